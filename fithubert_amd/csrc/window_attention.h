// What the entry points and the kernels of the window attention share: the problem as the kernels take it and how it is divided.
#pragma once
#include "common.cuh"

constexpr int FAR = 1 << 29;       // "no limit", and the largest position

struct WinArgs {
  int B, Tq, Tk, Hq, Hkv, G, dh, left, right, sinks;
  float scale, c;                  // c = scale log2(e)
  const int* key_len;
  const int* q_start;
  long q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs;
  int rows;                        // Tq * G
  int nsplit;                      // forward: workgroups that share a row block's keys; dk / dv: that share a sink block's rows
  int nsink;                       // dk / dv: key blocks that hold sinks
};

// Workgroups per row block: enough for every CU to hold a few, where the rows alone do not make them; at least two tiles of keys each.
static inline int fwd_splits(const WinArgs& a) {
  const long wgs = (long)a.B * a.Hkv * ((a.rows + 127) / 128), want = 768;
  const long span = (long)a.left + a.right + 128 / a.G + 1;
  const long tiles = ((span < a.Tk ? span : a.Tk) + 63) / 64 + (a.sinks + 63) / 64;
  long n = want / (wgs > 0 ? wgs : 1);
  if (n > tiles / 2) n = tiles / 2;
  return n < 2 ? 1 : n > 256 ? 256 : (int)n;
}
// sink blocks and the workgroups that share each one's rows
static inline void bwd_sinks(WinArgs& a) {
  a.nsink = (a.sinks + 127) / 128;
  long n = (a.rows + 1023) / 1024;
  a.nsplit = n < 1 ? 1 : n > 64 ? 64 : (int)n;
}
static inline size_t al16(size_t n) { return (n + 15) & ~(size_t)15; }

#define WIN_DECLARE(name)                                                                                                                     \
  int win_forward_##name(const WinArgs& a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st);  \
  int win_backward_##name(const WinArgs& a, const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, \
                          void* dq, void* dk, void* dv, char* scratch, hipStream_t st);
WIN_DECLARE(f32)
WIN_DECLARE(bf16)
WIN_DECLARE(f16)
#undef WIN_DECLARE
