// What the entry points and the kernels of the window attention share: the problem as the kernels take it and how it is divided.
#pragma once
#include "common.cuh"

constexpr int FAR = 1 << 29;             // more than the keys or the rows of an entry
constexpr int NO_LIMIT = 0x7fffffff;     // of left or right

struct WinArgs {
  int B, Tq, Tk, Hq, Hkv, G, dh, left, right, sinks;
  float scale, c;                  // c = scale log2(e)
  const int* key_len;
  const int* q_start;
  long q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs;
  int rows;                        // Tq * G
  unsigned magic;                  // floor(2^32 / G) + 1 (G = 1: 0)
  int nsplit;                      // forward: workgroups that share a row block's keys; dk / dv: that share a sink block's rows
  int nsink;                       // dk / dv: key blocks that hold sinks, where several workgroups share each
  // frame of a row (row < 2^29: the product is at most one too large)
  __device__ __forceinline__ int frame(int row) const {
    if (magic == 0u) return row;
    const int f = (int)__umulhi((unsigned)row, magic);
    return f * G > row ? f - 1 : f;
  }
  // The position of entry b's first row, clipped to +- FAR, and left and right as they are from there: what counts is where the first row's view begins and ends, and an end
  // clipped to +- FAR, past all keys whatever the row, hides and shows the same.  Sums and differences of positions, limits and keys then fit 32 bits.
  __device__ __forceinline__ int enter(int b) {
    const int first = q_start ? q_start[b] : 0, base = max(-FAR, min(FAR, first));
    left = left == NO_LIMIT ? base + FAR : base - (int)max((long)-FAR, min((long)FAR, (long)first - left));
    right = right == NO_LIMIT ? FAR - base : (int)max((long)-FAR, min((long)FAR, (long)first + right)) - base;
    return base;
  }
};

// How a forward call is laid out.  few: at most 32 rows per key head (win_few_kernel); otherwise rt 16-row tiles per wave, four waves; nsplit workgroups
// share each row block's keys.
struct WinPlan { int few, rt, nsplit; };
static inline WinPlan fwd_plan(const WinArgs& a, int dtype) {
  WinPlan p;
  const long heads = (long)a.B * a.Hkv, blocks2 = heads * ((a.rows + 127) / 128), blocks1 = heads * ((a.rows + 63) / 64);
  const long span = (long)a.left + a.right + 128 / a.G + 1;
  const long tiles = ((span < a.Tk ? span : a.Tk) + 63) / 64 + (a.sinks + 63) / 64;   // 64-key tiles that a row block sees
  p.few = a.rows <= (dtype == 0 && a.dh > 64 ? 16 : 32);   // (wide fp32 heads of 32 rows outgrow its registers)
  // 128-row blocks halve the reads of K and V; 64-row ones where those would leave CUs without work and the walk is short
  p.rt = !p.few && blocks2 < 512 && tiles < 16 ? 1 : 2;
  const long wgs = p.few ? heads : p.rt == 2 ? blocks2 : blocks1;
  // one workgroup per CU at least; a share is worth its join from eight tiles on (a wave's tiles of the few-row kernel: two)
  long n = wgs >= 256 ? 1 : (a.dh > 64 && !p.few ? 256 : 512) / (wgs > 0 ? wgs : 1);
  if (n > tiles / 8) n = tiles / 8;
  p.nsplit = n < 2 ? 1 : n > 256 ? 256 : (int)n;
  return p;
}
// Sink blocks (of `keys` keys) and the workgroups that share each one's rows: one per 1024 rows, but no more than four per CU in all -- where sinks are many their blocks fill the chip
// by themselves, and the shares' partial sums would only be written and read (30001 frames, all of them sinks, 4 key heads: 3.9 GB).  A block that nobody shares is
// one like the others: no partial sums, no join.
static inline void bwd_sinks(WinArgs& a, int keys) {
  a.nsink = (a.sinks + keys - 1) / keys;
  const long blocks = (long)a.B * a.Hkv * a.nsink, fill = blocks > 0 ? (1023 + blocks) / blocks : 1;
  long n = (a.rows + 1023) / 1024;
  if (n > 64) n = 64;
  if (n > fill) n = fill;
  if (n < 2) a.nsink = 0;
  a.nsplit = n < 2 ? 1 : (int)n;
}
// 16-key (16-row) tiles per wave of the backward passes: two where that still gives every CU two workgroups, and where the accumulators fit
static inline int bwd_tiles(const WinArgs& a, int dtype, long blocks128, bool dkv) {
  return dtype != 0 && a.dh <= (dkv ? 64 : 96) && blocks128 >= 512 ? 2 : 1;
}
static inline int dkv_keys(const WinArgs& a, int dtype) { return 64 * bwd_tiles(a, dtype, (long)a.B * a.Hkv * ((a.Tk + 127) / 128), true); }
static inline size_t al16(size_t n) { return (n + 15) & ~(size_t)15; }

#define WIN_DECLARE(name)                                                                                                                     \
  int win_forward_##name(const WinArgs& a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st);  \
  int win_backward_##name(const WinArgs& a, const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, \
                          void* dq, void* dk, void* dv, char* scratch, hipStream_t st);
WIN_DECLARE(f32)
WIN_DECLARE(bf16)
WIN_DECLARE(f16)
#undef WIN_DECLARE
