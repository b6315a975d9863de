// Entry points of the window attention: checks, the scratch they need, the choice of the element type (kernels: window_attention.cuh).
#include "window_attention.h"

namespace {

int check(int dtype, const fh_window_attention_desc* d) {
  if (dtype < 0 || dtype > 2) return -921;
  if (!d || d->B < 0 || d->Tq < 0 || d->Tk < 0 || d->Hq < 1 || d->Hkv < 1 || d->Hq % d->Hkv) return -922;
  if (d->dh < 8 || d->dh > 128 || d->dh % 8) return -923;
  if (d->B > 65535 || d->Hkv > 65535 || d->Tq >= FAR || d->Tk >= FAR || (long)d->Tq * (d->Hq / d->Hkv) >= FAR) return -924;
  if (!(d->scale > 0.f) || !(d->scale < INFINITY)) return -925;
  // a 64-row tile's places are 32-bit byte offsets from its first row
  const long far = 1 << 23, st[6] = {d->q_ts, d->q_hs, d->k_ts, d->k_hs, d->v_ts, d->v_hs};
  for (long x : st)
    if (x < 0 || x > far) return -929;
  if (d->q_bs < 0 || d->k_bs < 0 || d->v_bs < 0 || (long)d->Hq * d->dh > far) return -929;
  const long vec = dtype == 0 ? 4 : 8;
  if ((d->q_bs | d->q_ts | d->q_hs | d->k_bs | d->k_ts | d->k_hs | d->v_bs | d->v_ts | d->v_hs) % vec) return -926;
  return 0;
}
WinArgs args_of(const fh_window_attention_desc* d) {
  WinArgs a;
  a.B = d->B; a.Tq = d->Tq; a.Tk = d->Tk; a.Hq = d->Hq; a.Hkv = d->Hkv; a.G = d->Hq / d->Hkv; a.dh = d->dh;
  a.left = d->left < 0 ? NO_LIMIT : d->left;
  a.right = d->right < 0 ? NO_LIMIT : d->right;
  a.sinks = d->sinks < 0 ? 0 : d->sinks > d->Tk ? d->Tk : d->sinks;
  a.scale = d->scale;
  a.c = d->scale * 1.4426950408889634f;
  a.key_len = d->key_len; a.q_start = d->q_start;
  a.q_bs = d->q_bs; a.q_ts = d->q_ts; a.q_hs = d->q_hs;
  a.k_bs = d->k_bs; a.k_ts = d->k_ts; a.k_hs = d->k_hs;
  a.v_bs = d->v_bs; a.v_ts = d->v_ts; a.v_hs = d->v_hs;
  a.rows = d->Tq * a.G;
  a.magic = a.G == 1 ? 0u : (unsigned)(0x100000000ull / (unsigned)a.G) + 1u;
  a.nsplit = 1;
  a.nsink = 0;
  return a;
}

}  // namespace

extern "C" {

long fh_window_attention_scratch_bytes(int dtype, const fh_window_attention_desc* d, int backward) {
  if (check(dtype, d)) return -1;
  WinArgs a = args_of(d);
  if (!backward) {
    const int n = fwd_plan(a, dtype).nsplit;
    return n > 1 ? (long)a.B * a.Hkv * n * a.rows * (a.dh + 2) * 4 : 0;
  }
  const int keys = dkv_keys(a, dtype);
  bwd_sinks(a, keys);
  return (long)al16((size_t)a.B * a.Tq * a.Hq * 4) + (long)a.B * a.Hkv * a.nsink * a.nsplit * 2 * keys * a.dh * 4;
}

int fh_window_attention_forward(int dtype, const fh_window_attention_desc* d, const void* q, const void* k, const void* v, void* out,
                                float* lse, void* scratch, fh_stream_t stream) {
  if (int rc = check(dtype, d)) return rc;
  const WinArgs a = args_of(d);
  if (a.B == 0 || a.Tq == 0) return 0;
  if (!q || !out || (a.Tk > 0 && (!k || !v))) return -927;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)scratch) & 15) return -926;
  if (fh_window_attention_scratch_bytes(dtype, d, 0) > 0 && !scratch) return -928;
  return (dtype == 0 ? win_forward_f32 : dtype == 1 ? win_forward_bf16 : win_forward_f16)(a, q, k, v, out, lse, (float*)scratch, (hipStream_t)stream);
}

int fh_window_attention_backward(int dtype, const fh_window_attention_desc* d, const void* q, const void* k, const void* v, const void* out,
                                 const void* dout, const float* lse, void* dq, void* dk, void* dv, void* scratch, fh_stream_t stream) {
  if (int rc = check(dtype, d)) return rc;
  const WinArgs a = args_of(d);
  if (a.B == 0 || (a.Tq == 0 && a.Tk == 0)) return 0;
  if ((a.Tq > 0 && (!q || !out || !dout || !lse || !dq)) || (a.Tk > 0 && (!k || !v || !dk || !dv))) return -927;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)scratch) & 15) return -926;
  if (fh_window_attention_scratch_bytes(dtype, d, 1) > 0 && !scratch) return -928;
  return (dtype == 0 ? win_backward_f32 : dtype == 1 ? win_backward_bf16 : win_backward_f16)(a, q, k, v, out, dout, lse, dq, dk, dv, (char*)scratch,
                                                                                              (hipStream_t)stream);
}

}  // extern "C"
