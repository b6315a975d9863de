// One AdamW step over many tensors in one launch, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        g = grad * grad_scale
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The moments of all tensors lie in one flat buffer, every tensor padded to whole blocks of 256 elements.  A wave owns four
// neighbouring blocks, whatever tensors they belong to: a lane holds four consecutive elements of each, and all loads of the four
// blocks are in flight before the first is used.  The tensors travel as a table in the kernel's arguments (no device-side table to
// upload, so a captured launch is self-contained); a wave finds its tensor by counting, 64 entries per load, how many begin at or
// before its block.  More than FH_MANY tensors take several launches.
//
// 8 bits: m and r = sqrt(v) are held as e4m3 codes over one fp32 scale per block, its largest magnitude / 448.  The root is held
// instead of v because an e4m3 code spans 2^-9 .. 448 = 18.8 binades: for v itself that would lose elements whose gradients are
// 700 times smaller than their block's largest, for the root 5 * 10^5 times.  What is rounded is the new moment in fp32 -- the
// parameter moves by the unrounded one --, and it is rounded UP with the probability of its fraction: rounded to nearest, an
// average whose step (1 - b2) is far below a code's spacing of 1/16 would never leave its code.  The draws are 16 bits each of one
// hash of (seed, place), so a step can be repeated.  A root that is not zero never becomes zero (it divides).  An element that is
// not finite is held as the code's NaN and does not enter its block's scale: it harms itself alone, as it would in 32 bits.
// This file is compiled without contraction into fused multiply-adds: codes are a discontinuous function of the moments, and this
// way each is the same on every path and in any restatement that follows the formulas in fp32.
//
// Bound by HBM: 28 bytes per fp32 element with fp32 gradients and 32-bit moments, 16.06 with 8-bit ones, 10.06 with bf16 parameters
// and gradients.
#include "common.cuh"
#include "kernels.h"
#include <cmath>

namespace {

constexpr int FH_MANY = 160;      // tensors per launch: 22 bytes each, the table stays below the 4 KiB of a launch's arguments
constexpr int WAVE_BLOCKS = 4;    // blocks of 256 elements per wave
constexpr int WG_BLOCKS = 4 * WAVE_BLOCKS;
constexpr float E4M3_MAX = 448.f, TINY = 1e-30f;  // (TINY: the reciprocal of an empty block's scale stays finite)

struct ManyTable {
  void* p[FH_MANY];
  const void* g[FH_MANY];         // null: the tensor and its moments are left as they are
  int first[FH_MANY];             // first block of each tensor, counted from this launch's first
  unsigned short tail[FH_MANY];   // elements of its last block
};
struct ManyArgs {
  float b1, c1, b2, c2, eps, decay, rate, rbc2, gscale;  // c = 1 - b, decay = 1 - lr wd, rate = lr / bias correction, rbc2 = 1 / sqrt(bias correction)
  uint32_t key;
  int count, blocks;
  long block0;                    // this launch's first block in the flat moments
};

__device__ __forceinline__ float wave_max_dpp(float v) {
  // max over the 16 lanes of a row by four lane rotations inside the row, then over the rows
#define FH_ROW_MAX(ctrl) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, false)))
  FH_ROW_MAX(0x121);  // row_ror:1
  FH_ROW_MAX(0x122);
  FH_ROW_MAX(0x124);
  FH_ROW_MAX(0x128);
#undef FH_ROW_MAX
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// |x| * inv as an e4m3 code, rounded up where its fraction exceeds 1 - u; the quantum is 2^(e - 3), e >= -6 (subnormal codes below)
__device__ __forceinline__ uint32_t e4m3_code(float x, float inv, float u) {
  const float a = fabsf(x) * inv;
  const uint32_t ex = max(__float_as_uint(a) >> 23, 121u);
  const float k = floorf(a * __uint_as_float((257u - ex) << 23) + u);   // a / 2^(ex - 130): exact, below 16
  const uint32_t c = min(((ex - 120u) << 3) + (uint32_t)k - 8u, 0x7eu);
  return c | ((__float_as_uint(x) >> 24) & 0x80u);
}
__device__ __forceinline__ void e4m3_values(uint32_t c, float (&f)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  f[0] = lo[0]; f[1] = lo[1]; f[2] = hi[0]; f[3] = hi[1];
}

template <typename T> __device__ __forceinline__ void ld_upto4(const T* p, int cnt, bool vec, float (&f)[4]) {
  if (cnt >= 4 && vec) {
    ld4(p, f);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = e < cnt ? to_f(p[e]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void st_upto4(T* p, int cnt, bool vec, const float (&f)[4]) {
  if (cnt >= 4 && vec) {
    st4(p, f);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < cnt) p[e] = from_f<T>(f[e]);
  }
}

template <typename P, typename G, int BITS>
__global__ void __launch_bounds__(256) adamw_many_kernel(const ManyTable tab, const ManyArgs a, void* __restrict__ m_, float* __restrict__ m_scale,
                                                         void* __restrict__ v_, float* __restrict__ v_scale) {
  const int lane = threadIdx.x & 63;
  const int b0 = __builtin_amdgcn_readfirstlane(blockIdx.x * WG_BLOCKS + (threadIdx.x >> 6) * WAVE_BLOCKS);
  if (b0 >= a.blocks) return;
  int t = -1;                     // tensor of block b0: the last one that begins at or before it (empty tensors begin where the next does)
#pragma unroll
  for (int i = 0; i < (FH_MANY + 63) / 64; ++i) {
    const int j = i * 64 + lane;
    t += __popcll(__ballot(j < a.count && tab.first[min(j, FH_MANY - 1)] <= b0));
  }
  t = __builtin_amdgcn_readfirstlane(t);
  float p[WAVE_BLOCKS][4], g[WAVE_BLOCKS][4], m[WAVE_BLOCKS][4], v[WAVE_BLOCKS][4], ms[WAVE_BLOCKS], vs[WAVE_BLOCKS];
  uint32_t mc[WAVE_BLOCKS], vc[WAVE_BLOCKS];
  P* pp[WAVE_BLOCKS];
  int cnt[WAVE_BLOCKS];
  bool vec[WAVE_BLOCKS];
#pragma unroll
  for (int k = 0; k < WAVE_BLOCKS; ++k) {
    const int b = b0 + k;
    cnt[k] = -1;                  // (-1: nothing to do here)
    if (b < a.blocks) {
      while (t + 1 < a.count && tab.first[t + 1] <= b) ++t;
      const G* gp = (const G*)tab.g[t];
      if (gp) {
        const int last = (t + 1 < a.count ? tab.first[t + 1] : a.blocks) - 1;
        const long off = (long)(b - tab.first[t]) * 256 + lane * 4;
        const int in_block = b < last ? 256 : (int)tab.tail[t];
        pp[k] = (P*)tab.p[t] + off;
        cnt[k] = max(0, min(4, in_block - lane * 4));
        vec[k] = (((uintptr_t)tab.p[t] & (4 * sizeof(P) - 1)) | ((uintptr_t)gp & (4 * sizeof(G) - 1))) == 0;
        ld_upto4(gp + off, cnt[k], vec[k], g[k]);
        ld_upto4((const P*)pp[k], cnt[k], vec[k], p[k]);
        const long at = (a.block0 + b) * 256 + lane * 4;
        if constexpr (BITS == 8) {
          mc[k] = *(const uint32_t*)((const uint8_t*)m_ + at);
          vc[k] = *(const uint32_t*)((const uint8_t*)v_ + at);
          ms[k] = m_scale[a.block0 + b];
          vs[k] = v_scale[a.block0 + b];
        } else {
          ld4((const float*)m_ + at, m[k]);
          ld4((const float*)v_ + at, v[k]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < WAVE_BLOCKS; ++k) {
    if (cnt[k] < 0) continue;
    const long blk = a.block0 + b0 + k, at = blk * 256 + lane * 4;
    if constexpr (BITS == 8) {
      e4m3_values(mc[k], m[k]);
      e4m3_values(vc[k], v[k]);
    }
    float r[4], m_top = 0.f, r_top = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gr = g[k][e] * a.gscale;
      if constexpr (BITS == 8) {
        const float r0 = v[k][e] * vs[k];
        m[k][e] = m[k][e] * ms[k];
        v[k][e] = r0 * r0;
      }
      m[k][e] = m[k][e] * a.b1 + gr * a.c1;
      v[k][e] = v[k][e] * a.b2 + (gr * gr) * a.c2;
      r[e] = sqrtf(v[k][e]);
      p[k][e] = p[k][e] * a.decay - a.rate * (m[k][e] / (r[e] * a.rbc2 + a.eps));
      if constexpr (BITS == 8) {
        m_top = fmaxf(m_top, finite(m[k][e]) ? fabsf(m[k][e]) : 0.f);
        r_top = fmaxf(r_top, finite(r[e]) ? r[e] : 0.f);
      }
    }
    st_upto4(pp[k], cnt[k], vec[k], p[k]);
    if constexpr (BITS == 8) {
      m_top = fmaxf(wave_max_dpp(m_top), TINY);
      r_top = fmaxf(wave_max_dpp(r_top), TINY);
      const float m_inv = (1.f / m_top) * E4M3_MAX, r_inv = (1.f / r_top) * E4M3_MAX;
      uint32_t cm = 0, cr = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t h = fh_mix32(((uint32_t)at + e) ^ a.key);
        uint32_t x = e4m3_code(m[k][e], m_inv, (float)(h & 0xffffu) * (1.f / 65536.f));
        uint32_t y = e4m3_code(r[e], r_inv, (float)(h >> 16) * (1.f / 65536.f));
        if (r[e] > 0.f && y == 0u) y = 1u;
        if (!finite(m[k][e])) x = 0x7fu;
        if (!finite(r[e])) y = 0x7fu;
        cm |= x << (8 * e);
        cr |= y << (8 * e);
      }
      *(uint32_t*)((uint8_t*)m_ + at) = cm;
      *(uint32_t*)((uint8_t*)v_ + at) = cr;
      if (lane == 0) {
        m_scale[blk] = m_top * (1.f / E4M3_MAX);
        v_scale[blk] = r_top * (1.f / E4M3_MAX);
      }
    } else {
      st4((float*)m_ + at, m[k]);
      st4((float*)v_ + at, v[k]);
    }
  }
}

template <typename P, typename G> int launch_pg(const ManyTable& tab, const ManyArgs& a, int bits, void* m, float* ms, void* v, float* vs, hipStream_t st) {
  const dim3 grid((unsigned)((a.blocks + WG_BLOCKS - 1) / WG_BLOCKS)), block(256);
  if (bits == 8) hipLaunchKernelGGL((adamw_many_kernel<P, G, 8>), grid, block, 0, st, tab, a, m, ms, v, vs);
  else hipLaunchKernelGGL((adamw_many_kernel<P, G, 32>), grid, block, 0, st, tab, a, m, ms, v, vs);
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename P> int launch_p(int gdt, const ManyTable& tab, const ManyArgs& a, int bits, void* m, float* ms, void* v, float* vs, hipStream_t st) {
  if (gdt == 0) return launch_pg<P, float>(tab, a, bits, m, ms, v, vs, st);
  if (gdt == 1) return launch_pg<P, bf16>(tab, a, bits, m, ms, v, vs, st);
  return launch_pg<P, f16>(tab, a, bits, m, ms, v, vs, st);
}

}  // namespace

extern "C" {

long fh_adamw_many_blocks(const long* n, int count) {
  if (count < 0 || (count > 0 && !n)) return -1;
  long blocks = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0) return -1;
    blocks += (n[i] + 255) / 256;
  }
  return blocks;
}

int fh_adamw_many(int p_dtype, int g_dtype, void* const* p, const void* const* g, const long* n, int count, int bits, void* m, float* m_scale,
                  void* v, float* v_scale, double lr, double beta1, double beta2, double eps, double wd, long step, double grad_scale,
                  uint32_t seed, fh_stream_t stream) {
  if (p_dtype < 0 || p_dtype > 2 || g_dtype < 0 || g_dtype > 2) return -901;
  if (bits != 8 && bits != 32) return -902;
  if (count < 0 || step < 1) return -903;
  if (count > 0 && (!p || !g || !n)) return -904;
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1)) return -905;
  long total = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || (n[i] > 0 && g[i] && !p[i])) return -904;
    if ((uintptr_t)p[i] % fh_esize(p_dtype) || (uintptr_t)g[i] % fh_esize(g_dtype)) return -906;
    total += (n[i] + 255) / 256;
  }
  if (total == 0) return 0;
  if (!m || !v || (bits == 8 && (!m_scale || !v_scale))) return -904;
  if (((uintptr_t)m | (uintptr_t)v) & 15) return -906;
  ManyArgs a;
  a.b1 = (float)beta1; a.c1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2; a.c2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.decay = (float)(1.0 - lr * wd);
  a.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
  a.rbc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  a.gscale = (float)grad_scale;
  uint32_t key = seed * 0x9E3779B9u + 0x27D4EB2Fu;  // fh_mix32 on the host
  key ^= key >> 16; key *= 0x7feb352dU; key ^= key >> 15; key *= 0x846ca68bU; key ^= key >> 16;
  a.key = key;
  ManyTable tab;
  long block0 = 0;
  for (int i = 0; i < count;) {
    // as many tensors as the table holds and a launch's block count can count
    a.count = 0;
    a.block0 = block0;
    long blocks = 0;
    while (i < count && a.count < FH_MANY) {
      const long nb = (n[i] + 255) / 256;
      if (nb > 0x3fffffffL) return -903;  // one tensor of more than 2^38 elements
      if (blocks + nb > 0x3fffffffL) break;
      const int j = a.count++;
      tab.p[j] = p[i];
      tab.g[j] = n[i] > 0 ? g[i] : nullptr;
      tab.first[j] = (int)blocks;
      tab.tail[j] = (unsigned short)(n[i] - (nb - 1) * 256);
      blocks += nb;
      ++i;
    }
    a.blocks = (int)blocks;
    block0 += blocks;
    if (blocks == 0) continue;
    int rc;
    if (p_dtype == 0) rc = launch_p<float>(g_dtype, tab, a, bits, m, m_scale, v, v_scale, (hipStream_t)stream);
    else if (p_dtype == 1) rc = launch_p<bf16>(g_dtype, tab, a, bits, m, m_scale, v, v_scale, (hipStream_t)stream);
    else rc = launch_p<f16>(g_dtype, tab, a, bits, m, m_scale, v, v_scale, (hipStream_t)stream);
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
