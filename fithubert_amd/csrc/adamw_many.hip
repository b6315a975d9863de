// One AdamW step over many tensors in one launch, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        g = grad * grad_scale
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The moments of all tensors lie in one flat buffer, every tensor padded to whole blocks of 256 elements.  A wave owns four
// neighbouring blocks, whatever tensors they belong to; where they are whole blocks of one tensor (nearly always) all loads of the four
// are in flight before the first is used.  The tensors travel as a table in the kernel's arguments (no device-side table to
// upload, so a captured launch is self-contained); a wave finds its tensor by counting, 64 entries per load, how many begin at or
// before its block.  More than FH_MANY tensors take several launches.
//
// 8 bits: m and r = sqrt(v) are held as e4m3 codes over one fp32 scale per block, its largest magnitude / 448.  The root is held
// instead of v because an e4m3 code spans 2^-9 .. 448 = 18.8 binades: for v itself that would lose elements whose gradients are
// 700 times smaller than their block's largest, for the root 5 * 10^5 times.  What is rounded is the new moment in fp32 -- the
// parameter moves by the unrounded one --, and it is rounded UP with the probability of its fraction: rounded to nearest, an
// average whose step (1 - b2) is far below a code's spacing of 1/16 would never leave its code.  That keeps the average of r, not of v = r^2, which gains the
// rounding's variance: under steady gradients v is held 1 % (b2 = 0.9) to 5 % (0.98, 0.99) too large on average and stays there, so steps are up to 2.5 % shorter.  The draws are 16 bits each of one
// hash of (seed, place), so a step can be repeated.  A root that is not zero never becomes zero (it divides).  An element that is
// not finite is held as the code's NaN and does not enter its block's scale: it harms itself alone, as it would in 32 bits.
// This file is compiled without contraction into fused multiply-adds: codes are a discontinuous function of the moments, and this
// way each is the same on every path and in any restatement that follows the formulas in fp32.
//
// Bound by HBM: 28 bytes per fp32 element with fp32 gradients and 32-bit moments, 16.06 with 8-bit ones, 10.06 with bf16 parameters and
// gradients.  Measured (a copy runs at 5.0 to 5.2 TB/s): 300 M bf16 parameters, 8-bit moments, 380 tensors: 596 us = 5.1 TB/s; 30 M fp32
// parameters, 8-bit moments, 200 tensors: 87 us of kernel time (two launches; 5.6 TB/s, some of its 488 MB stay in the last cache from pass to pass).  With the compiler's IEEE division and square
// root, a software rounding to e4m3 and four elements per lane everywhere the first took 934 us: the arithmetic was the bound, not the bytes.
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

// max over the 64 (HALF: over each 32) lanes of a wave, in every one of them: four lane rotations inside the rows of 16, then over the rows
template <bool HALF> __device__ __forceinline__ float wave_max_dpp(float v) {
#define FH_ROW_MAX(ctrl) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, false)))
  FH_ROW_MAX(0x121);  // row_ror:1
  FH_ROW_MAX(0x122);
  FH_ROW_MAX(0x124);
  FH_ROW_MAX(0x128);
#undef FH_ROW_MAX
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  if constexpr (HALF) return v;
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// square root to nearest: v_sqrt_f32 is off by one unit at most, and s is too large (small) when x lies below (above) the product of s and its
// neighbour.  (hipcc's own adds a rescue of x < 2^-96; there this one may be a unit off.)
__device__ __forceinline__ float sqrt_near(float x) {
  const float s = __builtin_amdgcn_sqrtf(x), dn = __uint_as_float(__float_as_uint(s) - 1u), up = __uint_as_float(__float_as_uint(s) + 1u);
  float y = __builtin_fmaf(-dn, s, x) <= 0.f ? dn : s;
  return __builtin_fmaf(-up, s, x) > 0.f ? up : y;
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

// The step on N neighbouring elements of a lane, whose block is the N / 4th part of a wave.  BITS = 8: m, v hold code values on entry, ms / vs the block's
// scales; `at`: the first element's place in the flat moments.
template <int BITS, int N>
__device__ __forceinline__ void update(const ManyArgs& a, float (&p)[N], const float (&g)[N], float (&m)[N], float (&v)[N], float& ms, float& vs, uint32_t at,
                                       int (&cm)[N / 4], int (&cr)[N / 4]) {
  float m_top = 0.f, r_top = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float gr = g[e] * a.gscale;
    if constexpr (BITS == 8) {
      const float r0 = v[e] * vs;
      m[e] = m[e] * ms;
      v[e] = r0 * r0;
    }
    m[e] = m[e] * a.b1 + gr * a.c1;
    v[e] = v[e] * a.b2 + (gr * gr) * a.c2;
    const float r = sqrt_near(v[e]);
    // (v_rcp_f32 is off by one unit: nothing beside the 2^-24 of the other steps, and a tenth of a division)
    p[e] = p[e] * a.decay - a.rate * (m[e] * __builtin_amdgcn_rcpf(r * a.rbc2 + a.eps));
    if constexpr (BITS == 8) {
      v[e] = r;
      m_top = fmaxf(m_top, fabsf(m[e]));   // (a NaN loses against any number)
      r_top = fmaxf(r_top, r);
    }
  }
  if constexpr (BITS == 8) {
    constexpr bool HALF = N == 8;
    m_top = wave_max_dpp<HALF>(m_top);
    r_top = wave_max_dpp<HALF>(r_top);
    if (__any(!(m_top < INFINITY) || !(r_top < INFINITY))) {   // an infinity somewhere: the largest of the others
      m_top = r_top = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        m_top = fmaxf(m_top, fabsf(m[e]) < INFINITY ? fabsf(m[e]) : 0.f);
        r_top = fmaxf(r_top, v[e] < INFINITY ? v[e] : 0.f);
      }
      m_top = wave_max_dpp<HALF>(m_top);
      r_top = wave_max_dpp<HALF>(r_top);
    }
    m_top = fmaxf(m_top, TINY);
    r_top = fmaxf(r_top, TINY);
    const float m_inv = (1.f / m_top) * E4M3_MAX, r_inv = (1.f / r_top) * E4M3_MAX;
    ms = m_top * (1.f / E4M3_MAX);
    vs = r_top * (1.f / E4M3_MAX);
    // v_cvt_sr_fp8_f32 adds the draw below the code's last bit and cuts: floor(|x| / spacing + draw), subnormal codes included; infinities and
    // NaN become the code's NaN.  The largest element comes to 448 (1 + 2 2^-24) at most, which no draw of 16 bits lifts to the next code.
#define FH_CODE(i, e)                                                                                                  \
  {                                                                                                                    \
    const uint32_t h = fh_mix32((at + 4 * i + e) ^ a.key);                                                             \
    const float x = v[4 * i + e] * r_inv;                                                                              \
    cm[i] = __builtin_amdgcn_cvt_sr_fp8_f32(m[4 * i + e] * m_inv, (int)(h << 16), cm[i], e);                           \
    cr[i] = __builtin_amdgcn_cvt_sr_fp8_f32(x > 0.f ? fmaxf(x, 0x1p-9f) : x, (int)(h & 0xffff0000u), cr[i], e);        \
  }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      cm[i] = cr[i] = 0;
      FH_CODE(i, 0) FH_CODE(i, 1) FH_CODE(i, 2) FH_CODE(i, 3)
    }
#undef FH_CODE
  }
}

template <int N> __device__ __forceinline__ void ld_codes(const uint8_t* p, int (&c)[N / 4]) {
  if constexpr (N == 8) {
    const int2 x = *(const int2*)p;
    c[0] = x.x; c[1] = x.y;
  } else {
    c[0] = *(const int*)p;
  }
}
template <int N> __device__ __forceinline__ void st_codes(uint8_t* p, const int (&c)[N / 4]) {
  if constexpr (N == 8) *(int2*)p = make_int2(c[0], c[1]);
  else *(int*)p = c[0];
}
template <typename T, int N> __device__ __forceinline__ void ld_n(const T* p, float (&f)[N]) {
  if constexpr (N == 8 && sizeof(T) == 2) {
    unpack16<T>(ld16(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) ld4(p + i, f + i);
  }
}
template <typename T, int N> __device__ __forceinline__ void st_n(T* p, const float (&f)[N]) {
  if constexpr (N == 8 && sizeof(T) == 2) {
    st16(p, pack16<T>(f));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) st4(p + i, f + i);
  }
}

// four whole blocks of one tensor, everything aligned: N elements per lane and step, all loads in front of the first use
template <typename P, typename G, int BITS, int N>
__device__ __forceinline__ void four_blocks(const ManyArgs& a, P* __restrict__ p_, const G* __restrict__ g_, void* __restrict__ m_, float* __restrict__ m_scale,
                                            void* __restrict__ v_, float* __restrict__ v_scale, long blk, int lane) {
  constexpr int STEPS = 16 / N, LB = 256 / N;   // lanes per block
  float p[STEPS][N], g[STEPS][N], m[STEPS][N], v[STEPS][N], ms[STEPS], vs[STEPS];
  int cm[STEPS][N / 4], cr[STEPS][N / 4];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int off = k * 64 * N + lane * N;
    const long at = blk * 256 + off, b = blk + k * (N / 4) + lane / LB;
    ld_n<G, N>(g_ + off, g[k]);
    ld_n<P, N>(p_ + off, p[k]);
    if constexpr (BITS == 8) {
      ld_codes<N>((const uint8_t*)m_ + at, cm[k]);
      ld_codes<N>((const uint8_t*)v_ + at, cr[k]);
      ms[k] = m_scale[b];
      vs[k] = v_scale[b];
    } else {
      ld_n<float, N>((const float*)m_ + at, m[k]);
      ld_n<float, N>((const float*)v_ + at, v[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int off = k * 64 * N + lane * N;
    const long at = blk * 256 + off, b = blk + k * (N / 4) + lane / LB;
    if constexpr (BITS == 8) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        float f[4];
        e4m3_values((uint32_t)cm[k][i], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) m[k][4 * i + e] = f[e];
        e4m3_values((uint32_t)cr[k][i], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][4 * i + e] = f[e];
      }
    }
    update<BITS, N>(a, p[k], g[k], m[k], v[k], ms[k], vs[k], (uint32_t)at, cm[k], cr[k]);
    st_n<P, N>(p_ + off, p[k]);
    if constexpr (BITS == 8) {
      st_codes<N>((uint8_t*)m_ + at, cm[k]);
      st_codes<N>((uint8_t*)v_ + at, cr[k]);
      if (lane % LB == 0) {
        m_scale[b] = ms[k];
        v_scale[b] = vs[k];
      }
    } else {
      st_n<float, N>((float*)m_ + at, m[k]);
      st_n<float, N>((float*)v_ + at, v[k]);
    }
  }
}

template <typename P, typename G, int BITS>
__global__ void __launch_bounds__(256) adamw_many_kernel(const ManyTable tab, const ManyArgs a, void* __restrict__ m_, float* __restrict__ m_scale,
                                                         void* __restrict__ v_, float* __restrict__ v_scale) {
  // 16-bit parameters with 8-bit moments: eight elements per lane, so that parameters and gradients move 16 bytes at a time
  constexpr int N = BITS == 8 && sizeof(P) == 2 ? 8 : 4;
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
  {
    const int first = tab.first[t], end = t + 1 < a.count ? tab.first[t + 1] : a.blocks;
    P* pt = (P*)tab.p[t];
    const G* gt = (const G*)tab.g[t];
    if (gt && b0 + WAVE_BLOCKS + (tab.tail[t] < 256) <= end && (((uintptr_t)pt & (N * sizeof(P) - 1) & 15) | ((uintptr_t)gt & (N * sizeof(G) - 1) & 15)) == 0) {
      const long off = (long)(b0 - first) * 256;
      four_blocks<P, G, BITS, N>(a, pt + off, gt + off, m_, m_scale, v_, v_scale, a.block0 + b0, lane);
      return;
    }
  }
  // the ends of tensors, short and unaligned ones: block by block
  for (int k = 0; k < WAVE_BLOCKS && b0 + k < a.blocks; ++k) {
    const int b = b0 + k;
    while (t + 1 < a.count && tab.first[t + 1] <= b) ++t;
    const G* gp = (const G*)tab.g[t];
    if (!gp) continue;
    const int last = (t + 1 < a.count ? tab.first[t + 1] : a.blocks) - 1;
    const long off = (long)(b - tab.first[t]) * 256 + lane * 4, blk = a.block0 + b, at = blk * 256 + lane * 4;
    const int cnt = max(0, min(4, (b < last ? 256 : (int)tab.tail[t]) - lane * 4));
    P* pp = (P*)tab.p[t] + off;
    const bool vec = (((uintptr_t)tab.p[t] & (4 * sizeof(P) - 1)) | ((uintptr_t)gp & (4 * sizeof(G) - 1))) == 0;
    float p[4], g[4], m[4], v[4], ms = 0.f, vs = 0.f;
    int cm[1] = {0}, cr[1] = {0};
    ld_upto4(gp + off, cnt, vec, g);
    ld_upto4((const P*)pp, cnt, vec, p);
    if constexpr (BITS == 8) {
      e4m3_values(*(const uint32_t*)((const uint8_t*)m_ + at), m);
      e4m3_values(*(const uint32_t*)((const uint8_t*)v_ + at), v);
      ms = m_scale[blk];
      vs = v_scale[blk];
    } else {
      ld4((const float*)m_ + at, m);
      ld4((const float*)v_ + at, v);
    }
    update<BITS, 4>(a, p, g, m, v, ms, vs, (uint32_t)at, cm, cr);
    st_upto4(pp, cnt, vec, p);
    if constexpr (BITS == 8) {
      *(int*)((uint8_t*)m_ + at) = cm[0];
      *(int*)((uint8_t*)v_ + at) = cr[0];
      if (lane == 0) {
        m_scale[blk] = ms;
        v_scale[blk] = vs;
      }
    } else {
      st4((float*)m_ + at, m);
      st4((float*)v_ + at, v);
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
