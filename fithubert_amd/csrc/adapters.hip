// Low-rank adapters of many requests beside one frozen projection, forward and backward.
//
//   h = s_a x A_a^T          y  = x W^T + bias + h B_a^T          a: the adapter of the row's segment
//   G = s_a dy B_a           dx = dy W + G A_a          dA_a = sum over a's rows G^T x          dB_a = sum over a's rows dy^T h
//
// down:   h and G.  A workgroup owns 16 (long batches: 32) rows, its four waves split the long reduction (K or N) and join in LDS: one pass over x (dy), many
//         short workgroups, so that a handful of rows is as quick as its longest load chain.  Rows of several segments: one trip per segment
//         that the tile touches, dealt over grid.y where requests are short.  Bound by the reads of x (dy).
// y, dx:  the shared projection's product, the adapters' part added to its accumulators (see `project`); short requests' part by `up`, added as the
//         GEMM's residual operand.
// outer:  dA and dB in one launch: a workgroup owns 64 columns of one adapter's factor and walks that adapter's rows, whichever segments they lie in, 32
//         at a time per wave; long walks are dealt over several workgroups whose partial sums are added in order (no atomics).
// Rounding in 16-bit modes: h and G, which are the next products' operands.  Sums are fp32 and y (dx) is rounded once, the adapters' part being added inside the projection's product; but
// for many short requests (see `project`) the part is a residual operand and rounded on its way to it.
// Measured, warm, forward and backward of 16384 x 1024 -> 4096, rank 16, 4 adapters, 32 requests, bf16: h 11 us, y 122 (1.12 PFLOP/s of the projection alone), turn 5, G 45 (134 MB, 3.0 TB/s), dx 121,
// dA and dB 26 + 5; the call 322.  Forward of 9973 x 480 -> 1440, rank 8: 6 + 27 us, the call 28 -- 234 tiles of 256 x 256 for 256 CUs, each with eight steps of K: bound by filling and emptying
// one tile.  32 one-row requests, 768 -> 768, fp16: 4.9 + 6.7 us.  fp32, 1497 x 480 -> 480, rank 32, both directions: 70 us of kernels (y 19, dx 21, the rest 4 to 8 each).
#include "gemm_loops.cuh"
#include "kernels.h"
#include "attn_frag.cuh"

int fh_gemm_path_bf16(const GemmParams& p, int path, hipStream_t stream);  // gemm_bf16.hip
int fh_gemm_path_f16(const GemmParams& p, int path, hipStream_t stream);   // gemm_f16.hip

namespace {

struct Segs {
  const int* start;
  const int* which;
  const float* scaling;
  int n, adapters, M;
  __device__ __forceinline__ int begin(int s) const { return max(0, min(M, start[s])); }
  __device__ __forceinline__ int adapter(int s) const { const int a = which[s]; return a >= 0 && a < adapters ? a : -1; }
  // number of segments that end at or before `row`: the first one that may hold it.  The 64 lanes look at 64 places at a time.
  __device__ __forceinline__ int first_at(int row, int lane) const {
    int lo = 0, len = n;
    while (len > 0) {
      const int step = (len + 63) >> 6, at = lo + lane * step + step - 1;
      const int passed = __popcll(__ballot(at < lo + len && start[min(at, n - 1) + 1] <= row));
      lo += passed * step;
      len = step > 1 ? min(step - 1, lo + step - 1 > n ? n - lo : step - 1) : 0;
    }
    return __builtin_amdgcn_readfirstlane(min(lo, n));
  }
};

// The factors the other way round, for the backward pass: At[a][k][r] = A_a[r][k] and Bt[a][r][n] = B_a[n][r], 64 x 64 elements per workgroup.  (Gathered in place the
// products' fragments are eight loads each: down's product with dy took 47 us of them at 16384 x 4096, 16 adapter columns, against 30.)
template <typename T>
__global__ void __launch_bounds__(256) adapter_turn_kernel(const T* __restrict__ fa, const T* __restrict__ fb, T* __restrict__ ta, T* __restrict__ tb, int K, int N, int R) {
  __shared__ T tile[64][65];
  const int rt = (R + 63) / 64, na = rt * ((K + 63) / 64);
  const bool is_a = (int)blockIdx.x < na;
  const int n = is_a ? blockIdx.x : blockIdx.x - na, rows = is_a ? R : N, cols = is_a ? K : R;
  const int ct = (cols + 63) / 64, r0 = n / ct * 64, c0 = n % ct * 64;
  const long off = (long)blockIdx.y * rows * cols;
  const T* src = (is_a ? fa : fb) + off;
  T* dst = (is_a ? ta : tb) + off;
  const int c = threadIdx.x & 63;
  T v[16];   // (all loads in flight at once; those past the edge repeat the last row or column and are not stored)
  const T* at = src + min(c0 + c, cols - 1);
#pragma unroll
  for (int u = 0; u < 16; ++u) v[u] = at[(long)min(r0 + (int)(threadIdx.x >> 6) + 4 * u, rows - 1) * cols];
#pragma unroll
  for (int u = 0; u < 16; ++u) tile[(threadIdx.x >> 6) + 4 * u][c] = v[u];
  __syncthreads();
  for (int r = threadIdx.x >> 6; r < 64; r += 4)
    if (c0 + r < cols && r0 + c < rows) dst[(long)(c0 + r) * rows + r0 + c] = tile[c][r];
}

// out[row][r] = scaling[a] * sum_k x[row][k] f[a][r][k]   (h: f = A; G: f = Bt).  RT 16-row tiles per workgroup share the reads of f; a wave takes 128 bytes of
// every row at a time.
template <typename T, int NR, int RT>
__global__ void __launch_bounds__(256) adapter_down_kernel(const Segs g, const T* __restrict__ x, const T* __restrict__ f, T* __restrict__ out, int K, int R) {
  constexpr int KD = AT<T>::KD, VEC = ElemTraits<T>::VEC;
  typedef typename AT<T>::frag frag;
  __shared__ f32x4 part[4][NR * RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int i0 = blockIdx.x * 16 * RT, i1 = min(i0 + 16 * RT, g.M);
  const int s0 = g.first_at(i0, lane);
  if (blockIdx.y == 0) {
    // rows that no adapter's segment holds: zero (their own store below never comes)
    for (int n = threadIdx.x; n < 16 * RT * NR; n += 256) {
      const int row = i0 + n % (16 * RT), c = n / (16 * RT) * 16;
      if (row >= i1) continue;
      int s = s0;
      while (s < g.n && g.start[s + 1] <= row) ++s;
      if (s >= g.n || g.start[s] > row || g.adapter(s) < 0)
        for (int j = c; j < min(c + 16, R); ++j) out[(long)row * R + j] = from_f<T>(0.f);
    }
  }
  auto piece = [](const T* p, bool live) {
    union { V16 v; frag f; } u;
    u.v = v16_zero();
    if (live) u.v = ld16(p);
    return u.f;
  };
  bool more = true;   // (a segment that reaches i1 is the last: the next one need not be looked at)
  for (int s = s0 + (int)blockIdx.y; s < g.n && more; s += (int)gridDim.y) {
    const int begin = g.begin(s), end = g.begin(s + 1), a = g.adapter(s), b = max(begin, i0), e = min(end, i1);
    more = end < i1;
    if (b >= e || a < 0) continue;
    const T* fa = f + (long)a * K * R;
    const T* xr[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) xr[t] = x + (long)min(i0 + 16 * t + r, g.M - 1) * K;
    f32x4 acc[NR][RT];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int k = wave * 2 * KD; k < K; k += 8 * KD) {
      frag fx[2][RT], ff[2][NR];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k0 = k + u * KD + VEC * q;
#pragma unroll
        for (int t = 0; t < RT; ++t) fx[u][t] = piece(xr[t] + k0, k0 < K);
#pragma unroll
        for (int n = 0; n < NR; ++n) ff[u][n] = piece(fa + (long)(16 * n + r) * K + k0, 16 * n + r < R && k0 < K);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[n][t] = mma<T>(fx[u][t], ff[u][n], acc[n][t]);
    }
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int t = 0; t < RT; ++t) part[wave][n * RT + t][lane] = acc[n][t];
    __syncthreads();
    const float sc = g.scaling[a];
    for (int m = wave; m < NR * RT; m += 4) {
      f32x4 v = part[0][m][lane];
#pragma unroll
      for (int w = 1; w < 4; ++w)
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] += part[w][m][lane][c];
      const int col = 16 * (m / RT) + r;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int row = i0 + 16 * (m % RT) + 4 * q + c;
        if (row >= b && row < e && col < R) out[(long)row * R + col] = from_f<T>(v[c] * sc);   // rounded to the element type: the next product's operand
      }
    }
    __syncthreads();
  }
}

// out[i][j] = sum_r h[i][r] f[a][j][r], 0 for rows without an adapter   (y's part: f = B; dx's: f = At)
template <typename T>
__global__ void __launch_bounds__(256) adapter_up_kernel(const Segs g, const T* __restrict__ h, const T* __restrict__ f, T* __restrict__ out, int N, int R) {
  constexpr int KD = AT<T>::KD, VEC = ElemTraits<T>::VEC;
  typedef typename AT<T>::frag frag;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int i0 = blockIdx.x * 16, j0 = blockIdx.y * 256 + wave * 64, i1 = min(i0 + 16, g.M);
  if (j0 >= N) return;
  f32x4 acc[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  bool more = true;   // (a segment that reaches i1 is the last: the next one need not be looked at)
  for (int s = g.first_at(i0, threadIdx.x & 63); s < g.n && more; ++s) {
    const int begin = g.begin(s), end = g.begin(s + 1), a = g.adapter(s), b = max(begin, i0), e = min(end, i1);
    more = end < i1;
    if (b >= e || a < 0) continue;
    const T* fa = f + (long)a * N * R;
    const bool mine = i0 + r >= b && i0 + r < e;
    for (int k = 0; k < R; k += KD) {
      const int k0 = k + VEC * q;
      frag fh = zero_frag((frag*)nullptr);
      if (mine && k0 < R) {
        union { V16 v; frag f; } u;
        u.v = ld16(h + (long)(i0 + r) * R + k0);
        fh = u.f;
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int col = j0 + 16 * n + r;
        frag ff;
        ff = zero_frag((frag*)nullptr);
        if (col < N && k0 < R) {
          union { V16 v; frag f; } u;
          u.v = ld16(fa + (long)col * R + k0);
          ff = u.f;
        }
        // transposed: a lane holds four neighbouring columns of one row; rows of other requests keep their sum (a zero times this adapter's infinity would reach them)
        const f32x4 t = mma<T>(ff, fh, acc[n]);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[n][c] = mine ? t[c] : acc[n][c];
      }
    }
  }
  const int row = i0 + r;
  if (row < i1) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int col = j0 + 16 * n + 4 * q;
      float v[4] = {acc[n][0], acc[n][1], acc[n][2], acc[n][3]};
      if (col < N) st4(out + (long)row * N + col, v);
    }
  }
}

// The same products added to a wave's accumulators of the projection's GEMM, between its main loop and its epilogue: one rounding for the whole of y (dx), and
// no pass over it.
template <typename T> struct AdapterExtend {
  static constexpr bool STORES = true;
  Segs g;
  const T* h;
  const T* f;
  int N, R;
  // C = acc + bias, 32 rows at a time through LDS so that a row of 64 columns leaves as whole 128-byte lines.  The lanes exchange their values without a barrier of
  // the workgroup; the wave barriers keep the compiler from letting lanes whose columns lie past N run ahead (that condition is the same in every
  // pass, and threaded through them it had half of the lanes write all passes before the others read the first).
  __device__ __forceinline__ void store(const GemmParams& p, const f32x4 (&acc)[4][8], unsigned char* my, int row0, int col0, int lane) const {
    constexpr int ROW = 64 * 2 + 16;
    static_assert(32 * ROW <= EPI_WAVE, "a pass fits the wave's room");
    const int r = lane & 15, q = lane >> 4, col = col0 + 8 * (lane & 7);
    float b4[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int j = col0 + 16 * n + 4 * q;
#pragma unroll
      for (int e = 0; e < 4; ++e) b4[n][e] = 0.f;
      if (p.ep.bias && j < p.N) ld4(p.ep.bias + j, b4[n]);
    }
    unsigned char* wp = my + r * ROW + 8 * q;
    const unsigned char* lp = my + (lane >> 3) * ROW + (lane & 7) * 16;
#pragma unroll
    for (int h2 = 0; h2 < 4; ++h2) {
#pragma unroll
      for (int mm = 0; mm < 2; ++mm)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const f32x4& a = acc[n][2 * h2 + mm];
          uint2 pk;
          pk.x = pack2<T>(a[0] + b4[n][0], a[1] + b4[n][1]);
          pk.y = pack2<T>(a[2] + b4[n][2], a[3] + b4[n][3]);
          *reinterpret_cast<uint2*>(wp + mm * 16 * ROW + n * 32) = pk;
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      V16 v[4];
#pragma unroll
      for (int it = 0; it < 4; ++it) v[it] = ld16(lp + it * 8 * ROW);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int row = row0 + 32 * h2 + 8 * it + (lane >> 3);
        if (row < p.M && col < p.N) st16(reinterpret_cast<T*>(p.C) + (long)row * p.ldc + col, v[it]);
      }
    }
  }
  typedef typename AT<T>::frag frag;
  template <int NN, int NM> __device__ __forceinline__ void operator()(f32x4 (&acc)[NN][NM], int row0, int col0, int lane) const {
    // nothing below may be computed in front of the main loop and held across it: that loop counts its vector-memory operations, so it may not spill
    asm volatile("" : "+v"(lane));
    row0 = __builtin_amdgcn_readfirstlane(row0);
    col0 = __builtin_amdgcn_readfirstlane(col0);
    asm volatile("" : "+s"(row0), "+s"(col0));
    const int r = lane & 15, q = lane >> 4, row1 = min(row0 + 16 * NM, g.M);
    if (row0 >= g.M || col0 >= N) return;
    bool more = true;   // (a segment that reaches row1 is the last: the next one need not be looked at)
    for (int s = g.first_at(row0, lane); s < g.n && more; ++s) {
      const int begin = g.begin(s), end = g.begin(s + 1), a = g.adapter(s), b = max(begin, row0), e = min(end, row1);
      more = end < row1;
      if (b >= e || a < 0) continue;
      const T* fa = f + (long)a * N * R;
      for (int k = 0; k < R; k += AT<T>::KD) {
        const int k0 = k + ElemTraits<T>::VEC * q, kc = min(k0, R - ElemTraits<T>::VEC);
        // all operands in flight at once: rows and columns past the edge read the last ones, their products are dropped; ranks past it are zeros in both operands (h may be infinite)
        frag ff[NN], fh[NM];
#pragma unroll
        for (int n = 0; n < NN; ++n) ff[n] = *reinterpret_cast<const frag*>(fa + (long)min(col0 + 16 * n + r, N - 1) * R + kc);
#pragma unroll
        for (int m = 0; m < NM; ++m) fh[m] = *reinterpret_cast<const frag*>(h + (long)min(row0 + 16 * m + r, g.M - 1) * R + kc);
#pragma unroll
        for (int n = 0; n < NN; ++n)
          if (k0 >= R) ff[n] = zero_frag((frag*)nullptr);
#pragma unroll
        for (int m = 0; m < NM; ++m)
          if (k0 >= R) fh[m] = zero_frag((frag*)nullptr);
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          if (b >= row0 + 16 * m + 16 || e <= row0 + 16 * m) continue;
          const int row = row0 + 16 * m + r;
          const bool mine = row >= b && row < e;   // rows of other requests keep their sum
#pragma unroll
          for (int n = 0; n < NN; ++n) {
            const f32x4 t = mma<T>(ff[n], fh[m], acc[n][m]);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[n][m][c] = mine ? t[c] : acc[n][m][c];
          }
        }
      }
    }
  }
};
// The launch's parameters with everything that a plain X W^T + bias leaves unused as constants: the loops' epilogues fold to what is left.
__device__ __forceinline__ GemmParams plain_product(const GemmParams& a) {
  GemmParams p = a;
  GemmEpilogue& e = p.ep;
  e.alpha = 1.f; e.bias_gstride = 0; e.bias_mod = 0; e.preact = nullptr; e.act = FH_ACT_NONE; e.drop.p = 0.f; e.gelu_aux = nullptr; e.residual = nullptr;
  e.row_len = nullptr; e.out_f32 = 0; e.atomic = 0; e.idiv = e.jdiv = 0; e.si1 = e.si0 = e.sj1 = e.sj0 = 0; e.tail_cols = 0; e.aux_factor = 0;
  e.kd_teacher = nullptr; e.c0_wpart = nullptr;
  return p;
}
template <typename T, int YL> __global__ void __launch_bounds__(512) adapter_gemm_kernel(const GemmParams a, const AdapterExtend<T> ext) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  gemm_8ph_tile<T, FH_R_CONTIG, YL, false, AdapterExtend<T>>(a, lds, logical_block(1), 1, 0, ext);
}
template <typename T> __global__ void __launch_bounds__(256) adapter_gemm_small_kernel(const GemmParams a, const AdapterExtend<T> ext) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const GemmParams p = plain_product(a);
  gemm_small_tile<T, AdapterExtend<T>>(p, lds, ext);
}

// Few rows (a frame of each of some live requests): y whole, in one kernel behind `down`.  A workgroup owns 16 columns of 64 rows; its four waves split K straight from
// memory into the products' operands -- W is read once, by as many workgroups as N has 16s --, then a thread holds four columns of one row and adds
// that row's own adapter, whatever the other rows use: a tile of one-row requests costs no walk over them.
template <typename T>
__global__ void __launch_bounds__(256) adapter_few_kernel(const Segs g, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ bias,
                                                          const T* __restrict__ h, const T* __restrict__ f, T* __restrict__ y, int K, int N, int R) {
  constexpr int KD = AT<T>::KD, VEC = ElemTraits<T>::VEC;
  typedef typename AT<T>::frag frag;
  __shared__ f32x4 part[4][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 16, mt = min(4, (g.M - i0 + 15) >> 4);
  // the adapter of this thread's row in the end (row tile `wave`, row r): the segments' ends 64 at a time, one count per row
  const int row = i0 + 16 * wave + r, seg0 = g.first_at(min(i0 + 16 * wave, g.M), lane);
  int mine = seg0;
  for (int s = seg0; s < g.n; s += 64) {
    const int end = s + lane < g.n ? g.start[s + lane + 1] : 0x7fffffff;
    bool more = false;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int passed = __popcll(__ballot(end <= i0 + 16 * wave + k));
      if (k == r) mine += passed;
      more = passed == 64;
    }
    if (!more) break;
  }
  const int a = row < g.M && mine < g.n && g.start[mine] <= row ? g.adapter(mine) : -1;
  f32x4 acc[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const T* wr = w + (long)min(j0 + r, N - 1) * K;
  const T* xr[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) xr[m] = x + (long)min(i0 + 16 * m + r, g.M - 1) * K;
#pragma unroll 2
  for (int k = wave * 2 * KD; k < K; k += 8 * KD) {
    frag fw[2], fx[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k0 = k + u * KD + VEC * q;
      fw[u] = zero_frag((frag*)nullptr);
      if (k0 < K) fw[u] = *reinterpret_cast<const frag*>(wr + k0);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        fx[u][m] = zero_frag((frag*)nullptr);
        if (m < mt && k0 < K) fx[u][m] = *reinterpret_cast<const frag*>(xr[m] + k0);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (m < mt) acc[m] = mma<T>(fw[u], fx[u][m], acc[m]);
  }
#pragma unroll
  for (int m = 0; m < 4; ++m) part[wave][m][lane] = acc[m];
  __syncthreads();
  const int j = j0 + 4 * q;
  if (row >= g.M || j >= N) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += part[k][wave][lane][e];
  if (bias) {
    float b4[4];
    ld4(bias + j, b4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += b4[e];
  }
  if (a >= 0) {
    const T* fa = f + ((long)a * N + j) * R;
    const T* hr = h + (long)row * R;
    for (int k = 0; k < R; k += VEC) {
      float hv[VEC], fv[VEC];
      unpack16<T>(ld16(hr + k), hv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        unpack16<T>(ld16(fa + (long)e * R + k), fv);
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[e] = fmaf(hv[c], fv[c], v[e]);
      }
    }
  }
  st4(y + (long)row * N + j, v);
}

// fp32: C = X Y^T (+ bias) with the adapters' part, 64 x 64 per workgroup, 32 of the reduction at a time through two LDS buffers; a wave owns 32 x 32.  YL = FH_R_STRIDED: Y is read by
// its columns (dx: W[n][k] with the reduction over n) and turned on its way into LDS.  (The library's 128 x 128 fp32 loop with the part as residual: a
// 1497 x 480 x 480 product is 48 workgroups of it and took 52 us.)
template <int YL>
__global__ void __launch_bounds__(256) adapter_gemm_f32_kernel(const float* __restrict__ X, const float* __restrict__ Y, const float* __restrict__ bias, float* __restrict__ C,
                                                               int M, int N, int K, long ldy, const AdapterExtend<float> ext) {
  constexpr int BK = 32, ROW = BK + 4;
  __shared__ __attribute__((aligned(16))) float lds[2][2][64 * ROW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  const int tj_n = (N + 63) / 64, lb = xcd_remap(blockIdx.x, gridDim.x), ti = lb / tj_n, i0 = ti * 64, j0 = (lb - ti * tj_n) * 64;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  f32x4 px[2], py[2];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int n = tid + 256 * u, row = n >> 3, k = k0 + (n & 7) * 4;
      px[u] = py[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (i0 + row < M && k < K) px[u] = *reinterpret_cast<const f32x4*>(X + (long)(i0 + row) * K + k);
      if constexpr (YL == FH_R_CONTIG) {
        if (j0 + row < N && k < K) py[u] = *reinterpret_cast<const f32x4*>(Y + (long)(j0 + row) * ldy + k);
      } else {
        const int kr = k0 + (n >> 4), j = j0 + (n & 15) * 4;
        if (kr < K && j < N) py[u] = *reinterpret_cast<const f32x4*>(Y + (long)kr * ldy + j);
      }
    }
  };
  auto deposit = [&](int buf) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int n = tid + 256 * u;
      *reinterpret_cast<f32x4*>(&lds[buf][0][(n >> 3) * ROW + (n & 7) * 4]) = px[u];
      if constexpr (YL == FH_R_CONTIG) {
        *reinterpret_cast<f32x4*>(&lds[buf][1][(n >> 3) * ROW + (n & 7) * 4]) = py[u];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) lds[buf][1][((n & 15) * 4 + e) * ROW + (n >> 4)] = py[u][e];
      }
    }
  };
  f32x4 acc[2][2];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int m = 0; m < 2; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  fetch(0);
  int buf = 0;
  for (int k0 = 0; k0 < K; k0 += BK, buf ^= 1) {
    deposit(buf);   // (its readers of two steps ago have passed the barrier of the step in between)
    __syncthreads();
    if (k0 + BK < K) fetch(k0 + BK);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f32x4 fx[2], fy[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        fx[m] = *reinterpret_cast<const f32x4*>(&lds[buf][0][(wi + 16 * m + r) * ROW + ks * 16 + 4 * q]);
        fy[m] = *reinterpret_cast<const f32x4*>(&lds[buf][1][(wj + 16 * m + r) * ROW + ks * 16 + 4 * q]);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int m = 0; m < 2; ++m) acc[n][m] = mma<float>(fy[n], fx[m], acc[n][m]);
    }
  }
  ext(acc, i0 + wi, j0 + wj, lane);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int j = j0 + wj + 16 * n + 4 * q;
    if (j >= N) continue;
    float b4[4] = {0.f, 0.f, 0.f, 0.f};
    if (bias) ld4(bias + j, b4);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int row = i0 + wi + 16 * m + r;
      if (row >= M) continue;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[n][m][e] + b4[e];
      st4(C + (long)row * N + j, v);
    }
  }
}

// One gradient's sums: dst[a][r][c] (dA: by row) or dst[a][c][r] (dB) = sum over the rows of adapter a of u[row][r] v[row][c], in `wgs` workgroups per adapter: `splits`
// of the rows for every 64 columns.  With several splits: partial sums part[split][a] .. in the same layout.
template <typename T> struct Outer {
  const T* u;
  const T* v;
  T* dst;
  float* part;
  int C, splits, wgs;
};
template <typename T, int NR, bool BY_ROW>
__device__ __forceinline__ void outer_sums(const Segs& g, const Outer<T>& o, int wg, int R, unsigned char* lds) {
  const T* __restrict__ u = o.u;
  const T* __restrict__ v = o.v;
  const int C = o.C;
  constexpr int VEC = ElemTraits<T>::VEC, ES = sizeof(T);
  constexpr int RU = NR * 16 * ES + 16, RV = 64 * ES + 16;           // LDS row strides
  constexpr int PER = 32 * (RU + RV);                                // a wave's tiles
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int split = wg % o.splits, c0 = wg / o.splits * 64, a = blockIdx.y, ways = 4 * o.splits;
  unsigned char* tu = lds + wave * PER;
  unsigned char* tv = tu + 32 * RU;
  f32x4 acc[NR][4];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int m = 0; m < 4; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  int turn = 0;                                                      // blocks of 32 rows of this adapter seen so far
  for (int sb = 0; sb < g.n; sb += 64) {
    const int s = sb + lane;
    const bool ours = s < g.n && g.adapter(s) == a;
    const int b_ = ours ? g.begin(s) : 0, e_ = ours ? g.begin(s + 1) : 0;
    unsigned long long left = __ballot(b_ < e_);
    while (left) {
      const int j = __ffsll((unsigned long long)left) - 1;
      left &= left - 1;
      const int b = __builtin_amdgcn_readlane(b_, j), e = __builtin_amdgcn_readlane(e_, j), blocks = (e - b + 31) >> 5;
      // the blocks of this segment whose turn is ours: turn + k = split * 4 + wave modulo ways
      int k = (split * 4 + wave - turn % ways + ways) % ways;
      turn += blocks;
      for (; k < blocks; k += ways) {
        const int row0 = b + 32 * k;
        constexpr int PU = 32 * NR * 16 / VEC / 64, PV = 32 * 64 / VEC / 64;
        V16 xu[PU > 0 ? PU : 1], xv[PV];
#pragma unroll
        for (int p = 0; p < PU; ++p) {
          const int at = p * 64 + lane, row = at / (NR * 16 / VEC), col = (at % (NR * 16 / VEC)) * VEC;
          xu[p] = v16_zero();
          if (row0 + row < e && col < R) xu[p] = ld16(u + (long)(row0 + row) * R + col);
        }
#pragma unroll
        for (int p = 0; p < PV; ++p) {
          const int at = p * 64 + lane, row = at / (64 / VEC), col = (at % (64 / VEC)) * VEC;
          xv[p] = v16_zero();
          if (row0 + row < e && c0 + col < C) xv[p] = ld16(v + (long)(row0 + row) * C + c0 + col);
        }
#pragma unroll
        for (int p = 0; p < PU; ++p) {
          const int at = p * 64 + lane, row = at / (NR * 16 / VEC), col = (at % (NR * 16 / VEC)) * VEC;
          st16(tu + row * RU + col * ES, xu[p]);
        }
#pragma unroll
        for (int p = 0; p < PV; ++p) {
          const int at = p * 64 + lane, row = at / (64 / VEC), col = (at % (64 / VEC)) * VEC;
          st16(tv + row * RV + col * ES, xv[p]);
        }
        // (a wave reads only what it wrote itself, and LDS accesses of one wave stay in order)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if constexpr (ES == 2) {
          bf16x8 fv[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const unsigned char* p0 = tv + (8 * q + (i >> 2)) * RV + (16 * m + 4 * (i & 3)) * 2;
            union { struct { s16x4 lo, hi; } s; bf16x8 v; } w;
            w.s.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p0);
            w.s.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0 + 4 * RV));
            fv[m] = w.v;
          }
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            const unsigned char* p0 = tu + (8 * q + (i >> 2)) * RU + (16 * n + 4 * (i & 3)) * 2;
            union { struct { s16x4 lo, hi; } s; bf16x8 v; } w;
            w.s.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p0);
            w.s.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0 + 4 * RU));
#pragma unroll
            for (int m = 0; m < 4; ++m) acc[n][m] = BY_ROW ? mfma16<T>(fv[m], w.v, acc[n][m]) : mfma16<T>(w.v, fv[m], acc[n][m]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            float fu[NR], fv[4];
#pragma unroll
            for (int n = 0; n < NR; ++n) fu[n] = *reinterpret_cast<const float*>(tu + (4 * t + q) * RU + (16 * n + i) * 4);
#pragma unroll
            for (int m = 0; m < 4; ++m) fv[m] = *reinterpret_cast<const float*>(tv + (4 * t + q) * RV + (16 * m + i) * 4);
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
              for (int m = 0; m < 4; ++m)
                acc[n][m] = BY_ROW ? __builtin_amdgcn_mfma_f32_16x16x4f32(fv[m], fu[n], acc[n][m], 0, 0, 0)
                                   : __builtin_amdgcn_mfma_f32_16x16x4f32(fu[n], fv[m], acc[n][m], 0, 0, 0);
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
  // the four waves' sums, in their order
  f32x4* sum = reinterpret_cast<f32x4*>(lds);
  for (int w = 0; w < 4; ++w) {
    __syncthreads();
    if (wave == w) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          f32x4 t = acc[n][m];
          if (w > 0) {
            const f32x4 o = sum[(n * 4 + m) * 64 + lane];
#pragma unroll
            for (int c = 0; c < 4; ++c) t[c] += o[c];
          }
          sum[(n * 4 + m) * 64 + lane] = t;
        }
    }
  }
  __syncthreads();
  const long at = ((long)split * g.adapters + a) * C * R;
  auto put = [&](long n, const float* w) {
    if (o.splits > 1) st4(o.part + at + n, w);
    else st4(o.dst + at + n, w);
  };
  for (int t = wave; t < NR * 4; t += 4) {
    const int n = t >> 2, m = t & 3;
    const f32x4 f = sum[t * 64 + lane];
    const float w[4] = {f[0], f[1], f[2], f[3]};
    if constexpr (BY_ROW) {   // tile rows: columns c, tile columns: r
      const int c = c0 + 16 * m + 4 * q, rr = 16 * n + i;
      if (c < C && rr < R) put((long)rr * C + c, w);
    } else {
      const int rr = 16 * n + 4 * q, c = c0 + 16 * m + i;
      if (c < C && rr < R) put((long)c * R + rr, w);
    }
  }
}

// dA's workgroups first, dB's behind them: one launch, so that neither waits for the other's last rows
template <typename T, int NR>
__global__ void __launch_bounds__(256) adapter_outer_kernel(const Segs g, const Outer<T> da, const Outer<T> db, int R) {
  constexpr int PER = 32 * ((NR * 16 + 64) * (int)sizeof(T) + 32), SUM = NR * 4 * 64 * 16;   // (one wave's sums at the end)
  __shared__ __attribute__((aligned(16))) unsigned char lds[4 * PER > SUM ? 4 * PER : SUM];
  if ((int)blockIdx.x < da.wgs) outer_sums<T, NR, true>(g, da, blockIdx.x, R, lds);
  else outer_sums<T, NR, false>(g, db, blockIdx.x - da.wgs, R, lds);
}

// the splits' sums in their order: na x 256 x 4 elements of dA first, dB behind them
template <typename T> __global__ void __launch_bounds__(256) adapter_join_kernel(const Outer<T> da, const Outer<T> db, int na, long a4, long b4) {
  const bool is_a = (int)blockIdx.x < na;
  const Outer<T>& o = is_a ? da : db;
  const long n4 = is_a ? a4 : b4, i = (long)((int)blockIdx.x - (is_a ? 0 : na)) * 256 + threadIdx.x;
  if (i >= n4) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f}, f[4];
#pragma unroll 4
  for (int k = 0; k < o.splits; ++k) {
    ld4(o.part + ((long)k * n4 + i) * 4, f);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += f[e];
  }
  st4(o.dst + i * 4, s);
}

// ------------------------------------------------------------------------------------------------ host
int check(int dtype, const fh_adapter_desc* d) {
  if (dtype < 0 || dtype > 2) return -941;
  if (!d || d->M < 0 || d->K < 8 || d->N < 8 || d->K % 8 || d->N % 8) return -942;
  if (d->R < 8 || d->R > 128 || d->R % 8) return -943;
  if (d->n_adapters < 1 || d->n_adapters > 65535 || d->n_segments < 0 || d->M > (1 << 30)) return -944;
  if (d->n_segments > 0 && (!d->seg_start || !d->seg_adapter || !d->scaling)) return -945;
  return 0;
}
Segs segs_of(const fh_adapter_desc* d) {
  Segs g;
  g.start = d->seg_start; g.which = d->seg_adapter; g.scaling = d->scaling;
  g.n = d->n_segments; g.adapters = d->n_adapters; g.M = d->M;
  return g;
}
size_t al16(size_t n) { return (n + 15) & ~(size_t)15; }
// workgroups per adapter and 64-column tile: about four per CU in all, at least 256 rows each
int outer_splits(const fh_adapter_desc* d, int C) {
  const long wgs = (long)d->n_adapters * ((C + 63) / 64);
  long n = 1024 / wgs;
  if (n > (d->M + 255) / 256) n = (d->M + 255) / 256;
  return n < 1 ? 1 : (int)n;
}
size_t outer_bytes(const fh_adapter_desc* d, int C) {
  const int n = outer_splits(d, C);
  return n > 1 ? al16((size_t)n * d->n_adapters * C * d->R * 4) : 0;
}

// Whether requests are short on average, and the workgroups of adapter_few_kernel (see `project`)
bool brief(const fh_adapter_desc* d) { return (long)d->n_segments * 16 > d->M; }
long few_blocks(long M, long N) { return (M + 63) / 64 * ((N + 15) / 16); }
constexpr long FEW_BRIEF = 2048;
// Whether a 16-bit product of M x N with the reduction K takes the 256 x 256 8-phase loop: with W by its rows where its tiles give work to a good part of the CUs; with W by its columns, where the
// loop for small products needs W turned first, from 36 tiles on.  Both directions, rank 8 to 64, us with W turned | with the large loop: 18 tiles (600 rows, 2304 -> 1536) 93 | 128, 24 (3000, 1440 ->
// 480) 93 | 108, 32 (2000, 1024 -> 1024) 77 | 85, 36 (1400, 2304 -> 1536) 169 | 162, 48 (3000, 1024 -> 1024) 98 | 97, 72 (3000, 2304 -> 1536) 236 | 194.
bool large(long M, long N, long K, bool strided) {
  const long tiles = (M + 255) / 256 * ((N + 255) / 256);
  return K >= 128 && (tiles >= 96 || (strided && tiles >= 36 && N >= 128));
}
// Whether the backward pass turns W for dx: the loops for small products read it by its rows only.
bool turns_weight(int dtype, const fh_adapter_desc* d) {
  return dtype != 0 && (brief(d) ? few_blocks(d->M, d->K) <= FEW_BRIEF : !large(d->M, d->K, d->N, true));
}

size_t partial_bytes(const fh_adapter_desc* d) { return outer_bytes(d, d->K) + outer_bytes(d, d->N); }

template <typename T> int down(const Segs& g, const void* x, const void* f, void* out, int K, int R, hipStream_t st) {
  if (g.M == 0) return 0;
  // 32-row tiles where they still fill the chip twice over (two workgroups per CU: 16384 rows, the only size measured, 4096 columns, rank 16: 50 -> 36 us) and requests are
  // long enough on average to share them
  const bool wide = g.M >= 16384 && R <= 64 && (long)g.n * 64 <= g.M;
  const int tile = wide ? 32 : 16, tiles = (g.M + tile - 1) / tile;
  const long per = 1 + ((long)tile * g.n + g.M - 1) / g.M;   // segments that a tile touches
  const dim3 grid(tiles, per > 16 ? 16 : (int)per), block(256);
#define FH_DOWN(NR, RT) hipLaunchKernelGGL((adapter_down_kernel<T, NR, RT>), grid, block, 0, st, g, (const T*)x, (const T*)f, (T*)out, K, R)
  if (R <= 16) { if (wide) FH_DOWN(1, 2); else FH_DOWN(1, 1); }
  else if (R <= 32) { if (wide) FH_DOWN(2, 2); else FH_DOWN(2, 1); }
  else if (R <= 64) { if (wide) FH_DOWN(4, 2); else FH_DOWN(4, 1); }
  else FH_DOWN(8, 1);
#undef FH_DOWN
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename T> int up(const Segs& g, const void* h, const void* f, void* out, int N, int R, hipStream_t st) {
  hipLaunchKernelGGL((adapter_up_kernel<T>), dim3((g.M + 15) / 16, (N + 255) / 256), dim3(256), 0, st, g, (const T*)h, (const T*)f, (T*)out, N, R);
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename T> int outer(const fh_adapter_desc* d, const void* G, const void* x, void* da, const void* h, const void* dy, void* db, float* part, hipStream_t st) {
  const Segs g = segs_of(d);
  const int R = d->R;
  auto side = [&](const void* u, const void* v, void* dst, int C, float* p) {
    const int n = outer_splits(d, C);
    return Outer<T>{(const T*)u, (const T*)v, (T*)dst, p, C, n, dst ? (C + 63) / 64 * n : 0};
  };
  const Outer<T> a = side(G, x, da, d->K, part), b = side(h, dy, db, d->N, part + outer_bytes(d, d->K) / 4);
  const dim3 grid(a.wgs + b.wgs, d->n_adapters), block(256);
  if (R <= 16) hipLaunchKernelGGL((adapter_outer_kernel<T, 1>), grid, block, 0, st, g, a, b, R);
  else if (R <= 32) hipLaunchKernelGGL((adapter_outer_kernel<T, 2>), grid, block, 0, st, g, a, b, R);
  else if (R <= 64) hipLaunchKernelGGL((adapter_outer_kernel<T, 4>), grid, block, 0, st, g, a, b, R);
  else hipLaunchKernelGGL((adapter_outer_kernel<T, 8>), grid, block, 0, st, g, a, b, R);
  FH_CHECK_LAUNCH();
  auto quads = [&](const Outer<T>& o) { return o.wgs && o.splits > 1 ? (long)d->n_adapters * o.C * R / 4 : 0; };
  const long a4 = quads(a), b4 = quads(b), na = (a4 + 255) / 256, nb = (b4 + 255) / 256;
  if (na + nb > 0) {
    hipLaunchKernelGGL((adapter_join_kernel<T>), dim3((unsigned)(na + nb)), dim3(256), 0, st, a, b, (int)na, a4, b4);
    FH_CHECK_LAUNCH();
  }
  return 0;
}

// The projection's product with the adapters' part:
//   few rows (forward)        adapter_few_kernel, by its number of workgroups: with the whole of h's kernel, bf16 and rank 16, us against the next line's:
//                             1 x 480 -> 1440 7.2 | 18, 256 x 4096 -> 1024 35 | 44 (256 workgroups), 512 x 480 -> 1440 12.7 | 12.4 (720), 512 x 1024 -> 4096 48 | 35
//                             (2048), but 56 | 56 with one-row requests; fp32: 512 x 4096 -> 1024 98 | 131 (512), 1024 x 768 -> 768 36 | 33 (768)
//   requests under 16 rows    (on average; past the line above) the part on its own first (16-row tiles, many of them), then the GEMM's residual operand: a large tile would walk its
//                             requests one by one.  In 16-bit modes the part is rounded to the element type in between, off by half a step of itself, beside y's own rounding
//   fp32                      adapter_gemm_f32_kernel
//   16-bit                    inside the GEMM: the 256 x 256 8-phase loop where `large` says so, else the 64 x 64 one-trip loop (it takes W by its rows: a small backward pass turns W first)
template <typename T, int YL>
int project(int dtype, const fh_adapter_desc* d, GemmParams& p, const void* h, const void* f, hipStream_t st) {
  const Segs g = segs_of(d);
  const AdapterExtend<T> ext{g, (const T*)h, (const T*)f, p.N, d->R};
  const long few = few_blocks(p.M, p.N);
  if (YL == FH_R_CONTIG && few <= (brief(d) ? FEW_BRIEF : sizeof(T) == 4 ? 512 : 400)) {
    hipLaunchKernelGGL((adapter_few_kernel<T>), dim3((p.N + 15) / 16, (p.M + 63) / 64), dim3(256), 0, st, g, (const T*)p.X.p, (const T*)p.Y.p, p.ep.bias, (const T*)h, (const T*)f,
                       (T*)p.C, p.Kseg, p.N, d->R);
    FH_CHECK_LAUNCH();
    return 0;
  }
  if (!brief(d)) {
    if constexpr (sizeof(T) == 4) {
      const long tiles = (long)((p.M + 63) / 64) * ((p.N + 63) / 64);
      if (tiles <= 0x7fffffffL) {
        hipLaunchKernelGGL((adapter_gemm_f32_kernel<YL>), dim3((unsigned)tiles), dim3(256), 0, st, (const float*)p.X.p, (const float*)p.Y.p, p.ep.bias, (float*)p.C, p.M, p.N,
                           p.Kseg, p.Y.ld, ext);
        FH_CHECK_LAUNCH();
        return 0;
      }
    } else {
      const long tiles = (long)((p.M + 255) / 256) * ((p.N + 255) / 256);
      if (large(p.M, p.N, p.Kseg, YL == FH_R_STRIDED) && tiles <= 0x7fffffffL) {
        const size_t smem = 131072;
        if (int rc = (int)hipFuncSetAttribute((const void*)adapter_gemm_kernel<T, YL>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return rc;
        hipLaunchKernelGGL((adapter_gemm_kernel<T, YL>), dim3((unsigned)tiles), dim3(512), smem, st, p, ext);
        FH_CHECK_LAUNCH();
        return 0;
      }
      if constexpr (YL == FH_R_CONTIG) {
        const size_t smem = 2 * (size_t)64 * 512 * 2;
        if (int rc = (int)hipFuncSetAttribute((const void*)adapter_gemm_small_kernel<T>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return rc;
        hipLaunchKernelGGL((adapter_gemm_small_kernel<T>), dim3(((p.M + 63) / 64) * ((p.N + 63) / 64)), dim3(256), smem, st, p, ext);
        FH_CHECK_LAUNCH();
        return 0;
      }
    }
  }
  if (int rc = up<T>(g, h, f, p.C, p.N, d->R, st)) return rc;
  p.ep.residual = p.C;
  if constexpr (sizeof(T) == 4) return fh_gemm_launch(p, dtype, st);
  // The loop that an unmeasured shape takes, without the per-shape table: a measurement would run the launch several times, each on top of the last one's sum, and
  // the table is not for two threads (a backward pass runs on autograd's).
  const int loop = p.M >= 4096 && p.N >= 128 && p.Kseg >= 128 ? 8 : 2;
  return dtype == 2 ? fh_gemm_path_f16(p, loop, st) : fh_gemm_path_bf16(p, loop, st);
}

template <typename T>
int forward_t(int dtype, const fh_adapter_desc* d, const void* x, const void* w, const float* bias, const void* a, const void* b, void* h, void* y, hipStream_t st) {
  if (int rc = down<T>(segs_of(d), x, a, h, d->K, d->R, st)) return rc;
  GemmParams p = fh_gemm_params();
  p.X = fh_operand(x, FH_R_CONTIG, d->K);
  p.Y = fh_operand(w, FH_R_CONTIG, d->K);
  p.C = y;
  p.M = d->M; p.N = d->N; p.Kseg = d->K; p.ldc = d->N;
  p.ep.bias = bias;
  return project<T, FH_R_CONTIG>(dtype, d, p, h, b, st);
}
template <typename T>
int backward_t(int dtype, const fh_adapter_desc* d, const void* x, const void* w, const void* a, const void* b, const void* h, const void* dy, void* dx,
               void* da, void* db, char* scratch, hipStream_t st) {
  T* G = (T*)scratch;
  float* part = (float*)(scratch + al16((size_t)d->M * d->R * sizeof(T)));
  T* at = (T*)((char*)part + partial_bytes(d));
  T* bt = at + (long)d->n_adapters * d->K * d->R;
  T* wt = bt + (long)d->n_adapters * d->N * d->R;
  if ((dx || da) && d->M > 0) {
    const int rt = (d->R + 63) / 64;
    hipLaunchKernelGGL((adapter_turn_kernel<T>), dim3(rt * ((d->K + 63) / 64 + (d->N + 63) / 64), d->n_adapters), dim3(256), 0, st, (const T*)a, (const T*)b, at, bt, d->K,
                       d->N, d->R);
    FH_CHECK_LAUNCH();
    if (int rc = down<T>(segs_of(d), dy, bt, G, d->N, d->R, st)) return rc;
  }
  if (dx && d->M > 0) {
    GemmParams p = fh_gemm_params();
    p.X = fh_operand(dy, FH_R_CONTIG, d->N);
    p.C = dx;
    p.M = d->M; p.N = d->K; p.Kseg = d->N; p.ldc = d->K;
    int rc;
    if (turns_weight(dtype, d)) {
      hipLaunchKernelGGL((adapter_turn_kernel<T>), dim3((d->N + 63) / 64 * ((d->K + 63) / 64)), dim3(256), 0, st, (const T*)w, (const T*)nullptr, wt, (T*)nullptr, d->K, 0, d->N);
      FH_CHECK_LAUNCH();
      p.Y = fh_operand(wt, FH_R_CONTIG, d->N);
      rc = project<T, FH_R_CONTIG>(dtype, d, p, G, at, st);
    } else {
      p.Y = fh_operand(w, FH_R_STRIDED, d->K);
      rc = project<T, FH_R_STRIDED>(dtype, d, p, G, at, st);
    }
    if (rc) return rc;
  }
  if (da || db) return outer<T>(d, G, x, da, h, dy, db, part, st);
  return 0;
}

}  // namespace

extern "C" {

long fh_adapter_scratch_bytes(int dtype, const fh_adapter_desc* d, int backward) {
  if (check(dtype, d)) return -1;
  if (!backward) return 0;
  return (long)(al16((size_t)d->M * d->R * fh_esize(dtype)) + partial_bytes(d) + (size_t)d->n_adapters * d->R * ((size_t)d->K + d->N) * fh_esize(dtype) +
                (turns_weight(dtype, d) ? (size_t)d->K * d->N * fh_esize(dtype) : 0));
}

int fh_adapter_linear_forward(int dtype, const fh_adapter_desc* d, const void* x, const void* w, const float* bias, const void* a, const void* b,
                              void* h, void* y, void* scratch, fh_stream_t stream) {
  if (int rc = check(dtype, d)) return rc;
  (void)scratch;
  if (d->M == 0) return 0;
  if (!x || !w || !a || !b || !h || !y) return -946;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)a | (uintptr_t)b | (uintptr_t)h | (uintptr_t)y) & 15) return -947;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return forward_t<float>(dtype, d, x, w, bias, a, b, h, y, st);
  if (dtype == 1) return forward_t<bf16>(dtype, d, x, w, bias, a, b, h, y, st);
  return forward_t<f16>(dtype, d, x, w, bias, a, b, h, y, st);
}

int fh_adapter_linear_backward(int dtype, const fh_adapter_desc* d, const void* x, const void* w, const void* a, const void* b, const void* h,
                               const void* dy, void* dx, void* da, void* db, void* scratch, fh_stream_t stream) {
  if (int rc = check(dtype, d)) return rc;
  if (!dx && !da && !db) return 0;
  if (d->M > 0 && (!dy || ((dx || da) && (!a || !b)) || (dx && !w) || (da && !x) || (db && !h) || !scratch)) return -946;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)a | (uintptr_t)b | (uintptr_t)h | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)da | (uintptr_t)db | (uintptr_t)scratch) & 15)
    return -947;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return backward_t<float>(dtype, d, x, w, a, b, h, dy, dx, da, db, (char*)scratch, st);
  if (dtype == 1) return backward_t<bf16>(dtype, d, x, w, a, b, h, dy, dx, da, db, (char*)scratch, st);
  return backward_t<f16>(dtype, d, x, w, a, b, h, dy, dx, da, db, (char*)scratch, st);
}

}  // extern "C"
