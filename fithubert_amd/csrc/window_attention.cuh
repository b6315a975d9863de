// Attention inside a sliding window with a few first keys that stay visible ("sinks"), forward and backward.
//
//   row p sees key s:  s < key_len,  s <= p + right,  s >= p - left or s < sinks
//   P = softmax over the seen keys of scale q.k;  out = P v
//   dP = dout v^T,  D = sum_d dout out,  dS = scale P (dP - D);   dq = dS k,  dk = dS^T q,  dv = P^T dout
//
// Query heads that share a key head are ROWS of one problem: row = frame * G + (head inside the group), G = Hq / Hkv.  Keys and values are
// then staged once for all G heads, the sums of dk / dv over the group happen in registers, and one frame of a stream fills G rows of a
// tile instead of one.
//
// Forward: a workgroup owns 32 rows per wave, walks the 64-key tiles that its rows see (first the sinks' tiles, then the window's) through
// two LDS buffers, and keeps running maximum and sum per row.  Scores are computed transposed (keys x rows): a lane holds ONE row, the
// reductions are two row exchanges, and the probabilities are the second product's operand without leaving the registers.  A wave
// skips tiles that none of its rows sees; only tiles on a border of the window pay for the mask.  Few rows against many keys: the tiles
// are dealt over several workgroups, whose partial sums a second kernel joins.
// Backward: a pass over the rows for dq (the forward's walk), one over 128-key blocks for dk / dv (its rows are those between the block's
// window borders).  The blocks that hold sinks see every later row: their rows are dealt over several workgroups and joined.
// Two passes cost 7 products instead of 5, but no atomics: results repeat bit for bit.
#pragma once
#include "window_attention.h"
#include "attn_frag.cuh"

namespace {

template <typename T, int NDT> struct WT {
  static constexpr int KD = AT<T>::KD;
  static constexpr int NK = (NDT * 16 + KD - 1) / KD;   // fragments per row
  static constexpr int RS = NK * 64 + 16;               // LDS row stride (bytes): 16 bytes of skew against bank conflicts
  static constexpr int TILE = 64 * RS;
  static constexpr int VEC = ElemTraits<T>::VEC;
  typedef typename AT<T>::frag frag;
  // waves per SIMD that the register budget is cut for: wide heads hold their accumulators in registers alone
  static constexpr int OCC = NDT >= (sizeof(T) == 4 ? 6 : 9) ? 1 : 2;
  static constexpr int OCC_DKV = NDT >= (sizeof(T) == 4 ? 4 : 6) ? 1 : 2;
};

template <typename T, int NDT> __device__ __forceinline__ typename AT<T>::frag wfrag(const unsigned char* lds, int row, int ks, int lane) {
  return *reinterpret_cast<const typename AT<T>::frag*>(lds + row * WT<T, NDT>::RS + ks * 64 + (lane >> 4) * 16);
}

// acc[dt] += Tile^T[d tile dt][rows 32 m2 .. 32 m2 + 31] * P: P0 / P1 are the accumulator tiles of rows 0..15 / 16..31 of that range
template <typename T, int NDT>
__device__ __forceinline__ void wmma_transposed(const unsigned char* tile, int m2, const f32x4& P0, const f32x4& P1, f32x4 (&acc)[NDT], int lane) {
  constexpr int RS = WT<T, NDT>::RS;
  const int i = lane & 15, q = lane >> 4;
  if constexpr (sizeof(T) == 2) {
    union { V16 w; bf16x8 v; } pb;   // the rounding of the probabilities (or dS) to the element type: half a unit in 2^-8 (bf16) / 2^-11 of each
    pb.w.w[0] = pack2<T>(P0[0], P0[1]); pb.w.w[1] = pack2<T>(P0[2], P0[3]);
    pb.w.w[2] = pack2<T>(P1[0], P1[1]); pb.w.w[3] = pack2<T>(P1[2], P1[3]);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const unsigned char* a0 = tile + (32 * m2 + 4 * q + (i >> 2)) * RS + (16 * dt + 4 * (i & 3)) * 2;
      union { struct { s16x4 lo, hi; } s; bf16x8 v; } u;
      u.s.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a0);
      u.s.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a0 + 16 * RS));
      acc[dt] = mfma16<T>(u.v, pb.v, acc[dt]);
    }
  } else {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 32 * m2 + 16 * half + 4 * q + e;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const float a = *reinterpret_cast<const float*>(tile + row * RS + (16 * dt + i) * 4);
          acc[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, half ? P1[e] : P0[e], acc[dt], 0, 0, 0);
        }
      }
  }
}

// 64 rows of two tensors (K and V, or q and dout) on their way from memory to an LDS tile pair: fetch() requests them into registers, deposit()
// stores them -- a tile later, so that the latency lies under the tile in between.  A thread owns one 16-byte column of every RP-th row.
template <typename T, int NDT, int NT> struct Mover {
  static constexpr int VEC = WT<T, NDT>::VEC;
  static constexpr int CP = NDT * 16 / VEC;        // columns at the widest head
  static constexpr int RP = NT / CP;               // rows per pass
  static constexpr int NP = (64 + RP - 1) / RP;    // passes
  V16 pre[2][NP];
  int row, col, dst;
  bool live;
  __device__ __forceinline__ void init(int dh) {
    row = (int)threadIdx.x / CP;
    const int c = (int)threadIdx.x - row * CP;
    col = c * VEC;
    live = row < RP && col < dh;
    dst = row * WT<T, NDT>::RS + c * 16;
  }
  // at(row, first, second): the addresses of a row's channels in the two tensors; false: zeros
  template <typename F> __device__ __forceinline__ void fetch(F&& at) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      pre[0][j] = pre[1][j] = v16_zero();
      const T *x, *y;
      if (live && row + j * RP < 64 && at(row + j * RP, x, y)) {
        pre[0][j] = ld16(x + col);
        pre[1][j] = ld16(y + col);
      }
    }
  }
  __device__ __forceinline__ void deposit(unsigned char* pair) const {
#pragma unroll
    for (int j = 0; j < NP; ++j)
      if (live && row + j * RP < 64) {
        st16(pair + dst + j * RP * WT<T, NDT>::RS, pre[0][j]);
        st16(pair + WT<T, NDT>::TILE + dst + j * RP * WT<T, NDT>::RS, pre[1][j]);
      }
  }
};

__device__ __forceinline__ int clip_pos(int p) { return max(-FAR, min(FAR, p)); }

// (x, y, z) of the grid in an order that keeps neighbouring x on one XCD: they read the same keys
__device__ __forceinline__ void win_block(int& x, int& y, int& z) {
  const int lg = fh_xcd_logical_block(), gx = gridDim.x, gy = gridDim.y;
  x = lg % gx;
  const int yz = lg / gx;
  y = yz % gy;
  z = yz / gy;
}

// The 64-key tiles that the rows of frames [i0, i1] see: ns tiles from key 0 on (sinks), then those from tile `first` on, n in all.
struct TileWalk {
  int klen, lo, hi, ns, first, n;   // keys [lo, hi) and the sinks below hi are all that any of these rows sees
  __device__ __forceinline__ TileWalk(const WinArgs& a, int b, int p0, int p1) {
    klen = a.key_len ? max(0, min(a.key_len[b], a.Tk)) : a.Tk;
    lo = max(0, p0 - a.left);
    hi = max(0, min(klen, p1 + a.right + 1));
    const int last = lo < hi ? (hi + 63) >> 6 : 0;
    first = lo < hi ? lo >> 6 : 0;
    ns = (min(a.sinks, hi) + 63) >> 6;
    if (last > 0 && ns >= first) { ns = 0; first = min(first, (a.sinks > 0 ? 0 : first)); }
    n = ns + (last - first);
  }
  __device__ __forceinline__ int key0(int k) const { return (k < ns ? k : first + k - ns) << 6; }
};

// Which part of a 64-key tile the rows at positions [p0, p1] see.  0: nothing, 1: some of it, 2: all of it, every row
__device__ __forceinline__ int tile_sight(const WinArgs& a, int klen, int s0, int p0, int p1) {
  if (s0 >= klen || s0 > p1 + a.right || (s0 + 63 < p0 - a.left && s0 >= a.sinks)) return 0;
  if (s0 + 63 < klen && s0 + 63 <= p0 + a.right && (s0 >= p1 - a.left || s0 + 63 < a.sinks)) return 2;
  return 1;
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int NDT, int NW, bool SPLIT>
__global__ void __launch_bounds__(NW * 64, (WT<T, NDT>::OCC)) win_fwd_kernel(const WinArgs a, const T* __restrict__ q_, const T* __restrict__ k_, const T* __restrict__ v_,
                                                          T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part) {
  typedef WT<T, NDT> W;
  constexpr int NK = W::NK;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  int blk, h, bz;
  win_block(blk, h, bz);
  const int split = SPLIT ? bz % a.nsplit : 0, b = SPLIT ? bz / a.nsplit : bz;
  const int base = a.q_start ? clip_pos(a.q_start[b]) : 0;
  const int g0 = blk * 32 * NW, g1 = min(g0 + 32 * NW, a.rows) - 1;            // the workgroup's rows
  const int w0 = g0 + wave * 32, w1 = min(w0 + 31, a.rows - 1);                // the wave's
  const TileWalk walk(a, b, base + g0 / a.G, base + g1 / a.G);
  const int wp0 = base + w0 / a.G, wp1 = base + w1 / a.G;
  const T* qb = q_ + b * a.q_bs;
  const T* kb_ = k_ + b * a.k_bs + h * a.k_hs;
  const T* vb_ = v_ + b * a.v_bs + h * a.v_hs;
  zero_lds<T>(lds, 4 * W::TILE);                                               // (channels past dh are never written again)
  typename W::frag qf[2][NK];
  int pos[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int row = w0 + 16 * t + r, i = row / a.G, g = row - i * a.G;
    pos[t] = base + i;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) qf[t][ks] = gfrag<T>(qb + i * a.q_ts + (long)(h * a.G + g) * a.q_hs, row < a.rows, ks, lane, a.dh);
  }
  __syncthreads();
  Mover<T, NDT, NW * 64> mv;
  mv.init(a.dh);
  const int per = SPLIT ? (walk.n + a.nsplit - 1) / a.nsplit : walk.n;
  const int kt0 = split * per, kt1 = min(walk.n, kt0 + per);
  auto fetch = [&](int s0) {
    mv.fetch([&](int row, const T*& x, const T*& y) {
      const int s = s0 + row;
      x = kb_ + s * a.k_ts;
      y = vb_ + s * a.v_ts;
      return s < walk.hi && (s >= walk.lo || s < a.sinks);                     // what no row here sees is not read
    });
  };
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  f32x4 o[2][NDT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](const unsigned char* Ks, int s0, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const unsigned char* Vs = Ks + W::TILE;
    f32x4 s[4][2];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      s[kb][0] = s[kb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        const typename W::frag f = wfrag<T, NDT>(Ks, 16 * kb + r, ks, lane);
        s[kb][0] = mma<T>(f, qf[0][ks], s[kb][0]);
        s[kb][1] = mma<T>(f, qf[1][ks], s[kb][1]);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float mx = -INFINITY;
      const int hi = min(walk.klen - 1, pos[t] + a.right), lo = pos[t] - a.left;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (MASKED) {
            const int key = s0 + 16 * kb + 4 * q + e;
            if (key > hi || (key < lo && key >= a.sinks)) s[kb][t][e] = -INFINITY;
          }
          mx = fmaxf(mx, s[kb][t][e]);
        }
      const float mnew = fmaxf(m[t], xor_max(mx) * a.c);                        // c > 0: the maximum commutes with it
      const float ref = mnew == -INFINITY ? 0.f : mnew;                         // (a row that has seen nothing yet)
      const float alpha = fast_exp2(m[t] - ref);
      m[t] = mnew;
      float rs = 0.f;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = fast_exp2(fmaf(s[kb][t][e], a.c, -ref));
          rs += p;
          s[kb][t][e] = p;
        }
      l[t] = l[t] * alpha + xor_sum(rs);
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][dt][e] *= alpha;
      }
    }
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2)
#pragma unroll
      for (int t = 0; t < 2; ++t) wmma_transposed<T, NDT>(Vs, m2, s[2 * m2][t], s[2 * m2 + 1][t], o[t], lane);
  };

  if (kt0 < kt1) fetch(walk.key0(kt0));
  for (int kt = kt0; kt < kt1; ++kt) {
    unsigned char* Ks = lds + ((kt - kt0) & 1) * 2 * W::TILE;
    // the buffer's readers of two tiles ago have all passed the barrier of the tile in between
    mv.deposit(Ks);
    __syncthreads();
    if (kt + 1 < kt1) fetch(walk.key0(kt + 1));
    const int s0 = walk.key0(kt), sight = w0 < a.rows ? tile_sight(a, walk.klen, s0, wp0, wp1) : 0;
    if (sight == 2) compute(Ks, s0, std::false_type{});
    else if (sight == 1) compute(Ks, s0, std::true_type{});
  }

#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int row = w0 + 16 * t + r;
    if (row >= a.rows) continue;
    const int i = row / a.G, g = row - i * a.G;
    if constexpr (SPLIT) {
      // partial sums of this workgroup's keys: [entry][head][split][row][dh + 2] with the maximum and the sum behind the channels
      float* dst = part + ((((long)b * a.Hkv + h) * a.nsplit + split) * a.rows + row) * (a.dh + 2);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const int d = 16 * dt + 4 * q;
        if (d < a.dh) {
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[d + e] = o[t][dt][e];
        }
      }
      if (q == 0) { dst[a.dh] = m[t]; dst[a.dh + 1] = l[t]; }
    } else {
      const float inv = l[t] > 0.f ? 1.0f / l[t] : (l[t] == 0.f ? 0.f : l[t]);   // (NaN stays NaN)
      const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
      if (q == 0 && lse) lse[orow] = l[t] == 0.f ? INFINITY : m[t] + log2f(l[t]);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const int d = 16 * dt + 4 * q;
        if (d < a.dh) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = o[t][dt][e] * inv;
          st4(out + orow * a.dh + d, w);
        }
      }
    }
  }
}

// joins the partial sums of a row: one wave per row, two channels per lane
template <typename T>
__global__ void __launch_bounds__(256) win_join_kernel(const WinArgs a, const float* __restrict__ part, T* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6);     // row of [entry][head][row]
  if (n >= (long)a.B * a.Hkv * a.rows) return;
  const int row = (int)(n % a.rows);
  const long bh = n / a.rows;
  const int h = (int)(bh % a.Hkv), b = (int)(bh / a.Hkv), W = a.dh + 2;
  const float* src = part + (bh * a.nsplit * a.rows + row) * W;
  const long step = (long)a.rows * W;
  float m = -INFINITY;
  for (int s = lane; s < a.nsplit; s += 64) m = fmaxf(m, src[s * step + a.dh]);
  m = wave_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int s = 0; s < a.nsplit; ++s) {
    const float* p = src + s * step;
    const float w = fast_exp2(p[a.dh] - ref);
    l += w * p[a.dh + 1];
    if (2 * lane < a.dh) { o0 += w * p[2 * lane]; o1 += w * p[2 * lane + 1]; }
  }
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  const int i = row / a.G, g = row - i * a.G;
  const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
  if (lane == 0 && lse) lse[orow] = l == 0.f ? INFINITY : m + log2f(l);
  if (2 * lane < a.dh) {
    out[orow * a.dh + 2 * lane] = from_f<T>(o0 * inv);
    out[orow * a.dh + 2 * lane + 1] = from_f<T>(o1 * inv);
  }
}

// ------------------------------------------------------------------------------------------------ backward: dq, and D for the other pass
template <typename T, int NDT, int NW>
__global__ void __launch_bounds__(NW * 64, (WT<T, NDT>::OCC)) win_dq_kernel(const WinArgs a, const T* __restrict__ q_, const T* __restrict__ k_, const T* __restrict__ v_,
                                                         const T* __restrict__ out, const T* __restrict__ dout, const float* __restrict__ lse,
                                                         float* __restrict__ delta, T* __restrict__ dq) {
  typedef WT<T, NDT> W;
  constexpr int NK = W::NK;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  int blk, h, b;
  win_block(blk, h, b);
  const int base = a.q_start ? clip_pos(a.q_start[b]) : 0;
  const int g0 = blk * 32 * NW, g1 = min(g0 + 32 * NW, a.rows) - 1;
  const int w0 = g0 + wave * 32, w1 = min(w0 + 31, a.rows - 1);
  const TileWalk walk(a, b, base + g0 / a.G, base + g1 / a.G);
  const int wp0 = base + w0 / a.G, wp1 = base + w1 / a.G;
  const T* qb = q_ + b * a.q_bs;
  const T* kb_ = k_ + b * a.k_bs + h * a.k_hs;
  const T* vb_ = v_ + b * a.v_bs + h * a.v_hs;
  zero_lds<T>(lds, 4 * W::TILE);
  typename W::frag qf[2][NK], gf[2][NK];
  int pos[2];
  float ls[2], dl[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int row = w0 + 16 * t + r, i = row / a.G, g = row - i * a.G;
    const bool live = row < a.rows;
    const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
    pos[t] = base + i;
    ls[t] = live ? lse[orow] : INFINITY;
    float d = 0.f;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      qf[t][ks] = gfrag<T>(qb + i * a.q_ts + (long)(h * a.G + g) * a.q_hs, live, ks, lane, a.dh);
      gf[t][ks] = gfrag<T>(dout + orow * a.dh, live, ks, lane, a.dh);
      const typename W::frag of = gfrag<T>(out + orow * a.dh, live, ks, lane, a.dh);
      union { typename W::frag f; V16 v; } x, y;
      x.f = gf[t][ks];
      y.f = of;
      float fx[W::VEC], fy[W::VEC];
      unpack16<T>(x.v, fx);
      unpack16<T>(y.v, fy);
#pragma unroll
      for (int e = 0; e < W::VEC; ++e) d = fmaf(fx[e], fy[e], d);
    }
    dl[t] = xor_sum(d);
    if (live && q == 0) delta[orow] = dl[t];
  }
  __syncthreads();
  Mover<T, NDT, NW * 64> mv;
  mv.init(a.dh);
  auto fetch = [&](int s0) {
    mv.fetch([&](int row, const T*& x, const T*& y) {
      const int s = s0 + row;
      x = kb_ + s * a.k_ts;
      y = vb_ + s * a.v_ts;
      return s < walk.hi && (s >= walk.lo || s < a.sinks);                     // what no row here sees is not read
    });
  };
  f32x4 acc[2][NDT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) acc[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const unsigned char* Ks, int s0, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const unsigned char* Vs = Ks + W::TILE;
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2) {
      f32x4 s[2][2], dp[2][2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int kb = 2 * m2 + kk;
        s[kk][0] = s[kk][1] = dp[kk][0] = dp[kk][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
          const typename W::frag f = wfrag<T, NDT>(Ks, 16 * kb + r, ks, lane);
          s[kk][0] = mma<T>(f, qf[0][ks], s[kk][0]);
          s[kk][1] = mma<T>(f, qf[1][ks], s[kk][1]);
          const typename W::frag fv = wfrag<T, NDT>(Vs, 16 * kb + r, ks, lane);
          dp[kk][0] = mma<T>(fv, gf[0][ks], dp[kk][0]);
          dp[kk][1] = mma<T>(fv, gf[1][ks], dp[kk][1]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int hi = min(walk.klen - 1, pos[t] + a.right), lo = pos[t] - a.left;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float p = fast_exp2(fmaf(s[kk][t][e], a.c, -ls[t]));
            if constexpr (MASKED) {
              const int key = s0 + 16 * kb + 4 * q + e;
              if (key > hi || (key < lo && key >= a.sinks)) p = 0.f;
            }
            s[kk][t][e] = p * a.scale * (dp[kk][t][e] - dl[t]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) wmma_transposed<T, NDT>(Ks, m2, s[0][t], s[1][t], acc[t], lane);
    }
  };
  if (walk.n > 0) fetch(walk.key0(0));
  for (int kt = 0; kt < walk.n; ++kt) {
    unsigned char* Ks = lds + (kt & 1) * 2 * W::TILE;
    mv.deposit(Ks);
    __syncthreads();
    if (kt + 1 < walk.n) fetch(walk.key0(kt + 1));
    const int s0 = walk.key0(kt), sight = w0 < a.rows ? tile_sight(a, walk.klen, s0, wp0, wp1) : 0;
    if (sight == 2) compute(Ks, s0, std::false_type{});
    else if (sight == 1) compute(Ks, s0, std::true_type{});
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int row = w0 + 16 * t + r;
    if (row >= a.rows) continue;
    const int i = row / a.G, g = row - i * a.G;
    const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const int d = 16 * dt + 4 * q;
      if (d < a.dh) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = acc[t][dt][e];
        st4(dq + orow * a.dh + d, w);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
// A workgroup owns 128 keys (32 per wave) of one key head and walks the 64-row tiles that see them.  grid.x: nsink * nsplit workgroups for the
// blocks that hold sinks (partial sums), then one per remaining block.
template <typename T, int NDT>
__global__ void __launch_bounds__(256, (WT<T, NDT>::OCC_DKV)) win_dkv_kernel(const WinArgs a, const T* __restrict__ q_, const T* __restrict__ k_, const T* __restrict__ v_,
                                                      const T* __restrict__ dout, const float* __restrict__ lse, const float* __restrict__ delta,
                                                      T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
  typedef WT<T, NDT> W;
  constexpr int NK = W::NK;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  float* rowdata = reinterpret_cast<float*>(lds + 4 * W::TILE);   // two buffers of 64 x (lse | D | position)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  int x, h, b;
  win_block(x, h, b);
  const bool shared = x < a.nsink * a.nsplit;
  const int kb = shared ? x / a.nsplit : x - a.nsink * a.nsplit + a.nsink, split = shared ? x % a.nsplit : 0;
  const int base = a.q_start ? clip_pos(a.q_start[b]) : 0;
  const int klen = a.key_len ? max(0, min(a.key_len[b], a.Tk)) : a.Tk;
  const int s0 = kb * 128, k0 = s0 + wave * 32;                   // first key of the workgroup, of the wave
  const T* qb = q_ + b * a.q_bs;
  zero_lds<T>(lds, 4 * W::TILE);
  typename W::frag kf[2][NK], vf[2][NK];
  int plo[2], phi[2];                                             // positions that see this lane's keys
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int s = k0 + 16 * t + r;
    plo[t] = s - a.right;
    phi[t] = s >= klen ? -2 * FAR : s < a.sinks ? 2 * FAR : s + a.left;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      kf[t][ks] = gfrag<T>(k_ + b * a.k_bs + h * a.k_hs + s * a.k_ts, s < klen, ks, lane, a.dh);
      vf[t][ks] = gfrag<T>(v_ + b * a.v_bs + h * a.v_hs + s * a.v_ts, s < klen, ks, lane, a.dh);
    }
  }
  // rows that see a key of this block: frames [f0, f1), then the workgroup's share of their 64-row tiles
  const int last = min(s0 + 127, klen - 1);
  const int f0 = max(0, min(a.Tq, s0 - a.right - base));
  const int f1 = last < s0 ? f0 : s0 < a.sinks ? a.Tq : max(f0, min(a.Tq, last + a.left - base + 1));
  const int row0 = f0 * a.G, row1 = f1 * a.G;
  const int nt = (row1 - row0 + 63) >> 6, per = shared ? (nt + a.nsplit - 1) / a.nsplit : nt;
  const int t0 = split * per, t1 = min(nt, t0 + per);
  __syncthreads();
  Mover<T, NDT, 256> mv;
  mv.init(a.dh);
  float pre_l = 0.f, pre_d = 0.f;
  auto fetch = [&](int rt) {
    const int first = row0 + rt * 64;
    mv.fetch([&](int n, const T*& x, const T*& y) {
      const int row = first + n, i = row / a.G, g = row - i * a.G;
      x = qb + i * a.q_ts + (long)(h * a.G + g) * a.q_hs;
      y = dout + (((long)b * a.Tq + i) * a.Hq + h * a.G + g) * a.dh;
      return row < row1;
    });
    if (threadIdx.x < 64) {
      const int row = first + (int)threadIdx.x, i = row / a.G, g = row - i * a.G;
      const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
      pre_l = row < row1 ? lse[orow] : INFINITY;                  // +inf: the row's probabilities are 0
      pre_d = row < row1 ? delta[orow] : 0.f;
    }
  };
  f32x4 ak[2][NDT], av[2][NDT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) ak[t][dt] = av[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const unsigned char* Qs, const float* rd, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const unsigned char* Gs = Qs + W::TILE;
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2) {
      f32x4 p[2][2], ds[2][2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int rb = 2 * m2 + kk;
        p[kk][0] = p[kk][1] = ds[kk][0] = ds[kk][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
          const typename W::frag f = wfrag<T, NDT>(Qs, 16 * rb + r, ks, lane);
          p[kk][0] = mma<T>(f, kf[0][ks], p[kk][0]);
          p[kk][1] = mma<T>(f, kf[1][ks], p[kk][1]);
          const typename W::frag fg = wfrag<T, NDT>(Gs, 16 * rb + r, ks, lane);
          ds[kk][0] = mma<T>(fg, vf[0][ks], ds[kk][0]);
          ds[kk][1] = mma<T>(fg, vf[1][ks], ds[kk][1]);
        }
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(rd + 16 * rb + 4 * q);
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(rd + 64 + 16 * rb + 4 * q);
        const int* p4 = reinterpret_cast<const int*>(rd + 128 + 16 * rb + 4 * q);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float w = fast_exp2(fmaf(p[kk][t][e], a.c, -l4[e]));
            if constexpr (MASKED) {
              const int at = p4[e];
              if (at < plo[t] || at > phi[t]) w = 0.f;
            }
            p[kk][t][e] = w;
            ds[kk][t][e] = w * a.scale * (ds[kk][t][e] - d4[e]);
          }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        wmma_transposed<T, NDT>(Gs, m2, p[0][t], p[1][t], av[t], lane);
        wmma_transposed<T, NDT>(Qs, m2, ds[0][t], ds[1][t], ak[t], lane);
      }
    }
  };
  if (t0 < t1) fetch(t0);
  for (int rt = t0; rt < t1; ++rt) {
    unsigned char* Qs = lds + ((rt - t0) & 1) * 2 * W::TILE;
    float* rd = rowdata + ((rt - t0) & 1) * 192;
    mv.deposit(Qs);
    if (threadIdx.x < 64) {
      rd[threadIdx.x] = pre_l;
      rd[64 + threadIdx.x] = pre_d;
      reinterpret_cast<int*>(rd)[128 + threadIdx.x] = base + (row0 + rt * 64 + (int)threadIdx.x) / a.G;
    }
    __syncthreads();
    if (rt + 1 < t1) fetch(rt + 1);
    // positions of the tile's rows against those that see the wave's keys
    const int p0 = base + (row0 + rt * 64) / a.G, p1 = base + min(row0 + rt * 64 + 63, row1 - 1) / a.G, ke = min(k0 + 31, klen - 1);
    if (ke < k0 || p1 < k0 - a.right || (p0 > ke + a.left && k0 >= a.sinks)) continue;
    if (k0 + 31 < klen && p0 >= k0 + 31 - a.right && (p1 <= k0 + a.left || k0 + 31 < a.sinks)) compute(Qs, rd, std::false_type{});
    else compute(Qs, rd, std::true_type{});
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int s = k0 + 16 * t + r;
    if (s >= a.Tk) continue;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const int d = 16 * dt + 4 * q;
      if (d >= a.dh) continue;
      float wk[4], wv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) { wk[e] = ak[t][dt][e]; wv[e] = av[t][dt][e]; }
      if (shared) {
        // [entry][head][sink block][split][dk | dv][128][dh]
        float* dst = part + (((((long)b * a.Hkv + h) * a.nsink + kb) * a.nsplit + split) * 2 * 128 + (s - s0)) * a.dh + d;
        st4(dst, wk);
        st4(dst + 128 * a.dh, wv);
      } else {
        const long at = (((long)b * a.Tk + s) * a.Hkv + h) * a.dh + d;
        st4(dk + at, wk);
        st4(dv + at, wv);
      }
    }
  }
}

// sums the partial dk / dv of the sink blocks, in the order of the splits; a thread owns four channels of one key
template <typename T>
__global__ void __launch_bounds__(256) win_dkv_join_kernel(const WinArgs a, const float* __restrict__ part, T* __restrict__ dk, T* __restrict__ dv) {
  const int c4 = a.dh / 4;
  const long n = (long)blockIdx.x * 256 + threadIdx.x, total = (long)a.B * a.Hkv * a.nsink * 2 * 128 * c4;
  if (n >= total) return;
  const int c = (int)(n % c4);
  long k = n / c4;
  const int key = (int)(k % 128);
  k /= 128;
  const int which = (int)(k % 2);
  k /= 2;
  const int kb = (int)(k % a.nsink), s = kb * 128 + key;
  k /= a.nsink;
  const int h = (int)(k % a.Hkv), b = (int)(k / a.Hkv);
  if (s >= a.Tk) return;
  const float* src = part + (((((long)b * a.Hkv + h) * a.nsink + kb) * a.nsplit * 2 + which) * 128 + key) * a.dh + c * 4;
  float sum[4] = {0.f, 0.f, 0.f, 0.f}, f[4];
  for (int i = 0; i < a.nsplit; ++i) {
    ld4(src + (long)i * 2 * 128 * a.dh, f);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += f[e];
  }
  st4((which ? dv : dk) + (((long)b * a.Tk + s) * a.Hkv + h) * a.dh + c * 4, sum);
}

// ------------------------------------------------------------------------------------------------ launches
template <typename K> int set_lds(K kernel, size_t bytes) {
  if (bytes <= 64 * 1024) return 0;
  return (int)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename T, int NDT, int NW, bool SPLIT>
int run_fwd(const WinArgs& a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st) {
  const size_t smem = 4 * WT<T, NDT>::TILE;
  if (int rc = set_lds(win_fwd_kernel<T, NDT, NW, SPLIT>, smem)) return rc;
  const dim3 grid((a.rows + 32 * NW - 1) / (32 * NW), a.Hkv, a.B * a.nsplit), block(NW * 64);
  hipLaunchKernelGGL((win_fwd_kernel<T, NDT, NW, SPLIT>), grid, block, smem, st, a, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, part);
  FH_CHECK_LAUNCH();
  if (SPLIT) {
    const long rows = (long)a.B * a.Hkv * a.rows;
    hipLaunchKernelGGL((win_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, part, (T*)out, lse);
    FH_CHECK_LAUNCH();
  }
  return 0;
}
template <typename T, int NDT>
int fwd_t(WinArgs a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st) {
  a.nsplit = fwd_splits(a);
  return a.nsplit > 1 ? run_fwd<T, NDT, 4, true>(a, q, k, v, out, lse, part, st) : run_fwd<T, NDT, 4, false>(a, q, k, v, out, lse, part, st);
}
template <typename T, int NDT>
int bwd_t(WinArgs a, const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, void* dq, void* dk, void* dv,
          char* scratch, hipStream_t st) {
  float* delta = (float*)scratch;
  float* part = (float*)(scratch + al16((size_t)a.B * a.Tq * a.Hq * 4));
  const size_t smem = 4 * WT<T, NDT>::TILE, smem2 = smem + 2 * 192 * 4;
  if (int rc = set_lds(win_dq_kernel<T, NDT, 4>, smem)) return rc;
  if (int rc = set_lds(win_dkv_kernel<T, NDT>, smem2)) return rc;
  if (a.rows > 0) {
    hipLaunchKernelGGL((win_dq_kernel<T, NDT, 4>), dim3((a.rows + 127) / 128, a.Hkv, a.B), dim3(256), smem, st, a, (const T*)q, (const T*)k, (const T*)v,
                       (const T*)out, (const T*)dout, lse, delta, (T*)dq);
    FH_CHECK_LAUNCH();
  }
  if (a.Tk > 0) {
    bwd_sinks(a);
    const int nkb = (a.Tk + 127) / 128;
    hipLaunchKernelGGL((win_dkv_kernel<T, NDT>), dim3(a.nsink * a.nsplit + nkb - a.nsink, a.Hkv, a.B), dim3(256), smem2, st, a, (const T*)q, (const T*)k,
                       (const T*)v, (const T*)dout, lse, delta, (T*)dk, (T*)dv, part);
    FH_CHECK_LAUNCH();
    if (a.nsink > 0) {
      const long n = (long)a.B * a.Hkv * a.nsink * 2 * 128 * (a.dh / 4);
      hipLaunchKernelGGL((win_dkv_join_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, part, (T*)dk, (T*)dv);
      FH_CHECK_LAUNCH();
    }
  }
  return 0;
}
#define WIN_BY_DH(fn, T, ...)                                       \
  (a.dh <= 48   ? fn<T, 3>(a, __VA_ARGS__)                          \
   : a.dh <= 64 ? fn<T, 4>(a, __VA_ARGS__)                          \
   : a.dh <= 96 ? fn<T, 6>(a, __VA_ARGS__)                          \
                : fn<T, 8>(a, __VA_ARGS__))
}  // namespace

// one element type's entry points (window_attention_{f32,bf16,f16}.hip)
#define WIN_INSTANCE(name, T)                                                                                                                        \
  int win_forward_##name(const WinArgs& a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st) {        \
    return WIN_BY_DH(fwd_t, T, q, k, v, out, lse, part, st);                                                                                         \
  }                                                                                                                                                  \
  int win_backward_##name(const WinArgs& a, const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse,        \
                          void* dq, void* dk, void* dv, char* scratch, hipStream_t st) {                                                             \
    return WIN_BY_DH(bwd_t, T, q, k, v, out, dout, lse, dq, dk, dv, scratch, st);                                                                    \
  }
