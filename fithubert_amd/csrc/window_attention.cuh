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
// Forward: a workgroup owns 16 or 32 rows per wave, walks the 64-key tiles that its rows see (first the sinks' tiles, then the window's) through
// two LDS buffers, and keeps running maximum and sum per row.  Scores are computed transposed (keys x rows): a lane holds ONE row, the
// reductions are two row exchanges, and the probabilities are the second product's operand without leaving the registers.  A wave
// skips tiles that none of its rows sees; only tiles on a border of the window pay for the mask.  Few rows against many keys: the tiles
// are dealt over several workgroups, whose partial sums a second kernel joins.
// Backward: a pass over the rows for dq (the forward's walk), one over 64- or 128-key blocks for dk / dv (its rows are those between the block's
// window borders).  The blocks that hold sinks see every later row: their rows are dealt over several workgroups and joined.
// Two passes cost 7 products instead of 5, but no atomics: results repeat bit for bit.
//
// Bound, 30001 frames, 16 heads over 4, 64 channels, 1024 keys per row, bf16, by the counters: the forward's vector instructions occupy 76 % of its SIMD cycles (9.6 per score, of which the
// MFMAs and the exponentials are 1.1 each), beside 31 % of the matrix pipe; dq's 63 % and 43 %; dk / dv's 40 % and 37 %: two waves per SIMD (its accumulators) leave gaps.
// Measured there, warm, after 60 passes: forward 185 us (0.68 PFLOP/s of its two products), dq 210 (0.90 of three), dk / dv 292 + 6 (0.86 of four); the call 691.  8 x 375 frames, 12 heads
// of 40 channels, window 64 + 64: 10, 11, 11 us.  fp32, 2 x 499 frames: 22, 29, 49 us.  Streams are bound by the cache's bytes and the length of a wave's
// chain: one fp16 frame of 64 entries, 4 key heads, 1028 keys: 15.6 us (68 MB, 4.3 TB/s); 16 frames against 65536 keys of 128 channels: 24 + 5 us (67 MB, 3.5 TB/s
// with the partial sums' 17 MB).  (The comparisons of variants further down were taken a few passes after an idle GPU, where the same kernels take about a quarter longer.)
#pragma once
#include "window_attention.h"
#include "attn_frag.cuh"

namespace {

template <typename T, int NDT> struct WT {
  static constexpr int KD = AT<T>::KD;
  static constexpr int NK = (NDT * 16 + KD - 1) / KD;   // fragments per row
  static constexpr int CP = NK <= 2 ? 8 : NK <= 4 ? 16 : 32;      // 16-byte pieces of a row's room, a power of two
  static constexpr int RS = sizeof(T) == 2 ? CP * 16 : NK * 64 + 16; // LDS row stride (bytes)
  static constexpr int TILE = 64 * RS;
  static constexpr int VEC = ElemTraits<T>::VEC;
  typedef typename AT<T>::frag frag;
  static constexpr int OCC = sizeof(T) == 4 && NDT >= 6 ? 1 : 2;   // waves per SIMD that the registers are cut for
  // The backward passes pack P (dP - D) and scale the sums; in IEEE half, whose largest number is 65504, they pack dS = scale P (dP - D) itself: under a scaled loss
  // the former is past that 1 / scale = 6 to 11 times sooner than anything that the formulas name.
  static constexpr bool SCALED = ElemTraits<T>::DT == 2;
  // The 16-byte piece c of a row lies at place c ^ twist(row).  The LDS serves 256 bytes at a time: sixteen rows' fragments (one piece each), the column reads'
  // two pieces of eight rows; the twists put each of these on 64 different banks (rows of 128 bytes: even and odd rows lie on different halves
  // already).  fp32: no twist, 16 bytes of skew per row (its column reads are single floats; the twisted form took more registers and time).
  static __device__ __forceinline__ int twist(int row) {
    return sizeof(T) == 4 ? 0 : RS == 128 ? (row & 6) | ((row >> 3) & 1) : ((row & 7) << 1) | ((row >> 3) & 1);
  }
  static __device__ __forceinline__ int place(int row, int c) { return row * RS + ((c ^ twist(row)) << 4); }
};

// fragment ks of row 16 n + (lane & 15)
template <typename T, int NDT> __device__ __forceinline__ typename AT<T>::frag wfrag(const unsigned char* lds, int n, int ks, int lane) {
  typedef WT<T, NDT> W;
  const int x = (lane >> 4) ^ W::twist(lane & 15);
  return *reinterpret_cast<const typename W::frag*>(lds + (16 * n + (lane & 15)) * W::RS + ((x ^ ((ks & 3) << 2)) << 4) + (ks >> 2) * 256);
}

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
// two floats to two elements of T, to nearest: one instruction
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (ElemTraits<T>::DT == 2) {
    union { f16x2 v; uint32_t u; } c;
    c.v = __builtin_convertvector(f32x2{a, b}, f16x2);
    return c.u;
  } else {
    union { bf16x2 v; uint32_t u; } c;
    c.v = __builtin_convertvector(f32x2{a, b}, bf16x2);
    return c.u;
  }
}

// The second products' operand, a 16-row accumulator tile at a time.  16-bit modes round the probabilities (or dS) to the element type here, the matrix pipe's rate for
// the second products: off by at most 2^-8 (bf16), 2^-11 (fp16) of each; they are packed as soon as they exist, which halves the registers that wait for the other half.
template <typename T> struct Half2 {
  typedef uint2 type;
  static __device__ __forceinline__ uint2 pack(const f32x4& p) { return make_uint2(pack_pair<T>(p[0], p[1]), pack_pair<T>(p[2], p[3])); }
};
template <> struct Half2<float> {
  typedef f32x4 type;
  static __device__ __forceinline__ f32x4 pack(const f32x4& p) { return p; }
};

// The columns of rows 32 m2 .. 32 m2 + 31 of an LDS tile as first operands (one per 16 channels): transposing reads (16-bit).
template <typename T, int NDT> __device__ __forceinline__ void tile_columns(const unsigned char* tile, int m2, bf16x8 (&col)[NDT], int lane) {
  constexpr int RS = WT<T, NDT>::RS;
  const int i = lane & 15, q = lane >> 4, row = 4 * q + (i >> 2), y = ((i >> 1) & 1) ^ WT<T, NDT>::twist(row);
  const unsigned char* base = tile + (32 * m2 + row) * RS + (i & 1) * 8;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    const unsigned char* a0 = base + ((y ^ (2 * dt)) << 4);
    union { struct { s16x4 lo, hi; } s; bf16x8 v; } u;
    u.s.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a0);
    u.s.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a0 + 16 * RS));
    col[dt] = u.v;
  }
}
// acc[t][dt] += Tile^T[d tile dt][rows 32 m2 .. 32 m2 + 31] * P[t]: P0 / P1 are the packed accumulator tiles of rows 0..15 / 16..31 of that range
template <typename T, int NDT, int RT>
__device__ __forceinline__ void mma_columns(const bf16x8 (&col)[NDT], const uint2 (&P0)[RT], const uint2 (&P1)[RT], f32x4 (&acc)[RT][NDT]) {
  union { struct { uint2 lo, hi; } w; bf16x8 v; } pb[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    pb[t].w.lo = P0[t];
    pb[t].w.hi = P1[t];
  }
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t][dt] = mfma16<T>(col[dt], pb[t].v, acc[t][dt]);
}
template <typename T, int NDT, int RT>
__device__ __forceinline__ void wmma_transposed(const unsigned char* tile, int m2, const typename Half2<T>::type (&P0)[RT], const typename Half2<T>::type (&P1)[RT],
                                                f32x4 (&acc)[RT][NDT], int lane) {
  if constexpr (sizeof(T) == 2) {
    bf16x8 col[NDT];
    tile_columns<T, NDT>(tile, m2, col, lane);
    mma_columns<T, NDT, RT>(col, P0, P1, acc);
  } else {
    const int i = lane & 15, q = lane >> 4;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 32 * m2 + 16 * half + 4 * q + e;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const float a = *reinterpret_cast<const float*>(tile + WT<T, NDT>::place(row, 4 * dt + (i >> 2)) + (i & 3) * 4);
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, half ? P1[t][e] : P0[t][e], acc[t][dt], 0, 0, 0);
        }
      }
  }
}

// Waits for a fragment's loads here: left to its first use inside a loop, the wait would count the loop's own loads in flight as well (the counter is in
// order, and on the way into the loop there are none behind it) -- every tile would wait for the next one's.
template <typename F> __device__ __forceinline__ void landed(F& f) { asm volatile("" : "+v"(f)); }

// 64 rows of two tensors (K and V, or q and dout) on their way from memory to an LDS tile pair: fetch() requests them into registers, deposit()
// stores them -- a tile later, so that the latency lies under the tile in between.  A thread owns one 16-byte column of every RP-th row; where
// its rows lie from the tile's first one is the same for every tile (x_of, y_of: 32-bit byte offsets), so a whole tile costs a load per
// piece and no address arithmetic.
template <typename T, int NDT, int NT> struct Mover {
  typedef WT<T, NDT> W;
  static constexpr int VEC = WT<T, NDT>::VEC;
  static constexpr int CP = W::CP;                 // columns of a row's LDS room
  static constexpr int RP = NT / CP;               // rows per pass
  static constexpr int NP = 64 / RP;               // passes
  static_assert(NT % CP == 0 && 64 % RP == 0, "whole passes");
  V16 pre[2][NP];
  unsigned x_of[NP], y_of[NP];
  int row, col;
  bool live;
  // off(row, x, y): element offsets of a row from the tile's first row
  template <typename F> __device__ __forceinline__ void init(int dh, F&& off) {
    row = (int)threadIdx.x / CP;
    const int c = (int)threadIdx.x - row * CP;
    col = c * VEC;
    live = col < dh;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      unsigned x, y;
      off(row + j * RP, x, y);
      x_of[j] = (x + col) * sizeof(T);
      y_of[j] = (y + col) * sizeof(T);
    }
  }
  // the whole tile whose first rows are x, y
  __device__ __forceinline__ void fetch_whole(const T* x, const T* y) {
    if (live) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        pre[0][j] = ld16((const char*)x + x_of[j]);
        pre[1][j] = ld16((const char*)y + y_of[j]);
      }
    }
  }
  // at(row, first, second): the addresses of a row's channels in the two tensors; false: zeros
  template <typename F> __device__ __forceinline__ void fetch(F&& at) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      pre[0][j] = pre[1][j] = v16_zero();
      const T *x, *y;
      if (live && at(row + j * RP, x, y)) {
        pre[0][j] = ld16(x + col);
        pre[1][j] = ld16(y + col);
      }
    }
  }
  __device__ __forceinline__ void deposit(unsigned char* pair) const {
    if (live) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        // (rows 16 apart share their twist)
        const int at = sizeof(T) == 4 || RP % 16 == 0 ? W::place(row, col / VEC) + j * RP * W::RS : W::place(row + j * RP, col / VEC);
        st16(pair + at, pre[0][j]);
        st16(pair + W::TILE + at, pre[1][j]);
      }
    }
  }
};

// The same pair of tiles loaded straight into LDS (16-bit modes: rows without padding), 1 KiB of neighbouring places per wave and load: no registers in between (dk / dv of
// 64 channels: 254 -> 236), no LDS writes.  Lane i of a load fills the i-th 16 bytes behind the wave's; the twist is in WHICH piece of its row it asks for.
// (Issued from an asm statement: the compiler neither counts these loads nor drains them in front of LDS reads, `dma_wait` and the barrier order them.)
typedef __attribute__((address_space(3))) const unsigned char* lds_ptr_t;
template <typename T, int NDT, int NT> struct Dma {
  typedef WT<T, NDT> W;
  static constexpr int CP = W::CP, RP = NT / CP, NP = 64 / RP, LOADS = 2 * NP;
  static_assert(sizeof(T) == 2 && NT % CP == 0 && RP % 16 == 0 && 64 % RP == 0, "whole passes, one twist per thread");
  unsigned x_of[NP], y_of[NP], wave0;
  int row, col;
  bool live;
  template <typename F> __device__ __forceinline__ void init(int dh, F&& off) {
    row = (int)threadIdx.x / CP;
    col = (((int)threadIdx.x - row * CP) ^ W::twist(row)) * W::VEC;
    live = col < dh;
    wave0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      unsigned x, y;
      off(row + j * RP, x, y);
      x_of[j] = (x + col) * sizeof(T);
      y_of[j] = (y + col) * sizeof(T);
    }
  }
  static __device__ __forceinline__ void load(const char* src, unsigned dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(dst) : "memory");
  }
  // four bytes per lane
  static __device__ __forceinline__ void word(const float* src, unsigned dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(dst) : "memory");
  }
  // the whole tile whose first rows are x, y to the pair of tiles at `pair`
  __device__ __forceinline__ void whole(const T* x, const T* y, unsigned pair) const {
    if (live) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        load((const char*)x + x_of[j], pair + wave0 + j * RP * W::RS);
        load((const char*)y + y_of[j], pair + wave0 + j * RP * W::RS + W::TILE);
      }
    }
  }
  // at(row, first, second): the addresses of a row's channels in the two tensors
  template <typename F> __device__ __forceinline__ void rows(F&& at, unsigned pair) const {
    if (live) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const T *x, *y;
        at(row + j * RP, x, y);
        load((const char*)(x + col), pair + wave0 + j * RP * W::RS);
        load((const char*)(y + col), pair + wave0 + j * RP * W::RS + W::TILE);
      }
    }
  }
};
// all of this wave's loads but the N newest are there, and so is what every wave wrote; then the others' too
template <int N> __device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

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
// Which of a tile's 64 keys (or rows) a lane's row (key) meets, as one bit each: [lo, hi) and [0, first).  The lane keeps those at 4 q + e of every 16.
struct Meets {
  unsigned w[2];
  Meets() = default;
  static __device__ __forceinline__ unsigned long long below(int n) { return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1ull; }
  __device__ __forceinline__ Meets(int lo, int hi, int first, int q) {
    const unsigned long long m = (below(hi) & ~below(lo)) | below(first);
    w[0] = (unsigned)m >> (4 * q);
    w[1] = (unsigned)(m >> 32) >> (4 * q);
  }
  __device__ __forceinline__ int bits(int n16, int e) const { return __builtin_amdgcn_sbfe((int)w[n16 >> 1], 16 * (n16 & 1) + e, 1); }   // 0 or -1
  __device__ __forceinline__ float or_less(float x, int n16, int e) const {                                                             // x, or -inf
    const unsigned m = (unsigned)bits(n16, e);
    return __uint_as_float((__float_as_uint(x) & m) | (0xff800000u & ~m));
  }
  __device__ __forceinline__ float or_zero(float x, int n16, int e) const { return __uint_as_float(__float_as_uint(x) & (unsigned)bits(n16, e)); }
};

// One 64-key tile of the online softmax: s (keys x rows; a lane holds row t's keys 16 kb + 4 q + e) becomes the tile's probabilities up to the rows' running
// maximum, packed in ph; m, l and the sums o are brought to it.
template <typename T, int RT, bool MASKED, int NDT>
__device__ __forceinline__ void softmax_step(const WinArgs& a, f32x4 (&s)[4][RT], typename Half2<T>::type (&ph)[4][RT], int s0, int klen, const int (&pos)[RT], float (&m)[RT], float (&l)[RT],
                                             f32x4 (&o)[RT][NDT], int q) {
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float mx = -INFINITY;
    const int hi = min(klen, pos[t] + a.right + 1) - s0;
    const Meets meets(MASKED ? pos[t] - a.left - s0 : 0, hi, MASKED ? min(a.sinks - s0, hi) : 0, q);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (MASKED) s[kb][t][e] = meets.or_less(s[kb][t][e], kb, e);
        mx = fmaxf(mx, s[kb][t][e]);
      }
    // The reference that the exponents are taken against is moved only when a row's maximum has outgrown it by 2^8: P then stays below 256, which
    // costs no precision, and most tiles leave the sums as they are (moved at every new maximum, 60 % of a long window's tiles rescaled them).
    mx = xor_max(mx) * a.c;                                                   // c > 0: the maximum commutes with it
    if (__any(mx > m[t] + 8.f)) {
      const float mnew = fmaxf(m[t], mx), alpha = fast_exp2(m[t] - (mnew == -INFINITY ? 0.f : mnew));
      m[t] = mnew;
      l[t] *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][dt][e] *= alpha;
    }
    const float ref = m[t] == -INFINITY ? 0.f : m[t];                         // (a row that has seen nothing yet)
    float rs = 0.f;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = fast_exp2(fmaf(s[kb][t][e], a.c, -ref));
        rs += p;
        s[kb][t][e] = p;
      }
      ph[kb][t] = Half2<T>::pack(s[kb][t]);
    }
    l[t] += xor_sum(rs);
  }
}

// Pairs of 64-key tiles in LDS: the one in use and those on their way.  A second one on its way helps where workgroups share the keys and a CU holds one of them
// (16 frames against 65536: 28 -> 25.5 us); with several on a CU the others' work covers the loads (ten minutes of audio, forward: two 226 us, three 234).
template <typename T, bool SPLIT> constexpr int key_bufs() { return sizeof(T) == 2 && SPLIT ? 3 : 2; }

// A workgroup's walk over its tiles [kt0, kt1) of keys: work(tile's LDS, first key) on each, loads one or two tiles ahead.
template <typename T, int NDT, int BUFS, typename F>
__device__ __forceinline__ void walk_keys(const WinArgs& a, const TileWalk& walk, int kt0, int kt1, const T* kb_, const T* vb_, unsigned char* lds, F&& work) {
  typedef WT<T, NDT> W;
  const auto places = [&](int row, unsigned& x, unsigned& y) { x = row * (unsigned)a.k_ts; y = row * (unsigned)a.v_ts; };
  const auto whole = [&](int s0) { return s0 + 64 <= walk.hi && (s0 >= walk.lo || s0 + 64 <= a.sinks); };
  if constexpr (sizeof(T) == 2) {
    constexpr int AHEAD = BUFS - 1, LOADS = Dma<T, NDT, 256>::LOADS;
    Dma<T, NDT, 256> dma;
    dma.init(a.dh, places);
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)((lds_ptr_t)lds));
    auto send = [&](int kt, int buf) {
      const int s0 = walk.key0(kt);
      const unsigned pair = lds0 + buf * 2 * W::TILE;
      if (whole(s0)) dma.whole(kb_ + s0 * a.k_ts, vb_ + s0 * a.v_ts, pair);
      else
        dma.rows([&](int m, const T*& x, const T*& y) {
          // what no row here sees is not read: the nearest key that one sees instead, its probabilities are 0
          int s = s0 + m;
          if (s >= walk.hi || (s < walk.lo && s >= a.sinks)) s = walk.lo < walk.hi ? max(walk.lo, min(s, walk.hi - 1)) : 0;
          x = kb_ + s * a.k_ts;
          y = vb_ + s * a.v_ts;
        }, pair);
    };
    // A tile is sent for AHEAD tiles before it is worked on, to where the tile before the present one was: every wave has passed the barrier behind that.
    const int n = kt1 - kt0;
    for (int k = 0; k < AHEAD && k < n; ++k) send(kt0 + k, k);
    int buf = 0;
    for (int k = 0; k < n; ++k) {
      if (AHEAD == 2 && k + 1 < n) dma_wait<LOADS>();
      else dma_wait<0>();
      if (k + AHEAD < n) send(kt0 + k + AHEAD, buf == 0 ? BUFS - 1 : buf - 1);
      work(lds + buf * 2 * W::TILE, walk.key0(kt0 + k));
      buf = buf == BUFS - 1 ? 0 : buf + 1;
    }
  } else {
    Mover<T, NDT, 256> mv;
    mv.init(a.dh, places);
    auto fetch = [&](int s0) {
      if (whole(s0)) return mv.fetch_whole(kb_ + s0 * a.k_ts, vb_ + s0 * a.v_ts);
      mv.fetch([&](int row, const T*& x, const T*& y) {
        const int s = s0 + row;
        x = kb_ + s * a.k_ts;
        y = vb_ + s * a.v_ts;
        return s < walk.hi && (s >= walk.lo || s < a.sinks);                     // what no row here sees is not read
      });
    };
    if (kt0 < kt1) fetch(walk.key0(kt0));
    for (int kt = kt0; kt < kt1; ++kt) {
      unsigned char* tiles = lds + ((kt - kt0) & 1) * 2 * W::TILE;
      // the buffer's readers of two tiles ago have all passed the barrier of the tile in between
      mv.deposit(tiles);
      __syncthreads();
      if (kt + 1 < kt1) fetch(walk.key0(kt + 1));
      work(tiles, walk.key0(kt));
    }
  }
}

// Where several workgroups share a row block's keys: part[entry][head][share][row][dh] sums, behind them [entry][head][share][row] maximum and sum.
__device__ __forceinline__ long share_row(const WinArgs& a, int b, int h, int split, int row) { return (((long)b * a.Hkv + h) * a.nsplit + split) * a.rows + row; }
__device__ __forceinline__ float2* share_stat(const WinArgs& a, float* part, long n) {
  return reinterpret_cast<float2*>(part + (long)a.B * a.Hkv * a.nsplit * a.rows * a.dh) + n;
}

template <typename T, int NDT, int RT, bool SPLIT>
__global__ void __launch_bounds__(256, (WT<T, NDT>::OCC)) win_fwd_kernel(WinArgs a, const T* __restrict__ q_, const T* __restrict__ k_, const T* __restrict__ v_,
                                                          T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part) {
  typedef WT<T, NDT> W;
  constexpr int NK = W::NK;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  int blk, h, bz;
  win_block(blk, h, bz);
  const int split = SPLIT ? bz % a.nsplit : 0, b = SPLIT ? bz / a.nsplit : bz;
  const int base = a.enter(b);
  const int g0 = blk * 64 * RT, g1 = min(g0 + 64 * RT, a.rows) - 1;            // the workgroup's rows
  const int w0 = g0 + wave * 16 * RT, w1 = min(w0 + 16 * RT, a.rows) - 1;                // the wave's
  const TileWalk walk(a, b, base + a.frame(g0), base + a.frame(g1));
  const int wp0 = base + a.frame(min(w0, g1)), wp1 = base + a.frame(max(w1, 0));
  const T* qb = q_ + b * a.q_bs;
  const T* kb_ = k_ + b * a.k_bs + h * a.k_hs;
  const T* vb_ = v_ + b * a.v_bs + h * a.v_hs;
  zero_lds<T>(lds, 2 * key_bufs<T, SPLIT>() * W::TILE);                                               // (channels past dh are never written again)
  typename W::frag qf[RT][NK];
  int pos[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = w0 + 16 * t + r, i = a.frame(row), g = row - i * a.G;
    pos[t] = base + i;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) qf[t][ks] = gfrag<T>(qb + i * a.q_ts + (long)(h * a.G + g) * a.q_hs, row < a.rows, ks, lane, a.dh);
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) landed(qf[t][ks]);
  const int per = SPLIT ? (walk.n + a.nsplit - 1) / a.nsplit : walk.n;
  const int kt0 = split * per, kt1 = min(walk.n, kt0 + per);
  float m[RT], l[RT];
  f32x4 o[RT][NDT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto compute = [&](const unsigned char* Ks, int s0, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const unsigned char* Vs = Ks + W::TILE;
    f32x4 s[4][RT];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int t = 0; t < RT; ++t) s[kb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        const typename W::frag f = wfrag<T, NDT>(Ks, kb, ks, lane);
#pragma unroll
        for (int t = 0; t < RT; ++t) s[kb][t] = mma<T>(f, qf[t][ks], s[kb][t]);
      }
    }
    typename Half2<T>::type ph[4][RT];
    softmax_step<T, RT, MASKED>(a, s, ph, s0, walk.klen, pos, m, l, o, q);
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2) wmma_transposed<T, NDT, RT>(Vs, m2, ph[2 * m2], ph[2 * m2 + 1], o, lane);
  };

  walk_keys<T, NDT, key_bufs<T, SPLIT>()>(a, walk, kt0, kt1, kb_, vb_, lds, [&](const unsigned char* Ks, int s0) {
    const int sight = w0 < a.rows ? tile_sight(a, walk.klen, s0, wp0, wp1) : 0;
    if (sight == 2) compute(Ks, s0, std::false_type{});
    else if (sight == 1) compute(Ks, s0, std::true_type{});
  });

#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = w0 + 16 * t + r;
    if (row >= a.rows) continue;
    const int i = a.frame(row), g = row - i * a.G;
    if constexpr (SPLIT) {
      float* dst = part + share_row(a, b, h, split, row) * a.dh;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const int d = 16 * dt + 4 * q;
        if (d < a.dh) *reinterpret_cast<f32x4*>(dst + d) = o[t][dt];
      }
      if (q == 0) *share_stat(a, part, share_row(a, b, h, split, row)) = make_float2(m[t], l[t]);
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

// A few rows (at most 16 TT per key head: one new frame's query heads, or some frames') against a cache.  What counts is how many keys are on their way at a
// time, so the four waves of a workgroup walk tiles of their own, without a barrier: keys go straight from memory into the first product's operand
// registers, values through a tile of LDS that only this wave uses, and both are requested a tile ahead.  The waves' sums meet at the end.
template <typename T, int NDT, int TT>
__global__ void __launch_bounds__(256, NDT * TT * (int)sizeof(T) > 12 ? 1 : 2) win_few_kernel(WinArgs a, const T* __restrict__ q_, const T* __restrict__ k_,
                                                                                    const T* __restrict__ v_, T* __restrict__ out, float* __restrict__ lse,
                                                                                    float* __restrict__ part) {
  typedef WT<T, NDT> W;
  constexpr int NK = W::NK, CP = NDT * 16 / W::VEC;    // 16-byte pieces of a row = per lane and tile
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int base = a.enter(b);
  const int wp0 = base, wp1 = base + a.Tq - 1;
  const TileWalk walk(a, b, wp0, wp1);
  const T* qb = q_ + b * a.q_bs;
  const T* kb_ = k_ + b * a.k_bs + h * a.k_hs;
  const T* vb_ = v_ + b * a.v_bs + h * a.v_hs;
  unsigned char* tile = lds + wave * W::TILE;
  typename W::frag qf[TT][NK], kf[4][NK];
  V16 vf[CP];
  int pos[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int row = 16 * t + r, i = a.frame(row), g = row - i * a.G;
    pos[t] = base + i;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) qf[t][ks] = gfrag<T>(qb + i * a.q_ts + (long)(h * a.G + g) * a.q_hs, row < a.rows, ks, lane, a.dh);
  }
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) landed(qf[t][ks]);
  const int per = (walk.n + a.nsplit - 1) / a.nsplit, kt1 = min(walk.n, (split + 1) * per);
  auto fetch = [&](int s0) {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const int s = s0 + 16 * kb + r;
      const bool live = s < walk.hi && (s >= walk.lo || s < a.sinks);
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) kf[kb][ks] = gfrag<T>(kb_ + s * a.k_ts, live, ks, lane, a.dh);
    }
#pragma unroll
    for (int j = 0; j < CP; ++j) {
      const int at = j * 64 + lane, row = at / CP, col = (at % CP) * W::VEC, s = s0 + row;
      vf[j] = v16_zero();
      if (s < walk.hi && (s >= walk.lo || s < a.sinks) && col < a.dh) vf[j] = ld16(vb_ + s * a.v_ts + col);
    }
  };
  float m[TT], l[TT];
  f32x4 o[TT][NDT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int kt = split * per + wave;
  if (kt < kt1) fetch(walk.key0(kt));
  for (; kt < kt1; kt += 4) {
    const int s0 = walk.key0(kt);
    f32x4 s[4][TT];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        s[kb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) s[kb][t] = mma<T>(kf[kb][ks], qf[t][ks], s[kb][t]);
      }
#pragma unroll
    for (int j = 0; j < CP; ++j) {
      const int at = j * 64 + lane;
      st16(tile + W::place(at / CP, at % CP), vf[j]);
    }
    if (kt + 4 < kt1) fetch(walk.key0(kt + 4));
    typename Half2<T>::type ph[4][TT];
    if (tile_sight(a, walk.klen, s0, wp0, wp1) == 2) softmax_step<T, TT, false>(a, s, ph, s0, walk.klen, pos, m, l, o, q);
    else softmax_step<T, TT, true>(a, s, ph, s0, walk.klen, pos, m, l, o, q);
    // (a wave reads only what it wrote itself, and the LDS serves one wave's accesses in order: only the compiler has to be held back)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2) wmma_transposed<T, NDT, TT>(tile, m2, ph[2 * m2], ph[2 * m2 + 1], o, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // the four waves' sums: [wave][row][NDT * 16] over the tiles, the maxima and sums behind them
  constexpr int D = NDT * 16;
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);
  float* ml = sums + 4 * 16 * TT * D;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(sums + ((wave * TT + t) * 16 + r) * D + 16 * dt + 4 * q) = o[t][dt];
    if (q == 0) {
      ml[((wave * TT + t) * 16 + r) * 2] = m[t];
      ml[((wave * TT + t) * 16 + r) * 2 + 1] = l[t];
    }
  }
  __syncthreads();
  for (int n = threadIdx.x; n < a.rows * (D / 4); n += 256) {
    const int row = n / (D / 4), d = (n - row * (D / 4)) * 4;
    float top = -INFINITY, w[4], sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[(k * 16 * TT + row) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = fast_exp2(ml[(k * 16 * TT + row) * 2] - ref);
      sum += w[k] * ml[(k * 16 * TT + row) * 2 + 1];
      const f32x4 x = *reinterpret_cast<const f32x4*>(sums + (k * 16 * TT + row) * D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += w[k] * x[e];
    }
    if (d >= a.dh) continue;
    if (a.nsplit > 1) {
      const long n2 = share_row(a, b, h, split, row);
      *reinterpret_cast<f32x4*>(part + n2 * a.dh + d) = f32x4{v[0], v[1], v[2], v[3]};
      if (d == 0) *share_stat(a, part, n2) = make_float2(top, sum);
    } else {
      const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
      const int i = a.frame(row), g = row - i * a.G;
      const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
      if (d == 0 && lse) lse[orow] = sum == 0.f ? INFINITY : top + log2f(sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= inv;
      st4(out + orow * a.dh + d, v);
    }
  }
}

// Joins the shares of a row (at most 256), a workgroup per row: a thread per share for the weights, then 16 bytes of a share per thread, added over the groups of
// threads in their order.
template <typename T>
__global__ void __launch_bounds__(256) win_join_kernel(const WinArgs a, float* __restrict__ part, T* __restrict__ out, float* __restrict__ lse) {
  __shared__ float weight[256], acc[1024], top[4], total[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long n = blockIdx.x;                                     // row of [entry][head][row]
  const int row = (int)(n % a.rows);
  const long bh = n / a.rows;
  const int h = (int)(bh % a.Hkv), b = (int)(bh / a.Hkv), per = a.dh > 64 ? 32 : 16, c = tid % per * 4, first = tid / per, groups = 256 / per;
  const long at = share_row(a, b, h, 0, row);
  const float2 st = tid < a.nsplit ? *share_stat(a, part, at + (long)tid * a.rows) : make_float2(-INFINITY, 0.f);
  const float wm = wave_max(st.x);
  if (lane == 0) top[wave] = wm;
  __syncthreads();
  const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), ref = m == -INFINITY ? 0.f : m, w = fast_exp2(st.x - ref);
  weight[tid] = w;
  const float ws = wave_sum(w * st.y);
  if (lane == 0) total[wave] = ws;
  __syncthreads();
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < a.dh) {
#pragma unroll 8
    for (int s = first; s < a.nsplit; s += groups) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(part + (at + (long)s * a.rows) * a.dh + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += weight[s] * x[e];
    }
  }
  *reinterpret_cast<f32x4*>(acc + tid * 4) = f32x4{o[0], o[1], o[2], o[3]};
  __syncthreads();
  const int i = a.frame(row), g = row - i * a.G;
  const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
  const float l = total[0] + total[1] + total[2] + total[3], inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  if (tid == 0 && lse) lse[orow] = l == 0.f ? INFINITY : m + log2f(l);
  if (tid < a.dh) {
    float v = 0.f;
    for (int k = 0; k < groups; ++k) v += acc[k * per * 4 + tid];
    out[orow * a.dh + tid] = from_f<T>(v * inv);
  }
}

// ------------------------------------------------------------------------------------------------ backward: dq, and D for the other pass
template <typename T, int NDT, int RT>
__global__ void __launch_bounds__(256, (WT<T, NDT>::OCC)) win_dq_kernel(WinArgs a, const T* __restrict__ q_, const T* __restrict__ k_, const T* __restrict__ v_,
                                                         const T* __restrict__ out, const T* __restrict__ dout, const float* __restrict__ lse,
                                                         float* __restrict__ delta, T* __restrict__ dq) {
  typedef WT<T, NDT> W;
  constexpr int NK = W::NK;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  int blk, h, b;
  win_block(blk, h, b);
  const int base = a.enter(b);
  const int g0 = blk * 64 * RT, g1 = min(g0 + 64 * RT, a.rows) - 1;
  const int w0 = g0 + wave * 16 * RT, w1 = min(w0 + 16 * RT, a.rows) - 1;
  const TileWalk walk(a, b, base + a.frame(g0), base + a.frame(g1));
  const int wp0 = base + a.frame(min(w0, g1)), wp1 = base + a.frame(max(w1, 0));
  const T* qb = q_ + b * a.q_bs;
  const T* kb_ = k_ + b * a.k_bs + h * a.k_hs;
  const T* vb_ = v_ + b * a.v_bs + h * a.v_hs;
  zero_lds<T>(lds, 2 * key_bufs<T, false>() * W::TILE);
  typename W::frag qf[RT][NK], gf[RT][NK];
  int pos[RT];
  float ls[RT], dl[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = w0 + 16 * t + r, i = a.frame(row), g = row - i * a.G;
    const bool live = row < a.rows;
    const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
    pos[t] = base + i;
    ls[t] = live ? lse[orow] : INFINITY;
    if constexpr (W::SCALED) ls[t] -= log2f(a.scale);   // the exponential gives scale P
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
    dl[t] = xor_sum(d);   // (of the rounded output: in 32 bits it would cost its bytes again in both directions)
    if (live && q == 0) delta[orow] = -dl[t];   // (as the other pass wants it)
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    landed(ls[t]);
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      landed(qf[t][ks]);
      landed(gf[t][ks]);
    }
  }
  f32x4 acc[RT][NDT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) acc[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const unsigned char* Ks, int s0, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const unsigned char* Vs = Ks + W::TILE;
    Meets meets[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
      if constexpr (MASKED) {
        const int hi = min(walk.klen, pos[t] + a.right + 1) - s0;
        meets[t] = Meets(pos[t] - a.left - s0, hi, min(a.sinks - s0, hi), q);
      }
#pragma unroll
    for (int m2 = 0; m2 < 2; ++m2) {
      typename Half2<T>::type dsh[2][RT];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int kb = 2 * m2 + kk;
        f32x4 s[RT], dp[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
          dp[t] = f32x4{-dl[t], -dl[t], -dl[t], -dl[t]};   // dP - D out of the product itself
        }
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
          const typename W::frag f = wfrag<T, NDT>(Ks, kb, ks, lane), fv = wfrag<T, NDT>(Vs, kb, ks, lane);
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            s[t] = mma<T>(f, qf[t][ks], s[t]);
            dp[t] = mma<T>(fv, gf[t][ks], dp[t]);
          }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float p = fast_exp2(fmaf(s[t][e], a.c, -ls[t]));
            if constexpr (MASKED) p = meets[t].or_zero(p, kb, e);
            s[t][e] = p * dp[t][e];                        // dS / scale (SCALED: dS)
          }
          dsh[kk][t] = Half2<T>::pack(s[t]);
        }
      }
      wmma_transposed<T, NDT, RT>(Ks, m2, dsh[0], dsh[1], acc, lane);
    }
  };
  walk_keys<T, NDT, key_bufs<T, false>()>(a, walk, 0, walk.n, kb_, vb_, lds, [&](const unsigned char* Ks, int s0) {
    const int sight = w0 < a.rows ? tile_sight(a, walk.klen, s0, wp0, wp1) : 0;
    if (sight == 2) compute(Ks, s0, std::false_type{});
    else if (sight == 1) compute(Ks, s0, std::true_type{});
  });
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = w0 + 16 * t + r;
    if (row >= a.rows) continue;
    const int i = a.frame(row), g = row - i * a.G;
    const long orow = ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const int d = 16 * dt + 4 * q;
      if (d < a.dh) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ls[t] == INFINITY ? 0.f : W::SCALED ? acc[t][dt][e] : acc[t][dt][e] * a.scale;   // (a row without keys: whatever its gradient holds)
        st4(dq + orow * a.dh + d, w);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
// A workgroup owns 64 KT keys (16 KT per wave) of one key head and walks the 64-row tiles that see them: nkb blocks per head, and where the blocks that hold sinks are
// shared (nsink of them) nsplit workgroups with partial sums for each.
template <typename T, int NDT, int KT>
__global__ void __launch_bounds__(256, (WT<T, NDT>::OCC)) win_dkv_kernel(WinArgs a, const T* __restrict__ q_, const T* __restrict__ k_, const T* __restrict__ v_,
                                                      const T* __restrict__ dout, const float* __restrict__ lse, const float* __restrict__ delta,
                                                      T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part, int nkb) {
  typedef WT<T, NDT> W;
  constexpr int NK = W::NK;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  constexpr bool DMA = sizeof(T) == 2;
  float* rowdata = reinterpret_cast<float*>(lds + 4 * W::TILE);   // two buffers of 64 x (lse | -D)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  // one dimension: all blocks that are not shared first (each XCD a contiguous range: neighbours read the same rows), then the sink blocks' shares, which are
  // short and fill the CUs that the last round of the others leaves idle
  const int heads = a.B * a.Hkv, whole = heads * nkb, lin = blockIdx.x;
  const bool shared = lin >= whole;
  int kb, split = 0, bh;
  if (shared) {
    const int n = lin - whole, s = n / heads;
    bh = n - s * heads;
    kb = s / a.nsplit;
    split = s - kb * a.nsplit;
  } else {
    const int per = whole >> 3, rem = whole & 7, xcd = lin & 7, lg = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + (lin >> 3);
    bh = lg / nkb;
    kb = lg - bh * nkb + a.nsink;
  }
  const int b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int base = a.enter(b);
  const int klen = a.key_len ? max(0, min(a.key_len[b], a.Tk)) : a.Tk;
  const int s0 = kb * 64 * KT, k0 = s0 + wave * 16 * KT;                   // first key of the workgroup, of the wave
  const T* qb = q_ + b * a.q_bs;
  zero_lds<T>(lds, 4 * W::TILE);
  typename W::frag kf[KT][NK], vf[KT][NK];
  int rlo[KT], rhi[KT];                                           // rows [rlo, rhi) see this lane's keys
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int s = k0 + 16 * t + r;
    rlo[t] = max(0, min(a.Tq, s - a.right - base)) * a.G;
    rhi[t] = s >= klen ? 0 : s < a.sinks ? a.rows : max(0, min(a.Tq, s + a.left - base + 1)) * a.G;
    // a key that no row sees is not read: with zeros its dP is finite, so that its probabilities of 0 leave 0 of it
    const bool met = s < klen && rlo[t] < rhi[t];
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      kf[t][ks] = gfrag<T>(k_ + b * a.k_bs + h * a.k_hs + s * a.k_ts, met, ks, lane, a.dh);
      vf[t][ks] = gfrag<T>(v_ + b * a.v_bs + h * a.v_hs + s * a.v_ts, met, ks, lane, a.dh);
    }
  }
  // rows that see a key of this block: frames [f0, f1), then the workgroup's share of their 64-row tiles
  const int last = min(s0 + 64 * KT, klen) - 1;
  const int f0 = max(0, min(a.Tq, s0 - a.right - base));
  const int f1 = last < s0 ? f0 : s0 < a.sinks ? a.Tq : max(f0, min(a.Tq, last + a.left - base + 1));
  const int row0 = f0 * a.G, row1 = f1 * a.G;
  const int nt = (row1 - row0 + 63) >> 6, per = shared ? (nt + a.nsplit - 1) / a.nsplit : nt;
  const int t0 = split * per, t1 = min(nt, t0 + per);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      landed(kf[t][ks]);
      landed(vf[t][ks]);
    }
  // (a tile's first row is a frame's first head where 64 rows are whole frames: then its rows lie at the same places in every tile)
  const auto places = [&](int row, unsigned& x, unsigned& y) {
    const int i = a.frame(row), g = row - i * a.G;
    x = i * (unsigned)a.q_ts + g * (unsigned)a.q_hs;
    y = (i * (unsigned)a.Hq + g) * (unsigned)a.dh;
  };
  const auto address = [&](int row, const T*& x, const T*& y) {
    const int i = a.frame(row), g = row - i * a.G;
    x = qb + i * a.q_ts + (long)(h * a.G + g) * a.q_hs;
    y = dout + (((long)b * a.Tq + i) * a.Hq + h * a.G + g) * a.dh;
  };
  const bool even = 64 % a.G == 0;
  const auto stat = [&](int row) {   // a row's place in lse and delta
    const int i = a.frame(row), g = row - i * a.G;
    return ((long)b * a.Tq + i) * a.Hq + h * a.G + g;
  };
  f32x4 ak[KT][NDT], av[KT][NDT];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) ak[t][dt] = av[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const unsigned char* Qs, const float* rd, int first_row, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    Meets meets[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
      if constexpr (MASKED) meets[t] = Meets(rlo[t] - first_row, rhi[t] - first_row, 0, q);
    const unsigned char* Gs = Qs + W::TILE;
    // Three stages per 16 rows: the products S and dP - D, the probabilities and dS out of them, the products that sum dv and dk (32 rows at a
    // time).  They are issued one behind the other's successor -- the first stage of rows n + 1 with the second of rows n --, so that the matrix
    // pipe has work of this wave while its vector instructions run; two waves per SIMD alone leave both idle half of the time.
    f32x4 p[2][KT], ds[2][KT];
    typename Half2<T>::type ph[2][KT], dsh[2][KT];
    typename W::frag fq[2][NK], fg[2][NK];
    auto load = [&](int rb) {
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        fq[rb & 1][ks] = wfrag<T, NDT>(Qs, rb, ks, lane);
        fg[rb & 1][ks] = wfrag<T, NDT>(Gs, rb, ks, lane);
      }
    };
    auto first = [&](int rb) {
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(rd + 64 + 16 * rb + 4 * q);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        p[rb & 1][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        ds[rb & 1][t] = d4;                                  // -D: dP - D out of the product itself
      }
#pragma unroll
      for (int ks = 0; ks < NK; ++ks)
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          p[rb & 1][t] = mma<T>(fq[rb & 1][ks], kf[t][ks], p[rb & 1][t]);
          ds[rb & 1][t] = mma<T>(fg[rb & 1][ks], vf[t][ks], ds[rb & 1][t]);
        }
    };
    auto soft = [&](int rb) {
      const f32x4 l4 = *reinterpret_cast<const f32x4*>(rd + 16 * rb + 4 * q);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float w = fast_exp2(fmaf(p[rb & 1][t][e], a.c, -l4[e]));
          if constexpr (MASKED) w = meets[t].or_zero(w, rb, e);
          p[rb & 1][t][e] = w;
          ds[rb & 1][t][e] *= W::SCALED ? w * a.scale : w;   // dS / scale (SCALED: dS)
        }
        ph[rb & 1][t] = Half2<T>::pack(p[rb & 1][t]);
        dsh[rb & 1][t] = Half2<T>::pack(ds[rb & 1][t]);
      }
    };
#define FH_STAGE __builtin_amdgcn_sched_barrier(0);
    if constexpr (sizeof(T) == 2) {
      bf16x8 cg[NDT], cq[NDT];
      load(0);
      FH_STAGE load(1); first(0);
      FH_STAGE load(2); first(1); soft(0);
      FH_STAGE load(3); tile_columns<T, NDT>(Gs, 0, cg, lane); first(2); soft(1);
      FH_STAGE tile_columns<T, NDT>(Qs, 0, cq, lane); mma_columns<T, NDT, KT>(cg, ph[0], ph[1], av); 
      FH_STAGE tile_columns<T, NDT>(Gs, 1, cg, lane); mma_columns<T, NDT, KT>(cq, dsh[0], dsh[1], ak); soft(2);
      FH_STAGE first(3); tile_columns<T, NDT>(Qs, 1, cq, lane);
      FH_STAGE soft(3);
      mma_columns<T, NDT, KT>(cg, ph[0], ph[1], av);
      mma_columns<T, NDT, KT>(cq, dsh[0], dsh[1], ak);
    } else {
#pragma unroll
      for (int m2 = 0; m2 < 2; ++m2) {
        load(2 * m2);
        first(2 * m2);
        soft(2 * m2);
        load(2 * m2 + 1);
        first(2 * m2 + 1);
        soft(2 * m2 + 1);
        wmma_transposed<T, NDT, KT>(Gs, m2, ph[0], ph[1], av, lane);
        wmma_transposed<T, NDT, KT>(Qs, m2, dsh[0], dsh[1], ak, lane);
      }
    }
#undef FH_STAGE
  };
  // Neighbouring blocks see mostly the same rows, one block's worth further on.  Each begins its walk where the tile's place among all rows is a multiple of the
  // walk's length (and wraps): the workgroups of an XCD then read the same few tiles at the same time instead of as many as they are, which their
  // L2 does not hold (ten minutes of audio: 403 -> 387 us).
  const int n = t1 - t0;
  int rt = t0 + (n > 0 ? (n - ((row0 >> 6) + t0) % n) % n : 0);
  const auto after = [&](int tile) { return tile + 1 < t1 ? tile + 1 : t0; };
  auto work = [&](int buf, int tile) {
    const unsigned char* Qs = lds + buf * 2 * W::TILE;
    const float* rd = rowdata + buf * 128;
    const int at = row0 + tile * 64;
    // positions of the tile's rows against those that see the wave's keys
    const int p0 = base + a.frame(at), p1 = base + a.frame(min(at + 63, row1 - 1)), ke = min(k0 + 16 * KT, klen) - 1;
    if (ke < k0 || p1 < k0 - a.right || (p0 > ke + a.left && k0 >= a.sinks)) return;
    if (k0 + 16 * KT - 1 < klen && p0 >= k0 + 16 * KT - 1 - a.right && (p1 <= k0 + a.left || k0 + 16 * KT - 1 < a.sinks)) compute(Qs, rd, at, std::false_type{});
    else compute(Qs, rd, at, std::true_type{});
  };
  if constexpr (DMA) {
    Dma<T, NDT, 256> dma;
    dma.init(a.dh, places);
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)((lds_ptr_t)lds));
    auto send = [&](int tile, int buf) {
      const int first = row0 + tile * 64;
      const unsigned pair = lds0 + buf * 2 * W::TILE;
      if (first + 64 <= row1) {
        if (wave == (tile & 3)) {
          const long at = stat(first + lane);
          const unsigned dst = lds0 + 4 * W::TILE + buf * 512;
          dma.word(lse + at, dst);
          dma.word(delta + at, dst + 256);
        }
      } else if (wave == (tile & 3)) {
        const bool there = first + lane < row1;
        const long at = stat(min(first + lane, row1 - 1));
        rowdata[buf * 128 + lane] = there ? lse[at] : INFINITY;   // +inf: the row's probabilities are 0
        rowdata[buf * 128 + 64 + lane] = there ? delta[at] : 0.f;
      }
      if (even && first + 64 <= row1) {
        const T *x, *y;
        address(first, x, y);
        dma.whole(x, y, pair);
      } else {
        // (behind the last row: that row again, with probabilities of 0)
        dma.rows([&](int m, const T*& x, const T*& y) { address(min(first + m, row1 - 1), x, y); }, pair);
      }
    };
    // A tile is sent for when the one in front of it is worked on, to where the one in front of that was: every wave has passed the barrier behind it.  (Two on their way
    // measured no better: with two workgroups on a CU the other's work covers the loads.)
    if (n > 0) send(rt, 0);
    for (int k = 0; k < n; ++k) {
      dma_wait<0>();
      const int next = after(rt);
      if (k + 1 < n) send(next, (k + 1) & 1);
      work(k & 1, rt);
      rt = next;
    }
  } else {
    Mover<T, NDT, 256> mv;
    mv.init(a.dh, places);
    float pre_l = 0.f, pre_d = 0.f;
    auto fetch = [&](int tile) {
      const int first = row0 + tile * 64;
      if (even && first + 64 <= row1) {
        const T *x, *y;
        address(first, x, y);
        mv.fetch_whole(x, y);
      } else {
        mv.fetch([&](int m, const T*& x, const T*& y) {
          address(first + m, x, y);
          return first + m < row1;
        });
      }
      if (threadIdx.x < 64) {
        const bool there = first + lane < row1;
        const long at = stat(min(first + lane, row1 - 1));
        pre_l = there ? lse[at] : INFINITY;                       // +inf: the row's probabilities are 0
        pre_d = there ? delta[at] : 0.f;
      }
    };
    if (n > 0) fetch(rt);
    for (int k = 0; k < n; ++k) {
      mv.deposit(lds + (k & 1) * 2 * W::TILE);
      if (threadIdx.x < 64) {
        rowdata[(k & 1) * 128 + lane] = pre_l;
        rowdata[(k & 1) * 128 + 64 + lane] = pre_d;
      }
      __syncthreads();
      if (k + 1 < n) fetch(after(rt));
      work(k & 1, rt);
      rt = after(rt);
    }
  }
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int s = k0 + 16 * t + r;
    if (s >= a.Tk) continue;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const int d = 16 * dt + 4 * q;
      if (d >= a.dh) continue;
      float wk[4], wv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) { wk[e] = W::SCALED ? ak[t][dt][e] : ak[t][dt][e] * a.scale; wv[e] = av[t][dt][e]; }
      if (shared) {
        // [entry][head][sink block][split][dk | dv][keys][dh]
        float* dst = part + (((((long)b * a.Hkv + h) * a.nsink + kb) * a.nsplit + split) * 2 * 64 * KT + (s - s0)) * a.dh + d;
        st4(dst, wk);
        st4(dst + 64 * KT * a.dh, wv);
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
__global__ void __launch_bounds__(256) win_dkv_join_kernel(const WinArgs a, const float* __restrict__ part, T* __restrict__ dk, T* __restrict__ dv, int keys) {
  const int c4 = a.dh / 4;
  const long n = (long)blockIdx.x * 256 + threadIdx.x, total = (long)a.B * a.Hkv * a.nsink * 2 * keys * c4;
  if (n >= total) return;
  const int c = (int)(n % c4);
  long k = n / c4;
  const int key = (int)(k % keys);
  k /= keys;
  const int which = (int)(k % 2);
  k /= 2;
  const int kb = (int)(k % a.nsink), s = kb * keys + key;
  k /= a.nsink;
  const int h = (int)(k % a.Hkv), b = (int)(k / a.Hkv);
  if (s >= a.Tk) return;
  const float* src = part + (((((long)b * a.Hkv + h) * a.nsink + kb) * a.nsplit * 2 + which) * keys + key) * a.dh + c * 4;
  float sum[4] = {0.f, 0.f, 0.f, 0.f}, f[4];
#pragma unroll 8
  for (int i = 0; i < a.nsplit; ++i) {
    ld4(src + (long)i * 2 * keys * a.dh, f);
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

template <typename T, int NDT, int RT, bool SPLIT>
int run_fwd(const WinArgs& a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st) {
  const size_t smem = 2 * key_bufs<T, SPLIT>() * WT<T, NDT>::TILE;
  if (int rc = set_lds(win_fwd_kernel<T, NDT, RT, SPLIT>, smem)) return rc;
  const dim3 grid((a.rows + 64 * RT - 1) / (64 * RT), a.Hkv, a.B * a.nsplit), block(256);
  hipLaunchKernelGGL((win_fwd_kernel<T, NDT, RT, SPLIT>), grid, block, smem, st, a, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, part);
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename T, int NDT, int TT>
int run_few(const WinArgs& a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st) {
  const size_t ends = 4 * 16 * TT * (NDT * 16 + 2) * 4, tiles = 4 * WT<T, NDT>::TILE, smem = ends > tiles ? ends : tiles;
  if (int rc = set_lds(win_few_kernel<T, NDT, TT>, smem)) return rc;
  hipLaunchKernelGGL((win_few_kernel<T, NDT, TT>), dim3(a.nsplit, a.Hkv, a.B), dim3(256), smem, st, a, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, part);
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename T, int NDT>
int fwd_t(WinArgs a, const void* q, const void* k, const void* v, void* out, float* lse, float* part, hipStream_t st) {
  const WinPlan p = fwd_plan(a, ElemTraits<T>::DT);
  a.nsplit = p.nsplit;
  int rc;
  if (p.few) {
    if constexpr (sizeof(T) == 2 || NDT <= 4) rc = a.rows <= 16 ? run_few<T, NDT, 1>(a, q, k, v, out, lse, part, st) : run_few<T, NDT, 2>(a, q, k, v, out, lse, part, st);
    else rc = run_few<T, NDT, 1>(a, q, k, v, out, lse, part, st);
  }
  else if (p.nsplit > 1) rc = p.rt == 2 ? run_fwd<T, NDT, 2, true>(a, q, k, v, out, lse, part, st) : run_fwd<T, NDT, 1, true>(a, q, k, v, out, lse, part, st);
  else rc = p.rt == 2 ? run_fwd<T, NDT, 2, false>(a, q, k, v, out, lse, part, st) : run_fwd<T, NDT, 1, false>(a, q, k, v, out, lse, part, st);
  if (rc || p.nsplit == 1) return rc;
  hipLaunchKernelGGL((win_join_kernel<T>), dim3((unsigned)((long)a.B * a.Hkv * a.rows)), dim3(256), 0, st, a, part, (T*)out, lse);
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename T, int NDT, int RT>
int run_dq(const WinArgs& a, const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, float* delta, void* dq, hipStream_t st) {
  const size_t smem = 2 * key_bufs<T, false>() * WT<T, NDT>::TILE;
  if (int rc = set_lds(win_dq_kernel<T, NDT, RT>, smem)) return rc;
  hipLaunchKernelGGL((win_dq_kernel<T, NDT, RT>), dim3((a.rows + 64 * RT - 1) / (64 * RT), a.Hkv, a.B), dim3(256), smem, st, a, (const T*)q, (const T*)k, (const T*)v,
                     (const T*)out, (const T*)dout, lse, delta, (T*)dq);
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename T, int NDT, int KT>
int run_dkv(const WinArgs& a, const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* delta, void* dk, void* dv, float* part,
            hipStream_t st) {
  const size_t smem = 2 * (2 * WT<T, NDT>::TILE + 128 * 4);
  if (int rc = set_lds(win_dkv_kernel<T, NDT, KT>, smem)) return rc;
  const int nkb = (a.Tk + 64 * KT - 1) / (64 * KT) - a.nsink;
  const long wgs = (long)a.B * a.Hkv * (nkb + a.nsink * a.nsplit);
  if (wgs > 0x7fffffffL) return -930;
  hipLaunchKernelGGL((win_dkv_kernel<T, NDT, KT>), dim3((unsigned)wgs), dim3(256), smem, st, a, (const T*)q, (const T*)k, (const T*)v, (const T*)dout, lse, delta, (T*)dk,
                     (T*)dv, part, nkb);
  FH_CHECK_LAUNCH();
  return 0;
}
template <typename T, int NDT>
int bwd_t(WinArgs a, const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, void* dq, void* dk, void* dv,
          char* scratch, hipStream_t st) {
  constexpr int DT = ElemTraits<T>::DT;
  float* delta = (float*)scratch;
  float* part = (float*)(scratch + al16((size_t)a.B * a.Tq * a.Hq * 4));
  if (a.rows > 0) {
    int rc;
    if constexpr (DT != 0 && NDT <= 6) {
      rc = bwd_tiles(a, DT, (long)a.B * a.Hkv * ((a.rows + 127) / 128), false) == 2 ? run_dq<T, NDT, 2>(a, q, k, v, out, dout, lse, delta, dq, st)
                                                                                     : run_dq<T, NDT, 1>(a, q, k, v, out, dout, lse, delta, dq, st);
    } else {
      rc = run_dq<T, NDT, 1>(a, q, k, v, out, dout, lse, delta, dq, st);
    }
    if (rc) return rc;
  }
  if (a.Tk > 0) {
    const int keys = dkv_keys(a, DT);
    bwd_sinks(a, keys);
    int rc;
    if constexpr (DT != 0 && NDT <= 4) {
      rc = keys == 128 ? run_dkv<T, NDT, 2>(a, q, k, v, dout, lse, delta, dk, dv, part, st) : run_dkv<T, NDT, 1>(a, q, k, v, dout, lse, delta, dk, dv, part, st);
    } else {
      rc = run_dkv<T, NDT, 1>(a, q, k, v, dout, lse, delta, dk, dv, part, st);
    }
    if (rc) return rc;
    if (a.nsink > 0) {
      const long n = (long)a.B * a.Hkv * a.nsink * 2 * keys * (a.dh / 4);
      hipLaunchKernelGGL((win_dkv_join_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, part, (T*)dk, (T*)dv, keys);
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
