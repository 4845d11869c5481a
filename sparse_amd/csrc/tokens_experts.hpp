// tokens_experts.hpp -- the experts' products on the matrix cores: a block-diagonal matrix of dense blocks W[e] times a
// panel whose rows are grouped by block (offsets[e] .. offsets[e+1] are expert e's rows, tokens_order.hpp):
//
//   kForward   ys[r, f]    = sum_d xs[r, d]  W[e][f, d]        (both operands have the summed index side by side)
//   kGradX     dxs[r, d]   = sum_f dys[r, f] W[e][f, d]        (W has it down its rows)
//   kGradW     dW[e][f, d] = sum_r dys[r, f] xs[r, d]          (both have it down their rows)
//
// One workgroup computes a BM x BN tile of one expert's result; sums are in 32 bits (v_mfma_f32_16x16x32) and rounded
// once.  A step takes 64 of the summed index: each operand's 64-deep slice goes from memory to LDS without passing
// through registers (buffer_load ... lds, 16 bytes a lane), one step ahead of the products, in two buffers with one
// barrier a step.  The buffer descriptor ends at the expert's last row, so what a ragged tile would read beyond it is
// zero and costs no memory access.
//
// LDS layouts.  "Lying" operands (summed index side by side): row r is 128 bytes, its eight 16-byte chunks permuted by
// c ^ (r & 7); a fragment is one ds_read_b128.  "Standing" operands (summed index down the rows): row k is R elements,
// its 32-byte units permuted by a function of k; a fragment is two ds_read_b64_tr_b16, which hand a lane four k of one
// column.  Both permutations spread every group of lanes that is served at once over all 64 banks.  They are applied to
// the addresses the loads read from, since a load to LDS writes its 64 lanes side by side.
#pragma once

#include "tokens_common.hpp"

namespace samd {
namespace tok {

enum { kForward = 0, kGradX = 1, kGradW = 2 };

constexpr int kDepth = 64;  // of the summed index in a step

template <class T>
struct Mfma;
template <>
struct Mfma<bf16> {
  typedef __attribute__((ext_vector_type(8))) bf16 Frag;
  typedef __attribute__((ext_vector_type(4))) float Acc;
  static __device__ __forceinline__ Acc go(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mfma<f16> {
  typedef __attribute__((ext_vector_type(8))) f16 Frag;
  typedef __attribute__((ext_vector_type(4))) float Acc;
  static __device__ __forceinline__ Acc go(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

typedef __attribute__((ext_vector_type(4))) short Short4;
typedef __attribute__((address_space(3))) Short4 LdsShort4;
typedef __attribute__((address_space(3))) void LdsVoid;

struct ProductShape {
  int64_t rows;        // rows of the panels
  int64_t M, N, K;     // kForward / kGradX: M unused (an expert's rows), N columns of the result, K summed;
                       // kGradW: M x N = a block of dW, K unused
  int64_t ldA, ldB, ldC;
  int64_t blockB;      // elements from one block of W to the next (kForward, kGradX)
  int64_t blockC;      // elements from one block of dW to the next (kGradW)
  int X;
  int m_tiles, n_tiles;  // kForward / kGradX: m_tiles = upper bound over all experts; kGradW: of one block
};

// One operand's tile: R rows of the result's index, kDepth of the summed index.
// p: element (0, 0) of the tile's first step; `rest`: elements from p to behind the operand's last one.
template <class T, int R, bool STANDING, int NT, bool FAST>
struct Tile {
  static constexpr int kLoads = R * kDepth * (int)sizeof(T) / 16 / NT;  // 16-byte chunks a thread brings per step
  static_assert(kLoads >= 1 && R * kDepth * (int)sizeof(T) / 16 % NT == 0, "a tile is a whole number of loads for every thread");

  const T *p;
  int64_t ld, rest, summed;
  int64_t width;        // how much of the result's index there is from the tile's first on
  uint32_t off[FAST ? kLoads : 1];
  Piece<T> held[FAST ? 1 : kLoads];

  // the chunk that thread t's load i puts at LDS bytes (i * NT + t) * 16: its row in memory and its first column there
  static __device__ __forceinline__ void source(int i, int t, int *row, int *col) {
    const int at = i * NT + t;
    if (STANDING) {
      constexpr int per = R / 8;
      const int k = at / per, q = at % per;
      *row = k;
      *col = (((q >> 1) ^ spread(k)) << 4) + ((q & 1) << 3);
    } else {
      const int r = at >> 3, q = at & 7;
      *row = r;
      *col = (q ^ (r & 7)) << 3;
    }
  }
  static __device__ __forceinline__ int spread(int k) { return (k & 3) | (((k >> 3) & 1) << 2); }

  __device__ __forceinline__ void init(const T *base, int64_t ld_, int64_t rest_, int64_t summed_, int64_t width_) {
    p = base; ld = ld_; rest = rest_; summed = summed_; width = width_;
    if (FAST)
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        int r, c;
        source(i, threadIdx.x, &r, &c);
        off[i] = (uint32_t)(((int64_t)r * ld + c) * (int64_t)sizeof(T));
      }
  }

  // Starts bringing the step at summed index k0 into lds (FAST), or into registers.
  __device__ __forceinline__ void bring(T *lds, int64_t k0) {
    const int64_t step = STANDING ? k0 * ld : k0;
    if (FAST) {
      int64_t bytes = (rest - step) * (int64_t)sizeof(T);
      bytes = bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes;
      const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void *)(p + step), 0, (int)bytes, 0x00020000);
      // lying: columns beyond the summed index are the next row's, and are not read
      const bool dead = !STANDING && (((int)(threadIdx.x & 7) ^ (int)((threadIdx.x >> 3) & 7)) << 3) >= summed - k0;
      char *to = (char *)lds + wave_id() * (kWave * 16);
#pragma unroll
      for (int i = 0; i < kLoads; i++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (LdsVoid *)(to + i * NT * 16), 16, (int)(dead ? 0x80000000u : off[i]), 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        int r, c;
        source(i, threadIdx.x, &r, &c);
        const int64_t left = STANDING ? (k0 + r < summed ? width - c : 0) : (r < width ? summed - k0 - c : 0);
        held[i] = load_piece(p + step + r * ld + c, left);
      }
    }
  }
  __device__ __forceinline__ void put(T *lds) {
    if (!FAST)
#pragma unroll
      for (int i = 0; i < kLoads; i++) __builtin_memcpy((char *)lds + (i * NT + (int)threadIdx.x) * 16, &held[i], 16);
  }

  // Fragment of rows r0 .. r0+15 and summed index 32 kk .. 32 kk + 31: lane l has row r0 + l % 16, eight k from 8 (l / 16) on.
  static __device__ __forceinline__ typename Mfma<T>::Frag fragment(const T *lds, int r0, int kk) {
    const int l = lane_id();
    typename Mfma<T>::Frag f;
    if (STANDING) {
      const int q = (l & 15) >> 2;
      const int u = (r0 >> 4) ^ (q | (((l >> 4) & 1) << 2));
      const T *at = lds + (kk * 32 + (l >> 4) * 8 + q) * R + u * 16 + (l & 3) * 4;
      const Short4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4 *)at);
      const Short4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4 *)(at + 4 * R));
      __builtin_memcpy(&f, &a, 8);
      __builtin_memcpy((char *)&f + 8, &b, 8);
    } else {
      const int r = r0 + (l & 15);
      const T *at = lds + r * kDepth + (((kk * 4 + (l >> 4)) ^ (r & 7)) << 3);
      f = *(const typename Mfma<T>::Frag *)at;
    }
    return f;
  }
};

__device__ __forceinline__ int64_t clamped(const int32_t *offsets, int e, int64_t rows) {
  const int64_t v = offsets[e];
  return v < 0 ? 0 : v > rows ? rows : v;
}

// The expert whose m-tile `tile` is, counted over all experts; its first row and the expert's last.  False: there is none.
__device__ __forceinline__ bool find_tile(const int32_t *offsets, int X, int64_t rows, int bm, int tile, int *e, int64_t *r0, int64_t *r1) {
  const int l = lane_id();
  int before = 0;
  for (int e0 = 0; e0 < X; e0 += kWave) {
    const int mine = e0 + l;
    int64_t a = 0, b = 0;
    if (mine < X) {
      a = clamped(offsets, mine, rows);
      b = clamped(offsets, mine + 1, rows);
    }
    const int tiles = b > a ? (int)((b - a + bm - 1) / bm) : 0;
    int s = tiles;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(s, d, kWave);
      if (l >= d) s += o;
    }
    const uint64_t past = __ballot(before + s > tile);
    if (past) {
      const int w = __ffsll((unsigned long long)past) - 1;
      const int first = before + __shfl(s - tiles, w, kWave);
      *e = __builtin_amdgcn_readfirstlane(e0 + w);
      const int64_t ea = clamped(offsets, *e, rows), eb = clamped(offsets, *e + 1, rows);
      *r0 = ea + (int64_t)__builtin_amdgcn_readfirstlane(tile - first) * bm;
      *r1 = eb;
      return true;
    }
    before += __shfl(s, kWave - 1, kWave);
  }
  return false;
}

template <class T, class TO, bool ADD>
__device__ __forceinline__ void store_four(TO *p, const typename Mfma<T>::Acc &a, int64_t left) {
  if (left >= 4) {
    TO o[4];
    if (ADD) __builtin_memcpy(o, p, sizeof o);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (TO)(ADD ? (float)o[i] + a[i] : a[i]);
    __builtin_memcpy(p, o, sizeof o);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < left) p[i] = (TO)(ADD ? (float)p[i] + a[i] : a[i]);
  }
}

// A wave computes BM/WM x BN/WN of the tile, B's fragment as the first operand: a lane then holds four neighbouring
// columns of one row of the result.
template <class T, class TO, int KIND, int BM, int BN, int WM, int WN, bool FAST, bool ADD>
__global__ __launch_bounds__(WM *WN *kWave) void experts_kernel(TO *__restrict__ C, const T *__restrict__ A, const T *__restrict__ B,
                                                                const int32_t *__restrict__ offsets, ProductShape g) {
  constexpr int NT = WM * WN * kWave;
  constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  using TA = Tile<T, BM, KIND == kGradW, NT, FAST>;
  using TB = Tile<T, BN, KIND != kForward, NT, FAST>;
  using Acc = typename Mfma<T>::Acc;
  using Frag = typename Mfma<T>::Frag;
  __shared__ __align__(128) T a0[BM * kDepth];
  __shared__ __align__(128) T b0[BN * kDepth];
  __shared__ __align__(128) T a1[BM * kDepth];
  __shared__ __align__(128) T b1[BN * kDepth];

  const int id = (int)blockIdx.x;
  int e;
  int64_t m0, n0, m_end, summed;
  TA ta;
  TB tb;
  TO *out;
  if (KIND == kGradW) {
    const int per = g.m_tiles * g.n_tiles;
    e = id / per;
    const int t = id - e * per;
    m0 = (int64_t)(t / g.n_tiles) * BM;
    n0 = (int64_t)(t % g.n_tiles) * BN;
    m_end = g.M;
    const int64_t ra = clamped(offsets, e, g.rows), rb = clamped(offsets, e + 1, g.rows);
    summed = rb > ra ? rb - ra : 0;
    if (ADD && summed == 0) return;
    ta.init(A + ra * g.ldA + m0, g.ldA, summed ? (summed - 1) * g.ldA + g.M - m0 : 0, summed, g.M - m0);
    tb.init(B + ra * g.ldB + n0, g.ldB, summed ? (summed - 1) * g.ldB + g.N - n0 : 0, summed, g.N - n0);
    out = C + (int64_t)e * g.blockC;
  } else {
    if (!find_tile(offsets, g.X, g.rows, BM, id / g.n_tiles, &e, &m0, &m_end)) return;
    n0 = (int64_t)(id % g.n_tiles) * BN;
    summed = g.K;
    ta.init(A + m0 * g.ldA, g.ldA, (m_end - m0 - 1) * g.ldA + g.K, summed, m_end - m0);
    const T *w = B + (int64_t)e * g.blockB;
    if (KIND == kForward)
      tb.init(w + n0 * g.ldB, g.ldB, (g.N - n0 - 1) * g.ldB + g.K, summed, g.N - n0);
    else
      tb.init(w + n0, g.ldB, (g.K - 1) * g.ldB + g.N - n0, summed, g.N - n0);
    out = C;
  }

  const int wm = wave_id() / WN, wn = wave_id() % WN;
  Acc acc[NI][MI] = {};
  const auto step = [&](const T *sa, const T *sb, T *na, T *nb, int64_t k0) {
    __syncthreads();  // this step's slices have arrived, and nobody reads the other buffer any more
    const bool more = k0 + kDepth < summed;
    if (more) {
      ta.bring(na, k0 + kDepth);
      tb.bring(nb, k0 + kDepth);
    }
#pragma unroll
    for (int kk = 0; kk < kDepth / 32; kk++) {
      Frag fa[MI], fb[NI];
#pragma unroll
      for (int i = 0; i < MI; i++) fa[i] = TA::fragment(sa, wm * (BM / WM) + i * 16, kk);
#pragma unroll
      for (int j = 0; j < NI; j++) fb[j] = TB::fragment(sb, wn * (BN / WN) + j * 16, kk);
#pragma unroll
      for (int j = 0; j < NI; j++)
#pragma unroll
        for (int i = 0; i < MI; i++) acc[j][i] = Mfma<T>::go(fb[j], fa[i], acc[j][i]);
    }
    if (more) {
      ta.put(na);
      tb.put(nb);
    }
  };
  if (summed > 0) {
    ta.bring(a0, 0);
    tb.bring(b0, 0);
    ta.put(a0);
    tb.put(b0);
  }
  for (int64_t k0 = 0; k0 < summed; k0 += 2 * kDepth) {
    step(a0, b0, a1, b1, k0);
    if (k0 + kDepth < summed) step(a1, b1, a0, b0, k0 + kDepth);
  }

  const int l = lane_id();
#pragma unroll
  for (int i = 0; i < MI; i++) {
    const int64_t m = m0 + wm * (BM / WM) + i * 16 + (l & 15);
    if (m >= m_end) continue;
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const int64_t n = n0 + wn * (BN / WN) + j * 16 + (l >> 4) * 4;
      if (n < g.N) store_four<T, TO, ADD>(out + m * g.ldC + n, acc[j][i], g.N - n);
    }
  }
}

}  // namespace tok
}  // namespace samd
