// tokens_experts.hpp -- the experts' products on the matrix cores: a block-diagonal matrix of dense blocks W[e] times a
// panel whose rows are grouped by block (offsets[e] .. offsets[e+1] are expert e's rows, tokens_order.hpp):
//
//   kForward   ys[r, f]    = sum_d xs[r, d]  W[e][f, d]        (both operands have the summed index side by side)
//   kGradX     dxs[r, d]   = sum_f dys[r, f] W[e][f, d]        (W has it down its rows)
//   kGradW     dW[e][f, d] = sum_r dys[r, f] xs[r, d]          (both have it down their rows)
//
// One workgroup computes a BM x BN tile of one expert's result; sums are in 32 bits (v_mfma_f32_16x16x32) and rounded
// once.  A step takes 32, 64 or 128 of the summed index: each operand's slice of it goes from memory to LDS without passing
// through registers (buffer_load ... lds, 16 bytes a lane), some steps ahead of the products.  The buffer descriptor ends
// with the expert's last row (its last chunk of 16 bytes), so what a ragged tile would read beyond it is zero and costs no
// memory access.
//
// What bounds it: with few rows an expert the blocks' bytes (32 blocks of 4096 x 2048, 2 rows each: 75 us, 7.2 TB/s), with many the
// matrix cores and what they wait for at a tile's ends: 8 blocks of 4096 x 4096, 2048 rows each, 1380 to 1400 TFLOP/s forward,
// 1360 by xs, 1347 by W; 16 of 4096 x 2048, 1024 rows each, whose tiles have half the steps or fewer, 1220 to 1250, 1250 and
// 1156.  A library product of as many operations reaches 1520 to 1590.
//
// Forward, the order in which a row's products are added depends on the workgroup that its tile falls to: a row's last bits
// may change with the other rows of the batch, though not from call to call.
//
// LDS layouts.  "Lying" operands (summed index side by side): row r is a step's slice, its 16-byte chunks permuted by a
// function of r; a fragment is one ds_read_b128.  "Standing" operands (summed index down the rows): row k is R elements,
// its 32-byte units permuted by a function of k; a fragment is two ds_read_b64_tr_b16, which hand a lane four k of one
// column.  Both permutations spread every group of lanes that is served at once over all 64 banks.  They are applied to
// the addresses the loads read from, since a load to LDS writes its 64 lanes side by side.
#pragma once

#include "tokens_common.hpp"

#include <type_traits>

namespace samd {
namespace tok {

enum { kForward = 0, kGradX = 1, kGradW = 2 };

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
  int split;           // CUs the last round of tiles is spread over, or 1: it is left as it is
  bool stream;         // the result is written past the caches
  int m_tiles, n_tiles;  // kForward / kGradX: m_tiles = upper bound over all experts; kGradW: of one block
};

// A value that every lane has, known to be the same: what is computed from it stays in scalar registers (a descriptor that
// might differ between lanes would be loaded through lane by lane).
__device__ __forceinline__ int64_t same(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// One operand's tile: R rows of the result's index, DEPTH (32, 64 or 128) of the summed index.
// p: element (0, 0) of the tile's first step; `rest`: elements from p to behind the operand's last one.
template <class T, int R, int DEPTH, bool STANDING, int NT, bool FAST>
struct Tile {
  static constexpr int kLoads = R * DEPTH * (int)sizeof(T) / 16 / NT;  // 16-byte chunks a thread brings per step
  static_assert(kLoads >= 1 && R * DEPTH * (int)sizeof(T) / 16 % NT == 0, "a tile is a whole number of loads for every thread");

  const T *p;
  int64_t ld, rest, summed;  // FAST: rest in whole chunks
  int64_t width;        // how much of the result's index there is from the tile's first on
  int steps, first, now;  // FAST, lying: how many steps there are, which is taken first (then in turn), steps moved on
  uint32_t off[FAST ? kLoads : 1];
  __amdgpu_buffer_rsrc_t bounds;
  Piece<T> held[2][FAST ? 1 : kLoads];  // not FAST: two steps on their way to LDS

  // the chunk that thread t's load i puts at LDS bytes (i * NT + t) * 16: its row in memory and its first column there
  static __device__ __forceinline__ void source(int i, int t, int *row, int *col) {
    const int at = i * NT + t;
    if (STANDING) {
      constexpr int per = R / 8;
      const int k = at / per, q = at % per;
      *row = k;
      *col = (((q >> 1) ^ (spread(k) & (R / 16 - 1))) << 4) + ((q & 1) << 3);
    } else {
      constexpr int per = DEPTH / 8;
      const int r = at / per, q = at % per;
      *row = r;
      *col = (q ^ twist(r)) << 3;
    }
  }
  // ds_read_b128 serves 16 lanes at a time, over 64 banks: lanes 0-3, 12-15 and 20-27, then 4-11, 16-19 and 28-31, and the
  // same of the upper half.  Either set has to find its rows' chunks in 16 different places.
  static __device__ __forceinline__ int twist(int r) { return DEPTH == 128 ? r & 15 : DEPTH == 64 ? (r >> 1) & 7 : (4 - (r >> 2)) & 3; }
  static __device__ __forceinline__ int spread(int k) { return (k & 3) | (((k >> 3) & 1) << 2); }

  __device__ __forceinline__ void init(const T *base, int64_t ld_, int64_t rest_, int64_t summed_, int64_t width_, int first_) {
    p = (const T *)same(reinterpret_cast<int64_t>(base)); ld = ld_; rest = same(rest_); summed = summed_; width = width_;
    if (FAST) {
      // The descriptor ends with a whole chunk: of one that it ended in, the four bytes that hold its end would read as zero, and
      // a width that is odd would lose its last element.  Chunks begin on 16 bytes, so none reaches into memory that is not
      // there, and what lies behind the width is of columns that are not written.
      rest = (rest + 7) & ~(int64_t)7;
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        int r, c;
        source(i, threadIdx.x, &r, &c);
        off[i] = (uint32_t)(((int64_t)r * ld + c) * (int64_t)sizeof(T));
      }
      steps = (int)((summed + DEPTH - 1) / DEPTH);
      first = steps > 0 ? first_ / DEPTH % steps : 0;
      now = 0;
      bound();
    }
  }

  __device__ __forceinline__ void bound() {
    const int64_t bytes = rest * (int64_t)sizeof(T);
    bounds = __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)(bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes), 0x00020000);
  }

  // FAST: steps are counted from here on `by` further.  Standing: the descriptor moves along, so that offsets stay small
  // whatever the operand's size.
  __device__ __forceinline__ void move(int by) {
    now += by;
    if (!STANDING) return;
    p += by * DEPTH * ld;
    rest -= by * DEPTH * ld;
    bound();
  }

  // FAST: starts the loads of step `step` into lds.  ONCE: past the caches' order of use (non-temporal).
  template <bool ONCE = false>
  __device__ __forceinline__ void start(T *lds, int step) {
    int row, col;
    source(0, threadIdx.x, &row, &col);  // the same columns in every load of a thread: NT / (DEPTH / 8) rows on, twist() repeats
    bool dead = false;
    int at;
    if (STANDING) {
      at = (int)(step * DEPTH * ld * (int64_t)sizeof(T));
    } else {  // columns beyond the summed index are the next row's, and are not read
      int t = now + step;
      const bool over = t >= steps;
      t += first;
      if (t >= steps) t -= steps;
      dead = over || col >= (int)summed - t * DEPTH;
      at = t * DEPTH * (int)sizeof(T);
    }
    char *to = (char *)lds + wave_id() * (kWave * 16);
#pragma unroll
    for (int i = 0; i < kLoads; i++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(bounds, (LdsVoid *)(to + i * NT * 16), 16, (int)(dead ? 0x80000000u : off[i]), at, 0, ONCE ? 2 : 0);
  }

  // Not FAST: the step at summed index k0 into registers, and from there into lds.
  template <int SET>
  __device__ __forceinline__ void bring(int64_t k0) {
    const int64_t step = STANDING ? k0 * ld : k0;
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      int r, c;
      source(i, threadIdx.x, &r, &c);
      const int64_t left = STANDING ? (k0 + r < summed ? width - c : 0) : (r < width ? summed - k0 - c : 0);
      held[SET][FAST ? 0 : i] = load_piece(p + step + r * ld + c, left);
    }
  }
  template <int SET>
  __device__ __forceinline__ void put(T *lds) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) __builtin_memcpy((char *)lds + (i * NT + (int)threadIdx.x) * 16, &held[SET][FAST ? 0 : i], 16);
  }

  // Fragment of rows r0 .. r0+15 and summed index 32 kk .. 32 kk + 31: lane l has row r0 + l % 16, eight k from 8 (l / 16) on.
  static __device__ __forceinline__ typename Mfma<T>::Frag fragment(const T *lds, int r0, int kk) {
    const int l = lane_id();
    typename Mfma<T>::Frag f;
    if (STANDING) {
      const int q = (l & 15) >> 2;
      const int u = (r0 >> 4) ^ ((q | (((l >> 4) & 1) << 2)) & (R / 16 - 1));
      const T *at = lds + (kk * 32 + (l >> 4) * 8 + q) * R + u * 16 + (l & 3) * 4;
      const Short4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4 *)at);
      const Short4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4 *)(at + 4 * R));
      __builtin_memcpy(&f, &a, 8);
      __builtin_memcpy((char *)&f + 8, &b, 8);
    } else {
      const int r = r0 + (l & 15);
      const T *at = lds + r * DEPTH + (((kk * 4 + (l >> 4)) ^ twist(r)) << 3);
      f = *(const typename Mfma<T>::Frag *)at;
    }
    return f;
  }
};

__device__ __forceinline__ int64_t clamped(const int32_t *offsets, int e, int64_t rows) {
  const int64_t v = offsets[e];
  return v < 0 ? 0 : v > rows ? rows : v;
}

constexpr int kXcds = 8;  // workgroup i runs on die i % 8, each with an L2 of its own

// Tile `id` of m x n: every die has a run of neighbouring tiles, taken down columns of kDown tiles, so that the 32 tiles a
// die works on at a time share 8 tiles of one operand and 4 of the other out of its L2.
constexpr int kDown = 8;
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int *m, int *n) {
  const int group = t / (kDown * n_tiles), in = t - group * (kDown * n_tiles);
  const int high = min(kDown, m_tiles - group * kDown);
  *n = in / high;
  *m = group * kDown + in - *n * high;
}

// The place of workgroup `id` among `tiles`: every die has a run of them.  Negative: it has none.
__device__ __forceinline__ int place_of(int id, int tiles) {
  const int per = (tiles + kXcds - 1) / kXcds;
  const int t = id % kXcds * per + id / kXcds;
  return id / kXcds < per && t < tiles ? t : -1;
}

// The experts' m-tiles, 64 experts at a time: lane l has those of expert e0 + l, counted up to and with it.
struct TileCounts {
  int32_t a, b;   // the expert's rows
  int upto;
  __device__ __forceinline__ TileCounts(const int32_t *offsets, int e0, int X, int64_t rows, int bm) {
    const int e = e0 + lane_id();
    a = b = 0;
    if (e < X) {
      a = (int32_t)clamped(offsets, e, rows);
      b = (int32_t)clamped(offsets, e + 1, rows);
    }
    upto = (int)wave_inclusive_add_dpp(b > a ? (uint32_t)(b - a + bm - 1) / (uint32_t)bm : 0u);
  }
  __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(upto, kWave - 1); }
  // The expert (of these 64) whose tile the `tile`-th of these is; its first row in the tile, and the expert's last.
  __device__ __forceinline__ int find(int tile, int bm, int64_t *r0, int64_t *r1) const {
    const int w = __builtin_ctzll(__ballot(upto > tile));
    const int before = w > 0 ? __builtin_amdgcn_readlane(upto, w - 1) : 0;
    *r0 = __builtin_amdgcn_readlane(a, w) + (int64_t)(tile - before) * bm;
    *r1 = __builtin_amdgcn_readlane(b, w);
    return w;
  }
};

template <class T, class TO, bool ADD>
__device__ __forceinline__ void store_four(TO *p, const typename Mfma<T>::Acc &a, int64_t left) {
  typedef uint32_t __attribute__((ext_vector_type(sizeof(TO)), aligned(2), may_alias)) Four;
  if (left >= 4) {
    TO o[4];
    if (ADD) __builtin_memcpy(o, p, sizeof o);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (TO)(ADD ? (float)o[i] + a[i] : a[i]);
    Four q;
    __builtin_memcpy(&q, o, sizeof o);
    *(Four *)p = q;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < left) p[i] = (TO)(ADD ? (float)p[i] + a[i] : a[i]);
  }
}

// All but the last N loads of this wave have arrived and its LDS reads are done; then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void arrived() {
  static_assert(N < 64, "the counter has six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The operands of a tile whose rows begin at m0 and columns at n0 of expert e's result, which ends with row m_end.
template <int KIND, class T, class TA>
__device__ __forceinline__ void operand_a(TA &ta, int e, int64_t m0, int64_t m_end, int64_t summed, int first, const T *A, const int32_t *offsets, const ProductShape &g) {
  if (KIND == kGradW)
    ta.init(A + clamped(offsets, e, g.rows) * g.ldA + m0, g.ldA, summed ? (summed - 1) * g.ldA + g.M - m0 : 0, summed, g.M - m0, 0);
  else
    ta.init(A + m0 * g.ldA, g.ldA, (m_end - m0 - 1) * g.ldA + g.K, g.K, m_end - m0, first);
}
template <int KIND, class T, class TB>
__device__ __forceinline__ void operand_b(TB &tb, int e, int64_t n0, int64_t summed, int first, const T *B, const int32_t *offsets, const ProductShape &g) {
  if (KIND == kGradW)
    tb.init(B + clamped(offsets, e, g.rows) * g.ldB + n0, g.ldB, summed ? (summed - 1) * g.ldB + g.N - n0 : 0, summed, g.N - n0, 0);
  else if (KIND == kForward)
    tb.init(B + (int64_t)e * g.blockB + n0 * g.ldB, g.ldB, (g.N - n0 - 1) * g.ldB + g.K, g.K, g.N - n0, first);
  else
    tb.init(B + (int64_t)e * g.blockB + n0, g.ldB, (g.K - 1) * g.ldB + g.N - n0, g.K, g.N - n0, 0);
}
// Where a tile's sums begin (they go round to what lies before).  Rows of W that are a power of two apart would all be read
// at the same column at the same time, which meets in few of the memory's channels: so every die, and every expert on it,
// begins elsewhere; the tiles that share rows in an L2 stay together.  32 blocks of 4096 x 2048, 16 rows each: 97 -> 83 us;
// of 2048 x 4096, 94 -> 86; 96 rows each in tiles of 256 x 256: 133 -> 110; nothing where rows are 1.4 or 5 times a power of
// two apart, or W is in a cache.  (A beginning for every column of tiles: 32 x 64 as much, 128 x 128 up to 10 % slower.)
template <int KIND>
__device__ __forceinline__ int first_column(int e) { return KIND == kForward ? ((int)blockIdx.x % kXcds + e) * 768 : 0; }
// How long its sums are, and where its result goes.
template <int KIND>
__device__ __forceinline__ int64_t sum_length(int e, const int32_t *offsets, const ProductShape &g) {
  if (KIND != kGradW) return g.K;
  const int64_t ra = clamped(offsets, e, g.rows), rb = clamped(offsets, e + 1, g.rows);
  return same(rb > ra ? rb - ra : 0);
}
template <int KIND, class TO>
__device__ __forceinline__ TO *result_of(TO *C, int e, const ProductShape &g) { return KIND == kGradW ? C + (int64_t)e * g.blockC : C; }

// Where the workgroup's tile is.  False: it has none.
//
// A last round of a few tiles of 256 x 256 would leave most CUs idle for as long as any other: if it fills half of them or
// fewer (g.split: the launch has workgroups enough) each of its tiles is cut into its upper and its lower rows; *half =
// which, or -1.  (73 tiles after 256, forward: 262 us whole, 252 in halves, 272 in quarters; in the gradient by xs 301, 286,
// 308.)
template <int KIND, int BM, int BN>
__device__ __forceinline__ bool place_product(int *e, int64_t *m0, int64_t *n0, int64_t *m_end, int *half, const int32_t *offsets,
                                              const ProductShape &g) {
  const int id = (int)blockIdx.x;
  int m, n;
  *half = -1;
  if (KIND == kGradW) {
    // block after block of dW, each dealt to all dies: the blocks' costs differ with their experts' rows
    const int per = (g.m_tiles * g.n_tiles + kXcds - 1) / kXcds * kXcds;
    *e = id / per;
    const int t = place_of(id - *e * per, g.m_tiles * g.n_tiles);
    if (t < 0) return false;
    tile_at(t, g.m_tiles, g.n_tiles, &m, &n);
    *m0 = (int64_t)m * BM;
    *n0 = (int64_t)n * BN;
    *m_end = g.M;
    return true;
  }
  const TileCounts first(offsets, 0, g.X, g.rows, BM);  // all there are, as a rule
  int m_tiles = first.all();
  for (int e0 = kWave; e0 < g.X; e0 += kWave) m_tiles += TileCounts(offsets, e0, g.X, g.rows, BM).all();
  const int tiles = m_tiles * g.n_tiles;
  const int rest = tiles % g.split, whole = g.split > 1 && 2 * rest <= g.split ? tiles - rest : tiles;
  const int own = (whole + kXcds - 1) / kXcds * kXcds;  // workgroups of the whole tiles
  int t;
  if (id < own) {
    t = place_of(id, whole);
    if (t < 0) return false;
  } else {
    const int q = id - own;  // the halves of a tile go to one die
    t = whole + q / (2 * kXcds) * kXcds + q % kXcds;
    *half = q / kXcds % 2;
    if (t >= tiles) return false;
  }
  tile_at(t, m_tiles, g.n_tiles, &m, &n);
  if (m < first.all()) {
    *e = first.find(m, BM, m0, m_end);
  } else {
    m -= first.all();
    for (int e0 = kWave; e0 < g.X; e0 += kWave) {
      const TileCounts more(offsets, e0, g.X, g.rows, BM);
      if (m < more.all()) {
        *e = e0 + more.find(m, BM, m0, m_end);
        break;
      }
      m -= more.all();
    }
  }
  *n0 = (int64_t)n * BN;
  if (*half == 1) *m0 += BM / 2;
  return *m0 < *m_end;
}

// Sums in 32 bits, or added to what is there: every lane writes the four neighbouring columns that it holds.
template <class T, class TO, bool ADD, int BM, int BN, int WM, int WN, class Acc, int NI, int MI>
__device__ __forceinline__ void store_product(TO *out, const Acc (&acc)[NI][MI], int64_t m0, int64_t n0, int64_t m_end, const ProductShape &g) {
  const int l = lane_id(), wm = wave_id() / WN, wn = wave_id() % WN;
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

// Rounded to 16 bits: through `mine`, LDS that only this wave uses, so that a row leaves the wave in pieces of 16 bytes that
// lie side by side (a wave's 64 columns are a cache line; written four columns a lane, dW of 32 blocks of 4096 x 2048 for few
// rows, in four stages, took 214 us where this took 150).  The pieces of a row are permuted by the row's number: the lanes that write the same
// columns of 16 rows would all meet in a few banks.
template <class T, int BM, int BN, int WM, int WN, class Acc, int NI, int MI>
__device__ __forceinline__ void store_rounded(T *mine, T *out, const Acc (&acc)[NI][MI], int64_t m0, int64_t n0, int64_t m_end, const ProductShape &g) {
  constexpr int TM = BM / WM, TN = BN / WN, per = TN / 8;  // pieces in a row of the wave's tile
  const int l = lane_id();
  m0 += wave_id() / WN * TM;
  n0 += wave_id() % WN * TN;
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const int r = i * 16 + (l & 15), c = j * 2 + (l >> 5);
      T v[4];
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = (T)acc[j][i][k];
      __builtin_memcpy((char *)mine + (r * per + (c ^ (r & (per - 1)))) * 16 + ((l >> 4) & 1) * 8, v, 8);
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int q = 0; q < TM * per / kWave; q++) {
    const int at = q * kWave + l, r = at / per, c = at % per;
    Piece<T> v;
    __builtin_memcpy(&v, (const char *)mine + (r * per + (c ^ (r & (per - 1)))) * 16, 16);
    const int64_t m = m0 + r, n = n0 + c * 8;
    if (m < m_end) {
      if (g.stream) store_piece<true>(out + m * g.ldC + n, v, g.N - n);
      else store_piece<false>(out + m * g.ldC + n, v, g.N - n);
    }
  }
}

// Any strides and alignment: a step's chunks are loaded into registers two steps before its products, and put into one of
// two LDS buffers one step before.
// A wave computes BM/WM x BN/WN of the tile, B's fragment as the first operand: a lane then holds four neighbouring
// columns of one row of the result.
template <class T, class TO, int KIND, int BM, int BN, int DEPTH, int WM, int WN, bool ADD>
__global__ __launch_bounds__(WM *WN *kWave) void experts_any_kernel(TO *__restrict__ C, const T *__restrict__ A, const T *__restrict__ B,
                                                                    const int32_t *__restrict__ offsets, ProductShape g) {
  constexpr int NT = WM * WN * kWave;
  constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  using TA = Tile<T, BM, DEPTH, KIND == kGradW, NT, false>;
  using TB = Tile<T, BN, DEPTH, KIND != kForward, NT, false>;
  using Acc = typename Mfma<T>::Acc;
  using Frag = typename Mfma<T>::Frag;
  __shared__ __align__(128) T sa[2][BM * DEPTH];
  __shared__ __align__(128) T sb[2][BN * DEPTH];
  TA ta;
  TB tb;
  int e, half;
  int64_t m0, n0, m_end;
  if (!place_product<KIND, BM, BN>(&e, &m0, &n0, &m_end, &half, offsets, g)) return;
  const int64_t summed = sum_length<KIND>(e, offsets, g);
  if (ADD && summed == 0) return;
  operand_a<KIND>(ta, e, m0, m_end, summed, 0, A, offsets, g);
  operand_b<KIND>(tb, e, n0, summed, 0, B, offsets, g);
  TO *const out = result_of<KIND>(C, e, g);
  const int wm = wave_id() / WN, wn = wave_id() % WN;
  Acc acc[NI][MI] = {};
  // the products of the step in buffer SET; the next step goes from registers into the other one
  const auto step = [&](auto set, int64_t k0) {
    constexpr int SET = decltype(set)::value;
    __syncthreads();  // this step's slices are there, and nobody reads the other buffer any more
    ta.template put<SET ^ 1>(sa[SET ^ 1]);
    tb.template put<SET ^ 1>(sb[SET ^ 1]);
    ta.template bring<SET ^ 1>(k0 + 3 * DEPTH);  // nothing is read behind the end
    tb.template bring<SET ^ 1>(k0 + 3 * DEPTH);
#pragma unroll
    for (int kk = 0; kk < DEPTH / 32; kk++) {
      Frag fa[MI], fb[NI];
#pragma unroll
      for (int i = 0; i < MI; i++) fa[i] = TA::fragment(sa[SET], wm * (BM / WM) + i * 16, kk);
#pragma unroll
      for (int j = 0; j < NI; j++) fb[j] = TB::fragment(sb[SET], wn * (BN / WN) + j * 16, kk);
#pragma unroll
      for (int j = 0; j < NI; j++)
#pragma unroll
        for (int i = 0; i < MI; i++) acc[j][i] = Mfma<T>::go(fb[j], fa[i], acc[j][i]);
    }
  };
  if (summed > 0) {
    ta.template bring<0>(0);
    tb.template bring<0>(0);
    ta.template bring<1>(DEPTH);
    tb.template bring<1>(DEPTH);
    ta.template put<0>(sa[0]);
    tb.template put<0>(sb[0]);
    ta.template bring<0>(2 * DEPTH);
    tb.template bring<0>(2 * DEPTH);
    for (int64_t k0 = 0; k0 < summed; k0 += 2 * DEPTH) {  // a step behind the last multiplies zeros
      step(std::integral_constant<int, 0>(), k0);
      step(std::integral_constant<int, 1>(), k0 + DEPTH);
    }
  }
  if constexpr (std::is_same<T, TO>::value && !ADD) {
    static_assert(BM / WM * (BN / WN) * WM * WN <= 2 * BM * DEPTH, "every wave's part of the tile fits into A's two buffers");
    __syncthreads();
    store_rounded<T, BM, BN, WM, WN>(&sa[0][0] + wave_id() * (BM / WM * (BN / WN)), out, acc, m0, n0, m_end, g);
  } else {
    store_product<T, TO, ADD, BM, BN, WM, WN>(out, acc, m0, n0, m_end, g);
  }
}

// Rows that begin on 16 bytes: loads go to LDS by themselves, some steps ahead of the products.  Loads behind the end of the
// summed index are started like any others, read nothing and write zeros, so that the number of loads in flight, which a
// wait for the older ones counts (vmcnt counts down in order), is always the same.
//
// ONCE: B is read past the caches, for weights that no cache could hold anyway.

// Four waves, two or three workgroups on a CU.  Four stages of LDS, each DEPTH of the summed index: a stage's loads are
// started three steps before its products.  A step: read this stage's fragments, start the loads of the stage three on,
// wait for the fragments and for the wave's own loads of the next stage, barrier, products.  Behind the barrier every
// wave's loads of the next stage are there, and the stage before this one may be overwritten.
template <class T, class TO, int KIND, int BM, int BN, int DEPTH, int WM, int WN, bool ADD, bool ONCE>
__device__ __forceinline__ void multiply_small(int e, int64_t m0, int64_t n0, int64_t m_end, TO *C, const T *A, const T *B,
                                               const int32_t *offsets, const ProductShape &g) {
  constexpr int NT = WM * WN * kWave, S = 4, KK = DEPTH / 32;
  constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  using TA = Tile<T, BM, DEPTH, KIND == kGradW, NT, true>;
  using TB = Tile<T, BN, DEPTH, KIND != kForward, NT, true>;
  using Acc = typename Mfma<T>::Acc;
  using Frag = typename Mfma<T>::Frag;
  constexpr int L = TA::kLoads + TB::kLoads;
  // an array for each stage: what is read from one does not wait for loads into another
  __shared__ __align__(128) T a0[BM * DEPTH], a1[BM * DEPTH], a2[BM * DEPTH], a3[BM * DEPTH];
  __shared__ __align__(128) T b0[BN * DEPTH], b1[BN * DEPTH], b2[BN * DEPTH], b3[BN * DEPTH];
  TA ta;
  TB tb;
  const int64_t summed = sum_length<KIND>(e, offsets, g);
  if (ADD && summed == 0) return;
  const int first = first_column<KIND>(e);
  operand_a<KIND>(ta, e, m0, m_end, summed, first, A, offsets, g);
  operand_b<KIND>(tb, e, n0, summed, first, B, offsets, g);
  TO *const out = result_of<KIND>(C, e, g);
  const int wm = wave_id() / WN, wn = wave_id() % WN;
  Acc acc[NI][MI] = {};
  // the products of stage t, which is in sa, sb; na, nb take the stage three on
  const auto step = [&](const T *sa, const T *sb, T *na, T *nb, int t) {
    Frag fa[KK][MI], fb[KK][NI];
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
#pragma unroll
      for (int j = 0; j < NI; j++) fb[kk][j] = TB::fragment(sb, wn * (BN / WN) + j * 16, kk);
#pragma unroll
      for (int i = 0; i < MI; i++) fa[kk][i] = TA::fragment(sa, wm * (BM / WM) + i * 16, kk);
    }
    __builtin_amdgcn_sched_barrier(0);
    ta.start(na, t + S - 1);
    tb.template start<ONCE>(nb, t + S - 1);
    __builtin_amdgcn_sched_barrier(0);
    arrived<(S - 2) * L>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
      for (int j = 0; j < NI; j++)
#pragma unroll
        for (int i = 0; i < MI; i++) acc[j][i] = Mfma<T>::go(fb[kk][j], fa[kk][i], acc[j][i]);
  };
  if (summed > 0) {
    ta.start(a0, 0);
    tb.template start<ONCE>(b0, 0);
    ta.start(a1, 1);
    tb.template start<ONCE>(b1, 1);
    ta.start(a2, 2);
    tb.template start<ONCE>(b2, 2);
    arrived<(S - 2) * L>();
    for (int64_t k0 = 0; k0 < summed; k0 += S * DEPTH) {  // steps behind the last multiply zeros
      step(a0, b0, a3, b3, 0);
      step(a1, b1, a0, b0, 1);
      step(a2, b2, a1, b1, 2);
      step(a3, b3, a2, b2, 3);
      ta.move(S);
      tb.move(S);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may still write to LDS when the workgroup has ended
  }
  if constexpr (std::is_same<T, TO>::value && !ADD) {
    constexpr int part = BM / WM * (BN / WN);  // each wave has a stage's array to itself, one that its part of the tile fits into
    constexpr bool in_a = part <= BM * DEPTH;
    static_assert(WM * WN == 4 && part <= BN * DEPTH, "a wave's part of the tile fits into a stage's array");
    __syncthreads();
    T *const as[4] = {a0, a1, a2, a3}, *const bs[4] = {b0, b1, b2, b3};
    const int w = wave_id();
    T *mine = in_a ? as[0] : bs[0];
#pragma unroll
    for (int k = 1; k < 4; k++)
      if (w == k) mine = in_a ? as[k] : bs[k];
    store_rounded<T, BM, BN, WM, WN>(mine, out, acc, m0, n0, m_end, g);
  } else {
    store_product<T, TO, ADD, BM, BN, WM, WN>(out, acc, m0, n0, m_end, g);
  }
}

// dW of experts with few rows: nearly all of it is writing, so a workgroup keeps little (32 KiB of LDS, one slice of the rows
// at a time; 128 registers) and four of them on a CU overlap.  32 blocks of 4096 x 2048, 16 rows each: 90 us, 6.0 TB/s, where
// three workgroups take 102, and four stages and two workgroups 142; 128 rows: 136, 157 and 169; 256 rows: as long as tiles of
// 256 x 256.  Slices of 64: 16 rows 125; tiles of 64 x 256 and 64 x 128 3 and 10 % more.
template <class T, class TO, int BM, int BN, int DEPTH, int WM, int WN, bool ADD>
__global__ __launch_bounds__(WM *WN *kWave, 4) void experts_few_kernel(TO *__restrict__ C, const T *__restrict__ A, const T *__restrict__ B,
                                                                    const int32_t *__restrict__ offsets, ProductShape g) {
  constexpr int NT = WM * WN * kWave, KK = DEPTH / 32;
  constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  using TA = Tile<T, BM, DEPTH, true, NT, true>;
  using TB = Tile<T, BN, DEPTH, true, NT, true>;
  using Acc = typename Mfma<T>::Acc;
  using Frag = typename Mfma<T>::Frag;
  constexpr bool rounded = std::is_same<T, TO>::value && !ADD;
  __shared__ __align__(128) T lds[rounded ? BM * BN : (BM + BN) * DEPTH];
  static_assert((BM + BN) * DEPTH <= BM * BN, "the slices fit where the result goes later");
  T *const a = lds, *const b = lds + BM * DEPTH;
  int e, half;
  int64_t m0, n0, m_end;
  if (!place_product<kGradW, BM, BN>(&e, &m0, &n0, &m_end, &half, offsets, g)) return;
  const int64_t summed = sum_length<kGradW>(e, offsets, g);
  if (ADD && summed == 0) return;
  TA ta;
  TB tb;
  operand_a<kGradW>(ta, e, m0, m_end, summed, 0, A, offsets, g);
  operand_b<kGradW>(tb, e, n0, summed, 0, B, offsets, g);
  TO *const out = result_of<kGradW>(C, e, g);
  const int wm = wave_id() / WN, wn = wave_id() % WN;
  Acc acc[NI][MI] = {};
  for (int64_t k0 = 0; k0 < summed; k0 += DEPTH) {
    ta.start(a, 0);
    tb.start(b, 0);
    arrived<0>();
    Frag fa[KK][MI], fb[KK][NI];
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
#pragma unroll
      for (int j = 0; j < NI; j++) fb[kk][j] = TB::fragment(b, wn * (BN / WN) + j * 16, kk);
#pragma unroll
      for (int i = 0; i < MI; i++) fa[kk][i] = TA::fragment(a, wm * (BM / WM) + i * 16, kk);
    }
    ta.move(1);
    tb.move(1);
    __syncthreads();  // everybody has read
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
      for (int j = 0; j < NI; j++)
#pragma unroll
        for (int i = 0; i < MI; i++) acc[j][i] = Mfma<T>::go(fb[kk][j], fa[kk][i], acc[j][i]);
  }
  if constexpr (rounded)
    store_rounded<T, BM, BN, WM, WN>(lds + wave_id() * (BM / WM * (BN / WN)), out, acc, m0, n0, m_end, g);
  else
    store_product<T, TO, ADD, BM, BN, WM, WN>(out, acc, m0, n0, m_end, g);
}

// Eight waves, two on each SIMD, one workgroup on a CU.  LDS holds two steps of 64 of the summed index, so that a row gives
// whole cache lines; each has three parts that are loaded and given up by themselves: the upper rows, the lower rows, and
// all columns.  A step is two phases: read the columns' and the upper rows' fragments, multiply; read the lower rows'
// fragments, multiply.  What a phase has read is overwritten one phase later, with the same part two steps on (the lower
// rows: a step on, being younger), so every load has two phases of time.
//
// Waves 4 to 7 run one barrier behind waves 0 to 3, and every phase has one barrier before its products and one behind:
// while one wave of a SIMD feeds the matrix cores the other reads LDS and starts loads, and they change places.  A part is
// then read up to half a phase later by the second four, still before the barrier behind which it is overwritten, and
// waits count the loads that a barrier later all waves may need.
//
// Four stages of 32, as above but in turns, take 64 bytes of a lying operand's row at a time: 16 experts of 4096 x 2048,
// 1024 rows each, forward: 7 % slower than steps of 64 where both were timed in turn; the other two products are as fast either way.
template <class T>
struct Parts {  // [of the even and the odd steps]; an array each: what is read from one does not wait for loads into another
  T *up0, *up1, *low0, *low1, *col0, *col1;
};

template <class T, class TO, int KIND, int BM, int BN, bool ADD>
__device__ __forceinline__ void multiply_large(const Parts<T> lds, int e, int64_t m0, int64_t n0, int64_t m_end, TO *C, const T *A, const T *B,
                                               const int32_t *offsets, const ProductShape &g) {
  constexpr int WM = 2, WN = 4, NT = WM * WN * kWave, DEPTH = 64, KK = 2, HM = BM / 2;
  constexpr int MI = HM / WM / 16, NI = BN / WN / 16;
  using TA = Tile<T, HM, DEPTH, KIND == kGradW, NT, true>;
  using TB = Tile<T, BN, DEPTH, KIND != kForward, NT, true>;
  using Acc = typename Mfma<T>::Acc;
  using Frag = typename Mfma<T>::Frag;
  constexpr int kYounger = TB::kLoads + 2 * TA::kLoads;  // loads started since those that a phase waits for
  TA up, low;
  TB col;
  const int64_t summed = sum_length<KIND>(e, offsets, g);
  if (ADD && summed == 0) return;
  const int first = first_column<KIND>(e);
  operand_a<KIND>(up, e, m0, m_end, summed, first, A, offsets, g);
  operand_a<KIND>(low, e, m0 + HM, m_end, summed, first, A, offsets, g);
  operand_b<KIND>(col, e, n0, summed, first, B, offsets, g);
  TO *const out = result_of<KIND>(C, e, g);
  const int wm = wave_id() / WN, wn = wave_id() % WN;
  Acc acc[2][NI][MI] = {};
  Frag fb[KK][NI];
  const auto multiply = [&](const Frag(&fa)[KK][MI], Acc(&sum)[NI][MI]) {
    __builtin_amdgcn_sched_barrier(0);
    arrived<kYounger>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
      for (int j = 0; j < NI; j++)
#pragma unroll
        for (int i = 0; i < MI; i++) sum[j][i] = Mfma<T>::go(fb[kk][j], fa[kk][i], sum[j][i]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  // step t (0 or 1, counted from where the tiles were moved to), whose parts are u, l, c; other: where the lower rows of
  // the next step go
  const auto step = [&](T *u, const T *l, T *c, T *other, int t) {
    Frag fa[KK][MI];
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
#pragma unroll
      for (int j = 0; j < NI; j++) fb[kk][j] = TB::fragment(c, wn * (BN / WN) + j * 16, kk);
#pragma unroll
      for (int i = 0; i < MI; i++) fa[kk][i] = TA::fragment(u, wm * (HM / WM) + i * 16, kk);
    }
    __builtin_amdgcn_sched_barrier(0);
    low.start(other, t + 1);
    multiply(fa, acc[0]);
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
      for (int i = 0; i < MI; i++) fa[kk][i] = TA::fragment(l, wm * (HM / WM) + i * 16, kk);
    __builtin_amdgcn_sched_barrier(0);
    col.start(c, t + 2);
    up.start(u, t + 2);
    multiply(fa, acc[1]);
  };
  if (summed > 0) {
    col.start(lds.col0, 0);
    up.start(lds.up0, 0);
    low.start(lds.low0, 0);
    col.start(lds.col1, 1);
    up.start(lds.up1, 1);
    arrived<kYounger>();
    const bool second = wave_id() >= 4;
    if (second) __builtin_amdgcn_s_barrier();
    for (int64_t k0 = 0; k0 < summed; k0 += 2 * DEPTH) {  // a step behind the last multiplies zeros
      step(lds.up0, lds.low0, lds.col0, lds.low1, 0);
      step(lds.up1, lds.low1, lds.col1, lds.low0, 1);
      up.move(2);
      low.move(2);
      col.move(2);
    }
    if (!second) __builtin_amdgcn_s_barrier();        // as many barriers as the others
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may still write to LDS when the workgroup has ended
  }
  if constexpr (std::is_same<T, TO>::value && !ADD) {
    constexpr int part = HM / WM * (BN / WN);
    static_assert(2 * part <= HM * DEPTH, "two waves' parts of half the tile fit into an array of rows");
    __syncthreads();
    T *const rows[4] = {lds.up0, lds.up1, lds.low0, lds.low1};
    const int w = wave_id();
    T *mine = rows[0];
#pragma unroll
    for (int k = 1; k < 4; k++)
      if (w >> 1 == k) mine = rows[k];
    mine += (w & 1) * part;
    store_rounded<T, HM, BN, WM, WN>(mine, out, acc[0], m0, n0, m_end, g);
    __builtin_amdgcn_wave_barrier();
    store_rounded<T, HM, BN, WM, WN>(mine, out, acc[1], m0 + HM, n0, m_end, g);
  } else {
    store_product<T, TO, ADD, HM, BN, WM, WN>(out, acc[0], m0, n0, m_end, g);
    store_product<T, TO, ADD, HM, BN, WM, WN>(out, acc[1], m0 + HM, n0, m_end, g);
  }
}

template <class T, class TO, int KIND, int BM, int BN, int DEPTH, int WM, int WN, bool ADD, bool ONCE>
__global__ __launch_bounds__(WM *WN *kWave) void experts_kernel(TO *__restrict__ C, const T *__restrict__ A, const T *__restrict__ B,
                                                                const int32_t *__restrict__ offsets, ProductShape g) {
  int e, half;
  int64_t m0, n0, m_end;
  if (!place_product<KIND, BM, BN>(&e, &m0, &n0, &m_end, &half, offsets, g)) return;
  if constexpr (WM * WN == 4) {
    multiply_small<T, TO, KIND, BM, BN, DEPTH, WM, WN, ADD, ONCE>(e, m0, n0, m_end, C, A, B, offsets, g);
  } else {
    static_assert(WM == 2 && WN == 4 && DEPTH == 64 && !ONCE, "as multiply_large has it");
    __shared__ __align__(128) T up0[BM / 2 * DEPTH], up1[BM / 2 * DEPTH], low0[BM / 2 * DEPTH], low1[BM / 2 * DEPTH];
    __shared__ __align__(128) T col0[BN * DEPTH], col1[BN * DEPTH];
    const Parts<T> lds = {up0, up1, low0, low1, col0, col1};
    if constexpr (KIND != kGradW && BM == 256 && BN == 256) {
      if (half >= 0) {
        multiply_large<T, TO, KIND, BM / 2, BN, ADD>(lds, e, m0, n0, m_end, C, A, B, offsets, g);
        return;
      }
    }
    multiply_large<T, TO, KIND, BM, BN, ADD>(lds, e, m0, n0, m_end, C, A, B, offsets, g);
  }
}

}  // namespace tok
}  // namespace samd
