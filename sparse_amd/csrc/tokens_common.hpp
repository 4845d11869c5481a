// tokens_common.hpp -- what the kernels of tokens.hip share: element types, 16-byte pieces of a row, wave sums.
//
// Everything here works on rows of a dense row-major panel: `units` pieces of 16 bytes, the last one possibly short.
// Rows need no more alignment than their element: the hardware takes 128-bit global accesses at any element's address
// (a piece that crosses a cache line costs a second line), so odd widths and strides run the same kernels as round ones.
#pragma once

#include "common.hpp"
#include "scan.hpp"

namespace samd {
namespace tok {

using bf16 = __bf16;
using f16 = _Float16;

constexpr int kWave = 64;
constexpr int kThreads = kBlock;  // kWaves waves
static_assert(kThreads == kWaves * kWave, "a workgroup is a whole number of waves");

template <class T>
constexpr int kPer = 16 / (int)sizeof(T);  // elements of a 16-byte piece

template <class T>
struct Piece {
  T v[kPer<T>];
};

typedef uint32_t __attribute__((ext_vector_type(4), aligned(2), may_alias)) Quad;  // 16 bytes at any element's address
// (a copy of bytes instead is stored in parts where the compiler joins it with the elements of a tail)

// The `left` elements (kPer or fewer) of a piece at p; what is not there reads as zero.  ONCE: nobody will read them again
// soon, so they are not kept in the caches in the place of what will be (a non-temporal load).
template <bool ONCE = false, class T>
__device__ __forceinline__ Piece<T> load_piece(const T *p, int64_t left) {
  Piece<T> r = {};
  if (left >= kPer<T>) {
    if (ONCE) {
      const Quad q = __builtin_nontemporal_load((const Quad *)p);
      __builtin_memcpy(&r, &q, 16);
    } else {
      __builtin_memcpy(&r, p, 16);
    }
  } else if (left > 0) {
#pragma unroll
    for (int i = 0; i < kPer<T> - 1; i++)
      if (i < left) r.v[i] = p[i];
  }
  return r;
}

template <bool STREAM = false, class T>
__device__ __forceinline__ void store_piece(T *p, const Piece<T> &r, int64_t left) {
  if (left >= kPer<T>) {
    Quad q;
    __builtin_memcpy(&q, &r, 16);
    if (STREAM) __builtin_nontemporal_store(q, (Quad *)p);
    else *(Quad *)p = q;
  } else if (left > 0) {
#pragma unroll
    for (int i = 0; i < kPer<T> - 1; i++)
      if (i < left) p[i] = r.v[i];
  }
}

// A result larger than the L2s of the card (8 x 4 MiB) is written past them (non-temporal stores): its lines would push out
// what is being read.  A smaller one is left to the caches, where the next kernel finds it.  16384 rows of 8 KiB looked up:
// 43 -> 40 us; 32 blocks of dW, 512 MiB: 127 -> 101 us.
constexpr int64_t kStreamBytes = (int64_t)32 << 20;

// kPer<T> sums held in 32 bits, rounded once to TO (16 or 32 bits) and stored; ADD: added to what is there first.
template <class T, class TO, bool ADD, bool STREAM>
__device__ __forceinline__ void store_sums(TO *p, const float (&s)[kPer<T>], int64_t left) {
  if (left >= kPer<T>) {
    constexpr int n = kPer<T> / kPer<TO>;  // pieces of the result: one, or two of 32 bits from 16
    Piece<TO> o[n];
    if (ADD) __builtin_memcpy(o, p, sizeof o);
#pragma unroll
    for (int i = 0; i < kPer<T>; i++) {
      TO &x = o[i / kPer<TO>].v[i % kPer<TO>];
      x = (TO)(ADD ? (float)x + s[i] : s[i]);
    }
#pragma unroll
    for (int i = 0; i < n; i++) store_piece<STREAM>(p + i * kPer<TO>, o[i], kPer<TO>);
  } else if (left > 0) {
#pragma unroll
    for (int i = 0; i < kPer<T> - 1; i++)
      if (i < left) p[i] = (TO)(ADD ? (float)p[i] + s[i] : s[i]);
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
  return v;
}

__device__ __forceinline__ int lane_id() { return (int)(threadIdx.x & (kWave - 1)); }
// The same in every lane of a wave, and known to be: what is indexed by it is loaded once per wave.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave)); }

// A grid holds fewer than 2^32 threads along x.  A launch of more workgroups has several rows of kGridRow of them (of up to 1024
// threads), the last row whole as well: a kernel returns for a number behind its last one.
constexpr int kGridRowLog = 21;
constexpr int64_t kGridRow = (int64_t)1 << kGridRowLog;

inline dim3 grid_of(int64_t blocks, int threads) {
  if (blocks * threads < (int64_t)1 << 32) return dim3((unsigned)blocks);
  return dim3((unsigned)kGridRow, (unsigned)cdiv(blocks, kGridRow));
}

__device__ __forceinline__ int64_t block_number() { return ((int64_t)blockIdx.y << kGridRowLog) + blockIdx.x; }

// Among the waves of a launch of kThreads threads a workgroup.
__device__ __forceinline__ int64_t wave_number() { return block_number() * kWaves + wave_id(); }

// How a launch deals rows to waves.  Rows of 64 pieces or more: a wave takes `u` x 64 pieces of one row, `segs` waves a
// row.  Shorter rows: a power of two of lanes each (1 << lg), so that a wave takes several.
struct RowDeal {
  int lg;
  int64_t segs;
  int64_t waves;
};

inline RowDeal deal_rows(int64_t rows, int64_t units, int u) {
  RowDeal d;
  d.lg = 0;
  while (d.lg < 6 && ((int64_t)1 << d.lg) < units) d.lg++;
  d.segs = d.lg == 6 ? cdiv(units, (int64_t)kWave * u) : 1;
  d.waves = cdiv(rows, (int64_t)(kWave >> d.lg)) * d.segs;
  return d;
}

struct RowPlace {
  int64_t row, unit;  // this lane's row, and its first piece in it
};

// of the w-th wave of such a launch
__device__ __forceinline__ RowPlace my_row(int64_t w, int lg, int64_t segs, int u) {
  const int lane = lane_id();
  RowPlace r;
  if (lg == 6) {
    r.row = w / segs;
    r.unit = (w - r.row * segs) * (kWave * u) + lane;
  } else {
    r.row = w * (kWave >> lg) + (lane >> lg);
    r.unit = lane & ((1 << lg) - 1);
  }
  return r;
}

}  // namespace tok
}  // namespace samd
