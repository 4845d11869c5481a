// tokens_lookup_grad.hpp -- dE[v] = sum over i with id[i] = v of s f[i] dy[i]: the transposed record of a lookup times dy.
//
// The ids are ordered first (tokens_order.hpp), so that the rows of one v lie side by side in the order of the batch.  The
// ordered positions are cut into chunks of equal length, whatever runs they hold: a wave takes one chunk and 64 pieces of
// the row, loads eight rows of dy at a time and adds them in 32 bits, and writes a run when it ends.  A run that crosses
// chunk ends leaves a 32-bit sum for each chunk (head: the run came from an earlier chunk; tail: it began here), and a
// second launch adds those in order and writes the row.  So a vocabulary's commonest token costs as much as any others,
// no sum depends on timing, and dy is read once.  Rows without an id are zeroed by the waves of the first launch that
// have no chunk: a stream of writes beside a stream of reads.  Bound by the bytes of dy and dE where the table is large (16384
// rows into 131072 of 2048 bf16: 102 us, 5.9 TB/s); a small table by few waves and by launches in a row (32768 rows, 30 % of
// them padding, into 8192 of 1024 f16: 42 us, of which the order takes 16, the sums 19 at 3.2 TB/s, the join 6).
#pragma once

#include "tokens_order.hpp"

namespace samd {
namespace tok {

struct GradShape {
  int64_t n, V, D;
  int64_t ldy, ldE;
  int64_t segs;      // waves along a row of dy, 64 pieces each
  int64_t chunks;
  RowDeal fill;      // of the rows that are zeroed; no waves when sums are added to what is there
  int chunk;         // positions in a chunk: a multiple of 8
};

// Zeros are fastest from many short waves in the order of memory: 2 pieces of a row a lane; 16384 rows into 131072 of 2048 bf16
// 102 us, 4 pieces 117, 1 piece 150.
constexpr int kFillPieces = 2;

// Sum of a chunk's part of a run, as two rows of 32-bit sums per chunk: [chunk][head, tail][segs * 64 * kPer].
template <class T>
__device__ __forceinline__ float *chunk_sum(float *part, const GradShape &g, int64_t chunk, int tail, int64_t unit) {
  return part + ((chunk * 2 + tail) * g.segs * kWave + unit) * kPer<T>;
}

template <class T, class TO, bool ADD, bool STREAM>
__global__ __launch_bounds__(kThreads) void lookup_grad_kernel(TO *__restrict__ dE, const T *__restrict__ dy,
                                                               const float *__restrict__ vals, float scale,
                                                               const uint32_t *__restrict__ keys, const int32_t *__restrict__ items,
                                                               const uint8_t *__restrict__ named, float *__restrict__ part,
                                                               GradShape g) {
  constexpr int R = 8;
  const int64_t w = wave_number();
  const int lane = lane_id();
  const int64_t chunk = w / g.segs;
  if (chunk >= g.chunks) {  // zero the rows no id names (named: a byte for each row)
    if (ADD) return;
    const RowPlace at = my_row(w - g.chunks * g.segs, g.fill.lg, g.fill.segs, kFillPieces);
    if (at.row >= g.V || named[at.row]) return;
    const Piece<TO> z = {};
#pragma unroll
    for (int u = 0; u < kFillPieces; u++) {
      const int64_t c = (at.unit + u * kWave) * kPer<TO>;
      if (c < g.D) store_piece<STREAM>(dE + at.row * g.ldE + c, z, g.D - c);
    }
    return;
  }
  const int64_t unit = (w - chunk * g.segs) * kWave + lane;
  const int64_t c = unit * kPer<T>;
  const int64_t p0 = chunk * g.chunk, p1 = p0 + g.chunk < g.n ? p0 + g.chunk : g.n;
  const uint32_t none = (uint32_t)g.V;
  uint32_t run = keys[p0];
  bool from_before = p0 > 0 && keys[p0 - 1] == run;
  float s[kPer<T>] = {};
  for (int64_t p = p0; p < p1 && run != none; p += R) {
    uint32_t k[R];
    float f[R];
    Piece<T> x[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      k[r] = p + r < p1 ? keys[p + r] : none;
      const int64_t i = k[r] != none ? items[p + r] : 0;
      f[r] = vals ? scale * vals[i] : scale;
      x[r] = load_piece<!STREAM>(dy + i * g.ldy + c, k[r] != none ? g.D - c : 0);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (k[r] != run) {
        if (p + r >= p1) break;
        if (c < g.D) {
          if (from_before) {
            float *to = chunk_sum<T>(part, g, chunk, 0, unit);
#pragma unroll
            for (int i = 0; i < kPer<T>; i++) to[i] = s[i];
          } else {
            store_sums<T, TO, ADD, STREAM>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
          }
        }
        run = k[r];
        from_before = false;
#pragma unroll
        for (int i = 0; i < kPer<T>; i++) s[i] = 0.0f;
        if (run == none) break;
      }
#pragma unroll
      for (int i = 0; i < kPer<T>; i++) s[i] += f[r] * (float)x[r].v[i];
    }
  }
  if (run == none || c >= g.D) return;
  const bool goes_on = p1 < g.n && keys[p1] == run;
  if (from_before || goes_on) {
    float *to = chunk_sum<T>(part, g, chunk, from_before ? 0 : 1, unit);
#pragma unroll
    for (int i = 0; i < kPer<T>; i++) to[i] = s[i];
  } else {
    store_sums<T, TO, ADD, STREAM>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
  }
}

// One workgroup for each chunk and 64 pieces: returns at once unless a run begins in the chunk and goes on behind it.
// Its waves add a part of the run's chunk sums each, and the parts are added in order.
template <class T, class TO, bool ADD, bool STREAM>
__global__ __launch_bounds__(kThreads) void lookup_grad_join_kernel(TO *__restrict__ dE, const uint32_t *__restrict__ keys,
                                                                    float *__restrict__ part, GradShape g) {
  __shared__ float sums[kWaves][kWave][kPer<T>];
  const int64_t chunk = block_number() / g.segs;
  const int64_t p0 = chunk * g.chunk, p1 = p0 + g.chunk;
  if (p1 >= g.n) return;
  const uint32_t run = keys[p1 - 1];
  if (run == (uint32_t)g.V || keys[p1] != run || (p0 > 0 && keys[p0 - 1] == run)) return;
  // chunk sums of the run: this chunk's tail, then the heads of the chunks that begin with it (64 chunks looked at at once)
  int64_t count = 1;
  for (;;) {
    const int64_t q = (chunk + count + lane_id()) * g.chunk;
    const uint64_t other = ~__ballot(q < g.n && keys[q] == run);
    if (other) {
      count += __builtin_ctzll(other);
      break;
    }
    count += kWave;
  }
  const int64_t each = (count + kWaves - 1) / kWaves;
  const int64_t k0 = wave_id() * each, k1 = k0 + each < count ? k0 + each : count;
  const int64_t unit = (block_number() - chunk * g.segs) * kWave + lane_id();
  const int64_t c = unit * kPer<T>;
  float s[kPer<T>] = {};
  if (c < g.D) {
#pragma unroll 8
    for (int64_t k = k0; k < k1; k++) {
      const float *from = chunk_sum<T>(part, g, chunk + k, k == 0 ? 1 : 0, unit);
#pragma unroll
      for (int i = 0; i < kPer<T>; i++) s[i] += from[i];
    }
  }
#pragma unroll
  for (int i = 0; i < kPer<T>; i++) sums[wave_id()][lane_id()][i] = s[i];
  __syncthreads();
  if (wave_id() != 0 || c >= g.D) return;
  for (int v = 1; v < kWaves; v++)
#pragma unroll
    for (int i = 0; i < kPer<T>; i++) s[i] += sums[v][lane_id()][i];
  store_sums<T, TO, ADD, STREAM>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
}

// ------------------------------------------------------------------------------------------------ few ids
// Up to 256 ids in one launch, without a workspace.  The first `segs` workgroups take 64 pieces of the rows each: every
// one of them orders the ids for itself (an id's place is how many are smaller, its place in the batch being the low byte
// of what is compared; four threads share the counting for one id), its 16 waves sum a chunk each, and the runs that cross
// chunks are joined through LDS.  The other workgroups zero those of their rows that no id names.  The same sums in the
// same order every time.  For tables of fewer than 2^24 rows; beyond that the ordered path takes over.
// What every lane of a wave has read, as the scalar that it is: a wave then branches instead of masking its lanes.
__device__ __forceinline__ uint32_t one(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

constexpr int kFewIds = 256;
constexpr int64_t kFewTable = ((int64_t)1 << 24) - 1;
constexpr int kFewWaves = 16;
constexpr int kFewFillRows = 2048;

template <class T, class TO, class I, bool ADD, bool STREAM>
__global__ __launch_bounds__(kFewWaves *kWave) void lookup_grad_few_kernel(TO *__restrict__ dE, const T *__restrict__ dy,
                                                                           const I *__restrict__ ids, const float *__restrict__ vals,
                                                                           float scale, GradShape g, int fill_rows) {
  __shared__ __align__(16) uint32_t key[kFewIds];
  __shared__ uint32_t okey[kFewIds];
  __shared__ int oitem[kFewIds];
  __shared__ float part[kFewWaves][2][kWave][kPer<T>];
  const int n = (int)g.n, t = (int)threadIdx.x, lane = lane_id(), w = wave_id();
  const uint32_t none = (uint32_t)g.V;

  if ((int64_t)blockIdx.x >= g.segs) {
    if (ADD) return;
    uint8_t *named = (uint8_t *)&part[0][0][0][0];
    const int64_t first = ((int64_t)blockIdx.x - g.segs) * fill_rows;
    for (int r = t; r < fill_rows; r += kFewWaves * kWave) named[r] = 0;
    __syncthreads();
    if (t < n) {
      const int64_t v = (int64_t)ids[t];
      if (v >= first && v < g.V && v - first < fill_rows) named[v - first] = 1;
    }
    __syncthreads();
    const int lanes = 1 << g.fill.lg, each = kWave >> g.fill.lg;
    const Piece<TO> z = {};
    for (int r0 = w * each; r0 < fill_rows; r0 += kFewWaves * each) {
      const int r = r0 + lane / lanes;
      if (r >= fill_rows || first + r >= g.V || named[r]) continue;
      TO *row = dE + (first + r) * g.ldE;
      for (int64_t c = (int64_t)(lane & (lanes - 1)) * kPer<TO>; c < g.D; c += (int64_t)lanes * kPer<TO>) store_piece<STREAM>(row + c, z, g.D - c);
    }
    return;
  }

  if (t < kFewIds) {
    const int64_t v = t < n ? (int64_t)ids[t] : -1;
    key[t] = (v >= 0 && v < g.V ? (uint32_t)v : none) << 8 | (uint32_t)t;
  }
  __syncthreads();
  {
    const uint32_t mine = key[t >> 2];
    const int quarter = (n + 15) / 16 * 4;  // whole reads of four; what lies behind the n-th is larger than all before it
    int before = 0;
    for (int u = (t & 3) * quarter; u < ((t & 3) + 1) * quarter; u += 4) {
      const uint4 k = *(const uint4 *)&key[u];
      before += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
    }
    before += __shfl_xor(before, 1, kWave);
    before += __shfl_xor(before, 2, kWave);
    if ((t & 3) == 0 && (t >> 2) < n) {
      okey[before] = mine >> 8;
      oitem[before] = (int)(mine & 255);
    }
  }
  __syncthreads();

  const int64_t c = ((int64_t)blockIdx.x * kWave + lane) * kPer<T>;
  const int chunk = (n + kFewWaves - 1) / kFewWaves;
  const int p0 = w * chunk, p1 = p0 + chunk < n ? p0 + chunk : n;
  if (p0 < p1) {
    constexpr int R = 8;
    uint32_t run = one(okey[p0]);
    bool from_before = p0 > 0 && one(okey[p0 - 1]) == run;
    float s[kPer<T>] = {};
    for (int p = p0; p < p1 && run != none; p += R) {
      uint32_t k[R];
      float f[R];
      Piece<T> x[R];
#pragma unroll
      for (int r = 0; r < R; r++) {
        k[r] = p + r < p1 ? one(okey[p + r]) : none;
        const int i = k[r] != none ? (int)one(oitem[p + r]) : 0;
        f[r] = vals ? scale * vals[i] : scale;
        x[r] = load_piece(dy + (int64_t)i * g.ldy + c, k[r] != none ? g.D - c : 0);
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        if (k[r] != run) {
          if (p + r >= p1) break;
          if (from_before) {
#pragma unroll
            for (int i = 0; i < kPer<T>; i++) part[w][0][lane][i] = s[i];
          } else if (c < g.D) {
            store_sums<T, TO, ADD, STREAM>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
          }
          run = k[r];
          from_before = false;
#pragma unroll
          for (int i = 0; i < kPer<T>; i++) s[i] = 0.0f;
          if (run == none) break;
        }
#pragma unroll
        for (int i = 0; i < kPer<T>; i++) s[i] += f[r] * (float)x[r].v[i];
      }
    }
    if (run != none) {
      const bool goes_on = p1 < n && one(okey[p1]) == run;
      if (from_before || goes_on) {
#pragma unroll
        for (int i = 0; i < kPer<T>; i++) part[w][from_before ? 0 : 1][lane][i] = s[i];
      } else if (c < g.D) {
        store_sums<T, TO, ADD, STREAM>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
      }
    }
  }
  __syncthreads();
  if (p0 >= p1 || p1 >= n) return;
  const uint32_t run = one(okey[p1 - 1]);
  if (run == none || one(okey[p1]) != run || (p0 > 0 && one(okey[p0 - 1]) == run)) return;
  float s[kPer<T>];
#pragma unroll
  for (int i = 0; i < kPer<T>; i++) s[i] = part[w][1][lane][i];
  for (int v = w + 1; v * chunk < n && one(okey[v * chunk]) == run; v++)
#pragma unroll
    for (int i = 0; i < kPer<T>; i++) s[i] += part[v][0][lane][i];
  if (c < g.D) store_sums<T, TO, ADD, STREAM>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
}

}  // namespace tok
}  // namespace samd
