// tokens_lookup_grad.hpp -- dE[v] = sum over i with id[i] = v of s f[i] dy[i]: the transposed record of a lookup times dy.
//
// The ids are ordered first (tokens_order.hpp), so that the rows of one v lie side by side in the order of the batch.  The
// ordered positions are cut into chunks of equal length, whatever runs they hold: a wave takes one chunk and 64 pieces of
// the row, loads eight rows of dy at a time and adds them in 32 bits, and writes a run when it ends.  A run that crosses
// chunk ends leaves a 32-bit sum for each chunk (head: the run came from an earlier chunk; tail: it began here), and a
// second launch adds those in order and writes the row.  So a vocabulary's commonest token costs as much as any others,
// no sum depends on timing, and dy is read once.  Rows without an id are zeroed by the waves of the first launch that
// have no chunk: a stream of writes beside a stream of reads.  Bound by the bytes of dy and dE.
#pragma once

#include "tokens_order.hpp"

namespace samd {
namespace tok {

struct GradShape {
  int64_t n, V, D;
  int64_t ldy, ldE;
  int64_t segs;       // waves along a row of dy, 64 pieces each
  int64_t chunks;
  int64_t fill_segs;  // waves along a row of dE that is zeroed; 0: none are
  int chunk;          // positions in a chunk: a multiple of 8
};

constexpr int kFillPieces = 4;

// Sum of a chunk's part of a run, as two rows of 32-bit sums per chunk: [chunk][head, tail][segs * 64 * kPer].
template <class T>
__device__ __forceinline__ float *chunk_sum(float *part, const GradShape &g, int64_t chunk, int tail, int64_t unit) {
  return part + ((chunk * 2 + tail) * g.segs * kWave + unit) * kPer<T>;
}

template <class T, class TO, bool ADD>
__global__ __launch_bounds__(kThreads) void lookup_grad_kernel(TO *__restrict__ dE, const T *__restrict__ dy,
                                                               const float *__restrict__ vals, float scale,
                                                               const uint32_t *__restrict__ keys, const int32_t *__restrict__ items,
                                                               const uint32_t *__restrict__ marks, float *__restrict__ part,
                                                               GradShape g) {
  constexpr int R = 8;
  const int64_t w = (int64_t)blockIdx.x * kWaves + wave_id();
  const int lane = lane_id();
  const int64_t chunk = w / g.segs;
  if (chunk >= g.chunks) {  // zero the rows no id names
    if (ADD || g.fill_segs == 0) return;
    const int64_t f = w - g.chunks * g.segs, row = f / g.fill_segs;
    if (row >= g.V || (marks && ((marks[row >> 5] >> (row & 31)) & 1))) return;
    Piece<TO> z = {};
#pragma unroll
    for (int u = 0; u < kFillPieces; u++) {
      const int64_t c = (((f - row * g.fill_segs) * kFillPieces + u) * kWave + lane) * kPer<TO>;
      if (c < g.D) store_piece(dE + row * g.ldE + c, z, g.D - c);
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
      x[r] = load_piece(dy + i * g.ldy + c, k[r] != none ? g.D - c : 0);
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
            store_sums<T, TO, ADD>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
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
    store_sums<T, TO, ADD>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
  }
}

// One workgroup for each chunk and 64 pieces: returns at once unless a run begins in the chunk and goes on behind it.
// Its waves add a part of the run's chunk sums each, and the parts are added in order.
template <class T, class TO, bool ADD>
__global__ __launch_bounds__(kThreads) void lookup_grad_join_kernel(TO *__restrict__ dE, const uint32_t *__restrict__ keys,
                                                                    float *__restrict__ part, GradShape g) {
  __shared__ float sums[kWaves][kWave][kPer<T>];
  const int64_t chunk = blockIdx.x / g.segs;
  const int64_t p0 = chunk * g.chunk, p1 = p0 + g.chunk;
  if (p1 >= g.n) return;
  const uint32_t run = keys[p1 - 1];
  if (run == (uint32_t)g.V || keys[p1] != run || (p0 > 0 && keys[p0 - 1] == run)) return;
  int64_t lo = p1, hi = g.n;  // the end of the run: first position behind p1 with a larger key
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] <= run) lo = mid + 1; else hi = mid;
  }
  const int64_t count = (lo - 1) / g.chunk - chunk + 1;  // chunk sums of the run: this chunk's tail, then heads
  const int64_t each = (count + kWaves - 1) / kWaves;
  const int64_t k0 = wave_id() * each, k1 = k0 + each < count ? k0 + each : count;
  const int64_t unit = (blockIdx.x - chunk * g.segs) * kWave + lane_id();
  const int64_t c = unit * kPer<T>;
  float s[kPer<T>] = {};
  if (c < g.D) {
#pragma unroll 4
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
  store_sums<T, TO, ADD>(dE + (int64_t)run * g.ldE + c, s, g.D - c);
}

}  // namespace tok
}  // namespace samd
