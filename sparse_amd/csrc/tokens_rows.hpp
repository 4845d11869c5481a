// tokens_rows.hpp -- products with a record of one or a few entries per row, row by row of the dense panel:
//
//   lookup        y[i]  = s f[i] E[id[i]]                 one entry per row (S/mono.fut:95: col_idx[n], vals[n]) times a panel
//   lookup_dots   df[i] = s <dy[i], E[id[i]]>             its gradient by the values
//   dispatch      xs[pos[t,j]] = (w[t,j]) x[t]            rows into the order of their experts
//   combine       y[t]  = sum_j (w[t,j]) ys[pos[t,j]]     and back; the transpose of dispatch with the same places and weights
//   combine_grad  dys[pos[t,j]] = w[t,j] dy[t],  dw[t,j] = <dy[t], ys[pos[t,j]]>
//
// All of them are bound by the bytes of the rows (16384 tokens of 2048 bf16 to 8 places each: 604 MB, dispatch 121 us,
// combine 106 us; with ordinary loads and stores instead of streaming ones 172 and 160 us): every row is read once (dispatch reads a token's row once for all its
// places, combine_grad reads dy once for both of its results), nothing is held in memory between, sums are in 32 bits and
// are rounded once, in an order that depends on the record alone.
#pragma once

#include "tokens_common.hpp"

namespace samd {
namespace tok {

// ids outside 0 .. V-1 select nothing: a row of zeros (padding).
// One wave takes U x 64 pieces of a row: U independent 16-byte loads in flight for each lane, behind one id.
template <class T, class I, int U, bool STREAM>
__global__ __launch_bounds__(kThreads) void lookup_kernel(T *__restrict__ y, int64_t ldy, const T *__restrict__ E, int64_t ldE,
                                                          int64_t V, int64_t D, const I *__restrict__ ids, int64_t n,
                                                          const float *__restrict__ vals, float scale, int lg, int64_t segs) {
  const RowPlace at = my_row(wave_number(), lg, segs, U);
  if (at.row >= n) return;
  const int64_t id = (int64_t)ids[at.row];
  const bool any = id >= 0 && id < V;
  const float f = vals ? scale * vals[at.row] : scale;
  const bool copy = !vals && scale == 1.0f;
  const T *src = E + (any ? id : 0) * ldE;
  T *dst = y + at.row * ldy;
  Piece<T> p[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int64_t c = (at.unit + u * kWave) * kPer<T>;
    p[u] = load_piece(src + c, any ? D - c : 0);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int64_t c = (at.unit + u * kWave) * kPer<T>;
    if (c >= D) continue;
    if (!copy && any)
#pragma unroll
      for (int i = 0; i < kPer<T>; i++) p[u].v[i] = (T)(f * (float)p[u].v[i]);
    store_piece<STREAM>(dst + c, p[u], D - c);
  }
}

// One wave per row of dy.
template <class T, class I>
__global__ __launch_bounds__(kThreads) void lookup_dots_kernel(float *__restrict__ df, const T *__restrict__ dy, int64_t ldy,
                                                               const T *__restrict__ E, int64_t ldE, int64_t V, int64_t D,
                                                               const I *__restrict__ ids, int64_t n, float scale) {
  const int64_t row = wave_number();
  if (row >= n) return;
  const int64_t id = (int64_t)ids[row];
  float s = 0.0f;
  if (id >= 0 && id < V)
    for (int64_t c = (int64_t)lane_id() * kPer<T>; c < D; c += kWave * kPer<T>) {
      const Piece<T> a = load_piece(dy + row * ldy + c, D - c), b = load_piece(E + id * ldE + c, D - c);
#pragma unroll
      for (int i = 0; i < kPer<T>; i++) s += (float)a.v[i] * (float)b.v[i];
    }
  s = wave_sum(s);
  if (lane_id() == 0) df[row] = scale * s;
}

// pos < 0: the token has no such place.  A place is given to one (t, j) only, so no two waves write one row.
template <class T, int U, bool STREAM>
__global__ __launch_bounds__(kThreads) void dispatch_kernel(T *__restrict__ xs, int64_t ldxs, const T *__restrict__ x, int64_t ldx,
                                                            int64_t n, int64_t D, int K, const int32_t *__restrict__ pos,
                                                            int64_t slots, const float *__restrict__ w, int lg, int64_t segs) {
  const RowPlace at = my_row(wave_number(), lg, segs, U);
  if (at.row >= n) return;
  const T *src = x + at.row * ldx;
  Piece<T> p[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int64_t c = (at.unit + u * kWave) * kPer<T>;
    p[u] = load_piece<true>(src + c, D - c);
  }
  for (int j = 0; j < K; j++) {
    const int64_t to = pos[at.row * K + j];
    if (to < 0 || to >= slots) continue;
    const float f = w ? w[at.row * K + j] : 1.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t c = (at.unit + u * kWave) * kPer<T>;
      if (c >= D) continue;
      Piece<T> q = p[u];
      if (w)
#pragma unroll
        for (int i = 0; i < kPer<T>; i++) q.v[i] = (T)(f * (float)q.v[i]);
      store_piece<STREAM>(xs + to * ldxs + c, q, D - c);
    }
  }
}

// The places of four choices at once: their rows are loaded before the first is added.
template <class T, int U, bool STREAM>
__global__ __launch_bounds__(kThreads) void combine_kernel(T *__restrict__ y, int64_t ldy, const T *__restrict__ ys, int64_t ldys,
                                                           int64_t n, int64_t D, int K, const int32_t *__restrict__ pos,
                                                           int64_t slots, const float *__restrict__ w, int lg, int64_t segs) {
  constexpr int J = 4;
  const RowPlace at = my_row(wave_number(), lg, segs, U);
  if (at.row >= n) return;
  float s[U][kPer<T>] = {};
  for (int j0 = 0; j0 < K; j0 += J) {
    int64_t from[J];
    float f[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
      const bool in = j0 + j < K;
      from[j] = in ? pos[at.row * K + j0 + j] : -1;
      if (from[j] >= slots) from[j] = -1;
      f[j] = w && in ? w[at.row * K + j0 + j] : 1.0f;
    }
    Piece<T> p[J][U];
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t c = (at.unit + u * kWave) * kPer<T>;
        p[j][u] = load_piece<true>(ys + (from[j] < 0 ? 0 : from[j]) * ldys + c, from[j] < 0 ? 0 : D - c);
      }
#pragma unroll
    for (int j = 0; j < J; j++)
      if (from[j] >= 0)  // a place that is not there adds nothing, whatever its weight
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int i = 0; i < kPer<T>; i++) s[u][i] += f[j] * (float)p[j][u].v[i];
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int64_t c = (at.unit + u * kWave) * kPer<T>;
    if (c < D) store_sums<T, T, false, STREAM>(y + at.row * ldy + c, s[u], D - c);
  }
}

// W waves per token, side by side along its row; J choices at once share one reading of dy.  The dot products are summed
// lane, wave, token: the same order every time.
template <class T, int W, int J, bool STREAM>
__global__ __launch_bounds__(kThreads) void combine_grad_kernel(T *__restrict__ dys, int64_t lddys, float *__restrict__ dw,
                                                                const T *__restrict__ dy, int64_t lddy, const T *__restrict__ ys,
                                                                int64_t ldys, int64_t n, int64_t D, int K, const int32_t *__restrict__ pos,
                                                                int64_t slots, const float *__restrict__ w) {
  static_assert(W == 1 || W == kWaves, "a token has a wave or a workgroup");
  __shared__ float part[kWaves][J];
  const int64_t t = W == 1 ? wave_number() : block_number();
  if (t >= n) return;
  const int first = W == 1 ? lane_id() : (int)threadIdx.x;
  for (int j0 = 0; j0 < K; j0 += J) {
    int64_t at[J];
    float f[J], dot[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
      const bool in = j0 + j < K;
      at[j] = in ? pos[t * K + j0 + j] : -1;
      if (at[j] >= slots) at[j] = -1;
      f[j] = in ? w[t * K + j0 + j] : 0.0f;
      dot[j] = 0.0f;
    }
    for (int64_t c = (int64_t)first * kPer<T>; c < D; c += W * kWave * kPer<T>) {
      const Piece<T> g = load_piece<true>(dy + t * lddy + c, D - c);
      Piece<T> p[J];
#pragma unroll
      for (int j = 0; j < J; j++)
        if (at[j] >= 0) p[j] = load_piece<true>(ys + at[j] * ldys + c, D - c);
#pragma unroll
      for (int j = 0; j < J; j++) {
        if (at[j] < 0) continue;
        Piece<T> q;
#pragma unroll
        for (int i = 0; i < kPer<T>; i++) {
          dot[j] += (float)g.v[i] * (float)p[j].v[i];
          q.v[i] = (T)(f[j] * (float)g.v[i]);
        }
        store_piece<STREAM>(dys + at[j] * lddys + c, q, D - c);
      }
    }
#pragma unroll
    for (int j = 0; j < J; j++) {
      const float s = wave_sum(dot[j]);
      if (W == 1) {
        if (lane_id() == 0 && j0 + j < K) dw[t * K + j0 + j] = s;
      } else if (lane_id() == 0) {
        part[wave_id()][j] = s;
      }
    }
    if (W == 1) continue;
    __syncthreads();
    if (threadIdx.x < J && j0 + (int)threadIdx.x < K) {
      float s = 0.0f;
      for (int v = 0; v < kWaves; v++) s += part[v][threadIdx.x];
      dw[t * K + j0 + threadIdx.x] = s;
    }
    __syncthreads();
  }
}

}  // namespace tok
}  // namespace samd
