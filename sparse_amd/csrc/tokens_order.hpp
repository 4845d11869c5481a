// tokens_order.hpp -- the stable order of tokens by a small whole number: choices by expert (one pass over at most 1025
// bins), token ids by vocabulary row (digit passes of at most 1024 bins, lowest digit first).
//
// A pass ranks each item among the equal digits of its wave (one ballot per digit bit), counts the waves' digits in LDS,
// and turns the counts into places by one scan; nothing is ordered by an atomic, so equal inputs give equal orders.
// Few items (4096 choices, 2048 ids) are ordered by one workgroup in a single launch.  More are split over at most 128
// workgroups: one launch counts every workgroup's digits, the next adds up the counts of the workgroups before its own
// (a column of at most 128 numbers per bin, out of L2) and places its items; up to 8192 choices
// (4096 ids, whose digits are further from even) the second launch counts for itself: a launch less, and 15 us instead of 18
// for 4096 ids, but 22 instead of 17 for 8192.  Items are 4 to 16 bytes each against rows
// of hundreds or thousands, so these launches are bound by their latency and by the ballots of the ranks: a wave ranks
// only 64 items at a time where there are workgroups enough (16384 ids of 18 bits: 17 us in four launches; with two items
// a lane 27 us, by one workgroup 43 us).
#pragma once

#include "tokens_common.hpp"

namespace samd {
namespace tok {

constexpr int kMaxExperts = 1024;
constexpr int kMaxBins = kMaxExperts + 1;  // the last bin: choices that name no expert
constexpr int kIdBits = 10, kIdBins = 1 << kIdBits;  // of a split pass over ids, at most
constexpr int kOneGroupChoices = 4096, kOneGroupIds = 2048;  // what one workgroup orders by itself
constexpr int kSplitWaves = 8, kSplitThreads = kSplitWaves * kWave;
constexpr int kTile = kSplitThreads;       // items a workgroup of a split pass places at a time
constexpr int kMaxGroups = 128;
constexpr int kSelfChoices = 8192, kSelfIds = 4096;  // up to so many, each workgroup of a split pass counts them all

// Rank of every item among the items of its wave with the same digit that come before it.  The wave's items are
// first + i * 64 + lane; digit < 0: no item.  cnt[d] (this wave's own, zeroed by the caller) ends as the wave's counts.
template <int IPL>
__device__ __forceinline__ void wave_ranks(const int (&digit)[IPL], int (&rank)[IPL], int bits, volatile int *cnt) {
  const int lane = lane_id();
#pragma unroll
  for (int i = 0; i < IPL; i++) {
    uint64_t peers = __ballot(digit[i] >= 0);
    for (int b = 0; b < bits; b++) {
      const uint64_t set = __ballot((digit[i] >> b) & 1);
      peers &= ((digit[i] >> b) & 1) ? set : ~set;
    }
    if (digit[i] >= 0) {
      const int before = __popcll(peers & ((1ull << lane) - 1ull));
      const int old = cnt[digit[i]];
      rank[i] = old + before;
      __builtin_amdgcn_wave_barrier();
      if (before == 0) cnt[digit[i]] = old + __popcll(peers);
    } else {
      rank[i] = 0;
      __builtin_amdgcn_wave_barrier();
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Exclusive scan over the threads of a workgroup of NW waves.
template <int NW>
__device__ __forceinline__ int group_scan(int v, int *wave_total, int *total) {
  const int s = (int)wave_inclusive_add_dpp((uint32_t)v);
  if (lane_id() == kWave - 1) wave_total[wave_id()] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NW; w++) {
    if (w < wave_id()) before += wave_total[w];
    all += wave_total[w];
  }
  __syncthreads();
  *total = all;
  return before + s - v;
}

// cnt[w * stride + b] = wave w's count of bin b  ->  the place of the first of them (bins ascending, waves ascending).
template <int NW>
__device__ __forceinline__ void counts_to_places(int *cnt, int stride, int bins, int *wave_total) {
  const int per = (bins + NW * kWave - 1) / (NW * kWave);
  const int b0 = (int)threadIdx.x * per, b1 = min(b0 + per, bins);
  int mine = 0;
  for (int b = b0; b < b1; b++)
    for (int w = 0; w < NW; w++) mine += cnt[w * stride + b];
  int total;
  int at = group_scan<NW>(mine, wave_total, &total);
  for (int b = b0; b < b1; b++)
    for (int w = 0; w < NW; w++) {
      const int c = cnt[w * stride + b];
      cnt[w * stride + b] = at;
      at += c;
    }
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------ choices by expert
// pos[i] = place of choice i (-1: it names no expert), src[p] = the choice at place p (-1 behind the last one),
// offsets[e] = first place of expert e, offsets[X] = how many choices have a place.

template <class I>
__device__ __forceinline__ int expert_of(const I *chosen, int64_t i, int64_t n, int X) {
  if (i >= n) return -1;
  const int64_t e = (int64_t)chosen[i];
  return e >= 0 && e < X ? (int)e : X;
}

__device__ __forceinline__ void write_choice(int e, int X, int64_t i, int64_t place, int32_t *pos, int32_t *src) {
  pos[i] = e < X ? (int32_t)place : -1;
  src[place] = e < X ? (int32_t)i : -1;
}

template <class I, int NW, int IPL>
__global__ __launch_bounds__(NW *kWave) void route_small_kernel(const I *__restrict__ chosen, int n, int X, int bits,
                                                                int32_t *__restrict__ pos, int32_t *__restrict__ src,
                                                                int32_t *__restrict__ offsets) {
  __shared__ int cnt[NW * kMaxBins];
  __shared__ int wave_total[NW];
  const int bins = X + 1;
  for (int b = threadIdx.x; b < NW * bins; b += NW * kWave) cnt[b] = 0;
  __syncthreads();
  const int first = wave_id() * kWave * IPL + lane_id();
  int digit[IPL], rank[IPL];
#pragma unroll
  for (int i = 0; i < IPL; i++) digit[i] = expert_of(chosen, first + i * kWave, n, X);
  wave_ranks<IPL>(digit, rank, bits, cnt + wave_id() * bins);
  __syncthreads();
  counts_to_places<NW>(cnt, bins, bins, wave_total);
#pragma unroll
  for (int i = 0; i < IPL; i++)
    if (digit[i] >= 0) write_choice(digit[i], X, first + i * kWave, cnt[wave_id() * bins + digit[i]] + rank[i], pos, src);
  for (int b = threadIdx.x; b < bins; b += NW * kWave) offsets[b] = cnt[b];
}

// ------------------------------------------------------------------------------------------------ split passes
// The digits a pass orders by: choices (BY = 0), the lowest digit of the ids themselves (1), a later digit of keys (2).
template <int BY, class I>
struct Digits {
  const I *ids;
  const uint32_t *keys;
  int64_t n;
  int64_t V;      // experts, or rows of the table: what names none of them comes last
  int shift, mask;
  __device__ __forceinline__ uint32_t key(int64_t i) const {
    if (BY == 2) return keys[i];
    const int64_t v = (int64_t)ids[i];
    return (uint32_t)(v >= 0 && v < V ? v : V);
  }
  __device__ __forceinline__ int digit(uint32_t k) const { return BY == 0 ? (int)k : (int)((k >> shift) & (uint32_t)mask); }
};

// hist[g * bins + b] = how many of workgroup g's items have digit b.  `clear`: null, or words to zero on the way.
template <int BY, class I>
__global__ __launch_bounds__(kSplitThreads) void digit_count_kernel(Digits<BY, I> d, int64_t per_group, int bins, int *__restrict__ hist,
                                                                    uint32_t *__restrict__ clear, int64_t clear_words) {
  __shared__ int cnt[BY == 0 ? kMaxBins : kIdBins];
  for (int64_t k = (int64_t)blockIdx.x * kSplitThreads + threadIdx.x; k < clear_words; k += (int64_t)gridDim.x * kSplitThreads) clear[k] = 0;
  for (int b = threadIdx.x; b < bins; b += kSplitThreads) cnt[b] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * per_group, i1 = i0 + per_group < d.n ? i0 + per_group : d.n;
#pragma unroll 2
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kSplitThreads) atomicAdd(&cnt[d.digit(d.key(i))], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSplitThreads) hist[(int64_t)blockIdx.x * bins + b] = cnt[b];
}

struct PassOut {
  int32_t *pos, *src, *offsets;      // choices
  uint32_t *keys;                    // ids: the keys and the items in their new order
  int32_t *items;
  const int32_t *items_in;           // null: item i is i
  uint8_t *named;                    // null, or a byte for every row of the table (zeroed): set where an id names it
};

// hist == null: every workgroup counts all items for itself.
template <int BY, class I>
__global__ __launch_bounds__(kSplitThreads) void digit_place_kernel(Digits<BY, I> d, int64_t per_group, int bins, int bits,
                                                                    const int *__restrict__ hist, PassOut o) {
  constexpr int IPL = kTile / kSplitThreads;
  constexpr int kBins = BY == 0 ? kMaxBins : kIdBins;
  __shared__ int cnt[kSplitWaves * kBins];
  __shared__ int base[kBins];
  __shared__ int wave_total[kSplitWaves];
  const int groups = (int)gridDim.x, g = (int)blockIdx.x;
  const int64_t i0 = (int64_t)g * per_group, i1 = i0 + per_group < d.n ? i0 + per_group : d.n;

  // base[b] = items with a smaller digit, and those with digit b in workgroups before this one
  const int per = (bins + kSplitThreads - 1) / kSplitThreads;
  const int b0 = (int)threadIdx.x * per, b1 = min(b0 + per, bins);
  if (!hist) {
    for (int b = threadIdx.x; b < bins; b += kSplitThreads) cnt[b] = base[b] = 0;
    // a part of the rows' bytes is this workgroup's to clear and to set: it sees all ids here
    const int64_t words = o.named ? ((d.V + 3) / 4 + groups - 1) / groups : 0;
    const uint32_t v0 = (uint32_t)(g * words * 4), v1 = (uint32_t)(v0 + words * 4 < d.V ? v0 + words * 4 : d.V);
    for (int64_t k = g * words + threadIdx.x; k < (g + 1) * words && k < (d.V + 3) / 4; k += kSplitThreads) ((uint32_t *)o.named)[k] = 0;
    __syncthreads();
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < d.n; i += kSplitThreads) {
      const uint32_t key = d.key(i);
      const int v = d.digit(key);
      atomicAdd(&cnt[v], 1);
      if (i < i0) atomicAdd(&base[v], 1);
      if (o.named && key >= v0 && key < v1) o.named[key] = 1;
    }
    __syncthreads();
  }
  int all = 0;
  for (int b = b0; b < b1; b++) {
    if (hist) {
      int before = 0, total = 0;
#pragma unroll 16
      for (int k = 0; k < groups; k++) {
        const int c = hist[(int64_t)k * bins + b];
        total += c;
        before += k < g ? c : 0;
      }
      base[b] = before;
      cnt[b] = total;
    }
    all += cnt[b];
  }
  int unused;
  int at = group_scan<kSplitWaves>(all, wave_total, &unused);
  for (int b = b0; b < b1; b++) {
    if (BY == 0 && g == 0) o.offsets[b] = at;
    base[b] += at;
    at += cnt[b];
  }
  __syncthreads();

  for (int64_t t0 = i0; t0 < i1; t0 += kTile) {
    const int64_t first = t0 + wave_id() * (kWave * IPL) + lane_id();
    uint32_t key[IPL];
    int digit[IPL], rank[IPL];
#pragma unroll
    for (int i = 0; i < IPL; i++) {
      const int64_t at_i = first + i * kWave;
      key[i] = at_i < i1 ? d.key(at_i) : 0u;
      digit[i] = at_i < i1 ? d.digit(key[i]) : -1;
    }
    for (int b = threadIdx.x; b < kSplitWaves * bins; b += kSplitThreads) cnt[b] = 0;
    __syncthreads();
    int *mine = cnt + wave_id() * bins;
    wave_ranks<IPL>(digit, rank, bits, mine);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSplitThreads) {
      int run = base[b];
#pragma unroll
      for (int w = 0; w < kSplitWaves; w++) {
        const int c = cnt[w * bins + b];
        cnt[w * bins + b] = run;
        run += c;
      }
      base[b] = run;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IPL; i++) {
      if (digit[i] < 0) continue;
      const int64_t at_i = first + i * kWave;
      const int64_t place = mine[digit[i]] + rank[i];
      if (BY == 0) {
        write_choice(digit[i], (int)d.V, at_i, place, o.pos, o.src);
      } else {
        o.keys[place] = key[i];
        o.items[place] = o.items_in ? o.items_in[at_i] : (int32_t)at_i;
        if (o.named && hist && (int64_t)key[i] < d.V) o.named[key[i]] = 1;
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ ids by table row, small
// All passes of up to 2048 ids in one workgroup, keys and items in LDS between them.
constexpr int kSmallBits = 9;

template <class I, int IPL>
__global__ __launch_bounds__(1024) void id_sort_small_kernel(const I *__restrict__ ids, int n, int64_t V, int passes, int bits,
                                                             uint32_t *__restrict__ keys, int32_t *__restrict__ items,
                                                             uint8_t *__restrict__ named) {
  constexpr int NW = 16;
  __shared__ uint32_t skey[NW * kWave * IPL];
  __shared__ uint16_t sitem[NW * kWave * IPL];
  __shared__ int cnt[NW << kSmallBits];
  __shared__ int wave_total[NW];
  if (named) {  // a byte for every row of the table, a whole number of words
    for (int64_t k = threadIdx.x; k < (V + 3) / 4; k += NW * kWave) ((uint32_t *)named)[k] = 0;
    __syncthreads();
  }
  const int first = wave_id() * kWave * IPL + lane_id();
  const int bins = 1 << bits;
  uint32_t key[IPL];
  int32_t item[IPL];
  int digit[IPL], rank[IPL];
#pragma unroll
  for (int i = 0; i < IPL; i++) {
    const int at = first + i * kWave;
    key[i] = 0;
    item[i] = at;
    if (at < n) {
      const int64_t v = (int64_t)ids[at];
      key[i] = (uint32_t)(v >= 0 && v < V ? v : V);
      if (named && (int64_t)key[i] < V) named[key[i]] = 1;
    }
  }
  for (int p = 0; p < passes; p++) {
    for (int b = threadIdx.x; b < NW * bins; b += NW * kWave) cnt[b] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IPL; i++) digit[i] = first + i * kWave < n ? (int)((key[i] >> (p * bits)) & (uint32_t)(bins - 1)) : -1;
    wave_ranks<IPL>(digit, rank, bits, cnt + wave_id() * bins);
    __syncthreads();
    counts_to_places<NW>(cnt, bins, bins, wave_total);
    const bool last = p == passes - 1;
#pragma unroll
    for (int i = 0; i < IPL; i++)
      if (digit[i] >= 0) {
        const int place = cnt[wave_id() * bins + digit[i]] + rank[i];
        if (last) {
          keys[place] = key[i];
          items[place] = item[i];
        } else {
          skey[place] = key[i];
          sitem[place] = (uint16_t)item[i];
        }
      }
    __syncthreads();
    if (!last)
#pragma unroll
      for (int i = 0; i < IPL; i++)
        if (first + i * kWave < n) {
          key[i] = skey[first + i * kWave];
          item[i] = sitem[first + i * kWave];
        }
  }
}

}  // namespace tok
}  // namespace samd
