// tokens.hip -- the sparse_amd_tokens_* entries of include/sparse_amd.h: argument checks, workspaces, launches.
//
// These entries take plain device pointers with row strides and the stream to run on.  They allocate nothing, keep
// nothing from one call to the next and never wait, so they may be captured into a graph; the caller's device is the
// current one again when they return.
#include "tokens_rows.hpp"
#include "tokens_lookup_grad.hpp"
#include "tokens_experts.hpp"

#include <initializer_list>

using namespace samd;
using namespace samd::tok;

namespace {

struct OnDevice {
  std::lock_guard<std::mutex> g;
  int before = -1;
  explicit OnDevice(futhark_context *ctx) : g(ctx->mu) {
    if (ctx->own_stream && hipGetDevice(&before) == hipSuccess && before != ctx->device) (void)hipSetDevice(ctx->device);
    else before = -1;
    ctx->n_entries++;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// A context whose device could not be opened launches nothing; arguments are checked all the same, before that is looked at.
int need_device(futhark_context *ctx) {
  return ctx->own_stream ? 0 : set_error(ctx, "context has no usable HIP device; libsparse_amd has no CPU path");
}

// Runs `body` with the context locked and its device current; no exception leaves.
template <class F>
int entry(futhark_context *ctx, F body) {
  if (!ctx) return 1;
  try {
    OnDevice on(ctx);
    const int rc = body();
    return rc ? rc : need_device(ctx);
  } catch (...) {
    return 1;
  }
}

template <class T>
struct Tag { typedef T type; };

template <class F>
int by_type(futhark_context *ctx, const char *who, int type, F f) {
  switch (type) {
    case SPARSE_AMD_F32: return f(Tag<float>());
    case SPARSE_AMD_F16: return f(Tag<f16>());
    case SPARSE_AMD_BF16: return f(Tag<bf16>());
  }
  return set_error(ctx, "%s: unknown element type %d", who, type);
}

template <class F>
int by_type16(futhark_context *ctx, const char *who, int type, F f) {
  switch (type) {
    case SPARSE_AMD_F16: return f(Tag<f16>());
    case SPARSE_AMD_BF16: return f(Tag<bf16>());
    case SPARSE_AMD_F32: return set_error(ctx, "%s: the experts' products are offered for 16-bit elements", who);
  }
  return set_error(ctx, "%s: unknown element type %d", who, type);
}

template <class F>
int by_index(futhark_context *ctx, const char *who, int bits, F f) {
  if (bits == 32) return f(Tag<int32_t>());
  if (bits == 64) return f(Tag<int64_t>());
  return set_error(ctx, "%s: indices have 32 or 64 bits, not %d", who, bits);
}

int64_t type_size(int type) { return type == SPARSE_AMD_F32 ? 4 : 2; }

// A panel of `rows` rows of `cols` elements of `size` bytes, `ld` elements apart; null where there is none.
struct Panel {
  const char *name;
  const void *p;
  int64_t rows, cols, ld, size;
  int64_t bytes() const { return rows > 0 && cols > 0 ? ((rows - 1) * ld + cols) * size : 0; }
};

// Every panel has a place; the results (the first `outs` panels) have strides that keep their rows apart and share no byte
// with each other or with what is read.  Rows that are only read may lie over each other (a stride of zero: one row for all).
int check_panels(futhark_context *ctx, const char *who, int outs, std::initializer_list<Panel> panels) {
  int k = 0;
  for (const Panel &a : panels) {
    if (a.rows < 0 || a.cols < 0) return set_error(ctx, "%s: %s has a negative size", who, a.name);
    if (a.rows > 1 && a.ld < 0) return set_error(ctx, "%s: %s has a negative stride", who, a.name);
    if (k++ < outs && a.rows > 1 && a.ld < a.cols) return set_error(ctx, "%s: the rows of %s are %lld apart and %lld long", who, a.name, (long long)a.ld, (long long)a.cols);
    if (a.ld > ((int64_t)1 << 40) || a.rows > ((int64_t)1 << 40) || a.cols > ((int64_t)1 << 40) ||
        (a.rows > 0 && a.ld > 0 && a.rows > ((int64_t)1 << 56) / a.ld))
      return set_error(ctx, "%s: %s is too large", who, a.name);
    if (a.bytes() > 0 && !a.p) return set_error(ctx, "%s: %s is null", who, a.name);
    if (a.p && (uintptr_t)a.p % (uintptr_t)a.size) return set_error(ctx, "%s: %s is not aligned to its elements", who, a.name);
  }
  int i = 0;
  for (const Panel *a = panels.begin(); a != panels.end() && i < outs; a++, i++)
    for (const Panel *b = a + 1; b != panels.end(); b++) {
      const char *pa = (const char *)a->p, *pb = (const char *)b->p;
      if (a->bytes() > 0 && b->bytes() > 0 && pa < pb + b->bytes() && pb < pa + a->bytes())
        return set_error(ctx, "%s: %s overlaps %s", who, a->name, b->name);
    }
  return 0;
}

int check_blocks(futhark_context *ctx, const char *who, int64_t blocks) {
  if (blocks > 0x7fffffff) return set_error(ctx, "%s: more work than one launch can hold", who);
  return 0;
}

// As many for a kernel that takes its workgroups' numbers from the grid's first dimension alone.
int check_row(futhark_context *ctx, const char *who, int64_t blocks, int threads) {
  return check_blocks(ctx, who, blocks * threads < (int64_t)1 << 32 ? blocks : (int64_t)1 << 32);
}

#define TOK_LAUNCH(ctx, kernel, blocks, threads, stream, ...)                                                  \
  do {                                                                                                         \
    SAMD_TRY(need_device(ctx));                                                                                \
    hipLaunchKernelGGL(kernel, grid_of(blocks, threads), dim3((unsigned)(threads)), 0, stream, __VA_ARGS__);        \
    SAMD_LAUNCH_CHECK(ctx);                                                                                    \
  } while (0)

// Rows in pieces of U = 4 keep four loads in flight per lane; a launch too small to fill the card with such waves is
// spread over more of them instead.
constexpr int64_t kFullCard = 2048;

// ---------------------------------------------------------------- workspaces
struct Carve {  // adds up 256-byte aligned parts of a workspace
  char *base;
  int64_t used = 0;
  explicit Carve(void *p) : base((char *)p) {}
  template <class T>
  T *take(int64_t count) {
    T *p = base ? (T *)(base + used) : nullptr;
    used += (count * (int64_t)sizeof(T) + 255) & ~(int64_t)255;
    return p;
  }
};

struct Split {  // a split pass: its workgroups and how many items each has
  int64_t per_group;
  int groups;
  explicit Split(int64_t n) {
    per_group = cdiv(cdiv(n, kMaxGroups), kTile) * kTile;
    groups = (int)cdiv(n, per_group);
  }
};

struct GradPlan {
  GradShape g;
  bool small;
  int passes, bits;
  Split split;
  uint32_t *keys, *keys2;
  int32_t *items, *items2;
  int *hist;
  float *part;
  uint8_t *named;
  int64_t bytes;

  GradPlan(void *work, int type, int64_t n, int64_t V, int64_t D) : split(n > 0 ? n : 1) {
    const int64_t per = 16 / type_size(type);
    g = {};
    g.n = n; g.V = V; g.D = D;
    g.segs = cdiv(cdiv(D, per), kWave);
    // chunks of 32 read a key, an item and two chunk ends for 32 rows; where that leaves the card empty, chunks of 8
    g.chunk = cdiv(n, 32) * g.segs >= kFullCard ? 32 : 8;
    g.chunks = cdiv(n, g.chunk);
    small = n <= kOneGroupIds && V <= ((int64_t)1 << 22);  // one workgroup clears the rows' bytes too
    const int key_bits = bits_for(V + 1) > 0 ? bits_for(V + 1) : 1;
    const int most = small ? kSmallBits : kIdBits;
    passes = (key_bits + most - 1) / most;
    bits = (key_bits + passes - 1) / passes;
    Carve c(work);
    keys = c.take<uint32_t>(n);
    items = c.take<int32_t>(n);
    keys2 = small ? nullptr : c.take<uint32_t>(n);
    items2 = small ? nullptr : c.take<int32_t>(n);
    hist = n <= kSelfIds ? nullptr : c.take<int>((int64_t)split.groups << bits);
    named = c.take<uint8_t>(cdiv(V, 4) * 4);
    part = c.take<float>(g.chunks > 1 ? g.chunks * 2 * g.segs * kWave * per : 0);
    bytes = c.used;
  }

  // Workgroups of the launch that sums and zeroes (zeroes nothing until it has been told how), and of the one that joins.
  void zero(int out_type) { g.fill = deal_rows(g.V, cdiv(g.D, 16 / type_size(out_type)), kFillPieces); }
  int64_t sum_blocks() const { return cdiv(join_blocks() + g.fill.waves, kWaves); }
  int64_t join_blocks() const { return g.chunks * g.segs; }
};

int check_work(futhark_context *ctx, const char *who, const void *work, int64_t have, int64_t need) {
  if (need == 0) return 0;
  if (!work || have < need) return set_error(ctx, "%s: needs a workspace of %lld bytes, got %lld", who, (long long)need, (long long)(work ? have : 0));
  if ((uintptr_t)work % 256) return set_error(ctx, "%s: the workspace is not aligned to 256 bytes", who);
  return 0;
}

template <class I>
int order_ids(futhark_context *ctx, hipStream_t stream, const I *ids, const GradPlan &p, bool mark) {
  uint8_t *named = mark ? p.named : nullptr;
  const int n = (int)p.g.n;
  if (p.small) {
    if (n <= 1024)
      TOK_LAUNCH(ctx, (id_sort_small_kernel<I, 1>), 1, 1024, stream, ids, n, p.g.V, p.passes, p.bits, p.keys, p.items, named);
    else
      TOK_LAUNCH(ctx, (id_sort_small_kernel<I, 2>), 1, 1024, stream, ids, n, p.g.V, p.passes, p.bits, p.keys, p.items, named);
    return 0;
  }
  const int bins = 1 << p.bits, mask = bins - 1;
  const bool self = n <= kSelfIds;
  const int *hist = self ? nullptr : p.hist;
  for (int k = 0; k < p.passes; k++) {
    const bool to_first = (p.passes - 1 - k) % 2 == 0;
    PassOut o = {};
    o.keys = to_first ? p.keys : p.keys2;
    o.items = to_first ? p.items : p.items2;
    if (k == 0) {
      const Digits<1, I> d = {ids, nullptr, p.g.n, p.g.V, 0, mask};
      o.named = named;
      if (!self)
        TOK_LAUNCH(ctx, (digit_count_kernel<1, I>), p.split.groups, kSplitThreads, stream, d, p.split.per_group, bins, p.hist,
                   (uint32_t *)named, named ? cdiv(p.g.V, 4) : 0);
      TOK_LAUNCH(ctx, (digit_place_kernel<1, I>), p.split.groups, kSplitThreads, stream, d, p.split.per_group, bins, p.bits, hist, o);
    } else {
      o.items_in = to_first ? p.items2 : p.items;
      const Digits<2, I> d = {nullptr, to_first ? p.keys2 : p.keys, p.g.n, p.g.V, k * p.bits, mask};
      if (!self)
        TOK_LAUNCH(ctx, (digit_count_kernel<2, I>), p.split.groups, kSplitThreads, stream, d, p.split.per_group, bins, p.hist,
                   (uint32_t *)nullptr, (int64_t)0);
      TOK_LAUNCH(ctx, (digit_place_kernel<2, I>), p.split.groups, kSplitThreads, stream, d, p.split.per_group, bins, p.bits, hist, o);
    }
  }
  return 0;
}

template <class T, class TO, bool ADD, bool STREAM>
int sum_ids(futhark_context *ctx, hipStream_t stream, TO *dE, const T *dy, const float *vals, float scale, const GradPlan &p) {
  TOK_LAUNCH(ctx, (lookup_grad_kernel<T, TO, ADD, STREAM>), p.sum_blocks(), kThreads, stream, dE, dy, vals, scale, (const uint32_t *)p.keys,
             (const int32_t *)p.items, (const uint8_t *)p.named, p.part, p.g);
  if (p.g.chunks > 1)
    TOK_LAUNCH(ctx, (lookup_grad_join_kernel<T, TO, ADD, STREAM>), p.join_blocks(), kThreads, stream, dE, (const uint32_t *)p.keys, p.part, p.g);
  return 0;
}

template <class T, class TO, class I, bool ADD, bool STREAM>
int sum_few(futhark_context *ctx, hipStream_t stream, TO *dE, const T *dy, const I *ids, const float *vals, float scale, GradShape g) {
  const int64_t units = cdiv(g.D, kPer<TO>);
  g.fill = deal_rows(1, units, 1);
  // 16 to 128 KiB of zeros for a workgroup: two of them on every CU if there is that much
  const int64_t share = g.V * units * 16 / 512;
  const int64_t rows = (share < 16 * 1024 ? 16 * 1024 : share > 128 * 1024 ? 128 * 1024 : share) / (units * 16);
  const int fill_rows = (int)(rows < 1 ? 1 : rows > kFewFillRows ? kFewFillRows : rows);
  const int64_t blocks = g.segs + (ADD ? 0 : cdiv(g.V, fill_rows));
  SAMD_TRY(check_row(ctx, "lookup_grad", blocks, kFewWaves * kWave));
  TOK_LAUNCH(ctx, (lookup_grad_few_kernel<T, TO, I, ADD, STREAM>), blocks, kFewWaves * kWave, stream, dE, dy, ids, vals, scale, g, fill_rows);
  return 0;
}

template <class T, class TO, class I>
int sum_few_as(futhark_context *ctx, hipStream_t stream, bool add, TO *dE, const T *dy, const I *ids, const float *vals, float scale, const GradShape &g) {
  if (add) return sum_few<T, TO, I, true, false>(ctx, stream, dE, dy, ids, vals, scale, g);
  if (g.V * g.D * (int64_t)sizeof(TO) > kStreamBytes) return sum_few<T, TO, I, false, true>(ctx, stream, dE, dy, ids, vals, scale, g);
  return sum_few<T, TO, I, false, false>(ctx, stream, dE, dy, ids, vals, scale, g);
}

// The gradient's table: written past the caches when all of it is written and it is large.
template <class T, class TO>
int sum_ids_as(futhark_context *ctx, hipStream_t stream, bool add, TO *dE, const T *dy, const float *vals, float scale, const GradPlan &p) {
  if (add) return sum_ids<T, TO, true, false>(ctx, stream, dE, dy, vals, scale, p);
  if (p.g.V * p.g.D * (int64_t)sizeof(TO) > kStreamBytes) return sum_ids<T, TO, false, true>(ctx, stream, dE, dy, vals, scale, p);
  return sum_ids<T, TO, false, false>(ctx, stream, dE, dy, vals, scale, p);
}

// ---------------------------------------------------------------- experts
// Rows that begin on 16 bytes, and apart from each other: the buffer's end is what tells rows behind the last one.
template <class T>
bool direct_to_lds(const T *p, int64_t ld, int64_t width) {
  return (uintptr_t)p % 16 == 0 && ld >= width && ld % 8 == 0 && ld <= ((int64_t)1 << 20);
}

enum { kSteps = 0, kAny = 1, kFew = 2 };  // the kernel: experts_kernel, experts_any_kernel, experts_few_kernel
template <class T, class TO, int KIND, int BM, int BN, int DEPTH, int WM, int WN, bool ADD, bool ONCE = false, int KERNEL = kSteps>
int launch_experts(futhark_context *ctx, const char *who, hipStream_t stream, TO *C, const T *A, const T *B, const int32_t *offsets,
                   ProductShape g) {
  const int64_t n_tiles = cdiv(g.N, BN);
  int64_t m_tiles, blocks;
  if (KIND == kGradW) {
    m_tiles = cdiv(g.M, BM);
    blocks = g.X * (cdiv(m_tiles * n_tiles, kXcds) * kXcds);
  } else {
    // every expert with rows ends in one tile that may not be full
    m_tiles = g.rows / BM + (g.rows < g.X ? g.rows : g.X);
    blocks = m_tiles * n_tiles;
  }
  blocks = cdiv(blocks, kXcds) * kXcds;
  g.split = 1;
  if (KIND != kGradW && BM == 256 && BN == 256 && m_tiles * n_tiles > ctx->num_cu) {  // room for the halves of half a round
    g.split = ctx->num_cu;
    blocks += cdiv(ctx->num_cu / 2, kXcds) * kXcds + 4 * kXcds;
  }
  SAMD_TRY(check_row(ctx, who, blocks, WM * WN * kWave));
  g.m_tiles = (int)m_tiles;
  g.n_tiles = (int)n_tiles;
  if constexpr (KERNEL == kFew)
    TOK_LAUNCH(ctx, (experts_few_kernel<T, TO, BM, BN, DEPTH, WM, WN, ADD>), blocks, WM * WN * kWave, stream, C, A, B, offsets, g);
  else if constexpr (KERNEL == kAny)
    TOK_LAUNCH(ctx, (experts_any_kernel<T, TO, KIND, BM, BN, DEPTH, WM, WN, ADD>), blocks, WM * WN * kWave, stream, C, A, B, offsets, g);
  else
    TOK_LAUNCH(ctx, (experts_kernel<T, TO, KIND, BM, BN, DEPTH, WM, WN, ADD, ONCE>), blocks, WM * WN * kWave, stream, C, A, B, offsets, g);
  return 0;
}

template <class T, int KIND>
int experts_panels(futhark_context *ctx, const char *who, hipStream_t stream, T *C, const T *A, const T *B, const int32_t *offsets,
                   const ProductShape &g) {
  const bool fast = direct_to_lds(A, g.ldA, g.K) && g.K % 8 == 0 && direct_to_lds(B, g.ldB, KIND == kForward ? g.K : g.N) && g.blockB % 8 == 0;
  if (!fast) {
    if (g.rows <= 48 * g.X) return launch_experts<T, T, KIND, 32, 64, 128, 1, 4, false, false, kAny>(ctx, who, stream, C, A, B, offsets, g);
    return launch_experts<T, T, KIND, 128, 128, 64, 2, 2, false, false, kAny>(ctx, who, stream, C, A, B, offsets, g);
  }
  // The tile whose launch is estimated to end first: rounds of the card's CUs, at the time that a tile takes for 64 of the
  // summed index, or one pass over the blocks where no cache holds them, at the rate that a tile's loads reach (64 bytes of
  // every row of W at a time are slower than whole lines).  Both were fitted to the times of all five tiles for 2 to 2048
  // rows an expert in eleven shapes from 2 blocks of 2048 x 512 to 32 of 4096 x 2048, where the choice is 1.3 % behind the
  // fastest tile on average and 29 % at most; in six others, 256 wide to 8192, 2.9 % (from rates alone: 9 % and 82 %).
  // Small tiles waste fewer rows of a small expert, large ones read each operand less often: 32 experts of 4096 x 2048,
  // forward, 16 rows each: 32 x 64 83 us, 128 x 256 91, 256 x 256 94; 64 rows: 158, 99 and 102; 256 rows: 419, 193 and 182.
  struct Cost { int bm, bn; double step, rate; };  // microseconds, TB/s
  static const Cost forward[] = {{32, 64, 0.20, 6.4}, {64, 256, 0.93, 4.2}, {128, 128, 0.64, 5.2}, {128, 256, 0.92, 6.2}, {256, 256, 1.15, 5.2}};
  static const Cost grad_x[] = {{32, 64, 0.16, 4.8}, {64, 256, 0.83, 6.6}, {128, 128, 0.64, 5.1}, {128, 256, 1.15, 5.2}, {256, 256, 1.40, 5.2}};
  const Cost *const tiles = KIND == kForward ? forward : grad_x;
  const double used = (double)(g.rows < g.X ? g.rows : g.X), mean = (double)g.rows / used, bytes = used * g.N * g.K * sizeof(T);
  const bool cached = bytes <= (double)((int64_t)256 << 20);  // the card's last cache
  int best = 0;
  double least = 0;
  for (int i = 0; i < 5; i++) {
    // an expert's last tile is half full, if it has several
    const double full = mean / tiles[i].bm + 0.5, count = used * (full > 1 ? full : 1) * (double)cdiv(g.N, tiles[i].bn) / ctx->num_cu;
    double rounds = ceil(count);
    if (i == 4 && rounds > 1 && rounds - count >= 0.5) rounds -= 0.4;  // a last round of half tiles
    double t = rounds * ((double)g.K / 64) * tiles[i].step;
    if (!cached && bytes / tiles[i].rate * 1e-6 > t) t = bytes / tiles[i].rate * 1e-6;
    if (i == 0 || t < least) {
      best = i;
      least = t;
    }
  }
  // weights that no cache can hold until the next call are read past it where nearly every block is read once: 32 blocks
  // of 4096 x 2048, 94 -> 83 us; 8 of them, which it holds, 27 -> 33
  const bool once = 4 * mean <= 3 * tiles[best].bm && !cached;
  switch (best) {
    case 0:
      return once ? launch_experts<T, T, KIND, 32, 64, 64, 1, 4, false, true>(ctx, who, stream, C, A, B, offsets, g)
                  : launch_experts<T, T, KIND, 32, 64, 64, 1, 4, false>(ctx, who, stream, C, A, B, offsets, g);
    case 1:
      return once ? launch_experts<T, T, KIND, 64, 256, 32, 1, 4, false, true>(ctx, who, stream, C, A, B, offsets, g)
                  : launch_experts<T, T, KIND, 64, 256, 32, 1, 4, false>(ctx, who, stream, C, A, B, offsets, g);
    case 2: return launch_experts<T, T, KIND, 128, 128, 32, 2, 2, false>(ctx, who, stream, C, A, B, offsets, g);
    case 3: return launch_experts<T, T, KIND, 128, 256, 64, 2, 4, false>(ctx, who, stream, C, A, B, offsets, g);
    default: return launch_experts<T, T, KIND, 256, 256, 64, 2, 4, false>(ctx, who, stream, C, A, B, offsets, g);
  }
}

template <class T, class TO, bool ADD>
int experts_weights(futhark_context *ctx, const char *who, hipStream_t stream, TO *C, const T *A, const T *B, const int32_t *offsets,
                    const ProductShape &g) {
  // small tiles where large ones would leave CUs without work (a tile's sum is one workgroup's): 8 blocks of 512 x 256, 1024
  // rows each: 64 x 64 10 us, 128 x 128 14; 30 of 208 x 2024, 960 tiles of 128 x 128: 74 and 46
  const bool small = g.X * cdiv(g.M, 128) * cdiv(g.N, 128) <= 128;
  if (!(direct_to_lds(A, g.ldA, g.M) && direct_to_lds(B, g.ldB, g.N))) {
    if (small || g.rows <= 48 * g.X) return launch_experts<T, TO, kGradW, 64, 64, 32, 2, 2, ADD, false, kAny>(ctx, who, stream, C, A, B, offsets, g);
    return launch_experts<T, TO, kGradW, 128, 128, 64, 2, 2, ADD, false, kAny>(ctx, who, stream, C, A, B, offsets, g);
  }
  if (g.rows <= 160 * g.X) {
    // past the caches unless rows of dw share their lines: few sums leave the cache time to join the parts (110 blocks of
    // 2888 x 688, 16 rows each: 149 us, past it 187; 192 rows: 279 and 215)
    ProductShape few = g;
    few.stream = g.stream && (((uintptr_t)C | g.ldC * sizeof(TO) | g.blockC * sizeof(TO)) % 128 == 0 || g.rows > 64 * g.X);
    return launch_experts<T, TO, kGradW, 128, 128, 32, 2, 2, ADD, false, kFew>(ctx, who, stream, C, A, B, offsets, few);
  }
  if (small) return launch_experts<T, TO, kGradW, 64, 64, 32, 1, 4, ADD>(ctx, who, stream, C, A, B, offsets, g);
  // as above: tiles enough for every CU to have a large one
  if (g.X * cdiv(g.M, 256) * cdiv(g.N, 256) >= 256) return launch_experts<T, TO, kGradW, 256, 256, 64, 2, 4, ADD>(ctx, who, stream, C, A, B, offsets, g);
  return launch_experts<T, TO, kGradW, 128, 128, 32, 2, 2, ADD>(ctx, who, stream, C, A, B, offsets, g);
}

// Elements from a block's first to behind its last one.
int64_t block_span(int64_t F, int64_t D, int64_t ld) { return F > 0 && D > 0 ? (F - 1) * ld + D : 0; }

int check_experts(futhark_context *ctx, const char *who, int64_t rows, int64_t X, int64_t F, int64_t D, const int32_t *offsets) {
  if (rows < 0 || F < 0 || D < 0) return set_error(ctx, "%s: negative size", who);
  if (X < 1 || X > kMaxExperts) return set_error(ctx, "%s: %lld experts (1 to %d are offered)", who, (long long)X, kMaxExperts);
  if (rows > 0x7fffffff) return set_error(ctx, "%s: %lld rows (places have 31 bits)", who, (long long)rows);
  if (F > 0x3fffffff || D > 0x3fffffff) return set_error(ctx, "%s: a block of %lld x %lld is too large", who, (long long)F, (long long)D);
  if (!offsets) return set_error(ctx, "%s: offsets is null", who);
  return 0;
}

}  // namespace

extern "C" {

int sparse_amd_tokens_lookup(struct futhark_context *ctx, void *stream, int type, void *y, int64_t ldy, const void *table, int64_t V,
                             int64_t D, int64_t ldt, const void *ids, int id_bits, int64_t n, const float *vals, float scale) {
  return entry(ctx, [&]() -> int {
    const char *who = "lookup";
    return by_type(ctx, who, type, [&](auto t) {
      return by_index(ctx, who, id_bits, [&](auto it) -> int {
        typedef typename decltype(t)::type T;
        typedef typename decltype(it)::type I;
        SAMD_TRY(check_panels(ctx, who, 1, {{"the result", y, n, D, ldy, (int64_t)sizeof(T)}, {"the table", table, V, D, ldt, (int64_t)sizeof(T)},
                                            {"ids", ids, 1, n, n, (int64_t)sizeof(I)}, {"vals", vals, 1, vals ? n : 0, n, 4}}));
        if (n == 0 || D == 0) return 0;
        const hipStream_t s = (hipStream_t)stream;
        const int64_t units = cdiv(D, kPer<T>);
        RowDeal d = deal_rows(n, units, 4);
        const int u = d.lg == 6 && d.waves >= kFullCard ? 4 : 1;
        if (u == 1) d = deal_rows(n, units, 1);
        SAMD_TRY(check_blocks(ctx, who, cdiv(d.waves, kWaves)));
        const auto go = [&](auto kernel) -> int {
          TOK_LAUNCH(ctx, kernel, cdiv(d.waves, kWaves), kThreads, s, (T *)y, ldy, (const T *)table, ldt, V, D, (const I *)ids, n, vals, scale, d.lg, d.segs);
          return 0;
        };
        if (n * D * (int64_t)sizeof(T) > kStreamBytes) return u == 4 ? go(lookup_kernel<T, I, 4, true>) : go(lookup_kernel<T, I, 1, true>);
        return u == 4 ? go(lookup_kernel<T, I, 4, false>) : go(lookup_kernel<T, I, 1, false>);
      });
    });
  });
}

int sparse_amd_tokens_lookup_dots(struct futhark_context *ctx, void *stream, int type, float *dvals, const void *dy, int64_t ldy,
                                  const void *table, int64_t V, int64_t D, int64_t ldt, const void *ids, int id_bits, int64_t n,
                                  float scale) {
  return entry(ctx, [&]() -> int {
    const char *who = "lookup_dots";
    return by_type(ctx, who, type, [&](auto t) {
      return by_index(ctx, who, id_bits, [&](auto it) -> int {
        typedef typename decltype(t)::type T;
        typedef typename decltype(it)::type I;
        SAMD_TRY(check_panels(ctx, who, 1, {{"the result", dvals, 1, n, n, 4}, {"dy", dy, n, D, ldy, (int64_t)sizeof(T)},
                                            {"the table", table, V, D, ldt, (int64_t)sizeof(T)}, {"ids", ids, 1, n, n, (int64_t)sizeof(I)}}));
        if (n == 0) return 0;
        SAMD_TRY(check_blocks(ctx, who, cdiv(n, kWaves)));
        TOK_LAUNCH(ctx, (lookup_dots_kernel<T, I>), cdiv(n, kWaves), kThreads, (hipStream_t)stream, dvals, (const T *)dy, ldy, (const T *)table, ldt, V, D, (const I *)ids, n, scale);
        return 0;
      });
    });
  });
}

int64_t sparse_amd_tokens_lookup_grad_workspace(int type, int64_t n, int64_t V, int64_t D) {
  if (n <= 0 || (n <= kFewIds && V <= kFewTable) || V < 0 || D <= 0) return 0;
  return GradPlan(nullptr, type, n, V, D).bytes;
}

int sparse_amd_tokens_lookup_grad(struct futhark_context *ctx, void *stream, int type, int out_type, int accumulate, void *dtable,
                                  int64_t V, int64_t D, int64_t ldt, const void *dy, int64_t ldy, const void *ids, int id_bits, int64_t n,
                                  const float *vals, float scale, void *work, int64_t work_bytes) {
  return entry(ctx, [&]() -> int {
    const char *who = "lookup_grad";
    if (out_type != type && out_type != SPARSE_AMD_F32)
      return set_error(ctx, "%s: the gradient has the rows' element type or 32 bits", who);
    if (V > 0x7ffffffe || n > 0x7fffffff) return set_error(ctx, "%s: rows and ids are counted in 31 bits", who);
    return by_type(ctx, who, type, [&](auto t) {
      return by_index(ctx, who, id_bits, [&](auto it) -> int {
        typedef typename decltype(t)::type T;
        typedef typename decltype(it)::type I;
        SAMD_TRY(check_panels(ctx, who, 1, {{"the result", dtable, V, D, ldt, type_size(out_type)}, {"dy", dy, n, D, ldy, (int64_t)sizeof(T)},
                                            {"ids", ids, 1, n, n, (int64_t)sizeof(I)}, {"vals", vals, 1, vals ? n : 0, n, 4},
                                            {"the workspace", work, 1, work ? work_bytes : 0, work_bytes, 1}}));
        if (V == 0 || D == 0 || (n == 0 && accumulate)) return 0;
        const hipStream_t s = (hipStream_t)stream;
        GradPlan p(work, type, n, V, D);
        p.g.ldy = ldy;
        p.g.ldE = ldt;
        if (n == 0 || (n <= kFewIds && V <= kFewTable)) {
          if (out_type == type) return sum_few_as<T, T, I>(ctx, s, accumulate != 0, (T *)dtable, (const T *)dy, (const I *)ids, vals, scale, p.g);
          return sum_few_as<T, float, I>(ctx, s, accumulate != 0, (float *)dtable, (const T *)dy, (const I *)ids, vals, scale, p.g);
        }
        SAMD_TRY(check_work(ctx, who, work, work_bytes, p.bytes));
        // it is written before the last of what is read has been
        SAMD_TRY(check_panels(ctx, who, 1, {{"the workspace", work, 1, p.bytes, p.bytes, 1}, {"dy", dy, n, D, ldy, (int64_t)sizeof(T)},
                                            {"ids", ids, 1, n, n, (int64_t)sizeof(I)}, {"vals", vals, 1, vals ? n : 0, n, 4}}));
        if (!accumulate) p.zero(out_type);
        SAMD_TRY(check_blocks(ctx, who, p.sum_blocks()));
        SAMD_TRY(check_blocks(ctx, who, p.join_blocks()));
        SAMD_TRY(order_ids<I>(ctx, s, (const I *)ids, p, !accumulate));
        if (out_type == type) return sum_ids_as<T, T>(ctx, s, accumulate != 0, (T *)dtable, (const T *)dy, vals, scale, p);
        return sum_ids_as<T, float>(ctx, s, accumulate != 0, (float *)dtable, (const T *)dy, vals, scale, p);
      });
    });
  });
}

int64_t sparse_amd_tokens_route_workspace(int64_t n, int64_t X) {
  if (n <= kSelfChoices || X < 1) return 0;
  return (Split(n).groups * (X + 1) * (int64_t)sizeof(int) + 255) & ~(int64_t)255;
}

int sparse_amd_tokens_route(struct futhark_context *ctx, void *stream, const void *chosen, int id_bits, int64_t n, int64_t X, int32_t *pos,
                            int32_t *src, int32_t *offsets, void *work, int64_t work_bytes) {
  return entry(ctx, [&]() -> int {
    const char *who = "route";
    if (X < 1 || X > kMaxExperts) return set_error(ctx, "%s: %lld experts (1 to %d are offered)", who, (long long)X, kMaxExperts);
    if (n > 0x7fffffff) return set_error(ctx, "%s: %lld choices (places have 31 bits)", who, (long long)n);
    return by_index(ctx, who, id_bits, [&](auto it) -> int {
      typedef typename decltype(it)::type I;
      SAMD_TRY(check_panels(ctx, who, 3, {{"pos", pos, 1, n, n, 4}, {"src", src, 1, n, n, 4}, {"offsets", offsets, 1, X + 1, X + 1, 4},
                                          {"chosen", chosen, 1, n, n, (int64_t)sizeof(I)}, {"the workspace", work, 1, work ? work_bytes : 0, work_bytes, 1}}));
      const hipStream_t s = (hipStream_t)stream;
      const int bits = bits_for(X + 1);
      if (n <= 256)
        TOK_LAUNCH(ctx, (route_small_kernel<I, 4, 1>), 1, 256, s, (const I *)chosen, (int)n, (int)X, bits, pos, src, offsets);
      else if (n <= 1024)
        TOK_LAUNCH(ctx, (route_small_kernel<I, 16, 1>), 1, 1024, s, (const I *)chosen, (int)n, (int)X, bits, pos, src, offsets);
      else if (n <= kOneGroupChoices)
        TOK_LAUNCH(ctx, (route_small_kernel<I, 16, 4>), 1, 1024, s, (const I *)chosen, (int)n, (int)X, bits, pos, src, offsets);
      else {
        const int64_t need = sparse_amd_tokens_route_workspace(n, X);
        SAMD_TRY(check_work(ctx, who, work, work_bytes, need));
        SAMD_TRY(check_panels(ctx, who, 1, {{"the workspace", work, 1, need, need, 1}, {"chosen", chosen, 1, n, n, (int64_t)sizeof(I)}}));
        const Split sp(n);
        const Digits<0, I> d = {(const I *)chosen, nullptr, n, X, 0, 0};
        const bool self = n <= kSelfChoices;
        if (!self)
          TOK_LAUNCH(ctx, (digit_count_kernel<0, I>), sp.groups, kSplitThreads, s, d, sp.per_group, (int)X + 1, (int *)work, (uint32_t *)nullptr, (int64_t)0);
        PassOut o = {};
        o.pos = pos; o.src = src; o.offsets = offsets;
        TOK_LAUNCH(ctx, (digit_place_kernel<0, I>), sp.groups, kSplitThreads, s, d, sp.per_group, (int)X + 1, bits, self ? (const int *)nullptr : (const int *)work, o);
      }
      return 0;
    });
  });
}

int sparse_amd_tokens_dispatch(struct futhark_context *ctx, void *stream, int type, void *xs, int64_t ldxs, int64_t slots, const void *x,
                               int64_t ldx, int64_t n, int64_t D, int64_t K, const int32_t *pos, const float *weights) {
  return entry(ctx, [&]() -> int {
    const char *who = "dispatch";
    if (K < 0 || K > 0x7fffffff) return set_error(ctx, "%s: %lld places a row", who, (long long)K);
    return by_type(ctx, who, type, [&](auto t) -> int {
      typedef typename decltype(t)::type T;
      SAMD_TRY(check_panels(ctx, who, 1, {{"the result", xs, slots, D, ldxs, (int64_t)sizeof(T)}, {"x", x, n, D, ldx, (int64_t)sizeof(T)},
                                          {"pos", pos, n, K, K, 4}, {"weights", weights, weights ? n : 0, K, K, 4}}));
      if (n == 0 || D == 0 || K == 0) return 0;
      const hipStream_t s = (hipStream_t)stream;
      const int64_t units = cdiv(D, kPer<T>);
      RowDeal d = deal_rows(n, units, 4);
      const int u = d.lg == 6 && d.waves >= kFullCard ? 4 : 1;
      if (u == 1) d = deal_rows(n, units, 1);
      SAMD_TRY(check_blocks(ctx, who, cdiv(d.waves, kWaves)));
      const auto go = [&](auto kernel) -> int {
        TOK_LAUNCH(ctx, kernel, cdiv(d.waves, kWaves), kThreads, s, (T *)xs, ldxs, (const T *)x, ldx, n, D, (int)K, pos, slots, weights, d.lg, d.segs);
        return 0;
      };
      if (n * K * D * (int64_t)sizeof(T) > kStreamBytes) return u == 4 ? go(dispatch_kernel<T, 4, true>) : go(dispatch_kernel<T, 1, true>);
      return u == 4 ? go(dispatch_kernel<T, 4, false>) : go(dispatch_kernel<T, 1, false>);
    });
  });
}

int sparse_amd_tokens_combine(struct futhark_context *ctx, void *stream, int type, void *y, int64_t ldy, const void *ys, int64_t ldys,
                              int64_t slots, int64_t n, int64_t D, int64_t K, const int32_t *pos, const float *weights) {
  return entry(ctx, [&]() -> int {
    const char *who = "combine";
    if (K < 0 || K > 0x7fffffff) return set_error(ctx, "%s: %lld places a row", who, (long long)K);
    return by_type(ctx, who, type, [&](auto t) -> int {
      typedef typename decltype(t)::type T;
      SAMD_TRY(check_panels(ctx, who, 1, {{"the result", y, n, D, ldy, (int64_t)sizeof(T)}, {"ys", ys, slots, D, ldys, (int64_t)sizeof(T)},
                                          {"pos", pos, n, K, K, 4}, {"weights", weights, weights ? n : 0, K, K, 4}}));
      if (n == 0 || D == 0) return 0;
      const hipStream_t s = (hipStream_t)stream;
      const RowDeal d = deal_rows(n, cdiv(D, kPer<T>), 1);
      SAMD_TRY(check_blocks(ctx, who, cdiv(d.waves, kWaves)));
      const auto go = [&](auto kernel) -> int {
        TOK_LAUNCH(ctx, kernel, cdiv(d.waves, kWaves), kThreads, s, (T *)y, ldy, (const T *)ys, ldys, n, D, (int)K, pos, slots, weights, d.lg, d.segs);
        return 0;
      };
      return n * D * (int64_t)sizeof(T) > kStreamBytes ? go(combine_kernel<T, 1, true>) : go(combine_kernel<T, 1, false>);
    });
  });
}

int sparse_amd_tokens_combine_grad(struct futhark_context *ctx, void *stream, int type, void *dys, int64_t lddys, float *dweights,
                                   const void *dy, int64_t lddy, const void *ys, int64_t ldys, int64_t slots, int64_t n, int64_t D,
                                   int64_t K, const int32_t *pos, const float *weights) {
  return entry(ctx, [&]() -> int {
    const char *who = "combine_grad";
    if (K < 0 || K > 0x7fffffff) return set_error(ctx, "%s: %lld places a row", who, (long long)K);
    return by_type(ctx, who, type, [&](auto t) -> int {
      typedef typename decltype(t)::type T;
      SAMD_TRY(check_panels(ctx, who, 2, {{"dys", dys, slots, D, lddys, (int64_t)sizeof(T)}, {"dweights", dweights, n, K, K, 4},
                                          {"dy", dy, n, D, lddy, (int64_t)sizeof(T)}, {"ys", ys, slots, D, ldys, (int64_t)sizeof(T)},
                                          {"pos", pos, n, K, K, 4}, {"weights", weights, n, K, K, 4}}));
      if (n == 0 || K == 0) return 0;
      SAMD_TRY(check_blocks(ctx, who, n));
      const auto go = [&](auto waves, auto at_once) -> int {
        constexpr int W = decltype(waves)::value, J = decltype(at_once)::value;
        const auto kernel = n * K * D * (int64_t)sizeof(T) > kStreamBytes ? combine_grad_kernel<T, W, J, true> : combine_grad_kernel<T, W, J, false>;
        TOK_LAUNCH(ctx, kernel, W == 1 ? cdiv(n, kWaves) : n, kThreads, (hipStream_t)stream, (T *)dys, lddys, dweights, (const T *)dy, lddy, (const T *)ys, ldys, n, D, (int)K, pos, slots, weights);
        return 0;
      };
      const auto choose = [&](auto waves) -> int {
        return K <= 2 ? go(waves, std::integral_constant<int, 2>()) : K <= 4 ? go(waves, std::integral_constant<int, 4>()) : go(waves, std::integral_constant<int, 8>());
      };
      // choices that are not there cost their share of sums, registers and waiting: 8863 tokens of 1728 bf16, 1 place each, 8 at
      // once 50 us, 2 at once 21.  A wave to itself where a row is two rounds of it at most: 16384 tokens of 256, 4 places each,
      // a workgroup 106 us, a wave 31; of 2048, 8 places each, 212 and 293.
      return cdiv(D, kPer<T>) <= 2 * kWave ? choose(std::integral_constant<int, 1>()) : choose(std::integral_constant<int, kWaves>());
    });
  });
}

int sparse_amd_tokens_experts(struct futhark_context *ctx, void *stream, int type, void *ys, int64_t ldy, const void *xs, int64_t ldx,
                              int64_t rows, const void *w, int64_t X, int64_t F, int64_t D, int64_t ldw, int64_t blockw,
                              const int32_t *offsets) {
  return entry(ctx, [&]() -> int {
    const char *who = "experts";
    SAMD_TRY(check_experts(ctx, who, rows, X, F, D, offsets));
    return by_type16(ctx, who, type, [&](auto t) -> int {
      typedef typename decltype(t)::type T;
      SAMD_TRY(check_panels(ctx, who, 1, {{"the result", ys, rows, F, ldy, 2}, {"xs", xs, rows, D, ldx, 2},
                                          {"w", w, X, block_span(F, D, ldw), X > 1 ? blockw : block_span(F, D, ldw), 2}, {"a block of w", w, F, D, ldw, 2},
                                          {"offsets", offsets, 1, X + 1, X + 1, 4}}));
      if (rows == 0 || F == 0) return 0;
      ProductShape g = {};
      g.rows = rows; g.N = F; g.K = D; g.ldA = ldx; g.ldB = ldw; g.ldC = ldy; g.blockB = blockw; g.X = (int)X;
      g.stream = rows * F * 2 > kStreamBytes;
      return experts_panels<T, kForward>(ctx, who, (hipStream_t)stream, (T *)ys, (const T *)xs, (const T *)w, offsets, g);
    });
  });
}

int sparse_amd_tokens_experts_grad_x(struct futhark_context *ctx, void *stream, int type, void *dxs, int64_t ldx, const void *dys,
                                     int64_t ldy, int64_t rows, const void *w, int64_t X, int64_t F, int64_t D, int64_t ldw,
                                     int64_t blockw, const int32_t *offsets) {
  return entry(ctx, [&]() -> int {
    const char *who = "experts_grad_x";
    SAMD_TRY(check_experts(ctx, who, rows, X, F, D, offsets));
    return by_type16(ctx, who, type, [&](auto t) -> int {
      typedef typename decltype(t)::type T;
      SAMD_TRY(check_panels(ctx, who, 1, {{"the result", dxs, rows, D, ldx, 2}, {"dys", dys, rows, F, ldy, 2},
                                          {"w", w, X, block_span(F, D, ldw), X > 1 ? blockw : block_span(F, D, ldw), 2}, {"a block of w", w, F, D, ldw, 2},
                                          {"offsets", offsets, 1, X + 1, X + 1, 4}}));
      if (rows == 0 || D == 0) return 0;
      ProductShape g = {};
      g.rows = rows; g.N = D; g.K = F; g.ldA = ldy; g.ldB = ldw; g.ldC = ldx; g.blockB = blockw; g.X = (int)X;
      g.stream = rows * D * 2 > kStreamBytes;
      return experts_panels<T, kGradX>(ctx, who, (hipStream_t)stream, (T *)dxs, (const T *)dys, (const T *)w, offsets, g);
    });
  });
}

int sparse_amd_tokens_experts_grad_w(struct futhark_context *ctx, void *stream, int type, int out_type, int accumulate, void *dw,
                                     int64_t X, int64_t F, int64_t D, int64_t ldw, int64_t blockw, const void *dys, int64_t ldy,
                                     const void *xs, int64_t ldx, int64_t rows, const int32_t *offsets) {
  return entry(ctx, [&]() -> int {
    const char *who = "experts_grad_w";
    SAMD_TRY(check_experts(ctx, who, rows, X, F, D, offsets));
    if (out_type != type && out_type != SPARSE_AMD_F32)
      return set_error(ctx, "%s: the gradient has the rows' element type or 32 bits", who);
    return by_type16(ctx, who, type, [&](auto t) -> int {
      typedef typename decltype(t)::type T;
      if (X > 1 && blockw < block_span(F, D, ldw)) return set_error(ctx, "%s: the blocks of dw overlap", who);
      SAMD_TRY(check_panels(ctx, who, 1, {{"the result", dw, X, block_span(F, D, ldw), X > 1 ? blockw : block_span(F, D, ldw), type_size(out_type)},
                                          {"dys", dys, rows, F, ldy, 2}, {"xs", xs, rows, D, ldx, 2}, {"offsets", offsets, 1, X + 1, X + 1, 4}}));
      SAMD_TRY(check_panels(ctx, who, 1, {{"a block of the result", dw, F, D, ldw, type_size(out_type)}}));
      if (F == 0 || D == 0) return 0;
      ProductShape g = {};
      g.rows = rows; g.M = F; g.N = D; g.ldA = ldy; g.ldB = ldx; g.ldC = ldw; g.blockC = blockw; g.X = (int)X;
      g.stream = X * F * D * 2 > kStreamBytes;
      const hipStream_t s = (hipStream_t)stream;
      if (out_type == type)
        return accumulate ? experts_weights<T, T, true>(ctx, who, s, (T *)dw, (const T *)dys, (const T *)xs, offsets, g)
                          : experts_weights<T, T, false>(ctx, who, s, (T *)dw, (const T *)dys, (const T *)xs, offsets, g);
      return accumulate ? experts_weights<T, float, true>(ctx, who, s, (float *)dw, (const T *)dys, (const T *)xs, offsets, g)
                        : experts_weights<T, float, false>(ctx, who, s, (float *)dw, (const T *)dys, (const T *)xs, offsets, g);
    });
  });
}

}  // extern "C"
