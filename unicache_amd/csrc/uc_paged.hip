// Pages of the paged KV cache: handing them out, sharing, copying, thinning out and taking them back.
//
// All of it happens on the device, so that a captured graph can grow, fork and cut sequences.  What the
// calls do is a function of the tables and lengths alone: free pages go out lowest first, to the
// sequences in order, found by prefix sums over a bit for each page; reference counts and bits move by
// atomics whose order does not matter (a count's zero is seen by the one that makes it).
//
// Copies (the rows of open pages; the kept rows of thinned sequences) are bound by HBM (the latter 5.4 TB/s over 244 MB of
// reads and writes), the rest by latency: chains of short launches over a few kilobytes (reserve 2.3 us, a small
// reorder 11, count, give, list and commit of thinning 5 to 9 each).
#include "uc_paged.h"

namespace uc {
namespace pg {

int check_cache(const uc_paged_cache *c, int64_t layer, const char *what, Cache &out) {
  UC_REQUIRE(c != nullptr, "%s: cache is NULL", what);
  UC_REQUIRE(half_dtype(c->dtype), "%s: the cache must be bf16 or fp16", what);
  UC_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim must be 64 or 128", what);
  const int32_t b = c->page_tokens;
  UC_REQUIRE(b == 16 || b == 32 || b == 64 || b == 128 || b == 256, "%s: pages must have 16, 32, 64, 128 or 256 tokens", what);
  UC_REQUIRE(c->sequences > 0 && c->sequences <= kMostSequences, "%s: bad number of sequences", what);
  UC_REQUIRE(c->layers > 0 && c->layers < (1 << 20) && layer >= 0 && layer < c->layers, "%s: bad layer", what);
  UC_REQUIRE(c->pages > 0 && c->pages < (int64_t(1) << 30), "%s: bad number of pages", what);
  UC_REQUIRE(c->sequence_pages > 0 && c->sequence_pages <= (int64_t(1) << 30) / b, "%s: bad number of pages per sequence", what);
  UC_REQUIRE(c->sequences * c->sequence_pages < (int64_t(1) << 30), "%s: the table is too large", what);
  UC_REQUIRE(c->heads_kv > 0 && c->heads_kv < (1 << 24) && c->heads_kv * b * c->head_dim < (int64_t(1) << 30),
             "%s: bad number of KV heads", what);
  UC_REQUIRE(c->layers * c->pages < (int64_t(1) << 60) / (c->heads_kv * b * c->head_dim), "%s: the pool is too large", what);
  auto aligned = [](const void *p, uintptr_t n) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  UC_REQUIRE(aligned(c->key, 16) && aligned(c->value, 16), "%s: keys and values must be 16-byte aligned", what);
  UC_REQUIRE(aligned(c->table, 4) && aligned(c->lengths, 4), "%s: table and lengths must be 4-byte aligned", what);
  const bool none = c->granted == nullptr && c->references == nullptr && c->free_pages == nullptr;
  UC_REQUIRE(none || (aligned(c->granted, 4) && aligned(c->references, 4) && aligned(c->free_pages, 4)),
             "%s: granted, references and free_pages belong together", what);
  out.page = b;
  out.shift = __builtin_ctz(static_cast<uint32_t>(b));
  out.sequences = static_cast<int32_t>(c->sequences);
  out.width = static_cast<int32_t>(c->sequence_pages);
  out.pages = static_cast<int32_t>(c->pages);
  out.heads = static_cast<int32_t>(c->heads_kv);
  out.page_elems = static_cast<int32_t>(c->heads_kv * b * c->head_dim);
  out.layer_elems = int64_t(out.page_elems) * c->pages;
  out.table = c->table;
  out.lengths = c->lengths;
  out.key = static_cast<uint16_t *>(c->key) + layer * out.layer_elems;
  out.value = static_cast<uint16_t *>(c->value) + layer * out.layer_elems;
  return UC_OK;
}

namespace {

constexpr int kThreads = 1024;  // of the workgroup that hands out pages
constexpr int kListed = 8192;   // pages that it hands out at a time

struct Pool {
  int32_t *granted, *references;
  uint32_t *free;
};

// What atomics of this launch may have changed, past the CU's own cache.
template <class T>
__device__ __forceinline__ T fresh(const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Inclusive prefix sum over a workgroup of 1024, and its total.
__device__ __forceinline__ int32_t block_prefix(int32_t v, int32_t &total, int32_t *waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int32_t u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  __syncthreads();  // what stood in `waves` has been read
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) v += waves[w];
    total += waves[w];
  }
  return v;
}

struct Giver {
  int32_t waves[kThreads / 64];
  int32_t list[kListed];
};

__device__ __forceinline__ uint32_t free_word(const Pool &pool, int32_t pages, int32_t w) {
  if (w >= (pages + 31) / 32) return 0;
  const int32_t tail = pages - 32 * w;  // pages of this word
  return fresh(pool.free + w) & (tail >= 32 ? ~0u : (1u << tail) - 1u);
}

// Free pages, up to `want`, counted by a whole workgroup.
__device__ int32_t count_free(const Pool &pool, int32_t pages, int32_t want, Giver &g) {
  int32_t found = 0;
  for (int32_t w0 = 0; w0 < (pages + 31) / 32 && found < want; w0 += kThreads) {
    int32_t total;
    block_prefix(__popc(free_word(pool, pages, w0 + threadIdx.x)), total, g.waves);
    found += total;
  }
  return found < want ? found : want;
}

// Take the `want` lowest free pages: assign(rank, page) for each, by a whole workgroup.  Returns how many there were.
template <class F>
__device__ int32_t give_pages(const Pool &pool, int32_t pages, int32_t want, Giver &g, F assign) {
  int32_t found = 0;
  for (int32_t w0 = 0; w0 < (pages + 31) / 32 && found < want; w0 += kThreads) {
    const int32_t w = w0 + threadIdx.x;
    const uint32_t word = free_word(pool, pages, w);
    int32_t total;
    const int32_t count = __popc(word), first = found + block_prefix(count, total, g.waves) - count;
    const int32_t end = found + total < want ? found + total : want;
    if (count > 0 && first < end) {
      uint32_t rest = word;
      for (int32_t r = first; rest != 0 && r < end; ++r) rest &= rest - 1;
      pool.free[w] = rest;
    }
    for (int32_t base = found; base < end; base += kListed) {
      __syncthreads();
      uint32_t rest = word;
      for (int32_t r = first; rest != 0 && r < end && r < base + kListed; ++r) {
        if (r >= base) g.list[r - base] = 32 * w + __ffs(rest) - 1;
        rest &= rest - 1;
      }
      __syncthreads();
      for (int32_t r = base + threadIdx.x; r < end && r < base + kListed; r += kThreads) assign(r, g.list[r - base]);
    }
    found = end;
  }
  __syncthreads();
  return found;
}

// The last sequence s with first[s] <= rank: the one that page goes to (sequences that take none share their first).
__device__ __forceinline__ int32_t taker(const int32_t *first, int32_t n, int32_t rank) {
  int32_t lo = 0, hi = n - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) / 2;
    if (first[mid] <= rank) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// One page of a sequence's table is released.
__device__ __forceinline__ void release(const Pool &pool, int32_t page) {
  if (atomicSub(pool.references + page, 1) == 1) atomicOr(pool.free + page / 32, 1u << (page % 32));
}

// ---------------------------------------------------------------- reserve --
__global__ __launch_bounds__(kThreads) void reserve_kernel(Cache c, Pool pool, int32_t tokens, const int32_t *counts) {
  __shared__ Giver g;
  extern __shared__ int32_t first[];  // [S] the first page's rank
  auto wanted = [&](int32_t s, int32_t length) {  // tokens, within the table
    int32_t n = counts != nullptr ? counts[s] : tokens;
    n = n < 0 ? 0 : n > tokens ? tokens : n;
    return n < c.capacity() - length ? n : c.capacity() - length;
  };
  int32_t want = 0;
  for (int32_t s0 = 0; s0 < c.sequences; s0 += kThreads) {
    const int32_t s = s0 + threadIdx.x;
    int32_t need = 0, total;
    if (s < c.sequences) {
      const int32_t length = c.length(s);
      need = c.pages_of(length + wanted(s, length)) - c.pages_of(length);
    }
    const int32_t sum = block_prefix(need, total, g.waves);
    if (s < c.sequences) first[s] = want + sum - need;
    want += total;
  }
  __syncthreads();
  const int32_t found = give_pages(pool, c.pages, want, g, [&](int32_t rank, int32_t page) {
    const int32_t s = taker(first, c.sequences, rank);
    c.table[int64_t(s) * c.width + c.pages_of(c.length(s)) + rank - first[s]] = page;
    pool.references[page] = 1;
  });
  for (int32_t s = threadIdx.x; s < c.sequences; s += kThreads) {
    const int32_t length = c.length(s), n = wanted(s, length), held = c.pages_of(length);
    int32_t got = found - first[s];
    got = got < 0 ? 0 : got;
    const int64_t room = (int64_t(held) + got) * c.page - length;
    const int32_t granted = n < room ? n : static_cast<int32_t>(room);
    pool.granted[s] = granted;
    c.lengths[s] = length + granted;
  }
}

// ---------------------------------------------------------------- reorder --
struct Order {
  const int32_t *parents, *cut;
  int32_t *old_table;            // [S, M]
  int32_t *before, *length;      // [S] pages held before; tokens held now
  int32_t *source, *target;      // [S] the open page's copy; target -1: none
  int32_t *owner, *opens;        // [P] of pages that are some sequence's open page: the lowest such sequence, their number
};

__device__ __forceinline__ int32_t parent_of(const Cache &c, const Order &o, int32_t s) {
  const int32_t p = o.parents != nullptr ? o.parents[s] : s;
  return p < 0 || p >= c.sequences ? -1 : p;
}

// A sequence before and after.
struct Change {
  int32_t parent, before, after;  // pages
  int32_t now;                    // tokens
};

__device__ __forceinline__ Change change_of(const Cache &c, const Order &o, int32_t s) {
  Change x;
  x.parent = parent_of(c, o, s);
  x.before = c.pages_of(c.length(s));
  x.now = x.parent < 0 ? 0 : c.length(x.parent);
  if (o.cut != nullptr) {
    const int32_t cut = o.cut[s] < 0 ? 0 : o.cut[s];
    x.now = x.now < cut ? x.now : cut;
  }
  x.after = c.pages_of(x.now);
  return x;
}

// Entry i of a sequence, which it may hold no more, is released (i from 0 on, one at least).
__device__ __forceinline__ void release_entry(const Cache &c, const Pool &pool, const Order &o, int32_t s, int32_t i,
                                              const Change &x) {
  const int64_t at = int64_t(s) * c.width + i;
  if (i == 0) {
    o.before[s] = x.before;
    o.length[s] = x.now;
    o.target[s] = -1;
  }
  if (i < x.before) {
    const int32_t entry = c.table[at];
    o.old_table[at] = entry;
    if (c.is_page(entry) && !(x.parent == s && i < x.after)) release(pool, entry);
  }
  if (i == x.after - 1 && (x.now & (c.page - 1)) != 0) {
    const int32_t open = c.table[int64_t(x.parent) * c.width + i];
    if (c.is_page(open)) {
      o.owner[open] = c.sequences;
      o.opens[open] = 0;
    }
  }
}

// And what it holds now, held.
__device__ __forceinline__ void hold_entry(const Cache &c, const Pool &pool, const Order &o, int32_t s, int32_t i, int32_t p,
                                           int32_t before, int32_t now) {
  const int64_t at = int64_t(s) * c.width + i;
  const int32_t after = c.pages_of(now);
  if (i >= after) {
    if (i < before) c.table[at] = -1;
    return;
  }
  const int32_t entry = o.old_table[int64_t(p) * c.width + i];
  if (p != s) {
    c.table[at] = entry;
    if (c.is_page(entry) && atomicAdd(pool.references + entry, 1) == 0) {
      atomicAnd(pool.free + entry / 32, ~(1u << (entry % 32)));
    }
  }
  if (i == after - 1 && (now & (c.page - 1)) != 0 && c.is_page(entry)) {
    atomicMin(o.owner + entry, s);
    atomicAdd(o.opens + entry, 1);
  }
}

// Pages for the copies of open pages, and the new lengths.  One workgroup; first: [S] in LDS.
__device__ __forceinline__ void open_pages(const Cache &c, const Pool &pool, const Order &o, Giver &g, int32_t *first) {
  int32_t want = 0;
  for (int32_t s0 = 0; s0 < c.sequences; s0 += kThreads) {
    const int32_t s = s0 + threadIdx.x;
    int32_t need = 0, total;
    if (s < c.sequences) {
      const int32_t now = o.length[s];
      if ((now & (c.page - 1)) != 0) {
        const int32_t open = c.table[int64_t(s) * c.width + c.pages_of(now) - 1];
        // another sequence's, or held whole by one
        need = c.is_page(open) && (fresh(o.owner + open) != s || fresh(pool.references + open) != fresh(o.opens + open));
        o.source[s] = open;
      }
    }
    const int32_t sum = block_prefix(need, total, g.waves);
    if (s < c.sequences) first[s] = want + sum - need;
    want += total;
  }
  __syncthreads();
  auto copies = [&](int32_t s) { return first[s] != (s + 1 < c.sequences ? first[s + 1] : want); };
  const int32_t found = give_pages(pool, c.pages, want, g, [&](int32_t rank, int32_t page) {
    const int32_t s = taker(first, c.sequences, rank);
    o.target[s] = page;
    pool.references[page] = 1;
  });
  for (int32_t s = threadIdx.x; s < c.sequences; s += kThreads) {
    int32_t now = o.length[s];
    if (copies(s)) {
      const int64_t at = int64_t(s) * c.width + c.pages_of(now) - 1;
      const bool got = first[s] < found;
      atomicSub(pool.references + o.source[s], 1);
      c.table[at] = got ? o.target[s] : -1;
      if (!got) now &= ~(c.page - 1);
    }
    c.lengths[s] = now;
  }
}

// A row of workgroups a sequence, a thread an entry.
__global__ __launch_bounds__(256) void reorder_release_kernel(Cache c, Pool pool, Order o) {
  const int32_t s = blockIdx.y;
  const Change x = change_of(c, o, s);
  const int32_t end = x.before > x.after ? x.before : x.after;
  for (int32_t i = blockIdx.x * 256 + threadIdx.x; i < end || i == 0; i += gridDim.x * 256) release_entry(c, pool, o, s, i, x);
}

__global__ __launch_bounds__(256) void reorder_hold_kernel(Cache c, Pool pool, Order o) {
  const int32_t s = blockIdx.y, p = parent_of(c, o, s), before = o.before[s], now = o.length[s], after = c.pages_of(now);
  const int32_t end = before > after ? before : after;
  for (int32_t i = blockIdx.x * 256 + threadIdx.x; i < end; i += gridDim.x * 256) hold_entry(c, pool, o, s, i, p, before, now);
}

__global__ __launch_bounds__(kThreads) void reorder_open_kernel(Cache c, Pool pool, Order o) {
  __shared__ Giver g;
  extern __shared__ int32_t first[];
  open_pages(c, pool, o, g, first);
}

// All of it by one workgroup, for few entries a thread (8 sequences forked three times: 23.0 -> 20.5 us a call).
__global__ __launch_bounds__(kThreads) void reorder_small_kernel(Cache c, Pool pool, Order o) {
  __shared__ Giver g;
  __shared__ int32_t widest;
  extern __shared__ int32_t first[];
  if (threadIdx.x == 0) widest = 1;
  __syncthreads();
  for (int32_t s = threadIdx.x; s < c.sequences; s += kThreads) {
    const Change x = change_of(c, o, s);
    atomicMax(&widest, x.before > x.after ? x.before : x.after);
  }
  __syncthreads();
  const int64_t entries = int64_t(c.sequences) * widest;
  for (int64_t at = threadIdx.x; at < entries; at += kThreads) {
    const int32_t s = static_cast<int32_t>(at / widest);
    release_entry(c, pool, o, s, static_cast<int32_t>(at - int64_t(s) * widest), change_of(c, o, s));
  }
  __syncthreads();  // (one workgroup's accesses, and its atomics' in L2: no fence of a wider scope is needed)
  for (int64_t at = threadIdx.x; at < entries; at += kThreads) {
    const int32_t s = static_cast<int32_t>(at / widest);
    hold_entry(c, pool, o, s, static_cast<int32_t>(at - int64_t(s) * widest), parent_of(c, o, s), o.before[s], o.length[s]);
  }
  __syncthreads();
  open_pages(c, pool, o, g, first);
}

constexpr int64_t kSmallTable = 4 * kThreads;

// The rows of open pages into their copies: a workgroup a (sequence, layer and head).
__global__ __launch_bounds__(256) void reorder_copy_kernel(Cache c, Order o, int32_t row_bytes) {
  const int32_t s = blockIdx.y, target = o.target[s];
  if (target < 0) return;
  const int32_t layer = blockIdx.x / c.heads, head = blockIdx.x - layer * c.heads;
  const int32_t rows = o.length[s] & (c.page - 1), units = rows * (row_bytes / 16);
  const int64_t base = layer * c.layer_elems + int64_t(head) * c.page * (row_bytes / 2);
  const int64_t from = base + int64_t(o.source[s]) * c.page_elems, to = base + int64_t(target) * c.page_elems;
  for (int32_t i = threadIdx.x; i < units; i += 256) {
    const uint4 k = reinterpret_cast<const uint4 *>(c.key + from)[i], v = reinterpret_cast<const uint4 *>(c.value + from)[i];
    reinterpret_cast<uint4 *>(c.key + to)[i] = k;
    reinterpret_cast<uint4 *>(c.value + to)[i] = v;
  }
}

// ---------------------------------------------------------------- compact --
struct Thin {
  const uint8_t *keep;
  int64_t stride;
  int32_t tokens;
  int32_t *source;           // [P, page] of each page to come, in order: the tokens that move there
  int32_t *page;             // [P] the page
  int32_t *moves;            // [P] its sequence and place in that
  int32_t *first;            // [S] the first of a sequence's
  int32_t *length;           // [S] tokens before
  int32_t *kept, *whole;     // [S] tokens that stay; leading pages that do
  int32_t *count;            // [1] pages to come
};

// Eight tokens of sequence s, whose mask starts at keep: a bit for each that stays.  Tokens without a page (one holds all eight)
// do not: they have no rows to move, and a new page would show what it held before in their place.
__device__ __forceinline__ uint32_t stays_of(const Cache &c, const Thin &t, const uint8_t *keep, int32_t s, int32_t token,
                                             int32_t length) {
  uint32_t stays = 0;
  const bool held = c.is_page(c.table[int64_t(s) * c.width + (token >> c.shift)]);
  if (token + 8 <= length && token + 8 <= t.tokens && (reinterpret_cast<uintptr_t>(keep + token) & 7) == 0) {
    const uint2 w = *reinterpret_cast<const uint2 *>(keep + token);
#pragma unroll
    for (int i = 0; i < 8; ++i) stays |= (((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu) != 0 ? 1u << i : 0u;
    return held ? stays : 0;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int32_t at = token + i;
    if (at < length && (at >= t.tokens || keep[at] != 0)) stays |= 1u << i;
  }
  return held ? stays : 0;
}

// How many tokens a sequence keeps, and how many of its pages come before the first that loses one.
__global__ __launch_bounds__(kThreads) void thin_count_kernel(Cache c, Thin t) {
  __shared__ int32_t lost, kept;
  const int32_t s = blockIdx.x, length = c.length(s);
  const uint8_t *keep = t.keep + s * t.stride;
  if (threadIdx.x == 0) {
    lost = length;
    kept = 0;
  }
  __syncthreads();
  int32_t mine = 0, first = length;
  for (int32_t token = 8 * threadIdx.x; token < length; token += 8 * kThreads) {
    const uint32_t stays = stays_of(c, t, keep, s, token, length);
    const int32_t there = length - token >= 8 ? 8 : length - token;
    const uint32_t gone = ~stays & ((1u << there) - 1u);
    mine += __popc(stays);
    if (gone != 0 && first == length) first = token + __ffs(gone) - 1;
  }
  if (mine != 0) atomicAdd(&kept, mine);
  if (first != length) atomicMin(&lost, first);
  __syncthreads();
  if (threadIdx.x == 0) {
    t.length[s] = length;
    t.kept[s] = kept;
    t.whole[s] = lost < length ? lost >> c.shift : c.pages_of(length);
  }
}

// The tokens that move, page by page.
__global__ __launch_bounds__(kThreads) void thin_list_kernel(Cache c, Thin t) {
  __shared__ int32_t waves[kThreads / 64];
  const int32_t s = blockIdx.x, length = t.length[s], stay = t.whole[s] << c.shift;
  if (t.kept[s] <= stay) return;  // (also where nothing is lost)
  const uint8_t *keep = t.keep + s * t.stride;
  int32_t *source = t.source + (int64_t(t.first[s]) << c.shift) - stay;
  // (every token of the pages that stay is kept, so the count begins behind them)
  for (int32_t t0 = stay, kept = stay; t0 < length; t0 += 8 * kThreads) {
    const int32_t token = t0 + 8 * threadIdx.x;
    const uint32_t stays = token < length ? stays_of(c, t, keep, s, token, length) : 0;
    int32_t total;
    const int32_t count = __popc(stays);
    int32_t to = kept + block_prefix(count, total, waves) - count;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (stays & (1u << i)) source[to++] = token + i;
    }
    kept += total;
  }
}

// Pages to come.  One workgroup.
__global__ __launch_bounds__(kThreads) void thin_give_kernel(Cache c, Pool pool, Thin t) {
  __shared__ Giver g;
  extern __shared__ int32_t first[];  // [S]
  int32_t want = 0;
  auto need_of = [&](int32_t s) {
    const int32_t need = c.pages_of(t.kept[s]) - t.whole[s];
    return need < 0 ? 0 : need;
  };
  for (int32_t s0 = 0; s0 < c.sequences; s0 += kThreads) {
    const int32_t s = s0 + threadIdx.x;
    const int32_t need = s < c.sequences ? need_of(s) : 0;
    int32_t total;
    const int32_t sum = block_prefix(need, total, g.waves);
    if (s < c.sequences) first[s] = want + sum - need;
    want += total;
  }
  __syncthreads();
  const int32_t found = count_free(pool, c.pages, want, g);
  if (found < want) {  // some sequences stay as they are
    __shared__ int32_t most;
    if (threadIdx.x == 0) most = 0;
    __syncthreads();
    for (int32_t s = threadIdx.x; s < c.sequences; s += kThreads) {
      const int32_t need = need_of(s);
      if (first[s] + need <= found) {
        atomicMax(&most, first[s] + need);
      } else {
        t.kept[s] = t.length[s];
        t.whole[s] = c.pages_of(t.length[s]);
      }
    }
    __syncthreads();
    want = most;
  }
  give_pages(pool, c.pages, want, g, [&](int32_t rank, int32_t page) {
    const int32_t s = taker(first, c.sequences, rank);
    t.page[rank] = page;
    t.moves[rank] = s * c.width + t.whole[s] + rank - first[s];
    pool.references[page] = 1;
  });
  for (int32_t s = threadIdx.x; s < c.sequences; s += kThreads) t.first[s] = first[s];
  if (threadIdx.x == 0) *t.count = want;
}

// The kept rows into the pages to come: a workgroup takes one (page, layer and head) after another.
__global__ __launch_bounds__(256) void thin_copy_kernel(Cache c, Thin t, int32_t layers, int32_t chunks) {
  const int64_t parts = int64_t(layers) * c.heads, jobs = *t.count * parts;
  const int32_t elems = chunks * 8;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int32_t rank = static_cast<int32_t>(job / parts), at = t.moves[rank], part = static_cast<int32_t>(job % parts);
    const int32_t s = at / c.width, i = at - s * c.width, layer = part / c.heads, head = part - layer * c.heads;
    const int32_t first = i << c.shift, left = t.kept[s] - first, rows = left < c.page ? left : c.page;
    const int32_t *source = t.source + (int64_t(rank) << c.shift);
    const int64_t base = layer * c.layer_elems + int64_t(head) * c.page * elems;
    const int64_t to = base + int64_t(t.page[rank]) * c.page_elems;
    for (int32_t u = threadIdx.x; u < rows * chunks; u += 256) {
      const int32_t row = u / chunks, x = (u - row * chunks) * 8, token = source[row];
      const int32_t page = c.table[int64_t(s) * c.width + (token >> c.shift)];
      if (!c.is_page(page)) continue;
      const int64_t from = base + int64_t(page) * c.page_elems + (token & (c.page - 1)) * elems + x;
      const uint4 k = *reinterpret_cast<const uint4 *>(c.key + from), v = *reinterpret_cast<const uint4 *>(c.value + from);
      *reinterpret_cast<uint4 *>(c.key + to + row * elems + x) = k;
      *reinterpret_cast<uint4 *>(c.value + to + row * elems + x) = v;
    }
  }
}

// The pages left behind are released, and the new ones take their place.  A row of workgroups a sequence.
__global__ __launch_bounds__(256) void thin_commit_kernel(Cache c, Pool pool, Thin t) {
  const int32_t s = blockIdx.y, kept = t.kept[s], held = c.pages_of(t.length[s]), whole = t.whole[s], first = t.first[s];
  if (blockIdx.x == 0 && threadIdx.x == 0) c.lengths[s] = kept;
  for (int32_t i = whole + blockIdx.x * 256 + threadIdx.x; i < held; i += gridDim.x * 256) {
    const int64_t at = int64_t(s) * c.width + i;
    const int32_t entry = c.table[at];
    if (c.is_page(entry)) release(pool, entry);
    c.table[at] = i < c.pages_of(kept) ? t.page[first + i - whole] : -1;
  }
}

// ------------------------------------------------------------------ dense --
__global__ __launch_bounds__(256) void dense_kernel(Cache c, uint16_t *key, uint16_t *value, int32_t tokens, int32_t chunks) {
  const int32_t units = c.heads * chunks, s = blockIdx.y, elems = chunks * 8;
  const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= int64_t(tokens) * units) return;
  const int32_t token = static_cast<int32_t>(at / units), unit = static_cast<int32_t>(at - int64_t(token) * units);
  const int32_t head = unit / chunks, x = (unit - head * chunks) * 8;
  uint4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
  if (token < c.length(s)) {
    const int32_t page = c.table[int64_t(s) * c.width + (token >> c.shift)];
    if (c.is_page(page)) {
      const int64_t from = int64_t(page) * c.page_elems + ((head << c.shift) + (token & (c.page - 1))) * elems + x;
      k = *reinterpret_cast<const uint4 *>(c.key + from);
      v = *reinterpret_cast<const uint4 *>(c.value + from);
    }
  }
  const int64_t to = (int64_t(s) * tokens * units + at) * 8;
  *reinterpret_cast<uint4 *>(key + to) = k;
  *reinterpret_cast<uint4 *>(value + to) = v;
}

int check_pool(const uc_paged_cache *cache, const char *what, Cache &c, Pool &pool) {
  if (int rc = check_cache(cache, 0, what, c)) return rc;
  UC_REQUIRE(cache->references != nullptr, "%s: the cache has no references and free pages", what);
  pool = Pool{cache->granted, cache->references, cache->free_pages};
  return UC_OK;
}

int64_t pages_expected(const Cache &c, int64_t max_tokens) {
  const int64_t n = ceil_div(max_tokens < c.capacity() ? max_tokens : int64_t(c.capacity()), int64_t(c.page));
  return n > 0 ? n : 1;
}

// Workgroups for the entries of each sequence: 16 of them at most, which then take more than one entry a thread.
dim3 entry_groups(const Cache &c, int64_t widest) {
  const int64_t n = ceil_div(widest, int64_t(256));
  return dim3(static_cast<uint32_t>(n < 16 ? n : 16), c.sequences);
}

size_t first_bytes(const Cache &c) { return static_cast<size_t>(c.sequences) * sizeof(int32_t); }

// Workspaces in int32 words, every part on 16 bytes.
struct Parts {
  int64_t words = 0;
  int64_t take(int64_t n) {
    const int64_t at = words;
    words += (n + 3) / 4 * 4;
    return at;
  }
};

int64_t lay_out(const Cache &c, int32_t *base, Order &o) {
  Parts p;
  const int64_t s = c.sequences;
  o.old_table = base + p.take(s * c.width);
  o.before = base + p.take(s);
  o.length = base + p.take(s);
  o.source = base + p.take(s);
  o.target = base + p.take(s);
  o.owner = base + p.take(c.pages);
  o.opens = base + p.take(c.pages);
  return p.words * 4;
}

int64_t lay_out(const Cache &c, int32_t *base, Thin &t) {
  Parts p;
  const int64_t s = c.sequences;
  t.source = base + p.take(int64_t(c.pages) * c.page);
  t.page = base + p.take(c.pages);
  t.moves = base + p.take(c.pages);
  t.first = base + p.take(s);
  t.kept = base + p.take(s);
  t.whole = base + p.take(s);
  t.count = base + p.take(1);
  t.length = base + p.take(s);
  return p.words * 4;
}

}  // namespace
}  // namespace pg
}  // namespace uc

extern "C" int uc_paged_dense(const uc_paged_cache *cache, int64_t layer, void *out_key, void *out_value, int64_t tokens,
                              uc_stream_t stream) {
  using namespace uc;
  using namespace uc::pg;
  const char *what = "uc_paged_dense";
  Cache c;
  if (int rc = check_cache(cache, layer, what, c)) return rc;
  UC_REQUIRE(tokens >= 0 && tokens <= c.capacity(), "%s: bad number of tokens", what);
  if (tokens == 0) return UC_OK;
  UC_REQUIRE(out_key != nullptr && out_value != nullptr &&
                 ((reinterpret_cast<uintptr_t>(out_key) | reinterpret_cast<uintptr_t>(out_value)) & 15) == 0,
             "%s: out must be 16-byte aligned", what);
  const int32_t chunks = static_cast<int32_t>(cache->head_dim / 8);
  const int64_t groups = ceil_div(tokens * c.heads * chunks, int64_t(256));
  UC_REQUIRE(groups * c.sequences < (1 << 24), "%s: too many rows", what);
  hipLaunchKernelGGL(dense_kernel, dim3(static_cast<uint32_t>(groups), c.sequences), dim3(256), 0, as_stream(stream), c,
                     static_cast<uint16_t *>(out_key), static_cast<uint16_t *>(out_value), static_cast<int32_t>(tokens), chunks);
  return check_launch(what);
}

extern "C" int uc_paged_reserve(const uc_paged_cache *cache, int64_t tokens, const int32_t *counts, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::pg;
  const char *what = "uc_paged_reserve";
  Cache c;
  Pool pool;
  if (int rc = check_pool(cache, what, c, pool)) return rc;
  UC_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 30), "%s: bad number of tokens", what);
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kThreads), first_bytes(c), as_stream(stream), c, pool,
                     static_cast<int32_t>(tokens), counts);
  return check_launch(what);
}

extern "C" int64_t uc_paged_reorder_workspace_bytes(const uc_paged_cache *cache) {
  using namespace uc::pg;
  Cache c;
  Pool pool;
  Order o;
  if (check_pool(cache, "uc_paged_reorder", c, pool)) return -1;
  return lay_out(c, nullptr, o);
}

extern "C" int uc_paged_reorder(const uc_paged_cache *cache, const int32_t *parents, const int32_t *lengths,
                                int64_t max_tokens, void *workspace, int64_t workspace_bytes, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::pg;
  const char *what = "uc_paged_reorder";
  Cache c;
  Pool pool;
  Order o;
  if (int rc = check_pool(cache, what, c, pool)) return rc;
  UC_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                 workspace_bytes >= lay_out(c, static_cast<int32_t *>(workspace), o),
             "%s: workspace too small", what);
  UC_REQUIRE(cache->layers * c.heads * c.sequences < (1 << 24), "%s: too many layers, heads and sequences", what);
  UC_REQUIRE(max_tokens >= 0, "%s: negative max_tokens", what);
  o.parents = parents;
  o.cut = lengths;
  // what the launches are shaped for; they do with any lengths
  const int64_t widest = pages_expected(c, max_tokens);
  if (c.sequences * widest <= kSmallTable) {
    hipLaunchKernelGGL(reorder_small_kernel, dim3(1), dim3(kThreads), first_bytes(c), as_stream(stream), c, pool, o);
    if (int rc = check_launch(what)) return rc;
  } else {
    const dim3 groups = entry_groups(c, widest);
    hipLaunchKernelGGL(reorder_release_kernel, groups, dim3(256), 0, as_stream(stream), c, pool, o);
    if (int rc = check_launch(what)) return rc;
    hipLaunchKernelGGL(reorder_hold_kernel, groups, dim3(256), 0, as_stream(stream), c, pool, o);
    if (int rc = check_launch(what)) return rc;
    hipLaunchKernelGGL(reorder_open_kernel, dim3(1), dim3(kThreads), first_bytes(c), as_stream(stream), c, pool, o);
    if (int rc = check_launch(what)) return rc;
  }
  hipLaunchKernelGGL(reorder_copy_kernel, dim3(static_cast<uint32_t>(cache->layers * c.heads), c.sequences), dim3(256), 0,
                     as_stream(stream), c, o, static_cast<int32_t>(cache->head_dim * 2));
  return check_launch(what);
}

extern "C" int64_t uc_paged_compact_workspace_bytes(const uc_paged_cache *cache) {
  using namespace uc::pg;
  Cache c;
  Pool pool;
  Thin t;
  if (check_pool(cache, "uc_paged_compact", c, pool)) return -1;
  return lay_out(c, nullptr, t);
}

extern "C" int uc_paged_compact(const uc_paged_cache *cache, const uint8_t *keep, int64_t keep_stride, int64_t tokens,
                                int64_t max_tokens, void *workspace, int64_t workspace_bytes, uc_stream_t stream) {
  using namespace uc;
  using namespace uc::pg;
  const char *what = "uc_paged_compact";
  Cache c;
  Pool pool;
  Thin t;
  if (int rc = check_pool(cache, what, c, pool)) return rc;
  UC_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 30), "%s: bad number of tokens", what);
  UC_REQUIRE(tokens == 0 || keep != nullptr, "%s: keep is NULL", what);
  UC_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                 workspace_bytes >= lay_out(c, static_cast<int32_t *>(workspace), t),
             "%s: workspace too small", what);
  UC_REQUIRE(max_tokens >= 0, "%s: negative max_tokens", what);
  t.keep = keep;
  t.stride = keep_stride;
  t.tokens = static_cast<int32_t>(tokens);
  hipLaunchKernelGGL(thin_count_kernel, dim3(c.sequences), dim3(kThreads), 0, as_stream(stream), c, t);
  if (int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(thin_give_kernel, dim3(1), dim3(kThreads), first_bytes(c), as_stream(stream), c, pool, t);
  if (int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(thin_list_kernel, dim3(c.sequences), dim3(kThreads), 0, as_stream(stream), c, t);
  if (int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(thin_copy_kernel, dim3(4096), dim3(256), 0, as_stream(stream), c, t, static_cast<int32_t>(cache->layers),
                     static_cast<int32_t>(cache->head_dim / 8));
  if (int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(thin_commit_kernel, entry_groups(c, pages_expected(c, max_tokens)), dim3(256), 0, as_stream(stream), c,
                     pool, t);
  return check_launch(what);
}
