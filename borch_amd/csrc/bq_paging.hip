// Page tables of a paged cache, kept on the GPU: sequences are cut back, go over to others' pages (a beam
// search's forks), and new tokens get places. No call waits for the host, and all can be captured.
//
// The state: table [S][width] names each sequence's pages in order (-1 past the last), lens [S] its tokens,
// refs [pages] how many entries name a page. Pages are handed out in ascending order of their number,
// sequence after sequence, so that the same state and requests give the same tables. A page that is named
// several times is not written to: a sequence whose last page is partly filled and shared takes one of its own
// when it grows, and the caller moves the tokens there (bq_kv4_copy_pages).
//
// All of this is latency: the tables of a few hundred sequences are some 100 KB, and a launch of one workgroup is
// some eight look-ups one after another. 256 sequences of up to 128 pages: 3 us to cut, 8.6 to grow by a token each;
// 128 of 512 sequences ended and replaced by prompts of 4000 tokens, 200000 pages: 25 us in five launches.
#include "bq_kv4.h"

namespace bq {

struct Tables {
  int *table, *lens, *refs;
  int S, width, pages, page;
  FastDiv by_page;
};

__device__ __forceinline__ int pages_of(const Tables& a, int tokens) {
  return tokens <= 0 ? 0 : fdiv(tokens - 1, a.by_page.mul, a.by_page.shift) + 1;
}
__device__ __forceinline__ void add_ref(const Tables& a, int page, int by) {
  if ((unsigned)page < (unsigned)a.pages) atomicAdd(a.refs + page, by);
}

// A wave a sequence.
__global__ __launch_bounds__(256) void pages_cut_kernel(Tables a, const int* __restrict__ to) {
  const int s = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (s >= a.S) return;
  const int keep = min(a.lens[s], max(to[s], 0));
  int* row = a.table + (size_t)s * a.width;
  for (int c = pages_of(a, keep) + lane; c < a.width; c += 64) {
    const int page = row[c];
    if (page < 0) continue;
    add_ref(a, page, -1);
    row[c] = -1;
  }
  if (lane == 0) a.lens[s] = keep;  // this wave has read it
}

// Every row of the table becomes its parent's: a workgroup takes 2^`shift` columns of all rows through LDS,
// the last one the lengths. 8 columns above 128 rows, for more workgroups (192 rows of 24 pages: 13 us in 16 columns
// with divisions, so 5), fewer where LDS ends.
constexpr int FORK_ENTRIES = 16384, FORK_THREADS = 512, FORK_EACH = 4 * FORK_THREADS;
__global__ __launch_bounds__(FORK_THREADS) void pages_fork_kernel(Tables a, const int* __restrict__ parents, int shift) {
  extern __shared__ int old[];
  const bool lengths = blockIdx.x == gridDim.x - 1;
  const int column = blockIdx.x << shift, count = a.S << (lengths ? 0 : shift), bits = lengths ? 0 : shift;
  int* from = lengths ? a.lens : a.table;
  const size_t pitch = lengths ? 1 : a.width;
  const int c0 = lengths ? 0 : column, c1 = lengths ? 1 : a.width;
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += FORK_THREADS) {
    const int s = i >> bits, c = c0 + (i & ((1 << bits) - 1));
    old[i] = from[s * pitch + min(c, c1 - 1)];
  }
  __syncthreads();
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += FORK_THREADS) {
    const int s = i >> bits, e = i & ((1 << bits) - 1), p = parents[s], was = old[i];
    const int now = (unsigned)p < (unsigned)a.S ? old[(p << bits) + e] : lengths ? 0 : -1;
    if (now == was || c0 + e >= c1) continue;
    if (!lengths) {
      add_ref(a, was, -1);
      add_ref(a, now, 1);
    }
    from[s * pitch + c0 + e] = now;
  }
}

// Growing. BLOCK pages' free ones are found as 64 words of 64 bits, a lane's word each. Up to SOLO_PAGES pages the
// plan's waves read refs themselves, beyond it a launch before it writes the words down. One workgroup plans, since
// the tables change only where all find room; it also hands out the pages and writes the places, but those of many
// tokens (SOLO_ROWS) are launches of their own (16000 pages for 512000 tokens: 62 us by the plan alone, 16 with them).
constexpr int BLOCK = 4096, PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;
constexpr int MOST_SEQUENCES = 8192, MOST_BLOCKS = 4096;
constexpr int64_t SOLO_PAGES = (int64_t)BLOCK * PLAN_WAVES;
constexpr int SOLO_ROWS = 8192;

struct Grow {
  Tables t;
  const int* more;  // new tokens of each sequence
  int rows;         // room for their places
  int* cu;
  int64_t* slots;
  int *at, *moves, *ok;
  uint64_t* words;  // the workspace, or null: free pages; in each BLOCK, then before it; wanted pages before a sequence
  int *counts, *upto;
  bool solo;  // the plan hands out and writes the places
};

// Up to 64 words of free pages by one wave, the first for the pages from 64 `w0` on, lane l's the l-th.
__device__ __forceinline__ uint64_t free_words(const Tables& a, int w0, int n) {
  const int lane = threadIdx.x & 63;
  uint64_t mine = 0;
  for (int i = 0; i < n && (w0 + i) * 64 < a.pages; i += 16) {
    int refs[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) refs[e] = a.refs[min((w0 + i + e) * 64 + lane, a.pages - 1)];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint64_t free = __ballot((w0 + i + e) * 64 + lane < a.pages && refs[e] == 0);
      if (lane == i + e && i + e < n) mine = free;
    }
  }
  return mine;
}

// The sum of the lanes' values up to this one's own; what passes 32 bits stays at their largest.
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint32_t plus_lanes(uint32_t v) {
  return __builtin_elementwise_add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
  v = plus_lanes<0x111, 0xF>(v);  // from the lanes 1, 2, 4 and 8 before in a row of 16,
  v = plus_lanes<0x112, 0xF>(v);
  v = plus_lanes<0x114, 0xF>(v);
  v = plus_lanes<0x118, 0xF>(v);
  v = plus_lanes<0x142, 0xA>(v);  // the last of the row before into the second and fourth,
  return plus_lanes<0x143, 0xC>(v);  // lane 31's into the upper half
}

// A wave's words' free pages in ascending order: f(page, k), k from `rank` on and below `limit`.
template <typename F>
__device__ __forceinline__ void each_free(uint64_t word, int w0, int rank, int limit, F&& f) {
  const int lane = threadIdx.x & 63, upto = (int)wave_upto(__builtin_popcountll(word));
  const int before = upto - __builtin_popcountll(word), n = min(__shfl(upto, 63), limit - rank);
  for (int j0 = 0; j0 < n; j0 += 64) {
    const int j = j0 + lane;
    int l = 0;
#pragma unroll
    for (int d = 32; d; d /= 2) l += __shfl(before, l + d) <= j ? d : 0;
    int nth = j - __shfl(before, l), bit = 0;
    uint64_t w = (uint64_t)(uint32_t)__shfl((int)(word >> 32), l) << 32 | (uint32_t)__shfl((int)word, l);
#pragma unroll
    for (int d = 32; d; d /= 2) {
      const int low = __builtin_popcountll(w & ((1ull << d) - 1));
      const bool above = nth >= low;
      nth -= above ? low : 0;
      bit += above ? d : 0;
      w >>= above ? d : 0;
    }
    if (j < n) f((w0 + l) * 64 + bit, rank + j);
  }
}

__global__ __launch_bounds__(256) void pages_count_kernel(Grow g) {
  __shared__ int of[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w0 = blockIdx.x * 64 + wave * 16;
  const uint64_t word = free_words(g.t, w0, 16);
  if (lane < 16) g.words[w0 + lane] = word;
  const int n = (int)wave_upto(__builtin_popcountll(word));
  if (lane == 63) of[wave] = n;
  __syncthreads();
  if (threadIdx.x == 0) g.counts[blockIdx.x] = of[0] + of[1] + of[2] + of[3];
}

// The sums over the workgroup's threads before this one, and of all (at 32 bits' largest where they pass it, which
// is more than any caller has room for).
struct Pair {
  uint32_t pages, tokens;
};
__device__ __forceinline__ Pair plus(Pair a, Pair b) {
  return {__builtin_elementwise_add_sat(a.pages, b.pages), __builtin_elementwise_add_sat(a.tokens, b.tokens)};
}
__device__ __forceinline__ Pair scan_all(Pair v, Pair* waves, Pair* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Pair x = {wave_upto(v.pages), wave_upto(v.tokens)};
  __syncthreads();  // the last scan's sums are read
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  Pair before = {0, 0}, total = {0, 0};
#pragma unroll
  for (int i = 0; i < PLAN_WAVES; ++i) {
    if (i == wave) before = total;
    total = plus(total, waves[i]);
  }
  *all = total;
  const uint32_t p = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x.pages, 0x138, 0xF, 0xF, false);  // the lane before
  const uint32_t t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x.tokens, 0x138, 0xF, 0xF, false);
  return plus(before, {p, t});
}

// Where k lies among the running sums upto[0] = 0, ...: the last i in [lo, hi] with upto[i] <= k.
__device__ __forceinline__ int holder_of(const int* upto, int lo, int hi, int k) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (upto[mid] <= k) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Place i of the new tokens: of sequence s, whose first is `first`, with `len` tokens before them.
__device__ __forceinline__ void put_place(const Grow& g, int i, int s, int64_t len, int first) {
  const Tables& a = g.t;
  const int at = (int)(len + i - first), c = fdiv(at, a.by_page.mul, a.by_page.shift);
  const int page = a.table[(size_t)s * a.width + c];
  g.at[i] = at;
  g.slots[i] = (unsigned)page < (unsigned)a.pages ? (int64_t)page * a.page + (at - c * a.page) : -1;
}

// A free page to sequence s as its `nth` new one; `share`: the page that the first takes the place of, or -1.
template <int SCOPE>
__device__ __forceinline__ void give(const Grow& g, int page, int s, int nth, int len, int share) {
  const Tables& a = g.t;
  const int c = pages_of(a, len) + nth - (share >= 0 ? 1 : 0);
  if (share >= 0 && nth == 0) {
    __hip_atomic_fetch_add(a.refs + share, -1, __ATOMIC_RELAXED, SCOPE);
    g.moves[a.S + s] = page;
  }
  a.table[(size_t)s * a.width + c] = page;
  a.refs[page] = 1;
}

// What each sequence wants, one workgroup: nothing is written before it is known that all find room.
__global__ __launch_bounds__(PLAN_THREADS) void pages_grow_kernel(Grow g) {
  // pages and tokens before a sequence, its tokens, the page that it shares; pages free before a block. The first
  // three hold the shared pages' hash table before that: the page, the lowest sequence, how many.
  __shared__ int upto[MOST_SEQUENCES + 1], first[MOST_SEQUENCES + 1], held[MOST_SEQUENCES], share[MOST_SEQUENCES];
  __shared__ int blocks[MOST_BLOCKS + 1];
  __shared__ Pair waves[PLAN_WAVES];
  const Tables& a = g.t;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // the first of this thread's sequences, and refs if they are read here: on their way together
  const int mine = min(tid, a.S - 1), len0 = mine < 0 ? 0 : a.lens[mine], more0 = mine < 0 ? 0 : g.more[mine];
  int count = PLAN_WAVES, each = ((a.pages + 63) / 64 + PLAN_WAVES - 1) / PLAN_WAVES;  // words a block, 64 at most
  const uint64_t word = g.words ? 0 : free_words(a, wave * each, each);
  // the last page of each that grows, if it is partly filled and named elsewhere too
  bool bad = false, any = false;
  for (int s = tid; s < a.S; s += PLAN_THREADS) {
    const int len = s == tid ? len0 : a.lens[s], more = s == tid ? more0 : g.more[s];
    const int c = fdiv(max(len, 0), a.by_page.mul, a.by_page.shift);
    // width pages are fewer than 2^31 tokens
    bad |= more < 0 || len < 0 || (int64_t)len + more > (int64_t)a.width * a.page;
    int page = -1;
    if (len > 0 && more > 0 && c < a.width && len != c * a.page) {
      page = a.table[(size_t)s * a.width + c];
      if ((unsigned)page >= (unsigned)a.pages || a.refs[page] < 2) page = -1;
    }
    share[s] = page;
    any |= page >= 0;
  }
  // of those that share a page and grow the lowest keeps it where they are all that name it
  if (__syncthreads_or(any)) {
    int bits = 6;
    while (1 << bits < 2 * a.S && 1 << bits < MOST_SEQUENCES) ++bits;  // as many slots as sequences at least
    const int mask = (1 << bits) - 1;
    for (int i = tid; i <= mask; i += PLAN_THREADS) upto[i] = -1, first[i] = MOST_SEQUENCES, held[i] = 0;
    __syncthreads();
    for (int s = tid; s < a.S; s += PLAN_THREADS) {
      const int page = share[s];
      if (page < 0) continue;
      int h = (int)((uint32_t)page * 0x9E3779B1u >> (32 - bits));
      for (;; h = (h + 1) & mask) {
        const int was = atomicCAS(upto + h, -1, page);
        if (was == -1 || was == page) break;
      }
      atomicMin(first + h, s);
      atomicAdd(held + h, 1);
    }
    __syncthreads();
    for (int s = tid; s < a.S; s += PLAN_THREADS) {
      const int page = share[s];
      if (page < 0) continue;
      int h = (int)((uint32_t)page * 0x9E3779B1u >> (32 - bits));
      while (upto[h] != page) h = (h + 1) & mask;
      if (first[h] == s && held[h] == a.refs[page]) share[s] = -1;
    }
    __syncthreads();
  }
  Pair total = {0, 0};
  for (int s0 = 0; s0 < a.S; s0 += PLAN_THREADS) {
    const int s = s0 + tid;
    Pair want = {0, 0}, all;
    if (s < a.S) {
      const int len = max(s0 == 0 ? len0 : a.lens[s], 0), more = max(s0 == 0 ? more0 : g.more[s], 0);
      want.tokens = more;  // what does not fit is refused, whatever its pages
      want.pages = max(pages_of(a, (int)min((uint32_t)len + more, 0x7fffffffu)) - pages_of(a, len), 0) + (share[s] >= 0);
      held[s] = len;
    }
    const Pair before = scan_all(want, waves, &all);
    if (s < a.S) {
      const Pair from = plus(total, before);
      upto[s] = (int)min(from.pages, 0x7fffffffu);
      first[s] = (int)min(from.tokens, 0x7fffffffu);
    }
    total = plus(total, all);
  }
  bad |= total.tokens > (uint32_t)g.rows || total.pages > (uint32_t)a.pages;
  // the free pages, where any are wanted
  bool good = !__syncthreads_or(bad);
  const int wanted = good ? (int)total.pages : 0;
  if (wanted > 0) {
    Pair all;
    int free = 0;  // 2^24 at most
    if (!g.words) {
      const Pair before = scan_all({(uint32_t)__builtin_popcountll(word), 0}, waves, &all);
      if (lane == 0) blocks[wave] = (int)before.pages;
      free = (int)all.pages;
    } else {
      each = 64;
      count = (a.pages + BLOCK - 1) / BLOCK;
      for (int b0 = 0; b0 < count; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        const Pair before = scan_all({b < count ? (uint32_t)g.counts[b] : 0, 0}, waves, &all);
        if (b < count) blocks[b] = free + (int)before.pages;
        free += (int)all.pages;
      }
    }
    good = free >= wanted;
    __syncthreads();
    if (good && g.words && !g.solo) {  // a launch of its own hands them out
      for (int b = tid; b < count; b += PLAN_THREADS) g.counts[b] = blocks[b];
      for (int s = tid; s < a.S; s += PLAN_THREADS) g.upto[s] = upto[s];
    } else if (good) {
      for (int b = wave; b < count && blocks[b] < wanted; b += PLAN_WAVES)
        each_free(g.words ? g.words[b * 64 + lane] : word, b * each, blocks[b], wanted, [&](int page, int k) {
          const int s = holder_of(upto, 0, a.S - 1, k);
          give<__HIP_MEMORY_SCOPE_WORKGROUP>(g, page, s, k - upto[s], held[s], share[s]);
        });
    }
  }
  if (g.words && tid == 0) g.upto[a.S] = good ? wanted : 0;
  __syncthreads();
  for (int s = tid; s < a.S; s += PLAN_THREADS) {
    const int len = held[s];
    const bool own = good && share[s] >= 0;
    g.moves[s] = own ? share[s] : -1;
    if (!own) g.moves[a.S + s] = -1;
    g.moves[2 * a.S + s] = own ? len - fdiv(len, a.by_page.mul, a.by_page.shift) * a.page : 0;
    g.cu[s] = good ? first[s] : 0;
    if (good) a.lens[s] = len + (s == tid ? more0 : g.more[s]);
  }
  if (tid == 0) {
    g.cu[a.S] = good ? (int)total.tokens : 0;
    g.ok[0] = good ? 1 : 0;
  }
  if (g.solo)
    for (int i = tid; i < g.rows; i += PLAN_THREADS) {
      if (!good || i >= (int)total.tokens) {
        g.at[i] = -1;
        g.slots[i] = -1;
      } else {
        const int s = holder_of(first, 0, a.S - 1, i);
        put_place(g, i, s, held[s], first[s]);
      }
    }
}

// The pages of many new tokens, after the plan: a workgroup a block, a wave four of its words.
__global__ __launch_bounds__(1024) void pages_give_kernel(Grow g) {
  extern __shared__ int upto[];
  const Tables& a = g.t;
  const int lane = threadIdx.x & 63, w0 = threadIdx.x >> 6 << 2, b = blockIdx.x;
  const int wanted = g.upto[a.S], rank = g.counts[b];
  if (rank >= wanted) return;
  const uint64_t all = g.words[b * 64 + lane], mine = g.words[b * 64 + w0 + (lane & 3)];
  for (int s = threadIdx.x; s < a.S; s += 1024) upto[s] = g.upto[s];
  __syncthreads();
  const int n = __builtin_popcountll(all), before = rank + __shfl((int)wave_upto(n) - n, w0);
  if (before >= wanted) return;
  each_free(lane < 4 ? mine : 0, b * 64 + w0, before, wanted, [&](int page, int k) {
    const int s = holder_of(upto, 0, a.S - 1, k);
    give<__HIP_MEMORY_SCOPE_AGENT>(g, page, s, k - upto[s], a.lens[s] - (g.cu[s + 1] - g.cu[s]), g.moves[s]);
  });
}

// The last s with cu[s] <= k by one wave, 64 at a time.
__device__ __forceinline__ int wave_holder(const int* cu, int S, int k) {
  int lo = 0, n = S;
  while (n > 1) {
    const int step = (n + 63) >> 6, i = (int)(threadIdx.x & 63) * step;
    const int below = __builtin_popcountll(__ballot(i < n && cu[lo + min(i, n - 1)] <= k)) - 1;  // cu[lo] <= k
    lo += below * step;
    n = min(step, n - below * step);
  }
  return lo;
}

// The places of many new tokens, after their pages: a wave takes 256.
__global__ __launch_bounds__(256) void pages_places_kernel(Grow g) {
  const int lane = threadIdx.x & 63, S = g.t.S, all = S ? g.cu[S] : 0;
  const int64_t i0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 256;
  if (i0 >= g.rows) return;
  int lo = 0, hi = 0;
  if (i0 < all) {
    const int last = (int)min(i0 + 255, (int64_t)all - 1);
    lo = wave_holder(g.cu, S, (int)i0);
    hi = g.cu[lo + 1] > last ? lo : lo + wave_holder(g.cu + lo, S - lo, last);
  }
  int s[4], first[4], end[4], len[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = lo;
  if (lo < hi)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = holder_of(g.cu, lo, hi, (int)min(i0 + e * 64 + lane, (int64_t)all - 1));
  if (i0 < all)
#pragma unroll
    for (int e = 0; e < 4; ++e) first[e] = g.cu[s[e]], end[e] = g.cu[s[e] + 1], len[e] = g.t.lens[s[e]];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t at = i0 + e * 64 + lane;
    if (at < all && at < g.rows) put_place(g, (int)at, s[e], (int64_t)len[e] - (end[e] - first[e]), first[e]);
    else if (at < g.rows) g.at[at] = -1, g.slots[at] = -1;
  }
}

// The tokens of pages that go over to others, in up to CACHES caches: a workgroup a cache, move and head
// takes 32 tokens' codes and scales at a time as they lie.
constexpr int CACHES = 64;
struct Copy {
  struct {
    uint8_t* p[4];
    int pages, heads, page, dim;
  } c[CACHES];
  const int* moves;
  int S;
};
__global__ __launch_bounds__(256) void kv4_copy_pages_kernel(Copy a) {
  const auto& c = a.c[blockIdx.z];
  const int s = blockIdx.x, h = blockIdx.y;
  if (h >= c.heads) return;
  const int src = a.moves[s], dst = a.moves[a.S + s], blocks = (min(a.moves[2 * a.S + s], c.page) + 31) >> 5;
  if ((unsigned)src >= (unsigned)c.pages || (unsigned)dst >= (unsigned)c.pages || src == dst) return;
  const size_t from = (size_t)src * c.heads + h, to = (size_t)dst * c.heads + h;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int row = x & 1 ? c.dim / 32 : c.dim / 2;  // bytes of a token
    const int pieces = 32 * blocks * row / 16;
    const uint4* f = reinterpret_cast<const uint4*>(c.p[x] + from * c.page * row);
    uint4* t = reinterpret_cast<uint4*>(c.p[x] + to * c.page * row);
    for (int i = threadIdx.x; i < pieces; i += 256) t[i] = f[i];
  }
}

static int tables_of(const char* what, const bq_pages* p, Tables* out) {
  if (!p) return set_error(BQ_ERR_ARG, "%s: null tables", what);
  if (p->sequences < 0 || p->width < 0 || p->pages < 0 || p->page < 1 || p->page > 1 << 20)
    return set_error(BQ_ERR_ARG, "%s: bad sizes", what);
  if (p->sequences > MOST_SEQUENCES)
    return set_error(BQ_ERR_UNSUPPORTED, "%s: %lld sequences (%d at most)", what, (long long)p->sequences, MOST_SEQUENCES);
  if (p->pages > (int64_t)MOST_BLOCKS * BLOCK || p->width > 0x7fffffff / MOST_SEQUENCES ||
      p->width * p->page > 0x7fffffff - 8192)
    return set_error(BQ_ERR_ARG, "%s: size too large", what);
  if ((p->sequences && (!p->lens || (p->width && !p->table))) || (p->pages && !p->refs))
    return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  *out = Tables{p->table, p->lens, p->refs, (int)p->sequences, (int)p->width, (int)p->pages, (int)p->page,
                fast_div((uint32_t)p->page)};
  return BQ_OK;
}

}  // namespace bq

using namespace bq;

int bq_pages_cut(const bq_pages* pages, const int32_t* to, bq_stream_t stream) {
  const char* what = "bq_pages_cut";
  Tables a;
  if (const int rc = tables_of(what, pages, &a)) return rc;
  if (a.S == 0) return BQ_OK;
  if (!to) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  pages_cut_kernel<<<(a.S + 3) / 4, 256, 0, (hipStream_t)stream>>>(a, to);
  return check_launch(what);
}

int bq_pages_fork(const bq_pages* pages, const int32_t* parents, bq_stream_t stream) {
  const char* what = "bq_pages_fork";
  Tables a;
  if (const int rc = tables_of(what, pages, &a)) return rc;
  if (a.S == 0) return BQ_OK;
  if (!parents) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  int shift = 4;
  while (shift > 1 && (a.S << shift) > (shift > 3 ? FORK_EACH : FORK_ENTRIES)) --shift;  // S <= 8192: two columns at least
  const int tiles = (a.width + (1 << shift) - 1) >> shift;
  pages_fork_kernel<<<tiles + 1, FORK_THREADS, ((size_t)a.S << shift) * 4, (hipStream_t)stream>>>(a, parents, shift);
  return check_launch(what);
}

size_t bq_pages_grow_ws_bytes(int64_t sequences, int64_t pages) {
  if (sequences < 0 || sequences > MOST_SEQUENCES || pages <= SOLO_PAGES || pages > (int64_t)MOST_BLOCKS * BLOCK) return 0;
  return (size_t)((pages + BLOCK - 1) / BLOCK) * (64 * 8 + 4) + (sequences + 1) * 4;
}

int bq_pages_grow(const bq_pages* pages, const int32_t* more, int64_t rows, int32_t* cu, int64_t* slots, int32_t* at,
                  int32_t* moves, int32_t* ok, void* ws, size_t ws_bytes, bq_stream_t stream) {
  const char* what = "bq_pages_grow";
  Grow g;
  if (const int rc = tables_of(what, pages, &g.t)) return rc;
  if (rows < 0 || rows > 0x7fffffff - 8192) return set_error(BQ_ERR_ARG, "%s: %lld rows", what, (long long)rows);
  if (!cu || !ok || (rows && (!slots || !at)) || (g.t.S && (!more || !moves)))
    return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const size_t need = bq_pages_grow_ws_bytes(g.t.S, g.t.pages);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 7)))
    return set_error(BQ_ERR_ARG, "%s: a workspace of %zu bytes, given %zu", what, need, ws ? ws_bytes : 0);
  const int blocks = (g.t.pages + BLOCK - 1) / BLOCK;
  g.more = more;
  g.rows = (int)rows;
  g.cu = cu;
  g.slots = slots;
  g.at = at;
  g.moves = moves;
  g.ok = ok;
  g.words = need ? (uint64_t*)ws : nullptr;
  g.counts = need ? (int*)(g.words + (size_t)blocks * 64) : nullptr;
  g.upto = need ? g.counts + blocks : nullptr;
  g.solo = rows <= SOLO_ROWS;
  hipStream_t st = (hipStream_t)stream;
  if (need) pages_count_kernel<<<blocks, 256, 0, st>>>(g);
  pages_grow_kernel<<<1, PLAN_THREADS, 0, st>>>(g);
  if (need && !g.solo) pages_give_kernel<<<blocks, 1024, (size_t)g.t.S * 4, st>>>(g);
  if (!g.solo) pages_places_kernel<<<(unsigned)((rows + 1023) / 1024), 256, 0, st>>>(g);
  return check_launch(what);
}

int bq_kv4_copy_pages(const bq_kv4_cache* caches, int64_t count, const int32_t* moves, int64_t sequences,
                      bq_stream_t stream) {
  const char* what = "bq_kv4_copy_pages";
  if (count < 0 || sequences < 0 || sequences > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: bad sizes", what);
  if (count && !caches) return set_error(BQ_ERR_ARG, "%s: null cache", what);
  for (int64_t i = 0; i < count; ++i) {
    Kv4 c;
    if (const int rc = kv4_of(what, caches + i, nullptr, 0, 0, &c)) return rc;
  }
  if (count == 0 || sequences == 0) return BQ_OK;
  if (!moves) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  for (int64_t i0 = 0; i0 < count; i0 += CACHES) {
    Copy a;
    const int n = (int)(count - i0 < CACHES ? count - i0 : CACHES);
    int heads = 1;
    for (int i = 0; i < n; ++i) {
      const bq_kv4_cache& c = caches[i0 + i];
      a.c[i] = {{c.k, c.k_scales, c.v, c.v_scales}, (int)c.pages, (int)c.heads, (int)c.page, (int)c.dim};
      if (c.heads > heads) heads = (int)c.heads;
    }
    a.moves = moves;
    a.S = (int)sequences;
    kv4_copy_pages_kernel<<<dim3((unsigned)sequences, heads, n), 256, 0, (hipStream_t)stream>>>(a);
  }
  return check_launch(what);
}
