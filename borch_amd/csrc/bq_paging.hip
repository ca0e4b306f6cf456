// Page tables of a paged cache, kept on the GPU: sequences are cut back, go over to others' pages (a beam
// search's forks), and new tokens get places. No call waits for the host, and all can be captured.
//
// The state: table [S][width] names each sequence's pages in order (-1 past the last), lens [S] its tokens,
// refs [pages] how many entries name a page. Pages are handed out in ascending order of their number,
// sequence after sequence, so that the same state and requests give the same tables. A page that is named
// several times is not written to: a sequence whose last page is partly filled and shared takes one of its own
// when it grows, and the caller moves the tokens there (bq_kv4_copy_pages).
//
// All of this is latency: the tables of a few hundred sequences are some 100 KB.
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

// Every row of the table becomes its parent's: a workgroup takes `columns` columns of all rows through LDS,
// the last one the lengths.
constexpr int FORK_ENTRIES = 16384;
__global__ __launch_bounds__(256) void pages_fork_kernel(Tables a, const int* __restrict__ parents, int columns) {
  extern __shared__ int old[];
  const bool lengths = blockIdx.x == gridDim.x - 1;
  const int c0 = blockIdx.x * columns, n = lengths ? 1 : min(columns, a.width - c0);
  int* from = lengths ? a.lens : a.table + c0;
  const size_t pitch = lengths ? 1 : a.width;
  for (int i = threadIdx.x; i < a.S * n; i += 256) old[i] = from[i / n * pitch + i % n];
  __syncthreads();
  for (int i = threadIdx.x; i < a.S * n; i += 256) {
    const int s = i / n, p = parents[s], was = old[i];
    const int now = (unsigned)p < (unsigned)a.S ? old[p * n + i % n] : lengths ? 0 : -1;
    if (now == was) continue;
    if (!lengths) {
      add_ref(a, was, -1);
      add_ref(a, now, 1);
    }
    from[s * pitch + i % n] = now;
  }
}

struct Grow {
  Tables t;
  const int* more;  // new tokens of each sequence
  int rows;         // room for their places
  int* cu;
  int64_t* slots;
  int *at, *moves, *ok;
  const int* counts;  // free pages in each BLOCK of them, or null
};

constexpr int BLOCK = 4096, PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;
constexpr int MOST_SEQUENCES = 8192, MOST_BLOCKS = 4096;
constexpr int64_t SOLO_PAGES = (int64_t)BLOCK * PLAN_WAVES;  // a wave of the plan counts a block itself
constexpr int SOLO_ROWS = 8192;                             // places that the plan writes itself

// The free pages of block b by one wave: f(page, rank) in ascending order, from `rank` on until it says no.
template <typename F>
__device__ __forceinline__ int each_free(const Tables& a, int b, int rank, F&& f) {
  const int lane = threadIdx.x & 63, end = min(a.pages, (b + 1) * BLOCK);
  const uint64_t before = (1ull << lane) - 1;
  for (int i = b * BLOCK; i < end; i += 512) {
    int refs[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) refs[e] = a.refs[min(i + 64 * e + lane, end - 1)];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int p = i + 64 * e + lane;
      const uint64_t free = __ballot(p < end && refs[e] == 0);
      if ((free >> lane) & 1) f(p, rank + __builtin_popcountll(free & before));
      rank += __builtin_popcountll(free);
    }
  }
  return rank;
}

__global__ __launch_bounds__(256) void pages_count_kernel(Tables a, int* counts) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if ((int64_t)b * BLOCK >= a.pages) return;
  const int n = each_free(a, b, 0, [](int, int) {});
  if ((threadIdx.x & 63) == 0) counts[b] = n;
}

// The sum over the workgroup's threads before this one, and of all.
__device__ __forceinline__ int64_t scan_all(int64_t v, int64_t* waves, int64_t* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the last scan's sums are read
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < PLAN_WAVES; ++i) {
    const int64_t w = waves[i];
    before += i < wave ? w : 0;
    total += w;
  }
  *all = total;
  return before + x - v;
}

// The first i of n whose running sum upto[i] (without i itself) passes k, less one: where k lies.
__device__ __forceinline__ int holder_of(const int* upto, int n, int k) {
  int lo = 0, hi = n - 1;
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

// What each sequence wants, one workgroup: nothing is written before it is known that all find room.
__global__ __launch_bounds__(PLAN_THREADS) void pages_grow_kernel(Grow g) {
  __shared__ int upto[MOST_SEQUENCES + 1], first[MOST_SEQUENCES + 1], share[MOST_SEQUENCES];  // pages, tokens before; the shared page
  __shared__ int blocks[MOST_BLOCKS + 1];
  __shared__ int64_t waves[PLAN_WAVES];
  const Tables& a = g.t;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // the last page of each that grows, if it is partly filled and named elsewhere too
  bool bad = false, any = false;
  for (int s = tid; s < a.S; s += PLAN_THREADS) {
    const int len = a.lens[s], more = g.more[s];
    const int c = fdiv(max(len, 0), a.by_page.mul, a.by_page.shift);
    const int64_t after = ((int64_t)len + more + a.page - 1) / a.page;
    bad |= more < 0 || len < 0 || after > a.width;
    int page = -1;
    if (len > 0 && more > 0 && c < a.width && len != c * a.page) {
      page = a.table[(size_t)s * a.width + c];
      if ((unsigned)page >= (unsigned)a.pages || a.refs[page] < 2) page = -1;
    }
    share[s] = page;
    any |= page >= 0;
  }
  const bool shares = __syncthreads_or(any);
  // of those that share a page and grow the lowest keeps it where they are all that name it
  int64_t pages = 0, tokens = 0;
  for (int s0 = 0; s0 < a.S; s0 += PLAN_THREADS) {
    const int s = s0 + tid;
    int64_t want = 0, more = 0;
    if (s < a.S) {
      bool own = false;
      if (shares && share[s] >= 0) {
        const int page = share[s];
        int same = 0, lower = 0;
        for (int i = 0; i < a.S; ++i) {
          const int hit = share[i] == page;
          same += hit;
          lower += i < s ? hit : 0;
        }
        own = lower > 0 || same != a.refs[page];
      }
      const int64_t len = max(a.lens[s], 0);
      more = max(g.more[s], 0);
      want = (len + more + a.page - 1) / a.page - (len + a.page - 1) / a.page + own;
      if (own) want |= 1ll << 40;
    }
    const bool own = (want >> 40) & 1;
    want &= (1ll << 40) - 1;
    int64_t all, all_more;
    const int64_t w = pages + scan_all(want, waves, &all), m = tokens + scan_all(more, waves, &all_more);
    if (s < a.S) {
      upto[s] = (int)min(w, (int64_t)0x7fffffff);
      first[s] = (int)min(m, (int64_t)0x7fffffff);
      g.moves[s] = own ? 0 : -1;  // read again below
    }
    pages += all;
    tokens += all_more;
  }
  bad |= tokens > g.rows || pages > a.pages;
  // the free pages, where any are wanted
  const int count = (int)(((int64_t)a.pages + BLOCK - 1) / BLOCK);
  bool good = !__syncthreads_or(bad);
  if (good && pages > 0) {
    if (!g.counts) {
      if (wave < count) {
        const int n = each_free(a, wave, 0, [](int, int) {});
        if (lane == 0) blocks[wave] = n;
      }
    } else {
      for (int b = tid; b < count; b += PLAN_THREADS) blocks[b] = g.counts[b];
    }
    __syncthreads();
    int64_t free = 0;
    for (int b0 = 0; b0 < count; b0 += PLAN_THREADS) {
      const int b = b0 + tid, n = b < count ? blocks[b] : 0;
      int64_t all;
      const int64_t w = free + scan_all(n, waves, &all);
      if (b < count) blocks[b] = (int)w;
      free += all;
    }
    good = free >= pages;
    __syncthreads();
    if (good) {
      for (int b = wave; b < count && blocks[b] < pages; b += PLAN_WAVES)
        each_free(a, b, blocks[b], [&](int page, int k) {
          if (k >= pages) return;
          const int s = holder_of(upto, a.S, k), len = a.lens[s];
          const bool own = g.moves[s] == 0;
          const int nth = k - upto[s];
          int c = pages_of(a, len) + nth - (own ? 1 : 0);
          if (own && nth == 0) {
            add_ref(a, share[s], -1);
            g.moves[a.S + s] = page;
          }
          a.table[(size_t)s * a.width + c] = page;
          a.refs[page] = 1;
        });
    }
  }
  __syncthreads();
  for (int s = tid; s < a.S; s += PLAN_THREADS) {
    const int len = a.lens[s];
    const bool own = good && g.moves[s] == 0;
    g.moves[s] = own ? share[s] : -1;
    if (!own) g.moves[a.S + s] = -1;
    g.moves[2 * a.S + s] = own ? len - fdiv(len, a.by_page.mul, a.by_page.shift) * a.page : 0;
    g.cu[s] = good ? first[s] : 0;
  }
  if (tid == 0) {
    g.cu[a.S] = good ? (int)tokens : 0;
    g.ok[0] = good ? 1 : 0;
  }
  if (g.rows <= SOLO_ROWS)
    for (int i = tid; i < g.rows; i += PLAN_THREADS) {
      if (!good || i >= tokens) {
        g.at[i] = -1;
        g.slots[i] = -1;
      } else {
        const int s = holder_of(first, a.S, i);
        put_place(g, i, s, a.lens[s], first[s]);
      }
    }
  __syncthreads();
  if (good)
    for (int s = tid; s < a.S; s += PLAN_THREADS) a.lens[s] += g.more[s];
}

// The places of many new tokens, after the plan.
__global__ __launch_bounds__(256) void pages_places_kernel(Grow g) {
  const int i = blockIdx.x * 256 + threadIdx.x, S = g.t.S;
  if (i >= g.rows) return;
  if (i >= g.cu[S]) {
    g.at[i] = -1;
    g.slots[i] = -1;
    return;
  }
  const int s = holder_of(g.cu, S, i);
  put_place(g, i, s, (int64_t)g.t.lens[s] - (g.cu[s + 1] - g.cu[s]), g.cu[s]);
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
  int columns = 16;
  while (columns * a.S > FORK_ENTRIES) columns /= 2;  // S <= 8192: two at least
  const int tiles = (a.width + columns - 1) / columns;
  pages_fork_kernel<<<tiles + 1, 256, (size_t)columns * a.S * 4, (hipStream_t)stream>>>(a, parents, columns);
  return check_launch(what);
}

size_t bq_pages_grow_ws_bytes(int64_t pages) {
  return pages > SOLO_PAGES ? (size_t)((pages + BLOCK - 1) / BLOCK) * 4 : 0;
}

int bq_pages_grow(const bq_pages* pages, const int32_t* more, int64_t rows, int32_t* cu, int64_t* slots, int32_t* at,
                  int32_t* moves, int32_t* ok, void* ws, size_t ws_bytes, bq_stream_t stream) {
  const char* what = "bq_pages_grow";
  Grow g;
  if (const int rc = tables_of(what, pages, &g.t)) return rc;
  if (rows < 0 || rows > 0x7fffffff - 8192) return set_error(BQ_ERR_ARG, "%s: %lld rows", what, (long long)rows);
  if (!cu || !ok || (rows && (!slots || !at)) || (g.t.S && (!more || !moves)))
    return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const size_t need = bq_pages_grow_ws_bytes(g.t.pages);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 3)))
    return set_error(BQ_ERR_ARG, "%s: a workspace of %zu bytes, given %zu", what, need, ws ? ws_bytes : 0);
  g.more = more;
  g.rows = (int)rows;
  g.cu = cu;
  g.slots = slots;
  g.at = at;
  g.moves = moves;
  g.ok = ok;
  g.counts = need ? (const int*)ws : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (need) {
    const int blocks = (g.t.pages + BLOCK - 1) / BLOCK;
    pages_count_kernel<<<(blocks + 3) / 4, 256, 0, st>>>(g.t, (int*)ws);
  }
  pages_grow_kernel<<<1, PLAN_THREADS, 0, st>>>(g);
  if (rows > SOLO_ROWS) pages_places_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(g);
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
