// The 4-bit cache's own passes (its form: bq_kv4.h): new tokens quantized into their pages, the
// values it holds, and the eviction of the tokens that received least.
#include <math.h>

#include <type_traits>

#include "bq_kv4.h"

namespace bq {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v8f __attribute__((ext_vector_type(8)));

int kv4_of(const char* what, const bq_kv4_cache* c, const int* table, int64_t B, int64_t width, Kv4* out) {
  if (!c) return set_error(BQ_ERR_ARG, "%s: null cache", what);
  if (c->dim != 64 && c->dim != 128)
    return set_error(BQ_ERR_UNSUPPORTED, "%s: head width %lld (64 or 128)", what, (long long)c->dim);
  if (c->page < 32 || c->page % 32 || c->page > (1 << 20))
    return set_error(BQ_ERR_UNSUPPORTED, "%s: %lld tokens a page (a multiple of 32)", what, (long long)c->page);
  if (c->pages < 0 || c->heads < 1 || B < 0 || width < 0) return set_error(BQ_ERR_ARG, "%s: bad sizes", what);
  if (c->pages > 0x7fffffff || c->heads > 65535 || B > 0x7fffff || width * c->page > 0x7fffffff - 8192)
    return set_error(BQ_ERR_ARG, "%s: size too large", what);
  if (c->pages && (!c->k || !c->k_scales || !c->v || !c->v_scales))
    return set_error(BQ_ERR_ARG, "%s: null cache array", what);
  if (B && width && !table) return set_error(BQ_ERR_ARG, "%s: null table", what);
  if (((uintptr_t)c->k | (uintptr_t)c->k_scales | (uintptr_t)c->v | (uintptr_t)c->v_scales) & 15)
    return set_error(BQ_ERR_ARG, "%s: misaligned cache array", what);
  *out = Kv4{c->k, c->k_scales, c->v, c->v_scales, (int)c->pages, (int)c->heads, (int)c->page, table, (int)width,
             fast_div((uint32_t)c->page), fast_div((uint32_t)c->page / 32)};
  return BQ_OK;
}

template <typename T>
__device__ __forceinline__ v8f load8(const T* p) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    return v8f{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  } else if constexpr (__is_same(T, __bf16)) {
    return __builtin_convertvector(*reinterpret_cast<const v8bf*>(p), v8f);
  } else {
    return __builtin_convertvector(*reinterpret_cast<const v8h*>(p), v8f);
  }
}

// New tokens into their pages. Eight channels a thread, DIM / 8 threads a token's row, the largest
// magnitude of 32 channels over four lanes. The scale's exponent is the least that takes it to 6
// or below, read off its bits: 1.m 2^E fits for 1.m <= 1.5 with E - 2, else with E - 1. Scaling by
// a power of two is exact (what underflows rounds to 0 either way), so the codes are the
// hardware's rounding to nearest even of the exact quotient.
// A workgroup takes 2048 / DIM tokens, whose places it looks up once, and PARTS of their 2 heads rows
// (keys, then values), all loaded at once: with a row a thread the chain of lookups before each
// row was most of the time (6237 tokens, 8 heads of 128, f32: 15.5 -> 13.4 us, 4.3 TB/s).
constexpr int PARTS = 4;
template <typename T, int DIM>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4 c, const T* __restrict__ nk, const T* __restrict__ nv,
                                                         int64_t kt, int64_t kh, int64_t vt, int64_t vh, int n, int groups,
                                                         const int* __restrict__ lens, const int* __restrict__ cu, int B) {
  using At = Kv4At<DIM>;
  constexpr int P = DIM / 8;
  const int tile = blockIdx.x / groups, part0 = (blockIdx.x - tile * groups) * PARTS;
  const int i = tile * (256 / P) + threadIdx.x / P, piece = threadIdx.x % P;
  if (i >= n) return;  // whole rows
  v8f x[PARTS];
#pragma unroll
  for (int e = 0; e < PARTS; ++e) {
    const int part = min(part0 + e, 2 * c.heads - 1);
    const bool is_v = part >= c.heads;
    const T* from = is_v ? nv + i * vt + (part - c.heads) * vh : nk + i * kt + part * kh;
    x[e] = load8(from + 8 * piece);
  }
  int lo = 0, hi = B;  // the sequence: the last b with cu[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] <= i) lo = mid + 1;
    else hi = mid;
  }
  int at = -1, off = 0;
  if (lo < B) {  // else past the last sequence
    const int64_t pos = (int64_t)lens[lo] - cu[lo + 1] + i;
    if (i >= cu[lo] && pos >= 0 && pos < (int64_t)c.width * c.page) {  // else before the first
      const int pi = fdiv((int)pos, c.by_page.mul, c.by_page.shift);
      at = kv4_page(c, lo, pi);
      off = (int)pos - pi * c.page;
    }
  }
#pragma unroll
  for (int e = 0; e < PARTS; ++e) {
    uint32_t peak = 0;  // |x| as integers: ordered as the values, NaN above infinity
#pragma unroll
    for (int j = 0; j < 8; ++j) peak = max(peak, __float_as_uint(x[e][j]) & 0x7fffffffu);
    peak = max(peak, (uint32_t)__builtin_amdgcn_mov_dpp((int)peak, 0xB1, 0xF, 0xF, false));
    peak = max(peak, (uint32_t)__builtin_amdgcn_mov_dpp((int)peak, 0x4E, 0xF, 0xF, false));
    if (at < 0 || part0 + e >= 2 * c.heads) continue;
    const bool is_v = part0 + e >= c.heads, finite = peak < 0x7f800000u;
    const int h = is_v ? part0 + e - c.heads : part0 + e;
    int byte = (int)((peak + 0x3fffffu) >> 23) - 2;  // E - 2, one more above 1.5 2^E
    byte = finite ? max(byte, 1) : 255;
    uint32_t code = 0;
    if (finite) {
      const float r = __uint_as_float((uint32_t)(254 - byte) << 23);  // 2^(127 - byte), byte <= 253
#define BQ_CODE(K) \
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, __fmul_rn(x[e][2 * K], r), __fmul_rn(x[e][2 * K + 1], r), 1.0f, K)
      BQ_CODE(0);
      BQ_CODE(1);
      BQ_CODE(2);
      BQ_CODE(3);
#undef BQ_CODE
    }
    const size_t row = At::row(c, at, h, off);
    if (is_v) {
      if constexpr (DIM == 128) {
        *reinterpret_cast<uint32_t*>(c.v + At::v(row, off, piece)) = code;
      } else {
        *reinterpret_cast<uint16_t*>(c.v + At::v(row, off, 2 * piece)) = (uint16_t)code;
        *reinterpret_cast<uint16_t*>(c.v + At::v(row, off, 2 * piece + 1)) = (uint16_t)(code >> 16);
      }
      if (piece % 4 == 0) c.vs[At::vs(row, off, piece / 4)] = (uint8_t)byte;
    } else {
      *reinterpret_cast<uint32_t*>(c.k + At::k(row) + 4 * piece) = code;
      if (piece % 4 == 0) c.ks[At::ks(row, off, piece / 4)] = (uint8_t)byte;
    }
  }
}

// Four channels' values: codes in a half word, the scale's byte.
__device__ __forceinline__ float4 kv4_values(uint32_t codes, uint32_t byte) {
  const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0);
  const v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1);
  const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
  return make_float4(__fmul_rn(a[0], s), __fmul_rn(a[1], s), __fmul_rn(b[0], s), __fmul_rn(b[1], s));
}

// The cache's values in f32, [B][heads][most][DIM] of keys and values, zeros past each length and
// where a table names no page. Bound by its writes: four channels a thread, so that a wave's store
// is one contiguous KiB; a workgroup takes 32 tokens (one place in one page). 134 MB written in 24 us,
// 5.6 TB/s (a fill of 128 MiB writes 6.5); stores past the caches were no faster.
template <int DIM>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4 c, const int* __restrict__ lens, int most, int blocks,
                                                       float* __restrict__ k, float* __restrict__ v) {
  using At = Kv4At<DIM>;
  constexpr int LANES = DIM / 4, TOKENS = 256 / LANES, PASSES = 32 / TOKENS;
  const int bh = blockIdx.x / blocks, t0 = (blockIdx.x - bh * blocks) * 32;
  const int b = bh / c.heads, h = bh - b * c.heads;
  const int len = min(lens[b], most);
  const int pi = fdiv(t0, c.by_page.mul, c.by_page.shift);
  const int at = t0 < len ? kv4_page(c, b, pi) : -1;
  const int off0 = t0 - pi * c.page;
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  uint32_t kc[PASSES], vc[PASSES], kb[PASSES], vb[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int t = p * TOKENS + sub, off = off0 + t;
    kc[p] = vc[p] = 0;
    kb[p] = vb[p] = 127;
    if (at >= 0 && t0 + t < len) {
      const size_t row = At::row(c, at, h, off);
      kc[p] = *reinterpret_cast<const uint16_t*>(c.k + At::k(row) + 2 * lane);
      if constexpr (DIM == 128) vc[p] = *reinterpret_cast<const uint16_t*>(c.v + At::v(row, off, lane >> 1) + 2 * (lane & 1));
      else vc[p] = *reinterpret_cast<const uint16_t*>(c.v + At::v(row, off, lane));
      kb[p] = c.ks[At::ks(row, off, lane / 8)];
      vb[p] = c.vs[At::vs(row, off, lane / 8)];
    }
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int t = t0 + p * TOKENS + sub;
    if (t < most) {
      const size_t to = ((size_t)bh * most + t) * DIM + 4 * lane;
      *reinterpret_cast<float4*>(k + to) = kv4_values(kc[p], kb[p]);
      *reinterpret_cast<float4*>(v + to) = kv4_values(vc[p], vb[p]);
    }
  }
}

// ---------------------------------------------------------------- eviction

// A weight's place in the order, as unsigned integers, all above 0; -0 with 0, NaN above all.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __float_as_uint(__fadd_rn(w, 0.f));
  const uint32_t o = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return __builtin_isnan(w) ? 0xffffffffu : o;
}

constexpr int EVICT_WAVES = 16, EVICT_THREADS = EVICT_WAVES * 64;

// The sum of `v` over the workgroup's threads before this one; *all gets the sum of all.
__device__ __forceinline__ int scan_before(int v, int* waves, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the last scan's sums are read
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < EVICT_WAVES; ++i) {
    const int w = waves[i];
    before += i < wave ? w : 0;
    total += w;
  }
  *all = total;
  return before + x - v;
}

// Which tokens of a (sequence, head) stay: the `recent` last ones, and of the others (the old) the
// keep - recent of largest weight, ties to the earlier token.
// A radix select over order_of finds the least weight that stays and how many of its equals do: 12,
// 12 and 8 bits, a histogram in LDS each. The first digit spans sign, exponent and three bits of
// the mantissa, so that weights of one size fall into eight counters and the lanes of a wave seldom
// meet in one; the weights that share the digit found are then listed, and the other digits look at
// the list alone (a row with more such than the list holds is read again for each). Places and weights
// are written in order: each wave counts, by ballots, those that stay of its 256 tokens, one scan sums
// the counts, and what stays is put side by side in LDS first.
//
// Rows of up to 16384 weights: one workgroup does it all (kv4_select_kernel<true>). Longer ones are
// bound by instructions on one CU (16 rows of 65536: 47 us), so parts of 8192 weights take workgroups of
// their own, in three launches: the first digit's counts of each part (kv4_tally_kernel), the list
// (kv4_list_kernel), the rest (kv4_select_kernel<false>: every part resolves the list itself).
constexpr int EVICT_STEP = 16384, EVICT_PART = 8192, EVICT_LIST = 8192;
constexpr int EVICT_SOLO = EVICT_STEP;  // the longest row of one workgroup
typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));

struct Evict {
  const float* sums;
  int64_t sums_b, sums_h;
  const int* lens;
  int most, heads, keep, recent, parts;
  int *kept, *left;
  float* weights;
  // long rows: a part's counts of the first digit [rows][parts][4096], its tokens above the digit found
  // [rows][parts]; a row's list (order_of, token), its length, and the digit with what remains to keep
  uint16_t* slots;
  int* over;
  uint2* list;
  int* listed;
  int2* found;
};

// A row's weights and lengths.
struct Row {
  const float* w;
  int b, n, old;  // old: those before the latest, 0 where all stay
  __device__ __forceinline__ Row(const Evict& a, int row) : b(row / a.heads) {
    n = max(0, min(a.lens[b], a.most));
    old = n > a.keep ? n - a.recent : 0;
    w = a.sums + b * a.sums_b + (row - b * a.heads) * a.sums_h;
  }
  // f(i, o) for tokens i .. i + 3 of from .. to (at most `old`), o order_of their weights, 0 past `to`: the
  // threads side by side, a wave's 256 tokens or none. The next loads under this step's work.
  template <typename F>
  __device__ __forceinline__ void each(int most, int from, int to, F&& f) const {
    constexpr int LOADS = EVICT_STEP / (4 * EVICT_THREADS);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto load = [&](int i0, v4fu (&x)[LOADS]) {
#pragma unroll
      for (int e = 0; e < LOADS; ++e) {
        const int c = i0 + (e * EVICT_WAVES + wave) * 256, i = c + 4 * lane;
        if (c + 256 <= most) {
          x[e] = *reinterpret_cast<const v4fu*>(w + i);
        } else if (c < to) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[e][j] = w[min(i + j, to - 1)];
        }
      }
    };
    v4fu now[LOADS] = {}, next[LOADS] = {};
    if (from < to) load(from, now);
#pragma unroll 1
    for (int i0 = from; i0 < to; i0 += EVICT_STEP) {
      if (i0 + EVICT_STEP < to) load(i0 + EVICT_STEP, next);
#pragma unroll
      for (int e = 0; e < LOADS; ++e) {
        const int c = i0 + (e * EVICT_WAVES + wave) * 256, i = c + 4 * lane;
        if (c >= to) break;
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = order_of(now[e][j]);
        if (c + 256 > to)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = i + j < to ? o[j] : 0u;
        f(i, o);
      }
#pragma unroll
      for (int e = 0; e < LOADS; ++e) now[e] = next[e];
    }
  }
};

// The digit at which hist's counts from the largest down reach `need`, and what then remains of it: four
// counters a thread. need = 0: the largest digit, of which none stays. By the whole workgroup.
__device__ __forceinline__ int2 find_digit(const int* hist, int count, int need, int* waves, int* found) {
  const int tid = threadIdx.x;
  int c4[4], sum = 0, all;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = count - 1 - 4 * tid - e;
    c4[e] = d >= 0 ? hist[d] : 0;
    sum += c4[e];
  }
  int above = scan_before(sum, waves, &all);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((above < need && above + c4[e] >= need) || (need == 0 && tid == 0 && e == 0)) {
      found[0] = count - 1 - 4 * tid - e;
      found[1] = need - above;
    }
    above += c4[e];
  }
  __syncthreads();
  const int2 r = make_int2(found[0], found[1]);
  __syncthreads();
  return r;
}

// Long rows, first: a part's counts of the first digit (a part has at most 8192).
__global__ __launch_bounds__(EVICT_THREADS) void kv4_tally_kernel(Evict a) {
  __shared__ int hist[4096];
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts, tid = threadIdx.x, lo = part * EVICT_PART;
  const Row r(a, row);
  if (part == 0 && tid == 0) a.listed[row] = 0;
  if (lo >= r.old) return;
  for (int i = tid; i < 4096; i += EVICT_THREADS) hist[i] = 0;
  __syncthreads();
  r.each(a.most, lo, min(r.old, lo + EVICT_PART), [&](int, const uint32_t (&o)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (o[j]) atomicAdd(&hist[o[j] >> 20], 1);
  });
  __syncthreads();
  uint2* to = reinterpret_cast<uint2*>(a.slots + ((size_t)row * a.parts + part) * 4096) + tid;
  const int* h = hist + 4 * tid;
  *to = make_uint2((uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16);
}

// Then: the first digit from all parts' counts, this part's tokens above it counted and those of it listed.
__global__ __launch_bounds__(EVICT_THREADS) void kv4_list_kernel(Evict a) {
  __shared__ int hist[4096], waves[EVICT_WAVES], found[2], over, count, first;
  __shared__ uint32_t keys[EVICT_PART];
  __shared__ uint16_t tokens[EVICT_PART];
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts, tid = threadIdx.x, lo = part * EVICT_PART;
  const Row r(a, row);
  if (lo >= r.old) return;
  int c[4] = {0, 0, 0, 0};
  const uint2* from = reinterpret_cast<const uint2*>(a.slots + (size_t)row * a.parts * 4096) + tid;
  const int parts = (r.old + EVICT_PART - 1) / EVICT_PART;
  for (int p0 = 0; p0 < parts; p0 += 8) {
    uint2 x[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) x[p] = from[(size_t)min(p0 + p, parts - 1) * 1024];
#pragma unroll
    for (int p = 0; p < 8; ++p)
      if (p0 + p < parts) c[0] += x[p].x & 0xffff, c[1] += x[p].x >> 16, c[2] += x[p].y & 0xffff, c[3] += x[p].y >> 16;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) hist[4 * tid + e] = c[e];
  if (tid == 0) over = count = 0;
  __syncthreads();
  const int2 digit = find_digit(hist, 4096, a.keep - a.recent, waves, found);
  if (part == 0 && tid == 0) a.found[row] = digit;
  int mine = 0;
  r.each(a.most, lo, min(r.old, lo + EVICT_PART), [&](int i, const uint32_t (&o)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mine += (int)(o[j] >> 20) > digit.x;
      if (o[j] && (int)(o[j] >> 20) == digit.x) {
        const int at = atomicAdd(&count, 1);
        keys[at] = o[j];
        tokens[at] = (uint16_t)(i + j - lo);
      }
    }
  });
  atomicAdd(&over, mine);
  __syncthreads();
  if (tid == 0) {
    a.over[(size_t)row * a.parts + part] = over;
    first = atomicAdd(&a.listed[row], count);  // the list's order does not matter
  }
  __syncthreads();
  for (int x = tid; x < min(count, EVICT_LIST - first); x += EVICT_THREADS)
    a.list[(size_t)row * EVICT_LIST + first + x] = make_uint2(keys[x], (uint32_t)(lo + tokens[x]));
}

template <bool SOLO>  // the row is one workgroup's
__global__ __launch_bounds__(EVICT_THREADS) void kv4_select_kernel(Evict a) {
  __shared__ int hist[4096], waves[EVICT_WAVES], found[2], listed;
  __shared__ uint32_t list[EVICT_LIST];
  __shared__ int tokens[SOLO ? 1 : EVICT_LIST];
  const int row = SOLO ? blockIdx.x : blockIdx.x / a.parts, part = SOLO ? 0 : blockIdx.x - row * a.parts;
  const int tid = threadIdx.x, lane = tid & 63, keep = a.keep;
  const Row r(a, row);
  const int lo = part * EVICT_PART, hi = SOLO ? r.n : min(r.n, lo + EVICT_PART);  // this workgroup's tokens
  int* kept = a.kept + (size_t)row * keep;
  float* weights = a.weights + (size_t)row * keep;
  if (row % a.heads == 0 && part == 0 && tid == 0) a.left[r.b] = min(r.n, keep);
  // the latest (or all), and past the last
  for (int i = max(lo, r.old) + tid; i < hi; i += EVICT_THREADS) {
    const int to = min(r.n, keep) - r.n + i;
    kept[to] = i;
    weights[to] = r.w[i];
  }
  for (int i = max(lo, r.n) + tid; i < (SOLO ? keep : min(keep, lo + EVICT_PART)); i += EVICT_THREADS) {
    kept[i] = -1;
    weights[i] = 0.f;
  }
  if (lo >= r.old) return;

  uint32_t prefix = 0, mask = 0;  // weights of `prefix` in their bits of `mask` are still undecided
  int need = keep - a.recent;     // and so many of them stay
  bool fits = true;
  if constexpr (!SOLO) {
    const int2 digit = a.found[row];
    prefix = (uint32_t)digit.x << 20;
    mask = 0xfff00000u;
    need = digit.y;
    const int count = a.listed[row];
    fits = count <= EVICT_LIST;
    if (tid == 0) listed = min(count, EVICT_LIST);
    for (int i = tid; i < min(count, EVICT_LIST); i += EVICT_THREADS) {
      const uint2 x = a.list[(size_t)row * EVICT_LIST + i];
      list[i] = x.x;
      tokens[i] = (int)x.y;
    }
  } else if (tid == 0) {
    listed = 0;
  }
  for (int digit = SOLO ? 0 : 1; digit < 3; ++digit) {
    const int shift = digit == 0 ? 20 : digit == 1 ? 8 : 0, count = digit == 2 ? 256 : 4096;
    for (int i = tid; i < count; i += EVICT_THREADS) hist[i] = 0;
    __syncthreads();
    auto tally = [&](uint32_t o) {
      if (o && (o & mask) == prefix) atomicAdd(&hist[(o >> shift) & (count - 1)], 1);
    };
    if (digit > 0 && fits)
      for (int i = tid; i < listed; i += EVICT_THREADS) tally(list[i]);
    else
      r.each(a.most, 0, r.old, [&](int, const uint32_t (&o)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) tally(o[j]);
      });
    __syncthreads();
    const int2 d = find_digit(hist, count, need, waves, found);
    prefix |= (uint32_t)d.x << shift;
    mask |= (uint32_t)(count - 1) << shift;
    need = d.y;
    if (SOLO && digit == 0) {
      r.each(a.most, 0, r.old, [&](int, const uint32_t (&o)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (o[j] && (o[j] & mask) == prefix) {
            const int at = atomicAdd(&listed, 1);
            if (at < EVICT_LIST) list[at] = o[j];
          }
      });
      __syncthreads();
      fits = listed <= EVICT_LIST;
    }
  }
  const uint32_t least = prefix;  // weights above it stay
  const int equals = need;        // and so many that equal it

  // those that stay before this workgroup's tokens, and the equals among them
  int out = 0, same = 0;
  if (!SOLO && part > 0) {
    int over = 0, eq = 0;
    if (fits) {
      for (int p = tid; p < part; p += EVICT_THREADS) over += a.over[(size_t)row * a.parts + p];
      for (int i = tid; i < listed; i += EVICT_THREADS) {
        over += tokens[i] < lo && list[i] > least;
        eq += tokens[i] < lo && list[i] == least;
      }
    } else {
      r.each(a.most, 0, lo, [&](int, const uint32_t (&o)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          over += o[j] > least;
          eq += o[j] == least;
        }
      });
    }
    scan_before(over, waves, &out);
    scan_before(eq, waves, &same);
    out += min(same, equals);
  }

  const int end = min(hi, r.old);  // one step
  __syncthreads();
  // of each 256 tokens, those above `least` and, from 256 on, its equals
  if (tid < 512) hist[tid] = 0;
  __syncthreads();
  r.each(a.most, lo, end, [&](int i, const uint32_t (&o)[4]) {
    int over = 0, eq = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      over += (int)__popcll(__ballot(o[j] > least));
      eq += (int)__popcll(__ballot(o[j] == least));
    }
    if (lane == 0) {
      hist[(i - lo) >> 8] = over;
      hist[256 + ((i - lo) >> 8)] = eq;
    }
  });
  __syncthreads();
  int all_eq, all;
  const int eq_here = tid < 256 ? hist[256 + tid] : 0;
  const int eq_before = same + scan_before(eq_here, waves, &all_eq);
  const int stay = (tid < 256 ? hist[tid] : 0) + max(0, min(eq_here, equals - eq_before));
  const int before = scan_before(stay, waves, &all);
  if (tid < 256) {
    hist[tid] = before;
    hist[256 + tid] = equals - eq_before;  // so many of its equals stay
  }
  __syncthreads();
  auto below = [&](bool x) {  // lanes before this one with x
    const uint64_t m = __ballot(x);
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
  };
  uint16_t* staged = reinterpret_cast<uint16_t*>(list);
  static_assert(EVICT_STEP * 2 <= EVICT_LIST * 4 && EVICT_STEP <= 65536 && EVICT_PART <= EVICT_STEP, "staging");
  r.each(a.most, lo, end, [&](int i, const uint32_t (&o)[4]) {
    const int at = __builtin_amdgcn_readfirstlane((i - lo) >> 8), cut = __builtin_amdgcn_readfirstlane(hist[256 + at]);
    bool stays[4];
    if (cut <= 0 || cut >= 256) {  // no equal stays, or all
      const uint32_t from = cut <= 0 ? least : least - 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) stays[j] = o[j] > from;
    } else {
      int rank = 0;  // of the lane's first token among the equals
#pragma unroll
      for (int j = 0; j < 4; ++j) rank += below(o[j] == least);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        stays[j] = o[j] > least || (o[j] == least && rank < cut);
        rank += o[j] == least;
      }
    }
    int to = hist[at];
#pragma unroll
    for (int j = 0; j < 4; ++j) to += below(stays[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (stays[j]) staged[to] = (uint16_t)(i + j - lo);
      to += stays[j];
    }
  });
  __syncthreads();
  for (int x = tid; x < all; x += EVICT_THREADS) {
    const int i = lo + staged[x];
    kept[out + x] = i;
    weights[out + x] = r.w[i];
  }
}

// The kept tokens of each (sequence, head) to the new pages in order: codes and scales as they are.
// A workgroup takes 4096 / DIM destinations, whose rows and sources' rows it looks up once; k's rows
// move 16 bytes a thread, v's slices are put together where they go (a thread gathers one slice of a
// block of tokens) and the scales in v_scales' order. 2048 of 64 rows of 2500 on average, heads of 128:
// 12 us; 16384 of 16 rows of 57768, heads of 64: 17 us, where nearly every block is touched (81 MB, 4.8 TB/s).
template <int DIM>
__global__ __launch_bounds__(256) void kv4_move_kernel(Kv4 c, Kv4 to, const int* __restrict__ kept, int keep,
                                                       int blocks) {
  using At = Kv4At<DIM>;
  constexpr int TB = At::TB, CB = At::CB, TOK = 4096 / DIM;
  // rows in the arrays; a destination of -1: nothing to move; a source of -1: zeros (its entry is no page, and the
  // new page may hold anything)
  __shared__ long long from[TOK], dest[TOK];
  __shared__ int from_off[TOK], dest_off[TOK];
  const int bh = blockIdx.x / blocks, t0 = (blockIdx.x - bh * blocks) * TOK;
  const int b = bh / c.heads, h = bh - b * c.heads, tid = threadIdx.x;
  if (tid < TOK) {
    const int i = t0 + tid, src = i < keep ? kept[(size_t)bh * keep + i] : -1;
    long long row = -1, to_row = -1;
    if (src >= 0) {
      const int si = fdiv(src, c.by_page.mul, c.by_page.shift), di = fdiv(i, c.by_page.mul, c.by_page.shift);
      const int sp = kv4_page(c, b, si), dp = kv4_page(to, b, di);
      from_off[tid] = src - si * c.page;
      dest_off[tid] = i - di * c.page;
      if (sp >= 0) row = (long long)At::row(c, sp, h, from_off[tid]);
      if (dp >= 0) to_row = (long long)At::row(c, dp, h, dest_off[tid]);
    }
    from[tid] = row;
    dest[tid] = to_row;
  }
  __syncthreads();
  if (tid < 128) {  // k: 16 bytes
    const int t = tid / (DIM / 32), q = tid % (DIM / 32);
    if (dest[t] >= 0) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (from[t] >= 0) x = *reinterpret_cast<const uint4*>(c.k + At::k(from[t]) + 16 * q);
      *reinterpret_cast<uint4*>(c.k + At::k(dest[t]) + 16 * q) = x;
    }
  } else {  // v: a slice of TB tokens, CB bytes each
    const int t = (tid - 128) / 16 * TB, s = tid % 16;
#pragma unroll
    for (int e = 0; e < TB; ++e)
      if (dest[t + e] >= 0) {
        typedef std::conditional_t<DIM == 128, uint32_t, uint16_t> Slice;
        Slice x = 0;
        if (from[t + e] >= 0) x = *reinterpret_cast<const Slice*>(c.v + At::v(from[t + e], from_off[t + e], s));
        *reinterpret_cast<Slice*>(c.v + At::v(dest[t + e], dest_off[t + e], s)) = x;
      }
  }
  if (tid < TOK * CB) {
    const int t = tid % TOK, s = tid / TOK;
    if (dest[t] >= 0) {
      c.vs[At::vs(dest[t], dest_off[t], s)] = from[t] >= 0 ? c.vs[At::vs(from[t], from_off[t], s)] : (uint8_t)1;
      c.ks[At::ks(dest[t], dest_off[t], s)] = from[t] >= 0 ? c.ks[At::ks(from[t], from_off[t], s)] : (uint8_t)1;
    }
  }
}

template <typename T, int DIM>
static void append_of(const Kv4& c, const void* nk, const void* nv, int64_t n, int64_t kt, int64_t kh, int64_t vt,
                      int64_t vh, const int* lens, const int* cu, int B, hipStream_t st) {
  const int groups = (2 * c.heads + PARTS - 1) / PARTS;
  const int64_t tiles = (n + 2048 / DIM - 1) / (2048 / DIM);
  kv4_append_kernel<T, DIM><<<(unsigned)(tiles * groups), 256, 0, st>>>(c, (const T*)nk, (const T*)nv, kt, kh, vt, vh, (int)n,
                                                                       groups, lens, cu, B);
}

}  // namespace bq

using namespace bq;

int bq_kv4_append(const bq_kv4_cache* cache, const void* new_k, const void* new_v, int type, int64_t n,
                  int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, const int32_t* table, int64_t B,
                  int64_t width, const int32_t* lens, const int32_t* cu, bq_stream_t stream) {
  const char* what = "bq_kv4_append";
  Kv4 c;
  if (const int rc = kv4_of(what, cache, table, B, width, &c)) return rc;
  if (type < 0 || type > 2) return set_error(BQ_ERR_ARG, "%s: type %d", what, type);
  if (n < 0 || n > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: %lld tokens", what, (long long)n);
  if (n == 0 || B == 0 || width == 0 || c.pages == 0) return BQ_OK;
  if (!new_k || !new_v || !lens || !cu) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const int64_t size = type == KV4_F32 ? 4 : 2;
  if ((((uintptr_t)new_k | (uintptr_t)new_v) & 15) || (k_token | k_head | v_token | v_head) * size % 16)
    return set_error(BQ_ERR_ARG, "%s: rows that are not 16-byte aligned", what);
  if ((n + 15) / 16 * ((2 * c.heads + PARTS - 1) / PARTS) > 0x7fffffff)
    return set_error(BQ_ERR_ARG, "%s: size too large", what);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = cache->dim == 128;
#define BQ_APPEND(T)                                                                                            \
  (wide ? append_of<T, 128>(c, new_k, new_v, n, k_token, k_head, v_token, v_head, lens, cu, (int)B, st)         \
        : append_of<T, 64>(c, new_k, new_v, n, k_token, k_head, v_token, v_head, lens, cu, (int)B, st))
  if (type == KV4_F32) BQ_APPEND(float);
  else if (type == KV4_BF16) BQ_APPEND(__bf16);
  else BQ_APPEND(_Float16);
#undef BQ_APPEND
  return check_launch(what);
}

int bq_kv4_read(const bq_kv4_cache* cache, const int32_t* table, int64_t B, int64_t width, const int32_t* lens,
                int64_t most, float* k, float* v, bq_stream_t stream) {
  const char* what = "bq_kv4_read";
  Kv4 c;
  if (const int rc = kv4_of(what, cache, table, B, width, &c)) return rc;
  if (most < 0 || most > 0x7fffffff - 8192) return set_error(BQ_ERR_ARG, "%s: %lld tokens", what, (long long)most);
  if (most == 0 || B == 0) return BQ_OK;
  if (!lens || !k || !v) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  if (((uintptr_t)k | (uintptr_t)v) & 15) return set_error(BQ_ERR_ARG, "%s: misaligned output", what);
  const int64_t blocks = (most + 31) / 32;
  if (B * c.heads > 0x7fffffff / blocks) return set_error(BQ_ERR_ARG, "%s: size too large", what);  // within 64 bits
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)(B * c.heads * blocks);
  if (cache->dim == 128) kv4_read_kernel<128><<<grid, 256, 0, st>>>(c, lens, (int)most, (int)blocks, k, v);
  else kv4_read_kernel<64><<<grid, 256, 0, st>>>(c, lens, (int)most, (int)blocks, k, v);
  return check_launch(what);
}

// Parts a row is cut into, 0 for one workgroup.
static int64_t evict_parts(int64_t most, int64_t keep) {
  return most <= EVICT_SOLO ? 0 : ((most > keep ? most : keep) + EVICT_PART - 1) / EVICT_PART;
}

size_t bq_kv4_evict_ws_bytes(int64_t B, int64_t heads, int64_t most, int64_t keep) {
  if (B < 1 || heads < 1) return 0;
  const size_t parts = (size_t)evict_parts(most, keep), rows = (size_t)B * heads;
  return parts ? rows * (parts * (4096 * 2 + 4) + EVICT_LIST * 8 + 8 + 4) : 0;
}

int bq_kv4_evict(const bq_kv4_cache* cache, const float* sums, int64_t sums_b, int64_t sums_h, int64_t most,
                 const int32_t* table, int64_t B, int64_t width, const int32_t* lens, const int32_t* new_table,
                 int64_t new_width, int64_t keep, int64_t recent, int32_t* kept, float* weights, int32_t* left,
                 void* ws, size_t ws_bytes, bq_stream_t stream) {
  const char* what = "bq_kv4_evict";
  Kv4 c, to;
  if (const int rc = kv4_of(what, cache, table, B, width, &c)) return rc;
  if (const int rc = kv4_of(what, cache, new_table, B, new_width, &to)) return rc;
  if (most < 0 || most > 0x7fffffff - 8192) return set_error(BQ_ERR_ARG, "%s: %lld weights a row", what, (long long)most);
  if (keep < 1 || keep > 0x7fffffff - 8192) return set_error(BQ_ERR_ARG, "%s: keep %lld", what, (long long)keep);
  if (recent < 0 || recent > keep)
    return set_error(BQ_ERR_ARG, "%s: the %lld latest of %lld kept", what, (long long)recent, (long long)keep);
  if (new_width * c.page < keep)
    return set_error(BQ_ERR_ARG, "%s: the new pages hold %lld tokens of %lld kept", what,
                     (long long)(new_width * c.page), (long long)keep);
  if (B == 0) return BQ_OK;
  if (!lens || !kept || !weights || !left || (most && !sums)) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const int64_t blocks = (keep + 4096 / cache->dim - 1) / (4096 / cache->dim);
  if (B * c.heads > 0x7fffffff / blocks) return set_error(BQ_ERR_ARG, "%s: size too large", what);  // within 64 bits
  hipStream_t st = (hipStream_t)stream;
  const int64_t rows = B * c.heads, parts = evict_parts(most, keep);
  const size_t need = bq_kv4_evict_ws_bytes(B, c.heads, most, keep);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    return set_error(BQ_ERR_ARG, "%s: a workspace of %zu bytes, given %zu", what, need, ws ? ws_bytes : 0);
  if (rows * parts > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  Evict a = {sums, sums_b, sums_h, lens, (int)most, c.heads, (int)keep, (int)recent, (int)parts, kept, left, weights};
  if (parts) {
    a.slots = (uint16_t*)ws;
    a.list = (uint2*)(a.slots + (size_t)rows * parts * 4096);
    a.found = (int2*)(a.list + (size_t)rows * EVICT_LIST);
    a.listed = (int*)(a.found + rows);
    a.over = a.listed + rows;
    kv4_tally_kernel<<<(unsigned)(rows * parts), EVICT_THREADS, 0, st>>>(a);
    kv4_list_kernel<<<(unsigned)(rows * parts), EVICT_THREADS, 0, st>>>(a);
    kv4_select_kernel<false><<<(unsigned)(rows * parts), EVICT_THREADS, 0, st>>>(a);
  } else {
    kv4_select_kernel<true><<<(unsigned)rows, EVICT_THREADS, 0, st>>>(a);
  }
  if (const int rc = check_launch(what)) return rc;
  const unsigned grid = (unsigned)(B * c.heads * blocks);
  if (c.pages == 0) return BQ_OK;
  if (cache->dim == 128) kv4_move_kernel<128><<<grid, 256, 0, st>>>(c, to, kept, (int)keep, (int)blocks);
  else kv4_move_kernel<64><<<grid, 256, 0, st>>>(c, to, kept, (int)keep, (int)blocks);
  return check_launch(what);
}
