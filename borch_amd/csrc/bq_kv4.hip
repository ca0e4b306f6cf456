// The 4-bit cache's own passes (its form: bq_kv4.h): new tokens quantized into their pages, the
// values it holds, and the eviction of the tokens that received least.
#include <math.h>

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
// row was most of the time (6237 tokens, 8 heads of 128: 15.5 us).
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
    if (pos >= 0 && pos < (int64_t)c.width * c.page) {
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
// is one contiguous KiB; a workgroup takes 32 tokens (one place in one page).
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

// Which tokens stay, one workgroup a (sequence, head): the `recent` last ones, and of the others
// the keep - recent of largest weight, ties to the earlier token.
// A radix select over order_of finds the least weight that stays and how many of its equals do: 12,
// 12 and 8 bits, a histogram in LDS each. The first digit spans sign, exponent and three bits of
// the mantissa, so that weights of one size fall into eight counters and the lanes of a wave seldom
// meet in one; the weights that share the digit found are then listed in LDS, where the other
// digits take no time (a row with more such than the list holds is read again for each digit). Two
// passes write places and weights in order: each wave counts, by ballots, those that stay of its 256
// tokens, one scan sums the counts, and each lane knows its place.
// The passes' loops stay rolled, the next loads under this step's work: with a row held in registers, 64
// weights a thread, the straight code for them took longer to fetch than four more reads from L2
// (64 rows of 4096: 30 us; 16 of 65536: 52).
constexpr int EVICT_STEP = 4, EVICT_SPAN = 65536, EVICT_LIST = 8192;
typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));

__global__ __launch_bounds__(EVICT_THREADS) void kv4_select_kernel(const float* __restrict__ sums, int64_t sums_b,
                                                                   int64_t sums_h, int most, int heads,
                                                                   const int* __restrict__ lens, int keep, int recent,
                                                                   int* __restrict__ kept, float* __restrict__ weights,
                                                                   int* __restrict__ left) {
  __shared__ int hist[4096], waves[EVICT_WAVES], found[2], listed;
  __shared__ uint32_t list[EVICT_LIST];
  const int bh = blockIdx.x, b = bh / heads, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = max(0, min(lens[b], most)), old = n > keep ? n - recent : 0;  // all stay: none is looked at
  const float* w = sums + b * sums_b + (bh - b * heads) * sums_h;
  kept += (size_t)bh * keep;
  weights += (size_t)bh * keep;
  if (bh % heads == 0 && tid == 0) left[b] = min(n, keep);

  // f(i, o) for tokens i .. i + 3 of the old ones from .. to, o order_of their weights, 0 past them; the
  // threads side by side, a wave's 256 tokens or none
  auto load = [&](int i0, int to, v4fu (&x)[EVICT_STEP]) {
#pragma unroll
    for (int e = 0; e < EVICT_STEP; ++e) {
      const int c = i0 + (e * EVICT_WAVES + wave) * 256, i = c + 4 * lane;
      if (c + 256 <= most) {
        x[e] = *reinterpret_cast<const v4fu*>(w + i);
      } else if (c < to) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[e][j] = w[min(i + j, old - 1)];
      }
    }
  };
  constexpr int STEP = EVICT_STEP * EVICT_THREADS * 4;  // tokens
  auto each = [&](int from, int to, auto&& f, auto&& after) {  // after(i0): a step's tokens are done
    v4fu now[EVICT_STEP] = {}, next[EVICT_STEP] = {};
    load(from, to, now);
#pragma unroll 1
    for (int i0 = from; i0 < to; i0 += STEP) {
      if (i0 + STEP < to) load(i0 + STEP, to, next);
#pragma unroll
      for (int e = 0; e < EVICT_STEP; ++e) {
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
      after(i0);
#pragma unroll
      for (int e = 0; e < EVICT_STEP; ++e) now[e] = next[e];
    }
  };
  auto nothing = [](int) {};

  uint32_t least = 0;       // weights above this stay
  int equals = 0x7fffffff;  // and so many that equal it
  if (n > keep) {
    int need = keep - recent;
    uint32_t prefix = 0, mask = 0;
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 20 : digit == 1 ? 8 : 0, count = digit == 2 ? 256 : 4096;
      for (int i = tid; i < count; i += EVICT_THREADS) hist[i] = 0;
      if (tid == 0 && digit == 0) listed = 0;
      __syncthreads();
      // a 0, of no weight, is counted under all others, where `need` never comes
      auto tally = [&](uint32_t o) {
        if ((o & mask) == prefix) atomicAdd(&hist[(o >> shift) & (count - 1)], 1);
      };
      if (digit > 0 && listed <= EVICT_LIST)
        for (int i = tid; i < listed; i += EVICT_THREADS) tally(list[i]);
      else
        each(0, old, [&](int, const uint32_t (&o)[4]) {
#pragma unroll
          for (int j = 0; j < 4; ++j) tally(o[j]);
        }, nothing);
      __syncthreads();
      // the digit at which the counts from the largest down reach `need`: four counters a thread
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
        // need = 0: the largest digit, of which none stays
        if ((above < need && above + c4[e] >= need) || (need == 0 && tid == 0 && e == 0)) {
          found[0] = count - 1 - 4 * tid - e;
          found[1] = need - above;
        }
        above += c4[e];
      }
      __syncthreads();
      prefix |= (uint32_t)found[0] << shift;
      mask |= (uint32_t)(count - 1) << shift;
      need = found[1];
      if (digit == 0)
        each(0, old, [&](int, const uint32_t (&o)[4]) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((o[j] & mask) == prefix) {
              const int at = atomicAdd(&listed, 1);
              if (at < EVICT_LIST) list[at] = o[j];
            }
        }, nothing);
      __syncthreads();
    }
    least = prefix;
    equals = need;
  }
  int out = 0, same = 0;  // kept before this span, equals of `least` met before it
  for (int s0 = 0; s0 < old; s0 += EVICT_SPAN) {
    const int end = min(old, s0 + EVICT_SPAN);
    __syncthreads();
    // of each 256 tokens, those above `least` and, from 256 on, its equals
    if (tid < 512) hist[tid] = 0;
    __syncthreads();
    each(s0, end, [&](int i, const uint32_t (&o)[4]) {
      int over = 0, eq = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        over += (int)__popcll(__ballot(o[j] > least));
        eq += (int)__popcll(__ballot(o[j] == least));
      }
      if (lane == 0) {
        hist[(i - s0) >> 8] = over;
        hist[256 + ((i - s0) >> 8)] = eq;
      }
    }, nothing);
    __syncthreads();
    int all_eq, all;
    const int eq_here = tid < 256 ? hist[256 + tid] : 0;
    const int eq_before = same + scan_before(eq_here, waves, &all_eq);
    const int stay = (tid < 256 ? hist[tid] : 0) + max(0, min(eq_here, equals - eq_before));
    const int before = out + scan_before(stay, waves, &all);
    if (tid < 256) {
      hist[tid] = before;
      hist[256 + tid] = equals - eq_before;  // so many of its equals stay
    }
    int done = out;  // written
    uint16_t* staged = reinterpret_cast<uint16_t*>(list);  // of one step: STEP entries
    static_assert(STEP * 2 <= EVICT_LIST * 4 && EVICT_SPAN <= 65536, "staging");
    same += all_eq;
    out += all;
    __syncthreads();
    auto below = [&](bool b) {  // lanes before this one with b
      const uint64_t m = __ballot(b);
      return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    };
    each(s0, end, [&](int i, const uint32_t (&o)[4]) {
      const int at = __builtin_amdgcn_readfirstlane((i - s0) >> 8), cut = __builtin_amdgcn_readfirstlane(hist[256 + at]);
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
      int to = hist[at] - done;
#pragma unroll
      for (int j = 0; j < 4; ++j) to += below(stays[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (stays[j]) staged[to] = (uint16_t)(i + j - s0);
        to += stays[j];
      }
    }, [&](int i0) {
      // what stays of this step, from LDS: side by side, where each lane's own stores took most of the pass
      const int next = (i0 - s0 + STEP) >> 8, upto = i0 + STEP < end ? hist[next] : out;
      __syncthreads();
      for (int x = tid; x < upto - done; x += EVICT_THREADS) {
        const int i = s0 + staged[x];
        kept[done + x] = i;
        weights[done + x] = w[i];
      }
      __syncthreads();
      done = upto;
    });
  }
  for (int i = out + tid; i < keep; i += EVICT_THREADS) {  // the latest, and past the last
    const int from = old + i - out;
    kept[i] = from < n ? from : -1;
    weights[i] = from < n ? w[from] : 0.f;
  }
}

// The kept tokens of each (sequence, head) to the new pages in order: codes and scales as they are.
// A workgroup takes 4096 / DIM destinations, whose rows and sources' rows it looks up once; k's rows
// move 16 bytes a thread, v's slices are put together where they go (a thread gathers one slice of a
// block of tokens) and the scales in v_scales' order.
template <int DIM>
__global__ __launch_bounds__(256) void kv4_move_kernel(Kv4 c, Kv4 to, const int* __restrict__ kept, int keep,
                                                       int blocks) {
  using At = Kv4At<DIM>;
  constexpr int TB = At::TB, CB = At::CB, TOK = 4096 / DIM;
  __shared__ long long from[TOK], dest[TOK];  // rows in the arrays; a source of -1: nothing to move
  __shared__ int from_off[TOK], dest_off[TOK];
  const int bh = blockIdx.x / blocks, t0 = (blockIdx.x - bh * blocks) * TOK;
  const int b = bh / c.heads, h = bh - b * c.heads, tid = threadIdx.x;
  if (tid < TOK) {
    const int i = t0 + tid, src = i < keep ? kept[(size_t)bh * keep + i] : -1;
    long long row = -1;
    if (src >= 0) {
      const int si = fdiv(src, c.by_page.mul, c.by_page.shift), di = fdiv(i, c.by_page.mul, c.by_page.shift);
      const int sp = kv4_page(c, b, si), dp = kv4_page(to, b, di);
      from_off[tid] = src - si * c.page;
      dest_off[tid] = i - di * c.page;
      if (sp >= 0 && dp >= 0) {
        row = (long long)At::row(c, sp, h, from_off[tid]);
        dest[tid] = (long long)At::row(c, dp, h, dest_off[tid]);
      }
    }
    from[tid] = row;
  }
  __syncthreads();
  if (tid < 128) {  // k: 16 bytes
    const int t = tid / (DIM / 32), q = tid % (DIM / 32);
    if (from[t] >= 0)
      *reinterpret_cast<uint4*>(c.k + At::k(dest[t]) + 16 * q) = *reinterpret_cast<const uint4*>(c.k + At::k(from[t]) + 16 * q);
  } else {  // v: a slice of TB tokens, CB bytes each
    const int t = (tid - 128) / 16 * TB, s = tid % 16;
#pragma unroll
    for (int e = 0; e < TB; ++e)
      if (from[t + e] >= 0) {
        const uint8_t* p = c.v + At::v(from[t + e], from_off[t + e], s);
        uint8_t* at = c.v + At::v(dest[t + e], dest_off[t + e], s);
        if constexpr (DIM == 128) *reinterpret_cast<uint32_t*>(at) = *reinterpret_cast<const uint32_t*>(p);
        else *reinterpret_cast<uint16_t*>(at) = *reinterpret_cast<const uint16_t*>(p);
      }
  }
  if (tid < TOK * CB) {
    const int t = tid % TOK, s = tid / TOK;
    if (from[t] >= 0) {
      c.vs[At::vs(dest[t], dest_off[t], s)] = c.vs[At::vs(from[t], from_off[t], s)];
      c.ks[At::ks(dest[t], dest_off[t], s)] = c.ks[At::ks(from[t], from_off[t], s)];
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
  if (B * c.heads * blocks > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)(B * c.heads * blocks);
  if (cache->dim == 128) kv4_read_kernel<128><<<grid, 256, 0, st>>>(c, lens, (int)most, (int)blocks, k, v);
  else kv4_read_kernel<64><<<grid, 256, 0, st>>>(c, lens, (int)most, (int)blocks, k, v);
  return check_launch(what);
}

int bq_kv4_evict(const bq_kv4_cache* cache, const float* sums, int64_t sums_b, int64_t sums_h, int64_t most, const int32_t* table, int64_t B,
                 int64_t width, const int32_t* lens, const int32_t* new_table, int64_t new_width, int64_t keep,
                 int64_t recent, int32_t* kept, float* weights, int32_t* left, bq_stream_t stream) {
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
  if (B * c.heads * blocks > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  hipStream_t st = (hipStream_t)stream;
  kv4_select_kernel<<<(unsigned)(B * c.heads), EVICT_THREADS, 0, st>>>(sums, sums_b, sums_h, (int)most, c.heads, lens,
                                                                       (int)keep, (int)recent, kept, weights, left);
  if (const int rc = check_launch(what)) return rc;
  const unsigned grid = (unsigned)(B * c.heads * blocks);
  if (c.pages == 0) return BQ_OK;
  if (cache->dim == 128) kv4_move_kernel<128><<<grid, 256, 0, st>>>(c, to, kept, (int)keep, (int)blocks);
  else kv4_move_kernel<64><<<grid, 256, 0, st>>>(c, to, kept, (int)keep, (int)blocks);
  return check_launch(what);
}
