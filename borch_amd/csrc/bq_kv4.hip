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
template <typename T, int DIM>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4 c, const T* __restrict__ nk, const T* __restrict__ nv,
                                                         int64_t kt, int64_t kh, int64_t vt, int64_t vh, int first,
                                                         uint32_t items, FastDiv per_token, const int* __restrict__ lens,
                                                         const int* __restrict__ cu, int B) {
  using At = Kv4At<DIM>;
  constexpr int P = DIM / 8;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  if (id >= items) return;  // whole rows: items is a multiple of P
  int i = fdiv((int)id, per_token.mul, per_token.shift);
  int rest = (int)id - i * (2 * c.heads * P);
  i += first;
  const int piece = rest % P;
  rest /= P;
  const bool is_v = rest >= c.heads;
  const int h = is_v ? rest - c.heads : rest;
  const v8f x = load8(is_v ? nv + i * vt + h * vh + 8 * piece : nk + i * kt + h * kh + 8 * piece);
  int lo = 0, hi = B;  // the sequence: the last b with cu[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] <= i) lo = mid + 1;
    else hi = mid;
  }
  uint32_t peak = 0;  // |x| as integers: ordered as the values, NaN above infinity
#pragma unroll
  for (int e = 0; e < 8; ++e) peak = max(peak, __float_as_uint(x[e]) & 0x7fffffffu);
  peak = max(peak, (uint32_t)__shfl_xor((int)peak, 1));
  peak = max(peak, (uint32_t)__shfl_xor((int)peak, 2));
  if (lo >= B) return;  // past the last sequence
  const int64_t pos = (int64_t)lens[lo] - cu[lo + 1] + i;
  if (pos < 0 || pos >= (int64_t)c.width * c.page) return;
  const int pi = fdiv((int)pos, c.by_page.mul, c.by_page.shift);
  const int at = kv4_page(c, lo, pi), off = (int)pos - pi * c.page;
  if (at < 0) return;

  const bool finite = peak < 0x7f800000u;
  int byte = (int)((peak + 0x3fffffu) >> 23) - 2;  // E - 2, one more above 1.5 2^E
  byte = finite ? max(byte, 1) : 255;
  uint32_t code = 0;
  if (finite) {
    const float r = __uint_as_float((uint32_t)(254 - byte) << 23);  // 2^(127 - byte), byte <= 253
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, __fmul_rn(x[0], r), __fmul_rn(x[1], r), 1.0f, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, __fmul_rn(x[2], r), __fmul_rn(x[3], r), 1.0f, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, __fmul_rn(x[4], r), __fmul_rn(x[5], r), 1.0f, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, __fmul_rn(x[6], r), __fmul_rn(x[7], r), 1.0f, 3);
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

// A weight's place in the order: larger first as unsigned integers; -0 with 0, NaN above all.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (__builtin_isnan(w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(__fadd_rn(w, 0.f));
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of `v` over the workgroup's threads before this one; *all gets the sum of all.
__device__ __forceinline__ int scan_before(int v, int* waves, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, count = blockDim.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int before = 0, total = 0;
  for (int i = 0; i < count; ++i) {
    if (i < wave) before += waves[i];
    total += waves[i];
  }
  *all = total;
  return before + x - v;
}

// Which tokens stay, one workgroup a (sequence, head): the `recent` last ones, and of the others
// the keep - recent of largest weight, ties to the earlier token. A radix select from the top
// byte of order_of finds the least weight that stays and how many of its equals do; a pass in
// order then writes the places and weights.
constexpr int EVICT_THREADS = 1024;
__global__ __launch_bounds__(EVICT_THREADS) void kv4_select_kernel(const float* __restrict__ sums, int64_t sums_b,
                                                                   int64_t sums_h, int most, int heads, const int* __restrict__ lens,
                                                                   int keep, int recent, int* __restrict__ kept,
                                                                   float* __restrict__ weights, int* __restrict__ left) {
  __shared__ int hist[256], waves[EVICT_THREADS / 64], found[2];
  const int bh = blockIdx.x, b = bh / heads, tid = threadIdx.x;
  const int n = max(0, min(lens[b], most));
  const float* w = sums + b * sums_b + (bh - b * heads) * sums_h;
  kept += (size_t)bh * keep;
  weights += (size_t)bh * keep;
  if (bh % heads == 0 && tid == 0) left[b] = min(n, keep);
  uint32_t least = 0;      // weights above this stay
  int equals = 0x7fffffff;  // and so many that equal it
  const int old = n > keep ? n - recent : n;
  if (n > keep) {
    int need = keep - recent;
    uint32_t prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += EVICT_THREADS) {
        const uint32_t u = order_of(w[i]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {  // from the largest digit down
        int d = 255, rest = need;
        while (d > 0 && hist[d] < rest) rest -= hist[d--];
        found[0] = d;
        found[1] = rest;
      }
      __syncthreads();
      prefix |= (uint32_t)found[0] << shift;
      mask |= 255u << shift;
      need = found[1];
      __syncthreads();
    }
    least = prefix;
    equals = need;
  }
  int out = 0, same = 0;  // kept so far, equals of `least` met so far
  for (int i0 = 0; i0 < n; i0 += EVICT_THREADS) {
    const int i = i0 + tid;
    int stays = 0;
    float x = 0.f;
    if (n <= keep) {
      if (i < n) stays = 1, x = w[i];
    } else {
      uint32_t u = 0;
      if (i < n) x = w[i], u = order_of(x);
      int all;
      const int eq = i < old && u == least;
      const int rank = same + scan_before(eq, waves, &all);
      same += all;
      stays = i < n && (i >= old || u > least || (eq && rank < equals));
    }
    int all;
    const int to = out + scan_before(stays, waves, &all);
    out += all;
    if (stays && to < keep) {
      kept[to] = i;
      weights[to] = x;
    }
  }
  for (int i = out + tid; i < keep; i += EVICT_THREADS) {
    kept[i] = -1;
    weights[i] = 0.f;
  }
}

// The kept tokens of each (sequence, head) to the new pages in order: codes and scales as they are.
template <int DIM>
__global__ __launch_bounds__(256) void kv4_move_kernel(Kv4 c, Kv4 to, const int* __restrict__ kept, int keep,
                                                       int blocks) {
  using At = Kv4At<DIM>;
  constexpr int P = DIM / 8, TOKENS = 256 / P;
  const int bh = blockIdx.x / blocks, i = (blockIdx.x - bh * blocks) * TOKENS + threadIdx.x / P;
  if (i >= keep) return;
  const int b = bh / c.heads, h = bh - b * c.heads, piece = threadIdx.x % P;
  const int src = kept[(size_t)bh * keep + i];
  if (src < 0) return;
  const int si = fdiv(src, c.by_page.mul, c.by_page.shift), di = fdiv(i, c.by_page.mul, c.by_page.shift);
  const int sp = kv4_page(c, b, si), dp = kv4_page(to, b, di);
  if (sp < 0 || dp < 0) return;
  const int so = src - si * c.page, dof = i - di * c.page;
  const size_t sr = At::row(c, sp, h, so), dr = At::row(c, dp, h, dof);
  *reinterpret_cast<uint32_t*>(c.k + At::k(dr) + 4 * piece) = *reinterpret_cast<const uint32_t*>(c.k + At::k(sr) + 4 * piece);
  if constexpr (DIM == 128) {
    *reinterpret_cast<uint32_t*>(c.v + At::v(dr, dof, piece)) = *reinterpret_cast<const uint32_t*>(c.v + At::v(sr, so, piece));
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<uint16_t*>(c.v + At::v(dr, dof, 2 * piece + e)) =
          *reinterpret_cast<const uint16_t*>(c.v + At::v(sr, so, 2 * piece + e));
  }
  if (piece < DIM / 32) {
    c.ks[At::ks(dr, dof, piece)] = c.ks[At::ks(sr, so, piece)];
    c.vs[At::vs(dr, dof, piece)] = c.vs[At::vs(sr, so, piece)];
  }
}

template <typename T, int DIM>
static void append_of(const Kv4& c, const void* nk, const void* nv, int64_t n, int64_t kt, int64_t kh, int64_t vt,
                      int64_t vh, const int* lens, const int* cu, int B, hipStream_t st) {
  const int64_t per = 2 * (int64_t)c.heads * (DIM / 8);
  const int64_t most = 0x70000000 / per;  // tokens a launch
  const FastDiv by = fast_div((uint32_t)per);
  for (int64_t first = 0; first < n; first += most) {
    const int64_t items = (n - first < most ? n - first : most) * per;
    kv4_append_kernel<T, DIM><<<(unsigned)((items + 255) / 256), 256, 0, st>>>(
        c, (const T*)nk, (const T*)nv, kt, kh, vt, vh, (int)first, (uint32_t)items, by, lens, cu, B);
  }
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
  const int64_t blocks = (keep + 255 / (cache->dim / 8)) / (256 / (cache->dim / 8));
  if (B * c.heads * blocks > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  hipStream_t st = (hipStream_t)stream;
  kv4_select_kernel<<<(unsigned)(B * c.heads), EVICT_THREADS, 0, st>>>(sums, sums_b, sums_h, (int)most, c.heads, lens, (int)keep,
                                                                       (int)recent, kept, weights, left);
  if (const int rc = check_launch(what)) return rc;
  const unsigned grid = (unsigned)(B * c.heads * blocks);
  if (c.pages == 0) return BQ_OK;
  if (cache->dim == 128) kv4_move_kernel<128><<<grid, 256, 0, st>>>(c, to, kept, (int)keep, (int)blocks);
  else kv4_move_kernel<64><<<grid, 256, 0, st>>>(c, to, kept, (int)keep, (int)blocks);
  return check_launch(what);
}
