// Softmax attention over whole prompts: sequences of different lengths packed one after another,
// causal or not, each key-value head shared by a group of query heads; f32, bf16 and f16, heads of
// 64 or 128. out = sum_i p_i v_i over the sequence's tokens i (causal: up to the query's own), p =
// softmax(scale q . k_i).
//
// One pass over the keys with each query's running maximum and sum. A workgroup of four waves takes
// 128 queries of one head, 32 a wave, and walks the keys in tiles staged in LDS. The scores are
// computed transposed, S^T = k q^T on the 32 x 32 x 16 MFMA, so that lane l holds scores of query
// l % 32 alone (tokens 8 (i / 4) + 4 (l / 32) + i % 4 in register i): maxima and sums are over the
// lane's own registers and its one partner lane, and the exponentials are, register for register,
// the second operand of O^T = v^T p^T: its contracted index (tokens) is permuted to suit, groups of
// 4 tokens each, which is what the transposing LDS read takes of v's rows.
//
// The 16-bit types multiply as they are and p is rounded to their type (half a step of 2^-8 or
// 2^-11 on each term, where the output takes one as large). f32 operands are the exact sums of
// three bf16 pieces (bq_bf16x3.h), of whose nine products the six of weight 2^-18 and above are
// added. What the pieces cannot hold is taken apart: a score that is not finite is computed again
// in plain f32, a value that is not finite leaves the products (nonfinite_values).
#include <math.h>

#include "bq_bf16x3.h"
#include "bq_common.h"

namespace bq {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v8s __attribute__((ext_vector_type(8)));

constexpr int PROMPT_ROWS = 128;  // queries a workgroup
constexpr int PROMPT_WAVES = 4;

struct Prompt {
  const void *q, *k, *v;
  void* out;
  int64_t qt, qh, kt, kh, vt, vh;  // strides in elements
  const int* cu;
  int n, B, heads, group, tiles, causal;
  float scale2;  // scale * log2(e)
};

template <typename T>
struct Kind;
template <>
struct Kind<float> {
  static constexpr int P = 3, KT = 32;  // pieces, keys a tile
};
template <>
struct Kind<__bf16> {
  static constexpr int P = 1, KT = 64;
};
template <>
struct Kind<_Float16> {
  static constexpr int P = 1, KT = 64;
};

template <int P>
struct Frag {
  v8s p[P];
};

template <typename T>
__device__ __forceinline__ v16f mma(v8s a, v8s b, v16f c) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ v16f product(const Frag<Kind<T>::P>& a, const Frag<Kind<T>::P>& b, v16f c) {
  if constexpr (Kind<T>::P == 3) {  // the smallest first
    c = mma<T>(a.p[2], b.p[0], c);
    c = mma<T>(a.p[1], b.p[1], c);
    c = mma<T>(a.p[0], b.p[2], c);
    c = mma<T>(a.p[1], b.p[0], c);
    c = mma<T>(a.p[0], b.p[1], c);
  }
  return mma<T>(a.p[0], b.p[0], c);
}

// Eight floats as one operand.
template <typename T>
__device__ __forceinline__ Frag<Kind<T>::P> frag_of(const float x[8]) {
  Frag<Kind<T>::P> f;
  if constexpr (__is_same(T, _Float16)) {
    v8h h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
    f.p[0] = __builtin_bit_cast(v8s, h);
  } else if constexpr (__is_same(T, __bf16)) {
    f.p[0] = __builtin_bit_cast(v8s, make_uint4(bf2(x[0], x[1]), bf2(x[2], x[3]), bf2(x[4], x[5]), bf2(x[6], x[7])));
  } else {
    const Split8 s = split8(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
    f.p[0] = __builtin_bit_cast(v8s, s.p1);
    f.p[1] = __builtin_bit_cast(v8s, s.p2);
    f.p[2] = __builtin_bit_cast(v8s, s.p3);
  }
  return f;
}

// Eight elements as loaded.
template <typename T>
struct Piece {
  uint4 x[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
    x[0] = *reinterpret_cast<const uint4*>(p);
    if constexpr (sizeof(T) == 4) x[1] = *reinterpret_cast<const uint4*>(p + 4);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint4& v : x) v = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ Frag<Kind<T>::P> frag() const {
    if constexpr (sizeof(T) == 4) {
      const float y[8] = {__uint_as_float(x[0].x), __uint_as_float(x[0].y), __uint_as_float(x[0].z), __uint_as_float(x[0].w),
                          __uint_as_float(x[1].x), __uint_as_float(x[1].y), __uint_as_float(x[1].z), __uint_as_float(x[1].w)};
      return frag_of<T>(y);
    } else {
      return Frag<1>{{__builtin_bit_cast(v8s, x[0])}};
    }
  }
  // Whether an element's exponent is all ones.
  __device__ __forceinline__ bool odd() const {
    bool bad = false;
#pragma unroll
    for (const uint4& v : x) {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
        } else {
          constexpr uint32_t E = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
          bad |= (w[i] & E) == E || (w[i] & (E << 16)) == (E << 16);
        }
      }
    }
    return bad;
  }
};

// Where a 16-byte piece of a row lies in a staged tile. k's rows are read 16 at a time at one
// piece, v's four at a time over four pieces (64 bytes): XORed so that either covers all 64 banks.
template <int DIM>
__device__ __forceinline__ int k_at(int row, int piece) {
  return DIM == 128 ? row * 256 + ((piece ^ (row & 15)) << 4) : row * 128 + ((piece ^ ((row >> 1) & 7)) << 4);
}
template <int DIM>
__device__ __forceinline__ int v_at(int row, int piece) {
  return DIM == 128 ? row * 256 + ((piece ^ ((row & 3) << 2)) << 4) : row * 128 + ((piece ^ ((row & 2) << 1)) << 4);
}

typedef __attribute__((address_space(3))) v4s* lds_v4s;
__device__ __forceinline__ v4s read_tr(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(const __attribute__((address_space(3))) unsigned char*)p);
}

template <typename T, int DIM>
struct PromptTile {
  static constexpr int P = Kind<T>::P, KT = Kind<T>::KT, PLANE = KT * DIM * 2, STEPS = DIM / 16, VT = DIM / 32;
  static constexpr int PER = KT * DIM / 8 / (PROMPT_WAVES * 64);  // pieces a thread
  unsigned char k[P * PLANE], v[P * PLANE];
  int odd[2];  // whether v's tile holds a value that is not finite, tiles in turn

  // v's operand of 32 channels from 32 d, tokens of step s: lane l is channel 32 d + l % 32
  __device__ __forceinline__ Frag<P> v_frag(int d, int s) const {
    const int lane = threadIdx.x & 63;
    const int row = 16 * s + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), half = (lane & 1) * 8;
    Frag<P> f;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      const v4s a = read_tr(v + e * PLANE + v_at<DIM>(row, piece) + half);
      const v4s b = read_tr(v + e * PLANE + v_at<DIM>(row + 8, piece) + half);
      f.p[e] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }
};

// The scores of a lane that did not come out finite, in plain f32: infinities and NaN among q and k
// as f32 gives them.
__device__ __attribute__((noinline)) void plain_scores(const float* q, const float* k, int64_t kt, int dim, int tokens,
                                                       int half, float* s) {
  for (int i = 0; i < 16; ++i) {
    const int t = 8 * (i / 4) + 4 * half + i % 4;
    if (t >= tokens || __builtin_isfinite(s[i])) continue;
    float x = 0.f;
    for (int d = 0; d < dim; ++d) x = __fmaf_rn(q[d], k[t * kt + d], x);
    s[i] = x;
  }
}

template <typename T, int DIM>
__global__ __launch_bounds__(PROMPT_WAVES * 64, 2) void prompt_kernel(Prompt a) {
  using Tile = PromptTile<T, DIM>;
  constexpr int P = Tile::P, KT = Tile::KT, STEPS = Tile::STEPS, VT = Tile::VT, PER = Tile::PER, SUB = KT / 32;
  __shared__ __attribute__((aligned(16))) Tile tile;
  const int heads = a.heads * a.group;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, hh = lane >> 5;

  // this workgroup's head and place: places from the last down (the causal ones with most keys
  // first); with a multiple of 8 heads each XCD (ids modulo 8) keeps to its own
  int head = blockIdx.x % heads;
  if (heads % 8 == 0) head = (head % 8) * (heads / 8) + head / 8;
  int place = a.tiles - 1 - blockIdx.x / heads;
  // the sequence: tiles of what lies before cu[0], of each sequence, of what lies past the last
  // (those rows see nothing)
  int start = 0, end = 0, kv = 0;
  for (int base = 0; base < a.B + 2; base += 64) {
    const int i = base + lane;
    int s = 0, e = 0;
    if (i <= a.B + 1) {
      s = i == 0 ? 0 : min(max(a.cu[i - 1], 0), a.n);
      e = i == a.B + 1 ? a.n : min(max(a.cu[i], 0), a.n);
    }
    const int mine = max(0, e - s + PROMPT_ROWS - 1) / PROMPT_ROWS;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
    const uint64_t hit = __ballot(upto > place);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      place -= __shfl(upto - mine, at);
      start = __shfl(s, at);
      end = __shfl(e, at);
      kv = base + at > 0 && base + at <= a.B;
      break;
    }
    place -= __shfl(upto, 63);
    if (base + 64 >= a.B + 2) return;  // fewer tiles than the grid has
  }
  const int len = end - start, q0 = place * PROMPT_ROWS;
  const int qw = q0 + wave * 32, row = qw + n;  // the wave's first query, this lane's
  const int h = head / a.group;
  const T* q = (const T*)a.q + (int64_t)(start + row) * a.qt + head * a.qh;
  const T* k = (const T*)a.k + (int64_t)start * a.kt + h * a.kh;
  const T* v = (const T*)a.v + (int64_t)start * a.vt + h * a.vh;

  Frag<P> qf[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    Piece<T> x;
    x.clear();
    if (row < len) x.load(q + 16 * s + 8 * hh);
    qf[s] = x.frag();
  }
  const int keys = !kv ? 0 : a.causal ? min(len, q0 + PROMPT_ROWS) : len;  // that the workgroup sees
  const int wkeys = a.causal ? min(keys, qw + 32) : keys;                  // that the wave does
  const int sees = a.causal ? min(len, row + 1) : len;                     // that the lane does
  float m = -INFINITY, l = 0.f;
  v16f o[VT];
#pragma unroll
  for (int d = 0; d < VT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

  Piece<T> kr[PER], vr[PER];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int x = threadIdx.x + e * PROMPT_WAVES * 64, r = x / (DIM / 8), c = x % (DIM / 8);
      kr[e].clear();
      vr[e].clear();
      if (t0 + r < len) {
        kr[e].load(k + (int64_t)(t0 + r) * a.kt + 8 * c);
        vr[e].load(v + (int64_t)(t0 + r) * a.vt + 8 * c);
      }
    }
  };
  if (threadIdx.x < 2) tile.odd[threadIdx.x] = 0;
  if (keys > 0) fetch(0);
  for (int t0 = 0, turn = 0; t0 < keys; t0 += KT, turn ^= 1) {
    __syncthreads();  // the last tile is read, its flag too
    bool odd = false;
    // f32 asks of every tile, the others of those that a query sees in part
    const bool part = t0 + KT > len || (a.causal && t0 + KT > q0 + 1);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int x = threadIdx.x + e * PROMPT_WAVES * 64, r = x / (DIM / 8), c = x % (DIM / 8);
      const Frag<P> kf = kr[e].frag(), vf = vr[e].frag();
#pragma unroll
      for (int p = 0; p < P; ++p) {
        *reinterpret_cast<v8s*>(tile.k + p * Tile::PLANE + k_at<DIM>(r, c)) = kf.p[p];
        *reinterpret_cast<v8s*>(tile.v + p * Tile::PLANE + v_at<DIM>(r, c)) = vf.p[p];
      }
      if (P == 3 || part) odd |= vr[e].odd();
    }
    if (threadIdx.x == 0) tile.odd[turn ^ 1] = 0;
    if (odd) tile.odd[turn] = 1;
    __syncthreads();
    if (t0 + KT < keys) fetch(t0 + KT);
    if (t0 >= wkeys) continue;

    // S^T = k q^T
    v16f s[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
      for (int e = 0; e < STEPS; ++e) {
        Frag<P> kf;
#pragma unroll
        for (int p = 0; p < P; ++p)
          kf.p[p] = *reinterpret_cast<const v8s*>(tile.k + p * Tile::PLANE + k_at<DIM>(32 * u + n, 2 * e + hh));
        s[u] = product<T>(kf, qf[e], s[u]);
      }
    }
    if constexpr (P == 3) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        float zero = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = __fmaf_rn(s[u][i], 0.f, zero);
        if (zero != 0.f && row < len) {
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = s[u][i];
          plain_scores((const float*)q, (const float*)k + (int64_t)(t0 + 32 * u) * a.kt, a.kt, DIM, len - t0 - 32 * u, hh, x);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[u][i] = x[i];
        }
      }
    }

    // softmax, one step
    const bool edge = t0 + KT > len || (a.causal && t0 + KT > qw + 1);
    if (edge)
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t0 + 32 * u + 8 * (i / 4) + 4 * hh + i % 4 >= sees) s[u][i] = -INFINITY;
    float top = m;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
    top = fmaxf(top, __shfl_xor(top, 32));
    const float base = top == -INFINITY ? 0.f : top;
    if (__any(top > m)) {
      const float f = __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(m, base), a.scale2));
      l = __fmul_rn(l, f);
#pragma unroll
      for (int d = 0; d < VT; ++d) o[d] *= f;
      m = top;
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(s[u][i], base), a.scale2));
        l = __fadd_rn(l, s[u][i]);
      }

    // O^T += v^T p^T
    const bool taint = tile.odd[turn] != 0;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = s[u][8 * e + i];
        const Frag<P> pf = frag_of<T>(x);
        if (!taint) {
#pragma unroll
          for (int d = 0; d < VT; ++d) o[d] = product<T>(tile.v_frag(d, 2 * u + e), pf, o[d]);
        } else {
          // Values that are not finite leave the product, where they would meet the zeros of
          // tokens that a query does not see (and, in f32, pieces of either sign); what they come
          // to is counted by products of ones: infinities that meet a weight, by sign, and NaN (a
          // NaN that is seen, an infinity that meets a weight of 0).
          constexpr short ONE = __is_same(T, _Float16) ? 0x3c00 : 0x3f80;
          constexpr short E = __is_same(T, _Float16) ? 0x7c00 : 0x7f80;
          v8s seen, met, none;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int t = t0 + 32 * u + 16 * e + 8 * (i / 4) + 4 * hh + i % 4;
            seen[i] = t < sees ? ONE : 0;
            met[i] = t < sees && x[i] > 0.f ? ONE : 0;
            none[i] = t < sees && !(x[i] > 0.f) ? ONE : 0;
          }
#pragma unroll
          for (int d = 0; d < VT; ++d) {
            Frag<P> vf = tile.v_frag(d, 2 * u + e);
            v8s plus, minus, nan, inf;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const short y = vf.p[0][i], mag = y & 0x7fff;
              plus[i] = y == E ? ONE : 0;
              minus[i] = mag == E && y != E ? ONE : 0;
              inf[i] = mag == E ? ONE : 0;
              nan[i] = mag > E ? ONE : 0;
              if (mag >= E)
#pragma unroll
                for (int p = 0; p < P; ++p) vf.p[p][i] = 0;
            }
            o[d] = product<T>(vf, pf, o[d]);
            v16f zero;
#pragma unroll
            for (int i = 0; i < 16; ++i) zero[i] = 0.f;
            const v16f cp = mma<T>(plus, met, zero), cm = mma<T>(minus, met, zero);
            const v16f cn = mma<T>(inf, none, mma<T>(nan, seen, zero));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (cp[i] > 0.f) o[d][i] = __fadd_rn(o[d][i], INFINITY);
              if (cm[i] > 0.f) o[d][i] = __fadd_rn(o[d][i], -INFINITY);
              if (cn[i] > 0.f) o[d][i] = NAN;
            }
          }
        }
      }
  }

  l = __fadd_rn(l, __shfl_xor(l, 32));
  if (row >= len) return;
  const float d1 = l == 0.f ? 1.f : l;
  T* to = (T*)a.out + ((int64_t)(start + row) * heads + head) * DIM + 4 * hh;
#pragma unroll
  for (int d = 0; d < VT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y[4] = {__fdiv_rn(o[d][4 * i], d1), __fdiv_rn(o[d][4 * i + 1], d1), __fdiv_rn(o[d][4 * i + 2], d1),
                          __fdiv_rn(o[d][4 * i + 3], d1)};
      T* at = to + 32 * d + 8 * i;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(at) = make_float4(y[0], y[1], y[2], y[3]);
      } else if constexpr (__is_same(T, __bf16)) {
        *reinterpret_cast<uint2*>(at) = make_uint2(bf2(y[0], y[1]), bf2(y[2], y[3]));
      } else {
        typedef _Float16 v4h __attribute__((ext_vector_type(4)));
        *reinterpret_cast<v4h*>(at) = v4h{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
      }
    }
}

}  // namespace bq

using namespace bq;

int bq_prompt_attention(const void* q, const void* k, const void* v, int type, int64_t n, int64_t q_heads,
                        int64_t heads, int64_t dim, int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head,
                        int64_t v_token, int64_t v_head, const int32_t* cu, int64_t B, int causal, float scale,
                        void* out, bq_stream_t stream) {
  const char* what = "bq_prompt_attention";
  if (type < 0 || type > 2) return set_error(BQ_ERR_ARG, "%s: type %d", what, type);
  if (dim != 64 && dim != 128)
    return set_error(BQ_ERR_UNSUPPORTED, "%s: head width %lld (64 or 128)", what, (long long)dim);
  if (n < 0 || n > 0x7fffffff - 8192 || heads < 1 || q_heads < 1 || q_heads > 65535 || B < 0 || B > 0x7fffff)
    return set_error(BQ_ERR_ARG, "%s: bad sizes", what);
  if (q_heads % heads)
    return set_error(BQ_ERR_ARG, "%s: %lld query heads over %lld key-value heads", what, (long long)q_heads,
                     (long long)heads);
  if (!(scale > 0.f) || !(scale < 1e30f)) return set_error(BQ_ERR_ARG, "%s: scale %g", what, (double)scale);
  if (n == 0) return BQ_OK;
  if (!q || !k || !v || !cu || !out) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const int64_t size = type == 0 ? 4 : 2;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) ||
      (q_token | q_head | k_token | k_head | v_token | v_head) * size % 16)
    return set_error(BQ_ERR_ARG, "%s: rows that are not 16-byte aligned", what);
  // whatever the lengths are: a full tile for every 128 rows and one begun for each sequence
  const int64_t tiles = n / PROMPT_ROWS + (B + 2 < n ? B + 2 : n);
  if (tiles * q_heads > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  const Prompt a = {q, k, v, out, q_token, q_head, k_token, k_head, v_token, v_head, cu, (int)n, (int)B, (int)heads,
                    (int)(q_heads / heads), (int)tiles, causal ? 1 : 0, scale * 1.4426950408889634f};
  const unsigned grid = (unsigned)(tiles * q_heads);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = dim == 128;
#define BQ_PROMPT(T)                                                                        \
  (wide ? prompt_kernel<T, 128><<<grid, PROMPT_WAVES * 64, 0, st>>>(a)                      \
        : prompt_kernel<T, 64><<<grid, PROMPT_WAVES * 64, 0, st>>>(a))
  if (type == 0) BQ_PROMPT(float);
  else if (type == 1) BQ_PROMPT(__bf16);
  else BQ_PROMPT(_Float16);
#undef BQ_PROMPT
  return check_launch(what);
}
