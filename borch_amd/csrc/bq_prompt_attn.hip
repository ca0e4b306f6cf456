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
// The 16-bit types multiply as they are and p is rounded to their type: half a step of 2^-8 or 2^-11 on each
// term, where the output takes one as large (bf16, 8192 tokens: 2.1e-3 from float64 in the mean, 1.6e-3 by the
// output's rounding alone). p in two pieces would leave the output's rounding alone and take half as much
// matrix work again (8192 tokens 544 -> 706 us, 2048 and 1111 48 -> 55, 4096 of 64 channels 88 -> 117).
//
// In f32 p and v are the exact sums of three bf16 pieces (bq_bf16x3.h), of whose nine products the six of
// weight 2^-18 and above are added: a small weight on a large value keeps its bits. In the scores only
// the sum over the channels counts, so q and k are two fp16 pieces each, 22 bits below a power of two of
// their row (what a channel 2^-14 of the row's largest loses is 2^-38 of that largest), and of the four
// products three are added: half the matrix work of the bf16 pieces, each product within 3 2^-22. Taken again
// in plain f32 (plain_row) are outputs that do not come out finite, so that infinities and NaN act as f32 has
// them, and only on the queries that see them; in f32 those below 2^-109 (zero aside), where the up to 2^-134
// that the pieces take from such a value is more than a rounding, and those for whose scores the 2^-38 could
// count: a channel far above its row over rows that are small there (2^20 in q alone made the scores' error
// twelve times f32's own, 2^30 outputs worthless).
//
// Bound by the MFMAs at the clock that they leave: 8192 tokens, 32 heads of 128 over 8, bf16, causal:
// 520 to 575 us, 0.96 to 1.06 PFLOP/s, where the library's 8192^3 product reaches 1.21; 2048 and 1111
// tokens, 16 heads of 128 over 4, f32: 130 us, nine 16-bit products for two.
#include <math.h>

#include "bq_bf16x3.h"
#include "bq_common.h"
#include "bq_dma.h"

namespace bq {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v8s __attribute__((ext_vector_type(8)));

struct Prompt {
  const void *q, *k, *v;
  void* out;
  int64_t qt, qh, kt, kh, vt, vh;  // strides in elements
  const int* cu;
  int n, B, heads, group, tiles, causal;
  float scale2;    // scale * log2(e)
  void* ws;        // f32: the planes of k, then of v
  int* exponents;  // and of each row of k
};

// A workgroup's head and queries.
struct Place {
  int head, start, len, q0;  // the sequence's first row and length, the first query in it
  bool keys;                 // whether it is a sequence (else rows of none, which see nothing)
};

// Places from the last down (the causal ones with most keys first), the heads of one place side by
// side; with a multiple of 8 heads each XCD (ids modulo 8) keeps to its own. A place is a tile of
// what lies before cu[0], of each sequence in turn, or of what lies past the last. False: the grid
// has more workgroups than there are tiles.
template <int ROWS>  // of a place
__device__ __forceinline__ bool place_of(const Prompt& a, Place* out) {
  const int heads = a.heads * a.group, lane = threadIdx.x & 63;
  int head = blockIdx.x % heads;
  if (heads % 8 == 0) head = (head % 8) * (heads / 8) + head / 8;
  int place = a.tiles - 1 - blockIdx.x / heads;
  for (int base = 0; base < a.B + 2; base += 64) {
    const int i = base + lane;
    int s = 0, e = 0;
    if (i <= a.B + 1) {
      s = i == 0 ? 0 : min(max(a.cu[i - 1], 0), a.n);
      e = i == a.B + 1 ? a.n : min(max(a.cu[i], 0), a.n);
    }
    const int mine = max(0, e - s + ROWS - 1) / ROWS;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
    const uint64_t hit = __ballot(upto > place);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      // one value for the wave, in scalar registers
      const int start = __builtin_amdgcn_readlane(s, at), end = __builtin_amdgcn_readlane(e, at);
      place -= __builtin_amdgcn_readlane(upto - mine, at);
      *out = Place{head, start, end - start, place * ROWS, base + at > 0 && base + at <= a.B};
      return true;
    }
    place -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// f32 prompts of up to this many channels of a head (192 tokens of 64, 96 of 128) are split where they
// are used. With a launch for it and without, us: 102 tokens, 12 heads of 64 16.1, 12.2; 256 tokens
// 22.6, 21.9; 94 tokens, 16 heads of 128 20.1, 16.7; 128 tokens 20.3, 21.8; 512 tokens 43, 61.
constexpr int64_t PROMPT_DIRECT = 12288;

template <typename T>
struct Kind {
  static constexpr int P = sizeof(T) == 4 ? 3 : 1;   // pieces of v and p
  static constexpr int PK = sizeof(T) == 4 ? 2 : 1;  // of k and q
  // The maximum that is subtracted lags by up to 2^LAG, and the row's largest weight is 2^LIFT or more. In fp16
  // weights keep their 11 bits down to 2^-25 of the largest (at 2^0 those below 2^-14 were subnormal: where a
  // first token of values near 0 leads by e^14, outputs were off by 0.3 of their size), and none passes 2^15.5.
  // A lag of 2^4 costs nothing beside one of 2^8: 8192 tokens, 32 heads of 128, 569 and 571 us.
  static constexpr float LAG = __is_same(T, _Float16) ? 4.f : 8.f, LIFT = __is_same(T, _Float16) ? 11.f : 0.f;
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

// The scores' product: two fp16 pieces, the smaller terms first, or one of the 16-bit types.
template <typename T>
__device__ __forceinline__ v16f score(const Frag<Kind<T>::PK>& k, const Frag<Kind<T>::PK>& q, v16f c) {
  if constexpr (Kind<T>::PK == 2) {
    c = mma<_Float16>(k.p[1], q.p[0], c);
    c = mma<_Float16>(k.p[0], q.p[1], c);
    return mma<_Float16>(k.p[0], q.p[0], c);
  } else {
    return mma<T>(k.p[0], q.p[0], c);
  }
}

// The power of two that takes a row's largest magnitude (as bits) to [2^13, 2^14): its exponent. Rows
// that are not finite get any; their products are not finite.
__device__ __forceinline__ int row_exponent(uint32_t peak) { return max((int)(peak >> 23), 1) - 127 - 13; }
constexpr int NO_ROW = -139;  // of a row of zeros
// The largest over the wave.
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false));   // lanes 1 apart
  v = max(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false));   // 2
  v = max(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false));  // mirrored in 8
  v = max(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, false));  // and in 16
  const auto x = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = max((int)x[0], (int)x[1]);
  const auto y = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return max((int)y[0], (int)y[1]);
}
// Two fp16 pieces of x 2^-e.
__device__ __forceinline__ Frag<2> halves(const float x[8], int e) {
  v8h hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __builtin_ldexpf(x[i], -e);
    hi[i] = (_Float16)y;
    lo[i] = (_Float16)__fsub_rn(y, (float)hi[i]);
  }
  return Frag<2>{{__builtin_bit_cast(v8s, hi), __builtin_bit_cast(v8s, lo)}};
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

// Eight elements.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float x[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

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

__device__ __forceinline__ v16f zeros16() {
  v16f z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// v's operand of 32 channels from 32 d, tokens of step s: lane l is channel 32 d + l % 32
template <int DIM, int P>
__device__ __forceinline__ Frag<P> v_frag(const unsigned char* v, int plane, int d, int s) {
  const int lane = threadIdx.x & 63;
  const int row = 16 * s + 4 * (lane >> 5) + ((lane & 15) >> 2);
  const int piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), half = (lane & 1) * 8;
  Frag<P> f;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    const v4s a = read_tr(v + e * plane + v_at<DIM>(row, piece) + half);
    const v4s b = read_tr(v + e * plane + v_at<DIM>(row + 8, piece) + half);
    f.p[e] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// One query's attention by one wave in plain f32, for outputs that are not finite: what infinities
// among q, k and v come to is f32's matter, not that of pieces of either sign or of weights rounded
// to 0. Lane l scores keys l, l + 64, ..., and sums channels l (and l + 64). A score that is NaN or +infinity
// leaves NaN in every channel, whatever follows. A lane takes 16 bytes of its key at a time. Where all
// rows come here, 8192 tokens, 32 heads of 128 over 8, bf16: 1.7 ms for a NaN in the first key, 79 in the
// first value (with the whole row taken channel by channel 104 and 104), beside 0.57 where none is.
template <typename T, int DIM>
__device__ __attribute__((noinline)) void plain_row(const T* q, const T* k, int64_t kt, const T* v, int64_t vt, T* to,
                                                    int sees, float scale2) {
  constexpr int C = DIM / 64, E = 16 / sizeof(T);
  typedef T Piece __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f, o[C] = {};
  for (int t0 = 0; t0 < sees; t0 += 64) {
    const int t = t0 + lane;
    float s = -INFINITY;
    if (t < sees) {
      s = 0.f;
#pragma unroll 4
      for (int d = 0; d < DIM; d += E) {
        const Piece x = *reinterpret_cast<const Piece*>(q + d), y = *reinterpret_cast<const Piece*>(k + t * kt + d);
#pragma unroll
        for (int e = 0; e < E; ++e) s = __fmaf_rn((float)x[e], (float)y[e], s);
      }
    }
    if (__any(!(s < INFINITY))) {
      l = NAN;
      break;
    }
    float top = s;
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    top = fmaxf(top, m);
    const float base = top == -INFINITY ? 0.f : top;
    const float f = __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(m, base), scale2));
    const float p = t < sees ? __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(s, base), scale2)) : 0.f;
    m = top;
    l = __fadd_rn(__fmul_rn(l, f), wave_sum_fixed(p));
    for (int c = 0; c < C; ++c) o[c] = __fmul_rn(o[c], f);
    const int here = min(64, sees - t0);
    for (int j0 = 0; j0 < here; j0 += 16) {  // 16 rows of v on their way at once
      T x[16][C];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        for (int c = 0; c < C; ++c) x[j][c] = v[(t0 + min(j0 + j, here - 1)) * vt + lane + 64 * c];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), j0 + j));
        if (j0 + j < here)
          for (int c = 0; c < C; ++c) o[c] = __fmaf_rn(pj, (float)x[j][c], o[c]);
      }
    }
  }
  for (int c = 0; c < C; ++c) to[lane + 64 * c] = (T)__fdiv_rn(o[c], l == 0.f ? 1.f : l);
}

// The rows' outputs: lane (n, hh) holds channels 32 d + 8 i + 4 hh .. of its query; l is the row's
// sum. Rows with their bit in `again` by plain_row.
template <typename T, int DIM>
__device__ __forceinline__ void store_rows(const Prompt& a, const Place& at, int row, float l, const v16f (&o)[DIM / 32],
                                           uint32_t again) {
  const float r = __fdiv_rn(1.f, l == 0.f ? 1.f : l);
  T* to = (T*)a.out + ((int64_t)(at.start + row) * (a.heads * a.group) + at.head) * DIM + 4 * ((threadIdx.x >> 5) & 1);
  if (row < at.len)
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y[4] = {__fmul_rn(o[d][4 * i], r), __fmul_rn(o[d][4 * i + 1], r), __fmul_rn(o[d][4 * i + 2], r),
                          __fmul_rn(o[d][4 * i + 3], r)};
      T* p = to + 32 * d + 8 * i;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
      } else if constexpr (__is_same(T, __bf16)) {
        *reinterpret_cast<uint2*>(p) = make_uint2(bf2(y[0], y[1]), bf2(y[2], y[3]));
      } else {
        typedef _Float16 v4h __attribute__((ext_vector_type(4)));
        *reinterpret_cast<v4h*>(p) = v4h{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
      }
    }
  const int row0 = __builtin_amdgcn_readfirstlane(row), h = at.head / a.group;
#pragma unroll 1
  for (int i = 0; i < 32; ++i)
    if ((again >> i) & 1) {
      const int64_t q = at.start + row0 + i;
      const T* k = (const T*)a.k + (int64_t)at.start * a.kt + h * a.kh;
      const T* v = (const T*)a.v + (int64_t)at.start * a.vt + h * a.vh;
      plain_row<T, DIM>((const T*)a.q + q * a.qt + at.head * a.qh, k, a.kt, v, a.vt,
                        (T*)a.out + (q * (a.heads * a.group) + at.head) * DIM,
                        a.causal ? min(at.len, row0 + i + 1) : at.len, a.scale2);
    }
}

// Takes the values that are not finite out of a staged tile of v, which some query sees in part (they
// would meet that query's weights of 0), and returns whether the lane's query sees one: it sees
// the tile's first `sees` tokens. By the whole workgroup; found [KT].
template <typename T, int DIM, int KT, int WAVES>
__device__ __attribute__((noinline)) bool clear_values(unsigned char* v, int* found, int sees) {
  constexpr int P = Kind<T>::P, PLANE = KT * DIM * 2;
  constexpr uint32_t E = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
  if (threadIdx.x < KT) found[threadIdx.x] = 0;
  wait_lds();
  barrier();
  for (int x = threadIdx.x; x < KT * DIM / 2; x += WAVES * 64) {  // two values
    const int r = x / (DIM / 2), at = v_at<DIM>(r, x % (DIM / 2) / 4) + x % 4 * 4;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(v + at);
    const uint32_t keep = ((w & E) == E ? 0u : 0xffffu) | ((w & (E << 16)) == (E << 16) ? 0u : 0xffff0000u);
    if (keep != ~0u) {
      found[r] = 1;
      for (int p = 0; p < P; ++p) *reinterpret_cast<uint32_t*>(v + p * PLANE + at) &= keep;
    }
  }
  wait_lds();
  barrier();
  bool seen = false;
  for (int r = 0; r < min(KT, sees); ++r) seen |= found[r] != 0;
  wait_lds();
  barrier();  // before `found` is cleared again
  return seen;
}

// k's two planes and exponents and v's three planes, [piece][head][row][dim]: once a call, where every
// workgroup would split its tiles again.
template <int DIM>
__global__ __launch_bounds__(256) void prompt_split_kernel(Prompt a) {
  constexpr int LANES = DIM / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int piece = id % LANES;
  const uint32_t rest = (uint32_t)(id / LANES), i = rest / (uint32_t)(2 * a.heads);
  const int w = rest - i * (2 * a.heads), h = w % a.heads;
  if (i >= (uint32_t)a.n) return;  // whole rows
  const bool is_v = w >= a.heads;
  float x[8];
  load8((is_v ? (const float*)a.v + i * a.vt + h * a.vh : (const float*)a.k + i * a.kt + h * a.kh) + 8 * piece, x);
  uint32_t peak = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) peak = max(peak, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) peak = max(peak, (uint32_t)__shfl_xor((int)peak, d));
  const size_t plane = (size_t)a.heads * a.n * DIM, row = (size_t)h * a.n + i;
  short* to = (short*)a.ws + (is_v ? 2 * plane : 0) + row * DIM + 8 * piece;
  if (is_v) {
    const Frag<3> f = frag_of<float>(x);
#pragma unroll
    for (int e = 0; e < 3; ++e) *reinterpret_cast<v8s*>(to + e * plane) = f.p[e];
  } else {
    const int e = row_exponent(peak);
    const Frag<2> f = halves(x, e);
    *reinterpret_cast<v8s*>(to) = f.p[0];
    *reinterpret_cast<v8s*>(to + plane) = f.p[1];
    if (piece == 0) a.exponents[row] = e;
  }
}

// Tiles of KT keys and values come straight into LDS, rows past the sequence's end as zeros. The
// 16-bit types hold two tiles, the next one's loads under this one's products, one barrier a tile.
// f32 holds one (40 KB of planes at dim 128, so that two workgroups share a CU): the next keys load
// under this tile's second product, the next values under the next tile's first, two barriers.
// PARTS = 2: two waves take one half of each tile's keys each for the same 32 queries, joined in LDS at
// the end, where 128 queries a workgroup of four waves leave the GPU part empty. Four waves have 64
// queries then, in twice the workgroups, each half as long. (Heads of 64 in 16 bits take tiles of 128 keys, so
// that a wave has as much of a tile as without: 2048 tokens, 16 heads, f16: 29 -> 25 us.) f32 heads of 128,
// whose tile of 64 keys fills half of LDS, take eight waves and 128 queries.
// DIRECT (f32, short prompts): the workgroup splits its tiles itself, and no launch goes before.
template <typename T, int DIM, int PARTS, bool DIRECT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void prompt_kernel(Prompt a) {
  constexpr int P = Kind<T>::P, PK = Kind<T>::PK, KT = P == 3 ? 32 * PARTS : PARTS == 2 && DIM == 64 ? 128 : 64;
  constexpr int SUB = KT / 32 / PARTS, BUFS = P == 3 ? 1 : 2;
  constexpr int ALL = 32 * WAVES / PARTS;  // queries a workgroup
  constexpr int STEPS = DIM / 16, VT = DIM / 32, PLANE = KT * DIM * 2;
  constexpr int ROWS = 1024 / (DIM * 2);         // of a wave's load
  constexpr int PER = KT / ROWS / WAVES;  // loads a wave and plane
  __shared__ __attribute__((aligned(1024))) unsigned char lds[BUFS * (PK + P) * PLANE];
  __shared__ __attribute__((aligned(16))) int exponents[DIRECT ? PROMPT_DIRECT / DIM : KT];  // f32: of the tile's keys, or of all
  __shared__ int tops[WAVES];
  __shared__ int found[KT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hh = lane >> 5;
  Place at;
  if (!place_of<ALL>(a, &at)) return;
  const int len = at.len, q0 = at.q0;
  const int part = wave % PARTS, qw = q0 + wave / PARTS * 32, row = qw + n;  // the wave's first query, this lane's
  const int h = at.head / a.group;
  const int keys = !at.keys ? 0 : a.causal ? min(len, q0 + ALL) : len;  // that the workgroup sees
  const int wkeys = a.causal ? min(keys, qw + 32) : keys;                      // that the wave does
  const int sees = a.causal ? min(len, row + 1) : len;                         // that the lane does

  // k and v as loaded: the callers' rows, or the planes
  const size_t plane = (size_t)a.heads * a.n * DIM * 2;
  const int ktb = P == 3 ? DIM * 2 : (int)a.kt * 2, vtb = P == 3 ? DIM * 2 : (int)a.vt * 2;
  const char *k, *v;
  if constexpr (P == 3) {
    k = (const char*)a.ws + ((size_t)h * a.n + at.start) * (DIM * 2);
    v = k + 2 * plane;
  } else {
    k = (const char*)((const T*)a.k + (int64_t)at.start * a.kt + h * a.kh);
    v = (const char*)((const T*)a.v + (int64_t)at.start * a.vt + h * a.vh);
  }
  // of this wave's loads: the lane's place in LDS is its own, the piece the one that lies there
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  uint32_t ko[PER], vo[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int r = (wave * PER + e) * ROWS + lane / (DIM / 8), slot = lane % (DIM / 8);
    ko[e] = r * ktb + (k_at<DIM>(r, slot) & (DIM * 2 - 1));
    vo[e] = r * vtb + (v_at<DIM>(r, slot) & (DIM * 2 - 1));
  }
  auto fetch = [&](const char* from, int planes, int stride, const uint32_t (&off)[PER], int t0, uint32_t to) {
    const uint32_t bytes = (uint32_t)min((int64_t)(len - 1 - t0) * stride + DIM * 2, (int64_t)0x7fffffff);
#pragma unroll
    for (int p = 0; p < planes; ++p) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(from + p * plane + (int64_t)t0 * stride, bytes);
#pragma unroll
      for (int e = 0; e < PER; ++e) dma16(r, off[e], to + p * PLANE + (wave * PER + e) * 1024);
    }
  };
  Frag<PK> qf[STEPS];
  int q_e = 0;  // f32: the exponent of this lane's query
  const T* q = (const T*)a.q + (int64_t)(at.start + row) * a.qt + at.head * a.qh + 8 * hh;
  if constexpr (PK == 2) {
    float x[STEPS][8];
    uint32_t peak = 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = 0.f;
      if (row < len) load8(q + 16 * s, x[s]);
#pragma unroll
      for (int i = 0; i < 8; ++i) peak = max(peak, __float_as_uint(x[s][i]) & 0x7fffffffu);
    }
    peak = max(peak, (uint32_t)__shfl_xor((int)peak, 32));
    q_e = row_exponent(peak);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[s] = halves(x[s], q_e);
  } else {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row < len) x = *reinterpret_cast<const uint4*>(q + 16 * s);
      qf[s].p[0] = __builtin_bit_cast(v8s, x);
    }
  }
  const int* row_e = PK == 2 ? a.exponents + (size_t)h * a.n + at.start : nullptr;
  auto exponent = [&](int t0) {
    const int t = t0 + threadIdx.x;
    return PK == 2 && !DIRECT && threadIdx.x < KT && t < len ? row_e[t] : NO_ROW;
  };
  // What is added to a score times the scale, for a maximum, and the factor from the weights of one maximum
  // to those of another: f32 subtracts the maxima first, the 16-bit types what they add, rounded.
  auto shift_of = [&](float x) { return __fsub_rn(Kind<T>::LIFT, __fmul_rn(x, a.scale2)); };
  auto factor = [&](float from, float to) {
    return __builtin_amdgcn_exp2f(P == 3 ? __fmul_rn(__fsub_rn(from, to), a.scale2) : __fsub_rn(shift_of(to), shift_of(from)));
  };
  float m, l;
  int most_e;  // f32: the largest exponent among the keys that this thread put into LDS
  v16f o[VT];
  // Once; and where an output is not finite once more, with the values that are not out of the tiles
  // that some query sees in part. Rows that see one, or are not finite then, go to plain_row: what a
  // query does not see changes no bit of its output.
  bool odd = false;
  for (int again = 0;; again = 1) {
    m = -INFINITY, l = 0.f, most_e = NO_ROW;
#pragma unroll
    for (int d = 0; d < VT; ++d) o[d] = zeros16();
    if (!DIRECT && keys > 0) {
      fetch(k, PK, ktb, ko, 0, lds0);
      if constexpr (BUFS == 2) fetch(v, P, vtb, vo, 0, lds0 + PK * PLANE);
    }

    int e_next = exponent(0);  // loaded with the keys, put in LDS when they are there
    for (int t0 = 0, buf = 0; t0 < keys; t0 += KT, buf ^= BUFS - 1) {
      wait_dma_all();
      int* key_e = exponents + (DIRECT ? t0 : 0);
      if constexpr (DIRECT) {
        wait_lds();
        barrier();  // the last tile is read
#pragma unroll
        for (int e = 0; e < 2 * KT * DIM / 8 / (WAVES * 64); ++e) {
          constexpr int HALF = KT * DIM / 8;  // pieces of eight of k, then of v
          const int id = threadIdx.x + e * WAVES * 64, r = id % HALF / (DIM / 8), c = id % (DIM / 8);
          const bool is_v = id >= HALF;
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (t0 + r < len) {
            const int64_t at_row = at.start + t0 + r;
            const float* from = is_v ? (const float*)a.v + at_row * a.vt + h * a.vh
                                     : (const float*)a.k + at_row * a.kt + h * a.kh;
            load8(from + 8 * c, x);
          }
          if (is_v) {
            const Frag<3> f = frag_of<float>(x);
#pragma unroll
            for (int p = 0; p < 3; ++p)
              *reinterpret_cast<v8s*>(lds + (PK + p) * PLANE + v_at<DIM>(r, c)) = f.p[p];
          } else {
            uint32_t peak = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) peak = max(peak, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
            for (int d = 1; d < DIM / 8; d *= 2) peak = max(peak, (uint32_t)__shfl_xor((int)peak, d));
            const int ex = row_exponent(peak);
            const Frag<2> f = halves(x, ex);
#pragma unroll
            for (int p = 0; p < 2; ++p) *reinterpret_cast<v8s*>(lds + p * PLANE + k_at<DIM>(r, c)) = f.p[p];
            if (c == 0) key_e[r] = ex;
            most_e = max(most_e, ex);
          }
        }
      } else if (PK == 2 && threadIdx.x < KT) {
        key_e[threadIdx.x] = e_next;
        most_e = max(most_e, e_next);
      }
      wait_lds();
      barrier();  // the keys are there (both buffers: the values too), what is loaded over is read
      const unsigned char *tk = lds + buf * (PK + P) * PLANE, *tv = tk + PK * PLANE;
      auto middle = [&]() {  // f32: the values are there, the keys read
        if constexpr (DIRECT) return;
        wait_dma_all();
        wait_lds();
        barrier();
        if (t0 + KT < keys) {
          fetch(k, PK, ktb, ko, t0 + KT, lds0);
          e_next = exponent(t0 + KT);
        }
      };
      if constexpr (BUFS == 1 && !DIRECT) {
        fetch(v, P, vtb, vo, t0, lds0 + PK * PLANE);
      } else if (BUFS == 2 && t0 + KT < keys) {
        const uint32_t to = lds0 + (buf ^ 1) * (PK + P) * PLANE;
        fetch(k, PK, ktb, ko, t0 + KT, to);
        fetch(v, P, vtb, vo, t0 + KT, to + PK * PLANE);
      }
      const bool clears = again && (t0 + KT > len || (a.causal && t0 + KT > q0 + 1));
      const int tw = t0 + 32 * SUB * part;  // this wave's first key of the tile
      if (tw >= wkeys) {
        if constexpr (BUFS == 1) middle();
        if (clears) clear_values<T, DIM, KT, WAVES>(const_cast<unsigned char*>(tv), found, 0);
        continue;
      }

      tk += part * 32 * SUB * DIM * 2;
      tv += part * 32 * SUB * DIM * 2;

      // S^T = k q^T
      v16f s[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        s[u] = zeros16();
#pragma unroll
        for (int e = 0; e < STEPS; ++e) {
          Frag<PK> kf;
#pragma unroll
          for (int p = 0; p < PK; ++p)
            kf.p[p] = *reinterpret_cast<const v8s*>(tk + p * PLANE + k_at<DIM>(32 * u + n, 2 * e + hh));
          s[u] = score<T>(kf, qf[e], s[u]);
        }
      }

      if constexpr (PK == 2) {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // the next step's fragments under this one's products
#pragma unroll
        for (int i = 0; i < STEPS - 2; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int4 e = *reinterpret_cast<const int4*>(key_e + 32 * SUB * part + 8 * i + 4 * hh);
          s[0][4 * i] = __builtin_ldexpf(s[0][4 * i], e.x + q_e);
          s[0][4 * i + 1] = __builtin_ldexpf(s[0][4 * i + 1], e.y + q_e);
          s[0][4 * i + 2] = __builtin_ldexpf(s[0][4 * i + 2], e.z + q_e);
          s[0][4 * i + 3] = __builtin_ldexpf(s[0][4 * i + 3], e.w + q_e);
        }
      }

      // softmax, one step. The maximum that is subtracted lags (the weights' own size cancels in the
      // quotient), so that most steps rescale nothing.
      const bool edge = tw + 32 * SUB > len || (a.causal && tw + 32 * SUB > qw + 1);
      if (edge)
#pragma unroll
        for (int i = 0; i < 16 * SUB; ++i)
          if (tw + 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * hh + i % 4 >= sees) s[i / 16][i % 16] = -INFINITY;
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 16 * SUB; ++i) top = fmaxf(top, s[i / 16][i % 16]);
      top = max_xor32(top);
      const bool grew = __fmul_rn(__fsub_rn(top, m), a.scale2) > Kind<T>::LAG;
      if (__any(grew)) {
        const float f = grew ? factor(m, top) : 1.f;
        m = grew ? top : m;
        l = __fmul_rn(l, f);
#pragma unroll
        for (int d = 0; d < VT; ++d) o[d] *= f;
      }
      const float base = m == -INFINITY ? 0.f : m, shift = shift_of(base);
#pragma unroll
      for (int i = 0; i < 16 * SUB; ++i) {
        float x = s[i / 16][i % 16];
        // f32 subtracts the maximum first. The 16-bit types take one FMA (8192 tokens 560 -> 547 us): the
        // rounding of `shift` is a factor common to the row, which cancels while it stays near 1; beyond
        // 2^24 (scores that large) the row is taken again.
        x = P == 3 ? __fmul_rn(__fsub_rn(x, base), a.scale2) : __fmaf_rn(x, a.scale2, shift);
        s[i / 16][i % 16] = x = __builtin_amdgcn_exp2f(x);
        l = __fadd_rn(l, x);
      }
      if constexpr (P == 1) odd |= fabsf(shift) > 0x1p24f;
      if constexpr (BUFS == 1) middle();

      if (clears)
        odd |= clear_values<T, DIM, KT, WAVES>(const_cast<unsigned char*>(tv) - part * 32 * SUB * DIM * 2, found, sees - t0);

      // O^T += v^T p^T
#pragma unroll
      for (int e = 0; e < 2 * SUB; ++e) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = s[e / 2][8 * (e % 2) + i];
        const Frag<P> pf = frag_of<T>(x);
#pragma unroll
        for (int d = 0; d < VT; ++d) o[d] = product<T>(v_frag<DIM, P>(tv, PLANE, d, e), pf, o[d]);
      }
      if constexpr (P == 3) {  // the same, the weights' splitting between
        __builtin_amdgcn_sched_group_barrier(0x100, 12, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 80, 0);
#pragma unroll
        for (int i = 0; i < 6 * (2 * VT - 2); ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 12, 0);
      }
    }
    if constexpr (PARTS == 2) {  // the two halves' sums, in the place of the tiles
      float* to = reinterpret_cast<float*>(lds) + (wave >> 1) * (16 * VT + 3) * 64 + lane;
      wait_lds();
      barrier();
      if (part == 1) {
        to[0] = m;
        to[64] = l;
        to[128] = odd ? 1.f : 0.f;
#pragma unroll
        for (int i = 0; i < 16 * VT; ++i) to[(3 + i) * 64] = o[i / 16][i % 16];
      }
      wait_lds();
      barrier();
      if (part == 0) {
        const float m1 = to[0], now = fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 0.f : factor(m, now), f1 = m1 == -INFINITY ? 0.f : factor(m1, now);
        l = __fmaf_rn(l, f0, __fmul_rn(to[64], f1));
        odd |= to[128] != 0.f;
#pragma unroll
        for (int i = 0; i < 16 * VT; ++i)
          o[i / 16][i % 16] = __fmaf_rn(o[i / 16][i % 16], f0, __fmul_rn(to[(3 + i) * 64], f1));
      }
    }
    l = __fadd_rn(l, __shfl_xor(l, 32));
    float zero = __fmul_rn(l, 0.f);  // NaN beside a value that is not finite
#pragma unroll
    for (int d = 0; d < VT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) zero = __fmaf_rn(o[d][i], 0.f, zero);
    odd |= zero != 0.f;
    if constexpr (P == 3) {
      uint32_t least = ~0u;  // |o| as an integer, 0 as the largest
#pragma unroll
      for (int d = 0; d < VT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) least = min(least, (__float_as_uint(o[d][i]) << 1) - 1u);
      odd |= least < (__float_as_uint(__fmul_rn(l, 0x1p-109f)) << 1) - 1u;
      // What the scores lose of channels far below their row's largest: 2^-38 of either row's largest, below
      // 2^(exponent + 14), times dim channels of the other's. First by all keys that were here, which seldom
      // says more; then by those that the query sees.
      const float most = fmaxf(0x1p-17f, __fmul_rn(__fmul_rn(fabsf(m), a.scale2), 0x1p-22f));
      auto counts = [&](int e) { return __builtin_ldexpf(a.scale2, q_e + e + (DIM == 128 ? -2 : -3)) > most; };
      most_e = wave_max(most_e);
      if (lane == 0) tops[wave] = most_e;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) most_e = max(most_e, tops[w]);
      if (part == 0 && __any(row < len && counts(most_e))) {
        const int* e = DIRECT ? exponents : row_e;
        int seen = NO_ROW;
        for (int t = 0; t < wkeys; ++t) seen = max(seen, t < sees ? e[t] : NO_ROW);
        odd |= counts(seen);
      }
    }
    odd = odd && row < len && part == 0;
    if (again || !__syncthreads_or(odd)) break;
    odd = false;
  }
  if (part) return;
  const uint64_t who = __ballot(odd);
  store_rows<T, DIM>(a, at, row, l, o, (uint32_t)(who | who >> 32));
}

}  // namespace bq

using namespace bq;

size_t bq_prompt_attention_ws_bytes(int type, int64_t n, int64_t heads, int64_t dim) {
  if (type != 0 || n * dim <= PROMPT_DIRECT || heads < 1 || dim < 1) return 0;
  return (size_t)n * heads * (10 * dim + 4);  // two planes of k, three of v, an exponent a row of k
}

int bq_prompt_attention(const void* q, const void* k, const void* v, int type, int64_t n, int64_t q_heads,
                        int64_t heads, int64_t dim, int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head,
                        int64_t v_token, int64_t v_head, const int32_t* cu, int64_t B, int causal, float scale,
                        void* out, void* ws, size_t ws_bytes, bq_stream_t stream) {
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
  // a tile's rows within 32 bits, where the callers' own come into LDS (f32's are split first, or where used)
  if (k_token < 0 || v_token < 0 || (type && (k_token > 1 << 23 || v_token > 1 << 23)))
    return set_error(BQ_ERR_UNSUPPORTED, "%s: rows of k or v too far apart", what);
  // whatever the lengths are: a full tile for every 128 rows and one begun for each sequence
  const bool direct = type == 0 && n * dim <= PROMPT_DIRECT;
  const int64_t begun = B + 2 < n ? B + 2 : n;
  // The form (prompt_kernel's PARTS), by the workgroups of 128 queries that there would be, two of
  // which a CU holds at once. us in one part and in two, causal:
  //   16 bits, up to 512: bf16, 128 channels, 2048 + 1111 tokens of 16 heads (400) 57, 49; 1024 of 32 (256)
  //     28, 25; 2048 of 32 (512) 57, 56; 3000 of 32 (752) 87, 110; f16, 64 channels, 2048 of 16 (256) 34, 25
  //   f32, up to 768: 64 channels, 2048 + 1111 of 16 (400) 119, 84; 2048 of 32 (512) 122, 97; 4096 of 32
  //     (1024) 305, 318; 128 channels, and sequences of 256 tokens on average or more: 2048 + 1111 of 16
  //     159, 137; 2048 of 32 176, 161; 5542 in 8 of 16 (704) 260, 249; 4096 of 32 556, 570; 30 of 130
  //     tokens of 8 heads 40, 50
  const int64_t groups = (n + 127) / 128 * q_heads;
  const bool wide = dim == 128, two = type ? groups <= 512 : !direct && groups <= 768 && (!wide || n >= 256 * B);
  const bool eight = two && !type && wide, halves = two && !eight;
  const int64_t tiles = n / (halves ? 64 : 128) + begun;
  if (tiles * q_heads > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  const size_t need = bq_prompt_attention_ws_bytes(type, n, heads, dim);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    return set_error(BQ_ERR_ARG, "%s: a workspace of %zu bytes, given %zu", what, need, ws ? ws_bytes : 0);
  const Prompt a = {q, k, v, out, q_token, q_head, k_token, k_head, v_token, v_head, cu, (int)n, (int)B, (int)heads,
                    (int)(q_heads / heads), (int)tiles, causal ? 1 : 0, scale * 1.4426950408889634f, ws,
                    (int*)((char*)ws + (size_t)10 * n * heads * dim)};
  const unsigned grid = (unsigned)(tiles * q_heads);
  hipStream_t st = (hipStream_t)stream;
  if (need) {
    const int64_t blocks = (n * 2 * heads * (dim / 8) + 255) / 256;
    if (blocks > 0x7fffffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
    if (wide) prompt_split_kernel<128><<<(unsigned)blocks, 256, 0, st>>>(a);
    else prompt_split_kernel<64><<<(unsigned)blocks, 256, 0, st>>>(a);
  }
#define BQ_PROMPT(T, PARTS, DIRECT)                                                          \
  do {                                                                                       \
    if (wide) prompt_kernel<T, 128, PARTS, DIRECT, 4><<<grid, 256, 0, st>>>(a);              \
    else prompt_kernel<T, 64, PARTS, DIRECT, 4><<<grid, 256, 0, st>>>(a);                    \
  } while (0)
  if (type == 0) {
    if (direct) BQ_PROMPT(float, 1, true);
    else if (eight) prompt_kernel<float, 128, 2, false, 8><<<grid, 512, 0, st>>>(a);
    else if (halves) prompt_kernel<float, 64, 2, false, 4><<<grid, 256, 0, st>>>(a);
    else BQ_PROMPT(float, 1, false);
  } else if (type == 1) {
    if (halves) BQ_PROMPT(__bf16, 2, false);
    else BQ_PROMPT(__bf16, 1, false);
  } else {
    if (halves) BQ_PROMPT(_Float16, 2, false);
    else BQ_PROMPT(_Float16, 1, false);
  }
#undef BQ_PROMPT
  return check_launch(what);
}
