// Attention of chunks of new tokens over a cache held in 4 bits (its form: bq_kv4.h): prompts read in
// pieces, alone or beside sequences that add one token.
//
// Sequence b's new tokens are the rows cu[b] .. cu[b + 1] of q, the last ones of its lens[b] cached
// tokens: row i is token lens[b] - cu[b + 1] + i and sees the tokens up to itself,
// out = sum_i p_i v_i with p = softmax(scale q . k_i), zeros where it sees nothing.
//
// One pass over the keys with each row's running maximum and sum. The G = q_heads / heads query heads of a key-value
// head and the chunk's tokens are the rows of one product (row t G + j: token t, head j), so that the codes are
// expanded once for all that read them. The codes become bf16 exactly (a code has 2 significant bits, bf16 the
// exponents of f32). q enters as the exact sum of bf16 pieces (f32: 3, f16: 2, bf16: 1), the weights p as pieces too
// (f32: 3; the 16-bit types: 2, so that p's error is 2^-16 beside the output's rounding of 2^-11 or 2^-8; with one,
// bf16's outputs were 2.36e-3 of their size from float64 where rounding them alone is 1.67e-3, in 553 us for 702 of the
// case below), with f32 accumulation; the sum of the weights is of those before they are rounded. The scores are
// taken transposed, S^T = k q^T on the 32 x 32 x 16 MFMA, keys in an order (bits 2 and 3 of their number
// exchanged) that leaves 8 following tokens in 8 following registers of a lane: the exponentials are, register for
// register, the second operand of O^T = v^T p^T.
//
// Wide tiles, of sequences of many rows: a workgroup of four waves takes 128 rows, 32 a wave, and 64 keys at a time,
// whose codes, loaded one tile ahead, are expanded into LDS, two tiles in turn, one barrier a tile. Bound by the
// matrix units beside the exponentials and the expansion: 2048 tokens over 16384, 32 heads over 8 of 128, bf16:
// 702 us, 734 TFLOP/s, at 1.5 times the products (1.10 PFLOP/s of pieces); 8192 over 8192 735 us, 748 (the library's
// 8192^3 product: 1426). f16 550 and f32 380, at 2 and 3 times the products. With p of bf16 in one piece reading LDS
// took as long as the products, but with 64 rows a wave, which halves it, one wave a SIMD did not hide the exponentials
// (804 us where these were 555), and eight waves that share the codes took as long (567; in two halves that take turns
// between products and exponentials 630).
//
// Narrow tiles, of sequences of few rows: 32 rows, of which each wave takes every fourth 32 keys by itself, from
// memory into operands, joined in LDS at the end. Bound by the reading and the products beside it: 64 sequences of
// 4000 tokens and one new, bf16: 74 us, 3.7 TB/s (read alone: 7.0; with p in one piece 60 us); 512 of 1000: 180 us,
// 3.1 TB/s (167), where finding the tile and the first loads are a third of a workgroup's time.
//
// The maximum that is subtracted lags by up to 2^8 (the weights' own size cancels in the quotient) and is a whole
// number of powers of two, so that a weight is one FMA and one exp2 and all of a row's agree. In keys whose values are
// large it does not lag, so that no weight passes 1 there: f32 holds the sums as far as those of such weights.
//
// A tile's keys are cut into shares of up to `upper` units of 64 where the tiles alone would leave the GPU part empty;
// a second kernel joins the shares of a row.
#include "bq_dma.h"
#include "bq_kv4_pieces.h"

namespace bq {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct Chunk {
  Kv4 c;
  const int *lens, *cu;
  const void* q;
  int64_t qt, qh;  // strides in elements: token, head
  int n, group, B, max_len;
  int least;  // sequences of more rows than this take wide tiles
  struct Kind {
    int tiles, upper, most;  // that there can be; units a share; shares a tile at most
  };
  Kind wide, few;
  FastDiv by_group;
  float scale2;  // scale * log2(e)
  void* out;     // [n][heads * group][DIM]
  float *part, *stats;  // of each row, head and share: [n group][heads][most][DIM], [..][2]
};

constexpr int WIDE = 128, FEW = 32, KEYS = 64;  // rows a tile, of sequences of many and of few; keys a unit
constexpr float LAG = 8.f;  // by how many powers of two the maximum that is subtracted may lag
// A tile's sequence and rows.
struct Place {
  int b, start, rows, row0;  // b: -1 for rows of no sequence; the first row of q, the sequence's rows, the tile's first
  int base, len;             // the place in the cache of the sequence's first new token, and its tokens
};

template <int CONTROL, int ROWS>
__device__ __forceinline__ int plus_lanes(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_upto(int v) {  // the lanes' values up to this one's own
  v = plus_lanes<0x111, 0xF>(v);  // from the lanes 1, 2, 4 and 8 before in a row of 16,
  v = plus_lanes<0x112, 0xF>(v);
  v = plus_lanes<0x114, 0xF>(v);
  v = plus_lanes<0x118, 0xF>(v);
  v = plus_lanes<0x142, 0xA>(v);  // the last of the row before into the second and fourth,
  return plus_lanes<0x143, 0xC>(v);  // lane 31's into the upper half
}
// Where the i-th of what lies before cu[0], each sequence and what lies past the last ends.
__device__ __forceinline__ int end_at(const Chunk& a, int i) {
  const int x = min(max(a.cu[min(i, a.B)], 0), a.n);  // whatever i: loads under a condition would wait for one another
  return i > a.B ? a.n : x;
}
// From 64 of those ends, a lane each, and the one before: the rows of each, and its tiles if it takes such.
template <int TILE>
__device__ __forceinline__ int tiles_of(const Chunk& a, int end, int before, int* start, int* rows) {
  int x = __builtin_amdgcn_update_dpp(before, end, 0x138, 0xF, 0xF, false);  // the lane before's
  asm("" : "+v"(x));  // no operand of the difference: where `before` is 0 it became a v_subrev_u32_dpp, of the wrong sign
  *start = x;
  *rows = max(0, end - *start) * a.group;
  return (*rows > a.least) == (TILE == WIDE) ? (*rows + TILE - 1) / TILE : 0;
}
// Tile `last` from the last one on. Where there are more sequences than lanes their tiles are summed first, 64 at a
// time, the loads of eight such on their way: beside workgroups that stream, each wait is 1 to 2 us (512 sequences of
// one token: 178 us with one after another, 166 so).
template <int TILE>
__device__ __forceinline__ bool place_of(const Chunk& a, int last, Place* out) {
  const int lane = threadIdx.x & 63, rounds = (a.B + 2 + 63) >> 6, each = (rounds + 63) >> 6;  // rounds a lane's sum
  int from = 0, place = 0, s, rows;
  if (rounds > 1) {
    int sums = 0, before = 0;
    for (int r0 = 0; r0 < rounds; r0 += 8) {
      int ends[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) ends[k] = end_at(a, (r0 + k) * 64 + lane);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int sum = __builtin_amdgcn_readlane(wave_upto(tiles_of<TILE>(a, ends[k], before, &s, &rows)), 63);
        before = __builtin_amdgcn_readlane(ends[k], 63);
        sums += lane == (each == 1 ? r0 + k : (r0 + k) / each) ? sum : 0;
      }
    }
    const int upto = wave_upto(sums);
    place = __builtin_amdgcn_readlane(upto, 63) - 1 - last;
    if (place < 0) return false;
    const int l = __builtin_ctzll(__ballot(upto > place));
    place -= __builtin_amdgcn_readlane(upto - sums, l);
    from = l * each * 64;
  }
  for (int at = from; at < from + each * 64; at += 64) {
    const int mine = tiles_of<TILE>(a, end_at(a, at + lane), at ? end_at(a, at - 1) : 0, &s, &rows), upto = wave_upto(mine);
    if (rounds == 1) place = __builtin_amdgcn_readlane(upto, 63) - 1 - last;
    if (place < 0) return false;
    const uint64_t hit = __ballot(upto > place);
    if (hit) {
      const int l = __builtin_ctzll(hit), seq = at + l;
      const bool real = seq > 0 && seq <= a.B;
      place -= __builtin_amdgcn_readlane(upto - mine, l);
      out->b = real ? seq - 1 : -1;
      out->start = __builtin_amdgcn_readlane(s, l);
      out->rows = __builtin_amdgcn_readlane(rows, l);
      out->row0 = place * TILE;
      out->len = real ? max(0, min(a.lens[seq - 1], a.max_len)) : 0;
      out->base = real ? a.lens[seq - 1] - fdiv(out->rows, a.by_group.mul, a.by_group.shift) : 0;
      return true;
    }
    place -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// What row `row` of a sequence sees: its first so many tokens.
__device__ __forceinline__ int end_of(const Chunk& a, const Place& at, int row) {
  return max(0, min(at.len, at.base + fdiv(row, a.by_group.mul, a.by_group.shift) + 1));
}
// The units of the tile that holds `row`, and in how many shares they are cut.
template <int TILE>
__device__ __forceinline__ int units_of(const Chunk& a, const Place& at, int row0) {
  return (end_of(a, at, min(row0 + TILE, at.rows) - 1) + KEYS - 1) / KEYS;
}
__device__ __forceinline__ int shares_of(int upper, int units) { return max(1, (units + upper - 1) / upper); }
__device__ __forceinline__ int64_t slot_of(const Chunk& a, const Place& at, int row, int h) {  // of a row's first share
  return (((int64_t)at.start * a.group + row) * a.c.heads + h) * max(a.wide.most, a.few.most);
}

// Where 32 tokens lie: the first one's row in the cache's arrays, -1 where there is no page.
__device__ __forceinline__ int64_t row_of(const Chunk& a, const Place& at, int h, int blk) {
  const int i = fdiv(blk, a.c.by_blocks.mul, a.c.by_blocks.shift);
  const int page = 32 * blk < at.len ? kv4_page(a.c, at.b, i) : -1;
  return page < 0 ? -1 : ((int64_t)page * a.c.heads + h) * a.c.page + ((blk - i * (a.c.page >> 5)) << 5);
}
__device__ __forceinline__ int64_t of_lane(int64_t x, int lane) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, lane) |
         (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32;
}

// A row's weights are relative to 2^ref, ref the next whole number above its lagging maximum; or, where that
// passes 2^20, to the maximum itself.
constexpr float FAR = 0x1p20f;
__device__ __forceinline__ float ref_of(float m, float c) { return m == -INFINITY ? 0.f : ceilf(__fmul_rn(m, c)); }
// From weights of one maximum to those of another, each by what its side's are relative to.
__device__ __forceinline__ float factor(float from, float to, float c) {
  if (from == -INFINITY) return 0.f;
  const float a = ref_of(from, c), b = ref_of(to, c);
  const bool far_a = fabsf(a) > FAR, far_b = fabsf(b) > FAR;
  const float far = __fsub_rn(far_a ? from : 0.f, far_b ? to : 0.f), near = __fsub_rn(far_a ? 0.f : a, far_b ? 0.f : b);
  return __builtin_amdgcn_exp2f(__fmaf_rn(far, c, near));
}

// Where a 16-byte piece lies in LDS: row `row` of the keys, channels 8 piece ..; channel `ch` of the
// values, tokens 8 piece ... XORed so that 16 lanes cover all banks.
template <int DIM>
__device__ __forceinline__ int k_at(int row, int piece) {
  return DIM == 128 ? row * 256 + ((piece ^ (row & 15)) << 4) : row * 128 + ((piece ^ ((row >> 1) & 7)) << 4);
}
__device__ __forceinline__ int v_at(int ch, int piece) { return ch * 128 + ((piece ^ (((ch >> 1) ^ ((ch >> 4) & 3)) & 7)) << 4); }

constexpr uint32_t HUGE = 253;  // scale bytes from here on may make codes infinite or NaN
// Which of four bytes are: bits 7, 15, ... of the result. And those from 191 on, of values of up to 2^66 and more: of
// smaller ones 2^31 terms with weights of 2^8 stay far below f32's end.
__device__ __forceinline__ uint32_t huge_of(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x03030303u) & w & 0x80808080u; }
__device__ __forceinline__ uint32_t large_of(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x41414141u) & w & 0x80808080u; }
// Byte I of four as a scale of the expanding conversion, which takes a float's exponent and nothing else of it.
template <int I>
__device__ __forceinline__ float scale_byte(uint32_t w) {
  return __uint_as_float(I < 3 ? w << (23 - 8 * I) : w >> 1);
}

// One of the 256 pieces of 64 tokens' codes: of token p / 4 a quarter of the keys' channels, of tokens
// 4 (p / 16) .. + 3 channel slice p % 16 of the values. Pieces p / 128 lie in one block of 32 tokens.
template <int DIM>
struct Codes {
  uint32_t k[DIM / 32], v[DIM / 32], ks, vs;
  // `row`: of the block's first token (uniform)
  __device__ __forceinline__ void load_k(const Kv4& c, int64_t row, int p) {
    constexpr int CB = DIM / 32;
    const int t = (p & 127) >> 2, quarter = p & 3;
    const uint8_t* from = c.k + row * (DIM / 2) + (uint32_t)(t * (DIM / 2) + quarter * (DIM / 8));
    if constexpr (DIM == 128) {
      const uint4 x = *reinterpret_cast<const uint4*>(from);
      k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(from);
      k[0] = x.x, k[1] = x.y;
    }
    ks = (c.ks + row * CB)[(uint32_t)((((t & 3) * CB + quarter * CB / 4) << 3) + (t >> 2))];
  }
  __device__ __forceinline__ void load_v(const Kv4& c, int64_t row, int p) {
    constexpr int CB = DIM / 32;
    const int four = (p & 127) >> 4, n = p & 15;
    const uint8_t* from = c.v + row * (DIM / 2);
    if constexpr (DIM == 128) {
      const uint4 x = *reinterpret_cast<const uint4*>(from + (uint32_t)(four * 256 + n * 16));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(from + (uint32_t)((four >> 1) * 256 + n * 16 + (four & 1) * 8));
      v[0] = x.x, v[1] = x.y;
    }
    vs = *reinterpret_cast<const uint32_t*>(c.vs + row * CB + (uint32_t)(n * CB / 16 * 32 + 4 * four));
  }
  // Values of tokens from `len` on read as zeros; left: len minus the piece's first token.
  __device__ __forceinline__ void cut(int left) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i >= left) {
        vs = (vs & ~(255u << (8 * i))) | (127u << (8 * i));
        if constexpr (DIM == 128) v[i] = 0;
        else v[i >> 1] &= i & 1 ? 0xffffu : 0xffff0000u;
      }
  }
  __device__ __forceinline__ bool huge() const { return huge_of(vs) != 0; }
  __device__ __forceinline__ bool large() const { return large_of(vs) != 0; }
  // Into a tile in LDS, as bf16. CLEAR: what is not finite among the values becomes 0 (it is added at the end).
  __device__ __forceinline__ void expand_k(unsigned char* tk, int p) const {
    const int t = p >> 2, row = (t & ~12) | ((t & 4) << 1) | ((t & 8) >> 1);
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i)
      *reinterpret_cast<v8bf*>(tk + k_at<DIM>(row, (p & 3) * (DIM / 32) + i)) = codes8(k[i], scale_bits(ks));
  }
  template <bool CLEAR, int K>
  __device__ __forceinline__ void two(unsigned char* tv, int p, const float (&s)[4]) const {  // channels 2 K and + 1 of the slice
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DIM == 128) x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[i], s[i], K));
      else if (i & 1) x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[i >> 1], s[i], K + 2));
      else x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[i >> 1], s[i], K));
      if constexpr (CLEAR)
        x[i] &= ((x[i] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((x[i] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
    }
    const int ch = (p & 15) * (DIM / 16) + 2 * K, to = (p >> 4) >> 1, half = ((p >> 4) & 1) * 8;
    *reinterpret_cast<uint2*>(tv + v_at(ch, to) + half) =
        make_uint2(__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u));
    *reinterpret_cast<uint2*>(tv + v_at(ch + 1, to) + half) =
        make_uint2(__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u));
  }
  template <bool CLEAR>
  __device__ __forceinline__ void expand_v(unsigned char* tv, int p) const {
    const float s[4] = {scale_byte<0>(vs), scale_byte<1>(vs), scale_byte<2>(vs), scale_byte<3>(vs)};
    two<CLEAR, 0>(tv, p, s);
    two<CLEAR, 1>(tv, p, s);
    if constexpr (DIM == 128) {
      two<CLEAR, 2>(tv, p, s);
      two<CLEAR, 3>(tv, p, s);
    }
  }
};

__device__ __forceinline__ v16f zeros16() {
  v16f z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// What a wave keeps of 32 rows of one key-value head: the queries' pieces, the running maxima and sums, the outputs.
// Lane (n, hh) has row n; of the queries channels 16 s + 8 hh .. of step s, of the outputs 32 d + 8 i + 4 hh ...
// With DIRECT the contracted channels of step s are DIM / 2 hh + 8 s .., the outputs VT (8 (i / 4) + 4 hh + i % 4) + d.
template <typename T, int DIM, bool DIRECT>
struct Rows {
  static constexpr int QP = Q_PIECES<T>, PP = P_PIECES<T>, STEPS = DIM / 16, VT = DIM / 32;
  Pieces<QP> q[STEPS];
  float m, l;
  v16f o[VT];
  int row, end, sure, most;  // this lane's row; what it sees; what all the wave's rows see, and any does

  __device__ __forceinline__ void begin(const Chunk& a, const Place& at, int h, int first) {
    const int n = threadIdx.x & 31, hh = (threadIdx.x >> 5) & 1, last = at.rows - 1;
    row = first + n;
    end = end_of(a, at, min(row, last));
    sure = end_of(a, at, min(first, last));
    most = first <= last ? end_of(a, at, min(first + 31, last)) : 0;
    const int here = min(row, last);  // rows past the last are the last one's again, and not stored
    const int t = fdiv(here, a.by_group.mul, a.by_group.shift), j = here - t * a.group;
    const T* from = (const T*)a.q + (int64_t)(at.start + t) * a.qt + (int64_t)(h * a.group + j) * a.qh +
                    (DIRECT ? DIM / 2 : 8) * hh;
    float x[STEPS][8];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) load8f(from + (DIRECT ? 8 : 16) * s, x[s]);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) q[s] = split_q<QP>(x[s]);
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < VT; ++d) o[d] = zeros16();
  }

  // The scores of SUB times 32 keys, from row 32 sub of a tile on.
  template <int SUB>
  __device__ __forceinline__ void scores(const unsigned char* tk, int sub, v16f (&s)[SUB]) const {
    const int n = threadIdx.x & 31, hh = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      s[u] = zeros16();
#pragma unroll
      for (int e = 0; e < STEPS; ++e) {
        const v8bf kf = *reinterpret_cast<const v8bf*>(tk + k_at<DIM>(32 * (sub + u) + n, 2 * e + hh));
#pragma unroll
        for (int p = QP - 1; p >= 0; --p) s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q[e].p[p], s[u], 0, 0, 0);
      }
    }
  }

  // What is not seen leaves them (keys from `tok`; there: a bit for each 32 that has a page). Returns the maximum,
  // which the one that is subtracted follows where it is `lag` powers of two above.
  template <int SUB>
  __device__ __forceinline__ float raise(const Chunk& a, int tok, int there, v16f (&s)[SUB], float lag) {
    const int hh = (threadIdx.x >> 5) & 1;
    if (tok + 32 * SUB > sure || there != (1 << SUB) - 1)
#pragma unroll
      for (int i = 0; i < 16 * SUB; ++i)
        if (tok + 32 * (i / 16) + 16 * (i % 16 / 8) + 8 * hh + i % 8 >= end || !((there >> (i / 16)) & 1))
          s[i / 16][i % 16] = -INFINITY;
    float tops[4];  // four chains of maxima
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      tops[c] = s[0][c];
#pragma unroll
      for (int i = c + 4; i < 16 * SUB; i += 4) tops[c] = fmaxf(tops[c], s[i / 16][i % 16]);
    }
    const float top = max_xor32(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
    follow(a, top, lag);
    return top;
  }
  __device__ __forceinline__ void follow(const Chunk& a, float top, float lag) {
    const bool grew = __fmul_rn(__fsub_rn(top, m), a.scale2) > lag;
    if (__any(grew)) {
      const float f = grew ? factor(m, top, a.scale2) : 1.f;
      m = grew ? top : m;
      l = __fmul_rn(l, f);
#pragma unroll
      for (int d = 0; d < VT; ++d) o[d] *= f;
    }
  }
  // What is subtracted from the scores, times the scale.
  template <int SUB>
  __device__ __forceinline__ float base(const Chunk& a, v16f (&s)[SUB]) const {
    float ref = ref_of(m, a.scale2);
    const bool far = fabsf(ref) > FAR;
    if (__any(far)) {  // such rows' differences are taken here, exactly as far as f32 goes
#pragma unroll
      for (int i = 0; i < 16 * SUB; ++i)
        if (far) s[i / 16][i % 16] = __fsub_rn(s[i / 16][i % 16], m);
      if (far) ref = 0.f;
    }
    return ref;
  }

  // The weights of keys 16 e .. + 15, as the second product's operand, and their sum.
  template <int SUB>
  __device__ __forceinline__ Pieces<PP> weights(const Chunk& a, const v16f (&s)[SUB], float ref, int e, float* sum) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(__fmaf_rn(s[e / 2][8 * (e % 2) + i], a.scale2, -ref));
    const Pieces<PP> f = pieces_of<PP>(x);
    *sum = __fadd_rn(__fadd_rn(__fadd_rn(x[0], x[1]), __fadd_rn(x[2], x[3])),
                     __fadd_rn(__fadd_rn(x[4], x[5]), __fadd_rn(x[6], x[7])));
    return f;
  }

  __device__ __forceinline__ void products(const unsigned char* tv, int sub, int e, const Pieces<PP>& f) {
    const int n = threadIdx.x & 31, hh = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int d = 0; d < VT; ++d) {
      const v8bf vf = *reinterpret_cast<const v8bf*>(tv + v_at(32 * d + n, 4 * sub + 2 * e + hh));
#pragma unroll
      for (int p = PP - 1; p >= 0; --p) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, f.p[p], o[d], 0, 0, 0);
    }
  }

  // SUB times 32 keys from `tok`, in a tile's places from 32 sub on.
  template <int SUB>
  __device__ __forceinline__ void keys(const Chunk& a, const unsigned char* tk, const unsigned char* tv, int sub, int tok,
                                       int there, float lag) {
    v16f s[SUB];
    scores<SUB>(tk, sub, s);
    raise<SUB>(a, tok, there, s, lag);
    const float ref = base<SUB>(a, s);
    float sums[2 * SUB];
    if constexpr (QP == 1) {  // all weights first, as the registers allow (2048 tokens over 16384: 711 us in turn, 702 so)
      Pieces<PP> f[2 * SUB];
#pragma unroll
      for (int e = 0; e < 2 * SUB; ++e) f[e] = weights<SUB>(a, s, ref, e, sums + e);
#pragma unroll
      for (int e = 0; e < 2 * SUB; ++e) products(tv, sub, e, f[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 2 * SUB; ++e) products(tv, sub, e, weights<SUB>(a, s, ref, e, sums + e));
    }
    if constexpr (SUB == 2) l = __fadd_rn(l, __fadd_rn(__fadd_rn(sums[0], sums[1]), __fadd_rn(sums[2], sums[3])));
    else l = __fadd_rn(l, __fadd_rn(sums[0], sums[1]));
  }

  // What was left out of the products is added to the outputs of the rows that see it, whatever its weight,
  // and to no other's: to the N of them from `first` on in out()'s order, y(0) ...
  template <int N, typename Y>
  __device__ __forceinline__ void add_huge(const Chunk& a, const Place& at, int h, int blk0, int blk1, int first, Y&& y) {
    const int hh = (threadIdx.x >> 5) & 1;
    for (int blk = blk0; blk < blk1; ++blk) {
      const int64_t r0 = row_of(a, at, h, blk);
      if (r0 < 0) continue;
#pragma unroll 1
      for (int t = 0; t < 32; ++t) {
        if (32 * blk + t >= most) break;
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {  // four channels at a time
          const int ch = channel(first + 4 * i, hh);
          const uint32_t byte = a.c.vs[Kv4At<DIM>::vs(r0 + t, t, ch / 32)];
          if (byte < HUGE) continue;
          const uint32_t w = *reinterpret_cast<const uint16_t*>(a.c.v + Kv4At<DIM>::v(r0 + t, t, ch / (DIM / 16)) +
                                                                ch % (DIM / 16) / 2);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = (float)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w >> (8 * (e / 2)), scale_bits(byte), 0)[e & 1];
            if (!(fabsf(v) < INFINITY) && 32 * blk + t < end) y(4 * i + e) = __fadd_rn(y(4 * i + e), v);
          }
        }
      }
    }
  }

  // This lane's outputs in an order in which four at a time are neighbours: the x-th, and its channel.
  __device__ __forceinline__ float& out(int x) { return DIRECT ? ((float*)&o[x % VT])[x / VT] : ((float*)&o[x / 16])[x % 16]; }
  static __device__ __forceinline__ int channel(int x, int hh) {
    if constexpr (DIRECT) {
      const int i = x / VT;
      return VT * (8 * (i / 4) + 4 * hh + i % 4) + x % VT;
    } else {
      return 32 * (x / 16) + 8 * (x % 16 / 4) + 4 * hh + x % 4;
    }
  }

  // N outputs from `first` on into the output, or as one of the shares of a row.
  template <int N, typename Y>
  __device__ __forceinline__ void store(const Chunk& a, const Place& at, int h, int share, int shares, int first, Y&& y) {
    const int hh = (threadIdx.x >> 5) & 1;
    if (row >= at.rows) return;
    if (shares == 1) {
      const int t = fdiv(row, a.by_group.mul, a.by_group.shift), j = row - t * a.group;
      const float r = __fdiv_rn(1.f, l == 0.f ? 1.f : l);
      T* to = (T*)a.out + ((int64_t)(at.start + t) * a.c.heads * a.group + h * a.group + j) * DIM;
#pragma unroll
      for (int x = 0; x < N; x += 4)
        store4(to + channel(first + x, hh), __fmul_rn(y(x), r), __fmul_rn(y(x + 1), r), __fmul_rn(y(x + 2), r),
               __fmul_rn(y(x + 3), r));
    } else {
      const int64_t slot = slot_of(a, at, row, h) + share;
      float* to = a.part + slot * DIM;
#pragma unroll
      for (int x = 0; x < N; x += 4)
        *reinterpret_cast<float4*>(to + channel(first + x, hh)) = make_float4(y(x), y(x + 1), y(x + 2), y(x + 3));
      if (hh == 0 && first == 0) *reinterpret_cast<float2*>(a.stats + slot * 2) = make_float2(m, l);
    }
  }
};

// Which tile and share a workgroup has; false: none. Tiles from the last down (those with most keys first), the
// key-value heads side by side, the shares one after another: side by side, four heads' four shares of which some are
// none left half of the XCDs idle (f32, 512 rows beside 333 and 500: 146 -> 107 us).
template <int TILE>
__device__ __forceinline__ bool job_of(const Chunk& a, int id, Place* at, int* h, int* share, int* shares, int* u0, int* u1) {
  const Chunk::Kind& kind = TILE == WIDE ? a.wide : a.few;
  *h = id % a.c.heads;
  const int rest = id / a.c.heads;
  *share = rest / kind.tiles;
  if (!place_of<TILE>(a, rest - *share * kind.tiles, at)) return false;
  const int units = units_of<TILE>(a, *at, at->row0);
  *shares = shares_of(kind.upper, units);
  if (*share >= *shares) return false;
  *u0 = (uint32_t)units * *share / *shares;  // 2^25 units and 128 shares at most
  *u1 = (uint32_t)units * (*share + 1) / *shares;
  return true;
}

// Sequences of many rows: 32 rows a wave, tiles of 64 keys in LDS for all four.
template <typename T, int DIM>
__device__ __forceinline__ void wide_tile(const Chunk& a, int id, unsigned char* lds) {
  constexpr int KB = KEYS * DIM * 2, BUF = 2 * KB;  // bytes of a tile's keys, as many of its values
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Place at;
  int h, share, shares, u0, u1;
  if (!job_of<WIDE>(a, id, &at, &h, &share, &shares, &u0, &u1)) return;
  Rows<T, DIM, false> r;
  r.begin(a, at, h, at.row0 + 32 * wave);
  Codes<DIM> next;
  const int p = threadIdx.x, mine = wave >> 1;  // which of a unit's two blocks this wave's codes are of
  // the rows of 64 units' two blocks, a unit a lane: looked up one by one, each waited for the codes on their way
  int first = u0;
  int64_t rows[2];
  auto look = [&](int u) {
    first = u;
    rows[0] = row_of(a, at, h, 2 * (u + lane));
    rows[1] = row_of(a, at, h, 2 * (u + lane) + 1);
  };
  look(u0);
  int there = 0, loaded = 0;  // a bit for each block that has a page: of the unit expanded last, of the codes in `next`
  bool huge = false;          // whether there were values that may not be finite
  int* large = reinterpret_cast<int*>(lds + 2 * BUF);  // of each buffer: the last unit of large values
  if (threadIdx.x < 2) large[threadIdx.x] = -1;
  auto load = [&](int u) {
    if (u - first == 64) look(u);
    const int64_t r0 = of_lane(rows[0], u - first), r1 = of_lane(rows[1], u - first);
    loaded = (r0 >= 0 ? 1 : 0) | (r1 >= 0 ? 2 : 0);
    const int64_t row = max(mine ? r1 : r0, (int64_t)0);
    next.load_k(a.c, row, p);
    next.load_v(a.c, row, p);
  };
  auto expand = [&](int u, int buf) {
    there = loaded;
    // values that are not there are zeros; their scores are left out
    const bool gone = !((loaded >> mine) & 1);
    if (gone || KEYS * u + KEYS > at.len) next.cut(gone ? 0 : at.len - KEYS * u - 4 * (p >> 4));
    unsigned char *tk = lds + buf * BUF, *tv = tk + KB;
    next.expand_k(tk, p);
    const bool far_up = __any(next.large());
    if (far_up) {
      large[buf] = u;  // by whichever waves
      huge |= __any(next.huge());
      next.template expand_v<true>(tv, p);
    } else {
      next.template expand_v<false>(tv, p);
    }
  };
  if (u0 < u1) {
    load(u0);
    wait_lds();
    barrier();  // `large` is set
    expand(u0, 0);
    if (u0 + 1 < u1) load(u0 + 1);
  }
  for (int u = u0, buf = 0; u < u1; ++u, buf ^= 1) {
    wait_lds();
    barrier();  // this unit is there, the last one is read
    const int now = there;
    const unsigned char *tk = lds + buf * BUF, *tv = tk + KB;
    if (u + 1 < u1) {
      expand(u + 1, buf ^ 1);
      if (u + 2 < u1) load(u + 2);
    }
    const float lag = __builtin_amdgcn_readfirstlane(large[buf]) == u ? 0.f : LAG;
    if constexpr (Q_PIECES<T> == 3 && DIM == 128) {  // as the registers allow
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (KEYS * u + 32 * e < r.most) r.template keys<1>(a, tk, tv, e, KEYS * u + 32 * e, (now >> e) & 1, lag);
    } else {
      if (KEYS * u < r.most) r.template keys<2>(a, tk, tv, 0, KEYS * u, now, lag);
    }
  }
  auto y = [&](int x) -> float& { return r.out(x); };
  if (__syncthreads_or(huge)) r.template add_huge<DIM / 2>(a, at, h, 2 * u0, min(2 * u1, (at.len + 31) >> 5), 0, y);
  r.l = __fadd_rn(r.l, __shfl_xor(r.l, 32));
  r.template store<DIM / 2>(a, at, h, share, shares, 0, y);
}

// Sequences of few rows, where the products are small beside the reading: each wave takes every fourth 32 keys for
// the same 32 rows by itself, straight from memory into operands, without LDS and barriers: of the keys a lane
// takes its token's half of the channels, of the values 8 tokens' codes of its VT neighbouring channels (the
// loads hold twice that, and neighbouring lanes share them). The next keys load under the exponentials, the next
// values under the next scores. The four waves are joined at the end.
template <typename T, int DIM>
__device__ __forceinline__ void narrow_tile(const Chunk& a, int id, float* all) {
  constexpr int VT = DIM / 32, CB = DIM / 32, PP = P_PIECES<T>;
  constexpr int WORDS = 16 * VT + 2;
  constexpr int DEPTH = sizeof(T) == 4 && DIM == 128 ? 1 : 2;  // blocks on their way, as the registers allow
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hh = lane >> 5;
  Place at;
  int h, share, shares, u0, u1;
  if (!job_of<FEW>(a, id, &at, &h, &share, &shares, &u0, &u1)) return;
  Rows<T, DIM, true> r;
  const int b1 = min(2 * u1, (at.len + 31) >> 5);
  int blk = 2 * u0 + wave, first = 0;
  int64_t rows;  // of 64 of this wave's blocks, one a lane
  auto look = [&](int blk) {
    first = blk;
    rows = row_of(a, at, h, blk + 4 * lane);
  };
  // of the keys the lane's token (row n of the scores), of the values its channels
  const int t = (n & ~12) | ((n & 4) << 1) | ((n & 8) >> 1);
  const uint32_t k_off = t * (DIM / 2) + hh * (DIM / 4), ks_off = (((t & 3) * CB + hh * CB / 2) << 3) + (t >> 2);
  const uint32_t v_off = (n >> 1) * 16 + hh * (DIM == 128 ? 512 : 256), vs_off = n * CB / 32 * 32 + 8 * hh;
  const uint32_t v_take = DIM == 128 ? (n & 1 ? 0x07060302u : 0x05040100u) : (n & 1 ? 0x07050301u : 0x06040200u);
  struct Block {
    int64_t row;
    uint32_t k[DIM / 16], ks[CB / 2], v[2][DIM / 16], vs[2][2];
  } blocks[DEPTH];
  auto load_k = [&](Block& c) {
    const int64_t row = max(c.row, (int64_t)0);  // past the last block, or where there is no page, what is not looked at
    const uint8_t *from = a.c.k + row * (DIM / 2), *bytes = a.c.ks + row * CB;
#pragma unroll
    for (int i = 0; i < DIM / 64; ++i) {
      const v4u x = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(from + k_off + 16 * i));
#pragma unroll
      for (int j = 0; j < 4; ++j) c.k[4 * i + j] = x[j];
      c.ks[i] = bytes[ks_off + 8 * i];
    }
  };
  auto load_v = [&](Block& c) {
    const int64_t row = max(c.row, (int64_t)0);
    const uint8_t *from = a.c.v + row * (DIM / 2), *bytes = a.c.vs + row * CB;
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // 8 tokens: two blocks of 4 (dim 128), or one
#pragma unroll
      for (int i = 0; i < DIM / 64; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(from + v_off + e * (8 * DIM) + 256 * i);
        c.v[e][4 * i] = x.x, c.v[e][4 * i + 1] = x.y, c.v[e][4 * i + 2] = x.z, c.v[e][4 * i + 3] = x.w;
      }
      const uint2 y = *reinterpret_cast<const uint2*>(bytes + vs_off + 16 * e);
      c.vs[e][0] = y.x, c.vs[e][1] = y.y;
    }
  };
  auto find = [&](int blk) {  // blocks in turn
    if (blk - first == 4 * 64) look(blk);
    return blk < b1 ? of_lane(rows, (blk - first) >> 2) : -1;
  };
  look(blk);
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) {
    blocks[i].row = find(blk + 4 * i);
    if (blk < b1) {
      load_k(blocks[i]);
      load_v(blocks[i]);
    }
  }
  r.begin(a, at, h, at.row0);
  bool huge = false;
  auto body = [&](int blk, Block& c) {
    const bool there = c.row >= 0;
    c.row = find(blk + 4 * DEPTH);
    v16f s[1];
    s[0] = zeros16();
#pragma unroll
    for (int e = 0; e < DIM / 16; ++e) {
      const v8bf kf = codes8(c.k[e], scale_bits(c.ks[e * 8 / 32]));
#pragma unroll
      for (int p = Q_PIECES<T> - 1; p >= 0; --p) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, r.q[e].p[p], s[0], 0, 0, 0);
    }
    load_k(c);
    const float top = r.template raise<1>(a, 32 * blk, there, s, LAG);
    // values past the length, or of no page, read as zeros
    if (!there || 32 * blk + 32 > at.len) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!there || 32 * blk + 16 * e + 8 * hh + i >= at.len) {
            if constexpr (DIM == 128) c.v[e][i] = 0;
            else c.v[e][i / 2] &= i & 1 ? 0xffffu : 0xffff0000u;
            c.vs[e][i / 4] = (c.vs[e][i / 4] & ~(255u << (8 * (i & 3)))) | (127u << (8 * (i & 3)));
          }
    }
    const bool large = __any((large_of(c.vs[0][0]) | large_of(c.vs[0][1]) | large_of(c.vs[1][0]) | large_of(c.vs[1][1])) != 0);
    if (large) {
      huge |= __any((huge_of(c.vs[0][0]) | huge_of(c.vs[0][1]) | huge_of(c.vs[1][0]) | huge_of(c.vs[1][1])) != 0);
      r.follow(a, top, 0.f);
    }
    const float ref = r.template base<1>(a, s);
    float sums[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const Pieces<PP> f = r.template weights<1>(a, s, ref, e, sums + e);
      uint32_t x[8][VT / 2];  // token i's channels, two at a time
      auto four = [&]<int Z>() {
        const uint32_t b = c.vs[e][Z];
        const float s0 = scale_byte<0>(b), s1 = scale_byte<1>(b), s2 = scale_byte<2>(b), s3 = scale_byte<3>(b);
        if constexpr (DIM == 128) {  // the lane's halves of two tokens in one word
          const uint32_t w0 = __builtin_amdgcn_perm(c.v[e][4 * Z + 1], c.v[e][4 * Z], v_take);
          const uint32_t w1 = __builtin_amdgcn_perm(c.v[e][4 * Z + 3], c.v[e][4 * Z + 2], v_take);
          x[4 * Z][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s0, 0));
          x[4 * Z][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s0, 1));
          x[4 * Z + 1][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s1, 2));
          x[4 * Z + 1][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s1, 3));
          x[4 * Z + 2][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w1, s2, 0));
          x[4 * Z + 2][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w1, s2, 1));
          x[4 * Z + 3][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w1, s3, 2));
          x[4 * Z + 3][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w1, s3, 3));
        } else {  // its bytes of four
          const uint32_t w = __builtin_amdgcn_perm(c.v[e][2 * Z + 1], c.v[e][2 * Z], v_take);
          x[4 * Z][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s0, 0));
          x[4 * Z + 1][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s1, 1));
          x[4 * Z + 2][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s2, 2));
          x[4 * Z + 3][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s3, 3));
        }
      };
      four.template operator()<0>();
      four.template operator()<1>();
      if (large)  // what is not finite is added at the end
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int z = 0; z < VT / 2; ++z)
            x[i][z] &= ((x[i][z] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) |
                       ((x[i][z] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
#pragma unroll
      for (int d = 0; d < VT; ++d) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(x[2 * i + 1][d / 2], x[2 * i][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
        const v8bf vf = __builtin_bit_cast(v8bf, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int p = PP - 1; p >= 0; --p) r.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, f.p[p], r.o[d], 0, 0, 0);
      }
    }
    r.l = __fadd_rn(r.l, __fadd_rn(sums[0], sums[1]));
    load_v(c);
  };
  for (; blk < b1; blk += 4 * DEPTH) {
    body(blk, blocks[0]);
    if (DEPTH == 2 && blk + 4 < b1) body(blk + 4, blocks[DEPTH - 1]);
  }
  // a quarter of the outputs by each wave, from all four
  constexpr int N = DIM / 8;
  float* to = all + wave * (WORDS * 64) + lane;
  to[0] = r.m;
  to[64] = __fadd_rn(r.l, __shfl_xor(r.l, 32));
#pragma unroll
  for (int x = 0; x < DIM / 2; ++x) to[(2 + x) * 64] = r.out(x);
  huge = __syncthreads_or(huge);
  const float* from = all + lane;
  float ms[4], f[4], y[N];
#pragma unroll
  for (int w = 0; w < 4; ++w) ms[w] = from[w * (WORDS * 64)];
  r.m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  r.l = 0.f;
#pragma unroll
  for (int x = 0; x < N; ++x) y[x] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = ms[w] == r.m ? 1.f : factor(ms[w], r.m, a.scale2);
    r.l = __fmaf_rn(from[w * (WORDS * 64) + 64], f[w], r.l);
#pragma unroll
    for (int x = 0; x < N; ++x) y[x] = __fmaf_rn(from[(w * WORDS + 2 + wave * N + x) * 64], f[w], y[x]);
  }
  auto part = [&](int x) -> float& { return y[x]; };
  if (huge) r.template add_huge<N>(a, at, h, 2 * u0, b1, wave * N, part);
  r.template store<N>(a, at, h, share, shares, wave * N, part);
}

// Both in one launch, the wide tiles first; or narrow ones alone, with less LDS and fewer registers. Three workgroups a
// CU where 64 channels of 16-bit types allow it (f16's wide tiles took 176 registers of the 168 by themselves).
template <typename T, int DIM, bool WIDES>
__global__ __launch_bounds__(256, DIM == 64 && sizeof(T) == 2 ? 3 : 2) void kv4_chunk_kernel(Chunk a) {
  constexpr int TILES = WIDES ? 4 * KEYS * DIM * 2 : 0, JOIN = 4 * (DIM / 2 + 2) * 256, BYTES = TILES > JOIN ? TILES : JOIN;
  static_assert(!WIDES || BYTES >= TILES + 8);  // the tiles, and which of them hold large values
  __shared__ __attribute__((aligned(1024))) unsigned char lds[BYTES];
  const int wides = a.wide.tiles * a.wide.most * a.c.heads;
  if constexpr (WIDES)
    if ((int)blockIdx.x < wides) return wide_tile<T, DIM>(a, blockIdx.x, lds);
  narrow_tile<T, DIM>(a, blockIdx.x - wides, reinterpret_cast<float*>(lds));
}

// The shares of each row joined: a wave a row and head.
template <typename T, int DIM>
__global__ __launch_bounds__(256) void kv4_chunk_join_kernel(Chunk a) {
  constexpr int C = DIM / 64;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, heads = a.c.heads * a.group;
  if (id >= (int64_t)a.n * heads) return;
  const int i = (int)(id / heads), qh = (int)(id - (int64_t)i * heads), h = qh / a.group, j = qh - h * a.group;
  int lo = 0, hi = a.B;  // the last b with cu[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid + 1] <= i) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= a.B || i < a.cu[lo]) return;  // of no sequence: written as zeros
  Place at;
  const int e = min(max(a.cu[lo + 1], 0), a.n);
  at.b = lo;
  at.start = min(max(a.cu[lo], 0), a.n);
  at.rows = (e - at.start) * a.group;
  at.len = max(0, min(a.lens[lo], a.max_len));
  at.base = a.lens[lo] - (e - at.start);
  const int row = (i - at.start) * a.group + j;
  const int shares = at.rows > a.least ? shares_of(a.wide.upper, units_of<WIDE>(a, at, row / WIDE * WIDE))
                                       : shares_of(a.few.upper, units_of<FEW>(a, at, row / FEW * FEW));
  if (shares == 1) return;
  const int64_t slot = slot_of(a, at, row, h);
  float m = -INFINITY, l = 0.f, y[C] = {};
  // up to 64 shares at a time: their maxima and sums a lane each, then their rows, whose loads wait for nothing
  for (int s0 = 0; s0 < shares; s0 += 64) {
    const int mine = min(64, shares - s0);
    float2 st = make_float2(-INFINITY, 0.f);
    if (lane < mine) st = *reinterpret_cast<const float2*>(a.stats + (slot + s0 + lane) * 2);
    float now = st.x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) now = fmaxf(now, __shfl_xor(now, d));
    now = fmaxf(now, m);
    const float f = m == now ? 1.f : factor(m, now, a.scale2), e = st.x == now ? 1.f : factor(st.x, now, a.scale2);
    m = now;
    l = __fmaf_rn(l, f, wave_sum_fixed(__fmul_rn(st.y, e)));
#pragma unroll
    for (int c = 0; c < C; ++c) y[c] = fabsf(y[c]) < INFINITY ? __fmul_rn(y[c], f) : y[c];
    for (int i0 = 0; i0 < mine; i0 += 8) {
      float x[8][C];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) x[i][c] = a.part[(slot + s0 + min(i0 + i, mine - 1)) * DIM + C * lane + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float ei = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), min(i0 + i, mine - 1)));
        if (i0 + i < mine)
#pragma unroll
          for (int c = 0; c < C; ++c)  // what is not finite stays so, also where its factor is 0
            y[c] = fabsf(x[i][c]) < INFINITY ? __fmaf_rn(x[i][c], ei, y[c]) : __fadd_rn(y[c], x[i][c]);
      }
    }
  }
  const float r = __fdiv_rn(1.f, l == 0.f ? 1.f : l);
  T* to = (T*)a.out + id * DIM + C * lane;
#pragma unroll
  for (int c = 0; c < C; ++c) to[c] = (T)__fmul_rn(y[c], r);
}

// How the work is cut, whatever the lengths are.
//
// A sequence takes wide tiles from more than FEW_ROWS rows on; a call of up to FEW_ALL rows takes narrow tiles alone,
// for more workgroups. Above FEW_MOST rows, where every sequence may fill a wide tile, it takes them if the estimates
// below say so. In narrow and in wide tiles on one card, 32 heads over 8 of 128, bf16 unless said:
//   24 new tokens in each of 32 sequences of 3000 78 and 100 us, 32 of them 103 and 116, 1024 over 8192 in
//   f16 (4096 rows) 308 and 270: wide ones are taken; 12 in each of the 32 sequences (1536 rows, narrow either way) 55,
//   and 71 in the launch that has both
//   512 tokens (2048 rows) over 4096 62 and 72, over 16384 232 and 217, over 65536 925 and 810
//   128 tokens (512 rows) over 4096 28 and 36, over 16384 72 and 70, over 65536 252 and 218 (f16 288 and 263, f32 376
//   and 390; narrow ones are taken); 64 tokens over 65536 137 and 163
//   32 and 17 tokens over 65536 and 50001, 24 heads over 4, f16: 100 and 140
//
// Of the shares that a tile may be cut in that number is taken for which the estimated time is least: of the longest
// workgroup, of all the work over the workgroups that run at once and the longest begun last, or of whole rounds of
// equal ones; the workgroups that find no tile; and what the join writes and reads. Narrow tiles' usual length is what
// the cache's pages hold for each sequence: with the longest sequence's for all, one chunk of 1024 tokens beside 511
// sequences of one over 1000 took 866 us, so 230 (268 with weights in two pieces). So are wide tiles' where every
// sequence may have some (three chunks of 512, 500 and 333 tokens over 4096, 1500 and 777, f32: 130 -> 107 us). Narrow
// tiles beside wide ones are cut only where they would last longer: the join alone, over all rows, is 15 us of 2048
// tokens of 32 heads.
constexpr int64_t FEW_ROWS = 64, FEW_ALL = 2048, FEW_MOST = 512;
static_assert(2 * (FEW_ROWS + 1) > WIDE);
constexpr double FEW_UNIT_US = 1.2, NONE_US = 4.0;  // a unit of a narrow tile's; a workgroup that finds no tile
struct Cut {
  Chunk::Kind wide, few;
  int64_t least;
};
static Chunk::Kind kind_of(int64_t most_tiles, int64_t tiles, int64_t heads, int64_t units, double usual, int64_t at_once,
                           double unit_us, double share_us, double* took) {
  Chunk::Kind k = {(int)most_tiles, (int)units, 1};
  double least = 0.0;
  if (tiles < 1) tiles = 1;
  for (int64_t m = 1; m <= 128 && m <= units; ++m) {
    const int64_t all = tiles * heads * m, each = (units + m - 1) / m, none = most_tiles * heads * m - all;
    double length = (double)each;
    if (all > at_once) {
      const double work = tiles * heads * usual / at_once + each * (1.0 - (double)at_once / all);
      const double rounds = (all + at_once - 1) / at_once * usual / m;
      length = fmax(length, fmax(work, rounds));
    }
    const double us = fmax(length * unit_us + (none > 0 ? NONE_US * none / at_once : 0.0), *took) +
                      (m > 1 ? 4.0 + m * share_us : 0.0);
    if (m == 1 || us < least) {
      least = us;
      k.upper = (int)each;
      k.most = (int)((units + each - 1) / each);
    }
  }
  *took = least;
  return k;
}
static Cut cut_of(int type, int64_t n, int64_t B, int64_t heads, int64_t group, int64_t dim, int64_t max_len, int64_t tokens) {
  const int64_t units = max_len > 0 ? (max_len + KEYS - 1) / KEYS : 1, begun = B + 2 < n ? B + 2 : n, rows = n * group;
  const double share_us = (double)rows * heads * (2 * 4 * (dim + 2)) / 4e6;  // of all rows, written and read at 4 TB/s
  // workgroups that run at once (two a CU, three where the registers allow), and a unit's time in one of them then;
  // bf16's is that of weights in one piece: 2.6 for 64 channels, as measured with two, cuts 8192 tokens over 8192 in
  // two (562 us for 445), 2.9 for 128 changes nothing
  const int64_t at_once = dim == 64 && type ? 768 : 512;
  const double unit_us = dim == 64 ? (type == 0 ? 3.3 : type == 1 ? 2.0 : 2.4) : type == 0 ? 5.5 : type == 1 ? 2.3 : 3.7;
  const double mean = B < 1 ? 1.0 : (double)tokens / KEYS / B, usual = mean < units ? mean : (double)units;
  auto narrow_kind = [&](double each_us, double* took) {
    const int64_t tiles = (rows + FEW - 1) / FEW, some = B < n ? B : n;
    return kind_of(rows / FEW + begun, tiles > some ? tiles : some, heads, units, usual, at_once, each_us, share_us, took);
  };
  auto wide_kind = [&](double* took) {
    // more than FEW_ROWS rows are at most 2 tiles for every WIDE + 1
    const int64_t many = rows / (FEW_ROWS + 1), tiles = rows / WIDE + (begun < many ? begun : many);
    const int64_t most = 2 * rows / (WIDE + 1);
    return kind_of(tiles < most ? tiles : most, rows / WIDE, heads, units, B <= rows / WIDE ? usual : (double)units,
                   at_once, unit_us, share_us, took);
  };
  bool wide = rows > FEW_ALL;
  if (!wide && rows > FEW_MOST && B <= rows / WIDE) {  // a unit of a narrow tile's beside others of the same sequence
    const double each_us = dim == 64 ? (type == 0 ? 0.8 : type == 1 ? 0.5 : 0.66) : type == 0 ? 1.33 : type == 1 ? 0.66 : 0.97;
    double narrow_us = 0.0, wide_us = 0.0;
    narrow_kind(each_us, &narrow_us);
    wide_kind(&wide_us);
    wide = wide_us < narrow_us;
  }
  double took = 0.0;  // of the wide tiles, beside which the narrow ones run
  Cut c = {{0, 1, 1}, {}, 0x7fffffff};
  if (wide) {
    c.least = FEW_ROWS;
    c.wide = wide_kind(&took);
    const int64_t full = rows / FEW + begun, two = begun * (FEW_ROWS / FEW);
    c.few = kind_of(full < two ? full : two, B < 1 ? 1 : B, heads, units, usual, at_once, FEW_UNIT_US, share_us, &took);
  } else {
    c.few = narrow_kind(FEW_UNIT_US, &took);
  }
  return c;
}

template <typename T, int DIM>
static int launch(const char* what, const Chunk& a, hipStream_t st) {
  auto grid = [&](const Chunk::Kind& k) { return (unsigned)((int64_t)k.tiles * k.most * a.c.heads); };
  if (a.wide.tiles) kv4_chunk_kernel<T, DIM, true><<<grid(a.wide) + grid(a.few), 256, 0, st>>>(a);
  else kv4_chunk_kernel<T, DIM, false><<<grid(a.few), 256, 0, st>>>(a);
  if (a.wide.most > 1 || a.few.most > 1) {
    const int64_t rows = (int64_t)a.n * a.c.heads * a.group;
    kv4_chunk_join_kernel<T, DIM><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(a);
  }
  return check_launch(what);
}

}  // namespace bq

using namespace bq;

size_t bq_kv4_attend_chunk_ws_bytes(int type, int64_t n, int64_t B, int64_t q_heads, int64_t heads, int64_t dim,
                                    int64_t max_len, int64_t tokens) {
  if (n < 1 || B < 0 || heads < 1 || q_heads < heads || dim < 1 || max_len < 0 || tokens < 0) return 0;
  const Cut c = cut_of(type, n, B, heads, q_heads / heads, dim, max_len, tokens);
  const int most = c.wide.most > c.few.most ? c.wide.most : c.few.most;
  return most > 1 ? (size_t)n * q_heads * most * (dim + 2) * 4 : 0;
}

int bq_kv4_attend_chunk(const bq_kv4_cache* cache, const void* q, int type, int64_t n, int64_t q_heads, int64_t q_token,
                        int64_t q_head, const int32_t* table, int64_t B, int64_t width, const int32_t* lens,
                        const int32_t* cu, int64_t max_len, float scale, void* out, void* ws, size_t ws_bytes,
                        bq_stream_t stream) {
  const char* what = "bq_kv4_attend_chunk";
  Chunk a;
  if (const int rc = kv4_of(what, cache, table, B, width, &a.c)) return rc;
  if (type < 0 || type > 2) return set_error(BQ_ERR_ARG, "%s: type %d", what, type);
  if (n < 0 || n > 0x7fffffff - 8192 || q_heads < 1 || q_heads > 65535 || max_len < 0 || max_len > 0x7fffffff - 8192)
    return set_error(BQ_ERR_ARG, "%s: bad sizes", what);
  if (q_heads % cache->heads)
    return set_error(BQ_ERR_ARG, "%s: %lld query heads over %lld key-value heads", what, (long long)q_heads,
                     (long long)cache->heads);
  if (!(scale > 0.f) || !(scale < 1e30f)) return set_error(BQ_ERR_ARG, "%s: scale %g", what, (double)scale);
  if (n == 0) return BQ_OK;
  const int64_t group = q_heads / cache->heads;
  if (n * group > 0x7fffffff - 8192) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  const Cut cut = cut_of(type, n, B, cache->heads, group, cache->dim, max_len, cache->pages * cache->page);
  auto grid = [&](const Chunk::Kind& k) { return (int64_t)k.tiles * k.most * cache->heads; };
  if (grid(cut.wide) + grid(cut.few) > 0x7fffffff || n * q_heads > 0x7fffffffll * 4)
    return set_error(BQ_ERR_ARG, "%s: size too large", what);
  if (!q || !cu || !out || (B && !lens)) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const int64_t size = type == KV4_F32 ? 4 : 2;
  if ((((uintptr_t)q | (uintptr_t)out) & 15) || (q_token | q_head) * size % 16)
    return set_error(BQ_ERR_ARG, "%s: rows that are not 16-byte aligned", what);
  const size_t need = bq_kv4_attend_chunk_ws_bytes(type, n, B, q_heads, cache->heads, cache->dim, max_len,
                                                   cache->pages * cache->page);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    return set_error(BQ_ERR_ARG, "%s: a workspace of %zu bytes, given %zu", what, need, ws ? ws_bytes : 0);
  const int64_t held = cache->pages ? width * cache->page : 0;  // tokens that a sequence's pages have room for
  a.lens = lens;
  a.cu = cu;
  a.q = q;
  a.qt = q_token;
  a.qh = q_head;
  a.n = (int)n;
  a.group = (int)group;
  a.B = (int)B;
  a.max_len = (int)(max_len < held ? max_len : held);
  a.wide = cut.wide;
  a.few = cut.few;
  a.least = (int)cut.least;
  a.by_group = fast_div((uint32_t)group);
  a.scale2 = scale * 1.4426950408889634f;
  a.out = out;
  a.part = (float*)ws;
  a.stats = a.part + (need ? need / (cache->dim + 2) / 4 * cache->dim : 0);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = cache->dim == 128;
  if (type == KV4_F32) return wide ? launch<float, 128>(what, a, st) : launch<float, 64>(what, a, st);
  if (type == KV4_BF16) return wide ? launch<__bf16, 128>(what, a, st) : launch<__bf16, 64>(what, a, st);
  return wide ? launch<_Float16, 128>(what, a, st) : launch<_Float16, 64>(what, a, st);
}
