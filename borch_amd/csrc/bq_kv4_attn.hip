// Attention of the newest tokens over a cache held in 4 bits (its form: bq_kv4.h).
//
// For sequence b with n = lens[b] cached tokens, the newest T of them the queries', query token t
// of query head h sees the first n - T + 1 + t: out = sum_i p_i v_i with p = softmax(scale q . k_i),
// zeros where it sees nothing. The G = q_heads / heads query heads of a key-value head and the T
// tokens are the rows of one product, R = T G.
//
// A wave takes 32 cached tokens at a time, straight from memory into MFMA operands (no LDS): the
// scores transposed, S^T = k q^T, 16 x 16 x 32, so that lane (n, g) of column n = lane % 16 and
// g = lane / 16 holds row n's scores for tokens 8 g .. 8 g + 7, which is the second product's
// operand as it stands: O^T = v^T p^T. The codes become bf16 exactly (a code has 2 significant
// bits, bf16 the exponents of f32). q enters as the exact sum of bf16 pieces (f32: 3, f16: 2,
// bf16: 1) and p, in [0, 1], as pieces too (f32: 3, the 16-bit types: 2, so that p's error is
// 2^-17 where the output's rounding is 2^-9 or 2^-12), with f32 accumulation.
// The contracted index of the scores is permuted (lane group g takes a quarter of the channels) and
// so are the rows of v^T (row m of product j is channel DIM / 16 m + j), both to load whole pieces.
//
// Each row keeps its running maximum, sum and output (one pass over the cache). A workgroup of four
// waves takes tokens of one sequence for one key-value head and 16 RT rows, and joins its waves in
// LDS. Short caches: a workgroup a (sequence, head, rows). Long ones: all their units of 128 tokens
// in one line, cut into equal shares for as many workgroups as the GPU holds at once (lengths are
// the device's knowledge, and a share has one beginning and one end however unlike they are); a
// (sequence, head, rows) that lies in several shares leaves (maximum, sum, output) of each in the
// workspace, and a second kernel joins them. What the cached tokens received (the softmax weights
// summed over the rows) needs the final maximum and sum of each row: a last kernel takes the scores
// again, each token by one workgroup, so that sums are added without atomics, in one order.
//
// Bound by the codes, read once: 64 sequences of 200 to 16384 tokens, 8 heads of 128, bf16, 32 query
// heads: 338 MB in 63 us, 5.4 TB/s, and 5 us to join; two of 131072 and 100001, f32: 251 MB in 58 us,
// 4.3 TB/s. A streaming read of 4 GiB reaches 7.0 TB/s, a copy 4.75 (read and written).
#include <math.h>

#include "bq_kv4_pieces.h"

namespace bq {

struct Attend {
  Kv4 c;
  const int* lens;
  const void* q;
  int64_t qb, qt, qh;  // strides in elements: sequence, token, head
  int tokens, group, rows, row_groups, max_len, B;
  int shares, least;  // workgroups of the line (0: one a sequence, head and rows), the least units a share
  FastDiv by_group;
  float scale2;  // scale * log2(e)
  void* out;     // [B][tokens][heads * group][DIM]
  float *part, *stats;  // shares' first and last parts [2 shares][16 RT][DIM + 2]; [B heads][rows][2]
  float* weights;
  int64_t wb, wh;
};

// q's pieces as the score product's second operand: rows row0 .. + 15, step s, of lane (n, g) row
// row0 + n, channels DIM / 4 g + 8 s ..; rows past the last as zeros.
template <typename T, int DIM>
__device__ __forceinline__ Pieces<Q_PIECES<T>> q_frag(const Attend& a, int b, int h, int row0, int s) {
  constexpr int P = Q_PIECES<T>;
  const int lane = threadIdx.x & 63, row = row0 + (lane & 15), g = lane >> 4;
  const int t = fdiv(row, a.by_group.mul, a.by_group.shift), j = row - t * a.group;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (row < a.rows)
    load8f((const T*)a.q + b * a.qb + t * a.qt + (int64_t)(h * a.group + j) * a.qh + DIM / 4 * g + 8 * s, x);
  return split_q<P>(x);
}
// The operands of RT row tiles in LDS, once for the four waves (in registers they took a third of
// them in f32, and a wave a SIMD): a lane reads its own 16 bytes.
template <typename T, int DIM, int RT>
struct QTile {
  uint4 p[RT][DIM / 32][Q_PIECES<T>][64];
  __device__ __forceinline__ void fill(const Attend& a, int b, int h, int row0) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < (RT * (DIM / 32) + 3) / 4; ++i) {
      const int x = 4 * i + wave, r = x / (DIM / 32), s = x % (DIM / 32);
      if (x >= RT * (DIM / 32)) break;
      const Pieces<Q_PIECES<T>> f = q_frag<T, DIM>(a, b, h, row0 + 16 * r, s);
#pragma unroll
      for (int k = 0; k < Q_PIECES<T>; ++k) p[r][s][k][lane] = __builtin_bit_cast(uint4, f.p[k]);
    }
  }
  __device__ __forceinline__ v8bf at(int r, int s, int k) const {
    return __builtin_bit_cast(v8bf, p[r][s][k][threadIdx.x & 63]);
  }
};

// One row tile's in a wave's registers, for the sums (f32, 16 tokens of 32 heads over 16384: 61 -> 57 us
// for the call; in LDS there was room for three workgroups a CU).
template <typename T, int DIM>
struct QRegs {
  Pieces<Q_PIECES<T>> f[DIM / 32];
  __device__ __forceinline__ v8bf at(int, int s, int k) const { return f[s].p[k]; }
};

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
// 16 bytes of codes, read once a call: past the caches' other contents.
__device__ __forceinline__ uint4 codes_at(const uint8_t* p) {
  const v4u x = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p));
  return make_uint4(x[0], x[1], x[2], x[3]);
}

// What a lane loads of 32 tokens' keys: of token 8 (n / 4) + 4 t + n % 4, its quarter g of the
// channels (row n of score tile t), and the scale bytes of both tiles' tokens.
template <int DIM>
struct KBlock {
  uint32_t w[2][DIM / 32];
  uint32_t scales;
  __device__ __forceinline__ void load(const Kv4& c, int at, int h, int off0) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const size_t row = Kv4At<DIM>::row(c, at, h, off0);
    const uint8_t* p = c.k + Kv4At<DIM>::k(row) + (8 * (n >> 2) + (n & 3)) * (DIM / 2) + g * (DIM / 8);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (DIM == 128) {
        const uint4 x = codes_at(p + t * 4 * (DIM / 2));
        w[t][0] = x.x, w[t][1] = x.y, w[t][2] = x.z, w[t][3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p + t * 4 * (DIM / 2));
        w[t][0] = x.x, w[t][1] = x.y;
      }
    }
    scales = *reinterpret_cast<const uint16_t*>(c.ks + row * (DIM / 32) + ((n & 3) * (DIM / 32) + g * (DIM / 32) / 4) * 8 +
                                                2 * (n >> 2));
  }
  // The scores of 16 rows a tile, before the scale: [4 t + i] is token 8 g + 4 t + i
  template <typename T, int RT, typename Q>
  __device__ __forceinline__ void scores(const Q& q, float (&s)[RT][8]) const {
    v8bf kf[2][DIM / 32];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < DIM / 32; ++i) kf[t][i] = codes8(w[t][i], scale_bits((scales >> (8 * t)) & 255));
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      v4f acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int k = Q_PIECES<T> - 1; k >= 0; --k)  // the smallest pieces first
#pragma unroll
        for (int i = 0; i < DIM / 32; ++i) {
          const v8bf f = q.at(r, i, k);
#pragma unroll
          for (int t = 0; t < 2; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][i], f, acc[t], 0, 0, 0);
        }
#pragma unroll
      for (int e = 0; e < 8; ++e) s[r][e] = acc[e / 4][e % 4];
    }
  }
};

// Of 32 tokens' values: of tokens 8 g .. 8 g + 7, channel slice n (DIM / 16 channels).
template <int DIM>
struct VBlock {
  uint32_t w[8];  // token i's slice: 8 codes (DIM 128), or two tokens' 4 codes each
  uint32_t s[2];  // scale bytes, four tokens a dword
  __device__ __forceinline__ void load(const Kv4& c, int at, int h, int off0) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const size_t row = Kv4At<DIM>::row(c, at, h, off0);
    const uint8_t* p = c.v + row * (DIM / 2);
    if constexpr (DIM == 128) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 x = codes_at(p + (2 * g + e) * 256 + n * 16);
        w[4 * e] = x.x, w[4 * e + 1] = x.y, w[4 * e + 2] = x.z, w[4 * e + 3] = x.w;
      }
    } else {
      const uint4 x = codes_at(p + g * 256 + n * 16);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    }
    const uint2 y = *reinterpret_cast<const uint2*>(c.vs + row * (DIM / 32) + n * (DIM / 32) / 16 * 32 + 8 * g);
    s[0] = y.x, s[1] = y.y;
  }
  __device__ __forceinline__ uint32_t byte(int i) const { return (s[i >> 2] >> (8 * (i & 3))) & 255; }
  __device__ __forceinline__ void clear(int i) {  // token i reads as zeros
    s[i >> 2] = (s[i >> 2] & ~(255u << (8 * (i & 3)))) | (127u << (8 * (i & 3)));
    if constexpr (DIM == 128) w[i] = 0;
    else w[i >> 1] &= i & 1 ? 0xffffu : 0xffff0000u;
  }
  // The first operand of products 2 k and 2 k + 1 (channels DIM / 16 n + 2 k and + 1), 8 tokens each.
  template <int K>
  __device__ __forceinline__ void frags(v8bf& even, v8bf& odd) const {
    uint32_t e[4], o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b;
      if constexpr (DIM == 128) {
        a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[2 * i], scale_bits(byte(2 * i)), K));
        b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[2 * i + 1], scale_bits(byte(2 * i + 1)), K));
      } else {
        a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i], scale_bits(byte(2 * i)), K));
        b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i], scale_bits(byte(2 * i + 1)), K + 2));
      }
      e[i] = __builtin_amdgcn_perm(b, a, 0x05040100u);
      o[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    }
    even = __builtin_bit_cast(v8bf, make_uint4(e[0], e[1], e[2], e[3]));
    odd = __builtin_bit_cast(v8bf, make_uint4(o[0], o[1], o[2], o[3]));
  }
};

// exp2(c (s - m)) with an empty row's maximum, -infinity, taken as 0
__device__ __forceinline__ float weight_of(float s, float base, float c) {
  return __builtin_amdgcn_exp2f(__fmul_rn(__fsub_rn(s, base), c));
}
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

constexpr int UNIT = 128;  // tokens: a block of 32 a wave
// Places of the line that stand for the beginning and the end of a run (its queries, its pages, the
// join of the waves): a share of many short runs is not longer than one of few long ones.
constexpr int EDGE = 3;

__device__ __forceinline__ int len_of(const Attend& a, int b) { return max(0, min(a.lens[b], a.max_len)); }
__device__ __forceinline__ int units_of(int len) { return max(1, (len + UNIT - 1) / UNIT); }  // an empty one writes zeros

__device__ __forceinline__ int scan64(int v) {  // over the wave, this lane's with those before it
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(v, d);
    if (lane >= d) v += y;
  }
  return v;
}
// The line: sequence after sequence, per_b (heads times row groups) runs of each, EDGE places and then
// its units. Its length, and of the sequence `seq`, or of that in which place at(line) lies (seq < 0),
// the number and the place where its runs begin. Up to 64 sequences are looked at once.
template <typename F>
__device__ __forceinline__ int line_of(const Attend& a, int per_b, int seq, F&& at, int* which, int* begin) {
  const int lane = threadIdx.x & 63;
  auto mine = [&](int b0) { return b0 + lane < a.B ? (EDGE + units_of(len_of(a, b0 + lane))) * per_b : 0; };
  const int first = mine(0), upto0 = scan64(first);
  int line = __builtin_amdgcn_readlane(upto0, 63);
  for (int b0 = 64; b0 < a.B; b0 += 64) line += __builtin_amdgcn_readlane(scan64(mine(b0)), 63);
  const int x = seq < 0 ? at(line) : 0;
  int from = 0, u = first, upto = upto0;
  *which = max(seq, 0);
  *begin = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    if (b0) {
      u = mine(b0);
      upto = scan64(u);
    }
    const uint64_t hit = __ballot(seq < 0 ? from + upto > x : b0 + lane == seq);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      *which = b0 + l;
      *begin = from + __builtin_amdgcn_readlane(upto - u, l);
      break;
    }
    from += __builtin_amdgcn_readlane(upto, 63);
  }
  return line;
}
__device__ __forceinline__ int share_of(const Attend& a, int line) { return max(a.least, (line + a.shares - 1) / a.shares); }

template <typename T, int DIM, int RT>
__global__ __launch_bounds__(256, 2) void kv4_attend_kernel(Attend a) {
  constexpr int PP = P_PIECES<T>, NJ = DIM / 16, PITCH = DIM + 4;
  __shared__ __attribute__((aligned(16))) float so[4][16][PITCH];
  __shared__ float sm[4][16], sl[4][16];
  __shared__ QTile<T, DIM, RT> q;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int per_b = a.c.heads * a.row_groups, bpp = a.c.page >> 5;

  // this workgroup's places x0 .. x1 of the line
  int x0, x1, b, begin;
  if (a.shares) {
    const int line = line_of(a, per_b, -1, [&](int n) { return (int)blockIdx.x * share_of(a, n); }, &b, &begin);
    x0 = blockIdx.x * share_of(a, line);
    if (x0 >= line) return;
    x1 = min(line, x0 + share_of(a, line));
  } else {
    b = blockIdx.x / per_b;
    const int run = EDGE + units_of(len_of(a, b));
    begin = 0;
    x0 = (blockIdx.x - b * per_b) * run;
    x1 = x0 + run;
  }
  for (int x = x0; x < x1;) {
    const int len = len_of(a, b), units = units_of(len);
    const int pair = (x - begin) / (EDGE + units), h = pair / a.row_groups, row0 = (pair - h * a.row_groups) * 16 * RT;
    const int run = begin + pair * (EDGE + units) + EDGE;  // where this run's units begin
    const int u0 = max(0, x - run), u1 = min(units, x1 - run);
    x = run + units;  // the next run
    const int seq = b;
    if (x == begin + (EDGE + units) * per_b) {
      begin = x;
      ++b;
    }
    if (u0 >= u1) continue;  // its beginning only
    const int sure = len - a.tokens + 1;  // tokens that every row sees
    const int blocks = (len + 31) >> 5;

    // up to 64 units at a time: this wave's block of each, their pages one a lane; the first block's
    // codes are on their way while the queries are split
    int first, mine, pages;
    KBlock<DIM> k0, k1;
    VBlock<DIM> v0, v1;
    auto fetch = [&](int i, KBlock<DIM>& k, VBlock<DIM>& v) {
      const int blk = first + 4 * i;
      const int at = max(0, __builtin_amdgcn_readlane(pages, i));
      const int off0 = (blk - fdiv(blk, a.c.by_blocks.mul, a.c.by_blocks.shift) * bpp) << 5;
      k.load(a.c, at, h, off0);
      v.load(a.c, at, h, off0);
    };
    auto look = [&](int w0) {
      first = 4 * w0 + wave;
      mine = min(min(64, u1 - w0), blocks > first ? (blocks - first + 3) >> 2 : 0);
      pages = -1;
      if (lane < mine) pages = kv4_page(a.c, seq, fdiv(first + 4 * lane, a.c.by_blocks.mul, a.c.by_blocks.shift));
      if (mine > 0) fetch(0, k0, v0);
    };
    look(u0);
    q.fill(a, seq, h, row0);  // every wave has left the last run's: the join's barriers
    int end[RT];              // what this lane's row sees
    bool lost[RT];            // whether it sees a NaN value in its channels that left the products
    float m[RT], l[RT];
    v4f o[RT][NJ];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int t = fdiv(row0 + 16 * r + n, a.by_group.mul, a.by_group.shift);
      end[r] = min(len, sure + t);
      lost[r] = false;
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[r][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();

    for (int w0 = u0; w0 < u1; w0 += 64) {
      if (w0 > u0) look(w0);
      auto body = [&](int i, const KBlock<DIM>& kb, VBlock<DIM>& vb) {
        const int tok = (first + 4 * i) << 5;
        if (__builtin_amdgcn_readlane(pages, i) < 0) return;  // no page: nothing to see
        float s[RT][8];
        kb.template scores<T, RT>(q, s);
        if (tok + 32 > sure) {
          // The end: what a row does not see gets no weight, and no NaN of it (0 times NaN) may reach the
          // row, so such values leave the products (bit e: token 8 g + e of this lane's slice); past
          // the length everything does.
          uint32_t nans = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int t = tok + 8 * g + e;
#pragma unroll
            for (int r = 0; r < RT; ++r)
              if (t >= end[r]) s[r][e] = -INFINITY;
            if (t >= sure && (t >= len || vb.byte(e) == 255)) {
              if (t < len) nans |= 1u << e;
              vb.clear(e);
            }
          }
          if (__any(nans != 0)) {
            // the rows that do see one get NaN in its 32 channels. Lane (n, g) of O holds channels DIM / 4 g ..,
            // whose scale is that of v's slice 4 g, in the lanes of each token group u
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint64_t who = __ballot((nans >> e) & 1);
              for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int r = 0; r < RT; ++r) lost[r] |= ((who >> (16 * u + 4 * g)) & 1) && tok + 8 * u + e < end[r];
            }
          }
        }
        Pieces<PP> p[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          float top = s[r][0];
#pragma unroll
          for (int e = 1; e < 8; ++e) top = fmaxf(top, s[r][e]);
          top = max_xor32(max_xor16(top));
          // the maximum that is subtracted lags by up to 2^8 (the weights' own size cancels in the quotient)
          const bool grew = __fmul_rn(__fsub_rn(top, m[r]), a.scale2) > 8.f;
          if (__any(grew)) {
            const float f = grew ? weight_of(m[r], top, a.scale2) : 1.f;
            m[r] = grew ? top : m[r];
            l[r] = __fmul_rn(l[r], f);
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[r][j] *= f;
          }
          const float base = base_of(m[r]);
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            w[e] = weight_of(s[r][e], base, a.scale2);
            l[r] = __fadd_rn(l[r], w[e]);
          }
          p[r] = pieces_of<PP>(w);
        }
        auto product = [&]<int K>() {
          v8bf f[2];
          vb.template frags<K>(f[0], f[1]);
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
              for (int k = PP - 1; k >= 0; --k)
                o[r][2 * K + z] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[z], p[r].p[k], o[r][2 * K + z], 0, 0, 0);
        };
        product.template operator()<0>();
        product.template operator()<1>();
        if constexpr (DIM == 128) {
          product.template operator()<2>();
          product.template operator()<3>();
        }
      };
      for (int i = 0; i < mine; i += 2) {
        if (i + 1 < mine) fetch(i + 1, k1, v1);
        body(i, k0, v0);
        if (i + 1 >= mine) break;
        if (i + 2 < mine) fetch(i + 2, k0, v0);
        body(i + 1, k1, v1);
      }
    }

    // the four waves' rows together: lane (n, g) holds channels DIM / 4 g + DIM / 16 i + j of row n
    const size_t bh = (size_t)seq * a.c.heads + h;
    const bool whole = u0 == 0 && u1 == units;
    float* part = a.part + ((size_t)2 * blockIdx.x + (x0 <= run)) * (16 * RT) * (DIM + 2);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      l[r] = __fadd_rn(l[r], __shfl_xor(l[r], 16));
      l[r] = __fadd_rn(l[r], __shfl_xor(l[r], 32));
      __syncthreads();  // the last rows are read
      if (g == 0) {
        sm[wave][n] = m[r];
        sl[wave][n] = l[r];
      }
      const float nan = lost[r] ? NAN : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ; j += 4)
          *reinterpret_cast<float4*>(&so[wave][n][DIM / 4 * g + NJ * i + j]) =
              make_float4(__fadd_rn(o[r][j][i], nan), __fadd_rn(o[r][j + 1][i], nan), __fadd_rn(o[r][j + 2][i], nan),
                          __fadd_rn(o[r][j + 3][i], nan));
      __syncthreads();
      constexpr int LANES = DIM / 4;  // threads a row, four channels each
      for (int z = threadIdx.x; z < 16 * LANES; z += 256) {
        const int rr = z / LANES, c4 = z % LANES * 4, row = row0 + 16 * r + rr;
        if (row >= a.rows) continue;
        const float top = fmaxf(fmaxf(sm[0][rr], sm[1][rr]), fmaxf(sm[2][rr], sm[3][rr])), base = base_of(top);
        float sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = weight_of(sm[w][rr], base, a.scale2);
          const float4 v = *reinterpret_cast<const float4*>(&so[w][rr][c4]);
          sum = __fmaf_rn(f, sl[w][rr], sum);
          y.x = __fmaf_rn(f, v.x, y.x);
          y.y = __fmaf_rn(f, v.y, y.y);
          y.z = __fmaf_rn(f, v.z, y.z);
          y.w = __fmaf_rn(f, v.w, y.w);
        }
        if (!whole) {
          float* to = part + (16 * r + rr) * (DIM + 2);
          *reinterpret_cast<float2*>(to + c4) = make_float2(y.x, y.y);
          *reinterpret_cast<float2*>(to + c4 + 2) = make_float2(y.z, y.w);
          if (c4 == 0) *reinterpret_cast<float2*>(to + DIM) = make_float2(top, sum);
        } else {
          const float d = sum == 0.f ? 1.f : sum;
          const int t = fdiv(row, a.by_group.mul, a.by_group.shift), j = row - t * a.group;
          T* to = (T*)a.out + (((size_t)seq * a.tokens + t) * a.c.heads * a.group + h * a.group + j) * DIM + c4;
          store4(to, __fdiv_rn(y.x, d), __fdiv_rn(y.y, d), __fdiv_rn(y.z, d), __fdiv_rn(y.w, d));
          if (a.weights && c4 == 0) *reinterpret_cast<float2*>(a.stats + (bh * a.rows + row) * 2) = make_float2(top, d);
        }
      }
    }
  }
}

// The parts of one row joined, where its units lie in several shares: a workgroup a row, its waves the
// parts in turn.
template <typename T, int DIM, int RT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void kv4_join_kernel(Attend a) {
  __shared__ float sm[WAVES], sl[WAVES], so[WAVES][DIM];
  const int row = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rg = row / (16 * RT), units = units_of(len_of(a, b));
  int begin, seq;
  const int share = share_of(a, line_of(a, a.c.heads * a.row_groups, b, [](int) { return 0; }, &seq, &begin));
  begin += (h * a.row_groups + rg) * (EDGE + units) + EDGE;
  const int w0 = begin / share, w1 = (begin + units - 1) / share;
  if (w0 == w1) return;  // whole in one share, and written there
  const float* rows = a.part + (size_t)(row - rg * 16 * RT) * (DIM + 2);
  constexpr int C = DIM / 64;
  float top = -INFINITY, sum = 0.f, y[C] = {};
  auto part_of = [&](int w) { return rows + ((size_t)2 * w + (w * share <= begin)) * (16 * RT) * (DIM + 2); };
  // up to 64 of this wave's parts at a time: their maxima and sums a lane each, then their rows, whose
  // loads wait for nothing
  for (int f0 = w0 + wave; f0 <= w1; f0 += 64 * WAVES) {
    const int mine = min(64, (w1 - f0) / WAVES + 1);
    float2 ms = make_float2(-INFINITY, 0.f);
    if (lane < mine) ms = *reinterpret_cast<const float2*>(part_of(f0 + WAVES * lane) + DIM);
    float now = ms.x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) now = fmaxf(now, __shfl_xor(now, d));
    now = fmaxf(now, top);
    const float base = base_of(now), f = weight_of(top, base, a.scale2), e = weight_of(ms.x, base, a.scale2);
    top = now;
    sum = __fmaf_rn(sum, f, wave_sum_fixed(__fmul_rn(ms.y, e)));
#pragma unroll
    for (int c = 0; c < C; ++c) y[c] = __fmul_rn(y[c], f);
    for (int i0 = 0; i0 < mine; i0 += 8) {
      float x[8][C];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* p = part_of(f0 + WAVES * min(i0 + i, mine - 1)) + C * lane;  // past the last: a weight of 0
#pragma unroll
        for (int c = 0; c < C; ++c) x[i][c] = p[c];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float ei = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), i0 + i));
#pragma unroll
        for (int c = 0; c < C; ++c) y[c] = __fmaf_rn(x[i][c], ei, y[c]);
      }
    }
  }
  if (lane == 0) sm[wave] = top, sl[wave] = sum;
#pragma unroll
  for (int c = 0; c < C; ++c) so[wave][C * lane + c] = y[c];
  __syncthreads();
  if (wave) return;
  float now = sm[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) now = fmaxf(now, sm[w]);
  const float base = base_of(now);
  sum = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) y[c] = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float f = weight_of(sm[w], base, a.scale2);
    sum = __fmaf_rn(f, sl[w], sum);
#pragma unroll
    for (int c = 0; c < C; ++c) y[c] = __fmaf_rn(f, so[w][C * lane + c], y[c]);
  }
  const float d = sum == 0.f ? 1.f : sum;
  const int t = fdiv(row, a.by_group.mul, a.by_group.shift), j = row - t * a.group;
  T* to = (T*)a.out + (((size_t)b * a.tokens + t) * a.c.heads * a.group + h * a.group + j) * DIM + C * lane;
#pragma unroll
  for (int c = 0; c < C; ++c) to[c] = (T)__fdiv_rn(y[c], d);
  if (a.weights && lane == 0)
    *reinterpret_cast<float2*>(a.stats + (((size_t)b * a.c.heads + h) * a.rows + row) * 2) = make_float2(now, d);
}

// Of 8 tokens' weights a lane, 16 rows: lane n < 8 of a group gets the sum of token n over the rows.
__device__ __forceinline__ float over_rows(float (&total)[8]) {
  const int n = threadIdx.x & 15;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int d = 1; d < 16; d *= 2) total[e] = __fadd_rn(total[e], __shfl_xor(total[e], d));
  }
  float mine = total[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) mine = n == e ? total[e] : mine;
  return mine;
}

// What each cached token received, added to its sum: the scores once more, each row's weight from its
// final maximum and sum. A workgroup's waves take the row tiles in turn over the same 32 BLOCKS tokens;
// the rows of a tile are added over lanes, the tiles of a wave and the waves in order.
// Bound by the queries, which each workgroup loads and splits again: 64 tokens and two waves where the
// work is cut in shares, 32 and four else, where latency counts (us for the call, f32, 32 heads of 128
// over 8: 16 sequences of 8192, 8 tokens 144, 212; two of 1000, 16 tokens 25.9, 24.7).
template <typename T, int DIM, int WAVES, int BLOCKS>
__global__ __launch_bounds__(WAVES * 64) void kv4_weights_kernel(Attend a) {
  __shared__ float sums[WAVES][32 * BLOCKS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int blk = blockIdx.x * BLOCKS, h = blockIdx.y, b = blockIdx.z;
  const int len = len_of(a, b), tok = blk << 5;
  if (tok >= len) return;
  const size_t bh = (size_t)b * a.c.heads + h;
  KBlock<DIM> kb[BLOCKS] = {};
  int at[BLOCKS];
  float total[BLOCKS][8] = {};
#pragma unroll
  for (int z = 0; z < BLOCKS; ++z) {
    const int pi = fdiv(blk + z, a.c.by_blocks.mul, a.c.by_blocks.shift);
    at[z] = tok + 32 * z < len ? kv4_page(a.c, b, pi) : -1;
    if (at[z] >= 0) kb[z].load(a.c, at[z], h, (blk + z - pi * (a.c.page >> 5)) << 5);
  }
#pragma unroll 1
  for (int row0 = 16 * wave; row0 < a.rows; row0 += 16 * WAVES) {
    const int row = row0 + n, t = fdiv(row, a.by_group.mul, a.by_group.shift);
    const int end = row < a.rows ? min(len, len - a.tokens + 1 + t) : 0;
    float2 st = make_float2(0.f, 1.f);
    if (row < a.rows) st = *reinterpret_cast<const float2*>(a.stats + (bh * a.rows + row) * 2);
    QRegs<T, DIM> q;
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) q.f[i] = q_frag<T, DIM>(a, b, h, row0, i);
    const float base = base_of(st.x), part = __fdiv_rn(1.f, st.y);
#pragma unroll
    for (int z = 0; z < BLOCKS; ++z) {
      float s[1][8];
      kb[z].template scores<T, 1>(q, s);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (tok + 32 * z + 8 * g + e < end)
          total[z][e] = __fmaf_rn(weight_of(s[0][e], base, a.scale2), part, total[z][e]);
    }
  }
#pragma unroll
  for (int z = 0; z < BLOCKS; ++z) {
    const float mine = over_rows(total[z]);
    if (n < 8) sums[wave][32 * z + 8 * g + n] = mine;
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int z = 0; z < BLOCKS; ++z) {
    const int i = 32 * z + 8 * g + n;
    if (n < 8 && tok + i < len && at[z] >= 0) {
      float all = sums[0][i];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) all = __fadd_rn(all, sums[w][i]);
      float* to = a.weights + b * a.wb + h * a.wh + tok + i;
      *to = __fadd_rn(*to, all);
    }
  }
}

// The same of one row tile: a workgroup takes 128 tokens, its waves 32 each, the queries in LDS.
template <typename T, int DIM>
__global__ __launch_bounds__(256) void kv4_weights_one_kernel(Attend a) {
  __shared__ QTile<T, DIM, 1> q;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  const int blk = blockIdx.x * 4 + wave, h = blockIdx.y, b = blockIdx.z;
  const int len = len_of(a, b), tok = blk << 5;
  if ((int)blockIdx.x * 128 >= len) return;
  const int pi = fdiv(blk, a.c.by_blocks.mul, a.c.by_blocks.shift);
  const int at = tok < len ? kv4_page(a.c, b, pi) : -1;
  KBlock<DIM> kb = {};
  if (at >= 0) kb.load(a.c, at, h, (blk - pi * (a.c.page >> 5)) << 5);
  q.fill(a, b, h, 0);
  __syncthreads();
  const int end = n < a.rows ? min(len, len - a.tokens + 1 + fdiv(n, a.by_group.mul, a.by_group.shift)) : 0;
  float2 st = make_float2(0.f, 1.f);
  if (n < a.rows) st = *reinterpret_cast<const float2*>(a.stats + (((size_t)b * a.c.heads + h) * a.rows + n) * 2);
  float s[1][8], total[8];
  kb.template scores<T, 1>(q, s);
  const float base = base_of(st.x), part = __fdiv_rn(1.f, st.y);
#pragma unroll
  for (int e = 0; e < 8; ++e) total[e] = tok + 8 * g + e < end ? __fmul_rn(weight_of(s[0][e], base, a.scale2), part) : 0.f;
  const float mine = over_rows(total);
  const int t = tok + 8 * g + n;
  if (n < 8 && t < len && at >= 0) {
    float* to = a.weights + b * a.wb + h * a.wh + t;
    *to = __fadd_rn(*to, mine);
  }
}

// How the work is cut: row tiles a workgroup (of 16), and the most shares of the line, 0 for a
// workgroup a (sequence, head, rows): up to LEAST_UNITS units, where the line's second kernel costs more
// than it saves (us whole and cut, heads of 128: 300 tokens, f32 10.3, 14.1; 1000, 24 heads over 4, f32
// 14.3, 14.9, bf16 11.1, 14.7; 100 sequences of 1000, 32 over 8, bf16 30, 38; 1500, f32 18.8, 14.8; ten of
// 2000, bf16 23.4, 15.9).
struct Cut {
  int tiles, row_groups, shares;
};
// Two row tiles read the codes once for 32 rows, one lets more workgroups run at once: one up to
// ONE_TILE places of the line (us in one and in two, f16, heads of 128: 24 heads over 4, 16 tokens over
// 1100 (288 places) 15.0, 18.6; 32 over 8, two of 4000, 16 tokens (2240) 21.5, 24.6; 32 over 4, two of
// 65536, 4 tokens (8240) 40.2, 41.8; 32 over 8, four of 8192, 32 tokens (17152) 73.6, 70.9; sixteen of
// 16384, 8 tokens (33536) 126, 114).
constexpr int MOST_SHARES = 256 * 4;
constexpr int LEAST_UNITS = 8;
constexpr int ONE_TILE = 12 * 1024;
static Cut cut_of(int64_t B, int64_t heads, int64_t rows, int64_t max_len) {
  Cut c;
  const int64_t units = (max_len + UNIT - 1) / UNIT, groups = (rows + 15) / 16;
  c.tiles = groups == 1 || B * heads * groups <= ONE_TILE / (EDGE + units) ? 1 : 2;
  c.row_groups = (int)((groups + c.tiles - 1) / c.tiles);
  const int64_t line = B * heads * c.row_groups * (EDGE + units), most = MOST_SHARES;
  c.shares = units <= LEAST_UNITS ? 0 : (int)(line < most ? line : most);
  return c;
}

// As many shares as workgroups run at once, by the registers (64 sequences of unlike lengths, bf16,
// 2 / 3 / 4 a CU: 77, 69, 80 us; two of 131072, f32: 70, 64, 75). A row is joined by two waves where it has
// up to 16 parts on average, else by eight (us by two and by eight, heads of 128: 200 sequences of 2000,
// 32 heads over 8, bf16 94, 110; two of 131072 and 100001, f32 62.8, 61.3; one of 131072, 8 over 1, f32
// 23.4, 17.0).
template <typename T, int DIM, int RT>
static void launch_rows(Attend a, hipStream_t st) {
  constexpr int PER_CU = (RT == 1 ? 3 : 2) + (DIM == 64);
  if (a.shares > 256 * PER_CU) a.shares = 256 * PER_CU;
  const unsigned grid = a.shares ? a.shares : a.B * a.c.heads * a.row_groups;
  kv4_attend_kernel<T, DIM, RT><<<grid, 256, 0, st>>>(a);
  if (!a.shares) return;
  const dim3 rows(a.rows, a.c.heads, a.B);
  if (a.B * a.c.heads * a.row_groups >= a.shares / 16) kv4_join_kernel<T, DIM, RT, 2><<<rows, 128, 0, st>>>(a);
  else kv4_join_kernel<T, DIM, RT, 8><<<rows, 512, 0, st>>>(a);
}

template <typename T, int DIM>
static int launch(const char* what, const Attend& a, int tiles, hipStream_t st) {
  if (tiles == 1) launch_rows<T, DIM, 1>(a, st);
  else launch_rows<T, DIM, 2>(a, st);
  if (a.weights && a.max_len > 0) {
    if (a.rows <= 16)
      kv4_weights_one_kernel<T, DIM><<<dim3((a.max_len + 127) / 128, a.c.heads, a.B), 256, 0, st>>>(a);
    else if (a.shares)
      kv4_weights_kernel<T, DIM, 2, 2><<<dim3((a.max_len + 63) / 64, a.c.heads, a.B), 128, 0, st>>>(a);
    else
      kv4_weights_kernel<T, DIM, 4, 1><<<dim3((a.max_len + 31) / 32, a.c.heads, a.B), 256, 0, st>>>(a);
  }
  return check_launch(what);
}

// Whether the weights of B sequences and `heads` heads, `most` each, share no place: the one axis' rows lie within
// a step of the other.
static bool rows_apart(int64_t B, int64_t seq, int64_t heads, int64_t head, int64_t most) {
  auto nested = [&](int64_t n, int64_t step, int64_t outer_n, int64_t outer) {
    const __int128 in = step < 0 ? -(__int128)step : step, out = outer < 0 ? -(__int128)outer : outer;
    return (n < 2 || in >= most) && (outer_n < 2 || out >= (n - 1) * in + most);
  };
  return most == 0 || nested(heads, head, B, seq) || nested(B, seq, heads, head);
}

}  // namespace bq

using namespace bq;

size_t bq_kv4_attend_ws_bytes(int64_t B, int64_t heads, int64_t rows, int64_t dim, int64_t max_len, int weights) {
  if (B < 1 || heads < 1 || rows < 1 || dim < 1 || max_len < 0) return 0;
  const Cut c = cut_of(B, heads, rows, max_len);
  return (weights ? (size_t)B * heads * rows * 8 : 0) + (size_t)2 * c.shares * 16 * c.tiles * (dim + 2) * 4;
}

int bq_kv4_attend(const bq_kv4_cache* cache, const void* q, int type, int64_t tokens, int64_t q_heads, int64_t q_seq,
                  int64_t q_token, int64_t q_head, const int32_t* table, int64_t B, int64_t width, const int32_t* lens,
                  int64_t max_len, float scale, void* out, float* weights, int64_t w_seq, int64_t w_head, void* ws,
                  size_t ws_bytes, bq_stream_t stream) {
  const char* what = "bq_kv4_attend";
  Attend a;
  if (const int rc = kv4_of(what, cache, table, B, width, &a.c)) return rc;
  if (type < 0 || type > 2) return set_error(BQ_ERR_ARG, "%s: type %d", what, type);
  if (tokens < 0 || q_heads < 1 || max_len < 0 || max_len > 0x7fffffff - 8192)
    return set_error(BQ_ERR_ARG, "%s: bad sizes", what);
  if (q_heads % cache->heads)
    return set_error(BQ_ERR_ARG, "%s: %lld query heads over %lld key-value heads", what, (long long)q_heads,
                     (long long)cache->heads);
  if (!(scale > 0.f) || !(scale < 1e30f)) return set_error(BQ_ERR_ARG, "%s: scale %g", what, (double)scale);
  if (B == 0 || tokens == 0) return BQ_OK;
  const int64_t group = q_heads / cache->heads;
  if (tokens > 1 << 20 || group > 1 << 10 || B > 65535) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  const int64_t rows = tokens * group;
  if (rows > 1 << 20) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  const Cut cut = cut_of(B, cache->heads, rows, max_len);
  // the line and the places after its end that shares would begin at, within 32 bits
  if (B * cache->heads * cut.row_groups > (0x7fffffff - 8 * MOST_SHARES) / ((max_len + UNIT - 1) / UNIT + 1 + EDGE))
    return set_error(BQ_ERR_ARG, "%s: size too large", what);
  if (!q || !lens || !out) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const int64_t size = type == KV4_F32 ? 4 : 2;
  if ((((uintptr_t)q | (uintptr_t)out) & 15) || (q_seq | q_token | q_head) * size % 16)
    return set_error(BQ_ERR_ARG, "%s: rows that are not 16-byte aligned", what);
  const int64_t held = cache->pages ? width * cache->page : 0;  // tokens that a sequence's pages have room for
  // several workgroups would add to one place
  if (weights && !rows_apart(B, w_seq, cache->heads, w_head, max_len < held ? max_len : held))
    return set_error(BQ_ERR_ARG, "%s: weights of sequences or heads overlap", what);
  const size_t need = bq_kv4_attend_ws_bytes(B, cache->heads, rows, cache->dim, max_len, weights != nullptr);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    return set_error(BQ_ERR_ARG, "%s: a workspace of %zu bytes, given %zu", what, need, ws ? ws_bytes : 0);
  a.lens = lens;
  a.q = q;
  a.qb = q_seq;
  a.qt = q_token;
  a.qh = q_head;
  a.tokens = (int)tokens;
  a.group = (int)group;
  a.rows = (int)rows;
  a.row_groups = cut.row_groups;
  a.B = (int)B;
  a.shares = cut.shares;
  a.least = EDGE + 1;
  a.max_len = (int)(max_len < held ? max_len : held);
  a.by_group = fast_div((uint32_t)group);
  a.scale2 = scale * 1.4426950408889634f;
  a.out = out;
  a.stats = (float*)ws;
  a.part = a.stats + (weights ? (size_t)B * cache->heads * rows * 2 : 0);
  a.weights = weights;
  a.wb = w_seq;
  a.wh = w_head;
  hipStream_t st = (hipStream_t)stream;
  const bool wide = cache->dim == 128;
  if (type == KV4_F32) return wide ? launch<float, 128>(what, a, cut.tiles, st) : launch<float, 64>(what, a, cut.tiles, st);
  if (type == KV4_BF16) return wide ? launch<__bf16, 128>(what, a, cut.tiles, st) : launch<__bf16, 64>(what, a, cut.tiles, st);
  return wide ? launch<_Float16, 128>(what, a, cut.tiles, st) : launch<_Float16, 64>(what, a, cut.tiles, st);
}
