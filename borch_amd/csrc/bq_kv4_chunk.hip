// Attention of chunks of new tokens over a cache held in 4 bits (its form: bq_kv4.h): prompts read in
// pieces, alone or beside sequences that add one token.
//
// Sequence b's new tokens are the rows cu[b] .. cu[b + 1] of q, the last ones of its lens[b] cached
// tokens: row i is token lens[b] - cu[b + 1] + i and sees the tokens up to itself,
// out = sum_i p_i v_i with p = softmax(scale q . k_i), zeros where it sees nothing.
//
// One pass over the keys with each row's running maximum and sum. The G = q_heads / heads query heads
// of a key-value head and the chunk's tokens are the rows of one product (row t G + j: token t, head j),
// so that the codes are expanded once for all that read them. A workgroup of four waves takes a tile of
// 128 rows, 32 a wave, and 64 keys at a time: the codes, loaded one tile ahead, become bf16 exactly (a
// code has 2 significant bits, bf16 the exponents of f32) in LDS, two tiles in turn, one barrier a tile.
// The scores are taken transposed, S^T = k q^T on the 32 x 32 x 16 MFMA, keys in an order (bits 2 and 3 of
// their number exchanged) that leaves 8 following tokens in 8 following registers of a lane: the
// exponentials are, register for register, the second operand of O^T = v^T p^T. q enters as the exact sum of
// bf16 pieces (f32: 3, f16: 2, bf16: 1), p as pieces too (f32: 3, f16: 2, so that p's error is 2^-17 where
// the output's rounding is 2^-12; bf16: 1, half a step of 2^-8 on each term as the output), with f32
// accumulation. Tiles of up to 64 rows give two waves the halves of each 64 keys for the same rows; of up
// to 32, where a product is small beside the reading, each wave takes every fourth 32 keys by itself,
// without barriers. Such waves are joined in LDS at the end.
//
// The maximum that is subtracted lags by up to 2^8 (the weights' own size cancels in the quotient) and is
// a whole number of powers of two, so that a weight is one FMA and one exp2 and all of a row's agree.
//
// A tile's keys are cut into shares of up to `upper` units of 64 where the tiles alone would leave the GPU
// part empty; a second kernel joins the shares of a row.
#include "bq_dma.h"
#include "bq_kv4_pieces.h"

namespace bq {

typedef float v16f __attribute__((ext_vector_type(16)));

struct Chunk {
  Kv4 c;
  const int *lens, *cu;
  const void* q;
  int64_t qt, qh;  // strides in elements: token, head
  int n, group, B, max_len, tiles, upper, most;  // upper: units a share; most: shares a tile at most
  FastDiv by_group;
  float scale2;  // scale * log2(e)
  void* out;     // [n][heads * group][DIM]
  float *part, *stats;  // of each row, head and share: [n group][heads][most][DIM], [..][2]
};

constexpr int TILE = 128, KEYS = 64;  // rows a tile; keys a unit

// A tile's sequence and rows.
struct Place {
  int b, start, rows, row0;  // b: -1 for rows of no sequence; the first row of q, the sequence's rows, the tile's first
  int base, len;             // the place in the cache of the sequence's first new token, and its tokens
};

// Tile `place` of what lies before cu[0], of each sequence in turn, or of what lies past the last.
__device__ __forceinline__ bool place_of(const Chunk& a, int place, Place* out) {
  const int lane = threadIdx.x & 63;
  for (int at = 0; at < a.B + 2; at += 64) {
    const int i = at + lane;
    int s = 0, e = 0;
    if (i <= a.B + 1) {
      s = i == 0 ? 0 : min(max(a.cu[i - 1], 0), a.n);
      e = i == a.B + 1 ? a.n : min(max(a.cu[i], 0), a.n);
    }
    const int rows = max(0, e - s) * a.group, mine = (rows + TILE - 1) / TILE;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
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
      out->base = real ? a.lens[seq - 1] - (__builtin_amdgcn_readlane(e, l) - out->start) : 0;
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
__device__ __forceinline__ int units_of(const Chunk& a, const Place& at, int row0) {
  return (end_of(a, at, min(row0 + TILE, at.rows) - 1) + KEYS - 1) / KEYS;
}
__device__ __forceinline__ int shares_of(const Chunk& a, int units) { return max(1, (units + a.upper - 1) / a.upper); }

// A row's weights are relative to 2^ref, ref a whole number near its lagging maximum; or, where that
// passes 2^20, to the maximum itself.
constexpr float FAR = 0x1p20f;
__device__ __forceinline__ float ref_of(float m, float c) { return m == -INFINITY ? 0.f : rintf(__fmul_rn(m, c)); }
// From weights of one maximum to those of another.
__device__ __forceinline__ float factor(float from, float to, float c) {
  if (from == -INFINITY) return 0.f;
  const float a = ref_of(from, c), b = ref_of(to, c);
  return __builtin_amdgcn_exp2f(fmaxf(fabsf(a), fabsf(b)) > FAR ? __fmul_rn(__fsub_rn(from, to), c) : __fsub_rn(a, b));
}

// Where a 16-byte piece lies in LDS: row `row` of the keys, channels 8 piece ..; channel `ch` of the
// values, tokens 8 piece ... XORed so that 16 lanes cover all banks.
template <int DIM>
__device__ __forceinline__ int k_at(int row, int piece) {
  return DIM == 128 ? row * 256 + ((piece ^ (row & 15)) << 4) : row * 128 + ((piece ^ ((row >> 1) & 7)) << 4);
}
__device__ __forceinline__ int v_at(int ch, int piece) { return ch * 128 + ((piece ^ (((ch >> 1) ^ (ch >> 3)) & 7)) << 4); }

constexpr uint32_t HUGE = 253;  // scale bytes from here on may make codes infinite or NaN

// One of the 256 pieces of 64 tokens' codes: of token p / 4 a quarter of the keys' channels, of tokens
// 4 (p / 16) .. + 3 channel slice p % 16 of the values. Pieces p / 128 lie in one block of 32 tokens.
template <int DIM>
struct Codes {
  uint32_t k[DIM / 32], v[DIM / 32], ks, vs;
  __device__ __forceinline__ void load(const Kv4& c, int at, int h, int off0, int p) {
    const size_t row = Kv4At<DIM>::row(c, at, h, off0);
    const int t = (p & 127) >> 2, quarter = p & 3, four = (p & 127) >> 4, n = p & 15;
    const uint8_t* kp = c.k + (row + t) * (DIM / 2) + quarter * (DIM / 8);
    const uint8_t* vp = c.v + row * (DIM / 2);
    if constexpr (DIM == 128) {
      const uint4 x = *reinterpret_cast<const uint4*>(kp), y = *reinterpret_cast<const uint4*>(vp + four * 256 + n * 16);
      k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w;
      v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(kp);
      const uint2 y = *reinterpret_cast<const uint2*>(vp + (four >> 1) * 256 + n * 16 + (four & 1) * 8);
      k[0] = x.x, k[1] = x.y;
      v[0] = y.x, v[1] = y.y;
    }
    constexpr int CB = DIM / 32;
    ks = c.ks[row * CB + (((t & 3) * CB + quarter * CB / 4) << 3) + (t >> 2)];
    vs = *reinterpret_cast<const uint32_t*>(c.vs + row * CB + n * CB / 16 * 32 + 4 * four);
  }
  __device__ __forceinline__ void none() {
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) k[i] = v[i] = 0;
    ks = 127, vs = 0x7f7f7f7fu;
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
  __device__ __forceinline__ bool huge() const {
    return max(max(vs & 255, (vs >> 8) & 255), max((vs >> 16) & 255, vs >> 24)) >= HUGE;
  }
  // Into a tile in LDS, as bf16. What is not finite among the values becomes 0 (it is added at the end).
  __device__ __forceinline__ void expand(unsigned char* tk, unsigned char* tv, int p) const {
    const int t = p >> 2, row = (t & ~12) | ((t & 4) << 1) | ((t & 8) >> 1);
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i)
      *reinterpret_cast<v8bf*>(tk + k_at<DIM>(row, (p & 3) * (DIM / 32) + i)) = codes8(k[i], scale_bits(ks));
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = scale_bits((vs >> (8 * i)) & 255);
    const bool odd = huge();
    auto two = [&]<int K>() {
      uint32_t x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DIM == 128) x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[i], s[i], K));
        else if (i & 1) x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[i >> 1], s[i], K + 2));
        else x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[i >> 1], s[i], K));
        if (odd)
          x[i] &= ((x[i] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((x[i] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
      }
      const int ch = (p & 15) * (DIM / 16) + 2 * K, to = (p >> 4) >> 1, half = ((p >> 4) & 1) * 8;
      *reinterpret_cast<uint2*>(tv + v_at(ch, to) + half) =
          make_uint2(__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u));
      *reinterpret_cast<uint2*>(tv + v_at(ch + 1, to) + half) =
          make_uint2(__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u));
    };
    two.template operator()<0>();
    two.template operator()<1>();
    if constexpr (DIM == 128) {
      two.template operator()<2>();
      two.template operator()<3>();
    }
  }
};

__device__ __forceinline__ v16f zeros16() {
  v16f z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

template <typename T>
constexpr int W_PIECES = __is_same(T, float) ? 3 : __is_same(T, _Float16) ? 2 : 1;

template <typename T, int DIM>
__global__ __launch_bounds__(256, 2) void kv4_chunk_kernel(Chunk a) {
  constexpr int QP = Q_PIECES<T>, PP = W_PIECES<T>, STEPS = DIM / 16, VT = DIM / 32;
  constexpr int KB = KEYS * DIM * 2, BUF = 2 * KB;  // bytes of a tile's keys, as many of its values
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * BUF];
  __shared__ int flags[2][4];  // of each buffer what its waves found: 1 the block is there, 2 values that are huge
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hh = lane >> 5;
  const int h = blockIdx.x % a.c.heads, rest = blockIdx.x / a.c.heads, share = rest % a.most;
  Place at;
  if (!place_of(a, a.tiles - 1 - rest / a.most, &at)) return;
  const int units = units_of(a, at, at.row0), shares = shares_of(a, units);
  if (share >= shares) return;
  const int u0 = (int)((int64_t)units * share / shares), u1 = (int)((int64_t)units * (share + 1) / shares);
  const int rows = min(TILE, at.rows - at.row0);
  const int parts = rows <= 32 ? 4 : rows <= 64 ? 2 : 1, part = wave & (parts - 1);
  const int wrow = at.row0 + wave / parts * 32, row = wrow + n;  // the wave's first row and this lane's
  const int last = at.rows - 1;
  const int end = end_of(a, at, min(row, last));
  const int sure = end_of(a, at, min(wrow, last)), most_end = end_of(a, at, min(wrow + 31, last));
  const bool works = wrow <= last;
  const int bpp = a.c.page >> 5, blocks = (at.len + 31) >> 5;

  Pieces<QP> qf[STEPS];
  {
    const int t = fdiv(row, a.by_group.mul, a.by_group.shift), j = row - t * a.group;
    const T* q = (const T*)a.q + (int64_t)(at.start + t) * a.qt + (int64_t)(h * a.group + j) * a.qh + 8 * hh;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (row <= last && at.b >= 0) load8f(q + 16 * s, x);
      qf[s] = split_q<QP>(x);
    }
  }
  float m = -INFINITY, l = 0.f;
  v16f o[VT];
#pragma unroll
  for (int d = 0; d < VT; ++d) o[d] = zeros16();

  int huge = 0;  // whether there were values that may not be finite
  auto page_of = [&](int blk) {
    return blk < blocks ? kv4_page(a.c, at.b, fdiv(blk, a.c.by_blocks.mul, a.c.by_blocks.shift)) : -1;
  };
  auto off_of = [&](int blk) { return (blk - fdiv(blk, a.c.by_blocks.mul, a.c.by_blocks.shift) * bpp) << 5; };

  // SUB times 32 keys from `tok`, in a tile's places from 32 sub on; there: a bit for each 32 that has a page
  auto products = [&]<int SUB>(const unsigned char* tk, const unsigned char* tv, int sub, int tok, int there) {
    v16f s[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      s[u] = zeros16();
#pragma unroll
      for (int e = 0; e < STEPS; ++e) {
        const v8bf kf = *reinterpret_cast<const v8bf*>(tk + k_at<DIM>(32 * (sub + u) + n, 2 * e + hh));
#pragma unroll
        for (int p = QP - 1; p >= 0; --p) s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[e].p[p], s[u], 0, 0, 0);
      }
    }
    if (tok + 32 * SUB > sure || there != (1 << SUB) - 1)
#pragma unroll
      for (int i = 0; i < 16 * SUB; ++i)
        if (tok + 32 * (i / 16) + 16 * (i % 16 / 8) + 8 * hh + i % 8 >= end || !((there >> (i / 16)) & 1))
          s[i / 16][i % 16] = -INFINITY;
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * SUB; ++i) top = fmaxf(top, s[i / 16][i % 16]);
    top = max_xor32(top);
    const bool grew = __fmul_rn(__fsub_rn(top, m), a.scale2) > 8.f;
    if (__any(grew)) {
      const float f = grew ? factor(m, top, a.scale2) : 1.f;
      m = grew ? top : m;
      l = __fmul_rn(l, f);
#pragma unroll
      for (int d = 0; d < VT; ++d) o[d] *= f;
    }
    const float ref = ref_of(m, a.scale2);
    const bool far = fabsf(ref) > FAR;
    if (__any(far)) {
#pragma unroll
      for (int i = 0; i < 16 * SUB; ++i) {
        float x = s[i / 16][i % 16];
        x = far ? __fmul_rn(__fsub_rn(x, m), a.scale2) : __fmaf_rn(x, a.scale2, -ref);
        s[i / 16][i % 16] = x = __builtin_amdgcn_exp2f(x);
        l = __fadd_rn(l, x);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16 * SUB; ++i) {
        const float x = __builtin_amdgcn_exp2f(__fmaf_rn(s[i / 16][i % 16], a.scale2, -ref));
        s[i / 16][i % 16] = x;
        l = __fadd_rn(l, x);
      }
    }
#pragma unroll
    for (int e = 0; e < 2 * SUB; ++e) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = s[e / 2][8 * (e % 2) + i];
      const Pieces<PP> pf = pieces_of<PP>(x);
#pragma unroll
      for (int d = 0; d < VT; ++d) {
        const v8bf vf = *reinterpret_cast<const v8bf*>(tv + v_at(32 * d + n, 4 * sub + 2 * e + hh));
#pragma unroll
        for (int p = PP - 1; p >= 0; --p) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf.p[p], o[d], 0, 0, 0);
      }
    }
  };

  if (parts == 4) {  // each wave by itself: blocks of 32 keys 4 apart
    unsigned char *tk = lds + (wave >> 1) * BUF, *tv = tk + KB;
    const int sub = wave & 1, b1 = min(2 * u1, blocks), p0 = sub * 128 + lane;
    Codes<DIM> now[2];
    int page = -1, next_page = -1;
    auto load = [&](int blk) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (page < 0) {
          now[e].none();
        } else {
          now[e].load(a.c, page, h, off_of(blk), p0 + 64 * e);
          if (32 * blk + 32 > at.len) now[e].cut(at.len - 32 * blk - 4 * (((p0 + 64 * e) & 127) >> 4));
        }
      }
    };
    int blk = 2 * u0 + wave;
    if (blk < b1) {
      page = page_of(blk);
      next_page = page_of(blk + 4);
      load(blk);
    }
    for (; blk < b1; blk += 4) {
      // one wave's own part of LDS: its accesses there run in order
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const bool there = page >= 0;
      if (__any(now[0].huge() || now[1].huge())) huge = 1;
#pragma unroll
      for (int e = 0; e < 2; ++e) now[e].expand(tk, tv, p0 + 64 * e);
      page = next_page;
      next_page = page_of(blk + 8);
      if (blk + 4 < b1) load(blk + 4);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (there) products.template operator()<1>(tk, tv, sub, 32 * blk, 1);
    }
  } else {
    Codes<DIM> next;
    const int p = threadIdx.x, mine = wave >> 1;  // which of a unit's two blocks
    int page = -1, next_page = -1;
    auto load = [&](int u) {
      if (page < 0) {
        next.none();
      } else {
        next.load(a.c, page, h, off_of(2 * u + mine), p);
        if (KEYS * u + KEYS > at.len) next.cut(at.len - KEYS * u - 4 * (p >> 4));
      }
    };
    auto expand = [&](int buf) {
      const bool odd = __any(next.huge());
      if (lane == 0) flags[buf][wave] = (page >= 0 ? 1 : 0) | (odd ? 2 : 0);
      next.expand(lds + buf * BUF, lds + buf * BUF + KB, p);
    };
    if (u0 < u1) {
      page = page_of(2 * u0 + mine);
      next_page = page_of(2 * u0 + 2 + mine);
      load(u0);
      expand(0);
      page = next_page;
      if (u0 + 1 < u1) load(u0 + 1);
    }
    for (int u = u0, buf = 0; u < u1; ++u, buf ^= 1) {
      wait_lds();
      barrier();  // this unit is there, the last one is read
      if (u + 1 < u1) {
        next_page = page_of(2 * u + 4 + mine);
        expand(buf ^ 1);
        page = next_page;
        if (u + 2 < u1) load(u + 2);
      }
      const unsigned char *tk = lds + buf * BUF, *tv = tk + KB;
      const int f0 = flags[buf][0] | flags[buf][1], f1 = flags[buf][2] | flags[buf][3];
      const int there = __builtin_amdgcn_readfirstlane((f0 & 1) | (f1 & 1) << 1);
      huge |= __builtin_amdgcn_readfirstlane((f0 | f1) >> 1);
      const int tok = KEYS * u + 32 * part;
      if (!works || tok >= most_end) continue;
      if (parts == 1) products.template operator()<2>(tk, tv, 0, tok, there);
      else products.template operator()<1>(tk, tv, part, tok, (there >> part) & 1);
    }
  }

  l = __fadd_rn(l, __shfl_xor(l, 32));
  if (parts == 4) huge = __syncthreads_or(huge);  // each wave saw its own
  if (parts > 1) {  // the waves of the same rows, in the place of the tiles
    constexpr int WORDS = 16 * VT + 2;
    float* all = reinterpret_cast<float*>(lds);
    __syncthreads();
    if (part) {
      float* to = all + (wave - 1) * (WORDS * 64) + lane;
      to[0] = m;
      to[64] = l;
#pragma unroll
      for (int i = 0; i < 16 * VT; ++i) to[(2 + i) * 64] = o[i / 16][i % 16];
    }
    __syncthreads();
    if (part) return;
    for (int w = 1; w < parts; ++w) {
      const float* from = all + (wave + w - 1) * (WORDS * 64) + lane;
      const float m1 = from[0], now = fmaxf(m, m1);
      const float f0 = m == now ? 1.f : factor(m, now, a.scale2), f1 = m1 == now ? 1.f : factor(m1, now, a.scale2);
      m = now;
      l = __fmaf_rn(l, f0, __fmul_rn(from[64], f1));
#pragma unroll
      for (int i = 0; i < 16 * VT; ++i)
        o[i / 16][i % 16] = __fmaf_rn(o[i / 16][i % 16], f0, __fmul_rn(from[(2 + i) * 64], f1));
    }
  }
  if (huge) {
    // What was left out of the products is added to the outputs of the rows that see it, whatever its weight,
    // and to no other's: lane (n, hh) holds channels 32 d + 8 i + 4 hh .. of its row.
    for (int blk = 2 * u0; blk < min(2 * u1, blocks); ++blk) {
      const int page = page_of(blk), off0 = off_of(blk);
      if (page < 0) continue;
      const size_t r0 = Kv4At<DIM>::row(a.c, page, h, off0);
#pragma unroll 1
      for (int t = 0; t < 32; ++t) {
        if (32 * blk + t >= most_end) break;
#pragma unroll
        for (int d = 0; d < VT; ++d) {
          const uint32_t byte = a.c.vs[Kv4At<DIM>::vs(r0 + t, off0 + t, d)];
          if (byte < HUGE) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ch = 32 * d + 8 * i + 4 * hh;
            const uint32_t w = *reinterpret_cast<const uint16_t*>(
                a.c.v + Kv4At<DIM>::v(r0 + t, off0 + t, ch / (DIM / 16)) + ch % (DIM / 16) / 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = (float)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w >> (8 * (e / 2)), scale_bits(byte), 0)[e & 1];
              if (!(fabsf(y) < INFINITY) && 32 * blk + t < end) o[d][4 * i + e] = __fadd_rn(o[d][4 * i + e], y);
            }
          }
        }
      }
    }
  }
  if (row > last) return;
  const int t = fdiv(row, a.by_group.mul, a.by_group.shift), j = row - t * a.group;
  if (shares == 1) {
    const float r = __fdiv_rn(1.f, l == 0.f ? 1.f : l);
    T* to = (T*)a.out + ((int64_t)(at.start + t) * a.c.heads * a.group + h * a.group + j) * DIM + 4 * hh;
#pragma unroll
    for (int d = 0; d < VT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4(to + 32 * d + 8 * i, __fmul_rn(o[d][4 * i], r), __fmul_rn(o[d][4 * i + 1], r), __fmul_rn(o[d][4 * i + 2], r),
               __fmul_rn(o[d][4 * i + 3], r));
  } else {
    const int64_t slot = (((int64_t)at.start * a.group + row) * a.c.heads + h) * a.most + share;
    float* to = a.part + slot * DIM + 4 * hh;
#pragma unroll
    for (int d = 0; d < VT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(to + 32 * d + 8 * i) = make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
    if (hh == 0) *reinterpret_cast<float2*>(a.stats + slot * 2) = make_float2(m, l);
  }
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
  const int shares = shares_of(a, units_of(a, at, row / TILE * TILE));
  if (shares == 1) return;
  const int64_t slot = (((int64_t)at.start * a.group + row) * a.c.heads + h) * a.most;
  float m = -INFINITY, l = 0.f, y[C] = {};
  for (int s = lane; s < shares; s += 64) m = fmaxf(m, a.stats[(slot + s) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  for (int s = 0; s < shares; ++s) {
    const float2 st = *reinterpret_cast<const float2*>(a.stats + (slot + s) * 2);
    const float f = st.x == m ? 1.f : factor(st.x, m, a.scale2);
    l = __fmaf_rn(st.y, f, l);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float x = a.part[(slot + s) * DIM + C * lane + c];
      y[c] = fabsf(x) < INFINITY ? __fmaf_rn(x, f, y[c]) : __fadd_rn(y[c], x);  // also where f is 0
    }
  }
  const float r = __fdiv_rn(1.f, l == 0.f ? 1.f : l);
  T* to = (T*)a.out + id * DIM + C * lane;
#pragma unroll
  for (int c = 0; c < C; ++c) to[c] = (T)__fmul_rn(y[c], r);
}

// The tiles there can be, whatever the lengths are, the units of a share and the shares of a tile.
struct Cut {
  int64_t tiles;
  int upper, most;
};
static Cut cut_of(int64_t n, int64_t B, int64_t heads, int64_t group, int64_t max_len) {
  Cut c;
  const int64_t units = max_len > 0 ? (max_len + KEYS - 1) / KEYS : 1, begun = B + 2 < n ? B + 2 : n;
  c.tiles = n * group / TILE + begun;
  const int64_t want = (units * c.tiles * heads + 1023) / 1024;
  c.upper = (int)(want < 8 ? 8 : want);
  c.most = (int)((units + c.upper - 1) / c.upper);
  return c;
}

template <typename T, int DIM>
static int launch(const char* what, const Chunk& a, hipStream_t st) {
  kv4_chunk_kernel<T, DIM><<<(unsigned)((int64_t)a.tiles * a.most * a.c.heads), 256, 0, st>>>(a);
  if (a.most > 1) {
    const int64_t rows = (int64_t)a.n * a.c.heads * a.group;
    kv4_chunk_join_kernel<T, DIM><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(a);
  }
  return check_launch(what);
}

}  // namespace bq

using namespace bq;

size_t bq_kv4_attend_chunk_ws_bytes(int64_t n, int64_t B, int64_t q_heads, int64_t heads, int64_t dim, int64_t max_len) {
  if (n < 1 || B < 0 || heads < 1 || q_heads < heads || dim < 1 || max_len < 0) return 0;
  const Cut c = cut_of(n, B, heads, q_heads / heads, max_len);
  return c.most > 1 ? (size_t)n * q_heads * c.most * (dim + 2) * 4 : 0;
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
  const Cut cut = cut_of(n, B, cache->heads, group, max_len);
  if (cut.tiles * cut.most * cache->heads > 0x7fffffff || n * q_heads > 0x7fffffffll * 4)
    return set_error(BQ_ERR_ARG, "%s: size too large", what);
  if (!q || !cu || !out || (B && !lens)) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const int64_t size = type == KV4_F32 ? 4 : 2;
  if ((((uintptr_t)q | (uintptr_t)out) & 15) || (q_token | q_head) * size % 16)
    return set_error(BQ_ERR_ARG, "%s: rows that are not 16-byte aligned", what);
  const size_t need = bq_kv4_attend_chunk_ws_bytes(n, B, q_heads, cache->heads, cache->dim, max_len);
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
  a.tiles = (int)cut.tiles;
  a.upper = cut.upper;
  a.most = cut.most;
  a.by_group = fast_div((uint32_t)group);
  a.scale2 = scale * 1.4426950408889634f;
  a.out = out;
  a.part = (float*)ws;
  a.stats = a.part + (need ? (size_t)n * q_heads * cut.most * cache->dim : 0);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = cache->dim == 128;
  if (type == KV4_F32) return wide ? launch<float, 128>(what, a, st) : launch<float, 64>(what, a, st);
  if (type == KV4_BF16) return wide ? launch<__bf16, 128>(what, a, st) : launch<__bf16, 64>(what, a, st);
  return wide ? launch<_Float16, 128>(what, a, st) : launch<_Float16, 64>(what, a, st);
}
