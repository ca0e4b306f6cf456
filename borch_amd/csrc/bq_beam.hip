// A beam search's selection: of each request's W beams and V tokens the W best continuations.
//
// A candidate's score is scores[b][w] + (x[b w][v] - lse), lse = m + log sum_v exp(x - m) over the beam's
// logits x with their maximum m. Beams are compared with one another in 64 bits: two candidates whose scores
// differ by less than f32 shows would else come out in an order that the sum's rounding decides. So the sum
// and its exponentials are taken in 64 bits too, and everything else about a beam's own tokens goes by the logits
// as they are: within a beam their order is that of the scores.
//
// Two launches. The first reads the logits once: a workgroup takes a part of a beam's tokens, and each of its
// waves keeps the W best of what it reads, a candidate a lane in order (value and token as one 64-bit number,
// so that equals go to the lower token). Which logits are looked at alone is known from maxima: the W-th largest of a
// wave's 64 lanes' maxima is reached by W logits at least, so that less than the largest such bar of the four waves
// is never among the W best of the part, and only the 16 bytes whose maximum reaches it are read again. The
// exponentials need no maximum: f64 holds e^x for every logit within +-600, and parts with others are summed again
// against their maximum. The second launch joins a request's parts and beams.
//
// Bound by the exponentials, 10 operations in f64 and as many in 32 bits a logit, beside the reading: 64 requests of
// 8 beams and 128000 tokens in bf16 (131 MB) take 55 us for the first launch (the vector units busy for two thirds of
// it) and 9 for the second. 4 beams of 32000 in f32: 6 us each, latency.
#include <math.h>

#include "bq_common.h"

namespace bq {

constexpr int MOST_BEAMS = 64, PART_WAVES = 4;
constexpr int PIECES = 16, PART_BYTES = PIECES * PART_WAVES * 64 * 16;  // 16 bytes each of a lane; of a part

struct Beam {
  const void* x;
  int64_t pitch;  // elements from beam to beam
  const float* scores;
  const uint8_t* done;  // nullable
  int B, W, V, end, parts, per;  // per: tokens a part
  uint64_t* best;  // [B W][parts][W] candidates in order
  double2* sums;   // [B W][parts]: what the exponents are relative to, their sum (NaN where a logit is)
  float* out;
  int *parents, *tokens;
  uint8_t* ended;
};

// A logit and its token as one number: larger is better. -0 counts as 0; NaN does not come here.
__device__ __forceinline__ uint64_t rank_of(float x, int token) {
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.f));
  const uint32_t o = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return (uint64_t)o << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float logit_of(uint64_t r) {
  const uint32_t o = (uint32_t)(r >> 32);
  return __uint_as_float(o ^ (o & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int token_of(uint64_t r) { return (int)~(uint32_t)r; }

// The value of the lane before (wave_shr:1); the first lane's is not looked at.
__device__ __forceinline__ int lane_below(int v) { return __builtin_amdgcn_mov_dpp(v, 0x138, 0xF, 0xF, false); }

// Over the wave's lanes, in a fixed order: from the lanes 1, 2, 4 and 8 before in a row of 16, the row before's last,
// lane 31's. Lanes that have none before take `none`, or for the maximum their own.
template <int CONTROL, int ROWS>
__device__ __forceinline__ double from_lanes(double v, double none) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v), o = __builtin_bit_cast(uint64_t, none);
  const uint32_t lo = __builtin_amdgcn_update_dpp((int)o, (int)x, CONTROL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp((int)(o >> 32), (int)(x >> 32), CONTROL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double last_lane(double v) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)x, 63));
}
__device__ __forceinline__ double wave_sum(double v) {
  v += from_lanes<0x111, 0xF>(v, 0.0);
  v += from_lanes<0x112, 0xF>(v, 0.0);
  v += from_lanes<0x114, 0xF>(v, 0.0);
  v += from_lanes<0x118, 0xF>(v, 0.0);
  v += from_lanes<0x142, 0xA>(v, 0.0);
  v += from_lanes<0x143, 0xC>(v, 0.0);
  return last_lane(v);
}
__device__ __forceinline__ double wave_top(double v) {
  v = fmax(v, from_lanes<0x111, 0xF>(v, v));
  v = fmax(v, from_lanes<0x112, 0xF>(v, v));
  v = fmax(v, from_lanes<0x114, 0xF>(v, v));
  v = fmax(v, from_lanes<0x118, 0xF>(v, v));
  v = fmax(v, from_lanes<0x142, 0xA>(v, v));
  v = fmax(v, from_lanes<0x143, 0xC>(v, v));
  return last_lane(v);
}

// The best `W` so far, in order, lane i the i-th (0: none); `least` the W-th.
struct List {
  uint64_t mine, least;
  int W;
  __device__ __forceinline__ void clear(int w) { mine = 0, least = 0, W = w; }
  // every lane's candidate that is good enough, one after another
  __device__ __forceinline__ void add(uint64_t r) {
    const int lane = threadIdx.x & 63;
    uint64_t who = __ballot(r > least);
    while (who) {
      const int l = __builtin_ctzll(who);
      const uint64_t x = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(r >> 32), l) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)r, l);
      const uint64_t up = (uint64_t)(uint32_t)lane_below((int)(mine >> 32)) << 32 | (uint32_t)lane_below((int)mine);
      mine = mine > x ? mine : lane == 0 || up > x ? x : up;
      least = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), W - 1) << 32 |
              (uint32_t)__builtin_amdgcn_readlane((int)mine, W - 1);
      who &= who - 1;
      who &= __ballot(r > least);
    }
  }
};

// e^x in f64 for |x| <= 700: 2^(n / 32) from a table of n's low bits and n's others as its exponent, times a
// polynomial for 2^(f / 32), f within 1/2 of 0 (interpolated at Chebyshev's nodes; within 8e-14 of itself). NaN stays.
// The table's 32 entries are the 64 banks of LDS once each, so lanes read any of them without conflict.
__device__ __forceinline__ double exp_of(double x, const double* table) {
  constexpr double ROUND = 0x1.8p52, C = 0x1.71547652b82fep5;  // a sum with ROUND is a whole number in its low bits
  const double k = __builtin_fma(x, C, ROUND), f = __builtin_fma(x, C, -(k - ROUND));
  const int n = (int)__builtin_bit_cast(uint64_t, k);
  const uint64_t at = __builtin_bit_cast(uint64_t, table[n & 31]) + ((uint64_t)(uint32_t)((n >> 5) << 20) << 32);
  double p = __builtin_fma(f, 0x1.3b2b13640caa1p-27, 0x1.c6b167e0c48a8p-20);
  p = __builtin_fma(f, p, 0x1.ebfbdff8198e6p-13);
  p = __builtin_fma(f, p, 0x1.62e42fef6d05bp-6);
  p = __builtin_fma(f, p, 1.0);
  return p * __builtin_bit_cast(double, at);
}
constexpr float WITHIN = 600.f, LEAST = -700.f;  // parts whose maximum is within +-WITHIN; logits below LEAST add nothing

template <typename T>
__global__ __launch_bounds__(PART_WAVES * 64) void beam_part_kernel(Beam a) {
  constexpr int E = 16 / sizeof(T), U = 4;  // logits a load, loads on their way
  typedef T Vec __attribute__((ext_vector_type(E)));
  __shared__ uint64_t lists[PART_WAVES][MOST_BEAMS];
  __shared__ double sums[PART_WAVES];
  __shared__ float tops[PART_WAVES], bars[PART_WAVES], mosts[PIECES][PART_WAVES * 64];
  __shared__ double table[32];
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  if (a.done && a.done[row]) return;
  if (threadIdx.x < 32) table[threadIdx.x] = exp2(threadIdx.x / 32.0);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* x = (const T*)a.x + row * a.pitch;
  const int lo = min(part * a.per, a.V), hi = min(a.V, lo + a.per);
  // 16-byte pieces from the first aligned one on; what lies before and behind them is the first wave's
  const int head = min(hi - lo, (int)((E - ((uintptr_t)(x + lo) / sizeof(T)) % E) % E));
  const int pieces = (hi - lo - head) / E, tail = lo + head + pieces * E;
  float top = -INFINITY, bar = -INFINITY;  // bar: what a logit has to reach
  double sum[2] = {0.0, 0.0};
  List best;
  best.clear(a.W);
  auto add = [&](float v, int token) {
    const float y = v < LEAST ? LEAST : v;  // NaN stays
    sum[token & 1] += exp_of((double)y, table);
  };
  if (wave == 0) {
    const int i = lane < head ? lo + lane : lane >= 32 && tail + lane - 32 < hi ? tail + lane - 32 : -1;
    const float v = i >= 0 ? (float)x[i] : -INFINITY;
    if (i >= 0) add(v, i);
    top = fmaxf(top, v);
    best.add(i >= 0 && v == v ? rank_of(v, i) : 0);
  }
  // Each piece's maximum waits in LDS for the bar.
  const Vec* from = reinterpret_cast<const Vec*>(x + lo + head);
  float lane_most = -INFINITY;
  auto place = [&](int n) { return (n * PART_WAVES + wave) * 64 + lane; };  // this lane's n-th piece
  const int mine = pieces > wave * 64 ? (pieces - wave * 64 + PART_WAVES * 64 - 1) / (PART_WAVES * 64) : 0;
  for (int n0 = 0; n0 < mine; n0 += U) {
    Vec now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = __builtin_nontemporal_load(from + min(place(n0 + u), pieces - 1));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float most = -INFINITY;
      if (place(n0 + u) < pieces)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          add((float)now[u][e], e);
          most = fmaxf(most, (float)now[u][e]);
        }
      if (n0 + u < mine) mosts[n0 + u][threadIdx.x] = most;
      lane_most = fmaxf(lane_most, most);
    }
  }
  top = fmaxf(top, lane_most);
  for (int w = 0; w < a.W; ++w) {
    bar = wave_max(lane_most);
    const uint64_t who = __ballot(lane_most == bar);
    if (lane == __builtin_ctzll(who)) lane_most = -INFINITY;
  }
  if (lane == 0) bars[wave] = bar;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < PART_WAVES; ++w) bar = fmaxf(bar, bars[w]);
  for (int n = 0; n < mine; ++n) {
    const bool here = mosts[n][threadIdx.x] >= bar && place(n) < pieces;
    if (!__any(here)) continue;
    const Vec now = from[min(place(n), pieces - 1)];
    const int i = lo + head + place(n) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = (float)now[e];
      const bool may = here && v >= bar;
      if (__any(may)) best.add(may ? rank_of(v, i + e) : 0);
    }
  }
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  lists[wave][lane] = best.mine;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < PART_WAVES; ++w) top = fmaxf(top, tops[w]);
  double all = sum[0] + sum[1], base = 0.0;
  if (fabsf(top) > WITHIN) {  // sums against the maximum; of one that is not finite a NaN is kept, the rest is the join's
    base = (double)top;
    if (fabsf(top) < INFINITY) {
      all = 0.0;
      for (int i = lo + (int)threadIdx.x; i < hi; i += PART_WAVES * 64) all += exp((double)(float)x[i] - base);
    }
  }
  all = wave_sum(all);
  if (lane == 0) sums[wave] = all;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < PART_WAVES; ++w) best.add(lists[w][lane]);
  const size_t slot = (size_t)row * a.parts + part;
  if (lane < a.W) a.best[slot * a.W + lane] = best.mine;
  if (lane == 0) {
    double s = sums[0];
    for (int w = 1; w < PART_WAVES; ++w) s += sums[w];
    a.sums[slot] = make_double2(base, s);
  }
}

// One request: each beam's parts joined, then the beams. Candidates are in order of (score, beam, place in the
// beam's order), and a candidate's place among all is the number of those before it, beam by beam.
__global__ __launch_bounds__(1024) void beam_join_kernel(Beam a) {
  extern __shared__ unsigned char lds[];
  double* keys = reinterpret_cast<double*>(lds);             // [W][W]
  int* toks = reinterpret_cast<int*>(keys + a.W * a.W);      // [W][W]
  int* counts = toks + a.W * a.W;                            // [W]: a beam's candidates
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = a.W, most = min(W, a.V);
  for (int w = wave; w < W; w += blockDim.x >> 6) {
    const int row = b * W + w;
    const double score = (double)a.scores[row];
    double key = -INFINITY;
    int token = -1;
    if (a.done && a.done[row]) {
      key = score != score ? -INFINITY : score;
      token = lane == 0 ? a.end : -1;
    } else {
      List best;
      best.clear(W);
      const uint64_t* from = a.best + (size_t)row * a.parts * W;
      const int all = a.parts * W;
      uint64_t next = from[min(lane, all - 1)];  // on its way beside the sums
      double top = -INFINITY, sum = 0.0;
      bool nan = false;
      for (int p0 = 0; p0 < a.parts; p0 += 64) {
        const int p = p0 + lane;
        double2 s = make_double2(-INFINITY, 0.0);
        if (p < a.parts) s = a.sums[(size_t)row * a.parts + p];
        nan |= s.y != s.y;
        const double now = fmax(wave_top(s.x), top);
        const double add = wave_sum(s.x > -INFINITY ? s.y * exp(s.x - now) : 0.0);
        sum = (top > -INFINITY ? sum * exp(top - now) : 0.0) + add;
        top = now;
      }
      for (int i = lane; i - lane < all; i += 64) {
        const uint64_t now = next;
        next = from[min(i + 64, all - 1)];
        best.add(i < all ? now : 0);
      }
      const bool dead = __any(nan) || !(top > -INFINITY && top < INFINITY) || !(fabs(score) < INFINITY);
      if (dead) {
        token = lane;  // nothing tells its tokens apart
      } else {
        token = token_of(best.mine);
        key = score + ((double)logit_of(best.mine) - (top + log(sum)));
        if (key != key) key = -INFINITY;
      }
      if (lane >= most) token = -1;
    }
    if (lane < W) {
      keys[w * W + lane] = key;
      toks[w * W + lane] = token;
    }
    const uint64_t real = __ballot(lane < W && token >= 0);
    if (lane == 0) counts[w] = __builtin_popcountll(real);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < W * W; i += blockDim.x) {
    const int own = i / W, nth = i - own * W;
    if (nth >= counts[own]) continue;
    const double key = keys[i];
    int place = nth;
    for (int w = 0; w < W && place < W; ++w) {
      if (w == own) continue;
      int lo = 0, hi = counts[w];  // how many of w's come before
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const double k = keys[w * W + mid];
        if (k > key || (k == key && w < own)) lo = mid + 1;
        else hi = mid;
      }
      place += lo;
    }
    if (place < W) {
      const int row = b * W + own, to = b * W + place;
      a.out[to] = (float)key;
      a.parents[to] = row;
      a.tokens[to] = toks[i];
      if (a.ended) a.ended[to] = (a.done && a.done[row]) || toks[i] == a.end;
    }
  }
}

// The parts of a beam: enough workgroups for all CUs at once (8 a CU; twice as many or half measure within 2 %, four
// times as many 10 % more), of at least 2048 tokens each (1024: 5 beams of 7 requests, 50001 tokens 18.8 us for 16.9),
// and as few as a part has room for (16 logits less than it has, for a row that starts anywhere).
static int64_t parts_of(int type, int64_t rows, int64_t V) {
  const int64_t want = (2048 + rows - 1) / rows, most = (V + 2047) / 2048, room = PART_BYTES / (type == 0 ? 4 : 2) - 16;
  const int64_t least = (V + room - 1) / room, parts = want < most ? want : most;
  return parts < least ? least : parts;
}

}  // namespace bq

using namespace bq;

size_t bq_beam_select_ws_bytes(int type, int64_t B, int64_t W, int64_t V) {
  if (B < 1 || W < 1 || W > MOST_BEAMS || V < 1) return 0;
  return (size_t)(B * W * parts_of(type, B * W, V)) * (16 + 8 * W);
}

int bq_beam_select(const void* logits, int type, int64_t B, int64_t W, int64_t V, int64_t pitch, const float* scores,
                   const uint8_t* done, int64_t end, float* out, int32_t* parents, int32_t* tokens, uint8_t* ended,
                   void* ws, size_t ws_bytes, bq_stream_t stream) {
  const char* what = "bq_beam_select";
  if (type < 0 || type > 2) return set_error(BQ_ERR_ARG, "%s: type %d", what, type);
  if (B < 0 || W < 1 || V < 1) return set_error(BQ_ERR_ARG, "%s: bad sizes", what);
  if (W > MOST_BEAMS) return set_error(BQ_ERR_UNSUPPORTED, "%s: %lld beams (%d at most)", what, (long long)W, MOST_BEAMS);
  if (V > 0x7fffffff - 8192 || B > 0x7fffff) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  if (done && (end < 0 || end > 0x7fffffff)) return set_error(BQ_ERR_ARG, "%s: end token %lld", what, (long long)end);
  if (B == 0) return BQ_OK;
  if (parts_of(type, B * W, V) > 0x7fffffff / (B * W)) return set_error(BQ_ERR_ARG, "%s: size too large", what);
  if (!logits || !scores || !out || !parents || !tokens) return set_error(BQ_ERR_ARG, "%s: null pointer", what);
  const size_t need = bq_beam_select_ws_bytes(type, B, W, V);
  if (!ws || ws_bytes < need || ((uintptr_t)ws & 15))
    return set_error(BQ_ERR_ARG, "%s: a workspace of %zu bytes, given %zu", what, need, ws ? ws_bytes : 0);
  Beam a;
  a.x = logits;
  a.pitch = pitch;
  a.scores = scores;
  a.done = done;
  a.B = (int)B;
  a.W = (int)W;
  a.V = (int)V;
  a.end = end < 0 || end > 0x7fffffff ? -1 : (int)end;
  a.parts = (int)parts_of(type, B * W, V);
  a.per = (int)((V + a.parts - 1) / a.parts);
  a.sums = (double2*)ws;
  a.best = (uint64_t*)(a.sums + B * W * a.parts);
  a.out = out;
  a.parents = parents;
  a.tokens = tokens;
  a.ended = ended;
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)(B * W * a.parts);
  if (type == 0) beam_part_kernel<float><<<grid, PART_WAVES * 64, 0, st>>>(a);
  else if (type == 1) beam_part_kernel<__bf16><<<grid, PART_WAVES * 64, 0, st>>>(a);
  else beam_part_kernel<_Float16><<<grid, PART_WAVES * 64, 0, st>>>(a);
  beam_join_kernel<<<(unsigned)B, 64 * (W < 16 ? (int)W : 16), (size_t)W * W * 12 + W * 4, st>>>(a);
  return check_launch(what);
}
