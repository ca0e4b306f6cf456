// What the attention kernels over the 4-bit cache share: values as exact sums of bf16 pieces, codes to
// bf16, rows stored in the callers' types.
#pragma once

#include <math.h>

#include "bq_bf16x3.h"
#include "bq_kv4.h"

namespace bq {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));

template <typename T>
constexpr int Q_PIECES = __is_same(T, float) ? 3 : __is_same(T, _Float16) ? 2 : 1;
template <typename T>
constexpr int P_PIECES = __is_same(T, float) ? 3 : 2;

template <int P>
struct Pieces {
  v8bf p[P];
};

template <int P>
__device__ __forceinline__ Pieces<P> pieces_of(const float x[8]) {
  Pieces<P> r;
  uint32_t w[P][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      w[k][i] = bf2(a, b);
      if (k + 1 < P) {
        a = __fsub_rn(a, __uint_as_float(w[k][i] << 16));
        b = __fsub_rn(b, __uint_as_float(w[k][i] & 0xffff0000u));
      }
    }
  }
#pragma unroll
  for (int k = 0; k < P; ++k) r.p[k] = __builtin_bit_cast(v8bf, make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]));
  return r;
}

template <typename T>
__device__ __forceinline__ void load8f(const T* p, float x[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if constexpr (__is_same(T, __bf16)) {
    const v8bf a = *reinterpret_cast<const v8bf*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
  } else {
    const v8h a = *reinterpret_cast<const v8h*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
  }
}

// The pieces of queries. An infinity stays one (inf - inf left NaN in the second piece), and what f32
// holds above bf16's largest value does not become one. By whole waves.
template <int P>
__device__ __forceinline__ Pieces<P> split_q(const float x[8]) {
  Pieces<P> r = pieces_of<P>(x);
  if constexpr (P > 1) {
    constexpr float MOST = 0x1.fep127f;
    float peak = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) peak = fmaxf(peak, fabsf(x[i]));
    if (__any(peak > (P == 2 ? 65504.f : MOST))) {
      float y[8], z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool finite = fabsf(x[i]) < INFINITY;
        y[i] = finite ? fminf(fmaxf(x[i], -MOST), MOST) : x[i];
        y[i] = (float)(__bf16)y[i];
        z[i] = finite ? __fsub_rn(x[i], y[i]) : 0.f;
      }
      r.p[0] = pieces_of<1>(y).p[0];
      const Pieces<P - 1> rest = pieces_of<P - 1>(z);
#pragma unroll
      for (int k = 1; k < P; ++k) r.p[k] = rest.p[k - 1];
    }
  }
  return r;
}

__device__ __forceinline__ float scale_bits(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes (one dword, low half byte first) times a scale, in bf16, exactly.
__device__ __forceinline__ v8bf codes8(uint32_t w, float scale) {
  const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1),
             c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  } else if constexpr (__is_same(T, __bf16)) {
    *reinterpret_cast<uint2*>(p) = make_uint2(bf2(a, b), bf2(c, d));
  } else {
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4h*>(p) = v4h{(_Float16)a, (_Float16)b, (_Float16)c, (_Float16)d};
  }
}

}  // namespace bq
