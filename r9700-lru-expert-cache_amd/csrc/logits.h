// Rows of logits in vectors of 16 bytes, shared by the kernels that read them (log probabilities, losses):
// their elements, their maximum, and sums over a wave in a fixed order.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave.h"

namespace rlu {
namespace lp {

typedef unsigned int v4u __attribute__((ext_vector_type(4)));

constexpr float L2E = 1.44269504f;

template <int DT>
struct Elem;                               // 0 bf16, 1 f32, 2 f16: elements of 16 bytes, and the i-th
template <>
struct Elem<0> {
  static constexpr int N = 8, SIZE = 2;
  static constexpr uint32_t NINF = 0xff80;
  static __device__ __forceinline__ float get(v4u v, int i) {
    const uint32_t u = v[i / 2];
    return __uint_as_float(i % 2 ? u & 0xffff0000u : u << 16);
  }
};
template <>
struct Elem<1> {
  static constexpr int N = 4, SIZE = 4;
  static constexpr uint32_t NINF = 0xff800000u;
  static __device__ __forceinline__ float get(v4u v, int i) { return __uint_as_float(v[i]); }
};
template <>
struct Elem<2> {
  static constexpr int N = 8, SIZE = 2;
  static constexpr uint32_t NINF = 0xfc00;
  static __device__ __forceinline__ float get(v4u v, int i) {
    const uint32_t u = v[i / 2];
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(i % 2 ? u >> 16 : u));
  }
};

// A thread's maximum over its vectors.
template <int DT, int CV>
struct Max {
  static __device__ __forceinline__ float of(const v4u (&raw)[CV]) {
    float m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < CV; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = fmaxf(m, __uint_as_float(raw[k][i]));
    return m;
  }
};
// Of 16-bit floats without unpacking them: as signed integers they are in order from 0 up, and where none
// is up there the least unsigned one is the largest. (A NaN may or may not come out.)
typedef short v2s __attribute__((ext_vector_type(2)));
typedef unsigned short v2us __attribute__((ext_vector_type(2)));
template <int DT, int CV>
__device__ __forceinline__ float packed_max(const v4u (&raw)[CV]) {
  v2s hi = __builtin_bit_cast(v2s, (uint32_t)raw[0][0]);
#pragma unroll
  for (int k = 0; k < CV; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      hi = __builtin_elementwise_max(hi, __builtin_bit_cast(v2s, (uint32_t)raw[k][i]));
  const short h = hi[0] > hi[1] ? hi[0] : hi[1];
  v4u v = {};
  v[0] = (uint16_t)h;
  if (__ballot(h < 0)) {
    v2us lo = __builtin_bit_cast(v2us, (uint32_t)raw[0][0]);
#pragma unroll
    for (int k = 0; k < CV; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        lo = __builtin_elementwise_min(lo, __builtin_bit_cast(v2us, (uint32_t)raw[k][i]));
    if (h < 0) v[0] = lo[0] < lo[1] ? lo[0] : lo[1];
  }
  return Elem<DT>::get(v, 0);
}
template <int CV>
struct Max<0, CV> {
  static __device__ __forceinline__ float of(const v4u (&raw)[CV]) { return packed_max<0>(raw); }
};
template <int CV>
struct Max<2, CV> {
  static __device__ __forceinline__ float of(const v4u (&raw)[CV]) { return packed_max<2>(raw); }
};

template <int DT>
__device__ __forceinline__ float load_one(const uint8_t* row, long long i) {
  const uint8_t* p = row + i * Elem<DT>::SIZE;
  v4u v = {};
  v[0] = Elem<DT>::SIZE == 4 ? *reinterpret_cast<const uint32_t*>(p)
                             : *reinterpret_cast<const uint16_t*>(p);
  return Elem<DT>::get(v, 0);
}

template <int CTRL>
__device__ __forceinline__ float dppf(float v) {
  return __int_as_float(dpp<CTRL>(__float_as_int(v), __float_as_int(v)));
}
__device__ __forceinline__ float lane_f(float v, int l) {
  return __int_as_float(readlane(__float_as_int(v), l));
}
__device__ __forceinline__ float wave_max(float v) {   // wave-uniform; NaN only if all are
  v = fmaxf(v, dppf<0xb1>(v));
  v = fmaxf(v, dppf<0x4e>(v));
  v = fmaxf(v, dppf<0x141>(v));
  v = fmaxf(v, dppf<0x140>(v));
  return fmaxf(fmaxf(lane_f(v, 0), lane_f(v, 16)), fmaxf(lane_f(v, 32), lane_f(v, 48)));
}
__device__ __forceinline__ float wave_add(float v) {   // wave-uniform, in a fixed order
  v += dppf<0xb1>(v);
  v += dppf<0x4e>(v);
  v += dppf<0x141>(v);
  v += dppf<0x140>(v);
  return (lane_f(v, 0) + lane_f(v, 16)) + (lane_f(v, 32) + lane_f(v, 48));
}

__device__ __forceinline__ long long token_of(const void* tokens, int wide, int row) {
  return wide ? ((const long long*)tokens)[row] : ((const int*)tokens)[row];
}

}  // namespace lp
}  // namespace rlu
