// Shared by the adapters' kernels (lora.hip, lora_grad.hip): rows in tiles of one adapter each, 16-bit
// operands in fragments of 8 along a product's depth, 16 x 16 x 32 matrix instructions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "numerics.h"
#include "wave.h"

namespace rlu {
namespace lora {

typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int MAX_RANK = 128, MAX_ADAPTERS = 1024;

// A tile: rows order[start .. start + count) of one adapter; NONE: rows without one, BAD: ids past the last.
struct Tile {
  int adapter, start, count, pad;
};
constexpr int NONE = -1, BAD = -2;

struct Plan {
  const int* order;
  const Tile* tiles;
  const int* first;                        // [n + 3]: an adapter's first tile; NONE's, BAD's, and their number
  int n, rows, cap;                        // cap: tiles that there are at most
};

// D[i][j] += sum_k a[i][k] b[j][k]: lane l brings row / column l % 16 at k = 8 (l / 16) .. + 7, and holds column
// l % 16 at rows 4 (l / 16) .. + 3.
template <int DT>
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c) {
  if (DT == 0)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a),
                                                   __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ float to_f32(uint32_t b) {
  return DT == 0 ? bf16_to_f32((uint16_t)b) : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
template <int DT>
__device__ __forceinline__ uint32_t to_bits(float f) {
  return DT == 0 ? f32_to_bf16(f) : __builtin_bit_cast(uint16_t, (_Float16)f);
}

// n elements at p (8 or more: eight of them), zeros behind: p at any element's address.
__device__ __forceinline__ v4u load8(const uint16_t* p, int n) {
  v4u v = {};
  if (n >= 8) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) v[i / 2] |= (uint32_t)p[i] << i % 2 * 16;
  }
  return v;
}
__device__ __forceinline__ void store8(uint16_t* p, v4u v, int n) {
  if (n >= 8) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = (uint16_t)(v[i / 2] >> i % 2 * 16);
  }
}

// Four of 8 consecutive k of a lane's column, from a row-major [k][column] tile in LDS: lanes 4 r .. 4 r + 3 of
// each 16 point at four columns each of row r, lane i gets column i of rows 0 .. 3.
__device__ __forceinline__ v4s read_tr(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) v4s*)(__attribute__((address_space(3))) void*)p);
}

// A power of two that brings values of at most m in size to 2^10 .. 2^11: float16 has five bits of exponent.
__device__ __forceinline__ float scale_to(float m) {
  const int ex = (int)(__float_as_uint(m) >> 23);
  if (ex == 0 || ex >= 255) return 1.f;
  return __builtin_ldexpf(1.f, max(-100, min(100, 137 - ex)));
}

// f as the sum of two 16-bit values: 16 bits of it (22 in float16), for products with 8 (11)
template <int DT>
struct Split {
  uint32_t hi, lo;
  __device__ __forceinline__ explicit Split(float f) {
    hi = to_bits<DT>(f);
    const float r = f - to_f32<DT>(hi);
    lo = to_bits<DT>(r == r ? r : 0.f);                // (an infinity's rest)
  }
};

// A row of h or u, R floats, as fragments of both its parts: of the lane's 8 ranks of each 32. Returns by what sums
// with them are multiplied: float16's were brought into its range by a power of two.
template <int DT, int KS>
__device__ __forceinline__ float split_row(const float* row, int R, int g, v4u (&hi)[KS], v4u (&lo)[KS]) {
  float h[KS][8], m = 0.f;
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = 32 * k + 8 * g + e;
      h[k][e] = r < R ? row[r] : 0.f;
      m = fmaxf(m, fabsf(h[k][e]));
    }
  float by = 1.f;
  if (DT != 0) {
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    by = scale_to(m);
  }
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const Split<DT> p(h[k][e] * by), q(h[k][e + 1] * by);
      hi[k][e / 2] = p.hi | q.hi << 16;
      lo[k][e / 2] = p.lo | q.lo << 16;
    }
  return 1.f / by;
}

static inline bool sizes_ok(int dtype, int rows, int n, int size, int cap, int K, int N, int R) {
  return (dtype == 0 || dtype == 2) && rows >= 0 && n >= 1 && n <= MAX_ADAPTERS &&
         (size == 16 || size == 64) && K >= 1 && N >= 1 && K <= 1 << 24 && N <= 1 << 24 && R >= 1 &&
         R <= MAX_RANK && cap == (int)(rows / size + (rows < n + 2 ? rows : n + 2));
}

}  // namespace lora
}  // namespace rlu
