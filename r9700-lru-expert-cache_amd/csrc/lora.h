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
  const int* first;                        // [n + 5]: an adapter's first tile; NONE's, BAD's, their number; adapters
                                           // with rows, and the rows that have one
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

// Two of them in one word.
template <int DT>
__device__ __forceinline__ uint32_t to_bits2(float a, float b) {
  return DT == 0 ? f32x2_to_bf16(a, b) : to_bits<DT>(a) | to_bits<DT>(b) << 16;
}

// n elements at p (8 or more: eight of them), zeros behind: p at any element's address. ONCE: nobody asks
// for these again, so they need no place in the cache.
typedef v4u v4ua __attribute__((aligned(2)));
template <bool ONCE = false>
__device__ __forceinline__ v4u load8(const uint16_t* p, int n) {
  v4u v = {};
  if (n >= 8) {
    v = ONCE ? (v4u)__builtin_nontemporal_load((const v4ua*)p) : (v4u)*(const v4ua*)p;
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) v[i / 2] |= (uint32_t)p[i] << i % 2 * 16;
  }
  return v;
}
template <bool ONCE = false>
__device__ __forceinline__ void store8(uint16_t* p, v4u v, int n) {
  if (n >= 8) {
    if (ONCE) __builtin_nontemporal_store(v, (v4ua*)p);
    else *(v4ua*)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = (uint16_t)(v[i / 2] >> i % 2 * 16);
  }
}

typedef v4f v4fa __attribute__((aligned(4)));
__device__ __forceinline__ void load8(const float* p, int n, float (&h)[8]) {
  if (n >= 8) {
    const v4f a = *(const v4fa*)p, b = *(const v4fa*)(p + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < 4 ? a[i] : b[i - 4];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < n ? p[i] : 0.f;
  }
}

// Elements i .. i + 7 of a row of `all`, i a multiple of 8, in two steps: fetch asks for them, keep makes those past the
// row's end zeros, when they are there. WHOLE: all is a multiple of 8 too, so that eight are there or none: then both go
// without a branch, and a fetch ahead of its use waits for nothing (where its elements don't matter, keep is left out).
template <bool WHOLE, bool ONCE = false>
__device__ __forceinline__ v4u fetch(const uint16_t* p, int i, int all) {
  return WHOLE ? load8<ONCE>(p + (i < all ? i : 0), 8) : load8<ONCE>(p + i, all - i);
}
template <bool WHOLE>
__device__ __forceinline__ v4u keep(v4u v, int i, int all) {
  if (WHOLE)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i < all ? v[e] : 0u;
  return v;
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

// f as the sum of 16-bit values, the largest first, for products with 16-bit ones: all of its 24 bits in three of bf16; in
// two of float16 22, half a step of which is 2^-23 of f, no more than two additions of the float32 sums around it may lose.
// (bf16 in two parts, 16 bits, left 1.2e-4 between lora_1's outputs and what float32 rounds to, 9e-8 in three. The third one's cost, us:
// 8192 rows of [2560 -> 10240] in any order, R = 64 expand 81 -> 85, outer 95 -> 108, R = 128 121 -> 145 and 154 -> 175; R = 16
// 1 to 2%, dx with dA 25 -> 28)
template <int DT>
struct Split {
  static constexpr int N = DT == 0 ? 3 : 2;
  uint32_t part[N];
  __device__ __forceinline__ explicit Split(float f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      part[i] = DT == 0 ? f32_to_bf16_hw(f) : to_bits<DT>(f);
      f -= to_f32<DT>(part[i]);
      f = f == f ? f : 0.f;                            // (an infinity's rest)
    }
  }
};

// A lane's part of 16 rows from `row` on, 32 of their elements from `k` on, of a row-major tile in LDS.
template <int LD>
__device__ __forceinline__ v4u frag(const uint16_t* tile, int row, int k) {
  const int lane = lane_id();
  return *(const v4u*)&tile[(row + lane % 16) * LD + k + 8 * (lane / 16)];
}
// The same of 16 columns from `c` on, 32 rows from `k` on.
template <int LD>
__device__ __forceinline__ v4u frag_tr(const uint16_t* tile, int k, int c) {
  const int lane = lane_id(), col = lane % 16;
  const uint16_t* p = &tile[(k + 8 * (lane / 16) + col / 4) * LD + c + col % 4 * 4];
  return __builtin_bit_cast(v4u, __builtin_shufflevector(read_tr(p), read_tr(p + 4 * LD), 0, 1, 2, 3, 4, 5, 6, 7));
}

// A tile's rows of h or u, R floats each, as their 16-bit parts in LDS, and by what sums with them are multiplied:
// float16's are brought into its range by a power of two a row.
template <int DT, int MT, int KS>
struct Rows {
  static constexpr int T = 16 * MT, LD = 32 * KS + 8, PARTS = Split<DT>::N;
  uint16_t part[PARTS][T][LD];
  float back[T];
};
// rows: where the row-th of `count` rows lies
template <int DT, int MT, int KS, int NT, class At>
__device__ __forceinline__ void stage(Rows<DT, MT, KS>& s, int count, int R, At rows) {
  constexpr int PER = NT / (16 * MT), N = (4 * KS + PER - 1) / PER;    // threads a row, chunks of 8 a thread
  const int row = (int)threadIdx.x / PER, q = (int)threadIdx.x % PER;
  const float* from = rows(min(row, count - 1));
  float v[N][8], m = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = k * PER + q;
    load8(from + 8 * c, c < 4 * KS && row < count ? R - 8 * c : 0, v[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[k][e]));
  }
  float by = 1.f;
  if (DT != 0) {
#pragma unroll
    for (int d = 1; d < PER; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    by = scale_to(m);
    if (q == 0) s.back[row] = 1.f / by;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = k * PER + q;
    if (c >= 4 * KS) continue;
    v4u p[Split<DT>::N];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const Split<DT> a(v[k][e] * by), b(v[k][e + 1] * by);
#pragma unroll
      for (int i = 0; i < Split<DT>::N; ++i) p[i][e / 2] = a.part[i] | b.part[i] << 16;
    }
#pragma unroll
    for (int i = 0; i < Split<DT>::N; ++i) *(v4u*)&s.part[i][row][8 * c] = p[i];
  }
}

// ---- out = y + h W^T (TR: h W, with W [R][cols]), without y where there is none ------------------------------------
// A workgroup a tile (or 16 MT of its rows) and a strip of columns, a wave 64 columns at a time: W's part of them as it
// lies in memory through LDS into registers, then 16 rows after the other. Sums leave the matrix unit with a lane's
// neighbour another row; through LDS they come in rows of 128 bytes, as y and out are read and written.
// Bound by y read and out written: 8192 x 10240, R = 64 77 - 80 us, 4.4 TB/s; 1024 x 151936, R = 16 117 - 120 us, 5.3 TB/s; 160 x
// 151936, R = 16, 32 adapters 53 - 54 us, 4.7 TB/s with their 156 MB. The matrix unit is busy for 17% of the cycles, LDS for
// 28%. R over 64: 143 us at 8192 x 10240, as W's and h's 122 KB of LDS leave a CU one workgroup. At 8192 x 10240, R = 64, with h
// in two parts: 150 us with h's eight values loaded one by one, 112 by 16 bytes, 97 with W through LDS, 77 with the sums through
// it, 74 with y and out past the cache.
struct Out {
  const uint16_t *w, *y;
  long long ldy;
  uint16_t* out;
  long long ldo;
  int cols, R;
};
constexpr int EXPAND_NT = 256;
template <int DT, int MT, int KS, bool TR, int NT = EXPAND_NT>
struct ExpandLds {
  static constexpr int LD = TR ? 72 : 32 * KS + 8, SUM_LD = 68;
  static constexpr int W = TR ? 32 * KS * LD : 64 * LD, SUMS = 2 * 16 * SUM_LD;
  Rows<DT, MT, KS> h;
  alignas(16) uint16_t wave[NT / WAVE][W > SUMS ? W : SUMS];           // W, then a block's sums
};

// Rows without an adapter: out = y.
template <int NT = EXPAND_NT>
__device__ __forceinline__ void copy(const Out& f, const Plan& p, const Tile& t, int n0, int n1) {
  if (f.y == f.out && f.ldy == f.ldo) return;
  for (int r = (int)threadIdx.x / 32; r < t.count; r += NT / 32) {
    const size_t row = p.order[t.start + r];
    for (int c = n0 + (int)threadIdx.x % 32 * 8; c < n1; c += 256)
      store8(f.out + row * f.ldo + c, load8(f.y + row * f.ldy + c, f.cols - c), f.cols - c);
  }
}

// lds.h is staged; its barrier is to come.
template <int DT, int MT, int KS, bool WHOLE, bool TR, bool ADD, int NT = EXPAND_NT>
__device__ __forceinline__ void expand(const Out& f, const Plan& p, const Tile& t, int n0, int n1,
                                       ExpandLds<DT, MT, KS, TR, NT>& lds) {
  typedef ExpandLds<DT, MT, KS, TR, NT> L;
  constexpr int STEP = NT;                 // columns: 64 a wave
  constexpr bool ONCE = ADD && NT == EXPAND_NT;        // (what is more than a few tiles' outputs passes the cache by)
  const int lane = lane_id(), w = uniform((int)threadIdx.x / WAVE), col = lane % 16, g = lane / 16;
  const int r8 = lane / 8, c8 = lane % 8 * 8;
  size_t row[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int s = 0; s < 2; ++s) row[i][s] = p.order[t.start + min(16 * i + 8 * s + r8, t.count - 1)];
  const uint16_t* weights = f.w + (size_t)max(t.adapter, 0) * f.cols * f.R;       // (BAD: h is NaN)
  const int ranks = t.adapter == NONE ? 0 : f.R;       // (0 times whatever adapter 0 holds may be NaN)
  uint16_t* mine = lds.wave[w];
  float* sums = (float*)mine;
  __syncthreads();
  for (int c0 = n0 + w * 64; c0 < n1; c0 += STEP) {
    v4u wr[4 * KS], yv[MT][2];
#pragma unroll
    for (int i = 0; i < 4 * KS; ++i) {
      const int q = i * WAVE + lane;
      if (TR) wr[i] = fetch<WHOLE>(weights + (size_t)min(q / 8, f.R - 1) * f.cols, c0 + c8, q / 8 < ranks ? f.cols : 0);
      else wr[i] = fetch<WHOLE>(weights + (size_t)min(c0 + q / (4 * KS), f.cols - 1) * f.R, q % (4 * KS) * 8, ranks);
    }
    if (ADD)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) yv[i][s] = fetch<WHOLE, ONCE>(f.y + row[i][s] * f.ldy, c0 + c8, f.cols);
#pragma unroll
    for (int i = 0; i < 4 * KS; ++i) {
      const int q = i * WAVE + lane;
      if (TR) *(v4u*)&mine[q / 8 * L::LD + c8] = keep<WHOLE>(wr[i], c0 + c8, q / 8 < ranks ? f.cols : 0);
      else *(v4u*)&mine[q / (4 * KS) * L::LD + q % (4 * KS) * 8] = keep<WHOLE>(wr[i], q % (4 * KS) * 8, ranks);
    }
    wave_lds_sync();
    v4u wf[4][KS];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < KS; ++k)
        wf[j][k] = TR ? frag_tr<L::LD>(mine, 32 * k, 16 * j) : frag<L::LD>(mine, 16 * j, 32 * k);
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      v4f acc[4] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int p = Split<DT>::N - 1; p >= 0; --p) {
          const v4u h = frag<32 * KS + 8>(lds.h.part[p][0], 16 * i, 32 * k);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = mfma<DT>(wf[j][k], h, acc[j]);
        }
      if (DT != 0) {
        const float back = lds.h.back[16 * i + col];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] *= back;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) *(v4f*)&sums[col * L::SUM_LD + 16 * j + 4 * g] = acc[j];
      wave_lds_sync();
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const v4f a = *(const v4f*)&sums[(8 * s + r8) * L::SUM_LD + c8];
        const v4f b = *(const v4f*)&sums[(8 * s + r8) * L::SUM_LD + c8 + 4];
        v4u o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = e < 2 ? a[2 * e] : b[2 * e - 4], y = e < 2 ? a[2 * e + 1] : b[2 * e - 3];
          if (ADD) {
            x += to_f32<DT>(yv[i][s][e] & 0xffffu);
            y += to_f32<DT>(yv[i][s][e] >> 16);
          }
          o[e] = to_bits2<DT>(x, y);
        }
        if (16 * i + 8 * s + r8 < t.count) store8<ONCE>(f.out + row[i][s] * f.ldo + c0 + c8, o, f.cols - c0 - c8);
      }
      wave_lds_sync();
    }
  }
}

// Columns of a workgroup: as many as 32768 outputs have, where that leaves two workgroups for every CU (each of them
// stages h again).
static inline int strip_of(long long tiles, int rows, int N) {
  int strip = 32768 / rows;
  while (strip > 256 && tiles * ((N + strip - 1) / strip) < 512) strip /= 2;
  return strip;
}

static inline bool sizes_ok(int dtype, int rows, int n, int size, int cap, int K, int N, int R) {
  return (dtype == 0 || dtype == 2) && rows >= 0 && rows <= 1 << 24 && n >= 1 && n <= MAX_ADAPTERS &&
         (size == 16 || size == 64) && K >= 1 && N >= 1 && K <= 1 << 24 && N <= 1 << 24 && R >= 1 &&
         R <= MAX_RANK && cap == (int)(rows / size + (rows < n + 2 ? rows : n + 2));
}

}  // namespace lora
}  // namespace rlu
