// The dense fp8 block-scaled GEMM for any number of rows: y[M, n] bf16 = A[M, K] W[n, K]^T, A e4m3
// row-major with a float32 scale per row and 128 columns, W e4m3 in fragment order with one per 128 x 128
// block:  y = sum over 128-deep steps k of xs[m, k] ws[n / 128, k] (A_k W_k^T)[m, n].
//
// Bound, with many rows: the matrix cores at the clock that the chip's power leaves them (1.75 - 1.8 GHz
// under this load), with a multiply-add of every product by its scale beside them and both operands
// through LDS. A bare loop of 32 x 32 x 64 MFMAs and their scaling runs at 3.3 PFLOP/s on two waves a
// SIMD, this kernel at 2.1 (8192 x 10240 x 2560 in 194 - 207 us; 2048 x 151936 x 2560 in 757 - 838, 2.0), the
// library's fp8 product of 8192^3, which scales nothing, at 2.65. With few rows: the weights' read, and
// below about 256 tiles the length of one (1.0 us a step of the largest alone).
//
//   * A tile is 256 x 256, 192 x 256 or 128 x 128; a wave has 32 x 32 tiles, up to 4 x 2 of them (64 columns
//     of 128 rows), all in registers. W is the MFMA's first operand: a lane then holds one row of y, and its
//     scale is one register. 32 x 32 x 64 and not 16 x 16 x 128: half the operand reads and instructions,
//     3.3 against 2.8 PFLOP/s in the bare loop. Without scales the instruction is 8 bytes shorter.
//   * A step's rows and weights come straight to LDS, two steps of them. Rows are stored by chunks of 16
//     bytes, chunk q of row r at q ^ (r / 2 & 7): no bank conflicts (r & 7 instead: 13% of the cycles).
//     The weights are already in fragment order. Three steps of LDS with a smaller tile: 1.4 PFLOP/s where
//     two with this one had 1.7; one more step of weights alone (192 x 256) changed nothing.
//   * The scaling of a 32 x 32 tile is issued behind the products of the next one, so that the vector unit
//     works under the matrix cores; operand reads go out two at a time between products, ahead of need, and
//     a step's loads one or two a tile: in one go after the barrier they kept every wave from its products
//     (225 -> 209 us at 8192 x 10240). The second half of a row tile's depth is held once and not twice, and
//     what a lane can recompute it does: with 8 registers more the loop spills, and a spill's reload waits
//     for all loads to LDS (1.3 PFLOP/s).
//   * The weights' scales are scalar loads, a step ahead and just before the barrier: their wait is one for
//     every LDS read in flight. The rows' go to LDS, 8 steps at a time.
//   * Measured against one another and slower: the two waves of a SIMD taking turns at products and LDS reads
//     (1.56 PFLOP/s), products and scaling in the compiler's own order (1.7).
//   * Output through LDS to 16-byte pieces, stored without a place in the L2 (2048 x
//     151936: 895 against 915 us).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemm_common.h"
#include "head.h"
#include "numerics.h"
#include "rlu.h"
#include "wave.h"

namespace rlu {
namespace dense {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int GROUP = 4;               // row tiles walked together
constexpr int SC = 8;                  // steps of row scales staged at a time

__device__ __forceinline__ v16f mfma32(v8i a, v8i b, v16f c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void* lds_ptr;
constexpr int BUF_WORD3 = 0x00020000;  // raw buffer descriptor word 3 on gfx9 (no format)

// 16 / 4 bytes from a buffer at voff (a lane's) + soff to LDS at dst + lane * 16 / 4 (dst uniform)
__device__ __forceinline__ void to_lds16(__amdgpu_buffer_rsrc_t b, int voff, int soff, void* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_ptr)dst, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void to_lds4(__amdgpu_buffer_rsrc_t b, int voff, int soff, void* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_ptr)dst, 4, voff, soff, 0, 0);
}

// Barrier behind which every wave's loads to LDS so far have arrived (the fence of a barrier alone does not
// wait for them).
__device__ __forceinline__ void staged_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0f70);                  // vmcnt(0)
  lds_barrier();
}

// A wave has WM x WN tiles of 32 rows x 32 columns, a workgroup GM x GN waves.
template <int WM_, int WN_, int GM_, int GN_>
struct Cfg {
  static constexpr int WM = WM_, WN = WN_, GM = GM_, GN = GN_;
  static constexpr int BM = 32 * WM * GM, BN = 32 * WN * GN, NW = GM * GN;
  static constexpr int X = BM * 128, W = BN * 128;              // bytes of a step
  static constexpr int S = BM * SC * 4;                         // bytes of SC steps' row scales
  static constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW;      // loads of a wave
  static_assert(XI * 8 * NW == BM && WI * 8 * NW == BN, "the waves share the loads evenly");
  static constexpr int SLOTS = WM % 2 ? WM : 2;                 // row tiles' operands held
  static constexpr int LDS = 2 * (X + W) + 2 * S;
};

// A wave's loads of step kb, one at a time: j counts XI of rows (8 each, 8 lanes a row), then WI of half strips
// of weights; row_scales is one of XI parts, of the SC steps from kb on. ld(e, at, bytes, voffset, soffset): piece
// e of the step, through a buffer of `bytes` from byte `at` of the tile's operand on. Only the vector offset is
// sure to count in a buffer's range check, so what decides whether there is such a row lies in the base and the
// vector offset, the scalar one moves within a row or a strip alone, and past the last step or strip the buffer
// is empty: such a load touches no memory. (Masks, and one buffer for all rows of a wave and one for its strips: a
// condition is made a branch, with which the loop spills, and a buffer each took 20 scalar instructions more a
// step: 768 x 2560 x 2048 14.5 us, this 13.9.)
// A row's chunk q lies at q ^ (row / 2 & 7), so that 16 rows' reads of one chunk meet all 64 banks (by row & 7,
// row r and r + 8 shared theirs).
template <class C>
__host__ __device__ __forceinline__ int row_lane(int w, int lane, int K, int j) {
  return (8 * j + lane / 8) * K + ((lane ^ (8 * (w * C::XI + j) + lane / 8) / 2) & 7) * 16;
}
template <class C, class LD>
__host__ __device__ __forceinline__ void row_or_weights(int w, int lane, const int (&vx)[C::XI],
                                                        int rows, int cols, int K, int kb, int j,
                                                        const LD& ld) {
  const int live = (kb - K / 128) >> 31;
  if (j < C::XI) {
    const int r0 = 8 * w * C::XI;
    ld(w * C::XI + j, r0 * K, max(0, rows - r0) * K & live, vx[j], kb * 128);
  } else {
    const int e = w * C::WI + j - C::XI, c0 = w * C::WI / 2 * 16;
    static_assert(128 % (C::WI * 8) == 0 && C::WI % 2 == 0, "a wave's strips are there together");
    ld(e, c0 * K, (c0 < cols ? C::WI * 8 * K : 0) & live, lane * 16 + (j - C::XI) / 2 * 16 * K,
       kb * 2048 + (e & 1) * 1024);
  }
}
template <class C, class LD>
__host__ __device__ __forceinline__ void row_scales(int w, int lane, int rows, int K, int kb, int i,
                                                    const LD& ld) {
  const int nkg = K / 128, e = w * C::XI + i, j = (lane ^ (lane / 8 + 2 * e)) & 7;
  const int r0 = 8 * w * C::XI;
  // (SC steps on from kb: past a row's last they are the next one's, and not used)
  ld(e, (r0 * nkg + kb) * 4, max(0, (rows - r0) * nkg - kb) * 4 & (kb - nkg) >> 31,
     ((8 * i + lane / 8) * nkg + j) * 4, 0);
}

template <class C>
__global__ __launch_bounds__(C::NW * WAVE, 2) void dense_k(const uint8_t* __restrict__ qx,
                                                           const float* __restrict__ xs,
                                                           const uint8_t* __restrict__ wq,
                                                           const float* __restrict__ ws,
                                                           uint16_t* __restrict__ y,
                                                           long long ldy, int M, int n, int K) {
  extern __shared__ __align__(16) uint8_t lds[];
  uint8_t* lx = lds;                       // [2][BM rows][8 chunks of 16 B, swizzled]
  uint8_t* lw = lds + 2 * C::X;            // [2][BN / 16 strips][2][64 lanes][16 B]
  uint8_t* ls = lw + 2 * C::W;             // [2][BM / 8][8 rows][SC floats, swizzled]
  const int lane = lane_id();
  const int w = uniform((int)threadIdx.x / WAVE);
  const int nkg = K / 128;
  const int tm = (M + C::BM - 1) / C::BM;
  // workgroups go round the 8 XCDs: each XCD takes a run of tiles, in groups of GROUP row tiles
  // walked along the columns, so that the tiles it works on at a time share rows and weights
  const int tiles = (int)gridDim.x, tn = tiles / tm;
  const int xcd = (int)blockIdx.x & 7, per = tiles / 8, more = tiles % 8;
  const int id = xcd * per + min(xcd, more) + (int)blockIdx.x / 8;
  const int band = id / (GROUP * tn), gm = min(GROUP, tm - band * GROUP), at = id - band * GROUP * tn;
  const int m0 = (band * GROUP + at % gm) * C::BM, n0 = at / gm * C::BN;
  const int strips = (n + 127) / 128 * 8;
  const int rows = min(C::BM, M - m0), cols = min(C::BN, strips * 16 - n0);
  const uint8_t* gx = qx + (size_t)m0 * K;
  const uint8_t* gw = wq + (size_t)n0 * K;
  const float* gs = xs + (size_t)m0 * nkg;
  auto buf = [&](const void* p, int at, int bytes) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const uint8_t*)p + (unsigned)at), 0, bytes,
                                             BUF_WORD3);
  };
  int vx[C::XI];
#pragma unroll
  for (int j = 0; j < C::XI; ++j) vx[j] = row_lane<C>(w, lane, K, j);
  // A step's loads: XI + WI, and a part of the row scales that the steps from the next multiple of SC on read
  // (the last part again once all are on their way).
  constexpr int PIECES = C::XI + C::WI + 1;
  auto scales = [&](int b, int kb, int i) __attribute__((always_inline)) {
    row_scales<C>(w, lane, rows, K, kb, i,
                  [&](int e, int at, int bytes, int voff, int soff) __attribute__((always_inline)) {
      to_lds4(buf(gs, at, bytes), voff, soff, ls + b * C::S + e * 256);
    });
  };
  auto piece = [&](int b, int kb, int j) __attribute__((always_inline)) {
    if (j < C::XI + C::WI) {
      const bool x = j < C::XI;
      row_or_weights<C>(w, lane, vx, rows, cols, K, kb, j,
                        [&](int e, int at, int bytes, int voff, int soff)
                            __attribute__((always_inline)) {
        to_lds16(buf(x ? gx : gw, at, bytes), voff, soff,
                 (x ? lx + b * C::X : lw + b * C::W) + e * 1024);
      });
    } else {
      const int s = kb - 2, c = (s >> 3) + 1;
      static_assert(SC == 8, "s >> 3");
      scales(c & 1, c * SC, min(s & 7, C::XI - 1));
    }
  };

  const int wm = w % C::GM, wn = w / C::GM;
  const int r = lane & 31, g = lane >> 5;
  const int nb = uniform((n0 + wn * 32 * C::WN) / 128);
  const float* wsr = ws + (size_t)min(nb, strips / 8 - 1) * nkg;
  v16f acc[C::WM][C::WN];
#pragma unroll
  for (int t = 0; t < C::WM; ++t)
#pragma unroll
    for (int u = 0; u < C::WN; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][u][i] = 0.f;
  const uint8_t* pw = lw + wn * C::WN * 4096 + (r / 16) * 2048 + (32 * g + (r & 15)) * 16;
  // chunk 4 h + 2 g + i of a row lies at (that of h = i = 0) ^ (4 h + i)
  const int ox = wm * C::WM * 4096 + r * 128 + ((2 * g ^ (r / 2)) & 7) * 16;
  const uint8_t* ps = ls + wm * C::WM * 1024 + (r / 8) * 256 + (r & 7) * 32;

  v8i a[C::WN][2], x0[C::SLOTS], x1;
  v16f d[2];
  float f[C::SLOTS], sx, wsc = wsr[0], wsn;
  auto read_w = [&](int b, int u, int h) __attribute__((always_inline)) {
    const uint8_t* p = pw + b * C::W + u * 4096 + h * 1024;
    a[u][h] = pack8(*reinterpret_cast<const v4u*>(p), *reinterpret_cast<const v4u*>(p + 256));
  };
  auto read_x = [&](int b, int t, int h) __attribute__((always_inline)) {
    const uint8_t* p = lx + b * C::X + t * 4096;
    (h ? x1 : x0[t % C::SLOTS]) =
        pack8(*reinterpret_cast<const v4u*>(p + (ox ^ (64 * h))),
              *reinterpret_cast<const v4u*>(p + (ox ^ (64 * h + 16))));
  };
  auto read_s = [&](int kb, int t) __attribute__((always_inline)) {
    sx = *reinterpret_cast<const float*>(ps + t * 1024 + (kb / SC & 1) * C::S +
                                         ((kb ^ (r + 2 * (r / 8))) & 7) * 4);
  };
  constexpr int T = C::WM * C::WN;
  // (a part staged behind step s's barrier has arrived at that of step s + 1, before the reads for s + 2)
  static_assert(C::XI <= SC - 1, "all parts are there when the next SC steps begin");
  // Behind a step's barrier its buffer is free for step kb + 2, whose loads go out a few in each of the
  // WINDOW tiles from there on: in one go they kept every wave from its products.
  constexpr int WINDOW = T - 3 > C::WN ? T - 3 : C::WN, PER = (PIECES + WINDOW - 1) / WINDOW;
  // the step whose operands are in buffer b; the steps before and after it have buffer bn
  auto step = [&](int b, int bn, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int t = i / C::WN, u = i % C::WN;          // a tile, and in p the one before it
      const int p = (i + T - 1) % T;
      const bool last = t + 1 == C::WM;
      if (last && u == 0) {
        staged_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
      // the next row tile's operands are read between the products, a few at a time
      v16f z;
#pragma unroll
      for (int k = 0; k < 16; ++k) z[k] = 0.f;
      // the depth's second half goes first in every other tile: x1 is free again one product sooner
      const int h0 = u & 1, h1 = 1 - h0;
      d[i & 1] = mfma32(a[u][h0], h0 ? x1 : x0[t % C::SLOTS], z);
      // (the loop's first product waits for every read before it: none of the new ones)
      if (i == 0) __builtin_amdgcn_sched_barrier(0);
      if (last) read_w(bn, u, h0);
      if (u == 0) read_x(last ? bn : b, last ? 0 : t + 1, 0);
      else read_x(last ? bn : b, last ? 0 : t + 1, 1);
      // just ahead of the barrier, which waits for it: a scalar load's wait is one for all LDS reads
      if (i == T - C::WN - 1) wsn = wsr[min(kb + 1, nkg - 1)];
      __builtin_amdgcn_sched_barrier(0);
      d[i & 1] = mfma32(a[u][h1], h1 ? x1 : x0[t % C::SLOTS], d[i & 1]);
      if (last) read_w(bn, u, h1);
      if (u == 0) {
        f[t % C::SLOTS] = wsc * sx;
        read_s(last ? kb + 1 : kb, last ? 0 : t + 1);
      }
      const int q = (i + C::WN) % T;                   // tiles since the barrier
#pragma unroll
      for (int j = q * PER; j < (q + 1) * PER && j < PIECES; ++j)
        piece(last ? b : bn, last ? kb + 2 : kb + 1, j);
      __builtin_amdgcn_sched_barrier(0x3f4);
      acc[p / C::WN][p % C::WN] = __builtin_elementwise_fma(
          d[(i + 1) & 1], (v16f)(f[p / C::WN % C::SLOTS]), acc[p / C::WN][p % C::WN]);
      __builtin_amdgcn_sched_barrier(0);
    }
    wsc = wsn;
  };
  static_assert(C::WM > 1 && C::WN == 2, "a row tile's operands are read while the one before is used");
#pragma unroll
  for (int i = 0; i < C::XI; ++i) scales(0, 0, i);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < PIECES - 1; ++j)
      if (i == 0 || j < C::WN * PER) piece(i, i, j);
  staged_barrier();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int u = 0; u < C::WN; ++u) read_w(0, u, h);
    read_x(0, 0, h);
  }
  read_s(0, 0);
#pragma unroll
  for (int k = 0; k < 16; ++k) d[1][k] = 0.f;
  f[(C::WM - 1) % C::SLOTS] = 0.f;
  for (int kb = 0, b = 0; kb < nkg; ++kb) {
    const int bn = b ^ 1;
    step(b, bn, kb);
    b = bn;
  }
  acc[C::WM - 1][C::WN - 1] = __builtin_elementwise_fma(
      d[(T - 1) & 1], (v16f)(f[(C::WM - 1) % C::SLOTS]), acc[C::WM - 1][C::WN - 1]);
  // lane: row r of a tile, columns 8 (i / 4) + 4 g + i % 4. Through LDS (each wave its own part) to
  // whole 16-byte pieces of a row; a row's piece q lies at q ^ (row % CH)
  constexpr int CH = 4 * C::WN;
  staged_barrier();                                    // (the empty loads past the end, too)
  uint8_t* le = lds + w * (C::WM * 32 * CH * 16);
#pragma unroll
  for (int t = 0; t < C::WM; ++t)
#pragma unroll
    for (int u = 0; u < C::WN; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v16f& v = acc[t][u];
        const uint2 p = {f32_to_bf16(v[4 * i]) | (uint32_t)f32_to_bf16(v[4 * i + 1]) << 16,
                         f32_to_bf16(v[4 * i + 2]) | (uint32_t)f32_to_bf16(v[4 * i + 3]) << 16};
        *reinterpret_cast<uint2*>(le + (t * 32 + r) * (CH * 16) +
                                  (((u * 4 + i) ^ r) & (CH - 1)) * 16 + g * 8) = p;
      }
  wave_lds_sync();
  const long long row0 = m0 + wm * C::WM * 32;
  const int col0 = n0 + wn * C::WN * 32;
  if (ldy % 8 == 0 && (uintptr_t)y % 16 == 0) {
#pragma unroll
    for (int i = 0; i < C::WM * 32 * CH / WAVE; ++i) {
      const int row = i * (WAVE / CH) + lane / CH, q = lane % CH;
      const v4u p = *reinterpret_cast<const v4u*>(le + row * (CH * 16) + ((q ^ row) & (CH - 1)) * 16);
      uint16_t* o = y + (row0 + row) * ldy + col0 + q * 8;
      if (row0 + row < M) {
        if (col0 + q * 8 + 8 <= n) {
          __builtin_nontemporal_store(p, reinterpret_cast<v4u*>(o));
        } else {
          for (int k = 0; col0 + q * 8 + k < n; ++k) o[k] = (uint16_t)(p[k / 2] >> (k % 2 * 16));
        }
      }
    }
  } else {
    // rows at odd addresses: a lane a column, so that a row's part is still one piece
    static_assert(CH * 8 == WAVE, "a column a lane");
    const bool in = col0 + lane < n;
    uint16_t* o = y + row0 * ldy + col0 + lane;
#pragma unroll
    for (int i = 0; i < C::WM * 32; i += 16) {
      uint16_t v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k)
        v[k] = *reinterpret_cast<const uint16_t*>(
            le + (i + k) * (CH * 16) + (((lane / 8) ^ (i + k)) & (CH - 1)) * 16 + lane % 8 * 2);
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (in && row0 + i + k < M) o[(i + k) * ldy] = v[k];
    }
  }
}

template <class C>
static int launch(hipStream_t st, const uint8_t* qx, const float* xs, const uint8_t* wq,
                  const float* ws, uint16_t* y, long long ldy, int M, int n, int K) {
  const long long tiles =
      (long long)((M + C::BM - 1) / C::BM) * ((n + C::BN - 1) / C::BN);
  if (tiles > INT32_MAX) return -1;
  hipLaunchKernelGGL((dense_k<C>), dim3((unsigned)tiles), dim3(C::NW * WAVE), C::LDS, st, qx, xs,
                     wq, ws, y, ldy, M, n, K);
  return (int)hipGetLastError();
}

// The loads of a tile of `rows` x `cols` (weights' rows, by whole 16) of K by which dense_k would touch memory
// that it has no use for (all past the last step, row or strip; of the scales those behind the last row's), with
// only the vector offset in a buffer's range check, and those of its operands that a check of the vector and the
// scalar offset would drop.
template <class C>
static unsigned long long loads_wrong(int rows, int cols, int K) {
  unsigned long long bad = 0;
  const int nkg = K / 128;
  for (int w = 0; w < C::NW; ++w)
    for (int lane = 0; lane < WAVE; ++lane) {
      // own: the byte to load, -1 for none
      auto count = [&](long long own, int at, int bytes, int voff, int soff, int n) {
        const long long to = (long long)at + voff + soff;
        if (own < 0 ? voff < bytes : to != own || (long long)voff + soff + n > bytes) ++bad;
      };
      int vx[C::XI];
      for (int j = 0; j < C::XI; ++j) vx[j] = row_lane<C>(w, lane, K, j);
      for (int kb = 0; kb < nkg + 2 + SC; ++kb) {
        const bool live = kb < nkg;
        for (int j = 0; j < C::XI + C::WI; ++j)
          row_or_weights<C>(w, lane, vx, rows, cols, K, kb, j,
                            [&](int e, int at, int bytes, int voff, int soff) {
            if (j < C::XI) {                           // row r's chunk q lies at q ^ (r / 2 & 7)
              const int r = 8 * e + lane / 8, q = (lane ^ r / 2) & 7;
              count(live && r < rows ? (long long)r * K + kb * 128 + q * 16 : -1, at, bytes, voff,
                    soff, 16);
            } else {                                   // half h of strip s
              const int s = e / 2, h = e % 2;
              count(live && 16 * s < cols ? (long long)(s * nkg + kb) * 2048 + h * 1024 + lane * 16
                                          : -1,
                    at, bytes, voff, soff, 16);
            }
          });
        for (int i = 0; i < C::XI && kb % SC == 0; ++i)
          row_scales<C>(w, lane, rows, K, kb, i, [&](int e, int at, int bytes, int voff, int soff) {
            // step kb + j of row r at j ^ (r + 2 (r / 8)) & 7
            const int r = 8 * e + lane / 8, j = (lane ^ (r + r / 8 * 2)) & 7;
            const long long to = ((long long)r * nkg + kb + j) * 4;
            count(live && to < (long long)rows * nkg * 4 ? to : -1, at, bytes, voff, soff, 4);
          });
      }
    }
  return bad;
}

typedef Cfg<4, 2, 2, 4> Big;           // 256 x 256, one workgroup a CU
typedef Cfg<3, 2, 2, 4> Mid;           // 192 x 256, one
typedef Cfg<2, 2, 2, 2> Small;       // 128 x 128, two

// tiles of a shape that the fullest CU gets
template <class C>
static long long per_cu(int M, int n) {
  const long long t = (long long)((M + C::BM - 1) / C::BM) * ((n + C::BN - 1) / C::BN);
  return (t + device_cus() - 1) / device_cus();
}

}  // namespace dense
}  // namespace rlu

extern "C" int rlu_gemm_fp8blk_dense(const void* qx, const float* xs, const void* w,
                                     const float* ws, void* y, long long ldy, int M, int n,
                                     int K, hipStream_t stream) {
  using namespace rlu;
  if (M < 0 || n < 1 || K < 1 || ldy < n || n > INT32_MAX - 256 || M > INT32_MAX - 256) return -1;
  if (K % 128 || K > (1 << 22)) return -2;
  if (M == 0) return 0;
  if (!qx || !xs || !w || !ws || !y) return -1;
  if (((uintptr_t)qx | (uintptr_t)w) % 16 || ((uintptr_t)xs | (uintptr_t)ws) % 4 || (uintptr_t)y % 2)
    return -4;
  const auto* q = (const uint8_t*)qx;
  const auto* p = (const uint8_t*)w;
  auto* o = (uint16_t*)y;
  // Which kernel: the least of these estimates in us, each of a round of the CUs (fixed part, a 128-deep
  // step's) as measured. Tiles, with every CU busy: Big 8 + 1.6, Mid 6.5 + 1.22, Small 4 + 0.55 alone
  // on its CU and 6 + 0.95 for two, and 2.5 more where rows do not start at 16 bytes. The head's kernel,
  // 64 rows x 64 columns and K split over its waves: 3.7 + 1.35 for a wave's steps.
  //   rows x n x K           head / Big / Mid / Small (us)
  //   256 x 2560 x 2560      10.5 / 28.5 / 24.9 / 15.2    1024 x 2560     24 / 29 / 25.6 / 16
  //   4096 x 2560 x 2560     - / 34 / 31 / 39             2048 x 10240    - / 69 / 64 / 70
  //   128 x 151936 x 2560    192 / 119 / 114 / 104        160 x 151936    270 / 126 / 117 / 141
  //   256 x 151936 x 2560    373 / 138 / 173 / 158        512 x 32000     118 / 36 / 50 / 43
  //   617 x 1543 x 768       8.4 / - / - / 10.8
  // Up to 64 rows the head's kernel reads the weights once, as it does for gemm_fp8_block.
  const int steps = K / 128, sk = head::sk_of(K);
  if (M <= 64 && sk) return head::rows(q, xs, p, ws, o, ldy, M, n, K, stream);
  const long long ns = dense::per_cu<dense::Small>(M, n);
  const double odd = ldy % 8 || (uintptr_t)y % 16 ? 2.5 : 0;
  const double big = dense::per_cu<dense::Big>(M, n) * (8 + odd + 1.6 * steps);
  const double mid = dense::per_cu<dense::Mid>(M, n) * (6.5 + odd + 1.22 * steps);
  const double small =
      ns / 2 * (6 + odd + 0.95 * steps) + ns % 2 * (4 + odd + 0.55 * steps);
  const double tile = small < mid ? (small < big ? small : big) : mid < big ? mid : big;
  if (sk && M <= 65535 * 64) {
    const long long items = (n + 127) / 128 * 2, wgs = (items * sk + 3) / 4 * ((M + 63) / 64);
    if ((double)((wgs + device_cus() - 1) / device_cus()) * (3.7 + 1.35 * (steps / sk)) < tile)
      return head::rows(q, xs, p, ws, o, ldy, M, n, K, stream);
  }
  if (tile == small)
    return dense::launch<dense::Small>(stream, q, xs, p, ws, o, ldy, M, n, K);
  if (tile == mid) return dense::launch<dense::Mid>(stream, q, xs, p, ws, o, ldy, M, n, K);
  return dense::launch<dense::Big>(stream, q, xs, p, ws, o, ldy, M, n, K);
}

// Host only: counts into *bad, over the tiles of each shape that M x n ends in, the loads that would touch
// memory they should not with only the vector offset in the buffers' range check, and the operands' that
// would be dropped with both offsets in it. Returns -1 (bad sizes or NULL), -2 (K % 128 or too large).
extern "C" int rlu_selftest_dense_loads(int M, int n, int K, unsigned long long* bad) {
  using namespace rlu::dense;
  if (M < 1 || n < 1 || K < 1 || n > INT32_MAX - 256 || !bad) return -1;
  if (K % 128 || K > (1 << 22)) return -2;
  auto last = [&](auto c) {
    typedef decltype(c) C;
    const int rows = (M - 1) % C::BM + 1, cols = ((n + 127) / 128 * 128 - 1) % C::BN + 1;
    return loads_wrong<C>(rows, cols, K);
  };
  *bad = last(Big()) + last(Mid()) + last(Small());
  return 0;
}
