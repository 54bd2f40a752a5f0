// The dense fp8 block-scaled GEMM for many rows: y[M, n] bf16 = A[M, K] W[n, K]^T, A e4m3 row-major
// with a float32 scale per row and 128 columns, W e4m3 in fragment order with one per 128 x 128
// block.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemm_common.h"
#include "numerics.h"
#include "rlu.h"
#include "wave.h"

namespace rlu {
namespace dense {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int GROUP = 8;               // row tiles walked together
constexpr int SC = 8;                  // steps of row scales staged at a time

__device__ __forceinline__ v16f mfma32(v8i a, v8i b, v16f c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 127, 0, 127);
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

// Barrier behind which every wave's loads to LDS so far have arrived (the fence of a barrier alone
// does not wait for them).
__device__ __forceinline__ void staged_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0f70);                  // vmcnt(0)
  __syncthreads();
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
  static constexpr int LDS = 2 * (X + W + S);
};

template <class C>
__global__ __launch_bounds__(C::NW * WAVE, 2) void dense_k(const uint8_t* __restrict__ qx,
                                                           const float* __restrict__ xs,
                                                           const uint8_t* __restrict__ wq,
                                                           const float* __restrict__ ws,
                                                           uint16_t* __restrict__ y,
                                                           long long ldy, int M, int n, int K) {
  extern __shared__ __align__(16) uint8_t lds[];
  uint8_t* lx = lds;                                  // [2][BM rows][8 chunks of 16 B, swizzled]
  uint8_t* lw = lds + 2 * C::X;                       // [2][BN / 16 strips][2][64 lanes][16 B]
  uint8_t* ls = lw + 2 * C::W;                        // [2][BM / 8][8 rows][SC, swizzled] floats
  const int lane = lane_id();
  const int w = uniform((int)threadIdx.x / WAVE);
  const int nkg = K / 128;
  const int tm = (M + C::BM - 1) / C::BM;
  // workgroups go round the 8 XCDs: each XCD takes a run of tiles, in groups of GROUP row tiles
  // walked along the columns, so that the tiles it works on at a time share rows and weights
  const int tiles = (int)gridDim.x, tn = tiles / tm;
  const int xcd = (int)blockIdx.x & 7, per = tiles / 8, more = tiles % 8;
  const int id = xcd * per + min(xcd, more) + (int)blockIdx.x / 8;
  const int grp = id / (GROUP * tn), gm = min(GROUP, tm - grp * GROUP), at = id - grp * GROUP * tn;
  const int m0 = (grp * GROUP + at % gm) * C::BM, n0 = at / gm * C::BN;
  const int strips = (n + 127) / 128 * 8;
  const int rows = min(C::BM, M - m0), cols = min(C::BN, strips * 16 - n0);
  const uint8_t* gx = qx + (size_t)m0 * K;
  const uint8_t* gw = wq + (size_t)n0 * K;
  const float* gs = xs + (size_t)m0 * nkg;
  // past the last step the buffers have no bytes: such a load touches no memory
  auto buf = [&](const void* p, int bytes, bool live) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, live ? bytes : 0, BUF_WORD3);
  };
  // a wave's loads take 8 rows, 8 lanes a row; a row's chunk q lies at q ^ (row & 7)
  const int vx = lane / 8 * K + ((lane ^ (lane / 8)) & 7) * 16;
  const int vw = lane * 16;
  auto stage = [&](int b, int kb) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t bx = buf(gx, rows * K, kb < nkg);
    const __amdgpu_buffer_rsrc_t bw = buf(gw, cols * K, kb < nkg);
#pragma unroll
    for (int i = 0; i < C::XI; ++i)
      to_lds16(bx, vx, (w * C::XI + i) * 8 * K + kb * 128,
               lx + b * C::X + (w * C::XI + i) * 1024);
#pragma unroll
    for (int i = 0; i < C::WI; ++i) {
      const int s = w * C::WI + i;                     // half a strip's step
      to_lds16(bw, vw, (s / 2) * nkg * 2048 + kb * 2048 + (s & 1) * 1024,
               lw + b * C::W + s * 1024);
    }
  };
  // a wave's i-th load of the row scales of steps kb .. kb + SC
  auto scales = [&](int b, int kb, int i) __attribute__((always_inline)) {
    const int e = w * C::XI + i;
    const int j = (lane ^ (lane / 8 + 2 * e)) & 7;
    to_lds4(buf(gs, rows * nkg * 4, kb < nkg), (lane / 8 * nkg + j) * 4, (e * 8 * nkg + kb) * 4,
            ls + b * C::S + e * 256);
  };

  const int wm = w % C::GM, wn = w / C::GM;
  const int r = lane & 31, g = lane >> 5;
  const int nb = uniform((n0 + wn * 32 * C::WN) / 128);
  const float* wsr = ws + (size_t)min(nb, strips / 8 - 1) * nkg;
  float acc[C::WM][C::WN][16];
#pragma unroll
  for (int t = 0; t < C::WM; ++t)
#pragma unroll
    for (int u = 0; u < C::WN; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][u][i] = 0.f;
  const uint8_t* pw = lw + wn * C::WN * 4096 + (r / 16) * 2048 + (32 * g + (r & 15)) * 16;
  const uint8_t* px[4];                                // chunk 4 h + 2 g + i at [2 h + i]
#pragma unroll
  for (int c = 0; c < 4; ++c)
    px[c] = lx + wm * C::WM * 4096 + r * 128 + (((4 * (c / 2) + 2 * g + c % 2) ^ r) & 7) * 16;
  const uint8_t* ps = ls + wm * C::WM * 1024 + (r / 8) * 256 + (r & 7) * 32;

  v8i a[C::WN][2], x[2][2];
  v16f d[2];
  float f[2], sx[2], wsc;
  auto read_w = [&](int b, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* p = pw + b * C::W + u * 4096 + h * 1024;
      a[u][h] = pack8(*reinterpret_cast<const v4u*>(p), *reinterpret_cast<const v4u*>(p + 256));
    }
  };
  auto read_x = [&](int b, int kb, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      x[t & 1][h] = pack8(*reinterpret_cast<const v4u*>(px[2 * h] + b * C::X + t * 4096),
                          *reinterpret_cast<const v4u*>(px[2 * h + 1] + b * C::X + t * 4096));
    sx[t & 1] = *reinterpret_cast<const float*>(ps + t * 1024 + (kb / SC & 1) * C::S +
                                                ((kb ^ (r + 2 * (r / 8))) & 7) * 4);
  };
  // tile i = t WN + u of a step: its products, and the scaling of the tile before it
  auto tile = [&](int i) __attribute__((always_inline)) {
    const int t = i / C::WN, u = i % C::WN;
    v16f z;
#pragma unroll
    for (int k = 0; k < 16; ++k) z[k] = 0.f;
    d[i & 1] = mfma32(a[u][0], x[t & 1][0], z);
    d[i & 1] = mfma32(a[u][1], x[t & 1][1], d[i & 1]);
    constexpr int T = C::WM * C::WN;
    const int p = (i + T - 1) % T;
#pragma unroll
    for (int k = 0; k < 16; ++k)
      acc[p / C::WN][p % C::WN][k] =
          fmaf(d[(i + 1) & 1][k], f[p / C::WN & 1], acc[p / C::WN][p % C::WN][k]);
    if (u == 0) f[t & 1] = wsc * sx[t & 1];
  };
  static_assert(C::XI <= SC, "a step stages at most one part of the scales");
  auto step = [&](const int b, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < C::WM; ++t) {
      if (t == C::WM - 1) {
        staged_barrier();
        stage(b, kb + 2);
        // of the next SC steps' scales the part that this step stages
        scales((kb / SC + 1) & 1, (kb / SC + 1) * SC, kb % SC * C::XI / SC);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int u = 0; u < C::WN; ++u) {
        tile(t * C::WN + u);
        if (t + 1 == C::WM) read_w(b ^ 1, u);
        if (u == 0) {
          if (t + 1 < C::WM) read_x(b, kb, t + 1);
          else read_x(b ^ 1, kb + 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    wsc = wsr[min(kb + 1, nkg - 1)];
  };
  static_assert(C::WM % 2 == 0, "x alternates over a step's row tiles");
#pragma unroll
  for (int i = 0; i < C::XI; ++i) scales(0, 0, i);
  stage(0, 0);
  stage(1, 1);
  staged_barrier();
  wsc = wsr[0];
#pragma unroll
  for (int u = 0; u < C::WN; ++u) read_w(0, u);
  read_x(0, 0, 0);
#pragma unroll
  for (int k = 0; k < 16; ++k) d[1][k] = 0.f;
  f[0] = f[1] = 0.f;
  for (int kb = 0; kb < nkg; ++kb) step(kb & 1, kb);
#pragma unroll
  for (int k = 0; k < 16; ++k)
    acc[C::WM - 1][C::WN - 1][k] =
        fmaf(d[(C::WM * C::WN - 1) & 1][k], f[(C::WM - 1) & 1], acc[C::WM - 1][C::WN - 1][k]);
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
        const float* v = &acc[t][u][4 * i];
        const uint2 p = {f32_to_bf16(v[0]) | (uint32_t)f32_to_bf16(v[1]) << 16,
                         f32_to_bf16(v[2]) | (uint32_t)f32_to_bf16(v[3]) << 16};
        *reinterpret_cast<uint2*>(le + (t * 32 + r) * (CH * 16) +
                                  (((u * 4 + i) ^ r) & (CH - 1)) * 16 + g * 8) = p;
      }
  wave_lds_sync();
  const int row0 = m0 + wm * C::WM * 32, col0 = n0 + wn * C::WN * 32;
  if (ldy % 8 == 0 && (uintptr_t)y % 16 == 0) {
#pragma unroll
    for (int i = 0; i < C::WM * 32 * CH / WAVE; ++i) {
      const int row = i * (WAVE / CH) + lane / CH, q = lane % CH;
      const v4u p = *reinterpret_cast<const v4u*>(le + row * (CH * 16) + ((q ^ row) & (CH - 1)) * 16);
      uint16_t* o = y + (row0 + row) * ldy + col0 + q * 8;
      if (row0 + row < M) {
        if (col0 + q * 8 + 8 <= n) {
          *reinterpret_cast<v4u*>(o) = p;
        } else {
          for (int k = 0; col0 + q * 8 + k < n; ++k) o[k] = (uint16_t)(p[k / 2] >> (k % 2 * 16));
        }
      }
    }
  } else {
    constexpr int RW = WAVE / (CH * 8) > 0 ? WAVE / (CH * 8) : 1;   // rows a pass
    for (int i = 0; i < C::WM * 32 / RW; ++i)
#pragma unroll
      for (int c = lane % (CH * 8); c < CH * 8; c += WAVE) {
        const int row = i * RW + lane / (CH * 8);
        const uint16_t v = *reinterpret_cast<const uint16_t*>(
            le + row * (CH * 16) + (((c / 8) ^ row) & (CH - 1)) * 16 + c % 8 * 2);
        if (row0 + row < M && col0 + c < n) y[(row0 + row) * ldy + col0 + c] = v;
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

}  // namespace dense
}  // namespace rlu

extern "C" int rlu_gemm_fp8blk_dense(const void* qx, const float* xs, const void* w,
                                     const float* ws, void* y, long long ldy, int M, int n,
                                     int K, hipStream_t stream) {
  using namespace rlu;
  if (M < 0 || n < 1 || K < 1 || ldy < n) return -1;
  if (K % 128) return -2;
  if (M == 0) return 0;
  if (!qx || !xs || !w || !ws || !y) return -1;
  const auto* q = (const uint8_t*)qx;
  const auto* p = (const uint8_t*)w;
  return dense::launch<dense::Cfg<4, 2, 2, 4>>(stream, q, xs, p, ws, (uint16_t*)y, ldy, M, n, K);
}
