// Low-rank adapters of many requests beside a shared projection:
//   out[m] = y[m] + h[m] B_a^T, h[m] = s_a x[m] A_a^T, a = the row's adapter, A [n, R, K], B [n, N, R].
// Rows are put in order by adapter once for a batch, in tiles of 16 or 64 rows of one adapter, which the products of
// all its projections share.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lora.h"
#include "rlu.h"
#include "wave.h"

namespace rlu {
namespace lora {

// ---- rows by adapter: a stable counting sort in one workgroup ---------------------------------------------
// Each wave counts and later places a run of the rows, 64 at a time in order, so the order is the same on every run.
constexpr int PLAN_NT = 1024, PLAN_NW = PLAN_NT / WAVE;

__device__ __forceinline__ int key_of(const void* ids, int wide, int row, int n) {
  const long long id = wide ? ((const long long*)ids)[row] : (long long)((const int*)ids)[row];
  return id < 0 ? n : id >= n ? n + 1 : (int)id;
}

__global__ __launch_bounds__(PLAN_NT) void plan_k(const void* __restrict__ ids, int wide, int rows,
                                                  int n, int size, int* __restrict__ order,
                                                  Tile* __restrict__ tiles, int* __restrict__ first) {
  extern __shared__ int count[];           // [PLAN_NW][n + 2], then starts [n + 2], then first tiles [n + 3]
  const int groups = n + 2, tid = (int)threadIdx.x, lane = lane_id(), w = uniform(tid / WAVE);
  int* start = count + PLAN_NW * groups;
  int* tile0 = start + groups;
  for (int i = tid; i < PLAN_NW * groups; i += PLAN_NT) count[i] = 0;
  __syncthreads();
  const int run = (rows + PLAN_NT - 1) / PLAN_NT * WAVE, r0 = min(w * run, rows), r1 = min(r0 + run, rows);
  for (int r = r0 + lane; r < r1; r += WAVE) atomicAdd(&count[w * groups + key_of(ids, wide, r, n)], 1);
  __syncthreads();
  // per group: where each wave's rows begin within it
  for (int g = tid; g < groups; g += PLAN_NT) {
    int sum = 0;
    for (int i = 0; i < PLAN_NW; ++i) {
      const int c = count[i * groups + g];
      count[i * groups + g] = sum;
      sum += c;
    }
    start[g] = sum;
  }
  __syncthreads();
  if (w == 0) {                            // totals to starts, rows and tiles
    int at = 0, tile = 0;
    for (int g0 = 0; g0 < groups; g0 += WAVE) {
      const int g = g0 + lane, c = g < groups ? start[g] : 0, t = (c + size - 1) / size;
      const int sc = wave_incl_scan(c), st = wave_incl_scan(t);
      if (g < groups) {
        start[g] = at + sc - c;
        tile0[g] = tile + st - t;
        first[g] = tile + st - t;
      }
      at += readlane(sc, WAVE - 1);
      tile += readlane(st, WAVE - 1);
    }
    if (lane == 0) {
      first[groups] = tile;
      tile0[groups] = tile;
    }
  }
  __syncthreads();
  for (int g = tid; g < groups; g += PLAN_NT) {
    const int end = g + 1 < groups ? start[g + 1] : rows, t0 = tile0[g], t1 = tile0[g + 1];
    for (int t = t0; t < t1; ++t) {
      const int s = start[g] + (t - t0) * size;
      tiles[t] = {g < n ? g : g == n ? NONE : BAD, s, min(size, end - s), 0};
    }
  }
  int bits = 1;
  while (1 << bits < groups) ++bits;
  for (int r = r0; r < r1; r += WAVE) {    // (uniform: a wave's lanes place one row each)
    const bool in = r + lane < r1;
    const int key = in ? key_of(ids, wide, r + lane, n) : 0;
    const uint64_t same = match_any(key, in, bits);
    const int before = mbcnt(same);
    int to = 0;
    if (in) to = start[key] + count[w * groups + key] + before;
    wave_lds_sync();
    if (in && before == 0) count[w * groups + key] += (int)__popcll(same);
    wave_lds_sync();
    if (in) order[to] = r + lane;
  }
}

// ---- h = s x A^T ------------------------------------------------------------------------------------------
// A workgroup a tile and 64 ranks: its waves take turns at the depth, and are summed through LDS.
struct Fwd {
  const uint16_t* x;
  long long ldx;
  const uint16_t *a, *b;
  const float* scale;
  Plan p;
  int K, N, R;
  float* hidden;
  const uint16_t* y;
  long long ldy;
  uint16_t* out;
  long long ldo;
};

template <int DT, int MT, int RB>
__global__ __launch_bounds__(MT == 1 ? 512 : 256) void shrink_k(Fwd f) {
  constexpr int NW = MT == 1 ? 8 : 4, T = 16 * MT, W = 16 * RB;
  __shared__ float sums[NW][T][W];
  if ((int)blockIdx.x >= f.p.first[f.p.n + 2]) return;
  const Tile t = f.p.tiles[blockIdx.x];
  const int lane = lane_id(), w = uniform((int)threadIdx.x / WAVE), col = lane % 16, g = lane / 16;
  const int r0 = (int)blockIdx.y * W;
  if (t.adapter < 0) {
    const float v = t.adapter == NONE ? 0.f : __builtin_nanf("");
    for (int i = (int)threadIdx.x; i < t.count * W; i += NW * WAVE)
      if (r0 + i % W < f.R)
        f.hidden[(size_t)f.p.order[t.start + i / W] * f.R + r0 + i % W] = v;
    return;
  }
  const uint16_t *xp[MT], *ap[RB];
#pragma unroll
  for (int i = 0; i < MT; ++i)             // (rows past the tile's last: its last again, not stored)
    xp[i] = f.x + (size_t)f.p.order[t.start + min(16 * i + col, t.count - 1)] * f.ldx;
#pragma unroll
  for (int j = 0; j < RB; ++j)
    ap[j] = f.a + ((size_t)t.adapter * f.R + min(r0 + 16 * j + col, f.R - 1)) * f.K;
  v4f acc[MT][RB] = {};
#pragma unroll 2
  for (int k = w * 32; k < f.K; k += NW * 32) {
    const int kk = k + 8 * g;
    v4u xv[MT], av[RB];
#pragma unroll
    for (int i = 0; i < MT; ++i) xv[i] = load8(xp[i] + kk, f.K - kk);
#pragma unroll
    for (int j = 0; j < RB; ++j) av[j] = load8(ap[j] + kk, f.K - kk);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < RB; ++j) acc[i][j] = mfma<DT>(xv[i], av[j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < RB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[w][16 * i + 4 * g + e][16 * j + col] = acc[i][j][e];
  __syncthreads();
  const float s = f.scale[t.adapter];
  for (int i = (int)threadIdx.x; i < t.count * W; i += NW * WAVE) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) v += sums[k][i / W][i % W];
    if (r0 + i % W < f.R) f.hidden[(size_t)f.p.order[t.start + i / W] * f.R + r0 + i % W] = s * v;
  }
}

// ---- out = y + h B^T --------------------------------------------------------------------------------------
// h goes in as a sum of two 16-bit values, so that it is not rounded to the operands' type. Outputs come by four
// consecutive columns a lane and instruction: with rows of B handed out by fours, two of them make 16 bytes.
constexpr int STRIP = 512;                 // columns of a workgroup

template <int DT, int MT, int KS>
__global__ __launch_bounds__(256) void expand_k(Fwd f, int strips) {
  const int tile = (int)(blockIdx.x / (unsigned)strips), n0 = (int)(blockIdx.x % (unsigned)strips) * STRIP;
  if (tile >= f.p.first[f.p.n + 2]) return;
  const Tile t = f.p.tiles[tile];
  const int lane = lane_id(), w = uniform((int)threadIdx.x / WAVE), col = lane % 16, g = lane / 16;
  int row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) row[i] = f.p.order[t.start + min(16 * i + col, t.count - 1)];
  if (t.adapter == NONE) {
    if (f.y == f.out && f.ldy == f.ldo) return;
#pragma unroll
    for (int i = 0; i < MT; ++i)
      if (16 * i + col < t.count)
        for (int c = n0 + w * 32 + 8 * g; c < min(n0 + STRIP, f.N); c += 128)
          store8(f.out + (size_t)row[i] * f.ldo + c, load8(f.y + (size_t)row[i] * f.ldy + c, f.N - c),
                 f.N - c);
    return;
  }
  v4u hi[MT][KS], lo[MT][KS];
  float back[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    back[i] = split_row<DT, KS>(f.hidden + (size_t)row[i] * f.R, f.R, g, hi[i], lo[i]);
  const uint16_t* b = f.b + (size_t)max(t.adapter, 0) * f.N * f.R;       // (BAD: h is NaN)
  for (int c0 = n0 + w * 32; c0 < min(n0 + STRIP, f.N); c0 += 128) {
    v4u bv[2][KS];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = min(c0 + col / 4 * 8 + j * 4 + col % 4, f.N - 1);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        bv[j][k] = load8(b + (size_t)n * f.R + 32 * k + 8 * g, f.R - 32 * k - 8 * g);
    }
    const int c = c0 + 8 * g;
    v4u yv[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      yv[i] = v4u{};
      if (16 * i + col < t.count) yv[i] = load8(f.y + (size_t)row[i] * f.ldy + c, f.N - c);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      v4f acc[2] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[j] = mfma<DT>(bv[j][k], lo[i][k], acc[j]);
          acc[j] = mfma<DT>(bv[j][k], hi[i][k], acc[j]);
        }
      v4u o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = acc[e / 2][e % 2 * 2], q = acc[e / 2][e % 2 * 2 + 1];
        o[e] = to_bits<DT>(to_f32<DT>(yv[i][e] & 0xffffu) + (DT == 0 ? p : p * back[i])) |
               to_bits<DT>(to_f32<DT>(yv[i][e] >> 16) + (DT == 0 ? q : q * back[i])) << 16;
      }
      if (16 * i + col < t.count) store8(f.out + (size_t)row[i] * f.ldo + c, o, f.N - c);
    }
  }
}

template <int DT, int MT>
static void forward(const Fwd& f, hipStream_t stream) {
  const int strips = (f.N + STRIP - 1) / STRIP;
  const dim3 tiles((unsigned)f.p.cap), half((unsigned)f.p.cap, 2);
  const dim3 grid((unsigned)f.p.cap * strips);
#define RLU_SHRINK(RB, G) \
  hipLaunchKernelGGL((shrink_k<DT, MT, RB>), G, dim3(MT == 1 ? 512 : 256), 0, stream, f)
  if (f.R <= 16) RLU_SHRINK(1, tiles);
  else if (f.R <= 32) RLU_SHRINK(2, tiles);
  else if (f.R <= 64) RLU_SHRINK(4, tiles);
  else RLU_SHRINK(4, half);
#undef RLU_SHRINK
#define RLU_EXPAND(KS) \
  hipLaunchKernelGGL((expand_k<DT, MT, KS>), grid, dim3(256), 0, stream, f, strips)
  if (f.R <= 32) RLU_EXPAND(1);
  else if (f.R <= 64) RLU_EXPAND(2);
  else RLU_EXPAND(4);
#undef RLU_EXPAND
}

}  // namespace lora
}  // namespace rlu

extern "C" int rlu_lora_plan(const void* ids, int wide, int rows, int n, int size, int cap, int* order,
                             int* tiles, int* first, hipStream_t stream) {
  using namespace rlu::lora;
  if (!sizes_ok(0, rows, n, size, cap, 1, 1, 1) || (wide != 0 && wide != 1)) return -1;
  if (rows == 0) return 0;
  if (!ids || !order || !tiles || !first) return -1;
  if ((uintptr_t)tiles % 16 || ((uintptr_t)order | (uintptr_t)first) % 4) return -4;
  const size_t lds = ((PLAN_NW + 2) * (size_t)(n + 2) + 1) * sizeof(int);
  hipLaunchKernelGGL(plan_k, dim3(1), dim3(PLAN_NT), lds, stream, ids, wide, rows, n, size, order,
                     (Tile*)tiles, first);
  return (int)hipGetLastError();
}

extern "C" int rlu_lora_add(const void* x, long long ldx, const void* a, const void* b,
                            const float* scale, int dtype, const int* order, const int* tiles,
                            const int* first, int rows, int n, int size, int cap, int K, int N, int R,
                            float* hidden, const void* y, long long ldy, void* out, long long ldo,
                            hipStream_t stream) {
  using namespace rlu::lora;
  if (!sizes_ok(dtype, rows, n, size, cap, K, N, R) || ldx < 0 || ldy < 0) return -1;
  if (rows == 0) return 0;
  if (!x || !a || !b || !scale || !order || !tiles || !first || !hidden || !y || !out) return -1;
  if (rows > 1 && ldo < N) return -1;
  if ((long long)cap * ((N + STRIP - 1) / STRIP) > UINT32_MAX / 256 ||
      (long long)cap > UINT32_MAX / 512)
    return -1;                                         // (a launch counts its threads in 32 bits)
  if (((uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)y | (uintptr_t)out) % 2 ||
      ((uintptr_t)scale | (uintptr_t)hidden | (uintptr_t)order | (uintptr_t)first) % 4 ||
      (uintptr_t)tiles % 16)
    return -4;
  Fwd f = {(const uint16_t*)x, ldx, (const uint16_t*)a, (const uint16_t*)b, scale,
           {order, (const Tile*)tiles, first, n, rows, cap}, K, N, R, hidden, (const uint16_t*)y, ldy,
           (uint16_t*)out, ldo};
  if (dtype == 0 && size == 16) forward<0, 1>(f, stream);
  else if (dtype == 0) forward<0, 4>(f, stream);
  else if (size == 16) forward<2, 1>(f, stream);
  else forward<2, 4>(f, stream);
  return (int)hipGetLastError();
}
