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
// Each wave counts and later places a run of the rows, 64 at a time in order, so the order is the same on every run. One
// workgroup's chain of loads and barriers: 3 - 4 us up to 8192 rows, once for all the projections of a batch.
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
    int at = 0, tile = 0, live = 0;
    for (int g0 = 0; g0 < groups; g0 += WAVE) {
      const int g = g0 + lane, c = g < groups ? start[g] : 0, t = (c + size - 1) / size;
      const int sc = wave_incl_scan(c), st = wave_incl_scan(t);
      if (g < groups) {
        start[g] = at + sc - c;
        tile0[g] = tile + st - t;
        first[g] = tile + st - t;
      }
      live += (int)__popcll(__ballot(c > 0 && g < n));
      at += readlane(sc, WAVE - 1);
      tile += readlane(st, WAVE - 1);
    }
    if (lane == 0) {
      first[groups] = tile;
      first[groups + 1] = live;
      first[groups + 2] = start[n];
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

struct Fwd {
  const uint16_t* x;
  long long ldx;
  const uint16_t *a, *b;
  const float* scale;
  Plan p;
  int size, K, N, R;                       // size: rows of a tile
  float* hidden;
  const uint16_t* y;
  long long ldy;
  uint16_t* out;
  long long ldo;
};

// Part `sub` of a tile: 16 MT of its rows. Its tile, and none where it has no rows there.
template <int MT>
__device__ __forceinline__ Tile part_of(const Fwd& f, int block) {
  const int subs = f.size / (16 * MT), tile = block / subs, sub = block % subs;
  if (tile >= f.p.first[f.p.n + 2]) return {NONE, 0, 0, 0};
  Tile t = f.p.tiles[tile];
  t.start += sub * 16 * MT;
  t.count = min(16 * MT, t.count - sub * 16 * MT);
  return t;
}

// ---- h = s x A^T ------------------------------------------------------------------------------------------
// A workgroup 16 or 32 rows and 64 ranks: its waves take turns at the depth, 64 of it at a time, and are summed through
// LDS. Rows of x and of A come in pieces of 128 bytes a row and go through LDS: as the matrix unit wants them, with each
// lane's neighbour in another row, a load would take 64 accesses of 16 bytes (measured: 64 cache accesses a load).
// Bound by x: 8192 x 2560 with ranks of 64 19 - 20 us, 2.2 TB/s of x's 42 MB behind the writes of what ran before (three steps
// ahead 24, 16 rows a workgroup 20.5); 160 x 2560, R = 16, 32 adapters 5 - 6 us, a chain of five steps.
constexpr int SHRINK_NT = 512, DEPTH = 2;

template <int MT, int RB, int NT>
struct ShrinkLds {
  static constexpr int NW = NT / WAVE, T = 16 * MT, W = 16 * RB, LD = 64;
  static constexpr int TILES = NW * (T + W) * LD, SUMS = 2 * NW * T * W;
  alignas(16) uint16_t tiles[TILES > SUMS ? TILES : SUMS];             // rows of x and A, then each wave's sums
};

// Calls put(row, rank, h) for the rows of t and the ranks from r0 on.
template <int DT, int MT, int RB, bool WHOLE, int NT, class Put>
__device__ __forceinline__ void shrink(const Fwd& f, const Tile& t, int r0, ShrinkLds<MT, RB, NT>& lds, Put put) {
  typedef ShrinkLds<MT, RB, NT> L;
  constexpr int NW = L::NW, T = L::T, W = L::W, LD = L::LD;
  const int lane = lane_id(), w = uniform((int)threadIdx.x / WAVE), col = lane % 16, g = lane / 16;
  const int r8 = lane / 8, c8 = lane % 8 * 8;
  uint16_t *xt = lds.tiles + w * (T + W) * LD, *at = xt + T * LD;
  const uint16_t *xp[2 * MT], *ap[2 * RB];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i)         // (rows past the last: the last again, not stored)
    xp[i] = f.x + (size_t)f.p.order[t.start + min(8 * i + r8, t.count - 1)] * f.ldx;
#pragma unroll
  for (int j = 0; j < 2 * RB; ++j)
    ap[j] = f.a + ((size_t)t.adapter * f.R + min(r0 + 8 * j + r8, f.R - 1)) * f.K;
  v4u xv[DEPTH][2 * MT], av[DEPTH][2 * RB];
  auto load = [&](int d, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) xv[d][i] = fetch<WHOLE>(xp[i], k + c8, f.K);
#pragma unroll
    for (int j = 0; j < 2 * RB; ++j) av[d][j] = fetch<WHOLE>(ap[j], k + c8, f.K);
  };
  // chunks of 16 bytes swapped by the row, so that a fragment's 16 rows lie over all banks
  const int at16 = (lane % 8 ^ r8) * 8;
  auto fr = [&](const uint16_t* tile, int row, int k) __attribute__((always_inline)) {
    return *(const v4u*)&tile[(row + col) * LD + ((k / 8 + g) ^ (col % 8)) * 8];
  };
  v4f acc[MT][RB] = {};
  constexpr int STEP = NW * 64;
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (w * 64 + d * STEP < f.K) load(d, w * 64 + d * STEP);
  for (int k0 = w * 64; k0 < f.K; k0 += DEPTH * STEP)
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = k0 + d * STEP;
      if (k >= f.K) break;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) *(v4u*)&xt[(8 * i + r8) * LD + at16] = keep<WHOLE>(xv[d][i], k + c8, f.K);
#pragma unroll
      for (int j = 0; j < 2 * RB; ++j) *(v4u*)&at[(8 * j + r8) * LD + at16] = keep<WHOLE>(av[d][j], k + c8, f.K);
      wave_lds_sync();
      if (k + DEPTH * STEP < f.K) load(d, k + DEPTH * STEP);
#pragma unroll
      for (int s = 0; s < 64; s += 32) {
        v4u xf[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) xf[i] = fr(xt, 16 * i, s);
#pragma unroll
        for (int j = 0; j < RB; ++j) {
          const v4u af = fr(at, 16 * j, s);
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][j] = mfma<DT>(xf[i], af, acc[i][j]);
        }
      }
      wave_lds_sync();
    }
  __syncthreads();
  float* sums = (float*)lds.tiles;         // [NW][T][W]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < RB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[(w * T + 16 * i + 4 * g + e) * W + 16 * j + col] = acc[i][j][e];
  __syncthreads();
  const float s = f.scale[t.adapter];
  for (int i = (int)threadIdx.x; i < t.count * W; i += NT) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < NW; ++q) v += sums[q * T * W + i];
    if (r0 + i % W < f.R) put(i / W, r0 + i % W, s * v);
  }
}
// h of rows without an adapter, and of ids past the last
template <int NT, class Put>
__device__ __forceinline__ void bare(const Fwd& f, const Tile& t, int r0, int ranks, Put put) {
  const float v = t.adapter == NONE ? 0.f : __builtin_nanf("");
  for (int i = (int)threadIdx.x; i < t.count * ranks; i += NT)
    if (r0 + i % ranks < f.R) put(i / ranks, r0 + i % ranks, v);
}

template <int DT, int MT, int RB, bool WHOLE, int NT>
__global__ __launch_bounds__(NT) void shrink_k(Fwd f) {
  __shared__ ShrinkLds<MT, RB, NT> lds;
  const Tile t = part_of<MT>(f, (int)blockIdx.x);
  if (t.count <= 0) return;
  const int r0 = (int)blockIdx.y * 16 * RB;
  auto put = [&](int row, int r, float v) { f.hidden[(size_t)f.p.order[t.start + row] * f.R + r] = v; };
  if (t.adapter < 0) bare<NT>(f, t, r0, 16 * RB, put);
  else shrink<DT, MT, RB, WHOLE, NT>(f, t, r0, lds, put);
}

template <int DT, int MT, int KS, bool WHOLE>
__global__ __launch_bounds__(EXPAND_NT) void expand_k(Fwd f, int strips, int strip) {
  __shared__ ExpandLds<DT, MT, KS, false> lds;
  const int tile = (int)(blockIdx.x / (unsigned)strips);
  if (tile >= f.p.first[f.p.n + 2]) return;
  const Tile t = f.p.tiles[tile];
  const int n0 = (int)(blockIdx.x % (unsigned)strips) * strip, n1 = min(n0 + strip, f.N);
  const Out o = {f.b, f.y, f.ldy, f.out, f.ldo, f.N, f.R};
  if (t.adapter == NONE) return copy(o, f.p, t, n0, n1);
  stage<DT, MT, KS, EXPAND_NT>(lds.h, t.count, f.R, [&](int row) {
    return f.hidden + (size_t)f.p.order[t.start + row] * f.R;
  });
  expand<DT, MT, KS, WHOLE, false, true>(o, f.p, t, n0, n1, lds);
}

// Both in one launch where the tiles' strips have a CU each: every strip's workgroup works h out for itself.
// (in place, ranks of 16, us: 5 workgroups 5.9, two launches 7.4; 110 6.5 and 8.1; 360 12.0 and 9.5; ranks of 64
// and 240 workgroups 11.5 and 11.5)
constexpr int BOTH_STRIP = SHRINK_NT;      // columns: 64 a wave
template <int DT, int RB, bool WHOLE>
__global__ __launch_bounds__(SHRINK_NT) void both_k(Fwd f, int strips) {
  constexpr int KS = (RB + 1) / 2, LD = 16 * RB + 4;
  __shared__ union {
    ShrinkLds<1, RB, SHRINK_NT> first;
    ExpandLds<DT, 1, KS, false, SHRINK_NT> then;
  } lds;
  __shared__ float h[16 * LD];
  const int tile = (int)(blockIdx.x / (unsigned)strips), strip = (int)(blockIdx.x % (unsigned)strips);
  if (tile >= f.p.first[f.p.n + 2]) return;
  const Tile t = f.p.tiles[tile];
  const int n0 = strip * BOTH_STRIP, n1 = min(n0 + BOTH_STRIP, f.N);
  const Out o = {f.b, f.y, f.ldy, f.out, f.ldo, f.N, f.R};
  auto put = [&](int row, int r, float v) {
    h[row * LD + r] = v;
    if (strip == 0) f.hidden[(size_t)f.p.order[t.start + row] * f.R + r] = v;
  };
  if (t.adapter < 0) bare<SHRINK_NT>(f, t, 0, 16 * RB, put);
  else shrink<DT, 1, RB, WHOLE, SHRINK_NT>(f, t, 0, lds.first, put);
  if (t.adapter == NONE) return copy<SHRINK_NT>(o, f.p, t, n0, n1);
  __syncthreads();
  stage<DT, 1, KS, SHRINK_NT>(lds.then.h, t.count, f.R, [&](int row) { return (const float*)h + row * LD; });
  expand<DT, 1, KS, WHOLE, false, true, SHRINK_NT>(o, f.p, t, n0, n1, lds.then);
}

template <int DT, bool WHOLE>
static void forward(const Fwd& f, hipStream_t stream) {
  const int two = (f.N + BOTH_STRIP - 1) / BOTH_STRIP;
  if (f.size == 16 && f.R <= 64 && (long long)f.p.cap * two <= 256) {
    const dim3 grid(f.p.cap * two), block(SHRINK_NT);
    if (f.R <= 16) hipLaunchKernelGGL((both_k<DT, 1, WHOLE>), grid, block, 0, stream, f, two);
    else if (f.R <= 32) hipLaunchKernelGGL((both_k<DT, 2, WHOLE>), grid, block, 0, stream, f, two);
    else hipLaunchKernelGGL((both_k<DT, 4, WHOLE>), grid, block, 0, stream, f, two);
    return;
  }
  const int strip = strip_of(f.p.cap, f.size, f.N), strips = (f.N + strip - 1) / strip;
  // 64 ranks of 32 rows: half the threads, as the others' LDS (98 KB) would leave them a workgroup a CU and some CUs a second
  // one after it (8192 x 2560: 22.4 us, 19.5 so; 16 ranks of 1024 rows 8.3 and 9.4)
#define RLU_SHRINK(MT, RB, Y)                                                                      \
  hipLaunchKernelGGL((shrink_k<DT, MT, RB, WHOLE, MT * RB == 8 ? SHRINK_NT / 2 : SHRINK_NT>),      \
                     dim3(f.p.cap * (f.size / (16 * MT)), Y),                                      \
                     dim3(MT * RB == 8 ? SHRINK_NT / 2 : SHRINK_NT), 0, stream, f)
#define RLU_EXPAND(MT, KS)                                                                         \
  hipLaunchKernelGGL((expand_k<DT, MT, KS, WHOLE>), dim3(f.p.cap * strips), dim3(EXPAND_NT), 0,    \
                     stream, f, strips, strip)
#define RLU_FORWARD(MT, ALL)                                                                       \
  do {                                                                                             \
    if (f.R <= 16) RLU_SHRINK(MT, 1, 1);                                                           \
    else if (f.R <= 32) RLU_SHRINK(MT, 2, 1);                                                      \
    else RLU_SHRINK(MT, 4, f.R <= 64 ? 1 : 2);                                                     \
    if (f.R <= 32) RLU_EXPAND(ALL, 1);                                                             \
    else if (f.R <= 64) RLU_EXPAND(ALL, 2);                                                        \
    else RLU_EXPAND(ALL, 4);                                                                       \
  } while (0)
  if (f.size == 16) RLU_FORWARD(1, 1);
  else RLU_FORWARD(2, 4);
#undef RLU_FORWARD
#undef RLU_EXPAND
#undef RLU_SHRINK
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
  const long long parts = cap * (size / 16ll);
  if (cap * ((N + 255ll) / 256) > UINT32_MAX / EXPAND_NT || parts > UINT32_MAX / SHRINK_NT)
    return -1;                                         // (a launch counts its threads in 32 bits)
  if (((uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)y | (uintptr_t)out) % 2 ||
      ((uintptr_t)scale | (uintptr_t)hidden | (uintptr_t)order | (uintptr_t)first) % 4 ||
      (uintptr_t)tiles % 16)
    return -4;
  Fwd f = {(const uint16_t*)x, ldx, (const uint16_t*)a, (const uint16_t*)b, scale,
           {order, (const Tile*)tiles, first, n, rows, cap}, size, K, N, R, hidden, (const uint16_t*)y, ldy,
           (uint16_t*)out, ldo};
  const bool whole = (K | N | R) % 8 == 0;
  if (dtype == 0 && whole) forward<0, true>(f, stream);
  else if (dtype == 0) forward<0, false>(f, stream);
  else if (whole) forward<2, true>(f, stream);
  else forward<2, false>(f, stream);
  return (int)hipGetLastError();
}
