// The backward pass of out = y + h B^T, h = s x A^T, from dy [rows, N] and h as the forward pass left it:
//   u = s dy B, dx = u A; of each adapter over its own rows dA = u^T x, dB = dy^T h.
// Products over the rows (dA, dB) and over the rank (dx) need operands across the way they lie in memory: their tiles
// go through LDS as they are and are read transposed. h and u take part as sums of two 16-bit values each, laid out
// with a tile's rows next to each other.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lora.h"
#include "rlu.h"
#include "wave.h"

namespace rlu {
namespace lora {

constexpr int NT = 256, NW = NT / WAVE;

struct Bwd {
  const uint16_t *dy, *x;
  long long lddy, ldx;
  const uint16_t *a, *b;
  const float* scale;
  Plan p;
  int K, N, R, RP;                         // RP: R up to a multiple of 16
  const float* hidden;
  uint16_t* dx;
  long long lddx;
  uint16_t *da, *db;
  // workspace
  float* upart;                            // [us][rows][R], then the sum over us in the first
  int us;
  uint16_t *hp, *up;                       // [cap][2][RP][T]
  float *hs, *uscale;                      // [cap] what each tile's values were divided by (float16)
  float *pa, *pb;                          // [sa][2][R][K], [sb][2][N][R]
  int sa, sb;
};

// ---- u / s = dy B -----------------------------------------------------------------------------------------
// A workgroup a tile and a part of the columns, a wave 32 columns at a time.
template <int DT, int MT, int RB>
__global__ __launch_bounds__(NT) void u_k(Bwd f, int cols) {
  constexpr int T = 16 * MT, W = 16 * RB, LD = W + 8, Q = 32 * 2 * RB / WAVE;
  __shared__ uint16_t bt[NW][32][LD];
  __shared__ float sums[2][T][W];
  if ((int)blockIdx.x >= f.p.first[f.p.n]) return;     // (rows of real adapters come first)
  const Tile t = f.p.tiles[blockIdx.x];
  const int lane = lane_id(), w = uniform((int)threadIdx.x / WAVE), col = lane % 16, g = lane / 16;
  const int split = (int)blockIdx.y, r0 = (int)blockIdx.z * W;
  const int n0 = split * cols, n1 = min(n0 + cols, f.N);
  const uint16_t* b = f.b + (size_t)t.adapter * f.N * f.R + r0;
  const uint16_t* yp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    yp[i] = f.dy + (size_t)f.p.order[t.start + min(16 * i + col, t.count - 1)] * f.lddy;
  v4u yv[MT], bv[Q];
  auto load = [&](int n) {
#pragma unroll
    for (int i = 0; i < MT; ++i) yv[i] = load8(yp[i] + n + 8 * g, n1 - n - 8 * g);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int c = q * WAVE + lane, nn = n + c / (2 * RB), r = c % (2 * RB) * 8;
      bv[q] = load8(b + (size_t)nn * f.R + r, nn < n1 ? f.R - r0 - r : 0);
    }
  };
  v4f acc[MT][RB] = {};
  int n = n0 + w * 32;
  if (n < n1) load(n);
  while (n < n1) {
    v4u cur[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) cur[i] = yv[i];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int c = q * WAVE + lane;
      *(v4u*)&bt[w][c / (2 * RB)][c % (2 * RB) * 8] = bv[q];
    }
    wave_lds_sync();
    n += NW * 32;
    if (n < n1) load(n);
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const uint16_t* p = &bt[w][8 * g + col / 4][16 * j + col % 4 * 4];
      const v4s lo = read_tr(p), hi = read_tr(p + 4 * LD);
      const auto bf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][j] = mfma<DT>(cur[i], __builtin_bit_cast(v4u, bf), acc[i][j]);
    }
    wave_lds_sync();
  }
  auto put = [&](int k) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[k][16 * i + 4 * g + e][16 * j + col] = acc[i][j][e];
  };
  if (w >= 2) put(w - 2);
  __syncthreads();
  if (w < 2) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] += sums[w][16 * i + 4 * g + e][16 * j + col];
  }
  __syncthreads();
  if (w < 2) put(w);
  __syncthreads();
  for (int i = (int)threadIdx.x; i < t.count * W; i += NT)
    if (r0 + i % W < f.R)
      f.upart[((size_t)split * f.p.rows + f.p.order[t.start + i / W]) * f.R + r0 + i % W] =
          sums[0][i / W][i % W] + sums[1][i / W][i % W];
}

// ---- u over its parts; u and h laid out for the products over the rows ----------------------------------------
template <int DT, int T>
__global__ __launch_bounds__(NT) void pack_k(Bwd f) {
  constexpr int MAX = T * MAX_RANK;
  __shared__ float vals[MAX];              // [T][RP]
  __shared__ float top[NW];
  const int tile = (int)blockIdx.x, tid = (int)threadIdx.x, w = uniform(tid / WAVE);
  if (tile >= f.p.first[f.p.n + 2]) return;
  const Tile t = f.p.tiles[tile];
  if (t.adapter < 0) {                     // dx alone asks for these
    for (int i = tid; i < t.count * f.R; i += NT)
      f.upart[(size_t)f.p.order[t.start + i / f.R] * f.R + i % f.R] =
          t.adapter == NONE ? 0.f : __builtin_nanf("");
    return;
  }
  const float s = f.scale[t.adapter];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float m = 0.f;
    for (int i = tid; i < T * f.RP; i += NT) {
      const int row = i / f.RP, r = i % f.RP;
      float v = 0.f;
      if (row < t.count && r < f.R) {
        const size_t at = (size_t)f.p.order[t.start + row] * f.R + r;
        if (which == 0) {
          v = f.hidden[at];
        } else {
          for (int k = 0; k < f.us; ++k) v += f.upart[(size_t)k * f.p.rows * f.R + at];
          v *= s;
          f.upart[at] = v;
        }
      }
      vals[i] = v;
      m = fmaxf(m, fabsf(v));
    }
    float by = 1.f;
    if (DT != 0) {
#pragma unroll
      for (int d = 1; d < WAVE; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
      if (lane_id() == 0) top[w] = m;
    }
    __syncthreads();
    if (DT != 0) {
      by = scale_to(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
      if (tid == 0) (which == 0 ? f.hs : f.uscale)[tile] = 1.f / by;
    }
    uint16_t* to = (which == 0 ? f.hp : f.up) + (size_t)tile * 2 * f.RP * T;
    for (int i = tid; i < T * f.RP; i += NT) {
      const Split<DT> p(vals[i % T * f.RP + i / T] * by);
      to[i] = (uint16_t)p.hi;
      to[f.RP * T + i] = (uint16_t)p.lo;
    }
    __syncthreads();
  }
}

// ---- dx = u A ---------------------------------------------------------------------------------------------
template <int DT, int MT, int KS>
__global__ __launch_bounds__(NT) void dx_k(Bwd f, int strips) {
  constexpr int SC = KS == 4 ? 128 : 256, LD = SC + 8;
  __shared__ uint16_t at[32 * KS][LD];
  const int tile = (int)(blockIdx.x / (unsigned)strips), c0 = (int)(blockIdx.x % (unsigned)strips) * SC;
  if (tile >= f.p.first[f.p.n + 2]) return;
  const Tile t = f.p.tiles[tile];
  const int lane = lane_id(), tid = (int)threadIdx.x, w = uniform(tid / WAVE), col = lane % 16, g = lane / 16;
  int row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) row[i] = f.p.order[t.start + min(16 * i + col, t.count - 1)];
  const uint16_t* a = f.a + (size_t)max(t.adapter, 0) * f.R * f.K;
  const int R = t.adapter == NONE ? 0 : f.R;           // (0 times whatever adapter 0 holds may be NaN)
  for (int q = tid; q < 32 * KS * (SC / 8); q += NT) {
    const int r = q / (SC / 8), c = q % (SC / 8) * 8;
    *(v4u*)&at[r][c] = load8(a + (size_t)r * f.K + c0 + c, r < R ? f.K - c0 - c : 0);
  }
  v4u hi[MT][KS], lo[MT][KS];
  float back[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) back[i] = split_row<DT, KS>(f.upart + (size_t)row[i] * f.R, f.R, g, hi[i], lo[i]);
  __syncthreads();
#pragma unroll
  for (int b = 0; b < SC / 128; ++b) {
    const int cb = w * 32 + b * 128;
    v4u av[2][KS];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint16_t* p = &at[32 * k + 8 * g + col / 4][cb + col % 4 * 8 + j * 4];
        const v4s lo4 = read_tr(p), hi4 = read_tr(p + 4 * LD);
        av[j][k] = __builtin_bit_cast(v4u, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    const int c = c0 + cb + 8 * g;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      v4f acc[2] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[j] = mfma<DT>(av[j][k], lo[i][k], acc[j]);
          acc[j] = mfma<DT>(av[j][k], hi[i][k], acc[j]);
        }
      v4u o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = acc[e / 2][e % 2 * 2], q = acc[e / 2][e % 2 * 2 + 1];
        o[e] = to_bits<DT>(DT == 0 ? p : p * back[i]) | to_bits<DT>(DT == 0 ? q : q * back[i]) << 16;
      }
      if (16 * i + col < t.count) store8(f.dx + (size_t)row[i] * f.lddx + c, o, f.K - c);
    }
  }
}

// ---- dA = u^T x, dB = dy^T h ------------------------------------------------------------------------------
// A workgroup a strip of 256 columns and a run of tiles, a wave 64 of the columns, 32 rows at a time (or a tile of
// 16, both halves of its split values at once). An adapter whose tiles lie in one run is written as it is; one that
// goes over several leaves a part in each, which a launch after this one adds up in order.
constexpr int OUT_STRIP = 256;

struct Outer {
  const uint16_t* v;                       // x or dy
  long long ld;
  int cols, runs;
  const uint16_t* packed;                  // u or h
  const float* scales;
  uint16_t* out;
  float* parts;
};
template <bool SWAP>
__device__ __forceinline__ Outer outer_of(const Bwd& f) {
  return SWAP ? Outer{f.dy, f.lddy, f.N, f.sb, f.hp, f.hs, f.db, f.pb}
              : Outer{f.x, f.ldx, f.K, f.sa, f.up, f.uscale, f.da, f.pa};
}
// where element (r, c) of an adapter's gradient lies
template <bool SWAP>
__device__ __forceinline__ size_t place(const Outer& o, int R, int r, int c) {
  return SWAP ? (size_t)c * R + r : (size_t)r * o.cols + c;
}

template <int DT, int T, int RB, bool SWAP>
__device__ __forceinline__ void outer(const Bwd& f, int block, uint16_t (&xt)[NW][32][72]) {
  const Outer o = outer_of<SWAP>(f);
  const int strips = (o.cols + OUT_STRIP - 1) / OUT_STRIP, run = block / strips;
  const int lane = lane_id(), w = uniform((int)threadIdx.x / WAVE), col = lane % 16, g = lane / 16;
  const int c0 = block % strips * OUT_STRIP + w * 64;
  const int total = f.p.first[f.p.n], per = (total + o.runs - 1) / o.runs;
  const int t0 = run * per, t1 = min(t0 + per, total);
  if (t0 >= t1 || c0 >= o.cols) return;
  constexpr int STEPS = T == 64 ? 2 : 1, L = T == 64 ? 4 : 2;          // steps of a tile, loads of a step
  const int r0 = (int)blockIdx.y * 16 * RB;
  v4f acc[RB][4] = {};
  int tile = t0, step = 0;
  Tile t = f.p.tiles[tile];
  v4u xv[L];
  auto load = [&](const Tile& t, int step) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int m = step * 32 + i * 8 + lane / 8, c = c0 + lane % 8 * 8;
      xv[i] = load8(o.v + (size_t)f.p.order[t.start + min(m, t.count - 1)] * o.ld + c,
                    m < t.count ? o.cols - c : 0);
    }
  };
  load(t, 0);
  while (true) {
#pragma unroll
    for (int i = 0; i < L; ++i) *(v4u*)&xt[w][i * 8 + lane / 8][lane % 8 * 8] = xv[i];
    wave_lds_sync();
    const uint16_t* p = o.packed + (size_t)tile * 2 * f.RP * T;
    v4u hi[RB], lo[RB];
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const int r = r0 + 16 * j + col;
      const bool in = r < f.RP;
      if (T == 64) {
        hi[j] = load8(p + (size_t)r * T + step * 32 + 8 * g, in ? 8 : 0);
        lo[j] = load8(p + (size_t)(f.RP + r) * T + step * 32 + 8 * g, in ? 8 : 0);
      } else {
        hi[j] = load8(p + (size_t)(g / 2 * f.RP + r) * T + g % 2 * 8, in ? 8 : 0);
      }
    }
    const float back = DT != 0 ? o.scales[tile] : 1.f;
    // the next step's rows
    const Tile now = t;
    const int was = tile;
    if (step + 1 < STEPS && (step + 1) * 32 < t.count) {
      ++step;
    } else {
      step = 0;
      if (++tile < t1) t = f.p.tiles[tile];
    }
    if (tile < t1) load(t, step);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int k = T == 64 ? 8 * g : 8 * (g % 2);
      const uint16_t* q = &xt[w][k + col / 4][16 * c + col % 4 * 4];
      const v4s x0 = read_tr(q), x1 = read_tr(q + 4 * 72);
      const v4u xf = __builtin_bit_cast(v4u, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        v4f d = DT != 0 ? v4f{} : acc[j][c];
        if (T == 64) d = SWAP ? mfma<DT>(xf, lo[j], d) : mfma<DT>(lo[j], xf, d);
        d = SWAP ? mfma<DT>(xf, hi[j], d) : mfma<DT>(hi[j], xf, d);
        if (DT == 0) acc[j][c] = d;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][c][e] = fmaf(d[e], back, acc[j][c][e]);
      }
    }
    wave_lds_sync();
    if (tile == was) continue;
    if (tile < t1 && t.adapter == now.adapter) continue;
    // the adapter's last step here
    const int a = now.adapter, first = f.p.first[a], last = f.p.first[a + 1];
    const bool whole = first >= t0 && last <= t1;
    const size_t one = (size_t)f.R * o.cols;
    uint16_t* out = o.out + a * one;
    float* part = o.parts + ((size_t)run * 2 + (first >= t0)) * one;
#pragma unroll
    for (int j = 0; j < RB; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + 16 * j + (SWAP ? col : 4 * g + e);
          const int cc = c0 + 16 * c + (SWAP ? 4 * g + e : col);
          if (r >= f.R || cc >= o.cols) continue;
          const size_t at = place<SWAP>(o, f.R, r, cc);
          if (whole) out[at] = (uint16_t)to_bits<DT>(acc[j][c][e]);
          else part[at] = acc[j][c][e];
        }
        acc[j][c] = v4f{};
      }
    if (tile >= t1) return;
  }
}

template <int DT, int T, int RB>
__global__ __launch_bounds__(NT) void outer_k(Bwd f, int blocks_a) {
  __shared__ uint16_t xt[NW][32][72];
  const int b = (int)blockIdx.x;
  if (b < blocks_a) outer<DT, T, RB, false>(f, b, xt);
  else outer<DT, T, RB, true>(f, b - blocks_a, xt);
}

// Adapters that go over several runs: their parts, in order; those without rows: zeros.
template <int DT, bool SWAP>
__device__ __forceinline__ void join(const Bwd& f, int a, int block, int blocks) {
  const Outer o = outer_of<SWAP>(f);
  const int total = f.p.first[f.p.n], per = (total + o.runs - 1) / o.runs;
  const int first = f.p.first[a], last = f.p.first[a + 1];
  const size_t one = (size_t)f.R * o.cols;
  const int s0 = first < last ? first / per : 0, s1 = first < last ? (last - 1) / per : 0;
  if (first < last && s0 == s1) return;
  uint16_t* out = o.out + a * one;
  for (size_t i = (size_t)block * NT + threadIdx.x; i < one; i += (size_t)blocks * NT) {
    float v = 0.f;
    if (first < last)
      for (int s = s0; s <= s1; ++s) v += o.parts[((size_t)s * 2 + (s == s0)) * one + i];
    out[i] = (uint16_t)to_bits<DT>(v);
  }
}
template <int DT>
__global__ __launch_bounds__(NT) void join_k(Bwd f) {
  if (blockIdx.z == 0 && f.da) join<DT, false>(f, (int)blockIdx.y, (int)blockIdx.x, (int)gridDim.x);
  if (blockIdx.z == 1 && f.db) join<DT, true>(f, (int)blockIdx.y, (int)blockIdx.x, (int)gridDim.x);
}

// Parts of the columns of u, and runs of tiles of the gradients: workgroups for every CU, twice over.
static int parts_of(int blocks, int most) {
  const int want = blocks > 0 ? (512 + blocks - 1) / blocks : 1;
  return want < most ? want : most > 1 ? most : 1;
}
static void layout(Bwd& f, int size, long long* bytes) {
  f.RP = (f.R + 15) / 16 * 16;
  f.us = parts_of(f.p.cap, (f.N + 255) / 256);
  f.sa = parts_of((f.K + OUT_STRIP - 1) / OUT_STRIP, f.p.cap);
  f.sb = parts_of((f.N + OUT_STRIP - 1) / OUT_STRIP, f.p.cap);
  long long at = 0;
  auto take = [&](long long n) {
    const long long was = at;
    at += (n + 255) / 256 * 256;
    return was;
  };
  uint8_t* ws = (uint8_t*)f.upart;
  f.upart = (float*)(ws + take(4ll * f.us * f.p.rows * f.R));
  f.hp = (uint16_t*)(ws + take(4ll * f.p.cap * f.RP * size));
  f.up = (uint16_t*)(ws + take(4ll * f.p.cap * f.RP * size));
  f.hs = (float*)(ws + take(4ll * f.p.cap));
  f.uscale = (float*)(ws + take(4ll * f.p.cap));
  f.pa = (float*)(ws + take(f.sa > 1 ? 8ll * f.sa * f.R * f.K : 0));
  f.pb = (float*)(ws + take(f.sb > 1 ? 8ll * f.sb * f.R * f.N : 0));
  *bytes = at;
}

template <int DT, int MT>
static void backward(const Bwd& f, hipStream_t stream) {
  constexpr int T = 16 * MT;
  const unsigned cap = (unsigned)f.p.cap;
  const int cols = ((f.N + f.us - 1) / f.us + 31) / 32 * 32;
#define RLU_U(RB, Z) \
  hipLaunchKernelGGL((u_k<DT, MT, RB>), dim3(cap, f.us, Z), dim3(NT), 0, stream, f, cols)
  if (f.R <= 16) RLU_U(1, 1);
  else if (f.R <= 32) RLU_U(2, 1);
  else if (f.R <= 64) RLU_U(4, 1);
  else RLU_U(4, 2);
#undef RLU_U
  hipLaunchKernelGGL((pack_k<DT, T>), dim3(cap), dim3(NT), 0, stream, f);
  if (f.dx) {
    const int strips = f.R <= 64 ? (f.K + 255) / 256 : (f.K + 127) / 128;
#define RLU_DX(KS) \
  hipLaunchKernelGGL((dx_k<DT, MT, KS>), dim3(cap * strips), dim3(NT), 0, stream, f, strips)
    if (f.R <= 32) RLU_DX(1);
    else if (f.R <= 64) RLU_DX(2);
    else RLU_DX(4);
#undef RLU_DX
  }
  const int ba = f.da ? (f.K + OUT_STRIP - 1) / OUT_STRIP * f.sa : 0;
  const int bb = f.db ? (f.N + OUT_STRIP - 1) / OUT_STRIP * f.sb : 0;
  if (ba + bb == 0) return;
#define RLU_OUTER(RB, Y) \
  hipLaunchKernelGGL((outer_k<DT, T, RB>), dim3(ba + bb, Y), dim3(NT), 0, stream, f, ba)
  if (f.R <= 16) RLU_OUTER(1, 1);
  else if (f.R <= 32) RLU_OUTER(2, 1);
  else if (f.R <= 64) RLU_OUTER(4, 1);
  else RLU_OUTER(4, 2);
#undef RLU_OUTER
  const int per = (int)(((long long)f.R * (f.N > f.K ? f.N : f.K) + NT * 16 - 1) / (NT * 16));
  hipLaunchKernelGGL((join_k<DT>), dim3(per < 256 ? per : 256, f.p.n, 2), dim3(NT), 0, stream, f);
}

}  // namespace lora
}  // namespace rlu

static int grad_sizes(rlu::lora::Bwd& f, int dtype, int rows, int n, int size, int cap, int K, int N, int R,
                      long long* bytes) {
  using namespace rlu::lora;
  if (!sizes_ok(dtype, rows, n, size, cap, K, N, R)) return -1;
  f.p.rows = rows;
  f.p.cap = cap;
  f.p.n = n;
  f.K = K;
  f.N = N;
  f.R = R;
  layout(f, size, bytes);
  const long long strips = (N + OUT_STRIP - 1) / OUT_STRIP * (long long)f.sb +
                           (K + OUT_STRIP - 1) / OUT_STRIP * (long long)f.sa;
  if (2 * strips > UINT32_MAX / NT || (long long)cap * f.us * 2 > UINT32_MAX / NT ||
      (long long)cap * ((K + 127) / 128) > UINT32_MAX / NT)
    return -1;                                         // (a launch counts its threads in 32 bits)
  return 0;
}

extern "C" int rlu_lora_grad_workspace(int dtype, int rows, int n, int size, int cap, int K, int N, int R,
                                       long long* bytes) {
  rlu::lora::Bwd f = {};
  return bytes ? grad_sizes(f, dtype, rows, n, size, cap, K, N, R, bytes) : -1;
}

extern "C" int rlu_lora_grad(const void* dy, long long lddy, const void* x, long long ldx, const void* a,
                             const void* b, const float* scale, int dtype, const int* order,
                             const int* tiles, const int* first, int rows, int n, int size, int cap,
                             int K, int N, int R, const float* hidden, void* dx, long long lddx,
                             void* da, void* db, void* ws, hipStream_t stream) {
  using namespace rlu::lora;
  Bwd f = {};
  f.upart = (float*)ws;
  long long bytes;
  if (grad_sizes(f, dtype, rows, n, size, cap, K, N, R, &bytes) || lddy < 0 || ldx < 0) return -1;
  if (rows == 0) return 0;
  if (!dy || !x || !a || !b || !scale || !order || !tiles || !first || !hidden || !ws) return -1;
  if (dx && rows > 1 && lddx < K) return -1;
  if (((uintptr_t)dy | (uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)dx | (uintptr_t)da |
       (uintptr_t)db) % 2 ||
      ((uintptr_t)scale | (uintptr_t)hidden | (uintptr_t)order | (uintptr_t)first) % 4 ||
      ((uintptr_t)tiles | (uintptr_t)ws) % 16)
    return -4;
  f.dy = (const uint16_t*)dy;
  f.lddy = lddy;
  f.x = (const uint16_t*)x;
  f.ldx = ldx;
  f.a = (const uint16_t*)a;
  f.b = (const uint16_t*)b;
  f.scale = scale;
  f.p.order = order;
  f.p.tiles = (const Tile*)tiles;
  f.p.first = first;
  f.hidden = hidden;
  f.dx = (uint16_t*)dx;
  f.lddx = lddx;
  f.da = (uint16_t*)da;
  f.db = (uint16_t*)db;
  if (dtype == 0 && size == 16) backward<0, 1>(f, stream);
  else if (dtype == 0) backward<0, 4>(f, stream);
  else if (size == 16) backward<2, 1>(f, stream);
  else backward<2, 4>(f, stream);
  return (int)hipGetLastError();
}
