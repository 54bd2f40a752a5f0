// The backward pass of out = y + h B^T, h = s x A^T, from dy [rows, N] and h as the forward pass left it:
//   u = s dy B, dx = u A; of each adapter over its own rows dA = u^T x, dB = dy^T h.
// dy is read once, for u and for dB. Products over the rows (dA, dB) and over the rank (dx) need operands across the way
// they lie in memory: their tiles go through LDS as they are and are read transposed. h and u take part as sums of 16-bit
// values each (Split).
//
// Bound by dy: 1024 x 151936, R = 16, 2 adapters (dy 311 MB) 79 - 83 us for u and dB, then 10 for u over the strips, 9 for dx,
// dA and dB's parts, 4 for dA's. 8192 x [2560 -> 10240], 8 adapters: R = 16 48 + 8 + 28 + 5, R = 64 103 - 109 + 16 + 51 + 7, where the
// registers leave two workgroups a CU, R = 128 175 + 33 + 43 + 55 + 8, where dy and x are read for 64 ranks at a time. u's parts, R
// floats a row for each 256 columns, are R / 128 of dy's own bytes, written and read again. 96 x 2560 x 2560 with one adapter: 7, 3,
// 5 us, each launch a chain of a few loads.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lora.h"
#include "rlu.h"
#include "wave.h"

namespace rlu {
namespace lora {

constexpr int NT = 256, NW = NT / WAVE;
constexpr int OUTER = 256;                 // columns of a workgroup of the products over the rows

struct Bwd {
  const uint16_t *dy, *x;
  long long lddy, ldx;
  const uint16_t *a, *b;
  const float* scale;
  Plan p;
  int size, K, N, R;
  const float* hidden;
  uint16_t* dx;
  long long lddx;
  uint16_t *da, *db;
  // workspace
  float* upart;                            // [strips of N][rows R, and 64 that nobody reads]
  float* u;                                // [rows][R]
  float *pa, *pb;                          // [sa][2][R][K], [sb][2][N][R]
  int sa, sb;                              // runs of tiles
};

// ---- dA = u^T x; dB = dy^T h and u = s dy B ------------------------------------------------------------------------
// A workgroup a strip of 256 columns and a run of tiles, a wave 64 of the columns; of each adapter in the run 32 rows at a
// time (its rows lie one after the other in the order). An adapter whose tiles lie in one run is written as it is; one
// that goes over several leaves a part in each, which a launch after this one adds up in order.
// Rows come in pieces of 512 bytes, one step ahead of their products; no load in flight is branched on or selected from, and
// barriers wait for LDS alone (anything else waits for all loads at once). 1024 x 151936, us: 100 at first, 96 without such
// waits, 82 with 512 bytes a row past the cache; 69 without writing u's parts (39 MB). Two steps ahead: 117 - 143, for half the
// workgroups a CU. Two to four times the runs: 78 - 80, and 12 more to join.
struct Side {
  const uint16_t* v;                       // x or dy
  long long ld;
  int cols, runs;
  const float* h;                          // u or h
  uint16_t* out;
  float* parts;
};
template <bool DB>
__device__ __forceinline__ Side side_of(const Bwd& f) {
  return DB ? Side{f.dy, f.lddy, f.N, f.sb, f.hidden, f.db, f.pb}
            : Side{f.x, f.ldx, f.K, f.sa, f.u, f.da, f.pa};
}

// Runs: one for each adapter that has rows, or for 128 rows; for 64 rows where that leaves CUs without a workgroup (256 rows
// of one adapter, [2560 -> 2560], R = 64, us: in two of 128 44, in four of 64 27, in eight of 32 28). Adapters of up to twice
// that are not cut by a run's end: their parts and the join cost more than uneven runs (256 rows of 8 adapters over [2560 ->
// 10240], R = 16: 27 us cut, 20 not).
constexpr int FEWEST = 64;
struct Runs {
  int per, whole;                          // tiles of a run; tiles of an adapter that is not cut
};
__device__ __forceinline__ Runs runs_of(const Bwd& f, const Side& o) {
  const int total = f.p.first[f.p.n], live = f.p.first[f.p.n + 3], rows = f.p.first[f.p.n + 4];
  const int strips = (o.cols + OUTER - 1) / OUTER, each = strips * max(live, rows / 128) >= 256 ? 128 : FEWEST;
  const int use = max(1, min(o.runs, max(live, rows / each)));
  return {max(1, (total + use - 1) / use), 2 * each / f.size};
}
__device__ __forceinline__ bool in_one(const Bwd& f, const Runs& r, int a) { return f.p.first[a + 1] - f.p.first[a] <= r.whole; }
__device__ __forceinline__ int run_start(const Bwd& f, const Runs& r, int tile) {
  const int total = f.p.first[f.p.n];
  if (tile >= total) return total;
  const int a = f.p.tiles[tile].adapter;
  return in_one(f, r, a) ? f.p.first[a] : tile;
}

template <int DT, int RB, bool DB>
struct OuterLds {
  static constexpr int W = 16 * RB, UW = W + 4;       // (four rows apart lie 16 banks apart)
  alignas(16) uint16_t v[NW * 32 * 72];    // the step's rows [32][VLD]; before them each wave's part of B
  alignas(16) uint16_t h[Split<DT>::N][W * 40];       // the parts of h or u, [rank][row]
  float u[DB ? NW : 1][DB ? 32 * UW : 1];
  int row[2][DB ? 32 : 1];                 // where the rows of this step and of the one before lie
  float top[NW];
};

template <int DT, int RB, bool WHOLE, bool DB>
__device__ __forceinline__ void outer(const Bwd& f, int block, int r0, OuterLds<DT, RB, DB>& lds) {
  constexpr int W = 16 * RB, UW = W + 4, EACH = 32 * W / NT, LDB = W + 8, VLD = OUTER + 8;
  const Side o = side_of<DB>(f);
  const int strips = (o.cols + OUTER - 1) / OUTER, run = block / strips, strip = block % strips;
  const Runs r = runs_of(f, o);
  const int t0 = run_start(f, r, run * r.per), t1 = run_start(f, r, (run + 1) * r.per);
  const int lane = lane_id(), tid = (int)threadIdx.x, w = uniform(tid / WAVE), col = lane % 16, g = lane / 16;
  const int c0 = strip * OUTER + w * 64;
  uint16_t* mine = lds.v + w * 32 * 72;
  const int vr = w * 8 + lane / 32, vc = strip * OUTER + lane % 32 * 8;        // of the rows this lane brings
  const uint32_t spare = (uint32_t)f.p.rows * f.R;     // (rows of 64 more behind each strip's part)
  float* upart = f.upart + (size_t)strip * (spare + WAVE);
  for (int tile = t0; tile < t1;) {
    const int a = f.p.tiles[tile].adapter, first = f.p.first[a], last = f.p.first[a + 1], end = min(last, t1);
    const int p0 = f.p.tiles[tile].start, p1 = f.p.tiles[end - 1].start + f.p.tiles[end - 1].count;
    tile = end;
    v4u bu[2][RB];
    if (DB) {                              // this wave's 64 rows of B, as the second operand of u
      const uint16_t* b = f.b + (size_t)a * f.N * f.R;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const int q = i * WAVE + lane, n = c0 + 32 * k + q / (2 * RB), r = r0 + q % (2 * RB) * 8;
          const v4u v = fetch<WHOLE>(b + (size_t)min(n, f.N - 1) * f.R, r, n < f.N ? f.R : 0);
          *(v4u*)&mine[q / (2 * RB) * LDB + q % (2 * RB) * 8] = keep<WHOLE>(v, r, n < f.N ? f.R : 0);
        }
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < RB; ++j) bu[k][j] = frag_tr<LDB>(mine, 0, 16 * j);
        wave_lds_sync();
      }
      lds_barrier();                       // (the rows come to the same place)
    }
    const float s = DB ? f.scale[a] : 1.f;
    v4f acc[RB][4] = {};
    // of the next step: its rows' places, its rows, its h. Places are asked for before the rows of the step before: what
    // comes back in order is waited for in order.
    struct Places {
      int v[4], h[EACH];
    };
    const int hrow = tid / W * 2;          // (two rows of h, one below the other, a thread)
    auto places = [&](int pos) __attribute__((always_inline)) {        // (past the end: the last row again)
      Places n;
#pragma unroll
      for (int i = 0; i < 4; ++i) n.v[i] = f.p.order[min(pos + vr + 2 * i, p1 - 1)];
#pragma unroll
      for (int i = 0; i < EACH; ++i) n.h[i] = f.p.order[min(pos + hrow + i % 2 + i / 2 * (2 * NT / W), p1 - 1)];
      return n;
    };
    const int hcol = min(r0 + tid % W, f.R - 1);       // (NT is a multiple of W)
    int vrow[4], odd = 0;
    v4u vv[4];
    float hv[EACH];
    auto load = [&](const Places& at) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vrow[i] = at.v[i];
        vv[i] = fetch<WHOLE, true>(o.v + (uint64_t)(uint32_t)at.v[i] * (uint32_t)o.ld, vc, o.cols);
      }
#pragma unroll
      for (int i = 0; i < EACH; ++i) hv[i] = o.h[(uint32_t)at.h[i] * (uint32_t)f.R + hcol];
    };
    Places at = places(p0);
    {
      const Places next = places(p0 + 32);
      load(at);
      at = next;
    }
    for (int pos = p0; pos < p1; pos += 32) {
      float by = 1.f;
      if (DT != 0) {                       // float16: h and u into its range by a power of two a step
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < EACH; ++i) m = fmaxf(m, fabsf(hv[i]));
#pragma unroll
        for (int l = 1; l < WAVE; l *= 2) m = fmaxf(m, __shfl_xor(m, l));
        if (lane == 0) lds.top[w] = m;
        lds_barrier();
        by = scale_to(fmaxf(fmaxf(lds.top[0], lds.top[1]), fmaxf(lds.top[2], lds.top[3])));
      }
      if (pos + 32 > p1 || (strip + 1) * OUTER > o.cols)               // zeros past the last row and column
#pragma unroll
        for (int i = 0; i < 4; ++i)
          vv[i] = pos + vr + 2 * i < p1 ? keep<WHOLE>(vv[i], vc, o.cols) : v4u{};
#pragma unroll
      for (int i = 0; i < 4; ++i) *(v4u*)&lds.v[(vr + 2 * i) * VLD + lane % 32 * 8] = vv[i];
#pragma unroll
      for (int i = 0; i < EACH; i += 2) {
        const int row = hrow + i * (NT / W), n = tid % W < f.R - r0 ? p1 - pos - row : 0;
        const Split<DT> p(n > 0 ? hv[i] * by : 0.f), q(n > 1 ? hv[i + 1] * by : 0.f);
#pragma unroll
        for (int k = 0; k < Split<DT>::N; ++k)
          *(uint32_t*)&lds.h[k][tid % W * 40 + row] = p.part[k] | q.part[k] << 16;
      }
      if (DB && lane % 32 == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) lds.row[odd][vr + 2 * i] = vrow[i];
      }
      lds_barrier();
      const Places next = places(pos + 64);
      load(at);
      at = next;
      if (DB)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v4f u[RB] = {};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const v4u vf = frag<VLD>(lds.v, 16 * i, w * 64 + 32 * k);
#pragma unroll
            for (int j = 0; j < RB; ++j) u[j] = mfma<DT>(vf, bu[k][j], u[j]);
          }
#pragma unroll
          for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) lds.u[w][(16 * i + 4 * g + e) * UW + 16 * j + col] = u[j][e];
        }
      v4u vf[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) vf[c] = frag_tr<VLD>(lds.v, 0, w * 64 + 16 * c);
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        v4f sums[4] = {};
        v4f(&t)[4] = DT != 0 ? sums : acc[j];
#pragma unroll
        for (int k = Split<DT>::N - 1; k >= 0; --k) {
          const v4u h = frag<40>(lds.h[k], 16 * j, 0);
#pragma unroll
          for (int c = 0; c < 4; ++c) t[c] = DB ? mfma<DT>(vf[c], h, t[c]) : mfma<DT>(h, vf[c], t[c]);
        }
        if (DT != 0)
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][c][e] = fmaf(t[c][e], 1.f / by, acc[j][c][e]);
      }
      lds_barrier();
      if (DB) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          // (no branch around the store: the waits after one would be for all that is on its way, this store among
          // it. What lies past the last row or rank goes to a row that nobody reads.)
          const int q = tid + i * NT;
          const bool in = q / W < p1 - pos && q % W < f.R - r0;
          const int at = q / W * UW + q % W;
          upart[in ? (uint32_t)lds.row[odd][q / W] * (uint32_t)f.R + hcol : spare + lane] =
              s * ((lds.u[0][at] + lds.u[1][at]) + (lds.u[2][at] + lds.u[3][at]));
        }
      }
      odd ^= 1;
    }
    // 16 ranks at a time through the wave's part of LDS, then eight of the gradient's consecutive elements a lane
    const bool whole = first >= t0 && last <= t1;
    const size_t one = (size_t)f.R * o.cols;
    uint16_t* out = o.out + a * one;
    float* part = o.parts + ((size_t)run * 2 + (first >= t0)) * one;
    float* t = (float*)mine;
#pragma unroll
    for (int j = 0; j < RB; ++j) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          t[DB ? (16 * c + 4 * g + e) * 16 + col : (4 * g + e) * 68 + 16 * c + col] = acc[j][c][e];
      wave_lds_sync();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = i * WAVE + lane, r = r0 + 16 * j + (DB ? q % 2 * 8 : q / 8), cc = c0 + (DB ? q / 2 : q % 8 * 8);
        const v4f x = *(const v4f*)&t[DB ? q * 8 : q / 8 * 68 + q % 8 * 8];
        const v4f y = *(const v4f*)&t[DB ? q * 8 + 4 : q / 8 * 68 + q % 8 * 8 + 4];
        if (r >= f.R || cc >= o.cols || !o.out) continue;
        const size_t at = DB ? (size_t)cc * f.R + r : (size_t)r * o.cols + cc;
        const int n = DB ? f.R - r : o.cols - cc;
        if (whole) {
          const v4u v = {to_bits2<DT>(x[0], x[1]), to_bits2<DT>(x[2], x[3]), to_bits2<DT>(y[0], y[1]),
                         to_bits2<DT>(y[2], y[3])};
          store8(out + at, v, n);
        } else if (n >= 8) {
          *(v4fa*)(part + at) = x;
          *(v4fa*)(part + at + 4) = y;
        } else {
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (e < n) part[at + e] = e < 4 ? x[e] : y[e - 4];
        }
      }
      wave_lds_sync();
    }
    lds_barrier();                         // (the next adapter's rows come to the same place)
  }
}

template <int DT, int RB, bool WHOLE>
__global__ __launch_bounds__(NT, RB == 1 ? 3 : RB == 4 && DT != 0 ? 1 : 2) void outer_k(Bwd f) {
  __shared__ OuterLds<DT, RB, true> lds;
  outer<DT, RB, WHOLE, true>(f, (int)blockIdx.x, (int)blockIdx.y * 16 * RB, lds);
}

// Adapters that go over several runs: their parts, in order; those without rows: zeros. (zeros alone with only)
template <int DT, bool DB>
__device__ __forceinline__ void join(const Bwd& f, int a, int block, int blocks, bool only) {
  const Side o = side_of<DB>(f);
  const Runs r = runs_of(f, o);
  const int first = f.p.first[a], last = f.p.first[a + 1];
  const int s0 = first < last ? first / r.per : 0, s1 = first < last ? (last - 1) / r.per : -1;
  if (s0 == s1 || (first < last && (only || in_one(f, r, a)))) return;
  const size_t one = (size_t)f.R * o.cols;
  uint16_t* out = o.out + a * one;
  for (size_t i = 8 * ((size_t)block * NT + threadIdx.x); i < one; i += (size_t)blocks * NT * 8) {
    if (i + 8 <= one) {
      v4f x = {}, y = {};
#pragma unroll 4
      for (int s = s0; s <= s1; ++s) {
        const float* p = o.parts + ((size_t)s * 2 + (s == s0)) * one + i;
        x += *(const v4fa*)p;
        y += *(const v4fa*)(p + 4);
      }
      const v4u v = {to_bits2<DT>(x[0], x[1]), to_bits2<DT>(x[2], x[3]), to_bits2<DT>(y[0], y[1]),
                     to_bits2<DT>(y[2], y[3])};
      store8(out + i, v, 8);
    } else {
      for (size_t e = i; e < one; ++e) {
        float v = 0.f;
        for (int s = s0; s <= s1; ++s) v += o.parts[((size_t)s * 2 + (s == s0)) * one + e];
        out[e] = (uint16_t)to_bits<DT>(v);
      }
    }
  }
}
template <int DT>
__global__ __launch_bounds__(NT) void join_k(Bwd f) {
  join<DT, false>(f, (int)blockIdx.y, (int)blockIdx.x, (int)gridDim.x, false);
}

// ---- u over the strips --------------------------------------------------------------------------------------
// 32 times four ranks of a tile a workgroup, eight threads each. (8192 rows, 40 strips, R = 64: 25 us with a rank a thread, 15;
// 16 times four by 16 threads 16, 8 by 32 22)
__global__ __launch_bounds__(NT) void sum_k(Bwd f) {
  __shared__ v4f sums[8][32];
  if ((int)blockIdx.x >= f.p.first[f.p.n + 2]) return;
  const Tile t = f.p.tiles[blockIdx.x];
  const int e = (int)threadIdx.x % 32, q = (int)threadIdx.x / 32, i = (int)blockIdx.y * 32 + e;
  const int fours = (f.R + 3) / 4, r = i % fours * 4;
  const bool in = i < t.count * fours;
  const size_t at = in ? (size_t)f.p.order[t.start + i / fours] * f.R + r : 0;
  const int strips = (f.N + OUTER - 1) / OUTER;
  const size_t step = (size_t)f.p.rows * f.R + WAVE;
  v4f v = {};
  if (in && t.adapter >= 0)                            // (past the last rank: the next row's, or what is behind the last)
#pragma unroll 8
    for (int k = q; k < strips; k += 8) v += *(const v4fa*)(f.upart + k * step + at);
  sums[q][e] = v;
  __syncthreads();
  if (q || !in) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += sums[k][e];
  if (t.adapter == BAD) v = v4f{} + __builtin_nanf("");
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (r + k < f.R) f.u[at + k] = v[k];
}

// ---- what needs u, and what dB's launch left -------------------------------------------------------------------------
// dx, a tile and strip a workgroup; dA's strips and runs; dB's parts and both gradients' zeros, `joins` workgroups an
// adapter: one launch of work that does not wait for one another.
struct Last {
  int dx, da, joins;                       // workgroups (joins: of an adapter)
  int strips, strip;                       // of dx
  int passes;                              // of dA, 64 ranks each
};
template <int DT, int MT, int RB, int KS, bool WHOLE>
__global__ __launch_bounds__(NT, RB == 1 ? 3 : 2) void last_k(Bwd f, Last l) {
  __shared__ union {
    ExpandLds<DT, MT, KS, true> dx;
    OuterLds<DT, RB, false> da;
  } lds;
  int block = (int)blockIdx.x;
  if (block < l.dx) {
    const int tile = block / l.strips, n0 = block % l.strips * l.strip;
    if (tile >= f.p.first[f.p.n + 2]) return;
    const Tile t = f.p.tiles[tile];
    const Out o = {f.a, nullptr, 0, f.dx, f.lddx, f.K, f.R};
    stage<DT, MT, KS, EXPAND_NT>(lds.dx.h, t.count, f.R, [&](int row) {
      return f.u + (size_t)f.p.order[t.start + row] * f.R;
    });
    expand<DT, MT, KS, WHOLE, true, false>(o, f.p, t, n0, min(n0 + l.strip, f.K), lds.dx);
    return;
  }
  block -= l.dx;
  if (block < l.da) {
    const int pass = l.da / l.passes;
    outer<DT, RB, WHOLE, false>(f, block % pass, block / pass * 16 * RB, lds.da);
    return;
  }
  block -= l.da;
  const int a = block / l.joins;
  if (f.db) join<DT, true>(f, a, block % l.joins, l.joins, false);
  if (f.da) join<DT, false>(f, a, block % l.joins, l.joins, true);
}

// Runs, at most: as many workgroups as the CUs take at a time, two each, and three of up to 16 ranks. (strips: of all passes
// over the ranks. 8192 rows of [2560 -> 10240], us: R = 64 with 240 workgroups 190, 480 162, 760 178; R = 128 with 480 277, 560
// 314; 512 rows of 64 adapters, R = 16, with 480 47, 760 43)
static int runs_at_most(int strips, int rows, int n, int R) {
  const int slots = R <= 16 ? 768 : 512, want = strips < slots ? slots / strips : 1;
  const int most = rows / FEWEST > n ? rows / FEWEST : rows < n ? rows : n;
  return want < most ? want : most > 1 ? most : 1;
}
static void layout(Bwd& f, long long* bytes) {
  const int strips = (f.N + OUTER - 1) / OUTER, passes = f.R > 64 ? 2 : 1;
  f.sa = runs_at_most((f.K + OUTER - 1) / OUTER * passes, f.p.rows, f.p.n, f.R);
  f.sb = runs_at_most(strips * passes, f.p.rows, f.p.n, f.R);
  long long at = 0;
  auto take = [&](long long n) {
    const long long was = at;
    at += (n + 255) / 256 * 256;
    return was;
  };
  uint8_t* ws = (uint8_t*)f.upart;
  f.upart = (float*)(ws + take(4ll * strips * (1ll * f.p.rows * f.R + WAVE)));
  f.u = (float*)(ws + take(4ll * f.p.rows * f.R));
  f.pa = (float*)(ws + take(f.sa > 1 ? 8ll * f.sa * f.R * f.K : 0));
  f.pb = (float*)(ws + take(f.sb > 1 ? 8ll * f.sb * f.R * f.N : 0));
  *bytes = at;
}

template <int DT, bool WHOLE>
static void backward(const Bwd& f, const Last& l, hipStream_t stream) {
  const unsigned cap = (unsigned)f.p.cap;
  const int bb = (f.N + OUTER - 1) / OUTER * f.sb;
#define RLU_OUTER(RB, Y) hipLaunchKernelGGL((outer_k<DT, RB, WHOLE>), dim3(bb, Y), dim3(NT), 0, stream, f)
  if (f.R <= 16) RLU_OUTER(1, 1);
  else if (f.R <= 32) RLU_OUTER(2, 1);
  else RLU_OUTER(4, f.R <= 64 ? 1 : 2);
#undef RLU_OUTER
  if (f.dx || f.da)
    hipLaunchKernelGGL(sum_k, dim3(cap, (f.size * ((f.R + 3) / 4) + 31) / 32), dim3(NT), 0, stream, f);
  const auto blocks = [&](const Last& l) { return dim3((unsigned)(l.dx + l.da + l.joins * f.p.n)); };
#define RLU_LAST(MT, RB, KS, L) \
  hipLaunchKernelGGL((last_k<DT, MT, RB, KS, WHOLE>), blocks(L), dim3(NT), 0, stream, f, L)
#define RLU_LAST_OF(MT)                                                                         \
  do {                                                                                          \
    if (f.R <= 16) {                                                                            \
      RLU_LAST(MT, 1, 1, l);                                                                    \
    } else if (f.R <= 32) {                                                                     \
      RLU_LAST(MT, 2, 1, l);                                                                    \
    } else if (f.R <= 64) {                                                                     \
      RLU_LAST(MT, 4, 2, l);                                                                    \
    } else { /* (dx's 123 KB of LDS would leave dA one workgroup a CU: 531 us, 450 apart) */        \
      Last dx = l, rest = l;                                                                    \
      dx.da = dx.joins = rest.dx = 0;                                                           \
      if (dx.dx) RLU_LAST(MT, 4, 4, dx);                                                        \
      RLU_LAST(MT, 4, 2, rest);                                                                 \
    }                                                                                           \
  } while (0)
  if (f.size == 16) RLU_LAST_OF(1);
  else RLU_LAST_OF(4);
#undef RLU_LAST_OF
#undef RLU_LAST
  if (f.da && f.sa > 1) {
    const long long per = ((long long)f.R * f.K + NT * 8 - 1) / (NT * 8);
    hipLaunchKernelGGL((join_k<DT>), dim3(per < 512 ? per : 512, f.p.n), dim3(NT), 0, stream, f);
  }
}

}  // namespace lora
}  // namespace rlu

static int grad_sizes(rlu::lora::Bwd& f, rlu::lora::Last& l, int dtype, int rows, int n, int size, int cap, int K, int N, int R,
                      long long* bytes) {
  using namespace rlu::lora;
  if (!sizes_ok(dtype, rows, n, size, cap, K, N, R)) return -1;
  f.p.rows = rows;
  f.p.cap = cap;
  f.p.n = n;
  f.size = size;
  f.K = K;
  f.N = N;
  f.R = R;
  layout(f, bytes);
  const int strip = strip_of(cap, size, K);
  const long long strips = (K + strip - 1) / strip, most = (long long)R * (N > K ? N : K);
  // Workgroups for an adapter's parts: those of an adapter without any end at once, and of 64 adapters with 512 each that
  // took 50 us; with 32 each, one that has all of 8192 rows at R = 64 took 90 us more than with 128.
  const long long each = 8192 / n > 1 ? (8192 / n < 512 ? 8192 / n : 512) : 1;
  const long long joins = (most + NT * 8 - 1) / (NT * 8);
  const long long blocks = 2ll * ((N + OUTER - 1) / OUTER) * f.sb, dx = cap * strips,
                  da = ((K + OUTER - 1) / OUTER) * (R > 64 ? 2ll : 1ll) * f.sa;
  l = {(int)dx, (int)da, (int)(joins < each ? joins : each), (int)strips, strip, R > 64 ? 2 : 1};
  if (blocks > UINT32_MAX / NT || dx + da + (long long)l.joins * n > UINT32_MAX / NT ||
      (long long)cap * ((size * ((R + 3) / 4) + 31) / 32) > UINT32_MAX / NT)
    return -1;                                         // (a launch counts its threads in 32 bits)
  return 0;
}

extern "C" int rlu_lora_grad_workspace(int dtype, int rows, int n, int size, int cap, int K, int N, int R,
                                       long long* bytes) {
  rlu::lora::Bwd f = {};
  rlu::lora::Last l;
  return bytes ? grad_sizes(f, l, dtype, rows, n, size, cap, K, N, R, bytes) : -1;
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
  Last l;
  if (grad_sizes(f, l, dtype, rows, n, size, cap, K, N, R, &bytes) || lddy < 0 || ldx < 0 ||
      lddy > INT32_MAX || ldx > INT32_MAX)
    return -1;
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
  if (!dx) l.dx = 0;
  if (!da) l.da = 0;
  const bool whole = (K | N | R) % 8 == 0;
  if (dtype == 0 && whole) backward<0, true>(f, l, stream);
  else if (dtype == 0) backward<0, false>(f, l, stream);
  else if (whole) backward<2, true>(f, l, stream);
  else backward<2, false>(f, l, stream);
  return (int)hipGetLastError();
}
