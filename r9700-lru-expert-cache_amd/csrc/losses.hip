// Losses over rows of logits, with the logits' gradient: the clipped policy loss of a sampled token, and the
// divergence from a teacher's listed log probabilities. With p = softmax(x / T) both gradients are
//   dL/dx_i = c e^(x_i / T) for a token that the row does not list, and one value for each that it lists
// (the sampled token, the teacher's ids), so a row is read once for the sum over the unlisted tokens and once
// more, from the cache, for the gradient.
//
//   * The listed tokens are left out of that sum, and join it by their own exponentials: 1 - p of a nearly certain
//     token, and what is left beside a teacher's list, are then sums and not differences.
//   * Sums are taken against a thread's own running maximum, a chunk at a time.
//
// Bound by the logits read and the gradient written, at a copy's rate (4.91 TB/s): 4096 bf16 rows of 151936 with 20 listed
// tokens 498 - 506 us, 2048 float32 rows with the policy loss 513 - 517, 4.8 - 5.0 TB/s; without a gradient 207 and 204, 6.0
// TB/s. Vector instructions take 61% and 27% of the cycles. At first 617 and 708 us; then
//   * the gradient is stored past the caches, so that rows still to be read again stay there: 542 / 684;
//   * the second read asks for no place in them either: 517 / 555;
//   * it goes backwards, from what came last, and no more rows are in flight than the memory-side cache holds: 506 / 517;
//   * one wave works out a row's coefficients, a thousand instructions, for all: 498; 617 f16 rows of 32003 26 -> 23 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "logits.h"
#include "numerics.h"
#include "rlu.h"
#include "wave.h"

namespace rlu {
namespace loss {

using lp::Elem;
using lp::lane_f;
using lp::load_one;
using lp::Max;
using lp::token_of;
using lp::v4u;
using lp::wave_add;
using lp::wave_max;

constexpr int MAX_TOP = 32, MAX_V = 500000;
constexpr int MOST_NW = 16;
constexpr double LOG2_E = 1.44269504088896340736;

// Threads of a workgroup, and the vectors of 16 bytes that each of them takes at a time.
template <int THREADS, int VECTORS>
struct Shape {
  static constexpr int NT = THREADS, NW = NT / WAVE, CV = VECTORS, CHUNK = CV * NT;
};
constexpr int MAX_SEGS = WAVE;
enum { POLICY, DISTILL };
typedef v4u v4ua __attribute__((aligned(2)));          // (16 bytes at any element's address)

struct Args {
  const uint8_t* logits;
  long long ld;
  int R, V, nseg;
  const void* ids;                         // the sampled tokens [R] or the teacher's [R][top]
  int wide, top;
  const float *old, *adv, *ref;            // policy [R]; ref may be null
  const float* vals;                       // teacher [R][top]
  const float* weight;                     // [R] or null
  int rest;
  float k, inv_t, lo, hi, kl;              // k = log2(e) / T
  float *loss, *logprob;
  uint8_t* grad;
  long long ldg;
  const float* by;                         // null, or [R] step apart: the gradient alone, of rows whose factor is not 1
  long long step;
};

// A row's workgroup (Wide: of long float32 rows), and a segment's. (4096 bf16 rows of 151936 with 256 threads 556 us, 517 with
// 512 at that step; eight vectors a thread: 503, but 617 rows of 32003 37 us, 26 with four)
typedef Shape<512, 4> Usual;
typedef Shape<1024, 4> Wide;
typedef Shape<256, 2> Short;
// Rows that one chunk of these holds: the work that a row costs whatever its length, one wave's coefficients and the waits
// around them, then leaves the CU to more rows. (distill with 20 listed, bf16, in shapes of 512 / 256 / 64 threads, us: 40000
// x 500 418 / 215 / 87, 4476 x 1666 55 / 34 / 19; 4096 x 8000 57 / 35 / 39, 1159 x 8000 21.4 / 14.6 / 23)
typedef Shape<256, 4> Medium;
typedef Shape<64, 4> Small;

// The maximum of a row's unlisted logits and sum e^((x - m) / T) over them. Nothing: -inf, 0.
struct Part {
  float m, s;
};

// What a row's gradient is made of: f e^((x - m) / T) of an unlisted logit. The listed ones' are in LDS.
struct Coef {
  float m, f;
};

struct Row {
  const uint8_t* p;
  const v4u* pv;                           // vectors from the aligned address at or below its start
  int shift, nvec;
};
template <int DT>
__device__ __forceinline__ Row row_of(const Args& a, int row) {
  Row r;
  r.p = a.logits + (size_t)row * a.ld * Elem<DT>::SIZE;
  r.shift = (int)((uintptr_t)r.p % 16) / Elem<DT>::SIZE;
  r.pv = reinterpret_cast<const v4u*>(r.p - r.shift * Elem<DT>::SIZE);
  r.nvec = (r.shift + a.V + Elem<DT>::N - 1) / Elem<DT>::N;
  return r;
}

template <int DT>
__device__ __forceinline__ uint32_t bits_of(float x) {
  if (DT == 0) return f32_to_bf16(x);
  if (DT == 1) return __float_as_uint(x);
  return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// raw's element at of its CV vectors becomes b (a dynamic index would put raw into memory)
template <int DT, int CV>
__device__ __forceinline__ void put(v4u (&raw)[CV], int k, int e, uint32_t b) {
  const int word = k * 4 + (Elem<DT>::SIZE == 4 ? e : e / 2);
#pragma unroll
  for (int i = 0; i < CV * 4; ++i) {
    const uint32_t u = raw[i / 4][i % 4];
    const uint32_t w = Elem<DT>::SIZE == 4 ? b : e % 2 ? (u & 0xffffu) | b << 16
                                                       : (u & 0xffff0000u) | b;
    raw[i / 4][i % 4] = word == i ? w : u;
  }
}

// What a row lists, in LDS: ids out of range as -1.
struct Listed {
  int id[MAX_TOP];
  float grad[MAX_TOP];
  float m[MOST_NW], s[MOST_NW];
  Coef coef;
  uint32_t owns[MOST_NW * WAVE];           // bit j: the thread's vectors hold id[j]
};

// Of a thread's vectors from `from` on the first that holds a listed logit.
template <int DT>
__device__ __forceinline__ int next_of(const Listed& l, uint32_t owns, int shift, int from) {
  int next = 0x7fffffff;
  for (uint32_t b = owns; b; b &= b - 1) {
    const int v = (l.id[__ffs((int)b) - 1] + shift) / Elem<DT>::N;
    if (v >= from) next = min(next, v);
  }
  return next;
}
// Puts of(j) in the place of each listed logit j of the thread's chunk at `base`.
template <int DT, class S, class Of>
__device__ __forceinline__ void replace(v4u (&raw)[S::CV], const Listed& l, uint32_t owns, int shift,
                                        int base, Of of) {
  for (uint32_t b = owns; b; b &= b - 1) {
    const int j = __ffs((int)b) - 1, i = l.id[j] + shift, v = i / Elem<DT>::N;
    if (v >= base && v < base + S::CHUNK) put<DT>(raw, (v - base) / S::NT, i % Elem<DT>::N, of(j));
  }
}

// LAST: nobody asks for these again
template <int DT, class S, bool LAST>
__device__ __forceinline__ void load(v4u (&raw)[S::CV], const Row& r, int base) {
#pragma unroll
  for (int k = 0; k < S::CV; ++k) {
    const int v = base + k * S::NT + (int)threadIdx.x;
    if (v < r.nvec) {
      raw[k] = LAST ? __builtin_nontemporal_load(r.pv + v) : r.pv[v];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        raw[k][j] = Elem<DT>::SIZE == 4 ? Elem<DT>::NINF : Elem<DT>::NINF * 0x10001u;
    }
  }
}
// elements of the neighbours in a row's end vectors
template <int DT, class S>
__device__ __forceinline__ void trim(v4u (&raw)[S::CV], const Row& r, int V, int base) {
  typedef Elem<DT> E;
#pragma unroll
  for (int k = 0; k < S::CV; ++k) {
    const int v = base + k * S::NT + (int)threadIdx.x;
    if ((v == 0 && r.shift) || v == r.nvec - 1)
#pragma unroll
      for (int i = 0; i < E::N; ++i) {
        const int j = v * E::N + i - r.shift;
        if (j < 0 || j >= V) {
          if (E::SIZE == 4) raw[k][i] = E::NINF;
          else raw[k][i / 2] = i % 2 ? (raw[k][i / 2] & 0xffffu) | E::NINF << 16
                                     : (raw[k][i / 2] & 0xffff0000u) | E::NINF;
        }
      }
  }
}

// e^((x - m) / T) takes c = RN(m k) and one multiply-add an element; what that rounding changed, 2^fix, is
// taken back once. Where it is not small (or m infinite), and for NaN, m is subtracted first.
// k itself is rounded: every argument is off by the same share of itself, 1.3e-8 at T = 1 and at most 2^-24 (6e-8), and a usual
// row's sum by some 7e-8, one step of the float32 that it is given in. An argument's own rounding is up to 2^-24 of it too. k's
// rest as a second multiply-add was measured: 617 x 32003 f16 24.2 -> 25.8 us, 4096 x 151936 498 -> 501, 2048 float32 516 -> 519,
// and the errors of e^-80 and of what hangs on it the same within the roundings (2 to 4e-6).
struct Ref {
  float m, c, fix;
  bool far;
};
__device__ __forceinline__ Ref ref_of(float m, float k) {
  Ref r;
  r.m = m == -__builtin_inff() ? 0.f : m;
  r.c = r.m * k;
  r.far = !(fabsf(r.c) <= 16384.f);
  r.fix = r.far ? 0.f : -fmaf(r.m, k, -r.c);
  return r;
}

// Adds a thread's chunk to (m, s).
template <int DT, int CV>
__device__ __forceinline__ void add(const v4u (&raw)[CV], float k, float& m, float& s) {
  const float top = fmaxf(m, Max<DT, CV>::of(raw));
  const Ref r = ref_of(top, k);
  float t = 0.f;
  if (!__ballot(r.far)) {
#pragma unroll
    for (int i = 0; i < CV; ++i)
#pragma unroll
      for (int e = 0; e < Elem<DT>::N; ++e)
        t += __builtin_amdgcn_exp2f(fmaf(Elem<DT>::get(raw[i], e), k, -r.c));
    t *= __builtin_amdgcn_exp2f(r.fix);
  } else {
#pragma unroll
    for (int i = 0; i < CV; ++i)
#pragma unroll
      for (int e = 0; e < Elem<DT>::N; ++e)
        t += __builtin_amdgcn_exp2f((Elem<DT>::get(raw[i], e) - r.m) * k);
  }
  s = (m == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f((m - r.m) * k)) + t;
  m = top;
}

// (m, s) of two: order matters to no bit but the last
__device__ __forceinline__ Part join(Part a, float m, float k) {
  a.s = a.m == -__builtin_inff() ? a.s : a.s * __builtin_amdgcn_exp2f((a.m - m) * k);
  return {m, a.s};
}

// The sum over a row's vectors [v0, v1), of all threads: the same in each of them. raw: the first chunk. The last
// one is left in it.
template <int DT, class S>
__device__ __forceinline__ Part sum_of(const Args& a, const Row& r, Listed& l, uint32_t owns, int v0,
                                       int v1, v4u (&raw)[S::CV]) {
  const int lane = lane_id(), w = uniform((int)threadIdx.x / WAVE);
  float m = -__builtin_inff(), s = 0.f;
  int next = next_of<DT>(l, owns, r.shift, v0);
  for (int base = v0; base < v1; base += S::CHUNK) {
    v4u x[S::CV];
#pragma unroll
    for (int i = 0; i < S::CV; ++i) x[i] = raw[i];
    if (base + S::CHUNK < v1) load<DT, S, false>(raw, r, base + S::CHUNK);
    if (base == 0 || base + S::CHUNK >= r.nvec) trim<DT, S>(x, r, a.V, base);
    if (next < base + S::CHUNK) {
      replace<DT, S>(x, l, owns, r.shift, base, [](int) { return Elem<DT>::NINF; });
      next = next_of<DT>(l, owns, r.shift, base + S::CHUNK);
    }
    add<DT>(x, a.k, m, s);
  }
  const float wm = wave_max(m);
  s = wave_add(join({m, s}, wm, a.k).s);
  if (lane == 0) {
    l.m[w] = wm;
    l.s[w] = s;
  }
  __syncthreads();
  float top = l.m[0], sum = 0.f;
#pragma unroll
  for (int i = 1; i < S::NW; ++i) top = fmaxf(top, l.m[i]);
#pragma unroll
  for (int i = 0; i < S::NW; ++i) sum += join({l.m[i], l.s[i]}, top, a.k).s;
  return {top, sum};
}

// The loss and its coefficients from the unlisted logits' part, by the first wave; the listed ones' gradients go to LDS.
__device__ __forceinline__ Coef policy(const Args& a, Part u, float x, int row, float weight,
                                       bool bad, Listed& l, bool store) {
  const float inf = __builtin_inff(), nan = __builtin_nanf("");
  x = lane_f(x, 0);                        // -inf where the token is bad
  const float m = fmaxf(u.m, x);
  bad |= u.s != u.s || x != x || m == inf;
  const bool none = m == -inf;
  const float rest = join(u, m, a.k).s, e = none ? 0.f : __builtin_amdgcn_exp2f((x - m) * a.k);
  const float z = rest + e;
  float lp = x == m ? -log1pf(rest) : (x - m) * a.inv_t - logf(z);
  if (none) lp = -inf;
  if (bad) lp = nan;
  const float ratio = expf(lp - a.old[row]), adv = a.adv[row];
  const float held = ratio < a.lo ? a.lo : ratio > a.hi ? a.hi : ratio;
  const float gain = ratio * adv, bound = held * adv;
  const bool take = gain <= bound;
  float loss = -(take ? gain : bound), g = take ? -gain : 0.f;
  if (a.ref) {
    const float d = a.ref[row] - lp, over = expm1f(d);
    loss += a.kl * (over == inf ? inf : over - d);
    g -= a.kl * over;
  }
  if (loss != loss) g = nan;
  const float f = none && !bad ? 0.f : weight * g * a.inv_t / z;
  if (store && a.loss && threadIdx.x == 0) {
    a.loss[row] = weight * loss;
    a.logprob[row] = lp;
  }
  if (threadIdx.x == 0) l.grad[0] = f * rest;
  const float down = u.m == -inf ? 0.f : __builtin_amdgcn_exp2f((u.m - m) * a.k);
  return {u.m, -f * down};
}

__device__ __forceinline__ Coef distill(const Args& a, Part u, float x, float v, int id, int row,
                                        float weight, bool bad, Listed& l, bool store) {
  const float inf = __builtin_inff(), nan = __builtin_nanf("");
  const int lane = lane_id();
  const bool in = id >= 0;                 // (lanes that list a token; x and v -inf in the others)
  float ln_q, q, left, total;
  bool first = in;
  bad |= __ballot(in && x != x) || u.s != u.s;
  // the teacher's probabilities
  const float vm = wave_max(in ? v : -inf);
  if (a.rest) {
    ln_q = v;
    q = in ? expf(v) : 0.f;
    const uint64_t at = __ballot(in && v == vm);
    const bool lead = at && lane == __ffsll((unsigned long long)at) - 1;
    const float sum = wave_add(q), others = wave_add(lead ? 0.f : q);
    // what they leave: the leader's own 1 - q is small where it is nearly certain
    left = (at ? -expm1f(vm) : 1.f) - others;
    left = left > 0.f ? left : left == left ? 0.f : left;
    // what the loss counts: 1, or the listed ones' sum where it is over 1 by more than a teacher's rounded values explain,
    // or where no token is left for the rest, whose term the loss then lacks
    total = sum > 1.f + 0x1p-16f || u.s == 0.f ? sum : sum == sum ? 1.f : sum;
    if (!__ballot(in)) left = total = 0.f;
  } else {
    const float d = (v - vm) * a.inv_t;
    q = in && vm > -inf ? expf(d) : 0.f;
    const float sum = wave_add(q);
    ln_q = d - logf(sum);
    q = sum > 0.f ? q / sum : sum == sum ? 0.f : sum;
    left = 0.f;
    total = wave_add(q) > 0.f ? 1.f : 0.f;
  }
  // an id listed twice has its probabilities' sum and counts once
  float own = q;
  const uint64_t alike = match_any(id, in, 19);        // (MAX_V < 2^19)
  if (__ballot(alike & (alike - 1))) {
    first = in && __ffsll((unsigned long long)alike) - 1 == lane;
    for (int j = 0; j < a.top; ++j) own += alike >> j & 1 && j != lane ? lane_f(q, j) : 0.f;
  }
  const float xm = wave_max(in ? x : -inf), m = fmaxf(u.m, xm);
  bad |= m == inf || __ballot(in && !(q < inf));
  const bool none = m == -inf;
  const float e = none || !in ? 0.f : __builtin_amdgcn_exp2f((x - m) * a.k);
  const float rest = join(u, m, a.k).s;
  const uint64_t tops = __ballot(first && x == m);
  const bool lead = tops && lane == __ffsll((unsigned long long)tops) - 1;
  const float others = rest + wave_add(first && !lead ? e : 0.f);
  const float z = tops ? 1.f + others : others, ln_z = tops ? log1pf(others) : logf(others);
  float loss = wave_add(in && q > 0.f ? q * (ln_q - ((x - m) * a.inv_t - ln_z)) : 0.f);
  if (left > 0.f && u.s > 0.f)
    loss += left * (logf(left) - ((u.m - m) * a.inv_t + logf(u.s) - ln_z));
  if (none) loss = wave_add(q) > 0.f ? inf : 0.f;
  if (bad) loss = nan;
  if (store && a.loss && threadIdx.x == 0) a.loss[row] = weight * loss;
  const float w = (bad ? nan : weight) * a.inv_t;
  if (threadIdx.x < (unsigned)a.top) l.grad[lane] = none ? 0.f * w : w * (total * e / z - own);
  // relative to the unlisted logits' own maximum: their share of z may be below the smallest float
  const float down = u.m == -inf ? 0.f : __builtin_amdgcn_exp2f((u.m - m) * a.k);
  const float f = none ? 0.f : total * down / z - (u.s > 0.f ? left / u.s : 0.f);
  return {u.m, w * f};
}

// Two floats in 16 bits each.
template <int DT>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  return DT == 0 ? f32x2_to_bf16(a, b) : bits_of<DT>(a) | bits_of<DT>(b) << 16;
}

// The gradient of a row's vectors [v0, v1), the last chunk first: the cache has it still. raw: that chunk.
template <int DT, class S>
__device__ __forceinline__ void grad_of(const Args& a, const Row& r, const Listed& l, uint32_t owns,
                                        int row, int v0, int v1, Coef c, v4u (&raw)[S::CV]) {
  typedef Elem<DT> E;
  uint8_t* out = a.grad + (size_t)row * a.ldg * E::SIZE - r.shift * E::SIZE;
  const Ref ref = ref_of(c.m, a.k);
  const float f = c.f * __builtin_amdgcn_exp2f(ref.fix);
  for (int base = v0 + (v1 - v0 - 1) / S::CHUNK * S::CHUNK; base >= v0 && v0 < v1; base -= S::CHUNK) {
    v4u x[S::CV];
#pragma unroll
    for (int i = 0; i < S::CV; ++i) x[i] = raw[i];
    if (base > v0) load<DT, S, true>(raw, r, base - S::CHUNK);
#pragma unroll
    for (int i = 0; i < S::CV; ++i) {
      float g[E::N];
      if (!ref.far)
#pragma unroll
        for (int e = 0; e < E::N; ++e)
          g[e] = f * __builtin_amdgcn_exp2f(fmaf(E::get(x[i], e), a.k, -ref.c));
      else
#pragma unroll
        for (int e = 0; e < E::N; ++e)
          g[e] = f * __builtin_amdgcn_exp2f((E::get(x[i], e) - ref.m) * a.k);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[i][j] = E::SIZE == 4 ? __float_as_uint(g[j]) : pack<DT>(g[2 * j % E::N], g[(2 * j + 1) % E::N]);
    }
    if (owns) replace<DT, S>(x, l, owns, r.shift, base, [&](int j) { return bits_of<DT>(l.grad[j]); });
#pragma unroll
    for (int k = 0; k < S::CV; ++k) {
      const int v = base + k * S::NT + (int)threadIdx.x;
      uint8_t* to = out + (long long)v * 16;
      if ((v == 0 && r.shift) || v == r.nvec - 1) {
#pragma unroll
        for (int i = 0; i < E::N; ++i) {
          const int j = v * E::N + i - r.shift;
          if (j < 0 || j >= a.V) continue;
          if (E::SIZE == 4) ((uint32_t*)to)[i] = x[k][i];
          else ((uint16_t*)to)[i] = (uint16_t)(x[k][i / 2] >> i % 2 * 16);
        }
      } else if (v < r.nvec) {
        __builtin_nontemporal_store(x[k], (v4ua*)to);
      }
    }
  }
}

template <int DT, class S>
__device__ __forceinline__ void clear(const Args& a, const Row& r, int row, int v0, int v1) {
  typedef Elem<DT> E;
  uint8_t* out = a.grad + (size_t)row * a.ldg * E::SIZE - r.shift * E::SIZE;
  for (int v = v0 + (int)threadIdx.x; v < min(v1, r.nvec); v += S::NT) {
    uint8_t* to = out + (long long)v * 16;
    if ((v == 0 && r.shift) || v == r.nvec - 1) {
      for (int i = 0; i < E::N; ++i) {
        const int j = v * E::N + i - r.shift;
        if (j < 0 || j >= a.V) continue;
        if (E::SIZE == 4) ((uint32_t*)to)[i] = 0;
        else ((uint16_t*)to)[i] = 0;
      }
    } else {
      const v4u z = {};
      __builtin_memcpy(to, &z, 16);
    }
  }
}

// A row whose gradient stays as it is. (A float32 gradient is multiplied: by is for 16 bits.)
template <int DT>
__device__ __forceinline__ bool done(const Args& a, int row) {
  return Elem<DT>::SIZE == 2 && a.by && a.by[row * a.step] == 1.f;
}

// What the threads of a row know of what it lists.
struct Own {
  float x, v, weight;                      // of the lane's listed token
  int id;
  bool bad, skip;
};
template <int DT, int OP, class S>
__device__ __forceinline__ Own listed(const Args& a, const Row& r, int row, const float* xs, Listed& l) {
  const int lane = lane_id(), tid = (int)threadIdx.x, top = OP == POLICY ? 1 : a.top;
  Own o = {-__builtin_inff(), -__builtin_inff(), a.weight ? a.weight[row] : 1.f, -1, false, false};
  long long id = -1;
  if (lane < top) id = OP == POLICY ? token_of(a.ids, a.wide, row)
                                    : (long long)((const int*)a.ids)[(size_t)row * top + lane];
  o.bad = __ballot(id >= a.V);
  o.skip = o.weight == 0.f || (OP == POLICY && __ballot(id >= 0) == 0);
  if (Elem<DT>::SIZE == 2 && a.by) {       // (before the rounding to the logits' type)
    o.weight *= a.by[row * a.step];
    o.skip |= o.weight == 0.f;
  }
  o.id = id >= 0 && id < a.V ? (int)id : -1;
  float v = 0.f;
  if (OP == DISTILL && lane < top) v = a.vals[(size_t)row * top + lane];
  if (o.id >= 0) {
    o.x = xs ? xs[(size_t)row * top + lane] : load_one<DT>(r.p, o.id);
    if (OP == DISTILL) o.v = v;
  }
  if (tid < MAX_TOP) l.id[tid] = tid < top ? o.id : -1;
  l.owns[tid] = 0;
  __syncthreads();
  if (tid < WAVE && o.id >= 0) atomicOr(&l.owns[(o.id + r.shift) / Elem<DT>::N % S::NT], 1u << lane);
  __syncthreads();
  return o;
}

template <int OP>
__device__ __forceinline__ Coef coef(const Args& a, Part u, const Own& o, int row, Listed& l,
                                     bool store) {
  // (one wave for all: it is a thousand instructions)
  if (threadIdx.x < WAVE) {
    const Coef c = OP == POLICY ? policy(a, u, o.x, row, o.weight, o.bad, l, store)
                                : distill(a, u, o.x, o.v, o.id, row, o.weight, o.bad, l, store);
    if (threadIdx.x == 0) l.coef = c;
  }
  __syncthreads();
  return l.coef;
}

// A workgroup a row: its sum, its loss and, with GRAD, its gradient.
template <int DT, int OP, bool GRAD, class S>
__global__ __launch_bounds__(S::NT, S::NT == Wide::NT ? 8 : 1) void row_k(Args a) {
  __shared__ Listed l;
  const int row = (int)blockIdx.x;
  if (done<DT>(a, row)) return;
  const Row r = row_of<DT>(a, row);
  v4u raw[S::CV];
  load<DT, S, !GRAD>(raw, r, 0);
  const Own o = listed<DT, OP, S>(a, r, row, nullptr, l);
  if (o.skip) {
    if (a.loss && threadIdx.x == 0) {
      a.loss[row] = 0.f;
      if (OP == POLICY) a.logprob[row] = 0.f;
    }
    if (GRAD) clear<DT, S>(a, r, row, 0, r.nvec);
    return;
  }
  const uint32_t owns = l.owns[threadIdx.x];
  const Part u = sum_of<DT, S>(a, r, l, owns, 0, r.nvec, raw);
  const Coef c = coef<OP>(a, u, o, row, l, true);
  if (GRAD) grad_of<DT, S>(a, r, l, owns, row, 0, r.nvec, c, raw);
}

// Few rows: a workgroup for each of a row's segments, first their sums, then a launch that joins them and
// writes the loss and the segments' gradients. Bound by two launches' chains of loads: 8 bf16 rows of 151936 4.2 + 4.5 us,
// 20 with 20 listed tokens 5.0 + 6.8.
template <int DT, int OP, class S>
__global__ __launch_bounds__(S::NT) void segment_k(Args a, Part* __restrict__ parts,
                                                   float* __restrict__ xs) {
  __shared__ Listed l;
  const int row = (int)(blockIdx.x / (unsigned)a.nseg), seg = (int)(blockIdx.x % (unsigned)a.nseg);
  if (done<DT>(a, row)) return;
  const Row r = row_of<DT>(a, row);
  const int len = ((r.nvec + S::CHUNK - 1) / S::CHUNK + a.nseg - 1) / a.nseg * S::CHUNK;
  const int v0 = min(seg * len, r.nvec), v1 = min(v0 + len, r.nvec);
  v4u raw[S::CV];
  load<DT, S, false>(raw, r, v0);
  const Own o = listed<DT, OP, S>(a, r, row, nullptr, l);
  if (o.skip) return;
  // (the gradient may take the logits' place while other segments still ask for these)
  if (seg == 0 && (int)threadIdx.x < a.top) xs[(size_t)row * a.top + threadIdx.x] = o.x;
  const Part u = sum_of<DT, S>(a, r, l, l.owns[threadIdx.x], v0, v1, raw);
  if (threadIdx.x == 0) parts[blockIdx.x] = u;
}

template <int DT, int OP, bool GRAD, class S>
__global__ __launch_bounds__(S::NT) void finish_k(Args a, const Part* __restrict__ parts,
                                                  const float* __restrict__ xs) {
  __shared__ Listed l;
  const unsigned n = GRAD ? (unsigned)a.nseg : 1u;
  const int row = (int)(blockIdx.x / n), seg = (int)(blockIdx.x % n), lane = lane_id();
  if (done<DT>(a, row)) return;
  const Row r = row_of<DT>(a, row);
  const int len = ((r.nvec + S::CHUNK - 1) / S::CHUNK + a.nseg - 1) / a.nseg * S::CHUNK;
  const int v0 = min(seg * len, r.nvec), v1 = min(v0 + len, r.nvec);
  v4u raw[S::CV];
  if (GRAD && v0 < v1) load<DT, S, true>(raw, r, v0 + (v1 - v0 - 1) / S::CHUNK * S::CHUNK);
  Part u = {-__builtin_inff(), 0.f};
  if (lane < a.nseg) u = parts[(size_t)row * a.nseg + lane];
  const Own o = listed<DT, OP, S>(a, r, row, xs, l);
  if (o.skip) {
    if (a.loss && seg == 0 && threadIdx.x == 0) {
      a.loss[row] = 0.f;
      if (OP == POLICY) a.logprob[row] = 0.f;
    }
    if (GRAD) clear<DT, S>(a, r, row, v0, v1);
    return;
  }
  const float m = wave_max(u.m);
  u = {m, wave_add(join(u, m, a.k).s)};
  const Coef c = coef<OP>(a, u, o, row, l, seg == 0);
  if (GRAD) grad_of<DT, S>(a, r, l, l.owns[threadIdx.x], row, v0, v1, c, raw);
}

constexpr int SCALE_NT = 512;

// Rows of a gradient by a factor each; those whose factor is 1 are left as they are. (2048 float32 rows of 151936 480 us, by
// 1 6)
template <int DT>
__global__ __launch_bounds__(SCALE_NT) void scale_k(Args a, const float* __restrict__ by, long long step) {
  typedef Elem<DT> E;
  const int row = (int)(blockIdx.x / (unsigned)a.nseg), seg = (int)(blockIdx.x % (unsigned)a.nseg);
  const float f = by[row * step];
  if (f == 1.f) return;
  const Row r = row_of<DT>(a, row);
  for (int v = seg * SCALE_NT + (int)threadIdx.x; v < r.nvec; v += a.nseg * SCALE_NT) {
    uint8_t* to = (uint8_t*)(r.pv + v);
    if ((v == 0 && r.shift) || v == r.nvec - 1) {      // (the neighbours' elements are theirs)
      for (int i = 0; i < E::N; ++i) {
        const int j = v * E::N + i - r.shift;
        if (j < 0 || j >= a.V) continue;
        const uint32_t b = bits_of<DT>(load_one<DT>(r.p, j) * f);
        if (E::SIZE == 4) ((uint32_t*)to)[i] = b;
        else ((uint16_t*)to)[i] = (uint16_t)b;
      }
    } else {
      v4u x = r.pv[v];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = E::SIZE == 4 ? bits_of<DT>(E::get(x, j) * f)
                            : pack<DT>(E::get(x, 2 * j % E::N) * f, E::get(x, (2 * j + 1) % E::N) * f);
      *(v4u*)to = x;
    }
  }
}

// Vectors of a row, but for what its address adds.
static long long vectors(int dtype, int V) { return (long long)V * (dtype == 1 ? 4 : 2) / 16 + 1; }

// Segments of a row: one where the rows alone fill the chip, or a workgroup holds a row in its registers. (bf16, policy, us:
// 16 rows of 151936 8.5 in segments, 26 whole; 128 24.4 and 30.5; 192 33.8 and 33.3; 255 42.3 and 39.4; 8 of 15000 7.2 and 6.5
// and a launch less, 150 of them 9.1 and 7.3)
static int segments(int dtype, int R, int V) {
  if (R >= 192 || vectors(dtype, V) <= Usual::CHUNK) return 1;
  const int n = dtype == 1 ? 4 : 8;
  const int chunks = (V + 2 * n - 2) / n / Short::CHUNK + 1, want = R ? (768 + R - 1) / R : 1;
  const int most = chunks < MAX_SEGS ? chunks : MAX_SEGS;
  return want < most ? want : most;
}

static int check(const Args& a, int dtype, long long* bytes) {
  if (dtype < 0 || dtype > 2 || a.R < 0 || a.V < 1 || a.V > MAX_V || a.top < 1 || a.top > MAX_TOP)
    return -1;
  const long long segs = (long long)a.R * segments(dtype, a.R, a.V);
  if (segs > UINT32_MAX / Wide::NT) return -1;         // (a launch counts its threads in 32 bits)
  *bytes = segs * (long long)sizeof(Part) + 4ll * a.R * a.top;
  return 0;
}

template <int OP>
static int launch(Args a, int dtype, void* ws, hipStream_t stream) {
  long long bytes;
  if (check(a, dtype, &bytes) || a.ld < 0 || !(a.inv_t > 0.f) || !(a.k < __builtin_inff())) return -1;
  if (a.R == 0) return 0;
  if (a.by && dtype == 1) return -1;
  if (!a.logits || !ws || !(a.by ? (const void*)a.grad : a.loss)) return -1;
  if (a.grad && a.R > 1 && a.ldg < a.V) return -1;
  if (((uintptr_t)a.logits | (uintptr_t)a.grad) % (dtype == 1 ? 4 : 2) || (uintptr_t)ws % 8) return -4;
  a.nseg = segments(dtype, a.R, a.V);
  Part* parts = (Part*)ws;
  float* xs = (float*)(parts + (size_t)a.R * a.nseg);
  const dim3 rows((unsigned)a.R), all((unsigned)(a.R * a.nseg));
  // The second read comes from the memory-side cache as long as the rows in flight fit there (256 MB): four
  // workgroups a CU of rows up to 256 KB. Of longer ones two: float32's with twice the threads, 16-bit ones' kept to
  // two by LDS that they do not use, as more threads a row leave the vector unit idle between its passes.
  const long long vecs = vectors(dtype, a.V);
  const bool longer = (long long)a.V * (dtype == 1 ? 4 : 2) > 256 << 10;
#define RLU_ROW(DT, GRAD, S, LDS) \
  hipLaunchKernelGGL((row_k<DT, OP, GRAD, S>), rows, dim3(S::NT), LDS, stream, a)
#define RLU_LOSS(DT)                                                                               \
  do {                                                                                             \
    if (a.nseg == 1) {                                                                             \
      if (vecs <= Small::CHUNK && a.grad) RLU_ROW(DT, true, Small, 0);                             \
      else if (vecs <= Small::CHUNK) RLU_ROW(DT, false, Small, 0);                                 \
      else if (vecs <= Medium::CHUNK && a.grad) RLU_ROW(DT, true, Medium, 0);                      \
      else if (vecs <= Medium::CHUNK) RLU_ROW(DT, false, Medium, 0);                               \
      else if (!a.grad) RLU_ROW(DT, false, Usual, 0);                                              \
      else if (!longer) RLU_ROW(DT, true, Usual, 0);                                               \
      else if (DT == 1) RLU_ROW(1, true, Wide, 0);                                                 \
      else RLU_ROW(DT, true, Usual, 70 << 10);                                                     \
    } else {                                                                                       \
      hipLaunchKernelGGL((segment_k<DT, OP, Short>), all, dim3(Short::NT), 0, stream, a, parts, xs); \
      if (a.grad)                                                                                  \
        hipLaunchKernelGGL((finish_k<DT, OP, true, Short>), all, dim3(Short::NT), 0, stream, a,    \
                           parts, xs);                                                             \
      else                                                                                         \
        hipLaunchKernelGGL((finish_k<DT, OP, false, Short>), rows, dim3(Short::NT), 0, stream, a,  \
                           parts, xs);                                                             \
    }                                                                                              \
  } while (0)
  if (dtype == 0) RLU_LOSS(0);
  else if (dtype == 1) RLU_LOSS(1);
  else RLU_LOSS(2);
#undef RLU_LOSS
#undef RLU_ROW
  return (int)hipGetLastError();
}

}  // namespace loss
}  // namespace rlu

extern "C" int rlu_loss_workspace(int dtype, int R, int V, int top, long long* bytes) {
  rlu::loss::Args a = {};
  a.top = top;
  a.R = R;
  a.V = V;
  return bytes ? rlu::loss::check(a, dtype, bytes) : -1;
}

static int policy_args(rlu::loss::Args& a, const void* logits, long long ld, int R, int V, const void* tokens, int wide,
                       const float* old_logprobs, const float* advantages, const float* ref_logprobs,
                       const float* weight, float clip_low, float clip_high, float kl, float temperature) {
  if ((wide != 0 && wide != 1) || !(clip_low >= 0.f && clip_low <= 1.f) || !(clip_high >= 0.f)) return -1;
  if (!(temperature > 0.f) || !(kl >= 0.f && kl < __builtin_inff())) return -1;
  if (R > 0 && (!tokens || !old_logprobs || !advantages)) return -1;
  a.logits = (const uint8_t*)logits;
  a.ld = ld;
  a.R = R;
  a.V = V;
  a.ids = tokens;
  a.wide = wide;
  a.top = 1;
  a.old = old_logprobs;
  a.adv = advantages;
  a.ref = kl != 0.f ? ref_logprobs : nullptr;
  a.weight = weight;
  a.inv_t = 1.f / temperature;
  a.k = (float)(rlu::loss::LOG2_E / temperature);
  a.lo = 1.f - clip_low;
  a.hi = 1.f + clip_high;
  a.kl = kl;
  return 0;
}

extern "C" int rlu_policy_loss(const void* logits, int dtype, long long ld, int R, int V,
                               const void* tokens, int wide, const float* old_logprobs,
                               const float* advantages, const float* ref_logprobs,
                               const float* weight, float clip_low, float clip_high, float kl,
                               float temperature, float* loss, float* logprob, void* grad,
                               long long ldg, void* ws, hipStream_t stream) {
  rlu::loss::Args a = {};
  if (policy_args(a, logits, ld, R, V, tokens, wide, old_logprobs, advantages, ref_logprobs, weight, clip_low, clip_high,
                  kl, temperature) || (R > 0 && !logprob))
    return -1;
  a.loss = loss;
  a.logprob = logprob;
  a.grad = (uint8_t*)grad;
  a.ldg = ldg;
  return rlu::loss::launch<rlu::loss::POLICY>(a, dtype, ws, stream);
}

extern "C" int rlu_policy_grad_by(const void* logits, int dtype, long long ld, int R, int V, const void* tokens,
                                  int wide, const float* old_logprobs, const float* advantages,
                                  const float* ref_logprobs, const float* weight, float clip_low,
                                  float clip_high, float kl, float temperature, const float* by,
                                  long long step, void* grad, long long ldg, void* ws, hipStream_t stream) {
  rlu::loss::Args a = {};
  if (policy_args(a, logits, ld, R, V, tokens, wide, old_logprobs, advantages, ref_logprobs, weight, clip_low, clip_high,
                  kl, temperature) || (R > 0 && !by))
    return -1;
  a.grad = (uint8_t*)grad;
  a.ldg = ldg;
  a.by = by;
  a.step = step;
  return rlu::loss::launch<rlu::loss::POLICY>(a, dtype, ws, stream);
}

static int distill_args(rlu::loss::Args& a, const void* logits, long long ld, int R, int V, const int* top_ids,
                        const float* top_logprobs, int top, int rest, const float* weight, float temperature) {
  if ((rest != 0 && rest != 1) || !(temperature > 0.f)) return -1;
  if (R > 0 && (!top_ids || !top_logprobs)) return -1;
  a.logits = (const uint8_t*)logits;
  a.ld = ld;
  a.R = R;
  a.V = V;
  a.ids = top_ids;
  a.top = top;
  a.vals = top_logprobs;
  a.rest = rest;
  a.weight = weight;
  a.inv_t = 1.f / temperature;
  a.k = (float)(rlu::loss::LOG2_E / temperature);
  return 0;
}

extern "C" int rlu_distill_top(const void* logits, int dtype, long long ld, int R, int V,
                               const int* top_ids, const float* top_logprobs, int top, int rest,
                               const float* weight, float temperature, float* loss, void* grad,
                               long long ldg, void* ws, hipStream_t stream) {
  rlu::loss::Args a = {};
  if (distill_args(a, logits, ld, R, V, top_ids, top_logprobs, top, rest, weight, temperature)) return -1;
  a.loss = loss;
  a.grad = (uint8_t*)grad;
  a.ldg = ldg;
  return rlu::loss::launch<rlu::loss::DISTILL>(a, dtype, ws, stream);
}

extern "C" int rlu_distill_top_grad_by(const void* logits, int dtype, long long ld, int R, int V, const int* top_ids,
                                       const float* top_logprobs, int top, int rest, const float* weight,
                                       float temperature, const float* by, long long step, void* grad,
                                       long long ldg, void* ws, hipStream_t stream) {
  rlu::loss::Args a = {};
  if (distill_args(a, logits, ld, R, V, top_ids, top_logprobs, top, rest, weight, temperature) || (R > 0 && !by))
    return -1;
  a.grad = (uint8_t*)grad;
  a.ldg = ldg;
  a.by = by;
  a.step = step;
  return rlu::loss::launch<rlu::loss::DISTILL>(a, dtype, ws, stream);
}

extern "C" int rlu_scale_rows(void* x, int dtype, long long ld, int R, int V, const float* by,
                              long long step, hipStream_t stream) {
  using namespace rlu::loss;
  if (dtype < 0 || dtype > 2 || R < 0 || V < 1 || V > MAX_V || (R > 1 && ld < V)) return -1;
  if (R == 0) return 0;
  if (!x || !by) return -1;
  if ((uintptr_t)x % (dtype == 1 ? 4 : 2)) return -4;
  Args a = {};
  a.logits = (const uint8_t*)x;
  a.ld = ld;
  a.R = R;
  a.V = V;
  a.nseg = (V + SCALE_NT * 64 - 1) / (SCALE_NT * 64);              // (8 to 16 vectors a thread)
  if ((long long)R * a.nseg > UINT32_MAX / SCALE_NT) return -1;
  const dim3 grid((unsigned)(R * a.nseg));
  if (dtype == 0) hipLaunchKernelGGL((scale_k<0>), grid, dim3(SCALE_NT), 0, stream, a, by, step);
  else if (dtype == 1) hipLaunchKernelGGL((scale_k<1>), grid, dim3(SCALE_NT), 0, stream, a, by, step);
  else hipLaunchKernelGGL((scale_k<2>), grid, dim3(SCALE_NT), 0, stream, a, by, step);
  return (int)hipGetLastError();
}
