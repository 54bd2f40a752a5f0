// Log probabilities of given tokens, with rank, entropy and the n largest alternatives, in one read of
// the logits. With m = max x, Z = sum e^(x - m):
//   logprob = x_t - m - ln Z, entropy = ln Z - sum (x - m) e^(x - m) / Z,
//   rank = 1 + #{x > x_t} + #{j < t: x_j = x_t}, alternatives by value, the lowest index first.
//
// Bound: the read, 1.24 GB at 4096 x 151936 bf16 or 2048 x 151936 f32. float32 takes 187 + 5 us of it (6.6
// TB/s; a bare read 7.0). In 16 bits there are twice the elements and the vector unit has no cycle left, either:
// 195 - 210 us in a row of calls, up to 260 in the first milliseconds after other work; with 20 alternatives it
// is the limit, 240 - 265. An element is an unpacking, a multiply-add, an exponential (as long as four others),
// an add and a multiply-add, half an operation of the maximum and for the rank a comparison, 9.5 in all. Where
// the token is among the highest the comparisons are left out: 3%.
//
//   * A row is cut into segments of 32 KB, a workgroup each, that stay in registers between the maximum and
//     the sums: no running rescaling, and eight workgroups' loads in flight a CU (52 VGPRs; with alternatives 67,
//     and seven). Shorter ones where there would be under 256 (32 / 16 / 8 KB: 20 rows with 20 alternatives
//     14.1 / 13.9 / 15.0 us, one row without 7.7 / 6.4 / 6.1). A wave a row then joins them, 4 - 8 us, nearly all of it the chain of its steps.
//   * 16-bit logits are unpacked again for each pass and their maximum is taken packed: held unpacked they
//     took 256 VGPRs, and 4096 rows with 20 alternatives 1589 us, then 423.
//   * The maximum's own term is left out of Z: in a nearly certain row 1 + 1e-9 is 1, and entropy and the
//     likeliest token's log probability would be 0. Its thread's elements are summed again by its wave, an
//     element a lane (by a second pass of all, where Z came near 1: 230 us where this takes 201).
//   * The alternatives of a segment are its elements at or above the n-th largest of the maxima of 64 groups
//     of four threads, a little over n of them (of all 256 threads: 21 instead of 24 where n is 20, and four
//     times the comparisons, 268 us for 265; of each wave's own 64: three times as many). They are looked for
//     among the vectors of the threads that have any, a lane a vector, and there a lane an element (a lane an
//     element throughout: 278 for 265). Lists of fixed length hold them.
//   * Where a wave has more candidates than its list holds, the segment is read again once for each alternative.
//     That happens to runs of equal logits, to segments masked with a finite value of which fewer than n groups
//     keep anything else, and to float32 rows whose spread is lost in 16 bits (100 +- 0.1). 256 x 151936, 20 / 5 / 1
//     alternatives: 800 - 865 / 255 / 90 - 103 us, masked with -inf instead 35 - 40 us.
#include <float.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "logits.h"
#include "rlu.h"
#include "wave.h"

namespace rlu {
namespace lp {

constexpr int NT = 256, NW = NT / WAVE;    // threads and waves of a segment's workgroup
constexpr int MAX_TOP = 32, MAX_V = 500000;
constexpr int MAX_SEGS = WAVE;             // a row's segments, one to a lane of the joining wave
constexpr int CAP = 256;                   // candidates a wave lists
constexpr double LN2 = 0.693147180559945309;

// What a segment leaves of a row: its maximum, sum e^(x - m) - 1 (the maximum's own 1 left out: a nearly
// certain row's small terms would be lost beside it), sum log2(e^(x - m)) e^(x - m), and how many of its logits
// come before the token's. A segment of nothing: -inf, -1, 0.
struct Part {
  float m, rest, t;
  int before;
};

// unsigned keys in the order of the floats (the two zeros one), and back
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : 0xffffffffu));
}

// The compiler forgets what it unpacked: unpacking again costs one instruction an element, keeping the
// floats 64 registers.
template <int CV>
__device__ __forceinline__ void forget(v4u (&raw)[CV]) {
#pragma unroll
  for (int k = 0; k < CV; ++k) asm volatile("" : "+v"(raw[k]));
}

// log2(e^(x - m)) and its sums take c = RN(m log2 e), one multiply-add an element: with the same c in all
// of them its rounding is undone at the end. Where that rounding is not small (|m| past 4096, 2^-11; a row at
// the type's lowest value overflows there) base = m is taken off first.
struct Ref {
  float base, c;
};
__device__ __forceinline__ Ref ref_of(float m) {
  const bool far = !(fabsf(m) <= 4096.f), inf = fabsf(m) == __builtin_inff();
  return far && !inf ? Ref{m, 0.f} : Ref{0.f, m == -__builtin_inff() ? 0.f : m * L2E};
}
__device__ __forceinline__ void term(float x, Ref f, float& s, float& t) {
  const float y = fmaf(x - f.base, L2E, -f.c), e = __builtin_amdgcn_exp2f(y);
  s += e;
  t = fmaf(fmaxf(y, -200.f), e, t);        // (-inf times its zero)
}

// The sums of a thread's vectors, n of them. ANY: takes -inf and far maxima. COUNT: adds the wave's elements
// above thr(k) to before.
template <int DT, int CV, bool ANY, bool COUNT, class Thr>
__device__ __forceinline__ void sums(const v4u (&raw)[CV], int n, Ref f, Thr thr, float& s,
                                     float& t, int& before) {
  s = t = 0.f;
#pragma unroll
  for (int k = 0; k < CV; ++k) {
    if (k >= n) continue;                              // (uniform)
    const float above = COUNT ? thr(k) : 0.f;
#pragma unroll
    for (int i = 0; i < Elem<DT>::N; ++i) {
      const float x = Elem<DT>::get(raw[k], i);
      if (COUNT) before += __popcll(__ballot(x > above));
      if (ANY) {
        term(x, f, s, t);
      } else {
        const float y = fmaf(x, L2E, -f.c), e = __builtin_amdgcn_exp2f(y);
        s += e;
        t = fmaf(y, e, t);
      }
    }
  }
}

// One segment of one row: NT threads hold its CV * NT vectors of 16 bytes.
template <int DT, int CV, bool TOP>
__global__ __launch_bounds__(NT) void segment_k(const uint8_t* __restrict__ logits, long long ld,
                                                int V, int nseg, const void* __restrict__ tokens,
                                                int wide, int top, Part* __restrict__ parts,
                                                uint64_t* __restrict__ lists) {
  typedef Elem<DT> E;
  __shared__ float rtm[NT], rs[NW], rt[NW], rfrom;
  __shared__ int rbefore[NW], rcount[NW];
  __shared__ v4u one[CV];
  __shared__ uint64_t list[TOP ? NW : 1][TOP ? CAP : 1], rkey[NW];
  constexpr int BATCH = WAVE / CV;         // threads a wave lists from at a time
  __shared__ v4u near[TOP ? NW : 1][TOP ? WAVE : 1];
  __shared__ int near_v[TOP ? NW : 1][TOP ? BATCH : 1], hit[TOP ? NW : 1][TOP ? WAVE : 1];
  const int lane = lane_id(), tid = (int)threadIdx.x, w = uniform(tid / WAVE);
  const int row = (int)(blockIdx.x / (unsigned)nseg), seg = (int)(blockIdx.x % (unsigned)nseg);
  const uint8_t* p = logits + (size_t)row * ld * E::SIZE;
  // vectors from the aligned address at or below the row's start on; index = v N + i - shift
  const int shift = (int)((uintptr_t)p % 16) / E::SIZE;
  const v4u* pv = reinterpret_cast<const v4u*>(p - shift * E::SIZE);
  const int nvec = (shift + V + E::N - 1) / E::N, v0 = seg * CV * NT;
  v4u raw[CV];
#pragma unroll
  for (int k = 0; k < CV; ++k) {
    const int v = v0 + k * NT + tid;
    if (v < nvec) {
      raw[k] = __builtin_nontemporal_load(pv + v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[k][j] = E::SIZE == 4 ? E::NINF : E::NINF * 0x10001u;
    }
  }
  auto entry = [&](float x, int j) {                   // by value, then the lowest index
    return (uint64_t)key_of(x) << 32 | ~(uint32_t)j;
  };
  const long long tok = token_of(tokens, wide, row);
  const bool asked = tok >= 0 && tok < V;
  const float xt = asked ? load_one<DT>(p, tok) : __builtin_inff();
#pragma unroll
  for (int k = 0; k < CV; ++k) {           // elements of the neighbours in a row's end vectors
    const int v = v0 + k * NT + tid;
    if ((v == 0 && shift) || v == nvec - 1)
#pragma unroll
      for (int i = 0; i < E::N; ++i) {
        const int j = v * E::N + i - shift;
        if (j < 0 || j >= V) {
          if (E::SIZE == 4) raw[k][i] = E::NINF;
          else raw[k][i / 2] = i % 2 ? (raw[k][i / 2] & 0xffffu) | E::NINF << 16
                                     : (raw[k][i / 2] & 0xffff0000u) | E::NINF;
        }
      }
  }
  const float tm = Max<DT, CV>::of(raw);
  rtm[tid] = tm;
  __syncthreads();
  float om[NW], m;                         // the lane's threads of all waves
#pragma unroll
  for (int k = 0; k < NW; ++k) om[k] = rtm[k * WAVE + lane];
  const float gm = fmaxf(fmaxf(om[0], om[1]), fmaxf(om[2], om[3]));
  m = wave_max(gm);
  if (TOP && w == 0) {
    // a value that `top` of 64 groups of threads have an element at or above: the upper 16 bits of the
    // top-th largest of their maxima, bit by bit
    const uint32_t key = key_of(gm);
    uint32_t at = 0;
#pragma unroll
    for (int b = 15; b >= 0; --b) {
      const uint32_t c = at | 1u << b;
      if ((int)__popcll(__ballot(key >= c << 16)) >= top) at = c;
    }
    if (lane == 0) rfrom = at > 0x7fu ? of_key(at << 16) : -FLT_MAX;     // (finite ones only)
  }
  const Ref ref = ref_of(m);
  // vectors that the wave has, the token's, and the value just below its logit
  const int left = nvec - v0 - w * WAVE, n = left <= 0 ? 0 : min(CV, (left + NT - 1) / NT);
  const int tv = asked ? (int)((tok + shift) / E::N) : 0;
  const uint32_t ub = __float_as_uint(xt + 0.f);
  const float below = __uint_as_float(xt == 0.f ? 0x80000001u : xt > 0.f ? ub - 1 : ub + 1);
  const bool count = m >= xt, low = !(xt > -__builtin_inff());
  auto thr = [&](int k) __attribute__((always_inline)) {
    const int vw = v0 + k * NT + w * WAVE;             // the wave's first vector
    return vw + WAVE <= tv ? below : vw > tv ? xt : __builtin_inff();
  };
  auto none = [](int) { return 0.f; };
  float s, t;
  int before = 0;
  bool again = (n && __ballot(E::get(raw[0], 0) == -__builtin_inff())) || ref.base != 0.f;
  if (!again) {
    if (count && !low) sums<DT, CV, false, true>(raw, n, ref, thr, s, t, before);
    else sums<DT, CV, false, false>(raw, n, ref, none, s, t, before);
    again = __ballot(t != t);
  } else if (count && !low) {
#pragma unroll
    for (int k = 0; k < CV; ++k)
#pragma unroll
      for (int i = 0; i < E::N; ++i) before += __popcll(__ballot(E::get(raw[k], i) > thr(k)));
  }
  if (again) {
    forget(raw);
    sums<DT, CV, true, false>(raw, n, ref, none, s, t, before);
  }
  if (count) {                             // the vectors beside the token's, and a token at -inf
    forget(raw);
#pragma unroll
    for (int k = 0; k < CV; ++k) {
      const int vw = v0 + k * NT + w * WAVE;
      if (vw > tv || (!low && vw + WAVE <= tv)) {
        if (low)
#pragma unroll
          for (int i = 0; i < E::N; ++i) before += __popcll(__ballot(E::get(raw[k], i) > xt));
      } else {
#pragma unroll
        for (int i = 0; i < E::N; ++i) {
          const int j = (vw + lane) * E::N + i - shift;
          const float x = E::get(raw[k], i);
          before += __popcll(__ballot(x > xt || (x == xt && j >= 0 && j < (int)tok)));
        }
      }
    }
  }
  // The maximum's own 1 is left out: small terms would be lost beside it. The first thread that has it hands
  // its elements to the wave, which sums them again without the first that is equal to it.
  const uint64_t h0 = __ballot(om[0] == m), h1 = __ballot(om[1] == m), h2 = __ballot(om[2] == m);
  const int first = h0 ? 0 : h1 ? 1 : h2 ? 2 : 3;
  if (w == first && m > -__builtin_inff()) {
    const int f = __ffsll((unsigned long long)__ballot(tm == m)) - 1;
    if (lane == f) {
#pragma unroll
      for (int k = 0; k < CV; ++k) one[k] = raw[k];
      s = t = 0.f;
    }
    wave_lds_sync();
    const bool in = lane < CV * E::N;
    const float x = in ? load_one<DT>((const uint8_t*)one, lane) : 0.f;
    const uint64_t eq = __ballot(in && x == m);
    if (in && lane != __ffsll((unsigned long long)eq) - 1) term(x, ref, s, t);
  }
  s = wave_add(s);
  t = wave_add(t);
  if (lane == 0) {
    rs[w] = s;
    rt[w] = t;
    rbefore[w] = before;
  }
  __syncthreads();
  if (TOP) {
    // the elements from there on: of the threads that have any, BATCH at a time, their vectors that do
    // (a lane a vector), and of those the elements (a lane each)
    const float from = rfrom;
    forget(raw);
    uint64_t todo = __ballot(tm >= from);
    int count = 0;
    while (todo) {
      const int at = mbcnt(todo);
      const bool mine = (todo >> lane & 1) && at < BATCH;
      if (mine) {
#pragma unroll
        for (int k = 0; k < CV; ++k) near[w][at * CV + k] = raw[k];
        near_v[w][at] = v0 + tid;
      }
      wave_lds_sync();
      const int left = (int)__popcll(todo), n = left < BATCH ? left : BATCH;
      const v4u one_v[1] = {near[w][lane]};
      const bool has = lane < n * CV && Max<DT, 1>::of(one_v) >= from;
      const uint64_t hits = __ballot(has);
      const int nh = (int)__popcll(hits);
      if (has) hit[w][mbcnt(hits)] = lane;
      wave_lds_sync();
      for (int i = lane / E::N; i - lane / E::N < nh; i += WAVE / E::N) {
        const int of = hit[w][i < nh ? i : 0], e = lane % E::N;
        const float x = load_one<DT>((const uint8_t*)(near[w] + of), e);
        const bool in = i < nh && x >= from;
        const uint64_t all = __ballot(in);
        const int to = count + mbcnt(all);
        if (in && to < CAP)
          list[w][to] = entry(x, (near_v[w][of / CV] + of % CV * NT) * E::N + e - shift);
        count += (int)__popcll(all);
      }
      wave_lds_sync();
      todo &= ~__ballot(mine);
    }
    if (lane < 8 && count + lane < CAP) list[w][count + lane] = 0;      // (places are counted by 8)
    if (lane == 0) rcount[w] = count;
    __syncthreads();
  }
  s = (rs[0] + rs[1]) + (rs[2] + rs[3]);
  t = (rt[0] + rt[1]) + (rt[2] + rt[3]);
  if (tid == 0) {
    const float r = fmaf(m - ref.base, L2E, -ref.c);   // the maximum's own log2: what c's rounding left
    const float unit = __builtin_amdgcn_exp2f(-r);
    const bool some = m > -__builtin_inff();
    Part o;
    o.m = m;
    o.rest = m == __builtin_inff() ? __builtin_nanf("") : some ? s * unit : s - 1.f;
    o.t = some ? (t - r * s) * unit : 0.f;
    o.before = rbefore[0] + rbefore[1] + rbefore[2] + rbefore[3];
    parts[blockIdx.x] = o;
  }
  if (TOP) {
    uint64_t* out = lists + (size_t)blockIdx.x * top;
    int total = 0, most = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      total += rcount[k];
      most = max(most, rcount[k]);
    }
    if (most <= CAP) {                     // each candidate's place is how many come before it
      const int c1 = rcount[0], c2 = c1 + rcount[1], c3 = c2 + rcount[2];
      for (int j = tid; j < total; j += NT) {          // (mostly the first wave's alone)
        const int of = (j >= c1) + (j >= c2) + (j >= c3);
        const uint64_t key = list[of][j - (of == 0 ? 0 : of == 1 ? c1 : of == 2 ? c2 : c3)];
        int place = 0;
#pragma unroll
        for (int k = 0; k < NW; ++k)
          for (int l = 0; l < rcount[k]; l += 8)
#pragma unroll
            for (int o = 0; o < 8; ++o) place += list[k][l + o] > key;
        if (place < top) out[place] = key;
      }
      if (tid >= total && tid < top) out[tid] = 0;
    } else {                               // long runs of equal logits: one after the other
      uint64_t last = ~0ull;
      for (int n = 0; n < top; ++n) {
        uint64_t best = 0;
        if (last)
          for (int v = v0 + tid; v < min(v0 + CV * NT, nvec); v += NT)
            for (int i = 0; i < E::N; ++i) {
              const int j = v * E::N + i - shift;
              const float x = j >= 0 && j < V ? load_one<DT>(p, j) : -__builtin_inff();
              const uint64_t key = x >= -FLT_MAX ? entry(x, j) : 0;
              best = key < last && key > best ? key : best;
            }
        best = wave_reduce64(best, OpMax64());
        if (lane == 0) rkey[w] = best;
        __syncthreads();
        OpMax64 op;
        last = op(op(rkey[0], rkey[1]), op(rkey[2], rkey[3]));
        if (tid == 0) out[n] = last;
        __syncthreads();
      }
    }
  }
}

// Joins a row's segments: one wave a row. parts [R][nseg], lists [R][nseg][top] in falling order, 0 behind
// the last.
template <int DT, int K>
__global__ __launch_bounds__(WAVE) void join_k(const uint8_t* __restrict__ logits, long long ld,
                                               int V, int nseg, const void* __restrict__ tokens,
                                               int wide, int top, const Part* __restrict__ parts,
                                               const uint64_t* __restrict__ lists,
                                               float* __restrict__ logprob, int* __restrict__ rank,
                                               float* __restrict__ entropy,
                                               float* __restrict__ top_logprobs,
                                               int* __restrict__ top_ids) {
  extern __shared__ uint64_t heads[];      // [nseg][top], then WAVE chosen
  const int lane = lane_id(), row = (int)blockIdx.x;
  const float ninf = -__builtin_inff(), nan = __builtin_nanf("");
  const uint8_t* p = logits + (size_t)row * ld * Elem<DT>::SIZE;
  Part q = {ninf, -1.f, 0.f, 0};
  if (lane < nseg) q = parts[(size_t)row * nseg + lane];
  for (int i = lane; i < nseg * top; i += WAVE) heads[i] = lists[(size_t)row * nseg * top + i];
  const long long tok = token_of(tokens, wide, row);
  const float xt = tok >= 0 && tok < V ? load_one<DT>(p, tok) : 0.f;
  const float m = wave_max(q.m);
  const bool none = m == ninf;
  // the segment of the maximum keeps its rest, the others add all they have
  const uint64_t has = __ballot(q.m == m);
  const bool ref = lane == __ffsll((unsigned long long)has) - 1;
  const float d = (q.m - m) * L2E, a = __builtin_amdgcn_exp2f(d);
  float rest = q.rest, t = q.t;
  if (!ref) {
    rest = q.m > ninf ? a * (1.f + q.rest) : q.rest + 1.f;              // (a NaN stays)
    t = a > 0.f ? a * fmaf(d, 1.f + q.rest, q.t) : 0.f;
  }
  rest = wave_add(rest);
  t = wave_add(t);
  const int before = wave_sum(q.before);
  const bool bad = rest != rest;
  const float lz = none ? 0.f : log1pf(rest);
  auto score = [&](float x) { return bad ? nan : none ? ninf : (x - m) - lz; };
  if (lane == 0) {
    const bool in = tok >= 0 && tok < V;
    logprob[row] = tok < 0 ? 0.f : in ? score(xt) : nan;
    rank[row] = in && !bad ? 1 + before : 0;
    entropy[row] = bad ? nan : none ? 0.f : lz - (float)LN2 * t / (1.f + rest);
  }
  if (top == 0) return;
  wave_lds_sync();
  // a value that at least top are at or above: of the lists' entries at one depth the one that so many
  // lists reach it (its upper 16 bits, bit by bit); then the place of each from there on
  const int all = nseg * top;
  uint64_t mine = 0;
  int found = 0;
  const int deep = min(top, (2 * top + nseg - 1) / nseg), reach = (top + deep - 1) / deep;
  const uint32_t probe = lane < nseg ? (uint32_t)(heads[lane * top + deep - 1] >> 32) : 0;
  uint32_t at = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t c = at | 1u << b;
    if (__popcll(__ballot(probe >= c)) >= reach) at = c;
  }
  uint64_t key[K];
#pragma unroll
  for (int k = 0; k < K; ++k) key[k] = k * WAVE + lane < all ? heads[k * WAVE + lane] : 0;
  uint64_t* chosen = heads + all;
  chosen[lane] = 0;
  wave_lds_sync();
  int n = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool in = key[k] && (uint32_t)(key[k] >> 32) >= at;
    const uint64_t w = __ballot(in);
    const int to = n + mbcnt(w);
    if (in && to < WAVE) chosen[to] = key[k];
    n += __popcll(w);
  }
  wave_lds_sync();
  if (n <= WAVE) {
    found = min(n, top);
    const uint64_t own = lane < n ? chosen[lane] : 0;
    int place = 0;
    for (int k = 0; k < n; k += 8)         // (zeros behind the last)
#pragma unroll
      for (int l = 0; l < 8; ++l) place += chosen[k + l] > own;
    wave_lds_sync();
    if (lane < n) chosen[place] = own;
    wave_lds_sync();
    if (lane < found) mine = chosen[lane];
  } else {                                 // many equal ones: one after the other
    uint64_t head = lane < nseg ? heads[lane * top] : 0;
    int next = 1;
    for (; found < top; ++found) {
      const uint64_t best = wave_reduce64(head, OpMax64());
      if (best == 0) break;
      if (lane == found) mine = best;
      if (head == best) head = next < top ? heads[lane * top + next++] : 0;
    }
  }
  float* ol = top_logprobs + (size_t)row * top;
  int* oi = top_ids + (size_t)row * top;
  if (bad) {
    if (lane < top) {
      ol[lane] = nan;
      oi[lane] = -1;
    }
    return;
  }
  if (lane < found) {
    ol[lane] = score(of_key((uint32_t)(mine >> 32)));
    oi[lane] = (int)~(uint32_t)mine;
  }
  if (found < top) {                       // fewer finite ones: the first at -inf, all among 64
    const bool at = lane < V && load_one<DT>(p, lane) == ninf;
    const int place = found + mbcnt(__ballot(at));
    if (at && place < top) {
      ol[place] = ninf;
      oi[place] = lane;
    }
  }
}

// Vectors a thread holds, and segments of a row: the longest of which there is one for every CU.
struct Plan {
  int cv, nseg;
};
static Plan plan(int dtype, int R, int V) {
  const int n = dtype == 1 ? 4 : 8;
  const int chunks = (V + 2 * n - 2) / n / NT + 1;     // of NT vectors, wherever the row starts
  Plan p = {chunks >= 8 ? 8 : chunks > 2 ? 4 : chunks, 0};
  for (;; p.cv /= 2) {
    p.nseg = (chunks + p.cv - 1) / p.cv;
    const int half = (chunks + p.cv / 2 - 1) / (p.cv / 2 > 0 ? p.cv / 2 : 1);
    if (p.cv == 1 || half > MAX_SEGS || (long long)R * p.nseg >= 256) return p;
  }
}

}  // namespace lp
}  // namespace rlu

extern "C" int rlu_token_logprobs_workspace(int dtype, int R, int V, int top, long long* bytes) {
  using namespace rlu::lp;
  if (!bytes || dtype < 0 || dtype > 2 || R < 0 || V < 1 || V > MAX_V || top < 0 ||
      top > MAX_TOP || top > V)
    return -1;
  const long long segs = (long long)R * plan(dtype, R, V).nseg;
  if (segs > UINT32_MAX / NT) return -1;               // (a launch counts its threads in 32 bits)
  *bytes = segs * (sizeof(Part) + 8 * top);
  return 0;
}

extern "C" int rlu_token_logprobs(const void* logits, int dtype, long long ld, int R, int V,
                                  const void* tokens, int wide, int top, float* logprob, int* rank,
                                  float* entropy, float* top_logprobs, int* top_ids, void* ws,
                                  hipStream_t stream) {
  using namespace rlu::lp;
  long long bytes;
  if (rlu_token_logprobs_workspace(dtype, R, V, top, &bytes)) return -1;
  if (ld < 0 || (wide != 0 && wide != 1)) return -1;
  if (R == 0) return 0;
  if (!logits || !tokens || !logprob || !rank || !entropy || !ws) return -1;
  if (top && (!top_logprobs || !top_ids)) return -1;
  if ((uintptr_t)logits % (dtype == 1 ? 4 : 2) || (uintptr_t)ws % 8) return -4;
  const Plan pl = plan(dtype, R, V);
  const auto* x = (const uint8_t*)logits;
  auto* lists = (uint64_t*)ws;                         // (8-byte entries first: both aligned)
  auto* parts = (Part*)(lists + (size_t)R * pl.nseg * top);
  const dim3 grid((unsigned)(R * pl.nseg));
#define RLU_SEG(DT, CV, TOP)                                                                       \
  hipLaunchKernelGGL((segment_k<DT, CV, TOP>), grid, dim3(NT), 0, stream, x, ld, V, pl.nseg,       \
                     tokens, wide, top, parts, lists)
#define RLU_JOIN(DT, K)                                                                          \
  hipLaunchKernelGGL((join_k<DT, K>), dim3((unsigned)R), dim3(rlu::WAVE),                        \
                     top ? (pl.nseg * top + rlu::WAVE) * 8 : 0, stream, x, ld, V, pl.nseg, tokens, \
                     wide, top, parts, lists, logprob, rank, entropy, top_logprobs, top_ids)
#define RLU_CV(DT, TOP)                                                                            \
  do {                                                                                             \
    if (pl.cv == 8) RLU_SEG(DT, 8, TOP);                                                           \
    else if (pl.cv == 4) RLU_SEG(DT, 4, TOP);                                                      \
    else if (pl.cv == 2) RLU_SEG(DT, 2, TOP);                                                      \
    else RLU_SEG(DT, 1, TOP);                                                                      \
  } while (0)
#define RLU_DT(DT)                                                                                 \
  do {                                                                                             \
    if (top) RLU_CV(DT, true);                                                                     \
    else RLU_CV(DT, false);                                                                        \
    if (pl.nseg * top <= 4 * rlu::WAVE) RLU_JOIN(DT, 4);                                           \
    else if (pl.nseg * top <= 12 * rlu::WAVE) RLU_JOIN(DT, 12);                                    \
    else RLU_JOIN(DT, 32);                                                                         \
  } while (0)
  if (dtype == 0) RLU_DT(0);
  else if (dtype == 1) RLU_DT(1);
  else RLU_DT(2);
#undef RLU_DT
#undef RLU_CV
#undef RLU_JOIN
#undef RLU_SEG
  return (int)hipGetLastError();
}
