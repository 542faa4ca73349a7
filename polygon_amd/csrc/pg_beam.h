// Device functions of beam search's selection: exact scores, and the K best of what a wave holds in registers.
#pragma once
#include "pg_common.h"
#include "../../include/polygon_hip.h"

struct BeamSelect {
  const void* logits;
  long ld_group, ld_row;
  int n, K, V;
  const uint8_t* mask;
  long mask_group, mask_row;
  double inv_temp;
  const float* scores;
  const uint8_t* finished;
  int eos, pad, keep;
  float* scores_out;
  int32_t *parents, *tokens;
  uint8_t* finished_out;
};

// ---- keys -------------------------------------------------------------------------------------------------------------
// A number's bits in the order of the numbers; 0 stands for "nothing" (no number maps to 0).
__device__ __forceinline__ unsigned beam_order(float c) {
  const unsigned b = __float_as_uint(c);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float beam_unorder(unsigned o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o); }
// The order above the index counted down: one 64-bit maximum finds the best number and, among equal ones, the lowest index.
__device__ __forceinline__ unsigned long long beam_key(unsigned order, unsigned index) {
  return ((unsigned long long)order << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ unsigned beam_key_index(unsigned long long k) { return 0xFFFFFFFFu - (unsigned)k; }
__device__ __forceinline__ float beam_key_number(unsigned long long k) { return beam_unorder((unsigned)(k >> 32)); }

// ---- exact scores -----------------------------------------------------------------------------------------------------
// exp of d <= 0 in 64 bits: d = n ln 2 + r with |r| <= ln 2 / 2, the series of exp(r) to r^11 (remainder r^12 / 12! < 7e-15),
// times 2^n.  18 instructions where the library's, which serves every argument, takes about twice that.  Which candidate wins
// hangs on the normaliser, so 32 bits are not enough; 7e-15 is far below what a score's rounding to fp32 can tell.
__device__ __forceinline__ double beam_exp(double d) {
  d = fmax(d, -800.0);                       // -inf and all that underflows: 0
  const double n = rint(d * 1.4426950408889634074);
  double r = fma(n, -6.93147180369123816490e-01, d);   // ln 2 in two parts
  r = fma(n, -1.90821492927058770002e-10, r);
  double p = 1.0 / 39916800.0;
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}
// c of a candidate: the log-probability in 64 bits, rounded to fp32 once, added to the beam's score in fp32.
// (+ 0.0f: -0.0 and 0.0 are one score and go by the index.)
__device__ __forceinline__ float beam_score(float x, float m, double inv_temp, double lse, float s) {
  return (s + (float)(((double)x - (double)m) * inv_temp - lse)) + 0.0f;
}

// ---- reductions over 16 lanes (every lane gets the result; partners add the same two numbers, so all results are equal) ----
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
  const int i = __float_as_int(x);
  return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xF, 0xF, false));
}
template <int CTRL> __device__ __forceinline__ double dpp(double x) {
  const long long i = __double_as_longlong(x);
  const unsigned lo = __builtin_amdgcn_update_dpp((int)i, (int)i, CTRL, 0xF, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp((int)(i >> 32), (int)(i >> 32), CTRL, 0xF, 0xF, false);
  return __longlong_as_double(((long long)hi << 32) | lo);
}
// quad_perm [1,0,3,2], quad_perm [2,3,0,1], row_half_mirror, row_mirror
__device__ __forceinline__ float max16(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  return fmaxf(x, dpp<0x140>(x));
}
__device__ __forceinline__ double sum16(double x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  return x + dpp<0x140>(x);
}
__device__ __forceinline__ float readlane_f(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }
__device__ __forceinline__ float max64(float x) {
  x = max16(x);
  return fmaxf(fmaxf(readlane_f(x, 0), readlane_f(x, 16)), fmaxf(readlane_f(x, 32), readlane_f(x, 48)));
}
__device__ __forceinline__ double readlane_d(double x, int l) {
  const long long i = __double_as_longlong(x);
  const unsigned lo = __builtin_amdgcn_readlane((int)i, l), hi = __builtin_amdgcn_readlane((int)(i >> 32), l);
  return __longlong_as_double(((long long)hi << 32) | lo);
}
__device__ __forceinline__ double sum64(double x) {
  x = sum16(x);
  return (readlane_d(x, 0) + readlane_d(x, 16)) + (readlane_d(x, 32) + readlane_d(x, 48));
}
__device__ __forceinline__ unsigned long long max64(unsigned long long x) {
  for (int o = 32; o; o >>= 1) {
    const unsigned long long t = __shfl_xor(x, o);
    x = t > x ? t : x;
  }
  return x;
}
// lanes below this one that are set in m
__device__ __forceinline__ int lanes_before(unsigned long long m) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0));
}
// LDS written by some lanes of a wave and read by others of the same wave: in order in the hardware, kept so by the compiler
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- the K best of a wave's registers --------------------------------------------------------------------------------
// With one order per lane (each lane's best): a bound such that at least K lanes reach it, and few more - found by halving the
// interval of orders, where a step costs a comparison and a population count.  1 (everything) if fewer than K lanes have any.
// Any K of what reaches the bound are at least as good as it, so nothing below the bound can be among the K best.
__device__ __forceinline__ unsigned beam_bound(unsigned best, int K) {
  if (__popcll(__ballot(best != 0)) <= K) return 1;
  unsigned lo = best ? best : 0xFFFFFFFFu, hi = best;
  for (int o = 32; o; o >>= 1) {
    lo = min(lo, (unsigned)__shfl_xor(lo, o));
    hi = max(hi, (unsigned)__shfl_xor(hi, o));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi) + 1;        // (+inf is never an order here: no wrap)
  const int enough = K + 4 + K / 4;
  while (hi - lo > 1) {
    const unsigned mid = lo + (hi - lo) / 2;
    const int c = __popcll(__ballot(best >= mid));
    if (c >= K) {
      lo = mid;
      if (c <= enough) break;
    } else hi = mid;
  }
  return lo;
}

// Ranks `m` <= 128 different keys of list[] and puts the `keep` best into won[] in order (won[] beyond m: 0).
__device__ __forceinline__ void beam_rank(const unsigned long long* list, int m, unsigned long long* won, int keep, int lane) {
  if (lane < keep) won[lane] = 0;
  const unsigned long long a = lane < m ? list[lane] : 0, b = lane + 64 < m ? list[lane + 64] : 0;
  int ra = 0, rb = 0;
  if (m <= 64) {
    for (int j = 0; j < m; ++j) ra += list[j] > a;
  } else {
    for (int j = 0; j < m; ++j) {
      const unsigned long long o = list[j];
      ra += o > a;
      rb += o > b;
    }
  }
  wave_sync();
  if (lane < m && ra < keep) won[ra] = a;
  if (lane + 64 < m && rb < keep) won[rb] = b;
  wave_sync();
}

// The K best of a wave's N orders per lane (0: nothing) into won[0 .. K) (keys; 0 where there are fewer), by way of list[],
// room for 128.  index(i) is the index of a lane's i-th element.  above: only orders greater than it count.
// What reaches the bound is nearly always few; where it is not (ties all over) the keys are taken out one by one.
template <int N, class F>
__device__ __forceinline__ void beam_best(const unsigned (&order)[N], F index, unsigned above, int K, unsigned long long* list,
                                          unsigned long long* won, int lane) {
  unsigned best = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) best = max(best, order[i]);
  if (best <= above) best = 0;
  const unsigned bound = max(beam_bound(best, K), above + 1);
  int m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = order[i] >= bound;
    const unsigned long long b = __ballot(in);
    if (b) {
      const int at = m + lanes_before(b);
      if (in && at < 128) list[at] = beam_key(order[i], index(i));
      m += __popcll(b);
    }
  }
  wave_sync();
  if (m <= 128) {
    beam_rank(list, m, won, K, lane);
    return;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < K; ++j) {
    unsigned long long top = 0;
    if (last) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned long long k = order[i] >= bound ? beam_key(order[i], index(i)) : 0;
        if (k < last && k > top) top = k;
      }
    }
    last = max64(top);
    if (lane == 0) won[j] = last;
  }
  wave_sync();
}

// ---- the step's outputs -----------------------------------------------------------------------------------------------
// One wave; won[] holds the group's K keys by rank (order of c, index k * V + v), fin the finished beams as bits.
// keep: the best child of a beam takes the beam's place (won[] is by rank, so it is the lowest lane that names the parent),
// the others take the free places in ascending order, then come the entries without a candidate.  place[]: room for K.
__device__ __forceinline__ void beam_write(const BeamSelect& a, long g, const unsigned long long* won, unsigned fin, int* place,
                                           int lane) {
  const int K = a.K;
  const unsigned long long key = lane < K ? won[lane] : 0;
  const unsigned flat = beam_key_index(key);
  const int parent = key ? (int)(flat / (unsigned)a.V) : -1, v = key ? (int)(flat % (unsigned)a.V) : a.pad;
  int to = lane;
  if (a.keep) {
    unsigned long long first = 0;
    unsigned taken = 0;
    for (int p = 0; p < K; ++p) {
      const unsigned long long m = __ballot(parent == p);
      if (m) { first |= m & -m; taken |= 1u << p; }
    }
    const bool vacant = lane < K && !(taken >> lane & 1);
    const unsigned long long vacants = __ballot(vacant);
    if (vacant) place[lanes_before(vacants)] = lane;
    wave_sync();
    // entries that need a free place, in the order of their ranks: those without a candidate rank last by themselves
    const bool is_first = first >> lane & 1;
    const unsigned long long rest = __ballot(lane < K && !is_first);
    if (lane < K) to = is_first ? parent : place[lanes_before(rest)];
  }
  if (lane >= K) return;
  const long o = g * K + to;
  a.scores_out[o] = key ? beam_key_number(key) : -INFINITY;
  a.parents[o] = key ? parent : to;
  a.tokens[o] = v;
  a.finished_out[o] = !key || (fin >> parent & 1) || v == a.eos;
}
