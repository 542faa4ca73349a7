// Device functions of beam search's selection: exact scores, and the K best of what a wave holds in registers.
#pragma once
#include "pg_common.h"
#include "../../include/polygon_hip.h"

// What a running search adds to a step (pg_beam_search.hip).  Groups are positions of a dense prefix that shrinks; scores,
// finished flags and the history stay with the molecule.
struct BeamTrack {
  const int *n_dev, *mol;            // live positions; molecule at each
  uint8_t *parent, *token;           // this step's history, [molecules, K]
  uint8_t* live;                     // per position: some beam goes on
  int* last;                         // per molecule: steps recorded
  int step;
};
struct BeamSelect {
  const void* logits;
  long ld_group, ld_row;
  int n, K, V;
  const uint8_t* mask;
  long mask_group, mask_row;
  double inv_temp, scale;            // 1 / temp, log2(e) / temp
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
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float beam_unorder(unsigned o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o); }
// The order above the index counted down: one 64-bit maximum finds the best number and, among equal ones, the lowest index.
// A candidate's index is beam << 20 | symbol, which orders as beam * V + symbol does.  (+ 0.0f: -0.0 and 0.0 are one number.)
__device__ __forceinline__ unsigned long long beam_key(float c, unsigned index) {
  return ((unsigned long long)beam_order(c + 0.0f) << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ unsigned beam_key_index(unsigned long long k) { return 0xFFFFFFFFu - (unsigned)k; }
__device__ __forceinline__ float beam_key_number(unsigned long long k) { return beam_unorder((unsigned)(k >> 32)); }

// ---- exact scores -----------------------------------------------------------------------------------------------------
// 2^t of t <= 0 in 64 bits: t = n + f with |f| <= 1/2 (adding 1.5 * 2^52 leaves n in the low bits), 2^f = 1 + f q(f) with q fitted
// to the least largest relative error of 2^f on that interval, 8.1e-13 (Lawson's iteration), n added to the exponent.  13
// instructions, all at the full 64-bit rate, which is also that of fp32 here.  Which candidate wins hangs on the normaliser:
// 32 bits (6e-8) would let near ties flip; 8e-13 is a 70000th of what a score near 1 is rounded by (2^-24), less beside larger ones.
// 2^0 is exactly 1.
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
constexpr double BEAM_LOG2E = 1.4426950408889634074;
__device__ __forceinline__ double beam_exp2(double t) {
  t = fmax(t, -1000.0);                      // -inf and all that would underflow: 1e-301
  const double big = t + 6755399441055744.0, f = t - (big - 6755399441055744.0);
  double p = 1.3178933133195561237e-6;
  p = fma(p, f, 1.5309156473849579456e-5);
  p = fma(p, f, 1.5403825466894596854e-4);
  p = fma(p, f, 1.3333454859215948937e-3);
  p = fma(p, f, 9.618128616111247785e-3);
  p = fma(p, f, 5.550410935267969742e-2);
  p = fma(p, f, 2.4022650698110698366e-1);
  p = fma(p, f, 6.9314718054821182051e-1);
  p = fma(p, f, 1.0);
  u32x2 b = __builtin_bit_cast(u32x2, p);
  b.y += __builtin_bit_cast(u32x2, big).x << 20;
  return __builtin_bit_cast(double, b);
}
// ln of a softmax's sum, 1 <= z <= 2^20: the hardware's log2 (a few 1e-7 off) corrected once by what z falls short of its power,
// ln z = y ln 2 + ln(z 2^-y), the last factor within 1e-6 of 1.  As exact as beam_exp2; ln 1 is exactly 0.
__device__ __forceinline__ double beam_log(double z) {
  const double y = (double)__builtin_amdgcn_logf((float)z), r = fma(z, beam_exp2(-y), -1.0);
  return fma(y, 0.69314718055994530942, fma(-0.5 * r, r, r));
}
// the larger of three; NaN if one is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// a lane's largest number; NaN if it holds one
template <int N> __device__ __forceinline__ float max_nan(const float (&x)[N]) {
  float m = N % 2 ? x[0] : max3_nan(x[0], x[N - 1], x[N - 1]);
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) m = max3_nan(m, x[i], x[i + 1]);
  return m;
}
// c of a candidate: the log-probability in 64 bits, rounded to fp32 once, added to the beam's score in fp32.
__device__ __forceinline__ float beam_score(float x, float m, double inv_temp, double lse, float s) {
  return s + (float)(((double)x - (double)m) * inv_temp - lse);
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
// over the N = 16, 32 or 64 neighbouring lanes that hold a row
template <int N> __device__ __forceinline__ float max_row(float x) {
  if (N == 64) return max64(x);
  x = max16(x);
  return N == 32 ? fmaxf(x, __shfl_xor(x, 16)) : x;
}
template <int N> __device__ __forceinline__ double sum_row(double x) {
  if (N == 64) return sum64(x);
  x = sum16(x);
  return N == 32 ? x + __shfl_xor(x, 16) : x;
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
// With one number per lane (each lane's best; `some` > K lanes exceed `above`): a bound such that at least K lanes reach it,
// and few more - from the wave's best downwards in doubling strides, then by halving; a step costs one comparison and a
// population count.  Any K of what reaches the bound are at least as good as it, so nothing below it can be among the K best.
__device__ __forceinline__ float beam_bound(float best, float above, int K) {
  const unsigned mine = beam_order(best), none = beam_order(above);      // (never +inf: the sum below cannot wrap)
  unsigned hi = beam_order(max64(best)) + 1, lo, step = 1u << 20;        // an eighth of an octave to begin with
  const int enough = K + 4 + K / 4;
  for (;;) {
    lo = hi - none > step ? hi - step : none + 1;
    const int c = __popcll(__ballot(mine >= lo));
    if (c >= K) {
      if (c <= enough) return beam_unorder(lo);
      break;
    }
    hi = lo;
    step <<= 1;
  }
  while (hi - lo > 1) {
    const unsigned mid = lo + (hi - lo) / 2;
    const int c = __popcll(__ballot(mine >= mid));
    if (c >= K) {
      lo = mid;
      if (c <= enough) break;
    } else hi = mid;
  }
  return beam_unorder(lo);
}

// Ranks `m` <= 128 different keys of list[] and puts the K best into won[] in order (won[] beyond m: 0).
__device__ __forceinline__ void beam_rank(const unsigned long long* list, int m, unsigned long long* won, int K, int lane) {
  if (lane < K) won[lane] = 0;
  wave_sync();
  const unsigned long long a = lane < m ? list[lane] : 0;
  int ra = 0;
  if (m <= 64) {
#pragma unroll 4
    for (int j = 0; j < m; ++j) ra += list[j] > a;
  } else {
    const unsigned long long b = lane + 64 < m ? list[lane + 64] : 0;
    int rb = 0;
#pragma unroll 4
    for (int j = 0; j < m; ++j) {
      const unsigned long long o = list[j];
      ra += o > a;
      rb += o > b;
    }
    if (lane + 64 < m && rb < K) won[rb] = b;
  }
  wave_sync();
  if (lane < m && ra < K) won[ra] = a;
  wave_sync();
}

// Puts a few keys (at most 128 in all; the new length is returned) behind the `m` <= 64 that list[] already holds, the K best of
// a wave's N numbers per lane among them; only numbers above `above` (-inf: all) count.  index(i): of a lane's i-th number.
// best: the lane's largest number.  What reaches the bound is nearly always few; where it is not (ties all over) the K best of
// everything are taken out one by one, by way of won[].
template <int N, class F>
__device__ __forceinline__ int beam_collect(const float (&c)[N], F index, float best, float above, int K, unsigned long long* list, int m,
                                            unsigned long long* won, int lane) {
  const int some = __popcll(__ballot(best > above));
  float bound = some > K ? beam_bound(best, above, K) : beam_unorder(beam_order(above) + 1);
  const int m0 = m;
  auto put = [&]() {
    m = m0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = c[i] >= bound;
      const unsigned long long b = __ballot(in);
      if (b) {
        const int at = m + lanes_before(b);
        if (in && at < 128) list[at] = beam_key(c[i], index(i));
        m += __popcll(b);
      }
    }
    wave_sync();
  };
  put();
  const int limit = m0 + K + 24 > 64 ? 128 : 64;       // (a ranking of 64 costs as much as four steps here)
  if (m > limit) {
    // a few lanes hold most of it (rows of very different scores): halve by numbers instead of lanes
    unsigned lo = beam_order(bound), hi = beam_order(max64(best)) + 1;
    int all = m - m0;
    while (all + m0 > limit && hi - lo > 1) {
      const unsigned mid = lo + (hi - lo) / 2;
      const float f = beam_unorder(mid);
      int n = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) n += __popcll(__ballot(c[i] >= f));
      if (n >= K) { lo = mid; all = n; }
      else hi = mid;
    }
    bound = beam_unorder(lo);
    if (all + m0 <= 128) put();
  }
  if (m <= 128) return m;
  // (rare: written so that it needs no registers of its own - `zero` keeps the indices from being worked out ahead of the loop)
  float last = INFINITY;
  unsigned last_i = 0;
  const unsigned long long held = lane < m0 ? list[lane] : 0;           // (m0 <= 64)
  for (int j = 0; j < K; ++j) {
    unsigned zero = 0;
    asm volatile("" : "+v"(zero));
    auto next = [&](float f, unsigned i) { return f < last || (f == last && i > last_i); };
    float top = -INFINITY;
    if (held && next(beam_key_number(held), beam_key_index(held))) top = beam_key_number(held);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c[i] >= bound && next(c[i], index(i) + zero)) top = fmaxf(top, c[i]);
    top = max64(top);
    unsigned top_i = 0xFFFFFFFFu;
    if (held && beam_key_number(held) == top && next(top, beam_key_index(held))) top_i = beam_key_index(held);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c[i] == top && next(top, index(i) + zero)) top_i = min(top_i, index(i) + zero);
    for (int o = 32; o; o >>= 1) top_i = min(top_i, (unsigned)__shfl_xor(top_i, o));
    if (lane == 0) won[j] = top > -INFINITY ? beam_key(top, top_i) : 0;
    last = top;
    last_i = top_i;
  }
  wave_sync();
  const unsigned long long key = lane < K ? won[lane] : 0;
  if (lane < K) list[lane] = key;
  wave_sync();
  return __popcll(__ballot(key != 0));
}
// The same, ranked: the K best of both into won[0 .. K) (keys; 0 where there are fewer).
template <int N, class F>
__device__ __forceinline__ void beam_best(const float (&c)[N], F index, float best, float above, int K, unsigned long long* list, int m,
                                          unsigned long long* won, int lane) {
  beam_rank(list, beam_collect<N>(c, index, best, above, K, list, m, won, lane), won, K, lane);
}

// ---- the step's outputs -----------------------------------------------------------------------------------------------
// One wave; won[] holds the group's K keys by rank, fin the finished beams as bits.
// keep: the best child of a beam takes the beam's place (won[] is by rank, so it is the lowest lane that names the parent),
// the others take the free places in ascending order, then come the entries without a candidate.  place[]: room for K.
template <bool TRACK>
__device__ __forceinline__ void beam_write(const BeamSelect& a, const BeamTrack& tr, long g, long mol, const unsigned long long* won,
                                           unsigned fin, int* place, int lane) {
  const int K = a.K;
  const unsigned long long key = lane < K ? won[lane] : 0;
  const unsigned index = beam_key_index(key);
  const int parent = key ? (int)(index >> 20) : -1, v = key ? (int)(index & 0xFFFFFu) : a.pad;
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
  const bool done = lane < K && (!key || (fin >> parent & 1) || v == a.eos);
  if (TRACK) {
    const bool goes_on = __ballot(lane < K && !done) != 0;
    if (lane == 0) { tr.live[g] = goes_on; tr.last[mol] = tr.step; }
  }
  if (lane >= K) return;
  const long o = g * K + to, om = mol * K + to;      // (mol == g outside a search)
  a.scores_out[om] = key ? beam_key_number(key) : -INFINITY;
  a.finished_out[om] = done;
  a.parents[o] = key ? parent : to;
  a.tokens[o] = v;
  if (TRACK) { tr.parent[om] = key ? parent : to; tr.token[om] = v; }
}

// One step of a search (V <= 128): h [positions * K, H] times fcw [64 or 128, H] plus fcb, then the selection.
template <typename T>
int launch_beam_head(const BeamSelect& a, const BeamTrack& tr, const T* h, int H, const T* fcw, const float* fcb, hipStream_t st);
