// Beam search: selection over beams and vocabulary.
#include <math.h>
#include "pg_host.h"
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

// The score's bits in the order of the numbers, above the flat index counted down: one 64-bit maximum finds the best score
// and, among equal ones, the lowest index.  0 = no candidate (c is never NaN or -inf here).
__device__ __forceinline__ unsigned long long beam_key(float c, unsigned flat) {
  const unsigned b = __float_as_uint(c);
  const unsigned o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)o << 32) | (0xFFFFFFFFu - flat);
}
__device__ __forceinline__ unsigned beam_key_flat(unsigned long long k) { return 0xFFFFFFFFu - (unsigned)k; }
__device__ __forceinline__ float beam_key_score(unsigned long long k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// c of a candidate: the normaliser in 64 bits (which candidate wins hangs on it), rounded to fp32 once, added in fp32.
// (+ 0.0f: -0.0 and 0.0 are one score and go by the index.)
__device__ __forceinline__ float beam_score(float x, float m, double inv_temp, double lse, float s) {
  return (s + (float)(((double)x - (double)m) * inv_temp - lse)) + 0.0f;
}

// One workgroup per group: every row's maximum and normaliser, then K times the largest key below the last one.
template <typename T> __global__ __launch_bounds__(256) void beam_select_kernel(BeamSelect a) {
  __shared__ double red[4];
  __shared__ unsigned long long redk[4];
  __shared__ float rm[PG_MAX_BEAMS];
  __shared__ double rl[PG_MAX_BEAMS];
  __shared__ int rs[PG_MAX_BEAMS];       // 0 none, 1 alive, 2 finished
  __shared__ unsigned long long won[PG_MAX_BEAMS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long g = blockIdx.x;
  const T* x0 = (const T*)a.logits + g * a.ld_group;
  const uint8_t* m0 = a.mask ? a.mask + g * a.mask_group : nullptr;
  for (int k = 0; k < a.K; ++k) {
    const float s = a.scores[g * a.K + k];
    const bool fin = a.finished && a.finished[g * a.K + k];
    const bool ok = isfinite(s);
    float mx = -INFINITY;
    double sum = 0.0;
    if (ok && !fin) {
      const T* x = x0 + k * a.ld_row;
      const uint8_t* mk = m0 ? m0 + k * a.mask_row : nullptr;
      bool bad = false;
      for (int v = tid; v < a.V; v += 256) {
        const float f = to_f32<T>(x[v]);
        if (mk && !mk[v]) continue;
        bad |= !(f < INFINITY);
        mx = fmaxf(mx, f);
      }
      if (bad) mx = INFINITY;
      for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      if (lane == 0) red[wave] = mx;
      __syncthreads();
      mx = fmaxf(fmaxf((float)red[0], (float)red[1]), fmaxf((float)red[2], (float)red[3]));
      __syncthreads();
      if (isfinite(mx)) {
        for (int v = tid; v < a.V; v += 256)
          if (!mk || mk[v]) sum += exp(((double)to_f32<T>(x[v]) - (double)mx) * a.inv_temp);
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) red[wave] = sum;
        __syncthreads();
        sum = (red[0] + red[1]) + (red[2] + red[3]);
        __syncthreads();
      }
    }
    if (tid == 0) {
      rs[k] = !ok ? 0 : fin ? 2 : isfinite(mx) ? 1 : 0;
      rm[k] = mx;
      rl[k] = log(sum);
    }
  }
  __syncthreads();
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.K; ++j) {
    unsigned long long best = 0;
    if (last)
      for (int k = 0; k < a.K; ++k) {
        const float s = a.scores[g * a.K + k];
        if (rs[k] == 2 && tid == 0) {
          const unsigned long long key = beam_key(s + 0.0f, k * a.V + a.pad);
          if (key < last && key > best) best = key;
        }
        if (rs[k] != 1) continue;
        const T* x = x0 + k * a.ld_row;
        const uint8_t* mk = m0 ? m0 + k * a.mask_row : nullptr;
        for (int v = tid; v < a.V; v += 256) {
          if (mk && !mk[v]) continue;
          const float c = beam_score(to_f32<T>(x[v]), rm[k], a.inv_temp, rl[k], s);
          if (!(c > -INFINITY)) continue;
          const unsigned long long key = beam_key(c, k * a.V + v);
          if (key < last && key > best) best = key;
        }
      }
    for (int o = 32; o; o >>= 1) {
      const unsigned long long other = __shfl_xor(best, o);
      best = other > best ? other : best;
    }
    if (lane == 0) redk[wave] = best;
    __syncthreads();
    best = redk[0];
    for (int w = 1; w < 4; ++w) best = redk[w] > best ? redk[w] : best;
    last = best;
    if (tid == 0) won[j] = best;
    __syncthreads();
  }
  if (tid != 0) return;
  // read every flag before any is written: the outputs may be the inputs
  unsigned fin = 0, taken = 0;
  for (int k = 0; k < a.K; ++k) fin |= (unsigned)(rs[k] == 2) << k;
  int place[PG_MAX_BEAMS];
  for (int j = 0; j < a.K; ++j) {
    place[j] = j;
    if (!a.keep) continue;
    const int p = won[j] ? (int)(beam_key_flat(won[j]) / a.V) : -1;
    place[j] = -1;
    if (p >= 0 && !(taken >> p & 1)) { place[j] = p; taken |= 1u << p; }
  }
  for (int j = 0; j < a.K; ++j) {
    int p = place[j];
    if (p < 0) { p = __ffs(~taken) - 1; taken |= 1u << p; }
    const long o = g * a.K + p;
    if (won[j]) {
      const unsigned flat = beam_key_flat(won[j]);
      const int parent = flat / a.V, v = flat % a.V;
      a.scores_out[o] = beam_key_score(won[j]);
      a.parents[o] = parent;
      a.tokens[o] = v;
      a.finished_out[o] = (fin >> parent & 1) || v == a.eos;
    } else {
      a.scores_out[o] = -INFINITY;
      a.parents[o] = p;
      a.tokens[o] = a.pad;
      a.finished_out[o] = 1;
    }
  }
}

extern "C" size_t pg_beam_select_workspace_bytes(int dtype, int n, int K, int V) { return 0; }

extern "C" int pg_beam_select(int dtype, const void* logits, long ld_group, long ld_row, int n, int K, int V,
                              const uint8_t* mask, long mask_group, long mask_row, double temp, const float* scores,
                              const uint8_t* finished, int eos, int pad, int keep_slots, float* scores_out, int32_t* parents,
                              int32_t* tokens, uint8_t* finished_out, void* ws, size_t ws_bytes, void* stream) {
  PG_REQUIRE(dtype == PG_F32 || dtype == PG_BF16, "pg_beam_select: dtype %d is neither PG_F32 nor PG_BF16", dtype);
  PG_REQUIRE(n >= 0 && K >= 1 && K <= PG_MAX_BEAMS && V >= 1 && V <= PG_MAX_BEAM_V,
             "pg_beam_select: n=%d, K=%d outside [1,%d] or V=%d outside [1,%d]", n, K, PG_MAX_BEAMS, V, PG_MAX_BEAM_V);
  PG_REQUIRE(temp > 0.0 && isfinite(temp) && isfinite(1.0 / temp), "pg_beam_select: temperature must be positive and finite");
  PG_REQUIRE(pad >= 0 && pad < V && eos < V, "pg_beam_select: pad=%d outside [0,%d) or eos=%d not below it", pad, V, eos);
  if (n == 0) return PG_OK;
  PG_REQUIRE(logits && scores && scores_out && parents && tokens && finished_out, "pg_beam_select: NULL buffer");
  BeamSelect a = {logits, ld_group, ld_row, n, K, V, mask, mask_group, mask_row, 1.0 / temp, scores, finished, eos, pad, keep_slots,
                  scores_out, parents, tokens, finished_out};
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PG_BF16) hipLaunchKernelGGL(beam_select_kernel<bf16_t>, dim3(n), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(beam_select_kernel<float>, dim3(n), dim3(256), 0, st, a);
  PG_CHECK_LAUNCH();
  return PG_OK;
}
