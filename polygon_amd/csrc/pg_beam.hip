// Beam search: selection over beams and vocabulary.
#include <math.h>
#include "pg_beam.h"
#include "pg_host.h"
#include "pg_mma.h"
#include <type_traits>

// ---- short vocabularies (V <= 1024) -----------------------------------------------------------------------------------
// N = 16, 32 or 64 lanes hold a row (E neighbouring symbols per lane, wide loads), a wave 64 / N rows at a time, P times, and a
// group takes the G waves that its K rows need.  The logits are read once and stay in registers (at most 32 of them), and
// softmax's reductions stay inside a wave (for N = 16 inside DPP rows).  With G > 1 the first wave selects from the G waves'
// few best.  Bound by instructions (some 700 a wave at 8 x 51, half of them the selection, a fifth the 64-bit exponentials):
// 8192 x 8 x 51 fp32 14.5 us for 10.5 MB, 1024 x 32 x 128 bf16 with masks 19.0 us, one group 4.4 us, most of it latency (each launch
// by itself; back to back a call of 8192 x 8 x 51 takes 12.5).
// Measured against the chunked kernels below where those could start: 4096 x 8 x 129 19 us here, 63 there; 2000 x 8 x 1000 28 and 56.
constexpr int SW = 4;      // waves per workgroup, where G is not more
template <int W, int ROWS> struct ShortLds {
  unsigned long long list[W][128], won[W][PG_MAX_BEAMS];
  double sum[W][ROWS];
  int place[W][PG_MAX_BEAMS], many[W];
};
// Group g (none if !here), whose K rows of logits start at `logits` (global memory or LDS), by the G waves wave, wave + 1, .. of
// the workgroup (wave % G is one's place among them).  With G > 1 every wave of the workgroup must call it.
template <typename T, int N, int E, int P, int G, bool TRACK, int W>
__device__ __forceinline__ void beam_short(const BeamSelect& a, const BeamTrack& tr, const T* logits, long ld, long g, bool here, int wave,
                                           int lane, ShortLds<W, 64 / N * P>& lds) {
  constexpr int R = 64 / N;
  const int K = a.K, V = a.V, k0 = wave % G * (R * P), row = lane / N;
  const long mol = TRACK && here ? tr.mol[g] : g;
  // beam `lane`
  float s_mine = -INFINITY;
  bool fin_mine = false;
  if (here && lane < K) {
    s_mine = a.scores[mol * K + lane];
    fin_mine = a.finished && a.finished[mol * K + lane];
  }
  const unsigned fin = (unsigned)__ballot(fin_mine), alive = (unsigned)__ballot(isfinite(s_mine)), open = alive & ~fin;
  // the lane's symbols v0 .. v0+E-1 of its rows; the row's last lane reads the last E, and leaves out those it shares
  const int sub = lane % N * E, v0 = min(sub, max(V - E, 0));
  float x[P][E], m[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int k = k0 + p * R + row;
#pragma unroll
    for (int e = 0; e < E; ++e) x[p][e] = -INFINITY;
    if (!(open >> k & 1) || sub >= V) continue;
    const T* r = logits + k * ld + v0;
    const uint8_t* mk = a.mask ? a.mask + g * a.mask_group + k * a.mask_row + v0 : nullptr;
    if (V >= E) {
      T t[E];
      __builtin_memcpy(t, r, sizeof(t));
#pragma unroll
      for (int e = 0; e < E; ++e) x[p][e] = v0 + e >= sub ? to_f32<T>(t[e]) : -INFINITY;
      if (mk) {
        uint8_t ok[E];
        __builtin_memcpy(ok, mk, E);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!ok[e]) x[p][e] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < V && (!mk || mk[e])) x[p][e] = to_f32<T>(r[e]);
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const float mx = max_nan(x[p]);
    m[p] = max_row<N>(mx != mx ? INFINITY : mx);    // a NaN or +inf makes the row's maximum +inf, and the beam has no continuation
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += beam_exp2(((double)x[p][e] - (double)m[p]) * a.scale);
    sum = sum_row<N>(sum);
    if (lane % N == 0) lds.sum[wave][p * R + row] = sum;
  }
  wave_sync();
  // one logarithm for all rows
  if (lane < R * P) lds.sum[wave][lane] = beam_log(lds.sum[wave][lane]);
  wave_sync();
  float c[P * E], best = -INFINITY;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int k = k0 + p * R + row;
    const float s = __shfl(s_mine, k);
    const double lse = lds.sum[wave][p * R + row];
    const bool has = (open >> k & 1) && isfinite(m[p]), done = alive & fin & (1u << k);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float f = has ? beam_score(x[p][e], m[p], a.inv_temp, lse, s) : -INFINITY;
      if (done && v0 + e == a.pad && v0 + e >= sub) f = s;
      c[p * E + e] = f;
      best = fmaxf(best, f);
    }
  }
  unsigned long long *list = lds.list[wave], *won = lds.won[wave];
  auto index = [&](int i) { return (unsigned)(k0 + i / E * R + row) << 20 | (unsigned)(v0 + i % E); };
  if (G == 1) beam_best<P * E>(c, index, best, -INFINITY, K, list, 0, won, lane);
  else {   // every wave's few, unranked; the group's first wave selects from them
    const int many = beam_collect<P * E>(c, index, best, -INFINITY, K, list, 0, won, lane);
    if (lane == 0) lds.many[wave] = many;
    __syncthreads();
    if (wave % G != 0) return;
    float t[2 * G], top = -INFINITY;
    unsigned at[2 * G];
#pragma unroll
    for (int i = 0; i < 2 * G; ++i) {
      const int j = lane + i % 2 * 64;
      const unsigned long long key = j < lds.many[wave + i / 2] ? lds.list[wave + i / 2][j] : 0;
      t[i] = key ? beam_key_number(key) : -INFINITY;
      at[i] = beam_key_index(key);
      top = fmaxf(top, t[i]);
    }
    beam_best<2 * G>(t, [&](int i) { return at[i]; }, top, -INFINITY, K, list, 0, won, lane);
  }
  if (here) beam_write<TRACK>(a, tr, g, mol, won, fin, lds.place[wave], lane);
}
template <typename T, int N, int E, int P, int G>
__global__ __launch_bounds__(64 * (G > SW ? G : SW)) void beam_select_short_kernel(BeamSelect a) {
  constexpr int W = G > SW ? G : SW;
  __shared__ ShortLds<W, 64 / N * P> lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const long g = ((long)blockIdx.x * W + wave) / G;
  if (G == 1 && g >= a.n) return;
  beam_short<T, N, E, P, G, false>(a, BeamTrack{}, (const T*)a.logits + g * a.ld_group, a.ld_row, g, g < a.n, wave, lane, lds);
}

// A search's step from the top layer's states: vocabulary projection and selection in one launch.  A workgroup takes the whole
// groups that fit 32 rows (one tile of the matrix instruction); its four waves contract every fourth step of H each,
// straight from memory (the weights, 64 KB in bf16, stay in the L2s), their partial logits meet in LDS, and the selection reads
// them there.  For few rows it is bound by latency: 9.4 us for one group where the tiled product and the selection took 8.7 and
// 4.5; 11 instead of 15.4 + 7.2 us at 512 rows.  At 65536 rows it takes 49 instead of 25 + 13; used there too: those 11 us are 0.7 % of a
// step (the cells take 1510), rows shrink as molecules leave (median over a search of 65536 rows: 27 us), and a second path would
// serve only a search's first steps.
template <typename T, int E, int P, int G>
__global__ __launch_bounds__(64 * SW) void beam_head_kernel(BeamSelect a, BeamTrack tr, const T* __restrict__ h, int H,
                                                            const T* __restrict__ fcw, const float* __restrict__ fcb) {
  constexpr int VP = 16 * E, NT = VP / 32, LD = VP + 4, EPC = 16 / sizeof(T);
  __shared__ ShortLds<SW, 4 * P> lds;
  __shared__ __attribute__((aligned(16))) float part[2][32][LD];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, K = a.K;
  const int n = min(a.n, *tr.n_dev), per = 32 / K;
  const long g0 = (long)blockIdx.x * per;
  if (g0 >= n) return;                                  // uniform over the workgroup
  const int rows = (int)min((long)per, n - g0) * K;
  const int r = lane & 31, half = lane >> 5;
  const T* hr = h + (g0 * K + min(r, rows - 1)) * H + half * EPC;
  const T* wr = fcw + (long)r * H + half * EPC;
  f32x16 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
#pragma unroll 4
  for (int k = wave * 2 * EPC; k < H; k += SW * 2 * EPC) {      // (H is a multiple of 32)
    const uint4 x = *reinterpret_cast<const uint4*>(hr + k);
#pragma unroll
    for (int t = 0; t < NT; ++t) MmaOp<T>::run(acc[t], x, *reinterpret_cast<const uint4*>(wr + (long)t * 32 * H + k));
  }
  // the four partial sums through two tiles (four would not leave room for a second workgroup at 128 symbols)
  for (int turn = 0; turn < 2; ++turn) {
    if (wave >> 1 == turn) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float* y = &part[wave & 1][(i & 3) + 8 * (i >> 2) + 4 * half][t * 32 + r];
          *y = turn ? *y + acc[t][i] : acc[t][i];
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 32 * VP; i += 64 * SW) {
    const int y = i / VP, v = i % VP;
    part[0][y][v] = part[0][y][v] + part[1][y][v] + fcb[v];
  }
  __syncthreads();
  for (int q = 0; q < per; q += SW / G) {
    const int mine = q + wave / G;
    const bool here = mine < per && g0 + mine < n;
    beam_short<float, 16, E, P, G, true>(a, tr, &part[0][here ? mine * K : 0][0], LD, g0 + mine, here, wave, lane, lds);
    if (G > 1) __syncthreads();
  }
}

// ---- long vocabularies ------------------------------------------------------------------------------------------------
// The vocabulary is split into chunks; a wave walks through its chunk in tiles of 64 x 16 symbols held in registers, with a
// running maximum and 64-bit sum of the softmax and the K + 1 best logits so far (a tile's symbols at or below the last of them
// are out at one comparison per lane).  A chunk leaves (max, sum, K + 1 keys of logit and symbol).  A workgroup per group then
// joins the chunks' sums, turns their keys into scores and selects.  Where that would be many keys for one workgroup (few
// groups, many chunks), a workgroup per row first merges the row's chunks into one.
// 64 x 8 x 131072 fp32 (268 MB): 73.7 us, 3.6 TB/s, and 7.0 us for the join.  Reading alone takes 44 us; the exponentials add 26
// (17 instructions a symbol; matrix units do not help an exponential), the later tiles' selection 13: the vector units are busy
// 70 % of the time.  Not kept: tiles of 32 symbols a lane (87 us: fewer waves), the next tile loaded ahead into registers (77), or
// through LDS (70.5: some 3 %, for aligned rows only, and a second variant of the loop); more or fewer waves gain nothing.
constexpr int LE = 16, TILE = 64 * LE, LONG_KEYS = PG_MAX_BEAMS + 1;
struct BeamChunk {
  double sum;
  float max;       // +inf: a NaN or +inf was seen
  int pad;
};
struct BeamLong {
  int tiles, chunks;             // tiles of a chunk; chunks of a row
  BeamChunk* part;               // [n * K, chunks]
  unsigned long long* keys;      // [n * K, chunks, K + 1], best first, 0 behind the last
};
template <typename T>
__global__ __launch_bounds__(64 * SW) void beam_chunk_kernel(BeamSelect a, BeamLong l) {
  __shared__ unsigned long long list_s[SW][128], won_s[SW][LONG_KEYS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long u = (long)blockIdx.x * SW + __builtin_amdgcn_readfirstlane(wave);
  const long row = u / l.chunks;
  const int chunk = (int)(u - row * l.chunks), K = a.K, V = a.V, L = K + 1;
  if (row >= (long)a.n * K) return;
  if (!isfinite(a.scores[row]) || (a.finished && a.finished[row])) return;     // the join does not look at this row
  const long g = row / K;
  const int k = (int)(row - g * K);
  const T* r = (const T*)a.logits + g * a.ld_group + k * a.ld_row;
  const uint8_t* mk = a.mask ? a.mask + g * a.mask_group + k * a.mask_row : nullptr;
  constexpr int W = 16 / sizeof(T);
  float mx = -INFINITY;
  double sum = 0.0;
  bool bad = false;
  float above = -INFINITY;       // the last of the L best so far (-inf: fewer than L)
  unsigned long long *list = list_s[wave], *won = won_s[wave];
  bool fresh = false;            // there are keys behind the ranked ones
  int m = 0;                     // keys in list[], at most 48 between tiles: the L best when it was last ranked, and later ones
  auto settle = [&]() {          // won[] becomes the list
    const unsigned long long key = lane < L ? won[lane] : 0;
    if (key) list[lane] = key;
    m = __popcll(__ballot(key != 0));
    const unsigned last = __builtin_amdgcn_readlane((int)(key >> 32), L - 1);
    above = last ? beam_unorder(last) : -INFINITY;
    wave_sync();
  };
  for (int t = 0; t < l.tiles; ++t) {
    const long b = ((long)chunk * l.tiles + t) * TILE;
    if (b >= V) break;
    // 16-byte loads: W = 4 (fp32) or 8 (bf16) neighbouring symbols per lane and load, a wave's loads dense, all in flight together
    float x[LE];
    if (b + TILE <= V) {
      T e[LE];
#pragma unroll
      for (int q = 0; q < LE / W; ++q) __builtin_memcpy(e + q * W, r + b + (q * 64 + lane) * W, 16);
      if (mk) {
        uint8_t ok[LE];
#pragma unroll
        for (int q = 0; q < LE / W; ++q) __builtin_memcpy(ok + q * W, mk + b + (q * 64 + lane) * W, W);
#pragma unroll
        for (int i = 0; i < LE; ++i) x[i] = ok[i] ? to_f32<T>(e[i]) : -INFINITY;
      } else {
#pragma unroll
        for (int i = 0; i < LE; ++i) x[i] = to_f32<T>(e[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < LE; ++i) {
        const long v = b + (i / W * 64 + lane) * W + i % W;
        x[i] = v < V && (!mk || mk[v]) ? to_f32<T>(r[v]) : -INFINITY;
      }
    }
    const float top = max_nan(x);
    bad |= top != top || top == INFINITY;
    const float all = max64(top);
    if (!(all > -INFINITY) || all == INFINITY) continue;
    if (all > mx) {
      sum *= beam_exp2(((double)mx - (double)all) * a.scale);
      mx = all;
    }
#pragma unroll
    for (int i = 0; i < LE; ++i) {
      sum += beam_exp2(((double)x[i] - (double)mx) * a.scale);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // four at a time: enough to hide their latency, and few registers
    }
    if (!__ballot(top > above)) continue;
    // what the tile has above the last of the best is put behind them, and the list is ranked when it has grown: a stale bound
    // lets a few more in, which is cheaper than a ranking per tile
    const int m0 = m;
    if (__popcll(__ballot(top > above)) <= 32) {
#pragma unroll
      for (int i = 0; i < LE; ++i) {
        const bool in = x[i] > above;
        const unsigned long long some = __ballot(in);
        if (some) {
          const int at = m + lanes_before(some);
          if (in && at < 128) list[at] = beam_key(x[i], (unsigned)(b + (i / W * 64 + lane) * W + i % W));
          m += __popcll(some);
        }
      }
      fresh = m > m0 || fresh;
      if (m <= 48) continue;
    }
    if (m > m0 && m <= 128) beam_rank(list, m, won, L, lane);
    else beam_best<LE>(x, [&](int i) { return (unsigned)(b + (i / W * 64 + lane) * W + i % W); }, top, above, L, list, m0, won, lane);
    settle();
    fresh = false;
  }
  if (fresh) { beam_rank(list, m, won, L, lane); settle(); }
  const bool any_bad = __ballot(bad) != 0;
  sum = sum64(sum);
  if (lane == 0) l.part[row * l.chunks + chunk] = {sum, any_bad ? INFINITY : mx, 0};
  if (lane < L) l.keys[(row * l.chunks + chunk) * L + lane] = lane < m ? list[lane] : 0;
}

// One workgroup per row: its chunks' maxima, sums and keys become those of one chunk, l2's.
__global__ __launch_bounds__(64 * SW) void beam_merge_kernel(BeamSelect a, BeamLong l, BeamLong l2) {
  constexpr int B = 8;           // keys per lane and turn
  __shared__ unsigned long long list_s[SW][128], won_s[SW][LONG_KEYS];
  __shared__ int many[SW];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, L = a.K + 1;
  const long row = blockIdx.x;
  if (!isfinite(a.scores[row]) || (a.finished && a.finished[row])) return;
  if (wave == 0) {
    const BeamChunk* part = l.part + row * l.chunks;
    float mx = -INFINITY;
    double sum = 0.0;
    for (int c = lane; c < l.chunks; c += 64) mx = fmaxf(mx, part[c].max);
    mx = max64(mx);
    if (isfinite(mx))
      for (int c = lane; c < l.chunks; c += 64) sum += part[c].sum * beam_exp2(((double)part[c].max - (double)mx) * a.scale);
    sum = sum64(sum);
    if (lane == 0) l2.part[row] = {sum, mx, 0};
  }
  // every wave the best of its turns (the chunks, and so the symbols, ascend: an equal logit that comes later has the higher
  // index and stays out), then the four lists
  const unsigned long long* keys = l.keys + row * (long)l.chunks * L;
  unsigned long long *list = list_s[wave], *won = won_s[wave];
  const int total = l.chunks * L;
  float above = -INFINITY;
  int m = 0;
  for (int e0 = wave * 64 * B; e0 < total; e0 += SW * 64 * B) {
    float x[B], top = -INFINITY;
    unsigned at[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int e = e0 + i * 64 + lane;
      const unsigned long long key = e < total ? keys[e] : 0;
      x[i] = key ? beam_key_number(key) : -INFINITY;
      at[i] = beam_key_index(key);
      top = fmaxf(top, x[i]);
    }
    if (!__ballot(top > above)) continue;
    beam_best<B>(x, [&](int i) { return at[i]; }, top, above, L, list, m, won, lane);
    const unsigned long long key = lane < L ? won[lane] : 0;
    if (key) list[lane] = key;
    m = __popcll(__ballot(key != 0));
    const unsigned last = __builtin_amdgcn_readlane((int)(key >> 32), L - 1);
    above = last ? beam_unorder(last) : -INFINITY;
    wave_sync();
  }
  if (lane == 0) many[wave] = m;
  __syncthreads();
  if (wave != 0) return;
  // (4 x 33 keys would not fit the 128 that a ranking takes: two by two)
  for (int w = 1; w < SW; ++w) {
    if (lane < many[w]) list[m + lane] = list_s[w][lane];
    wave_sync();
    beam_rank(list, m + many[w], won, L, lane);
    const unsigned long long key = lane < L ? won[lane] : 0;
    if (key) list[lane] = key;
    m = __popcll(__ballot(key != 0));
    wave_sync();
  }
  if (lane < L) l2.keys[row * L + lane] = lane < m ? list[lane] : 0;
}

// One workgroup per group.  The first JKEEP entries of every thread are loaded before anything else and stay in registers (that
// is all of them: more are merged first), their latency behind the rows' sums, which 16 lanes each work out.
// Bound by latency: a chain of loads, two exchanges through LDS, and the ranking of some 2 K keys.
constexpr int JW = 4, JLIST = 1024, JKEEP = 10;
template <typename T>
__global__ __launch_bounds__(64 * JW) void beam_join_kernel(BeamSelect a, BeamLong l) {
  __shared__ unsigned long long list[JLIST], won[PG_MAX_BEAMS], red[JW];
  __shared__ double lse_s[PG_MAX_BEAMS];
  __shared__ float max_s[PG_MAX_BEAMS], score_s[PG_MAX_BEAMS];
  __shared__ int place[PG_MAX_BEAMS], again[64 * JW], have, stop;
  __shared__ unsigned best_s[64 * JW];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, K = a.K, V = a.V;
  const long g = blockIdx.x;
  const int L = K + 1, per_row = l.chunks * L, total = K * per_row;
  const unsigned long long* keys = l.keys + g * (long)total;
  float s_mine = -INFINITY;
  bool fin_mine = false;
  if (lane < K) {
    s_mine = a.scores[g * K + lane];
    fin_mine = a.finished && a.finished[g * K + lane];
  }
  const unsigned fin = (unsigned)__ballot(fin_mine), alive = (unsigned)__ballot(isfinite(s_mine)), open = alive & ~fin;
  // (a row that is not open was not written: its entries are not looked at)
  unsigned long long kept[JKEEP];
#pragma unroll
  for (int i = 0; i < JKEEP; ++i) {
    const int e = tid + i * 64 * JW;
    kept[i] = e < total && (open >> (e / per_row) & 1) ? keys[e] : 0;
  }
  if (wave == 0 && lane < K) score_s[lane] = s_mine;
  // every row's maximum and normaliser from its chunks, 16 lanes a row
  for (int k0 = wave * 4; k0 < K; k0 += 4 * JW) {
    const int k = k0 + (lane >> 4), c0 = lane & 15;
    const bool here = open >> k & 1;          // (false for k >= K)
    const BeamChunk* part = l.part + (g * K + k) * l.chunks;
    float mx = -INFINITY;
    double sum = 0.0;
    if (here)
      for (int c = c0; c < l.chunks; c += 16) mx = fmaxf(mx, part[c].max);
    mx = max16(mx);
    if (here && isfinite(mx))
      for (int c = c0; c < l.chunks; c += 16) sum += part[c].sum * beam_exp2(((double)part[c].max - (double)mx) * a.scale);
    sum = sum16(sum);
    if (c0 == 0 && k < K) { max_s[k] = mx; lse_s[k] = beam_log(sum); }
  }
  if (tid == 0) have = 0;
  __syncthreads();
  // entry e of the group's K * chunks * L, as a key of its score (0: none)
  auto scored = [&](int e, unsigned long long key) -> unsigned long long {
    const int k = e / per_row;
    if (!key || !isfinite(max_s[k])) return 0;
    const float c = beam_score(beam_key_number(key), max_s[k], a.inv_temp, lse_s[k], score_s[k]);
    return c > -INFINITY ? beam_key(c, (unsigned)k << 20 | beam_key_index(key)) : 0;
  };
  auto ended = [&](int k) -> unsigned long long {      // a finished beam's own candidate
    return alive & fin & (1u << k) ? beam_key(score_s[k], (unsigned)k << 20 | (unsigned)a.pad) : 0;
  };
#pragma unroll
  for (int i = 0; i < JKEEP; ++i)
    if (tid + i * 64 * JW < total) kept[i] = scored(tid + i * 64 * JW, kept[i]);
  auto each = [&](auto f) {
    if (tid < K) f(ended(tid));
#pragma unroll
    for (int i = 0; i < JKEEP; ++i) f(kept[i]);
  };
  // a bound that at least K of the threads' bests reach (found in every wave alike)
  unsigned best = 0;
  each([&](unsigned long long key) { best = max(best, (unsigned)(key >> 32)); });
  best_s[tid] = best;
  __syncthreads();
  unsigned b4[JW], bound = 1;
#pragma unroll
  for (int w = 0; w < JW; ++w) b4[w] = best_s[w * 64 + lane];
  {
    int some = 0;
    unsigned lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
    for (int w = 0; w < JW; ++w) {
      some += __popcll(__ballot(b4[w] != 0));
      if (b4[w]) lo = min(lo, b4[w]);
      hi = max(hi, b4[w]);
    }
    for (int o = 32; o; o >>= 1) {
      lo = min(lo, (unsigned)__shfl_xor(lo, o));
      hi = max(hi, (unsigned)__shfl_xor(hi, o));
    }
    if (some > K) {
      hi += 1;
      while (hi - lo > 1) {
        const unsigned mid = lo + (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int w = 0; w < JW; ++w) c += __popcll(__ballot(b4[w] >= mid));
        if (c >= K) {
          lo = mid;
          if (c <= K + 4 + K / 4) break;
        } else hi = mid;
      }
      bound = lo;
    }
  }
  auto put = [&](unsigned long long key) {
    if ((unsigned)(key >> 32) < bound) return;
    const int at = atomicAdd(&have, 1);       // the list's order does not matter: its keys are ranked
    if (at < JLIST) list[at] = key;
  };
  each(put);
  if (tid < K) won[tid] = 0;
  __syncthreads();
  const int m = have;
  if (m <= JLIST) {
    for (int i = tid; i < m; i += 64 * JW) {
      const unsigned long long key = list[i];
      int r = 0;
      for (int j = 0; j < m; ++j) r += list[j] > key;
      if (r < K) won[r] = key;
    }
  } else {   // ties all over: the keys one by one
    unsigned long long last = ~0ull;
    for (int j = 0; j < K; ++j) {
      unsigned long long top = 0;
      each([&](unsigned long long key) { if (key < last && key > top) top = key; });
      top = max64(top);
      if (lane == 0) red[wave] = top;
      __syncthreads();
      for (int w = 0; w < JW; ++w) top = red[w] > top ? red[w] : top;
      last = top;
      if (tid == 0) won[j] = top;
      __syncthreads();
    }
  }
  __syncthreads();
  // A chunk's list goes by the logit, the selection by the score, and rounding can give symbols with different logits one
  // score: then the lower index counts.  What a list left out can only matter if its last entry, the K + 1st, still has the score of
  // the group's last winner (it cannot have a better one: K others of the list are as good) and a lower logit could have it too;
  // such a chunk is read again for the symbols of that score.  (Logits that tie by being equal are listed by index already.)
  // That is at most one chunk of a group, read up to K times by this workgroup alone - slow where a merged row, which is one chunk,
  // has one score all over.  All logits zero, fp32, against ordinary ones: 4 x 8 x 32001 53 and 17 us, 64 x 8 x 131072 232 and 81,
  // 1 x 8 x 131072 861 and 20, 1 x 32 x 131072 3490 and 40, 1 x 32 x 2^20 26300 and 78.
  const unsigned edge = (unsigned)(won[K - 1] >> 32);
  if (edge == 0) {
    if (wave == 0) beam_write<false>(a, BeamTrack{}, g, g, won, fin, place, lane);
    return;
  }
  for (int base = 0; base < K * l.chunks; base += 64 * JW) {
    if (tid == 0) have = 0;
    __syncthreads();
    {
      const int kc = base + tid, k = kc / l.chunks;       // (beam, chunk)
      bool near = false;
      if (kc < K * l.chunks && (open >> k & 1)) {
        const unsigned long long key = keys[kc * L + K];
        // the list's last entry has the edge's score, so has the next lower number of the logits' type, and the chunk does not
        // start behind the last winner
        if ((unsigned)(scored(kc * L + K, key) >> 32) == edge) {
          const float lower = beam_unorder((unsigned)(key >> 32) - (sizeof(T) == 2 ? 0x10000u : 1u));
          near = (unsigned)(beam_key(beam_score(lower, max_s[k], a.inv_temp, lse_s[k], score_s[k]), 0) >> 32) == edge &&
                 ((unsigned)k << 20 | (unsigned)(kc % l.chunks) * l.tiles * TILE) < beam_key_index(won[K - 1]);
        }
      }
      if (near) again[atomicAdd(&have, 1)] = kc;
    }
    __syncthreads();
    const int again_n = have;
    for (int i = 0; i < again_n; ++i) {
      const int k = again[i] / l.chunks, c = again[i] % l.chunks;
      const T* r = (const T*)a.logits + g * a.ld_group + k * a.ld_row;
      const uint8_t* mk = a.mask ? a.mask + g * a.mask_group + k * a.mask_row : nullptr;
      const long v1 = min((long)V, (long)(c + 1) * l.tiles * TILE);
      // the symbols of the edge's score, lowest first, until one does not beat the last winner
      unsigned long long last = ~0ull;
      for (int round = 0; round < K; ++round) {
        unsigned long long top = 0;
        for (long v = (long)c * l.tiles * TILE + tid; v < v1; v += 64 * JW) {
          if (mk && !mk[v]) continue;
          const float sc = beam_score(to_f32<T>(r[v]), max_s[k], a.inv_temp, lse_s[k], score_s[k]);
          const unsigned long long key = beam_key(sc, (unsigned)k << 20 | (unsigned)v);
          if ((unsigned)(key >> 32) != edge) continue;
          if (key < last && key > top) top = key;
        }
        top = max64(top);
        if (lane == 0) red[wave] = top;
        __syncthreads();
        for (int w = 0; w < JW; ++w) top = red[w] > top ? red[w] : top;
        last = top;
        if (tid == 0) {      // into the winners, if it beats the last one and is not there yet
          bool in = top > won[K - 1];
          for (int j = 0; j < K; ++j) in &= won[j] != top;
          if (in) {
            int j = K - 1;
            for (; j > 0 && won[j - 1] < top; --j) won[j] = won[j - 1];
            won[j] = top;
          }
          stop = top == 0 || top < won[K - 1];
        }
        __syncthreads();
        if (stop) break;
      }
      __syncthreads();
    }
    __syncthreads();
  }
  if (wave == 0) beam_write<false>(a, BeamTrack{}, g, g, won, fin, place, lane);
}

constexpr int SHORT_V = 1024;
// Tiles per chunk: as long as there are waves enough for the card (4 on each of its 1024 SIMDs) a chunk is made longer - the
// K + 1 best so far make the next tile cheap, and there are fewer lists to join.
static BeamLong long_plan(int n, int K, int V) {
  BeamLong l = {};
  const long tiles = (V + TILE - 1) / TILE, rows = (long)n * K;
  l.tiles = (int)std::max<long>(1, std::min<long>(tiles, rows * tiles / 4096));
  l.chunks = (int)((tiles + l.tiles - 1) / l.tiles);
  return l;
}

// A group's keys that its one workgroup of the join takes without a merge: what it holds in registers.  Measured, a whole call: one
// group, K = 16, 131072 symbols (34816 keys) 27 us with the merge and 117 without; four groups, K = 8, 32001 symbols (2304) 20.7
// with and 18.0 without.
static bool long_merges(const BeamLong& l, int K) { return l.chunks > 1 && (long)K * (K + 1) * l.chunks > JKEEP * 64 * JW; }
struct LongWs { size_t part, keys, part2, keys2, total; };
static LongWs long_ws(const BeamLong& l, int n, int K) {
  LongWs w;
  size_t p = 0;
  auto take = [&](size_t bytes) { size_t r = p; p = align_up(p + bytes, 256); return r; };
  const size_t rows = (size_t)n * K, merged = long_merges(l, K) ? rows : 0;
  w.part = take(rows * l.chunks * sizeof(BeamChunk)); w.keys = take(rows * l.chunks * (K + 1) * 8);
  w.part2 = take(merged * sizeof(BeamChunk)); w.keys2 = take(merged * (K + 1) * 8);
  w.total = p;
  return w;
}

extern "C" size_t pg_beam_select_workspace_bytes(int dtype, int n, int K, int V) {
  (void)dtype;
  return n < 1 || K < 1 || V <= SHORT_V ? 0 : long_ws(long_plan(n, K, V), n, K).total;
}

template <int I> using Int = std::integral_constant<int, I>;
// Waves per group: the least power of two whose waves of `rows` rows each hold K
template <class F> static void with_waves(int K, int rows, F f) {
  if (K <= rows) f(Int<1>{});
  else if (K <= 2 * rows) f(Int<2>{});
  else if (K <= 4 * rows) f(Int<4>{});
  else if (K <= 8 * rows) f(Int<8>{});
  else f(Int<16>{});
}
// f(N, E, P, G): the narrowest kernel that holds V symbols and K beams.  Up to 4 beams one row per 16 lanes (P = 1) instead of two:
// 8192 groups of 4 x 51 8.3 us against 10.0, 65536 of 4 x 128 57 against 78, one of 1 x 51 3.5 against 3.9.
template <class F> static void with_short_shape(int V, int K, F f) {
  auto shape = [&](auto n, auto e, auto p) { with_waves(K, 64 / n * p, [&](auto g) { if constexpr (g * (64 / n * p) <= PG_MAX_BEAMS) f(n, e, p, g); }); };
  if (V <= 64) K <= 4 ? f(Int<16>{}, Int<4>{}, Int<1>{}, Int<1>{}) : shape(Int<16>{}, Int<4>{}, Int<2>{});
  else if (V <= 128) K <= 4 ? f(Int<16>{}, Int<8>{}, Int<1>{}, Int<1>{}) : shape(Int<16>{}, Int<8>{}, Int<2>{});
  else if (V <= 256) shape(Int<32>{}, Int<8>{}, Int<4>{});
  else if (V <= 512) shape(Int<64>{}, Int<8>{}, Int<4>{});
  else shape(Int<64>{}, Int<16>{}, Int<2>{});
}
template <typename T> static int launch_short(const BeamSelect& a, hipStream_t st) {
  with_short_shape(a.V, a.K, [&](auto n, auto e, auto p, auto g) {
    constexpr int W = g > SW ? g : SW;
    hipLaunchKernelGGL((beam_select_short_kernel<T, n, e, p, g>), dim3(cdiv((long)a.n * g, W)), dim3(64 * W), 0, st, a);
  });
  PG_CHECK_LAUNCH();
  return PG_OK;
}
template <typename T>
int launch_beam_head(const BeamSelect& a, const BeamTrack& tr, const T* h, int H, const T* fcw, const float* fcb, hipStream_t st) {
  PG_REQUIRE(a.V <= PG_MAX_V && a.K <= PG_MAX_BEAMS && H % 32 == 0, "beam search: V=%d, K=%d or H=%d out of range", a.V, a.K, H);
  with_short_shape(a.V, a.K, [&](auto n, auto e, auto p, auto g) {
    if constexpr (n == 16) hipLaunchKernelGGL((beam_head_kernel<T, e, p, g>), dim3(cdiv(a.n, 32 / a.K)), dim3(64 * SW), 0, st, a, tr, h, H, fcw, fcb);
  });
  PG_CHECK_LAUNCH();
  return PG_OK;
}
template int launch_beam_head<float>(const BeamSelect&, const BeamTrack&, const float*, int, const float*, const float*, hipStream_t);
template int launch_beam_head<bf16_t>(const BeamSelect&, const BeamTrack&, const bf16_t*, int, const bf16_t*, const float*, hipStream_t);

template <typename T> static int beam_select_t(const BeamSelect& a, void* ws, size_t ws_bytes, hipStream_t st) {
  if (a.V <= SHORT_V) return launch_short<T>(a, st);
  BeamLong l = long_plan(a.n, a.K, a.V);
  const LongWs w = long_ws(l, a.n, a.K);
  if (!ws || ws_bytes < w.total) PG_FAIL(PG_ERR_WORKSPACE, "pg_beam_select: workspace too small (%zu < %zu)", ws_bytes, w.total);
  const long rows = (long)a.n * a.K, lists = rows * l.chunks;
  PG_REQUIRE(lists < (1L << 26), "pg_beam_select: n=%d, K=%d, V=%d are too many rows for one call", a.n, a.K, a.V);
  l.part = at<BeamChunk>(ws, w.part);
  l.keys = at<unsigned long long>(ws, w.keys);
  hipLaunchKernelGGL(beam_chunk_kernel<T>, dim3(cdiv(lists, SW)), dim3(64 * SW), 0, st, a, l);
  PG_CHECK_LAUNCH();
  if (long_merges(l, a.K)) {
    BeamLong l2 = l;
    l2.tiles = l.tiles * l.chunks; l2.chunks = 1;
    l2.part = at<BeamChunk>(ws, w.part2);
    l2.keys = at<unsigned long long>(ws, w.keys2);
    hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)rows), dim3(64 * SW), 0, st, a, l, l2);
    PG_CHECK_LAUNCH();
    l = l2;
  }
  hipLaunchKernelGGL(beam_join_kernel<T>, dim3(a.n), dim3(64 * JW), 0, st, a, l);
  PG_CHECK_LAUNCH();
  return PG_OK;
}

extern "C" int pg_beam_select(int dtype, const void* logits, long ld_group, long ld_row, int n, int K, int V,
                              const uint8_t* mask, long mask_group, long mask_row, double temp, const float* scores,
                              const uint8_t* finished, int eos, int pad, int keep_slots, float* scores_out, int32_t* parents,
                              int32_t* tokens, uint8_t* finished_out, void* ws, size_t ws_bytes, void* stream) {
  PG_REQUIRE(dtype == PG_F32 || dtype == PG_BF16, "pg_beam_select: dtype %d is neither PG_F32 nor PG_BF16", dtype);
  PG_REQUIRE(n >= 0 && K >= 1 && K <= PG_MAX_BEAMS && V >= 1 && V <= PG_MAX_BEAM_V,
             "pg_beam_select: n=%d, K=%d outside [1,%d] or V=%d outside [1,%d]", n, K, PG_MAX_BEAMS, V, PG_MAX_BEAM_V);
  PG_REQUIRE(temp > 0.0 && isfinite(temp) && isfinite(2.0 / temp), "pg_beam_select: temperature must be positive and finite");
  PG_REQUIRE(pad >= 0 && pad < V && eos < V, "pg_beam_select: pad=%d outside [0,%d) or eos=%d not below it", pad, V, eos);
  PG_REQUIRE((long)n * K < 1L << 24, "pg_beam_select: n * K = %ld is not below 2^24", (long)n * K);
  if (n == 0) return PG_OK;
  PG_REQUIRE(logits && scores && scores_out && parents && tokens && finished_out, "pg_beam_select: NULL buffer");
  const BeamSelect a = {logits, ld_group, ld_row, n, K, V, mask, mask_group, mask_row, 1.0 / temp, BEAM_LOG2E / temp, scores, finished, eos, pad, keep_slots,
                        scores_out, parents, tokens, finished_out};
  return dtype == PG_BF16 ? beam_select_t<bf16_t>(a, ws, ws_bytes, (hipStream_t)stream)
                          : beam_select_t<float>(a, ws, ws_bytes, (hipStream_t)stream);
}
