// VAE.beam_search: the K most probable strings of every latent, by beam search over the GRU decoder.
//
// A row is one beam: group (molecule) p's beams are rows p*K .. p*K + K-1.  Per step: L GRU cells, vocabulary projection
// and selection (pg_beam.hip, one launch, places kept), reorder of the 2 L state planes (only beams with more than one child move).  Beams
// end at different lengths: every COMPACT_EVERY steps the molecules whose beams have all ended leave, and the others close
// up, so the cells run over a shrinking prefix whose length only the device knows - nothing is waited for.  What is recorded
// per step is a parent and a symbol per beam (2 bytes); the strings are traced back at the end.
#include <math.h>
#include "pg_beam.h"
#include "pg_gemm.h"
#include "pg_gru.h"
#include "pg_host.h"
#include "pg_layout.h"
#include "pg_pages.h"

int shadow_join(hipStream_t st);   // pg_vae.hip

// A compaction costs one launch of 6 us and the moves of what closes up; a step of the default decoder takes 60 us for a few
// rows and 1.6 ms for 65536.  Whole searches, 99 steps of the bf16 default decoder: 1 latent x 5 beams 2.0 ms, 64 x 8 6.1 ms,
// 1024 x 8 12.3 ms, 8192 x 8 77.6 ms (72.1 of them the cells, 2.9 projection and selection, 2.4 reorder, 0.1 compaction).
constexpr int COMPACT_EVERY = 8;

// Latents of one turn.  The cells and the products read states and latents by 32-bit byte offsets into a descriptor of 2 GiB, and
// the cells' grid counts tiles of 64 rows in its second dimension: a call beyond that decodes its latents in turns of one size, one after
// another in the same workspace.
static long latent_bytes(const pg_dims* d, int dtype, int K) { return std::max((long)K * d->Hd, (long)d->Dz) * (dtype == PG_BF16 ? 2 : 4); }
static int turn_size(const pg_dims* d, int dtype, int n, int K) {
  const long most = std::min(((1L << 31) - 1) / latent_bytes(d, dtype, K), 65535L * 64 / K);
  return cdiv(n, cdiv(n, most));
}

struct SearchWs {
  size_t zop, zproj, h0_32, h0_op, carry[PG_MAX_LAYERS], hop[PG_MAX_LAYERS][2], tok, parents, mol, count, live, last, scores,
      finished, hist, compact, total;
};
static SearchWs search_ws_layout(const pg_dims* d, int dtype, long n, int K, int max_len) {
  const size_t es = dtype == PG_BF16 ? 2 : 4, rows = n * K, Hd = d->Hd, Dz = d->Dz;
  SearchWs w;
  size_t p = 0;
  auto take = [&](size_t bytes) { size_t r = p; p = align_up(p + bytes, 256); return r; };
  w.zop = take(n * Dz * es); w.zproj = take(n * 3 * Hd * 4); w.h0_32 = take(n * Hd * 4); w.h0_op = take(n * Hd * es);
  for (int l = 0; l < d->L; ++l) {
    w.carry[l] = take(rows * Hd * 4);
    w.hop[l][0] = take(rows * Hd * es); w.hop[l][1] = take(rows * Hd * es);
  }
  w.tok = take(rows * 4); w.parents = take(rows * 4);
  w.mol = take(n * 4); w.count = take(2 * 4); w.live = take(n); w.last = take(n * 4);
  w.scores = take(rows * 4); w.finished = take(rows);
  w.hist = take(2 * rows * (max_len - 1));
  w.compact = take(pg_pages_compact_workspace_bytes((int)n));
  w.total = p;
  return w;
}

__global__ __launch_bounds__(256) void search_init_kernel(int n, int K, int bos, int* __restrict__ tok, int* __restrict__ mol,
                                                          int* __restrict__ count, int* __restrict__ last, float* __restrict__ scores,
                                                          uint8_t* __restrict__ finished) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i == 0) count[0] = n;
  if (i < n) { mol[i] = (int)i; last[i] = 0; }
  if (i < (long)n * K) {
    tok[i] = bos;
    scores[i] = i % K == 0 ? 0.0f : -INFINITY;      // one beam per latent to begin with
    finished[i] = 0;
  }
}

// The strings, best first (equal scores: lower place first): beam (molecule, rank) walks its history back.
__global__ __launch_bounds__(256) void search_trace_kernel(int n, int K, int max_len, int bos, int pad, int eos, const float* __restrict__ scores,
                                                           const int* __restrict__ last, const uint8_t* __restrict__ parent,
                                                           const uint8_t* __restrict__ token, uint8_t* __restrict__ tokens,
                                                           int32_t* __restrict__ end_pads, float* __restrict__ out) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)n * K) return;
  const long mol = i / K, step = (long)n * K;
  int at = (int)(i - mol * K), rank = 0;
  const float s = scores[i];
  for (int j = 0; j < K; ++j) {
    const float o = scores[mol * K + j];
    rank += o > s || (o == s && j < at);
  }
  const long to = mol * K + rank;
  uint8_t* row = tokens + to * max_len;
  out[to] = s;
  int end = s > -INFINITY ? max_len : 0;            // (a place without a hypothesis is the empty string)
  const int t1 = s > -INFINITY ? last[mol] : 0;
  for (int t = max_len - 1; t > t1; --t) row[t] = (uint8_t)pad;
  for (int t = t1; t > 0; --t) {
    const long h = (t - 1) * step + mol * K + at;
    const int v = token[h];
    row[t] = (uint8_t)v;
    if (v == eos) end = t + 1;                      // (behind its eos a beam appends pad: the first eos is the last seen here)
    at = parent[h];
  }
  row[0] = (uint8_t)bos;
  end_pads[to] = end;
}

template <typename T>
static int search_t(const pg_dims* d, int dtype, const float* params, const void* shadow, void* ws, int n, int K, int max_len,
                    const float* z, const uint8_t* allowed, double temp, uint8_t* tokens, int32_t* end_pads, float* scores,
                    hipStream_t st) {
  const ParamOff po = param_offsets(d);
  const ShadowOff so = shadow_offsets(d, dtype);
  const SearchWs w = search_ws_layout(d, dtype, n, K, max_len);
  const int Hd = d->Hd, Dz = d->Dz, L = d->L, rows = n * K;
  const long es = sizeof(T);
  int *tok = at<int>(ws, w.tok), *mol = at<int>(ws, w.mol), *count = at<int>(ws, w.count), *last = at<int>(ws, w.last);
  float* beam_scores = at<float>(ws, w.scores);
  uint8_t *finished = at<uint8_t>(ws, w.finished), *live = at<uint8_t>(ws, w.live), *hist = at<uint8_t>(ws, w.hist);
  const long half = (long)rows * (max_len - 1);
  hipLaunchKernelGGL(search_init_kernel, dim3(cdiv(rows, 256)), dim3(256), 0, st, n, K, d->bos, tok, mol, count, last, beam_scores, finished);
  PG_CHECK_LAUNCH();
  T* z_op = at<T>(ws, w.zop);
  PG_TRY(convert_to<T>(z, z_op, (long)n * Dz, st));
  {
    GemmEpi<T> e;
    e.C32 = at<float>(ws, w.zproj); e.ldc = 3 * Hd;
    PG_TRY(launch_gemm_nt<T>(z_op, Dz, at<T>(shadow, so.wih0z), Dz, n, 3 * Hd, Dz, e, st));
  }
  {
    GemmEpi<T> e;
    e.bias = params + po.lat_b; e.C32 = at<float>(ws, w.h0_32); e.Ct = at<T>(ws, w.h0_op); e.ldc = Hd;
    PG_TRY(launch_gemm_nt<T>(z_op, Dz, at<T>(shadow, so.lat_w), Dz, n, Hd, Dz, e, st));
  }
  {   // h0 into the first beam of every molecule, in all layers; the other places have no beam yet
    pg_plane dst[2 * PG_MAX_LAYERS], src[2 * PG_MAX_LAYERS];
    for (int l = 0; l < L; ++l) {
      dst[2 * l] = {at<char>(ws, w.carry[l]), (long)K * Hd * 4, (long)Hd * 4};
      src[2 * l] = {at<char>(ws, w.h0_32), (long)Hd * 4, (long)Hd * 4};
      dst[2 * l + 1] = {at<char>(ws, w.hop[l][0]), (long)K * Hd * es, (long)Hd * es};
      src[2 * l + 1] = {at<char>(ws, w.h0_op), (long)Hd * es, (long)Hd * es};
    }
    PG_TRY(pg_pages_fork(dst, src, 2 * L, n, n, mol, st));
  }
  int cur = 0;      // which of the two counts is the present one
  for (int i = 1; i < max_len; ++i) {
    const int p = (i - 1) & 1;
    for (int l = 0; l < L; ++l) {
      GruFwdArgs<T> a;
      a.rows = rows; a.H = Hd;
      a.groups_dev = count + cur; a.group_rows = K;
      a.hprev_op = at<T>(ws, w.hop[l][p]);
      a.hprev32 = at<float>(ws, w.carry[l]);
      a.Whh = at<T>(shadow, so.whh[l]);
      a.bhn = params + po.dec_bhh[l] + 2 * Hd;
      if (l == 0) {
        a.gi_mode = PG_GI_TABLE;
        a.table = at<float>(shadow, so.tab_dec);
        a.tok = tok;
        a.zproj = at<float>(ws, w.zproj);
      } else {
        a.gi_mode = PG_GI_FUSED;
        a.x = at<T>(ws, w.hop[l - 1][p ^ 1]);
        a.Kx = Hd;
        a.Wih = at<T>(shadow, so.wih[l]);
        a.bias_gi = at<float>(shadow, so.bias_gi[l]);
      }
      a.h_op = at<T>(ws, w.hop[l][p ^ 1]);
      a.h32 = at<float>(ws, w.carry[l]);
      PG_TRY(launch_gru_fwd<T>(a, st));
    }
    const BeamSelect sel = {nullptr, 0, 0, n, K, d->V, allowed, 0, 0, 1.0 / temp, BEAM_LOG2E / temp, beam_scores, finished, d->eos, d->pad,
                            1, beam_scores, at<int>(ws, w.parents), tok, finished};
    const BeamTrack tr = {count + cur, mol, hist + (long)(i - 1) * rows, hist + half + (long)(i - 1) * rows, live, last, i};
    PG_TRY(launch_beam_head<T>(sel, tr, at<T>(ws, w.hop[L - 1][p ^ 1]), Hd, at<T>(shadow, so.fc_w), at<float>(shadow, so.fc_b), st));
    if (i + 1 == max_len) break;
    pg_plane planes[2 * PG_MAX_LAYERS + 3];
    int np = 0;
    for (int l = 0; l < L; ++l) {
      planes[np++] = {at<char>(ws, w.carry[l]), (long)Hd * 4, (long)Hd * 4};
      planes[np++] = {at<char>(ws, w.hop[l][p ^ 1]), (long)Hd * es, (long)Hd * es};
    }
    if (K > 1) PG_TRY(launch_pages_reorder(planes, np, n, count + cur, K, at<int>(ws, w.parents), st));
    if (i % COMPACT_EVERY == 0) {
      for (int q = 0; q < np; ++q) { planes[q].pitch *= K; planes[q].bytes *= K; }      // a page is a molecule's K rows
      planes[np++] = {at<char>(ws, w.zproj), 3L * Hd * 4, 3L * Hd * 4};
      planes[np++] = {tok, 4L * K, 4L * K};
      planes[np++] = {mol, 4, 4};
      PG_TRY(launch_pages_compact(planes, np, n, count + cur, live, count + (cur ^ 1), nullptr, at<char>(ws, w.compact), st));
      cur ^= 1;
    }
  }
  hipLaunchKernelGGL(search_trace_kernel, dim3(cdiv(rows, 256)), dim3(256), 0, st, n, K, max_len, d->bos, d->pad, d->eos, beam_scores, last,
                     hist, hist + half, tokens, end_pads, scores);
  PG_CHECK_LAUNCH();
  return PG_OK;
}

static int check_search(const pg_dims* d, int dtype, int n, int K, int max_len) {
  PG_TRY(check_dims(d, dtype));
  PG_REQUIRE(n >= 1 && K >= 1 && K <= PG_MAX_BEAMS && (long)n * K < 1L << 24, "pg_beam_search: n=%d, K=%d (K <= %d, n * K < 2^24)", n, K,
             PG_MAX_BEAMS);
  PG_REQUIRE(max_len >= 2 && max_len <= 1 << 20, "pg_beam_search: max_len=%d outside [2, 2^20]", max_len);
  PG_REQUIRE(latent_bytes(d, dtype, K) < 1L << 31, "pg_beam_search: one latent's %d beams of %d units do not fit an operand of 2 GiB", K, d->Hd);
  return PG_OK;
}
extern "C" size_t pg_beam_search_workspace_bytes(const pg_dims* d, int dtype, int n, int K, int max_len) {
  return check_search(d, dtype, n, K, max_len) == PG_OK ? search_ws_layout(d, dtype, turn_size(d, dtype, n, K), K, max_len).total : 0;
}
extern "C" int pg_beam_search(const pg_dims* d, int dtype, const float* params, const void* shadow, void* ws, size_t ws_bytes, int n,
                              int K, int max_len, const float* z, const uint8_t* allowed, double temp, uint8_t* tokens,
                              int32_t* end_pads, float* scores, void* stream) {
  PG_TRY(check_search(d, dtype, n, K, max_len));
  PG_REQUIRE(params && shadow && ws && z && tokens && end_pads && scores, "pg_beam_search: NULL buffer");
  PG_REQUIRE(temp > 0.0 && isfinite(temp) && isfinite(2.0 / temp), "pg_beam_search: temperature must be positive and finite");
  const int m = turn_size(d, dtype, n, K);
  const size_t need = search_ws_layout(d, dtype, m, K, max_len).total;
  if (ws_bytes < need) PG_FAIL(PG_ERR_WORKSPACE, "pg_beam_search: workspace too small (%zu < %zu)", ws_bytes, need);
  PG_TRY(check_persist());
  PG_TRY(shadow_join((hipStream_t)stream));
  for (int r = 0; r < n; r += m) {
    const auto search = dtype == PG_BF16 ? search_t<bf16_t> : search_t<float>;
    const long row = (long)r * K;
    PG_TRY(search(d, dtype, params, shadow, ws, std::min(m, n - r), K, max_len, z + (long)r * d->Dz, allowed, temp, tokens + row * max_len,
                  end_pads + row, scores + row, (hipStream_t)stream));
  }
  return PG_OK;
}
