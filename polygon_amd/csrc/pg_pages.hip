// Pages of a cache of decoder states: reorder inside groups, fork, compaction.
#include "pg_host.h"
#include "../../include/polygon_hip.h"

struct Planes {
  pg_plane p[PG_MAX_PLANES];
};

// Two planes of `pages` pages share bytes: their spans overlap, unless they interleave with one pitch.
static bool planes_share(const pg_plane& a, long na, const pg_plane& b, long nb) {
  if (na < 1 || nb < 1) return false;
  const uintptr_t a0 = (uintptr_t)a.base, b0 = (uintptr_t)b.base;
  if (a0 + (na - 1) * a.pitch + a.bytes <= b0 || b0 + (nb - 1) * b.pitch + b.bytes <= a0) return false;
  if (a.pitch != b.pitch) return true;
  const long d = (long)((b0 >= a0 ? b0 - a0 : (uintptr_t)a.pitch - (a0 - b0) % a.pitch) % a.pitch);   // b's column relative to a's
  return d < a.bytes || d + b.bytes > a.pitch;
}
static int check_planes(const char* who, const pg_plane* planes, int n_planes, long pages) {
  PG_REQUIRE(planes && n_planes >= 1 && n_planes <= PG_MAX_PLANES, "%s: %d planes outside [1,%d]", who, n_planes, PG_MAX_PLANES);
  for (int i = 0; i < n_planes; ++i) {
    PG_REQUIRE(planes[i].bytes >= 1 && planes[i].pitch >= planes[i].bytes, "%s: plane %d has %ld bytes at a pitch of %ld", who, i,
               planes[i].bytes, planes[i].pitch);
    PG_REQUIRE(pages == 0 || planes[i].base, "%s: plane %d is NULL", who, i);
    for (int j = 0; j < i; ++j)
      PG_REQUIRE(!planes_share(planes[i], pages, planes[j], pages), "%s: planes %d and %d share bytes", who, j, i);
  }
  return PG_OK;
}

// In place: a thread owns one byte column of a group's K pages, reads what moves before it writes, so any parents will do.
__global__ __launch_bounds__(256) void pages_reorder_kernel(Planes pl, int K, const int32_t* __restrict__ parents) {
  const pg_plane p = pl.p[blockIdx.y];
  const long g = blockIdx.x;
  unsigned char* base = (unsigned char*)p.base + g * K * p.pitch;
  for (long c = threadIdx.x; c < p.bytes; c += blockDim.x) {
    unsigned char v[PG_MAX_BEAMS];
#pragma unroll
    for (int j = 0; j < PG_MAX_BEAMS; ++j)
      if (j < K) {
        const unsigned from = parents[g * K + j];
        v[j] = base[(from < (unsigned)K ? from : j) * p.pitch + c];
      }
#pragma unroll
    for (int j = 0; j < PG_MAX_BEAMS; ++j)
      if (j < K) base[j * p.pitch + c] = v[j];
  }
}

__global__ __launch_bounds__(256) void pages_fork_kernel(Planes dst, Planes src, int n_src, const int32_t* __restrict__ index) {
  const pg_plane d = dst.p[blockIdx.y], s = src.p[blockIdx.y];
  const long i = blockIdx.x;
  const unsigned from = index[i];
  if (from >= (unsigned)n_src) return;
  const unsigned char* x = (const unsigned char*)s.base + from * s.pitch;
  unsigned char* y = (unsigned char*)d.base + i * d.pitch;
  for (long c = threadIdx.x; c < d.bytes; c += blockDim.x) y[c] = x[c];
}

// One workgroup: count, then the map and move[i] = the page that goes to the i-th dead place below count, dead[i].
__global__ __launch_bounds__(1024) void pages_plan_kernel(int n, const uint8_t* __restrict__ live, int32_t* __restrict__ count,
                                                          int32_t* __restrict__ map, int32_t* __restrict__ dead,
                                                          int32_t* __restrict__ move) {
  __shared__ int part[1024];
  const int tid = threadIdx.x;
  const long per = (n + 1023L) / 1024, p0 = min((long)n, tid * per), p1 = min((long)n, p0 + per);
  int mine = 0;
  for (long p = p0; p < p1; ++p) mine += live[p] != 0;
  part[tid] = mine;
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    const int add = tid >= o ? part[tid - o] : 0;
    __syncthreads();
    part[tid] += add;
    __syncthreads();
  }
  const int total = part[1023];
  if (tid == 0) count[0] = total;
  // live pages before p0, and (for the pages at or behind count) live pages in [count, p0): the moves are as many as the dead
  // places below count, and the live pages below count are count less that
  int before = part[tid] - mine;
  __shared__ int low;
  if (tid == 0) low = 0;
  __syncthreads();
  int below = 0;
  for (long p = p0; p < p1 && p < total; ++p) below += live[p] != 0;
  atomicAdd(&low, below);
  __syncthreads();
  for (long p = p0; p < p1; ++p) {
    const bool l = live[p] != 0;
    if (p < total) {
      if (!l) dead[p - before] = (int)p;
      map[p] = l ? (int)p : -1;
    } else if (l) move[before - low] = (int)p;
    else map[p] = -1;
    before += l;
  }
  __syncthreads();
  for (int i = tid; i < total - low; i += 1024) map[move[i]] = dead[i];
}
__global__ __launch_bounds__(256) void pages_move_kernel(Planes pl, int n, const int32_t* __restrict__ count,
                                                         const int32_t* __restrict__ map, const int32_t* __restrict__ move) {
  const pg_plane p = pl.p[blockIdx.y];
  const long old = (long)count[0] + blockIdx.x;       // pages at or behind count
  if (old >= n) return;
  const int to = map[old];
  if (to < 0) return;
  const unsigned char* x = (const unsigned char*)p.base + old * p.pitch;
  unsigned char* y = (unsigned char*)p.base + to * p.pitch;
  for (long c = threadIdx.x; c < p.bytes; c += blockDim.x) y[c] = x[c];
}

extern "C" int pg_pages_reorder(const pg_plane* planes, int n_planes, int n_groups, int K, const int32_t* parents, void* stream) {
  PG_REQUIRE(n_groups >= 0 && K >= 1 && K <= PG_MAX_BEAMS, "pg_pages_reorder: n_groups=%d or K=%d outside [1,%d]", n_groups, K,
             PG_MAX_BEAMS);
  PG_TRY(check_planes("pg_pages_reorder", planes, n_planes, (long)n_groups * K));
  if (n_groups == 0) return PG_OK;
  PG_REQUIRE(parents, "pg_pages_reorder: parents is NULL");
  Planes pl;
  memcpy(pl.p, planes, n_planes * sizeof(pg_plane));
  hipLaunchKernelGGL(pages_reorder_kernel, dim3(n_groups, n_planes), dim3(256), 0, (hipStream_t)stream, pl, K, parents);
  PG_CHECK_LAUNCH();
  return PG_OK;
}

extern "C" int pg_pages_fork(const pg_plane* dst, const pg_plane* src, int n_planes, int n_dst, int n_src, const int32_t* index,
                             void* stream) {
  PG_REQUIRE(n_dst >= 0 && n_src >= 0, "pg_pages_fork: n_dst=%d, n_src=%d", n_dst, n_src);
  PG_TRY(check_planes("pg_pages_fork: dst", dst, n_planes, n_dst));
  PG_REQUIRE(src, "pg_pages_fork: src is NULL");
  for (int i = 0; i < n_planes; ++i) {
    PG_REQUIRE(src[i].bytes == dst[i].bytes && src[i].pitch >= src[i].bytes, "pg_pages_fork: plane %d has %ld bytes in dst, %ld at a pitch of %ld in src",
               i, dst[i].bytes, src[i].bytes, src[i].pitch);
    PG_REQUIRE(n_src == 0 || src[i].base, "pg_pages_fork: plane %d of src is NULL", i);
    for (int j = 0; j < n_planes; ++j)
      PG_REQUIRE(!planes_share(dst[j], n_dst, src[i], n_src), "pg_pages_fork: plane %d of dst shares bytes with plane %d of src", j, i);
  }
  if (n_dst == 0 || n_src == 0) return PG_OK;
  PG_REQUIRE(index, "pg_pages_fork: index is NULL");
  Planes d, s;
  memcpy(d.p, dst, n_planes * sizeof(pg_plane));
  memcpy(s.p, src, n_planes * sizeof(pg_plane));
  hipLaunchKernelGGL(pages_fork_kernel, dim3(n_dst, n_planes), dim3(256), 0, (hipStream_t)stream, d, s, n_src, index);
  PG_CHECK_LAUNCH();
  return PG_OK;
}

extern "C" size_t pg_pages_compact_workspace_bytes(int n_pages) { return n_pages < 1 ? 256 : align_up((size_t)n_pages * 4, 256) * 2; }

extern "C" int pg_pages_compact(const pg_plane* planes, int n_planes, int n_pages, const uint8_t* live, int32_t* count, int32_t* map,
                                void* ws, size_t ws_bytes, void* stream) {
  PG_REQUIRE(n_pages >= 0, "pg_pages_compact: n_pages=%d", n_pages);
  PG_TRY(check_planes("pg_pages_compact", planes, n_planes, n_pages));
  PG_REQUIRE(count && (n_pages == 0 || (live && map)), "pg_pages_compact: NULL buffer");
  if (ws == nullptr || ws_bytes < pg_pages_compact_workspace_bytes(n_pages))
    PG_FAIL(PG_ERR_WORKSPACE, "pg_pages_compact: workspace too small (%zu < %zu)", ws_bytes, pg_pages_compact_workspace_bytes(n_pages));
  Planes pl;
  memcpy(pl.p, planes, n_planes * sizeof(pg_plane));
  int32_t *dead = at<int32_t>(ws, 0), *move = at<int32_t>(ws, align_up((size_t)n_pages * 4, 256));
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(1024), 0, st, n_pages, live, count, map, dead, move);
  PG_CHECK_LAUNCH();
  if (n_pages == 0) return PG_OK;
  hipLaunchKernelGGL(pages_move_kernel, dim3(n_pages, n_planes), dim3(256), 0, st, pl, n_pages, count, map, move);
  PG_CHECK_LAUNCH();
  return PG_OK;
}
