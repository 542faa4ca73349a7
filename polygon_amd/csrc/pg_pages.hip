// Pages of a cache of decoder states: reorder inside groups, fork, compaction.
#include "pg_pages.h"
#include "pg_host.h"
#include <numeric>

// What a move kernel needs of a cache: its planes, and how their columns are dealt out to waves.  A lane takes 16 bytes, so a wave
// covers PG_SEG = 1024 bytes of one page, or - pages of at most 512 bytes - 64 / lanes neighbouring groups of pages at once
// (lanes: the power of two that holds one).  Units are counted in blocks of 64 groups: a block has 64 * segments units of a wide
// plane and `lanes` of a narrow one; first[] is where each plane's begin.
constexpr int PG_SEG = 1024;
struct Planes {
  pg_plane p[PG_MAX_PLANES];
  int first[PG_MAX_PLANES + 1];
  int lanes[PG_MAX_PLANES];        // 64: a wide plane
  int n;
};
static int make_planes(const char* who, const pg_plane* planes, int n, Planes* out) {
  long at = 0;
  for (int i = 0; i < n; ++i) {
    out->p[i] = planes[i];
    out->first[i] = (int)at;
    int lanes = 1;
    while (lanes < 64 && lanes * 16L < planes[i].bytes) lanes *= 2;
    out->lanes[i] = lanes;
    at += lanes == 64 ? 64 * ((planes[i].bytes + PG_SEG - 1) / PG_SEG) : lanes;
    PG_REQUIRE(at < (1L << 30), "%s: pages of more than 2^34 bytes", who);
  }
  out->first[n] = (int)at;
  out->n = n;
  return PG_OK;
}
static bool any_narrow(const Planes& pl) {
  for (int i = 0; i < pl.n; ++i)
    if (pl.lanes[i] < 64) return true;
  return false;
}
// MIX: some planes are narrow, and units are dealt out in blocks of 64 groups.  Otherwise group by group, with less arithmetic and
// fewer registers per wave.  Three planes of 2 KB and three of 1 KB, all wide, in blocks instead: reorder of 8192 groups of 4 56.5 us
// against 50.3, compaction of 8192 pages of 8 such rows 59.6 against 52.9.  Pages of 64 and 128 bytes by a wave per group and plane
// instead: reorder of 8192 groups of 8 11.4 us against 5.1; of 512 and 256 bytes 13.2 against 10.2 (64 groups: 3.8 against 4.4).
template <bool MIX> __host__ __device__ __forceinline__ long plane_units(const Planes& pl, long groups) {
  return MIX ? (groups + 63) / 64 * pl.first[pl.n] : groups * (pl.first[pl.n] / 64);
}

// Two planes of na and nb pages share bytes (or, where their pitches differ, may: then only planes are told apart whose columns
// differ in rows of the pitches' greatest common divisor, at which the pages of both recur).  A single page has no pitch.
static bool planes_share(const pg_plane& a, long na, const pg_plane& b, long nb) {
  if (na < 1 || nb < 1) return false;
  const uintptr_t a0 = (uintptr_t)a.base, b0 = (uintptr_t)b.base;
  if (a0 + (na - 1) * a.pitch + a.bytes <= b0 || b0 + (nb - 1) * b.pitch + b.bytes <= a0) return false;
  const uintptr_t row = std::gcd(na > 1 ? a.pitch : 0, nb > 1 ? b.pitch : 0);
  if (row == 0) return true;
  const long d = (long)(b0 >= a0 ? (b0 - a0) % row : (row - (a0 - b0) % row) % row);   // b's column relative to a's
  return d < a.bytes || d + b.bytes > (long)row;
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

// What a call reads as flags or indices, or writes beside the pages, lies outside them: workgroups move pages while others still
// read the indices.
static int check_apart(const char* who, const pg_plane* planes, int n_planes, long pages, const char* what, const void* at, long bytes) {
  for (int i = 0; i < n_planes; ++i)
    PG_REQUIRE(!planes_share(planes[i], pages, pg_plane{(void*)at, bytes, bytes}, bytes > 0), "%s: %s shares bytes with plane %d",
               who, what, i);
  return PG_OK;
}

// One lane's 16 bytes of a page, `left` >= 1 of them inside it.  Any alignment: the hardware takes unaligned wide accesses.
__device__ __forceinline__ uint4 page_load(const unsigned char* p, long left) {
  uint4 v = {0, 0, 0, 0};
  if (left >= 16) { __builtin_memcpy(&v, p, 16); return v; }
  int o = 0;
  if (left & 8) { __builtin_memcpy(&v.x, p, 4); __builtin_memcpy(&v.y, p + 4, 4); o = 8; }
  if (left & 4) { __builtin_memcpy(&v.z, p + o, 4); o += 4; }
  if (left & 2) { unsigned short h; __builtin_memcpy(&h, p + o, 2); v.w = h; o += 2; }
  if (left & 1) v.w |= (unsigned)p[o] << 16;
  return v;
}
__device__ __forceinline__ void page_store(unsigned char* p, long left, const uint4& v) {
  if (left >= 16) { __builtin_memcpy(p, &v, 16); return; }
  int o = 0;
  if (left & 8) { __builtin_memcpy(p, &v.x, 4); __builtin_memcpy(p + 4, &v.y, 4); o = 8; }
  if (left & 4) { __builtin_memcpy(p + o, &v.z, 4); o += 4; }
  if (left & 2) { const unsigned short h = (unsigned short)v.w; __builtin_memcpy(p + o, &h, 2); o += 2; }
  if (left & 1) p[o] = (unsigned char)(v.w >> 16);
}
// A lane's place in unit u: plane i (wave-uniform), group g, column col.  wide: g is the wave's (uniform).
struct Place {
  int i;
  bool wide;
  long g, col;
};
template <bool MIX> __device__ __forceinline__ Place unit_place(const Planes& pl, long u, int lane) {
  const int per = MIX ? pl.first[pl.n] : pl.first[pl.n] / 64;
  const long block = u / per;
  int r = (int)(u - block * per);
  if (!MIX) r *= 64;
  Place p;
  p.i = 0;
  while (p.i + 1 < pl.n && r >= pl.first[p.i + 1]) ++p.i;
  r -= pl.first[p.i];
  p.wide = !MIX || pl.lanes[p.i] == 64;
  if (!MIX) {
    p.g = block;
    p.col = (long)(r / 64) * PG_SEG + lane * 16;
  } else if (p.wide) {
    const int segs = (pl.first[p.i + 1] - pl.first[p.i]) / 64, q = r / segs;
    p.g = block * 64 + q;
    p.col = (long)(r - q * segs) * PG_SEG + lane * 16;
  } else {
    p.g = block * 64 + (r * 64 + lane) / pl.lanes[p.i];
    p.col = lane % pl.lanes[p.i] * 16;
  }
  return p;
}

// Moves of pages: R pages at a time in one column segment; every load of a wave is issued before its first store.
// REORDER: the R pages are a group's K (<= R) and the sources lie among them, so whatever the parents are no page is
// overwritten before all of the segment's sources are in registers, and no other wave touches this segment of the group.
// Pages that keep their state are not touched.  Fork: the R pages are consecutive pages of dst, their sources pages of src.
// Bound by HBM where pages are wide - 16 bytes per lane, up to R loads in flight per wave: half of 65536 pages of 9 KB moving in
// groups of 8 (604 MB) 118 us, 5.1 TB/s, a fork of 8192 pages to 65536 (679 MB) 128 us, 5.3 TB/s; a 1 GiB copy reaches 5.06.
template <int R, bool REORDER, bool MIX>
__global__ __launch_bounds__(256) void pages_move_kernel(Planes dst, Planes src, long groups, int K, long n_dst, unsigned n_src,
                                                         const int32_t* __restrict__ from, const int* __restrict__ groups_dev) {
  const int lane = threadIdx.x & 63;
  if (groups_dev) groups = min(groups, (long)*groups_dev);
  const long units = plane_units<MIX>(dst, groups);
  for (long u = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < units; u += (long)gridDim.x * 4) {
    const Place at = unit_place<MIX>(dst, u, lane);
    const long left = at.g < groups ? dst.p[at.i].bytes - at.col : 0;
    const long page0 = at.g * K, dp = dst.p[at.i].pitch, sp = REORDER ? dp : src.p[at.i].pitch;
    unsigned char* d = (unsigned char*)dst.p[at.i].base + page0 * dp + at.col;
    const unsigned char* s = REORDER ? d : (const unsigned char*)src.p[at.i].base + at.col;
    int f[R];
    uint4 v[R];
    if (at.wide) {          // one group: its sources are scalars
      const int mine = lane < K && at.g < groups && page0 + lane < n_dst ? from[page0 + lane] : -1;
#pragma unroll
      for (int j = 0; j < R; ++j) f[j] = __builtin_amdgcn_readlane(mine, j);
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const bool moves = j < K && (unsigned)f[j] < (REORDER ? (unsigned)K : n_src) && !(REORDER && f[j] == j);
        f[j] = moves ? f[j] : -1;
        if (f[j] >= 0 && left > 0) v[j] = page_load(s + f[j] * sp, left);
      }
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (f[j] >= 0 && left > 0) page_store(d + j * dp, left, v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < R; ++j) f[j] = j < K && left > 0 && page0 + j < n_dst ? from[page0 + j] : -1;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const bool moves = j < K && (unsigned)f[j] < (REORDER ? (unsigned)K : n_src) && !(REORDER && f[j] == j);
        f[j] = moves ? f[j] : -1;
        if (f[j] >= 0) v[j] = page_load(s + f[j] * sp, left);
      }
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (f[j] >= 0) page_store(d + j * dp, left, v[j]);
    }
  }
}
// waves of 4 per workgroup; more units than this many workgroups hold are taken in rounds
static int move_grid(long units) { return (int)std::min<long>((units + 3) / 4, 1 << 20); }

// ---- compaction -------------------------------------------------------------------------------------------------------
// With count live pages, the i-th dead page below count is filled by the i-th live page at or behind it: as few moves as there
// can be, and no page is both read and written.  before(p) = live pages before p gives every place at once: a dead p < count
// is hole number p - before(p), a live p >= count is mover number before(p) - before(count).

// the live flags of pages p0 .. p0+7 (those below n) as 8 bits
__device__ __forceinline__ unsigned live_bits8(const uint8_t* __restrict__ live, long p0, long n) {
  unsigned long long w = 0;
  if (p0 + 8 <= n) {
    __builtin_memcpy(&w, live + p0, 8);
    w |= w >> 4; w |= w >> 2; w |= w >> 1;
    w &= 0x0101010101010101ull;
    return (unsigned)((w * 0x0102040810204080ull) >> 56);   // byte i -> bit i
  }
  unsigned m = 0;
  for (int i = 0; i < 8; ++i)
    if (p0 + i < n && live[p0 + i]) m |= 1u << i;
  return m;
}
// sum over the workgroup of all threads before this one; *total = over all
template <int NT> __device__ __forceinline__ int block_before(int x, int* total, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(s, o);
    if (lane >= o) s += t;
  }
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int b = 0, t = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    b += w < wave ? part[w] : 0;
    t += part[w];
  }
  *total = t;
  return b + s - x;
}
// The moves ("groups" of one page), one wave per MV consecutive units: MV loads in flight, then the stores.
constexpr int MV = 4;
template <bool MIX, typename I>
__device__ __forceinline__ void move_pages(const Planes& pl, long moves, const I* hole, const I* mover) {
  const int lane = threadIdx.x & 63;
  const long units = plane_units<MIX>(pl, moves);
  for (long u = ((long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * MV; u < units; u += (long)gridDim.x * 4 * MV) {
    uint4 v[MV];
    unsigned char* to[MV];
    long left[MV];
#pragma unroll
    for (int j = 0; j < MV; ++j) {
      left[j] = 0;
      if (u + j < units) {
        const Place at = unit_place<MIX>(pl, u + j, lane);
        if (at.g < moves) {
          const pg_plane& p = pl.p[at.i];
          left[j] = p.bytes - at.col;
          to[j] = (unsigned char*)p.base + hole[at.g] * p.pitch + at.col;
          if (left[j] > 0) v[j] = page_load((const unsigned char*)p.base + mover[at.g] * p.pitch + at.col, left[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < MV; ++j)
      if (left[j] > 0) page_store(to[j], left[j], v[j]);
  }
}
static int compact_grid(const Planes& pl, bool mix, long n) {
  const long units = mix ? plane_units<true>(pl, n / 2) : plane_units<false>(pl, n / 2);
  return (int)std::max<long>(1, std::min<long>((units + 4 * MV - 1) / (4 * MV), 2048));
}

// Up to PLAN_PAGES pages: ONE launch, every workgroup works the plan out for itself (n flag bytes from L2, a scan, the moves'
// ends as 16-bit lists in LDS) and takes its share of the moves.  8192 pages of 72 KB, half live (302 MB): 66 us, 4.5 TB/s, some
// 5 us of it the plan; 64 pages 7 us.  Units in flight per wave (MV) 8: 76 us; 1024 or 4096 workgroups 72 and 76.
// 16384 is as many flags as 256 threads hold in 64 bits each, and up to there this is the faster way: pages of 2 KB, half live, 300
// pages 5.8 us against 9.4 with the plan in a launch of its own, 4096 pages 6.7 and 9.6, 16384 pages 12.8 and 19.7.
constexpr int PLAN_PAGES = 16384;
template <bool MIX>
__global__ __launch_bounds__(256) void pages_compact_kernel(Planes pl, int n, const int* __restrict__ n_dev,
                                                            const uint8_t* __restrict__ live, int32_t* __restrict__ count,
                                                            int32_t* __restrict__ map) {
  if (n_dev) n = min(n, *n_dev);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ unsigned long long bits[256];
  __shared__ int before[256], part[4], low_s;
  const int tid = threadIdx.x;
  const int per = n <= 2048 ? 8 : n <= 4096 ? 16 : n <= 8192 ? 32 : 64;      // flags per thread (n <= 256 * per)
  unsigned long long mine = 0;
  for (int i = 0; i < per && (long)tid * per + i < n; i += 8) mine |= (unsigned long long)live_bits8(live, (long)tid * per + i, n) << i;
  int total;
  const int b = block_before<256>(__popcll(mine), &total, part);
  bits[tid] = mine;
  before[tid] = b;
  // before(count): from the thread that owns page `count`; all of them if that is no page
  const int end = total - tid * per;                        // my first `end` pages lie below count
  if (tid == 0 && total == n) low_s = total;
  if (total < n && end >= 0 && end < per) low_s = b + __popcll(mine & ((1ull << end) - 1));
  __syncthreads();
  const int low = low_s, moves = total - low;
  unsigned short *hole = reinterpret_cast<unsigned short*>(smem), *mover = hole + n / 2;
  const unsigned long long below = end >= 64 ? ~0ull : end > 0 ? (1ull << end) - 1 : 0;
  const int own_n = min(per, n - tid * per);                // my flags
  const unsigned long long own = own_n >= 64 ? ~0ull : own_n > 0 ? (1ull << own_n) - 1 : 0;
  for (unsigned long long h = ~mine & below & own; h; h &= h - 1) {
    const int i = __ffsll(h) - 1;
    hole[tid * per + i - (b + __popcll(mine & ((1ull << i) - 1)))] = (unsigned short)(tid * per + i);
  }
  for (unsigned long long h = mine & ~below; h; h &= h - 1) {
    const int i = __ffsll(h) - 1;
    mover[b + __popcll(mine & ((1ull << i) - 1)) - low] = (unsigned short)(tid * per + i);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) count[0] = total;
  for (int p = blockIdx.x * 256 + tid; map && p < n; p += gridDim.x * 256) {
    const int t = p / per, i = p % per;
    const bool l = bits[t] >> i & 1;
    map[p] = !l ? -1 : p < total ? p : (int)hole[before[t] + __popcll(bits[t] & ((1ull << i) - 1)) - low];
  }
  move_pages<MIX>(pl, moves, hole, mover);
}

// More pages: the plan by one workgroup into the workspace, then the moves.  Bound by that workgroup's walk through the flags: pages of
// 4 bytes, half live, 65536 of them 61 us, 300000 267 us, a million 1.02 ms (pages of 2 KB: 66, 344 us and 1.31 ms).
__global__ __launch_bounds__(1024) void pages_plan_kernel(int n, const int* __restrict__ n_dev,
                                                          const uint8_t* __restrict__ live, int32_t* __restrict__ count,
                                                          int32_t* __restrict__ map, int32_t* __restrict__ moves,
                                                          int32_t* __restrict__ hole, int32_t* __restrict__ mover) {
  if (n_dev) n = min(n, *n_dev);
  __shared__ int part[16], part2[16];
  const int tid = threadIdx.x;
  const long per = ((n + 1023L) / 1024 + 7) / 8 * 8, p0 = min((long)n, tid * per), p1 = min((long)n, p0 + per);
  int mine = 0;
  for (long p = p0; p < p1; p += 8) mine += __popc(live_bits8(live, p, p1));
  int total, low;
  int before = block_before<1024>(mine, &total, part);
  int under = 0;
  for (long p = p0; p < p1 && p < total; p += 8) under += __popc(live_bits8(live, p, min(p1, (long)total)));
  block_before<1024>(under, &low, part2);
  if (tid == 0) { count[0] = total; moves[0] = total - low; }
  for (long p = p0; p < p1; p += 8) {
    const unsigned m = live_bits8(live, p, p1);
    for (int i = 0; i < 8 && p + i < p1; ++i) {
      const bool l = m >> i & 1;
      const long q = p + i;
      if (q < total) {
        if (!l) hole[q - before] = (int)q;
        if (map) map[q] = l ? (int)q : -1;
      } else if (l) mover[before - low] = (int)q;
      else if (map) map[q] = -1;
      before += l;
    }
  }
  __syncthreads();
  if (map)
    for (int i = tid; i < total - low; i += 1024) map[mover[i]] = hole[i];
}
template <bool MIX>
__global__ __launch_bounds__(256) void pages_compact_move_kernel(Planes pl, const int32_t* __restrict__ moves,
                                                                 const int32_t* __restrict__ hole, const int32_t* __restrict__ mover) {
  move_pages<MIX>(pl, moves[0], hole, mover);
}

int launch_pages_reorder(const pg_plane* planes, int n_planes, int n_groups, const int* groups_dev, int K, const int32_t* parents,
                         hipStream_t st) {
  Planes pl;
  PG_TRY(make_planes("pg_pages_reorder", planes, n_planes, &pl));
  const long pages = (long)n_groups * K;
  // R registers of 16 bytes per lane: the narrowest instantiation that holds the group
  const bool mix = any_narrow(pl);
  const int grid = move_grid(mix ? plane_units<true>(pl, n_groups) : plane_units<false>(pl, n_groups));
  auto go = [&](auto mixed, auto plain) {
    hipLaunchKernelGGL(mix ? mixed : plain, dim3(grid), dim3(256), 0, st, pl, pl, (long)n_groups, K, pages, 0u, parents, groups_dev);
  };
  if (K <= 8) go(pages_move_kernel<8, true, true>, pages_move_kernel<8, true, false>);
  else if (K <= 16) go(pages_move_kernel<16, true, true>, pages_move_kernel<16, true, false>);
  else go(pages_move_kernel<32, true, true>, pages_move_kernel<32, true, false>);
  PG_CHECK_LAUNCH();
  return PG_OK;
}
extern "C" int pg_pages_reorder(const pg_plane* planes, int n_planes, int n_groups, int K, const int32_t* parents, void* stream) {
  PG_REQUIRE(n_groups >= 0 && K >= 1 && K <= PG_MAX_BEAMS, "pg_pages_reorder: n_groups=%d or K=%d outside [1,%d]", n_groups, K,
             PG_MAX_BEAMS);
  PG_TRY(check_planes("pg_pages_reorder", planes, n_planes, (long)n_groups * K));
  if (n_groups == 0) return PG_OK;
  PG_REQUIRE(parents, "pg_pages_reorder: parents is NULL");
  PG_TRY(check_apart("pg_pages_reorder", planes, n_planes, (long)n_groups * K, "parents", parents, (long)n_groups * K * 4));
  return launch_pages_reorder(planes, n_planes, n_groups, nullptr, K, parents, (hipStream_t)stream);
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
  PG_TRY(check_apart("pg_pages_fork", dst, n_planes, n_dst, "index", index, n_dst * 4L));
  Planes d, s;
  PG_TRY(make_planes("pg_pages_fork", dst, n_planes, &d));
  PG_TRY(make_planes("pg_pages_fork", src, n_planes, &s));
  constexpr int R = 8;
  const long groups = cdiv(n_dst, R);
  const bool mix = any_narrow(d);
  const int grid = move_grid(mix ? plane_units<true>(d, groups) : plane_units<false>(d, groups));
  auto* kernel = mix ? pages_move_kernel<R, false, true> : pages_move_kernel<R, false, false>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, d, s, groups, R, (long)n_dst, (unsigned)n_src, index, (const int*)nullptr);
  PG_CHECK_LAUNCH();
  return PG_OK;
}

// number of moves | holes | movers (n / 2 of each at most)
static size_t compact_list_bytes(int n) { return align_up((size_t)n / 2 * 4 + 4, 256); }
extern "C" size_t pg_pages_compact_workspace_bytes(int n_pages) {
  return n_pages <= PLAN_PAGES ? 0 : 256 + 2 * compact_list_bytes(n_pages);
}

int launch_pages_compact(const pg_plane* planes, int n_planes, int n_pages, const int* n_dev, const uint8_t* live, int32_t* count,
                         int32_t* map, void* ws, hipStream_t st) {
  Planes pl;
  PG_TRY(make_planes("pg_pages_compact", planes, n_planes, &pl));
  const bool mix = any_narrow(pl);
  const int grid = compact_grid(pl, mix, n_pages);
  if (n_pages <= PLAN_PAGES) {
    auto* kernel = mix ? pages_compact_kernel<true> : pages_compact_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), (size_t)(n_pages / 2) * 4, st, pl, n_pages, n_dev, live, count, map);
    PG_CHECK_LAUNCH();
    return PG_OK;
  }
  int32_t *moves = at<int32_t>(ws, 0), *hole = at<int32_t>(ws, 256), *mover = at<int32_t>(ws, 256 + compact_list_bytes(n_pages));
  hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(1024), 0, st, n_pages, n_dev, live, count, map, moves, hole, mover);
  PG_CHECK_LAUNCH();
  auto* kernel = mix ? pages_compact_move_kernel<true> : pages_compact_move_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, pl, moves, hole, mover);
  PG_CHECK_LAUNCH();
  return PG_OK;
}
extern "C" int pg_pages_compact(const pg_plane* planes, int n_planes, int n_pages, const uint8_t* live, int32_t* count, int32_t* map,
                                void* ws, size_t ws_bytes, void* stream) {
  PG_REQUIRE(n_pages >= 0, "pg_pages_compact: n_pages=%d", n_pages);
  PG_TRY(check_planes("pg_pages_compact", planes, n_planes, n_pages));
  PG_REQUIRE(count && (n_pages == 0 || (live && map)), "pg_pages_compact: NULL buffer");
  const size_t need = pg_pages_compact_workspace_bytes(n_pages);
  if (ws_bytes < need || (need && !ws)) PG_FAIL(PG_ERR_WORKSPACE, "pg_pages_compact: workspace too small (%zu < %zu)", ws_bytes, need);
  const struct { const char* what; const void* at; size_t bytes; } beside[] = {
      {"live", live, (size_t)n_pages}, {"count", count, 4}, {"map", map, n_pages * 4ul}, {"the workspace", ws, need}};
  for (const auto& b : beside) {
    PG_TRY(check_apart("pg_pages_compact", planes, n_planes, n_pages, b.what, b.at, (long)b.bytes));
    for (const auto* o = beside; o < &b; ++o)
      PG_REQUIRE((uintptr_t)o->at + o->bytes <= (uintptr_t)b.at || (uintptr_t)b.at + b.bytes <= (uintptr_t)o->at || !o->bytes || !b.bytes,
                 "pg_pages_compact: %s and %s share bytes", o->what, b.what);
  }
  return launch_pages_compact(planes, n_planes, n_pages, nullptr, live, count, map, ws, (hipStream_t)stream);
}
