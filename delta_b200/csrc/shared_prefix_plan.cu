// The plan of the attention over shared prefixes (shared_prefix.cuh): one block, a thread per group and per row.  Everything that comes
// from the device's tables is checked here, so the kernels that follow the plan stay inside their tensors (page ids they check
// themselves).  The tables are asked for at once; then it is two scans over the block and a search for every range and piece.
#include "shared_prefix.cuh"

namespace {
using namespace shared_prefix;
constexpr int THREADS = 1024;
static_assert(THREADS >= MAX_ROWS && THREADS > MAX_GROUPS, "a thread per row and per group");

struct Shared {
  int member[MAX_ROWS];                                 // a row's place in members, -1: of no group
  int start[MAX_GROUPS + 1], prefix[MAX_GROUPS];
  int tile[MAX_GROUPS + 1], seg[MAX_GROUPS + 1];        // groups: first tile and first segment in their line
  int own[MAX_ROWS], len[MAX_ROWS];                     // keys read with the group, all keys
  int piece[MAX_ROWS + 1];                              // rows: first piece
  int warp[3][33];
};

// The last place whose value is not above v; a[0] <= v.
__device__ __forceinline__ int last_not_above(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Sums over the threads before this one of N values, and over all; one sync.
template <int N>
__device__ __forceinline__ void scan(const int (&v)[N], int (&before)[N], int (&total)[N], int (*s)[33], int tid) {
  const int lane = tid & 31, warp = tid >> 5;
  int to[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    to[i] = v[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, to[i], o);
      if (lane >= o) to[i] += a;
    }
    if (lane == 31) s[i][warp] = to[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int w = s[i][lane];                     // THREADS / 32 = 32 warps
    int sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += a;
    }
    sum = __shfl_sync(0xffffffffu, w, 31);
    const int mine = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
    before[i] = mine + to[i] - v[i];
    total[i] = sum;
  }
}

__global__ void __launch_bounds__(THREADS) shared_prefix_plan_kernel(const DkSharedPrefixParams p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, G = p.H / p.KV, rpt = p.qr / G, max_keys = p.max_pages * p.ps;
  const Plan plan(p);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int member = tid < p.n_members && p.groups > 0 ? p.members[tid] : -1;
  int len = tid < p.rows ? p.kv_len[tid] : 0;
  int a = 0, b = 0, k = 0;
  if (tid <= p.groups && p.groups > 0) a = p.group_start[tid];
  if (tid < p.groups) {
    b = p.group_start[tid + 1];
    k = p.group_prefix[tid];
  }
  s.member[tid] = -1;
  if (tid <= p.groups) {
    if (a < 0 || a > p.n_members || (tid < p.groups && (b < a || b > p.n_members || k < 0 || k > max_keys))) {
      const bool at_start = a < 0 || a > p.n_members, at_end = b < a || b > p.n_members;
      dk_report(p.err, DK_DEV_BAD_GROUP, tid, at_start ? a : at_end ? b : k, at_start || at_end ? p.n_members : max_keys);
      a = min(max(a, 0), p.n_members);
      b = a;
      k = 0;
    }
    s.start[tid] = a;
    // one row shares nothing, and what saves few keys is read by each row itself
    if (tid < p.groups) s.prefix[tid] = (long long)(b - a - 1) * k >= max(p.min_saved, 1) ? k / p.ps * p.ps : 0;
  }
  __syncthreads();
  if (tid < p.n_members && p.groups > 0 && tid >= s.start[0] && tid < s.start[p.groups] &&
      (member < 0 || member >= p.rows || atomicCAS(&s.member[member], -1, tid) != -1))
    dk_report(p.err, DK_DEV_BAD_GROUP, last_not_above(s.start, p.groups, tid), member, p.rows);
  __syncthreads();
  // a group's segments and the tiles of each, a row's tiles
  const int n = tid < p.groups ? s.start[tid + 1] - s.start[tid] : 0, shared = tid < p.groups ? s.prefix[tid] : 0;
  const int g_segs = n > 0 && shared > 0 ? cdiv(n, rpt) * p.KV : 0, g_tiles = g_segs > 0 ? cdiv(shared, p.kt) : 0;
  int own = 0, row_tiles = 0;
  if (tid < p.rows) {
    const int m = s.member[tid];
    int declared = 0;
    if (m >= 0) {
      const int g = last_not_above(s.start, p.groups, m);
      if (m - s.start[g] < s.start[g + 1] - s.start[g]) {
        own = s.prefix[g];
        declared = own > 0 ? own : min(max(p.group_prefix[g], 0), max_keys) / p.ps * p.ps;
      }
    }
    if (len < declared || len > max_keys) {
      dk_report(p.err, DK_DEV_BAD_GROUP, tid, len, len < declared ? declared : max_keys);
      len = own;
    }
    row_tiles = max(1, cdiv(len - own, p.rows_kt));       // a row without a key of its own has an empty piece
    s.own[tid] = own;
    s.len[tid] = len;
  }
  const int v[3] = {g_segs * g_tiles, g_segs, row_tiles};
  int before[3], total[3];
  scan<3>(v, before, total, s.warp, tid);
  const int Q = max(1, min(cdiv(total[0], p.grid), CAP)), ranges = cdiv(total[0], Q);
  const int C = max(MIN_ROW_TILES, cdiv(total[2] * p.KV, p.rows_grid));
  if (tid <= p.groups) {
    s.tile[tid] = before[0];
    s.seg[tid] = before[1];
  }
  __syncthreads();       // (the sums of the warps are read before they are written again)
  const int row_pieces = tid < p.rows ? cdiv(row_tiles, C) : 0;
  const int v2[1] = {row_pieces * p.KV};
  int before2[1], total2[1];
  scan<1>(v2, before2, total2, s.warp, tid);
  if (tid < p.rows) {
    s.piece[tid] = before2[0];
    plan.rows[2 * tid] = before2[0];
    plan.rows[2 * tid + 1] = row_pieces;
  }
  if (tid == 0) {
    plan.head[0] = ranges;
    plan.head[1] = total2[0];
  }
  __syncthreads();
  // groups: a thread per range walks the segments it holds
  for (int r = tid; r < ranges; r += THREADS) {
    int lo = r * Q;
    const int hi = min(total[0], lo + Q);
    int g = last_not_above(s.tile, p.groups, lo);          // the last one: groups without tiles before it start at the same place
    const int first_seg = s.seg[g] + (lo - s.tile[g]) / cdiv(s.prefix[g], p.kt);
    int seg = first_seg;
    while (lo < hi) {
      const int tiles = cdiv(s.prefix[g], p.kt), i = seg - s.seg[g], j0 = lo - s.tile[g] - i * tiles, j1 = min(tiles, j0 + hi - lo);
      const int m0 = s.start[g] + i / p.KV * rpt, row = p.members[m0];
      GroupPiece x;
      x.first = m0;
      x.rows = min(rpt, s.start[g + 1] - m0);
      x.kvh = i % p.KV;
      x.id = seg + r;
      x.key0 = j0 * p.kt;
      x.limit = min(s.prefix[g], j1 * p.kt);
      x.table_row = row >= 0 && row < p.rows ? row : 0;    // (recorded above)
      x.unused = 0;
      plan.group_pieces[seg + r] = x;
      lo += j1 - j0;
      ++seg;
      if (lo < hi)
        while (seg >= s.seg[g + 1]) ++g;                   // there is a later segment, so this ends at its group
    }
    plan.ranges[2 * r] = first_seg + r;
    plan.ranges[2 * r + 1] = seg - first_seg;
  }
  // rows: a thread per piece
  for (int id = tid; id < total2[0]; id += THREADS) {
    const int row = last_not_above(s.piece, p.rows, id);
    const int shared_keys = s.own[row], keys = s.len[row], tiles = max(1, cdiv(keys - shared_keys, p.rows_kt)), pieces = cdiv(tiles, C), per = cdiv(tiles, pieces);
    const int kvh = (id - s.piece[row]) / pieces, i = (id - s.piece[row]) % pieces;
    RowPiece x;
    x.row = row;
    x.kvh = kvh;
    x.key0 = min(keys, shared_keys + i * per * p.rows_kt);
    x.limit = min(keys, shared_keys + (i + 1) * per * p.rows_kt);
    x.index = i;
    x.pieces = pieces;
    x.first_id = id - i;
    x.group_id = x.group_n = x.r0 = x.unused[0] = x.unused[1] = 0;
    if (shared_keys > 0) {
      const int m = s.member[row], g = last_not_above(s.start, p.groups, m), at = m - s.start[g], t = cdiv(shared_keys, p.kt), seg = at / rpt * p.KV + kvh;
      const int first = s.tile[g] + seg * t, f = first / Q;
      x.group_id = s.seg[g] + seg + f;
      x.group_n = (first + t - 1) / Q - f + 1;
      x.r0 = at % rpt * G;
    }
    plan.row_pieces[id] = x;
  }
}
}  // namespace

int dk_shared_prefix_plan_launch(const DkSharedPrefixParams& p, cudaStream_t stream) {
  shared_prefix_plan_kernel<<<1, THREADS, 0, stream>>>(p);
  return dk_check_launch("shared_prefix_plan");
}
