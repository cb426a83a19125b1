// How the attention over shared prefixes cuts its work: the arguments, the pieces and where the partial results lie.
//
// Work comes in segments.  A segment of a group is a tile of its queries (``rpt`` rows with their G query heads of one
// key-value head) over the group's shared keys; a segment of a row is its G query heads over the keys it holds alone.  A segment
// is walked in tiles of keys, and cut into pieces of whole tiles:
//
//   groups  the tiles of all segments stand in one line, which is cut into ranges of Q tiles, as many as blocks run at once: every block
//           has the same number of tiles whatever the groups are, and at most one segment is cut at each border.  A piece is what a
//           range holds of a segment, and its number is segment + range: every step from one piece to the next moves to the next
//           segment or the next range, so no two pieces have one number and those of a segment follow one another.
//   rows    every segment is cut into equal pieces of at most C tiles, numbered through, and a block takes every ``grid``-th.  C is what
//           levels the blocks, but a number of its own for each kernel at least: the pieces of a cut segment go through memory, which takes as long as several tiles.
//
// All this is worked out on the device from the tables, so that a captured call follows them.  Whatever comes from the tables is checked here, so
// the kernels stay inside their tensors (page ids they check themselves).
#pragma once
#include "common.cuh"

#define DK_DEV_BAD_GROUP 5

struct DkSharedPrefixParams {
  const void* q;             // row r, head h at q + r * q_stride + h * hd
  void* out;                 // the same with out_stride
  const void* kv;            // [num_pages, 2, KV, ps, hd]
  const int* block_table;    // [rows, max_pages]
  const int* kv_len;         // [rows] keys each row reads
  const int* members;        // [n_members] rows, group by group
  const int* group_start;    // [groups + 1] first member of each group
  const int* group_prefix;   // [groups] shared keys (rounded down to whole pages)
  float* work;               // the rows' pieces, counters, the pieces' results
  int* err;                  // device error record, 4 ints; or null
  long long q_stride, out_stride;   // elements
  int rows, groups, n_members, H, KV, hd, ps, max_pages, num_pages, dtype;
  float scale;
  unsigned long long call;          // set by the launcher: what says that this call's list of the rows' pieces is there (attention_shared_prefix_rows.cu)
  // set by the launcher: how the work is cut (queries and keys of a group's tile, keys of a row's), query heads of a key-value head, rows of a
  // group's tile, the blocks that compute, the most pieces there can be, the keys that a group must save for its prefix to be read apart, and the tiles that a range of long segments has at least
  // (and the tiles that the groups may have together: where the tables ask for more, every row reads its keys alone)
  int qr, kt, rows_kt, G, rpt, grid, rows_grid, group_pieces, row_pieces, min_saved, least_tiles, max_tiles;
};

namespace shared_prefix {
constexpr int MAX_ROWS = 1024, MAX_GROUPS = 1023, MAX_G = 32;
constexpr int CAP = 48;            // tiles of a range, so also the most pieces of one
constexpr int NOBODY = 0x7fffffff;

__host__ __device__ constexpr int cdiv(int a, int b) { return (a + b - 1) / b; }
// the same for a that seldom passes b (a division by a number the compiler does not know takes some hundred cycles)
__device__ __forceinline__ int few(int a, int b) { return a <= 0 ? 0 : a <= b ? 1 : cdiv(a, b); }
__host__ __device__ constexpr int round4(int a) { return (a + 3) / 4 * 4; }

// A piece of a group: the first member's place in ``members``, how many rows, the key-value head, its number, the first key, the key behind the last,
// the row whose table is read.
struct __align__(16) GroupPiece {
  int first, rows, kvh, id, key0, limit, table_row, unused;
};
// A piece of a row: its place among its segment's pieces, how many those are and the first one's number; the pieces of its group's segment (first number,
// how many: 0 for none) and the row's first query in them.
struct __align__(16) RowPiece {
  int row, kvh, key0, limit, index, pieces, first_id, group_id, group_n, r0, unused[2];
};
constexpr int ROW_INTS = sizeof(RowPiece) / 4;

// Floats of one piece's results: of a group as [hd / 4 + 1][queries][4] (neighbouring queries lie side by side; the last row of four holds maximum and
// sum, then nothing); of a row as [query][hd], then {maximum, sum} per query.
__host__ __device__ __forceinline__ long long group_piece_floats(int qr, int hd) { return (long long)qr * (hd + 4); }
__host__ __device__ __forceinline__ long long row_piece_floats(int G, int hd) { return ((long long)G * (hd + 2) + 3) / 4 * 4; }

// The work buffer: how many pieces the rows have, nothing, the call whose list this is (64 bits), their records, a counter per row and key-value head, the results of groups' pieces, of rows' pieces.
__host__ __device__ __forceinline__ long long front_ints(const DkSharedPrefixParams& p) { return 4 + (long long)p.row_pieces * ROW_INTS; }
// Fills in the most pieces that there can be with these sizes, whatever the device's tables say, and tells what they need.
// Groups of n_g rows and k_g keys have ceil(n_g / rpt) ceil(k_g / kt) tiles for a key-value head, at most (n_g / rpt + 1) (k_g / kt + 1).  Their pages are
// distinct, or some are held by two groups (a part of all rows shares more than all do): sum k_g <= 2 pool.  So the sum is at most
// (n / rpt + 2 pool / longest) longest / kt and a tile for every segment, which is what the working memory is made for.  Tables that ask for more are right all the
// same: their rows read alone.  (64 rows with tables of 131,072 tokens, 32 heads on 8 of 128, a pool of 262,144 tokens: 90 MB; with 32 groups of full tables 412.)
struct Bounds {
  long long tiles, pieces, work_floats;
};
static inline Bounds bounds(DkSharedPrefixParams& p) {
  Bounds b;
  const int G = p.G = p.H / p.KV, rpt = p.rpt = p.qr / G;
  const long long keys = (long long)p.max_pages * p.ps, segments = (long long)p.KV * (p.groups > 0 ? p.n_members / rpt + p.groups : 0);
  const long long pool = (long long)p.num_pages * p.ps, longest = keys < pool ? keys : pool, any = segments * ((keys + p.kt - 1) / p.kt);
  const long long held = segments + p.KV * ((p.n_members + rpt - 1) / rpt * ((longest + p.kt - 1) / p.kt) + (2 * pool + p.kt - 1) / p.kt);
  const long long of_groups = any < held ? any : held, capped = (of_groups + CAP - 1) / CAP;
  const long long ranges = capped > p.grid ? capped : (of_groups < p.grid ? of_groups : (long long)p.grid);      // (no range is empty)
  const long long group_pieces = segments > 0 ? segments + ranges : 0;
  const long long row_pieces = (long long)p.rows * p.KV + p.rows_grid;      // a segment's last piece, and tiles / C of full ones, which are no more than blocks
  p.max_tiles = (int)of_groups;
  b.tiles = any + (long long)p.rows * p.KV * ((keys + p.rows_kt - 1) / p.rows_kt);
  b.pieces = group_pieces + row_pieces;
  p.group_pieces = (int)group_pieces;
  p.row_pieces = (int)row_pieces;
  b.work_floats = front_ints(p) + round4(p.rows * p.KV) + group_pieces * group_piece_floats(p.qr, p.hd) + row_pieces * row_piece_floats(G, p.hd);
  return b;
}
__device__ __forceinline__ unsigned long long* list_of_call(const DkSharedPrefixParams& p) { return reinterpret_cast<unsigned long long*>(p.work + 2); }
__device__ __forceinline__ RowPiece* row_pieces(const DkSharedPrefixParams& p) { return reinterpret_cast<RowPiece*>(p.work + 4); }
__device__ __forceinline__ int* counters(const DkSharedPrefixParams& p) { return reinterpret_cast<int*>(p.work + front_ints(p)); }
__host__ __device__ __forceinline__ float* group_results(const DkSharedPrefixParams& p, int id) {
  return p.work + front_ints(p) + round4(p.rows * p.KV) + id * group_piece_floats(p.qr, p.hd);
}
__device__ __forceinline__ float* row_results(const DkSharedPrefixParams& p, int id) {
  return group_results(p, p.group_pieces) + id * row_piece_floats(p.H / p.KV, p.hd);
}

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

// The tables of a call in shared memory, checked, and how they are cut.
struct Cut {
  int *start, *prefix, *declared, *tile, *seg;      // groups: first member [groups + 1], keys read apart, keys said to be shared, first tile and segment in their line
  int *member, *len, *own, *piece;                  // rows: place in members (the first of several; NOBODY: of no group), keys, keys read with the group, first piece
  int* sums;
  int Q, tiles, ranges, C, pieces;                  // tiles of a range, tiles of the line, ranges; tiles of a row's piece, rows' pieces
  static __host__ __device__ constexpr int ints(int rows, int groups) { return 5 * groups + 1 + 4 * rows + 4 * 32; }
  __device__ __forceinline__ Cut(int* s, int rows, int groups)
      : start(s), prefix(start + groups + 1), declared(prefix + groups), tile(declared + groups), seg(tile + groups), member(seg + groups), len(member + rows),
        own(len + rows), piece(own + rows), sums(piece + rows) {}
};

// Tiles of a range, for a line of ``tiles`` in ``segments``.  Long segments are cut into ranges of up to ``least_tiles`` even where that leaves blocks
// idle: every piece is one more for the rows to read, eight at a time.  (Tensor cores, 8 rows x 4,096 keys, 1, 2 and 4 tiles a range: 21.6, 18.6 and 17.4 us.)
__device__ __forceinline__ int range_tiles(const DkSharedPrefixParams& p, int tiles, int segments) {
  return min(max(few(tiles, p.grid), min(p.least_tiles, tiles > 24 * segments ? 4 : max(1, few(tiles, 8 * segments)))), CAP);
}

// Sums of N values over the threads before this one, and over all; one sync.
template <int N, int NT, typename Sync>
__device__ __forceinline__ void scan(const int* v, int* before, int* total, int* s, int tid, Sync sync) {
  const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) before[i] = v[i];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int a = __shfl_up_sync(0xffffffffu, before[i], o);
      if (lane >= o) before[i] += a;
    }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (lane == 31) s[i * 32 + warp] = before[i];
    total[i] = 0;
    before[i] -= v[i];
  }
  sync();
  for (int w = 0; w < NT / 32; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = s[i * 32 + w];
      total[i] += x;
      if (w < warp) before[i] += x;
    }
}

// Fills in ``c`` by a block of NT threads.  KT, ROWS_KT: p.kt, p.rows_kt; MIN_ROW_TILES: the least C.  Ends with a sync.
// Starts of groups that are out of order or out of range could make groups overlap and pieces outnumber the work buffer, and groups that repeat the same pages
// may be more tiles than it has room for: then there is no group, and every row reads its keys alone.  So does a row that is shorter than its group's
// prefix; one whose length fits no table reads nothing.  A row that is named twice belongs to its first place: every block that works the tables out finds the same pieces.
template <int KT, int ROWS_KT, int MIN_ROW_TILES, int NT>
__device__ __forceinline__ void make_cut(const DkSharedPrefixParams& p, Cut& c, int tid) {
  const auto sync = [] { __syncthreads(); };
  const int max_keys = p.max_pages * p.ps;
  // what the steps below read is asked for at once
  const int m_first = tid < p.n_members && p.groups > 0 ? p.members[tid] : -1;
  for (int r = tid; r < p.rows; r += NT) {
    c.len[r] = p.kv_len[r];
    c.member[r] = NOBODY;
  }
  bool out_of_order = false;
  if (tid == 0) c.sums[0] = 0;
  sync();
  for (int g = tid; g <= p.groups; g += NT) {
    int a = 0, b = 0, k = 0;
    if (p.groups > 0) a = p.group_start[g];
    if (g < p.groups) {
      b = p.group_start[g + 1];
      k = p.group_prefix[g];
    }
    const bool at_start = a < 0 || a > p.n_members, at_end = g < p.groups && (b < a || b > p.n_members);
    out_of_order |= at_start || at_end;
    if (at_start || at_end || k < 0 || k > max_keys) {
      dk_report(p.err, DK_DEV_BAD_GROUP, g, at_start ? a : at_end ? b : k, at_start || at_end ? p.n_members : max_keys);
      k = 0;
    }
    c.start[g] = a;
    if (g < p.groups) {
      k = k / p.ps * p.ps;
      c.declared[g] = k;
      c.prefix[g] = (long long)(b - a - 1) * k >= p.min_saved ? k : 0;      // one row shares nothing, and what saves few keys is read by each row itself
      if (c.prefix[g] > 0) atomicAdd(&c.sums[0], few(b - a, p.rpt) * p.KV * cdiv(k, KT));
    }
  }
  if (__syncthreads_or(out_of_order) || c.sums[0] > p.max_tiles) {
    for (int g = tid; g <= p.groups; g += NT) {
      c.start[g] = 0;
      if (g < p.groups) c.declared[g] = c.prefix[g] = 0;
    }
    sync();
  }
  if (p.groups > 0) {
    const int end = c.start[p.groups];
    for (int m = tid; m < end; m += NT) {
      if (m < c.start[0]) continue;
      const int row = m == tid ? m_first : p.members[m];
      const int other = row < 0 || row >= p.rows ? -1 : atomicMin(&c.member[row], m);
      if (other != NOBODY) dk_report(p.err, DK_DEV_BAD_GROUP, last_not_above(c.start, p.groups, max(m, other)), row, p.rows);
    }
  }
  sync();
  // neighbouring threads take neighbouring groups and rows
  const int g_per = cdiv(p.groups, NT), g0 = min(p.groups, tid * g_per), g1 = min(p.groups, g0 + g_per);
  const int r_per = cdiv(p.rows, NT), r0 = min(p.rows, tid * r_per), r1 = min(p.rows, r0 + r_per);
  auto segments = [&](int g) {
    const int n = c.start[g + 1] - c.start[g];
    return c.prefix[g] > 0 ? few(n, p.rpt) * p.KV : 0;
  };
  int v[4] = {0, 0, 0, 0}, before[4], total[4];
  for (int g = g0; g < g1; ++g) {
    const int x = segments(g);
    v[0] += x * cdiv(c.prefix[g], KT);
    v[1] += x;
  }
  for (int r = r0; r < r1; ++r) {
    const int m = c.member[r];
    int len = c.len[r], own = 0, said = 0;
    if (m != NOBODY) {
      const int g = last_not_above(c.start, p.groups, m);
      if (m - c.start[g] < c.start[g + 1] - c.start[g]) {
        own = c.prefix[g];
        said = c.declared[g];
      }
    }
    if (len < said || len > max_keys) {
      dk_report(p.err, DK_DEV_BAD_GROUP, r, len, len < said ? said : max_keys);
      own = 0;
      if (len < 0 || len > max_keys) c.len[r] = len = 0;
    }
    c.own[r] = own;
    const int tiles = max(1, cdiv(len - own, ROWS_KT));       // a row without a key of its own has an empty piece
    c.piece[r] = tiles;
    v[2] += tiles;
    v[3] += cdiv(tiles, MIN_ROW_TILES) * p.KV;
  }
  scan<4, NT>(v, before, total, c.sums, tid, sync);
  c.tiles = total[0];
  c.Q = range_tiles(p, total[0], total[1]);
  c.ranges = cdiv(total[0], c.Q);
  c.C = total[2] * p.KV <= MIN_ROW_TILES * p.rows_grid ? MIN_ROW_TILES : cdiv(total[2] * p.KV, p.rows_grid);
  for (int g = g0; g < g1; ++g) {
    c.tile[g] = before[0];
    c.seg[g] = before[1];
    const int x = segments(g);
    before[0] += x * cdiv(c.prefix[g], KT);
    before[1] += x;
  }
  if (c.C != MIN_ROW_TILES) {
    sync();                     // (the sums were read)
    v[0] = 0;
    for (int r = r0; r < r1; ++r) v[0] += cdiv(c.piece[r], c.C) * p.KV;
    scan<1, NT>(v, before + 3, total + 3, c.sums, tid, sync);
  }
  c.pieces = total[3];
  for (int r = r0; r < r1; ++r) {
    const int n = cdiv(c.piece[r], c.C) * p.KV;
    c.piece[r] = before[3];
    before[3] += n;
  }
  sync();
}

// Segment that holds tile ``x`` of the groups' line.
template <int KT>
__device__ __forceinline__ int segment_at(const DkSharedPrefixParams& p, const Cut& c, int x) {
  const int g = last_not_above(c.tile, p.groups, x);       // the last one: groups without tiles before it start at the same place
  return c.seg[g] + (x - c.tile[g]) / cdiv(c.prefix[g], KT);
}
template <int KT>
__device__ __forceinline__ int range_pieces(const DkSharedPrefixParams& p, const Cut& c, int range, int& first_seg) {
  const int lo = range * c.Q, hi = min(c.tiles, lo + c.Q);
  first_seg = segment_at<KT>(p, c, lo);
  return segment_at<KT>(p, c, hi - 1) - first_seg + 1;
}
// What range ``range`` holds of segment ``seg``.
template <int KT>
__device__ __forceinline__ GroupPiece group_piece(const DkSharedPrefixParams& p, const Cut& c, int range, int seg) {
  const int lo = range * c.Q, hi = min(c.tiles, lo + c.Q), g = last_not_above(c.seg, p.groups, seg);
  const int tiles = cdiv(c.prefix[g], KT), i = seg - c.seg[g], a = c.tile[g] + i * tiles, qt = i < p.KV ? 0 : i / p.KV, m0 = c.start[g] + qt * p.rpt;
  const int row = p.members[m0];
  GroupPiece x;
  x.first = m0;
  x.rows = min(p.rpt, c.start[g + 1] - m0);
  x.kvh = i - qt * p.KV;
  x.id = seg + range;
  x.key0 = max(0, lo - a) * KT;
  x.limit = min(c.prefix[g], min(tiles, hi - a) * KT);
  x.table_row = row >= 0 && row < p.rows ? row : 0;        // (a row out of range was recorded)
  x.unused = 0;
  return x;
}
// Piece number ``id`` of the rows.
template <int KT, int ROWS_KT>
__device__ __forceinline__ RowPiece row_piece(const DkSharedPrefixParams& p, const Cut& c, int id) {
  const int row = last_not_above(c.piece, p.rows, id), shared = c.own[row], keys = c.len[row];
  const int tiles = max(1, cdiv(keys - shared, ROWS_KT)), pieces = few(tiles, c.C), per = pieces == 1 ? tiles : cdiv(tiles, pieces), at = id - c.piece[row];
  RowPiece x;
  x.row = row;
  x.kvh = pieces == 1 ? at : at / pieces;
  x.index = at - x.kvh * pieces;
  x.key0 = min(keys, shared + x.index * per * ROWS_KT);
  x.limit = min(keys, shared + (x.index + 1) * per * ROWS_KT);
  x.pieces = pieces;
  x.first_id = id - x.index;
  x.group_id = x.group_n = x.r0 = x.unused[0] = x.unused[1] = 0;
  if (shared > 0) {
    const int m = c.member[row], g = last_not_above(c.start, p.groups, m), i = m - c.start[g], qt = i < p.rpt ? 0 : i / p.rpt;
    const int t = cdiv(shared, KT), seg = qt * p.KV + x.kvh, a = c.tile[g] + seg * t, f = a / c.Q, l = (a + t - 1) / c.Q;
    x.group_id = c.seg[g] + seg + f;
    x.group_n = l - f + 1;
    x.r0 = (i - qt * p.rpt) * p.G;
  }
  return x;
}
}  // namespace shared_prefix
