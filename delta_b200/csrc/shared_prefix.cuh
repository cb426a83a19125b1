// How the attention over shared prefixes cuts its work: the arguments, the lists of pieces that blocks take, and where the
// partial results lie.
//
// Work comes in segments.  A segment of a group is a tile of its queries (``rpt`` rows with their G query heads of
// one key-value head) over the group's shared keys; a segment of a row is its G query heads over the keys it holds
// alone.  A segment is walked in tiles of KT keys.  The tiles of all segments stand in one line, which is cut into ranges
// of Q tiles (as many ranges as blocks run at once): so every block has the same number of tiles whatever the prefixes, the
// rows and their lengths are, and at most one segment is cut at each border.  A piece is what a range holds of a segment.
// Pieces are numbered segment + range: every step from one piece to the next moves to the next segment or to the next
// range, so no two pieces have one number.
//
// The kernel on the FMA units has groups and rows in one line; on the tensor cores each has a line and a kernel of its own.
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
  float* work;               // row records and counters, then the pieces' partial results
  int* err;                  // device error record, 4 ints; or null
  long long q_stride, out_stride;   // elements
  int rows, groups, n_members, H, KV, hd, ps, max_pages, num_pages, dtype;
  float scale;
  // set by the launcher: blocks over the line of groups (or the only line) and over the line of rows, pieces of groups that the
  // work buffer holds, and the keys that a group must save for its prefix to be read apart
  int grid, rows_grid, group_pieces, min_saved;
};

namespace shared_prefix {
constexpr int MAX_ROWS = 1024, MAX_GROUPS = 1024, MAX_G = 32;
constexpr int CAP = 96;            // tiles of a range, so also the most pieces of one
constexpr int ROW_INTS = 8;        // a row's record for the merge

__host__ __device__ constexpr int cdiv(int a, int b) { return (a + b - 1) / b; }
__host__ __device__ constexpr int round4(int a) { return (a + 3) / 4 * 4; }

// Floats of one piece: of a group as [hd / 4][rows][4] (neighbouring rows lie side by side), then {maximum, sum} per row.
__host__ __device__ __forceinline__ long long group_piece_floats(int qr, int hd) { return (long long)qr * (hd + 2); }
__host__ __device__ __forceinline__ long long row_piece_floats(int G, int hd) { return ((long long)G * (hd + 2) + 3) / 4 * 4; }
// ints at the front of the work buffer: a record per row, a counter per row and key-value head
__host__ __device__ __forceinline__ int front_ints(int rows, int KV) { return round4(rows * ROW_INTS) + round4(rows * KV); }

// The most pieces there can be with these sizes, whatever the device's tables say.
struct Bounds {
  long long tiles, group_pieces, row_pieces, floats;
};
static inline Bounds bounds(const DkSharedPrefixParams& p, int qr, int kt, int grid, int rows_kt, int rows_grid) {
  Bounds b;
  const int G = p.H / p.KV, rpt = qr / G;
  const long long keys = (long long)p.max_pages * p.ps, segments = (long long)p.KV * (p.groups > 0 ? p.n_members / rpt + p.groups : 0);
  const long long of_groups = segments * ((keys + kt - 1) / kt), of_rows = (long long)p.rows * p.KV * ((keys + rows_kt - 1) / rows_kt);
  auto ranges = [&](long long n, int blocks) { return (n + CAP - 1) / CAP > blocks ? (n + CAP - 1) / CAP : (long long)blocks; };
  b.tiles = of_groups + of_rows;
  b.group_pieces = segments > 0 ? segments + ranges(of_groups, grid) : 0;
  b.row_pieces = (long long)p.rows * p.KV + ranges(b.tiles, rows_grid);
  b.floats = front_ints(p.rows, p.KV) + b.group_pieces * group_piece_floats(qr, p.hd) + b.row_pieces * row_piece_floats(G, p.hd);
  return b;
}
__device__ __forceinline__ int* row_record(const DkSharedPrefixParams& p, int row) { return reinterpret_cast<int*>(p.work) + row * ROW_INTS; }
__device__ __forceinline__ int* counters(const DkSharedPrefixParams& p) { return reinterpret_cast<int*>(p.work) + round4(p.rows * ROW_INTS); }
__device__ __forceinline__ float* group_piece(const DkSharedPrefixParams& p, int qr, int id) {
  return p.work + front_ints(p.rows, p.KV) + id * group_piece_floats(qr, p.hd);
}
__device__ __forceinline__ float* row_piece(const DkSharedPrefixParams& p, int qr, int id) {
  return group_piece(p, qr, p.group_pieces) + id * row_piece_floats(p.H / p.KV, p.hd);
}

// The tables of a call in shared memory.
struct Tables {
  int *member, *start, *prefix, *tile, *seg, *line;
  // [rows] the row's place in members, -1: of no group; [groups + 1]; [groups] keys that are read apart; [groups] first tile and segment in the
  // line of groups; what walk_line works in
  static __host__ __device__ constexpr int ints(int rows, int groups) { return rows + 4 * groups + 1 + 64 + 4; }
  __device__ __forceinline__ Tables(int* s, int rows, int groups)
      : member(s), start(s + rows), prefix(start + groups + 1), tile(prefix + groups), seg(tile + groups), line(seg + groups) {}
};

// The last group that starts at member m or before it.
__device__ __forceinline__ int group_of(const DkSharedPrefixParams& p, const Tables& t, int m) {
  int lo = 0, hi = p.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.start[mid] <= m) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Starts and prefixes of the groups, checked.  ROWS: also each row's place among the members.  Ends with a sync.
template <bool ROWS, int NT, typename Sync>
__device__ void load_tables(const DkSharedPrefixParams& p, const Tables& t, int tid, Sync sync) {
  const int max_keys = p.max_pages * p.ps;
  // what the steps below read is asked for at once
  const int m_first = ROWS && tid < p.n_members ? p.members[tid] : -1;
  for (int g = tid; g <= p.groups; g += NT) {
    int a = 0, b = 0, k = 0;
    if (p.groups > 0) a = p.group_start[g];
    if (g < p.groups) {
      b = p.group_start[g + 1];
      k = p.group_prefix[g];
    }
    if (a < 0 || a > p.n_members || (g < p.groups && (b < a || k < 0 || k > max_keys))) {
      dk_report(p.err, DK_DEV_BAD_GROUP, g, a < 0 || a > p.n_members ? a : (b < a ? b : k), b < a ? p.n_members : max_keys);
      a = min(max(a, 0), p.n_members);
      k = 0;
    }
    t.start[g] = a;
    // one row shares nothing, and what saves few keys is read by each row itself
    if (g < p.groups) t.prefix[g] = (long long)(min(b, p.n_members) - a - 1) * k >= max(p.min_saved, 1) ? k / p.ps * p.ps : 0;
  }
  if (ROWS)
    for (int r = tid; r < p.rows; r += NT) t.member[r] = -1;
  sync();
  if (ROWS && p.groups > 0) {
    const int end = min(t.start[p.groups], p.n_members);
    for (int m = tid; m < end; m += NT) {
      if (m < t.start[0]) continue;
      const int row = m == tid ? m_first : p.members[m];
      if (row < 0 || row >= p.rows || atomicCAS(&t.member[row], -1, m) != -1) dk_report(p.err, DK_DEV_BAD_GROUP, group_of(p, t, m), row, p.rows);
    }
  }
  if (ROWS) sync();
}

// An entry of a line: a group or a row, with its segments and the tiles of each.
struct Entry {
  int segments, tiles;
};
template <int KT>
__device__ __forceinline__ Entry group_entry(const DkSharedPrefixParams& p, const Tables& t, int g, int rpt) {
  const int n = t.start[g + 1] - t.start[g], k = t.prefix[g];
  return n > 0 && k > 0 ? Entry{cdiv(n, rpt) * p.KV, cdiv(k, KT)} : Entry{0, 0};
}
// Keys that are read with the row's group, and all of its keys (checked).
__device__ __forceinline__ int row_prefix(const DkSharedPrefixParams& p, const Tables& t, int row) {
  const int m = t.member[row];
  if (m < 0) return 0;
  const int g = group_of(p, t, m);
  return m - t.start[g] < t.start[g + 1] - t.start[g] ? t.prefix[g] : 0;
}
__device__ __forceinline__ int row_keys(const DkSharedPrefixParams& p, const Tables& t, int row, int n, bool report) {
  const int m = t.member[row], max_keys = p.max_pages * p.ps;
  const int shared = m >= 0 ? min(max(p.group_prefix[group_of(p, t, m)], 0), max_keys) / p.ps * p.ps : 0;
  if (n < shared || n > max_keys) {
    if (report) dk_report(p.err, DK_DEV_BAD_GROUP, row, n, n < shared ? shared : max_keys);
    n = row_prefix(p, t, row);
  }
  return n;
}

struct Line {
  int pieces, total, Q;     // pieces of the range, tiles of the line, tiles of a range
  bool more;                // whether range + grid exists
};
// Walks a line of entries: ``at(e, x, tile, segment)`` for every entry by the thread that owns it, then, behind a sync, ``emit(e, x, i, segment,
// tile, j0, j1, place, Q)`` for segment i of entry e that the range holds from its tile j0 to j1, at ``place`` of the range's list.  Ends with a sync.
template <int NT, typename Sync, typename Of, typename At, typename Emit>
__device__ Line walk_line(int entries, int grid, int range, int* s, int tid, Sync sync, Of of, At at, Emit emit) {
  const int lane = tid & 31, warp = tid >> 5;
  const int per = cdiv(entries, NT), e0 = min(entries, tid * per), e1 = min(entries, e0 + per);
  int tiles = 0, segs = 0;
  for (int e = e0; e < e1; ++e) {
    const Entry x = of(e);
    tiles += x.segments * x.tiles;
    segs += x.segments;
  }
  int tiles_to = tiles, segs_to = segs;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, tiles_to, o), b = __shfl_up_sync(0xffffffffu, segs_to, o);
    if (lane >= o) {
      tiles_to += a;
      segs_to += b;
    }
  }
  if (lane == 31) {
    s[warp] = tiles_to;
    s[32 + warp] = segs_to;
  }
  if (tid == 0) s[64] = s[65] = -1;
  sync();
  Line l;
  l.total = 0;
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) {
      tiles_to += s[w];
      segs_to += s[32 + w];
    }
    l.total += s[w];
  }
  l.Q = max(1, min(cdiv(l.total, grid), CAP));
  const int lo = range * l.Q, hi = min(l.total, lo + l.Q);
  l.more = (range + grid) * l.Q < l.total;
  const int first_tile = tiles_to - tiles, first_seg = segs_to - segs;
  int a = first_tile, seg = first_seg;
  for (int e = e0; e < e1; ++e) {
    const Entry x = of(e);
    const int end = a + x.segments * x.tiles;
    if (a <= lo && lo < end) s[64] = seg + (lo - a) / x.tiles;
    if (a < hi && hi <= end) s[65] = seg + (hi - 1 - a) / x.tiles;
    at(e, x, a, seg);
    a = end;
    seg += x.segments;
  }
  sync();
  const int seg0 = s[64];
  l.pieces = lo < hi ? s[65] - seg0 + 1 : 0;
  a = first_tile;
  seg = first_seg;
  for (int e = e0; e < e1; ++e) {
    const Entry x = of(e);
    const int end = a + x.segments * x.tiles;
    if (lo < hi && x.segments > 0 && a < hi && end > lo) {
      const int i0 = max(0, (lo - a) / x.tiles), i1 = min(x.segments - 1, (hi - 1 - a) / x.tiles);
      for (int i = i0; i <= i1; ++i) {
        const int b = a + i * x.tiles;
        emit(e, x, i, seg + i, b, max(0, lo - b), min(x.tiles, hi - b), seg + i - seg0, l.Q);
      }
    }
    a = end;
    seg += x.segments;
  }
  sync();
  return l;
}

// A piece of a group, 16 bytes: x the place of its first member (bit 31 set), y key-value head, rows and number, z first key, w key behind the last.
// A piece of a row in the line of both: x the row.
struct Piece {
  int first, kvh, n_rows, id, key0, limit;
  bool of_group;
  __device__ __forceinline__ Piece(const int4& d)
      : first(d.x & 0x7fffffff), kvh(d.y & 255), n_rows((d.y >> 8) & 255), id((unsigned)d.y >> 16), key0(d.z), limit(d.w), of_group(d.x < 0) {}
};
template <int KT>
__device__ __forceinline__ int4 piece_of_group(const DkSharedPrefixParams& p, const Tables& t, int g, int rpt, int i, int id, int j0, int j1) {
  const int m0 = t.start[g] + i / p.KV * rpt, n = min(rpt, t.start[g + 1] - m0);
  return make_int4((int)(0x80000000u | (unsigned)m0), (i % p.KV) | (n << 8) | (id << 16), j0 * KT, min(t.prefix[g], j1 * KT));
}
}  // namespace shared_prefix
