// How the attention over shared prefixes cuts its work: the arguments, the list of pieces that a block takes, and
// where the partial results lie.  Used by the kernel on the FMA units, the one on the tensor cores and the merge.
//
// Work comes in segments.  A segment of a group is a tile of its queries (``rpt`` rows with their G query heads of
// one key-value head) over the group's shared keys; a segment of a row is its G query heads over the keys it holds
// alone.  A segment is walked in tiles of KT keys.  All tiles of all segments, groups first, stand in one line, which
// is cut into ranges of Q tiles (as many ranges as blocks run at once): so every block has the same number of tiles
// whatever the prefixes, the rows and their lengths are, and at most one segment is cut at each border.  A piece is
// what a range holds of a segment.  Pieces are numbered segment + range: every step from one piece to the next
// moves to the next segment or to the next range, so no two pieces have one number.
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
  float* work;               // row records, then the pieces' partial results
  int* err;                  // device error record, 4 ints; or null
  long long q_stride, out_stride;   // elements
  int rows, groups, n_members, H, KV, hd, ps, max_pages, num_pages, dtype;
  float scale;
  int grid, prefix_pieces;   // set by the launcher: blocks of the first kernel, pieces of groups that the work buffer holds
};

namespace shared_prefix {
constexpr int MAX_ROWS = 1024, MAX_GROUPS = 1024, MAX_G = 32;
constexpr int CAP = 96;            // tiles of a range, so also the most pieces of one
constexpr int ROW_INTS = 8;        // a row's record for the merge

// ints of shared memory that build() works in
__host__ __device__ constexpr int scratch_ints(int rows, int groups) { return rows + 4 * groups + 1 + 2 * 32 + 8; }
__host__ __device__ constexpr int cdiv(int a, int b) { return (a + b - 1) / b; }

struct Piece {
  int first;      // of a group: its first member's place in ``members``; of a row: the row
  int kvh, n_rows, id, key0, limit;
  bool of_group;
  __device__ __forceinline__ Piece(const int4& d)
      : first(d.x & 0x7fffffff), kvh(d.y & 255), n_rows((d.y >> 8) & 255), id((unsigned)d.y >> 16), key0(d.z), limit(d.w), of_group(d.x < 0) {}
};

// Floats of one piece: outputs as [hd / 4][rows][4] (neighbouring rows lie side by side), then {maximum, sum} per row.
__host__ __device__ __forceinline__ long long group_piece_floats(int qr, int hd) { return (long long)qr * (hd + 2); }
__host__ __device__ __forceinline__ long long row_piece_floats(int G, int hd) { return ((long long)G * (hd + 2) + 3) / 4 * 4; }

struct Bounds {
  long long tiles_of_groups, tiles, group_pieces, row_pieces, floats;
};
// The most there can be with these sizes, whatever the device's tables say.
static inline Bounds bounds(const DkSharedPrefixParams& p, int qr, int kt, int grid) {
  Bounds b;
  const int G = p.H / p.KV, rpt = qr / G;
  const long long keys = (long long)p.max_pages * p.ps, tiles = (keys + kt - 1) / kt;
  const long long segments = (long long)p.KV * (p.groups > 0 ? p.n_members / rpt + p.groups : 0);
  b.tiles_of_groups = segments * tiles;
  b.tiles = b.tiles_of_groups + (long long)p.rows * p.KV * tiles;
  auto ranges = [&](long long n) { return (n + CAP - 1) / CAP > grid ? (n + CAP - 1) / CAP : (long long)grid; };
  b.group_pieces = segments > 0 ? segments + ranges(b.tiles_of_groups) : 0;
  b.row_pieces = (long long)p.rows * p.KV + ranges(b.tiles);
  b.floats = ((long long)p.rows * ROW_INTS + 3) / 4 * 4 + b.group_pieces * group_piece_floats(qr, p.hd) + b.row_pieces * row_piece_floats(G, p.hd);
  return b;
}
__device__ __forceinline__ float* group_piece(const DkSharedPrefixParams& p, int qr, int id) {
  return p.work + (p.rows * ROW_INTS + 3) / 4 * 4 + id * group_piece_floats(qr, p.hd);
}
__device__ __forceinline__ float* row_piece(const DkSharedPrefixParams& p, int qr, int id) {
  return group_piece(p, qr, p.prefix_pieces) + id * row_piece_floats(p.H / p.KV, p.hd);
}

// Fills ``list`` with the pieces of range number ``range`` and returns how many there are; ``ranges_left`` tells whether a range
// ``range + grid`` exists.  Called by NT threads that can be synchronised with ``sync``; ``s`` holds scratch_ints ints.  With
// ``write_rows`` the rows' records for the merge are written too.
template <int KT, int NT, typename Sync>
__device__ int build(const DkSharedPrefixParams& p, int rpt, int range, int4* list, int* s, int tid, Sync sync, bool write_rows, bool& ranges_left) {
  int* s_member = s;                       // [rows] the row's place in members, -1: of no group
  int* s_start = s_member + p.rows;        // [groups + 1]
  int* s_prefix = s_start + p.groups + 1;  // [groups] shared keys
  int* s_tile = s_prefix + p.groups;       // [groups] first tile
  int* s_seg = s_tile + p.groups;          // [groups] first segment
  int* s_warp = s_seg + p.groups;          // [2][32]
  int* s_out = s_warp + 64;                // first segment of the range, last one, segments of groups
  const int lane = tid & 31, warp = tid >> 5;
  const int max_keys = p.max_pages * p.ps;
  for (int r = tid; r < p.rows; r += NT) s_member[r] = -1;
  for (int g = tid; g <= p.groups; g += NT) {
    int a = p.groups > 0 ? p.group_start[g] : 0;
    if (a < 0 || a > p.n_members) {
      dk_report(p.err, DK_DEV_BAD_GROUP, g, a, p.n_members);
      a = 0;
    }
    s_start[g] = a;
    if (g < p.groups) {
      int k = p.group_prefix[g];
      if (k < 0 || k > max_keys) {
        dk_report(p.err, DK_DEV_BAD_GROUP, g, k, max_keys);
        k = 0;
      }
      s_prefix[g] = k / p.ps * p.ps;
    }
  }
  if (tid == 0) s_out[0] = s_out[1] = -1;
  sync();
  auto group_of = [&](int m) {             // the last group that starts at m or before it
    int lo = 0, hi = p.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_start[mid] <= m) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  for (int g = tid; g < p.groups; g += NT)
    if (s_start[g + 1] < s_start[g]) dk_report(p.err, DK_DEV_BAD_GROUP, g, s_start[g + 1], s_start[g]);
  if (p.groups > 0)
    for (int m = s_start[0] + tid; m < s_start[p.groups]; m += NT) {
      const int row = p.members[m];
      if (row < 0 || row >= p.rows || atomicCAS(&s_member[row], -1, m) != -1) dk_report(p.err, DK_DEV_BAD_GROUP, group_of(m), row, p.rows);
    }
  sync();
  // An entry is a group or a row.  Neighbouring threads take neighbouring runs of entries.
  struct Entry {
    int segments, tiles, prefix, len;
  };
  auto entry = [&](int e, bool report) {
    Entry x = {0, 0, 0, 0};
    if (e < p.groups) {
      const int n = s_start[e + 1] - s_start[e];
      x.prefix = s_prefix[e];
      if (n > 0 && x.prefix > 0) {
        x.tiles = cdiv(x.prefix, KT);
        x.segments = cdiv(n, rpt) * p.KV;
      }
    } else {
      const int row = e - p.groups, m = s_member[row];
      x.prefix = m >= 0 ? s_prefix[group_of(m)] : 0;
      x.len = p.kv_len[row];
      if (x.len < x.prefix || x.len > max_keys) {
        if (report) dk_report(p.err, DK_DEV_BAD_GROUP, row, x.len, x.len < x.prefix ? x.prefix : max_keys);
        x.len = x.prefix;
      }
      x.tiles = cdiv(x.len - x.prefix, KT);
      x.segments = x.tiles > 0 ? p.KV : 0;
    }
    return x;
  };
  const int entries = p.groups + p.rows, per = cdiv(entries, NT);
  const int e0 = min(entries, tid * per), e1 = min(entries, e0 + per);
  int tiles = 0, segs = 0;
  for (int e = e0; e < e1; ++e) {
    const Entry x = entry(e, write_rows);
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
    s_warp[warp] = tiles_to;
    s_warp[32 + warp] = segs_to;
  }
  sync();
  int total = 0;
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) {
      tiles_to += s_warp[w];
      segs_to += s_warp[32 + w];
    }
    total += s_warp[w];
  }
  const int Q = max(1, min(cdiv(total, p.grid), CAP));
  const int lo = range * Q, hi = min(total, lo + Q);
  ranges_left = (range + p.grid) * Q < total;
  int at = tiles_to - tiles, seg = segs_to - segs;
  for (int e = e0; e < e1; ++e) {
    const Entry x = entry(e, false);
    const int end = at + x.segments * x.tiles;
    if (e < p.groups) {
      s_tile[e] = at;
      s_seg[e] = seg;
    }
    if (at <= lo && lo < end) s_out[0] = seg + (lo - at) / x.tiles;
    if (at < hi && hi <= end) s_out[1] = seg + (hi - 1 - at) / x.tiles;
    if (e == p.groups - 1) s_out[2] = seg + x.segments;      // segments of groups
    at = end;
    seg += x.segments;
  }
  if (p.groups == 0 && tid == 0) s_out[2] = 0;
  sync();
  const int first_seg = s_out[0], group_segs = s_out[2];
  at = tiles_to - tiles;
  seg = segs_to - segs;
  for (int e = e0; e < e1; ++e) {
    const Entry x = entry(e, false);
    const int end = at + x.segments * x.tiles;
    const bool of_group = e < p.groups;
    if (lo < hi && x.segments > 0 && at < hi && end > lo) {
      const int i0 = max(0, (lo - at) / x.tiles), i1 = min(x.segments - 1, (hi - 1 - at) / x.tiles);
      for (int i = i0; i <= i1; ++i) {
        const int a = at + i * x.tiles, j0 = max(0, lo - a), j1 = min(x.tiles, hi - a);
        int4 d;
        if (of_group) {
          const int m0 = s_start[e] + (i / p.KV) * rpt, n = min(rpt, s_start[e + 1] - m0);
          d.x = (int)(0x80000000u | (unsigned)m0);
          d.y = (i % p.KV) | (n << 8) | ((seg + i + range) << 16);
          d.z = j0 * KT;
          d.w = min(x.prefix, j1 * KT);
        } else {
          d.x = e - p.groups;
          d.y = i | (1 << 8) | ((seg + i - group_segs + range) << 16);
          d.z = x.prefix + j0 * KT;
          d.w = min(x.len, x.prefix + j1 * KT);
        }
        list[seg + i - first_seg] = d;
      }
    }
    if (write_rows && !of_group) {
      const int row = e - p.groups, m = s_member[row];
      int* rec = reinterpret_cast<int*>(p.work) + row * ROW_INTS;
      int r[ROW_INTS] = {0, 0, 0, 0, seg - group_segs, at, x.tiles, Q};
      const int g = m >= 0 ? group_of(m) : 0, i = m - s_start[g];
      if (x.prefix > 0 && i < s_start[g + 1] - s_start[g]) {      // (a start below the one before it was recorded)
        const int pt = cdiv(x.prefix, KT), qt = i / rpt;
        r[0] = s_seg[g] + qt * p.KV;
        r[1] = s_tile[g] + qt * p.KV * pt;
        r[2] = pt;
        r[3] = i % rpt * (p.H / p.KV);
      }
      for (int i = 0; i < ROW_INTS; ++i) rec[i] = r[i];
    }
    at = end;
    seg += x.segments;
  }
  const int n = lo < hi ? s_out[1] - first_seg + 1 : 0;
  sync();
  return n;
}
}  // namespace shared_prefix
