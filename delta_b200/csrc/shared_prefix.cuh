// How the attention over shared prefixes cuts its work: the arguments, the plan and where the partial results lie.
//
// Work comes in segments.  A segment of a group is a tile of its queries (``rpt`` rows with their G query heads of one
// key-value head) over the group's shared keys; a segment of a row is its G query heads over the keys it holds alone.  A segment
// is walked in tiles of keys, and cut into pieces of whole tiles:
//
//   groups  the tiles of all segments stand in one line, which is cut into ranges of Q tiles, as many as blocks run at once: every block
//           has the same number of tiles whatever the groups are, and at most one segment is cut at each border.  A piece is what a
//           range holds of a segment, and its number is segment + range: every step from one piece to the next moves to the next
//           segment or the next range, so no two pieces have one number and those of a range follow one another.
//   rows    every segment is cut into equal pieces of at most C tiles, numbered through, and a block takes every ``grid``-th.  C is what
//           levels the blocks, but eight tiles at least: a cut costs a row about as much as three tiles, since its pieces go through memory.
//
// One small kernel works the plan out from the tables on the device, so that a captured call follows them, and the kernels that
// compute read it.  A plan holds for every layer that has the same tables.
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
  int* plan;
  float* work;               // counters, then the pieces' partial results
  int* err;                  // device error record, 4 ints; or null
  long long q_stride, out_stride;   // elements
  int rows, groups, n_members, H, KV, hd, ps, max_pages, num_pages, dtype;
  float scale;
  // set by the launcher: how the work is cut (queries and keys of a group's tile, keys of a row's), the blocks that compute, the most pieces and
  // ranges there can be, and the keys that a group must save for its prefix to be read apart
  int qr, kt, rows_kt, grid, rows_grid, group_ranges, group_pieces, row_pieces, min_saved;
};

namespace shared_prefix {
constexpr int MAX_ROWS = 1024, MAX_GROUPS = 1023, MAX_G = 32;
constexpr int CAP = 48;            // tiles of a range, so also the most pieces of one
constexpr int MIN_ROW_TILES = 8;

__host__ __device__ constexpr int cdiv(int a, int b) { return (a + b - 1) / b; }
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
// The plan in ints: {ranges of groups, pieces of rows, 0, 0}, per range {first piece, pieces}, per row {first piece, pieces of a segment}, the pieces.
constexpr int HEAD = 4, GROUP_INTS = sizeof(GroupPiece) / 4, ROW_INTS = sizeof(RowPiece) / 4;
struct Plan {
  int *head, *ranges, *rows;
  GroupPiece* group_pieces;
  RowPiece* row_pieces;
  __host__ __device__ __forceinline__ Plan(const DkSharedPrefixParams& p)
      : head(p.plan), ranges(head + HEAD), rows(ranges + round4(2 * p.group_ranges)), group_pieces(reinterpret_cast<GroupPiece*>(rows + round4(2 * p.rows))),
        row_pieces(reinterpret_cast<RowPiece*>(group_pieces + p.group_pieces)) {}
};

// Floats of one piece's results: of a group as [hd / 4][queries][4] (neighbouring rows lie side by side), then {maximum, sum} per query; of a row as
// [query][hd], then the same.
__host__ __device__ __forceinline__ long long group_piece_floats(int qr, int hd) { return (long long)qr * (hd + 2); }
__host__ __device__ __forceinline__ long long row_piece_floats(int G, int hd) { return ((long long)G * (hd + 2) + 3) / 4 * 4; }

// Fills in the most ranges and pieces that there can be with these sizes, whatever the device's tables say, and tells what they need.
struct Bounds {
  long long tiles, group_ranges, group_pieces, row_pieces, plan_ints, work_floats;
};
static inline Bounds bounds(DkSharedPrefixParams& p) {
  Bounds b;
  const int G = p.H / p.KV, rpt = p.qr / G;
  const long long keys = (long long)p.max_pages * p.ps, segments = (long long)p.KV * (p.groups > 0 ? p.n_members / rpt + p.groups : 0);
  const long long of_groups = segments * ((keys + p.kt - 1) / p.kt);
  b.tiles = of_groups + (long long)p.rows * p.KV * ((keys + p.rows_kt - 1) / p.rows_kt);
  b.group_ranges = segments > 0 ? ((of_groups + CAP - 1) / CAP > p.grid ? (of_groups + CAP - 1) / CAP : (long long)p.grid) : 0;
  b.group_pieces = segments > 0 ? segments + b.group_ranges : 0;
  b.row_pieces = (long long)p.rows * p.KV + p.rows_grid;      // a segment's last piece, and tiles / C of full ones, which are no more than blocks
  b.plan_ints = HEAD + 2 * b.group_ranges + 4 + 2ll * p.rows + 4 + b.group_pieces * GROUP_INTS + b.row_pieces * ROW_INTS;
  b.work_floats = round4(p.rows * p.KV) + b.group_pieces * group_piece_floats(p.qr, p.hd) + b.row_pieces * row_piece_floats(G, p.hd);
  p.group_ranges = (int)b.group_ranges;
  p.group_pieces = (int)b.group_pieces;
  p.row_pieces = (int)b.row_pieces;
  return b;
}
__device__ __forceinline__ int* counters(const DkSharedPrefixParams& p) { return reinterpret_cast<int*>(p.work); }
__device__ __forceinline__ float* group_results(const DkSharedPrefixParams& p, int id) {
  return p.work + round4(p.rows * p.KV) + id * group_piece_floats(p.qr, p.hd);
}
__device__ __forceinline__ float* row_results(const DkSharedPrefixParams& p, int id) {
  return group_results(p, p.group_pieces) + id * row_piece_floats(p.H / p.KV, p.hd);
}
}  // namespace shared_prefix
