// Attention over shared prefixes on the tcgen05 tensor cores, bfloat16, heads of 64 or 128: the keys that the rows of a group share.  (The
// mathematics is in attention_shared_prefix.cu, how the work is cut in shared_prefix.cuh, the rows' own keys and the merge in
// attention_shared_prefix_rows.cu.)
//
// A block walks its pieces one after the other: up to 128 queries (rows of a group with their G heads of one key-value head)
// over tiles of 128 keys.  Both products are tcgen05.mma with accumulators in tensor memory:
//
//   S = Q K^T   A = Q [128 x hd], B = K [128 keys x hd] from shared memory, K-major; S[128 x 128] float
//   O += P V    A = P [128 x 128 keys] bfloat16 from shared memory, B = V as it lies in the cache ("MN-major"); O[128 x hd] float
//
// Tiles alternate between two halves of the block that do not wait for each other (half w: softmax warps 4w..4w+3, scores S_w,
// accumulator O_w, weights P_w; tiles w, w + 2, ...), merged at the end of a piece: while one half exponentiates, the tensor
// cores work for the other.  Warps without a query exponentiate nothing.
//
//   warps 0-7   softmax: thread r of a half owns query r.  They also fetch the queries, whose rows lie anywhere: the next
//               piece's are asked for before the merge of this one and stored when its last scores are made.
//   warps 8, 9  producers of K and V by TMA: a tile whose pages follow one another in the pool is one box per 64 columns,
//               else a box per page.  Pages behind the piece's last key are not fetched.  Warp 8 first lists the block's pieces.
//   warp 10     issues the score products
//   warp 11     issues P V over the 16-key blocks that hold keys, and clears what the last of them holds behind the last key
//               (a page's rest may hold anything, and 0 times infinity is no zero)
//
// A call is short (a tile of 128 keys takes a microsecond) and a kernel's instructions are fetched anew at every launch, about two bytes a cycle and
// SM: loops are kept rolled, and the scores are read twice from tensor memory, 32 columns at a time, instead of once into 128 registers.
// What bounds a long line of tiles is shared memory: 224 KB a tile (128 as operands of the two products, 64 of pages coming in, 32 of weights) at 128 bytes a
// cycle are 1,792 of the 1,918 cycles that a tile takes (48 rows behind 30,000 keys).  So neither scores fetched ahead of the exponentials (51 to 53 us),
// chunks of 16 or 64 columns (52 to 56) nor two products to an instruction (51) help.  Weights as an operand in tensor memory would take 64 KB off: over the scores they
// come from, since the halves' scores and accumulators fill it, so that a half's next scores wait for its product (not built).
// The last block computes nothing: it works out the pieces of the rows' kernel, which may start as soon as they are there.
//
// Every wait is bounded; when one gives up the block records it, waits (bounded again) for the copies and products it has under
// way, frees its tensor memory and returns.
#include "shared_prefix.cuh"
#include "tcgen05_helpers.cuh"
#include "ring.cuh"

namespace {
using namespace shared_prefix;
constexpr int QT = 128;            // queries of a tile (rows of both products)
constexpr int KT = 128;            // keys of a tile
constexpr int ROWS_KT = 64;        // keys of a tile of the rows' kernel
constexpr int MIN_ROW_TILES = 16;  // (48 rows of 200 to 1,000 keys of their own, 8 and 16: 58.7 and 56.3 us)
constexpr int HALF_THREADS = 128;
constexpr int PRODUCER_WARP0 = 8, MMA_WARP = 10;
constexpr int THREADS = (MMA_WARP + 2) * 32;
constexpr int BOX_BYTES = 128 * 128;   // 128 rows of one 128-byte swizzle row each
constexpr float RESCALE_STEP = 8.f;    // in powers of two
constexpr int TMEM_COLS = 512;
constexpr int COL_S = 0, COL_O = 2 * KT;

template <int HD>
struct Layout {
  static constexpr int HALVES = HD / 64;
  static constexpr int Q_BYTES = HALVES * BOX_BYTES;
  static constexpr int TILE_BYTES = HALVES * BOX_BYTES;   // one K or V tile
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + Q_BYTES;           // two of each
  static constexpr int OFF_V = OFF_K + 2 * TILE_BYTES;
  static constexpr int OFF_P = OFF_V + 2 * TILE_BYTES;    // P of each half: two boxes [128 x 64 keys]
  static constexpr int P_BYTES = 2 * BOX_BYTES;
  static constexpr int TOTAL = OFF_P + 2 * P_BYTES + 1024;   // 1024 to start on a swizzle boundary
  static_assert(4 * Cut::ints(MAX_ROWS, MAX_GROUPS) <= OFF_P, "the last block's tables");
};

// 2^x by the special-function unit (two units in the last place; results below 2^-126 become 0)
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ void block_barrier() {
  __syncwarp();
  asm volatile("bar.sync 1, %0;\n" ::"n"(THREADS) : "memory");
}
__device__ __noinline__ bool long_wait(uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity); }
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity) || long_wait(bar, parity); }

// The pieces of range ``range`` into ``list``, by one warp: a lane per group, first for the length of the line, then for what the range holds.
// Returns how many; ``ranges`` gets the number of ranges.  The same cut as make_cut's, which also reports what is wrong in the tables.
__device__ __forceinline__ int list_pieces(const DkSharedPrefixParams& p, int range, GroupPiece* list, int lane, int& ranges) {
  const int max_keys = p.max_pages * p.ps;
  int Q = 1, lo = 0, hi = 0, first_seg = -1, last_seg = -1;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int tile_base = 0, seg_base = 0;
    bool out_of_order = false;
#pragma unroll 1
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      const int g = g0 + lane;
      int a = 0, b = 0, k = 0;
      if (g < p.groups) {
        a = p.group_start[g];
        b = p.group_start[g + 1];
        k = p.group_prefix[g];
      }
      const bool bad = a < 0 || b < a || b > p.n_members;
      out_of_order |= __any_sync(0xffffffffu, bad);
      if (bad || k < 0 || k > max_keys) a = b = k = 0;
      k &= -p.ps;               // whole pages (a power of two)
      const int tiles = (long long)(b - a - 1) * k >= p.min_saved ? cdiv(k, KT) : 0, segs = tiles > 0 ? few(b - a, p.rpt) * p.KV : 0;
      int at = segs * tiles, seg = segs;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, at, o), y = __shfl_up_sync(0xffffffffu, seg, o);
        if (lane >= o) {
          at += x;
          seg += y;
        }
      }
      const int tile_end = __shfl_sync(0xffffffffu, at, 31), seg_end = __shfl_sync(0xffffffffu, seg, 31);
      if (pass == 1) {
        at += tile_base - segs * tiles;
        seg += seg_base - segs;
        const int end = at + segs * tiles;
        const unsigned with_first = __ballot_sync(0xffffffffu, at <= lo && lo < end);
        if (with_first) first_seg = __shfl_sync(0xffffffffu, seg + (tiles > 0 && lo > at ? (lo - at) / tiles : 0), __ffs(with_first) - 1);
        const unsigned with_last = __ballot_sync(0xffffffffu, at < hi && hi <= end);
        if (with_last) last_seg = __shfl_sync(0xffffffffu, seg + (tiles > 0 && hi > at ? (hi - 1 - at) / tiles : 0), __ffs(with_last) - 1);
        if (segs > 0 && at < hi && end > lo) {
#pragma unroll 1
          for (int i = lo > at ? (lo - at) / tiles : 0; i < segs && at + i * tiles < hi; ++i) {
            const int qt = i < p.KV ? 0 : i / p.KV, m0 = a + qt * p.rpt, row = p.members[m0], from = at + i * tiles;
            list[seg + i - first_seg] = {m0, min(p.rpt, b - m0), i - qt * p.KV, seg + i + range, max(0, lo - from) * KT, min(k, min(tiles, hi - from) * KT),
                                         row >= 0 && row < p.rows ? row : 0, 0};
          }
        }
      }
      tile_base += tile_end;
      seg_base += seg_end;
    }
    if (pass == 0) {
      if (out_of_order || tile_base > p.max_tiles) tile_base = seg_base = 0;      // as make_cut has it
      Q = range_tiles(p, tile_base, seg_base);
      ranges = cdiv(tile_base, Q);
      lo = range * Q;
      hi = min(tile_base, lo + Q);
      if (lo >= hi) return 0;
    }
  }
  return last_seg - first_seg + 1;
}

// What the rows' kernel needs: its pieces, and the counters cleared.  The list is published for its blocks that start before this kernel's end.
// (A function of its own: inlined it made the other blocks' code slower. 48 rows behind 30,000 keys 52.1 and 50.7 us, 64 behind 2,048 24.8 and 24.0, the mixed
// call 33.6 and 32.9, 8 rows behind 4,096 16.6 and 17.0.)
template <int HD>
__device__ __noinline__ void prepare_rows(const DkSharedPrefixParams p, int* tables, int tid) {
  for (int i = tid; i < p.rows * p.KV; i += THREADS) counters(p)[i] = 0;
  Cut cut(tables, p.rows, p.groups);
  make_cut<KT, ROWS_KT, MIN_ROW_TILES, THREADS>(p, cut, tid);
  for (int id = tid; id < cut.pieces; id += THREADS) row_pieces(p)[id] = row_piece<KT, ROWS_KT>(p, cut, id);
  if (tid == 0) *reinterpret_cast<int*>(p.work) = cut.pieces;
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    asm volatile("st.release.gpu.global.u64 [%0], %1;\n" ::"l"(list_of_call(p)), "l"(p.call) : "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  }
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) attention_shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap map_kv,
                                                                                const __grid_constant__ CUtensorMap map_run,
                                                                                const DkSharedPrefixParams p) {
  using L = Layout<HD>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  // barriers: q_full, k_full[2], v_full[2], s_full[2], p_full[2], o_done[2], s_free[2], merge, piece_done.  Those in pairs belong to the
  // tiles of one parity of their pieces; what a wait needs is how many of them the block has had.
  __shared__ __align__(8) unsigned long long bars[15];
  __shared__ GroupPiece list[CAP];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  __shared__ int n_listed, n_ranges;
  // row_stat(w)[query]: maximum and sum of half w's tiles, over the half's P, which is not read any more by then
  auto row_stat = [&](int w) { return reinterpret_cast<float2*>(smem + L::OFF_P + w * L::P_BYTES); };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (blockIdx.x + 1 == gridDim.x) {
    prepare_rows<HD>(p, reinterpret_cast<int*>(smem), tid);
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");      // the rows' kernel may start wherever there is room, once its pieces are there
  const int ps = p.ps, G = p.G;
  const uint32_t bar0 = s2u(&bars[0]);
  const uint32_t q_full = bar0, k_full = bar0 + 8, v_full = k_full + 16, s_full = v_full + 16, p_full = s_full + 16, o_done = p_full + 16,
                 s_free = o_done + 16, merge_bar = s_free + 16, piece_done = merge_bar + 8;
  if (tid == 0) {
    const unsigned counts[15] = {2 * HALF_THREADS, 1, 1, 1, 1, 1, 1, HALF_THREADS, HALF_THREADS, 1, 1, HALF_THREADS, HALF_THREADS, 2 * HALF_THREADS, 2 * HALF_THREADS};
#pragma unroll
    for (int i = 0; i < 15; ++i) mbar_init(bar0 + 8 * i, counts[i]);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(s2u(&tmem_slot), TMEM_COLS);
  const uint32_t sm_q = s2u(smem + L::OFF_Q), sm_k = s2u(smem + L::OFF_K), sm_v = s2u(smem + L::OFF_V), sm_p = s2u(smem + L::OFF_P);
  int had0 = 0, had1 = 0;   // tiles of each parity in the pieces before the current one
  int asked0 = 0, asked1 = 0;   // producers: tiles of each parity asked for so far
  int n_done = 0;           // pieces before the current one
  int had_w = 0, had_other = 0;       // softmax: tiles of this half and of the other one so far
  for (int range = blockIdx.x;; range += gridDim.x - 1) {
    if (warp == PRODUCER_WARP0) {
      int ranges = 0;
      const int n = list_pieces(p, range, list, lane, ranges);
      if (lane == 0) {
        n_listed = n;
        n_ranges = ranges;
      }
    }
    tc_fence_before();
    block_barrier();
    tc_fence_after();
    const int n_pieces = n_listed;       // (read before the second barrier: behind it the next list is made)
    const bool more = range + (int)gridDim.x - 1 < n_ranges;
    const uint32_t tmem = tmem_slot;
    if (warp < PRODUCER_WARP0) {
      // ------------------------------------------------------------- softmax
      const int w = warp >> 2;                            // which half: its tiles are w, w + 2, ...
      const int r = (warp & 3) * 32 + lane;               // query of this thread = lane of the TMEM
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t t_s = tmem + lane_base + COL_S + w * KT;
      const uint32_t t_o = tmem + lane_base + COL_O + w * HD;
      const float sl2 = p.scale * 1.4426950408889634f;
      // This half's columns of the queries: LANES neighbouring lanes fetch a row's 16-byte chunks, so a warp's request covers whole lines.
      constexpr int LANES = HD / 16, AT_ONCE = 32 / LANES;       // lanes to a row, rows to a request
      const int qi = r / G, qh = r - qi * G;
      uint4 qv[LANES];
      auto ask_q = [&](const GroupPiece& pc) {      // (a row of the tile without a query gets some other: nothing comes of it)
        const int row = qi < pc.rows ? p.members[pc.first + qi] : -1;
        const long long mine = row >= 0 && row < p.rows ? row * p.q_stride + (pc.kvh * G + qh) * HD : -1;
#pragma unroll
        for (int x = 0; x < LANES; ++x) {
          const long long at = __shfl_sync(0xffffffffu, mine, x * AT_ONCE + lane / LANES);
          qv[x] = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.q) + (at < 0 ? 0 : at) + w * (HD / 2) + lane % LANES * 8);
        }
      };
      auto store_q = [&] {
        const int col = w * LANES + lane % LANES;       // 16-byte chunk of a query's row
#pragma unroll
        for (int x = 0; x < LANES; ++x) {
          const int to = (warp & 3) * 32 + x * AT_ONCE + lane / LANES;
          *reinterpret_cast<uint4*>(smem + L::OFF_Q + (col / 8) * BOX_BYTES + to * 128 + (((col % 8) ^ (to & 7)) << 4)) = qv[x];
        }
        fence_async_smem();
        mbar_arrive(q_full);
      };
      // Queries are fetched in front of every piece (i = -1: the first one's), stored when all scores of the piece before are made.
      bool good = true;
#pragma unroll 1
      for (int i = -1; good && i < n_pieces; ++i) {
        GroupPiece pc = {};
        int n_tiles = 0, queries = 0, mine = 0;
        float m_used = -INFINITY, l_sum = 0.f;
        bool busy = false;
        if (i >= 0) {
          pc = list[i];
          n_tiles = cdiv(pc.limit - pc.key0, KT);
          queries = pc.rows * G;
          busy = (warp & 3) * 32 < queries;       // some thread of this warp has a query
          // P (under which the maxima and sums of the piece before lay) and the accumulators are free again
          if (n_done > 0) {
            const bool ok = wait(piece_done, (n_done - 1) & 1);
            if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
          }
        }
#pragma unroll 1
        for (int j = w; j < n_tiles; j += 2, ++mine) {
          const int ord = had_w + mine;
          bool ok = wait(s_full + 8 * w, ord & 1);
          if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
          tc_fence_after();
          const int n = pc.limit - pc.key0 - j * KT;      // keys of this tile and those behind it
          float factor = 1.f;
          bool grow = false;
          if (busy) {
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // four chains instead of one long one
#pragma unroll 1
            for (int c = 0; c < KT; c += 32) {
              float v[32];
              tmem_ld32_nowait(t_s + c, v);
              tmem_wait_ld();
              if (n < KT) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (c + k >= n) v[k] = -INFINITY;
              }
#pragma unroll
              for (int k = 0; k < 32; ++k) mx4[k & 3] = fmaxf(mx4[k & 3], v[k]);
            }
            const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl2);
            grow = m_new > m_used + RESCALE_STEP;      // also the first finite maximum of a row
            if (grow) {
              factor = m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_new);
              m_used = m_new;
            }
          }
          if (mine > 0) {
            // P V of this half's tile before is done: its P may be overwritten, and O_w is at rest
            ok = wait(o_done + 8 * w, (ord - 1) & 1);
            if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
            if (__any_sync(0xffffffffu, grow)) {
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                float o[32];
                tmem_ld32_nowait(t_o + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= factor;
                tmem_st32(t_o + c * 32, o);
              }
              tmem_wait_st();
              tc_fence_before();
            }
          }
          if (busy) {
            // exponentials, their sum in 32 bits, and P rounded to bfloat16 (what the product takes) in the layout of a 128-byte swizzle
            const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
            float sum4[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t p_row = sm_p + w * L::P_BYTES + r * 128;
#pragma unroll 1
            for (int c = 0; c < KT; c += 32) {
              float v[32];
              tmem_ld32_nowait(t_s + c, v);
              tmem_wait_ld();
              if (c == KT - 32) {        // the scores are read: those of the half's next tile may be made
                tc_fence_before();
                mbar_arrive(s_free + 8 * w);
              }
              if (n < KT) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (c + k >= n) v[k] = -INFINITY;
              }
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                v[k] = fast_exp2(fmaf(v[k], sl2, neg_m));
                sum4[k & 3] += v[k];
              }
              const uint32_t addr = p_row + (c >> 6) * BOX_BYTES;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr + ((((c >> 3) & 7) + k ^ (r & 7)) << 4)), "r"(pack2(v[8 * k], v[8 * k + 1])),
                             "r"(pack2(v[8 * k + 2], v[8 * k + 3])), "r"(pack2(v[8 * k + 4], v[8 * k + 5])), "r"(pack2(v[8 * k + 6], v[8 * k + 7])) : "memory");
            }
            l_sum = l_sum * factor + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
            fence_async_smem();
          } else {
            mbar_arrive(s_free + 8 * w);
          }
          mbar_arrive(p_full + 8 * w);
        }
        had_w += (n_tiles + 1 - w) / 2;
        had_other += (n_tiles + w) / 2;
        if (!good) break;
        bool ok = true;
        if (i + 1 < n_pieces) {
          ask_q(list[i + 1]);
          if (had_other > 0) ok = wait(s_full + 8 * (w ^ 1), (had_other - 1) & 1);
          store_q();
        }
        if (mine > 0) ok = wait(o_done + 8 * w, (had_w - 1) & 1) && ok;
        if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
        if (i < 0) continue;
        // merge of the two halves: each tells the other its maximum and sum, then writes half of the columns
        row_stat(w)[r] = make_float2(m_used, l_sum);
        tc_fence_before();
        mbar_arrive(merge_bar);
        ok = wait(merge_bar, n_done & 1);
        if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
        tc_fence_after();
        const float2 other = row_stat(w ^ 1)[r];
        const float m_all = fmaxf(m_used, other.x);
        const float f_mine = m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_all);
        const float f_other = other.x == -INFINITY ? 0.f : fast_exp2(other.x - m_all);
        const float f0 = w == 0 ? f_mine : f_other, f1 = w == 0 ? f_other : f_mine;
        const bool two = n_tiles > 1;                     // O_1 holds nothing when there was one tile
        float* part = group_results(p, pc.id) + 4 * r;
        if (busy) {
#pragma unroll 1
          for (int c = w * (HD / 2); c < (w + 1) * (HD / 2); c += 32) {
            float o0[32], o1[32];
            tmem_ld32_nowait(tmem + lane_base + COL_O + c, o0);
            if (two) tmem_ld32_nowait(tmem + lane_base + COL_O + HD + c, o1);
            tmem_wait_ld();
            if (r < queries) {
#pragma unroll
              for (int k = 0; k < 32; ++k) o0[k] = two ? o0[k] * f0 + o1[k] * f1 : o0[k] * f0;
#pragma unroll
              for (int k = 0; k < 8; ++k)
                *reinterpret_cast<float4*>(part + (size_t)(c / 4 + k) * (4 * QT)) = make_float4(o0[4 * k], o0[4 * k + 1], o0[4 * k + 2], o0[4 * k + 3]);
            }
          }
          if (r < queries && w == 0) *reinterpret_cast<float4*>(part + (size_t)QT * HD) = make_float4(m_all, l_sum * f_mine + other.y * f_other, 0.f, 0.f);
        }
        // accumulators and the other half's maximum and sum were read: the next piece may overwrite them
        tc_fence_before();
        mbar_arrive(piece_done);
        ++n_done;
      }
    } else if (warp < MMA_WARP) {
      // ----------------------------------------------------------- producers
      const int kind = warp - PRODUCER_WARP0;     // 0: K, 1: V
      const uint32_t full = kind ? v_full : k_full, done = kind ? o_done : s_full, sm_dst = kind ? sm_v : sm_k;
      const int ppt = KT / ps;      // pages per tile, at most 16
#pragma unroll 1
      for (int i = 0; i < n_pieces && !failed; ++i) {
        const GroupPiece w = list[i];
        const int n_tiles = cdiv(w.limit - w.key0, KT);
        const int* table = p.block_table + (size_t)w.table_row * p.max_pages;
#pragma unroll 1
        for (int j = 0; j < n_tiles; ++j) {
          const int c = j & 1, ord = (c ? had1 : had0) + j / 2;     // the ord-th tile of its parity in this block
          const int kb = w.key0 + j * KT, pages = min(ppt, cdiv(w.limit - kb, ps)), lp = kb / ps + lane;
          int page = -1;
          if (lane < pages) {
            page = table[lp];          // below max_pages: limits were checked
            if (page < 0 || page >= p.num_pages) {
              dk_report(p.err, DK_DEV_BAD_PAGE, w.table_row, lp, page);
              page = -1;
            }
          }
          const int first = __shfl_sync(0xffffffffu, page, 0);
          const bool run = __all_sync(0xffffffffu, lane >= ppt || (page >= 0 && page == first + lane));
          const int held = __popc(__ballot_sync(0xffffffffu, page >= 0));
          bool ok = true;
          if (ord >= 1) ok = wait(done + 8 * c, (ord - 1) & 1);
          if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; break; }
          if (lane == 0) mbar_expect_tx(full + 8 * c, (uint32_t)(held * ps * 128 * L::HALVES));
          __syncwarp();
          const uint32_t dst = sm_dst + c * L::TILE_BYTES;
          if (run) {
            if (lane == 0)
              for (int half = 0; half < L::HALVES; ++half)
                tma_load_4d(dst + half * BOX_BYTES, &map_run, half * 64, 0, kind * p.KV + w.kvh, first, full + 8 * c);
          } else if (page >= 0) {
            const int grow = ((page * 2 + kind) * p.KV + w.kvh) * ps;    // row of the cache seen as [pages * 2 * KV * ps, hd]
            for (int half = 0; half < L::HALVES; ++half)
              tma_load_2d(dst + half * BOX_BYTES + lane * ps * 128, &map_kv, half * 64, grow, full + 8 * c);
          }
          if (c) asked1 = ord + 1; else asked0 = ord + 1;
        }
        if (failed) break;
        had0 += (n_tiles + 1) / 2;
        had1 += n_tiles / 2;
      }
    } else {
      // ------------------------------------------- issuers: the scores (warp 10), P V (warp 11)
      const bool scores = warp == MMA_WARP, leader = elect_one();
      const uint32_t idesc = scores ? instr_desc_bf16(QT, KT, false) : instr_desc_bf16(QT, HD, true);
      const uint32_t operand = scores ? k_full : v_full, ready = scores ? s_free : p_full, result = scores ? s_full : o_done;
      auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };
      bool ok = true;
#pragma unroll 1
      for (int i = 0; ok && i < n_pieces; ++i) {
        const GroupPiece w = list[i];
        const int n_tiles = cdiv(w.limit - w.key0, KT);
        if (scores) ok = wait_all(q_full, n_done & 1);
        int j = 0;
#pragma unroll 1
        for (; ok && j < n_tiles; ++j) {
          const int c = j & 1, ord = (c ? had1 : had0) + j / 2, n = min(KT, w.limit - w.key0 - j * KT), blocks = scores ? HD / 16 : cdiv(n, 16);
          if (!wait_all(operand + 8 * c, ord & 1)) { ok = false; break; }
          if (!scores && n % 16 != 0) {          // rows n to 16 blocks - 1 of V, eight 16-byte chunks each
            const int chunks = (blocks * 16 - n) * 8;
            for (int x = lane; x < chunks * L::HALVES; x += 32)
              *reinterpret_cast<uint4*>(smem + L::OFF_V + c * L::TILE_BYTES + x / chunks * BOX_BYTES + n * 128 + x % chunks * 16) = make_uint4(0u, 0u, 0u, 0u);
            fence_async_smem();
            __syncwarp();
          }
          // the scores' buffer was read (from the second tile of its parity on), or P is written
          if ((!scores || ord >= 1) && !wait_all(ready + 8 * c, (scores ? ord - 1 : ord) & 1)) { ok = false; break; }
          tc_fence_after();
          if (leader) {
            const uint64_t da = smem_desc_k_major(scores ? sm_q : sm_p + c * L::P_BYTES);
            const uint64_t db = scores ? smem_desc_k_major(sm_k + c * L::TILE_BYTES) : smem_desc_mn_major(sm_v + c * L::TILE_BYTES, BOX_BYTES);
            const uint32_t d = tmem + (scores ? COL_S + c * KT : COL_O + c * HD);
#pragma unroll 1
            for (int kk = 0; kk < blocks; ++kk) {      // 16 further: 32 bytes along a row, or two groups of 8 rows of V; start addresses count 16 bytes
              const uint64_t along = (uint64_t)(((kk / 4) * BOX_BYTES + (kk % 4) * 32) >> 4);
              umma(d, da + along, db + (scores ? along : (uint64_t)(kk * (2048 >> 4))), idesc, (kk > 0 || (!scores && j > 1)) ? 1u : 0u);
            }
            umma_commit(result + 8 * c);
          }
          __syncwarp();
        }
        had0 += (j + 1) / 2;
        had1 += j / 2;
        ++n_done;
      }
      if (!ok) failed = 1;
    }
    block_barrier();
    if (failed || !more) break;
  }
  if (warp >= PRODUCER_WARP0 && lane == 0) {      // what this warp has under way ends before the block leaves
    const bool producer = warp < MMA_WARP;
    const uint32_t bar = producer ? (warp == PRODUCER_WARP0 ? k_full : v_full) : (warp == MMA_WARP ? s_full : o_done);
    ring_drain(producer ? asked0 : had0, 1, [&](int, uint32_t parity) { return long_wait(bar, parity); });
    ring_drain(producer ? asked1 : had1, 1, [&](int, uint32_t parity) { return long_wait(bar + 8, parity); });
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (failed && tid == 0) dk_report(p.err, DK_DEV_TIMEOUT, (int)blockIdx.x, (int)gridDim.x, n_listed);
  if (warp == MMA_WARP) tmem_dealloc(tmem_slot, TMEM_COLS);
}

template <int HD>
int launch(const DkSharedPrefixParams& p, cudaStream_t stream) {
  using L = Layout<HD>;
  CUtensorMap map_kv, map_run;
  DK_REQUIRE(make_tensor_map_bf16(&map_kv, p.kv, (long long)p.num_pages * 2 * p.KV * p.ps, HD, HD, p.ps), "attention_shared_prefix: cannot encode the tensor map of the cache");
  // the cache as [page][K|V, head][offset][hd]: a run of pages of one head in one box
  const unsigned long long dims[4] = {(unsigned long long)HD, (unsigned long long)p.ps, (unsigned long long)(2 * p.KV), (unsigned long long)p.num_pages};
  const unsigned long long strides[3] = {(unsigned long long)HD * 2, (unsigned long long)p.ps * HD * 2, (unsigned long long)2 * p.KV * p.ps * HD * 2};
  DK_REQUIRE(make_tensor_map_bf16_4d(&map_run, p.kv, dims, strides, p.ps, KT / p.ps), "attention_shared_prefix: cannot encode the tensor map of runs of pages");
  static bool configured_on[DK_MAX_DEVICES] = {false};
  bool& configured = configured_on[dk_current_device()];
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(attention_shared_prefix_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);
    if (e != cudaSuccess) {
      dk_set_error("attention_shared_prefix: cannot get %d bytes of shared memory: %s", L::TOTAL, cudaGetErrorString(e));
      return DK_ERR_LAUNCH;
    }
    configured = true;
  }
  attention_shared_prefix_tc_kernel<HD><<<p.groups > 0 ? p.grid + 1 : 1, THREADS, L::TOTAL, stream>>>(map_kv, map_run, p);
  return dk_check_launch("attention_shared_prefix_tc");
}
}  // namespace

bool dk_shared_prefix_tc_takes(const DkSharedPrefixParams& p) {
  return p.dtype == DK_BF16 && p.H / p.KV <= 16 && (p.hd == 64 || p.hd == 128) && (p.ps == 8 || p.ps == 16 || p.ps == 32 || p.ps == 64 || p.ps == 128) &&
         (long long)p.num_pages * 2 * p.KV * p.ps < (1ll << 31);
}

int dk_shared_prefix_tc_launch(const DkSharedPrefixParams& p, cudaStream_t stream) { return p.hd == 64 ? launch<64>(p, stream) : launch<128>(p, stream); }
