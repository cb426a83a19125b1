// Attention over shared prefixes, bfloat16: the keys that each row holds alone, and the merge with the pieces that the
// kernel of the groups (attention_shared_prefix_tc.cu) leaves.
//
// A row's G <= 16 query heads of one key-value head are the columns of warp-level MMA tiles; the kernel is bound by the bytes of
// K and V, which nobody shares, so the legacy MMA is enough.  Two blocks run on an SM and take pieces in turn; their tiles of 64 keys flow
// through a ring without a stop between pieces:
//
//   warp 4     fetches by TMA: a tile's K and V (one box per 64 columns where its pages follow one another in the pool, else a
//              box per page; pages behind the last key are left out), and with a segment's first tile its queries
//   warps 0-3  16 keys of a tile each, as S^T = K Q^T and O^T += V^T P^T: the queries are the eight columns of an MMA, so that none of it is
//              spent on empty rows (an MMA takes a warp some 35 cycles here, which was most of the time with queries as its 16 rows).  Each
//              warp has a maximum of its own; they are merged at a piece's end.
//
// Behind a piece's last tile the pieces of its row's group are added to it, in the order of their keys: they come through the ring as well, up to eight
// a stage, one box each.  (Of a segment that is cut, only the first piece adds them.)  The result is rounded once.  Where a segment is cut, each block
// leaves its piece's results in the work buffer and counts itself; the one that comes last adds them all, in their order, so the result does not depend on
// who that is.  This kernel starts while that one runs and waits for its end before it touches what it wrote, but for the list of pieces: the block that
// writes it publishes it with a release of the call's number, and a block of this kernel that acquires that number may read the list; one that does not
// waits for the other kernel's end.  The number is nobody else's, and it is taken back before this kernel ends, so a replayed call does not find its last one.
#include "shared_prefix.cuh"
#include "tcgen05_helpers.cuh"
#include "mma_helpers.cuh"
#include "ring.cuh"
#include <atomic>

namespace {
using namespace shared_prefix;
constexpr int TILE = 64;           // keys of a tile
constexpr int QR = 128;            // queries of a group's piece
constexpr int LISTED = 32;         // pieces whose records lie in shared memory at once
constexpr int MERGED = 8;          // pieces of a group in a stage, at most
constexpr int ROWS = 16;           // queries of a piece, at most
constexpr int WARPS = 4, THREADS = (WARPS + 1) * 32;

// One block of five stages an SM where two of three do not fit (heads of 128 with more than 8 to a key-value head).
template <int HD, bool LOW>
struct Ring {
  static constexpr int HALVES = HD / 64;
  static constexpr int KV_BYTES = HALVES * TILE * 128;               // one of K and V
  static constexpr int Q_BYTES = (LOW ? 8 : ROWS) * HD * 2;
  static constexpr int STAGE = (2 * KV_BYTES + Q_BYTES + 1023) / 1024 * 1024;
  static constexpr int STAGES = HD == 128 && LOW ? 3 : 5;
  static constexpr int BLOCKS = HD == 128 && !LOW ? 1 : 2;            // on an SM
  static constexpr int TOTAL = STAGES * STAGE + 1024;                // 1024 to start on a swizzle boundary
};

// The 8 x 8 matrix of 16-bit entries that lies over the warp as a fragment, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
// Byte offset of 16-byte chunk ``chunk`` of key ``key`` in a K or V tile: 64 columns side by side, rows of 128 bytes, 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_offset(int key, int chunk) {
  return (uint32_t)((chunk >> 3) * (TILE * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __noinline__ bool long_wait(uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity); }
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity) || long_wait(bar, parity); }
// 2^x by the special-function unit (two units in the last place; results below 2^-126 become 0)
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void warps_barrier() { asm volatile("bar.sync 1, %0;\n" ::"n"(WARPS * 32) : "memory"); }

template <int HD, bool LOW>
__global__ void __launch_bounds__(THREADS, Ring<HD, LOW>::BLOCKS) attention_shared_prefix_rows_kernel(const __grid_constant__ CUtensorMap map_kv,
                                                                                  const __grid_constant__ CUtensorMap map_run,
                                                                                  const __grid_constant__ CUtensorMap map_merge,
                                                                                  const DkSharedPrefixParams p) {
  using R = Ring<HD, LOW>;
  constexpr int NQ = LOW ? 1 : 2, ROWS_USED = 8 * NQ;      // tiles of eight queries
  constexpr int KB = HD / 16, MT = HD / 16;   // blocks of 16 columns: the depth of K Q^T, the rows of V^T P^T
  constexpr int STEP = WARPS * 32 / ROWS_USED, PASSES = HD / 4 / STEP;      // at a piece's end: threads to a query, groups of four columns of each
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long bars[2 * R::STAGES];   // full, then empty
  __shared__ RowPiece list[LISTED];
  __shared__ float s_max[2][WARPS][ROWS], s_sum[2][WARPS][ROWS];      // in turns for the pieces
  __shared__ int s_last;
  __shared__ bool listed;
  __shared__ volatile int failed, stuck;      // a wait of the producer, of one of the four warps gave up
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
  const int ps = p.ps, G = p.G;
  const uint32_t full = s2u(&bars[0]), empty = full + 8 * R::STAGES, ring = s2u(smem);
  if (tid == 0) {
    for (int s = 0; s < R::STAGES; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, WARPS);
    }
    failed = stuck = 0;
    unsigned long long seen;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];\n" : "=l"(seen) : "l"(list_of_call(p)) : "memory");
    listed = seen == p.call;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  const float sl2 = p.scale * 1.4426950408889634f;
  int n_tile = 0;                 // tiles this block has had
  bool waited = false;
  // the pieces of a group in a stage: G queries each in a slot of its own
  const int slot_bytes = (G * 16 * (HD / 4 + 1) + 127) / 128 * 128, per_stage = min(MERGED, R::STAGE / slot_bytes);
  if (!listed) asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int all_pieces = __ldcg(reinterpret_cast<const int*>(p.work));
  for (int first = blockIdx.x; first < p.row_pieces; first += gridDim.x * LISTED) {
    // (records behind the last piece are read with the others, so that nothing waits for the count, and not used)
    for (int x = tid; x < LISTED * (ROW_INTS / 4); x += THREADS) {
      const int id = first + x / (ROW_INTS / 4) * (int)gridDim.x;
      if (id < p.row_pieces) reinterpret_cast<int4*>(list)[x] = __ldcg(reinterpret_cast<const int4*>(row_pieces(p) + id) + x % (ROW_INTS / 4));
    }
    const int n_pieces = first < all_pieces ? min(LISTED, cdiv(all_pieces - first, (int)gridDim.x)) : 0;
    if (n_pieces == 0) break;
    __syncthreads();
    if (warp == WARPS) {
      // ---------------------------------------------------------------- producer
      const int rows_of_box = min(ps, TILE), ppt = TILE / rows_of_box;      // a tile's pages, at most 8
      int n = n_tile;
      for (int i = 0; i < n_pieces && !failed; ++i) {
        const RowPiece& w = list[i];
        const int* table = p.block_table + (size_t)w.row * p.max_pages;
        const int kvh = w.kvh, limit = w.limit;
        int kb = w.key0;
        do {
          const int held_pages = min(ppt, cdiv(limit - kb, rows_of_box)), lp = kb / ps + lane;
          int page = -1;
          if (lane < held_pages) {
            page = table[lp];            // below max_pages: limits were checked
            if (page < 0 || page >= p.num_pages) {
              dk_report(p.err, DK_DEV_BAD_PAGE, w.row, lp, page);
              page = -1;
            }
          }
          const int first = __shfl_sync(0xffffffffu, page, 0);
          const bool run = ppt > 1 && __all_sync(0xffffffffu, lane >= ppt || (page >= 0 && page == first + lane));
          const int held = __popc(__ballot_sync(0xffffffffu, page >= 0));
          const int s = ring_slot(n, R::STAGES);
          bool ok = true;
          if (n >= R::STAGES) ok = wait(empty + 8 * s, ring_parity(n - R::STAGES, R::STAGES));
          if (!__all_sync(0xffffffffu, ok && !stuck)) { failed = 1; break; }
          const uint32_t k_dst = ring + s * R::STAGE, v_dst = k_dst + R::KV_BYTES, bar = full + 8 * s;
          const bool with_q = kb == w.key0 && limit > w.key0;
          if (lane == 0) {
            mbar_expect_tx(bar, (uint32_t)(held * rows_of_box * 128 * R::HALVES * 2 + (with_q ? G * HD * 2 : 0)));
            if (with_q)
              bulk_load(v_dst + R::KV_BYTES, reinterpret_cast<const __nv_bfloat16*>(p.q) + w.row * p.q_stride + kvh * G * HD, (uint32_t)(G * HD * 2), bar);
          }
          __syncwarp();
          if (run) {
            if (lane == 0)
              for (int half = 0; half < R::HALVES; ++half) {
                tma_load_4d(k_dst + half * (TILE * 128), &map_run, half * 64, 0, kvh, first, bar);
                tma_load_4d(v_dst + half * (TILE * 128), &map_run, half * 64, 0, p.KV + kvh, first, bar);
              }
          } else if (page >= 0) {
            const int grow = (page * 2 * p.KV + kvh) * ps + kb % ps;      // row of the cache seen as [pages * 2 * KV * ps, hd]
            for (int half = 0; half < R::HALVES; ++half) {
              tma_load_2d(k_dst + half * (TILE * 128) + lane * rows_of_box * 128, &map_kv, half * 64, grow, bar);
              tma_load_2d(v_dst + half * (TILE * 128) + lane * rows_of_box * 128, &map_kv, half * 64, grow + p.KV * ps, bar);
            }
          }
          ++n;
          kb += TILE;
        } while (kb < limit);
        if (failed || w.index != 0 || w.group_n == 0) continue;
        if (!waited) {          // the pieces of the groups
          asm volatile("griddepcontrol.wait;\n" ::: "memory");
          asm volatile("fence.proxy.async;\n" ::: "memory");       // written with ordinary stores, read by TMA
          waited = true;
        }
        for (int x = 0; x < w.group_n; x += per_stage, ++n) {
          const int s = ring_slot(n, R::STAGES), m = min(per_stage, w.group_n - x);
          bool ok = true;
          if (n >= R::STAGES) ok = wait(empty + 8 * s, ring_parity(n - R::STAGES, R::STAGES));
          if (!__all_sync(0xffffffffu, ok && !stuck)) { failed = 1; break; }
          if (lane == 0) mbar_expect_tx(full + 8 * s, (uint32_t)(m * G * 16 * (HD / 4 + 1)));
          __syncwarp();
          if (lane < m) tma_load_3d(ring + s * R::STAGE + lane * slot_bytes, &map_merge, w.r0 * 4, 0, w.group_id + x + lane, full + 8 * s);
        }
      }
      if (lane == 0) ring_drain(n, R::STAGES, [&](int slot, uint32_t parity) { return long_wait(full + 8 * slot, parity); });   // its copies have arrived
      __syncwarp();
      n_tile = n;
    } else {
      // ---------------------------------------------------------------- the four warps
      int n = n_tile;
      bool bad = false, dead = false;         // bad: some warp of these gave up a wait; dead: this one did
      for (int i = 0; i < n_pieces && !bad; ++i) {
        const RowPiece w = list[i];
        // S^T = K Q^T and O^T += V^T P^T: the queries are the eight columns of an MMA, a warp's 16 keys its rows and then its depth.  A thread has
        // queries 2 tq and 2 tq + 1 (and 8 more behind them).
        uint32_t qb[KB][NQ][2];
        float o[MT][NQ][4], m_run[NQ][2], l_run[NQ][2];
#pragma unroll
        for (int x = 0; x < NQ; ++x) {
#pragma unroll
          for (int k = 0; k < MT; ++k) o[k][x][0] = o[k][x][1] = o[k][x][2] = o[k][x][3] = 0.f;
          m_run[x][0] = m_run[x][1] = -INFINITY;
          l_run[x][0] = l_run[x][1] = 0.f;
        }
        int kb = w.key0, s;
        for (;;) {
          s = ring_slot(n, R::STAGES);
          if (!dead && !wait(full + 8 * s, ring_parity(n, R::STAGES))) {
            dead = true;
            stuck = 1;
          }
          const uint32_t k_tile = ring + s * R::STAGE, v_tile = k_tile + R::KV_BYTES;
          const int keys = min(16, w.limit - kb - warp * 16);      // of this warp
          if (kb == w.key0) {
            // (rows from G on hold whatever lay there: a query's scores depend on nobody else's)
            const uint32_t q = v_tile + R::KV_BYTES;
#pragma unroll
            for (int k = 0; k < KB; k += 2)
#pragma unroll
              for (int x = 0; x < NQ; ++x)
                ldmatrix_x4(qb[k][x][0], qb[k][x][1], qb[k + 1][x][0], qb[k + 1][x][1], q + (x * 8 + (lane & 7)) * (HD * 2) + (2 * k + (lane >> 3)) * 16);
          }
          if (keys > 0) {
            uint32_t a[KB][4];
            const int row = warp * 16 + (lane & 7);
#pragma unroll
            for (int k = 0; k < KB; ++k) ldmatrix_x4(a[k][0], a[k][1], a[k][2], a[k][3], k_tile + tile_offset(row + ((lane >> 3) & 1) * 8, 2 * k + (lane >> 4)));
            float sc[NQ][4], odd[NQ][4];      // two chains of products: even and odd k-blocks
#pragma unroll
            for (int x = 0; x < NQ; ++x)
#pragma unroll
              for (int c = 0; c < 4; ++c) sc[x][c] = odd[x][c] = 0.f;
#pragma unroll
            for (int k = 0; k < KB; k += 2)
#pragma unroll
              for (int x = 0; x < NQ; ++x) {
                mma_bf16(sc[x], a[k], qb[k][x][0], qb[k][x][1]);
                mma_bf16(odd[x], a[k + 1], qb[k + 1][x][0], qb[k + 1][x][1]);
              }
            // V's fragments are asked for before the softmax, into the registers of K's: keys are the depth now
            uint32_t v[MT][4];
#pragma unroll
            for (int k = 0; k < MT; ++k)
              ldmatrix_x4_trans(v[k][0], v[k][1], v[k][2], v[k][3], v_tile + tile_offset(row + (lane >> 4) * 8, 2 * k + ((lane >> 3) & 1)));
            if (keys < 16) {
              // what lies behind the last key may be anything, and 0 times infinity is no zero
              const uint32_t low = (2 * tq < keys ? 0xffffu : 0u) | (2 * tq + 1 < keys ? 0xffff0000u : 0u);
              const uint32_t high = (2 * tq + 8 < keys ? 0xffffu : 0u) | (2 * tq + 9 < keys ? 0xffff0000u : 0u);
#pragma unroll
              for (int k = 0; k < MT; ++k) {
                v[k][0] &= low;
                v[k][1] &= low;
                v[k][2] &= high;
                v[k][3] &= high;
              }
            }
            uint32_t pb[NQ][2];
            bool moved = false;
            float keep[NQ][2];
#pragma unroll
            for (int x = 0; x < NQ; ++x) {
#pragma unroll
              for (int c = 0; c < 4; ++c) sc[x][c] = g + (c >> 1) * 8 < keys ? (sc[x][c] + odd[x][c]) * sl2 : -INFINITY;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float mx = fmaxf(sc[x][c], sc[x][c + 2]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                const float m_new = fmaxf(m_run[x][c], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
                keep[x][c] = fast_exp2(m_run[x][c] - m_use);       // 0 before the first key
                moved |= m_new != m_run[x][c];
                m_run[x][c] = m_new;
                sc[x][c] = fast_exp2(sc[x][c] - m_use);
                sc[x][c + 2] = fast_exp2(sc[x][c + 2] - m_use);
                l_run[x][c] = l_run[x][c] * keep[x][c] + (sc[x][c] + sc[x][c + 2]);        // the sum in 32 bits; the weights are rounded to bfloat16 for the product
              }
              pb[x][0] = transposed(pack_bf16(sc[x][0], sc[x][1]));
              pb[x][1] = transposed(pack_bf16(sc[x][2], sc[x][3]));
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
              for (int k = 0; k < MT; ++k)
#pragma unroll
                for (int x = 0; x < NQ; ++x)
#pragma unroll
                  for (int c = 0; c < 4; ++c) o[k][x][c] *= keep[x][c & 1];
            }
#pragma unroll
            for (int k = 0; k < MT; ++k)
#pragma unroll
              for (int x = 0; x < NQ; ++x) mma_bf16(o[k][x], v[k], pb[x][0], pb[x][1]);
          }
          ++n;
          kb += TILE;
          if (kb >= w.limit) break;       // (the last tile's stage is kept for what follows)
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + 8 * s);
        }
        // ---- the segment's end: the four warps' results added in the last tile's stage, under their common maximum
        float(*maxima)[ROWS] = s_max[i & 1], (*sums)[ROWS] = s_sum[i & 1];
#pragma unroll
        for (int x = 0; x < NQ; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l_run[x][c] += __shfl_xor_sync(0xffffffffu, l_run[x][c], d);
            if (g == 0) {
              maxima[warp][x * 8 + 2 * tq + c] = m_run[x][c];
              sums[warp][x * 8 + 2 * tq + c] = l_run[x][c];
            }
          }
        warps_barrier();
        bad = stuck != 0;       // set before this barrier or behind the next one: the same for all four warps
        if (bad) break;
        float* scratch = reinterpret_cast<float*>(smem + s * R::STAGE);       // [warp][query][HD + 4]
#pragma unroll
        for (int x = 0; x < NQ; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int q = x * 8 + 2 * tq + c;
            const float M = fmaxf(fmaxf(maxima[0][q], maxima[1][q]), fmaxf(maxima[2][q], maxima[3][q]));
            const float f = M == -INFINITY ? 0.f : fast_exp2(m_run[x][c] - M);
#pragma unroll
            for (int k = 0; k < MT; ++k) {
              scratch[(warp * ROWS_USED + q) * (HD + 4) + k * 16 + g] = o[k][x][c] * f;
              scratch[(warp * ROWS_USED + q) * (HD + 4) + k * 16 + g + 8] = o[k][x][c + 2] * f;
            }
          }
        warps_barrier();
        // from here on a thread has one query and PASSES times four columns (neighbouring threads have neighbouring queries, as the pieces lie)
        const int q = tid % ROWS_USED, c4 = tid / ROWS_USED;
        float M = fmaxf(fmaxf(maxima[0][q], maxima[1][q]), fmaxf(maxima[2][q], maxima[3][q])), L = 0.f;
        float4 acc[PASSES];
#pragma unroll
        for (int j = 0; j < PASSES; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int y = 0; y < WARPS; ++y) {
          L += M == -INFINITY ? 0.f : sums[y][q] * fast_exp2(maxima[y][q] - M);
#pragma unroll
          for (int j = 0; j < PASSES; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(scratch + (y * ROWS_USED + q) * (HD + 4) + (c4 + j * STEP) * 4);
            acc[j] = make_float4(acc[j].x + v.x, acc[j].y + v.y, acc[j].z + v.z, acc[j].w + v.w);
          }
        }
        fence_async_smem();       // the stage is TMA's again
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * s);
        // ``count`` pieces added, under their common maximum: piece y has {maximum, sum} at ml(y) and four columns at at(y, c)
        auto add = [&](int count, auto ml, auto at) {
          float2 m[MERGED];
          float m_new = M;
#pragma unroll
          for (int y = 0; y < MERGED; ++y) {
            m[y] = make_float2(-INFINITY, 0.f);
            if (y < count) m[y] = ml(y);
            m_new = fmaxf(m_new, m[y].x);
          }
          const float m_use = m_new == -INFINITY ? 0.f : m_new, have = fast_exp2(M - m_use);
          M = m_new;
          L *= have;
#pragma unroll
          for (int j = 0; j < PASSES; ++j) acc[j] = make_float4(acc[j].x * have, acc[j].y * have, acc[j].z * have, acc[j].w * have);
#pragma unroll
          for (int y = 0; y < MERGED; ++y)
            if (y < count) {
              const float f = fast_exp2(m[y].x - m_use);
              L = fmaf(f, m[y].y, L);
#pragma unroll
              for (int j = 0; j < PASSES; ++j) {
                const float4 v = at(y, c4 + j * STEP);
                acc[j] = make_float4(fmaf(f, v.x, acc[j].x), fmaf(f, v.y, acc[j].y), fmaf(f, v.z, acc[j].z), fmaf(f, v.w, acc[j].w));
              }
            }
        };
        if (w.index == 0)
          for (int x = 0; x < w.group_n; x += per_stage, ++n) {
            s = ring_slot(n, R::STAGES);
            if (!dead && !wait(full + 8 * s, ring_parity(n, R::STAGES))) {
              dead = true;
              stuck = 1;
            }
            const unsigned char* part = smem + s * R::STAGE + q * 16;
            if (q < G)
              add(min(per_stage, w.group_n - x), [&](int y) { return *reinterpret_cast<const float2*>(part + y * slot_bytes + HD / 4 * G * 16); },
                  [&](int y, int c) { return *reinterpret_cast<const float4*>(part + y * slot_bytes + c * G * 16); });
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * s);
          }
        bool finish = true;
        if (w.pieces > 1) {
          if (!waited) {          // the last call's pieces are nobody's any more
            asm volatile("griddepcontrol.wait;\n" ::: "memory");
            waited = true;
          }
          if (q < G) {
            float* part = row_results(p, w.first_id + w.index);
#pragma unroll
            for (int j = 0; j < PASSES; ++j) *reinterpret_cast<float4*>(part + (size_t)q * HD + (c4 + j * STEP) * 4) = acc[j];
            if (c4 == 0) *reinterpret_cast<float2*>(part + (size_t)G * HD + 2 * q) = make_float2(M, L);
          }
          __threadfence();
          warps_barrier();
          if (tid == 0) s_last = atomicAdd(&counters(p)[w.row * p.KV + w.kvh], 1) == w.pieces - 1;
          warps_barrier();
          finish = s_last != 0;
          if (finish && q < G) {
            __threadfence();
            const long long rs = row_piece_floats(G, HD);
            M = -INFINITY;
            L = 0.f;
            for (int x = 0; x < w.pieces; x += MERGED) {
              const float* from = row_results(p, w.first_id + x);
              add(min(MERGED, w.pieces - x), [&](int y) { return __ldcg(reinterpret_cast<const float2*>(from + y * rs + (size_t)G * HD + 2 * q)); },
                  [&](int y, int c) { return __ldcg(reinterpret_cast<const float4*>(from + y * rs + (size_t)q * HD + c * 4)); });
            }
          }
        }
        if (finish && q < G) {
          const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);      // no key: zeros; a NaN stays one
          __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out) + w.row * p.out_stride + (w.kvh * G + q) * HD;
#pragma unroll
          for (int j = 0; j < PASSES; ++j)
            *reinterpret_cast<uint2*>(out + (c4 + j * STEP) * 4) = make_uint2(pack_bf16(acc[j].x * inv, acc[j].y * inv), pack_bf16(acc[j].z * inv, acc[j].w * inv));
        }
      }
      n_tile = n;
    }
    __syncthreads();
    if (failed || stuck) {
      if (tid == 0) dk_report(p.err, DK_DEV_TIMEOUT, (int)blockIdx.x, (int)gridDim.x, n_pieces);
      break;
    }
  }
  asm volatile("griddepcontrol.wait;\n" ::: "memory");       // what follows this kernel follows the other one too
  if (blockIdx.x == 0 && tid == 0) asm volatile("st.relaxed.gpu.global.u64 [%0], %1;\n" ::"l"(list_of_call(p)), "l"(0ull) : "memory");      // (others may still look)
}

bool make_map_of_pieces(CUtensorMap* m, const float* base, int pieces, int G, int hd) {
  TensorMapEncodeFn fn = tensor_map_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {4 * QR, (cuuint64_t)(hd / 4 + 1), (cuuint64_t)pieces};
  const cuuint64_t strides[2] = {16 * QR, (cuuint64_t)(4 * group_piece_floats(QR, hd))};
  const cuuint32_t box[3] = {(cuuint32_t)(4 * G), (cuuint32_t)(hd / 4 + 1), 1}, one[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool LOW>
int launch(const DkSharedPrefixParams& p, cudaStream_t stream) {
  using R = Ring<HD, LOW>;
  CUtensorMap map_kv, map_run, map_merge;
  const int rows = p.ps < TILE ? p.ps : TILE;
  DK_REQUIRE(make_tensor_map_bf16(&map_kv, p.kv, (long long)p.num_pages * 2 * p.KV * p.ps, HD, HD, rows), "attention_shared_prefix: cannot encode the tensor map of the cache");
  // the cache as [page][K|V, head][offset][hd]: a run of pages of one head in one box
  const unsigned long long dims[4] = {(unsigned long long)HD, (unsigned long long)p.ps, (unsigned long long)(2 * p.KV), (unsigned long long)p.num_pages};
  const unsigned long long strides[3] = {(unsigned long long)HD * 2, (unsigned long long)p.ps * HD * 2, (unsigned long long)2 * p.KV * p.ps * HD * 2};
  DK_REQUIRE(make_tensor_map_bf16_4d(&map_run, p.kv, dims, strides, rows, TILE / rows), "attention_shared_prefix: cannot encode the tensor map of runs of pages");
  // the results of groups' pieces as [piece][hd / 4 + 1][queries x 4]: G queries of a piece in one box
  DK_REQUIRE(make_map_of_pieces(&map_merge, group_results(p, 0), p.group_pieces > 0 ? p.group_pieces : 1, p.H / p.KV, HD), "attention_shared_prefix: cannot encode the tensor map of the pieces");
  static bool configured_on[DK_MAX_DEVICES] = {false};
  bool& configured = configured_on[dk_current_device()];
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(attention_shared_prefix_rows_kernel<HD, LOW>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::TOTAL);
    if (e != cudaSuccess) {
      dk_set_error("attention_shared_prefix: cannot get %d bytes of shared memory: %s", R::TOTAL, cudaGetErrorString(e));
      return DK_ERR_LAUNCH;
    }
    configured = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows_grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = R::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // it may start while the kernel of the groups runs
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, attention_shared_prefix_rows_kernel<HD, LOW>, map_kv, map_run, map_merge, p);
  if (e != cudaSuccess) {
    dk_set_error("attention_shared_prefix: launch of the rows' kernel failed: %s", cudaGetErrorString(e));
    return DK_ERR_LAUNCH;
  }
  return dk_check_launch("attention_shared_prefix_rows");
}
}  // namespace

unsigned long long dk_shared_prefix_call_number() {
  static std::atomic<unsigned long long> calls{0};
  return 0x9e3779b97f4a7c15ull * (calls.fetch_add(1) + 1);       // (odd, so no two are alike; and never 0)
}
int dk_shared_prefix_rows_tile() { return TILE; }
int dk_shared_prefix_rows_grid(const DkSharedPrefixParams& p) { return (p.hd == 128 && p.H / p.KV > 8 ? 1 : 2) * dk_sm_count(); }
int dk_shared_prefix_rows_launch(const DkSharedPrefixParams& p, cudaStream_t stream) {
  const bool low = p.H / p.KV <= 8;
  if (p.hd == 64) return low ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
  return low ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}
