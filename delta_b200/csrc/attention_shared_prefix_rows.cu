// Attention over shared prefixes, bfloat16: the keys that each row holds alone, and the merge with the pieces that the
// kernel of the groups (attention_shared_prefix_tc.cu) leaves.
//
// A row's G <= 16 query heads of one key-value head are the rows of a warp-level MMA tile; the kernel is bound by the bytes of
// K and V, which nobody shares, so the legacy MMA is enough.  Two blocks run on an SM and take pieces in turn; their tiles of 64 keys flow
// through a ring without a stop between pieces:
//
//   warp 4     fetches by TMA: a tile's K and V (one box per 64 columns where its pages follow one another in the pool, else a
//              box per page; pages behind the last key are left out), and with a segment's first tile its queries
//   warps 0-3  S = Q K^T for 16 keys each, the maximum over the tile through shared memory, P in bfloat16 through shared
//              memory, O += P V for a quarter of the columns each.  So all warps share one maximum, and nothing has to be merged
//              between them at a segment's end.
//
// Behind a piece's last tile the pieces of its row's group are added to it, in the order of their keys: they come through the ring as well, up to eight
// a stage, one box each.  (Of a segment that is cut, only the first piece adds them.)  The result is rounded once.  Where a segment is cut, each block
// leaves its piece's results in the work buffer and counts itself; the one that comes last adds them all, in their order, so the result does not depend on
// who that is.  This kernel starts while that one runs and waits for its end before it touches what it wrote; the list of pieces and the cleared counters
// alone are there before: the block that writes them lets this kernel start when they are.
#include "shared_prefix.cuh"
#include "tcgen05_helpers.cuh"
#include "mma_helpers.cuh"
#include "ring.cuh"

namespace {
using namespace shared_prefix;
constexpr int TILE = 64;           // keys of a tile
constexpr int QR = 128;            // queries of a group's piece
constexpr int LISTED = 32;         // pieces whose records lie in shared memory at once
constexpr int MERGED = 8;          // pieces of a group in a stage, at most
constexpr int ROWS = 16;           // rows of the MMA tile
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

// LOW: at most 8 query heads; rows 8..15 of the MMA tile are then empty and their accumulators two registers that stay zero.
template <bool LOW>
__device__ __forceinline__ void mma_rows(float* c, float (&zero)[2], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (LOW) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(zero[0]), "+f"(zero[1])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
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
  constexpr int NR = LOW ? 1 : 2;             // rows of the tile a thread keeps (g, and g + 8)
  constexpr int KB = HD / 16;                 // k-blocks of Q K^T
  constexpr int NT = HD / WARPS / 8;          // n-tiles of P V of a warp
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long bars[2 * R::STAGES];   // full, then empty
  __shared__ RowPiece list[LISTED];
  __shared__ __align__(16) unsigned char s_p[ROWS * TILE * 2];      // weights [row][key], 16-byte chunks exchanged by the row
  __shared__ float s_max[WARPS][ROWS], s_sum[WARPS][ROWS];
  __shared__ int s_last;
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
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  const float sl2 = p.scale * 1.4426950408889634f;
  int n_tile = 0;                 // tiles this block has had
  bool waited = false;
  // the pieces of a group in a stage: G queries each in a slot of its own
  const int slot_bytes = (G * 16 * (HD / 4 + 1) + 127) / 128 * 128, per_stage = min(MERGED, R::STAGE / slot_bytes);
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
      bool bad = false;
      for (int i = 0; i < n_pieces && !bad; ++i) {
        const RowPiece w = list[i];
        uint32_t qa[KB][4];
        float o[NT][2 * NR], zero[2] = {0.f, 0.f}, m_run[NR], l_run[NR];
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int c = 0; c < 2 * NR; ++c) o[k][c] = 0.f;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          m_run[r] = -INFINITY;
          l_run[r] = 0.f;
        }
        int kb = w.key0;
        do {
          const int s = ring_slot(n, R::STAGES);
          if (!wait(full + 8 * s, ring_parity(n, R::STAGES))) stuck = 1;
          const uint32_t k_tile = ring + s * R::STAGE, v_tile = k_tile + R::KV_BYTES;
          const int keys = min(TILE, w.limit - kb);
          if (kb == w.key0 && keys > 0) {
            // (rows from G on hold whatever lay there: a row of the products depends on its own queries alone)
            const uint32_t q = v_tile + R::KV_BYTES;
            if (LOW) {
#pragma unroll
              for (int k = 0; k < KB; k += 2) {
                ldmatrix_x4(qa[k][0], qa[k][2], qa[k + 1][0], qa[k + 1][2], q + (lane & 7) * (HD * 2) + (2 * k + (lane >> 3)) * 16);
                qa[k][1] = qa[k][3] = qa[k + 1][1] = qa[k + 1][3] = 0u;
              }
            } else {
#pragma unroll
              for (int k = 0; k < KB; ++k)
                ldmatrix_x4(qa[k][0], qa[k][1], qa[k][2], qa[k][3], q + ((lane & 7) + ((lane >> 3) & 1) * 8) * (HD * 2) + (2 * k + (lane >> 4)) * 16);
            }
          }
          // fragments first, then four chains of products: even and odd k-blocks of two groups of eight keys
          float sc[2][2 * NR], odd[2][2 * NR], mx[NR];
          uint32_t kf[2][KB / 2][4];
#pragma unroll
          for (int k = 0; k < KB / 2; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              ldmatrix_x4(kf[j][k][0], kf[j][k][1], kf[j][k][2], kf[j][k][3], k_tile + tile_offset(warp * 16 + j * 8 + (lane & 7), 4 * k + (lane >> 3)));
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 2 * NR; ++c) sc[j][c] = odd[j][c] = 0.f;
#pragma unroll
          for (int k = 0; k < KB / 2; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma_rows<LOW>(sc[j], zero, qa[2 * k], kf[j][k][0], kf[j][k][1]);
              mma_rows<LOW>(odd[j], zero, qa[2 * k + 1], kf[j][k][2], kf[j][k][3]);
            }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 2 * NR; ++c) sc[j][c] += odd[j][c];
          // V's fragments are asked for before the softmax
          uint32_t vf[TILE / 16][NT / 2][4];
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk)
#pragma unroll
            for (int k = 0; k < NT / 2; ++k)
              ldmatrix_x4_trans(vf[kk][k][0], vf[kk][k][1], vf[kk][k][2], vf[kk][k][3],
                                v_tile + tile_offset(kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, warp * NT + 2 * k + (lane >> 4)));
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            mx[r] = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float& v = sc[j][2 * r + c];
                v = warp * 16 + j * 8 + 2 * tq + c < keys ? v * sl2 : -INFINITY;
                mx[r] = fmaxf(mx[r], v);
              }
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            if (tq == 0) s_max[warp][g + 8 * r] = mx[r];
          }
          warps_barrier();
          // written by these warps only, before this barrier or behind the next one: the same for all four
          bad = stuck != 0;
          if (bad) break;
          float keep[NR];
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const int row = g + 8 * r;
            const float m_new = fmaxf(fmaxf(m_run[r], fmaxf(s_max[0][row], s_max[1][row])), fmaxf(s_max[2][row], s_max[3][row]));
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            keep[r] = fast_exp2(m_run[r] - m_use);       // 0 before the first key
            m_run[r] = m_new;
            l_run[r] *= keep[r];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float p0 = fast_exp2(sc[j][2 * r] - m_use), p1 = fast_exp2(sc[j][2 * r + 1] - m_use);
              l_run[r] += p0 + p1;        // the sum in 32 bits; the weights are rounded to bfloat16 for the product
              const int key = warp * 16 + j * 8 + 2 * tq;
              *reinterpret_cast<uint32_t*>(s_p + row * (TILE * 2) + (((key >> 3) ^ (row & 7)) << 4) + (key & 7) * 2) = pack_bf16(p0, p1);
            }
          }
          warps_barrier();
#pragma unroll
          for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int c = 0; c < 2 * NR; ++c) o[k][c] *= keep[c >> 1];
          uint32_t a[TILE / 16][4];
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk) {
            const int arow = (lane & 7) + ((lane >> 3) & 1) * 8;      // rows 0-7, 8-15 of keys 0-7, then of keys 8-15
            ldmatrix_x4(a[kk][0], a[kk][1], a[kk][2], a[kk][3], s2u(s_p) + arow * (TILE * 2) + (((2 * kk + (lane >> 4)) ^ (arow & 7)) << 4));
            if (LOW) a[kk][1] = a[kk][3] = 0u;
          }
          if (keys < TILE) {
            // what lies behind the last key may be anything, and 0 times infinity is no zero
#pragma unroll
            for (int kk = 0; kk < TILE / 16; ++kk) {
              const int k0 = kk * 16 + 2 * tq;
              const uint32_t low = (k0 < keys ? 0xffffu : 0u) | (k0 + 1 < keys ? 0xffff0000u : 0u);
              const uint32_t high = (k0 + 8 < keys ? 0xffffu : 0u) | (k0 + 9 < keys ? 0xffff0000u : 0u);
#pragma unroll
              for (int k = 0; k < NT / 2; ++k) {
                vf[kk][k][0] &= low;
                vf[kk][k][1] &= high;
                vf[kk][k][2] &= low;
                vf[kk][k][3] &= high;
              }
            }
          }
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk)
#pragma unroll
            for (int k = 0; k < NT / 2; ++k) {
              mma_rows<LOW>(o[2 * k], zero, a[kk], vf[kk][k][0], vf[kk][k][1]);
              mma_rows<LOW>(o[2 * k + 1], zero, a[kk], vf[kk][k][2], vf[kk][k][3]);
            }
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + 8 * s);
          ++n;
          kb += TILE;
        } while (kb < w.limit);
        if (bad) break;
        // ---- the segment's end: sums over the warps, then the merge
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
          l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
          if (tq == 0) s_sum[warp][g + 8 * r] = l_run[r];
        }
        warps_barrier();
#pragma unroll
        for (int r = 0; r < NR; ++r) l_run[r] = (s_sum[0][g + 8 * r] + s_sum[1][g + 8 * r]) + (s_sum[2][g + 8 * r] + s_sum[3][g + 8 * r]);
        // {maximum, sum, outputs} of a piece added to this thread's queries
        auto add = [&](int r, float m, float l, const float (&v)[2 * NT]) {
          const float m_new = fmaxf(m_run[r], m), m_use = m_new == -INFINITY ? 0.f : m_new;
          const float have = fast_exp2(m_run[r] - m_use), f = fast_exp2(m - m_use);
          m_run[r] = m_new;
          l_run[r] = l_run[r] * have + l * f;
#pragma unroll
          for (int k = 0; k < 2 * NT; ++k) o[k / 2][2 * r + k % 2] = o[k / 2][2 * r + k % 2] * have + v[k] * f;
        };
        if (w.index == 0)
          for (int x = 0; x < w.group_n; x += per_stage, ++n) {
            const int s = ring_slot(n, R::STAGES), m = min(per_stage, w.group_n - x);
            if (!wait(full + 8 * s, ring_parity(n, R::STAGES))) stuck = 1;
            // the stage's pieces at once: their common maximum first, so that nothing but the sums is done one after the other
            const unsigned char* part = smem + s * R::STAGE;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              const int qh = g + 8 * r;
              if (qh >= G) continue;
              float f[MERGED], m_new = m_run[r];
#pragma unroll
              for (int y = 0; y < MERGED; ++y) {
                f[y] = y < m ? *reinterpret_cast<const float*>(part + y * slot_bytes + (HD / 4 * G + qh) * 16) : -INFINITY;
                m_new = fmaxf(m_new, f[y]);
              }
              const float m_use = m_new == -INFINITY ? 0.f : m_new, have = fast_exp2(m_run[r] - m_use);
              m_run[r] = m_new;
              l_run[r] *= have;
#pragma unroll
              for (int k = 0; k < 2 * NT; ++k) o[k / 2][2 * r + k % 2] *= have;
#pragma unroll
              for (int y = 0; y < MERGED; ++y)
                if (y < m) {
                  const unsigned char* from = part + y * slot_bytes;
                  const float w_y = fast_exp2(f[y] - m_use);
                  l_run[r] += w_y * *reinterpret_cast<const float*>(from + (HD / 4 * G + qh) * 16 + 4);
#pragma unroll
                  for (int k = 0; k < NT; ++k) {
                    const float2 v = *reinterpret_cast<const float2*>(from + (((warp * NT + k) * 2 + tq / 2) * G + qh) * 16 + (tq & 1) * 8);
                    o[k][2 * r] = fmaf(w_y, v.x, o[k][2 * r]);
                    o[k][2 * r + 1] = fmaf(w_y, v.y, o[k][2 * r + 1]);
                  }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * s);
          }
        bool finish = true;
        if (w.pieces > 1) {
          if (!waited) {          // the counters were cleared by the kernel of the groups
            asm volatile("griddepcontrol.wait;\n" ::: "memory");
            waited = true;
          }
          float* part = row_results(p, w.first_id + w.index);
#pragma unroll
          for (int r = 0; r < NR; ++r)
            if (g + 8 * r < G) {
#pragma unroll
              for (int k = 0; k < NT; ++k)
                *reinterpret_cast<float2*>(part + (size_t)(g + 8 * r) * HD + (warp * NT + k) * 8 + 2 * tq) = make_float2(o[k][2 * r], o[k][2 * r + 1]);
              if (warp == 0 && tq == 0) *reinterpret_cast<float2*>(part + (size_t)G * HD + 2 * (g + 8 * r)) = make_float2(m_run[r], l_run[r]);
            }
          __threadfence();
          warps_barrier();
          if (tid == 0) s_last = atomicAdd(&counters(p)[w.row * p.KV + w.kvh], 1) == w.pieces - 1;
          warps_barrier();
          finish = s_last != 0;
          if (finish) {
            __threadfence();
            constexpr int AT_ONCE = 4;        // pieces asked for together, added in order
            const long long rs = row_piece_floats(G, HD);
            const float* rp = row_results(p, w.first_id);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              m_run[r] = -INFINITY;
              l_run[r] = 0.f;
#pragma unroll
              for (int k = 0; k < NT; ++k) o[k][2 * r] = o[k][2 * r + 1] = 0.f;
              if (g + 8 * r >= G) continue;
              for (int x = 0; x < w.pieces; x += AT_ONCE) {
                float2 ml[AT_ONCE];
                float v[AT_ONCE][2 * NT];
#pragma unroll
                for (int y = 0; y < AT_ONCE; ++y)
                  if (x + y < w.pieces) {
                    const float* from = rp + (x + y) * rs;
                    ml[y] = __ldcg(reinterpret_cast<const float2*>(from + (size_t)G * HD + 2 * (g + 8 * r)));
#pragma unroll
                    for (int k = 0; k < NT; ++k) {
                      const float2 f = __ldcg(reinterpret_cast<const float2*>(from + (size_t)(g + 8 * r) * HD + (warp * NT + k) * 8 + 2 * tq));
                      v[y][2 * k] = f.x;
                      v[y][2 * k + 1] = f.y;
                    }
                  }
#pragma unroll
                for (int y = 0; y < AT_ONCE; ++y)
                  if (x + y < w.pieces) add(r, ml[y].x, ml[y].y, v[y]);
              }
            }
          }
        }
        if (finish) {
#pragma unroll
          for (int r = 0; r < NR; ++r)
            if (g + 8 * r < G) {
              const float inv = l_run[r] > 0.f ? 1.f / l_run[r] : (l_run[r] == 0.f ? 0.f : l_run[r]);      // no key: zeros; a NaN stays one
              __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out) + w.row * p.out_stride + (w.kvh * G + g + 8 * r) * HD;
#pragma unroll
              for (int k = 0; k < NT; ++k)
                *reinterpret_cast<__nv_bfloat162*>(out + (warp * NT + k) * 8 + 2 * tq) = __floats2bfloat162_rn(o[k][2 * r] * inv, o[k][2 * r + 1] * inv);
            }
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

int dk_shared_prefix_rows_tile() { return TILE; }
int dk_shared_prefix_rows_grid(const DkSharedPrefixParams& p) { return (p.hd == 128 && p.H / p.KV > 8 ? 1 : 2) * dk_sm_count(); }
int dk_shared_prefix_rows_launch(const DkSharedPrefixParams& p, cudaStream_t stream) {
  const bool low = p.H / p.KV <= 8;
  if (p.hd == 64) return low ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
  return low ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
}
