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
//               else a box per page.  Pages behind the piece's last key are not fetched.
//   warp 10     issues the score products
//   warp 11     issues P V over the 16-key blocks that hold keys, and clears what the last of them holds behind the last key
//               (a page's rest may hold anything, and 0 times infinity is no zero)
//   warps 8-11  together make the list of the range's pieces
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
  static constexpr int OFF_K = OFF_Q + Q_BYTES;           // two of each; the list is made here, before they are filled
  static constexpr int OFF_V = OFF_K + 2 * TILE_BYTES;
  static constexpr int OFF_P = OFF_V + 2 * TILE_BYTES;    // P of each half: two boxes [128 x 64 keys]
  static constexpr int P_BYTES = 2 * BOX_BYTES;
  static constexpr int TOTAL = OFF_P + 2 * P_BYTES + 1024;   // 1024 to start on a swizzle boundary
  static_assert(4 * Cut::ints(0, MAX_GROUPS) <= 4 * TILE_BYTES, "the list is made in the buffers of K and V");
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
  asm volatile("bar.sync 2, %0;\n" ::"n"(THREADS) : "memory");
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
  __shared__ int n_listed, ranges_left;
  // row_stat(w)[query]: maximum and sum of half w's tiles, over the half's P, which is not read any more by then
  auto row_stat = [&](int w) { return reinterpret_cast<float2*>(smem + L::OFF_P + w * L::P_BYTES); };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");      // the rows' kernel may start wherever there is room
  for (int i = blockIdx.x * THREADS + tid; i < p.rows * p.KV; i += gridDim.x * THREADS) counters(p)[i] = 0;
  const int ps = p.ps, G = p.G;
  const uint32_t bar0 = s2u(&bars[0]);
  const uint32_t q_full = bar0, k_full = bar0 + 8, v_full = k_full + 16, s_full = v_full + 16, p_full = s_full + 16, o_done = p_full + 16,
                 s_free = o_done + 16, merge_bar = s_free + 16, piece_done = merge_bar + 8;
  if (tid == 0) {
    mbar_init(q_full, 2 * HALF_THREADS);
    for (int w = 0; w < 2; ++w) {
      mbar_init(k_full + 8 * w, 1);
      mbar_init(v_full + 8 * w, 1);
      mbar_init(s_full + 8 * w, 1);
      mbar_init(p_full + 8 * w, HALF_THREADS);
      mbar_init(o_done + 8 * w, 1);
      mbar_init(s_free + 8 * w, HALF_THREADS);
    }
    mbar_init(merge_bar, 2 * HALF_THREADS);
    mbar_init(piece_done, 2 * HALF_THREADS);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(s2u(&tmem_slot), TMEM_COLS);
  if (warp == PRODUCER_WARP0 && lane < 2)
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(lane ? &map_run : &map_kv)) : "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t sm_q = s2u(smem + L::OFF_Q), sm_k = s2u(smem + L::OFF_K), sm_v = s2u(smem + L::OFF_V), sm_p = s2u(smem + L::OFF_P);
  int had0 = 0, had1 = 0;   // tiles of each parity in the pieces before the current one
  int n_done = 0;           // pieces before the current one

  // 384 threads x 168 registers = 128 x 64 + 256 x 216 and some
  if (warp >= PRODUCER_WARP0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n");
    int asked0 = 0, asked1 = 0;   // producers: tiles of each parity asked for so far
    const int kind = warp - PRODUCER_WARP0;     // 0: K, 1: V
    const uint32_t full = kind ? v_full : k_full, done = kind ? o_done : s_full, sm_dst = kind ? sm_v : sm_k;
    for (int range = blockIdx.x;; range += gridDim.x) {
      {
        const int t4 = tid - PRODUCER_WARP0 * 32;
        auto sync = [] { asm volatile("bar.sync 1, 128;\n" ::: "memory"); };
        Cut cut(reinterpret_cast<int*>(smem + L::OFF_K), 0, p.groups);
        make_cut<false, KT, KT, 128>(p, cut, t4, sync);
        int n = 0, first_seg = 0;
        if (range < cut.ranges) n = min(range_pieces<KT>(p, cut, range, first_seg), CAP);
        if (t4 < n) list[t4] = group_piece<KT>(p, cut, range, first_seg + t4);
        if (t4 == 0) {
          n_listed = n;
          ranges_left = range + (int)gridDim.x < cut.ranges;
        }
        fence_async_smem();       // the buffers are TMA's from here on
      }
      block_barrier();
      const int n_pieces = n_listed;       // (read before the second barrier: behind it the next list is made)
      const bool more = ranges_left != 0;
      if (warp < MMA_WARP) {
        // ----------------------------------------------------------- producers
        const int ppt = KT / ps;      // pages per tile, at most 16
        for (int i = 0; i < n_pieces && !failed; ++i) {
          const GroupPiece w = list[i];
          const int n_tiles = cdiv(w.limit - w.key0, KT);
          const int* table = p.block_table + (size_t)w.table_row * p.max_pages;
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
            if (ord >= 1) ok = mbar_wait(done + 8 * c, (ord - 1) & 1);
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
      } else if (warp == MMA_WARP) {
        // ------------------------------------------- issuer of the scores
        const bool leader = elect_one();
        const uint32_t idesc_s = instr_desc_bf16(QT, KT, false);
        auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); };
        const uint64_t da0 = smem_desc_k_major(sm_q);
        bool ok = true;
        for (int i = 0; ok && i < n_pieces; ++i) {
          const GroupPiece w = list[i];
          const int n_tiles = cdiv(w.limit - w.key0, KT);
          ok = wait_all(q_full, n_done & 1);
          int j = 0;
          for (; ok && j < n_tiles; ++j) {
            const int c = j & 1, ord = (c ? had1 : had0) + j / 2;
            if (ord >= 1 && !wait_all(s_free + 8 * c, (ord - 1) & 1)) { ok = false; break; }
            if (!wait_all(k_full + 8 * c, ord & 1)) { ok = false; break; }
            tc_fence_after();
            const uint64_t db0 = smem_desc_k_major(sm_k + c * L::TILE_BYTES);
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk) {
                const uint64_t off = (uint64_t)(((kk / 4) * BOX_BYTES + (kk % 4) * 32) >> 4);   // start addresses count 16 bytes
                umma(tmem + COL_S + c * KT, da0 + off, db0 + off, idesc_s, kk > 0 ? 1u : 0u);
              }
              umma_commit(s_full + 8 * c);
            }
            __syncwarp();
          }
          had0 += (j + 1) / 2;
          had1 += j / 2;
          ++n_done;
        }
        if (!ok) failed = 1;
      } else {
        // ------------------------------------------ issuer of P V
        const bool leader = elect_one();
        const uint32_t idesc_o = instr_desc_bf16(QT, HD, true);
        auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); };
        bool ok = true;
        for (int i = 0; ok && i < n_pieces; ++i) {
          const GroupPiece w = list[i];
          const int n_tiles = cdiv(w.limit - w.key0, KT);
          int j = 0;
          for (; ok && j < n_tiles; ++j) {
            const int c = j & 1, ord = (c ? had1 : had0) + j / 2;
            if (!wait_all(v_full + 8 * c, ord & 1)) { ok = false; break; }
            const int n = min(KT, w.limit - w.key0 - j * KT), blocks = cdiv(n, 16);
            if (n % 16 != 0) {          // rows n to 16 blocks - 1 of both halves, eight 16-byte chunks each
              const int chunks = (blocks * 16 - n) * 8;
              for (int x = lane; x < chunks * L::HALVES; x += 32)
                *reinterpret_cast<uint4*>(smem + L::OFF_V + c * L::TILE_BYTES + x / chunks * BOX_BYTES + n * 128 + x % chunks * 16) = make_uint4(0u, 0u, 0u, 0u);
              fence_async_smem();
              __syncwarp();
            }
            if (!wait_all(p_full + 8 * c, ord & 1)) { ok = false; break; }
            tc_fence_after();
            const uint64_t dp0 = smem_desc_k_major(sm_p + c * L::P_BYTES);
            const uint64_t dv0 = smem_desc_mn_major(sm_v + c * L::TILE_BYTES, BOX_BYTES);
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < KT / 16; ++kk)   // 16 keys further: 32 bytes along a row of P, two groups of 8 rows of V
                if (kk < blocks)
                  umma(tmem + COL_O + c * HD, dp0 + (uint64_t)(((kk / 4) * BOX_BYTES + (kk % 4) * 32) >> 4),
                       dv0 + (uint64_t)(kk * (2048 >> 4)), idesc_o, (j > 1 || kk > 0) ? 1u : 0u);
              umma_commit(o_done + 8 * c);
            }
            __syncwarp();
          }
          had0 += (j + 1) / 2;
          had1 += j / 2;
        }
        if (!ok) failed = 1;
      }
      block_barrier();
      if (failed || !more) break;
    }
    if (lane == 0) {      // what this warp has under way ends before the block leaves
      const uint32_t bar = warp < MMA_WARP ? full : (warp == MMA_WARP ? s_full : o_done);
      ring_drain(warp < MMA_WARP ? asked0 : had0, 1, [&](int, uint32_t parity) { return mbar_wait(bar, parity); });
      ring_drain(warp < MMA_WARP ? asked1 : had1, 1, [&](int, uint32_t parity) { return mbar_wait(bar + 8, parity); });
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
    // ------------------------------------------------------------- softmax
    const int w = warp >> 2;                            // which half: its tiles are w, w + 2, ...
    const int r = (warp & 3) * 32 + lane;               // query of this thread = lane of the TMEM
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_base + COL_S + w * KT;
    const uint32_t t_o = tmem + lane_base + COL_O + w * HD;
    const float sl2 = p.scale * 1.4426950408889634f;
    constexpr int QC = HD / 16;                         // 16-byte chunks of a query that this half fetches
    const int qi = r / G, qh = r - qi * G;
    auto ask_q = [&](const GroupPiece& pc, uint4 (&v)[QC]) {
      int row = -1;
      if (qi < pc.rows) row = p.members[pc.first + qi];
      const bool held = row >= 0 && row < p.rows;
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.q) + (held ? row : 0) * p.q_stride + (pc.kvh * G + qh) * HD + w * (HD / 2));
#pragma unroll
      for (int c = 0; c < QC; ++c) v[c] = held ? src[c] : make_uint4(0u, 0u, 0u, 0u);
    };
    auto store_q = [&](const uint4 (&v)[QC]) {
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        const int col = w * QC + c;       // 16-byte chunk of the query's row
        *reinterpret_cast<uint4*>(smem + L::OFF_Q + (col / 8) * BOX_BYTES + r * 128 + (((col % 8) ^ (r & 7)) << 4)) = v[c];
      }
      fence_async_smem();
      mbar_arrive(q_full);
    };
    bool good = true;
    int had_w = 0, had_other = 0;       // tiles of this half and of the other one so far
    // While the list is made these warps walk once through what they do with a tile and at a piece's end, on whatever lies in the buffers, without a wait,
    // an arrival or a store to global memory: the instructions are fetched then and not behind the first scores (3.2 us for a first tile against 1.9).
    bool dry = true;
    for (;;) {
      int n_pieces = 1;
      bool more = true;
      if (!dry) {
        block_barrier();
        n_pieces = n_listed;       // (read before the second barrier: behind it the next list is made)
        more = ranges_left != 0;
        if (n_pieces > 0) {
          uint4 v[QC];
          ask_q(list[0], v);
          store_q(v);
        }
      }
#pragma unroll 1
      for (int i = 0; good && i < n_pieces; ++i) {
        GroupPiece pc;
        if (dry) pc = {0, 0, 0, 0, 0, 2 * KT - 1, 0, 0};
        else pc = list[i];
        const int n_tiles = cdiv(pc.limit - pc.key0, KT), queries = pc.rows * G;
        const bool busy = dry || (warp & 3) * 32 < queries;      // some thread of this warp has a query
        float m_used = -INFINITY, l_sum = 0.f;
        int mine = 0;
        // P (under which the maxima and sums of the piece before lay) and the accumulators are free again
        if (n_done > 0) {
          bool ok = mbar_wait(piece_done, (n_done - 1) & 1);
          if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
        }
        for (int j = w; j < n_tiles; j += 2, ++mine) {
          const int ord = had_w + mine;
          bool ok = dry || mbar_wait(s_full + 8 * w, ord & 1);
          if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
          tc_fence_after();
          if (!busy) {
            mbar_arrive(s_free + 8 * w);
            if (mine > 0) {
              ok = mbar_wait(o_done + 8 * w, (ord - 1) & 1);
              if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
            }
            mbar_arrive(p_full + 8 * w);
            continue;
          }
          float v[KT];
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) tmem_ld32_nowait(t_s + c * 32, v + c * 32);
          tmem_wait_ld();
          tc_fence_before();
          if (!dry) mbar_arrive(s_free + 8 * w);
          const int n = pc.limit - pc.key0 - j * KT;
          if (n < KT) {
#pragma unroll
            for (int k = 0; k < KT; ++k)
              if (k >= n) v[k] = -INFINITY;
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // four chains instead of one long one
#pragma unroll
          for (int k = 0; k < KT; k += 4) {
            mx4[0] = fmaxf(mx4[0], v[k]);
            mx4[1] = fmaxf(mx4[1], v[k + 1]);
            mx4[2] = fmaxf(mx4[2], v[k + 2]);
            mx4[3] = fmaxf(mx4[3], v[k + 3]);
          }
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          const float m_new = fmaxf(m_used, mx * sl2);
          const bool grow = m_new > m_used + RESCALE_STEP;      // also the first finite maximum of a row
          float factor = 1.f;
          if (grow) {
            factor = m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_new);
            m_used = m_new;
          }
          const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
          if (mine > 0) {
            // P V of this half's tile before is done: its P may be overwritten, and O_w is at rest
            ok = mbar_wait(o_done + 8 * w, (ord - 1) & 1);
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
          // exponentials, their sum in 32 bits, and P rounded to bfloat16 (what the product takes) in the layout of a 128-byte swizzle
          float sum4[4] = {0.f, 0.f, 0.f, 0.f};
          const uint32_t p_row = sm_p + w * L::P_BYTES + r * 128;
#pragma unroll
          for (int c = 0; c < KT / 8; ++c) {
            float e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              e[k] = fast_exp2(fmaf(v[c * 8 + k], sl2, neg_m));
              sum4[k & 3] += e[k];
            }
            const uint32_t addr = p_row + (c / 8) * BOX_BYTES + (((c % 8) ^ (r & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(pack2(e[0], e[1])), "r"(pack2(e[2], e[3])),
                         "r"(pack2(e[4], e[5])), "r"(pack2(e[6], e[7])) : "memory");
          }
          l_sum = l_sum * factor + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
          fence_async_smem();
          if (!dry) mbar_arrive(p_full + 8 * w);
        }
        // the next piece's queries, under way while the last products run; stored when all scores of this piece are made
        if (!dry) {
          had_w += (n_tiles + 1 - w) / 2;
          had_other += (n_tiles + w) / 2;
        }
        if (good && !dry) {
          bool ok = true;
          if (i + 1 < n_pieces) {
            uint4 v[QC];
            ask_q(list[i + 1], v);
            if (had_other > 0) ok = mbar_wait(s_full + 8 * (w ^ 1), (had_other - 1) & 1);
            store_q(v);
          }
          if (mine > 0) ok = mbar_wait(o_done + 8 * w, (had_w - 1) & 1) && ok;
          if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; }
        }
        // merge of the two halves: each tells the other its maximum and sum, then writes half of the columns
        if (!good) break;
        row_stat(w)[r] = make_float2(m_used, l_sum);
        tc_fence_before();
        if (!dry) mbar_arrive(merge_bar);
        {
          bool ok = dry || mbar_wait(merge_bar, n_done & 1);
          if (!__all_sync(0xffffffffu, ok && !failed)) { failed = 1; good = false; break; }
        }
        tc_fence_after();
        const float2 other = row_stat(w ^ 1)[r];
        const float m_all = fmaxf(m_used, other.x);
        const float f_mine = m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_all);
        const float f_other = other.x == -INFINITY ? 0.f : fast_exp2(other.x - m_all);
        const float l_all = l_sum * f_mine + other.y * f_other;
        const float f0 = w == 0 ? f_mine : f_other, f1 = w == 0 ? f_other : f_mine;
        const bool two = n_tiles > 1;                     // O_1 holds nothing when there was one tile
        float* part = group_results(p, pc.id);
        if (!busy) {
          tc_fence_before();
          mbar_arrive(piece_done);
        } else {
          constexpr int OC = HD / 64;                       // chunks of 32 columns this thread writes
#pragma unroll
          for (int c = 0; c < OC; ++c) {
            float o0[32], o1[32];
            const uint32_t col = (uint32_t)(w * (HD / 2) + c * 32);
            tmem_ld32_nowait(tmem + lane_base + COL_O + col, o0);
            if (two) tmem_ld32_nowait(tmem + lane_base + COL_O + HD + col, o1);
            tmem_wait_ld();
            if (c == OC - 1) {
              // accumulators and the other half's maximum and sum are in registers: the next piece may overwrite them
              tc_fence_before();
              if (!dry) mbar_arrive(piece_done);
            }
            if (r < queries) {
#pragma unroll
              for (int k = 0; k < 32; ++k) o0[k] = two ? o0[k] * f0 + o1[k] * f1 : o0[k] * f0;
#pragma unroll
              for (int k = 0; k < 8; ++k)
                *reinterpret_cast<float4*>(part + ((size_t)(col / 4 + k) * QT + r) * 4) = make_float4(o0[4 * k], o0[4 * k + 1], o0[4 * k + 2], o0[4 * k + 3]);
            }
          }
          if (r < queries && w == 0) *reinterpret_cast<float4*>(part + (size_t)QT * HD + 4 * r) = make_float4(m_all, l_all, 0.f, 0.f);
        }
        if (!dry) ++n_done;
      }
      if (dry) {
        dry = false;
        continue;
      }
      block_barrier();
      if (failed || !more) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (failed && tid == 0) dk_report(p.err, DK_DEV_TIMEOUT, (int)blockIdx.x, (int)gridDim.x, n_listed);
  if (warp == MMA_WARP) tmem_dealloc(tmem, TMEM_COLS);
}

template <int HD>
int launch(const DkSharedPrefixParams& p, cudaStream_t stream) {
  using L = Layout<HD>;
  CUtensorMap map_kv, map_run;
  const long long kv_rows = (long long)p.num_pages * 2 * p.KV * p.ps;
  DK_REQUIRE(kv_rows < (1ll << 31), "attention_shared_prefix: the cache of one layer has too many rows for a tensor map coordinate");
  DK_REQUIRE(make_tensor_map_bf16(&map_kv, p.kv, kv_rows, HD, HD, p.ps), "attention_shared_prefix: cannot encode the tensor map of the cache");
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
  attention_shared_prefix_tc_kernel<HD><<<p.groups > 0 ? p.grid : 1, THREADS, L::TOTAL, stream>>>(map_kv, map_run, p);      // (one block clears the counters)
  return dk_check_launch("attention_shared_prefix_tc");
}
}  // namespace

bool dk_shared_prefix_tc_takes(const DkSharedPrefixParams& p) {
  return p.dtype == DK_BF16 && p.H / p.KV <= 16 && (p.hd == 64 || p.hd == 128) && (p.ps == 8 || p.ps == 16 || p.ps == 32 || p.ps == 64 || p.ps == 128) &&
         (long long)p.num_pages * 2 * p.KV * p.ps < (1ll << 31);
}

int dk_shared_prefix_tc_launch(const DkSharedPrefixParams& p, cudaStream_t stream) { return p.hd == 64 ? launch<64>(p, stream) : launch<128>(p, stream); }
