// Attention of single tokens whose rows share leading pages: each row r of the batch has one query per head and
// reads kv_len[r] keys through its row of the block table,
//
//   out[r, h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(scale q[r, h] K[j] - m),   j < kv_len[r],
//
// and the rows of a group read the same first keys, which are fetched once for all of them (shared_prefix.cuh cuts
// the work).  A first kernel leaves, for every piece, the outputs relative to the piece's own maximum with that
// maximum and the sum; a second one merges the pieces of a row, which are few, in the order of their keys:
//
//   m = max_i m_i,   out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i      (maxima in units of log2).
//
// This file holds the merge and the kernel on the FMA units: 32-bit keys and values, and every head size and page
// size that the kernels on the tensor cores (attention_shared_prefix_tc.cu, attention_shared_prefix_rows.cu) do not take.  A block of 128 threads
// keeps 32 queries; K and V of a tile of 32 keys lie in shared memory as floats, and those of the next tile are on their way while this one is
// computed.  A thread has four queries and two keys of the scores, then four queries and eight columns of the result, two products to an instruction.
//
// 8 rows of 32 query heads on 4 of 128 behind 2,048 shared keys: 35.0 us.  Of these 2.7 go into the tables, 1 into the list of pieces, 5 until the first
// keys are there, 7.5 into a tile with two or three blocks to an SM, 2 into a piece's results and 5 into the merge.  32 rows behind 4,096 keys and 8 behind 1,000: 134 us, a quarter of
// the FMA units' rate: latency of shared memory between four barriers a tile, which three warps to a scheduler do not hide.  (A fourth block to an SM: 40 us for
// the small call, since its ranges are half as long and the merge reads twice the pieces.  Weights kept twice, ready to be multiplied in pairs: 36.4.  Loops rolled
// to two steps: 35.7 and 142.  Tiles of 64 keys with 4 x 4 scores to a thread and two blocks to an SM: 55 and 171.)
#include "shared_prefix.cuh"
#include "mma_helpers.cuh"

// attention_shared_prefix_tc.cu
bool dk_shared_prefix_tc_takes(const DkSharedPrefixParams& p);
int dk_shared_prefix_tc_launch(const DkSharedPrefixParams& p, cudaStream_t stream);
// attention_shared_prefix_rows.cu
unsigned long long dk_shared_prefix_call_number();
int dk_shared_prefix_rows_tile();
int dk_shared_prefix_rows_grid(const DkSharedPrefixParams& p);
int dk_shared_prefix_rows_launch(const DkSharedPrefixParams& p, cudaStream_t stream);

namespace {
using namespace shared_prefix;
constexpr int QR = 32;        // queries of a tile
constexpr int KT = 32;        // keys of a tile
constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int SHARE = 16;     // threads that share four queries
constexpr int P_STRIDE = QR + 4;
constexpr int BLOCKS = 3;     // of an SM

// rows four floats apart from a multiple of 32: threads that read neighbouring rows meet no bank twice
__host__ __device__ constexpr int row_stride(int hd) { return hd + 4; }
static size_t smem_floats(int hd) { return (size_t)(QR + 2 * KT) * row_stride(hd) + (size_t)KT * P_STRIDE; }

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&raw.x), b = *reinterpret_cast<const __nv_bfloat162*>(&raw.y);
  return make_float4(__low2float(a), __high2float(a), __low2float(b), __high2float(b));
}

// Two floats in one register pair: a product and a sum of both is one instruction.
using two = unsigned long long;
__device__ __forceinline__ two pack(float a, float b) {
  two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(two v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ two fma2(two a, two b, two c) {
  two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ two mul2(two a, two b) {
  two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// HDM: the head size rounded up to 64, 128 or 256 (sizes the registers)
template <typename T, int HDM>
__global__ void __launch_bounds__(THREADS, HDM <= 128 ? BLOCKS : 1) attention_shared_prefix_kernel(const DkSharedPrefixParams p) {
  constexpr int OC = HDM <= 64 ? 1 : HDM / 64;     // groups of four output columns of a thread
  extern __shared__ __align__(16) float smem[];
  const int hd = p.hd, ks = row_stride(hd);
  float* s_q = smem;                   // [QR][hd + 4]
  float* s_k = s_q + QR * ks;          // [KT][hd + 4]
  float* s_v = s_k + KT * ks;          // [KT][hd + 4]
  float* s_p = s_v + KT * ks;          // [KT][QR + 4]
  __shared__ GroupPiece list[CAP];
  __shared__ long long s_row[2][KT];   // where a key's row of K begins in the cache, -1: there is none; of this tile and the next
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q4 = tid / SHARE * 4, c = tid % SHARE;
  const int G = p.G, inv_g = 65535 / G + 1;        // x / G = x * inv_g >> 16 for the x below QR
  const float sl2 = p.scale * 1.4426950408889634f;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");      // the merge may be put in place (it waits for this kernel's end)
  Cut cut(reinterpret_cast<int*>(smem), p.rows, p.groups);
  auto tables = [&] { make_cut<KT, KT, 2, THREADS>(p, cut, tid); };
  tables();
  // every row's first piece for the merge
  if (blockIdx.x == 0)
    for (int i = tid; i < p.rows * p.KV; i += THREADS) {
      const int row = i / p.KV, n = ((row + 1 < p.rows ? cut.piece[row + 1] : cut.pieces) - cut.piece[row]) / p.KV;
      row_pieces(p)[i] = row_piece<KT, KT>(p, cut, cut.piece[row] + i % p.KV * n);
    }
  const int n_ranges = cut.ranges, n_row_pieces = cut.pieces;
  // first the pieces of the block's ranges of groups, then its pieces of rows
  int range = blockIdx.x, next_row = gridDim.x - 1 - blockIdx.x, listed = 0, at = 0;
  bool of_group = range < n_ranges, list_made = false;
  for (;;) {
    if (at == listed) {
      // a list of pieces at a time; the tables are laid out where the tiles lie
      if (list_made) tables();
      list_made = true;
      at = listed = 0;
      of_group = range < n_ranges;
      if (of_group) {
        int first_seg;
        listed = min(range_pieces<KT>(p, cut, range, first_seg), CAP);
        if (tid < listed) list[tid] = group_piece<KT>(p, cut, range, first_seg + tid);
        range += gridDim.x;
      } else if (next_row < n_row_pieces) {
        listed = min(CAP, cdiv(n_row_pieces - next_row, (int)gridDim.x));
        if (tid < listed) {
          const int id = next_row + tid * (int)gridDim.x;
          const RowPiece x = row_piece<KT, KT>(p, cut, id);
          list[tid] = {x.row, 1, x.kvh, id, x.key0, x.limit, x.row, 0};
        }
        next_row += listed * gridDim.x;
      }
      __syncthreads();
      if (listed == 0) break;
    }
    const GroupPiece w = list[at++];
    const int rows = w.rows * G;
    auto row_at = [&](int k) { return of_group ? p.members[w.first + k] : w.first; };
    const int* table = p.block_table + (size_t)w.table_row * p.max_pages;
    two o[4][OC][2];
    float m_run[4], l_run[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m_run[i] = -INFINITY;
      l_run[i] = 0.f;
#pragma unroll
      for (int k = 0; k < OC; ++k) o[i][k][0] = o[i][k][1] = 0;
    }
    auto look_up = [&](int kb, int which) {       // by the first KT threads
      if (tid >= KT) return;
      long long row = -1;
      if (kb + tid < w.limit) {
        const int lp = (kb + tid) / p.ps, page = table[lp];        // below max_pages: limits were checked
        if (page < 0 || page >= p.num_pages) dk_report(p.err, DK_DEV_BAD_PAGE, w.table_row, lp, page);
        else row = (((long long)page * 2 * p.KV + w.kvh) * p.ps + (kb + tid - lp * p.ps)) * hd;
      }
      s_row[which][tid] = row;
    };
    auto fetch = [&](float* to, int which, long long kind) {       // zeros where there is none
#pragma unroll 1
      for (int key = warp; key < KT; key += WARPS) {
        const long long row = s_row[which][key];
        const T* src = reinterpret_cast<const T*>(p.kv) + (row < 0 ? 0 : row + kind);
        for (int col = lane * 4; col < hd; col += 128) {
          if constexpr (sizeof(T) == 4) cp_async_16(smem_u32(to + key * ks + col), src + col, row >= 0);
          else *reinterpret_cast<float4*>(to + key * ks + col) = row >= 0 ? load4(src + col) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      cp_async_commit();
    };
    const long long values = (long long)p.KV * p.ps * hd;        // from a key's row to its value's
    int q_row[QR / WARPS];        // asked for with the first pages
#pragma unroll
    for (int i = 0; i < QR / WARPS; ++i) {
      const int qr = warp + i * WARPS;
      q_row[i] = qr < rows ? row_at(qr * inv_g >> 16) : -1;
    }
    look_up(w.key0, 0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QR / WARPS; ++i) {        // the queries, on their way with the first keys
      const int qr = warp + i * WARPS, row = q_row[i];
      const bool there = row >= 0 && row < p.rows;
      const T* src = reinterpret_cast<const T*>(p.q) + (there ? row * p.q_stride + (w.kvh * G + qr - (qr * inv_g >> 16) * G) * hd : 0);
      for (int col = lane * 4; col < hd; col += 128) {
        if constexpr (sizeof(T) == 4) cp_async_16(smem_u32(s_q + qr * ks + col), src + col, there);
        else *reinterpret_cast<float4*>(s_q + qr * ks + col) = there ? load4(src + col) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    fetch(s_k, 0, 0);
    fetch(s_v, 0, values);
    int which = 0;
    const bool busy = warp * 8 < rows;        // some of the warp's eight queries is one
#pragma unroll 1
    for (int kb = w.key0; kb < w.limit; kb += KT, which ^= 1) {
      look_up(kb + KT, which ^ 1);
      cp_async_wait<1>();
      __syncthreads();        // the keys are there
      float s[4][2];
      if (busy) {
        two t[4][2];        // even and odd places of the head apart
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i][0] = t[i][1] = 0;
#pragma unroll 8
        for (int d = 0; d < hd; d += 4) {
          ulonglong2 a[4], b[2];
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const ulonglong2*>(s_q + (q4 + i) * ks + d);
#pragma unroll
          for (int j = 0; j < 2; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(s_k + (c + j * SHARE) * ks + d);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) t[i][j] = fma2(a[i].x, b[j].x, fma2(a[i].y, b[j].y, t[i][j]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 v = unpack(t[i][j]);
            s[i][j] = v.x + v.y;
          }
      }
      __syncthreads();        // the keys are no longer read
      fetch(s_k, which ^ 1, 0);
      if (busy) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[i][j] = kb + c + j * SHARE < w.limit ? s[i][j] * sl2 : -INFINITY;
            mx = fmaxf(mx, s[i][j]);
          }
#pragma unroll
          for (int x = 1; x < SHARE; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float m_new = fmaxf(m_run[i], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
          const float keep = exp2f(m_run[i] - m_use);       // 0 before the first key
          m_run[i] = m_new;
          s[i][0] = exp2f(s[i][0] - m_use);
          s[i][1] = exp2f(s[i][1] - m_use);
          l_run[i] = l_run[i] * keep + (s[i][0] + s[i][1]);
          const two keep2 = pack(keep, keep);
#pragma unroll
          for (int k = 0; k < OC; ++k) {
            o[i][k][0] = mul2(o[i][k][0], keep2);
            o[i][k][1] = mul2(o[i][k][1], keep2);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float4*>(s_p + (c + j * SHARE) * P_STRIDE + q4) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
      }
      cp_async_wait<1>();
      __syncthreads();        // the values and the weights are there
      if (busy) {
#pragma unroll 8
        for (int key = 0; key < KT; ++key) {        // (behind the last key weights and values are zeros)
          const float4 x = *reinterpret_cast<const float4*>(s_p + key * P_STRIDE + q4);
          const two e[4] = {pack(x.x, x.x), pack(x.y, x.y), pack(x.z, x.z), pack(x.w, x.w)};
#pragma unroll
          for (int k = 0; k < OC; ++k)
            if (k * 64 + c * 4 < hd) {
              const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(s_v + key * ks + k * 64 + c * 4);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[i][k][0] = fma2(e[i], v.x, o[i][k][0]);
                o[i][k][1] = fma2(e[i], v.y, o[i][k][1]);
              }
            }
        }
      }
      __syncthreads();        // the values are no longer read
      fetch(s_v, which ^ 1, values);
    }
    cp_async_wait<0>();
    // a query's columns and a column's queries lie one step apart
    float* part = of_group ? group_results(p, w.id) : row_results(p, w.id);
    const int per_query = of_group ? 4 : hd, per_column = of_group ? QR : 1;
    float* to = part + q4 * per_query + c * 4 * per_column;
    float* ml = part + (of_group ? QR : G) * hd + (of_group ? 4 : 2) * q4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int x = 1; x < SHARE; x <<= 1) l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], x);
      if (q4 + i < rows) {
#pragma unroll
        for (int k = 0; k < OC; ++k)
          if (k * 64 + c * 4 < hd) *reinterpret_cast<ulonglong2*>(to + i * per_query + k * 64 * per_column) = make_ulonglong2(o[i][k][0], o[i][k][1]);
        if (c == 0) *reinterpret_cast<float2*>(ml + i * (of_group ? 4 : 2)) = make_float2(m_run[i], l_run[i]);
      }
    }
    __syncthreads();          // the queries may be overwritten
  }
}

// One block per (key-value head, row, eight groups of four columns): thread (head, column group, lane), heads fastest.  A lane takes every ``lanes``-th
// piece, eight at a time; the lanes' results are joined in their order.
constexpr int MERGE_COLS = 8, MERGE_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(MERGE_THREADS) attention_shared_prefix_merge_kernel(const DkSharedPrefixParams p) {
  const int kvh = blockIdx.x, row = blockIdx.y, G = p.G;
  __shared__ float4 s_o[MERGE_THREADS];
  __shared__ float2 s_ml[MERGE_THREADS];
  const int places = G * MERGE_COLS, lanes = MERGE_THREADS / places, place = threadIdx.x % places, lane = threadIdx.x / places, g = place % G,
            c4 = blockIdx.z * MERGE_COLS + place / G;
  const bool mine = c4 * 4 < p.hd && lane < lanes;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const RowPiece w = row_pieces(p)[row * p.KV + kvh];
  const long long gs = group_piece_floats(QR, p.hd), rs = row_piece_floats(G, p.hd);
  const float* gp = group_results(p, w.group_id);
  const float* rp = row_results(p, w.first_id);
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float2 ml, const float4 o) {
    const float m_new = fmaxf(M, ml.x), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float keep = exp2f(M - m_use), f = exp2f(ml.x - m_use);
    M = m_new;
    L = L * keep + ml.y * f;
    acc.x = acc.x * keep + o.x * f;
    acc.y = acc.y * keep + o.y * f;
    acc.z = acc.z * keep + o.z * f;
    acc.w = acc.w * keep + o.w * f;
  };
  if (mine) {
    constexpr int AT_ONCE = 8;        // pieces asked for together
    const int pieces = w.group_n + w.pieces;
#pragma unroll 1
    for (int i = lane; i < pieces; i += AT_ONCE * lanes) {
      float2 ml[AT_ONCE];
      float4 o[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int n = i + j * lanes;
        if (n < w.group_n) {
          ml[j] = *reinterpret_cast<const float2*>(gp + n * gs + (size_t)QR * p.hd + 4 * (w.r0 + g));
          o[j] = *reinterpret_cast<const float4*>(gp + n * gs + ((size_t)c4 * QR + w.r0 + g) * 4);
        } else if (n < pieces) {
          ml[j] = *reinterpret_cast<const float2*>(rp + (n - w.group_n) * rs + (size_t)G * p.hd + 2 * g);
          o[j] = *reinterpret_cast<const float4*>(rp + (n - w.group_n) * rs + (size_t)g * p.hd + c4 * 4);
        }
      }
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
        if (i + j * lanes < pieces) add(ml[j], o[j]);
    }
  }
  s_o[threadIdx.x] = acc;
  s_ml[threadIdx.x] = make_float2(M, L);
  __syncthreads();
  if (!mine || lane != 0) return;
  for (int k = 1; k < lanes; ++k) add(s_ml[k * places + place], s_o[k * places + place]);
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);      // no key: zeros; a NaN stays one
  T* out = reinterpret_cast<T*>(p.out) + row * p.out_stride + (kvh * G + g) * p.hd + c4 * 4;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(out) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  }
}

template <typename T, int HDM>
int launch(const DkSharedPrefixParams& p, cudaStream_t stream) {
  const size_t need = smem_floats(p.hd), tables = Cut::ints(p.rows, p.groups);
  const size_t smem = 4 * (need > tables ? need : tables);
  static size_t granted_on[DK_MAX_DEVICES] = {0};
  size_t& granted = granted_on[dk_current_device()];
  if (smem > granted) {
    cudaError_t e = cudaFuncSetAttribute(attention_shared_prefix_kernel<T, HDM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) {
      dk_set_error("attention_shared_prefix: cannot get %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
      return DK_ERR_LAUNCH;
    }
    granted = smem;
  }
  attention_shared_prefix_kernel<T, HDM><<<p.grid, THREADS, smem, stream>>>(p);
  return dk_check_launch("attention_shared_prefix");
}

template <typename T>
int launch_sized(const DkSharedPrefixParams& p, cudaStream_t stream) {
  if (p.hd <= 64) return launch<T, 64>(p, stream);
  if (p.hd <= 128) return launch<T, 128>(p, stream);
  return launch<T, 256>(p, stream);
}

int fma_grid() { return BLOCKS * dk_sm_count(); }

int merge(const DkSharedPrefixParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.KV, p.rows, cdiv(p.hd, 4 * MERGE_COLS));
  cfg.blockDim = dim3(MERGE_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // its launch overlaps the first kernel's end; it waits for its results
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = p.dtype == DK_F32 ? cudaLaunchKernelEx(&cfg, attention_shared_prefix_merge_kernel<float>, p)
                                    : cudaLaunchKernelEx(&cfg, attention_shared_prefix_merge_kernel<__nv_bfloat16>, p);
  if (e != cudaSuccess) {
    dk_set_error("attention_shared_prefix: launch of the merge failed: %s", cudaGetErrorString(e));
    return DK_ERR_LAUNCH;
  }
  return dk_check_launch("attention_shared_prefix_merge");
}
}  // namespace

namespace {
int check_sizes(DkSharedPrefixParams& p) {
  DK_REQUIRE(p.dtype == DK_F32 || p.dtype == DK_BF16, "attention_shared_prefix: unknown element type %d", p.dtype);
  DK_REQUIRE(p.rows >= 0 && p.rows <= MAX_ROWS && p.groups >= 0 && p.groups <= MAX_GROUPS && p.n_members >= 0 && p.n_members <= MAX_ROWS,
             "attention_shared_prefix: %d rows in %d groups with %d members; at most %d rows and %d groups are taken", p.rows, p.groups,
             p.n_members, MAX_ROWS, MAX_GROUPS);
  DK_REQUIRE(p.KV >= 1 && p.KV <= 128 && p.H >= p.KV && p.H % p.KV == 0 && p.H / p.KV <= MAX_G,
             "attention_shared_prefix: %d query heads and %d key-value heads; 1 to %d to each of at most 128 are taken", p.H, p.KV, MAX_G);
  DK_REQUIRE(p.hd >= 4 && p.hd <= 256 && p.hd % 4 == 0, "attention_shared_prefix: head size %d is no multiple of 4 up to 256", p.hd);
  DK_REQUIRE(p.ps >= 1 && p.max_pages >= 1 && p.num_pages >= 1 && (long long)p.max_pages * p.ps < (1ll << 30),
             "attention_shared_prefix: tables of %d pages of %d tokens", p.max_pages, p.ps);
  if (p.n_members == 0) p.groups = 0;
  return 0;
}

// How the work is cut: by the tensor cores' kernels where they take the sizes, else for the FMA units.  Returns which.
bool cut_for(DkSharedPrefixParams& p) {
  const bool tc = dk_shared_prefix_tc_takes(p);
  p.qr = tc ? 128 : QR;
  p.kt = tc ? 128 : KT;
  p.grid = tc ? dk_sm_count() - 1 : fma_grid();      // (one block of the tensor cores' first kernel prepares the second)
  p.rows_kt = tc ? dk_shared_prefix_rows_tile() : KT;
  p.rows_grid = tc ? dk_shared_prefix_rows_grid(p) : fma_grid();
  p.min_saved = 1;
  p.least_tiles = tc ? 4 : 1;
  return tc;
}

int sizes(DkSharedPrefixParams& p, bool* tc, long long* floats) {
  if (int rc = check_sizes(p)) return rc;
  *tc = cut_for(p);
  const Bounds b = bounds(p);
  DK_REQUIRE(b.tiles < (1ll << 30) && b.pieces < (1ll << 24), "attention_shared_prefix: %d rows of %d key-value heads over tables of %d pages are too much for one call",
             p.rows, p.KV, p.max_pages);
  *floats = b.work_floats;
  return 0;
}
}  // namespace

// Floats of working memory that a call with these sizes needs.
extern "C" int dk_attention_shared_prefix_floats(int rows, int groups, int n_members, int H, int KV, int hd, int ps, int max_pages, int num_pages, int dtype, long long* floats) {
  DkSharedPrefixParams p = {};
  p.rows = rows; p.groups = groups; p.n_members = n_members; p.H = H; p.KV = KV; p.hd = hd; p.ps = ps; p.max_pages = max_pages; p.num_pages = num_pages; p.dtype = dtype;
  bool tc;
  return sizes(p, &tc, floats);
}

extern "C" int dk_attention_shared_prefix(const void* q, long long q_stride, void* out, long long out_stride, const void* kv, const int* block_table, const int* kv_len,
                                          const int* members, const int* group_start, const int* group_prefix, void* work, long long work_floats, int rows, int groups,
                                          int n_members, int H, int KV, int hd, int ps, int max_pages, int num_pages, float scale, int dtype, int* err, cudaStream_t stream) {
  DkSharedPrefixParams p = {};
  p.q = q; p.out = out; p.kv = kv; p.block_table = block_table; p.kv_len = kv_len; p.members = members; p.group_start = group_start; p.group_prefix = group_prefix;
  p.work = (float*)work; p.err = err; p.q_stride = q_stride; p.out_stride = out_stride;
  p.rows = rows; p.groups = groups; p.n_members = n_members; p.H = H; p.KV = KV; p.hd = hd; p.ps = ps; p.max_pages = max_pages; p.num_pages = num_pages; p.dtype = dtype;
  p.scale = scale;
  bool tc;
  long long need;
  int rc = sizes(p, &tc, &need);
  if (rc != 0 || rows == 0) return rc;
  DK_REQUIRE(q && out && kv && block_table && kv_len && work && (p.groups == 0 || (members && group_start && group_prefix)), "attention_shared_prefix: a tensor is missing");
  {
    // a row's pieces are read and written in no order
    const long long size = dtype == DK_F32 ? 4 : 2, row = (long long)H * hd, away = ((const char*)out - (const char*)q) / size;
    const bool apart = away >= (rows - 1) * q_stride + row || -away >= (rows - 1) * out_stride + row;
    const long long in_row = q_stride > 0 ? ((away % q_stride) + q_stride) % q_stride : 0;
    DK_REQUIRE(apart || (q_stride == out_stride && in_row >= row && in_row + row <= q_stride), "attention_shared_prefix: the results would overwrite queries that are still read");
  }
  DK_REQUIRE(work_floats >= need, "attention_shared_prefix: %lld floats of working memory are given, %lld are needed", work_floats, need);
  DK_REQUIRE(scale > 0.f, "attention_shared_prefix: the scale of the scores must be positive");
  DK_REQUIRE(q_stride % 4 == 0 && out_stride % 4 == 0 && ((uintptr_t)q % 16) == 0 && ((uintptr_t)kv % 16) == 0 && ((uintptr_t)out % 16) == 0 && ((uintptr_t)work % 16) == 0,
             "attention_shared_prefix: tensors must start on 16-byte boundaries, rows on multiples of 4 entries");
  DK_REQUIRE(!tc || q_stride % 8 == 0, "attention_shared_prefix: rows of queries must lie a multiple of 8 entries apart, not %lld", q_stride);
  if (tc) {
    p.call = dk_shared_prefix_call_number();
    rc = dk_shared_prefix_tc_launch(p, stream);
    return rc != 0 ? rc : dk_shared_prefix_rows_launch(p, stream);
  }
  rc = dtype == DK_F32 ? launch_sized<float>(p, stream) : launch_sized<__nv_bfloat16>(p, stream);
  return rc != 0 ? rc : merge(p, stream);
}
