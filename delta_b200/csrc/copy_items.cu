// Copies among the items (pages, slots) of tensors, as if every item were read before any is written: new[dst_i] = old[src_i].
// An item may be read by several copies and may be the source of one and the target of another (a cache that is compacted
// moves pages in chains and cycles), so the host puts the copies in an order in which nothing is overwritten that is still to
// be read: the copy that reads an item comes before the one that writes it.  Every copy has at most one such successor, so
// the copies form trees and cycles; a cycle is opened by keeping the first overwritten item in a register.
//
// A thread owns one unit (16 bytes where sizes and addresses allow it) at one place of an item and carries it through the
// whole list: units at different places never meet, so nothing has to be synchronised however the copies depend on
// one another.  Components that do not depend on one another are dealt to lanes (blockIdx.y).  The list travels in the kernel's arguments up to
// 1,500 copies, so there is one launch and no copy from the host.
//
// Bound by the bytes it moves.  With the device full of blocks a thread reads one copy at a time (16 layers, 1,100 pages of 32 KB: 179 us = 6.4 TB/s;
// two reads ahead 192, four 208, eight 235); a few long chains leave it nearly empty, and then four reads stand in front of four writes, which the
// order allows: a reader stands before its writer or beside it.
#include "common.cuh"
#include <algorithm>
#include <new>
#include <utility>
#include <vector>

struct DkCopyTensor {
  void* base;
  long long item_stride, layer_stride;     // bytes
  int layers, item_bytes;
  int token_bytes, tokens;                 // bytes of one token in a row of tokens, tokens in a row; 0: items are copied whole
};

namespace {
constexpr int THREADS = 256;
constexpr int MAX_TENSORS = 32;
constexpr int FEW = 96, INLINE = 1500;     // copies that travel in the arguments of the two kernels
constexpr int FULL = 8;                    // blocks for an SM from which on threads need not read ahead
constexpr int SAVE = 1, TAKE = 2;          // keep the target's old unit; write the kept unit

struct Tensor {
  char* base;
  long long item_stride, layer_stride;
  int layers, units, unit, first_block, layer_blocks;
  int units_per_token, tokens;             // 0: whole items
};
template <int N>
struct Args {
  Tensor t[MAX_TENSORS];
  int n_tensors, lanes;
  const int4* list;                        // {source, target, tokens, flags}; null: in ``copies``
  const int* starts;                       // [lanes + 1]
  int4 copies[N];
  short inline_starts[N + 2];
};
static_assert(sizeof(Args<FEW>) <= 4096 && sizeof(Args<INLINE>) <= 32764, "a kernel's arguments");

template <int AHEAD, typename U>
__device__ __forceinline__ void carry(const Tensor& t, const int4* list, int begin, int end) {
  const int block = (int)blockIdx.x - t.first_block, layer = block / t.layer_blocks;
  const unsigned unit = (unsigned)(block - layer * t.layer_blocks) * blockDim.x + threadIdx.x;      // (an item may have 2^31 - 1 units, and its last block ends behind them)
  if (unit >= (unsigned)t.units) return;
  char* place = t.base + layer * t.layer_stride + (long long)unit * sizeof(U);
  const int token = t.units_per_token > 0 ? (int)(unit / (unsigned)t.units_per_token % (unsigned)t.tokens) : 0;
  U kept = U();
  for (int i = begin; i < end; i += AHEAD) {
    U v[AHEAD];
    int to[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      to[j] = -1;
      if (i + j < end) {
        const int4 c = list[i + j];
        if (c.w & SAVE) kept = *reinterpret_cast<const U*>(place + c.y * t.item_stride);
        if (token < c.z) {
          to[j] = c.y;
          if (c.w & TAKE) v[j] = kept;
          else v[j] = *reinterpret_cast<const U*>(place + c.x * t.item_stride);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (to[j] >= 0) *reinterpret_cast<U*>(place + to[j] * t.item_stride) = v[j];
  }
}

template <int N, int AHEAD>
__global__ void __launch_bounds__(THREADS) copy_items_kernel(const __grid_constant__ Args<N> a) {
  int k = 0;
  while (k + 1 < a.n_tensors && (int)blockIdx.x >= a.t[k + 1].first_block) ++k;
  const Tensor& t = a.t[k];
  const int4* list = a.list ? a.list : a.copies;
  const int begin = a.list ? a.starts[blockIdx.y] : a.inline_starts[blockIdx.y];
  const int end = a.list ? a.starts[blockIdx.y + 1] : a.inline_starts[blockIdx.y + 1];
  switch (t.unit) {
    case 16: carry<AHEAD, uint4>(t, list, begin, end); break;
    case 8: carry<AHEAD, uint2>(t, list, begin, end); break;
    case 4: carry<AHEAD, uint32_t>(t, list, begin, end); break;
    case 2: carry<AHEAD, unsigned short>(t, list, begin, end); break;
    default: carry<AHEAD, unsigned char>(t, list, begin, end); break;
  }
}

// Puts the copies in order.  list: {source, target, tokens, flags} of at most n copies, lane by lane; starts[lanes + 1].  Returns the copies
// left (a copy of an item to itself is none), or a negative code.
int order_copies(const int* src, const int* dst, const int* tokens, int n, long long n_items, int whole, int want_lanes, int4* list, int* starts, int* lanes) {
  DK_REQUIRE(n >= 0, "copy_items: a negative number of copies");
  for (int i = 0; i < n; ++i) {
    DK_REQUIRE(src[i] >= 0 && src[i] < n_items && dst[i] >= 0 && dst[i] < n_items, "copy_items: copy %d goes from item %d to item %d of %lld", i, src[i], dst[i], n_items);
    DK_REQUIRE(tokens == nullptr || (tokens[i] >= 0 && tokens[i] <= whole), "copy_items: copy %d asks for %d tokens of an item of %d", i, tokens ? tokens[i] : 0, whole);
  }
  // which copy writes an item: a table of the items, or, where there are far more items than copies, the copies sorted by their targets
  const bool direct = n_items <= 64ll * n;
  std::vector<int> by_target(direct ? (size_t)n_items : (size_t)n, -1);
  if (direct) {
    for (int i = 0; i < n; ++i) {
      DK_REQUIRE(by_target[dst[i]] < 0, "copy_items: item %d is written twice", dst[i]);
      by_target[dst[i]] = i;
    }
  } else {
    for (int i = 0; i < n; ++i) by_target[i] = i;
    std::sort(by_target.begin(), by_target.end(), [&](int a, int b) { return dst[a] < dst[b]; });
    for (int i = 1; i < n; ++i) DK_REQUIRE(dst[by_target[i]] != dst[by_target[i - 1]], "copy_items: item %d is written twice", dst[by_target[i]]);
  }
  auto writer = [&](int item) {
    if (direct) return by_target[item];
    const auto it = std::lower_bound(by_target.begin(), by_target.end(), item, [&](int a, int v) { return dst[a] < v; });
    return it == by_target.end() || dst[*it] != item ? -1 : *it;
  };
  // next[i]: the copy that writes what copy i reads
  std::vector<int> next(n, -1), readers(n, 0), root(n);
  auto find = [&](int i) {
    while (root[i] != i) i = root[i] = root[root[i]];
    return i;
  };
  for (int i = 0; i < n; ++i) root[i] = i;
  auto moot = [&](int i) { return src[i] == dst[i] || (tokens != nullptr && tokens[i] == 0); };
  for (int i = 0; i < n; ++i) {
    if (moot(i)) continue;
    const int j = writer(src[i]);
    if (j < 0 || moot(j)) continue;
    next[i] = j;
    ++readers[j];
    root[find(i)] = find(j);
  }
  std::vector<int> order, flags(n, 0);
  order.reserve(n);
  std::vector<char> done(n, 0);
  for (int i = 0; i < n; ++i)
    if (!moot(i) && readers[i] == 0) order.push_back(i);
  for (size_t k = 0; k < order.size(); ++k) {
    done[order[k]] = 1;
    const int j = next[order[k]];
    if (j >= 0 && --readers[j] == 0) order.push_back(j);
  }
  for (int i = 0; i < n; ++i) {              // what is left are cycles
    if (moot(i) || done[i]) continue;
    int last = i;
    for (int j = i; !done[j]; j = next[j]) {
      done[j] = 1;
      order.push_back(j);
      last = j;
    }
    flags[i] |= SAVE;
    flags[last] |= TAKE;
  }
  // components one after the other, dealt to lanes of about the same length
  const int left = (int)order.size();
  std::vector<int> count(n + 1, 0), first(n, -1);
  for (int i : order) ++count[find(i)];
  const int target = std::max(1, (left + std::max(1, want_lanes) - 1) / std::max(1, want_lanes));
  int at = 0, lane = 0;
  starts[0] = 0;
  for (int i : order) {
    const int c = find(i);
    if (first[c] >= 0) continue;
    if (at - starts[lane] >= target) starts[++lane] = at;
    first[c] = at;
    at += count[c];
  }
  starts[lane + 1] = at;
  *lanes = left > 0 ? lane + 1 : 0;
  for (int i : order) list[first[find(i)]++] = make_int4(src[i], dst[i], tokens ? tokens[i] : (whole > 0 ? whole : 1), flags[i]);
  return left;
}

// Tensors that share memory would be copied in two places at once, each overwriting what the other reads.
int check_apart(const DkCopyTensor* tensors, int n_tensors, long long n_items) {
  DK_REQUIRE(n_tensors >= 1, "copy_items: there is no tensor");
  if (n_tensors == 1) return 0;
  std::vector<std::pair<const char*, long long>> spans;
  spans.reserve(n_tensors);
  for (int k = 0; k < n_tensors; ++k)
    if (tensors[k].layers > 0 && tensors[k].item_bytes > 0)
      spans.push_back({(const char*)tensors[k].base, (tensors[k].layers - 1) * tensors[k].layer_stride + n_items * tensors[k].item_stride});
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    DK_REQUIRE(spans[i].first >= spans[i - 1].first + spans[i - 1].second, "copy_items: two of the tensors share memory");
  return 0;
}

// Fills a.t with up to MAX_TENSORS; returns the blocks that one lane takes, or a negative code.  ``threads``: of a block.
template <int N>
int lay_out(const DkCopyTensor* tensors, int n_tensors, Args<N>& a, int& threads) {
  n_tensors = std::min(n_tensors, MAX_TENSORS);
  int most = 1;
  for (int k = 0; k < n_tensors; ++k) {
    const DkCopyTensor& x = tensors[k];
    DK_REQUIRE((x.base != nullptr || x.item_bytes == 0) && x.layers >= 0 && x.item_bytes >= 0 && x.token_bytes >= 0 && x.tokens >= 0, "copy_items: tensor %d is missing, or its items have no size that is taken", k);
    long long bits = (long long)(uintptr_t)x.base | x.item_stride | x.layer_stride | x.item_bytes | x.token_bytes;
    int unit = 16;
    while (unit > 1 && bits % unit != 0) unit /= 2;
    Tensor& t = a.t[k];
    t.base = (char*)x.base;
    t.item_stride = x.item_stride;
    t.layer_stride = x.layer_stride;
    t.layers = x.layers;
    t.unit = unit;
    t.units = x.item_bytes / unit;
    t.units_per_token = x.token_bytes / unit;
    t.tokens = x.tokens > 0 ? x.tokens : 1;
    if (t.units > most) most = t.units;
  }
  threads = most >= THREADS ? THREADS : (most + 31) / 32 * 32;
  long long blocks = 0;
  for (int k = 0; k < n_tensors; ++k) {
    Tensor& t = a.t[k];
    t.first_block = (int)blocks;
    t.layer_blocks = (int)std::max(1ll, ((long long)t.units + threads - 1) / threads);
    blocks += (long long)t.layers * t.layer_blocks;
    DK_REQUIRE(blocks < (1ll << 31) - 1, "copy_items: items of too many bytes");
  }
  a.n_tensors = n_tensors;
  return (int)blocks;
}

// As many lanes as leave eight copies to each (a fork's one source is then read for every eighth target only: 63 targets, one and eight to a lane, 18.3 and
// 11.2 us), while there are fewer than LEVEL blocks for an SM, which is enough to level the ends.
int lanes_for(int blocks, int n) {
  constexpr int LEVEL = 64, EACH = 8;
  const long long want = blocks > 0 ? ((long long)LEVEL * dk_sm_count() + blocks - 1) / blocks : 1;
  return (int)std::max(1ll, std::min({want, (long long)(n + EACH - 1) / EACH, 65535ll}));
}

template <int N>
int launch(const Args<N>& a, int blocks, int lanes, int threads, cudaStream_t stream) {
  if (blocks == 0 || lanes <= 0) return 0;
  const dim3 grid(blocks, lanes);
  if ((long long)blocks * lanes >= (long long)FULL * dk_sm_count()) copy_items_kernel<N, 1><<<grid, threads, 0, stream>>>(a);
  else copy_items_kernel<N, 4><<<grid, threads, 0, stream>>>(a);
  return dk_check_launch("copy_items");
}

// One launch for every MAX_TENSORS tensors.
template <int N>
int launch_all(const DkCopyTensor* tensors, int n_tensors, Args<N>& a, int lanes, cudaStream_t stream) {
  for (int k = 0; k < n_tensors; k += MAX_TENSORS) {
    int threads = THREADS;
    const int blocks = lay_out(tensors + k, n_tensors - k, a, threads);
    if (blocks < 0) return blocks;
    const int rc = launch(a, blocks, lanes, threads, stream);
    if (rc != 0) return rc;
  }
  return 0;
}

template <int N>
int copy_inline(const DkCopyTensor* tensors, int n_tensors, const int* src, const int* dst, const int* tokens, int n, long long n_items, cudaStream_t stream) {
  Args<N> a = {};
  int threads = THREADS, lanes = 0;
  const int blocks = lay_out(tensors, n_tensors, a, threads);
  if (blocks < 0) return blocks;
  int s[N + 2];
  const int rc = order_copies(src, dst, tokens, n, n_items, tensors[0].tokens, lanes_for(blocks, n), a.copies, s, &lanes);
  if (rc < 0) return rc;
  for (int i = 0; i <= lanes; ++i) a.inline_starts[i] = (short)s[i];
  return launch_all(tensors, n_tensors, a, lanes, stream);
}

int copy_all(const DkCopyTensor* tensors, int n_tensors, const int* src, const int* dst, const int* tokens, int n, long long n_items, const int* list, const int* starts,
             int lanes, cudaStream_t stream) {
  if (list == nullptr) {
    DK_REQUIRE(n <= INLINE, "copy_items: %d copies need a list on the device", n);
    if (const int rc = check_apart(tensors, n_tensors, n_items)) return rc;
    return n <= FEW ? copy_inline<FEW>(tensors, n_tensors, src, dst, tokens, n, n_items, stream)
                    : copy_inline<INLINE>(tensors, n_tensors, src, dst, tokens, n, n_items, stream);
  }
  Args<1> a = {};
  a.list = reinterpret_cast<const int4*>(list);
  a.starts = starts;
  return launch_all(tensors, n_tensors, a, lanes, stream);
}

int order_all(const DkCopyTensor* tensors, int n_tensors, const int* src, const int* dst, const int* tokens, int n, long long n_items, int* list, int* starts) {
  if (const int rc = check_apart(tensors, n_tensors, n_items)) return rc;
  Args<1> a = {};
  int threads = THREADS, lanes = 0;
  const int blocks = lay_out(tensors, n_tensors, a, threads);
  if (blocks < 0) return blocks;
  const int rc = order_copies(src, dst, tokens, n, n_items, tensors[0].tokens, lanes_for(blocks, n), reinterpret_cast<int4*>(list), starts, &lanes);
  return rc < 0 ? rc : lanes;
}

// {address, bytes} of dense tensors [slots, ...] as tensors of items.
std::vector<DkCopyTensor> dense(const long long* pairs, int n, long long slots) {
  std::vector<DkCopyTensor> out(n);
  for (int k = 0; k < n; ++k) {
    const long long item = slots > 0 ? pairs[2 * k + 1] / slots : 0;
    out[k] = {(void*)pairs[2 * k], item, 0, item > 0 ? 1 : 0, item < (1ll << 31) ? (int)item : -1, 0, 0};      // (-1: refused as a negative size)
  }
  return out;
}

template <typename F>
int guarded(int n, F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    dk_set_error("copy_items: no memory on the host to order %d copies", n);
    return DK_ERR_ARG;
  }
}
}  // namespace

extern "C" int dk_sizeof_copy_tensor() { return (int)sizeof(DkCopyTensor); }
extern "C" int dk_copy_items_inline() { return INLINE; }

// Puts n copies in order for a list on the device: list [n][4] ints and starts [n + 2].  Returns the number of lanes (0: nothing to copy) or a negative code.
extern "C" int dk_copy_items_order(const DkCopyTensor* tensors, int n_tensors, const int* src, const int* dst, const int* tokens, int n, long long n_items, int* list, int* starts) {
  return guarded(n, [&] { return order_all(tensors, n_tensors, src, dst, tokens, n, n_items, list, starts); });
}

// The copies of src and dst (host) when there are at most INLINE of them, else those of a list on the device that dk_copy_items_order made.
extern "C" int dk_copy_items(const DkCopyTensor* tensors, int n_tensors, const int* src, const int* dst, const int* tokens, int n, long long n_items,
                             const int* list, const int* starts, int lanes, cudaStream_t stream) {
  return guarded(n, [&] { return copy_all(tensors, n_tensors, src, dst, tokens, n, n_items, list, starts, lanes, stream); });
}

// The same two for dense tensors [slots, ...], each given by its address and bytes.
extern "C" int dk_copy_slots_order(const long long* pairs, int n_tensors, const int* src, const int* dst, int n, long long slots, int* list, int* starts) {
  return guarded(n, [&] {
    const std::vector<DkCopyTensor> t = dense(pairs, n_tensors, slots);
    return order_all(t.data(), n_tensors, src, dst, nullptr, n, slots, list, starts);
  });
}
extern "C" int dk_copy_slots(const long long* pairs, int n_tensors, const int* src, const int* dst, int n, long long slots, const int* list, const int* starts, int lanes,
                             cudaStream_t stream) {
  return guarded(n, [&] {
    const std::vector<DkCopyTensor> t = dense(pairs, n_tensors, slots);
    return copy_all(t.data(), n_tensors, src, dst, nullptr, n, slots, list, starts, lanes, stream);
  });
}
