// Eviction from a paged K/V cache by accumulated attention weight for sm_100a (B200).
//
// Every kv head of a sequence with more than `budget` tokens keeps its newest `recent` tokens and, of the others, the budget -
// recent with the largest weights, of equal weights the earlier ones; shorter sequences keep all. What is kept goes to other
// pages, in the order of the tokens, each head's rows to the same places.
//
// What bounds it: reading the weights once, and reading and writing the rows that are kept (8 D bytes a row of keys and values).
// Two kernels:
//
//   * The choice, a CTA per (sequence, kv head): the weights become 32-bit keys in the order of the numbers, in shared memory
//     while they fit. A radix search from the top (11, 11 and 10 bits, a histogram each) finds the key of the last one to be
//     kept and how many of the keys equal to it are; one pass in the order of the tokens then writes the list of what is kept.
//   * The move, all SMs: a row's 16-byte pieces by neighbouring threads, eight pieces in flight per thread. Sources and
//     destinations are different pages, so that the rows can move in any order and pages shared with another sequence stay as
//     they are.
#include "sm100_ptx.cuh"
#include "fa2_launch.h"
#include "fa2_paged_params.h"

namespace fa2 {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr int kHeld = 48 * 1024;   // keys that shared memory holds

// Larger numbers have larger keys; both zeroes are one, and NaN is above all.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  if (f != f) return 0xffffffffu;
  if (f == 0.f) return 0x80000000u;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Sum over the threads before this one, and over all.
__device__ __forceinline__ int block_scan(int x, int* s_warp, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int y = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) y += z;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = y;
  __syncthreads();
  int w = s_warp[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, w, d);
    if (lane >= d) w += z;
  }
  all = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return y - x + (warp > 0 ? before : 0);
}
static_assert(kSelectWarps == 32, "the scan takes one warp sum a lane");

// HELD: the table has room for no more tokens than shared memory has for keys. Otherwise a sequence whose keys fit after all still has
// them there, and those of a longer one are read again in every pass.
template <bool HELD>
__global__ void __launch_bounds__(kSelectThreads, 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_key[];
  __shared__ int s_bin[kBins];
  __shared__ int s_warp[32];
  __shared__ int s_found, s_above;
  const int tid = threadIdx.x;
  const int b = blockIdx.x / p.heads_k, hk = blockIdx.x - b * p.heads_k;
  early_wait();
  early_trigger();
  const int64_t most = min(p.from.capacity(), static_cast<int64_t>(INT32_MAX - 8 * kSelectThreads));
  const int given = p.seqlens[b];
  const int n = cut_length(given, most);
  if (tid == 0 && given > most && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedTooLong));
  int32_t* kept = p.kept + static_cast<int64_t>(blockIdx.x) * p.budget;
  const int n_kept = min(n, p.budget);
  if (hk == 0 && tid == 0) p.seqlens_out[b] = n_kept;
  for (int i = n_kept + tid; i < p.budget; i += kSelectThreads) kept[i] = -1;
  if (n <= p.budget) {
    for (int i = tid; i < n; i += kSelectThreads) kept[i] = i;
    return;
  }
  const int others = n - p.recent, wanted = p.budget - p.recent;  // wanted < others
  for (int i = tid; i < p.recent; i += kSelectThreads) kept[wanted + i] = others + i;
  if (wanted == 0) return;

  auto read = [&](int i) {
    const int page = p.from.page_of(b, i);
    if (page < 0) {
      if (p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedBadPage));
      return 0u;  // the first to go
    }
    return order_key(p.mass[(static_cast<int64_t>(page) * p.heads_k + hk) * p.from.page_size.d + p.from.page_size.mod(i)]);
  };
  const bool held = HELD || others <= kHeld;
  if (held)
    for (int i = tid; i < others; i += kSelectThreads) s_key[i] = read(i);
  auto key_at = [&](int i) { return held ? s_key[i] : read(i); };

  // ---- the key of the last one to be kept: `prefix` are its bits above `shift`, `above` counts the larger keys
  uint32_t prefix = 0;
  int above = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kBins; i += kSelectThreads) s_bin[i] = 0;
    __syncthreads();
    for (int i = tid; i < others; i += kSelectThreads) {
      const uint32_t k = key_at(i);
      if (pass == 0 || k >> (shift + bits) == prefix) atomicAdd(&s_bin[(k >> shift) & ((1u << bits) - 1)], 1);
    }
    __syncthreads();
    // Thread t has the bins 2047 - 2 t and 2046 - 2 t: from the top.
    const int hi = s_bin[kBins - 1 - 2 * tid], lo = s_bin[kBins - 2 - 2 * tid];
    int all;
    const int before = above + block_scan(hi + lo, s_warp, all);
    if (before < wanted && before + hi + lo >= wanted) {
      const bool first = before + hi >= wanted;
      s_found = first ? kBins - 1 - 2 * tid : kBins - 2 - 2 * tid;
      s_above = first ? before : before + hi;
    }
    __syncthreads();
    prefix = prefix << bits | static_cast<uint32_t>(s_found);
    above = s_above;
    __syncthreads();
  }
  const int ties = wanted - above;  // of the keys equal to `prefix` the first ones

  // ---- the list, four neighbouring tokens a thread at a time
  int done_above = 0, done_ties = 0;
  for (int i0 = 0; i0 < others; i0 += 4 * kSelectThreads) {
    const int first = i0 + 4 * tid;
    int larger = 0, equal = 0;
    uint32_t k[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      k[e] = 0;
      if (first + e < others) {
        k[e] = key_at(first + e);
        larger += k[e] > prefix;
        equal += k[e] == prefix;
      }
    }
    int all;
    const int scan = block_scan(larger | equal << 16, s_warp, all);  // at most 4096 each
    int at_above = done_above + (scan & 0xffff), at_ties = done_ties + (scan >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (first + e < others) {
        const bool is_tie = k[e] == prefix;
        if (k[e] > prefix || (is_tie && at_ties < ties)) kept[at_above + min(at_ties, ties)] = first + e;
        at_above += k[e] > prefix;
        at_ties += is_tie;
      }
    done_above += all & 0xffff;
    done_ties += all >> 16;
    if (done_above == above && done_ties >= ties) break;
  }
}

constexpr int kMoveThreads = 256, kMoveRows = 4;  // rows a thread has in flight

// PIECES: 16-byte pieces of a row where they are known, 0: any number.
template <int PIECES>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  early_wait();
  early_trigger();
  const int pieces = PIECES > 0 ? PIECES : p.head_dim / 8, per_pass = kMoveThreads / pieces;  // rows at a time
  const int row_in = threadIdx.x / pieces, piece = threadIdx.x - row_in * pieces;
  const int b = blockIdx.x / p.heads_k, hk = blockIdx.x - b * p.heads_k;
  const int n = p.seqlens_out[b];
  if (row_in >= per_pass) return;
  const int32_t* kept = p.kept + static_cast<int64_t>(blockIdx.x) * p.budget;
  const int64_t step = static_cast<int64_t>(gridDim.y) * per_pass * kMoveRows;
  for (int64_t j0 = static_cast<int64_t>(blockIdx.y) * per_pass * kMoveRows + row_in; j0 < n; j0 += step) {
    int from[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) from[u] = j0 + u * per_pass < n ? kept[j0 + u * per_pass] : -1;
    uint4 kw[kMoveRows], vw[kMoveRows];
    float mw[kMoveRows];
    int64_t to_page[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      to_page[u] = -1;
      if (from[u] < 0) continue;
      const int page = p.from.page_of(b, from[u]);
      const int to = p.to.page_of(b, static_cast<int>(j0) + u * per_pass);
      if (page < 0 || to < 0) {
        if (p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedBadPage));
        continue;
      }
      to_page[u] = to;
      const int row = p.from.page_size.mod(from[u]);
      kw[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.k) + page * p.ks.outer + row * p.ks.row + hk * p.ks.head + piece * 8);
      vw[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.v) + page * p.vs.outer + row * p.vs.row + hk * p.vs.head + piece * 8);
      if (piece == 0) mw[u] = p.mass[(static_cast<int64_t>(page) * p.heads_k + hk) * p.from.page_size.d + row];
    }
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      if (to_page[u] < 0) continue;
      const int row = p.from.page_size.mod(static_cast<int>(j0) + u * per_pass);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k) + to_page[u] * p.ks.outer + row * p.ks.row + hk * p.ks.head + piece * 8) = kw[u];
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v) + to_page[u] * p.vs.outer + row * p.vs.row + hk * p.vs.head + piece * 8) = vw[u];
      if (piece == 0) p.mass[(to_page[u] * p.heads_k + hk) * p.from.page_size.d + row] = mw[u];
    }
  }
}

}  // namespace

namespace {

template <bool HELD>
cudaError_t launch_select(const EvictParams& p, size_t smem, cudaStream_t stream) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(evict_select_kernel<HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeld * 4);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch_grid(true, evict_select_kernel<HELD>, dim3(p.batch * p.heads_k), kSelectThreads, smem, stream, p);
}

}  // namespace

cudaError_t launch_paged_evict(const EvictParams& p, int sm_count, cudaStream_t stream) {
  const int units = p.batch * p.heads_k;
  const int64_t most = p.from.capacity();
  cudaError_t e = most <= kHeld ? launch_select<true>(p, static_cast<size_t>(most) * 4, stream) : launch_select<false>(p, kHeld * 4, stream);
  if (e != cudaSuccess) return e;
  const int rows = kMoveThreads / (p.head_dim / 8) * kMoveRows;
  const int64_t blocks = (static_cast<int64_t>(p.budget) + rows - 1) / rows, fill = (64 * static_cast<int64_t>(sm_count) + units - 1) / units;
  const dim3 grid(units, static_cast<unsigned>(blocks < fill ? blocks : fill));
  if (p.head_dim == 128) return launch_grid(true, evict_move_kernel<16>, grid, kMoveThreads, 0, stream, p);
  if (p.head_dim == 64) return launch_grid(true, evict_move_kernel<8>, grid, kMoveThreads, 0, stream, p);
  return launch_grid(true, evict_move_kernel<0>, grid, kMoveThreads, 0, stream, p);
}

}  // namespace fa2
