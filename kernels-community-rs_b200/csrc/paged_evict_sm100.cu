// Eviction from a paged K/V cache by accumulated attention weight for sm_100a (B200).
//
// Every kv head of a sequence with more than `budget` tokens keeps its newest `recent` tokens and, of the others, the budget -
// recent with the largest weights, of equal weights the earlier ones; shorter sequences keep all. What is kept goes to other
// pages, in the order of the tokens, each head's rows to the same places.
//
// What bounds it: reading the weights once, and reading and writing the rows that are kept (8 D bytes a row of keys and values).
// Two kernels:
//
//   * The choice, a cluster of 1 to 8 CTAs per (sequence, kv head), so that few of them use more of the GPU. The weights become
//     32-bit keys in the order of the numbers, in shared memory where they fit; else they are read again in every pass. A radix
//     search from the top (11, 11 and 10 bits, a histogram each, the CTAs' added up over distributed shared memory) finds the key
//     of the last one to be kept and how many of the keys equal to it are; one pass in the order of the tokens then writes the
//     list of what is kept. It is bound by the latency of its steps, a few thousand cycles.
//   * The move, all SMs: a row's 16-byte pieces by neighbouring threads, one of K and one of V in flight in each of 2048 threads per
//     SM. (Two or four rows a thread, and fewer threads, are slower: B16 Hk4 16384 -> 6000 87 and 92 us a call where one took
//     83, all with an earlier choice.)
//     Sources and destinations are different pages, so that the rows can move in any order and pages shared with another
//     sequence stay as they are.
#include <algorithm>

#include "sm100_ptx.cuh"
#include "fa2_launch.h"
#include "fa2_paged_params.h"

namespace fa2 {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kBins = 2048;
constexpr int kRoundKeys = 4 * kSelectThreads;        // four neighbouring keys a thread
constexpr int kHeld = 4 * kRoundKeys;                 // keys that shared memory holds

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
static_assert(kSelectThreads == 32 * 32, "the scan takes one warp sum a lane");

// Four neighbouring words of the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ int4 peer_words(const int* word, uint32_t rank) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(peer_smem(smem_u32(word), rank)) : "memory");
  return v;
}

__device__ __forceinline__ int peer_word(const int* word, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(peer_smem(smem_u32(word), rank)) : "memory");
  return v;
}

template <int CTAS>
__global__ void __launch_bounds__(kSelectThreads, 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
  __shared__ __align__(16) int s_bin[3][kBins];   // one for each pass: the other CTAs may still read the one before
  extern __shared__ __align__(16) uint4 s_key[];
  __shared__ int s_eight[CTAS > 1 ? 3 : 1][kBins / 8];
  __shared__ int s_warp[32];
  __shared__ __align__(16) int s_count[4];       // keys above and equal to the last one's
  __shared__ int s_found, s_above;
  const int tid = threadIdx.x;
  const int unit = blockIdx.x / CTAS, rank = blockIdx.x - unit * CTAS;
  const int b = unit / p.heads_k, hk = unit - b * p.heads_k;
  for (int i = tid; i < 3 * kBins; i += kSelectThreads) s_bin[0][i] = 0;
  early_wait();
  early_trigger();
  auto meet = [&]() {  // all threads of the cluster; what they wrote to shared memory is seen by all
    __syncwarp();
    if constexpr (CTAS > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
  };
  const int64_t most = min(p.from.capacity(), static_cast<int64_t>(INT32_MAX - 8 * kRoundKeys));
  const int given = p.seqlens[b];
  const int n = cut_length(given, most);
  if (tid == 0 && given > most && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedTooLong));
  int32_t* kept = p.kept + static_cast<int64_t>(unit) * p.budget;
  const int n_kept = min(n, p.budget), at = rank * kSelectThreads + tid;
  if (hk == 0 && at == 0) p.seqlens_out[b] = n_kept;
  for (int i = n_kept + at; i < p.budget; i += CTAS * kSelectThreads) kept[i] = -1;
  if (n <= p.budget) {
    for (int i = at; i < n; i += CTAS * kSelectThreads) kept[i] = i;
    return;
  }
  const int others = n - p.recent, wanted = p.budget - p.recent;  // wanted < others
  for (int i = at; i < p.recent; i += CTAS * kSelectThreads) kept[wanted + i] = others + i;
  if (wanted == 0) return;

  // ---- this CTA's tokens, and their keys
  const int slice = ((others + CTAS - 1) / CTAS + 3) / 4 * 4;
  const int begin = min(others, rank * slice), end = min(others, begin + slice);
  const bool by_four = p.from.page_size.d % 4 == 0 && reinterpret_cast<uintptr_t>(p.mass) % 16 == 0;  // four neighbours are on one page
  auto weights = [&](int page) { return p.mass + (static_cast<int64_t>(page) * p.heads_k + hk) * p.from.page_size.d; };
  auto no_page = [&]() {
    if (p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedBadPage));
  };
  // Four tokens from i on; a token of a page that cannot be is the first to go.
  auto read = [&](int i, uint32_t (&k)[4]) {
    k[0] = k[1] = k[2] = k[3] = 0;
    if (by_four) {
      const int page = p.from.page_of(b, i);
      if (page < 0) return no_page();
      const float4 w = *reinterpret_cast<const float4*>(weights(page) + p.from.page_size.mod(i));
      k[0] = order_key(w.x), k[1] = order_key(w.y), k[2] = order_key(w.z), k[3] = order_key(w.w);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < end) {
          const int page = p.from.page_of(b, i + e);
          if (page < 0) no_page();
          else k[e] = order_key(weights(page)[p.from.page_size.mod(i + e)]);
        }
    }
  };
  const bool held = slice <= kHeld;
  if (held) {
    for (int i = begin + 4 * tid; i < end; i += kRoundKeys) {
      uint32_t k[4];
      read(i, k);
      s_key[(i - begin) / 4] = make_uint4(k[0], k[1], k[2], k[3]);
    }
  }
  // Four keys of this thread's own.
  auto keys = [&](int i, uint32_t (&k)[4]) {
    if (!held) return read(i, k);
    const uint4 w = s_key[(i - begin) / 4];
    k[0] = w.x, k[1] = w.y, k[2] = w.z, k[3] = w.w;
  };

  // ---- the key of the last one to be kept: `prefix` are its bits so far, `above` counts the larger keys
  uint32_t prefix = 0;
  int above = 0;
  __syncthreads();  // the histograms are clear
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    int* bin = s_bin[pass];
#pragma unroll 1
    for (int i = begin + 4 * tid; i < end; i += kRoundKeys) {
      uint32_t k[4];
      keys(i, k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < end && (pass == 0 || k[e] >> (shift + bits) == prefix)) atomicAdd(&bin[(k[e] >> shift) & ((1u << bits) - 1)], 1);
    }
    // Threads 0 to 255 have eight bins each, from the top. The CTAs exchange the sums of eight first, and of the eight in question the bins.
    const int* eight = bin + kBins - 8 - 8 * tid;
    int mine = 0;
    __syncthreads();
    if (tid < kBins / 8) {
      const int4 v = *reinterpret_cast<const int4*>(eight), w = *reinterpret_cast<const int4*>(eight + 4);
      mine = v.x + v.y + v.z + v.w + w.x + w.y + w.z + w.w;
    }
    if constexpr (CTAS > 1) {
      if (tid < kBins / 8) s_eight[pass][tid] = mine;
      meet();
      if (tid < kBins / 8) {
        mine = 0;
#pragma unroll
        for (int r = 0; r < CTAS; ++r) mine += peer_word(&s_eight[pass][tid], r);
      }
    }
    int upto = mine;  // keys in this thread's bins and above, of those that this pass looks at
    if (tid < kBins / 8) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, upto, d);
        if ((tid & 31) >= d) upto += z;
      }
      if ((tid & 31) == 31) s_warp[tid >> 5] = upto;
    }
    __syncthreads();
    if (tid < kBins / 8) {
      upto += above - mine;
#pragma unroll
      for (int w = 0; w < kBins / 256; ++w)
        if (w < tid >> 5) upto += s_warp[w];
      if (upto < wanted && upto + mine >= wanted) {
#pragma unroll
        for (int h = 1; h >= 0; --h) {
          int4 v = make_int4(0, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < CTAS; ++r) {
            const int4 x = CTAS > 1 ? peer_words(eight + 4 * h, r) : *reinterpret_cast<const int4*>(eight + 4 * h);
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
          }
          const int count[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 3; e >= 0; --e) {
            if (upto < wanted && upto + count[e] >= wanted) {
              s_found = kBins - 8 - 8 * tid + 4 * h + e;
              s_above = upto;
            }
            upto += count[e];
          }
        }
      }
    }
    __syncthreads();
    prefix = prefix << bits | static_cast<uint32_t>(s_found);
    above = s_above;
  }
  const int ties = wanted - above;  // of the keys equal to `prefix` the first ones

  // ---- the list: the keys above and equal to it in the CTAs before this one, then in the threads before
  if (tid < 2) s_count[tid] = 0;
  __syncthreads();
  int done_above = 0, done_ties = 0;
  if constexpr (CTAS > 1) {
    int larger = 0, equal = 0;
#pragma unroll 1
    for (int i = begin + 4 * tid; i < end; i += kRoundKeys) {
      uint32_t k[4];
      keys(i, k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < end) {
          larger += k[e] > prefix;
          equal += k[e] == prefix;
        }
    }
    larger = __reduce_add_sync(0xffffffffu, larger);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if ((tid & 31) == 0) {
      atomicAdd(&s_count[0], larger);
      atomicAdd(&s_count[1], equal);
    }
    meet();
#pragma unroll
    for (int r = 0; r < CTAS; ++r) {
      const int4 v = peer_words(s_count, r);
      if (r < rank) {
        done_above += v.x;
        done_ties += v.y;
      }
    }
    __syncwarp();
    cluster_arrive();  // no CTA ends while another one reads its shared memory
  }
#pragma unroll 1
  for (int i0 = begin; i0 < end && (done_above < above || done_ties < ties); i0 += kRoundKeys) {
    const int i = i0 + 4 * tid;
    uint32_t k[4];
    int count = 0;  // larger ones in the lower half, equal ones in the upper half: at most 4096 each
    if (i < end) {
      keys(i, k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < end) count += (k[e] > prefix ? 1 : 0) + (k[e] == prefix ? 1 << 16 : 0);
    }
    int all;
    const int before = block_scan(count, s_warp, all);
    int at_above = done_above + (before & 0xffff), at_ties = done_ties + (before >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < end) {
        const bool larger = k[e] > prefix, tie = k[e] == prefix;
        const int place = list_place(at_above, at_ties, ties, wanted);
        if (place >= 0 && (larger || (tie && at_ties < ties))) kept[place] = i + e;
        at_above += larger;
        at_ties += tie;
      }
    done_above += all & 0xffff;
    done_ties += all >> 16;
  }
  if constexpr (CTAS > 1) {
    __syncwarp();
    cluster_wait();
  }
}

constexpr int kMoveThreads = 256;

// PIECES: 16-byte pieces of a row where they are known, 0: any number.
template <int PIECES>
__global__ void __launch_bounds__(kMoveThreads, 8) evict_move_kernel(const __grid_constant__ EvictParams p) {
  early_wait();
  early_trigger();
  const int pieces = PIECES > 0 ? PIECES : p.head_dim / 8, per_pass = kMoveThreads / pieces;  // rows at a time
  const int row_in = threadIdx.x / pieces, piece = threadIdx.x - row_in * pieces;
  const int b = blockIdx.x / p.heads_k, hk = blockIdx.x - b * p.heads_k;
  const int n = p.seqlens_out[b];
  if (row_in >= per_pass) return;
  const int32_t* kept = p.kept + static_cast<int64_t>(blockIdx.x) * p.budget;
  const int64_t step = static_cast<int64_t>(gridDim.y) * per_pass;
  for (int64_t j = static_cast<int64_t>(blockIdx.y) * per_pass + row_in; j < n; j += step) {
    const int from = kept[j];
    const int page = p.from.page_of(b, from), to = p.to.page_of(b, static_cast<int>(j));
    if (page < 0 || to < 0) {
      if (p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedBadPage));
      continue;
    }
    const int row = p.from.page_size.mod(from), to_row = p.from.page_size.mod(static_cast<int>(j));
    uint16_t *k = static_cast<uint16_t*>(p.k) + hk * p.ks.head + piece * 8, *v = static_cast<uint16_t*>(p.v) + hk * p.vs.head + piece * 8;
    const uint4 kw = *reinterpret_cast<const uint4*>(k + page * p.ks.outer + row * p.ks.row);
    const uint4 vw = *reinterpret_cast<const uint4*>(v + page * p.vs.outer + row * p.vs.row);
    const int64_t at = static_cast<int64_t>(page) * p.heads_k + hk, to_at = static_cast<int64_t>(to) * p.heads_k + hk;
    const float w = piece == 0 ? p.mass[at * p.from.page_size.d + row] : 0.f;
    *reinterpret_cast<uint4*>(k + to * p.ks.outer + to_row * p.ks.row) = kw;
    *reinterpret_cast<uint4*>(v + to * p.vs.outer + to_row * p.vs.row) = vw;
    if (piece == 0) p.mass[to_at * p.from.page_size.d + to_row] = w;
  }
}

}  // namespace

namespace {

template <int CTAS>
cudaError_t launch_select(const EvictParams& p, cudaStream_t stream) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(evict_select_kernel<CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeld * 4);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int64_t slice = (p.from.capacity() / CTAS + 8) / 4 * 4;  // the most that a CTA can have
  return launch_clusters(CTAS, evict_select_kernel<CTAS>, dim3(static_cast<unsigned>(p.batch * p.heads_k) * CTAS), kSelectThreads,
                         static_cast<size_t>(std::min<int64_t>(slice, kHeld)) * 4, stream, p);
}

}  // namespace

cudaError_t launch_paged_evict(const EvictParams& p, int sm_count, cudaStream_t stream) {
  const int units = p.batch * p.heads_k;
  const int64_t most = p.from.capacity();
  // Clusters where there are SMs for them and more than 8192 keys for a CTA: their barriers and the exchange take longer than that many
  // keys. us a call of B1 Hk8 from 8192 tokens with 1 CTA 12.1, with 2 13.2; from 16384 with 1 17.5, with 2 16.5; from 32768 with 1 35.8,
  // with 2 22.2, with 4 17.1; from 131072 with 1 129, with 4 51.6, with 8 24.4; of B8 Hk8 from 8192 with 1 20.7, with 2 22.3; of B16 Hk4
  // from 16384 with 1 82.3, with 2 80.7. (Four for 16384 tokens of few heads would take 14.1, for more heads there are no SMs.)
  const int64_t ctas = std::min<int64_t>((most + 8191) / 8192, sm_count / units);
  cudaError_t e = ctas >= 8 ? launch_select<8>(p, stream) : ctas >= 4 ? launch_select<4>(p, stream) : ctas >= 2 ? launch_select<2>(p, stream)
                                                                                                             : launch_select<1>(p, stream);
  if (e != cudaSuccess) return e;
  const int rows = kMoveThreads / (p.head_dim / 8);
  const int64_t blocks = (static_cast<int64_t>(p.budget) + rows - 1) / rows, fill = (64 * static_cast<int64_t>(sm_count) + units - 1) / units;
  const dim3 grid(units, static_cast<unsigned>(blocks < fill ? blocks : fill));
  if (p.head_dim == 128) return launch_grid(true, evict_move_kernel<16>, grid, kMoveThreads, 0, stream, p);
  if (p.head_dim == 64) return launch_grid(true, evict_move_kernel<8>, grid, kMoveThreads, 0, stream, p);
  return launch_grid(true, evict_move_kernel<0>, grid, kMoveThreads, 0, stream, p);
}

}  // namespace fa2
