// Attention of the newest tokens of each sequence over a paged K/V cache for sm_100a (B200), and the weights it gives each key.
//
//   O = softmax(f(Q K^T)) V over the keys of the sequence's pages, f the scale and the soft cap; running maximum m and sum l.
//
// What bounds it: reading K and V once, 4 D bytes a key and kv head; 4 D operations for each of them and each query row, 1 to 32
// operations a byte. So:
//
//   * The query rows of a kv head (row r = query r / group, head r % group) share its K and V: up to 32 rows are one unit of work.
//   * The lengths are on the device. Every CTA, one per SM, adds up the sequences' 16-key tiles and takes an equal share of the list
//     of all (sequence, kv head, row tile, key tile); a share may begin and end inside a unit. A CTA leaves its part of a unit that it
//     does not cover alone in the workspace, and a second kernel, which waits beside the first, adds the parts up (and the keys' weights).
//   * Each warp walks key tiles of its own and keeps a queue of two or more of them in flight, 130 to 170 KB per SM: TMA boxes of 64
//     columns where a tile lies in one page, else copies of 16 bytes by cp.async, a row's neighbouring pieces by neighbouring lanes
//     (131072 keys of 8 heads at D128 in pages of 100, 64 and 16 90 us, of 7 91, of 1 101). One bulk copy for each row, for any page
//     size, took 14 cycles a row: 18 B/clk per SM, where the measured copy rate is 23. The queue goes on over the ends of units: the next
//     unit's copies start before the warps' parts of the last one are added up.
//   * The products are transposed, S^T = K Q^T and O^T = V^T P^T, by mma.sync m16n8k16: the keys (the columns of V) are the 16, 8
//     query rows the 8, so that 8 rows, one token's heads in most models, waste nothing. Which d a k index means is free as long as
//     K and Q agree, and so is which column of V a row of O^T is: a lane reads 16 bytes of shared memory at a time, and the
//     pairs of keys that a fragment of V^T wants come from two such reads by byte permutes. P's fragments are transposed by movmatrix.
//     (tcgen05 would multiply 128 rows at a time and hold P in another memory; 8 rows leave it nothing to win.)
//   * P goes into P V as the sum of two 16-bit numbers, so that its rounding is 2^-16 (fp16: 2^-22) of it in place of 2^-8 (2^-11), and
//     the output's error is its own rounding. fp16's subnormals end that for small P: in fp16 P is 2^7 times as large, which leaves an
//     error of at most 2^-32 of the row's largest weight for each key (without, 2^-25: a first key with nearly all the weight took the
//     weight of the thousands behind it, 6 % of an output made by their values). mma.sync issues once in 16 cycles per
//     scheduler here; up to 16 rows memory hides that, with 32 rows the products bound the call (96 of them for 16 keys: the tensor pipe
//     is busy 90 % of an SM's active cycles). A value that is not finite gives a result that is not finite, though an infinity may become
//     a NaN by the two products.
//   * Keys that no row sees are not read or count as zero, whatever lies there. Where some rows see a key and others do not, P's
//     zero meets its value, and a value that is not finite would make a NaN of it: such values take a path of their own.
//
// Measured (us a call, share of the measured copy rate): B1 H32/8 D128 8192 keys 14.6 (35 %; start of the kernel, the dependent reads of
// length, table and keys, and the join are 8 of them), 131072 keys 90 (91 %), 262144 168 (98 %); B32 4096 keys 90 (92 %); at D64 131072
// keys 55 (75 %), at D96 92 (67 %), at D192 131 (94 %), at D256 166 (99 %). 131072 keys of 8 heads with 16 rows 91 (90 %), 24 113 (73 %),
// 32 117 (70 %), 40 208, 64 212, 96 308, 128 426 (19 %: every 32 rows read K and V again). 300 sequences of 100 tokens, 4 rows 63 (30 %).
#include "sm100_ptx.cuh"
#include "fa2_launch.h"
#include "fa2_paged_params.h"

namespace fa2 {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A: 64-column parts of the head dim. NT: 8-row tiles of a warp. TEAM: warps that work on the same keys, each on its own rows.
template <int A, int NT, int TEAM>
struct Cfg {
  static constexpr int D = A * 64;
  static constexpr int kRows = 8 * NT * TEAM;
  static constexpr int kWarps = A == 1 ? (NT == 1 ? 14 : NT == 2 ? 12 : 8) : A == 2 ? (NT == 1 ? 10 : 8) : A == 3 ? (TEAM == 1 ? 7 : 8) : (TEAM == 1 ? 5 : 8);
  static constexpr int kTeams = kWarps / TEAM;
  static constexpr int kThreads = kWarps * 32;
  // A tile's 16 rows of K, then of V: 64 columns at a time, rows of 128 bytes whose 16-byte pieces are swizzled by the row.
  static constexpr int kPart = 2048;
  static constexpr int kVOff = A * kPart, kStageBytes = 2 * A * kPart;  // of a team
  static constexpr int kStages = A == 1 ? (NT < 4 ? 3 : 5) : A == 3 && TEAM > 1 ? 3 : 2;
  static constexpr int kQueueBytes = kTeams * kStages * kStageBytes;
  static constexpr bool kQInRegs = A * NT <= 4;          // else its fragments stay in shared memory
  static constexpr int kQBytes = kQInRegs ? 0 : TEAM * NT * A * 2 * 512;
  static constexpr int kRowFloats = D + 4;               // a row of a warp's O when the warps' parts become one, 8 rows at a time
  static constexpr int kPartOff = kQueueBytes + kQBytes, kPartBytes = kWarps * 8 * kRowFloats * 4;
  static constexpr int kBarOff = kPartOff + kPartBytes;
  static constexpr int kSmemBytes = kBarOff + kTeams * kStages * 8;
  static_assert(kSmemBytes <= 227 * 1024 - 6144, "shared memory");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  const int bytes = there ? 16 : 0;  // 0: zeroes
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// An arrival of this thread at a barrier, once its copies so far are there.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
  return w;
}
__device__ __forceinline__ void sts16(uint32_t at, uint4 w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  float2 f;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(w));
  return f;
}
// Two numbers as the sum of two 16-bit ones each.
template <bool BF16>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack2<BF16>(x, y);
  const float2 h = unpack2<BF16>(hi);
  lo = pack2<BF16>(x - h.x, y - h.y);
}
// Does a word of two 16-bit numbers hold an infinity or NaN?
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}
// exp2(m - m_tot) with m = -inf (a part that saw no key) giving 0 also when m_tot = -inf.
__device__ __forceinline__ float part_scale(float m, float m_tot) { return m == -INFINITY ? 0.f : ex2(m - m_tot); }

// The transpose of an 8 x 8 matrix of 16-bit numbers, two of a row in each lane.
__device__ __forceinline__ uint32_t transposed(uint32_t w) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}

// A unit: up to 8 NT TEAM query rows of a kv head of a sequence, and the part of its 16-key tiles that a share has.
struct Segment {
  int b, hk, rt;       // sequence, kv head, row tile
  int unit;            // within the sequence
  int length;          // keys of the sequence
  int first, tiles;    // its key tiles [first, first + tiles)
  int j0, j1;          // the share's
  int64_t start;       // list index of the unit's first tile
  int end_all, begin_all;  // keys outside [begin_all, end_all) are seen by no row
};
// Four columns of a row's end, and with the first of them the LSE (+inf for a row that saw no key) and what turns scores into weights.
template <bool BF16>
__device__ __forceinline__ void store_row(const PagedParams& p, int b, int hk, int row, int col, const float4& acc, float top, float total) {
  const int q = p.group.div(row), group = static_cast<int>(p.group.d), h = hk * group + row - q * group;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (col < p.head_dim)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.o) + b * p.os.outer + q * p.os.row + h * p.os.head + col) =
        make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
  if (col == 0) {
    p.lse[(static_cast<int64_t>(b) * p.heads + h) * p.seqlen_q + q] = total == 0.f ? INFINITY : (top + log2f(total)) * kLn2;
    if (p.stats != nullptr) __stcg(p.stats + (static_cast<int64_t>(b) * p.heads_k + hk) * p.rows + row, make_float2(top, inv));
  }
}

// TILED: pages are whole tiles, so that a tile is one TMA box for each 64 columns of K and of V. Otherwise its rows lie in two or more
// pages, and are copied 16 bytes at a time.
template <int A, int NT, int TEAM, bool BF16, bool TILED>
__global__ void __launch_bounds__((Cfg<A, NT, TEAM>::kThreads), 1) fwd_paged_kernel(const __grid_constant__ PagedParams p) {
  using C = Cfg<A, NT, TEAM>;
  constexpr int D = C::D, W = C::kWarps, R = C::kRows, kStages = C::kStages, kTeams = C::kTeams;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t s_sum[W];
  __shared__ int64_t s_before;        // tiles of the sequences before s_first
  __shared__ int s_first, s_length;   // ... and its length
  __shared__ float s_m[W][8], s_l[W][8];
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int team = warp / TEAM, mate = warp - team * TEAM;  // its first warp starts the copies
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff) + team * kStages;  // this team's
  const WaitCtl ctl{&s_abort};
  if (tid == 0) s_abort = 0;
  if (mate == 0 && lane < kStages) mbar_init(&bars[lane], TILED ? 1 : 32);
  mbar_fence_init();
  if (TILED && tid == 0) {
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
  }
  if (tid == 0) {
    s_first = 0;
    s_before = 0;
    s_length = 0;
  }
  // The warps' first waits read s_abort, and an elected lane arms barriers that other lanes have set up: nothing else orders these
  // for short batches. It stands beside the end of the grid before.
  __syncthreads();
  early_wait();
  early_trigger();

  // ---- this CTA's share of the tile list
  const int64_t most = min(static_cast<int64_t>(p.most_keys), p.table.capacity());
  const int units_per_seq = p.heads_k * p.row_tiles;
  auto length_of = [&](int b) {
    const int n = p.seqlens[b];
    if (n > most && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedTooLong));
    return cut_length(n, most);
  };
  auto list_of = [&](int length) { return static_cast<int64_t>(tiles_of(length, p.seqlen_q, p.window, kPagedTile)) * units_per_seq; };
  auto warp_scan = [&](int64_t x) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    return x;
  };
  // Sum over the threads up to this one, and over all.
  auto scan = [&](int64_t x, int64_t& all) {
    x = warp_scan(x);
    __syncthreads();
    if (lane == 31) s_sum[warp] = x;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w == warp) x += all;
      all += s_sum[w];
    }
    return x;
  };
  Segment seg;
  int64_t n_tiles, ctas, lo, hi;
  // No CTA has nothing (a unit's parts are neighbours' parts), and none has less than a few tiles where there are more.
  auto take_share = [&]() {
    ctas = max(min((n_tiles + kPagedMinShare - 1) / kPagedMinShare, static_cast<int64_t>(gridDim.x)), static_cast<int64_t>(1));
    lo = share_begin(blockIdx.x, n_tiles, ctas);
    hi = share_begin(blockIdx.x + 1, n_tiles, ctas);
  };
  // Then the sequence that tile lo belongs to: its number of tiles before reaches lo last.
  if (p.batch <= 32) {  // every warp for itself
    const int length = lane < p.batch ? length_of(lane) : 0;
    const int64_t n = lane < p.batch ? list_of(length) : 0, upto = warp_scan(n);
    n_tiles = __shfl_sync(0xffffffffu, upto, 31);
    take_share();
    const uint32_t found = __ballot_sync(0xffffffffu, upto - n <= lo && lo < upto);
    seg.b = found != 0 ? __ffs(found) - 1 : 0;
    seg.start = __shfl_sync(0xffffffffu, upto - n, seg.b);
    seg.length = __shfl_sync(0xffffffffu, length, seg.b);
  } else {
    const int length = tid < p.batch ? length_of(tid) : 0;
    int64_t n = tid < p.batch ? list_of(length) : 0, all;
    int64_t upto = scan(n, all);
    n_tiles = all;
    if (p.batch > C::kThreads) {
      int64_t more = 0, rest;
      for (int b = tid + C::kThreads; b < p.batch; b += C::kThreads) more += list_of(length_of(b));
      scan(more, rest);
      n_tiles += rest;
    }
    take_share();
    auto look = [&](int b, int seq_length) {
      if (upto - n <= lo && lo < upto) {
        s_first = b;
        s_before = upto - n;
        s_length = seq_length;
      }
    };
    look(tid, length);
    for (int b0 = C::kThreads; b0 < p.batch && all <= lo; b0 += C::kThreads) {
      const int b = b0 + tid, seq_length = b < p.batch ? length_of(b) : 0;
      const int64_t before = all;
      n = b < p.batch ? list_of(seq_length) : 0;
      upto = scan(n, all) + before;
      all += before;
      look(b, seq_length);
    }
    __syncthreads();
    seg.b = s_first;
    seg.start = s_before;
    seg.length = s_length;
  }
  if (blockIdx.x >= ctas) {  // no copy has been started
    if (tid == 0) p.shared[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  auto open_sequence = [&]() {
    seg.first = first_seen_tile(seg.length, p.seqlen_q, p.window, kPagedTile);
    seg.tiles = tiles_of(seg.length, p.seqlen_q, p.window, kPagedTile);
    seg.end_all = seg.length;
    seg.begin_all = p.window < 0 ? 0 : max(0, seg.length - p.seqlen_q - p.window);
  };
  // The part of the unit that begins at seg.start which lies in [x, hi).
  auto open_unit = [&](int64_t x) {
    seg.hk = seg.unit / p.row_tiles;
    seg.rt = seg.unit - seg.hk * p.row_tiles;
    seg.j0 = static_cast<int>(x - seg.start);
    seg.j1 = static_cast<int>(min(static_cast<int64_t>(seg.tiles), hi - seg.start));
  };
  open_sequence();
  {
    const int64_t before = lo - seg.start;
    seg.unit = static_cast<int>(before < (1ll << 31) ? static_cast<uint32_t>(before) / static_cast<uint32_t>(seg.tiles) : before / seg.tiles);
    seg.unit = min(seg.unit, units_per_seq - 1);
    seg.start += static_cast<int64_t>(seg.unit) * seg.tiles;
  }
  open_unit(lo);

  const uint32_t queue = smem_u32(smem) + team * (kStages * C::kStageBytes);
  const uint32_t q_smem = smem_u32(smem) + C::kQueueBytes + lane * 16;
  const float inv_cap = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
  const float cap_l2 = p.softcap * kLog2e;
  const int group = static_cast<int>(p.group.d);
  // Where this lane's pieces lie in 64 columns of a stage. K: pieces 2 t4 and 2 t4 + 1 of key g (of key g + 8 1024 bytes further); V:
  // piece g of keys 2 t4 and 2 t4 + 1 (of keys 2 t4 + 8 and + 9 1024 bytes further). Of the eight lanes that a shared-memory access
  // serves at once no two have the same banks: even pieces of two rows, or two pieces of four even rows.
  const uint32_t k_at[2] = {static_cast<uint32_t>(g * 128 + ((2 * t4 ^ g) << 4)), static_cast<uint32_t>(g * 128 + ((2 * t4 + 1 ^ g) << 4))};
  const uint32_t v_at[2] = {static_cast<uint32_t>(C::kVOff + 2 * t4 * 128 + ((g ^ 2 * t4) << 4)),
                            static_cast<uint32_t>(C::kVOff + (2 * t4 + 1) * 128 + ((g ^ (2 * t4 + 1)) << 4))};
  int stage = 0, phase = 0;                             // the next one to be read

  // ---- copies of 16 keys of the present segment
  auto first_key = [&](int j) { return (seg.first + j) * kPagedTile; };
  // The table's entry for a tile (TILED), or for key `lane % 16` of it. It is looked at when it is used: a
  // step later, so that nothing waits for it.
  auto look_up = [&](int j) {
    const int key = first_key(j) + (TILED ? 0 : lane & 15);
    if (j >= seg.j1 || key >= seg.end_all || (!TILED && key < seg.begin_all)) return -1;
    return p.table.pages[seg.b * p.table.stride + p.table.page_size.div(key)];
  };
  // Starts the copies of tile j into a stage that all lanes of the team have read, and returns a bit for each of its keys that some row sees.
  auto issue = [&](int j, int page, int to_stage) {
    const int key0 = first_key(j);
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.table.num_pages)) {
      const int key = key0 + (TILED ? 0 : lane & 15);
      if (key < seg.end_all && key >= (TILED ? 0 : seg.begin_all) && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedBadPage));
      page = -1;
    }
    const uint32_t at = queue + to_stage * C::kStageBytes;
    uint32_t seen;
    if constexpr (TILED) {
      seen = page < 0 ? 0u : bit_range(seg.begin_all - key0, min(seg.end_all - key0, 16));
      if (mate == 0 && elect_one()) {
        mbar_expect_tx(&bars[to_stage], page < 0 ? 0 : C::kStageBytes);
        if (page >= 0) {
          const int row = p.table.page_size.mod(key0);
#pragma unroll
          for (int i = 0; i < A; ++i) {
            tma_load_4d(smem + (at - smem_u32(smem)) + i * C::kPart, &p.tm_k, &bars[to_stage], i * 64, seg.hk, row, page);
            tma_load_4d(smem + (at - smem_u32(smem)) + C::kVOff + i * C::kPart, &p.tm_v, &bars[to_stage], i * 64, seg.hk, row, page);
          }
        }
      }
      __syncwarp();
    } else {
      seen = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
      const int row = p.table.page_size.mod(key0 + (lane & 15));
      const int64_t k_row = page < 0 ? 0 : page * p.ks.outer + row * p.ks.row;
      const int64_t v_row = page < 0 ? 0 : page * p.vs.outer + row * p.vs.row;
      if (mate == 0) {
        // Neighbouring lanes take neighbouring pieces of a row; what is not there is zero.
#pragma unroll
        for (int i = 0; i < A * 4; ++i) {
          const int r = (lane + 32 * i) / (A * 8), c = lane + 32 * i - r * (A * 8);
          const bool there = (seen >> r & 1) && c * 8 < p.head_dim;
          const uint32_t to = at + (c >> 3) * C::kPart + r * 128 + (((c ^ r) & 7) << 4);
          const int64_t k_from = __shfl_sync(0xffffffffu, k_row, r) + c * 8, v_from = __shfl_sync(0xffffffffu, v_row, r) + c * 8;
          copy16(to, static_cast<const uint16_t*>(p.k) + seg.hk * p.ks.head + (there ? k_from : 0), there);
          copy16(to + C::kVOff, static_cast<const uint16_t*>(p.v) + seg.hk * p.vs.head + (there ? v_from : 0), there);
        }
        copies_arrive(&bars[to_stage]);
      }
    }
    return seen;
  };
  uint32_t seen_of[kStages];  // of the tiles in the queue, the oldest first
  int next_page;              // of the tile behind them
  // Fills the queue with the segment's first tiles.
  auto fill = [&]() {
    int page[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) page[i] = look_up(seg.j0 + team + i * kTeams);
    next_page = look_up(seg.j0 + team + kStages * kTeams);
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      seen_of[i] = 0;
      if (seg.j0 + team + i * kTeams < seg.j1) seen_of[i] = issue(seg.j0 + team + i * kTeams, page[i], stage + i < kStages ? stage + i : stage + i - kStages);
    }
  };
  fill();

  constexpr int kSlot = R * (D + 2);  // floats of a part in the workspace

  for (bool more = true; more;) {
    const int row0 = seg.rt * R;
    const int rows = min(R, p.rows - row0);
    const int my_row0 = row0 + 8 * NT * mate, my_rows = rows - 8 * NT * mate;  // this warp's; it may have none
    // Keys [same_lo, same_hi) are seen by every row of the call.
    const int same_hi = seg.length - p.seqlen_q + 1;
    const int same_lo = p.window < 0 ? 0 : seg.length - 1 - p.window;
    // What query q sees: keys [from(q), to(q)).
    auto to = [&](int q) { return seg.length - p.seqlen_q + q + 1; };
    auto from = [&](int q) { return p.window < 0 ? 0 : to(q) - 1 - p.window; };

    // ---- Q: of row g of each 8-row tile the pieces that K has, as B fragments of k-steps 2 i and 2 i + 1
    uint4 qf[C::kQInRegs ? NT * A * 2 : 1];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (!C::kQInRegs && (n > 0 || warp >= TEAM * NT)) continue;  // in shared memory each tile is written by one warp
      const int tile = C::kQInRegs ? mate * NT + n : warp, r = row0 + 8 * tile + g, q = p.group.div(r);
      const uint16_t* base = static_cast<const uint16_t*>(p.q) + seg.b * p.qs.outer + q * p.qs.row + (seg.hk * group + r - q * group) * p.qs.head;
#pragma unroll
      for (int i = 0; i < A * 2; ++i) {
        const int e = (8 * (i >> 1) + 2 * t4 + (i & 1)) * 8;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (r < p.rows && e < p.head_dim) w = *reinterpret_cast<const uint4*>(base + e);
        if constexpr (C::kQInRegs) qf[n * (A * 2) + i] = w;
        else sts16(q_smem + (tile * (A * 2) + i) * 512, w);
      }
    }
    if constexpr (!C::kQInRegs) __syncthreads();

    // Rows of this thread: my_row0 + 8 n + 2 t4 + e.
    float m[NT][2], l[NT][2];
    float o[A * 4][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < A * 4; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
    }

    for (int j = seg.j0 + team; j < seg.j1; j += kTeams) {
      warp_wait(&bars[stage], phase, ctl, kWaitPaged + 1);
      const uint32_t at = queue + stage * C::kStageBytes;
      const uint32_t seen = seen_of[0];
      const int key0 = first_key(j);
      // ---- scores, transposed: of keys key0 + g and + 8 (s[2], s[3]) for rows 2 t4 and 2 t4 + 1 of each tile
      constexpr int kSums = NT == 1 ? 2 : NT;  // chains of products: one alone would be waited for at each step
      float s[kSums][4];
#pragma unroll
      for (int n = 0; n < kSums; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int i = 0; i < A * 2; ++i) {
        const uint4 w0 = lds16(at + k_at[i & 1] + (i >> 1) * C::kPart), w1 = lds16(at + k_at[i & 1] + (i >> 1) * C::kPart + 1024);
        const uint32_t a0[4] = {w0.x, w1.x, w0.y, w1.y}, a1[4] = {w0.z, w1.z, w0.w, w1.w};
        uint4 b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (C::kQInRegs) b[n] = qf[n * (A * 2) + i];
          else b[n] = lds16(q_smem + ((mate * NT + n) * (A * 2) + i) * 512);
        }
        // Neighbouring products have different sums.
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<BF16>(s[n], a0, b[n].x, b[n].y);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<BF16>(s[NT == 1 ? 1 : n], a1, b[n].z, b[n].w);
      }
      if constexpr (NT == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] += s[1][e];
      }
      const bool uneven = key0 + 16 > same_hi || key0 < same_lo;  // rows of the call see different keys of these
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (p.softcap > 0.f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = cap_l2 * tanhf(s[n][e] * inv_cap);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] *= p.scale_log2;
        }
      }
      if (uneven || seen != 0xffffu) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = g + 8 * (e >> 1), q = p.group.div(my_row0 + 8 * n + 2 * t4 + (e & 1));
            if (!(seen >> k & 1) || key0 + k >= to(q) || key0 + k < from(q)) s[n][e] = -INFINITY;
          }
      }
      if (p.scores != nullptr) {
        float* out = p.scores + ((static_cast<int64_t>(seg.b) * p.heads_k + seg.hk) * p.rows + my_row0 + 2 * t4) * p.score_stride + key0 + g;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (8 * n + 2 * t4 + (e & 1) < my_rows) __stcg(out + (8 * n + (e & 1)) * p.score_stride + 8 * (e >> 1), s[n][e]);
      }
      // ---- the levels that P is relative to: the row maxima, in fp16 less 7. They hold until some score exceeds the maximum by more than
      // 8 (in the log2 domain): P is then at most 2^8, in fp16 2^15, which costs neither of the two formats nor the fp32 sums any
      // precision, and O is rarely rescaled. Sums and levels go together to what adds up parts, so that the 7 cancels there.
      constexpr float kBelow = BF16 ? 0.f : 7.f;
      bool more = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) more = more || fmaxf(s[n][e], s[n][2 + e]) > m[n][e] + (8.f + kBelow);
      if (__any_sync(0xffffffffu, more)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(s[n][e], s[n][2 + e]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16)) - kBelow, m[n][e]);
            const float f = part_scale(m[n][e], x);
            m[n][e] = x;
            l[n][e] *= f;
#pragma unroll
            for (int i = 0; i < A * 4; ++i) {
              o[i][n][e] *= f;
              o[i][n][2 + e] *= f;
            }
          }
      }
      uint32_t p_hi[NT][2], p_lo[NT][2];  // B fragments: keys 2 t4, + 1 (and + 8, + 9) of row g
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float b0 = m[n][0] == -INFINITY ? 0.f : m[n][0], b1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float e0 = ex2(s[n][2 * h] - b0), e1 = ex2(s[n][2 * h + 1] - b1);
          l[n][0] += e0;
          l[n][1] += e1;
          uint32_t hi, lo;
          split2<BF16>(e0, e1, hi, lo);
          p_hi[n][h] = transposed(hi);
          p_lo[n][h] = transposed(lo);
        }
      }
      // ---- O^T += V^T P^T: row g of output tile 4 i + h is column 64 i + 8 g + 2 h, row g + 8 the one behind it
      auto value = [&](int r, int i) { return lds16(at + v_at[r & 1] + (r >> 1) * 1024 + i * C::kPart); };  // of key 2 t4 + (r & 1) + 8 (r / 2)
      bool apart = false;
      if (uneven && p.seqlen_q > 1) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < A * 4; ++i) {
          const uint4 w = value(i & 3, i >> 2);
          if (seen >> (2 * t4 + (i & 1) + 8 * (i >> 1 & 1)) & 1) odd = odd || not_finite<BF16>(w.x) || not_finite<BF16>(w.y) || not_finite<BF16>(w.z) || not_finite<BF16>(w.w);
        }
        apart = __any_sync(0xffffffffu, odd);
      }
      // Calls f(output tile, its A fragment); `keep` masks the keys 2 t4 and 2 t4 + 1, and those 8 behind, by halves of a word.
      auto values = [&](uint32_t keep0, uint32_t keep1, auto&& f) {
#pragma unroll
        for (int i = 0; i < A; ++i) {
          uint4 w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) w[r] = value(r, i);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            auto word = [&](const uint4& v) { return h == 0 ? v.x : h == 1 ? v.y : h == 2 ? v.z : v.w; };
            const uint32_t a[4] = {__byte_perm(word(w[0]), word(w[1]), 0x5410) & keep0, __byte_perm(word(w[0]), word(w[1]), 0x7632) & keep0,
                                   __byte_perm(word(w[2]), word(w[3]), 0x5410) & keep1, __byte_perm(word(w[2]), word(w[3]), 0x7632) & keep1};
            f(4 * i + h, a);
          }
        }
      };
      auto add_all = [&](int i, const uint32_t (&a)[4]) {
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<BF16>(o[i][n], a, p_hi[n][0], p_hi[n][1]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<BF16>(o[i][n], a, p_lo[n][0], p_lo[n][1]);
      };
      // What was not copied, or lies under a mask of all rows, may be anything: it counts as zero.
      auto halves = [](uint32_t bits) { return (bits & 1 ? 0xffffu : 0u) | (bits & 2 ? 0xffff0000u : 0u); };
      if (seen == 0xffffu && !apart) {
        values(0xffffffffu, 0xffffffffu, add_all);
      } else if (!apart) {
        values(halves(seen >> (2 * t4)), halves(seen >> (2 * t4 + 8)), add_all);
      } else {
        // One query at a time, with the values that it does not see at zero, into the rows of that query alone.
        for (int q = p.group.div(my_row0); q <= p.group.div(my_row0 + max(min(my_rows, 8 * NT), 1) - 1); ++q) {
          const uint32_t sees = seen & bit_range(from(q) - key0, to(q) - key0);
          values(halves(sees >> (2 * t4)), halves(sees >> (2 * t4 + 8)), [&](int i, const uint32_t (&a)[4]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<BF16>(c, a, p_hi[n][0], p_hi[n][1]);
              mma16816<BF16>(c, a, p_lo[n][0], p_lo[n][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (p.group.div(my_row0 + 8 * n + 2 * t4 + (e & 1)) == q) o[i][n][e] += c[e];
            }
          });
        }
      }
      // ---- the stage is free: the next tile's copies
#pragma unroll
      for (int i = 0; i + 1 < kStages; ++i) seen_of[i] = seen_of[i + 1];
      __syncwarp();
      if constexpr (TEAM > 1) asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TEAM * 32) : "memory");
      if (j + kStages * kTeams < seg.j1) {
        seen_of[kStages - 1] = issue(j + kStages * kTeams, next_page, stage);
        next_page = look_up(j + (kStages + 1) * kTeams);
      }
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }

    // ---- the next unit's copies start, then the warps' parts become one, 8 rows at a time
    const Segment done = seg;
    const bool whole = done.j0 == 0 && done.j1 == done.tiles;
    const int64_t next = done.start + done.j1;
    more = next < hi;
    if (more) {
      seg.start += seg.tiles;
      if (++seg.unit == units_per_seq) {
        seg.unit = 0;
        if (++seg.b >= p.batch) more = false;
        else {
          seg.length = length_of(seg.b);
          open_sequence();
        }
      }
      if (more) {
        open_unit(next);
        fill();
      }
    }
    float* const slot = p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (done.j0 == 0 ? 1 : 0)) * kSlot;
    float* const parts = reinterpret_cast<float*>(smem + C::kPartOff);  // [warp][8 rows][D + 4]
    const int teams = min(kTeams, done.j1 - done.j0);  // those that had a tile
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (8 * n >= rows) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[n][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int r = 2 * t4 + e;
        if (g == 0) {
          s_m[warp][r] = m[n][e];
          s_l[warp][r] = x;
        }
        if (team < teams && 8 * n + r < my_rows) {
          float* row = parts + (warp * 8 + r) * C::kRowFloats + 8 * g;
#pragma unroll
          for (int i = 0; i < A; ++i) {
            *reinterpret_cast<float4*>(row + i * 64) = make_float4(o[4 * i][n][e], o[4 * i][n][2 + e], o[4 * i + 1][n][e], o[4 * i + 1][n][2 + e]);
            *reinterpret_cast<float4*>(row + i * 64 + 4) = make_float4(o[4 * i + 2][n][e], o[4 * i + 2][n][2 + e], o[4 * i + 3][n][e], o[4 * i + 3][n][2 + e]);
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < TEAM * 8 * (D / 4); i += C::kThreads) {
        const int r = i / (D / 4) % 8, x = i / (D / 4) / 8, col = i % (D / 4) * 4;
        const int row = 8 * (NT * x + n) + r;  // of the unit: row r of the n-th tile of the x-th warp of each team
        if (row >= rows) continue;
        float top = -INFINITY;
        for (int w = x; w < teams * TEAM; w += TEAM) top = fmaxf(top, s_m[w][r]);
        float total = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int w = x; w < teams * TEAM; w += TEAM) {
          const float f = part_scale(s_m[w][r], top);
          const float4 v = *reinterpret_cast<const float4*>(parts + (w * 8 + r) * C::kRowFloats + col);
          total += f * s_l[w][r];
          acc.x += f * v.x;
          acc.y += f * v.y;
          acc.z += f * v.z;
          acc.w += f * v.w;
        }
        if (whole) {
          store_row<BF16>(p, done.b, done.hk, row0 + row, col, acc, top, total);
        } else {
          __stcg(reinterpret_cast<float4*>(slot + row * D + col), acc);
          if (col == 0) {
            __stcg(slot + R * D + row, top);
            __stcg(slot + R * D + R + row, total);
          }
        }
      }
      __syncthreads();
    }
    // A unit that this CTA begins is known by it to paged_tail_kernel: in how many parts it comes.
    if (p.units != nullptr && done.j0 == 0 && tid == 0)
      p.units[(static_cast<int64_t>(done.b) * p.heads_k + done.hk) * p.row_tiles + done.rt] =
          make_int2(blockIdx.x, whole ? 0 : share_owner(done.start + done.tiles - 1, n_tiles, ctas) - static_cast<int>(blockIdx.x) + 1);
    if (!more && tid == 0) {
      const int c_last = share_owner(done.start + done.tiles - 1, n_tiles, ctas);
      p.shared[blockIdx.x] = make_int4(whole || done.j0 > 0 ? 0 : c_last - static_cast<int>(blockIdx.x) + 1, done.b, done.hk, done.rt);
    }
  }
  if (s_abort) {
    // A wait ran out: copies may still be in flight, give them about a millisecond before the memory is given back.
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {
    }
  }
  __syncthreads();
  if (tid == 0) report_abort(&s_abort, p.status);
}

// ---- what is left when the parts are there: the units that several CTAs share, and the weights. A kernel of its own, which starts
// early and waits beside the attention. (With flags in memory, by which the last CTA of a unit knew itself, a call ended with two fences
// and two round trips to memory: B1 H32/8 Sk 8192 D128 17.3 us in place of 14.9.)
constexpr int kTailThreads = 128;

// Slot 2 c holds the part of a segment that began before CTA c's share, 2 c + 1 that of one that began in it: the first part.
__device__ __forceinline__ const float* part_of(const PagedParams& p, int c_first, int i, int64_t slot) {
  return p.partials + (2 * static_cast<int64_t>(c_first + i) + (i == 0 ? 1 : 0)) * slot;
}

// A row's maximum, sum and four columns, and the same with another part added.
struct RowPart {
  float top, total;
  float4 acc;
};
__device__ __forceinline__ void add_part(RowPart& a, float top, float total, const float4& v) {
  const float above = fmaxf(a.top, top), f = part_scale(a.top, above), g = part_scale(top, above);
  a.top = above;
  a.total = f * a.total + g * total;
  a.acc.x = f * a.acc.x + g * v.x;
  a.acc.y = f * a.acc.y + g * v.y;
  a.acc.z = f * a.acc.z + g * v.z;
  a.acc.w = f * a.acc.w + g * v.w;
}

// Adds up the parts of row r of a unit, in the order of the keys: a block has a row, a thread four columns of some neighbouring
// parts. (A single unit of 8192 keys at D256 comes in 128 parts.) i: a unit (by_unit), or the CTA whose share the unit begins in.
template <bool BF16>
__device__ __forceinline__ void join_parts(const PagedParams& p, int grid, int i, int r, bool by_unit, int d, int unit_rows, RowPart* s_part) {
  int c = i;
  int4 unit;  // parts, sequence, kv head, row tile
  if (by_unit) {
    const int2 parts = p.units[i];
    const int b = i / (p.heads_k * p.row_tiles), rest = i - b * (p.heads_k * p.row_tiles), hk = rest / p.row_tiles;
    c = parts.x;
    unit = make_int4(parts.y, b, hk, rest - hk * p.row_tiles);
  } else {
    unit = p.shared[c];
  }
  const int n_parts = unit.x, row = unit.w * unit_rows + r;
  if (!parts_there(c, n_parts, grid) || row >= p.rows) return;
  const int64_t slot = static_cast<int64_t>(unit_rows) * (d + 2);
  const int columns = d / 4, groups = kTailThreads / columns, group = threadIdx.x / columns, col = (threadIdx.x - group * columns) * 4;
  const int per = (n_parts + groups - 1) / groups, end = min(n_parts, (group + 1) * per);
  RowPart sum{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  if (group < groups) {
    constexpr int kBatch = 8;  // parts whose loads are in flight together
    for (int c0 = group * per; c0 < end; c0 += kBatch) {
      float4 v[kBatch];
      float pm[kBatch], pl[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (c0 + e < end) {
          const float* src = part_of(p, c, c0 + e, slot);
          v[e] = __ldcg(reinterpret_cast<const float4*>(src + r * d + col));
          pm[e] = __ldcg(src + unit_rows * d + r);
          pl[e] = __ldcg(src + unit_rows * d + unit_rows + r);
        }
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (c0 + e < end) add_part(sum, pm[e], pl[e], v[e]);
    }
    if (group > 0) s_part[threadIdx.x] = sum;
  }
  __syncthreads();
  if (group == 0) {
    for (int x = 1; x < groups && x * per < n_parts; ++x) {
      const RowPart o = s_part[threadIdx.x + x * columns];
      add_part(sum, o.top, o.total, o.acc);
    }
    store_row<BF16>(p, unit.y, unit.z, row, col, sum.acc, sum.top, sum.total);
  }
}

// mass[page][kv head][row] += sum over the query rows of exp2(score - maximum) / sum, four keys a thread; the sum is in the order of
// the rows, and the addition is atomic because sequences may share a page. The rows' maxima and sums are those of the unit where
// one CTA has it, else they come from the parts.
__device__ __forceinline__ void add_weights(const PagedParams& p, int grid, int unit, int block, int blocks, int d, int unit_rows, float2* s_stats) {
  const int b = unit / p.heads_k, hk = unit - b * p.heads_k;
  const int length = cut_length(p.seqlens[b], min(static_cast<int64_t>(p.most_keys), p.table.capacity()));
  const int lo = p.window < 0 ? 0 : max(0, length - p.seqlen_q - p.window);
  const int64_t step = 4 * static_cast<int64_t>(blocks) * kTailThreads;
  int64_t key = lo / 4 * 4 + 4 * (static_cast<int64_t>(block) * kTailThreads + threadIdx.x);
  if (key - 4 * threadIdx.x >= length) return;
  const int64_t slot = static_cast<int64_t>(unit_rows) * (d + 2);
  for (int r = threadIdx.x; r < p.rows; r += kTailThreads) {
    const int rt = r / unit_rows, in = r - rt * unit_rows;
    const int2 parts = p.units[static_cast<int64_t>(unit) * p.row_tiles + rt];
    float2 stat;
    if (!parts_there(parts.x, parts.y, grid)) {  // whole (or, of lengths that changed meanwhile, nothing that is known)
      stat = __ldcg(p.stats + static_cast<int64_t>(unit) * p.rows + r);
    } else {
      float top = -INFINITY, total = 0.f;
#pragma unroll 8
      for (int i = 0; i < parts.y; ++i) {
        const float* src = part_of(p, parts.x, i, slot) + unit_rows * d + in;
        const float m = __ldcg(src), l = __ldcg(src + unit_rows), above = fmaxf(top, m);
        total = total * part_scale(top, above) + l * part_scale(m, above);
        top = above;
      }
      stat = make_float2(top, total == 0.f ? 0.f : 1.f / total);
    }
    s_stats[r] = stat;
  }
  __syncthreads();
  const bool by_four = p.table.page_size.d % 4 == 0;
  for (; key < length; key += step) {
    const float* from = p.scores + static_cast<int64_t>(unit) * p.rows * p.score_stride + key;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int r = 0; r < p.rows; ++r) {
      const float4 s = __ldcg(reinterpret_cast<const float4*>(from + r * p.score_stride));
      const float2 stat = s_stats[r];
      auto weight = [&](float x) { return x == -INFINITY ? 0.f : ex2(x - stat.x) * stat.y; };
      sum[0] += weight(s.x), sum[1] += weight(s.y), sum[2] += weight(s.z), sum[3] += weight(s.w);
    }
    int page = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = static_cast<int>(key) + e;
      if (at < lo || at >= length) continue;
      if (page < 0 || !by_four) page = p.table.page_of(b, at);
      if (page >= 0)
        atomicAdd(p.mass + (static_cast<int64_t>(page) * p.heads_k + hk) * p.table.page_size.d + p.table.page_size.mod(at), sum[e]);
    }
  }
}

// Blocks: `joins` for the rows of the shared units, of which there are `listed` at most, then `blocks` for the weights of each
// (sequence, kv head).
template <bool BF16>
__global__ void __launch_bounds__(kTailThreads) paged_tail_kernel(const __grid_constant__ PagedParams p, int grid, int listed, int joins, int blocks, int d, int unit_rows) {
  __shared__ union {
    float2 stats[kPagedMaxRows];
    RowPart part[kTailThreads];
  } s;
  early_wait();
  early_trigger();
  const int i = blockIdx.x;
  if (i < joins) {
    join_parts<BF16>(p, grid, i % listed, i / listed, listed != grid, d, unit_rows, s.part);
  } else {
    const int unit = (i - joins) / blocks;
    add_weights(p, grid, unit, i - joins - unit * blocks, blocks, d, unit_rows, s.stats);
  }
}

template <int A, int NT, int TEAM, bool BF16, bool TILED>
cudaError_t launch_one(const PagedParams& p, int grid, cudaStream_t stream) {
  using C = Cfg<A, NT, TEAM>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(fwd_paged_kernel<A, NT, TEAM, BF16, TILED>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch_grid(true, fwd_paged_kernel<A, NT, TEAM, BF16, TILED>, dim3(grid), C::kThreads, C::kSmemBytes, stream, p);
}

template <int A, int NT, int TEAM, bool BF16>
cudaError_t pick_copies(const PagedParams& p, int grid, cudaStream_t stream) {
  return p.tiled ? launch_one<A, NT, TEAM, BF16, true>(p, grid, stream) : launch_one<A, NT, TEAM, BF16, false>(p, grid, stream);
}

template <int A, bool BF16>
cudaError_t pick_rows(const PagedParams& p, int grid, cudaStream_t stream) {
  const int rows = paged_unit_rows(p.rows);
  if (rows == 8) return pick_copies<A, 1, 1, BF16>(p, grid, stream);
  if (rows == 16) return pick_copies<A, 2, 1, BF16>(p, grid, stream);
  // A warp has registers for 32 rows of 128 columns; of more columns two warps take 16 rows each of the same keys. (Where one can, two
  // are slower: 32 rows against 131072 keys of 8 heads at D128 134 us, with one 120.)
  if constexpr (A <= 2) return pick_copies<A, 4, 1, BF16>(p, grid, stream);
  else return pick_copies<A, 2, 2, BF16>(p, grid, stream);
}

template <bool BF16>
cudaError_t pick_dim(const PagedParams& p, int grid, cudaStream_t stream) {
  if (p.head_dim <= 64) return pick_rows<1, BF16>(p, grid, stream);
  if (p.head_dim <= 128) return pick_rows<2, BF16>(p, grid, stream);
  if (p.head_dim <= 192) return pick_rows<3, BF16>(p, grid, stream);
  return pick_rows<4, BF16>(p, grid, stream);
}

}  // namespace

cudaError_t launch_fwd_paged(const PagedParams& p, int grid, int sm_count, bool bf16, cudaStream_t stream) {
  if (p.rows <= 0 || p.rows > kPagedMaxRows || p.head_dim <= 0 || p.head_dim > 256 || grid <= 0) return cudaErrorInvalidValue;
  const cudaError_t e = bf16 ? pick_dim<true>(p, grid, stream) : pick_dim<false>(p, grid, stream);
  if (e != cudaSuccess) return e;
  const int64_t units = static_cast<int64_t>(p.batch) * p.heads_k, keys = 4 * kTailThreads;
  const int d = (p.head_dim + 63) / 64 * 64, unit_rows = paged_unit_rows(p.rows);
  const int listed = paged_join_by_unit(units * p.row_tiles, grid, p.rows) ? static_cast<int>(units) * p.row_tiles : grid;
  const int joins = listed * (p.rows < unit_rows ? p.rows : unit_rows);
  // Blocks for every key that there can be, but no more than fill the GPU a few times over: lengths are known on the device only.
  const int64_t every = (static_cast<int64_t>(p.most_keys) + 3 + keys - 1) / keys, fill = (32 * static_cast<int64_t>(sm_count) + units - 1) / units;
  const int blocks = p.mass != nullptr ? static_cast<int>(every < fill ? every : fill) : 0;
  const dim3 all(static_cast<unsigned>(joins + units * blocks));
  if (bf16) return launch_grid(true, paged_tail_kernel<true>, all, kTailThreads, 0, stream, p, grid, listed, joins, blocks, d, unit_rows);
  return launch_grid(true, paged_tail_kernel<false>, all, kTailThreads, 0, stream, p, grid, listed, joins, blocks, d, unit_rows);
}

}  // namespace fa2
