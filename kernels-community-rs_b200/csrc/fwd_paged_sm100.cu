// Attention of the newest tokens of each sequence over a paged K/V cache for sm_100a (B200), and the weights it gives each key.
//
//   O = softmax(f(Q K^T)) V over the keys of the sequence's pages, f the scale and the soft cap; running maximum m and sum l.
//
// What bounds it: reading K and V once (4 D bytes a key and kv head, 4 D operations for each of them and each query row: 1 to 16
// operations a byte). So:
//
//   * The query rows of a kv head (row r = query r / group, head r % group) are the M of one product, 16 at a time.
//   * The lengths are on the device. Every CTA, one per SM, adds up the sequences' key tiles and takes an equal share of the list
//     of all (sequence, kv head, key tile); a share may begin and end inside a unit. A CTA leaves its part of a unit that it does
//     not cover alone in the workspace, and whichever sees a unit's last part done adds the parts up, in the order of the keys.
//   * A thread's copies are its own. mma.sync takes B fragments whose k index may be permuted freely as long as A's is alike, and
//     n is only a name; so lane (g, t) = (lane / 4, lane % 4) takes 16-byte pieces t, t + 4, ... of key g's row as two k-steps of
//     Q K^T, and pieces g, g + 8, ... of the rows of keys 2t, 2t + 1, 2t + 8, 2t + 9 as columns of P V. Every lane therefore reads
//     from shared memory only what it copied there itself (cp.async): a queue per thread, without barriers between threads, with
//     any page size, and free of bank conflicts because a copy's 32 pieces lie side by side. Each of the 8 (4) warps of a CTA
//     walks its own keys, 16 at a time, with about 190 KB of copies in flight per SM.
//   * P goes into P V as the sum of two 16-bit numbers, so that its rounding is 2^-16 (2^-21) instead of 2^-9 (2^-12) of it, and
//     the output's error is its own rounding. The tensor cores are idle most of the time anyway.
//   * Keys that no row sees are not read: their rows are zeroes and their scores -inf. Where some rows see a key and others do
//     not, P's zero meets its value, and a value that is not finite would make a NaN of it: such values take a path of their own.
#include "sm100_ptx.cuh"
#include "fa2_launch.h"
#include "fa2_paged_params.h"

namespace fa2 {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int A>  // 64-column parts of the head dim
struct Cfg {
  static constexpr int D = A * 64;
  static constexpr int kWarps = A > 2 ? 4 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTileKeys = kWarps * 16;
  static constexpr int kPieces = 8 * A;                  // 16-byte pieces a lane copies for 16 keys: K and V
  static constexpr int kStageBytes = kPieces * 32 * 16;  // of a warp
  static constexpr int kStages = A == 1 ? 5 : A == 3 ? 4 : 3;
  static constexpr int kQueueBytes = kWarps * kStages * kStageBytes;
  static constexpr int kRowFloats = D + 4;               // a row of a warp's O when the warps' parts become one
  static_assert(kPagedRows * kRowFloats * 4 <= kStages * kStageBytes, "the parts take the place of the queue");
  static constexpr int kSmemBytes = kQueueBytes;
  static_assert(kSmemBytes <= 227 * 1024 - 4096, "shared memory");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  const int bytes = there ? 16 : 0;  // 0: zeroes
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
  return w;
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

// A unit: 16 query rows of a kv head of a sequence, and the part of its key tiles that a share has.
struct Segment {
  int b, hk, rt;       // sequence, kv head, row tile
  int length;          // keys of the sequence
  int first, tiles;    // its key tiles [first, first + tiles)
};

template <int A, bool BF16>
__global__ void __launch_bounds__(Cfg<A>::kThreads, 1) fwd_paged_kernel(const __grid_constant__ PagedParams p) {
  using C = Cfg<A>;
  constexpr int D = C::D, W = C::kWarps, kKeys = C::kTileKeys;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_sum[W];
  __shared__ int64_t s_before;        // tiles of the sequences before s_first
  __shared__ int s_first;
  __shared__ float s_m[W][kPagedRows], s_l[W][kPagedRows];
  __shared__ uint32_t s_seen[W][C::kStages];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
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
  auto tiles_in = [&](int b) { return tiles_of(length_of(b), p.seqlen_q, p.window, kKeys); };
  int64_t mine = 0;
  for (int b = tid; b < p.batch; b += C::kThreads) mine += tiles_in(b);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if (lane == 0) s_sum[warp] = mine;
  __syncthreads();
  int64_t n_tiles = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) n_tiles += s_sum[w];
  n_tiles *= units_per_seq;
  const int64_t ctas = min(n_tiles, static_cast<int64_t>(gridDim.x));  // none of them has nothing: a unit's parts are neighbours' parts
  if (blockIdx.x >= ctas) return;
  const int64_t lo = share_begin(blockIdx.x, n_tiles, ctas), hi = share_begin(blockIdx.x + 1, n_tiles, ctas);
  if (tid == 0) {
    s_first = 0;
    s_before = 0;
  }
  // the sequence that tile lo belongs to: its number of tiles before reaches lo last
  {
    int64_t carry = 0;
    for (int b0 = 0; b0 < p.batch; b0 += C::kThreads) {
      const int b = b0 + tid;
      const int64_t n = b < p.batch ? static_cast<int64_t>(tiles_in(b)) * units_per_seq : 0;
      int64_t x = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      __syncthreads();
      if (lane == 31) s_sum[warp] = x;
      __syncthreads();
      int64_t before = carry, all = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < warp) before += s_sum[w];
        all += s_sum[w];
      }
      before += x - n;
      if (before <= lo && lo < before + n) {
        s_first = b;
        s_before = before;
      }
      carry += all;
      if (carry > lo) break;
    }
    __syncthreads();
  }
  Segment seg;
  seg.b = s_first;
  int64_t seg_start;  // list index of the segment's unit
  int unit;           // within the sequence
  auto open_sequence = [&]() {
    seg.length = length_of(seg.b);
    seg.first = first_seen_tile(seg.length, p.seqlen_q, p.window, kKeys);
    seg.tiles = tiles_of(seg.length, p.seqlen_q, p.window, kKeys);
  };
  open_sequence();
  unit = static_cast<int>(min((lo - s_before) / seg.tiles, static_cast<int64_t>(units_per_seq - 1)));
  seg_start = s_before + static_cast<int64_t>(unit) * seg.tiles;

  const uint32_t queue = smem_u32(smem) + warp * (C::kStages * C::kStageBytes) + lane * 16;
  const float inv_cap = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
  const float cap_l2 = p.softcap * kLog2e;

  for (int64_t x = lo; x < hi;) {
    seg.hk = unit / p.row_tiles;
    seg.rt = unit - seg.hk * p.row_tiles;
    const int j0 = static_cast<int>(x - seg_start);
    const int j1 = static_cast<int>(min(static_cast<int64_t>(seg.tiles), hi - seg_start));
    // Rows of this thread: query and head.
    const int r0 = seg.rt * 16 + g, r1 = r0 + 8;
    const int q0 = p.group.div(r0), q1 = p.group.div(r1);
    const int group = static_cast<int>(p.group.d);
    const int rows = min(kPagedRows, p.rows - seg.rt * 16);
    const int end_all = seg.length;                          // keys from here on are seen by no row
    const int begin_all = p.window < 0 ? 0 : max(0, static_cast<int>(max(static_cast<int64_t>(seg.length) - p.seqlen_q - p.window, static_cast<int64_t>(0))));
    // What each row sees: [lo, hi).
    const int hi0 = seg.length - p.seqlen_q + q0 + 1, hi1 = seg.length - p.seqlen_q + q1 + 1;
    const int lo0 = p.window < 0 ? 0 : hi0 - 1 - p.window, lo1 = p.window < 0 ? 0 : hi1 - 1 - p.window;
    // Keys [same_lo, same_hi) are seen by every row of the call.
    const int same_hi = seg.length - p.seqlen_q + 1;
    const int same_lo = p.window < 0 ? 0 : seg.length - 1 - p.window;

    // ---- Q: pieces t4 + 4 i of rows g and g + 8 as A fragments of k-steps 2 i and 2 i + 1
    uint32_t qf[A * 4][4];
    {
      const uint16_t* base = static_cast<const uint16_t*>(p.q) + seg.b * p.qs.outer + (seg.hk * group) * p.qs.head;
      const uint16_t* a0 = base + q0 * p.qs.row + (r0 - q0 * group) * p.qs.head;
      const uint16_t* a1 = base + q1 * p.qs.row + (r1 - q1 * group) * p.qs.head;
#pragma unroll
      for (int i = 0; i < A * 2; ++i) {
        const int e = (t4 + 4 * i) * 8;
        uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
        if (r0 < p.rows && e < p.head_dim) w0 = *reinterpret_cast<const uint4*>(a0 + e);
        if (r1 < p.rows && e < p.head_dim) w1 = *reinterpret_cast<const uint4*>(a1 + e);
        qf[2 * i][0] = w0.x, qf[2 * i][1] = w1.x, qf[2 * i][2] = w0.y, qf[2 * i][3] = w1.y;
        qf[2 * i + 1][0] = w0.z, qf[2 * i + 1][1] = w1.z, qf[2 * i + 1][2] = w0.w, qf[2 * i + 1][3] = w1.w;
      }
    }

    // ---- copies of 16 keys
    const uint16_t* k_head = static_cast<const uint16_t*>(p.k) + seg.hk * p.ks.head;
    const uint16_t* v_head = static_cast<const uint16_t*>(p.v) + seg.hk * p.vs.head;
    auto first_key = [&](int j) { return (seg.first + j) * kKeys + warp * 16; };
    // The page of key `lane % 16` of the warp's 16, looked up one step ahead of its copies.
    auto look_up = [&](int j) {
      const int key = first_key(j) + (lane & 15);
      if (j >= j1 || key >= end_all || key < begin_all) return -1;
      const int page = p.table.page_of(seg.b, key);
      if (page < 0 && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedBadPage));
      return page;
    };
    int next_page = look_up(j0);
    auto issue = [&](int j, int stage) {
      const int page = next_page;
      const uint32_t seen = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
      if (lane == 0) s_seen[warp][stage] = seen;
      if (j < j1) {
        const int row = p.table.page_size.mod(first_key(j) + (lane & 15));
        const int64_t k_row = page < 0 ? 0 : page * p.ks.outer + row * p.ks.row;
        const int64_t v_row = page < 0 ? 0 : page * p.vs.outer + row * p.vs.row;
        const uint32_t at = queue + stage * C::kStageBytes;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int key = g + 8 * half;
          const uint16_t* src = k_head + __shfl_sync(0xffffffffu, k_row, key) + t4 * 8;
          const bool there = seen >> key & 1;
#pragma unroll
          for (int i = 0; i < A * 2; ++i) {
            const bool in = there && (t4 + 4 * i) * 8 < p.head_dim;
            copy16(at + (half * (A * 2) + i) * 512, in ? src + i * 32 : k_head, in);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = 2 * t4 + (r & 1) + 8 * (r >> 1);
          const uint16_t* src = v_head + __shfl_sync(0xffffffffu, v_row, key) + g * 8;
          const bool there = seen >> key & 1;
#pragma unroll
          for (int i = 0; i < A; ++i) {
            const bool in = there && (g + 8 * i) * 8 < p.head_dim;
            copy16(at + (A * 4 + r * A + i) * 512, in ? src + i * 64 : v_head, in);
          }
        }
        next_page = look_up(j + 1);
      }
      copies_commit();
    };

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[A * 8][4];
#pragma unroll
    for (int i = 0; i < A * 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    int stage_in = 0, stage_out = 0;
#pragma unroll
    for (int s = 0; s < C::kStages - 1; ++s) {
      issue(j0 + s, stage_in);
      ++stage_in;
    }
    for (int j = j0; j < j1; ++j) {
      issue(j + C::kStages - 1, stage_in);
      if (++stage_in == C::kStages) stage_in = 0;
      copies_wait<C::kStages - 1>();
      __syncwarp();  // the words of seen keys are another lane's
      const uint32_t at = queue + stage_out * C::kStageBytes;
      const uint32_t seen = s_seen[warp][stage_out];
      if (++stage_out == C::kStages) stage_out = 0;
      const int key0 = first_key(j);
      if (key0 >= end_all) continue;  // past the end of the sequence
      // ---- scores of keys key0 + 2 t4, + 1 (s[0]) and + 8, + 9 (s[1])
      float s[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < A * 2; ++i) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint4 w = lds16(at + (half * (A * 2) + i) * 512);
          mma16816<BF16>(s[half], qf[2 * i], w.x, w.y);
          mma16816<BF16>(s[half], qf[2 * i + 1], w.z, w.w);
        }
      }
      if (p.softcap > 0.f) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = cap_l2 * tanhf(s[i][e] * inv_cap);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] *= p.scale_log2;
      }
      const bool uneven = key0 + 16 > same_hi || key0 < same_lo;  // rows of the call see different keys of these
      if (uneven || seen != 0xffffu) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = 2 * t4 + (e & 1) + 8 * i, key = key0 + n;
            if (!(seen >> n & 1) || key >= ((e & 2) ? hi1 : hi0) || key < ((e & 2) ? lo1 : lo0)) s[i][e] = -INFINITY;
          }
      }
      if (p.scores != nullptr) {
        float* to = p.scores + ((static_cast<int64_t>(seg.b) * p.heads_k + seg.hk) * p.rows + r0) * p.score_stride + key0 + 2 * t4;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (r0 < p.rows) __stcg(reinterpret_cast<float2*>(to + 8 * i), make_float2(s[i][0], s[i][1]));
          if (r1 < p.rows) __stcg(reinterpret_cast<float2*>(to + 8 * p.score_stride + 8 * i), make_float2(s[i][2], s[i][3]));
        }
      }
      // ---- row maxima over the four lanes of a row, rescale
      float x0 = fmaxf(max3(s[0][0], s[0][1], s[1][0]), s[1][1]);
      float x1 = fmaxf(max3(s[0][2], s[0][3], s[1][2]), s[1][3]);
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
      }
      const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
        const float a0 = part_scale(m0, n0), a1 = part_scale(m1, n1);
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int i = 0; i < A * 8; ++i) {
          o[i][0] *= a0;
          o[i][1] *= a0;
          o[i][2] *= a1;
          o[i][3] *= a1;
        }
        m0 = n0;
        m1 = n1;
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t hi_p[4], lo_p[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float e0 = ex2(s[i][0] - b0), e1 = ex2(s[i][1] - b0), e2 = ex2(s[i][2] - b1), e3 = ex2(s[i][3] - b1);
        l0 += e0 + e1;
        l1 += e2 + e3;
        split2<BF16>(e0, e1, hi_p[2 * i], lo_p[2 * i]);
        split2<BF16>(e2, e3, hi_p[2 * i + 1], lo_p[2 * i + 1]);
      }
      // ---- O += P V: output tile 8 i + j holds columns 64 i + 8 n + j for n = 0..7
      bool apart = false;
      if (uneven && p.seqlen_q > 1) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < A * 4; ++i) {
          const uint4 w = lds16(at + (A * 4 + i) * 512);
          odd = odd || not_finite<BF16>(w.x) || not_finite<BF16>(w.y) || not_finite<BF16>(w.z) || not_finite<BF16>(w.w);
        }
        apart = __any_sync(0xffffffffu, odd);
      }
      auto columns = [&](int i, const uint4 (&w)[4], int jj, uint32_t& c0, uint32_t& c1) {
        const uint32_t pick = jj & 1 ? 0x7632u : 0x5410u;
        auto word = [&](const uint4& v) { return jj < 2 ? v.x : jj < 4 ? v.y : jj < 6 ? v.z : v.w; };
        c0 = __byte_perm(word(w[0]), word(w[1]), pick);
        c1 = __byte_perm(word(w[2]), word(w[3]), pick);
      };
      if (!apart) {
#pragma unroll
        for (int i = 0; i < A; ++i) {
          uint4 w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) w[r] = lds16(at + (A * 4 + r * A + i) * 512);
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) {
            uint32_t c0, c1;
            columns(i, w, jj, c0, c1);
            mma16816<BF16>(o[8 * i + jj], hi_p, c0, c1);
            mma16816<BF16>(o[8 * i + jj], lo_p, c0, c1);
          }
        }
      } else {
        // One query at a time, with the values that it does not see at zero, into the rows of that query alone.
        for (int q = p.group.div(seg.rt * 16); q <= p.group.div(seg.rt * 16 + rows - 1); ++q) {
          const int to = seg.length - p.seqlen_q + q + 1, from = p.window < 0 ? 0 : to - 1 - p.window;
          uint32_t keep[2];  // of the keys 2 t4 and 2 t4 + 1, and of those 8 behind, by halves of a word
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = key0 + 2 * t4 + 8 * h;
            keep[h] = (key >= from && key < to ? 0xffffu : 0u) | (key + 1 >= from && key + 1 < to ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int i = 0; i < A; ++i) {
            uint4 w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = lds16(at + (A * 4 + r * A + i) * 512);
#pragma unroll
            for (int jj = 0; jj < 8; ++jj) {
              uint32_t c0, c1;
              columns(i, w, jj, c0, c1);
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<BF16>(c, hi_p, c0 & keep[0], c1 & keep[1]);
              mma16816<BF16>(c, lo_p, c0 & keep[0], c1 & keep[1]);
              if (q0 == q) o[8 * i + jj][0] += c[0], o[8 * i + jj][1] += c[1];
              if (q1 == q) o[8 * i + jj][2] += c[2], o[8 * i + jj][3] += c[3];
            }
          }
        }
      }
    }
    copies_wait<0>();

    // ---- the warps' parts become one
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (t4 == 0) {
      s_m[warp][g] = m0;
      s_m[warp][g + 8] = m1;
      s_l[warp][g] = l0;
      s_l[warp][g + 8] = l1;
    }
    float* const parts = reinterpret_cast<float*>(smem);  // [warp][row][D + 4]; a warp's is inside its own queue
    constexpr int kWarpFloats = C::kStages * C::kStageBytes / 4;
    {
      float* row0 = parts + warp * kWarpFloats + g * C::kRowFloats + 16 * t4;
      float* row1 = row0 + 8 * C::kRowFloats;
#pragma unroll
      for (int i = 0; i < A; ++i)
#pragma unroll
        for (int h = 0; h < 4; ++h) {  // four columns: n = 2 t4 + h / 2, j = 4 (h % 2) ...
          const int jj = 8 * i + 4 * (h & 1), e = h >> 1;
          if (g < rows) *reinterpret_cast<float4*>(row0 + i * 64 + h * 4) = make_float4(o[jj][e], o[jj + 1][e], o[jj + 2][e], o[jj + 3][e]);
          if (g + 8 < rows) *reinterpret_cast<float4*>(row1 + i * 64 + h * 4) = make_float4(o[jj][2 + e], o[jj + 1][2 + e], o[jj + 2][2 + e], o[jj + 3][2 + e]);
        }
    }
    __syncthreads();
    const bool whole = j0 == 0 && j1 == seg.tiles;
    constexpr int kPart = kPagedRows * (D + 2);
    float* part = p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (j0 == 0 ? 1 : 0)) * kPart;
    auto store_out = [&](int r, int col, float4 v) {
      if (col >= p.head_dim) return;
      const int row = seg.rt * 16 + r, q = p.group.div(row), h = seg.hk * group + row - q * group;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.o) + seg.b * p.os.outer + q * p.os.row + h * p.os.head + col) =
          make_uint2(pack2<BF16>(v.x, v.y), pack2<BF16>(v.z, v.w));
    };
    // A row's end: LSE (+inf for a row that saw no key), and what turns scores into weights.
    auto store_stats = [&](int r, float m, float l) {
      const int row = seg.rt * 16 + r, q = p.group.div(row), h = seg.hk * group + row - q * group;
      p.lse[(static_cast<int64_t>(seg.b) * p.heads + h) * p.seqlen_q + q] = l == 0.f ? INFINITY : (m + log2f(l)) * kLn2;
      if (p.stats != nullptr)
        __stcg(p.stats + (static_cast<int64_t>(seg.b) * p.heads_k + seg.hk) * p.rows + row, make_float2(m, l == 0.f ? 0.f : 1.f / l));
    };
    for (int i = tid; i < rows * (D / 4); i += C::kThreads) {
      const int r = i / (D / 4), col = i % (D / 4) * 4;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, s_m[w][r]);
      float l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = part_scale(s_m[w][r], m);
        const float4 v = *reinterpret_cast<const float4*>(parts + w * kWarpFloats + r * C::kRowFloats + col);
        l += f * s_l[w][r];
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store_out(r, col, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        if (col == 0) store_stats(r, m, l);
      } else {
        __stcg(reinterpret_cast<float4*>(part + r * D + col), acc);
        if (col == 0) {
          __stcg(part + kPagedRows * D + r, m);
          __stcg(part + kPagedRows * D + kPagedRows + r, l);
        }
      }
    }
    __syncthreads();  // the parts are in memory; the queue is free again
    if (!whole) {
      // CTAs whose shares touch this unit: the owners of its first and its last tile. Slot 2 c holds a segment that began before
      // CTA c's share, 2 c + 1 one that began in it.
      const int c_first = share_owner(seg_start, n_tiles, ctas);
      const int c_last = share_owner(seg_start + seg.tiles - 1, n_tiles, ctas);
      auto slot_of = [&](int c) { return 2 * c + (c == c_first ? 1 : 0); };
      if (warp == 0) {
        // One flag per part, set to the launch's number once the part is in memory: a flag left over from another launch, or
        // from other use of the memory, is not set. Whoever sees all of a unit's flags set merges: the last to set one does
        // (store, fence, load); two may, and then both write the same bits.
        volatile unsigned long long* flags = p.flags;
        if (lane == 0) {
          asm volatile("fence.acq_rel.gpu;" ::: "memory");
          flags[slot_of(blockIdx.x)] = p.launch_tag;
        }
        __syncwarp();
        asm volatile("fence.sc.gpu;" ::: "memory");
        bool all = true;
        for (int c = c_first + lane; c <= c_last; c += 32) all = all && flags[slot_of(c)] == p.launch_tag;
        all = __all_sync(0xffffffffu, all);
        asm volatile("fence.acq_rel.gpu;" ::: "memory");
        if (all) {
          // A replayed graph launches with the same number: it has to find the flags clear.
          for (int c = c_first + lane; c <= c_last; c += 32) flags[slot_of(c)] = 0;
        }
        if (lane == 0) s_last = all ? 1 : 0;
      }
      __syncthreads();
      if (s_last) {
        const int n_parts = c_last - c_first + 1;
        for (int i = tid; i < rows * (D / 4); i += C::kThreads) {
          const int r = i / (D / 4), col = i % (D / 4) * 4;
          float m = -INFINITY, l = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          constexpr int kBatch = 8;
          for (int c0 = 0; c0 < n_parts; c0 += kBatch) {
            float4 v[kBatch];
            float pm[kBatch], pl[kBatch];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
              pm[e] = -INFINITY;
              if (c0 + e < n_parts) {
                const float* from = p.partials + static_cast<int64_t>(slot_of(c_first + c0 + e)) * kPart;
                v[e] = __ldcg(reinterpret_cast<const float4*>(from + r * D + col));
                pm[e] = __ldcg(from + kPagedRows * D + r);
                pl[e] = __ldcg(from + kPagedRows * D + kPagedRows + r);
              }
            }
            float top = m;
#pragma unroll
            for (int e = 0; e < kBatch; ++e) top = fmaxf(top, pm[e]);
            const float f = part_scale(m, top);
            l *= f;
            acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
            m = top;
#pragma unroll
            for (int e = 0; e < kBatch; ++e)
              if (c0 + e < n_parts) {
                const float f = part_scale(pm[e], m);
                l += f * pl[e];
                acc.x += f * v[e].x;
                acc.y += f * v[e].y;
                acc.z += f * v[e].z;
                acc.w += f * v[e].w;
              }
          }
          const float inv = l == 0.f ? 0.f : 1.f / l;
          store_out(r, col, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
          if (col == 0) store_stats(r, m, l);
        }
      }
    }
    // ---- the next unit
    x = seg_start + j1;
    if (j1 == seg.tiles) {
      seg_start += seg.tiles;
      if (++unit == units_per_seq) {
        unit = 0;
        if (++seg.b >= p.batch) break;
        if (x < hi) open_sequence();
      }
    }
  }
}

// mass[page][kv head][row] += sum over the query rows of exp2(score - maximum) / sum. One thread a key; the sum is in the order of
// the rows, and the addition is atomic because sequences may share a page.
template <int kMassThreads>
__global__ void __launch_bounds__(kMassThreads) paged_mass_kernel(const __grid_constant__ PagedParams p) {
  __shared__ float2 s_stats[kPagedMaxRows];
  early_wait();
  early_trigger();
  const int unit = blockIdx.x, b = unit / p.heads_k, hk = unit - b * p.heads_k;
  const int length = cut_length(p.seqlens[b], min(static_cast<int64_t>(p.most_keys), p.table.capacity()));
  const int64_t lo = p.window < 0 ? 0 : max(static_cast<int64_t>(length) - p.seqlen_q - p.window, static_cast<int64_t>(0));
  const int64_t step = static_cast<int64_t>(gridDim.y) * kMassThreads;
  if (lo / 16 * 16 + blockIdx.y * kMassThreads >= length) return;
  for (int r = threadIdx.x; r < p.rows; r += kMassThreads) s_stats[r] = __ldcg(p.stats + static_cast<int64_t>(unit) * p.rows + r);
  __syncthreads();
  for (int64_t key = lo / 16 * 16 + blockIdx.y * kMassThreads + threadIdx.x; key < length; key += step) {
    if (key < lo) continue;
    const float* from = p.scores + static_cast<int64_t>(unit) * p.rows * p.score_stride + key;
    float sum = 0.f;
    for (int r = 0; r < p.rows; ++r) {
      const float s = __ldcg(from + r * p.score_stride);
      if (s != -INFINITY) sum += ex2(s - s_stats[r].x) * s_stats[r].y;
    }
    const int page = p.table.page_of(b, static_cast<int>(key));
    if (page >= 0)
      atomicAdd(p.mass + (static_cast<int64_t>(page) * p.heads_k + hk) * p.table.page_size.d + p.table.page_size.mod(static_cast<int>(key)), sum);
  }
}

template <int A, bool BF16>
cudaError_t launch_one(const PagedParams& p, int grid, cudaStream_t stream) {
  using C = Cfg<A>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(fwd_paged_kernel<A, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch_grid(true, fwd_paged_kernel<A, BF16>, dim3(grid), C::kThreads, C::kSmemBytes, stream, p);
}

template <bool BF16>
cudaError_t pick_dim(const PagedParams& p, int grid, cudaStream_t stream) {
  if (p.head_dim <= 64) return launch_one<1, BF16>(p, grid, stream);
  if (p.head_dim <= 128) return launch_one<2, BF16>(p, grid, stream);
  if (p.head_dim <= 192) return launch_one<3, BF16>(p, grid, stream);
  return launch_one<4, BF16>(p, grid, stream);
}

}  // namespace

cudaError_t launch_fwd_paged(const PagedParams& p, int grid, bool bf16, cudaStream_t stream) {
  if (p.rows <= 0 || p.rows > kPagedMaxRows || p.head_dim <= 0 || p.head_dim > 256 || grid <= 0) return cudaErrorInvalidValue;
  return bf16 ? pick_dim<true>(p, grid, stream) : pick_dim<false>(p, grid, stream);
}

cudaError_t launch_paged_mass(const PagedParams& p, int sm_count, cudaStream_t stream) {
  constexpr int kMassThreads = 256;
  const int units = p.batch * p.heads_k;
  const int64_t blocks = (static_cast<int64_t>(p.most_keys) + 15 + kMassThreads - 1) / kMassThreads;
  // Blocks for every key that there can be, but no more than fill the GPU a few times over: lengths are known on the device only.
  const int64_t most = (16 * static_cast<int64_t>(sm_count) + units - 1) / units;
  const int y = static_cast<int>(blocks < most ? blocks : most);
  return launch_grid(true, paged_mass_kernel<kMassThreads>, dim3(units, y), kMassThreads, 0, stream, p);
}

}  // namespace fa2
