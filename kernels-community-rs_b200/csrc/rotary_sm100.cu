// Rotary positions with several axes for sm_100a (B200), alone and with the append of new tokens to a paged cache.
//
//   y0 = x0 cos a - x1 sin a,  y1 = x1 cos a + x0 sin a,   a = position[axis(pair)] * inv_freq[pair]
//
// for the pairs (x0, x1) of a head's first elements; the others are copied. The gradient is the turn by -a.
//
// What bounds it: 4 bytes of memory traffic an element. The angles of a token serve all of its heads: a warp starts the loads of
// its first heads, works out the cosines and sines of its token meanwhile, one sincos a pair, and then streams the heads
// through. (A table of cosines and sines in memory would add 8 bytes a pair and a lookup.)
//
// Angles: a position of 2^20 times a frequency of 1 in 32 bits is off by 0.03 to 0.06 rad. The frequency goes, by way of fp64,
// into turns as a fixed-point fraction of 64 bits; times the position, modulo 2^64, that is the angle's fraction of a turn, off by
// at most position * (2^-52 * frequency's turns + 2^-64), the constant and the product each rounded once (and 2^-54 * position where a
// negative frequency is brought above 0). What is left to round is that fraction to 24 bits.
#include "sm100_ptx.cuh"
#include "fa2_launch.h"
#include "fa2_paged_params.h"

namespace fa2 {

namespace {

constexpr int kThreads = 128;

// cos and sin of position * frequency.
__device__ __forceinline__ float2 turn_of(int64_t position, float frequency) {
  double t = static_cast<double>(frequency) * 0.15915494309189533577;  // 1 / (2 pi)
  t -= floor(t);
  const uint64_t u = __double2ull_rn(t * 18446744073709551616.0);
  const int64_t fraction = static_cast<int64_t>(u * static_cast<uint64_t>(position));  // [-1/2, 1/2) turns
  float s, c;
  sincospif(static_cast<float>(fraction) * 0x1p-63f, &s, &c);
  if (!isfinite(frequency)) s = c = __int_as_float(0x7fffffff);
  return make_float2(c, s);
}

__device__ __forceinline__ float2 turn_of_pair(const RotaryParams& p, int b, int s, int pair) {
  const int axis = axis_of_pair(pair, p.axes, p.sections, p.in_turns != 0);
  const int64_t at = axis * p.pos_axis + b * p.pos_batch + s * p.pos_row;
  const int64_t position = p.positions64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
  float2 cs = turn_of(position, p.inv_freq[pair]);
  if (p.negate) cs.y = -cs.y;
  return cs;
}

// Where a new token goes: element offsets of its row (head 0) in the pools, or -1 where it is not written. The weights that lie there
// are those of the row's last token: this one's start at 0, for the heads first_head, first_head + 32 and so on.
__device__ __forceinline__ longlong2 cache_row(const RotaryParams& p, int token, int b, int s, int first_head) {
  int sequence = b, i = s;
  if (p.cu_seqlens != nullptr) {
    // the last sequence that begins at or before the token
    int lo = 0, hi = p.sequences;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_seqlens[mid] <= token) lo = mid + 1;
      else hi = mid;
    }
    sequence = lo - 1;
    if (sequence < 0 || token >= p.cu_seqlens[sequence + 1]) return make_longlong2(-1, -1);
    i = token - p.cu_seqlens[sequence];
  } else if (p.seqlens_new != nullptr && s >= p.seqlens_new[b]) {
    return make_longlong2(-1, -1);
  }
  const int before = p.seqlens[sequence];
  const int64_t slot = static_cast<int64_t>(before) + i;
  const int page = before < 0 || slot >= p.table.capacity() ? -1 : p.table.page_of(sequence, static_cast<int>(slot));
  if (page < 0) {
    if (p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(kPagedBadPage));
    return make_longlong2(-1, -1);
  }
  const int row = p.table.page_size.mod(static_cast<int>(slot));
  if (p.mass != nullptr)
    for (int h = first_head; h < p.heads_k; h += 32) p.mass[(static_cast<int64_t>(page) * p.heads_k + h) * p.table.page_size.d + row] = 0.f;
  return make_longlong2(page * p.kos.outer + row * p.kos.row, page * p.vos.outer + row * p.vos.row);
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  float2 f;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(w));
  return f;
}

// One head of one token: its rows in memory, and whether it is turned.
struct Head {
  const uint16_t* in;
  uint16_t* out;   // null: not written
  bool turned;
};
template <bool APPEND>
__device__ __forceinline__ Head head_of(const RotaryParams& p, int b, int s, int h, const longlong2& row) {
  Head r;
  r.turned = true;
  if (h < p.heads) {
    r.in = static_cast<const uint16_t*>(p.q) + b * p.qs.outer + s * p.qs.row + h * p.qs.head;
    r.out = static_cast<uint16_t*>(p.q_out) + b * p.qos.outer + s * p.qos.row + h * p.qos.head;
    return r;
  }
  h -= p.heads;
  if (!APPEND || h < p.heads_k) {
    r.in = static_cast<const uint16_t*>(p.k) + b * p.ks.outer + s * p.ks.row + h * p.ks.head;
    r.out = static_cast<uint16_t*>(p.k_out);
    if constexpr (!APPEND) r.out += b * p.kos.outer + s * p.kos.row + h * p.kos.head;
    else r.out = row.x < 0 ? nullptr : r.out + row.x + h * p.kos.head;
    return r;
  }
  h -= p.heads_k;
  r.in = static_cast<const uint16_t*>(p.v) + b * p.vs.outer + s * p.vs.row + h * p.vs.head;
  r.out = row.y < 0 ? nullptr : static_cast<uint16_t*>(p.v_out) + row.y + h * p.vos.head;
  r.turned = false;
  return r;
}

// 16 bytes at a time: every row 16-byte aligned, pairs a multiple of 8. A lane has 16 elements of a head: 8 pairs, or 16 (at a head's
// end 8) elements that are copied. A warp takes a token, or with few tokens 1 / 2^warps_log of a token's heads, and goes through the
// heads with its pairs' cosines and sines in registers.
template <bool BF16, bool NEIGHBOURS, bool APPEND>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ __align__(16) float s_turn[kThreads / 32][2][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  early_wait();
  early_trigger();
  const int w = blockIdx.x * (kThreads / 32) + warp, token = w >> p.warps_log;
  if (token >= p.tokens) return;
  const int b = p.seqlen.div(token), s = token - b * static_cast<int>(p.seqlen.d);
  const int items = static_cast<int>(p.items.d), at_once = 32 / items;  // heads of a warp at a time
  const int mine = lane / items, c = lane - mine * items, chunks = p.pairs / 8, n = p.pairs;
  const bool pairs = c < chunks;
  const int e0 = pairs && !NEIGHBOURS ? 8 * c : 16 * c, e1 = pairs && !NEIGHBOURS ? n + 8 * c : 16 * c + 8;
  const int heads = static_cast<int>(p.heads_all.d), step = at_once << p.warps_log;
  int h0 = mine < at_once ? (w & ((1 << p.warps_log) - 1)) * at_once + mine : heads;

  // Heads that are loaded together; while they are turned, the loads of as many more are in flight. With 64 registers a thread, 32
  // warps to an SM, one is best: forward of B4 S8192 H32/8 D128 109 us, of B2 S4093 H16/16 25.4; two 113 and 27.7 (80 registers);
  // four at a time and none ahead 150 and 32.
  constexpr int kBatch = 1;
  uint4 w0[2][kBatch], w1[2][kBatch];
  // A head that is only copied (a value) has its elements in their order.
  auto first_of = [&](bool turned) { return turned ? e0 : 16 * c; };
  auto second_of = [&](bool turned) { return turned ? e1 : 16 * c + 8; };
  auto load = [&](int set, int h) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (h + u * step < heads) {
        const Head x = head_of<APPEND>(p, b, s, h + u * step, make_longlong2(0, 0));
        w0[set][u] = *reinterpret_cast<const uint4*>(x.in + first_of(x.turned));
        if (second_of(x.turned) < p.head_dim) w1[set][u] = *reinterpret_cast<const uint4*>(x.in + second_of(x.turned));
      }
  };
  load(0, h0);
  for (int i = lane; i < n; i += 32) {
    const float2 cs = turn_of_pair(p, b, s, i);
    s_turn[warp][0][i] = cs.x;
    s_turn[warp][1][i] = cs.y;
  }
  longlong2 row = make_longlong2(0, 0);
  if constexpr (APPEND) row = cache_row(p, token, b, s, (w & ((1 << p.warps_log) - 1)) == 0 ? lane : p.heads_k);  // one of a token's warps
  __syncwarp();
  float cs[16];  // cosines, then sines
  if (pairs) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 f = *reinterpret_cast<const float4*>(&s_turn[warp][k >> 1][8 * c + 4 * (k & 1)]);
      cs[4 * k] = f.x;
      cs[4 * k + 1] = f.y;
      cs[4 * k + 2] = f.z;
      cs[4 * k + 3] = f.w;
    }
  }
  auto turn = [&](int set, int first) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (first + u * step >= heads) break;
      const Head h = head_of<APPEND>(p, b, s, first + u * step, row);
      const uint4 x0 = w0[set][u], x1 = w1[set][u];
      uint32_t a[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
      if (h.turned && pairs) {
        if constexpr (NEIGHBOURS) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 x = unpack2<BF16>(a[j]);
            a[j] = pack2<BF16>(x.x * cs[j] - x.y * cs[8 + j], x.y * cs[j] + x.x * cs[8 + j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 x = unpack2<BF16>(a[j]), y = unpack2<BF16>(a[4 + j]);
            const float c0 = cs[2 * j], c1 = cs[2 * j + 1], s0 = cs[8 + 2 * j], s1 = cs[9 + 2 * j];
            a[j] = pack2<BF16>(x.x * c0 - y.x * s0, x.y * c1 - y.y * s1);
            a[4 + j] = pack2<BF16>(y.x * c0 + x.x * s0, y.y * c1 + x.y * s1);
          }
        }
      }
      if (APPEND && h.out == nullptr) continue;
      *reinterpret_cast<uint4*>(h.out + first_of(h.turned)) = make_uint4(a[0], a[1], a[2], a[3]);
      if (second_of(h.turned) < p.head_dim) *reinterpret_cast<uint4*>(h.out + second_of(h.turned)) = make_uint4(a[4], a[5], a[6], a[7]);
    }
  };
  for (; h0 < heads; h0 += 2 * kBatch * step) {
    load(1, h0 + kBatch * step);
    turn(0, h0);
    load(0, h0 + 2 * kBatch * step);
    turn(1, h0 + kBatch * step);
  }
}

// Any strides and any number of pairs, two bytes at a time: a block a token. A thread reads both elements of a pair before it writes
// either, so that the result may lie where the input was.
template <bool BF16, bool APPEND>
__global__ void __launch_bounds__(kThreads) rotary_any_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float2 s_turn[128];
  __shared__ longlong2 s_row;
  const int tid = threadIdx.x, n = p.pairs;
  early_wait();
  early_trigger();
  const int t = blockIdx.x, b = p.seqlen.div(t), s = t - b * static_cast<int>(p.seqlen.d);
  for (int i = tid; i < n; i += kThreads) s_turn[i] = turn_of_pair(p, b, s, i);
  if (tid < 32) {
    const longlong2 place = APPEND ? cache_row(p, t, b, s, tid) : make_longlong2(0, 0);
    if (tid == 0) s_row = place;
  }
  __syncthreads();
  const longlong2 row = s_row;
  const int heads = static_cast<int>(p.heads_all.d), items = p.head_dim - n;  // of a head: its pairs, then the elements behind them
  auto value = [](uint16_t x) { return unpack2<BF16>(x).x; };
  for (int i = tid; i < heads * items; i += kThreads) {
    const int h = i / items, item = i - h * items;
    const Head r = head_of<APPEND>(p, b, s, h, row);
    if (r.out == nullptr) continue;
    if (item >= n) {
      r.out[n + item] = r.in[n + item];
      continue;
    }
    const int e0 = p.neighbours ? 2 * item : item, e1 = p.neighbours ? 2 * item + 1 : n + item;
    uint16_t x0 = r.in[e0], x1 = r.in[e1];
    if (r.turned) {
      const float2 cs = s_turn[item];
      const float f0 = value(x0), f1 = value(x1);
      x0 = static_cast<uint16_t>(pack2<BF16>(f0 * cs.x - f1 * cs.y, 0.f));
      x1 = static_cast<uint16_t>(pack2<BF16>(f1 * cs.x + f0 * cs.y, 0.f));
    }
    r.out[e0] = x0;
    r.out[e1] = x1;
  }
}

template <bool BF16, bool APPEND>
cudaError_t pick(const RotaryParams& p, bool vectors, cudaStream_t stream) {
  if (!vectors) return launch_grid(true, rotary_any_kernel<BF16, APPEND>, dim3(p.tokens), kThreads, 0, stream, p);
  const int64_t warps = static_cast<int64_t>(p.tokens) << p.warps_log;
  const dim3 grid(static_cast<unsigned>((warps + kThreads / 32 - 1) / (kThreads / 32)));
  if (p.neighbours) return launch_grid(true, rotary_kernel<BF16, true, APPEND>, grid, kThreads, 0, stream, p);
  return launch_grid(true, rotary_kernel<BF16, false, APPEND>, grid, kThreads, 0, stream, p);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, bool bf16, bool append, bool vectors, cudaStream_t stream) {
  if (p.tokens <= 0 || p.warps_log < 0 || p.warps_log > 8 || p.pairs < 0 || p.pairs > 128) return cudaErrorInvalidValue;
  if (append) return bf16 ? pick<true, true>(p, vectors, stream) : pick<false, true>(p, vectors, stream);
  return bf16 ? pick<true, false>(p, vectors, stream) : pick<false, false>(p, vectors, stream);
}

}  // namespace fa2
