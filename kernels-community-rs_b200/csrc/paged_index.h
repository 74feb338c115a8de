// Index arithmetic of the operators on a paged K/V cache, shared by the kernels and the host: which page and row hold a token,
// how the attention's key tiles are divided over the CTAs, which axis turns a pair.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FA2_BOTH __host__ __device__ __forceinline__
#else
#define FA2_BOTH inline
#endif

namespace fa2 {

// Division of 0 <= n < 2^31 by a fixed d >= 1. With 2^(l-1) < d <= 2^l and m = ceil(2^(31+l) / d), that is m d = 2^(31+l) + e with
// e < d: n m / 2^(31+l) = n / d + n e / (d 2^(31+l)), and what is too much is below 2^-l <= 1 / d, so the floor is the same.
struct FastDiv {
  uint32_t d = 1, mul = 0, shift = 0;
  FA2_BOTH int div(int n) const {
    if (d == 1) return n;
#ifdef __CUDA_ARCH__
    return static_cast<int>(__umulhi(static_cast<uint32_t>(n), mul) >> shift);
#else
    return static_cast<int>(((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> 32) >> shift);
#endif
  }
  FA2_BOTH int mod(int n) const { return n - div(n) * static_cast<int>(d); }
};
inline FastDiv make_div(int d) {
  FastDiv f;
  f.d = static_cast<uint32_t>(d);
  if (d > 1) {
    int l = 0;
    while ((1ll << l) < d) ++l;
    f.mul = static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d);
    f.shift = static_cast<uint32_t>(l - 1);
  }
  return f;
}

// A pool of pages, and the pages of each sequence in order. Nothing on the device is trusted: a page outside the pool is not
// touched, and neither is a row past the pages that a sequence's row of the table has room for.
struct PageTable {
  const int32_t* pages;   // [batch, max_pages]
  int64_t stride;         // elements between the rows of the table
  int max_pages, num_pages;
  FastDiv page_size;
  FA2_BOTH int64_t capacity() const { return static_cast<int64_t>(max_pages) * page_size.d; }
  // The page that holds token `slot` of sequence b, or -1.
  FA2_BOTH int page_of(int b, int slot) const {
    if (slot < 0 || slot >= capacity()) return -1;
    const int page = pages[b * stride + page_size.div(slot)];
    return static_cast<uint32_t>(page) < static_cast<uint32_t>(num_pages) ? page : -1;
  }
};

// A length from the device, cut to what there can be.
FA2_BOTH int cut_length(int length, int64_t most) {
  return length < 0 ? 0 : length > most ? static_cast<int>(most) : length;
}

// The keys that some row of a call sees: the rows are the last seqlen_q tokens of `length`, and with a window >= 0 a row at place
// r sees the keys from r - window on. First key, a multiple of `tile`.
FA2_BOTH int first_seen_tile(int length, int seqlen_q, int window, int tile) {
  if (window < 0) return 0;
  const int64_t lo = static_cast<int64_t>(length) - seqlen_q - window;
  return lo > 0 ? static_cast<int>(lo / tile) : 0;
}
// Tiles of a sequence; one without keys has one, whose rows are written as empty.
FA2_BOTH int tiles_of(int length, int seqlen_q, int window, int tile) {
  const int end = static_cast<int>((static_cast<int64_t>(length) + tile - 1) / tile);
  const int n = end - first_seen_tile(length, seqlen_q, window, tile);
  return n > 0 ? n : 1;
}
// CTA c of `grid` has the tiles [share_begin(c), share_begin(c + 1)) of the list; share_owner gives the CTA of a tile. Lists of
// usual lengths get by with 32-bit divisions.
FA2_BOTH bool share_is_small(int64_t tiles, int64_t grid) { return tiles < (1 << 24) && grid < 255; }
FA2_BOTH int64_t share_begin(int64_t c, int64_t tiles, int64_t grid) {
  if (share_is_small(tiles, grid)) return static_cast<uint32_t>(c) * static_cast<uint32_t>(tiles) / static_cast<uint32_t>(grid);
  return c * tiles / grid;
}
FA2_BOTH int share_owner(int64_t tile, int64_t tiles, int64_t grid) {
  if (share_is_small(tiles, grid))
    return static_cast<int>((static_cast<uint32_t>(tile + 1) * static_cast<uint32_t>(grid) + static_cast<uint32_t>(tiles) - 1) / static_cast<uint32_t>(tiles) - 1);
  return static_cast<int>(((tile + 1) * grid + tiles - 1) / tiles - 1);
}

// Are the parts of CTAs [first, first + n) parts of a call with `grid` CTAs? What the attention has left in the workspace says so of
// every unit, unless the lengths were written to while it ran.
FA2_BOTH bool parts_there(int first, int n, int grid) { return first >= 0 && n > 0 && n <= grid - first; }

// Where a kept token goes in an eviction's list: `larger` keys and `ties` equal ones lie before it, of which the first `most_ties`
// are kept. -1: nowhere, which only weights that are written to while the eviction reads them can make of a token that is kept.
FA2_BOTH int list_place(int larger, int ties, int most_ties, int wanted) {
  const int at = larger + (ties < most_ties ? ties : most_ties);
  return at < wanted ? at : -1;
}

// Which axis turns pair i. In sections: the first sections[0] pairs belong to axis 0, and so on. In turns: of `axes` neighbours
// each axis has one, until its section is used up; what is left belongs to axis 0.
constexpr int kMaxAxes = 4;
FA2_BOTH int axis_of_pair(int i, int axes, const int32_t* sections, bool in_turns) {
  if (in_turns) {
    const int a = i % axes;
    return i < axes * sections[a] ? a : 0;
  }
  int a = 0;
  for (int end = sections[0]; a + 1 < axes && i >= end; end += sections[a]) ++a;
  return a;
}

}  // namespace fa2
