// Kernel-side parameter blocks of the operators on a paged K/V cache.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged_index.h"

namespace fa2 {

// Codes of the status word besides WaitSite's.
enum PagedFault : int {
  kPagedBadPage = 100,   // an entry of a block table names no page of the pool, or a token lies past the table's row
  kPagedTooLong = 101,   // a length exceeds the table's row, or the bound that the caller gave
};

// Strides of a tensor in elements: {batch (or page), row, head}.
struct Strides3 {
  int64_t outer, row, head;
};

// Rotary positions: q -> q_out, k -> k_out. With `append` k_out and v_out are the pools of the cache.
struct RotaryParams {
  const void *q, *k, *v;        // null: not there
  void *q_out, *k_out, *v_out;
  Strides3 qs, ks, vs, qos, kos, vos;
  int tokens;                   // batch * seqlen
  FastDiv seqlen, heads_all, items;  // rows per batch entry; heads of q, k (and v); 16-element items of a head
  int heads, heads_k, head_dim, pairs;
  int warps_log;                // 2^warps_log warps share the heads of a token
  const void* positions;
  int64_t pos_axis, pos_batch, pos_row;
  int positions64;
  const float* inv_freq;
  int axes, in_turns, neighbours, negate;  // neighbours: a pair is two neighbouring elements
  int32_t sections[kMaxAxes];
  // append
  PageTable table;
  const int32_t* seqlens;       // tokens already in the cache
  const int32_t* cu_seqlens;    // packed: the tokens of sequence b are [cu[b], cu[b + 1])
  const int32_t* seqlens_new;   // dense: only the first of each sequence's rows are tokens
  int sequences;
  float* mass;                  // [pages, heads_k, page_size]: a new token's weights start at 0; or null
  int* status;
};

// Attention of the newest tokens over a paged cache (fwd_paged_sm100.cu).
struct PagedParams {
  CUtensorMap tm_k, tm_v;       // 4-D: (D, heads, rows of a page, pages), box (64, 1, 16, 1); used where tiled
  int tiled;                    // page_size is a multiple of 16
  const void *q, *k, *v;
  void* o;
  float* lse;                   // [batch, heads, seqlen_q]
  Strides3 qs, ks, vs, os;
  PageTable table;
  const int32_t* seqlens;
  int most_keys;                // longer sequences are cut to it
  int batch, heads, heads_k, seqlen_q, head_dim;
  FastDiv group;                // heads / heads_k
  int rows, row_tiles;          // seqlen_q * group, in tiles of paged_unit_rows
  int window;
  float scale, scale_log2, softcap;
  float* partials;              // 2 slots per CTA
  int4* shared;                 // of the unit that begins in a CTA's share and ends in another: its parts (0: there is none), sequence, kv head, row tile
  float* scores;                // [batch, heads_k, rows, score_stride] in the log2 domain, or null
  int64_t score_stride;
  float2* stats;                // [batch, heads_k, rows]: row maximum (log2 domain; fp16: less 7), 1 / row sum, where one CTA has the row's unit
  int2* units;                  // [batch, heads_k, row_tiles]: first CTA and number of its parts (0: it is whole); null where nothing asks for it
  float* mass;                  // [pages, heads_k, page_size]
  int* status;
};

// Eviction (paged_evict_sm100.cu).
struct EvictParams {
  void *k, *v;
  float* mass;
  Strides3 ks, vs;
  PageTable from, to;
  const int32_t* seqlens;
  int32_t* seqlens_out;
  int32_t* kept;                // [batch, heads_k, budget]
  int batch, heads_k, head_dim, budget, recent;
  int* status;
};

cudaError_t launch_rotary(const RotaryParams& p, bool bf16, bool append, bool vectors, cudaStream_t stream);

constexpr int kPagedMaxRows = 128;   // query rows per kv head
constexpr int kPagedTile = 16;       // keys of a tile
constexpr int kPagedMinShare = 4;    // tiles of a CTA's share at least, where there are that many
// Query rows of a unit.
inline int paged_unit_rows(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }
// Are the shared units found by looking at all units (fewer than CTAs), or at what each CTA has begun? With a block for each row the
// latter leaves most of the blocks nothing to do, which costs with many rows. us a call at D128, by units and by CTAs: 16 rows
// against 8192 keys of 8 heads 20.0 and 21.2, 32 rows 28.1 and 31.2, against 131072 116.6 and 119.4, B4 12 rows 8192 keys 34.7 and 35.2.
// Up to 8 rows it is the other way about: 4 rows against 2048 keys of 8 heads 10.8 and 10.3, 8192 17.2 and 16.7,
// 131072 91.3 and 89.9, B4 8192 keys 31.8 and 31.5, D64 12.8 and 12.4, D256 23.1 and 22.1; only 8 rows of a single head gain by units,
// 11.8 and 12.1. Why was not found out.
inline bool paged_join_by_unit(int64_t units, int grid, int rows) { return units < grid && rows > 8; }
// Floats of a partial result: O of a unit's rows, their maxima and sums.
inline int64_t paged_part_floats(int head_dim, int rows) { return paged_unit_rows(rows) * (static_cast<int64_t>((head_dim + 63) / 64 * 64) + 2); }
cudaError_t launch_fwd_paged(const PagedParams& p, int grid, int sm_count, bool bf16, cudaStream_t stream);

cudaError_t launch_paged_evict(const EvictParams& p, int sm_count, cudaStream_t stream);

}  // namespace fa2
