// Host side of the operators on a paged K/V cache: argument checks and launches.
#include "../../include/fa2_b200.h"
#include "fa2_paged_params.h"
#include "fa2_runtime.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <initializer_list>

namespace {

using fa2::DeviceScope;
using fa2::fail;
using fa2::get_runtime;
using fa2::make_div;
using fa2::PageTable;
using fa2::Runtime;
using fa2::Strides3;

constexpr int kMostRows = INT_MAX - 65536;  // tokens or keys that 32-bit indices are used for

Strides3 strides(const int64_t* s) { return Strides3{s[0], s[1], s[2]}; }

bool addressable(const void* ptr, const int64_t* stride) {
  if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] % 8 != 0) return false;
  return true;
}

bool aligned4(std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return false;
  return true;
}

// A tensor [batch, rows, heads, .] that is turned in place has to stay where it is.
bool apart_or_in_place(const void* in, const int64_t* in_stride, const void* out, const int64_t* out_stride, int batch, int rows, int heads) {
  if (in != out) return true;
  return (batch <= 1 || in_stride[0] == out_stride[0]) && (rows <= 1 || in_stride[1] == out_stride[1]) && (heads <= 1 || in_stride[2] == out_stride[2]);
}

int check_types(int dtype, int head_dim) {
  if (dtype != FA2_F16 && dtype != FA2_BF16) return fail(FA2_E_TYPE, "tensors must be float16 or bfloat16");
  if (head_dim < 8 || head_dim > 256 || head_dim % 8 != 0)
    return fail(FA2_E_VALUE, "head dim must be a multiple of 8 up to 256, got %d", head_dim);
  return FA2_OK;
}

int check_cache(const fa2_paged_cache* c) {
  if (c == nullptr) return fail(FA2_E_VALUE, "cache is null");
  if (c->size != static_cast<int64_t>(sizeof(fa2_paged_cache))) return fail(FA2_E_VALUE, "fa2_paged_cache has an unknown size");
  if (const int rc = check_types(c->dtype, c->head_dim)) return rc;
  if (c->reserved != 0) return fail(FA2_E_VALUE, "reserved must be 0");
  if (c->num_pages <= 0 || c->page_size <= 0 || c->max_pages <= 0)
    return fail(FA2_E_VALUE, "num_pages, page_size and max_pages must be positive, got %d, %d and %d", c->num_pages, c->page_size, c->max_pages);
  if (c->batch <= 0 || c->batch > 65535 || c->heads_k <= 0 || c->heads_k > 65535)
    return fail(FA2_E_VALUE, "batch and heads must each be in 1..=65535, got %d and %d", c->batch, c->heads_k);
  if (static_cast<int64_t>(c->batch) * c->heads_k > kMostRows) return fail(FA2_E_VALUE, "batch * heads_k must be below %d", kMostRows);
  if (c->k == nullptr || c->v == nullptr || c->block_table == nullptr || c->seqlens_k == nullptr)
    return fail(FA2_E_VALUE, "k, v, block_table and seqlens_k must be non-null");
  if (!aligned4({c->attn_mass, c->block_table, c->seqlens_k})) return fail(FA2_E_VALUE, "attn_mass, block_table and seqlens_k must be 4-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (c->k_stride[i] < 0 || c->v_stride[i] < 0) return fail(FA2_E_VALUE, "strides of k and v must not be negative");
  if (!addressable(c->k, c->k_stride) || !addressable(c->v, c->v_stride))
    return fail(FA2_E_VALUE, "k and v must be 16-byte aligned, with outer strides that are multiples of 8 elements");
  return FA2_OK;
}

PageTable table_of(const fa2_paged_cache* c, const int32_t* pages, int64_t stride, int max_pages) {
  PageTable t;
  t.pages = pages;
  t.stride = stride;
  t.max_pages = max_pages;
  t.num_pages = c->num_pages;
  t.page_size = make_div(c->page_size);
  return t;
}
PageTable table_of(const fa2_paged_cache* c) { return table_of(c, c->block_table, c->block_table_stride, c->max_pages); }

int rotary_params(const fa2_rotary_args* a, fa2::RotaryParams* p) {
  if (a == nullptr) return fail(FA2_E_VALUE, "args is null");
  if (a->size != static_cast<int64_t>(sizeof(fa2_rotary_args))) return fail(FA2_E_VALUE, "fa2_rotary_args has an unknown size");
  if (const int rc = check_types(a->dtype, a->head_dim)) return rc;
  if (a->reserved != 0) return fail(FA2_E_VALUE, "reserved must be 0");
  if (a->batch < 0 || a->seqlen < 0 || static_cast<int64_t>(a->batch) * a->seqlen > kMostRows)
    return fail(FA2_E_VALUE, "batch * seqlen must be in 0..=%d, got %d and %d", kMostRows, a->batch, a->seqlen);
  if ((a->q != nullptr && (a->heads <= 0 || a->heads > 65535)) || (a->k != nullptr && (a->heads_k <= 0 || a->heads_k > 65535)))
    return fail(FA2_E_VALUE, "heads must be in 1..=65535, got %d and %d", a->heads, a->heads_k);
  if (a->axes < 1 || a->axes > fa2::kMaxAxes) return fail(FA2_E_VALUE, "axes must be in 1..=%d, got %d", fa2::kMaxAxes, a->axes);
  int64_t pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->sections[i] < 0) return fail(FA2_E_VALUE, "sections must not be negative");
    pairs += a->sections[i];
  }
  if (pairs < 1 || 2 * pairs > a->head_dim)
    return fail(FA2_E_VALUE, "sections must add up to 1..=%d pairs, got %lld", a->head_dim / 2, static_cast<long long>(pairs));
  if (a->interleaved_axes)
    for (int i = 1; i < a->axes; ++i)
      if (a->sections[i] > 0 && a->axes * (a->sections[i] - 1) + i >= pairs)
        return fail(FA2_E_VALUE, "interleaved_axes: axis %d has more pairs than its turns among %lld", i, static_cast<long long>(pairs));
  if (a->position_bits != 32 && a->position_bits != 64) return fail(FA2_E_VALUE, "position_bits must be 32 or 64");
  *p = fa2::RotaryParams{};
  p->tokens = a->batch * a->seqlen;
  p->heads = a->q != nullptr ? a->heads : 0;
  p->heads_k = a->k != nullptr ? a->heads_k : 0;
  p->head_dim = a->head_dim;
  p->pairs = static_cast<int>(pairs);
  if (p->tokens == 0 || p->heads + p->heads_k == 0) return FA2_OK;
  if (a->positions == nullptr || a->inv_freq == nullptr) return fail(FA2_E_VALUE, "positions and inv_freq must be non-null");
  if (reinterpret_cast<uintptr_t>(a->positions) % (a->position_bits / 8) || reinterpret_cast<uintptr_t>(a->inv_freq) % 4)
    return fail(FA2_E_VALUE, "positions and inv_freq must be aligned to their elements");
  if (a->q != nullptr && a->q_out == nullptr) return fail(FA2_E_VALUE, "q_out is null");
  for (const void* t : {a->q, static_cast<const void*>(a->q_out), a->k})
    if (reinterpret_cast<uintptr_t>(t) % 2) return fail(FA2_E_VALUE, "tensors must be aligned to their elements");
  if (a->q != nullptr && !apart_or_in_place(a->q, a->q_stride, a->q_out, a->q_out_stride, a->batch, a->seqlen, a->heads))
    return fail(FA2_E_VALUE, "q_out is q, but its strides are others");
  p->q = a->q;
  p->q_out = a->q_out;
  p->k = a->k;
  p->k_out = a->k_out;
  p->qs = strides(a->q_stride);
  p->qos = strides(a->q_out_stride);
  p->ks = strides(a->k_stride);
  p->kos = strides(a->k_out_stride);
  p->seqlen = make_div(a->seqlen);
  p->items = make_div((a->head_dim + 15) / 16);
  p->positions = a->positions;
  p->positions64 = a->position_bits == 64;
  p->pos_axis = a->position_stride[0];
  p->pos_batch = a->position_stride[1];
  p->pos_row = a->position_stride[2];
  p->inv_freq = a->inv_freq;
  p->axes = a->axes;
  memcpy(p->sections, a->sections, sizeof(p->sections));
  p->in_turns = a->interleaved_axes != 0;
  p->neighbours = a->interleaved_pairs != 0;
  p->negate = a->inverse != 0;
  return FA2_OK;
}

int rotary_launch(fa2::RotaryParams* p, int dtype, bool append, bool vectors, Runtime* rt, cudaStream_t stream) {
  const int heads = p->heads + p->heads_k + (append ? p->heads_k : 0);
  p->heads_all = make_div(heads);
  // A warp has a token's heads to itself where that fills the GPU with 16 warps per SM; else they are shared, down to a head a lane.
  const int64_t fill = 16 * static_cast<int64_t>(rt->sm_count);
  const int at_once = 32 / static_cast<int>(p->items.d);
  p->warps_log = 0;
  while ((static_cast<int64_t>(p->tokens) << p->warps_log) < fill && (at_once << p->warps_log) < heads && p->warps_log < 8) ++p->warps_log;
  p->status = rt->status;
  const cudaError_t e = fa2::launch_rotary(*p, dtype == FA2_BF16, append, vectors, stream);
  if (e != cudaSuccess) return fail(FA2_E_RUNTIME, "rotary launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

// What a call of fa2_paged_fwd takes besides its arguments.
struct FwdPlan {
  int most_keys = 0, rows = 0, row_tiles = 0, grid = 0;
  int64_t score_stride = 0;
  int64_t list_bytes = 0, part_bytes = 0, unit_bytes = 0, stat_bytes = 0, score_bytes = 0;
  int64_t bytes() const { return list_bytes + part_bytes + unit_bytes + stat_bytes + score_bytes; }
};
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

int plan_fwd(const fa2_paged_fwd_args* a, int sm_count, FwdPlan* f) {
  const fa2_paged_cache* c = a->cache;
  const int64_t capacity = std::min<int64_t>(static_cast<int64_t>(c->max_pages) * c->page_size, kMostRows);
  f->most_keys = static_cast<int>(a->max_seqlen_k > 0 ? std::min<int64_t>(a->max_seqlen_k, capacity) : capacity);
  f->rows = a->seqlen_q * (a->heads / c->heads_k);
  const int unit_rows = fa2::paged_unit_rows(f->rows);
  f->row_tiles = (f->rows + unit_rows - 1) / unit_rows;
  const int64_t most_tiles = static_cast<int64_t>(c->batch) * c->heads_k * f->row_tiles * ((f->most_keys + static_cast<int64_t>(fa2::kPagedTile) - 1) / fa2::kPagedTile);
  f->grid = static_cast<int>(std::min<int64_t>(sm_count, (most_tiles + fa2::kPagedMinShare - 1) / fa2::kPagedMinShare));
  f->list_bytes = round256(static_cast<int64_t>(f->grid) * 16);
  f->part_bytes = round256(2 * static_cast<int64_t>(f->grid) * fa2::paged_part_floats(c->head_dim, f->rows) * 4);
  const int64_t units = static_cast<int64_t>(c->batch) * c->heads_k * f->row_tiles;
  if (c->attn_mass != nullptr || fa2::paged_join_by_unit(units, f->grid, f->rows)) f->unit_bytes = round256(units * 8);
  if (c->attn_mass != nullptr) {
    const int64_t rows = static_cast<int64_t>(c->batch) * c->heads_k * f->rows;
    f->score_stride = (f->most_keys + 15) / 16 * 16;
    f->stat_bytes = round256(rows * 8);
    if (rows > (INT64_MAX >> 8) / f->score_stride) return fail(FA2_E_VALUE, "the scores of this call do not fit an address space");
    f->score_bytes = round256(rows * f->score_stride * 4);
  }
  return FA2_OK;
}

int check_fwd(const fa2_paged_fwd_args* a) {
  if (a == nullptr) return fail(FA2_E_VALUE, "args is null");
  if (a->size != static_cast<int64_t>(sizeof(fa2_paged_fwd_args))) return fail(FA2_E_VALUE, "fa2_paged_fwd_args has an unknown size");
  if (const int rc = check_cache(a->cache)) return rc;
  if (a->heads <= 0 || a->heads > 65535 || a->heads % a->cache->heads_k != 0)
    return fail(FA2_E_VALUE, "num_heads (%d) must be a multiple of num_heads_k (%d)", a->heads, a->cache->heads_k);
  if (a->seqlen_q < 0) return fail(FA2_E_VALUE, "seqlen_q must not be negative");
  if (static_cast<int64_t>(a->seqlen_q) * (a->heads / a->cache->heads_k) > fa2::kPagedMaxRows)
    return fail(FA2_E_VALUE, "at most %d query rows per kv head (seqlen_q * num_heads / num_heads_k), got %lld: a longer chunk goes in "
                "pieces, each with lengths up to its own last token", fa2::kPagedMaxRows, static_cast<long long>(a->seqlen_q) * (a->heads / a->cache->heads_k));
  if (!std::isfinite(a->softmax_scale)) return fail(FA2_E_VALUE, "softmax_scale must be finite");
  if (!std::isfinite(a->softcap) || a->softcap < 0.f) return fail(FA2_E_VALUE, "softcap must be finite and not negative");
  if (a->max_seqlen_k < 0) return fail(FA2_E_VALUE, "max_seqlen_k must not be negative");
  return FA2_OK;
}

}  // namespace

extern "C" {

int fa2_rotary(const fa2_rotary_args* args, void* stream) {
  fa2::RotaryParams p;
  int rc = rotary_params(args, &p);
  if (rc != FA2_OK) return rc;
  if (p.tokens == 0 || p.heads + p.heads_k == 0) return FA2_OK;
  if (p.k != nullptr && (p.k_out == nullptr || reinterpret_cast<uintptr_t>(p.k_out) % 2))
    return fail(FA2_E_VALUE, "k_out must be non-null and aligned to its elements");
  if (p.k != nullptr && !apart_or_in_place(p.k, args->k_stride, p.k_out, args->k_out_stride, args->batch, args->seqlen, args->heads_k))
    return fail(FA2_E_VALUE, "k_out is k, but its strides are others");
  const DeviceScope scope(p.q != nullptr ? p.q : p.k);
  Runtime* rt = nullptr;
  if ((rc = get_runtime(scope.device(), &rt)) != FA2_OK) return rc;
  const bool vectors = p.pairs % 8 == 0 &&
                       (p.q == nullptr || (addressable(p.q, args->q_stride) && addressable(p.q_out, args->q_out_stride))) &&
                       (p.k == nullptr || (addressable(p.k, args->k_stride) && addressable(p.k_out, args->k_out_stride)));
  return rotary_launch(&p, args->dtype, false, vectors, rt, static_cast<cudaStream_t>(stream));
}

int fa2_paged_append(const fa2_paged_append_args* args, void* stream) {
  if (args == nullptr) return fail(FA2_E_VALUE, "args is null");
  if (args->size != static_cast<int64_t>(sizeof(fa2_paged_append_args))) return fail(FA2_E_VALUE, "fa2_paged_append_args has an unknown size");
  fa2::RotaryParams p;
  int rc = rotary_params(args->turn, &p);
  if (rc != FA2_OK) return rc;
  if ((rc = check_cache(args->cache)) != FA2_OK) return rc;
  const fa2_rotary_args* t = args->turn;
  const fa2_paged_cache* c = args->cache;
  if (t->k == nullptr && p.tokens > 0) return fail(FA2_E_VALUE, "k is null");
  if (t->heads_k != c->heads_k || t->head_dim != c->head_dim) return fail(FA2_E_VALUE, "k must have the cache's heads and head dim");
  if (t->dtype != c->dtype) return fail(FA2_E_TYPE, "k and the cache must share dtype");
  if (args->cu_seqlens != nullptr && (t->batch != 1 || args->seqlens_new != nullptr))
    return fail(FA2_E_VALUE, "with cu_seqlens the batch of the new tokens is 1 and seqlens_new is null");
  if (args->cu_seqlens == nullptr && t->batch != c->batch) return fail(FA2_E_VALUE, "the new tokens must have the cache's batch");
  if (p.tokens == 0) return FA2_OK;
  if (args->v == nullptr || reinterpret_cast<uintptr_t>(args->v) % 2) return fail(FA2_E_VALUE, "v must be non-null and aligned to its elements");
  if (!aligned4({args->cu_seqlens, args->seqlens_new})) return fail(FA2_E_VALUE, "cu_seqlens and seqlens_new must be 4-byte aligned");
  const DeviceScope scope(c->k);
  Runtime* rt = nullptr;
  if ((rc = get_runtime(scope.device(), &rt)) != FA2_OK) return rc;
  p.k_out = c->k;
  p.v_out = c->v;
  p.kos = strides(c->k_stride);
  p.vos = strides(c->v_stride);
  p.v = args->v;
  p.vs = strides(args->v_stride);
  p.table = table_of(c);
  p.seqlens = c->seqlens_k;
  p.cu_seqlens = args->cu_seqlens;
  p.seqlens_new = args->seqlens_new;
  p.sequences = c->batch;
  p.mass = c->attn_mass;
  const bool vectors = p.pairs % 8 == 0 && addressable(p.k, t->k_stride) && addressable(p.v, args->v_stride) &&
                       (p.q == nullptr || (addressable(p.q, t->q_stride) && addressable(p.q_out, t->q_out_stride)));
  return rotary_launch(&p, t->dtype, true, vectors, rt, static_cast<cudaStream_t>(stream));
}

int64_t fa2_paged_fwd_workspace_bytes(const fa2_paged_fwd_args* args) {
  if (check_fwd(args) != FA2_OK || args->seqlen_q == 0) return 0;
  const DeviceScope scope(args->cache->k);
  Runtime* rt = nullptr;
  FwdPlan f;
  if (get_runtime(scope.device(), &rt) != FA2_OK || plan_fwd(args, rt->sm_count, &f) != FA2_OK) return 0;
  return f.bytes();
}

int fa2_paged_fwd(const fa2_paged_fwd_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_fwd(args);
  if (rc != FA2_OK) return rc;
  if (args->seqlen_q == 0) return FA2_OK;
  const fa2_paged_cache* c = args->cache;
  if (args->q == nullptr || args->out == nullptr || args->lse == nullptr) return fail(FA2_E_VALUE, "q, out and lse must be non-null");
  if (!aligned4({args->lse})) return fail(FA2_E_VALUE, "lse must be 4-byte aligned");
  if (!addressable(args->q, args->q_stride) || !addressable(args->out, args->o_stride))
    return fail(FA2_E_VALUE, "q and out must be 16-byte aligned, with outer strides that are multiples of 8 elements");
  const DeviceScope scope(c->k);
  Runtime* rt = nullptr;
  if ((rc = get_runtime(scope.device(), &rt)) != FA2_OK) return rc;
  FwdPlan f;
  if ((rc = plan_fwd(args, rt->sm_count, &f)) != FA2_OK) return rc;
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < f.bytes())
    return fail(FA2_E_VALUE, "the workspace must be 256-byte aligned and have %lld bytes", static_cast<long long>(f.bytes()));
  fa2::PagedParams p{};
  p.q = args->q;
  p.k = c->k;
  p.v = c->v;
  p.o = args->out;
  p.lse = args->lse;
  p.qs = strides(args->q_stride);
  p.ks = strides(c->k_stride);
  p.vs = strides(c->v_stride);
  p.os = strides(args->o_stride);
  p.table = table_of(c);
  // A tensor map needs strides other than zero; heads or pages that share their memory are copied like pages of other sizes.
  const bool apart = (c->heads_k == 1 || (c->k_stride[2] > 0 && c->v_stride[2] > 0)) && (c->page_size == 1 || (c->k_stride[1] > 0 && c->v_stride[1] > 0)) &&
                     (c->num_pages == 1 || (c->k_stride[0] > 0 && c->v_stride[0] > 0));
  p.tiled = c->page_size % fa2::kPagedTile == 0 && apart;
  if (p.tiled) {
    const bool wide = c->head_dim * 2 % 256 == 0;
    if ((rc = fa2::make_map(&p.tm_k, c->k, c->dtype, 2, c->head_dim, c->heads_k, c->page_size, c->num_pages, c->k_stride[2], c->k_stride[1],
                            c->k_stride[0], 64, fa2::kPagedTile, "k", wide)) != FA2_OK)
      return rc;
    if ((rc = fa2::make_map(&p.tm_v, c->v, c->dtype, 2, c->head_dim, c->heads_k, c->page_size, c->num_pages, c->v_stride[2], c->v_stride[1],
                            c->v_stride[0], 64, fa2::kPagedTile, "v", wide)) != FA2_OK)
      return rc;
  }
  p.seqlens = c->seqlens_k;
  p.most_keys = f.most_keys;
  p.batch = c->batch;
  p.heads = args->heads;
  p.heads_k = c->heads_k;
  p.seqlen_q = args->seqlen_q;
  p.head_dim = c->head_dim;
  p.group = make_div(args->heads / c->heads_k);
  p.rows = f.rows;
  p.row_tiles = f.row_tiles;
  p.window = args->window_left >= f.most_keys ? -1 : args->window_left;  // a window of all keys is none
  p.scale = args->softmax_scale;
  p.scale_log2 = args->softmax_scale * 1.4426950408889634f;
  p.softcap = args->softcap;
  char* at = static_cast<char*>(workspace);
  p.shared = reinterpret_cast<int4*>(at);
  p.partials = reinterpret_cast<float*>(at += f.list_bytes);
  at += f.part_bytes;
  if (f.unit_bytes > 0) p.units = reinterpret_cast<int2*>(at);
  if (c->attn_mass != nullptr) {
    p.stats = reinterpret_cast<float2*>(at += f.unit_bytes);
    p.scores = reinterpret_cast<float*>(at += f.stat_bytes);
    p.score_stride = f.score_stride;
    p.mass = c->attn_mass;
  }
  p.status = rt->status;
  const cudaError_t e = fa2::launch_fwd_paged(p, f.grid, rt->sm_count, c->dtype == FA2_BF16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(FA2_E_RUNTIME, "paged forward launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

int fa2_paged_evict(const fa2_paged_evict_args* args, void* stream) {
  if (args == nullptr) return fail(FA2_E_VALUE, "args is null");
  if (args->size != static_cast<int64_t>(sizeof(fa2_paged_evict_args))) return fail(FA2_E_VALUE, "fa2_paged_evict_args has an unknown size");
  int rc = check_cache(args->cache);
  if (rc != FA2_OK) return rc;
  const fa2_paged_cache* c = args->cache;
  if (args->reserved != 0) return fail(FA2_E_VALUE, "reserved must be 0");
  if (c->attn_mass == nullptr) return fail(FA2_E_VALUE, "attn_mass is null");
  if (args->budget < 1 || args->budget > kMostRows || args->recent < 0 || args->recent > args->budget)
    return fail(FA2_E_VALUE, "budget must be in 1..=%d and recent in 0..=budget, got %d and %d", kMostRows, args->budget, args->recent);
  if (args->dst_block_table == nullptr || args->seqlens_out == nullptr || args->kept == nullptr || args->dst_max_pages <= 0)
    return fail(FA2_E_VALUE, "dst_block_table, seqlens_out and kept must be non-null, dst_max_pages positive");
  if (!aligned4({args->dst_block_table, args->seqlens_out, args->kept})) return fail(FA2_E_VALUE, "dst_block_table, seqlens_out and kept must be 4-byte aligned");
  const DeviceScope scope(c->k);
  Runtime* rt = nullptr;
  if ((rc = get_runtime(scope.device(), &rt)) != FA2_OK) return rc;
  fa2::EvictParams p{};
  p.k = c->k;
  p.v = c->v;
  p.mass = c->attn_mass;
  p.ks = strides(c->k_stride);
  p.vs = strides(c->v_stride);
  p.from = table_of(c);
  p.to = table_of(c, args->dst_block_table, args->dst_block_table_stride, args->dst_max_pages);
  p.seqlens = c->seqlens_k;
  p.seqlens_out = args->seqlens_out;
  p.kept = args->kept;
  p.batch = c->batch;
  p.heads_k = c->heads_k;
  p.head_dim = c->head_dim;
  p.budget = args->budget;
  p.recent = args->recent;
  p.status = rt->status;
  const cudaError_t e = fa2::launch_paged_evict(p, rt->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(FA2_E_RUNTIME, "eviction launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

}  // extern "C"
