/*
 * C ABI of the B200 (sm_100a) FlashAttention-2 library, libfa2_b200.so.
 *
 * Plain pointers and sizes only: device pointers are raw CUDA addresses, `stream` is a
 * cudaStream_t / CUstream passed as void*. Every call enqueues work on `stream` and returns
 * without synchronising. Return value: 0 on success, a negative FA2_E_* code on failure;
 * fa2_last_error() returns the message of the last failure on the calling thread.
 *
 * These entry points are what the host layer of the reference crate (flash-attn2-rs, Rust)
 * would bind through `extern "C"` in place of its own cuLaunchKernel calls; the tvm-ffi
 * operator symbols (__tvm_ffi_fwd, ...) in libflash_attn2_b200.so sit on top of them.
 * All tensors use the reference layouts: Q/O [B, Sq, H, D], K/V [B, Sk, Hk, D] (last stride 1),
 * LSE fp32 [B, H, Sq]; packed (varlen) Q/O [total_q, H, D], K/V [total_k, Hk, D],
 * LSE fp32 [H, total_q].
 */
#ifndef FA2_B200_H_
#define FA2_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define FA2_API __attribute__((visibility("default")))
#else
#define FA2_API
#endif

#define FA2_F16 0
#define FA2_BF16 1

#define FA2_OK 0
#define FA2_E_VALUE (-1)   /* bad shape / stride / argument value */
#define FA2_E_TYPE (-2)    /* bad dtype */
#define FA2_E_RUNTIME (-3) /* CUDA failure, or a kernel reported a stalled pipeline */

/* Strides are in elements: {batch, row, head}; the head_dim stride is 1. In packed mode
 * the batch stride is ignored. head_dim is a multiple of 8 up to 256, the reference's range
 * (flash-attn2-rs/src/host/tiles.rs:1): up to 128 on the two-stage kernels, above on kernels with
 * smaller tiles (fwd_wide_sm100.cu, bwd_wide_sm100.cu) or on pairs of CTAs (bwd_wide_pair_sm100.cu). */
typedef struct fa2_fwd_args {
  const void* q;
  const void* k;
  const void* v;
  void* out;                   /* [B, Sq, H, D] (or packed), same dtype as q */
  float* lse;                  /* contiguous fp32 [B, H, Sq] (or [H, total_q]) */
  const float* alibi_slopes;   /* fp32 [H] or [B, H], or NULL */
  int32_t alibi_batch_stride;  /* 0 for [H], H for [B, H] */
  int32_t dtype;               /* FA2_F16 or FA2_BF16 */
  int32_t batch, seqlen_q, seqlen_k, heads, heads_k, head_dim;
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3];
  float softmax_scale;
  int32_t causal;
  int32_t window_left, window_right; /* < 0 = unbounded, as passed by the caller */
  float softcap;                     /* 0 = off */
  /* packed (varlen) mode when cu_seqlens_q != NULL: device int32 [batch + 1] each;
   * seqlen_q / seqlen_k are then the maxima and total_q / total_k the packed row counts */
  const int32_t* cu_seqlens_q;
  const int32_t* cu_seqlens_k;
  int32_t total_q, total_k;
  int32_t zero_tensors; /* packed mode: clear out (0) and LSE (-inf) first, as the reference's flag does */
} fa2_fwd_args;

/* Dense forward. The bits of a head do not depend on the batch and the other heads of the call. Replaces launch_forward + flash_attn_fwd of the reference
 * (flash-attn2-rs/src/host/forward/mod.rs:449-813, src/device/forward/dense.rs:472-590).
 * Empty Sk gives O = 0 and LSE = +inf (forward/mod.rs:548-582). */
FA2_API int fa2_fwd(const fa2_fwd_args* args, void* stream);

/* The same with scratch memory: a call with few query rows, or whose (batch, head) work does not fill the GPU, is split
 * along the keys as well. How, and with it the order of its sums, follows from the sizes of the whole call; a call repeats
 * itself bit for bit. `workspace` is 256-byte aligned, its contents are irrelevant; without it, or with less than
 * fa2_fwd_workspace_bytes() bytes of it, the call does with what needs none. */
FA2_API int fa2_fwd_with_workspace(const fa2_fwd_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* Bytes of scratch memory that call can use for these arguments (0: none); reads the shapes, the window and the
 * pointers' device only. */
FA2_API int64_t fa2_fwd_workspace_bytes(const fa2_fwd_args* args);

/* Packed variable-length forward driven by cu_seqlens on the device, no host read of the
 * metadata. Replaces varlen_fwd (flash-attn2-rs/src/host/varlen/mod.rs:21-630,
 * src/device/varlen/mod.rs:30-318,445-578). */
FA2_API int fa2_varlen_fwd(const fa2_fwd_args* args, void* stream);

/* delta[b,h,s] = sum_d dO*O in fp32, rows padded to a multiple of 128 and the padding zeroed:
 * delta is [B, H, ceil(Sq/128)*128]. Replaces bwd_preprocess
 * (flash-attn2-rs/src/host/backward.rs:628-737, src/device/backward/reduce.rs:40-108). */
typedef struct fa2_bwd_preprocess_args {
  const void* dout;
  const void* out;
  float* delta;
  int32_t dtype;
  int32_t batch, seqlen_q, heads, head_dim;
  int64_t do_stride[3], o_stride[3];
  /* packed mode (varlen_preprocess, src/device/varlen/backward.rs:53-132):
   * delta is [H, total_q + 128*batch], sequence b starts at cu_seqlens_q[b] + 128*b */
  const int32_t* cu_seqlens_q;
  int32_t total_q;
} fa2_bwd_preprocess_args;
FA2_API int fa2_bwd_preprocess(const fa2_bwd_preprocess_args* args, void* stream);

/* Backward: dQ, dK, dV from Q, K, V, dO, LSE and delta. dQ is accumulated in fp32 in
 * `dq_accum` (fa2_bwd_workspace_bytes() bytes, 16-byte aligned, need not be cleared) and
 * converted to the 16-bit dQ at the end. `which` selects outputs: bit 0 = dQ, bit 1 = dK and dV.
 * A dense dQ-only call (which = 1, the deterministic bwd_dq of the reference) up to head dim 128 has a
 * kernel of its own that sums dQ in key order, so dQ is bit-reproducible; it needs no workspace. Elsewhere
 * the workspace is the accumulator (B*Sq*H*D floats, rounded up to 256 bytes), for a packed dQ-only call up to
 * head dim 128 followed by one 32-bit turn counter per 32 query rows of every (batch, head): with them it adds the
 * key blocks' contributions in a fixed order; a workspace that only holds the accumulator is accepted too
 * (arrival order). dK and dV never use atomics and are always bit-reproducible. Head dims above 128 always add dQ in
 * arrival order. A dQ-only call (which = 1) may pass dk = dv = NULL, a dK/dV-only call dq = dq_accum = NULL.
 * Replaces backward_component + the `backward` and `backward_kv` kernels
 * (flash-attn2-rs/src/host/backward.rs:14-566, src/device/backward/dq.rs:12-302,438-576,
 *  src/device/backward/dkv.rs:15-266,865-1012). */
typedef struct fa2_bwd_args {
  const void* q;
  const void* k;
  const void* v;
  const void* dout;
  const float* lse;    /* [B, H, Sq] (or [H, total_q]) */
  const float* delta;  /* layout of fa2_bwd_preprocess */
  void* dq;            /* [B, Sq, H, D] contiguous, input dtype */
  void* dk;            /* [B, Sk, Hk, D] contiguous */
  void* dv;
  void* dq_accum;      /* fp32 workspace */
  int64_t dq_accum_bytes;
  int32_t dtype;
  int32_t batch, seqlen_q, seqlen_k, heads, heads_k, head_dim;
  int64_t q_stride[3], k_stride[3], v_stride[3], do_stride[3];
  float softmax_scale;
  int32_t causal;
  int32_t window_left, window_right;
  int32_t which;
  const int32_t* cu_seqlens_q;
  const int32_t* cu_seqlens_k;
  int32_t total_q, total_k;
  /* Optional cudaEvent_t handles recorded on `stream` right before and right after the main
   * dQ/dK/dV kernel (not the memset / convert around it), for per-kernel timing. May be NULL. */
  void* ev_kernel_start;
  void* ev_kernel_stop;
  /* Score transforms of the forward pass that produced `lse` (flash-attn2-rs/src/host/backward.rs:15-34
   * takes the same two): ALiBi slopes ([H] with alibi_batch_stride 0, or [B, H] with stride H; NULL
   * for none) and the softcap (0 for none). */
  const float* alibi_slopes;
  int32_t alibi_batch_stride;
  float softcap;
} fa2_bwd_args;
FA2_API int64_t fa2_bwd_workspace_bytes(const fa2_bwd_args* args);
FA2_API int fa2_bwd(const fa2_bwd_args* args, void* stream);

/* What a backward call can do besides. */
typedef struct fa2_bwd_options {
  int64_t size; /* sizeof(fa2_bwd_options) */
  /* With `out` (the forward's output) the call computes delta itself, into the memory `delta` points to,
   * and clears the accumulator in the same pass: one kernel instead of fa2_bwd_preprocess and a fill.
   * NULL: `delta` is an input. */
  const void* out;
  int64_t o_stride[3];
  /* 1: several CTAs may share a key block when there are too few of them for the GPU (dense, head dims up to 128);
   * the workspace then has room for their fp32 parts. They are shared only in a workspace that is 256-byte aligned. dK and dV are the same bits every time either way, but not the
   * same with and without. */
  int32_t share_key_blocks;
  int32_t reserved; /* 0 */
  /* Taken and ignored: a hint that a which = 2 call may run beside the which = 1 call before it. Calls run in the order of
   * their stream. */
  int64_t beside_dq;
} fa2_bwd_options;
FA2_API int64_t fa2_bwd_workspace_bytes_with_options(const fa2_bwd_args* args, const fa2_bwd_options* options);
FA2_API int fa2_bwd_with_options(const fa2_bwd_args* args, const fa2_bwd_options* options, void* stream);

/* Views the kernels cannot address (base not 16-byte aligned, or an outer stride that is not a
 * multiple of 8 elements) are copied into a packed tensor first, as prepare_attention_tensor does
 * (flash-attn2-rs/src/host/layout.rs:80-100, kernel src/device/layout.rs:4-35). The C ABI does not
 * allocate: the caller tests the view with fa2_layout_is_addressable() (1 = usable as it is) and, if
 * needed, packs it into its own contiguous buffer with fa2_pack_16bit(): `shape` is [n0, n1, n2, d]
 * (use n0 = 1 for packed [total, H, D] tensors), `outer_strides` the element strides of n0, n1, n2;
 * the last dimension has stride 1. */
FA2_API int fa2_layout_is_addressable(const void* ptr, const int64_t* outer_strides, int32_t n_outer);
FA2_API int fa2_pack_16bit(const void* src, void* dst, const int64_t shape[4], const int64_t outer_strides[3],
                           void* stream);

/* Copy of a 16-bit tensor [n0, n1, n2, d] (unit last stride) between two layouts given by their outer element
 * strides: the general form of fa2_pack_16bit. The operator layer uses it to copy a result that was computed
 * into a temporary back into a supplied `out` the kernels cannot write in place (not addressable, or
 * overlapping an input), as the reference does (flash-attn2-rs/src/host/forward/mod.rs:367-375, 832-840,
 * src/host/layout.rs:458-512). */
FA2_API int fa2_copy_16bit(const void* src, const int64_t src_strides[3], void* dst, const int64_t dst_strides[3],
                           const int64_t shape[4], void* stream);

/* Backward that allocates nothing. No counterpart in the reference crate (its host layer always
 * allocates its workspaces through the tvm-ffi environment allocator).
 *
 * For callers that may not call cudaMalloc at all - a serving loop whose device memory was
 * partitioned up front, an embedding runtime that owns the device heap, a sandboxed plugin host -
 * this variant of fa2_bwd keeps the fp32 dQ accumulator (and the kernels' status word) in device
 * arrays that are part of the library image. It ignores args->dq_accum / dq_accum_bytes; the caller
 * still passes every input and output. Neither this call nor anything it reaches calls cudaMalloc,
 * cudaFree or an allocating library routine.
 *
 * Limits and rules:
 *  - dense tensors only, which = 3, head_dim up to 128, and batch * seqlen_q * heads * head_dim must not exceed
 *    FA2_BWD_STATIC_MAX_ELEMENTS (4,194,304: a 16 MiB array that every GPU which loads the
 *    library holds until the process exits); larger problems are rejected with FA2_E_VALUE;
 *  - the first call on a device looks up the arrays' device addresses (cudaGetSymbolAddress, with
 *    that device current). Make that first call outside any stream capture;
 *  - all calls share the one accumulator: each call clears the part it uses, and two calls whose
 *    GPU work overlaps (different streams, or different threads) race on it. Serialise them;
 *  - the kernels' pipeline status of these calls lands in the library image too; read it with
 *    fa2_bwd_static_status(), not fa2_device_status() (which reads the word of the allocating
 *    entry points and allocates it on first use);
 *  - lse and delta usually come from fa2_fwd and fa2_bwd_preprocess. fa2_bwd_preprocess allocates
 *    nothing; fa2_fwd (like fa2_bwd and fa2_device_status) allocates one 64-byte status block per
 *    device on its first call, so a host that cannot allocate later makes that first call while it
 *    still can. */
#define FA2_BWD_STATIC_MAX_ELEMENTS 4194304
FA2_API int fa2_bwd_static(const fa2_bwd_args* args, void* stream);

/* Status word of the fa2_bwd_static calls on `device`, with the meaning of fa2_device_status():
 * synchronises the device, returns 0 when every pipeline wait of those calls completed, else the code
 * of the first wait that ran out, and clears the word. It copies from and to the array in the
 * library image and allocates nothing. No counterpart in the reference crate. */
FA2_API int fa2_bwd_static_status(int device);

/* ---------------------------------------------------------------------------------------------------------------
 * Operators on a paged K/V cache: rotary positions, append, attention of the newest tokens, eviction. Every struct starts
 * with its own size. The reference's counterparts of the cache (append with rotary, paged decoding) are
 * flash-attn2-rs/src/host/cache/mod.rs:321,382 and src/device/varlen/paged.rs:26-299; positions with several axes and the
 * eviction have none. */

/* A pool of pages k, v [num_pages, page_size, heads_k, head_dim] with any outer strides {page, row, head} (in elements,
 * multiples of 8; 16-byte aligned bases), and who has which pages. Token t of sequence b lies in row t % page_size of page
 * block_table[b][t / page_size]. Two sequences may have pages in common where nothing writes to them. Entries are checked on
 * the device: a page outside the pool is neither read nor written, its keys are seen by no row, and fa2_device_status() says
 * 100; where a length exceeds what the table has room for (or max_seqlen_k) it is cut, and the status is 101. Lengths,
 * tables and weights are not to be written while a call reads them. */
typedef struct fa2_paged_cache {
  int64_t size; /* sizeof(fa2_paged_cache) */
  void* k;
  void* v;
  int64_t k_stride[3], v_stride[3];
  float* attn_mass;           /* contiguous fp32 [num_pages, heads_k, page_size], or NULL: weight that each key has got. The append
                               * starts it at 0, the attention adds to it, the eviction moves it with the key; entries of rows that
                               * hold no token may be anything */
  const int32_t* block_table; /* device int32 [batch, max_pages], unit stride in a row; entries that no token needs are ignored */
  int64_t block_table_stride;
  const int32_t* seqlens_k;   /* device int32 [batch]: tokens in the cache */
  int32_t num_pages, page_size, max_pages, batch, heads_k, head_dim, dtype;
  int32_t reserved;           /* 0 */
} fa2_paged_cache;

/* Rotary positions with several axes (time, height, width, ...). The first 2 * (sections[0] + ... ) elements of a head are
 * pairs: elements i and i + n of n pairs, or with interleaved_pairs elements 2 i and 2 i + 1; the rest is copied. A pair is
 * turned by position[axis] * inv_freq[pair], exact to a few 1e-7 rad at any position below 2^31 (frequencies up to 1).
 * Which axis: the first sections[0] pairs have axis 0, the next sections[1] axis 1 and so on; with interleaved_axes pair i has
 * axis i % axes while i < axes * sections[i % axes], and axis 0 behind that. inverse = 1 turns back: the gradient.
 * In place: q_out may be q and k_out may be k, with the same strides. Otherwise nothing that is written may overlap anything that is
 * read, and no two rows of an output each other. */
typedef struct fa2_rotary_args {
  int64_t size; /* sizeof(fa2_rotary_args) */
  const void* q; /* [batch, seqlen, heads, head_dim], or NULL */
  void* q_out;
  const void* k; /* [batch, seqlen, heads_k, head_dim], or NULL */
  void* k_out;   /* ignored by fa2_paged_append */
  int64_t q_stride[3], q_out_stride[3], k_stride[3], k_out_stride[3]; /* {batch, row, head}, any; the last stride is 1 */
  const void* positions;  /* device [axes, batch, seqlen], int32 or int64 */
  int64_t position_stride[3]; /* {axis, batch, row} */
  const float* inv_freq;  /* device fp32, one per pair */
  int32_t position_bits;  /* 32 or 64 */
  int32_t dtype;
  int32_t batch, seqlen, heads, heads_k, head_dim;
  int32_t axes;           /* 1..4 */
  int32_t sections[4];
  int32_t interleaved_axes, interleaved_pairs, inverse;
  int32_t reserved;       /* 0 */
} fa2_rotary_args;
FA2_API int fa2_rotary(const fa2_rotary_args* args, void* stream);

/* New tokens: turn->q is turned into turn->q_out, turn->k into the cache behind the seqlens_k tokens that each sequence has
 * there, and v is copied beside it; seqlens_k stays as it is. Dense: row i of sequence b is its new token i, and with
 * seqlens_new only the first seqlens_new[b] rows are. Packed (cu_seqlens; turn->batch is 1): the new tokens of sequence b are
 * the rows [cu_seqlens[b], cu_seqlens[b + 1]). The new tokens lie outside the pools. Other rows are not written to the cache; every row of q is turned. With
 * cache->attn_mass the new tokens' entries are set to 0: a row of the pool may hold the weight of a token that lay there before. */
typedef struct fa2_paged_append_args {
  int64_t size; /* sizeof(fa2_paged_append_args) */
  const fa2_rotary_args* turn;
  const fa2_paged_cache* cache;
  const void* v;
  int64_t v_stride[3];
  const int32_t* cu_seqlens;  /* device int32 [cache->batch + 1], or NULL */
  const int32_t* seqlens_new; /* device int32 [cache->batch], or NULL */
} fa2_paged_append_args;
FA2_API int fa2_paged_append(const fa2_paged_append_args* args, void* stream);

/* Attention of the last seqlen_q tokens of every sequence (which the cache holds already) over its pages: token i of them sees
 * the keys up to itself, with window_left >= 0 no more than window_left before it. At most 128 query rows per kv head
 * (seqlen_q * heads / heads_k); a longer chunk of a prompt, once it is in the cache, goes in pieces, each with the seqlens_k that end
 * at its own last token. A row without keys gives O = 0 and LSE = +inf. With cache->attn_mass the weights of each key,
 * summed over the query rows of its kv head, are added to it. The workspace is 256-byte aligned and may hold anything;
 * fa2_paged_fwd_workspace_bytes() bytes of it are needed (it grows with max_seqlen_k where there is attn_mass). A call
 * repeats itself bit for bit, attn_mass of pages that sequences share excepted. */
typedef struct fa2_paged_fwd_args {
  int64_t size; /* sizeof(fa2_paged_fwd_args) */
  const fa2_paged_cache* cache;
  const void* q; /* [batch, seqlen_q, heads, head_dim] */
  void* out;
  float* lse;    /* contiguous fp32 [batch, heads, seqlen_q] */
  int64_t q_stride[3], o_stride[3];
  int32_t seqlen_q, heads;
  float softmax_scale;
  int32_t window_left; /* < 0 = unbounded */
  float softcap;       /* 0 = off */
  int32_t max_seqlen_k; /* bound on seqlens_k, or 0: what the table has room for */
} fa2_paged_fwd_args;
FA2_API int64_t fa2_paged_fwd_workspace_bytes(const fa2_paged_fwd_args* args);
FA2_API int fa2_paged_fwd(const fa2_paged_fwd_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* Eviction. Of a sequence with more than `budget` tokens every kv head keeps its newest `recent` tokens and, of the others, the
 * budget - recent with the largest attn_mass (of equal ones the earlier; NaN counts as the largest). Shorter sequences keep
 * all. The rows that are kept, with their attn_mass, go in their order to the pages of dst_block_table; the old pages stay as
 * they are. No page of dst_block_table may be one that block_table names, or be named twice. seqlens_out[b] is the new
 * length, kept[b][head] lists the old places of the rows, -1 behind the last. */
typedef struct fa2_paged_evict_args {
  int64_t size; /* sizeof(fa2_paged_evict_args) */
  const fa2_paged_cache* cache; /* with attn_mass */
  const int32_t* dst_block_table; /* device int32 [batch, dst_max_pages] */
  int64_t dst_block_table_stride;
  int32_t dst_max_pages, budget, recent;
  int32_t reserved; /* 0 */
  int32_t* seqlens_out; /* [batch] */
  int32_t* kept;        /* [batch, heads_k, budget] */
} fa2_paged_evict_args;
FA2_API int fa2_paged_evict(const fa2_paged_evict_args* args, void* stream);

/* Message of the last failed call on this thread ("" if none). */
FA2_API const char* fa2_last_error(void);

/* Synchronises `device` and returns the kernels' status word: 0 = every pipeline wait
 * completed; otherwise the code of the first wait that ran out (the kernels bound every
 * wait instead of spinning forever), 100 or 101 = a call on a paged cache met a page or a length that cannot be. Clears the
 * word. Negative on CUDA failure. */
FA2_API int fa2_device_status(int device);

/* Number of SMs the persistent kernels size their grids for on `device`. */
FA2_API int fa2_sm_count(int device);

#ifdef __cplusplus
}
#endif
#endif /* FA2_B200_H_ */
