/*
 * akt_amd.h - C ABI of the gfx950 attention kernel library (libakt_amd.so).
 *
 * Every entry point takes plain device pointers, element strides and sizes,
 * launches asynchronously on the given HIP stream (passed as void*; NULL is
 * the default stream) and returns AKT_OK or an error code; on error
 * akt_last_error() returns a message for the calling thread.  Nothing here
 * synchronises the stream or allocates device memory: the split-KV decode
 * entry points take a caller-owned workspace of the size reported by the
 * matching *_workspace_size() function.
 *
 * Workspace contract (all decode entry points): the first
 * min(AKT_WORKSPACE_ZERO_BYTES, workspace size) bytes hold scheduling and
 * per-unit arrival counters and must be zero before a workspace is first
 * used; every call leaves them zero again when it completes.  (The counters
 * of calls with more than 32768 units past that prefix are zero-filled by the
 * call itself.)  A workspace may be reused by any decode entry point, but
 * only by calls ordered on one stream (calls that overlap in time must use
 * different workspaces).
 *
 * Tensor element types: q/k/v/o and KV pools are IEEE fp16 (entry points with a dtype
 * argument also take bf16, and akt_paged_kv_append and akt_paged_copy move any 2-byte
 * elements); page tables, kept-token indices and counts are int32;
 * MagicPIG K/L and LSE are fp32.
 * Strides are in elements.  The innermost (head_dim) stride must be 1 and
 * every row must start 16-byte aligned.
 *
 * Reference interfaces replaced (KiritoHugh/attention_kernel_triton):
 *   prefill_flash_attention.py:342                       flash_attention_prefill
 *   prefill_flash_attention_var_len_padding.py:348       flash_attention_prefill(varlen=)
 *   decode_flash_attention_redundant.py:233              flash_attention_decode
 *   decode_flash_attention_redundant_var_len_paged.py:228  flash_attention_decode_paged
 *   sparsetoken_decode_flash_attention_redundant.py:127  sparsetoken_flash_attention_decode
 *   sparsetoken_decode_flash_attention_redundant_var_len_paged.py:170
 *                                                        sparsetoken_flash_attention_decode_paged
 *   magicpig_sparsetoken_decode_flash_attention_redundant_var_len_paged_with_norm.py:166
 *                                                        magicpig_sparsetoken_flash_attention_decode_paged
 *   sparsetoken_decode_flash_attention_redundant.py:283-295 (kept-index selection, harness code)
 *   prefill_flash_attention.py:331-334 (stubbed LSE store)  akt_prefill_fwd_lse, akt_merge_states
 *   sparse_decode_flash_attention.py:13-15 (CSR index note)   akt_sparse_decode_*csr_fwd
 *   decode_flash_attention_redundant_var_len_paged.py:349-353 (page tables, harness)
 *                                                        akt_paged_kv_append
 * Without a counterpart there: akt_chunk_paged_fwd, akt_rotary_fwd,
 * akt_paged_kv_append_rotary and akt_paged_copy, which serve a paged cache beyond
 * single-token decode; akt_shared_prefix_paged_fwd, akt_attention_weights_paged,
 * akt_kept_index_heaviest and akt_paged_keep, which keep what is read and held of one small.
 */
#ifndef AKT_AMD_H
#define AKT_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AKT_OK 0
#define AKT_ERR_INVALID_ARGUMENT 1 /* shape, stride, alignment or value check failed */
#define AKT_ERR_UNSUPPORTED 2      /* a valid request this build has no kernel for   */
#define AKT_ERR_WORKSPACE 3        /* workspace missing or smaller than required      */
#define AKT_ERR_HIP 4              /* the HIP runtime reported an error at launch     */

/* Element types for entry points that accept more than one. */
#define AKT_DTYPE_F16 0
#define AKT_DTYPE_F32 1
#define AKT_DTYPE_BF16 2

/* Message describing the last failure on the calling thread ("" if none). */
const char* akt_last_error(void);

/* ABI version of this header (bumped on any signature or contract change). */
#define AKT_ABI_VERSION 2
int akt_abi_version(void);

/* Bytes at the start of a decode workspace that must be zero before its first
 * use: a 256-byte counter header and 32768 int32 arrival counters. */
#define AKT_WORKSPACE_ZERO_BYTES (256u + 32768u * 4u)

/*
 * Causal / non-causal GQA prefill, O = softmax(scale * Q K^T [+ causal]) V.
 * Replaces prefill_flash_attention.py:342 and, with varlen != NULL,
 * prefill_flash_attention_var_len_padding.py:348.
 *   q, o: [batch, num_q_heads, seq_len, head_dim]; k, v: [batch, num_kv_heads,
 *   seq_len, head_dim]; q head h reads kv head h / (num_q_heads / num_kv_heads).
 *   varlen: optional device array [batch] of valid lengths (int32 when
 *   varlen_bits == 32, int64 when 64, ignored when varlen == NULL).  Query
 *   blocks of 64 rows that start at or beyond a sequence's length are not
 *   written (as in the reference); rows < length never read keys >= length
 *   when causal.
 *   head_dim: 64, 128, 192 or 256.
 */
int akt_prefill_fwd(const void* q, const void* k, const void* v, void* o,
                    int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                    int64_t seq_len, int64_t head_dim,
                    const int64_t q_stride[4], const int64_t k_stride[4],
                    const int64_t v_stride[4], const int64_t o_stride[4],
                    float softmax_scale, int causal,
                    const void* varlen, int varlen_bits, void* stream);

/*
 * akt_prefill_fwd plus the natural-log softmax normaliser of every computed
 * row: lse[b, h, s] = ln sum_k exp(scale * q_s . k) over the keys row s
 * attends (fp32, strides lse_stride[0..2] over batch, head, row).  Rows that
 * akt_prefill_fwd leaves unwritten are left unwritten here too.  The
 * reference computes the same quantity and leaves its store commented out
 * (prefill_flash_attention.py:331-334); this is its public form, for
 * chunked prefill and akt_merge_states.
 */
int akt_prefill_fwd_lse(const void* q, const void* k, const void* v, void* o, float* lse,
                        int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                        int64_t seq_len, int64_t head_dim,
                        const int64_t q_stride[4], const int64_t k_stride[4],
                        const int64_t v_stride[4], const int64_t o_stride[4],
                        const int64_t lse_stride[3], float softmax_scale, int causal,
                        const void* varlen, int varlen_bits, void* stream);

/*
 * akt_prefill_fwd / akt_prefill_fwd_lse for either element type: q, k, v and
 * o are all fp16 (dtype AKT_DTYPE_F16) or all bf16 (AKT_DTYPE_BF16); lse may
 * be NULL (no normaliser; lse_stride is then ignored).  With bf16 both MFMA
 * products run in bf16 and the probabilities are rounded to bf16 for P.V (the
 * fp16 path rounds them to fp16, as the reference's prefill does at
 * prefill_flash_attention.py:94).  The reference's prefill kernels take fp16
 * only (their P.V casts P to fp16); this entry point has no counterpart there.
 */
int akt_prefill_fwd_ex(const void* q, const void* k, const void* v, void* o, float* lse,
                       int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                       int64_t seq_len, int64_t head_dim,
                       const int64_t q_stride[4], const int64_t k_stride[4],
                       const int64_t v_stride[4], const int64_t o_stride[4],
                       const int64_t lse_stride[3], float softmax_scale, int causal,
                       const void* varlen, int varlen_bits, int dtype, void* stream);

/*
 * Merge attention states computed over disjoint key sets.  For each of
 * `rows` (query, head) rows and n_parts parts i:
 *   lse_out = ln sum_i exp(lse_i),  o_out = sum_i exp(lse_i - lse_out) o_i.
 * Parts with lse_i = -inf contribute nothing; a row with no contributing
 * part gets o_out = 0 and lse_out = -inf.  No reference counterpart: it is
 * the combine the reference's stubbed LSE stores
 * (prefill_flash_attention.py:331-334, decode_flash_attention_redundant.py:225-228)
 * would feed, for chunked prefill / decode and per-GPU shards.
 *   o_parts: [n_parts, rows, head_dim] of type o_parts_dtype (AKT_DTYPE_F16 or
 *   AKT_DTYPE_F32), strides o_parts_stride[0..1] (head_dim stride 1);
 *   lse_parts: fp32 [n_parts, rows], strides lse_parts_stride[0..1];
 *   o_out: [rows, head_dim] of type o_out_dtype, row stride o_out_row_stride;
 *   lse_out: optional fp32 [rows], stride lse_out_row_stride.
 *   head_dim: a multiple of 8 up to 512.
 */
int akt_merge_states(const void* o_parts, int o_parts_dtype, const float* lse_parts,
                     void* o_out, int o_out_dtype, float* lse_out, int64_t n_parts,
                     int64_t rows, int64_t head_dim, const int64_t o_parts_stride[2],
                     const int64_t lse_parts_stride[2], int64_t o_out_row_stride,
                     int64_t lse_out_row_stride, void* stream);

/*
 * Single-token GQA decode over a dense cache.  Replaces
 * decode_flash_attention_redundant.py:233.
 *   q: [batch, num_q_heads, 1, head_dim] (strides q_stride[0], [1], -, [3]);
 *   k, v: [batch, num_kv_heads, seq_len, head_dim];
 *   o: contiguous [batch, num_q_heads, head_dim] fp16;
 *   lse: optional contiguous [batch, num_q_heads] fp32 (natural log of the
 *   softmax normaliser of the scaled scores).  head_dim: 64, 128 or 256.
 *   chunk_tokens: split-KV chunk length: 128, 256, 512 or 640 tokens, 0 = automatic
 *   (a hint: pages that do not hold whole 16-token groups, and paged batches
 *   over 1024 sequences, use 256).  Automatic dense calls large enough to gain
 *   run the stream-K kernel (see akt_decode_paged_fwd); the workspace size then
 *   depends on the current device.
 */
size_t akt_decode_workspace_size(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                 int64_t seq_len, int64_t head_dim, int64_t chunk_tokens);
int akt_decode_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                   int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                   int64_t seq_len, int64_t head_dim,
                   const int64_t q_stride[4], const int64_t k_stride[4],
                   const int64_t v_stride[4], float softmax_scale, int64_t chunk_tokens,
                   void* workspace, size_t workspace_bytes, void* stream);

/*
 * Paged var-len GQA decode.  Replaces
 * decode_flash_attention_redundant_var_len_paged.py:228.
 *   kv_cache: [num_pool_pages, 2, num_kv_heads, page_size, head_dim] (K at
 *   [:,0], V at [:,1]) with strides kv_stride[5];
 *   kv_page_indptr [batch+1], kv_page_indices [total_pages],
 *   kv_last_page_len [batch]: int32 CSR page table.  Sequence b has
 *   (indptr[b+1]-indptr[b]-1)*page_size + last_page_len[b] tokens (0 when it
 *   has no pages; last_page_len is clamped to [0, page_size]).  Page ids
 *   outside [0, num_pool_pages) are skipped.  indptr must lie in
 *   [0, total_pages] and not decrease; where it does not, its entries are taken
 *   clamped and as a running maximum, and nothing outside the arrays is touched.
 *   o: contiguous [batch, num_q_heads, head_dim]; lse optional [batch, num_q_heads].
 *   chunk_tokens 0 (automatic) runs the stream-K kernel when batch <= 1024,
 *   page_size is a multiple of 16 and the launch is not small: every wave of
 *   the launch takes a fixed range of 16-token groups.  Its workspace has room
 *   for one partial per wave the device keeps resident plus one per (sequence,
 *   head group), more than the kernel stores (one per workgroup and one per
 *   unit that reaches into another workgroup's range), so the workspace size
 *   depends on the current device.  Otherwise, and for the
 *   explicit lengths 128, 256, 512 or 640, the chunked split kernel runs.
 */
size_t akt_decode_paged_workspace_size(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                       int64_t head_dim, int64_t page_size, int64_t total_pages,
                                       int64_t chunk_tokens);
int akt_decode_paged_fwd(const void* q, const void* kv_cache, const int32_t* kv_page_indptr,
                         const int32_t* kv_page_indices, const int32_t* kv_last_page_len,
                         void* o, float* lse, int64_t batch, int64_t num_q_heads,
                         int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                         int64_t total_pages, int64_t num_pool_pages,
                         const int64_t q_stride[4], const int64_t kv_stride[5],
                         float softmax_scale, int64_t chunk_tokens,
                         void* workspace, size_t workspace_bytes, void* stream);

/*
 * akt_decode_paged_fwd without a workspace argument: no reference
 * counterpart.  It is for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc), and it allocates nothing.  The split-KV workspace is a
 * file-scope device array of AKT_NOALLOC_SCRATCH_BYTES that every GPU the
 * library runs on holds until the process ends; its counter area is
 * zero-filled (by a fill kernel on `stream`) at the first call on a device,
 * and every launch leaves its counters at zero again.  A call whose workspace
 * (akt_decode_paged_workspace_size of the same arguments) exceeds the array
 * fails with AKT_ERR_INVALID_ARGUMENT.  All calls on one GPU share the array:
 * calls that overlap in time on one GPU race, so order them (one stream).
 * Results are bit-identical to akt_decode_paged_fwd's.
 */
#define AKT_NOALLOC_SCRATCH_BYTES (32u << 20)
int akt_decode_paged_fwd_noalloc(const void* q, const void* kv_cache,
                                 const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                                 const int32_t* kv_last_page_len, void* o, float* lse,
                                 int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                 int64_t head_dim, int64_t page_size, int64_t total_pages,
                                 int64_t num_pool_pages, const int64_t q_stride[4],
                                 const int64_t kv_stride[5], float softmax_scale,
                                 int64_t chunk_tokens, void* stream);

/*
 * Sparse-token decode over a dense cache.  Replaces
 * sparsetoken_decode_flash_attention_redundant.py:127.
 *   sparse_ind: [batch, num_q_heads, l_max] int32 kept token indices
 *   (ascending in the reference harness; order does not matter here), entry
 *   i is used when i < sparse_nnz[b, h] (nnz is clamped to [0, l_max]).
 *   Indices outside [0, seq_len) are skipped.  A head with no kept tokens
 *   produces o = 0 and lse = -inf.
 *   ind_stride: strides of sparse_ind over (batch, head) (last stride 1);
 *   nnz_stride: strides of sparse_nnz over (batch, head).
 */
size_t akt_sparse_decode_workspace_size(int64_t batch, int64_t num_q_heads, int64_t head_dim,
                                        int64_t l_max, int64_t num_splits);
int akt_sparse_decode_fwd(const void* q, const void* k, const void* v,
                          const int32_t* sparse_ind, const int32_t* sparse_nnz,
                          void* o, float* lse, int64_t batch, int64_t num_q_heads,
                          int64_t num_kv_heads, int64_t seq_len, int64_t head_dim, int64_t l_max,
                          const int64_t q_stride[4], const int64_t k_stride[4],
                          const int64_t v_stride[4], const int64_t ind_stride[2],
                          const int64_t nnz_stride[2], float softmax_scale, int64_t num_splits,
                          void* workspace, size_t workspace_bytes, void* stream);

/*
 * Sparse-token decode over a paged var-len cache.  Replaces
 * sparsetoken_decode_flash_attention_redundant_var_len_paged.py:170.
 * Kept token t of sequence b lives in page
 * kv_page_indices[kv_page_indptr[b] + t / page_size], slot t % page_size.
 * Tokens whose logical page is outside the sequence's page list, or whose
 * page id is outside [0, num_pool_pages), are skipped.
 */
int akt_sparse_decode_paged_fwd(const void* q, const void* kv_cache,
                                const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                                const int32_t* sparse_ind, const int32_t* sparse_nnz,
                                void* o, float* lse, int64_t batch, int64_t num_q_heads,
                                int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                int64_t num_pool_pages, int64_t l_max,
                                const int64_t q_stride[4], const int64_t kv_stride[5],
                                const int64_t ind_stride[2], const int64_t nnz_stride[2],
                                float softmax_scale, int64_t num_splits,
                                void* workspace, size_t workspace_bytes, void* stream);

/*
 * MagicPIG "with norm" sparse paged decode.  Replaces
 * magicpig_sparsetoken_decode_flash_attention_redundant_var_len_paged_with_norm.py:166.
 * Score of kept token i: q.k_i / sqrt(head_dim) - ln(u_i) with
 *   c = q.k_i / (|q| |k_i| + 1e-8) clamped to [-1+1e-7, 1-1e-7],
 *   p = clamp(1 - acos(c)/pi, 0, 1), x = p^K,
 *   u = max(1 - (1-x)^L - L x (1-x)^(L-1), 1e-10),
 * with per-(batch, q head) K, L: contiguous fp32 [batch, num_q_heads].  u is
 * evaluated in fp32 in the equal form -expm1((L-1) g(-x) + g((L-1) x)),
 * g(y) = log1p(y) - y, which does not cancel for x in [0, 1) and L >= 1 (a
 * few fp32 ulps of relative error in u); x >= 1 or (L-1) x <= -1 fall back to
 * the formula as written.
 * Workspace size: akt_sparse_decode_workspace_size().
 */
int akt_magicpig_decode_paged_fwd(const void* q, const void* kv_cache,
                                  const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                                  const int32_t* sparse_ind, const int32_t* sparse_nnz,
                                  const float* lsh_k, const float* lsh_l,
                                  void* o, float* lse, int64_t batch, int64_t num_q_heads,
                                  int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                  int64_t num_pool_pages, int64_t l_max,
                                  const int64_t q_stride[4], const int64_t kv_stride[5],
                                  const int64_t ind_stride[2], const int64_t nnz_stride[2],
                                  int64_t num_splits, void* workspace, size_t workspace_bytes,
                                  void* stream);

/*
 * Sparse-token decode with kept indices in CSR form (inds + ptr) instead of
 * the -1-padded [batch, num_q_heads, l_max] rows: row u = b * num_q_heads + h
 * keeps the tokens inds[ptr[u] .. ptr[u+1]) (int32 token positions, int64
 * row pointer [batch * num_q_heads + 1]).  The second index format proposed
 * in sparse_decode_flash_attention.py:13-15 (no padding, no l_max); results
 * equal akt_sparse_decode_fwd on the same kept tokens.  max_nnz is a planning
 * hint (the longest row) for the automatic split count and the workspace size
 * (akt_sparse_decode_workspace_size with l_max = max_nnz); rows of any length
 * are handled.  Other arguments as akt_sparse_decode_fwd.
 */
int akt_sparse_decode_csr_fwd(const void* q, const void* k, const void* v, const int32_t* inds,
                              const int64_t* ptr, void* o, float* lse, int64_t batch,
                              int64_t num_q_heads, int64_t num_kv_heads, int64_t seq_len,
                              int64_t head_dim, int64_t max_nnz, const int64_t q_stride[4],
                              const int64_t k_stride[4], const int64_t v_stride[4],
                              float softmax_scale, int64_t num_splits, void* workspace,
                              size_t workspace_bytes, void* stream);

/*
 * Sparse paged decode (and, with lsh_k / lsh_l given, the MagicPIG with-norm
 * variant) with CSR kept indices; see akt_sparse_decode_csr_fwd for the CSR
 * format and akt_sparse_decode_paged_fwd / akt_magicpig_decode_paged_fwd for
 * the rest.  Scale 1/sqrt(head_dim).
 */
int akt_sparse_decode_paged_csr_fwd(const void* q, const void* kv_cache,
                                    const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                                    const int32_t* inds, const int64_t* ptr, const float* lsh_k,
                                    const float* lsh_l, void* o, float* lse, int64_t batch,
                                    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                    int64_t page_size, int64_t num_pool_pages, int64_t max_nnz,
                                    const int64_t q_stride[4], const int64_t kv_stride[5],
                                    int64_t num_splits, void* workspace, size_t workspace_bytes,
                                    void* stream);

/*
 * Paged KV cache write side: append new tokens into the page pool.
 * Sequence b's n_b = append_indptr[b+1] - append_indptr[b] new tokens
 * (rows of k_new / v_new: [total_new, num_kv_heads, head_dim], strides
 * *_new_stride[0..2]) become the last n_b logical positions of b under the
 * page table kv_page_indptr / kv_page_indices / kv_last_page_len, which must
 * already include them (see attention_kernel_triton_amd.paged_kv.PagedKVCache).
 * Writes pool[page, 0, h, slot] (K) and pool[page, 1, h, slot] (V) with the
 * decode kernels' addressing; tokens whose position or page id is outside
 * the table or pool are skipped.  No reference counterpart: the reference's
 * tests build page tables by hand
 * (decode_flash_attention_redundant_var_len_paged.py:349-353).
 */
int akt_paged_kv_append(const void* k_new, const void* v_new, const int32_t* append_indptr,
                        void* kv_cache, const int32_t* kv_page_indptr,
                        const int32_t* kv_page_indices, const int32_t* kv_last_page_len,
                        int64_t batch, int64_t total_new, int64_t num_kv_heads,
                        int64_t head_dim, int64_t page_size, int64_t num_pool_pages,
                        const int64_t k_new_stride[3], const int64_t v_new_stride[3],
                        const int64_t kv_stride[5], void* stream);

/*
 * Attention of several new tokens per sequence over a paged cache (chunked
 * prefill, verification of drafted tokens, mixed batches, single tokens).  No
 * reference counterpart.
 *   q: [total_q, num_q_heads, head_dim], strides q_stride[3]; sequence b's n_b query
 *   tokens are rows q_indptr[b] .. q_indptr[b+1] - 1 (int32 [batch+1]).
 *   kv_cache and page table as akt_decode_paged_fwd; len_b counts the new tokens, whose
 *   K and V the caller has written (akt_paged_kv_append).
 *   causal != 0: query i of sequence b sits at position len_b - n_b + i and sees the keys
 *   0 .. that position; 0: every query sees all len_b keys.
 *   o: contiguous [total_q, num_q_heads, head_dim]; lse: optional contiguous fp32
 *   [total_q, num_q_heads], ln sum_j exp(softmax_scale q.k_j).  Rows that see no key get
 *   o = 0 and lse = -inf; rows of q that belong to no sequence are not written.
 *   Keys of pages outside [0, num_pool_pages) are skipped.  q_indptr must lie in
 *   [0, total_q] and kv_page_indptr in [0, total_pages], neither decreasing; entries
 *   that do not are taken clamped and touch nothing outside the arrays.
 *   Masked K and V (later tokens, slots past len_b, skipped pages) never reach a row,
 *   whatever they hold; infinities and NaNs of V that a row sees reach it (as NaN where
 *   the probability rounds to 0).  dtype: AKT_DTYPE_F16 or AKT_DTYPE_BF16 (q, kv_cache and o; P is
 *   rounded to it for P.V, the sums are fp32).  head_dim: 64, 128 or 256;
 *   num_q_heads / num_kv_heads up to 128; total_pages * page_size below 2^30.
 *   The workspace follows the decode entry points' contract and may be shared with them;
 *   its size depends on the current device.
 */
size_t akt_chunk_paged_workspace_size(int64_t batch, int64_t total_q, int64_t num_q_heads,
                                      int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                      int64_t total_pages);
int akt_chunk_paged_fwd(const void* q, const int32_t* q_indptr, const void* kv_cache,
                        const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                        const int32_t* kv_last_page_len, void* o, float* lse, int64_t batch,
                        int64_t total_q, int64_t num_q_heads, int64_t num_kv_heads,
                        int64_t head_dim, int64_t page_size, int64_t total_pages,
                        int64_t num_pool_pages, const int64_t q_stride[3],
                        const int64_t kv_stride[5], float softmax_scale, int causal, int dtype,
                        void* workspace, size_t workspace_bytes, void* stream);

/*
 * Rotary positions of dense q [batch, num_q_heads, seq_len, head_dim] and, with
 * num_kv_heads > 0, k [batch, num_kv_heads, seq_len, head_dim], into contiguous q_out and
 * k_out.  No reference counterpart.
 *   Frequency f < rotary_dim / 2 turns dims (f, f + rotary_dim / 2), or (2 f, 2 f + 1) when
 *   interleaved, at position t by the angle t * inv_freq[f] (device fp64
 *   [rotary_dim / 2]; the angle is formed in 64 bits) and scales them by factor; dims from
 *   rotary_dim on are copied.  transpose != 0 applies the transposed map: the
 *   negative angles, the same factor (the gradient of the inputs from that of the
 *   outputs; at factor 1 the inverse).
 *   positions: optional device array, element (b, s) at b * position_stride[0] +
 *   s * position_stride[1], int32 or int64 by position_bits; NULL: 0 .. seq_len - 1.
 *   head_dim: a multiple of 8 up to 1024; rotary_dim: even, up to head_dim.  A launch has
 *   fewer than 2^32 work items: calls of batch * seq_len * head_dim from 2^35 on may be
 *   refused.
 *   dtype: AKT_DTYPE_F16 or AKT_DTYPE_BF16.
 */
int akt_rotary_fwd(const void* q, const void* k, void* q_out, void* k_out,
                   const double* inv_freq, const void* positions, int position_bits,
                   int64_t batch, int64_t num_q_heads, int64_t num_kv_heads, int64_t seq_len,
                   int64_t head_dim, int64_t rotary_dim, const int64_t q_stride[4],
                   const int64_t k_stride[4], const int64_t position_stride[2], int interleaved,
                   int transpose, float factor, int dtype, void* stream);

/*
 * akt_paged_kv_append with rotary positions: k_new is rotated (as akt_rotary_fwd) by its
 * token's position in its sequence and written into the pool, v_new is written as it is,
 * and q [total_new, num_q_heads, head_dim] (rows as k_new's) is rotated by the same
 * positions into contiguous q_out.  A token whose page lies outside the table or pool is
 * not stored, its q is rotated; rows that belong to no sequence are not written.
 * total_pages * page_size must be below 2^30, total_new at most 2^26 - 4.
 * No reference counterpart.
 */
int akt_paged_kv_append_rotary(const void* q, const void* k_new, const void* v_new, void* q_out,
                               const int32_t* append_indptr, void* kv_cache,
                               const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                               const int32_t* kv_last_page_len, const double* inv_freq,
                               int64_t batch, int64_t total_new, int64_t num_q_heads,
                               int64_t num_kv_heads, int64_t head_dim, int64_t rotary_dim,
                               int64_t page_size, int64_t total_pages, int64_t num_pool_pages,
                               const int64_t q_stride[3], const int64_t k_new_stride[3],
                               const int64_t v_new_stride[3], const int64_t kv_stride[5],
                               int interleaved, float factor, int dtype, void* stream);

/*
 * akt_paged_kv_append_rotary for sequences that have lost tokens: position_offset[b] (int32
 * [batch]; NULL: 0) is added to the positions of sequence b's tokens.
 */
int akt_paged_kv_append_rotary_at(
    const void* q, const void* k_new, const void* v_new, void* q_out, const int32_t* append_indptr,
    void* kv_cache, const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
    const int32_t* kv_last_page_len, const int32_t* position_offset, const double* inv_freq,
    int64_t batch, int64_t total_new, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
    int64_t rotary_dim, int64_t page_size, int64_t total_pages, int64_t num_pool_pages,
    const int64_t q_stride[3], const int64_t k_new_stride[3], const int64_t v_new_stride[3],
    const int64_t kv_stride[5], int interleaved, float factor, int dtype, void* stream);

/*
 * Copies the first num_tokens[i] slots (NULL: all page_size; clamped to [0, page_size]) of
 * page src[i] to page dst[i], K and V of every head, for i < n.  A pair with a page outside
 * [0, num_pool_pages), or the same page twice, is skipped.  All copies of a call run at
 * once: no page may be the destination of two of them, or the source of one and
 * the destination of another.  Up to 2^24 - 1 blocks of 16 KiB (a page takes one at
 * least) are copied by a call; more are refused.  No reference counterpart.
 */
int akt_paged_copy(void* kv_cache, const int32_t* src, const int32_t* dst,
                   const int32_t* num_tokens, int64_t n, int64_t num_kv_heads, int64_t head_dim,
                   int64_t page_size, int64_t num_pool_pages, const int64_t kv_stride[5],
                   void* stream);

/*
 * akt_chunk_paged_fwd for sequences that share prefixes: each prefix's K and V are read once for
 * all of its group.  No reference counterpart.
 *   group_indptr int32 [groups + 1]: group i is sequences group_indptr[i] .. group_indptr[i + 1]
 *   - 1 (a sequence outside [group_indptr[0], group_indptr[groups]) has no prefix).
 *   prefix_page_indptr [groups + 1], prefix_page_indices [prefix_pages], prefix_last_page_len
 *   [groups]: the prefixes' page table, in the form of the sequences' own.
 * A sequence's keys are its group's prefix, then its own (the table kv_page_*, which counts its new
 * tokens).  Every query token sees the whole prefix; of the own keys query i of n_b, at own
 * position len_b - n_b + i, sees those up to its own position (causal) or all.
 * The rest is as in akt_chunk_paged_fwd; so is the workspace, and the first
 * AKT_WORKSPACE_ZERO_BYTES of it that every call leaves zero.  Besides the parts of cut units it holds
 * two 32-bit states, 2 (4 head_dim + 16) bytes, for each query row and head.  total_q * num_q_heads
 * must be below 2^25.  Two launches.
 */
size_t akt_shared_prefix_paged_workspace_size(int64_t batch, int64_t total_q, int64_t num_q_heads,
                                              int64_t num_kv_heads, int64_t head_dim,
                                              int64_t page_size, int64_t total_pages,
                                              int64_t groups, int64_t prefix_pages);
int akt_shared_prefix_paged_fwd(
    const void* q, const int32_t* q_indptr, const void* kv_cache, const int32_t* kv_page_indptr,
    const int32_t* kv_page_indices, const int32_t* kv_last_page_len, const int32_t* group_indptr,
    const int32_t* prefix_page_indptr, const int32_t* prefix_page_indices,
    const int32_t* prefix_last_page_len, void* o, float* lse, int64_t batch, int64_t total_q,
    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
    int64_t total_pages, int64_t groups, int64_t prefix_pages, int64_t num_pool_pages,
    const int64_t q_stride[3], const int64_t kv_stride[5], float softmax_scale, int causal,
    int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Adds the attention that cached tokens draw to sums over calls.  No reference counterpart.
 *   weights[rows[b], h, j] += sum over the tokens i of sequence b that see key j and the query
 *   heads of kv head h of exp(softmax_scale * q_i . k_j - lse_i)
 * for the keys j < min(len_b, row_len).  q [total_q, num_q_heads, head_dim], q_indptr, the page
 * table and causal are those of an attention call, lse (contiguous fp32 [total_q, num_q_heads]) what
 * it returned; rows of q with lse -inf count nothing.
 *   weights: fp32 [num_rows, num_kv_heads, row_len], strides weight_stride[0..1], unit in the last; no
 *   two rows may overlap.
 *   rows: int32 [batch], the row of each sequence (NULL: b); no row may be named twice, and a
 *   sequence whose row is outside [0, num_rows) is left out.
 *   window: only the last `window` tokens of each sequence count.
 * Keys on pages outside the pool are skipped.  head_dim: 64, 128 or 256; dtype AKT_DTYPE_F16 or
 * AKT_DTYPE_BF16 (q and the cache).  The workspace is a decode workspace: its first
 * AKT_WORKSPACE_ZERO_BYTES are zero before the first call and after every call.
 */
size_t akt_attention_weights_paged_workspace_size(int64_t batch, int64_t total_q,
                                                  int64_t num_q_heads, int64_t num_kv_heads,
                                                  int64_t head_dim, int64_t page_size,
                                                  int64_t total_pages);
int akt_attention_weights_paged(
    const void* q, const int32_t* q_indptr, const float* lse, const void* kv_cache,
    const int32_t* kv_page_indptr, const int32_t* kv_page_indices, const int32_t* kv_last_page_len,
    float* weights, const int32_t* rows, int64_t batch, int64_t total_q, int64_t num_q_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t total_pages,
    int64_t num_pool_pages, int64_t num_rows, int64_t row_len, const int64_t q_stride[3],
    const int64_t kv_stride[5], const int64_t weight_stride[2], float softmax_scale, int causal,
    int64_t window, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Kept tokens close up within a cache, in place.  For each (sequence b, kv head h) and j <
 * min(sparse_nnz[b, h], keep, len_b): slot j takes K and V of token sparse_ind[b, h, j], which must
 * be at or behind slot j and before len_b (other entries are skipped: their slots stay).
 *   sparse_ind: contiguous int32 [batch, num_kv_heads, keep]; sparse_nnz: [batch, num_kv_heads].
 *   dst_page_indices: NULL, or int32 [total_pages] in the place of kv_page_indices for the slots
 *   written; where the two differ the page must be in no sequence of the call.
 *   weights: NULL, or sums as in akt_attention_weights_paged, which move along; those of slots from
 *   the count on, up to len_b, become 0.
 * No page may be written for two sequences, nor written for one and read for another.  The cache
 * is moved as 16-bit words; head_dim a multiple of 8 up to 1024.
 */
int akt_paged_keep(void* kv_cache, const int32_t* kv_page_indptr, const int32_t* kv_page_indices,
                   const int32_t* kv_last_page_len, const int32_t* dst_page_indices,
                   const int32_t* sparse_ind, const int32_t* sparse_nnz, float* weights,
                   const int32_t* rows, int64_t batch, int64_t num_kv_heads, int64_t head_dim,
                   int64_t page_size, int64_t total_pages, int64_t num_pool_pages, int64_t keep,
                   int64_t num_rows, int64_t row_len, const int64_t kv_stride[5],
                   const int64_t weight_stride[2], void* stream);

/*
 * The heaviest entries of rows of sums, as kept-token lists.  For each (sequence b, head h), of
 * the first len = min(lengths[b], row_len) entries of weights[rows[b], h]: the first `first`, the
 * last `recent` and the heaviest of the others, `keep` in all (all len where there are no more),
 * ascending in sparse_ind [batch, num_heads, keep], -1 behind them; their number in sparse_nnz
 * [batch, num_heads].  Of equal sums the lower index is kept; NaN counts as the heaviest.
 * weights, num_rows, row_len, weight_stride and rows as in akt_attention_weights_paged (a row may
 * be named twice here; a sequence whose row is outside [0, num_rows) keeps nothing).
 */
int akt_kept_index_heaviest(const float* weights, const int32_t* lengths, const int32_t* rows,
                            int32_t* sparse_ind, int32_t* sparse_nnz, int64_t batch,
                            int64_t num_heads, int64_t num_rows, int64_t row_len,
                            const int64_t weight_stride[2], int64_t keep, int64_t first,
                            int64_t recent, void* stream);

/*
 * Kept-token index selection (the reference harness step at
 * sparsetoken_decode_flash_attention_redundant.py:283-295 and
 * sparsetoken_decode_flash_attention_redundant_var_len_paged.py:341-353).
 * For each of `rows` rows: kept = {j < n_r : keep(r, j)} in ascending order,
 * where n_r = row_len[r] (or n when row_len == NULL) and keep(r, j) is
 *   mask[r * mask_row_stride + j] != 0            (akt_kept_index_from_mask)
 *   uniform[r * row_stride + j] < kept_ratio      (akt_kept_index_from_uniform)
 * If ensure_nonempty and nothing is kept, index 0 is kept.
 * Writes sparse_ind[r * l_max + i] = kept[i] for i < min(|kept|, l_max) and -1
 * for the rest of the row, and sparse_nnz[r] = |kept|.
 */
int akt_kept_index_from_mask(const uint8_t* mask, int64_t rows, int64_t n,
                             int64_t mask_row_stride, const int32_t* row_len,
                             int32_t* sparse_ind, int64_t l_max, int32_t* sparse_nnz,
                             int ensure_nonempty, void* stream);
int akt_kept_index_from_uniform(const float* uniform, float kept_ratio, int64_t rows, int64_t n,
                                int64_t row_stride, const int32_t* row_len,
                                int32_t* sparse_ind, int64_t l_max, int32_t* sparse_nnz,
                                int ensure_nonempty, void* stream);

/*
 * Kernel timer (diagnostics; no counterpart in the reference, which times
 * whole Python calls with triton.testing.do_bench).  While enabled, every
 * entry point above records a HIP event pair around its dominant kernel
 * (akt_shared_prefix_paged_fwd: around each of its two) on
 * the launch stream.  akt_kernel_timer_read() waits for the recorded events
 * and returns the summed elapsed milliseconds and the number of launches;
 * akt_kernel_timer_enable() discards what was recorded.
 */
int akt_kernel_timer_enable(int enable);
int akt_kernel_timer_read(double* total_ms, int64_t* launches);

/*
 * Read-rate ceilings (diagnostics; no counterpart in the reference, which has
 * no bandwidth model).  They measure, on the caller's data, how fast the
 * device streams the bytes a paged decode reads, with no arithmetic:
 *   akt_diag_paged_gather reads the K and V block (page_size x head_dim fp16,
 *   contiguous: kv_stride[3] == head_dim) of every (CSR page position, kv
 *   head) pair of kv_page_indices[0 .. total_pages), as the decode kernels
 *   address them (page ids outside [0, num_pool_pages) read page 0); blocks
 *   of 2, 4, 8 or 16 KB.
 *   akt_diag_stream_read reads `bytes` (a multiple of 16) from `data` in order.
 * Both write nothing but possibly one word of `sink` (a device uint32).
 */
int akt_diag_paged_gather(const void* kv_cache, const int32_t* kv_page_indices,
                          int64_t total_pages, int64_t num_kv_heads, int64_t head_dim,
                          int64_t page_size, int64_t num_pool_pages, const int64_t kv_stride[5],
                          uint32_t* sink, void* stream);
int akt_diag_stream_read(const void* data, int64_t bytes, uint32_t* sink, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AKT_AMD_H */
