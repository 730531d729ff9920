/*
 * gqa_fa_b200.h - C ABI of the B200 (sm_100a) GQA flash-attention library.
 *
 * The library replaces the three Triton launches of the reference's training
 * path and the one launch of its inference path (zzhhjjj/gemma-triton-flash-attn):
 *
 *   gqafa_fwd  <- FlashAttnGQAFunction.forward launch of _flash_attn_gqa_kernel
 *                 with STORE_LSE=True          (flash_attn/attention.py:1454-1468)
 *              <- attention_flash_gqa launch with STORE_LSE=False, lse == NULL
 *                                              (flash_attn/attention.py:583-603)
 *   gqafa_bwd  <- FlashAttnGQAFunction.backward: the dQ launch with the delta
 *                 prologue (flash_attn/attention.py:1506-1523) followed by the
 *                 packed dK/dV launch (flash_attn/attention.py:1602-1620)
 *
 * Conventions (all taken from the reference):
 *   - q is [B, H_Q, N, D]; k, v are [B, H_KV, N, D]; H_Q % H_KV == 0 and query
 *     head h reads KV head h / (H_Q / H_KV)   (attention.py:272).
 *   - Tensors are fp16 or bf16 (dtype code below) with arbitrary strides in
 *     elements, given as {stride_b, stride_h, stride_n, stride_d}; stride_d must
 *     be 1, the others multiples of 8 elements (16 bytes), pointers 16-byte
 *     aligned. Transposed views such as HF's [B, N, H, D] storage are accepted
 *     without a copy.
 *   - head_dim is 64, 128, 256 or 512 (the reference accepts powers of two up to
 *     512, docs/api.md:63); other values return GQAFA_ERR_UNSUPPORTED.
 *   - causal != 0 applies k <= q. window > 0 additionally applies q - k < window,
 *     and only when causal != 0 (attention.py:289-293, 347-356). window >= N is
 *     treated as full causal (attention.py:1442-1443).
 *   - softmax_scale multiplies Q K^T. The reference fixes it at 1/sqrt(D)
 *     (attention.py:1461); passing another value is how the HF adapter avoids
 *     pre-multiplying q (hf_integration.py:55-58).
 *   - lse is fp32 [B, H_Q, N] contiguous, natural log, including the scale
 *     (attention.py:384-388). delta is fp32 [B, H_Q, N] contiguous scratch that
 *     gqafa_bwd fills with rowsum(dO * O) (attention.py:738-742).
 *   - Outputs have the dtype of q. dq/dk/dv have the shapes of q/k/v.
 *   - Work is launched on `stream` (a cudaStream_t, NULL = legacy default) of
 *     the current CUDA device; nothing is allocated and nothing synchronises.
 *
 * Return value: GQAFA_OK, or an error code; gqafa_last_error() then returns a
 * message (thread-local).
 */
#ifndef GQA_FA_B200_H
#define GQA_FA_B200_H

#if defined(__GNUC__)
#define GQAFA_API __attribute__((visibility("default")))
#else
#define GQAFA_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define GQAFA_DTYPE_FP16 0
#define GQAFA_DTYPE_BF16 1

#define GQAFA_OK 0
#define GQAFA_ERR_INVALID 1     /* bad shape, stride, pointer or flag   */
#define GQAFA_ERR_UNSUPPORTED 2 /* valid but not implemented (head_dim) */
#define GQAFA_ERR_CUDA 3        /* a CUDA runtime / driver call failed   */

/* Forward. lse may be NULL (inference path, no LSE written). */
GQAFA_API int gqafa_fwd(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
              const void* v, const long long* v_strides, void* o, const long long* o_strides, float* lse,
              int batch, int heads_q, int heads_kv, int seqlen, int head_dim, float softmax_scale,
              int causal, int window, int dtype, void* stream);

/* Forward with a key length different from the query length (a KV cache:
 * decode or chunked prefill). q and o are [B, H_Q, seqlen_q, D], k and v
 * [B, H_KV, seqlen_k, D], lse (may be NULL) [B, H_Q, seqlen_q]. With causal
 * != 0 the queries are the last seqlen_q of the seqlen_k positions (query row
 * r sits at key position r + seqlen_k - seqlen_q, so seqlen_k >= seqlen_q is
 * required) and a window counts back from that position; without causal every
 * query sees all seqlen_k keys. Replaces the same forward launch as gqafa_fwd
 * (flash_attn/attention.py:583-603): the reference takes the key length from q
 * (attention.py:552-553) and so reads the wrong range of a longer cache; this
 * entry takes both lengths. There is no backward for seqlen_k != seqlen_q. */
GQAFA_API int gqafa_fwd_kv(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
              const void* v, const long long* v_strides, void* o, const long long* o_strides, float* lse,
              int batch, int heads_q, int heads_kv, int seqlen_q, int seqlen_k, int head_dim,
              float softmax_scale, int causal, int window, int dtype, void* stream);

/* Backward. Reads q, k, v, o, dout and lse; writes dq, dk, dv and delta. */
GQAFA_API int gqafa_bwd(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
              const void* v, const long long* v_strides, const void* o, const long long* o_strides,
              const void* dout, const long long* dout_strides, const float* lse, void* dq,
              const long long* dq_strides, void* dk, const long long* dk_strides, void* dv,
              const long long* dv_strides, float* delta, int batch, int heads_q, int heads_kv,
              int seqlen, int head_dim, float softmax_scale, int causal, int window, int dtype,
              void* stream);

/* One stage of gqafa_bwd, same arguments: stage 0 = dQ with the delta
 * prologue (replaces the dQ launch, flash_attn/attention.py:1506-1523),
 * 1 = dK and 2 = dV (together they replace the packed dK/dV launch,
 * flash_attn/attention.py:1602-1620). Stage 0 must run before 1 (dK reads
 * delta). For per-kernel timing and profiling; gqafa_bwd runs all three. */
GQAFA_API int gqafa_bwd_stage(int stage, const void* q, const long long* q_strides, const void* k,
                              const long long* k_strides, const void* v, const long long* v_strides,
                              const void* o, const long long* o_strides, const void* dout,
                              const long long* dout_strides, const float* lse, void* dq,
                              const long long* dq_strides, void* dk, const long long* dk_strides, void* dv,
                              const long long* dv_strides, float* delta, int batch, int heads_q,
                              int heads_kv, int seqlen, int head_dim, float softmax_scale, int causal,
                              int window, int dtype, void* stream);

/* gqafa_bwd without the delta argument, for callers that cannot allocate
 * device memory (an FFI binding that only holds its input and output tensors,
 * or a process whose device memory is planned up front and may not call
 * cudaMalloc). No counterpart in the reference. The delta workspace lives in
 * a fixed 4 MiB device array inside the library, which limits B * H_Q * N to
 * 1,048,576 (larger sizes return GQAFA_ERR_INVALID). The first call on a
 * device looks up the array's address, so make it before any CUDA stream
 * capture. All calls share the array: calls whose kernels overlap on the GPU
 * race on it. Allocates nothing. */
GQAFA_API int gqafa_bwd_noalloc(const void* q, const long long* q_strides, const void* k,
                                const long long* k_strides, const void* v, const long long* v_strides,
                                const void* o, const long long* o_strides, const void* dout,
                                const long long* dout_strides, const float* lse, void* dq,
                                const long long* dq_strides, void* dk, const long long* dk_strides, void* dv,
                                const long long* dv_strides, int batch, int heads_q, int heads_kv, int seqlen,
                                int head_dim, float softmax_scale, int causal, int window, int dtype,
                                void* stream);

/* Materialised backward. The reference's dK/dV launch recomputes
 * S = Q K^T and dP = dO V^T for every (key tile, query block)
 * (flash_attn/attention.py:1602-1620) after its dQ launch already computed
 * them (flash_attn/attention.py:1506-1523). gqafa_bwd_ws instead has the dQ
 * kernel also write P and dS (16-bit, the attended 128 x 256 blocks only) to a
 * caller-provided workspace and computes dK and dV from them in one kernel:
 * 10 instead of 16 head_dim-sized MACs per attended (query, key) pair, and
 * the softmax elementwise work done once. Same arguments and results as
 * gqafa_bwd, plus the workspace (256-byte aligned device memory, any
 * contents). gqafa_bwd_workspace_size returns the bytes it needs
 * (2 * B * H_Q * blocks * 64 KiB, independent of head_dim), 0 where the
 * materialised path does not apply (gqafa_bwd_ws then runs gqafa_bwd and
 * ignores the workspace), or -1 for invalid or unsupported sizes. */
GQAFA_API long long gqafa_bwd_workspace_size(int batch, int heads_q, int heads_kv, int seqlen, int head_dim,
                                             int causal, int window);
GQAFA_API int gqafa_bwd_ws(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
                           const void* v, const long long* v_strides, const void* o, const long long* o_strides,
                           const void* dout, const long long* dout_strides, const float* lse, void* dq,
                           const long long* dq_strides, void* dk, const long long* dk_strides, void* dv,
                           const long long* dv_strides, float* delta, int batch, int heads_q, int heads_kv,
                           int seqlen, int head_dim, float softmax_scale, int causal, int window, int dtype,
                           void* stream, void* workspace, long long workspace_bytes);
/* gqafa_bwd_ws (workspace non-NULL) or gqafa_bwd (workspace NULL) with dk and
 * dv written as fp32 (float, element strides as for the 16-bit tensors; dq
 * stays in the input dtype). No counterpart in the reference: for callers
 * that split the query heads of one KV group over several devices and add the
 * partial dK / dV up (the multi-GPU head split), so that the partials are not
 * rounded to 16 bits before the sum. */
GQAFA_API int gqafa_bwd_partial(const void* q, const long long* q_strides, const void* k,
                                const long long* k_strides, const void* v, const long long* v_strides,
                                const void* o, const long long* o_strides, const void* dout,
                                const long long* dout_strides, const float* lse, void* dq,
                                const long long* dq_strides, void* dk, const long long* dk_strides, void* dv,
                                const long long* dv_strides, float* delta, int batch, int heads_q, int heads_kv,
                                int seqlen, int head_dim, float softmax_scale, int causal, int window, int dtype,
                                void* stream, void* workspace, long long workspace_bytes);
/* One kernel of gqafa_bwd_ws: stage 0 = dQ + delta + P/dS, 1 = dK + dV
 * (needs stage 0's workspace contents). For per-kernel timing. */
GQAFA_API int gqafa_bwd_ws_stage(int stage, const void* q, const long long* q_strides, const void* k,
                                 const long long* k_strides, const void* v, const long long* v_strides,
                                 const void* o, const long long* o_strides, const void* dout,
                                 const long long* dout_strides, const float* lse, void* dq,
                                 const long long* dq_strides, void* dk, const long long* dk_strides, void* dv,
                                 const long long* dv_strides, float* delta, int batch, int heads_q, int heads_kv,
                                 int seqlen, int head_dim, float softmax_scale, int causal, int window, int dtype,
                                 void* stream, void* workspace, long long workspace_bytes);

/* Row-range variants for splitting one (batch, KV-group) unit across GPUs
 * by sequence blocks (no counterpart in the reference, whose launches always
 * cover every row). Same arguments as gqafa_fwd / gqafa_bwd_stage plus
 * [row_begin, row_end): row_begin a multiple of 128, row_end a multiple of 128
 * or N. gqafa_fwd_rows writes the O and LSE rows of that query range (keys:
 * all). gqafa_bwd_stage_rows stage 0 writes the dQ and delta rows of that
 * query range; stages 1 and 2 write the dK / dV rows of that key range and
 * read lse and delta of every query row, so those must be complete. */
GQAFA_API int gqafa_fwd_rows(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
                             const void* v, const long long* v_strides, void* o, const long long* o_strides,
                             float* lse, int batch, int heads_q, int heads_kv, int seqlen, int head_dim,
                             float softmax_scale, int causal, int window, int dtype, void* stream, int row_begin,
                             int row_end);
GQAFA_API int gqafa_bwd_stage_rows(int stage, const void* q, const long long* q_strides, const void* k,
                                   const long long* k_strides, const void* v, const long long* v_strides,
                                   const void* o, const long long* o_strides, const void* dout,
                                   const long long* dout_strides, const float* lse, void* dq,
                                   const long long* dq_strides, void* dk, const long long* dk_strides, void* dv,
                                   const long long* dv_strides, float* delta, int batch, int heads_q,
                                   int heads_kv, int seqlen, int head_dim, float softmax_scale, int causal,
                                   int window, int dtype, void* stream, int row_begin, int row_end);

/* ---------------------------------------------------------------------------
 * Serving from a paged KV cache held in 4 bits (no counterpart in the
 * reference). The cache is one uint8 array of num_pages pages of
 * gqafa_kv4_page_bytes bytes, 16-byte aligned; page_size (tokens of a page) is
 * 16, 32, 64, 128 or 256. Values are held as s * (c - z) in groups of 64 along
 * head_dim: a 4-bit code c each, and a scale s of 4 significant bits and a zero
 * point z in 0..15 per group (4.25 bits a value; layout in csrc/kv4_layout.cuh).
 * s * (c - z) is exact in fp16 and bf16.
 *
 * Integer arrays are int32 device memory. A request's token t lies in page
 * block_table[b][t / page_size]; a slot is page * page_size + t % page_size.
 * Lengths, tables and slots are read on the device, so a captured graph can be
 * replayed with new ones. Entries that are out of range never leave the given
 * arrays: a slot outside the cache is skipped, a page outside the pool is
 * replaced by page 0 (read as zeros by gqafa_kv4_read and by attention of many
 * rows), a length beyond the block table is clamped to it; the
 * first such entry is recorded in the status word (gqafa_device_status: 16
 * page, 17 slot, 18 length), and the results of that request are undefined.
 * Nothing is allocated and nothing synchronises.
 * ------------------------------------------------------------------------- */

/* Bytes of one page (keys and values of all heads), -1 for invalid sizes. */
GQAFA_API long long gqafa_kv4_page_bytes(int heads_kv, int head_dim, int page_size);

/* The plan of a step. Request b has kv_lens[b] cached tokens and gets
 * new_lens[b] more (0..max_new), or is finished (negative: its pages go back).
 * free_pages is a ring of num_free page ids (each in 0..num_free-1) whose live
 * part starts at free_state[0] and holds free_state[1] ids. Requests take free
 * pages in request order. A request is refused (accepted 0, nothing added)
 * when its length would pass the block table or max_new, or when the pages
 * wanted by it and the requests before it pass the free count. Pages given
 * back are written behind the live part of the ring, for later steps.
 * Outputs: block table [batch][cols] (-1 where unused), lengths after the
 * step, tokens added, slot and position of every new token [batch][max_new]
 * (-1 behind the last one), accepted, and the ring's new state. Inputs other
 * than the dead part of the ring are not written; outputs may not overlap
 * them. */
GQAFA_API int gqafa_kv4_plan(const int* kv_lens, const int* new_lens, const int* block_table, long long table_stride,
                             int* free_pages, const int* free_state, int batch, int cols, int num_free, int page_size,
                             int max_new, int* out_block_table, int* out_kv_lens, int* out_new_lens, int* out_slot_map,
                             int* out_positions, int* out_accepted, int* out_free_state, void* stream);

/* Quantise k and v [batch, heads_kv, seqlen, head_dim] into the slots of
 * slot_map [batch][seqlen] (-1: skip the token). Slots must be distinct. A
 * group of 64 values with an infinity or a NaN reads back as NaN. */
GQAFA_API int gqafa_kv4_append(const void* k, const long long* k_strides, const void* v, const long long* v_strides,
                               const int* slot_map, long long slot_stride, void* pages, long long num_pages, int batch,
                               int heads_kv, int seqlen, int head_dim, int page_size, int dtype, void* stream);

/* Cached keys and values as contiguous [batch, heads_kv, seqlen, head_dim]
 * tensors (32-byte aligned): row i of request b is position starts[b] + i
 * (starts NULL or negative: 0), zeros from kv_lens[b] on. */
GQAFA_API int gqafa_kv4_read(const void* pages, long long num_pages, const int* block_table, long long table_stride,
                             int cols, const int* kv_lens, const int* starts, void* k, void* v, int batch,
                             int heads_kv, int seqlen, int head_dim, int page_size, int dtype, void* stream);

/* Attention of q [batch, heads_q, seqlen_q, head_dim] over the cache. Request
 * b has kv_lens[b] keys; its first q_lens[b] query rows (q_lens NULL: all) are
 * the last of those positions: row r sits at kv_lens[b] - q_lens[b] + r. With
 * causal != 0 a row sees the keys up to its own position, and with window > 0
 * the last `window` of them; without causal every row sees all keys. Rows from
 * q_lens[b] on, and rows that see no key, get zeros (lse -inf). Rows that see a
 * key with a group that is not finite get NaNs (lse too); a value group that is
 * not finite makes its 64 dims NaN in the rows that see its token. lse may be
 * NULL, else fp32 [batch, heads_q, seqlen_q]. max_kv_len is an upper bound of
 * kv_lens that the host knows (0: the block table's capacity); it sizes the
 * launch and the workspace. Where a request is longer all the same, no access
 * leaves the buffers, but its rows may be wrong, and then status 18 is recorded.
 * workspace: gqafa_kv4_attend_workspace_size bytes (called with the same sizes,
 * and the same max_kv_len and window or larger ones; 0 stands for any length, a
 * window counts only with causal), 256-byte aligned, any contents, not shared by
 * calls that overlap on the GPU. Many query rows also want room for the keys and
 * values of a request in 16 bits: the size call includes it for a max_kv_len
 * above 0 (so pass cols * page_size there rather than 0, and window 0 without
 * causal); in a workspace without it they take the slower way of few rows. */
GQAFA_API long long gqafa_kv4_attend_workspace_size(int batch, int heads_q, int heads_kv, int seqlen_q, int head_dim,
                                                    int max_kv_len, int window);
GQAFA_API int gqafa_kv4_attend(const void* q, const long long* q_strides, const void* pages, long long num_pages,
                               const int* block_table, long long table_stride, int cols, const int* kv_lens,
                               const int* q_lens, void* o, const long long* o_strides, float* lse, int batch,
                               int heads_q, int heads_kv, int seqlen_q, int head_dim, int page_size, int max_kv_len,
                               float softmax_scale, int causal, int window, int dtype, void* workspace,
                               long long workspace_bytes, void* stream);

/* 1 if (head_dim, dtype) has a compiled kernel set, else 0. */
GQAFA_API int gqafa_supported(int head_dim, int dtype);

/* Message of the last failed call on this thread ("" if none). */
GQAFA_API const char* gqafa_last_error(void);

/* Synchronises `device` and returns its kernel status word (0 = every kernel
 * finished its pipeline; otherwise the code of the first bounded wait that
 * timed out). reset != 0 clears the word afterwards. Returns -1 on a CUDA
 * error. Not for the hot path. */
GQAFA_API int gqafa_device_status(int device, int reset);

/* Diagnostics, not for the hot path: point the kernels at a device buffer of
 * 9 zeroed unsigned 64-bit counters (NULL turns it off). Kernels that support
 * it (the head_dim-512 backward) then add the cycles each role spends waiting:
 * [0] producer on free ring stages, [1] MMA issuer on score operands, [2] on
 * accumulate operands, [3] on the row warps, [4] row warps on scores, [5] row
 * warps' elementwise work, [6] epilogue, [7] CTA lifetime, [8] CTA count. */
GQAFA_API int gqafa_set_wait_counters(void* device_counters);

/* Test knob (no counterpart in the reference, whose Triton kernels have no
 * bounded waits): every mbarrier wait of later launches gives up after
 * `wait_limit_cycles` clock cycles (<= 0 restores the default of 2e9, about
 * one second), and with `skip_loads` != 0 the kernels' TMA producers issue
 * nothing, so every wait runs into that bound. A timed-out launch records a
 * non-zero code in the status word (gqafa_device_status), frees its tensor
 * memory and returns; its outputs are undefined. Used by the tests of the
 * timeout path; process-wide, not for production use. */
GQAFA_API int gqafa_set_test_waits(long long wait_limit_cycles, int skip_loads);

/* Library version string. */
GQAFA_API const char* gqafa_version(void);

#ifdef __cplusplus
}
#endif
#endif /* GQA_FA_B200_H */
