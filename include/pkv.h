/*
 * pkv.h — C ABI of the MI355X (gfx950) PersistentKV paged decode-attention engine.
 *
 * Every entry point takes plain device pointers, sizes and a HIP stream passed as
 * `void*` (a hipStream_t; NULL selects the null stream).  Outputs, the split workspace
 * and the merge counters are owned by the caller, exactly as in the reference op surface,
 * and the library allocates no device memory.  A direct launch (num_splits == 1) of fewer
 * than 128 (row, kv head) pairs splits itself internally when the caller's workspace can
 * hold the partial states (pkv_direct_workspace_bytes gives the size for the full split;
 * a smaller or empty workspace gives a smaller split or the single launch, with the same
 * result to fp32 rounding; PKV_DIRECT_SPLIT=0 in the environment turns this off).  Calls
 * enqueue work asynchronously and never synchronise the host.
 * Errors are reported as a pkv_status code; a one-line message describing the last
 * failure on the calling thread is available from pkv_last_error().
 *
 * Layouts (all row-major, contiguous):
 *   q / q_source   [rows, num_q_heads, 128]                   fp16 or bf16
 *   k_pages/v_pages[num_pages, num_kv_heads, page_size, 128]  same dtype as q (fp8 e4m3
 *                                                             for the *_fp8 entries)
 *   block_table    [batch, max_pages]                         int32 physical page ids
 *   seq_lens       [batch]                                    int32 tokens per row
 *   output         [out_rows, num_q_heads, 128]               same dtype as q
 *   work_items     [num_tasks, 5] int32 = {row, kv_head, split, tile_begin, tile_end}
 *                  (tiles are 32-token units, independent of page_size)
 *   split_offsets  [batch + 1]                                int32 prefix sum of row splits
 *   merge_counters [batch, num_kv_heads]                      int32, zero on entry and exit
 *   workspace      fp32 [m: n][l: n][acc: n x 128] with n = batch*num_q_heads*num_splits
 *                  (grid split) or total_partial_slots*num_q_heads (work queue),
 *                  16-byte aligned (as any torch allocation is; others are rejected).
 *
 * Query head h reads KV head h / G with G = num_q_heads / num_kv_heads.  The softmax
 * scale is fixed at 1/sqrt(128).  G may be any integer in [1, 32]; the reference accepts
 * only {1, 2, 4, 8}.  Reference citations are into ahmed123hds/persistentkv-attention.
 */
#ifndef PKV_H_
#define PKV_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PKV_HEAD_DIM 128     /* kernels/persistentkv_attention.cuh:26 (PKV_D) */
#define PKV_TILE_TOKENS 32   /* kernels/persistentkv_attention.cuh:28 (PKV_TILE) */
#define PKV_MAX_GROUP 32     /* largest supported Hq / Hkv */

typedef enum pkv_status {
  PKV_OK = 0,
  PKV_ERR_INVALID_ARGUMENT = 1,  /* a shape, pointer or size is inconsistent */
  PKV_ERR_UNSUPPORTED = 2,       /* a valid request this build does not implement */
  PKV_ERR_WORKSPACE_TOO_SMALL = 3,
  PKV_ERR_LAUNCH = 4,            /* the HIP runtime rejected a kernel launch */
  PKV_ERR_CAPACITY = 5           /* a host builder output buffer is too small */
} pkv_status;

typedef enum pkv_dtype { PKV_DTYPE_F16 = 0, PKV_DTYPE_BF16 = 1 } pkv_dtype;

/* Text of the most recent error on this thread ("" when none). */
const char* pkv_last_error(void);
/* Static name of a status code. */
const char* pkv_status_string(int status);
/* Library version as major*10000 + minor*100 + patch. */
int pkv_version(void);

/* ---------------------------------------------------------------------------------
 * Workspace sizing.
 * ------------------------------------------------------------------------------- */

/* Bytes of split workspace for the grid-split ops; 0 when num_splits <= 1.
 * Replaces persistentkv_workspace_bytes, kernels/persistentkv_attention.cuh:891-898. */
size_t pkv_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_splits);

/* Bytes of workspace for the work-queue op (total_partial_slots partial states per head).
 * Replaces persistentkv_partition_workqueue_workspace sizing, cuh:915-927. */
size_t pkv_workqueue_workspace_bytes(int32_t total_partial_slots, int32_t num_q_heads);

/* Bytes of workspace with which a direct launch (num_splits == 1) of the grid ops and of
 * pkv_attention_contiguous runs its full internal split: about 256 units of work for a
 * batch of few (row, kv head) pairs, whose partial states are merged by a second launch.
 * 0 when that launch is not split.  The reference's direct path takes no workspace
 * (cuh:929-946); this entry has no counterpart there. */
size_t pkv_direct_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                  int32_t context);

/* Bytes of workspace with which a split launch (num_splits > 1) of the grid ops and of
 * pkv_attention_contiguous runs its full internal sub-split: a launch of fewer
 * batch * num_kv_heads * num_splits units than about 3/4 of the CUs cuts each split into
 * sub-splits, to about one unit per CU (at least 2 tiles of 32 tokens each), merged
 * together.  pkv_workspace_bytes(batch, num_q_heads, num_splits) when the launch is not
 * sub-split; with that size (the reference's) the partial states keep the reference's
 * layout; sizes in between give fewer sub-splits, with the same result to fp32 rounding
 * (PKV_SPLIT_SUBDIVIDE=0 in the environment turns this off).  No counterpart in the
 * reference, whose split launches use exactly the caller's split (cuh:947-974). */
size_t pkv_split_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                 int32_t context, int32_t num_splits);

/* ---------------------------------------------------------------------------------
 * The four ops.  Argument order follows the torch op surface of
 * tests/persistentkv_torch_extension.cu, with the tensor shapes spelled out.
 * ------------------------------------------------------------------------------- */

/* Every row attends to exactly `context` tokens.
 * Replaces persistentkv_paged_attention (tests/persistentkv_torch_extension.cu:35-93)
 * and persistentkv_paged_dispatch (kernels/persistentkv_attention.cuh:1114-1136). */
int pkv_paged_attention(
    const void* q, const void* k_pages, const void* v_pages,
    const int32_t* block_table, void* output,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t context, int32_t num_splits, int32_t dtype, void* stream);

/* Row b attends to seq_lens[b] tokens; bucket_context bounds num_splits.
 * Replaces persistentkv_paged_attention_masked (extension.cu:95-157) and
 * persistentkv_paged_masked_dispatch (cuh:1138-1161). */
int pkv_paged_attention_masked(
    const void* q, const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens, void* output,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t num_splits, int32_t dtype, void* stream);

/* Row b reads query row q_indices[b] of q_source and writes output row out_indices[b].
 * Replaces persistentkv_paged_attention_indexed (extension.cu:159-228) and
 * persistentkv_paged_masked_indexed_dispatch (cuh:1163-1189). */
int pkv_paged_attention_indexed(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t num_splits, int32_t dtype, void* stream);

/* Compact work queue: one partial state per work item, then a segmented LSE merge
 * (or, with fused_merge != 0, the last work item of each (row, kv head) merges).
 * Replaces persistentkv_paged_attention_workqueue (extension.cu:230-317) and
 * persistentkv_paged_workqueue_indexed_dispatch (cuh:1191-1261).
 * Work-queue contract (the reference's, cuh:294-363, :648-716, :753-784):
 * - item (row, kvh, split, tile_begin, tile_end) writes the state of its own 32-token
 *   tile range into slot split_offsets[row] + split; a negative bound stands for the
 *   row-local split bound (cuh:330-337); a range without tiles writes the neutral state;
 *   items with row, kvh, split or slot out of range are ignored;
 * - row b's output folds the slots [split_offsets[b], split_offsets[b + 1]): every slot
 *   when num_tasks >= num_kv_heads x (split_offsets[batch] - split_offsets[0]) (a queue
 *   that writes each slot once, the queues on which the reference reads no unwritten
 *   memory); otherwise the slots of splits whose row-local range is empty are skipped
 *   (the builder's queues emit no item for them, and the reference then merges
 *   uninitialised memory);
 * - the fused merge waits for one arrival per slot in the first case (the reference's
 *   row_splits arrivals, cuh:659) and one per non-empty split in the second, and also
 *   merges rows of one slot (which the reference leaves unwritten). */
int pkv_paged_attention_workqueue(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, int32_t* merge_counters,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, int32_t fused_merge,
    int32_t dtype, void* stream);

/* pkv_paged_attention_workqueue without the workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid allocation).  It has no counterpart in the reference.  The partial states
 * go to a 16 MiB static scratch array in the library's code object (one per GPU, held
 * until the process ends); the call allocates nothing.  It returns
 * PKV_ERR_WORKSPACE_TOO_SMALL when pkv_workqueue_workspace_bytes(total_partial_slots,
 * num_q_heads) exceeds 16 MiB.  Every call on one GPU shares that GPU's scratch: calls
 * that overlap on one GPU (on other streams, or graph replays running at the same time)
 * race and give wrong results.  The scratch's address is taken on the calling thread's
 * current HIP device, which must be the device of `stream`.  Same results, bit for bit, as
 * pkv_paged_attention_workqueue with a workspace of exactly
 * pkv_workqueue_workspace_bytes(total_partial_slots, num_q_heads) bytes (the same
 * schedule, see pkv_workqueue_schedule). */
int pkv_paged_attention_workqueue_noalloc(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, int32_t* merge_counters,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, int32_t fused_merge,
    int32_t dtype, void* stream);

/* Which schedule pkv_paged_attention_workqueue (and its fp8 and append variants) runs
 * for these sizes on the current device: 1 = the balanced schedule, 0 = one workgroup per
 * work item.  The balanced schedule streams every (row, kv head) pair's tiles [0, T) with
 * an equal share per wave (2 waves per CU, 4 with fp8 K/V) and merges the pieces; it
 * applies when fused_merge == 0, G = num_q_heads / num_kv_heads <= 16, page_size is a
 * multiple of 16, batch <= 256 and the workspace holds
 * pkv_workqueue_balanced_workspace_bytes (one threshold for every K/V dtype).
 * Streaming [0, T) is the reference's result for the queue pkv_build_workqueue (the
 * reference's compile_persistentkv_metadata) builds.  The decode checks on the device that
 * the caller's queue is exactly that one; for any other queue the merge stage computes
 * each (row, kv head) pair from the items' own tile ranges instead (slower), so both
 * schedules give the reference's result, to fp32 rounding, on every queue that writes
 * each slot once, and the builder's result on the builder's queues.  No counterpart in
 * the reference. */
int pkv_workqueue_schedule(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                           int32_t page_size, size_t workspace_bytes, int32_t fused_merge);

/* Workspace bytes the balanced schedule needs on the current device, sized for its
 * largest wave count (4 per CU): the partial states,
 * (batch * num_kv_heads + 4 * CUs) * (num_q_heads / num_kv_heads) rounded up to even,
 * times 130 * 4 bytes, then a 16-byte plan entry per (row, kv head) pair (the waves that
 * hold the pair's tiles, written by the decode stage for the merge stage), then 4 bytes
 * per CU (each decode workgroup's part of the queue check); 0 for sizes it never takes
 * (G > 16 or batch > 256).  A complete queue's reference-sized workspace
 * (pkv_workqueue_workspace_bytes) often holds it already (C4: 2.66 MB against 2.26 MB).
 * No counterpart in the reference. */
size_t pkv_workqueue_balanced_workspace_bytes(int32_t batch, int32_t num_q_heads,
                                              int32_t num_kv_heads);

/* One stage of pkv_paged_attention_workqueue (fused_merge == 0), in whichever schedule
 * pkv_workqueue_schedule names: stage 1 = the decode kernel, 2 = the merge.  Stage 1 then
 * stage 2 on one stream equal the combined call bit for bit; they exist for per-kernel
 * timing and for callers that overlap the merge with other work.  Both stages take the
 * same arguments, the same workspace and workspace_bytes in particular (they choose the
 * schedule and where its partial states and plan lie): stage 2 folds what the last stage
 * 1 wrote into that workspace, so another step's stage 1 in between changes its result.
 * kv_fp8 != 0 selects the fp8 K/V pages of pkv_paged_attention_workqueue_fp8 with
 * k_scale / v_scale.  The reference launches both from one host function
 * (cuh:1005-1017); it has no separate entry points. */
int pkv_paged_attention_workqueue_stage(
    int32_t stage, const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, int32_t kv_fp8, float k_scale,
    float v_scale, int32_t dtype, void* stream);

/* The two stages of the per-item schedule of pkv_paged_attention_workqueue with
 * fused_merge == 0 (one workgroup per work item, partial states in the reference's slot
 * format (split_offsets[b] + s) * Hq + qh), callable on their own.  Running decode then
 * merge on one stream equals the combined call when it takes the per-item schedule
 * (pkv_workqueue_schedule == 0).  The reference launches both from one host function
 * (cuh:1005-1017); it has no separate entry points. */
int pkv_workqueue_decode(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, const int32_t* q_indices,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, int32_t dtype, void* stream);

/* num_tasks and num_kv_heads are the queue's item count and Hkv.  When num_tasks >=
 * num_kv_heads x (split_offsets[batch] - split_offsets[0]) (a queue that writes every
 * slot) the merge folds every slot of a row, as the reference's does (cuh:766-780);
 * otherwise (the builder's queues, whose splits without tiles emit no item) it skips the
 * slots whose row-local bounds are empty.  num_tasks < 0 selects the second rule. */
int pkv_workqueue_merge(
    const int32_t* seq_lens, const int32_t* split_offsets, const int32_t* out_indices,
    void* output, int32_t out_rows,
    const void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t total_partial_slots,
    int32_t num_tasks, int32_t num_kv_heads, int32_t dtype, void* stream);

/* ---------------------------------------------------------------------------------
 * fp8 K/V: the same ops over K and V pages of OCP fp8 e4m3 (1 byte per element, same
 * [num_pages, num_kv_heads, page_size, 128] layout) dequantised with per-tensor scales,
 * K = k_scale * k8 and V = v_scale * v8.  q / output keep `dtype` (fp16 or bf16).
 * page_size must be a multiple of 16; k_scale must be positive and finite.  The
 * reference names fp8 / dequantising paged decode as future work
 * (paper/persistentkv_mlsys_workshop.tex:688-690); these entries have no counterpart
 * in its code and follow the signatures of the 2-byte ops they extend.
 * ------------------------------------------------------------------------------- */

/* pkv_paged_attention_indexed with fp8 K/V. */
int pkv_paged_attention_indexed_fp8(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t num_splits, float k_scale, float v_scale,
    int32_t dtype, void* stream);

/* pkv_paged_attention_workqueue with fp8 K/V. */
int pkv_paged_attention_workqueue_fp8(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, int32_t* merge_counters,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, int32_t fused_merge,
    float k_scale, float v_scale, int32_t dtype, void* stream);

/* pkv_workqueue_decode with fp8 K/V (stage 1 only; pkv_workqueue_merge is unchanged). */
int pkv_workqueue_decode_fp8(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, const int32_t* q_indices,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, float k_scale, float v_scale,
    int32_t dtype, void* stream);

/* ---------------------------------------------------------------------------------
 * From a prompt to the cache, and decode over block-scaled fp8.  No counterpart in the
 * reference, whose harness builds its metadata on the host and starts from filled pools.
 * Token-major inputs (q, k, v, k_new, v_new) are [tokens, heads, 128] with a stride between
 * tokens in elements (a multiple of 8, at least heads * 128), so that the column ranges of
 * one fused projection's output need no copy; their heads lie next to one another.  Tensors
 * are 16-byte aligned.
 * ------------------------------------------------------------------------------- */

/* The metadata of one step, from lengths on the GPU.  Row b holds cached_lens[b] tokens, and
 * seq_lens[b] after the step (a row that shrinks takes no tokens and keeps its pages until
 * cached_lens goes down too: those behind it are then the caller's to return; negative lengths
 * count as 0):
 *   token_offsets [batch + 1]  where row b's new tokens start in packed order, and their count
 *   block_table   [batch, max_pages]  the pages that row b needs beyond the
 *                 ceil(cached / page_size) it has are entered, taken in row order from the
 *                 end of the list free_pages[0, num_free); other entries stay as they are
 *   slot_mapping  [slots]  page * page_size + offset of every new token in packed order; -1
 *                 for tokens past the table or without a page, and behind the last token
 *   num_free_out  [1]  num_free less the pages taken; negative when that many were missing
 *                 (the entries concerned are -1).  It must not be num_free: the inputs
 *                 stay as they are, and a repeated call gives the same result.
 * A step with a negative num_free_out must not be used: tokens without a page have no slot, and
 * the entries of -1 would count as pages held once cached_lens has moved on.  With cached_lens
 * and num_free as they were, and pages returned to the list or rows left out (seq_lens =
 * cached_lens), the same call builds it again.
 * num_free [1] counts as clamped to [0, free_capacity].  At most 8000 rows, and 2^31 - 1 new
 * tokens.  Pages are returned by pkv_free_rows, or where no row was ever forked by the caller, who
 * copies entries to the end of free_pages; a page that other rows hold must not go there. */
int pkv_build_block_tables(
    const int32_t* cached_lens, const int32_t* seq_lens, const int32_t* free_pages,
    const int32_t* num_free, int32_t* block_table, int32_t* token_offsets, int32_t* slot_mapping,
    int32_t* num_free_out, int32_t batch, int32_t free_capacity, int32_t max_pages, int32_t slots,
    int32_t page_size, void* stream);

/* Causal attention over whole prompts: sequence b is the tokens [token_offsets[b],
 * token_offsets[b + 1]) of q [tokens, num_q_heads, 128] and of k, v [tokens, num_kv_heads,
 * 128]; its token i attends to its tokens 0 ... i.  output [tokens, num_q_heads, 128],
 * contiguous; rows outside every sequence are left as they are.  It may be q itself if q is
 * contiguous too (q_stride = num_q_heads * 128, or one token); otherwise it must not overlap q,
 * and never k or v (refused).  Offsets must not decrease and count as clamped to [0, tokens].
 * G = num_q_heads / num_kv_heads in [1, 32]; (tokens * G / 128 + batch) * num_kv_heads must be
 * below 2^24.  An infinity or NaN in K or V reaches the tokens from its own on, and no other (a
 * key of score -inf has weight 0).  K and V of the call are all that is attended to: tokens that
 * the cache holds already are not, so a row that continues a cached prefix (cached_lens > 0 in
 * pkv_build_block_tables) must not go in for its new tokens alone (pkv_paged_prefill_attention
 * is for those). */
int pkv_prefill_attention(
    const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
    int64_t v_stride, const int32_t* token_offsets, void* output, int32_t batch, int32_t tokens,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype, void* stream);

/* Writes k_new[t] and v_new[t] ([num_kv_heads, 128], dtype f16 or bf16) to slot
 * slot_mapping[t] (page * page_size + offset) of the pools [num_pages, num_kv_heads,
 * page_size, 128] of the same dtype.  Slots outside the pools are skipped; a slot may occur
 * only once in a call.  tokens * num_kv_heads must be below 2^28. */
int pkv_write_kv(const void* k_new, int64_t k_stride, const void* v_new, int64_t v_stride,
                 void* k_pages, void* v_pages, const int32_t* slot_mapping, int32_t tokens,
                 int32_t num_kv_heads, int32_t head_dim, int32_t num_pages, int32_t page_size,
                 int32_t dtype, void* stream);

/* pkv_write_kv into fp8 (OCP e4m3) pools with kv_scales [num_pages, num_kv_heads, 2] (K's
 * scale, V's scale; 8-byte aligned).  Scales are powers of two in [2^-60, 2^60], the smallest
 * with amax <= 448 scale over the finite values the block receives; elements are stored as
 * e4m3(clamp(x / scale, -448, 448)), rounded to nearest even, NaN as NaN.  An infinity is so
 * stored as 448 scale: the largest value that its block can hold, and 448 * 2^-60 where all of
 * the block's finite values are zero.  A page whose first
 * written offset is 0 starts anew.  Otherwise the tokens before it stay: the scale is at
 * least the old one (rounded up to a power of two), and where it grows, those tokens are
 * stored again under it (exact but for subnormals).  The tokens of one page must follow one
 * another in slot_mapping, each in the slot behind its predecessor's, without gaps; a call that
 * breaks this (slots 5 and 7 of a page, a page's tokens in two places, a slot twice) leaves the
 * pages concerned with unspecified values. */
int pkv_write_kv_fp8_block(const void* k_new, int64_t k_stride, const void* v_new,
                           int64_t v_stride, void* k_pages, void* v_pages, float* kv_scales,
                           const int32_t* slot_mapping, int32_t tokens, int32_t num_kv_heads,
                           int32_t head_dim, int32_t num_pages, int32_t page_size, int32_t dtype,
                           void* stream);

/* pkv_paged_attention_masked over such pools: K = kv_scales[p, h, 0] * k8 and
 * V = kv_scales[p, h, 1] * v8 for every page p and KV head h.  Scales count as clamped to
 * [2^-60, 2^60] (NaN as the lower end) and need not be powers of two.  page_size must be a
 * multiple of 16; rows of length 0 give zeros; lengths are clamped to the table, page ids
 * into the pool.  At most 16000 rows, and fewer than 2^24 output rows (batch * num_q_heads).
 * The workspace is required:
 * pkv_fp8_block_workspace_bytes on the same device, for any lengths; it holds nothing
 * between calls, and calls that may overlap need one each.  output may be q itself, but must not
 * overlap it otherwise (refused). */
int pkv_paged_attention_fp8_block(
    const void* q, const void* k_pages, const void* v_pages, const float* kv_scales,
    const int32_t* block_table, const int32_t* seq_lens, void* output, void* workspace,
    size_t workspace_size, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t num_pages, int32_t page_size, int32_t max_pages, int32_t dtype,
    void* stream);
size_t pkv_fp8_block_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads);

/* ---------------------------------------------------------------------------------
 * A further turn over rows that are cached.  No counterpart in the reference.
 * ------------------------------------------------------------------------------- */

/* The norm of every head of q [tokens, num_q_heads, 128] and k [tokens, num_kv_heads, 128] and its
 * rotation by position, in 32 bits, rounded once:
 *   y = x * (mean(x^2) + eps)^(-1/2) * weight       (weight null: y = x)
 *   a' = a cos - b sin,  b' = b cos + a sin          for the pairs (a, b) of the first rotary_dim dims
 * Pairs are dims (i, i + rotary_dim / 2), or with `interleaved` (2 i, 2 i + 1).  Weights are fp32
 * [128] (*_weight_heads = 1) or one row a head ([heads, 128], *_weight_heads = heads).  cos_sin is
 * fp32 [max_positions, rotary_dim]: the cosines of the rotary_dim / 2 angles, then their sines.
 * rotary_dim is a multiple of 16 up to 128, eps (where a weight is given) in [2^-100, 2^100].
 * positions [tokens] count as clamped to the table.  An output is its own input (same pointer and
 * stride), or overlaps neither the inputs nor the other output (refused).  Strides between tokens
 * as for the token-major inputs above, the outputs' too. */
int pkv_norm_rope(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                  const float* q_weight, int32_t q_weight_heads, const float* k_weight,
                  int32_t k_weight_heads, const float* cos_sin, const int32_t* positions, void* q_out,
                  int64_t q_out_stride, void* k_out, int64_t k_out_stride, int32_t tokens,
                  int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim,
                  int32_t max_positions, int32_t interleaved, float eps, int32_t dtype, void* stream);

/* pkv_norm_rope and pkv_write_kv in one pass: k goes, normed and rotated, and v, as it is, to slot
 * slot_mapping[t] of the pools (which no other tensor of the call may overlap); slots outside them
 * are skipped, and a slot may occur only once.  q_out as above. */
int pkv_norm_rope_write_kv(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                           const void* v, int64_t v_stride, const float* q_weight,
                           int32_t q_weight_heads, const float* k_weight, int32_t k_weight_heads,
                           const float* cos_sin, const int32_t* positions, void* q_out,
                           int64_t q_out_stride, void* k_pages, void* v_pages,
                           const int32_t* slot_mapping, int32_t tokens, int32_t num_q_heads,
                           int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim,
                           int32_t max_positions, int32_t interleaved, float eps, int32_t num_pages,
                           int32_t page_size, int32_t dtype, void* stream);

/* Pages that several rows hold.  page_shares [num_pages] counts the holders of a page beyond the
 * first: 0 for a page that one row holds and for a free one, so pages that pkv_build_block_tables
 * hands out need nothing done.  All zero at the start; only these three operators write it.  What one
 * of the three writes, its workspace among it, must not overlap another tensor of its call (refused).
 *
 * Forks: row children[i] of the table becomes a copy of row parents[i], for i < num_forks (at most
 * 8000).  Of the parent's lens[parent] tokens, full pages are shared (entries copied, page_shares one
 * more); a part-filled last page is the child's own: taken from the end of the list free_pages[0,
 * num_free) in the order of i, entered in its table row, and named in copy_src[i], copy_dst[i]
 * (the parent's page and the child's; -1, -1 where there is none) for pkv_copy_pages, once for every
 * layer's pools.  num_free_out is num_free less the pages taken; negative when that many were
 * missing: then nothing else is written but -1 to the copy lists, and the call can be repeated.  Such
 * a count must not become num_free, which is still the list's, nor may the children get lengths.
 * Lengths are the caller's: the children's are set by it.  A child's row must hold no pages (its entries
 * are written over, not returned).  Pairs whose rows are outside the table,
 * or the same, are skipped; a row must not be a child twice, nor a child and a parent in one call
 * (unspecified entries and counts, nothing outside the tables).  num_free counts as clamped to [0,
 * free_capacity], lengths to the table.  num_free_out must not be num_free. */
int pkv_fork_rows(const int32_t* parents, const int32_t* children, const int32_t* lens,
                  int32_t* block_table, int32_t* page_shares, const int32_t* free_pages,
                  const int32_t* num_free, int32_t* num_free_out, int32_t* copy_src, int32_t* copy_dst,
                  int32_t num_forks, int32_t batch, int32_t max_pages, int32_t num_pages,
                  int32_t free_capacity, int32_t page_size, void* stream);

/* Rows that end: every page that holds tokens of the rows `rows` [num_rows] (at most 8000) loses one
 * holder, and pages that had no other go, in ascending order, to free_pages[num_free] and behind;
 * num_free_out is the new count.  A row listed twice counts once; rows outside the table are
 * skipped.  Table and lengths stay as they are (the caller sets the rows' lengths to 0).  The list
 * must have a place for every page (free_capacity >= num_pages).  The workspace, of
 * pkv_page_workspace_bytes(num_pages), holds nothing between calls; calls that may overlap need one
 * each, and must not share lists. */
int pkv_free_rows(const int32_t* rows, const int32_t* lens, const int32_t* block_table,
                  int32_t* page_shares, int32_t* free_pages, const int32_t* num_free,
                  int32_t* num_free_out, void* workspace, size_t workspace_size, int32_t num_rows,
                  int32_t batch, int32_t max_pages, int32_t num_pages, int32_t free_capacity,
                  int32_t page_size, void* stream);

/* Pages moved to the front of the pool, so that those in use (the ones that free_pages[0, num_free)
 * does not name; U of them) are 0 ... U - 1 and the rest can be given back.  A page below U stays; the
 * used page of the highest id goes to the lowest free id, and so on:
 *   page_map [num_pages]        every used page's new id; -1 for free ones
 *   block_table_out             the table [batch, max_pages] with its ids mapped (free pages' as -1;
 *                               entries that are no ids stay); it alone may be its input, block_table itself
 *   page_shares_out             the counts at the new ids, 0 behind; not page_shares itself
 *   free_pages_out              num_pages - 1 down to U, so that the lowest is taken first (it and
 *                               free_pages have free_capacity >= num_pages places; not free_pages itself)
 *   num_free_out [1]            num_pages - U; not num_free itself
 *   copy_src, copy_dst          [num_copies >= num_pages / 2] the moves, for pkv_copy_pages, once for
 *                               every layer's pools; -1 behind them
 * The inputs stay as they are but where the table is said to be its own output.  Workspace as above. */
int pkv_compact_pages(const int32_t* block_table, const int32_t* page_shares, const int32_t* free_pages,
                      const int32_t* num_free, int32_t* page_map, int32_t* block_table_out,
                      int32_t* page_shares_out, int32_t* free_pages_out, int32_t* num_free_out,
                      int32_t* copy_src, int32_t* copy_dst, void* workspace, size_t workspace_size,
                      int32_t batch, int32_t max_pages, int32_t num_pages, int32_t free_capacity,
                      int32_t num_copies, void* stream);
size_t pkv_page_workspace_bytes(int32_t num_pages);

/* Page copy_dst[i] of the pools [num_pages, num_kv_heads, page_size, 128] (elements of 1 or 2 bytes)
 * becomes page copy_src[i], and its kv_scales [num_pages, num_kv_heads, 2] too (or null).  Entries
 * that are not ids of the pool, and copies of a page to itself, are skipped.  No page may be written
 * twice, nor written and read, in one call. */
int pkv_copy_pages(const int32_t* copy_src, const int32_t* copy_dst, void* k_pages, void* v_pages,
                   float* kv_scales, int32_t num_copies, int32_t num_pages, int32_t num_kv_heads,
                   int32_t page_size, int32_t head_dim, int32_t element_bytes, void* stream);

/* Attention of the newest tokens of every row over its pages, which hold them already (2-byte
 * pools).  Row b has seq_lens[b] tokens; the n of the call are q's tokens [token_offsets[b],
 * token_offsets[b + 1]), at positions seq_lens[b] - n ... seq_lens[b] - 1, and each attends to the
 * row's tokens up to its own: a second turn over a cached prefix, a piece of a prompt, one token,
 * or none.  A token at a negative position (more new tokens than the row has) sees nothing: 0.
 * output [tokens, num_q_heads, 128], contiguous; rows outside every sequence are left as they are;
 * it may be a contiguous q itself, otherwise it must not overlap q (refused), nor the pools.  Any
 * page_size; G = num_q_heads / num_kv_heads in [1, 32].  Tokens past the table are not attended to
 * (positions are those of seq_lens as given; negative lengths count as 0), page ids count as clamped
 * into the pool, offsets (which must not decrease) to [0, tokens].  Page slots past a row's length are
 * not read.  An infinity or NaN in K or V reaches the tokens that see its key, and no other.
 * (tokens * G / 128 + batch) * num_kv_heads must be below 2^24 less ten for every compute unit of
 * the GPU and five for every KV head.  The workspace is required: pkv_paged_prefill_workspace_bytes on the
 * same device, for any lengths (with 256 compute units up to 199 MB, from tokens * G = 128 on, and 17 MB
 * up to tokens * G = 32); it holds nothing between calls, and calls that may overlap need one each. */
int pkv_paged_prefill_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages,
                                const int32_t* block_table, const int32_t* seq_lens,
                                const int32_t* token_offsets, void* output, void* workspace,
                                size_t workspace_size, int32_t batch, int32_t tokens, int32_t num_q_heads,
                                int32_t num_kv_heads, int32_t head_dim, int32_t num_pages,
                                int32_t page_size, int32_t max_pages, int32_t dtype, void* stream);
size_t pkv_paged_prefill_workspace_bytes(int32_t batch, int32_t tokens, int32_t num_q_heads, int32_t num_kv_heads);

/* ---------------------------------------------------------------------------------
 * Contiguous-layout decode: K and V are [batch, num_kv_heads, context, 128] (every row
 * holds `context` tokens) and q / output are [batch, num_q_heads, 128].
 * ------------------------------------------------------------------------------- */

/* GQA decode over contiguous K/V, unsplit (num_splits == 1, no workspace) or split
 * (workspace of pkv_workspace_bytes(batch, num_q_heads, num_splits) bytes).
 * Replaces persistentkv_dispatch (cuh:1077-1090) and persistentkv_split_dispatch
 * (cuh:1092-1108) over PkvContiguousAccessor (cuh:128-178). */
int pkv_attention_contiguous(
    const void* q, const void* k, const void* v, void* output,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t context,
    int32_t head_dim, int32_t num_splits, int32_t dtype, void* stream);

/* Query-head baseline: each query head streams its KV head on its own, so every K/V
 * byte is read G times (the redundant GQA traffic the grouped path removes).  Same
 * output as pkv_attention_contiguous.  Replaces persistentkv_baseline_dispatch
 * (cuh:1263-1282) and pkv_query_head_baseline_kernel (cuh:786-889). */
int pkv_attention_query_head_baseline(
    const void* q, const void* k, const void* v, void* output,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t context,
    int32_t head_dim, int32_t dtype, void* stream);

/* ---------------------------------------------------------------------------------
 * Host scheduling: split policy, cost model and compact work-queue builder.
 * Pure host code (no GPU needed).  "Reference" mode reproduces
 * tests/benchmark_serving_trace.py bit for bit; "mi355x" mode is re-tuned for 256 CUs.
 * ------------------------------------------------------------------------------- */

typedef enum pkv_policy { PKV_POLICY_REFERENCE = 0, PKV_POLICY_MI355X = 1 } pkv_policy;

typedef enum pkv_route {
  PKV_ROUTE_FLASHINFER = 0,   /* the reference's fallback route (reference policy only;
                                 this engine has no such route) */
  PKV_ROUTE_BUCKET = 1,       /* length-bucket split grid (paged_attention_indexed); with
                                 1 split, the direct launch */
  PKV_ROUTE_WORKQUEUE = 2     /* compact work queue (paged_attention_workqueue) */
} pkv_route;

/* Constants of the roofline cost model (benchmark_serving_trace.py:33-43). */
typedef struct pkv_cost_model {
  int32_t num_q_heads;        /* HQ */
  int32_t num_kv_heads;       /* HKV */
  int32_t head_dim;           /* DIM */
  int32_t compute_units;      /* SM_COUNT */
  double read_gbps;           /* ROOFLINE_READ_GBPS */
  double launch_overhead_us;  /* LAUNCH_OVERHEAD_US */
  double min_ctas_per_cu;     /* MIN_CTAS_PER_SM */
  int32_t supported_group;    /* SUPPORTED_PERSISTENTKV_GQA; 0 accepts every G */
  int32_t min_long_context;   /* 16384 in the reference's adaptive gate (:457) */
  int32_t policy;             /* pkv_policy used for the split choices */
  /* MI355X policy only (no counterpart in the reference's model): fixed costs of this
   * engine's launches, fitted to measured step times (profiles/cost_model_calibration.json,
   * persistentkv-attention_amd/pkv_calibrate.py). */
  double unit_round_us;       /* per round of two workgroups per CU of a split grid */
  double grid_merge_us;       /* a split grid's merge kernel */
  double queue_merge_us;      /* the work queue's merge kernel (balanced schedule) */
} pkv_cost_model;

/* Fills *model with the reference constants (RTX 3060) or the MI355X constants. */
void pkv_cost_model_preset(int32_t policy, pkv_cost_model* model);

/* choose_workqueue_row_splits, benchmark_serving_trace.py:370-393. */
int32_t pkv_choose_workqueue_row_splits(
    int32_t length, int32_t active_count, int32_t requested_splits,
    int32_t auto_splits, int32_t num_kv_heads, int32_t policy);

/* choose_splits, benchmark_serving_trace.py:328-367. */
int32_t pkv_choose_splits(
    const int32_t* lengths, int32_t count, int32_t requested_splits,
    int32_t auto_splits, int32_t single_bucket, int32_t num_kv_heads, int32_t policy);

/* model_bucket_splits / model_workqueue_splits, benchmark_serving_trace.py:396-415. */
int32_t pkv_model_bucket_splits(
    const int32_t* lengths, int32_t count, int32_t num_kv_heads, int32_t policy);
int32_t pkv_model_workqueue_splits(
    const int32_t* lengths, int32_t count, int32_t num_kv_heads, int32_t policy);

/* estimate_route_ms, benchmark_serving_trace.py:418-442.  `lengths` are the active
 * rows' current lengths. */
double pkv_estimate_route_ms(
    const int32_t* lengths, int32_t count, int32_t route, int32_t splits,
    const pkv_cost_model* model);

/* choose_adaptive_route_cost_model, benchmark_serving_trace.py:445-488.  Returns the
 * chosen pkv_route and writes its split count and estimate.  With model->policy ==
 * PKV_POLICY_MI355X it never returns PKV_ROUTE_FLASHINFER: every step, for any G, length
 * and active count, goes to the cheaper of PKV_ROUTE_BUCKET (splits from
 * pkv_model_bucket_splits, priced as one ragged grid launch plus its merge) and
 * PKV_ROUTE_WORKQUEUE (splits from pkv_model_workqueue_splits). */
int32_t pkv_choose_adaptive_route(
    const int32_t* lengths, int32_t count, const pkv_cost_model* model,
    int32_t* out_splits, double* out_estimated_ms);

/* Sizes the compact work queue for one decode step without building it.  num_q_heads
 * only matters for PKV_POLICY_MI355X, whose item size depends on the kernel that
 * G = num_q_heads / num_kv_heads selects; the reference policy ignores it. */
int pkv_workqueue_size(
    const int32_t* lengths, int32_t count, int32_t requested_splits,
    int32_t auto_splits, int32_t num_q_heads, int32_t num_kv_heads, int32_t policy,
    int32_t* out_num_tasks, int32_t* out_total_partial_slots);

/* Builds one decode step's work-queue metadata, bit-exact with the work-queue branch of
 * compile_persistentkv_metadata (benchmark_serving_trace.py:668-729).
 *   lengths[count], request_ids[count]: the active rows in step order.
 *   page_indptr[count+1], page_ids[]: each active row's reserved physical pages (CSR).
 * Outputs (host buffers):
 *   block_table[count * table_cols]: row r = its first ceil(max_len/page_size) pages,
 *     padded with its last reserved page; *out_table_cols receives the width.
 *   seq_lens[count], q_indices[count] (= request_ids), out_indices[count] (= r),
 *   work_items[5 * work_capacity], split_offsets[count + 1].
 * Returns PKV_ERR_CAPACITY (with the needed sizes written) when a buffer is too small. */
int pkv_build_workqueue(
    const int32_t* lengths, const int32_t* request_ids, int32_t count,
    const int32_t* page_indptr, const int32_t* page_ids,
    int32_t page_size, int32_t requested_splits, int32_t auto_splits,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t policy,
    int32_t* block_table, int32_t table_capacity, int32_t* out_table_cols,
    int32_t* seq_lens, int32_t* q_indices, int32_t* out_indices,
    int32_t* work_items, int32_t work_capacity, int32_t* out_num_tasks,
    int32_t* split_offsets, int32_t* out_total_partial_slots);

/* round_bucket_length, benchmark_serving_trace.py:316-321: `length` rounded up to a
 * multiple of bucket_tokens, then to a multiple of page_size (at least one page), capped
 * at the row's allocated_pages * page_size; `length` itself when bucket_tokens <= 0. */
int32_t pkv_round_bucket_length(int32_t length, int32_t bucket_tokens, int32_t allocated_pages,
                                int32_t page_size);

/* use_single_bucket_for_state, benchmark_serving_trace.py:491-504: 1 when the step's rows
 * go through one ragged bucket (requested, or adaptive with at least max(3, count - 1)
 * distinct lengths among count > 1 rows). */
int32_t pkv_use_single_bucket(const int32_t* lengths, int32_t count,
                              int32_t requested_single_bucket, int32_t adaptive_route);

/* Builds one decode step's length-bucket metadata, bit-exact with the bucket branch of
 * compile_persistentkv_metadata (benchmark_serving_trace.py:731-780): rows grouped by
 * pkv_round_bucket_length of their length (one bucket of max(lengths) when
 * pkv_use_single_bucket), buckets in order of first appearance, rows of a bucket in step
 * order.  Bucket j (j < *out_bucket_count <= count) holds bucket_rows[j] rows, which are
 * entries [sum of earlier bucket_rows, + bucket_rows[j]) of seq_lens (the row's length),
 * q_indices (its request id) and out_indices (its position in the step), and one
 * [bucket_rows[j], bucket_table_cols[j] = ceil(bucket_lengths[j] / page_size)] block
 * table, stored after the earlier buckets' tables in `tables`, each row its first
 * reserved pages padded with its last one.  bucket_splits[j] is choose_splits over the
 * bucket's lengths (pkv_choose_splits with `policy`).  Every bucket is one
 * pkv_paged_attention_indexed launch with bucket_context = bucket_lengths[j] (:986-1000).
 * Returns PKV_ERR_CAPACITY with *out_table_elems set when `tables` is too small. */
int pkv_build_buckets(const int32_t* lengths, const int32_t* request_ids, int32_t count,
                      const int32_t* page_indptr, const int32_t* page_ids, int32_t page_size,
                      int32_t requested_splits, int32_t auto_splits, int32_t bucket_tokens,
                      int32_t single_bucket, int32_t adaptive_route, int32_t num_kv_heads,
                      int32_t policy, int32_t* out_bucket_count, int32_t* bucket_lengths,
                      int32_t* bucket_rows, int32_t* bucket_splits, int32_t* bucket_table_cols,
                      int32_t* seq_lens, int32_t* q_indices, int32_t* out_indices,
                      int32_t* tables, int64_t table_capacity, int64_t* out_table_elems);

/* ---------------------------------------------------------------------------------
 * KV-cache append: the write of each row's newest token before its decode step.
 * No counterpart in the reference, whose harness grows the lengths without writing K/V
 * (tests/benchmark_serving_trace.py:285-298); fused KV-cache writes are future work in
 * paper/persistentkv_mlsys_workshop.tex:689.
 * ------------------------------------------------------------------------------- */

/* Writes k_new[b] and v_new[b] ([num_kv_heads, 128] each, dtype f16 or bf16, batch rows)
 * into the pools ([num_pages, num_kv_heads, page_size, 128], same dtype) at token position
 * seq_lens[b] - 1: page block_table[b * max_pages + pos / page_size], slot
 * pos % page_size.  Rows with seq_lens[b] <= 0, a position past the table, or a page id
 * outside [0, num_pages) are skipped.  Asynchronous on `stream`. */
int pkv_append_kv(const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                  const int32_t* block_table, const int32_t* seq_lens, int32_t batch,
                  int32_t num_kv_heads, int32_t head_dim, int32_t num_pages, int32_t page_size,
                  int32_t max_pages, int32_t dtype, void* stream);

/* pkv_append_kv into fp8 (OCP e4m3) pools: each element is stored as
 * e4m3(clamp(x / scale, -448, 448)), rounded to nearest even (torch's float8_e4m3fn cast),
 * with k_scale for K and v_scale for V.  `dtype` is that of k_new and v_new. */
int pkv_append_kv_fp8(const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                      const int32_t* block_table, const int32_t* seq_lens, int32_t batch,
                      int32_t num_kv_heads, int32_t head_dim, int32_t num_pages,
                      int32_t page_size, int32_t max_pages, float k_scale, float v_scale,
                      int32_t dtype, void* stream);

/* Decode with the append fused in: the result and the pools afterwards equal
 * pkv_append_kv(k_new, v_new, ...) followed by the op without the suffix, in one decode
 * launch.  The newest token of each row (position seq_lens[b] - 1) is read from k_new /
 * v_new ([batch, num_kv_heads, 128], `dtype`) by the waves whose tiles hold it (one, or one
 * of each workgroup that shares the unit's output dims), one of which also writes it into
 * the pools.  Page sizes that are not multiples of 16 run pkv_append_kv first on the same
 * stream.  (fp8 pools: the *_fp8_append entries below.)  A row's tail slot must not be read
 * through another (row, position) of the same step (no two rows share a tail page, as
 * in any copy-on-write cache).  No counterpart in the reference (see pkv_append_kv). */
int pkv_paged_attention_masked_append(
    const void* q, const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens, void* output,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t num_splits, const void* k_new, const void* v_new,
    int32_t dtype, void* stream);

int pkv_paged_attention_indexed_append(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t num_splits, const void* k_new, const void* v_new,
    int32_t dtype, void* stream);

/* pkv_paged_attention_workqueue with the append fused in (as above). */
int pkv_paged_attention_workqueue_append(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, int32_t* merge_counters,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, int32_t fused_merge,
    const void* k_new, const void* v_new, int32_t dtype, void* stream);

/* The fp8-K/V ops with the append: k_new / v_new are in `dtype` and stored as
 * pkv_append_kv_fp8 stores them, e4m3(clamp(x / k_scale)) and e4m3(clamp(x / v_scale)).
 * Same result as pkv_append_kv_fp8 followed by the fp8 op.  That is also what they run, two
 * launches in stream order, in the indexed op and in the work-queue op's per-item schedule.
 * In its balanced schedule (pkv_workqueue_schedule names the schedule of a call: it follows
 * from the workspace size, fused_merge, G, page_size and batch) the decode writes the tokens
 * itself, and a row's tail slot must not be read through another (row, position) of the
 * same step, as above: of two rows that share a tail page, each may then read the other's
 * slot before or after it is written.  Callers with shared tail pages run pkv_append_kv_fp8
 * and the op without the suffix.  v_scale must be positive. */
int pkv_paged_attention_indexed_fp8_append(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t num_splits, float k_scale, float v_scale,
    const void* k_new, const void* v_new, int32_t dtype, void* stream);

int pkv_paged_attention_workqueue_fp8_append(
    const void* q_source, int32_t q_rows,
    const void* k_pages, const void* v_pages,
    const int32_t* block_table, const int32_t* seq_lens,
    const int32_t* work_items, int32_t num_tasks,
    const int32_t* split_offsets, int32_t* merge_counters,
    const int32_t* q_indices, const int32_t* out_indices,
    void* output, int32_t out_rows,
    void* workspace, size_t workspace_bytes,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t num_pages, int32_t page_size, int32_t max_pages,
    int32_t bucket_context, int32_t total_partial_slots, int32_t fused_merge,
    float k_scale, float v_scale, const void* k_new, const void* v_new,
    int32_t dtype, void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* PKV_H_ */
