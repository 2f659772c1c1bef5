/*
 * tierkv_hip.h -- C ABI of the MI355X (gfx950) tiered paged KV-cache path.
 *
 * Plain pointers and sizes only: device pointers for tensors, a hipStream_t
 * passed as void*, int status codes.  Every launch is asynchronous on the
 * given stream and never synchronises.  The library keeps no pointer past a
 * call.  Citations are file:line in xiaoMartintin/Paged_TierKV.
 *
 * Tier states: 0 HOT (fp16), 1 WARM (quantized), 2 COLD (evicted)
 * (tierkv_policy.py:14-16, csrc/block_manager.cpp:9-13).
 *
 * Pool layouts (tierkv_policy.py:122-135, 828-841):
 *   hot_k/hot_v   fp16  [hot_slots,  kv_heads, block_size, head_dim]
 *   warm_k/warm_v       [warm_slots, kv_heads, block_size, head_dim]
 *     TIERKV_WARM_REF_U8:    uint8 codes, k/v_scale and k/v_zero fp16
 *                            [warm_slots, kv_heads, block_size, 1]
 *                            (quantize_fp16_to_int8, tierkv_policy.py:21-36)
 *     TIERKV_WARM_ABSMAX_I8: int8 codes, k/v_scale fp32 [warm_slots, kv_heads],
 *                            k/v_zero unused (NULL)
 *   block_table / block_states / block_lengths: int32 [batch, table_stride],
 *     indexed by logical block; the table holds the slot of the block's
 *     state-specific pool (compact layout) or a physical id that indexes both
 *     pools (dense layout); COLD entries are never dereferenced.
 */
#ifndef TIERKV_HIP_H
#define TIERKV_HIP_H

#include <stdint.h>

#if defined(__GNUC__)
#define TIERKV_API __attribute__((visibility("default")))
#else
#define TIERKV_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes (the Python layer maps 1 -> ValueError, others -> RuntimeError). */
#define TIERKV_OK 0
#define TIERKV_ERR_INVALID 1     /* bad argument / shape */
#define TIERKV_ERR_UNSUPPORTED 2 /* configuration outside the kernels' support */
#define TIERKV_ERR_HIP 3         /* HIP launch/runtime error */
#define TIERKV_ERR_WORKSPACE 4   /* workspace too small */
#define TIERKV_ERR_STATE 5       /* BlockManager rule violation (RuntimeError) */

#define TIERKV_DTYPE_F16 0
#define TIERKV_DTYPE_BF16 1
#define TIERKV_DTYPE_F32 2 /* logits of tierkv_sample_tokens, norm weights, rows read back */

#define TIERKV_WARM_REF_U8 0
#define TIERKV_WARM_ABSMAX_I8 1

#define TIERKV_COLD_ZERO_LOGIT 0 /* reference: COLD tokens enter softmax with K=V=0 */
#define TIERKV_COLD_MASKED 1     /* COLD blocks contribute nothing */

/* Flag OR'ed into a decode call's splits_hint (whose low bits are the split
 * factor, 0 = automatic): each wave takes a fixed share of the workgroup's
 * tiles instead of taking them from a shared counter, so the attention output
 * is the same bits on every call over the same inputs, as the reference's
 * Triton kernel is.  The bits are those of the launch's wave and split counts
 * (its plan), which follow from its shape in any workspace of at least
 * tierkv_decode_workspace_bytes; in a smaller one with no room for that plan
 * they are those of one other plan, whatever the size.  Costs about 1 % of
 * the launch time (2-3 % with score sums). */
#define TIERKV_DECODE_DETERMINISTIC 0x40000000

/* Message of the last failing call on this thread ("" if none). */
TIERKV_API const char* tierkv_last_error(void);

/* Library/ABI version, for the Python loader's compatibility check. */
TIERKV_API int32_t tierkv_abi_version(void);

/* ---------------------------------------------------------------------- */
/* Decode attention.  Replaces the launch in tierkv_decode_attention
 * (tierkv_triton.py:272-465) of _tierkv_decode_attention_kernel
 * (tierkv_triton.py:45-145) and the split/reduce pair (147-264).
 *
 * query  [batch, num_heads, head_dim] (== [B, H, 1, D] contiguous), f16/bf16.
 * out    [batch, num_heads, head_dim] (== [B, 1, H, D]), same dtype as query.
 * score_sums  NULL, or fp32 [batch, num_heads, table_stride]: per (head,
 *   block) sum of softmax probabilities (tierkv_triton.py:121-145), zero for
 *   blocks >= the sequence's block count.
 * seq_num_blocks  NULL (every sequence has num_blocks blocks) or device
 *   int32 [batch] (each clamped to num_blocks).
 * workspace  device scratch of at least tierkv_decode_workspace_bytes(...)
 *   bytes, zero-filled before its first use; its first 4 bytes are an error
 *   word the kernels set non-zero when they skip a block whose slot or state
 *   is out of range.  It also holds the split-arrival counters, which every
 *   launch leaves at zero, so one workspace serves launches of any shape
 *   (and graph replays) on one stream; launches that share it must not
 *   overlap.
 * scaling  softmax scale (head_dim ** -0.5 in modeling_llama.py:315).
 * splits_hint  split factor per (sequence, kv head) (0: chosen from the
 *   launch size), optionally | TIERKV_DECODE_DETERMINISTIC.  Without the
 *   flag, tiles are handed to waves as they free up: outputs agree with the
 *   fp32 reference within tolerance but their last bits can differ between
 *   calls.  Score sums are the same bits either way.
 */
TIERKV_API int32_t tierkv_decode_attention(
    const void* query, int32_t query_dtype, void* out, float* score_sums,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths,
    int64_t table_stride, const int32_t* seq_num_blocks, int32_t num_blocks,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero,
    int32_t warm_format, int32_t cold_mode,
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim,
    float scaling, int32_t splits_hint,
    void* workspace, int64_t workspace_bytes, void* stream);

/* tierkv_decode_attention without a workspace argument and without any
 * allocation.  No counterpart in the reference: it is for callers that cannot
 * allocate device memory -- code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc.  The scratch is a 16 MiB device
 * array in the library (one copy per GPU, held until the process ends; its
 * address is taken and the array zeroed on the first call on each device,
 * with that device current, and that first call waits for the fill, so it
 * must not be under stream capture); launches that
 * cannot run in 16 MiB fail with TIERKV_ERR_WORKSPACE.
 * Every call on a GPU shares that GPU's array: calls that overlap on one GPU
 * (different streams, or host threads) race.  Blocks skipped for an
 * out-of-range slot or state set the array's error word, which
 * tierkv_decode_noalloc_error_word reads.  Arguments and results otherwise
 * as tierkv_decode_attention; the stream must belong to the current
 * device. */
TIERKV_API int32_t tierkv_decode_attention_noalloc(
    const void* query, int32_t query_dtype, void* out, float* score_sums,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths,
    int64_t table_stride, const int32_t* seq_num_blocks, int32_t num_blocks,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero,
    int32_t warm_format, int32_t cold_mode,
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim,
    float scaling, int32_t splits_hint, void* stream);

/* The error word of the current device's allocation-free scratch (bit 1: a
 * resident block with an out-of-range slot was skipped; bit 2: a state that
 * is none of HOT/WARM/COLD), 0 before the first allocation-free launch on
 * the device; cleared when clear != 0.  Synchronises the device (a copy, no
 * allocation; not under stream capture).  Accessor of
 * tierkv_decode_attention_noalloc, likewise without a counterpart in the
 * reference. */
TIERKV_API int32_t tierkv_decode_noalloc_error_word(int32_t clear, int32_t* word);

/* Workspace bytes with which tierkv_decode_attention plans freely for this
 * shape and for every shorter row.  A launch given less takes the best plan
 * that fits; it is refused only below tierkv_decode_workspace_least_bytes. */
TIERKV_API int64_t tierkv_decode_workspace_bytes(
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t num_blocks,
    int32_t block_size, int32_t head_dim, int32_t with_scores, int32_t splits_hint);

/* The fewest workspace bytes that tierkv_decode_attention accepts for this
 * shape: those of enough splits to put about 2048 waves on the chip, or of
 * the hint. */
TIERKV_API int64_t tierkv_decode_workspace_least_bytes(
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t num_blocks,
    int32_t block_size, int32_t head_dim, int32_t with_scores, int32_t splits_hint);

/* ---------------------------------------------------------------------- */
/* Demotion HOT -> WARM.  Replaces CompactTieredKVTensorPool.demote_to_warm
 * (tierkv_policy.py:1042-1068) / TieredKVTensorPool.demote_to_warm (329-361)
 * and quantize_fp16_to_int8 (21-36), batched: job i quantizes tiles
 * src_k/src_v[src_index[i]] (fp16 [kv_heads, block_size, head_dim], first
 * lengths[i] tokens) into warm slot dst_slot[i].  Jobs whose indices are out
 * of range are skipped (the Python layer validates them before launch).
 *   REF_U8: per (token, head) codes/scale/zero bit-exact with the
 *     reference's fp16 op sequence; tokens >= length are left untouched
 *     (pad_tail = 0, compact demote_to_warm) or zero-padded with scale 1 /
 *     zero 0 (pad_tail = 1, write_warm_block 989-995 / dense 350-356).
 *   ABSMAX_I8: scale = max|x| / 127 over the valid tokens of the (block,
 *     head) tile, codes rint(x / scale) clamped to [-127, 127]; tail codes 0.
 * table_pos  NULL, or int32 [n]: flat indices into block_table/block_states
 *   whose entries become (dst_slot[i], WARM) -- the _set_metadata rewrite
 *   (tierkv_policy.py:917-926); negative entries are skipped.
 */
TIERKV_API int32_t tierkv_demote_to_warm(
    const void* src_k, const void* src_v, int64_t src_tiles,
    const int32_t* src_index, const int32_t* dst_slot, const int32_t* lengths, int32_t n,
    void* warm_k, void* warm_v, int64_t warm_slots,
    void* k_scale, void* k_zero, void* v_scale, void* v_zero,
    int32_t warm_format, int32_t pad_tail,
    int32_t* block_table, int32_t* block_states, const int32_t* table_pos,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* Quantization of a prompt's blocks straight into WARM slots, without fp16
 * tiles in between: write_warm_block (tierkv_policy.py:969-1002) as
 * append_prefill_with_policy (1722-1766) calls it, batched.  Job i quantizes
 * tokens [src_tok[i], src_tok[i] + lengths[i]) of sequence src_seq[i] of the
 * fp16 sources src_k/src_v [src_seqs, kv_heads, src_tokens, head_dim] into
 * warm slot dst_slot[i], with the codecs and pad_tail of
 * tierkv_demote_to_warm.  Jobs out of range are skipped. */
TIERKV_API int32_t tierkv_quantize_tokens(
    const void* src_k, const void* src_v, int64_t src_seqs, int32_t src_tokens,
    const int32_t* src_seq, const int32_t* src_tok, const int32_t* dst_slot, const int32_t* lengths, int32_t n,
    void* warm_k, void* warm_v, int64_t warm_slots,
    void* k_scale, void* k_zero, void* v_scale, void* v_zero, int32_t warm_format, int32_t pad_tail,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* Promotion WARM -> HOT.  Replaces promote_to_hot (tierkv_policy.py:1087-1115,
 * 375-402) with dequantize_int8_to_fp16 (39-44): job i dequantizes the first
 * lengths[i] tokens of warm slot src_slot[i] into hot slot dst_slot[i]
 * (REF_U8: fp16 per-op rounding; ABSMAX_I8: fp16(fp32(q) * scale)).
 * table_pos as in tierkv_demote_to_warm, entries become (dst_slot[i], HOT). */
TIERKV_API int32_t tierkv_promote_to_hot(
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero,
    const int32_t* src_slot, const int32_t* dst_slot, const int32_t* lengths, int32_t n,
    void* hot_k, void* hot_v, int64_t hot_slots, int32_t warm_format,
    int32_t* block_table, int32_t* block_states, const int32_t* table_pos,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* ---------------------------------------------------------------------- */
/* KV append into HOT slots.  Replaces the tensor copies of write_hot_tokens
 * (tierkv_policy.py:934-967; dense pool 238-267): job i copies tokens
 * [src_tok[i], src_tok[i] + count[i]) of sequence src_seq[i] of the fp16
 * sources src_k/src_v [src_seqs, kv_heads, src_tokens, head_dim] into HOT
 * slot dst_slot[i] at rows [dst_pos[i], dst_pos[i] + count[i]); with
 * zero_tail the slot's rows past the written range are zeroed, as the
 * reference does.  Jobs whose ranges fall outside their tensors are skipped. */
TIERKV_API int32_t tierkv_write_hot_tokens(
    const void* src_k, const void* src_v, int64_t src_seqs, int32_t src_tokens,
    const int32_t* src_seq, const int32_t* src_tok, const int32_t* count,
    const int32_t* dst_slot, const int32_t* dst_pos, int32_t n, int32_t zero_tail,
    void* hot_k, void* hot_v, int64_t hot_slots,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* The same copy for at most 4 jobs given in HOST memory, jobs_host = int32
 * [n][5] = {src_seq, src_tok, count, dst_slot, dst_pos}: the jobs travel in
 * the kernel's arguments, so a decode step's single-token append needs no
 * host-to-device copy of its plan (write_hot_tokens, tierkv_policy.py:934-967,
 * as called once per layer and step by append_to_layer, 1768-1816). */
TIERKV_API int32_t tierkv_write_hot_tokens_inline(
    const void* src_k, const void* src_v, int64_t src_seqs, int32_t src_tokens, const int32_t* jobs_host, int32_t n,
    int32_t zero_tail, void* hot_k, void* hot_v, int64_t hot_slots,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* Batched runtime (one layer of B sequences whose tables live on the device).
 * Free-slot stacks: int32 [capacity] arrays whose first `top` entries are free
 * slots; ctl is int32 [4] = {hot_top, warm_top, error bits, last append
 * applied (1) or refused (0)}.  Error bits: 1 no free HOT slot, 2 no free
 * WARM slot, 4 a table row is full, 8 a sequence's last block was not HOT. */

/* Append `tokens` new tokens per sequence from src_k/src_v [batch, kv_heads,
 * tokens, head_dim] fp16 at the end of each sequence's block list: the open
 * block first (the last block, when open_blocks[b] != 0), then new HOT blocks
 * popped from hot_free in sequence order (deterministic slot ids).
 * open_blocks [batch] is 1 while the last block was left partially filled by
 * an append; a prefill sets it to 0, since the reference starts decode
 * tokens in a new block (append_prefill_with_policy resets the open block,
 * tierkv_policy.py:1764-1766).  seq_num_blocks, open_blocks and the table
 * rows are updated on the device.  All-or-nothing when slots run out.  The
 * per-step part of append_to_layer (tierkv_policy.py:1768-1816) for a batch
 * of sequences, without host involvement.  blocks_hint: the block count the
 * caller expects every sequence to hold before the append (the lockstep
 * count a decode loop tracks), or 0; with it the last blocks' entries are
 * read together with the counts (one memory round trip less).  Results do
 * not depend on it. */
TIERKV_API int32_t tierkv_runtime_append(
    const void* src_k, const void* src_v, int32_t tokens,
    int32_t* block_table, int32_t* block_states, int32_t* block_lengths, int64_t table_stride,
    int32_t* seq_num_blocks, int32_t* open_blocks, int32_t batch, int32_t blocks_hint,
    void* hot_k, void* hot_v, int64_t hot_slots, int32_t* hot_free, int32_t* ctl,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* tierkv_runtime_append with the decode step's rotary embedding fused in, for
 * fp16 models: K is rotated on its way into the pool, q is rotated into q_out
 * (contiguous fp16 [batch, num_heads, tokens, head_dim]), V is copied.  The
 * rotation is transformers' apply_rotary_pos_emb in its fp16 op order,
 * fp16(fp16(x * cos) + fp16(rotate_half(x) * sin)), so both are bit-identical
 * to it; it replaces the ~10 elementwise launches per layer that the HF hook
 * (modeling_llama.py:376-377) spends on the rotation.  q / k / v are fp16
 * [batch, heads, tokens, head_dim] with element strides (head_dim contiguous;
 * HF's projection views need no copy); cos / sin are fp16 [Bc, tokens,
 * head_dim] with strides (stride_b 0 broadcasts one row set over the batch).
 * head_dim a multiple of 16; every stride a multiple of 8 elements; every
 * pointer 16-byte aligned. */
TIERKV_API int32_t tierkv_runtime_append_rope(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t, int32_t num_heads, void* q_out,
    const void* k, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t,
    const void* v, int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t,
    const void* cos, const void* sin, int64_t cs_stride_b, int64_t cs_stride_t, int32_t tokens,
    int32_t* block_table, int32_t* block_states, int32_t* block_lengths, int64_t table_stride,
    int32_t* seq_num_blocks, int32_t* open_blocks, int32_t batch, int32_t blocks_hint,
    void* hot_k, void* hot_v, int64_t hot_slots, int32_t* hot_free, int32_t* ctl,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* One policy tick for one layer, entirely on the device: block scores from the
 * decode kernel's probability sums (block_scores_from_probability_sums,
 * tierkv_policy.py:1905-1912), stable-rank tier labels with reserved HOT
 * {0, n-1} and sticky COLD (enforce_budget mode 1 / enforce_tiered_budget
 * mode 2, 1391-1477), slot allocation (pops before pushes, in (sequence,
 * block) order) and the demote / promote data movement (sync_storage_states,
 * 1849-1867).  A migration that finds no free slot leaves its block as it is
 * and sets an error bit.  scratch: at least
 * tierkv_runtime_tick_scratch_bytes(...) bytes. */
TIERKV_API int32_t tierkv_runtime_tick(
    const float* score_sums, int64_t sums_stride, int32_t num_heads,
    int32_t* block_table, int32_t* block_states, int32_t* block_lengths, int64_t table_stride,
    const int32_t* seq_num_blocks, int32_t batch, int32_t hot_budget, int32_t warm_budget, int32_t mode,
    void* hot_k, void* hot_v, int64_t hot_slots, int32_t* hot_free,
    void* warm_k, void* warm_v, int64_t warm_slots, int32_t* warm_free,
    void* k_scale, void* k_zero, void* v_scale, void* v_zero, int32_t warm_format,
    int32_t* ctl, void* scratch, int64_t scratch_bytes, int32_t max_demotions, int32_t max_promotions,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

TIERKV_API int64_t tierkv_runtime_tick_scratch_bytes(int32_t batch, int64_t table_stride,
                                                      int32_t max_demotions, int32_t max_promotions);

/* Prefill block scores without materialising the attention probabilities.
 * Replaces compute_block_scores on the prefill attention weights
 * (tierkv_policy.py:1380-1389 via modeling_llama.py:282-292), per sequence:
 *   mass[b, blk] = sum_{h, q} sum_{t in blk} p[b, h, q, t] / (H * T) / len(blk)
 * with p the causal softmax of scaling * q . k.  q [B, H, T, D] and k
 * [B, H_kv, T, D] are fp16 or bf16 with the given element strides (head_dim
 * contiguous, strides multiples of 8, 16-byte aligned); head_dim 64 or 128,
 * GQA group <= 8, block_size a multiple of 16, T <= 32768.  mass is fp32
 * [B, ceil(T / block_size)].  One MFMA pass over K up to 4096 tokens, two
 * above; deterministic (fixed reduction order).  workspace: at least
 * tierkv_prefill_block_mass_workspace_bytes(B, H_kv, T) bytes, no
 * initialisation needed; with tierkv_prefill_block_mass_full_workspace_bytes,
 * which are twice as many for short launches of groups above four heads, those
 * run as two sets of heads side by side (another summation order; results
 * follow from the shape and from which of the two sizes is reached). */
TIERKV_API int64_t tierkv_prefill_block_mass_workspace_bytes(int32_t batch, int32_t num_kv_heads, int32_t tokens);
TIERKV_API int64_t tierkv_prefill_block_mass_full_workspace_bytes(int32_t batch, int32_t num_heads,
                                                                  int32_t num_kv_heads, int32_t tokens);
TIERKV_API int32_t tierkv_prefill_block_mass(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
    const void* k, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t, int32_t dtype,
    float* mass, int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t tokens, int32_t head_dim,
    int32_t block_size, float scaling, void* workspace, int64_t workspace_bytes, void* stream);

/* Tier telemetry without a host sync: adds one layer's per-tier block and
 * token counts over sequences b < batch and blocks i < seq_num_blocks[b] into
 * counts int64[6] = {HOT, WARM, COLD blocks, HOT, WARM, COLD tokens} on the
 * device; the caller reads them back when it wants the numbers.  The counts
 * collect_memory_metrics derives from the tables (tierkv_policy.py:1193-1317,
 * 489-654) with one `.item()` sync per counter and layer. */
TIERKV_API int32_t tierkv_tier_counts(const int32_t* block_states, const int32_t* block_lengths,
                                      int64_t table_stride, const int32_t* seq_num_blocks, int32_t batch,
                                      int64_t* counts, void* stream);

/* Table writes planned on the host: dst[pairs[2i]] = pairs[2i + 1] for
 * i < n, positions distinct, out-of-range positions skipped; pairs is an
 * 8-byte-aligned int32 device array.  Replaces the per-entry device writes of
 * _set_metadata, set_block_entry, set_block_state and sync_gpu_block_tables
 * (tierkv_policy.py:917-926, 1019-1040, 1164-1174; dense pool 269-290,
 * 450-477), which the reference issues as one launch per table entry. */
TIERKV_API int32_t tierkv_scatter_i32(int32_t* dst, int64_t dst_len, const int32_t* pairs, int32_t n,
                                      void* stream);

/* The same writes for at most 16 pairs given in HOST memory (int32 [n][2]),
 * carried in the kernel's arguments: a decode step's table update (the open
 * block's length, a new block's entries) needs no host-to-device copy. */
TIERKV_API int32_t tierkv_scatter_i32_inline(int32_t* dst, int64_t dst_len, const int32_t* pairs_host, int32_t n,
                                             void* stream);

/* One decode step of a layer in one call: the token write of
 * tierkv_write_hot_tokens_inline (n_jobs 0..4), the table writes of
 * tierkv_scatter_i32_inline (n_pairs 0..16), then tierkv_decode_attention,
 * in stream order, each validated as its own entry point validates it; every
 * check runs before the first launch, so a call that returns an argument
 * error has queued nothing.  It
 * replaces the three calls the reference's decode forward makes per layer
 * and step (append_to_layer's token write, the table update it queues, and
 * tierkv_decode_attention: modeling_llama.py:419-456, tierkv_policy.py:
 * 1768-1816, 1869-1872), so that a host-bound caller pays one C call.  The
 * fields are those of the three entry points (8-byte fields first, so the
 * layout has no interior padding); tierkv_decode_step_size() returns
 * sizeof(TierkvDecodeStep) for bindings to check theirs against. */
typedef struct TierkvDecodeStep {
  const void* src_k;        /* token write: fp16 [src_seqs, kv_heads, src_tokens, head_dim] */
  const void* src_v;
  void* hot_k;              /* HOT pools: written by the token write, read by the decode */
  void* hot_v;
  int32_t* table_dst;       /* table writes: int32 [table_len] */
  const void* query;        /* decode: as tierkv_decode_attention */
  void* out;
  float* score_sums;
  const int32_t* block_table;
  const int32_t* block_states;
  const int32_t* block_lengths;
  const int32_t* seq_num_blocks;
  const void* warm_k;
  const void* warm_v;
  const void* k_scale;
  const void* k_zero;
  const void* v_scale;
  const void* v_zero;
  void* workspace;
  int64_t src_seqs;
  int64_t hot_slots;
  int64_t table_len;
  int64_t table_stride;
  int64_t warm_slots;
  int64_t workspace_bytes;
  int32_t src_tokens;
  int32_t n_jobs;
  int32_t zero_tail;
  int32_t n_pairs;
  int32_t query_dtype;
  int32_t num_blocks;
  int32_t warm_format;
  int32_t cold_mode;
  int32_t batch;
  int32_t num_heads;
  int32_t num_kv_heads;
  int32_t block_size;
  int32_t head_dim;
  float scaling;
  int32_t splits_hint;
  int32_t jobs[4][5];       /* {src_seq, src_tok, count, dst_slot, dst_pos} */
  int32_t pairs[16][2];     /* {table index, value} */
} TierkvDecodeStep;

TIERKV_API int32_t tierkv_decode_step(const TierkvDecodeStep* step, void* stream);
TIERKV_API int64_t tierkv_decode_step_size(void);

/* ---------------------------------------------------------------------- */
/* A serving step over requests of different lengths.  The reference serves
 * one sequence per table (tierkv_policy.py:1768-1816, modeling_llama.py:
 * 419-456); these take a batch whose requests bring different numbers of new
 * tokens, packed as rows: request b's are rows [cu[b], cu[b + 1]).
 * A call may be several launches that pass state on through its workspace:
 * calls that share one go to one stream, and a host thread starts one only
 * after another thread's has returned. */

/* Table entries of the new tokens' blocks, and where each packed row goes.
 * new_tokens int32 [batch] (device) tokens per request, >= 0.  The open block
 * (open_blocks[b] != 0, last, HOT, not full) is filled first, then new HOT
 * blocks are popped from hot_free [hot_slots] in (request, block) order;
 * block_table / block_states / block_lengths [batch, table_stride],
 * seq_num_blocks, open_blocks and ctl are updated as by tierkv_runtime_append
 * (a request without new tokens keeps all of its words).  Outputs:
 *   slots     int32 [num_rows] slot * block_size + position of each row, -1
 *             for rows behind the last request
 *   positions int32 [num_rows] the row's position in its request, or -1
 *   cu_tokens int32 [batch + 1] first row of each request
 *   context   int32 [batch] tokens each request holds after the step
 * All or nothing: when the stack or a table row is too short, a length is
 * negative or there are more tokens than num_rows (error bit 16), the tables
 * stay as they are, every row is -1, cu_tokens is 0 and ctl[3] is 0.
 * batch <= 4096.  slots, positions and workspace 16-byte aligned; workspace:
 * tierkv_slot_map_workspace_bytes(batch) bytes, no initialisation needed. */
TIERKV_API int64_t tierkv_slot_map_workspace_bytes(int32_t batch);
TIERKV_API int32_t tierkv_build_slot_map(
    const int32_t* new_tokens, int32_t batch, int32_t num_rows,
    int32_t* block_table, int32_t* block_states, int32_t* block_lengths, int64_t table_stride,
    int32_t* seq_num_blocks, int32_t* open_blocks, const int32_t* hot_free, int64_t hot_slots, int32_t* ctl,
    int32_t block_size, int32_t* slots, int32_t* positions, int32_t* cu_tokens, int32_t* context,
    void* workspace, int64_t workspace_bytes, void* stream);

/* Copy packed K/V rows into HOT slots: row r of key / value [num_rows,
 * kv_heads, head_dim] (fp16 or bf16, element strides, head_dim contiguous)
 * becomes row slots[r] = slot * block_size + position of hot_k / hot_v, in
 * fp16 (bf16 values past its range become infinities).  Rows whose slot is
 * negative or outside the pool are skipped; slots that are written are
 * distinct.  write_hot_tokens (tierkv_policy.py:934-967) by rows. */
TIERKV_API int32_t tierkv_write_slots(
    const void* key, int64_t k_stride_t, int64_t k_stride_h, const void* value, int64_t v_stride_t, int64_t v_stride_h,
    int32_t dtype, const int32_t* slots, int32_t num_rows, void* hot_k, void* hot_v, int64_t hot_slots,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* Per-head norms and rotation by position of packed query and key rows, and
 * the write of keys and values into HOT slots, in one pass.  Row r stands at
 * positions[r] of its context (tierkv_build_slot_map gives them).  For each
 * head of q (with q_weight) and of k (with k_weight; NULL: no norm)
 *   x' = x * rsqrt(mean(x^2) + eps) * weight,
 * then the pairs (a, b) of the first rotary_dim dims, (i, i + rotary_dim / 2)
 * or (2 i, 2 i + 1) when interleaved, turn by the angle positions[r] * inv_freq[i]
 * (formed in 64 bits) and are scaled by attention_scaling; the other dims pass.
 *   q  [num_rows, num_heads, head_dim], k / v [num_rows, num_kv_heads, head_dim],
 *      fp16 or bf16, element strides, head_dim contiguous; weights [head_dim],
 *      in that dtype or fp32; inv_freq fp32 [rotary_dim / 2], rotary_dim even
 *   q_out, k_out  contiguous rows of the same dtype (k_out may be NULL where
 *      the keys go to pools); they do not overlap the inputs
 *   slots NULL (then value and pools are NULL), or the pool row slot *
 *      block_size + position of each row: k rotated and v as it is are written
 *      there in fp16, as tierkv_write_slots does; negative and outside ones
 *      are skipped, those written are distinct
 * Rows whose position is negative are left out: nothing of them is written.
 * 32-bit arithmetic, one rounding.  apply_rotary_pos_emb and write_hot_tokens
 * (modeling_llama.py:376-377, tierkv_policy.py:934-967) by rows; the norms
 * have no counterpart in the reference.  head_dim up to 256, fewer than 2^26
 * rows. */
TIERKV_API int32_t tierkv_rotate_rows(
    const void* query, int64_t q_stride_t, int64_t q_stride_h, void* q_out,
    const void* key, int64_t k_stride_t, int64_t k_stride_h, void* k_out,
    const void* value, int64_t v_stride_t, int64_t v_stride_h, int32_t dtype,
    const int32_t* positions, int32_t num_rows,
    const float* inv_freq, int32_t rotary_dim, int32_t interleaved, float attention_scaling,
    const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps,
    const int32_t* slots, void* hot_k, void* hot_v, int64_t hot_slots,
    int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* Packed K/V rows quantized into WARM slots as a step writes them: row r of
 * key / value (as tierkv_write_slots takes them; bf16 rows become fp16 first)
 * becomes row slots[r] = slot * block_size + position of warm_k / warm_v.
 * Rows whose slot is negative or outside the pool are skipped; slots that are
 * written are distinct.
 *   REF_U8: each (row, head) by itself, the codes, scale and zero point of
 *     tierkv_demote_to_warm.
 *   ABSMAX_I8: a block's rows are consecutive in the call, with no skipped row
 *     among them (what a block's rows in several places of one call give is
 *     not defined).  With p the lowest
 *     position written of a block and s its scale (0 where p = 0, a block that
 *     starts anew), the scale becomes s' = max(|s|, max|x| / 127) of the rows
 *     written; the rows before p, which the block holds, become rint(code * s /
 *     s') and those written rint(x / s').  Every other row of the block holds
 *     nothing afterwards.  Each growth rounds held codes again, by up to half
 *     a step of the scale then: in a block of b tokens filled one by one, the
 *     values of position p end within (b - p) / 2 steps of the last scale.
 * write_warm_block (tierkv_policy.py:969-1002) by rows.  head_dim up to 256. */
TIERKV_API int32_t tierkv_quantize_rows(
    const void* key, int64_t k_stride_t, int64_t k_stride_h, const void* value, int64_t v_stride_t, int64_t v_stride_h,
    int32_t dtype, const int32_t* slots, int32_t num_rows,
    void* warm_k, void* warm_v, int64_t warm_slots,
    void* k_scale, void* k_zero, void* v_scale, void* v_zero, int32_t warm_format,
    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* Tokens of a tiered cache read back as packed rows.  Request b's rows
 * [cu_tokens[b], cu_tokens[b + 1]) of out_k / out_v [num_rows, num_kv_heads,
 * head_dim] (fp16, bf16 or fp32) become its tokens of ordinal start[b] (0 when
 * negative), start[b] + 1, ... over the valid tokens of its blocks: HOT as
 * they are, WARM as code * scale (ABSMAX_I8) or (code - zero) * scale (REF_U8)
 * in 32 bits, rounded once; tokens of evicted blocks, of blocks whose slot is
 * out of range, and past what the request holds are 0.  Rows of no request
 * are not written.  reconstruct_layer (tierkv_policy.py:1818-1841) for a
 * batch.  head_dim up to 256, block_size up to 64, batch up to 65535. */
TIERKV_API int32_t tierkv_read_rows(
    const int32_t* start, const int32_t* cu_tokens, int32_t num_rows,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths, int64_t table_stride,
    const int32_t* seq_num_blocks, int32_t num_blocks,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero, int32_t warm_format,
    void* out_k, void* out_v, int32_t out_dtype,
    int32_t batch, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, void* stream);

/* Attention of several query tokens per request over the tiered cache.
 * Request b's query rows [cu_tokens[b], cu_tokens[b + 1]) are the last n_b of
 * the L_b tokens that its row of the tables holds (valid tokens of all blocks
 * below its block count, evicted ones included); row i sees the tokens up to
 * its own, ordinals 0 .. L_b - n_b + i, with the tiers, WARM formats and COLD
 * modes of tierkv_decode_attention.  A row that sees nothing becomes 0; rows
 * of out behind the last request are not written.
 *   query  [num_rows, num_heads, head_dim], fp16 / bf16, element strides that
 *          are multiples of 8, head_dim contiguous, 16-byte aligned
 *   out    [num_rows, num_heads, head_dim] contiguous, the query's dtype
 *   max_tokens  an upper bound of the requests' new tokens (num_rows will do):
 *          with it small calls launch less.  Of a request that brings more, or
 *          whose range ends past num_rows, the first max_tokens rows that
 *          there are see what they see in any case, the others are not
 *          written, and bit 4 of the error word is set (nothing is launched,
 *          and no bit set, when max_tokens or num_rows is 0)
 * head_dim a multiple of 8 up to 128, block_size up to 64, any GQA group.
 * Probabilities and WARM values are rounded to fp16 once (WARM values past its
 * range become infinite); logits, statistics and sums are 32-bit.
 * The same inputs give the same bits on every call.  workspace: as
 * tierkv_decode_attention's (one buffer may serve both, in stream order), at
 * least tierkv_extend_workspace_bytes(...) bytes, zero-filled before its
 * first use; the error word is set as there when a block is skipped, and to 4
 * when rows are not computed (max_tokens, or packed ranges that overlap). */
TIERKV_API int64_t tierkv_extend_workspace_bytes(int32_t batch, int32_t num_rows, int32_t max_tokens,
                                                 int32_t num_heads, int32_t num_kv_heads, int32_t num_blocks,
                                                 int32_t block_size, int32_t head_dim);
TIERKV_API int32_t tierkv_extend_attention(
    const void* query, int64_t q_stride_t, int64_t q_stride_h, int32_t query_dtype, void* out,
    const int32_t* cu_tokens, int32_t num_rows, int32_t max_tokens,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths, int64_t table_stride,
    const int32_t* seq_num_blocks, int32_t num_blocks,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero,
    int32_t warm_format, int32_t cold_mode,
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, float scaling,
    void* workspace, int64_t workspace_bytes, void* stream);

/* tierkv_extend_attention for requests that share prefixes, each prefix read
 * once for the rows of all its requests.  Every row of request b sees all
 * tokens of prefix prefix_of[b] (a row of the prefix tables; negative, or not
 * below num_prefixes: none), then the request's own tokens as there.
 *   prefix_of  int32 [batch] (device), requests of a prefix in any order
 *   prefix_table / prefix_states / prefix_lengths  int32 [num_prefixes,
 *      prefix_stride], of the same pools, with prefix_num_blocks (NULL: all
 *      num_prefix_blocks of them) as seq_num_blocks; blocks may also be in
 *      requests' tables, and a prefix may have no request
 * batch + num_prefixes <= 4096; where max_tokens is 512 rows per kv head or
 * more, prefix and own tables together hold fewer than 2^31 tokens.  The
 * prefix adds no position of its own: the keys are in the cache with the
 * positions that they were rotated by.
 * workspace: as there, tierkv_prefix_workspace_bytes(...) bytes of these
 * sizes (-1 for sizes that no call takes; fewer rows may take more, since
 * their tables are cut into more parts; a max_tokens of up to 64 rows per kv
 * head takes at most twice what a larger one does).  absmax values enter the
 * products exactly, code * 2^e with the rest of the scale on the
 * probabilities; other roundings, arguments, limits and errors as there.  The
 * same inputs give the same bits. */
TIERKV_API int64_t tierkv_prefix_workspace_bytes(int32_t batch, int32_t num_prefixes, int32_t num_rows,
                                                 int32_t max_tokens, int32_t num_heads, int32_t num_kv_heads,
                                                 int32_t num_blocks, int32_t num_prefix_blocks, int32_t block_size,
                                                 int32_t head_dim);
TIERKV_API int32_t tierkv_prefix_attention(
    const void* query, int64_t q_stride_t, int64_t q_stride_h, int32_t query_dtype, void* out,
    const int32_t* cu_tokens, int32_t num_rows, int32_t max_tokens,
    const int32_t* block_table, const int32_t* block_states, const int32_t* block_lengths, int64_t table_stride,
    const int32_t* seq_num_blocks, int32_t num_blocks,
    const int32_t* prefix_of, const int32_t* prefix_table, const int32_t* prefix_states, const int32_t* prefix_lengths,
    int64_t prefix_stride, const int32_t* prefix_num_blocks, int32_t num_prefix_blocks, int32_t num_prefixes,
    const void* hot_k, const void* hot_v, int64_t hot_slots,
    const void* warm_k, const void* warm_v, int64_t warm_slots,
    const void* k_scale, const void* k_zero, const void* v_scale, const void* v_zero,
    int32_t warm_format, int32_t cold_mode,
    int32_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t block_size, int32_t head_dim, float scaling,
    void* workspace, int64_t workspace_bytes, void* stream);

/* Next tokens from logits [batch, vocab] (fp16, bf16 or fp32, rows
 * row_stride elements apart) and one random number in [0, 1) per row.
 * Weights are whole numbers W_i = rint(2^42 exp((x_i - max x) / T)), 0 for
 * -inf and NaN.  Of the tokens in the order (logit descending, index
 * ascending): the first top_k (off when <= 0); of these those whose sum of
 * weights before them is below top_p times their total, one at least (off
 * when >= 1); of these those with W_i >= 2^42 min(min_p, 1).  tokens[b] is
 * the smallest index whose running sum of what is left, in index order,
 * exceeds floor(uniforms[b] * total); probs (or NULL) gets W / total.
 * temperature <= 0 (or NaN) takes the first of the largest logits, with
 * probability 1; a row with no logit above -inf gives token -1, probability
 * 0.  Each limit is a device array [batch] or, where that is NULL, one value
 * for all rows.  vocab <= 2^20, batch <= 65536.  The same inputs give the
 * same tokens on every call.  workspace: tierkv_sample_workspace_bytes(batch,
 * vocab) bytes, 16-byte aligned, of which the first
 * TIERKV_SAMPLE_COUNTER_BYTES are zero before the first call; every call
 * leaves them so, and one workspace serves calls of any shape on one stream. */
#define TIERKV_SAMPLE_COUNTER_BYTES 524288
TIERKV_API int64_t tierkv_sample_workspace_bytes(int32_t batch, int32_t vocab);
TIERKV_API int32_t tierkv_sample_tokens(
    const void* logits, int32_t dtype, int64_t row_stride, int32_t batch, int32_t vocab, const float* uniforms,
    const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
    const float* top_p, float top_p_all, const float* min_p, float min_p_all,
    int64_t* tokens, float* probs, void* workspace, int64_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------- */
/* Block scores.  Per-block probability mass from softmax probabilities
 * probs fp32 [batch, num_heads, tokens] -> out fp32 [batch, tokens/block_size]:
 * sequential sum over heads, pairwise tree over the block's tokens, / heads,
 * / max(len, 1).  lengths NULL (full blocks) or int32 [batch, n_blocks].
 * The quantity of compute_block_scores (tierkv_policy.py:1380-1389) and
 * block_scores_from_probability_sums (1905-1912) for a batch of sequences. */
TIERKV_API int32_t tierkv_block_mass_from_probs(
    const float* probs, const int32_t* lengths, float* out,
    int32_t batch, int32_t num_heads, int32_t tokens, int32_t block_size, void* stream);

/* block_scores_from_probability_sums (tierkv_policy.py:1905-1912), batched:
 * score_sums fp32 [batch, num_heads, sums_stride], lengths int32
 * [batch, len_stride] -> out fp32 [batch, num_blocks]. */
TIERKV_API int32_t tierkv_block_scores_from_sums(
    const float* score_sums, int64_t sums_stride, const int32_t* lengths, int64_t len_stride,
    float* out, int32_t batch, int32_t num_heads, int32_t num_blocks, void* stream);

/* Tier labels.  TierKVPolicyEngine.enforce_tiered_budget (mode 2,
 * tierkv_policy.py:1434-1477) and enforce_budget (mode 1 with
 * demoted_state, 1391-1432) for a batch of sequences: reserved HOT
 * {0, n-1}, stable descending rank of the remaining scores, COLD sticky.
 * mode 0 (hot_only) copies cur_states.  scores fp32 [batch, n]; cur_states
 * and new_states int32 [batch, states_stride]. */
TIERKV_API int32_t tierkv_tier_labels(
    const float* scores, const int32_t* cur_states, int32_t* new_states, int64_t states_stride,
    int32_t batch, int32_t num_blocks, int32_t hot_budget, int32_t warm_budget,
    int32_t mode, int32_t demoted_state, void* stream);

/* ---------------------------------------------------------------------- */
/* BlockManager (host).  Replaces the pybind11 class of
 * csrc/block_manager.cpp:22-134 with identical allocation order and errors:
 * TIERKV_ERR_STATE carries the reference's message in tierkv_last_error(). */
typedef struct tierkv_block_manager tierkv_block_manager;

TIERKV_API int32_t tierkv_bm_create(int32_t total_blocks, tierkv_block_manager** out);   /* :24-34 */
TIERKV_API void tierkv_bm_destroy(tierkv_block_manager* bm);
TIERKV_API int32_t tierkv_bm_allocate_block(tierkv_block_manager* bm, int32_t seq_id, int32_t* physical_idx); /* :36-49 */
TIERKV_API int32_t tierkv_bm_free_sequence(tierkv_block_manager* bm, int32_t seq_id);   /* :51-62 */
TIERKV_API int32_t tierkv_bm_update_block_state(tierkv_block_manager* bm, int32_t seq_id,
                                     int32_t logical_id, int32_t state);     /* :64-77 */
/* Batched state write for logical ids [0, n) (a device policy tick's result);
 * same checks as update_block_state, applied to every entry before any write. */
TIERKV_API int32_t tierkv_bm_set_block_states(tierkv_block_manager* bm, int32_t seq_id,
                                   const int32_t* states, int32_t n);
TIERKV_API int32_t tierkv_bm_num_blocks(const tierkv_block_manager* bm, int32_t seq_id, int32_t* n);
/* Copy up to capacity entries; *n receives the full count (:79-105). */
TIERKV_API int32_t tierkv_bm_get_physical_indices(const tierkv_block_manager* bm, int32_t seq_id,
                                       int32_t* out, int32_t capacity, int32_t* n);
TIERKV_API int32_t tierkv_bm_get_states(const tierkv_block_manager* bm, int32_t seq_id,
                             int32_t* out, int32_t capacity, int32_t* n);
TIERKV_API int32_t tierkv_bm_num_free(const tierkv_block_manager* bm, int32_t* n);

#ifdef __cplusplus
}
#endif

#endif /* TIERKV_HIP_H */
