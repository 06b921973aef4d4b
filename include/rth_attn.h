/*
 * C ABI of the MI355X attention hot path (libruntherder_attn.so).
 *
 * Every entry point takes plain device pointers, host int sizes and a HIP
 * stream passed as void* (NULL = the null stream), enqueues its work
 * asynchronously, never synchronizes and never allocates, so calls are
 * HIP-graph capturable. Return value: RTH_OK, or an error code with a message
 * available from rth_last_error_string() (thread-local).
 *
 * Element types at the boundary:
 *   bf16  -> uint16_t (raw bfloat16 bits)
 *   E4M3  -> uint8_t  (OCP FP8 E4M3FN: bias 7, max 448, 0x7F/0xFF NaN)
 *
 * Layouts follow the reference engine (reference paths):
 *   q, out   [n_new, num_q_heads, head_dim] bf16           (backend.h:31-41)
 *   k, v     [max_seq_len, num_kv_heads, head_dim] E4M3   (kv_view.h:7-13)
 *   k_scale, v_scale [max_seq_len, num_kv_heads] fp32, one dequant scale per
 *            (token, kv_head); value = float(code) * scale  (kv_view.h:7-13)
 *   cache_len / at_pos are DEVICE-resident ints, unchecked against the cache
 *   size (the caller owns that bound), as in the reference.
 */
#ifndef RTH_ATTN_H
#define RTH_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    RTH_OK              = 0,
    RTH_ERR_INVALID_ARG = 1, /* argument check failed (message says which) */
    RTH_ERR_HIP         = 2, /* HIP runtime / launch error */
};

/* Message of the last failing call on this thread ("" if none). */
const char* rth_last_error_string(void);

/* Replaces kernels::quantize_kv_fp8 (reference
 * include/runtherder/kernels/quantization.cuh:50-57). Per row of head_dim bf16:
 * scale = amax/448, q = E4M3_satfinite(x * (448/amax)); row r is written at
 * destination row r + (*at_pos) * rows_per_pos. head_dim % 8 == 0,
 * 8 <= head_dim <= 16384. Bit-exact with the reference's arithmetic. */
int rth_kv_quantize_fp8(uint8_t* q, float* scale, const uint16_t* x,
                        const int* at_pos, int rows_per_pos, int num_rows,
                        int head_dim, void* stream);

/* Given-scale variant (no reference counterpart): scale[dst] is an input and
 * q = E4M3_satfinite(x * (1/scale[dst])). Used to fill caches whose scales are
 * set by the caller (e.g. per-head calibration). Same constraints. */
int rth_kv_quantize_fp8_scaled(uint8_t* q, const float* scale,
                               const uint16_t* x, const int* at_pos,
                               int rows_per_pos, int num_rows, int head_dim,
                               void* stream);

/* Replaces the two quantize_kv_fp8 launches of engine::KVCache::append
 * (reference include/runtherder/engine/kv_cache.h:62-78) with one launch:
 * quantizes k and v ([n_new, num_kv_heads, head_dim] bf16) into one layer's
 * slabs at rows *at_pos .. *at_pos + n_new - 1. */
int rth_kv_append_fp8(uint8_t* k_cache, uint8_t* v_cache, float* k_scale,
                      float* v_scale, const uint16_t* k, const uint16_t* v,
                      const int* at_pos, int n_new, int num_kv_heads,
                      int head_dim, void* stream);

/* Replaces kernels::flash_split_scratch_floats (reference
 * include/runtherder/kernels/flash_decode.cuh:16-24): floats of decode
 * scratch for max_splits splits, Hq*S*2 + Hq*S*D, laid out as [Hq*S] m,
 * [Hq*S] l, [Hq*S*D] acc like the reference's. No initialization needed. */
size_t rth_split_scratch_floats(int num_q_heads, int head_dim, int max_splits);

/* Split count AdaptiveAttention uses on `device` for num_kv_heads kv heads:
 * the decode kernel runs one wave per (kv head, split) unit, eight per
 * compute unit, so this is 8 * CUs / num_kv_heads (256 for 8 kv heads on
 * MI355X), capped at 1024. */
int rth_default_num_splits(int num_kv_heads, int device);

/* Replaces kernels::flash_decode_split_bf16 (reference
 * include/runtherder/kernels/flash_decode.cuh:45-59): one query token,
 * attends *cache_len + 1 keys, split-K over num_splits key ranges with a
 * log-sum-exp merge (two kernels: splits, then merge). `partial` is
 * caller-owned scratch of rth_split_scratch_floats(Hq, D, num_splits) floats.
 * head_dim in {32,64,128,256,512}; 64/128/256 run the MFMA split kernel when
 * the group of G = Hq/Hkv q heads splits into equal blocks of 4..16 heads
 * (G itself when G <= 16) with block * head_dim <= 2048, the rest the VALU
 * split kernel (rth_decode_path). */
int rth_attn_decode_split(uint16_t* out, const uint16_t* q, const uint8_t* k,
                          const uint8_t* v, const float* k_scale,
                          const float* v_scale, float* partial, int num_splits,
                          const int* cache_len, int num_q_heads,
                          int num_kv_heads, int head_dim, float scale,
                          void* stream);

enum {
    RTH_DECODE_MFMA = 1, /* bf16 MFMA split kernel */
    RTH_DECODE_VALU = 2, /* VALU split kernel (DPP / shuffle reductions) */
};

/* No counterpart in the reference: which split kernel rth_attn_decode_split,
 * rth_attn_decode_split_noalloc and rth_attn_decode_append_split run for this
 * shape (RTH_DECODE_MFMA or RTH_DECODE_VALU), 0 if the shape is not
 * supported; it follows rth_set_decode_kernel. The paged, RoPE and q/k-norm
 * entries always run the MFMA kernel and accept the shapes this reports as
 * RTH_DECODE_MFMA under the automatic choice (path 0), whatever the switch. */
int rth_decode_path(int num_q_heads, int num_kv_heads, int head_dim);

/* No counterpart in the reference: process-wide choice of the split kernel
 * for rth_attn_decode_split, rth_attn_decode_split_noalloc and
 * rth_attn_decode_append_split, for measurement and tuning (the paged, RoPE
 * and q/k-norm entries ignore it). path 0 (the
 * default) = the MFMA kernel wherever it supports the shape, the VALU kernel
 * elsewhere; RTH_DECODE_VALU = the VALU kernel for every shape. Results of
 * the two kernels agree within the attention tolerance, not bit for bit.
 * Not synchronized with calls in flight on other host threads. */
int rth_set_decode_kernel(int path);

/* No counterpart in the reference: rth_attn_decode_split without the
 * `partial` argument, for callers that cannot allocate (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc). It calls no
 * hipMalloc/hipFree and no allocating library routine: the split partials
 * live in a fixed 16 MiB device array (2^22 floats) that each GPU holds from
 * the library's load until the process ends. Rejects shapes with
 * num_q_heads * num_splits * (head_dim + 2) > 2^22 floats
 * (RTH_ERR_INVALID_ARG). Every call on one GPU shares that GPU's array:
 * calls that overlap on one GPU (several streams or host threads) race and
 * must be serialized by the caller. Output is bit-identical to
 * rth_attn_decode_split with the same arguments. */
int rth_attn_decode_split_noalloc(uint16_t* out, const uint16_t* q, const uint8_t* k,
                                  const uint8_t* v, const float* k_scale,
                                  const float* v_scale, int num_splits,
                                  const int* cache_len, int num_q_heads, int num_kv_heads,
                                  int head_dim, float scale, void* stream);

/* No counterpart in the reference: KVCache::append(layer, k_new, v_new, 1,
 * cache_len) followed by the decode call (reference
 * src/model/supported/llama/llama3.cu:232-234 with n_new == 1) in one call
 * of two kernels instead of three. The new token ([Hkv, D] bf16) is
 * quantized into row *cache_len of the layer's cache slabs (bytes identical
 * to rth_kv_append_fp8) and attended with the *cache_len earlier keys;
 * output equals rth_kv_append_fp8 + rth_attn_decode_split. Same shapes and
 * scratch as rth_attn_decode_split. */
int rth_attn_decode_append_split(uint16_t* out, const uint16_t* q, uint8_t* k_cache,
                                 uint8_t* v_cache, float* k_scale, float* v_scale,
                                 const uint16_t* k_new, const uint16_t* v_new,
                                 float* partial, int num_splits, const int* cache_len,
                                 int num_q_heads, int num_kv_heads, int head_dim,
                                 float scale, void* stream);

/* Replaces kernels::flash_prefill_bf16 (reference
 * include/runtherder/kernels/flash_prefill.cuh:26-39): causal attention of
 * n_new queries at positions *cache_len .. *cache_len + n_new - 1 over keys
 * 0 .. *cache_len + n_new - 1. head_dim == 128. */
int rth_attn_prefill(uint16_t* out, const uint16_t* q, const uint8_t* k,
                     const uint8_t* v, const float* k_scale,
                     const float* v_scale, int n_new, const int* cache_len,
                     int num_q_heads, int num_kv_heads, int head_dim,
                     float scale, void* stream);

/* No counterpart in the reference: the causal attention of rth_attn_prefill
 * split over the keys, for calls after a long cache (speculative-decoding
 * verification, prefill chunks), instead of one workgroup per q tile
 * streaming every key (reference flash_prefill.cu:34-241 walks all keys
 * serially per tile: n_new = 4 at 32K keys costs ~50x a decode step).
 * n_new <= 80 (at head_dim 128 with splits that give the key runs a
 * workgroup per compute unit: <= 40), or head_dim != 128: the decode split
 * kernel over (block of tokens, kv head) units, token t over the first
 * *cache_len + t + 1 keys (shapes of the MFMA decode kernel, rth_decode_path
 * == RTH_DECODE_MFMA: head_dim 64 / 128 / 256; n_new <= 256), and the decode's
 * merge. Beyond, at head_dim 128: the flash prefill with each block of 128
 * rows (tokens x q heads of a kv head) split over num_splits runs of key
 * tiles, and a merge of their own. n_new's K/V must already be in the cache
 * (as for rth_attn_prefill). partial: rth_split_scratch_floats(n_new *
 * num_q_heads, head_dim, num_splits) floats, no initialization needed;
 * 1 <= n_new <= 4096. Results match rth_attn_prefill within the attention
 * tolerance (a different summation order). */
int rth_attn_prefill_split(uint16_t* out, const uint16_t* q, const uint8_t* k,
                           const uint8_t* v, const float* k_scale, const float* v_scale,
                           float* partial, int num_splits, int n_new, const int* cache_len,
                           int num_q_heads, int num_kv_heads, int head_dim, float scale,
                           void* stream);
int rth_attn_prefill_split_paged(uint16_t* out, const uint16_t* q, const uint8_t* k,
                                 const uint8_t* v, const float* k_scale,
                                 const float* v_scale, const int* block_table,
                                 int block_size, float* partial, int num_splits, int n_new,
                                 const int* cache_len, int num_q_heads, int num_kv_heads,
                                 int head_dim, float scale, void* stream);

/* Replaces kernels::attention_causal_bf16 (reference
 * include/runtherder/kernels/attention.cuh:21-34): the same causal attention
 * as rth_attn_prefill at any n_new, by the plain two-pass algorithm.
 * head_dim <= 512. */
int rth_attn_naive(uint16_t* out, const uint16_t* q, const uint8_t* k,
                   const uint8_t* v, const float* k_scale, const float* v_scale,
                   int n_new, const int* cache_len, int num_q_heads,
                   int num_kv_heads, int head_dim, float scale, void* stream);

/* *pos += delta on device. No counterpart in the reference (which advances
 * the decode position with a host copy, reference
 * include/runtherder/engine/context.h:41-45); lets one captured graph hold
 * several decode steps. */
int rth_advance_position(int* pos, int delta, void* stream);

/* Replaces kernels::rope_bf16 (reference include/runtherder/kernels/
 * rope.cuh:16-25): in-place rotate-half RoPE on q [seq_len, Hq, D] and
 * k [seq_len, Hkv, D] bf16; token t rotates by positions[t] (device array)
 * with inv_freq [D/2] (device). head_dim even, <= 256. sin/cos are taken in
 * double precision of the fp32 angle, rounded to fp32. */
int rth_rope_bf16(uint16_t* q, uint16_t* k, const int* positions,
                  const float* inv_freq, int seq_len, int num_q_heads,
                  int num_kv_heads, int head_dim, void* stream);

/* No counterpart in the reference: fuses the caller sequence
 * rope_bf16(q, k) then KVCache::append(layer, k, v, n_new, at_pos)
 * (reference src/model/supported/llama/llama3.cu:228-232) into one launch.
 * q is rotated in place exactly as rth_rope_bf16 does; rotated K and V rows
 * are quantized into the layer's cache slabs at rows *at_pos .. *at_pos +
 * n_new - 1, byte-identical to rth_rope_bf16 followed by rth_kv_append_fp8.
 * The k input is read only (left unrotated, unlike the two-step sequence).
 * head_dim in {64, 128, 256}. */
int rth_rope_append_fp8(uint16_t* q, uint8_t* k_cache, uint8_t* v_cache,
                        float* k_scale, float* v_scale, const uint16_t* k,
                        const uint16_t* v, const int* positions,
                        const float* inv_freq, const int* at_pos, int n_new,
                        int num_q_heads, int num_kv_heads, int head_dim,
                        void* stream);

/* Paged KV cache (no counterpart in the reference, whose README plans paged
 * attention, README.md:142-143): the cache slabs hold physical blocks of
 * block_size positions ([num_blocks * block_size, Hkv, D] E4M3 and
 * [num_blocks * block_size, Hkv] fp32 scales); logical position p of the
 * sequence lives at physical position block_table[p / block_size] *
 * block_size + p % block_size. block_table is a device int array covering
 * every block up to the last position used; block_size is a power of two
 * >= 32. Each entry below equals its contiguous counterpart on the gathered
 * cache, bit for bit. */
int rth_kv_append_fp8_paged(uint8_t* k_cache, uint8_t* v_cache, float* k_scale,
                            float* v_scale, const uint16_t* k, const uint16_t* v,
                            const int* at_pos, int n_new, int num_kv_heads, int head_dim,
                            const int* block_table, int block_size, void* stream);
int rth_attn_decode_split_paged(uint16_t* out, const uint16_t* q, const uint8_t* k,
                                const uint8_t* v, const float* k_scale, const float* v_scale,
                                const int* block_table, int block_size, float* partial,
                                int num_splits, const int* cache_len, int num_q_heads,
                                int num_kv_heads, int head_dim, float scale, void* stream);
int rth_attn_decode_append_split_paged(uint16_t* out, const uint16_t* q, uint8_t* k_cache,
                                       uint8_t* v_cache, float* k_scale, float* v_scale,
                                       const int* block_table, int block_size,
                                       const uint16_t* k_new, const uint16_t* v_new,
                                       float* partial, int num_splits, const int* cache_len,
                                       int num_q_heads, int num_kv_heads, int head_dim,
                                       float scale, void* stream);
/* No counterpart in the reference: fuses the per-layer decode step
 * rope_bf16(q, k, positions, inv_freq) -> KVCache::append(layer, k, v, 1,
 * cache_len) -> AttentionBackend::run(out, q, view, 1, cache_len) (reference
 * src/model/supported/llama/llama3.cu:228-234) into the two launches of
 * rth_attn_decode_append_split. q and k_new ([Hq, D] and [Hkv, D] bf16,
 * unrotated) are read only: both are rotated in registers by the angles of
 * positions[0] with rth_rope_bf16's arithmetic, so the cache row written at
 * *cache_len is byte-identical to rth_rope_bf16 + rth_kv_append_fp8 and the
 * output is bit-identical to rth_attn_decode_append_split on the rotated q
 * and k. Shapes
 * rth_decode_path reports as RTH_DECODE_MFMA under the automatic choice
 * (head_dim 64, 128, 256); others fail with an error. block_table == NULL (or the first entry point): the
 * contiguous layout. */
int rth_attn_decode_rope_append_split(uint16_t* out, const uint16_t* q, uint8_t* k_cache,
                                      uint8_t* v_cache, float* k_scale, float* v_scale,
                                      const uint16_t* k_new, const uint16_t* v_new,
                                      const int* positions, const float* inv_freq,
                                      float* partial, int num_splits, const int* cache_len,
                                      int num_q_heads, int num_kv_heads, int head_dim,
                                      float scale, void* stream);
int rth_attn_decode_rope_append_split_paged(uint16_t* out, const uint16_t* q, uint8_t* k_cache,
                                            uint8_t* v_cache, float* k_scale, float* v_scale,
                                            const int* block_table, int block_size,
                                            const uint16_t* k_new, const uint16_t* v_new,
                                            const int* positions, const float* inv_freq,
                                            float* partial, int num_splits,
                                            const int* cache_len, int num_q_heads,
                                            int num_kv_heads, int head_dim, float scale,
                                            void* stream);
/* No counterpart in the reference: the Qwen3 decode step,
 * rmsnorm_bf16_forward(q, q_norm) and (k, k_norm) per head -> rope_bf16 ->
 * KVCache::append -> run (reference src/model/supported/llama/
 * qwen3.cu:189-202), in the two launches of rth_attn_decode_append_split.
 * q and k_new are read only; the cache row equals rth_qk_norm_rope_append_fp8's
 * byte for byte, and the output is bit-identical to
 * rth_attn_decode_append_split on q and
 * k_new after rth_rmsnorm_bf16 (per head) and rth_rope_bf16. Shapes as
 * rth_attn_decode_rope_append_split. */
int rth_attn_decode_qk_norm_rope_append_split(
    uint16_t* out, const uint16_t* q, uint8_t* k_cache, uint8_t* v_cache, float* k_scale,
    float* v_scale, const uint16_t* k_new, const uint16_t* v_new, const uint16_t* q_norm,
    const uint16_t* k_norm, float eps, const int* positions, const float* inv_freq,
    float* partial, int num_splits, const int* cache_len, int num_q_heads, int num_kv_heads,
    int head_dim, float scale, void* stream);
int rth_attn_decode_qk_norm_rope_append_split_paged(
    uint16_t* out, const uint16_t* q, uint8_t* k_cache, uint8_t* v_cache, float* k_scale,
    float* v_scale, const int* block_table, int block_size, const uint16_t* k_new,
    const uint16_t* v_new, const uint16_t* q_norm, const uint16_t* k_norm, float eps,
    const int* positions, const float* inv_freq, float* partial, int num_splits,
    const int* cache_len, int num_q_heads, int num_kv_heads, int head_dim, float scale,
    void* stream);
int rth_attn_prefill_paged(uint16_t* out, const uint16_t* q, const uint8_t* k,
                           const uint8_t* v, const float* k_scale, const float* v_scale,
                           const int* block_table, int block_size, int n_new,
                           const int* cache_len, int num_q_heads, int num_kv_heads,
                           int head_dim, float scale, void* stream);

/* No counterpart in the reference: fuses the Qwen3 caller sequence
 * rmsnorm_bf16_forward(q, q_norm) [per q head], rmsnorm_bf16_forward(k,
 * k_norm) [per kv head], rope_bf16(q, k), KVCache::append(k, v) (reference
 * src/model/supported/llama/qwen3.cu:189-200) into one launch. q is
 * normalized and rotated in place; the cache receives exactly the bytes of
 * rth_rmsnorm_bf16 + rth_rope_bf16 + rth_kv_append_fp8; k is read only.
 * q_norm, k_norm: [head_dim] bf16 gains. head_dim in {64, 128, 256}. */
int rth_qk_norm_rope_append_fp8(uint16_t* q, uint8_t* k_cache, uint8_t* v_cache,
                                float* k_scale, float* v_scale, const uint16_t* k,
                                const uint16_t* v, const uint16_t* q_norm,
                                const uint16_t* k_norm, float eps, const int* positions,
                                const float* inv_freq, const int* at_pos, int n_new,
                                int num_q_heads, int num_kv_heads, int head_dim,
                                void* stream);

/* Replaces kernels::rmsnorm_bf16_forward (reference include/runtherder/
 * kernels/rmsnorm.cuh:14-22): y = bf16((x * rrms) * g) per row of
 * x [num_tokens, hidden_dim] bf16, rrms = 1 / sqrt(sum(x^2) / hidden_dim +
 * eps) with a correctly rounded sqrt and division; y may alias x.
 * hidden_dim a multiple of 8, <= 16384. The sum of squares runs over
 * rth_rmsnorm_lanes(hidden_dim) lane partials in a fixed order. */
int rth_rmsnorm_bf16(uint16_t* y, const uint16_t* x, const uint16_t* g, int num_tokens,
                     int hidden_dim, float eps, void* stream);

/* Lanes per row of rth_rmsnorm_bf16's reduction (the next power of two of
 * hidden_dim / 8, at most 64); 0 for an invalid hidden_dim. No reference
 * counterpart: lets a checker restate the summation order. */
int rth_rmsnorm_lanes(int hidden_dim);

/* ---- a batch of sequences (no counterparts in the reference, which serves one
 * sequence at a time) -------------------------------------------------------
 *
 * Packed rows: the tokens of num_seqs sequences one behind the other; sequence
 * b holds rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (cu_seqlens: num_seqs + 1
 * device ints, ascending; bounds past num_rows are taken as num_rows). What rows
 * behind the last sequence hold does not matter, and they are not written. Row strides are in
 * elements, multiples of 8, at least heads * head_dim and at most 2^24 (so q, k
 * and v may be slices of one projection's rows). Rows of q, k, v and out start 16-byte aligned.
 *
 * Block tables of a batch: [num_seqs, table_blocks] device ints; entry i of row
 * b is the page of positions i * block_size .. (i + 1) * block_size - 1 of
 * sequence b, an entry outside 0 .. num_blocks - 1 names no page. Slabs hold
 * num_blocks pages of block_size positions (a power of two >= 32). num_seqs <=
 * 4096. */

/* Causal attention over whole prompts: row t of sequence b attends rows
 * cu_seqlens[b] .. t, straight from the bf16 k and v ([rows, Hkv, D], no
 * cache). head_dim 64, 128, 256; any Hq / Hkv. out may not overlap the inputs.
 * A key that a row does not see leaves no trace in it, whatever k and v hold there. */
int rth_attn_packed(uint16_t* out, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                    const int* cu_seqlens, int num_seqs, int num_rows, int64_t out_stride,
                    int64_t q_stride, int64_t k_stride, int64_t v_stride, int num_q_heads,
                    int num_kv_heads, int head_dim, float scale, void* stream);

/* Appends a batch's K and V rows ([rows, Hkv, D] bf16, packed; cu_seqlens NULL:
 * one row per sequence, row b of sequence b) to the sequences' pages: row t of
 * sequence b at position at_pos[b] + t - cu_seqlens[b] of it, byte for byte
 * as rth_kv_append_fp8_paged would. A row whose position lies outside the table, or
 * whose table entry names no page, is not stored. Rows of one call go to positions of
 * their own (sequences that share a page do not both write to it). head_dim % 8 == 0, 8 <=
 * head_dim <= 512. */
int rth_kv_append_fp8_batch(uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale,
                            const uint16_t* k, const uint16_t* v, int64_t k_stride,
                            int64_t v_stride, const int* cu_seqlens, const int* at_pos,
                            int num_seqs, int num_rows, int num_kv_heads, int head_dim,
                            const int* block_tables, int table_blocks, int num_blocks,
                            int block_size, void* stream);

/* Decode attention of a batch, one query token per sequence (q, out [num_seqs,
 * Hq, D]): sequence b attends keys 0 .. lens[b] - 1. The first *prefix_len of
 * them are the same for every sequence and lie in the pages of prefix_table
 * [prefix_blocks]: they are read and multiplied once for the whole batch. The
 * others lie in the sequence's own row of block_tables, at their own positions
 * (so tables that rth_pages_fork made can be passed whole, with any one of
 * their rows as prefix_table). prefix_table and prefix_len NULL: nothing is shared. lens[b] <= 0:
 * an unused slot, its output row is zeros. A sequence shorter than the prefix sees
 * its lens[b] keys of it (where those that a longer one sees are finite: the rows of a kv head
 * are one product, in which a NaN or an infinity times a weight of 0 is a NaN; what no
 * sequence sees does not matter). Keys past a table's end, and keys whose
 * table entry names no page, are left out. head_dim 64, 128, 256; any Hq / Hkv;
 * num_seqs * Hq <= 2^24, num_seqs * table_blocks * block_size <= 2^35.
 * partial: rth_batch_scratch_floats floats, 16-byte aligned, no
 * initialization needed, not shared by calls that overlap (graphs included). */
size_t rth_batch_scratch_floats(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim);
int rth_attn_decode_batch(uint16_t* out, int64_t out_stride, const uint16_t* q, int64_t q_stride,
                          const uint8_t* k, const uint8_t* v, const float* k_scale,
                          const float* v_scale, const int* block_tables, int table_blocks,
                          int num_blocks, int block_size, const int* lens,
                          const int* prefix_table, int prefix_blocks, const int* prefix_len,
                          float* partial, int num_seqs, int num_q_heads, int num_kv_heads,
                          int head_dim, float scale, void* stream);

/* Pages of a paged cache of num_layers layers (slabs [num_layers, num_blocks *
 * block_size, Hkv, D] and [.., Hkv]; head_dim % 8 == 0), with the bookkeeping on the device: refs
 * [num_blocks] counts the table entries that hold each page, a page with refs
 * <= 0 is free, and the lowest free pages are given out first. A table entry < 0
 * holds no page. `work` is scratch of rth_pages_work_ints ints (no
 * initialization needed, not shared by calls that overlap); *status gets bit 0
 * when the free pages did not suffice and bit 1 when a table is too short, and the call has
 * then changed nothing else. Calls on one pool run one behind the other (one
 * stream, or ordered streams). */
size_t rth_pages_work_ints(int num_blocks);

/* Copies page src[i] to page dst[i] in every layer, i < count. The dst pages are
 * distinct, and none of them is a src page; ids that name no page are skipped. */
int rth_pages_copy(uint8_t* k, uint8_t* v, float* k_scale, float* v_scale, int num_layers,
                   int num_blocks, int block_size, int num_kv_heads, int head_dim,
                   const int* src, const int* dst, int count, void* stream);

/* Gives sequence b the pages it lacks for positions lens[b] .. lens[b] +
 * n_new[b] - 1 (entries of its table row that are < 0), in order of b. */
int rth_pages_reserve(int* refs, int* work, int* status, int num_blocks, int block_size,
                      int* block_tables, int table_blocks, const int* lens, const int* n_new,
                      int num_seqs, void* stream);

/* Child i becomes a copy of sequence parents[i] of the source tables: it shares
 * the parent's filled pages (refs + 1) and gets, where the last one is part
 * filled, a page of its own with a copy of the filled rows of every layer.
 * dst_tables [num_children, table_blocks] and dst_lens are written whole and
 * may not overlap the source's; what they held before is to be freed first. A
 * parent outside 0 .. num_src - 1 gives an empty child. num_children <= 4096. */
int rth_pages_fork(uint8_t* k, uint8_t* v, float* k_scale, float* v_scale, int num_layers,
                   int num_blocks, int block_size, int num_kv_heads, int head_dim, int* refs,
                   int* work, int* status, int* dst_tables, int* dst_lens,
                   const int* src_tables, const int* src_lens, int table_blocks, int num_src,
                   const int* parents, int num_children, void* stream);

/* Frees the sequences with drop[b] != 0 (drop NULL: all): refs - 1 for each
 * page of their rows, entries -1, lengths 0. */
int rth_pages_free(int* refs, int num_blocks, int* block_tables, int table_blocks, int* lens,
                   const int* drop, int num_seqs, void* stream);

/* Moves the pages in use down to 0 .. (their number) - 1: those above, lowest
 * first, into the free ones below, lowest first, in every layer; the tables
 * (all that hold pages of the pool) and refs follow. */
int rth_pages_compact(uint8_t* k, uint8_t* v, float* k_scale, float* v_scale, int num_layers,
                      int num_blocks, int block_size, int num_kv_heads, int head_dim, int* refs,
                      int* work, int* block_tables, int table_blocks, int num_seqs,
                      void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RTH_ATTN_H */
