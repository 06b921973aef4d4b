// Attention and cache append of a batch of sequences, forwarding to the C ABI
// (no reference counterparts: the reference serves one sequence at a time).
// rth_attn.h's batch section says what packed rows and block tables are.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp8.h>
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include <rth_attn.h>
#include <runtherder/device/check.h>

namespace runtherder::kernels {

// Causal attention over whole prompts, straight from bf16 k and v (no cache).
// Strides are in elements from one token's row to the next.
inline void flash_packed_bf16(__hip_bfloat16*       out,
                              const __hip_bfloat16* q,
                              const __hip_bfloat16* k,
                              const __hip_bfloat16* v,
                              const int*            cu_seqlens,
                              int                   num_seqs,
                              int                   num_rows,
                              std::int64_t          out_stride,
                              std::int64_t          q_stride,
                              std::int64_t          k_stride,
                              std::int64_t          v_stride,
                              int                   num_q_heads,
                              int                   num_kv_heads,
                              int                   head_dim,
                              float                 scale,
                              hipStream_t           stream = nullptr) {
    RUNTHERDER_RTH_CHECK(rth_attn_packed(
        reinterpret_cast<std::uint16_t*>(out), reinterpret_cast<const std::uint16_t*>(q),
        reinterpret_cast<const std::uint16_t*>(k), reinterpret_cast<const std::uint16_t*>(v),
        cu_seqlens, num_seqs, num_rows, out_stride, q_stride, k_stride, v_stride, num_q_heads,
        num_kv_heads, head_dim, scale, stream));
}

// Floats of flash_decode_batch_bf16's scratch on the current device.
[[nodiscard]] inline std::size_t batch_scratch_floats(int num_seqs, int num_q_heads,
                                                      int num_kv_heads, int head_dim) {
    return rth_batch_scratch_floats(num_seqs, num_q_heads, num_kv_heads, head_dim);
}

// One query token of each sequence over a paged cache; the first *prefix_len
// keys, in the pages of prefix_table, are shared (both null: none are).
inline void flash_decode_batch_bf16(__hip_bfloat16*       out,
                                    std::int64_t          out_stride,
                                    const __hip_bfloat16* q,
                                    std::int64_t          q_stride,
                                    const __hip_fp8_e4m3* k,
                                    const __hip_fp8_e4m3* v,
                                    const float*          k_scale,
                                    const float*          v_scale,
                                    const int*            block_tables,
                                    int                   table_blocks,
                                    int                   num_blocks,
                                    int                   block_size,
                                    const int*            lens,
                                    const int*            prefix_table,
                                    int                   prefix_blocks,
                                    const int*            prefix_len,
                                    float*                partial,
                                    int                   num_seqs,
                                    int                   num_q_heads,
                                    int                   num_kv_heads,
                                    int                   head_dim,
                                    float                 scale,
                                    hipStream_t           stream = nullptr) {
    RUNTHERDER_RTH_CHECK(rth_attn_decode_batch(
        reinterpret_cast<std::uint16_t*>(out), out_stride,
        reinterpret_cast<const std::uint16_t*>(q), q_stride,
        reinterpret_cast<const std::uint8_t*>(k), reinterpret_cast<const std::uint8_t*>(v),
        k_scale, v_scale, block_tables, table_blocks, num_blocks, block_size, lens,
        prefix_table, prefix_blocks, prefix_len, partial, num_seqs, num_q_heads, num_kv_heads,
        head_dim, scale, stream));
}

}  // namespace runtherder::kernels
