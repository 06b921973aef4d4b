// Attention of a batch of sequences (no reference counterpart): whole prompts
// packed one behind the other, and one token of each sequence over a paged
// cache whose first pages all may share. Owns the decode's scratch, so the
// decodes of one object run one behind the other (one stream, or ordered
// streams; a captured graph counts).
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include <runtherder/attention/backend.h>
#include <runtherder/attention/kv_view.h>
#include <runtherder/check.h>
#include <runtherder/device/memory.h>
#include <runtherder/kernels/batch.h>

namespace runtherder::attention {

class BatchAttention {
public:
    // max_seqs: of one decode.
    BatchAttention(const AttnConfig& config, int max_seqs) : config_(config), max_seqs_(max_seqs) {
        RUNTHERDER_CHECK(max_seqs >= 1, "BatchAttention max_seqs must be >= 1");
        RUNTHERDER_CHECK(kernels::batch_scratch_floats(max_seqs, config.num_q_heads,
                                                       config.num_kv_heads, config.head_dim) > 0,
                         "BatchAttention serves head_dim 64, 128 and 256, up to 4096 sequences");
        std::size_t most = 0;
        for (int n = 1; n <= max_seqs; ++n) {
            most = std::max(most, kernels::batch_scratch_floats(n, config.num_q_heads,
                                                                config.num_kv_heads,
                                                                config.head_dim));
        }
        partial_ = device::make_device_unique<float>(most);
    }

    // Causal attention of num_seqs prompts (out, q [rows, Hq, D], k, v [rows,
    // Hkv, D]; strides in elements, 0: rows without gaps).
    void run_packed(__hip_bfloat16* out, const __hip_bfloat16* q, const __hip_bfloat16* k,
                    const __hip_bfloat16* v, const int* cu_seqlens, int num_seqs, int num_rows,
                    hipStream_t stream, std::int64_t q_stride = 0, std::int64_t k_stride = 0,
                    std::int64_t v_stride = 0) const {
        const std::int64_t qo = static_cast<std::int64_t>(config_.num_q_heads) * config_.head_dim;
        const std::int64_t kv = static_cast<std::int64_t>(config_.num_kv_heads) * config_.head_dim;
        kernels::flash_packed_bf16(out, q, k, v, cu_seqlens, num_seqs, num_rows, qo,
                                   q_stride != 0 ? q_stride : qo, k_stride != 0 ? k_stride : kv,
                                   v_stride != 0 ? v_stride : kv, config_.num_q_heads,
                                   config_.num_kv_heads, config_.head_dim, config_.scale, stream);
    }

    // One token of each of the view's sequences (out, q [seqs, Hq, D]) over
    // its keys 0 .. lens[b] - 1. The first *prefix_len lie in the pages of
    // prefix_table for all of them (both null: nothing is shared).
    void run_decode(__hip_bfloat16* out, const __hip_bfloat16* q, const KVBatchView& kv,
                    const int* lens, hipStream_t stream, const int* prefix_table = nullptr,
                    int prefix_blocks = 0, const int* prefix_len = nullptr) {
        RUNTHERDER_CHECK(kv.num_seqs <= max_seqs_, "BatchAttention was made for fewer sequences");
        const std::int64_t row = static_cast<std::int64_t>(config_.num_q_heads) * config_.head_dim;
        kernels::flash_decode_batch_bf16(out, row, q, row, kv.k, kv.v, kv.k_scale, kv.v_scale,
                                         kv.block_tables, kv.table_blocks, kv.num_blocks,
                                         kv.block_size, lens, prefix_table, prefix_blocks,
                                         prefix_len, partial_.get(), kv.num_seqs,
                                         config_.num_q_heads, config_.num_kv_heads,
                                         config_.head_dim, config_.scale, stream);
    }

    [[nodiscard]] int max_seqs() const noexcept { return max_seqs_; }

private:
    AttnConfig                     config_;
    int                            max_seqs_;
    device::DeviceUniquePtr<float> partial_;
};

}  // namespace runtherder::attention
