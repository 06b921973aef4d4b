// Device helpers of the batch operators (packed prompts, batch decode, batch
// append, pages): where a workgroup's part of a batch of sequences lies.
#pragma once

#include "device_common.hpp"

namespace rth {

constexpr int kMaxBatchSeqs = 4096;   // sequences of one batch call

template <int kCtrl>
__device__ __forceinline__ int dpp_i(int x) {
    return __builtin_amdgcn_update_dpp(0, x, kCtrl, 0xF, 0xF, false);
}

// x, as a value of its own: what is computed from it is computed there, not kept
// in registers from an earlier use.
__device__ __forceinline__ int again(int x) {
    asm("" : "+v"(x));
    return x;
}

// x, the same in every lane, in a scalar register (a division leaves it in
// vector ones).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Sum over the wave, in every lane: lane exchanges within rows of 16, then the
// two cross-row swaps. Every lane must be active.
__device__ __forceinline__ int wave_sum_i(int v) {
    v += dpp_i<0xB1>(v);    // quad_perm [1,0,3,2]
    v += dpp_i<0x4E>(v);    // quad_perm [2,3,0,1]
    v += dpp_i<0x141>(v);   // row_half_mirror
    v += dpp_i<0x140>(v);   // row_mirror
    const auto a = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(v),
                                                    static_cast<uint32_t>(v), false, false);
    v            = static_cast<int>(a[0] + a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(v),
                                                    static_cast<uint32_t>(v), false, false);
    return static_cast<int>(b[0] + b[1]);
}

// Maximum over the wave, likewise.
__device__ __forceinline__ int wave_max_i(int v) {
    v = max(v, dpp_i<0xB1>(v));
    v = max(v, dpp_i<0x4E>(v));
    v = max(v, dpp_i<0x141>(v));
    v = max(v, dpp_i<0x140>(v));
    const auto a = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(v),
                                                    static_cast<uint32_t>(v), false, false);
    v            = max(static_cast<int>(a[0]), static_cast<int>(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(v),
                                                    static_cast<uint32_t>(v), false, false);
    return max(static_cast<int>(b[0]), static_cast<int>(b[1]));
}

// Set bits of `mask` below this lane.
__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// Sequence and token bounds of a packed batch: cu[b] .. cu[b + 1] clamped into
// the rows that exist, so that no bound of a caller's array leads outside them.
__device__ __forceinline__ int clamp_rows(int x, int num_rows) {
    return min(max(x, 0), num_rows);
}

}  // namespace rth
