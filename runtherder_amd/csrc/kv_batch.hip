// Append of a batch's K and V rows into the pages of its sequences, gfx950.
//
// Token t of sequence b (cu[b] <= t < cu[b + 1]; without cu, token t is sequence
// t's one) goes to position p = at_pos[b] + t - cu[b], which lies at row
// table_b[p / block] * block + p % block of the slabs. Per (token, kv head) row:
// scale = amax / 448 and code = E4M3(x * (448 / amax)), bit for bit as the
// append of one sequence (kv_quant.hip). A token that has no page (its position
// past the table, a table entry that names no page, a row behind the last
// sequence) is not stored.
//
// Bound by bytes (6 D + 8 per row of K and V together) for prompts, and for one
// token per sequence by the chain of dependent reads cu -> at_pos -> table; the
// row itself is loaded before that chain. A wave finds its rows' sequences by
// counting, 64 bounds at a time, how many sequences end at or before the row.
#include "batch_common.hpp"
#include "launch.hpp"

namespace rth {
namespace {

constexpr int kAppendBlock = 256;

struct AppendSlab {
    uint8_t*        q;
    float*          scale;
    const uint16_t* x;
    int64_t         stride;   // elements per token
};

template <int kLanes>   // lanes per row, 8 elements each
__global__ __launch_bounds__(kAppendBlock) void append_batch_kernel(
    AppendSlab s0, AppendSlab s1, const int* __restrict__ cu, const int* __restrict__ at_pos,
    int num_seqs, int num_rows, int hkv, int head_dim, const int* __restrict__ tables,
    int table_blocks, int num_blocks, int block_shift) {
    constexpr int    kRows = kWave / kLanes;   // of a wave
    const AppendSlab s     = blockIdx.y == 0 ? s0 : s1;
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int sub = lane % kLanes, mine = lane / kLanes;
    const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * kAppendBlock + threadIdx.x - lane) / kLanes;
    const int64_t row  = row0 + mine;
    const int64_t end  = static_cast<int64_t>(num_rows) * hkv;
    const bool    has  = row < end && 8 * sub < head_dim;
    const int     tok  = static_cast<int>(row / hkv), kvh = static_cast<int>(row % hkv);

    u32x4 x = {};
    if (has) {
        x = *reinterpret_cast<const u32x4*>(s.x + tok * s.stride + static_cast<int64_t>(kvh) * head_dim +
                                            8 * sub);
    }
    // The sequence of each of the wave's tokens.
    int seq = tok;
    if (cu != nullptr) {
        seq = 0;
        const int first = static_cast<int>(row0 / hkv);
        const int last  = static_cast<int>((min(row0 + kRows, end) - 1) / hkv);
        for (int b0 = 0; b0 < num_seqs; b0 += kWave) {
            const int b   = b0 + lane;
            const int top = b < num_seqs ? cu[b + 1] : INT32_MAX;
            for (int t = first; t <= last; ++t) {
                const int n = __popcll(__ballot(top <= t));
                seq += t == tok ? n : 0;
            }
        }
    }
    int64_t dst = -1;
    if (has && seq < num_seqs) {
        const int64_t p = static_cast<int64_t>(at_pos[seq]) + (cu != nullptr ? tok - cu[seq] : 0);
        if (p >= 0 && (p >> block_shift) < table_blocks && (cu == nullptr || tok >= cu[seq])) {
            const int page = tables[static_cast<int64_t>(seq) * table_blocks + (p >> block_shift)];
            if (page >= 0 && page < num_blocks) {
                const int64_t at = (static_cast<int64_t>(page) << block_shift) +
                                   (p & ((int64_t{1} << block_shift) - 1));
                dst = at * hkv + kvh;
            }
        }
    }

    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        amax = fmaxf(amax, fabsf(__uint_as_float(x[e] << 16)));
        amax = fmaxf(amax, fabsf(__uint_as_float(x[e] & 0xffff0000u)));
    }
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) {
        amax = wave_xor_max(amax, m);
    }
    if (dst < 0) {
        return;
    }
    const float inv = amax > 0.0f ? kE4M3Max / amax : 0.0f;
    if (sub == 0) {
        s.scale[dst] = amax / kE4M3Max;
    }
    uint32_t lo = 0, hi = 0;
    lo = e4m3x2_pack<false>(__uint_as_float(x.x << 16) * inv, __uint_as_float(x.x & 0xffff0000u) * inv, lo);
    lo = e4m3x2_pack<true>(__uint_as_float(x.y << 16) * inv, __uint_as_float(x.y & 0xffff0000u) * inv, lo);
    hi = e4m3x2_pack<false>(__uint_as_float(x.z << 16) * inv, __uint_as_float(x.z & 0xffff0000u) * inv, hi);
    hi = e4m3x2_pack<true>(__uint_as_float(x.w << 16) * inv, __uint_as_float(x.w & 0xffff0000u) * inv, hi);
    *reinterpret_cast<u32x2*>(s.q + dst * head_dim + 8 * sub) = u32x2{lo, hi};
}

}  // namespace

hipError_t kv_append_batch_launch(uint8_t* k_q, uint8_t* v_q, float* k_scale, float* v_scale,
                                  const uint16_t* k, const uint16_t* v, int64_t k_stride,
                                  int64_t v_stride, const int* cu_seqlens, const int* at_pos,
                                  int num_seqs, int num_rows, int num_kv_heads, int head_dim,
                                  const int* block_tables, int table_blocks, int num_blocks,
                                  int block_shift, hipStream_t stream) {
    int lanes = 1;
    while (8 * lanes < head_dim) {
        lanes <<= 1;
    }
    const int64_t rows = static_cast<int64_t>(num_rows) * num_kv_heads;
    const int64_t per  = kAppendBlock / lanes;
    const dim3    grid(static_cast<unsigned>((rows + per - 1) / per), 2);
    const AppendSlab sk{k_q, k_scale, k, k_stride}, sv{v_q, v_scale, v, v_stride};
    switch (lanes) {
#define RTH_CASE(L)                                                                            \
    case L:                                                                                    \
        append_batch_kernel<L><<<grid, kAppendBlock, 0, stream>>>(                             \
            sk, sv, cu_seqlens, at_pos, num_seqs, num_rows, num_kv_heads, head_dim, block_tables, \
            table_blocks, num_blocks, block_shift);                                            \
        break;
        RTH_CASE(1)
        RTH_CASE(2)
        RTH_CASE(4)
        RTH_CASE(8)
        RTH_CASE(16)
        RTH_CASE(32)
        RTH_CASE(64)
#undef RTH_CASE
        default:
            return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace rth
