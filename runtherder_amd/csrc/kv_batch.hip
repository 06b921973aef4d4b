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
//
// 8 kv heads, head_dim 128: 64 sequences of one token 7.4 us, which is the call's own time
// on the host (kernel 3); 9 prompts, 9687 tokens, 15.7 us = 3.8 TB/s.
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

// kLanes lanes per row, kChunks chunks of 8 elements each (chunk sub + c * kLanes).
template <int kLanes, int kChunks>
__global__ __launch_bounds__(kAppendBlock) void append_batch_kernel(
    AppendSlab s0, AppendSlab s1, const int* __restrict__ cu, const int* __restrict__ at_pos,
    int num_seqs, int num_rows, int hkv, int head_dim, const int* __restrict__ tables,
    int table_blocks, int num_blocks, int block_shift) {
    constexpr uint32_t kRows = kWave / kLanes;   // of a wave
    const AppendSlab s    = blockIdx.y == 0 ? s0 : s1;
    const int        lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int        sub = lane % kLanes, mine = lane / kLanes;
    const uint32_t   heads = static_cast<uint32_t>(hkv);
    const uint32_t   end   = static_cast<uint32_t>(num_rows) * heads;   // below 2^31
    const uint32_t   row0  = static_cast<uint32_t>(
        uniform(static_cast<int>((blockIdx.x * kAppendBlock + (threadIdx.x & ~(kWave - 1u))) / kLanes)));
    const uint32_t row = row0 + mine;
    const bool     has = row < end;
    const int      tok = static_cast<int>(row / heads), kvh = static_cast<int>(row - tok * heads);

    u32x4           x[kChunks];
    const uint16_t* from = s.x + tok * s.stride + static_cast<int64_t>(kvh) * head_dim;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int e = 8 * (sub + c * kLanes);
        x[c]        = u32x4{};
        if (has && e < head_dim) {
            x[c] = *reinterpret_cast<const u32x4*>(from + e);
        }
    }
    // The sequence of each of the wave's tokens.
    int seq = tok;
    if (cu != nullptr) {
        seq = 0;
        const int first = static_cast<int>(row0 / heads);
        const int last  = static_cast<int>((min(row0 + kRows, end) - 1) / heads);
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
        const int     begin = cu != nullptr ? cu[seq] : tok;
        const int64_t p     = static_cast<int64_t>(at_pos[seq]) + tok - begin;
        if (tok >= begin && p >= 0 && (p >> block_shift) < table_blocks) {
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
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            amax = fmaxf(amax, fabsf(__uint_as_float(x[c][e] << 16)));
            amax = fmaxf(amax, fabsf(__uint_as_float(x[c][e] & 0xffff0000u)));
        }
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
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int e = 8 * (sub + c * kLanes);
        auto      f = [&](uint32_t w, bool hi) { return __uint_as_float(hi ? w & 0xffff0000u : w << 16) * inv; };
        uint32_t  lo = 0, hi = 0;
        lo = e4m3x2_pack<false>(f(x[c].x, false), f(x[c].x, true), lo);
        lo = e4m3x2_pack<true>(f(x[c].y, false), f(x[c].y, true), lo);
        hi = e4m3x2_pack<false>(f(x[c].z, false), f(x[c].z, true), hi);
        hi = e4m3x2_pack<true>(f(x[c].w, false), f(x[c].w, true), hi);
        if (e < head_dim) {
            *reinterpret_cast<u32x2*>(s.q + dst * head_dim + e) = u32x2{lo, hi};
        }
    }
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
    // Large appends: half the lanes per row, so that each has two loads in flight and a
    // wave's search of the sequences serves twice the rows; small ones finish
    // sooner with the wider groups.
    const int64_t rows  = static_cast<int64_t>(num_rows) * num_kv_heads;
    const bool    large = 2 * rows >= 32768 && lanes >= 8;
    lanes               = large ? lanes / 2 : lanes;
    const int64_t per   = kAppendBlock / lanes;
    const dim3    grid(static_cast<unsigned>((rows + per - 1) / per), 2);
    const AppendSlab sk{k_q, k_scale, k, k_stride}, sv{v_q, v_scale, v, v_stride};
#define RTH_APPEND(L, C)                                                                          \
    append_batch_kernel<L, C><<<grid, kAppendBlock, 0, stream>>>(                                 \
        sk, sv, cu_seqlens, at_pos, num_seqs, num_rows, num_kv_heads, head_dim, block_tables,     \
        table_blocks, num_blocks, block_shift)
#define RTH_CASE(L)            \
    case L:                    \
        if (large) {           \
            RTH_APPEND(L, 2);  \
        } else {               \
            RTH_APPEND(L, 1);  \
        }                      \
        break;
    switch (lanes) {
        case 1:
            RTH_APPEND(1, 1);
            break;
        case 2:
            RTH_APPEND(2, 1);
            break;
        RTH_CASE(4)
        RTH_CASE(8)
        RTH_CASE(16)
        RTH_CASE(32)
        case 64:
            RTH_APPEND(64, 1);
            break;
        default:
            return hipErrorInvalidValue;
    }
#undef RTH_CASE
#undef RTH_APPEND
    return hipGetLastError();
}

}  // namespace rth
