// Causal attention over whole prompts, packed one behind the other, gfx950.
//
// For row t of sequence b (cu[b] <= t < cu[b + 1]) and q head h of kv head
// h / G: out[t, h] = sum over cu[b] <= u <= t of softmax_u(scale * q[t, h] .
// k[u, h / G]) * v[u, h / G], from the bf16 K and V rows themselves (no cache).
//
//  * Rows: the G q heads of a kv head are packed token by token (row r of a
//    sequence: token r / G, head r % G), 32 kQ rows per wave, four waves per
//    workgroup. A workgroup finds its (sequence, row block) itself: block w in
//    order of the block's index within its sequence, longest first, so that the
//    last workgroups to start are short ones, whatever mix of lengths the batch
//    holds; no plan, no workspace and one launch.
//  * Keys in tiles of 64 (32 at head_dim 256), K and V rows through registers into two LDS buffers (the next tile's
//    loads run under this tile's products).
//  * S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_bf16: a lane owns
//    a query row, so the softmax needs no lane exchange but for a new maximum; P^T
//    goes from the score registers into the second product as it is: the V^T
//    operand is read (ds_read_b64_tr_b16) in the scores' key order.
//  * Softmax in base 2 with a lazy reference maximum in fp32; P is rounded to
//    bf16 (half a step, 2^-9 of each weight) for the matrix product, the row
//    sum is taken from the fp32 values.
#include <algorithm>

#include "attn_tile.hpp"
#include "launch.hpp"

namespace rth {
namespace {

// Which (sequence, block of `bm` rows) workgroup w of a kv head takes: blocks
// in descending order of their index j within the sequence (their work grows
// with j), within one j in order of the sequences. nblk[b]: blocks of sequence
// b, in LDS. False: w is past the last block.
struct BlockOf {
    int seq, j;
};
__device__ __forceinline__ bool find_block(int w, const int* nblk, int num_seqs, int lane,
                                           BlockOf& at) {
    // blocks with index >= t
    auto from = [&](int t) {
        int n = 0;
        for (int b = lane; b < num_seqs; b += kWave) {
            n += max(0, nblk[b] - t);
        }
        return __builtin_amdgcn_readfirstlane(wave_sum_i(n));
    };
    if (w >= from(0)) {
        return false;
    }
    // The largest t with from(t) > w, and from(t + 1).
    int lo = 0, hi = 1, above = from(1);
    while (above > w) {
        lo    = hi;
        hi    = 2 * hi;
        above = from(hi);
    }
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, f = from(mid);
        if (f > w) {
            lo = mid;
        } else {
            hi    = mid;
            above = f;
        }
    }
    int rank = w - above;   // among the sequences with more than lo blocks
    for (int b0 = 0; b0 < num_seqs; b0 += kWave) {
        const int      b    = b0 + lane;
        const bool     mine = b < num_seqs && nblk[b] > lo;
        const uint64_t m    = __ballot(mine);
        const int      n    = __popcll(m);
        if (rank < n) {
            const uint64_t hit = __ballot(mine && lanes_below(m) == rank);
            at                 = {b0 + __ffsll(static_cast<unsigned long long>(hit)) - 1, lo};
            return true;
        }
        rank -= n;
    }
    return false;
}

template <int D, int kQ>
__global__ __launch_bounds__(kPThr, kQ == 1 && D < 256 ? 2 : 1) void flash_packed_kernel(
    uint16_t* __restrict__ out, const uint16_t* __restrict__ q, const uint16_t* __restrict__ k,
    const uint16_t* __restrict__ v, const int* __restrict__ cu, int num_seqs, int num_rows,
    int64_t out_stride, int64_t q_stride, int64_t k_stride, int64_t v_stride, int group, int hkv,
    float scale_log2) {
    using T           = AttnTile<D>;
    constexpr int kPN = T::kN;
    constexpr int kBM = 32 * kQ * kPW;
    constexpr int kCpr   = D / 8;          // 16-byte chunks per row
    constexpr int kCopy  = kPThr / kCpr;   // rows of one copy step
    constexpr int kSteps = kPN / kCopy;
    constexpr int kTiles = 2 * T::kBytes > 4 * kMaxBatchSeqs ? 2 * T::kBytes : 4 * kMaxBatchSeqs;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kTiles];

    const int tid  = static_cast<int>(threadIdx.x);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int lane = tid & (kWave - 1);
    const int col  = lane & 31;
    const int h    = lane >> 5;
    const int bid  = static_cast<int>(blockIdx.x);
    const int w    = bid / hkv, hb = bid % hkv;
    // The blocks of one kv head on one XCD (workgroup id modulo 8), where they
    // share its K and V rows in L2.
    const int kvh = (hkv & 7) == 0 ? (hb & 7) * (hkv >> 3) + (hb >> 3) : hb;

    BlockOf at;
    {
        int* nblk = reinterpret_cast<int*>(lds);
        for (int b = tid; b < num_seqs; b += kPThr) {
            const int n = clamp_rows(cu[b + 1], num_rows) - clamp_rows(cu[b], num_rows);
            nblk[b] = static_cast<int>((static_cast<int64_t>(max(n, 0)) * group + kBM - 1) / kBM);
        }
        __syncthreads();
        const bool found = find_block(w, nblk, num_seqs, lane, at);
        __syncthreads();
        if (!found) {
            return;
        }
    }
    const int seq   = __builtin_amdgcn_readfirstlane(at.seq);
    const int j     = __builtin_amdgcn_readfirstlane(at.j);
    const int first = clamp_rows(cu[seq], num_rows);
    const int n     = clamp_rows(cu[seq + 1], num_rows) - first;
    const int rows  = n * group;
    const int r0    = j * kBM;
    const int n_tiles = (min(r0 + kBM, rows) - 1) / group / kPN + 1;

    // Rows of this lane; past the sequence's last they repeat it and store nothing.
    int my_row[kQ], my_tok[kQ];
    const int wr0 = r0 + wave * 32 * kQ;
#pragma unroll
    for (int a = 0; a < kQ; ++a) {
        my_row[a] = min(wr0 + 32 * a + col, rows - 1);
        my_tok[a] = my_row[a] / group;
    }
    // The wave's first and last token, for the tiles it masks or skips.
    const int w_first = min(wr0, rows - 1) / group;
    const int w_last  = min(wr0 + 32 * kQ - 1, rows - 1) / group;
    const bool idle   = wr0 >= rows;

    const int64_t row0 = first;
    const uint16_t* kh = k + row0 * k_stride + static_cast<int64_t>(kvh) * D;
    const uint16_t* vh = v + row0 * v_stride + static_cast<int64_t>(kvh) * D;
    const int crow = tid / kCpr, cchunk = tid % kCpr;
    u32x4 kreg[kSteps], vreg[kSteps];
    auto load = [&](int i) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int64_t r = min(i * kPN + s * kCopy + crow, n - 1);
            kreg[s] = *reinterpret_cast<const u32x4*>(kh + r * k_stride + 8 * cchunk);
            vreg[s] = *reinterpret_cast<const u32x4*>(vh + r * v_stride + 8 * cchunk);
        }
    };
    auto store = [&](int i) {
        uint8_t* b = lds + (i & 1) * T::kBytes;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int r = s * kCopy + crow;
            *reinterpret_cast<u32x4*>(b + r * T::kKPitch + 16 * cchunk)         = kreg[s];
            *reinterpret_cast<u32x4*>(b + T::kK + r * T::kVPitch + 16 * cchunk) = vreg[s];
        }
    };

    load(0);
    QueryRows<D, kQ> rq;
#pragma unroll
    for (int a = 0; a < kQ; ++a) {
        const int64_t t = my_tok[a];
        rq.load_q(a, q + (row0 + t) * q_stride +
                         (static_cast<int64_t>(kvh) * group + (my_row[a] - my_tok[a] * group)) * D, h);
    }
    rq.clear();
    store(0);

    for (int i = 0; i < n_tiles; ++i) {
        __syncthreads();
        if (i + 1 < n_tiles) {
            load(i + 1);
        }
        const uint8_t* kb = lds + (i & 1) * T::kBytes;
        const uint8_t* vb = kb + T::kK;
        if (!idle && i * kPN <= w_last) {
#pragma unroll
            for (int hf = 0; hf < kPN / 32; ++hf) {
                const int key0 = i * kPN + 32 * hf;
                int       lim[kQ];
#pragma unroll
                for (int a = 0; a < kQ; ++a) {
                    lim[a] = my_tok[a] - key0 - 4 * h;
                }
                rq.template half<false>(kb, vb, hf, lane, scale_log2, nullptr, nullptr,
                                        key0 + 31 > w_first, lim);
            }
        }
        if (i + 1 < n_tiles) {
            store(i + 1);
        }
    }
    if (idle) {
        return;
    }
#pragma unroll
    for (int a = 0; a < kQ; ++a) {
        const float inv = 1.0f / wave_xor_sum(rq.l_run[a], 32);
        const int   r   = again(wr0 + 32 * a + col);
        if (r < rows) {
            const int64_t t = r / group;
            uint16_t* orow = out + (row0 + t) * out_stride +
                             (static_cast<int64_t>(kvh) * group + (r - t * group)) * D;
#pragma unroll
            for (int b = 0; b < D / 32; ++b) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    u32x2 x;
                    x.x = pack_bf16x2(rq.o[a][b][4 * g] * inv, rq.o[a][b][4 * g + 1] * inv);
                    x.y = pack_bf16x2(rq.o[a][b][4 * g + 2] * inv, rq.o[a][b][4 * g + 3] * inv);
                    *reinterpret_cast<u32x2*>(orow + 32 * b + 8 * g + 4 * h) = x;
                }
            }
        }
    }
}

template <int D, int kQ>
hipError_t launch_packed(uint16_t* out, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                         const int* cu, int num_seqs, int num_rows, int64_t out_stride,
                         int64_t q_stride, int64_t k_stride, int64_t v_stride, int hq, int hkv,
                         float scale, hipStream_t stream) {
    constexpr int kBM = 32 * kQ * kPW;
    const int     group = hq / hkv;
    // Most row blocks that the rows can make up in num_seqs sequences.
    const int64_t packed = static_cast<int64_t>(num_rows) * group;
    const int64_t blocks = std::min<int64_t>(packed, packed / kBM + num_seqs);
    flash_packed_kernel<D, kQ><<<dim3(static_cast<unsigned>(blocks * hkv)), kPThr, 0, stream>>>(
        out, q, k, v, cu, num_seqs, num_rows, out_stride, q_stride, k_stride, v_stride, group, hkv,
        scale * kLog2e);
    return hipGetLastError();
}

}  // namespace

hipError_t flash_packed_launch(uint16_t* out, const uint16_t* q, const uint16_t* k,
                               const uint16_t* v, const int* cu_seqlens, int num_seqs,
                               int num_rows, int64_t out_stride, int64_t q_stride,
                               int64_t k_stride, int64_t v_stride, int num_q_heads,
                               int num_kv_heads, int head_dim, float scale, hipStream_t stream) {
#define RTH_PACKED(D, Q)                                                                          \
    return launch_packed<D, Q>(out, q, k, v, cu_seqlens, num_seqs, num_rows, out_stride, q_stride, \
                               k_stride, v_stride, num_q_heads, num_kv_heads, scale, stream)
    switch (head_dim) {
        case 64:
            RTH_PACKED(64, 1);
        case 128:
            RTH_PACKED(128, 1);
        case 256:
            RTH_PACKED(256, 1);
        default:
            return hipErrorInvalidValue;
    }
#undef RTH_PACKED
}

}  // namespace rth
