// Causal attention over whole prompts, packed one behind the other, gfx950.
//
// For row t of sequence b (cu[b] <= t < cu[b + 1]) and q head h of kv head
// h / G: out[t, h] = sum over cu[b] <= u <= t of softmax_u(scale * q[t, h] .
// k[u, h / G]) * v[u, h / G], from the bf16 K and V rows themselves (no cache).
//
//  * Rows: the G q heads of a kv head are packed token by token (row r of a
//    sequence: token r / G, head r % G), 32 rows per wave, four or eight waves per
//    workgroup. A workgroup finds its (sequence, row block) itself: block w in
//    order of the block's index within its sequence, longest first, so that the
//    last workgroups to start are short ones, whatever mix of lengths the batch
//    holds; no plan, no workspace and one launch.
//  * Keys in tiles of 64, K and V rows through registers into two LDS buffers
//    each: the loads of K(i + 2) and V(i + 1) run under the products of tiles i and i + 1,
//    with one barrier per tile.
//  * The tile loop is attn_tile.hpp's: softmax of half a tile under the
//    products of its neighbours.
//  * A key past a row's diagonal weighs zero, but zero times a non-finite value is
//    NaN: V tiles that reach past a diagonal are stored without their non-finite
//    values, and the rows that do see such a value get it back at the end (1 to
//    3 % of the time; a sequence must not hear what stands behind it).
//
// Bound by the matrix units: 16384 tokens, 32 q heads on 8, head_dim 128, 1.95 to
// 2.03 ms = 1.13 to 1.08 PFLOP/s of the causal products, against 1.38 for a large matrix
// product. Ragged prompts (12 of 40 to 1100 tokens, 97 us) pay beside that 6 of a
// workgroup's 22 us for finding its block, the first tile and the rows of q and out.
#include <algorithm>
#include <type_traits>

#include "attn_tile.hpp"
#include "launch.hpp"

namespace rth {
namespace {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Which (sequence, block of rows) workgroup w of a kv head takes: blocks in
// descending order of their index j within the sequence (their work grows with
// j), within one j in order of the sequences. blocks(b0): the blocks of sequence
// b0 + lane. False: w is past the last block.
struct BlockOf {
    int seq, j;
};
template <typename F>
__device__ __forceinline__ bool find_block(int w, int num_seqs, F blocks, BlockOf& at) {
    // blocks with index >= t
    auto from = [&](int t) {
        int n = 0;
        for (int b0 = 0; b0 < num_seqs; b0 += kWave) {
            n += max(0, blocks(b0) - t);
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
        const bool     mine = blocks(b0) > lo;
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

// The same for up to a wave of sequences (lane b: n blocks): each lane sums for an index of
// its own (one prompt of 200 tokens, against one index after the other, 10.8 -> 10.2 us;
// 30 ragged ones 165 -> 166).
__device__ __forceinline__ bool find_block_of_wave(int w, int num_seqs, int n, int lane, BlockOf& at) {
    int step = 1;
    while (__any(n > step * kWave)) {
        step *= kWave;
    }
    int lo = 0, above = 0;
    for (;; step /= kWave) {
        const int t = lo + lane * step;
        int       from = 0;   // blocks with index >= t
        for (int b = 0; b < num_seqs; ++b) {
            from += max(0, __builtin_amdgcn_readlane(n, b) - t);
        }
        const int over = __popcll(__ballot(from > w));   // (from falls with t)
        if (over == 0) {
            return false;
        }
        above = over < kWave ? __builtin_amdgcn_readlane(from, over) : above;
        lo += (over - 1) * step;
        if (step == 1) {
            break;
        }
    }
    const bool     mine = n > lo;
    const uint64_t hit  = __ballot(mine && lanes_below(__ballot(mine)) == w - above);
    at = {__ffsll(static_cast<unsigned long long>(hit)) - 1, lo};
    return true;
}

template <int D, int kW>   // kW waves of 32 rows
__global__ __launch_bounds__(kW * kWave, D < 256 ? 2 : 1) void flash_packed_kernel(
    uint16_t* __restrict__ out, const uint16_t* __restrict__ q, const uint16_t* __restrict__ k,
    const uint16_t* __restrict__ v, const int* __restrict__ cu, int num_seqs, int num_rows,
    int64_t out_stride, int64_t q_stride, int64_t k_stride, int64_t v_stride, int group, int hkv,
    float scale_log2) {
    using T              = AttnTile<D>;
    constexpr int kThr   = kW * kWave;
    constexpr int kBM    = 32 * kW;
    constexpr int kCpr   = D / 8;         // 16-byte chunks per row
    constexpr int kCopy  = kThr / kCpr;   // rows of one copy step
    constexpr int kSteps = T::kN / kCopy;
    static_assert(T::kBytes >= 4 * kMaxBatchSeqs, "the block counts of a batch fit the tiles");
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::kBytes];
    __shared__ int                                  odd;   // a V tile at the diagonal has values that are not finite

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
    int     first, n;   // the sequence's rows
    {
        auto bound = [&](int b) { return b <= num_seqs ? clamp_rows(cu[b], num_rows) : 0; };
        auto count = [&](int rows) {
            return static_cast<int>((static_cast<int64_t>(max(rows, 0)) * group + kBM - 1) / kBM);
        };
        bool found;
        if (num_seqs <= kWave) {   // every wave by itself, from registers
            const int from = bound(lane), to = bound(lane + 1);
            found = find_block_of_wave(w, num_seqs, lane < num_seqs ? count(to - from) : 0, lane, at);
            if (found) {
                first = __builtin_amdgcn_readlane(from, uniform(at.seq));
                n     = __builtin_amdgcn_readlane(to, uniform(at.seq)) - first;
            }
        } else {
            int* nblk = reinterpret_cast<int*>(lds);
            for (int b = tid; b < num_seqs; b += kThr) {
                nblk[b] = count(bound(b + 1) - bound(b));
            }
            __syncthreads();
            found = find_block(
                w, num_seqs, [&](int b0) { return b0 + lane < num_seqs ? nblk[b0 + lane] : 0; }, at);
            __syncthreads();
            if (found) {
                first = uniform(bound(at.seq));
                n     = uniform(bound(at.seq + 1)) - first;
            }
        }
        if (!found) {
            return;
        }
    }
    const int j     = __builtin_amdgcn_readfirstlane(at.j);
    const int rows  = n * group;
    const int r0    = j * kBM;
    const int n_tiles = (min(r0 + kBM, rows) - 1) / group / T::kN + 1;

    // This lane's row; past the sequence's last it repeats that and stores nothing.
    const int wr0    = r0 + wave * 32;
    const int my_row = min(wr0 + col, rows - 1);
    const int my_tok = my_row / group;
    // The wave's first token (halves past it are masked), and its halves.
    const int w_first = min(wr0, rows - 1) / group;
    const int mine    = wr0 < rows ? (min(wr0 + 31, rows - 1) / group) / 32 + 1 : -1;

    const int64_t   row0 = first;
    const uint16_t* kh   = k + row0 * k_stride + static_cast<int64_t>(kvh) * D;
    const uint16_t* vh   = v + row0 * v_stride + static_cast<int64_t>(kvh) * D;
    const int       crow = tid / kCpr, cchunk = tid % kCpr;
    u32x4 kreg[kSteps], vreg[kSteps];
    // Tile i of x: a scalar base and a 32-bit offset per lane. A row past the
    // sequence's last repeats it: every key past a row's own is masked.
    auto load = [&](const uint16_t* x, int64_t stride, int i, u32x4 (&reg)[kSteps]) {
        const uint8_t* base = reinterpret_cast<const uint8_t*>(x + static_cast<int64_t>(i) * T::kN * stride);
        const uint32_t pitch = 2u * static_cast<uint32_t>(stride);
        const int      last  = n - 1 - i * T::kN;
        if (last >= T::kN - 1) {
            const uint32_t off = static_cast<uint32_t>(crow) * pitch + 16u * static_cast<uint32_t>(cchunk);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                reg[s] = *reinterpret_cast<const u32x4*>(base + static_cast<int64_t>(s * kCopy) * pitch + off);
            }
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int r = min(s * kCopy + crow, last);
                reg[s] = *reinterpret_cast<const u32x4*>(
                    base + (static_cast<uint32_t>(r) * pitch + 16u * static_cast<uint32_t>(cchunk)));
            }
        }
    };
    auto store = [&](uint32_t to, int pitch, const u32x4 (&reg)[kSteps]) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            *reinterpret_cast<u32x4*>(lds + to + (s * kCopy + crow) * pitch + 16 * cchunk) = reg[s];
        }
    };

    // A weight of 0 takes nothing from a finite value, but from an infinity or a
    // NaN it does: in the tiles where some row of the block does not see every key,
    // such values of V are made 0, and given to the rows that see them at the end.
    const int diagonal = r0 / group / T::kN;   // the first such tile
    auto      store_v  = [&](int i) {
        if (i >= diagonal) {
            u16x2 top = {};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, vreg[s][e] & 0x7fff7fffu));
                }
            }
            if (__any(top.x >= 0x7f80 || top.y >= 0x7f80)) {
                odd = 1;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x  = vreg[s][e];
                        const bool     lo = (x & 0x7f80u) == 0x7f80u, hi = (x & 0x7f800000u) == 0x7f800000u;
                        vreg[s][e] = x & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
                    }
                }
            }
        }
        store(T::v_at(i), T::kVPitch, vreg);
    };

    // Row `x` of the wave's 32 (those that exist) in q or out: whole rows of D
    // elements, kRowLanes lanes each, kRowsAt rows at once.
    constexpr int kRowLanes = D / 8, kRowsAt = kWave / kRowLanes, kRowSteps = 32 / kRowsAt;
    constexpr int kRowPitch = 2 * D + 16;
    const int     have  = min(rows - wr0, 32);   // (negative: an idle wave)
    const int     token = uniform(wr0 / group), left = wr0 - token * group;
    const float   part  = 1.0f / static_cast<float>(group);
    auto row_at = [&](int x, int64_t stride) {
        // Exact: (left + x + 1/2) / group lies at least 1 / (2 group) from a whole number.
        const int n = static_cast<int>((static_cast<float>(left + x) + 0.5f) * part);
        return (row0 + token + n) * stride + (static_cast<int64_t>(kvh) * group + (left + x - n * group)) * D;
    };

    load(kh, k_stride, 0, kreg);
    QueryRows<D, false, kW == 8> rq;
    rq.lane = lane;
    if constexpr (kW == 4) {
        // q in whole rows, to the operand layout through LDS (a lane's own row in
        // pieces of 32 bytes: 64 x 128 tokens x 32 heads 63 us, with whole rows 42).
        uint8_t* area = lds + T::v_at(0) + wave * 32 * kRowPitch;
        static_assert(kW * 32 * kRowPitch <= 2 * T::kV, "the waves' rows fit the V tiles");
        const int r = lane / kRowLanes, chunk = lane % kRowLanes;
        u32x4     x[kRowSteps];
        if (have > 0) {
#pragma unroll
            for (int s = 0; s < kRowSteps; ++s) {
                x[s] = *reinterpret_cast<const u32x4*>(
                    q + row_at(min(s * kRowsAt + r, have - 1), q_stride) + 8 * chunk);
            }
#pragma unroll
            for (int s = 0; s < kRowSteps; ++s) {
                *reinterpret_cast<u32x4*>(area + (s * kRowsAt + r) * kRowPitch + 16 * chunk) = x[s];
            }
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                rq.qf[c] = *reinterpret_cast<const bf16x8*>(area + col * kRowPitch + 32 * c + 16 * h);
            }
        }
        load(vh, v_stride, 0, vreg);
        __syncthreads();
    } else {
        if (have > 0) {
            rq.load_q(q + row_at(min(col, have - 1), q_stride));
        }
        load(vh, v_stride, 0, vreg);
    }
    rq.clear();
    store(T::k_at(0), T::kKPitch, kreg);
    // The first step multiplies zero weights with the "tile before".
    {
        const u32x4 zero[kSteps] = {};
        store(T::v_at(1), T::kVPitch, zero);
    }
    if (tid == 0) {
        odd = 0;
    }
    if (n_tiles > 1) {
        load(kh, k_stride, 1, kreg);
    }
    __syncthreads();
    if (mine > 0) {
        rq.first_scores(lds + T::k_at(0));
    }
    for (int i = 0; i < n_tiles; ++i) {
        auto half = [&](auto par, uint32_t k_at, uint32_t v_at) {
            constexpr int kPar = decltype(par)::value;
            const int     j    = 2 * i + kPar;
            // (The step past the last half, all of it masked, adds that half's P V.)
            if (j <= mine) {
                rq.head(lds + k_at, lds + v_at);
                rq.template step<kPar>(lds + k_at, lds + v_at, scale_log2, nullptr, j == 0,
                                       32 * j + 31 > w_first, my_tok - 32 * j - 4 * h);
            }
        };
        half(std::integral_constant<int, 0>{}, T::k_at(i) + 32 * T::kKPitch, T::v_at(i + 1) + 32 * T::kVPitch);
        // K(i + 1) over K(i - 1), V(i) over V(i - 2): last read before the barrier before.
        if (i + 1 < n_tiles) {
            store(T::k_at(i + 1), T::kKPitch, kreg);
        }
        store_v(i);
        __syncthreads();
        if (i + 2 < n_tiles) {
            load(kh, k_stride, i + 2, kreg);
        }
        if (i + 1 < n_tiles) {
            load(vh, v_stride, i + 1, vreg);
        }
        half(std::integral_constant<int, 1>{}, T::k_at(i + 1), T::v_at(i));
    }
    if (mine == 2 * n_tiles) {
        rq.last(lds + T::v_at(n_tiles - 1) + 32 * T::kVPitch);
    }
    if (mine > 0 && odd != 0) {   // (every store_v lies before a barrier of the loop)
        for (int u = diagonal * T::kN; u <= min(wr0 + 31, rows - 1) / group; ++u) {
            const uint16_t* vr = vh + static_cast<int64_t>(u) * v_stride + 4 * h;
#pragma unroll
            for (int b = 0; b < D / 32; ++b) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = bf16_to_f32(vr[32 * b + 8 * (e >> 2) + (e & 3)]);
                    if (u <= my_tok && !(fabsf(x) < INFINITY)) {
                        rq.o[b][e] += x;
                    }
                }
            }
        }
    }
    // O to bf16 rows in LDS, stored as whole rows.
    const float inv = 1.0f / wave_xor_sum(rq.l_run, 32);
    __syncthreads();   // the tiles are done with
    if (mine < 0) {
        return;
    }
    static_assert(kW * 32 * kRowPitch <= T::kBytes, "the waves' rows fit the tiles");
    const int ln   = again(lane);
    uint8_t*  area = lds + wave * 32 * kRowPitch;
    uint8_t*  to   = area + (ln & 31) * kRowPitch + 8 * (ln >> 5);
#pragma unroll
    for (int b = 0; b < D / 32; ++b) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            u32x2 x;
            x.x = pack_bf16x2(rq.o[b][4 * g] * inv, rq.o[b][4 * g + 1] * inv);
            x.y = pack_bf16x2(rq.o[b][4 * g + 2] * inv, rq.o[b][4 * g + 3] * inv);
            *reinterpret_cast<u32x2*>(to + 64 * b + 16 * g) = x;
        }
    }
    const int r = ln / kRowLanes, chunk = ln % kRowLanes;
#pragma unroll
    for (int s = 0; s < kRowSteps; ++s) {
        const int x = s * kRowsAt + r;
        if (x < have) {
            *reinterpret_cast<u32x4*>(out + row_at(x, out_stride) + 8 * chunk) =
                *reinterpret_cast<const u32x4*>(area + x * kRowPitch + 16 * chunk);
        }
    }
}

template <int D, int kW>
hipError_t launch_packed(uint16_t* out, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                         const int* cu, int num_seqs, int num_rows, int64_t out_stride,
                         int64_t q_stride, int64_t k_stride, int64_t v_stride, int hq, int hkv,
                         float scale, hipStream_t stream) {
    constexpr int kBM = 32 * kW;
    const int     group = hq / hkv;
    // Most row blocks that the rows can make up in num_seqs sequences.
    const int64_t packed = static_cast<int64_t>(num_rows) * group;
    const int64_t blocks = std::min<int64_t>(packed, packed / kBM + num_seqs);
    flash_packed_kernel<D, kW><<<dim3(static_cast<unsigned>(blocks * hkv)), kW * kWave, 0, stream>>>(
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
    int        cus = 0;
    hipError_t e   = device_cu_count(&cus);
    if (e != hipSuccess) {
        return e;
    }
    // Eight waves a workgroup (256 rows, one workgroup of two waves per SIMD: half the
    // copies of K and V per row, and the wave priority) where there are long
    // sequences and 1.75 workgroups per compute unit of them; else four (128 rows, two
    // workgroups per compute unit), whose blocks waste less at the diagonal and even out
    // better. Four / eight, us: 1 x 8192 tokens, 32 heads 552 / 495, 1 x 4096 160 / 135,
    // 4 x 2000 156 / 145, 4 x 2000 of 16 heads 86 / 79, but 8 x 1000 94 / 95, 16 x 500
    // 64 / 73, 1 x 2048 54 / 57, 1 x 4096 of 16 heads 99 / 103; head_dim 64 1 x 4096
    // 114 / 100, 16 x 500 44 / 46.
    const int64_t wide = static_cast<int64_t>(num_rows) * num_q_heads / 256;
    const bool    eight = num_rows / num_seqs >= 1500 && 4 * wide >= 7 * static_cast<int64_t>(cus);
#define RTH_PACKED(D, W)                                                                          \
    return launch_packed<D, W>(out, q, k, v, cu_seqlens, num_seqs, num_rows, out_stride, q_stride, \
                               k_stride, v_stride, num_q_heads, num_kv_heads, scale, stream)
    switch (head_dim) {
        case 64:
            if (eight) {
                RTH_PACKED(64, 8);
            }
            RTH_PACKED(64, 4);
        case 128:
            if (eight) {
                RTH_PACKED(128, 8);
            }
            RTH_PACKED(128, 4);
        case 256:
            RTH_PACKED(256, 4);
        default:
            return hipErrorInvalidValue;
    }
#undef RTH_PACKED
}

}  // namespace rth
