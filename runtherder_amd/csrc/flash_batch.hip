// Decode attention of a batch: one query token of each sequence over a paged
// OCP E4M3 cache, the sequences sharing the pages of a prefix, gfx950.
//
// For sequence b and q head h of kv head h / G: out[b, h] = sum over keys
// p < lens[b] of softmax_p(scale * scale * q[b, h] . k[p, h / G]) v[p, h / G]; the
// first prefix_len keys lie in the pages of the prefix table for every
// sequence, the others in the sequence's own table. lens[b] <= 0: zeros.
#include <algorithm>

#include "attn_tile.hpp"
#include "launch.hpp"

namespace rth {
namespace {

// Waves of an own-key workgroup: at head_dim 256 a wave needs over 256 registers.
template <int D>
constexpr int kBWaves = D == 256 ? 4 : 8;
constexpr int kBTile  = 32;   // keys per tile of a wave

// Exclusive prefix sum over the wave's lanes, and the total.
__device__ __forceinline__ int wave_exclusive_i(int v, int lane, int& total) {
    int x = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int y = __shfl_up(x, d, kWave);
        x += lane >= d ? y : 0;
    }
    total = __shfl(x, kWave - 1, kWave);
    return x - v;
}

struct BatchView {
    const uint8_t* k;
    const uint8_t* v;
    const float*   ks;
    const float*   vs;
    const int*     tables;
    int            table_blocks;
    const int*     lens;
    const int*     prefix_table;
    int            prefix_blocks;
    const int*     prefix_len;
    int            num_blocks, block_shift, num_seqs, group, hkv;
};

// Own keys [from, to) of sequence b: behind the prefix, as far as its table goes.
struct OwnKeys {
    int from, to;
    __device__ __forceinline__ int tiles() const {
        return to > from ? (to - 1) / kBTile - from / kBTile + 1 : 0;
    }
};
__device__ __forceinline__ OwnKeys own_keys(const BatchView& t, int b, int prefix) {
    const int64_t room = static_cast<int64_t>(t.table_blocks) << t.block_shift;
    return {prefix, static_cast<int>(min(static_cast<int64_t>(t.lens[b]), room))};
}
__device__ __forceinline__ int prefix_keys(const BatchView& t) {
    if (t.prefix_len == nullptr) {
        return 0;
    }
    const int64_t room = static_cast<int64_t>(t.prefix_blocks) << t.block_shift;
    return static_cast<int>(min(static_cast<int64_t>(max(*t.prefix_len, 0)), room));
}

// Tiles per slot such that all sequences' runs of that many tiles (the last one
// shorter) fit in num_slots slots.
__device__ __forceinline__ int tiles_per_slot(int total_tiles, int num_seqs, int num_slots) {
    return max(1, (total_tiles + num_slots - num_seqs - 1) / (num_slots - num_seqs));
}

template <int D>
struct BatchTile {
    static constexpr int kPitch = D + 16;                 // bytes per row in LDS
    static constexpr int kCpr   = D / 16;                 // 16-byte chunks per row
    static constexpr int kRows  = kWave / kCpr;           // rows of one load
    static constexpr int kSteps = kBTile / kRows;
    static constexpr int kBytes = 2 * kBTile * kPitch + 2 * kBTile * 4;
};

template <int D>
__global__ __launch_bounds__(kBWaves<D> * kWave, D == 256 ? 1 : 2) void batch_own_kernel(
    const uint16_t* __restrict__ q, int64_t q_stride, BatchView t, float* __restrict__ partial,
    int* __restrict__ plan, int num_slots, float scale_log2, int nqb) {
    using T = BatchTile<D>;
    constexpr int kKS = D / 16, kDB = D / 32;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBWaves<D>][T::kBytes];

    const int tid  = static_cast<int>(threadIdx.x);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int lane = tid & (kWave - 1);
    const int col = lane & 31, h = lane >> 5;
    const int slot = static_cast<int>(blockIdx.x);
    const int unit = static_cast<int>(blockIdx.y) * kBWaves<D> + wave;   // (kv head, block of q heads)
    if (unit >= t.hkv * nqb) {
        return;
    }
    const int kvh = unit / nqb, qb = unit % nqb;

    const int prefix = prefix_keys(t);
    int       total  = 0;
    for (int b0 = 0; b0 < t.num_seqs; b0 += kWave) {
        const int b = b0 + lane;
        total += wave_sum_i(b < t.num_seqs ? own_keys(t, b, prefix).tiles() : 0);
    }
    const int per = tiles_per_slot(total, t.num_seqs, num_slots);
    int seq = -1, run = 0, base = 0;
    for (int b0 = 0; b0 < t.num_seqs; b0 += kWave) {
        const int b    = b0 + lane;
        const int runs = b < t.num_seqs ? (own_keys(t, b, prefix).tiles() + per - 1) / per : 0;
        int       sum;
        const int before = base + wave_exclusive_i(runs, lane, sum);
        const uint64_t hit = __ballot(slot >= before && slot < before + runs);
        if (slot == 0 && unit == 0 && b < t.num_seqs) {
            plan[2 * b]     = before;
            plan[2 * b + 1] = runs;
        }
        if (hit != 0) {
            const int at = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            seq          = b0 + at;
            run          = slot - __shfl(before, at, kWave);
            if (slot != 0) {
                break;
            }
        }
        base += sum;
    }
    if (seq < 0) {
        return;
    }
    seq                = __builtin_amdgcn_readfirstlane(seq);
    run                = __builtin_amdgcn_readfirstlane(run);
    const OwnKeys keys = own_keys(t, seq, prefix);
    const int t0 = keys.from / kBTile + run * per;
    const int t1 = min(t0 + per, (keys.to - 1) / kBTile + 1);
    const int* table = t.tables + static_cast<int64_t>(seq) * t.table_blocks;

    const int hq      = t.hkv * t.group;
    const int my_head = kvh * t.group + min(qb * 32 + col, t.group - 1);
    const uint16_t* qr = q + seq * q_stride + static_cast<int64_t>(my_head) * D;
    bf16x8 qf[kKS];   // k-step 2 j + e of lane (row, h): d = 32 j + 16 h + 8 e .. + 7
#pragma unroll
    for (int s = 0; s < kKS; ++s) {
        qf[s] = *reinterpret_cast<const bf16x8*>(qr + 32 * (s >> 1) + 16 * h + 8 * (s & 1));
    }

    uint8_t* lk = lds[wave];
    uint8_t* lv = lk + kBTile * T::kPitch;
    float*   ls = reinterpret_cast<float*>(lv + kBTile * T::kPitch);
    const int     lrow = lane / T::kCpr, lchunk = lane % T::kCpr;
    const int64_t stride = static_cast<int64_t>(t.hkv) * D;

    f32x16 o[kDB];
#pragma unroll
    for (int b = 0; b < kDB; ++b) {
        o[b] = f32x16{};
    }
    float m_ref = 0.0f, l_run = 0.0f;
    bool  start = true;
    for (int i = t0; i < t1; ++i) {
        const int key0 = i * kBTile;
        const int page = table[key0 >> t.block_shift];
        if (page < 0 || page >= t.num_blocks) {
            continue;
        }
        const int64_t row0 = (static_cast<int64_t>(page) << t.block_shift) +
                             (key0 & ((1 << t.block_shift) - 1));
        const int lo = max(keys.from - key0, 0), hi = min(keys.to - key0, kBTile);   // rows that count
#pragma unroll
        for (int s = 0; s < T::kSteps; ++s) {
            const int  r    = s * T::kRows + lrow;
            const bool live = r >= lo && r < hi;
            const int64_t at = (row0 + r) * stride + static_cast<int64_t>(kvh) * D + 16 * lchunk;
            u32x4 kx = {}, vx = {};
            if (live) {
                kx = *reinterpret_cast<const u32x4*>(t.k + at);
                vx = *reinterpret_cast<const u32x4*>(t.v + at);
            }
            *reinterpret_cast<u32x4*>(lk + r * T::kPitch + 16 * lchunk) = kx;
            *reinterpret_cast<u32x4*>(lv + r * T::kPitch + 16 * lchunk) = vx;
        }
        {
            const bool    live = col >= lo && col < hi;
            const int64_t at   = (row0 + col) * t.hkv + kvh;
            ls[lane] = live ? (h == 0 ? t.ks[at] * scale_log2 : t.vs[at]) : 0.0f;
        }
        __builtin_amdgcn_wave_barrier();
        f32x16 s = {};
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(lk + col * T::kPitch + 32 * j + 16 * h);
            bf16x8 a0, a1;
            e4m3x16_to_bf16x8x2(w, a0, a1);
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, qf[2 * j], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a1, qf[2 * j + 1], s, 0, 0, 0);
        }
        f32x4 vf[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 kf = *reinterpret_cast<const f32x4*>(ls + 8 * g + 4 * h);
            vf[g]          = *reinterpret_cast<const f32x4*>(ls + 32 + 8 * g + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 8 * g + 4 * h + e;
                s[4 * g + e] = r >= lo && r < hi ? fmaf(s[4 * g + e], kf[e], -m_ref) : -INFINITY;
            }
        }
        bf16x8 p[2];
        float  sum;
        auto   weights = [&]() {
            sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = __builtin_amdgcn_exp2f(s[e]);
                sum += x;
                p[e >> 3][e & 7] = static_cast<__bf16>(x * vf[e >> 2][e & 3]);
            }
        };
        weights();
        if (start || __any(!(sum <= 0x1p20f))) {
            float top = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) {
                top = fmaxf(top, s[e]);
            }
            top               = wave_xor_max(top, 32);
            const float up    = start ? (top == -INFINITY ? 0.0f : top) : fmaxf(top, 0.0f);
            const float alpha = start ? 1.0f : __builtin_amdgcn_exp2f(-up);
            m_ref += up;
            l_run *= alpha;
#pragma unroll
            for (int b = 0; b < kDB; ++b) {
                o[b] *= alpha;
            }
            s -= up;
            weights();
            start = false;
        }
        l_run += sum;
        // V^T: lane (d, h), the keys of p: 16 c + 4 h + 0..3 and 16 c + 8 + 4 h + 0..3.
        const int l16 = lane & 15, rr = l16 >> 1;
        const uint8_t* vp = lv + (4 * h + (rr & 3) + 8 * (rr >> 2)) * T::kPitch +
                            16 * ((lane >> 4) & 1) + 8 * (l16 & 1);
#pragma unroll
        for (int b = 0; b < kDB; ++b) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                typedef int i32x2 __attribute__((ext_vector_type(2)));
                typedef __attribute__((address_space(3))) i32x2* LdsPtr;
                const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (LdsPtr)const_cast<uint8_t*>(vp + 16 * c * T::kPitch + 32 * b));
                const u32x2 u = {static_cast<uint32_t>(w.x), static_cast<uint32_t>(w.y)};
                o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e4m3x8_to_bf16x8(u), p[c], o[b], 0, 0, 0);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    l_run = wave_xor_sum(l_run, 32);
    if (qb * 32 + col < t.group) {
        const int64_t rows = static_cast<int64_t>(num_slots) * hq;
        const int64_t row  = static_cast<int64_t>(slot) * hq + my_head;
        if (h == 0) {
            partial[row]        = start ? -INFINITY : m_ref;
            partial[rows + row] = l_run;
        }
        float* po = partial + 2 * rows + row * D + 4 * h;
#pragma unroll
        for (int b = 0; b < kDB; ++b) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 x = {o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]};
                *reinterpret_cast<f32x4*>(po + 32 * b + 8 * g) = x;
            }
        }
    }
}

// Key tiles of one prefix split, and how many splits have keys.
struct PrefixRuns {
    int per, live;
};
template <int D>
__device__ __forceinline__ PrefixRuns prefix_runs(int prefix, int num_splits) {
    const int tiles = (prefix + AttnTile<D>::kN - 1) / AttnTile<D>::kN;
    const int per   = max((tiles + num_splits - 1) / num_splits, 1);
    return {per, (tiles + per - 1) / per};
}

template <int D, int kQ>
__global__ __launch_bounds__(kPThr, kQ == 1 && D < 256 ? 2 : 1) void batch_prefix_kernel(
    const uint16_t* __restrict__ q, int64_t q_stride, BatchView t, float* __restrict__ partial,
    int num_splits, float scale_log2) {
    using T           = AttnTile<D>;
    constexpr int kBM    = 32 * kQ * kPW;
    constexpr int kCpr   = D / 16;         // 16-code chunks per row
    constexpr int kCopy  = kPThr / kCpr;   // rows of one copy step
    constexpr int kSteps = T::kN / kCopy < 1 ? 1 : T::kN / kCopy;
    static_assert(kCopy <= T::kN, "");
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][T::kBytes];
    __shared__ __attribute__((aligned(16))) float   fac[2][2][T::kN];

    const int prefix = prefix_keys(t);
    const PrefixRuns runs  = prefix_runs<D>(prefix, num_splits);
    const int split = static_cast<int>(blockIdx.y);
    if (split >= runs.live) {
        return;
    }
    const int tid  = static_cast<int>(threadIdx.x);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int lane = tid & (kWave - 1);
    const int col = lane & 31, h = lane >> 5;
    const int bid = static_cast<int>(blockIdx.x);
    const int blk = bid / t.hkv, hb = bid % t.hkv;
    const int kvh  = (t.hkv & 7) == 0 ? (hb & 7) * (t.hkv >> 3) + (hb >> 3) : hb;
    const int rows = t.num_seqs * t.group;
    const int hq   = t.hkv * t.group;
    const int wr0  = blk * kBM + wave * 32 * kQ;
    const bool idle = wr0 >= rows;

    int my_row[kQ], my_end[kQ];   // row, and how many prefix keys it sees
#pragma unroll
    for (int a = 0; a < kQ; ++a) {
        my_row[a] = min(wr0 + 32 * a + col, rows - 1);
        my_end[a] = min(prefix, t.lens[my_row[a] / t.group]);
    }
    const int tile0 = split * runs.per, tile1 = min(tile0 + runs.per, (prefix + T::kN - 1) / T::kN);

    const int crow = tid / kCpr, cchunk = tid % kCpr;
    const int64_t stride = static_cast<int64_t>(t.hkv) * D;
    u32x4 kreg[kSteps], vreg[kSteps];
    float freg;
    auto load = [&](int i) {
        // A row past the prefix, or on a page that is not there, is zeros.
        auto place = [&](int r, int64_t& row) {
            const int key  = i * T::kN + r;
            const int page = key < prefix ? t.prefix_table[key >> t.block_shift] : -1;
            row = (static_cast<int64_t>(page) << t.block_shift) + (key & ((1 << t.block_shift) - 1));
            return page >= 0 && page < t.num_blocks;
        };
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            int64_t row;
            kreg[s] = u32x4{};
            vreg[s] = u32x4{};
            if (place(s * kCopy + crow, row)) {
                const int64_t at = row * stride + static_cast<int64_t>(kvh) * D + 16 * cchunk;
                kreg[s] = *reinterpret_cast<const u32x4*>(t.k + at);
                vreg[s] = *reinterpret_cast<const u32x4*>(t.v + at);
            }
        }
        // Factors: of K by the first kN threads, of V by the next.
        freg = 0.0f;
        int64_t row;
        if (tid < 2 * T::kN && place(tid % T::kN, row)) {
            freg = tid < T::kN ? t.ks[row * t.hkv + kvh] * scale_log2 : t.vs[row * t.hkv + kvh];
        }
    };
    auto store = [&](int i) {
        uint8_t* b = lds[i & 1];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int r = s * kCopy + crow;
            bf16x8 x, y;
            e4m3x16_to_bf16x8x2(kreg[s], x, y);
            *reinterpret_cast<bf16x8*>(b + r * T::kKPitch + 32 * cchunk)      = x;
            *reinterpret_cast<bf16x8*>(b + r * T::kKPitch + 32 * cchunk + 16) = y;
            e4m3x16_to_bf16x8x2(vreg[s], x, y);
            *reinterpret_cast<bf16x8*>(b + T::kK + r * T::kVPitch + 32 * cchunk)      = x;
            *reinterpret_cast<bf16x8*>(b + T::kK + r * T::kVPitch + 32 * cchunk + 16) = y;
        }
        if (tid < 2 * T::kN) {
            fac[i & 1][tid / T::kN][tid % T::kN] = freg;
        }
    };

    load(tile0);
    QueryRows<D, kQ> rq;
#pragma unroll
    for (int a = 0; a < kQ; ++a) {
        const int b = my_row[a] / t.group;
        rq.load_q(a, q + b * q_stride + (static_cast<int64_t>(kvh) * t.group + (my_row[a] - b * t.group)) * D, h);
    }
    rq.clear();
    store(tile0);
    for (int i = tile0; i < tile1; ++i) {
        __syncthreads();
        if (i + 1 < tile1) {
            load(i + 1);
        }
        if (!idle) {
#pragma unroll
            for (int hf = 0; hf < T::kN / 32; ++hf) {
                const int key0 = i * T::kN + 32 * hf;
                const int page = key0 < prefix ? t.prefix_table[key0 >> t.block_shift] : -1;
                if (page < 0 || page >= t.num_blocks) {
                    continue;
                }
                int  lim[kQ];
                bool masked = false;
#pragma unroll
                for (int a = 0; a < kQ; ++a) {
                    lim[a] = my_end[a] - 1 - key0 - 4 * h;
                    masked = masked || my_end[a] < key0 + 32;
                }
                rq.template half<true>(lds[i & 1], lds[i & 1] + T::kK, hf, lane, scale_log2, fac[i & 1][0],
                                       fac[i & 1][1], __any(masked), lim);
            }
        }
        if (i + 1 < tile1) {
            store(i + 1);
        }
    }
    if (idle) {
        return;
    }
    // Partials: [splits, B, Hq] m, l, then O.
    const int64_t all = static_cast<int64_t>(num_splits) * t.num_seqs * hq;
#pragma unroll
    for (int a = 0; a < kQ; ++a) {
        const float l = wave_xor_sum(rq.l_run[a], 32);
        if (wr0 + 32 * a + col < rows) {
            const int     b   = my_row[a] / t.group;
            const int64_t row = (static_cast<int64_t>(split) * t.num_seqs + b) * hq + kvh * t.group +
                                (my_row[a] - b * t.group);
            if (h == 0) {
                partial[row]       = l == 0.0f ? -INFINITY : rq.m_ref[a];
                partial[all + row] = l;
            }
            float* po = partial + 2 * all + row * D + 4 * h;
#pragma unroll
            for (int db = 0; db < D / 32; ++db) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 x = {rq.o[a][db][4 * g], rq.o[a][db][4 * g + 1],
                                     rq.o[a][db][4 * g + 2], rq.o[a][db][4 * g + 3]};
                    *reinterpret_cast<f32x4_a4*>(po + 32 * db + 8 * g) = x;
                }
            }
        }
    }
}

template <int D>
__global__ __launch_bounds__(D) void batch_merge_kernel(uint16_t* __restrict__ out,
                                                       int64_t out_stride, BatchView t,
                                                       const float* __restrict__ own,
                                                       const int* __restrict__ plan,
                                                       int num_slots,
                                                       const float* __restrict__ shared,
                                                       int num_splits) {
    const int hq = t.hkv * t.group;
    const int b = static_cast<int>(blockIdx.x) / hq, head = static_cast<int>(blockIdx.x) % hq;
    const int d = static_cast<int>(threadIdx.x);
    const int first = plan[2 * b], n_own = plan[2 * b + 1];
    const int n_pre = prefix_runs<D>(prefix_keys(t), num_splits).live;
    const int64_t own_rows = static_cast<int64_t>(num_slots) * hq;
    const int64_t pre_rows = static_cast<int64_t>(num_splits) * t.num_seqs * hq;
    float top = -INFINITY, l = 0.0f, acc = 0.0f;
    auto add = [&](const float* part, int64_t rows, int64_t row) {
        const float m = part[row];
        if (m == -INFINITY) {
            return;
        }
        const float up = fmaxf(top, m);
        const float f0 = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - up);
        const float f1 = m != m ? m : __builtin_amdgcn_exp2f(m - up);
        l   = l * f0 + f1 * part[rows + row];
        acc = acc * f0 + f1 * part[2 * rows + row * D + d];
        top = up;
    };
    if (t.lens[b] > 0) {
        for (int s = 0; s < n_pre; ++s) {
            add(shared, pre_rows, (static_cast<int64_t>(s) * t.num_seqs + b) * hq + head);
        }
        for (int s = first; s < first + n_own; ++s) {
            add(own, own_rows, static_cast<int64_t>(s) * hq + head);
        }
    }
    out[b * out_stride + static_cast<int64_t>(head) * D + d] =
        f32_to_bf16_bits(l == 0.0f ? 0.0f : acc / l);
}

// How a launch is split: own slots, prefix splits.
struct BatchPlan {
    int slots, splits, q_blocks;
};
BatchPlan batch_plan(int num_seqs, int hq, int hkv, int cus) {
    const int group = hq / hkv;
    const int nqb   = (group + 31) / 32;
    const int blocks = (num_seqs * group + 32 * kPW - 1) / (32 * kPW) * hkv;
    BatchPlan p;
    p.q_blocks = nqb;
    p.slots    = num_seqs + std::max(8, 8 * cus / (hkv * nqb));
    p.splits   = std::max(1, std::min(256, (2 * cus + blocks - 1) / blocks));
    return p;
}

std::size_t plan_floats(int num_seqs) { return (2 * static_cast<std::size_t>(num_seqs) + 3) & ~std::size_t{3}; }

template <int D>
hipError_t launch_batch(uint16_t* out, int64_t out_stride, const uint16_t* q, int64_t q_stride,
                        const BatchView& t, float* partial, const BatchPlan& p, float scale,
                        hipStream_t stream) {
    const int   hq         = t.hkv * t.group;
    const float scale_log2 = scale * kLog2e;
    int*        plan       = reinterpret_cast<int*>(partial);
    float*      own        = partial + plan_floats(t.num_seqs);
    float*      shared     = own + static_cast<std::size_t>(p.slots) * hq * (D + 2);
    if (t.prefix_len != nullptr) {
        const int blocks = (t.num_seqs * t.group + 32 * kPW - 1) / (32 * kPW) * t.hkv;
        batch_prefix_kernel<D, 1><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(p.splits)),
                                    kPThr, 0, stream>>>(q, q_stride, t, shared, p.splits, scale_log2);
    }
    const int units = t.hkv * p.q_blocks;
    batch_own_kernel<D><<<dim3(static_cast<unsigned>(p.slots),
                               static_cast<unsigned>((units + kBWaves<D> - 1) / kBWaves<D>)),
                          kBWaves<D> * kWave, 0, stream>>>(q, q_stride, t, own, plan, p.slots, scale_log2,
                                                        p.q_blocks);
    batch_merge_kernel<D><<<dim3(static_cast<unsigned>(t.num_seqs * hq)), D, 0, stream>>>(
        out, out_stride, t, own, plan, p.slots, shared, p.splits);
    return hipGetLastError();
}

}  // namespace

std::size_t batch_scratch_floats(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                                 int cus) {
    const BatchPlan p = batch_plan(num_seqs, num_q_heads, num_kv_heads, cus);
    return plan_floats(num_seqs) +
           (static_cast<std::size_t>(p.slots) + static_cast<std::size_t>(p.splits) * num_seqs) *
               num_q_heads * (head_dim + 2);
}

hipError_t flash_batch_launch(uint16_t* out, int64_t out_stride, const uint16_t* q,
                              int64_t q_stride, const uint8_t* k, const uint8_t* v,
                              const float* k_scale, const float* v_scale, const int* block_tables,
                              int table_blocks, int num_blocks, int block_shift, const int* lens,
                              const int* prefix_table, int prefix_blocks, const int* prefix_len,
                              float* partial, int num_seqs, int num_q_heads, int num_kv_heads,
                              int head_dim, float scale, hipStream_t stream) {
    int        cus = 0;
    hipError_t e   = device_cu_count(&cus);
    if (e != hipSuccess) {
        return e;
    }
    const BatchPlan p = batch_plan(num_seqs, num_q_heads, num_kv_heads, cus);
    const BatchView t{k, v, k_scale, v_scale, block_tables, table_blocks, lens, prefix_table,
                      prefix_blocks, prefix_len, num_blocks, block_shift, num_seqs,
                      num_q_heads / num_kv_heads, num_kv_heads};
    switch (head_dim) {
        case 64:
            return launch_batch<64>(out, out_stride, q, q_stride, t, partial, p, scale, stream);
        case 128:
            return launch_batch<128>(out, out_stride, q, q_stride, t, partial, p, scale, stream);
        case 256:
            return launch_batch<256>(out, out_stride, q, q_stride, t, partial, p, scale, stream);
        default:
            return hipErrorInvalidValue;
    }
}

}  // namespace rth
