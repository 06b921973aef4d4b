// Decode attention of a batch: one query token of each sequence over a paged
// OCP E4M3 cache, the sequences sharing the pages of a prefix, gfx950.
//
// For sequence b and q head h of kv head h / G: out[b, h] = sum over keys
// p < lens[b] of softmax_p(scale * q[b, h] . k[p, h / G]) v[p, h / G]; the first
// prefix_len keys lie in the pages of the prefix table for every sequence, the
// others in the sequence's own table. lens[b] <= 0: zeros.
//
// The softmax over both parts is joined from partials (m, l, O per row and part
// of its keys: maximum in log2 units, sum and unnormalized output against it):
//
//  * The prefix: the B * G query rows of a kv head are the columns of one
//    product against its keys. Few rows (prefix_units): 16 rows per
//    workgroup, whose waves take the prefix's tiles in turn and join their
//    results in LDS, so that a partial leaves the workgroup once; the codes go
//    to bf16 operands in each wave's registers. Many rows (prefix_tiles):
//    128 or 256 rows per workgroup share each tile, converted to bf16 once as it is
//    staged in LDS, in attn_tile.hpp's pipeline.
//  * Own keys (own_units, the other workgroups of the launch): the tiles of all
//    sequences are dealt out in runs of equal length, so that long sequences
//    spread over the chip and short ones do not wait for them; a wave per
//    (run, kv head or two). The number of runs fits the scratch whatever the lengths,
//    which live on the device.
//  * A wave's tile: K and V codes and scales of 32 keys (at head_dim 64 of two kv heads), one tile in
//    registers ahead, through the wave's own LDS (no barriers): K rows are read
//    back in the MFMA layout, V transposed by ds_read_b64_tr_b8. E4M3 codes are
//    exact in bf16; the per-key scales are applied in fp32 to the scores and to
//    P, which is rounded to bf16 (half a step, 2^-8 of each weight) for
//    the bf16 MFMA; the row sum takes the fp32 weights.
//  * batch_merge_kernel joins the partials of a row.
//
// 32 q heads on 8, head_dim 128: 4 sequences behind 1000 shared keys 10 us (two
// launches and the chain table -> page -> tile), 32 behind 8192 27 us (the same chain, four
// rounds of tiles and 52 MB), 128 behind 32768 112 us (69 GFLOP, 0.62 PFLOP/s; in the tile
// loop 0.9, the rest is its start, the own keys and 35 MB of partials); 48 sequences of 100 to
// 6000 own keys, head_dim 64, 35 us (bytes: 4.5 TB/s).
#include <algorithm>
#include <type_traits>

#include "attn_tile.hpp"
#include "launch.hpp"

namespace rth {
namespace {

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

    __device__ __forceinline__ bool is_page(int p) const { return p >= 0 && p < num_blocks; }
    // Physical row of key `key` on page `page`.
    __device__ __forceinline__ int64_t row(int page, int key) const {
        return (static_cast<int64_t>(page) << block_shift) + (key & ((1 << block_shift) - 1));
    }
};

__device__ __forceinline__ int prefix_keys(const BatchView& t) {
    if (t.prefix_len == nullptr) {
        return 0;
    }
    const int64_t room = static_cast<int64_t>(t.prefix_blocks) << t.block_shift;
    return static_cast<int>(min(static_cast<int64_t>(max(*t.prefix_len, 0)), room));
}

constexpr int kHalf = 32;   // keys of one score block

// How many of the prefix's keys some sequence sees. The others may never have
// been written, and a weight of 0 takes a NaN from them: they are not read.
__device__ __forceinline__ int prefix_seen(const BatchView& t, int prefix, int lane) {
    int n = 0;
    for (int b0 = 0; b0 < t.num_seqs; b0 += 4 * kWave) {   // four loads on the way
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            n = max(n, t.lens[min(b0 + i * kWave + lane, t.num_seqs - 1)]);
        }
    }
    return min(prefix, uniform(wave_max_i(n)));
}

// Keys [from, to) of a run of tiles of n keys.
struct Keys {
    int from, to;
    __device__ __forceinline__ int tiles(int n) const {
        return to > from ? (to - 1) / n - from / n + 1 : 0;
    }
};
// Sequence b's own keys: behind the prefix, as far as its table goes.
__device__ __forceinline__ Keys own_keys(const BatchView& t, int b, int prefix) {
    const int64_t room = static_cast<int64_t>(t.table_blocks) << t.block_shift;
    return {prefix, static_cast<int>(min(static_cast<int64_t>(t.lens[b]), room))};
}

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

// Tiles per run such that all sequences' runs of that many tiles (the last one
// of each shorter) fit in num_slots slots: the fewest, by bisection, for up to
// kChunks waves of sequences (tiles[c]: of sequence 64 c + lane), else as many as
// always do (128 sequences of 1000 to 4000 keys, 155 -> 123 us).
template <int kChunks>
__device__ __forceinline__ int tiles_per_slot(int total_tiles, const int (&tiles)[kChunks], int num_seqs,
                                              int num_slots) {
    int hi = max(1, (total_tiles + num_slots - num_seqs - 1) / (num_slots - num_seqs));
    if (num_seqs > kChunks * kWave) {
        return hi;
    }
    int lo = max(1, (total_tiles + num_slots - 1) / num_slots);
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        int       runs = 0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            if (c * kWave < num_seqs) {
                runs += (tiles[c] + mid - 1) / mid;
            }
        }
        if (uniform(wave_sum_i(runs)) <= num_slots) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    return hi;
}

// How a launch is split. Prefix: splits of the keys for each block of rows;
// own keys: slots of runs.
struct BatchPlan {
    int q_blocks;      // blocks of 16 q heads of a kv head
    int head_units;    // kv heads, by the tiles of a wave
    int slots;
    int waves;         // of a workgroup
    int splits;        // of the prefix
    int row_blocks;    // of the prefix's rows, of a kv head
    int least, most;   // tiles of a split: least, and up to most of them before the second
                       // half of the splits is used (a partial costs as much as some tiles)
    int tile_waves;    // 0: prefix_units takes the prefix; else the waves of a block of prefix_tiles's rows
};

// Units of one prefix split, and how many splits have keys.
struct PrefixRuns {
    int per, live;
};
__device__ __forceinline__ PrefixRuns prefix_runs(int tiles, const BatchPlan& p) {
    const int half = max(p.splits / 2, 1);
    const int want = min(max((tiles + half - 1) / half, p.least), p.most);
    const int per  = max((tiles + p.splits - 1) / p.splits, want);
    return {per, (tiles + per - 1) / per};
}

// ---- a wave against tiles of its own ------------------------------------------

// A wave's tile: 32 keys of a kv head, at head_dim 64 of two neighbours, so that
// its loads take whole 128-byte lines (48 sequences of 100 to 6000 own keys, one head's
// 64 keys -> two heads' 32: 45 -> 35 us).
template <int D>
struct WaveTile {
    static constexpr int kRowsQ  = 16;                    // query rows of a wave
    static constexpr int kN      = kHalf;                 // keys
    static constexpr int kHeads  = D == 64 ? 2 : 1;
    static constexpr int kPitch  = D + 16;                // bytes per row in LDS
    // V rows 16.. lie this much further: the transposing reads take
    // rows 16 apart at once, which no pitch spreads over the banks.
    static constexpr int kSkew   = D == 64 ? 32 : D == 128 ? 16 : 64;
    static constexpr int kKHead  = kN * kPitch;           // a head's K, and V
    static constexpr int kVHead  = kN * kPitch + kSkew;
    static constexpr int kCpr    = D / 16;                // 16-byte chunks per row of a head
    static constexpr int kLine   = kHeads * kCpr;         // of all heads
    static constexpr int kRows   = kWave / kLine;         // keys of one load
    static constexpr int kLoads  = kN / kRows;
    static constexpr int kV      = kHeads * kKHead;       // where V, and the factors start
    static constexpr int kF      = kV + kHeads * kVHead;
    static constexpr int kBytes  = kF + 2 * kHeads * kN * 4;
    static constexpr int kArea   = kRowsQ * (D + 2);      // floats a wave hands over
    template <int kW>   // waves of a workgroup
    static constexpr int kLds = std::max(kW * kBytes, kW / 2 * kHeads * kArea * 4);
};

// 16 query rows (the columns of v_mfma_f32_16x16x32_bf16, lane l: row l % 16) of a
// wave. (With 32 and v_mfma_f32_32x32x16 the operands and sums take twice the
// registers, so half the waves have loads in flight.)
template <int D>
struct WaveRows {
    using T = WaveTile<D>;
    static constexpr int kKS = D / 32, kDB = D / 16, kHeads = T::kHeads;

    const BatchView& t;
    uint8_t*         lds;   // the wave's
    int              lane, kvh;   // kvh: the first of the tile's heads
    int              heads;       // how many it has
    float            scale_log2;
    bf16x8 qf[kHeads][kKS];   // k-step 2 j + e of lane (row, g): d = 64 j + 16 g + 8 e .. + 7
    f32x4  o[kHeads][kDB];    // lane (row, g): d = 16 b + 4 g .. + 3
    float  m_ref[kHeads], l_run[kHeads];
    bool   start;

    u32x4 kreg[T::kLoads], vreg[T::kLoads];
    float freg[kHeads];
    int   lo, hi;   // rows of the loaded tile that count
    bool  there;

    __device__ __forceinline__ WaveRows(const BatchView& view, uint8_t* l, int ln, int kv, float sc)
        : t(view), lds(l), lane(ln), kvh(kv), heads(min(view.hkv - kv, kHeads)), scale_log2(sc),
          start(true) {
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            m_ref[u] = 0.0f;
            l_run[u] = 0.0f;
#pragma unroll
            for (int b = 0; b < kDB; ++b) {
                o[u][b] = f32x4{};
            }
        }
    }

    // row: the lane's row of the first head; `next`: as far as the next head's. (A head
    // that is not there gets the first one's.)
    __device__ __forceinline__ void load_q(const uint16_t* row, int next) {
        const int g = lane >> 4;
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            const uint16_t* x = row + (u < heads ? u * next : 0);
#pragma unroll
            for (int s = 0; s < kKS; ++s) {
                qf[u][s] = *reinterpret_cast<const bf16x8*>(x + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
            }
        }
    }

    // The table entry of tile i, in every lane.
    __device__ __forceinline__ int entry(const int* table, int i, int to) const {
        const int key = i * T::kN;
        return key < to ? table[key >> t.block_shift] : -1;
    }

    // Codes are read once (nontemporal).
    static __device__ __forceinline__ u32x4 codes(const uint8_t* p, uint32_t off) {
        return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + off));
    }

    // Loads tile i, on page e. Rows outside [from, to) repeat one inside (their V is made
    // zeros as it is staged, and their factors are).
    __device__ __forceinline__ void load(int i, const Keys& keys, int e) {
        const int ln = again(lane);   // (addresses: computed anew for each tile)
        const uint32_t stride = static_cast<uint32_t>(t.hkv) * D;
        const uint32_t r0 = static_cast<uint32_t>(ln / T::kLine);
        const uint32_t chunk = static_cast<uint32_t>(ln % (heads < kHeads ? T::kCpr : T::kLine));
        const int page = uniform(e), key0 = i * T::kN;
        lo    = max(keys.from - key0, 0);
        hi    = min(keys.to - key0, T::kN);
        there = t.is_page(page) && lo < hi;
        if (!there) {   // (the first page's rows, which nothing uses)
            lo = 0;
            hi = T::kN;
        }
        const int64_t  row = t.row(there ? page : 0, key0);
        const int64_t  at  = row * stride + static_cast<int64_t>(kvh) * D;
        const uint8_t* kp  = t.k + at;
        const uint8_t* vp  = t.v + at;
        if (lo == 0 && hi == T::kN) {
            const uint32_t off = r0 * stride + 16u * chunk;
#pragma unroll
            for (int s = 0; s < T::kLoads; ++s) {
                const uint32_t more = static_cast<uint32_t>(s * T::kRows) * stride;
                kreg[s] = codes(kp + more, off);
                vreg[s] = codes(vp + more, off);
            }
        } else {
#pragma unroll
            for (int s = 0; s < T::kLoads; ++s) {
                const int      r   = min(max(s * T::kRows + static_cast<int>(r0), lo), hi - 1);
                const uint32_t off = static_cast<uint32_t>(r) * stride + 16u * chunk;
                kreg[s] = codes(kp, off);
                vreg[s] = codes(vp, off);
            }
        }
        // Factors: lanes 0..31 of K, the others of V.
        const float* f = (ln < 32 ? t.ks : t.vs) + row * t.hkv + kvh +
                         static_cast<uint32_t>(min(max(ln & 31, lo), hi - 1)) * static_cast<uint32_t>(t.hkv);
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            freg[u] = f[u < heads ? u : 0];
        }
    }

    __device__ __forceinline__ void stage() {
        const int ln = again(lane);
        const int r0 = ln / T::kLine, head = ln % T::kLine / T::kCpr, chunk = ln % T::kCpr;
        float*     f    = reinterpret_cast<float*>(lds + T::kF);
        const bool edge = lo > 0 || hi < T::kN;
        uint8_t*   at   = lds + r0 * T::kPitch + 16 * chunk;
#pragma unroll
        for (int s = 0; s < T::kLoads; ++s) {
            const int r = s * T::kRows;
            u32x4     v = vreg[s];
            if (edge && (r + r0 < lo || r + r0 >= hi)) {
                v = u32x4{};
            }
            *reinterpret_cast<u32x4*>(at + head * T::kKHead + r * T::kPitch) = kreg[s];
            *reinterpret_cast<u32x4*>(at + T::kV + head * T::kVHead + r * T::kPitch + (r >= 16 ? T::kSkew : 0)) = v;
        }
        const int  r  = ln & 31;
        const bool in = r >= lo && r < hi;
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            f[(ln < 32 ? 0 : kHeads * T::kN) + u * T::kN + r] = in ? freg[u] * (ln < 32 ? scale_log2 : 1.0f) : 0.0f;
        }
    }

    // The staged keys of head u, of which this lane's row sees rows lo .. hi - 1.
    __device__ __forceinline__ void keys_of(int u, int lo, int hi) {
        const int      ln = again(lane), row = ln & 15, g = ln >> 4;
        const uint8_t* lk = lds + u * T::kKHead;
        const uint8_t* lv = lds + T::kV + u * T::kVHead;
        const float*   ls = reinterpret_cast<const float*>(lds + T::kF) + u * T::kN;
        // Register 4 a + e of a lane: key 16 a + 4 g + e of the tile.
        float s[8];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            pin();   // operand reads ahead of the marks would not fit the registers
            f32x4 x = {};
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(lk + (16 * a + row) * T::kPitch + 64 * j + 16 * g);
                bf16x8 a0, a1;
                e4m3x16_to_bf16x8x2(w, a0, a1);
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, qf[u][2 * j], x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, qf[u][2 * j + 1], x, 0, 0, 0);
            }
            const f32x4 kf = *reinterpret_cast<const f32x4*>(ls + 16 * a + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[4 * a + e] = fmaf(x[e], kf[e], -m_ref[u]);
            }
        }
        if (__any(lo > 0 || hi < T::kN)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = 16 * (e >> 2) + 4 * g + (e & 3);
                s[e]        = r >= lo && r < hi ? s[e] : -INFINITY;
            }
        }
        pin();
        bf16x8 p;
        float  sum;
        auto   weights = [&]() {
            sum = 0.0f;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const f32x4 vf = *reinterpret_cast<const f32x4*>(ls + kHeads * T::kN + 16 * a + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = __builtin_amdgcn_exp2f(s[4 * a + e]);
                    sum += x;
                    p[4 * a + e] = static_cast<__bf16>(x * vf[e]);
                }
            }
        };
        weights();
        // A new reference maximum (lazy, as in attn_tile.hpp).
        const bool high = !(sum <= 0x1p20f);
        if (__any(start || high)) {
            float top = s[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) {
                top = fmaxf(top, s[e]);
            }
            top = wave_xor_max(wave_xor_max(top, 16), 32);
            const bool  need  = wave_xor_max(wave_xor_max(high ? 1.0f : 0.0f, 16), 32) != 0.0f;
            const float up    = start ? (top == -INFINITY ? 0.0f : top) : need ? fmaxf(top, 0.0f) : 0.0f;
            const float alpha = start ? 1.0f : __builtin_amdgcn_exp2f(-up);
            m_ref[u] += up;
            l_run[u] *= alpha;
#pragma unroll
            for (int b = 0; b < kDB; ++b) {
                o[u][b] *= alpha;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[e] -= up;
            }
            weights();
        }
        l_run[u] += sum;
        pin();
        // V^T: lane (d, g), the keys of p: 4 g + 0..3 and 16 + 4 g + 0..3. A group of
        // 16 lanes reads eight keys' 16 d and gets them transposed: ln i points at
        // eight d of key i / 2.
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) i32x2* LdsPtr;
        const int rr = (ln & 15) >> 1;
        const uint8_t* vp = lv + (4 * g + (rr & 3)) * T::kPitch +
                            (rr >> 2) * (16 * T::kPitch + T::kSkew) + 8 * (ln & 1);
#pragma unroll
        for (int b = 0; b < kDB; ++b) {
            const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsPtr)const_cast<uint8_t*>(vp + 16 * b));
            const u32x2 x = {static_cast<uint32_t>(w.x), static_cast<uint32_t>(w.y)};
            o[u][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3x8_to_bf16x8(x), p, o[u][b], 0, 0, 0);
            if (b % 4 == 3) {
                pin();
            }
        }
    }

    // Tiles first, first + step, .. below last over keys [from, to) of a
    // table; this lane's row sees those below `end`.
    __device__ __forceinline__ void run(const int* table, const Keys& keys, int first, int last,
                                        int step, int end) {
        if (first >= last) {
            return;
        }
        int e = entry(table, first, keys.to);
        int next = entry(table, first + step, first + step < last ? keys.to : 0);
        load(first, keys, e);
        for (int i = first; i < last; i += step) {
            const bool is = there;
            e             = next;
            stage();
            if (i + 2 * step < last) {
                next = entry(table, i + 2 * step, keys.to);
            }
            if (i + step < last) {
                load(i + step, keys, e);
            }
            if (is) {
                const int key0 = i * T::kN;
#pragma unroll
                for (int u = 0; u < kHeads; ++u) {
                    if (u < heads) {
                        keys_of(u, keys.from - key0, min(keys.to, end) - key0);
                    }
                }
                start = false;
            }
        }
    }

    __device__ __forceinline__ static float row_sum(float x) {
        return wave_xor_sum(wave_xor_sum(x, 16), 32);
    }

    // m, l (summed over the row's lanes) and O of this lane's row of head u, as one of
    // `rows` partials at `part`.
    __device__ __forceinline__ void write(int u, float* part, int64_t rows, int64_t row, float m, float l) const {
        const int g = lane >> 4;
        if (g == 0) {
            part[row]        = m;
            part[rows + row] = l;
        }
        float* po = part + 2 * rows + row * D + 4 * g;
#pragma unroll
        for (int b = 0; b < kDB; ++b) {
            *reinterpret_cast<f32x4_a4*>(po + 16 * b) = o[u][b];
        }
    }

    // Joins the results of the workgroup's waves into wave 0's, by halves: the
    // upper half of the waves left hands over through LDS. m and l: as write().
    template <int kW>
    __device__ __forceinline__ void join(float* all, int wave, float (&m)[kHeads], float (&l)[kHeads]) {
#pragma unroll
        for (int n = kW / 2; n > 0; n >>= 1) {
            __syncthreads();   // tiles, or the step before, are done with
            // A wave's area, for each head: [D / 16][64 lanes] quads of O, then m and l of 16 rows.
            float* a = all + (wave % n) * kHeads * T::kArea;
            if (wave >= n && wave < 2 * n) {
#pragma unroll
                for (int u = 0; u < kHeads; ++u) {
#pragma unroll
                    for (int b = 0; b < kDB; ++b) {
                        *reinterpret_cast<f32x4*>(a + u * T::kArea + (b * kWave + lane) * 4) = o[u][b];
                    }
                    if (lane < 16) {
                        a[u * T::kArea + 16 * D + lane]      = m[u];
                        a[u * T::kArea + 16 * D + 16 + lane] = l[u];
                    }
                }
            }
            __syncthreads();
            if (wave < n) {
#pragma unroll
                for (int u = 0; u < kHeads; ++u) {
                    const float* x  = a + u * T::kArea;
                    const float  m1 = x[16 * D + (lane & 15)], l1 = x[16 * D + 16 + (lane & 15)];
                    const float top = m1 != m1 ? m1 : fmaxf(m[u], m1);
                    const float f0 = m[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[u] - top);
                    const float f1 = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - top);
                    l[u] = f0 * l[u] + f1 * l1;
                    m[u] = top;
#pragma unroll
                    for (int b = 0; b < kDB; ++b) {
                        const f32x4 y = *reinterpret_cast<const f32x4*>(x + (b * kWave + lane) * 4);
                        o[u][b] = f0 * o[u][b] + f1 * y;
                    }
                }
            }
        }
    }
};

// Workgroup `bid` of the prefix, few rows: (split, block of 16 rows, kv head), the
// waves taking the split's tiles in turn.
template <int D, int kW>
__device__ __forceinline__ void prefix_units(uint8_t* lds, int bid, int prefix,
                                             const uint16_t* __restrict__ q, int64_t q_stride,
                                             const BatchView& t, float* __restrict__ shared,
                                             const BatchPlan& bp, float scale_log2) {
    using T = WaveTile<D>;
    const int tid  = static_cast<int>(threadIdx.x);
    const int wave = uniform(tid / kWave), lane = tid & (kWave - 1), col = lane & 15;
    const int hq   = t.hkv * t.group;
    const int tiles = (prefix + T::kN - 1) / T::kN;
    const PrefixRuns runs = prefix_runs(tiles, bp);
    const int at = uniform(bid / bp.head_units), kvh = (bid - at * bp.head_units) * T::kHeads;
    const int split = uniform(at / bp.row_blocks), rb = at - split * bp.row_blocks;
    if (split >= runs.live) {
        return;
    }
    const int rows = t.num_seqs * t.group;
    const int row  = min(rb * 16 + col, rows - 1);
    const int b = row / t.group, head = kvh * t.group + (row - b * t.group);
    WaveRows<D> w(t, lds + wave * T::kBytes, lane, kvh, scale_log2);
    w.load_q(q + b * q_stride + static_cast<int64_t>(head) * D, t.group * D);
    const int first = split * runs.per;
    w.run(t.prefix_table, Keys{0, prefix_seen(t, prefix, lane)}, first + wave, min(first + runs.per, tiles),
          kW, t.lens[b]);
    const int64_t all = static_cast<int64_t>(bp.splits) * t.num_seqs * hq;
    float m[T::kHeads], l[T::kHeads];
#pragma unroll
    for (int u = 0; u < T::kHeads; ++u) {
        l[u] = w.row_sum(w.l_run[u]);
        m[u] = l[u] == 0.0f ? -INFINITY : w.m_ref[u];
    }
    w.template join<kW>(reinterpret_cast<float*>(lds), wave, m, l);
#pragma unroll
    for (int u = 0; u < T::kHeads; ++u) {
        if (wave == 0 && rb * 16 + col < rows && u < w.heads) {
            w.write(u, shared, all, (static_cast<int64_t>(split) * t.num_seqs + b) * hq + head + u * t.group, m[u],
                    l[u]);
        }
    }
}

// Workgroup `bid` of the own keys: (slot, group of kW units: the kv heads of a tile, block of 16 q heads of each).
template <int D, int kW>
__device__ __forceinline__ void own_units(uint8_t* lds, int bid, int prefix,
                                          const uint16_t* __restrict__ q, int64_t q_stride,
                                          const BatchView& t, float* __restrict__ own,
                                          int* __restrict__ plan, const BatchPlan& bp,
                                          float scale_log2) {
    using T = WaveTile<D>;
    const int tid  = static_cast<int>(threadIdx.x);
    const int wave = uniform(tid / kWave), lane = tid & (kWave - 1), col = lane & 15;
    const int hq   = t.hkv * t.group;
    const int units  = bp.head_units * bp.q_blocks;
    const int slot = uniform((bid * kW + wave) / units), unit = bid * kW + wave - slot * units;
    if (slot >= bp.slots) {
        return;
    }
    const int of = uniform(unit / bp.q_blocks), qb = unit - of * bp.q_blocks, kvh = of * T::kHeads;

    // Which run of which sequence this slot is. Slot 0 writes the plan down.
    constexpr int kChunks = 4;
    int           tiles[kChunks] = {}, total = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int b = c * kWave + lane;
        tiles[c]    = b < t.num_seqs ? own_keys(t, b, prefix).tiles(T::kN) : 0;
        total += tiles[c];
    }
    for (int b0 = kChunks * kWave; b0 < t.num_seqs; b0 += kWave) {
        const int b = b0 + lane;
        total += b < t.num_seqs ? own_keys(t, b, prefix).tiles(T::kN) : 0;
    }
    total         = uniform(wave_sum_i(total));
    const int per = tiles_per_slot(total, tiles, t.num_seqs, bp.slots);
    int seq = -1, run = 0, base = 0;
    for (int b0 = 0; b0 < t.num_seqs; b0 += kWave) {
        const int b    = b0 + lane;
        const int runs = b < t.num_seqs ? (own_keys(t, b, prefix).tiles(T::kN) + per - 1) / per : 0;
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
    seq             = uniform(seq);
    run             = uniform(run);
    const Keys keys = own_keys(t, seq, prefix);
    const int t0 = keys.from / T::kN + run * per;
    const int t1 = min(t0 + per, (keys.to - 1) / T::kN + 1);
    const int head = kvh * t.group + min(qb * 16 + col, t.group - 1);
    WaveRows<D> w(t, lds + wave * T::kBytes, lane, kvh, scale_log2);
    w.load_q(q + seq * q_stride + static_cast<int64_t>(head) * D, t.group * D);
    w.run(t.tables + static_cast<int64_t>(seq) * t.table_blocks, keys, t0, t1, 1, keys.to);
#pragma unroll
    for (int u = 0; u < T::kHeads; ++u) {
        const float l = w.row_sum(w.l_run[u]);
        if (qb * 16 + col < t.group && u < w.heads) {
            w.write(u, own, static_cast<int64_t>(bp.slots) * hq,
                    static_cast<int64_t>(slot) * hq + head + u * t.group, l == 0.0f ? -INFINITY : w.m_ref[u], l);
        }
    }
}

// ---- many rows against the prefix ------------------------------------------------

template <int D>
struct PrefixLds {
    using T = AttnTile<D>;
    __attribute__((aligned(16))) uint8_t tiles[T::kBytes];
    __attribute__((aligned(16))) float   fac[4][2 * T::kN];   // ring of four tiles
};

// Workgroup `bid` of the prefix: (split, block of 32 kW rows, kv head). kG groups of
// kW waves share its tiles, each with a part of the split of its own, and join
// their results in LDS: a split of few rows is done in half the time, and its partial is
// written once.
template <int D, int kW, int kG>
__device__ __forceinline__ void prefix_tiles(PrefixLds<D> (&sm)[kG], int bid, int prefix,
                                             const uint16_t* __restrict__ q, int64_t q_stride,
                                             const BatchView& t, float* __restrict__ partial,
                                             const BatchPlan& bp, float scale_log2) {
    using T              = AttnTile<D>;
    constexpr int kThr   = kW * kWave;     // of a group
    constexpr int kCpr   = D / 16;         // 16-code chunks per row
    constexpr int kCopy  = kThr / kCpr;    // rows of one copy step
    constexpr int kSteps = kCopy < T::kN ? T::kN / kCopy : 1;
    constexpr bool kSome = kCopy > T::kN;  // more threads than chunks
    const int num_splits = bp.splits;
    const int tiles  = (prefix + T::kN - 1) / T::kN;
    const PrefixRuns runs  = prefix_runs(tiles, bp);
    const int at0   = uniform(bid / t.hkv), hb = bid - at0 * t.hkv;
    const int split = uniform(at0 / bp.row_blocks), blk = at0 - split * bp.row_blocks;
    if (split >= runs.live) {
        return;
    }
    const int group = kG == 1 ? 0 : uniform(static_cast<int>(threadIdx.x) / kThr);
    const int tid   = static_cast<int>(threadIdx.x) - group * kThr;
    const int wave = uniform(tid / kWave);
    const int lane = tid & (kWave - 1);
    uint8_t* const lds = sm[group].tiles;
    auto&          fac = sm[group].fac;
    const int col = lane & 31, h = lane >> 5;
    const int kvh  = uniform((t.hkv & 7) == 0 ? (hb & 7) * (t.hkv >> 3) + (hb >> 3) : hb);
    const int rows = t.num_seqs * t.group;
    const int hq   = t.hkv * t.group;
    const int wr0  = (blk * kW + wave) * 32;
    const bool idle = wr0 >= rows;
    const int my_row = min(wr0 + col, rows - 1);
    const int my_seq = my_row / t.group;
    // The split's tiles, and this group's of them (rounds: the first group's).
    const int all_tiles = min(runs.per, tiles - split * runs.per);
    const int rounds    = (all_tiles + kG - 1) / kG;
    const int tile0     = split * runs.per + group * rounds;
    const int n_tiles   = min(rounds, all_tiles - group * rounds);

    int seen_to = prefix;   // (found out below, while the first table entries are on the way)

    // A thread copies 16 codes of a row in each copy step; the rows of a wave
    // lie in one half of the tile, so in one page, and their base is scalar.
    constexpr int kWaveRows = kWave / kCpr;
    static_assert(kHalf % kWaveRows == 0, "a wave's rows of a copy step lie in one half");
    const uint32_t stride = static_cast<uint32_t>(t.hkv) * D;
    u32x4 kreg[kSteps], vreg[kSteps];
    float freg = 0.0f;
    // The pages of a tile's halves, as loaded (in every lane), then as scalars: first
    // rows, and which halves have a page.
    struct Entries {
        int lo, hi;
    };
    struct Pages {
        int64_t lo, hi;
        int     there;
        __device__ __forceinline__ int64_t row(int u) const {
            const int64_t a = lo, b = hi;
            return u != 0 ? b : a;
        }
    };
    auto entries = [&](int i) {
        const int key = (tile0 + i) * T::kN;
        auto of = [&](int k) { return i < n_tiles && k < prefix ? t.prefix_table[k >> t.block_shift] : -1; };
        return Entries{of(key), of(key + kHalf)};
    };
    auto pages = [&](int i, const Entries& e) {
        const int key = (tile0 + i) * T::kN, lo = uniform(e.lo), hi = uniform(e.hi);
        return Pages{t.row(t.is_page(lo) ? lo : 0, key), t.row(t.is_page(hi) ? hi : 0, key + kHalf),
                     (t.is_page(lo) && key < seen_to ? 1 : 0) | (t.is_page(hi) && key + kHalf < seen_to ? 2 : 0)};
    };
    // The row of half u that row r of it reads: past the keys that are seen, the last one.
    auto row_of = [&](int i, int u, int r) {
        return static_cast<uint32_t>(min(r, max(seen_to - 1 - (tile0 + i) * T::kN - u * kHalf, 0)));
    };
    auto load = [&](const uint8_t* x, int i, const Pages& p, u32x4 (&reg)[kSteps]) {
        const int tt = again(tid), crow = tt / kCpr, cchunk = tt % kCpr;   // (computed anew: registers)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int u = kSteps * kCopy / kHalf > 1 || kSome ? (s * kCopy + wave * kWaveRows) / kHalf & 1 : 0;
            // (A half without a page is zeros: its weights are 0, and stay so.)
            reg[s] = u32x4{};
            if ((!kSome || wave * kWaveRows < T::kN) && (p.there >> u & 1) != 0) {
                const uint8_t* base = x + p.row(u) * stride + static_cast<int64_t>(kvh) * D;
                const uint32_t off = row_of(i, u, (s * kCopy + crow) & (kHalf - 1)) * stride + 16u * cchunk;
                reg[s] = *reinterpret_cast<const u32x4*>(base + off);
            }
        }
    };
    // Factors: of K by the first wave, of V by the second.
    auto load_fac = [&](int i, const Pages& p) {
        if (wave < 2) {
            const int      u = lane >> 5;
            const float*   x = (wave == 0 ? t.ks : t.vs) + kvh;
            const int64_t  r = p.row(u) + row_of(i, u, lane & 31);
            freg = (p.there >> u & 1) != 0 ? x[r * t.hkv] * (wave == 0 ? scale_log2 : 1.0f) : 0.0f;
        }
    };
    auto store = [&](uint32_t to, int pitch, const u32x4 (&reg)[kSteps]) {
        const int tt = again(tid), crow = tt / kCpr, cchunk = tt % kCpr;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (!kSome || wave * kWaveRows < T::kN) {
                bf16x8 x, y;
                e4m3x16_to_bf16x8x2(reg[s], x, y);
                uint8_t* at = lds + to + (s * kCopy + crow) * pitch + 32 * cchunk;
                *reinterpret_cast<bf16x8*>(at)      = x;
                *reinterpret_cast<bf16x8*>(at + 16) = y;
            }
        }
    };
    auto store_fac = [&](int i) {
        if (wave < 2) {
            fac[i & 3][wave * T::kN + lane] = freg;
        }
    };

    // pa, pb: pages of tiles i and i + 1 (at iteration i), e2, e3: entries of the two after.
    const Entries e0 = entries(0), e1 = entries(1);
    Entries       e2 = entries(2), e3 = entries(3);
    seen_to  = prefix_seen(t, prefix, lane);
    Pages pa = pages(0, e0), pb = pages(1, e1);
    if (n_tiles > 0) {
        load(t.k, 0, pa, kreg);
        load_fac(0, pa);
    }
    const int my_end = min(prefix, t.lens[my_seq]);   // keys this row sees
    QueryRows<D, true, kW == 8> rq;
    rq.lane = lane;
    rq.load_q(q + my_seq * q_stride +
              (static_cast<int64_t>(kvh) * t.group + (my_row - my_seq * t.group)) * D);
    if (n_tiles > 0) {
        load(t.v, 0, pa, vreg);
        store(T::k_at(0), T::kKPitch, kreg);
        store_fac(0);
    }
    rq.clear();
    {   // The first step multiplies zero weights with the "tile before".
        const u32x4 zero[kSteps] = {};
        store(T::v_at(1), T::kVPitch, zero);
    }
    if (n_tiles > 1) {
        load(t.k, 1, pb, kreg);
        load_fac(1, pb);
    }
    __syncthreads();
    const int key0 = tile0 * T::kN;
    // Halves with keys; a half that reaches past w_end is masked.
    const int mine = idle || n_tiles <= 0 ? -1 : (min(prefix - key0, n_tiles * T::kN) + kHalf - 1) / kHalf;
    int       w_end;
    {
        int m = my_end;
#pragma unroll
        for (int d = 1; d < kHalf; d <<= 1) {
            m = min(m, __shfl_xor(m, d, kWave));
        }
        w_end = __builtin_amdgcn_readfirstlane(m);
    }
    bool seen = false;   // a half with a page
    if (mine > 0) {
        rq.first_scores(lds + T::k_at(0));
    }
    for (int i = 0; i < rounds; ++i) {
        auto half = [&](auto par, uint32_t k_at, uint32_t v_at) {
            constexpr int kPar = decltype(par)::value;
            const int     j    = 2 * i + kPar, at = key0 + 32 * j;
            // (The step past the last half, all of it masked, adds that half's P V.)
            if (j <= mine) {
                rq.head(lds + k_at, lds + v_at, fac[i & 3] + kPar * kHalf);
                const bool is  = j < mine && (pa.there >> kPar & 1) != 0;
                const int  lim = is ? my_end - 1 - at - 4 * h : -1;
                rq.template step<kPar>(lds + k_at, lds + v_at, scale_log2, fac[i & 3] + T::kN + kPar * kHalf,
                                       is && !seen, !is || at + 32 > w_end, lim);
                seen = seen || is;
            }
        };
        half(std::integral_constant<int, 0>{}, T::k_at(i) + 32 * T::kKPitch, T::v_at(i + 1) + 32 * T::kVPitch);
        // K(i + 1) over K(i - 1), V(i) over V(i - 2): last read before the barrier before.
        if (i + 1 < n_tiles) {
            store(T::k_at(i + 1), T::kKPitch, kreg);
            store_fac(i + 1);
        }
        if (i < n_tiles) {
            store(T::v_at(i), T::kVPitch, vreg);
        }
        __syncthreads();
        const Pages pc = pages(i + 2, e2);
        e2 = e3;
        e3 = entries(i + 4);
        if (i + 2 < n_tiles) {
            load(t.k, i + 2, pc, kreg);
            load_fac(i + 2, pc);
        }
        if (i + 1 < n_tiles) {
            load(t.v, i + 1, pb, vreg);
        }
        half(std::integral_constant<int, 1>{}, T::k_at(i + 1), T::v_at(i));
        pa = pb;
        pb = pc;
    }
    if (mine == 2 * rounds) {
        rq.last(lds + T::v_at(rounds - 1) + 32 * T::kVPitch);
    }
    float l = wave_xor_sum(rq.l_run, 32);
    float m = l == 0.0f ? -INFINITY : rq.m_ref;
    if constexpr (kG == 2) {
        // The second group hands over: [D / 8][64 lanes] quads of O, then m and l.
        float* area = reinterpret_cast<float*>(sm) + wave * 32 * (D + 2);
        static_assert(kW * 32 * (D + 2) * 4 <= static_cast<int>(sizeof(sm)), "");
        __syncthreads();
        if (group == 1) {
#pragma unroll
            for (int b = 0; b < D / 32; ++b) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 x = {rq.o[b][4 * g], rq.o[b][4 * g + 1], rq.o[b][4 * g + 2], rq.o[b][4 * g + 3]};
                    *reinterpret_cast<f32x4*>(area + ((b * 4 + g) * kWave + lane) * 4) = x;
                }
            }
            if (h == 0) {
                area[32 * D + col]      = m;
                area[32 * D + 32 + col] = l;
            }
        }
        __syncthreads();
        if (group == 1) {
            return;
        }
        const float m1 = area[32 * D + col], l1 = area[32 * D + 32 + col];
        const float top = m1 != m1 ? m1 : fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        const float f1 = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - top);
        m = top;
        l = f0 * l + f1 * l1;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(area + ((b * 4 + g) * kWave + lane) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    rq.o[b][4 * g + i] = f0 * rq.o[b][4 * g + i] + f1 * x[i];
                }
            }
        }
    }
    if (idle) {
        return;
    }
    // Partials: [splits, B, Hq] m, l, then O.
    const int64_t all = static_cast<int64_t>(num_splits) * t.num_seqs * hq;
    const int     ln = again(lane), r = uniform(wr0) + (ln & 31), h2 = ln >> 5;
    if (r < rows) {
        const int     b   = r / again(t.group);
        const int     g   = r - b * t.group;
        const int64_t row = (static_cast<int64_t>(split) * t.num_seqs + b) * hq + kvh * t.group + g;
        if (h2 == 0) {
            partial[row]       = m;
            partial[all + row] = l;
        }
        float* po = partial + 2 * all + row * D + 4 * h2;
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 x = {rq.o[db][4 * g], rq.o[db][4 * g + 1], rq.o[db][4 * g + 2],
                                 rq.o[db][4 * g + 3]};
                *reinterpret_cast<f32x4_a4*>(po + 32 * db + 8 * g) = x;
            }
        }
    }
}

// Workgroups: first the prefix's, then those of the own keys. kG > 0: the prefix by
// prefix_tiles, two waves per SIMD (head_dim 256: one); kG == 0 and four waves: by
// prefix_units, three (two); kG == 0 and eight waves: there is none, and workgroups of
// eight waves take all heads of a run together where there are as many (48 sequences of 100
// to 6000 keys, one workgroup of eight per compute unit against three of four: 60 -> 54
// us; two tiles ahead instead of one: 54 -> 56).
constexpr int batch_waves(int w, int g) { return w * (g > 0 ? g : 1); }
constexpr int batch_per_simd(int d, int w, int g) {
    return g > 0 ? (d < 256 ? 2 : 1) : w == 8 ? 2 : d < 256 ? 3 : 2;
}
template <int D, int kW, int kG>
__global__ __launch_bounds__(batch_waves(kW, kG) * kWave, batch_per_simd(D, kW, kG)) void batch_kernel(
    const uint16_t* __restrict__ q, int64_t q_stride, BatchView t, float* __restrict__ own,
    int* __restrict__ plan, float* __restrict__ shared, BatchPlan bp, int prefix_wgs,
    float scale_log2) {
    constexpr int kWaves = batch_waves(kW, kG);
    union Lds {
        __attribute__((aligned(16))) uint8_t units[WaveTile<D>::template kLds<kWaves>];
        PrefixLds<D> tiles[kG > 0 ? kG : 1];
    };
    __shared__ std::conditional_t<(kG > 0), Lds, uint8_t[WaveTile<D>::template kLds<kWaves>]> lds;
    uint8_t*  units  = reinterpret_cast<uint8_t*>(&lds);
    const int bid    = static_cast<int>(blockIdx.x);
    const int prefix = prefix_keys(t);
    if constexpr (kG > 0 || kW == 4) {
        if (bid < prefix_wgs) {
            if constexpr (kG > 0) {
                prefix_tiles<D, kW, kG>(lds.tiles, bid, prefix, q, q_stride, t, shared, bp, scale_log2);
            } else {
                prefix_units<D, kWaves>(units, bid, prefix, q, q_stride, t, shared, bp, scale_log2);
            }
            return;
        }
    }
    own_units<D, kWaves>(units, bid - prefix_wgs, prefix, q, q_stride, t, own, plan, bp, scale_log2);
}

// ---- joining a row's partials ------------------------------------------------------

// A workgroup of kW waves joins the partials of a row: each group of D / 4 lanes (four floats a
// lane) every kGroups-th one against a maximum of its own, four on the way
// at a time, so that nothing waits for the maximum of all; then the groups.
template <int D, int kW>
__global__ __launch_bounds__(kW * kWave) void batch_merge_kernel(
    uint16_t* __restrict__ out, int64_t out_stride, BatchView t, const float* __restrict__ own,
    const int* __restrict__ plan, const float* __restrict__ shared, BatchPlan bp) {
    constexpr int kLanes  = D / 4;
    constexpr int kGroups = kW * kWave / kLanes;
    constexpr int kAtOnce = 4;
    __shared__ float                              top_s[kGroups], sum_s[kGroups];
    __shared__ __attribute__((aligned(16))) float acc_s[kGroups][D];
    const int tid = static_cast<int>(threadIdx.x);
    const int hq  = t.hkv * t.group;
    // Rows whose prefix partials the same XCD wrote (prefix_tiles's kv heads): they may be
    // in its L2 still (32 sequences after 8192 keys 26.9 -> 24.7 us, 64 after 2048 27.1 -> 24.3).
    const int wg = static_cast<int>(blockIdx.x);
    const int xcds = bp.tile_waves != 0 && (t.hkv & 7) == 0 ? 8 : 1;
    const int at0 = wg / xcds, part = hq / xcds;
    const int b = uniform(at0 / part), head = at0 - b * part + (wg - at0 * xcds) * part;
    const int first = plan[2 * b], n_own = plan[2 * b + 1];
    const int prefix = prefix_keys(t);
    const int n_tile = bp.tile_waves != 0 ? AttnTile<D>::kN : WaveTile<D>::kN;
    const int n_pre =
        prefix > 0 ? prefix_runs((prefix + n_tile - 1) / n_tile, bp).live : 0;
    const int64_t own_rows = static_cast<int64_t>(bp.slots) * hq;
    const int64_t pre_rows = static_cast<int64_t>(bp.splits) * t.num_seqs * hq;
    const int n = t.lens[b] > 0 ? n_pre + n_own : 0;
    const int group = tid / kLanes, d = 4 * (tid % kLanes);

    float top = -INFINITY, l = 0.0f;
    f32x4 acc = {};
    for (int s0 = group; s0 < n; s0 += kAtOnce * kGroups) {
        float m[kAtOnce], lv[kAtOnce];
        f32x4 v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int  s   = s0 + i * kGroups;
            const bool pre = s < n_pre;
            m[i]           = -INFINITY;
            lv[i]          = 0.0f;
            v[i]           = f32x4{};
            if (s < n) {
                const float*  x    = pre ? shared : own;
                const int64_t rows = pre ? pre_rows : own_rows;
                const int64_t at   = pre ? (static_cast<int64_t>(s) * t.num_seqs + b) * hq + head
                                         : static_cast<int64_t>(first + s - n_pre) * hq + head;
                m[i]  = x[at];
                lv[i] = x[rows + at];
                v[i]  = *reinterpret_cast<const f32x4_a4*>(x + 2 * rows + at * D + d);
            }
        }
        float up = top;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            up = fmaxf(up, m[i]);
        }
        const float f0 = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - up);
        l *= f0;
        acc *= f0;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const float f = m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - up);
            l += f * lv[i];
            acc += f * v[i];
        }
        top = up;
    }
    *reinterpret_cast<f32x4*>(&acc_s[group][d]) = acc;
    if (d == 0) {
        top_s[group] = top;
        sum_s[group] = l;
    }
    __syncthreads();
    if (tid >= kLanes) {
        return;
    }
    float all = -INFINITY;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        all = fmaxf(all, top_s[g]);
    }
    f32x4 o     = {};
    float total = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        // (A sum of NaN alone has no maximum: it passes on by the product.)
        const float f = top_s[g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top_s[g] - all);
        total += f * sum_s[g];
        o += f * *reinterpret_cast<const f32x4*>(&acc_s[g][d]);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    u32x2       x;
    x.x = pack_bf16x2(o[0] * inv, o[1] * inv);
    x.y = pack_bf16x2(o[2] * inv, o[3] * inv);
    *reinterpret_cast<u32x2*>(out + b * out_stride + static_cast<int64_t>(head) * D + d) = x;
}

// `shared`: there is a prefix (its length is known on the device only).
BatchPlan batch_plan(int num_seqs, int hq, int hkv, int head_dim, int cus, bool shared) {
    const int group = hq / hkv, rows = num_seqs * group;
    BatchPlan p;
    p.q_blocks   = (group + 15) / 16;
    p.head_units = head_dim == 64 ? (hkv + 1) / 2 : hkv;
    p.tile_waves = !shared || rows <= 64 ? 0 : head_dim < 256 && rows > 128 ? 8 : 4;
    const int per_block = p.tile_waves == 0 ? 16 : 32 * p.tile_waves;
    p.row_blocks = (rows + per_block - 1) / per_block;
    p.waves = head_dim == 256 || (p.tile_waves == 0 && shared) ? 4 : 8;
    // A tile per group of waves for short prefixes (32 sequences after 1000 keys, tiles
    // of a split 8 -> 2: 23 -> 17 us), eight before more than half the splits write partials
    // (64 after 8192, 4 -> 8: 39 -> 34; head_dim 256, whose tiles take twice as
    // long, 64 after 8000, 4 -> 8: 45 -> 48).
    p.least = p.tile_waves != 0 ? p.waves / p.tile_waves : 3;
    p.most  = p.tile_waves != 0 && head_dim == 256 ? 4 : 8;
    // Rounds of the chip's workgroups: one for a launch of units (three or, at
    // head_dim 256, two per compute unit), half of it the prefix's; prefix tiles
    // take up to one round of their own, one workgroup per compute unit.
    const int round = cus * (p.tile_waves != 0 || p.waves == 8 ? 1 : head_dim == 256 ? 2 : 3);
    const int wgs  = p.row_blocks * (p.tile_waves == 0 ? p.head_units : hkv);
    const int most = p.tile_waves == 0 ? round / 2 : round;
    p.splits         = shared ? std::max(1, std::min(256, most / wgs)) : 0;
    const int left   = shared && p.tile_waves == 0 ? std::max(round - wgs * p.splits, round / 4) : round;
    p.slots = std::max(left * p.waves / (p.head_units * p.q_blocks), num_seqs + std::max(8, num_seqs / 4));
    return p;
}

std::size_t plan_floats(int num_seqs) { return (2 * static_cast<std::size_t>(num_seqs) + 3) & ~std::size_t{3}; }

template <int D>
hipError_t launch_batch(uint16_t* out, int64_t out_stride, const uint16_t* q, int64_t q_stride,
                        const BatchView& t, float* partial, const BatchPlan& p, int cus,
                        float scale, hipStream_t stream) {
    const int   hq         = t.hkv * t.group;
    const float scale_log2 = scale * kLog2e;
    int*        plan       = reinterpret_cast<int*>(partial);
    float*      own        = partial + plan_floats(t.num_seqs);
    float*      shared     = own + static_cast<std::size_t>(p.slots) * hq * (D + 2);
    const int   pre        = p.row_blocks * (p.tile_waves == 0 ? p.head_units : t.hkv) * p.splits;
    const dim3  grid(static_cast<unsigned>(pre + (p.slots * p.head_units * p.q_blocks + p.waves - 1) / p.waves));
    const dim3  block(static_cast<unsigned>(p.waves * kWave));
#define RTH_BATCH(W, G)                                                                        \
    batch_kernel<D, W, G><<<grid, block, 0, stream>>>(q, q_stride, t, own, plan, shared, p, pre, \
                                                      scale_log2)
    if (p.tile_waves == 0 && p.waves == 4) {
        RTH_BATCH(4, 0);
    } else if constexpr (D == 256) {
        RTH_BATCH(4, 1);
    } else if (p.tile_waves == 0) {
        RTH_BATCH(8, 0);
    } else if (p.tile_waves == 4) {
        RTH_BATCH(4, 2);
    } else {
        RTH_BATCH(8, 1);
    }
#undef RTH_BATCH
    // Four waves a row, one where four fill the chip more than once (200 sequences after 3000
    // keys, head_dim 64, 50 -> 44 us; 256 apart 84 -> 80; 128 after 32768 equal).
    const dim3 rows(static_cast<unsigned>(t.num_seqs * hq));
    if (static_cast<int64_t>(t.num_seqs) * hq * 4 <= 32 * static_cast<int64_t>(cus)) {
        batch_merge_kernel<D, 4><<<rows, 4 * kWave, 0, stream>>>(out, out_stride, t, own, plan, shared, p);
    } else {
        batch_merge_kernel<D, 1><<<rows, kWave, 0, stream>>>(out, out_stride, t, own, plan, shared, p);
    }
    return hipGetLastError();
}

}  // namespace

std::size_t batch_scratch_floats(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                                 int cus) {
    std::size_t rows = 0;
    for (const bool shared : {false, true}) {
        const BatchPlan p = batch_plan(num_seqs, num_q_heads, num_kv_heads, head_dim, cus, shared);
        rows = std::max(rows, static_cast<std::size_t>(p.slots) +
                                  static_cast<std::size_t>(p.splits) * num_seqs);
    }
    return plan_floats(num_seqs) + rows * num_q_heads * (head_dim + 2);
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
    const BatchPlan p =
        batch_plan(num_seqs, num_q_heads, num_kv_heads, head_dim, cus, prefix_len != nullptr);
    const BatchView t{k, v, k_scale, v_scale, block_tables, table_blocks, lens, prefix_table,
                      prefix_blocks, prefix_len, num_blocks, block_shift, num_seqs,
                      num_q_heads / num_kv_heads, num_kv_heads};
    switch (head_dim) {
        case 64:
            return launch_batch<64>(out, out_stride, q, q_stride, t, partial, p, cus, scale, stream);
        case 128:
            return launch_batch<128>(out, out_stride, q, q_stride, t, partial, p, cus, scale, stream);
        case 256:
            return launch_batch<256>(out, out_stride, q, q_stride, t, partial, p, cus, scale, stream);
        default:
            return hipErrorInvalidValue;
    }
}

}  // namespace rth
