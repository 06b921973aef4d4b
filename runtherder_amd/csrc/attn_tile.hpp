// The tile loop of the batch attention kernels: query rows in registers against
// tiles of keys whose K and V rows lie in LDS as bf16.
#pragma once

#include "batch_common.hpp"

namespace rth {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Rows of a K or V tile in LDS: 16 bytes between K rows spread the operand
// reads (16 bytes of 32 rows) over the banks, 64 bytes those of V^T (64 bytes
// of four rows). K and V have two buffers each, tile i in buffer i % 2.
template <int D>
struct AttnTile {
    static constexpr int kN      = 64;   // keys
    static constexpr int kKPitch = 2 * D + 16;
    static constexpr int kVPitch = 2 * D + 64;
    static constexpr int kK      = kN * kKPitch;
    static constexpr int kV      = kN * kVPitch;
    static constexpr int kBytes  = 2 * (kK + kV);
    static __device__ __forceinline__ uint32_t k_at(int tile) { return (tile & 1) * kK; }
    static __device__ __forceinline__ uint32_t v_at(int tile) { return 2 * kK + (tile & 1) * kV; }
};

// Keeps the instruction scheduler from moving anything across.
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

// 32 query rows of a wave (lane l: row l % 32) and what they have gathered.
// S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_bf16, so that a lane
// owns a query row and the softmax needs no lane exchange but for a new maximum;
// P^T goes from the score registers into the second product as it is, because
// V^T is read (ds_read_b64_tr_b16) in the scores' key order. Softmax in base 2,
// fp32, with a lazy reference maximum: it moves at the first keys, and when a
// row's sum of 32 weights passes 2^20; one reference for the sum and for O, so
// the result does not depend on it. P is rounded to bf16 (half a step, 2^-8 of
// each weight) for the matrix product, the row sum takes the fp32 values.
//
// Software pipelined by halves of a tile (32 keys): one step does the softmax
// of half j under the P V products of half j - 1 and the scores of half j + 1,
// which alternate (neither waits for the other) in the order written here.
// kPrio (one workgroup of two waves per SIMD): a wave holds priority over the
// first two thirds of a step, so that it does not give up its place between
// its MFMAs; held to the end, the other wave's came in too late.
// kScaled: every key has a factor of its own for its scores (times scale *
// log2 e) and one for its values, read from LDS; else all share scale_log2.
template <int D, bool kScaled, bool kPrio>
struct QueryRows {
    using T = AttnTile<D>;
    static constexpr int kSteps = D / 16;   // MFMAs of a half's scores, and of its P V
    static constexpr int kDB    = D / 32;   // d blocks of O^T
    static constexpr int kAhead = 3;        // operand reads ahead of their MFMA

    bf16x8 qf[kSteps];   // k-step c of lane (row, h): d = 16 c + 8 h .. + 7
    f32x16 o[kDB];
    f32x16 s[2];         // scores of half j in s[j % 2]
    bf16x8 p[2];         // P^T of the half before
    bf16x8 ka[kAhead + 1], va[kAhead + 1];
    f32x4  fk[4];        // key factors of half j
    float  m_ref, l_run;
    int    lane;

    __device__ __forceinline__ void clear() {
        m_ref = 0.0f;
        l_run = 0.0f;
#pragma unroll
        for (int b = 0; b < kDB; ++b) {
            o[b] = f32x16{};
        }
        p[0] = bf16x8{};
        p[1] = bf16x8{};
    }

    __device__ __forceinline__ void load_q(const uint16_t* row) {
        const int h = lane >> 5;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            qf[c] = *reinterpret_cast<const bf16x8*>(row + 16 * c + 8 * h);
        }
    }

    // K operand of k-step c of the half whose K rows start at `at`: lane
    // (key, h), d = 16 c + 8 h .. + 7.
    __device__ __forceinline__ void read_k(const uint8_t* at, int c) {
        ka[c & kAhead] = *reinterpret_cast<const bf16x8*>(at + (lane & 31) * T::kKPitch + 32 * c +
                                                          16 * (lane >> 5));
    }
    // V^T operand of MFMA c of a half's P V (d block c % kDB, 16 keys c / kDB):
    // lane (d, h), keys 4 h .. + 3 and 8 + 4 h .. + 3 of them. A group of 16
    // lanes reads four keys' 16 d and gets them transposed: lane i points at four
    // d of key i / 4.
    __device__ __forceinline__ void read_v(const uint8_t* at, int c) {
        typedef __attribute__((address_space(3))) s16x4* LdsPtr;
        const int      l16 = lane & 15;
        const uint8_t* x   = at + (4 * (lane >> 5) + (l16 >> 2)) * T::kVPitch +
                           32 * ((lane >> 4) & 1) + 8 * (l16 & 3) + 16 * (c / kDB) * T::kVPitch +
                           64 * (c % kDB);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)const_cast<uint8_t*>(x));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (LdsPtr)const_cast<uint8_t*>(x + 8 * T::kVPitch));
        const s16x8 ab = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        va[c & kAhead] = __builtin_bit_cast(bf16x8, ab);
    }
    __device__ __forceinline__ void qk(f32x16& x, int c) {
        x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[c & kAhead], qf[c], c == 0 ? f32x16{} : x, 0, 0, 0);
    }
    __device__ __forceinline__ void pv(int c) {
        o[c % kDB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[c & kAhead], p[c / kDB], o[c % kDB], 0, 0, 0);
    }

    // The reads that a step starts with: operands, and (kScaled) the key factors kf
    // of half j.
    __device__ __forceinline__ void head(const uint8_t* k_at, const uint8_t* v_at,
                                         const float* kf = nullptr) {
#pragma unroll
        for (int c = 0; c < kAhead; ++c) {
            read_v(v_at, c);
            read_k(k_at, c);
            if constexpr (kScaled) {
                if (c == 0) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        fk[g] = *reinterpret_cast<const f32x4*>(kf + 8 * g + 4 * (lane >> 5));
                    }
                }
            }
        }
    }

    // Scores of the first half, before the first step.
    __device__ __forceinline__ void first_scores(const uint8_t* k_at) {
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            read_k(k_at, c);
            qk(s[0], c);
        }
    }

    // Softmax of half j (in s[kPar], kPar = j % 2), P V of half j - 1 (V rows from v_at),
    // scores of half j + 1 (K rows from k_at), after head(k_at, v_at, kf).
    // masked: key r of half j counts as far as r <= lim (lim: less 4 h). vf: the
    // value factors of half j.
    template <int kPar>
    __device__ __forceinline__ void step(const uint8_t* k_at, const uint8_t* v_at, float scale_log2,
                                         const float* vf, bool start, bool masked, int lim) {
        f32x16&   x = s[kPar];
        f32x16&   y = s[kPar ^ 1];
        const int h = lane >> 5;
        f32x4     fv[4];
        bf16x8    pn[2];
        float     sum[2] = {0.0f, 0.0f};
        // Register e of a lane: key 8 (e / 4) + 4 h + e % 4 of the half.
        auto scale4 = [&](int g) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[4 * g + e] = fmaf(x[4 * g + e], kScaled ? fk[g][e] : scale_log2, -m_ref);
            }
        };
        auto exp4 = [&](int g) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = __builtin_amdgcn_exp2f(x[4 * g + e]);
                sum[e & 1] += w[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pn[g >> 1][4 * (g & 1) + e] = static_cast<__bf16>(kScaled ? w[e] * fv[g][e] : w[e]);
            }
        };
        if constexpr (kPrio) {
            __builtin_amdgcn_s_setprio(1);
        }
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            pv(c);
            if (c + kAhead < kSteps) {
                read_v(v_at, c + kAhead);
            }
            if (c == 1) {
                scale4(2);
                scale4(3);
            }
            pin();
            if (c == 1 && masked) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    x[e] = 8 * (e >> 2) + (e & 3) > lim ? -INFINITY : x[e];
                }
            }
            qk(y, c);
            if (c + kAhead < kSteps) {
                read_k(k_at, c + kAhead);
            }
            if (c == 0) {
                scale4(0);
                scale4(1);
            }
            if constexpr (kScaled) {
                if (c <= 1) {
#pragma unroll
                    for (int g = 2 * c; g < 2 * c + 2; ++g) {
                        fv[g] = *reinterpret_cast<const f32x4*>(vf + 8 * g + 4 * h);
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (c == 2 + g * (kSteps - 2) / 4) {
                    exp4(g);
                }
            }
            pin();
            if constexpr (kPrio) {
                if (c == 2 * kSteps / 3) {
                    __builtin_amdgcn_s_setprio(0);
                }
            }
        }
        const bool high = !(sum[0] + sum[1] <= 0x1p20f);
        if (__any(start || high)) {
            float top = x[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) {
                top = fmaxf(top, x[e]);
            }
            top = wave_xor_max(top, 32);
            // (Rows that need no new reference keep theirs: a row's result does not
            // depend on the others of its wave.)
            const bool  need  = wave_xor_max(high ? 1.0f : 0.0f, 32) != 0.0f;
            const float up    = start ? (top == -INFINITY ? 0.0f : top) : need ? fmaxf(top, 0.0f) : 0.0f;
            const float alpha = start ? 1.0f : __builtin_amdgcn_exp2f(-up);
            m_ref += up;
            l_run *= alpha;
#pragma unroll
            for (int b = 0; b < kDB; ++b) {
                o[b] *= alpha;
            }
            x -= up;
            sum[0] = sum[1] = 0.0f;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                exp4(g);
            }
        }
        l_run += sum[0] + sum[1];
        p[0] = pn[0];
        p[1] = pn[1];
    }

    // P V of the last half.
    __device__ __forceinline__ void last(const uint8_t* v_at) {
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            read_v(v_at, c);
            pv(c);
        }
    }
};

}  // namespace rth
