// The tile step of the batch attention kernels: query rows in registers against
// a tile of keys whose K and V rows lie in LDS as bf16.
#pragma once

#include "batch_common.hpp"

namespace rth {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kPW   = 4;    // waves per workgroup
constexpr int kPThr = kPW * kWave;

// Rows of a K or V tile in LDS: 16 bytes between K rows spread the operand
// reads (16 bytes of 32 rows) over the banks, 64 bytes those of V^T (64 bytes
// of four rows).
template <int D>
struct AttnTile {
    static constexpr int kN      = D == 256 ? 32 : 64;   // keys
    static constexpr int kKPitch = 2 * D + 16;
    static constexpr int kVPitch = 2 * D + 64;
    static constexpr int kK      = kN * kKPitch;
    static constexpr int kBytes  = kK + kN * kVPitch;
};

// 32 kQ query rows of a wave (lane l: rows l % 32 of each block of 32) and what
// they have gathered: S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_32x32x16_bf16, so that a lane owns a query row and the softmax
// needs no lane exchange but for a new maximum; P^T goes from the score
// registers into the second product as it is, because V^T is read
// (ds_read_b64_tr_b16) in the scores' key order. Softmax in base 2, fp32, with a
// lazy reference maximum: it moves at the first keys, and when a row's sum of 32
// weights passes 2^20; one reference for the sum and for O, so the result
// does not depend on it. P is rounded to bf16 (half a step, 2^-9 of each weight)
// for the matrix product, the row sum takes the fp32 values.
template <int D, int kQ>
struct QueryRows {
    static constexpr int kKS = D / 16;   // k-steps of a score
    static constexpr int kDB = D / 32;   // d blocks of O^T

    bf16x8 qf[kQ][kKS];   // k-step s of lane (row, h): d = 16 s + 8 h .. + 7
    f32x16 o[kQ][kDB];
    float  m_ref[kQ], l_run[kQ];
    bool   start;

    __device__ __forceinline__ void clear() {
        start = true;
#pragma unroll
        for (int a = 0; a < kQ; ++a) {
            m_ref[a] = 0.0f;
            l_run[a] = 0.0f;
#pragma unroll
            for (int b = 0; b < kDB; ++b) {
                o[a][b] = f32x16{};
            }
        }
    }

    __device__ __forceinline__ void load_q(int a, const uint16_t* row, int h) {
#pragma unroll
        for (int s = 0; s < kKS; ++s) {
            qf[a][s] = *reinterpret_cast<const bf16x8*>(row + 16 * s + 8 * h);
        }
    }

    // Keys 32 hf .. + 31 of the tile at kb, vb. kScaled: kf, vf hold the tile's
    // key factors (times scale * log2 e) and value factors, else every key's
    // factor is scale_log2. masked: key r of the half counts for block a as
    // far as r <= lim[a] (lim: less 4 h).
    template <bool kScaled>
    __device__ __forceinline__ void half(const uint8_t* kb, const uint8_t* vb, int hf, int lane,
                                         float scale_log2, const float* kf, const float* vf,
                                         bool masked, const int (&lim)[kQ]) {
        using T       = AttnTile<D>;
        const int col = lane & 31, h = lane >> 5;
        if constexpr (D == 256) {   // operand reads ahead of the marks would not fit the registers
            __builtin_amdgcn_sched_barrier(0);
        }
        f32x16    s[kQ];
#pragma unroll
        for (int a = 0; a < kQ; ++a) {
            s[a] = f32x16{};
        }
#pragma unroll
        for (int c = 0; c < kKS; ++c) {
            const bf16x8 x = *reinterpret_cast<const bf16x8*>(kb + (32 * hf + col) * T::kKPitch +
                                                              32 * c + 16 * h);
#pragma unroll
            for (int a = 0; a < kQ; ++a) {
                s[a] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, qf[a][c], s[a], 0, 0, 0);
            }
            if constexpr (D == 256) {
                if (c % 4 == 3) {
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        // Register e of a lane: key 8 (e / 4) + 4 h + e % 4 of the half.
        f32x4 fk[4], fv[4];
        if constexpr (kScaled) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                fk[g] = *reinterpret_cast<const f32x4*>(kf + 32 * hf + 8 * g + 4 * h);
                fv[g] = *reinterpret_cast<const f32x4*>(vf + 32 * hf + 8 * g + 4 * h);
            }
        }
        bf16x8 p[kQ][2];
        float  sum[kQ];
        auto   weights = [&](int a) {
            float t0 = 0.0f, t1 = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = __builtin_amdgcn_exp2f(s[a][e]);
                ((e & 1) != 0 ? t1 : t0) += x;
                p[a][e >> 3][e & 7] = static_cast<__bf16>(kScaled ? x * fv[e >> 2][e & 3] : x);
            }
            sum[a] = t0 + t1;
        };
#pragma unroll
        for (int a = 0; a < kQ; ++a) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[a][e] = fmaf(s[a][e], kScaled ? fk[e >> 2][e & 3] : scale_log2, -m_ref[a]);
            }
            if (masked) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[a][e] = 8 * (e >> 2) + (e & 3) > lim[a] ? -INFINITY : s[a][e];
                }
            }
            weights(a);
            if (start || __any(!(sum[a] <= 0x1p20f))) {
                float top = s[a][0];
#pragma unroll
                for (int e = 1; e < 16; ++e) {
                    top = fmaxf(top, s[a][e]);
                }
                top = wave_xor_max(top, 32);
                const float up    = start ? (top == -INFINITY ? 0.0f : top) : fmaxf(top, 0.0f);
                const float alpha = start ? 1.0f : __builtin_amdgcn_exp2f(-up);
                m_ref[a] += up;
                l_run[a] *= alpha;
#pragma unroll
                for (int b = 0; b < kDB; ++b) {
                    o[a][b] *= alpha;
                }
                s[a] -= up;
                weights(a);
            }
            l_run[a] += sum[a];
        }
        start = false;
        // V^T: lane (d, h), keys 16 c + 4 h .. + 3 and 16 c + 8 + 4 h .. + 3. A
        // group of 16 lanes reads four keys' 16 d and gets them transposed: lane i
        // points at four d of key i / 4.
        const int l16 = lane & 15;
        const uint8_t* vp = vb + (32 * hf + 4 * h + (l16 >> 2)) * T::kVPitch +
                            32 * ((lane >> 4) & 1) + 8 * (l16 & 3);
#pragma unroll
        for (int b = 0; b < kDB; ++b) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                typedef __attribute__((address_space(3))) s16x4* LdsPtr;
                const uint8_t* at = vp + 16 * c * T::kVPitch + 64 * b;
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (LdsPtr)const_cast<uint8_t*>(at));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (LdsPtr)const_cast<uint8_t*>(at + 8 * T::kVPitch));
                const s16x8  xy = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
                const bf16x8 va = __builtin_bit_cast(bf16x8, xy);
#pragma unroll
                for (int a = 0; a < kQ; ++a) {
                    o[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, p[a][c], o[a][b], 0, 0, 0);
                }
            }
            if constexpr (D == 256) {
                if (b % 2 == 1) {
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
};

}  // namespace rth
