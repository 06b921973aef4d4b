// Drives the C++ layer's batch calls as a serving loop does: prompts packed
// one behind the other, their K and V into pages, a sequence freed, another
// forked, decode steps over the shared pages, the parents freed, the pool
// compacted, one more step. Outputs are checked against 64-bit attention over
// the oracle's codes. Needs a GPU; run by tests/test_gpu_batch_flow.py.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include <runtherder/attention/batch.h>
#include <runtherder/engine/page_pool.h>
#include <runtherder/engine/paged_kv_cache.h>

#include "rth_oracle.h"

using runtherder::attention::AttnConfig;
using runtherder::attention::BatchAttention;
using runtherder::engine::PagedKVCache;
using runtherder::engine::PagePool;

namespace {

constexpr int   kHq = 8, kHkv = 2, kD = 64, kLayers = 2, kBlock = 64, kWidth = 4, kPages = 24;
constexpr float kScale = 0.125f;

template <typename T>
struct Dev {
    explicit Dev(const std::vector<T>& h) : n(h.size()), p(runtherder::device::make_device_unique<T>(n)) { set(h); }
    void set(const std::vector<T>& h) {
        RUNTHERDER_HIP_CHECK(hipMemcpy(p.get(), h.data(), n * sizeof(T), hipMemcpyHostToDevice));
    }
    std::vector<T> get() const {
        std::vector<T> h(n);
        RUNTHERDER_HIP_CHECK(hipMemcpy(h.data(), p.get(), n * sizeof(T), hipMemcpyDeviceToHost));
        return h;
    }
    T*                                     ptr() const { return p.get(); }
    std::size_t                            n;
    runtherder::device::DeviceUniquePtr<T> p;
};

__hip_bfloat16*       bf(const Dev<uint16_t>& d) { return reinterpret_cast<__hip_bfloat16*>(d.ptr()); }

std::vector<uint16_t> normal(std::size_t n, uint64_t seed) {
    std::vector<uint16_t> x(n);
    rth_ref_fill_normal_bf16(x.data(), static_cast<int64_t>(n), seed);
    return x;
}

// Keys and values of one sequence, [keys][Hkv][D].
struct Rows {
    std::vector<float> k, v;
    int                keys() const { return static_cast<int>(k.size()) / (kHkv * kD); }
    void push(const uint16_t* kr, const uint16_t* vr, bool quantize) {
        add(k, kr, quantize);
        add(v, vr, quantize);
    }
    static void add(std::vector<float>& to, const uint16_t* x, bool quantize) {
        uint8_t code[kHkv * kD];
        float   s[kHkv];
        if (quantize) {
            rth_ref_quantize_kv_fp8(code, s, x, 0, kHkv, kHkv, kD);
        }
        for (int i = 0; i < kHkv * kD; ++i) {
            to.push_back(quantize ? rth_ref_e4m3_decode(code[i]) * s[i / kD] : rth_ref_bf16_to_f32(x[i]));
        }
    }
};

// Worst |got - want| against its bound: half a bf16 step (2^-8) of the output, the
// same of every weight (P is rounded to bf16), and the fp32 of scores and sums, 64 *
// 2^-24 per unit of the largest score of about 32 (log2 units).
double check(const uint16_t* got, const uint16_t* q, const Rows& rows, int keys) {
    double worst = 0.0;
    for (int h = 0; h < kHq; ++h) {
        const int           kvh = h / (kHq / kHkv);
        std::vector<double> p(keys);
        double              m = -1e300, sum = 0.0;
        for (int u = 0; u < keys; ++u) {
            double s = 0.0;
            for (int d = 0; d < kD; ++d) {
                s += static_cast<double>(rth_ref_bf16_to_f32(q[h * kD + d])) * rows.k[(u * kHkv + kvh) * kD + d];
            }
            p[u] = s * kScale;
            m    = std::fmax(m, p[u]);
        }
        for (double& x : p) {
            x = std::exp(x - m);
            sum += x;
        }
        for (int d = 0; d < kD; ++d) {
            double o = 0.0, w = 0.0;
            for (int u = 0; u < keys; ++u) {
                const double x = p[u] / sum * rows.v[(u * kHkv + kvh) * kD + d];
                o += x;
                w += std::fabs(x);
            }
            const double tol = (std::fabs(o) + w) / 256 + w * 2048.0 / 16777216.0 + 1e-30;
            const double err = std::fabs(rth_ref_bf16_to_f32(got[h * kD + d]) - o) / tol;
            worst            = err <= worst ? worst : err;   // (NaN counts)
        }
    }
    return worst;
}

int expect(bool ok, const char* what, double x) {
    std::printf("%s %.4g %s\n", what, x, ok ? "OK" : "FAIL");
    std::fflush(stdout);
    return ok ? 0 : 1;
}

int run() {
    int                    fails = 0;
    const std::vector<int> lens = {70, 1, 133}, cu = {0, 70, 71, 204};
    const int              rows = cu.back(), kv = kHkv * kD, qo = kHq * kD;
    const auto             q = normal(static_cast<std::size_t>(rows) * qo, 1);
    // K and V are slices of one projection's rows.
    const auto  kvr = normal(static_cast<std::size_t>(rows) * 2 * kv, 2);
    hipStream_t stream = nullptr;
    RUNTHERDER_HIP_CHECK(hipStreamCreate(&stream));
    PagedKVCache   cache(kLayers, kPages, kBlock, kHkv, kD);
    PagePool       pool(kPages, kBlock);
    BatchAttention attn(AttnConfig{kHq, kHkv, kD, kScale}, 4);

    Dev<uint16_t> dq(q), dkv(kvr), dout(std::vector<uint16_t>(q.size()));
    Dev<int>      dcu(cu), dlens(std::vector<int>(3, 0)), dnew(lens), at(std::vector<int>(3, 0));
    Dev<int>      tables(std::vector<int>(3 * kWidth, -1));
    attn.run_packed(bf(dout), bf(dq), bf(dkv), bf(dkv) + kv, dcu.ptr(), 3, rows, stream, 0, 2 * kv, 2 * kv);
    pool.reserve(tables.ptr(), kWidth, dlens.ptr(), dnew.ptr(), 3, stream);
    for (int layer = 0; layer < kLayers; ++layer) {
        cache.append_batch(layer, bf(dkv), bf(dkv) + kv, dcu.ptr(), at.ptr(), 3, rows,
                           tables.ptr(), kWidth, stream, 2 * kv, 2 * kv);
    }
    RUNTHERDER_HIP_CHECK(hipStreamSynchronize(stream));
    const auto out = dout.get();
    double     worst = 0.0;
    Rows       last;   // sequence 2 in the cache
    for (int b = 0; b < 3; ++b) {
        Rows r;
        for (int t = cu[b]; t < cu[b + 1]; ++t) {
            const uint16_t* x = kvr.data() + static_cast<std::size_t>(t) * 2 * kv;
            r.push(x, x + kv, false);
            if (b == 2) {
                last.push(x, x + kv, true);
            }
            worst = std::fmax(worst, check(out.data() + static_cast<std::size_t>(t) * qo,
                                           q.data() + static_cast<std::size_t>(t) * qo, r, t - cu[b] + 1));
        }
    }
    fails += expect(worst <= 1.0, "packed prompts, worst error of its bound", worst);

    // Four children of sequence 2 (133 keys: two full pages, five keys of a third).
    dlens.set(lens);
    Dev<int> drop(std::vector<int>{0, 1, 0}), parents(std::vector<int>(4, 2));
    Dev<int> ctables(std::vector<int>(4 * kWidth, -1)), clens(std::vector<int>(4, 0)), ones(std::vector<int>(4, 1));
    Dev<int> shared(std::vector<int>{128});
    pool.free(tables.ptr(), kWidth, dlens.ptr(), drop.ptr(), 3, stream);
    pool.fork(cache, ctables.ptr(), clens.ptr(), tables.ptr(), dlens.ptr(), kWidth, 3, parents.ptr(), 4, stream);
    RUNTHERDER_HIP_CHECK(hipStreamSynchronize(stream));
    fails += expect(clens.get() == std::vector<int>(4, 133), "lengths of the children", clens.get()[0]);
    std::vector<Rows>    seq(4, last);
    std::vector<int>     now(4, 133);
    Dev<uint16_t>        sq(std::vector<uint16_t>(4 * qo)), sk(std::vector<uint16_t>(4 * kv)),
        sv(std::vector<uint16_t>(4 * kv)), so(std::vector<uint16_t>(4 * qo)), so1(std::vector<uint16_t>(4 * qo));
    for (int step = 0; step < 4; ++step) {
        const auto hq = normal(4 * qo, 10 + step), hk = normal(4 * kv, 20 + step), hv = normal(4 * kv, 30 + step);
        sq.set(hq), sk.set(hk), sv.set(hv);
        pool.reserve(ctables.ptr(), kWidth, clens.ptr(), ones.ptr(), 4, stream);
        for (int layer = 0; layer < kLayers; ++layer) {
            cache.append_batch(layer, bf(sk), bf(sv), nullptr, clens.ptr(), 4, 4, ctables.ptr(), kWidth, stream);
        }
        RUNTHERDER_HIP_CHECK(hipStreamSynchronize(stream));
        for (int b = 0; b < 4; ++b) {
            seq[b].push(hk.data() + b * kv, hv.data() + b * kv, true);
            ++now[b];
        }
        clens.set(now);
        // The children share 128 keys; layer 0 reads them as a prefix, layer 1 apart.
        attn.run_decode(bf(so), bf(sq), cache.batch_view(0, ctables.ptr(), kWidth, 4), clens.ptr(), stream,
                        ctables.ptr() + kWidth, kWidth, shared.ptr());
        attn.run_decode(bf(so1), bf(sq), cache.batch_view(1, ctables.ptr(), kWidth, 4), clens.ptr(), stream);
        RUNTHERDER_HIP_CHECK(hipStreamSynchronize(stream));
        const auto o = so.get(), o1 = so1.get();
        worst = 0.0;
        for (int b = 0; b < 4; ++b) {
            worst = std::fmax(worst, check(o.data() + b * qo, hq.data() + b * qo, seq[b], now[b]));
            worst = std::fmax(worst, check(o1.data() + b * qo, hq.data() + b * qo, seq[b], now[b]));
        }
        fails += expect(worst <= 1.0, "decode step, worst error of its bound", worst);
        if (step == 2) {
            // The parents go, the pages move down: 2 shared ones and 4 own.
            pool.free(tables.ptr(), kWidth, dlens.ptr(), nullptr, 3, stream);
            pool.compact(cache, ctables.ptr(), kWidth, 4, stream);
            attn.run_decode(bf(so1), bf(sq), cache.batch_view(0, ctables.ptr(), kWidth, 4), clens.ptr(), stream,
                            ctables.ptr(), kWidth, shared.ptr());
            RUNTHERDER_HIP_CHECK(hipStreamSynchronize(stream));
            fails += expect(so1.get() == o, "the same after compaction", 0);
            int live = 0, top = -1;
            std::vector<int> refs(kPages);
            RUNTHERDER_HIP_CHECK(hipMemcpy(refs.data(), pool.refs(), kPages * sizeof(int), hipMemcpyDeviceToHost));
            for (int i = 0; i < kPages; ++i) {
                live += refs[i] > 0;
                top = refs[i] > 0 ? i : top;
            }
            fails += expect(live == 6 && top == 5 && refs[0] + refs[1] + refs[2] + refs[3] + refs[4] + refs[5] == 12,
                            "pages in use, the lowest ones", live);
        }
    }
    int status = -1;
    RUNTHERDER_HIP_CHECK(hipMemcpy(&status, pool.status(), sizeof(int), hipMemcpyDeviceToHost));
    fails += expect(status == 0, "status", status);
    RUNTHERDER_HIP_CHECK(hipStreamDestroy(stream));
    return fails;
}

}  // namespace

int main() {
    const int fails = run();
    std::printf("%s\n", fails == 0 ? "ALL OK" : "FAILURES");
    return fails == 0 ? 0 : 1;
}
