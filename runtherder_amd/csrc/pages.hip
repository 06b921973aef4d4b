// Pages of a paged KV cache: copying, reserving, forking, freeing and compacting
// them, with the bookkeeping in device memory, gfx950.
//
// refs[page] counts the block-table entries that hold a page; a page with refs
// <= 0 is free. A table entry < 0 holds none. Pages are given out lowest first,
// so the result of a call does not depend on the order of its workgroups, nor
// on the calls that freed the pages, and the pool stays dense.
//
// Two kinds of kernels: one workgroup does the bookkeeping (ranks by prefix
// sums over refs, no atomics where an order could show), then as many as fill
// the chip move the rows of all layers. Moving is bound by the copy's bytes:
// 2 * (2 D + 8) per (row, kv head, layer); the bookkeeping by one read of refs
// and the latency of its few steps.
//
// 8 kv heads, head_dim 128, pages of 64 keys: 48 pages of 32 layers copied in 81 us
// (5.2 TB/s of reads and writes, a large copy's rate; 67 us where the last-level cache holds
// some of them), a pool of 256 pages compacted in 119 us; freeing 8 children and forking 8,
// 28 layers, 16 us: three launches and a chain of reads.
#include <algorithm>

#include "batch_common.hpp"
#include "launch.hpp"

namespace rth {
namespace {

constexpr int kPlanThr   = 1024;
constexpr int kPlanWaves = kPlanThr / kWave;
constexpr int kPlanRefs  = 8;       // refs of a thread per step
constexpr int kMoveThr   = 256;

// Sum over the workgroup and the exclusive prefix of this thread's value;
// `sums` holds one int per wave. Every thread calls it.
__device__ __forceinline__ int block_exclusive(int v, int* sums, int& total) {
    const int tid = static_cast<int>(threadIdx.x), lane = tid & (kWave - 1), wave = tid / kWave;
    int x = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int y = __shfl_up(x, d, kWave);
        x += lane >= d ? y : 0;
    }
    if (lane == kWave - 1) {
        sums[wave] = x;
    }
    __syncthreads();
    int before = 0;
    total      = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? sums[w] : 0;
        total += sums[w];
    }
    __syncthreads();
    return before + x - v;
}

// Ranks the pages of [from, to) that are free (kFree) or in use, in ascending
// order, into list[0 .. most - 1]; how many there are, or at least `most`.
template <bool kFree>
__device__ __forceinline__ int list_pages(const int* refs, int from, int to, int* list, int most,
                                          int* sums) {
    int found = 0;
    for (int at = from; at < to && found < most; at += kPlanThr * kPlanRefs) {
        const int p0 = at + static_cast<int>(threadIdx.x) * kPlanRefs;
        uint32_t  is = 0;
#pragma unroll
        for (int i = 0; i < kPlanRefs; ++i) {
            const int r = p0 + i < to ? refs[p0 + i] : (kFree ? 1 : 0);
            is |= ((r <= 0) == kFree ? 1u : 0u) << i;
        }
        int total;
        int rank = found + block_exclusive(__popc(is), sums, total);
#pragma unroll
        for (int i = 0; i < kPlanRefs; ++i) {
            if (((is >> i) & 1u) != 0) {
                if (rank < most) {
                    list[rank] = p0 + i;
                }
                ++rank;
            }
        }
        found += total;
    }
    return found;
}

__device__ __forceinline__ bool is_page(int p, int num_blocks) { return p >= 0 && p < num_blocks; }

// ---- moving rows ------------------------------------------------------------

struct Move {
    int src, dst, rows;
};

// rows of page src to page dst in layer l: K (half 0) or V with its scales.
__device__ __forceinline__ void move_rows(const PageSlabs& s, const Move& m, int64_t layer, int half) {
    const int64_t page_rows = static_cast<int64_t>(s.block_size) * s.hkv;
    const int64_t all       = static_cast<int64_t>(s.num_blocks) * page_rows;
    const int64_t n         = static_cast<int64_t>(m.rows) * s.hkv;
    uint8_t*       codes = half == 0 ? s.k : s.v;
    float*         scale = half == 0 ? s.ks : s.vs;
    const int64_t  from = layer * all + m.src * page_rows, to = layer * all + m.dst * page_rows;
    const u32x4*   a = reinterpret_cast<const u32x4*>(codes + from * s.head_dim);
    u32x4*         b = reinterpret_cast<u32x4*>(codes + to * s.head_dim);
    const int64_t  bytes = n * s.head_dim, n16 = bytes / 16;
    const int      tid = static_cast<int>(threadIdx.x);
    int64_t i = tid;
    // Four loads on the way, and stores past the caches (48 pages of 32 layers,
    // the same ones each time, 85 us; so 67, and with such loads as well 76).
    for (; i + 3 * kMoveThr < n16; i += 4 * kMoveThr) {
        u32x4 x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            x[c] = a[i + c * kMoveThr];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            __builtin_nontemporal_store(x[c], b + i + c * kMoveThr);
        }
    }
    for (; i < n16; i += kMoveThr) {
        b[i] = a[i];
    }
    // (A row of an odd multiple of 8 codes leaves 8 bytes.)
    if (tid < (bytes - 16 * n16) / 4) {
        reinterpret_cast<uint32_t*>(b + n16)[tid] = reinterpret_cast<const uint32_t*>(a + n16)[tid];
    }
    for (int64_t r = tid; r < n; r += kMoveThr) {
        scale[to + r] = scale[from + r];
    }
}

// Moves count pages (src[i] -> dst[i]); rows[i] rows, or all where rows is null.
// count_at: the count, where the device made it. Ids that name no page, and a
// page onto itself, are skipped.
__global__ __launch_bounds__(kMoveThr) void move_pages_kernel(PageSlabs s, const int* __restrict__ src,
                                                             const int* __restrict__ dst,
                                                             const int* __restrict__ rows, int count,
                                                             const int* __restrict__ count_at) {
    const int     n     = count_at != nullptr ? *count_at : count;
    const int64_t units = static_cast<int64_t>(n) * s.layers * 2;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int half = static_cast<int>(u & 1), i = static_cast<int>((u >> 1) % n);
        const Move m{src[i], dst[i], rows != nullptr ? rows[i] : s.block_size};
        if (is_page(m.src, s.num_blocks) && is_page(m.dst, s.num_blocks) && m.src != m.dst) {
            move_rows(s, m, (u >> 1) / n, half);
        }
    }
}

hipError_t move_pages(const PageSlabs& s, const int* src, const int* dst, const int* rows, int count,
                      const int* count_at, hipStream_t stream) {
    int        cus = 0;
    hipError_t e   = device_cu_count(&cus);
    if (e != hipSuccess) {
        return e;
    }
    const int64_t units = static_cast<int64_t>(count) * s.layers * 2;
    const int64_t grid  = std::min<int64_t>(units, static_cast<int64_t>(cus) * 16);
    move_pages_kernel<<<dim3(static_cast<unsigned>(std::max<int64_t>(grid, 1))), kMoveThr, 0, stream>>>(
        s, src, dst, rows, count, count_at);
    return hipGetLastError();
}

// ---- bookkeeping --------------------------------------------------------------

// work: [num_blocks] pages found.
__global__ __launch_bounds__(kPlanThr) void reserve_kernel(int* refs, int* work, int* status,
                                                          int num_blocks, int block_size, int* tables,
                                                          int table_blocks, const int* lens,
                                                          const int* n_new, int num_seqs) {
    __shared__ int need[kMaxBatchSeqs];
    __shared__ int sums[kPlanWaves];
    __shared__ int too_long;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & (kWave - 1), wave = tid / kWave;
    if (tid == 0) {
        too_long = 0;
    }
    __syncthreads();
    // Entries [first, last) of a sequence's row that have to hold a page.
    auto range = [&](int b, int& first, int& last) {
        const int     len = max(lens[b], 0);
        const int64_t to  = static_cast<int64_t>(len) + max(n_new[b], 0);
        first             = len / block_size;
        last              = static_cast<int>((to + block_size - 1) / block_size);
        if (lens[b] < 0 || n_new[b] <= 0) {
            last = first;
        }
    };
    for (int b = wave; b < num_seqs; b += kPlanWaves) {
        int first, last, n = 0;
        range(b, first, last);
        if (last > table_blocks) {
            if (lane == 0) {
                too_long = 1;
            }
            last = first;
        }
        for (int i0 = first; i0 < last; i0 += kWave) {
            const int i = i0 + lane;
            n += __popcll(__ballot(i < last && tables[static_cast<int64_t>(b) * table_blocks + i] < 0));
        }
        if (lane == 0) {
            need[b] = n;
        }
    }
    __syncthreads();
    // need[b] -> the rank of its first page.
    int total = 0;
    for (int b0 = 0; b0 < num_seqs; b0 += kPlanThr) {
        const int b = b0 + tid, n = b < num_seqs ? need[b] : 0;
        int       sum;
        const int before = block_exclusive(n, sums, sum);
        if (b < num_seqs) {
            need[b] = total + before;
        }
        total += sum;
    }
    if (too_long != 0) {
        if (tid == 0) {
            atomicOr(status, 2);
        }
        return;
    }
    const int found = total > 0 ? list_pages<true>(refs, 0, num_blocks, work, min(total, num_blocks), sums) : 0;
    if (found < total) {
        if (tid == 0) {
            atomicOr(status, 1);
        }
        return;
    }
    __syncthreads();   // work is whole (one workgroup: its own global writes)
    for (int i = tid; i < total; i += kPlanThr) {
        refs[work[i]] = 1;
    }
    for (int b = wave; b < num_seqs; b += kPlanWaves) {
        int first, last, rank = need[b];
        range(b, first, last);
        for (int i0 = first; i0 < last; i0 += kWave) {
            const int i    = i0 + lane;
            int*      e    = tables + static_cast<int64_t>(b) * table_blocks + i;
            const bool is  = i < last && *e < 0;
            const uint64_t m = __ballot(is);
            if (is) {
                *e = work[rank + lanes_below(m)];
            }
            rank += __popcll(m);
        }
    }
}

// work: [num_blocks] pages found, then count, src, dst, rows of the moves.
__global__ __launch_bounds__(kPlanThr) void fork_kernel(int* refs, int* work, int* moves, int* status,
                                                       int num_blocks, int block_size, int* dst_tables,
                                                       int* dst_lens, const int* src_tables,
                                                       const int* src_lens, int table_blocks,
                                                       int num_src, const int* parents,
                                                       int num_children) {
    __shared__ int rank_of[kMaxBatchSeqs];   // of a child's own page, or -1
    __shared__ int sums[kPlanWaves];
    const int tid = static_cast<int>(threadIdx.x), lane = tid & (kWave - 1), wave = tid / kWave;
    const int64_t room = static_cast<int64_t>(table_blocks) * block_size;
    auto length = [&](int p) {
        return p >= 0 && p < num_src
                   ? static_cast<int>(min(static_cast<int64_t>(max(src_lens[p], 0)), room))
                   : 0;
    };
    int total = 0;
    for (int c0 = 0; c0 < num_children; c0 += kPlanThr) {
        const int c   = c0 + tid;
        int       has = 0;
        if (c < num_children) {
            const int p = parents[c], len = length(p);
            has = len % block_size != 0 &&
                  is_page(src_tables[static_cast<int64_t>(p) * table_blocks + len / block_size], num_blocks);
        }
        int       sum;
        const int before = block_exclusive(has, sums, sum);
        if (c < num_children) {
            rank_of[c] = has != 0 ? total + before : -1;
        }
        total += sum;
    }
    const int found = total > 0 ? list_pages<true>(refs, 0, num_blocks, work, min(total, num_blocks), sums) : 0;
    if (found < total) {
        if (tid == 0) {
            atomicOr(status, 1);
            moves[0] = 0;
        }
        return;
    }
    __syncthreads();
    int* src  = moves + 1;
    int* dst  = src + num_children;
    int* rows = dst + num_children;
    if (tid == 0) {
        moves[0] = total;
    }
    for (int i = tid; i < total; i += kPlanThr) {
        refs[work[i]] = 1;
    }
    for (int c = wave; c < num_children; c += kPlanWaves) {
        const int  p = parents[c], len = length(p), full = len / block_size, rank = rank_of[c];
        const int* from = src_tables + static_cast<int64_t>(max(p, 0)) * table_blocks;
        int*       to   = dst_tables + static_cast<int64_t>(c) * table_blocks;
        for (int i = lane; i < table_blocks; i += kWave) {
            int e = -1;
            if (i < full) {
                e = from[i];
                if (is_page(e, num_blocks)) {
                    atomicAdd(&refs[e], 1);
                } else {
                    e = -1;
                }
            } else if (i == full && rank >= 0) {
                e          = work[rank];
                src[rank]  = from[i];
                dst[rank]  = e;
                rows[rank] = len % block_size;
            }
            to[i] = e;
        }
        if (lane == 0) {
            dst_lens[c] = len;
        }
    }
}

__global__ __launch_bounds__(kMoveThr) void free_kernel(int* refs, int num_blocks, int* tables,
                                                       int table_blocks, int* lens, const int* drop) {
    const int b = static_cast<int>(blockIdx.x);
    if (drop != nullptr && drop[b] == 0) {
        return;
    }
    int* row = tables + static_cast<int64_t>(b) * table_blocks;
    for (int i = static_cast<int>(threadIdx.x); i < table_blocks; i += kMoveThr) {
        const int e = row[i];
        if (is_page(e, num_blocks)) {
            atomicAdd(&refs[e], -1);
        }
        row[i] = -1;
    }
    if (threadIdx.x == 0) {
        lens[b] = 0;
    }
}

// work: the new name of each page, then count, src, dst.
__global__ __launch_bounds__(kPlanThr) void compact_kernel(int* refs, int* work, int* moves, int num_blocks) {
    __shared__ int sums[kPlanWaves];
    const int tid = static_cast<int>(threadIdx.x);
    int       n   = 0;
    for (int p = tid; p < num_blocks; p += kPlanThr) {
        n += refs[p] > 0 ? 1 : 0;
    }
    int live;
    block_exclusive(n, sums, live);
    int* src = moves + 1;
    int* dst = src + num_blocks;
    const int holes  = list_pages<true>(refs, 0, live, dst, num_blocks, sums);
    const int movers = list_pages<false>(refs, live, num_blocks, src, num_blocks, sums);
    __syncthreads();
    for (int p = tid; p < num_blocks; p += kPlanThr) {
        work[p] = p;
    }
    __syncthreads();
    const int count = min(holes, movers);   // equal
    for (int i = tid; i < count; i += kPlanThr) {
        work[src[i]] = dst[i];
        refs[dst[i]] = refs[src[i]];
        refs[src[i]] = 0;
    }
    if (tid == 0) {
        moves[0] = count;
    }
}

__global__ __launch_bounds__(kMoveThr) void rename_kernel(int* tables, int64_t entries, const int* name,
                                                         int num_blocks) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kMoveThr + threadIdx.x;
    if (i < entries) {
        const int e = tables[i];
        if (is_page(e, num_blocks)) {
            tables[i] = name[e];
        }
    }
}

}  // namespace

hipError_t pages_copy_launch(const PageSlabs& s, const int* src, const int* dst, int count,
                             hipStream_t stream) {
    return move_pages(s, src, dst, nullptr, count, nullptr, stream);
}

hipError_t pages_reserve_launch(int* refs, int* work, int* status, int num_blocks, int block_size,
                                int* tables, int table_blocks, const int* lens, const int* n_new,
                                int num_seqs, hipStream_t stream) {
    reserve_kernel<<<1, kPlanThr, 0, stream>>>(refs, work, status, num_blocks, block_size, tables,
                                               table_blocks, lens, n_new, num_seqs);
    return hipGetLastError();
}

hipError_t pages_fork_launch(const PageSlabs& s, int* refs, int* work, int* status,
                             int* dst_tables, int* dst_lens, const int* src_tables,
                             const int* src_lens, int table_blocks, int num_src,
                             const int* parents, int num_children, hipStream_t stream) {
    int* moves = work + s.num_blocks;
    fork_kernel<<<1, kPlanThr, 0, stream>>>(refs, work, moves, status, s.num_blocks, s.block_size,
                                            dst_tables, dst_lens, src_tables, src_lens, table_blocks,
                                            num_src, parents, num_children);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    return move_pages(s, moves + 1, moves + 1 + num_children, moves + 1 + 2 * num_children,
                      num_children, moves, stream);
}

hipError_t pages_free_launch(int* refs, int num_blocks, int* tables, int table_blocks, int* lens,
                             const int* drop, int num_seqs, hipStream_t stream) {
    free_kernel<<<num_seqs, kMoveThr, 0, stream>>>(refs, num_blocks, tables, table_blocks, lens, drop);
    return hipGetLastError();
}

hipError_t pages_compact_launch(const PageSlabs& s, int* refs, int* work, int* tables,
                                int table_blocks, int num_seqs, hipStream_t stream) {
    int* moves = work + s.num_blocks;
    compact_kernel<<<1, kPlanThr, 0, stream>>>(refs, work, moves, s.num_blocks);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    const int64_t entries = static_cast<int64_t>(num_seqs) * table_blocks;
    rename_kernel<<<dim3(static_cast<unsigned>((entries + kMoveThr - 1) / kMoveThr)), kMoveThr, 0, stream>>>(
        tables, entries, work, s.num_blocks);
    e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    return move_pages(s, moves + 1, moves + 1 + s.num_blocks, nullptr, (s.num_blocks + 1) / 2, moves, stream);
}

}  // namespace rth
