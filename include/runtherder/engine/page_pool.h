// Which pages of a paged cache are in use, on the device (no reference
// counterpart): refs[page] counts the block-table entries that hold it, refs
// <= 0 is free, and the lowest free pages are given out first. Block tables
// are [seqs, table_blocks] device ints, -1 where there is no page. Nothing here
// waits for the device: what a call could not do for lack of pages (or of
// table entries) it leaves undone and says in *status(), which stays set until
// the caller clears it. Calls on one pool run one behind the other.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>

#include <rth_attn.h>
#include <runtherder/check.h>
#include <runtherder/device/check.h>
#include <runtherder/device/memory.h>
#include <runtherder/engine/paged_kv_cache.h>

namespace runtherder::engine {

class PagePool {
public:
    static constexpr int kOutOfPages = 1, kTableTooShort = 2;   // bits of *status()

    PagePool(int num_blocks, int block_size) : num_blocks_(num_blocks), block_size_(block_size) {
        RUNTHERDER_CHECK(num_blocks >= 1, "PagePool num_blocks must be >= 1");
        RUNTHERDER_CHECK(block_size >= 32 && (block_size & (block_size - 1)) == 0,
                         "PagePool block_size must be a power of two >= 32");
        refs_   = device::make_device_unique<int>(num_blocks);
        status_ = device::make_device_unique<int>(1);
        work_   = device::make_device_unique<int>(rth_pages_work_ints(num_blocks));
        RUNTHERDER_HIP_CHECK(hipMemset(refs_.get(), 0, static_cast<std::size_t>(num_blocks) * sizeof(int)));
        RUNTHERDER_HIP_CHECK(hipMemset(status_.get(), 0, sizeof(int)));
        RUNTHERDER_HIP_CHECK(hipDeviceSynchronize());
    }

    // Pages for positions lens[b] .. lens[b] + n_new[b] - 1 of sequence b, where
    // its table row has none yet.
    void reserve(int* block_tables, int table_blocks, const int* lens, const int* n_new,
                 int num_seqs, hipStream_t stream) {
        RUNTHERDER_RTH_CHECK(rth_pages_reserve(refs_.get(), work_.get(), status_.get(), num_blocks_,
                                               block_size_, block_tables, table_blocks, lens, n_new,
                                               num_seqs, stream));
    }

    // Sequence i of dst becomes a copy of sequence parents[i] of src: filled
    // pages are shared, a part-filled last page is copied, in all layers of
    // cache, into a page of the child's own. The dst tables hold no pages before.
    void fork(PagedKVCache& cache, int* dst_tables, int* dst_lens, const int* src_tables,
              const int* src_lens, int table_blocks, int num_src, const int* parents,
              int num_children, hipStream_t stream) {
        const auto c = of(cache);
        RUNTHERDER_RTH_CHECK(rth_pages_fork(c.k, c.v, c.k_scale, c.v_scale, c.num_layers,
                                            num_blocks_, block_size_, c.num_kv_heads, c.head_dim,
                                            refs_.get(), work_.get(), status_.get(), dst_tables,
                                            dst_lens, src_tables, src_lens, table_blocks, num_src,
                                            parents, num_children, stream));
    }

    // Frees the sequences with drop[b] != 0 (null: all): their pages lose one
    // reference, their table rows hold none, their lengths are 0.
    void free(int* block_tables, int table_blocks, int* lens, const int* drop, int num_seqs,
              hipStream_t stream) {
        RUNTHERDER_RTH_CHECK(rth_pages_free(refs_.get(), num_blocks_, block_tables, table_blocks,
                                            lens, drop, num_seqs, stream));
    }

    // Moves the pages in use down to the lowest ones, in all layers of cache, and
    // renames them in block_tables, which are all the tables that hold pages of
    // the pool.
    void compact(PagedKVCache& cache, int* block_tables, int table_blocks, int num_seqs,
                 hipStream_t stream) {
        const auto c = of(cache);
        RUNTHERDER_RTH_CHECK(rth_pages_compact(c.k, c.v, c.k_scale, c.v_scale, c.num_layers,
                                               num_blocks_, block_size_, c.num_kv_heads, c.head_dim,
                                               refs_.get(), work_.get(), block_tables, table_blocks,
                                               num_seqs, stream));
    }

    [[nodiscard]] int* refs() noexcept { return refs_.get(); }       // [num_blocks], device
    [[nodiscard]] int* status() noexcept { return status_.get(); }   // one device int
    [[nodiscard]] int  num_blocks() const noexcept { return num_blocks_; }
    [[nodiscard]] int  block_size() const noexcept { return block_size_; }

private:
    [[nodiscard]] PagedKVCache::AllLayers of(PagedKVCache& cache) const {
        RUNTHERDER_CHECK(cache.num_blocks() == num_blocks_ && cache.block_size() == block_size_,
                         "the pool and the cache differ in their blocks");
        return cache.all_layers();
    }

    int                          num_blocks_, block_size_;
    device::DeviceUniquePtr<int> refs_, status_, work_;
};

}  // namespace runtherder::engine
