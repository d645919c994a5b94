#pragma once
// A paged key/value cache and the operators of a serving step over it (no counterpart in the reference, whose KVCache
// holds one batch of one length).  Requests of different lengths share one pool of pages; a step's batch says which new
// positions of which requests it computes and in which pages they lie.  The caller hands pages out; everything it says
// about them is checked on the host when the batch is made, before any kernel reads it.  A PagePool counts who holds which
// page; requests are forked, and what is left of a pool moved to its front, by copies that the operators below queue.

#include "dl/ops.h"

#include <memory>
#include <span>
#include <vector>

namespace dl::nn {

/// One pool of pages per layer: keys and values [pages, kv_heads, page_size, head_dim], f32 or bf16, on a GPU.
/// page_size is a power of two from 16 to 1024, head_dim 16, 32, 64 or 128.
class DL_API PagedKVCache {
public:
    PagedKVCache(Index layers, Index pages, Index page_size, Index kv_heads, Index head_dim, TensorOptions options);
    Index layers() const { return static_cast<Index>(key_.size()); }
    Index pages() const { return pages_; }
    Index page_size() const { return page_size_; }
    Index kv_heads() const { return kv_heads_; }
    Index head_dim() const { return head_dim_; }
    DType dtype() const { return options_.dtype; }
    Device device() const { return options_.device; }
    /// The live storage of a layer.
    const Tensor& key(Index layer) const { return key_.at(static_cast<std::size_t>(layer)); }
    const Tensor& value(Index layer) const { return value_.at(static_cast<std::size_t>(layer)); }

private:
    Index pages_, page_size_, kv_heads_, head_dim_;
    TensorOptions options_;
    std::vector<Tensor> key_, value_;
};

/// What one step computes: sequence b holds lengths[b] positions and gets counts[b] new ones (0: none this time), and its
/// position p lies in page tables[b * width + p / page_size].  The new positions' rows of a step lie one sequence after
/// another ([tokens, heads, head_dim], tokens the sum of the counts).  With `shared` > 0 (whole pages) the first `shared`
/// positions of every sequence with new ones lie in the same pages, and attention reads them once for the whole batch.
/// A page that the step writes belongs to one place of one sequence with new positions; the pages of the others are not
/// looked at, so the caller sees to it that a step writes none that they still need.  Made once and used for every layer; the
/// cache may be another one of the same layout.  Making it copies the plan to the device and waits for the library's stream.
class DL_API PagedBatch {
public:
    struct Plan;
    PagedBatch(const PagedKVCache& cache, Index heads, std::span<const Index> lengths, std::span<const Index> counts,
               std::span<const Index> tables, Index width, Index shared = 0);
    Index tokens() const;
    const Plan& plan() const { return *plan_; }

private:
    std::shared_ptr<const Plan> plan_;
};

/// Which pages of a cache are held, and by how many page tables.  Host bookkeeping alone; used by one thread at a time.
/// Ids below zero (the empty places of a table) are passed over; an id beyond the pool is refused, and a refused call
/// changes nothing.
class DL_API PagePool {
public:
    explicit PagePool(Index pages);
    Index pages() const { return static_cast<Index>(holders_.size()); }
    /// Pages that nobody holds.
    Index available() const { return available_; }
    Index references(Index page) const;
    /// `count` free pages, the lowest ones, each held once from now on.
    std::vector<Index> take(Index count);
    /// One more holder of each page, free ones among them (a pool made anew from tables).
    void claim(std::span<const Index> pages);
    /// One more holder of each page, all of them held.
    void share(std::span<const Index> pages);
    /// One holder fewer of each page; without any it is free.  Work queued that reads it has the old contents still: what
    /// writes it next is queued behind.
    void release(std::span<const Index> pages);

private:
    void check(std::span<const Index> pages) const;
    std::vector<Index> holders_;
    Index available_, lowest_ = 0; // no page below `lowest_` is free
};

} // namespace dl::nn

namespace dl {

/// Writes the step's keys (rotated at their positions) and values, [tokens, kv_heads, head_dim], to their pages of
/// `layer`, and returns the queries [tokens, heads, head_dim] rotated likewise (an undefined tensor when there are none).
/// All three are f32 or bf16 and may be views of one projection output; cosine and sine as for rotary_positions, with a
/// row for every position of the step (on the cache's device, or they are copied there, and waited for, in each call).  What of
/// them lies in this layer's pages is taken as it was before the call.  A bf16 cache rounds each key and value once.
DL_API Tensor paged_append(const nn::PagedKVCache& cache, Index layer, const nn::PagedBatch& batch,
                           const std::optional<Tensor>& query, const Tensor& key, const Tensor& value,
                           const Tensor& cosine, const Tensor& sine, RotaryLayout layout);

/// Attention of the step's (rotated) queries [tokens, heads, head_dim], f32 or bf16, over the pages of `layer`: the row
/// at position p sees the positions 0 .. p of its sequence, its own included (append first).  f32 [tokens, heads, head_dim].
/// What a row does not see may hold anything.  Products keep all bits of an f32 (of f32 queries and weights by f32 keys and
/// values down to 2^-22 of each product), for finite scores q k / sqrt(head_dim) whose products' magnitudes sum below 2^29 and
/// for values up to 1e36 over the number of keys that the row sees: they are summed with weights of up to 2^8 before the division.
/// Where a row sees a value that is not finite, that entry of it is not finite either.
DL_API Tensor paged_attention(const nn::PagedKVCache& cache, Index layer, const nn::PagedBatch& batch, const Tensor& query);

/// Copies page sources[i] to page targets[i] in every layer, keys and values, of each only the first rows[i] positions (an
/// empty `rows`: whole pages); what else a target holds stays.  Every source is taken as it was before the call, whichever
/// order the pairs stand in; no page is a target twice.
DL_API void paged_copy(const nn::PagedKVCache& cache, std::span<const Index> sources, std::span<const Index> targets,
                       std::span<const Index> rows = {});

/// Tables [parents, width] of new requests that go on from position lengths[p] of request p = parents[i] (a row of `tables`
/// [sequences, width], all of its pages up to there held): the whole pages in front are shared, a partly filled last one is
/// copied, as far as it is filled, to a page taken from the pool, and the rest of a row is -1.  With too few free pages
/// the call is refused and the pool stays as it was.  (Of this cache: in another whose pages the same tables name, paged_copy
/// copies the last ones.)
DL_API std::vector<Index> paged_fork(const nn::PagedKVCache& cache, nn::PagePool& pool, std::span<const Index> tables, Index width,
                                     std::span<const Index> lengths, std::span<const Index> parents);

/// Moves the held pages to the front of the pool: those beyond the first n, n the number of held pages, go to the free ones
/// among them, in ascending order; their ids in `tables` become the new ones.  The tables are all that holds pages: a page
/// stands in them as often as the pool counts.  Returns how many pages were moved.  (It moves this cache's pages: two caches whose
/// pages share tables and a pool, a draft model's beside the target's, cannot be compacted, since one call renames them for both.)
DL_API Index paged_compact(const nn::PagedKVCache& cache, nn::PagePool& pool, std::span<Index> tables);

} // namespace dl
