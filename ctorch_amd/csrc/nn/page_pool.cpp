// Who holds which page of a paged cache, and the copies that fork and compact requests (include/dl/paged.h).
#include "nn/ops_internal.h"

#include "dl/paged.h"

#include <algorithm>
#include <stdexcept>
#include <unordered_map>

namespace dl::detail {

// Staged copies keep the call's meaning where a page is read by one pair and written by another: such sources are first
// copied to memory of their own.  (Compaction and forks have none.)
void copy_pages(const std::vector<void*>& pools, Index pages, Index heads, Index page, Index row_bytes, Device device,
                std::span<const Index> sources, std::span<const Index> targets, std::span<const Index> rows, const char* operation) {
    const std::string name(operation);
    const auto refuse = [&](const std::string& what) { throw std::invalid_argument(name + ": " + what); };
    if (sources.size() != targets.size() || (!rows.empty() && rows.size() != sources.size()))
        refuse("needs a target (and, if given, rows) for each source");
    const Index units = row_bytes / 16 * page * heads; // 16 bytes each
    if (units > 1 << 27) refuse("pages of more than 2 GiB");
    std::vector<std::uint8_t> written(static_cast<std::size_t>(pages), 0);
    for (std::size_t i = 0; i < sources.size(); ++i) {
        for (const Index id : {sources[i], targets[i]})
            if (id < 0 || id >= pages) refuse(std::to_string(id) + " is not one of " + std::to_string(pages));
        if (!rows.empty() && (rows[i] < 0 || rows[i] > page)) refuse("rows of a page must be from 0 to " + std::to_string(page));
        auto& mark = written[static_cast<std::size_t>(targets[i])];
        if (mark) refuse(std::to_string(targets[i]) + " would be written twice");
        mark = 1;
    }
    std::vector<dlk_page_pair> stage, copy;
    std::unordered_map<Index, std::pair<std::int32_t, std::size_t>> places; // of staged sources, and their pairs
    for (std::size_t i = 0; i < sources.size(); ++i) {
        const auto from = static_cast<std::int32_t>(sources[i]), to = static_cast<std::int32_t>(targets[i]);
        const auto n = static_cast<std::int32_t>(rows.empty() ? page : rows[i]);
        if (n == 0 || from == to) continue;
        if (!written[static_cast<std::size_t>(from)]) {
            copy.push_back({from, to, n});
            continue;
        }
        const auto [place, fresh] = places.try_emplace(from, static_cast<std::int32_t>(places.size()), stage.size());
        if (fresh) stage.push_back({from, ~place->second.first, n});
        else stage[place->second.second].rows = std::max(stage[place->second.second].rows, n);
        copy.push_back({~place->second.first, to, n});
    }
    if (copy.empty()) return;
    GpuContext& context = gpu_context(device.index);
    // a launch has fewer than 2^32 threads, of 64 bytes each
    const std::size_t most = std::min<std::size_t>(pools.size(), DLK_PAGE_POOLS);
    const std::size_t pairs = std::clamp<std::size_t>((1u << 30) / (static_cast<std::size_t>(units) * most), 1, DLK_PAGE_PAIRS);
    dlk_page_copy_params p{};
    p.heads = static_cast<int>(heads);
    p.page = static_cast<int>(page);
    p.row_units = static_cast<int>(row_bytes / 16);
    Tensor staging; // released to the pool in stream order
    if (!places.empty()) {
        p.staged = static_cast<int>(places.size());
        staging = empty_tensor({static_cast<Index>(most), p.staged, heads, page, row_bytes / 4}, DType::f32, device);
        p.staging = mutable_data(staging);
    }
    for (std::size_t first = 0; first < pools.size(); first += most) {
        p.pool_count = static_cast<int>(std::min(most, pools.size() - first));
        std::copy_n(pools.begin() + static_cast<std::ptrdiff_t>(first), p.pool_count, p.pools);
        for (const auto* list : {&stage, &copy})
            for (std::size_t i = 0; i < list->size(); i += pairs) {
                p.count = static_cast<int>(std::min(pairs, list->size() - i));
                std::copy_n(list->begin() + static_cast<std::ptrdiff_t>(i), p.count, p.pairs);
                hip_check(dlk_page_copy(&p, context.stream), operation);
            }
    }
}

} // namespace dl::detail

namespace dl::nn {

PagePool::PagePool(Index pages) : available_(pages) {
    if (pages <= 0 || pages > INT32_MAX) throw std::invalid_argument("page pool: pages must be positive, below 2^31");
    holders_.resize(static_cast<std::size_t>(pages), 0);
}

void PagePool::check(std::span<const Index> pages) const {
    for (const Index id : pages)
        if (id >= this->pages()) throw std::out_of_range("page pool: page " + std::to_string(id) + " is not in the pool");
}

Index PagePool::references(Index page) const {
    if (page < 0 || page >= pages()) throw std::out_of_range("page pool: page " + std::to_string(page) + " is not in the pool");
    return holders_[static_cast<std::size_t>(page)];
}

std::vector<Index> PagePool::take(Index count) {
    if (count < 0) throw std::invalid_argument("page pool: a count below zero");
    if (count > available_)
        throw std::runtime_error("page pool: " + std::to_string(count) + " pages wanted, " + std::to_string(available_) + " are free");
    std::vector<Index> out;
    out.reserve(static_cast<std::size_t>(count));
    for (; static_cast<Index>(out.size()) < count; ++lowest_)
        if (auto& n = holders_[static_cast<std::size_t>(lowest_)]; n == 0) n = 1, out.push_back(lowest_);
    available_ -= count;
    return out;
}

void PagePool::claim(std::span<const Index> pages) {
    check(pages);
    for (const Index id : pages)
        if (id >= 0 && holders_[static_cast<std::size_t>(id)]++ == 0) --available_;
}

void PagePool::share(std::span<const Index> pages) {
    check(pages);
    for (const Index id : pages)
        if (id >= 0 && holders_[static_cast<std::size_t>(id)] == 0)
            throw std::invalid_argument("page pool: page " + std::to_string(id) + " is not held");
    claim(pages);
}

void PagePool::release(std::span<const Index> pages) {
    check(pages);
    for (std::size_t i = 0; i < pages.size(); ++i) {
        if (pages[i] < 0) continue;
        auto& n = holders_[static_cast<std::size_t>(pages[i])];
        if (n == 0) { // (perhaps since this call: what it did is taken back)
            for (std::size_t j = 0; j < i; ++j)
                if (pages[j] >= 0 && holders_[static_cast<std::size_t>(pages[j])]++ == 0) --available_;
            throw std::invalid_argument("page pool: page " + std::to_string(pages[i]) + " is not held");
        }
        if (--n == 0) ++available_;
    }
    for (const Index id : pages)
        if (id >= 0) lowest_ = std::min(lowest_, id);
}

} // namespace dl::nn

namespace dl {

using namespace detail;

void paged_copy(const nn::PagedKVCache& cache, std::span<const Index> sources, std::span<const Index> targets,
                std::span<const Index> rows) {
    std::vector<void*> pools;
    for (Index layer = 0; layer < cache.layers(); ++layer) {
        pools.push_back(mutable_data(cache.key(layer)));
        pools.push_back(mutable_data(cache.value(layer)));
    }
    copy_pages(pools, cache.pages(), cache.kv_heads(), cache.page_size(), cache.head_dim() * (cache.dtype() == DType::bf16 ? 2 : 4),
               cache.device(), sources, targets, rows, "paged_copy");
}

std::vector<Index> paged_fork(const nn::PagedKVCache& cache, nn::PagePool& pool, std::span<const Index> tables, Index width,
                              std::span<const Index> lengths, std::span<const Index> parents) {
    const auto refuse = [](const std::string& what) { throw std::invalid_argument("paged_fork: " + what); };
    const Index batch = static_cast<Index>(lengths.size()), page = cache.page_size();
    if (pool.pages() != cache.pages()) refuse("the pool counts other pages than the cache has");
    if (width <= 0 || (batch > 0 && width > INT32_MAX / batch) || tables.size() != static_cast<std::size_t>(batch * width))
        refuse("tables must be [sequences, width]");
    std::vector<Index> children, sources, rows, slots; // slots: where the copied pages' ids go
    children.reserve(parents.size() * static_cast<std::size_t>(width));
    for (const Index b : parents) {
        if (b < 0 || b >= batch) refuse("parent " + std::to_string(b) + " is not one of the sequences");
        const Index length = lengths[static_cast<std::size_t>(b)];
        if (length < 0 || length > width * page) refuse("sequence " + std::to_string(b) + " has positions outside its table");
        const Index whole = length / page, used = (length + page - 1) / page;
        const Index* row = tables.data() + b * width;
        for (Index i = 0; i < used; ++i)
            if (row[i] < 0 || row[i] >= cache.pages() || pool.references(row[i]) == 0)
                refuse("page " + std::to_string(row[i]) + " of sequence " + std::to_string(b) + " is not held");
        if (used > whole) {
            sources.push_back(row[whole]);
            rows.push_back(length - whole * page);
            slots.push_back(static_cast<Index>(children.size()) + whole);
        }
        children.insert(children.end(), row, row + whole);
        children.insert(children.end(), static_cast<std::size_t>(width - whole), -1);
    }
    const auto targets = pool.take(static_cast<Index>(slots.size()));
    try {
        paged_copy(cache, sources, targets, rows);
    } catch (...) {
        pool.release(targets);
        throw;
    }
    pool.share(children);
    for (std::size_t i = 0; i < slots.size(); ++i) children[static_cast<std::size_t>(slots[i])] = targets[i];
    return children;
}

Index paged_compact(const nn::PagedKVCache& cache, nn::PagePool& pool, std::span<Index> tables) {
    const auto refuse = [](const std::string& what) { throw std::invalid_argument("paged_compact: " + what); };
    if (pool.pages() != cache.pages()) refuse("the pool counts other pages than the cache has");
    std::vector<Index> seen(static_cast<std::size_t>(cache.pages()), 0);
    for (const Index id : tables) {
        if (id >= cache.pages()) refuse("page " + std::to_string(id) + " is not in the cache");
        if (id >= 0) ++seen[static_cast<std::size_t>(id)];
    }
    for (Index id = 0; id < cache.pages(); ++id)
        if (pool.references(id) != seen[static_cast<std::size_t>(id)])
            refuse("page " + std::to_string(id) + " is held " + std::to_string(pool.references(id)) + " times and stands " +
                   std::to_string(seen[static_cast<std::size_t>(id)]) + " times in the tables");
    const Index live = cache.pages() - pool.available();
    std::vector<Index> sources, targets;
    for (Index id = live; id < cache.pages(); ++id)
        if (seen[static_cast<std::size_t>(id)]) sources.push_back(id);
    for (Index id = 0; id < live; ++id)
        if (!seen[static_cast<std::size_t>(id)]) targets.push_back(id);
    paged_copy(cache, sources, targets);
    std::vector<Index> moved(static_cast<std::size_t>(cache.pages()), -1);
    for (std::size_t i = 0; i < sources.size(); ++i) moved[static_cast<std::size_t>(sources[i])] = targets[i];
    nn::PagePool renamed(cache.pages());
    for (Index& id : tables)
        if (id >= 0 && moved[static_cast<std::size_t>(id)] >= 0) id = moved[static_cast<std::size_t>(id)];
    renamed.claim(tables);
    pool = std::move(renamed);
    return static_cast<Index>(sources.size());
}

} // namespace dl
