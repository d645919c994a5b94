// The paged key/value cache, the plan of a step over it, and its two operators (include/dl/paged.h).
#include "nn/paged_plan.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <numeric>
#include <stdexcept>

namespace dl::nn {

using namespace dl::detail;

PagedKVCache::PagedKVCache(Index layers, Index pages, Index page_size, Index kv_heads, Index head_dim,
                           TensorOptions options)
    : pages_(pages), page_size_(page_size), kv_heads_(kv_heads), head_dim_(head_dim), options_(options) {
    if (layers <= 0 || pages <= 0 || kv_heads <= 0)
        throw std::invalid_argument("paged cache: layers, pages and kv_heads must be positive");
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
        throw std::invalid_argument("paged cache: the page size must be a power of two from 16 to 1024");
    if (head_dim != 16 && head_dim != 32 && head_dim != 64 && head_dim != 128)
        throw std::invalid_argument("paged cache: head size 16, 32, 64 or 128");
    if (options.dtype != DType::f32 && options.dtype != DType::bf16)
        throw std::invalid_argument("paged cache: pages must be f32 or bf16");
    if (pages > INT32_MAX || kv_heads > INT32_MAX / 1024)
        throw std::invalid_argument("paged cache: too many pages or heads");
    require_gpu(options.device, "paged cache");
    const Shape shape{pages, kv_heads, page_size, head_dim};
    for (Index layer = 0; layer < layers; ++layer) {
        key_.push_back(empty_tensor(shape, options.dtype, options.device));
        value_.push_back(empty_tensor(shape, options.dtype, options.device));
    }
}

namespace {

// Row tiles of one kind that see `seen` keys each, for every KV head, and what their work-groups take.
struct Load {
    std::vector<Index> seen;
    Index kv_heads, head_dim, rows, used_rows; // used: the most rows that a tile really has
    bool f32;
    bool merged; // the rows are merged anyway (with a prefix)
    bool beside; // there are tiles of many rows in the launch
};

// Keys per item: the split with the smallest time by this account, in microseconds (measured on MI355X).  `slots` work-groups
// run at once; `rate` is what each takes in a microsecond then, in keys.
// Few rows: memory gives 5.4 TB/s to all.  The items run in rounds of `slots`; in the last, of fewer, each is faster, up to
// three times, and the longest counts.  An item takes 4 more to begin and to end, a merge 6, and the partials, written and
// read, their bytes at 2.5 TB/s.
// Many rows: 8500 / (products of a pair's entry, twice the head size), what the matrix cores do: 22 keys for bf16 pages and
// heads of 64, 11 for heads of 128 or f32 pages; a work-group with a CU to itself 1.75 times that.  An item takes 5 more; the
// last ones, the longest having come first, run a sixth of an item alone.  The bytes of partials go at 2.5 TB/s, of a prefix at 1.5
// (fitted: it stands too for the items of few rows of the same launch, which are accounted for apart).
// (8 sequences of 32768 keys, a row each: 64 items of 2048 keys a head 133 us, of 768 124, of 256 139.  64 runs of 5 after up to
// 1000, f32: items of 256 61 us, whole 48.  3000 new rows after 1000: whole 335 us, in 512 keys 366.  16 runs of 192 rows
// after up to 2000 keys, 256 work-groups: whole 58 us, in 1024 keys 44.  Over 120 batches of few rows the choice is 4 % off
// the best of seven sizes in the mean, a third at most, over 36 of many 1.5 and 12 %.)
Index chunk_of(const Load& load) {
    if (load.seen.empty()) return 256;
    const bool many = load.rows == 128, wide = load.head_dim == 128;
    // fitted: no more than registers and LDS leave room for (up to 8 for f32 heads of 16, 3 for bf16 queries at bf16 heads of 128,
    // 3 or 4 for heads of 16 and 32 beside items of many rows)
    const Index per_cu = many || load.beside ? 2 : !load.f32 ? (wide ? 2 : 4) : load.rows == 32 && load.head_dim >= 64 ? 2 : wide ? 3 : 4;
    const double slots = 256.0 * static_cast<double>(per_cu), heads = static_cast<double>(load.kv_heads);
    const double dim = static_cast<double>(load.head_dim), partial = heads * static_cast<double>(load.used_rows) * dim * 8.0;
    const double rate = many ? 8500.0 / (dim * (load.f32 ? 12.0 : 6.0)) : 5.4e6 / (slots * dim * (load.f32 ? 8.0 : 4.0));
    const Index longest = *std::max_element(load.seen.begin(), load.seen.end());
    const double work = static_cast<double>(std::accumulate(load.seen.begin(), load.seen.end(), Index(0)));
    double best = 0.0;
    Index chosen = 0;
    for (Index chunk = 128, step = 1;; chunk += 128 * step) {
        Index items = 0, partials = 0;
        for (const Index keys : load.seen) {
            const Index n = (keys + chunk - 1) / chunk;
            items += n;
            if (n > 1 || load.merged) partials += n;
        }
        const double n = static_cast<double>(items), most = static_cast<double>(std::min(chunk, longest));
        double time;
        if (many) {
            time = std::max(most / rate / 1.75 + 5.0, (work / rate + 5.0 * n) * heads / slots + most / rate / 6.0);
        } else {
            const double rounds = std::floor(n * heads / slots), rest = n * heads - rounds * slots;
            time = rounds * (4.0 + work / n / rate);
            if (rest > 0.0) time += 4.0 + most / (rate * std::min(slots / rest, 3.0));
        }
        if (partials > 0)
            time += (load.merged ? 0.0 : 6.0) + static_cast<double>(partials) * partial / (many && load.merged ? 1.5e6 : 2.5e6);
        if (chosen == 0 || time < best) best = time, chosen = chunk;
        if (chunk >= longest) return chosen;
        if (chunk >= 1024 * step) step *= 2;
    }
}

} // namespace

PagedBatch::PagedBatch(const PagedKVCache& cache, Index heads, std::span<const Index> lengths, std::span<const Index> counts,
                       std::span<const Index> tables, Index width, Index shared) {
    const Index batch = static_cast<Index>(lengths.size()), page = cache.page_size();
    const auto refuse = [](const std::string& what) { throw std::invalid_argument("paged batch: " + what); };
    if (heads <= 0 || heads % cache.kv_heads() != 0) refuse("heads must be a multiple of the cache's kv_heads");
    if (heads > INT32_MAX / 1024) refuse("too many heads");
    if (batch <= 0 || counts.size() != lengths.size()) refuse("needs a length and a count for each of its sequences");
    if (width <= 0 || width > INT32_MAX / batch || tables.size() != static_cast<std::size_t>(batch * width))
        refuse("tables must be [sequences, width]");
    if (shared < 0 || shared % page != 0) refuse("the shared prefix must be whole pages");

    auto plan = std::make_shared<Plan>();
    plan->heads = heads;
    plan->kv_heads = cache.kv_heads();
    plan->head_dim = cache.head_dim();
    plan->page_size = page;
    plan->pages = cache.pages();
    plan->dtype = cache.dtype();
    plan->device = cache.device();

    const Index group = heads / cache.kv_heads();
    int shift = 0;
    while ((Index(1) << shift) < page) ++shift;

    // every id that a kernel will follow, and the pages that the step writes
    std::vector<std::uint8_t> written(static_cast<std::size_t>(cache.pages()), 0);
    Index tokens = 0, front = -1;
    for (Index b = 0; b < batch; ++b) {
        const Index length = lengths[b], count = counts[b];
        if (length < 0 || count < 0 || length > width * page || count > width * page - length || length + count > (1 << 30))
            refuse("sequence " + std::to_string(b) + " has positions outside its table");
        if (count == 0) continue;
        const Index used = (length + count + page - 1) / page;
        for (Index i = 0; i < used; ++i) {
            const Index id = tables[b * width + i];
            if (id < 0 || id >= cache.pages())
                refuse("page " + std::to_string(id) + " of sequence " + std::to_string(b) + " is not in the cache");
        }
        for (Index i = length / page; i < used; ++i) {
            auto& mark = written[static_cast<std::size_t>(tables[b * width + i])];
            if (mark) refuse("page " + std::to_string(tables[b * width + i]) + " would be written at two places");
            mark = 1;
        }
        if (shared > length) refuse("sequence " + std::to_string(b) + " does not hold the shared prefix");
        if (front < 0) front = b;
        if (!std::equal(tables.begin() + b * width, tables.begin() + b * width + shared / page, tables.begin() + front * width))
            refuse("sequence " + std::to_string(b) + " does not begin with the shared pages");
        tokens += count;
        plan->last = std::max(plan->last, length + count - 1);
    }
    for (Index b = 0; b < batch; ++b) // a page that is written appears nowhere else
        for (Index i = 0; counts[b] > 0 && i < lengths[b] / page; ++i)
            if (written[static_cast<std::size_t>(tables[b * width + i])])
                refuse("page " + std::to_string(tables[b * width + i]) + " is written and belongs to another place too");
    if (tokens > INT32_MAX / heads || tokens >= 1 << 30) refuse("too many new positions");
    plan->tokens = tokens;

    // Row tiles: of 128 for the waves to split, and what is left, if it is no more than 32, like runs of few rows in one of
    // 16 or 32, whose keys they split: its 128 would take as long as full ones.  (16 runs of 144 rows after up to 2000 keys,
    // bf16, heads of 64: 54 us with the last 16 in a tile of 128, 33 in one of 16.  Two tiles of 32 for 33 to 64 rows gain
    // a tenth where keys are few, and lose up to a third on f32 pages.)  The runs of few rows settle which of the two, 16
    // where all of them fit: 32 take more registers (32 tokens of 4096 keys: 39 us, 48 us).
    auto& lists = plan->lists;
    lists[DLK_PAGED_MANY].rows = 128;
    Index& few = lists[DLK_PAGED_FEW].rows;
    few = 0;
    Index tails = 16;
    const auto settle = [&](Index rows) {
        if (rows > 0 && rows <= 32) few = std::max<Index>(few, rows <= 16 ? 16 : 32);
        if (rows % 128 > 16 && rows % 128 <= 32) tails = 32;
    };
    for (Index b = 0; b < batch; ++b) settle(counts[b] * group);
    if (shared > 0) settle(tokens * group);
    if (few == 0) few = tails;
    struct Tile {
        Index begin, end;
        int kind;
    };
    const auto tiles_of = [&](Index rows) {
        std::vector<Tile> tiles;
        for (Index row = 0; row < rows; row += 128)
            tiles.push_back({row, std::min(rows, row + 128), rows - row <= few ? DLK_PAGED_FEW : DLK_PAGED_MANY});
        return tiles;
    };

    // how many keys an item takes: of the runs' own (behind the shared ones), and of the shared ones
    Load loads[2];
    bool beside = shared > 0 && tokens * group > few;
    for (Index b = 0; b < batch; ++b) beside = beside || counts[b] * group > few;
    const auto load_of = [&](int kind, bool merged) {
        return Load{{}, cache.kv_heads(), cache.head_dim(), lists[kind].rows, 1, cache.dtype() == DType::f32, merged, beside};
    };
    for (int kind = 0; kind < 2; ++kind) loads[kind] = load_of(kind, shared > 0);
    for (Index b = 0; b < batch; ++b) {
        const auto tiles = tiles_of(counts[b] * group);
        for (const Tile& tile : tiles) {
            if (tile.kind != tiles[0].kind) continue; // (what is left of a run of many goes along)
            loads[tile.kind].seen.push_back(lengths[b] - shared + (tile.end - 1) / group + 1);
            loads[tile.kind].used_rows = std::max(loads[tile.kind].used_rows, tile.end - tile.begin);
        }
    }
    const Index chunks[2] = {chunk_of(loads[0]), chunk_of(loads[1])};

    std::vector<dlk_paged_item> items[2];
    std::vector<dlk_paged_merge> merges;
    std::vector<Index> positions, places;
    positions.reserve(static_cast<std::size_t>(tokens));
    places.reserve(static_cast<std::size_t>(tokens));
    const auto place = [](Index n) { return static_cast<int32_t>(n); }; // (checked below)
    if (shared > 0 && tokens > 0) {
        const Index rows = tokens * group;
        const auto tiles = tiles_of(rows);
        Load load = load_of(tiles[0].kind, true);
        for (const Tile& tile : tiles)
            if (tile.kind == tiles[0].kind) load.seen.push_back(shared), load.used_rows = std::max(load.used_rows, tile.end - tile.begin);
        const Index chunk = chunk_of(load);
        plan->shared_splits = (shared + chunk - 1) / chunk;
        plan->shared_stride = rows;
        plan->partials = plan->shared_splits * rows;
        for (Index s = 0; s < plan->shared_splits; ++s)
            for (const Tile& tile : tiles)
                items[tile.kind].push_back({0, place(tile.begin), place(tile.end), place(front * width), place(s * chunk),
                                            place(std::min(shared, (s + 1) * chunk)), 1 << 30, place(s * rows + tile.begin)});
    }
    Index token = 0;
    for (Index b = 0; b < batch; ++b) {
        const Index count = counts[b], first = lengths[b] - shared, keys = first + count, rows = count * group;
        if (count == 0) continue;
        const auto tiles = tiles_of(rows);
        const Index chunk = chunks[tiles[0].kind], splits = (keys + chunk - 1) / chunk;
        const bool whole = splits == 1 && shared == 0;
        for (const Tile& tile : tiles) {
            const Index sees = first + (tile.end - 1) / group + 1; // keys of the tile's last row
            for (Index s = 0; s < splits && s * chunk < sees; ++s)
                items[tile.kind].push_back({place(token), place(tile.begin), place(tile.end), place(b * width + shared / page),
                                            place(s * chunk), place(std::min(sees, (s + 1) * chunk)), place(first),
                                            whole ? -1 : place(plan->partials + s * rows + tile.begin)});
        }
        for (Index i = 0; i < count; ++i) {
            const Index position = lengths[b] + i;
            positions.push_back(position);
            places.push_back((tables[b * width + position / page] << shift) + position % page);
            if (!whole)
                merges.push_back({place(token + i), place(plan->partials + i * group), place(rows), place((first + i) / chunk + 1),
                                  place((token + i) * group)});
        }
        if (!whole) plan->partials += splits * rows;
        token += count;
    }
    // the longest first, so that the last work-groups to start are short
    std::stable_sort(items[DLK_PAGED_MANY].begin(), items[DLK_PAGED_MANY].end(), [](const auto& a, const auto& b) {
        return a.key_end - a.key_begin > b.key_end - b.key_begin;
    });
    for (int i = 0; i < 2; ++i) lists[i].count = static_cast<Index>(items[i].size());
    plan->merge_count = static_cast<Index>(merges.size());
    if (plan->partials > INT32_MAX / cache.kv_heads() ||
        !dlk_paged_fits(lists[0].count + lists[1].count, plan->merge_count, static_cast<int>(heads), static_cast<int>(cache.kv_heads()),
                        static_cast<int>(cache.head_dim())))
        refuse("too many new positions");
    for (const auto& merge : merges) plan->merge_most = std::max<Index>(plan->merge_most, merge.count + plan->shared_splits);

    // one copy to the device
    std::vector<std::int32_t> ids(tables.size());
    for (std::size_t i = 0; i < ids.size(); ++i)
        ids[i] = tables[i] >= 0 && tables[i] < cache.pages() ? static_cast<std::int32_t>(tables[i]) : 0;
    std::vector<char> bytes;
    const auto put = [&](const auto& array) {
        const std::size_t at = (bytes.size() + 15) / 16 * 16, size = array.size() * sizeof(array[0]);
        bytes.resize(at + size);
        if (size) std::memcpy(bytes.data() + at, array.data(), size);
        return at;
    };
    plan->tables = put(ids);
    for (int i = 0; i < 2; ++i) lists[i].items = put(items[i]);
    plan->merges = put(merges);
    plan->positions = put(positions);
    plan->places = put(places);
    bytes.resize((bytes.size() + 7) / 8 * 8);
    plan->blob = from_host(bytes.data(), {static_cast<Index>(bytes.size() / 8)}, DType::i64, false, cache.device());
    plan_ = std::move(plan);
}

Index PagedBatch::tokens() const { return plan_->tokens; }

} // namespace dl::nn

namespace dl {

using namespace detail;

namespace {
// the step's plan belongs to caches of this layout
const nn::PagedBatch::Plan& plan_for(const nn::PagedKVCache& cache, Index layer, const nn::PagedBatch& batch,
                                     const char* operation) {
    const auto& plan = batch.plan();
    if (plan.kv_heads != cache.kv_heads() || plan.head_dim != cache.head_dim() || plan.page_size != cache.page_size() ||
        plan.pages != cache.pages() || plan.dtype != cache.dtype() || !(plan.device == cache.device()))
        throw std::invalid_argument(std::string(operation) + ": the batch was made for a cache of another layout");
    if (layer < 0 || layer >= cache.layers()) throw std::out_of_range(std::string(operation) + ": layer out of range");
    return plan;
}

void check_rows(const Tensor& t, Index tokens, Index heads, Index dim, Device device, const char* operation,
                const char* what) {
    if (t.shape() != Shape{tokens, heads, dim})
        throw std::invalid_argument(std::string(operation) + ": " + what + " must be " + shape_string({tokens, heads, dim}) +
                                    ", got " + shape_string(t.shape()));
    if (t.dtype() != DType::f32 && t.dtype() != DType::bf16)
        throw std::invalid_argument(std::string(operation) + ": " + what + " must be f32 or bf16");
    if (!(t.device() == device)) throw std::invalid_argument(std::string(operation) + ": " + what + " on another device");
}

// What lies in the pages that a call writes would be read while it changes: it is read from a copy.
Tensor apart_from(const nn::PagedKVCache& cache, Index layer, const Tensor& t) {
    if (!t.defined()) return t; // (its reader refuses it)
    const auto& storage = TensorAccess::impl(t)->storage;
    for (const Tensor* pages : {&cache.key(layer), &cache.value(layer)})
        if (storage == TensorAccess::impl(*pages)->storage) return t.clone();
    return t;
}

int page_shift(Index page_size) {
    int shift = 0;
    while ((Index(1) << shift) < page_size) ++shift;
    return shift;
}
} // namespace

Tensor paged_append(const nn::PagedKVCache& cache, Index layer, const nn::PagedBatch& batch,
                    const std::optional<Tensor>& query, const Tensor& key, const Tensor& value, const Tensor& cosine,
                    const Tensor& sine, RotaryLayout layout) {
    constexpr const char* name = "paged_append";
    const auto& plan = plan_for(cache, layer, batch, name);
    const Index kv = cache.kv_heads(), dim = cache.head_dim();
    check_rows(key, plan.tokens, kv, dim, cache.device(), name, "key");
    check_rows(value, plan.tokens, kv, dim, cache.device(), name, "value");
    if (query) check_rows(*query, plan.tokens, plan.heads, dim, cache.device(), name, "query");
    RotaryTables tables(apart_from(cache, layer, cosine), apart_from(cache, layer, sine), dim, cache.device(), name);
    if (plan.last >= tables.capacity())
        throw std::out_of_range(std::string(name) + ": position " + std::to_string(plan.last) + " lies beyond the tables");
    GpuContext& context = gpu_of(key, name);
    dlk_rotary_params p{};
    tables.fill(p, layout, name);
    Tensor out = query ? empty_tensor(query->shape(), DType::f32, cache.device()) : Tensor{};
    if (plan.tokens == 0) return out;
    Tensor q, k, v;
    p.tokens = plan.tokens;
    p.dim = static_cast<int>(dim);
    if (query) {
        p.q = row_segment(apart_from(cache, layer, *query), q, plan.heads, name);
        p.out = static_cast<float*>(mutable_data(out));
    }
    p.k = row_segment(apart_from(cache, layer, key), k, kv, name);
    p.v = row_segment(apart_from(cache, layer, value), v, kv, name);
    p.positions = plan.at<Index>(plan.positions);
    p.places = plan.at<Index>(plan.places);
    p.k_pages = mutable_data(cache.key(layer));
    p.v_pages = mutable_data(cache.value(layer));
    p.pages_bf16 = cache.dtype() == DType::bf16;
    p.page_shift = page_shift(cache.page_size());
    hip_check(dlk_rotary(&p, context.stream), name);
    return out;
}

Tensor paged_attention(const nn::PagedKVCache& cache, Index layer, const nn::PagedBatch& batch, const Tensor& query) {
    constexpr const char* name = "paged_attention";
    const auto& plan = plan_for(cache, layer, batch, name);
    const Index kv = cache.kv_heads(), dim = cache.head_dim();
    check_rows(query, plan.tokens, plan.heads, dim, cache.device(), name, "query");
    GpuContext& context = gpu_of(query, name);
    Tensor out = empty_tensor(query.shape(), DType::f32, cache.device());
    if (plan.tokens == 0) return out;
    // the kernels read 16 bytes of a row at a time
    const Index align = query.dtype() == DType::bf16 ? 8 : 4;
    const auto& strides = query.strides();
    const bool direct = strides[2] == 1 && strides[0] % align == 0 && strides[1] % align == 0 &&
                        reinterpret_cast<std::uintptr_t>(query.data<void>()) % 16 == 0;
    Tensor q = query;
    if (!direct) {
        q = empty_tensor(query.shape(), query.dtype(), query.device());
        copy_into(q, query);
    }
    dlk_paged_params p{};
    p.q = q.data<void>();
    p.q_bf16 = q.dtype() == DType::bf16;
    p.q_row = q.strides()[0];
    p.q_head = q.strides()[1];
    p.k = cache.key(layer).data<void>();
    p.v = cache.value(layer).data<void>();
    p.kv_bf16 = cache.dtype() == DType::bf16;
    p.page_shift = page_shift(cache.page_size());
    p.H = static_cast<int>(plan.heads);
    p.KV = static_cast<int>(kv);
    p.hd = static_cast<int>(dim);
    p.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim)));
    p.tables = plan.at<std::int32_t>(plan.tables);
    p.out = static_cast<float*>(mutable_data(out));
    p.shared_splits = static_cast<int>(plan.shared_splits);
    p.shared_stride = static_cast<int>(plan.shared_stride);
    p.merges = plan.at<dlk_paged_merge>(plan.merges);
    p.merge_count = static_cast<int>(plan.merge_count);
    p.merge_most = static_cast<int>(plan.merge_most);
    // partials, released to the pool in stream order
    const Index rows = plan.partials * kv;
    Tensor partials = rows > 0 ? empty_tensor({rows * (dim + 2)}, DType::f32, cache.device()) : Tensor{};
    p.partial_o = rows > 0 ? static_cast<float*>(mutable_data(partials)) : nullptr;
    p.partial_ml = rows > 0 ? p.partial_o + rows * dim : nullptr;
    p.places = static_cast<int>(plan.partials);
    for (int i = 0; i < 2; ++i)
        p.lists[i] = {plan.at<dlk_paged_item>(plan.lists[i].items), static_cast<int>(plan.lists[i].count), static_cast<int>(plan.lists[i].rows)};
    hip_check(dlk_paged_attention(&p, context.stream), name);
    return out;
}

} // namespace dl
