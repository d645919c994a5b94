// The paged key/value cache, the plan of a step over it, and its two operators (include/dl/paged.h).
#include "nn/paged_plan.h"

#include <algorithm>
#include <cmath>
#include <cstring>
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

constexpr Index kTileKeys = 32, kWaveTiles = 4 * kTileKeys; // keys of a wave's tile, and of a work-group's four

Index round_up(Index value, Index to) { return (value + to - 1) / to * to; }

// Keys per item where the row tiles see `total` keys in all: about `wanted` work-groups over the KV heads, of two rounds of
// the four waves' tiles at least.
Index chunk_of(Index total, Index kv_heads, Index wanted) {
    return std::max<Index>(2 * kWaveTiles, round_up((total * kv_heads + wanted - 1) / wanted, kWaveTiles));
}

} // namespace

PagedBatch::PagedBatch(const PagedKVCache& cache, Index heads, std::span<const Index> lengths, std::span<const Index> counts,
                       std::span<const Index> tables, Index width, Index shared) {
    const Index batch = static_cast<Index>(lengths.size()), page = cache.page_size();
    const auto refuse = [](const std::string& what) { throw std::invalid_argument("paged batch: " + what); };
    if (heads <= 0 || heads % cache.kv_heads() != 0) refuse("heads must be a multiple of the cache's kv_heads");
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
    if (tokens > INT32_MAX / heads) refuse("too many new positions");
    plan->tokens = tokens;

    // the runs' rows over their own keys (behind the shared ones), split where that gives more work-groups
    const Index rows_of = 16 * plan->row_tiles;
    Index total = 0;
    for (Index b = 0; b < batch; ++b)
        if (counts[b] > 0) total += (counts[b] * group + rows_of - 1) / rows_of * (lengths[b] + counts[b] - shared);
    constexpr Index kWanted = 1024; // work-groups
    const Index chunk = chunk_of(total, cache.kv_heads(), kWanted);

    std::vector<dlk_paged_item> items, shared_items;
    std::vector<dlk_paged_merge> merges;
    std::vector<Index> positions, places;
    positions.reserve(static_cast<std::size_t>(tokens));
    places.reserve(static_cast<std::size_t>(tokens));
    Index token = 0;
    for (Index b = 0; b < batch; ++b) {
        const Index count = counts[b], first = lengths[b] - shared, keys = first + count, rows = count * group;
        if (count == 0) continue;
        const Index splits = (keys + chunk - 1) / chunk;
        const bool whole = splits == 1 && shared == 0;
        for (Index row = 0; row < rows; row += rows_of) {
            const Index end = std::min(rows, row + rows_of);
            const Index seen = first + (end - 1) / group + 1; // keys that the tile's last row sees
            for (Index s = 0; s < splits && s * chunk < seen; ++s)
                items.push_back({static_cast<int32_t>(token), static_cast<int32_t>(row), static_cast<int32_t>(end),
                                 static_cast<int32_t>(b * width + shared / page), static_cast<int32_t>(s * chunk),
                                 static_cast<int32_t>(std::min(seen, (s + 1) * chunk)), static_cast<int32_t>(first),
                                 whole ? -1 : static_cast<int32_t>(plan->slots + row / rows_of * splits + s)});
        }
        for (Index i = 0; i < count; ++i) {
            const Index position = lengths[b] + i;
            positions.push_back(position);
            places.push_back((tables[b * width + position / page] << shift) + position % page);
            if (!whole)
                merges.push_back({static_cast<int32_t>(token + i), static_cast<int32_t>(i * group),
                                  static_cast<int32_t>(plan->slots), static_cast<int32_t>(splits),
                                  static_cast<int32_t>((first + i) / chunk + 1), static_cast<int32_t>((token + i) * group)});
        }
        if (!whole) plan->slots += (rows + rows_of - 1) / rows_of * splits;
        token += count;
    }
    if (shared > 0 && tokens > 0) {
        const Index rows = tokens * group;
        const Index shared_rows = 16 * plan->shared_row_tiles, tiles = (rows + shared_rows - 1) / shared_rows;
        const Index part = chunk_of(tiles * shared, cache.kv_heads(), kWanted);
        const Index splits = (shared + part - 1) / part;
        plan->shared_splits = static_cast<int>(splits);
        for (Index s = 0; s < splits; ++s)
            for (Index tile = 0; tile < tiles; ++tile)
                shared_items.push_back({0, static_cast<int32_t>(tile * shared_rows),
                                        static_cast<int32_t>(std::min(rows, (tile + 1) * shared_rows)),
                                        static_cast<int32_t>(front * width), static_cast<int32_t>(s * part),
                                        static_cast<int32_t>(std::min(shared, (s + 1) * part)), 1 << 30,
                                        static_cast<int32_t>(tile * splits + s)});
        plan->shared_slots = tiles * splits;
    }
    if (std::max<Index>({static_cast<Index>(items.size()), static_cast<Index>(shared_items.size()), plan->slots,
                         plan->shared_slots}) > INT32_MAX / cache.kv_heads())
        refuse("too many new positions");
    plan->item_count = static_cast<Index>(items.size());
    plan->shared_count = static_cast<Index>(shared_items.size());
    plan->merge_count = static_cast<Index>(merges.size());

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
    plan->items = put(items);
    plan->shared_items = put(shared_items);
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
    RotaryTables tables(cosine, sine, dim, cache.device(), name);
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
        p.q = row_segment(*query, q, plan.heads, name);
        p.out = static_cast<float*>(mutable_data(out));
    }
    p.k = row_segment(key, k, kv, name);
    p.v = row_segment(value, v, kv, name);
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
    p.items = plan.at<dlk_paged_item>(plan.items);
    p.item_count = static_cast<int>(plan.item_count);
    p.row_tiles = plan.row_tiles;
    p.shared_items = plan.at<dlk_paged_item>(plan.shared_items);
    p.shared_count = static_cast<int>(plan.shared_count);
    p.shared_row_tiles = plan.shared_row_tiles;
    p.shared_splits = plan.shared_splits;
    p.merges = plan.at<dlk_paged_merge>(plan.merges);
    p.merge_count = static_cast<int>(plan.merge_count);
    // partials, released to the pool in stream order
    const Index own_rows = plan.slots * kv * 16 * plan.row_tiles;
    const Index shared_rows = plan.shared_slots * kv * 16 * plan.shared_row_tiles;
    Tensor partials;
    if (own_rows + shared_rows > 0) {
        partials = empty_tensor({(own_rows + shared_rows) * (dim + 2)}, DType::f32, cache.device());
        p.partial_o = static_cast<float*>(mutable_data(partials));
        p.shared_o = p.partial_o + own_rows * dim;
        p.partial_ml = p.shared_o + shared_rows * dim;
        p.shared_ml = p.partial_ml + 2 * own_rows;
    }
    hip_check(dlk_paged_attention(&p, context.stream), name);
    return out;
}

} // namespace dl
