// Entries of <dl/decoder_c_api.h> for serving loops: page pools, forks and compaction, the gated delta rule, experts.
#include "api/common.h"
#include "core/tensor_impl.h"

#include <algorithm>
#include <stdexcept>

using namespace dl::capi;

namespace {
// `count` ids at `data`, which may be NULL only where there are none
template <class T> std::span<T> ids(T* data, int64_t count, const char* what) {
    if (count < 0) throw std::invalid_argument(std::string(what) + ": a count below zero");
    if (count > 0) require(data, what);
    return {data, static_cast<std::size_t>(count)};
}

int64_t table_ids(int64_t sequences, int64_t width) {
    if (sequences < 0 || width <= 0 || (sequences > 0 && width > INT32_MAX / sequences))
        throw std::invalid_argument("tables must be [sequences, width]");
    return sequences * width;
}
} // namespace

extern "C" {

dl_status dl_page_pool_create(int64_t pages, dl_page_pool** output) {
    return make_handle(output, [&] { return dl::nn::PagePool(pages); });
}

void dl_page_pool_release(dl_page_pool* pool) { delete pool; }

dl_status dl_page_pool_available(const dl_page_pool* pool, int64_t* available) {
    return invoke([&] { require(available, "available slot") = require(pool, "pool").value.available(); });
}

dl_status dl_page_pool_references(const dl_page_pool* pool, int64_t page, int64_t* references) {
    return invoke([&] { require(references, "references slot") = require(pool, "pool").value.references(page); });
}

dl_status dl_page_pool_take(dl_page_pool* pool, int64_t count, int64_t* pages) {
    return invoke([&] {
        auto& p = require(pool, "pool").value;
        if (count > 0) require(pages, "pages");
        std::ranges::copy(p.take(count), pages);
    });
}

dl_status dl_page_pool_claim(dl_page_pool* pool, int64_t count, const int64_t* pages) {
    return invoke([&] { require(pool, "pool").value.claim(ids(pages, count, "pages")); });
}

dl_status dl_page_pool_share(dl_page_pool* pool, int64_t count, const int64_t* pages) {
    return invoke([&] { require(pool, "pool").value.share(ids(pages, count, "pages")); });
}

dl_status dl_page_pool_give_back(dl_page_pool* pool, int64_t count, const int64_t* pages) {
    return invoke([&] { require(pool, "pool").value.release(ids(pages, count, "pages")); });
}

dl_status dl_paged_cache_copy(dl_paged_cache* cache, int64_t count, const int64_t* sources, const int64_t* targets,
                              const int64_t* rows) {
    return invoke([&] {
        dl::paged_copy(require(cache, "cache").value, ids(sources, count, "sources"), ids(targets, count, "targets"),
                       rows ? ids(rows, count, "rows") : std::span<const int64_t>{});
    });
}

dl_status dl_paged_cache_fork(dl_paged_cache* cache, dl_page_pool* pool, int64_t sequences, const int64_t* tables, int64_t width,
                              const int64_t* lengths, int64_t children, const int64_t* parents, int64_t* forked) {
    return invoke([&] {
        const auto all = ids(tables, table_ids(sequences, width), "tables");
        const auto own = ids(forked, table_ids(children, width), "forked");
        std::ranges::copy(dl::paged_fork(require(cache, "cache").value, require(pool, "pool").value, all, width,
                                         ids(lengths, sequences, "lengths"), ids(parents, children, "parents")),
                          own.begin());
    });
}

dl_status dl_paged_cache_compact(dl_paged_cache* cache, dl_page_pool* pool, int64_t count, int64_t* tables, int64_t* moved) {
    return invoke([&] {
        const auto n = dl::paged_compact(require(cache, "cache").value, require(pool, "pool").value, ids(tables, count, "tables"));
        if (moved) *moved = n;
    });
}

dl_status dl_delta_states_create(int64_t layers, int64_t slots, int64_t heads, int64_t key_dim, int64_t value_dim,
                                 dl_device device, dl_delta_states** output) {
    return make_handle(output, [&] { return dl::nn::DeltaStates(layers, slots, heads, key_dim, value_dim, convert(device)); });
}

void dl_delta_states_release(dl_delta_states* states) { delete states; }

dl_status dl_delta_states_tensor(const dl_delta_states* states, int64_t layer, dl_tensor** output) {
    return make_handle(output, [&] {
        const auto& s = require(states, "states").value;
        if (layer < 0 || layer >= s.layers()) throw std::out_of_range("delta states: layer out of range");
        return s.state(layer).detach();
    });
}

dl_status dl_delta_states_copy(dl_delta_states* states, int64_t count, const int64_t* sources, const int64_t* targets) {
    return invoke([&] {
        dl::delta_copy(require(states, "states").value, ids(sources, count, "sources"), ids(targets, count, "targets"));
    });
}

dl_status dl_delta_batch_create(const dl_delta_states* states, int64_t key_heads, int64_t requests, const int64_t* sources,
                                const int64_t* targets, const int64_t* counts, dl_delta_batch** output) {
    return make_handle(output, [&] {
        return dl::nn::DeltaBatch(require(states, "states").value, key_heads, ids(sources, requests, "sources"),
                                  ids(targets, requests, "targets"), ids(counts, requests, "counts"));
    });
}

void dl_delta_batch_release(dl_delta_batch* batch) { delete batch; }

dl_status dl_gated_delta(dl_delta_states* states, int64_t layer, const dl_delta_batch* batch, const dl_tensor* query,
                         const dl_tensor* key, const dl_tensor* value, const dl_tensor* decay, const dl_tensor* rate,
                         const double* scale, dl_tensor** output) {
    return make_handle(output, [&] {
        return dl::gated_delta(require(states, "states").value, layer, require(batch, "batch").value, require(query, "query").value,
                               require(key, "key").value, require(value, "value").value, require(decay, "decay").value,
                               require(rate, "rate").value, scale ? std::optional<double>{*scale} : std::nullopt);
    });
}

dl_status dl_expert_mixture(const dl_tensor* input, const dl_tensor* router, const dl_tensor* gate, const dl_tensor* up,
                            const dl_tensor* down, int64_t top, int32_t normalise, dl_tensor** output, dl_tensor** chosen,
                            dl_tensor** weights) {
    for (dl_tensor** slot : {output, chosen, weights})
        if (slot) *slot = nullptr;
    return invoke([&] {
        require(output, "output slot");
        auto mixed = dl::expert_mixture(require(input, "input").value, require(router, "router").value, require(gate, "gate").value,
                                        require(up, "up").value, require(down, "down").value, top, normalise != 0);
        auto y = std::make_unique<dl_tensor>(dl_tensor{mixed.output});
        auto c = chosen ? std::make_unique<dl_tensor>(dl_tensor{mixed.chosen}) : nullptr;
        auto w = weights ? std::make_unique<dl_tensor>(dl_tensor{mixed.weights}) : nullptr;
        *output = y.release();
        if (chosen) *chosen = c.release();
        if (weights) *weights = w.release();
    });
}

dl_status dl_expert_mixture_create(int64_t dimensions, int64_t hidden, int64_t experts, int64_t top, int32_t normalise,
                                   dl_tensor_options options, dl_module** output) {
    return make_handle(output, [&] {
        return std::shared_ptr<dl::nn::UnaryModule>(
            std::make_shared<dl::nn::ExpertMixture>(dimensions, hidden, experts, top, normalise != 0, convert(options)));
    });
}

} // extern "C"
