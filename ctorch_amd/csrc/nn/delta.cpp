// The states of the gated delta rule, the plan of a step over them, and its operator (include/dl/delta.h).
#include "nn/delta_plan.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <stdexcept>

namespace dl::nn {

using namespace dl::detail;

DeltaStates::DeltaStates(Index layers, Index slots, Index heads, Index key_dim, Index value_dim, Device device)
    : slots_(slots), heads_(heads), key_dim_(key_dim), value_dim_(value_dim), device_(device) {
    if (layers <= 0 || slots <= 0 || heads <= 0)
        throw std::invalid_argument("delta states: layers, slots and heads must be positive");
    if (key_dim != 32 && key_dim != 64 && key_dim != 128)
        throw std::invalid_argument("delta states: key_dim must be 32, 64 or 128");
    if (value_dim <= 0 || value_dim % 32 != 0 || value_dim > 256)
        throw std::invalid_argument("delta states: value_dim must be a multiple of 32 up to 256");
    if (slots > INT32_MAX || heads > 16384)
        throw std::invalid_argument("delta states: too many slots or heads");
    require_gpu(device, "delta states");
    for (Index layer = 0; layer < layers; ++layer)
        state_.push_back(zeros({slots, heads, key_dim, value_dim}, {.dtype = DType::f32, .device = device}));
}

DeltaBatch::DeltaBatch(const DeltaStates& states, Index key_heads, std::span<const Index> sources,
                       std::span<const Index> targets, std::span<const Index> counts) {
    const auto refuse = [](const std::string& what) { throw std::invalid_argument("delta batch: " + what); };
    if (key_heads <= 0 || states.heads() % key_heads != 0) refuse("the states' heads must be a multiple of key_heads");
    if (counts.empty() || sources.size() != counts.size() || targets.size() != counts.size())
        refuse("needs a source, a target and a count for each of its requests");
    auto plan = std::make_shared<Plan>();
    plan->heads = states.heads();
    plan->key_heads = key_heads;
    plan->key_dim = states.key_dim();
    plan->value_dim = states.value_dim();
    plan->slots = states.slots();
    plan->device = states.device();

    std::vector<Index> writer(static_cast<std::size_t>(states.slots()), -1);
    const auto batch = static_cast<Index>(counts.size());
    for (Index b = 0; b < batch; ++b) {
        if (counts[b] < 0) refuse("a count below zero");
        if (counts[b] == 0) continue;
        if (targets[b] < 0 || targets[b] >= states.slots()) refuse("slot " + std::to_string(targets[b]) + " is not among the states");
        if (sources[b] < -1 || sources[b] >= states.slots()) refuse("slot " + std::to_string(sources[b]) + " is not among the states");
        auto& mark = writer[static_cast<std::size_t>(targets[b])];
        if (mark >= 0) refuse("slot " + std::to_string(targets[b]) + " would be written by two requests");
        mark = b;
        if (counts[b] > (1 << 30) - plan->tokens) refuse("too many new tokens");
        plan->tokens += counts[b];
    }
    if (plan->tokens > INT32_MAX / states.heads()) refuse("too many new tokens");
    // Up to so many tokens a request's go one after the other, 0.6 to 1 us each; more in chunks, which take two launches and, where
    // requests, heads and columns make more work-groups than run at once, rounds of 5 us.  Measured on MI355X, us one by one / in
    // chunks: one request of 32 heads of 128 x 128, 16 tokens 18.7 / 19.8, 24 26.4 / 20.2; 16 such requests, 32 tokens 54 / 99, 64
    // 88 / 107; one request of 8 heads of 64 x 64 in f32, 24 tokens 18.0 / 19.4, 48 33.5 / 19.5; 16 such 24 tokens 18 / 28, 48 33 / 28.
    Index busy = 0;
    for (const Index count : counts) busy += count > 0;
    // (a launch has fewer than 2^32 threads: so many columns of 16)
    if (busy > (1 << 22) / (states.heads() * (states.value_dim() / 16))) refuse("too many requests at once");
    const Index few = std::min<Index>(64, 16 + 3 * (busy * states.heads() * (states.value_dim() / 16) / 256));
    // (of chunks and heads: 26 KB of workspace each, and the keys' copies)
    constexpr Index most = 8192;
    const Index round_chunks = std::max<Index>(1, most / states.heads());
    std::vector<dlk_delta_item> items, rest; // rest: requests of many tokens, then what is left of them
    std::vector<dlk_delta_chunk> chunks;
    Index token = 0;
    for (Index b = 0; b < batch; ++b) {
        if (counts[b] == 0) continue;
        if (sources[b] >= 0) {
            const Index by = writer[static_cast<std::size_t>(sources[b])];
            if (by >= 0 && by != b) refuse("slot " + std::to_string(sources[b]) + " is written by one request and read by another");
        }
        (counts[b] <= few ? items : rest)
            .push_back({static_cast<int32_t>(sources[b]), static_cast<int32_t>(targets[b]), static_cast<int32_t>(token),
                        static_cast<int32_t>(counts[b]), 0, 0});
        token += counts[b];
    }
    plan->few = static_cast<Index>(items.size());
    while (!rest.empty()) {
        // the requests side by side, each by as many chunks as leave some for all
        const Index each = std::max<Index>(1, round_chunks / static_cast<Index>(rest.size()));
        Plan::Round round{static_cast<Index>(items.size()), 0, static_cast<Index>(chunks.size()), 0};
        std::vector<dlk_delta_item> left;
        for (dlk_delta_item& item : rest) {
            if (round.chunks >= round_chunks) {
                left.push_back(item);
                continue;
            }
            const Index n = std::min<Index>((item.count + 63) / 64, std::min(each, round_chunks - round.chunks));
            dlk_delta_item now = item;
            now.count = static_cast<int32_t>(std::min<Index>(item.count, 64 * n));
            now.chunk = static_cast<int32_t>(round.chunks);
            for (Index i = 0; i < n; ++i)
                chunks.push_back({static_cast<int32_t>(item.token + 64 * i), static_cast<int32_t>(std::min<Index>(64, item.count - 64 * i))});
            round.chunks += n;
            round.items += 1;
            items.push_back(now);
            if (now.count < item.count) left.push_back({item.target, item.target, item.token + now.count, item.count - now.count, 0, 0});
        }
        plan->rounds.push_back(round);
        rest = std::move(left);
    }
    plan->chunks = items.size() * sizeof(dlk_delta_item);
    std::vector<char> bytes(plan->chunks + chunks.size() * sizeof(dlk_delta_chunk));
    if (!items.empty()) {
        std::memcpy(bytes.data(), items.data(), plan->chunks);
        if (!chunks.empty()) std::memcpy(bytes.data() + plan->chunks, chunks.data(), bytes.size() - plan->chunks);
        plan->blob = from_host(bytes.data(), {static_cast<Index>(bytes.size() / 8)}, DType::i64, false, states.device());
    }
    plan_ = std::move(plan);
}

Index DeltaBatch::tokens() const { return plan_->tokens; }

} // namespace dl::nn

namespace dl {

using namespace detail;

namespace {
// A segment of rows whose pieces of 16 bytes a kernel reads whole, from a copy where they are not aligned, or lie in the
// states, which the call writes.
dlk_row_segment aligned_rows(const Tensor& t, Tensor& held, Index tokens, Index heads, Index dim, const Tensor& states,
                             const char* what) {
    const std::string name("gated_delta");
    if (t.shape() != Shape{tokens, heads, dim})
        throw std::invalid_argument(name + ": " + what + " must be " + shape_string({tokens, heads, dim}) + ", got " + shape_string(t.shape()));
    if (t.dtype() != DType::f32 && t.dtype() != DType::bf16) throw std::invalid_argument(name + ": " + what + " must be f32 or bf16");
    if (!(t.device() == states.device())) throw std::invalid_argument(name + ": " + what + " on another device");
    const Index align = t.dtype() == DType::bf16 ? 8 : 4;
    const auto& strides = t.strides();
    // (64 rows lie within 2^32 entries, which a kernel counts in 32 bits)
    const bool direct = strides[2] == 1 && strides[0] % align == 0 && strides[1] % align == 0 && strides[0] < (1 << 26) &&
                        reinterpret_cast<std::uintptr_t>(t.data<void>()) % 16 == 0 &&
                        TensorAccess::impl(t)->storage != TensorAccess::impl(states)->storage;
    held = t;
    if (!direct) {
        held = empty_tensor(t.shape(), t.dtype(), t.device());
        copy_into(held, t);
    }
    dlk_row_segment s{};
    s.x = held.data<void>();
    s.bf16 = held.dtype() == DType::bf16;
    s.heads = static_cast<int>(heads);
    s.row = held.strides()[0];
    s.head = held.strides()[1];
    return s;
}

Tensor gates(const Tensor& t, Index tokens, Index heads, const Tensor& states, const char* what) {
    const std::string name("gated_delta");
    if (t.shape() != Shape{tokens, heads})
        throw std::invalid_argument(name + ": " + what + " must be " + shape_string({tokens, heads}) + ", got " + shape_string(t.shape()));
    if (t.dtype() != DType::f32 && t.dtype() != DType::bf16) throw std::invalid_argument(name + ": " + what + " must be f32 or bf16");
    if (!(t.device() == states.device())) throw std::invalid_argument(name + ": " + what + " on another device");
    if (TensorAccess::impl(t)->storage == TensorAccess::impl(states)->storage) return contiguous_f32(t.clone());
    return contiguous_f32(t);
}
} // namespace

Tensor gated_delta(const nn::DeltaStates& states, Index layer, const nn::DeltaBatch& batch, const Tensor& query,
                   const Tensor& key, const Tensor& value, const Tensor& decay, const Tensor& rate, std::optional<double> scale) {
    constexpr const char* name = "gated_delta";
    const auto& plan = batch.plan();
    if (plan.heads != states.heads() || plan.key_dim != states.key_dim() || plan.value_dim != states.value_dim() ||
        plan.slots != states.slots() || !(plan.device == states.device()))
        throw std::invalid_argument(std::string(name) + ": the batch was made for states of another layout");
    if (layer < 0 || layer >= states.layers()) throw std::out_of_range(std::string(name) + ": layer out of range");
    if (scale && !(std::abs(*scale) <= std::numeric_limits<float>::max()))
        throw std::invalid_argument(std::string(name) + ": the scale must be finite in f32");
    const Tensor& state = states.state(layer);
    Tensor q, k, v;
    dlk_delta_params p{};
    // (the kernels take queries and keys of one type)
    const bool mixed = query.dtype() != key.dtype() && is_floating(query.dtype()) && is_floating(key.dtype());
    const auto alike = [&](const Tensor& t) { return mixed && t.dtype() == DType::bf16 ? t.astype(DType::f32) : t; };
    p.q = aligned_rows(alike(query), q, plan.tokens, plan.key_heads, plan.key_dim, state, "query");
    p.k = aligned_rows(alike(key), k, plan.tokens, plan.key_heads, plan.key_dim, state, "key");
    p.v = aligned_rows(value, v, plan.tokens, plan.heads, plan.value_dim, state, "value");
    const Tensor g = gates(decay, plan.tokens, plan.heads, state, "decay"), b = gates(rate, plan.tokens, plan.heads, state, "rate");
    GpuContext& context = gpu_of(state, name);
    Tensor out = empty_tensor({plan.tokens, plan.heads, plan.value_dim}, DType::f32, states.device());
    if (plan.tokens == 0) return out;
    p.decay = g.data<float>();
    p.rate = b.data<float>();
    p.states = static_cast<float*>(mutable_data(state));
    p.out = static_cast<float*>(mutable_data(out));
    p.heads = static_cast<int>(plan.heads);
    p.group = static_cast<int>(plan.heads / plan.key_heads);
    p.key_dim = static_cast<int>(plan.key_dim);
    p.value_dim = static_cast<int>(plan.value_dim);
    p.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(plan.key_dim)));
    const auto* items = reinterpret_cast<const dlk_delta_item*>(plan.blob.data<char>());
    const auto* chunks = reinterpret_cast<const dlk_delta_chunk*>(plan.blob.data<char>() + plan.chunks);
    Tensor workspace; // of the largest round; released to the pool in stream order
    Index most = 0;
    for (const auto& round : plan.rounds) most = std::max(most, round.chunks);
    if (most > 0) {
        p.chunk_count = static_cast<int>(most);
        workspace = empty_tensor({dlk_delta_workspace(&p) / 4}, DType::f32, states.device());
    }
    p.items = items;
    p.item_count = static_cast<int>(plan.few);
    hip_check(dlk_delta_step(&p, context.stream), name);
    for (const auto& round : plan.rounds) {
        p.items = items + round.first;
        p.item_count = static_cast<int>(round.items);
        p.chunks = chunks + round.first_chunk;
        p.chunk_count = static_cast<int>(round.chunks);
        hip_check(dlk_delta_chunks(&p, mutable_data(workspace), context.stream), name);
    }
    return out;
}

void delta_copy(const nn::DeltaStates& states, std::span<const Index> sources, std::span<const Index> targets) {
    std::vector<void*> pools;
    for (Index layer = 0; layer < states.layers(); ++layer) pools.push_back(mutable_data(states.state(layer)));
    copy_pages(pools, states.slots(), states.heads(), states.key_dim(), states.value_dim() * 4, states.device(), sources, targets, {},
               "delta_copy");
}

} // namespace dl
