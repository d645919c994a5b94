// The paged cache's host side without a GPU, on the device of host_checks.cpp: what a step's batch refuses, and what the
// plan it makes has the kernels read and write.  Run by tests/test_paged_rules.py.
//
//   paged_checks plan PAGES PAGE_SIZE KV HEADS HEAD_DIM BF16 SHARED WIDTH LENGTHS COUNTS TABLES
//       (lists are separated by commas)  makes the batch, walks its items and merges as the kernels do, and prints the
//       numbers of tokens, items, prefix items and merges; any place out of range, key left out or seen twice, slot
//       written twice or read unwritten is an error
//   paged_checks call CASE    an operator called with arguments that it refuses (its error), or with nothing to do
#define main host_checks_main
#include "host_checks.cpp"
#undef main

#include "nn/paged_plan.h"

#include <functional>
#include <limits>
#include <optional>
#include <set>

namespace {

using dl::Index;
using dl::nn::PagedBatch;
using dl::nn::PagedKVCache;

std::vector<Index> list(const char* text) {
    std::vector<Index> out;
    for (const char* at = text; *at;) {
        char* end = nullptr;
        out.push_back(std::strtoll(at, &end, 10));
        at = *end ? end + 1 : end;
    }
    return out;
}

void expect(bool holds, const char* what) {
    if (!holds) throw std::logic_error(std::string("plan: ") + what);
}

int plan(char** arg) {
    auto at = [&](int i) { return std::atoll(arg[i]); };
    const Index pages = at(0), page_size = at(1), KV = at(2), H = at(3), shared = at(6), width = at(7);
    const PagedKVCache cache(1, pages, page_size, KV, at(4), {.dtype = at(5) ? dl::DType::bf16 : dl::DType::f32, .device = dl::Device::gpu(0)});
    const auto lengths = list(arg[8]), counts = list(arg[9]), tables = list(arg[10]);
    const PagedBatch batch(cache, H, lengths, counts, tables, width, shared);
    const auto& p = batch.plan();
    const Index G = H / KV, T = p.tokens;

    // the tokens' sequences, positions and places
    std::vector<Index> seq, position;
    for (std::size_t b = 0; b < lengths.size(); ++b)
        for (Index i = 0; i < counts[b]; ++i) seq.push_back(static_cast<Index>(b)), position.push_back(lengths[b] + i);
    expect(static_cast<Index>(seq.size()) == T, "tokens");
    std::set<Index> written;
    for (Index t = 0; t < T; ++t) {
        expect(p.at<Index>(p.positions)[t] == position[t], "position");
        const Index place = p.at<Index>(p.places)[t];
        expect(place == tables[seq[t] * width + position[t] / page_size] * page_size + position[t] % page_size, "place");
        expect(place >= 0 && place < pages * page_size && written.insert(place).second, "place written twice");
    }

    // seen[row]: the keys (positions) that the items give the row, per slot; whole: rows whose output an item writes
    using Keys = std::vector<char>;
    std::map<std::pair<Index, Index>, Keys> whole;                      // (token, g)
    std::map<Index, std::pair<std::pair<Index, Index>, Keys>> partials; // place -> row, keys
    Index fronts = 0;
    for (int kind = 0; kind < 2; ++kind) {
        const auto& list = p.lists[kind];
        const auto* items = p.at<dlk_paged_item>(list.items);
        const Index rows = list.rows;
        expect(kind == DLK_PAGED_MANY ? rows == 128 : rows == 16 || rows == 32, "rows of a list");
        for (Index n = 0; n < list.count; ++n) {
            const dlk_paged_item& i = items[n];
            const bool front = i.first == 1 << 30;
            fronts += front;
            expect(i.row_end > i.row_begin && i.row_end - i.row_begin <= rows, "rows of an item");
            expect(i.key_begin >= 0 && i.key_begin % 32 == 0 && i.key_end > i.key_begin, "keys of an item");
            expect(i.slot == -1 || (i.slot >= 0 && i.slot + i.row_end - i.row_begin <= p.partials), "slot");
            for (Index r = i.row_begin; r < i.row_end; ++r) {
                const Index token = i.token + r / G;
                expect(token >= 0 && token < T, "token of a row");
                Keys keys(static_cast<std::size_t>(position[token]) + 1, 0);
                for (Index key = i.key_begin; key < std::min<Index>(i.key_end, i.first + r / G + 1); ++key) {
                    const Index entry = i.table + key / page_size;
                    expect(entry >= 0 && entry < static_cast<Index>(tables.size()), "table entry");
                    const Index where = (front ? 0 : shared) + key;
                    expect(where < static_cast<Index>(keys.size()), "key behind the row");
                    expect(p.at<std::int32_t>(p.tables)[entry] == tables[seq[token] * width + where / page_size], "page");
                    expect((key & (page_size - 1)) == where % page_size, "row of a page");
                    keys[static_cast<std::size_t>(where)] += 1;
                }
                const auto row = std::pair(token, r % G);
                if (i.slot < 0) expect(whole.emplace(row, keys).second, "output written twice");
                else expect(partials.emplace(i.slot + r - i.row_begin, std::pair(row, keys)).second, "slot written twice");
            }
            // the pages that the item's loads may touch, to the end of its last tile's live keys
            for (Index key = i.key_begin; key < i.key_end; ++key) {
                const Index id = p.at<std::int32_t>(p.tables)[i.table + key / page_size];
                expect(id >= 0 && id < pages, "page of an item");
            }
        }
    }
    const auto* merges = p.at<dlk_paged_merge>(p.merges);
    for (Index n = 0; n < p.merge_count; ++n) {
        const dlk_paged_merge& m = merges[n];
        for (Index g = 0; g < G; ++g) {
            Keys keys(static_cast<std::size_t>(position[m.token]) + 1, 0);
            auto add = [&](Index slot) {
                const auto found = partials.find(slot);
                expect(found != partials.end(), "merge of a slot that nobody writes");
                expect(found->second.first == std::pair<Index, Index>(m.token, g), "merge of another row's slot");
                for (std::size_t k = 0; k < keys.size(); ++k) keys[k] += found->second.second[k];
            };
            for (Index s = 0; s < m.count; ++s) add(m.slot + s * m.stride + g);
            for (Index s = 0; s < p.shared_splits; ++s) add(m.shared_slot + s * p.shared_stride + g);
            expect(whole.emplace(std::pair(Index(m.token), g), keys).second, "output written twice");
        }
    }
    expect(static_cast<Index>(whole.size()) == T * G, "row without an output");
    for (const auto& [row, keys] : whole)
        for (char n : keys) expect(n == 1, "key left out or seen twice");
    std::printf("%lld %lld %lld %lld\n", static_cast<long long>(T), static_cast<long long>(p.lists[0].count + p.lists[1].count - fronts),
                static_cast<long long>(fronts), static_cast<long long>(p.merge_count));
    return 0;
}

int call(const std::string& name) {
    const dl::Device gpu = dl::Device::gpu(0);
    const dl::TensorOptions f32{.dtype = dl::DType::f32, .device = gpu};
    auto tensor = [&](dl::Shape shape, dl::DType dtype = dl::DType::f32) { return empty_tensor(shape, dtype, gpu); };
    auto host = [&](dl::Shape shape, dl::DType dtype = dl::DType::f32) { return empty_tensor(shape, dtype, dl::Device::cpu()); };
    const double inf = std::numeric_limits<double>::infinity();
    const Index one[] = {20}, two[] = {3}, none[] = {0}, pages[] = {1, 2, 0, 3};
    PagedKVCache cache(2, 8, 16, 2, 32, f32);
    const PagedBatch batch(cache, 4, one, two, pages, 4), idle(cache, 4, one, none, pages, 4);
    const auto c = tensor({64, 16}), s = tensor({64, 16}), q = tensor({3, 4, 32}), k = tensor({3, 2, 32}), v = tensor({3, 2, 32});
    using dl::RotaryLayout;
    using Kind = dl::RotaryScaling::Kind;
    auto append = [&](const auto& key, const auto& value, const auto& cosine, const auto& sine, Index layer = 0,
                      const PagedBatch* step = nullptr, std::optional<dl::Tensor> query = std::nullopt, RotaryLayout layout = RotaryLayout::half) {
        return dl::paged_append(cache, layer, step ? *step : batch, query ? query : std::optional<dl::Tensor>{q}, key, value, cosine, sine, layout);
    };
    // three rows out of a page
    auto page_rows = [&](const dl::Tensor& pages) { return pages.select(0, 5).transpose(0, 1).narrow(0, 0, 3); };
    const auto x = tensor({5, 2, 32});
    const auto at = tensor({5}, dl::DType::i64);
    const auto ids = tensor({2, 3}, dl::DType::i64);
    const auto target = tensor({2, 4, 10}), draft = tensor({2, 3, 10}), u = tensor({2, 4});
    fake.launches = 0;
    std::map<std::string, std::function<void()>> cases{
        {"cache layers", [&] { PagedKVCache(0, 8, 16, 2, 32, f32); }},
        {"cache pages", [&] { PagedKVCache(1, 0, 16, 2, 32, f32); }},
        {"cache page size 8", [&] { PagedKVCache(1, 8, 8, 2, 32, f32); }},
        {"cache page size 24", [&] { PagedKVCache(1, 8, 24, 2, 32, f32); }},
        {"cache page size 2048", [&] { PagedKVCache(1, 8, 2048, 2, 32, f32); }},
        {"cache head 48", [&] { PagedKVCache(1, 8, 16, 2, 48, f32); }},
        {"cache heads", [&] { PagedKVCache(1, 8, 16, 0, 32, f32); }},
        {"cache f64", [&] { PagedKVCache(1, 8, 16, 2, 32, {.dtype = dl::DType::f64, .device = gpu}); }},
        {"cache on the host", [&] { PagedKVCache(1, 8, 16, 2, 32, {}); }},
        {"cache elements", [&] { PagedKVCache(1, Index(1) << 30, 1024, Index(1) << 20, 128, f32); }},
        {"cache bytes", [&] { PagedKVCache(1, Index(1) << 30, 1024, Index(1) << 15, 128, f32); }},
        {"batch heads", [&] { PagedBatch(cache, Index(1) << 30, one, none, pages, 4); }},
        {"batch of too many items", [&] { // (17 million work-groups; the pages are never touched)
             const Index n = 1 << 14;
             const PagedKVCache wide(1, n, 16, 1024, 16, {.dtype = dl::DType::bf16, .device = gpu});
             std::vector<Index> lengths(n, 0), counts(n, 1), own(n);
             for (Index i = 0; i < n; ++i) own[i] = i;
             PagedBatch(wide, 1024, lengths, counts, own, 1);
         }},
        {"batch of too many merges", [&] { // (its rows are some million work-groups, joined by 17)
             const Index n = 1 << 22;
             const PagedKVCache narrow(1, n / 16 + 1, 16, 1, 128, {.dtype = dl::DType::bf16, .device = gpu});
             std::vector<Index> own(n / 16 + 1);
             for (std::size_t i = 0; i < own.size(); ++i) own[i] = static_cast<Index>(i);
             const Index length[] = {16}, count[] = {n};
             PagedBatch(narrow, 32, length, count, own, n / 16 + 1, 16);
         }},
        {"append layer", [&] { append(k, v, c, s, 2); }},
        {"append layer below", [&] { append(k, v, c, s, -1); }},
        {"append rows", [&] { append(tensor({4, 2, 32}), v, c, s); }},
        {"append heads", [&] { append(k, tensor({3, 4, 32}), c, s); }},
        {"append query heads", [&] { append(k, v, c, s, 0, nullptr, tensor({3, 8, 32})); }},
        {"append type", [&] { append(tensor({3, 2, 32}, dl::DType::f64), v, c, s); }},
        {"append host rows", [&] { append(host({3, 2, 32}), v, c, s); }},
        {"append short tables", [&] { append(k, v, tensor({22, 16}), tensor({22, 16})); }},
        {"append wide tables", [&] { append(k, v, tensor({64, 17}), tensor({64, 17})); }},
        {"append unequal tables", [&] { append(k, v, c, tensor({64, 8})); }},
        {"append empty tables", [&] { append(k, v, tensor({64, 0}), tensor({64, 0})); }},
        {"append undefined tables", [&] { append(k, v, dl::Tensor{}, s); }},
        {"append undefined sines", [&] { append(k, v, c, dl::Tensor{}); }},
        {"append undefined rows", [&] { append(dl::Tensor{}, v, c, s); }},
        {"append layout", [&] { append(k, v, c, s, 0, nullptr, std::nullopt, static_cast<RotaryLayout>(7)); }},
        {"append nothing", [&] { append(tensor({0, 2, 32}), tensor({0, 2, 32}), c, s, 0, &idle, tensor({0, 4, 32})); }},
        {"append rows of the pages", [&] { append(page_rows(cache.key(0)), page_rows(cache.value(0)), c, s); }},
        {"append rows of another layer", [&] { append(page_rows(cache.key(1)), page_rows(cache.value(1)), c, s); }},
        {"attend other cache", [&] { dl::paged_attention(PagedKVCache(2, 8, 32, 2, 32, f32), 0, batch, q); }},
        {"attend other type", [&] { dl::paged_attention(PagedKVCache(2, 8, 16, 2, 32, {.dtype = dl::DType::bf16, .device = gpu}), 0, batch, q); }},
        {"attend fewer pages", [&] { dl::paged_attention(PagedKVCache(2, 7, 16, 2, 32, f32), 0, batch, q); }},
        {"attend layer", [&] { dl::paged_attention(cache, 2, batch, q); }},
        {"attend rows", [&] { dl::paged_attention(cache, 0, batch, tensor({4, 4, 32})); }},
        {"attend flat", [&] { dl::paged_attention(cache, 0, batch, tensor({3, 128})); }},
        {"attend type", [&] { dl::paged_attention(cache, 0, batch, tensor({3, 4, 32}, dl::DType::i64)); }},
        {"attend host rows", [&] { dl::paged_attention(cache, 0, batch, host({3, 4, 32})); }},
        {"attend nothing", [&] { dl::paged_attention(cache, 0, idle, tensor({0, 4, 32})); }},
        {"rotary rank", [&] { dl::rotary_positions(tensor({5, 32}), at, c, s); }},
        {"rotary positions", [&] { dl::rotary_positions(x, tensor({4}, dl::DType::i64), c, s); }},
        {"rotary positions type", [&] { dl::rotary_positions(x, tensor({5}), c, s); }},
        {"rotary host positions", [&] { dl::rotary_positions(x, host({5}, dl::DType::i64), c, s); }},
        {"rotary host rows", [&] { dl::rotary_positions(host({5, 2, 32}), at, c, s); }},
        {"rotary type", [&] { dl::rotary_positions(tensor({5, 2, 32}, dl::DType::f64), at, c, s); }},
        {"rotary wide tables", [&] { dl::rotary_positions(tensor({5, 2, 30}), at, c, s); }},
        {"rotary layout", [&] { dl::rotary_positions(x, at, c, s, static_cast<RotaryLayout>(2)); }},
        {"rotary heads", [&] { dl::rotary_positions(tensor({1, Index(1) << 31, 2}, dl::DType::bf16), tensor({1}, dl::DType::i64), c, s); }},
        {"rotary nothing", [&] { dl::rotary_positions(tensor({0, 2, 32}), tensor({0}, dl::DType::i64), c, s); }},
        {"tables odd", [&] { dl::rotary_tables(7, 4); }},
        {"tables empty", [&] { dl::rotary_tables(8, 0); }},
        {"tables base", [&] { dl::rotary_tables(8, 4, 0.0); }},
        {"tables kind", [&] { dl::rotary_tables(8, 4, 10.0, {.kind = static_cast<Kind>(9)}); }},
        {"tables factor", [&] { dl::rotary_tables(8, 4, 10.0, {.kind = Kind::linear, .factor = 0.0}); }},
        {"tables trained", [&] { dl::rotary_tables(8, 4, 10.0, {.kind = Kind::parts, .factor = 2.0}); }},
        {"tables turns", [&] { dl::rotary_tables(8, 4, 10.0, {.kind = Kind::parts, .factor = 2.0, .trained = 8, .slow_turns = 4.0, .fast_turns = 4.0}); }},
        {"tables one pair", [&] { dl::rotary_tables(2, 4, 10.0, {.kind = Kind::base, .factor = 2.0}); }},
        {"tables magnitude", [&] { dl::rotary_tables(8, 4, 10.0, {.magnitude = inf}); }},
        {"verify ids", [&] { dl::verify_drafted(tensor({2, 3}), target, draft, 1.0, u); }},
        {"verify target", [&] { dl::verify_drafted(ids, draft, draft, 1.0, u); }},
        {"verify draft", [&] { dl::verify_drafted(ids, target, target, 1.0, u); }},
        {"verify uniforms", [&] { dl::verify_drafted(ids, target, draft, 1.0, tensor({2, 3})); }},
        {"verify uniforms type", [&] { dl::verify_drafted(ids, target, draft, 1.0, tensor({2, 4}, dl::DType::f64)); }},
        {"verify vocabulary", [&] { dl::verify_drafted(ids, tensor({2, 4, 0}), std::nullopt, 1.0, u); }},
        {"verify drafts", [&] {
             const Index n = (1 << 20) + 1;
             dl::verify_drafted(tensor({1, n}, dl::DType::i64), tensor({1, n + 1, 1}), std::nullopt, 1.0, tensor({1, n + 1}));
         }},
        {"verify rows", [&] {
             const Index n = 1 << 24;
             dl::verify_drafted(tensor({n, 0}, dl::DType::i64), tensor({n, 1, 1}), std::nullopt, 1.0, tensor({n, 1}));
         }},
        {"verify temperature", [&] { dl::verify_drafted(ids, target, draft, inf, u); }},
        {"verify temperature nan", [&] { dl::verify_drafted(ids, target, draft, inf - inf, u); }},
        {"verify logits type", [&] { dl::verify_drafted(ids, tensor({2, 4, 10}, dl::DType::f64), std::nullopt, 1.0, u); }},
        {"verify host ids", [&] { dl::verify_drafted(host({2, 3}, dl::DType::i64), target, draft, 1.0, u); }},
        {"verify host draft", [&] { dl::verify_drafted(ids, target, host({2, 3, 10}), 1.0, u); }},
        {"verify nothing", [&] { dl::verify_drafted(tensor({0, 3}, dl::DType::i64), tensor({0, 4, 10}), std::nullopt, 1.0, tensor({0, 4})); }},
    };
    cases.at(name)();
    std::printf("%zu\n", fake.launches);
    return 0;
}

} // namespace

int main(int argc, char** argv) {
    try {
        if (argc == 13 && std::strcmp(argv[1], "plan") == 0) return plan(argv + 2);
        if (argc == 3 && std::strcmp(argv[1], "call") == 0) return call(argv[2]);
    } catch (const std::exception& error) {
        std::fprintf(stderr, "%s\n", error.what());
        return 1;
    }
    std::fprintf(stderr, "see the head of paged_checks.cpp\n");
    return 2;
}
