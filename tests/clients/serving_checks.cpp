// Page pools, forks, compaction, the gated delta rule's batches and a layer of experts without a GPU, on the device of
// host_checks.cpp.  The copy of pages runs on the host (dlk_page_copy below takes the kernel's place, pair after pair in the
// order given to it backwards, so that a pair that depends on another of its launch is found out).  Run by
// tests/test_serving_rules.py.
//
//   serving_checks copy PAGES HEADS PAGE BYTES POOLS SOURCES TARGETS ROWS
//       copy_pages over pools whose bytes are known (lists separated by commas; ROWS "-": whole pages); every byte is
//       checked against the copy from the pools as they were
//   serving_checks fork PAGES PAGE WIDTH TABLES LENGTHS PARENTS      the tables of the new requests, then the holders of each page
//   serving_checks compact PAGES PAGE TABLES                         the tables, the pages moved
//   serving_checks hidden ENTRIES UNIT LAID      the room of a pair's hidden entries; each one's place, and what is zeroed with it
//   serving_checks call CASE    an operator called with arguments that it refuses (its error), or with nothing to do (launches)
#define main host_checks_main
#include "host_checks.cpp"
#undef main

#include "dl/delta.h"
#include "dl/paged.h"
#include "kernels/experts_layout.h"
#include "nn/ops_internal.h"

#include <functional>
#include <limits>

namespace {

using dl::DType;
using dl::Index;
using dl::Tensor;
using dl::nn::DeltaBatch;
using dl::nn::DeltaStates;
using dl::nn::PagedKVCache;
using dl::nn::PagePool;
using List = std::vector<Index>;

bool broken = false; // the next copy fails

List list(const char* text) {
    List out;
    if (std::strcmp(text, "-") == 0) return out;
    for (const char* at = text; *at;) {
        char* end = nullptr;
        out.push_back(std::strtoll(at, &end, 10));
        at = *end ? end + 1 : end;
    }
    return out;
}

void print(const List& ids) {
    for (const Index id : ids) std::printf("%lld ", static_cast<long long>(id));
    std::printf("\n");
}

int copy(char** arg) {
    const Index pages = std::atoll(arg[0]), heads = std::atoll(arg[1]), page = std::atoll(arg[2]), bytes = std::atoll(arg[3]);
    const int count = std::atoi(arg[4]);
    const List sources = list(arg[5]), targets = list(arg[6]), rows = list(arg[7]);
    const Index size = heads * page * bytes;
    std::vector<std::vector<unsigned char>> held(count, std::vector<unsigned char>(static_cast<std::size_t>(pages * size)));
    std::vector<void*> pools;
    for (int i = 0; i < count; ++i) {
        for (std::size_t at = 0; at < held[i].size(); ++at) held[i][at] = static_cast<unsigned char>((at * 2654435761u + i * 97u) >> 13);
        pools.push_back(held[i].data());
    }
    auto want = held;
    for (int i = 0; i < count; ++i)
        for (std::size_t n = 0; n < sources.size(); ++n)
            for (Index h = 0; h < heads; ++h)
                std::copy_n(held[i].data() + sources[n] * size + h * page * bytes, (rows.empty() ? page : rows[n]) * bytes,
                            want[i].data() + targets[n] * size + h * page * bytes);
    dl::detail::copy_pages(pools, pages, heads, page, bytes, dl::Device::gpu(0), sources, targets, rows, "copy");
    for (int i = 0; i < count; ++i)
        if (held[i] != want[i]) throw std::logic_error("pool " + std::to_string(i) + " differs");
    return 0;
}

PagedKVCache cache_of(Index pages, Index page) {
    return PagedKVCache(1, pages, page, 1, 16, {.dtype = DType::f32, .device = dl::Device::gpu(0)});
}

int fork(char** arg) {
    const Index pages = std::atoll(arg[0]), page = std::atoll(arg[1]), width = std::atoll(arg[2]);
    const List tables = list(arg[3]), lengths = list(arg[4]), parents = list(arg[5]);
    PagePool pool(pages);
    pool.claim(tables);
    print(dl::paged_fork(cache_of(pages, page), pool, tables, width, lengths, parents));
    List holders;
    for (Index i = 0; i < pages; ++i) holders.push_back(pool.references(i));
    print(holders);
    return 0;
}

int compact(char** arg) {
    const Index pages = std::atoll(arg[0]), page = std::atoll(arg[1]);
    List tables = list(arg[2]);
    PagePool pool(pages);
    pool.claim(tables);
    const Index moved = dl::paged_compact(cache_of(pages, page), pool, tables);
    print(tables);
    print({moved});
    return 0;
}

int hidden(char** arg) {
    const int entries = std::atoi(arg[0]), unit = std::atoi(arg[1]);
    const bool laid = std::atoi(arg[2]) != 0;
    List places, zeros;
    for (int i = 0; i < entries; ++i) {
        places.push_back(dlk::hidden_place(i, entries, unit, laid));
        zeros.push_back(dlk::hidden_zero(i, entries, unit, laid));
    }
    print({dlk::hidden_line(entries, unit, laid)});
    print(places);
    print(zeros);
    return 0;
}

int call(const std::string& name) {
    const dl::Device gpu = dl::Device::gpu(0);
    const auto tensor = [&](dl::Shape shape, DType dtype = DType::f32) { return dl::detail::empty_tensor(shape, dtype, gpu); };
    const auto host = [&](dl::Shape shape) { return dl::detail::empty_tensor(shape, DType::f32, dl::Device::cpu()); };
    const PagedKVCache cache = cache_of(8, 16);
    PagePool pool(8);
    pool.claim(List{0, 1, 2});
    const List tables{0, 1, 2}, lengths{40};
    const auto fork = [&](const List& t, Index w, const List& l, const List& p) { dl::paged_fork(cache, pool, t, w, l, p); };

    const DeltaStates states(2, 6, 4, 32, 64, gpu);
    const auto batch = [&](const List& s, const List& t, const List& c, Index key_heads = 2) { return DeltaBatch(states, key_heads, s, t, c); };
    const DeltaBatch step = batch({-1, 2}, {0, 2}, {1, 2}), idle = batch({9}, {-5}, {0});
    const Tensor q = tensor({3, 2, 32}), v = tensor({3, 4, 64}), g = tensor({3, 4});
    const auto delta = [&](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& b, Index layer = 0,
                           std::optional<double> scale = std::nullopt) { dl::gated_delta(states, layer, step, q, k, v, g, b, scale); };
    const auto rows_of = [&](const Tensor& t) { return t.select(0, 5).narrow(0, 0, 3).narrow(1, 0, 2).narrow(2, 0, 32); };

    const Tensor x = tensor({3, 16}), router = tensor({4, 16}), up = tensor({4, 8, 16}), down = tensor({4, 16, 8});
    const auto mix = [&](const Tensor& x, const Tensor& r, const Tensor& g, const Tensor& u, const Tensor& d, Index top = 2) {
        dl::expert_mixture(x, r, g, u, d, top);
    };
    fake.launches = 0;
    const std::map<std::string, std::function<void()>> cases = {
        {"pool empty", [&] { PagePool(0); }},
        {"pool large", [&] { PagePool(Index(1) << 31); }},
        {"copy unequal", [&] { dl::paged_copy(cache, List{1, 2}, List{3}); }},
        {"copy rows unequal", [&] { dl::paged_copy(cache, List{1}, List{3}, List{1, 2}); }},
        {"copy source", [&] { dl::paged_copy(cache, List{8}, List{3}); }},
        {"copy target", [&] { dl::paged_copy(cache, List{1}, List{-1}); }},
        {"copy twice", [&] { dl::paged_copy(cache, List{1, 2}, List{3, 3}); }},
        {"copy rows", [&] { dl::paged_copy(cache, List{1}, List{3}, List{17}); }},
        {"copy rows below", [&] { dl::paged_copy(cache, List{1}, List{3}, List{-1}); }},
        {"copy nothing", [&] { dl::paged_copy(cache, {}, {}); }},
        {"copy itself", [&] { dl::paged_copy(cache, List{1, 2}, List{1, 3}, List{16, 0}); }},
        {"copy large", [&] { dl::detail::copy_pages({nullptr}, 4, 1 << 20, 1024, 512, gpu, List{0}, List{1}, {}, "copy"); }},
        {"fork other pool", [&] {
             PagePool other(9);
             dl::paged_fork(cache, other, tables, 3, lengths, List{0});
         }},
        {"fork tables", [&] { fork(tables, 2, lengths, {0}); }},
        {"fork parent", [&] { fork(tables, 3, lengths, {1}); }},
        {"fork parent below", [&] { fork(tables, 3, lengths, {-1}); }},
        {"fork length", [&] { fork(tables, 3, {49}, {0}); }},
        {"fork length below", [&] { fork(tables, 3, {-1}, {0}); }},
        {"fork missing page", [&] { fork({0, 1, -1}, 3, lengths, {0}); }},
        {"fork page beyond", [&] { fork({0, 1, 8}, 3, lengths, {0}); }},
        {"fork free page", [&] { fork({0, 1, 3}, 3, lengths, {0}); }},
        {"fork too many", [&] {
             try {
                 fork(tables, 3, lengths, {0, 0, 0, 0, 0, 0});
             } catch (const std::runtime_error& error) {
                 if (pool.available() != 5 || pool.references(0) != 1) throw std::logic_error("the pool changed");
                 throw;
             }
         }},
        {"fork failing", [&] { // what was taken is given back
             broken = true;
             try {
                 fork(tables, 3, lengths, {0});
             } catch (const std::runtime_error& error) {
                 if (pool.available() != 5 || pool.references(0) != 1 || pool.references(3) != 0) throw std::logic_error("the pool changed");
                 throw;
             }
         }},
        {"compact other pool", [&] {
             PagePool other(9);
             List t = tables;
             dl::paged_compact(cache, other, t);
         }},
        {"compact beyond", [&] { List t{0, 1, 8}; dl::paged_compact(cache, pool, t); }},
        {"compact missing", [&] { List t{0, 1}; dl::paged_compact(cache, pool, t); }},
        {"compact twice", [&] { List t{0, 1, 2, 2}; dl::paged_compact(cache, pool, t); }},
        {"compact nothing", [&] { List t{0, 1, 2}; dl::paged_compact(cache, pool, t); }},
        {"states layers", [&] { DeltaStates(0, 1, 1, 32, 32, gpu); }},
        {"states key_dim", [&] { DeltaStates(1, 1, 1, 48, 32, gpu); }},
        {"states value_dim", [&] { DeltaStates(1, 1, 1, 32, 48, gpu); }},
        {"states wide", [&] { DeltaStates(1, 1, 1, 32, 288, gpu); }},
        {"states slots", [&] { DeltaStates(1, Index(1) << 31, 1, 32, 32, gpu); }},
        {"states host", [&] { DeltaStates(1, 1, 1, 32, 32, dl::Device::cpu()); }},
        {"batch key_heads", [&] { batch({0}, {0}, {1}, 3); }},
        {"batch no key_heads", [&] { batch({0}, {0}, {1}, 0); }},
        {"batch empty", [&] { batch({}, {}, {}); }},
        {"batch unequal", [&] { batch({0}, {0, 1}, {1}); }},
        {"batch count", [&] { batch({0}, {0}, {-1}); }},
        {"batch target", [&] { batch({0}, {6}, {1}); }},
        {"batch no target", [&] { batch({0}, {-1}, {1}); }},
        {"batch source", [&] { batch({6}, {0}, {1}); }},
        {"batch source below", [&] { batch({-2}, {0}, {1}); }},
        {"batch written twice", [&] { batch({0, 1}, {3, 3}, {1, 1}); }},
        {"batch read and written", [&] { batch({0, 1}, {1, 2}, {1, 1}); }},
        {"batch read and written before", [&] { batch({1, 0}, {2, 1}, {1, 1}); }},
        {"batch many", [&] { batch({0, 1}, {2, 3}, {1 << 30, 1}); }},
        {"batch many requests", [&] {
             const List none(20, -1), counts(20, 1);
             List targets(20);
             for (Index i = 0; i < 20; ++i) targets[static_cast<std::size_t>(i)] = i;
             DeltaBatch(DeltaStates(1, 20, 16384, 32, 256, gpu), 1, none, targets, counts);
         }},
        {"states heads", [&] { DeltaStates(1, 1, 16385, 32, 32, gpu); }},
        {"experts large", [&] { mix(tensor({1, 1}), tensor({1024, 1}), tensor({1024, 32769, 1}), tensor({1024, 32769, 1}), tensor({1024, 1, 32769}), 1); }},
        {"batch many heads", [&] { batch({0}, {2}, {1 << 29}); }},
        {"delta other states", [&] { dl::gated_delta(DeltaStates(2, 6, 4, 32, 32, gpu), 0, step, q, q, v, g, g); }},
        {"delta fewer slots", [&] { dl::gated_delta(DeltaStates(2, 5, 4, 32, 64, gpu), 0, step, q, q, v, g, g); }},
        {"delta layer", [&] { delta(q, q, v, g, g, 2); }},
        {"delta layer below", [&] { delta(q, q, v, g, g, -1); }},
        {"delta query", [&] { delta(tensor({2, 2, 32}), q, v, g, g); }},
        {"delta key heads", [&] { delta(q, tensor({3, 4, 32}), v, g, g); }},
        {"delta value", [&] { delta(q, q, tensor({3, 4, 32}), g, g); }},
        {"delta type", [&] { delta(q, q, tensor({3, 4, 64}, DType::f64), g, g); }},
        {"delta host", [&] { delta(q, host({3, 2, 32}), v, g, g); }},
        {"delta decay", [&] { delta(q, q, v, tensor({3, 2}), g); }},
        {"delta rate type", [&] { delta(q, q, v, g, tensor({3, 4}, DType::i64)); }},
        {"delta host decay", [&] { delta(q, q, v, host({3, 4}), g); }},
        {"delta scale beyond f32", [&] { delta(q, q, v, g, g, 0, -1e39); }},
        {"delta scale", [&] { delta(q, q, v, g, g, 0, std::numeric_limits<double>::infinity()); }},
        {"delta undefined", [&] { delta(Tensor{}, q, v, g, g); }},
        {"delta undefined rate", [&] { delta(q, q, v, g, Tensor{}); }},
        {"delta nothing", [&] {
             dl::gated_delta(states, 0, idle, tensor({0, 2, 32}), tensor({0, 2, 32}), tensor({0, 4, 64}), tensor({0, 4}), tensor({0, 4}));
         }},
        {"delta rows of the states", [&] { delta(rows_of(states.state(0)), q, v, g, g); }},
        {"delta rows of another layer", [&] { delta(rows_of(states.state(1)), q, v, g, g); }},
        {"states copy twice", [&] { dl::delta_copy(states, List{0, 1}, List{2, 2}); }},
        {"states copy beyond", [&] { dl::delta_copy(states, List{6}, List{2}); }},
        {"experts router", [&] { mix(x, tensor({4, 8}), up, up, down); }},
        {"experts router rank", [&] { mix(x, tensor({4, 16, 1}), up, up, down); }},
        {"experts gate", [&] { mix(x, router, tensor({3, 8, 16}), up, down); }},
        {"experts up", [&] { mix(x, router, up, tensor({4, 9, 16}), down); }},
        {"experts down", [&] { mix(x, router, up, up, tensor({4, 8, 16})); }},
        {"experts top", [&] { mix(x, router, up, up, down, 5); }},
        {"experts no top", [&] { mix(x, router, up, up, down, 0); }},
        {"experts top beyond", [&] { mix(x, tensor({80, 16}), tensor({80, 8, 16}), tensor({80, 8, 16}), tensor({80, 16, 8}), 65); }},
        {"experts many", [&] { mix(x, tensor({1025, 16}), tensor({1025, 1, 16}), tensor({1025, 1, 16}), tensor({1025, 16, 1}), 1); }},
        {"experts types", [&] { mix(x, router, up, up, tensor({4, 16, 8}, DType::bf16)); }},
        {"experts weight type", [&] { mix(x, tensor({4, 16}, DType::f64), up, up, down); }},
        {"experts input type", [&] { mix(tensor({3, 16}, DType::i64), router, up, up, down); }},
        {"experts host", [&] { mix(host({3, 16}), router, up, up, down); }},
        {"experts host weights", [&] { mix(x, router, host({4, 8, 16}), up, down); }},
        {"experts strides", [&] { mix(x, router, tensor({4, 8, 32}).narrow(2, 0, 16), up, down); }},
        {"experts no width", [&] { mix(tensor({3, 0}), tensor({4, 0}), tensor({4, 8, 0}), tensor({4, 8, 0}), tensor({4, 0, 8})); }},
        {"experts undefined", [&] { mix(x, router, Tensor{}, up, down); }},
        {"experts nothing", [&] { mix(tensor({0, 16}), router, up, up, down); }},
        {"experts module", [&] { dl::nn::ExpertMixture(16, 8, 4, 5); }},
    };
    cases.at(name)();
    std::printf("%zu\n", fake.launches);
    return 0;
}

} // namespace

extern "C" int dlk_page_copy(const dlk_page_copy_params* p, dlh_stream) {
    if (std::exchange(broken, false)) return hipErrorOutOfMemory;
    fake.launches += 1;
    const Index row = Index(16) * p->row_units, size = row * p->page * p->heads;
    if (p->count < 1 || p->count > DLK_PAGE_PAIRS || p->pool_count < 1 || p->pool_count > DLK_PAGE_POOLS) return hipErrorInvalidValue;
    for (int z = 0; z < p->pool_count; ++z)
        for (int i = p->count - 1; i >= 0; --i) {
            const dlk_page_pair pair = p->pairs[i];
            char* pool = static_cast<char*>(p->pools[z]);
            char* staged = static_cast<char*>(p->staging) + size * p->staged * z;
            const char* from = pair.from >= 0 ? pool + size * pair.from : staged + size * ~pair.from;
            char* to = pair.to >= 0 ? pool + size * pair.to : staged + size * ~pair.to;
            if ((pair.from < 0 && ~pair.from >= p->staged) || (pair.to < 0 && ~pair.to >= p->staged)) return hipErrorInvalidValue;
            for (int h = 0; h < p->heads; ++h) std::memcpy(to + row * p->page * h, from + row * p->page * h, row * pair.rows);
        }
    return 0;
}

int main(int argc, char** argv) {
    try {
        if (argc == 10 && std::strcmp(argv[1], "copy") == 0) return copy(argv + 2);
        if (argc == 8 && std::strcmp(argv[1], "fork") == 0) return fork(argv + 2);
        if (argc == 5 && std::strcmp(argv[1], "compact") == 0) return compact(argv + 2);
        if (argc == 5 && std::strcmp(argv[1], "hidden") == 0) return hidden(argv + 2);
        if (argc == 3 && std::strcmp(argv[1], "call") == 0) return call(argv[2]);
    } catch (const std::exception& error) {
        std::fprintf(stderr, "%s\n", error.what());
        return 1;
    }
    std::fprintf(stderr, "see the head of serving_checks.cpp\n");
    return 2;
}
