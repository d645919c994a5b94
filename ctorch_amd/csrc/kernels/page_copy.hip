// Copies of pages within pools that share one layout (see dlk_page_copy_params in kernels.h): the keys and values of every
// layer of a paged cache, or the states of every layer.  Bound by memory: each byte is read and written once, 16 of them a
// thread's step: 229 MB moved in 16 layers' pages of 64 KB 87 us, 5.3 TB/s read and written; 157 MB to four copies of each page
// 49 us; three copies of 8 rows of a 16 KB page in 16 layers 3.2 us, of a call's 13.  What a launch needs to know comes with its arguments, so that a call copies nothing to the device first
// and waits for nothing.
#include "kernels/device_common.h"

#include <algorithm>

namespace dlk {
namespace {

constexpr int kThreads = 256, kSteps = 4; // 16 KB a work-group
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
static_assert(sizeof(dlk_page_copy_params) <= 4096, "the arguments of a launch");

// A work-group per piece of (pair, pool).  Of a head's `page` rows the pair's first `rows` are copied: unit i of the pair
// lies in head i / (rows * units), at unit i % (rows * units) of the head's.
__global__ __launch_bounds__(kThreads) void page_copy(const dlk_page_copy_params p) {
    const dlk_page_pair pair = p.pairs[blockIdx.y];
    const uint32_t span = static_cast<uint32_t>(pair.rows) * p.row_units, head_units = static_cast<uint32_t>(p.page) * p.row_units;
    const uint32_t count = span * p.heads;
    const int64_t page_units = static_cast<int64_t>(head_units) * p.heads;
    u32x4* pool = static_cast<u32x4*>(p.pools[blockIdx.z]);
    u32x4* staged = static_cast<u32x4*>(p.staging) + page_units * p.staged * blockIdx.z;
    const u32x4* from = pair.from >= 0 ? pool + page_units * pair.from : staged + page_units * ~pair.from;
    u32x4* to = pair.to >= 0 ? pool + page_units * pair.to : staged + page_units * ~pair.to;
    const uint32_t first = blockIdx.x * (kThreads * kSteps) + threadIdx.x;
    u32x4 held[kSteps];
    uint32_t at[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const uint32_t i = first + s * kThreads;
        at[s] = i / span * head_units + i % span;
        if (i < count) held[s] = from[at[s]];
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
        if (first + s * kThreads < count) to[at[s]] = held[s];
}

} // namespace
} // namespace dlk

extern "C" int dlk_page_copy(const dlk_page_copy_params* p, dlh_stream stream) {
    using namespace dlk;
    if (p->count <= 0 || p->pool_count <= 0) return 0;
    if (p->count > DLK_PAGE_PAIRS || p->pool_count > DLK_PAGE_POOLS || p->row_units <= 0 || p->page <= 0 || p->heads <= 0 ||
        static_cast<int64_t>(p->page) * p->row_units * p->heads > INT32_MAX / 2)
        return hipErrorInvalidValue;
    int most = 0;
    for (int i = 0; i < p->count; ++i) {
        const dlk_page_pair& pair = p->pairs[i];
        if (pair.rows <= 0 || pair.rows > p->page || ((pair.from < 0 || pair.to < 0) && !p->staging)) return hipErrorInvalidValue;
        if (~pair.from >= p->staged || ~pair.to >= p->staged) return hipErrorInvalidValue;
        most = std::max(most, pair.rows);
    }
    const int units = most * p->row_units * p->heads;
    const dim3 grid((units + kThreads * kSteps - 1) / (kThreads * kSteps), p->count, p->pool_count);
    page_copy<<<grid, kThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(*p);
    return hipGetLastError();
}
