// Rows at given positions: out of a step's queries, keys and values (f32 or bf16, any strides between rows and heads)
// the rotated queries, and the rotated keys and the values in their places of a paged cache (see dlk_rotary_params in
// kernels.h).  Pair (a, b) of a row at position t becomes (a c - b s, a s + b c) with c, s = cosine, sine[t]; the pairs
// are neighbours (2 i, 2 i + 1) or lie half the rotated part apart, and entries behind that part are copied.  All of it in
// f32; a bf16 page rounds once, to nearest even.
#include "kernels/device_common.h"

#include <algorithm>

namespace dlk {
namespace {

constexpr int kThreads = 256;
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float load_one(const void* x, int bf16, int64_t at) {
    return bf16 ? bf16_to_f32(static_cast<const uint16_t*>(x)[at]) : static_cast<const float*>(x)[at];
}

// Any head size, part, stride and alignment: a thread per pair (or copied entry) of a head.
__global__ __launch_bounds__(kThreads) void rotary_entries(const dlk_rotary_params p) {
    const int pairs = p.part / 2, units = p.dim - pairs;
    const int heads = p.q.heads + p.k.heads + p.v.heads;
    const int64_t total = p.tokens * heads * units, step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += step) {
        const int unit = static_cast<int>(i % units);
        int head = static_cast<int>(i / units % heads);
        const int64_t token = i / units / heads;
        const bool query = head < p.q.heads, key = !query && head < p.q.heads + p.k.heads;
        head -= query ? 0 : key ? p.q.heads : p.q.heads + p.k.heads;
        const dlk_row_segment s = query ? p.q : key ? p.k : p.v;
        const int64_t from = token * s.row + head * s.head;
        // the entries that this thread writes: a pair, or one copied entry (values: two copied ones of the part)
        int first = p.half ? unit : 2 * unit, second = p.half ? unit + pairs : 2 * unit + 1;
        const bool pair = unit < pairs;
        if (!pair) first = second = pairs + unit;
        float a = load_one(s.x, s.bf16, from + first), b = pair ? load_one(s.x, s.bf16, from + second) : a;
        if (pair && (query || key)) {
            const int64_t position = p.positions[token];
            const bool inside = position >= 0 && position < p.capacity;
            const int64_t at = inside ? position * pairs + unit : 0;
            const float c = inside ? p.cosine[at] : NAN, sn = inside ? p.sine[at] : NAN;
            const float x = a, y = b;
            a = x * c - y * sn;
            b = x * sn + y * c;
        }
        if (query) {
            float* to = p.out + (token * p.q.heads + head) * p.dim;
            to[first] = a;
            if (pair) to[second] = b;
            continue;
        }
        const int64_t place = p.places[token], size = int64_t(1) << p.page_shift;
        const int64_t to = (((place >> p.page_shift) * p.k.heads + head) * size + (place & (size - 1))) * p.dim;
        void* pages = key ? p.k_pages : p.v_pages;
        if (p.pages_bf16) {
            static_cast<uint16_t*>(pages)[to + first] = f32_to_bf16(a);
            if (pair) static_cast<uint16_t*>(pages)[to + second] = f32_to_bf16(b);
        } else {
            static_cast<float*>(pages)[to + first] = a;
            if (pair) static_cast<float*>(pages)[to + second] = b;
        }
    }
}

} // namespace
} // namespace dlk

extern "C" int dlk_rotary(const dlk_rotary_params* params, dlh_stream stream_handle) {
    const dlk_rotary_params& p = *params;
    const int heads = p.q.heads + p.k.heads + p.v.heads;
    if (p.tokens < 0 || p.dim <= 0 || p.part < 0 || p.part % 2 != 0 || p.part > p.dim || heads <= 0 || p.k.heads != p.v.heads ||
        (p.q.heads && !p.out) || (p.k.heads && !(p.k_pages && p.v_pages && p.places)))
        return static_cast<int>(hipErrorInvalidValue);
    if (p.tokens == 0) return 0;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_handle);
    const int64_t total = p.tokens * heads * (p.dim - p.part / 2);
    const int blocks = static_cast<int>(std::min<int64_t>((total + dlk::kThreads - 1) / dlk::kThreads, 1 << 16));
    hipLaunchKernelGGL(dlk::rotary_entries, dim3(blocks), dim3(dlk::kThreads), 0, stream, p);
    return static_cast<int>(hipGetLastError());
}
