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
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float load_one(const void* x, int bf16, int64_t at) {
    return bf16 ? bf16_to_f32(static_cast<const uint16_t*>(x)[at]) : static_cast<const float*>(x)[at];
}

// Whole 16-byte pieces: a thread takes 8 entries of a head, four pairs or eight copied ones (dim and part multiples of 8,
// rows 16-byte aligned).  HALF: the pairs' second entries lie part / 2 behind the first.  Bound by memory: 4093 bf16 rows of 32
// x 128 to f32 19.7 us (5.2 TB/s; a thread per pair 62 us), four f32 prompts into their pages, 182 MB, 35 us (83 us).
template <bool HALF>
__global__ __launch_bounds__(kThreads) void rotary_pieces(const dlk_rotary_params p) {
    const uint32_t units = static_cast<uint32_t>(p.dim) / 8, heads = p.q.heads + p.k.heads + p.v.heads;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x, rows = i / units;
    if (rows >= static_cast<uint32_t>(p.tokens) * heads) return;
    const int unit = static_cast<int>(i % units), pairs = p.part / 2;
    const int64_t token = rows / heads;
    int head = static_cast<int>(rows % heads);
    const bool query = head < p.q.heads, key = !query && head < p.q.heads + p.k.heads;
    head -= query ? 0 : key ? p.q.heads : p.q.heads + p.k.heads;
    const dlk_row_segment s = query ? p.q : key ? p.k : p.v;
    // entries first .. +4 and second .. +4: in the rotated part of HALF the four pairs' first and second ones
    const bool pair = 4 * unit < pairs;
    const int first = HALF && pair ? 4 * unit : 8 * unit, second = HALF && pair ? first + pairs : first + 4;
    const int64_t from = token * s.row + head * s.head;
    f32x4 a, b;
    if (s.bf16) {
        const uint16_t* row = static_cast<const uint16_t*>(s.x) + from;
        const u32x2 x = *reinterpret_cast<const u32x2*>(row + first), y = *reinterpret_cast<const u32x2*>(row + second);
        a = f32x4{bf16_lo(x.x), bf16_hi(x.x), bf16_lo(x.y), bf16_hi(x.y)};
        b = f32x4{bf16_lo(y.x), bf16_hi(y.x), bf16_lo(y.y), bf16_hi(y.y)};
    } else {
        const float* row = static_cast<const float*>(s.x) + from;
        a = *reinterpret_cast<const f32x4*>(row + first);
        b = *reinterpret_cast<const f32x4*>(row + second);
    }
    if (pair && (query || key)) {
        const int64_t position = p.positions[token];
        const bool inside = position >= 0 && position < p.capacity;
        const int64_t at = inside ? position * pairs + 4 * unit : 0;
        f32x4 c = *reinterpret_cast<const f32x4*>(p.cosine + at), sn = *reinterpret_cast<const f32x4*>(p.sine + at);
        if (!inside) c = sn = f32x4{NAN, NAN, NAN, NAN};
        if constexpr (HALF) {
            const f32x4 x = a, y = b;
            a = x * c - y * sn;
            b = x * sn + y * c;
        } else {
            const f32x4 x = a, y = b;
            a = f32x4{x[0] * c[0] - x[1] * sn[0], x[0] * sn[0] + x[1] * c[0], x[2] * c[1] - x[3] * sn[1], x[2] * sn[1] + x[3] * c[1]};
            b = f32x4{y[0] * c[2] - y[1] * sn[2], y[0] * sn[2] + y[1] * c[2], y[2] * c[3] - y[3] * sn[3], y[2] * sn[3] + y[3] * c[3]};
        }
    }
    if (query) {
        float* to = p.out + (token * p.q.heads + head) * p.dim;
        *reinterpret_cast<f32x4*>(to + first) = a;
        *reinterpret_cast<f32x4*>(to + second) = b;
        return;
    }
    const int64_t place = p.places[token], size = int64_t(1) << p.page_shift;
    const int64_t to = (((place >> p.page_shift) * p.k.heads + head) * size + (place & (size - 1))) * p.dim;
    void* pages = key ? p.k_pages : p.v_pages;
    if (p.pages_bf16) {
        uint16_t* row = static_cast<uint16_t*>(pages) + to;
        *reinterpret_cast<bf16x4*>(row + first) = __builtin_convertvector(a, bf16x4);
        *reinterpret_cast<bf16x4*>(row + second) = __builtin_convertvector(b, bf16x4);
    } else {
        float* row = static_cast<float*>(pages) + to;
        *reinterpret_cast<f32x4*>(row + first) = a;
        *reinterpret_cast<f32x4*>(row + second) = b;
    }
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
    const auto whole = [](const dlk_row_segment& s) {
        const int align = s.bf16 ? 8 : 4; // entries of 16 bytes
        return s.heads == 0 || (s.row % align == 0 && s.head % align == 0 && reinterpret_cast<uintptr_t>(s.x) % 16 == 0);
    };
    const int64_t pieces = p.tokens * heads * (p.dim / 8);
    if (p.dim % 8 == 0 && p.part % 8 == 0 && pieces < INT32_MAX && whole(p.q) && whole(p.k) && whole(p.v) &&
        reinterpret_cast<uintptr_t>(p.cosine) % 16 == 0 && reinterpret_cast<uintptr_t>(p.sine) % 16 == 0) {
        const dim3 grid(static_cast<unsigned>((pieces + dlk::kThreads - 1) / dlk::kThreads));
        if (p.half) hipLaunchKernelGGL(dlk::rotary_pieces<true>, grid, dim3(dlk::kThreads), 0, stream, p);
        else hipLaunchKernelGGL(dlk::rotary_pieces<false>, grid, dim3(dlk::kThreads), 0, stream, p);
        return static_cast<int>(hipGetLastError());
    }
    const int64_t total = p.tokens * heads * (p.dim - p.part / 2);
    const int blocks = static_cast<int>(std::min<int64_t>((total + dlk::kThreads - 1) / dlk::kThreads, 1 << 16));
    hipLaunchKernelGGL(dlk::rotary_entries, dim3(blocks), dim3(dlk::kThreads), 0, stream, p);
    return static_cast<int>(hipGetLastError());
}
