// The gated delta rule token by token (see dlk_delta_params in kernels.h): for single and drafted tokens, whose time is that
// of the states' way from memory and back.
//   a = e^decay,  w = rate (v - a S^T k),  out = scale (a S^T q + (k . q) w),  S = a S + k w^T
// so that both products with the state are taken before it changes, in one pass over it and one exchange between lanes.
#include "kernels/device_common.h"

namespace dlk {
namespace {

constexpr int kThreads = 256;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// N (a multiple of 4) neighbouring entries of a row, in f32
template <int N>
__device__ __forceinline__ void load_entries(const void* x, int bf16, int64_t at, float (&out)[N]) {
    if (bf16) {
        const u32x2* from = reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(x) + at);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x2 w = from[i];
            out[4 * i] = bf16_lo(w.x), out[4 * i + 1] = bf16_hi(w.x);
            out[4 * i + 2] = bf16_lo(w.y), out[4 * i + 3] = bf16_hi(w.y);
        }
    } else {
        const f32x4* from = reinterpret_cast<const f32x4*>(static_cast<const float*>(x) + at);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const f32x4 w = from[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) out[4 * i + j] = w[j];
        }
    }
}

// The sum over the lanes that differ in bits 3, 4 and 5 alone.
__device__ __forceinline__ float sum_over_rows(float x) {
    x += __shfl_xor(x, 8);
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// A wave holds 32 columns of a head's state: 8 lanes side by side with 4 columns each, 8 groups of them with DK / 8 rows each.
// Columns know nothing of one another, so waves do not either.
template <int DK>
__global__ __launch_bounds__(kThreads) void delta_step(const dlk_delta_params p) {
    constexpr int R = DK / 8;
    const int lane = threadIdx.x % kWave;
    const uint32_t slices = p.value_dim / 32;
    const uint32_t unit = (blockIdx.x * kThreads + threadIdx.x) / kWave;
    if (unit >= static_cast<uint32_t>(p.item_count) * p.heads * slices) return;
    const int slice = unit % slices, head = unit / slices % p.heads;
    const dlk_delta_item item = p.items[unit / slices / p.heads];
    const int row = lane / 8 * R, column = slice * 32 + lane % 8 * 4;
    const int64_t within = static_cast<int64_t>(row) * p.value_dim + column, size = static_cast<int64_t>(DK) * p.value_dim;

    f32x4 s[R];
    if (item.source >= 0) {
        const float* from = p.states + (static_cast<int64_t>(item.source) * p.heads + head) * size + within;
#pragma unroll
        for (int i = 0; i < R; ++i) s[i] = *reinterpret_cast<const f32x4*>(from + i * p.value_dim);
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) s[i] = 0.0f;
    }
    for (int t = 0; t < item.count; ++t) {
        const int64_t token = item.token + t;
        float q[R], k[R], v[4];
        load_entries(p.q.x, p.q.bf16, token * p.q.row + head / p.group * p.q.head + row, q);
        load_entries(p.k.x, p.k.bf16, token * p.k.row + head / p.group * p.k.head + row, k);
        load_entries(p.v.x, p.v.bf16, token * p.v.row + head * p.v.head + column, v);
        const float a = expf(p.decay[token * p.heads + head]), rate = p.rate[token * p.heads + head];
        f32x4 sk = 0.0f, sq = 0.0f;
        float kq = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk[j] = fmaf(k[i], s[i][j], sk[j]);
                sq[j] = fmaf(q[i], s[i][j], sq[j]);
            }
            kq = fmaf(k[i], q[i], kq);
        }
        kq = sum_over_rows(kq);
        f32x4 w, out;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = rate * (v[j] - a * sum_over_rows(sk[j]));
            out[j] = p.scale * (a * sum_over_rows(sq[j]) + kq * w[j]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = fmaf(k[i], w[j], a * s[i][j]);
        if (lane < 8) *reinterpret_cast<f32x4*>(p.out + (token * p.heads + head) * p.value_dim + column) = out;
    }
    float* to = p.states + (static_cast<int64_t>(item.target) * p.heads + head) * size + within;
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<f32x4*>(to + i * p.value_dim) = s[i];
}

} // namespace
} // namespace dlk

extern "C" int dlk_delta_step(const dlk_delta_params* p, dlh_stream stream) {
    using namespace dlk;
    const int64_t waves = static_cast<int64_t>(p->item_count) * p->heads * (p->value_dim / 32);
    const int64_t groups = (waves + kThreads / kWave - 1) / (kThreads / kWave);
    if (p->value_dim <= 0 || p->value_dim % 32 != 0 || p->group <= 0 || groups > DLK_MOST_GROUPS) return hipErrorInvalidValue;
    if (groups == 0) return 0;
    hipStream_t at = reinterpret_cast<hipStream_t>(stream);
    switch (p->key_dim) {
    case 32: delta_step<32><<<groups, kThreads, 0, at>>>(*p); break;
    case 64: delta_step<64><<<groups, kThreads, 0, at>>>(*p); break;
    case 128: delta_step<128><<<groups, kThreads, 0, at>>>(*p); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
