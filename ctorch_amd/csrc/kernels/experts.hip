// A layer of experts over few rows (see dlk_experts_params in kernels.h).
#include "kernels/device_common.h"

namespace dlk {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float entry(const void* x, int bf16, int64_t at) {
    return bf16 ? bf16_to_f32(static_cast<const uint16_t*>(x)[at]) : static_cast<const float*>(x)[at];
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// A work-group per row: the logits in f64, which hold products of two f32 exactly, so that rows choose as the exact logits do
// but for ties within 1e-15 of them; then one wave picks the best one after another.
__global__ __launch_bounds__(kThreads) void experts_route(const dlk_experts_params p) {
    __shared__ double logits[DLK_EXPERTS_MOST];
    const int64_t token = blockIdx.x;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    for (int e = wave; e < p.experts; e += kThreads / kWave) {
        double sum = 0.0;
        for (int i = lane; i < p.dim; i += kWave)
            sum = fma(static_cast<double>(entry(p.x, p.x_bf16, token * p.dim + i)),
                      static_cast<double>(entry(p.router, p.router_bf16, static_cast<int64_t>(e) * p.dim + i)), sum);
        sum = wave_sum_f64(sum);
        if (lane == 0) logits[e] = sum;
    }
    __syncthreads();
    if (wave != 0) return;
    uint32_t taken = 0; // of this lane's experts lane, lane + 64, ...
    double largest = 0.0, all = 0.0, mine = 0.0, picked = 0.0;
    int64_t own = 0;
    for (int j = 0; j < p.top; ++j) {
        double best = 0.0;
        int64_t at = p.experts; // none
        for (int e = lane, n = 0; e < p.experts; e += kWave, ++n)
            if (!(taken >> n & 1) && (at == p.experts || prefer(logits[e], e, best, at))) best = logits[e], at = e;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const double other = __shfl_xor(best, d);
            const int64_t index = __shfl_xor(static_cast<long long>(at), d);
            if (index < p.experts && (at == p.experts || prefer(other, index, best, at))) best = other, at = index;
        }
        if (static_cast<int>(at) % kWave == lane) taken |= 1u << at / kWave;
        if (j == 0) {
            largest = best;
            double sum = 0.0;
            for (int e = lane; e < p.experts; e += kWave) sum += exp(logits[e] - largest);
            all = wave_sum_f64(sum);
        }
        const double weight = exp(best - largest);
        picked += weight;
        if (j == lane) mine = weight, own = at;
    }
    if (lane < p.top) {
        p.chosen[token * p.top + lane] = own;
        p.weights[token * p.top + lane] = static_cast<float>(mine / (p.normalise ? picked : all));
    }
}

// Any sizes and alignments: a wave per pair (row, chosen expert) and hidden entry.
__global__ __launch_bounds__(kThreads) void experts_hidden_any(const dlk_experts_params p) {
    const int lane = threadIdx.x % kWave;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kWave, step = static_cast<int64_t>(gridDim.x) * kThreads / kWave;
    for (int64_t u = unit; u < p.tokens * p.top * p.hidden; u += step) {
        const int64_t pair = u / p.hidden, row = p.chosen[pair] * p.hidden + u % p.hidden;
        float g = 0.0f, h = 0.0f;
        for (int i = lane; i < p.dim; i += kWave) {
            const float x = entry(p.x, p.x_bf16, pair / p.top * p.dim + i);
            g = fmaf(x, entry(p.gate, p.weights_bf16, row * p.dim + i), g);
            h = fmaf(x, entry(p.up, p.weights_bf16, row * p.dim + i), h);
        }
        g = wave_sum(g), h = wave_sum(h);
        if (lane == 0) p.act[u] = g / (1.0f + expf(-g)) * h;
    }
}

// and a wave per row and output entry, the chosen experts in order
__global__ __launch_bounds__(kThreads) void experts_down_any(const dlk_experts_params p) {
    const int lane = threadIdx.x % kWave;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kWave, step = static_cast<int64_t>(gridDim.x) * kThreads / kWave;
    for (int64_t u = unit; u < p.tokens * p.dim; u += step) {
        float y = 0.0f;
        for (int j = 0; j < p.top; ++j) {
            const int64_t pair = u / p.dim * p.top + j, row = p.chosen[pair] * p.dim + u % p.dim;
            float sum = 0.0f;
            for (int i = lane; i < p.hidden; i += kWave)
                sum = fmaf(p.act[pair * p.hidden + i], entry(p.down, p.weights_bf16, row * p.hidden + i), sum);
            y = fmaf(p.weights[pair], wave_sum(sum), y);
        }
        if (lane == 0) p.y[u] = y;
    }
}

} // namespace
} // namespace dlk

extern "C" int dlk_experts(const dlk_experts_params* p, dlh_stream stream) {
    using namespace dlk;
    if (p->experts <= 0 || p->experts > DLK_EXPERTS_MOST || p->top <= 0 || p->top > p->experts || p->top > DLK_EXPERTS_TOP_MOST ||
        p->dim <= 0 || p->hidden <= 0 || p->tokens <= 0 || p->tokens > DLK_MOST_GROUPS)
        return hipErrorInvalidValue;
    hipStream_t at = reinterpret_cast<hipStream_t>(stream);
    const auto groups = [](int64_t waves) { return static_cast<unsigned>(waves / 4 + 1 < 16384 ? waves / 4 + 1 : 16384); };
    experts_route<<<static_cast<unsigned>(p->tokens), kThreads, 0, at>>>(*p);
    experts_hidden_any<<<groups(p->tokens * p->top * p->hidden), kThreads, 0, at>>>(*p);
    experts_down_any<<<groups(p->tokens * p->dim), kThreads, 0, at>>>(*p);
    return hipGetLastError();
}
