// Verification of drafted tokens against a target model's logits (see dlk_verify_params in kernels.h).  With p and q the
// softmax of the target's and the draft's logits over the temperature, draft x of step i is kept while u_i q_i(x) < p_i(x);
// the token after the kept ones is drawn from max(p - q, 0) at the first refusal, or from p behind the last draft, as the
// first index whose cumulative weight exceeds u times the total.  Without draft logits a draft is certain (q(x) = 1).
// A decision compares two products and a draw finds a place in a sum over the vocabulary, so that everything behind the
// logits is in f64: the decisions are those of the exact probabilities, in any order of summation.
#include "kernels/device_common.h"

namespace dlk {
namespace {

constexpr int kThreads = 256, kDrawThreads = 1024, kDrawWaves = kDrawThreads / kWave;

__device__ __forceinline__ double wave_sum64(double v) {
    for (int offset = kWave / 2; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, kWave);
    return v;
}

// a work-group per row of logits: the largest (a NaN wins, then the lower index, as dl_argmax), and the sum
__global__ __launch_bounds__(kThreads) void verify_rows(const dlk_verify_params p) {
    __shared__ double sums[kThreads / kWave], scores[kThreads / kWave];
    __shared__ int64_t indices[kThreads / kWave];
    const int64_t per = p.drafts + 1 + (p.draft ? p.drafts : 0), b = blockIdx.x / per, r = blockIdx.x % per;
    const float* x = r <= p.drafts ? p.target + (b * (p.drafts + 1) + r) * p.vocabulary
                                   : p.draft + (b * p.drafts + r - p.drafts - 1) * p.vocabulary;
    double best = 0.0;
    int64_t index = -1;
    for (int64_t i = threadIdx.x; i < p.vocabulary; i += kThreads)
        if (index < 0 || prefer(x[i], i, best, index)) { best = x[i]; index = i; }
    auto join = [&](double s, int64_t j) {
        if (j >= 0 && (index < 0 || prefer(s, j, best, index))) { best = s; index = j; }
    };
    for (int offset = kWave / 2; offset > 0; offset >>= 1) {
        const double s = __shfl_xor(best, offset, kWave);
        join(s, __shfl_xor(index, offset, kWave));
    }
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) { scores[wave] = best; indices[wave] = index; }
    __syncthreads();
    for (int w = 0; w < kThreads / kWave; ++w) join(scores[w], indices[w]);
    double sum = 0.0;
    if (p.inverse > 0.0)
        for (int64_t i = threadIdx.x; i < p.vocabulary; i += kThreads) sum += exp((x[i] - best) * p.inverse);
    sum = wave_sum64(sum);
    if (threadIdx.x % kWave == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    dlk_verify_row out{0.0, static_cast<float>(best), static_cast<int32_t>(index)};
    for (int w = 0; w < kThreads / kWave; ++w) out.sum += sums[w];
    p.rows[b * (2 * p.drafts + 1) + r] = out;
}

// a work-group per sequence: the drafts kept, and the draw
__global__ __launch_bounds__(kDrawThreads) void verify_draw(const dlk_verify_params p) {
    __shared__ int stop;
    __shared__ double parts[kDrawWaves];
    __shared__ int64_t chosen;
    const int64_t b = blockIdx.x, n = p.drafts, V = p.vocabulary;
    const int t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const int64_t* drafted = p.drafted + b * n;
    const dlk_verify_row* rows = p.rows + b * (2 * n + 1);
    const float* uniforms = p.uniforms + b * (n + 1);
    if (t == 0) { stop = static_cast<int>(n); chosen = -1; }
    __syncthreads();
    for (int i = t; i < n; i += kDrawThreads) {
        const int64_t x = drafted[i];
        bool keep = x >= 0 && x < V;
        if (keep && p.inverse > 0.0) {
            const float* target = p.target + (b * (n + 1) + i) * V;
            double q = 1.0;
            if (p.draft)
                q = exp((static_cast<double>(p.draft[(b * n + i) * V + x]) - rows[n + 1 + i].largest) * p.inverse) /
                    rows[n + 1 + i].sum;
            keep = uniforms[i] * q < exp((static_cast<double>(target[x]) - rows[i].largest) * p.inverse) / rows[i].sum;
        } else if (keep) {
            keep = x == rows[i].index;
        }
        if (!keep) atomicMin(&stop, i);
    }
    __syncthreads();
    const int kept = stop;
    const bool refused = kept < n && drafted[kept] >= 0;
    int64_t drawn = rows[kept].index;
    if (p.inverse > 0.0) {
        const float* target = p.target + (b * (n + 1) + kept) * V;
        const float* draft = p.draft ? p.draft + (b * n + kept) * V : nullptr;
        const dlk_verify_row pr = rows[kept], qr = rows[n + 1 + (refused && p.draft ? kept : 0)];
        const int64_t out = refused ? drafted[kept] : -1;
        bool over = refused; // weights max(p - q, 0), else p
        auto weight = [&](int64_t i) {
            double w = exp((static_cast<double>(target[i]) - pr.largest) * p.inverse) / pr.sum;
            if (over) {
                const double q = draft ? exp((static_cast<double>(draft[i]) - qr.largest) * p.inverse) / qr.sum
                                       : i == out ? 1.0 : 0.0;
                w = fmax(w - q, 0.0);
            }
            return w;
        };
        // sums of the waves' equal slices of [begin, end)
        auto slices = [&](int64_t begin, int64_t end) {
            const int64_t per = (end - begin + kDrawWaves - 1) / kDrawWaves;
            const int64_t from = begin + wave * per, to = min(end, from + per);
            double s = 0.0;
            for (int64_t i = from + lane; i < to; i += kWave) s += weight(i);
            s = wave_sum64(s);
            __syncthreads();
            if (lane == 0) parts[wave] = s;
            __syncthreads();
            return per;
        };
        int64_t begin = 0, end = V, per = slices(0, V);
        double total = 0.0;
        for (int w = 0; w < kDrawWaves; ++w) total += parts[w];
        if (over && !(total > 0.0)) { // no weight over the draft's: the target's own
            over = false;
            per = slices(0, V);
            total = 0.0;
            for (int w = 0; w < kDrawWaves; ++w) total += parts[w];
        }
        if (total > 0.0 && total < INFINITY) {
            const double aim = uniforms[n] * total;
            double reach = 0.0;
            for (int level = 0; level < 2; ++level) {
                // the first slice that reaches past the aim, or the last one with any weight
                int slice = -1, filled = 0;
                double before = reach, filled_before = reach;
                for (int w = 0; w < kDrawWaves; ++w) {
                    if (parts[w] > 0.0) { filled = w; filled_before = before; }
                    if (slice < 0 && before + parts[w] > aim) slice = w;
                    if (slice < 0) before += parts[w];
                }
                if (slice < 0) { slice = filled; before = filled_before; }
                reach = before;
                begin = begin + slice * per;
                end = min(end, begin + per);
                if (level == 0) per = slices(begin, end);
            }
            if (wave == 0) {
                int64_t found = -1, filled = -1;
                for (int64_t at = begin; at < end && found < 0; at += kWave) {
                    const double w = at + lane < end ? weight(at + lane) : 0.0;
                    double sum = w;
                    for (int offset = 1; offset < kWave; offset <<= 1) {
                        const double up = __shfl_up(sum, offset, kWave);
                        if (lane >= offset) sum += up;
                    }
                    const uint64_t past = __ballot(reach + sum > aim && w > 0.0), some = __ballot(w > 0.0);
                    if (past) found = at + __builtin_ctzll(past);
                    if (some) filled = at + 63 - __builtin_clzll(some);
                    reach += __shfl(sum, kWave - 1, kWave);
                }
                if (lane == 0) chosen = found >= 0 ? found : filled;
            }
            __syncthreads();
            if (chosen >= 0) drawn = chosen;
        }
    }
    for (int64_t i = t; i <= n; i += kDrawThreads) p.tokens[b * (n + 1) + i] = i < kept ? drafted[i] : i == kept ? drawn : -1;
    if (t == 0) p.accepted[b] = kept;
}

} // namespace
} // namespace dlk

extern "C" int dlk_verify(const dlk_verify_params* params, dlh_stream stream_handle) {
    const dlk_verify_params& p = *params;
    if (p.batch < 0 || p.drafts < 0 || p.vocabulary <= 0 || p.vocabulary > INT32_MAX || p.drafts > INT32_MAX)
        return static_cast<int>(hipErrorInvalidValue);
    if (p.batch == 0) return 0;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_handle);
    const int64_t rows = p.batch * (p.drafts + 1 + (p.draft ? p.drafts : 0));
    if (rows > INT32_MAX) return static_cast<int>(hipErrorInvalidValue);
    hipLaunchKernelGGL(dlk::verify_rows, dim3(rows), dim3(dlk::kThreads), 0, stream, p);
    hipLaunchKernelGGL(dlk::verify_draw, dim3(p.batch), dim3(dlk::kDrawThreads), 0, stream, p);
    return static_cast<int>(hipGetLastError());
}
