// Verification of drafted tokens against a target model's logits (see dlk_verify_params in kernels.h).  With p and q the
// softmax of the target's and the draft's logits over the temperature, draft x of step i is kept while u_i q_i(x) < p_i(x);
// the token after the kept ones is drawn from max(p - q, 0) at the first refusal, or from p behind the last draft, as the
// first index whose cumulative weight exceeds u times the total.  Without draft logits a draft is certain (q(x) = 1).
//
// A decision compares two products and a draw finds a place in a sum over the vocabulary, so that everything behind the
// logits is in f64, with exponentials off by 1.1e-12: decisions are those of the exact probabilities, in any order of
// summation, but where a number lies that close to its border.
//
// Three launches.  verify_rows reads every logit once, slices of a row as work-groups, and leaves each slice's largest and
// sum.  verify_weights decides what is kept and sums the weights of the row behind it, 1024 entries a work-group.  verify_draw
// finds the part of 1024 and in it the index.  The first is bound by the read and the f64 instructions, which a work-group does one
// after the other (32 runs of 7 drafts over 32000 entries, 61 MB: 19 us), the others by round trips to memory (7 and 8 us).  A
// greedy verification needs the largest only and no sums.
#include "kernels/device_common.h"

#include <algorithm>

namespace dlk {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kHeld = 16; // entries of a slice per thread
constexpr int kDraw = DLK_VERIFY_DRAW, kDrawHeld = kDraw / kThreads;

// A shifted copy of v across the wave's lanes (CONTROL), zero where nothing arrives or ROWS leaves the row out.
template <int CONTROL, int ROWS> __device__ __forceinline__ double shifted(double v) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CONTROL, ROWS, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CONTROL, ROWS, 0xf, false));
}

// sums of the lanes up to each: within rows of 16 lanes, then the rows before, in registers
__device__ __forceinline__ double wave_scan64(double v) {
    v += shifted<0x111, 0xf>(v);
    v += shifted<0x112, 0xf>(v);
    v += shifted<0x114, 0xf>(v);
    v += shifted<0x118, 0xf>(v);
    v += shifted<0x142, 0xa>(v); // rows 1 and 3 take lane 15 of the row before
    v += shifted<0x143, 0xc>(v); // the upper half lane 31
    return v;
}

__device__ __forceinline__ double lane_of(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}

__device__ __forceinline__ double wave_sum64(double v) { return lane_of(wave_scan64(v), kWave - 1); }

// a b + c with c in scalar registers (the compiler copies such a constant into vector registers before each use)
__device__ __forceinline__ double fma_constant(double a, double b, double c) {
    double d;
    __asm__("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
}

// exp((l - largest) * inverse) for l <= largest, to a relative 1.1e-12, far below what separates any two numbers compared
// here: (l - largest) inverse = n ln 2 + r, |r| <= ln 2 / 2, and the polynomial of degree 8 through exp at the Chebyshev
// points of that range.  n is found in f32, where being off by one part in 10^6 only moves r.  A third of the instructions
// of the library's exp, which bound the pass over the logits.  0 below exp(-700); a NaN stays.
// WIDE: n is found from the difference in f64, for temperatures whose inverse, or the difference of two logits times it, f32
// does not hold (-inf times an inverse that became 0 is no number).  An instruction an entry more, so only for those.
template <bool WIDE> struct Exponential {
    double largest, inverse;
    float largest32, inverse32;
    __device__ __forceinline__ Exponential(double largest_, double inverse_)
        : largest(largest_), inverse(inverse_), largest32(static_cast<float>(largest_)), inverse32(static_cast<float>(inverse_)) {}
    __device__ __forceinline__ double operator()(float l) const {
        const double x = (static_cast<double>(l) - largest) * inverse;
        const float about = WIDE ? static_cast<float>(x) : (l - largest32) * inverse32;
        const float n = __builtin_rintf(about * 1.44269504f);
        const double nd = n;
        const double r = __builtin_fma(nd, -0x1.62e42fefa39efp-1, x);
        double y = fma_constant(r, 0x1.a15a60062d0e8p-16, 0x1.a1aa939e66a93p-13);
        y = fma_constant(y, r, 0x1.6c164de86c8c8p-10);
        y = fma_constant(y, r, 0x1.1110809f385f2p-7);
        y = fma_constant(y, r, 0x1.555555742d972p-5);
        y = fma_constant(y, r, 0x1.555555a279c87p-3);
        y = fma_constant(y, r, 0x1.fffffffff71b2p-2);
        y = fma_constant(y, r, 0x1.ffffffffd382fp-1);
        y = __builtin_fma(y, r, 1.0);
        // 2^n: n onto the exponent (y is near 1, n above -1011)
        const int high = __double2hiint(y) + (static_cast<int>(n) << 20);
        const bool none = about < -700.0f;
        return __hiloint2double(none ? 0 : high, none ? 0 : __double2loint(y));
    }
};

__device__ __forceinline__ int64_t slice_begin(const dlk_verify_params& p, int64_t slice) {
    return min(slice * p.slice, p.vocabulary);
}
__device__ __forceinline__ const float* target_row(const dlk_verify_params& p, int64_t b, int64_t i) {
    return p.target + (b * (p.drafts + 1) + i) * p.vocabulary;
}
__device__ __forceinline__ const dlk_verify_slice* slices_of(const dlk_verify_params& p, int64_t b, int64_t row) {
    return p.rows + (b * (2 * p.drafts + 1) + row) * p.slices;
}

template <bool GREEDY, bool WIDE>
__global__ __launch_bounds__(kThreads) void verify_rows(const dlk_verify_params p) {
    __shared__ double sums[kWaves];
    __shared__ float tops[kWaves];
    __shared__ int64_t indices[kWaves];
    const int t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const uint32_t per_batch = static_cast<uint32_t>(p.drafts + 1 + (p.draft ? p.drafts : 0));
    const uint32_t row = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
    const int64_t b = row / per_batch, r = row % per_batch;
    const float* x = r <= p.drafts ? target_row(p, b, r) : p.draft + (b * p.drafts + r - p.drafts - 1) * p.vocabulary;
    const int64_t begin = slice_begin(p, slice), end = slice_begin(p, slice + 1);
    const int length = static_cast<int>(end - begin);
    dlk_verify_slice out{0.0, -INFINITY, -1};
    float held[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) held[j] = t + j * kThreads < length ? x[begin + t + j * kThreads] : -INFINITY;
    if constexpr (GREEDY) {
        float top = held[0]; // (a slice has an entry; a thread without one says so below)
        int at = 0;
#pragma unroll
        for (int j = 1; j < kHeld; ++j)
            if (t + j * kThreads < length && (held[j] > top || (held[j] != held[j] && top == top))) top = held[j], at = j;
        double best = top;
        int64_t index = t < length ? begin + t + at * kThreads : -1;
        auto join = [&](double s, int64_t j) {
            if (j >= 0 && (index < 0 || prefer(s, j, best, index))) { best = s; index = j; }
        };
        for (int offset = kWave / 2; offset > 0; offset >>= 1) {
            const double s = __shfl_xor(best, offset, kWave);
            join(s, __shfl_xor(index, offset, kWave));
        }
        if (lane == 0) { sums[wave] = best; indices[wave] = index; }
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) join(sums[w], indices[w]);
        out.largest = static_cast<float>(best);
        out.index = static_cast<int32_t>(index);
    } else {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) top = fmaxf(top, held[j]); // (a NaN is passed over here and spoils the sum below)
        top = wave_max(top);
        if (lane == 0) tops[wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
        const Exponential<WIDE> weight(top == -INFINITY ? 0.0 : top, p.inverse);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < kHeld; j += 4)
            if (j * kThreads < length) // (what lies behind the slice weighs nothing)
                sum += (weight(held[j]) + weight(held[j + 1])) + (weight(held[j + 2]) + weight(held[j + 3]));
        sum = wave_sum64(sum);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) out.sum += sums[w];
        out.largest = top;
    }
    if (t == 0) p.rows[(b * (2 * p.drafts + 1) + r) * p.slices + slice] = out;
}

// What a row's probabilities are made of: exp((l - largest) / T) * scale.
struct Row {
    double largest, scale;
};

__device__ __forceinline__ int64_t greedy_of(const dlk_verify_params& p, const dlk_verify_slice* slices) {
    double best = 0.0;
    int64_t index = -1;
    for (int i = 0; i < p.slices; ++i) {
        const int64_t j = slices[i].index;
        if (j >= 0 && (index < 0 || prefer(slices[i].largest, j, best, index))) { best = slices[i].largest; index = j; }
    }
    return index;
}

constexpr int kTeam = 8;                     // lanes that join a row's slices
constexpr int kStep = kThreads / kTeam / 2;  // drafts looked at in one round, target and draft rows side by side

struct Decision {
    int kept;
    bool refused; // a draft was refused there
    Row p, q;     // of the row behind the kept ones: the target's, and the refused draft's
};

// What is kept of sequence b, by the whole work-group.
template <bool WIDE> __device__ __forceinline__ Decision decide(const dlk_verify_params& p, int64_t b) {
    __shared__ int stop;
    __shared__ Row rows[2][kStep];
    const int t = threadIdx.x, n = static_cast<int>(p.drafts), team = t / kTeam, member = t % kTeam;
    const int64_t* drafted = p.drafted + b * n;
    if (t == 0) stop = n;
    __syncthreads();
    for (int first = 0;; first += kStep) {
        // what the comparisons need besides the rows' sums, asked for first
        const int step = first + t;
        const bool tests = t < kStep && step < n;
        const int64_t x = tests ? drafted[step] : -1;
        const bool inside = x >= 0 && x < p.vocabulary;
        const float target_logit = inside ? target_row(p, b, step)[x] : 0.0f;
        const float draft_logit = inside && p.draft ? p.draft[(b * n + step) * p.vocabulary + x] : 0.0f;
        const float uniform = tests ? p.uniforms[b * (n + 1) + step] : 0.0f;
        const bool draft = team >= kStep;
        const int i = first + team % kStep;
        const bool any = draft ? p.draft && i < n : i <= n;
        const dlk_verify_slice* slices = slices_of(p, b, any ? (draft ? n + 1 + i : i) : 0);
        double largest = -INFINITY, sum = 0.0;
        for (int begin = 0; begin < p.slices; begin += 8 * kTeam) {
            dlk_verify_slice held[8];
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 8; ++k) held[k] = slices[min(begin + member + kTeam * k, p.slices - 1)];
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, held[k].largest); // (repeated ones do not matter)
#pragma unroll
            for (int offset = kTeam / 2; offset > 0; offset >>= 1) top = fmaxf(top, __shfl_xor(top, offset, kWave));
            const double next = fmax(largest, static_cast<double>(top));
            const Exponential<WIDE> weight(next == -INFINITY ? 0.0 : next, p.inverse); // (slices of -inf weigh nothing)
            if (begin > 0) sum *= weight(static_cast<float>(largest));
            largest = next;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (begin + member + kTeam * k < p.slices) sum += held[k].sum * weight(held[k].largest);
        }
#pragma unroll
        for (int offset = kTeam / 2; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset, kWave);
        if (member == 0 && any) rows[draft][i - first] = {largest, 1.0 / sum};
        __syncthreads();
        if (tests) {
            bool keep = inside;
            if (keep) {
                double q = 1.0;
                if (p.draft) q = Exponential<WIDE>(rows[1][t].largest, p.inverse)(draft_logit) * rows[1][t].scale;
                keep = uniform * q < Exponential<WIDE>(rows[0][t].largest, p.inverse)(target_logit) * rows[0][t].scale;
            }
            if (!keep) atomicMin(&stop, step);
        }
        __syncthreads();
        const int kept = stop;
        if (kept < first + kStep) {
            const bool refused = kept < n && drafted[kept] >= 0;
            return {kept, refused, rows[0][kept - first], refused && p.draft ? rows[1][kept - first] : Row{0.0, 0.0}};
        }
        __syncthreads(); // the rows are written again
    }
}

// What the token behind the kept ones is drawn with: p, less q where a draft was refused.
template <bool WIDE> struct Weights {
    const float* target;
    const float* draft; // the refused draft's row, or NULL
    Exponential<WIDE> p, q;
    double p_scale, q_scale;
    int64_t out;        // a certain draft that was refused, or -1
    __device__ __forceinline__ Weights(const dlk_verify_params& v, int64_t b, const Decision& d)
        : target(target_row(v, b, d.kept)),
          draft(d.refused && v.draft ? v.draft + (b * v.drafts + d.kept) * v.vocabulary : nullptr), p(d.p.largest, v.inverse),
          q(d.q.largest, v.inverse), p_scale(d.p.scale), q_scale(d.q.scale),
          out(d.refused && !v.draft ? v.drafted[b * v.drafts + d.kept] : -1) {}
    // the target's weight of entry i, whose logits are l and, with a draft's row, m, and what it has over the draft's.  Both
    // products are rounded before they are subtracted: fused into the subtraction, one would leave the other's rounding where
    // the two are equal, and rows that agree would be drawn from by that instead of by p.
    __device__ __forceinline__ double of(float l, float m, int64_t i, double& over) const {
#pragma clang fp contract(off)
        const double w = p(l) * p_scale;
        const double rest = w - (draft ? q(m) * q_scale : i == out ? 1.0 : 0.0);
        over = rest < 0.0 ? 0.0 : rest; // (a NaN stays)
        return w;
    }
};

// a work-group per 1024 entries of a sequence's row
template <bool WIDE> __global__ __launch_bounds__(kThreads) void verify_weights(const dlk_verify_params p) {
    __shared__ double sums[2][kWaves];
    const int t = threadIdx.x;
    const uint32_t parts = static_cast<uint32_t>((p.vocabulary + kDraw - 1) / kDraw), part = blockIdx.x % parts;
    const int64_t b = blockIdx.x / parts;
    const Decision d = decide<WIDE>(p, b);
    if (part == 0 && t == 0) {
        p.accepted[b] = d.kept;
        p.decisions[4 * b] = d.p.largest;
        p.decisions[4 * b + 1] = d.p.scale;
        p.decisions[4 * b + 2] = d.q.largest;
        p.decisions[4 * b + 3] = d.refused ? d.q.scale : -1.0;
    }
    const Weights<WIDE> weights(p, b, d);
    const int64_t begin = static_cast<int64_t>(part) * kDraw;
    float l[kDrawHeld], m[kDrawHeld];
#pragma unroll
    for (int j = 0; j < kDrawHeld; ++j) {
        const int64_t i = begin + t + j * kThreads;
        l[j] = i < p.vocabulary ? weights.target[i] : -INFINITY;
        m[j] = i < p.vocabulary && weights.draft ? weights.draft[i] : -INFINITY;
    }
    double own = 0.0, over = 0.0;
#pragma unroll
    for (int j = 0; j < kDrawHeld; ++j) {
        double rest;
        const double w = weights.of(l[j], m[j], begin + t + j * kThreads, rest);
        own += w; // (nothing behind the row)
        over += rest;
    }
    own = wave_sum64(own);
    over = wave_sum64(over);
    if (t % kWave == 0) {
        sums[0][t / kWave] = over;
        sums[1][t / kWave] = own;
    }
    __syncthreads();
    if (t < 2) p.drawn[2 * (b * parts + part) + t] = (sums[t][0] + sums[t][1]) + (sums[t][2] + sums[t][3]);
}

// a work-group per sequence
template <bool WIDE> __global__ __launch_bounds__(kThreads) void verify_draw(const dlk_verify_params p) {
    __shared__ double sums[kWaves];
    __shared__ int first_index, last_index;
    __shared__ double best_s[kWaves];
    __shared__ int64_t index_s[kWaves];
    const int t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const int64_t b = blockIdx.x, n = p.drafts;
    const int64_t token = t < n ? p.drafted[b * n + t] : -1; // (asked for early; the ones beyond at the end)
    int kept = 0;
    int64_t drawn = -1;
    if (p.inverse > 0.0) {
        const int parts = static_cast<int>((p.vocabulary + kDraw - 1) / kDraw);
        const double* weight_of = p.drawn + 2 * b * parts;
        const double early_over = weight_of[2 * min(lane, parts - 1)], early_own = weight_of[2 * min(lane, parts - 1) + 1];
        const float uniform = p.uniforms[b * (n + 1) + n];
        kept = static_cast<int>(p.accepted[b]);
        const Decision d{kept, !(p.decisions[4 * b + 3] < 0.0), {p.decisions[4 * b], p.decisions[4 * b + 1]},
                         {p.decisions[4 * b + 2], p.decisions[4 * b + 3]}};
        const Weights<WIDE> weights(p, b, d);
        // every wave goes over the parts' sums alike, 64 at a time: of max(p - q, 0), or of p where that is zero or nothing
        // was refused
        int of = d.refused ? 0 : 1;
        auto sums_from = [&](int at) {
            if (at + lane >= parts) return 0.0;
            return at > 0 ? weight_of[2 * (at + lane) + of] : of == 0 ? early_over : early_own;
        };
        double first = wave_scan64(sums_from(0));
        auto total_of = [&] {
            double s = lane_of(first, kWave - 1);
            for (int at = kWave; at < parts; at += kWave) s += wave_sum64(sums_from(at));
            return s;
        };
        double total = total_of();
        if (of == 0 && !(total > 0.0) && total == total) {
            of = 1;
            first = wave_scan64(sums_from(0));
            total = total_of();
        }
        if (total > 0.0 && total < INFINITY) {
            const double aim = uniform * total;
            // the first part that reaches past the aim, or the last with any weight
            int part = -1, filled = 0;
            double reach = 0.0, before = 0.0, before_filled = 0.0;
            for (int at = 0; at < parts && part < 0; at += kWave) {
                const double own = sums_from(at), sum = at == 0 ? first : wave_scan64(own);
                const uint64_t past = __ballot(own > 0.0 && reach + sum > aim), some = __ballot(own > 0.0);
                if (past) {
                    part = at + __builtin_ctzll(past);
                    before = reach + lane_of(sum - own, part - at);
                }
                if (some) {
                    filled = at + 63 - __builtin_clzll(some);
                    before_filled = reach + lane_of(sum - own, filled - at);
                }
                reach += lane_of(sum, kWave - 1);
            }
            if (part < 0) { part = filled; before = before_filled; }
            // its entries, a run of them per thread, in order
            const int64_t begin = static_cast<int64_t>(part) * kDraw + t * kDrawHeld;
            float l[kDrawHeld], m[kDrawHeld];
#pragma unroll
            for (int j = 0; j < kDrawHeld; ++j) {
                l[j] = begin + j < p.vocabulary ? weights.target[begin + j] : -INFINITY;
                m[j] = begin + j < p.vocabulary && weights.draft ? weights.draft[begin + j] : -INFINITY;
            }
            double held[kDrawHeld], own = 0.0;
#pragma unroll
            for (int j = 0; j < kDrawHeld; ++j) {
                double over;
                const double w = weights.of(l[j], m[j], begin + j, over);
                held[j] = of == 0 ? over : w;
                own += held[j];
            }
            const double sum = wave_scan64(own);
            if (lane == kWave - 1) sums[wave] = sum;
            if (t == 0) { first_index = INT32_MAX; last_index = -1; }
            __syncthreads();
            double at = before + (sum - own);
            for (int w = 0; w < wave; ++w) at += sums[w];
            int found = INT32_MAX, last = -1;
#pragma unroll
            for (int j = 0; j < kDrawHeld; ++j) {
                at += held[j];
                if (held[j] > 0.0) {
                    last = static_cast<int>(begin + j);
                    if (found == INT32_MAX && at > aim) found = last;
                }
            }
            if (found != INT32_MAX) atomicMin(&first_index, found);
            if (last >= 0) atomicMax(&last_index, last);
            __syncthreads();
            drawn = first_index != INT32_MAX ? first_index : last_index;
        }
        if (drawn < 0) { // no sum to draw by: the row's argmax
            const float* x = weights.target;
            double best = 0.0;
            int64_t index = -1;
            auto join = [&](double s, int64_t j) {
                if (j >= 0 && (index < 0 || prefer(s, j, best, index))) { best = s; index = j; }
            };
            for (int64_t i = t; i < p.vocabulary; i += kThreads) join(x[i], i);
            for (int offset = kWave / 2; offset > 0; offset >>= 1) {
                const double s = __shfl_xor(best, offset, kWave);
                join(s, __shfl_xor(index, offset, kWave));
            }
            if (lane == 0) { best_s[wave] = best; index_s[wave] = index; }
            __syncthreads();
            for (int w = 0; w < kWaves; ++w) join(best_s[w], index_s[w]);
            drawn = index;
        }
    } else {
        if (t == 0) first_index = static_cast<int>(n);
        __syncthreads();
        for (int i = t; i < n; i += kThreads)
            if (p.drafted[b * n + i] != greedy_of(p, slices_of(p, b, i))) atomicMin(&first_index, i);
        __syncthreads();
        kept = first_index;
        drawn = greedy_of(p, slices_of(p, b, kept));
        if (t == 0) p.accepted[b] = kept;
    }
    for (int64_t i = t; i <= n; i += kThreads)
        p.tokens[b * (n + 1) + i] = i < kept ? (i == t ? token : p.drafted[b * n + i]) : i == kept ? drawn : -1;
}

} // namespace
} // namespace dlk

extern "C" int dlk_verify_slices(int64_t rows, int64_t vocabulary) {
    // whole slices that a work-group's registers hold, more of them while the rows are few for 256 CUs
    const int64_t most = dlk::kThreads * dlk::kHeld, fewest = (vocabulary + most - 1) / most;
    const int64_t wanted = std::min<int64_t>((vocabulary + 511) / 512, 1024 / std::max<int64_t>(rows, 1));
    return static_cast<int>(std::min<int64_t>(std::max(fewest, wanted), INT32_MAX));
}

extern "C" int dlk_verify(const dlk_verify_params* params, dlh_stream stream_handle) {
    const dlk_verify_params& p = *params;
    if (p.batch < 0 || p.drafts < 0 || p.vocabulary <= 0 || p.vocabulary > INT32_MAX || p.drafts > (1 << 20) || p.slices <= 0 ||
        p.slice <= 0 || p.slice > dlk::kThreads * dlk::kHeld || p.slice * p.slices < p.vocabulary)
        return static_cast<int>(hipErrorInvalidValue);
    if (p.batch == 0) return 0;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_handle);
    const int64_t groups = p.batch * (p.drafts + 1 + (p.draft ? p.drafts : 0)) * p.slices;
    const int64_t parts = p.batch * ((p.vocabulary + dlk::kDraw - 1) / dlk::kDraw);
    if (groups > DLK_MOST_GROUPS || parts > DLK_MOST_GROUPS) return static_cast<int>(hipErrorInvalidValue);
    const dim3 threads(dlk::kThreads), rows(groups), sequences(p.batch);
    // between 2^-100 and 2^100 f32 holds the inverse, and two logits that are further apart than f32 counts weigh nothing
    const bool wide = p.inverse < 0x1p-100 || p.inverse > 0x1p100;
    if (!(p.inverse > 0.0)) {
        hipLaunchKernelGGL((dlk::verify_rows<true, false>), rows, threads, 0, stream, p);
        hipLaunchKernelGGL(dlk::verify_draw<false>, sequences, threads, 0, stream, p);
    } else if (wide) {
        hipLaunchKernelGGL((dlk::verify_rows<false, true>), rows, threads, 0, stream, p);
        hipLaunchKernelGGL(dlk::verify_weights<true>, dim3(parts), threads, 0, stream, p);
        hipLaunchKernelGGL(dlk::verify_draw<true>, sequences, threads, 0, stream, p);
    } else {
        hipLaunchKernelGGL((dlk::verify_rows<false, false>), rows, threads, 0, stream, p);
        hipLaunchKernelGGL(dlk::verify_weights<false>, dim3(parts), threads, 0, stream, p);
        hipLaunchKernelGGL(dlk::verify_draw<false>, sequences, threads, 0, stream, p);
    }
    return static_cast<int>(hipGetLastError());
}
