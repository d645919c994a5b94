// The gated delta rule token by token (see dlk_delta_params in kernels.h): for single and drafted tokens, whose time is that
// of the states' way from memory and back.
//   a = e^decay,  w = rate (v - a S^T k),  out = scale (a S^T q + (k . q) w),  S = a S + k w^T
// so that both products with the state are taken before it changes, in one pass over it and one exchange between lanes.
#include "kernels/parts.h"

namespace dlk {
namespace {

constexpr int kThreads = 256;

// N neighbouring entries of a row as they lie in memory, and in f32.
template <int N, bool BF16> struct Entries {
    static constexpr int WORDS = BF16 ? N / 2 : N;
    uint32_t word[WORDS];
    __device__ __forceinline__ void load(const void* x, int64_t at) {
        const char* from = static_cast<const char*>(x) + at * (BF16 ? 2 : 4);
        if constexpr (WORDS == 2) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(from);
            word[0] = w.x, word[1] = w.y;
        } else {
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i) {
                const u32x4 w = reinterpret_cast<const u32x4*>(from)[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) word[4 * i + j] = w[j];
            }
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (BF16) return i % 2 ? bf16_hi(word[i / 2]) : bf16_lo(word[i / 2]);
        else return __uint_as_float(word[i]);
    }
};

// The sum over the lanes that differ in bits 3, 4 and 5 alone.
__device__ __forceinline__ float sum_over_rows(float x) {
    constexpr int kRotate8 = 0x128; // row_ror:8, of 16 lanes
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x), kRotate8, 0xf, 0xf, false));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A wave holds 32 columns of a head's state: 8 lanes side by side with 4 columns each, 8 groups of them with DK / 8 rows each.
// Columns know nothing of one another, so waves do not either.  The next token's rows are on their way while one is worked
// on (a token more takes 0.95 us; its rows waited for 1.35).  64 requests' states of 32 x 128 x 128, 268 MB: 44.7 us, 6.0 TB/s.
template <int DK, bool BF16, bool V_BF16>
__global__ __launch_bounds__(kThreads) void delta_step(const dlk_delta_params p) {
    constexpr int R = DK / 8;
    const int lane = threadIdx.x % kWave;
    const uint32_t slices = p.value_dim / 32;
    const auto shared = [](uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); };
    const uint32_t unit = shared((blockIdx.x * kThreads + threadIdx.x) / kWave);
    if (unit >= static_cast<uint32_t>(p.item_count) * p.heads * slices) return;
    const int slice = shared(unit % slices), head = shared(unit / slices % p.heads), key_head = shared(head / p.group);
    const dlk_delta_item* own = p.items + shared(unit / slices / p.heads);
    const int source = shared(own->source), target = shared(own->target), first = shared(own->token), count = shared(own->count);
    const int row = lane / 8 * R, column = slice * 32 + lane % 8 * 4;
    const uint32_t within = row * p.value_dim + column;
    const int64_t size = static_cast<int64_t>(DK) * p.value_dim;

    struct Token {
        Entries<R, BF16> q, k;
        Entries<4, V_BF16> v;
        float decay, rate;
    };
    const auto load = [&](int t, Token& to) {
        const int64_t token = first + t;
        to.q.load(p.q.x, token * p.q.row + key_head * p.q.head + row);
        to.k.load(p.k.x, token * p.k.row + key_head * p.k.head + row);
        to.v.load(p.v.x, token * p.v.row + head * p.v.head + column);
        to.decay = p.decay[token * p.heads + head];
        to.rate = p.rate[token * p.heads + head];
    };
    Token next;
    load(0, next);
    f32x4 s[R];
    if (source >= 0) {
        const float* from = p.states + (static_cast<int64_t>(source) * p.heads + head) * size;
#pragma unroll
        for (int i = 0; i < R; ++i) s[i] = *reinterpret_cast<const f32x4*>(from + within + i * p.value_dim);
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) s[i] = 0.0f;
    }
    for (int t = 0; t < count; ++t) {
        const Token now = next;
        if (t + 1 < count) load(t + 1, next);
        const float a = expf(now.decay);
        f32x4 sk = 0.0f, sq = 0.0f;
        float kq = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk[j] = fmaf(now.k[i], s[i][j], sk[j]);
                sq[j] = fmaf(now.q[i], s[i][j], sq[j]);
            }
            kq = fmaf(now.k[i], now.q[i], kq);
        }
        kq = sum_over_rows(kq);
        f32x4 w, out;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = now.rate * (now.v[j] - a * sum_over_rows(sk[j]));
            out[j] = p.scale * (a * sum_over_rows(sq[j]) + kq * w[j]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = fmaf(now.k[i], w[j], a * s[i][j]);
        if (lane < 8) *reinterpret_cast<f32x4*>(p.out + (static_cast<int64_t>(first + t) * p.heads + head) * p.value_dim + column) = out;
    }
    float* to = p.states + (static_cast<int64_t>(target) * p.heads + head) * size;
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<f32x4*>(to + within + i * p.value_dim) = s[i];
}

template <int DK> void launch(const dlk_delta_params& p, unsigned groups, hipStream_t at) {
    if (p.k.bf16) {
        if (p.v.bf16) delta_step<DK, true, true><<<groups, kThreads, 0, at>>>(p);
        else delta_step<DK, true, false><<<groups, kThreads, 0, at>>>(p);
    } else {
        if (p.v.bf16) delta_step<DK, false, true><<<groups, kThreads, 0, at>>>(p);
        else delta_step<DK, false, false><<<groups, kThreads, 0, at>>>(p);
    }
}

} // namespace
} // namespace dlk

extern "C" int dlk_delta_step(const dlk_delta_params* p, dlh_stream stream) {
    using namespace dlk;
    const int64_t waves = static_cast<int64_t>(p->item_count) * p->heads * (p->value_dim / 32);
    const int64_t groups = (waves + kThreads / kWave - 1) / (kThreads / kWave);
    if (p->value_dim <= 0 || p->value_dim % 32 != 0 || p->group <= 0 || groups > DLK_MOST_GROUPS || p->q.bf16 != p->k.bf16)
        return hipErrorInvalidValue;
    if (groups == 0) return 0;
    hipStream_t at = reinterpret_cast<hipStream_t>(stream);
    switch (p->key_dim) {
    case 32: launch<32>(*p, static_cast<unsigned>(groups), at); break;
    case 64: launch<64>(*p, static_cast<unsigned>(groups), at); break;
    case 128: launch<128>(*p, static_cast<unsigned>(groups), at); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
