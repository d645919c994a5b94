// A layer of experts over few rows (see dlk_experts_params in kernels.h): the router in f64, the hidden entries of the chosen
// experts, their output entries, and the weighted sum.  Bound by memory: a few rows read each chosen expert's matrices once.  16 rows
// through 8 of 64 bf16 experts of 1024 x 2048: router 12 us, hidden entries 90 (5.3 TB/s), outputs 50 (4.8 TB/s), sum 4.8; 200 rows
// through 4 of 32 of 768 x 2048: 8, 47, 32 and 4.8; one row through 2 of 16 of 704 x 1024: 4.4, 4.3, and 3.8 for outputs and sum.
//
// Products keep all bits of an f32: bf16 matrices go into v_mfma_f32_16x16x32_bf16 as they are, rows as three bf16 parts that
// hold all 24 bits (bf16 rows are one); f32 matrices and rows go into v_mfma_f32_16x16x4_f32.
#include "kernels/experts_layout.h"
#include "kernels/parts.h"

#include <algorithm>
#include <type_traits>

namespace dlk {
namespace {

constexpr uint32_t kBeyond = 1u << 31; // an offset behind every buffer's end
constexpr int kPairs = 8000; // (row, chosen expert) pairs of a launch: the list of an expert's in LDS, beside 48 KB of rows in 64

__device__ __forceinline__ float entry(const void* x, int bf16, int64_t at) {
    return bf16 ? bf16_to_f32(static_cast<const uint16_t*>(x)[at]) : static_cast<const float*>(x)[at];
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ void eight(const void* x, int bf16, int64_t at, float (&v)[8]) {
    if (bf16) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(x) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    } else {
        const f32x4* from = reinterpret_cast<const f32x4*>(static_cast<const float*>(x) + at);
        const f32x4 a = from[0], b = from[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    }
}

struct Plan {          // what a launch's kernels hand on
    uint16_t* pick;    // [tokens, top]: the chosen experts
    double* logits;    // [tokens, experts], or NULL: the router's kernel takes them
    char* rows;        // x as the products read it (see `planes` and experts_layout.h), or NULL: p.x itself
    char* act;         // the hidden entries: f32 (`whole`), or three parts
    bool whole, laid;  // laid: in pieces, see experts_layout.h
    float* partial;    // [tokens, top, dim]: outputs of each pair
    int planes;        // bf16 matrices: parts of a row of x; 0: f32 matrices, f32 rows
};

// A row's logits in f64, which hold products of two f32 exactly, so that rows choose as the exact logits do but for ties within
// 1e-15 of them: two experts at a time for wave `wave` of `waves`.  Bound by the conversions to f64 and, for few rows, by one way to
// memory, so all of a wave's loads of 2048 entries are made at once.  WIDE: pieces of 8 entries (dim a multiple of 8, 16-byte aligned).
template <bool WIDE>
__device__ __forceinline__ void take_logits(const dlk_experts_params& p, int64_t token, int wave, int waves, double* logits) {
    const int lane = threadIdx.x % kWave;
    for (int first = 2 * wave; first < p.experts; first += 2 * waves) {
        if constexpr (WIDE) {
            constexpr int N = 2, U = 4; // experts, and steps at a time
            double sum[N] = {};
            for (int i = lane * 8; i < p.dim; i += U * kWave * 8) {
                float x[U][8], w[U][N][8];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int at = min(i + u * kWave * 8, p.dim - 8);
                    eight(p.x, p.x_bf16, token * p.dim + at, x[u]);
#pragma unroll
                    for (int n = 0; n < N; ++n) eight(p.router, p.router_bf16, static_cast<int64_t>(min(first + n, p.experts - 1)) * p.dim + at, w[u][n]);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u * kWave * 8 < p.dim)
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int j = 0; j < 8; ++j) sum[n] = fma(static_cast<double>(x[u][j]), static_cast<double>(w[u][n][j]), sum[n]);
            }
            // lanes that differ in the lowest bit share the two sums out
            const bool odd = lane & 1;
            double z = (odd ? sum[1] : sum[0]) + __shfl_xor(odd ? sum[0] : sum[1], 1);
#pragma unroll
            for (int d = 2; d < kWave; d *= 2) z += __shfl_xor(z, d);
            if (lane < N && first + lane < p.experts) logits[first + lane] = z;
        } else {
            constexpr int U = 16;
            double sum[2] = {};
            const int64_t row[2] = {static_cast<int64_t>(first) * p.dim, static_cast<int64_t>(min(first + 1, p.experts - 1)) * p.dim};
            const auto entries = [&](auto x_bf16, auto router_bf16) { // (a type looked up at each load would have each waited for)
                for (int i = lane; i < p.dim; i += U * kWave) {
                    float x[U], w[U][2];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int at = min(i + u * kWave, p.dim - 1);
                        x[u] = entry(p.x, x_bf16, token * p.dim + at);
#pragma unroll
                        for (int n = 0; n < 2; ++n) w[u][n] = entry(p.router, router_bf16, row[n] + at);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (i + u * kWave < p.dim)
#pragma unroll
                            for (int n = 0; n < 2; ++n) sum[n] = fma(static_cast<double>(x[u]), static_cast<double>(w[u][n]), sum[n]);
                }
            };
            const std::true_type yes;
            const std::false_type no;
            if (p.x_bf16) p.router_bf16 ? entries(yes, yes) : entries(yes, no);
            else p.router_bf16 ? entries(no, yes) : entries(no, no);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const double z = wave_sum_f64(sum[n]);
                if (lane == 0 && first + n < p.experts) logits[first + n] = z;
            }
        }
    }
}

// A row as the products read it, by `threads` threads.
template <bool WIDE> __device__ __forceinline__ void lay_row(const dlk_experts_params& p, const Plan& plan, int64_t token, int thread, int threads) {
    if (!plan.rows) return;
    if constexpr (WIDE) {
        for (int i = thread * 8; i < p.dim; i += threads * 8) {
            float v[8];
            eight(p.x, p.x_bf16, token * p.dim + i, v);
            if (plan.planes == 0) {
                f32x4* to = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(plan.rows) + token * p.dim + i);
                to[0] = f32x4{v[0], v[1], v[2], v[3]}, to[1] = f32x4{v[4], v[5], v[6], v[7]};
            }
            for (int part = 0; part < plan.planes; ++part)
                *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(plan.rows) + (part * p.tokens + token) * p.dim + i) = cut(v);
        }
    } else {
        const int unit = p.weights_bf16 ? 8 : 4, line = laid_width(p.dim, unit), whole = p.dim / unit * unit;
        for (int i = thread; i < line; i += threads) {
            const int from = i < whole ? i : i - whole + p.dim - unit;
            float v = i < whole || from >= whole ? entry(p.x, p.x_bf16, token * p.dim + from) : 0.0f;
            if (plan.planes == 0) reinterpret_cast<float*>(plan.rows)[token * line + i] = v;
            for (int part = 0; part < plan.planes; ++part)
                reinterpret_cast<uint16_t*>(plan.rows)[(part * p.tokens + token) * line + i] = cut(v);
        }
    }
}

// Work-groups that share a row's logits, where one would take long.
constexpr int kLogits = 256, kLogitsExperts = kLogits / kWave * 2;
template <bool WIDE>
__global__ __launch_bounds__(kLogits) void experts_logits(const dlk_experts_params p, const Plan plan) {
    const int64_t token = blockIdx.y;
    take_logits<WIDE>(p, token, blockIdx.x * (kLogits / kWave) + threadIdx.x / kWave, gridDim.x * (kLogits / kWave), plan.logits + token * p.experts);
    lay_row<WIDE>(p, plan, token, blockIdx.x * kLogits + threadIdx.x, gridDim.x * kLogits);
}

// A work-group per row: an expert's rank is the number of those that are preferred to it.  OWN: it takes the logits by itself.
constexpr int kRoute = 1024;
template <bool WIDE, bool OWN>
__global__ __launch_bounds__(kRoute) void experts_route(const dlk_experts_params p, const Plan plan) {
    __shared__ double logits[DLK_EXPERTS_MOST];
    __shared__ int slots[DLK_EXPERTS_TOP_MOST];
    const int64_t token = blockIdx.x;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if constexpr (OWN) {
        lay_row<WIDE>(p, plan, token, threadIdx.x, kRoute);
        take_logits<WIDE>(p, token, wave, kRoute / kWave, logits);
    } else {
        if (static_cast<int>(threadIdx.x) < p.experts) logits[threadIdx.x] = plan.logits[token * p.experts + threadIdx.x];
    }
    __syncthreads();
    for (int first = 0; first < p.experts; first += kRoute / 16) { // 16 lanes an expert
        const int e = first + threadIdx.x / 16;
        int before = 0;
        if (e < p.experts) {
            const double z = logits[e];
            for (int f = threadIdx.x % 16; f < p.experts; f += 16) before += f != e && prefer(logits[f], f, z, e);
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) before += __shfl_xor(before, d);
        if (threadIdx.x % 16 == 0 && e < p.experts && before < p.top) slots[before] = e;
    }
    __syncthreads();
    if (wave != 0) return;
    const double largest = logits[slots[0]];
    const int own = slots[min(lane, p.top - 1)];
    const double mine = lane < p.top ? exp(logits[own] - largest) : 0.0;
    double all = mine;
    if (!p.normalise) {
        all = 0.0;
        for (int e = lane; e < p.experts; e += kWave) all += exp(logits[e] - largest);
    }
    all = wave_sum_f64(all);
    if (lane < p.top) {
        p.chosen[token * p.top + lane] = own;
        plan.pick[token * p.top + lane] = static_cast<uint16_t>(own);
        p.weights[token * p.top + lane] = static_cast<float>(mine / all);
    }
}

// The pairs of expert `e`, in order, to `list`; `counts` is scratch.  Each of the WAVES waves looks through a run of them, twice.
template <int WAVES> __device__ __forceinline__ int collect(const uint16_t* pick, int pairs, int e, uint16_t* list, int* counts) {
    constexpr int THREADS = WAVES * kWave;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int run = ((pairs + THREADS - 1) / THREADS) * kWave, begin = wave * run, end = min(pairs, begin + run);
    int count = 0;
    for (int i = begin + lane; i - lane < end; i += kWave) count += __popcll(__ballot(i < end && pick[i] == e));
    if (lane == 0) counts[wave] = count;
    __syncthreads();
    int at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        at += w < wave ? counts[w] : 0;
        all += counts[w];
    }
    for (int i = begin + lane; i - lane < end; i += kWave) {
        const bool own = i < end && pick[i] == e;
        const uint64_t mask = __ballot(own);
        if (own) list[at + __popcll(mask & ((1ull << lane) - 1))] = static_cast<uint16_t>(i);
        at += __popcll(mask);
    }
    __syncthreads();
    return all;
}

// 16 bytes from any address that an entry may have
typedef u32x4 __attribute__((aligned(2))) LooseWords;
__device__ __forceinline__ u32x4 load_loose(const char* at) { return *reinterpret_cast<const LooseWords*>(at); }

// Lanes l and l ^ 8 change places with half of what they hold (see below).
__device__ __forceinline__ void exchange(u32x4 (&w)[2]) {
    constexpr int kRotate8 = 0x128; // row_ror:8, of 16 lanes
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int a = static_cast<int>(w[0][j]), b = static_cast<int>(w[1][j]);
        w[0][j] = __builtin_amdgcn_update_dpp(a, b, kRotate8, 0xf, 0xc, false);
        w[1][j] = __builtin_amdgcn_update_dpp(b, a, kRotate8, 0xf, 0x3, false);
    }
}

// An entry of a pair: a hidden one as the next product reads it, or an output.
template <bool GATE>
__device__ __forceinline__ void keep(const dlk_experts_params& p, const Plan& plan, int pair, int row, float v, float up) {
    if constexpr (!GATE) plan.partial[static_cast<int64_t>(pair) * p.dim + row] = v;
    else {
        const int unit = p.weights_bf16 ? 8 : 4;
        const bool laid = plan.laid;
        const int64_t line = hidden_line(p.hidden, unit, laid), from = pair * line;
        const auto put = [&](int at, float x) {
            if (plan.whole) reinterpret_cast<float*>(plan.act)[from + at] = x;
            else
#pragma unroll
                for (int part = 0; part < 3; ++part) reinterpret_cast<uint16_t*>(plan.act)[part * p.tokens * p.top * line + from + at] = cut(x);
        };
        put(hidden_place(row, p.hidden, unit, laid), v / (1.0f + expf(-v)) * up);
        const int zero = hidden_zero(row, p.hidden, unit, laid);
        if (zero >= 0) put(zero, 0.0f);
    }
}

// One chosen expert's products with the rows that chose it, which are the columns here, 16 at a time.  16 R rows of its
// matrices (GATE: of gate and up, and silu(gate) * up of both; else of down) are a wave's own, or, SPLIT, 16 a work-group's whose
// waves share the sum's index and join their sums in LDS.  A ring of D steps of 128 bytes a row is on its way from memory.
// A work-group stands for expert blockIdx.y, or, where there are fewer pairs than experts, for the expert of pair blockIdx.y
// if that is its first.
template <bool GATE, bool F32, int PARTS, int R, bool SPLIT, bool LOOSE>
__global__ __launch_bounds__(SPLIT ? 512 : 256) void experts_rows(const dlk_experts_params p, const Plan plan) {
    constexpr int WAVES = SPLIT ? 8 : 4, THREADS = WAVES * kWave, TILES = GATE ? 2 * R : R;
    constexpr int ROOM = 15 / (TILES + PARTS), D = SPLIT || ROOM < 2 ? 2 : ROOM > 4 ? 4 : ROOM;
    constexpr int SIZE = F32 ? 4 : 2, PAD = 20;
    static_assert(!SPLIT || R == 1);
    extern __shared__ uint16_t list[];
    __shared__ int counts[WAVES];
    __shared__ float sums[SPLIT ? WAVES : 1][TILES][16][PAD];
    const int pairs = static_cast<int>(p.tokens) * p.top;
    const bool few = pairs < p.experts;
    const int e = few ? plan.pick[blockIdx.y] : blockIdx.y;

    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, n = lane % 16, g = lane / 16;
    const int width = GATE ? p.dim : p.hidden, height = GATE ? p.hidden : p.dim;
    const uint32_t matrix_row = static_cast<uint32_t>(width) * SIZE, matrix = matrix_row * static_cast<uint32_t>(height);
    const uint32_t row_bytes = LOOSE ? laid_width(width, 16 / SIZE) * SIZE : matrix_row; // of the rows, as they are laid out
    const int first_row = (SPLIT ? blockIdx.x : blockIdx.x * WAVES + wave) * 16 * R;
    const auto resource = [](const void* at, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, bytes, kBufferFlags);
    };
    const auto of_expert = [&](const void* w) { return static_cast<const char*>(w) + static_cast<int64_t>(e) * matrix; };
    const __amdgpu_buffer_rsrc_t w0 = resource(of_expert(GATE ? p.gate : p.down), matrix), w1 = resource(of_expert(GATE ? p.up : p.down), matrix);
    const uint32_t x_rows = GATE ? static_cast<uint32_t>(p.tokens) : static_cast<uint32_t>(pairs), plane = x_rows * row_bytes;
    const __amdgpu_buffer_rsrc_t x = resource(GATE ? (plan.rows ? plan.rows : static_cast<const char*>(p.x)) : plan.act, plane * PARTS);
    uint32_t w_at[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = first_row + 16 * r + 8 * i + n % 8;
            w_at[r][i] = LOOSE ? min(row, height - 1) * matrix_row : row < height ? row * matrix_row : kBeyond;
        }

    const int steps = (static_cast<int>(row_bytes) + 127) / 128, per = SPLIT ? (steps + WAVES - 1) / WAVES : steps;
    const int begin = SPLIT ? wave * per : 0, end = min(steps, begin + per);
    const int turn = static_cast<int>((blockIdx.x * WAVES + wave + blockIdx.y * 5u) * 7u % static_cast<uint32_t>(steps));
    struct Held {
        u32x4 w[TILES][2], x[2][PARTS];
    };
    // (what lies behind a row's end or the wave's run is read as zero, from beyond the buffer)
    const auto of_step = [&](int step) {
        const int turned = SPLIT ? step : step + turn < steps ? step + turn : step + turn - steps;
        return static_cast<uint32_t>(step < end ? turned : steps) * 128;
    };
    const auto load_weights = [&](int step, Held& to) {
        const uint32_t k = of_step(step) + g * 32 + n / 8 * 16;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (LOOSE) {
                    const uint32_t at = w_at[r][i] + min(k, matrix_row - 16);
                    to.w[r][i] = load_loose(of_expert(GATE ? p.gate : p.down) + at);
                    if constexpr (GATE) to.w[R + r][i] = load_loose(of_expert(p.up) + at);
                } else {
                    const uint32_t at = k < row_bytes ? w_at[r][i] + k : kBeyond;
                    to.w[r][i] = __builtin_amdgcn_raw_buffer_load_b128(w0, at, 0, 0);
                    if constexpr (GATE) to.w[R + r][i] = __builtin_amdgcn_raw_buffer_load_b128(w1, at, 0, 0);
                }
            }
    };
    Held ring[D]; // (the weights' on their way while the rows are looked up)
#pragma unroll
    for (int d = 0; d < D; ++d) load_weights(begin + d, ring[d]);
    const int count = collect<WAVES>(plan.pick, pairs, e, list, counts);
    if (few && list[0] != blockIdx.y) return;
    for (int first = 0; first < count; first += 16) {
        const int own = first + n;
        const uint32_t x_at = own < count ? static_cast<uint32_t>(GATE ? list[own] / p.top : list[own]) * row_bytes : kBeyond;
        f32x4 sum[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) sum[i] = 0.0f;
        const auto load_rows = [&](int step, Held& to) {
            const uint32_t k = of_step(step) + g * 32;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int part = 0; part < PARTS; ++part) // (x_at may lie behind the end by itself)
                    to.x[i][part] = __builtin_amdgcn_raw_buffer_load_b128(x, k + 16 * i < row_bytes ? x_at + part * plane + k + 16 * i : kBeyond, 0, 0);
        };
        const auto multiply = [&](Held& of) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) exchange(of.w[i]);
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (F32) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[i] = product(__uint_as_float(of.w[i][h][j]), __uint_as_float(of.x[h][0][j]), sum[i]);
                    } else {
#pragma unroll
                        for (int part = PARTS - 1; part >= 0; --part) sum[i] = product(of.w[i][h], of.x[h][part], sum[i]);
                    }
                }
        };
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (first > 0) load_weights(begin + d, ring[d]);
            load_rows(begin + d, ring[d]);
        }
        for (int step = begin; step < end; step += D)
#pragma unroll
            for (int d = 0; d < D; ++d) {
                multiply(ring[d]);
                load_weights(step + D + d, ring[d]);
                load_rows(step + D + d, ring[d]);
            }
        if constexpr (SPLIT) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) *reinterpret_cast<f32x4*>(&sums[wave][i][n][4 * g]) = sum[i];
            __syncthreads();
            for (int i = threadIdx.x; i < 256; i += THREADS) {
                const int r = i % 16, column = i / 16, row = first_row + r, at = first + column;
                if (row >= height || at >= count) continue;
                float v = 0.0f, up = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    v += sums[w][0][column][r];
                    if constexpr (GATE) up += sums[w][1][column][r];
                }
                keep<GATE>(p, plan, list[at], row, v, up);
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = first_row + 16 * r + 4 * g + j;
                    if (row < height && own < count) keep<GATE>(p, plan, list[own], row, sum[r][j], GATE ? sum[TILES - R + r][j] : 0.0f);
                }
        }
    }
}

// The same for experts that many rows chose: the rows pass through LDS, 128 bytes of up to 16 NT of them at a time, for the
// work-group's waves, which have 16 R rows of the matrices each.  (Read by each wave for itself they took most of the time: of
// 25 rows an expert through 32 experts of 768 x 2048, 58 us to the hidden entries and 57 back, through LDS 45 and 31.)
template <bool GATE, bool F32, int PARTS, int R, int NT, int WAVES, bool LOOSE>
__global__ __launch_bounds__(WAVES * kWave) void experts_blocks(const dlk_experts_params p, const Plan plan) {
    constexpr int THREADS = WAVES * kWave, TILES = GATE ? 2 * R : R, D = TILES > 2 ? 2 : 4;
    constexpr int SIZE = F32 ? 4 : 2, ROWS = 16 * NT, UNITS = PARTS * ROWS * 8, STAGED = (UNITS + THREADS - 1) / THREADS;
    extern __shared__ uint16_t list[];
    __shared__ int counts[WAVES];
    __shared__ u32x4 held[2][UNITS]; // [part][row][8 pieces of 16 bytes, in an order of the row's own]
    const int pairs = static_cast<int>(p.tokens) * p.top, e = blockIdx.y;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, n = lane % 16, g = lane / 16;
    const int width = GATE ? p.dim : p.hidden, height = GATE ? p.hidden : p.dim;
    const uint32_t matrix_row = static_cast<uint32_t>(width) * SIZE, matrix = matrix_row * static_cast<uint32_t>(height);
    const uint32_t row_bytes = LOOSE ? laid_width(width, 16 / SIZE) * SIZE : matrix_row; // of the rows, as they are laid out
    const int first_row = (blockIdx.x * WAVES + wave) * 16 * R;
    const auto resource = [](const void* at, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, bytes, kBufferFlags);
    };
    const auto of_expert = [&](const void* w) { return static_cast<const char*>(w) + static_cast<int64_t>(e) * matrix; };
    const __amdgpu_buffer_rsrc_t w0 = resource(of_expert(GATE ? p.gate : p.down), matrix), w1 = resource(of_expert(GATE ? p.up : p.down), matrix);
    const uint32_t x_rows = GATE ? static_cast<uint32_t>(p.tokens) : static_cast<uint32_t>(pairs), plane = x_rows * row_bytes;
    const __amdgpu_buffer_rsrc_t x = resource(GATE ? (plan.rows ? plan.rows : static_cast<const char*>(p.x)) : plan.act, plane * PARTS);
    uint32_t w_at[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = first_row + 16 * r + 8 * i + n % 8;
            w_at[r][i] = LOOSE ? min(row, height - 1) * matrix_row : row < height ? row * matrix_row : kBeyond;
        }
    const int steps = (static_cast<int>(row_bytes) + 127) / 128;
    const int turn = static_cast<int>((blockIdx.x + blockIdx.y * 5u) * 7u % static_cast<uint32_t>(steps));
    const auto turned = [&](int step) { return static_cast<uint32_t>(step >= steps ? steps : step + turn < steps ? step + turn : step + turn - steps) * 128; };
    struct Weights {
        u32x4 w[TILES][2];
    };
    const auto load = [&](int step, Weights& to) {
        const uint32_t k = turned(step) + g * 32 + n / 8 * 16;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (LOOSE) {
                    const uint32_t at = w_at[r][i] + min(k, matrix_row - 16);
                    to.w[r][i] = load_loose(of_expert(GATE ? p.gate : p.down) + at);
                    if constexpr (GATE) to.w[R + r][i] = load_loose(of_expert(p.up) + at);
                } else {
                    const uint32_t at = k < row_bytes ? w_at[r][i] + k : kBeyond;
                    to.w[r][i] = __builtin_amdgcn_raw_buffer_load_b128(w0, at, 0, 0);
                    if constexpr (GATE) to.w[R + r][i] = __builtin_amdgcn_raw_buffer_load_b128(w1, at, 0, 0);
                }
            }
    };
    Weights ring[D]; // (on its way while the rows are looked up)
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, ring[d]);
    const int count = collect<WAVES>(plan.pick, pairs, e, list, counts);
    for (int first = 0; first < count; first += ROWS) {
        const int blocks = min(NT, (count - first + 15) / 16); // of 16 columns, that hold rows
        uint32_t x_at[STAGED];
#pragma unroll
        for (int i = 0; i < STAGED; ++i) {
            const int unit = threadIdx.x + i * THREADS, row = unit / 8 % ROWS, at = first + row;
            x_at[i] = unit < UNITS && at < count
                          ? static_cast<uint32_t>(GATE ? list[at] / p.top : list[at]) * row_bytes + unit / (8 * ROWS) * plane : kBeyond;
        }
        f32x4 sum[NT][TILES];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < TILES; ++i) sum[t][i] = 0.0f;
        u32x4 coming[STAGED];
        const auto fetch = [&](int step) {
            const uint32_t k = turned(step);
#pragma unroll
            for (int i = 0; i < STAGED; ++i) {
                const uint32_t at = k + threadIdx.x % 8 * 16;
                coming[i] = __builtin_amdgcn_raw_buffer_load_b128(x, at < row_bytes ? x_at[i] + at : kBeyond, 0, 0);
            }
        };
        const auto stage = [&](int buffer) {
#pragma unroll
            for (int i = 0; i < STAGED; ++i) {
                const int unit = threadIdx.x + i * THREADS;
                if (UNITS % THREADS == 0 || unit < UNITS) held[buffer][unit ^ (unit / 8 % 8)] = coming[i];
            }
        };
        const auto multiply = [&](Weights& of, int buffer) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) exchange(of.w[i]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (t >= blocks) break;
                    u32x4 rows[PARTS];
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const int row = part * ROWS + 16 * t + n;
                        rows[part] = held[buffer][row * 8 + ((2 * g + h) ^ (row % 8))];
                    }
#pragma unroll
                    for (int i = 0; i < TILES; ++i) {
                        if constexpr (F32) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                sum[t][i] = product(__uint_as_float(of.w[i][h][j]), __uint_as_float(rows[0][j]), sum[t][i]);
                        } else {
#pragma unroll
                            for (int part = PARTS - 1; part >= 0; --part) sum[t][i] = product(of.w[i][h], rows[part], sum[t][i]);
                        }
                    }
                }
        };
        fetch(0);
        if (first > 0)
#pragma unroll
            for (int d = 0; d < D; ++d) load(d, ring[d]);
        stage(0);
        fetch(1);
        __syncthreads();
        for (int step = 0; step < steps; step += D)
#pragma unroll
            for (int d = 0; d < D; ++d) {
                static_assert(D % 2 == 0, "a buffer for each other step");
                stage((d + 1) % 2);
                fetch(step + d + 2);
                multiply(ring[d], d % 2);
                load(step + D + d, ring[d]);
                __syncthreads();
            }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int at = first + 16 * t + n;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = first_row + 16 * r + 4 * g + j;
                    if (row < height && at < count) keep<GATE>(p, plan, list[at], row, sum[t][r][j], GATE ? sum[t][TILES - R + r][j] : 0.0f);
                }
        }
    }
}

// The hidden entries of single rows (see below): a wave has R of a pair's, and reads their rows of both matrices side by side, x from
// where it lies.  1 row through 8 of 64 bf16 experts of 1024 x 2048: 13.1 us, 5.1 TB/s, where matrix products took 19.8.
template <bool F32, bool X_BF16, bool LOOSE> __global__ __launch_bounds__(256) void experts_hidden_single(const dlk_experts_params p, const Plan plan) {
    constexpr int N = F32 ? 4 : 8, R = 2, U = 4;
    const int lane = threadIdx.x % kWave, pair = blockIdx.y;
    const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * 4 + threadIdx.x / kWave) * R);
    if (row >= p.hidden) return;
    const int pieces = LOOSE ? (p.dim + N - 1) / N : p.dim / N;
    constexpr int SIZE = F32 ? 4 : 2, X_SIZE = X_BF16 ? 2 : 4, WORDS = X_BF16 ? N / 2 : N;
    const char* x = static_cast<const char*>(p.x) + static_cast<int64_t>(pair / p.top) * p.dim * X_SIZE;
    const int64_t matrix = static_cast<int64_t>(plan.pick[pair]) * p.hidden;
    const char* from[2][R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t at = (matrix + min(row + r, p.hidden - 1)) * p.dim * SIZE;
        from[0][r] = static_cast<const char*>(p.gate) + at;
        from[1][r] = static_cast<const char*>(p.up) + at;
    }
    const auto four = [](const char* at) { return LOOSE ? load_loose(at) : *reinterpret_cast<const u32x4*>(at); };
    float sum[2][R] = {};
    for (int first = lane; first < pieces; first += U * kWave) {
        u32x4 w[U][2][R];
        uint32_t held[U][WORDS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(first + u * kWave, pieces - 1), at = LOOSE ? min(i * N, p.dim - N) : i * N;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int r = 0; r < R; ++r) w[u][m][r] = four(from[m][r] + at * SIZE);
            if constexpr (WORDS == 2) {
                typedef u32x2 __attribute__((aligned(2))) Loose;
                const char* own = x + at * X_SIZE;
                const u32x2 a = LOOSE ? *reinterpret_cast<const Loose*>(own) : *reinterpret_cast<const u32x2*>(own);
                held[u][0] = a.x, held[u][1] = a.y;
            } else {
#pragma unroll
                for (int c = 0; c < WORDS / 4; ++c) {
                    const u32x4 a = four(x + at * X_SIZE + 16 * c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) held[u][4 * c + j] = a[j];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (first + u * kWave < pieces)
#pragma unroll
                for (int c = 0; c < N; ++c) {
                    float a = !X_BF16 ? __uint_as_float(held[u][c]) : c % 2 ? bf16_hi(held[u][c / 2]) : bf16_lo(held[u][c / 2]);
                    if (LOOSE && c < (first + u * kWave + 1) * N - p.dim) a = 0.0f; // (the last piece holds what the one before it does)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const u32x4 v = w[u][m][r];
                            sum[m][r] = fmaf(a, F32 ? __uint_as_float(v[c % 4]) : c % 2 ? bf16_hi(v[c / 2]) : bf16_lo(v[c / 2]), sum[m][r]);
                        }
                }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float gate = wave_sum(sum[0][r]), up = wave_sum(sum[1][r]);
        if (lane == 0 && row + r < p.hidden) keep<true>(p, plan, pair, row + r, gate, up);
    }
}

// The outputs of single rows, and their weighted sums with them: a column of a matrix product's sixteen would be all that is used, and
// its partial sums would need another launch.  A wave has R outputs of a row and goes through the chosen experts' entries 16 bytes of a
// matrix a lane, all of them side by side.  (f32 hidden entries, which it reads once for R outputs.)  1 row through 8 of 64 bf16 experts
// of 1024 x 2048: 10.6 us, 3.2 TB/s.
template <bool F32> __global__ __launch_bounds__(256) void experts_down_single(const dlk_experts_params p, const float* act) {
    constexpr int N = F32 ? 4 : 8, R = 2, U = 4;
    const int lane = threadIdx.x % kWave;
    const int64_t token = blockIdx.y;
    const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * 4 + threadIdx.x / kWave) * R);
    if (row >= p.dim) return;
    const int pieces = p.hidden / N, all = p.top * pieces;
    const char* down = static_cast<const char*>(p.down);
    float y[R] = {};
    for (int first = lane; first < all; first += U * kWave) {
        u32x4 w[U][R];
        f32x4 a[U][N / 4];
        float weight[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(first + u * kWave, all - 1), j = i / pieces, at = i % pieces;
            const int64_t pair = token * p.top + j, expert = p.chosen[pair];
            weight[u] = first + u * kWave < all ? p.weights[pair] : 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r)
                w[u][r] = *reinterpret_cast<const u32x4*>(down + ((expert * p.dim + min(row + r, p.dim - 1)) * pieces + at) * 16);
#pragma unroll
            for (int c = 0; c < N / 4; ++c) a[u][c] = *reinterpret_cast<const f32x4*>(act + pair * p.hidden + at * N + 4 * c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < N; ++c) {
                    const float v = F32 ? __uint_as_float(w[u][r][c % 4]) : c % 2 ? bf16_hi(w[u][r][c / 2]) : bf16_lo(w[u][r][c / 2]);
                    sum = fmaf(a[u][c / 4][c % 4], v, sum);
                }
                if (first + u * kWave < all) y[r] = fmaf(weight[u], sum, y[r]);
            }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        y[r] = wave_sum(y[r]);
        if (lane == 0 && row + r < p.dim) p.y[token * p.dim + row + r] = y[r];
    }
}

// The weighted sum of a row's outputs, in the order of its choice.  A thread has N neighbouring entries.
template <int N> __global__ __launch_bounds__(256) void experts_join(const dlk_experts_params p, const float* partial) {
    struct alignas(4 * N) Entries {
        float v[N];
    };
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, units = p.dim / N;
    if (i >= p.tokens * units) return;
    const int64_t token = i / units;
    const Entries* from = reinterpret_cast<const Entries*>(partial) + token * p.top * units + i % units;
    Entries y{};
#pragma unroll 4
    for (int j = 0; j < p.top; ++j) {
        const Entries x = from[j * units];
        const float w = p.weights[token * p.top + j];
#pragma unroll
        for (int c = 0; c < N; ++c) y.v[c] = fmaf(w, x.v[c], y.v[c]);
    }
    reinterpret_cast<Entries*>(p.y)[i] = y;
}

// Any sizes and alignments, entry by entry: a wave per expert and hidden entry, for up to 8 of the rows that chose it at a time.
__global__ __launch_bounds__(256) void experts_hidden_any(const dlk_experts_params p, const Plan plan) {
    constexpr int WAVES = 4, N = 8;
    extern __shared__ uint16_t list[];
    __shared__ int counts[WAVES];
    const int pairs = static_cast<int>(p.tokens) * p.top, e = blockIdx.y;
    const int count = collect<WAVES>(plan.pick, pairs, e, list, counts);
    const int lane = threadIdx.x % kWave, row = blockIdx.x * WAVES + threadIdx.x / kWave;
    if (row >= p.hidden) return;
    const int64_t at = (static_cast<int64_t>(e) * p.hidden + row) * p.dim;
    for (int first = 0; first < count; first += N) {
        float g[N] = {}, h[N] = {};
        int64_t rows[N];
#pragma unroll
        for (int n = 0; n < N; ++n) rows[n] = static_cast<int64_t>(list[min(first + n, count - 1)] / p.top) * p.dim;
#pragma unroll 2
        for (int i = lane; i < p.dim; i += kWave) {
            const float wg = entry(p.gate, p.weights_bf16, at + i), wu = entry(p.up, p.weights_bf16, at + i);
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (first + n < count) {
                    const float x = entry(p.x, p.x_bf16, rows[n] + i);
                    g[n] = fmaf(x, wg, g[n]);
                    h[n] = fmaf(x, wu, h[n]);
                }
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (first + n < count) {
                const float a = wave_sum(g[n]), b = wave_sum(h[n]);
                if (lane == 0) keep<true>(p, plan, list[first + n], row, a, b);
            }
    }
}

// and a wave per row and output entry, the chosen experts in order.
__global__ __launch_bounds__(256) void experts_down_any(const dlk_experts_params p, const float* act) {
    const int lane = threadIdx.x % kWave;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kWave, step = static_cast<int64_t>(gridDim.x) * 256 / kWave;
    for (int64_t u = unit; u < p.tokens * p.dim; u += step) {
        float y = 0.0f;
        for (int j = 0; j < p.top; ++j) {
            const int64_t pair = u / p.dim * p.top + j, row = p.chosen[pair] * p.dim + u % p.dim;
            float sum = 0.0f;
            for (int i = lane; i < p.hidden; i += kWave)
                sum = fmaf(act[pair * p.hidden + i], entry(p.down, p.weights_bf16, row * p.hidden + i), sum);
            y = fmaf(p.weights[pair], wave_sum(sum), y);
        }
        if (lane == 0) p.y[u] = y;
    }
}

bool aligned(const void* at) { return reinterpret_cast<uintptr_t>(at) % 16 == 0; }
bool wide(const dlk_experts_params& p) { return p.dim % 8 == 0 && aligned(p.x) && aligned(p.router); }
// A work-group takes a row's logits by itself unless they are many: 16 rows and 64 experts of 2048 entries 13.9 us, by several
// work-groups 6.7 and 4.7 with the launch behind it (4 rows and 128 experts, the whole call: 102 and 88 us); but 1 row and 16 experts of
// 1024 4.8, or 3.8 and 2.5, and the small call's 24 us become 27.
bool shared_logits(const dlk_experts_params& p) { return static_cast<int64_t>(p.experts) * p.dim >= 1 << 17; }
int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// Each product takes the matrix cores where its rows have a piece of 16 bytes at least, at offsets of 32 bits; loose: where
// its matrices' rows do not begin at multiples of 16 bytes.
// Few rows go one by one through a product where their experts are others or its matrices stay in the last cache (128 MB, each
// row's counted).  Measured on MI355X, us a call with matrix products / outputs one by one / both: 1 row through 8 of 64 experts of 1024 x
// 2048 41 / 38 / 32, 4 rows 79 / 73 / 69, 16 rows through 8 of 128 of them 252 / 244 / 242, 4 rows through 4 of 16 of 704 x 1024 34 / 28 / 21, 8
// rows through 2 of them 34 / 27 / 22, 20 rows through 2 of 8 of 256 x 512 25 / 21 / 21; but 4 rows through 8 of 8 of 1024 x 2048 41 / 38 / 53,
// 16 rows through 8 of 64 of them (537 MB) 150 / 172, 60 rows through 2 of 16 of 704 x 1024 37 / 45.  Of bf16 matrices off their alignment
// a wave's 1024 bytes in a row take one line more, the matrix products' 8 rows of 128 bytes eight: 16 rows through 8 of 64 of 1024 x 2047
// 289 / 227 (first the hidden entries with matrix products, then one by one), 16 rows through 4 of 32 of 704 x 2047 124 / 76, 64 rows through
// 2 of 64 of 1024 x 2047 290 / 222, 8 rows through 8 of 8 of them 114 / 87; but 32 rows through 8 of 64 295 / 371, 64 rows through 2 of 32 of 704 x
// 1023 75 / 87.
bool single_rows(const dlk_experts_params& p, int matrices, bool loose) {
    const int64_t pairs = p.tokens * p.top, bytes = static_cast<int64_t>(p.dim) * p.hidden * (p.weights_bf16 ? 2 : 4) * matrices;
    if (loose && p.weights_bf16) return (p.tokens <= 64 && pairs <= 2 * p.experts) || (p.tokens <= 32 && pairs * bytes <= 1 << 29);
    return p.tokens <= 32 && (pairs <= p.experts || pairs * bytes <= 1 << 27);
}
struct Layout {
    bool gate, down, single_gate, single, loose_gate, loose_down;
    int planes; // of x: parts (bf16 matrices) or 0
    int64_t logits, rows, act, partial, bytes;
};
Layout layout(const dlk_experts_params& p) {
    Layout l{};
    const int64_t pairs = p.tokens * p.top;
    const int unit = p.weights_bf16 ? 8 : 4, size = p.weights_bf16 ? 2 : 4, held = p.weights_bf16 ? 6 : 4;
    const int64_t x_line = laid_width(p.dim, unit), act_line = laid_width(p.hidden, unit);
    const bool fits = std::max(p.tokens * x_line, pairs * act_line) * held <= INT32_MAX && static_cast<int64_t>(p.dim) * p.hidden * size <= INT32_MAX;
    l.gate = fits && p.dim >= unit;
    l.down = fits && p.hidden >= unit;
    l.loose_gate = p.dim % unit != 0 || !aligned(p.gate) || !aligned(p.up);
    l.loose_down = p.hidden % unit != 0 || !aligned(p.down);
    l.single = l.down && !l.loose_down && single_rows(p, 1, false);
    if (l.single) l.down = false;
    // (x as it is where its rows are what the products read; else laid out by the router's kernel)
    l.single_gate = l.gate && single_rows(p, 2, l.loose_gate);
    const bool laid = !l.single_gate && (p.weights_bf16 != p.x_bf16 || p.dim % unit != 0 || !aligned(p.x));
    l.planes = p.weights_bf16 ? (p.x_bf16 ? 1 : 3) : 0;
    l.logits = up16(pairs * 2); // behind the choice
    l.rows = l.logits + (shared_logits(p) ? up16(p.tokens * p.experts * 8) : 0);
    l.act = l.rows + (l.gate && laid ? up16(p.tokens * x_line * held) : 0);
    l.partial = l.act + up16(l.down ? pairs * act_line * held : pairs * p.hidden * 4);
    l.bytes = l.partial + (l.down ? pairs * p.dim * 4 : 0);
    return l;
}

template <bool GATE, bool F32, int PARTS, bool LOOSE> void rows_of(const dlk_experts_params& p, const Plan& plan, hipStream_t at) {
    const int pairs = static_cast<int>(p.tokens) * p.top, height = GATE ? p.hidden : p.dim;
    const int active = std::min(pairs, p.experts), tiles = (height + 15) / 16;
    const auto launch = [&](auto r, auto split) {
        constexpr int R = decltype(r)::value;
        constexpr bool SPLIT = decltype(split)::value;
        const int per = R * (SPLIT ? 1 : 4);
        experts_rows<GATE, F32, PARTS, R, SPLIT, LOOSE><<<dim3((tiles + per - 1) / per, active), SPLIT ? 512 : 256, pairs * 2, at>>>(p, plan);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    const std::true_type split;
    const std::false_type whole;
    const auto blocks = [&](auto r, auto nt, auto waves) {
        constexpr int R = decltype(r)::value, NT = decltype(nt)::value, WAVES = decltype(waves)::value;
        experts_blocks<GATE, F32, PARTS, R, NT, WAVES, LOOSE><<<dim3((tiles + R * WAVES - 1) / (R * WAVES), p.experts), WAVES * kWave, pairs * 2, at>>>(p, plan);
    };
    const integral_constant<int, 8> eight;
    const integral_constant<int, 6> six;
    // What fills the chip: 16 rows of a matrix a work-group whose waves share the sum, until the chosen experts have a tile for each
    // of 1024 waves, and then as many tiles a wave as leave 1024 waves busy, so that what a wave reads of the rows serves more of
    // them.  Measured on MI355X, us a call (both products and the rest), bf16 matrices of 2048 x 1024, by what the gates' product takes,
    // shared / 1 / 2 / 4 tiles a wave: 8 experts (512 tiles) 61 / 67 / 83 / 113; 16 78 / 70 / 85 / 116; 32 117 / 105 / 99 / 129; 64 170 /
    // 159 / 154 / 149.  f32 matrices take twice the registers and one tile: 32 experts 165 / 161 / 165 / 221.
    // Through LDS where all experts are read anyway: 16 rows through 4 of 64 experts of 512 x 1024 58 / 55 / 51 / 68, through LDS 51; through
    // 4 of 32 of 704 x 2048 79 / 87 / 78 / 107 and 67; where many rows share an expert from fewer tiles on: 100 rows through 4 of 16
    // of 704 x 1024 64 shared, 56 through LDS, 30 rows through 2 of them 37 and 40.  Loads off their alignment take longer, less so
    // where each is made once (16 rows through 4 of 32 experts of 704 x 2047: 129 us a call more with four tiles a wave than through LDS), and
    // f32 rows are twice as long (8 rows through 8 of 64 experts of 1024 x 2048: 255 and 237).
    const int64_t all = static_cast<int64_t>(active) * tiles;
    if (all < (pairs >= 8 * p.experts ? 512 : 1024)) launch(one, split);
    else if (pairs < p.experts || (!LOOSE && !F32 && p.tokens <= 16 && all >= 4096)) {
        if constexpr (F32) launch(one, whole);
        else if (all < 2048) launch(one, whole);
        else if (all < 4096) launch(two, whole);
        else launch(four, whole);
    } else {
        // 6, 8 or 16 tiles a work-group, by what the CU with most of them has (us a call by what the gates' product
        // takes: 200 rows through 4 of 32 experts of 768 x 2048, 48 tiles of each, 87 with 6, 90 and 122 with the others; 40 rows through 4 of 64 of
        // 512 x 1024, 32 of each, 66, 53 and 66; 40 rows through 8 of 64 of 1024 x 2048, 64 of each, 181, 168 and 169)
        const auto most = [&](int rows) { return (static_cast<int64_t>(p.experts) * ((tiles + rows - 1) / rows) + 255) / 256 * rows; };
        if (most(6) < most(16) && most(6) < most(8)) blocks(one, four, six);
        else if (most(8) < most(16)) blocks(one, four, eight);
        else blocks(two, four, eight);
    }
}

template <bool GATE, bool F32, int PARTS> void rows_of(const dlk_experts_params& p, const Plan& plan, bool loose, hipStream_t at) {
    if (loose) rows_of<GATE, F32, PARTS, true>(p, plan, at);
    else rows_of<GATE, F32, PARTS, false>(p, plan, at);
}

} // namespace
} // namespace dlk

extern "C" int64_t dlk_experts_rows(const dlk_experts_params* p) {
    // pairs that an expert's list holds, and planes of x and of the hidden entries below 2 GiB
    const int64_t most = std::max<int64_t>(p->dim, p->top * static_cast<int64_t>(p->hidden)) * 12;
    return std::max<int64_t>(1, std::min<int64_t>(dlk::kPairs / p->top, INT32_MAX / most));
}

extern "C" int64_t dlk_experts_workspace(const dlk_experts_params* p) { return dlk::layout(*p).bytes; }

extern "C" int dlk_experts(const dlk_experts_params* p, dlh_stream stream) {
    using namespace dlk;
    if (p->experts <= 0 || p->experts > DLK_EXPERTS_MOST || p->top <= 0 || p->top > p->experts || p->top > DLK_EXPERTS_TOP_MOST ||
        p->dim <= 0 || p->hidden <= 0 || p->tokens <= 0 || p->tokens > dlk_experts_rows(p) || !p->workspace)
        return hipErrorInvalidValue;
    hipStream_t at = reinterpret_cast<hipStream_t>(stream);
    const Layout l = layout(*p);
    char* space = static_cast<char*>(p->workspace);
    const Plan plan{reinterpret_cast<uint16_t*>(space), reinterpret_cast<double*>(space + l.logits), l.act > l.rows ? space + l.rows : nullptr, space + l.act, !l.down || !p->weights_bf16, l.down,
                    reinterpret_cast<float*>(space + l.partial), l.planes};
    const auto tokens = static_cast<unsigned>(p->tokens);
    if (shared_logits(*p)) {
        const dim3 groups((p->experts + kLogitsExperts - 1) / kLogitsExperts, tokens);
        if (wide(*p)) experts_logits<true><<<groups, kLogits, 0, at>>>(*p, plan);
        else experts_logits<false><<<groups, kLogits, 0, at>>>(*p, plan);
        experts_route<true, false><<<tokens, kRoute, 0, at>>>(*p, plan);
    } else if (wide(*p)) experts_route<true, true><<<tokens, kRoute, 0, at>>>(*p, plan);
    else experts_route<false, true><<<tokens, kRoute, 0, at>>>(*p, plan);
    if (l.single_gate) {
        const auto launch = [&](auto f32, auto x_bf16) {
            const dim3 groups((p->hidden + 7) / 8, tokens * p->top);
            if (l.loose_gate || !aligned(p->x)) experts_hidden_single<f32.value, x_bf16.value, true><<<groups, 256, 0, at>>>(*p, plan);
            else experts_hidden_single<f32.value, x_bf16.value, false><<<groups, 256, 0, at>>>(*p, plan);
        };
        const std::true_type yes;
        const std::false_type no;
        if (p->weights_bf16) p->x_bf16 ? launch(no, yes) : launch(no, no);
        else p->x_bf16 ? launch(yes, yes) : launch(yes, no);
    } else if (!l.gate) {
        const dim3 groups((p->hidden + 3) / 4, p->experts);
        const int list = static_cast<int>(p->tokens) * p->top * 2;
        experts_hidden_any<<<groups, 256, list, at>>>(*p, plan);
    } else if (!p->weights_bf16) rows_of<true, true, 1>(*p, plan, l.loose_gate, at);
    else if (p->x_bf16) rows_of<true, false, 1>(*p, plan, l.loose_gate, at);
    else rows_of<true, false, 3>(*p, plan, l.loose_gate, at);
    if (l.single) {
        const dim3 groups((p->dim + 7) / 8, tokens);
        const float* act = reinterpret_cast<const float*>(plan.act);
        if (p->weights_bf16) experts_down_single<false><<<groups, 256, 0, at>>>(*p, act);
        else experts_down_single<true><<<groups, 256, 0, at>>>(*p, act);
        return hipGetLastError();
    }
    if (!l.down) {
        const int64_t waves = p->tokens * p->dim;
        experts_down_any<<<static_cast<unsigned>(std::min<int64_t>(waves / 4 + 1, 16384)), 256, 0, at>>>(*p, reinterpret_cast<const float*>(plan.act));
        return hipGetLastError();
    }
    if (p->weights_bf16) rows_of<false, false, 3>(*p, plan, l.loose_down, at);
    else rows_of<false, true, 1>(*p, plan, l.loose_down, at);
    const int64_t entries = p->tokens * p->dim;
    if (p->dim % 4 == 0 && aligned(p->y)) experts_join<4><<<static_cast<unsigned>((entries / 4 + 255) / 256), 256, 0, at>>>(*p, plan.partial);
    else experts_join<1><<<static_cast<unsigned>((entries + 255) / 256), 256, 0, at>>>(*p, plan.partial);
    return hipGetLastError();
}
