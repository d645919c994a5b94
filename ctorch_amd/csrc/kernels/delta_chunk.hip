// The gated delta rule over prompts, 64 tokens (a chunk) at a time (see dlk_delta_params in kernels.h).
//
// Within a chunk, with G_i the sum of its decays up to token i, b the rates and S the state before it, the writes w_i obey
//   w_i = b_i (v_i - e^G_i S^T k_i - sum_(j < i) e^(G_i - G_j) (k_i . k_j) w_j),
// a triangular system whose matrix 1 + A, A_ij = b_i e^(G_i - G_j) (k_i . k_j), knows nothing of the states.  So a first launch takes
// T = (1 + A)^-1 and P_ij = e^(G_i - G_j) (q_i . k_j), j <= i, of all chunks at once, and a second goes through each request's
// chunks in order with what is left, for 16 columns of the state a work-group (columns know nothing of one another):
//   R = b (V - e^G K S);   W = T R;   out = scale (e^G Q S + P W);   S = e^G_64 S + K^T (e^(G_64 - G) W)
//
// All exact to f32.  bf16 queries and keys go into the matrix cores as they are, what else is a factor there (S, R, W, T, P, f32
// queries and keys) as three bf16 parts that hold all 24 bits; of a product of two such, the three smallest of nine part
// products are left out, below 2^-24 of it.  Sums of decays are of 64 bits, since differences of long sums are taken.  (The
// f32 instruction would take 2.7 times as long as six bf16 ones.)
//
// What is not finite stays behind its token: a matrix product would take it to the tokens before as well, by way of the zeros behind a
// triangle.  So entries of the products' right factors that are not finite (R, W, and in the inverse A) go in as zeros, and the
// tokens' outputs from the first of them on, and the state, become NaN.  (1 to 2 % of a prompt's time.)
//
// A bf16 prompt of 8191 tokens through 32 heads of 128 x 128 takes 70 us in the first launch and 304 in the second; 6 f32 ones of 6725
// in all through 16 heads of 64 x 128 45 and 158.
#include "kernels/parts.h"

#include <algorithm>

namespace dlk {
namespace {

constexpr int kThreads = 256, kWaves = 4, kTile = 256, kTiles = 10; // 16 x 16 tiles on and below the diagonal of 64 x 64
__device__ __forceinline__ int tile_of(int i, int j) { return i * (i + 1) / 2 + j; }

// the compiler keeps LDS accesses of a wave in order across this (the hardware does by itself)
__device__ __forceinline__ void wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// The entries of a row as PARTS bf16 parts (one: they are bf16; three: f32).
template <int PARTS> __device__ __forceinline__ void eight_of(const dlk_row_segment& s, int64_t at, u32x4 (&to)[PARTS]) {
    if constexpr (PARTS == 1) {
        to[0] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(s.x) + at);
    } else {
        float v[8];
        const f32x4* from = reinterpret_cast<const f32x4*>(static_cast<const float*>(s.x) + at);
        const f32x4 a = from[0], b = from[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
#pragma unroll
        for (int part = 0; part < PARTS; ++part) to[part] = cut(v);
    }
}

__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) <= 3.4028234664e38f); }
// x, or, where it is not finite, zero; `first` goes down to `row` then.
__device__ __forceinline__ float finite_of(float x, int row, int& first) {
    const bool bad = not_finite(x);
    first = bad ? min(first, row) : first;
    return bad ? 0.0f : x;
}

// sum + a b, the smallest part products first
template <int A, int B> __device__ __forceinline__ f32x4 multiply(const u32x4 (&a)[A], const u32x4 (&b)[B], f32x4 sum) {
    constexpr int LAST = (A > B ? A : B) - 1;
#pragma unroll
    for (int order = LAST; order >= 0; --order)
#pragma unroll
        for (int i = 0; i < A; ++i)
            if (order - i >= 0 && order - i < B) sum = product(a[i], b[order - i], sum);
    return sum;
}

// ------------------------------------------------------------------------------------------------ the chunks by themselves
// A work-group per chunk and key head; wave w has the chunk's tokens 16 w to 16 w + 15 as rows.
template <int DK, int PARTS> __global__ __launch_bounds__(kThreads, 3) void delta_prepare(const dlk_delta_params p) {
    constexpr int STEPS = DK / 32, LINE = 64 + 8, WIDE = 64 + 4;
    __shared__ union {
        uint16_t turned[DK][LINE];
        struct {
            float system[64][WIDE], inverse[4][16][20];
        };
    } room; // (first the one, then the other)
    auto& turned = room.turned;
    auto& system = room.system;
    auto& inverse = room.inverse;
    __shared__ double reach[kWaves][64];
    __shared__ int first_bad[2]; // the first token whose row of A is not finite (of every other head)
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, n = lane % 16, g = lane / 16;
    const int key_heads = p.heads / p.group, key_head = blockIdx.x % key_heads;
    const int64_t index = blockIdx.x / key_heads;
    dlk_delta_chunk chunk = p.chunks[index];
    chunk.token = __builtin_amdgcn_readfirstlane(chunk.token), chunk.count = __builtin_amdgcn_readfirstlane(chunk.count);
    const int64_t place = index * key_heads + key_head;

    u32x4 k[STEPS][PARTS], q[STEPS][PARTS];
    {
        const int row = 16 * wave + n;
        const int64_t token = chunk.token + min(row, chunk.count - 1);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            eight_of<PARTS>(p.k, token * p.k.row + key_head * p.k.head + 32 * s + 8 * g, k[s]);
            eight_of<PARTS>(p.q, token * p.q.row + key_head * p.q.head + 32 * s + 8 * g, q[s]);
            if (row >= chunk.count)
#pragma unroll
                for (int part = 0; part < PARTS; ++part) k[s][part] = 0, q[s][part] = 0;
        }
    }
    // for the second launch: keys with the tokens side by side, and the parts of f32 ones
    const int64_t plane = static_cast<int64_t>(p.chunk_count) * key_heads * 64 * DK;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
        if constexpr (PARTS > 1)
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int64_t at = part * plane + (place * 64 + 16 * wave + n) * DK + 32 * s + 8 * g;
                *reinterpret_cast<u32x4*>(p.key_parts + at) = k[s][part];
                *reinterpret_cast<u32x4*>(p.query_parts + at) = q[s][part];
            }
        if (part > 0) __syncthreads();
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                turned[32 * s + 8 * g + i][16 * wave + n] = static_cast<uint16_t>(i % 2 ? k[s][part][i / 2] >> 16 : k[s][part][i / 2]);
        __syncthreads();
        for (int i = threadIdx.x; i < DK * 8; i += kThreads)
            *reinterpret_cast<u32x4*>(p.turned_keys + part * plane + (place * DK + i / 8) * 64 + i % 8 * 8) =
                *reinterpret_cast<const u32x4*>(&turned[i / 8][i % 8 * 8]);
    }
    f32x4 kk[4], qk[4]; // row 16 wave + 4 g + r, column 16 j + n
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk[j] = 0.0f, qk[j] = 0.0f;
        if (j > wave) continue;
        const int row = 16 * j + n;
        const int64_t token = chunk.token + min(row, chunk.count - 1);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            u32x4 column[PARTS];
            eight_of<PARTS>(p.k, token * p.k.row + key_head * p.k.head + 32 * s + 8 * g, column);
            kk[j] = multiply(k[s], column, kk[j]);
            qk[j] = multiply(q[s], column, qk[j]);
        }
    }
    if (threadIdx.x == 0) first_bad[0] = 64;
    __syncthreads();
    for (int h = 0; h < p.group; ++h) {
        const int head = key_head * p.group + h;
        const int64_t own = index * p.heads + head;
        // lane i: token i
        const int64_t gate = (chunk.token + min(lane, chunk.count - 1)) * p.heads + head;
        const float decay = p.decay[gate], rate = lane < chunk.count ? p.rate[gate] : 0.0f;
        // (e^-1000 is 0; sums with -inf would have no differences)
        double sum = lane >= chunk.count ? 0.0 : decay < -1000.0f ? -1000.0 : static_cast<double>(decay);
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double before = __shfl_up(sum, d);
            if (lane >= d) sum += before;
        }
        reach[wave][lane] = sum;
        wave_order();
        if (wave == 0) {
            float* to = p.gates + own * 192;
            to[lane] = expf(static_cast<float>(sum));
            to[64 + lane] = expf(static_cast<float>(reach[0][63] - sum));
            to[128 + lane] = rate;
        }
        int bad = 64; // of the rows that this lane has entries of, the first that is not finite, from 16 wave + 4 g on
        float* within = p.within + own * kTiles * kTile;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > wave) continue;
            const double to = reach[wave][16 * j + n];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * wave + 4 * g + r, at = 16 * j + n;
                const float fade = expf(static_cast<float>(reach[wave][i] - to)), factor = __shfl(rate, i) * fade;
                system[i][at] = finite_of(i > at ? factor * kk[j][r] : 0.0f, r, bad);
                within[tile_of(wave, j) * kTile + (4 * g + r) * 16 + n] = i >= at && at < chunk.count ? fade * qk[j][r] : 0.0f;
            }
        }
        if (threadIdx.x == 0) first_bad[(h + 1) % 2] = 64;
        __syncthreads();
        // The inverse of each diagonal tile by substitution, a column a lane (four times over),
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            f32x4 row[4];
#pragma unroll
            for (int j = 0; j < (i + 3) / 4; ++j) row[j] = *reinterpret_cast<const f32x4*>(&system[16 * wave + i][16 * wave + 4 * j]);
            x[i] = i == n ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; ++j) x[i] = fmaf(-row[j / 4][j % 4], x[j], x[i]);
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0); // (all rows read at once would take the registers of another wave)
        }
        f32x4 solved[4]; // [tile row]: rows 4 g + r, column n
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float own_row = g == 0 ? x[r] : g == 1 ? x[4 + r] : g == 2 ? x[8 + r] : x[12 + r];
            solved[0][r] = own_row;
            inverse[wave][4 * g + r][n] = own_row;
        }
        __syncthreads();
        // and the tiles below it, in order: X_ij = -X_ii sum_(j <= k < i) A_ik X_kj; wave j has column j of tiles.
        // (A result's lane layout is that of the next product's right factor, if its index runs over 4 g + r.)
#pragma unroll
        for (int step = 0; step < 4; ++step) {
            const int i = wave + step;
            if (i > 3) break;
            if (step > 0) {
                f32x4 below = 0.0f;
#pragma unroll
                for (int t = 0; t < step; ++t) {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(&system[16 * i + n][16 * (wave + t) + 4 * g]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) below = product(a[r], solved[t][r], below);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) below[r] = finite_of(below[r], 16 * step + r, bad);
                const f32x4 a = *reinterpret_cast<const f32x4*>(&inverse[i][n][4 * g]);
                solved[step] = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) solved[step] = product(a[r], -below[r], solved[step]);
            }
        }
        if (bad < 64) atomicMin(&first_bad[h % 2], 16 * wave + 4 * g + bad);
        __syncthreads();
#pragma unroll
        for (int step = 0; step < 4; ++step)
            if (wave + step < 4)
#pragma unroll
                for (int r = 0; r < 4; ++r) system[16 * (wave + step) + 4 * g + r][16 * wave + n] = solved[step][r];
        __syncthreads();
        if (wave == 0 && lane >= first_bad[h % 2]) p.gates[own * 192 + lane] = __builtin_nanf("");
        // in parts, 8 entries a thread
        uint16_t* solution = p.solution + own * 3 * kTiles * kTile;
        for (int i = threadIdx.x; i < kTiles * 32; i += kThreads) {
            const int tile = i / 32, row = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, column = tile - tile_of(row, 0);
            const f32x4* from = reinterpret_cast<const f32x4*>(&system[16 * row + i / 2 % 16][16 * column + i % 2 * 8]);
            const f32x4 a = from[0], b = from[1];
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
#pragma unroll
            for (int part = 0; part < 3; ++part) *reinterpret_cast<u32x4*>(solution + part * kTiles * kTile + i * 8) = cut(v);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ chunk after chunk
// A work-group per request, head and 16 columns of the state.  What counts is how long a chunk takes, not how much there is to
// do: a prompt's chunks follow one another, and a chunk's three products wait for each other at three barriers, 2.4 us of 128 x 128 (the
// products alone, at the matrix cores' rate, 0.7).  So the waves share it by what waits for what: waves 0 to 3 hold the state (DK / 4
// rows each; of 32: waves 0 and 1, 16 each) and take it to the next chunk by way of R and W, 16 tokens each, and waves 4 to 7 make
// the outputs of 16 tokens each beside them.  What the next chunk's products read is asked for as soon as this one's have used theirs
// (and not before: its registers are the same).  32 columns a work-group would halve the reads of keys and queries, but leave half of the
// CUs idle where one prompt of 32 heads is all there is.
template <int DK, int PARTS, bool V_BF16>
__global__ __launch_bounds__(2 * kThreads) __attribute__((amdgpu_waves_per_eu(2, PARTS == 1 && DK < 128 ? 4 : 2))) void delta_scan(const dlk_delta_params p) {
    constexpr int STEPS = DK / 32, OWN = DK > 64 ? DK / 64 : 1, LINE_S = DK + 8, LINE = 64 + 8;
    __shared__ uint16_t state_parts[3][16][LINE_S], right[3][16][LINE], write[3][16][LINE], late[3][16][LINE];
    __shared__ float gates[2][192];
    __shared__ int first_bad[16]; // of a column, the first token whose write is not finite (since then of every chunk: the state is not)
    const int lane = threadIdx.x % kWave, n = lane % 16, g = lane / 16;
    const int role = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wave = role % kWaves;
    // (work-groups go to the 8 dies in turn; the slices of a head read the same chunks, from the cache of one of them)
    const int slices = p.value_dim / 16, pairs = p.item_count * p.heads;
    const int pair = static_cast<int>(blockIdx.x / (8 * slices) * 8 + blockIdx.x % 8);
    if (pair >= pairs) return;
    const auto shared = [](int x) { return __builtin_amdgcn_readfirstlane(x); }; // (by the whole wave, which the compiler cannot know)
    const int first_column = shared(blockIdx.x / 8 % slices) * 16, head = shared(pair % p.heads), key_head = shared(head / p.group);
    const int key_heads = shared(p.heads / p.group);
    dlk_delta_item item = p.items[shared(pair / p.heads)];
    item = {shared(item.source), shared(item.target), shared(item.token), shared(item.count), shared(item.chunk), 0};
    const int chunks = (item.count + 63) / 64;
    const auto tokens_of = [&](int c) { return min(64, item.count - 64 * c); };
    const int64_t plane = static_cast<int64_t>(p.chunk_count) * key_heads * 64 * DK;
    // the places of chunk c: of its key head, and of its head
    const auto key_place = [&](int c) { return static_cast<int64_t>(item.chunk + c) * key_heads + key_head; };
    const auto place = [&](int c) { return static_cast<int64_t>(item.chunk + c) * p.heads + head; };
    const auto column_parts = [&](const uint16_t* from, int line, u32x4 (&to)[3]) {
#pragma unroll
        for (int part = 0; part < 3; ++part) to[part] = *reinterpret_cast<const u32x4*>(from + part * 16 * line);
    };
    // Offsets of a lane are the same for all chunks but the last, which may end early: reads behind it take its last row.
    // (32 bits behind an address that the whole wave shares; a 64-bit product a lane takes as long as a dozen other instructions.)
    const int last_row = tokens_of(chunks - 1) - 1;
    const auto at_row = [&](int row, int64_t stride, int c) {
        return static_cast<uint32_t>(c + 1 < chunks ? row : min(row, last_row)) * static_cast<uint32_t>(stride);
    };
    // rows 16 wave + n of the chunk's keys or queries, entries 32 s + 8 g to + 7
    const auto load_rows = [&](const dlk_row_segment& rows, const uint16_t* parts, int c, u32x4 (&to)[STEPS][PARTS]) {
        if constexpr (PARTS == 1) {
            const uint16_t* from = static_cast<const uint16_t*>(rows.x) + (item.token + 64 * static_cast<int64_t>(c)) * rows.row + key_head * rows.head;
            const uint32_t at = at_row(16 * wave + n, rows.row, c) + 8 * g;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) to[s][0] = *reinterpret_cast<const u32x4*>(from + at + 32 * s);
        } else {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint16_t* from = parts + part * plane + key_place(c) * 64 * DK;
                const uint32_t at = static_cast<uint32_t>((16 * wave + n) * DK + 8 * g);
#pragma unroll
                for (int s = 0; s < STEPS; ++s) to[s][part] = *reinterpret_cast<const u32x4*>(from + at + 32 * s);
            }
        }
    };
    // Those rows times the state's columns, all read from LDS before the first product; two sums, since products that follow
    // one another wait for each other.
    const auto times_state = [&](const u32x4 (&rows)[STEPS][PARTS]) {
        u32x4 b[STEPS][3];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) column_parts(&state_parts[0][n][32 * s + 8 * g], LINE_S, b[s]);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < STEPS; s += 2)
#pragma unroll
            for (int order = 2; order >= 0; --order)
#pragma unroll
                for (int i = 0; i < PARTS && i <= order; ++i)
#pragma unroll
                    for (int t = 0; t < 2 && s + t < STEPS; ++t) sum[t] = product(rows[s + t][i], b[s + t][order - i], sum[t]);
        return sum[0] + sum[1];
    };
    // tiles of a triangle: what lies behind it is read as zero, from beyond the buffer
    const auto tiles_at = [&](const void* at, int bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, kTiles * kTile * bytes, kBufferFlags);
    };
    const auto tile_offset = [&](int s, int size) {
        const int tile = 2 * s + g / 2;
        return tile > wave ? 1u << 30 : static_cast<uint32_t>((tile_of(wave, tile) * kTile + n * 16 + g % 2 * 8) * size);
    };
    // rows of a triangle, parts [2 steps of 32 columns], times columns in LDS
    const auto triangle = [&](const u32x4 (&rows)[2][3], const uint16_t (&columns)[3][16][LINE], f32x4 sum) {
        f32x4 small = 0.0f;
        u32x4 b[2][3];
#pragma unroll
        for (int s = 0; s < 2; ++s) column_parts(&columns[0][n][32 * s + 8 * g], LINE, b[s]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (2 * s > wave) break;
            small = product(rows[s][2], b[s][0], small);
            sum = product(rows[s][1], b[s][0], sum);
            small = product(rows[s][1], b[s][1], small);
            sum = product(rows[s][0], b[s][1], sum);
            small = product(rows[s][0], b[s][2], small);
            sum = product(rows[s][0], b[s][0], sum);
        }
        return sum + small;
    };

    if (role >= kWaves) {
        u32x4 q[STEPS][PARTS];
        float coming[3];       // (wave 0) the next chunk's gates
        f32x4 within[2][2];    // rows 16 wave + n, columns 32 s + 8 g to + 7; behind the triangle: zeros
        const int out_row = p.heads * p.value_dim;
        const auto load_gates = [&](int c) {
#pragma unroll
            for (int i = 0; i < 3; ++i) coming[i] = (p.gates + place(c) * 192)[static_cast<uint32_t>(64 * i + lane)];
        };
        const auto keep_gates = [&](int c) {
            if (wave == 0)
#pragma unroll
                for (int i = 0; i < 3; ++i) gates[c % 2][64 * i + lane] = coming[i];
        };
        const auto load_within = [&](int c) {
            const __amdgpu_buffer_rsrc_t from = tiles_at(p.within + place(c) * kTiles * kTile, 4);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    within[s][i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, tile_offset(s, 4) + 16 * i, 0, 0));
        };
        load_gates(0);
        load_rows(p.q, p.query_parts, 0, q);
        load_within(0);
        keep_gates(0);
        if (role == kWaves && lane < 16) first_bad[lane] = 64;
        load_gates(min(1, chunks - 1));
        __syncthreads();
        for (int c = 0; c < chunks; ++c) {
            const int next = min(c + 1, chunks - 1), tokens = tokens_of(c);
            f32x4 out = times_state(q) * *reinterpret_cast<const f32x4*>(&gates[c % 2][16 * wave + 4 * g]);
            __builtin_amdgcn_sched_barrier(0);
            load_rows(p.q, p.query_parts, next, q);
            keep_gates(c + 1);
            __builtin_amdgcn_sched_barrier(0);
            load_gates(min(c + 2, chunks - 1));
            __syncthreads();
            u32x4 rows[2][3];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float a[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = within[s][i / 4][i % 4];
#pragma unroll
                for (int part = 0; part < 3; ++part) rows[s][part] = cut(a);
            }
            __builtin_amdgcn_sched_barrier(0);
            load_within(next);
            __syncthreads();
            const int bad = first_bad[n];
            out = triangle(rows, write, out) * p.scale;
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = 16 * wave + 4 * g + i < bad ? out[i] : __builtin_nanf("");
            // Rows behind the chunk's end lie behind the buffer's.  (Of stores under a condition the compiler could not tell how
            // many came before a load, and would wait for them all.)
            float* to = p.out + ((item.token + 64 * static_cast<int64_t>(c)) * p.heads + head) * p.value_dim + first_column;
            const __amdgpu_buffer_rsrc_t rows_out = __builtin_amdgcn_make_buffer_rsrc(to, 0, ((tokens - 1) * out_row + 16) * 4, kBufferFlags);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(out[i]), rows_out, ((16 * wave + 4 * g + i) * out_row + n) * 4, 0, 0);
            __syncthreads();
        }
        return;
    }

    const bool holds = 16 * OWN * kWaves <= DK || 16 * OWN * wave < DK;
    f32x4 state[OWN]; // rows 16 (OWN wave + t) + 4 g + r
    const auto row_of = [&](int t, int r) { return 16 * (OWN * wave + t) + 4 * g + r; };
    const auto state_at = [&](int slot) {
        return p.states + (static_cast<int64_t>(slot) * p.heads + head) * DK * p.value_dim + first_column;
    };
#pragma unroll
    for (int t = 0; t < OWN; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) state[t][r] = holds && item.source >= 0 ? state_at(item.source)[row_of(t, r) * p.value_dim + n] : 0.0f;
    // four neighbouring rows of a column, in parts
    const auto part4 = [&](f32x4 v, uint16_t* to, int line) {
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            uint32_t w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w[r] = __float_as_uint(v[r]);
                v[r] -= __uint_as_float(w[r] & 0xffff0000u);
            }
            *reinterpret_cast<u32x2*>(to + part * 16 * line) =
                u32x2{__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), __builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
        }
    };
    const auto keep_state = [&] {
        if (holds)
#pragma unroll
            for (int t = 0; t < OWN; ++t) part4(state[t], &state_parts[0][n][row_of(t, 0)], LINE_S);
    };
    // entries of four neighbouring tokens' rows, zero where they are not finite
    const auto finite_rows = [&](f32x4 v) {
        if (not_finite(v[0]) || not_finite(v[1]) || not_finite(v[2]) || not_finite(v[3]))
#pragma unroll
            for (int i = 3; i >= 0; --i)
                if (not_finite(v[i])) {
                    atomicMin(&first_bad[n], 16 * wave + 4 * g + i);
                    v[i] = 0.0f;
                }
        return v;
    };
    u32x4 k[STEPS][PARTS], keys[OWN][2][PARTS], solution[2][3];
    uint32_t v[4]; // as they lie in memory
    const auto load_values = [&](int c) {
        const int64_t from = (item.token + 64 * static_cast<int64_t>(c)) * p.v.row + head * p.v.head + first_column;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t at = at_row(16 * wave + 4 * g + r, p.v.row, c) + n;
            if constexpr (V_BF16) v[r] = (static_cast<const uint16_t*>(p.v.x) + from)[at];
            else v[r] = (static_cast<const uint32_t*>(p.v.x) + from)[at];
        }
    };
    const auto load_solution = [&](int c) { // row 16 wave + n, columns 32 s + 8 g to + 7; behind the triangle: zeros
        const __amdgpu_buffer_rsrc_t from = tiles_at(p.solution + place(c) * 3 * kTiles * kTile, 6);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int part = 0; part < 3; ++part)
                solution[s][part] = __builtin_amdgcn_raw_buffer_load_b128(from, tile_offset(s, 2) + part * kTiles * kTile * 2, 0, 0);
    };
    const auto load_keys = [&](int c) {
        if (holds)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint16_t* from = p.turned_keys + part * plane + key_place(c) * DK * 64;
                const uint32_t at = static_cast<uint32_t>((16 * OWN * wave + n) * 64 + 8 * g);
#pragma unroll
                for (int t = 0; t < OWN; ++t)
#pragma unroll
                    for (int s = 0; s < 2; ++s) keys[t][s][part] = *reinterpret_cast<const u32x4*>(from + at + 16 * t * 64 + 32 * s);
            }
    };

    load_rows(p.k, p.key_parts, 0, k);
    load_values(0);
    load_solution(0);
    load_keys(0);
    keep_state();
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
        const int next = min(c + 1, chunks - 1), tokens = tokens_of(c);
        const float* own = &gates[c % 2][16 * wave + 4 * g];
        const f32x4 since = *reinterpret_cast<const f32x4*>(own), left = *reinterpret_cast<const f32x4*>(own + 64), rate = *reinterpret_cast<const f32x4*>(own + 128);
        const float whole = gates[c % 2][63];
        const f32x4 ks = times_state(k);
        __builtin_amdgcn_sched_barrier(0);
        load_rows(p.k, p.key_parts, next, k);
        f32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = 16 * wave + 4 * g + i < tokens ? rate[i] * (__uint_as_float(V_BF16 ? v[i] << 16 : v[i]) - since[i] * ks[i]) : 0.0f;
        part4(finite_rows(r), &right[0][n][16 * wave + 4 * g], LINE);
        __syncthreads();
        const f32x4 w = finite_rows(triangle(solution, right, f32x4{0.0f, 0.0f, 0.0f, 0.0f}));
        __builtin_amdgcn_sched_barrier(0);
        load_solution(next);
        part4(w * left, &late[0][n][16 * wave + 4 * g], LINE);
        part4(w, &write[0][n][16 * wave + 4 * g], LINE);
#pragma unroll
        for (int t = 0; t < OWN; ++t) state[t] *= whole;
        __builtin_amdgcn_sched_barrier(0);
        load_values(next);
        __syncthreads();
        if (holds) {
            u32x4 b[2][3];
#pragma unroll
            for (int s = 0; s < 2; ++s) column_parts(&late[0][n][32 * s + 8 * g], LINE, b[s]);
            const bool bad = first_bad[n] < 64;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int order = 2; order >= 0; --order)
#pragma unroll
                    for (int i = 0; i < PARTS && i <= order; ++i)
#pragma unroll
                        for (int t = 0; t < OWN; ++t) state[t] = product(keys[t][s][i], b[s][order - i], state[t]);
            if (bad)
#pragma unroll
                for (int t = 0; t < OWN; ++t) state[t] = __builtin_nanf("");
        }
        __builtin_amdgcn_sched_barrier(0);
        load_keys(next);
        keep_state();
        __syncthreads();
    }
    if (holds)
#pragma unroll
        for (int t = 0; t < OWN; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) state_at(item.target)[row_of(t, r) * p.value_dim + n] = state[t][r];
}

template <int DK, int PARTS> void launch(const dlk_delta_params& p, hipStream_t at) {
    const int slices = p.value_dim / 16;
    delta_prepare<DK, PARTS><<<static_cast<unsigned>(p.chunk_count) * (p.heads / p.group), kThreads, 0, at>>>(p);
    const unsigned groups = (static_cast<unsigned>(p.item_count) * p.heads + 7) / 8 * 8 * slices;
    if (p.v.bf16) delta_scan<DK, PARTS, true><<<groups, 2 * kThreads, 0, at>>>(p);
    else delta_scan<DK, PARTS, false><<<groups, 2 * kThreads, 0, at>>>(p);
}

int parts_of(const dlk_delta_params* p) { return p->k.bf16 ? 1 : 3; }

struct Layout {
    int64_t solution, within, gates, turned, keys, queries, bytes;
};
Layout layout(const dlk_delta_params* p) {
    Layout l{};
    const int64_t heads = static_cast<int64_t>(p->chunk_count) * p->heads, parts = parts_of(p);
    const int64_t rows = static_cast<int64_t>(p->chunk_count) * (p->heads / p->group) * 64 * p->key_dim * parts * 2;
    l.within = heads * 3 * kTiles * kTile * 2;
    l.gates = l.within + heads * kTiles * kTile * 4;
    l.turned = l.gates + heads * 192 * 4;
    l.keys = l.turned + rows;
    l.queries = l.keys + (parts > 1 ? rows : 0);
    l.bytes = l.queries + (parts > 1 ? rows : 0);
    return l;
}

} // namespace
} // namespace dlk

extern "C" int64_t dlk_delta_workspace(const dlk_delta_params* p) { return dlk::layout(p).bytes; }

extern "C" int dlk_delta_chunks(const dlk_delta_params* given, void* workspace, dlh_stream stream) {
    using namespace dlk;
    dlk_delta_params p = *given;
    if (p.item_count <= 0 || p.chunk_count <= 0) return 0;
    const int64_t prepared = static_cast<int64_t>(p.chunk_count) * (p.heads / p.group);
    const int64_t scanned = (static_cast<int64_t>(p.item_count) * p.heads + 7) / 8 * 8 * (p.value_dim / 16);
    if (p.value_dim <= 0 || p.value_dim % 16 != 0 || p.group <= 0 || prepared > DLK_MOST_GROUPS || 2 * scanned > DLK_MOST_GROUPS || !workspace ||
        p.q.bf16 != p.k.bf16)
        return hipErrorInvalidValue;
    const Layout l = layout(&p);
    char* at = static_cast<char*>(workspace);
    p.solution = reinterpret_cast<uint16_t*>(at);
    p.within = reinterpret_cast<float*>(at + l.within);
    p.gates = reinterpret_cast<float*>(at + l.gates);
    p.turned_keys = reinterpret_cast<uint16_t*>(at + l.turned);
    p.key_parts = reinterpret_cast<uint16_t*>(at + l.keys);
    p.query_parts = reinterpret_cast<uint16_t*>(at + l.queries);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const bool bf16 = parts_of(&p) == 1;
    switch (p.key_dim) {
    case 32: bf16 ? launch<32, 1>(p, s) : launch<32, 3>(p, s); break;
    case 64: bf16 ? launch<64, 1>(p, s) : launch<64, 3>(p, s); break;
    case 128: bf16 ? launch<128, 1>(p, s) : launch<128, 3>(p, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
