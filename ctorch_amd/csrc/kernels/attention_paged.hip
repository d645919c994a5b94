// Attention over the pages of a paged cache (see dlk_paged_params in kernels.h): each row of a run of tokens over the
// keys up to its own position, o = sum_j softmax_j(q k_j / sqrt(hd)) v_j, the keys found through the run's page table.
// f32 or bf16 pages, head size 16, 32, 64 or 128, page sizes that are powers of two from 16.
//
// A work-group takes an item, up to 16 NT rows (token r / G, query head r % G of the KV head's group) over a range of
// keys, for one KV head; its four waves split the range, stream it in tiles of 32 keys from memory into registers and keep
// their own online softmax (base 2, log2 e folded into the query's scale), and merge in LDS.  Per tile and 16 rows:
//   S^T[16 keys][16 rows] = K[16][hd] Q[16][hd]^T    (v_mfma_f32_16x16x32_bf16, A = 16 key rows as they are stored)
//   O^T[16 d][16 rows]   += V^T[16 d][32 keys] P^T   (A = V^T, transposed through the wave's own LDS tile)
// so a lane holds the scores of one row, and they are the B operand of the second product as they come.  Queries and
// probabilities are split into bf16 hi + lo (and f32 keys and values too), which keeps f32 accuracy: two products for
// bf16 pages, three for f32 ones (the lo * lo term is below 2^-16 of the product).  Row sums come out of one more product
// whose A operand is all ones.  A tile of 32 keys is two halves of 16, each in one page; keys past the range read as zero
// from the buffer range and are masked, so that what a page holds behind the sequence never counts, not even a NaN.
// An item that is all its rows see writes the output, the others (o, max, sum) partials that paged_merge joins.
#include "kernels/device_common.h"

namespace dlk {
namespace {

constexpr int kTileKeys = 32, kWaves = 4, kThreads = kWaves * kWave;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// bf16 hi and lo parts of eight f32 values (x = hi + lo to 2^-16; x - hi is exact in f32)
__device__ __forceinline__ void split8(const f32x8 v, bf16x8& hi, bf16x8& lo) {
    const u32x4 h = __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8));
    const f32x8 back = {__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u),
                        __uint_as_float(h.y << 16), __uint_as_float(h.y & 0xffff0000u),
                        __uint_as_float(h.z << 16), __uint_as_float(h.z & 0xffff0000u),
                        __uint_as_float(h.w << 16), __uint_as_float(h.w & 0xffff0000u)};
    hi = __builtin_bit_cast(bf16x8, h);
    lo = __builtin_convertvector(v - back, bf16x8);
}

__device__ __forceinline__ void split4(const u32x4 w, u32x2& hi, u32x2& lo) {
    const f32x4 v = __builtin_bit_cast(f32x4, w);
    const u32x2 h = __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4));
    const f32x4 back = {__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u),
                        __uint_as_float(h.y << 16), __uint_as_float(h.y & 0xffff0000u)};
    hi = h;
    lo = __builtin_bit_cast(u32x2, __builtin_convertvector(v - back, bf16x4));
}

// maximum over the four lanes that hold one row's scores (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float max_over_row(float x) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ bf16x8 load_query(const dlk_paged_params& p, int64_t at, int d, float scale, bf16x8& lo) {
    f32x8 x;
    if (p.q_bf16) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.q) + at + d);
        x = f32x8{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y), bf16_lo(w.z), bf16_hi(w.z), bf16_lo(w.w), bf16_hi(w.w)};
    } else {
        const float* row = static_cast<const float*>(p.q) + at + d;
        const f32x4 a = *reinterpret_cast<const f32x4*>(row), b = *reinterpret_cast<const f32x4*>(row + 4);
        x = f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    }
    bf16x8 hi;
    split8(x * scale, hi, lo);
    return hi;
}

template <typename KT, int HD, int NT>
__global__ __launch_bounds__(kThreads) void paged_stream(const dlk_paged_params p, const dlk_paged_item* items, float* partial_o,
                                                         float* partial_ml) {
    constexpr bool F32 = sizeof(KT) == 4;
    constexpr int PLANES = F32 ? 2 : 1;               // bf16 planes of the staged V^T
    constexpr int KS = HD < 32 ? 1 : HD / 32;         // k steps of the score product
    constexpr int DT = HD / 16;                       // 16-wide head-dim tiles of the output
    constexpr int KL = F32 ? 2 : 1;                   // 16-byte loads of a K fragment (8 values)
    constexpr int DPP = 16 / static_cast<int>(sizeof(KT)); // head-dim values of a 16-byte piece
    constexpr int PIECES = HD / DPP;                  // pieces of a row
    constexpr int VI = (PIECES + 7) / 8;              // V pieces per lane and key (64 lanes: 8 key pairs x 8 pieces)
    constexpr int VSTRIDE = kTileKeys + 4;            // bf16 per staged V^T row: 18 words spread the accesses over the banks
    constexpr int ROW = HD * static_cast<int>(sizeof(KT));
    constexpr int ROWS = 16 * NT;
    constexpr int STAGE = kWaves * PLANES * HD * VSTRIDE * 2, MERGE = kWaves * ROWS * HD * 4;
    // the staged V^T tiles, and after the last tile the waves' outputs
    __shared__ __attribute__((aligned(16))) char area[STAGE > MERGE ? STAGE : MERGE];
    __shared__ float m_s[kWaves][ROWS], l_s[kWaves][ROWS];

    const int t = threadIdx.x, lane = t % kWave, q = lane / 16, col = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int kvh = static_cast<int>(blockIdx.x) % p.KV;
    const dlk_paged_item item = items[blockIdx.x / p.KV];
    const int G = p.H / p.KV;
    const int32_t* table = p.tables + item.table;

    // the item's keys in four runs of whole tiles
    const int all = (item.key_end - item.key_begin + kTileKeys - 1) / kTileKeys;
    const int per_wave = (all + kWaves - 1) / kWaves;
    const int w_begin = item.key_begin + min(wave * per_wave, all) * kTileKeys;
    const int w_end = min(item.key_end, w_begin + per_wave * kTileKeys);
    const int tiles = max(0, (w_end - w_begin + kTileKeys - 1) / kTileKeys);

    struct Tile {
        u32x4 k[2][KS][KL];
        u32x4 v[2][VI][2];
    };
    const int kp = lane % 8, piece = lane / 8; // V: keys 2 kp, 2 kp + 1 of a half, pieces piece + 8 i
    const int k_offset = 8 * q < HD ? col * ROW + 8 * q * static_cast<int>(sizeof(KT)) : INT32_MAX / 2; // (past the range)
    auto load = [&](int tile, Tile& dst) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int key = w_begin + tile * kTileKeys + 16 * u;
            const int live = max(0, min(16, w_end - key));
            const int page = table[min(key, w_end - 1) >> p.page_shift];
            const int64_t at = ((static_cast<int64_t>(page) * p.KV + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
            const __amdgpu_buffer_rsrc_t kres = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<KT*>(static_cast<const KT*>(p.k)) + at * HD, 0, live * ROW, kBufferFlags);
            const __amdgpu_buffer_rsrc_t vres = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<KT*>(static_cast<const KT*>(p.v)) + at * HD, 0, live * ROW, kBufferFlags);
#pragma unroll
            for (int st = 0; st < KS; ++st)
#pragma unroll
                for (int e = 0; e < KL; ++e)
                    dst.k[u][st][e] = __builtin_amdgcn_raw_buffer_load_b128(
                        kres, k_offset + 32 * st * static_cast<int>(sizeof(KT)) + 16 * e, 0, 0);
#pragma unroll
            for (int i = 0; i < VI; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    dst.v[u][i][e] = __builtin_amdgcn_raw_buffer_load_b128(
                        vres, (2 * kp + e) * ROW + (min(piece + 8 * i, PIECES - 1)) * 16, 0, 0);
        }
    };

    // the rows as the B operand, in base 2: column col of tile nt is row row_begin + 16 nt + col
    bf16x8 qh[NT][KS], ql[NT][KS];
    int limit[NT]; // the last key that the row sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = min(item.row_begin + 16 * nt + col, item.row_end - 1);
        limit[nt] = min(item.first + row / G, w_end - 1);
        const int64_t at = (item.token + row / G) * p.q_row + static_cast<int64_t>(kvh * G + row % G) * p.q_head;
#pragma unroll
        for (int st = 0; st < KS; ++st)
            qh[nt][st] = load_query(p, at, min(32 * st + 8 * q, HD - 8), p.scale * 1.4426950408889634f, ql[nt][st]);
    }
    const int all_see = min(item.first + item.row_begin / G, w_end - 1); // the last key that every row sees

    f32x4 o[NT][DT], l[NT];
    float m_run[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_run[nt] = -INFINITY;
        l[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
    uint16_t* my_vt = reinterpret_cast<uint16_t*>(area) + wave * PLANES * HD * VSTRIDE;
    uint32_t* vt_words = reinterpret_cast<uint32_t*>(my_vt);

    auto use = [&](int tile, const Tile& cur) {
        // (a wave's LDS operations complete in order: the fences only keep the compiler from moving them past each other)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        // V^T of the tile into the wave's LDS tile: a word is a key pair of one head-dim row
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < VI; ++i) {
                if (PIECES < 8 && piece >= PIECES) continue;
                const u32x4 a = cur.v[u][i][0], c = cur.v[u][i][1];
                const int d0 = DPP * (piece + 8 * i), word = 8 * u + kp;
                if constexpr (F32) {
                    u32x2 h0, l0, h1, l1;
                    split4(a, h0, l0);
                    split4(c, h1, l1);
                    const uint32_t hw[4] = {(h0.x & 0xffffu) | (h1.x << 16), (h0.x >> 16) | (h1.x & 0xffff0000u),
                                            (h0.y & 0xffffu) | (h1.y << 16), (h0.y >> 16) | (h1.y & 0xffff0000u)};
                    const uint32_t lw[4] = {(l0.x & 0xffffu) | (l1.x << 16), (l0.x >> 16) | (l1.x & 0xffff0000u),
                                            (l0.y & 0xffffu) | (l1.y << 16), (l0.y >> 16) | (l1.y & 0xffff0000u)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        vt_words[(d0 + e) * (VSTRIDE / 2) + word] = hw[e];
                        vt_words[(HD + d0 + e) * (VSTRIDE / 2) + word] = lw[e];
                    }
                } else {
                    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        vt_words[(d0 + 2 * e) * (VSTRIDE / 2) + word] = (aw[e] & 0xffffu) | (cw[e] << 16);
                        vt_words[(d0 + 2 * e + 1) * (VSTRIDE / 2) + word] = (aw[e] >> 16) | (cw[e] & 0xffff0000u);
                    }
                }
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        // scores of both halves
        f32x4 s[NT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                bf16x8 kh, kl;
                if constexpr (F32)
                    split8(__builtin_bit_cast(f32x8, __builtin_shufflevector(cur.k[u][st][0], cur.k[u][st][KL - 1], 0, 1, 2, 3,
                                                                              4, 5, 6, 7)), kh, kl);
                else kh = __builtin_bit_cast(bf16x8, cur.k[u][st][0]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    s[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kh, qh[nt][st], s[nt][u], 0, 0, 0);
                    s[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kh, ql[nt][st], s[nt][u], 0, 0, 0);
                    if constexpr (F32) s[nt][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kl, qh[nt][st], s[nt][u], 0, 0, 0);
                }
            }
        }
        const int key0 = w_begin + tile * kTileKeys;
        bf16x8 ph[NT], pl[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (key0 + kTileKeys - 1 > all_see) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (key0 + 16 * u + 4 * q + j > limit[nt]) s[nt][u][j] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[nt][u][j]);
            const float m_new = fmaxf(m_run[nt], max_over_row(mx));
            // a row that has seen no key yet (masked so far, or scores of -inf) keeps a finite base: exp2(-inf) = 0
            const float base = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = __builtin_amdgcn_exp2f(m_run[nt] - base);
            m_run[nt] = m_new;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[nt][u][j] = __builtin_amdgcn_exp2f(s[nt][u][j] - base);
            if (!__all(alpha == 1.0f)) {
                l[nt] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[nt][d] *= alpha;
            }
            split8(f32x8{s[nt][0][0], s[nt][0][1], s[nt][0][2], s[nt][0][3], s[nt][1][0], s[nt][1][1], s[nt][1][2],
                         s[nt][1][3]}, ph[nt], pl[nt]);
            l[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, ph[nt], l[nt], 0, 0, 0);
            l[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pl[nt], l[nt], 0, 0, 0);
        }
        // lane (d = 16 dt + col, q) supplies V[keys 4 q .. +4 and 16 + 4 q .. +4][d]
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int at = (16 * dt + col) * VSTRIDE + 4 * q;
            const u32x2 lo4 = *reinterpret_cast<const u32x2*>(my_vt + at);
            const u32x2 hi4 = *reinterpret_cast<const u32x2*>(my_vt + at + 16);
            const bf16x8 a = __builtin_bit_cast(bf16x8, u32x4{lo4.x, lo4.y, hi4.x, hi4.y});
            bf16x8 al = a;
            if constexpr (F32) {
                const u32x2 llo4 = *reinterpret_cast<const u32x2*>(my_vt + HD * VSTRIDE + at);
                const u32x2 lhi4 = *reinterpret_cast<const u32x2*>(my_vt + HD * VSTRIDE + at + 16);
                al = __builtin_bit_cast(bf16x8, u32x4{llo4.x, llo4.y, lhi4.x, lhi4.y});
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, ph[nt], o[nt][dt], 0, 0, 0);
                o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pl[nt], o[nt][dt], 0, 0, 0);
                if constexpr (F32) o[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(al, ph[nt], o[nt][dt], 0, 0, 0);
            }
        }
    };
    if (tiles > 0) {
        // two tiles a turn, so that the buffers are named statically; the next tile is in flight while one is used
        Tile a, c;
        load(0, a);
        for (int tile = 0;;) {
            if (tile + 1 >= tiles) { use(tile, a); break; }
            load(tile + 1, c);
            use(tile, a);
            ++tile;
            if (tile + 1 >= tiles) { use(tile, c); break; }
            load(tile + 1, a);
            use(tile, c);
            ++tile;
        }
    }

    // merge the waves: a lane holds O[row col][d = 16 dt + 4 q + j] and the row's sum in every entry of l
    __syncthreads();
    float* o_s = reinterpret_cast<float*>(area);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (q == 0) {
            m_s[wave][16 * nt + col] = m_run[nt];
            l_s[wave][16 * nt + col] = l[nt][0];
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            *reinterpret_cast<f32x4*>(o_s + (wave * ROWS + 16 * nt + col) * HD + 16 * dt + 4 * q) = o[nt][dt];
    }
    __syncthreads();
    const int rows = item.row_end - item.row_begin;
    for (int i = t; i < rows * HD; i += kThreads) {
        const int r = i / HD, d = i % HD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, m_s[w][r]);
        const float base = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float weight = __builtin_amdgcn_exp2f(m_s[w][r] - base);
            L += weight * l_s[w][r];
            O += weight * o_s[(w * ROWS + r) * HD + d];
        }
        if (item.slot < 0) {
            const int row = item.row_begin + r;
            p.out[(static_cast<int64_t>(item.token + row / G) * p.H + kvh * G + row % G) * HD + d] = O / L;
        } else {
            const int64_t at = (static_cast<int64_t>(item.slot) * p.KV + kvh) * ROWS + r;
            partial_o[at * HD + d] = O;
            if (d == 0) {
                partial_ml[2 * at] = M;
                partial_ml[2 * at + 1] = L;
            }
        }
    }
}

// Joins the partials of a row: those of its own run's splits and those of the prefix that the batch shares.  A wave per
// (token, query head).
template <int HD>
__global__ __launch_bounds__(kThreads) void paged_merge(const dlk_paged_params p) {
    const int lane = threadIdx.x % kWave;
    const int unit = static_cast<int>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (unit >= p.merge_count * p.H) return;
    const dlk_paged_merge merge = p.merges[unit / p.H];
    const int h = unit % p.H, G = p.H / p.KV, kvh = h / G;
    const int rows = 16 * p.row_tiles, row = merge.row + h % G;
    const int shared_rows = 16 * p.shared_row_tiles, shared_row = merge.shared_row + h % G;
    auto place = [&](int i) { // split i of the row's own run
        return (static_cast<int64_t>(merge.slot + row / rows * merge.stride + i) * p.KV + kvh) * rows + row % rows;
    };
    auto shared_place = [&](int i) {
        return (static_cast<int64_t>(shared_row / shared_rows * p.shared_splits + i) * p.KV + kvh) * shared_rows +
               shared_row % shared_rows;
    };
    constexpr int PER = HD < kWave ? 1 : HD / kWave;
    float M = -INFINITY, L = 0.0f, O[PER] = {};
    auto add = [&](const float* o, const float* ml, int64_t at) {
        const float m = ml[2 * at], m_new = fmaxf(M, m), base = m_new == -INFINITY ? 0.0f : m_new;
        const float keep = __builtin_amdgcn_exp2f(M - base), weight = __builtin_amdgcn_exp2f(m - base);
        M = m_new;
        L = L * keep + weight * ml[2 * at + 1];
#pragma unroll
        for (int e = 0; e < PER; ++e) O[e] = O[e] * keep + weight * o[at * HD + min(lane * PER + e, HD - 1)];
    };
    for (int i = 0; i < merge.count; ++i) add(p.partial_o, p.partial_ml, place(i));
    for (int i = 0; i < p.shared_splits; ++i) add(p.shared_o, p.shared_ml, shared_place(i));
    float* out = p.out + (static_cast<int64_t>(merge.token) * p.H + h) * HD;
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (lane * PER + e < HD) out[lane * PER + e] = O[e] / L;
}

template <typename KT, int HD, int NT>
int launch_stream(const dlk_paged_params& p, const dlk_paged_item* items, int count, float* o, float* ml, hipStream_t stream) {
    hipLaunchKernelGGL((paged_stream<KT, HD, NT>), dim3(count * p.KV), dim3(kThreads), 0, stream, p, items, o, ml);
    return static_cast<int>(hipGetLastError());
}

template <typename KT, int HD>
int launch_rows(const dlk_paged_params& p, const dlk_paged_item* items, int count, int row_tiles, float* o, float* ml,
                hipStream_t stream) {
    if (count == 0) return 0;
    if (row_tiles == 1) return launch_stream<KT, HD, 1>(p, items, count, o, ml, stream);
    return static_cast<int>(hipErrorInvalidValue);
}

template <typename KT, int HD> int launch(const dlk_paged_params& p, hipStream_t stream) {
    int status = launch_rows<KT, HD>(p, p.shared_items, p.shared_count, p.shared_row_tiles, p.shared_o, p.shared_ml, stream);
    if (status == 0) status = launch_rows<KT, HD>(p, p.items, p.item_count, p.row_tiles, p.partial_o, p.partial_ml, stream);
    if (status != 0 || p.merge_count == 0) return status;
    const int64_t units = static_cast<int64_t>(p.merge_count) * p.H;
    hipLaunchKernelGGL((paged_merge<HD>), dim3((units + kWaves - 1) / kWaves), dim3(kThreads), 0, stream, p);
    return static_cast<int>(hipGetLastError());
}

template <typename KT> int launch_heads(const dlk_paged_params& p, hipStream_t stream) {
    switch (p.hd) {
    case 16: return launch<KT, 16>(p, stream);
    case 32: return launch<KT, 32>(p, stream);
    case 64: return launch<KT, 64>(p, stream);
    case 128: return launch<KT, 128>(p, stream);
    default: return static_cast<int>(hipErrorInvalidValue);
    }
}

} // namespace
} // namespace dlk

extern "C" int dlk_paged_attention(const dlk_paged_params* params, dlh_stream stream_handle) {
    const dlk_paged_params& p = *params;
    const int align = p.q_bf16 ? 8 : 4; // elements of 16 bytes
    if (p.KV <= 0 || p.H <= 0 || p.H % p.KV != 0 || p.page_shift < 4 || p.q_row % align != 0 || p.q_head % align != 0 ||
        reinterpret_cast<uintptr_t>(p.q) % 16 != 0 || (p.merge_count > 0 && !p.merges))
        return static_cast<int>(hipErrorInvalidValue);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_handle);
    return p.kv_bf16 ? dlk::launch_heads<uint16_t>(p, stream) : dlk::launch_heads<float>(p, stream);
}
