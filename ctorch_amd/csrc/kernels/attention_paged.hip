// Attention over the pages of a paged cache (see dlk_paged_params in kernels.h): each row of a run of tokens over the
// keys up to its own position, o = sum_j softmax_j(q k_j / sqrt(hd)) v_j, the keys found through the run's page table.
// f32 or bf16 pages, head size 16, 32, 64 or 128, page sizes that are powers of two from 16.
//
// Products are exact to f32 on the matrix cores.  bf16 keys and values go in as they are stored (v_mfma_f32_16x16x32_bf16)
// against queries and probabilities cut into three bf16 parts of 8 bits each, which hold all 24 bits of an f32: three
// products (bf16 queries are one part).  (Two parts, 2^-17 off, gave outputs 4e-6 off the 64-bit ones, three 7e-7.)  f32
// pages take the f32 matrix instruction where memory is the bound, and three by three parts where the products are, the
// three terms left out that are 2^-22 of a product at most together (typically 2^-24): six products, 2.7 times the f32
// instruction's rate.
//   S^T[16 keys][16 rows] = K[16][hd] Q[16][hd]^T    so that a lane holds scores of one row (lane % 16),
//   O^T[16 d][16 rows]   += V^T[16 d][keys] P^T       and they are the second product's right operand as they come.
// The softmax runs in base 2 with the running base and sum of each row; keys past a range are masked and their values
// read as zero, so that what a page holds behind the sequence never counts, not even a NaN.  An item that is all its rows
// see writes the output, the others (o, base, sum) partials that paged_merge joins.
#include "kernels/device_common.h"

namespace dlk {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// The nearest bf16 of each value, and the rest (exact): three parts hold all 24 bits.
// (Kept as words: vectors of bf16 that cross a branch are taken apart into halves.)
template <int PARTS> __device__ __forceinline__ void cut8(f32x8 v, u32x4 (&part)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const u32x4 h = part[i] = __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8));
        if (i + 1 < PARTS)
            v -= f32x8{__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16),
                       __uint_as_float(h.y & 0xffff0000u), __uint_as_float(h.z << 16), __uint_as_float(h.z & 0xffff0000u),
                       __uint_as_float(h.w << 16), __uint_as_float(h.w & 0xffff0000u)};
    }
}

// The first 8 bits of four values, and the rest: cut off, so that no finite key or value becomes infinite.
__device__ __forceinline__ u32x2 cut4(f32x4& v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    v -= __builtin_bit_cast(f32x4, w & 0xffff0000u);
    return u32x2{__builtin_amdgcn_perm(w.y, w.x, 0x07060302u), __builtin_amdgcn_perm(w.w, w.z, 0x07060302u)};
}

__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), sum, 0, 0, 0);
}
__device__ __forceinline__ f32x16 product(u32x4 a, u32x4 b, f32x16 sum) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), sum, 0, 0, 0);
}

// over the lanes that hold one row's scores: l and l ^ 32, and of ROWS = 16 rows a wave l ^ 16 and l ^ 48 too
template <int ROWS, typename Op> __device__ __forceinline__ float over_row(float x, Op op) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(h[0]), __uint_as_float(h[1]));
    if constexpr (ROWS == 32) return x;
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int ROWS> __device__ __forceinline__ float max_over_row(float x) {
    return over_row<ROWS>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int ROWS> __device__ __forceinline__ float sum_over_row(float x) {
    return over_row<ROWS>(x, [](float a, float b) { return a + b; });
}

// the compiler keeps LDS accesses of a wave in order across this (the hardware does by itself)
__device__ __forceinline__ void wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// What the host wrote for the step, read through the scalar cache: page ids and items are the same for a whole wave, and a
// vector load of them would make every buffer descriptor behind it a loop over the lanes.
template <typename T> using Planned = const __attribute__((address_space(4))) T;
template <typename T> __device__ __forceinline__ Planned<T>* planned(const T* pointer) { return (Planned<T>*)(pointer); }

__device__ __forceinline__ dlk_paged_item item_of(const dlk_paged_list& list, int n) {
    Planned<dlk_paged_item>* from = planned(list.items) + n;
    return {from->token, from->row_begin, from->row_end, from->table, from->key_begin, from->key_end, from->first, from->slot};
}

// 8 entries of a query row, unscaled
__device__ __forceinline__ f32x8 query8(const dlk_paged_params& p, int64_t at) {
    if (p.q_bf16) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.q) + at);
        return f32x8{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y), bf16_lo(w.z), bf16_hi(w.z), bf16_lo(w.w), bf16_hi(w.w)};
    }
    const float* row = static_cast<const float*>(p.q) + at;
    const f32x4 a = *reinterpret_cast<const f32x4*>(row), b = *reinterpret_cast<const f32x4*>(row + 4);
    return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// The four values at V[keys at .. +4 rows][d], d = the lane's column of a 16-wide block, out of row-major bf16 LDS rows of
// STRIDE: the 16 lanes of a group read 4 rows of 16 between them, and each receives a column (ds_read_b64_tr_b16).
template <int STRIDE> __device__ __forceinline__ u32x2 column4(const uint16_t* block, int col) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const uint16_t* from = block + (col / 4) * STRIDE + 4 * (col % 4);
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(from)));
}

// A value that some of a tile's rows do not see must not reach them, and zero times an infinity or a NaN would.  So the
// tiles that are like that are looked over: what is not finite goes into the products as zero, and if there was any, it is
// added to the rows that see it in the end, key by key (infinities and NaN add up the same in any order).
__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }
template <typename KT, int N> __device__ __forceinline__ bool clear_not_finite(u32x4 (&pieces)[N]) {
    if constexpr (sizeof(KT) == 4) {
        uint64_t any = 0;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            bool piece = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool word = not_finite(__uint_as_float(pieces[n][i]));
                pieces[n][i] = word ? 0u : pieces[n][i];
                piece |= word;
            }
            any |= __ballot(piece);
        }
        return any != 0;
    } else {
        uint32_t sum = 0; // (an exponent of ones carries into the sign)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum |= (pieces[n][i] & 0x7f807f80u) + 0x00800080u;
        if (!__any((sum & 0x80008000u) != 0)) return false;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = pieces[n][i];
                pieces[n][i] &= (not_finite(__uint_as_float(w)) ? 0xffffu : ~0u) & (not_finite(__uint_as_float(w << 16)) ? 0xffff0000u : ~0u);
            }
        return true;
    }
}
// An entry, and four, of a row of values.
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(uint16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ f32x4 four(const float* from) { return *reinterpret_cast<const f32x4*>(from); }
__device__ __forceinline__ f32x4 four(const uint16_t* from) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(from);
    return f32x4{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
}
template <typename KT> __device__ __forceinline__ const KT* value_row(const dlk_paged_params& p, Planned<int32_t>* table, int kvh, int key) {
    const int64_t page = table[key >> p.page_shift];
    return static_cast<const KT*>(p.v) + (((page * p.KV + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * (int64_t(1) * p.hd);
}

// Weights of a row whose base is not set yet: any score sets it.  (Scores stay below 2^30: s c - base is one fma, off by the
// rounding of the base, a factor that the weights and their sum share.)
constexpr float kNoBase = -1e30f;
// How far (in powers of two) a score may lie above its row's base before the base follows.
constexpr float kSlack = 8.0f;

// The softmax of T rows a lane: base[i] is what row i's weights exp2(s c - base) are taken from, l[i] the lane's share of
// their sum.  The base need not be the row's maximum: f32 weights up to 2^8 are as exact, so it moves only when a score
// passes it by more, mostly once, and the row's lanes do not have to compare their scores before that.  S: a vector of a
// row's scores, N of them; O: one of a row's outputs, D of them.
template <int ROWS, int T, int N, int D, typename S, typename O>
__device__ __forceinline__ void settle(const S (&s)[T][N], float (&base)[T], float (&l)[T], float c, O (&outputs)[T][D]) {
    constexpr int LENGTH = sizeof(S) / 4;
    float top[T];
    bool passed = false;
#pragma unroll
    for (int i = 0; i < T; ++i) {
        top[i] = s[i][0][0];
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int j = 0; j < LENGTH; ++j) top[i] = fmaxf(top[i], s[i][u][j]);
        passed |= top[i] * c > base[i] + kSlack;
    }
    if (__any(passed)) {
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const float next = fmaxf(base[i], max_over_row<ROWS>(top[i]) * c), keep = __builtin_amdgcn_exp2f(base[i] - next);
            base[i] = next;
            l[i] *= keep;
#pragma unroll
            for (int d = 0; d < D; ++d) outputs[i][d] *= keep;
        }
    }
}
template <int N, typename S> __device__ __forceinline__ void soften(S (&s)[N], float base, float& l, float c) {
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(S) / 4); ++j) {
            s[u][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], c, -base));
            l += s[u][j];
        }
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 NT rows over a range of keys: the four waves split the range, each streams its run in tiles of 16 NU keys from
// memory into registers and keeps its own softmax, and they merge in LDS.  Bound by memory: a tile's keys and values are
// asked for as soon as the registers of the ones before are free, and the waves of a SIMD hide each other's waits.  (32
// tokens over up to 4096 bf16 keys, 8 heads of 64: 34 us, 4.9 TB/s; 8 over up to 32768, heads of 128: 122 us, 5.4 TB/s.)
//
// bf16: V goes through the wave's own LDS tile, stored as it comes and read back by columns; the cut queries of two row
// tiles stay in LDS, where one tile's fit the registers.  f32: no LDS; with the keys of step j of the second product chosen
// as 4 q + j (q = lane / 16), its right operand is the score register j, and its left one 16 bytes of a V row, whose four
// entries belong to four output tiles (tile e, row i is head entry 4 i + e).
template <typename KT, int HD, int NT, int QP> struct Few {
    static constexpr bool F32 = sizeof(KT) == 4;
    static constexpr int NU = F32 && HD == 128 ? 1 : 2; // 16-key halves of a tile (f32 heads of 128: registers)
    static constexpr int KEYS = 16 * NU, ROWS = 16 * NT;
    static constexpr int VSTRIDE = HD + 16;             // bf16 of a staged V row: the column reads hit no bank twice
    static constexpr bool QLDS = !F32 && NT > 1;        // the cut queries, in LDS
    // LDS: V tiles and queries, then the waves' outputs; and the waves' bases and sums
    static constexpr int STAGE = F32 ? 0 : kWaves * KEYS * VSTRIDE * 2, QUERIES = QLDS ? QP * ROWS * VSTRIDE * 2 : 0;
    static constexpr int MERGE = kWaves * ROWS * HD * 4;
    static constexpr int AREA = STAGE + QUERIES > MERGE ? STAGE + QUERIES : MERGE, LDS = AREA + 2 * kWaves * ROWS * 4;
};

template <typename KT, int HD, int NT, int QP>
__device__ __forceinline__ void attend_few(const dlk_paged_params& p, int block, char* area) {
    using S = Few<KT, HD, NT, QP>;
    constexpr bool F32 = S::F32, QLDS = S::QLDS;
    constexpr int NU = S::NU, KEYS = S::KEYS, ROWS = S::ROWS, VSTRIDE = S::VSTRIDE, STAGE = S::STAGE;
    constexpr int KS = HD < 32 ? 1 : HD / 32;         // bf16: k steps of the score product
    constexpr int KF = HD / 16;                       // f32: 16-byte pieces of a key per lane
    constexpr int DT = HD / 16;                       // output tiles
    constexpr int E = HD >= 64 ? 4 : HD / 16;         // f32: entries of a V row per lane and load
    constexpr int VL = HD / 16 / E;                   // f32: such loads of a V row
    constexpr int PIECES = HD / 8;                    // bf16: 16-byte pieces of a row
    constexpr int VI = (16 * PIECES + kWave - 1) / kWave; // bf16: V pieces per lane and half
    constexpr int ROW = HD * static_cast<int>(sizeof(KT));
    float(*m_s)[ROWS] = reinterpret_cast<float(*)[ROWS]>(area + S::AREA);
    float(*l_s)[ROWS] = m_s + kWaves;

    const int t = threadIdx.x, lane = t % kWave, q = lane / 16, col = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int kvh = block % p.KV;
    const dlk_paged_item item = item_of(p.lists[DLK_PAGED_FEW], block / p.KV);
    const int G = p.H / p.KV;
    Planned<int32_t>* table = planned(p.tables) + item.table;
    const float c = p.scale * 1.4426950408889634f;

    // the item's keys in four runs of whole tiles
    const int all = (item.key_end - item.key_begin + KEYS - 1) / KEYS;
    const int per_wave = (all + kWaves - 1) / kWaves;
    const int w_begin = item.key_begin + min(wave * per_wave, all) * KEYS;
    const int w_end = min(item.key_end, w_begin + per_wave * KEYS);
    const int tiles = max(0, (w_end - w_begin + KEYS - 1) / KEYS);

    constexpr int kBeyond = INT32_MAX / 2; // an offset past every range: reads as zero
    const int k_offset = F32 || 8 * q < HD ? col * ROW + 16 * q : kBeyond;
    // the 16 rows of a half: their place, and how many bytes of them are within the run
    auto half_of = [&](int tile, int u, int& bytes) {
        const int key = w_begin + tile * KEYS + 16 * u;
        bytes = __builtin_amdgcn_readfirstlane(max(0, min(16, w_end - key)) * ROW);
        const int page = table[min(key, w_end - 1) >> p.page_shift];
        return (((static_cast<int64_t>(page) * p.KV + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * HD;
    };
    u32x4 k[NU][F32 ? KF : KS], v[NU][F32 ? 4 * VL : VI];
    auto load_keys = [&](int tile) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            int bytes;
            const int64_t at = half_of(tile, u, bytes);
            const __amdgpu_buffer_rsrc_t rows =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<KT*>(static_cast<const KT*>(p.k)) + at, 0, bytes, kBufferFlags);
#pragma unroll
            for (int st = 0; st < (F32 ? KF : KS); ++st) k[u][st] = __builtin_amdgcn_raw_buffer_load_b128(rows, k_offset + 64 * st, 0, 0);
        }
    };
    auto load_values = [&](int tile) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            int bytes;
            const int64_t at = half_of(tile, u, bytes);
            const __amdgpu_buffer_rsrc_t rows =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<KT*>(static_cast<const KT*>(p.v)) + at, 0, bytes, kBufferFlags);
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < VL; ++i) {
                        const int offset = (4 * q + j) * ROW + (64 * i + E * col) * 4;
                        u32x4& to = v[u][j * VL + i];
                        if constexpr (E == 4) to = __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0);
                        if constexpr (E == 2) {
                            const u32x2 two = __builtin_amdgcn_raw_buffer_load_b64(rows, offset, 0, 0);
                            to = u32x4{two.x, two.y, 0u, 0u};
                        }
                        if constexpr (E == 1) to = u32x4{__builtin_amdgcn_raw_buffer_load_b32(rows, offset, 0, 0), 0u, 0u, 0u};
                    }
            } else {
#pragma unroll
                for (int i = 0; i < VI; ++i) // the half's rows are one piece of memory, read in order
                    v[u][i] = __builtin_amdgcn_raw_buffer_load_b128(rows, 16 * (lane + kWave * i), 0, 0);
            }
        }
    };
    if (tiles > 0) {
        load_keys(0);
        load_values(0);
    }

    // the rows as the right operand: column col of tile nt is row row_begin + 16 nt + col
    u32x4 qb[QLDS ? 1 : NT][KS][QP];
    f32x4 qf[NT][KF];
    int limit[NT]; // the last key that the row sees
    uint16_t* q_s = reinterpret_cast<uint16_t*>(area + STAGE);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = min(item.row_begin + 16 * nt + col, item.row_end - 1);
        limit[nt] = min(item.first + row / G, w_end - 1);
        const int64_t at = (item.token + row / G) * p.q_row + static_cast<int64_t>(kvh * G + row % G) * p.q_head;
        if constexpr (F32) {
#pragma unroll
            for (int st = 0; st < KF; ++st) { // entries 16 st + 4 q .. +4
                const f32x8 x = query8(p, at + 16 * st + 8 * (q / 2));
                qf[nt][st] = q % 2 ? f32x4{x[4], x[5], x[6], x[7]} : f32x4{x[0], x[1], x[2], x[3]};
            }
        } else {
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                u32x4(&parts)[QP] = qb[QLDS ? 0 : nt][st];
                if (QLDS && wave != nt) continue; // wave nt cuts row tile nt for all
                cut8<QP>(query8(p, at + min(32 * st + 8 * q, HD - 8)), parts);
                if (QLDS && 8 * q < HD) {
#pragma unroll
                    for (int part = 0; part < QP; ++part)
                        *reinterpret_cast<u32x4*>(q_s + (part * ROWS + 16 * nt + col) * VSTRIDE + 32 * st + 8 * q) = parts[part];
                }
            }
        }
    }
    if (QLDS) __syncthreads();
    const int every = item.first + item.row_begin / G, all_see = min(every, w_end - 1); // the last key that every row sees

    f32x4 o[NT][DT];
    float base[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        base[nt] = kNoBase;
        l[nt] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto entry_of = [&](int dt, int j) { return F32 ? 16 * E * (dt / E) + E * (4 * q + j) + dt % E : 16 * dt + 4 * q + j; }; // of o[.][dt][j]
    uint16_t* my_v = reinterpret_cast<uint16_t*>(area) + wave * KEYS * VSTRIDE;

    bool spoiled = false;
    for (int tile = 0; tile < tiles; ++tile) {
        const int key0 = w_begin + tile * KEYS;
        auto look = [&] {
            if (min(key0 + KEYS, w_end) - 1 <= every) return; // (every row sees all of it)
            for (auto& half : v) spoiled |= clear_not_finite<KT>(half);
        };
        if constexpr (!F32) {
            look();
            wave_order();
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < VI; ++i) {
                    const int at = lane + kWave * i;
                    if (16 * PIECES >= kWave || at < 16 * PIECES)
                        *reinterpret_cast<u32x4*>(my_v + (16 * u + at / PIECES) * VSTRIDE + 8 * (at % PIECES)) = v[u][i];
                }
            wave_order();
            if (tile + 1 < tiles) load_values(tile + 1);
        }
        f32x4 s[NT][NU];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u = 0; u < NU; ++u) s[nt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < (F32 ? KF : KS); ++st)
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int u = 0; u < NU; ++u)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            s[nt][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[u][st][e]), qf[nt][st][e], s[nt][u], 0, 0, 0);
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int part = QP - 1; part >= 0; --part) {
                        u32x4 x = qb[QLDS ? 0 : nt][st][part];
                        if constexpr (QLDS)
                            x = *reinterpret_cast<const u32x4*>(q_s + (part * ROWS + 16 * nt + col) * VSTRIDE + min(32 * st + 8 * q, HD - 8));
#pragma unroll
                        for (int u = 0; u < NU; ++u)
                            s[nt][u] = product(k[u][st], x, s[nt][u]);
                    }
            }
        if (tile + 1 < tiles) load_keys(tile + 1);
        u32x4 pb[NT][3];
        if (key0 + KEYS - 1 > all_see) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (key0 + 16 * u + 4 * q + j > limit[nt]) s[nt][u][j] = -INFINITY;
        }
        settle<16>(s, base, l, c, o);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            soften(s[nt], base[nt], l[nt], c);
            if constexpr (!F32)
                cut8<3>(f32x8{s[nt][0][0], s[nt][0][1], s[nt][0][2], s[nt][0][3], s[nt][NU - 1][0], s[nt][NU - 1][1],
                              s[nt][NU - 1][2], s[nt][NU - 1][3]}, pb[nt]);
        }
        if constexpr (F32) {
            look();
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < VL; ++i)
#pragma unroll
                        for (int e = 0; e < E; ++e)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                o[nt][i * E + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[u][j * VL + i][e]), s[nt][u][j], o[nt][i * E + e], 0, 0, 0);
            if (tile + 1 < tiles) load_values(tile + 1);
        } else {
            // lane (d = 16 dt + col, q) supplies V[keys 4 q .. +4 and 16 + 4 q .. +4][d], as its probabilities lie
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const u32x2 a = column4<VSTRIDE>(my_v + 4 * q * VSTRIDE + 16 * dt, col);
                const u32x2 b = column4<VSTRIDE>(my_v + (16 + 4 * q) * VSTRIDE + 16 * dt, col);
                const u32x4 columns = {a.x, a.y, b.x, b.y};
#pragma unroll
                for (int part = 2; part >= 0; --part)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) o[nt][dt] = product(columns, pb[nt][part], o[nt][dt]);
            }
        }
    }
    if (spoiled) {
#pragma unroll 1
        for (int key = w_begin + max(0, every + 1 - w_begin) / KEYS * KEYS; key < w_end; ++key) {
            const KT* row = value_row<KT>(p, table, kvh, key);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = value_of(row[entry_of(dt, j)]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        if (not_finite(x) && key <= limit[nt]) o[nt][dt][j] += x;
                }
        }
    }

    // merge the waves
    __syncthreads();
    float* o_s = reinterpret_cast<float*>(area);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float sum = sum_over_row<16>(l[nt]);
        if (q == 0) {
            m_s[wave][16 * nt + col] = base[nt];
            l_s[wave][16 * nt + col] = sum;
        }
        float* row = o_s + (wave * ROWS + 16 * nt + col) * HD;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) row[entry_of(dt, j)] = o[nt][dt][j];
    }
    __syncthreads();
    const int rows = item.row_end - item.row_begin;
    for (int i = t; i < rows * HD; i += kThreads) {
        const int r = i / HD, d = i % HD;
        float M = kNoBase;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, m_s[w][r]);
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float weight = __builtin_amdgcn_exp2f(m_s[w][r] - M);
            L += weight * l_s[w][r];
            O += weight * o_s[(w * ROWS + r) * HD + d];
        }
        if (item.slot < 0) {
            const int row = item.row_begin + r;
            p.out[(static_cast<int64_t>(item.token + row / G) * p.H + kvh * G + row % G) * HD + d] = O / L;
        } else {
            const int64_t at = static_cast<int64_t>(kvh) * p.places + item.slot + r;
            p.partial_o[at * HD + d] = O;
            if (d == 0) {
                p.partial_ml[2 * at] = M;
                p.partial_ml[2 * at + 1] = L;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ many rows
// 128 rows over a range of keys, 32 a wave, in tiles of 32 keys that pass through LDS for all waves: while one tile is used
// the next is staged into the other buffer, from the registers that then receive the one after it, so that a tile costs one
// barrier.  v_mfma_f32_32x32x16_bf16: a lane holds 16 scores of row lane % 32, of the keys 8 (i / 4) + 4 (lane / 32) + i % 4.
// (The matrix cores and the vector ALUs, which cut the weights and stage the tiles, have about as much to do here, and the
// 32 x 32 instruction leaves the vector ALUs more room than two of 16 x 16: three vector instructions beside each of the
// latter cost 26 % of its rate, beside the former 12 %.)  f32 pages are cut into three bf16 planes as they are staged, once
// for the 128 rows.  (3000 new rows of 32 heads after 1000: f32 pages, heads of 64 340 us, of 128 645 us; bf16 183 and 330 us:
// 0.95 to 1.1 PF/s of the products that run, where a large bf16 product reaches 1.2.  f32 queries over bf16 pages at heads of 128
// take all 256 registers and spill 5.)
template <typename KT, int HD> struct Many {
    static constexpr int PLANES = sizeof(KT) == 4 ? 3 : 1;
    static constexpr int BUFFERS = sizeof(KT) == 4 && HD == 128 ? 1 : 2; // (LDS of two work-groups a CU)
    static constexpr int KEYS = 32, STRIDE = HD + 16;                    // bf16 of a staged row
    static constexpr int LDS = 2 * BUFFERS * PLANES * KEYS * STRIDE * 2;
};

template <typename KT, int HD, int QP>
__device__ __forceinline__ void attend_many(const dlk_paged_params& p, int block, char* area) {
    using S = Many<KT, HD>;
    constexpr bool F32 = sizeof(KT) == 4;
    constexpr int PLANES = S::PLANES, BUFFERS = S::BUFFERS, KEYS = S::KEYS, STRIDE = S::STRIDE;
    constexpr int KS = HD / 16, DT = HD < 32 ? 1 : HD / 32; // (heads of 16: half an output tile is left)
    constexpr bool EARLY = HD <= 64;                  // a tile's keys are read ahead of the softmax (registers)
    constexpr int DPP = 16 / static_cast<int>(sizeof(KT)), PIECES = HD / DPP;
    constexpr int ROW = HD * static_cast<int>(sizeof(KT));
    // a half of 16 keys is one piece of memory of BLOCK 16-byte pieces: several passes of all threads, or part of them
    constexpr int BLOCK = 16 * PIECES, PASSES = BLOCK / kThreads, LOADS = PASSES ? 2 * PASSES : 1;
    constexpr int TEAM = BLOCK < kWave ? kWave : BLOCK; // threads of a half, where one pass takes both
    typedef uint16_t Planes[PLANES][KEYS * STRIDE];
    Planes* const ks = reinterpret_cast<Planes*>(area);
    Planes* const vs = ks + BUFFERS;

    const int t = threadIdx.x, lane = t % kWave, half = lane / 32, r = lane % 32;
    const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const int kvh = block % p.KV;
    const dlk_paged_item item = item_of(p.lists[DLK_PAGED_MANY], block / p.KV);
    const int G = p.H / p.KV;
    Planned<int32_t>* table = planned(p.tables) + item.table;
    const float c = p.scale * 1.4426950408889634f;
    const int tiles = (item.key_end - item.key_begin + KEYS - 1) / KEYS;
    // the last key that every row sees; the tiles behind it hold keys that some row does not see
    const int every = item.first + item.row_begin / G;
    auto end_of = [&](int tile) { return min(item.key_begin + (tile + 1) * KEYS, item.key_end); };
    __shared__ int spoiled[kWaves]; // what a wave staged behind `every` was not all finite
    if (lane == 0) spoiled[wave] = 0;

    auto half_of = [&](int i) { return PASSES ? i / (PASSES ? PASSES : 1) : wave * kWave / TEAM; };
    auto piece_of = [&](int i) { return PASSES ? t + kThreads * (i % (PASSES ? PASSES : 1)) : t % TEAM; };
    const bool loads = PASSES || (t / TEAM < 2 && t % TEAM < BLOCK);
    u32x4 kr[LOADS], vr[LOADS];
    // the pages of a tile's halves: asked for a tile before the loads that need them
    struct Pages {
        int of[2];
    };
    auto pages_of = [&](int tile) {
        const int key = item.key_begin + tile * KEYS;
        return Pages{{table[min(key, item.key_end - 1) >> p.page_shift], table[min(key + 16, item.key_end - 1) >> p.page_shift]}};
    };
    auto load = [&](int tile, const Pages& pages, const void* pool, u32x4 (&to)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int key = item.key_begin + tile * KEYS + 16 * half_of(i);
            const int bytes = __builtin_amdgcn_readfirstlane(max(0, min(16, item.key_end - key)) * ROW); // what lies behind reads as zero
            const int page = half_of(i) == 0 ? pages.of[0] : pages.of[1];
            const int64_t at = (((static_cast<int64_t>(page) * p.KV + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * HD;
            to[i] = __builtin_amdgcn_raw_buffer_load_b128(
                __builtin_amdgcn_make_buffer_rsrc(const_cast<KT*>(static_cast<const KT*>(pool)) + at, 0, bytes, kBufferFlags),
                loads ? 16 * piece_of(i) : INT32_MAX / 2, 0, 0);
        }
    };
    auto stage = [&](const u32x4 (&from)[LOADS], Planes& planes) {
        if (!loads) return;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int to = (16 * half_of(i) + piece_of(i) / PIECES) * STRIDE + DPP * (piece_of(i) % PIECES);
            if constexpr (F32) {
                f32x4 x = __builtin_bit_cast(f32x4, from[i]);
#pragma unroll
                for (int plane = 0; plane < PLANES; ++plane) *reinterpret_cast<u32x2*>(&planes[plane][to]) = cut4(x);
            } else {
                *reinterpret_cast<u32x4*>(&planes[0][to]) = from[i];
            }
        }
    };
    auto load_keys = [&](int tile, const Pages& pages) { load(tile, pages, p.k, kr); };
    auto load_values = [&](int tile, const Pages& pages) { load(tile, pages, p.v, vr); };
    auto stage_keys = [&](int buffer) { stage(kr, ks[buffer]); };
    auto look = [&](int tile) {
        if (end_of(tile) - 1 <= every) return;
        if (clear_not_finite<KT>(vr)) spoiled[wave] = 1;
    };
    auto stage_values = [&](int buffer) { stage(vr, vs[buffer]); };
    Pages pages = pages_of(0);
    load_keys(0, pages);
    load_values(0, pages);
    pages = pages_of(1);

    // this lane's row
    u32x4 qb[KS][QP];
    const int first_row = item.row_begin + 32 * wave, row = min(first_row + r, item.row_end - 1);
    const int limit = min(item.first + row / G, item.key_end - 1);
    const int64_t query = (item.token + row / G) * p.q_row + static_cast<int64_t>(kvh * G + row % G) * p.q_head;
#pragma unroll
    for (int st = 0; st < KS; ++st) cut8<QP>(query8(p, query + 16 * st + 8 * half), qb[st]);
    // the last key that every row of the wave sees, and the last that any does
    const int all_see = min(item.first + min(first_row, item.row_end - 1) / G, item.key_end - 1);
    const int any_sees = first_row < item.row_end ? min(item.first + min(first_row + 31, item.row_end - 1) / G, item.key_end - 1) : -1;

    f32x16 o[1][DT];
    float base[1] = {kNoBase}, l[1] = {0.0f};
#pragma unroll
    for (int d = 0; d < DT; ++d) o[0][d] = f32x16{};

    auto key_of = [&](int buffer, int st, int plane) {
        return *reinterpret_cast<const u32x4*>(&ks[buffer][plane][r * STRIDE + 16 * st + 8 * half]);
    };
    auto read_keys = [&](int buffer, u32x4 (&to)[KS][PLANES]) {
#pragma unroll
        for (int st = 0; st < KS; ++st)
#pragma unroll
            for (int plane = 0; plane < PLANES; ++plane) to[st][plane] = key_of(buffer, st, plane);
    };
    auto score = [&](int buffer, const u32x4 (&read)[KS][PLANES], f32x16& s) {
        s = f32x16{};
#pragma unroll
        for (int st = 0; st < KS; ++st)
#pragma unroll
            for (int plane = PLANES - 1; plane >= 0; --plane) {
                const u32x4 k = EARLY ? read[st][plane] : key_of(buffer, st, plane);
#pragma unroll
                for (int part = QP - 1; part >= 0; --part)
                    if (part + plane <= 2) s = product(k, qb[st][part], s);
            }
    };
    auto hide = [&](int tile, f32x16& s) {
        const int key0 = item.key_begin + tile * KEYS;
        if (key0 + KEYS - 1 <= all_see) return;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (key0 + 8 * (i / 4) + 4 * half + i % 4 > limit) s[i] = -INFINITY;
    };
    auto weigh = [&](f32x16 (&s)[1], u32x4 (&pb)[2][3]) {
        soften(s, base[0], l[0], c);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            cut8<3>(f32x8{s[0][8 * u], s[0][8 * u + 1], s[0][8 * u + 2], s[0][8 * u + 3], s[0][8 * u + 4], s[0][8 * u + 5],
                          s[0][8 * u + 6], s[0][8 * u + 7]}, pb[u]);
    };
    // lane (d = 32 dt + r, half) supplies V[keys 16 u + 4 half .. +4 and 8 behind them][d], as its weights lie
    auto add = [&](int buffer, const u32x4 (&pb)[2][3]) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int plane = PLANES - 1; plane >= 0; --plane) {
                    const uint16_t* block = &vs[buffer][plane][(16 * u + 4 * half) * STRIDE + 32 * dt + 16 * (r / 16)];
                    const u32x2 a = column4<STRIDE>(block, r % 16), b = column4<STRIDE>(block + 8 * STRIDE, r % 16);
                    const u32x4 v = {a.x, a.y, b.x, b.y};
#pragma unroll
                    for (int part = 2; part >= 0; --part)
                        if (part + plane <= 2) o[0][dt] = product(v, pb[u][part], o[0][dt]);
                }
    };
    // tiles that some row of the wave sees
    const int mine = any_sees < item.key_begin ? 0 : min(tiles, (any_sees - item.key_begin) / KEYS + 1);
    f32x16 s[1][1];
    u32x4 keys[KS][PLANES];
    if constexpr (BUFFERS == 2) {
        // Tile t's weights are worked out while the products of tile t + 1's scores run, and tile t + 1's values and tile
        // t + 2's keys are staged while those of its outputs do.  (Loads behind the last tile read nothing.)  The buffers'
        // numbers are constants, so that the compiler sees that the reads and writes of a step are apart.
        stage_keys(0);
        load_keys(1, pages);
        look(0);
        stage_values(0);
        load_values(1, pages);
        pages = pages_of(2); // of tile t + 2
        __syncthreads();
        stage_keys(1);
        load_keys(2, pages);
        if (EARLY) read_keys(0, keys);
        if (mine > 0) score(0, keys, s[0][0]);
        __syncthreads();
        auto step = [&](int tile, auto buffer) {
            constexpr int B = decltype(buffer)::value;
            look(tile + 1); // (here, where no products are in flight: a branch in the midst of them costs 5 %)
            const Pages ahead = pages_of(tile + 3);
            u32x4 pb[2][3];
            f32x16 next;
            if (EARLY) read_keys(1 - B, keys);
            hide(tile, s[0][0]);
            settle<32>(s, base, l, c, o);
            score(1 - B, keys, next); // (of no use behind the last tile)
            weigh(s[0], pb);
            stage_keys(B);
            stage_values(1 - B);
            load_keys(tile + 3, ahead);
            load_values(tile + 2, pages);
            add(B, pb);
            s[0][0] = next;
            pages = ahead;
            __syncthreads();
        };
        int tile = 0;
        for (; tile + 1 < mine; tile += 2) {
            step(tile, std::integral_constant<int, 0>{});
            step(tile + 1, std::integral_constant<int, 1>{});
        }
        if (tile < mine) step(tile++, std::integral_constant<int, 0>{});
        for (; tile < tiles; ++tile) { // the other waves' tiles
            const Pages ahead = pages_of(tile + 3);
            stage_keys(tile % 2);
            look(tile + 1);
            stage_values((tile + 1) % 2);
            load_keys(tile + 3, ahead);
            load_values(tile + 2, pages);
            pages = ahead;
            __syncthreads();
        }
    } else {
        stage_keys(0);
        look(0);
        stage_values(0);
        load_keys(1, pages);
        load_values(1, pages);
        __syncthreads();
        for (int tile = 0; tile < tiles; ++tile) {
            pages = pages_of(tile + 2);
            if (tile < mine) {
                u32x4 pb[2][3];
                score(0, keys, s[0][0]);
                hide(tile, s[0][0]);
                settle<32>(s, base, l, c, o);
                weigh(s[0], pb);
                add(0, pb);
            }
            __syncthreads();
            stage_keys(0);
            look(tile + 1);
            stage_values(0);
            load_keys(tile + 2, pages);
            load_values(tile + 2, pages);
            __syncthreads();
        }
    }

    // lane holds O[row r][d = 32 dt + 8 (i / 4) + 4 half + i % 4]
    if (item.key_end - 1 > every && (spoiled[0] | spoiled[1] | spoiled[2] | spoiled[3])) { // (a barrier ended the last tile)
#pragma unroll 1
        for (int key = item.key_begin + max(0, every + 1 - item.key_begin) / KEYS * KEYS; key < item.key_end; ++key) {
            const KT* from = value_row<KT>(p, table, kvh, key) + 4 * half;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (32 * dt + 8 * i >= HD) continue;
                    const f32x4 x = four(from + 32 * dt + 8 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (not_finite(x[j]) && key <= limit) o[0][dt][4 * i + j] += x[j];
                }
        }
    }
    const float sum = sum_over_row<32>(l[0]);
    if (first_row + r >= item.row_end) return;
    const bool whole = item.slot < 0;
    const int64_t at = static_cast<int64_t>(kvh) * p.places + item.slot + row - item.row_begin;
    float* out = whole ? p.out + (static_cast<int64_t>(item.token + row / G) * p.H + kvh * G + row % G) * HD : p.partial_o + at * HD;
    const float scale = whole ? 1.0f / sum : 1.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (32 * dt + 8 * i < HD)
                *reinterpret_cast<f32x4*>(out + 32 * dt + 8 * i + 4 * half) =
                    f32x4{o[0][dt][4 * i], o[0][dt][4 * i + 1], o[0][dt][4 * i + 2], o[0][dt][4 * i + 3]} * scale;
    if (!whole && half == 0) {
        p.partial_ml[2 * at] = base[0];
        p.partial_ml[2 * at + 1] = sum;
    }
}

// One launch for all items: the ones of many rows first, which take longest, and beside them those of few, which wait for
// memory where the others wait for the matrix cores.
template <typename KT, int HD, int NT, int QP, bool FEW, bool MANY>
__global__ __launch_bounds__(kThreads, MANY || NT > 1 || (sizeof(KT) == 2 && QP > 1) ? 2 : 3) void paged_attend(const dlk_paged_params p) {
    constexpr int FQ = sizeof(KT) == 4 ? 1 : QP; // the f32 instruction takes queries as they are
    constexpr int A = FEW ? Few<KT, HD, NT, FQ>::LDS : 0, B = MANY ? Many<KT, HD>::LDS : 0;
    __shared__ __attribute__((aligned(16))) char area[A > B ? A : B];
    const int block = static_cast<int>(blockIdx.x), many = p.lists[DLK_PAGED_MANY].count * p.KV;
    if constexpr (FEW && MANY) {
        if (block < many) attend_many<KT, HD, QP>(p, block, area);
        else attend_few<KT, HD, NT, FQ>(p, block - many, area);
    } else if constexpr (MANY) {
        attend_many<KT, HD, QP>(p, block, area);
    } else {
        attend_few<KT, HD, NT, FQ>(p, block, area);
    }
}

// ------------------------------------------------------------------------------------------------ the merge
// Joins the partials of a token's rows: those of the prefix that the batch shares, then those of its own run's splits.  16
// bytes a lane, so that a wave takes 256 / HD heads at once; W waves take the splits in turn, AHEAD of them asked for at once,
// rows and sums together.  Bound by the two round trips to memory (the record, the partials: 5 us in all), or by the partials'
// bytes (up to two of each of 3000 rows of 32 heads of 64: 17 us).
template <int HD, int W>
__global__ __launch_bounds__(kThreads) void paged_merge(const dlk_paged_params p) {
    constexpr int LANES = HD / 4, HEADS = kWave / LANES, AHEAD = 8;
    __shared__ float m_s[kWaves][HEADS], l_s[kWaves][HEADS];
    __shared__ f32x4 o_s[kWaves][kWave];
    const int t = threadIdx.x, lane = t % kWave, all = __builtin_amdgcn_readfirstlane(t / kWave), wave = all % W;
    const uint32_t groups = (p.H + HEADS - 1) / HEADS; // of heads
    const uint32_t unit = min(blockIdx.x * (kWaves / W) + all / W, p.merge_count * groups - 1);
    Planned<dlk_paged_merge>* merge = planned(p.merges) + unit / groups;
    const int token = merge->token, shared = p.shared_splits, count = shared + merge->count;
    const int h = min(static_cast<int>(unit % groups) * HEADS + lane / LANES, p.H - 1), G = p.H / p.KV;
    // where the row's first partials are, and how far apart
    const int64_t row = static_cast<int64_t>(h / G) * p.places + h % G, own_at = row + merge->slot, front_at = row + merge->shared_slot;
    const int64_t own_step = merge->stride, front_step = p.shared_stride;
    const int d = lane % LANES * 4;
    float M = kNoBase, L = 0.0f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int begin = wave; begin < count; begin += W * AHEAD) {
        float m[AHEAD], l[AHEAD];
        f32x4 x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = min(begin + W * k, count - 1);
            const bool in_front = i < shared;
            const int64_t at = in_front ? front_at + i * front_step : own_at + (i - shared) * own_step;
            m[k] = p.partial_ml[2 * at];
            l[k] = p.partial_ml[2 * at + 1];
            x[k] = *reinterpret_cast<const f32x4*>(p.partial_o + at * HD + d);
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) top = fmaxf(top, m[k]); // (repeated ones do not matter)
        const float keep = __builtin_amdgcn_exp2f(M - top);
        M = top;
        L *= keep;
        O *= keep;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (begin + W * k >= count) break;
            const float weight = __builtin_amdgcn_exp2f(m[k] - M);
            L += weight * l[k];
            O += weight * x[k];
        }
    }
    if constexpr (W > 1) {
        if (d == 0) {
            m_s[wave][lane / LANES] = M;
            l_s[wave][lane / LANES] = L;
        }
        o_s[wave][lane] = O;
        __syncthreads();
        if (wave != 0) return;
        L = 0.0f;
        O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, m_s[w][lane / LANES]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float weight = __builtin_amdgcn_exp2f(m_s[w][lane / LANES] - M);
            L += weight * l_s[w][lane / LANES];
            O += weight * o_s[w][lane];
        }
    }
    *reinterpret_cast<f32x4*>(p.out + (static_cast<int64_t>(token) * p.H + h) * HD + d) = O / L;
}

template <typename KT, int HD, int QP> int launch_items(const dlk_paged_params& p, hipStream_t stream) {
    const dlk_paged_list &few_list = p.lists[DLK_PAGED_FEW], &many_list = p.lists[DLK_PAGED_MANY];
    const int64_t blocks = (static_cast<int64_t>(few_list.count) + many_list.count) * p.KV;
    const int few = few_list.count > 0 ? few_list.rows : 0;
    const bool many = many_list.count > 0;
    if (blocks == 0) return 0;
    if (blocks > DLK_MOST_GROUPS || (few != 0 && few != 16 && few != 32) || (many && many_list.rows != 128)) return static_cast<int>(hipErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(blocks)), threads(kThreads);
    if (many && few == 32) hipLaunchKernelGGL((paged_attend<KT, HD, 2, QP, true, true>), grid, threads, 0, stream, p);
    else if (many && few == 16) hipLaunchKernelGGL((paged_attend<KT, HD, 1, QP, true, true>), grid, threads, 0, stream, p);
    else if (many) hipLaunchKernelGGL((paged_attend<KT, HD, 1, QP, false, true>), grid, threads, 0, stream, p);
    else if (few == 32) hipLaunchKernelGGL((paged_attend<KT, HD, 2, QP, true, false>), grid, threads, 0, stream, p);
    else hipLaunchKernelGGL((paged_attend<KT, HD, 1, QP, true, false>), grid, threads, 0, stream, p);
    return static_cast<int>(hipGetLastError());
}

// waves of a merge
int64_t merge_units(int64_t merges, int64_t H, int64_t hd) { return merges * ((H + 256 / hd - 1) / (256 / hd)); }

template <typename KT, int HD> int launch(const dlk_paged_params& p, hipStream_t stream) {
    const int status = p.q_bf16 ? launch_items<KT, HD, 1>(p, stream) : launch_items<KT, HD, 3>(p, stream);
    if (status != 0) return status;
    if (p.merge_count == 0) return 0;
    const int64_t units = merge_units(p.merge_count, p.H, HD);
    // up to 8 splits are one round trip of one wave, and more waves than a launch has are not needed
    if (p.merge_most <= 8 || units > DLK_MOST_GROUPS) hipLaunchKernelGGL((paged_merge<HD, 1>), dim3(static_cast<unsigned>((units + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, p);
    else hipLaunchKernelGGL((paged_merge<HD, kWaves>), dim3(static_cast<unsigned>(units)), dim3(kThreads), 0, stream, p);
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

extern "C" int dlk_paged_fits(int64_t items, int64_t merges, int H, int KV, int hd) {
    return items <= DLK_MOST_GROUPS / KV && dlk::merge_units(merges, H, hd) <= static_cast<int64_t>(DLK_MOST_GROUPS) * dlk::kWaves;
}

extern "C" int dlk_paged_attention(const dlk_paged_params* params, dlh_stream stream_handle) {
    const dlk_paged_params& p = *params;
    const int align = p.q_bf16 ? 8 : 4; // elements of 16 bytes
    if (p.KV <= 0 || p.H <= 0 || p.H % p.KV != 0 || p.page_shift < 4 || p.q_row % align != 0 || p.q_head % align != 0 ||
        reinterpret_cast<uintptr_t>(p.q) % 16 != 0 || (p.merge_count > 0 && !p.merges) ||
        !dlk_paged_fits(static_cast<int64_t>(p.lists[0].count) + p.lists[1].count, p.merge_count, p.H, p.KV, p.hd))
        return static_cast<int>(hipErrorInvalidValue);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_handle);
    return p.kv_bf16 ? dlk::launch_heads<uint16_t>(p, stream) : dlk::launch_heads<float>(p, stream);
}
