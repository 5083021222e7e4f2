// Attention of a few rows a sequence on the matrix units: 16 rows to a block, all of its waves at the keys.
//
// A tile of 64 keys is dealt out to the four waves, 16 keys each, and everything is computed transposed, as in rt_attention_tile.h, in 16 x 16 products:
//     S^T = K Q^T      lane l: query l % 16, keys 4 h .. 4 h + 3 of the wave's 16, h = l / 16
//     O^T += V^T P^T   over the wave's 16 keys, whose weights are in the registers that S^T was computed into
// so that a lane has four scores of a tile, where the tiles of 128 rows leave a single token's 64 scores to 32 registers of two lanes in a row of 32 and three waves idle: what
// is done to a score there (its cap takes 7 to 13 instructions) counts 8 times as much.  Every wave keeps its own m, l and O; they are joined in LDS when the block's keys are
// walked, and the block's part then goes the way of rt_attention_tile.h's.
//
// What bounds it: HBM.  bf16, 32 tokens of 200 to 6000 keys, 32 heads on 8 of 128, capped and biased: 107 us, 4.1 TB/s (a copy 4.9); in the tiles of 128 rows 130, with the cap
// or without.  Loads that do not stay in the L2s (at_to_lds<true>) 106, others 113.
#ifndef RT_ATTENTION_FEW_H
#define RT_ATTENTION_FEW_H

#include "rt_attention_tile.h"

typedef float v4f32 __attribute__((ext_vector_type(4)));
typedef _Float16 v4h16 __attribute__((ext_vector_type(4)));

constexpr uint32_t AF_ROWS = 16;

template <typename T, int DT> struct FewShape {
    static constexpr int CE = 16 / sizeof(T);                  // elements of a chunk
    static constexpr int STEPS = (DT + 4 * CE - 1) / (4 * CE); // groups of four chunks in a row
    static constexpr int BLOCKS = (DT + 15) / 16;              // 16-column blocks of the result
    static constexpr int KT = 64;
    static constexpr int CHUNKS = DT / CE;
    static constexpr int LOADS = (KT * CHUNKS + AT_BLOCK - 1) / AT_BLOCK;
    static constexpr int TILE = (KT * CHUNKS * 16 + 1023) / 1024 * 1024;
    static constexpr int LDS = 4 * TILE + 256;
};

template <typename T> struct AfMma;
template <> struct AfMma<half_t> {
    static __device__ __forceinline__ v4f32 qk(v4u k, v4u q, v4f32 s) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, k), __builtin_bit_cast(v8h, q), s, 0, 0, 0);
    }
    static __device__ __forceinline__ v4f32 pv(v2u v, v2u w, v4f32 o) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4h16, v), __builtin_bit_cast(v4h16, w), o, 0, 0, 0);
    }
};
template <> struct AfMma<bf16_t> {
    static __device__ __forceinline__ v4f32 qk(v4u k, v4u q, v4f32 s) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, k), __builtin_bit_cast(v8b, q), s, 0, 0, 0);
    }
    static __device__ __forceinline__ v4f32 pv(v2u v, v2u w, v4f32 o) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4s, v), __builtin_bit_cast(v4s, w), o, 0, 0, 0);
    }
};
template <> struct AfMma<float> {
    static __device__ __forceinline__ v4f32 one(float x, float y, v4f32 s) { return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, s, 0, 0, 0); }
};

// over the four lanes of a query, which are 16 apart
__device__ __forceinline__ float af_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, at_other(x));
}
__device__ __forceinline__ float af_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + at_other(x);
}
__device__ __forceinline__ void af_settle(float last) {
    at_in_order();
    asm volatile("" : : "s"(__builtin_amdgcn_readfirstlane(__float_as_uint(last))));
    at_in_order();
}

template <typename T, int DT, bool EXACT, bool PAGED>
__global__ void __launch_bounds__(AT_BLOCK) attention_few_kernel(AttnArgs a, AttnPartial part) {
    typedef FewShape<T, DT> S;
    constexpr int KT = S::KT, CE = S::CE;
    constexpr float LIFT = AT_LIFT<T, true>, LOWER = 1.0f / (1 << AT_LIFT<T, true>);
    extern __shared__ __align__(16) unsigned char smem[];
    lds_byte* const lds = (lds_byte*)smem;
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 16, quarter = lane / 16;
    const uint32_t D = EXACT ? DT : a.dim, chunks = D / CE, pitch = D * sizeof(T);

    // ---- which rows, which keys: as in attention_tile_kernel, 16 rows to a tile
    uint32_t b, g, tile, piece_at, piece, stride;
    if (PAGED) {
        stride = a.kv_heads;
        g = blockIdx.x % a.kv_heads;
        uint32_t at = blockIdx.x / a.kv_heads;
        piece = part.split ? __builtin_amdgcn_readfirstlane(at_piece<KT, true, true, AF_ROWS>(a)) : 0x7fffffffu;
        b = __builtin_amdgcn_readfirstlane(at_locate<KT, true, AF_ROWS>(a, piece, at));
        if (b >= a.seqs) return;
        tile = __builtin_amdgcn_readfirstlane(at);
        piece_at = 0;
    } else {
        const uint32_t pairs = stride = a.seqs * a.kv_heads, pair = blockIdx.x % pairs, at = blockIdx.x / pairs;
        b = pair / a.kv_heads;
        g = pair - b * a.kv_heads;
        piece = part.piece;
        tile = part.row_tiles - 1 - at / part.pieces;
        piece_at = at % part.pieces;
    }
    const AttnSeq s = at_seq<PAGED>(a, b);
    if (PAGED) {
        const uint32_t span = at_span<KT, true>(a, b, s), at = tile;
        piece = at_piece_of(piece, span);
        const uint32_t pieces = (span + piece - 1) / piece;
        tile = at / pieces;
        piece_at = at - tile * pieces;
        tile = at_row_tiles<AF_ROWS>(a, s) - 1 - tile;
    }
    const uint32_t all = s.count * a.group, row0 = tile * AF_ROWS, rows = all - row0 < AF_ROWS ? all - row0 : AF_ROWS;
    const AttnTexts texts = !PAGED ? at_texts(a, b) : AttnTexts{};
    const AttnWalk w = at_walk<KT, true>(a, texts, b, s, row0, rows);
    const uint32_t tile0 = piece_at * piece, tile1 = w.tiles - tile0 < piece || tile0 >= w.tiles ? w.tiles : tile0 + piece;
    const bool whole = w.tiles <= piece;
    if (tile0 >= w.tiles && piece_at > 0) return;
    if (!whole && blockIdx.x + (uint64_t)((w.tiles + piece - 1) / piece - 1 - piece_at) * stride >= gridDim.x) return;          // starts that decrease

    // ---- this lane's row
    const uint32_t row = row0 + (col < rows ? col : rows - 1), j = fd_div(row, a.group_div), h = g * a.group + (row - j * a.group);
    AttnRow me;
    if (!PAGED && a.documents) {
        const int32_t p_a = at_position(s, fd_div(row0, a.group_div)), p_z = at_position(s, fd_div(row0 + rows - 1, a.group_div));
        const uint32_t da = at_document(a, texts, b, p_a), dz = at_document(a, texts, b, p_z);
        me = at_in_document(a, texts, b, s, at_position(s, j), at_document_of(a, texts, b, at_position(s, j), da, dz));
    } else {
        me = at_in_text(a, at_position(s, j), 0, s.keys, a.prefix ? a.prefix[b] : 0);
    }
    const float slope = a.slopes ? at_slope(a, h) : 0.0f;

    v4u q[S::STEPS];
    {
        const T* from = (const T*)a.q + b * a.q_b + h * a.q_h + (uint64_t)(s.first + j) * a.q_t;
        const uint32_t flip = a.c < 0.0f ? AtMma<T>::SIGNS : 0;
#pragma unroll
        for (int i = 0; i < S::STEPS; i++) {
            q[i] = v4u{0, 0, 0, 0};
            if ((4 * i + quarter) * CE < D) q[i] = *(const v4u*)(from + (4 * i + quarter) * CE);
            q[i] ^= v4u{flip, flip, flip, flip};
        }
    }
    const bool changed = a.most != 0.0f || a.slopes;
    const float c = changed ? 1.0f : fmaxf(__builtin_fabsf(a.c), 1e-37f);

    // ---- this lane's part of a tile's loads
    uint32_t l_row[S::LOADS], l_k[S::LOADS], l_v[S::LOADS];
    const uint32_t slots = KT * chunks, loads = (slots + 63) / 64;
#pragma unroll
    for (int i = 0; i < S::LOADS; i++) {
        uint32_t slot = (i * AT_WAVES + wave) * 64 + lane;
        slot = slot < slots ? slot : slots - 1;
        const uint32_t rr = slot / chunks, cc = slot - rr * chunks;
        const uint32_t tk = at_turn_k(rr, chunks), tv = at_turn_v<T>(rr, chunks);
        l_row[i] = rr;
        l_k[i] = (cc >= tk ? cc - tk : cc + chunks - tk) * 16;
        l_v[i] = (cc >= tv ? cc - tv : cc + chunks - tv) * 16;
    }
    const unsigned char* kb = (const unsigned char*)a.k + (g * a.k_h + (PAGED ? 0 : b * a.k_b)) * sizeof(T);
    const unsigned char* vb = (const unsigned char*)a.v + (g * a.v_h + (PAGED ? 0 : b * a.v_b)) * sizeof(T);
    const uint64_t k_row = a.k_t * sizeof(T), v_row = a.v_t * sizeof(T), k_page = PAGED ? a.k_b * sizeof(T) : 0;
    auto start_of = [&](uint32_t n) -> int32_t { return n < w.head ? (PAGED ? 0 : w.start) + (int32_t)(n * KT) : w.from + (int32_t)((n - w.head) * KT); };
    // the rows of this lane's chunks of a tile: keys beyond the last are that one, those without a page lie in page 0
    auto look = [&](uint32_t n, uint32_t& slot) -> int32_t {
        int32_t t = start_of(n) + (int32_t)lane;
        t = t < s.keys ? t : s.keys - 1;
        return at_page(a, b, (uint32_t)t, slot);
    };
    auto fetch = [&](uint32_t n, lds_byte* to, int32_t page, uint32_t slot) __attribute__((always_inline)) {
        const int32_t t0 = start_of(n);
        to += wave * 1024;
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) {
            uint64_t ko, vo;
            if (PAGED) {
                int32_t pg = __shfl(page, (int)l_row[i]);
                const uint32_t sl = (uint32_t)__shfl((int)slot, (int)l_row[i]);
                pg = pg < 0 ? 0 : pg;
                ko = vo = (uint64_t)(uint32_t)pg * k_page + sl * k_row;
            } else {
                int32_t t = t0 + (int32_t)l_row[i];
                t = t < s.keys ? t : s.keys - 1;
                ko = (uint64_t)(uint32_t)t * k_row;
                vo = (uint64_t)(uint32_t)t * v_row;
            }
            if (i * AT_WAVES + wave >= loads) break;
            at_to_lds<true>(kb + ko + l_k[i], to + i * AT_WAVES * 1024);
            at_to_lds<true>(vb + vo + l_v[i], to + i * AT_WAVES * 1024 + S::TILE);
        }
    };

    // ---- where this lane reads a tile: a chunk of key 16 wave + col; of keys 16 wave + 4 quarter .. + 3 the columns of a block
    uint32_t k_at[S::STEPS], v_at[S::BLOCKS];
    const uint32_t k_key = 16 * wave + col;
#pragma unroll
    for (int i = 0; i < S::STEPS; i++) {
        uint32_t cc = 4 * i + quarter;
        cc = cc < chunks ? cc : 0;                              // beyond the row: replaced by 0 below
        cc += at_turn_k(k_key, chunks);
        k_at[i] = k_key * pitch + (cc >= chunks ? cc - chunks : cc) * 16;
    }
    const uint32_t v_key = 16 * wave + 4 * quarter + (sizeof(T) == 2 ? col / 4 : 0);
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++) {
        if (sizeof(T) == 2) {                                   // lane 4 r + x of each 16 gives the address of four of row r's columns
            uint32_t cc = 2 * i + (lane % 4) / 2;
            if (cc >= chunks) cc = 0;                           // columns of nobody
            cc += at_turn_v<T>(v_key, chunks);
            if (cc >= chunks) cc -= chunks;
            v_at[i] = S::TILE + v_key * pitch + cc * 16 + (lane % 2) * 8;
        } else {
            v_at[i] = S::TILE + v_key * pitch + (i * 16 + col < D ? i * 16 + col : 0) * 4;
        }
    }

    v4f32 o[S::BLOCKS];
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++) o[i] = v4f32{0};
    float m = -INFINITY, l = 0.0f;                              // of this wave's keys; l: of this lane's

    // All products of a tile, also those of columns beyond the rows' (of zeros, and to columns of nobody), so that no branch lies between a product and the next read of its sum:
    // there the compiler counts the wait states of one way round only, and rows of 8 and 16 columns lost their last tile's fourth columns
    auto step = [&](uint32_t n, const lds_byte* cur, uint64_t there) __attribute__((always_inline)) {
        const int32_t t0 = start_of(n) + (int32_t)(16 * wave), t1 = t0 + 4 * (int32_t)quarter;       // this wave's first key, this lane's
        v4f32 x = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < S::STEPS; i++) {
            v4u k = at_lds16(cur + k_at[i]);
            if ((EXACT ? DT % (4 * CE) != 0 : true) && (4 * i + 4) * CE > (int)D && (4 * i + quarter) * CE >= D) k = v4u{0, 0, 0, 0};
            if constexpr (sizeof(T) == 2) {
                x = AfMma<T>::qk(k, q[i], x);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) x = AfMma<T>::one(__uint_as_float(k[e]), __uint_as_float(q[i][e]), x);
            }
        }
        af_settle(x[3]);
        if (changed) {
            if (a.most != 0.0f) {
                const float most_in = __builtin_fabsf(a.most_in);
                if (sizeof(T) == 4 || a.most > AT_COARSE) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float y = x[e] * most_in;
                        if (sizeof(T) == 2) asm volatile("" : "+v"(y));   // shares nothing with the others
                        x[e] = at_capped<T, true>(a.most, y);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = at_capped<T, false>(a.most, x[e] * most_in);
                }
            } else {
                const float cc = __builtin_fabsf(a.c);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] *= cc;
            }
            if (a.slopes) {
                const float far = (float)(me.p - t1);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(-slope, __builtin_fabsf(far - (float)e), x[e]);
            }
        }
        const uint32_t have = (uint32_t)(there >> (16 * wave + 4 * quarter));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int32_t t = t1 + e;
            const bool seen = t <= me.limit && t >= me.lo && (me.p - t < a.window || t < me.front) && (!PAGED || (have >> e) & 1);
            x[e] = seen ? x[e] : -INFINITY;
        }
        const float top = af_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))) * c;
        if (__ballot(top > m)) {
            const float m_new = fmaxf(m, top), old = at_exp2(m - (m_new == -INFINITY ? 0.0f : m_new));
            m = m_new;
            l *= old;
#pragma unroll
            for (int i = 0; i < S::BLOCKS; i++) o[i] *= old;
        }
        const float base = m == -INFINITY ? 0.0f : m - LIFT;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] = at_exp2(__builtin_fmaf(x[e], c, -base));
            l += x[e];
        }
        if constexpr (sizeof(T) == 2) {
            const v2u weights = {AtMma<T>::pack(x[0], x[1]), AtMma<T>::pack(x[2], x[3])};
#pragma unroll
            for (int i = 0; i < S::BLOCKS; i++)
                o[i] = AfMma<T>::pv(at_lds_turned(cur + v_at[i]), weights, o[i]);
        } else {
#pragma unroll
            for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i] = AfMma<T>::one(at_lds4(cur + (v_at[i] + e * pitch)), x[e], o[i]);
        }
    };

    int32_t page = 0, page1 = 0;                                // of key `lane` of the tile that is loaded next, and of the one after
    uint32_t slot = 0, slot1 = 0;
    uint64_t there = ~0ull, there1 = ~0ull;                     // keys that have a page: of the tile at hand, of the next
    if (tile0 < tile1) {
        if (PAGED) {
            page = look(tile0, slot);
            there1 = __ballot(page >= 0);
        }
        fetch(tile0, lds, page, slot);
        if (PAGED && tile0 + 1 < tile1) page1 = look(tile0 + 1, slot1);
    }
    auto turn = [&](uint32_t n, lds_byte* next, const lds_byte* cur) __attribute__((always_inline)) {
        there = there1;
        page = page1;
        slot = slot1;
        if (PAGED) there1 = __ballot(page >= 0);
        at_wait_memory();                                       // this wave's loads have arrived
        __syncthreads();                                        // and everyone's; and everyone is done with the other stage
        if (n + 1 < tile1) fetch(n + 1, next, page, slot);
        if (PAGED && n + 2 < tile1) page1 = look(n + 2, slot1);
        step(n, cur, there);
    };
    for (uint32_t n = tile0; n < tile1; n += 2) {
        turn(n, lds + 2 * S::TILE, lds);
        if (n + 1 < tile1) turn(n + 1, lds, lds + 2 * S::TILE);
    }

    // ---- the waves' results joined: O^T of each as [row][column], m and l behind
    af_settle(o[S::BLOCKS - 1][3]);
    l = af_sum(l);
    const uint32_t width = D + 2;
    float* const mine = (float*)smem + (wave * AF_ROWS + col) * width;
    __syncthreads();                                            // everyone is done with the tiles
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t d = 16 * i + 4 * quarter + e;
            if (d < D) mine[d] = o[i][e];
        }
    if (quarter == 0) {
        mine[D] = m;
        mine[D + 1] = l;
    }
    __syncthreads();
    // 16 threads to a row
    const uint32_t r = threadIdx.x / 16, x16 = threadIdx.x % 16;
    const float* const from = (const float*)smem + r * width;
    float factor[AT_WAVES], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (uint32_t n = 0; n < AT_WAVES; n++) top = fmaxf(top, from[n * AF_ROWS * width + D]);
#pragma unroll
    for (uint32_t n = 0; n < AT_WAVES; n++) {
        factor[n] = at_exp2(from[n * AF_ROWS * width + D] - (top == -INFINITY ? 0.0f : top));
        sum = __builtin_fmaf(factor[n], from[n * AF_ROWS * width + D + 1], sum);
    }
    const uint32_t rj = fd_div(row0 + (r < rows ? r : rows - 1), a.group_div), rh = g * a.group + (row0 + (r < rows ? r : rows - 1) - rj * a.group);
    const float inv = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : LOWER;
    const uint64_t part_at = (uint64_t)blockIdx.x * AF_ROWS + r;
    T* const y = (T*)a.y + b * a.y_b + rh * a.y_h + (uint64_t)(s.first + rj) * a.y_t;
    bool fine = __builtin_isfinite(sum) && top < INFINITY;
    for (uint32_t d = 4 * x16; d < D; d += 64) {
        float out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t n = 0; n < AT_WAVES; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = __builtin_fmaf(factor[n], from[n * AF_ROWS * width + d + e], out[e]);
#pragma unroll
        for (int e = 0; e < 4; e++) fine = fine && __builtin_isfinite(out[e]);
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] *= inv;
        if (r >= rows) continue;
        if (!whole) {
            at_leave(part.o + part_at * D + d, out[0], out[1]);
            at_leave(part.o + part_at * D + d + 2, out[2], out[3]);
        } else if constexpr (sizeof(T) == 2) {
            *(v2u*)(y + d) = v2u{AtMma<T>::pack(out[0], out[1]), AtMma<T>::pack(out[2], out[3])};
        } else {
            *(v4f32*)(y + d) = v4f32{out[0], out[1], out[2], out[3]};
        }
    }
    if (r < rows && x16 == 0) {
        if (!whole) at_leave(part.ml + 2 * part_at, top, sum * LOWER);
        else if (a.lse) a.lse[b * a.l_b + rh * a.l_h + (uint64_t)(s.first + rj) * a.l_t] = at_lse(top, sum * LOWER);
    }
    // a row whose result is not finite is computed again, over its visible keys alone
    const uint64_t bad = __ballot(r < rows && !fine);
    for (uint32_t n = 0; n < 4; n++) {                          // this wave's rows
        const uint32_t again = wave * 4 + n;
        if (!((bad >> (16 * n)) & 0xffff)) continue;
        at_wait_memory();                                       // what was written of it first has been
        at_again<T, DT, PAGED, KT, true, true>(a, part, b, g, s, w, tile0, tile1, row0 + again, (uint64_t)blockIdx.x * AF_ROWS + again, whole);
    }
    if (whole) return;
    const uint32_t used = (w.tiles + piece - 1) / piece, first = blockIdx.x - piece_at * stride;
    if (at_last(part.arrivals + first, used, (volatile uint32_t*)(smem + S::LDS - 16)))
        at_join<T, true, AF_ROWS>(a, part, s, b, g, row0, 0, rows, first, stride, used, (float*)smem);
}

// One token to a sequence on average, and no more rows of a KV head than a tile's; tiles that LDS holds.  bf16, 32 heads on 8 of 128, cap and bias, us here | in tiles of 128 rows:
// a token to each of 64 sequences of 300 keys 35 | 39, of 1500 82 | 96; of 256 91 | 104 and 275 | 324; of 512 200 | 225 and 570 | 664.  The host knows no more of the tokens than their
// number, so one sequence may have them all, whose row tiles then walk the same keys: 64 tokens of 1000 keys 24 | 44, of 8000 85 | 178; 128 41 | 49 and 144 | 175; 256 71 | 66 and
// 267 | 184 (260 with loads that stay in the L2s); 512 123 | 138 and 511 | 239.
template <typename T> bool at_fits_few(const AttnArgs& a, bool paged) {
    return a.group <= AF_ROWS && (paged ? a.tokens <= a.seqs : (uint64_t)a.tokens * a.group <= AF_ROWS) && a.dim * sizeof(T) <= 512;
}

template <typename T, int DT, bool EXACT, bool PAGED> int at_launch_few(rt_device* dev, AttnArgs& a, bool* done) {
    typedef FewShape<T, DT> S;
    AttnPartial part = {};
    const uint64_t most_blocks = AT_MOST_PARTS / (AF_ROWS * ((uint64_t)a.dim + 2) * sizeof(float)), per = PAGED ? a.kv_heads : (uint64_t)a.seqs * a.kv_heads;
    uint64_t items;
    if (PAGED) {
        const uint64_t tiles = ((uint64_t)a.tokens * a.group) / AF_ROWS + a.seqs;
        items = tiles + AT_TARGET_FEW / a.kv_heads + 1;         // as in at_launch_tile
        part.split = a.cap > AT_LEAST_TILES_FEW * S::KT && items * per <= RT_ARRIVALS && items * per <= most_blocks;
        if (!part.split) items = tiles;
    } else {
        part.row_tiles = 1;
        uint64_t span = (a.cap + S::KT - 1) / S::KT;
        if (a.window != AT_FAR && !a.documents && !a.prefix) {
            const uint64_t w = ((uint64_t)a.window + AT_ROWS) / S::KT + 2 + ((uint64_t)a.sinks + S::KT - 1) / S::KT;
            span = w < span ? w : span;
        }
        uint64_t piece = at_piece_for<true, AF_ROWS>(per, span * per);
        piece = at_piece_of((uint32_t)(piece > span ? span : piece), (uint32_t)span);
        if ((span + piece - 1) / piece * per > (most_blocks < RT_ARRIVALS ? most_blocks : RT_ARRIVALS)) piece = span;
        part.piece = (uint32_t)piece;
        part.pieces = (uint32_t)((span + piece - 1) / piece);
        part.split = part.pieces > 1;
        items = part.pieces;
    }
    const uint64_t blocks = items * per;
    *done = blocks <= AT_MOST_BLOCKS;
    if (!*done) return RT_OK;
    const size_t row_count = part.split ? (size_t)blocks * AF_ROWS : 0;
    void* p = nullptr;
    int rc = at_workspace(dev, a, row_count * ((size_t)a.dim + 2) * sizeof(float), &p);
    if (rc) return rc;
    part.ml = (float*)p;
    part.o = part.ml + 2 * row_count;
    part.arrivals = dev->arrivals;
    const auto kernel = attention_few_kernel<T, DT, EXACT, PAGED>;
    static_assert(S::LDS <= 160 * 1024 && AT_WAVES * AF_ROWS * (DT + 2) * 4 <= S::LDS - 16 && AT_MOST_PIECES * AF_ROWS * 4 <= S::LDS - 16, "LDS");
    static bool raised[16] = {};                                // per GPU; setting it twice does no harm
    if (S::LDS > 64 * 1024 && !(dev->ordinal < 16 && raised[dev->ordinal])) {
        RT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS));
        if (dev->ordinal < 16) raised[dev->ordinal] = true;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(AT_BLOCK), S::LDS, dev->stream, a, part);
    RT_CHECK_LAUNCH("attention_few_kernel");
    return RT_OK;
}

template <typename T> int at_dispatch_few(rt_device* dev, AttnArgs& a, bool paged, bool* done) {
#define RT_FEW(DT, EXACT) return paged ? at_launch_few<T, DT, EXACT, true>(dev, a, done) : at_launch_few<T, DT, EXACT, false>(dev, a, done)
    if (a.dim == 64) RT_FEW(64, true);
    if (a.dim == 80) RT_FEW(80, true);
    if (a.dim == 96) RT_FEW(96, true);
    if (a.dim == 128) RT_FEW(128, true);
    if (a.dim < 64) RT_FEW(64, false);
    if (a.dim < 128) RT_FEW(128, false);
    if constexpr (sizeof(T) == 2) {
        if (a.dim == 256) RT_FEW(256, true);
        RT_FEW(256, false);
    }
    *done = false;
    return RT_OK;
#undef RT_FEW
}

#endif
