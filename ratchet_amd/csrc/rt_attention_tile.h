// Attention on the matrix units: 128 query rows to a block, 32 to a wave, the keys in tiles through LDS.
//
// A row is a (token, head of the group) pair, so the heads that share a KV head share its tiles.  Everything is computed transposed, with the queries
// along the columns of the 32 x 32 products:
//     S^T = K Q^T      K from LDS (16-byte chunks of a key's row), Q in registers for the whole walk
//     O^T += V^T P^T   V^T read transposed from LDS, P^T the registers that S^T was computed into
// In the products' layout lane l holds column l % 32 and, of every 8 rows, the 4 at 4 * (l / 32): a query's scores lie in two lanes, so
// its maximum and sum are a walk over registers and one exchange.  The operand layout of P^T (8 keys a lane and step) is that of the S^T registers
// if the 16 keys of a step are taken in the order {4h..4h+3, 8+4h..8+4h+3}, h = l / 32, and any order will do as long as V^T is read in the same one.
//
// What hidden keys hold is kept out of the scores by a select and out of the maxima and sums by that; their values meet a weight of 0, and 0 times
// what is not finite is NaN, which stays.  So a row tile whose result is not finite is computed again, one row at a time, over the visible keys only.
//
// Roundings below f32: the weights of 16-bit types are rounded to the type for the second product, as its operands have to be (their f32 values make the sums);
// everything else, scores, m, l and O, is f32.  An m that lags by up to AT_SLACK powers of two makes weights up to 2^8: rounded relative to themselves.  f16's small numbers
// are not: they end at 2^-24, and thousands of keys below that against the row's largest can be most of a result.  f16 weights are therefore held 2^AT_LIFT larger,
// to 2^14 at most (f16's largest is 2^16; scores beyond 2^24, whose own rounding may pass that, make a row that is computed again): relative to the largest they
// go down to 2^-30 at least, where rows are few to 2^-38.  l and O carry the same factor until the row is finished or its part is left.
//
// What bounds it, by counters: 8192 tokens of 32 heads of 96 with a window of 2047, bf16: 227 to 244 us, 745 to 800 TFLOP/s of the visible pairs' products; the
// matrix units are busy 47 % and the vector units (scores to weights: six to seven instructions each, by the counters) 62 % of the time, and three waves of a SIMD have both overlap
// only in part.  f32, [4,6,1500,64]: 154 us, 79 % of it the matrix units, whose f32 products do an eighth of the 16-bit ones' work.  Single tokens, 64 of about
// 4600 keys in bf16: 242 us, the keys and values once at 5.0 TB/s; a copy reaches 5.2.
//
// Changed scores are vector instructions on top: f16, 4096 tokens of 16 heads on 8 of 256 with a window of 2048, capped, 225 us; bf16, 2048 tokens of 32 heads of 128, biased by
// distance 63, plain 54; 12 texts in 8192 tokens of 32 heads on 8 of 128 116, of which about 40 are what four rounds of blocks take whatever their keys.
#ifndef RT_ATTENTION_TILE_H
#define RT_ATTENTION_TILE_H

#include "rt_attention.h"
#include "rt_attention_order.h"

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

constexpr uint32_t AT_ROWS = 128, AT_WAVES = 4, AT_BLOCK = 64 * AT_WAVES;
constexpr int AT_SLACK = 8;                      // powers of two that a row's weights may lie above its m
template <typename T, bool FEW> constexpr int AT_LIFT = 0;
template <> inline constexpr int AT_LIFT<half_t, false> = 14 - AT_SLACK;
template <> inline constexpr int AT_LIFT<half_t, true> = 14;
// How far the keys of row tiles are shared out over blocks.  Single tokens (FEW): to AT_TARGET_FEW items, in pieces of no fewer than two tiles, which costs little as
// their parts are small (one token's 2051 keys 17.9 us, with four tiles at least 19.3; 16 tokens 53 us at 1024 items, 61 at 512, 58 at 2048; 64 ragged
// ones 255, 277, 251).  Others leave and join 64 KB a row tile and piece: only where the row tiles do not fill the chip by themselves (AT_ENOUGH), and to
// AT_TARGET items (Phi-2 prompt, 512 row tiles: 45 us whole, 55 to 57 shared out; chunks, 320 row tiles: 152 us at 256 items, 125 at 768, 142 at 1536;
// encoder, 288: 202, 149, 140).
constexpr uint32_t AT_TARGET_FEW = 1024, AT_TARGET = 768, AT_ENOUGH = 512, AT_LEAST_TILES_FEW = 2, AT_LEAST_TILES = 4;
// Blocks of 16 rows of 128 columns that the chip holds at once, two a CU.  Four sequences of up to 6000 keys, 8 KV heads: 22 us in one round of pieces of four tiles, 31 in two of
// pieces of two; one of 1000 keys 13 us in pieces of two, 17 of four; of 6000 20 and 19
constexpr uint32_t AT_AT_ONCE = 512;
constexpr uint32_t AT_SHORT = 40;                // tiles of keys to a row tile
constexpr size_t AT_MOST_PARTS = 1u << 30;       // bytes of parts; a launch that would leave more shares nothing out
constexpr uint32_t AT_MOST_PIECES = 60;          // of a row tile: their factors for its 128 rows fit the LDS of the smallest tiles
// Rows of a sequence and KV head, on average, up to which a launch joins its own pieces.  The average, as the rows of each are known on the device alone: a step of 60 tokens
// and one piece of a prompt is then few rows as well.  It is the faster for it (us, as few rows | as many: bf16, 32 heads on 8 of 128, up to 8000 keys, a piece of 60 tokens
// 219 | 225, of 180 231 | 281; f32, up to 4000 keys, 180 487 | 760; 32 heads of 80, up to 2000 keys, 700 171 | 198) but for short caches (up to 400 keys, 180 42 | 36; 8
// sequences, 25 64 | 55) and received weights, whose scores are then added up row after row (180 395 | 327; 700 563 | 412).
constexpr uint32_t AT_FEW_ROWS = 16;
constexpr uint32_t AT_JOIN_ROWS = 16;            // rows to a block of the joining kernel
constexpr uint64_t AT_MOST_BLOCKS = (1u << 24) - 1;   // of a launch, which has fewer than 2^32 threads; more rows go to the kernel for any

// ------------------------------------------------------------------------------------------------- who does what
// Tiles of KT keys that a tile of rows of sequence s may see at most; 1 where there are no keys, for the block that writes the zeros
template <int KT, bool SCORED> __device__ __forceinline__ uint32_t at_span(const AttnArgs& a, uint32_t b, const AttnSeq& s) {
    uint32_t n = ((uint32_t)s.keys + KT - 1) / KT;
    if (a.window != AT_FAR) {
        int32_t front = a.sinks;
        if (SCORED && a.prefix && a.prefix[b] > front) front = a.prefix[b];
        const uint64_t w = ((uint64_t)a.window + AT_ROWS) / KT + 2 + ((uint64_t)front + KT - 1) / KT;
        n = w < n ? (uint32_t)w : n;
    }
    return n ? n : 1;
}
template <uint32_t ROWS> __device__ __forceinline__ uint32_t at_row_tiles(const AttnArgs& a, const AttnSeq& s) { return (s.count * a.group + ROWS - 1) / ROWS; }

template <typename T> __device__ __forceinline__ T at_wave_sum(T x) {
#pragma unroll
    for (int i = 32; i; i >>= 1) x += __shfl_xor(x, i);
    return x;
}

// Tiles in a piece of the keys, for `tiles` row tiles in all that have `work` tiles of keys to walk
template <bool FEW, uint32_t ROWS> __host__ __device__ __forceinline__ uint32_t at_piece_for(uint64_t tiles, uint64_t work) {
    if (!FEW && tiles >= AT_ENOUGH) return 0x7fffffffu;
    constexpr uint32_t target = FEW ? AT_TARGET_FEW : AT_TARGET, least = FEW ? AT_LEAST_TILES_FEW : AT_LEAST_TILES;
    uint64_t n = (work + target - 1) / target;
    if (ROWS != AT_ROWS && n < 4) {                             // blocks of 16 rows: as many as the chip holds at once, while that asks for no more than four tiles
        const uint64_t once = (work + AT_AT_ONCE - 1) / AT_AT_ONCE;
        n = once < 4 ? once : 4;
    }
    return n < least ? least : n > 0x7fffffffu ? 0x7fffffffu : (uint32_t)n;
}
// The same from the device's lengths; the same in every wave.
template <int KT, bool FEW, bool SCORED, uint32_t ROWS> __device__ __forceinline__ uint32_t at_piece(const AttnArgs& a) {
    uint64_t work = 0;
    uint32_t tiles = 0;
    for (uint32_t b = __lane_id(); b < a.seqs; b += 64) {
        const AttnSeq s = at_seq<true>(a, b);
        const uint32_t span = at_span<KT, SCORED>(a, b, s), less = FEW ? 0 : s.count / (2 * KT);           // causal: the middle row of the new ones lacks half of them
        work += (uint64_t)at_row_tiles<ROWS>(a, s) * (span > 2 * less ? span - less : (span + 1) / 2);
        tiles += at_row_tiles<ROWS>(a, s);
    }
    return at_piece_for<FEW, ROWS>((uint64_t)at_wave_sum(tiles) * a.kv_heads, at_wave_sum(work) * a.kv_heads);
}
// ... and in a piece of this sequence's: pieces of the same size
__host__ __device__ __forceinline__ uint32_t at_piece_of(uint32_t piece, uint32_t span) {
    uint32_t n = (span + piece - 1) / piece;
    n = n < AT_MOST_PIECES ? n : AT_MOST_PIECES;
    return (span + n - 1) / n;
}

// Sequence b's items are numbered row tile by row tile, at_items of them, after those of the sequences before it.
template <int KT, bool SCORED, uint32_t ROWS> __device__ __forceinline__ uint32_t at_items(const AttnArgs& a, uint32_t b, uint32_t piece) {
    const AttnSeq s = at_seq<true>(a, b);
    const uint32_t span = at_span<KT, SCORED>(a, b, s), n = at_piece_of(piece, span);
    return at_row_tiles<ROWS>(a, s) * ((span + n - 1) / n);
}
// The sequence that item `at` belongs to (a.seqs: none); `at` becomes its number there.  All lanes of a wave take part.
template <int KT, bool SCORED, uint32_t ROWS> __device__ __forceinline__ uint32_t at_locate(const AttnArgs& a, uint32_t piece, uint32_t& at) {
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.seqs; b0 += 64) {
        const uint32_t b = b0 + __lane_id(), n = b < a.seqs ? at_items<KT, SCORED, ROWS>(a, b, piece) : 0;
        uint32_t sum = n;                                       // of this lane and those below
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) {
            const uint32_t x = __shfl_up(sum, i);
            if ((int)__lane_id() >= i) sum += x;
        }
        const uint64_t holds = __ballot(at >= before + sum - n && at < before + sum);
        if (holds) {
            const int lane = __builtin_ctzll(holds);
            at -= before + __shfl(sum, lane) - __shfl(n, lane);
            return b0 + lane;
        }
        before += __shfl(sum, 63);
    }
    return a.seqs;
}
template <int KT, bool SCORED, uint32_t ROWS> __device__ __forceinline__ uint32_t at_before(const AttnArgs& a, uint32_t piece, uint32_t until) {
    uint32_t sum = 0;
    for (uint32_t b = __lane_id(); b < until; b += 64) sum += at_items<KT, SCORED, ROWS>(a, b, piece);
    return at_wave_sum(sum);
}

// A row tile's walk over the keys: `tiles` of them, the first `head` from key `start` on, the others from key `from` on
struct AttnWalk {
    uint32_t tiles, head;
    int32_t start, from;
};
template <int KT, bool SCORED> __device__ __forceinline__ AttnWalk at_walk(const AttnArgs& a, const AttnTexts& texts, uint32_t b, const AttnSeq& s, uint32_t row0, uint32_t rows) {
    const uint32_t j0 = fd_div(row0, a.group_div), j1 = fd_div(row0 + rows - 1, a.group_div);
    AttnRow r0 = at_row<SCORED>(a, texts, b, s, j0);
    int32_t last = at_row<SCORED>(a, texts, b, s, j1).limit;
    if (SCORED) {                                               // the same in all lanes, which the compiler cannot know
        r0.p = __builtin_amdgcn_readfirstlane(r0.p);
        r0.lo = __builtin_amdgcn_readfirstlane(r0.lo);
        r0.front = __builtin_amdgcn_readfirstlane(r0.front);
        last = __builtin_amdgcn_readfirstlane(last);
    }
    const int32_t start = SCORED ? r0.lo / KT * KT : 0;
    AttnWalk w = {0, 0, start, start};
    if (last < r0.lo) return w;
    if (a.window != AT_FAR) {
        // the first key of the first row's window; what later texts of the tile keep in front lies behind it
        const int32_t first = r0.p - a.window + 1;
        const int32_t from = first > r0.lo ? first / KT * KT : start;
        const int32_t front = r0.front < from ? r0.front : from;
        const uint32_t head = front > start ? ((uint32_t)(front - start) + KT - 1) / KT : 0;
        if (start + (int32_t)(head * KT) < from) {
            w.head = head;
            w.from = from;
            if (from > last) {                                  // rows beyond the last key there is room for: only the front is left
                const uint32_t most = (uint32_t)(last - start) / KT + 1;
                w.tiles = head < most ? head : most;
                return w;
            }
        }
    }
    w.tiles = w.head + (uint32_t)(last - w.from) / KT + 1;
    return w;
}

// ----------------------------------------------------------------------------------------------------- elements
template <typename T> struct AtMma;
template <> struct AtMma<half_t> {
    static __device__ __forceinline__ v16f qk(v4u k, v4u q, v16f s) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, k), __builtin_bit_cast(v8h, q), s, 0, 0, 0);
    }
    // round to nearest even, as all roundings here
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        typedef _Float16 v2h __attribute__((ext_vector_type(2)));
        const v2h p = {(_Float16)x, (_Float16)y};
        return __builtin_bit_cast(uint32_t, p);
    }
    static constexpr uint32_t SIGNS = 0x80008000u;
};
template <> struct AtMma<bf16_t> {
    static __device__ __forceinline__ v16f qk(v4u k, v4u q, v16f s) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, k), __builtin_bit_cast(v8b, q), s, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        // not written as an instruction: one that reads an exponential has to keep a state away from it, which the compiler sees to only for its own
        typedef __bf16 v2b __attribute__((ext_vector_type(2)));
        typedef float v2f __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{x, y}), v2b));
    }
    static constexpr uint32_t SIGNS = 0x80008000u;
};
template <> struct AtMma<float> {
    static __device__ __forceinline__ v16f one(uint32_t k, uint32_t q, v16f s) {
        return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k), __uint_as_float(q), s, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float, float) { return 0; }
    static constexpr uint32_t SIGNS = 0x80000000u;
};

// The products of a pair of chunks, added to a score's SUMS sums: s and the others
template <typename T, int SUMS> __device__ __forceinline__ void at_score(v4u k, v4u q, v16f& s, v16f (&others)[SUMS]) {
    if constexpr (sizeof(T) == 2) {
        s = AtMma<T>::qk(k, q, s);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (e % SUMS == 0) s = AtMma<T>::one(k[e], q[e], s);
            else others[e % SUMS] = AtMma<T>::one(k[e], q[e], others[e % SUMS]);
        }
    }
}
template <int SUMS> __device__ __forceinline__ void at_join_sums(v16f& s, v16f (&others)[SUMS]) {
    if constexpr (SUMS == 4) s = (s + others[1]) + (others[2] + others[3]);
    if constexpr (SUMS == 2) s = s + others[1];
}

typedef __attribute__((address_space(3))) unsigned char lds_byte;
__device__ __forceinline__ v4u at_lds16(const lds_byte* at) { return *(const __attribute__((address_space(3))) v4u*)at; }
__device__ __forceinline__ float at_lds4(const lds_byte* at) { return *(const __attribute__((address_space(3))) float*)at; }
// Lane i of each 16 gives the address of 4 elements and receives, of the 4 rows that lanes 4r .. 4r + 3 address, column i
__device__ __forceinline__ v2u at_lds_turned(const lds_byte* at) {
    return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)const_cast<lds_byte*>(at)));
}
// 16 bytes a lane from memory to LDS, lane i's to at + 16 i (at: the same in all lanes).  Whoever reads them waits for vmcnt(0) first.  Written as an instruction, which
// has no result the compiler could misplace: after the builtin the compiler holds every LDS read for a possible flat access in flight, and waits
// for all reads where it needs one (s_waitcnt lgkmcnt(0) before each product).
template <bool ONCE = false> __device__ __forceinline__ void at_to_lds(const void* from, lds_byte* at) {
    if (ONCE) asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(from), "{m0}"((uint32_t)(uintptr_t)at) : "memory");
    else asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"((uint32_t)(uintptr_t)at) : "memory");
}
// The same with a base that all lanes share.  s_nop 4: a scalar register that a vector instruction wrote (v_readlane) may be read five states later.
__device__ __forceinline__ void at_to_lds(const void* base, uint32_t offset, lds_byte* at) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"((uint32_t)(uintptr_t)at) : "memory");
}
__device__ __forceinline__ void at_wait_memory() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// x and the other half's value of the same column
__device__ __forceinline__ float at_other(float x) {
    typedef unsigned int v2 __attribute__((ext_vector_type(2)));
    const v2 r = __builtin_bit_cast(v2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return __uint_as_float(__lane_id() < 32 ? r[1] : r[0]);
}

// ------------------------------------------------------------------------------------------------------- shape
// Head dims up to DT columns; EXACT: DT itself, known to the compiler.  WIDE: 64 keys to a tile whatever the columns: half as many steps, whose barriers, maxima and waits a
// single wave of a SIMD hides from nobody (16 capped heads of 256, 4096 tokens with a window of 2048, f16: 268 -> 224 us), where the registers let
template <typename T, int DT, bool WIDE = false> struct AtShape {
    static constexpr int CE = 16 / sizeof(T);                  // elements of a chunk
    static constexpr int STEPS = (DT + 2 * CE - 1) / (2 * CE); // pairs of chunks in a row
    static constexpr int BLOCKS = (DT + 31) / 32;              // 32-column blocks of the result
    static constexpr int KT = sizeof(T) == 2 && (DT <= 128 || WIDE) ? 64 : 32;
    static constexpr int HALVES = KT / 32;
    // Sums that a score is kept in while it grows: a f32 product adds two columns at a time, and 128 additions in a row lose twice what 32 do (a 16-bit one adds 16)
    static constexpr int SUMS = sizeof(T) == 2 || DT <= 64 ? 1 : DT <= 128 ? 2 : 4;
    static constexpr int CHUNKS = DT / CE;                     // of a row, at most
    static constexpr int LOADS = (KT * CHUNKS + AT_BLOCK - 1) / AT_BLOCK;      // of a tile of keys (or values), by each wave
    // a wave's last load of a tile may reach beyond it, and so may the transposed reads of the last block of columns
    static constexpr int TILE = (KT * CHUNKS * 16 + 1023) / 1024 * 1024;
    static constexpr int LDS = 4 * TILE + 256;
    static constexpr int WAVES = DT > 128 ? 1 : DT > (sizeof(T) == 2 ? 96 : 64) ? 2 : 3;             // of a SIMD: what its registers are shared by
};

// 16-byte chunks of a row are rotated by an amount that goes by the row, so that what the lanes of one access read spreads over the banks: keys are read a
// chunk from each of 16 rows at a time, values 32 bytes from each of 8 rows.
__device__ __forceinline__ uint32_t at_turn_k(uint32_t row, uint32_t chunks) {
    const uint32_t z = chunks % 16 == 0 ? 4 : chunks % 8 == 0 ? 3 : chunks % 4 == 0 ? 2 : chunks % 2 == 0 ? 1 : 0;
    return (row & 15) >> (4 - z);
}
template <typename T> __device__ __forceinline__ uint32_t at_turn_v(uint32_t row, uint32_t chunks) {
    if (sizeof(T) == 4 || chunks % 2) return 0;
    const uint32_t z = chunks % 16 == 0 ? 3 : chunks % 8 == 0 ? 2 : chunks % 4 == 0 ? 1 : 0;
    return 2 * ((row & 7) >> (3 - z));
}

// Left to itself the compiler reads an operand from LDS, waits for it and multiplies, one at a time.  A step is therefore written in the order it runs in: reads
// some products in front of their uses, the next keys' exponentials between the products of the last, and a fence for the scheduler after each product.
__device__ __forceinline__ void at_in_order() { __builtin_amdgcn_sched_barrier(0); }
// After a chain of products, `sum` being the last one's: reads it in the products' own block, so that the matrix unit is waited for there. Left to the reads behind a
// branch over a few instructions, the compiler counts the wait states of the longer way only, and what comes the shorter way reads sums that are not there yet (f32
// rows of 80 columns were off by 4e-2 for it)
__device__ __forceinline__ void at_settle(const v16f& sum) {
    at_in_order();
    asm volatile("" : : "s"(__builtin_amdgcn_readfirstlane(__float_as_uint(sum[15]))));
    at_in_order();
}

// One row over the keys of tiles [tile0, tile1) of a walk, a lane to a key for the scores and to columns for the result: visible keys alone are touched.
template <typename T, int DT, bool PAGED, int KT, bool SCORED>
__device__ __forceinline__ void at_row_again(const AttnArgs& a, uint32_t b, uint32_t g, AttnSeq s, AttnWalk w, uint32_t tile0, uint32_t tile1, uint32_t row, float* o, float& m_out,
                                          float& l_out) {
    constexpr int COLS = (DT + 63) / 64;
    const uint32_t lane = __lane_id(), D = a.dim, j = fd_div(row, a.group_div), h = g * a.group + (row - j * a.group);
    const T* q = (const T*)a.q + b * a.q_b + h * a.q_h + (uint64_t)(s.first + j) * a.q_t;
    const T* k = (const T*)a.k + g * a.k_h + (PAGED ? 0 : b * a.k_b);
    const T* v = (const T*)a.v + g * a.v_h + (PAGED ? 0 : b * a.v_b);
    const AttnRow r = at_row<SCORED>(a, SCORED && !PAGED ? at_texts(a, b) : AttnTexts{}, b, s, j);
    const float slope = SCORED && a.slopes ? at_slope(a, h) : 0.0f;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < COLS; i++) o[i] = 0.0f;
    for (uint32_t tile = tile0; tile < tile1; tile++) {
        const int32_t t = (tile < w.head ? w.start + (int32_t)(tile * KT) : w.from + (int32_t)((tile - w.head) * KT)) + (int32_t)lane;
        bool seen = lane < KT && at_sees<SCORED>(a, r, t);
        uint64_t k_at = 0, v_at = 0;
        if (seen) {
            if (PAGED) {
                uint32_t slot;
                const int32_t page = at_page(a, b, (uint32_t)t, slot);
                seen = page >= 0;
                k_at = (uint64_t)(seen ? page : 0) * a.k_b + slot * a.k_t;
                v_at = (uint64_t)(seen ? page : 0) * a.v_b + slot * a.v_t;
            } else {
                k_at = (uint64_t)t * a.k_t;
                v_at = (uint64_t)t * a.v_t;
            }
        }
        float x = -INFINITY;
        if (seen) {
            float dot = 0.0f;
            for (uint32_t d = 0; d < D; d++) dot = __builtin_fmaf(Ar<T>::widen(q[d]), Ar<T>::widen(k[k_at + d]), dot);
            x = at_changed<T, SCORED>(a, dot, slope, r.p - t);
        }
        uint64_t todo = __ballot(seen);
        if (!todo) continue;
        float top = x;
        for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
        const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.0f : m_new;
        const float old = at_exp2(m - base), e = seen ? at_exp2(x - base) : 0.0f;
        m = m_new;
        l = __builtin_fmaf(l, old, at_wave_sum(e));
#pragma unroll
        for (int i = 0; i < COLS; i++) o[i] *= old;
        while (todo) {
            const int src = __builtin_ctzll(todo);
            todo &= todo - 1;
            const float ei = __shfl(e, src);
            const uint64_t from = __shfl(v_at, src);
#pragma unroll
            for (int i = 0; i < COLS; i++)
                if (i * 64 + lane < D) o[i] = __builtin_fmaf(ei, Ar<T>::widen(v[from + i * 64 + lane]), o[i]);
        }
    }
    m_out = m;
    l_out = l;
}

// Where the keys of a row tile are shared out over blocks (pieces), each block leaves its part of the result.  Who joins them:
//   few rows (single tokens): the block that comes last.  Each counts itself in when its part is written, which for few rows is a few hundred bytes; parts then travel
//       between blocks of one launch, and each XCD has an L2 of its own, so they are written and read as agent-scope atomics, which go past it, and a
//       block counts itself in only when its writes have been acknowledged.
//   many rows: a launch of its own, 16 rows to a block.  The last block alone would read a whole row tile's parts (64 KB each) through one CU (see AT_FEW_ROWS for what is few).
struct AttnPartial {
    float* o;                      // [blocks][AT_ROWS][dim], unnormalised
    float* ml;                     // [blocks][AT_ROWS][2]: m (of scaled scores, base 2), l
    uint32_t* arrivals;            // [blocks]: of a row tile's first block
    uint32_t split;                // 0: each block walks all keys
    uint32_t pieces;               // contiguous: pieces of the keys a row tile is split into, `piece` tiles each
    uint32_t piece;
    uint32_t row_tiles;            // contiguous: of each batch entry
    uint32_t round;                // see at_turned
};

// Contiguous: which row tile, counted from the last, has place `at` in the launch.  A launch that the chip holds at once is not balanced by blocks that come later: where
// a CU gets one block of each `round` tiles, every other round runs backwards, so that a long causal walk shares its CU with a short one.
// Which launches are turned: rt_attention_order.h.
__device__ __forceinline__ uint32_t at_turned(const AttnPartial& part, uint32_t at) {
    if (part.round == 0) return at;
    const uint32_t n = at / part.round, first = n * part.round, count = part.row_tiles - first < part.round ? part.row_tiles - first : part.round;
    return n & 1 ? first + count - 1 - (at - first) : at;
}

__device__ __forceinline__ void at_leave(float* to, float x, float y) {
    const uint64_t both = (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x);
    __hip_atomic_store((uint64_t*)to, both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void at_take(const float* from, float& x, float& y) {
    const uint64_t both = __hip_atomic_load((const uint64_t*)from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = __uint_as_float((uint32_t)both);
    y = __uint_as_float((uint32_t)(both >> 32));
}

// Called by all threads of a block that has left its part.  True in the block that comes last of `used`.
__device__ __forceinline__ bool at_last(uint32_t* arrivals, uint32_t used, volatile uint32_t* shared) {
    at_wait_memory();                                              // this wave's part is where the others will read it
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = __hip_atomic_fetch_add(arrivals, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == used - 1;
        *shared = last;
        if (last) __hip_atomic_store(arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *shared != 0;
}

template <bool ATOMIC> __device__ __forceinline__ void at_put(float* to, float x, float y) {
    if (ATOMIC) {
        at_leave(to, x, y);
    } else {
        typedef float v2f __attribute__((ext_vector_type(2)));
        *(v2f*)to = v2f{x, y};
    }
}
template <bool ATOMIC> __device__ __forceinline__ void at_get(const float* from, float& x, float& y) {
    if (ATOMIC) {
        at_take(from, x, y);
    } else {
        typedef float v2f __attribute__((ext_vector_type(2)));
        const v2f both = *(const v2f*)from;
        x = both[0];
        y = both[1];
    }
}

// Joins `used` parts, `stride` blocks apart from block `first` on, of rows r0 .. r1 - 1 of the row tile at row0.  factors: LDS for (r1 - r0) * used floats.
// First each row's factors 2^(m_k - m) / l, then the sums, eight parts in flight.
template <typename T, bool ATOMIC, uint32_t ROWS>
__device__ __forceinline__ void at_join(const AttnArgs& a, const AttnPartial& part, const AttnSeq& s, uint32_t b, uint32_t g, uint32_t row0, uint32_t r0, uint32_t r1, uint64_t first,
                                        uint64_t stride, uint32_t used, float* factors) {
    const uint32_t D = a.dim, quads = D / 4, n = r1 - r0;
    // the factors: 16 lanes to a row
    const uint32_t part_lane = threadIdx.x % 16;
    for (uint32_t i0 = 0; i0 < n; i0 += AT_BLOCK / 16) {
        const uint32_t i = i0 + threadIdx.x / 16;
        float mk[(AT_MOST_PIECES + 15) / 16], lk[(AT_MOST_PIECES + 15) / 16], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (uint32_t u = 0; u < (AT_MOST_PIECES + 15) / 16; u++) {
            const uint32_t k = part_lane + 16 * u;
            mk[u] = -INFINITY;
            lk[u] = 0.0f;
            if (i < n && k < used) at_get<ATOMIC>(part.ml + 2 * ((first + k * stride) * ROWS + r0 + i), mk[u], lk[u]);
        }
#pragma unroll
        for (uint32_t u = 0; u < (AT_MOST_PIECES + 15) / 16; u++) m = fmaxf(m, mk[u]);
#pragma unroll
        for (int x = 8; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (uint32_t u = 0; u < (AT_MOST_PIECES + 15) / 16; u++) {
            mk[u] = at_exp2(mk[u] - base);
            l = __builtin_fmaf(mk[u], lk[u], l);
        }
#pragma unroll
        for (int x = 8; x; x >>= 1) l += __shfl_xor(l, x);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (uint32_t u = 0; u < (AT_MOST_PIECES + 15) / 16; u++)
            if (i < n && part_lane + 16 * u < used) factors[i * used + part_lane + 16 * u] = mk[u] * inv;
        if (a.lse && i < n && part_lane == 0) {
            const uint32_t row = row0 + r0 + i, j = fd_div(row, a.group_div), h = g * a.group + (row - j * a.group);
            a.lse[b * a.l_b + h * a.l_h + (uint64_t)(s.first + j) * a.l_t] = at_lse(m, l);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n * quads; i += AT_BLOCK) {
        const uint32_t r = i / quads, d = (i - r * quads) * 4;
        const float* from = part.o + (first * ROWS + r0 + r) * D + d;
        const uint64_t next = stride * ROWS * D;
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t k0 = 0; k0 < used; k0 += 8) {
            float x[8][4];
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) {
                const uint32_t k = k0 + u < used ? k0 + u : used - 1;
                at_get<ATOMIC>(from + k * next, x[u][0], x[u][1]);
                at_get<ATOMIC>(from + k * next + 2, x[u][2], x[u][3]);
            }
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) {
                const float f = k0 + u < used ? factors[r * used + k0 + u] : 0.0f;
                if (k0 + u < used)
#pragma unroll
                    for (int y = 0; y < 4; y++) o[y] = __builtin_fmaf(f, x[u][y], o[y]);
            }
        }
        const uint32_t row = row0 + r0 + r, j = fd_div(row, a.group_div), h = g * a.group + (row - j * a.group);
        T* y = (T*)a.y + b * a.y_b + h * a.y_h + (uint64_t)(s.first + j) * a.y_t + d;
        if constexpr (sizeof(T) == 2) {
            *(v2u*)y = v2u{AtMma<T>::pack(o[0], o[1]), AtMma<T>::pack(o[2], o[3])};
        } else {
            typedef float v4f __attribute__((ext_vector_type(4)));
            *(v4f*)y = v4f{o[0], o[1], o[2], o[3]};
        }
    }
}

// A tile's rows computed again where they are not finite: row `row`, by a wave, to y or to its part
template <typename T, int DT, bool PAGED, int KT, bool SCORED, bool ATOMIC>
__device__ __forceinline__ void at_again(const AttnArgs& a, const AttnPartial& part, uint32_t b, uint32_t g, const AttnSeq& s, const AttnWalk& w, uint32_t tile0, uint32_t tile1,
                                         uint32_t row, uint64_t part_at, bool whole) {
    const uint32_t lane = __lane_id(), D = a.dim;
    float oo[(DT + 63) / 64], mm, ll;
    at_row_again<T, DT, PAGED, KT, SCORED>(a, b, g, s, w, tile0, tile1, row, oo, mm, ll);
    const uint32_t jj = fd_div(row, a.group_div), hh = g * a.group + (row - jj * a.group);
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    T* y = (T*)a.y + b * a.y_b + hh * a.y_h + (uint64_t)(s.first + jj) * a.y_t;
#pragma unroll
    for (uint32_t i = 0; i < (DT + 63) / 64; i++) {
        const float next = __shfl_down(oo[i], 1);
        if (i * 64 + lane >= D) continue;
        if (whole) y[i * 64 + lane] = Ar<T>::conv(oo[i] * inv);
        else if (lane % 2 == 0) at_put<ATOMIC>(part.o + part_at * D + i * 64 + lane, oo[i], next);
    }
    if (lane == 0 && !whole) at_put<ATOMIC>(part.ml + 2 * part_at, mm, ll);
    if (lane == 0 && whole && a.lse) a.lse[b * a.l_b + hh * a.l_h + (uint64_t)(s.first + jj) * a.l_t] = at_lse(mm, ll);
}

// FEW: pieces are joined by the block that comes last (a joining launch took 10 to 13 us more), and scores are left where they are
// wanted.  Waves of a SIMD: as many as the registers let, four where the rows have 64 columns and no page table is followed (encoder in f32: 146.5 us a call, with three 148.7)
template <typename T, int DT, bool EXACT, bool PAGED, bool FEW, bool SCORED>
__global__ void __launch_bounds__(AT_BLOCK) __attribute__((amdgpu_waves_per_eu(AtShape<T, DT>::WAVES + (DT <= 64 && EXACT && !PAGED && !FEW && !SCORED), AtShape<T, DT>::WAVES + (DT <= 64 && EXACT && !PAGED && !FEW && !SCORED)))) attention_tile_kernel(AttnArgs a, AttnPartial part) {
    typedef AtShape<T, DT, SCORED && EXACT> S;
    constexpr int KT = S::KT, CE = S::CE;
    constexpr float LIFT = AT_LIFT<T, FEW>, LOWER = 1.0f / (1 << AT_LIFT<T, FEW>);              // the weights' factor is 2^LIFT, 1 / LOWER
    constexpr int SUMS = sizeof(T) == 4 && (PAGED || FEW) ? (S::SUMS > 2 ? S::SUMS : 2) : S::SUMS;  // 64 columns have registers for two where three waves share them
    extern __shared__ __align__(16) unsigned char smem[];
    lds_byte* const lds = (lds_byte*)smem;
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 32, half = lane / 32;
    const uint32_t D = EXACT ? DT : a.dim, chunks = D / CE, pitch = D * sizeof(T);

    // ---- which rows, which keys
    uint32_t b, g, tile, piece_at, piece, stride;               // stride: in blocks, from piece to piece of a row tile
    if (PAGED) {
        stride = a.kv_heads;
        g = blockIdx.x % a.kv_heads;
        uint32_t at = blockIdx.x / a.kv_heads;
        piece = part.split ? __builtin_amdgcn_readfirstlane(at_piece<KT, FEW, SCORED, AT_ROWS>(a)) : 0x7fffffffu;
        b = __builtin_amdgcn_readfirstlane(at_locate<KT, SCORED, AT_ROWS>(a, piece, at));
        if (b >= a.seqs) return;
        tile = __builtin_amdgcn_readfirstlane(at);
        piece_at = 0;
    } else {
        const uint32_t pairs = stride = a.seqs * a.kv_heads, pair = blockIdx.x % pairs, at = blockIdx.x / pairs;
        b = pair / a.kv_heads;
        g = pair - b * a.kv_heads;
        piece = part.piece;
        tile = part.row_tiles - 1 - at_turned(part, at / part.pieces);          // the longest walks first
        piece_at = at % part.pieces;
    }
    const AttnSeq s = at_seq<PAGED>(a, b);
    if (PAGED) {
        const uint32_t span = at_span<KT, SCORED>(a, b, s), at = tile;
        piece = at_piece_of(piece, span);
        const uint32_t pieces = (span + piece - 1) / piece;
        tile = at / pieces;
        piece_at = at - tile * pieces;
        tile = at_row_tiles<AT_ROWS>(a, s) - 1 - tile;
    }
    const uint32_t all = s.count * a.group, row0 = tile * AT_ROWS, rows = all - row0 < AT_ROWS ? all - row0 : AT_ROWS;
    const AttnTexts texts = SCORED && !PAGED ? at_texts(a, b) : AttnTexts{};
    const AttnWalk w = at_walk<KT, SCORED>(a, texts, b, s, row0, rows);
    const uint32_t tile0 = piece_at * piece, tile1 = w.tiles - tile0 < piece || tile0 >= w.tiles ? w.tiles : tile0 + piece;
    const bool whole = w.tiles <= piece;                        // no other block has keys of these rows
    if (tile0 >= w.tiles && piece_at > 0) return;
    // Starts that decrease can count more items than there are blocks: a row tile whose pieces are not all there is left alone (its counter would stay up).
    if (!whole && blockIdx.x + (uint64_t)((w.tiles + piece - 1) / piece - 1 - piece_at) * stride >= gridDim.x) return;

    // ---- this lane's row
    const uint32_t r = wave * 32 + col, row = row0 + (r < rows ? r : rows - 1);
    const uint32_t j = fd_div(row, a.group_div), h = g * a.group + (row - j * a.group);
    // and what all rows of the wave see, and any of them
    const bool busy = wave * 32 < rows;
    const uint32_t ja = fd_div(row0 + (busy ? wave * 32 : 0), a.group_div), jz = fd_div(row0 + (wave * 32 + 31 < rows ? wave * 32 + 31 : rows - 1), a.group_div);
    int32_t limit, p, limit_a, limit_z, p_a, p_z;
    int32_t front = a.sinks, front_a = a.sinks, front_z = a.sinks, lo = 0, lo_a = 0, lo_z = 0;
    if constexpr (SCORED) {
        AttnRow me, ra, rz;
        if (!PAGED && a.documents) {
            const uint32_t da = at_document(a, texts, b, at_position(s, ja)), dz = at_document(a, texts, b, at_position(s, jz));
            ra = at_in_document(a, texts, b, s, at_position(s, ja), da);
            rz = at_in_document(a, texts, b, s, at_position(s, jz), dz);
            me = at_in_document(a, texts, b, s, at_position(s, j), at_document_of(a, texts, b, at_position(s, j), da, dz));
        } else {
            const int32_t prefix = a.prefix ? a.prefix[b] : 0;
            me = at_in_text(a, at_position(s, j), 0, s.keys, prefix);
            ra = at_in_text(a, at_position(s, ja), 0, s.keys, prefix);
            rz = at_in_text(a, at_position(s, jz), 0, s.keys, prefix);
        }
        const auto one = [](int32_t x) __attribute__((always_inline)) { return (int32_t)__builtin_amdgcn_readfirstlane(x); };      // the same in all lanes
        limit = me.limit; limit_a = one(ra.limit); limit_z = one(rz.limit);
        p = me.p; p_a = one(ra.p); p_z = one(rz.p);
        front = me.front; front_a = one(ra.front); front_z = one(rz.front);
        if (!PAGED) {
            lo = me.lo; lo_a = one(ra.lo); lo_z = one(rz.lo);
        }
    } else {
        limit = at_limit(a, s, j); limit_a = at_limit(a, s, ja); limit_z = at_limit(a, s, jz);
        p = at_position(s, j); p_a = at_position(s, ja); p_z = at_position(s, jz);
    }

    v4u q[S::STEPS];
    {
        const T* from = (const T*)a.q + b * a.q_b + h * a.q_h + (uint64_t)(s.first + j) * a.q_t;
        const uint32_t flip = a.c < 0.0f ? AtMma<T>::SIGNS : 0;
#pragma unroll
        for (int i = 0; i < S::STEPS; i++) {
            q[i] = v4u{0, 0, 0, 0};
            if ((2 * i + half) * CE < D) q[i] = *(const v4u*)(from + (2 * i + half) * CE);
            q[i] ^= v4u{flip, flip, flip, flip};
        }
    }
    // |scale| log2 e; never 0, so that a hidden key's -inf stays
    // capped scores are in units of log2 e from there on; others get their bias in units of the products, divided by c, which then need no product of their own (unless c is next to 0)
    const bool changed = SCORED && (a.most != 0.0f || (a.slopes && __builtin_fabsf(a.c) < 0x1p-40f));
    const float c = changed ? 1.0f : fmaxf(__builtin_fabsf(a.c), 1e-37f);
    const float slope = SCORED && a.slopes ? at_slope(a, h) / c : 0.0f;

    // ---- this lane's part of a tile's loads: LDS chunk `slot` belongs to row slot / chunks
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
    const uint32_t k_row = (uint32_t)(a.k_t * sizeof(T)), v_row = (uint32_t)(a.v_t * sizeof(T));
    const uint32_t k_page = PAGED ? (uint32_t)(a.k_b * sizeof(T)) : 0;
    auto start_of = [&](uint32_t n) -> int32_t { return n < w.head ? (SCORED && !PAGED ? w.start : 0) + (int32_t)(n * KT) : w.from + (int32_t)((n - w.head) * KT); };
    // paged: the page of key `lane` of tile n, and its row there
    auto look = [&](uint32_t n, uint32_t& slot) -> int32_t {
        int32_t t = start_of(n) + (int32_t)(lane % KT);
        t = t < s.keys ? t : s.keys - 1;
        return at_page(a, b, (uint32_t)t, slot);
    };
    // contiguous: offsets of this lane's chunks from a whole tile's first key
    uint32_t k_off[S::LOADS], v_off[S::LOADS];
#pragma unroll
    for (int i = 0; i < S::LOADS; i++) {
        k_off[i] = l_row[i] * k_row + l_k[i];
        v_off[i] = l_row[i] * v_row + l_v[i];
    }
    // paged: offsets of the rows of this lane's chunks of the next tile, worked out from its pages before the loads can be issued
    uint64_t next_off[S::LOADS];
    auto prepare = [&](int32_t page, uint32_t slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) {
            int32_t pg = __shfl(page, (int)l_row[i]);
            const uint32_t sl = (uint32_t)__shfl((int)slot, (int)l_row[i]);
            pg = pg < 0 ? 0 : pg;
            next_off[i] = (uint64_t)(uint32_t)pg * k_page + sl * k_row;
        }
    };
    auto fetch = [&](uint32_t n, lds_byte* to) __attribute__((always_inline)) {
        const int32_t t0 = start_of(n);
        to += wave * 1024;
        if (PAGED) {
#pragma unroll
            for (int i = 0; i < S::LOADS; i++) {
                if (i * AT_WAVES + wave >= loads) break;
                at_to_lds<FEW>(kb + next_off[i] + l_k[i], to + i * AT_WAVES * 1024);
                at_to_lds<FEW>(vb + next_off[i] + l_v[i], to + i * AT_WAVES * 1024 + S::TILE);
            }
            return;
        }
        // Offsets within a tile fit 32 bits (the caller saw to it), its first key's need not.  The last tile's rows beyond the last key are that key's.
        const unsigned char* k0 = kb + (uint64_t)(uint32_t)t0 * k_row;
        const unsigned char* v0 = vb + (uint64_t)(uint32_t)t0 * v_row;
        const bool cut = t0 + KT > s.keys;
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) {
            if (i * AT_WAVES + wave >= loads) break;
            uint32_t ko = k_off[i], vo = v_off[i];
            if (cut && t0 + (int32_t)l_row[i] >= s.keys) {
                const uint32_t beyond = (uint32_t)(t0 + (int32_t)l_row[i] - (s.keys - 1));
                ko -= beyond * k_row;
                vo -= beyond * v_row;
            }
            at_to_lds(k0, ko, to + i * AT_WAVES * 1024);
            at_to_lds(v0, vo, to + i * AT_WAVES * 1024 + S::TILE);
        }
    };

    // ---- where this lane reads a tile
    uint32_t k_at[S::STEPS], v_at[S::BLOCKS];
#pragma unroll
    for (int i = 0; i < S::STEPS; i++) {
        uint32_t cc = 2 * i + half;
        cc = cc < chunks ? cc : 0;                              // beyond the row: replaced by 0 below
        cc += at_turn_k(col, chunks);
        k_at[i] = col * pitch + (cc >= chunks ? cc - chunks : cc) * 16;
    }
    const uint32_t v_key = 4 * half + (lane % 16) / 4;
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++) {
        if (sizeof(T) == 2) {
            uint32_t cc = 4 * i + 2 * ((lane / 16) & 1);
            if (cc >= chunks) cc = 0;                           // columns of nobody
            cc += at_turn_v<T>(v_key, chunks);
            if (cc >= chunks) cc -= chunks;
            v_at[i] = S::TILE + v_key * pitch + cc * 16 + (lane % 4) * 8;
        } else {
            v_at[i] = S::TILE + 4 * half * pitch + (i * 32 + col < D ? i * 32 + col : 0) * 4;
        }
    }

    v16f o[S::BLOCKS];
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++) o[i] = v16f{0};
    float m = -INFINITY, l = 0.0f;                              // l: of this lane's half of the keys
    if (SCORED && a.slopes && !__builtin_isfinite(slope)) l = __builtin_nanf("");                // beyond f32 in units of the products: computed again, a row at a time

    int32_t page = 0;                                           // of this lane's key of the tile after next
    uint32_t slot = 0;
    uint64_t there = ~0ull, there1 = ~0ull;                     // keys of the tile at hand that have a page, and of the next
    if (tile0 < tile1) {
        if (PAGED) {
            page = look(tile0, slot);
            there1 = __ballot(page >= 0);
            prepare(page, slot);
        }
        fetch(tile0, lds);
        if (PAGED && tile0 + 1 < tile1) page = look(tile0 + 1, slot);
    }
    // One tile: the loads of the next one go into `next` while this one is read from `cur`.  The wait for them stands at the top of the next step.
    auto step = [&](uint32_t n, lds_byte* next, const lds_byte* cur) __attribute__((always_inline)) {
        if (n + 1 < tile1) fetch(n + 1, next);
        if (PAGED && n + 2 < tile1) page = look(n + 2, slot);                   // arrives while this tile is worked on
        const int32_t t0 = start_of(n);
        if (!busy || t0 > limit_z || (SCORED && !PAGED && t0 + KT <= lo_a) || (t0 >= (SCORED ? front_z : a.sinks) && p_a - (t0 + KT - 1) >= a.window)) return;

        constexpr int N = S::STEPS * S::HALVES, AHEAD = N < 4 ? N : 4;
        v16f x[S::HALVES], others[S::HALVES][SUMS];
#pragma unroll
        for (int kk = 0; kk < S::HALVES; kk++) {
            x[kk] = v16f{0};
#pragma unroll
            for (int z = 1; z < SUMS; z++) others[kk][z] = v16f{0};
        }
        v4u k[N];
        auto read_k = [&](int at) __attribute__((always_inline)) {              // product `at`: step at / HALVES of half at % HALVES
            const int i = at / S::HALVES, kk = at % S::HALVES;
            if (!EXACT && (uint32_t)(2 * i * CE) >= D) return;
            k[at] = at_lds16(cur + (k_at[i] + kk * 32 * pitch));
        };
#pragma unroll
        for (int at = 0; at < AHEAD; at++) read_k(at);
        at_in_order();
#pragma unroll
        for (int at = 0; at < N; at++) {
            const int i = at / S::HALVES, kk = at % S::HALVES;
            if (EXACT || (uint32_t)(2 * i * CE) < D) {
                if ((EXACT ? DT % (2 * CE) != 0 : true) && (2 * i + 2) * CE > (int)D && half) k[at] = v4u{0, 0, 0, 0};
                at_score<T>(k[at], q[i], x[kk], others[kk]);
            }
            if (at + AHEAD < N) read_k(at + AHEAD);
            at_in_order();
        }
        at_settle(SUMS == 1 ? x[S::HALVES - 1] : others[S::HALVES - 1][SUMS - 1]);
#pragma unroll
        for (int kk = 0; kk < S::HALVES; kk++) at_join_sums(x[kk], others[kk]);
        const auto each_seen = [&](auto f) __attribute__((always_inline)) {     // each score of the tile, and whether its row sees its key
            // key t = 32 kk + (e % 4) + 8 (e / 4) + 4 half of the tile: p - t < window as t > p - window, which saturates where there is no window
            int32_t lim = limit - t0 - 4 * (int32_t)half, from = __builtin_elementwise_sub_sat(p - t0 - 4 * (int32_t)half, a.window), sink = (SCORED ? front : a.sinks) - t0 - 4 * (int32_t)half, low = lo - t0 - 4 * (int32_t)half;
            asm volatile("" : "+v"(lim), "+v"(from), "+v"(sink));               // nothing of this is worth registers outside of masked tiles
            if (SCORED && !PAGED) asm volatile("" : "+v"(low));
            const uint64_t have = there >> (4 * half);
#pragma unroll
            for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int32_t t = 32 * kk + e % 4 + 8 * (e / 4);
                    float score = x[kk][e];
                    f(score, t <= lim && (t > from || t < sink) && (!SCORED || PAGED || t >= low) && (!PAGED || (have >> t) & 1));
                    x[kk][e] = score;
                }
        };
        if (changed) {
            if (a.most != 0.0f) {
                bool near = false;
                if (sizeof(T) == 2) {
                    float far = 0.0f;
#pragma unroll
                    for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
                        for (int e = 0; e < 16; e++) far = fmaxf(far, __builtin_fabsf(x[kk][e]));
                    near = __ballot(!(far <= a.near_limit)) == 0;
                    if (!near && a.most > AT_COARSE) {          // what hidden keys hold does not have the rows computed again
                        far = 0.0f;
                        each_seen([&](float& score, bool seen) __attribute__((always_inline)) { far = fmaxf(far, seen ? __builtin_fabsf(score) : 0.0f); });
                        near = __ballot(!(far <= a.near_limit)) == 0;
                    }
                }
                if (near) {                                     // half of what the exponential and the reciprocal take
#pragma unroll
                    for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float z = x[kk][e] * x[kk][e];
                            x[kk][e] *= __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(a.near[3], z, a.near[2]), z, a.near[1]), z, a.near[0]);
                        }
                } else {
                    const float most_in = __builtin_fabsf(a.most_in);
                    if (sizeof(T) == 2 && a.most > AT_COARSE) l = __builtin_nanf("");             // computed again, a row at a time (with FINE ones here as well, 80 columns took 14 % more)
#pragma unroll
                    for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
                        for (int e = 0; e < 16; e++) x[kk][e] = at_capped<T, sizeof(T) == 4>(a.most, x[kk][e] * most_in);
                }
            }
            if (a.most == 0.0f) {
                const float cc = __builtin_fabsf(a.c);
#pragma unroll
                for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
                    for (int e = 0; e < 16; e++) x[kk][e] *= cc;
            }
        }
        if (SCORED && a.slopes) {
            const float far = (float)(p - t0 - 4 * (int32_t)half);              // distance of the tile's first key of this half
#pragma unroll
            for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
                for (int e = 0; e < 16; e++) x[kk][e] = __builtin_fmaf(-slope, __builtin_fabsf(far - (float)(32 * kk + e % 4 + 8 * (e / 4))), x[kk][e]);
        }
        if (t0 + KT - 1 > limit_a || (SCORED && !PAGED && t0 < lo_z) || (t0 + KT > (SCORED ? front_a : a.sinks) && p_z - t0 >= a.window) || (PAGED && there != ~0ull)) {
            each_seen([&](float& score, bool seen) __attribute__((always_inline)) { score = seen ? score : -INFINITY; });
        }
        if (FEW && a.scores && r < rows) {
            typedef float v4f __attribute__((ext_vector_type(4)));
            float* to = a.scores + ((uint64_t)(s.first + j) * a.heads + h) * a.score_pitch + (uint32_t)t0 + 4 * half;
#pragma unroll
            for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) *(v4f*)(to + 32 * kk + 8 * (e / 4)) = v4f{x[kk][e] * c, x[kk][e + 1] * c, x[kk][e + 2] * c, x[kk][e + 3] * c};
        }
        float top = x[0][0];
#pragma unroll
        for (int kk = 0; kk < S::HALVES; kk++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, x[kk][e]);
        top = fmaxf(top, at_other(top)) * c;
        // m follows the maximum at a distance: a weight of up to 2^AT_SLACK loses nothing in f32, f16 or bf16, and of 32 rows one has a new maximum in nearly every tile
        if (__ballot(top > m + (FEW ? 0.0f : (float)AT_SLACK))) {
            const float m_new = fmaxf(m, top), old = at_exp2(m - (m_new == -INFINITY ? 0.0f : m_new));
            m = m_new;
            l *= old;
#pragma unroll
            for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[i][e] *= old;
        }
        const float base = m == -INFINITY ? 0.0f : m - LIFT;
        if constexpr (sizeof(T) == 2) {
            constexpr int GROUPS = 2 * S::HALVES, P = GROUPS * S::BLOCKS, FRONT = 4;           // groups of 16 keys
            v4u v[P], w[GROUPS];
            auto read_v = [&](int at) __attribute__((always_inline)) {          // product `at`: columns at % BLOCKS of group at / BLOCKS
                const int i = at % S::BLOCKS, u = at / S::BLOCKS;
                if (!EXACT && (uint32_t)(32 * i) >= D) return;
                const uint32_t from = v_at[i] + 16 * u * pitch;
                const v2u lo = at_lds_turned(cur + from), hi = at_lds_turned(cur + (from + 8 * pitch));
                v[at] = v4u{lo[0], lo[1], hi[0], hi[1]};
            };
            // the exponentials of weights 2e, 2e + 1 of group u's 8 in this lane, and, later, what is made of them: a wave would wait for an exponential it uses at once
            auto weigh = [&](int u, int e) __attribute__((always_inline)) {
                x[u / 2][8 * (u % 2) + 2 * e] = at_exp2(__builtin_fmaf(x[u / 2][8 * (u % 2) + 2 * e], c, -base));
                x[u / 2][8 * (u % 2) + 2 * e + 1] = at_exp2(__builtin_fmaf(x[u / 2][8 * (u % 2) + 2 * e + 1], c, -base));
            };
            auto finish = [&](int u) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float w0 = x[u / 2][8 * (u % 2) + 2 * e], w1 = x[u / 2][8 * (u % 2) + 2 * e + 1];
                    l += w0 + w1;
                    w[u][e] = AtMma<T>::pack(w0, w1);
                }
            };
#pragma unroll
            for (int at = 0; at < FRONT; at++) read_v(at);
#pragma unroll
            for (int e = 0; e < 4; e++) weigh(0, e);
            finish(0);
            at_in_order();
#pragma unroll
            for (int at = 0; at < P; at++) {
                const int i = at % S::BLOCKS, u = at / S::BLOCKS;
                if (EXACT || (uint32_t)(32 * i) < D) o[i] = AtMma<T>::qk(v[at], w[u], o[i]);
                if (at + FRONT < P) read_v(at + FRONT);
                if (u + 1 < GROUPS)
#pragma unroll
                    for (int e = 4 * i / S::BLOCKS; e < 4 * (i + 1) / S::BLOCKS; e++) weigh(u + 1, e);
                if (i == S::BLOCKS - 1 && u + 1 < GROUPS) finish(u + 1);
                at_in_order();
            }
        } else {
            constexpr int P = 16 * S::HALVES * S::BLOCKS, FRONT = 8;
            float v[P], w[16 * S::HALVES];
            auto read_v = [&](int at) __attribute__((always_inline)) {          // product `at`: columns at % BLOCKS of the two keys of register at / BLOCKS
                const int i = at % S::BLOCKS, e = at / S::BLOCKS;
                if (!EXACT && (uint32_t)(32 * i) >= D) return;
                v[at] = at_lds4(cur + (v_at[i] + (32 * (e / 16) + e % 4 + 8 * (e % 16 / 4)) * pitch));
            };
            auto weigh = [&](int e) __attribute__((always_inline)) {
                w[e] = at_exp2(__builtin_fmaf(x[e / 16][e % 16], c, -base));
                l += w[e];
            };
#pragma unroll
            for (int at = 0; at < FRONT; at++) read_v(at);
            weigh(0);
            at_in_order();
#pragma unroll
            for (int at = 0; at < P; at++) {
                const int i = at % S::BLOCKS, e = at / S::BLOCKS;
                if (EXACT || (uint32_t)(32 * i) < D) o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[at], w[e], o[i], 0, 0, 0);
                if (at + FRONT < P) read_v(at + FRONT);
                if (i == 0 && e + 1 < 16 * S::HALVES) weigh(e + 1);
                at_in_order();
            }
        }
    };
    auto turn = [&](uint32_t n, lds_byte* next, const lds_byte* cur) __attribute__((always_inline)) {
        if (PAGED) {
            there = there1;
            there1 = __ballot(page >= 0);
            prepare(page, slot);
        }
        at_wait_memory();                                       // this wave's loads have arrived
        __syncthreads();                                        // and everyone's; and everyone is done with the other stage
        step(n, next, cur);
    };
    for (uint32_t n = tile0; n < tile1; n += 2) {               // two at a time: the stages' addresses are then constants
        turn(n, lds + 2 * S::TILE, lds);
        if (n + 1 < tile1) turn(n + 1, lds, lds + 2 * S::TILE);
    }

    // ---- result: lane's columns of d are 32 i + 8 (e / 4) + 4 half + e % 4
    at_settle(o[S::BLOCKS - 1]);
    l += at_other(l);
    bool fine = __builtin_isfinite(l) && m < INFINITY;
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (32 * i + 8 * (e / 4) + 4 * half < D) fine = fine && __builtin_isfinite(o[i][e]);
    if (__ballot(r < rows && !fine)) {
        const uint32_t end = wave * 32 + 32 < rows ? wave * 32 + 32 : rows;
        for (uint32_t rr = wave * 32; rr < end; rr++)
            at_again<T, DT, PAGED, KT, SCORED, FEW>(a, part, b, g, s, w, tile0, tile1, row0 + rr, (uint64_t)blockIdx.x * AT_ROWS + rr, whole);
    } else if (r < rows && whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* y = (T*)a.y + b * a.y_b + h * a.y_h + (uint64_t)(s.first + j) * a.y_t;
#pragma unroll
        for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t d = 32 * i + 8 * (e / 4) + 4 * half;
                if (d >= D) continue;
                if constexpr (sizeof(T) == 2) {
                    const v2u put = {AtMma<T>::pack(o[i][e] * inv, o[i][e + 1] * inv), AtMma<T>::pack(o[i][e + 2] * inv, o[i][e + 3] * inv)};
                    *(v2u*)(y + d) = put;
                } else {
                    typedef float v4f __attribute__((ext_vector_type(4)));
                    *(v4f*)(y + d) = v4f{o[i][e] * inv, o[i][e + 1] * inv, o[i][e + 2] * inv, o[i][e + 3] * inv};
                }
            }
        if (a.lse && half == 0) a.lse[b * a.l_b + h * a.l_h + (uint64_t)(s.first + j) * a.l_t] = at_lse(m, l * LOWER);
    } else if (r < rows) {
        const uint64_t part_at = (uint64_t)blockIdx.x * AT_ROWS + r;
#pragma unroll
        for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t d = 32 * i + 8 * (e / 4) + 4 * half;
                if (d >= D) continue;
                if (FEW) {
                    at_leave(part.o + part_at * D + d, o[i][e] * LOWER, o[i][e + 1] * LOWER);
                    at_leave(part.o + part_at * D + d + 2, o[i][e + 2] * LOWER, o[i][e + 3] * LOWER);
                } else {
                    typedef float v4f __attribute__((ext_vector_type(4)));
                    *(v4f*)(part.o + part_at * D + d) = v4f{o[i][e] * LOWER, o[i][e + 1] * LOWER, o[i][e + 2] * LOWER, o[i][e + 3] * LOWER};
                }
            }
        if (half == 0) at_put<FEW>(part.ml + 2 * part_at, m, l * LOWER);
    }
    if (!FEW || whole) return;
    const uint32_t used = (w.tiles + piece - 1) / piece, first = blockIdx.x - piece_at * stride;
    if (at_last(part.arrivals + first, used, (volatile uint32_t*)(smem + S::LDS - 16)))
        at_join<T, true, AT_ROWS>(a, part, s, b, g, row0, 0, rows, first, stride, used, (float*)smem);
}

// Parts of a row to the row: bound by reading them, 512 bytes a row, piece and 128 columns, and by the launch (encoder: 10 us, ragged chunks: 16 us with their search).
// blockIdx.y: which AT_JOIN_ROWS of a row tile.  blockIdx.x: paged: KV head, sequence and row tile of it, a row tile having more than one piece; contiguous: as the tiles' blocks
template <typename T, int KT, bool PAGED, bool SCORED> __global__ void __launch_bounds__(AT_BLOCK) attention_join_kernel(AttnArgs a, AttnPartial part, uint32_t tile_blocks) {
    __shared__ float factors[AT_JOIN_ROWS * AT_MOST_PIECES];
    uint32_t b, g, tile, piece, pieces;
    uint64_t first, stride;
    AttnSeq s;
    if (PAGED) {
        // numbered as the items are, with one piece a row tile
        g = blockIdx.x % a.kv_heads;
        uint32_t at = blockIdx.x / a.kv_heads;
        b = __builtin_amdgcn_readfirstlane(at_locate<KT, SCORED, AT_ROWS>(a, 0x7fffffffu, at));
        if (b >= a.seqs) return;
        s = at_seq<true>(a, b);
        tile = __builtin_amdgcn_readfirstlane(at);
        const uint32_t span = at_span<KT, SCORED>(a, b, s), all = __builtin_amdgcn_readfirstlane(at_piece<KT, false, SCORED, AT_ROWS>(a));
        piece = at_piece_of(all, span);
        pieces = (span + piece - 1) / piece;
        if (pieces == 1) return;
        stride = a.kv_heads;
        first = (__builtin_amdgcn_readfirstlane(at_before<KT, SCORED, AT_ROWS>(a, all, b)) + (uint64_t)(at_row_tiles<AT_ROWS>(a, s) - 1 - tile) * pieces) * stride + g;
    } else {
        stride = (uint64_t)a.seqs * a.kv_heads;
        const uint32_t pair = (uint32_t)(blockIdx.x % stride);
        b = pair / a.kv_heads;
        g = pair - b * a.kv_heads;
        tile = (uint32_t)(blockIdx.x / stride);
        s = at_seq<false>(a, b);
        piece = part.piece;
        first = (uint64_t)(part.row_tiles - 1 - tile) * part.pieces * stride + pair;
    }
    const uint32_t all_rows = s.count * a.group, row0 = tile * AT_ROWS, rows = all_rows - row0 < AT_ROWS ? all_rows - row0 : AT_ROWS;
    const AttnWalk w = at_walk<KT, SCORED>(a, SCORED && !PAGED ? at_texts(a, b) : AttnTexts{}, b, s, row0, rows);
    const uint32_t r0 = blockIdx.y * AT_JOIN_ROWS, r1 = r0 + AT_JOIN_ROWS < rows ? r0 + AT_JOIN_ROWS : rows;
    if (w.tiles <= piece || r0 >= rows) return;
    const uint32_t used = (w.tiles + piece - 1) / piece;
    if (first + (used - 1) * stride >= tile_blocks) return;     // as in the tiles' kernel: starts that decrease
    at_join<T, false, AT_ROWS>(a, part, s, b, g, row0, r0, r1, first, stride, used, factors);
}

template <typename T, int DT, bool EXACT, bool PAGED, bool SCORED> int at_launch_tile(rt_device* dev, AttnArgs& a, bool* done) {
    typedef AtShape<T, DT, SCORED && EXACT> S;
    AttnPartial part = {};
    const bool few = (uint64_t)a.tokens * a.group <= (uint64_t)AT_FEW_ROWS * (PAGED ? a.seqs : 1);
    const uint64_t most_blocks = AT_MOST_PARTS / (AT_ROWS * ((uint64_t)a.dim + 2) * sizeof(float));
    uint64_t join_tiles, items;                                 // row tiles; blocks per KV head (paged) or per (batch entry, KV head)
    const uint64_t per = PAGED ? a.kv_heads : (uint64_t)a.seqs * a.kv_heads;
    if (PAGED) {
        const uint64_t tiles = ((uint64_t)a.tokens * a.group) / AT_ROWS + a.seqs;
        // sum over the row tiles of ceil(span / piece): no more than work / piece, which is at most the target, and one for each row tile
        const uint32_t target = few ? AT_TARGET_FEW : AT_TARGET, least = few ? AT_LEAST_TILES_FEW : AT_LEAST_TILES;
        items = tiles + (few ? 1 : 2) * target / a.kv_heads + 1;                // (twice where the work is a causal mean, at least half of the spans)
        const bool enough = !few && ((uint64_t)a.tokens * a.group + AT_ROWS - 1) / AT_ROWS * per >= AT_ENOUGH;                // at least so many row tiles
        part.split = a.cap > least * S::KT && items * per <= RT_ARRIVALS && items * per <= most_blocks && !enough;
        if (!part.split) items = tiles;
        join_tiles = tiles * per;
    } else {
        part.row_tiles = (uint32_t)(((uint64_t)a.tokens * a.group + AT_ROWS - 1) / AT_ROWS);
        uint64_t span = (a.cap + S::KT - 1) / S::KT;
        if (a.window != AT_FAR && !a.documents && !a.prefix) {  // (where texts and prefixes end is known on the device)
            const uint64_t w = ((uint64_t)a.window + AT_ROWS) / S::KT + 2 + ((uint64_t)a.sinks + S::KT - 1) / S::KT;
            span = w < span ? w : span;
        }
        const uint64_t less = a.causal ? a.tokens / (2 * S::KT) : 0, mean = span > 2 * less ? span - less : (span + 1) / 2;
        const uint64_t tiles = part.row_tiles * per;
        uint64_t piece = few ? at_piece_for<true, AT_ROWS>(tiles, mean * tiles) : at_piece_for<false, AT_ROWS>(tiles, mean * tiles);
        // a block to each CU and short walks of 16-bit tiles, one to two microseconds each: parts and their joining cost more than the CUs that end early leave idle.
        // 32 heads of 64, 96 and 128, whole | shared out, us: causal 1024 tokens 21, 25, 29 | 27, 29, 40; 1024 of 2048 keys, all visible 40, 48, 58 | 40, 51, 71; of
        // 2560 47, 58, 72 | 46, 58, 82; of 4096 74, 88, 110 | 69, 89, 116; 8 heads, causal 4096 67, 78, 93 | 45, 62, 82.  A f32 tile takes four times as long
        if (!few && sizeof(T) == 2 && tiles >= (uint64_t)dev->num_cus && span <= AT_SHORT) piece = span;
        piece = at_piece_of((uint32_t)(piece > span ? span : piece), (uint32_t)span);
        if (part.row_tiles * ((span + piece - 1) / piece) * per > (most_blocks < RT_ARRIVALS ? most_blocks : RT_ARRIVALS)) piece = span;
        part.piece = (uint32_t)piece;
        part.pieces = (uint32_t)((span + piece - 1) / piece);
        part.split = part.pieces > 1;
        items = (uint64_t)part.row_tiles * part.pieces;
        constexpr uint64_t HELD = 160 * 1024 / S::LDS < S::WAVES ? 160 * 1024 / S::LDS : S::WAVES;             // blocks of a CU at once
        if (a.causal && part.pieces == 1) part.round = at_round(tiles, per, (uint64_t)dev->num_cus, HELD);
        join_tiles = part.row_tiles * per;
    }
    const uint64_t blocks = items * per;
    *done = blocks <= AT_MOST_BLOCKS;
    if (!*done) return RT_OK;
    const size_t row_count = part.split ? (size_t)blocks * AT_ROWS : 0;
    a.score_pitch = (a.cap + 63) / 64 * 64;
    size_t score_bytes = PAGED && few && a.want_scores ? (size_t)a.tokens * a.heads * a.score_pitch * sizeof(float) : 0;
    if (score_bytes > AT_MOST_SCORES) score_bytes = 0;
    void* p = nullptr;
    int rc = at_workspace(dev, a, row_count * ((size_t)a.dim + 2) * sizeof(float) + score_bytes, &p);
    if (rc) return rc;
    part.ml = (float*)p;
    part.o = part.ml + 2 * row_count;
    a.scores = score_bytes ? part.o + row_count * a.dim : nullptr;
    part.arrivals = dev->arrivals;
    const auto kernel = few ? attention_tile_kernel<T, DT, EXACT, PAGED, true, SCORED> : attention_tile_kernel<T, DT, EXACT, PAGED, false, SCORED>;
    static_assert(S::LDS <= 160 * 1024 && AT_MOST_PIECES * AT_ROWS * 4 <= S::LDS - 16, "LDS");
    static bool raised[2][16] = {};                             // per GPU; setting it twice does no harm
    if (S::LDS > 64 * 1024 && !(dev->ordinal < 16 && raised[few][dev->ordinal])) {
        RT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS));
        if (dev->ordinal < 16) raised[few][dev->ordinal] = true;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(AT_BLOCK), S::LDS, dev->stream, a, part);
    RT_CHECK_LAUNCH("attention_tile_kernel");
    if (part.split && !few) {
        hipLaunchKernelGGL((attention_join_kernel<T, S::KT, PAGED, SCORED>), dim3((unsigned)join_tiles, AT_ROWS / AT_JOIN_ROWS), dim3(AT_BLOCK), 0, dev->stream, a, part, (uint32_t)blocks);
        RT_CHECK_LAUNCH("attention_join_kernel");
    }
    return RT_OK;
}

// rt_attention_few.h: calls of a few rows a sequence
template <typename T> bool at_fits_few(const AttnArgs& a, bool paged);
template <typename T> int at_dispatch_few(rt_device* dev, AttnArgs& a, bool paged, bool* done);

template <typename T, bool SCORED> int at_dispatch_tile(rt_device* dev, AttnArgs& a, bool paged, bool* done) {
    // rows of whole 16-byte chunks on 16-byte boundaries; 32-bit offsets of the rows of a tile, or in a page, and of pages
    const uint64_t e = sizeof(T), most = 0xffffffffull / e, far = (1ull << 31) / 64 / e;
    const uint64_t strides[] = {a.dim, a.q_b, a.q_h, a.q_t, a.k_b, a.k_h, a.k_t, a.v_b, a.v_h, a.v_t, a.y_b, a.y_h, a.y_t};
    bool fits = rt_aligned(a.q, 16) && rt_aligned(a.k, 16) && rt_aligned(a.v, 16) && rt_aligned(a.y, 16) && a.k_t <= far && a.v_t <= far && (!paged || a.k_b <= most) &&
                (uint64_t)a.tokens * a.group <= 0x7fffffffull && a.dim <= 256;
    for (uint64_t x : strides) fits = fits && x * e % 16 == 0;
    *done = fits;
    if (!fits) return RT_OK;
    if constexpr (SCORED) {
        if (at_fits_few<T>(a, paged)) {
            const int rc = at_dispatch_few<T>(dev, a, paged, done);
            if (rc || *done) return rc;
        }
    }
#define RT_TILE(DT, EXACT) return paged ? at_launch_tile<T, DT, EXACT, true, SCORED>(dev, a, done) : at_launch_tile<T, DT, EXACT, false, SCORED>(dev, a, done)
    if (a.dim == 64) RT_TILE(64, true);
    if (a.dim == 80) RT_TILE(80, true);
    if (a.dim == 96) RT_TILE(96, true);
    if (a.dim == 128) RT_TILE(128, true);
    if (a.dim == 192) RT_TILE(192, true);
    if (a.dim == 256) RT_TILE(256, true);
    // f16, 32 heads, causal 2048 tokens: 40 columns 50 us, in the variant for 128 66; 192 and 256 columns 101 and 123 us (with turned rounds 130 and 160, and then with each
    // step's columns tested 248 and 262; f32 603 and 904, 1549 and 2720)
    if (a.dim < 64) RT_TILE(64, false);
    if (a.dim < 128) RT_TILE(128, false);
    RT_TILE(256, false);
#undef RT_TILE
}

#endif
