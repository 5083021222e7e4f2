// Rotary positions of tokens: every row its own position, pairs of halves or of neighbours, part of the head, any table of frequencies; alone, or
// with the rotated keys and the values going to the pages of the cache.
//
//     theta = position * f_i        (x1, x2) -> factor * (x1 cos theta - x2 sin theta, x1 sin theta + x2 cos theta)
// of columns (i, dim/2 + i), or (2i, 2i + 1) where interleaved; columns from dim on pass through.
//
// Angles are exact: the table holds f_i / 2 pi as a 64-bit fraction of a turn, and position * fraction mod 2^64 is the angle's fraction of a turn, 2^-65 * |position| off at most.
// What is left of the nearest quarter turn, at most an eighth, becomes a float (relative error 2^-24) and goes through the Taylor series of sine and cosine, to x^9 and x^10:
// the terms left out are below 2e-9.  So far positions are as good as near ones, and a negative position turns back.
//
// What bounds it: memory.  A block owns some tokens, computes a sine and cosine of each (token, frequency) once, into LDS, and its threads then turn two vectors each of all
// heads, whose loads are in flight before the sines.  f16, 8192 tokens of 64 heads of 96 columns: 41 us, 4.9 TB/s, what a copy reaches.  What a step adds is little next to a
// launch: 64 tokens of 40 heads of 128 columns 5 us, with the cache (the token's sequence, its length and page come one after the other) 6.
#include <math.h>

#include <algorithm>

#include "rt_attention.h"

namespace {

constexpr int BLOCK = 256, TRIP = 2;              // units of two vectors that a thread has in flight
constexpr uint32_t MOST_HALF = 512;               // frequencies
constexpr uint32_t PAIRS = 2 * MOST_HALF;         // (token, frequency) pairs of a block: LDS for their sines and cosines
constexpr uint32_t GRID_ROW = 1u << 22;           // blocks to a row of the grid: an extent of a launch has fewer than 2^32 threads

struct RopeRows {
    const void* x[3];                              // the heads of a token: queries, keys, values (rope_tokens: the first alone)
    void* y[3];                                    // keys and values of a paged call: the pages
    uint64_t x_token[3], x_head[3];                // strides, in vectors
    uint64_t y_token, y_head;                      // of the first
    uint32_t heads[3];
    bool in_place;                                 // y[0] is x[0]
    const int32_t* positions;                      // NULL in paged calls
    const int32_t *table, *lens, *starts;
    uint32_t seqs, table_len, n_pages, page_len;
    const uint64_t* turns;
    float factor;
    uint32_t tokens, half, hv, rv, row_v, units;   // units that turn, vectors that turn (of a row), vectors and units per row
    uint32_t ntok, head_chunk, chunks;             // tokens of a block; heads of a block, blocks to a token's heads
    FastDiv page_div, half_div, unit_div, row_units_div, chunk_div;   // by page_len, half, units, units * head_chunk, chunks
};

// sine and cosine of `turn` / 2^64 turns
__device__ __forceinline__ void sincos_turn(uint64_t turn, float& sn, float& cs) {
    const uint64_t near = turn + (1ull << 61);     // quarter turns, rounded
    const uint32_t quarter = (uint32_t)(near >> 62);
    const int64_t rest = (int64_t)(turn - ((uint64_t)quarter << 62));
    const float f = __builtin_fmaf((float)(uint32_t)rest, 0x1p-64f, (float)(int32_t)(rest >> 32) * 0x1p-32f);
    const float x = f * 6.283185307179586f, z = x * x;
    const float s = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
    sn = quarter & 2 ? -a : a;
    cs = (quarter + 1) & 2 ? -b : b;
}

// Where a token of a paged call goes
struct Place {
    int32_t position;
    uint32_t page, slot;
    uint32_t mine, there;                          // it belongs to a sequence; and its page exists
};
__device__ __forceinline__ Place find_place(const RopeRows& a, uint32_t token) {
    Place p = {0, 0, 0, 0, 0};
    const uint32_t b = at_find(a.starts, a.seqs, token);
    if (b == a.seqs) return p;
    const int32_t top = (int32_t)a.tokens;
    int32_t lo = a.starts[b], hi = a.starts[b + 1];
    lo = lo < 0 ? 0 : lo;
    hi = hi > top ? top : hi;
    if ((int32_t)token < lo || (int32_t)token >= hi) return p;
    int32_t len = a.lens[b];
    len = len < 0 ? 0 : len < AT_MOST_TOKENS ? len : AT_MOST_TOKENS;
    p.mine = 1;
    p.position = len - hi + (int32_t)token;
    if (p.position < 0) return p;
    uint32_t at;
    fd_divmod((uint32_t)p.position, a.page_div, at, p.slot);
    if (at >= a.table_len) return p;
    p.page = (uint32_t)a.table[(uint64_t)b * a.table_len + at];
    p.there = p.page < a.n_pages;
    return p;
}

template <int VB> struct VecOf;
template <> struct VecOf<16> { typedef v4u type; };
template <> struct VecOf<4> { typedef uint32_t type; };
template <> struct VecOf<2> { typedef uint16_t type; };
template <typename T, int VB> union Vec {
    typename VecOf<VB>::type u;
    T e[VB / sizeof(T)];
    __device__ __forceinline__ Vec() {}
};

template <typename T, int VB, bool INTER, bool PAGED> __global__ void __launch_bounds__(BLOCK) rope_tokens_kernel(RopeRows a) {
    constexpr int VE = VB / sizeof(T);
    typedef typename VecOf<VB>::type V;
    __shared__ float s_sn[PAIRS], s_cs[PAIRS];
    __shared__ Place s_place[PAGED ? BLOCK : 1];
    const uint32_t tid = threadIdx.x;
    uint32_t block, chunk;
    fd_divmod(blockIdx.y * GRID_ROW + blockIdx.x, a.chunk_div, block, chunk);
    const uint64_t first64 = (uint64_t)block * a.ntok;
    if (first64 >= a.tokens) return;
    const uint32_t first = (uint32_t)first64, ntok = a.tokens - first < a.ntok ? a.tokens - first : a.ntok;
    const uint32_t all_heads = a.heads[0] + a.heads[1] + a.heads[2], head0 = chunk * a.head_chunk;
    const uint32_t n_heads = all_heads - head0 < a.head_chunk ? all_heads - head0 : a.head_chunk;
    const uint32_t items = ntok * a.head_chunk * a.units;

    struct Item {
        uint32_t tok, head, unit, one, two;        // vectors of the row; two == row_v: there is none
        int which;                                 // of x
        bool live, turned;
        Vec<T, VB> a, b;
    };
    Item it[TRIP];
    auto load = [&](uint32_t at) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < TRIP; k++) {
            Item& i = it[k];
            const uint32_t n = at + k * BLOCK + tid;
            uint32_t rest;
            fd_divmod(n < items ? n : 0, a.row_units_div, i.tok, rest);
            fd_divmod(rest, a.unit_div, i.head, i.unit);
            i.live = n < items && i.head < n_heads;
            i.head += head0;
            i.which = 0;
            if (PAGED) {
                if (i.head >= a.heads[0]) {
                    i.head -= a.heads[0];
                    i.which = 1;
                    if (i.head >= a.heads[1]) {
                        i.head -= a.heads[1];
                        i.which = 2;
                    }
                }
            }
            i.turned = i.which != 2 && i.unit < a.hv;
            i.one = INTER ? 2 * i.unit : i.unit < a.hv ? i.unit : 2 * i.unit;
            i.two = INTER || i.unit >= a.hv ? i.one + 1 : i.unit + a.hv;
            if (a.in_place && i.which == 0 && !i.turned) i.live = false;
            if (i.live) {
                const V* from = (const V*)(i.which == 0 ? a.x[0] : i.which == 1 ? a.x[1] : a.x[2]);
                const uint64_t ts = i.which == 0 ? a.x_token[0] : i.which == 1 ? a.x_token[1] : a.x_token[2], hs = i.which == 0 ? a.x_head[0] : i.which == 1 ? a.x_head[1] : a.x_head[2];
                from += (first + i.tok) * ts + i.head * hs;
                i.a.u = from[i.one];
                if (i.two < a.row_v) i.b.u = from[i.two];
            }
        }
    };
    load(0);
    // the first frequency of each thread is on its way while the tokens are found
    uint32_t t_first = 0, i_first = 0;
    fd_divmod(tid, a.half_div, t_first, i_first);
    uint64_t turn = tid < ntok * a.half ? a.turns[i_first] : 0;
    if (PAGED) {
        for (uint32_t t = tid / 64; t < ntok; t += BLOCK / 64) {
            const Place p = find_place(a, first + t);
            if (tid % 64 == 0) s_place[t] = p;
        }
        __syncthreads();
    }
    for (uint32_t n = tid; n < ntok * a.half; n += BLOCK) {
        uint32_t t, i;
        fd_divmod(n, a.half_div, t, i);
        if (n != tid) turn = a.turns[i];
        const int64_t position = PAGED ? s_place[t].position : a.positions[first + t];
        float sn, cs;
        sincos_turn((uint64_t)position * turn, sn, cs);
        s_sn[n] = sn * a.factor;
        s_cs[n] = cs * a.factor;
    }
    __syncthreads();
    for (uint32_t at = 0; at < items;) {
        Item now[TRIP];
#pragma unroll
        for (int k = 0; k < TRIP; k++) {
            Item& i = it[k];
            now[k] = i;
            if (!i.live || !i.turned) continue;
            const uint32_t f = i.tok * a.half;
            if (INTER && VE > 1) {
#pragma unroll
                for (int e = 0; e + 1 < VE; e += 2) {
                    const uint32_t g = f + (i.one * VE + e) / 2;
                    const float cs = s_cs[g], sn = s_sn[g], x1 = Ar<T>::widen(i.a.e[e]), x2 = Ar<T>::widen(i.a.e[e + 1]);
                    now[k].a.e[e] = Ar<T>::conv(__builtin_fmaf(x1, cs, -(x2 * sn)));
                    now[k].a.e[e + 1] = Ar<T>::conv(__builtin_fmaf(x1, sn, x2 * cs));
                }
                if (i.two < a.rv)
#pragma unroll
                    for (int e = 0; e + 1 < VE; e += 2) {
                        const uint32_t g = f + (i.two * VE + e) / 2;
                        const float cs = s_cs[g], sn = s_sn[g], x1 = Ar<T>::widen(i.b.e[e]), x2 = Ar<T>::widen(i.b.e[e + 1]);
                        now[k].b.e[e] = Ar<T>::conv(__builtin_fmaf(x1, cs, -(x2 * sn)));
                        now[k].b.e[e + 1] = Ar<T>::conv(__builtin_fmaf(x1, sn, x2 * cs));
                    }
            } else {
#pragma unroll
                for (int e = 0; e < VE; e++) {
                    const uint32_t g = f + i.unit * VE + e;
                    const float cs = s_cs[g], sn = s_sn[g], x1 = Ar<T>::widen(i.a.e[e]), x2 = Ar<T>::widen(i.b.e[e]);
                    now[k].a.e[e] = Ar<T>::conv(__builtin_fmaf(x1, cs, -(x2 * sn)));
                    now[k].b.e[e] = Ar<T>::conv(__builtin_fmaf(x1, sn, x2 * cs));
                }
            }
        }
        at += TRIP * BLOCK;
        if (at < items) load(at);
#pragma unroll
        for (int k = 0; k < TRIP; k++) {
            const Item& i = now[k];
            if (!i.live) continue;
            V* to;
            if (i.which == 0) {
                if (PAGED && !s_place[i.tok].mine) continue;
                to = (V*)a.y[0] + (first + i.tok) * a.y_token + i.head * a.y_head;
            } else {
                const Place& p = s_place[PAGED ? i.tok : 0];
                if (!p.there) continue;
                to = (V*)(i.which == 1 ? a.y[1] : a.y[2]) + (((uint64_t)p.page * a.heads[1] + i.head) * a.page_len + p.slot) * a.row_v;
            }
            to[i.one] = i.a.u;
            if (i.two < a.row_v) to[i.two] = i.b.u;
        }
    }
}

template <typename T, int VB> void launch(rt_device* dev, const RopeRows& a, bool interleaved, bool paged, dim3 grid) {
#define RT_RT(I, P) hipLaunchKernelGGL((rope_tokens_kernel<T, VB, I, P>), grid, dim3(BLOCK), 0, dev->stream, a)
    if (interleaved && paged) RT_RT(true, true);
    else if (interleaved) RT_RT(true, false);
    else if (paged) RT_RT(false, true);
    else RT_RT(false, false);
#undef RT_RT
}

// a: everything but the vectors' sizes, with strides in elements
int run(rt_device* dev, int dt, RopeRows& a, uint32_t dim, uint32_t head_dim, bool interleaved, bool paged) {
    const uint32_t e = (uint32_t)rt_dt_bytes(dt);
    // the widest vector that all rows, their halves and the rotated columns are whole numbers of
    uint32_t vb = 16;
    for (; vb > e; vb = vb == 16 ? 4 : e) {
        bool fits = (uint64_t)head_dim * e % vb == 0 && (uint64_t)(interleaved ? dim : dim / 2) * e % vb == 0 && a.y_token * e % vb == 0 && a.y_head * e % vb == 0;
        for (int i = 0; i < (paged ? 3 : 1); i++) fits = fits && a.x_token[i] * e % vb == 0 && a.x_head[i] * e % vb == 0 && rt_aligned(a.x[i], vb) && rt_aligned(a.y[i], vb);
        if (fits) break;
    }
    const uint32_t ve = vb / e;
    for (int i = 0; i < 3; i++) {
        a.x_token[i] /= ve;
        a.x_head[i] /= ve;
    }
    a.y_token /= ve;
    a.y_head /= ve;
    a.half = dim / 2;
    a.row_v = head_dim / ve;
    a.units = (a.row_v + 1) / 2;
    a.rv = dim / ve;
    a.hv = (a.rv + 1) / 2;                         // (halves: rv is even)
    const uint32_t heads = a.heads[0] + a.heads[1] + a.heads[2];
    const uint64_t row_units = (uint64_t)heads * a.units;
    RT_REQUIRE(row_units < 1ull << 31, RT_ERR_SIZE, "rope: rows of %u heads of %u columns", heads, head_dim);
    // Tokens of few heads share a block, a unit to a thread, as far as there are blocks for all CUs.  f16, one token to a block | several: 65536 tokens of a head of 64 columns
    // 50 us | 8, of 8 heads of 128 57 | 41, 8192 of a head of 128 8.8 | 4.2, cache and all for 16 pieces of 1000 tokens of 1 + 1 heads of 40 19 | 7; two units to a thread
    // 41 | 43 for 8 heads, and a block's sines in 2 KB of LDS in place of 8 14 us for 65536 tokens of a head of 128 in place of 13.
    a.ntok = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({PAIRS / a.half, BLOCK / row_units, a.tokens / (uint32_t)dev->num_cus}));
    a.head_chunk = heads;
    if (a.ntok == 1 && row_units * a.tokens < 2ull * dev->num_cus * BLOCK) {
        const uint32_t per = BLOCK / a.units > 1 ? BLOCK / a.units : 1;           // few tokens: a unit to a thread, blocks share a token's heads
        a.head_chunk = per < heads ? per : heads;
    }
    a.chunks = (heads + a.head_chunk - 1) / a.head_chunk;
    a.half_div = make_fastdiv(a.half);
    a.unit_div = make_fastdiv(a.units);
    a.row_units_div = make_fastdiv(a.units * a.head_chunk);
    a.chunk_div = make_fastdiv(a.chunks);
    const uint64_t blocks = ((uint64_t)a.tokens + a.ntok - 1) / a.ntok * a.chunks;
    RT_REQUIRE(blocks < 1ull << 32 && blocks <= 65535ull * GRID_ROW, RT_ERR_SIZE, "rope: too many tokens");
    const dim3 grid((unsigned)(blocks < GRID_ROW ? blocks : GRID_ROW), (unsigned)((blocks + GRID_ROW - 1) / GRID_ROW));
    if (dt == RT_F32) {
        if (vb == 16) launch<float, 16>(dev, a, interleaved, paged, grid);
        else launch<float, 4>(dev, a, interleaved, paged, grid);
    } else if (dt == RT_F16) {
        if (vb == 16) launch<half_t, 16>(dev, a, interleaved, paged, grid);
        else if (vb == 4) launch<half_t, 4>(dev, a, interleaved, paged, grid);
        else launch<half_t, 2>(dev, a, interleaved, paged, grid);
    } else {
        if (vb == 16) launch<bf16_t, 16>(dev, a, interleaved, paged, grid);
        else if (vb == 4) launch<bf16_t, 4>(dev, a, interleaved, paged, grid);
        else launch<bf16_t, 2>(dev, a, interleaved, paged, grid);
    }
    RT_CHECK_LAUNCH("rope_tokens_kernel");
    return RT_OK;
}

int table_rules(const char* who, int dt, uint32_t head_dim, const uint64_t* turns, uint32_t dim, float factor, int interleaved) {
    RT_REQUIRE(rt_is_float_dt(dt), RT_ERR_DTYPE, "%s: dtype %d is not F32, F16 or BF16", who, dt);
    RT_REQUIRE(head_dim > 0, RT_ERR_SHAPE, "%s: zero extent", who);
    RT_REQUIRE(dim > 0 && dim % 2 == 0 && dim <= head_dim, RT_ERR_SHAPE, "%s: dim %u must be positive, even and <= %u", who, dim, head_dim);
    RT_REQUIRE(dim / 2 <= MOST_HALF && head_dim <= 1u << 16, RT_ERR_SIZE, "%s: %u of %u columns", who, dim, head_dim);
    RT_REQUIRE(isfinite(factor), RT_ERR_ARG, "%s: factor is not finite", who);
    RT_REQUIRE(interleaved == 0 || interleaved == 1, RT_ERR_ARG, "%s: interleaved is %d", who, interleaved);
    RT_REQUIRE(turns, RT_ERR_NULL_POINTER, "%s: NULL table", who);
    RT_REQUIRE(rt_aligned(turns, 8), RT_ERR_ALIGN, "%s: misaligned table", who);
    return RT_OK;
}

// Whether two of the rows [tokens, heads, dim] share an element
bool rows_overlap(uint32_t tokens, uint32_t heads, uint32_t dim, uint64_t token, uint64_t head) {
    const bool token_first = heads == 1 || (tokens > 1 && token < head);           // the smaller stride
    const uint64_t near = token_first ? token : head, far = token_first ? head : token;
    const uint32_t n_near = token_first ? tokens : heads, n_far = token_first ? heads : tokens;
    return (n_near > 1 && near < dim) || (n_far > 1 && far < (n_near - 1) * near + dim);
}

}  // namespace

extern "C" {

int rt_rope_turns(uint32_t dim, double base, const double* divisors, uint64_t* turns) {
    RT_REQUIRE(dim > 0 && dim % 2 == 0, RT_ERR_SHAPE, "rt_rope_turns: dim %u must be positive and even", dim);
    RT_REQUIRE(turns, RT_ERR_NULL_POINTER, "rt_rope_turns: NULL turns");
    RT_REQUIRE(base > 0 && isfinite(base), RT_ERR_ARG, "rt_rope_turns: base must be positive and finite");
    for (uint32_t i = 0; divisors && i < dim / 2; i++) RT_REQUIRE(divisors[i] > 0 && isfinite(divisors[i]), RT_ERR_ARG, "rt_rope_turns: divisor %u is not positive and finite", i);
    for (uint32_t i = 0; i < dim / 2; i++) {
        long double f = powl((long double)base, -2.0L * i / dim) / 6.283185307179586476925286766559005768L;
        if (divisors) f /= divisors[i];
        f -= floorl(f);
        const long double n = roundl(f * 0x1p64L);
        turns[i] = n < 0x1p64L ? (uint64_t)n : 0;
    }
    return RT_OK;
}

int rt_rope_tokens(rt_device* dev, int dt, const void* x, const uint64_t x_strides[2], void* y, const uint64_t y_strides[2], uint32_t tokens, uint32_t heads, uint32_t head_dim,
                   const int32_t* positions, const uint64_t* turns, uint32_t dim, float factor, int interleaved) {
    static const char* const who = "rt_rope_tokens";
    RopeRows a = {};
    RT_REQUIRE(heads > 0, RT_ERR_SHAPE, "%s: zero extent", who);
    RT_REQUIRE(heads <= 65535, RT_ERR_SIZE, "%s: %u heads", who, heads);
    int rc = table_rules(who, dt, head_dim, turns, dim, factor, interleaved);
    if (rc) return rc;
    if ((rc = rt_rows_rules(who, "x", tokens, heads, head_dim, x_strides, &a.x_token[0], &a.x_head[0]))) return rc;
    if ((rc = rt_rows_rules(who, "y", tokens, heads, head_dim, y_strides, &a.y_token, &a.y_head))) return rc;
    RT_REQUIRE(!rows_overlap(tokens, heads, head_dim, a.y_token, a.y_head), RT_ERR_ARG, "%s: elements of y overlap", who);
    RT_REQUIRE(x && y && positions, RT_ERR_NULL_POINTER, "%s: NULL operand", who);
    const size_t e = (size_t)rt_dt_bytes(dt);
    RT_REQUIRE(rt_aligned(x, e) && rt_aligned(y, e) && rt_aligned(positions, 4), RT_ERR_ALIGN, "%s: misaligned pointer", who);
    RT_REQUIRE(x != y || (a.x_token[0] == a.y_token && a.x_head[0] == a.y_head), RT_ERR_ARG, "%s: y is x with other strides", who);
    rc = rt_enter(dev);
    if (rc) return rc;
    a.x[0] = x;
    a.y[0] = y;
    a.in_place = x == y;
    a.heads[0] = heads;
    a.positions = positions;
    a.turns = turns;
    a.factor = factor;
    a.tokens = tokens;
    return run(dev, dt, a, dim, head_dim, interleaved != 0, false);
}

int rt_paged_rope_append(rt_device* dev, int dt, const rt_paged_kv* kv, const int32_t* starts, uint32_t tokens, const void* q, const uint64_t q_strides[2], uint32_t heads,
                         void* y, const uint64_t y_strides[2], const void* k, const uint64_t k_strides[2], const void* v, const uint64_t v_strides[2], const uint64_t* turns,
                         uint32_t dim, float factor, int interleaved) {
    static const char* const who = "rt_paged_rope_append";
    RopeRows a = {};
    RT_REQUIRE(kv, RT_ERR_NULL_POINTER, "%s: NULL cache", who);
    RT_REQUIRE(heads > 0, RT_ERR_SHAPE, "%s: zero extent", who);
    RT_REQUIRE(heads <= 65535, RT_ERR_SIZE, "%s: %u heads", who, heads);
    int rc = table_rules(who, dt, kv->head_dim, turns, dim, factor, interleaved);
    if (rc) return rc;
    const size_t e = (size_t)rt_dt_bytes(dt);
    if ((rc = rt_paged_rules(who, kv, e))) return rc;
    const uint32_t d = kv->head_dim;
    if ((rc = rt_rows_rules(who, "q", tokens, heads, d, q_strides, &a.x_token[0], &a.x_head[0]))) return rc;
    if ((rc = rt_rows_rules(who, "y", tokens, heads, d, y_strides, &a.y_token, &a.y_head))) return rc;
    if ((rc = rt_rows_rules(who, "k", tokens, kv->kv_heads, d, k_strides, &a.x_token[1], &a.x_head[1]))) return rc;
    if ((rc = rt_rows_rules(who, "v", tokens, kv->kv_heads, d, v_strides, &a.x_token[2], &a.x_head[2]))) return rc;
    RT_REQUIRE(!rows_overlap(tokens, heads, d, a.y_token, a.y_head), RT_ERR_ARG, "%s: elements of y overlap", who);
    RT_REQUIRE(q && y && k && v && starts, RT_ERR_NULL_POINTER, "%s: NULL operand", who);
    RT_REQUIRE(rt_aligned(q, e) && rt_aligned(y, e) && rt_aligned(k, e) && rt_aligned(v, e) && rt_aligned(starts, 4), RT_ERR_ALIGN, "%s: misaligned pointer", who);
    RT_REQUIRE(q != y || (a.x_token[0] == a.y_token && a.x_head[0] == a.y_head), RT_ERR_ARG, "%s: y is q with other strides", who);
    rc = rt_enter(dev);
    if (rc) return rc;
    a.x[0] = q; a.x[1] = k; a.x[2] = v;
    a.y[0] = y; a.y[1] = kv->k; a.y[2] = kv->v;
    a.in_place = q == y;
    a.heads[0] = heads;
    a.heads[1] = a.heads[2] = kv->kv_heads;
    a.table = kv->table; a.lens = kv->lens; a.starts = starts;
    a.seqs = kv->seqs; a.table_len = kv->table_len; a.n_pages = kv->pages; a.page_len = kv->page_len;
    a.page_div = make_fastdiv(kv->page_len);
    a.turns = turns;
    a.factor = factor;
    a.tokens = tokens;
    return run(dev, dt, a, dim, d, interleaved != 0, true);
}

}  // extern "C"
