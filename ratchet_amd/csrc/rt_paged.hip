// The paged KV cache: append of new rows, and eviction by accumulated attention weight.
#include "rt_attention.h"

namespace {

constexpr int BLOCK = 256;

// ---------------------------------------------------------------------------------------------------- append
struct AppendArgs {
    const void* src[2];
    void* pages[2];
    uint64_t token[2], head[2];    // strides of the sources, in vectors
    const int32_t *table, *lens, *starts;
    uint32_t n_pages, kv_heads, page_len, row_v, seqs, table_len, tokens;
    FastDiv page_div, row_div;     // by page_len; by vectors per row
};

// A block to a token: the wave finds the token's sequence, then the block's threads move the vectors of all its heads, keys and values alike.
// Moves each row once; bound by memory for prompts (157 MB in f16: 31.7 us, 5.0 TB/s) and by the chain starts -> lens and table -> store for single tokens (64: 2.8 us).
constexpr uint32_t APPEND_ROW = 1u << 22;           // blocks to a row of the grid: an extent of a launch has fewer than 2^32 threads

template <typename VecT> __global__ void __launch_bounds__(BLOCK) paged_append_kernel(AppendArgs a) {
    const uint32_t token = blockIdx.y * APPEND_ROW + blockIdx.x;
    if (token >= a.tokens) return;
    const uint32_t b = at_find(a.starts, a.seqs, token);
    if (b == a.seqs) return;
    const int32_t top = (int32_t)a.tokens;
    int32_t lo = a.starts[b], hi = a.starts[b + 1];
    lo = lo < 0 ? 0 : lo;
    hi = hi > top ? top : hi;
    if ((int32_t)token < lo || (int32_t)token >= hi) return;
    int32_t len = a.lens[b];
    len = len < 0 ? 0 : len < AT_MOST_TOKENS ? len : AT_MOST_TOKENS;
    const int32_t t = len - hi + (int32_t)token;
    if (t < 0) return;
    uint32_t at, slot;
    fd_divmod((uint32_t)t, a.page_div, at, slot);
    if (at >= a.table_len) return;
    const uint32_t page = (uint32_t)a.table[(uint64_t)b * a.table_len + at];
    if (page >= a.n_pages) return;
    const uint32_t per = a.kv_heads * a.row_v;
    for (uint32_t i = threadIdx.x; i < 2 * per; i += BLOCK) {
        const uint32_t which = i >= per, e = which ? i - per : i;
        uint32_t h, c;
        fd_divmod(e, a.row_div, h, c);
        const VecT x = ((const VecT*)a.src[which])[token * a.token[which] + h * a.head[which] + c];
        ((VecT*)a.pages[which])[(((uint64_t)page * a.kv_heads + h) * a.page_len + slot) * a.row_v + c] = x;
    }
}

// -------------------------------------------------------------------------------------------------- eviction
struct EvictArgs {
    const int32_t* lens;
    const float* weights;
    float* weights_out;
    uint32_t* kept;                // scratch: [seqs, kv_heads, keep] tokens that stay, in order
    uint32_t* counts;              // scratch: [seqs, kv_heads] how many
    uint32_t kv_heads, cap, keep, first, recent;
};

constexpr int SELECT_BLOCK = 1024;

// Weights in an order that unsigned integers have: larger is kept; NaN below everything, -0 and +0 alike
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A block to a (sequence, KV head).  The weight of the last token that stays is found digit by digit, eight bits at a time from the top
// (a histogram of the candidates that share the digits found so far); then one walk over the tokens writes the list of those that stay and
// moves their weights.  A round takes SELECT_ROUND tokens, 64 * SELECT_EACH of them in a row to a wave: one round's weights stay in registers
// from the first digit to the walk.  A weight moves to an index at or below its own and a round reads its tokens before it writes, so weights_out may be weights.
// Bound by its own chain of four histograms, a barrier or two each: 12 us for 8 blocks of 4100 tokens, 13 for 256 of up to 4096.
constexpr uint32_t SELECT_EACH = 8, SELECT_WAVES = SELECT_BLOCK / 64, SELECT_ROUND = SELECT_BLOCK * SELECT_EACH;
constexpr uint32_t SELECT_COPIES = 4;            // of the histogram: weights crowd into few digits, and lanes that meet in a bin wait for each other

__global__ void __launch_bounds__(SELECT_BLOCK) evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t hist[2][SELECT_COPIES][256], counts[SELECT_WAVES][2], digit, above;
    const uint32_t g = blockIdx.x, b = blockIdx.y, pair = b * a.kv_heads + g, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int32_t raw = a.lens[b];
    const uint32_t len = raw < 0 ? 0 : (uint32_t)raw < a.cap ? (uint32_t)raw : a.cap;
    const float* w = a.weights + (uint64_t)pair * a.cap;
    float* out = a.weights_out + (uint64_t)pair * a.cap;
    uint32_t* kept = a.kept + (uint64_t)pair * a.keep;
    if (len <= a.keep) {
        for (uint32_t t = tid; t < len; t += SELECT_BLOCK) {
            kept[t] = t;
            if (out != w) out[t] = w[t];
        }
        if (tid == 0) a.counts[pair] = len;
        return;
    }
    const uint32_t lo = a.first, hi = len - a.recent, need = a.keep - a.first - a.recent;      // candidates [lo, hi): more than need
    const bool once = len <= SELECT_ROUND;
    float x[SELECT_EACH];
    const uint32_t mine = wave * (64 * SELECT_EACH) + lane;     // this thread's first token of a round; the others follow 64 apart
    auto load = [&](uint32_t t0) {
#pragma unroll
        for (uint32_t i = 0; i < SELECT_EACH; i++) x[i] = t0 + mine + 64 * i < len ? w[t0 + mine + 64 * i] : 0.0f;
    };
    if (once) load(0);
    hist[0][tid / 256][tid % 256] = 0;
    __syncthreads();
    uint32_t found = 0, left = need;               // the digits so far; how many of the candidates that share them stay
    if (need)
        for (int shift = 24; shift >= 0; shift -= 8) {
            uint32_t* h = hist[(shift / 8 + 1) & 1][0];         // digits 3, 2, 1, 0
            for (uint32_t t0 = 0; t0 < len; t0 += SELECT_ROUND) {
                if (!once) load(t0);
#pragma unroll
                for (uint32_t i = 0; i < SELECT_EACH; i++) {
                    const uint32_t t = t0 + mine + 64 * i, key = weight_key(x[i]);
                    if (t >= lo && t < hi && (shift == 24 || (key >> (shift + 8)) == (found >> (shift + 8)))) atomicAdd(&h[(lane % SELECT_COPIES) * 256 + ((key >> shift) & 255)], 1u);
                }
            }
            __syncthreads();
            if (wave == 0) {                       // lane's digits: 255 - 4 lane and the three below; sums from the top
                uint32_t n[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    n[i] = 0;
#pragma unroll
                    for (uint32_t y = 0; y < SELECT_COPIES; y++) n[i] += h[y * 256 + 255 - 4 * lane - i];
                    sum += n[i];
                }
                uint32_t upto = sum;
#pragma unroll
                for (int i = 1; i < 64; i <<= 1) {
                    const uint32_t y = __shfl_up(upto, i);
                    if ((int)lane >= i) upto += y;
                }
                uint32_t before = upto - sum;
                if (before < left && upto >= left) {            // one lane: the digit is among its four
                    uint32_t i = 0;
                    while (i < 3 && before + n[i] < left) before += n[i++];
                    digit = 255 - 4 * lane - i;
                    above = before;
                }
            } else {                                           // the other one is cleared for the next digit
                for (uint32_t i = tid - 64; i < SELECT_COPIES * 256; i += SELECT_BLOCK - 64) hist[(shift / 8) & 1][0][i] = 0;
            }
            __syncthreads();
            found |= digit << shift;
            left -= above;
        }
    // tokens above `found` stay, and the first `left` of those that equal it
    uint32_t at = 0, equal_before = 0;
    for (uint32_t t0 = 0; t0 < len; t0 += SELECT_ROUND) {
        if (!once) load(t0);
        uint32_t more_n = 0, equal_n = 0;
        uint64_t more[SELECT_EACH], equal[SELECT_EACH];
#pragma unroll
        for (uint32_t i = 0; i < SELECT_EACH; i++) {
            const uint32_t t = t0 + mine + 64 * i, key = weight_key(x[i]);
            const bool fixed = t < len && (t < lo || t >= hi), open = t >= lo && t < hi && need;
            more[i] = __ballot(fixed || (open && key > found));
            equal[i] = __ballot(open && key == found);
            more_n += (uint32_t)__popcll(more[i]);
            equal_n += (uint32_t)__popcll(equal[i]);
        }
        if (lane == 0) {
            counts[wave][0] = more_n;
            counts[wave][1] = equal_n;
        }
        __syncthreads();
        // tokens of waves before this one that stay, and the round's totals
        uint32_t m = lane < SELECT_WAVES ? counts[lane][0] : 0, q = lane < SELECT_WAVES ? counts[lane][1] : 0;
#pragma unroll
        for (int i = 1; i < (int)SELECT_WAVES; i <<= 1) {
            const uint32_t ym = __shfl_up(m, i), yq = __shfl_up(q, i);
            if ((int)lane >= i) {
                m += ym;
                q += yq;
            }
        }
        uint32_t more_before = wave ? __shfl(m, (int)wave - 1) : 0, equal_at = equal_before + (wave ? __shfl(q, (int)wave - 1) : 0);
        // equal ones stay while there is room: min(equal ones before, left) of those before a token
        const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
        for (uint32_t i = 0; i < SELECT_EACH; i++) {
            const uint32_t t = t0 + mine + 64 * i, e = equal_at + (uint32_t)__popcll(equal[i] & below);
            const uint32_t gone_before = equal_before < left ? equal_before : left;            // equal ones that earlier rounds placed: counted in `at`
            const uint32_t to = at + more_before + (uint32_t)__popcll(more[i] & below) + (e < left ? e : left) - gone_before;
            if ((more[i] >> lane) & 1 || ((equal[i] >> lane) & 1 && e < left)) {
                kept[to] = t;
                out[to] = x[i];
            }
            more_before += (uint32_t)__popcll(more[i]);
            equal_at += (uint32_t)__popcll(equal[i]);
        }
        const uint32_t all_more = __shfl(m, (int)SELECT_WAVES - 1), all_equal = __shfl(q, (int)SELECT_WAVES - 1);
        const uint32_t was = equal_before < left ? equal_before : left;
        equal_before += all_equal;
        at += all_more + (equal_before < left ? equal_before : left) - was;
        __syncthreads();                                        // before the next round's counts, and before it reads what others may write
    }
    if (tid == 0) a.counts[pair] = a.keep;
}

struct MoveArgs {
    void* pages[2];
    const int32_t *table, *table_out;
    int32_t* lens_out;
    const uint32_t *kept, *counts;
    uint32_t n_pages, kv_heads, page_len, row_v, table_len, keep, slices, slice_v, rows;   // rows: of each block
    FastDiv page_div, slice_div;
};

// A block moves some vectors (a slice) of the rows that stay of one (sequence, KV head), keys or values, `rows` of them, MOVE_EACH a thread and step.  In
// place it is all rows, in order: a row moves to an index at or below its own, so when a step has read its rows the places it writes hold nothing that a
// later step reads.  8 sequences of 32 heads of 80 in f16 cut to 2048 tokens: into other pages 71 to 76 us, bound by memory: 164 MB written and 186 read (rows of 160 bytes end
// inside lines of 128), 4.6 to 4.9 TB/s.  In place 71 us for 92 MB written and 173 read (rows that stay where they are are left alone, and the slices of a row are read through
// two L2s), bound by the chain list -> table -> row of each step; one sequence of 8 heads of 128, 4100 tokens to 1024: 4.4 us elsewhere, 12.6 in four steps in place.
constexpr uint32_t MOVE_EACH = 4;

template <typename VecT> __global__ void __launch_bounds__(BLOCK) evict_move_kernel(MoveArgs a) {
    const uint32_t part = blockIdx.x % (2 * a.slices), pair = blockIdx.x / (2 * a.slices), which = part & 1, slice = part >> 1;
    const uint32_t b = pair / a.kv_heads, g = pair - b * a.kv_heads, count = a.counts[pair];
    if (part == 0 && g == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.lens_out[b] = (int32_t)count;
    const uint32_t step = BLOCK / a.slice_v, begin = blockIdx.y * a.rows;
    if (begin >= count) return;
    const uint32_t end = count - begin < a.rows ? count : begin + a.rows;
    VecT* pages = (VecT*)a.pages[which];
    uint32_t r, c;
    fd_divmod(threadIdx.x, a.slice_div, r, c);
    c += slice * a.slice_v;
    const bool mine = r < step && c < a.row_v;
    const int32_t* from_table = a.table + (uint64_t)b * a.table_len;
    const int32_t* to_table = a.table_out + (uint64_t)b * a.table_len;
    const uint32_t* kept = a.kept + (uint64_t)pair * a.keep;
    for (uint32_t i0 = begin; i0 < end; i0 += step * MOVE_EACH) {
        VecT x[MOVE_EACH];
        uint64_t to[MOVE_EACH];
        bool put[MOVE_EACH];
        uint32_t t[MOVE_EACH];
#pragma unroll
        for (uint32_t k = 0; k < MOVE_EACH; k++) {
            const uint32_t i = i0 + k * step + r;
            put[k] = mine && i < end;
            t[k] = put[k] ? kept[i] : 0;
        }
#pragma unroll
        for (uint32_t k = 0; k < MOVE_EACH; k++) {
            x[k] = VecT{};
            to[k] = 0;
            if (!put[k]) continue;
            uint32_t at, slot;
            fd_divmod(t[k], a.page_div, at, slot);
            const uint32_t src = (uint32_t)from_table[at];
            const uint64_t from = (((uint64_t)src * a.kv_heads + g) * a.page_len + slot) * a.row_v + c;
            fd_divmod(i0 + k * step + r, a.page_div, at, slot);
            const uint32_t dst = (uint32_t)to_table[at];
            to[k] = (((uint64_t)dst * a.kv_heads + g) * a.page_len + slot) * a.row_v + c;
            put[k] = dst < a.n_pages && !(src < a.n_pages && from == to[k]);
            if (put[k] && src < a.n_pages) x[k] = pages[from];
        }
#pragma unroll
        for (uint32_t k = 0; k < MOVE_EACH; k++) asm volatile("" : "+v"(x[k]));                  // the values have arrived before anyone writes
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < MOVE_EACH; k++)
            if (put[k]) pages[to[k]] = x[k];
    }
}

}  // namespace

extern "C" {

int rt_paged_append(rt_device* dev, int elem_bytes, const rt_paged_kv* kv, const int32_t* starts, uint32_t tokens, const void* k, const uint64_t k_strides[2],
                    const void* v, const uint64_t v_strides[2]) {
    static const char* const who = "rt_paged_append";
    RT_REQUIRE(elem_bytes == 2 || elem_bytes == 4, RT_ERR_ARG, "%s: elem_bytes must be 2 or 4, got %d", who, elem_bytes);
    int rc = rt_paged_rules(who, kv, (size_t)elem_bytes);
    if (rc) return rc;
    uint64_t st[2][2];
    if ((rc = rt_rows_rules(who, "k", tokens, kv->kv_heads, kv->head_dim, k_strides, &st[0][0], &st[0][1]))) return rc;
    if ((rc = rt_rows_rules(who, "v", tokens, kv->kv_heads, kv->head_dim, v_strides, &st[1][0], &st[1][1]))) return rc;
    RT_REQUIRE(k && v && starts, RT_ERR_NULL_POINTER, "%s: NULL operand", who);
    RT_REQUIRE(rt_aligned(k, (size_t)elem_bytes) && rt_aligned(v, (size_t)elem_bytes) && rt_aligned(starts, 4), RT_ERR_ALIGN, "%s: misaligned pointer", who);
    RT_REQUIRE((uint64_t)kv->kv_heads * kv->head_dim < 1u << 30, RT_ERR_SIZE, "%s: %u heads of %u columns", who, kv->kv_heads, kv->head_dim);
    rc = rt_enter(dev);
    if (rc) return rc;
    int vb = 16;
    for (; vb > elem_bytes; vb >>= 1) {
        bool fits = (uint64_t)kv->head_dim * elem_bytes % vb == 0 && rt_aligned(kv->k, (size_t)vb) && rt_aligned(kv->v, (size_t)vb) && rt_aligned(k, (size_t)vb) &&
                    rt_aligned(v, (size_t)vb);
        for (int i = 0; i < 4; i++) fits = fits && st[i / 2][i % 2] * elem_bytes % vb == 0;
        if (fits) break;
    }
    AppendArgs a;
    const uint32_t per = (uint32_t)(vb / elem_bytes);
    a.src[0] = k; a.src[1] = v;
    a.pages[0] = kv->k; a.pages[1] = kv->v;
    for (int i = 0; i < 2; i++) {
        a.token[i] = st[i][0] / per;
        a.head[i] = st[i][1] / per;
    }
    a.table = kv->table; a.lens = kv->lens; a.starts = starts;
    a.n_pages = kv->pages; a.kv_heads = kv->kv_heads; a.page_len = kv->page_len; a.seqs = kv->seqs; a.table_len = kv->table_len;
    a.row_v = kv->head_dim / per;
    a.tokens = tokens;
    a.page_div = make_fastdiv(kv->page_len);
    a.row_div = make_fastdiv(a.row_v);
    const dim3 grid(tokens < APPEND_ROW ? tokens : APPEND_ROW, (tokens + APPEND_ROW - 1) / APPEND_ROW), block(BLOCK);
    if (vb == 16) hipLaunchKernelGGL((paged_append_kernel<v4u>), grid, block, 0, dev->stream, a);
    else if (vb == 8) hipLaunchKernelGGL((paged_append_kernel<v2u>), grid, block, 0, dev->stream, a);
    else if (vb == 4) hipLaunchKernelGGL((paged_append_kernel<uint32_t>), grid, block, 0, dev->stream, a);
    else hipLaunchKernelGGL((paged_append_kernel<uint16_t>), grid, block, 0, dev->stream, a);
    RT_CHECK_LAUNCH("paged_append_kernel");
    return RT_OK;
}

int rt_paged_evict(rt_device* dev, int elem_bytes, const rt_paged_kv* kv, const float* weights, uint32_t keep, uint32_t first, uint32_t recent,
                   const int32_t* table_out, int32_t* lens_out, float* weights_out) {
    static const char* const who = "rt_paged_evict";
    RT_REQUIRE(elem_bytes == 2 || elem_bytes == 4, RT_ERR_ARG, "%s: elem_bytes must be 2 or 4, got %d", who, elem_bytes);
    int rc = rt_paged_rules(who, kv, (size_t)elem_bytes);
    if (rc) return rc;
    const uint32_t cap = kv->table_len * kv->page_len;
    RT_REQUIRE(keep > 0 && keep <= cap, RT_ERR_ARG, "%s: keep is %u of at most %u tokens", who, keep, cap);
    RT_REQUIRE((uint64_t)first + recent <= keep, RT_ERR_ARG, "%s: first %u and recent %u exceed keep %u", who, first, recent, keep);
    RT_REQUIRE((uint64_t)kv->kv_heads * kv->head_dim < 1u << 30, RT_ERR_SIZE, "%s: %u heads of %u columns", who, kv->kv_heads, kv->head_dim);
    RT_REQUIRE(weights && table_out && lens_out && weights_out, RT_ERR_NULL_POINTER, "%s: NULL operand", who);
    RT_REQUIRE(rt_aligned(weights, 4) && rt_aligned(table_out, 4) && rt_aligned(lens_out, 4) && rt_aligned(weights_out, 4), RT_ERR_ALIGN, "%s: misaligned pointer", who);
    const uint64_t pairs = (uint64_t)kv->seqs * kv->kv_heads;
    RT_REQUIRE(pairs <= RT_MAX_NUMEL / cap, RT_ERR_SIZE, "%s: weights are too large", who);
    int vb = 16;
    for (; vb > elem_bytes; vb >>= 1)
        if ((uint64_t)kv->head_dim * elem_bytes % vb == 0 && rt_aligned(kv->k, (size_t)vb) && rt_aligned(kv->v, (size_t)vb)) break;
    MoveArgs m;
    m.row_v = (uint32_t)((uint64_t)kv->head_dim * elem_bytes / vb);
    m.slice_v = m.row_v < (uint32_t)BLOCK ? m.row_v : BLOCK;
    // an extent of a launch has fewer than 2^32 threads (narrower slices, below, make no more than 8 blocks a CU)
    RT_REQUIRE(pairs * 2 * ((m.row_v + m.slice_v - 1) / m.slice_v) < (1ull << 32) / BLOCK, RT_ERR_SIZE, "%s: %u sequences, %u KV heads of %u columns", who, kv->seqs, kv->kv_heads,
               kv->head_dim);
    rc = rt_enter(dev);
    if (rc) return rc;
    void* scratch;
    if ((rc = rt_scratch(dev, (size_t)(pairs * (1 + (uint64_t)keep)) * sizeof(uint32_t), &scratch))) return rc;
    EvictArgs e;
    e.lens = kv->lens;
    e.weights = weights; e.weights_out = weights_out;
    e.counts = (uint32_t*)scratch;
    e.kept = e.counts + pairs;
    e.kv_heads = kv->kv_heads; e.cap = cap; e.keep = keep; e.first = first; e.recent = recent;
    hipLaunchKernelGGL(evict_select_kernel, dim3(kv->kv_heads, kv->seqs), dim3(SELECT_BLOCK), 0, dev->stream, e);
    RT_CHECK_LAUNCH("evict_select_kernel");
    m.pages[0] = kv->k; m.pages[1] = kv->v;
    m.table = kv->table; m.table_out = table_out; m.lens_out = lens_out;
    m.kept = e.kept; m.counts = e.counts;
    m.n_pages = kv->pages; m.kv_heads = kv->kv_heads; m.page_len = kv->page_len; m.table_len = kv->table_len; m.keep = keep;
    // Elsewhere: whole rows.  In place the rows of a pair cannot be shared out, but their columns can: slices of 64 bytes at least, as many
    // as give four blocks a CU.
    const bool in_place = table_out == kv->table;
    if (in_place)
        while (m.slice_v > 4 && pairs * 2 * ((m.row_v + m.slice_v - 1) / m.slice_v) < 4ull * dev->num_cus) m.slice_v = (m.slice_v + 1) / 2;
    m.slices = (m.row_v + m.slice_v - 1) / m.slice_v;
    m.page_div = make_fastdiv(kv->page_len);
    m.slice_div = make_fastdiv(m.slice_v);
    const uint32_t one_step = BLOCK / m.slice_v * MOVE_EACH;
    m.rows = one_step;                                          // of a block: one step where that gives no more than eight blocks a CU, as many as it takes otherwise
    const uint64_t wanted = pairs * 2 * m.slices * keep / (8ull * dev->num_cus);
    if (wanted > m.rows) m.rows = (uint32_t)((wanted + one_step - 1) / one_step * one_step);
    if (in_place) m.rows = keep;
    const dim3 grid((unsigned)(pairs * 2 * m.slices), (keep + m.rows - 1) / m.rows), block(BLOCK);
    if (vb == 16) hipLaunchKernelGGL((evict_move_kernel<v4u>), grid, block, 0, dev->stream, m);
    else if (vb == 8) hipLaunchKernelGGL((evict_move_kernel<v2u>), grid, block, 0, dev->stream, m);
    else if (vb == 4) hipLaunchKernelGGL((evict_move_kernel<uint32_t>), grid, block, 0, dev->stream, m);
    else hipLaunchKernelGGL((evict_move_kernel<uint16_t>), grid, block, 0, dev->stream, m);
    RT_CHECK_LAUNCH("evict_move_kernel");
    return RT_OK;
}

}  // extern "C"
