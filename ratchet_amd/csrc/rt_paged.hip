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
// Moves each row once; bound by memory for prompts and by the chain starts -> lens and table -> store for single tokens.
template <typename VecT> __global__ void __launch_bounds__(BLOCK) paged_append_kernel(AppendArgs a) {
    const uint32_t token = blockIdx.x;
    const uint32_t b = at_find(a.starts, a.seqs, token);
    if (b == a.seqs) return;
    const int32_t top = (int32_t)a.tokens;
    int32_t lo = a.starts[b], hi = a.starts[b + 1];
    lo = lo < 0 ? 0 : lo;
    hi = hi > top ? top : hi;
    if ((int32_t)token < lo || (int32_t)token >= hi) return;
    int32_t len = a.lens[b];
    len = len < 0 ? 0 : len;
    const int32_t t = len - hi + (int32_t)token;               // both below 2^31
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
    const int32_t *table, *lens;
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

// exclusive sums over the block of two flags a thread, in thread order; totals to all
__device__ __forceinline__ void block_ranks(bool x, bool y, uint32_t* lds, uint32_t& rank_x, uint32_t& rank_y, uint32_t& total_x, uint32_t& total_y) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint64_t bx = __ballot(x), by = __ballot(y), below = ((uint64_t)1 << lane) - 1;
    if (lane == 0) {
        lds[2 * wave] = (uint32_t)__popcll(bx);
        lds[2 * wave + 1] = (uint32_t)__popcll(by);
    }
    __syncthreads();
    rank_x = (uint32_t)__popcll(bx & below);
    rank_y = (uint32_t)__popcll(by & below);
    total_x = total_y = 0;
    for (uint32_t i = 0; i < SELECT_BLOCK / 64; i++) {
        if (i < wave) {
            rank_x += lds[2 * i];
            rank_y += lds[2 * i + 1];
        }
        total_x += lds[2 * i];
        total_y += lds[2 * i + 1];
    }
    __syncthreads();
}

// A block to a (sequence, KV head).  The weight of the last token that stays is found digit by digit, eight bits at a time from the top
// (a histogram of the candidates that share the digits found so far); then one walk over the tokens writes the list of those that stay and
// moves their weights.  A weight moves to an index at or below its own and a walk's step reads its tokens before it writes, so weights_out may be weights.
__global__ void __launch_bounds__(SELECT_BLOCK) evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t hist[256], ranks[2 * SELECT_BLOCK / 64], digit, above;
    const uint32_t g = blockIdx.x, b = blockIdx.y, pair = b * a.kv_heads + g, tid = threadIdx.x;
    int32_t raw = a.lens[b];
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
    uint32_t found = 0, left = need;               // the digits so far; how many of the candidates that share them stay
    if (need)
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (uint32_t t = lo + tid; t < hi; t += SELECT_BLOCK) {
                const uint32_t key = weight_key(w[t]);
                if (shift == 24 || (key >> (shift + 8)) == (found >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t sum = 0;
                int d = 255;
                for (; d > 0 && sum + hist[d] < left; d--) sum += hist[d];
                digit = (uint32_t)d;
                above = sum;
            }
            __syncthreads();
            found |= digit << shift;
            left -= above;
            __syncthreads();
        }
    // tokens above `found` stay, and the first `left` of those that equal it
    uint32_t at = 0, equal_before = 0;
    for (uint32_t t0 = 0; t0 < len; t0 += SELECT_BLOCK) {
        const uint32_t t = t0 + tid;
        const bool here = t < len, fixed = here && (t < lo || t >= hi), open = here && !fixed && need;
        const float x = here ? w[t] : 0.0f;
        const uint32_t key = weight_key(x);
        const bool more = fixed || (open && key > found), equal = open && key == found;
        uint32_t r_more, r_equal, n_more, n_equal;
        block_ranks(more, equal, ranks, r_more, r_equal, n_more, n_equal);
        // of the equal ones before this thread's, so many stay
        const uint32_t room = left > equal_before ? left - equal_before : 0;
        const uint32_t to = at + r_more + (r_equal < room ? r_equal : room);
        if (more || (equal && r_equal < room)) {
            kept[to] = t;
            out[to] = x;
        }
        at += n_more + (n_equal < room ? n_equal : room);
        equal_before += n_equal;
    }
    if (tid == 0) a.counts[pair] = a.keep;
}

struct MoveArgs {
    void* pages[2];
    const int32_t *table, *table_out;
    int32_t* lens_out;
    const uint32_t *kept, *counts;
    uint32_t n_pages, kv_heads, page_len, row_v, seqs, table_len, keep, slices, slice_v, rows;   // rows: of each block
    FastDiv page_div, slice_div;
};

// A block moves some vectors (a slice) of the rows that stay of one (sequence, KV head), keys or values, `rows` of them; in place it is all rows, in order:
// a row moves to an index at or below its own, so when a step has read its rows the places it writes hold nothing that a later step reads.
template <typename VecT> __global__ void __launch_bounds__(BLOCK) evict_move_kernel(MoveArgs a) {
    const uint32_t part = blockIdx.x % (2 * a.slices), pair = blockIdx.x / (2 * a.slices), which = part & 1, slice = part >> 1;
    const uint32_t b = pair / a.kv_heads, g = pair - b * a.kv_heads, count = a.counts[pair];
    if (part == 0 && g == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.lens_out[b] = (int32_t)count;
    const uint32_t c0 = slice * a.slice_v, width = a.row_v - c0 < a.slice_v ? a.row_v - c0 : a.slice_v;
    const uint32_t step = BLOCK / a.slice_v, begin = blockIdx.y * a.rows, end = count - begin < a.rows ? count : begin + a.rows;
    if (begin >= count) return;
    VecT* pages = (VecT*)a.pages[which];
    uint32_t r, c;
    fd_divmod(threadIdx.x, a.slice_div, r, c);
    const int32_t* from_table = a.table + (uint64_t)b * a.table_len;
    const int32_t* to_table = a.table_out + (uint64_t)b * a.table_len;
    for (uint32_t i0 = begin; i0 < end; i0 += step) {
        const uint32_t i = i0 + r;
        const bool mine = r < step && c < width && i < end;
        VecT x = {};
        uint64_t to = 0, from = 0;
        bool put = false;
        if (mine) {
            uint32_t at, slot;
            const uint32_t t = a.kept[(uint64_t)pair * a.keep + i];
            fd_divmod(t, a.page_div, at, slot);
            const uint32_t src = (uint32_t)from_table[at];
            from = (((uint64_t)src * a.kv_heads + g) * a.page_len + slot) * a.row_v + c0 + c;
            fd_divmod(i, a.page_div, at, slot);
            const uint32_t dst = (uint32_t)to_table[at];
            to = (((uint64_t)dst * a.kv_heads + g) * a.page_len + slot) * a.row_v + c0 + c;
            put = dst < a.n_pages && !(src < a.n_pages && from == to);
            if (put && src < a.n_pages) x = pages[from];
        }
        asm volatile("" : "+v"(x));                            // the value has arrived before anyone writes
        __syncthreads();
        if (put) pages[to] = x;
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
    const dim3 grid(tokens), block(BLOCK);
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
    rc = rt_enter(dev);
    if (rc) return rc;
    int vb = 16;
    for (; vb > elem_bytes; vb >>= 1)
        if ((uint64_t)kv->head_dim * elem_bytes % vb == 0 && rt_aligned(kv->k, (size_t)vb) && rt_aligned(kv->v, (size_t)vb)) break;
    void* scratch;
    if ((rc = rt_scratch(dev, (size_t)(pairs * (1 + (uint64_t)keep)) * sizeof(uint32_t), &scratch))) return rc;
    EvictArgs e;
    e.table = kv->table; e.lens = kv->lens;
    e.weights = weights; e.weights_out = weights_out;
    e.counts = (uint32_t*)scratch;
    e.kept = e.counts + pairs;
    e.kv_heads = kv->kv_heads; e.cap = cap; e.keep = keep; e.first = first; e.recent = recent;
    hipLaunchKernelGGL(evict_select_kernel, dim3(kv->kv_heads, kv->seqs), dim3(SELECT_BLOCK), 0, dev->stream, e);
    RT_CHECK_LAUNCH("evict_select_kernel");
    MoveArgs m;
    m.pages[0] = kv->k; m.pages[1] = kv->v;
    m.table = kv->table; m.table_out = table_out; m.lens_out = lens_out;
    m.kept = e.kept; m.counts = e.counts;
    m.n_pages = kv->pages; m.kv_heads = kv->kv_heads; m.page_len = kv->page_len; m.seqs = kv->seqs; m.table_len = kv->table_len; m.keep = keep;
    m.row_v = (uint32_t)((uint64_t)kv->head_dim * elem_bytes / vb);
    m.slice_v = m.row_v < 4 ? m.row_v : 4;
    m.slices = (m.row_v + m.slice_v - 1) / m.slice_v;
    m.page_div = make_fastdiv(kv->page_len);
    m.slice_div = make_fastdiv(m.slice_v);
    m.rows = table_out == kv->table || keep < 256 ? keep : 256;
    const uint64_t blocks = pairs * 2 * m.slices, chunks = (keep + m.rows - 1) / m.rows;
    RT_REQUIRE(blocks <= 0x7fffffffull && chunks <= 65535, RT_ERR_SIZE, "%s: too many rows", who);
    const dim3 grid((unsigned)blocks, (unsigned)chunks), block(BLOCK);
    if (vb == 16) hipLaunchKernelGGL((evict_move_kernel<v4u>), grid, block, 0, dev->stream, m);
    else if (vb == 8) hipLaunchKernelGGL((evict_move_kernel<v2u>), grid, block, 0, dev->stream, m);
    else if (vb == 4) hipLaunchKernelGGL((evict_move_kernel<uint32_t>), grid, block, 0, dev->stream, m);
    else hipLaunchKernelGGL((evict_move_kernel<uint16_t>), grid, block, 0, dev->stream, m);
    RT_CHECK_LAUNCH("evict_move_kernel");
    return RT_OK;
}

}  // extern "C"
