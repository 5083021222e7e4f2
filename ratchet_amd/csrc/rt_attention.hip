// Attention: the entry points, the choice of the kernel, and the kernels that take any head dim, stride and alignment.
#include <math.h>

#include "rt_attention.h"

namespace {

constexpr int WAVES = 4, BLOCK = 64 * WAVES;
constexpr uint32_t GRID_ROW = 1u << 22;          // blocks to a row of the grid: an extent of a launch has fewer than 2^32 threads

// A wave to a (query, head) row.  A lane computes the score of one key of a tile of 64; the tile's weights then go round the wave, key by key, and
// each lane adds them to its columns.  Hidden keys are skipped there, so nothing they hold is ever multiplied.
// Simple, and 50 to 800 times slower than the tiles: bound by its scalar dot products and uncoalesced key reads ([4,6,1500,64] f32 14.5 ms, with tiles 0.15)
template <typename T, bool PAGED, bool SCORED>
__global__ void __launch_bounds__(BLOCK) attention_any_kernel(AttnArgs a, uint64_t rows) {
    const uint32_t lane = threadIdx.x % 64;
    const uint64_t row = ((uint64_t)blockIdx.y * GRID_ROW + blockIdx.x) * WAVES + threadIdx.x / 64;
    if (row >= rows) return;
    const uint32_t h = (uint32_t)(row % a.heads);
    uint64_t at = row / a.heads;
    uint32_t b, j;
    AttnSeq s;
    if (PAGED) {
        b = at_find(a.starts, a.seqs, (uint32_t)at);
        if (b == a.seqs) return;
        s = at_seq<true>(a, b);
        if (at < s.first || at - s.first >= s.count) return;
        j = (uint32_t)at - s.first;
    } else {
        b = (uint32_t)(at / a.tokens);
        j = (uint32_t)(at % a.tokens);
        s = at_seq<false>(a, b);
    }
    const uint32_t g = h / a.group, D = a.dim;
    const T* q = (const T*)a.q + b * a.q_b + h * a.q_h + (uint64_t)(s.first + j) * a.q_t;
    const T* k = (const T*)a.k + g * a.k_h + (PAGED ? 0 : b * a.k_b);
    const T* v = (const T*)a.v + g * a.v_h + (PAGED ? 0 : b * a.v_b);
    const AttnRow r = at_row<SCORED>(a, SCORED ? at_texts(a, b) : AttnTexts{}, b, s, j);
    const float slope = SCORED && a.slopes ? at_slope(a, h) : 0.0f;
    float m = -INFINITY, l = 0.0f, o[AT_MAX_DIM / 64];
#pragma unroll
    for (int i = 0; i < AT_MAX_DIM / 64; i++) o[i] = 0.0f;
    for (int32_t t0 = r.lo / 64 * 64; t0 <= r.limit; t0 += 64) {
        if (t0 >= r.front && r.p - (t0 + 63) >= a.window) continue;
        const int32_t t = t0 + (int32_t)lane;
        bool seen = at_sees<SCORED>(a, r, t);
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
#pragma unroll
        for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
        const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.0f : m_new;
        const float old = at_exp2(m - base), w = seen ? at_exp2(x - base) : 0.0f;
        m = m_new;
        float sum = w;
#pragma unroll
        for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
        l = __builtin_fmaf(l, old, sum);
#pragma unroll
        for (int i = 0; i < AT_MAX_DIM / 64; i++) o[i] *= old;
        while (todo) {
            const int src = __builtin_ctzll(todo);
            todo &= todo - 1;
            const float wi = __shfl(w, src);
            const uint64_t from = __shfl(v_at, src);
#pragma unroll
            for (int i = 0; i < AT_MAX_DIM / 64; i++)
                if (i * 64 + lane < D) o[i] = __builtin_fmaf(wi, Ar<T>::widen(v[from + i * 64 + lane]), o[i]);
        }
    }
    T* y = (T*)a.y + b * a.y_b + h * a.y_h + (uint64_t)(s.first + j) * a.y_t;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;             // NaN stays NaN; a row that sees nothing is 0
#pragma unroll
    for (int i = 0; i < AT_MAX_DIM / 64; i++)
        if (i * 64 + lane < D) y[i * 64 + lane] = Ar<T>::conv(o[i] * inv);
    if (a.lse && lane == 0) a.lse[b * a.l_b + h * a.l_h + (uint64_t)(s.first + j) * a.l_t] = at_lse(m, l);
}

// Received weights from finished statistics: a wave owns 64 keys of a KV head, computes each query's scores with them again and adds
// 2^(s - lse) up in the order of the queries and heads.
template <typename T>
__global__ void __launch_bounds__(64) attention_weights_any_kernel(AttnArgs a, const float* weights, float* out) {
    const uint32_t lane = threadIdx.x, g = blockIdx.y, b = blockIdx.z;
    const AttnSeq s = at_seq<true>(a, b);
    const int32_t t0 = (int32_t)blockIdx.x * 64, t = t0 + (int32_t)lane;
    if (t0 >= s.keys) return;
    uint32_t slot = 0;
    const int32_t page = t < s.keys ? at_page(a, b, (uint32_t)t, slot) : -1;
    const uint64_t at = ((uint64_t)b * a.kv_heads + g) * a.cap + (uint32_t)t;
    const T* k = (const T*)a.k + g * a.k_h + (uint64_t)(page < 0 ? 0 : page) * a.k_b + slot * a.k_t;
    float sum = t < s.keys && t < s.shift ? weights[at] : 0.0f;
    for (uint32_t j = 0; j < s.count; j++) {
        const int32_t limit = at_limit(a, s, j), p = at_position(s, j);
        if (t0 > limit || (t0 >= a.sinks && p - (t0 + 63) >= a.window)) continue;
        const bool seen = page >= 0 && at_visible(a, t, limit, p);
        for (uint32_t h = g * a.group; h < (g + 1) * a.group; h++) {
            const T* q = (const T*)a.q + h * a.q_h + (uint64_t)(s.first + j) * a.q_t;
            const float lse = a.lse[h * a.l_h + (uint64_t)(s.first + j) * a.l_t];
            if (!seen || lse == -INFINITY) continue;           // a row whose scores are all -inf weighs nothing
            float dot = 0.0f;
            for (uint32_t d = 0; d < a.dim; d++) dot = __builtin_fmaf(Ar<T>::widen(q[d]), Ar<T>::widen(k[d]), dot);
            sum += at_exp2(__builtin_fmaf(lse, -1.4426950408889634f, dot * a.c));
        }
    }
    if (t < s.keys) out[at] = sum;
}

template <typename T> int launch_any(rt_device* dev, const AttnArgs& a, bool paged, const float* weights, float* weights_out) {
    const uint64_t rows = (uint64_t)(paged ? 1 : a.seqs) * a.tokens * a.heads, blocks = (rows + WAVES - 1) / WAVES;
    RT_REQUIRE(blocks <= 65535ull * GRID_ROW, RT_ERR_SIZE, "attention: too many rows");
    const dim3 grid((unsigned)(blocks < GRID_ROW ? blocks : GRID_ROW), (unsigned)((blocks + GRID_ROW - 1) / GRID_ROW));
    if (paged && a.scored) hipLaunchKernelGGL((attention_any_kernel<T, true, true>), grid, dim3(BLOCK), 0, dev->stream, a, rows);
    else if (paged) hipLaunchKernelGGL((attention_any_kernel<T, true, false>), grid, dim3(BLOCK), 0, dev->stream, a, rows);
    else if (a.scored) hipLaunchKernelGGL((attention_any_kernel<T, false, true>), grid, dim3(BLOCK), 0, dev->stream, a, rows);
    else hipLaunchKernelGGL((attention_any_kernel<T, false, false>), grid, dim3(BLOCK), 0, dev->stream, a, rows);
    RT_CHECK_LAUNCH("attention_any_kernel");
    if (weights_out) {
        hipLaunchKernelGGL((attention_weights_any_kernel<T>), dim3((a.cap + 63) / 64, a.kv_heads, a.seqs), dim3(64), 0, dev->stream, a, weights, weights_out);
        RT_CHECK_LAUNCH("attention_weights_any_kernel");
    }
    return RT_OK;
}

int dispatch(rt_device* dev, int dt, AttnArgs& a, bool paged, const float* weights, float* weights_out) {
    bool done;
    int rc;
    if (a.scored) rc = dt == RT_F32 ? rt_attention_scored_f32(dev, a, paged, &done) : dt == RT_F16 ? rt_attention_scored_f16(dev, a, paged, &done) : rt_attention_scored_bf16(dev, a, paged, &done);
    else rc = dt == RT_F32 ? rt_attention_tile_f32(dev, a, paged, &done) : dt == RT_F16 ? rt_attention_tile_f16(dev, a, paged, &done) : rt_attention_tile_bf16(dev, a, paged, &done);
    if (rc || (done && !weights_out)) return rc;
    if (done) {
        switch (dt) {
            case RT_F32: return rt_attention_weights_f32(dev, a, weights, weights_out);
            case RT_F16: return rt_attention_weights_f16(dev, a, weights, weights_out);
            default: return rt_attention_weights_bf16(dev, a, weights, weights_out);
        }
    }
    void* none = nullptr;
    if ((rc = at_workspace(dev, a, 0, &none))) return rc;
    switch (dt) {
        case RT_F32: return launch_any<float>(dev, a, paged, weights, weights_out);
        case RT_F16: return launch_any<half_t>(dev, a, paged, weights, weights_out);
        default: return launch_any<bf16_t>(dev, a, paged, weights, weights_out);
    }
}

constexpr uint32_t MOST_TOKENS = AT_MOST_TOKENS;

int head_rules(const char* who, int dt, uint32_t heads, uint32_t kv_heads, uint32_t dim, float scale, uint32_t window, uint32_t sinks, AttnArgs& a) {
    RT_REQUIRE(rt_is_float_dt(dt), RT_ERR_DTYPE, "%s: dtype %d is not F32, F16 or BF16", who, dt);
    RT_REQUIRE(heads > 0 && kv_heads > 0 && dim > 0, RT_ERR_SHAPE, "%s: zero extent", who);
    RT_REQUIRE(heads % kv_heads == 0, RT_ERR_SHAPE, "%s: %u heads are no multiple of %u KV heads", who, heads, kv_heads);
    RT_REQUIRE(kv_heads <= 65535, RT_ERR_SIZE, "%s: %u KV heads", who, kv_heads);
    RT_REQUIRE(dim <= (uint32_t)AT_MAX_DIM, RT_ERR_SIZE, "%s: head dim %u exceeds %d", who, dim, AT_MAX_DIM);
    RT_REQUIRE(isfinite(scale), RT_ERR_ARG, "%s: scale is not finite", who);
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.group = heads / kv_heads;
    a.group_div = make_fastdiv(a.group);
    a.dim = dim;
    a.c = scale * 1.4426950408889634f;
    a.window = window == 0 || window >= MOST_TOKENS ? AT_FAR : (int32_t)window;               // as far as positions go
    a.sinks = sinks > MOST_TOKENS ? AT_MOST_TOKENS : (int32_t)sinks;
    return RT_OK;
}

// What changes or masks the scores; `documents`: the call may have them
int score_rules(const char* who, const rt_scores* scores, float scale, uint32_t batch, bool documents, bool causal, AttnArgs& a) {
    RT_REQUIRE(scores, RT_ERR_NULL_POINTER, "%s: NULL scores", who);
    RT_REQUIRE(scores->cap >= 0.0f && isfinite(scores->cap), RT_ERR_ARG, "%s: cap must be finite and not negative", who);
    RT_REQUIRE(scores->cap == 0.0f || isfinite(2.0f * scores->cap * 1.4426950408889634f), RT_ERR_ARG, "%s: cap is too large", who);        // at_capped multiplies by its double
    RT_REQUIRE(scores->cap == 0.0f || isfinite(scale / scores->cap), RT_ERR_ARG, "%s: scale / cap is not finite", who);
    RT_REQUIRE(documents || !scores->documents, RT_ERR_ARG, "%s: sequences are not cut into documents", who);
    RT_REQUIRE(!scores->documents == !scores->n_documents, RT_ERR_SHAPE, "%s: %u documents", who, scores->n_documents);
    RT_REQUIRE(!scores->prefix || causal, RT_ERR_ARG, "%s: a prefix needs causal attention", who);
    RT_REQUIRE(scores->n_documents <= (uint32_t)AT_MOST_TOKENS && (uint64_t)batch * (scores->n_documents + 1ull) <= RT_MAX_NUMEL, RT_ERR_SIZE, "%s: %u documents", who, scores->n_documents);
    RT_REQUIRE(rt_aligned(scores->slopes, 4) && rt_aligned(scores->documents, 4) && rt_aligned(scores->prefix, 4), RT_ERR_ALIGN, "%s: misaligned pointer", who);
    a.scored = scores->cap != 0.0f || scores->slopes || scores->documents || scores->prefix;       // else it is attention as it ever was
    a.most = scores->cap * 1.4426950408889634f;
    a.most_in = scores->cap != 0.0f ? scale / scores->cap : 0.0f;
    // tanh y = y (t0 + t1 y^2 + t2 y^4 + t3 y^6), through its values at Chebyshev's points of y^2 <= 0.16 and 1e-7 of it off at most.  Where k^6 is too small for f32, y - y^3 / 3,
    // 2^-23 of it off below 2^-5.  Only where no power of scale / cap leaves f32's range
    const float k = a.most_in < 0.0f ? -a.most_in : a.most_in;
    a.near_limit = -1.0f;
    if (k > 0x1p-19f && k < 0x1p16f && a.most > 0x1p-16f && (a.most < 0x1p16f || k < 1.0f)) {
        static const double tanh_terms[4] = {0.9999999013476046, -0.3333135628726226, 0.1327087433318406, -0.04754934670684051};
        double power = (double)a.most * k;
        for (int i = 0; i < 4; i++, power *= (double)k * k) a.near[i] = (float)(tanh_terms[i] * power);
        a.near_limit = 0.4f / k;
    } else if (k <= 0x1p-19f && a.most > 1.0f) {                  // (a scale of 0 too: capped scores are 0)
        const double c = (double)a.most * k;
        a.near[0] = (float)c;
        a.near[1] = (float)(-c * k * k / 3);
        a.near_limit = k > 0x1p-55f ? 0x1p-5f / k : 0x1p50f;
    }
    a.slopes = scores->slopes;
    a.documents = scores->documents;
    a.n_documents = scores->n_documents;
    a.prefix = scores->prefix;
    return RT_OK;
}

// The last extent's stride is 1; elements of one tensor lie below 2^40.  A stride of an extent of 1 is never taken, so it does not decide about the layout: 0.
int stride_rules(const char* who, const char* what, const uint32_t shape[4], const uint64_t* strides, uint64_t out[4]) {
    unsigned __int128 dense = 1, last = 0;
    for (int i = 3; i >= 0; i--) {
        RT_REQUIRE(strides || dense <= RT_MAX_NUMEL, RT_ERR_SIZE, "%s: %s is too large", who, what);
        out[i] = shape[i] == 1 ? 0 : strides ? strides[i] : (uint64_t)dense;
        dense *= shape[i];
        last += (unsigned __int128)(shape[i] - 1) * out[i];
    }
    RT_REQUIRE(last < RT_MAX_NUMEL, RT_ERR_SIZE, "%s: %s is too large", who, what);
    RT_REQUIRE(shape[3] == 1 || out[3] == 1, RT_ERR_ARG, "%s: the last stride of %s is not 1", who, what);
    return RT_OK;
}

// Whether two index tuples can name the same element: extents in the order of their strides, each stride beyond what the smaller ones span
bool may_overlap(const uint32_t shape[4], const uint64_t strides[4]) {
    int order[4] = {0, 1, 2, 3};
    for (int i = 1; i < 4; i++)
        for (int j = i; j > 0 && strides[order[j]] < strides[order[j - 1]]; j--) {
            const int t = order[j];
            order[j] = order[j - 1];
            order[j - 1] = t;
        }
    uint64_t span = 0;
    for (int i = 0; i < 4; i++) {
        const int at = order[i];
        if (shape[at] == 1) continue;
        if (strides[at] <= span) return true;
        span += (uint64_t)(shape[at] - 1) * strides[at];
    }
    return false;
}

}  // namespace

int rt_paged_rules(const char* who, const rt_paged_kv* kv, size_t elem_bytes) {
    RT_REQUIRE(kv, RT_ERR_NULL_POINTER, "%s: NULL cache", who);
    RT_REQUIRE(kv->pages > 0 && kv->kv_heads > 0 && kv->page_len > 0 && kv->head_dim > 0 && kv->seqs > 0 && kv->table_len > 0, RT_ERR_SHAPE,
               "%s: zero extent in the cache", who);
    RT_REQUIRE(kv->seqs <= 65535 && kv->kv_heads <= 65535, RT_ERR_SIZE, "%s: %u sequences, %u KV heads", who, kv->seqs, kv->kv_heads);
    RT_REQUIRE(kv->pages <= 0x7fffffffu, RT_ERR_SIZE, "%s: %u pages", who, kv->pages);
    RT_REQUIRE((uint64_t)kv->table_len * kv->page_len <= MOST_TOKENS, RT_ERR_SIZE, "%s: a table of %u pages of %u tokens is too long", who, kv->table_len, kv->page_len);
    RT_REQUIRE((uint64_t)kv->page_len * kv->head_dim <= RT_MAX_NUMEL / kv->kv_heads && (uint64_t)kv->page_len * kv->head_dim * kv->kv_heads <= RT_MAX_NUMEL / kv->pages,
               RT_ERR_SIZE, "%s: cache too large", who);
    RT_REQUIRE(kv->k && kv->v && kv->table && kv->lens, RT_ERR_NULL_POINTER, "%s: NULL pointer in the cache", who);
    RT_REQUIRE(rt_aligned(kv->k, elem_bytes) && rt_aligned(kv->v, elem_bytes) && rt_aligned(kv->table, 4) && rt_aligned(kv->lens, 4), RT_ERR_ALIGN,
               "%s: misaligned pointer in the cache", who);
    return RT_OK;
}

int rt_rows_rules(const char* who, const char* what, uint32_t tokens, uint32_t heads, uint32_t dim, const uint64_t strides[2], uint64_t* token, uint64_t* head) {
    *token = tokens == 1 ? 0 : strides ? strides[0] : (uint64_t)heads * dim;                  // of an extent of 1: as in stride_rules
    *head = heads == 1 ? 0 : strides ? strides[1] : dim;
    RT_REQUIRE(tokens > 0, RT_ERR_SHAPE, "%s: no tokens", who);
    RT_REQUIRE(tokens <= MOST_TOKENS, RT_ERR_SIZE, "%s: %u tokens", who, tokens);
    RT_REQUIRE(*token < RT_MAX_NUMEL / tokens && *head < RT_MAX_NUMEL / heads, RT_ERR_SIZE, "%s: %s is too large", who, what);
    return RT_OK;
}

namespace {

int attention(const char* who, rt_device* dev, int dt, const void* q, const uint32_t q_shape[4], const uint64_t q_strides[4], const void* k, const uint64_t k_strides[4],
                 const void* v, const uint64_t v_strides[4], const uint32_t kv_shape[4], const int32_t* lens, void* y, const uint64_t y_strides[4], float* lse,
                 float scale, int causal, uint32_t window, uint32_t sinks, const rt_scores* scores, bool scored) {
    AttnArgs a = {};
    RT_REQUIRE(q_shape && kv_shape, RT_ERR_NULL_POINTER, "%s: NULL shape", who);
    int rc = head_rules(who, dt, q_shape[1], kv_shape[1], q_shape[3], scale, window, sinks, a);
    if (rc) return rc;
    RT_REQUIRE(q_shape[0] > 0 && q_shape[2] > 0 && kv_shape[2] > 0, RT_ERR_SHAPE, "%s: zero extent", who);
    RT_REQUIRE(q_shape[0] == kv_shape[0] && q_shape[3] == kv_shape[3], RT_ERR_SHAPE, "%s: q and k differ in batch or head dim", who);
    RT_REQUIRE(q_shape[0] <= 65535, RT_ERR_SIZE, "%s: batch %u", who, q_shape[0]);
    RT_REQUIRE(q_shape[2] <= MOST_TOKENS && kv_shape[2] <= MOST_TOKENS, RT_ERR_SIZE, "%s: %u queries, %u keys", who, q_shape[2], kv_shape[2]);
    RT_REQUIRE(causal == 0 || causal == 1, RT_ERR_ARG, "%s: causal is %d", who, causal);
    RT_REQUIRE(causal || (window == 0 && sinks == 0), RT_ERR_ARG, "%s: a window needs causal attention", who);
    if (scored && (rc = score_rules(who, scores, scale, q_shape[0], true, causal != 0, a))) return rc;
    uint64_t qs[4], ks[4], vs[4], ys[4];
    if ((rc = stride_rules(who, "q", q_shape, q_strides, qs))) return rc;
    if ((rc = stride_rules(who, "k", kv_shape, k_strides, ks))) return rc;
    if ((rc = stride_rules(who, "v", kv_shape, v_strides, vs))) return rc;
    if ((rc = stride_rules(who, "y", q_shape, y_strides, ys))) return rc;
    RT_REQUIRE(!may_overlap(q_shape, ys), RT_ERR_ARG, "%s: elements of y overlap", who);
    RT_REQUIRE(q && k && v && y, RT_ERR_NULL_POINTER, "%s: NULL operand", who);
    const size_t e = (size_t)rt_dt_bytes(dt);
    RT_REQUIRE(rt_aligned(q, e) && rt_aligned(k, e) && rt_aligned(v, e) && rt_aligned(y, e) && rt_aligned(lse, 4) && rt_aligned(lens, 4), RT_ERR_ALIGN,
               "%s: misaligned pointer", who);
    rc = rt_enter(dev);
    if (rc) return rc;
    a.q = q; a.k = k; a.v = v; a.y = y; a.lse = lse; a.lens = lens;
    a.q_b = qs[0]; a.q_h = qs[1]; a.q_t = qs[2];
    a.k_b = ks[0]; a.k_h = ks[1]; a.k_t = ks[2];
    a.v_b = vs[0]; a.v_h = vs[1]; a.v_t = vs[2];
    a.y_b = ys[0]; a.y_h = ys[1]; a.y_t = ys[2];
    a.l_t = 1; a.l_h = q_shape[2]; a.l_b = (uint64_t)q_shape[1] * q_shape[2];
    a.seqs = q_shape[0];
    a.tokens = q_shape[2];
    a.cap = kv_shape[2];
    a.causal = causal;
    return dispatch(dev, dt, a, false, nullptr, nullptr);
}

int paged_attention(const char* who, rt_device* dev, int dt, const void* q, const uint64_t q_strides[2], uint32_t tokens, uint32_t heads, const rt_paged_kv* kv,
                       const int32_t* starts, void* y, float* lse, const float* weights, float* weights_out, float scale, uint32_t window, uint32_t sinks,
                    const rt_scores* scores, bool scored) {
    AttnArgs a = {};
    RT_REQUIRE(kv, RT_ERR_NULL_POINTER, "%s: NULL cache", who);
    int rc = head_rules(who, dt, heads, kv->kv_heads, kv->head_dim, scale, window, sinks, a);
    if (rc) return rc;
    const size_t e = (size_t)rt_dt_bytes(dt);
    if ((rc = rt_paged_rules(who, kv, e))) return rc;
    if ((rc = rt_rows_rules(who, "q", tokens, heads, kv->head_dim, q_strides, &a.q_t, &a.q_h))) return rc;
    if (scored && (rc = score_rules(who, scores, scale, kv->seqs, false, true, a))) return rc;
    RT_REQUIRE(q && starts && y, RT_ERR_NULL_POINTER, "%s: NULL operand", who);
    RT_REQUIRE(!weights == !weights_out, RT_ERR_NULL_POINTER, "%s: weights and weights_out go together", who);
    RT_REQUIRE((uint64_t)tokens * heads <= RT_MAX_NUMEL / kv->head_dim, RT_ERR_SIZE, "%s: y is too large", who);
    RT_REQUIRE(!weights || (uint64_t)kv->seqs * kv->kv_heads <= RT_MAX_NUMEL / ((uint64_t)kv->table_len * kv->page_len), RT_ERR_SIZE, "%s: weights are too large", who);
    RT_REQUIRE(rt_aligned(q, e) && rt_aligned(y, e) && rt_aligned(starts, 4) && rt_aligned(lse, 4) && rt_aligned(weights, 4) && rt_aligned(weights_out, 4),
               RT_ERR_ALIGN, "%s: misaligned pointer", who);
    rc = rt_enter(dev);
    if (rc) return rc;
    a.q = q; a.k = kv->k; a.v = kv->v; a.y = y; a.lse = lse; a.lens = kv->lens; a.table = kv->table; a.starts = starts;
    a.k_t = a.v_t = kv->head_dim;
    a.k_h = a.v_h = (uint64_t)kv->page_len * kv->head_dim;
    a.k_b = a.v_b = a.k_h * kv->kv_heads;
    a.y_h = kv->head_dim;
    a.y_t = (uint64_t)heads * kv->head_dim;
    a.l_h = 1; a.l_t = heads;
    a.seqs = kv->seqs;
    a.tokens = tokens;
    a.cap = kv->table_len * kv->page_len;
    a.pages = kv->pages;
    a.table_len = kv->table_len;
    a.page_div = make_fastdiv(kv->page_len);
    a.causal = 1;
    a.want_scores = weights_out != nullptr;
    a.own_lse = weights_out && !lse ? (size_t)tokens * heads * sizeof(float) : 0;
    return dispatch(dev, dt, a, true, weights, weights_out);
}

}  // namespace

extern "C" {

int rt_attention(rt_device* dev, int dt, const void* q, const uint32_t q_shape[4], const uint64_t q_strides[4], const void* k, const uint64_t k_strides[4],
                 const void* v, const uint64_t v_strides[4], const uint32_t kv_shape[4], const int32_t* lens, void* y, const uint64_t y_strides[4], float* lse,
                 float scale, int causal, uint32_t window, uint32_t sinks) {
    return attention("rt_attention", dev, dt, q, q_shape, q_strides, k, k_strides, v, v_strides, kv_shape, lens, y, y_strides, lse, scale, causal, window, sinks, nullptr, false);
}

int rt_attention_scored(rt_device* dev, int dt, const void* q, const uint32_t q_shape[4], const uint64_t q_strides[4], const void* k, const uint64_t k_strides[4],
                        const void* v, const uint64_t v_strides[4], const uint32_t kv_shape[4], const int32_t* lens, void* y, const uint64_t y_strides[4], float* lse,
                        float scale, int causal, uint32_t window, uint32_t sinks, const rt_scores* scores) {
    return attention("rt_attention_scored", dev, dt, q, q_shape, q_strides, k, k_strides, v, v_strides, kv_shape, lens, y, y_strides, lse, scale, causal, window, sinks, scores, true);
}

int rt_paged_attention(rt_device* dev, int dt, const void* q, const uint64_t q_strides[2], uint32_t tokens, uint32_t heads, const rt_paged_kv* kv,
                       const int32_t* starts, void* y, float* lse, const float* weights, float* weights_out, float scale, uint32_t window, uint32_t sinks) {
    return paged_attention("rt_paged_attention", dev, dt, q, q_strides, tokens, heads, kv, starts, y, lse, weights, weights_out, scale, window, sinks, nullptr, false);
}

int rt_paged_attention_scored(rt_device* dev, int dt, const void* q, const uint64_t q_strides[2], uint32_t tokens, uint32_t heads, const rt_paged_kv* kv,
                              const int32_t* starts, void* y, float* lse, float scale, uint32_t window, uint32_t sinks, const rt_scores* scores) {
    return paged_attention("rt_paged_attention_scored", dev, dt, q, q_strides, tokens, heads, kv, starts, y, lse, nullptr, nullptr, scale, window, sinks, scores, true);
}

}  // extern "C"
