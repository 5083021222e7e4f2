// What the attention kernels share: the problem as one set of arguments for contiguous and paged caches, and where its rows are.
//
// For one query row at position p (its head reads KV head head / G):
//     s_t = c * q.k_t  over the visible keys t, c = scale * log2(e)        m = max s_t,  l = sum 2^(s_t - m)
//     o = sum 2^(s_t - m) v_t / l                                          lse = ln 2 * (m + log2 l)
// where the call changes its scores (SCORED), with z = scale * q.k_t: s_t = log2(e) * (cap tanh(z / cap) - slope |p - t|)
// Keys are walked in tiles; m, l and o are kept running in f32 and o, l are scaled by 2^(m_old - m_new) where a tile raises m.
#ifndef RT_ATTENTION_H
#define RT_ATTENTION_H

#include "rt_arith.h"
#include "rt_internal.h"

constexpr int AT_MAX_DIM = 512;                  // columns of a head
constexpr int32_t AT_FAR = 0x7fffffff;           // window of a call without one
constexpr int32_t AT_MOST_TOKENS = 1 << 30;      // rows, keys and positions lie below it, and their differences in 32 bits

struct AttnArgs {
    const void* q;
    const void* k;
    const void* v;
    void* y;
    float* lse;                    // NULL: not wanted
    const int32_t* table;          // paged only
    const int32_t* lens;           // contiguous: NULL = all keys
    const int32_t* starts;         // paged only
    uint64_t q_b, q_h, q_t;        // elements from batch entry to batch entry, head to head, token to token (q_b = 0 where paged)
    uint64_t k_b, k_h, k_t;        // contiguous: the same of k; paged: page to page, head to head, token to token
    uint64_t v_b, v_h, v_t;
    uint64_t y_b, y_h, y_t;
    uint64_t l_b, l_h, l_t;        // of lse
    uint32_t seqs, heads, kv_heads, group, dim;
    uint32_t tokens;               // rows of q per batch entry (contiguous) or in all (paged)
    uint32_t cap;                  // keys that there is room for: Sk, or table_len * page_len
    uint32_t pages, table_len;
    FastDiv page_div;              // by page_len
    FastDiv group_div;             // by group
    float c;                       // scale * log2(e)
    int32_t causal, window, sinks;
    size_t own_lse;                // bytes of lse that the call itself needs and keeps at the front of the workspace
    float* scores;                 // NULL, or [tokens, heads, score_pitch]: c q.k of each row and key, -inf where hidden, left for the received weights
    uint32_t score_pitch;
    bool want_scores;              // the caller has use for them
    // calls that change or mask their scores (rt_scores)
    bool scored;
    float most, most_in;           // cap * log2(e), 0: none; scale / cap
    float near[4], near_limit;     // 16-bit products up to near_limit take the polynomial x (near[0] + near[1] x^2 + ..) for the capped score
    const float* slopes;
    const int32_t* documents;
    uint32_t n_documents;
    const int32_t* prefix;
};

// Scores of up to this size are kept between the attention of few rows and the sum of its weights; 64 bytes of q and k a score is what it would take to have them again
constexpr size_t AT_MOST_SCORES = 256u << 20;

// The device's workspace with room for lse, if it is the call's own (a.lse is then set), and `bytes` behind it
static inline int at_workspace(rt_device* dev, AttnArgs& a, size_t bytes, void** rest) {
    const size_t front = (a.own_lse + 255) / 256 * 256;
    if (front + bytes == 0) return RT_OK;
    void* p;
    int rc = rt_scratch(dev, front + bytes, &p);
    if (rc) return rc;
    if (front) a.lse = (float*)p;
    *rest = (unsigned char*)p + front;
    return RT_OK;
}

// The matrix-unit kernels (rt_attention_tile.h), a source to each element type.  RT_OK with *done = false where the operands are not laid out for them, or are too many rows for a launch
int rt_attention_tile_f32(rt_device* dev, AttnArgs& a, bool paged, bool* done);
int rt_attention_tile_f16(rt_device* dev, AttnArgs& a, bool paged, bool* done);
int rt_attention_tile_bf16(rt_device* dev, AttnArgs& a, bool paged, bool* done);
// The same for calls that change or mask their scores
int rt_attention_scored_f32(rt_device* dev, AttnArgs& a, bool paged, bool* done);
int rt_attention_scored_f16(rt_device* dev, AttnArgs& a, bool paged, bool* done);
int rt_attention_scored_bf16(rt_device* dev, AttnArgs& a, bool paged, bool* done);
// Received weights of a paged call that the kernel above took (rt_attention_weights.h); a.lse holds its rows' statistics
int rt_attention_weights_f32(rt_device* dev, const AttnArgs& a, const float* weights, float* out);
int rt_attention_weights_f16(rt_device* dev, const AttnArgs& a, const float* weights, float* out);
int rt_attention_weights_bf16(rt_device* dev, const AttnArgs& a, const float* weights, float* out);

#ifdef __HIPCC__

// One sequence's part of a call
struct AttnSeq {
    uint32_t first, count;         // its rows of q
    int32_t keys;                  // keys there are
    int32_t shift;                 // position of row j: j + shift
};

template <bool PAGED> __device__ __forceinline__ AttnSeq at_seq(const AttnArgs& a, uint32_t b) {
    AttnSeq s;
    if (PAGED) {
        const int32_t top = (int32_t)a.tokens;
        int32_t lo = a.starts[b], hi = a.starts[b + 1];
        lo = lo < 0 ? 0 : lo > top ? top : lo;
        hi = hi < lo ? lo : hi > top ? top : hi;
        int32_t len = a.lens[b];
        len = len < 0 ? 0 : len < AT_MOST_TOKENS ? len : AT_MOST_TOKENS;
        s.first = (uint32_t)lo;
        s.count = (uint32_t)(hi - lo);
        s.keys = len < (int32_t)a.cap ? len : (int32_t)a.cap;
        s.shift = len - (int32_t)s.count;
    } else {
        int32_t len = (int32_t)a.cap;
        if (a.lens) {
            len = a.lens[b];
            len = len < 0 ? 0 : len > (int32_t)a.cap ? (int32_t)a.cap : len;
        }
        s.first = 0;
        s.count = a.tokens;
        s.keys = len;
        s.shift = len - (int32_t)a.tokens;
    }
    return s;
}

// The last key that row j may see: its own position, or the last key where the call is not causal
__device__ __forceinline__ int32_t at_limit(const AttnArgs& a, const AttnSeq& s, uint32_t j) {
    const int32_t p = (int32_t)j + s.shift;
    return a.causal && p < s.keys - 1 ? p : s.keys - 1;
}
// Position that the window counts from
__device__ __forceinline__ int32_t at_position(const AttnSeq& s, uint32_t j) { return (int32_t)j + s.shift; }
__device__ __forceinline__ bool at_visible(const AttnArgs& a, int32_t t, int32_t limit, int32_t p) {
    return t <= limit && (p - t < a.window || t < a.sinks);
}

// What a row sees: keys lo .. limit, but where p - t >= window those before `front` alone.  Over rows in order none of the four decreases.
struct AttnRow {
    int32_t p, limit, lo, front;
};
__device__ __forceinline__ int32_t at_between(int32_t x, int32_t low, int32_t high) { return x < low ? low : x > high ? high : x; }
// The row at position p of a text that holds keys lo .. hi - 1
__device__ __forceinline__ AttnRow at_in_text(const AttnArgs& a, int32_t p, int32_t lo, int32_t hi, int32_t prefix) {
    const int32_t seen = at_between(prefix, 0, hi - lo), wide = a.sinks > seen ? a.sinks : seen;
    AttnRow r = {p, hi - 1, lo, wide < hi - lo ? lo + wide : hi};
    if (a.causal) {
        const int32_t own = p < hi - 1 ? p : hi - 1, shared = lo + seen - 1;
        r.limit = own > shared ? own : shared;
        if (r.limit < lo) r.limit = lo - 1;
    }
    return r;
}
__device__ __forceinline__ uint32_t at_find(const int32_t* starts, uint32_t seqs, uint32_t token);

// The texts of one entry of a call with documents, by all lanes of a wave: up to 63 are looked at once, a lane to a text, and what is asked of them later is a vote of the lanes
struct AttnTexts {
    int32_t start, prefix;                         // of text `lane`, where all fit
};
__device__ __forceinline__ AttnTexts at_texts(const AttnArgs& a, uint32_t b) {
    AttnTexts t = {AT_FAR, 0};
    if (a.documents && a.n_documents < 64) {
        const uint32_t lane = __lane_id();
        if (lane <= a.n_documents) t.start = a.documents[(uint64_t)b * (a.n_documents + 1) + lane];
        if (a.prefix && lane < a.n_documents) t.prefix = a.prefix[(uint64_t)b * a.n_documents + lane];
    }
    return t;
}
// The document of position p, the same in all lanes: the last that begins at or before it; n_documents or above where it is in none
__device__ __forceinline__ uint32_t at_document(const AttnArgs& a, const AttnTexts& t, uint32_t b, int32_t p) {
    if (a.n_documents < 64) return (uint32_t)__popcll(__ballot(t.start <= p)) - 1;         // (none in front of the first: the largest number)
    return __builtin_amdgcn_readfirstlane(at_find(a.documents + (uint64_t)b * (a.n_documents + 1), a.n_documents + 1, (uint32_t)p));
}
// Where document d begins (n_documents: where the last one ends).  d may differ from lane to lane, all of which take part
__device__ __forceinline__ int32_t at_start(const AttnArgs& a, const AttnTexts& t, uint32_t b, uint32_t d) {
    return a.n_documents < 64 ? __shfl(t.start, (int)d) : a.documents[(uint64_t)b * (a.n_documents + 1) + d];
}
__device__ __forceinline__ AttnRow at_in_document(const AttnArgs& a, const AttnTexts& t, uint32_t b, const AttnSeq& s, int32_t p, uint32_t d) {
    const bool none = d >= a.n_documents;          // in front of the first, or behind the last: a text without keys
    const uint32_t from = !none ? d : d == a.n_documents ? d : 0, to = !none ? d + 1 : from;
    const int32_t lo = at_between(at_start(a, t, b, from), 0, s.keys), hi = at_between(at_start(a, t, b, to), lo, s.keys);
    int32_t prefix = 0;
    if (a.prefix) {
        prefix = a.n_documents < 64 ? __shfl(t.prefix, (int)(none ? 0 : d)) : a.prefix[(uint64_t)b * a.n_documents + (none ? 0 : d)];
        if (none) prefix = 0;
    }
    return at_in_text(a, p, lo, hi, prefix);
}
// The document of position p, a lane's own, among those from da to dz, the same in all lanes, that at_document names for the first and the last row: the last that begins at or
// before it, in as many steps as their number has bits, so that texts without tokens (an array that repeats its end) are not walked one by one.  All lanes take part.
__device__ __forceinline__ uint32_t at_document_of(const AttnArgs& a, const AttnTexts& t, uint32_t b, int32_t p, uint32_t da, uint32_t dz) {
    const uint32_t first = da > a.n_documents ? 0 : da + 1;    // da may be `none in front`, beyond all numbers
    if (dz > a.n_documents || dz < first) return da;
    const uint32_t count = dz - first + 1;
    uint32_t n = 0;                                // of them begin at or before p
    for (uint32_t step = 1u << (31 - __builtin_clz(count)); step; step >>= 1) {
        const uint32_t at = n + step;
        const int32_t start = at_start(a, t, b, first + (at <= count ? at : 1) - 1);
        if (at <= count && start <= p) n = at;
    }
    return n ? first + n - 1 : da;
}
// Row j of sequence b; all lanes take part, with the same row
template <bool SCORED> __device__ __forceinline__ AttnRow at_row(const AttnArgs& a, const AttnTexts& t, uint32_t b, const AttnSeq& s, uint32_t j) {
    const int32_t p = at_position(s, j);
    if (!SCORED) return AttnRow{p, at_limit(a, s, j), 0, a.sinks};
    if (a.documents) return at_in_document(a, t, b, s, p, at_document(a, t, b, p));
    return at_in_text(a, p, 0, s.keys, a.prefix ? a.prefix[b] : 0);
}
template <bool SCORED> __device__ __forceinline__ bool at_sees(const AttnArgs& a, const AttnRow& r, int32_t t) {
    return t <= r.limit && (!SCORED || t >= r.lo) && (r.p - t < a.window || t < r.front);
}

// cap * tanh(z / cap) in units of log2(e), y = z / cap: tanh y = 1 - 2 / (e^2y + 1), off by less than 2^-21 of the cap.  For a cap up to AT_COARSE that is less than a 16-bit
// weight's rounding; for a larger one it is too much of small ones, and FINE ones below 1/8 take the series to y^5, 2^-22 of it off at most.
// In f32 the exponential of |y|, with a Newton step for the reciprocal, is off by 2^-22 at most, and those below 1/2 take the polynomial through tanh's values at Chebyshev's
// points of y^2 <= 1/4, 2^-26 of it off at most.
constexpr float AT_COARSE = 1024.0f;               // in units of log2(e)
template <typename T, bool FINE> __device__ __forceinline__ float at_capped(float cap, float y) {
    const float z = y * y;
    if (sizeof(T) == 2) {
        const float t = __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y * 2.885390081777927f) + 1.0f), cap);
        return FINE && __builtin_fabsf(y) < 0.125f ? cap * y * __builtin_fmaf(z, __builtin_fmaf(z, 2.0f / 15, -1.0f / 3), 1.0f) : t;
    }
    const float d = __builtin_amdgcn_exp2f(__builtin_fabsf(y) * 2.885390081777927f) + 1.0f, near_r = __builtin_amdgcn_rcpf(d);
    const float r = d < 0x1p100f ? near_r * __builtin_fmaf(-d, near_r, 2.0f) : 0.0f;
    const float t = __builtin_copysignf(__builtin_fmaf(-2.0f * cap, r, cap), y);
    const float near = cap * (y * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 0.017131344f, -0.052984239f), 0.133247505f), -0.33333068f), 0.99999999f));
    return __builtin_fabsf(y) < 0.5f ? near : t;
}
// The score, in units of log2(e), of a product q.k; slope: in the same units
template <typename T, bool SCORED> __device__ __forceinline__ float at_changed(const AttnArgs& a, float dot, float slope, int32_t distance) {
    if (!SCORED) return dot * a.c;
    float x = a.most != 0.0f ? at_capped<T, true>(a.most, dot * a.most_in) : dot * a.c;
    if (a.slopes) x = __builtin_fmaf(-slope, __builtin_fabsf((float)distance), x);
    return x;
}

// A head's slope in units of log2(e).  One that passes f32's largest there stays finite, so that at distance 0 it takes nothing: a bias that leaves a row its own key
__device__ __forceinline__ float at_slope(const AttnArgs& a, uint32_t h) {
    const float slope = a.slopes[h], x = slope * 1.4426950408889634f;
    return __builtin_isfinite(slope) ? fminf(fmaxf(x, -3.4028235e38f), 3.4028235e38f) : x;
}

// The page of token t, or -1 if there is none
__device__ __forceinline__ int32_t at_page(const AttnArgs& a, uint32_t b, uint32_t t, uint32_t& slot) {
    uint32_t at;
    fd_divmod(t, a.page_div, at, slot);
    const int32_t page = a.table[(uint64_t)b * a.table_len + at];
    return (uint32_t)page < a.pages ? page : -1;
}

// The last sequence whose rows start at or before `token`, found by the 64 lanes of a wave: 64 entries of `starts` at a time, then the
// stretch between two of them.  seqs if there is none.  Every lane takes part.
__device__ __forceinline__ uint32_t at_find(const int32_t* starts, uint32_t seqs, uint32_t token) {
    const uint32_t lane = __lane_id();
    uint32_t lo = 0, n = seqs;
    while (true) {
        const uint32_t step = (n + 63) / 64, at = lo + lane * step;
        const bool before = lane * step < n && starts[at] <= (int32_t)token;
        const uint32_t count = (uint32_t)__popcll(__ballot(before));
        if (count == 0) return seqs;               // only in the first round
        lo += (count - 1) * step;
        if (step == 1) return lo;
        n = n - (count - 1) * step < step ? n - (count - 1) * step : step;
    }
}

__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float at_lse(float m, float l) { return (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f; }

#endif
#endif
