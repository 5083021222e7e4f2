// What the attention kernels share: the problem as one set of arguments for contiguous and paged caches, and where its rows are.
//
// For one query row at position p (its head reads KV head head / G):
//     s_t = c * q.k_t  over the visible keys t, c = scale * log2(e)        m = max s_t,  l = sum 2^(s_t - m)
//     o = sum 2^(s_t - m) v_t / l                                          lse = ln 2 * (m + log2 l)
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
