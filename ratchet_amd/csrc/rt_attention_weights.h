// The attention weight that cached tokens receive from a call's queries, from the finished statistics of its rows:
//     out[t] = (t is new ? 0 : weights[t]) + sum over the rows that see t of 2^(c q.k_t - lse / ln 2)
// A wave owns 32 keys of a KV head. They are the rows of the 32 x 32 products S^T = K Q^T and stay in registers while the queries that may see
// them go by, 32 at a time; each lane adds up the weights of its own query column, and the columns are summed once at the end: no atomics, one order.
#ifndef RT_ATTENTION_WEIGHTS_H
#define RT_ATTENTION_WEIGHTS_H

#include "rt_attention_tile.h"

constexpr uint32_t AW_KEYS = 32 * AT_WAVES;      // of a block
constexpr uint32_t AW_MOST_BLOCKS = 8192;        // each takes every AW_MOST_BLOCKS-th item of a larger call

// Items are numbered sequence by sequence, AW_KEYS keys each; see at_locate
__device__ __forceinline__ uint32_t aw_locate(const AttnArgs& a, uint32_t& at) {
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.seqs; b0 += 64) {
        const uint32_t b = b0 + __lane_id(), n = b < a.seqs ? ((uint32_t)at_seq<true>(a, b).keys + AW_KEYS - 1) / AW_KEYS : 0;
        uint32_t sum = n;
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

template <typename T, int DT, bool EXACT>
__global__ void __launch_bounds__(AT_BLOCK, DT > 128 ? 1 : 2) attention_weights_kernel(AttnArgs a, const float* weights, float* out) {
    typedef AtShape<T, DT> S;
    constexpr int CE = S::CE;
    extern __shared__ __align__(16) unsigned char smem[];
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 32, half = lane / 32;
    const uint32_t D = EXACT ? DT : a.dim, chunks = D / CE, pitch = D * sizeof(T);
    constexpr uint32_t PART = (32 * S::CHUNKS * 16 + 1023) / 1024 * 1024;       // a wave's keys in LDS
    lds_byte* const lds = (lds_byte*)smem + wave * PART;
    const float c = a.c;
    for (uint32_t item = blockIdx.x;; item += gridDim.x) {
        const uint32_t g = item % a.kv_heads;
        uint32_t at = item / a.kv_heads;
        const uint32_t b = __builtin_amdgcn_readfirstlane(aw_locate(a, at));
        if (b >= a.seqs) return;
        const AttnSeq s = at_seq<true>(a, b);
        const int32_t t0 = (int32_t)(__builtin_amdgcn_readfirstlane(at) * AW_KEYS + wave * 32);
        if (t0 >= s.keys) continue;

        uint32_t slot;
        const int32_t mine = t0 + (int32_t)col, page = at_page(a, b, (uint32_t)(mine < s.keys ? mine : s.keys - 1), slot);
        const uint64_t w_at = ((uint64_t)b * a.kv_heads + g) * a.cap;
        const float before = mine < s.keys && mine < s.shift ? weights[w_at + (uint32_t)mine] : 0.0f;
        const uint32_t there = (uint32_t)__ballot(page >= 0);   // both halves say the same
        const unsigned char* kb = (const unsigned char*)a.k + g * a.k_h * sizeof(T);
        const uint32_t slots = 32 * chunks;
        for (uint32_t i = 0; i < (slots + 63) / 64; i++) {
            uint32_t at_slot = i * 64 + lane;
            at_slot = at_slot < slots ? at_slot : slots - 1;
            const uint32_t rr = at_slot / chunks, cc = at_slot - rr * chunks, tk = at_turn_k(rr, chunks);
            const int32_t pg = __shfl(page, (int)rr);
            const uint64_t off = (uint64_t)(pg < 0 ? 0 : pg) * (a.k_b * sizeof(T)) + (uint32_t)__shfl((int)slot, (int)rr) * (uint64_t)pitch;
            at_to_lds(kb + off + (cc >= tk ? cc - tk : cc + chunks - tk) * 16, lds + i * 1024);
        }

        // the rows that may see one of these keys: positions from t0 on and, where no sink is among them, up to the last key's window
        int64_t j0 = (int64_t)t0 - s.shift, j1 = s.count;
        if (a.window != AT_FAR && t0 >= a.sinks) {
            const int64_t x = (int64_t)t0 + 31 + a.window - s.shift;
            j1 = x < j1 ? x : j1;
        }
        j0 = j0 < 0 ? 0 : j0;
        const uint32_t r0 = j0 < j1 ? (uint32_t)j0 * a.group : 0, r1 = j0 < j1 ? (uint32_t)j1 * a.group : 0;

        auto load = [&](uint32_t r, v4u (&q)[S::STEPS], float& lse, uint32_t& j) __attribute__((always_inline)) {
            const uint32_t row = r + col < r1 ? r + col : r1 - 1;
            j = fd_div(row, a.group_div);
            const uint32_t h = g * a.group + (row - j * a.group);
            const T* from = (const T*)a.q + h * a.q_h + (uint64_t)(s.first + j) * a.q_t;
#pragma unroll
            for (int i = 0; i < S::STEPS; i++) {
                q[i] = v4u{0, 0, 0, 0};
                if ((2 * i + half) * CE < D) q[i] = *(const v4u*)(from + (2 * i + half) * CE);
            }
            lse = a.lse[h * a.l_h + (uint64_t)(s.first + j) * a.l_t] * -1.4426950408889634f;
        };
        float sum[16];
#pragma unroll
        for (int e = 0; e < 16; e++) sum[e] = 0.0f;
        v4u k[S::STEPS], q[S::STEPS], q2[S::STEPS];
        float lse = 0.0f, lse2 = 0.0f;
        uint32_t j = 0, j2 = 0;
        if (r0 < r1) load(r0, q, lse, j);
        at_wait_memory();                                       // the keys are in LDS
#pragma unroll
        for (int i = 0; i < S::STEPS; i++) {
            uint32_t cc = 2 * i + half;
            const bool in = cc < chunks;
            cc = (in ? cc : 0) + at_turn_k(col, chunks);
            k[i] = at_lds16(lds + (col * pitch + (cc >= chunks ? cc - chunks : cc) * 16));
            if (!in) k[i] = v4u{0, 0, 0, 0};
        }
        for (uint32_t r = r0; r < r1; r += 32) {
            if (r + 32 < r1) load(r + 32, q2, lse2, j2);
            v16f x = {0};
#pragma unroll
            for (int i = 0; i < S::STEPS; i++) {
                if (EXACT || (uint32_t)(2 * i * CE) < D) x = AtMma<T>::qk(k[i], q[i], x);
            }
            const int32_t limit = at_limit(a, s, j), p = at_position(s, j);
            const bool real = r + col < r1;
            // whether every row sees every key of the 32: nearly all tiles of a prompt
            const bool clear = real && t0 + 31 <= limit && (p - t0 < a.window || t0 + 31 < a.sinks) && there == ~0u;
            if (__ballot(clear) == ~0ull) {
#pragma unroll
                for (int e = 0; e < 16; e++) sum[e] += at_exp2(__builtin_fmaf(x[e], c, lse));
            } else {
                const int32_t lim = real ? limit - t0 - 4 * (int32_t)half : -1, near = p - t0 - 4 * (int32_t)half, sink = a.sinks - t0 - 4 * (int32_t)half;
                const uint32_t have = there >> (4 * half);
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int32_t t = e % 4 + 8 * (e / 4);
                    const bool seen = t <= lim && (near - t < a.window || t < sink) && (have >> t) & 1;
                    sum[e] += seen ? at_exp2(__builtin_fmaf(x[e], c, lse)) : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < S::STEPS; i++) q[i] = q2[i];
            lse = lse2;
            j = j2;
        }
        // over the 32 columns; the lane with column n keeps key n: element e of half h is key e % 4 + 8 (e / 4) + 4 h
        float total = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            float x = sum[e];
#pragma unroll
            for (int i = 16; i; i >>= 1) x += __shfl_xor(x, i);
            const uint32_t key = e % 4 + 8 * (e / 4);
            const float other = at_other(x);
            if (col == key) total = half ? other : x;
            if (col == key + 4) total = half ? x : other;
        }
        if (half == 0 && mine < s.keys) out[w_at + (uint32_t)mine] = before + total;
    }
}

// The same from scores that the attention left (few rows): a thread to a key, its rows one after the other.  Reads a score a row and key, coalesced.
constexpr uint32_t AW_SCORE_BLOCK = 128;
static __global__ void __launch_bounds__(AW_SCORE_BLOCK) attention_weights_of_scores_kernel(AttnArgs a, const float* weights, float* out) {
    const uint32_t g = blockIdx.y, b = blockIdx.z;
    const AttnSeq s = at_seq<true>(a, b);
    const int32_t t = (int32_t)(blockIdx.x * AW_SCORE_BLOCK + threadIdx.x);
    if (t >= s.keys) return;
    const uint64_t at = ((uint64_t)b * a.kv_heads + g) * a.cap + (uint32_t)t;
    float sum = t < s.shift ? weights[at] : 0.0f;
    for (uint32_t j = 0; j < s.count; j++) {
        if (!at_visible(a, t, at_limit(a, s, j), at_position(s, j))) continue;                 // its score may never have been written
        const uint64_t row = (uint64_t)(s.first + j) * a.heads + g * a.group;
        for (uint32_t h = 0; h < a.group; h++) {
            const float x = a.scores[(row + h) * a.score_pitch + (uint32_t)t];
            sum += x == -INFINITY ? 0.0f : at_exp2(__builtin_fmaf(a.lse[row + h], -1.4426950408889634f, x));
        }
    }
    out[at] = sum;
}

template <typename T, int DT, bool EXACT> int aw_launch(rt_device* dev, const AttnArgs& a, const float* weights, float* out) {
    typedef AtShape<T, DT> S;
    const uint64_t items = (uint64_t)a.seqs * ((a.cap + AW_KEYS - 1) / AW_KEYS) * a.kv_heads;
    const unsigned blocks = items < AW_MOST_BLOCKS ? (unsigned)items : (AW_MOST_BLOCKS + a.kv_heads - 1) / a.kv_heads * a.kv_heads;
    constexpr int LDS = AT_WAVES * ((32 * S::CHUNKS * 16 + 1023) / 1024 * 1024);
    const auto kernel = attention_weights_kernel<T, DT, EXACT>;
    static bool raised[16] = {};
    if (LDS > 64 * 1024 && !(dev->ordinal < 16 && raised[dev->ordinal])) {
        RT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
        if (dev->ordinal < 16) raised[dev->ordinal] = true;
    }
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(AT_BLOCK), LDS, dev->stream, a, weights, out);
    RT_CHECK_LAUNCH("attention_weights_kernel");
    return RT_OK;
}

template <typename T> int aw_dispatch(rt_device* dev, const AttnArgs& a, const float* weights, float* out) {
    if (a.scores) {
        const dim3 grid((a.cap + AW_SCORE_BLOCK - 1) / AW_SCORE_BLOCK, a.kv_heads, a.seqs);
        hipLaunchKernelGGL(attention_weights_of_scores_kernel, grid, dim3(AW_SCORE_BLOCK), 0, dev->stream, a, weights, out);
        RT_CHECK_LAUNCH("attention_weights_of_scores_kernel");
        return RT_OK;
    }
    if (a.dim == 64) return aw_launch<T, 64, true>(dev, a, weights, out);
    if (sizeof(T) == 2 && a.dim == 80) return aw_launch<T, 80, true>(dev, a, weights, out);
    if (sizeof(T) == 2 && a.dim == 96) return aw_launch<T, 96, true>(dev, a, weights, out);
    if (sizeof(T) == 2 && a.dim == 128) return aw_launch<T, 128, true>(dev, a, weights, out);
    if (a.dim <= 128) return aw_launch<T, 128, false>(dev, a, weights, out);
    return aw_launch<T, 256, false>(dev, a, weights, out);
}

#endif
