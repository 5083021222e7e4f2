// The attention weight that cached tokens receive from a call's queries, from the finished statistics of its rows:
//     out[t] = (t is new ? 0 : weights[t]) + sum over the rows that see t of 2^(c q.k_t - lse / ln 2)
// A wave owns 32 keys of a KV head.  They are the rows of the 32 x 32 products S^T = K Q^T and stay in registers while the queries that may see
// them go by, 64 at a time; each lane adds up the weights of its own query column, and the columns are summed once at the end: no atomics, one order.
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

constexpr int AW_ROWS = 64;                      // queries to a stage

template <typename T, int DT, bool EXACT> struct AwShape : AtShape<T, DT> {
    typedef AtShape<T, DT> S;
    static constexpr int PART = (32 * S::CHUNKS * 16 + 1023) / 1024 * 1024;     // a wave's keys in LDS, on their way to registers
    static constexpr int ROWS_AT = (AW_ROWS * S::CHUNKS * 16 + 1023) / 1024 * 1024;            // where a stage keeps its rows' lse
    static constexpr int STAGE = ROWS_AT + AW_ROWS * 4;
    static constexpr int STAGES = 3 * STAGE <= 160 * 1024 ? 3 : 2;              // of queries in LDS
    static constexpr int LDS = STAGES * STAGE > AT_WAVES * PART ? STAGES * STAGE : AT_WAVES * PART;
    static constexpr int LOADS = (AW_ROWS * S::CHUNKS + AT_BLOCK - 1) / AT_BLOCK;               // of a stage's rows, by each wave, at most
    // of the youngest stage, those that every wave has issued: what may still be in flight when the one before it is needed
    static constexpr int LEAST = EXACT && STAGES == 3 ? AW_ROWS * S::CHUNKS / AT_BLOCK : 0;
};

// 4 bytes a lane from memory to LDS, lane i's to at + 4 i
__device__ __forceinline__ void aw_to_lds4(const void* from, lds_byte* at) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "{m0}"((uint32_t)(uintptr_t)at) : "memory");
}
template <int N> __device__ __forceinline__ void aw_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// The block's four waves share the queries, which go through stages of LDS, two on their way while one is worked on (one where rows are too wide for three).  Two
// prompts of up to 1900 tokens, 32 heads of 80 in f16: 52 us.  Bound by its vector instructions, nine a score (a quarter-rate exponential among them), and by the triangle: by counters
// a CU works 77 % of the time, as the blocks of the first keys walk the most queries, and its vector units 70 % of that, its matrix units 18 %.
template <typename T, int DT, bool EXACT>
__global__ void __launch_bounds__(AT_BLOCK, DT > 128 ? 1 : DT > 96 || sizeof(T) == 4 ? 2 : 3) attention_weights_kernel(AttnArgs a, const float* weights, float* out) {
    typedef AwShape<T, DT, EXACT> S;
    constexpr int CE = S::CE;
    extern __shared__ __align__(16) unsigned char smem[];
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 32, half = lane / 32;
    const uint32_t D = EXACT ? DT : a.dim, chunks = D / CE, pitch = D * sizeof(T);
    lds_byte* const lds = (lds_byte*)smem;
    const float c = a.c;
    uint32_t k_at[S::STEPS];                                    // chunk 2 i + half of row col: keys and queries alike
#pragma unroll
    for (int i = 0; i < S::STEPS; i++) {
        uint32_t cc = 2 * i + half;
        cc = (cc < chunks ? cc : 0) + at_turn_k(col, chunks);
        k_at[i] = col * pitch + (cc >= chunks ? cc - chunks : cc) * 16;
    }
    for (uint32_t item = blockIdx.x;; item += gridDim.x) {
        const uint32_t g = item % a.kv_heads;
        uint32_t at = item / a.kv_heads;
        const uint32_t b = __builtin_amdgcn_readfirstlane(aw_locate(a, at));
        if (b >= a.seqs) return;
        const AttnSeq s = at_seq<true>(a, b);
        const int32_t tb = (int32_t)(__builtin_amdgcn_readfirstlane(at) * AW_KEYS), t0 = tb + (int32_t)wave * 32;
        const bool busy = t0 < s.keys;

        // ---- this wave's keys, through LDS to registers
        const int32_t mine = t0 + (int32_t)col;
        uint32_t slot = 0;
        const int32_t page = at_page(a, b, (uint32_t)(mine < s.keys ? mine : s.keys - 1), slot);
        const uint64_t w_at = ((uint64_t)b * a.kv_heads + g) * a.cap;
        const float before = mine < s.keys && mine < s.shift ? weights[w_at + (uint32_t)mine] : 0.0f;
        const uint32_t there = (uint32_t)__ballot(page >= 0);   // both halves say the same
        const unsigned char* kb = (const unsigned char*)a.k + g * a.k_h * sizeof(T);
        const uint32_t slots = 32 * chunks;
        __syncthreads();                                        // the item before this one is done with LDS
        for (uint32_t i = 0; i < (slots + 63) / 64; i++) {
            uint32_t at_slot = i * 64 + lane;
            at_slot = at_slot < slots ? at_slot : slots - 1;
            const uint32_t rr = at_slot / chunks, cc = at_slot - rr * chunks, tk = at_turn_k(rr, chunks);
            const int32_t pg = __shfl(page, (int)rr);
            const uint64_t off = (uint64_t)(pg < 0 ? 0 : pg) * (a.k_b * sizeof(T)) + (uint32_t)__shfl((int)slot, (int)rr) * (uint64_t)pitch;
            at_to_lds(kb + off + (cc >= tk ? cc - tk : cc + chunks - tk) * 16, lds + wave * S::PART + i * 1024);
        }
        v4u k[S::STEPS];
        at_wait_memory();
#pragma unroll
        for (int i = 0; i < S::STEPS; i++) {
            k[i] = at_lds16(lds + (wave * S::PART + k_at[i]));
            if ((2 * i + half) >= chunks) k[i] = v4u{0, 0, 0, 0};
        }
        __syncthreads();

        // ---- the rows that may see one of the block's keys: positions from the first key on and, where no sink is among them, up to the last key's window
        int64_t j0 = (int64_t)tb - s.shift, j1 = s.count;
        if (a.window != AT_FAR && tb >= a.sinks) {
            const int64_t x = (int64_t)tb + AW_KEYS - 1 + a.window - s.shift;
            j1 = x < j1 ? x : j1;
        }
        j0 = j0 < 0 ? 0 : j0;
        const uint32_t r0 = j0 < j1 ? (uint32_t)j0 * a.group : 0, r1 = j0 < j1 ? (uint32_t)j1 * a.group : 0;
        const uint32_t stages = (r1 - r0 + AW_ROWS - 1) / AW_ROWS, loads = (AW_ROWS * chunks + 63) / 64;
        auto fetch = [&](uint32_t n, uint32_t stage) __attribute__((always_inline)) {
            lds_byte* const to = lds + stage * S::STAGE;
#pragma unroll
            for (int i = 0; i < S::LOADS; i++) {
                if (i * AT_WAVES + wave >= loads) break;
                uint32_t at_slot = (i * AT_WAVES + wave) * 64 + lane;
                at_slot = at_slot < AW_ROWS * chunks ? at_slot : AW_ROWS * chunks - 1;
                const uint32_t rr = at_slot / chunks, cc = at_slot - rr * chunks, tk = at_turn_k(rr, chunks);
                uint32_t row = r0 + n * AW_ROWS + rr;
                row = row < r1 ? row : r1 - 1;
                const uint32_t j = fd_div(row, a.group_div), h = g * a.group + (row - j * a.group);
                const unsigned char* from = (const unsigned char*)a.q + (h * a.q_h + (uint64_t)(s.first + j) * a.q_t) * sizeof(T);
                at_to_lds(from + (cc >= tk ? cc - tk : cc + chunks - tk) * 16, to + (i * AT_WAVES + wave) * 1024);
            }
            if (wave == AT_WAVES - 1) {
                uint32_t row = r0 + n * AW_ROWS + lane;
                row = row < r1 ? row : r1 - 1;
                const uint32_t j = fd_div(row, a.group_div), h = g * a.group + (row - j * a.group);
                aw_to_lds4(a.lse + h * a.l_h + (uint64_t)(s.first + j) * a.l_t, to + S::ROWS_AT);
            }
        };
        float sum[16];
#pragma unroll
        for (int e = 0; e < 16; e++) sum[e] = 0.0f;
        if (stages > 0) fetch(0, 0);
        if (S::STAGES == 3 && stages > 1) fetch(1, 1);
        uint32_t stage = 0;
        for (uint32_t n = 0; n < stages; n++) {
            if (n + 1 < stages) aw_wait<S::LEAST>();
            else aw_wait<0>();
            __syncthreads();                                    // this stage is there, and everyone is done with the one before
            if (n + S::STAGES - 1 < stages) fetch(n + S::STAGES - 1, stage == 0 ? S::STAGES - 1 : stage - 1);
            const lds_byte* const cur = lds + stage * S::STAGE;
            stage = stage == S::STAGES - 1 ? 0 : stage + 1;
            if (!busy) continue;
            constexpr int N = 2 * S::STEPS, AHEAD = N < 4 ? N : 4;
            v16f x[2] = {v16f{0}, v16f{0}}, others[2][S::SUMS];
#pragma unroll
            for (int z = 1; z < S::SUMS; z++) others[0][z] = others[1][z] = v16f{0};
            v4u q[N];
            auto read_q = [&](int p) __attribute__((always_inline)) {
                if (!EXACT && (uint32_t)(p / 2 * 2 * CE) >= D) return;
                q[p] = at_lds16(cur + (k_at[p / 2] + p % 2 * 32 * pitch));
            };
#pragma unroll
            for (int p = 0; p < AHEAD; p++) read_q(p);
            float lse[2] = {at_lds4(cur + S::ROWS_AT + col * 4) * -1.4426950408889634f, at_lds4(cur + S::ROWS_AT + (col + 32) * 4) * -1.4426950408889634f};
#pragma unroll
            for (int y = 0; y < 2; y++) lse[y] = lse[y] == INFINITY ? -INFINITY : lse[y];       // a row whose scores are all -inf weighs nothing
            at_in_order();
#pragma unroll
            for (int p = 0; p < N; p++) {
                // where the row ends in a half chunk, both operands' other half holds what is not theirs: k's is 0 and q's has to be
                if ((EXACT ? DT % (2 * CE) != 0 : true) && (p / 2 * 2 + 2) * CE > (int)D && half) q[p] = v4u{0, 0, 0, 0};
                if (EXACT || (uint32_t)(p / 2 * 2 * CE) < D) at_score<T>(k[p / 2], q[p], x[p % 2], others[p % 2]);
                if (p + AHEAD < N) read_q(p + AHEAD);
                at_in_order();
            }
            at_settle(S::SUMS == 1 ? x[1] : others[1][S::SUMS - 1]);
            at_join_sums(x[0], others[0]);
            at_join_sums(x[1], others[1]);
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const uint32_t row = r0 + n * AW_ROWS + 32 * y + col;
                const bool real = row < r1;
                const uint32_t j = fd_div(real ? row : r1 - 1, a.group_div);
                const int32_t limit = at_limit(a, s, j), p = at_position(s, j);
                // whether every row sees every key of the 32: nearly all tiles of a prompt
                const bool clear = real && t0 + 31 <= limit && (p - t0 < a.window || t0 + 31 < a.sinks) && there == ~0u;
                if (__ballot(clear) == ~0ull) {
#pragma unroll
                    for (int e = 0; e < 16; e++) sum[e] += at_exp2(__builtin_fmaf(x[y][e], c, lse[y]));
                } else {
                    const int32_t lim = real ? limit - t0 - 4 * (int32_t)half : -1, near = p - t0 - 4 * (int32_t)half, sink = a.sinks - t0 - 4 * (int32_t)half;
                    const uint32_t have = there >> (4 * half);
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int32_t t = e % 4 + 8 * (e / 4);
                        const bool seen = t <= lim && (near - t < a.window || t < sink) && (have >> t) & 1;
                        sum[e] += seen ? at_exp2(__builtin_fmaf(x[y][e], c, lse[y])) : 0.0f;
                    }
                }
            }
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
    typedef AwShape<T, DT, EXACT> S;
    const uint64_t items = (uint64_t)a.seqs * ((a.cap + AW_KEYS - 1) / AW_KEYS) * a.kv_heads;
    const unsigned blocks = items < AW_MOST_BLOCKS ? (unsigned)items : (AW_MOST_BLOCKS + a.kv_heads - 1) / a.kv_heads * a.kv_heads;
    static_assert(S::LDS <= 160 * 1024, "LDS");
    constexpr int LDS = S::LDS;
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
    if (a.dim == 80) return aw_launch<T, 80, true>(dev, a, weights, out);
    if (a.dim == 96) return aw_launch<T, 96, true>(dev, a, weights, out);
    if (a.dim == 128) return aw_launch<T, 128, true>(dev, a, weights, out);
    if (a.dim == 192) return aw_launch<T, 192, true>(dev, a, weights, out);
    if (a.dim == 256) return aw_launch<T, 256, true>(dev, a, weights, out);
    if (a.dim < 64) return aw_launch<T, 64, false>(dev, a, weights, out);
    if (a.dim < 128) return aw_launch<T, 128, false>(dev, a, weights, out);
    return aw_launch<T, 256, false>(dev, a, weights, out);
}

#endif
