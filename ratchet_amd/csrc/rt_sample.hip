// Sampling of tokens from rows of logits: temperature, top-k, top-p, min-p, from given random numbers.
//
//     w_i = exp((x_i - max x) / temperature)                  in 64-bit floats, rounded to multiples of 2^-scale (fixed point in 64 bits)
//     K: the top_k largest logits; P: of K, in descending order, those with (sum of the w before) < top_p * (sum of K's w); M: w_i >= min_p
//     token: the first index whose cumulative kept weight, by index, exceeds uniform * (sum of the kept w)
// All three filters keep a front of the same order, larger logits first and of equal ones the lower index, so what they keep is a cut in it: a logit and
// the index up to which its equals stay.  Sums of fixed-point numbers are the same in any order and on any split, so atomics and waves need no order.
//
// A block to a row, a sixteenth of the row to a wave; the row is read again for every walk over it, from the L2.  NaN fails every comparison here, and so is never kept.
//   temperature alone: the waves' sums of weights, then the one wave's share that holds the border is dealt out to all threads again
//   top-k: the kth largest of the threads' maxima, to a step of a histogram, bounds the kth largest logit; what reaches it is listed, and a list of up to 1024 is sorted,
//          cut and drawn from by itself
//   top-p: a histogram of the weights over 2048 equal steps of the logit names the step the cut lies in; its members are listed and sorted for
//          the cut.  A step of too many members is cut into 2048 again, down to equals
// What bounds it: vector instructions, some 25 for a weight in 64 bits, twice for each logit where many are kept, and the chain of barriers between the phases.  256 rows of
// 32064 f32 with top-p 38 us: maximum 3.5, histogram 12.4 (of which its atomics 40 clocks a wave), the step's members 4.5, their order 1.4, weights of what is kept 4.8, search
// 4.3.  64 rows of 50295 f16 with top-k around 50 14.5 us.  One row of 51865 f32, all of it kept, 23 us: one CU reads it at 9 GB/s a wave and fetches the code for the first time.
#include <math.h>

#include "rt_arith.h"
#include "rt_internal.h"

namespace {

constexpr int BLOCK = 1024, WAVES = BLOCK / 64;
constexpr uint32_t BINS = 2048, LIST = 1024;
constexpr uint32_t MOST_VOCAB = 1u << 24;

// 2^f = 1 + f q(f) for |f| <= 1/2: q interpolates at Chebyshev's points, the result is 4e-14 off at most
constexpr int TERMS = 9;
constexpr double EXP2[TERMS] = {0x1.62e42fefa39efp-1, 0x1.ebfbdff823cedp-3, 0x1.c6b08d7047e8bp-5, 0x1.3b2ab7181b757p-7, 0x1.5d87fe86f8348p-10, 0x1.4308ac85aa619p-13,
                                0x1.ffcb952673288p-17, 0x1.63d136368c2cep-20, 0x1.b63871c687389p-24};

struct SampleArgs {
    const void* x;
    uint64_t stride;
    uint32_t vocab;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t* top_k;
    int32_t* tokens;
    float* probs;
    double magic;                                  // 2^(52 - scale): added to a weight, it leaves its fixed-point form in the low bits
    double exp2[TERMS];                            // here they are one load; as constants in the code, two instructions each
};

// an order that unsigned integers have; -0 as +0
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// a logit and its index as one number: what comes first is larger
__device__ __forceinline__ uint64_t place_of(float x, int32_t i) { return (uint64_t)key_of(x) << 32 | (0xffffffffu - (uint32_t)i); }
__device__ __forceinline__ int32_t index_of(uint64_t place) { return (int32_t)(0xffffffffu - (uint32_t)place); }

struct Shared {
    uint64_t hist[BINS];                           // or what a list is sorted in, and the weights of a sorted one
    uint64_t places[LIST];
    uint64_t sums[WAVES];
    uint64_t before, cut, total;                   // (cut: a place)
    uint32_t bin, n, found;
};

// Sums over lanes by data moves between them that need no LDS: rows of 16 lanes, then the last lane of a row to the next ones
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, true);
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t moved(uint64_t x) {
    return (uint64_t)moved<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)x);
}
__device__ __forceinline__ uint64_t row_upto(uint64_t x) {      // of this lane and those below in its row
    x += moved<0x111, 0xf>(x);
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    return x;
}
__device__ __forceinline__ uint64_t wave_upto(uint64_t x) {     // of this lane and those below
    x = row_upto(x);
    x += moved<0x142, 0xa>(x);
    x += moved<0x143, 0xc>(x);
    return x;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t x, uint32_t lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), (int)lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane);
}
// the largest of the lanes, in all of them
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    uint32_t y;
    y = moved<0x111, 0xf>(x), x = y > x ? y : x;
    y = moved<0x112, 0xf>(x), x = y > x ? y : x;
    y = moved<0x114, 0xf>(x), x = y > x ? y : x;
    y = moved<0x118, 0xf>(x), x = y > x ? y : x;
    y = moved<0x142, 0xa>(x), x = y > x ? y : x;
    y = moved<0x143, 0xc>(x), x = y > x ? y : x;
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// What is kept: logits above x, and those that equal it up to index i
struct Cut {
    float x;
    int32_t i;
    __device__ __forceinline__ bool keeps(float v, int32_t at) const { return v > x || (v == x && at <= i); }
};
__device__ __forceinline__ Cut cut_at(uint64_t place) { return Cut{of_key((uint32_t)(place >> 32)), index_of(place)}; }

template <typename T> struct Row {
    static constexpr int VE = 16 / sizeof(T);
    const SampleArgs& a;
    Shared& s;
    const v4u* base;                               // the aligned vectors that cover the row
    uint32_t shift, covered, vectors, per_wave, its, v0, v1;   // elements in front of the row; this wave's vectors
    uint32_t lane, wave, tid;
    float max;
    double step;                                   // log2(e) / temperature

    __device__ __forceinline__ Row(const SampleArgs& a, Shared& s, uint32_t row) : a(a), s(s) {
        const uintptr_t at = (uintptr_t)((const T*)a.x + row * a.stride);
        shift = (uint32_t)(at & 15) / sizeof(T);
        base = (const v4u*)(at & ~(uintptr_t)15);
        covered = a.vocab + shift;
        vectors = (covered + VE - 1) / VE;
        per_wave = (vectors + WAVES - 1) / WAVES;
        its = (per_wave + 63) / 64;
        tid = threadIdx.x;
        lane = tid % 64;
        wave = __builtin_amdgcn_readfirstlane(tid / 64);
        v0 = wave * per_wave;
        v0 = v0 < vectors ? v0 : vectors;
        v1 = v0 + per_wave < vectors ? v0 + per_wave : vectors;
        max = 0.0f;
        step = 0.0;
    }
    // vector `it` of this lane; elements that are none of the row's are NaN
    __device__ __forceinline__ v4u vector(uint32_t it) const {
        const uint32_t v = v0 + it * 64 + lane;
        Vec16<T> x;
        x.u = v4u{~0u, ~0u, ~0u, ~0u};
        if (v < v1) {
            x.u = base[v];
            if (v == 0 || v == vectors - 1) {
                Vec16<T> none;
                none.u = v4u{~0u, ~0u, ~0u, ~0u};
#pragma unroll
                for (int e = 0; e < VE; e++) {
                    const uint32_t c = v * VE + e;
                    if (c < shift || c >= covered) x.e[e] = none.e[e];
                }
            }
        }
        return x.u;
    }
    // f(logit, index) for this thread's share.  Loops stay loops: straight code, which a wave runs once, would wait for its own instructions
    template <typename F> __device__ __forceinline__ void each(F f) const {
        v4u next = vector(0);
#pragma unroll 1
        for (uint32_t it = 0; it < its; it++) {
            Vec16<T> x;
            x.u = next;
            next = vector(it + 1);                              // beyond the last: nothing is loaded
            const int32_t i = (int32_t)((v0 + it * 64 + lane) * VE) - (int32_t)shift;
#pragma unroll
            for (int e = 0; e < VE; e++) f(Ar<T>::widen(x.e[e]), i + e);
        }
    }
    __device__ __forceinline__ double weight(float x) const {
        const double y = fmax(((double)x - (double)max) * step, -100.0), n = rint(y), f = y - n;
        double q = a.exp2[TERMS - 1];
#pragma unroll
        for (int t = TERMS - 2; t >= 0; t--) q = __builtin_fma(q, f, a.exp2[t]);
        return ldexp(__builtin_fma(q, f, 1.0), (int)n);
    }
    __device__ __forceinline__ uint64_t fixed(double w) const { return (uint64_t)__double_as_longlong(w + a.magic) & ((1ull << 52) - 1); }

    // the sum over the block of what each thread brings; upto: of this thread and those below
    __device__ __forceinline__ uint64_t block_sum(uint64_t x, uint64_t* upto = nullptr) {
        const uint64_t mine = wave_upto(x);
        __syncthreads();
        if (lane == 63) s.sums[wave] = mine;
        __syncthreads();
        const uint64_t waves = row_upto(lane < WAVES ? s.sums[lane] : 0);
        if (upto) *upto = mine + (wave ? lane_of(waves, wave - 1) : 0);
        return lane_of(waves, WAVES - 1);
    }
    // the largest two numbers of the block, each among the threads' own
    __device__ __forceinline__ void block_max(uint32_t& x, uint32_t& y) {
        x = wave_max(x);
        y = wave_max(y);
        __syncthreads();
        if (lane == 0) s.sums[wave] = (uint64_t)x << 32 | y;
        __syncthreads();
        const uint64_t both = s.sums[lane % WAVES];
        x = wave_max((uint32_t)(both >> 32));
        y = wave_max((uint32_t)both);
    }
    // the lowest and highest key of the block; a thread without one brings low above high
    __device__ __forceinline__ void key_range(uint32_t& low, uint32_t& high) {
        low = ~low;
        block_max(low, high);
        low = ~low;
    }
    // below `whole` and, taken into [0, 1), uniform of it: a sum of whole numbers exceeds u * whole if it exceeds its whole part
    __device__ __forceinline__ static uint64_t part_of(float uniform, uint64_t whole) {
        const double u = uniform >= 0.0f ? (uniform < 1.0f ? uniform : 1.0f - 0x1p-24f) : 0.0f;
        return (uint64_t)(u * (double)whole);
    }

    // The n numbers of the threads below n, none of them 0, in descending order: a bitonic sort, between lanes where partners are in one wave.  Uses the first half of s.hist.
    // Few are counted, several threads to a number, which takes fewer barriers and moves (64 rows of 50295 f16, two such sorts, us counted | bitonic: up to 40 of k 16.7 | 21.4,
    // up to 100 22.9 | 25.3, up to 200 25.4 | 27.8).
    __device__ __forceinline__ uint64_t sorted(uint64_t x, uint32_t n) {
        uint32_t pad = 64;
        while (pad < n) pad <<= 1;
        if (pad <= 256) {
            uint64_t* const to = s.hist + 256;
            uint32_t* const rank = (uint32_t*)(s.hist + 512);
            __syncthreads();
            if (tid < pad) {
                s.hist[tid] = x;
                to[tid] = 0;
                rank[tid] = 0;
            }
            __syncthreads();
            const uint32_t t = tid & (pad - 1);
            const uint64_t me = s.hist[t];
            uint32_t ahead = 0;
            for (uint32_t j = tid / pad; j < n; j += BLOCK / pad) ahead += s.hist[j] > me;
            if (t < n) atomicAdd(&rank[t], ahead);
            __syncthreads();
            if (tid < n) to[rank[tid]] = x;
            __syncthreads();
            x = tid < pad ? to[tid] : 0;
            __syncthreads();
            return x;
        }
#pragma unroll 1
        for (uint32_t size = 2; size <= pad; size <<= 1)
#pragma unroll 1
            for (uint32_t stride = size / 2; stride; stride >>= 1) {
                uint64_t other = 0;
                if (stride >= 64) {
                    __syncthreads();
                    s.hist[tid] = x;
                    __syncthreads();
                    other = s.hist[tid ^ stride];
                } else if (wave * 64 < pad) {                   // (the others' numbers are 0, and stay there)
                    other = __shfl_xor(x, (int)stride);
                } else {
                    continue;
                }
                const bool larger = ((tid & stride) == 0) == ((tid & size) == 0);
                x = (x > other) == larger ? x : other;
            }
        __syncthreads();
        return x;
    }

    // The first index at which the sum of metric(logit, index), by index, exceeds `target`, or where `fraction` that part of the whole sum, `total`; mine: what this
    // thread's share adds to it.  First among the waves' shares, then among the threads, to which the one share is dealt out again.
    template <typename F> __device__ __forceinline__ int32_t search(uint64_t mine, bool fraction, float uniform, uint64_t target, F metric, uint64_t& total) {
        const uint64_t share = wave_upto(mine);
        __syncthreads();
        if (lane == 63) s.sums[wave] = share;
        if (tid == 0) s.found = a.vocab - 1;
        __syncthreads();
        uint64_t upto = row_upto(lane < WAVES ? s.sums[lane] : 0);
        total = lane_of(upto, WAVES - 1);
        if (fraction) target = part_of(uniform, total);
        uint32_t w = (uint32_t)__popcll(__ballot(lane < WAVES && upto <= target));
        w = w < WAVES ? w : WAVES - 1;
        w = __builtin_amdgcn_readfirstlane(w);
        uint64_t before = w ? lane_of(upto, w - 1) : 0;
        uint32_t c0 = w * per_wave * VE, c1 = (w + 1) * per_wave * VE;
        c0 = c0 > shift ? c0 : shift;
        c1 = c1 < covered ? c1 : covered;
        c1 = c1 > c0 ? c1 : c0;
        const uint32_t some = c0 < c1 ? c0 : shift;             // an element that is there
        const T* x = (const T*)base;
        const uint32_t rounds = (c1 - c0 + BLOCK - 1) / BLOCK, first = c0 + wave * rounds * 64 + lane;         // of 64 neighbours to a wave
        uint64_t sum = 0;
        auto weigh = [&](uint32_t round) -> uint64_t {
            const uint32_t c = first + round * 64;
            const T v = x[c < c1 ? c : some];
            return c < c1 ? metric(Ar<T>::widen(v), (int32_t)(c - shift)) : 0;
        };
#pragma unroll 1
        for (uint32_t n = 0; n < rounds; n++) sum += weigh(n);
        const uint64_t sub = wave_upto(sum);
        __syncthreads();
        if (lane == 63) s.sums[wave] = sub;
        __syncthreads();
        upto = before + row_upto(lane < WAVES ? s.sums[lane] : 0);
        w = (uint32_t)__popcll(__ballot(lane < WAVES && upto <= target));
        w = __builtin_amdgcn_readfirstlane(w < WAVES ? w : WAVES - 1);
        if (wave == w) {
            before = w ? lane_of(upto, w - 1) : before;
#pragma unroll 1
            for (uint32_t n = 0; n < rounds; n++) {
                const uint64_t here = before + wave_upto(weigh(n)), beyond = __ballot(here > target);
                before = lane_of(here, 63);
                if (!beyond) continue;
                if (lane == (uint32_t)__builtin_ctzll(beyond)) s.found = first + n * 64 - shift;
                break;
            }
        }
        __syncthreads();
        return (int32_t)s.found;
    }

    __device__ __forceinline__ void clear() {
        __syncthreads();
        for (uint32_t i = tid; i < BINS; i += BLOCK) s.hist[i] = 0;
        if (tid == 0) {
            s.n = 0;
            s.bin = BINS;
        }
        __syncthreads();
    }
    // Into s.bin and s.before: the bin of the histogram at which the sum from the top, and offset, reaches `want`, and the sum in front of it.  s.bin stays BINS if none does.
    __device__ __forceinline__ void find_bin(uint64_t offset, double want) {
        __syncthreads();
        uint64_t h[BINS / BLOCK], sum = 0, upto;
#pragma unroll
        for (uint32_t i = 0; i < BINS / BLOCK; i++) {
            h[i] = s.hist[tid * (BINS / BLOCK) + i];
            sum += h[i];
        }
        block_sum(sum, &upto);
        uint64_t before = offset + upto - sum;
#pragma unroll
        for (uint32_t i = 0; i < BINS / BLOCK; i++) {
            if ((double)before < want && !((double)(before + h[i]) < want)) {
                s.bin = tid * (BINS / BLOCK) + i;
                s.before = before;
            }
            before += h[i];
        }
        __syncthreads();
    }
    __device__ __forceinline__ void list(float x, int32_t i) {
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < LIST) s.places[at] = place_of(x, i);
    }

    // The cut among the members of a step, those with member(x, i), which s.places lists where they are not too many: the last of them that has less than `want` in front of it,
    // `before` being what lies in front of them all.  metric(x): what one weighs.
    template <typename In, typename M> __device__ __forceinline__ Cut cut_in_step(uint64_t before, double want, In member, M metric) {
        __syncthreads();
        uint32_t low = 0xffffffffu, high = 0;
        if (s.n > LIST) {
            each([&](float x, int32_t i) {
                if (!member(x, i)) return;
                const uint32_t key = key_of(x);
                low = key < low ? key : low;
                high = key > high ? key : high;
            });
            key_range(low, high);
        }
        while (s.n > LIST && low < high) {
            // steps of whole keys between the lowest and the highest
            uint32_t down = 0;
            while ((high - low) >> down >= BINS) down++;
            auto among = [&](float x, int32_t i) -> bool { return member(x, i) && key_of(x) >= low && key_of(x) <= high; };
            clear();
            each([&](float x, int32_t i) {
                if (among(x, i)) atomicAdd((unsigned long long*)&s.hist[(high - key_of(x)) >> down], (unsigned long long)metric(x));
            });
            find_bin(before, want);
            const uint32_t bin = s.bin < BINS ? s.bin : (high - low) >> down;    // (the last sum is the members' whole: it reaches what is wanted)
            if (s.bin < BINS) before = s.before;
            uint32_t l = 0xffffffffu, h = 0;
            each([&](float x, int32_t i) {
                if (!among(x, i) || (high - key_of(x)) >> down != bin) return;
                const uint32_t key = key_of(x);
                l = key < l ? key : l;
                h = key > h ? key : h;
                list(x, i);
            });
            key_range(l, h);
            low = l;
            high = h;
        }
        const uint32_t n = s.n;
        if (n > LIST) {
            // all alike: as many as it takes, the lower indices first
            const float same = of_key(low);
            const uint64_t w = metric(same);
            uint32_t keep = n;
            if (w) {
                const double more = (want - (double)before) / (double)w;
                keep = more < (double)n ? (uint32_t)more : n;
                while (keep > 0 && !((double)(before + (keep - 1) * w) < want)) keep--;
                while (keep < n && (double)(before + keep * w) < want) keep++;
            }
            uint64_t mine = 0, total;
            auto is = [&](float x, int32_t i) -> uint64_t { return x == same && member(x, i); };
            each([&](float x, int32_t i) { mine += is(x, i); });
            return Cut{same, search(mine, false, 0.0f, keep ? keep - 1 : 0, is, total)};
        }
        const uint64_t me = sorted(tid < n ? s.places[tid] : 0, n);
        const uint64_t w = tid < n ? metric(of_key((uint32_t)(me >> 32))) : 0;
        uint64_t upto;
        if (tid == 0) s.cut = 0;                                // (all of them; but one place always is where the sum reaches what is wanted)
        block_sum(w, &upto);
        upto += before;
        if (tid < n && (double)(upto - w) < want && !((double)upto < want)) s.cut = me;
        __syncthreads();
        return s.cut ? cut_at(s.cut) : Cut{-INFINITY, -1};
    }

    // A bound that at least k <= 1024 logits reach: that k of the threads' own maxima do, by a histogram of them over equal steps down to `least`, the smallest that is not -inf.  -inf
    // if so many threads have none
    __device__ __forceinline__ float reached_by(uint32_t k, float mine, float least) {
        float per = BINS / (max - least);
        per = per < 1e30f ? per : 1e30f;
        clear();
        if (mine >= least) {
            const float b = (max - mine) * per;
            atomicAdd((unsigned long long*)&s.hist[b < (float)(BINS - 1) ? (uint32_t)b : BINS - 1], 1ull);
        }
        find_bin(0, (double)k);
        const uint32_t bin = s.bin;
        if (bin == BINS) return -INFINITY;
        return bin < BINS - 1 && per > 0x1p-64f && per < 0x1p64f ? max - ((float)bin + 1.5f) / per : least;        // (half a step out, for the roundings)
    }

    // Draws from the n places of s.places, which hold all that may be kept: the first k of them, of those the ones with less than p of their weight
    // in front of them, of those the ones that weigh min_p.
    __device__ __forceinline__ void draw(uint32_t n, uint32_t k, float p, double min_p, float uniform, int32_t* token, float* prob) {
        uint64_t* const heavy = s.hist + LIST;
        __syncthreads();
        k = k < n ? k : n;
        const uint64_t place = sorted(tid < n ? s.places[tid] : 0, n);
        const double w = tid < k ? weight(of_key((uint32_t)(place >> 32))) : 0.0;
        uint64_t f = tid < k ? fixed(w) : 0, upto;
        heavy[tid] = f;
        const uint64_t total = block_sum(f, &upto);
        const double want = p > 0.0f ? (double)p * (double)total : 0.5;
        const bool stays = tid < k && (!(p < 1.0f) || (double)(upto - f) < want) && w >= min_p;
        const uint32_t kept = (uint32_t)block_sum(stays, nullptr);
        if (tid == kept - 1) s.total = upto;
        // those that stay, by index
        const uint64_t by = sorted(tid < kept ? place << 32 | (tid + 1) : 0, kept);
        const uint64_t whole = s.total, target = part_of(uniform, whole);
        f = tid < kept ? heavy[(uint32_t)by - 1] : 0;
        block_sum(f, &upto);
        if (tid < kept && upto > target && upto - f <= target) {                // one does
            *token = index_of(by >> 32);
            if (prob) *prob = (float)((double)f / (double)whole);
        }
    }
};

template <typename T> __global__ void __launch_bounds__(BLOCK) sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const uint32_t row = blockIdx.x;
    Row<T> r(a, s, row);
    const float temperature = a.temperature ? a.temperature[row] : 1.0f, uniform = a.uniform[row];
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p_raw = a.min_p ? a.min_p[row] : 0.0f;
    int32_t* const token_at = a.tokens + row;
    float* const prob_at = a.probs ? a.probs + row : nullptr;
    float mine = -INFINITY;
    r.each([&](float x, int32_t) { mine = fmaxf(mine, x); });
    uint32_t high = key_of(mine), low = mine > -INFINITY ? ~high : 0;
    r.block_max(high, low);
    r.max = of_key(high);
    const float least = of_key(~low);              // of the threads' maxima
    uint64_t total;
    if (r.max == -INFINITY || r.max == INFINITY || !(temperature > 0.0f)) {
        // nothing to choose from; equals that share all the weight; or, greedy, the first of the largest
        auto top = [&](float x, int32_t) -> uint64_t { return x == r.max && x > -INFINITY; };
        uint64_t n = 0;
        r.each([&](float x, int32_t i) { n += top(x, i); });
        uint64_t m = r.block_sum(n);
        if (!(temperature > 0.0f)) m = m < 1 ? m : 1;
        if (k > 0 && (uint64_t)k < m) m = (uint64_t)k;
        if (top_p < 1.0f && m) {
            const double want = top_p > 0.0f ? ceil((double)top_p * (double)m) : 1.0;
            m = want < 1.0 ? 1 : want < (double)m ? (uint64_t)want : m;
        }
        const int32_t token = r.search(n, false, 0.0f, r.part_of(uniform, m), top, total);
        if (r.tid == 0) {
            *token_at = m ? token : -1;
            if (prob_at) *prob_at = m ? (float)(1.0 / (double)m) : 0.0f;
        }
        return;
    }
    r.step = 1.4426950408889634 / (double)temperature;
    const double min_p = min_p_raw > 0.0f ? (min_p_raw < 1.0f ? min_p_raw : 1.0f) : 0.0;
    Cut cut = {-INFINITY, -1};
    // top-k counts, then top-p weighs.  What lies 48 temperatures below the largest weighs 0 in fixed point: whether it is among the k does not matter
    for (int phase = 0; phase < 2; phase++) {
        const bool counts = phase == 0;
        if (counts ? k <= 0 || (uint32_t)k >= a.vocab : !(top_p < 1.0f)) continue;
        const Cut front = cut;
        const float p = top_p > 0.0f ? top_p : 0.0f;
        float floor;
        if (counts) {
            floor = (uint32_t)k <= BLOCK ? r.reached_by((uint32_t)k, mine, least) : -INFINITY;
            floor = fmaxf(floor, r.max - 48.0f * temperature);
        } else {
            // all of those below this weigh less than half of what may be dropped; 0.7 is a little above ln 2
            floor = p > 0.0f ? r.max - temperature * 0.7f * __builtin_amdgcn_logf(2.0f * (float)a.vocab / (1.0f - p)) : r.max;
        }
        floor = fmaxf(floor, -3.4028235e38f);                   // (of an endless temperature: all that are finite)
        const bool all = front.x == -INFINITY;                  // nothing is cut yet: what is not finite weighs 0 and lies below the floor
        auto in = [&](float x, int32_t i) -> bool { return x >= floor && (all || front.keeps(x, i)); };
        // Listed, where as many hardly ever pass a list, which is then a walk for nothing (64 rows of 50295 f16, us listed | cut by a histogram: k 20 12.6 | 42, 200 18.7 | 49,
        // 500 33 | 49; 700 59 | 50).  None is listed yet
        if (counts && (uint32_t)k <= LIST / 2) {
            r.each([&](float x, int32_t i) {
                if (in(x, i)) r.list(x, i);
            });
            __syncthreads();
            if (s.n <= LIST) {
                r.draw(s.n, (uint32_t)k, top_p, min_p, uniform, token_at, prob_at);
                return;
            }
        }
        float per = BINS / (r.max - floor);                     // equal steps of the logit between the floor and the largest
        per = per < 1e30f ? per : 1e30f;
        auto bin_of = [&](float x) -> uint32_t {
            const float b = (r.max - x) * per;
            return b < (float)(BINS - 1) ? (uint32_t)b : BINS - 1;
        };
        auto metric = [&](float x) -> uint64_t { return counts ? 1 : r.fixed(r.weight(x)); };
        r.clear();
        uint64_t sum = 0;
        r.each([&](float x, int32_t i) {
            if (all || front.keeps(x, i)) {
                const uint64_t w = metric(x);
                sum += w;
                if (x >= floor) atomicAdd((unsigned long long*)&s.hist[bin_of(x)], (unsigned long long)w);
            }
        });
        const uint64_t whole = r.block_sum(sum);
        const double want = counts ? (double)k : p > 0.0f ? (double)p * (double)whole : 0.5;
        r.find_bin(0, want);
        const uint32_t bin = s.bin;
        const uint64_t before = s.before;
        if (bin == BINS) continue;                              // fewer than k
        // the step's ends, half a step out (a rounded end passes no logit that the end itself does not): few logits lie between them
        const float width = 1.0f / per;
        const bool narrow = per > 0x1p-64f && per < 0x1p64f;
        const float above = bin > 0 && narrow ? r.max - ((float)bin - 0.5f) * width : INFINITY, below = bin < BINS - 1 && narrow ? r.max - ((float)bin + 1.5f) * width : floor;
        r.each([&](float x, int32_t i) {
            if (x >= below && x <= above && in(x, i) && bin_of(x) == bin) r.list(x, i);
        });
        cut = r.cut_in_step(before, want, [&](float x, int32_t i) -> bool { return in(x, i) && bin_of(x) == bin; }, metric);
    }
    auto kept = [&](float x, int32_t i) -> uint64_t {
        if (!(x >= cut.x) || !cut.keeps(x, i)) return 0;        // most fail the first
        const double w = r.weight(x);
        return w >= min_p ? r.fixed(w) : 0;
    };
    uint64_t sum = 0;
    r.each([&](float x, int32_t i) { sum += kept(x, i); });
    const int32_t token = r.search(sum, true, uniform, 0, kept, total);
    if (r.tid == 0) {
        *token_at = token;
        if (prob_at) *prob_at = (float)((double)kept(Ar<T>::widen(((const T*)a.x)[row * a.stride + token]), token) / (double)total);
    }
}

template <typename T> int launch(rt_device* dev, const SampleArgs& a, uint32_t rows) {
    hipLaunchKernelGGL((sample_kernel<T>), dim3(rows), dim3(BLOCK), 0, dev->stream, a);
    RT_CHECK_LAUNCH("sample_kernel");
    return RT_OK;
}

}  // namespace

extern "C" int rt_sample(rt_device* dev, int dt, const void* x, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float* temperature, const int32_t* top_k,
                         const float* top_p, const float* min_p, const float* uniform, int32_t* tokens, float* probs) {
    static const char* const who = "rt_sample";
    RT_REQUIRE(rt_is_float_dt(dt), RT_ERR_DTYPE, "%s: dtype %d is not F32, F16 or BF16", who, dt);
    RT_REQUIRE(rows > 0 && vocab > 0, RT_ERR_SHAPE, "%s: zero extent", who);
    RT_REQUIRE(vocab <= MOST_VOCAB && rows < (1u << 22), RT_ERR_SIZE, "%s: %u rows of %u", who, rows, vocab);
    RT_REQUIRE(row_stride < RT_MAX_NUMEL / rows, RT_ERR_SIZE, "%s: rows are too far apart", who);
    RT_REQUIRE(x && uniform && tokens, RT_ERR_NULL_POINTER, "%s: NULL operand", who);
    RT_REQUIRE(rt_aligned(x, (size_t)rt_dt_bytes(dt)) && rt_aligned(temperature, 4) && rt_aligned(top_k, 4) && rt_aligned(top_p, 4) && rt_aligned(min_p, 4) &&
                   rt_aligned(uniform, 4) && rt_aligned(tokens, 4) && rt_aligned(probs, 4),
               RT_ERR_ALIGN, "%s: misaligned pointer", who);
    int rc = rt_enter(dev);
    if (rc) return rc;
    SampleArgs a;
    a.x = x;
    a.stride = row_stride;
    a.vocab = vocab;
    a.temperature = temperature; a.top_p = top_p; a.min_p = min_p; a.uniform = uniform; a.top_k = top_k;
    a.tokens = tokens; a.probs = probs;
    int scale = 46;                                             // the sum of the weights, at most vocab, stays below 2^62; 46 bits to a weight up to 2^16 tokens
    while ((uint64_t)vocab << scale > 1ull << 62) scale--;
    a.magic = ldexp(1.0, 52 - scale);
    for (int t = 0; t < TERMS; t++) a.exp2[t] = EXP2[t];
    switch (dt) {
        case RT_F32: return launch<float>(dev, a, rows);
        case RT_F16: return launch<half_t>(dev, a, rows);
        default: return launch<bf16_t>(dev, a, rows);
    }
}
