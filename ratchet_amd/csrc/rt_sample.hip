// Sampling of tokens from rows of logits: temperature, top-k, top-p, min-p, from given random numbers.
//
//     w_i = exp((x_i - max x) / temperature)                  in 64-bit floats, rounded to multiples of 2^-scale (fixed point in 64 bits)
//     K: the top_k largest logits; P: of K, in descending order, those with (sum of the w before) < top_p * (sum of K's w); M: w_i >= min_p
//     token: the first index whose cumulative kept weight, by index, exceeds uniform * (sum of the kept w)
// All three filters keep a front of the same order, larger logits first and of equal ones the lower index, so what they keep is a cut in it: a logit and
// the index up to which its equals stay.  Sums of fixed-point numbers are the same in any order and on any split, so atomics and waves need no order.
//
// A block to a row, a sixteenth of the row to a wave, the logits in registers where they fit.  A cut is found by a histogram of the weights (or counts)
// over 2048 equal steps of the logit, then by comparing the few members of the step it lies in; a step with too many members is cut into 2048 again.
#include <math.h>

#include "rt_arith.h"
#include "rt_internal.h"

namespace {

constexpr int BLOCK = 1024, WAVES = BLOCK / 64;
constexpr uint32_t BINS = 2048, LIST = 1024, NO_CUT = 0;       // NO_CUT: a key below all keys
constexpr uint32_t MOST_VOCAB = 1u << 24;

struct SampleArgs {
    const void* x;
    uint64_t stride;
    uint32_t vocab;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t* top_k;
    int32_t* tokens;
    float* probs;
    double magic;                                  // 2^(52 - scale): added to a weight, it leaves its fixed-point form in the low bits
};

// an order that unsigned integers have; -0 as +0
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Shared {
    uint64_t hist[BINS];
    uint64_t list_key[LIST];                       // key, then the index from the top, so that what comes first is larger
    uint64_t list_w[LIST];
    uint64_t wave_sum[WAVES];
    uint32_t wave_a[WAVES], wave_b[WAVES];
    uint64_t before;
    uint32_t bin, count, low, high;
    uint64_t cut;
    uint32_t found;
};

template <typename T> __device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
    for (int i = 32; i; i >>= 1) x += __shfl_xor(x, i);
    return x;
}
template <typename T> __device__ __forceinline__ T wave_upto(T x) {              // of this lane and those below
    const int lane = (int)__lane_id();
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const T y = __shfl_up(x, i);
        if (lane >= i) x += y;
    }
    return x;
}

// ITS: vectors that a lane holds; 0: the row is read again for every walk over it
template <typename T, int ITS> struct Row {
    static constexpr int VE = 16 / sizeof(T);
    const SampleArgs& a;
    Shared& s;
    const v4u* base;                               // the aligned vectors that cover the row
    uint32_t shift, covered, vectors, per_wave, its, v0, v1;   // elements in front of the row; this wave's vectors
    uint32_t lane, wave, tid;
    bool infinite;                                 // the largest is +inf: those are 0, the others -inf
    float max;
    double step;                                   // log2(e) / temperature
    float r[ITS ? ITS * VE : 1];

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
        infinite = false;
        max = 0.0f;
        step = 0.0;
    }
    __device__ __forceinline__ float clean(float x) const {                    // NaN ranks with -inf
        x = x == x ? x : -INFINITY;
        return infinite ? (x == INFINITY ? 0.0f : -INFINITY) : x;
    }
    __device__ __forceinline__ void vector(uint32_t it, float* to) const {
        const uint32_t v = v0 + it * 64 + lane;
        Vec16<T> x;
        if (v < v1) x.u = base[v];
#pragma unroll
        for (int e = 0; e < VE; e++) {
            const uint32_t c = v * VE + e;
            to[e] = v < v1 && c >= shift && c < covered ? clean(Ar<T>::widen(x.e[e])) : -INFINITY;
        }
    }
    __device__ __forceinline__ void load() {
        if constexpr (ITS != 0) {
#pragma unroll
            for (int it = 0; it < ITS; it++)
                if ((uint32_t)it < its) vector(it, r + it * VE);
        }
    }
    // f(logit, index) for this thread's share; elements beyond the row are -inf
    template <typename F> __device__ __forceinline__ void each(F f) const {
        if constexpr (ITS != 0) {
#pragma unroll
            for (int it = 0; it < ITS; it++)
                if ((uint32_t)it < its)
#pragma unroll
                    for (int e = 0; e < VE; e++) f(r[it * VE + e], (v0 + it * 64 + lane) * VE + e - shift);
        } else {
            for (uint32_t it = 0; it < its; it++) {
                float x[VE];
                vector(it, x);
#pragma unroll
                for (int e = 0; e < VE; e++) f(x[e], (v0 + it * 64 + lane) * VE + e - shift);
            }
        }
    }
    __device__ __forceinline__ double weight(float x) const {
        // 2^y = 2^n (1 + f q(f)), n the nearest integer: q interpolates at Chebyshev's points, 4e-14 off at most
        const double y = fmax(((double)x - (double)max) * step, -100.0), n = rint(y), f = y - n;
        double q = 0x1.b63871c687389p-24;
        q = __builtin_fma(q, f, 0x1.63d136368c2cep-20);
        q = __builtin_fma(q, f, 0x1.ffcb952673288p-17);
        q = __builtin_fma(q, f, 0x1.4308ac85aa619p-13);
        q = __builtin_fma(q, f, 0x1.5d87fe86f8348p-10);
        q = __builtin_fma(q, f, 0x1.3b2ab7181b757p-7);
        q = __builtin_fma(q, f, 0x1.c6b08d7047e8bp-5);
        q = __builtin_fma(q, f, 0x1.ebfbdff823cedp-3);
        q = __builtin_fma(q, f, 0x1.62e42fefa39efp-1);
        return ldexp(__builtin_fma(q, f, 1.0), (int)n);
    }
    __device__ __forceinline__ uint64_t fixed(double w) const { return (uint64_t)__double_as_longlong(w + a.magic) & ((1ull << 52) - 1); }

    // the sum over the block of what each thread brings
    __device__ __forceinline__ uint64_t block_sum(uint64_t x) {
        x = wave_sum(x);
        if (lane == 0) s.wave_sum[wave] = x;
        __syncthreads();
        const uint64_t all = wave_sum(lane < WAVES ? s.wave_sum[lane] : 0);
        __syncthreads();
        return all;
    }
    __device__ __forceinline__ float block_max(float x) {
#pragma unroll
        for (int i = 32; i; i >>= 1) x = fmaxf(x, __shfl_xor(x, i));
        if (lane == 0) s.wave_a[wave] = __float_as_uint(x);
        __syncthreads();
        x = __uint_as_float(s.wave_a[lane % WAVES]);
#pragma unroll
        for (int i = WAVES / 2; i; i >>= 1) x = fmaxf(x, __shfl_xor(x, i));
        __syncthreads();
        return x;
    }

    // The first index at which the sum of metric(logit, index), by index, exceeds `target`, which is below `total`, the sum of them all; before: the sum in front of it.
    // First among the waves' shares, whose sums each thread brings its part of, then among the threads, to which the one share is dealt out again.
    template <typename F> __device__ __forceinline__ uint32_t search(uint64_t mine, bool fraction, float uniform, uint64_t target, F metric, uint64_t& total) {
        const uint64_t share = wave_sum(mine);
        if (lane == 0) s.wave_sum[wave] = share;
        __syncthreads();
        uint64_t upto = wave_upto(lane < WAVES ? s.wave_sum[lane] : 0);
        total = __shfl(upto, WAVES - 1);
        if (fraction) {
            const double u = uniform >= 0.0f ? (uniform < 1.0f ? uniform : 1.0f - 0x1p-24f) : 0.0f;
            target = (uint64_t)(u * (double)total);             // a sum exceeds u * total if it exceeds its whole part
        }
        const uint64_t ahead = __ballot(lane < WAVES && upto <= target);
        uint32_t w = (uint32_t)__popcll(ahead);
        w = w < WAVES ? w : WAVES - 1;
        uint64_t before = w ? __shfl(upto, (int)w - 1) : 0;
        uint32_t c0 = w * per_wave * VE, c1 = (w + 1) * per_wave * VE;
        c0 = c0 > shift ? c0 : shift;
        c1 = c1 < covered ? c1 : covered;
        c1 = c1 > c0 ? c1 : c0;
        const uint32_t each_has = (c1 - c0 + BLOCK - 1) / BLOCK, c = c0 + tid * each_has;
        const T* x = (const T*)base;
        uint64_t sum = 0;
        for (uint32_t i = 0; i < each_has; i++)
            if (c + i < c1) sum += metric(clean(Ar<T>::widen(x[c + i])), c + i - shift);
        upto = wave_upto(sum);
        __syncthreads();
        if (lane == 63) s.wave_sum[wave] = upto;
        if (tid == 0) s.found = a.vocab - 1;
        __syncthreads();
        const uint64_t waves_before = wave_sum(lane < wave ? s.wave_sum[lane] : 0);
        before += waves_before + upto - sum;
        if (before <= target && before + sum > target) {
            for (uint32_t i = 0; i < each_has; i++) {
                if (c + i >= c1) break;
                before += metric(clean(Ar<T>::widen(x[c + i])), c + i - shift);
                if (before > target) {
                    s.found = c + i - shift;
                    break;
                }
            }
        }
        __syncthreads();
        const uint32_t found = s.found;
        __syncthreads();
        return found;
    }

    // Into s.bin and s.before: the bin of the histogram at which the sum from the top reaches `want`, and the sum in front of it.  s.bin is BINS if none does.
    __device__ __forceinline__ void find_bin(uint64_t offset, double want) {
        __syncthreads();
        if (tid == 0) s.bin = BINS;
        uint64_t h[BINS / BLOCK], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < BINS / BLOCK; i++) {
            h[i] = s.hist[tid * (BINS / BLOCK) + i];
            sum += h[i];
        }
        uint64_t upto = wave_upto(sum);
        if (lane == 63) s.wave_sum[wave] = upto;
        __syncthreads();
        uint64_t before = offset + wave_sum(lane < wave ? s.wave_sum[lane] : 0) + upto - sum;
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
    __device__ __forceinline__ void clear() {
        __syncthreads();
        for (uint32_t i = tid; i < BINS; i += BLOCK) s.hist[i] = 0;
        if (tid == 0) {
            s.count = 0;
            s.low = 0xffffffffu;
            s.high = 0;
        }
        __syncthreads();
    }

    // The cut at which the sum of the metric, in descending order, reaches `want`: the key of a logit and, from the top, the last index of its equals
    // that stays, as one number; what is kept is >= it.  in(x, i): takes part; floor: what lies below need not; metric(x): its weight.
    template <typename In, typename M> __device__ uint64_t select(double want, float floor, In in, M metric) {
        // equal steps of the logit between the floor and the largest
        float per = BINS / (max - floor);
        per = per < 1e30f ? per : 1e30f;
        auto bin_of = [&](float x) -> uint32_t {
            const float b = (max - x) * per;
            return b < (float)(BINS - 1) ? (uint32_t)b : BINS - 1;
        };
        clear();
        each([&](float x, uint32_t i) {
            if (x >= floor && in(x, i)) atomicAdd((unsigned long long*)&s.hist[bin_of(x)], (unsigned long long)metric(x));
        });
        find_bin(0, want);
        if (s.bin == BINS) return NO_CUT;
        uint32_t bin = s.bin;
        uint64_t before = s.before;
        auto gather = [&](float x, uint32_t i) {
            const uint32_t at = atomicAdd(&s.count, 1u), key = key_of(x);
            atomicMin(&s.low, key);
            atomicMax(&s.high, key);
            if (at < LIST) {
                s.list_key[at] = (uint64_t)key << 32 | (0xffffffffu - i);
                s.list_w[at] = metric(x);
            }
        };
        each([&](float x, uint32_t i) {
            if (x >= floor && bin_of(x) == bin && in(x, i)) gather(x, i);
        });
        __syncthreads();
        while (s.count > LIST && s.low < s.high) {
            // steps of whole keys between the lowest and the highest of the members
            const uint32_t low = s.low, high = s.high;
            uint32_t down = 0;
            while ((high - low) >> down >= BINS) down++;
            clear();
            each([&](float x, uint32_t i) {
                const uint32_t key = key_of(x);
                if (key >= low && key <= high && in(x, i)) atomicAdd((unsigned long long*)&s.hist[(high - key) >> down], (unsigned long long)metric(x));
            });
            find_bin(before, want);
            bin = s.bin < BINS ? s.bin : (high - low) >> down;  // (the last sum is the members': it reaches what is wanted)
            if (s.bin < BINS) before = s.before;
            each([&](float x, uint32_t i) {
                const uint32_t key = key_of(x);
                if (key >= low && key <= high && (high - key) >> down == bin && in(x, i)) gather(x, i);
            });
            __syncthreads();
        }
        const uint32_t n = s.count;
        uint64_t cut;
        if (n > LIST) {
            // all alike: as many as it takes, the lower indices first
            const uint32_t key = s.low;
            const uint64_t w = s.list_w[0];
            uint32_t keep = n;
            if (w) {
                const double more = (want - (double)before) / (double)w;
                keep = more < (double)n ? (uint32_t)more : n;
                while (keep > 0 && !((double)(before + (keep - 1) * w) < want)) keep--;
                while (keep < n && (double)(before + keep * w) < want) keep++;
            }
            uint64_t mine = 0, total;
            auto same = [&](float x, uint32_t i) -> uint64_t { return key_of(x) == key && in(x, i); };
            each([&](float x, uint32_t i) { mine += same(x, i); });
            const uint32_t last = search(mine, false, 0.0f, keep - 1, same, total);
            cut = (uint64_t)key << 32 | (0xffffffffu - last);
        } else {
            // each member adds up those in front of it
            if (tid == 0) s.cut = ~0ull;
            __syncthreads();
            if (tid < n) {
                const uint64_t me = s.list_key[tid];
                uint64_t sum = before;
                for (uint32_t j = 0; j < n; j++) sum += s.list_key[j] > me ? s.list_w[j] : 0;
                if ((double)sum < want) atomicMin((unsigned long long*)&s.cut, (unsigned long long)me);
            }
            __syncthreads();
            cut = s.cut;
        }
        __syncthreads();
        return cut;
    }

    // A bound that at least k logits reach: the kth largest of the threads' own maxima, rounded down to a step of whole keys
    __device__ __forceinline__ float reached_by(uint32_t k, float mine) {
        const uint32_t key = key_of(mine);
        clear();
        if (mine > -INFINITY) {
            atomicMin(&s.low, key);
            atomicMax(&s.high, key);
        }
        __syncthreads();
        const uint32_t low = s.low, high = s.high;
        uint32_t down = 0;
        while ((high - low) >> down >= BINS) down++;
        if (mine > -INFINITY) atomicAdd((unsigned long long*)&s.hist[(high - key) >> down], 1ull);
        find_bin(0, (double)k);
        if (s.bin == BINS) return -INFINITY;
        const uint64_t far = ((uint64_t)(s.bin + 1) << down) - 1;
        uint32_t bound = far < high - low ? high - (uint32_t)far : low;
        bound = bound & 0x80000000u ? bound & 0x7fffffffu : ~bound;
        return __uint_as_float(bound);
    }
};

template <typename T, int ITS> __global__ void __launch_bounds__(BLOCK) sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const uint32_t row = blockIdx.x;
    Row<T, ITS> r(a, s, row);
    const float temperature = a.temperature ? a.temperature[row] : 1.0f, uniform = a.uniform[row];
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p_raw = a.min_p ? a.min_p[row] : 0.0f;
    r.load();
    float mine = -INFINITY;
    r.each([&](float x, uint32_t) { mine = fmaxf(mine, x); });
    r.max = r.block_max(mine);
    if (r.max == -INFINITY) {                      // nothing to choose from
        if (r.tid == 0) {
            a.tokens[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
        }
        return;
    }
    uint64_t total;
    if (r.max == INFINITY) {
        r.infinite = true;
        r.max = 0.0f;
        r.load();
        mine = -INFINITY;
        r.each([&](float x, uint32_t) { mine = fmaxf(mine, x); });
    }
    if (!(temperature > 0.0f)) {                   // greedy: the first of the largest
        uint64_t n = 0;
        auto top = [&](float x, uint32_t) -> uint64_t { return x == r.max; };
        r.each([&](float x, uint32_t i) { n += top(x, i); });
        const uint32_t token = r.search(n, false, 0.0f, 0, top, total);
        if (r.tid == 0) {
            a.tokens[row] = (int32_t)token;
            if (a.probs) a.probs[row] = 1.0f;
        }
        return;
    }
    r.step = 1.4426950408889634 / (double)temperature;
    const double min_p = min_p_raw > 0.0f ? (min_p_raw < 1.0f ? min_p_raw : 1.0f) : 0.0;
    uint64_t cut = NO_CUT;
    auto above = [&](float x, uint32_t i) -> bool { return ((uint64_t)key_of(x) << 32 | (0xffffffffu - i)) >= cut && x > -INFINITY; };
    if (k > 0 && (uint32_t)k < a.vocab) {
        const float floor = (uint32_t)k <= BLOCK ? r.reached_by((uint32_t)k, mine) : -INFINITY;
        cut = r.select((double)k, floor, [](float x, uint32_t) -> bool { return x > -INFINITY; }, [](float) -> uint64_t { return 1; });
    }
    if (top_p < 1.0f) {
        uint64_t sum = 0;
        r.each([&](float x, uint32_t i) {
            if (above(x, i)) sum += r.fixed(r.weight(x));
        });
        sum = r.block_sum(sum);
        // all of those below this weigh less than half of what may be dropped
        const float p = top_p > 0.0f ? top_p : 0.0f;
        const float floor = p > 0.0f ? r.max - temperature * 0.7f * __builtin_amdgcn_logf(2.0f * (float)a.vocab / (1.0f - p)) : r.max;
        const double want = p > 0.0f ? (double)p * (double)sum : 0.5;
        const uint64_t cut_p = r.select(want, floor, above, [&](float x) -> uint64_t { return r.fixed(r.weight(x)); });
        cut = cut_p > cut ? cut_p : cut;
    }
    auto kept = [&](float x, uint32_t i) -> uint64_t {
        if (!above(x, i)) return 0;
        const double w = r.weight(x);
        return w >= min_p ? r.fixed(w) : 0;
    };
    uint64_t sum = 0;
    r.each([&](float x, uint32_t i) { sum += kept(x, i); });
    const uint32_t token = r.search(sum, true, uniform, 0, kept, total);
    if (r.tid == 0) {
        a.tokens[row] = (int32_t)token;
        if (a.probs) a.probs[row] = (float)((double)kept(r.clean(Ar<T>::widen(((const T*)a.x)[row * a.stride + token])), token) / (double)total);
    }
}

template <typename T> int launch(rt_device* dev, const SampleArgs& a, uint32_t rows) {
    hipLaunchKernelGGL((sample_kernel<T, 0>), dim3(rows), dim3(BLOCK), 0, dev->stream, a);
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
    switch (dt) {
        case RT_F32: return launch<float>(dev, a, rows);
        case RT_F16: return launch<half_t>(dev, a, rows);
        default: return launch<bf16_t>(dev, a, rows);
    }
}
