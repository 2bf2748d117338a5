// The next tokens of a batch from its logits and given random numbers.
//
//   t = temperature, m = max x:  w_v = exp((x_v - m) / t)            in the order (x descending, index ascending):
//   top-k: the first k;  top-p: while the mass before a token is below p times that of the first k (the first always);
//   min-p: w >= min(min_p, 1).  The token is the first one, by index, at which the kept mass reached exceeds u times all of it.
//   t not above 0, or m not finite: the lowest index of the largest logit (NaN above all numbers).
//
// Weights are integers, 2^bits exp(..) rounded, so that sums do not depend on their order: a histogram's atomics and any
// split of the row give the same token.  With b = 62 - log2(vocab) bits (45 at 128000 tokens) a sum of all of them is exact in
// 64 bits, and each is off by half of 2^-b, so that borders between tokens move by at most vocab 2^-(b + 1) of the mass, which the
// largest weight alone makes 1: 1.8e-9 at 128000 tokens and 3e-5 at 2^24 where all roundings go one way, some 1e-12 where they are
// random.
//
// A row is split over workgroups and takes four launches: the largest logit; weights, their sums by workgroup and a
// histogram of counts and masses over 1/32 steps of log2 w; the mass of all tokens in steps above those where top-k or top-p end,
// and a list of the tokens in these; the end's place in that list, the workgroup's part in which the number lies, and the
// token in it.  Short rows, and rows with more than kList tokens in the steps where the filters end, are one workgroup's, which
// finds the end digit by digit of the logits' bits.  That is not for equal logits alone: flat rows have them too, as logits of
// deviation 1 and top-p 0.9 from some 128000 tokens on.  128 such rows of 128000 bfloat16 take 324 us instead of 75, of 256000 633, a
// single one of 151936 in float32 230 instead of 33.
//
// 128 rows of 128000 bfloat16 logits with all filters: 70 us, of which the largest logit takes 10.5, masses and histogram 22
// (exponentials in 64 bits), the list 23 (those of the kept tokens again), the draw 17.  Sums by granules of 512 tokens instead
// of by workgroup took the draw from 27 to 17, the list's early test and the ends read once 91 to 87 in all, gathering the kept
// tokens the list from 25 to 23.  Units read ahead and a histogram without its atomics change nothing: instructions bound
// it.  One row of 49152 is latency: four launches of 3, 5, 7 and 9 us.
#include "serving.h"

namespace flux {
namespace {

// Larger values have larger keys, NaN the largest; zeros of both signs have one.
__device__ __forceinline__ uint32_t key_of(float value) {
    const int bits = __float_as_int(value + 0.0f);
    return value != value ? ~0u : static_cast<uint32_t>(bits ^ (bits >> 31 | static_cast<int>(0x80000000u)));
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// A token's place in the order, the first ones largest; never 0.
__device__ __forceinline__ uint64_t rank_of(float value, uint32_t index) {
    return static_cast<uint64_t>(key_of(value)) << 32 | ~index;
}

// 2^(-j / 32).
__constant__ double kRoots[32] = {
    0x1.0000000000000p+0, 0x1.f50765b6e4540p-1, 0x1.ea4afa2a490dap-1, 0x1.dfc97337b9b5fp-1,
    0x1.d5818dcfba487p-1, 0x1.cb720dcef9069p-1, 0x1.c199bdd85529cp-1, 0x1.b7f76f2fb5e47p-1,
    0x1.ae89f995ad3adp-1, 0x1.a5503b23e255dp-1, 0x1.9c49182a3f090p-1, 0x1.93737b0cdc5e5p-1,
    0x1.8ace5422aa0dbp-1, 0x1.82589994cce13p-1, 0x1.7a11473eb0187p-1, 0x1.71f75e8ec5f74p-1,
    0x1.6a09e667f3bcdp-1, 0x1.6247eb03a5585p-1, 0x1.5ab07dd485429p-1, 0x1.5342b569d4f82p-1,
    0x1.4bfdad5362a27p-1, 0x1.44e086061892dp-1, 0x1.3dea64c123422p-1, 0x1.371a7373aa9cbp-1,
    0x1.306fe0a31b715p-1, 0x1.29e9df51fdee1p-1, 0x1.2387a6e756238p-1, 0x1.1d4873168b9aap-1,
    0x1.172b83c7d517bp-1, 0x1.11301d0125b51p-1, 0x1.0b5586cf9890fp-1, 0x1.059b0d3158574p-1};

// The first 32 threads': 2^(bits + j / 32) in LDS.
__device__ __forceinline__ void fill_roots(double* roots, int bits) {
    const int j = threadIdx.x;
    if (j < 32) roots[j] = ldexp(kRoots[(32 - j) & 31], j ? bits + 1 : bits);
}

// 2^bits exp((x - top) / t), rounded.  In steps of 1/32 below the largest logit, (x - top) / t log2(e) = (n + f) / 32 with
// |f| <= 1/2: 2^(n / 32) from a table of 32 (one for each bank pair of the LDS: no conflicts) and 2^(f / 32) by its
// Taylor series, whose first term left out, (ln 2 / 64)^6 / 6!, is 2^-48.7.  Rounding to integers is an addition that leaves no
// bits below them: 1.5 2^52 for n, 2^52 for the weight.
struct Weigher {
    const double* roots;  // in LDS
    double top, rate;     // rate: 32 log2(e) / t
    int none;             // step of what weighs nothing: 2^(-1 - 1/32), which is rounded to 0

    __device__ __forceinline__ Weigher(const double* table, double largest, double by, int bits)
        : roots(table), top(largest), rate(by), none(32 * (bits + 1) + 1) {}
    // -n, and f.  `none` for all beyond it, and for NaN (-inf at an infinite temperature).
    __device__ __forceinline__ int step_of(float x, double& f) const {
        const double y = __builtin_fmax((static_cast<double>(x) - top) * rate, static_cast<double>(-none));
        const double n = y + 0x1.8p52;
        f = y - (n - 0x1.8p52);
        return -static_cast<int>(__double_as_longlong(n));
    }
    __device__ __forceinline__ double series(double f) const {
        double p = 0x1.5d87fe78a6731p-35;
        p = fma(p, f, 0x1.3b2ab6fba4e77p-27);
        p = fma(p, f, 0x1.c6b08d704a0c0p-20);
        p = fma(p, f, 0x1.ebfbdff82c58fp-13);
        p = fma(p, f, 0x1.62e42fefa39efp-6);
        return fma(p, f, 1.0);
    }
    __device__ __forceinline__ double root(int step) const {  // n / 32's whole part goes to the exponent
        const int n = -step;
        const int64_t whole = static_cast<int64_t>(n >> 5) << 52;
        return __longlong_as_double(__double_as_longlong(roots[n & 31]) + whole);
    }
    __device__ __forceinline__ double power(int step, double f) const { return series(f) * root(step); }
    __device__ __forceinline__ uint64_t weight(int step, double f) const {
        return __double_as_longlong(fma(series(f), root(step), 0x1p52)) - __double_as_longlong(0x1p52);
    }
    __device__ __forceinline__ uint64_t operator()(float x) const {
        double f;
        const int step = step_of(x, f);
        return weight(step, f);
    }
};

template <int kThreads>
__device__ __forceinline__ uint64_t block_best(uint64_t v, unsigned long long* words) {
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(v), step, kWave);
        v = other > v ? other : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) words[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) v = words[w] > v ? words[w] : v;
    return v;
}

// Inclusive prefix sums over the workgroup's threads, and the total.
template <int kThreads>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, unsigned long long* words, uint64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint64_t below = __shfl_up(static_cast<unsigned long long>(v), step, kWave);
        if (lane >= step) v += below;
    }
    __syncthreads();
    if (lane == 63) words[wave] = v;
    __syncthreads();
    uint64_t all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
        if (w < wave) v += words[w];
        all += words[w];
    }
    *total = all;
    return v;
}

// Of several values a thread, each by itself.
template <int kThreads, int kValues>
__device__ __forceinline__ void block_scan(const uint64_t (&v)[kValues], unsigned long long* words, uint64_t (&reached)[kValues], uint64_t (&total)[kValues]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < kValues; ++i) reached[i] = v[i], total[i] = 0;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            const uint64_t below = __shfl_up(static_cast<unsigned long long>(reached[i]), step, kWave);
            if (lane >= step) reached[i] += below;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kValues; ++i)
        if (lane == 63) words[i * (kThreads / kWave) + wave] = reached[i];
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            const uint64_t sum = words[i * (kThreads / kWave) + w];
            if (w < wave) reached[i] += sum;
            total[i] += sum;
        }
    }
}

// What a row asks for.
struct RowOptions {
    uint32_t greedy;
    bool draws;        // not greedy
    int64_t k;         // vocab: all
    float p;           // 1: all
    uint64_t least;    // weight that min-p asks for
    double rate, top;
};

// As they are given: read while the largest logit is not known yet.
struct GivenOptions {
    float temperature, p, least;
    int64_t k;
    __device__ __forceinline__ GivenOptions(const SampleArgs& a, int64_t row) {
        temperature = a.temperature ? a.temperature[row] : 1.0f;
        k = a.top_k ? a.top_k[row] : 0;
        p = a.top_p ? a.top_p[row] : 1.0f;
        least = a.min_p ? a.min_p[row] : 0.0f;
    }
};

__device__ __forceinline__ RowOptions options_of(const SampleArgs& a, const GivenOptions& given, int bits, uint64_t best) {
    RowOptions o;
    o.greedy = ~static_cast<uint32_t>(best);
    const float top = value_of(static_cast<uint32_t>(best >> 32));
    o.draws = given.temperature > 0.0f && fabsf(top) < INFINITY;
    o.k = given.k > 0 && given.k < a.vocab ? given.k : a.vocab;
    o.p = given.p < 1.0f ? (given.p > 0.0f ? given.p : 0.0f) : 1.0f;
    const float least = given.least;
    o.least = least > 0.0f ? static_cast<uint64_t>(ceil(ldexp(static_cast<double>(least < 1.0f ? least : 1.0f), bits))) : 0;
    o.top = top;
    o.rate = 32.0 * 1.44269504088896340736 / static_cast<double>(given.temperature);
    return o;
}

// The mass before which a token is kept by top-p, at least 1: the first always is.
__device__ __forceinline__ uint64_t mass_limit(float p, uint64_t all) {
    const double mass = ceil(static_cast<double>(p) * static_cast<double>(all));
    return mass >= 1.0 ? static_cast<uint64_t>(mass) : 1;
}
// The mass that the token has to exceed.
__device__ __forceinline__ uint64_t drawn_mass(float uniform, uint64_t all) {
    const double wanted = uniform > 0.0f ? static_cast<double>(uniform) * static_cast<double>(all) : 0.0;
    return wanted < static_cast<double>(all - 1) ? static_cast<uint64_t>(wanted) : all - 1;
}

// Logits that a thread reads at once.
template <class T>
struct Unit {
    static constexpr int kWidth = 16 / sizeof(T);
    T value[kWidth];
    // Those from `v` on, -inf from `end` on.
    __device__ __forceinline__ void load(const T* row, int64_t v, int64_t end, bool wide) {
        if (wide && v + kWidth <= end) {
            const uint4 quad = *reinterpret_cast<const uint4*>(row + v);
            __builtin_memcpy(value, &quad, 16);
        } else {
#pragma unroll
            for (int j = 0; j < kWidth; ++j) value[j] = v + j < end ? row[v + j] : static_cast<T>(-INFINITY);
        }
    }
    __device__ __forceinline__ float operator[](int j) const { return static_cast<float>(value[j]); }
};

// The token of the part [from, to) of a row at which the kept mass, `before` in front of the part, exceeds `target`; kept are
// tokens ranked `end` or higher that weigh `least` or more.
template <class T, int kThreads>
__device__ void draw_in(const SampleArgs& a, int64_t row, const T* in, bool wide, int64_t from, int64_t to, const Weigher& weigh,
                        uint64_t end, uint64_t least, uint64_t before, uint64_t target, uint64_t all, unsigned long long* words) {
    using U = Unit<T>;
    constexpr int kAhead = 2;  // units of a thread that are read and summed at once
    uint64_t running = before;
    for (int64_t base = from; base < to; base += kAhead * kThreads * U::kWidth) {
        U units[kAhead];
        uint64_t sums[kAhead], totals[kAhead];
        auto weight_of = [&](float x, int64_t v) -> uint64_t {
            const uint64_t w = v < to && rank_of(x, static_cast<uint32_t>(v)) >= end ? weigh(x) : 0;
            return w < least ? 0 : w;
        };
        auto at = [&](int i) { return base + U::kWidth * (i * kThreads + static_cast<int>(threadIdx.x)); };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) units[i].load(in, at(i), to, wide);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            sums[i] = 0;
            if (at(i) < to) {
#pragma unroll
                for (int j = 0; j < U::kWidth; ++j) sums[i] += weight_of(units[i][j], at(i) + j);
            }
        }
        uint64_t reached[kAhead];
        block_scan<kThreads>(sums, words, reached, totals);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            uint64_t sum = running + reached[i] - sums[i];
            if (sum <= target && sum + sums[i] > target) {
#pragma unroll
                for (int j = 0; j < U::kWidth; ++j) {
                    const float x = units[i][j];
                    const uint64_t w = weight_of(x, at(i) + j);
                    if (sum <= target && sum + w > target) {
                        double f;
                        const int step = weigh.step_of(x, f);
                        a.tokens[row] = at(i) + j;
                        a.probabilities[row] = static_cast<float>(weigh.power(step, f) / static_cast<double>(all));
                    }
                    sum += w;
                }
            }
            running += totals[i];
        }
        if (running > target) return;
    }
}

// ---------------------------------------------------------------------------
// One workgroup a row.
constexpr int kRowThreads = 1024;
constexpr int kDigitBins = 2048;

struct DigitShared {
    unsigned long long mass[kDigitBins];
    uint32_t count[kDigitBins];
    unsigned long long words[2 * kRowThreads / kWave];
    unsigned long long word, above;
    uint32_t index;
    double roots[32];
};

// The last token kept, where the count reaches `limit` (kCount) or the mass does: eleven, eleven and ten bits of the keys in
// turn, then the equal logits by index.  `mass`: of all kept.
template <bool kCount, class T, int kThreads>
__device__ uint64_t find_end(const T* row, int64_t vocab, bool wide, const Weigher& weigh, uint64_t limit, DigitShared& s, uint64_t* mass) {
    using U = Unit<T>;
    uint32_t prefix = 0;
    uint64_t above_count = 0, above_mass = 0, last_count = 0, last_mass = 0;
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : (digit == 1 ? 10 : 0), bins = digit == 2 ? 1024 : 2048;
        const int fixed = digit == 0 ? 32 : (digit == 1 ? 21 : 10);
        __syncthreads();
        for (int b = threadIdx.x; b < kDigitBins; b += kThreads) s.mass[b] = 0, s.count[b] = 0;
        if (threadIdx.x == 0) s.index = 0;  // a bin, also when the logits change during the call
        __syncthreads();
        for (int64_t v = U::kWidth * static_cast<int>(threadIdx.x); v < vocab; v += U::kWidth * kThreads) {
            U unit;
            unit.load(row, v, vocab, wide);
#pragma unroll
            for (int j = 0; j < U::kWidth; ++j) {
                const uint32_t key = key_of(unit[j]);
                if (v + j >= vocab || (fixed < 32 && (key ^ prefix) >> fixed)) continue;
                const uint32_t bin = key >> shift & (bins - 1);
                atomicAdd(s.count + bin, 1u);
                const uint64_t w = weigh(unit[j]);
                if (w) atomicAdd(s.mass + bin, static_cast<unsigned long long>(w));
            }
        }
        __syncthreads();
        // Each thread looks at some bins, the first one at the highest.
        constexpr int kEach = kDigitBins / kThreads;
        const int high = bins - 1 - kEach * static_cast<int>(threadIdx.x);
        uint64_t counts = 0, masses = 0;
        for (int j = 0; j < kEach && high - j >= 0; ++j) counts += s.count[high - j], masses += s.mass[high - j];
        uint64_t total;
        uint64_t count_before = above_count + block_scan<kThreads>(counts, s.words, &total) - counts;
        uint64_t mass_before = above_mass + block_scan<kThreads>(masses, s.words, &total) - masses;
        for (int j = 0; j < kEach && high - j >= 0; ++j) {
            const uint64_t c = s.count[high - j], m = s.mass[high - j];
            const uint64_t reached = kCount ? count_before : mass_before, added = kCount ? c : m;
            if (reached < limit && reached + added >= limit) {
                s.index = high - j;
                s.word = mass_before;
                s.above = count_before;
            }
            count_before += c;
            mass_before += m;
        }
        __syncthreads();
        const int bin = s.index;
        above_mass = s.word;
        above_count = s.above;
        last_count = s.count[bin];
        last_mass = s.mass[bin];
        prefix |= static_cast<uint32_t>(bin) << shift;
    }
    const uint64_t each = last_mass / last_count;  // they are equal
    const uint64_t ties = kCount ? limit - above_count : (limit - 1 - above_mass) / each + 1;
    *mass = above_mass + each * ties;
    if (ties >= last_count) return static_cast<uint64_t>(prefix) << 32;
    uint64_t found = 0;  // the index of the last of the equal ones that is kept
    for (int64_t base = 0; base < vocab && found < ties; base += U::kWidth * kThreads) {
        const int64_t v = base + U::kWidth * static_cast<int>(threadIdx.x);
        U unit;
        unit.load(row, v, vocab, wide);
        uint64_t mine = 0;
#pragma unroll
        for (int j = 0; j < U::kWidth; ++j) mine += v + j < vocab && key_of(unit[j]) == prefix;
        uint64_t total;
        uint64_t before = found + block_scan<kThreads>(mine, s.words, &total) - mine;
#pragma unroll
        for (int j = 0; j < U::kWidth; ++j)
            if (v + j < vocab && key_of(unit[j]) == prefix && ++before == ties) s.index = static_cast<uint32_t>(v + j);
        found += total;
    }
    __syncthreads();
    return static_cast<uint64_t>(prefix) << 32 | ~s.index;
}

template <class T, int kThreads>
__device__ void sample_row(const SampleArgs& a, int64_t row, const RowOptions& o, int bits, bool wide, DigitShared& s) {
    using U = Unit<T>;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const Weigher weigh(s.roots, o.top, o.rate, bits);
    uint64_t end = 0, mass = 0;
    if (o.k < a.vocab) end = find_end<true, T, kThreads>(in, a.vocab, wide, weigh, o.k, s, &mass);
    if (mass == 0) {
        uint64_t sum = 0;
        for (int64_t v = U::kWidth * static_cast<int>(threadIdx.x); v < a.vocab; v += U::kWidth * kThreads) {
            U unit;
            unit.load(in, v, a.vocab, wide);
#pragma unroll
            for (int j = 0; j < U::kWidth; ++j) sum += weigh(unit[j]);
        }
        block_scan<kThreads>(sum, s.words, &mass);
    }
    if (o.p < 1.0f) end = find_end<false, T, kThreads>(in, a.vocab, wide, weigh, mass_limit(o.p, mass), s, &mass);
    if (o.least > 0) {
        uint64_t sum = 0;
        for (int64_t v = U::kWidth * static_cast<int>(threadIdx.x); v < a.vocab; v += U::kWidth * kThreads) {
            U unit;
            unit.load(in, v, a.vocab, wide);
#pragma unroll
            for (int j = 0; j < U::kWidth; ++j) {
                const uint64_t w = rank_of(unit[j], static_cast<uint32_t>(v + j)) >= end && v + j < a.vocab ? weigh(unit[j]) : 0;
                sum += w < o.least ? 0 : w;
            }
        }
        block_scan<kThreads>(sum, s.words, &mass);
    }
    draw_in<T, kThreads>(a, row, in, wide, 0, a.vocab, weigh, end, o.least, 0, drawn_mass(a.uniforms[row], mass), mass, s.words);
}

template <class T>
__global__ void __launch_bounds__(kRowThreads) sample_row_kernel(SampleArgs a, int bits, bool wide) {
    using U = Unit<T>;
    __shared__ DigitShared s;
    const int64_t row = blockIdx.x;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    fill_roots(s.roots, bits);
    const GivenOptions given(a, row);
    uint64_t best = 0;
    for (int64_t v = U::kWidth * static_cast<int>(threadIdx.x); v < a.vocab; v += U::kWidth * kRowThreads) {
        U unit;
        unit.load(in, v, a.vocab, wide);
#pragma unroll
        for (int j = 0; j < U::kWidth; ++j) {
            const uint64_t rank = rank_of(unit[j], static_cast<uint32_t>(v + j));
            best = v + j < a.vocab && rank > best ? rank : best;
        }
    }
    best = block_best<kRowThreads>(best, s.words);
    const RowOptions o = options_of(a, given, bits, best);
    if (!o.draws) {
        if (threadIdx.x == 0) a.tokens[row] = o.greedy, a.probabilities[row] = 1.0f;
        return;
    }
    sample_row<T, kRowThreads>(a, row, o, bits, wide, s);
}

// ---------------------------------------------------------------------------
// Several workgroups a row.
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / kWave;
constexpr int kSteps = 1600;  // more than those of weights that are not 0, 32 (bits + 1): rows of this kind have at most 48 bits
constexpr int kList = 1024;   // tokens in the steps where top-k and top-p end
constexpr int kMostParts = 64;
constexpr int kGranules = 2048;

struct SampleSplit {
    int parts;       // of a row
    int64_t part;    // tokens
    int units;       // a wave's in a row: a granule, of 64 units' tokens each
    int granules;    // of a row, at most kGranules
    int part_granules;
    unsigned long long* best;    // [rows, parts]
    unsigned long long* mass;    // [rows, granules]
    unsigned long long* masses;  // [rows, kSteps]
    unsigned long long* list;    // [rows, kList] ranks
    struct Ends* ends;           // [rows]
    uint32_t* counts;            // [rows, kSteps]
    uint32_t* listed;            // [rows]
};

// Where the kept tokens of a row end, as far as its histogram tells: steps below `sure` are kept, the end is in the list, that
// is the steps [sure, last] and `by_count`, in which the k-th token is.  kSteps: none.
struct Ends {
    int sure, last, by_count;
    uint64_t count_before, mass_before;  // of the step by_count
    uint64_t mass_sure;  // of the steps below `sure`
    uint64_t mass_all;
};

// All parts of a row on one XCD (block index modulo 8), whose L2 then holds the row and its histogram.
__device__ __forceinline__ bool place_of(const SampleArgs& a, const SampleSplit& s, int64_t& row, int& part) {
    const uint32_t j = blockIdx.x / 8;
    row = static_cast<int64_t>(j / s.parts) * 8 + blockIdx.x % 8;
    part = j % s.parts;
    return row < a.rows;
}

// A part's tokens, by each wave in granules: `each` has a unit and its first token, `all` the granule's number and the sum
// of what `each` returned.
template <class T, class Each, class All>
__device__ __forceinline__ void walk(const SampleArgs& a, const SampleSplit& s, int64_t row, int part, bool wide, Each each, All all) {
    using U = Unit<T>;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const int64_t granule = static_cast<int64_t>(s.units) * kWave * U::kWidth;
    const int64_t from = part * s.part, to = from + s.part < a.vocab ? from + s.part : a.vocab;
    const int lane = threadIdx.x & 63;
    int number = part * s.part_granules + (threadIdx.x >> 6);
    for (int64_t start = from + (threadIdx.x >> 6) * granule; start < to; start += kWaves * granule, number += kWaves) {
        uint64_t sum = 0;
        for (int u = 0; u < s.units; ++u) {
            const int64_t v = start + (u * kWave + lane) * U::kWidth;
            U unit;
            unit.load(in, v, to, wide);
            sum += each(unit, v);
        }
        all(number, sum);
    }
}
__device__ __forceinline__ uint64_t wave_sum_of(uint64_t v) {
#pragma unroll
    for (int step = 1; step < 64; step *= 2) v += __shfl_xor(static_cast<unsigned long long>(v), step, kWave);
    return v;
}

template <class T>
__global__ void __launch_bounds__(kThreads) sample_best_kernel(SampleArgs a, SampleSplit s, bool wide) {
    using U = Unit<T>;
    __shared__ unsigned long long words[kWaves];
    int64_t row;
    int part;
    if (!place_of(a, s, row, part)) return;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const int64_t from = part * s.part, to = from + s.part < a.vocab ? from + s.part : a.vocab;
    uint64_t best = 0;
#pragma unroll 4
    for (int64_t v = from + U::kWidth * static_cast<int>(threadIdx.x); v < to; v += U::kWidth * kThreads) {
        U unit;
        unit.load(in, v, to, wide);
#pragma unroll
        for (int j = 0; j < U::kWidth; ++j) {
            const uint64_t rank = rank_of(unit[j], static_cast<uint32_t>(v + j));
            best = v + j < to && rank > best ? rank : best;
        }
    }
    best = block_best<kThreads>(best, words);
    if (threadIdx.x == 0) s.best[row * s.parts + part] = best;
    for (int b = part * kThreads + threadIdx.x; b < kSteps; b += s.parts * kThreads)
        s.masses[row * kSteps + b] = 0, s.counts[row * kSteps + b] = 0;
    if (part == 0 && threadIdx.x == 0) s.listed[row] = 0;
}

__device__ __forceinline__ RowOptions row_options(const SampleArgs& a, const SampleSplit& s, int64_t row, int bits, unsigned long long* words) {
    const GivenOptions given(a, row);
    uint64_t best = threadIdx.x < static_cast<uint32_t>(s.parts) ? s.best[row * s.parts + threadIdx.x] : 0;  // at most kMostParts
    return options_of(a, given, bits, block_best<kThreads>(best, words));
}

template <class T>
__global__ void __launch_bounds__(kThreads) sample_mass_kernel(SampleArgs a, SampleSplit s, int bits, bool wide) {
    using U = Unit<T>;
    __shared__ unsigned long long words[kWaves];
    __shared__ double roots[32];
    __shared__ unsigned long long masses[kSteps];
    __shared__ uint32_t counts[kSteps];
    int64_t row;
    int part;
    if (!place_of(a, s, row, part)) return;
    fill_roots(roots, bits);
    const RowOptions o = row_options(a, s, row, bits, words);
    if (!o.draws) {
        if (part == 0 && threadIdx.x == 0) a.tokens[row] = o.greedy, a.probabilities[row] = 1.0f;
        return;
    }
    const bool by_count = o.k < a.vocab, by_mass = o.p < 1.0f, filtered = by_count || by_mass;
    if (filtered) {
        for (int b = threadIdx.x; b < kSteps; b += kThreads) masses[b] = 0, counts[b] = 0;
        __syncthreads();
    }
    const Weigher weigh(roots, o.top, o.rate, bits);
    if (!filtered) {
        __syncthreads();
        walk<T>(a, s, row, part, wide, [&](const U& unit, int64_t) {
            uint64_t sum = 0;
#pragma unroll
            for (int j = 0; j < U::kWidth; ++j) {
                const uint64_t w = weigh(unit[j]);
                sum += w < o.least ? 0 : w;
            }
            return sum;
        }, [&](int granule, uint64_t sum) {
            sum = wave_sum_of(sum);
            if ((threadIdx.x & 63) == 0) s.mass[row * s.granules + granule] = sum;
        });
        return;
    }
    walk<T>(a, s, row, part, wide, [&](const U& unit, int64_t) -> uint64_t {
#pragma unroll
        for (int j = 0; j < U::kWidth; ++j) {
            double f;
            const int step = weigh.step_of(unit[j], f);
            if (step >= weigh.none) continue;
            if (by_count) atomicAdd(counts + step, 1u);
            if (by_mass) atomicAdd(masses + step, static_cast<unsigned long long>(weigh.weight(step, f)));
        }
        return 0;
    }, [](int, uint64_t) {});
    __syncthreads();
    for (int b = threadIdx.x; b < kSteps; b += kThreads) {
        if (counts[b]) atomicAdd(s.counts + row * kSteps + b, counts[b]);
        if (masses[b]) atomicAdd(s.masses + row * kSteps + b, masses[b]);
    }
}

struct EndsShared {
    unsigned long long words[2 * kWaves];
    int step;
    unsigned long long count, mass, own_mass;
};

// A thread's steps of the row's histogram.
constexpr int kStepsEach = (kSteps + kThreads - 1) / kThreads;
struct ThreadSteps {
    uint64_t mass[kStepsEach];
    uint32_t count[kStepsEach];
    __device__ __forceinline__ ThreadSteps(const SampleSplit& s, int64_t row) {
#pragma unroll
        for (int j = 0; j < kStepsEach; ++j) {
            const int b = kStepsEach * static_cast<int>(threadIdx.x) + j;
            mass[j] = b < kSteps ? s.masses[row * kSteps + b] : 0;
            count[j] = b < kSteps ? s.counts[row * kSteps + b] : 0;
        }
    }
};

__device__ Ends ends_of(const ThreadSteps& steps, const RowOptions& o, int64_t vocab, EndsShared& shared) {
    const int b0 = kStepsEach * threadIdx.x;
    const uint64_t(&mass)[kStepsEach] = steps.mass;
    uint64_t count[kStepsEach], sums[2] = {0, 0}, before[2], all[2];
#pragma unroll
    for (int j = 0; j < kStepsEach; ++j) {
        count[j] = steps.count[j];
        sums[0] += mass[j];
        sums[1] += count[j];
    }
    block_scan<kThreads>(sums, shared.words, before, all);
    const uint64_t all_mass = all[0], all_count = all[1], mass_before = before[0] - sums[0], count_before = before[1] - sums[1];
    // The first step at which the sum reaches the limit.
    auto reach = [&](uint64_t limit, uint64_t before, const uint64_t (&added)[kStepsEach]) {
        __syncthreads();
        if (threadIdx.x == 0) shared.step = kSteps;
        __syncthreads();
        uint64_t mass_at = mass_before, at = before;
#pragma unroll
        for (int j = 0; j < kStepsEach; ++j) {
            if (at < limit && at + added[j] >= limit)
                shared.step = b0 + j, shared.count = at, shared.mass = mass_at, shared.own_mass = mass[j];
            at += added[j];
            mass_at += mass[j];
        }
        __syncthreads();
        return shared.step;
    };
    Ends e{kSteps, kSteps, kSteps, 0, 0, all_mass, all_mass};
    uint64_t low = all_mass, high = all_mass;
    if (o.k < vocab && all_count >= static_cast<uint64_t>(o.k)) {
        e.by_count = reach(o.k, count_before, count);
        e.count_before = shared.count;
        e.mass_before = e.mass_sure = shared.mass;
        e.sure = e.last = e.by_count;
        low = e.mass_before;
        high = e.by_count < kSteps ? e.mass_before + shared.own_mass : all_mass;
    }
    if (o.p < 1.0f) {
        e.last = reach(mass_limit(o.p, high), mass_before, mass);
        e.sure = reach(mass_limit(o.p, low), mass_before, mass);
        e.mass_sure = shared.mass;
    }
    return e;
}

template <class T>
__global__ void __launch_bounds__(kThreads) sample_list_kernel(SampleArgs a, SampleSplit s, int bits, bool wide) {
    using U = Unit<T>;
    __shared__ EndsShared shared;
    __shared__ double roots[32];
    __shared__ unsigned long long found[kList], gathered[kWaves][kWave * U::kWidth];
    __shared__ uint32_t count, first;
    int64_t row;
    int part;
    if (!place_of(a, s, row, part)) return;
    fill_roots(roots, bits);
    const ThreadSteps steps(s, row);
    const RowOptions o = row_options(a, s, row, bits, shared.words);
    if (!o.draws || (o.k >= a.vocab && o.p >= 1.0f)) return;
    const Ends e = ends_of(steps, o, a.vocab, shared);
    if (threadIdx.x == 0 && part == 0) s.ends[row] = e;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const Weigher weigh(roots, o.top, o.rate, bits);
    // Most logits are far below the ends.  Their step to three roundings of 2^-24, of halves whose difference does not overflow, or
    // an earlier one where the rate is beyond float32's, is off by less than 2^-10 of a step: what lies a whole step behind the
    // last is left out by it.
    const int last = e.by_count < kSteps && e.by_count > e.last ? e.by_count : e.last;
    const float top = 0.5f * static_cast<float>(o.top), rate = 2.0f * (o.rate < 0x1p126 ? static_cast<float>(o.rate) : 0x1p126f);
    const float far = -static_cast<float>(last + 1);
    // The others of a wave's unit are gathered, so that a few of them do not take all lanes through the exponential.
    unsigned long long* near = gathered[threadIdx.x >> 6];
    const int lane = threadIdx.x & 63;
    walk<T>(a, s, row, part, wide, [&](const U& unit, int64_t v) {
        int held = 0;
#pragma unroll
        for (int j = 0; j < U::kWidth; ++j) {
            const bool is_near = !((0.5f * unit[j] - top) * rate < far);
            const uint64_t lanes = __ballot(is_near);
            if (is_near) near[held + __popcll(lanes & ((uint64_t{1} << lane) - 1))] = rank_of(unit[j], static_cast<uint32_t>(v + j));
            held += __popcll(lanes);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint64_t sum = 0;
        for (int i = lane; i < held; i += kWave) {
            const uint64_t rank = near[i];
            double f;
            const int step = weigh.step_of(value_of(static_cast<uint32_t>(rank >> 32)), f);
            if (step < e.sure) {
                const uint64_t w = weigh.weight(step, f);
                sum += w < o.least ? 0 : w;
            } else if (step < weigh.none && (step <= e.last || step == e.by_count)) {
                const uint32_t at = atomicAdd(&count, 1u);
                if (at < kList) found[at] = rank;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        return sum;
    }, [&](int granule, uint64_t sum) {
        sum = wave_sum_of(sum);
        if ((threadIdx.x & 63) == 0) s.mass[row * s.granules + granule] = sum;
    });
    __syncthreads();
    if (threadIdx.x == 0) first = count ? atomicAdd(s.listed + row, count) : 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count && i < kList; i += kThreads)
        if (first + i < kList) s.list[row * kList + first + i] = found[i];
}

struct DrawShared {
    unsigned long long sorted[kList];
    unsigned long long mass[kGranules];
    unsigned long long end, before;
    int index;
};

template <class T>
__global__ void __launch_bounds__(kThreads) sample_draw_kernel(SampleArgs a, SampleSplit s, int bits, bool wide) {
    __shared__ union {
        DrawShared draw;
        DigitShared digits;
    } u;
    __shared__ EndsShared shared;
    __shared__ double roots[32];
    const int64_t row = blockIdx.x;
    fill_roots(roots, bits);
    const RowOptions o = row_options(a, s, row, bits, shared.words);
    if (!o.draws) return;
    const Weigher weigh(roots, o.top, o.rate, bits);
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    DrawShared& d = u.draw;
    const int64_t granule = static_cast<int64_t>(s.units) * kWave * Unit<T>::kWidth;
    constexpr int kGranulesEach = kGranules / kThreads;
#pragma unroll
    for (int i = 0; i < kGranulesEach; ++i) {
        const int g = i * kThreads + static_cast<int>(threadIdx.x);
        d.mass[g] = g < s.granules ? s.mass[row * s.granules + g] : 0;
    }
    uint64_t end = 0;
    if (o.k < a.vocab || o.p < 1.0f) {
        const uint32_t listed = s.listed[row];
        if (listed > kList) {
            __syncthreads();
            fill_roots(u.digits.roots, bits);
            __syncthreads();
            sample_row<T, kThreads>(a, row, o, bits, wide, u.digits);
            return;
        }
        const Ends e = s.ends[row];
        // In their order, by a bitonic network; a rank is never 0, which fills the list up to a power of two.
        uint32_t places = 2;
        while (places < listed) places *= 2;
        for (uint32_t i = threadIdx.x; i < places; i += kThreads) d.sorted[i] = i < listed ? s.list[row * kList + i] : 0;
        if (threadIdx.x == 0) d.end = ~0ull;
        __syncthreads();
        for (uint32_t run = 2; run <= places; run *= 2) {
            for (uint32_t apart = run / 2; apart > 0; apart /= 2) {
                const uint32_t i = 2 * threadIdx.x - (threadIdx.x & (apart - 1));  // one pair a thread
                if (i < places) {
                    const uint64_t x = d.sorted[i], y = d.sorted[i + apart];
                    if ((x < y) == ((i & run) == 0)) d.sorted[i] = y, d.sorted[i + apart] = x;
                }
                __syncthreads();
            }
        }
        constexpr int kEach = kList / kThreads;
        const uint32_t i0 = kEach * threadIdx.x;
        uint64_t w[kEach], sum = 0, counted = 0, below = 0;
        bool of_count[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            w[j] = 0;
            of_count[j] = false;
            if (i0 + j < listed) {
                double f;
                const int step = weigh.step_of(value_of(static_cast<uint32_t>(d.sorted[i0 + j] >> 32)), f);
                w[j] = weigh.weight(step, f);
                of_count[j] = step == e.by_count;
                below += step < e.by_count;
            }
            sum += w[j];
        }
        uint64_t first_of_count, total;
        block_scan<kThreads>(below, shared.words, &first_of_count);
        // The mass of the first k: the step by_count's tokens up to the k-th one.
        const uint64_t kept_of_count = e.by_count < kSteps ? o.k - e.count_before : 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (of_count[j] && i0 + j < first_of_count + kept_of_count) counted += w[j];
        block_scan<kThreads>(counted, shared.words, &total);
        const uint64_t first_k = e.by_count < kSteps ? e.mass_before + total : e.mass_all;
        const uint64_t limit = o.p < 1.0f ? mass_limit(o.p, first_k) : ~uint64_t{0};
        // Kept of the list: up to the k-th token, and while the mass before is below the limit.  Between the steps [sure, last]
        // and by_count others are left out of the list: what follows them is beyond the limit.
        uint64_t reached = e.mass_sure + block_scan<kThreads>(sum, shared.words, &total) - sum;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const bool kept = i0 + j < listed && reached < limit && (!of_count[j] || i0 + j < first_of_count + kept_of_count);
            if (kept) {
                const uint32_t index = ~static_cast<uint32_t>(d.sorted[i0 + j]);
                if (w[j] >= o.least) atomicAdd(d.mass + index / static_cast<uint32_t>(granule), static_cast<unsigned long long>(w[j]));
            }
            const uint64_t lanes = __ballot(kept);
            if (lanes && (threadIdx.x & 63) == 63 - static_cast<uint32_t>(__builtin_clzll(lanes))) atomicMin(&d.end, d.sorted[i0 + j]);  // the wave's last
            reached += w[j];
        }
        __syncthreads();
        if (listed) end = d.end;
    }
    __syncthreads();
    uint64_t all, mass[kGranulesEach], masses = 0;
#pragma unroll
    for (int i = 0; i < kGranulesEach; ++i) masses += mass[i] = d.mass[kGranulesEach * threadIdx.x + i];
    uint64_t before = block_scan<kThreads>(masses, shared.words, &all) - masses;
    const uint64_t target = drawn_mass(a.uniforms[row], all);
    if (threadIdx.x == 0) d.index = 0, d.before = 0;  // a granule of the row, also when the logits change during the call
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kGranulesEach; ++i) {
        if (mass[i] && before <= target && before + mass[i] > target) d.index = kGranulesEach * threadIdx.x + i, d.before = before;
        before += mass[i];
    }
    __syncthreads();
    const int64_t from = d.index * granule, to = from + granule < a.vocab ? from + granule : a.vocab;
    draw_in<T, kThreads>(a, row, in, wide, from, to, weigh, end, o.least, d.before, target, all, shared.words);
}

// Rows up to this many tokens are one workgroup's.
constexpr int64_t kShortRow = 8192;
// About four workgroups a CU, and parts of whole granules for every wave.
SampleSplit split_of(int64_t rows, int64_t vocab, int size, void* workspace, size_t* bytes) {
    SampleSplit s{};
    const int64_t unit = kWave * 16 / size;  // tokens that a wave reads at once
    s.units = 1;
    while ((vocab + s.units * unit - 1) / (s.units * unit) > kGranules) s.units *= 2;
    const int64_t granule = s.units * unit, step = kWaves * granule;
    int64_t parts = (1024 + rows - 1) / rows;
    if (parts > kMostParts) parts = kMostParts;
    s.part = ((vocab + parts - 1) / parts + step - 1) / step * step;
    s.parts = static_cast<int>((vocab + s.part - 1) / s.part);
    s.part_granules = static_cast<int>(s.part / granule);
    s.granules = static_cast<int>((vocab + granule - 1) / granule);
    auto* at = static_cast<unsigned long long*>(workspace);
    s.best = at;
    s.mass = s.best + rows * s.parts;
    s.masses = s.mass + rows * s.granules;
    s.list = s.masses + rows * kSteps;
    s.ends = reinterpret_cast<Ends*>(s.list + rows * kList);
    s.counts = reinterpret_cast<uint32_t*>(s.ends + rows);
    s.listed = s.counts + rows * kSteps;
    *bytes = static_cast<size_t>(rows) * (8 * s.parts + 8 * s.granules + 8 * kSteps + 8 * kList + sizeof(Ends) + 4 * kSteps) + static_cast<size_t>(rows + rows % 2) * 4;
    return s;
}

template <class T>
hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
    int bits = 51;
    while (a.vocab > (int64_t{1} << (62 - bits))) --bits;  // not the vocabulary shifted, which does not fit
    const bool wide = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.logits_stride * sizeof(T) % 16 == 0;
    const auto rows = static_cast<uint32_t>(a.rows);
    if (a.vocab <= kShortRow) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(sample_row_kernel<T>), dim3(rows), dim3(kRowThreads), 0, stream, a, bits, wide);
        return hipGetLastError();
    }
    size_t bytes = 0;
    const SampleSplit s = split_of(a.rows, a.vocab, sizeof(T), a.workspace, &bytes);
    const dim3 grid((rows + 7) / 8 * 8 * static_cast<uint32_t>(s.parts));
    hipLaunchKernelGGL(HIP_KERNEL_NAME(sample_best_kernel<T>), grid, dim3(kThreads), 0, stream, a, s, wide);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(sample_mass_kernel<T>), grid, dim3(kThreads), 0, stream, a, s, bits, wide);
    if (a.top_k || a.top_p) hipLaunchKernelGGL(HIP_KERNEL_NAME(sample_list_kernel<T>), grid, dim3(kThreads), 0, stream, a, s, bits, wide);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(sample_draw_kernel<T>), dim3(rows), dim3(kThreads), 0, stream, a, s, bits, wide);
    return hipGetLastError();
}

}  // namespace

size_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
    if (vocab <= kShortRow) return 0;
    size_t bytes = 0;
    split_of(rows, vocab, 4, nullptr, &bytes);  // float32 has the most granules
    return bytes;
}

hipError_t launch_logits_sample(const SampleArgs& args, Type type, hipStream_t stream) {
    switch (type) {
        case Type::kFloat32: return launch_sample<float>(args, stream);
        case Type::kFloat16: return launch_sample<_Float16>(args, stream);
        default: return launch_sample<__bf16>(args, stream);
    }
}

}  // namespace flux
