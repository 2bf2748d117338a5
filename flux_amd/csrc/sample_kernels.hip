// The next tokens of a batch from its logits and given random numbers.
//
//   t = temperature, m = max x:  w_v = exp((x_v - m) / t)            in the order (x descending, index ascending):
//   top-k: the first k;  top-p: while the mass before a token is below p times that of the first k (the first always);
//   min-p: w >= min(min_p, 1).  The token is the first one, by index, at which the kept mass reached exceeds u times all of it.
//   t not above 0, or m not finite: the lowest index of the largest logit (NaN above all numbers).
//
// Weights are integers, 2^kBits exp(..) rounded, so that sums do not depend on their order: a histogram's atomics and any
// split of the row give the same token.  With 62 - log2(vocab) bits (45 at 128000 tokens) a sum of all of them is exact in
// 64 bits, and each is off by half of 2^-45: borders between tokens move by less than 1e-11 of the mass.
#include "serving.h"

namespace flux {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;

// Larger values have larger keys, NaN the largest; zeros of both signs have one.
__device__ __forceinline__ uint32_t key_of(float value) {
    const int bits = __float_as_int(value + 0.0f);
    return value != value ? ~0u : static_cast<uint32_t>(bits ^ (bits >> 31 | static_cast<int>(0x80000000u)));
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// 2^bits exp2((x - top) rate), rounded; rate = log2(e) / temperature.  2^f for |f| <= 1/2 by its Taylor series: the first
// term left out, (ln 2 / 2)^13 / 13!, is below 2^-52.
struct Weigher {
    double top, rate;
    int bits;

    __device__ __forceinline__ double exponent(float x) const { return (static_cast<double>(x) - top) * rate; }
    __device__ __forceinline__ double power(double y) const {
        const double n = __builtin_rint(y);
        const double f = (y - n) * 0.69314718055994530942;
        double p = 1.0 / 479001600.0;
        p = fma(p, f, 1.0 / 39916800.0);
        p = fma(p, f, 1.0 / 3628800.0);
        p = fma(p, f, 1.0 / 362880.0);
        p = fma(p, f, 1.0 / 40320.0);
        p = fma(p, f, 1.0 / 5040.0);
        p = fma(p, f, 1.0 / 720.0);
        p = fma(p, f, 1.0 / 120.0);
        p = fma(p, f, 1.0 / 24.0);
        p = fma(p, f, 1.0 / 6.0);
        p = fma(p, f, 0.5);
        p = fma(p, f, 1.0);
        p = fma(p, f, 1.0);
        return __builtin_amdgcn_ldexp(p, static_cast<int>(n) + bits);
    }
    // An integer below 2^52 by the addition of 2^52; NaN (an infinite temperature's -inf) weighs nothing.
    __device__ __forceinline__ uint64_t operator()(float x) const {
        const double y = exponent(x);
        if (!(y >= -(bits + 1))) return 0;
        return __double_as_longlong(power(y) + 0x1p52) - __double_as_longlong(0x1p52);
    }
};

struct Shared {
    unsigned long long mass[kBins];
    uint32_t count[kBins];
    unsigned long long sums[kWaves];
    unsigned long long word, above;
    uint32_t index;
};

__device__ __forceinline__ uint64_t shuffle_up(uint64_t v, int by) {
    return static_cast<uint64_t>(__shfl_up(static_cast<unsigned long long>(v), by, kWave));
}

// Inclusive prefix sums over the workgroup's threads, and the total.
__device__ uint64_t block_scan(uint64_t v, unsigned long long* sums, uint64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint64_t below = shuffle_up(v, step);
        if (lane >= step) v += below;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    uint64_t all = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) v += sums[w];
        all += sums[w];
    }
    *total = all;
    return v;
}

// The end of the kept tokens in the order: those with keys above `key`, and the first `ties` of those with it.
struct End {
    uint32_t key;
    uint32_t ties;
    uint64_t mass;  // of all kept
};

// The token where the count reaches `limit` (kCount) or the mass does: eleven, eleven and ten bits of its key in turn.
template <bool kCount, class T>
__device__ End find_end(const T* row, int64_t vocab, const Weigher& weigh, uint64_t limit, Shared& s) {
    uint32_t prefix = 0;
    uint64_t above_count = 0, above_mass = 0;
    uint64_t last_count = 0, last_mass = 0;
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : (digit == 1 ? 10 : 0), bins = digit == 2 ? 1024 : 2048;
        const int fixed = digit == 0 ? 32 : (digit == 1 ? 21 : 10);
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += kThreads) s.mass[b] = 0, s.count[b] = 0;
        __syncthreads();
        for (int64_t v = threadIdx.x; v < vocab; v += kThreads) {
            const float x = static_cast<float>(row[v]);
            const uint32_t key = key_of(x);
            if (fixed < 32 && (key ^ prefix) >> fixed) continue;
            const uint32_t bin = key >> shift & (bins - 1);
            atomicAdd(s.count + bin, 1u);
            const uint64_t w = weigh(x);
            if (w) atomicAdd(s.mass + bin, static_cast<unsigned long long>(w));
        }
        __syncthreads();
        // Thread t looks at the bins from the highest on: 2 t and 2 t + 1 below it.
        const int high = bins - 1 - 2 * static_cast<int>(threadIdx.x), low = high - 1;
        const bool mine = high >= 0;
        const uint64_t c0 = mine ? s.count[high] : 0, c1 = mine && low >= 0 ? s.count[low] : 0;
        const uint64_t m0 = mine ? s.mass[high] : 0, m1 = mine && low >= 0 ? s.mass[low] : 0;
        uint64_t total;
        const uint64_t counts = above_count + block_scan(c0 + c1, s.sums, &total);
        const uint64_t masses = above_mass + block_scan(m0 + m1, s.sums, &total);
        const uint64_t reached = kCount ? counts : masses, added = kCount ? c0 + c1 : m0 + m1, first = kCount ? c0 : m0;
        if (reached >= limit && reached - added < limit) {
            s.index = reached - added + first >= limit ? high : low;
            s.word = masses - m0 - m1;
            s.above = counts - c0 - c1;
        }
        __syncthreads();
        const int bin = s.index;
        above_mass = s.word;
        above_count = s.above;
        const int of = bins - 1 - bin;
        if (of & 1) above_mass += s.mass[bin + 1], above_count += s.count[bin + 1];
        last_count = s.count[bin];
        last_mass = s.mass[bin];
        prefix |= static_cast<uint32_t>(bin) << shift;
    }
    __syncthreads();
    End end;
    end.key = prefix;
    const uint64_t each = last_count ? last_mass / last_count : 0;  // they are equal
    end.ties = static_cast<uint32_t>(kCount ? limit - above_count : (limit - 1 - above_mass) / each + 1);
    end.mass = above_mass + each * end.ties;
    return end;
}

template <class T>
__global__ void __launch_bounds__(kThreads) sample_row_kernel(SampleArgs a, int bits) {
    __shared__ Shared s;
    const int64_t row = blockIdx.x;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    // The largest logit and its lowest index.
    uint64_t best = 0;
    for (int64_t v = threadIdx.x; v < a.vocab; v += kThreads) {
        const uint64_t rank = static_cast<uint64_t>(key_of(static_cast<float>(in[v]))) << 32 | ~static_cast<uint32_t>(v);
        best = rank > best ? rank : best;
    }
    if (threadIdx.x == 0) s.word = 0;
    __syncthreads();
    atomicMax(&s.word, static_cast<unsigned long long>(best));
    __syncthreads();
    best = s.word;
    const uint32_t greedy = ~static_cast<uint32_t>(best);
    const float top = static_cast<float>(in[greedy]);
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    if (!(temperature > 0.0f) || !(fabsf(top) < INFINITY)) {
        if (threadIdx.x == 0) a.tokens[row] = greedy, a.probabilities[row] = 1.0f;
        return;
    }
    const Weigher weigh{static_cast<double>(top), 1.44269504088896340736 / static_cast<double>(temperature), bits};
    End end{0, ~0u, 0};
    const int64_t k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, least = a.min_p ? a.min_p[row] : 0.0f;
    if (k > 0 && k < a.vocab) end = find_end<true, T>(in, a.vocab, weigh, k, s);
    if (p < 1.0f) {
        if (end.mass == 0) {
            uint64_t sum = 0;
            for (int64_t v = threadIdx.x; v < a.vocab; v += kThreads) sum += weigh(static_cast<float>(in[v]));
            block_scan(sum, s.sums, &end.mass);
        }
        const double mass = ceil(static_cast<double>(p) * static_cast<double>(end.mass));
        end = find_end<false, T>(in, a.vocab, weigh, mass >= 1.0 ? static_cast<uint64_t>(mass) : 1, s);
    }
    const uint64_t floor_mass =
        least > 0.0f ? static_cast<uint64_t>(ceil(ldexp(static_cast<double>(least < 1.0f ? least : 1.0f), bits))) : 0;

    // Twice over the row by index: the kept mass, then the place where it is reached.
    uint64_t target = 0, all = 0;
    for (int pass = 0; pass < 2; ++pass) {
        uint64_t running = 0, ties = 0;
        for (int64_t base = 0; base < a.vocab; base += kThreads) {
            const int64_t v = base + threadIdx.x;
            const float x = v < a.vocab ? static_cast<float>(in[v]) : -INFINITY;
            const uint32_t key = v < a.vocab ? key_of(x) : 0;
            const bool tie = v < a.vocab && key == end.key;
            uint64_t of_block;
            const uint64_t rank = ties + block_scan(tie, s.sums, &of_block);
            ties += of_block;
            uint64_t w = v < a.vocab && (key > end.key || (tie && rank <= end.ties)) ? weigh(x) : 0;
            if (w < floor_mass) w = 0;
            const uint64_t reached = running + block_scan(w, s.sums, &of_block);
            if (pass == 1 && w && reached > target && reached - w <= target) {
                a.tokens[row] = v;
                a.probabilities[row] = static_cast<float>(weigh.power(weigh.exponent(x)) / static_cast<double>(all));
            }
            running += of_block;
            if (pass == 1 && running > target) return;
        }
        all = running;
        const double u = a.uniforms[row];
        const double wanted = u > 0.0 ? u * static_cast<double>(all) : 0.0;
        target = wanted < static_cast<double>(all - 1) ? static_cast<uint64_t>(wanted) : all - 1;
    }
}

}  // namespace

size_t sample_workspace_bytes(int64_t rows, int64_t vocab) { return 0; }

hipError_t launch_logits_sample(const SampleArgs& a, Type type, hipStream_t stream) {
    int bits = 51;
    while (bits > 0 && (a.vocab << bits) > (int64_t{1} << 62)) --bits;
    const dim3 grid(static_cast<uint32_t>(a.rows));
    switch (type) {
        case Type::kFloat32: hipLaunchKernelGGL(sample_row_kernel<float>, grid, dim3(kThreads), 0, stream, a, bits); break;
        case Type::kFloat16: hipLaunchKernelGGL(sample_row_kernel<_Float16>, grid, dim3(kThreads), 0, stream, a, bits); break;
        default: hipLaunchKernelGGL(sample_row_kernel<__bf16>, grid, dim3(kThreads), 0, stream, a, bits);
    }
    return hipGetLastError();
}

}  // namespace flux
