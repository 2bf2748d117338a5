// Logits of a batch on their way to the next token: penalties for the tokens of a row's history, a bias, a grammar's
// bit mask, and the lowest index of the largest result.
//
//   c = occurrences of v in the row's history
//   x = c > 0 ? (x > 0 ? x / repetition : x * repetition) : x;  x -= frequency * c;  x -= c > 0 ? presence : 0
//   x += bias;  x = allowed ? x : -inf;  rounded once to the logits' type
//
// One workgroup takes kChunk tokens of a row: it requests its logits, counts the row's history into LDS meanwhile
// (integers, so the order of the additions does not show), then writes.  Few tokens are in a history: a bit per token
// says which, and only those take the penalties' path, whose results replace the counts.  The best token is looked for by
// unit: a unit's largest value first (maximum keeps a NaN), its place in the unit once for the workgroup's best.
// HBM and the latency of its phases bound a batch (128 rows of 128000 in bfloat16, 65.5 MB: 22 us with histories of 4096,
// a bias and a mask, 24 if stored through the caches; 13.4 us without them, where a copy takes 10.5), launches one row.
#include "serving.h"

namespace flux {
namespace {

// A value and an index as one number: the larger value's is larger, NaN's the largest, of equal values the lower index's
// (zeros of both signs are equal).  Never 0, which stands for nothing.
__device__ __forceinline__ uint64_t rank_of(float value, uint32_t index) {
    const int bits = __float_as_int(value + 0.0f);
    const uint32_t order = value != value ? ~0u : static_cast<uint32_t>(bits ^ (bits >> 31 | static_cast<int>(0x80000000u)));
    return static_cast<uint64_t>(order) << 32 | ~index;
}

__device__ __forceinline__ uint32_t wave_max_word(uint32_t v) {
    auto with = [&](uint32_t other) { v = v > other ? v : other; };
    with(__builtin_amdgcn_update_dpp(0, v, kDppRowRor8, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, v, kDppRowRor4, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, v, kDppQuadXor2, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, v, kDppQuadXor1, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, v, kDppRowBcast15, 0xA, 0xF, false));
    with(__builtin_amdgcn_update_dpp(0, v, kDppRowBcast31, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

__device__ __forceinline__ uint64_t wave_best(uint64_t rank) {
    const uint32_t order = static_cast<uint32_t>(rank >> 32);
    const uint32_t highest = wave_max_word(order);
    return static_cast<uint64_t>(highest) << 32 | wave_max_word(order == highest ? static_cast<uint32_t>(rank) : 0u);
}

__device__ __forceinline__ uint32_t select_bits(uint32_t mask, uint32_t one, uint32_t other) {
    return (one & mask) | (other & ~mask);
}
// All ones where bit j of `bits` is set.
__device__ __forceinline__ uint32_t mask_of(uint32_t bits, int j) { return static_cast<int>(bits << (31 - j)) >> 31; }

typedef float FloatPair __attribute__((ext_vector_type(2)));

// The logits of one 16-byte load (kWide) or one logit, as 32-bit words.
template <class T, bool kWide>
struct Unit {
    static constexpr int kPer = kWide && sizeof(T) == 2 ? 2 : 1;  // logits of a word
    static constexpr int kWords = kWide ? 4 : 1;
    static constexpr int kWidth = kWords * kPer;
    uint32_t word[kWords];

    static __device__ __forceinline__ float value(uint32_t word, int odd) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(word);
        else return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(odd ? word >> 16 : word)));
    }
    __device__ __forceinline__ float operator[](int j) const { return value(word[j / kPer], j % kPer); }
    __device__ __forceinline__ void load(const T* from) {
        if constexpr (kWide) {
            const uint4 quad = *reinterpret_cast<const uint4*>(from);
            word[0] = quad.x, word[1] = quad.y, word[2] = quad.z, word[3] = quad.w;
        } else if constexpr (sizeof(T) == 4) {
            word[0] = __float_as_uint(*from);
        } else {
            word[0] = __builtin_bit_cast(uint16_t, *from);
        }
    }
    __device__ __forceinline__ void store(T* to) const {
        if constexpr (kWide) store_past_caches(to, Quad{word[0], word[1], word[2], word[3]});
        else *to = static_cast<T>(value(word[0], 0));
    }
    __device__ __forceinline__ void round(const float (&y)[kWidth]) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            if constexpr (sizeof(T) == 4) {
                word[w] = __float_as_uint(y[w]);
            } else {
                typedef T Pair __attribute__((ext_vector_type(2)));
                word[w] = __builtin_bit_cast(uint32_t, __builtin_convertvector((FloatPair{y[w * kPer], y[w * kPer + kPer - 1]}), Pair));
            }
        }
    }
};

template <class T, int kChunk, int kThreads, bool kWide>
__global__ void __launch_bounds__(kThreads) logits_kernel(LogitsArgs a, int chunks) {
    using U = Unit<T, kWide>;
    constexpr int kWidth = U::kWidth;
    constexpr int kUnits = kChunk / (kThreads * kWidth);
    constexpr int kWords = kUnits * U::kWords;
    static_assert(kUnits * kWidth <= 32, "one bit for each of a thread's logits");
    constexpr int kIds = 4;  // of the history, per thread and round
    __shared__ uint32_t counts[kChunk];  // then the logits with their penalties
    __shared__ uint32_t seen[kChunk / 32];  // a bit per token of the history
    __shared__ unsigned long long best;
    const int64_t row = blockIdx.x / chunks;
    const uint32_t c0 = blockIdx.x % chunks * kChunk;
    const int size = static_cast<int>(a.vocab - c0 < kChunk ? a.vocab - c0 : kChunk);
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + c0;
    T* out = static_cast<T*>(a.out) + row * a.vocab + c0;
    const float* bias = a.bias ? a.bias + row * a.bias_stride + c0 : nullptr;
    const int32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride + c0 / 32 : nullptr;

    // All loads first, of the last unit where there is none: a use or a branch between them would wait for each.
    U held[kUnits];
    uint32_t bits[kUnits];
    alignas(16) float shift[kUnits][kWidth];
    auto place_of = [&](int u) {
        const int v = kWidth * (threadIdx.x + kThreads * u);
        return v < size ? v : size - kWidth;
    };
#pragma unroll
    for (int u = 0; u < kUnits; ++u) held[u].load(in + place_of(u));
    if (allowed) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) bits[u] = allowed[place_of(u) / 32];
    }
    if (bias) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const float* from = bias + place_of(u);
            if constexpr (kWide) {
#pragma unroll
                for (int j = 0; j < kWidth; j += 4)
                    *reinterpret_cast<float4*>(shift[u] + j) = *reinterpret_cast<const float4*>(from + j);
            } else {
                shift[u][0] = *from;
            }
        }
    }
    const float repetition = a.repetition ? a.repetition[row] : 1.0f;
    const float frequency = a.frequency ? a.frequency[row] : 0.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f;
    if (threadIdx.x == 0) best = 0;
    uint32_t hits = 0;  // of this thread's logits, those in the history
    if (a.history) {
        // The ids of a row's whole width are requested before its length is known.
        const int64_t* ids = a.history + row * a.history_stride;
        int64_t id[kIds];
#pragma unroll
        for (int j = 0; j < kIds; ++j) {
            const int64_t t = threadIdx.x + kThreads * j;
            id[j] = t < a.history_width ? ids[t] : -1;
        }
        int64_t n = a.history_lengths ? a.history_lengths[row] : a.history_width;
        n = n < a.history_width ? n : a.history_width;
        for (int v = 4 * threadIdx.x; v < kChunk; v += 4 * kThreads) *reinterpret_cast<uint4*>(counts + v) = make_uint4(0, 0, 0, 0);
        for (int w = threadIdx.x; w < kChunk / 32; w += kThreads) seen[w] = 0;
        __syncthreads();
        for (int64_t t = threadIdx.x; t < n; t += kIds * kThreads) {
#pragma unroll
            for (int j = 0; j < kIds; ++j) {
                const uint32_t v = static_cast<uint32_t>(id[j]) - c0;
                if ((id[j] >> 32 == 0) & (v < static_cast<uint32_t>(size)) & (t + kThreads * j < n)) {
                    atomicAdd(counts + v, 1u);
                    atomicOr(seen + v / 32, 1u << (v % 32));
                }
            }
#pragma unroll
            for (int j = 0; j < kIds; ++j) {
                const int64_t next = t + (kIds + j) * kThreads;
                id[j] = next < n ? ids[next] : -1;
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int v = kWidth * (threadIdx.x + kThreads * u);
            hits |= (seen[v / 32] >> (v % 32) & ((1u << kWidth) - 1u)) << (kWidth * u);
        }
        for (uint32_t rest = hits; rest; rest &= rest - 1) {
#pragma clang fp contract(off)
            const int which = __ffs(rest) - 1, of = which / U::kPer;
            uint32_t words[kWords];
#pragma unroll
            for (int w = 0; w < kWords; ++w) words[w] = held[w / U::kWords].word[w % U::kWords];
#pragma unroll
            for (int half = kWords / 2; half >= 1; half /= 2) {
                const uint32_t upper = of & half ? ~0u : 0u;
#pragma unroll
                for (int w = 0; w < half; ++w) words[w] = select_bits(upper, words[w + half], words[w]);
            }
            uint32_t* place = counts + kWidth * (threadIdx.x + kThreads * (which / kWidth)) + which % kWidth;
            float x = U::value(words[0], which % U::kPer);
            x = x > 0.0f ? x / repetition : x * repetition;
            x = x - frequency * static_cast<float>(*place);
            x = x - presence;
            *place = __float_as_uint(x);
        }
    } else {
        __syncthreads();
    }

    float value = -INFINITY;
    int at = kWidth * threadIdx.x;  // the lowest index that this thread looks at: right where all are -inf
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int v = kWidth * (threadIdx.x + kThreads * u);
        if (v >= size) continue;
        float y[kWidth];
#pragma unroll
        for (int j = 0; j < kWidth; ++j) y[j] = held[u][j];
        const uint32_t mine = hits >> (kWidth * u) & ((1u << kWidth) - 1u);
        if (mine) {
            alignas(16) uint32_t penalised[kWidth];  // all read: a branch for each costs more
            if constexpr (kWide) {
#pragma unroll
                for (int j = 0; j < kWidth; j += 4)
                    *reinterpret_cast<uint4*>(penalised + j) = *reinterpret_cast<const uint4*>(counts + v + j);
            } else {
                penalised[0] = counts[v];
            }
#pragma unroll
            for (int j = 0; j < kWidth; ++j)
                y[j] = __uint_as_float(select_bits(mask_of(mine, j), penalised[j], __float_as_uint(y[j])));
        }
        if (bias) {
#pragma unroll
            for (int j = 0; j < kWidth; ++j) y[j] += shift[u][j];
        }
        if (allowed) {
#pragma unroll
            for (int j = 0; j < kWidth; ++j)
                y[j] = __uint_as_float(select_bits(mask_of(bits[u] >> (v % 32), j), __float_as_uint(y[j]), 0xff800000u));
        }
        held[u].round(y);
        held[u].store(out + v);
        float highest = y[0];
#pragma unroll
        for (int j = 1; j < kWidth; ++j) highest = __builtin_elementwise_maximum(highest, y[j]);
        highest = static_cast<float>(static_cast<T>(highest));  // rounding keeps the order
        const bool better = !(highest <= value) & (value == value);  // larger than all before, or the first NaN
        value = better ? highest : value;
        at = better ? v : at;
    }
    const uint64_t rank = at < size ? rank_of(value, at) : 0;
    const uint64_t of_wave = wave_best(rank);
    if ((threadIdx.x & 63) == 0) atomicMax(&best, static_cast<unsigned long long>(of_wave));
    __syncthreads();
    if (rank != best) return;
    // One thread is left: which of its unit's logits is it?
    uint32_t index = 0;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        if (kWidth * (threadIdx.x + kThreads * u) != static_cast<uint32_t>(at)) continue;
#pragma unroll
        for (int j = kWidth - 1; j >= 0; --j)
            if (held[u][j] == value || held[u][j] != held[u][j]) index = c0 + at + j;
    }
    if (chunks == 1) a.tokens[row] = index;
    else static_cast<uint64_t*>(a.workspace)[blockIdx.x] = rank_of(value, index);
}

// One wave per row over its chunks' best.
__global__ void __launch_bounds__(64) logits_token_kernel(const uint64_t* __restrict__ best, int64_t* tokens, int chunks) {
    const int64_t row = blockIdx.x;
    uint64_t rank = 0;
    for (int c = threadIdx.x; c < chunks; c += 64) {
        const uint64_t other = best[row * chunks + c];
        rank = rank > other ? rank : other;
    }
    rank = wave_best(rank);
    if (threadIdx.x == 0) tokens[row] = ~static_cast<uint32_t>(rank);
}

// Tokens of a workgroup: 8192 with 512 threads (the batch above; 4096 with 256, which read the history twice as
// often, take 3 us more), unless that leaves CUs without one.
constexpr int kLargeChunk = 8192, kSmallChunk = 2048;
int logits_chunk(int64_t rows, int64_t vocab) {
    return rows * ((vocab + kLargeChunk - 1) / kLargeChunk) >= 256 ? kLargeChunk : kSmallChunk;
}
int logits_chunks(int64_t rows, int64_t vocab) {
    const int chunk = logits_chunk(rows, vocab);
    return static_cast<int>((vocab + chunk - 1) / chunk);
}

template <class T, int kChunk, int kThreads>
hipError_t launch_chunks(const LogitsArgs& a, int chunks, bool wide, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(a.rows * chunks));
    if (wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(logits_kernel<T, kChunk, kThreads, true>), grid, dim3(kThreads), 0, stream, a, chunks);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(logits_kernel<T, kChunk, kThreads, false>), grid, dim3(kThreads), 0, stream, a, chunks);
    return hipGetLastError();
}

template <class T>
hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
    const int chunks = logits_chunks(a.rows, a.vocab);
    constexpr int64_t kWidth = 16 / sizeof(T);
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool wide = a.vocab % kWidth == 0 && a.logits_stride % kWidth == 0 && aligned(a.logits) && aligned(a.out) &&
                      (!a.bias || (aligned(a.bias) && a.bias_stride % 4 == 0));
    const hipError_t launched = logits_chunk(a.rows, a.vocab) == kLargeChunk
                                    ? launch_chunks<T, kLargeChunk, 512>(a, chunks, wide, stream)
                                    : launch_chunks<T, kSmallChunk, 256>(a, chunks, wide, stream);
    if (launched != hipSuccess || chunks == 1) return launched;
    hipLaunchKernelGGL(logits_token_kernel, dim3(static_cast<uint32_t>(a.rows)), dim3(64), 0, stream,
                       static_cast<const uint64_t*>(a.workspace), a.tokens, chunks);
    return hipGetLastError();
}

}  // namespace

size_t logits_workspace_bytes(int64_t rows, int64_t vocab) {
    const int chunks = logits_chunks(rows, vocab);
    return chunks > 1 ? static_cast<size_t>(rows) * chunks * sizeof(uint64_t) : 0;
}

hipError_t launch_logits_process(const LogitsArgs& args, Type type, hipStream_t stream) {
    switch (type) {
        case Type::kFloat32: return launch_logits<float>(args, stream);
        case Type::kFloat16: return launch_logits<_Float16>(args, stream);
        default: return launch_logits<__bf16>(args, stream);
    }
}

}  // namespace flux
