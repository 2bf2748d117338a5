// Logits of a batch on their way to the next token: penalties for the tokens of a row's history, a bias, a grammar's
// bit mask, and the lowest index of the largest result.
//
//   c = occurrences of v in the row's history
//   x = c > 0 ? (x > 0 ? x / repetition : x * repetition) : x;  x -= frequency * c;  x -= c > 0 ? presence : 0
//   x += bias;  x = allowed ? x : -inf;  rounded once to the logits' type
//
// One workgroup takes kChunk tokens of a row: it requests its logits, counts the row's history into LDS meanwhile
// (integers, so the order of the additions does not show), then writes.  Few tokens are in a history: a bit per token
// says which, and only those take the penalties' path.  HBM-bound for a batch, launch-bound for one row.
#include "serving.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace flux {
namespace {

struct Candidate {
    int64_t index;
    float value;
};

template <class T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }

__device__ __forceinline__ void keep_better(float& value, int64_t& index, float other, int64_t other_index) {
    if (argmax_precedes(other, other_index, value, index)) {
        value = other;
        index = other_index;
    }
}

__device__ __forceinline__ void wave_best(float& value, int64_t& index) {
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const float v = __shfl_xor(value, step, kWave);
        const int64_t i = __shfl_xor(static_cast<long long>(index), step, kWave);
        keep_better(value, index, v, i);
    }
}

template <class T, int kChunk, int kThreads, bool kWide>
__global__ void __launch_bounds__(kThreads) logits_kernel(LogitsArgs a, int chunks) {
    constexpr int kWidth = kWide ? 16 / static_cast<int>(sizeof(T)) : 1;
    constexpr int kUnits = kChunk / (kThreads * kWidth);
    constexpr int kIds = 4;  // of the history, per thread and round
    __shared__ uint32_t counts[kChunk];
    __shared__ uint32_t seen[kChunk / 32];  // a bit per token of the history
    __shared__ Candidate best[kThreads / kWave];
    const int64_t row = blockIdx.x / chunks;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x % chunks) * kChunk;
    const int size = static_cast<int>(a.vocab - c0 < kChunk ? a.vocab - c0 : kChunk);
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + c0;
    T* out = static_cast<T*>(a.out) + row * a.vocab + c0;
    const float* bias = a.bias ? a.bias + row * a.bias_stride + c0 : nullptr;
    const int32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride + c0 / 32 : nullptr;

    struct alignas(16) Unit {
        T x[kWidth];
    };
    Unit held[kUnits];
    uint32_t bits[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int v = kWidth * (threadIdx.x + kThreads * u);
        bits[u] = ~0u;
        if (v >= size) continue;
        if constexpr (kWide) {
            *reinterpret_cast<uint4*>(held[u].x) = *reinterpret_cast<const uint4*>(in + v);
        } else {
            held[u].x[0] = in[v];
        }
        if (allowed) bits[u] = static_cast<uint32_t>(allowed[v / 32]) >> (v % 32);
    }
    const float repetition = a.repetition ? a.repetition[row] : 1.0f;
    const float frequency = a.frequency ? a.frequency[row] : 0.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f;
    if (a.history) {
        int64_t n = a.history_lengths ? a.history_lengths[row] : a.history_width;
        n = n < a.history_width ? n : a.history_width;
        const int64_t* ids = a.history + row * a.history_stride;
        for (int v = 4 * threadIdx.x; v < kChunk; v += 4 * kThreads) *reinterpret_cast<uint4*>(counts + v) = make_uint4(0, 0, 0, 0);
        for (int w = threadIdx.x; w < kChunk / 32; w += kThreads) seen[w] = 0;
        int64_t id[kIds];
#pragma unroll
        for (int j = 0; j < kIds; ++j) id[j] = threadIdx.x + kThreads * j < n ? ids[threadIdx.x + kThreads * j] : -1;
        __syncthreads();
        for (int64_t t = threadIdx.x; t < n; t += kIds * kThreads) {
#pragma unroll
            for (int j = 0; j < kIds; ++j)
                if (id[j] >= c0 && id[j] < c0 + size) {
                    const int v = static_cast<int>(id[j] - c0);
                    if (atomicAdd(counts + v, 1u) == 0) atomicOr(seen + v / 32, 1u << (v % 32));
                }
#pragma unroll
            for (int j = 0; j < kIds; ++j) {
                const int64_t next = t + (kIds + j) * kThreads;
                id[j] = next < n ? ids[next] : -1;
            }
        }
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
        for (int j = 0; j < kWidth; ++j) y[j] = to_float(held[u].x[j]);
        if (a.history) {
            uint32_t mine = seen[v / 32] >> (v % 32) & ((1u << kWidth) - 1u);
            while (mine) {
#pragma clang fp contract(off)
                const int which = __ffs(mine) - 1;
                mine &= mine - 1;
                float x = y[0];
#pragma unroll
                for (int j = 1; j < kWidth; ++j) x = which == j ? y[j] : x;
                x = x > 0.0f ? x / repetition : x * repetition;
                x = x - frequency * static_cast<float>(counts[v + which]);
                x = x - presence;
#pragma unroll
                for (int j = 0; j < kWidth; ++j) y[j] = which == j ? x : y[j];
            }
        }
        if (bias) {
            alignas(16) float shift[kWidth];
            if constexpr (kWide) {
#pragma unroll
                for (int j = 0; j < kWidth; j += 4)
                    *reinterpret_cast<float4*>(shift + j) = *reinterpret_cast<const float4*>(bias + v + j);
            } else {
                shift[0] = bias[v];
            }
#pragma unroll
            for (int j = 0; j < kWidth; ++j) y[j] += shift[j];
        }
#pragma unroll
        for (int j = 0; j < kWidth; ++j) {
            held[u].x[j] = static_cast<T>(bits[u] >> j & 1u ? y[j] : -INFINITY);
            // Larger than all before, or the first NaN.
            const float x = to_float(held[u].x[j]);
            const bool better = !(x <= value) & (value == value);
            value = better ? x : value;
            at = better ? v + j : at;
        }
        if constexpr (kWide) {
            *reinterpret_cast<uint4*>(out + v) = *reinterpret_cast<const uint4*>(held[u].x);
        } else {
            out[v] = held[u].x[0];
        }
    }
    int64_t index = at < size ? c0 + at : INT64_MAX;
    wave_best(value, index);
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = Candidate{index, value};
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / kWave; ++w) keep_better(value, index, best[w].value, best[w].index);
        if (chunks == 1) a.tokens[row] = index;
        else static_cast<Candidate*>(a.workspace)[blockIdx.x] = Candidate{index, value};
    }
}

// One wave per row over its chunks' best.
__global__ void __launch_bounds__(64) logits_token_kernel(const Candidate* __restrict__ best, int64_t* tokens,
                                                          int chunks) {
    const int64_t row = blockIdx.x;
    float value = -INFINITY;
    int64_t index = INT64_MAX;
    for (int c = threadIdx.x; c < chunks; c += 64) {
        const Candidate other = best[row * chunks + c];
        keep_better(value, index, other.value, other.index);
    }
    wave_best(value, index);
    if (threadIdx.x == 0) tokens[row] = index;
}

// Tokens of a workgroup: 8192, which read the history least often, unless that leaves CUs without one.
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
                       static_cast<const Candidate*>(a.workspace), a.tokens, chunks);
    return hipGetLastError();
}

}  // namespace

size_t logits_workspace_bytes(int64_t rows, int64_t vocab) {
    const int chunks = logits_chunks(rows, vocab);
    return chunks > 1 ? static_cast<size_t>(rows) * chunks * sizeof(Candidate) : 0;
}

hipError_t launch_logits_process(const LogitsArgs& args, Type type, hipStream_t stream) {
    switch (type) {
        case Type::kFloat32: return launch_logits<float>(args, stream);
        case Type::kFloat16: return launch_logits<_Float16>(args, stream);
        default: return launch_logits<__bf16>(args, stream);
    }
}

}  // namespace flux
