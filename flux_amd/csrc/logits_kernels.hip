// Logits of a batch on their way to the next token: penalties for the tokens of a row's history, a bias, a grammar's
// bit mask, and the lowest index of the largest result.
//
//   c = occurrences of v in the row's history
//   x = c > 0 ? (x > 0 ? x / repetition : x * repetition) : x;  x -= frequency * c;  x -= c > 0 ? presence : 0
//   x += bias;  x = allowed ? x : -inf;  rounded once to the logits' type
//
// One workgroup takes kChunk tokens of a row: it counts the row's history into LDS (integers, so the order of the
// additions does not show), then reads and writes its logits once.  HBM-bound for a batch, launch-bound for one row.
#include "serving.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace flux {
namespace {

constexpr int kLogitThreads = 512;
constexpr int kChunk = 8192;

struct Candidate {
    int64_t index;
    float value;
    float pad;
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

template <class T, bool kWide>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(LogitsArgs a, int chunks) {
    __shared__ uint32_t counts[kChunk];
    __shared__ Candidate best[kLogitThreads / kWave];
    const int64_t row = blockIdx.x / chunks;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x % chunks) * kChunk;
    const int size = static_cast<int>(a.vocab - c0 < kChunk ? a.vocab - c0 : kChunk);
    if (a.history) {
        for (int v = threadIdx.x; v < size; v += kLogitThreads) counts[v] = 0;
        __syncthreads();
        int64_t n = a.history_lengths ? a.history_lengths[row] : a.history_width;
        n = n < a.history_width ? n : a.history_width;
        const int64_t* ids = a.history + row * a.history_stride;
        for (int64_t t = threadIdx.x; t < n; t += kLogitThreads) {
            const int64_t v = ids[t] - c0;
            if (v >= 0 && v < size) atomicAdd(counts + v, 1u);
        }
        __syncthreads();
    }
    const float repetition = a.repetition ? a.repetition[row] : 1.0f;
    const float frequency = a.frequency ? a.frequency[row] : 0.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + c0;
    T* out = static_cast<T*>(a.out) + row * a.vocab + c0;
    const float* bias = a.bias ? a.bias + row * a.bias_stride + c0 : nullptr;
    const int32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride + c0 / 32 : nullptr;

    float value = -INFINITY;
    int64_t index = INT64_MAX;
    constexpr int kWidth = kWide ? 16 / static_cast<int>(sizeof(T)) : 1;
    for (int v = kWidth * threadIdx.x; v < size; v += kWidth * kLogitThreads) {
        alignas(16) T x[kWidth];
        alignas(16) float shift[kWidth];
        if constexpr (kWide) {
            *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(in + v);
            if (bias) {
#pragma unroll
                for (int j = 0; j < kWidth; j += 4)
                    *reinterpret_cast<float4*>(shift + j) = *reinterpret_cast<const float4*>(bias + v + j);
            }
        } else {
            x[0] = in[v];
            if (bias) shift[0] = bias[v];
        }
        const uint32_t bits = allowed ? static_cast<uint32_t>(allowed[v / 32]) >> (v % 32) : ~0u;
#pragma unroll
        for (int j = 0; j < kWidth; ++j) {
#pragma clang fp contract(off)
            float y = to_float(x[j]);
            const uint32_t count = a.history ? counts[v + j] : 0;
            if (count > 0) {
                y = y > 0.0f ? y / repetition : y * repetition;
                y = y - frequency * static_cast<float>(count);
                y = y - presence;
            }
            if (bias) y = y + shift[j];
            if (!(bits >> j & 1u)) y = -INFINITY;
            x[j] = static_cast<T>(y);
            keep_better(value, index, to_float(x[j]), c0 + v + j);
        }
        if constexpr (kWide) {
            *reinterpret_cast<uint4*>(out + v) = *reinterpret_cast<const uint4*>(x);
        } else {
            out[v] = x[0];
        }
    }
    wave_best(value, index);
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = Candidate{index, value, 0.0f};
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLogitThreads / kWave; ++w) keep_better(value, index, best[w].value, best[w].index);
        if (chunks == 1) a.tokens[row] = index;
        else static_cast<Candidate*>(a.workspace)[blockIdx.x] = Candidate{index, value, 0.0f};
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

int logits_chunks(int64_t vocab) { return static_cast<int>((vocab + kChunk - 1) / kChunk); }

template <class T>
hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
    const int chunks = logits_chunks(a.vocab);
    constexpr int64_t kWidth = 16 / sizeof(T);
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool wide = a.vocab % kWidth == 0 && a.logits_stride % kWidth == 0 && aligned(a.logits) && aligned(a.out) &&
                      (!a.bias || (aligned(a.bias) && a.bias_stride % 4 == 0));
    const dim3 grid(static_cast<uint32_t>(a.rows * chunks));
    if (wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(logits_kernel<T, true>), grid, dim3(kLogitThreads), 0, stream, a, chunks);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(logits_kernel<T, false>), grid, dim3(kLogitThreads), 0, stream, a, chunks);
    const hipError_t launched = hipGetLastError();
    if (launched != hipSuccess || chunks == 1) return launched;
    hipLaunchKernelGGL(logits_token_kernel, dim3(static_cast<uint32_t>(a.rows)), dim3(64), 0, stream,
                       static_cast<const Candidate*>(a.workspace), a.tokens, chunks);
    return hipGetLastError();
}

}  // namespace

size_t logits_workspace_bytes(int64_t rows, int64_t vocab) {
    const int chunks = logits_chunks(vocab);
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
