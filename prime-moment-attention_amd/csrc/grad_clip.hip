// The norm over many tensors and their scaling by min(1, max_norm / (norm + 1e-6)).
//
// The tensors come as a table in the kernel's arguments, counted in slots of 8 elements (a
// tensor's last one may be ragged); a workgroup has a span of slots that lie one after the
// other over all tensors, so that spans are equal whatever the tensors' sizes.  Squares are
// summed in 64 bits, where those of fp32 neither overflow nor vanish, and each span's sum is
// stored; the scaling's workgroups each add these in the same order.

#include "prime_kernels.h"

namespace prime {

namespace {

constexpr int kThreads = 256, kSlot = 8;

struct __attribute__((packed, aligned(2))) Raw {  // 16 bytes, wherever they start
    u32x4 v;
};

template <int DT>
__device__ __forceinline__ void load_slot(const char *p, float (&x)[kSlot]) {
    if constexpr (DT == PRIME_F32) {
        const u32x4 a = reinterpret_cast<const Raw *>(p)[0].v, b = reinterpret_cast<const Raw *>(p)[1].v;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(a[j]), x[j + 4] = __uint_as_float(b[j]);
    } else {
        const u32x4 v = reinterpret_cast<const Raw *>(p)->v;
#pragma unroll
        for (int j = 0; j < kSlot; ++j) {
            const uint32_t u = v[j / 2];
            if constexpr (DT == PRIME_BF16) x[j] = __uint_as_float(j & 1 ? u & 0xFFFF0000u : u << 16);
            else x[j] = h16_bits_to_f32(static_cast<uint16_t>(j & 1 ? u >> 16 : u));
        }
    }
}
template <int DT>
__device__ __forceinline__ void store_slot(char *p, const float (&x)[kSlot]) {
    if constexpr (DT == PRIME_F32) {
        u32x4 a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = __float_as_uint(x[j]), b[j] = __float_as_uint(x[j + 4]);
        reinterpret_cast<Raw *>(p)[0].v = a;
        reinterpret_cast<Raw *>(p)[1].v = b;
    } else {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < kSlot; j += 2) {
            if constexpr (DT == PRIME_BF16) v[j / 2] = f32_to_bf16_bits(x[j]) | static_cast<uint32_t>(f32_to_bf16_bits(x[j + 1])) << 16;
            else v[j / 2] = f32_to_h16_bits(x[j]) | static_cast<uint32_t>(f32_to_h16_bits(x[j + 1])) << 16;
        }
        reinterpret_cast<Raw *>(p)->v = v;
    }
}

__device__ __forceinline__ double wave_sum_f64(double x) {
    for (int o = 32; o; o >>= 1) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint64_t y = static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(u >> 32), o, kWave)) << 32 |
                           __shfl_xor(static_cast<uint32_t>(u), o, kWave);
        x += __builtin_bit_cast(double, y);
    }
    return x;
}
// over the workgroup, in every thread, in a fixed order
__device__ __forceinline__ double block_sum(double x, double *red) {
    x = wave_sum_f64(x);
    __syncthreads();
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// f(dtype, pointer, elements) over the tensors' pieces that the workgroup's span holds
template <typename F>
__device__ __forceinline__ void each_piece(const GradTable &t, F f) {
    const uint32_t slots = t.first[t.count];
    const uint64_t start = blockIdx.x * static_cast<uint64_t>(t.span), behind = start + t.span;
    if (start >= slots) return;
    const uint32_t begin = static_cast<uint32_t>(start), end = behind < slots ? static_cast<uint32_t>(behind) : slots;
    int lo = 0, hi = t.count - 1;  // the last tensor that starts at `begin` or before
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= begin) lo = mid;
        else hi = mid - 1;
    }
    for (uint32_t at = begin; at < end; ++lo) {
        const uint32_t stop = min(end, t.first[lo + 1]);
        const uint64_t word = t.data[lo];
        const int dt = static_cast<int>(word >> 62);
        const int64_t from = static_cast<int64_t>(at - t.first[lo]) * kSlot;
        const int64_t size = t.size[lo] - from, most = static_cast<int64_t>(stop - at) * kSlot;
        f(dt, reinterpret_cast<char *>(word & ((1ull << 62) - 1)) + from * (dt == PRIME_F32 ? 4 : 2), size < most ? size : most);
        at = stop;
    }
}

template <int DT>
__device__ __forceinline__ double square_sum(const char *p, int64_t size) {
    constexpr int U = 4, es = DT == PRIME_F32 ? 4 : 2;
    double acc[2] = {};
    const int64_t whole = size / kSlot;
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < whole; i += U * kThreads) {
        float x[U][kSlot];
#pragma unroll
        for (int u = 0; u < U; ++u) load_slot<DT>(p + (i + u * kThreads) * (kSlot * es), x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < kSlot; ++j) acc[j & 1] = fma(static_cast<double>(x[u][j]), static_cast<double>(x[u][j]), acc[j & 1]);
    }
    for (; i < whole; i += kThreads) {
        float x[kSlot];
        load_slot<DT>(p + i * (kSlot * es), x);
#pragma unroll
        for (int j = 0; j < kSlot; ++j) acc[j & 1] = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), acc[j & 1]);
    }
    if (const int64_t j = whole * kSlot + threadIdx.x; j < size) {
        const double x = load_elem(p, j, DT);
        acc[0] = fma(x, x, acc[0]);
    }
    return acc[0] + acc[1];
}

template <int DT>
__device__ __forceinline__ void scale_piece(char *p, int64_t size, float c) {
    constexpr int U = 4, es = DT == PRIME_F32 ? 4 : 2;
    const int64_t whole = size / kSlot;
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < whole; i += U * kThreads) {
        float x[U][kSlot];
#pragma unroll
        for (int u = 0; u < U; ++u) load_slot<DT>(p + (i + u * kThreads) * (kSlot * es), x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < kSlot; ++j) x[u][j] *= c;
            store_slot<DT>(p + (i + u * kThreads) * (kSlot * es), x[u]);
        }
    }
    for (; i < whole; i += kThreads) {
        float x[kSlot];
        load_slot<DT>(p + i * (kSlot * es), x);
#pragma unroll
        for (int j = 0; j < kSlot; ++j) x[j] *= c;
        store_slot<DT>(p + i * (kSlot * es), x);
    }
    if (const int64_t j = whole * kSlot + threadIdx.x; j < size) store_elem(p, j, DT, load_elem(p, j, DT) * c);
}

}  // namespace

// parts[blockIdx.x]: the span's sum of squares
__global__ __launch_bounds__(kThreads) void grad_squares_kernel(const GradTable t, double *parts) {
    __shared__ double red[kThreads / kWave];
    double sum = 0.0;
    each_piece(t, [&](int dt, char *p, int64_t size) {
        if (dt == PRIME_BF16) sum += square_sum<PRIME_BF16>(p, size);
        else if (dt == PRIME_F16) sum += square_sum<PRIME_F16>(p, size);
        else sum += square_sum<PRIME_F32>(p, size);
    });
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

__device__ __forceinline__ double parts_sum(const double *parts, int count, double *red) {
    double sum = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += kThreads) sum += parts[i];
    return block_sum(sum, red);
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const double *parts, int count, float *norm) {
    __shared__ double red[kThreads / kWave];
    const double sum = parts_sum(parts, count, red);
    if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(sum));
}

// parts: the sums of squares, whose root is written to `norm`; or null, `norm` being given.
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(const GradTable t, const double *parts, int count,
                                                              float *norm, double max_norm) {
    __shared__ double red[kThreads / kWave];
    double total;
    if (parts) {
        total = sqrt(parts_sum(parts, count, red));
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
    } else {
        total = *norm;
    }
    const float c = static_cast<float>(max_norm / (total + 1e-6));
    if (c >= 1.f || max_norm == __builtin_inf()) return;  // (a NaN scales)
    each_piece(t, [&](int dt, char *p, int64_t size) {
        if (dt == PRIME_BF16) scale_piece<PRIME_BF16>(p, size, c);
        else if (dt == PRIME_F16) scale_piece<PRIME_F16>(p, size, c);
        else scale_piece<PRIME_F32>(p, size, c);
    });
}

hipError_t launch_grad_squares(const GradTable &t, int blocks, double *parts, hipStream_t stream) {
    hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(kThreads), 0, stream, t, parts);
    return hipGetLastError();
}
hipError_t launch_grad_norm(const double *parts, int count, float *norm, hipStream_t stream) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kThreads), 0, stream, parts, count, norm);
    return hipGetLastError();
}
hipError_t launch_grad_scale(const GradTable &t, int blocks, const double *parts, int count, float *norm,
                             double max_norm, hipStream_t stream) {
    hipLaunchKernelGGL(grad_scale_kernel, dim3(blocks), dim3(kThreads), 0, stream, t, parts, count, norm, max_norm);
    return hipGetLastError();
}

}  // namespace prime
