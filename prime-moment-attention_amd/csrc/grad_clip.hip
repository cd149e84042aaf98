// The norm over many tensors and their scaling by min(1, max_norm / (norm + 1e-6)).
//
// The tensors come as a table in the kernel's arguments, cut into blocks of kGradBlock elements
// (a tensor's last one may be short): the loads of a block are on their way at once, so that a
// small tensor costs as much time as one, and a wave has a span of blocks that lie one after
// the other over all tensors.  Squares are summed in 64 bits, where those of fp32 neither
// overflow nor vanish, and each workgroup's sum is stored; the scaling's workgroups each add
// these in the same order.
//
// Bound by memory, but for small models, where two launches are (us on the device, sums and
// scaling): 124 M elements fp32 133 + 168, 4.9 TB/s, a copy's rate; bf16 69 + 76; the sums alone
// 84 and 45 (5.9 and 5.5 TB/s), where no scaling's writes are still on their way out of the
// caches.  28 small fp32 tensors 4.1 + 5.1; 80 tensors, 34 M elements, mostly
// bf16, whose norm clips nothing 15 + 4.9.  (Sums in fp32 are no faster; nor is scaling from the end, what the sums read last.)

#include "prime_kernels.h"
#include "row_vec.h"

namespace prime {

namespace {

constexpr int kThreads = 256, kSlot = 8;

template <int DT>
__device__ __forceinline__ void load_slot(const char *p, float (&x)[kSlot]) {
    constexpr int V = kVec<DT>;
    u32x4 v[kSlot / V];
#pragma unroll
    for (int i = 0; i < kSlot / V; ++i) v[i] = reinterpret_cast<const Raw *>(p)[i].v;
#pragma unroll
    for (int i = 0; i < kSlot / V; ++i) widen<DT>(v[i], reinterpret_cast<float(&)[V]>(x[i * V]));
}
template <int DT>
__device__ __forceinline__ void store_slot(char *p, const float (&x)[kSlot]) {
    constexpr int V = kVec<DT>;
#pragma unroll
    for (int i = 0; i < kSlot / V; ++i) reinterpret_cast<Raw *>(p)[i].v = narrow<DT>(reinterpret_cast<const float(&)[V]>(x[i * V]));
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

// f(dtype, pointer, elements) over the blocks of the wave's span
template <typename F>
__device__ __forceinline__ void each_block(const GradTable &t, F f) {
    const uint32_t blocks = t.first[t.count];
    const uint64_t start = (blockIdx.x * static_cast<uint64_t>(kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)) * t.span;
    if (start >= blocks) return;
    const uint32_t begin = static_cast<uint32_t>(start), end = start + t.span < blocks ? static_cast<uint32_t>(start + t.span) : blocks;
    uint32_t b = begin;
    // the tensor with block b: the last that starts there or before; each lane looks at three
    int k = -1;
#pragma unroll
    for (int q = 0; q < kGradTable / kWave; ++q) {
        const int i = q * kWave + threadIdx.x % kWave;
        const uint32_t first = t.first[i];
        k += __popcll(__ballot(i < t.count && first <= b));
    }
    for (; b < end; ++k) {
        // the span's blocks of tensor k
        const uint32_t first = t.first[k], stop = min(end, t.first[k + 1]);
        const uint64_t word = t.data[k];
        const int dt = static_cast<int>(word >> 62);
        char *data = reinterpret_cast<char *>(word & ((1ull << 62) - 1));
        const int64_t size = t.size[k];
        for (; b < stop; ++b) {
            const int64_t skip = static_cast<int64_t>(b - first) * kGradBlock;
            f(dt, data + skip * (dt == PRIME_F32 ? 4 : 2), static_cast<int>(min(size - skip, static_cast<int64_t>(kGradBlock))));
        }
    }
}

// g(slot's address, values) over a block, all its loads before the first use; then the elements
// behind the last whole slot: one(address).
template <int DT, typename G, typename E>
__device__ __forceinline__ void each_slot(char *p, int size, G g, E one) {
    constexpr int es = DT == PRIME_F32 ? 4 : 2, bytes = kSlot * es, U = kGradBlock / (kSlot * kWave);
    const int whole = size / kSlot, lane = threadIdx.x % kWave;
    if (whole) {
        float x[U][kSlot];
#pragma unroll
        for (int u = 0; u < U; ++u) load_slot<DT>(p + min(lane + u * kWave, whole - 1) * bytes, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lane + u * kWave < whole) g(p + (lane + u * kWave) * bytes, x[u]);
    }
    if (const int j = whole * kSlot + lane; j < size) one(p + j * es);
}

template <int DT>
__device__ __forceinline__ double square_sum(char *p, int size) {
    double acc[2] = {};
    each_slot<DT>(
        p, size,
        [&](char *, const float (&x)[kSlot]) {
#pragma unroll
            for (int j = 0; j < kSlot; ++j) acc[j & 1] = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), acc[j & 1]);
        },
        [&](char *q) {
            const double x = load_elem(q, 0, DT);
            acc[0] = fma(x, x, acc[0]);
        });
    return acc[0] + acc[1];
}

template <int DT>
__device__ __forceinline__ void scale_block(char *p, int size, float c, float power) {
    each_slot<DT>(
        p, size,
        [&](char *q, float (&x)[kSlot]) {
#pragma unroll
            for (int j = 0; j < kSlot; ++j) x[j] = x[j] * c * power;
            store_slot<DT>(q, x);
        },
        [&](char *q) { store_elem(q, 0, DT, load_elem(q, 0, DT) * c * power); });
}

}  // namespace

// parts[blockIdx.x]: the sum of squares of the workgroup's four spans
__global__ __launch_bounds__(kThreads) void grad_squares_kernel(const GradTable t, double *parts) {
    __shared__ double red[kThreads / kWave];
    double sum = 0.0;
    each_block(t, [&](int dt, char *p, int size) {
        if (dt == PRIME_BF16) sum += square_sum<PRIME_BF16>(p, size);
        else if (dt == PRIME_F16) sum += square_sum<PRIME_F16>(p, size);
        else sum += square_sum<PRIME_F32>(p, size);
    });
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

__device__ __forceinline__ double parts_sum(const double *parts, int count, double *red) {
    constexpr int U = 8;
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += U * kThreads) {
        double x[U];  // all loads first
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = parts[min(i + u * kThreads, count - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) sum += i + u * kThreads < count ? x[u] : 0.0;
    }
    return block_sum(sum, red);
}

// One workgroup: the norm, and the whole sum in parts[0] for the scaling of several tables.
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(double *parts, int count, float *norm) {
    __shared__ double red[kThreads / kWave];
    const double sum = parts_sum(parts, count, red);  // (behind its barriers all parts are read)
    if (threadIdx.x != 0) return;
    *norm = static_cast<float>(sqrt(sum));
    if (count) parts[0] = sum;
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
    // One fp32 number would lose bits of a factor near fp32's least or below it: then 2^100 times
    // the factor, and the power of two, which rounds nothing more, behind the product.
    const double factor = max_norm / (total + 1e-6);
    if (static_cast<float>(factor) >= 1.f || max_norm == __builtin_inf()) return;  // (a NaN scales)
    const float power = factor < 0x1p-100 ? 0x1p-100f : 1.f, c = static_cast<float>(factor / power);
    each_block(t, [&](int dt, char *p, int size) {
        if (dt == PRIME_BF16) scale_block<PRIME_BF16>(p, size, c, power);
        else if (dt == PRIME_F16) scale_block<PRIME_F16>(p, size, c, power);
        else scale_block<PRIME_F32>(p, size, c, power);
    });
}

hipError_t launch_grad_squares(const GradTable &t, int blocks, double *parts, hipStream_t stream) {
    hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(kThreads), 0, stream, t, parts);
    return hipGetLastError();
}
hipError_t launch_grad_norm(double *parts, int count, float *norm, hipStream_t stream) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kThreads), 0, stream, parts, count, norm);
    return hipGetLastError();
}
hipError_t launch_grad_scale(const GradTable &t, int blocks, const double *parts, int count, float *norm,
                             double max_norm, hipStream_t stream) {
    hipLaunchKernelGGL(grad_scale_kernel, dim3(blocks), dim3(kThreads), 0, stream, t, parts, count, norm, max_norm);
    return hipGetLastError();
}

}  // namespace prime
