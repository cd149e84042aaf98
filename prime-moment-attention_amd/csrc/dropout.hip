// Dropout with the residual add, its mask never stored:
//   out = residual + (keep ? x / (1 - p) : 0)
// Element e (counted over the rows, whatever their strides) is kept where its 16
// random bits are at least n = round(65536 p); 1 - p is 1 - n / 65536, so the
// expectation is exact.  The bits of elements 8 j .. 8 j + 7 are the four words,
// low halves first, of one block of Philox4x32-10 (J. Salmon, M. Moraes, R. Dror,
// D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011: the rounds and the
// constants are the paper's) with counter (j, offset + call) and key seed.

#include "prime_kernels.h"

namespace prime {

// Ten rounds; k is the same in every lane.
__device__ __forceinline__ void philox(uint64_t block, uint64_t counter, uint64_t seed, uint32_t (&w)[4]) {
    uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32);
    uint32_t c2 = static_cast<uint32_t>(counter), c3 = static_cast<uint32_t>(counter >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(p0);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

__global__ __launch_bounds__(256) void dropout_add_kernel(const DropoutArgs a) {
    const int64_t block = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, total = a.rows * a.cols;
    if (block * 8 >= total) return;
    uint32_t w[4];
    philox(block, static_cast<uint64_t>(a.rng[1]) + static_cast<uint64_t>(a.call), static_cast<uint64_t>(a.rng[0]), w);
    int64_t row = block * 8 / a.cols, col = block * 8 % a.cols;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (block * 8 + j < total) {
            const uint32_t bits = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
            float v = bits >= a.cut ? load_elem(a.x, row * a.ldx + col, a.dt) * a.scale : 0.f;
            if (a.residual) v += load_elem(a.residual, row * a.ldr + col, a.dt);
            store_elem(a.out, row * a.ldo + col, a.dt, v);
        }
        if (++col == a.cols) col = 0, ++row;
    }
}

hipError_t launch_dropout_add(const DropoutArgs &a, hipStream_t stream) {
    const int64_t blocks = (a.rows * a.cols + 7) / 8;
    hipLaunchKernelGGL(dropout_add_kernel, dim3(static_cast<unsigned>((blocks + 255) / 256)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace prime
