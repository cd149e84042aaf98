// Dropout with the residual add, its mask never stored:
//   out = residual + (keep ? x / (1 - p) : 0)
// Element e (counted over the rows, whatever their strides) is kept where its 16
// random bits are at least n = round(65536 p); 1 - p is 1 - n / 65536, so the
// expectation is exact.  The bits of elements 8 j .. 8 j + 7 are the four words,
// low halves first, of one block of Philox4x32-10 (J. Salmon, M. Moraes, R. Dror,
// D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011: the rounds and the
// constants are the paper's) with counter (j, offset + call) and key seed.
//
// Bound by memory: 65536 x 768 bf16 moves 302 MB in 47 us (6.4 TB/s) with a residual and 201 MB
// in 33 us (6.0 TB/s) without; the ten rounds, some 60 integer instructions for eight
// elements, hide behind the loads.  Two or four blocks a lane: 48 and 49 us, and 0.4 and 0.9 us
// more at 1000 x 513 (3.3 us).  Element by element, as rows take that start anywhere: 179 us.
// The loads past the caches: 106 us for fp32 with plain ones, 105 with these (without a
// residual 73, 68; for bf16 31, 33); stores past them too: 111.

#include "prime_kernels.h"

namespace prime {

constexpr int kDropThreads = 256;

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

__device__ __forceinline__ bool kept(const uint32_t (&w)[4], int j, uint32_t cut) {
    return (j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu) >= cut;
}

// One lane, eight elements: a 16-byte access in 16-bit types, two in fp32.
template <int DT>
struct Eight {
    static constexpr int N = DT == PRIME_F32 ? 2 : 1;
    u32x4 v[N];
    __device__ __forceinline__ void load(const void *p, int64_t e) {
        const u32x4 *q = reinterpret_cast<const u32x4 *>(static_cast<const char *>(p) + e * (2 * N));
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __builtin_nontemporal_load(q + i);
    }
    __device__ __forceinline__ void store(void *p, int64_t e) const {
        u32x4 *q = reinterpret_cast<u32x4 *>(static_cast<char *>(p) + e * (2 * N));
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = v[i];
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (DT == PRIME_F32) return __uint_as_float(v[j / 4][j % 4]);
        const uint32_t u = v[0][j / 2];
        if constexpr (DT == PRIME_BF16) return __uint_as_float(j & 1 ? u & 0xFFFF0000u : u << 16);
        return h16_bits_to_f32(static_cast<uint16_t>(j & 1 ? u >> 16 : u));
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j += DT == PRIME_F32 ? 1 : 2) {
            if constexpr (DT == PRIME_F32) v[j / 4][j % 4] = __float_as_uint(f[j]);
            else if constexpr (DT == PRIME_BF16) v[0][j / 2] = f32_to_bf16_bits(f[j]) | static_cast<uint32_t>(f32_to_bf16_bits(f[j + 1])) << 16;
            else v[0][j / 2] = f32_to_h16_bits(f[j]) | static_cast<uint32_t>(f32_to_h16_bits(f[j + 1])) << 16;
        }
    }
};

// Rows whose blocks of eight start on 16 bytes.  FLAT: the rows lie one after the other, so
// the elements are one row of any length.  The loads first, the random bits while they are
// under way.
template <int DT, bool RES, bool FLAT>
__global__ __launch_bounds__(kDropThreads) void dropout_add_kernel(const DropoutArgs a) {
    const int64_t block = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x, e = block * 8, total = a.rows * a.cols;
    if (e >= total) return;
    int64_t ox = e, orr = e, oo = e;
    if constexpr (!FLAT) {
        const int64_t row = e / a.cols, col = e % a.cols;
        ox = row * a.ldx + col, orr = row * a.ldr + col, oo = row * a.ldo + col;
    }
    const bool all = !FLAT || e + 8 <= total;
    Eight<DT> x, r;
    if (all) {
        x.load(a.x, ox);
        if constexpr (RES) r.load(a.residual, orr);
    }
    uint32_t w[4];
    philox(block, static_cast<uint64_t>(a.rng[1]) + static_cast<uint64_t>(a.call), static_cast<uint64_t>(a.rng[0]), w);
    if (all) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            f[j] = kept(w, j, a.cut) ? x.get(j) * a.scale : 0.f;
            if constexpr (RES) f[j] += r.get(j);
        }
        x.set(f);
        x.store(a.out, oo);
    } else {  // the last elements of one long row
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (e + j >= total) continue;
            float f = kept(w, j, a.cut) ? load_elem(a.x, e + j, DT) * a.scale : 0.f;
            if constexpr (RES) f += load_elem(a.residual, e + j, DT);
            store_elem(a.out, e + j, DT, f);
        }
    }
}

// Any rows: element by element.
__global__ __launch_bounds__(kDropThreads) void dropout_any_kernel(const DropoutArgs a) {
    const int64_t block = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x, total = a.rows * a.cols;
    if (block * 8 >= total) return;
    uint32_t w[4];
    philox(block, static_cast<uint64_t>(a.rng[1]) + static_cast<uint64_t>(a.call), static_cast<uint64_t>(a.rng[0]), w);
    int64_t row = block * 8 / a.cols, col = block * 8 % a.cols;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (block * 8 + j < total) {
            float v = kept(w, j, a.cut) ? load_elem(a.x, row * a.ldx + col, a.dt) * a.scale : 0.f;
            if (a.residual) v += load_elem(a.residual, row * a.ldr + col, a.dt);
            store_elem(a.out, row * a.ldo + col, a.dt, v);
        }
        if (++col == a.cols) col = 0, ++row;
    }
}

namespace {

template <int DT>
void run(const DropoutArgs &a, bool flat, dim3 grid, hipStream_t s) {
    const dim3 block(kDropThreads);
    if (a.residual && flat) hipLaunchKernelGGL((dropout_add_kernel<DT, true, true>), grid, block, 0, s, a);
    else if (a.residual) hipLaunchKernelGGL((dropout_add_kernel<DT, true, false>), grid, block, 0, s, a);
    else if (flat) hipLaunchKernelGGL((dropout_add_kernel<DT, false, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((dropout_add_kernel<DT, false, false>), grid, block, 0, s, a);
}

}  // namespace

hipError_t launch_dropout_add(const DropoutArgs &a, hipStream_t stream) {
    const int64_t blocks = (a.rows * a.cols + 7) / 8, es = a.dt == PRIME_F32 ? 4 : 2;
    const dim3 grid(static_cast<unsigned>((blocks + kDropThreads - 1) / kDropThreads));
    auto starts = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    auto aligned = [&](const void *p, int64_t ld) { return starts(p) && ld * es % 16 == 0; };
    const bool flat = a.rows == 1 || (a.ldx == a.cols && a.ldo == a.cols && (!a.residual || a.ldr == a.cols));
    const bool wide = flat ? starts(a.x) && starts(a.out) && starts(a.residual)
                           : a.cols % 8 == 0 && aligned(a.x, a.ldx) && aligned(a.out, a.ldo) &&
                                 (!a.residual || aligned(a.residual, a.ldr));
    if (!wide) hipLaunchKernelGGL(dropout_any_kernel, grid, dim3(kDropThreads), 0, stream, a);
    else if (a.dt == PRIME_BF16) run<PRIME_BF16>(a, flat, grid, stream);
    else if (a.dt == PRIME_F16) run<PRIME_F16>(a, flat, grid, stream);
    else run<PRIME_F32>(a, flat, grid, stream);
    return hipGetLastError();
}

}  // namespace prime
