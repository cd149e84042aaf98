// One token per row of logits from one given uniform number: temperature, top-k,
// top-p and min-p.  Tokens are ranked by logit, equal ones by index; the kept set is
// a prefix of that ranking, described by the last kept value's key and how many
// tokens of that value (its first ones by index) are kept.  The token is the first
// kept one, by index, whose running mass exceeds uniform * (mass of the kept set).
//
// Masses are whole numbers, w = rint(2^42 exp((x - max) / T)) with the exponential
// in fp64: sums are exact, so their order does not matter and shared-memory atomics
// give the same token every time, and a border is missed by at most 2^-42 of the
// largest mass per token.  A vocabulary of up to 2^20 keeps every sum below 2^62.
//
// The ranking is never sorted: a radix descent over the order-preserving keys, eight
// bits at a time, finds the k-th key by counts and the key where top_p falls by masses.

#include "prime_kernels.h"

namespace prime {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / kWave;
constexpr double kMassOne = 4398046511104.0;  // 2^42

// order-preserving image of a logit; NaN counts as -infinity, -0 as +0
__device__ __forceinline__ uint32_t logit_key(float x) {
    if (x != x) x = -__builtin_inff();
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// exp(d), d <= 0, to the last bits of fp64: 2^n times the Taylor polynomial of
// degree 13 on |f| <= ln(2)/2 (next term 4e-18); 0 below e^-30, whose mass is 0.
__device__ __forceinline__ double exp_neg(double d) {
    if (!(d > -30.0)) return 0.0;
    const double n = __builtin_rint(d * 1.4426950408889634074);
    double f = fma(n, -0.69314718055994528623, d);
    f = fma(n, -2.3190468138462995584e-17, f);
    double p = 1.0 / 6227020800.0;
    p = fma(p, f, 1.0 / 479001600.0);
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
    return ldexp(p, static_cast<int>(n));
}

// What a row's tokens are weighed by.
struct RowScale {
    float top;       // the largest logit
    double inv_t;
    double min_w;    // least kept exp(), from min_p
    bool flat;       // no logit above -infinity: all count as equal

    __device__ __forceinline__ uint64_t mass(uint32_t key) const {
        if (flat) return static_cast<uint64_t>(kMassOne);
        const float x = key_logit(key);
        if (x == top) return static_cast<uint64_t>(kMassOne);
        if (x == -__builtin_inff()) return 0;
        const double e = exp_neg((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
        return static_cast<uint64_t>(__builtin_rint(e * kMassOne));
    }
    // whether min_p keeps it
    __device__ __forceinline__ bool heavy(uint32_t key) const {
        if (flat) return true;
        const float x = key_logit(key);
        if (x == top) return true;
        if (x == -__builtin_inff()) return false;
        return exp_neg((static_cast<double>(x) - static_cast<double>(top)) * inv_t) >= min_w;
    }
};

__device__ __forceinline__ uint64_t shfl_up_u64(uint64_t v, int o) {
    const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), o, kWave);
    const uint32_t hi = __shfl_up(static_cast<uint32_t>(v >> 32), o, kWave);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {  // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint64_t u = shfl_up_u64(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

struct SampleShared {
    uint64_t hist[256];
    uint64_t part[kSampleWaves];
    uint64_t value;
    uint32_t word;
};

// exclusive sum over the block's threads, and the total
__device__ __forceinline__ uint64_t block_scan(SampleShared &sh, uint64_t v, uint64_t &total) {
    const uint64_t inc = wave_scan_u64(v);
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.part[wave] = inc;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
    for (int i = 0; i < kSampleWaves; ++i) {
        if (i == wave) before = total;
        total += sh.part[i];
    }
    return before + inc - v;
}

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleArgs a) {
    __shared__ SampleShared sh;
    const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    const char *base = static_cast<const char *>(a.logits) + row * a.stride_n * (DT == PRIME_F32 ? 4 : 2);
    auto key_at = [&](int j) { return logit_key(load_elem(base, j, DT)); };
    const float T = a.temperatures ? a.temperatures[row] : a.temperature;
    const float top_p = a.top_ps ? a.top_ps[row] : a.top_p, min_p = a.min_ps ? a.min_ps[row] : a.min_p;
    int top_k = a.top_ks ? a.top_ks[row] : a.top_k;
    if (!(T > 0.f)) top_k = 1;
    if (top_k <= 0 || top_k > V) top_k = V;

    // the largest key
    uint32_t best = 0;
    for (int j = tid; j < V; j += kSampleThreads) best = max(best, key_at(j));
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) best = max(best, static_cast<uint32_t>(__shfl_xor(best, o, kWave)));
    if ((tid & 63) == 0) sh.part[tid >> 6] = best;
    __syncthreads();
    for (int i = 0; i < kSampleWaves; ++i) best = max(best, static_cast<uint32_t>(sh.part[i]));
    RowScale rs;
    rs.top = key_logit(best);
    rs.flat = rs.top == -__builtin_inff();
    rs.inv_t = T > 0.f ? 1.0 / static_cast<double>(T) : 1.0;
    rs.min_w = min_p > 0.f ? static_cast<double>(min_p < 1.f ? min_p : 1.f) : 0.0;

    // the kept prefix: keys above `last`, and the first `ties` tokens of key `last`
    uint32_t last = 0;
    uint64_t ties = 0;
    auto descend = [&](auto weight, uint64_t need, uint32_t floor_key, uint64_t floor_weight, uint32_t &key,
                       uint64_t &above) {
        // the largest key with weight(keys >= it) >= need; above = weight(keys > it).  Keys below
        // floor_key weigh nothing, floor_key itself floor_weight in all.
        uint32_t prefix = 0;
        above = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) sh.hist[tid] = 0;
            __syncthreads();
            for (int j = tid; j < V; j += kSampleThreads) {
                const uint32_t k = key_at(j);
                if ((shift == 24 || (k ^ prefix) >> (shift + 8) == 0) && k > floor_key)
                    atomicAdd(reinterpret_cast<unsigned long long *>(&sh.hist[k >> shift & 255]),
                              static_cast<unsigned long long>(weight(k)));
            }
            if (tid == 0 && floor_weight && (shift == 24 || (floor_key ^ prefix) >> (shift + 8) == 0))
                atomicAdd(reinterpret_cast<unsigned long long *>(&sh.hist[floor_key >> shift & 255]),
                          static_cast<unsigned long long>(floor_weight));
            __syncthreads();
            if (tid == 0) {
                uint64_t sum = above;
                int d = 255;
                while (d > 0 && sum + sh.hist[d] < need) sum += sh.hist[d--];
                sh.value = sum;
                sh.word = prefix | static_cast<uint32_t>(d) << shift;
            }
            __syncthreads();
            above = sh.value;
            prefix = sh.word;
        }
        key = prefix;
    };
    if (rs.flat) {
        last = best;
        ties = top_k;
    } else if (top_k < V) {
        uint64_t above;
        descend([](uint32_t) { return uint64_t(1); }, top_k, 0, 0, last, above);
        ties = top_k - above;
    }
    const bool cut_p = top_p < 1.f;
    if (cut_p) {
        uint64_t mine = 0, total;
        if (!rs.flat)
            for (int j = tid; j < V; j += kSampleThreads) {
                const uint32_t k = key_at(j);
                if (k > last) mine += rs.mass(k);
            }
        const uint64_t floor_mass = ties * rs.mass(last);
        block_scan(sh, mine, total);
        total += floor_mass;
        const double want = static_cast<double>(top_p > 0.f ? top_p : 0.f) * static_cast<double>(total);
        uint64_t need = static_cast<uint64_t>(__builtin_ceil(want));
        need = need < 1 ? 1 : need > total ? total : need;
        if (rs.flat) {
            ties = (need + static_cast<uint64_t>(kMassOne) - 1) / static_cast<uint64_t>(kMassOne);
        } else {
            uint32_t key;
            uint64_t above;
            descend([&](uint32_t k) { return rs.mass(k); }, need, last, floor_mass, key, above);
            const uint64_t w = rs.mass(key);
            last = key;
            ties = (need - above + w - 1) / w;
        }
    }

    // mass of the kept set, then the token: tiles of one element a thread in index order
    const uint32_t best_key = best;
    auto kept_mass = [&](uint32_t k, uint64_t tie_rank) -> uint64_t {
        if (rs.flat) return tie_rank < ties ? static_cast<uint64_t>(kMassOne) : 0;
        if (k < last || (k == last && tie_rank >= ties)) return 0;
        if (k != best_key && !rs.heavy(k)) return 0;
        return rs.mass(k);
    };
    uint64_t mine = 0, total, tie_before = 0;
    for (int j0 = 0; j0 < V; j0 += kSampleThreads) {
        const int j = j0 + tid;
        const uint32_t k = j < V ? key_at(j) : 0;
        const bool tie = j < V && (rs.flat || k == last);
        uint64_t tile_ties;
        const uint64_t rank = block_scan(sh, tie, tile_ties) + tie_before;
        tie_before += tile_ties;
        if (j < V) mine += kept_mass(k, rank);
    }
    block_scan(sh, mine, total);
    const double u = a.uniforms[row];
    const double at = u > 0.0 ? u * static_cast<double>(total) : 0.0;
    uint64_t target = at < static_cast<double>(total) ? static_cast<uint64_t>(at) : total - 1;
    target = target < total ? target : total - 1;
    uint64_t before = 0;
    tie_before = 0;
    for (int j0 = 0; j0 < V; j0 += kSampleThreads) {
        const int j = j0 + tid;
        const uint32_t k = j < V ? key_at(j) : 0;
        const bool tie = j < V && (rs.flat || k == last);
        uint64_t tile_ties, tile_mass;
        const uint64_t rank = block_scan(sh, tie, tile_ties) + tie_before;
        tie_before += tile_ties;
        const uint64_t m = j < V ? kept_mass(k, rank) : 0;
        const uint64_t lo = before + block_scan(sh, m, tile_mass);
        if (lo <= target && target < lo + m) a.out[row] = j;
        before += tile_mass;
        if (before > target) break;  // the same for every thread
    }
}

hipError_t launch_sample(const SampleArgs &a, hipStream_t stream) {
    const dim3 grid(a.n), block(kSampleThreads);
    if (a.dt == PRIME_BF16) hipLaunchKernelGGL(sample_kernel<PRIME_BF16>, grid, block, 0, stream, a);
    else if (a.dt == PRIME_F16) hipLaunchKernelGGL(sample_kernel<PRIME_F16>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(sample_kernel<PRIME_F32>, grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace prime
