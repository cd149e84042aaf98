// One token per row of logits from one given uniform number: temperature, top-k,
// top-p and min-p.  Tokens are ranked by logit, equal ones by index; the kept set is
// a prefix of that ranking: the tokens above a value `last`, and of those equal to it
// the ones up to an index.  The token is the first kept one, by index, whose running
// mass exceeds uniform * (mass of the kept set).
//
// Masses are whole numbers, w = rint(2^42 exp((x - max) / T)), the exponential in fp64:
// sums are exact, so their order does not matter and shared-memory atomics give the same
// token every time, and a border is missed by at most 2^-42 of the largest mass per
// token.  A vocabulary of up to 2^20 keeps every sum below 2^62.
//
// One workgroup a row, a contiguous part a wave; every pass reads the row again, from the
// caches after the first.  The ranking is never sorted.  A cut
// adds weights (ones for top-k, masses for top-p) into buckets of equal width in the logit,
// finds the bucket in which the wanted sum is reached, and compares the tokens of that one
// bucket with each other; should it hold too many, a radix descent over the
// order-preserving keys of all tokens takes its place.

#include "prime_kernels.h"

namespace prime {

constexpr uint64_t kMass = 1ull << 42;  // the largest token's
constexpr int kBuckets = 2048, kList = 1024;
constexpr int kSampleSmall = 4096;  // up to here a row takes 4 waves, else 16
constexpr float kBucketSpan = 30.5f;  // a token this many T below the largest has mass 0
constexpr float kInf = __builtin_inff();

// order-preserving image of a logit, -0 as +0
__device__ __forceinline__ uint32_t logit_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// What the tokens of a row are weighed by.
struct RowScale {
    float top;        // the largest logit
    double rate;      // log2(e) / T
    double least;     // log2 of min_p; -infinity without
    float per_half;   // buckets per half a unit of the logit

    __device__ __forceinline__ double exponent(float x) const {  // of 2, at most 0
        return (static_cast<double>(x) - static_cast<double>(top)) * rate;
    }
    // 2^t as a mass: 2^f on |f| <= 1/2 by its Chebyshev interpolant of degree 9 (1.4e-14
    // off), scaled and rounded to a whole number by one addition to 2^52.
    __device__ static __forceinline__ uint64_t mass_of(double t) {
        constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: adding it rounds to a whole number
        t = fmax(t, -64.0);
        const double r = t + kRound, f = t - (r - kRound);
        double p = 1.0212097549811005e-07;
        p = fma(p, f, 1.3259945262689143e-06);
        p = fma(p, f, 1.5252640059770786e-05);
        p = fma(p, f, 0.00015403432339553542);
        p = fma(p, f, 0.001333355825801874);
        p = fma(p, f, 0.009618129195951041);
        p = fma(p, f, 0.05550410866428854);
        p = fma(p, f, 0.24022650695631514);
        p = fma(p, f, 0.6931471805599526);
        p = fma(p, f, 1.0);
        const uint32_t n = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, r));  // low word: the whole number
        const double scale = __builtin_bit_cast(double, static_cast<uint64_t>((n + 1023u + 42u) << 20) << 32);
        return __builtin_bit_cast(uint64_t, fma(p, scale, 4503599627370496.0)) - 0x4330000000000000ull;
    }
    __device__ __forceinline__ uint64_t mass(float x) const { return mass_of(exponent(x)); }
    // bucket of x, false for tokens whose mass is 0 (and for NaN); monotone: every step is
    __device__ __forceinline__ bool bucket(float x, int &b) const {
        const float f = fmaf(-0.5f, x, 0.5f * top) * per_half;
        b = static_cast<int>(f);
        return f < static_cast<float>(kBuckets - 1);
    }
};

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int lane) {
    return static_cast<uint64_t>(__shfl(static_cast<uint32_t>(v >> 32), lane, kWave)) << 32 |
           __shfl(static_cast<uint32_t>(v), lane, kWave);
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {  // inclusive
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), o, kWave), hi = __shfl_up(static_cast<uint32_t>(v >> 32), o, kWave);
        if (lane >= o) v += static_cast<uint64_t>(hi) << 32 | lo;
    }
    return v;
}

template <int WAVES>
struct SampleShared {
    uint64_t hist[kBuckets];
    uint64_t list_w[kList];
    float list_x[kList];
    uint64_t part[WAVES];
    uint64_t sum, ties;
    float last;
    int bucket, n, index;
};

// exclusive sum over the threads, and the total
template <int WAVES>
__device__ __forceinline__ uint64_t block_scan(SampleShared<WAVES> &sh, uint64_t v, uint64_t &total) {
    const uint64_t inc = wave_scan_u64(v);
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == kWave - 1) sh.part[wave] = inc;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        if (i == wave) before = total;
        total += sh.part[i];
    }
    return before + inc - v;
}

// A row: wave w has the chunks [w per, (w + 1) per) of 64 lanes with VE elements each.
// Elements past the vocabulary are -infinity.
template <int DT>
struct SampleRow {
    static constexpr int VE = DT == PRIME_F32 ? 4 : 8, es = DT == PRIME_F32 ? 4 : 2;
    const char *base;
    int vocab, per, start;  // start: the lane's first element
    bool wide, infinite;    // 16-byte loads; some logit is +infinity: those are 0, all others -infinity

    __device__ __forceinline__ int index(int i) const { return start + i * (kWave * VE); }
    __device__ __forceinline__ u32x4 fetch(int i) const {
        constexpr uint32_t none = DT == PRIME_F32 ? 0xFF800000u : DT == PRIME_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
        const int e = index(i);
        u32x4 v = {none, none, none, none};
        if (wide && e + VE <= vocab) {
            v = *reinterpret_cast<const u32x4 *>(base + static_cast<int64_t>(e) * es);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                if (e + j >= vocab) continue;
                if constexpr (DT == PRIME_F32) {
                    v[j] = reinterpret_cast<const uint32_t *>(base)[e + j];
                } else {
                    const uint32_t h = reinterpret_cast<const uint16_t *>(base)[e + j];
                    v[j / 2] = j & 1 ? (v[j / 2] & 0xFFFFu) | h << 16 : (v[j / 2] & 0xFFFF0000u) | h;
                }
            }
        }
        return v;
    }
    __device__ __forceinline__ void widen(const u32x4 &v, float (&x)[VE]) const {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if constexpr (DT == PRIME_F32) x[j] = __uint_as_float(v[j]);
            else if constexpr (DT == PRIME_BF16) x[j] = __uint_as_float(j & 1 ? v[j / 2] & 0xFFFF0000u : v[j / 2] << 16);
            else x[j] = h16_bits_to_f32(static_cast<uint16_t>(j & 1 ? v[j / 2] >> 16 : v[j / 2]));
            if (infinite) x[j] = x[j] == kInf ? 0.f : -kInf;
        }
    }
    // f(i, x) over the lane's chunks, the next ones under way
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        constexpr int U = 2;
        u32x4 next[U];
#pragma unroll
        for (int k = 0; k < U; ++k) next[k] = fetch(k);
        for (int i0 = 0; i0 < per; i0 += U) {
            u32x4 now[U];
#pragma unroll
            for (int k = 0; k < U; ++k) now[k] = next[k], next[k] = fetch(i0 + U + k);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                float x[VE];
                widen(now[k], x);
                if (i0 + k < per) f(i0 + k, x);
            }
        }
    }
};

// The cut: over the tokens above `last` and `ties` tokens equal to it (none for -infinity),
// in rank order, the shortest prefix with weight of at least wanted(sum of all weights).
// WEIGH: masses, else ones.  Left as it is where all of them are needed.
template <bool WEIGH, int DT, int WAVES, typename F>
__device__ __forceinline__ void cut(SampleShared<WAVES> &sh, const SampleRow<DT> &row, const RowScale &rs,
                                    float &last, uint64_t &ties, F wanted) {
    constexpr int kThreads = WAVES * kWave, kPer = kBuckets / kThreads, VE = SampleRow<DT>::VE;
    const int tid = threadIdx.x;
    const float floor = last;
    const uint64_t floor_w = ties ? ties * (WEIGH ? rs.mass(floor) : 1) : 0;
    auto add = [](uint64_t *p, uint64_t w) {
        atomicAdd(reinterpret_cast<unsigned long long *>(p), static_cast<unsigned long long>(w));
    };
    __syncthreads();
    for (int b = tid; b < kBuckets; b += kThreads) sh.hist[b] = 0;
    if (tid == 0) sh.n = 0, sh.bucket = -1;
    __syncthreads();
    row.each([&](int, const float (&x)[VE]) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < VE; ++j) any |= x[j] > floor;
        if (!any) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            int b;
            const uint64_t w = WEIGH ? rs.mass(x[j]) : 1;
            if (rs.bucket(x[j], b) && x[j] > floor) add(&sh.hist[b], w);
        }
    });
    int floor_b = -1;
    if (floor_w && !rs.bucket(floor, floor_b)) floor_b = -1;
    if (tid == 0 && floor_b >= 0) add(&sh.hist[floor_b], floor_w);
    __syncthreads();
    uint64_t mine = 0, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += sh.hist[tid * kPer + i];
    uint64_t before = block_scan(sh, mine, total);
    const uint64_t want = wanted(total);
    if (want > total) return;  // (the same for every thread)
    if (before < want && want <= before + mine) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint64_t w = sh.hist[tid * kPer + i];
            if (before < want && want <= before + w) sh.bucket = tid * kPer + i, sh.sum = before;
            before += w;
        }
    }
    __syncthreads();
    const int bucket = sh.bucket;
    const uint64_t above = sh.sum;
    row.each([&](int, const float (&x)[VE]) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            int b;
            if (rs.bucket(x[j], b) && b == bucket && x[j] > floor) {
                const int n = atomicAdd(&sh.n, 1);
                if (n < kList) sh.list_x[n] = x[j], sh.list_w[n] = WEIGH ? rs.mass(x[j]) : 1;
            }
        }
    });
    if (tid == 0 && floor_b == bucket) {
        const int n = atomicAdd(&sh.n, 1);
        if (n < kList) sh.list_x[n] = floor, sh.list_w[n] = floor_w;
    }
    __syncthreads();
    const int n = sh.n;
    auto found = [&](float x, uint64_t over) {  // `over`: the weight of the tokens above x
        const uint64_t w = WEIGH ? rs.mass(x) : 1;
        sh.last = x;
        sh.ties = (want - over + w - 1) / w;
    };
    if (n <= kList) {
        for (int i = tid; i < n; i += kThreads) {
            const float x = sh.list_x[i];
            uint64_t over = above, equal = 0;
            for (int j = 0; j < n; ++j) {
                const float y = sh.list_x[j];
                const uint64_t w = sh.list_w[j];
                over += y > x ? w : 0;
                equal += y == x ? w : 0;
            }
            if (over < want && want <= over + equal) found(x, over);
        }
    } else {
        // the largest key with enough weight at and above it, eight bits at a time
        uint32_t prefix = 0;
        uint64_t over = 0;
        const uint32_t floor_key = logit_key(floor);
        for (int shift = 24; shift >= 0; shift -= 8) {
            auto inside = [&](uint32_t k) { return shift == 24 || (k ^ prefix) >> (shift + 8) == 0; };
            __syncthreads();
            if (tid < 256) sh.hist[tid] = 0;
            __syncthreads();
            row.each([&](int, const float (&x)[VE]) {
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const uint32_t k = logit_key(x[j]);
                    if (x[j] > floor && inside(k)) add(&sh.hist[k >> shift & 255], WEIGH ? rs.mass(x[j]) : 1);
                }
            });
            if (tid == 0 && floor_w && inside(floor_key)) add(&sh.hist[floor_key >> shift & 255], floor_w);
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                while (d > 0 && over + sh.hist[d] < want) over += sh.hist[d--];
                sh.sum = over;
                sh.n = static_cast<int>(prefix | static_cast<uint32_t>(d) << shift);
            }
            __syncthreads();
            over = sh.sum;
            prefix = static_cast<uint32_t>(sh.n);
        }
        if (tid == 0) found(key_logit(prefix), over);
    }
    __syncthreads();
    last = sh.last;
    ties = sh.ties;
}

template <int DT, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void sample_kernel(const SampleArgs a) {
    __shared__ SampleShared<WAVES> sh;
    using Row = SampleRow<DT>;
    constexpr int VE = Row::VE;
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave), r = blockIdx.x;
    Row row;
    row.base = static_cast<const char *>(a.logits) + r * a.stride_n * Row::es;
    row.vocab = a.vocab;
    row.per = (a.vocab + WAVES * kWave * VE - 1) / (WAVES * kWave * VE);
    row.start = (wave * row.per * kWave + lane) * VE;
    row.wide = reinterpret_cast<uintptr_t>(row.base) % 16 == 0;
    row.infinite = false;
    const float T = a.temperatures ? a.temperatures[r] : a.temperature;
    const float top_p = a.top_ps ? a.top_ps[r] : a.top_p, min_p = a.min_ps ? a.min_ps[r] : a.min_p;
    int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    const double u = a.uniforms[r];
    if (top_k <= 0 || top_k > a.vocab) top_k = a.vocab;

    // the largest logit (fmaxf passes over NaN)
    RowScale rs;
    float top = -kInf;
    row.each([&](int, const float (&x)[VE]) {
#pragma unroll
        for (int j = 0; j < VE; ++j) top = fmaxf(top, x[j]);
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
    if (lane == 0) sh.list_x[wave] = top;
    if (tid == 0) sh.index = a.vocab;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) top = fmaxf(top, sh.list_x[i]);

    // uniform * total as a whole number below total
    auto target_of = [&](uint64_t total) {
        const double t = u > 0.0 ? u * static_cast<double>(total) : 0.0;
        const uint64_t whole = t < static_cast<double>(total) ? static_cast<uint64_t>(t) : total - 1;
        return whole < total ? whole : total - 1;
    };
    auto share = [&](uint64_t total) {  // the weight that top_p asks for
        const double t = __builtin_ceil(static_cast<double>(top_p > 0.f ? top_p : 0.f) * static_cast<double>(total));
        const uint64_t want = static_cast<uint64_t>(t);
        return want < 1 ? 1 : want > total ? total : want;
    };
    if (top == -kInf) {  // nothing to choose from: all logits count as equal
        uint64_t n = T > 0.f ? top_k : 1;
        if (top_p < 1.f) n = (share(n * kMass) + kMass - 1) / kMass;
        if (tid == 0) a.out[r] = static_cast<int64_t>(target_of(n * kMass) / kMass);
        return;
    }
    if (!(T > 0.f) || top_k == 1 || top_p <= 0.f) {  // the first of the largest
        int first = a.vocab;
        row.each([&](int i, const float (&x)[VE]) {
#pragma unroll
            for (int j = VE - 1; j >= 0; --j)
                if (x[j] == top) first = min(first, row.index(i) + j);
        });
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) first = min(first, __shfl_xor(first, o, kWave));
        if (lane == 0) atomicMin(&sh.index, first);
        __syncthreads();
        if (tid == 0) a.out[r] = sh.index;
        return;
    }
    row.infinite = top == kInf;
    rs.top = row.infinite ? 0.f : top;
    rs.rate = 1.4426950408889634074 / static_cast<double>(T);
    rs.least = min_p > 0.f ? log2(static_cast<double>(min_p < 1.f ? min_p : 1.f)) : -1e300;
    rs.per_half = fminf(2.f * (kBuckets - 1) / (kBucketSpan * T), 1e30f);

    float last = -kInf;
    uint64_t ties = 0;
    if (top_k < a.vocab) cut<false>(sh, row, rs, last, ties, [&](uint64_t) { return static_cast<uint64_t>(top_k); });
    if (top_p < 1.f) cut<true>(sh, row, rs, last, ties, share);

    // the index up to which tokens equal to `last` are kept
    int tie_index = -1;
    if (ties) {
        int mine = 0;
        row.each([&](int, const float (&x)[VE]) {
#pragma unroll
            for (int j = 0; j < VE; ++j) mine += x[j] == last;
        });
        uint64_t total;
        const uint64_t in_wave = wave_scan_u64(mine);
        block_scan(sh, mine, total);
        tie_index = a.vocab;
        if (total > ties) {
            uint64_t before = 0;
            for (int i = 0; i < wave; ++i) before += sh.part[i];
            if (before < ties && ties <= before + shfl_u64(in_wave, kWave - 1)) {
                // this wave's chunks one after the other, lanes in order within one
                int left = static_cast<int>(ties - before);
                row.each([&](int i, const float (&x)[VE]) {
                    int n = 0;
#pragma unroll
                    for (int j = 0; j < VE; ++j) n += x[j] == last;
                    const int inc = static_cast<int>(wave_scan_u64(n)), all = __shfl(inc, kWave - 1, kWave);
                    int skip = left - (inc - n);  // the skip-th of this lane's is the one
                    if (left > 0 && skip >= 1 && skip <= n) {
#pragma unroll
                        for (int j = 0; j < VE; ++j)
                            if (x[j] == last && --skip == 0) sh.index = row.index(i) + j;
                    }
                    left -= all;
                });
            }
            __syncthreads();
            tie_index = sh.index;
        }
    }

    auto chunk_masses = [&](int i, const float (&x)[VE], uint64_t (&m)[VE]) {
        bool keep[VE], any = false;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            keep[j] = x[j] > last || (x[j] == last && row.index(i) + j <= tie_index);
            any |= keep[j];
            m[j] = 0;
        }
        if (!any) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const double t = rs.exponent(x[j]);
            const uint64_t w = RowScale::mass_of(t);
            m[j] = keep[j] && t >= rs.least ? w : 0;
        }
    };
    uint64_t mine = 0, total;
    row.each([&](int i, const float (&x)[VE]) {
        uint64_t m[VE];
        chunk_masses(i, x, m);
#pragma unroll
        for (int j = 0; j < VE; ++j) mine += m[j];
    });
    block_scan(sh, mine, total);
    const uint64_t target = target_of(total);
    uint64_t before = 0;
    for (int i = 0; i < wave; ++i) before += sh.part[i];
    if (target < before || target - before >= sh.part[wave]) return;
    // this wave has the token: its chunks one after the other
    bool done = false;
    row.each([&](int i, const float (&x)[VE]) {
        if (done) return;  // the same in every lane
        uint64_t m[VE], sum = 0;
        chunk_masses(i, x, m);
#pragma unroll
        for (int j = 0; j < VE; ++j) sum += m[j];
        const uint64_t inc = wave_scan_u64(sum), all = shfl_u64(inc, kWave - 1);
        if (target - before < all) {
            uint64_t at = before + inc - sum;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                if (at <= target && target < at + m[j]) a.out[r] = row.index(i) + j;
                at += m[j];
            }
            done = true;
        }
        before += all;
    });
}

namespace {

template <int DT>
void run(const SampleArgs &a, hipStream_t s) {
    if (a.vocab <= kSampleSmall) hipLaunchKernelGGL((sample_kernel<DT, 4>), dim3(a.n), dim3(4 * kWave), 0, s, a);
    else hipLaunchKernelGGL((sample_kernel<DT, 16>), dim3(a.n), dim3(16 * kWave), 0, s, a);
}

}  // namespace

hipError_t launch_sample(const SampleArgs &a, hipStream_t stream) {
    if (a.dt == PRIME_BF16) run<PRIME_BF16>(a, stream);
    else if (a.dt == PRIME_F16) run<PRIME_F16>(a, stream);
    else run<PRIME_F32>(a, stream);
    return hipGetLastError();
}

}  // namespace prime
