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
constexpr double kLightest = -43.5;    // a token of weight 2^-43.5 or less has mass 0
constexpr float kBucketSpan = 30.5f;  // so has one this many T below the largest
constexpr float kInf = __builtin_inff();

// order-preserving image of a logit, -0 as +0
__device__ __forceinline__ uint32_t logit_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// a b + c with c from scalar registers (left alone, the compiler copies c into the
// accumulator first: a move for every multiply-add)
__device__ __forceinline__ double fma_s(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// What the tokens of a row are weighed by.
struct RowScale {
    float top;        // the largest logit
    double rate;      // log2(e) / T
    double least;     // log2 of min_p, at least kLightest
    float per_half;   // buckets per half a unit of the logit

    __device__ __forceinline__ double exponent(float x) const {  // of 2, at most 0
        return (static_cast<double>(x) - static_cast<double>(top)) * rate;
    }
    // 2^t as a mass, -44 <= t <= 0 (below, the result means nothing): 2^f on |f| <= 1/2 by
    // its Chebyshev interpolant of degree 9 (1.4e-14 off), scaled and rounded to a whole
    // number by one addition to 2^52.
    __device__ static __forceinline__ uint64_t mass_of(double t) {
        constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: adding it rounds to a whole number
        const double r = t + kRound, f = t - (r - kRound);
        double p = fma_s(1.0212097549811005e-07, f, 1.3259945262689143e-06);
        p = fma_s(p, f, 1.5252640059770786e-05);
        p = fma_s(p, f, 0.00015403432339553542);
        p = fma_s(p, f, 0.001333355825801874);
        p = fma_s(p, f, 0.009618129195951041);
        p = fma_s(p, f, 0.05550410866428854);
        p = fma_s(p, f, 0.24022650695631514);
        p = fma_s(p, f, 0.6931471805599526);
        p = fma(p, f, 1.0);
        const uint32_t n = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, r));  // low word: the whole number
        const double scale = __builtin_bit_cast(double, static_cast<uint64_t>((n + 1023u + 42u) << 20) << 32);
        uint64_t w = __builtin_bit_cast(uint64_t, fma(p, scale, 4503599627370496.0)) - 0x4330000000000000ull;
        asm("" : "+v"(w));  // computed for every token: a branch around it costs more than it saves
        return w;
    }
    __device__ __forceinline__ uint64_t mass(float x) const {
        const double t = exponent(x);
        return select(t >= kLightest, mass_of(t));
    }
    __device__ static __forceinline__ uint64_t select(bool keep, uint64_t w) { return keep ? w : 0; }
    // bucket of x, false for tokens whose mass is 0 (and for NaN); monotone: every step is
    __device__ __forceinline__ bool bucket(float x, int &b) const {
        const float f = fmaf(-0.5f, x, 0.5f * top) * per_half;
        b = static_cast<int>(f);
        return f < static_cast<float>(kBuckets - 1);
    }
};

// v of lane 63
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
    return static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63)) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {  // 0 where the move has no source
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xF, false);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
// inclusive sum over the lanes, on the vector unit: shifts within rows of 16, then the last
// lane of row 0 (2) into row 1 (3), then lane 31 into rows 2 and 3
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
    v += dpp_u64<0x111, 0xF>(v);
    v += dpp_u64<0x112, 0xF>(v);
    v += dpp_u64<0x114, 0xF>(v);
    v += dpp_u64<0x118, 0xF>(v);
    v += dpp_u64<0x142, 0xA>(v);
    v += dpp_u64<0x143, 0xC>(v);
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
    int bucket, n, index, owner;
    bool whole;
};

// exclusive sum over the threads, the sum over the waves before, and the total
template <int WAVES>
__device__ __forceinline__ uint64_t block_scan(SampleShared<WAVES> &sh, uint64_t v, uint64_t &waves, uint64_t &total) {
    const uint64_t inc = wave_scan_u64(v);
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == kWave - 1) sh.part[wave] = inc;
    __syncthreads();
    waves = total = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const uint64_t p = sh.part[i];
        waves += i < wave ? p : 0;
        total += p;
    }
    return waves + inc - v;
}

// A row: wave w has the chunks [w per, (w + 1) per) of 64 lanes with VE elements each.
// Elements past the vocabulary are -infinity.
// The first `staged` chunks of every wave are in LDS once stage() has run.
template <int DT>
struct SampleRow {
    static constexpr int VE = DT == PRIME_F32 ? 4 : 8, es = DT == PRIME_F32 ? 4 : 2;
    const char *base;
    int vocab, per, start;  // start: the lane's first element
    bool wide;              // 16-byte loads
    u32x4 *lds;             // the lane's place in the staged chunks, `lds_step` between two
    int staged, lds_step;

    __device__ __forceinline__ int index(int i) const { return start + i * (kWave * VE); }
    __device__ __forceinline__ u32x4 fetch(int i) const { return i < staged ? lds[i * lds_step] : load(i); }
    __device__ __forceinline__ u32x4 load(int i) const {
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
        }
    }
    // f(i, x) over the lane's chunks, U loads in flight
    template <int U, typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int i0 = 0; i0 < per; i0 += U) {
            u32x4 v[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (i0 + k < per) v[k] = fetch(i0 + k);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (i0 + k < per) {
                    float x[VE];
                    widen(v[k], x);
                    f(i0 + k, x);
                }
            }
        }
    }
    // the first pass: f over the row as it comes from memory, into LDS what has place there
    template <typename F>
    __device__ __forceinline__ void stage(F f) {
        constexpr int U = 8;
        for (int i0 = 0; i0 < per; i0 += U) {
            u32x4 v[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (i0 + k < per) v[k] = load(i0 + k);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (i0 + k >= per) continue;
                if (i0 + k < staged) lds[(i0 + k) * lds_step] = v[k];
                float x[VE];
                widen(v[k], x);
                f(i0 + k, x);
            }
        }
    }
    // the same for passes with much to compute, the next load under way
    template <typename F>
    __device__ __forceinline__ void each_heavy(F f) const {
        u32x4 next = fetch(0);
        for (int i = 0; i < per; ++i) {
            const u32x4 now = next;
            if (i + 1 < per) next = fetch(i + 1);
            float x[VE];
            widen(now, x);
            f(i, x);
        }
    }
};

// How many tokens are equal to `value`; `nth` of that count gives n, and the index of the
// n-th of them, from 1, is returned (any index where there are fewer).
template <int DT, int WAVES, typename F>
__device__ __forceinline__ int find_equal(SampleShared<WAVES> &sh, const SampleRow<DT> &row, float value, F nth) {
    constexpr int VE = SampleRow<DT>::VE;
    uint64_t count = 0, before, total;
    row.template each<4>([&](int, const float (&x)[VE]) {
#pragma unroll
        for (int j = 0; j < VE; ++j) count += x[j] == value;
    });
    block_scan(sh, count, before, total);
    const uint64_t n = nth(total);
    if (before < n && n <= before + sh.part[threadIdx.x / kWave]) {
        // this wave's chunks one after the other, lanes in order within one
        int left = static_cast<int>(n - before);
        row.template each<4>([&](int i, const float (&x)[VE]) {
            int all = 0, lower = 0;  // of the chunk, of the lanes below
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const uint64_t b = __ballot(x[j] == value);
                all += __popcll(b);
                lower += __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(b >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(b), 0));
            }
            int skip = left - lower;  // the skip-th of this lane's is the one
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (x[j] == value && --skip == 0) sh.index = row.index(i) + j;
            left -= all;
        });
    }
    __syncthreads();
    return sh.index;
}

// The cut: over the tokens above `last` and `ties` tokens equal to it (none for -infinity),
// in rank order, the shortest prefix with weight of at least wanted(sum of all weights).
// WEIGH: masses, else ones.  Left as it is where all of them are needed.  whole: the tokens
// equal to the new `last` are known to be all kept.
template <bool WEIGH, int DT, int WAVES, typename F>
__device__ __forceinline__ void cut(SampleShared<WAVES> &sh, const SampleRow<DT> &row, const RowScale &rs,
                                    float &last, uint64_t &ties, bool &whole, F wanted) {
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
    auto fill = [&](int, const float (&x)[VE]) {
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
    };
    if constexpr (WEIGH) row.each_heavy(fill);
    else row.template each<4>(fill);
    int floor_b = -1;
    if (floor_w && !rs.bucket(floor, floor_b)) floor_b = -1;
    if (tid == 0 && floor_b >= 0) add(&sh.hist[floor_b], floor_w);
    __syncthreads();
    uint64_t mine = 0, waves, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += sh.hist[tid * kPer + i];
    uint64_t before = block_scan(sh, mine, waves, total);
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
    row.template each<4>([&](int, const float (&x)[VE]) {
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
    // `over`: the weight of the tokens above x; `equal`: of those equal to it, where known
    auto found = [&](float x, uint64_t over, uint64_t equal) {
        const uint64_t w = WEIGH ? rs.mass(x) : 1, n = (want - over + w - 1) / w;
        sh.last = x;
        sh.ties = n;
        sh.whole = x != floor && n * w == equal;
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
            if (over < want && want <= over + equal) found(x, over, equal);
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
            row.each_heavy([&](int, const float (&x)[VE]) {
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
        if (tid == 0) found(key_logit(prefix), over, 0);
    }
    __syncthreads();
    last = sh.last;
    ties = sh.ties;
    whole = sh.whole;
}

template <int DT, int WAVES, int STAGED>
__global__ __launch_bounds__(WAVES *kWave) void sample_kernel(const SampleArgs a) {
    __shared__ SampleShared<WAVES> sh;
    __shared__ u32x4 stage[STAGED > 0 ? STAGED * WAVES * kWave : 1];
    using Row = SampleRow<DT>;
    constexpr int VE = Row::VE;
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave), r = blockIdx.x;
    Row row;
    row.base = static_cast<const char *>(a.logits) + r * a.stride_n * Row::es;
    row.vocab = a.vocab;
    row.per = (a.vocab + WAVES * kWave * VE - 1) / (WAVES * kWave * VE);
    row.start = (wave * row.per * kWave + lane) * VE;
    row.wide = reinterpret_cast<uintptr_t>(row.base) % 16 == 0;
    row.staged = STAGED;
    row.lds = stage + tid;
    row.lds_step = WAVES * kWave;
    const float T = a.temperatures ? a.temperatures[r] : a.temperature;
    const float top_p = a.top_ps ? a.top_ps[r] : a.top_p, min_p = a.min_ps ? a.min_ps[r] : a.min_p;
    int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    const double u = a.uniforms[r];
    if (top_k <= 0 || top_k > a.vocab) top_k = a.vocab;

    // the largest logit (fmaxf passes over NaN)
    RowScale rs;
    float top = -kInf;
    row.stage([&](int, const float (&x)[VE]) {
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
        row.template each<4>([&](int i, const float (&x)[VE]) {
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
    if (top == kInf) {  // the infinite ones share the weight
        const int index = find_equal(sh, row, top, [&](uint64_t n) {
            if (n > static_cast<uint64_t>(top_k)) n = top_k;
            if (top_p < 1.f) n = (share(n * kMass) + kMass - 1) / kMass;
            return target_of(n * kMass) / kMass + 1;
        });
        if (tid == 0) a.out[r] = index;
        return;
    }
    rs.top = top;
    rs.rate = 1.4426950408889634074 / static_cast<double>(T);
    rs.least = min_p > 0.f ? fmax(log2(static_cast<double>(min_p < 1.f ? min_p : 1.f)), kLightest) : kLightest;
    rs.per_half = fminf(2.f * (kBuckets - 1) / (kBucketSpan * T), 1e30f);

    // kept are the tokens above `last`; where the cut runs through equal ones (split), also
    // those equal to it up to tie_index
    float last = -kInf;
    uint64_t ties = 0;
    bool whole = true;
    if (top_k < a.vocab) cut<false>(sh, row, rs, last, ties, whole, [&](uint64_t) { return static_cast<uint64_t>(top_k); });
    if (top_p < 1.f) cut<true>(sh, row, rs, last, ties, whole, share);
    int tie_index = -1;
    bool split = ties && !whole;
    if (split)
        tie_index = find_equal(sh, row, last, [&](uint64_t total) {
            split = total > ties;
            return ties;
        });
    // all tokens equal to `last` are kept: the ones above the next value below it (below 0
    // that is not -0)
    if (ties && !split) last = key_logit(logit_key(last) - (last == 0.f ? 2 : 1));

    auto token_mass = [&](float x, int index, bool equals) -> uint64_t {
        const double t = rs.exponent(x);
        const uint64_t w = RowScale::mass_of(t);
        bool keep = x > last;
        if (equals) keep |= (x == last) & (index <= tie_index);
        return RowScale::select(keep & (t >= rs.least), w);
    };
    auto chunk_mass = [&](int i, const float (&x)[VE]) {
        float most = x[0];
        uint64_t sum = 0;
#pragma unroll
        for (int j = 1; j < VE; ++j) most = fmaxf(most, x[j]);
        if (most >= last) {
            if (split) {
#pragma unroll
                for (int j = 0; j < VE; ++j) sum += token_mass(x[j], row.index(i) + j, true);
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j) sum += token_mass(x[j], 0, false);
            }
        }
        return sum;
    };
    uint64_t mine = 0, total, before;
    row.each_heavy([&](int i, const float (&x)[VE]) { mine += chunk_mass(i, x); });
    block_scan(sh, mine, before, total);
    const uint64_t target = target_of(total);
    // the wave with the token, then its chunks, taken by all waves 64 lanes' sums each
    if (lane == 0 && before <= target && target - before < sh.part[wave]) sh.owner = wave, sh.sum = before;
    __syncthreads();
    before = sh.sum;
    const int shift = sh.owner - wave;
    row.start += shift * row.per * (kWave * VE);
    row.lds += shift * kWave;
    constexpr int kRound = kBuckets / kWave;  // chunks whose sums fit
    for (int i0 = 0; i0 < row.per; i0 += kRound) {
        const int n = min(kRound, row.per - i0);
        __syncthreads();
        for (int i = wave; i < n; i += WAVES) {
            float x[VE];
            row.widen(row.fetch(i0 + i), x);
            sh.hist[i * kWave + lane] = chunk_mass(i0 + i, x);
        }
        __syncthreads();
        if (wave) continue;
        // in order: lane by lane, chunk by chunk; here a lane takes n sums in a row
        uint64_t sum = 0;
        for (int k = 0; k < n; ++k) sum += sh.hist[lane * n + k];
        const uint64_t inc = wave_scan_u64(sum);
        uint64_t at = before + inc - sum;
        if (at <= target && target < before + inc) {
            int k = lane * n;
            while (target - at >= sh.hist[k]) at += sh.hist[k++];
            // sum k is lane k % 64's of chunk k / 64
            const int other = k % kWave - lane;
            SampleRow<DT> its = row;
            its.start += other * VE;
            its.lds += other;
            float x[VE];
            its.widen(its.fetch(i0 + k / kWave), x);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const int index = its.index(i0 + k / kWave) + j;
                const uint64_t m = token_mass(x[j], index, split);
                if (at <= target && target < at + m) a.out[r] = index;
                at += m;
            }
        }
        before += last_lane(inc);
    }
}

namespace {

template <int DT, int WAVES, int STAGED>
void launch(const SampleArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((sample_kernel<DT, WAVES, STAGED>), dim3(a.n), dim3(WAVES * kWave), 0, s, a);
}

template <int DT>
void run(const SampleArgs &a, hipStream_t s) {
    if (a.vocab <= kSampleSmall) launch<DT, 4, DT == PRIME_F32 ? 4 : 2>(a, s);
    else if (a.n <= 256) launch<DT, 16, 8>(a, s);
    else launch<DT, 16, 0>(a, s);
}

}  // namespace

hipError_t launch_sample(const SampleArgs &a, hipStream_t stream) {
    if (a.dt == PRIME_BF16) run<PRIME_BF16>(a, stream);
    else if (a.dt == PRIME_F16) run<PRIME_F16>(a, stream);
    else run<PRIME_F32>(a, stream);
    return hipGetLastError();
}

}  // namespace prime
