// Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits,
// and the gradient of the first two.  With l = log2(e), C the row's largest logit times l and
//   d_j = x_j l - C,   S = sum_j 2^d_j,   T = sum_j 2^d_j d_j,   L = log2 S:
//   logprob = ln 2 (d_t - L),   entropy = ln 2 (L - T / S),   p_j = 2^(d_j - L)
//   dx_j = g (delta_jt - p_j) - h p_j (log p_j + entropy).
// d_j is one multiply-add, rounded once, and the same for whatever C is, so that C need not
// be the exact product: S, T and d_t are all relative to it.
//
// The sums of powers of 2 hold where the row's largest logit is between kLowest and kHighest: the
// product C is then below 2^24, so that rounding it moves all d_j by 1/2 at most, and 2^d, S, T and
// what rescales them stay finite.  References begin at kLowest, so that in such a row a mask, whatever
// its size, comes to 0.  Other rows (a largest logit beyond, infinities that are the largest, nothing
// but masks, NaN) are summed again by differences (Careful), two more passes over the row (512 x
// 50304 bf16 of such rows alone, with 5 alternatives and the entropy: 80 us, the ties of equal masks among
// them, for 17.5); the backward finds their largest and sum in place of C and L.
//
// A forward reads a row once, the likeliest tokens' vectors again; a backward reads it and writes
// its gradient.  8192 x 50304 bf16 (us on the device): 139 forward (824 MB, 5.9 TB/s, a read's
// rate; 164 while the caches write back the last gradient), 167 with 5 alternatives and the
// entropy, 250 backward behind it (1.65 GB, 6.6 TB/s).  A row has one compute unit, whose vector unit
// bounds few rows (2.6 us of exponentials and sums for 50304 logits, 11000 cycles of a
// workgroup's first 22000 with what it waits for), and each meeting of its waves costs
// some 0.3 us: 1 x 50304 5.8, with 5 alternatives 8.4, with 20 10.4; 256 x 50304 with 5 and the
// entropy 12.9.

#include <type_traits>

#include "prime_kernels.h"
#include "row_vec.h"

namespace prime {

namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -1e7f, kHighest = 1e7f;  // times log2(e) below 2^24
constexpr float kFar = -2e38f;                     // an exponent that may be the end of fp32
constexpr float kFloor = -1e4f;                    // 2^kFloor = 0: for 0 times an exponent of -infinity

// The reference C of a largest logit m, the same number wherever it is used: contracted into a
// difference it would be another one.
__device__ __forceinline__ float reference(float m) {
#pragma clang fp contract(off)
    const float c = m * kLog2e;
    return c;
}

// -0 as +0, NaN as -infinity: the order of the likeliest tokens
__device__ __forceinline__ uint32_t rank_key(float x) {
    if (x != x) x = -kInf;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Largest over the lanes, in every lane, on the vector unit.
__device__ __forceinline__ float wave_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
    x = fmaxf(x, xor_lane<8>(x));
    x = fmaxf(x, xor_lane<4>(x));
    x = fmaxf(x, xor_lane<2>(x));
    return fmaxf(x, xor_lane<1>(x));
}

// One row of a group of threads: WAVES waves of one workgroup, or (WAVES = 1) one wave of a
// workgroup that has several rows.
template <int WAVES>
struct Group {
    static constexpr int kThreads = WAVES * kWave;
    float *red;  // shared, 4 WAVES
    __device__ __forceinline__ int thread() const { return threadIdx.x % kThreads; }
    __device__ __forceinline__ void sync() const {
        if constexpr (WAVES > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __device__ float sum(float x) const {
        x = wave_sum(x);
        if constexpr (WAVES > 1) {
            sync();
            if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
            sync();
            x = red[0];
            for (int w = 1; w < WAVES; ++w) x += red[w];
        }
        return x;
    }
    __device__ float max(float x) const {
        x = wave_max(x);
        if constexpr (WAVES > 1) {
            sync();
            if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
            sync();
            x = red[0];
            for (int w = 1; w < WAVES; ++w) x = fmaxf(x, red[w]);
        }
        return x;
    }
    __device__ uint64_t max(uint64_t x) const {
        for (int o = 32; o; o >>= 1)
            x = max_u64(x, static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(x >> 32), o, kWave)) << 32 |
                               __shfl_xor(static_cast<uint32_t>(x), o, kWave));
        if constexpr (WAVES > 1) {
            uint64_t *r = reinterpret_cast<uint64_t *>(red);
            sync();
            if (threadIdx.x % kWave == 0) r[threadIdx.x / kWave] = x;
            sync();
            x = r[0];
            for (int w = 1; w < WAVES; ++w) x = max_u64(x, r[w]);
        }
        return x;
    }
};

// A row summed by differences from its largest value, which may be infinite.
struct Careful {
    float top, log_sum, mean;  // largest; log S; sum p (x - top)
    bool nan;
    __device__ __forceinline__ float diff(float x) const { return x == top ? 0.f : x - top; }
    __device__ __forceinline__ float logprob(float x) const {
        return nan ? __builtin_nanf("") : top == -kInf ? -kInf : diff(x) - log_sum;
    }
    __device__ __forceinline__ float entropy() const { return nan ? __builtin_nanf("") : top == -kInf ? 0.f : log_sum - mean; }
};

template <int DT, int WAVES>
__device__ __noinline__ Careful careful(const Group<WAVES> g, const char *row, int vocab) {
    Careful c;
    float top = -kInf, bad = 0.f, s = 0.f, t = 0.f;
    auto each = [&](auto f) {
        constexpr int U = 8;
        for (int j = g.thread(); j < vocab; j += U * g.kThreads) {
            float x[U];  // all loads first
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = load_elem(row, min(j + u * g.kThreads, vocab - 1), DT);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j + u * g.kThreads < vocab) f(x[u]);
        }
    };
    each([&](float x) {
        top = fmaxf(top, x);
        bad += x != x ? 1.f : 0.f;
    });
    c.top = g.max(top);
    c.nan = g.sum(bad) > 0.f;
    each([&](float x) {
        const float d = c.diff(x), e = __expf(d);
        s += e;
        t += e > 0.f ? e * d : 0.f;
    });
    s = g.sum(s), t = g.sum(t);
    c.log_sum = logf(s), c.mean = t / s;
    return c;
}

}  // namespace

namespace {

// What a group keeps in LDS.
template <int WAVES>
struct Shared {
    static constexpr int kList = WAVES == 1 ? 512 : 1024;
    __attribute__((aligned(16))) float red[4 * WAVES];
    uint64_t list[kList];
    float best[kWave];
    uint32_t count;
    static constexpr int kBatches = 8;
    float batch[kBatches][WAVES * kWave];  // each lane's largest of its first batches of vectors
};

// A value that at least `top` of the row's logits reach, and not many more: `best` is each
// lane's largest, `mine` the wave's, which is in sh.best.  The `top`-th largest of the j largest
// lanes of every wave: with W waves and j = top / W rounded up.
template <int WAVES>
__device__ __forceinline__ float threshold(const Group<WAVES> &g, Shared<WAVES> &sh, float best, float mine, int top) {
    const int lane = threadIdx.x % kWave;
    int count = WAVES;
#pragma unroll 1
    for (; count < top; count += WAVES) {
        if (lane == __builtin_ctzll(__ballot(best == mine))) best = -kInf;
        mine = wave_max(best);
        if (WAVES > 1 && lane == 0) sh.best[count + threadIdx.x / kWave] = mine;
    }
    if constexpr (WAVES == 1) return mine;
    if (count > WAVES) g.sync();
    const float x = lane < count ? sh.best[lane] : -kInf;
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < count; ++o) {
        const float y = sh.best[o];
        rank += y > x || (y == x && o < lane);
    }
    return sh.best[__builtin_ctzll(__ballot(lane < count && rank == top - 1))];
}

// The `top` first tokens in the order of rank_key, equal ones by index: write(rank, token,
// logit).  Those at the threshold or above are listed and ranked among each other; if they are
// too many, those above it, and the first ones equal to it by index (a row with few tokens that
// are not -infinity, or with equal logits); if these are too many, one after the other.
// A lane whose largest is below the threshold reads nothing again, another one only the batches
// and vectors whose largest is not.  (The last vectors kept in registers instead: 11.1 us for 8.8
// at 1 x 50304 with 5, 201 for 165 at 8192 rows with the entropy.)
// best, mine: the lane's and the wave's largest; tail: those of its vectors from `full` on.
template <int DT, int WAVES, int U, typename W>
__device__ __forceinline__ void likeliest(const Group<WAVES> &g, Shared<WAVES> &sh, const char *row, int vocab, int top,
                                          float best, float mine, int full, const float (&tail)[U], W write) {
    constexpr int VE = kVec<DT>, kThreads = WAVES * kWave, kList = Shared<WAVES>::kList;
    const int tid = g.thread(), whole = vocab / VE;
    const uint32_t bar = rank_key(threshold<WAVES>(g, sh, best, mine, top)), own = rank_key(best);
    auto gather = [&](uint32_t least) {  // how many have a key of at least `least`; the first kList are listed
        auto take = [&](float x, int j) {
            const uint32_t k = rank_key(x);
            if (k < least) return;
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < kList) sh.list[at] = static_cast<uint64_t>(k) << 32 | static_cast<uint32_t>(~j);
        };
        auto take_vector = [&](const u32x4 &v, int i) {
            float x[VE];
            widen<DT>(v, x);
#pragma unroll
            for (int e = 0; e < VE; ++e) take(x[e], i * VE + e);
        };
        if (own >= least) {
            int i = tid;
#pragma unroll 1
            for (int b = 0; i - tid < full; i += U * kThreads, ++b) {
                if (b < Shared<WAVES>::kBatches && rank_key(sh.batch[b][tid]) < least) continue;
                u32x4 v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = reinterpret_cast<const Raw *>(row)[i + u * kThreads].v;
#pragma unroll
                for (int u = 0; u < U; ++u) take_vector(v[u], i + u * kThreads);
            }
            uint32_t reach = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) reach |= (i + u * kThreads < whole && rank_key(tail[u]) >= least) << u;
#pragma unroll 1
            for (; reach; reach &= reach - 1) {
                const int at = i + __builtin_ctz(reach) * kThreads;
                take_vector(reinterpret_cast<const Raw *>(row)[at].v, at);
            }
            if (const int j = whole * VE + tid; j < vocab) take(load_elem(row, j, DT), j);
        }
        g.sync();
        return sh.count;
    };
    uint32_t count = gather(bar);
    int equal = 0;  // of the tokens at the threshold, how many are still wanted
    if (count > kList) {
        g.sync();
        if (tid == 0) sh.count = 0;
        g.sync();
        count = gather(bar + 1);
        equal = count < static_cast<uint32_t>(top) ? top - count : 0;
    }
    auto give = [&](int rank, uint64_t key) { write(rank, static_cast<int>(~static_cast<uint32_t>(key)), key_logit(key >> 32)); };
    if (count <= kList) {
        for (uint32_t c = tid; c < count; c += kThreads) {
            const uint64_t key = sh.list[c];
            int rank = 0;
#pragma unroll 4
            for (uint32_t o = 0; o < count; ++o) rank += sh.list[o] > key;
            if (rank < top) give(rank, key);
        }
        if (equal && tid < kWave) {  // one wave, in the order of the tokens
            int rank = top - equal;
            for (int j0 = 0; j0 < vocab && rank < top; j0 += kWave) {
                const int j = j0 + tid;
                const bool is = j < vocab && rank_key(load_elem(row, j, DT)) == bar;
                const uint64_t all = __ballot(is);
                const int at = rank + __popcll(all & ((1ull << tid) - 1));
                if (is && at < top) write(at, j, key_logit(bar));
                rank += __popcll(all);
            }
        }
        return;
    }
    uint64_t last = ~0ull;
#pragma unroll 1
    for (int r = 0; r < top; ++r) {
        uint64_t next = 0;
        for (int j = tid; j < vocab; j += kThreads) {
            const uint64_t key = static_cast<uint64_t>(rank_key(load_elem(row, j, DT))) << 32 | static_cast<uint32_t>(~j);
            if (key < last) next = max_u64(next, key);
        }
        last = g.max(next);
        if (tid == 0) give(r, last);
    }
}

}  // namespace

// WAVES > 1: one row a workgroup.  WAVES = 1: one row a wave, four a workgroup.
// A thread takes U vectors at once, whose largest logit then moves its reference once: 64 (32)
// logits a rescaling.
template <int DT, int WAVES, bool ENTROPY>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void logprobs_kernel(const LogprobsArgs a) {
    constexpr int VE = kVec<DT>, U = WAVES == 16 ? 8 : 4, es = DT == PRIME_F32 ? 4 : 2, kThreads = WAVES * kWave;
    __shared__ Shared<WAVES> shared[WAVES == 1 ? 4 : 1];
    Shared<WAVES> &sh = shared[WAVES == 1 ? threadIdx.x / kWave : 0];
    const Group<WAVES> g{sh.red};
    const int row = WAVES == 1 ? blockIdx.x * 4 + threadIdx.x / kWave : blockIdx.x;
    if (WAVES == 1 && row >= a.n) return;
    const int tid = g.thread();
    if (a.top && tid == 0) sh.count = 0;  // (read behind the meeting below)
    const char *base = static_cast<const char *>(a.logits) + a.stride_n * es * row;
    const int64_t token = a.tokens[row];
    const bool known = token != a.ignore, inside = token >= 0 && token < a.vocab;
    if (!ENTROPY && !a.top && !known) {  // nothing of this row is asked for
        if (tid == 0) {
            a.logprobs[row] = 0.f;
            if (a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.f;
        }
        return;
    }
    float top = -kInf, m = kLowest, c = reference(kLowest), s = 0.f, t = 0.f;
    auto add = [&](auto count, const float *x) {
        constexpr int N = decltype(count)::value;
        float tm = x[0];
#pragma unroll
        for (int j = 1; j < N; ++j) tm = fmaxf(tm, x[j]);
        top = fmaxf(top, tm);
        m = fmaxf(m, tm);
        const float nc = reference(m), by = c - nc, f = __builtin_amdgcn_exp2f(by);
        if constexpr (ENTROPY) t = f * fmaf(by, s, t);
        s *= f;
        c = nc;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float d = fmaf(x[j], kLog2e, -c), e = __builtin_amdgcn_exp2f(d);
            s += e;
            if constexpr (ENTROPY) t = fmaf(e, fmaxf(d, kFloor), t);
        }
        return tm;
    };
    const int whole = a.vocab / VE, full = whole / (U * kThreads) * (U * kThreads);  // vectors
    int i = tid;
    for (int b = 0; i - tid < full; i += U * kThreads, ++b) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = reinterpret_cast<const Raw *>(base)[i + u * kThreads].v;
        float x[U][VE];
#pragma unroll
        for (int u = 0; u < U; ++u) widen<DT>(v[u], x[u]);
        const float most = add(std::integral_constant<int, U * VE>{}, &x[0][0]);
        if (a.top && b < Shared<WAVES>::kBatches) sh.batch[b][tid] = most;
    }
    float tail[U];  // the largest of each of the last vectors
#pragma unroll
    for (int u = 0; u < U; ++u) tail[u] = -kInf;
    if (i - tid < whole) {  // all on their way at once
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i - tid + u * kThreads < whole) v[u] = reinterpret_cast<const Raw *>(base)[min(i + u * kThreads, whole - 1)].v;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i - tid + u * kThreads >= whole) break;
            if (i + u * kThreads >= whole) continue;
            float x[VE];
            widen<DT>(v[u], x);
            tail[u] = add(std::integral_constant<int, VE>{}, x);
        }
    }
    if (const int j = whole * VE + tid; j < a.vocab) {
        const float x = load_elem(base, j, DT);
        add(std::integral_constant<int, 1>{}, &x);
    }
    const float at_token = inside ? load_elem(base, token, DT) : 0.f;
    // the wave's, then all waves'
    const float mine = wave_max(top);
    float all = mine, C = reference(fmaxf(all, kLowest)), by = c - C, f = __builtin_amdgcn_exp2f(by);
    if constexpr (ENTROPY) t = wave_sum(f * fmaf(by, s, t));
    s = wave_sum(s * f);
    if constexpr (WAVES > 1) {
        if (threadIdx.x % kWave == 0) {
            float *r = sh.red + threadIdx.x / kWave * 4;
            r[0] = all, r[1] = s, r[2] = t;
            sh.best[threadIdx.x / kWave] = mine;
        }
        g.sync();
        for (int w = 0; w < WAVES; ++w) all = fmaxf(all, sh.red[4 * w]);
        C = reference(fmaxf(all, kLowest)), s = 0.f, t = 0.f;
#pragma unroll 4
        for (int w = 0; w < WAVES; ++w) {
            const f32x4 r = *reinterpret_cast<const f32x4 *>(sh.red + 4 * w);
            by = reference(fmaxf(r[0], kLowest)) - C, f = __builtin_amdgcn_exp2f(by);
            if constexpr (ENTROPY) t = fmaf(f, fmaf(by, r[1], r[2]), t);
            s = fmaf(f, r[1], s);
        }
    }
    const bool fine = s > 0.f && all > kLowest && all < kHighest;  // (a NaN is in s)
    const float L = log2f(s);
    Careful k{};
    if (!fine) k = careful<DT, WAVES>(g, base, a.vocab);
    auto logprob = [&](float x) {
        if (!fine) return k.logprob(x);
        const float d = fmaf(x, kLog2e, -C);
        return d > kFar ? (d - L) * kLn2 : x - all;  // (in powers of 2 it may be beyond fp32)
    };
    if (tid == 0) {
        a.logprobs[row] = !known ? 0.f : inside ? logprob(at_token) : __builtin_nanf("");
        // (where one token has all the probability this may round to -3e-8; the gradient cancels that
        // against the same in log p, so that it is left as it is)
        if constexpr (ENTROPY) a.entropy[row] = fine ? (L - t / s) * kLn2 : k.entropy();
        if (a.stats) {  // (an ordinary row's L is above -1: its largest d is -1/2 at least)
            a.stats[2 * row] = fine ? C : k.nan ? __builtin_nanf("") : k.top;
            a.stats[2 * row + 1] = fine ? L : -1.f - k.log_sum;
        }
    }
    if (a.top)
        likeliest<DT, WAVES>(g, sh, base, a.vocab, a.top, top, mine, full, tail, [&](int rank, int id, float x) {
            const int64_t at = static_cast<int64_t>(row) * a.top + rank;
            a.top_tokens[at] = id;
            a.top_logprobs[at] = logprob(x);
        });
}

// The gradient of part blockIdx.x of row blockIdx.y's logits.  (At 8192 x 50304 bf16 2, 4 and 8
// vectors a thread take 281, 275 and 310 us, one call after the other.)
constexpr int kBackThreads = 256, kBackUnroll = 4;

template <int DT>
__global__ __launch_bounds__(kBackThreads) void logprobs_backward_kernel(const LogprobsArgs a) {
    constexpr int VE = kVec<DT>, U = kBackUnroll, es = DT == PRIME_F32 ? 4 : 2;
    const int64_t row = blockIdx.y;
    const char *base = static_cast<const char *>(a.logits) + a.stride_n * es * row;
    char *out = static_cast<char *>(a.dlogits) + a.stride_d * es * row;
    const int64_t token = a.tokens[row];
    float gl = token != a.ignore && a.dlogprobs ? a.dlogprobs[row] : 0.f;
    const float h = a.dentropy ? a.dentropy[row] : 0.f;
    if (a.dlogprobs && token != a.ignore && (token < 0 || token >= a.vocab)) gl = __builtin_nanf("");
    const int first = blockIdx.x * (kBackThreads * U * VE) + threadIdx.x * VE;
    const float C = a.stats[2 * row], L = a.stats[2 * row + 1];
    const bool none = gl == 0.f && h == 0.f, fine = L > -1.f;
    const float H = a.dentropy && !none ? a.entropy[row] : 0.f;
    const Careful k{C, -1.f - L, 0.f, C != C};  // as the forward left it
    // p (a0 + a1 log2 p), and g at the token
    const float a0 = -(gl + h * H), a1 = -h * kLn2;
    const int at = token >= 0 && token < a.vocab && (fine || k.top != -kInf) ? static_cast<int>(token) : -1;
    auto grad = [&](float x) {
        const float d = fmaxf(fmaf(x, kLog2e, -C) - L, kFloor);
        return __builtin_amdgcn_exp2f(d) * fmaf(a1, d, a0);
    };
    auto careful_grad = [&](float x) {
        if (k.nan) return __builtin_nanf("");
        if (k.top == -kInf) return 0.f;
        const float d = k.diff(x) - k.log_sum;
        return __expf(d) * (a0 - h * fmaxf(d, kFloor));
    };
    u32x4 v[U];
    if (!none) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = first + u * kBackThreads * VE;
            if (e + VE <= a.vocab) v[u] = reinterpret_cast<const Raw *>(base + static_cast<int64_t>(e) * es)->v;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = first + u * kBackThreads * VE;
        if (e + VE <= a.vocab) {
            float x[VE];
            if (none) {
#pragma unroll
                for (int j = 0; j < VE; ++j) x[j] = 0.f;
            } else if (widen<DT>(v[u], x); fine) {
#pragma unroll
                for (int j = 0; j < VE; ++j) x[j] = grad(x[j]);
            } else {
#pragma unroll 1
                for (int j = 0; j < VE; ++j) x[j] = careful_grad(x[j]);
            }
            if (!none && at >= e && at < e + VE) {
#pragma unroll
                for (int j = 0; j < VE; ++j) x[j] = e + j == at ? gl + x[j] : x[j];
            }
            reinterpret_cast<Raw *>(out + static_cast<int64_t>(e) * es)->v = narrow<DT>(x);
        } else {
            for (int j = e; j < a.vocab; ++j) {
                float x = 0.f;
                if (!none) {
                    x = load_elem(base, j, DT);
                    x = (fine ? grad(x) : careful_grad(x)) + (j == at ? gl : 0.f);
                }
                store_elem(out, j, DT, x);
            }
        }
    }
}

namespace {

template <int DT, int WAVES>
void forward(const LogprobsArgs &a, hipStream_t s) {
    const dim3 grid(WAVES == 1 ? (a.n + 3) / 4 : a.n), block(WAVES == 1 ? 256 : WAVES * kWave);
    if (a.entropy) hipLaunchKernelGGL((logprobs_kernel<DT, WAVES, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((logprobs_kernel<DT, WAVES, false>), grid, block, 0, s, a);
}

// Bytes of a row that one wave takes, against four waves (us): 20000 x 1500 bf16 14.2 / 25.9, x 3000
// 20 / 29, x 6000 43.0 / 42.2, x 3000 fp32 41.7 / 39.
constexpr int kWaveRow = 8192;

template <int DT>
void run(LogprobsArgs a, bool backward, hipStream_t s) {
    constexpr int es = DT == PRIME_F32 ? 4 : 2;
    const int part = kBackThreads * kBackUnroll * kVec<DT>, parts = (a.vocab + part - 1) / part, n = a.n;
    // a launch has below 2^32 threads and 2^16 rows in a grid's second dimension
    const int most = backward ? 65535 : 1 << 21;
    for (int64_t row = 0; row < n; row += most) {  // (the last sum may pass 2^31)
        a.n = n - row < most ? static_cast<int>(n - row) : most;
        if (backward) {
            hipLaunchKernelGGL(logprobs_backward_kernel<DT>, dim3(parts, a.n), dim3(kBackThreads), 0, s, a);
        } else if (static_cast<int64_t>(a.vocab) * es <= kWaveRow) {
            forward<DT, 1>(a, s);
        } else if (n >= 512 || a.vocab <= 16384) {
            // against 16 waves (us): 600 x 50304 bf16 13.2 / 20.8, 511 with 5 alternatives and the
            // entropy 25.7-27.9 / 24.8; 1 x 10000 2.8 / 3.7, 1 x 16000 with 20 9.5 / 7.4
            forward<DT, 4>(a, s);
        } else {
            forward<DT, 16>(a, s);
        }
        a.logits = static_cast<const char *>(a.logits) + a.stride_n * es * a.n;
        a.tokens += a.n;
        if (a.stats) a.stats += 2 * static_cast<int64_t>(a.n);
        if (a.entropy) a.entropy += a.n;
        if (backward) {
            a.dlogits = static_cast<char *>(a.dlogits) + a.stride_d * es * a.n;
            if (a.dlogprobs) a.dlogprobs += a.n;
            if (a.dentropy) a.dentropy += a.n;
        } else {
            a.logprobs += a.n;
            a.top_logprobs += static_cast<int64_t>(a.n) * a.top;
            a.top_tokens += static_cast<int64_t>(a.n) * a.top;
        }
    }
}

}  // namespace

hipError_t launch_logprobs(const LogprobsArgs &a, bool backward, hipStream_t stream) {
    if (a.dt == PRIME_BF16) run<PRIME_BF16>(a, backward, stream);
    else if (a.dt == PRIME_F16) run<PRIME_F16>(a, backward, stream);
    else run<PRIME_F32>(a, backward, stream);
    return hipGetLastError();
}

}  // namespace prime
