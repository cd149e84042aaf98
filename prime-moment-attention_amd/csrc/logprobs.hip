// Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits,
// and the gradient of the first two.  With l = log2(e), C the row's largest logit times l and
//   d_j = x_j l - C,   S = sum_j 2^d_j,   T = sum_j 2^d_j d_j,   L = log2 S:
//   logprob = ln 2 (d_t - L),   entropy = ln 2 (L - T / S),   p_j = 2^(d_j - L)
//   dx_j = g (delta_jt - p_j) - h p_j (log p_j + entropy).
// d_j is one multiply-add, rounded once, and the same for whatever C is, so that C need not
// be the exact product: S, T and d_t are all relative to it.
//
// The sums of powers of 2 hold for logits whose product with l is finite.  A row with others
// (infinities that are its largest, NaN, values near the ends of fp32, nothing but -infinity)
// shows in S and in the largest value, and is summed again by differences (Careful); the
// backward knows it by a NaN in the row's C.

#include <type_traits>

#include "prime_kernels.h"

namespace prime {

namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -2e38f, kHighest = 2e38f;  // times log2(e) finite
constexpr float kFloor = -1e4f;                      // 2^kFloor = 0: for 0 times an exponent of -infinity

struct __attribute__((packed, aligned(2))) Raw {  // 16 bytes of a row, wherever it starts
    u32x4 v;
};

template <int DT>
constexpr int kVec = DT == PRIME_F32 ? 4 : 8;  // elements of 16 bytes

template <int DT>
__device__ __forceinline__ void widen(const u32x4 &v, float (&x)[kVec<DT>]) {
#pragma unroll
    for (int j = 0; j < kVec<DT>; ++j) {
        if constexpr (DT == PRIME_F32) x[j] = __uint_as_float(v[j]);
        else if constexpr (DT == PRIME_BF16) x[j] = __uint_as_float(j & 1 ? v[j / 2] & 0xFFFF0000u : v[j / 2] << 16);
        else x[j] = h16_bits_to_f32(static_cast<uint16_t>(j & 1 ? v[j / 2] >> 16 : v[j / 2]));
    }
}

template <int DT>
__device__ __forceinline__ u32x4 narrow(const float (&x)[kVec<DT>]) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < kVec<DT>; j += DT == PRIME_F32 ? 1 : 2) {
        if constexpr (DT == PRIME_F32) v[j] = __float_as_uint(x[j]);
        else if constexpr (DT == PRIME_BF16) v[j / 2] = f32_to_bf16_bits(x[j]) | static_cast<uint32_t>(f32_to_bf16_bits(x[j + 1])) << 16;
        else v[j / 2] = f32_to_h16_bits(x[j]) | static_cast<uint32_t>(f32_to_h16_bits(x[j + 1])) << 16;
    }
    return v;
}

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

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, kWave));
    return x;
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
    for (int j = g.thread(); j < vocab; j += g.kThreads) {
        const float x = load_elem(row, j, DT);
        top = fmaxf(top, x);
        bad += x != x ? 1.f : 0.f;
    }
    c.top = g.max(top);
    c.nan = g.sum(bad) > 0.f;
    for (int j = g.thread(); j < vocab; j += g.kThreads) {
        const float d = c.diff(load_elem(row, j, DT)), e = __expf(d);
        s += e;
        t += e > 0.f ? e * d : 0.f;
    }
    s = g.sum(s), t = g.sum(t);
    c.log_sum = logf(s), c.mean = t / s;
    return c;
}

}  // namespace

// WAVES > 1: one row a workgroup.  WAVES = 1: one row a wave, four a workgroup.
template <int DT, int WAVES, bool ENTROPY>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void logprobs_kernel(const LogprobsArgs a) {
    constexpr int VE = kVec<DT>, U = 4, es = DT == PRIME_F32 ? 4 : 2, kThreads = WAVES * kWave;
    __shared__ __attribute__((aligned(8))) float red[4 * WAVES];
    const Group<WAVES> g{red};
    const int row = WAVES == 1 ? blockIdx.x * 4 + threadIdx.x / kWave : blockIdx.x;
    if (WAVES == 1 && row >= a.n) return;
    const int tid = g.thread();
    const char *base = static_cast<const char *>(a.logits) + a.stride_n * es * row;
    const int64_t token = a.tokens[row];
    const bool known = token != a.ignore;
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
        const float nc = reference(m), by = c - nc, f = exp2f(by);
        if constexpr (ENTROPY) t = f * fmaf(by, s, t);
        s *= f;
        c = nc;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float d = fmaf(x[j], kLog2e, -c), e = __builtin_amdgcn_exp2f(d);
            s += e;
            if constexpr (ENTROPY) t = fmaf(e, fmaxf(d, kFloor), t);
        }
    };
    const int whole = a.vocab / VE;  // vectors
    int i = tid;
    for (; i + (U - 1) * kThreads < whole; i += U * kThreads) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = reinterpret_cast<const Raw *>(base)[i + u * kThreads].v;
        float x[U][VE];
#pragma unroll
        for (int u = 0; u < U; ++u) widen<DT>(v[u], x[u]);
        add(std::integral_constant<int, U * VE>{}, &x[0][0]);
    }
    for (; i < whole; i += kThreads) {
        float x[VE];
        widen<DT>(reinterpret_cast<const Raw *>(base)[i].v, x);
        add(std::integral_constant<int, VE>{}, x);
    }
    if (const int j = whole * VE + tid; j < a.vocab) {
        const float x = load_elem(base, j, DT);
        add(std::integral_constant<int, 1>{}, &x);
    }
    const float all = g.max(top);
    const float C = reference(fmaxf(all, kLowest)), by = c - C, f = exp2f(by);
    if constexpr (ENTROPY) t = g.sum(f * fmaf(by, s, t));
    s = g.sum(s * f);
    const bool fine = s > 0.f && s < kInf && all > kLowest && all < kHighest;  // (NaN: false)
    const float L = log2f(s);
    Careful k{};
    if (!fine) k = careful<DT, WAVES>(g, base, a.vocab);
    auto logprob = [&](float x) {
        if (!fine) return k.logprob(x);
        const float d = fmaf(x, kLog2e, -C);
        return d > kLowest ? (d - L) * kLn2 : x - all;  // (in powers of 2 it may be beyond fp32)
    };
    if (tid == 0) {
        float lp = 0.f;
        if (known) lp = token >= 0 && token < a.vocab ? logprob(load_elem(base, token, DT)) : __builtin_nanf("");
        a.logprobs[row] = lp;
        if constexpr (ENTROPY) a.entropy[row] = fine ? (L - t / s) * kLn2 : k.entropy();
        if (a.stats) a.stats[2 * row] = fine ? C : __builtin_nanf(""), a.stats[2 * row + 1] = L;
    }
    // the likeliest, one after the other: the largest key below the last one's
    uint64_t last = ~0ull;
    for (int r = 0; r < a.top; ++r) {
        uint64_t best = 0;
        for (int j = tid; j < a.vocab; j += kThreads) {
            const uint64_t key = static_cast<uint64_t>(rank_key(load_elem(base, j, DT))) << 32 | static_cast<uint32_t>(~j);
            if (key < last) best = max_u64(best, key);
        }
        last = g.max(best);
        if (tid == 0) {
            const int64_t id = static_cast<uint32_t>(~last);
            a.top_tokens[static_cast<int64_t>(row) * a.top + r] = id;
            a.top_logprobs[static_cast<int64_t>(row) * a.top + r] = logprob(load_elem(base, id, DT));
        }
    }
}

// The gradient of part blockIdx.x of row blockIdx.y's logits.
constexpr int kBackThreads = 256, kBackUnroll = 4;

template <int DT>
__global__ __launch_bounds__(kBackThreads) void logprobs_backward_kernel(const LogprobsArgs a) {
    constexpr int VE = kVec<DT>, U = kBackUnroll, es = DT == PRIME_F32 ? 4 : 2;
    __shared__ __attribute__((aligned(8))) float red[4 * kBackThreads / kWave];
    const int64_t row = blockIdx.y;
    const char *base = static_cast<const char *>(a.logits) + a.stride_n * es * row;
    char *out = static_cast<char *>(a.dlogits) + a.stride_d * es * row;
    const int64_t token = a.tokens[row];
    float gl = token != a.ignore && a.dlogprobs ? a.dlogprobs[row] : 0.f;
    const float h = a.dentropy ? a.dentropy[row] : 0.f;
    if (token != a.ignore && (token < 0 || token >= a.vocab)) gl = __builtin_nanf("");
    const int first = blockIdx.x * (kBackThreads * U * VE) + threadIdx.x * VE;
    const float C = a.stats[2 * row], L = a.stats[2 * row + 1];
    const bool none = gl == 0.f && h == 0.f, fine = C == C;
    const float H = a.dentropy && !none ? a.entropy[row] : 0.f;
    Careful k{};
    if (!none && !fine) k = careful<DT>(Group<kBackThreads / kWave>{red}, base, a.vocab);
    // p (a0 + a1 log2 p), and g at the token
    const float a0 = -(gl + h * H), a1 = -h * kLn2;
    auto grad = [&](float x, int j) {
        float r = 0.f;
        if (fine) {
            const float d = fmaxf(fmaf(x, kLog2e, -C) - L, kFloor);
            r = __builtin_amdgcn_exp2f(d) * fmaf(a1, d, a0);
        } else if (k.nan) {
            return __builtin_nanf("");
        } else if (k.top == -kInf) {
            return 0.f;
        } else {
            const float d = k.diff(x) - k.log_sum;
            r = __expf(d) * (a0 - h * fmaxf(d, kFloor));
        }
        return j == token ? gl + r : r;
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
            } else {
                widen<DT>(v[u], x);
#pragma unroll
                for (int j = 0; j < VE; ++j) x[j] = grad(x[j], e + j);
            }
            reinterpret_cast<Raw *>(out + static_cast<int64_t>(e) * es)->v = narrow<DT>(x);
        } else {
            for (int j = e; j < a.vocab; ++j) store_elem(out, j, DT, none ? 0.f : grad(load_elem(base, j, DT), j));
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

template <int DT>
void run(LogprobsArgs a, bool backward, hipStream_t s) {
    constexpr int es = DT == PRIME_F32 ? 4 : 2;
    const int part = kBackThreads * kBackUnroll * kVec<DT>, parts = (a.vocab + part - 1) / part, n = a.n;
    // a launch has below 2^32 threads and 2^16 rows in a grid's second dimension
    const int most = backward ? 65535 : 1 << 21;
    for (int row = 0; row < n; row += most) {
        a.n = n - row < most ? n - row : most;
        if (backward) {
            hipLaunchKernelGGL(logprobs_backward_kernel<DT>, dim3(parts, a.n), dim3(kBackThreads), 0, s, a);
        } else if (a.vocab <= 2048) {
            forward<DT, 1>(a, s);
        } else if (n >= 512) {
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
