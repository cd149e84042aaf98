// Gated linear recurrence: per sequence and channel
//   D_t = clamp(softplus(step_t), kStepMin, kStepMax),  z_t = D_t / tau,  a_t = exp(-z_t)
//   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gate_t) x_t,   y_t = h_t
// and its gradients.  Elementwise over channels: a lane owns V neighbouring ones.
//
// One pass over the data.  A workgroup takes a span of kSpan tokens by 64 V channels,
// each of its waves kGatedTile of the tokens: the gates go into registers, the wave's
// tokens fold into (a's product - 1, end state from zero), the folds meet in LDS, and
// every wave then runs its tokens once more from its true state, with two fused
// multiply-adds and the rounding's remainder a token instead of the gates.
// Spans hand their state on through a workspace word per span and channel.  Every
// kChain-th span publishes its end state, the others their fold, so that a span needs
// the last published state and at most kChain - 1 folds, which are there as soon as
// those spans have read their inputs; which of them it takes is fixed by its number,
// so the result does not depend on timing.  Spans are numbered by a counter in the order
// in which workgroups start, time first: whatever a workgroup waits for belongs to one
// that started before it, so every wait ends.
//
// a is carried as a - 1 = expm1(-z): next to 1 (long memories) a itself has
// lost the decay's low bits, and with it the error of h grows by 2^-25 times
// the memory's length in tokens.  1 - a^2 = -(a - 1)(2 + (a - 1)) loses nothing.

#include <type_traits>

#include "prime_kernels.h"

namespace prime {

constexpr float kStepMin = 1e-4f, kStepMax = 50.f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWaves = 8, kThreads = kWaves * kWave, kSpan = kWaves * kGatedTile;
constexpr int kChain = 16;

// ------------------------------------------------------------------- gates
// expm1(-z), z >= 0: the Taylor polynomial below 1/16 (next term 1.3e-7 of the value),
// else exp2 (its rounding is 2^-24 / (1/16) of the value at most).
__device__ __forceinline__ float expm1_neg(float z) {
    float p = fmaf(-1.f / 24.f, z, 1.f / 6.f);
    p = fmaf(p, z, -0.5f);
    p = fmaf(p, z, 1.f);
    const float far = __builtin_amdgcn_exp2f(-z * kLog2e) - 1.f;
    return z < 0.0625f ? -z * p : far;
}

// softplus, unclamped, and e = exp(-|s|) for its derivative: max(s, 0) + log(1 + e), with
// log(1 + e) / e on [0, 1] its Chebyshev interpolant of degree 8 (3.4e-8 off at most), so
// that small e loses nothing.  maximum and minimum hand NaN on.
__device__ __forceinline__ float softplus(float s, float &e) {
    e = __builtin_amdgcn_exp2f(-fabsf(s) * kLog2e);
    float p = 0.0051261018961668015f;
    p = fmaf(p, e, -0.029074065387248993f);
    p = fmaf(p, e, 0.0775160863995552f);
    p = fmaf(p, e, -0.13602247834205627f);
    p = fmaf(p, e, 0.19076880812644958f);
    p = fmaf(p, e, -0.2483539879322052f);
    p = fmaf(p, e, 0.3331812024116516f);
    p = fmaf(p, e, -0.4999944567680359f);
    p = fmaf(p, e, 0.9999999403953552f);
    return fmaf(p, e, __builtin_elementwise_maximum(s, 0.f));
}

__device__ __forceinline__ float clamp_step(float d) {
    return __builtin_elementwise_minimum(__builtin_elementwise_maximum(d, kStepMin), kStepMax);
}

__device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-g * kLog2e));
}

// a - 1 and b = sqrt(1 - a^2) sigmoid(g) x of one token
__device__ __forceinline__ void gates(float x, float s, float g, float inv_tau, float &am1, float &b) {
    float e;
    am1 = expm1_neg(clamp_step(softplus(s, e)) * inv_tau);
    b = __builtin_amdgcn_sqrtf(-am1 * (2.f + am1)) * sigmoid(g) * x;
}

// h <- h + (am1 h + b), `lo` keeping what the sum's rounding drops.  Without it a state
// that hardly changes is rounded the same way every token: h = 3 at z = 5e-8 moves by
// 0.63 of its spacing, which rounds to 1, and decays 1.6 times too fast.
__device__ __forceinline__ void advance(float &h, float &lo, float am1, float b) {
    const float d = fmaf(am1, h, b) + lo, next = h + d;
    lo = d - (next - h);
    h = next;
}

// A fold (A, H): the tokens take a state h to h + (A h + H).  One more token:
__device__ __forceinline__ void fold_token(float &A, float &H, float am1, float b) {
    A += fmaf(am1, A, am1);
    H += fmaf(am1, H, b);
}

// ------------------------------------------------------------------- access
// V elements of type DT as they lie in memory
template <int DT, int V>
struct Packed {
    static constexpr int bytes = V * (DT == PRIME_F32 ? 4 : 2);
    using type = typename std::conditional<bytes == 2, uint16_t,
                 typename std::conditional<bytes == 4, uint32_t,
                 typename std::conditional<bytes == 8, uint2, uint4>::type>::type>::type;
};

template <int DT, int V>
__device__ __forceinline__ void unpack(const typename Packed<DT, V>::type &p, float (&f)[V]) {
    if constexpr (DT == PRIME_F32) {
        __builtin_memcpy(f, &p, sizeof(f));
    } else {
        uint16_t h[V];
        __builtin_memcpy(h, &p, sizeof(h));
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = DT == PRIME_BF16 ? bf16_bits_to_f32(h[i]) : h16_bits_to_f32(h[i]);
    }
}

template <int DT, int V>
__device__ __forceinline__ typename Packed<DT, V>::type pack(const float (&f)[V]) {
    typename Packed<DT, V>::type p;
    if constexpr (DT == PRIME_F32) {
        __builtin_memcpy(&p, f, sizeof(f));
    } else {
        uint16_t h[V];
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = DT == PRIME_BF16 ? f32_to_bf16_bits(f[i]) : f32_to_h16_bits(f[i]);
        __builtin_memcpy(&p, h, sizeof(h));
    }
    return p;
}

// A row of a view: rows are the same for a whole wave, so the address is a scalar and the
// lane's offset.
template <int DT, int V>
__device__ __forceinline__ const typename Packed<DT, V>::type &at(const GatedView &v, int b, int l, uint32_t c) {
    constexpr int es = DT == PRIME_F32 ? 4 : 2;
    const char *row = static_cast<const char *>(v.data) + (b * v.sb + l * v.sl) * es;
    return *reinterpret_cast<const typename Packed<DT, V>::type *>(row + c * es);
}
template <int DT, int V>
__device__ __forceinline__ typename Packed<DT, V>::type &at_out(const GatedView &v, int b, int l, uint32_t c) {
    return const_cast<typename Packed<DT, V>::type &>(at<DT, V>(v, b, l, c));
}

// -------------------------------------------------------------- spans' chain
// A workspace word: two floats, of which the first is never the all-ones NaN that the
// words are filled with before.
constexpr uint64_t kEmpty = ~0ull;

__device__ __forceinline__ void publish(uint64_t *w, float first, float second) {
    uint32_t f = __float_as_uint(first);
    f = f == 0xFFFFFFFFu ? 0x7FC00000u : f;
    __hip_atomic_store(w, static_cast<uint64_t>(f) << 32 | __float_as_uint(second), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t peek(const uint64_t *w) {
    return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What reaches span g (counted from where the recurrence starts): the published end state
// of the last chain head before it, then the folds between.  `words` is this channel's
// word of span 0, `stride` apart; called for g > 0 only.
__device__ __forceinline__ void chain_in(const uint64_t *words, int64_t stride, int g, float &h, float &lo) {
    constexpr int U = 5;  // words in flight, three rounds at most
    static_assert((kChain - 1) % U == 0, "rounds of U folds");
    const int head = (g - 1) / kChain * kChain, n = g - 1 - head;
    uint64_t first = peek(words + head * stride);
    for (int j0 = 0; j0 < n || j0 == 0; j0 += U) {
        uint64_t w[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (j0 + j < n) w[j] = peek(words + (head + 1 + j0 + j) * stride);
        if (j0 == 0) {
            while (first == kEmpty) {
                __builtin_amdgcn_s_sleep(1);
                first = peek(words + head * stride);
            }
            h = __uint_as_float(static_cast<uint32_t>(first));
            lo = __uint_as_float(static_cast<uint32_t>(first >> 32));
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (j0 + j >= n) continue;
            while (w[j] == kEmpty) {
                __builtin_amdgcn_s_sleep(1);
                w[j] = peek(words + (head + 1 + j0 + j) * stride);
            }
            advance(h, lo, __uint_as_float(static_cast<uint32_t>(w[j] >> 32)), __uint_as_float(static_cast<uint32_t>(w[j])));
        }
    }
}

template <int V>
struct SpanShared {
    float A[kWaves][kWave * V], H[kWaves][kWave * V];  // the waves' folds
    float h[kWave * V], lo[kWave * V];                 // what reaches the span
    int span;
};

// The workgroup's place.
struct Place {
    int g, b, wave;  // span in time order, sequence, wave
    uint32_t c;      // first channel of the lane
    bool in;         // the lane has channels
};
template <int V>
__device__ __forceinline__ Place place(const GatedArgs &a, SpanShared<V> &sh) {
    int id = blockIdx.x;
    if (a.G > 1) {  // the counter starts at -1
        if (threadIdx.x == 0) sh.span = static_cast<int>(atomicAdd(a.counter, 1u) + 1u);
        __syncthreads();
        id = __builtin_amdgcn_readfirstlane(sh.span);
    }
    const int groups = (a.C + kWave * V - 1) / (kWave * V), cols = a.B * groups, col = id % cols;
    Place p;
    p.g = id / cols;
    p.b = col / groups;
    p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t c = (col % groups * kWave + threadIdx.x % kWave) * V;
    p.in = c < static_cast<uint32_t>(a.C);
    p.c = p.in ? c : 0;  // lanes past the last channel read the first and write nothing
    return p;
}

// Every wave's fold to where its wave starts: h, lo from the span's start over the folds of
// the waves before it (`order` is the wave's place in time).  Wave 0 also gets what the
// span needs from the chain and publishes what the chain needs from the span.
template <int V, bool REVERSE>
__device__ __forceinline__ void join(const GatedArgs &a, SpanShared<V> &sh, const Place &p, int g, const float *start,
                                     const float (&A)[V], const float (&H)[V], float (&h)[V], float (&lo)[V]) {
    const int lane = threadIdx.x % kWave, order = REVERSE ? kWaves - 1 - p.wave : p.wave;
#pragma unroll
    for (int i = 0; i < V; ++i) sh.A[order][lane * V + i] = A[i], sh.H[order][lane * V + i] = H[i];
    __syncthreads();
    if (p.wave == 0) {
        const int64_t row = static_cast<int64_t>(p.b) * a.C + p.c;
        uint64_t *words = a.words + static_cast<int64_t>(p.b) * a.G * a.C + p.c;
        if (g + 1 < a.G && g % kChain && p.in) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float fa = 0.f, fh = 0.f;
                for (int w = 0; w < kWaves; ++w) fold_token(fa, fh, sh.A[w][lane * V + i], sh.H[w][lane * V + i]);
                publish(words + static_cast<int64_t>(g) * a.C + i, fa, fh);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float sh_h = 0.f, sh_lo = 0.f;
            if (g == 0) {
                if (start) sh_h = start[row + i];
            } else if (p.in) {
                chain_in(words + i, a.C, g, sh_h, sh_lo);
            }
            sh.h[lane * V + i] = sh_h;
            sh.lo[lane * V + i] = sh_lo;
            if (g + 1 < a.G && g % kChain == 0 && p.in) {
                for (int w = 0; w < kWaves; ++w) advance(sh_h, sh_lo, sh.A[w][lane * V + i], sh.H[w][lane * V + i]);
                publish(words + static_cast<int64_t>(g) * a.C + i, sh_lo, sh_h);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = sh.h[lane * V + i];
        lo[i] = sh.lo[lane * V + i];
        for (int w = 0; w < order; ++w) advance(h[i], lo[i], sh.A[w][lane * V + i], sh.H[w][lane * V + i]);
    }
}

// ------------------------------------------------------------------ forward
template <int DT, int V>
__global__ __launch_bounds__(kThreads) void gated_scan_kernel(const GatedArgs a) {
    __shared__ SpanShared<V> sh;
    constexpr int T = kGatedTile;
    const Place p = place<V>(a, sh);
    const int l0 = p.g * kSpan + p.wave * T, n = min(T, a.L - l0);  // n <= 0: nothing of the wave's is left
    float am1[T][V], b[T][V], A[V], H[V], inv_tau[V], h[V], lo[V];
#pragma unroll
    for (int i = 0; i < V; ++i) inv_tau[i] = 1.f / a.tau[p.c + i], A[i] = H[i] = 0.f;
    {
        typename Packed<DT, V>::type xs[T], ss[T], gs[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int l = min(l0 + t, a.L - 1);
            xs[t] = at<DT, V>(a.x, p.b, l, p.c);
            ss[t] = at<DT, V>(a.step, p.b, l, p.c);
            gs[t] = at<DT, V>(a.gate, p.b, l, p.c);
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float x[V], s[V], g[V];
            unpack<DT, V>(xs[t], x);
            unpack<DT, V>(ss[t], s);
            unpack<DT, V>(gs[t], g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                gates(x[i], s[i], g[i], inv_tau[i], am1[t][i], b[t][i]);
                if (t >= n) am1[t][i] = b[t][i] = 0.f;
                fold_token(A[i], H[i], am1[t][i], b[t][i]);
            }
        }
    }
    join<V, false>(a, sh, p, p.g, a.state_in, A, H, h, lo);
    if (!p.in || n <= 0) return;
    if (a.ckpt) {
        float *o = a.ckpt + (static_cast<int64_t>(p.b) * a.tiles + l0 / T) * a.C + p.c;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = h[i];
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
        for (int i = 0; i < V; ++i) advance(h[i], lo[i], am1[t][i], b[t][i]);
        if (t < n) at_out<DT, V>(a.y, p.b, l0 + t, p.c) = pack<DT, V>(h);
    }
    if (a.state_out && l0 + n == a.L) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.state_out[static_cast<int64_t>(p.b) * a.C + p.c + i] = h[i];
    }
}

// Few tokens: a lane walks them.
template <int DT, int V>
__global__ __launch_bounds__(256) void gated_step_kernel(const GatedArgs a) {
    const int groups = (a.C + blockDim.x * V - 1) / (blockDim.x * V), b = blockIdx.x / groups;
    const uint32_t c = (blockIdx.x % groups * blockDim.x + threadIdx.x) * V;
    if (c >= static_cast<uint32_t>(a.C)) return;
    const int64_t row = static_cast<int64_t>(b) * a.C + c;
    float inv_tau[V], h[V], lo[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        inv_tau[i] = 1.f / a.tau[c + i];
        h[i] = a.state_in ? a.state_in[row + i] : 0.f;
        lo[i] = 0.f;
    }
    if (a.ckpt) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.ckpt[row + i] = h[i];
    }
    for (int l = 0; l < a.L; ++l) {
        float x[V], s[V], g[V];
        unpack<DT, V>(at<DT, V>(a.x, b, l, c), x);
        unpack<DT, V>(at<DT, V>(a.step, b, l, c), s);
        unpack<DT, V>(at<DT, V>(a.gate, b, l, c), g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float am1, bt;
            gates(x[i], s[i], g[i], inv_tau[i], am1, bt);
            advance(h[i], lo[i], am1, bt);
        }
        at_out<DT, V>(a.y, b, l, c) = pack<DT, V>(h);
    }
    if (a.state_out) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.state_out[row + i] = h[i];
    }
}

// ----------------------------------------------------------------- backward
// With G_t the whole gradient of h_t, r_t = a_t G_t is what token t - 1 receives:
//   G_t = dy_t + r_{t+1},
// the forward's recurrence in reversed time, with the decay of the token behind.  The
// wave's states come again from its checkpoint, then
//   dz = G (a^2 / n  sigmoid x - a h_{t-1}),  n = sqrt(1 - a^2).
template <int DT, int V>
__global__ __launch_bounds__(kThreads) void gated_bwd_kernel(const GatedArgs a) {
    __shared__ SpanShared<V> sh;
    constexpr int T = kGatedTile;
    const Place p = place<V>(a, sh);
    const int span = a.G - 1 - p.g, l0 = span * kSpan + p.wave * T, n = min(T, a.L - l0);
    const int64_t row = static_cast<int64_t>(p.b) * a.C + p.c;
    float inv_tau[V], A[V], R[V];
    // a token: x, dy, a - 1, h_{t-1}, sigmoid(gate), sigmoid(gate) / n, z, d z / d step
    float xs[T][V], dys[T][V], am1[T][V], h[T][V], sg[T][V], sn[T][V], z[T][V], dzds[T][V];
#pragma unroll
    for (int i = 0; i < V; ++i) inv_tau[i] = 1.f / a.tau[p.c + i], A[i] = R[i] = 0.f;
    {
        typename Packed<DT, V>::type px[T], ps[T], pg[T], pd[T];
        float hc[V], hl[V];
        const float *ck = a.ckpt + (static_cast<int64_t>(p.b) * a.tiles + min(l0 / T, a.tiles - 1)) * a.C + p.c;
#pragma unroll
        for (int i = 0; i < V; ++i) hc[i] = ck[i], hl[i] = 0.f;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int l = min(l0 + t, a.L - 1);
            px[t] = at<DT, V>(a.x, p.b, l, p.c);
            ps[t] = at<DT, V>(a.step, p.b, l, p.c);
            pg[t] = at<DT, V>(a.gate, p.b, l, p.c);
            pd[t] = at<DT, V>(a.dy, p.b, l, p.c);
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float s[V], g[V];
            unpack<DT, V>(px[t], xs[t]);
            unpack<DT, V>(ps[t], s);
            unpack<DT, V>(pg[t], g);
            unpack<DT, V>(pd[t], dys[t]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float e;
                const float soft = softplus(s[i], e);
                const float sp = __builtin_amdgcn_rcpf(1.f + e) * (s[i] < 0.f ? e : 1.f);  // softplus'
                dzds[t][i] = soft < kStepMin || soft > kStepMax ? 0.f : inv_tau[i] * sp;
                z[t][i] = clamp_step(soft) * inv_tau[i];
                am1[t][i] = expm1_neg(z[t][i]);
                const float q = -am1[t][i] * (2.f + am1[t][i]);
                sg[t][i] = sigmoid(g[i]);
                sn[t][i] = sg[t][i] * __builtin_amdgcn_rsqf(q);
                h[t][i] = hc[i];
                advance(hc[i], hl[i], am1[t][i], q * sn[t][i] * xs[t][i]);
                if (t >= n) am1[t][i] = dys[t][i] = 0.f;
            }
        }
#pragma unroll
        for (int t = T - 1; t >= 0; --t) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float G = dys[t][i] + R[i];
                R[i] = fmaf(am1[t][i], G, G);
                A[i] += fmaf(am1[t][i], A[i], am1[t][i]);
            }
        }
    }
    float G[V], lo[V], behind[V], dtau[V];
    join<V, true>(a, sh, p, p.g, a.dstate_out, A, R, G, lo);
#pragma unroll
    for (int i = 0; i < V; ++i) behind[i] = dtau[i] = 0.f;
#pragma unroll
    for (int t = T - 1; t >= 0; --t) {
        float dx[V], ds[V], dg[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            advance(G[i], lo[i], behind[i], dys[t][i]);
            behind[i] = am1[t][i];
            const float al = 1.f + am1[t][i], q = -am1[t][i] * (2.f + am1[t][i]);
            dx[i] = G[i] * (q * sn[t][i]);
            dg[i] = dx[i] * xs[t][i] * (1.f - sg[t][i]);
            const float dz = al * G[i] * fmaf(al * sn[t][i], xs[t][i], -h[t][i]);
            ds[i] = dz * dzds[t][i];
            if (t < n) dtau[i] = fmaf(-dz, z[t][i], dtau[i]);
        }
        if (t < n && p.in) {
            at_out<DT, V>(a.dx, p.b, l0 + t, p.c) = pack<DT, V>(dx);
            at_out<DT, V>(a.dstep, p.b, l0 + t, p.c) = pack<DT, V>(ds);
            at_out<DT, V>(a.dgate, p.b, l0 + t, p.c) = pack<DT, V>(dg);
        }
    }
    if (l0 == 0 && a.dstate_in && p.in) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.dstate_in[row + i] = fmaf(behind[i], G[i], G[i]);
    }
    // the span's part of dtau, wave by wave
    const int lane = threadIdx.x % kWave;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) sh.A[p.wave][lane * V + i] = dtau[i];
    __syncthreads();
    if (p.wave || !p.in) return;
    float *part = a.dtau_part + (static_cast<int64_t>(p.b) * a.G + span) * a.C + p.c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float sum = 0.f;
        for (int w = 0; w < kWaves; ++w) sum += sh.A[w][lane * V + i];
        part[i] = sum * inv_tau[i];
    }
}

// dtau[c] = the sum of the spans' parts: 16 waves each take every 16th, in order, then
// their sums in order.
__global__ __launch_bounds__(1024) void gated_dtau_kernel(const GatedArgs a) {
    __shared__ float part[16][kWave];
    const int c = blockIdx.x * kWave + threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t n = static_cast<int64_t>(a.B) * a.G;
    float s = 0.f;
    if (c < a.C) {
#pragma unroll 8
        for (int64_t j = wave; j < n; j += 16) s += a.dtau_part[j * a.C + c];
    }
    part[wave][threadIdx.x % kWave] = s;
    __syncthreads();
    if (wave || c >= a.C) return;
    for (int w = 1; w < 16; ++w) s += part[w][threadIdx.x];
    a.dtau[c] = s;
}

// The chain's words and the counter before them, all ones.
__global__ __launch_bounds__(256) void gated_fill_kernel(uint4 *p, int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i < n) p[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// ------------------------------------------------------------------ launch
namespace {

constexpr int kStepTokens = 4;  // up to here a lane walks the tokens

// Whether every row allows V channels a lane.
bool lanes_of(const GatedArgs &a, int v) {
    const int es = a.dt == PRIME_F32 ? 4 : 2;
    if (a.C % v) return false;
    for (const GatedView *t : {&a.x, &a.step, &a.gate, &a.y, &a.dy, &a.dx, &a.dstep, &a.dgate})
        if (t->data && (reinterpret_cast<uintptr_t>(t->data) % (v * es) || t->sb % v || t->sl % v)) return false;
    return true;
}

int spans_grid(const GatedArgs &a, int v) { return a.B * ((a.C + kWave * v - 1) / (kWave * v)) * a.G; }

void fill(const GatedArgs &a, hipStream_t s) {
    if (a.G == 1) return;
    const int64_t n = static_cast<int64_t>(gated_chain_bytes(a.B, a.L, a.C) / 16);
    hipLaunchKernelGGL(gated_fill_kernel, dim3((n + 255) / 256), dim3(256), 0, s, reinterpret_cast<uint4 *>(a.counter), n);
}

template <int DT, int V>
void forward(const GatedArgs &a, hipStream_t s) {
    if (a.L <= kStepTokens) {
        const int lanes = (a.C + V - 1) / V, block = lanes >= 256 ? 256 : (lanes + kWave - 1) / kWave * kWave;
        hipLaunchKernelGGL((gated_step_kernel<DT, V>), dim3(a.B * ((lanes + block - 1) / block)), dim3(block), 0, s, a);
        return;
    }
    fill(a, s);
    hipLaunchKernelGGL((gated_scan_kernel<DT, V>), dim3(spans_grid(a, V)), dim3(kThreads), 0, s, a);
}

template <int DT>
void backward(const GatedArgs &a, hipStream_t s) {
    fill(a, s);
    hipLaunchKernelGGL((gated_bwd_kernel<DT, 1>), dim3(spans_grid(a, 1)), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(gated_dtau_kernel, dim3((a.C + kWave - 1) / kWave), dim3(1024), 0, s, a);
}

template <int DT>
void run(const GatedArgs &a, bool bwd, hipStream_t s) {
    if (bwd) return backward<DT>(a, s);
    if (DT != PRIME_F32 && lanes_of(a, 2)) return forward<DT, 2>(a, s);
    return forward<DT, 1>(a, s);
}

}  // namespace

int gated_spans(int L) { return (L + kSpan - 1) / kSpan; }

// a 16-byte head with the counter, and a word per span and channel; 0 for one span
size_t gated_chain_bytes(int B, int L, int C) {
    const int G = gated_spans(L);
    return G == 1 ? 0 : 16 + (static_cast<size_t>(B) * G * C * sizeof(uint64_t) + 15) / 16 * 16;
}

hipError_t launch_gated_scan(const GatedArgs &a, bool bwd, hipStream_t s) {
    if (a.dt == PRIME_BF16) run<PRIME_BF16>(a, bwd, s);
    else if (a.dt == PRIME_F16) run<PRIME_F16>(a, bwd, s);
    else run<PRIME_F32>(a, bwd, s);
    return hipGetLastError();
}

}  // namespace prime
