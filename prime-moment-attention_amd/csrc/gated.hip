// Gated linear recurrence: per sequence and channel
//   D_t = clamp(softplus(step_t), kStepMin, kStepMax),  z_t = D_t / tau,  a_t = exp(-z_t)
//   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gate_t) x_t,   y_t = h_t
// and its gradients.  Elementwise over channels: a lane owns one.
//
// One pass over the data.  A workgroup takes a span of kSpan tokens by 64 channels,
// each of its waves kGatedTile of the tokens.  A wave scans its tokens from zero, keeping
// each token's state and the product of a up to it, and folds them into (sum of z, end
// state); the folds meet in LDS, and once the wave knows the state it starts from, a token
// is one fused multiply-add away: h_t = (from zero) + (product) (start).
// Spans hand their state on through a workspace word per span and channel.  Every
// kChain-th span publishes its end state, the others their fold, so that a span needs
// the last published state and at most kChain - 1 folds, which are there as soon as
// those spans have read their inputs; which of them it takes is fixed by its number,
// so the result does not depend on timing.  Spans are numbered by a counter in the order
// in which workgroups start, time first: whatever a workgroup waits for belongs to one
// that started before it, so every wait ends.
//
// What bounds it.  A token is read once and written once: 8 x 8192 x 768 bf16 is 403 MB, 79
// us at the 5.1 TB/s of a large copy; its 49 vector instructions, five of them at a quarter of
// the rate, take as long again.  Together 111 us (3.6 TB/s); 65536 x 512 fp32, twice the bytes
// a token, 107 us (5.0 TB/s).  The backward, 32 x 2048 x 768 bf16, 79 instructions a token: 717 MB
// with the checkpoints, 141 us, takes 158-175.  (With a - 1 alone, which is wrong for quick
// forgetting, 46 and 71 instructions: 106, 106 and 154-166 us.)  Tried early, in us for that bf16
// forward, that fp32 one and the backward, then 112, 113 and 174: 4 waves a span 116, 138, 181; 16 waves 125, 106,
// 179; tiles of 8 tokens 161, 128, 187; a state published every 32nd span 123, 117, 171.
//
// A decay is held in one of two forms.  Next to 1 (long memories) a itself has lost the low bits
// of 1 - a, and with it the error of h grows by 2^-25 times the memory's length in tokens:
// there it is a - 1 = expm1(-z), and h + ((a - 1) h + b).  Far from 1 that sum rounds b at the
// spacing of the h that is to be forgotten (h = 1e7 and a = e^-25 leave nothing of b = 0.3):
// there it is a, and a h + b.  So a token is off by roundings of |a h| + |b| in either form.

#include <type_traits>

#include "prime_kernels.h"

namespace prime {

constexpr float kStepMin = 1e-4f, kStepMax = 50.f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWaves = 8, kThreads = kWaves * kWave, kSpan = kWaves * kGatedTile;
constexpr int kChain = 16;

// ------------------------------------------------------------------- gates
// z in binary logarithms: z = D log2(e) / tau, a = 2^-z.  1 - a below 1/16, its Taylor
// polynomial (next term 3e-8 of the value).
constexpr float kNear = 0.0625f;
__device__ __forceinline__ float loss(float z) {
    constexpr float l = 0.693147180559945f;
    float p = fmaf(-l * l * l * l / 24.f, z, l * l * l / 6.f);
    p = fmaf(p, z, -l * l / 2.f);
    p = fmaf(p, z, l);
    return z * p;
}

// A decay's number m: a - 1 (negative or -0) where it is near 1, else a (positive or +0).
__device__ __forceinline__ bool near_one(float m) { return __float_as_int(m) < 0; }

// of a run of tokens: exp2 - 1 is exact up to z = 1
__device__ __forceinline__ float decay(float z) {
    const float e = __builtin_amdgcn_exp2f(-z);
    return z < kNear ? -loss(z) : z <= 1.f ? e - 1.f : e;
}

// a h + b, and a h, for a token
__device__ __forceinline__ float step_on(float h, bool near, float m, float b) { return (near ? h : 0.f) + fmaf(m, h, b); }
__device__ __forceinline__ float decayed(float h, bool near, float m) { return fmaf(m, h, near ? h : 0.f); }

// softplus, unclamped, and e = exp(-|s|) for its derivative: max(s, 0) + log(1 + e), with
// log(1 + e) / e on [0, 1] its Chebyshev interpolant of degree 7 (2.2e-7 off at most), so
// that small e loses nothing.  maximum and minimum hand NaN on.
__device__ __forceinline__ float softplus(float s, float &e) {
    e = __builtin_amdgcn_exp2f(-fabsf(s) * kLog2e);
    float p = -0.00837115291506052f;
    p = fmaf(p, e, 0.04349390044808388f);
    p = fmaf(p, e, -0.1068500280380249f);
    p = fmaf(p, e, 0.1768747717142105f);
    p = fmaf(p, e, -0.24474774301052094f);
    p = fmaf(p, e, 0.3327192962169647f);
    p = fmaf(p, e, -0.49997174739837646f);
    p = fmaf(p, e, 0.9999997615814209f);
    return fmaf(p, e, __builtin_elementwise_maximum(s, 0.f));
}

__device__ __forceinline__ float clamp_step(float d) {
    return __builtin_elementwise_minimum(__builtin_elementwise_maximum(d, kStepMin), kStepMax);
}

// tau between 1e-30 and 1e33: past them 1 / tau, or 1 - a^2 >= 2e-4 / tau, is no normal number and
// a gradient the product of 0 and infinity.
__device__ __forceinline__ float held(float tau) {
    return __builtin_elementwise_minimum(__builtin_elementwise_maximum(tau, 1e-30f), 1e33f);
}

// sigmoid, and e = exp(-g): 1 - sigmoid is e sigmoid, which an open gate does not cancel (at
// g = 12 a subtraction is off by a hundredth of it)
__device__ __forceinline__ float sigmoid(float g, float &e) {
    e = __builtin_amdgcn_exp2f(-g * kLog2e);
    return __builtin_amdgcn_rcpf(1.f + e);
}

// A token's decay, and 1 - a^2: d (2 - d) with d = 1 - a near 1, else 1 - a a (exp2's rounding is
// 2^-24 / (ln(2) / 16) of it at most).
__device__ __forceinline__ float token_decay(float z, bool &near, float &m) {
    const float d = loss(z), a = __builtin_amdgcn_exp2f(-z);
    near = z < kNear;
    m = near ? -d : a;
    return fmaf(-m, m, near ? d + d : 1.f);
}

// z, the decay and b = sqrt(1 - a^2) sigmoid(g) x of one token, of none (a = 1, b = 0) without
// `in`; rate = log2(e) / tau
__device__ __forceinline__ void gates(bool in, float x, float s, float g, float rate, float &z, bool &near, float &m,
                                      float &b) {
    float e, eg;
    z = clamp_step(softplus(s, e)) * rate;
    z = in ? z : 0.f;
    b = __builtin_amdgcn_sqrtf(token_decay(z, near, m)) * sigmoid(g, eg) * x;
    b = in ? b : 0.f;
}

// h <- a h + b, `lo` keeping what a decay near 1 would drop of it by rounding.  Without it a
// state that hardly changes is rounded the same way every time: h = 3 at z = 5e-8 moves by
// 0.63 of its spacing a token, which rounds to 1, and decays 1.6 times too fast.
__device__ __forceinline__ void advance(float &h, float &lo, float m, float b) {
    const bool near = near_one(m);
    const float d = fmaf(m, h, b), dl = d + lo, next = h + dl;
    lo = near ? dl - (next - h) : 0.f;
    h = near ? next : d;
}

// ------------------------------------------------------------------- access
template <int DT>
using Elem = typename std::conditional<DT == PRIME_F32, float, uint16_t>::type;

template <int DT>
__device__ __forceinline__ float widen(Elem<DT> p) {
    if constexpr (DT == PRIME_F32) return p;
    else return DT == PRIME_BF16 ? bf16_bits_to_f32(p) : h16_bits_to_f32(p);
}
template <int DT>
__device__ __forceinline__ Elem<DT> narrow(float f) {
    if constexpr (DT == PRIME_F32) return f;
    else return DT == PRIME_BF16 ? f32_to_bf16_bits(f) : f32_to_h16_bits(f);
}

// The rows of a view one after the other, at an offset of the lane's: the row's address is
// the same for a whole wave and stays in scalar registers.
struct Rows {
    char *row;
    int64_t step;
    __device__ __forceinline__ Rows(const GatedView &v, int es, int b, int l)
        : row(static_cast<char *>(v.data) + (b * v.sb + l * v.sl) * es), step(v.sl * es) {}
    // PAST: past the caches, each element being used once
    template <typename P, bool PAST>
    __device__ __forceinline__ P load(uint32_t offset) const {
        const P *p = reinterpret_cast<const P *>(row + offset);
        if constexpr (PAST) return __builtin_nontemporal_load(p);
        else return *p;
    }
    template <bool PAST, typename P>
    __device__ __forceinline__ void store(uint32_t offset, P v) const {
        P *p = reinterpret_cast<P *>(row + offset);
        if constexpr (PAST) __builtin_nontemporal_store(v, p);
        else *p = v;
    }
    __device__ __forceinline__ void next(bool more = true) { row += more ? step : 0; }
};

// An offset whose widening to 64 bits stays beside its uses, where it becomes part of the
// load instead of a 64-bit addition a load.
__device__ __forceinline__ uint32_t here(uint32_t offset) {
    asm("" : "+v"(offset));
    return offset;
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

// v computed before what follows: before the wait for a state that others wait for in turn.
__device__ __forceinline__ float ready(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

// What reaches span g (counted from where the recurrence starts): the published end state
// of the last chain head before it, then the folds between.  The folds are there early and
// are joined first, so that from one head's state to the next one's is one word's way.
// `words` is this channel's word of span 0, `stride` apart; called for g > 0 only.
__device__ __forceinline__ void chain_in(const uint64_t *words, int64_t stride, int g, float &h, float &lo) {
    constexpr int U = 3;  // words in flight; more spill the backward's registers
    const int head = (g - 1) / kChain * kChain, n = g - 1 - head;
    uint64_t first = peek(words + head * stride);
    float Z = 0.f, H = 0.f;
    for (int j0 = 0; j0 < n; j0 += U) {
        uint64_t w[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (j0 + j < n) w[j] = peek(words + (head + 1 + j0 + j) * stride);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (j0 + j >= n) continue;
            while (w[j] == kEmpty) {
                __builtin_amdgcn_s_sleep(1);
                w[j] = peek(words + (head + 1 + j0 + j) * stride);
            }
            const float z = __uint_as_float(static_cast<uint32_t>(w[j] >> 32)), m = decay(z);
            Z += z;
            H = step_on(H, near_one(m), m, __uint_as_float(static_cast<uint32_t>(w[j])));
        }
    }
    const float m = ready(decay(Z));
    while (first == kEmpty) {
        __builtin_amdgcn_s_sleep(1);
        first = peek(words + head * stride);
    }
    h = __uint_as_float(static_cast<uint32_t>(first));
    lo = __uint_as_float(static_cast<uint32_t>(first >> 32));
    advance(h, lo, m, H);
}

// A fold (z, H): the tokens take a state h to 2^-z h + H.
struct SpanShared {
    float z[kWaves][kWave], m[kWaves][kWave], H[kWaves][kWave];  // the waves' folds, m = decay(z)
    float h[kWave], lo[kWave];                 // what reaches the span
    int span;
};

// The workgroup's place.
struct Place {
    int g, b, wave, lane;  // span in the recurrence's order, sequence, wave, lane
    uint32_t c;            // the lane's channel
    bool in;               // it has one
};
__device__ __forceinline__ Place place(const GatedArgs &a, SpanShared &sh) {
    int id = blockIdx.x;
    if (a.G > 1) {  // the counter starts at -1
        if (threadIdx.x == 0) sh.span = static_cast<int>(atomicAdd(a.counter, 1u) + 1u);
        __syncthreads();
        id = __builtin_amdgcn_readfirstlane(sh.span);
    }
    const int groups = (a.C + kWave - 1) / kWave, cols = a.B * groups, col = id % cols;
    Place p;
    p.g = id / cols;
    p.b = col / groups;
    p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    p.lane = threadIdx.x % kWave;
    const uint32_t c = col % groups * kWave + p.lane;
    p.in = c < static_cast<uint32_t>(a.C);
    p.c = p.in ? c : 0;  // lanes past the last channel read the first and write nothing
    return p;
}

// From every wave's fold to where the wave starts: h, lo after the span's start and the folds
// of the waves before it in the recurrence's order.  Wave 0 gets what the span needs from the
// chain and publishes what the chain needs from the span.
template <bool REVERSE>
__device__ __forceinline__ void join(const GatedArgs &a, SpanShared &sh, const Place &p, const float *start, float z,
                                     float m, float H, float &h, float &lo) {
    const int order = REVERSE ? kWaves - 1 - p.wave : p.wave;
    sh.z[order][p.lane] = z, sh.m[order][p.lane] = m, sh.H[order][p.lane] = H;
    __syncthreads();
    if (p.wave == 0) {
        uint64_t *words = a.words + static_cast<int64_t>(p.b) * a.G * a.C + p.c, *mine = words + static_cast<int64_t>(p.g) * a.C;
        const bool on = p.g + 1 < a.G && p.in, head = p.g % kChain == 0;
        float fz = 0.f, fh = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float wm = sh.m[w][p.lane];
            fz += sh.z[w][p.lane];
            fh = step_on(fh, near_one(wm), wm, sh.H[w][p.lane]);
        }
        const float m = ready(decay(fz));
        if (on && !head) publish(mine, fz, fh);
        h = lo = 0.f;
        if (p.g == 0) {
            if (start) h = start[static_cast<int64_t>(p.b) * a.C + p.c];
        } else if (p.in) {
            chain_in(words, a.C, p.g, h, lo);
        }
        sh.h[p.lane] = h, sh.lo[p.lane] = lo;
        if (on && head) {
            advance(h, lo, m, fh);
            publish(mine, lo, h);
        }
    }
    __syncthreads();
    h = sh.h[p.lane], lo = sh.lo[p.lane];
    for (int w = 0; w < order; ++w) advance(h, lo, sh.m[w][p.lane], sh.H[w][p.lane]);
}

// A wave's tokens: all kGatedTile of them (the loops below then have no branch in them),
// or the n < kGatedTile before the sequence's end, if any.
template <typename F>
__device__ __forceinline__ void for_tokens(int n, F f) {
    if (n >= kGatedTile) f(std::true_type{}, kGatedTile);
    else if (n > 0) f(std::false_type{}, n);
}

// ------------------------------------------------------------------ forward
template <int DT, bool LINES>
__global__ __launch_bounds__(kThreads) void gated_scan_kernel(const GatedArgs a) {
    __shared__ SpanShared sh;
    constexpr int T = kGatedTile, es = sizeof(Elem<DT>);
    using P = Elem<DT>;
    const Place p = place(a, sh);
    const int l0 = p.g * kSpan + p.wave * T, left = a.L - l0;  // left <= 0: nothing of the wave's is left
    float h[T], prod[T], zs = 0.f, H = 0.f;                    // state from zero, product of a, per token
    for_tokens(left, [&](auto full, int n) {
        Rows rx(a.x, es, p.b, l0), rs(a.step, es, p.b, l0), rg(a.gate, es, p.b, l0);
        const uint32_t o = here(p.c * es);
        P px[T], ps[T], pg[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            px[t] = rx.load<P, LINES>(o), ps[t] = rs.load<P, LINES>(o), pg[t] = rg.load<P, LINES>(o);
            const bool more = full || t + 1 < n;
            rx.next(more), rs.next(more), rg.next(more);
            __builtin_amdgcn_sched_barrier(0);  // else all rows' addresses are held at once, and spilled
        }
        const float rate = kLog2e / held(a.tau[p.c]);
        float pr = 1.f;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float z, m, b;
            bool near;
            gates(full || t < n, widen<DT>(px[t]), widen<DT>(ps[t]), widen<DT>(pg[t]), rate, z, near, m, b);
            H = step_on(H, near, m, b);
            pr = decayed(pr, near, m);
            zs += z;
            h[t] = H, prod[t] = pr;
        }
    });
    const float m = decay(zs);
    float carry, lo;
    join<false>(a, sh, p, a.state_in, zs, m, H, carry, lo);
    if (!p.in || left <= 0) return;
    if (a.ckpt) a.ckpt[(static_cast<int64_t>(p.b) * a.tiles + l0 / T) * a.C + p.c] = carry;
    for_tokens(left, [&](auto full, int n) {
        Rows ry(a.y, es, p.b, l0);
        const uint32_t o = here(p.c * es);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            if (full || t < n) ry.store<true>(o, narrow<DT>(fmaf(prod[t], carry, h[t])));
            ry.next();
        }
    });
    if (a.state_out && left <= T) {
        advance(carry, lo, m, H);
        a.state_out[static_cast<int64_t>(p.b) * a.C + p.c] = carry;
    }
}

template <typename P>
__device__ __forceinline__ P *elem(const GatedView &v, int b, uint32_t c) {
    return static_cast<P *>(v.data) + b * v.sb + c;
}

// Few tokens: a lane walks them, kWalk on their way at a time.  One token of 256 x 768 bf16:
// 3.5 us, all of it the launch and one way through memory (3.1 MB are 0.6 us).
constexpr int kWalk = 4;
template <int DT>
__global__ __launch_bounds__(256) void gated_step_kernel(const GatedArgs a) {
    using P = Elem<DT>;
    const int groups = (a.C + blockDim.x - 1) / blockDim.x, b = blockIdx.x / groups;
    const uint32_t c = blockIdx.x % groups * blockDim.x + threadIdx.x;
    if (c >= static_cast<uint32_t>(a.C)) return;
    const int64_t row = static_cast<int64_t>(b) * a.C + c;
    const P *rx = elem<P>(a.x, b, c), *rs = elem<P>(a.step, b, c), *rg = elem<P>(a.gate, b, c);
    P *ry = elem<P>(a.y, b, c);
    const float rate = kLog2e / held(a.tau[c]);
    float h = a.state_in ? a.state_in[row] : 0.f, lo = 0.f;
    for (int l0 = 0; l0 < a.L; l0 += kWalk) {
        if (a.ckpt && l0 % kGatedTile == 0) a.ckpt[(static_cast<int64_t>(b) * a.tiles + l0 / kGatedTile) * a.C + c] = h;
        P px[kWalk], ps[kWalk], pg[kWalk];
#pragma unroll
        for (int t = 0; t < kWalk; ++t) {
            if (l0 + t >= a.L) break;
            px[t] = *rx, ps[t] = *rs, pg[t] = *rg;
            rx += a.x.sl, rs += a.step.sl, rg += a.gate.sl;
        }
#pragma unroll
        for (int t = 0; t < kWalk; ++t) {
            if (l0 + t >= a.L) break;
            float z, m, bt;
            bool near;
            gates(true, widen<DT>(px[t]), widen<DT>(ps[t]), widen<DT>(pg[t]), rate, z, near, m, bt);
            advance(h, lo, m, bt);
            *ry = narrow<DT>(h);
            ry += a.y.sl;
        }
    }
    if (a.state_out) a.state_out[row] = h;
}

// ----------------------------------------------------------------- backward
// With G_t the whole gradient of h_t, r_t = a_t G_t is what token t - 1 receives:
//   G_t = dy_t + r_{t+1},
// the forward's recurrence in reversed time.  Every gradient is G_t times a number that
// does not depend on it, n = sqrt(1 - a^2), s = sigmoid(gate):
//   dx = G n s        dgate = G n s (1 - s) x        dz = G (a^2 / n  s x - a h_{t-1})
//   dstep = dz d z / d step                          dtau = -sum dz z / tau
// so a wave takes its states again from its checkpoint, keeps those four numbers a token
// instead of the inputs, and multiplies once its G is known (125 registers, 4 waves a SIMD).
template <int DT, bool LINES>
__global__ __launch_bounds__(kThreads, 4) void gated_bwd_kernel(const GatedArgs a) {
    __shared__ SpanShared sh;
    constexpr int T = kGatedTile, es = sizeof(Elem<DT>);
    using P = Elem<DT>;
    const Place p = place(a, sh);
    const int span = a.G - 1 - p.g, l0 = span * kSpan + p.wave * T, left = a.L - l0;
    const float inv_tau = 1.f / held(a.tau[p.c]), rate = inv_tau * kLog2e;
    float cx[T], cg[T], cs[T], cz[T];  // what G is multiplied by for dx, dgate, dstep, -dtau tau^2
    float G[T], prod[T];               // G from r = 0 behind the wave; the product of the a behind a token
    float zs = 0.f, R = 0.f;
    for_tokens(left, [&](auto full, int n) {
        P px[T], ps[T], pg[T], pd[T];
        Rows rx(a.x, es, p.b, l0), rs(a.step, es, p.b, l0), rg(a.gate, es, p.b, l0), rd(a.dy, es, p.b, l0);
        const uint32_t o = here(p.c * es);
        float h = a.ckpt[(static_cast<int64_t>(p.b) * a.tiles + l0 / T) * a.C + p.c], pr = 1.f;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            px[t] = rx.load<P, LINES>(o), ps[t] = rs.load<P, LINES>(o), pg[t] = rg.load<P, LINES>(o), pd[t] = rd.load<P, LINES>(o);
            const bool more = full || t + 1 < n;
            rx.next(more), rs.next(more), rg.next(more), rd.next(more);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float x = widen<DT>(px[t]), s = widen<DT>(ps[t]), d = widen<DT>(pd[t]);
            float e, eg;
            const float soft = softplus(s, e), step = clamp_step(soft), z = step * rate;
            bool near;
            float m;
            const float q = token_decay(z, near, m), rq = __builtin_amdgcn_rsqf(q), al = near ? 1.f + m : m;
            const float sp = __builtin_amdgcn_rcpf(1.f + e) * (s < 0.f ? e : 1.f);  // softplus'
            const float sg = sigmoid(widen<DT>(pg[t]), eg), sn = sg * rq;
            cx[t] = q * sn;
            const float b = cx[t] * x, w = al * fmaf(al * sn, x, -h);
            cg[t] = b * fminf(eg * sg, 1.f);  // (an infinite e times 0 is the 1 of a shut gate)
            cs[t] = step == soft ? w * inv_tau * sp : 0.f;
            cz[t] = w * step;
            h = step_on(h, near, m, b);
            const bool in = full || t < n;
            zs += in ? z : 0.f;
            G[t] = in ? d : 0.f, prod[t] = in ? m : -0.f;
        }
#pragma unroll
        for (int t = T - 1; t >= 0; --t) {
            const float m = prod[t];
            const bool near = near_one(m);
            G[t] += R;
            prod[t] = pr;
            R = decayed(G[t], near, m);
            pr = decayed(pr, near, m);
        }
    });
    float carry, lo, dtau = 0.f;
    const float m = decay(zs);
    join<true>(a, sh, p, a.dstate_out, zs, m, R, carry, lo);
    if (left > 0 && p.in) {
        for_tokens(left, [&](auto full, int n) {
            Rows rx(a.dx, es, p.b, l0), rs(a.dstep, es, p.b, l0), rg(a.dgate, es, p.b, l0);
            const uint32_t o = here(p.c * es);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const float Gt = fmaf(prod[t], carry, G[t]);
                if (full || t < n) {
                    dtau = fmaf(-Gt, cz[t], dtau);
                    rx.store<LINES>(o, narrow<DT>(Gt * cx[t]));
                    rs.store<LINES>(o, narrow<DT>(Gt * cs[t]));
                    rg.store<LINES>(o, narrow<DT>(Gt * cg[t]));
                }
                rx.next(), rs.next(), rg.next();
            }
        });
        if (l0 == 0 && a.dstate_in) {
            advance(carry, lo, m, R);
            a.dstate_in[static_cast<int64_t>(p.b) * a.C + p.c] = carry;
        }
    }
    // the span's part of dtau = -sum dz D / tau^2, wave by wave
    __syncthreads();
    sh.z[p.wave][p.lane] = dtau;
    __syncthreads();
    if (p.wave || !p.in) return;
    float sum = 0.f;
    for (int w = 0; w < kWaves; ++w) sum += sh.z[w][p.lane];
    a.dtau_part[(static_cast<int64_t>(p.b) * a.G + span) * a.C + p.c] = sum * inv_tau * inv_tau;
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

// Whether a lane walks the tokens: a few always (8 tokens of 768 bf16 channels: 1 sequence 4.3
// us, spans 5.1; 256 sequences 6.2, 17.3), more where the sequences fill the chip without the
// waves that share a span (32 tokens: 256 sequences 18.3 us, 22.8; 171, which are 2052 waves,
// 16.2, 16.5; 128 14.2, 13.6; 16 9.4, 5.0).  16 tokens could be walked from 1032 waves on: 86
// sequences 6.8 us, the spans that they get here 8.6; 64 6.3, 5.9.
bool walks(const GatedArgs &a) {
    return a.L <= 8 || (a.L <= 32 && static_cast<int64_t>(a.B) * ((a.C + kWave - 1) / kWave) >= 2048);
}

int spans_grid(const GatedArgs &a) { return a.B * ((a.C + kWave - 1) / kWave) * a.G; }

void fill(const GatedArgs &a, hipStream_t s) {
    if (a.G == 1) return;
    const int64_t n = static_cast<int64_t>(gated_chain_bytes(a.B, a.L, a.C) / 16);
    hipLaunchKernelGGL(gated_fill_kernel, dim3((n + 255) / 256), dim3(256), 0, s, reinterpret_cast<uint4 *>(a.counter), n);
}

// Whether every row starts on a 128-byte line.
bool lines(const GatedArgs &a, bool bwd) {
    const int es = a.dt == PRIME_F32 ? 4 : 2;
    auto one = [&](const GatedView &v) {
        return reinterpret_cast<uintptr_t>(v.data) % 128 == 0 && (a.L == 1 || v.sl * es % 128 == 0) &&
               (a.B == 1 || v.sb * es % 128 == 0);
    };
    return one(a.x) && one(a.step) && one(a.gate) && (bwd ? one(a.dy) && one(a.dx) && one(a.dstep) && one(a.dgate) : one(a.y));
}

template <int DT, bool LINES>
void run_spans(const GatedArgs &a, bool bwd, hipStream_t s) {
    fill(a, s);
    if (bwd) hipLaunchKernelGGL((gated_bwd_kernel<DT, LINES>), dim3(spans_grid(a)), dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((gated_scan_kernel<DT, LINES>), dim3(spans_grid(a)), dim3(kThreads), 0, s, a);
}

// Accesses go past the caches where every row starts on a line: 65536 x 512 fp32 takes 115 us
// with plain ones, 110 so, the backwards of that and of 32 x 2048 x 768 bf16 192, 177 and 175, 165
// (8 x 8192 x 768 bf16 117 either way).  Else neighbouring channel groups share lines, which the
// caches then put together: 8 x 8192 x 1000 bf16 202 us past them, 169 through them, the backward
// 410, 284; fp32 285, 241 and 544, 465; 501 channels bf16 113, 86 and 236, 161.  (The forward's
// stores go past them in either case: up to 5 us less.)
template <int DT>
void run(const GatedArgs &a, bool bwd, hipStream_t s) {
    if (!bwd && walks(a)) {
        const int block = a.C >= 256 ? 256 : (a.C + kWave - 1) / kWave * kWave;
        hipLaunchKernelGGL(gated_step_kernel<DT>, dim3(a.B * ((a.C + block - 1) / block)), dim3(block), 0, s, a);
        return;
    }
    if (lines(a, bwd)) run_spans<DT, true>(a, bwd, s);
    else run_spans<DT, false>(a, bwd, s);
    if (bwd) hipLaunchKernelGGL(gated_dtau_kernel, dim3((a.C + kWave - 1) / kWave), dim3(1024), 0, s, a);
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
