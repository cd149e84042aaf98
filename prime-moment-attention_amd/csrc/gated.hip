// Gated linear recurrence: per sequence and channel
//   D_t = clamp(softplus(step_t), kStepMin, kStepMax),  z_t = D_t / tau,  a_t = exp(-z_t)
//   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gate_t) x_t,   y_t = h_t
// and its gradients.  Elementwise over channels, so a lane owns V neighbouring
// channels and walks the tokens; the state stays in its registers, fp32.
//
// Time is cut into G segments of seg_len tokens (a multiple of kGatedTile)
// where B * C lanes cannot fill the chip: a first kernel folds every segment
// into (sum of z, end state from zero), the second starts each segment from
// the fold of those before it.  The order of every sum is fixed by the sizes.
//
// a is carried as a - 1 = expm1(-z): next to 1 (long memories) a itself has
// lost the decay's low bits, and with it the error of h grows by 2^-25 times
// the memory's length in tokens.  1 - a^2 = -(a - 1)(2 + (a - 1)) loses nothing.

#include <type_traits>

#include "prime_kernels.h"

namespace prime {

constexpr float kStepMin = 1e-4f, kStepMax = 50.f;
constexpr float kLog2e = 1.44269504088896340736f;

// ------------------------------------------------------------------- gates
// log(1 + e), 0 <= e <= 1, as 2 atanh(w), w = e / (2 + e) <= 1/3: the odd series
// to w^15 (next term 1.2e-9), no cancellation for small e.
__device__ __forceinline__ float log1p_unit(float e) {
    const float w = e * __builtin_amdgcn_rcpf(2.f + e), u = w * w;
    float p = 1.f / 15.f;
    p = fmaf(p, u, 1.f / 13.f);
    p = fmaf(p, u, 1.f / 11.f);
    p = fmaf(p, u, 1.f / 9.f);
    p = fmaf(p, u, 1.f / 7.f);
    p = fmaf(p, u, 1.f / 5.f);
    p = fmaf(p, u, 1.f / 3.f);
    p = fmaf(p, u, 1.f);
    return 2.f * w * p;
}

// exp(-z) - 1 for z >= 0: the Taylor polynomial below 1/2 (next term 1.1e-8), else exp2.
__device__ __forceinline__ float expm1_neg(float z) {
    float p = -1.f / 40320.f;
    p = fmaf(p, z, 1.f / 5040.f);
    p = fmaf(p, z, -1.f / 720.f);
    p = fmaf(p, z, 1.f / 120.f);
    p = fmaf(p, z, -1.f / 24.f);
    p = fmaf(p, z, 1.f / 6.f);
    p = fmaf(p, z, -1.f / 2.f);
    p = fmaf(p, z, 1.f);
    const float far = __builtin_amdgcn_exp2f(-z * kLog2e) - 1.f;
    return z < 0.5f ? -z * p : far;
}

// softplus, unclamped, and e = exp(-|s|) for its derivative.  (Selects, not fmax: NaN stays.)
__device__ __forceinline__ float softplus(float s, float &e) {
    e = __builtin_amdgcn_exp2f(-fabsf(s) * kLog2e);
    return (s < 0.f ? 0.f : s) + log1p_unit(e);
}

__device__ __forceinline__ float clamp_step(float d) {
    d = d < kStepMin ? kStepMin : d;
    return d > kStepMax ? kStepMax : d;
}

__device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-g * kLog2e));
}

// z and a - 1 of one token
__device__ __forceinline__ void decay(float s, float inv_tau, float &z, float &am1) {
    float e;
    z = clamp_step(softplus(s, e)) * inv_tau;
    am1 = expm1_neg(z);
}

// h <- h + (am1 h + b), `lo` keeping what the sum's rounding drops.  Without it a state
// that hardly changes is rounded the same way every token: h = 3 at z = 5e-8 moves by
// 0.63 of its spacing, which rounds to 1, and decays 1.6 times too fast.
__device__ __forceinline__ void advance(float &h, float &lo, float am1, float b) {
    const float d = fmaf(am1, h, b) + lo, next = h + d;
    lo = d - (next - h);
    h = next;
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

template <int DT, int V>
__device__ __forceinline__ const typename Packed<DT, V>::type *at(const GatedView &v, int b, int64_t l, int c) {
    const int64_t e = b * v.sb + l * v.sl + c;
    return reinterpret_cast<const typename Packed<DT, V>::type *>(
        static_cast<const char *>(v.data) + e * (DT == PRIME_F32 ? 4 : 2));
}
template <int DT, int V>
__device__ __forceinline__ typename Packed<DT, V>::type *at_out(const GatedView &v, int b, int64_t l, int c) {
    return const_cast<typename Packed<DT, V>::type *>(at<DT, V>(v, b, l, c));
}

// The lane's place: V channels from c, sequence b, segment g (blockIdx.x = b * G + g);
// false for lanes past the last channel.
template <int V>
__device__ __forceinline__ bool place(const GatedArgs &a, int &c, int &b, int &g) {
    c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    b = blockIdx.x / a.G;
    g = blockIdx.x % a.G;
    return c < a.C;
}

// The fold of the segments before g, from the state before the first.
template <int V>
__device__ __forceinline__ void carry_in(const GatedArgs &a, int b, int g, int c, float (&h)[V], float (&lo)[V]) {
    const int64_t row = static_cast<int64_t>(b) * a.C + c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = a.G > 1 ? a.ws_h0[row + i] : (a.state_in ? a.state_in[row + i] : 0.f);
        lo[i] = 0.f;
    }
    for (int j = 0; j < g; ++j) {
        const int64_t o = (static_cast<int64_t>(b) * a.G + j) * a.C + c;
#pragma unroll
        for (int i = 0; i < V; ++i) advance(h[i], lo[i], expm1_neg(a.ws_z[o + i]), a.ws_h[o + i]);
    }
}

// ------------------------------------------------------------------ forward
// One segment's (sum of z, end state from zero); segment 0 also copies the incoming
// state, which the last segment of the second kernel may overwrite (in-place states).
template <int DT, int V>
__global__ __launch_bounds__(kGatedThreads) void gated_summary_kernel(const GatedArgs a) {
    int c, b, g;
    if (!place<V>(a, c, b, g)) return;
    float inv_tau[V], h[V], lo[V], zs[V];
#pragma unroll
    for (int i = 0; i < V; ++i) inv_tau[i] = 1.f / a.tau[c + i], h[i] = 0.f, lo[i] = 0.f, zs[i] = 0.f;
    const int l0 = g * a.seg_len, l1 = min(l0 + a.seg_len, a.L);
#pragma unroll 4
    for (int l = l0; l < l1; ++l) {
        float x[V], s[V], gt[V];
        unpack<DT, V>(*at<DT, V>(a.x, b, l, c), x);
        unpack<DT, V>(*at<DT, V>(a.step, b, l, c), s);
        unpack<DT, V>(*at<DT, V>(a.gate, b, l, c), gt);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float z, am1;
            decay(s[i], inv_tau[i], z, am1);
            const float n = __builtin_amdgcn_sqrtf(-am1 * (2.f + am1));
            advance(h[i], lo[i], am1, n * sigmoid(gt[i]) * x[i]);
            zs[i] += z;
        }
    }
    const int64_t o = (static_cast<int64_t>(b) * a.G + g) * a.C + c, row = static_cast<int64_t>(b) * a.C + c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        a.ws_z[o + i] = zs[i];
        a.ws_h[o + i] = h[i];
        if (g == 0) a.ws_h0[row + i] = a.state_in ? a.state_in[row + i] : 0.f;
    }
}

template <int DT, int V>
__global__ __launch_bounds__(kGatedThreads) void gated_scan_kernel(const GatedArgs a) {
    int c, b, g;
    if (!place<V>(a, c, b, g)) return;
    float inv_tau[V], h[V], lo[V];
#pragma unroll
    for (int i = 0; i < V; ++i) inv_tau[i] = 1.f / a.tau[c + i];
    carry_in<V>(a, b, g, c, h, lo);
    const int l0 = g * a.seg_len, l1 = min(l0 + a.seg_len, a.L);
#pragma unroll 4
    for (int l = l0; l < l1; ++l) {
        if (a.ckpt && l % kGatedTile == 0) {
            float *o = a.ckpt + (static_cast<int64_t>(b) * a.tiles + l / kGatedTile) * a.C + c;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = h[i];
        }
        float x[V], s[V], gt[V];
        unpack<DT, V>(*at<DT, V>(a.x, b, l, c), x);
        unpack<DT, V>(*at<DT, V>(a.step, b, l, c), s);
        unpack<DT, V>(*at<DT, V>(a.gate, b, l, c), gt);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float z, am1;
            decay(s[i], inv_tau[i], z, am1);
            const float n = __builtin_amdgcn_sqrtf(-am1 * (2.f + am1));
            advance(h[i], lo[i], am1, n * sigmoid(gt[i]) * x[i]);
        }
        *at_out<DT, V>(a.y, b, l, c) = pack<DT, V>(h);
    }
    if (a.state_out && g == a.G - 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.state_out[static_cast<int64_t>(b) * a.C + c + i] = h[i];
    }
}

// ----------------------------------------------------------------- backward
// With G_t the whole gradient of h_t, r_t = a_t G_t is what token t - 1 receives:
//   G_t = dy_t + r_{t+1}, advanced as G <- G + (am1 G + dy) with the am1 of the token behind.
// A segment folds into (sum of z, r of its first token from r = 0).
template <int DT, int V>
__global__ __launch_bounds__(kGatedThreads) void gated_bwd_summary_kernel(const GatedArgs a) {
    int c, b, g;
    if (!place<V>(a, c, b, g)) return;
    float inv_tau[V], G[V], lo[V], am1[V], zs[V];
#pragma unroll
    for (int i = 0; i < V; ++i) inv_tau[i] = 1.f / a.tau[c + i], G[i] = lo[i] = am1[i] = zs[i] = 0.f;
    const int l0 = g * a.seg_len, l1 = min(l0 + a.seg_len, a.L);
#pragma unroll 4
    for (int l = l1 - 1; l >= l0; --l) {
        float s[V], dy[V];
        unpack<DT, V>(*at<DT, V>(a.step, b, l, c), s);
        unpack<DT, V>(*at<DT, V>(a.dy, b, l, c), dy);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float z;
            advance(G[i], lo[i], am1[i], dy[i]);
            decay(s[i], inv_tau[i], z, am1[i]);
            zs[i] += z;
        }
    }
    const int64_t o = (static_cast<int64_t>(b) * a.G + g) * a.C + c;
#pragma unroll
    for (int i = 0; i < V; ++i) a.ws_z[o + i] = zs[i], a.ws_h[o + i] = fmaf(am1[i], G[i], G[i]);
}

// Gradients of one segment, a tile of kGatedTile tokens at a time from its end:
// the tile's states come again from its checkpoint, then
//   dz = G (a^2 / n  sigmoid x - a h_{t-1}),  n = sqrt(1 - a^2).
template <int DT, int V>
__global__ __launch_bounds__(kGatedThreads) void gated_bwd_kernel(const GatedArgs a) {
    int c, b, g;
    if (!place<V>(a, c, b, g)) return;
    constexpr int T = kGatedTile;
    float inv_tau[V], G[V], lo[V], am1[V], dtau[V];
    const int64_t row = static_cast<int64_t>(b) * a.C + c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        inv_tau[i] = 1.f / a.tau[c + i];
        dtau[i] = lo[i] = am1[i] = 0.f;
        G[i] = a.dstate_out ? a.dstate_out[row + i] : 0.f;
    }
    for (int j = a.G - 1; j > g; --j) {
        const int64_t o = (static_cast<int64_t>(b) * a.G + j) * a.C + c;
#pragma unroll
        for (int i = 0; i < V; ++i) advance(G[i], lo[i], expm1_neg(a.ws_z[o + i]), a.ws_h[o + i]);
    }
    const int l0 = g * a.seg_len, l1 = min(l0 + a.seg_len, a.L);
    for (int t0 = l0 + (l1 - 1 - l0) / T * T; t0 >= l0; t0 -= T) {
        float h[T][V];  // the state before each token
        float hc[V], hl[V];
        const float *ck = a.ckpt + (static_cast<int64_t>(b) * a.tiles + t0 / T) * a.C + c;
#pragma unroll
        for (int i = 0; i < V; ++i) hc[i] = ck[i], hl[i] = 0.f;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int l = min(t0 + t, l1 - 1);
            float x[V], s[V], gt[V];
            unpack<DT, V>(*at<DT, V>(a.x, b, l, c), x);
            unpack<DT, V>(*at<DT, V>(a.step, b, l, c), s);
            unpack<DT, V>(*at<DT, V>(a.gate, b, l, c), gt);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[t][i] = hc[i];
                float z, d;
                decay(s[i], inv_tau[i], z, d);
                advance(hc[i], hl[i], d, __builtin_amdgcn_sqrtf(-d * (2.f + d)) * sigmoid(gt[i]) * x[i]);
            }
        }
#pragma unroll
        for (int t = T - 1; t >= 0; --t) {
            const int l = t0 + t;
            if (l >= l1) continue;
            float x[V], s[V], gt[V], dy[V], dx[V], ds[V], dg[V];
            unpack<DT, V>(*at<DT, V>(a.x, b, l, c), x);
            unpack<DT, V>(*at<DT, V>(a.step, b, l, c), s);
            unpack<DT, V>(*at<DT, V>(a.gate, b, l, c), gt);
            unpack<DT, V>(*at<DT, V>(a.dy, b, l, c), dy);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float e;
                advance(G[i], lo[i], am1[i], dy[i]);
                const float soft = softplus(s[i], e), z = clamp_step(soft) * inv_tau[i];
                am1[i] = expm1_neg(z);
                const float q = -am1[i] * (2.f + am1[i]), rq = __builtin_amdgcn_rsqf(q), n = q * rq, sg = sigmoid(gt[i]);
                const float al = 1.f + am1[i], Gx = G[i] * x[i];
                dx[i] = G[i] * n * sg;
                dg[i] = Gx * n * sg * (1.f - sg);
                const float dz = al * (al * rq * sg * Gx - G[i] * h[t][i]);
                const float sp = __builtin_amdgcn_rcpf(1.f + e) * (s[i] < 0.f ? e : 1.f);  // softplus'
                ds[i] = soft < kStepMin || soft > kStepMax ? 0.f : dz * inv_tau[i] * sp;
                dtau[i] -= dz * z * inv_tau[i];
            }
            *at_out<DT, V>(a.dx, b, l, c) = pack<DT, V>(dx);
            *at_out<DT, V>(a.dstep, b, l, c) = pack<DT, V>(ds);
            *at_out<DT, V>(a.dgate, b, l, c) = pack<DT, V>(dg);
        }
    }
    const int64_t o = (static_cast<int64_t>(b) * a.G + g) * a.C + c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        a.dtau_part[o + i] = dtau[i];
        if (g == 0 && a.dstate_in) a.dstate_in[row + i] = fmaf(am1[i], G[i], G[i]);
    }
}

// dtau[c] = the sum of the segments' parts, in order
__global__ __launch_bounds__(kGatedThreads) void gated_dtau_kernel(const GatedArgs a) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.C) return;
    float s = 0.f;
    for (int64_t j = 0; j < static_cast<int64_t>(a.B) * a.G; ++j) s += a.dtau_part[j * a.C + c];
    a.dtau[c] = s;
}

// ------------------------------------------------------------------ launch
namespace {

// Channels a lane: 4 bytes where every row allows it.
int lane_channels(const GatedArgs &a) {
    const int es = a.dt == PRIME_F32 ? 4 : 2, v = 2;
    if (a.C % v) return 1;
    for (const GatedView *t : {&a.x, &a.step, &a.gate, &a.y, &a.dy, &a.dx, &a.dstep, &a.dgate})
        if (t->data && (reinterpret_cast<uintptr_t>(t->data) % (v * es) || t->sb % v || t->sl % v)) return 1;
    return v;
}

// whole waves, at most kGatedThreads
dim3 threads(int lanes) { return dim3(lanes >= kGatedThreads ? kGatedThreads : (lanes + kWave - 1) / kWave * kWave); }

template <int DT, int V>
void forward(const GatedArgs &a, hipStream_t s) {
    const dim3 block = threads(a.C / V), grid(a.B * a.G, (a.C / V + block.x - 1) / block.x);
    if (a.G > 1) hipLaunchKernelGGL((gated_summary_kernel<DT, V>), grid, block, 0, s, a);
    hipLaunchKernelGGL((gated_scan_kernel<DT, V>), grid, block, 0, s, a);
}

template <int DT, int V>
void backward(const GatedArgs &a, hipStream_t s) {
    const dim3 block = threads(a.C / V), grid(a.B * a.G, (a.C / V + block.x - 1) / block.x);
    if (a.G > 1) hipLaunchKernelGGL((gated_bwd_summary_kernel<DT, V>), grid, block, 0, s, a);
    hipLaunchKernelGGL((gated_bwd_kernel<DT, V>), grid, block, 0, s, a);
    hipLaunchKernelGGL(gated_dtau_kernel, dim3((a.C + kGatedThreads - 1) / kGatedThreads), dim3(kGatedThreads), 0, s,
                       a);
}

template <int DT>
void run(const GatedArgs &a, bool bwd, hipStream_t s) {
    if (lane_channels(a) == 2) return bwd ? backward<DT, 2>(a, s) : forward<DT, 2>(a, s);
    return bwd ? backward<DT, 1>(a, s) : forward<DT, 1>(a, s);
}

}  // namespace

int gated_segments(int B, int L, int C, int *seg_len) {
    // about 4096 waves of 64 lanes with two channels each, segments of whole tiles
    const int64_t lanes = static_cast<int64_t>(B) * ((C + 1) / 2), tiles = (L + kGatedTile - 1) / kGatedTile;
    int64_t g = 4096 * 64 / lanes;
    g = g < 1 ? 1 : g > 64 ? 64 : g;
    if (g > tiles) g = tiles;
    const int64_t per = (tiles + g - 1) / g;
    *seg_len = static_cast<int>(per * kGatedTile);
    return static_cast<int>((tiles + per - 1) / per);
}

hipError_t launch_gated_scan(const GatedArgs &a, bool bwd, hipStream_t s) {
    if (a.dt == PRIME_BF16) run<PRIME_BF16>(a, bwd, s);
    else if (a.dt == PRIME_F16) run<PRIME_F16>(a, bwd, s);
    else run<PRIME_F32>(a, bwd, s);
    return hipGetLastError();
}

}  // namespace prime
