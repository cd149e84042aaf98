// Embedding lookup y_i = scale W[id_i], and its gradient dW[v] = scale sum_{i: id_i = v} dy_i.
//
// The gradient sorts the tokens by id, equal ones in their order, and sums over the sorted
// rows in fp32, each row of dy read once and each row of dW written once: no atomics on
// floats, so the order of every sum is fixed.
//   sort    counting passes of up to kMaxBits bits, from the lowest; a token without a
//           gradient (padding, an id outside the table) gets the key V and comes last
//   sum     a thread has 16 bytes of columns of a chunk of sorted rows.  An id whose rows all
//           lie in the chunk is finished there; one that reaches over its end or its start
//           leaves a part
//   join    the parts of ids that reach over a chunk's end, in order
// The rows of ids that do not occur are written as zeros by further workgroups of the sum.

#include "prime_kernels.h"

namespace prime {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kSortItems = 1024;  // at least, of a workgroup
constexpr int kSortBlocks = 512;  // at most
constexpr int kChunk = 32;        // sorted rows
constexpr int kZeroRows = 64;     // rows of the table that a workgroup looks at

struct __attribute__((packed, aligned(2))) Raw {  // 16 bytes of a row, wherever it starts
    u32x4 v;
};
template <int DT>
constexpr int kVec = DT == PRIME_F32 ? 4 : 8;

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

// The VE columns of a vector of a row of C: the last vector ends with the row, and where C is
// not a multiple of VE it shares columns with the one before.  Rows shorter than a vector go
// element by element.
template <int DT>
struct Columns {
    static constexpr int VE = kVec<DT>, es = DT == PRIME_F32 ? 4 : 2;
    int64_t offset;  // bytes
    int short_row;   // C where it is below VE, else 0
    __device__ __forceinline__ Columns(int vec, int C) {
        short_row = C < VE ? C : 0;
        const int e = vec * VE;
        offset = static_cast<int64_t>(short_row ? 0 : e + VE <= C ? e : C - VE) * es;
    }
    __device__ __forceinline__ u32x4 load(const void *row) const {
        const char *p = static_cast<const char *>(row) + offset;
        if (short_row == 0) return reinterpret_cast<const Raw *>(p)->v;
        uint16_t h[8] = {};
        for (int k = 0; k < short_row * (es / 2); ++k) h[k] = reinterpret_cast<const uint16_t *>(p)[k];
        return __builtin_bit_cast(u32x4, h);
    }
    __device__ __forceinline__ void store(void *row, const u32x4 &v) const {
        char *p = static_cast<char *>(row) + offset;
        if (short_row == 0) {
            reinterpret_cast<Raw *>(p)->v = v;
            return;
        }
        struct Halves { uint16_t h[8]; } h = __builtin_bit_cast(Halves, v);
        for (int k = 0; k < short_row * (es / 2); ++k) reinterpret_cast<uint16_t *>(p)[k] = h.h[k];
    }
};

__device__ __forceinline__ int64_t load_id(const EmbeddingArgs &a, int64_t i) {
    return a.ids64 ? static_cast<const int64_t *>(a.ids)[i] : static_cast<const int32_t *>(a.ids)[i];
}

__device__ __forceinline__ uint32_t sort_key(const EmbeddingArgs &a, int64_t i) {
    const int64_t id = load_id(a, i);
    return id < 0 || id >= a.V || id == a.padding ? static_cast<uint32_t>(a.V) : static_cast<uint32_t>(id);
}

}  // namespace

// Rows [first, first + rows) of the output, 16 bytes a thread.
template <int DT, bool SCALE>
__global__ __launch_bounds__(kThreads) void embedding_kernel(const EmbeddingArgs a, int64_t first, int rows, int vecs) {
    constexpr int VE = kVec<DT>, es = Columns<DT>::es;
    const uint32_t item = blockIdx.x * kThreads + threadIdx.x, r = item / static_cast<uint32_t>(vecs);
    if (r >= static_cast<uint32_t>(rows)) return;
    const Columns<DT> at(item - r * vecs, a.C);
    const int64_t i = first + r, id = load_id(a, i);
    u32x4 v = {0, 0, 0, 0};
    if (id >= 0 && id < a.V) {
        v = at.load(static_cast<const char *>(a.weight) + id * a.ldw * es);
        if constexpr (SCALE) {
            float x[VE];
            widen<DT>(v, x);
#pragma unroll
            for (int j = 0; j < VE; ++j) x[j] *= a.scale;
            v = narrow<DT>(x);
        }
    }
    at.store(static_cast<char *>(a.out) + i * a.C * es, v);
}

// One counting pass: keys and positions in, their digits' counts out, or (SCATTER) both in the
// digits' order.  FIRST: the keys are the ids', the positions the tokens' own.
template <bool FIRST, bool SCATTER>
__global__ __launch_bounds__(kThreads) void embedding_sort_kernel(const EmbeddingArgs a, const uint32_t *keys,
                                                                  const uint32_t *index, uint32_t *keys_out,
                                                                  uint32_t *index_out, uint32_t *hist, int shift,
                                                                  int bits, int items) {
    __shared__ uint32_t count[kWaves][kMaxBins];
    __shared__ uint32_t wave_total[kWaves];
    const int bins = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    for (int b = tid; b < kWaves * kMaxBins; b += kThreads) (&count[0][0])[b] = 0;
    __syncthreads();
    // a wave has `items` / kWaves tokens that lie one after the other
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * items + wave * (items / kWaves);
    const int64_t end = begin + items / kWaves < a.n ? begin + items / kWaves : a.n;
    auto key_of = [&](int64_t i) { return FIRST ? sort_key(a, i) : keys[i]; };
    for (int64_t i = begin + lane; i < end; i += kWave) atomicAdd(&count[wave][key_of(i) >> shift & (bins - 1)], 1u);
    __syncthreads();
    if constexpr (!SCATTER) {
        for (int b = tid; b < bins; b += kThreads) {
            uint32_t sum = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += count[w][b];
            hist[static_cast<int64_t>(blockIdx.x) * bins + b] = sum;
        }
    } else {
        // where each digit of this workgroup starts: behind the lower digits of all workgroups
        // and behind its own of the workgroups before.  Thread t has the digits 2 t, 2 t + 1.
        uint32_t total[2] = {}, before[2] = {};
        const int blocks = gridDim.x;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int b = 2 * tid + k;
            if (b >= bins) continue;
#pragma unroll 8
            for (int q = 0; q < blocks; ++q) {
                const uint32_t h = hist[static_cast<int64_t>(q) * bins + b];
                total[k] += h;
                before[k] += q < static_cast<int>(blockIdx.x) ? h : 0;
            }
        }
        uint32_t sum = total[0] + total[1], scan = sum;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const uint32_t v = __shfl_up(scan, o, kWave);
            scan += lane >= o ? v : 0;
        }
        if (lane == kWave - 1) wave_total[wave] = scan;
        __syncthreads();
        scan -= sum;
        for (int w = 0; w < wave; ++w) scan += wave_total[w];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int b = 2 * tid + k;
            if (b >= bins) continue;
            uint32_t at = scan + before[k];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const uint32_t c = count[w][b];
                count[w][b] = at;
                at += c;
            }
            scan += total[k];
        }
        __syncthreads();
        // 64 tokens at a time: those of one digit find each other by its bits
        volatile uint32_t *next = count[wave];
        for (int64_t i0 = begin; i0 < end; i0 += kWave) {
            const int64_t i = i0 + lane;
            const bool in = i < end;
            const uint32_t key = in ? key_of(i) : 0, digit = key >> shift & (bins - 1);
            uint64_t peers = __ballot(in);
            for (int b = 0; b < bits; ++b) {
                const uint64_t one = __ballot(digit >> b & 1);
                peers &= digit >> b & 1 ? one : ~one;
            }
            const int below = __popcll(peers & ((1ull << lane) - 1));
            uint32_t at = 0;
            if (in) at = next[digit];
            __builtin_amdgcn_wave_barrier();
            if (in && below == 0) next[digit] = at + __popcll(peers);
            __builtin_amdgcn_wave_barrier();
            if (in) {
                keys_out[at + below] = key;
                index_out[at + below] = FIRST ? static_cast<uint32_t>(i) : index[i];
            }
        }
    }
}

// Workgroups below `sum_blocks`: chunks of sorted rows, 16 bytes of columns a thread.  The
// others: the table's rows without a token.  part: [chunks][2][vecs VE], of the id that reaches
// in from the chunk before (0) and of the one that begins here and reaches on (1).
template <int DT>
__global__ __launch_bounds__(kThreads) void embedding_sum_kernel(const EmbeddingArgs a, const uint32_t *keys,
                                                                 const uint32_t *index, float *part, int vecs,
                                                                 uint32_t sum_blocks) {
    constexpr int VE = kVec<DT>, es = Columns<DT>::es;
    const uint32_t V = static_cast<uint32_t>(a.V), n = static_cast<uint32_t>(a.n);
    char *dw = static_cast<char *>(a.dweight);
    if (blockIdx.x >= sum_blocks) {
        __shared__ uint32_t absent[kZeroRows];
        const uint32_t first = (blockIdx.x - sum_blocks) * kZeroRows;
        if (threadIdx.x < kZeroRows) {
            const uint32_t v = first + threadIdx.x;
            uint32_t lo = 0, hi = n;  // the first place with a key of at least v
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                if (keys[mid] < v) lo = mid + 1;
                else hi = mid;
            }
            absent[threadIdx.x] = v < V && !(lo < n && keys[lo] == v);
        }
        __syncthreads();
        const uint32_t items = static_cast<uint32_t>(vecs) * kZeroRows;
        for (uint32_t q = threadIdx.x; q < items; q += kThreads) {
            const uint32_t r = q / vecs;
            if (absent[r])
                Columns<DT>(q - r * vecs, a.C).store(dw + static_cast<int64_t>(first + r) * a.C * es, u32x4{0, 0, 0, 0});
        }
        return;
    }
    const uint32_t item = blockIdx.x * kThreads + threadIdx.x, chunk = item / static_cast<uint32_t>(vecs);
    const uint32_t begin = chunk * kChunk;
    if (begin >= n) return;
    const int vec = item - chunk * vecs;
    const Columns<DT> at(vec, a.C);
    const uint32_t end = begin + kChunk < n ? begin + kChunk : n;
    const uint32_t prior = begin > 0 ? keys[begin - 1] : ~0u, follows = end < n ? keys[end] : ~0u;
    float acc[VE] = {};
    uint32_t cur = keys[begin];
    bool reaches_in = cur == prior;
    auto finish = [&](bool reaches_on) {
        if (cur >= V) return;
        if (reaches_in || reaches_on) {
            float *p = part + ((static_cast<int64_t>(chunk) * 2 + (reaches_in ? 0 : 1)) * vecs + vec) * VE;
#pragma unroll
            for (int j = 0; j < VE; ++j) p[j] = acc[j];
        } else {
            float x[VE];
#pragma unroll
            for (int j = 0; j < VE; ++j) x[j] = acc[j] * a.scale;
            at.store(dw + static_cast<int64_t>(cur) * a.C * es, narrow<DT>(x));
        }
    };
    constexpr int U = 8;
    for (uint32_t i = begin; i < end; i += U) {
        uint32_t key[U];
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            key[u] = i + u < end ? keys[i + u] : V;
            v[u] = u32x4{0, 0, 0, 0};
            if (key[u] < V) v[u] = at.load(static_cast<const char *>(a.dy) + static_cast<int64_t>(index[i + u]) * a.ldy * es);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= end) break;
            if (key[u] != cur) {
                finish(false);
                cur = key[u];
                reaches_in = false;
#pragma unroll
                for (int j = 0; j < VE; ++j) acc[j] = 0.f;
            }
            float x[VE];
            widen<DT>(v[u], x);
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] += x[j];
        }
    }
    finish(cur == follows);
}

// The ids that begin in a chunk and reach over its end: their parts, in order.
template <int DT>
__global__ __launch_bounds__(kThreads) void embedding_join_kernel(const EmbeddingArgs a, const uint32_t *keys,
                                                                  const float *part, int vecs) {
    constexpr int VE = kVec<DT>, es = Columns<DT>::es;
    const uint32_t n = static_cast<uint32_t>(a.n);
    const uint32_t item = blockIdx.x * kThreads + threadIdx.x, chunk = item / static_cast<uint32_t>(vecs);
    const uint32_t begin = chunk * kChunk, end = begin + kChunk;
    if (end >= n) return;
    const uint32_t key = keys[end];
    if (key >= static_cast<uint32_t>(a.V) || keys[end - 1] != key || (keys[begin] == key && begin > 0 && keys[begin - 1] == key))
        return;
    const int vec = item - chunk * vecs;
    float acc[VE];
    const float *p = part + ((static_cast<int64_t>(chunk) * 2 + 1) * vecs + vec) * VE;
#pragma unroll
    for (int j = 0; j < VE; ++j) acc[j] = p[j];
    for (uint32_t c = chunk + 1; c * kChunk < n && keys[c * kChunk] == key; ++c) {
        p = part + ((static_cast<int64_t>(c) * 2) * vecs + vec) * VE;
#pragma unroll
        for (int j = 0; j < VE; ++j) acc[j] += p[j];
    }
#pragma unroll
    for (int j = 0; j < VE; ++j) acc[j] *= a.scale;
    Columns<DT>(vec, a.C).store(static_cast<char *>(a.dweight) + static_cast<int64_t>(key) * a.C * es, narrow<DT>(acc));
}

namespace {

struct Plan {
    int passes, bits, blocks, items;
    int64_t chunks;
    size_t keys_bytes, hist_bytes, part_bytes;
};
Plan plan(int64_t n, int64_t V, int C) {
    Plan p{};
    int bits = 1;
    while (bits < 32 && (static_cast<int64_t>(1) << bits) <= V) ++bits;  // keys 0 .. V
    p.passes = (bits + kMaxBits - 1) / kMaxBits;
    p.bits = (bits + p.passes - 1) / p.passes;
    const int64_t per = (n + kSortBlocks - 1) / kSortBlocks, items = per < kSortItems ? kSortItems : (per + kThreads - 1) / kThreads * kThreads;
    p.items = static_cast<int>(items);
    p.blocks = static_cast<int>((n + items - 1) / items);
    p.chunks = (n + kChunk - 1) / kChunk;
    auto round = [](size_t b) { return (b + 255) / 256 * 256; };
    p.keys_bytes = round(static_cast<size_t>(n) * 4);
    p.hist_bytes = round(static_cast<size_t>(p.blocks) * (size_t{1} << p.bits) * 4);
    p.part_bytes = static_cast<size_t>(p.chunks) * 2 * ((static_cast<size_t>(C) + 7) / 8 * 8) * 4;
    return p;
}

template <int DT>
void run(const EmbeddingArgs &a, hipStream_t s) {
    const int vecs = (a.C + kVec<DT> - 1) / kVec<DT>;
    const int64_t most = (int64_t{1} << 30) / vecs;  // rows of a launch
    for (int64_t first = 0; first < a.n; first += most) {
        const int rows = static_cast<int>(a.n - first < most ? a.n - first : most);
        const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(rows) * vecs + kThreads - 1) / kThreads));
        if (a.scale == 1.f) hipLaunchKernelGGL((embedding_kernel<DT, false>), grid, dim3(kThreads), 0, s, a, first, rows, vecs);
        else hipLaunchKernelGGL((embedding_kernel<DT, true>), grid, dim3(kThreads), 0, s, a, first, rows, vecs);
    }
}

template <int DT>
void run_backward(const EmbeddingArgs &a, hipStream_t s) {
    const Plan p = plan(a.n, a.V, a.C);
    const int vecs = (a.C + kVec<DT> - 1) / kVec<DT>;
    char *w = static_cast<char *>(a.workspace);
    uint32_t *buf[4];
    for (int i = 0; i < 4; ++i) buf[i] = reinterpret_cast<uint32_t *>(w + i * p.keys_bytes);
    uint32_t *hist = reinterpret_cast<uint32_t *>(w + 4 * p.keys_bytes);
    float *part = reinterpret_cast<float *>(w + 4 * p.keys_bytes + p.hist_bytes);
    const uint32_t *keys = nullptr, *index = nullptr;
    const dim3 grid(p.blocks), block(kThreads);
    for (int i = 0; i < p.passes; ++i) {
        uint32_t *ko = buf[i % 2 * 2], *io = buf[i % 2 * 2 + 1];
        const int shift = i * p.bits;
        if (i == 0) {
            hipLaunchKernelGGL((embedding_sort_kernel<true, false>), grid, block, 0, s, a, keys, index, ko, io, hist, shift, p.bits, p.items);
            hipLaunchKernelGGL((embedding_sort_kernel<true, true>), grid, block, 0, s, a, keys, index, ko, io, hist, shift, p.bits, p.items);
        } else {
            hipLaunchKernelGGL((embedding_sort_kernel<false, false>), grid, block, 0, s, a, keys, index, ko, io, hist, shift, p.bits, p.items);
            hipLaunchKernelGGL((embedding_sort_kernel<false, true>), grid, block, 0, s, a, keys, index, ko, io, hist, shift, p.bits, p.items);
        }
        keys = ko, index = io;
    }
    const uint32_t sum_blocks = static_cast<uint32_t>((p.chunks * vecs + kThreads - 1) / kThreads);
    const uint32_t zero_blocks = static_cast<uint32_t>((a.V + kZeroRows - 1) / kZeroRows);
    hipLaunchKernelGGL(embedding_sum_kernel<DT>, dim3(sum_blocks + zero_blocks), block, 0, s, a, keys, index, part, vecs, sum_blocks);
    hipLaunchKernelGGL(embedding_join_kernel<DT>, dim3(sum_blocks), block, 0, s, a, keys, part, vecs);
}

}  // namespace

size_t embedding_workspace_bytes(int64_t n, int64_t V, int C) {
    const Plan p = plan(n, V, C);
    return 4 * p.keys_bytes + p.hist_bytes + p.part_bytes;
}

bool embedding_grid_fits(int64_t n, int64_t V, int C, int dt) {
    const Plan p = plan(n, V, C);
    const int64_t vecs = (C + (dt == PRIME_F32 ? 3 : 7)) / (dt == PRIME_F32 ? 4 : 8);
    return p.chunks * vecs + ((V + kZeroRows - 1) / kZeroRows + 1) * kThreads < (int64_t{1} << 32) - kThreads;
}

hipError_t launch_embedding(const EmbeddingArgs &a, bool backward, hipStream_t stream) {
    if (a.dt == PRIME_BF16) backward ? run_backward<PRIME_BF16>(a, stream) : run<PRIME_BF16>(a, stream);
    else if (a.dt == PRIME_F16) backward ? run_backward<PRIME_F16>(a, stream) : run<PRIME_F16>(a, stream);
    else backward ? run_backward<PRIME_F32>(a, stream) : run<PRIME_F32>(a, stream);
    return hipGetLastError();
}

}  // namespace prime
