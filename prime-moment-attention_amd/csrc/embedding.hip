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
// The sort is short and leaves most of the card idle: further workgroups of its launches fill
// the whole gradient with zeros meanwhile, which the rows with a token then replace.

#include "prime_kernels.h"

namespace prime {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kFewTokens = 8192;
constexpr int kSortItems = 4096;  // at least, of a workgroup
constexpr int kSortBlocks = 512;  // at most
constexpr int kChunk = 32;        // sorted rows
constexpr int kRows = 8;          // of a chunk, on their way at once

// The part [from, to) of the gradient's 16-byte blocks that a launch's workgroups from `block`
// on fill with zeros.
struct Fill {
    int block;
    int64_t from, to;
};

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

// A workgroup's share of the gradient's zeros: 16-byte stores over [from, to) of the table's
// 16-byte blocks, the elements before the first and behind the last by the share that has
// them.
__device__ __forceinline__ void fill_zeros(const EmbeddingArgs &a, const Fill &f) {
    const int es = a.dt == PRIME_F32 ? 4 : 2;
    char *dw = static_cast<char *>(a.dweight);
    const uintptr_t begin = reinterpret_cast<uintptr_t>(dw), end = begin + a.V * a.C * es;
    const uintptr_t first = (begin + 15) & ~uintptr_t{15}, last = end & ~uintptr_t{15};
    constexpr int U = 4;
    u32x4 *p = reinterpret_cast<u32x4 *>(first);
    const int64_t at = f.from + static_cast<int64_t>(blockIdx.x - f.block) * (kSortThreads * U) + threadIdx.x;
    const int64_t blocks = first < last ? static_cast<int64_t>(last - first) / 16 : 0, to = f.to < blocks ? f.to : blocks;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (at + u * kSortThreads < to) p[at + u * kSortThreads] = u32x4{0, 0, 0, 0};
    if (f.from == 0 && blockIdx.x == f.block) {
        const uintptr_t head = first < end ? first : end, tail = last > head ? last : head;
        for (uintptr_t q = begin + threadIdx.x * 2; q < head; q += kSortThreads * 2) *reinterpret_cast<uint16_t *>(q) = 0;
        for (uintptr_t q = tail + threadIdx.x * 2; q < end; q += kSortThreads * 2) *reinterpret_cast<uint16_t *>(q) = 0;
    }
}

// The sum of v over the threads before this one.
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t *wave_total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t scan = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t u = __shfl_up(scan, o, kWave);
        scan += lane >= o ? u : 0;
    }
    if (lane == kWave - 1) wave_total[wave] = scan;
    __syncthreads();
    uint32_t before = scan - v;
    for (int w = 0; w < wave; ++w) before += wave_total[w];
    return before;
}

// Items [begin, end) of a wave to the places that `next` counts up for their digits, 64 at a
// time: those of one digit find each other by its bits.
template <typename K, typename P>
__device__ __forceinline__ void place_items(volatile uint32_t *next, int64_t begin, int64_t end, int shift, int bits, K key_of, P put) {
    const int lane = threadIdx.x % kWave;
    for (int64_t i0 = begin; i0 < end; i0 += kWave) {
        const int64_t i = i0 + lane;
        const bool in = i < end;
        const uint32_t key = in ? key_of(i) : 0, digit = key >> shift & ((1u << bits) - 1);
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
        if (in) put(at + below, key, i);
    }
}

// One counting pass: keys and positions in, their digits' counts out, or (SCATTER) both in the
// digits' order.  FIRST: the keys are the ids', the positions the tokens' own.  Workgroups from
// `fill.block` on write zeros meanwhile.
template <bool FIRST, bool SCATTER>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(const EmbeddingArgs a, const uint32_t *keys,
                                                                      const uint32_t *index, uint32_t *keys_out,
                                                                      uint32_t *index_out, uint32_t *hist, int shift,
                                                                      int bits, int items, const Fill fill) {
    __shared__ uint32_t count[kSortWaves][kMaxBins];
    __shared__ uint32_t total[kSortThreads], before[kSortThreads], wave_total[kSortWaves];
    if (static_cast<int>(blockIdx.x) >= fill.block) {
        fill_zeros(a, fill);
        return;
    }
    const int bins = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, blocks = fill.block;
    if constexpr (SCATTER) {
        // each digit's count in all workgroups and in those before this one, by threads that
        // share the workgroups between them
        const int bin = tid & (bins - 1), share = kSortThreads / bins;
        uint32_t t = 0, b = 0;
#pragma unroll 8
        for (int q = tid / bins; q < blocks; q += share) {
            const uint32_t h = hist[static_cast<int64_t>(q) * bins + bin];
            t += h;
            b += q < static_cast<int>(blockIdx.x) ? h : 0;
        }
        total[tid] = t, before[tid] = b;
    }
    for (int b = tid; b < kSortWaves * kMaxBins; b += kSortThreads) (&count[0][0])[b] = 0;
    __syncthreads();
    // a wave has `items` / kSortWaves tokens that lie one after the other
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * items + wave * (items / kSortWaves);
    const int64_t end = begin + items / kSortWaves < a.n ? begin + items / kSortWaves : a.n;
    auto key_of = [&](int64_t i) { return FIRST ? sort_key(a, i) : keys[i]; };
#pragma unroll 4
    for (int64_t i = begin + lane; i < end; i += kWave) atomicAdd(&count[wave][key_of(i) >> shift & (bins - 1)], 1u);
    __syncthreads();
    uint32_t here = 0, all = 0;
    if (tid < bins) {
        if constexpr (SCATTER) {
            for (int q = tid; q < kSortThreads; q += bins) all += total[q], here += before[q];
        } else {
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) all += count[w][tid];
            hist[static_cast<int64_t>(blockIdx.x) * bins + tid] = all;
        }
    }
    if constexpr (SCATTER) {
        here += scan_before(all, wave_total);
        if (tid < bins) {
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const uint32_t c = count[w][tid];
                count[w][tid] = here;
                here += c;
            }
        }
        __syncthreads();
        place_items(count[wave], begin, end, shift, bits, key_of, [&](uint32_t at, uint32_t key, int64_t i) {
            keys_out[at] = key;
            index_out[at] = FIRST ? static_cast<uint32_t>(i) : index[i];
        });
    }
}

// All passes over at most kFewTokens tokens by one workgroup, in LDS; the others write zeros.
__global__ __launch_bounds__(kSortThreads) void embedding_sort_few_kernel(const EmbeddingArgs a, uint32_t *keys_out,
                                                                          uint32_t *index_out, int passes, int bits,
                                                                          const Fill fill) {
    __shared__ uint32_t count[kSortWaves][kMaxBins];
    __shared__ uint32_t wave_total[kSortWaves];
    __shared__ uint32_t keys[2][kFewTokens];
    __shared__ uint16_t index[2][kFewTokens];
    if (static_cast<int>(blockIdx.x) >= fill.block) {
        fill_zeros(a, fill);
        return;
    }
    const int bins = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, n = static_cast<int>(a.n);
    const int items = (n + kSortThreads - 1) / kSortThreads * kWave, begin = wave * items, end = min(begin + items, n);
#pragma unroll 4
    for (int i = tid; i < n; i += kSortThreads) keys[0][i] = sort_key(a, i), index[0][i] = static_cast<uint16_t>(i);
    for (int p = 0; p < passes; ++p) {
        const uint32_t *k = keys[p & 1];
        const uint16_t *x = index[p & 1];
        const int shift = p * bits;
        for (int b = tid; b < kSortWaves * kMaxBins; b += kSortThreads) (&count[0][0])[b] = 0;
        __syncthreads();
        for (int i = begin + lane; i < end; i += kWave) atomicAdd(&count[wave][k[i] >> shift & (bins - 1)], 1u);
        __syncthreads();
        uint32_t all = 0;
        if (tid < bins) {
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) all += count[w][tid];
        }
        uint32_t here = scan_before(all, wave_total);
        if (tid < bins) {
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const uint32_t c = count[w][tid];
                count[w][tid] = here;
                here += c;
            }
        }
        __syncthreads();
        const bool last = p + 1 == passes;
        place_items(count[wave], begin, end, shift, bits, [&](int64_t i) { return k[i]; }, [&](uint32_t at, uint32_t key, int64_t i) {
            if (last) {
                keys_out[at] = key;
                index_out[at] = x[i];
            } else {
                keys[~p & 1][at] = key;
                index[~p & 1][at] = x[i];
            }
        });
        __syncthreads();
    }
}

// Chunks of sorted rows, 16 bytes of columns a thread.  part: [chunks][2][vecs VE], of the id
// that reaches in from the chunk before (0) and of the one that begins here and reaches on (1).
template <int DT>
__global__ __launch_bounds__(kThreads) void embedding_sum_kernel(const EmbeddingArgs a, const uint32_t *keys,
                                                                 const uint32_t *index, float *part, int vecs) {
    constexpr int VE = kVec<DT>, es = Columns<DT>::es;
    const uint32_t V = static_cast<uint32_t>(a.V), n = static_cast<uint32_t>(a.n);
    char *dw = static_cast<char *>(a.dweight);
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
    constexpr int U = kRows;
    uint32_t key[U], row[U];
    auto fetch = [&](uint32_t i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = i + u < end ? i + u : end - 1;
            key[u] = keys[q], row[u] = index[q];
        }
    };
    fetch(begin);
    for (uint32_t i = begin; i < end; i += U) {
        u32x4 v[U];
        uint32_t k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = key[u];
            v[u] = u32x4{0, 0, 0, 0};
            if (k[u] < V) v[u] = at.load(static_cast<const char *>(a.dy) + static_cast<int64_t>(row[u]) * a.ldy * es);
        }
        if (i + U < end) fetch(i + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= end) break;
            if (k[u] != cur) {
                finish(false);
                cur = k[u];
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

// The ids that begin in chunk blockIdx.x and reach over its end: their parts, wave w the w-th,
// (w + 4)-th .. of them, then the waves' sums; four columns a lane.
template <int DT>
__global__ __launch_bounds__(kThreads) void embedding_join_kernel(const EmbeddingArgs a, const uint32_t *keys,
                                                                  const float *part, int vecs) {
    constexpr int VE = kVec<DT>;
    __shared__ f32x4 sums[kWaves][kWave];
    __shared__ uint32_t reach[kWaves];
    const uint32_t n = static_cast<uint32_t>(a.n), chunk = blockIdx.x, begin = chunk * kChunk, end = begin + kChunk;
    if (end >= n) return;
    const uint32_t key = keys[end];
    if (key >= static_cast<uint32_t>(a.V) || keys[end - 1] != key || (begin > 0 && keys[begin - 1] == key)) return;
    // the chunks behind that begin with the id: the keys are sorted, so they are the first ones
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t count = 0;
    for (;;) {
        const uint64_t at = (static_cast<uint64_t>(chunk) + 1 + count + threadIdx.x) * kChunk;
        const uint32_t here = __popcll(__ballot(at < n && keys[at] == key));
        if (lane == 0) reach[wave] = here;
        __syncthreads();
        const uint32_t all = reach[0] + reach[1] + reach[2] + reach[3];
        __syncthreads();
        count += all;
        if (all < kThreads) break;
    }
    const int slot = (blockIdx.y * kWave + lane) * 4, width = vecs * VE;  // columns as the parts have them
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (slot < width) {
        // part 0 is this chunk's, part c > 0 that of the c-th chunk behind
        auto part_of = [&](uint32_t c) {
            return *reinterpret_cast<const f32x4 *>(part + (static_cast<int64_t>(chunk + c) * 2 + (c == 0)) * width + slot);
        };
#pragma unroll 8
        for (uint32_t c = wave; c <= count; c += kWaves) acc += part_of(c);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || slot >= width) return;
    acc = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    const int vec = slot / VE, first = a.C < VE ? 0 : vec * VE + VE <= a.C ? vec * VE : a.C - VE, col = first + slot % VE;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (col + j < a.C) store_elem(a.dweight, static_cast<int64_t>(key) * a.C + col + j, DT, acc[j] * a.scale);
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
    const int64_t per = (n + kSortBlocks - 1) / kSortBlocks;
    const int64_t items = per < kSortItems ? kSortItems : (per + kSortThreads - 1) / kSortThreads * kSortThreads;
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
    const dim3 sort(kSortThreads);
    // the launches of the sort, each with its share of the zeros
    const bool few = a.n <= kFewTokens;
    const int launches = few ? 1 : 2 * p.passes;
    const int64_t zeros = a.V * a.C * Columns<DT>::es / 16 + 1, share = (zeros + launches - 1) / launches;
    int launch = 0;
    auto next = [&](int blocks, Fill &f) {
        f.block = blocks;
        f.from = share * launch++;
        f.to = f.from + share;
        constexpr int per = kSortThreads * 4;
        return dim3(static_cast<unsigned>(blocks + (share + per - 1) / per));
    };
    Fill f;
    if (few) {
        const dim3 grid = next(1, f);
        hipLaunchKernelGGL(embedding_sort_few_kernel, grid, sort, 0, s, a, buf[0], buf[1], p.passes, p.bits, f);
        keys = buf[0], index = buf[1];
    }
    for (int i = 0; i < p.passes && !few; ++i) {
        uint32_t *ko = buf[i % 2 * 2], *io = buf[i % 2 * 2 + 1];
        const int shift = i * p.bits;
        for (int scatter = 0; scatter < 2; ++scatter) {
            const dim3 grid = next(p.blocks, f);
            const auto kernel = i == 0 ? (scatter ? embedding_sort_kernel<true, true> : embedding_sort_kernel<true, false>)
                                       : (scatter ? embedding_sort_kernel<false, true> : embedding_sort_kernel<false, false>);
            hipLaunchKernelGGL(kernel, grid, sort, 0, s, a, keys, index, ko, io, hist, shift, p.bits, p.items, f);
        }
        keys = ko, index = io;
    }
    const dim3 grid(static_cast<unsigned>((p.chunks * vecs + kThreads - 1) / kThreads)), block(kThreads);
    hipLaunchKernelGGL(embedding_sum_kernel<DT>, grid, block, 0, s, a, keys, index, part, vecs);
    const dim3 join(static_cast<unsigned>(p.chunks), static_cast<unsigned>((vecs * kVec<DT> + 4 * kWave - 1) / (4 * kWave)));
    if (p.chunks > 1) hipLaunchKernelGGL(embedding_join_kernel<DT>, join, block, 0, s, a, keys, part, vecs);
}

}  // namespace

size_t embedding_workspace_bytes(int64_t n, int64_t V, int C) {
    const Plan p = plan(n, V, C);
    return 4 * p.keys_bytes + p.hist_bytes + p.part_bytes;
}

bool embedding_grid_fits(int64_t n, int64_t V, int C, int dt) {
    const Plan p = plan(n, V, C);
    const int64_t vecs = (C + (dt == PRIME_F32 ? 3 : 7)) / (dt == PRIME_F32 ? 4 : 8), limit = (int64_t{1} << 32) - kSortThreads;
    const int64_t fill = V * C * (dt == PRIME_F32 ? 4 : 2) / 64 + kSortThreads;  // threads, of one launch at most
    return p.chunks * vecs < limit && p.chunks * kThreads < limit && fill + p.blocks * kSortThreads < limit;
}

hipError_t launch_embedding(const EmbeddingArgs &a, bool backward, hipStream_t stream) {
    if (a.dt == PRIME_BF16) backward ? run_backward<PRIME_BF16>(a, stream) : run<PRIME_BF16>(a, stream);
    else if (a.dt == PRIME_F16) backward ? run_backward<PRIME_F16>(a, stream) : run<PRIME_F16>(a, stream);
    else backward ? run_backward<PRIME_F32>(a, stream) : run<PRIME_F32>(a, stream);
    return hipGetLastError();
}

}  // namespace prime
