// Embedding lookup y_i = scale W[id_i], and its gradient dW[v] = scale sum_{i: id_i = v} dy_i.
//
// The gradient puts the tokens of one id side by side, in their order, and sums over these rows
// in fp32, each row of dy read once: no atomics on floats, so the order of every sum is fixed.
//   group   (token, id) pairs in the order of their ids' low bits, then of the others; a token
//           without a gradient (padding, an id outside the table) gets the id V and comes
//           last.  Up to kGroupTokens tokens in one launch, else by counting passes (sort)
//   sum     a wave has 64 vectors of columns of a chunk of rows.  An id whose rows end before
//           the next chunk does is finished where it begins; a longer one leaves a part in
//           each chunk
//   join    the parts of the long ones, in a fixed order
// Grouping leaves the memory system idle: further workgroups of its launches fill the whole
// gradient with zeros meanwhile, which the rows with a token then replace.

#include "prime_kernels.h"

namespace prime {

namespace {

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kGroups = 128;           // by the ids' low bits
constexpr int kGroupList = 2048;       // tokens of a group that are sorted in LDS
constexpr int kGroupTokens = 1 << 14;
constexpr int kSortItems = 4096;       // at least, of a workgroup
constexpr int kSortBlocks = 512;       // at most
constexpr int kFewRows = 16384;        // tokens, below which chunks are short
constexpr int kRows = 8;               // of a chunk, on their way at once, twice

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
// not a multiple of VE it shares columns with the one before.  SHORT: rows shorter than a
// vector, element by element.
template <int DT, bool SHORT>
struct Columns {
    static constexpr int VE = kVec<DT>, es = DT == PRIME_F32 ? 4 : 2;
    int64_t offset;  // bytes
    int C;
    __device__ __forceinline__ Columns(int vec, int C_) : C(C_) {
        const int e = vec * VE;
        offset = static_cast<int64_t>(SHORT ? 0 : e + VE <= C ? e : C - VE) * es;
    }
    __device__ __forceinline__ u32x4 load(const void *row) const {
        const char *p = static_cast<const char *>(row) + offset;
        if constexpr (!SHORT) return reinterpret_cast<const Raw *>(p)->v;
        uint16_t h[8] = {};
        for (int k = 0; k < C * (es / 2); ++k) h[k] = reinterpret_cast<const uint16_t *>(p)[k];
        return __builtin_bit_cast(u32x4, h);
    }
    __device__ __forceinline__ void store(void *row, const u32x4 &v) const {
        char *p = static_cast<char *>(row) + offset;
        if constexpr (!SHORT) {
            reinterpret_cast<Raw *>(p)->v = v;
            return;
        }
        struct Halves { uint16_t h[8]; } h = __builtin_bit_cast(Halves, v);
        for (int k = 0; k < C * (es / 2); ++k) reinterpret_cast<uint16_t *>(p)[k] = h.h[k];
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
template <int DT, bool SCALE, bool SHORT>
__global__ __launch_bounds__(kThreads) void embedding_kernel(const EmbeddingArgs a, int64_t first, int rows, int vecs) {
    constexpr int VE = kVec<DT>, es = Columns<DT, SHORT>::es;
    const uint32_t item = blockIdx.x * kThreads + threadIdx.x, r = item / static_cast<uint32_t>(vecs);
    if (r >= static_cast<uint32_t>(rows)) return;
    const Columns<DT, SHORT> at(item - r * vecs, a.C);
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

// 64 items of a wave (`in`: those that there are) to the places that `next` counts up for their
// digits: those of one digit find each other by its bits.
template <typename P>
__device__ __forceinline__ void place_64(volatile uint32_t *next, uint2 item, bool in, int shift, int bits, P put) {
    const int lane = threadIdx.x % kWave;
    const uint32_t digit = item.x >> shift & ((1u << bits) - 1);
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
    if (in) put(at + below, item);
}
// Items [begin, end) of a wave, four loads ahead.
template <typename K, typename P>
__device__ __forceinline__ void place_items(volatile uint32_t *next, int64_t begin, int64_t end, int shift, int bits, K item_of, P put) {
    const int lane = threadIdx.x % kWave;
    constexpr int U = 4;
    for (int64_t i0 = begin; i0 < end; i0 += U * kWave) {
        uint2 items[U];
#pragma unroll
        for (int u = 0; u < U; ++u) items[u] = item_of(min(i0 + u * kWave + lane, end - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) place_64(next, items[u], i0 + u * kWave + lane < end, shift, bits, put);
    }
}

// A counting pass of one workgroup over `count` items: every digit's place, then the items there.
template <typename K, typename P>
__device__ __forceinline__ void sort_pass(uint32_t (*tally)[kMaxBins], uint32_t *wave_total, uint32_t count, int shift,
                                          int bits, K item_of, P put) {
    const int bins = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const uint32_t items = (count + kSortThreads - 1) / kSortThreads * kWave, begin = min(wave * items, count), end = min(begin + items, count);
    for (int b = tid; b < kSortWaves * kMaxBins; b += kSortThreads) (&tally[0][0])[b] = 0;
    __syncthreads();
    for (uint32_t i = begin + lane; i < end; i += kWave) atomicAdd(&tally[wave][item_of(i).x >> shift & (bins - 1)], 1u);
    __syncthreads();
    uint32_t all = 0;
    if (tid < bins) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) all += tally[w][tid];
    }
    uint32_t here = scan_before(all, wave_total);
    if (tid < bins) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const uint32_t c = tally[w][tid];
            tally[w][tid] = here;
            here += c;
        }
    }
    __syncthreads();
    place_items(tally[wave], begin, end, shift, bits, item_of, put);
    __syncthreads();
}

// Workgroup g < kGroups: the tokens whose ids have the low bits g, in the order of the others.
// Each reads all ids, so where its tokens go it knows by itself: behind those of lower groups.
// Workgroup kGroups: the places behind all of them, for tokens without a gradient.  The
// others write zeros.
__global__ __launch_bounds__(kSortThreads) void embedding_group_kernel(const EmbeddingArgs a, uint2 *pairs, uint2 *other,
                                                                       int passes, int bits, const Fill fill) {
    constexpr int kLow = __builtin_ctz(kGroups);
    __shared__ uint32_t tally[kSortWaves][kMaxBins];
    __shared__ uint32_t wave_total[kSortWaves], wave_lower[kSortWaves];
    __shared__ uint2 list[2][kGroupList];
    if (static_cast<int>(blockIdx.x) >= fill.block) {
        fill_zeros(a, fill);
        return;
    }
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, n = static_cast<int>(a.n);
    const uint32_t group = blockIdx.x, V = static_cast<uint32_t>(a.V), padding = static_cast<uint32_t>(a.padding);
    // a wave has the tokens [begin, end), U 64s of them at a time
    constexpr int U = 8;
    const int items = (n + kSortThreads - 1) / kSortThreads * kWave, begin = min(wave * items, n), end = min(begin + items, n);
    auto each = [&](auto f) {
        for (int i0 = begin; i0 < end; i0 += U * kWave) {
            uint2 word[U];  // all loads first
            if (a.ids64) {
#pragma unroll
                for (int u = 0; u < U; ++u) word[u] = static_cast<const uint2 *>(a.ids)[min(i0 + u * kWave + lane, n - 1)];
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) word[u] = uint2{static_cast<const uint32_t *>(a.ids)[min(i0 + u * kWave + lane, n - 1)], 0};
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * kWave + lane;
                f(word[u].x, i < end && word[u].y == 0 && word[u].x < V && word[u].x != padding, i);
            }
        }
    };
    uint32_t mine = 0, lower = 0;  // of the wave
    each([&](uint32_t id, bool valid, int) {
        const uint32_t low = id & (kGroups - 1);
        mine += __popcll(__ballot(valid && low == group));
        lower += __popcll(__ballot(valid && low < group));
    });
    if (lane == 0) wave_total[wave] = mine, wave_lower[wave] = lower;
    __syncthreads();
    uint32_t base = 0, count = 0, at = 0;  // the group's first place and its tokens; the wave's first among them
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
        at += w < wave ? wave_total[w] : 0;
        count += wave_total[w];
        base += wave_lower[w];
    }
    if (group == kGroups) {
        for (uint32_t i = base + tid; i < static_cast<uint32_t>(n); i += kSortThreads) pairs[i] = uint2{V, 0};
        return;
    }
    if (count == 0) return;
    const bool in_lds = count <= kGroupList;
    // round r writes to `pairs` where passes - r is even
    uint2 *first = passes == 0 ? pairs + base : in_lds ? list[0] : (passes & 1 ? other : pairs) + base;
    each([&](uint32_t id, bool valid, int i) {
        const bool in = valid && (id & (kGroups - 1)) == group;
        const uint64_t all = __ballot(in);
        if (in) first[at + __popcll(all & ((1ull << lane) - 1))] = uint2{id, static_cast<uint32_t>(i)};
        at += __popcll(all);
    });
    __syncthreads();
    for (int p = 0; p < passes; ++p) {
        const int shift = kLow + p * bits;
        uint2 *to = (passes - p) & 1 ? pairs + base : other + base;
        if (in_lds) {
            const uint2 *from = list[p & 1];
            if (p + 1 == passes)
                sort_pass(tally, wave_total, count, shift, bits, [&](uint32_t i) { return from[i]; }, [&](uint32_t i, uint2 v) { pairs[base + i] = v; });
            else
                sort_pass(tally, wave_total, count, shift, bits, [&](uint32_t i) { return from[i]; }, [&](uint32_t i, uint2 v) { list[~p & 1][i] = v; });
        } else {
            const uint2 *from = (passes - p) & 1 ? other + base : pairs + base;
            sort_pass(tally, wave_total, count, shift, bits, [&](uint32_t i) { return from[i]; }, [&](uint32_t i, uint2 v) { to[i] = v; });
        }
    }
}

// One counting pass over many tokens: their digits' counts, or (SCATTER) the pairs in the
// digits' order.  FIRST: the pairs are the ids' and the tokens' own.  ONE: a workgroup has
// kSortItems tokens, which its threads hold.  Workgroups from `fill.block` on write zeros
// meanwhile.
template <bool FIRST, bool SCATTER, bool ONE>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(const EmbeddingArgs a, const uint2 *pairs,
                                                                      uint2 *pairs_out, uint32_t *hist, int shift,
                                                                      int bits, int items, const Fill fill) {
    constexpr int R = kSortItems / kSortThreads;
    __shared__ uint32_t count[kSortWaves][kMaxBins];
    __shared__ uint32_t total[kSortThreads], before[kSortThreads], wave_total[kSortWaves];
    if (static_cast<int>(blockIdx.x) >= fill.block) {
        fill_zeros(a, fill);
        return;
    }
    const int bins = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, blocks = fill.block;
    if constexpr (ONE) items = kSortItems;
    // a wave has `items` / kSortWaves tokens that lie one after the other
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * items + wave * (items / kSortWaves);
    const int64_t end = begin + items / kSortWaves < a.n ? begin + items / kSortWaves : a.n;
    auto item_of = [&](int64_t i) { return FIRST ? uint2{sort_key(a, i), static_cast<uint32_t>(i)} : pairs[i]; };
    uint2 held[R];
    if constexpr (ONE) {
#pragma unroll
        for (int r = 0; r < R; ++r) held[r] = item_of(min(begin + r * kWave + lane, a.n - 1));
    }
    if constexpr (SCATTER) {
        // each digit's count in all workgroups and in those before this one, by threads that
        // share the workgroups between them
        constexpr int U = 8;
        const int bin = tid & (bins - 1), share = kSortThreads / bins;
        uint32_t t = 0, b = 0;
        for (int q = tid / bins; q < blocks; q += U * share) {
            uint32_t h[U];
#pragma unroll
            for (int u = 0; u < U; ++u) h[u] = hist[static_cast<int64_t>(min(q + u * share, blocks - 1)) * bins + bin];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                t += q + u * share < blocks ? h[u] : 0;
                b += q + u * share < static_cast<int>(blockIdx.x) ? h[u] : 0;
            }
        }
        total[tid] = t, before[tid] = b;
    }
    for (int b = tid; b < kSortWaves * kMaxBins; b += kSortThreads) (&count[0][0])[b] = 0;
    __syncthreads();
    auto tally = [&](uint2 item) { atomicAdd(&count[wave][item.x >> shift & (bins - 1)], 1u); };
    if constexpr (ONE) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (begin + r * kWave + lane < end) tally(held[r]);
    } else {
        for (int64_t i = begin + lane; i < end; i += kWave) tally(item_of(i));
    }
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
        auto put = [&](uint32_t at, uint2 v) { pairs_out[at] = v; };
        if constexpr (ONE) {
#pragma unroll
            for (int r = 0; r < R; ++r) place_64(count[wave], held[r], begin + r * kWave + lane < end, shift, bits, put);
        } else {
            place_items(count[wave], begin, end, shift, bits, item_of, put);
        }
    }
}

// A wave: 64 vectors of columns of the K rows of a chunk.  Lane l knows the pair l behind the
// chunk's begin, K of this chunk and K of the next, so that all decisions are the wave's.  An id
// is finished by the chunk in which it begins if it ends before the next one does; else it is
// long, and each chunk leaves its part of it.  part: [chunks][2][vecs VE], of the long id that
// reaches in from the chunk before (0) and of the one that begins here (1).
template <int DT, bool SHORT, int K>
__global__ __launch_bounds__(kThreads) void embedding_sum_kernel(const EmbeddingArgs a, const uint2 *pairs, float *part,
                                                                 int vecs, uint32_t chunks) {
    constexpr int VE = kVec<DT>, es = Columns<DT, SHORT>::es, U = kRows;
    static_assert(2 * K <= kWave && K % U == 0, "");
    const uint32_t V = static_cast<uint32_t>(a.V), n = static_cast<uint32_t>(a.n);
    const uint32_t chunk = blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (chunk >= chunks) return;
    const uint32_t begin = chunk * K;
    const int lane = threadIdx.x % kWave, vec = blockIdx.y * kWave + lane;
    const uint32_t place = begin + lane;
    const uint2 none = {~0u, 0};
    uint2 pair = place < n ? pairs[place] : none;
    const uint32_t prior = begin > 0 ? pairs[begin - 1].x : ~0u, older = begin >= 2 * K ? pairs[begin - K - 1].x : ~0u;
    const uint32_t first = __builtin_amdgcn_readfirstlane(pair.x);
    if (first >= V) return;
    // where ids begin
    uint32_t before = __shfl_up(pair.x, 1, kWave);
    if (lane == 0) before = prior;
    constexpr uint64_t kHere = (1ull << K) - 1, kWindow = K == 32 ? ~0ull : (1ull << (2 * K)) - 1;
    const uint64_t starts = __ballot(pair.x != before) & kWindow, own = starts & kHere;
    // the id that reaches in: long if it fills this chunk or the one before
    const bool reaches_in = !(starts & 1), lead = reaches_in && (own == 0 || older == first);
    int from = 0, to = K;
    bool tail = false;  // the last one that begins here is long
    if (own) {
        if (reaches_in && !lead) from = __builtin_ctzll(own);
        const uint64_t later = starts & ~kHere;
        tail = later == 0;
        if (!tail) to = __builtin_ctzll(later);
    } else if (!lead) {
        return;
    }
    const int last_start = own ? 63 - __builtin_clzll(own) : -1;
    to = min(to, static_cast<int>(__popcll(__ballot(pair.x < V))));  // (those without a gradient come last)
    if (from >= to) return;
    const bool in_row = vec < vecs;
    const Columns<DT, SHORT> at(in_row ? vec : vecs - 1, a.C);
    const char *dy = static_cast<const char *>(a.dy) + at.offset;
    const int64_t pitch = a.ldy * es;
    float acc[VE] = {};
    u32x4 v[2][U];
    auto fetch = [&](u32x4 (&w)[U], int r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int q = r + u < to ? r + u : to - 1;
            const uint32_t row = __builtin_amdgcn_readlane(pair.y, q);
            const char *p = dy + row * pitch;
            if constexpr (SHORT) w[u] = at.load(p);
            else w[u] = reinterpret_cast<const Raw *>(p)->v;
        }
    };
    auto add = [&](const u32x4 (&w)[U], int r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int q = r + u;
            if (q >= to) break;
            float x[VE];
            widen<DT>(w[u], x);
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] += x[j];
            if (q + 1 < to && !(starts >> (q + 1) & 1)) continue;
            // the last row of an id, or of its part
            const uint32_t id = __builtin_amdgcn_readlane(pair.x, q);
            const bool head = lead && (own == 0 || q < __builtin_ctzll(own));
            if (in_row && id < V) {
                if (head || (tail && q >= last_start)) {
                    float *p = part + ((static_cast<int64_t>(chunk) * 2 + (head ? 0 : 1)) * vecs + vec) * VE;
#pragma unroll
                    for (int j = 0; j < VE; ++j) p[j] = acc[j];
                } else {
#pragma unroll
                    for (int j = 0; j < VE; ++j) acc[j] *= a.scale;
                    at.store(static_cast<char *>(a.dweight) + static_cast<int64_t>(id) * a.C * es, narrow<DT>(acc));
                }
            }
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] = 0.f;
        }
    };
    fetch(v[0], from);
    for (int r = from; r < to; r += 2 * U) {
        if (r + U < to) fetch(v[1], r + U);
        add(v[0], r);
        if (r + 2 * U < to) fetch(v[0], r + 2 * U);
        if (r + U < to) add(v[1], r + U);
    }
}

// The long ids' parts: workgroup b looks for them at the chunks b, b + gridDim.x, ..; of an id's
// parts wave w has the w-th, (w + 16)-th .., of four columns a lane, then the waves' sums.
template <int DT, int K>
__global__ __launch_bounds__(kSortThreads) void embedding_join_kernel(const EmbeddingArgs a, const uint2 *pairs,
                                                                      const float *part, int vecs, uint32_t chunks) {
    constexpr int VE = kVec<DT>;
    __shared__ f32x4 sums[kSortWaves][kWave];
    __shared__ uint32_t found[kSortThreads], reach[kSortWaves];
    __shared__ int list;
    const uint32_t n = static_cast<uint32_t>(a.n);
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int slot = (blockIdx.y * kWave + lane) * 4, width = vecs * VE;  // columns as the parts have them
    for (uint64_t c0 = blockIdx.x; c0 < chunks; c0 += static_cast<uint64_t>(gridDim.x) * kSortThreads) {
        if (threadIdx.x == 0) list = 0;
        __syncthreads();
        const uint64_t c = c0 + static_cast<uint64_t>(threadIdx.x) * gridDim.x, begin = c * K;
        if (begin + 2 * K <= n) {
            const uint32_t id = pairs[begin + K - 1].x;
            if (id < static_cast<uint32_t>(a.V) && pairs[begin + 2 * K - 1].x == id && !(begin > 0 && pairs[begin - 1].x == id))
                found[atomicAdd(&list, 1)] = static_cast<uint32_t>(c);
        }
        __syncthreads();
        for (int f = 0; f < list; ++f) {
            const uint32_t chunk = found[f], id = pairs[static_cast<uint64_t>(chunk) * K + K - 1].x;
            // the chunks behind that begin with the id are the first ones
            uint32_t count = 0;
            for (;;) {
                const uint64_t at = (static_cast<uint64_t>(chunk) + 1 + count + threadIdx.x) * K;
                const uint32_t here = __popcll(__ballot(at < n && pairs[at].x == id));
                if (lane == 0) reach[wave] = here;
                __syncthreads();
                uint32_t all = 0;
                for (int w = 0; w < kSortWaves; ++w) all += reach[w];
                __syncthreads();
                count += all;
                if (all < kSortThreads) break;
            }
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            if (slot < width) {
                // part 0 is this chunk's, part c > 0 that of the c-th chunk behind
                constexpr int U = 8;
                for (uint32_t q = wave; q <= count; q += U * kSortWaves) {
                    f32x4 x[U];  // all loads first
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const uint32_t c = min(q + u * kSortWaves, count);
                        x[u] = *reinterpret_cast<const f32x4 *>(part + (static_cast<int64_t>(chunk + c) * 2 + (c == 0)) * width + slot);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (q + u * kSortWaves <= count) acc += x[u];
                }
            }
            sums[wave][lane] = acc;
            __syncthreads();
            if (wave == 0 && slot < width) {
                for (int w = 1; w < kSortWaves; ++w) acc += sums[w][lane];
                const int vec = slot / VE, first = a.C < VE ? 0 : vec * VE + VE <= a.C ? vec * VE : a.C - VE, col = first + slot % VE;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < a.C) store_elem(a.dweight, static_cast<int64_t>(id) * a.C + col + j, DT, acc[j] * a.scale);
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

namespace {

struct Plan {
    bool grouped;        // in one launch
    int passes, bits;    // of the sort, or of a group
    int blocks, items;   // of the sort
    int chunk;           // rows
    int64_t chunks;
    size_t pairs_bytes, hist_bytes, part_bytes;
};
Plan plan(int64_t n, int64_t V, int C) {
    Plan p{};
    p.grouped = n <= kGroupTokens;
    int bits = 0;  // of the ids; of the sort's keys 0 .. V
    while (bits < 32 && (static_cast<int64_t>(1) << bits) < V + !p.grouped) ++bits;
    if (p.grouped) bits = bits > __builtin_ctz(kGroups) ? bits - __builtin_ctz(kGroups) : 0;
    p.passes = (bits + kMaxBits - 1) / kMaxBits;
    p.bits = p.passes ? (bits + p.passes - 1) / p.passes : 0;
    const int64_t per = (n + kSortBlocks - 1) / kSortBlocks;
    const int64_t items = per < kSortItems ? kSortItems : (per + kSortThreads - 1) / kSortThreads * kSortThreads;
    p.items = static_cast<int>(items);
    p.blocks = static_cast<int>((n + items - 1) / items);
    p.chunk = n < kFewRows ? 8 : 32;
    p.chunks = (n + p.chunk - 1) / p.chunk;
    auto round = [](size_t b) { return (b + 255) / 256 * 256; };
    p.pairs_bytes = round(static_cast<size_t>(n) * 8);
    p.hist_bytes = p.grouped ? 0 : round(static_cast<size_t>(p.blocks) * (size_t{1} << p.bits) * 4);
    p.part_bytes = static_cast<size_t>(p.chunks) * 2 * ((static_cast<size_t>(C) + 7) / 8 * 8) * 4;
    return p;
}

template <int DT>
void run(const EmbeddingArgs &a, hipStream_t s) {
    const int vecs = (a.C + kVec<DT> - 1) / kVec<DT>;
    const int64_t most = (int64_t{1} << 30) / vecs;  // rows of a launch
    const bool scales = a.scale != 1.f, is_short = a.C < kVec<DT>;
    const auto kernel = is_short ? (scales ? embedding_kernel<DT, true, true> : embedding_kernel<DT, false, true>)
                                 : (scales ? embedding_kernel<DT, true, false> : embedding_kernel<DT, false, false>);
    for (int64_t first = 0; first < a.n; first += most) {
        const int rows = static_cast<int>(a.n - first < most ? a.n - first : most);
        const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(rows) * vecs + kThreads - 1) / kThreads));
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a, first, rows, vecs);
    }
}

template <int DT, int K>
void sum_and_join(const EmbeddingArgs &a, const Plan &p, const uint2 *pairs, float *part, hipStream_t s) {
    const int vecs = (a.C + kVec<DT> - 1) / kVec<DT>, slabs = (vecs + kWave - 1) / kWave;
    const uint32_t chunks = static_cast<uint32_t>(p.chunks);
    const dim3 grid((chunks + kThreads / kWave - 1) / (kThreads / kWave), slabs);
    const auto kernel = a.C < kVec<DT> ? embedding_sum_kernel<DT, true, K> : embedding_sum_kernel<DT, false, K>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a, pairs, part, vecs, chunks);
    if (a.n < 2 * K) return;  // (no long id)
    const dim3 join(chunks < 256 ? chunks : 256, (vecs * kVec<DT> + 4 * kWave - 1) / (4 * kWave));
    hipLaunchKernelGGL((embedding_join_kernel<DT, K>), join, dim3(kSortThreads), 0, s, a, pairs, part, vecs, chunks);
}

using SortKernel = void (*)(EmbeddingArgs, const uint2 *, uint2 *, uint32_t *, int, int, int, Fill);
SortKernel sort_kernel(bool first, bool scatter, bool one) {
    if (one) {
        if (first) return scatter ? embedding_sort_kernel<true, true, true> : embedding_sort_kernel<true, false, true>;
        return scatter ? embedding_sort_kernel<false, true, true> : embedding_sort_kernel<false, false, true>;
    }
    if (first) return scatter ? embedding_sort_kernel<true, true, false> : embedding_sort_kernel<true, false, false>;
    return scatter ? embedding_sort_kernel<false, true, false> : embedding_sort_kernel<false, false, false>;
}

template <int DT>
void run_backward(const EmbeddingArgs &a, hipStream_t s) {
    const Plan p = plan(a.n, a.V, a.C);
    char *w = static_cast<char *>(a.workspace);
    uint2 *buf[2] = {reinterpret_cast<uint2 *>(w), reinterpret_cast<uint2 *>(w + p.pairs_bytes)};
    uint32_t *hist = reinterpret_cast<uint32_t *>(w + 2 * p.pairs_bytes);
    float *part = reinterpret_cast<float *>(w + 2 * p.pairs_bytes + p.hist_bytes);
    const dim3 threads(kSortThreads);
    // the launches, each with its share of the zeros
    const int launches = p.grouped ? 1 : 2 * p.passes;
    const int64_t zeros = a.V * a.C * (DT == PRIME_F32 ? 4 : 2) / 16 + 1, share = (zeros + launches - 1) / launches;
    int launch = 0;
    auto next = [&](int blocks, Fill &f) {
        f.block = blocks;
        f.from = share * launch++;
        f.to = f.from + share;
        constexpr int per = kSortThreads * 4;
        return dim3(static_cast<unsigned>(blocks + (share + per - 1) / per));
    };
    Fill f;
    const uint2 *pairs = buf[0];
    if (p.grouped) {
        const dim3 grid = next(kGroups + 1, f);
        hipLaunchKernelGGL(embedding_group_kernel, grid, threads, 0, s, a, buf[0], buf[1], p.passes, p.bits, f);
    } else {
        for (int i = 0; i < p.passes; ++i) {
            uint2 *to = buf[i & 1];
            for (int scatter = 0; scatter < 2; ++scatter) {
                const dim3 grid = next(p.blocks, f);
                hipLaunchKernelGGL(sort_kernel(i == 0, scatter, p.items == kSortItems), grid, threads, 0, s, a, pairs, to, hist, i * p.bits, p.bits, p.items, f);
            }
            pairs = to;
        }
    }
    if (p.chunk == 8) sum_and_join<DT, 8>(a, p, pairs, part, s);
    else sum_and_join<DT, 32>(a, p, pairs, part, s);
}

}  // namespace

size_t embedding_workspace_bytes(int64_t n, int64_t V, int C) {
    const Plan p = plan(n, V, C);
    return 2 * p.pairs_bytes + p.hist_bytes + p.part_bytes;
}

bool embedding_grid_fits(int64_t n, int64_t V, int C, int dt) {
    const Plan p = plan(n, V, C);
    const int64_t vecs = (C + (dt == PRIME_F32 ? 3 : 7)) / (dt == PRIME_F32 ? 4 : 8), limit = (int64_t{1} << 32) - kSortThreads;
    const int64_t fill = V * C * (dt == PRIME_F32 ? 4 : 2) / 64 + kSortThreads;  // threads, of one launch at most
    return (p.chunks + 3) * ((vecs + kWave - 1) / kWave) * kWave < limit && fill + (p.blocks + kGroups + 1) * kSortThreads < limit;
}

hipError_t launch_embedding(const EmbeddingArgs &a, bool backward, hipStream_t stream) {
    if (a.dt == PRIME_BF16) backward ? run_backward<PRIME_BF16>(a, stream) : run<PRIME_BF16>(a, stream);
    else if (a.dt == PRIME_F16) backward ? run_backward<PRIME_F16>(a, stream) : run<PRIME_F16>(a, stream);
    else backward ? run_backward<PRIME_F32>(a, stream) : run<PRIME_F32>(a, stream);
    return hipGetLastError();
}

}  // namespace prime
