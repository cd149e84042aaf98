// Embedding lookup y_i = scale W[id_i], and its gradient dW[v] = scale sum_{i: id_i = v} dy_i.
//
// The gradient takes the tokens of one id side by side, in their order, and sums over these rows
// (those of many tokens by parts) in fp32, each row of dy read once: no atomics on floats, so the
// order of every sum is fixed.
//   order   pairs (id, token) such that equal ids lie together, a token without a gradient
//           (padding, an id outside the table) with the id V and behind all others; and which
//           ids occur.  Made by the lookup, for which it is all but free: its few workgroups
//           wait for memory while those that look up fill its bandwidth.  Up to kGroupTokens
//           tokens in one launch, else by counting passes
//   sum     a wave has 64 vectors of columns of a chunk of pairs.  An id whose rows end before
//           the next chunk does is finished where it begins; a longer one leaves a part in
//           each chunk.  Further workgroups write the zeros of the ids that do not occur
//   join    the parts of the long ones, in a fixed order
//
// All three are bound by memory.  65536 tokens x 768 bf16 of a table of 50304, ids of a language's
// frequencies (us on the device): the lookup alone 23-25 (100 MB written, the table's rows in
// the caches: 4.1 TB/s of writes); with the order, four launches of 10-12, 44; the sums 36.8
// (100 MB of dy read, 77 MB of gradient written: 4.8 TB/s, a copy's rate); the join 7.4.  2331 x
// 501 fp32 of 10000: 8.7, 15 and 4.  One token's lookup takes 1.8.

#include <type_traits>

#include "prime_kernels.h"
#include "row_vec.h"

namespace prime {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
// (128 groups and the one behind them, each reading all ids, are half of the workgroups that fit.
// A group of 2048 pairs, twice, and its counts are 66 KB of LDS)
constexpr int kGroups = 128;           // by the ids' low bits
constexpr int kGroupList = 2048;       // tokens of a group that are sorted in LDS
// Ranked / sorted in two passes, us: 2331 tokens 7.6 / 9.7, 8000 10.2 / 10.9; 16000 of ranked ids 18.8 / 17.0.
constexpr int kGroupRanked = 256;      // .. that are ranked by comparing each with each
// One launch against two passes of two launches (us, with the lookup of 768 bf16): 16000 tokens of
// ranked ids 18.7 / 30, of one id, which one workgroup then has, 40 / 34; 32000 tokens 25 / 35
// and 74 / 40; 65536 of one id 136.
constexpr int kGroupTokens = 1 << 14;
constexpr int kSortItems = 4096;       // at least, of a workgroup
constexpr int kSortBlocks = 512;       // at most
// Two chunks are one pair a lane.  Chunks of 8 pairs at 12000 tokens: sums and join 20.9 us for 24
// with ranked ids, 44 for 23 with one id.
constexpr int kChunk = 32;             // pairs
constexpr int kRows = 8;               // of a chunk, on their way at once, twice (4: 35.4 us for 36.5; 16: 46 for 43)
constexpr int kZeroRows = 64;          // of the table, that a workgroup writes where their ids do not occur

// A launch's share of the lookup: rows [first, first + rows) by the workgroups from `block` on,
// `vecs` vectors of 16 bytes each.
struct Share {
    int block;
    int64_t first;
    int rows, vecs;
};

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

// 16 bytes a thread of a row of the output; the last vector of a row ends with it, and where the
// row is no multiple of 16 bytes shares some with the one before.  Without a scale bytes are
// copied, whatever their type.
__device__ __forceinline__ void look_up(const EmbeddingArgs &a, const Share &share, uint32_t item) {
    const uint32_t r = item / static_cast<uint32_t>(share.vecs);
    if (r >= static_cast<uint32_t>(share.rows)) return;
    const int es = a.dt == PRIME_F32 ? 4 : 2, bytes = a.C * es, at = min(static_cast<int>(item - r * share.vecs) * 16, bytes - 16);
    const int64_t i = share.first + r, id = load_id(a, i);
    const bool inside = id >= 0 && id < a.V;
    const char *from = static_cast<const char *>(a.weight) + (inside ? id : 0) * a.ldw * es;
    char *to = static_cast<char *>(a.out) + i * bytes;
    if (at < 0) {  // a row shorter than a vector
        for (int j = 0; j < a.C; ++j) store_elem(to, j, a.dt, inside ? load_elem(from, j, a.dt) * a.scale : 0.f);
        return;
    }
    u32x4 v = {0, 0, 0, 0};
    if (inside) v = reinterpret_cast<const Raw *>(from + at)->v;
    auto scaled = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        float x[kVec<DT>];
        widen<DT>(v, x);
#pragma unroll
        for (int j = 0; j < kVec<DT>; ++j) x[j] *= a.scale;
        v = narrow<DT>(x);
    };
    if (a.scale != 1.f && inside) {
        if (a.dt == PRIME_BF16) scaled(std::integral_constant<int, PRIME_BF16>{});
        else if (a.dt == PRIME_F16) scaled(std::integral_constant<int, PRIME_F16>{});
        else scaled(std::integral_constant<int, PRIME_F32>{});
    }
    reinterpret_cast<Raw *>(to + at)->v = v;
}
// by the workgroups of a launch that makes the order
__device__ __forceinline__ void look_up(const EmbeddingArgs &a, const Share &share) {
    look_up(a, share, (blockIdx.x - share.block) * kSortThreads + threadIdx.x);
}

__global__ __launch_bounds__(kThreads) void embedding_kernel(const EmbeddingArgs a, const Share share) {
    look_up(a, share, blockIdx.x * kThreads + threadIdx.x);
}

// Where it is kept whether an id occurs: a group's ids lie together.
__device__ __forceinline__ int64_t occurs_at(int64_t id, int64_t V) {
    return id % kGroups * ((V + kGroups - 1) / kGroups) + id / kGroups;
}

// The sum of v over the threads before this one.
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t *wave_total) {  // a value a wave
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

// Bound by latency: three reads of the ids, which the caches hold, and a sort in LDS: 8.7 us at 2331
// tokens, the lookup among them.
// Workgroup g < kGroups: the tokens whose ids have the low bits g, in the order of the others.
// Each reads all ids, so where its tokens go it knows by itself: behind those of lower groups.
// Workgroup kGroups: the places behind all of them, for tokens without a gradient.  The
// others look up.
__global__ __launch_bounds__(kSortThreads) void embedding_group_kernel(const EmbeddingArgs a, uint2 *pairs, uint2 *other,
                                                                       uint8_t *occurs, int passes, int bits, const Share share) {
    constexpr int kLow = __builtin_ctz(kGroups);
    __shared__ uint32_t tally[kSortWaves][kMaxBins];
    __shared__ uint32_t wave_total[kSortWaves], wave_lower[kSortWaves];
    __shared__ uint2 list[2][kGroupList];
    if (static_cast<int>(blockIdx.x) >= share.block) {
        look_up(a, share);
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
    const int64_t ids = (a.V + kGroups - 1) / kGroups;  // of a group
    if (group < kGroups)
        for (int64_t i = tid; i < ids; i += kSortThreads) occurs[group * ids + i] = 0;
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
        if (in) {
            first[at + __popcll(all & ((1ull << lane) - 1))] = uint2{id, static_cast<uint32_t>(i)};
            occurs[group * ids + (id >> kLow)] = 1;
        }
        at += __popcll(all);
    });
    __syncthreads();
    if (passes && count <= kGroupRanked) {  // each by its rank among the others
        if (tid < static_cast<int>(count)) {
            const uint2 item = list[0][tid];
            uint32_t rank = 0;
#pragma unroll 8
            for (uint32_t o = 0; o < count; ++o) {
                const uint32_t id = list[0][o].x;
                rank += (id < item.x) | ((id == item.x) & (o < static_cast<uint32_t>(tid)));
            }
            pairs[base + rank] = item;
        }
        return;
    }
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
// kSortItems tokens, which its threads hold.  Workgroups from `share.block` on look up.  The
// first launch clears `occurs`, the second sets it.  At 65536 tokens the 16 workgroups that sort
// take 5-8 us of the 10-12 of a launch, which the lookup's share fills (all shares being equal;
// 1 : 2 or 2 : 3 for counting and placing is within a microsecond of that).
template <bool FIRST, bool SCATTER, bool ONE>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(const EmbeddingArgs a, const uint2 *pairs,
                                                                      uint2 *pairs_out, uint8_t *occurs,
                                                                      uint32_t *hist, int shift, int bits, int items,
                                                                      const Share share) {
    constexpr int R = kSortItems / kSortThreads;
    __shared__ uint32_t count[kSortWaves][kMaxBins];
    __shared__ uint32_t total[kSortThreads], before[kSortThreads], wave_total[kSortWaves];
    if constexpr (FIRST && !SCATTER) {
        const int64_t ids = (a.V + kGroups - 1) / kGroups * kGroups, step = static_cast<int64_t>(gridDim.x) * kSortThreads;
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * kSortThreads + threadIdx.x; i < ids; i += step) occurs[i] = 0;
    }
    if (static_cast<int>(blockIdx.x) >= share.block) {
        look_up(a, share);
        return;
    }
    const int bins = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, blocks = share.block;
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
        const int bin = tid & (bins - 1), parts = kSortThreads / bins;
        uint32_t t = 0, b = 0;
        for (int q = tid / bins; q < blocks; q += U * parts) {
            uint32_t h[U];
#pragma unroll
            for (int u = 0; u < U; ++u) h[u] = hist[static_cast<int64_t>(min(q + u * parts, blocks - 1)) * bins + bin];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                t += q + u * parts < blocks ? h[u] : 0;
                b += q + u * parts < static_cast<int>(blockIdx.x) ? h[u] : 0;
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
        auto put = [&](uint32_t at, uint2 v) {
            pairs_out[at] = v;
            if (FIRST && v.x < static_cast<uint32_t>(a.V)) occurs[occurs_at(v.x, a.V)] = 1;
        };
        if constexpr (ONE) {
#pragma unroll
            for (int r = 0; r < R; ++r) place_64(count[wave], held[r], begin + r * kWave + lane < end, shift, bits, put);
        } else {
            place_items(count[wave], begin, end, shift, bits, item_of, put);
        }
    }
}

// The ids that reach over a chunk and the next: a section of kThreads chunks has its count, and
// for each the chunk in which it begins, how many chunks behind it it reaches, and the id.
struct LongIds {
    uint32_t *count;  // [sections]
    uint4 *list;      // [sections][kThreads]
};

__device__ __forceinline__ void list_long(const EmbeddingArgs &a, const uint2 *pairs, const LongIds &longs, uint32_t chunks) {
    __shared__ uint32_t listed;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    constexpr int K = kChunk;
    const uint32_t n = static_cast<uint32_t>(a.n), chunk = blockIdx.x * kThreads + threadIdx.x;
    const uint64_t begin = static_cast<uint64_t>(chunk) * K;
    if (begin + 2 * K <= n) {
        const uint32_t id = pairs[begin + K - 1].x, ahead = pairs[begin + 2 * K - 1].x, prior = begin > 0 ? pairs[begin - 1].x : ~id;
        if (id < static_cast<uint32_t>(a.V) && ahead == id && prior != id) {
            // the chunks behind that begin with the id are the first ones: by doubling, then halving
            uint32_t in = chunk + 1, step = 1;  // `in` begins with it
            while (in + step < chunks && pairs[static_cast<uint64_t>(in + step) * K].x == id) in += step, step *= 2;
            for (; step; step /= 2)
                if (in + step < chunks && pairs[static_cast<uint64_t>(in + step) * K].x == id) in += step;
            longs.list[blockIdx.x * kThreads + atomicAdd(&listed, 1u)] = uint4{chunk, in - chunk, id, 0};
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) longs.count[blockIdx.x] = listed;
}

// A wave: 64 vectors of columns of the rows of a chunk.  Lane l knows the pair l behind the
// chunk's begin, those of this chunk and of the next, so that all decisions are the wave's.  An id
// is finished by the chunk in which it begins if it ends before the next one does; else it is
// long, and each chunk leaves its part of it.  part: [chunks][2][vecs VE], of the long id that
// reaches in from the chunk before (0) and of the one that begins here (1).  The first list_blocks
// workgroups list the long ids, those from sum_blocks on write zeros for kZeroRows rows each,
// where their ids do not occur.  ONCE: dy is read past the caches.
// Reads are random rows of dy, each once, two batches of kRows rows of 1 KB on their way in a wave.
template <int DT, bool SHORT, bool ONCE>
__global__ __launch_bounds__(kThreads) void embedding_sum_kernel(const EmbeddingArgs a, const uint2 *pairs,
                                                                 const uint8_t *occurs, const LongIds longs, float *part,
                                                                 int vecs, uint32_t chunks, uint32_t list_blocks,
                                                                 uint32_t sum_blocks) {
    constexpr int VE = kVec<DT>, es = Columns<DT, SHORT>::es, U = kRows, K = kChunk;
    static_assert(2 * K == kWave && K % U == 0, "");
    const uint32_t V = static_cast<uint32_t>(a.V), n = static_cast<uint32_t>(a.n);
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (blockIdx.x < list_blocks) {
        list_long(a, pairs, longs, chunks);
        return;
    }
    if (blockIdx.x >= sum_blocks) {
        constexpr int kRowsOfWave = kZeroRows / (kThreads / kWave);
        const int64_t first = static_cast<int64_t>(blockIdx.x - sum_blocks) * kZeroRows + wave * kRowsOfWave, id = first + lane;
        uint64_t absent = __ballot(lane < kRowsOfWave && id < a.V && !occurs[id < a.V ? occurs_at(id, a.V) : 0]);
        for (; absent; absent &= absent - 1) {
            char *row = static_cast<char *>(a.dweight) + (first + __builtin_ctzll(absent)) * a.C * es;
            for (int q = lane; q < vecs; q += kWave) Columns<DT, SHORT>(q, a.C).store(row, u32x4{0, 0, 0, 0});
        }
        return;
    }
    const uint32_t groups = (chunks + kThreads / kWave - 1) / (kThreads / kWave), block = blockIdx.x - list_blocks, slab = block / groups;
    const uint32_t chunk = (block - slab * groups) * (kThreads / kWave) + wave;
    if (chunk >= chunks) return;
    const uint32_t begin = chunk * K;
    const int vec = slab * kWave + lane;
    const uint32_t place = begin + lane;
    const uint2 none = {~0u, 0};
    uint2 pair = place < n ? pairs[place] : none;
    const uint32_t prior = begin > 0 ? pairs[begin - 1].x : ~0u, older = begin >= 2 * K ? pairs[begin - K - 1].x : ~0u;
    const uint32_t first = __builtin_amdgcn_readfirstlane(pair.x);
    if (first >= V) return;
    // where ids begin
    uint32_t before = __shfl_up(pair.x, 1, kWave);
    if (lane == 0) before = prior;
    constexpr uint64_t kHere = (1ull << K) - 1;
    const uint64_t starts = __ballot(pair.x != before), own = starts & kHere;
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
            else if constexpr (ONCE) w[u] = __builtin_nontemporal_load(&reinterpret_cast<const Raw *>(p)->v);
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

// The long ids' parts: of all sections' ids workgroup b has the b-th, (b + gridDim.x)-th ..; of an
// id's parts the workgroup's r-th row of L lanes has the r-th, (r + rows)-th .., of four columns
// a lane, then the rows' sums.  One workgroup reads some 50 GB/s, so narrow slabs bring more of
// them to an id: 65536 tokens of one id x 768, 6 MB of parts, take 15 us.  The slabs of an id begin at
// different places of x, so on different XCDs (all at the same: 37).
template <int DT, int L>
__global__ __launch_bounds__(kThreads) void embedding_join_kernel(const EmbeddingArgs a, const LongIds longs,
                                                                  const float *part, int vecs, uint32_t sections) {
    constexpr int VE = kVec<DT>, kRowsOfLanes = kThreads / L;
    __shared__ f32x4 sums[kWaves][L];
    __shared__ uint32_t wave_total[kWaves];
    __shared__ uint4 found;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, col = threadIdx.x % L, row = threadIdx.x / L;
    const int slot = (blockIdx.y * L + col) * 4, width = vecs * VE;  // columns as the parts have them
    for (uint32_t s0 = 0; s0 < sections; s0 += kThreads) {
        const uint32_t section = s0 + threadIdx.x, own = section < sections ? longs.count[section] : 0;
        const uint32_t before = scan_before(own, wave_total);
        uint32_t total = 0;
        for (int w = 0; w < kWaves; ++w) total += wave_total[w];
        for (uint32_t e = (blockIdx.x + blockIdx.y) % gridDim.x; e < total; e += gridDim.x) {
            if (before <= e && e < before + own) found = longs.list[section * kThreads + e - before];
            __syncthreads();
            const uint4 entry = found;
            const uint32_t chunk = entry.x, reach = entry.y, id = entry.z;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            if (slot < width) {
                // part 0 is this chunk's, part c > 0 that of the c-th chunk behind
                constexpr int U = 8;
                for (uint32_t q = row; q <= reach; q += U * kRowsOfLanes) {
                    f32x4 x[U];  // all loads first
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const uint32_t c = min(q + u * kRowsOfLanes, reach);
                        x[u] = *reinterpret_cast<const f32x4 *>(part + (static_cast<int64_t>(chunk + c) * 2 + (c == 0)) * width + slot);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (q + u * kRowsOfLanes <= reach) acc += x[u];
                }
            }
            if constexpr (L == 16) {
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = sum_lane32(sum_lane16(acc[j]));
            }
            if (lane < L) sums[wave][lane] = acc;
            __syncthreads();
            if (threadIdx.x < L && slot < width) {
                for (int w = 1; w < kWaves; ++w) acc += sums[w][col];
                const int vec = slot / VE, first = a.C < VE ? 0 : vec * VE + VE <= a.C ? vec * VE : a.C - VE, at = first + slot % VE;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < a.C) store_elem(a.dweight, static_cast<int64_t>(id) * a.C + at + j, DT, acc[j] * a.scale);
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

namespace {

// The order of n tokens in a buffer of the caller's: the pairs, which ids occur, then what only
// the making needs.
struct Plan {
    bool grouped;        // in one launch
    int passes, bits;    // of the sort, or of a group
    int blocks, items;   // of the sort
    int64_t chunks;
    size_t occurs, other, hist, bytes;  // where they begin, and the end
};
Plan plan(int64_t n, int64_t V) {
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
    p.blocks = p.grouped ? kGroups + 1 : static_cast<int>((n + items - 1) / items);
    p.chunks = (n + kChunk - 1) / kChunk;
    auto round = [](size_t b) { return (b + 255) / 256 * 256; };
    p.occurs = round(static_cast<size_t>(n) * 8);
    p.other = p.occurs + round(static_cast<size_t>(V + kGroups - 1) / kGroups * kGroups);
    p.hist = p.other + round(static_cast<size_t>(n) * 8);
    p.bytes = p.hist + (p.grouped ? 0 : round(static_cast<size_t>(p.blocks) * (size_t{1} << p.bits) * 4));
    return p;
}

using SortKernel = void (*)(EmbeddingArgs, const uint2 *, uint2 *, uint8_t *, uint32_t *, int, int, int,
                            Share);
SortKernel sort_kernel(bool first, bool scatter, bool one) {
    if (one) {
        if (first) return scatter ? embedding_sort_kernel<true, true, true> : embedding_sort_kernel<true, false, true>;
        return scatter ? embedding_sort_kernel<false, true, true> : embedding_sort_kernel<false, false, true>;
    }
    if (first) return scatter ? embedding_sort_kernel<true, true, false> : embedding_sort_kernel<true, false, false>;
    return scatter ? embedding_sort_kernel<false, true, false> : embedding_sort_kernel<false, false, false>;
}

void run(const EmbeddingArgs &a, hipStream_t s) {
    const int es = a.dt == PRIME_F32 ? 4 : 2, vecs = (a.C * es + 15) / 16;
    const int64_t most = (int64_t{1} << 30) / vecs;  // rows of a launch
    Share share{0, 0, 0, vecs};
    if (!a.order) {
        for (; share.first < a.n; share.first += most) {
            share.rows = static_cast<int>(a.n - share.first < most ? a.n - share.first : most);
            const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(share.rows) * vecs + kThreads - 1) / kThreads));
            hipLaunchKernelGGL(embedding_kernel, grid, dim3(kThreads), 0, s, a, share);
        }
        return;
    }
    const Plan p = plan(a.n, a.V);
    char *w = static_cast<char *>(a.order);
    uint2 *buf[2] = {reinterpret_cast<uint2 *>(w), reinterpret_cast<uint2 *>(w + p.other)};
    uint8_t *occurs = reinterpret_cast<uint8_t *>(w + p.occurs);
    uint32_t *hist = reinterpret_cast<uint32_t *>(w + p.hist);
    const dim3 threads(kSortThreads);
    share.block = p.blocks;
    // the launches, each with its share of the rows
    const int launches = p.grouped ? 1 : 2 * p.passes;
    int64_t left = a.n;
    auto next = [&](int launch) {
        const int64_t fair = (left + launches - launch - 1) / (launches - launch);
        share.first = a.n - left;
        share.rows = static_cast<int>(fair < most ? fair : most);
        left -= share.rows;
        return dim3(static_cast<unsigned>(p.blocks + (static_cast<int64_t>(share.rows) * vecs + kSortThreads - 1) / kSortThreads));
    };
    if (p.grouped) {
        const dim3 grid = next(0);
        hipLaunchKernelGGL(embedding_group_kernel, grid, threads, 0, s, a, buf[0], buf[1], occurs, p.passes, p.bits, share);
    }
    const uint2 *pairs = nullptr;
    for (int i = 0; i < p.passes && !p.grouped; ++i) {
        uint2 *to = buf[(p.passes - 1 - i) & 1];
        for (int scatter = 0; scatter < 2; ++scatter) {
            const dim3 grid = next(2 * i + scatter);
            hipLaunchKernelGGL(sort_kernel(i == 0, scatter, p.items == kSortItems), grid, threads, 0, s, a, pairs, to, occurs, hist,
                               i * p.bits, p.bits, p.items, share);
        }
        pairs = to;
    }
    if (left) {  // more rows than the launches of the order take
        EmbeddingArgs rest = a;
        const int64_t done = a.n - left;
        rest.order = nullptr;
        rest.n = left;
        rest.ids = static_cast<const char *>(a.ids) + done * (a.ids64 ? 8 : 4);
        rest.out = static_cast<char *>(a.out) + done * a.C * es;
        run(rest, s);
    }
}

// The backward's workspace: the parts, the long ids.
struct Parts {
    size_t sections, counts, lists, bytes;
};
Parts parts(const Plan &p, int C) {
    Parts w{};
    w.sections = static_cast<size_t>(p.chunks + kThreads - 1) / kThreads;
    w.lists = static_cast<size_t>(p.chunks) * 2 * ((static_cast<size_t>(C) + 7) / 8 * 8) * 4;
    w.counts = w.lists + w.sections * kThreads * sizeof(uint4);
    w.bytes = w.counts + w.sections * 4;
    return w;
}

template <int DT>
void run_backward(const EmbeddingArgs &a, hipStream_t s) {
    const Plan p = plan(a.n, a.V);
    const int vecs = (a.C + kVec<DT> - 1) / kVec<DT>, slabs = (vecs + kWave - 1) / kWave;
    const bool joins = a.n >= 2 * kChunk;  // (else no id is long)
    const Parts space = parts(p, a.C);
    const uint32_t chunks = static_cast<uint32_t>(p.chunks), waves = kThreads / kWave, sections = static_cast<uint32_t>(space.sections);
    const uint32_t list_blocks = joins ? sections : 0, sum_blocks = list_blocks + (chunks + waves - 1) / waves * slabs;
    const uint32_t zero_blocks = static_cast<uint32_t>((a.V + kZeroRows - 1) / kZeroRows);
    const char *o = static_cast<const char *>(a.order);
    const uint2 *pairs = reinterpret_cast<const uint2 *>(o);
    const uint8_t *occurs = reinterpret_cast<const uint8_t *>(o + p.occurs);
    char *w = static_cast<char *>(a.workspace);
    float *part = reinterpret_cast<float *>(w);
    const LongIds longs{reinterpret_cast<uint32_t *>(w + space.counts), reinterpret_cast<uint4 *>(w + space.lists)};
    // a dy of 64 MB or more, twice what the L2 caches hold together: past them.  (Past / through them, x 768 bf16, us:
    // last touched long ago, 131072 tokens 55 / 75, 65536 36 / 40-43, 32768 27 / 22; just
    // written, 59 / 51, 39.6 / 37, 22.5 / 21.)
    const bool once = a.n * a.C * (DT == PRIME_F32 ? 4 : 2) >= int64_t{1} << 26;
    const auto kernel = a.C < kVec<DT> ? embedding_sum_kernel<DT, true, false> : once ? embedding_sum_kernel<DT, false, true> : embedding_sum_kernel<DT, false, false>;
    hipLaunchKernelGGL(kernel, dim3(sum_blocks + zero_blocks), dim3(kThreads), 0, s, a, pairs, occurs, longs, part, vecs, chunks,
                       list_blocks, sum_blocks);
    if (!joins) return;
    // some 1500 workgroups, an id's columns over y of them: slabs of 64 columns, or of 256 for wide rows
    // (64 / 256, us: 65536 tokens of one id x 1024 15 / 46, x 2048 19 / 54; 16384 x 4096 of ranked ids
    // 6.7 / 5.2, of one 6.6 / 14.4; x 8192 11.5 / 6.7 and 19 / 16.6)
    const uint32_t width = vecs * kVec<DT>, cols = width <= 4096 ? 64 : 256, y = (width + cols - 1) / cols;
    const uint32_t x = y < 6 ? 256 : y < 96 ? 1536 / y : 16;
    const auto join = cols == 64 ? embedding_join_kernel<DT, 16> : embedding_join_kernel<DT, 64>;
    hipLaunchKernelGGL(join, dim3(x, y), dim3(kThreads), 0, s, a, longs, part, vecs, sections);
}

}  // namespace

size_t embedding_order_bytes(int64_t n, int64_t V) { return plan(n, V).bytes; }

size_t embedding_workspace_bytes(int64_t n, int C) { return parts(plan(n, 1), C).bytes; }

// (threads of a launch are below 2^32)
bool embedding_grid_fits(int64_t n, int64_t V, int C, int dt) {
    const int64_t vecs = (C + (dt == PRIME_F32 ? 3 : 7)) / (dt == PRIME_F32 ? 4 : 8), slabs = (vecs + kWave - 1) / kWave;
    const int64_t chunks = plan(n, V).chunks, limit = (int64_t{1} << 32) - kSortThreads;
    const int64_t sum = (chunks + 3) * slabs * kWave + ((V + kZeroRows - 1) / kZeroRows + 2 + chunks / kThreads) * kThreads;
    return sum < limit;
}

hipError_t launch_embedding(const EmbeddingArgs &a, bool backward, hipStream_t stream) {
    if (!backward) run(a, stream);
    else if (a.dt == PRIME_BF16) run_backward<PRIME_BF16>(a, stream);
    else if (a.dt == PRIME_F16) run_backward<PRIME_F16>(a, stream);
    else run_backward<PRIME_F32>(a, stream);
    return hipGetLastError();
}

}  // namespace prime
