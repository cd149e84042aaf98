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
// One workgroup a row, a contiguous part a wave.  The first pass finds the largest logit and
// puts the row into LDS where it fits (else the later ones read the caches).  The ranking is
// never sorted: tokens are counted in cells of equal width in the logit (count_cells), and the
// counts tell in which cell top-k ends, and between which cells top_p ends.  Where no more
// tokens are left than the workgroup has threads, they are gathered in the order of their
// indices, one a thread, and compared only within the cell or bucket in which a cut falls
// (equal tokens that top-k cuts away past that number are found by their indices before).
// Where more are left, the masses of all are summed once, those near top_p's border in
// separate parts (cut_once).  What either cannot decide (a border in a cell of more than kList
// tokens) is left to buckets of masses and, at the last, a radix descent over the tokens'
// order-preserving keys (cut).
//
// What bounds it.  A row belongs to one CU, whose fp64 rate is the floor of a pass over masses
// (21 instructions a token, 4.9 cycles each: 50304 tokens 9 us); the rest is fetching code that
// runs once and barriers.  One row of 50304 bf16: 19 us without cuts, 17 with top_k 50, 13 with
// min_p 0.1, 34 with top_p 0.9 where the tokens down to its border can be gathered, else 38 (of
// these: 4 to load, 7 for counts and bounds, 14 for the masses, 7 for the border, 6 for the token).
// 256 rows, one a CU, take what the slowest takes: 45 us with every kind of cut, 22 with min_p 0.1.
// 512 x 50304 fp32 without cuts: 103 MB, 20 us to read, but the row comes in nearly twice: 44 us.

#include <type_traits>

#include "prime_kernels.h"
#include "row_vec.h"

namespace prime {

constexpr uint64_t kMass = 1ull << 42;  // the largest token's
constexpr int kBuckets = 2048, kList = 1024;
constexpr int kCells = 2 * kBuckets;     // half buckets, for counts
constexpr float kBucketSpan = 30.5f;  // a token this many T below the largest has mass 0
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
    double least;     // log2 of min_p; below every exponent without
    float per_half;   // buckets per half a unit of the logit
    float step;       // log2 of the weight from one cell to the next

    __device__ __forceinline__ double exponent(float x) const {  // of 2, at most 0
        return (static_cast<double>(x) - static_cast<double>(top)) * rate;
    }
    // 2^t as a mass, t <= 0: 2^f on |f| <= 1/2 by its Chebyshev interpolant of degree 9
    // (1.4e-14 off), scaled and rounded to a whole number by one addition to 2^52.  Below
    // 2^-44 (and for NaN, of a NaN or of -infinity times a rate of 0) that is 0.
    static constexpr uint64_t kBits = 0x4330000000000000ull;  // of 2^52
    __device__ static __forceinline__ uint64_t mass_of(double t) {
        uint64_t w = mass_bits(t) - kBits;
        asm("" : "+v"(w));  // computed for every token: a branch around it costs more than it saves
        return w;
    }
    __device__ static __forceinline__ uint64_t mass_bits(double t) {  // the mass and kBits
        constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: adding it rounds to a whole number
        t = fmax(t, -44.0);
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
        return __builtin_bit_cast(uint64_t, fma(p, scale, 4503599627370496.0));
    }
    __device__ __forceinline__ uint64_t mass(float x) const { return mass_of(exponent(x)); }
    __device__ static __forceinline__ uint64_t select(bool keep, uint64_t w) { return keep ? w : 0; }
    // bucket of x, false for tokens whose mass is 0 (and for NaN); monotone: every step is
    __device__ __forceinline__ float place(float x) const {
#pragma clang fp contract(off)  // the same number wherever it is asked for
        return fmaf(-0.5f, x, 0.5f * top) * per_half;
    }
    // cell of x, as bucket()
    __device__ __forceinline__ bool cell(float x, int &c) const {
        const float f = place(x) * 2.f;
        c = static_cast<int>(f);
        return f < static_cast<float>(kCells - 2);
    }
    __device__ __forceinline__ bool bucket(float x, int &b) const {
        const float f = place(x);
        b = static_cast<int>(f);
        return f < static_cast<float>(kBuckets - 1);
    }
};

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int lane) {
    return static_cast<uint64_t>(__shfl(static_cast<uint32_t>(v >> 32), lane, kWave)) << 32 |
           __shfl(static_cast<uint32_t>(v), lane, kWave);
}
// v of one lane, the same for all
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
    return static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane)) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ uint64_t last_lane(uint64_t v) { return lane_u64(v, kWave - 1); }
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
    uint64_t sum, rest;
    float last;
    int bucket, n, index, owner, low, high, found;
    uint8_t list_wave[kList];
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

// A row: wave w has the chunks [w per, (w + 1) per) of 64 lanes with VE elements each.  A
// chunk past the vocabulary's end becomes the last VE elements, those that an earlier chunk
// has as -infinity.  STAGED > 0: per is at most that, and after the first pass the row is in LDS.
template <int DT, int STAGED>
struct SampleRow {
    static constexpr int VE = DT == PRIME_F32 ? 4 : 8, es = DT == PRIME_F32 ? 4 : 2;
    const char *base;
    int vocab, per, start;  // start: the lane's first element
    int whole;              // the wave's chunks that lie before the vocabulary's end
    __device__ __forceinline__ void place(int wave, int lane) {
        whole = (vocab - wave * per * (kWave * VE)) / (kWave * VE);
        start = (wave * per * kWave + lane) * VE;
    }
    u32x4 *lds;             // the lane's place in the staged chunks, `lds_step` between two
    int lds_step;

    __device__ __forceinline__ int index(int i) const {
        const int e = start + i * (kWave * VE);
        return i < whole ? e : max(0, min(e, vocab - VE));
    }
    __device__ __forceinline__ u32x4 load(int i) const {
        if constexpr (STAGED > 0) {
            if (vocab < VE) {
                uint16_t h[8] = {};
                for (int k = 0; k < vocab * (es / 2); ++k) h[k] = reinterpret_cast<const uint16_t *>(base)[k];
                return __builtin_bit_cast(u32x4, h);
            }
        }
        return reinterpret_cast<const Raw *>(base + static_cast<int64_t>(index(i)) * es)->v;
    }
    __device__ __forceinline__ void mask(int i, u32x4 &v) const {
        constexpr uint32_t none = DT == PRIME_F32 ? 0xFF800000u : DT == PRIME_BF16 ? 0xFF80u : 0xFC00u;  // -infinity
        if (i < whole) return;
        const int e = start + i * (kWave * VE), first = index(i);
        if (first == e && first + VE <= vocab) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if (first + j >= e && first + j < vocab) continue;
            if constexpr (DT == PRIME_F32) v[j] = none;
            else v[j / 2] = j & 1 ? (v[j / 2] & 0xFFFFu) | none << 16 : (v[j / 2] & 0xFFFF0000u) | none;
        }
    }
    // chunk i as it was loaded or staged; what was loaded is masked after
    template <bool FIRST = false>
    __device__ __forceinline__ u32x4 get(int i) const {
        if constexpr (STAGED > 0 && !FIRST) return lds[i * lds_step];
        else return load(i);
    }
    template <bool FIRST = false>
    __device__ __forceinline__ void finish(int i, u32x4 &v) const {
        if constexpr (STAGED == 0 || FIRST) mask(i, v);
        if constexpr (STAGED > 0 && FIRST) lds[i * lds_step] = v;
    }
    __device__ __forceinline__ void fetch(int i, float (&x)[VE]) const {
        u32x4 v = get(i);
        finish(i, v);
        widen(v, x);
    }
    // element j of chunk i
    __device__ __forceinline__ float one(int i, int j) const {
        using P = typename std::conditional<DT == PRIME_F32, float, uint16_t>::type;
        const int e = start + i * (kWave * VE), at = index(i) + j;
        if (at < e || at >= vocab) return -kInf;
        P p;
        if constexpr (STAGED > 0) p = reinterpret_cast<const P *>(lds + i * lds_step)[j];
        else p = reinterpret_cast<const P *>(base)[at];
        if constexpr (DT == PRIME_F32) return p;
        else return DT == PRIME_BF16 ? bf16_bits_to_f32(p) : h16_bits_to_f32(p);
    }
    __device__ __forceinline__ void widen(const u32x4 &v, float (&x)[VE]) const {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if constexpr (DT == PRIME_F32) x[j] = __uint_as_float(v[j]);
            else if constexpr (DT == PRIME_BF16) x[j] = __uint_as_float(j & 1 ? v[j / 2] & 0xFFFF0000u : v[j / 2] << 16);
            else x[j] = h16_bits_to_f32(static_cast<uint16_t>(j & 1 ? v[j / 2] >> 16 : v[j / 2]));
        }
    }
    // f(i, x) over the lane's chunks, the next ones on their way.  (One copy of f: with a row
    // or two the time is in fetching instructions.)
    template <bool FIRST = false, bool BACK = false, typename F>
    __device__ __forceinline__ void each(F f) const {
        auto at = [&](int i) { return BACK ? per - 1 - i : i; };
        constexpr int D = STAGED == 0 ? 4 : !FIRST ? 2 : STAGED < 8 ? STAGED : 8;
        u32x4 next[D];
#pragma unroll
        for (int k = 0; k < D; ++k)
            if (k < per) next[k] = get<FIRST>(at(k));
#pragma unroll 1
        for (int i = 0; i < per; ++i) {
            u32x4 now = next[0];
#pragma unroll
            for (int k = 0; k + 1 < D; ++k) next[k] = next[k + 1];
            if (i + D < per) next[D - 1] = get<FIRST>(at(i + D));
            finish<FIRST>(at(i), now);
            float x[VE];
            widen(now, x);
            f(at(i), x);
        }
    }
};

// How many tokens are equal to `value`; `nth` of that count gives n, and the index of the
// n-th of them, from 1, is returned (any index where there are fewer).
template <int DT, int WAVES, int STAGED, typename F>
__device__ __forceinline__ int find_equal(SampleShared<WAVES> &sh, const SampleRow<DT, STAGED> &row, float value, F nth) {
    constexpr int VE = SampleRow<DT, STAGED>::VE;
    uint64_t count = 0, before, total;
    row.each([&](int, const float (&x)[VE]) {
#pragma unroll
        for (int j = 0; j < VE; ++j) count += x[j] == value;
    });
    block_scan(sh, count, before, total);
    const uint64_t n = nth(total);
    if (before < n && n <= before + sh.part[threadIdx.x / kWave]) {
        // this wave's chunks one after the other, lanes in order within one
        int left = static_cast<int>(n - before);
        row.each([&](int i, const float (&x)[VE]) {
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

// Thread t's sum over hist[t kPer ..], the sum before it, and the total.
template <int WAVES>
__device__ __forceinline__ uint64_t scan_hist(SampleShared<WAVES> &sh, uint64_t &mine, uint64_t &total) {
    constexpr int kPer = kBuckets / (WAVES * kWave);
    uint64_t waves;
    mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += sh.hist[threadIdx.x * kPer + i];
    return block_scan(sh, mine, waves, total);
}
// The bucket in which the sum reaches `want` (at most the total) into sh.bucket, the sum
// before it into sh.sum; `before`, `mine` as scan_hist gives them.
template <int WAVES>
__device__ __forceinline__ void locate(SampleShared<WAVES> &sh, uint64_t before, uint64_t mine, uint64_t want) {
    constexpr int kPer = kBuckets / (WAVES * kWave);
    if (before < want && want <= before + mine) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint64_t w = sh.hist[threadIdx.x * kPer + i];
            if (before < want && want <= before + w) sh.bucket = threadIdx.x * kPer + i, sh.sum = before;
            before += w;
        }
    }
    __syncthreads();
}
__device__ __forceinline__ void lds_add(uint64_t *p, uint64_t w) {
    atomicAdd(reinterpret_cast<unsigned long long *>(p), static_cast<unsigned long long>(w));
}

template <int N>
__device__ __forceinline__ float largest(const float (&x)[N]) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, x[j]);
    return m;
}

// The cut: over the tokens above `last` and `ties` tokens equal to it (none for -infinity),
// in rank order, the shortest prefix with weight of at least wanted(sum of all weights).
// WEIGH: masses, else ones.  Left as it is where all of them are needed.  whole: the tokens
// equal to the new `last` are known to be all kept.
template <bool WEIGH, int DT, int WAVES, int STAGED, typename F>
__device__ __forceinline__ void cut(SampleShared<WAVES> &sh, const SampleRow<DT, STAGED> &row, const RowScale &rs,
                                    float &last, uint64_t &ties, bool &whole, F wanted) {
    constexpr int kThreads = WAVES * kWave, VE = SampleRow<DT, STAGED>::VE;
    const int tid = threadIdx.x;
    const float floor = last;
    const uint64_t floor_w = ties ? ties * (WEIGH ? rs.mass(floor) : 1) : 0;
    uint64_t before, mine, total;
    __syncthreads();
    for (int b = tid; b < kBuckets; b += kThreads) sh.hist[b] = 0;
    if (tid == 0) sh.n = 0;
    __syncthreads();
    auto fill = [&](int, const float (&x)[VE]) {
        int b;
        const float most = largest(x);
        if (!(rs.bucket(most, b) & (most > floor))) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const bool in = rs.bucket(x[j], b) & (x[j] > floor);
            const uint64_t w = WEIGH ? RowScale::mass_of(rs.exponent(x[j])) : 1;
            if (in) lds_add(&sh.hist[b], w);
        }
    };
    row.each(fill);
    int floor_b = -1;
    if (floor_w && !rs.bucket(floor, floor_b)) floor_b = -1;
    if (tid == 0 && floor_b >= 0) lds_add(&sh.hist[floor_b], floor_w);
    __syncthreads();
    before = scan_hist(sh, mine, total);
    const uint64_t want = wanted(total);
    if (want > total) return;  // (the same for every thread)
    locate(sh, before, mine, want);
    const int bucket = sh.bucket;
    const uint64_t above = sh.sum;
    row.each([&](int, const float (&x)[VE]) {
        int b;
        if (!(rs.bucket(largest(x), b) & (b <= bucket))) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if (rs.bucket(x[j], b) & (b == bucket) & (x[j] > floor)) {
                const int n = atomicAdd(&sh.n, 1);
                if (n < kList) sh.list_x[n] = x[j];
            }
        }
    });
    __syncthreads();
    const int own = sh.n, n = own + (floor_b == bucket);  // the floor's tokens count as one more
    if (n <= kList) {
        for (int i = tid; i < own; i += kThreads) sh.list_w[i] = WEIGH ? rs.mass(sh.list_x[i]) : 1;
        if (tid == 0 && n > own) sh.list_x[own] = floor, sh.list_w[own] = floor_w;
        __syncthreads();
    }
    // `over`: the weight of the tokens above x; `equal`: of those equal to it, where known
    auto found = [&](float x, uint64_t over, uint64_t equal) { sh.last = x, sh.sum = over, sh.rest = equal; };
    if (n <= kList) {
        for (int i = tid; i < n; i += kThreads) {
            const float x = sh.list_x[i];
            uint64_t over = above, equal = 0;
#pragma unroll 8
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
            row.each([&](int, const float (&x)[VE]) {
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const uint32_t k = logit_key(x[j]);
                    if (x[j] > floor && inside(k)) lds_add(&sh.hist[k >> shift & 255], WEIGH ? rs.mass(x[j]) : 1);
                }
            });
            if (tid == 0 && floor_w && inside(floor_key)) lds_add(&sh.hist[floor_key >> shift & 255], floor_w);
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
    const uint64_t w = WEIGH ? rs.mass(last) : 1;
    ties = WEIGH ? (want - sh.sum + w - 1) / w : want - sh.sum;
    whole = last != floor && ties * w == sh.rest;
}

// The cells' token counts, in the histogram's place.  False where all of a row is one cell
// (a temperature above any use).
template <int DT, int WAVES, int STAGED>
__device__ __forceinline__ bool count_cells(SampleShared<WAVES> &sh, const SampleRow<DT, STAGED> &row, const RowScale &rs) {
    constexpr int VE = SampleRow<DT, STAGED>::VE;
    if (!(rs.step < 1.f)) return false;
    uint32_t *counts = reinterpret_cast<uint32_t *>(sh.hist);
    __syncthreads();
    for (int b = threadIdx.x; b < kCells; b += WAVES * kWave) counts[b] = 0;
    if (threadIdx.x == 0) sh.low = 0, sh.high = kCells - 1, sh.n = 1 << 30, sh.found = 0;
    __syncthreads();
    row.each([&](int, const float (&x)[VE]) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            int b;
            if (rs.cell(x[j], b)) atomicAdd(&counts[b], 1u);
        }
    });
    __syncthreads();
    return true;
}

// Where a cut falls, from the counts: in one of the cells low .. high, with `above` tokens
// above those and `tokens` up to their end.
struct Bounds {
    int low, high, above, tokens;
};

// top-k: one cell, or (false) none, where no more than k tokens weigh anything.
template <int WAVES>
__device__ __forceinline__ bool bound_count(SampleShared<WAVES> &sh, int k, Bounds &out) {
    constexpr int kPer = kCells / (WAVES * kWave);
    const uint32_t *counts = reinterpret_cast<uint32_t *>(sh.hist);
    uint64_t n = 0, waves, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) n += counts[threadIdx.x * kPer + i];
    int to = static_cast<int>(block_scan(sh, n, waves, total));
    if (static_cast<uint64_t>(k) >= total) return false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c = counts[threadIdx.x * kPer + i];
        if (to < k && k <= to + c) sh.high = threadIdx.x * kPer + i, sh.low = to, sh.n = to + c;
        to += c;
    }
    __syncthreads();
    out = {sh.high, sh.high, sh.low, sh.n};
    return true;
}

// The cut by top-k, from its cell's tokens.  False, and nothing decided, where those are too many
// to compare.
template <int DT, int WAVES, int STAGED>
__device__ __forceinline__ bool cut_cell(SampleShared<WAVES> &sh, const SampleRow<DT, STAGED> &row, const RowScale &rs,
                                         const Bounds &bounds, int k, float &last, uint64_t &ties, bool &whole) {
    constexpr int VE = SampleRow<DT, STAGED>::VE;
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    row.each([&](int, const float (&x)[VE]) {
        int c;
        if (!(rs.cell(largest(x), c) & (c <= bounds.high))) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if (rs.cell(x[j], c) & (c == bounds.high)) {
                const int n = atomicAdd(&sh.n, 1);
                if (n < kList) sh.list_x[n] = x[j];
            }
        }
    });
    __syncthreads();
    const int n = sh.n;
    if (n > kList) return false;
    for (int i = threadIdx.x; i < n; i += WAVES * kWave) {
        const float x = sh.list_x[i];
        int over = bounds.above, equal = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const float y = sh.list_x[j];
            over += y > x;
            equal += y == x;
        }
        if (over < k && k <= over + equal) sh.last = x, sh.sum = over, sh.rest = equal;
    }
    __syncthreads();
    last = sh.last;
    ties = k - sh.sum;
    whole = ties == sh.rest;
    return true;
}

// top_p: a token of cell c weighs 2^(-(c + 1/2) step) give or take 0.2 step of that (a uniform
// place in the cell), so the counts give every prefix's mass up to 0.2 step sqrt(sum of the
// cells' squared masses); the bounds leave six times that, and 5e-5 of the total for roundings.
// They may miss, where tokens lie in their cells other than by chance: what comes after finds
// out, and falls back.
template <int WAVES>
__device__ __forceinline__ void bound_mass(SampleShared<WAVES> &sh, const RowScale &rs, float top_p, Bounds &out) {
    constexpr int kPer = kCells / (WAVES * kWave);
    const uint32_t *counts = reinterpret_cast<uint32_t *>(sh.hist);
    // masses in 2^-22 of the largest (below 2^42 in all) with the tokens' number behind, so that
    // one sum over the threads does
    uint64_t mass[kPer], to = 0, all, waves;
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = threadIdx.x * kPer + i;
        const uint32_t n = counts[b];
        const float w = static_cast<float>(n) * __builtin_amdgcn_exp2f(-rs.step * (static_cast<float>(b) + 0.5f));
        mass[i] = static_cast<uint64_t>(w * 4194304.f + 0.5f) << 21 | n;
        squares += w * w;
        to += mass[i];
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) squares += __shfl_xor(squares, o, kWave);
    if (threadIdx.x % kWave == 0) sh.list_x[threadIdx.x / kWave] = squares;
    to = block_scan(sh, to, waves, all);
    squares = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) squares += sh.list_x[i];
    const float sum = static_cast<float>(all >> 21), want = top_p * sum;
    const float margin = 1.2f * rs.step * 4194304.f * __builtin_amdgcn_sqrtf(squares) + 5e-5f * sum;
    const float from = want - margin, end = want + margin;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = threadIdx.x * kPer + i;
        const float before = static_cast<float>(to >> 21);
        to += mass[i];
        const float after = static_cast<float>(to >> 21);
        if (before < from && from <= after) sh.low = b;
        if (before < end && end <= after) sh.high = b, sh.n = static_cast<int>(to & 0x1FFFFF);
    }
    __syncthreads();
    out = {sh.low, sh.high, 0, sh.n};
}

// The cut by masses over all tokens (no top-k before it, no min_p behind) with each one's mass
// computed once, which gives the kept masses of the lanes' waves along with the cut (mass: of
// tokens above `last`, or equal to it where all of those are kept; count: of the tokens equal
// to it otherwise).  Masses of tokens above the bounds are added up in the lanes, only those
// between them go into shared sums, at most kRange parts of the bounds for each wave.
// False, and nothing decided, where the bounds miss the cut, or a part holds too many tokens to
// compare.
template <int DT, int WAVES, int STAGED, typename F>
__device__ __forceinline__ bool cut_once(SampleShared<WAVES> &sh, const SampleRow<DT, STAGED> &row, const RowScale &rs,
                                         const Bounds &bounds, F share, float &last, uint64_t &ties, bool &whole,
                                         uint64_t &mass, uint64_t &count) {
    constexpr int kThreads = WAVES * kWave, VE = SampleRow<DT, STAGED>::VE, kRange = 2 * kWave;
    static_assert(WAVES * kRange <= kBuckets, "the waves' sums take the histogram's place");
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const int low = bounds.low, range = bounds.high - low + 1;
    if (range < 1) return false;
    uint64_t waves;
    __syncthreads();
    if (tid == 0) sh.n = 0;
    uint64_t *sums = sh.hist;  // [wave][kRange]
    for (int b = tid; b < WAVES * kRange; b += kThreads) sums[b] = 0;
    __syncthreads();
    // the bounds as logits, and the parts between them: `width` cells each
    const int join = (range + kRange - 1) / kRange, parts = join > 1 ? (range + join - 1) / join : range * (kRange / range);
    const float width = join > 1 ? static_cast<float>(join) : 1.f / static_cast<float>(kRange / range);
    const float cell = 1.f / rs.per_half, from = static_cast<float>(low), fine = 1.f / width;
    const float high_x = rs.top - from * cell, low_x = rs.top - static_cast<float>(bounds.high + 1) * cell;
    auto part = [&](float x) { return max(0, min(parts - 1, static_cast<int>((rs.place(x) * 2.f - from) * fine))); };
    uint64_t rest = 0;
    mass = 0;
    row.each([&](int, const float (&x)[VE]) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const uint64_t w = RowScale::mass_bits(rs.exponent(x[j]));
            rest += w;
            mass += x[j] > high_x ? w - RowScale::kBits : 0;
            if ((x[j] <= high_x) & (x[j] >= low_x)) lds_add(&sums[wave * kRange + part(x[j])], w - RowScale::kBits);
        }
        rest -= VE * RowScale::kBits;
    });
    uint64_t all, above;
    block_scan(sh, rest, waves, all);
    block_scan(sh, mass, waves, above);
    const uint64_t want = share(all);
    // every wave finds the part for itself: lane k has the parts 2 k and 2 k + 1
    uint64_t even = 0, odd = 0;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) even += sums[k * kRange + 2 * lane], odd += sums[k * kRange + 2 * lane + 1];
    const uint64_t to_even = above + wave_scan_u64(even + odd) - odd, to_odd = to_even + odd;
    const uint64_t hit_even = __ballot(to_even - even < want && want <= to_even);
    const uint64_t hit_odd = __ballot(to_even < want && want <= to_odd);
    if (!(hit_even | hit_odd)) return false;
    const int owner = __builtin_ctzll(hit_even | hit_odd), found = 2 * owner + (hit_even ? 0 : 1);
    const uint64_t over0 = shfl_u64(hit_even ? to_even - even : to_even, owner);
    // (half a cell around the part: nearly all tokens are told by two comparisons)
    const float part_high = fminf(high_x, rs.top - (from + static_cast<float>(found) * width - 0.5f) * cell);
    const float part_low = fmaxf(low_x, rs.top - (from + static_cast<float>(found + 1) * width + 0.5f) * cell);
    row.each([&](int, const float (&x)[VE]) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if (!((x[j] <= part_high) & (x[j] >= part_low))) continue;
            if (part(x[j]) == found) {
                const int n = atomicAdd(&sh.n, 1);
                if (n < kList) sh.list_x[n] = x[j], sh.list_wave[n] = static_cast<uint8_t>(wave);
            }
        }
    });
    __syncthreads();
    const int n = sh.n;
    if (n > kList) return false;
    for (int i = tid; i < n; i += kThreads) sh.list_w[i] = rs.mass(sh.list_x[i]);
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const float x = sh.list_x[i];
        uint64_t over = over0, equal = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const float y = sh.list_x[j];
            const uint64_t w = sh.list_w[j];
            over += y > x ? w : 0;
            equal += y == x ? w : 0;
        }
        if (over < want && want <= over + equal) sh.last = x, sh.sum = over, sh.rest = equal;
    }
    __syncthreads();
    last = sh.last;
    const uint64_t w = rs.mass(last);
    ties = (want - sh.sum + w - 1) / w;
    whole = ties * w == sh.rest;
    count = 0;
    for (int k = lane; k < found; k += kWave) mass += sums[wave * kRange + k];
    for (int i = lane; i < n; i += kWave) {
        const float x = sh.list_x[i];
        if (sh.list_wave[i] != wave) continue;
        if (x > last || (whole && x == last)) mass += sh.list_w[i];
        else count += x == last;
    }
    return true;
}

template <int DT, int WAVES, int STAGED>
__global__ __launch_bounds__(WAVES *kWave) void sample_kernel(const SampleArgs a) {
    __shared__ SampleShared<WAVES> sh;
    __shared__ u32x4 stage[STAGED > 0 ? STAGED * WAVES * kWave : 1];
    using Row = SampleRow<DT, STAGED>;
    constexpr int VE = Row::VE;
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave), r = blockIdx.x;
    Row row;
    row.base = static_cast<const char *>(a.logits) + r * a.stride_n * Row::es;
    row.vocab = a.vocab;
    row.per = (a.vocab + WAVES * kWave * VE - 1) / (WAVES * kWave * VE);
    row.place(wave, lane);
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
    row.template each<true>([&](int, const float (&x)[VE]) {
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
        row.each([&](int i, const float (&x)[VE]) {
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
    rs.least = min_p > 0.f ? log2(static_cast<double>(min_p < 1.f ? min_p : 1.f)) : -1e300;
    rs.per_half = fminf(2.f * (kBuckets - 1) / (kBucketSpan * T), 1e30f);
    rs.step = static_cast<float>(rs.rate / static_cast<double>(rs.per_half));

    auto masses = [&](const float (&x)[VE]) {  // of a chunk
        uint64_t sum = 0;
#pragma unroll
        for (int j = 0; j < VE; ++j) sum += RowScale::mass_bits(rs.exponent(x[j]));
        return sum - VE * RowScale::kBits;
    };
    // Few tokens are left as a rule by top-k, where min_p alone cuts, or above top_p's bounds:
    // one thread takes each, in the order of their indices, and the rest is a few sums over the
    // threads.  (top_p alone also needs the mass of all.)
    Bounds bounds{0, kCells - 1, 0, 1 << 30};
    const bool counted = (top_k < a.vocab || top_p < 1.f) && count_cells(sh, row, rs);
    const bool by_count = counted && top_k < a.vocab && bound_count(sh, top_k, bounds);
    if (counted && !by_count) top_k = a.vocab;
    const bool by_mass = counted && !by_count && top_p < 1.f;
    if (by_mass) bound_mass(sh, rs, top_p, bounds);
    // kept are the tokens above `last`, and of those equal to it the first `ties`
    float last = -kInf;
    uint64_t ties = 0;
    bool whole = true;
    // where the last cell holds too many tokens, as it does with many equal ones, top-k's cut first
    const bool celled = by_count && bounds.tokens > WAVES * kWave && cut_cell(sh, row, rs, bounds, top_k, last, ties, whole);
    const bool exact = celled && top_k <= WAVES * kWave;
    const int last_tie = exact && !whole ? find_equal(sh, row, last, [&](uint64_t) { return ties; }) : a.vocab;
    if (by_count || by_mass ? exact || bounds.tokens <= WAVES * kWave : top_k == a.vocab && top_p >= 1.f && min_p > 0.f) {
        uint64_t all_mass = 0, waves, total;
        // nothing below this weighs: what min_p leaves, with room for rounding, or the bounds'
        // end, in cells
        const float far = top + static_cast<float>(rs.least / rs.rate), room = 1e-5f * (fabsf(top) + fabsf(far));
        const float least_x = exact ? last : counted ? -__FLT_MAX__ : fmaxf(far - room, -__FLT_MAX__);
        const float end = static_cast<float>(bounds.high + 1);
        auto stays = [&](float x) { return (x >= least_x) & (rs.place(x) * 2.f < end); };
        auto drop_ties = [&](int i, float (&x)[VE]) {
            if (last_tie >= a.vocab) return;
#pragma unroll
            for (int j = 0; j < VE; ++j) x[j] = x[j] == last && row.index(i) + j > last_tie ? -kInf : x[j];
        };
        uint64_t n = 0, sum = 0, first = 0, all;
        int *list_i = reinterpret_cast<int *>(sh.list_w);
        // Up to 64 are gathered as they come and put in order by one wave, which saves the pass that
        // counts them (top_k 50, 8 x 32000 fp32: 15.8 -> 13.9 us, 64 x 50304 bf16 21.7 -> 17.9; a pass
        // over 4096 tokens costs less than the ordering, 1 x 4000 9.7 -> 10.6).
        const bool few = WAVES > 4 && by_count && !exact && bounds.tokens <= kWave;
        if (few) {
            row.each([&](int i, const float (&x)[VE]) {
                if (!stays(largest(x))) return;
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    if (!stays(x[j])) continue;
                    const int k = atomicAdd(&sh.found, 1);
                    sh.list_x[k] = x[j], list_i[k] = row.index(i) + j;
                }
            });
            __syncthreads();
            all = bounds.tokens;
            if (wave == 0) {
                const float x = sh.list_x[lane];
                const int index = list_i[lane];
                int place = 0;
                for (int j = 0; j < bounds.tokens; ++j) place += __builtin_amdgcn_readlane(index, j) < index;
                if (lane < bounds.tokens) sh.list_x[place] = x, list_i[place] = index;
            }
        } else {
            row.each([&](int i, float (&x)[VE]) {
                drop_ties(i, x);
#pragma unroll
                for (int j = 0; j < VE; ++j) n += stays(x[j]);
                if (by_mass) sum += masses(x);
            });
            block_scan(sh, n, first, all);
            if (by_mass) block_scan(sh, sum, waves, all_mass);
        }
        bool closed = all <= WAVES * kWave;
        if (closed) {
            int at = static_cast<int>(first);
            if (!few) row.each([&](int i, float (&x)[VE]) {
                if (!__any(stays(largest(x)))) return;
                drop_ties(i, x);
                int chunk = 0, place = at;
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const uint64_t b = __ballot(stays(x[j]));
                    chunk += __popcll(b);
                    place += __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(b >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(b), 0));
                }
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    if (stays(x[j])) {
                        sh.list_x[place] = x[j], list_i[place] = row.index(i) + j;
                        ++place;
                    }
                }
                at += chunk;
            });
            __syncthreads();
            // One wave can do without barriers (8 x 32000 fp32, top_k 50: 17.0 -> 15.9 us; with top_p
            // behind it 18.8 -> 19.2, so not there)
            if (all <= kWave && !(top_p < 1.f)) {
                if (wave) return;
                const int number = static_cast<int>(all);
                const bool mine = lane < number;
                const float x = mine ? sh.list_x[lane] : -kInf;
                const double t = rs.exponent(mine ? x : top);
                uint64_t w = RowScale::select(mine && rs.place(x) < static_cast<float>(kBuckets - 1), RowScale::mass_of(t));
                if (by_count && !exact) {
                    int c;
                    const bool in = rs.cell(x, c) && c == bounds.high;
                    int rank = bounds.above;
                    for (uint64_t set = __ballot(in); set; set &= set - 1) {
                        const int j = __builtin_ctzll(set);
                        const float y = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), j));
                        rank += (y > x) | ((y == x) & (j < lane));
                    }
                    w = RowScale::select(!in || rank < top_k, w);
                }
                w = RowScale::select(t >= rs.least, w);
                const uint64_t to = wave_scan_u64(w), target = target_of(last_lane(to));
                if (to <= target + w && target < to && w) a.out[r] = list_i[lane];
                return;
            }
            const bool mine = tid < static_cast<int>(all);
            const float x = mine ? sh.list_x[tid] : -kInf;
            const int index = mine ? list_i[tid] : 0;
            const double t = rs.exponent(mine ? x : top);
            uint64_t w = RowScale::select(mine, RowScale::mass_of(t));
            int b;
            if (!rs.bucket(x, b)) b = kBuckets, w = 0;
            // the weight ranked before this token within its bucket, among those `in` it
            auto before_in_bucket = [&](bool in, uint64_t weight) {
                uint64_t over = 0;
                __syncthreads();
                if (tid == 0) sh.n = 0;
                __syncthreads();
                if (in) {
                    const int k = atomicAdd(&sh.n, 1);
                    sh.list_x[k] = x, sh.list_w[k] = weight << 10 | tid;  // (a mass is below 2^43)
                }
                __syncthreads();
                if (in) {
                    const int m = sh.n;
#pragma unroll 8
                    for (int k = 0; k < m; ++k) {
                        const float y = sh.list_x[k];
                        const uint64_t v = sh.list_w[k];
                        over += y > x || (y == x && static_cast<int>(v & 1023) < tid) ? v >> 10 : 0;
                    }
                }
                return over;
            };
            if (by_count && !exact) {
                int c;
                const bool in = rs.cell(x, c) && c == bounds.high;
                const uint64_t rank = bounds.above + before_in_bucket(in, 1);
                w = in && rank >= static_cast<uint64_t>(top_k) ? 0 : w;
            }
            if (top_p < 1.f) {
                __syncthreads();
                for (int k = tid; k < kBuckets; k += WAVES * kWave) sh.hist[k] = 0;
                __syncthreads();
                if (w) lds_add(&sh.hist[b], w);
                __syncthreads();
                uint64_t part;
                const uint64_t before = scan_hist(sh, part, total), want = share(by_mass ? all_mass : total);
                closed = want <= total;  // (else the bounds have missed)
                if (closed) {
                    locate(sh, before, part, want);
                    const int bucket = sh.bucket;
                    const uint64_t over = sh.sum + before_in_bucket(w && b == bucket, w);
                    w = b > bucket || (b == bucket && over >= want) ? 0 : w;
                }
            }
            w = RowScale::select(t >= rs.least, w);
            const uint64_t to = block_scan(sh, w, waves, total), target = target_of(total);
            if (closed && to <= target && target < to + w) a.out[r] = index;
        }
        if (closed) return;
    }

    // Else
    uint64_t mass = 0, count = 0;  // the lane's kept ones, once summed
    if (top_k < a.vocab && !celled)
        cut<false>(sh, row, rs, last, ties, whole, [&](uint64_t) { return static_cast<uint64_t>(top_k); });
    const bool summed =
        by_mass && !(min_p > 0.f) && cut_once(sh, row, rs, bounds, share, last, ties, whole, mass, count);
    if (top_p < 1.f && !summed) cut<true>(sh, row, rs, last, ties, whole, share);

    // The row is summed (once more): the masses above `last`, and the tokens equal to it,
    // of which the first `ties` weigh.  Where all of them are kept, they are the ones above the
    // next value below it (below 0 that is not -0).
    if (whole && ties) {
        last = key_logit(logit_key(last) - (last == 0.f ? 2 : 1));
        ties = 0;
    }
    const double tie_t = ties ? rs.exponent(last) : 0.0;
    const uint64_t tie_w = ties && tie_t >= rs.least ? RowScale::mass_of(tie_t) : 0;
    auto sum_of = [&](uint64_t mass, uint64_t count) { return mass + tie_w * (count < ties ? count : ties); };
    auto token = [&](float x) {
        const double t = rs.exponent(x);
        return RowScale::select((x > last) & (t >= rs.least), RowScale::mass_of(t));
    };
    const bool plain = last == -kInf && !(min_p > 0.f);
    auto add_chunk = [&](const float (&x)[VE], uint64_t &mass, uint64_t &count) {
        if (plain) {
            mass += masses(x);
            return;
        }
        if (!(largest(x) >= last)) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) mass += token(x[j]);
        if (ties) {
#pragma unroll
            for (int j = 0; j < VE; ++j) count += x[j] == last;
        }
    };
    uint64_t all_mass, all_count, mass0, count0;  // ..0: before what is looked at
    if (!summed) {
        mass = count = 0;
        row.template each<false, true>([&](int, const float (&x)[VE]) { add_chunk(x, mass, count); });
    }
    const uint64_t wave_count = ties ? last_lane(wave_scan_u64(count)) : 0;
    count0 = all_count = 0;
    if (ties) block_scan(sh, count, count0, all_count);
    block_scan(sh, mass, mass0, all_mass);
    const uint64_t target = target_of(sum_of(all_mass, all_count));
    // the wave with the token, then its chunks, taken by all waves 64 lanes' sums each
    if (lane == 0 && sum_of(mass0, count0) <= target && target < sum_of(mass0 + sh.part[wave], count0 + wave_count))
        sh.owner = wave, sh.sum = mass0, sh.rest = count0;
    __syncthreads();
    mass0 = sh.sum, count0 = sh.rest;
    const int shift = sh.owner - wave;
    row.place(__builtin_amdgcn_readfirstlane(sh.owner), lane);
    row.lds += shift * kWave;
    // the lane that has the target among its (mass, count), which follow each other lane by lane,
    // or -1; mass0, count0 move to before that lane, or behind all
    auto pick = [&](uint64_t m, uint64_t c) {
        const uint64_t mi = wave_scan_u64(m), ci = ties ? wave_scan_u64(c) : 0;
        const uint64_t hit = __ballot(target < sum_of(mass0 + mi, count0 + ci));
        const int l = hit ? __builtin_ctzll(hit) : kWave - 1;
        mass0 += shfl_u64(hit ? mi - m : mi, l);
        count0 += ties ? shfl_u64(hit ? ci - c : ci, l) : 0;
        return hit ? l : -1;
    };
    constexpr int kRound = kBuckets / kWave;  // chunks whose sums fit
    static_assert(sizeof(sh.list_w) >= kBuckets * sizeof(int), "the counts take the list's place");
    int *counts = reinterpret_cast<int *>(sh.list_w);
    bool done = false;
    for (int i0 = 0; i0 < row.per; i0 += kRound) {
        const int n = min(kRound, row.per - i0);
        __syncthreads();
        for (int i = wave; i < n; i += WAVES) {
            float x[VE];
            row.fetch(i0 + i, x);
            uint64_t m = 0, c = 0;
            add_chunk(x, m, c);
            sh.hist[i * kWave + lane] = m;
            counts[i * kWave + lane] = static_cast<int>(c);
        }
        __syncthreads();
        if (wave || done) continue;
        // in order, chunk by chunk: the lane whose n sums in a row have the target, then the sum,
        // then the token
        uint64_t m = 0, c = 0;
#pragma unroll 8
        for (int k = 0; k < n; ++k) m += sh.hist[lane * n + k], c += counts[lane * n + k];
        const int l = pick(m, c);
        if (l < 0) continue;
        const bool one = lane < n;
        const int k = l * n + pick(one ? sh.hist[l * n + lane] : 0, one ? counts[l * n + lane] : 0);
        const int i = i0 + k / kWave, other = k % kWave - lane;  // lane k % 64's of chunk k / 64
        Row its = row;
        its.start += other * VE;
        its.lds += other;
        const float x = lane < VE ? its.one(i, lane) : -kInf;
        if (pick(token(x), ties && x == last) == lane) a.out[r] = its.index(i) + lane;
        done = true;
    }
}

namespace {

template <int DT, int WAVES, int STAGED>
void launch(const SampleArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((sample_kernel<DT, WAVES, STAGED>), dim3(a.n), dim3(WAVES * kWave), 0, s, a);
}

// Up to 4096 tokens take 4 waves, more 16.  Without cuts, with top_k 50 and with top_p 0.9: 256 x 4000
// bf16 7.4, 9.7 and 16.7 us (16 waves 10.0, 10.3 and 21.5), one row 6.7, 9.1 and 15.6 (8.7, 9.4 and
// 20.2); fp32 7.6, 10.3 and 15.6 (9.3, 9.4 and 18.4), one row 6.9, 9.6 and 14.6 (8.1, 8.4 and 17.0):
// of these only fp32 with top_k would take less with 16.  Rows
// go through LDS where they fit (131072 bytes) and each has a CU to itself: 64 x 50304 bf16 20,
// 18 and 42 us (8 waves without LDS 21, 22, 47).  With more rows than CUs, two smaller
// workgroups on each hide one's memory behind the other's arithmetic: 512 x 50304 bf16 36, 33
// and 71 us (one of 16 waves at a time 45, 38, 86), fp32 42, 49 and 80 (49, 55, 100).
template <int DT>
void run(const SampleArgs &a, hipStream_t s) {
    constexpr int kLds = 8, kChunk = kWave * (DT == PRIME_F32 ? 4 : 8);
    if (a.vocab <= 4096) launch<DT, 4, 4096 / (4 * kChunk)>(a, s);
    else if (a.n > 256) launch<DT, 8, 0>(a, s);
    else if (a.vocab <= kLds * 16 * kChunk) launch<DT, 16, kLds>(a, s);
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
