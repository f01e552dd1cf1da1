// One row number drawn from each score row (vdb_sample_dev): temperature, top-k, top-p, min-p, a row filter, and a
// uniform number given by the caller.
//
// What remains of a row after the filters is a prefix of the order (score descending, row number ascending): a
// smallest score and how many of the rows that share it.  It is found without sorting:
//   - top-k, or min-p alone, leaves few rows: those at or above a bound (no fewer than k rows reach the k-th largest of
//     the maxima of k groups or more) go to a list in LDS, in row order, and everything else happens there;
//   - top-p alone takes a histogram of the weights over the distance from the best score, and then the scores of the one
//     bin in which the border lies, narrowed by their ordered bit patterns.
// Weights exp((z - max) / tau) are taken in double, to 2^-50, rounded to multiples of 2^-s (2^-45 at 131072 scores) and added as
// 64-bit integers: sums are exact and do not depend on the order in which threads add.  s is as large as the sum of a row of
// weights of 1 allows; a border lies within vocab * 2^-(s+1) of that of unrounded weights, 2^-29 of the best one's weight at 131072.
//
// Two forms.  Short rows: a block of 1024 threads takes a row through all its passes.  Long rows are streamed by the whole
// chip: one pass takes the maxima of groups of 32 scores (the floor: n * vocab values read once), a block per row finishes
// the rows that a list settles from those maxima, and for the others two more passes add up weights.  A top-k above LIST_MAX / 2, a
// list or a border's bin of more than LIST_MAX scores send a row through all its passes by one block, behind the passes that
// the chip went through: of 131072 bf16 scores of standard deviation 1, one row 103 us with top-k 5000, 222 with temperature 2
// and top-p 0.5, 256 rows 131 and 319 us (131 with top-p 0.9, whose bin is small enough).
#include "vdb_internal.h"
#include "values.h"

#include <algorithm>

namespace vdb {

// Passes over a whole row by one block take ROW_NT threads.  Everything else that a block does for a row is a chain of short
// steps between barriers, and every instruction of such a step costs each wave of a SIMD its turn: FEW_NT threads, two waves
// a SIMD (one row of 131072 bf16 scores, top-k 400: 23 us; with 256 threads 30, with 1024 27).
static constexpr int ROW_NT = 1024, ROW_WAVES = ROW_NT / 64, FEW_NT = 512;
static constexpr int LIST_MAX = 2048, BINS = 2048, EXP_STEPS = 1024, GROUPS = 64, AHEAD = 4, PAIRS = 256;
typedef unsigned long long u64;
static constexpr float LOWEST = -3.4028234663852886e38f;

struct SampleArgs {
    int64_t vocab, ld;
    int smaller_first;
    const float* uniform;
    const float* d_temperature; float temperature;
    const int32_t* d_top_k; int top_k;
    const float* d_top_p; float top_p;
    const float* d_min_p; float min_p;
    const uint32_t* mask; int64_t mask_ld;
    int64_t* out_row; float* out_logp;
    int shift;                       // weights are multiples of 2^-shift
};
// what a row asks for
struct Settings {
    float tau, top_p, min_p, uniform;
    int top_k;
    __device__ __forceinline__ Settings(const SampleArgs& a, int64_t row)
        : tau(a.d_temperature ? a.d_temperature[row] : a.temperature), top_p(a.d_top_p ? a.d_top_p[row] : a.top_p),
          min_p(a.d_min_p ? a.d_min_p[row] : a.min_p), uniform(a.uniform[row]), top_k(a.d_top_k ? a.d_top_k[row] : a.top_k) {}
    __device__ __forceinline__ bool first_of_best() const { return !(tau > 0.0f) || top_k == 1 || top_p <= 0.0f; }
    __device__ __forceinline__ bool by_count() const { return top_k > 1; }
    __device__ __forceinline__ bool by_mass() const { return top_p < 1.0f; }
    __device__ __forceinline__ u64 least_weight(int shift) const {
        return min_p > 0.0f ? (u64)ceil(fmin((double)min_p, 1.0) * (double)((u64)1 << shift)) : 0;
    }
    // no score below weighs min_p of the best
    __device__ __forceinline__ float min_p_bound(float best) const {
        const double lowest = (double)best + log(fmin((double)min_p, 1.0)) * (double)tau;
        return (float)fmax(lowest - (fabs(lowest) + fabs((double)best)) * 1e-6, (double)LOWEST);
    }
    // running sum > uniform * total, as integers
    __device__ __forceinline__ u64 goal(u64 total) const {
        const double g = (double)uniform * (double)total;
        const u64 least = g >= 0.0 ? (u64)floor(g) + 1 : 1;
        return least <= total ? least : total;
    }
};

// Ordered pattern of a score that can be drawn: larger score, larger pattern.  -0 counts as +0; 0 for NaN and -inf.
__device__ __forceinline__ uint32_t pattern(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return z > -INFINITY ? o : 0u;
}
__device__ __forceinline__ float score_of(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }

// A row's pieces: what cannot be drawn (filtered, behind the end) is -inf; a NaN fails every comparison and never counts.
template <class T> struct Source {
    const T* z;
    int vocab;
    const uint32_t* mask;
    bool flip, infinite;             // infinite: the best is +inf; those rows weigh 1, the others nothing
    static __device__ __forceinline__ uint32_t nothing() { return sizeof(T) == 4 ? 0xff800000u : (__is_same(T, bf16_t) ? 0xff80ff80u : 0xfc00fc00u); }
    __device__ __forceinline__ Piece<T> load(int at) const {
        constexpr int N = Piece<T>::N;
        Piece<T> x;
        if (at + N <= vocab) x = load_piece(z + at);
        else {
            float v[N];
            load_values(z, at, vocab, flip ? INFINITY : -INFINITY, v);
            x.set(v);
        }
        return x;
    }
    __device__ __forceinline__ Source(const T* scores, const SampleArgs& a, int64_t row)
        : z(scores + row * a.ld), vocab((int)a.vocab), mask(a.mask ? a.mask + row * a.mask_ld : nullptr), flip(a.smaller_first != 0), infinite(false) {}
    // one score
    __device__ __forceinline__ float one(int at) const {
        if (at >= vocab || (mask && !((mask[at >> 5] >> (at & 31)) & 1u))) return -INFINITY;
        float x = (float)z[at];
        if (flip) x = -x;
        if (infinite) x = x == INFINITY ? 0.0f : -INFINITY;
        return x > -INFINITY ? x : -INFINITY;
    }
    __device__ __forceinline__ uint32_t bits(int at) const { return mask && at < vocab ? mask[at >> 5] >> (at & 31) : 0xffffffffu; }   // N divides 32
    __device__ __forceinline__ void finish(Piece<T>& x, uint32_t bits) const {
        if (flip) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x.raw[i] ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
        }
        if (mask) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t keep;
                if constexpr (sizeof(T) == 4) keep = 0u - ((bits >> i) & 1u);
                else keep = ((0u - ((bits >> (2 * i)) & 1u)) & 0xffffu) | ((0u - ((bits >> (2 * i + 1)) & 1u)) << 16);
                x.raw[i] = (x.raw[i] & keep) | (nothing() & ~keep);
            }
        }
        if (infinite) only_infinite(x);
    }
    static __device__ __forceinline__ void only_infinite(Piece<T>& x) {
        constexpr int N = Piece<T>::N;
        float y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = x.get(e) == INFINITY ? 0.0f : -INFINITY;
        x.set(y);
    }
};

// The weight exp((z - best) / tau) as a multiple of 2^-s: with x = (z - best) c, c = 1024 log2(e) / tau, and k = x rounded,
// 2^(x / 1024) = 2^(k >> 10) table[k & 1023] q(x - k), q a cubic (its remainder is below 2^-50 for |x - k| <= 1/2).  Adding
// 2^(52 - s) leaves the multiple in the low mantissa bits.  Nine double instructions, 8 cycles each, and as many others,
// are what streaming weights is bound by (33.5M of them: 36 us; with 32 entries and degree 5, free of bank conflicts, 41 us).
struct FixedExp {
    double best, c, round_to;        // round_to = 2^(52 - s)
    float cut;                       // scores below weigh nothing (2^-40 of the best)
    const double* table;             // 2^(j / 1024), in LDS
    static constexpr double NEAREST = 6755399441055744.0;            // 1.5 * 2^52: the nearest integer in the low bits
    __device__ __forceinline__ FixedExp(float best_, float tau, int shift, const double* t)
        : best(best_), c(EXP_STEPS * 1.4426950408889634073599 / (double)tau), round_to((double)((u64)1 << (52 - shift))),
          cut((float)fmax((double)best_ - 40.0 * 0.69314718055994530942 * (double)tau, (double)LOWEST)), table(t) {}
    // Distances from the best are binned in steps of 1/32 of a power of two.  Scores of bin b lie in [*lo, *hi]; what else
    // does is told apart by its bin.
    __device__ __forceinline__ void bin_range(int b, float* lo, float* hi) const {
        const double h = best - (32.0 * b - 0.6) / c, l = best - (32.0 * b + 31.6) / c;
        *hi = (float)fmin(best, h + fabs(h) * 2.4e-7);
        *lo = (float)fmax(l - fabs(l) * 2.4e-7, (double)cut);
    }
    __device__ __forceinline__ int bin(float z) const {
        const int k = (int)(uint32_t)__double_as_longlong(fma((double)z - best, c, NEAREST));
        return (int)min((uint32_t)-k >> 5, (uint32_t)(BINS - 1));
    }
    // the same without the table, for a few scores: exp2() to the last bits of a double
    __device__ __forceinline__ u64 directly(float z) const {
        const double w = exp2(((double)z - best) * (c / EXP_STEPS));
        return z >= cut ? (u64)__double_as_longlong(w + round_to) - (u64)__double_as_longlong(round_to) : 0;
    }
    __device__ __forceinline__ u64 operator()(float z) const { return from(z, cut); }
    // 0 for scores below `least`, which is not below cut
    __device__ __forceinline__ u64 from(float z, float least) const {
        constexpr double L = 0.69314718055994530942 / EXP_STEPS;
        const double d = (double)z - best;
        const double a = fma(d, c, NEAREST);
        const int k = (int)(uint32_t)__double_as_longlong(a);
        const double f = fma(d, c, -(a - NEAREST));
        double q = fma(f, L * L * L / 6, L * L / 2);
        q = fma(f, q, L);
        q = fma(f, q, 1.0);
        const u64 t = (u64)__double_as_longlong(table[k & (EXP_STEPS - 1)]);
        const double scale = __longlong_as_double((long long)(t + ((u64)(uint32_t)(k >> 10) << 52)));
        const u64 r = (u64)__double_as_longlong(fma(scale, q, round_to)) - (u64)__double_as_longlong(round_to);
        return z >= least ? r : 0;
    }
};

struct SampleShared {
    double table[EXP_STEPS];
    u64 bin[BINS];
    float list_z[LIST_MAX];
    uint32_t list_at[LIST_MAX];
    u64 part[ROW_WAVES * GROUPS];     // per part of the row, in row order: counts or weights, then their exclusive prefix
    u64 pair_sum[PAIRS], pair_w[PAIRS];
    uint32_t pair_rank[PAIRS];
    u64 few_w[64];
    uint32_t few_key[64];
    u64 red[ROW_WAVES];
    u64 found_sum;
    uint32_t found, first, listed, few;
};

// Sums over a wave by data-parallel moves (rows of 16 lanes, then their last lanes passed on): a shuffle through LDS costs
// a hundred cycles a step, and these stand once in every step of every pass.
template <int CTRL, int ROWS> __device__ __forceinline__ u64 add_moved(u64 v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return v + (((u64)hi << 32) | lo);
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
    v = add_moved<0x111, 0xf>(v);        // row_shr:1, 2, 4, 8
    v = add_moved<0x112, 0xf>(v);
    v = add_moved<0x114, 0xf>(v);
    v = add_moved<0x118, 0xf>(v);
    v = add_moved<0x142, 0xa>(v);        // row_bcast:15 into rows 1 and 3
    return add_moved<0x143, 0xc>(v);     // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ u64 last_lane(u64 v) {
    return ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}
__device__ __forceinline__ u64 wave_sum(u64 v) { return last_lane(wave_scan(v)); }
// Helpers of a block's first NT threads (the others have ended, or take part elsewhere in no barrier).
// exclusive prefix of v; *total = its sum
template <int NT> __device__ __forceinline__ u64 block_scan(SampleShared& sh, u64 v, u64* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 inc = wave_scan(v);
    __syncthreads();
    if (lane == 63) sh.red[wave] = inc;
    __syncthreads();
    u64 all = 0, base = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const u64 r = sh.red[w];
        base += w < wave ? r : 0;
        all += r;
    }
    *total = all;
    return base + inc - v;
}
template <int NT> __device__ __forceinline__ u64 block_total(SampleShared& sh, u64 v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) v += sh.red[w];
    return v;
}
// the parts' exclusive prefix in place; -> their sum
template <int NT> __device__ __forceinline__ u64 scan_parts(SampleShared& sh, int parts) {
    constexpr int PER = ROW_WAVES * GROUPS / NT;
    __syncthreads();
    const int at = threadIdx.x * PER;
    u64 v[PER], sum = 0, total;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += v[j] = at + j < parts ? sh.part[at + j] : 0;
    u64 run = block_scan<NT>(sh, sum, &total);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (at + j < parts) sh.part[at + j] = run;
        run += v[j];
    }
    __syncthreads();
    return total;
}
template <int NT> __device__ __forceinline__ void clear_bins(SampleShared& sh) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < BINS / NT; ++j) sh.bin[j * NT + threadIdx.x] = 0;
    __syncthreads();
}
// 2^(j / 1024), by exp's series to the last bits of a double
struct ExpTable {
    double v[EXP_STEPS];
    constexpr ExpTable() : v() {
        for (int j = 0; j < EXP_STEPS; ++j) {
            const double x = 0.69314718055994530942 * j / EXP_STEPS;
            double sum = 1.0;
            for (int k = 20; k >= 1; --k) sum = 1.0 + sum * x / k;
            v[j] = sum;
        }
    }
};
__device__ constexpr ExpTable EXP_TABLE{};
template <int NT> __device__ __forceinline__ void make_table(double* table) {
#pragma unroll
    for (int j = 0; j < EXP_STEPS / NT; ++j) table[j * NT + threadIdx.x] = EXP_TABLE.v[j * NT + threadIdx.x];
}
// the first bin, from the top or from the bottom, at which the running sum, from `above`, reaches target: sh.found its
// number in that order (BINS: none), sh.found_sum the sum before it
template <int NT> __device__ __forceinline__ void find_bin(SampleShared& sh, u64 above, u64 target, bool from_top) {
    constexpr int PER = BINS / NT;
    __syncthreads();
    const int at = PER * threadIdx.x;
    u64 v[PER], sum = 0, total;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += v[j] = sh.bin[from_top ? BINS - 1 - at - j : at + j];
    if (threadIdx.x == 0) sh.found = BINS;
    u64 run = above + block_scan<NT>(sh, sum, &total);          // its barriers order the write above with those below
    if (run < target && run + sum >= target) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (run < target && run + v[j] >= target) {
                sh.found = (uint32_t)(at + j);
                sh.found_sum = run;
            }
            run += v[j];
        }
    }
    __syncthreads();
}

// Keys [first, last] in parts of 2^shift, at most BINS of them; the last part ends with the range.
struct KeyRange {
    uint32_t first, last;
    __host__ __device__ constexpr int part_shift() const {
        int shift = 0;
        while ((last - first) >> shift >= (uint32_t)BINS) ++shift;
        return shift;
    }
    __host__ __device__ constexpr KeyRange part(uint32_t b, int shift) const {
        // compared before it is added: row numbers are searched as ~row, whose last part lies next to 2^32
        const uint32_t lo = first + (b << shift), width = (1u << shift) - 1;
        return {lo, last - lo > width ? lo + width : last};
    }
};
constexpr bool parts_cover(KeyRange r) {
    const int shift = r.part_shift();
    const uint32_t most = (r.last - r.first) >> shift;
    const KeyRange begin = r.part(0, shift), end = r.part(most, shift);
    return most < (uint32_t)BINS && begin.first == r.first && (most == 0 || r.part(most - 1, shift).last == end.first - 1) && end.first <= end.last && end.last == r.last;
}
static_assert(parts_cover({~1u, ~0u}) && parts_cover({~4097u, ~0u}) && parts_cover({~50257u, ~0u}) && parts_cover({~131072u, ~0u}) &&
              parts_cover({~(1u << 24), ~0u}) && parts_cover({0u, ~0u}) && parts_cover({7u, 7u}) && parts_cover({0x007fffffu, 0xff800000u}), "parts of a key range");

// 11 bits of a search: the part of [*lo, *hi] in which the running sum of the weights, by descending key and from *above,
// reaches target (false: it does not; nothing changes).  each calls f(key, weight), weight a function.
template <int NT, class Each>
__device__ __forceinline__ bool narrow_step(SampleShared& sh, Each&& each, uint32_t* lo, uint32_t* hi, u64* above, u64 target) {
    const KeyRange range{*lo, *hi};
    const int shift = max(21 - __clz(range.last - range.first), 0);            // part_shift() at once: 21 = 32 - log2 BINS
    clear_bins<NT>(sh);
    each([&](uint32_t key, auto&& weight) {
        if (key < range.first || key > range.last) return;
        const u64 v = weight();
        if (v) atomicAdd(&sh.bin[(key - range.first) >> shift], v);
    });
    find_bin<NT>(sh, *above, target, true);
    if (sh.found == BINS) return false;
    const KeyRange part = range.part(BINS - 1 - sh.found, shift);
    *above = sh.found_sum;
    *lo = part.first;
    *hi = part.last;
    return true;
}
// The key among those of each(f) in [lo, hi] at which the running sum of the weights, by descending key and from `above`,
// reaches target (0 < target; where it is not reached: lo); *sum_above = the sum before it.  What a step leaves is settled at
// once by a wave that compares all pairs, if it is few.
template <int NT, class Each>
__device__ __forceinline__ uint32_t narrow(SampleShared& sh, Each&& each, uint32_t lo, uint32_t hi, u64 above, u64 target, u64* sum_above) {
    while (lo < hi && narrow_step<NT>(sh, each, &lo, &hi, &above, target) && lo < hi) {
        if (threadIdx.x == 0) sh.few = 0;
        __syncthreads();
        each([&](uint32_t key, auto&& weight) {
            if (key < lo || key > hi) return;
            const u64 v = weight();
            if (!v) return;
            const uint32_t i = atomicAdd(&sh.few, 1u);
            if (i < 64) { sh.few_key[i] = key; sh.few_w[i] = v; }
        });
        __syncthreads();
        const uint32_t few = sh.few;
        if (few <= 64) {
            if (threadIdx.x < few) {
                const uint32_t key = sh.few_key[threadIdx.x];
                u64 before = above, upto = above;
                for (uint32_t j = 0; j < few; ++j) {
                    const u64 v = sh.few_w[j];
                    if (sh.few_key[j] > key) before += v;
                    if (sh.few_key[j] >= key) upto += v;
                }
                if (before < target && upto >= target) {         // equal keys write the same
                    sh.found = key;
                    sh.found_sum = before;
                }
            }
            __syncthreads();
            lo = sh.found;
            above = sh.found_sum;
            break;
        }
    }
    *sum_above = above;
    return lo;
}
__device__ __forceinline__ u64 one_each() { return 1; }
// A bound that no fewer than k of the scores of each(f) reach, and few more: the lower end of the part in which the k-th
// largest lies.  lowest, best: their range.  LOWEST where there are fewer than k.
template <int NT, class Each> __device__ __forceinline__ float bound_of(SampleShared& sh, Each&& each, float lowest, float best, int k) {
    uint32_t lo = pattern(lowest), hi = pattern(best);
    u64 above = 0;
    if (!narrow_step<NT>(sh, each, &lo, &hi, &above, (u64)k)) return LOWEST;
    if (hi - lo >= 1u << 16) narrow_step<NT>(sh, each, &lo, &hi, &above, (u64)k);        // a range around zero holds most patterns
    return score_of(lo);
}
// lanes with `want` add to the list; the number of all that wanted is in sh.listed
__device__ __forceinline__ void append(SampleShared& sh, bool want, float z, uint32_t at) {
    const unsigned long long m = __ballot(want);
    if (!m) return;
    const int lane = threadIdx.x & 63;
    uint32_t from = 0;
    if (lane == 0) from = atomicAdd(&sh.listed, (uint32_t)__popcll(m));
    from = (uint32_t)__builtin_amdgcn_readfirstlane((int)from) + (uint32_t)__popcll(m & ((1ull << lane) - 1));
    if (want && from < LIST_MAX) {
        sh.list_z[from] = z;
        sh.list_at[from] = at;
    }
}
// smallest and largest over the block, of values that are not NaN
template <int CTRL, int ROWS> __device__ __forceinline__ float moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
template <int NT> __device__ __forceinline__ void block_range(SampleShared& sh, float& lowest, float& best) {
#define VDB_RANGE_STEP(CTRL, ROWS) { best = fmaxf(best, moved<CTRL, ROWS>(best)); lowest = fminf(lowest, moved<CTRL, ROWS>(lowest)); }
    VDB_RANGE_STEP(0x111, 0xf) VDB_RANGE_STEP(0x112, 0xf) VDB_RANGE_STEP(0x114, 0xf) VDB_RANGE_STEP(0x118, 0xf)      // as wave_scan
    VDB_RANGE_STEP(0x142, 0xa) VDB_RANGE_STEP(0x143, 0xc)
#undef VDB_RANGE_STEP
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.red[threadIdx.x >> 6] = ((u64)__float_as_uint(lowest) << 32) | __float_as_uint(best);
    __syncthreads();
    best = -INFINITY;
    lowest = INFINITY;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const u64 r = sh.red[w];
        best = fmaxf(best, __uint_as_float((uint32_t)r));
        lowest = fminf(lowest, __uint_as_float((uint32_t)(r >> 32)));
    }
}

// The log-probability of score z comes from the score: a weight near the cut holds few bits (ten of 2^-35 at 131072 scores).
__device__ __forceinline__ void write_draw(const SampleArgs& a, int64_t row, uint32_t at, float z, float tau, const FixedExp& weigh, u64 total) {
    a.out_row[row] = at;
    if (a.out_logp) a.out_logp[row] = (float)(((double)z - weigh.best) / (double)tau - log((double)total / (double)((u64)1 << a.shift)));
}
__device__ __forceinline__ void write_certain(const SampleArgs& a, int64_t row, int64_t at) {
    a.out_row[row] = at;
    if (a.out_logp) a.out_logp[row] = at < 0 ? -INFINITY : 0.0f;
}
// how many rows at a cut remain whose weights before it are `above`: those with less than target before them
__device__ __forceinline__ int64_t ties_within(double target, u64 above, u64 w) {
    return max((int64_t)1, (int64_t)ceil((target - (double)above) / (double)w));
}

// Of the rows at a cut, each(f) calling f(row), the first `ties` remain: the first one that is out (or 2^32 - 1).
template <int NT, class Each> __device__ __forceinline__ uint32_t first_tie_out(SampleShared& sh, Each&& each, int64_t ties, uint32_t vocab) {
    if (ties == INT64_MAX) return 0xffffffffu;
    u64 count = 0, ignored;
    each([&](uint32_t) { ++count; });
    if ((int64_t)block_total<NT>(sh, count) <= ties) return 0xffffffffu;
    return ~narrow<NT>(sh, [&](auto&& f) { each([&](uint32_t at) { f(~at, one_each); }); }, ~vocab, 0xffffffffu, 0, (u64)ties + 1, &ignored);
}

// ---------------------------------------------------------------- the draw from a list
// `listed` <= LIST_MAX scores and their rows in sh.list_*, in any order, among them all that remain.
template <int NT> __device__ __forceinline__ void draw_listed(SampleShared& sh, const SampleArgs& a, int64_t row, const Settings& set, const FixedExp& weigh, int listed) {
    constexpr int LIST_ITEMS = LIST_MAX / NT;
    const int tid = threadIdx.x;
    const u64 least_w = set.least_weight(a.shift);
    if (listed <= PAIRS) {
        // every item's rank, the weights ranked before it, and, once it is known what remains, those of lower rows: by
        // comparing all pairs, the block's threads in slices of the list
        int log_width = 6;
        while ((1 << log_width) < listed) ++log_width;
        const int i = tid & ((1 << log_width) - 1), slice = tid >> log_width, slices = NT >> log_width;
        const float zi = i < listed ? sh.list_z[i] : 0.0f;
        const uint32_t at = i < listed ? sh.list_at[i] : 0;
        u64 w = 0;
        if (tid < listed) w = weigh.directly(zi);
        if (tid < PAIRS) { sh.pair_rank[tid] = 0; sh.pair_sum[tid] = 0; sh.pair_w[tid] = w; }
        __syncthreads();
        if (i < listed) {
            uint32_t rank = 0;
            u64 before = 0;
            for (int j = slice; j < listed; j += slices) {
                const float zj = sh.list_z[j];
                if (zj > zi || (zj == zi && sh.list_at[j] < at)) {
                    ++rank;
                    before += sh.pair_w[j];
                }
            }
            if (rank) {
                atomicAdd(&sh.pair_rank[i], rank);
                atomicAdd(&sh.pair_sum[i], before);
            }
        }
        __syncthreads();
        if (set.by_count() && tid < listed && sh.pair_rank[tid] >= (uint32_t)set.top_k) w = 0;
        if (set.by_mass()) {
            const double target = (double)block_total<NT>(sh, w) * (double)set.top_p;
            if (tid < listed && sh.pair_rank[tid] > 0 && !((double)sh.pair_sum[tid] < target)) w = 0;
        }
        if (w < least_w) w = 0;
        __syncthreads();
        if (tid < PAIRS) { sh.pair_w[tid] = w; sh.pair_sum[tid] = 0; }
        const u64 all = block_total<NT>(sh, w), least = set.goal(all);
        if (i < listed) {
            u64 before = 0;
            for (int j = slice; j < listed; j += slices)
                if (sh.list_at[j] < at) before += sh.pair_w[j];
            if (before) atomicAdd(&sh.pair_sum[i], before);
        }
        __syncthreads();
        if (tid < listed && w && sh.pair_sum[tid] < least && sh.pair_sum[tid] + w >= least) write_draw(a, row, at, zi, set.tau, weigh, all);
        return;
    }
    make_table<NT>(sh.table);
    __syncthreads();
    u64 w[LIST_ITEMS];
    float z[LIST_ITEMS];
    uint32_t at[LIST_ITEMS];
#pragma unroll
    for (int q = 0; q < LIST_ITEMS; ++q) {
        const int i = q * NT + tid;
        z[q] = i < listed ? sh.list_z[i] : -INFINITY;
        at[q] = i < listed ? sh.list_at[i] : 0;
        w[q] = weigh(z[q]);
    }
    float cut = -INFINITY;
    int64_t ties = INT64_MAX;
    float lowest = INFINITY, best = -INFINITY;
#pragma unroll
    for (int q = 0; q < LIST_ITEMS; ++q) {
        best = fmaxf(best, z[q]);
        if (z[q] > -INFINITY) lowest = fminf(lowest, z[q]);
    }
    block_range<NT>(sh, lowest, best);
    const uint32_t bottom = pattern(lowest), top = pattern(best);
    if (set.by_count() && set.top_k < listed) {
        u64 above;
        cut = score_of(narrow<NT>(sh, [&](auto&& f) {
#pragma unroll
            for (int q = 0; q < LIST_ITEMS; ++q) f(pattern(z[q]), one_each);
        }, bottom, top, 0, (u64)set.top_k, &above));
        ties = set.top_k - (int64_t)above;
    }
    if (set.by_mass()) {
        u64 sum = 0;
#pragma unroll
        for (int q = 0; q < LIST_ITEMS; ++q) sum += z[q] > cut ? w[q] : 0;
        const u64 over = block_total<NT>(sh, sum), w_cut = ties < INT64_MAX ? weigh(cut) : 0;
        const double target = (double)(over + w_cut * (u64)(ties < INT64_MAX ? ties : 0)) * (double)set.top_p;
        const u64 least = max((u64)ceil(target), (u64)1);
        if (over >= least) {
            u64 above;
            const float floor_z = cut;
            cut = score_of(narrow<NT>(sh, [&](auto&& f) {
#pragma unroll
                for (int q = 0; q < LIST_ITEMS; ++q)
                    if (z[q] > floor_z) f(pattern(z[q]), [&] { return w[q]; });
            }, bottom, top, 0, least, &above));
            ties = ties_within(target, above, weigh(cut));
        } else if (w_cut) {
            ties = min(ties, ties_within(target, over, w_cut));
        }
    }
    const uint32_t tie_end = first_tie_out<NT>(sh, [&](auto&& f) {
#pragma unroll
        for (int q = 0; q < LIST_ITEMS; ++q)
            if (z[q] == cut) f(at[q]);
    }, ties, (uint32_t)a.vocab);
    u64 sum = 0;
#pragma unroll
    for (int q = 0; q < LIST_ITEMS; ++q) {
        if (!(z[q] > cut || (z[q] == cut && at[q] < tie_end)) || w[q] < least_w) w[q] = 0;
        sum += w[q];
    }
    const u64 all = block_total<NT>(sh, sum);
    u64 before;
    // the row, from the first, at which the running sum reaches the goal
    const uint32_t drawn = ~narrow<NT>(sh, [&](auto&& f) {
#pragma unroll
        for (int q = 0; q < LIST_ITEMS; ++q)
            if (w[q]) f(~at[q], [&] { return w[q]; });
    }, ~(uint32_t)a.vocab, 0xffffffffu, 0, set.goal(all), &before);
#pragma unroll
    for (int q = 0; q < LIST_ITEMS; ++q)
        if (w[q] && at[q] == drawn) write_draw(a, row, drawn, z[q], set.tau, weigh, all);
}

// ---------------------------------------------------------------- a row by one block
// Pieces of a loop, AHEAD loads in flight while the ones before are worked on: f(step, first element, piece) for steps
// [from, to), `at(step)` the first element of this lane's piece; `prologue` runs while the first loads are under way.  A step is
// kept apart from the next (sched_barrier): the compiler would interleave them and run out of registers.
template <class T, class At, class F, class P>
__device__ __forceinline__ void stream_pieces(const Source<T>& src, int from, int to, At&& at, F&& f, P&& prologue) {
    Piece<T> next[AHEAD];
    uint32_t bits[AHEAD];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = t0 + j < to ? at(t0 + j) : src.vocab;
            next[j] = src.load(i);
            bits[j] = src.bits(i);
        }
    };
    fetch(from);
    prologue();
#pragma unroll 1
    for (int t0 = from; t0 < to; t0 += AHEAD) {
        Piece<T> now[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            now[j] = next[j];
            src.finish(now[j], bits[j]);
        }
        if (t0 + AHEAD < to) fetch(t0 + AHEAD);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            if (t0 + j < to) f(t0 + j, at(t0 + j), now[j]);
        }
    }
}

template <class T> struct RowPasses {
    static constexpr int N = Piece<T>::N;
    Source<T> src;
    int tid, lane, wave;
    // the parts of the row: a wave's contiguous share in up to GROUPS groups of `per_group` steps of 64 pieces
    int steps, per_group, groups, parts, share;
    __device__ __forceinline__ RowPasses(const Source<T>& s)
        : src(s), tid(threadIdx.x), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
        steps = ((src.vocab + ROW_WAVES - 1) / ROW_WAVES + 64 * N - 1) / (64 * N);
        per_group = (steps + GROUPS - 1) / GROUPS;
        groups = (steps + per_group - 1) / per_group;
        parts = ROW_WAVES * groups;
        share = steps * 64 * N;
    }
    // every score, in no order: f(z)
    template <class F> __device__ __forceinline__ void each(F&& f) const {
        stream_pieces(src, 0, (src.vocab + ROW_NT * N - 1) / (ROW_NT * N), [&](int t) { return (t * ROW_NT + tid) * N; },
                      [&](int, int, const Piece<T>& v) {
#pragma unroll
                          for (int e = 0; e < N; ++e) f(v.get(e));
                      }, [] {});
    }
    // the steps [from, to) of the wave's share, in order: f(step, first element, piece)
    template <class F> __device__ __forceinline__ void in_order(int from, int to, F&& f) const {
        stream_pieces(src, from, to, [&](int t) { return wave * share + (t * 64 + lane) * N; }, f, [] {});
    }
    // sh.part = the running sums of value(piece, first element) before each part; -> their sum
    template <class Value> __device__ __forceinline__ u64 sum_parts(SampleShared& sh, Value&& value) const {
        __syncthreads();
        u64 sum = 0;
        in_order(0, steps, [&](int t, int at, const Piece<T>& v) {
            sum += value(v, at);
            if ((t + 1) % per_group == 0 || t + 1 == steps) {
                sum = wave_sum(sum);
                if (lane == 0) sh.part[wave * groups + t / per_group] = sum;
                sum = 0;
            }
        });
        return scan_parts<ROW_NT>(sh, parts);
    }
    // the parts of the wave that hold(sum before, sum up to): f(sum before, group)
    template <class Hold, class F> __device__ __forceinline__ void parts_that(const SampleShared& sh, u64 total, Hold&& hold, F&& f) const {
        for (int g = 0; g < groups; ++g) {
            const int k = wave * groups + g;
            const u64 from = sh.part[k], to = k + 1 < parts ? sh.part[k + 1] : total;
            if (hold(from, to)) f(from, g);
        }
    }
    // The scores at or above thr to the list; -> their number, of which the list holds LIST_MAX.
    __device__ __forceinline__ int compact(SampleShared& sh, float thr) const {
        __syncthreads();
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        stream_pieces(src, 0, (src.vocab + ROW_NT * N - 1) / (ROW_NT * N), [&](int t) { return (t * ROW_NT + tid) * N; },
                      [&](int, int at, const Piece<T>& v) {
                          float top = v.get(0);
#pragma unroll
                          for (int e = 1; e < N; ++e) top = fmaxf(top, v.get(e));
                          if (!__ballot(top >= thr)) return;
#pragma unroll
                          for (int e = 0; e < N; ++e) append(sh, v.get(e) >= thr, v.get(e), (uint32_t)(at + e));
                      }, [] {});
        __syncthreads();
        return (int)sh.listed;
    }
};

template <class T> __device__ __forceinline__ void sample_whole_row(SampleShared& sh, const T* scores, const SampleArgs& a, int64_t row) {
    constexpr int N = Piece<T>::N;
    RowPasses<T> pass(Source<T>(scores, a, row));
    const int tid = threadIdx.x;
    const Settings set(a, row);
    // ---- the largest score of each thread, and of the row
    float mine = -INFINITY;
    pass.each([&](float z) { mine = fmaxf(mine, z); });
    float best = mine, lowest = mine > -INFINITY ? mine : INFINITY;
    if (tid == 0) sh.first = 0xffffffffu;
    block_range<ROW_NT>(sh, lowest, best);
    if (best == -INFINITY) {
        if (tid == 0) write_certain(a, row, -1);
        return;
    }
    if (set.first_of_best()) {
        uint32_t at = 0xffffffffu;
        if (mine == best) {
#pragma unroll 1
            for (int i = tid * N; i < pass.src.vocab && at == 0xffffffffu; i += ROW_NT * N) {
                Piece<T> v = pass.src.load(i);
                pass.src.finish(v, pass.src.bits(i));
#pragma unroll
                for (int e = N - 1; e >= 0; --e)
                    if (v.get(e) == best) at = (uint32_t)(i + e);
            }
            atomicMin(&sh.first, at);
        }
        __syncthreads();
        if (tid == 0) write_certain(a, row, sh.first);
        return;
    }
    if (best == INFINITY) {
        pass.src.infinite = true;
        mine = mine == INFINITY ? 0.0f : -INFINITY;
        best = lowest = 0.0f;
    }
    const FixedExp weigh(best, set.tau, a.shift, sh.table);
    const u64 least_w = set.least_weight(a.shift);

    // ---- few rows can remain: a list of them
    float thr = -INFINITY;
    if (set.by_count() && set.top_k <= ROW_NT) {
        thr = bound_of<ROW_NT>(sh, [&](auto&& f) { f(pattern(mine), one_each); }, lowest, best, set.top_k);
    } else if (!set.by_count() && !set.by_mass() && least_w) {
        thr = set.min_p_bound(best);
    }
    if (thr > -INFINITY) {
        const int listed = pass.compact(sh, thr);
        if (listed <= LIST_MAX) {
            if (tid >= FEW_NT) return;                           // barriers wait for the waves that have not ended
            return draw_listed<FEW_NT>(sh, a, row, set, weigh, listed);
        }
    }
    make_table<ROW_NT>(sh.table);                        // the next barrier is clear_bins' or sum_parts'

    // ---- the lowest score that remains (cut), and how many of the rows at it
    float cut = -INFINITY;
    int64_t ties = INT64_MAX;
    // The score, from the best, at which the running sum of value(z) reaches target(total); false where scores that weigh
    // anything do not reach it.
    auto find_cut = [&](auto&& value, auto&& target, float* at, u64* above) {
        clear_bins<ROW_NT>(sh);
        u64 sum = 0;
        pass.each([&](float z) {
            if (z >= weigh.cut) {
                const u64 v = value(z);
                sum += v;
                if (v) atomicAdd(&sh.bin[weigh.bin(z)], v);
            }
        });
        const u64 least = target(block_total<ROW_NT>(sh, sum));
        find_bin<ROW_NT>(sh, 0, least, false);
        const int b = (int)sh.found;
        if (b == BINS) return false;
        const u64 before = sh.found_sum;
        float lo, hi;
        weigh.bin_range(b, &lo, &hi);
        // the bin's scores go to the list, where they fit; else they are picked out of the row again in each step
        __syncthreads();
        if (tid == 0) sh.found = 0;
        __syncthreads();
        pass.each([&](float z) {
            if (z < lo || z > hi || !(z >= weigh.cut) || weigh.bin(z) != b) return;
            const uint32_t to = atomicAdd(&sh.found, 1u);
            if (to < LIST_MAX) sh.list_z[to] = z;
        });
        __syncthreads();
        const int members = (int)sh.found;
        __syncthreads();
        *at = score_of(narrow<ROW_NT>(sh, [&](auto&& f) {
            if (members <= LIST_MAX) {
                for (int i = tid; i < members; i += ROW_NT) {
                    const float z = sh.list_z[i];
                    f(pattern(z), [&] { return value(z); });
                }
            } else {
                pass.each([&](float z) {
                    if (z >= lo && z <= hi && z >= weigh.cut && weigh.bin(z) == b) f(pattern(z), [&] { return value(z); });
                });
            }
        }, pattern(lo), pattern(hi), before, least, above));
        return true;
    };
    if (set.by_count()) {
        u64 above;
        float at;
        if (find_cut([](float) { return (u64)1; }, [&](u64) { return (u64)set.top_k; }, &at, &above)) {
            cut = at;
            ties = set.top_k - (int64_t)above;
        }
    }
    if (set.by_mass()) {
        const float floor_z = cut;
        const u64 w_cut = ties < INT64_MAX ? weigh(cut) : 0;
        u64 above = 0, over = 0;
        float at = 0.0f;
        double target = 0.0;
        if (find_cut([&](float z) { return z > floor_z ? weigh(z) : (u64)0; },
                     [&](u64 total) {
                         over = total;
                         target = (double)(total + w_cut * (u64)(ties < INT64_MAX ? ties : 0)) * (double)set.top_p;
                         return max((u64)ceil(target), (u64)1);
                     },
                     &at, &above)) {
            cut = at;
            ties = ties_within(target, above, weigh(at));
        } else if (w_cut) {
            ties = min(ties, ties_within(target, over, w_cut));
        }
    }

    // ---- the draw
    __syncthreads();
    if (tid == 0) sh.first = 0xffffffffu;             // rows at the cut from this one on are out
    if (ties < INT64_MAX) {
        auto ties_in = [&](const Piece<T>& v) {
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) c += v.get(e) == cut ? 1 : 0;
            return c;
        };
        const u64 total = pass.sum_parts(sh, [&](const Piece<T>& v, int) { return (u64)ties_in(v); });
        pass.parts_that(sh, total, [&](u64 from, u64 to) { return (int64_t)from <= ties && (int64_t)to > ties; }, [&](u64 before, int g) {
            int64_t run = (int64_t)before;
            pass.in_order(g * pass.per_group, min((g + 1) * pass.per_group, pass.steps), [&](int, int at, const Piece<T>& v) {
                const uint32_t c = ties_in(v);
                const u64 inc = wave_scan(c);
                int64_t k = run + (int64_t)inc - c;
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (v.get(e) == cut) {
                        if (k == ties) sh.first = (uint32_t)(at + e);
                        ++k;
                    }
                run += (int64_t)last_lane(inc);
            });
        });
    }
    __syncthreads();
    const uint32_t tie_end = sh.first;
    auto weight_at = [&](float z, uint32_t at) {
        const u64 w = weigh(z);
        return (z > cut || (z == cut && at < tie_end)) && w >= least_w ? w : (u64)0;
    };
    const u64 total = pass.sum_parts(sh, [&](const Piece<T>& v, int at) {
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) sum += weight_at(v.get(e), (uint32_t)(at + e));
        return sum;
    });
    const u64 least = set.goal(total);
    pass.parts_that(sh, total, [&](u64 from, u64 to) { return from < least && to >= least; }, [&](u64 before, int g) {
        u64 run = before;
        pass.in_order(g * pass.per_group, min((g + 1) * pass.per_group, pass.steps), [&](int, int at, const Piece<T>& v) {
            u64 w[N], sum = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) sum += w[e] = weight_at(v.get(e), (uint32_t)(at + e));
            const u64 inc = wave_scan(sum);
            u64 k = run + inc - sum;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (k < least && k + w[e] >= least) write_draw(a, row, (uint32_t)(at + e), v.get(e), set.tau, weigh, total);
                k += w[e];
            }
            run += last_lane(inc);
        });
    });
}

template <class T> __global__ void __launch_bounds__(ROW_NT) sample_kernel(const T* __restrict__ scores, SampleArgs a) {
    __shared__ SampleShared sh;
    sample_whole_row(sh, scores, a, blockIdx.x);
}

// ---------------------------------------------------------------- long rows, by the whole chip
// 1 sample_groups: the maxima of groups of 32 scores and of the blocks' slices (and the histograms cleared)
// 2 sample_pick: a block per row finishes the rows that the best score or a list settles, from the maxima and the few groups
//   that reach the bound, and marks the others; beside them, where settings ask for it, blocks of their own take the weights,
//   by parts of the row, and by distance from the best where top-p asks for it
// 3 sample_border (a block per row): the draw from the parts, or the bin in which the border of top-p lies
// 4 sample_above: the weights above that bin by parts, and the bin's members
// 5 sample_rest (a block per row): the border among the members and the draw; rows for which a list was too short go through
//   all passes by one block
static constexpr int GROUP = 32, STREAM_NT = 256, STREAM_PIECES = 4;
enum RowMode { ROW_DONE = 0, ROW_WHOLE = 1, ROW_SUM = 2, ROW_MASS = 3, ROW_LIST = 4 };
struct RowState {
    u64 above, least;                // weights above the bin of the border; the running sum that the border reaches
    double target;
    float best;
    int mode, bin;
    uint32_t members;
};
static constexpr int PARTS = ROW_WAVES * GROUPS;                 // at most, per row
static constexpr int WEIGH_PARTS = 4 * (FEW_NT / 64), ABOVE_PARTS = 4 * (STREAM_NT / 64);             // parts of a streaming block: four a wave
struct SampleWork {
    float* group_max; int groups;    // [n][groups]
    float* slice_max; int slices;    // [n][slices], slices as of fp32 rows at most
    RowState* state;                 // [n]
    u64* hist;                       // [n][BINS]
    u64* part; int parts, part_len;    // [n][PARTS], scores of a part (a multiple of 512)
    float* member_z; uint32_t* member_at;           // [n][LIST_MAX]
    int64_t bytes;
};
static SampleWork sample_work(void* base, int64_t n, int64_t vocab) {
    SampleWork w{};
    char* at = (char*)base;
    auto take = [&](int64_t bytes) {
        char* here = at;
        at += round_up64(bytes, 256);
        return here;
    };
    w.groups = (int)((vocab + GROUP - 1) / GROUP);
    w.part_len = (int)round_up64((vocab + PARTS - 1) / PARTS, 512);
    w.parts = (int)((vocab + w.part_len - 1) / w.part_len);
    w.group_max = (float*)take(n * w.groups * 4);
    w.slices = ceil_div(vocab, STREAM_NT * Piece<float>::N * STREAM_PIECES);
    w.slice_max = (float*)take(n * w.slices * 4);
    w.state = (RowState*)take(n * sizeof(RowState));
    w.hist = (u64*)take(n * BINS * 8);
    w.part = (u64*)take(n * PARTS * 8);
    w.member_z = (float*)take(n * LIST_MAX * 4);
    w.member_at = (uint32_t*)take(n * LIST_MAX * 4);
    w.bytes = at - (char*)base;
    return w;
}
// What a row's settings make of it, before its scores are seen.  Min-p alone mostly leaves few rows where it is 1/64 or more.
__host__ __device__ static inline RowMode mode_of(float tau, int top_k, float top_p, float min_p) {
    if (!(tau > 0.0f) || top_k == 1 || top_p <= 0.0f) return ROW_LIST;
    if (top_k > 1) return top_k <= LIST_MAX / 2 ? ROW_LIST : ROW_WHOLE;
    if (top_p < 1.0f) return ROW_MASS;
    return min_p >= 0.015625f ? ROW_LIST : ROW_SUM;
}

template <class T>
__global__ void __launch_bounds__(STREAM_NT) sample_groups_kernel(const T* __restrict__ scores, SampleArgs a, SampleWork w, int slices) {
    constexpr int N = Piece<T>::N;
    const int64_t row = blockIdx.x / slices;
    const int slice = (int)(blockIdx.x - row * slices);
    const Source<T> src(scores, a, row);
    Piece<T> x[STREAM_PIECES];
    uint32_t bits[STREAM_PIECES];
    const int first = (slice * STREAM_PIECES * STREAM_NT + (int)threadIdx.x) * N;
#pragma unroll
    for (int j = 0; j < STREAM_PIECES; ++j) {
        x[j] = src.load(first + j * STREAM_NT * N);
        bits[j] = src.bits(first + j * STREAM_NT * N);
    }
    for (int b = slice * STREAM_NT + threadIdx.x; b < BINS; b += slices * STREAM_NT) w.hist[row * BINS + b] = 0;
    if (slice == 0 && threadIdx.x == 0) w.state[row] = RowState{};
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < STREAM_PIECES; ++j) {
        const int at = first + j * STREAM_NT * N;
        src.finish(x[j], bits[j]);
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, x[j].get(e));
        m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0xB1, 0xf, 0xf, false)));      // quad_perm:[1,0,3,2]
        m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x4E, 0xf, 0xf, false)));      // quad_perm:[2,3,0,1]
        if (N == 4) m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x141, 0xf, 0xf, false)));   // row_half_mirror
        if (threadIdx.x % (GROUP / N) == 0 && at < src.vocab) w.group_max[row * w.groups + at / GROUP] = m;
        top = fmaxf(top, m);
    }
    __shared__ float tops[STREAM_NT / 64];
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < STREAM_NT / 64; ++i) top = fmaxf(top, tops[i]);
        w.slice_max[row * w.slices + slice] = top;
    }
}

// A row's group maxima, every FEW_NT-th of them a thread's: the first HELD in registers (rows of up to 131072 scores), the
// others read again in each pass.
struct GroupMaxima {
    static constexpr int HELD = 4096 / FEW_NT;
    const float* max;
    int groups;
    float held[HELD];
    __device__ __forceinline__ GroupMaxima(const SampleWork& work, int64_t row) : max(work.group_max + row * work.groups), groups(work.groups) {
#pragma unroll
        for (int q = 0; q < HELD; ++q) held[q] = q * FEW_NT + (int)threadIdx.x < groups ? max[q * FEW_NT + threadIdx.x] : -INFINITY;
    }
    // f(group, maximum)
    template <class F> __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
        for (int q = 0; q < HELD; ++q) f(q * FEW_NT + (int)threadIdx.x, held[q]);
        for (int g = HELD * FEW_NT + threadIdx.x; g < groups; g += FEW_NT) f(g, max[g]);
    }
};

template <class T> __device__ __forceinline__ void sample_pick(SampleShared& sh, const T* scores, const SampleArgs& a, const SampleWork& work, int64_t row) {
    const Source<T> src(scores, a, row);
    const Settings set(a, row);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const GroupMaxima groups(work, row);
    float best = -INFINITY, lowest = INFINITY;
    groups.each([&](int, float m) {
        best = fmaxf(best, m);
        if (m > -INFINITY) lowest = fminf(lowest, m);
    });
    const float mine = best;
    if (tid == 0) { sh.first = 0xffffffffu; sh.listed = sh.found = 0; }
    block_range<FEW_NT>(sh, lowest, best);
    if (best == -INFINITY) {
        if (tid == 0) write_certain(a, row, -1);
        return;
    }
    if (set.first_of_best()) {
        if (mine == best) {
            uint32_t first = 0xffffffffu;
            groups.each([&](int g, float m) { if (m == best) first = min(first, (uint32_t)g); });
            atomicMin(&sh.first, first);
        }
        __syncthreads();
        if (tid < GROUP) {
            const int at = (int)sh.first * GROUP + tid;
            const unsigned long long m = __ballot(src.one(at) == best);
            if (tid == 0) write_certain(a, row, (int64_t)sh.first * GROUP + __builtin_ctzll(m));
        }
        return;
    }
    const int mode = best == INFINITY ? ROW_WHOLE : mode_of(set.tau, set.top_k, set.top_p, set.min_p);
    if (mode == ROW_LIST) {
        const FixedExp weigh(best, set.tau, a.shift, sh.table);
        const float thr = !set.by_count() ? set.min_p_bound(best) : bound_of<FEW_NT>(sh, [&](auto&& f) {
            groups.each([&](int, float m) { f(pattern(m), one_each); });
        }, lowest, best, set.top_k);
        // the groups that reach the bound, and their scores that do
        uint32_t* group = (uint32_t*)sh.bin;
        __syncthreads();
        if (tid == 0) sh.found = 0;
        __syncthreads();
        groups.each([&](int g, float m) {
            if (!(m >= thr)) return;
            const uint32_t i = atomicAdd(&sh.found, 1u);
            if (i < LIST_MAX) group[i] = (uint32_t)g;
        });
        __syncthreads();
        const int found = (int)sh.found;
        if (found <= LIST_MAX) {
            // a piece a lane, two at a time: GROUP / N lanes a group
            constexpr int N = Piece<T>::N, LANES = GROUP / N, WAVE = 64 / LANES;
            for (int k0 = wave * WAVE + lane / LANES; k0 - lane / LANES < found; k0 += 2 * WAVE * (FEW_NT / 64)) {
                const int k1 = k0 + WAVE * (FEW_NT / 64);
                const int at0 = k0 < found ? (int)group[k0] * GROUP + (lane % LANES) * N : src.vocab;
                const int at1 = k1 < found ? (int)group[k1] * GROUP + (lane % LANES) * N : src.vocab;
                Piece<T> x0 = src.load(at0), x1 = src.load(at1);
                src.finish(x0, src.bits(at0));
                src.finish(x1, src.bits(at1));
#pragma unroll
                for (int e = 0; e < N; ++e) append(sh, x0.get(e) >= thr, x0.get(e), (uint32_t)(at0 + e));
#pragma unroll
                for (int e = 0; e < N; ++e) append(sh, x1.get(e) >= thr, x1.get(e), (uint32_t)(at1 + e));
            }
            __syncthreads();
            const int listed = (int)sh.listed;
            __syncthreads();
            if (listed <= LIST_MAX) return draw_listed<FEW_NT>(sh, a, row, set, weigh, listed);
        }
    }
    if (tid == 0) {
        work.state[row].best = best;
        work.state[row].mode = mode == ROW_LIST ? ROW_WHOLE : mode;
    }
}

// The parts of a row from p0 on, four a wave: out[part] = the sum of f(piece, first element)
template <class T, class F, class P>
__device__ __forceinline__ void stream_parts(const Source<T>& src, const SampleWork& work, int p0, u64* out, F&& f, P&& prologue) {
    constexpr int N = Piece<T>::N, EACH = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = p0 + EACH * wave, end = min(first + EACH, work.parts), steps = work.part_len / (64 * N);
    u64 sum = 0;
    stream_pieces(src, 0, max(end - first, 0) * steps, [&](int t) { return first * work.part_len + (t * 64 + lane) * N; },
                  [&](int t, int at, const Piece<T>& v) {
                      sum += f(v, at);
                      if ((t + 1) % steps) return;
                      sum = wave_sum(sum);
                      if (lane == 0) out[first + t / steps] = sum;
                      sum = 0;
                  }, prologue);
}
// A row's weights by parts, and by distance from the best where top-p asks for it.
template <class T>
__device__ __forceinline__ void sample_weigh(SampleShared& sh, const T* __restrict__ scores, const SampleArgs& a, const SampleWork& work, int64_t row, int cut,
                                             int slices) {
    constexpr int N = Piece<T>::N;
    const Settings set(a, row);
    const int mode = mode_of(set.tau, set.top_k, set.top_p, set.min_p);
    if (mode != ROW_SUM && mode != ROW_MASS) return;
    float best = -INFINITY;
    for (int i = threadIdx.x & 63; i < slices; i += 64) best = fmaxf(best, work.slice_max[row * work.slices + i]);
    best = wave_max(best);
    if (!(fabsf(best) < INFINITY)) return;
    const Source<T> src(scores, a, row);
    const FixedExp weigh(best, set.tau, a.shift, sh.table);
    const u64 least_w = mode == ROW_SUM ? set.least_weight(a.shift) : 0;
    stream_parts(src, work, cut * WEIGH_PARTS, work.part + row * PARTS, [&](const Piece<T>& v, int) {
        u64 w[N], sum = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = weigh(v.get(e));
        if (mode == ROW_MASS) {
            // no branch between the scores: their chains of dependent steps overlap
#pragma unroll
            for (int e = 0; e < N; ++e) atomicAdd(&sh.bin[weigh.bin(v.get(e))], w[e]);
        } else if (least_w) {
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = w[e] >= least_w ? w[e] : 0;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum += w[e];
        return sum;
    }, [&] {
        make_table<FEW_NT>(sh.table);
        if (mode == ROW_MASS)
            for (int b = threadIdx.x; b < BINS; b += FEW_NT) sh.bin[b] = 0;
        __syncthreads();
    });
    if (mode != ROW_MASS) return;
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += FEW_NT)
        if (sh.bin[b]) atomicAdd(&work.hist[row * BINS + b], sh.bin[b]);
}

template <class T>
__global__ void __launch_bounds__(STREAM_NT) sample_above_kernel(const T* __restrict__ scores, SampleArgs a, SampleWork work, int cuts) {
    constexpr int N = Piece<T>::N;
    __shared__ double table[EXP_STEPS];
    __shared__ float member_z[LIST_MAX];
    __shared__ uint32_t member_at[LIST_MAX];
    __shared__ uint32_t members, base;
    const int64_t row = blockIdx.x / cuts;
    const int slice = (int)(blockIdx.x - row * cuts);
    RowState& state = work.state[row];
    if (state.mode != ROW_MASS) return;
    const float best = state.best;
    const int b = state.bin;
    const Source<T> src(scores, a, row);
    const Settings set(a, row);
    const FixedExp weigh(best, set.tau, a.shift, table);
    const u64 least_w = set.least_weight(a.shift);
    float lo, hi;
    weigh.bin_range(b, &lo, &hi);
    const float beyond = score_of(pattern(hi) + 1);              // the next larger score
    stream_parts(src, work, slice * ABOVE_PARTS, work.part + row * PARTS, [&](const Piece<T>& v, int at) {
        float top = v.get(0);
#pragma unroll
        for (int e = 1; e < N; ++e) top = fmaxf(top, v.get(e));
        u64 sum = 0;
        if (!__ballot(top >= lo)) return sum;
        u64 w[N];
        bool near = false;
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = weigh.from(v.get(e), beyond);
        if (least_w) {
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = w[e] >= least_w ? w[e] : 0;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            sum += w[e];
            near |= v.get(e) >= lo && v.get(e) <= hi;
        }
        if (near) {
            // the bin's own scores, and those beside it that the bin's range takes in
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float z = v.get(e);
                if (!(z >= lo && z <= hi)) continue;
                const int bin = weigh.bin(z);
                if (bin < b) {
                    const u64 w_e = weigh(z);
                    sum += w_e >= least_w ? w_e : 0;
                } else if (bin == b) {
                    const uint32_t to = atomicAdd(&members, 1u);
                    if (to < LIST_MAX) { member_z[to] = z; member_at[to] = (uint32_t)(at + e); }
                }
            }
        }
        return sum;
    }, [&] {
        make_table<STREAM_NT>(table);
        if (threadIdx.x == 0) members = 0;
        __syncthreads();
    });
    __syncthreads();
    const uint32_t mine = members;
    if (threadIdx.x == 0 && mine) base = atomicAdd(&state.members, mine);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < min(mine, (uint32_t)LIST_MAX); i += STREAM_NT) {
        const uint32_t to = base + i;
        if (to >= LIST_MAX) break;
        work.member_z[row * LIST_MAX + to] = member_z[i];
        work.member_at[row * LIST_MAX + to] = member_at[i];
    }
}

// Blocks below n: a row each.  The others, `cuts` a row: the weights of rows that ask for them.  A list takes one block as long
// as the weights take the chip (25 and 15 us), so both go side by side.
template <class T>
__global__ void __launch_bounds__(FEW_NT) sample_pick_kernel(const T* __restrict__ scores, SampleArgs a, SampleWork work, int n, int cuts, int slices) {
    __shared__ SampleShared sh;
    const int block = (int)blockIdx.x - n;
    if (block < 0) return sample_pick(sh, scores, a, work, blockIdx.x);
    sample_weigh(sh, scores, a, work, block / cuts, block % cuts, slices);
}

// The row's parts, of `total` after scan_parts: the one that holds the goal, read again by the first wave.
template <class T, class Weight>
__device__ __forceinline__ void draw_from_parts(SampleShared& sh, const Source<T>& src, const SampleArgs& a, const SampleWork& work, int64_t row,
                                                const Settings& set, const FixedExp& weigh, u64 total, Weight&& weight_at) {
    constexpr int N = Piece<T>::N;
    const int tid = threadIdx.x, lane = tid & 63;
    const u64 least = set.goal(total);
    for (int i = tid; i < work.parts; i += FEW_NT) {
        const u64 from = sh.part[i], to = i + 1 < work.parts ? sh.part[i + 1] : total;
        if (from < least && to >= least) {
            sh.found = (uint32_t)i;
            sh.found_sum = from;
        }
    }
    __syncthreads();
    if (tid >= 64) return;
    u64 run = sh.found_sum;
    const int start = (int)sh.found * work.part_len, end = start + work.part_len;
    for (int at0 = start; at0 < end && run < least; at0 += 64 * N) {
        const int at = at0 + lane * N;
        Piece<T> v = src.load(at);
        src.finish(v, src.bits(at));
        u64 w[N], sum = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) sum += w[e] = weight_at(v.get(e), (uint32_t)(at + e));
        const u64 inc = wave_scan(sum);
        u64 k = run + inc - sum;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (k < least && k + w[e] >= least) write_draw(a, row, (uint32_t)(at + e), v.get(e), set.tau, weigh, total);
            k += w[e];
        }
        run += last_lane(inc);
    }
}

template <class T> __global__ void __launch_bounds__(FEW_NT) sample_border_kernel(const T* __restrict__ scores, SampleArgs a, SampleWork work) {
    __shared__ SampleShared sh;
    const int64_t row = blockIdx.x;
    RowState& state = work.state[row];
    const int mode = state.mode, tid = threadIdx.x;
    if (mode != ROW_SUM && mode != ROW_MASS) return;
    const float best = state.best;
    const Settings set(a, row);
    u64 part = 0;
    for (int i = tid; i < work.parts; i += FEW_NT) part += sh.part[i] = work.part[row * PARTS + i];
    if (mode == ROW_MASS) {
        for (int b = tid; b < BINS; b += FEW_NT) sh.bin[b] = work.hist[row * BINS + b];
        const double target = (double)block_total<FEW_NT>(sh, part) * (double)set.top_p;
        const u64 least = max((u64)ceil(target), (u64)1);
        find_bin<FEW_NT>(sh, 0, least, false);
        if (tid == 0) {
            state.above = sh.found_sum;
            state.least = least;
            state.target = target;
            state.bin = (int)sh.found;
        }
        return;
    }
    make_table<FEW_NT>(sh.table);
    const u64 total = scan_parts<FEW_NT>(sh, work.parts), least_w = set.least_weight(a.shift);
    const FixedExp weigh(best, set.tau, a.shift, sh.table);
    draw_from_parts(sh, Source<T>(scores, a, row), a, work, row, set, weigh, total, [&](float z, uint32_t) {
        const u64 w = weigh(z);
        return w >= least_w ? w : (u64)0;
    });
}

template <class T> __global__ void __launch_bounds__(ROW_NT) sample_rest_kernel(const T* __restrict__ scores, SampleArgs a, SampleWork work) {
    __shared__ SampleShared sh;
    const int64_t row = blockIdx.x;
    const RowState state = work.state[row];
    const int tid = threadIdx.x;
    if (state.mode == ROW_WHOLE || (state.mode == ROW_MASS && state.members > LIST_MAX)) return sample_whole_row(sh, scores, a, row);
    if (state.mode != ROW_MASS || tid >= FEW_NT) return;         // barriers wait for the waves that have not ended
    const Settings set(a, row);
    const Source<T> src(scores, a, row);
    const int members = (int)state.members;
    for (int i = tid; i < work.parts; i += FEW_NT) sh.part[i] = work.part[row * PARTS + i];
    for (int i = tid; i < members; i += FEW_NT) {
        sh.list_z[i] = work.member_z[row * LIST_MAX + i];
        sh.list_at[i] = work.member_at[row * LIST_MAX + i];
    }
    make_table<FEW_NT>(sh.table);
    __syncthreads();
    const FixedExp weigh(state.best, set.tau, a.shift, sh.table);
    const u64 least_w = set.least_weight(a.shift);
    float cut = -INFINITY;
    uint32_t tie_end = 0xffffffffu;              // rows at the cut from this one on are out
    auto weight_at = [&](float z, uint32_t at) {
        const u64 w = weigh(z);
        return (z > cut || (z == cut && at < tie_end)) && w >= least_w ? w : (u64)0;
    };
    float lo, hi;
    weigh.bin_range(state.bin, &lo, &hi);
    u64 above;
    cut = score_of(narrow<FEW_NT>(sh, [&](auto&& f) {
        for (int i = tid; i < members; i += FEW_NT) {
            const float z = sh.list_z[i];
            f(pattern(z), [&] { return weigh(z); });
        }
    }, pattern(lo), pattern(hi), state.above, state.least, &above));
    tie_end = first_tie_out<FEW_NT>(sh, [&](auto&& f) {
        for (int i = tid; i < members; i += FEW_NT)
            if (sh.list_z[i] == cut) f(sh.list_at[i]);
    }, ties_within(state.target, above, weigh(cut)), (uint32_t)a.vocab);
    __syncthreads();
    for (int i = tid; i < members; i += FEW_NT) {
        const u64 w = weight_at(sh.list_z[i], sh.list_at[i]);
        if (w) atomicAdd(&sh.part[sh.list_at[i] / (uint32_t)work.part_len], w);
    }
    const u64 total = scan_parts<FEW_NT>(sh, work.parts);
    draw_from_parts(sh, src, a, work, row, set, weigh, total, weight_at);
}

// Short rows go to one block each: what the other form saves in passes it loses in launches.  Rows of 32768 scores, by one
// block each and by the whole chip: one row with top-k 50 11 and 13 us, 256 rows with settings of every kind 46 and 57 us, 1024
// rows 106 and 100 us.  Few rows with top-p alone take two passes of weights, for which one block is slow: 1, 16, 64, 128 rows
// of 32768 44, 45, 45, 46 us by a block and 31, 33, 36, 42 by the chip, of 20000 37, 37, 37, 38 and 31, 33, 35, 40, of 12000
// 26 to 28 and 31 to 36.
static bool by_whole_chip(int64_t vocab) { return vocab > 32768; }
static bool few_rows(int64_t n, int64_t vocab) { return n <= 64 && vocab > 16384; }
static bool whole_chip_pays(int64_t n, const SampleArgs& a) {
    const bool top_p_alone = !a.d_top_k && a.top_k <= 0 && (a.d_top_p || (a.top_p > 0.0f && a.top_p < 1.0f)) && (a.d_temperature || a.temperature > 0.0f);
    return by_whole_chip(a.vocab) || (few_rows(n, a.vocab) && top_p_alone);
}
static const int64_t SAMPLE_BATCH = 1024;           // rows at a time by the whole chip: bounds the workspace (59 MB at 131072 scores)

template <class T> static int launch_long_rows(const T* z, int64_t n, const SampleArgs& a, const SampleWork& w, hipStream_t s) {
    const dim3 rows((unsigned)n), few(FEW_NT);
    const int slices = ceil_div(a.vocab, STREAM_NT * Piece<T>::N * STREAM_PIECES);
    hipLaunchKernelGGL(sample_groups_kernel<T>, dim3((unsigned)(n * slices)), dim3(STREAM_NT), 0, s, z, a, w, slices);
    VDB_HIP(hipGetLastError());
    // whether rows can need their weights, and a border among them
    const bool all_known = !a.d_temperature && !a.d_top_k && !a.d_top_p && !a.d_min_p;
    const RowMode mode = mode_of(a.temperature, a.top_k, a.top_p, a.min_p);
    const bool listed = all_known ? mode == ROW_LIST || mode == ROW_WHOLE
                                  : (!a.d_temperature && !(a.temperature > 0.0f)) || (!a.d_top_k && a.top_k >= 1) || (!a.d_top_p && a.top_p <= 0.0f);
    const int weigh_cuts = ceil_div(w.parts, WEIGH_PARTS), cuts = ceil_div(w.parts, ABOVE_PARTS);
    hipLaunchKernelGGL(sample_pick_kernel<T>, dim3((unsigned)(listed ? n : n + n * weigh_cuts)), few, 0, s, z, a, w, (int)n, weigh_cuts, slices);
    VDB_HIP(hipGetLastError());
    if (!listed) {
        hipLaunchKernelGGL(sample_border_kernel<T>, rows, few, 0, s, z, a, w);
        VDB_HIP(hipGetLastError());
        if (a.d_top_p || a.top_p < 1.0f) {
            hipLaunchKernelGGL(sample_above_kernel<T>, dim3((unsigned)(n * cuts)), dim3(STREAM_NT), 0, s, z, a, w, cuts);
            VDB_HIP(hipGetLastError());
        }
    }
    hipLaunchKernelGGL(sample_rest_kernel<T>, rows, dim3(ROW_NT), 0, s, z, a, w);
    VDB_HIP(hipGetLastError());
    return VDB_OK;
}

template <class T> static int launch_sample(const T* z, int64_t n, const SampleArgs& a, void* d_work, hipStream_t s) {
    const bool whole_chip = whole_chip_pays(n, a);
    const int64_t batch = whole_chip ? SAMPLE_BATCH : (int64_t)1 << 21;           // a launch holds fewer than 2^32 threads
    const SampleWork w = whole_chip ? sample_work(d_work, std::min(n, batch), a.vocab) : SampleWork{};
    for (int64_t r = 0; r < n; r += batch) {
        const int64_t m = std::min(n - r, batch);
        SampleArgs b = a;
        b.uniform += r;
        if (b.d_temperature) b.d_temperature += r;
        if (b.d_top_k) b.d_top_k += r;
        if (b.d_top_p) b.d_top_p += r;
        if (b.d_min_p) b.d_min_p += r;
        if (b.mask) b.mask += r * b.mask_ld;
        b.out_row += r;
        if (b.out_logp) b.out_logp += r;
        if (whole_chip) VDB_TRY(launch_long_rows(z + r * a.ld, m, b, w, s));
        else {
            hipLaunchKernelGGL(sample_kernel<T>, dim3((unsigned)m), dim3(ROW_NT), 0, s, z + r * a.ld, b);
            VDB_HIP(hipGetLastError());
        }
    }
    return VDB_OK;
}

}  // namespace vdb

using namespace vdb;

int vdb_sample_workspace(int64_t n, int64_t vocab, int64_t* bytes) {
    VDB_REQUIRE(bytes, "null pointer for the workspace size");
    VDB_REQUIRE(n >= 0 && vocab >= 1 && vocab <= ((int64_t)1 << 24), "bad sizes for sampling: %lld rows of %lld scores (at most 2^24)", (long long)n,
                (long long)vocab);
    *bytes = by_whole_chip(vocab) || few_rows(n, vocab) ? sample_work(nullptr, std::min(n, SAMPLE_BATCH), vocab).bytes : 0;
    return VDB_OK;
}

int vdb_sample_dev(const void* d_scores, int type, int64_t n, int64_t vocab, int64_t ld, int smaller_first, const float* d_uniform,
                   const float* d_temperature, float temperature, const int32_t* d_top_k, int top_k, const float* d_top_p, float top_p,
                   const float* d_min_p, float min_p, const uint32_t* d_mask, int64_t mask_ld, int64_t* d_out_row, float* d_out_logp,
                   void* d_work, int64_t work_bytes, void* stream) {
    int64_t need = 0;
    VDB_REQUIRE(valid_type(type), "unknown value type %d", type);
    VDB_TRY(vdb_sample_workspace(n, vocab, &need));
    VDB_REQUIRE(n < ((int64_t)1 << 31) - 1 && ld >= 0, "bad sizes for sampling: %lld rows, leading dimension %lld", (long long)n, (long long)ld);
    VDB_REQUIRE(mask_ld == 0 || mask_ld >= (vocab + 31) / 32, "a mask over %lld scores takes %lld words a row, its rows lie %lld apart", (long long)vocab,
                (long long)((vocab + 31) / 32), (long long)mask_ld);
    VDB_REQUIRE(n == 0 || (d_scores && d_uniform && d_out_row), "null pointer in sampling from %lld rows", (long long)n);
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    const SampleArgs a{vocab, ld, smaller_first, d_uniform, d_temperature, temperature, d_top_k, top_k, d_top_p, top_p, d_min_p, min_p,
                       d_mask, mask_ld, d_out_row, d_out_logp, std::min(52, 62 - bits)};
    if (!whole_chip_pays(n, a)) need = 0;
    VDB_REQUIRE(work_bytes >= need && (d_work || need == 0), "the workspace of %lld bytes is too small for this sampling (%lld needed)",
                (long long)work_bytes, (long long)need);
    VDB_REQUIRE(aligned_work(d_work), "a workspace begins at a multiple of 16 bytes");
    if (n == 0) return VDB_OK;
    VDB_TRY(ensure_init());
    (void)hipSetDevice(ctx().device);
    return with_type(type, [&](auto* p) -> int {
        typedef std::remove_pointer_t<decltype(p)> T;
        return launch_sample((const T*)d_scores, n, a, d_work, (hipStream_t)stream);
    });
}
