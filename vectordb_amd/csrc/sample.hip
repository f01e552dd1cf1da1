// One row number drawn from each score row (vdb_sample_dev): temperature, top-k, top-p, min-p, a row filter, and a
// uniform number given by the caller.
//
// What remains of a row after the filters is a prefix of the order (score descending, row number ascending): a
// smallest score and how many of the rows that share it.  That score is found without sorting: a histogram of the
// scores' ordered bit patterns, eight bits at a time, counts (top-k) or adds weights (top-p) until one pattern is
// left.  Weights exp((z - max) / tau) are taken in double and added as 64-bit integers (multiples of 2^-s), so sums do
// not depend on the order in which threads add, and the draw is the one of the definition.
#include "vdb_internal.h"
#include "values.h"

#include <algorithm>

namespace vdb {

static constexpr int SAMPLE_NT = 1024, SAMPLE_WAVES = SAMPLE_NT / 64;
typedef unsigned long long u64;

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

// Ordered pattern of a score: larger score, larger pattern; 0 = cannot be drawn.  -0 counts as +0.
__device__ __forceinline__ uint32_t pattern(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (z != z || z == -INFINITY) ? 0u : o;
}
__device__ __forceinline__ float score_of(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }

template <class T> struct Row {
    const T* z;
    int64_t vocab;
    const uint32_t* mask;
    int flip;
    // ordered patterns of the elements [at, at + N)
    __device__ __forceinline__ void load(int64_t at, uint32_t* o) const {
        constexpr int N = Piece<T>::N;
        float x[N];
        load_values(z, at, vocab, NAN, x);
        uint32_t bits = 0xffffffffu;
        if (mask && at < vocab) bits = mask[at >> 5] >> (at & 31);      // N divides 32: one word holds the piece
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t p = pattern(flip ? -x[e] : x[e]);
            o[e] = (bits >> e) & 1u ? p : 0u;
        }
    }
};

struct Weigher {
    double per_log2;                 // log2(e) / tau
    uint32_t best;
    double best_z, unit;
    __device__ __forceinline__ u64 operator()(uint32_t o) const {
        if (o == best) return (u64)unit;
        const double t = ((double)score_of(o) - best_z) * per_log2;
        return t >= -40.0 ? (u64)(exp2(t) * unit + 0.5) : 0ull;       // a NaN (tau = inf under scores of inf) is no weight
    }
    __device__ __forceinline__ double exact(uint32_t o) const {
        if (o == best) return 1.0;
        return exp2(((double)score_of(o) - best_z) * per_log2);
    }
};

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <class T>
__global__ void __launch_bounds__(SAMPLE_NT) sample_kernel(const T* __restrict__ scores, SampleArgs a) {
    constexpr int N = Piece<T>::N;
    __shared__ u64 bin[256];
    __shared__ u64 red[SAMPLE_WAVES + 1];
    __shared__ u64 chosen_above;
    __shared__ int chosen_bin;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x, vocab = a.vocab;
    const Row<T> r{scores + row * a.ld, vocab, a.mask ? a.mask + row * a.mask_ld : nullptr, a.smaller_first};
    const float tau = a.d_temperature ? a.d_temperature[row] : a.temperature;
    const float top_p = a.d_top_p ? a.d_top_p[row] : a.top_p;
    const float min_p = a.d_min_p ? a.d_min_p[row] : a.min_p;
    const bool greedy = !(tau > 0.0f);
    int64_t top_k = a.d_top_k ? a.d_top_k[row] : a.top_k;
    if (greedy) top_k = 1;
    const int64_t seg = (vocab + SAMPLE_WAVES - 1) / SAMPLE_WAVES;
    const int64_t step = 64 * N, seg_len = (seg + step - 1) / step * step;          // a wave's contiguous part
    const int64_t w_lo = min((int64_t)wave * seg_len, vocab), w_hi = min(w_lo + seg_len, vocab);

    // the largest score
    uint32_t best = 0;
    for (int64_t i = (int64_t)tid * N; i < vocab; i += SAMPLE_NT * N) {
        uint32_t o[N];
        r.load(i, o);
#pragma unroll
        for (int e = 0; e < N; ++e) best = max(best, o[e]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, o));
    if (lane == 0) red[wave] = best;
    __syncthreads();
    for (int w = 0; w < SAMPLE_WAVES; ++w) best = max(best, (uint32_t)red[w]);
    if (best == 0) {
        if (tid == 0) {
            a.out_row[row] = -1;
            if (a.out_logp) a.out_logp[row] = -INFINITY;
        }
        return;
    }
    const Weigher weigh{1.4426950408889634073599 / (greedy ? 1.0 : (double)tau), best, (double)score_of(best), ldexp(1.0, a.shift)};

    // the prefix: scores above `cut`, and the first `ties` rows at it
    uint32_t cut = 0;
    int64_t ties = INT64_MAX;
    // narrow to one pattern: the first, from the top, at which the running sum of `value` reaches `target`
    auto narrow = [&](auto&& value, u64 target, u64* above_out) {
        uint32_t known = 0;
        u64 above = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) bin[tid] = 0;
            __syncthreads();
            for (int64_t i = (int64_t)tid * N; i < vocab; i += SAMPLE_NT * N) {
                uint32_t o[N];
                r.load(i, o);
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (o[e] && (shift == 24 || (o[e] >> (shift + 8)) == known)) {
                        const u64 v = value(o[e]);
                        if (v) atomicAdd(&bin[(o[e] >> shift) & 255], v);
                    }
            }
            __syncthreads();
            if (tid == 0) {
                u64 run = above;
                int b = 255;
                for (; b > 0; --b) {
                    if (run + bin[b] >= target) break;
                    run += bin[b];
                }
                chosen_above = run;
                chosen_bin = b;
            }
            __syncthreads();
            above = chosen_above;
            known = (known << 8) | (uint32_t)chosen_bin;
        }
        *above_out = above;
        return known;
    };
    auto block_total = [&](u64 v) {
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) red[wave] = v;
        __syncthreads();
        v = 0;
        for (int w = 0; w < SAMPLE_WAVES; ++w) v += red[w];
        return v;
    };
    auto sum_over = [&](auto&& value) {
        u64 v = 0;
        for (int64_t i = (int64_t)tid * N; i < vocab; i += SAMPLE_NT * N) {
            uint32_t o[N];
            r.load(i, o);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (o[e]) v += value(o[e]);
        }
        return block_total(v);
    };

    if (top_k > 0) {
        const u64 usable = sum_over([](uint32_t) { return (u64)1; });
        if ((u64)top_k < usable) {
            u64 above;
            cut = narrow([](uint32_t) { return (u64)1; }, (u64)top_k, &above);
            ties = top_k - (int64_t)above;
        }
    }
    if (top_p < 1.0f) {
        const u64 over = sum_over([&](uint32_t o) { return o > cut ? weigh(o) : 0ull; });
        const u64 at_cut = cut && ties < INT64_MAX ? weigh(cut) * (u64)ties : 0ull;
        const double target = (double)(over + at_cut) * (double)top_p;
        // a row remains iff the weights before it are less than target: the first row is kept, and the last kept one is
        // where the running sum, itself included, reaches the target
        u64 least = target > 0.0 ? (u64)ceil(target) : 0ull;
        if (least == 0) least = 1;
        u64 above;
        const uint32_t c2 = over && (double)over >= target ? narrow([&](uint32_t o) { return o > cut ? weigh(o) : 0ull; }, least, &above) : cut;
        if (c2 != cut) {
            const u64 w = weigh(c2);
            const double left = (target - (double)above) / (double)w;
            cut = c2;
            ties = left >= 9.0e18 ? INT64_MAX : max((int64_t)1, (int64_t)ceil(left));
        } else if (at_cut) {
            const double left = (target - (double)over) / (double)weigh(cut);
            ties = min(ties, max((int64_t)1, (int64_t)ceil(left)));
        }
    }
    const double least_w = min_p > 0.0f ? fmin((double)min_p, 1.0) : 0.0;
    const bool use_min = min_p > 0.0f;
    if (use_min && cut && weigh.exact(cut) < least_w) ties = 0;

    // the weight of a row at the cut counts for the first `ties` rows there, in row order
    int64_t tie_end = vocab;                  // rows at the cut from here on are out
    if (cut && ties < INT64_MAX) {
        u64 mine = 0;
        for (int64_t i = w_lo + lane * N; i < w_hi; i += step) {
            uint32_t o[N];
            r.load(i, o);
#pragma unroll
            for (int e = 0; e < N; ++e) mine += (i + e < w_hi && o[e] == cut) ? 1 : 0;
        }
        mine = wave_sum(mine);
        __syncthreads();
        if (lane == 0) red[wave] = mine;
        if (tid == 0) chosen_above = (u64)vocab;
        __syncthreads();
        int64_t run = 0;
        for (int w = 0; w < wave; ++w) run += (int64_t)red[w];
        if (run <= ties && run + (int64_t)mine > ties) {
            // the first row that is out lies in this wave's part
            for (int64_t i0 = w_lo; i0 < w_hi; i0 += step) {
                const int64_t i = i0 + lane * N;
                uint32_t o[N];
                r.load(i, o);
                int cnt = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) cnt += o[e] == cut ? 1 : 0;
                int inc = cnt;
#pragma unroll
                for (int s = 1; s < 64; s <<= 1) {
                    const int t = __shfl_up(inc, s);
                    if (lane >= s) inc += t;
                }
                int64_t at = run + inc - cnt;
                const bool here = at <= ties && at + cnt > ties;
                if (here) {
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (o[e] == cut) {
                            if (at == ties) chosen_above = (u64)(i + e);
                            ++at;
                        }
                }
                if (__ballot(here)) break;
                run += __shfl(inc, 63);
            }
        }
        __syncthreads();
        tie_end = (int64_t)chosen_above;
    }
    auto remaining = [&](uint32_t o, int64_t i) -> u64 {
        if (o == 0 || o < cut || (o == cut && i >= tie_end)) return 0;
        if (use_min && weigh.exact(o) < least_w) return 0;
        return weigh(o);
    };
    // weights by wave part, then the part and the row at which the running sum exceeds uniform * total
    u64 mine = 0;
    for (int64_t i = w_lo + lane * N; i < w_hi; i += step) {
        uint32_t o[N];
        r.load(i, o);
#pragma unroll
        for (int e = 0; e < N; ++e) mine += remaining(o[e], i + e);
    }
    mine = wave_sum(mine);
    __syncthreads();
    if (lane == 0) red[wave] = mine;
    __syncthreads();
    u64 total = 0, run = 0;
    for (int w = 0; w < SAMPLE_WAVES; ++w) {
        if (w < wave) run += red[w];
        total += red[w];
    }
    // running sum > uniform * total, as integers: at least floor(uniform * total) + 1
    const double goal = (double)a.uniform[row] * (double)total;
    u64 least = goal >= 0.0 ? (u64)floor(goal) + 1 : 1;
    if (!(least <= total)) least = total;
    if (run < least && run + mine >= least) {
        for (int64_t i0 = w_lo; i0 < w_hi; i0 += step) {
            const int64_t i = i0 + lane * N;
            uint32_t o[N];
            r.load(i, o);
            u64 w[N], sum = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) sum += w[e] = remaining(o[e], i + e);
            u64 inc = sum;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const u64 t = __shfl_up(inc, s);
                if (lane >= s) inc += t;
            }
            u64 at = run + inc - sum;
            const bool here = at < least && at + sum >= least;
            if (here) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (at < least && at + w[e] >= least) {
                        a.out_row[row] = i + e;
                        if (a.out_logp) a.out_logp[row] = (float)log((double)w[e] / (double)total);
                    }
                    at += w[e];
                }
            }
            if (__ballot(here)) break;
            run += __shfl(inc, 63);
        }
    }
}

}  // namespace vdb

using namespace vdb;

int vdb_sample_workspace(int64_t n, int64_t vocab, int64_t* bytes) {
    VDB_REQUIRE(bytes, "null pointer for the workspace size");
    VDB_REQUIRE(n >= 0 && vocab >= 1 && vocab <= ((int64_t)1 << 24), "bad sizes for sampling: %lld rows of %lld scores (at most 2^24)", (long long)n,
                (long long)vocab);
    *bytes = 0;
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
    VDB_REQUIRE(work_bytes >= need && (d_work || need == 0), "the workspace of %lld bytes is too small for this sampling (%lld needed)",
                (long long)work_bytes, (long long)need);
    if (n == 0) return VDB_OK;
    VDB_TRY(ensure_init());
    (void)hipSetDevice(ctx().device);
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    const SampleArgs a{vocab, ld, smaller_first, d_uniform, d_temperature, temperature, d_top_k, top_k, d_top_p, top_p, d_min_p, min_p,
                       d_mask, mask_ld, d_out_row, d_out_logp, std::min(52, 62 - bits)};
    return with_type(type, [&](auto* p) -> int {
        typedef std::remove_pointer_t<decltype(p)> T;
        hipLaunchKernelGGL(sample_kernel<T>, dim3((unsigned)n), dim3(SAMPLE_NT), 0, (hipStream_t)stream, (const T*)d_scores, a);
        VDB_HIP(hipGetLastError());
        return VDB_OK;
    });
}
