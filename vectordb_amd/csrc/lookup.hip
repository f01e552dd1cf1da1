// Rows of a table by number (vdb_lookup_dev) and the gradient of that table (vdb_lookup_grad_dev).
//
// lookup: out[i] = scale * table[rows[i]].  A copy of n rows in 16-byte pieces, four a thread; what bounds it is HBM traffic,
// n * dim values written and as many read (from cache where rows repeat): 131072 x 2048 bf16 185 us, 5.8 TB/s.
//
// gradient: table_grad[r] = scale * sum over {i : rows[i] == r} of grad[i].  The positions i are sorted by row number, stable,
// so the members of a row lie side by side in ascending i; the sorted positions are cut into chunks of 8 to 64, a group of
// threads adds the rows of a chunk in order, and a row that crosses chunks has its parts added in chunk order by a
// second launch.  No atomics on values: the order of every sum is fixed by the row numbers.  Bound: grad read once,
// table_grad written once (rows without members as zeros): 131072 x 2048 bf16 into 131072 fp32 rows 387 us, 4.2 TB/s.
#include "vdb_internal.h"
#include "values.h"

#include <algorithm>

namespace vdb {

// ---------------------------------------------------------------- lookup
// A block takes `take` rows, `pieces` pieces of 16 bytes each, AHEAD of them a thread at a time.  inverse = ceil(2^32 / pieces):
// the row of piece x is the upper half of x * inverse (exact below 2^16), x itself lies in the only row otherwise.
static constexpr int LOOKUP_NT = 256, LOOKUP_AHEAD = 4;
template <class Ti, class To>
__global__ void __launch_bounds__(LOOKUP_NT) lookup_kernel(const Ti* __restrict__ table, int64_t n_rows, int dim, int64_t ld,
                                                           const int64_t* __restrict__ rows, int64_t n, float scale, To* __restrict__ out,
                                                           int64_t ld_out, int take, uint32_t pieces, uint32_t inverse) {
    constexpr int N = Piece<Ti>::N;
    const int64_t first = (int64_t)blockIdx.x * take;
    const uint32_t mine = (uint32_t)min((int64_t)take, n - first), all = mine * pieces;
    for (uint32_t x0 = threadIdx.x; x0 < all; x0 += LOOKUP_AHEAD * LOOKUP_NT) {
        int64_t r[LOOKUP_AHEAD];
        uint32_t i[LOOKUP_AHEAD], c[LOOKUP_AHEAD];
        Piece<Ti> v[LOOKUP_AHEAD];
#pragma unroll
        for (int u = 0; u < LOOKUP_AHEAD; ++u) {
            const uint32_t x = min(x0 + u * LOOKUP_NT, all - 1);
            i[u] = pieces == 1 ? x : take == 1 ? 0 : __umulhi(x, inverse);
            c[u] = (x - i[u] * pieces) * N;
            r[u] = rows[first + i[u]];
        }
        if (dim >= N) {
            // a piece that would end behind the row is the row's last N values: what two threads write there is the same
#pragma unroll
            for (int u = 0; u < LOOKUP_AHEAD; ++u) {
                c[u] = min(c[u], (uint32_t)(dim - N));
                v[u] = Piece<Ti>{};
                if (r[u] >= 0 && r[u] < n_rows) v[u] = load_piece(table + r[u] * ld + c[u]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < LOOKUP_AHEAD; ++u) {
                float y[N];
                load_values(table + r[u] * ld, 0, r[u] >= 0 && r[u] < n_rows ? dim : 0, 0.0f, y);
                v[u].set(y);
            }
        }
#pragma unroll
        for (int u = 0; u < LOOKUP_AHEAD; ++u) {
            if (x0 + u * LOOKUP_NT >= all) break;
            const bool known = r[u] >= 0 && r[u] < n_rows;
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = known ? scale * v[u].get(e) : 0.0f;
            store_values<To, N>(out + (first + i[u]) * ld_out, c[u], dim, y);
        }
    }
}

// ---------------------------------------------------------------- stable radix sort of the positions by row number
static constexpr int SORT_NT = 256, SORT_WAVES = SORT_NT / 64, SORT_MAX_BITS = 10, SORT_BLOCKS = 512;

struct SortPlan {
    int passes, bits;          // digits of `bits` bits; keys are 0 .. n_rows (n_rows = no row)
    int blocks;
    int64_t wave_keys;         // keys of one wave, a multiple of 64
};
static SortPlan sort_plan(int64_t n, int64_t n_rows) {
    SortPlan p;
    int key_bits = 1;
    while (((int64_t)1 << key_bits) <= n_rows) ++key_bits;
    p.passes = (key_bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
    p.bits = (key_bits + p.passes - 1) / p.passes;
    // a wave takes its keys 64 at a time, each step waiting for the last: few of them, until the blocks' histograms
    // would outgrow what they save
    p.wave_keys = std::max<int64_t>(128, round_up64((n + SORT_BLOCKS * SORT_WAVES - 1) / (SORT_BLOCKS * SORT_WAVES), 64));
    p.blocks = (int)((n + p.wave_keys * SORT_WAVES - 1) / (p.wave_keys * SORT_WAVES));
    return p;
}

__device__ __forceinline__ int key_of(const int64_t* rows, const int* keys, int64_t i, int64_t n_rows) {
    if (!rows) return keys[i];
    const int64_t r = rows[i];
    return (int)(r >= 0 && r < n_rows ? r : n_rows);
}

// Zeros for table rows, written by blocks behind those of a sort launch: the sort waits on latencies and leaves the
// memory idle.  Rows [r0, r1) of `units` 16-bit units, `ld` units apart: rows that lie back to back as one stretch from 16-byte
// border to border (449640 x 597 fp16 row by row: 210 us, so 102), else a group of 1 << log_tpr threads takes a row.
struct Fill {
    uint16_t* out;
    int64_t r0, r1, units, ld;
    int log_tpr;
};
__device__ static void fill_rows(const Fill& f, int64_t block, int64_t blocks, int nt) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    if (f.units == f.ld) {
        uint16_t *lo = f.out + f.r0 * f.ld, *hi = f.out + f.r1 * f.ld;
        uint16_t* border = (uint16_t*)(((uintptr_t)lo + 15) & ~(uintptr_t)15);
        uint16_t* from = border < hi ? border : hi;
        const int64_t pieces = (hi - from) / 8;
        const int64_t share = (pieces + blocks - 1) / blocks, end = min((block + 1) * share, pieces);
        for (int64_t i = block * share + threadIdx.x; i < end; i += nt) ((u32x4*)from)[i] = zero;
        if (block == 0 && threadIdx.x < 8) {
            if (lo + threadIdx.x < from) lo[threadIdx.x] = 0;
            if (from + pieces * 8 + threadIdx.x < hi) from[pieces * 8 + threadIdx.x] = 0;
        }
        return;
    }
    const int per = nt >> f.log_tpr;
    for (int64_t r = f.r0 + block * per + (threadIdx.x >> f.log_tpr); r < f.r1; r += blocks * per) {
        uint16_t* dst = f.out + r * f.ld;
        for (int64_t c = (threadIdx.x & ((1 << f.log_tpr) - 1)) * 8; c < f.units; c += (int64_t)8 << f.log_tpr) {
            if (c + 8 <= f.units) __builtin_memcpy(dst + c, &zero, 16);
            else
                for (int64_t e = c; e < f.units; ++e) dst[e] = 0;
        }
    }
}

// hist[digit][block]
__global__ void __launch_bounds__(SORT_NT) sort_hist_kernel(const int64_t* __restrict__ rows, const int* __restrict__ keys, int64_t n,
                                                            int64_t n_rows, int shift, int bits, int64_t wave_keys, int* __restrict__ hist,
                                                            int blocks, Fill fill) {
    extern __shared__ int cnt[];
    if ((int)blockIdx.x >= blocks) return fill_rows(fill, (int)blockIdx.x - blocks, (int)gridDim.x - blocks, SORT_NT);
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += SORT_NT) cnt[d] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * wave_keys * SORT_WAVES, hi = min(lo + wave_keys * SORT_WAVES, n);
    for (int64_t i = lo + threadIdx.x; i < hi; i += SORT_NT) atomicAdd(&cnt[(key_of(rows, keys, i, n_rows) >> shift) & (bins - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += SORT_NT) hist[(int64_t)d * blocks + blockIdx.x] = cnt[d];
}

// inclusive prefix over a wave
__device__ __forceinline__ int wave_prefix(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(v, o);
        if (lane >= o) v += t;
    }
    return v;
}
// one wave per digit: exclusive prefix of its counts over the blocks, all loaded at once, and their total
__global__ void __launch_bounds__(64) sort_scan_kernel(int* __restrict__ hist, int blocks, int* __restrict__ totals) {
    int* h = hist + (int64_t)blockIdx.x * blocks;
    int v[SORT_BLOCKS / 64], run = 0;
#pragma unroll
    for (int j = 0; j < SORT_BLOCKS / 64; ++j) v[j] = j * 64 + (int)threadIdx.x < blocks ? h[j * 64 + threadIdx.x] : 0;
#pragma unroll
    for (int j = 0; j < SORT_BLOCKS / 64; ++j) {
        if (j * 64 >= blocks) break;
        const int s = wave_prefix(v[j]);
        if (j * 64 + (int)threadIdx.x < blocks) h[j * 64 + threadIdx.x] = run + s - v[j];
        run += __shfl(s, 63);
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// Lanes of the wave whose digit equals this lane's (lanes without a key are in nobody's set).  All the bits that a digit can
// have, unrolled: those above it are zero in every lane (a loop over its own bits takes a tenth longer).
__device__ __forceinline__ unsigned long long same_digit(int d, bool have) {
    unsigned long long m = __ballot(have);
    uint32_t lo = (uint32_t)m, hi = (uint32_t)(m >> 32);
#pragma unroll
    for (int b = 0; b < SORT_MAX_BITS; ++b) {
        const int mine = (d << (31 - b)) >> 31;                      // all ones or none
        const unsigned long long one = __ballot(mine != 0);
        lo &= ~((uint32_t)one ^ (uint32_t)mine);
        hi &= ~((uint32_t)(one >> 32) ^ (uint32_t)mine);
    }
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ int lanes_below(unsigned long long m) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

__global__ void __launch_bounds__(SORT_NT) sort_scatter_kernel(const int64_t* __restrict__ rows, const int* __restrict__ keys,
                                                               const int* __restrict__ pos, int64_t n, int64_t n_rows, int shift, int bits,
                                                               int64_t wave_keys, const int* __restrict__ hist, const int* __restrict__ totals,
                                                               int* __restrict__ keys_out, int* __restrict__ pos_out, int blocks, Fill fill) {
    extern __shared__ int lds[];
    if ((int)blockIdx.x >= blocks) return fill_rows(fill, (int)blockIdx.x - blocks, (int)gridDim.x - blocks, SORT_NT);
    constexpr int MOST = (1 << SORT_MAX_BITS) / SORT_NT;
    const int bins = 1 << bits;
    int* start = lds;                         // [SORT_WAVES][bins]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // a contiguous run of digits per thread: their totals and what the blocks before have of them
    const int per = (bins + SORT_NT - 1) / SORT_NT;
    int total[MOST], before[MOST];
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
        const int d = tid * per + j;
        const bool mine = j < per && d < bins;
        total[j] = mine ? totals[d] : 0;
        before[j] = mine ? hist[(int64_t)d * blocks + blockIdx.x] : 0;
    }
    for (int d = tid; d < SORT_WAVES * bins; d += SORT_NT) start[d] = 0;
    __syncthreads();
    const int64_t lo = ((int64_t)blockIdx.x * SORT_WAVES + wave) * wave_keys, hi = min(lo + wave_keys, n);
    int* mine = start + wave * bins;
    for (int64_t i = lo + lane; i < hi; i += 64) atomicAdd(&mine[(key_of(rows, keys, i, n_rows) >> shift) & (bins - 1)], 1);
    __shared__ int wave_total[SORT_WAVES];
    int sum = 0;
#pragma unroll
    for (int j = 0; j < MOST; ++j) sum += total[j];
    const int upto = wave_prefix(sum);
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    int run = upto - sum;
    for (int w = 0; w < wave; ++w) run += wave_total[w];
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
        const int d = tid * per + j;
        if (j >= per || d >= bins) break;
        int at = run + before[j];
        run += total[j];
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int c = start[w * bins + d];
            start[w * bins + d] = at;
            at += c;
        }
    }
    __syncthreads();
    for (int64_t i0 = lo; i0 < hi; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool have = i < hi;
        const int key = have ? key_of(rows, keys, i, n_rows) : 0;
        const int d = (key >> shift) & (bins - 1);
        const unsigned long long m = same_digit(d, have);
        if (have) {
            const int rank = lanes_below(m);
            const int base = mine[d];
            // the wave's LDS operations run in order: every lane has its base before the last of its set moves it on
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (rank == __popcll(m) - 1) mine[d] = base + rank + 1;
            keys_out[base + rank] = key;
            pos_out[base + rank] = pos ? pos[i] : (int)i;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Up to COUNT_MAX positions: each by itself counts those that come before it, smaller rows and equal ones of earlier positions, and
// has its place, in one launch over the whole chip: n^2 comparisons of two instructions.  8192 positions take 10 us, where the
// 6 launches of the digits take 26 and one block that sorted in LDS took 21; at 16384 both forms are even.
// A block takes 16 * KEYS positions, KEYS a thread, and all the keys into LDS; its 16 threads of a share go through a 64th of them.
static constexpr int COUNT_NT = 1024, COUNT_LANES = 16, COUNT_SHARES = COUNT_NT / COUNT_LANES, COUNT_MAX = 12288;         // keys in less than 64 KB of LDS

template <int KEYS>
__global__ void __launch_bounds__(COUNT_NT) sort_count_kernel(const int64_t* __restrict__ rows, int n, int64_t n_rows, int blocks, int* __restrict__ keys_out,
                                                              int* __restrict__ pos_out, Fill fill) {
    constexpr int TAKE = COUNT_LANES * KEYS, AHEAD = 4;
    extern __shared__ __align__(16) int lds[];
    if ((int)blockIdx.x >= blocks) return fill_rows(fill, (int)blockIdx.x - blocks, (int)gridDim.x - blocks, COUNT_NT);
    __shared__ int before[COUNT_NT / 64][TAKE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, room = (n + 3) & ~3;
    for (int i0 = tid; i0 < room; i0 += AHEAD * COUNT_NT) {
        int64_t r[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) r[u] = rows[min(i0 + u * COUNT_NT, n - 1)];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * COUNT_NT;
            if (i < room) lds[i] = i >= n ? 0x7fffffff : r[u] >= 0 && r[u] < n_rows ? (int)r[u] : (int)n_rows;
        }
    }
    __syncthreads();
    const int first = (int)blockIdx.x * TAKE, share = tid / COUNT_LANES;
    int key[KEYS], at[KEYS];
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        const int i = first + k * COUNT_LANES + (tid & (COUNT_LANES - 1));
        key[k] = lds[min(i, n - 1)];
        // equal ones among the block's own positions
        const int j = first + share;
        at[k] = share < TAKE && j < i && j < n && lds[j] == key[k];
    }
#pragma unroll 4
    for (int q = share; q < room / 4; q += COUNT_SHARES) {
        const int4 other = *(const int4*)(lds + 4 * q);
        const int equal = 4 * q < first;
#pragma unroll
        for (int k = 0; k < KEYS; ++k) {
            const int least = key[k] + equal;
            at[k] += (other.x < least) + (other.y < least) + (other.z < least) + (other.w < least);
        }
    }
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
        at[k] += __shfl_xor(at[k], 16);
        at[k] += __shfl_xor(at[k], 32);
        if (lane < COUNT_LANES) before[wave][k * COUNT_LANES + lane] = at[k];
    }
    __syncthreads();
    if (tid >= TAKE || first + tid >= n) return;
    int place = 0;
#pragma unroll
    for (int w = 0; w < COUNT_NT / 64; ++w) place += before[w][tid];
    keys_out[place] = lds[first + tid];
    pos_out[place] = first + tid;
}

// ---------------------------------------------------------------- sums of the sorted rows
// The rows of a batch of SEG_BATCH positions are in flight together; a chunk is as many batches as still fill the chip, one at
// least (10240 rows of 384 values: 22 us with four).
static constexpr int SEG_BATCH = 8;

// first position whose key is not below r, found by a whole wave: 64 probes a step (n and keys are below 2^31)
__device__ __forceinline__ int64_t lower_bound_wave(const int* __restrict__ keys, int64_t n, int64_t r) {
    uint32_t a = 0, b = (uint32_t)n;                       // the answer lies in [a, b]
    while (a < b) {
        const uint32_t step = (b - a + 63) >> 6, at = a + step * ((threadIdx.x & 63) + 1) - 1;
        const uint32_t below = (uint32_t)__popcll(__ballot(at < b && (int64_t)keys[at < b ? at : a] < r));
        b = min(b, a + step * (below + 1) - 1);
        a += step * below;
    }
    return a;
}

template <class To, int N> __device__ __forceinline__ void put_row(To* row, int c, int dim, float scale, const float* acc, bool accumulate) {
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = scale * acc[e];
    if (accumulate) {
        if (c + N <= dim) {
            To old[N];
            __builtin_memcpy(old, row + c, sizeof(old));
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = (float)old[e] + x[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c + e < dim) x[e] = (float)row[c + e] + x[e];
        }
    }
    store_values<To, N>(row, c, dim, x);
}

// sums of a part of a row lie in whole pieces
__host__ __device__ static inline int64_t part_pitch(int dim) { return ((int64_t)dim + 7) & ~7; }

static constexpr int ZERO_ROWS = 64;                        // table rows that a block writes zeros to, at most

// zeros to those of the `count` table rows from r0 on that are not named
template <class To>
__device__ __forceinline__ void zero_rows(const int* named, To* out, int64_t r0, int count, int64_t n_rows, int dim, int64_t ld_out, int log_zero, int nt) {
    constexpr int N = Piece<To>::N;
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = 0.0f;
    for (int j = threadIdx.x >> log_zero; j < count && r0 + j < n_rows; j += nt >> log_zero) {
        if (named[j]) continue;
        To* dst = out + (r0 + j) * ld_out;
        for (int c = (threadIdx.x & ((1 << log_zero) - 1)) * N; c < dim; c += N << log_zero) store_values<To, N>(dst, c, dim, x);
    }
}

// The piece at column c of a batch of rows.  A piece that ends behind the row is read from the row's last N values (skip of them
// belong to the piece before).
template <class T>
__device__ __forceinline__ void load_rows(const T* grad, int64_t ld, const int* from, int c, int dim, int skip, Piece<T>* x) {
    constexpr int N = Piece<T>::N;
    if (dim >= N) {
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) x[q] = load_piece(grad + (int64_t)from[q] * ld + (c - skip));
    } else {
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) {
            float v[N];
            load_values(grad + (int64_t)from[q] * ld, c, dim, 0.0f, v);
            x[q].set(v);
        }
    }
}
template <class T> __device__ __forceinline__ void drop_neighbours(int skip, Piece<T>* x) {
    if (!skip) return;
#pragma unroll
    for (int q = 0; q < SEG_BATCH; ++q) x[q].drop_first(skip);
}

// Blocks below zero_from: a group of 1 << log_tpr threads takes the chunk g of sorted positions; columns in slices of
// blockIdx.y.  A row that neither starts before the chunk nor goes on behind it is finished here; the part of a row that
// started before goes to part[g][0], of one that starts here and goes on to part[g][1].
// The other blocks write zeros to those of zero_each table rows that no position names (slice 0 alone).  A launch takes the blocks
// from block0 on.
template <class Tg, class To>
__global__ void __launch_bounds__(256) seg_sum_kernel(const Tg* __restrict__ grad, int64_t ld, const int* __restrict__ keys,
                                                      const int* __restrict__ pos, int64_t n, float scale, To* __restrict__ out,
                                                      int64_t n_rows, int dim, int64_t ld_out, int accumulate, float* __restrict__ part,
                                                      int chunk, int64_t chunks, int log_tpr, int block0, int zero_from, int log_zero, int zero_each) {
    const int block = block0 + (int)blockIdx.x;
    if (block >= zero_from) {
        if (blockIdx.y) return;
        __shared__ int64_t range[2];
        __shared__ int named[ZERO_ROWS];
        const int64_t r0 = (int64_t)(block - zero_from) * zero_each;
        if (threadIdx.x < ZERO_ROWS) named[threadIdx.x] = 0;
        if (threadIdx.x < 128) {
            const int64_t at = lower_bound_wave(keys, n, r0 + (threadIdx.x >> 6) * zero_each);
            if ((threadIdx.x & 63) == 0) range[threadIdx.x >> 6] = at;
        }
        __syncthreads();
        if (range[1] - range[0] <= 8 * 256) {
            for (int64_t p = range[0] + threadIdx.x; p < range[1]; p += 256) named[keys[p] - r0] = 1;
        } else if ((int)threadIdx.x < zero_each) {            // rows named many times: each looks for itself (131072 positions of 10 rows: 161 us to go through)
            const int64_t r = r0 + threadIdx.x;
            uint32_t a = (uint32_t)range[0], b = (uint32_t)range[1];
            while (a < b) {
                const uint32_t mid = a + ((b - a) >> 1);
                if (keys[mid] < r) a = mid + 1;
                else b = mid;
            }
            named[threadIdx.x] = a < (uint32_t)range[1] && keys[a] == r;
        }
        __syncthreads();
        zero_rows(named, out, r0, zero_each, n_rows, dim, ld_out, log_zero, 256);
        return;
    }
    constexpr int N = Piece<Tg>::N;
    const int64_t g = (int64_t)block * (256 >> log_tpr) + (threadIdx.x >> log_tpr);
    const int c = ((blockIdx.y << log_tpr) + (threadIdx.x & ((1 << log_tpr) - 1))) * N;
    if (g >= chunks || c >= dim) return;
    const int64_t p0 = g * chunk, p1 = min(p0 + chunk, n);
    const int before = p0 > 0 ? keys[p0 - 1] : -1, behind = p1 < n ? keys[p1] : -1;
    const int64_t pitch = part_pitch(dim);
    const int skip = dim >= N ? max(c + N - dim, 0) : 0;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    int key[SEG_BATCH], from[SEG_BATCH];
#pragma unroll
    for (int q = 0; q < SEG_BATCH; ++q) key[q] = keys[min(p0 + q, n - 1)];
#pragma unroll
    for (int q = 0; q < SEG_BATCH; ++q) from[q] = pos[min(p0 + q, n - 1)];
    for (int64_t b = p0; b < p1; b += SEG_BATCH) {
        if (key[0] >= n_rows) break;                     // the positions without a row come last
        // No branch around the loads: where one joins, the compiler waits for loads that are still under way (1000000 x 64 fp32
        // rows 220 us, so 149).
        Piece<Tg> x[SEG_BATCH];
        int next[SEG_BATCH];
        load_rows(grad, ld, from, c, dim, skip, x);
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) next[q] = keys[min(b + SEG_BATCH + q, n - 1)];
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) from[q] = pos[min(b + SEG_BATCH + q, n - 1)];
        drop_neighbours(skip, x);
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) {
            const int cur = key[q];
            if (b + q >= p1 || cur >= n_rows) break;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += x[q].get(e);
            const bool end = b + q + 1 == p1;
            if (!end && (q + 1 < SEG_BATCH ? key[q + 1] : next[0]) == cur) continue;
            const bool open = end && behind == cur;
            if (cur == before || open) store_values<float, N>(part + (g * 2 + (cur == before ? 0 : 1)) * pitch, c, pitch, acc);
            else put_row<To, N>(out + (int64_t)cur * ld_out, c, dim, scale, acc, accumulate);
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) key[q] = next[q];
    }
}

// Up to FEW_MAX positions in one launch, without a workspace: a block takes a position; where it is the first of its row, the
// rows of all positions that name the row are added in order, eight loads in flight.  The blocks behind write zeros to those of
// zero_each table rows that no position names.  Bound by the latency of two loads: 10 or 128 positions of 384 fp32 added to their
// rows 3 us, sorted first 8 and 10; 128 positions of one row 15 and 10.
static constexpr int FEW_MAX = 128;
template <class Tg, class To>
__global__ void __launch_bounds__(256) seg_few_kernel(const Tg* __restrict__ grad, int64_t ld, const int64_t* __restrict__ rows, int n, float scale,
                                                      To* __restrict__ out, int64_t n_rows, int dim, int64_t ld_out, int accumulate, int log_zero, int zero_each) {
    __shared__ int key[FEW_MAX];
    __shared__ int named[ZERO_ROWS];
    const int nt = (int)blockDim.x, tid = threadIdx.x, lane = tid & 63;
    for (int i = tid; i < FEW_MAX; i += nt) {
        const int64_t r = i < n ? rows[i] : -1;
        key[i] = r >= 0 && r < n_rows ? (int)r : -1;
    }
    if (tid < ZERO_ROWS) named[tid] = 0;
    __syncthreads();
    if ((int)blockIdx.x >= n) {
        if (blockIdx.y) return;
        const int64_t r0 = (int64_t)((int)blockIdx.x - n) * zero_each;
        for (int i = tid; i < n; i += nt)
            if (key[i] >= r0 && key[i] < r0 + zero_each) named[key[i] - r0] = 1;
        __syncthreads();
        zero_rows(named, out, r0, zero_each, n_rows, dim, ld_out, log_zero, nt);
        return;
    }
    constexpr int N = Piece<Tg>::N;
    const int mine = key[blockIdx.x], c = ((int)blockIdx.y * nt + tid) * N;
    if (mine < 0) return;
    unsigned long long same[2] = {__ballot(key[lane] == mine), __ballot(key[64 + lane] == mine)};
    if ((same[0] ? __builtin_ctzll(same[0]) : 64 + __builtin_ctzll(same[1])) != (int)blockIdx.x || c >= dim) return;
    const int skip = dim >= N ? max(c + N - dim, 0) : 0;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    while (same[0] | same[1]) {
        int from[SEG_BATCH], count = 0;
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) {
            const int half = same[0] ? 0 : 1;
            const bool some = (same[0] | same[1]) != 0;
            from[q] = some ? 64 * half + __builtin_ctzll(same[half]) : (int)blockIdx.x;
            if (some) same[half] &= same[half] - 1;
            count += some;
        }
        Piece<Tg> x[SEG_BATCH];
        load_rows(grad, ld, from, c, dim, skip, x);
        drop_neighbours(skip, x);
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) {
            if (q >= count) break;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += x[q].get(e);
        }
    }
    put_row<To, N>(out + (int64_t)mine * ld_out, c, dim, scale, acc, accumulate);
}

// The rows that cross chunks.  A block looks at JOIN_CHUNKS chunks and takes 256 columns (blockIdx.y): a row that starts
// in one of them and goes on has its parts, here and in the following chunks, added in order; up to SEG_BATCH parts by one
// wave (the block's waves take such rows side by side), more by all waves, a contiguous run of parts each.  What takes the
// time is the latency of the parts' loads (2 us a batch: other XCDs wrote them), so as many as possible are in flight, and
// a row's chunks are counted by a wave's probes at once (one after the other: 26 us, so 23, for 131072 rows of 2048 values
// named as often as words are).
static constexpr int JOIN_NT = 1024, JOIN_WAVES = JOIN_NT / 64, JOIN_CHUNKS = 32;

// parts [lo, hi) of the row that starts in chunk g: [g][1], then [g + 1][0], [g + 2][0], ...
template <int N> __device__ __forceinline__ void add_parts(const float* part, int64_t pitch, int64_t g, int64_t lo, int64_t hi, int c, float* acc) {
    for (int64_t j = lo; j < hi; j += SEG_BATCH) {
        float x[SEG_BATCH][N];
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q) {
            const int64_t k = min(j + q, hi - 1);
            __builtin_memcpy(x[q], part + ((g + k) * 2 + (k == 0 ? 1 : 0)) * pitch + c, N * 4);
        }
#pragma unroll
        for (int q = 0; q < SEG_BATCH; ++q)
            if (j + q < hi) {
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] += x[q][e];
            }
    }
}

template <class To>
__global__ void __launch_bounds__(JOIN_NT) seg_join_kernel(const int* __restrict__ keys, int64_t n, float scale, To* __restrict__ out, int64_t n_rows,
                                                           int dim, int64_t ld_out, int accumulate, const float* __restrict__ part, int chunk,
                                                           int64_t chunks) {
    constexpr int N = 4;
    __shared__ float sums[JOIN_WAVES][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.y * 256 + lane * N;
    const bool active = c < dim;
    const int64_t pitch = part_pitch(dim);
    const int64_t first = (int64_t)blockIdx.x * JOIN_CHUNKS;
    // key at the start of chunk j
    auto border = [&](int64_t j) { return keys[min(j * chunk, n - 1)]; };
    int row;                             // of the last position of chunk first + lane
    bool starts, many;
    {
        const int64_t g = first + min(lane, JOIN_CHUNKS - 1), p1 = min((g + 1) * chunk, n);
        row = keys[p1 - 1];
        const int next = border(g + 1), prev = keys[max(p1 - chunk - 1, (int64_t)0)], far = border(g + SEG_BATCH);
        starts = lane < JOIN_CHUNKS && g + 1 < chunks && row < n_rows && next == row && !(g > 0 && prev == row);
        many = starts && g + SEG_BATCH < chunks && far == row;
    }
    const unsigned long long few = __ballot(starts && !many), long_ones = __ballot(many);
    int turn = 0;
    for (unsigned long long todo = few; todo; todo &= todo - 1, ++turn) {
        if (turn % JOIN_WAVES != wave) continue;
        const int at = __builtin_ctzll(todo), cur = __shfl(row, at);
        const int64_t g = first + at;
        const int count = __builtin_ctzll(~__ballot(lane == 0 || (lane < SEG_BATCH && g + lane < chunks && border(g + lane) == cur)));
        if (!active) continue;
        float acc[N] = {0.0f, 0.0f, 0.0f, 0.0f};
        add_parts<N>(part, pitch, g, 0, count, c, acc);
        put_row<To, N>(out + (int64_t)cur * ld_out, c, dim, scale, acc, accumulate);
    }
    for (unsigned long long todo = long_ones; todo; todo &= todo - 1) {
        const int at = __builtin_ctzll(todo), cur = __shfl(row, at);
        const int64_t g = first + at;
        // the chunks from g on that begin with the row (g itself counts): 64 probes a step
        uint32_t count = SEG_BATCH, most = (uint32_t)(chunks - g);             // it lies in [count, most]
        while (count < most) {
            const uint32_t step = (most - count + 63) >> 6, probe = count + step * (lane + 1) - 1;
            const uint32_t same = (uint32_t)__popcll(__ballot(probe < most && border(g + probe) == cur));
            most = min(most, count + step * (same + 1) - 1);
            count += step * same;
        }
        const uint32_t per = (count + JOIN_WAVES - 1) / JOIN_WAVES, lo = min(wave * per, count), hi = min(lo + per, count);
        float acc[N] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (active) add_parts<N>(part, pitch, g, lo, hi, c, acc);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < N; ++e) sums[wave][lane * N + e] = acc[e];
        __syncthreads();
        if (wave == 0 && active) {
            for (int w = 1; w < JOIN_WAVES; ++w)
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] += sums[w][lane * N + e];
            put_row<To, N>(out + (int64_t)cur * ld_out, c, dim, scale, acc, accumulate);
        }
    }
}

// threads of a group that takes a row: a power of two that covers the row's pieces, at most a block
static int log_threads(int pieces) {
    int l = 0;
    while (l < 8 && (1 << l) < pieces) ++l;
    return l;
}

int launch_lookup(const void* table, int table_type, int64_t n_rows, int dim, int64_t ld, const int64_t* rows, int64_t n, float scale,
                  void* out, int out_type, int64_t ld_out, hipStream_t s) {
    if (n <= 0) return VDB_OK;
    return with_type(table_type, [&](auto* ti) -> int {
        return with_type(out_type, [&](auto* to) -> int {
            typedef std::remove_pointer_t<decltype(ti)> Ti;
            typedef std::remove_pointer_t<decltype(to)> To;
            // rows for one piece a thread, for four where that still leaves eight blocks a CU (88769 x 1672 fp32 by a block a
            // row, two pieces a thread: 185 us, so 164)
            const int64_t pieces = (dim + Piece<Ti>::N - 1) / Piece<Ti>::N;
            const int each = n * pieces >= (int64_t)8 * ctx().num_cus * LOOKUP_AHEAD * LOOKUP_NT ? LOOKUP_AHEAD : 1;
            const int take = ceil_div(each * LOOKUP_NT, pieces);
            const uint32_t inverse = pieces > 1 ? (uint32_t)((((int64_t)1 << 32) + pieces - 1) / pieces) : 0;
            const int64_t most = ((int64_t)1 << 23) * take;           // a launch holds fewer than 2^32 threads
            for (int64_t i = 0; i < n; i += most) {
                const int64_t m = std::min(most, n - i);
                hipLaunchKernelGGL((lookup_kernel<Ti, To>), dim3(ceil_div(m, take)), dim3(LOOKUP_NT), 0, s, (const Ti*)table, n_rows, dim, ld, rows + i, m,
                                   scale, (To*)out + i * ld_out, ld_out, take, (uint32_t)pieces, inverse);
                VDB_HIP(hipGetLastError());
            }
            return VDB_OK;
        });
    });
}

// ---------------------------------------------------------------- workspace of the gradient
struct GradWork {
    int *keys[2], *pos[2], *hist, *totals;
    float* part;
    int64_t bytes;
};
static int seg_chunk(int64_t n, int dim) {
    if (n <= 32) return 32;                                           // a single chunk needs no second launch
    const int64_t lanes = n * ((dim + 3) / 4);
    // 131072 x 2048: parts written and joined cost 37 us with chunks of 32, 20 us with 64, the sums 348 and 352 us; 131072 x 64 as
    // a whole 59 us with 256 K lanes or more, 54 with 128 K, 56 with 64 K
    for (int chunk = 64; chunk > 8; chunk >>= 1)
        if (lanes / chunk >= (int64_t)128 * 1024) return chunk;
    return 8;
}
// Whether the whole table is zeroed beside the sort, and the named rows written over it: where those are few (10240 x 384
// into 100000 rows: 28 us with the sort, which takes 12 by itself), else the sums' launch writes zeros to the other rows alone.
static bool fill_first(int64_t n, int64_t n_rows) { return n > 0 && n <= n_rows / 4; }
static GradWork grad_work(void* base, int64_t n, int64_t n_rows, int dim) {
    const SortPlan p = sort_plan(n, n_rows);
    GradWork w{};
    char* at = (char*)base;
    auto take = [&](int64_t bytes) {
        char* here = at;
        at += round_up64(bytes, 256);
        return here;
    };
    for (int i = 0; i < 2; ++i) w.keys[i] = (int*)take(n * 4);
    for (int i = 0; i < 2; ++i) w.pos[i] = (int*)take(n * 4);
    if (n > COUNT_MAX) {
        w.hist = (int*)take(((int64_t)p.blocks << p.bits) * 4);
        w.totals = (int*)take(((int64_t)1 << p.bits) * 4);
    }
    const int chunk = seg_chunk(n, dim);
    w.part = (float*)take((n + chunk - 1) / chunk * 2 * part_pitch(dim) * 4);
    w.bytes = at - (char*)base;
    return w;
}

static int launch_sort(const int64_t* rows, int64_t n, int64_t n_rows, const GradWork& w, Fill fill, const int** keys, const int** pos, hipStream_t s) {
    const SortPlan p = sort_plan(n, n_rows);
    const int bins = 1 << p.bits;
    *keys = w.keys[(p.passes + 1) & 1];
    *pos = w.pos[(p.passes + 1) & 1];
    if (n <= 0) return VDB_OK;
    // Zeros of 32 to 128 KB a block, two blocks a CU where there are that many, for rows that lie back to back (697 MB by 1024 threads:
    // 133 us, with 32 or 256 KB a block 139 and 153, by two blocks a CU in turn 164); else blocks that go through the rows in turn.
    auto fill_blocks = [&](int64_t lo, int64_t hi, int threads) {
        fill.r0 = lo;
        fill.r1 = hi;
        const int64_t bytes = (hi - lo) * fill.units * 2;
        if (fill.units != fill.ld) return (int)std::min<int64_t>((bytes + 32767) / 32768, (int64_t)ctx().num_cus * 2048 / threads);
        const int64_t share = std::min(std::max<int64_t>(bytes / (2 * ctx().num_cus), 1 << 15), (int64_t)1 << 17);
        return (int)std::min<int64_t>((bytes + share - 1) / share, 1 << 20);
    };
    const int64_t fill_end = fill.out ? n_rows : 0;
    if (n <= COUNT_MAX) {
        const int per = std::min(std::max(ceil_div(n, COUNT_LANES * ctx().num_cus), 1), 3), blocks = ceil_div(n, COUNT_LANES * per);
        const int extra = fill_blocks(0, fill_end, COUNT_NT);
        auto kernel = per == 1 ? sort_count_kernel<1> : per == 2 ? sort_count_kernel<2> : sort_count_kernel<3>;
        hipLaunchKernelGGL(kernel, dim3(blocks + extra), dim3(COUNT_NT), (size_t)round_up64(n, 4) * 4, s, rows, (int)n, n_rows, blocks, w.keys[0], w.pos[0], fill);
        VDB_HIP(hipGetLastError());
        *keys = w.keys[0];
        *pos = w.pos[0];
        return VDB_OK;
    }
    const int shares = 2 * p.passes;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int64_t* src_rows = pass == 0 ? rows : nullptr;
        const int* src_keys = pass == 0 ? nullptr : w.keys[(pass + 1) & 1];
        const int* src_pos = pass == 0 ? nullptr : w.pos[(pass + 1) & 1];
        int extra = fill_blocks(fill_end * (2 * pass) / shares, fill_end * (2 * pass + 1) / shares, SORT_NT);
        hipLaunchKernelGGL(sort_hist_kernel, dim3(p.blocks + extra), dim3(SORT_NT), bins * 4, s, src_rows, src_keys, n, n_rows, pass * p.bits, p.bits,
                           p.wave_keys, w.hist, p.blocks, fill);
        VDB_HIP(hipGetLastError());
        hipLaunchKernelGGL(sort_scan_kernel, dim3(bins), dim3(64), 0, s, w.hist, p.blocks, w.totals);
        VDB_HIP(hipGetLastError());
        extra = fill_blocks(fill_end * (2 * pass + 1) / shares, fill_end * (2 * pass + 2) / shares, SORT_NT);
        hipLaunchKernelGGL(sort_scatter_kernel, dim3(p.blocks + extra), dim3(SORT_NT), SORT_WAVES * bins * 4, s, src_rows, src_keys, src_pos,
                           n, n_rows, pass * p.bits, p.bits, p.wave_keys, w.hist, w.totals, w.keys[pass & 1], w.pos[pass & 1], p.blocks, fill);
        VDB_HIP(hipGetLastError());
    }
    return VDB_OK;
}

// whether few positions go by themselves: the zeros of a large table are written faster by the other form (10 positions into 10000 x 384 fp32
// 6 us, 9 sorted first, 30000 x 384 12 and 13, 100000 x 384 28 and 26)
static const int64_t FEW_TABLE = (int64_t)1 << 24;
static bool by_few(int64_t n, int64_t n_rows, int dim) { return n <= FEW_MAX && n_rows <= FEW_TABLE / dim; }

static int launch_few(const void* grad, int grad_type, int64_t ld, const int64_t* rows, int n, float scale, void* out, int out_type, int64_t n_rows,
                      int dim, int64_t ld_out, int accumulate, hipStream_t s) {
    return with_type(out_type, [&](auto* to) -> int {
        typedef std::remove_pointer_t<decltype(to)> To;
        return with_type(grad_type, [&](auto* tg) -> int {
            typedef std::remove_pointer_t<decltype(tg)> Tg;
            const int pieces = (dim + Piece<Tg>::N - 1) / Piece<Tg>::N, l = std::min(std::max(log_threads(pieces), 6), 8), nt = 1 << l;
            const int lz = std::min(log_threads((dim + Piece<To>::N - 1) / Piece<To>::N), l);
            const int zero_each = std::min(std::max(2048 / dim, 1), ZERO_ROWS), zeros = accumulate ? 0 : ceil_div(n_rows, zero_each);
            if (n + zeros == 0) return VDB_OK;
            hipLaunchKernelGGL((seg_few_kernel<Tg, To>), dim3(n + zeros, ceil_div(pieces, nt)), dim3(nt), 0, s, (const Tg*)grad, ld, rows, n, scale,
                               (To*)out, n_rows, dim, ld_out, accumulate, lz, zero_each);
            VDB_HIP(hipGetLastError());
            return VDB_OK;
        });
    });
}

static int launch_lookup_grad(const void* grad, int grad_type, int64_t ld, const int64_t* rows, int64_t n, float scale, void* out, int out_type,
                              int64_t n_rows, int dim, int64_t ld_out, int accumulate, void* work, hipStream_t s) {
    const GradWork w = grad_work(work, n, n_rows, dim);
    const int *keys = nullptr, *pos = nullptr;
    const bool filled = !accumulate && fill_first(n, n_rows);
    const int half = out_type == VDB_VALUE_F32 ? 2 : 1;              // 16-bit units of a value
    const Fill fill{filled ? (uint16_t*)out : nullptr, 0, 0, (int64_t)dim * half, ld_out * half, log_threads((dim * half + 7) / 8)};
    VDB_TRY(launch_sort(rows, n, n_rows, w, fill, &keys, &pos, s));
    const int chunk = seg_chunk(n, dim);
    const int64_t chunks = (n + chunk - 1) / chunk;
    return with_type(out_type, [&](auto* to) -> int {
        typedef std::remove_pointer_t<decltype(to)> To;
        return with_type(grad_type, [&](auto* tg) -> int {
            typedef std::remove_pointer_t<decltype(tg)> Tg;
            const int pieces = (dim + Piece<Tg>::N - 1) / Piece<Tg>::N, l = log_threads(pieces);
            const int lz = log_threads((dim + Piece<To>::N - 1) / Piece<To>::N);
            // two blocks a CU for the zeros of small tables (1963 x 469 bf16 into 4316 rows: 22 us with 64 rows each, so 18)
            const int zero_each = (int)std::min<int64_t>(std::max<int64_t>(n_rows / (2 * ctx().num_cus), 8), ZERO_ROWS);
            const int sums = ceil_div(chunks, 256 >> l), zeros = accumulate || filled ? 0 : ceil_div(n_rows, zero_each);
            const int most = 1 << 23;                                      // a launch holds fewer than 2^32 threads
            for (int block0 = 0; block0 < sums + zeros; block0 += most) {
                hipLaunchKernelGGL((seg_sum_kernel<Tg, To>), dim3(std::min(sums + zeros - block0, most), ceil_div(pieces, 1 << l)), dim3(256), 0, s,
                                   (const Tg*)grad, ld, keys, pos, n, scale, (To*)out, n_rows, dim, ld_out, accumulate, w.part, chunk, chunks, l, block0,
                                   sums, lz, zero_each);
                VDB_HIP(hipGetLastError());
            }
            if (chunks > 1) {
                hipLaunchKernelGGL((seg_join_kernel<To>), dim3(ceil_div(chunks - 1, JOIN_CHUNKS), ceil_div(dim, 256)), dim3(JOIN_NT), 0, s, keys, n, scale,
                                   (To*)out, n_rows, dim, ld_out, accumulate, w.part, chunk, chunks);
                VDB_HIP(hipGetLastError());
            }
            return VDB_OK;
        });
    });
}

}  // namespace vdb

using namespace vdb;

static const int64_t LOOKUP_MAX = ((int64_t)1 << 31) - 1;

int vdb_lookup_dev(const void* d_table, int table_type, int64_t n_rows, int dim, int64_t ld, const int64_t* d_rows, int64_t n, float scale,
                   void* d_out, int out_type, int64_t ld_out, void* stream) {
    VDB_REQUIRE(valid_type(table_type) && valid_type(out_type), "unknown value type (table %d, out %d)", table_type, out_type);
    VDB_REQUIRE(n >= 0 && n < LOOKUP_MAX && n_rows >= 0 && n_rows < LOOKUP_MAX && dim >= 1 && ld >= 0 && ld_out >= dim,
                "bad sizes for a lookup: %lld of %lld rows, dimension %d, leading dimensions %lld and %lld", (long long)n, (long long)n_rows, dim,
                (long long)ld, (long long)ld_out);
    VDB_REQUIRE(n == 0 || (d_rows && d_out && (d_table || n_rows == 0)), "null pointer in a lookup of %lld rows", (long long)n);
    if (n == 0) return VDB_OK;
    VDB_TRY(ensure_init());
    (void)hipSetDevice(ctx().device);
    return launch_lookup(d_table, table_type, n_rows, dim, ld, d_rows, n, scale, d_out, out_type, ld_out, (hipStream_t)stream);
}

static int check_grad_sizes(int64_t n, int64_t n_rows, int dim) {
    // what the sort's 32-bit keys, positions and counts hold
    const int64_t most = (int64_t)1 << 30;
    VDB_REQUIRE(n >= 0 && n < most && n_rows >= 0 && n_rows < most && dim >= 1 && dim <= 1 << 23,
                "bad sizes for a lookup gradient: %lld rows into %lld, dimension %d", (long long)n, (long long)n_rows, dim);
    return VDB_OK;
}

static int64_t grad_bytes(int64_t n, int64_t n_rows, int dim) { return by_few(n, n_rows, dim) ? 0 : grad_work(nullptr, n, n_rows, dim).bytes; }

int vdb_lookup_grad_workspace(int64_t n, int64_t n_rows, int dim, int64_t* bytes) {
    VDB_REQUIRE(bytes, "null pointer for the workspace size");
    VDB_TRY(check_grad_sizes(n, n_rows, dim));
    *bytes = grad_bytes(n, n_rows, dim);
    return VDB_OK;
}

int vdb_lookup_grad_dev(const void* d_grad, int grad_type, int64_t ld, const int64_t* d_rows, int64_t n, float scale, void* d_table_grad,
                        int table_type, int64_t n_rows, int dim, int64_t ld_table, int accumulate, void* d_work, int64_t work_bytes, void* stream) {
    VDB_REQUIRE(valid_type(grad_type) && valid_type(table_type), "unknown value type (grad %d, table_grad %d)", grad_type, table_type);
    VDB_TRY(check_grad_sizes(n, n_rows, dim));
    VDB_REQUIRE(ld >= 0 && ld_table >= dim, "bad leading dimensions %lld and %lld for a lookup gradient of dimension %d", (long long)ld,
                (long long)ld_table, dim);
    VDB_REQUIRE((n == 0 || (d_grad && d_rows)) && (n_rows == 0 || d_table_grad), "null pointer in a lookup gradient");
    const int64_t need = grad_bytes(n, n_rows, dim);
    VDB_REQUIRE(work_bytes >= need && (d_work || need == 0), "the workspace of %lld bytes is too small for this lookup gradient (%lld needed)",
                (long long)work_bytes, (long long)need);
    VDB_REQUIRE(aligned_work(d_work), "a workspace begins at a multiple of 16 bytes");
    if (n_rows == 0 || (n == 0 && accumulate)) return VDB_OK;
    VDB_TRY(ensure_init());
    (void)hipSetDevice(ctx().device);
    if (by_few(n, n_rows, dim) || (accumulate && n <= FEW_MAX))
        return launch_few(d_grad, grad_type, ld, d_rows, (int)n, scale, d_table_grad, table_type, n_rows, dim, ld_table, accumulate, (hipStream_t)stream);
    return launch_lookup_grad(d_grad, grad_type, ld, d_rows, n, scale, d_table_grad, table_type, n_rows, dim, ld_table, accumulate, d_work,
                              (hipStream_t)stream);
}
