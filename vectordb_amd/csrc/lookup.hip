// Rows of a table by number (vdb_lookup_dev) and the gradient of that table (vdb_lookup_grad_dev).
//
// lookup: out[i] = scale * table[rows[i]].  A copy of n rows; what bounds it is HBM traffic, n * dim values read and
// written.  A group of threads (a power of two, up to a block) takes a row in 16-byte pieces.
//
// gradient: table_grad[r] = scale * sum over {i : rows[i] == r} of grad[i].  The positions i are sorted by row number
// with a stable radix sort, so the members of a row lie side by side in ascending i; the sorted positions are cut into
// chunks of SEG_CHUNK, a group of threads adds the rows of a chunk in order, and a row that crosses chunks has its
// parts added in chunk order by a second launch.  No atomics on values: the order of every sum is fixed by the row
// numbers.  Bound: grad read once, table_grad written once (rows without members as zeros).
#include "vdb_internal.h"
#include "values.h"

#include <algorithm>

namespace vdb {

// ---------------------------------------------------------------- lookup
template <class Ti, class To>
__global__ void __launch_bounds__(256) lookup_kernel(const Ti* __restrict__ table, int64_t n_rows, int dim, int64_t ld,
                                                     const int64_t* __restrict__ rows, int64_t n, float scale, To* __restrict__ out,
                                                     int64_t ld_out, int log_tpr) {
    constexpr int N = Piece<Ti>::N;
    const int tpr = 1 << log_tpr;
    const int64_t i = (int64_t)blockIdx.x * (256 >> log_tpr) + (threadIdx.x >> log_tpr);
    if (i >= n) return;
    const int64_t r = rows[i];
    const bool known = r >= 0 && r < n_rows;
    const Ti* src = table + (known ? r : 0) * ld;
    To* dst = out + i * ld_out;
    for (int c = (threadIdx.x & (tpr - 1)) * N; c < dim; c += tpr * N) {
        float x[N];
        if (known) {
            load_values(src, c, dim, 0.0f, x);
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] *= scale;
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = 0.0f;
        }
        store_values<To, N>(dst, c, dim, x);
    }
}

// ---------------------------------------------------------------- stable radix sort of the positions by row number
static constexpr int SORT_NT = 256, SORT_WAVES = SORT_NT / 64, SORT_MAX_BITS = 10;

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
    // 512 keys a wave until there are 1024 blocks, more beyond
    p.wave_keys = std::max<int64_t>(512, round_up64((n + 1024 * SORT_WAVES - 1) / (1024 * SORT_WAVES), 64));
    p.blocks = (int)((n + p.wave_keys * SORT_WAVES - 1) / (p.wave_keys * SORT_WAVES));
    return p;
}

__device__ __forceinline__ int key_of(const int64_t* rows, const int* keys, int64_t i, int64_t n_rows) {
    if (!rows) return keys[i];
    const int64_t r = rows[i];
    return (int)(r >= 0 && r < n_rows ? r : n_rows);
}

// hist[digit][block]
__global__ void __launch_bounds__(SORT_NT) sort_hist_kernel(const int64_t* __restrict__ rows, const int* __restrict__ keys, int64_t n,
                                                            int64_t n_rows, int shift, int bits, int64_t wave_keys, int* __restrict__ hist) {
    extern __shared__ int cnt[];
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += SORT_NT) cnt[d] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * wave_keys * SORT_WAVES, hi = min(lo + wave_keys * SORT_WAVES, n);
    for (int64_t i = lo + threadIdx.x; i < hi; i += SORT_NT) atomicAdd(&cnt[(key_of(rows, keys, i, n_rows) >> shift) & (bins - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += SORT_NT) hist[(int64_t)d * gridDim.x + blockIdx.x] = cnt[d];
}

// one wave per digit: exclusive prefix of its counts over the blocks, and their total
__global__ void __launch_bounds__(64) sort_scan_kernel(int* __restrict__ hist, int blocks, int* __restrict__ totals) {
    int* h = hist + (int64_t)blockIdx.x * blocks;
    int run = 0;
    for (int b0 = 0; b0 < blocks; b0 += 64) {
        const int b = b0 + threadIdx.x;
        const int v = b < blocks ? h[b] : 0;
        int s = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(s, o);
            if ((int)threadIdx.x >= o) s += t;
        }
        if (b < blocks) h[b] = run + s - v;
        run += __shfl(s, 63);
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// lanes of the wave whose digit equals this lane's (lanes without a key are in nobody's set)
__device__ __forceinline__ unsigned long long same_digit(int d, int bits, bool have) {
    unsigned long long m = __ballot(have);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long one = __ballot((d >> b) & 1);
        m &= ((d >> b) & 1) ? one : ~one;
    }
    return m;
}

__global__ void __launch_bounds__(SORT_NT) sort_scatter_kernel(const int64_t* __restrict__ rows, const int* __restrict__ keys,
                                                               const int* __restrict__ pos, int64_t n, int64_t n_rows, int shift, int bits,
                                                               int64_t wave_keys, const int* __restrict__ hist, const int* __restrict__ totals,
                                                               int* __restrict__ keys_out, int* __restrict__ pos_out) {
    extern __shared__ int lds[];
    const int bins = 1 << bits;
    int* start = lds;                         // [SORT_WAVES][bins]
    int* scan = lds + SORT_WAVES * bins;      // [SORT_NT]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int d = tid; d < SORT_WAVES * bins; d += SORT_NT) start[d] = 0;
    __syncthreads();
    const int64_t lo = ((int64_t)blockIdx.x * SORT_WAVES + wave) * wave_keys, hi = min(lo + wave_keys, n);
    int* mine = start + wave * bins;
    for (int64_t i = lo + lane; i < hi; i += 64) atomicAdd(&mine[(key_of(rows, keys, i, n_rows) >> shift) & (bins - 1)], 1);
    // exclusive prefix of the digit totals: a contiguous run of digits per thread, then over the threads
    const int per = (bins + SORT_NT - 1) / SORT_NT;
    int sum = 0;
    for (int j = 0; j < per; ++j) {
        const int d = tid * per + j;
        if (d < bins) sum += totals[d];
    }
    scan[tid] = sum;
    __syncthreads();
    for (int o = 1; o < SORT_NT; o <<= 1) {
        const int t = tid >= o ? scan[tid - o] : 0;
        __syncthreads();
        scan[tid] += t;
        __syncthreads();
    }
    int run = tid > 0 ? scan[tid - 1] : 0;
    for (int j = 0; j < per; ++j) {
        const int d = tid * per + j;
        if (d >= bins) break;
        int at = run + hist[(int64_t)d * gridDim.x + blockIdx.x];
        run += totals[d];
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
        const unsigned long long m = same_digit(d, bits, have);
        if (have) {
            const int rank = __popcll(m & ((1ull << lane) - 1));
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

// ---------------------------------------------------------------- sums of the sorted rows
static constexpr int SEG_CHUNK = 32;

template <class To, int N> __device__ __forceinline__ void put_row(To* row, int c, int dim, float scale, const float* acc, bool accumulate) {
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = scale * acc[e];
    if (accumulate) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (c + e < dim) x[e] = (float)row[c + e] + x[e];
    }
    store_values<To, N>(row, c, dim, x);
}

// A group of 1 << log_tpr threads takes the chunk of SEG_CHUNK sorted positions g; columns in slices of blockIdx.y.
// A row that neither starts before the chunk nor goes on behind it is finished here; the part of a row that started
// before goes to part[g][0], of one that starts here and goes on to part[g][1].
template <class Tg, class To>
__global__ void __launch_bounds__(256) seg_sum_kernel(const Tg* __restrict__ grad, int64_t ld, const int* __restrict__ keys,
                                                      const int* __restrict__ pos, int64_t n, float scale, To* __restrict__ out,
                                                      int64_t n_rows, int dim, int64_t ld_out, int accumulate, float* __restrict__ part,
                                                      int64_t chunks, int log_tpr) {
    constexpr int N = Piece<Tg>::N;
    const int64_t g = (int64_t)blockIdx.x * (256 >> log_tpr) + (threadIdx.x >> log_tpr);
    const int c = ((blockIdx.y << log_tpr) + (threadIdx.x & ((1 << log_tpr) - 1))) * N;
    if (g >= chunks || c >= dim) return;
    const int64_t p0 = g * SEG_CHUNK, p1 = min(p0 + SEG_CHUNK, n);
    const int before = p0 > 0 ? keys[p0 - 1] : -1, behind = p1 < n ? keys[p1] : -1;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    int cur = keys[p0];
    for (int64_t p = p0; p < p1 && cur < n_rows; ++p) {
        float x[N];
        load_values(grad + (int64_t)pos[p] * ld, c, dim, 0.0f, x);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += x[e];
        const int next = p + 1 < p1 ? keys[p + 1] : -1;
        if (next == cur) continue;
        const bool open = p + 1 == p1 && behind == cur;
        if (cur == before || open) store_values<float, N>(part + (g * 2 + (cur == before ? 0 : 1)) * dim, c, dim, acc);
        else put_row<To, N>(out + (int64_t)cur * ld_out, c, dim, scale, acc, accumulate);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.0f;
        cur = next < 0 ? cur : next;
    }
}

// The rows that cross chunks: the chunk in which such a row starts adds the parts of the following ones in order.
template <class To>
__global__ void __launch_bounds__(256) seg_join_kernel(const int* __restrict__ keys, int64_t n, float scale, To* __restrict__ out, int64_t n_rows,
                                                       int dim, int64_t ld_out, int accumulate, const float* __restrict__ part, int64_t chunks,
                                                       int log_tpr) {
    constexpr int N = 4;
    const int64_t g = (int64_t)blockIdx.x * (256 >> log_tpr) + (threadIdx.x >> log_tpr);
    const int c = ((blockIdx.y << log_tpr) + (threadIdx.x & ((1 << log_tpr) - 1))) * N;
    if (g + 1 >= chunks || c >= dim) return;
    const int64_t p0 = g * SEG_CHUNK;
    const int cur = keys[p0 + SEG_CHUNK - 1];
    if (cur >= n_rows || keys[p0 + SEG_CHUNK] != cur || (p0 > 0 && keys[p0 - 1] == cur)) return;
    float acc[N];
    load_values(part + (g * 2 + 1) * dim, c, dim, 0.0f, acc);
    for (int64_t h = g + 1; h < chunks; ++h) {
        float x[N];
        load_values(part + h * 2 * dim, c, dim, 0.0f, x);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += x[e];
        const int64_t end = (h + 1) * SEG_CHUNK;
        if (end >= n || keys[end] != cur) break;
    }
    put_row<To, N>(out + (int64_t)cur * ld_out, c, dim, scale, acc, accumulate);
}

// zeros for the rows that no position names
template <class To>
__global__ void __launch_bounds__(256) seg_zero_kernel(const int* __restrict__ keys, int64_t n, To* __restrict__ out, int64_t n_rows, int dim,
                                                       int64_t ld_out, int log_tpr) {
    constexpr int N = Piece<To>::N;
    const int64_t r = (int64_t)blockIdx.x * (256 >> log_tpr) + (threadIdx.x >> log_tpr);
    if (r >= n_rows) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < r) lo = mid + 1;
        else hi = mid;
    }
    if (lo < n && keys[lo] == r) return;
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = 0.0f;
    for (int c = (threadIdx.x & ((1 << log_tpr) - 1)) * N; c < dim; c += N << log_tpr) store_values<To, N>(out + r * ld_out, c, dim, x);
}

// threads per row: a power of two that covers the row's pieces, at most a block
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
            const int l = log_threads((dim + Piece<Ti>::N - 1) / Piece<Ti>::N);
            hipLaunchKernelGGL((lookup_kernel<Ti, To>), dim3(ceil_div(n, 256 >> l)), dim3(256), 0, s, (const Ti*)table, n_rows, dim, ld, rows, n,
                               scale, (To*)out, ld_out, l);
            VDB_HIP(hipGetLastError());
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
static GradWork grad_work(void* base, int64_t n, int64_t n_rows, int dim) {
    const SortPlan p = sort_plan(n, n_rows);
    GradWork w;
    char* at = (char*)base;
    auto take = [&](int64_t bytes) {
        char* here = at;
        at += round_up64(bytes, 256);
        return here;
    };
    for (int i = 0; i < 2; ++i) w.keys[i] = (int*)take(n * 4);
    for (int i = 0; i < 2; ++i) w.pos[i] = (int*)take(n * 4);
    w.hist = (int*)take(((int64_t)p.blocks << p.bits) * 4);
    w.totals = (int*)take(((int64_t)1 << p.bits) * 4);
    w.part = (float*)take((n + SEG_CHUNK - 1) / SEG_CHUNK * 2 * dim * 4);
    w.bytes = at - (char*)base;
    return w;
}

static int launch_lookup_grad(const void* grad, int grad_type, int64_t ld, const int64_t* rows, int64_t n, float scale, void* out, int out_type,
                              int64_t n_rows, int dim, int64_t ld_out, int accumulate, void* work, hipStream_t s) {
    const GradWork w = grad_work(work, n, n_rows, dim);
    const SortPlan p = sort_plan(n, n_rows);
    const int bins = 1 << p.bits;
    for (int pass = 0; pass < p.passes && n > 0; ++pass) {
        const int64_t* src_rows = pass == 0 ? rows : nullptr;
        const int* src_keys = pass == 0 ? nullptr : w.keys[(pass + 1) & 1];
        const int* src_pos = pass == 0 ? nullptr : w.pos[(pass + 1) & 1];
        hipLaunchKernelGGL(sort_hist_kernel, dim3(p.blocks), dim3(SORT_NT), bins * 4, s, src_rows, src_keys, n, n_rows, pass * p.bits, p.bits,
                           p.wave_keys, w.hist);
        VDB_HIP(hipGetLastError());
        hipLaunchKernelGGL(sort_scan_kernel, dim3(bins), dim3(64), 0, s, w.hist, p.blocks, w.totals);
        VDB_HIP(hipGetLastError());
        hipLaunchKernelGGL(sort_scatter_kernel, dim3(p.blocks), dim3(SORT_NT), (SORT_WAVES * bins + SORT_NT) * 4, s, src_rows, src_keys, src_pos, n,
                           n_rows, pass * p.bits, p.bits, p.wave_keys, w.hist, w.totals, w.keys[pass & 1], w.pos[pass & 1]);
        VDB_HIP(hipGetLastError());
    }
    const int* keys = w.keys[(p.passes + 1) & 1];
    const int* pos = w.pos[(p.passes + 1) & 1];
    const int64_t chunks = (n + SEG_CHUNK - 1) / SEG_CHUNK;
    return with_type(out_type, [&](auto* to) -> int {
        typedef std::remove_pointer_t<decltype(to)> To;
        if (!accumulate) {
            const int l = log_threads((dim + Piece<To>::N - 1) / Piece<To>::N);
            hipLaunchKernelGGL((seg_zero_kernel<To>), dim3(ceil_div(n_rows, 256 >> l)), dim3(256), 0, s, keys, n, (To*)out, n_rows, dim, ld_out, l);
            VDB_HIP(hipGetLastError());
        }
        if (n <= 0) return VDB_OK;
        return with_type(grad_type, [&](auto* tg) -> int {
            typedef std::remove_pointer_t<decltype(tg)> Tg;
            const int pieces = (dim + Piece<Tg>::N - 1) / Piece<Tg>::N, l = log_threads(pieces);
            hipLaunchKernelGGL((seg_sum_kernel<Tg, To>), dim3(ceil_div(chunks, 256 >> l), ceil_div(pieces, 1 << l)), dim3(256), 0, s, (const Tg*)grad,
                               ld, keys, pos, n, scale, (To*)out, n_rows, dim, ld_out, accumulate, w.part, chunks, l);
            VDB_HIP(hipGetLastError());
            const int joins = (dim + 3) / 4, lj = log_threads(joins);
            hipLaunchKernelGGL((seg_join_kernel<To>), dim3(ceil_div(chunks, 256 >> lj), ceil_div(joins, 1 << lj)), dim3(256), 0, s, keys, n, scale,
                               (To*)out, n_rows, dim, ld_out, accumulate, w.part, chunks, lj);
            VDB_HIP(hipGetLastError());
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
    VDB_REQUIRE(n >= 0 && n < LOOKUP_MAX && n_rows >= 0 && n_rows < LOOKUP_MAX && dim >= 1,
                "bad sizes for a lookup gradient: %lld rows into %lld, dimension %d", (long long)n, (long long)n_rows, dim);
    return VDB_OK;
}

int vdb_lookup_grad_workspace(int64_t n, int64_t n_rows, int dim, int64_t* bytes) {
    VDB_REQUIRE(bytes, "null pointer for the workspace size");
    VDB_TRY(check_grad_sizes(n, n_rows, dim));
    *bytes = grad_work(nullptr, n, n_rows, dim).bytes;
    return VDB_OK;
}

int vdb_lookup_grad_dev(const void* d_grad, int grad_type, int64_t ld, const int64_t* d_rows, int64_t n, float scale, void* d_table_grad,
                        int table_type, int64_t n_rows, int dim, int64_t ld_table, int accumulate, void* d_work, int64_t work_bytes, void* stream) {
    VDB_REQUIRE(valid_type(grad_type) && valid_type(table_type), "unknown value type (grad %d, table_grad %d)", grad_type, table_type);
    VDB_TRY(check_grad_sizes(n, n_rows, dim));
    VDB_REQUIRE(ld >= 0 && ld_table >= dim, "bad leading dimensions %lld and %lld for a lookup gradient of dimension %d", (long long)ld,
                (long long)ld_table, dim);
    VDB_REQUIRE((n == 0 || (d_grad && d_rows)) && (n_rows == 0 || d_table_grad), "null pointer in a lookup gradient");
    const int64_t need = grad_work(nullptr, n, n_rows, dim).bytes;
    VDB_REQUIRE(work_bytes >= need && (d_work || need == 0), "the workspace of %lld bytes is too small for this lookup gradient (%lld needed)",
                (long long)work_bytes, (long long)need);
    if (n_rows == 0 || (n == 0 && accumulate)) return VDB_OK;
    VDB_TRY(ensure_init());
    (void)hipSetDevice(ctx().device);
    return launch_lookup_grad(d_grad, grad_type, ld, d_rows, n, scale, d_table_grad, table_type, n_rows, dim, ld_table, accumulate, d_work,
                              (hipStream_t)stream);
}
