// Distillation of score rows from a teacher's k best scores (vdb_distill_dev, vdb_distill_grad_dev,
// vdb_distill_step_dev).  With z a row of scores, c = log2(e) / tau, m = max z, S = sum_v 2^((z_v - m) c):
//   loss = tau^2 sum_j p_j (log p_j - (z_{r_j} - m) / tau + log S),   dz_v = w tau (M 2^((z_v - m) c) / S - sum_{r_j = v} p_j)
// p_j and their sum M come from the teacher's list alone.  The loss needs one pass over the row with the running
// maximum and sum; the gradient one pass that reads z and writes dz.  Both are bound by HBM: n * vocab values read,
// and as many written for the gradient.
#include "vdb_internal.h"
#include "values.h"

#include <algorithm>

namespace vdb {

static constexpr float LOG2E = 1.44269504088896340736f;

// v_exp_f32: 1 ulp, results below 2^-126 are zero
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// a running maximum and the sum of 2^((x - max) c) behind it
struct MaxSum {
    float m, s;
};
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
    const float m = fmaxf(a.m, b.m), base = finite_base(m);
    return {m, a.s * exp2_fast((a.m - base) * c) + b.s * exp2_fast((b.m - base) * c)};
}
// an empty part is (-inf, 0): its factor 2^(-inf) is 0; a sum that is NaN stays NaN
template <int NT> __device__ __forceinline__ MaxSum block_join(MaxSum v, float c, MaxSum* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = join(v, MaxSum{__shfl_xor(v.m, o), __shfl_xor(v.s, o)}, c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = join(v, red[w], c);
    return v;
}
template <int NT> __device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
    return v;
}
template <int NT> __device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v += red[w];
    return v;
}

// The teacher's list of one row in LDS: row numbers (-1: unfilled) and probabilities p_j; log p_j by the same formula
// where it is needed.  Returns M = sum p_j (0: nothing filled).
struct Teacher {
    const float* scores; const int64_t* rows; int k; int64_t ld_scores, ld_rows; const float* lse; float inv_tau;
};
template <int NT> __device__ static float teacher_row(const Teacher& t, int64_t row, int64_t vocab, int* at, float* logp, float* red) {
    const float* sc = t.scores + row * t.ld_scores;
    const int64_t* rw = t.rows + row * t.ld_rows;
    float top = -INFINITY;
    for (int j = threadIdx.x; j < t.k; j += NT) {
        const int64_t r = rw[j];
        const float x = sc[j];
        const bool filled = r >= 0 && r < vocab && x != -INFINITY;
        at[j] = filled ? (int)r : -1;
        logp[j] = filled ? x : -INFINITY;
        if (filled) top = fmaxf(top, x);
    }
    // fmaxf drops a NaN score; it comes back through the sum
    top = finite_base(block_max<NT>(top, red));
    float norm;
    if (t.lse) {
        norm = t.lse[row];
    } else {
        float s = 0.0f;
        for (int j = threadIdx.x; j < t.k; j += NT)
            if (at[j] >= 0) s += expf((logp[j] - top) * t.inv_tau);
        norm = logf(block_sum<NT>(s, red));
    }
    float m = 0.0f;
    for (int j = threadIdx.x; j < t.k; j += NT) {
        if (at[j] < 0) continue;
        const float l = t.lse ? logp[j] * t.inv_tau - norm : (logp[j] - top) * t.inv_tau - norm;
        logp[j] = l;
        m += expf(l);
    }
    return block_sum<NT>(m, red);
}

// ---------------------------------------------------------------- loss
static constexpr int LOSS_NT = 256;

template <class T>
__global__ void __launch_bounds__(LOSS_NT) distill_loss_kernel(const T* __restrict__ scores, int64_t vocab, int64_t ld, Teacher t, float tau,
                                                               float* __restrict__ loss, float* __restrict__ stats) {
    constexpr int N = Piece<T>::N;
    extern __shared__ float lds[];
    int* at = (int*)lds;
    float* logp = lds + t.k;
    __shared__ MaxSum red[LOSS_NT / 64];
    const int64_t row = blockIdx.x;
    const T* z = scores + row * ld;
    const float mass = teacher_row<LOSS_NT>(t, row, vocab, at, logp, (float*)red);
    if (mass == 0.0f && !stats) {
        if (threadIdx.x == 0) loss[row] = 0.0f;
        return;
    }
    const float c = LOG2E * t.inv_tau;
    MaxSum v{-INFINITY, 0.0f};
    for (int64_t i = (int64_t)threadIdx.x * N; i < vocab; i += LOSS_NT * N) {
        float x[N];
        load_values(z, i, vocab, -INFINITY, x);
        float top = v.m;
#pragma unroll
        for (int e = 0; e < N; ++e) top = fmaxf(top, x[e]);
        const float base = finite_base(top);
        float s = v.s * exp2_fast((v.m - base) * c);
#pragma unroll
        for (int e = 0; e < N; ++e) s += exp2_fast((x[e] - base) * c);
        v = {top, s};
    }
    v = block_join<LOSS_NT>(v, c, red);
    const float logs = logf(v.s), base = finite_base(v.m);
    float sum = 0.0f;
    for (int j = threadIdx.x; j < t.k; j += LOSS_NT) {
        if (at[j] < 0) continue;
        const float l = logp[j], p = expf(l), x = (float)z[at[j]];
        if (p == 0.0f) continue;
        const float logq = x == -INFINITY ? -INFINITY : (x - base) * t.inv_tau - logs;
        sum += p * (l - logq);
    }
    sum = block_sum<LOSS_NT>(sum, (float*)red);
    if (threadIdx.x == 0) {
        loss[row] = mass == 0.0f ? 0.0f : tau * tau * sum;
        if (stats) {
            stats[2 * row] = v.m;
            stats[2 * row + 1] = logs;
        }
    }
}

// ---------------------------------------------------------------- gradient
static constexpr int GRAD_NT = 256, SLOTS = VDB_DISTILL_MAX_K / GRAD_NT;

template <class T>
__global__ void __launch_bounds__(GRAD_NT) distill_grad_kernel(const T* scores, int64_t vocab, int64_t ld, Teacher t, float tau,
                                                               const float* __restrict__ stats, const float* __restrict__ grad_loss, T* grad,
                                                               int64_t ld_grad, int64_t part) {
    constexpr int N = Piece<T>::N;
    extern __shared__ float lds[];
    int* at = (int*)lds;
    float* prob = lds + t.k;
    __shared__ MaxSum red[GRAD_NT / 64];
    const int64_t row = blockIdx.x;
    const int64_t lo = (int64_t)blockIdx.y * part, hi = min(lo + part, vocab);
    const T* z = scores + row * ld;
    T* dz = grad + row * ld_grad;
    const float mass = teacher_row<GRAD_NT>(t, row, vocab, at, prob, (float*)red);
    const float w = grad_loss[row] * tau;
    if (w == 0.0f || mass == 0.0f) {
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = 0.0f;
        for (int64_t i = lo + threadIdx.x * N; i < hi; i += GRAD_NT * N) store_values<T, N>(dz, i, hi, x);
        return;
    }
    const float c = LOG2E * t.inv_tau, base = finite_base(stats[2 * row]), logs = stats[2 * row + 1];
    const float a = logs == -INFINITY ? 0.0f : w * mass * expf(-logs);
    // the columns of the teacher's slots: their scores are taken before the gradient may overwrite them; slots that
    // name the same row are added up, in order, by the first of them
    for (int j = threadIdx.x; j < t.k; j += GRAD_NT) prob[j] = at[j] < 0 ? 0.0f : expf(prob[j]);
    __syncthreads();
    float fix[SLOTS];
    bool mine[SLOTS];
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
        const int j = threadIdx.x + q * GRAD_NT, r = j < t.k ? at[j] : -1;
        mine[q] = r >= lo && r < hi;
        if (!mine[q]) continue;
        float p = 0.0f;
        for (int i = 0; i < t.k; ++i)
            if (at[i] == r) {
                if (i < j) mine[q] = false;
                p += prob[i];
            }
        fix[q] = a * exp2_fast(((float)z[r] - base) * c) - w * p;
    }
    __syncthreads();
    for (int64_t i = lo + threadIdx.x * N; i < hi; i += GRAD_NT * N) {
        float x[N];
        load_values(z, i, hi, 0.0f, x);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = a * exp2_fast((x[e] - base) * c);
        store_values<T, N>(dz, i, hi, x);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < SLOTS; ++q)
        if (mine[q]) dz[at[threadIdx.x + q * GRAD_NT]] = (T)fix[q];
}

// ---------------------------------------------------------------- launches
static int distill_parts(int64_t n, int64_t vocab, int64_t step, int64_t* part) {
    // enough blocks to fill the chip several times over, each with at least one step of work
    const int64_t want = std::max<int64_t>(1, (8 * (int64_t)ctx().num_cus + n - 1) / std::max<int64_t>(n, 1));
    const int64_t steps = (vocab + step - 1) / step;
    const int64_t parts = std::min({want, steps, (int64_t)65535});
    *part = (steps + parts - 1) / parts * step;
    return (int)((vocab + *part - 1) / *part);
}

static int launch_loss(const void* scores, int type, int64_t n, int64_t vocab, int64_t ld, const Teacher& t, float tau, float* loss, float* stats,
                       hipStream_t s) {
    return with_type(type, [&](auto* p) -> int {
        typedef std::remove_pointer_t<decltype(p)> T;
        hipLaunchKernelGGL(distill_loss_kernel<T>, dim3((unsigned)n), dim3(LOSS_NT), (size_t)t.k * 8, s, (const T*)scores, vocab, ld, t, tau, loss, stats);
        VDB_HIP(hipGetLastError());
        return VDB_OK;
    });
}

static int launch_grad(const void* scores, int type, int64_t n, int64_t vocab, int64_t ld, const Teacher& t, float tau, const float* stats,
                       const float* grad_loss, void* grad, int64_t ld_grad, hipStream_t s) {
    return with_type(type, [&](auto* p) -> int {
        typedef std::remove_pointer_t<decltype(p)> T;
        int64_t part;
        const int parts = distill_parts(n, vocab, GRAD_NT * Piece<T>::N, &part);
        hipLaunchKernelGGL(distill_grad_kernel<T>, dim3((unsigned)n, parts), dim3(GRAD_NT), (size_t)t.k * 8, s, (const T*)scores, vocab, ld, t, tau,
                           stats, grad_loss, (T*)grad, ld_grad, part);
        VDB_HIP(hipGetLastError());
        return VDB_OK;
    });
}

// arguments first, so that a bad call is refused before anything touches the GPU
static int check_distill(const void* d_scores, int type, int64_t n, int64_t vocab, int64_t ld, const float* d_teacher, const int64_t* d_rows, int k,
                         int64_t ld_teacher, int64_t ld_rows, float temperature) {
    const int64_t most = ((int64_t)1 << 31) - 1;
    VDB_REQUIRE(valid_type(type), "unknown value type %d", type);
    VDB_REQUIRE(n >= 0 && n < most && vocab >= 1 && vocab < most && ld >= 0, "bad sizes for a distillation: %lld rows of %lld scores, leading dimension %lld",
                (long long)n, (long long)vocab, (long long)ld);
    VDB_REQUIRE(k >= 0 && k <= VDB_DISTILL_MAX_K && ld_teacher >= 0 && ld_rows >= 0, "a teacher's list takes 0 to %d slots, got %d (leading dimensions %lld, %lld)",
                VDB_DISTILL_MAX_K, k, (long long)ld_teacher, (long long)ld_rows);
    VDB_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, "the temperature of a distillation lies in [1e-6, 1e6], got %g", (double)temperature);
    VDB_REQUIRE(n == 0 || (d_scores && (k == 0 || (d_teacher && d_rows))), "null pointer in a distillation of %lld rows", (long long)n);
    return VDB_OK;
}
static int check_gradient(int64_t n, int64_t vocab, int64_t ld, const void* d_scores, const float* d_grad_loss, const void* d_grad, int64_t ld_grad) {
    VDB_REQUIRE(n == 0 || (d_grad_loss && d_grad), "null pointer in the gradient of a distillation of %lld rows", (long long)n);
    VDB_REQUIRE(ld_grad >= vocab, "rows of %lld gradients do not fit a leading dimension of %lld", (long long)vocab, (long long)ld_grad);
    VDB_REQUIRE(d_grad != d_scores || ld_grad == ld || n <= 1, "a gradient in place of the scores takes their leading dimension (%lld, got %lld)",
                (long long)ld, (long long)ld_grad);
    return VDB_OK;
}
static int enter() {
    VDB_TRY(ensure_init());
    (void)hipSetDevice(ctx().device);
    return VDB_OK;
}

}  // namespace vdb

using namespace vdb;

int vdb_distill_workspace(int64_t n, int64_t vocab, int64_t* bytes) {
    VDB_REQUIRE(bytes, "null pointer for the workspace size");
    VDB_REQUIRE(n >= 0 && vocab >= 1, "bad sizes for a distillation: %lld rows of %lld scores", (long long)n, (long long)vocab);
    *bytes = n * 2 * (int64_t)sizeof(float);
    return VDB_OK;
}

int vdb_distill_dev(const void* d_scores, int type, int64_t n, int64_t vocab, int64_t ld, const float* d_teacher, const int64_t* d_rows, int k,
                    int64_t ld_teacher, int64_t ld_rows, const float* d_teacher_lse, float temperature, float* d_loss, float* d_stats, void* d_work,
                    int64_t work_bytes, void* stream) {
    VDB_TRY(check_distill(d_scores, type, n, vocab, ld, d_teacher, d_rows, k, ld_teacher, ld_rows, temperature));
    VDB_REQUIRE(n == 0 || d_loss, "null pointer in a distillation of %lld rows", (long long)n);
    (void)d_work; (void)work_bytes;
    if (n == 0) return VDB_OK;
    VDB_TRY(enter());
    const Teacher t{d_teacher, d_rows, k, ld_teacher, ld_rows, d_teacher_lse, 1.0f / temperature};
    return launch_loss(d_scores, type, n, vocab, ld, t, temperature, d_loss, d_stats, (hipStream_t)stream);
}

int vdb_distill_grad_dev(const void* d_scores, int type, int64_t n, int64_t vocab, int64_t ld, const float* d_teacher, const int64_t* d_rows, int k,
                         int64_t ld_teacher, int64_t ld_rows, const float* d_teacher_lse, float temperature, const float* d_stats,
                         const float* d_grad_loss, void* d_grad, int64_t ld_grad, void* stream) {
    VDB_TRY(check_distill(d_scores, type, n, vocab, ld, d_teacher, d_rows, k, ld_teacher, ld_rows, temperature));
    VDB_REQUIRE(n == 0 || d_stats, "null pointer in the gradient of a distillation of %lld rows", (long long)n);
    VDB_TRY(check_gradient(n, vocab, ld, d_scores, d_grad_loss, d_grad, ld_grad));
    if (n == 0) return VDB_OK;
    VDB_TRY(enter());
    const Teacher t{d_teacher, d_rows, k, ld_teacher, ld_rows, d_teacher_lse, 1.0f / temperature};
    return launch_grad(d_scores, type, n, vocab, ld, t, temperature, d_stats, d_grad_loss, d_grad, ld_grad, (hipStream_t)stream);
}

int vdb_distill_step_dev(const void* d_scores, int type, int64_t n, int64_t vocab, int64_t ld, const float* d_teacher, const int64_t* d_rows, int k,
                         int64_t ld_teacher, int64_t ld_rows, const float* d_teacher_lse, float temperature, const float* d_grad_loss,
                         float* d_loss, float* d_stats, void* d_grad, int64_t ld_grad, void* d_work, int64_t work_bytes, void* stream) {
    int64_t need = 0;
    VDB_TRY(check_distill(d_scores, type, n, vocab, ld, d_teacher, d_rows, k, ld_teacher, ld_rows, temperature));
    VDB_TRY(vdb_distill_workspace(n, vocab, &need));
    VDB_REQUIRE(work_bytes >= need && (d_work || need == 0), "the workspace of %lld bytes is too small for this distillation (%lld needed)",
                (long long)work_bytes, (long long)need);
    VDB_REQUIRE(n == 0 || d_loss, "null pointer in a distillation of %lld rows", (long long)n);
    VDB_TRY(check_gradient(n, vocab, ld, d_scores, d_grad_loss, d_grad, ld_grad));
    if (n == 0) return VDB_OK;
    VDB_TRY(enter());
    float* stats = d_stats ? d_stats : (float*)d_work;
    const Teacher t{d_teacher, d_rows, k, ld_teacher, ld_rows, d_teacher_lse, 1.0f / temperature};
    VDB_TRY(launch_loss(d_scores, type, n, vocab, ld, t, temperature, d_loss, stats, (hipStream_t)stream));
    return launch_grad(d_scores, type, n, vocab, ld, t, temperature, stats, d_grad_loss, d_grad, ld_grad, (hipStream_t)stream);
}
