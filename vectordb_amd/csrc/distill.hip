// Distillation of score rows from a teacher's k best scores (vdb_distill_dev, vdb_distill_grad_dev,
// vdb_distill_step_dev).  With z a row of scores, c = log2(e) / tau, m = max z, S = sum_v 2^((z_v - m) c):
//   loss = tau^2 sum_j p_j (log p_j - (z_{r_j} - m) / tau + log S),   dz_v = w tau (M 2^((z_v - m) c) / S - sum_{r_j = v} p_j)
// p_j and their sum M come from the teacher's list alone.
//   loss       one pass over the row with the running maximum and sum; few long rows in parts, joined by a second launch
//   gradient   one pass that reads z and writes dz
//   both       a row that fits a block's registers is read once: maximum, sum and gradient from there; longer rows take the
//              two passes above
// All are bound by HBM: n * vocab values read (twice for the two passes), and as many written for the gradient.  Measured: loss
// of 4096 x 131072 bf16 184 us (5.8 TB/s), gradient of 5000 x 8191 bf16 34 us (5.0 TB/s), both of 4096 x 32768 bf16 110 us
// (4.9 TB/s), of 8000 x 8000 bf16 50 us (5.3 TB/s).  Rows need not be aligned.
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
// A barrier for what was written to LDS; loads and stores of global memory stay under way.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// Over a block, for all threads; one barrier, behind which everything written to LDS before is there too.  An empty part
// is (-inf, 0): its factor 2^(-inf) is 0; a sum that is NaN stays NaN.
template <int NT> __device__ __forceinline__ MaxSum block_join(MaxSum v, float c, MaxSum* red) {
    const float m = wave_max(v.m);
    const float s = wave_sum(v.s * exp2_fast((v.m - finite_base(m)) * c));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = {m, s};
    lds_barrier();
    MaxSum r{-INFINITY, 0.0f};
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) r.m = fmaxf(r.m, red[w].m);
    const float base = finite_base(r.m);
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) r.s += red[w].s * exp2_fast((red[w].m - base) * c);
    return r;
}

// The teacher's list of one row in LDS, up to a multiple of four slots: row numbers (-1: unfilled), log p_j and the rows' scores.
struct Teacher {
    const float* scores; const int64_t* rows; int k; int64_t ld_scores, ld_rows; const float* lse; float inv_tau;
    __host__ __device__ int room() const { return (k + 3) & ~3; }
    size_t lds() const { return (size_t)room() * 20; }
};
struct List {
    int *at, *where;                 // where, fix: see fix_slots
    float *logp, *score, *fix;
    __device__ __forceinline__ List(const Teacher& t, float* lds)
        : at((int*)lds), where((int*)lds + t.room()), logp(lds + 2 * t.room()), score(lds + 3 * t.room()), fix(lds + 4 * t.room()) {}
};
// Every wave goes through the list for itself, without a barrier: it is short, and what a block waits for costs more.  The
// first wave leaves it in LDS, with the scores of rows in [lo, hi).  Returns M = sum p_j: 0 where nothing is filled, 1 where
// the list is a distribution of its own.
template <class T>
__device__ __forceinline__ float teacher_row(const Teacher& t, int64_t row, const T* z, int64_t vocab, int64_t lo, int64_t hi, const List& list) {
    const float* sc = t.scores + row * t.ld_scores;
    const int64_t* rw = t.rows + row * t.ld_rows;
    const int lane = threadIdx.x & 63;
    auto slot = [&](int j, float* x) {
        const int64_t r = j < t.k ? rw[j] : -1;
        *x = j < t.k ? sc[j] : -INFINITY;
        const bool filled = r >= 0 && r < vocab && *x != -INFINITY;
        if (!filled) *x = -INFINITY;
        return filled ? (int)r : -1;
    };
    // The first slot of a lane stays in registers.  fmaxf drops a NaN score; it comes back through the sum.
    float x0, top, norm = 0.0f, mass = 1.0f;
    const int r0 = slot(lane, &x0);
    bool some = r0 >= 0;
    top = x0;
    for (int j = lane + 64; j < t.room(); j += 64) {
        float x;
        some |= slot(j, &x) >= 0;
        top = fmaxf(top, x);
    }
    if (!__ballot(some)) mass = 0.0f;
    top = t.lse ? 0.0f : finite_base(wave_max(top));
    if (t.lse) norm = t.lse[row];
    float sum = r0 >= 0 ? expf((x0 - top) * t.inv_tau - norm) : 0.0f;
    for (int j = lane + 64; j < t.room(); j += 64) {
        float x;
        if (slot(j, &x) >= 0) sum += expf((x - top) * t.inv_tau - norm);
    }
    sum = wave_sum(sum);
    if (t.lse) mass = sum;
    else norm = logf(sum);
    if (threadIdx.x < 64)
        for (int j = lane; j < t.room(); j += 64) {
            float x = x0;
            const int r = j == lane ? r0 : slot(j, &x);
            list.at[j] = r;
            list.logp[j] = (x - top) * t.inv_tau - norm;
            list.score[j] = r >= lo && r < hi ? (float)z[r] : 0.0f;
        }
    return mass;
}

// ---------------------------------------------------------------- rows at 16-byte borders
// The pieces of a row counted from the 16-byte border at or before its start: piece i holds the elements
// [i * N - off, i * N - off + N) of the row, those outside [lo, hi) as `fill`.
template <class T> __device__ __forceinline__ int border_off(const T* row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); }

template <class T> __device__ __forceinline__ Piece<T> load_between(const T* row, int64_t at, int64_t lo, int64_t hi, float fill) {
    constexpr int N = Piece<T>::N;
    Piece<T> x;
    if (at >= lo && at + N <= hi) x = load_piece(row + at);
    else {
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = at + e >= lo && at + e < hi ? (float)row[at + e] : fill;
        x.set(v);
    }
    return x;
}
template <class T> __device__ __forceinline__ void store_between(T* row, int64_t at, int64_t lo, int64_t hi, const float* x) {
    constexpr int N = Piece<T>::N;
    if (at >= lo && at + N <= hi) {
        Piece<T> v;
        v.set(x);
        store_piece(row + at, v);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (at + e >= lo && at + e < hi) row[at + e] = (T)x[e];
    }
}

template <class T> __device__ __forceinline__ Piece<T> all_of(float x) {
    float v[Piece<T>::N];
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e) v[e] = x;
    Piece<T> r;
    r.set(v);
    return r;
}

// the scores of AHEAD pieces into a running maximum and sum
static constexpr int AHEAD = 4;
template <class T> __device__ __forceinline__ void add_pieces(MaxSum& v, const Piece<T>* x, float c) {
    constexpr int N = Piece<T>::N;
    float top = v.m;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) top = fmaxf(top, x[j].get(e));
    const float base = finite_base(top);
    float s = v.s * exp2_fast((v.m - base) * c);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) t += exp2_fast((x[j].get(e) - base) * c);
        s += t;
    }
    v = {top, s};
}

// The loss of a row from the maximum and the sum, and the stats, by the block's first wave.
__device__ __forceinline__ void write_loss(const Teacher& t, const List& list, float mass, float tau, MaxSum v, float logs,
                                           int64_t row, float* loss, float* stats) {
    if (threadIdx.x >= 64) return;
    const float base = finite_base(v.m);
    float sum = 0.0f;
    for (int j = threadIdx.x; j < t.k; j += 64) {
        if (list.at[j] < 0) continue;
        const float l = list.logp[j], p = expf(l), x = list.score[j];
        if (p == 0.0f) continue;
        const float logq = x == -INFINITY ? -INFINITY : (x - base) * t.inv_tau - logs;
        sum += p * (l - logq);
    }
    sum = wave_sum(sum);
    if (threadIdx.x == 0) {
        loss[row] = mass == 0.0f ? 0.0f : tau * tau * sum;
        if (stats) {
            stats[2 * row] = v.m;
            stats[2 * row + 1] = logs;
        }
    }
}

// The gradient at the teacher's rows in [lo, hi).  Slots that name the same row are added up, in order, by the first of them;
// the others have nothing to write (-1).  The threads behind the first wave begin, as the first writes the loss.  The list is
// there for all threads; scores are no longer read, they may lie where the gradient goes.
template <int NT>
__device__ __forceinline__ void fix_slots(const Teacher& t, const List& list, float a, float w, float base, float c, int64_t lo, int64_t hi) {
    for (int j = (threadIdx.x + NT - 64) % NT; j < t.k; j += NT) {
        const int r = list.at[j];
        int where = -1;
        if (r >= lo && r < hi) {
            where = r;
            float p = expf(list.logp[j]);
            int same = 0;
#pragma unroll 4
            for (int i = 0; i < t.room(); i += 4) {
                const int4 other = *(const int4*)(list.at + i);
                same += (other.x == r) + (other.y == r) + (other.z == r) + (other.w == r);
            }
            if (same > 1)                                     // rare: most lists name a row once
                for (int i = 0; i < t.k; ++i)
                    if (i != j && list.at[i] == r) {
                        if (i < j) where = -1;
                        p += expf(list.logp[i]);
                    }
            list.fix[j] = a * exp2_fast((list.score[j] - base) * c) - w * p;
        }
        list.where[j] = where;
    }
}
// ... over the gradient of all scores.  Each wave takes the rows that lie in its own pieces (piece i, counted from `off` elements
// before the row, is thread (i - first) % NT's): its stores reach memory in their order, so none has to be waited for.
template <int NT, class T>
__device__ __forceinline__ void write_slots(const Teacher& t, const List& list, T* dz, int off, int64_t first) {
    lds_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int j = threadIdx.x & 63; j < t.k; j += 64) {
        const int r = list.where[j];
        if (r >= 0 && (uint32_t)((r + (int64_t)off) / Piece<T>::N - first) % NT / 64 == threadIdx.x / 64) dz[r] = (T)list.fix[j];
    }
}

// ---------------------------------------------------------------- loss
// blockIdx.y: the part of the row; one part: the loss at once, else its maximum and sum to `parts`
template <class T, int NT>
__global__ void __launch_bounds__(NT) distill_loss_kernel(const T* __restrict__ scores, int64_t row0, int64_t vocab, int64_t ld, Teacher t, float tau,
                                                          float* __restrict__ loss, float* __restrict__ stats, int64_t part_pieces, MaxSum* __restrict__ parts) {
    constexpr int N = Piece<T>::N;
    extern __shared__ __align__(16) float lds[];
    const List list(t, lds);
    __shared__ MaxSum red[NT / 64];
    const int64_t row = row0 + blockIdx.x;
    const T* z = scores + row * ld;
    const float c = LOG2E * t.inv_tau;
    const int64_t first = (int64_t)blockIdx.y * part_pieces, full = min(first + part_pieces, vocab / N);
    MaxSum v{-INFINITY, 0.0f};
    for (int64_t i = first + threadIdx.x; i < full; i += AHEAD * NT) {
        Piece<T> x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            x[j] = all_of<T>(-INFINITY);
            if (i + j * NT < full) x[j] = load_piece(z + (i + j * NT) * N);
        }
        add_pieces(v, x, c);
    }
    // what is left of the row, less than a piece
    const int64_t whole = vocab / N, left = whole * N + threadIdx.x;
    if (first <= whole && whole < first + part_pieces && left < vocab) v = join(v, {(float)z[left], 1.0f}, c);
    float mass = 0.0f;
    if (!parts && threadIdx.x < 64) mass = teacher_row(t, row, z, vocab, 0, vocab, list);
    v = block_join<NT>(v, c, red);
    if (parts) {
        if (threadIdx.x == 0) parts[row * gridDim.y + blockIdx.y] = v;
        return;
    }
    write_loss(t, list, mass, tau, v, logf(v.s), row, loss, stats);
}

template <class T>
__global__ void __launch_bounds__(256) distill_join_kernel(const T* __restrict__ scores, int64_t row0, int64_t vocab, int64_t ld, Teacher t, float tau,
                                                           float* __restrict__ loss, float* __restrict__ stats, const MaxSum* __restrict__ parts, int n_parts) {
    extern __shared__ __align__(16) float lds[];
    const List list(t, lds);
    __shared__ MaxSum red[4];
    const int64_t row = row0 + blockIdx.x;
    const float c = LOG2E * t.inv_tau;
    MaxSum v{-INFINITY, 0.0f};
    for (int i = threadIdx.x; i < n_parts; i += 256) v = join(v, parts[row * n_parts + i], c);
    float mass = 0.0f;
    if (threadIdx.x < 64) mass = teacher_row(t, row, scores + row * ld, vocab, 0, vocab, list);
    v = block_join<256>(v, c, red);
    write_loss(t, list, mass, tau, v, logf(v.s), row, loss, stats);
}

// ---------------------------------------------------------------- gradient
static constexpr int GRAD_NT = 256;

template <class T>
__global__ void __launch_bounds__(GRAD_NT) distill_grad_kernel(const T* scores, int64_t row0, int64_t vocab, int64_t ld, Teacher t, float tau,
                                                               const float* __restrict__ stats, const float* __restrict__ grad_loss, T* grad,
                                                               int64_t ld_grad, int64_t part_pieces) {
    constexpr int N = Piece<T>::N;
    extern __shared__ __align__(16) float lds[];
    const List list(t, lds);
    const int64_t row = row0 + blockIdx.x;
    const T* z = scores + row * ld;
    T* dz = grad + row * ld_grad;
    // pieces at the borders of the gradient: what is written matters more than what is read (where both lie alike: both)
    const int off = border_off(dz);
    const int64_t first = (int64_t)blockIdx.y * part_pieces, last = min(first + part_pieces, (vocab + off + N - 1) / N);
    const int64_t lo = max((int64_t)0, first * N - off), hi = min(vocab, last * N - off);
    const float w = grad_loss[row] * tau;
    const float mass = teacher_row(t, row, z, vocab, lo, hi, list);
    if (w == 0.0f || mass == 0.0f) {
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = 0.0f;
        for (int64_t i = first + threadIdx.x; i < last; i += GRAD_NT) store_between(dz, i * N - off, lo, hi, x);
        return;
    }
    const float c = LOG2E * t.inv_tau, base = finite_base(stats[2 * row]), logs = stats[2 * row + 1];
    const float a = logs == -INFINITY ? 0.0f : w * mass * expf(-logs);
    lds_barrier();
    fix_slots<GRAD_NT>(t, list, a, w, base, c, lo, hi);
    const int64_t from = off ? 1 : 0, full = min(last, (vocab + off) / N);
    for (int64_t i = first + threadIdx.x; i < full; i += AHEAD * GRAD_NT) {
        Piece<T> x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int64_t at = i + j * GRAD_NT;
            x[j] = all_of<T>(0.0f);
            if (at >= from && at < full) x[j] = load_piece(z + at * N - off);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int64_t at = i + j * GRAD_NT;
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = a * exp2_fast((x[j].get(e) - base) * c);
            x[j].set(y);
            if (at >= from && at < full) store_piece(dz + at * N - off, x[j]);
        }
    }
    // the pieces that the row fills in part, by the threads whose turn it is: the first, the last
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
        const int64_t at = side ? last - 1 : 0;
        if (side ? full == last || at < max(first, from) : first > 0 || !off) continue;
        if ((at - first) % GRAD_NT != threadIdx.x) continue;
        const Piece<T> x = load_between(z, at * N - off, lo, hi, 0.0f);
        float y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = a * exp2_fast((x.get(e) - base) * c);
        store_between(dz, at * N - off, lo, hi, y);
    }
    write_slots<GRAD_NT>(t, list, dz, off, first);
}

// ---------------------------------------------------------------- loss and gradient, the row in registers
// The pieces as they are, but nothing computed from them before: else the compiler keeps the unpacked scores of one pass
// for the next, twice as many registers as the row, and spills.
template <class T, int NP> __device__ __forceinline__ void forget_unpacked(Piece<T> (&x)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t r = x[p].raw[i];
            asm volatile("" : "+v"(r));
            x[p].raw[i] = r;
        }
}

template <class T, int NT, int NP>
__global__ void __launch_bounds__(NT) distill_step_kernel(const T* scores, int64_t row0, int64_t vocab, int64_t ld, Teacher t, float tau,
                                                          const float* __restrict__ grad_loss, float* __restrict__ loss, float* __restrict__ stats,
                                                          T* grad, int64_t ld_grad) {
    constexpr int N = Piece<T>::N;
    extern __shared__ __align__(16) float lds[];
    const List list(t, lds);
    __shared__ MaxSum red[NT / 64];
    const int64_t row = row0 + blockIdx.x;
    const T* z = scores + row * ld;
    T* dz = grad + row * ld_grad;
    const int full = (int)(vocab / N);
    const float c = LOG2E * t.inv_tau, w = grad_loss[row] * tau;
    Piece<T> x[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int at = p * NT + threadIdx.x;
        x[p] = all_of<T>(-INFINITY);
        if (at < full) x[p] = load_piece(z + at * N);
    }
    // the piece that the row fills in part, and the thread whose it is
    const bool partial = full * N < vocab && full % NT == threadIdx.x;
    if (partial) {
        const Piece<T> tail = load_between(z, (int64_t)full * N, 0, vocab, -INFINITY);
#pragma unroll
        for (int p = 0; p < NP; ++p)
            if (p == full / NT) x[p] = tail;
    }
    // while the row is under way
    const float mass = teacher_row(t, row, z, vocab, 0, vocab, list);
    // the thread's maximum and its sum behind it, then the block's: one barrier
    MaxSum v{-INFINITY, 0.0f};
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int e = 0; e < N; ++e) v.m = fmaxf(v.m, x[p].get(e));
    forget_unpacked(x);
    const float mine = finite_base(v.m);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        float u = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) u += exp2_fast((x[p].get(e) - mine) * c);
        v.s += u;
    }
    v = block_join<NT>(v, c, red);
    const float logs = logf(v.s), base = finite_base(v.m);
    write_loss(t, list, mass, tau, v, logs, row, loss, stats);
    const bool none = w == 0.0f || mass == 0.0f;
    const float a = none || logs == -INFINITY ? 0.0f : w * mass * expf(-logs);
    if (!none) fix_slots<NT>(t, list, a, w, base, c, 0, vocab);
    forget_unpacked(x);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        float y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = a * exp2_fast((x[p].get(e) - base) * c);
        x[p].set(y);
    }
    if (none) {                          // 0 x NaN or infinity among the scores
#pragma unroll
        for (int p = 0; p < NP; ++p) x[p] = all_of<T>(0.0f);
    }
#pragma unroll
    for (int p = 0; p < NP; ++p)
        if (p * NT + (int)threadIdx.x < full) store_piece(dz + (p * NT + threadIdx.x) * N, x[p]);
    if (partial) {
        Piece<T> tail = x[0];
#pragma unroll
        for (int p = 0; p < NP; ++p)
            if (p == full / NT) tail = x[p];
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (full * N + e < vocab) dz[full * N + e] = (T)tail.get(e);
    }
    if (!none) write_slots<NT>(t, list, dz, 0, 0);
}

// ---------------------------------------------------------------- launches
// A launch holds fewer than 2^32 threads: rows in batches of 2^21 blocks.
template <class F> static int in_batches(int64_t n, F&& launch) {
    const int64_t most = (int64_t)1 << 21;
    for (int64_t row0 = 0; row0 < n; row0 += most) {
        launch(row0, (unsigned)std::min(most, n - row0));
        VDB_HIP(hipGetLastError());
    }
    return VDB_OK;
}

// Parts of a row in pieces of 16 bytes: as many as `blocks` allow, each of at least `least` pieces.
static int parts_of(int64_t n, int64_t vocab, int per_piece, int64_t blocks, int64_t least, int64_t* part_pieces) {
    const int64_t pieces = vocab / per_piece + 2;                      // whatever the row's offset from a border
    const int64_t parts = std::max<int64_t>(1, std::min({blocks / std::max<int64_t>(n, 1), pieces / least, (int64_t)1024}));
    *part_pieces = (pieces + parts - 1) / parts;
    return (int)((pieces + *part_pieces - 1) / *part_pieces);
}
// The loss: a block of 256 threads a row, of 1024 where there are few blocks (1 x 131072 bf16 9.9 us, 13.5 by 256), and parts of a
// row, joined by a second launch, while they find a CU each (16 x 131072 fp32 7.9 us, 10.4 in one part; 500 x 32768 13.8,
// 16.6 in two).
static const int64_t LOSS_WIDE = 512, LOSS_PART = 4096;                // blocks; pieces of a part
static int loss_parts(int64_t n, int64_t vocab, int per_piece, int64_t* part_pieces) {
    const bool pays = vocab / per_piece + 2 >= 4 * LOSS_PART;          // two parts save less than the second launch takes
    return parts_of(n, vocab, per_piece, pays ? ctx().num_cus : 0, LOSS_PART, part_pieces);
}

static int launch_loss(const void* scores, int type, int64_t n, int64_t vocab, int64_t ld, const Teacher& t, float tau, float* loss, float* stats,
                       void* work, hipStream_t s) {
    return with_type(type, [&](auto* p) -> int {
        typedef std::remove_pointer_t<decltype(p)> T;
        int64_t part;
        const int parts = loss_parts(n, vocab, Piece<T>::N, &part);
        MaxSum* partial = parts > 1 ? (MaxSum*)work : nullptr;
        const size_t lds = t.lds();
        const T* z = (const T*)scores;
        return in_batches(n, [&](int64_t row0, unsigned rows) {
            const dim3 grid(rows, (unsigned)parts);
            if (n * parts <= LOSS_WIDE)
                hipLaunchKernelGGL((distill_loss_kernel<T, 1024>), grid, dim3(1024), lds, s, z, row0, vocab, ld, t, tau, loss, stats, part, partial);
            else
                hipLaunchKernelGGL((distill_loss_kernel<T, 256>), grid, dim3(256), lds, s, z, row0, vocab, ld, t, tau, loss, stats, part, partial);
            if (parts > 1) hipLaunchKernelGGL(distill_join_kernel<T>, dim3(rows), dim3(256), lds, s, z, row0, vocab, ld, t, tau, loss, stats, partial, parts);
        });
    });
}

static int launch_grad(const void* scores, int type, int64_t n, int64_t vocab, int64_t ld, const Teacher& t, float tau, const float* stats,
                       const float* grad_loss, void* grad, int64_t ld_grad, hipStream_t s) {
    return with_type(type, [&](auto* p) -> int {
        typedef std::remove_pointer_t<decltype(p)> T;
        int64_t part;
        // parts of a step of AHEAD pieces or more, up to 32 blocks a CU (2048 x 50021 fp16 92 us, with 8 or 64 a CU 96)
        const int parts = parts_of(n, vocab, Piece<T>::N, 32 * (int64_t)ctx().num_cus + n - 1, AHEAD * GRAD_NT, &part);
        return in_batches(n, [&](int64_t row0, unsigned rows) {
            hipLaunchKernelGGL(distill_grad_kernel<T>, dim3(rows, (unsigned)parts), dim3(GRAD_NT), t.lds(), s, (const T*)scores, row0, vocab, ld, t, tau, stats,
                               grad_loss, (T*)grad, ld_grad, part);
        });
    });
}

// Whether a row fits the registers of a block, and how: its threads, its pieces a thread.  As few pieces as the row allows, so that
// several blocks share a CU and one loads while another computes: 8000 x 2000 bf16 takes 20.6 us by 64 threads, 41.5 by 256;
// 4096 x 32768 bf16 109.7 us (4.9 TB/s) by 1024 threads of 4, 133 by 512 of 16.  Two blocks of 512 with 16 pieces fit a CU, one of
// 1024 with 8: 2048 x 50024 f16 89 against 113 us, but 16 x 32768 f32, where blocks are alone, takes the wide one.  A row
// of more than 8192 pieces takes a whole CU: 1000 x 131072 bf16 121 us against 167 in two passes of a split row, 1 x 131072 18.0
// against 14.8.
struct StepShape {
    int nt, np;
};
static StepShape step_shape(int64_t n, int64_t vocab, int per_piece) {
    const int64_t pieces = (vocab + per_piece - 1) / per_piece;
    const bool few = n < 2 * (int64_t)ctx().num_cus;
    if (pieces <= 256) return {64, 4};
    if (pieces <= 1024) return {256, 4};
    if (pieces <= 2048) return {512, 4};
    if (pieces <= 4096) return {1024, 4};
    if (pieces <= 8192) return few ? StepShape{1024, 8} : StepShape{512, 16};
    if (pieces <= 16384 && !few) return {1024, 16};
    return {0, 0};
}

static int launch_step(const void* scores, int type, int64_t n, int64_t vocab, int64_t ld, const Teacher& t, float tau, const float* grad_loss,
                       float* loss, float* stats, void* grad, int64_t ld_grad, const StepShape& shape, hipStream_t s) {
    return with_type(type, [&](auto* p) -> int {
        typedef std::remove_pointer_t<decltype(p)> T;
        auto go = [&](auto kernel, int nt) {
            return in_batches(n, [&](int64_t row0, unsigned rows) {
                hipLaunchKernelGGL(kernel, dim3(rows), dim3((unsigned)nt), t.lds(), s, (const T*)scores, row0, vocab, ld, t, tau, grad_loss, loss, stats,
                                   (T*)grad, ld_grad);
            });
        };
        if (shape.nt == 64) return go(distill_step_kernel<T, 64, 4>, 64);
        if (shape.nt == 256) return go(distill_step_kernel<T, 256, 4>, 256);
        if (shape.nt == 512 && shape.np == 4) return go(distill_step_kernel<T, 512, 4>, 512);
        if (shape.nt == 512) return go(distill_step_kernel<T, 512, 16>, 512);
        if (shape.np == 4) return go(distill_step_kernel<T, 1024, 4>, 1024);
        if (shape.np == 8) return go(distill_step_kernel<T, 1024, 8>, 1024);
        return go(distill_step_kernel<T, 1024, 16>, 1024);
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

// the workspace: the stats of a step in two passes (whatever the type: fp32 rows have the most pieces), then the parts of long rows
static int64_t distill_stats_bytes(int64_t n, int64_t vocab) {
    return step_shape(n, vocab, 4).nt ? 0 : round_up64(n * 2 * (int64_t)sizeof(float), 256);
}

int vdb_distill_workspace(int64_t n, int64_t vocab, int64_t* bytes) {
    VDB_REQUIRE(bytes, "null pointer for the workspace size");
    VDB_REQUIRE(n >= 0 && vocab >= 1, "bad sizes for a distillation: %lld rows of %lld scores", (long long)n, (long long)vocab);
    int64_t part;
    const int parts = loss_parts(n, vocab, 4, &part);
    *bytes = distill_stats_bytes(n, vocab) + (parts > 1 ? n * parts * (int64_t)sizeof(MaxSum) : 0);
    return VDB_OK;
}
static int check_work(int64_t n, int64_t vocab, const void* d_work, int64_t work_bytes) {
    int64_t need = 0;
    VDB_TRY(vdb_distill_workspace(n, vocab, &need));
    VDB_REQUIRE(work_bytes >= need && (d_work || need == 0), "the workspace of %lld bytes is too small for this distillation (%lld needed)",
                (long long)work_bytes, (long long)need);
    VDB_REQUIRE(aligned_work(d_work), "a workspace begins at a multiple of 16 bytes");
    return VDB_OK;
}

int vdb_distill_dev(const void* d_scores, int type, int64_t n, int64_t vocab, int64_t ld, const float* d_teacher, const int64_t* d_rows, int k,
                    int64_t ld_teacher, int64_t ld_rows, const float* d_teacher_lse, float temperature, float* d_loss, float* d_stats, void* d_work,
                    int64_t work_bytes, void* stream) {
    VDB_TRY(check_distill(d_scores, type, n, vocab, ld, d_teacher, d_rows, k, ld_teacher, ld_rows, temperature));
    VDB_REQUIRE(n == 0 || d_loss, "null pointer in a distillation of %lld rows", (long long)n);
    VDB_TRY(check_work(n, vocab, d_work, work_bytes));
    if (n == 0) return VDB_OK;
    VDB_TRY(enter());
    const Teacher t{d_teacher, d_rows, k, ld_teacher, ld_rows, d_teacher_lse, 1.0f / temperature};
    return launch_loss(d_scores, type, n, vocab, ld, t, temperature, d_loss, d_stats, (char*)d_work + distill_stats_bytes(n, vocab), (hipStream_t)stream);
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
    VDB_TRY(check_distill(d_scores, type, n, vocab, ld, d_teacher, d_rows, k, ld_teacher, ld_rows, temperature));
    VDB_TRY(check_work(n, vocab, d_work, work_bytes));
    VDB_REQUIRE(n == 0 || d_loss, "null pointer in a distillation of %lld rows", (long long)n);
    VDB_TRY(check_gradient(n, vocab, ld, d_scores, d_grad_loss, d_grad, ld_grad));
    if (n == 0) return VDB_OK;
    VDB_TRY(enter());
    const Teacher t{d_teacher, d_rows, k, ld_teacher, ld_rows, d_teacher_lse, 1.0f / temperature};
    const StepShape shape = step_shape(n, vocab, type == VDB_VALUE_F32 ? 4 : 8);
    if (shape.nt)
        return launch_step(d_scores, type, n, vocab, ld, t, temperature, d_grad_loss, d_loss, d_stats, d_grad, ld_grad, shape, (hipStream_t)stream);
    float* stats = d_stats ? d_stats : (float*)d_work;
    VDB_TRY(launch_loss(d_scores, type, n, vocab, ld, t, temperature, d_loss, stats, (char*)d_work + distill_stats_bytes(n, vocab), (hipStream_t)stream));
    return launch_grad(d_scores, type, n, vocab, ld, t, temperature, stats, d_grad_loss, d_grad, ld_grad, (hipStream_t)stream);
}
