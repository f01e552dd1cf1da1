// Loads and stores of fp32 / bf16 / fp16 rows for the operators on row tables and score rows: 16-byte pieces at any
// alignment the element type allows (gfx950 reads and writes them in one instruction wherever they lie), converted to
// fp32 and back with one rounding to nearest even.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/vdb_core.h"

namespace vdb {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <class T> struct Piece {
    static constexpr int N = 16 / (int)sizeof(T);     // elements of one 16-byte piece
    u32x4 raw;
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i]);
        else if constexpr (__is_same(T, bf16_t)) return __uint_as_float((i & 1) ? (raw[i >> 1] & 0xffff0000u) : (raw[i >> 1] << 16));
        else return (float)__builtin_bit_cast(f16_t, (uint16_t)((i & 1) ? (raw[i >> 1] >> 16) : (raw[i >> 1] & 0xffffu)));
    }
    // the first n elements away, the others to the front
    __device__ __forceinline__ void drop_first(int n) {
        const int bytes = n * (int)sizeof(T);
        if (bytes & 8) raw = u32x4{raw[2], raw[3], 0u, 0u};
        if (bytes & 4) raw = u32x4{raw[1], raw[2], raw[3], 0u};
        if (bytes & 2) raw = u32x4{raw[0] >> 16 | raw[1] << 16, raw[1] >> 16 | raw[2] << 16, raw[2] >> 16 | raw[3] << 16, raw[3] >> 16};
    }
    __device__ __forceinline__ void set(const float* x) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = __float_as_uint(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                typedef float f32x2 __attribute__((ext_vector_type(2)));
                typedef T T2 __attribute__((ext_vector_type(2)));
                const f32x2 pair = {x[2 * i], x[2 * i + 1]};
                raw[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, T2));
            }
        }
    }
};

template <class T> __device__ __forceinline__ Piece<T> load_piece(const T* p) {
    Piece<T> r;
    __builtin_memcpy(&r.raw, p, 16);
    return r;
}
template <class T> __device__ __forceinline__ void store_piece(T* p, const Piece<T>& v) { __builtin_memcpy(p, &v.raw, 16); }

// The elements [at, at + N) of a row of `len`, those behind its end as `fill`.
template <class T> __device__ __forceinline__ void load_values(const T* row, int64_t at, int64_t len, float fill, float* x) {
    if (at + Piece<T>::N <= len) {
        const Piece<T> v = load_piece(row + at);
#pragma unroll
        for (int i = 0; i < Piece<T>::N; ++i) x[i] = v.get(i);
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T>::N; ++i) x[i] = at + i < len ? (float)row[at + i] : fill;
    }
}

// N fp32 values to the elements [at, at + N) of a row of `len`, rounded once; what lies behind the row's end is dropped.
template <class T, int N> __device__ __forceinline__ void store_values(T* row, int64_t at, int64_t len, const float* x) {
    if (at + N <= len) {
        T v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (T)x[i];
        __builtin_memcpy(row + at, v, N * sizeof(T));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < len) row[at + i] = (T)x[i];
    }
}

// Over a wave by data-parallel moves (rows of 16 lanes, then their last lanes passed on), for all lanes.
template <int CTRL, int ROWS> __device__ __forceinline__ float moved(float v, float other) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(other), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ __forceinline__ float wave_sum(float v) {
    v += moved<0x111, 0xf>(v, 0.0f);          // row_shr:1, 2, 4, 8
    v += moved<0x112, 0xf>(v, 0.0f);
    v += moved<0x114, 0xf>(v, 0.0f);
    v += moved<0x118, 0xf>(v, 0.0f);
    v += moved<0x142, 0xa>(v, 0.0f);          // row_bcast:15 into rows 1 and 3
    v += moved<0x143, 0xc>(v, 0.0f);          // row_bcast:31 into rows 2 and 3
    return last_lane(v);
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, moved<0x111, 0xf>(v, v));
    v = fmaxf(v, moved<0x112, 0xf>(v, v));
    v = fmaxf(v, moved<0x114, 0xf>(v, v));
    v = fmaxf(v, moved<0x118, 0xf>(v, v));
    v = fmaxf(v, moved<0x142, 0xa>(v, v));
    v = fmaxf(v, moved<0x143, 0xc>(v, v));
    return last_lane(v);
}

// host side: vdb_value_type codes to template arguments
static inline bool valid_type(int type) { return type == VDB_VALUE_F32 || type == VDB_VALUE_BF16 || type == VDB_VALUE_F16; }

static inline bool aligned_work(const void* work) { return ((uintptr_t)work & 15) == 0; }

template <class F> static int with_type(int type, F&& f) {
    if (type == VDB_VALUE_F32) return f((float*)nullptr);
    if (type == VDB_VALUE_BF16) return f((bf16_t*)nullptr);
    return f((f16_t*)nullptr);
}

}  // namespace vdb
