// Rows of a model's activations and tables, read and written in units of 16
// bytes: shared by the operators around the optimizer step.
//
// A unit is Unit<T>::n consecutive elements of one row, converted to fp32.
// Rows need no alignment beyond their element's: gfx950's global loads and
// stores of 16 bytes take any address, so a width that is odd keeps the wide
// accesses, and only a row's last, shorter unit goes element by element.
#pragma once

#include "common.hpp"

namespace cresso {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Unit { static constexpr int n = 16 / (int)sizeof(T); };

// 16 bytes at an address that is aligned to its element alone
struct __attribute__((packed, aligned(2), may_alias)) Raw16h { u32x4 v; };
struct __attribute__((packed, aligned(4), may_alias)) Raw16w { u32x4 v; };
struct __attribute__((packed, aligned(2), may_alias)) Raw8h { u32x2 v; };
typedef uint16_t __attribute__((may_alias)) raw16_t;
typedef uint32_t __attribute__((may_alias)) raw32_t;

template <typename T> __device__ __forceinline__ u32x4 load16(const T* p) {
    if constexpr (sizeof(T) == 4) return ((const CRESSO_GLOBAL Raw16w*)p)->v;
    else return ((const CRESSO_GLOBAL Raw16h*)p)->v;
}
template <typename T> __device__ __forceinline__ void store16(T* p, u32x4 v) {
    if constexpr (sizeof(T) == 4) ((CRESSO_GLOBAL Raw16w*)p)->v = v;
    else ((CRESSO_GLOBAL Raw16h*)p)->v = v;
}
// four 16-bit elements
template <typename T> __device__ __forceinline__ void store8(T* p, u32x2 v) {
    static_assert(sizeof(T) == 2, "16-bit elements");
    ((CRESSO_GLOBAL Raw8h*)p)->v = v;
}

// two 16-bit elements of a word as floats
template <typename T> __device__ __forceinline__ void widen2(uint32_t w, float& lo, float& hi);
template <> __device__ __forceinline__ void widen2<__hip_bfloat16>(uint32_t w, float& lo, float& hi) {
    lo = __builtin_bit_cast(float, w << 16);
    hi = __builtin_bit_cast(float, w & 0xffff0000u);
}
template <> __device__ __forceinline__ void widen2<__half>(uint32_t w, float& lo, float& hi) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    lo = (float)h[0];
    hi = (float)h[1];
}
// two floats rounded to nearest even
template <typename T> __device__ __forceinline__ uint32_t narrow2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t narrow2<__hip_bfloat16>(float lo, float hi) {
    const f32x2v v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
template <> __device__ __forceinline__ uint32_t narrow2<__half>(float lo, float hi) {
    const f32x2v v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

template <typename T> __device__ __forceinline__ void widen(u32x4 r, float (&v)[Unit<T>::n]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = r[i];   // a copy: a bit cast of a vector's element takes the vector's first
            v[i] = __builtin_bit_cast(float, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) widen2<T>(r[i], v[2 * i], v[2 * i + 1]);
    }
}
template <typename T> __device__ __forceinline__ u32x4 narrow(const float (&v)[Unit<T>::n]) {
    u32x4 r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = narrow2<T>(v[2 * i], v[2 * i + 1]);
    }
    return r;
}

// A row's last unit of `left` < Unit<T>::n elements; what is beyond reads 0.
template <typename T> __device__ __forceinline__ u32x4 load_part(const T* p, int left) {
    if constexpr (sizeof(T) == 4) {
        u32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < left) r[i] = ((const CRESSO_GLOBAL raw32_t*)p)[i];
        return r;
    } else {
        u32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < left) r[i / 2] |= (uint32_t)((const CRESSO_GLOBAL raw16_t*)p)[i] << (16 * (i & 1));
        return r;
    }
}
template <typename T> __device__ __forceinline__ void store_part(T* p, u32x4 r, int left) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < left) ((CRESSO_GLOBAL raw32_t*)p)[i] = r[i];
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < left) ((CRESSO_GLOBAL raw16_t*)p)[i] = (uint16_t)(r[i / 2] >> (16 * (i & 1)));
    }
}

// Unit u of a row of `width` elements (0 beyond it).
template <typename T> __device__ __forceinline__ u32x4 load_unit(const T* row, int64_t u, int64_t width) {
    constexpr int E = Unit<T>::n;
    const int64_t at = u * E, left = width - at;
    if (left >= E) return load16(row + at);
    if (left > 0) return load_part(row + at, (int)left);
    return u32x4{0, 0, 0, 0};
}
template <typename T> __device__ __forceinline__ void store_unit(T* row, int64_t u, int64_t width, u32x4 v) {
    constexpr int E = Unit<T>::n;
    const int64_t at = u * E, left = width - at;
    if (left >= E) store16(row + at, v);
    else if (left > 0) store_part(row + at, v, (int)left);
}

// The same past the caches, for what is not read again soon.
template <typename T> __device__ __forceinline__ void store_unit_past(T* row, int64_t u, int64_t width, u32x4 v) {
    constexpr int E = Unit<T>::n;
    const int64_t at = u * E, left = width - at;
    if (left >= E) {
        if constexpr (sizeof(T) == 4) __builtin_nontemporal_store(v, &((CRESSO_GLOBAL Raw16w*)(row + at))->v);
        else __builtin_nontemporal_store(v, &((CRESSO_GLOBAL Raw16h*)(row + at))->v);
    } else if (left > 0) {
        store_part(row + at, v, (int)left);
    }
}

inline int32_t launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? CRESSO_OK : hip_fail(e, what);
}
// row-element dtypes of these operators
inline bool row_dtype(int32_t c) { return c == CRESSO_F32 || c == CRESSO_BF16 || c == CRESSO_F16; }

// Rows of `width` elements that are read: at a stride that leaves each its own
// elements, or all of them at one place (stride 0).
inline bool row_stride_ok(const void* p, int64_t rows, int64_t width, int64_t stride) {
    return !p || rows < 2 || stride == 0 || stride >= width;
}

// Runs fn(T{}) for the element type of `code` (checked by row_dtype before).
template <typename F> inline void with_row_dtype(int32_t code, F&& fn) {
    if (code == CRESSO_F32) fn(float{});
    else if (code == CRESSO_BF16) fn(__hip_bfloat16{});
    else fn(__half{});
}

}  // namespace cresso
