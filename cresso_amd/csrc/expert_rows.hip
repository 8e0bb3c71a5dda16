// Rows on their way from tokens to experts and back.
//
//   dispatch: rows[place(t,k)] = x[t]
//   combine:  out[t] = sum over k of w[t,k] * rows[place(t,k)]          (its gradient without weights is dispatch's)
//   gradient: d_rows[place(t,k)] = w[t,k] * d_out[t],  d_w[t,k] = d_out[t] . rows[place(t,k)]
//
// Each token's lanes read its row once and write, or read, its slots' rows, 16
// bytes a lane; sums are fp32, over k in order.  Many tokens are bound by HBM:
// 16384 x 2048 bf16, two experts a token: dispatch 34.9 us (5.8 TB/s read and
// written), combine 44.2 (4.6), its gradient 68.3 (4.9).  Few are bound by the
// chain of loads of one token, whose lanes take its columns four units at a time
// and its slots one after another (two at a time in combine): 8 x 2048 with two
// experts 3.0, 3.4 and 5.5 us, 333 x 1001 fp32 with three 4.6, 5.3 and 10.1, but 8 x 7168
// with eight 15.0, 20.7 and 41.8.  8 to 64 lanes a token, as its row has units, so that narrow rows leave no lanes idle.
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

constexpr int ER_NT = 256;
constexpr int ER_MAX_TOP = 32;
constexpr int64_t ER_MAX_TOKENS = (1 << 26) - 16;   // a launch has fewer than 2^32 threads: 64 a token, in workgroups of 4 tokens or more

struct RowsArgs {
    const void *x, *d_out;         // rows that are read
    const int32_t *experts, *places;
    const float* weights;
    void* out;
    float* d_weights;
    int64_t x_stride, d_out_stride, tokens, width, slots;
    int32_t top, lanes;            // lanes of a token: a power of two, 8 to 64
};

// The token of this thread's lanes, and its lane among them.
__device__ __forceinline__ int64_t token_of(const RowsArgs& a, int& lane) {
    lane = threadIdx.x & (a.lanes - 1);
    return (int64_t)blockIdx.x * (ER_NT / a.lanes) + threadIdx.x / a.lanes;
}
// A slot's row, or -1 for a place that is none.
__device__ __forceinline__ int64_t slot_place(const RowsArgs& a, int64_t slot) {
    const int64_t p = a.places[slot];
    return p >= 0 && p < a.slots ? p : -1;
}

// A row is read once and held while it is written to each of its slots.
template <typename T> __global__ __launch_bounds__(ER_NT) void dispatch_kernel(RowsArgs a) {
    int lane;
    const int64_t token = token_of(a, lane);
    if (token >= a.tokens) return;
    constexpr int E = Unit<T>::n, U = 4;
    const int64_t units = (a.width + E - 1) / E;
    const T* row = (const T*)a.x + token * a.x_stride;
    for (int64_t u0 = lane; u0 < units; u0 += (int64_t)a.lanes * U) {
        u32x4 r[U];
#pragma unroll
        for (int i = 0; i < U; ++i) r[i] = load_unit(row, u0 + i * a.lanes, a.width);
        for (int k = 0; k < a.top; ++k) {
            const int64_t place = slot_place(a, token * a.top + k);
            if (place < 0) continue;
            const bool there = a.experts[token * a.top + k] >= 0;
            T* to = (T*)a.out + place * a.width;
#pragma unroll
            for (int i = 0; i < U; ++i) store_unit(to, u0 + i * a.lanes, a.width, there ? r[i] : u32x4{0, 0, 0, 0});
        }
    }
}

// Four units of a row on their way a lane: 44 us for 16384 x 2048 bf16, 51 with one.
template <typename T> __global__ __launch_bounds__(ER_NT) void combine_kernel(RowsArgs a) {
    int lane;
    const int64_t token = token_of(a, lane);
    if (token >= a.tokens) return;
    constexpr int E = Unit<T>::n, U = 4;
    const int64_t units = (a.width + E - 1) / E;
    for (int64_t u0 = lane; u0 < units; u0 += (int64_t)a.lanes * U) {
        float sum[U][E] = {};
#pragma unroll 2
        for (int k = 0; k < a.top; ++k) {
            const int64_t slot = token * a.top + k, place = slot_place(a, slot);
            const bool there = place >= 0 && a.experts[slot] >= 0;
            if (!there) continue;
            const float w = a.weights ? a.weights[slot] : 1.0f;
            const T* row = (const T*)a.x + place * a.x_stride;
            u32x4 r[U];
#pragma unroll
            for (int i = 0; i < U; ++i) r[i] = load_unit(row, u0 + i * a.lanes, a.width);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float v[E];
                widen<T>(r[i], v);
#pragma unroll
                for (int e = 0; e < E; ++e) sum[i][e] = fmaf(w, v[e], sum[i][e]);
            }
        }
        T* to = (T*)a.out + token * a.width;
#pragma unroll
        for (int i = 0; i < U; ++i) store_unit(to, u0 + i * a.lanes, a.width, narrow<T>(sum[i]));
    }
}

// Both gradients in one pass over d_out and rows, four units of each on their way a lane (16384 x
// 2048 bf16 from memory 66 us, one of each 74); a token's lanes join their products in a fixed order.
template <typename T> __global__ __launch_bounds__(ER_NT) void combine_backward_kernel(RowsArgs a) {
    int lane;
    const int64_t token = token_of(a, lane);
    if (token >= a.tokens) return;
    constexpr int E = Unit<T>::n, U = 4;
    const int64_t units = (a.width + E - 1) / E;
    const T* by = (const T*)a.d_out + token * a.d_out_stride;
    for (int k = 0; k < a.top; ++k) {
        const int64_t slot = token * a.top + k, place = slot_place(a, slot);
        const bool there = place >= 0 && a.experts[slot] >= 0;
        float dot = 0.0f;
        if (place >= 0) {
            const float w = a.weights ? a.weights[slot] : 1.0f;
            const T* row = (const T*)a.x + place * a.x_stride;
            T* to = (T*)a.out + place * a.width;
            const bool dots = there && a.d_weights;
            for (int64_t u0 = lane; u0 < units; u0 += (int64_t)a.lanes * U) {
                u32x4 r[U], g[U];
#pragma unroll
                for (int i = 0; i < U; ++i) g[i] = load_unit(by, u0 + i * a.lanes, a.width);
#pragma unroll
                for (int i = 0; i < U; ++i) r[i] = dots ? load_unit(row, u0 + i * a.lanes, a.width) : u32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float d[E], v[E];
                    widen<T>(g[i], d);
                    if (dots) {
                        widen<T>(r[i], v);
#pragma unroll
                        for (int e = 0; e < E; ++e) dot = fmaf(d[e], v[e], dot);
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e) d[e] = there ? d[e] * w : 0.0f;
                    if (a.out) store_unit(to, u0 + i * a.lanes, a.width, narrow<T>(d));
                }
            }
        }
        if (a.d_weights) {
            for (int m = a.lanes / 2; m >= 1; m >>= 1) dot += __shfl_xor(dot, m, kWave);
            if (lane == 0) a.d_weights[slot] = there ? dot : 0.0f;
        }
    }
}

int32_t check_rows(const char* what, int32_t dtype, int64_t tokens, int32_t top, int64_t width) {
    if (!row_dtype(dtype)) return fail(CRESSO_E_UNSUPPORTED, "%s: dtype %d not supported (f32, bf16, f16)", what, dtype);
    if (tokens < 0 || width < 0) return fail(CRESSO_E_INVALID, "%s: negative size", what);
    if (top < 1 || top > ER_MAX_TOP) return fail(CRESSO_E_UNSUPPORTED, "%s: %d experts a token, 1 to %d are taken", what, top, ER_MAX_TOP);
    if (tokens > ER_MAX_TOKENS || tokens * top >= (int64_t)1 << 31 || width >= (int64_t)1 << 31)
        return fail(CRESSO_E_UNSUPPORTED, "%s: %lld rows of %lld are more than one call takes", what, (long long)(tokens * top), (long long)width);
    return CRESSO_OK;
}
RowsArgs rows_args(int32_t dtype, int64_t tokens, int32_t top, int64_t width, const int32_t* experts, const int32_t* places) {
    RowsArgs a{};
    a.experts = experts;
    a.places = places;
    a.tokens = tokens;
    a.top = top;
    a.width = width;
    a.slots = tokens * top;
    const int64_t units = (width * (dtype == CRESSO_F32 ? 4 : 2) + 15) / 16;
    a.lanes = 8;
    while (a.lanes < kWave && a.lanes < units) a.lanes *= 2;
    return a;
}
dim3 rows_grid(const RowsArgs& a) { return dim3((uint32_t)((a.tokens + ER_NT / a.lanes - 1) / (ER_NT / a.lanes))); }
}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" int32_t cresso_dispatch_rows(const void* x, int64_t x_stride, int32_t dtype, int64_t tokens, int32_t top, int64_t width,
                                        const int32_t* experts, const int32_t* places, void* rows, void* stream) {
    const int32_t rc = check_rows("dispatch", dtype, tokens, top, width);
    if (rc != CRESSO_OK) return rc;
    if (tokens == 0 || width == 0) return CRESSO_OK;
    if (!x || !experts || !places || !rows) return fail(CRESSO_E_INVALID, "dispatch: null argument");
    if (!row_stride_ok(x, tokens, width, x_stride)) return fail(CRESSO_E_INVALID, "dispatch: row stride %lld below the width", (long long)x_stride);
    RowsArgs a = rows_args(dtype, tokens, top, width, experts, places);
    a.x = x;
    a.x_stride = x_stride;
    a.out = rows;
    with_row_dtype(dtype, [&](auto t) {
        hipLaunchKernelGGL(dispatch_kernel<decltype(t)>, rows_grid(a), dim3(ER_NT), 0, (hipStream_t)stream, a);
    });
    return launched("dispatch");
}

extern "C" int32_t cresso_combine_rows(const void* rows, int64_t rows_stride, int32_t dtype, int64_t tokens, int32_t top, int64_t width,
                                       const int32_t* experts, const int32_t* places, const float* weights, void* out, void* stream) {
    const int32_t rc = check_rows("combine", dtype, tokens, top, width);
    if (rc != CRESSO_OK) return rc;
    if (tokens == 0 || width == 0) return CRESSO_OK;
    if (!rows || !experts || !places || !out) return fail(CRESSO_E_INVALID, "combine: null argument");
    if (!row_stride_ok(rows, tokens * top, width, rows_stride))
        return fail(CRESSO_E_INVALID, "combine: row stride %lld below the width", (long long)rows_stride);
    RowsArgs a = rows_args(dtype, tokens, top, width, experts, places);
    a.x = rows;
    a.x_stride = rows_stride;
    a.weights = weights;
    a.out = out;
    with_row_dtype(dtype, [&](auto t) {
        hipLaunchKernelGGL(combine_kernel<decltype(t)>, rows_grid(a), dim3(ER_NT), 0, (hipStream_t)stream, a);
    });
    return launched("combine");
}

extern "C" int32_t cresso_combine_backward(const void* rows, int64_t rows_stride, const void* d_out, int64_t d_out_stride, int32_t dtype,
                                           int64_t tokens, int32_t top, int64_t width, const int32_t* experts, const int32_t* places,
                                           const float* weights, void* d_rows, float* d_weights, void* stream) {
    const int32_t rc = check_rows("combine gradient", dtype, tokens, top, width);
    if (rc != CRESSO_OK) return rc;
    if (tokens == 0 || (!d_rows && !d_weights)) return CRESSO_OK;
    if (!experts || !places || (width > 0 && (!d_out || (d_weights && !rows)))) return fail(CRESSO_E_INVALID, "combine gradient: null argument");
    if (!row_stride_ok(rows, tokens * top, width, rows_stride) || !row_stride_ok(d_out, tokens, width, d_out_stride))
        return fail(CRESSO_E_INVALID, "combine gradient: row strides %lld and %lld, the width is %lld", (long long)rows_stride,
                    (long long)d_out_stride, (long long)width);
    RowsArgs a = rows_args(dtype, tokens, top, width, experts, places);
    a.x = rows;
    a.x_stride = rows_stride;
    a.d_out = d_out;
    a.d_out_stride = d_out_stride;
    a.weights = weights;
    a.out = d_rows;
    a.d_weights = d_weights;
    with_row_dtype(dtype, [&](auto t) {
        hipLaunchKernelGGL(combine_backward_kernel<decltype(t)>, rows_grid(a), dim3(ER_NT), 0, (hipStream_t)stream, a);
    });
    return launched("combine gradient");
}
