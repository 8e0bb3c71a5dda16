// Product with a weight that is held in 8-bit floating point (e4m3), one fp32
// scale for each 128 x 128 block:
//
//   y[m,n] = sum over blocks b of k:  s[n/128,b] * sum_{k in b} r[m,k]*w[n,k]
//   r[m,k] = 2^e * e4m3(x[m,k] * 2^-e),  e: the smallest whole number with max_{k in b} |x[m,k]| <= 448 * 2^e, at least -117
//
// and the gradient of x, the same with the roles of n and k exchanged (w read
// along n).  A power of two loses nothing against a free scale, since e4m3 is
// a floating point format, and costs no rounding of its own: r has four
// significant bits and is held exactly as bf16, as is each e4m3 value.  So
// the products are formed by the bf16 matrix instructions, exactly and with
// sums of 24 bits.  The 8-bit matrix instructions are not used: they align the
// products of a group before they add them and keep 13 bits below the largest
// (2^16 + 2^2 - 2^16 gives 0), which is 1.4e-5 of the result for normally
// distributed numbers against 6e-9, and more where products differ in size.
// A block's partial sum is multiplied by its fp32 scale when it is added to
// the fp32 accumulator.
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int BP = 128;            // block of a scale
constexpr int BP_NT = 256;
constexpr int BP_TM = 128, BP_TN = 128;
constexpr int BP_MIN_EXP = -117;   // the smallest step, 2^-9 * 2^-117, is a normal number

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// ---------------------------------------------------------------------------
// x rounded to e4m3 times a power of two, as bf16: 16 lanes hold one row's 128
// elements
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(BP_NT) void round_rows_kernel(const T* x, int64_t rows, int64_t width, int64_t stride,
                                                           uint16_t* q, int64_t q_stride) {
    const int64_t blocks = q_stride / BP;
    const int64_t job = ((int64_t)blockIdx.x * BP_NT + threadIdx.x) / 16;
    const int part = threadIdx.x & 15;
    if (job >= rows * blocks) return;
    const int64_t row = job / blocks, b = job - row * blocks, at = b * BP + part * 8;
    float v[8];
    const T* p = x + row * stride;
    if constexpr (sizeof(T) == 4) {
        float lo[4], hi[4];
        widen<T>(load_unit(p, at / 4, width), lo);
        widen<T>(load_unit(p, at / 4 + 1, width), hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = lo[i];
            v[4 + i] = hi[i];
        }
    } else {
        widen<T>(load_unit(p, at / 8, width), v);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.0f);
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, kWave));
    int e = 0;
    if (top > 0.0f) {
        const float f = frexpf(top, &e);   // top = f * 2^e, 0.5 <= f < 1; 448 = 0.875 * 2^9
        e = max(BP_MIN_EXP, e - 9 + (f > 0.875f));
    }
    const float unit = ldexpf(1.0f, e);
    const float most = e == 120 ? 240.0f : 448.0f;   // 256 * 2^120 is beyond fp32
    u32x4 r;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        float t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t[i] = ldexpf(v[2 * h + i], -e);
            // the format has no infinities
            t[i] = fabsf(t[i]) < INFINITY ? fminf(fmaxf(t[i], -most), most) : __builtin_nanf("");
        }
        const uint32_t pair = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
        r[h] = narrow2<__hip_bfloat16>(__builtin_amdgcn_cvt_f32_fp8(pair, 0) * unit, __builtin_amdgcn_cvt_f32_fp8(pair, 1) * unit);
    }
    *(u32x4*)(q + row * q_stride + at) = r;
}

// ---------------------------------------------------------------------------
// The weight's other layout: along n for the gradient (TURN), or only with
// rows padded to whole 16-byte pieces.  64 x 64 bytes a block.
// ---------------------------------------------------------------------------
template <bool TURN>
__global__ __launch_bounds__(BP_NT) void lay_out_kernel(const uint8_t* w, int64_t rows, int64_t cols, int64_t stride,
                                                        uint8_t* out, int64_t out_stride) {
    __shared__ uint8_t tile[64][68];
    const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
    for (int i = threadIdx.x; i < 64 * 64; i += BP_NT) {
        const int r = i / 64, c = i & 63;
        tile[r][c] = r0 + r < rows && c0 + c < cols ? w[(r0 + r) * stride + c0 + c] : 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += BP_NT) {
        const int a = i / 64, b = i & 63;
        if constexpr (TURN) {
            if (c0 + a < cols && r0 + b < out_stride) out[(c0 + a) * out_stride + r0 + b] = tile[b][a];
        } else {
            if (r0 + a < rows && c0 + b < out_stride) out[(r0 + a) * out_stride + c0 + b] = tile[a][b];
        }
    }
}

// ---------------------------------------------------------------------------
// out[m][n] = sum_k r[m][k] w[n][k] with scales.  r is padded to whole blocks
// of k (zeros); w's rows hold `depth` bytes, a multiple of 16.
// ---------------------------------------------------------------------------
struct ProductArgs {
    const uint16_t* r;
    const uint8_t* w;
    const float* scales;
    void* out;
    int64_t rows, cols, depth;          // m, n, k
    int64_t r_stride, w_stride, out_stride;
    int64_t scale_n, scale_k;           // strides of the scales along n's and k's blocks
};

// Byte offsets in the tiles, whose rows are one block of k: 256 bytes of r,
// 128 of w.  The 16-byte pieces of a row change places by the row's number, so
// that 16 rows' pieces of one column lie in different banks.
__device__ __forceinline__ int r_at(int row, int piece) { return row * 256 + ((piece ^ (row & 15)) * 16); }
__device__ __forceinline__ int w_at(int row, int piece) { return row * 128 + ((piece ^ ((row >> 1) & 7)) * 16); }

// eight e4m3 values as bf16
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T>
__global__ __launch_bounds__(BP_NT) void product_kernel(ProductArgs a) {
    __shared__ __align__(16) uint8_t rt[BP_TM * 256], wt[BP_TN * 128];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int64_t m0 = (int64_t)blockIdx.y * BP_TM, n0 = (int64_t)blockIdx.x * BP_TN;
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int l16 = lane & 15, quad = lane >> 4;
    f32x4 acc[4][4];   // [n][m]
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    const int64_t blocks = (a.depth + BP - 1) / BP;
    for (int64_t b = 0; b < blocks; ++b) {
        u32x4 gr[8], gw[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int piece = tid + i * BP_NT, row = piece >> 4, col = piece & 15;
            gr[i] = u32x4{0, 0, 0, 0};
            if (m0 + row < a.rows) gr[i] = *(const u32x4*)(a.r + (m0 + row) * a.r_stride + b * BP + col * 8);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int piece = tid + i * BP_NT, row = piece >> 3, col = piece & 7;
            const int64_t k = b * BP + col * 16;
            gw[i] = u32x4{0, 0, 0, 0};
            if (n0 + row < a.cols && k < a.depth) gw[i] = *(const u32x4*)(a.w + (n0 + row) * a.w_stride + k);
        }
        const float sc = a.scales[n0 / BP * a.scale_n + b * a.scale_k];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int piece = tid + i * BP_NT;
            *(u32x4*)(rt + r_at(piece >> 4, piece & 15)) = gr[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int piece = tid + i * BP_NT;
            *(u32x4*)(wt + w_at(piece >> 3, piece & 7)) = gw[i];
        }
        __syncthreads();
        f32x4 p[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) p[i][j] = f32x4{0, 0, 0, 0};
        // a lane's k: 32 of its quarter of the block, 8 for each of four steps
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 fw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) fw[i] = *(const u32x4*)(wt + w_at(wn + i * 16 + l16, quad * 2 + h));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                bf16x8 fr[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) fr[j] = *(const bf16x8*)(rt + r_at(wm + j * 16 + l16, quad * 4 + h * 2 + s));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bf16x8 f = widen8(fw[i][2 * s], fw[i][2 * s + 1]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, fr[j], p[i][j], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] += p[i][j][e] * sc;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t m = m0 + wm + j * 16 + l16;
        if (m >= a.rows) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t n = n0 + wn + i * 16 + quad * 4;
            T* to = (T*)a.out + m * a.out_stride + n;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < a.cols) to[e] = from_w<T>(acc[i][j][e]);
        }
    }
}

// Blocks of a weight to e4m3 and their scales, 16 rows of 16 lanes at a time.
template <typename T>
__global__ __launch_bounds__(BP_NT) void quantize_blocks_kernel(const T* w, int64_t rows, int64_t cols, int64_t stride,
                                                                uint8_t* q, float* scales) {
    __shared__ float part[BP_NT / kWave];
    const int64_t r0 = (int64_t)blockIdx.y * BP, c0 = (int64_t)blockIdx.x * BP;
    const int r_part = threadIdx.x / 16, c_part = threadIdx.x & 15;
    constexpr int E = Unit<T>::n, U = 8 / E;
    float top = 0.0f;
    const auto load = [&](int i, float (&v)[8]) {
        const int64_t r = r0 + i * 16 + r_part;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
        if (r >= rows) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float t[E];
            widen<T>(load_unit(w + r * stride, (c0 + c_part * 8) / E + u, cols), t);
#pragma unroll
            for (int k = 0; k < E; ++k) v[u * E + k] = t[k];
        }
    };
    for (int i = 0; i < 8; ++i) {
        float v[8];
        load(i, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k]) < INFINITY ? fabsf(v[k]) : 0.0f);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, kWave));
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = top;
    __syncthreads();
    for (int i = 0; i < BP_NT / kWave; ++i) top = fmaxf(top, part[i]);
    // a block of zeros, or of numbers too small to divide by, takes the scale 1
    const float scale = top >= 0x1p-100f ? top / 448.0f : 1.0f;
    if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = scale;
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + i * 16 + r_part, c = c0 + c_part * 8;
        if (r >= rows) continue;
        float v[8];
        load(i, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float t = v[k] / scale;
            t = fabsf(t) < INFINITY ? fminf(fmaxf(t, -448.0f), 448.0f) : __builtin_nanf("");
            if (c + k < cols) q[r * cols + c + k] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(t, t, 0, false);
        }
    }
}

struct ProductLayout {
    int64_t r, w, total, r_stride, w_stride;
};
// rows x cols outputs of depth `depth`; copy: the weight is laid out anew
ProductLayout product_layout(int64_t rows, int64_t cols, int64_t depth, bool copy) {
    ProductLayout o{};
    int64_t off = 0;
    const auto take = [&](int64_t b) { const int64_t at = off; off = up(off + b, 256); return at; };
    o.r_stride = up(depth, BP);
    o.r = take(rows * o.r_stride * 2);
    o.w_stride = up(depth, 16);
    if (copy) o.w = take(cols * o.w_stride);
    o.total = std::max<int64_t>(off, 256);
    return o;
}

int32_t check_product(const char* what, int64_t rows, int64_t cols, int64_t depth, int32_t dtype) {
    if (!row_dtype(dtype)) return fail(CRESSO_E_UNSUPPORTED, "%s: dtype %d not supported (f32, bf16, f16)", what, dtype);
    if (rows < 0 || cols < 0 || depth < 0) return fail(CRESSO_E_INVALID, "%s: negative size", what);
    if (rows >= (int64_t)1 << 22 || cols >= (int64_t)1 << 21 || depth >= (int64_t)1 << 21 || rows * (depth / BP + 1) >= (int64_t)1 << 28)
        return fail(CRESSO_E_UNSUPPORTED, "%s: %lld x %lld x %lld is more than one call takes", what, (long long)rows,
                    (long long)cols, (long long)depth);
    return CRESSO_OK;
}
bool needs_copy(const void* w, int64_t w_stride, int64_t depth, int32_t turned) {
    return turned || depth % 16 || w_stride % 16 || ((uintptr_t)w & 15);
}

}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" size_t cresso_block_product_workspace_bytes(int64_t rows, int64_t cols, int64_t depth, const void* w,
                                                       int64_t w_stride, int32_t turned) {
    if (check_product("block product", rows, cols, depth, CRESSO_F32) != CRESSO_OK) return 0;
    return (size_t)product_layout(rows, cols, depth, needs_copy(w, w_stride, depth, turned)).total;
}

extern "C" int32_t cresso_block_product(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols,
                                        int64_t depth, const void* w, int64_t w_stride, const float* scales,
                                        int64_t scale_stride, int32_t turned, void* out, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const int32_t rc = check_product("block product", rows, cols, depth, dtype);
    if (rc != CRESSO_OK) return rc;
    if (rows == 0 || cols == 0) return CRESSO_OK;
    if (!out || (depth > 0 && (!x || !w || !scales))) return fail(CRESSO_E_INVALID, "block product: null argument");
    const bool copy = needs_copy(w, w_stride, depth, turned);
    const ProductLayout o = product_layout(rows, cols, depth, copy);
    if (!workspace || workspace_bytes < (size_t)o.total)
        return fail(CRESSO_E_INVALID, "block product: workspace of %zu bytes, %lld needed", workspace_bytes, (long long)o.total);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    ProductArgs a{};
    a.r = (const uint16_t*)(ws + o.r);
    a.r_stride = o.r_stride;
    a.w = copy ? (uint8_t*)ws + o.w : (const uint8_t*)w;
    a.w_stride = copy ? o.w_stride : w_stride;
    a.scales = scales;
    a.scale_n = turned ? 1 : scale_stride;
    a.scale_k = turned ? scale_stride : 1;
    a.out = out;
    a.out_stride = cols;
    a.rows = rows;
    a.cols = cols;
    a.depth = copy ? o.w_stride : depth;
    if (depth > 0) {
        if (copy) {
            const int64_t r = turned ? depth : cols, c = turned ? cols : depth;   // the weight as it is held
            const dim3 grid((uint32_t)(up(c, 64) / 64), (uint32_t)(up(r, 64) / 64));
            if (turned)
                hipLaunchKernelGGL(lay_out_kernel<true>, grid, dim3(BP_NT), 0, st, (const uint8_t*)w, r, c, w_stride,
                                   (uint8_t*)ws + o.w, o.w_stride);
            else
                hipLaunchKernelGGL(lay_out_kernel<false>, grid, dim3(BP_NT), 0, st, (const uint8_t*)w, r, c, w_stride,
                                   (uint8_t*)ws + o.w, o.w_stride);
        }
        const int64_t jobs = rows * (o.r_stride / BP);
        with_row_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            hipLaunchKernelGGL(round_rows_kernel<T>, dim3((uint32_t)((jobs * 16 + BP_NT - 1) / BP_NT)), dim3(BP_NT), 0, st,
                               (const T*)x, rows, depth, x_stride, (uint16_t*)(ws + o.r), o.r_stride);
        });
    }
    with_row_dtype(dtype, [&](auto t) {
        const dim3 grid((uint32_t)((cols + BP_TN - 1) / BP_TN), (uint32_t)((rows + BP_TM - 1) / BP_TM));
        hipLaunchKernelGGL(product_kernel<decltype(t)>, grid, dim3(BP_NT), 0, st, a);
    });
    return launched("block product");
}

extern "C" int32_t cresso_block_quantize(const void* w, int64_t w_stride, int32_t dtype, int64_t rows, int64_t cols,
                                         void* values, float* scales, void* stream) {
    const int32_t rc = check_product("block quantization", rows, cols, 0, dtype);
    if (rc != CRESSO_OK) return rc;
    if (rows == 0 || cols == 0) return CRESSO_OK;
    if (!w || !values || !scales) return fail(CRESSO_E_INVALID, "block quantization: null argument");
    with_row_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const dim3 grid((uint32_t)(up(cols, BP) / BP), (uint32_t)(up(rows, BP) / BP));
        hipLaunchKernelGGL(quantize_blocks_kernel<T>, grid, dim3(BP_NT), 0, (hipStream_t)stream, (const T*)w, rows, cols,
                           w_stride, (uint8_t*)values, scales);
    });
    return launched("block quantization");
}
