// The norm over a set of gradients, and the set clipped by it.
//
//   n = s * (sum over all elements of g^2)^(1/2)   or   s * max |g|
//   out = g * s * c,   c = max_norm / n where n is finite and above max_norm, else 1
//
// Two passes over the data, each one launch over all tensors: the elements are
// cut into chunks of 32 KB, and each workgroup takes an equal run of chunks,
// whatever tensors they belong to.  The second pass begins where the first one
// ended, with what the last cache still holds, and where c * s is 1 and the
// tensors are clipped in place it reads nothing but the norm.
//
// Squares and their sums are fp64: gradients of 1e-30 and of 1e30 count as they
// are, and no order of the tensors changes more than the last bits.  fp64
// gradients whose own squares leave that range are scaled by a power of two and
// have sums of their own.  A thread's sum, the waves' and the workgroups' are
// joined in a fixed order.
//
// Bound by HBM.  840 fp32 adapters of 220 MB, nothing to clip: 35 us for the norm
// (6.3 TB/s) and 4 for the second kernel; 199 bf16 tensors of 1.2 B elements to
// fp32: 432 us (5.6 TB/s) and 1490 (4.8 TB/s read and written).  fp64 gradients
// with their three sums: 2^28 of them in 362 us, as with one (368).  With stores
// past the caches both together take 3012 instead of 1943.
#include "row_ops.hpp"

#include <algorithm>
#include <cmath>

namespace cresso {
namespace {

constexpr int CL_NT = 256;
constexpr int CL_UNITS = 8;                           // 16-byte units a thread holds of a chunk
constexpr int CL_CHUNK = CL_NT * CL_UNITS * 16;       // bytes
constexpr int CL_MAX_BLOCKS = 1024;                   // partial sums: each workgroup of the second pass adds them all up (2048 are no faster)
constexpr int CL_FILL = 250;                          // 16-byte entries of one fill launch: its arguments stay below 4 KB

// What a tensor is to the kernels: its elements from chunk `first` on, `tail` of them in its last chunk.
struct ClipEntry {
    const void* in;
    uint32_t first;
    uint32_t tail_types;   // tail << 5 | written << 4 | type << 2 | type of the output, types as CRESSO_*
};
static_assert(sizeof(ClipEntry) == 16 && (CL_CHUNK / 2) < (1 << 27), "entry");
struct ClipFill {
    u32x4 e[CL_FILL];      // entries, or two addresses of outputs each
};
struct ClipArgs {
    ClipEntry* table;
    void** outs;           // of the entries; NULL: each is its own output
    double* partials;      // [CL_SUMS][CL_MAX_BLOCKS]
    float* norm;
    uint32_t count, chunks, blocks;
    double max_norm, scale;
    int32_t write, in_place;   // write: there are outputs; in_place: every one is its input
};

int64_t element_bytes(int32_t code) { return code == CRESSO_F64 ? 8 : code == CRESSO_F32 ? 4 : 2; }

// The table, from the arguments of the launch to memory: thread i copies 16 bytes.
// 1.4 us a launch of 250 entries; nothing of the host's memory has to outlive the call.
__global__ __launch_bounds__(CL_FILL) void clip_fill_kernel(ClipFill f, u32x4* to, uint32_t count) {
    // the arguments' own memory, so that the lane's index needs no copy of them
    const auto* from = (const __attribute__((address_space(4))) u32x4*)__builtin_amdgcn_kernarg_segment_ptr();
    if (threadIdx.x < count) to[threadIdx.x] = from[threadIdx.x];
}

// Index of the entry that holds `chunk`: how many begin at or before it, less one.
__device__ __forceinline__ uint32_t entry_of(const ClipArgs& a, uint32_t chunk) {
    __shared__ uint32_t found[CL_NT / kWave];
    uint32_t n = 0;
    for (uint32_t i = threadIdx.x; i < a.count; i += CL_NT) n += a.table[i].first <= chunk ? 1u : 0u;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) n += __shfl_xor(n, m, kWave);
    if ((threadIdx.x & (kWave - 1)) == 0) found[threadIdx.x / kWave] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < CL_NT / kWave; ++w) n += found[w];
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)n) - 1;
}

// ---------------------------------------------------------------------------
// units of 16 bytes as doubles
// ---------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ u32x4 clip_load(const T* p) {
    if constexpr (sizeof(T) == 8) return load16((const float*)p);
    else return load16(p);
}
template <typename T> __device__ __forceinline__ double clip_value(u32x4 r, int i);
template <> __device__ __forceinline__ double clip_value<float>(u32x4 r, int i) {
    const uint32_t w = r[i];
    return (double)__builtin_bit_cast(float, w);
}
template <> __device__ __forceinline__ double clip_value<double>(u32x4 r, int i) {
    const uint64_t w = (uint64_t)r[2 * i] | (uint64_t)r[2 * i + 1] << 32;
    return __builtin_bit_cast(double, w);
}
template <> __device__ __forceinline__ double clip_value<__hip_bfloat16>(u32x4 r, int i) {
    const uint32_t w = i & 1 ? r[i / 2] & 0xffff0000u : r[i / 2] << 16;
    return (double)__builtin_bit_cast(float, w);
}
template <> __device__ __forceinline__ double clip_value<__half>(u32x4 r, int i) {
    const uint32_t w = r[i / 2];
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    return (double)(float)h[i & 1];
}

// What a norm is the root of: a sum of squares; for fp64 gradients three, so
// that no square leaves a double's range; or the largest magnitude.
enum ClipKind { CLIP_SQUARES, CLIP_WIDE, CLIP_LARGEST };
constexpr int CL_SUMS = 3;   // doubles of a partial sum, at most
// Squares of 2^-480 to 2^480 stay above 2^-960 and, 2^44 of them added up, below
// 2^1004; larger magnitudes are added up as those of g / 2^600, smaller ones of g * 2^600.
constexpr double CL_HIGH = 0x1p480, CL_LOW = 0x1p-480, CL_DOWN = 0x1p-600, CL_UP = 0x1p600;

// A largest magnitude is the largest pattern of |g| as a double: patterns order
// as the magnitudes do, NaN above infinity.
template <ClipKind KIND> struct ClipSum {
    static constexpr int N = KIND == CLIP_WIDE ? CL_SUMS : 1;
    double v[N];   // squares, those of large and of small numbers; or the largest
    template <typename T> __device__ __forceinline__ void add(double g) {
        if constexpr (KIND == CLIP_LARGEST) {
            largest(fabs(g));
        } else if constexpr (KIND == CLIP_WIDE && sizeof(T) == 8) {
            const double size = fabs(g);
            const bool high = size > CL_HIGH, low = size < CL_LOW;   // NaN is neither
            const double mid = high || low ? 0.0 : g, down = high ? g * CL_DOWN : 0.0, up = low ? g * CL_UP : 0.0;
            v[0] = fma(mid, mid, v[0]);
            v[1] = fma(down, down, v[1]);
            v[2] = fma(up, up, v[2]);
        } else {
            v[0] = fma(g, g, v[0]);
        }
    }
    __device__ __forceinline__ void largest(double o) {
        const uint64_t x = (uint64_t)__double_as_longlong(v[0]), y = (uint64_t)__double_as_longlong(o);
        v[0] = __longlong_as_double((long long)(x > y ? x : y));
    }
    __device__ __forceinline__ void join(const ClipSum& o) {
        if constexpr (KIND == CLIP_LARGEST) {
            largest(o.v[0]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += o.v[i];
        }
    }
    __device__ __forceinline__ double norm() const {
        if constexpr (KIND == CLIP_LARGEST) return v[0];
        if constexpr (KIND == CLIP_WIDE) {   // the sums that are far below another add nothing to it
            if (v[1] > 0.0) return sqrt(v[1] + v[0] * CL_DOWN * CL_DOWN) * CL_UP;
            if (v[0] == 0.0) return sqrt(v[2]) * CL_DOWN;
            return sqrt(v[0] + v[2] * CL_DOWN * CL_DOWN);
        }
        return sqrt(v[0]);
    }
};

template <typename T, ClipKind KIND> __device__ __forceinline__ void clip_sum(const T* at, uint32_t left, ClipSum<KIND> (&sum)[2]) {
    constexpr int E = 16 / (int)sizeof(T);
    constexpr uint32_t whole = CL_CHUNK / sizeof(T);
    if (left == whole) {
        u32x4 r[CL_UNITS];
#pragma unroll
        for (int u = 0; u < CL_UNITS; ++u) r[u] = clip_load(at + (uint32_t)(u * CL_NT + threadIdx.x) * E);
#pragma unroll
        for (int u = 0; u < CL_UNITS; ++u)
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i & 1].template add<T>(clip_value<T>(r[u], i));
        return;
    }
    for (uint32_t u = threadIdx.x * E; u < left; u += CL_NT * E) {
        if (u + E <= left) {
            const u32x4 r = clip_load(at + u);
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i & 1].template add<T>(clip_value<T>(r, i));
        } else {
            for (uint32_t i = u; i < left; ++i) {
                if constexpr (sizeof(T) == 8) sum[0].template add<T>(at[i]);
                else sum[0].template add<T>((double)to_f(at[i]));
            }
        }
    }
}

// Everybody's sums joined: lanes, then waves, in their order.
template <ClipKind KIND> __device__ __forceinline__ void clip_join(ClipSum<KIND>& s, ClipSum<KIND>* lds) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        ClipSum<KIND> o;
#pragma unroll
        for (int i = 0; i < ClipSum<KIND>::N; ++i) o.v[i] = __shfl_xor(s.v[i], m, kWave);
        s.join(o);
    }
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = s;
    __syncthreads();
    s = lds[0];
#pragma unroll
    for (int w = 1; w < CL_NT / kWave; ++w) s.join(lds[w]);
}

__device__ __forceinline__ void clip_run(const ClipArgs& a, uint32_t& lo, uint32_t& hi) {
    lo = (uint32_t)((uint64_t)blockIdx.x * a.chunks / a.blocks);
    hi = (uint32_t)((uint64_t)(blockIdx.x + 1) * a.chunks / a.blocks);
}

template <ClipKind KIND> __global__ __launch_bounds__(CL_NT) void clip_norm_kernel(ClipArgs a) {
    __shared__ ClipSum<KIND> lds[CL_NT / kWave];
    uint32_t lo, hi;
    clip_run(a, lo, hi);
    uint32_t e = entry_of(a, lo);
    ClipSum<KIND> sum[2] = {};
    ClipEntry t = a.table[e];
    uint32_t end = e + 1 < a.count ? a.table[e + 1].first : a.chunks;
    for (uint32_t c = lo; c < hi; ++c) {
        if (c == end) {
            t = a.table[++e];
            end = e + 1 < a.count ? a.table[e + 1].first : a.chunks;
        }
        const char* at = (const char*)t.in + (uint64_t)(c - t.first) * CL_CHUNK;
        const uint32_t tail = t.tail_types >> 5, type = (t.tail_types >> 2) & 3;
        const bool last = c + 1 == end;
        if (type == CRESSO_F32) clip_sum<float>((const float*)at, last ? tail : CL_CHUNK / 4, sum);
        else if (type == CRESSO_BF16) clip_sum<__hip_bfloat16>((const __hip_bfloat16*)at, last ? tail : CL_CHUNK / 2, sum);
        else if (type == CRESSO_F16) clip_sum<__half>((const __half*)at, last ? tail : CL_CHUNK / 2, sum);
        else clip_sum<double>((const double*)at, last ? tail : CL_CHUNK / 8, sum);
    }
    sum[0].join(sum[1]);
    clip_join(sum[0], lds);
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < ClipSum<KIND>::N; ++i) a.partials[i * CL_MAX_BLOCKS + blockIdx.x] = sum[0].v[i];
    }
}

// The E elements of r times f (and late), in fp64, rounded to fp32 and where `out` has 16
// bits from there: off by at most 2^-24 of the result more than half a step.
template <typename T, typename O> __device__ __forceinline__ void clip_scale_unit(u32x4 r, O* out, double f, double late) {
    constexpr int E = 16 / (int)sizeof(T);
    if constexpr (sizeof(O) == 8) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint64_t v = (uint64_t)__double_as_longlong(clip_value<T>(r, i) * f * late);
            w[2 * i] = (uint32_t)v;
            w[2 * i + 1] = (uint32_t)(v >> 32);
        }
        store16((float*)out, w);
    } else {
        constexpr int EO = Unit<O>::n;   // a unit of 16 bytes in is one or two of fp32 out
#pragma unroll
        for (int h = 0; h < E / EO; ++h) {
            float v[EO];
#pragma unroll
            for (int i = 0; i < EO; ++i) v[i] = (float)(clip_value<T>(r, h * EO + i) * f);
            store16(out + h * EO, narrow<O>(v));
        }
    }
}
template <typename T, typename O> __device__ __forceinline__ void clip_scale(const T* in, O* out, uint32_t left, double f, double late = 1.0) {
    constexpr int E = 16 / (int)sizeof(T);
    if (left == CL_CHUNK / sizeof(T)) {
        u32x4 r[CL_UNITS];
#pragma unroll
        for (int u = 0; u < CL_UNITS; ++u) r[u] = clip_load(in + (uint32_t)(u * CL_NT + threadIdx.x) * E);
#pragma unroll
        for (int u = 0; u < CL_UNITS; ++u) clip_scale_unit<T, O>(r[u], out + (uint32_t)(u * CL_NT + threadIdx.x) * E, f, late);
        return;
    }
    for (uint32_t u = threadIdx.x * E; u < left; u += CL_NT * E) {
        if (u + E <= left) {
            clip_scale_unit<T, O>(clip_load(in + u), out + u, f, late);
        } else {
            for (uint32_t i = u; i < left; ++i) {
                if constexpr (sizeof(T) == 8) out[i] = in[i] * f * late;
                else out[i] = from_w<O>((float)((double)to_f(in[i]) * f));
            }
        }
    }
}

template <ClipKind KIND> __global__ __launch_bounds__(CL_NT) void clip_scale_kernel(ClipArgs a) {
    __shared__ ClipSum<KIND> lds[CL_NT / kWave];
    ClipSum<KIND> sum = {};
#pragma unroll
    for (int i = 0; i < CL_MAX_BLOCKS / CL_NT; ++i) {
        const uint32_t at = i * CL_NT + threadIdx.x;
        if (at >= a.blocks) continue;
        ClipSum<KIND> o;
#pragma unroll
        for (int k = 0; k < ClipSum<KIND>::N; ++k) o.v[k] = a.partials[k * CL_MAX_BLOCKS + at];
        sum.join(o);
    }
    clip_join(sum, lds);
    const double norm = sum.norm() * fabs(a.scale);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
    if (!a.write) return;
    double f = a.scale, late = 1.0;   // late: of fp64 gradients, where max_norm / norm has too few bits by itself
    if (norm > a.max_norm && norm < INFINITY) {
        double by = a.max_norm / norm;
        if (by < 0x1p-960) {
            by = a.max_norm * CL_UP / norm;
            late = CL_DOWN;
        }
        f *= by;
    }
    const double whole = f * late;
    if (a.in_place && whole == 1.0) return;
    uint32_t lo, hi;
    clip_run(a, lo, hi);
    uint32_t e = entry_of(a, hi - 1);
    ClipEntry t = a.table[e];
    uint32_t end = e + 1 < a.count ? a.table[e + 1].first : a.chunks;
    for (uint32_t c = hi; c-- > lo;) {   // backwards: what was read last is still in a cache
        if (c < t.first) {
            end = t.first;
            t = a.table[--e];
        }
        void* const to = a.outs ? a.outs[e] : const_cast<void*>(t.in);
        if (!(t.tail_types & 16) || (to == t.in && whole == 1.0)) continue;
        const uint32_t tail = t.tail_types >> 5, types = t.tail_types & 15, type = types >> 2;
        const uint32_t size = type == CRESSO_F64 ? 8 : type == CRESSO_F32 ? 4 : 2, out_size = (types & 3) == CRESSO_F64 ? 8 : (types & 3) == CRESSO_F32 ? 4 : 2;
        const uint64_t first = (uint64_t)(c - t.first) * (CL_CHUNK / size);
        const char* in = (const char*)t.in + first * size;
        char* out = (char*)to + first * out_size;
        const uint32_t left = c + 1 == end ? tail : CL_CHUNK / size;
        if (types == (CRESSO_F32 << 2 | CRESSO_F32)) clip_scale((const float*)in, (float*)out, left, whole);
        else if (types == (CRESSO_BF16 << 2 | CRESSO_BF16)) clip_scale((const __hip_bfloat16*)in, (__hip_bfloat16*)out, left, whole);
        else if (types == (CRESSO_BF16 << 2 | CRESSO_F32)) clip_scale((const __hip_bfloat16*)in, (float*)out, left, whole);
        else if (types == (CRESSO_F16 << 2 | CRESSO_F16)) clip_scale((const __half*)in, (__half*)out, left, whole);
        else if (types == (CRESSO_F16 << 2 | CRESSO_F32)) clip_scale((const __half*)in, (float*)out, left, whole);
        else clip_scale((const double*)in, (double*)out, left, f, late);
    }
}

bool clip_dtype(int32_t c) { return c >= CRESSO_F32 && c <= CRESSO_BF16; }

int32_t check_clip(const cresso_grad_desc* g, int32_t count, uint32_t& entries, uint32_t& chunks) {
    if (count < 0 || (count > 0 && !g)) return fail(CRESSO_E_INVALID, "gradient norm: null argument or negative count");
    int64_t total = 0;
    entries = 0;
    for (int32_t i = 0; i < count; ++i) {
        if (!clip_dtype(g[i].dtype)) return fail(CRESSO_E_UNSUPPORTED, "gradient norm: dtype %d not supported (f32, f64, f16, bf16)", g[i].dtype);
        if (g[i].numel < 0) return fail(CRESSO_E_INVALID, "gradient norm: tensor %d has a negative size", i);
        if (g[i].numel > 0 && !g[i].grad) return fail(CRESSO_E_INVALID, "gradient norm: tensor %d is null", i);
        if (g[i].out && g[i].out_dtype != g[i].dtype && (g[i].out_dtype != CRESSO_F32 || g[i].dtype == CRESSO_F64))
            return fail(CRESSO_E_UNSUPPORTED, "gradient norm: tensor %d of dtype %d to dtype %d (its own or, of 16 bits, f32)", i, g[i].dtype,
                        g[i].out_dtype);
        const int64_t per = CL_CHUNK / element_bytes(g[i].dtype);
        total += g[i].numel / per + (g[i].numel % per ? 1 : 0);
        if (total >= (int64_t)1 << 31) return fail(CRESSO_E_UNSUPPORTED, "gradient norm: more elements than one call takes");
        entries += g[i].numel > 0;
    }
    chunks = (uint32_t)total;
    return CRESSO_OK;
}
// entries, then their outputs
size_t clip_bytes(uint32_t entries) { return CL_SUMS * CL_MAX_BLOCKS * sizeof(double) + (size_t)entries * sizeof(ClipEntry) + ((size_t)entries + 1) / 2 * 16; }
}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" size_t cresso_clip_workspace_bytes(const cresso_grad_desc* grads, int32_t count) {
    uint32_t entries, chunks;
    if (check_clip(grads, count, entries, chunks) != CRESSO_OK) return 0;
    return clip_bytes(entries);
}

extern "C" int32_t cresso_clip_gradients(const cresso_grad_desc* grads, int32_t count, int32_t norm_kind, double max_norm,
                                         double grad_scale, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    uint32_t entries, chunks;
    const int32_t rc = check_clip(grads, count, entries, chunks);
    if (rc != CRESSO_OK) return rc;
    if (norm_kind != CRESSO_NORM_2 && norm_kind != CRESSO_NORM_MAX)
        return fail(CRESSO_E_INVALID, "gradient norm: unknown norm %d", norm_kind);
    if (!(max_norm >= 0.0)) return fail(CRESSO_E_INVALID, "gradient norm: max_norm must not be negative");
    if (!std::isfinite(grad_scale)) return fail(CRESSO_E_INVALID, "gradient norm: grad_scale must be finite");
    if (!norm) return fail(CRESSO_E_INVALID, "gradient norm: null norm");
    const size_t need = clip_bytes(entries);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
        return fail(CRESSO_E_INVALID, "gradient norm: workspace of %zu bytes at %p, %zu at a multiple of 16 needed", workspace_bytes, workspace, need);
    hipStream_t st = (hipStream_t)stream;
    ClipArgs a{};
    a.partials = (double*)workspace;
    a.table = (ClipEntry*)((char*)workspace + CL_SUMS * CL_MAX_BLOCKS * sizeof(double));
    a.norm = norm;
    a.count = entries;
    a.chunks = chunks;
    a.blocks = std::min<uint32_t>(chunks, CL_MAX_BLOCKS);
    a.max_norm = max_norm;
    a.scale = grad_scale;
    a.in_place = 1;
    ClipFill f;
    uint32_t held = 0;
    u32x4* to = (u32x4*)a.table;
    const auto flush = [&] {
        if (held) hipLaunchKernelGGL(clip_fill_kernel, dim3(1), dim3(CL_FILL), 0, st, f, to, held);
        to += held;
        held = 0;
    };
    uint32_t first = 0;
    bool wide = false;
    for (int32_t i = 0; i < count; ++i) {
        const cresso_grad_desc& g = grads[i];
        if (!g.numel) continue;
        const int64_t per = CL_CHUNK / element_bytes(g.dtype);
        const uint32_t n = (uint32_t)((g.numel + per - 1) / per), tail = (uint32_t)(g.numel - (int64_t)(n - 1) * per);
        const ClipEntry e = {g.grad, first, tail << 5 | (g.out ? 16u : 0u) | (uint32_t)g.dtype << 2 | (uint32_t)(g.out ? g.out_dtype : 0)};
        f.e[held++] = __builtin_bit_cast(u32x4, e);
        first += n;
        wide |= g.dtype == CRESSO_F64;
        if (g.out) a.write = 1;
        if (g.out && g.out != g.grad) a.in_place = 0;
        if (held == CL_FILL) flush();
    }
    if (!a.in_place) {   // behind the entries
        a.outs = (void**)(a.table + entries);
        uint64_t pair[2] = {0, 0};
        uint32_t half = 0;
        for (int32_t i = 0; i < count; ++i) {
            if (!grads[i].numel) continue;
            pair[half++] = (uint64_t)(uintptr_t)grads[i].out;
            if (half < 2) continue;
            f.e[held++] = u32x4{(uint32_t)pair[0], (uint32_t)(pair[0] >> 32), (uint32_t)pair[1], (uint32_t)(pair[1] >> 32)};
            half = 0;
            if (held == CL_FILL) flush();
        }
        if (half) f.e[held++] = u32x4{(uint32_t)pair[0], (uint32_t)(pair[0] >> 32), 0u, 0u};
    }
    flush();
    const auto run = [&](auto norm_kernel, auto scale_kernel) {
        if (a.blocks) hipLaunchKernelGGL(norm_kernel, dim3(a.blocks), dim3(CL_NT), 0, st, a);
        hipLaunchKernelGGL(scale_kernel, dim3(a.write ? std::max(1u, a.blocks) : 1), dim3(CL_NT), 0, st, a);
    };
    if (norm_kind == CRESSO_NORM_MAX) run(clip_norm_kernel<CLIP_LARGEST>, clip_scale_kernel<CLIP_LARGEST>);
    else if (wide) run(clip_norm_kernel<CLIP_WIDE>, clip_scale_kernel<CLIP_WIDE>);
    else run(clip_norm_kernel<CLIP_SQUARES>, clip_scale_kernel<CLIP_SQUARES>);
    return launched("gradient norm");
}
