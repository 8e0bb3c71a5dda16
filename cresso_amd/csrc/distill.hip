// Loss against a teacher's top logits, and its gradient.  For a row z of
// student logits, with temperature t, mix a and weight w:
//
//   p = softmax over the teacher's present entries of teacher/t
//   q = softmax(z/t),  r = softmax(z)
//   loss = w * (a*t^2 * sum p*(log p - log q) + (1-a) * -log r[label])
//   dz   = w * (a*t * (q - p) + (1-a) * (r - onehot(label)))
//
// The row's maximum m and the sums of exp((z-m)/t) and exp(z-m) come from one
// pass over the row (a running maximum, sums rescaled when it grows), so the
// loss reads each logit once.  The gradient needs them all before its first
// element and reads the row again, from its end, where the caches still hold
// it; it is written as if there were no
// teacher and no label; their few places are written again afterwards from
// logits that were read before, so it may take the logits' own memory: the
// same rows at the same stride.  Any other share in what is read is refused,
// since a workgroup would overwrite what another has yet to read.
//
// Exponents are kept in base 2: (z-m)*c with c = log2(e)/t.  The difference
// comes first, so that the largest logit's exponent is 0 at any size and the
// others are off by 2^-24 of themselves: z*c - m*c, though one operation less,
// is off by 2^-24 of m*c, which from 2^31 on (a row, or a thread's part of
// one, that holds only mask values) is more than fp32 has exponents.  It took
// the loss of 512 x 32000 bf16 in 11.4 us, the difference takes 11.9.  Where t is 1 or
// 2, exp(z-m) is exp((z-m)/t) or its square: one transcendental operation per
// logit instead of two, which is what bounds the passes next to HBM.
//
// A row without weight, or without any teacher entry and label, is not read:
// its loss and gradient are 0 whatever it holds.  Entries with an index
// outside the vocabulary are absent; an index given twice counts twice.  Where
// the mix leaves nothing of a term (1: of the label's, 0: of the teacher's), its
// entries count as absent, so that an infinite term does not become NaN.
//
// 4096 x 131072 bf16, loss and gradient: 490 us for 1.07 GB read, read again and
// written (4.4 TB/s for the first and the last).  Rows kept in registers
// between the passes took 861 us: 256 KB leave one workgroup to a CU, with part
// of the row spilled, and nothing on its way while it computes.  The loss of
// 512 x 32000 bf16: 12 us (33 MB in one round of workgroups, most of it start
// and end); of 301 x 50257 fp32: 20 us, and the gradient 24 us (4.9 TB/s).
#include "overlap.hpp"
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

constexpr int DI_MAX_WAVES = 8;
constexpr int DI_MAX_TOP = 1024;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

enum { DI_LOSS, DI_BOTH, DI_GRAD };

struct DistillLds {
    float red[DI_MAX_WAVES][3];
    float soft;                     // 1: the row has a teacher
    int32_t index[DI_MAX_TOP + 1];  // the teacher's entries, then the label; -1: absent
    float p[DI_MAX_TOP + 1];
    float z[DI_MAX_TOP + 1];
};

__device__ __forceinline__ int64_t load_int(const void* p, int32_t bytes, int64_t i) {
    return bytes == 8 ? ((const CRESSO_GLOBAL int64_t*)p)[i] : (int64_t)((const CRESSO_GLOBAL int32_t*)p)[i];
}
__device__ __forceinline__ float load_any(const void* p, int32_t code, int64_t i) {
    if (code == CRESSO_F32) return ((const float*)p)[i];
    if (code == CRESSO_BF16) return to_f(((const __hip_bfloat16*)p)[i]);
    return to_f(((const __half*)p)[i]);
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, kWave));
    return v;
}
// a maximum to subtract: 0 for a row whose every entry is -inf
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

// The exponentials of a row against its maximum.  P: how exp(z-m) comes
// about.  0: it is not wanted; 1, 2: that power of exp((z-m)/t); -1: neither.
template <int P> struct RowExp {
    float c;   // log2(e) / t
    float m;   // finite, or a logit's own infinity
    __device__ __forceinline__ float soft2(float v) const { return (v - m) * c; }
    __device__ __forceinline__ float hard2(float v) const { return P > 0 ? (float)P * soft2(v) : (v - m) * LOG2E; }
    // exp(z-m), given exp((z-m)/t)
    __device__ __forceinline__ float hard(float v, float t) const { return P == 1 ? t : P == 2 ? t * t : fexp2(hard2(v)); }
};
template <int P> __device__ __forceinline__ RowExp<P> row_exp(const cresso_distill_desc& d) { return {LOG2E / d.temperature, 0.0f}; }

// A sum against another maximum; one that holds nothing yet has none.
__device__ __forceinline__ float moved(float sum, float by2) { return sum == 0.0f ? 0.0f : sum * fexp2(by2); }

// A thread's running maximum and sums; x is set to the maximum.
template <int P> struct RowSums {
    float top = -INFINITY, st = 0.0f, s1 = 0.0f;
    template <int E> __device__ __forceinline__ void add(const float (&v)[E], RowExp<P>& x) {
        float um = v[0];
#pragma unroll
        for (int e = 1; e < E; ++e) um = fmaxf(um, v[e]);
        if (um > top) {
            const float before = x.m;
            top = um;
            x.m = um;
            st = moved(st, x.soft2(before));
            if (P) s1 = moved(s1, x.hard2(before));
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float t = fexp2(x.soft2(v[e]));
            st += t;
            if (P) s1 += x.hard(v[e], t);
        }
    }
};
// Joins the threads' sums: x is set to the row's maximum m; l_t, l_1: log2 of
// the sums against it.  One barrier.
template <int P>
__device__ __forceinline__ void join_sums(DistillLds& s, RowSums<P> r, RowExp<P>& x, float& m, float& l_t, float& l_1) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    const float wm = wave_max(r.top);
    const float own = x.m;
    x.m = base_of(wm);
    r.st = wave_sum(moved(r.st, x.soft2(own)));
    r.s1 = P ? wave_sum(moved(r.s1, x.hard2(own))) : 0.0f;
    if (lane == 0) {
        s.red[wave][0] = wm;
        s.red[wave][1] = r.st;
        s.red[wave][2] = r.s1;
    }
    __syncthreads();
    m = s.red[0][0];
#pragma unroll 1
    for (int k = 1; k < waves; ++k) m = fmaxf(m, s.red[k][0]);
    m = base_of(m);
    x.m = m;
    float st = 0.0f, s1 = 0.0f;
#pragma unroll 1
    for (int k = 0; k < waves; ++k) {
        const float of = base_of(s.red[k][0]);
        st += moved(s.red[k][1], x.soft2(of));
        if (P) s1 += moved(s.red[k][2], x.hard2(of));
    }
    l_t = log2f(st);
    l_1 = P ? log2f(s1) : 0.0f;
}

// The row's weight; its teacher's entries and label, and the logits at their
// places, go to LDS.  -> whether the row gives anything.  One barrier.
template <typename T>
__device__ __forceinline__ bool row_begins(const cresso_distill_desc& d, DistillLds& s, const T* z, int64_t row, float& w, int32_t& label) {
    w = d.weights ? d.weights[row] : d.weight;
    bool some = false;
#pragma unroll 1
    for (int j = threadIdx.x; j < d.top; j += blockDim.x) {
        const int64_t v = load_int(d.index, d.index_bytes, row * d.index_stride + j);
        const bool on = v >= 0 && v < d.vocab && d.mix != 0.0f;
        s.index[j] = on ? (int32_t)v : -1;
        s.p[j] = on ? load_any(d.teacher, d.teacher_dtype, row * d.teacher_stride + j) : -INFINITY;
        s.z[j] = on ? to_f(z[v]) : 0.0f;
        some |= on;
    }
    label = -1;
    if (d.labels && d.mix != 1.0f) {
        const int64_t l = load_int(d.labels, d.label_bytes, row);
        if (l != d.ignore_index && l >= 0 && l < d.vocab) label = (int32_t)l;
    }
    if (threadIdx.x == 0) {
        s.index[d.top] = label;
        s.p[d.top] = 0.0f;
        s.z[d.top] = label >= 0 ? to_f(z[label]) : 0.0f;
    }
    some = __syncthreads_or(some);
    return w != 0.0f && (some || label >= 0);
}

// The first wave: the teacher's distribution in its logits' place, and, if
// `loss`, the row's loss.
template <int P>
__device__ __forceinline__ void teacher_of(const cresso_distill_desc& d, DistillLds& s, int64_t row, float w, int32_t label, const RowExp<P>& x,
                                           float l_t, float l_1, bool loss) {
    const int lane = threadIdx.x & (kWave - 1);
    float top = -INFINITY, total = 0.0f, kl = 0.0f;
#pragma unroll 1
    for (int j = lane; j < d.top; j += kWave) {
        top = fmaxf(top, s.p[j]);
    }
    const RowExp<0> a{x.c, base_of(wave_max(top))};
#pragma unroll 1
    for (int j = lane; j < d.top; j += kWave) total += fexp2(a.soft2(s.p[j]));
    total = wave_sum(total);
    const bool any = !(total == 0.0f);   // entries that all are -inf are no teacher
    const float l_total = log2f(total);
#pragma unroll 1
    for (int j = lane; j < d.top; j += kWave) {
        const float a2 = a.soft2(s.p[j]), v = s.z[j];
        const float p = any && s.index[j] >= 0 ? fexp2(a2) / total : 0.0f;
        if (!(p == 0.0f)) kl += p * ((a2 - l_total) - (x.soft2(v) - l_t));
        s.p[j] = p;
    }
    kl = wave_sum(kl);
    if (lane == 0) {
        s.soft = any ? 1.0f : 0.0f;
        const float hard = label >= 0 ? l_1 - x.hard2(s.z[d.top]) : 0.0f;
        if (loss) d.loss[row] = w * LN2 * (d.mix * d.temperature * d.temperature * kl + (1.0f - d.mix) * hard);
    }
}

// The gradient without the teacher's and the label's own terms.
template <int P> struct RowGrad {
    RowExp<P> x;
    float kt, k1;   // factors of exp((z-m)/t) and exp(z-m)
    __device__ __forceinline__ float of(float v) const {
        const float t = fexp2(x.soft2(v));
        return P ? fmaf(k1, x.hard(v, t), kt * t) : kt * t;
    }
};
template <int P>
__device__ __forceinline__ RowGrad<P> row_grad(const cresso_distill_desc& d, const RowExp<P>& x, float g, bool soft, bool hard, float l_t,
                                               float l_1) {
    return {x, soft ? g * d.mix * d.temperature * fexp2(-l_t) : 0.0f, hard ? g * (1.0f - d.mix) * fexp2(-l_1) : 0.0f};
}
// The places of the teacher and the label, after the others are written (a barrier before).
template <typename T, int P>
__device__ __forceinline__ void patch_row(const cresso_distill_desc& d, const DistillLds& s, T* out, const RowGrad<P>& r, float g,
                                          int32_t label) {
    const float kt = g * d.mix * d.temperature, k1 = g * (1.0f - d.mix);
#pragma unroll 1
    for (int j = threadIdx.x; j <= d.top; j += blockDim.x) {
        const int32_t v = s.index[j];
        if (v < 0) continue;
        float p = 0.0f;
        bool first = true;
#pragma unroll 1
        for (int k = 0; k < d.top; ++k)
            if (s.index[k] == v) {
                first &= k >= j;
                p += s.p[k];
            }
        if (!first) continue;
        out[v] = from_w<T>(r.of(s.z[j]) - kt * p - (v == label ? k1 : 0.0f));
    }
}
// The units of a row, NT threads side by side: fn(unit, raw) for each of a
// thread's, with the loads of four of them on their way at a time.  The units
// that all threads have whole lie at addresses of a common base and a 32-bit
// place of the thread's own.  BACK: from the row's end, where a pass before
// has read last and the caches still hold it.
constexpr int DI_AHEAD = 4;
template <typename T, int NT, bool BACK, typename F> __device__ __forceinline__ void for_units(const T* z, int64_t vocab, F&& fn) {
    constexpr int E = Unit<T>::n, PIECE = NT * E;
    const int fours = (int)(vocab / (PIECE * DI_AHEAD)), tid = threadIdx.x;
    const uint32_t place = (uint32_t)tid * E;
    const auto rest = [&] {
        for (int64_t u = (int64_t)fours * DI_AHEAD * NT + tid; u * E < vocab; u += NT) fn(u, load_unit(z, u, vocab));
    };
    if (BACK) rest();
    for (int f = 0; f < fours; ++f) {
        const int i = (BACK ? fours - 1 - f : f) * DI_AHEAD;
        const T* p = z + (int64_t)i * PIECE;
        u32x4 raw[DI_AHEAD];
#pragma unroll
        for (int k = 0; k < DI_AHEAD; ++k) raw[k] = load16(p + k * PIECE + place);
#pragma unroll
        for (int k = 0; k < DI_AHEAD; ++k) fn((int64_t)(i + k) * NT + tid, raw[k]);
    }
    if (!BACK) rest();
}
// a unit's logits; beyond the row's end -inf, which adds nothing
template <typename T> __device__ __forceinline__ void logits_of(u32x4 r, int64_t u, int64_t vocab, float (&v)[Unit<T>::n]) {
    constexpr int E = Unit<T>::n;
    widen<T>(r, v);
    if ((u + 1) * E > vocab) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (u * E + e >= vocab) v[e] = -INFINITY;
    }
}
__device__ __forceinline__ void put_stats(const cresso_distill_desc& d, int64_t row, float m, float l_t, float l_1) {
    if (!d.stats || threadIdx.x) return;
    d.stats[3 * row] = m;
    d.stats[3 * row + 1] = l_t;
    d.stats[3 * row + 2] = l_1;
}

// A workgroup per row: the loss, or the gradient from the loss's maximum and sums.
template <typename T, int MODE, int P, int NT>
__global__ __launch_bounds__(NT) void distill_kernel(cresso_distill_desc d) {
    constexpr int E = Unit<T>::n;
    __shared__ DistillLds s;
    const int64_t row = blockIdx.x, vocab = d.vocab, units = (vocab + E - 1) / E;
    const T* z = (const T*)d.logits + row * d.logits_stride;
    T* out = (T*)d.grad + row * d.grad_stride;
    float w, m, l_t, l_1;
    int32_t label;
    if (!row_begins(d, s, z, row, w, label)) {
        if (MODE != DI_GRAD) {
            if (threadIdx.x == 0) d.loss[row] = 0.0f;
            put_stats(d, row, 0.0f, 0.0f, 0.0f);
        }
        if (MODE != DI_LOSS) {
            for (int64_t u = threadIdx.x; u < units; u += NT) store_unit(out, u, vocab, u32x4{0, 0, 0, 0});
        }
        return;
    }
    RowExp<P> x = row_exp<P>(d);
    if (MODE == DI_GRAD) {
        m = d.stats[3 * row];
        l_t = d.stats[3 * row + 1];
        l_1 = d.stats[3 * row + 2];
        x.m = m;
    } else {
        RowSums<P> sums;
        for_units<T, NT, false>(z, vocab, [&](int64_t u, u32x4 raw) {
            float v[E];
            logits_of<T>(raw, u, vocab, v);
            sums.add(v, x);
        });
        join_sums(s, sums, x, m, l_t, l_1);
        put_stats(d, row, m, l_t, l_1);
    }
    if (threadIdx.x < kWave) teacher_of(d, s, row, w, label, x, l_t, l_1, MODE != DI_GRAD);
    if (MODE == DI_LOSS) return;
    __syncthreads();
    const float g = MODE == DI_GRAD ? w * d.d_loss[d.d_loss_stride * row] : w;
    const RowGrad<P> r = row_grad(d, x, g, s.soft != 0.0f, label >= 0, l_t, l_1);
    for_units<T, NT, MODE == DI_BOTH>(z, vocab, [&](int64_t u, u32x4 raw) {
        float v[E];
        widen<T>(raw, v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = r.of(v[e]);
        store_unit_past(out, u, vocab, narrow<T>(v));
    });
    __syncthreads();
    patch_row(d, s, out, r, g, label);
}

// The sum of the rows' losses, in a fixed order in fp64.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* loss, int64_t rows, float* total) {
    __shared__ double lds[16];
    double v[1] = {0.0};
    for (int64_t i = threadIdx.x; i < rows; i += 1024) v[0] += (double)loss[i];
    block_sum<1>(v, lds);
    if (threadIdx.x == 0) *total = (float)v[0];
}

int32_t check_distill(const char* what, const cresso_distill_desc* d) {
    if (!d) return fail(CRESSO_E_INVALID, "%s: null argument", what);
    if (!row_dtype(d->dtype) || !row_dtype(d->teacher_dtype))
        return fail(CRESSO_E_UNSUPPORTED, "%s: dtypes %d and %d (f32, bf16, f16)", what, d->dtype, d->teacher_dtype);
    if (d->rows < 0 || d->vocab < 1 || d->vocab >= (int64_t)1 << 31 || d->rows >= (int64_t)1 << 23)
        return fail(CRESSO_E_UNSUPPORTED, "%s: %lld rows of %lld logits", what, (long long)d->rows, (long long)d->vocab);
    if (d->top < 0 || d->top > DI_MAX_TOP)
        return fail(CRESSO_E_UNSUPPORTED, "%s: %d entries per row (at most %d)", what, d->top, DI_MAX_TOP);
    if ((d->index_bytes != 4 && d->index_bytes != 8) || (d->labels && d->label_bytes != 4 && d->label_bytes != 8))
        return fail(CRESSO_E_INVALID, "%s: indexes of 4 or 8 bytes are wanted", what);
    if (!(d->temperature > 0.0f) || !(d->mix >= 0.0f && d->mix <= 1.0f))
        return fail(CRESSO_E_INVALID, "%s: temperature must be positive and mix within 0..1", what);
    if (d->rows > 0 && (!d->logits || (d->top > 0 && (!d->index || !d->teacher))))
        return fail(CRESSO_E_INVALID, "%s: null argument", what);
    const struct { const void* p; int64_t width, stride; const char* name; } spans[] = {
        {d->logits, d->vocab, d->logits_stride, "logits"}, {d->index, d->top, d->index_stride, "teacher's indexes"},
        {d->teacher, d->top, d->teacher_stride, "teacher's logits"}, {d->d_loss, 1, d->d_loss_stride, "gradient that arrives"}};
    for (const auto& v : spans)
        if (!row_stride_ok(v.p, d->rows, v.width, v.stride))
            return fail(CRESSO_E_INVALID, "%s: row stride %lld of the %s below the width", what, (long long)v.stride, v.name);
    if (d->grad && d->rows > 1 && d->grad_stride < d->vocab)
        return fail(CRESSO_E_INVALID, "%s: row stride %lld of the gradient below the width", what, (long long)d->grad_stride);
    if (d->grad) {
        const char* with = distill_overlap(*d);
        if (with) return fail(CRESSO_E_INVALID, "%s: the gradient's memory overlaps the %s", what, with);
    }
    return CRESSO_OK;
}

// Calls fn(T, P) for the logits' type and the way to exp(z-m).
template <typename F> void with_exp(const cresso_distill_desc& d, F&& fn) {
    using std::integral_constant;
    with_row_dtype(d.dtype, [&](auto t) {
        if (!d.labels || d.mix == 1.0f) fn(t, integral_constant<int, 0>{});
        else if (d.temperature == 1.0f) fn(t, integral_constant<int, 1>{});
        else if (d.temperature == 2.0f) fn(t, integral_constant<int, 2>{});
        else fn(t, integral_constant<int, -1>{});
    });
}
template <int MODE> void launch_distill(const cresso_distill_desc& d, hipStream_t st) {
    with_exp(d, [&](auto t, auto p) {
        using T = decltype(t);
        constexpr int P = decltype(p)::value;
        const auto go = [&](auto kernel, int threads) {
            hipLaunchKernelGGL(kernel, dim3((uint32_t)d.rows), dim3(threads), 0, st, d);
        };
        const int64_t units = (d.vocab + Unit<T>::n - 1) / Unit<T>::n;
        // Long rows take 512 threads (4096 x 131072 bf16: 494 us, 550 with 256, 569
        // with 1024); where there are rows enough for more workgroups at once,
        // shorter ones fewer (4096 x 32000: 140 us with 256, 147 with 512; 8192 x
        // 1000: 35 us with 64, 46 with 256).  Rows enough are more than two to a CU:
        // loss and gradient of 384, 512, 576, 768 and 1024 rows x 16000 take 18.4, 19.0,
        // 20.7, 21.7 and 24.3 us with 256, 17.8, 18.1, 20.6, 21.5 and 27.7 with 512; of
        // 32000 24.5, 25.9, 28.5, 31.1, 40.7 and 23.2, 24.2, 28.3, 31.1, 44.3; the loss
        // alone of 32000 11.3, 11.8, 13.1, 13.8, 16.5 and 11.3, 11.7, 13.7, 14.5, 19.7.
        if (units <= 256) go(distill_kernel<T, MODE, P, 64>, 64);
        else if (units <= 6144 && d.rows > 512) go(distill_kernel<T, MODE, P, 256>, 256);
        else go(distill_kernel<T, MODE, P, 512>, 512);
    });
}
}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" int32_t cresso_distill_loss(const cresso_distill_desc* desc, void* stream) {
    const int32_t rc = check_distill("distillation loss", desc);
    if (rc != CRESSO_OK) return rc;
    if (!desc->total && desc->rows == 0) return CRESSO_OK;
    if (desc->rows > 0 && (!desc->loss || (desc->grad && !desc->stats))) return fail(CRESSO_E_INVALID, "distillation loss: null argument");
    hipStream_t st = (hipStream_t)stream;
    if (desc->rows > 0) {
        if (desc->grad) launch_distill<DI_BOTH>(*desc, st);
        else launch_distill<DI_LOSS>(*desc, st);
    }
    if (desc->total) hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st, desc->loss, desc->rows, desc->total);
    return launched("distillation loss");
}

extern "C" int32_t cresso_distill_backward(const cresso_distill_desc* desc, void* stream) {
    const int32_t rc = check_distill("distillation gradient", desc);
    if (rc != CRESSO_OK || desc->rows == 0) return rc;
    if (!desc->grad || !desc->stats || !desc->d_loss) return fail(CRESSO_E_INVALID, "distillation gradient: null argument");
    launch_distill<DI_GRAD>(*desc, (hipStream_t)stream);
    return launched("distillation gradient");
}
