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
// loss reads each logit once.  The gradient is written by a second pass over
// the row as if there were no teacher and no label; their few places are
// written again afterwards from logits that were read before, so it may take
// the logits' own memory.  Bound by HBM and, where both exponentials of each
// logit are needed in both passes, by the transcendental rate.
//
// A row without weight, or without any teacher entry and label, is not read:
// its loss and gradient are 0 whatever it holds.  Entries with an index
// outside the vocabulary are absent; an index given twice counts twice.
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

constexpr int DI_NT = 512;
constexpr int DI_WAVES = DI_NT / kWave;
constexpr int DI_MAX_TOP = 1024;
constexpr float LOG2E = 1.4426950408889634f;

enum { DI_LOSS, DI_BOTH, DI_GRAD };

struct DistillLds {
    float red[DI_WAVES][3];
    float row[8];                   // m, log sums, has teacher
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

template <typename T, int MODE>
__global__ __launch_bounds__(DI_NT) void distill_kernel(cresso_distill_desc d) {
    constexpr int E = Unit<T>::n;
    __shared__ DistillLds s;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int64_t row = blockIdx.x, vocab = d.vocab, units = (vocab + E - 1) / E;
    const T* z = (const T*)d.logits + row * d.logits_stride;
    T* out = (T*)d.grad + row * d.grad_stride;
    const float w = d.weights ? d.weights[row] : d.weight;
    const bool two = d.labels != nullptr;   // the batch has labels: both sums are kept

    // the teacher's entries and the label
    bool some = false;
    for (int j = tid; j < d.top; j += DI_NT) {
        const int64_t v = load_int(d.index, d.index_bytes, row * d.index_stride + j);
        const bool on = v >= 0 && v < vocab;
        s.index[j] = on ? (int32_t)v : -1;
        some |= on;
    }
    int64_t label = -1;
    if (two) {
        label = load_int(d.labels, d.label_bytes, row);
        if (label == d.ignore_index || label < 0 || label >= vocab) label = -1;
    }
    if (tid == 0) s.index[d.top] = (int32_t)label;
    const bool teacher = __syncthreads_or(some);
    if (w == 0.0f || (!teacher && label < 0)) {
        if (MODE != DI_GRAD && tid == 0) {
            d.loss[row] = 0.0f;
            if (d.stats) d.stats[3 * row] = d.stats[3 * row + 1] = d.stats[3 * row + 2] = 0.0f;
        }
        if (MODE != DI_LOSS)
            for (int64_t u = tid; u < units; u += DI_NT) store_unit(out, u, vocab, u32x4{0, 0, 0, 0});
        return;
    }
    const float ct = LOG2E / d.temperature;

    float m, log_t, log_1;   // maximum; log of the sums of exp((z-m)/t) and exp(z-m)
    if (MODE == DI_GRAD) {
        m = d.stats[3 * row];
        log_t = d.stats[3 * row + 1];
        log_1 = d.stats[3 * row + 2];
    } else {
        float top = -INFINITY, st = 0.0f, s1 = 0.0f;
        for (int64_t u = tid; u < units; u += DI_NT) {
            float v[E];
            widen<T>(load_unit(z, u, vocab), v);
            if (u == units - 1) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (u * E + e >= vocab) v[e] = -INFINITY;
            }
            float um = v[0];
#pragma unroll
            for (int e = 1; e < E; ++e) um = fmaxf(um, v[e]);
            if (um > top) {
                st *= fexp2((top - um) * ct);
                s1 *= fexp2((top - um) * LOG2E);
                top = um;
            }
            const float b = base_of(top);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                st += fexp2((v[e] - b) * ct);
                if (two) s1 += fexp2((v[e] - b) * LOG2E);
            }
        }
        const float wm = wave_max(top), wb = base_of(wm);
        st = wave_sum(st * fexp2((top - wb) * ct));
        s1 = wave_sum(s1 * fexp2((top - wb) * LOG2E));
        if (lane == 0) {
            s.red[wave][0] = wm;
            s.red[wave][1] = st;
            s.red[wave][2] = s1;
        }
        __syncthreads();
        m = s.red[0][0];
        for (int k = 1; k < DI_WAVES; ++k) m = fmaxf(m, s.red[k][0]);
        m = base_of(m);
        st = s1 = 0.0f;
        for (int k = 0; k < DI_WAVES; ++k) {
            st += s.red[k][1] * fexp2((s.red[k][0] - m) * ct);
            s1 += s.red[k][2] * fexp2((s.red[k][0] - m) * LOG2E);
        }
        log_t = logf(st);
        log_1 = two ? logf(s1) : 0.0f;
    }

    if (wave == 0) {   // the teacher's distribution; the loss
        float a_top = -INFINITY, total = 0.0f, kl = 0.0f;
        for (int j = lane; j < d.top; j += kWave) {
            const float a = s.index[j] >= 0 ? load_any(d.teacher, d.teacher_dtype, row * d.teacher_stride + j) : -INFINITY;
            s.p[j] = a;
            a_top = fmaxf(a_top, a);
        }
        a_top = base_of(wave_max(a_top));
        for (int j = lane; j < d.top; j += kWave) total += fexp2((s.p[j] - a_top) * ct);
        total = wave_sum(total);
        // entries that all are -inf: no teacher
        const bool any = !(total == 0.0f);
        const float log_total = logf(total);
        for (int j = lane; j < d.top; j += kWave) {
            const float a = s.p[j];
            const float p = any && s.index[j] >= 0 ? fexp2((a - a_top) * ct) / total : 0.0f;
            const float v = s.index[j] >= 0 ? to_f(z[s.index[j]]) : 0.0f;
            if (!(p == 0.0f)) kl += p * (((a - a_top) - (v - m)) / d.temperature - log_total + log_t);
            s.p[j] = p;
            s.z[j] = v;
        }
        kl = wave_sum(kl);
        if (lane == 0) {
            float hard = 0.0f;
            s.p[d.top] = 0.0f;
            if (label >= 0) {
                const float v = to_f(z[label]);
                s.z[d.top] = v;
                hard = log_1 - (v - m);
            }
            s.row[0] = any ? 1.0f : 0.0f;
            if (MODE != DI_GRAD) {
                d.loss[row] = w * (d.mix * d.temperature * d.temperature * kl + (1.0f - d.mix) * hard);
                if (d.stats) {
                    d.stats[3 * row] = m;
                    d.stats[3 * row + 1] = log_t;
                    d.stats[3 * row + 2] = log_1;
                }
            }
        }
    }
    if (MODE == DI_LOSS) return;
    __syncthreads();
    const float g = MODE == DI_GRAD ? w * d.d_loss[d.d_loss_stride * row] : w;
    const bool soft = s.row[0] != 0.0f, hard = label >= 0;
    const float kt = g * d.mix * d.temperature, k1 = g * (1.0f - d.mix);
    const float bt = log_t * LOG2E, b1 = log_1 * LOG2E;
    const auto grad_of = [&](float v) {
        float r = 0.0f;
        if (soft) r = kt * fexp2((v - m) * ct - bt);
        if (hard) r += k1 * fexp2((v - m) * LOG2E - b1);
        return r;
    };
    for (int64_t u = tid; u < units; u += DI_NT) {
        float v[E];
        widen<T>(load_unit(z, u, vocab), v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = grad_of(v[e]);
        store_unit(out, u, vocab, narrow<T>(v));
    }
    __syncthreads();   // the places below were written above
    for (int j = tid; j <= d.top; j += DI_NT) {
        const int32_t v = s.index[j];
        if (v < 0) continue;
        float p = 0.0f;
        bool first = true;
        for (int k = 0; k < d.top; ++k)
            if (s.index[k] == v) {
                first &= k >= j;
                p += s.p[k];
            }
        if (first) out[v] = from_w<T>(grad_of(s.z[j]) - kt * p - (v == label ? k1 : 0.0f));
    }
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
    return CRESSO_OK;
}

template <int MODE> void launch_distill(const cresso_distill_desc& d, hipStream_t st) {
    with_row_dtype(d.dtype, [&](auto t) {
        hipLaunchKernelGGL((distill_kernel<decltype(t), MODE>), dim3((uint32_t)d.rows), dim3(DI_NT), 0, st, d);
    });
}

}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" int32_t cresso_distill_loss(const cresso_distill_desc* desc, void* stream) {
    const int32_t rc = check_distill("distillation loss", desc);
    if (rc != CRESSO_OK) return rc;
    if (!desc->total && desc->rows == 0) return CRESSO_OK;
    if (desc->rows > 0 && !desc->loss) return fail(CRESSO_E_INVALID, "distillation loss: null argument");
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
