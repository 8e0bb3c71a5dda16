// The seam between two blocks of a network, in one pass over its rows:
//
//   yn = y * ry,  ry = 1/sqrt(mean(y^2) + eps)         norm after the block (with gain w1)
//   H  = s*h + a*(yn*w1),  a = act(g)                  gate and scaled residual
//   Hn = H * rh,  rh = 1/sqrt(mean(H^2) + eps)
//   n  = Hn * w2                                       norm before the next block
//
// and its gradient from dH (what arrives at H directly) and dn:
//
//   e = dn*w2,   d = dH + rh*(e - Hn*mean(e*Hn))       everything that arrives at H
//   dh = s*d,    ds = sum d*h,   dw2 = sum dn*Hn
//   dw1 = sum d*a*yn,   dg = act'(g) * sum d*yn*w1
//   dy = ry*(d*a*w1 - yn*mean(d*a*w1*yn))
//
// d is linear in mean(e*Hn), so with t = dH + rh*e and q = a*w1*yn
//   mean(d*q) = mean(t*q) - rh*mean(e*Hn)*mean(Hn*q)
// and one round of three sums per row serves both norms.  Where nothing arrives
// at n, or there is no norm after the block, its terms are left out: a factor
// of 0 would make an infinite element the whole row's NaN.
//
// Both directions are bound by HBM: 4 rows of traffic forward (h, y in; H, n
// out), 6 backward (h, y, dH, dn in; dh, dy out).  A row stays in registers
// from its load to its store; the gradients of what is shared by rows are kept
// in registers over a worker's rows, written once per worker as fp32 and added
// by a second kernel in worker order.  All sums are fp32.
//
// 16384 x 4096 bf16, a gate and a scale per channel: forward 99 us (537 MB, 5.4
// TB/s), gradient 170 us (805 MB, 4.7 TB/s) and 5.2 us for the sums of 256
// workers.  8 x 2048 bf16 forward: 4.4 us, latency of the loads and of two
// sums over four waves.  1533 x 1001 fp32: 8.6, 13.7 and 5.4 us.
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

constexpr int RN_MIN_NT = 256;
constexpr int RN_SUM_NT = 1024;
constexpr int RN_MAX_WIDTH = 16384;
constexpr int RN_WIDE = 4096;       // above, the gradient holds no row in registers
constexpr int RN_FWD_BLOCKS = 2048;

struct SeamArgs {
    cresso_residual_norm_desc d;
    int64_t workers, worker_rows, workers_per_gate, gates_per_worker;   // gradient
    float* partial;                                                      // [4][workers][padded width]
    int64_t padded;
};

__device__ __forceinline__ float act_of(int32_t act, float g) {
    if (act == CRESSO_GATE_SIGMOID) return 1.0f / (1.0f + expf(-g));
    if (act == CRESSO_GATE_TANH) return tanhf(g);
    return g;
}
// act'(g) from act(g)
__device__ __forceinline__ float act_slope(int32_t act, float a) {
    if (act == CRESSO_GATE_SIGMOID) return a * (1.0f - a);
    if (act == CRESSO_GATE_TANH) return (1.0f - a) * (1.0f + a);
    return 1.0f;
}

// Unit u of a vector of either the rows' type or fp32.
template <typename T>
__device__ __forceinline__ void load_vec(const void* p, int32_t code, int64_t u, int64_t width, float (&v)[Unit<T>::n]) {
    if constexpr (sizeof(T) == 4) {
        widen<T>(load_unit((const T*)p, u, width), v);
    } else {
        if (code == CRESSO_F32) {
            float lo[4], hi[4];
            widen<float>(load_unit((const float*)p, 2 * u, width), lo);
            widen<float>(load_unit((const float*)p, 2 * u + 1, width), hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = lo[i];
                v[4 + i] = hi[i];
            }
        } else {
            widen<T>(load_unit((const T*)p, u, width), v);
        }
    }
}
template <typename T>
__device__ __forceinline__ void store_vec(void* p, int32_t code, int64_t u, int64_t width, const float (&v)[Unit<T>::n]) {
    if constexpr (sizeof(T) == 4) {
        store_unit((T*)p, u, width, narrow<T>(v));
    } else {
        if (code == CRESSO_F32) {
            const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
            store_unit((float*)p, 2 * u, width, narrow<float>(lo));
            store_unit((float*)p, 2 * u + 1, width, narrow<float>(hi));
        } else {
            store_unit((T*)p, u, width, narrow<T>(v));
        }
    }
}
template <typename T> __device__ __forceinline__ int64_t vec_bytes(int32_t code) {
    return sizeof(T) == 4 || code == CRESSO_F32 ? 4 : 2;
}
__device__ __forceinline__ const char* gate_row(const cresso_residual_norm_desc& d, int64_t row, int64_t bytes) {
    return (const char*)d.gate + row / d.rows_per_gate * d.gate_stride * bytes;
}

// Sums of V values over the WPR waves of a row; every thread gets them.
// `turn` alternates between two areas, so one barrier a call is enough.
template <int WPR, int V>
__device__ __forceinline__ void row_sum(float (&x)[V], float* lds, int turn) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = wave_total(x[i]);
    if constexpr (WPR == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x[i]), 63));
    } else {
        const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, slot = wave / WPR;
        float* at = lds + (turn & 1) * (16 * V);
        if (lane == kWave - 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) at[wave * V + i] = x[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) s += at[(slot * WPR + w) * V + i];
            x[i] = s;
        }
    }
}

// waves per row WPR, units per thread NU: a unit a thread as long as a workgroup
// has room, so that a row's loads are one instruction a wave and its sums few
// steps.  What all rows share is read once and kept in registers.
template <typename T, int WPR, int NU>
__global__ __launch_bounds__(WPR * 64 < RN_MIN_NT ? RN_MIN_NT : WPR * 64) void seam_forward_kernel(SeamArgs a) {
    constexpr int E = Unit<T>::n, NT = WPR * 64 < RN_MIN_NT ? RN_MIN_NT : WPR * 64, SLOTS = NT / (WPR * 64);
    __shared__ float lds[2 * 16];
    const cresso_residual_norm_desc& d = a.d;
    const int slot = threadIdx.x / (WPR * 64), tid = threadIdx.x % (WPR * 64);
    const int64_t width = d.width;
    const float inv = 1.0f / (float)width;
    float w1[NU][E], w2[NU][E], sc[NU][E], ga[NU][E];
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int64_t u = tid + i * (WPR * 64);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w1[i][e] = w2[i][e] = ga[i][e] = 1.0f;
            sc[i][e] = d.scale;
        }
        if (d.post) load_vec<T>(d.post, d.post_dtype, u, width, w1[i]);
        if (d.pre) load_vec<T>(d.pre, d.pre_dtype, u, width, w2[i]);
        if (d.scale_vec) load_vec<T>(d.scale_vec, d.scale_dtype, u, width, sc[i]);
        if (d.gate && d.rows_per_gate == d.rows) {
            load_vec<T>(d.gate, d.gate_dtype, u, width, ga[i]);
#pragma unroll
            for (int e = 0; e < E; ++e) ga[i][e] = act_of(d.act, ga[i][e]);
        }
    }
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * SLOTS; r0 < d.rows; r0 += (int64_t)gridDim.x * SLOTS) {
        const int64_t row = r0 + slot;
        const bool on = row < d.rows;
        u32x4 hr[NU], yr[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int64_t u = tid + i * (WPR * 64);
            hr[i] = yr[i] = u32x4{0, 0, 0, 0};
            if (on) {
                hr[i] = load_unit((const T*)d.residual + row * d.residual_stride, u, width);
                if (d.update) yr[i] = load_unit((const T*)d.update + row * d.update_stride, u, width);
            }
        }
        if (d.gate && d.rows_per_gate != d.rows && on) {
            const char* g = gate_row(d, row, vec_bytes<T>(d.gate_dtype));
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                load_vec<T>(g, d.gate_dtype, tid + i * (WPR * 64), width, ga[i]);
#pragma unroll
                for (int e = 0; e < E; ++e) ga[i][e] = act_of(d.act, ga[i][e]);
            }
        }
        float ry = 1.0f, rh = 0.0f;
        if (d.update && d.post) {
            float ss[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float y[E];
                widen<T>(yr[i], y);
#pragma unroll
                for (int e = 0; e < E; ++e) ss[0] += y[e] * y[e];
            }
            row_sum<WPR>(ss, lds, turn++);
            ry = rsqrtf(ss[0] * inv + d.eps);
        }
        float H[NU][E], ss[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            float h[E], y[E];
            widen<T>(hr[i], h);
            widen<T>(yr[i], y);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                H[i][e] = sc[i][e] * h[e];
                if (d.update) H[i][e] += ga[i][e] * (y[e] * ry * w1[i][e]);
                ss[0] += H[i][e] * H[i][e];   // beyond the row's end H is 0
            }
        }
        if (d.pre) {
            row_sum<WPR>(ss, lds, turn++);
            rh = rsqrtf(ss[0] * inv + d.eps);
        }
        if (on) {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int64_t u = tid + i * (WPR * 64);
                if (d.out) store_unit((T*)d.out + row * width, u, width, narrow<T>(H[i]));
                if (d.pre) {
#pragma unroll
                    for (int e = 0; e < E; ++e) H[i][e] *= rh * w2[i][e];
                    store_unit((T*)d.normed + row * width, u, width, narrow<T>(H[i]));
                }
            }
            if (d.stats && tid == 0) {
                d.stats[2 * row] = ry;
                d.stats[2 * row + 1] = rh;
            }
        }
    }
}

// which of the four shared gradients, in `partial` and in the reduction
enum { G_POST, G_PRE, G_SCALE, G_GATE };

// FULL: something arrives at n, and there is a norm after the block.  The other
// forms ask for either on the way (in one kernel for all of them 16384 x 2048
// fp32 takes 183 us, 176 as it is).
template <typename T, int WPR, int NU, bool FULL>
__global__ __launch_bounds__(WPR * 64 < RN_MIN_NT ? RN_MIN_NT : WPR * 64) void seam_backward_kernel(SeamArgs a) {
    constexpr int E = Unit<T>::n, NT = WPR * 64 < RN_MIN_NT ? RN_MIN_NT : WPR * 64, SLOTS = NT / (WPR * 64);
    __shared__ float lds[2 * 16 * 3];
    const cresso_residual_norm_desc& d = a.d;
    const int slot = threadIdx.x / (WPR * 64), tid = threadIdx.x % (WPR * 64);
    const int64_t width = d.width, worker = (int64_t)blockIdx.x * SLOTS + slot;
    const float inv = 1.0f / (float)width;
    const bool normed = FULL || d.d_normed, post = FULL || d.post;
    // the worker's rows: whole gates' rows, or a part of one gate's
    int64_t first, last;
    if (a.workers_per_gate == 1) {
        first = worker * a.worker_rows;
        last = min(d.rows, first + a.worker_rows);
    } else {
        const int64_t g = worker / a.workers_per_gate, j = worker - g * a.workers_per_gate;
        first = g * d.rows_per_gate + j * a.worker_rows;
        last = min((g + 1) * d.rows_per_gate, first + a.worker_rows);
    }
    if (worker >= a.workers) first = last = 0;
    float w1[NU][E], w2[NU][E], sc[NU][E], ga[NU][E];
    float d1[NU][E] = {}, d2[NU][E] = {}, ds[NU][E] = {}, dg[NU][E] = {};
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int64_t u = tid + i * (WPR * 64);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w1[i][e] = w2[i][e] = ga[i][e] = 1.0f;
            sc[i][e] = d.scale;
        }
        if (d.post) load_vec<T>(d.post, d.post_dtype, u, width, w1[i]);
        if (d.pre) load_vec<T>(d.pre, d.pre_dtype, u, width, w2[i]);
        if (d.scale_vec) load_vec<T>(d.scale_vec, d.scale_dtype, u, width, sc[i]);
    }
    int64_t gate = -1;
    int turn = 0;
    u32x4 hr[NU], yr[NU], ar[NU], nr[NU];   // the row, and the next one's on their way
    u32x4 hn[NU], yn_[NU], an[NU], nn[NU];
    float ry = 1.0f, rh = 0.0f, ry_n = 1.0f, rh_n = 0.0f;
    const auto fetch = [&](int64_t row) {
        const bool on = row < last;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int64_t u = tid + i * (WPR * 64);
            hn[i] = yn_[i] = an[i] = nn[i] = u32x4{0, 0, 0, 0};
            if (on) {
                hn[i] = load_unit((const T*)d.residual + row * d.residual_stride, u, width);
                if (d.update) yn_[i] = load_unit((const T*)d.update + row * d.update_stride, u, width);
                if (d.d_out) an[i] = load_unit((const T*)d.d_out + row * d.d_out_stride, u, width);
                if (d.d_normed) nn[i] = load_unit((const T*)d.d_normed + row * d.d_normed_stride, u, width);
            }
        }
        if (on && d.post) ry_n = d.stats[2 * row];
        if (on && d.d_normed) rh_n = d.stats[2 * row + 1];
    };
    fetch(first);
    for (int64_t k = 0; k < a.worker_rows; ++k) {   // the same count for every slot: the row sums hold a barrier
        const int64_t row = first + k;
        const bool on = row < last;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            hr[i] = hn[i];
            yr[i] = yn_[i];
            ar[i] = an[i];
            nr[i] = nn[i];
        }
        ry = ry_n;
        rh = rh_n;
        fetch(row + 1);
        if (on && d.gate && row / d.rows_per_gate != gate) {
            gate = row / d.rows_per_gate;
            const char* g = gate_row(d, row, vec_bytes<T>(d.gate_dtype));
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                load_vec<T>(g, d.gate_dtype, tid + i * (WPR * 64), width, ga[i]);
#pragma unroll
                for (int e = 0; e < E; ++e) ga[i][e] = act_of(d.act, ga[i][e]);
            }
        }
        float ss[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            float h[E], y[E], t[E], dn[E];
            widen<T>(hr[i], h);
            widen<T>(yr[i], y);
            widen<T>(ar[i], t);
            widen<T>(nr[i], dn);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float q = d.update ? ga[i][e] * w1[i][e] * (y[e] * ry) : 0.0f;
                if (normed) {
                    const float Hn = (sc[i][e] * h[e] + q) * rh, en = dn[e] * w2[i][e];
                    ss[0] += en * Hn;
                    ss[1] += q * (t[e] + rh * en);
                    ss[2] += q * Hn;
                } else {
                    ss[1] += q * t[e];
                }
            }
        }
        row_sum<WPR>(ss, lds, turn++);
        const float c1 = rh * ss[0] * inv;            // rh * mean(e*Hn)
        const float c2 = (normed ? ss[1] - c1 * ss[2] : ss[1]) * inv;   // mean(d*q)
        if (on) {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int64_t u = tid + i * (WPR * 64);
                float h[E], y[E], t[E], dn[E], dh[E], dy[E];
                widen<T>(hr[i], h);
                widen<T>(yr[i], y);
                widen<T>(ar[i], t);
                widen<T>(nr[i], dn);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float yn = d.update ? y[e] * ry : 0.0f;
                    float D = t[e];
                    if (normed) {
                        const float Hn = (sc[i][e] * h[e] + ga[i][e] * w1[i][e] * yn) * rh;
                        D = t[e] + rh * (dn[e] * w2[i][e]) - Hn * c1;
                        d2[i][e] += dn[e] * Hn;
                    }
                    dh[e] = sc[i][e] * D;
                    ds[i][e] += D * h[e];
                    const float da = D * ga[i][e];
                    d1[i][e] += da * yn;
                    dg[i][e] += D * (yn * w1[i][e]);
                    dy[e] = da * w1[i][e];
                    if (post) dy[e] = ry * (dy[e] - yn * c2);
                }
                if (d.d_residual) store_unit((T*)d.d_residual + row * width, u, width, narrow<T>(dh));
                if (d.d_update) store_unit((T*)d.d_update + row * width, u, width, narrow<T>(dy));
            }
            // the last of a gate's rows, all of them this worker's: its gradient is complete
            if (d.d_gate && a.workers_per_gate == 1 && (row + 1) % d.rows_per_gate == 0) {
                char* to = (char*)d.d_gate + gate * width * vec_bytes<T>(d.gate_dtype);
#pragma unroll
                for (int i = 0; i < NU; ++i) {
#pragma unroll
                    for (int e = 0; e < E; ++e) dg[i][e] *= act_slope(d.act, ga[i][e]);
                    store_vec<T>(to, d.gate_dtype, tid + i * (WPR * 64), width, dg[i]);
#pragma unroll
                    for (int e = 0; e < E; ++e) dg[i][e] = 0.0f;
                }
            }
        }
    }
    if (worker >= a.workers) return;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int64_t u = tid + i * (WPR * 64);
        const auto put = [&](int which, const float (&v)[E]) {
            float* to = a.partial + ((int64_t)which * a.workers + worker) * a.padded;
            store_vec<T>(to, CRESSO_F32, u, width, v);
        };
        if (d.d_post) put(G_POST, d1[i]);
        if (d.d_pre) put(G_PRE, d2[i]);
        if (d.d_scale) put(G_SCALE, ds[i]);
        if (d.d_gate && a.workers_per_gate > 1) put(G_GATE, dg[i]);
    }
}

// The same for rows of more than 4096 elements (512 threads, NU units each),
// whose registers would not hold a row, its parameters and the shared sums: only
// the sums stay in registers.  A row is read twice, the second time from L2, and
// its parameters with it: 8192 x 8192 bf16 346 us with the sums, 1361 as
// above with the row's registers spilled.  (Above 8192 elements the sums alone pass what is
// left beside a unit's numbers, and some of them lie in scratch memory.)
template <typename T, int NU, bool FULL>
__global__ __launch_bounds__(512) void seam_backward_wide_kernel(SeamArgs a) {
    constexpr int E = Unit<T>::n, WPR = 8, NT = 512;
    __shared__ float lds[2 * 16 * 3];
    const cresso_residual_norm_desc& d = a.d;
    const int tid = threadIdx.x;
    const int64_t width = d.width, worker = blockIdx.x;
    const float inv = 1.0f / (float)width;
    const bool normed = FULL || d.d_normed, post = FULL || d.post;
    int64_t first, last;
    if (a.workers_per_gate == 1) {
        first = worker * a.worker_rows;
        last = min(d.rows, first + a.worker_rows);
    } else {
        const int64_t g = worker / a.workers_per_gate, j = worker - g * a.workers_per_gate;
        first = g * d.rows_per_gate + j * a.worker_rows;
        last = min((g + 1) * d.rows_per_gate, first + a.worker_rows);
    }
    float d1[NU][E] = {}, d2[NU][E] = {}, ds[NU][E] = {}, dg[NU][E] = {};
    struct Part {
        float h[E], y[E], t[E], dn[E], w1[E], w2[E], sc[E], ga[E];
    };
    const auto load = [&](int64_t row, int64_t u) {
        Part p;
        u32x4 r[4] = {};
        r[0] = load_unit((const T*)d.residual + row * d.residual_stride, u, width);
        if (d.update) r[1] = load_unit((const T*)d.update + row * d.update_stride, u, width);
        if (d.d_out) r[2] = load_unit((const T*)d.d_out + row * d.d_out_stride, u, width);
        if (d.d_normed) r[3] = load_unit((const T*)d.d_normed + row * d.d_normed_stride, u, width);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            p.w1[e] = p.w2[e] = p.ga[e] = 1.0f;
            p.sc[e] = d.scale;
        }
        if (d.post) load_vec<T>(d.post, d.post_dtype, u, width, p.w1);
        if (d.pre) load_vec<T>(d.pre, d.pre_dtype, u, width, p.w2);
        if (d.scale_vec) load_vec<T>(d.scale_vec, d.scale_dtype, u, width, p.sc);
        if (d.gate) {
            load_vec<T>(gate_row(d, row, vec_bytes<T>(d.gate_dtype)), d.gate_dtype, u, width, p.ga);
#pragma unroll
            for (int e = 0; e < E; ++e) p.ga[e] = act_of(d.act, p.ga[e]);
        }
        widen<T>(r[0], p.h);
        widen<T>(r[1], p.y);
        widen<T>(r[2], p.t);
        widen<T>(r[3], p.dn);
        return p;
    };
    int turn = 0;
    for (int64_t row = first; row < last; ++row) {
        const float ry = d.post ? d.stats[2 * row] : 1.0f, rh = d.d_normed ? d.stats[2 * row + 1] : 0.0f;
        float ss[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (int i = 0; i < NU; ++i) {
            const Part p = load(row, tid + i * NT);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float q = d.update ? p.ga[e] * p.w1[e] * (p.y[e] * ry) : 0.0f;
                if (normed) {
                    const float Hn = (p.sc[e] * p.h[e] + q) * rh, en = p.dn[e] * p.w2[e];
                    ss[0] += en * Hn;
                    ss[1] += q * (p.t[e] + rh * en);
                    ss[2] += q * Hn;
                } else {
                    ss[1] += q * p.t[e];
                }
            }
        }
        row_sum<WPR>(ss, lds, turn++);
        const float c1 = rh * ss[0] * inv;
        const float c2 = (normed ? ss[1] - c1 * ss[2] : ss[1]) * inv;
        const bool gate_ends = d.d_gate && a.workers_per_gate == 1 && (row + 1) % d.rows_per_gate == 0;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int64_t u = tid + i * NT;
            const Part p = load(row, u);
            float dh[E], dy[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float yn = d.update ? p.y[e] * ry : 0.0f;
                float D = p.t[e];
                if (normed) {
                    const float Hn = (p.sc[e] * p.h[e] + p.ga[e] * p.w1[e] * yn) * rh;
                    D = p.t[e] + rh * (p.dn[e] * p.w2[e]) - Hn * c1;
                    d2[i][e] += p.dn[e] * Hn;
                }
                dh[e] = p.sc[e] * D;
                ds[i][e] += D * p.h[e];
                const float da = D * p.ga[e];
                d1[i][e] += da * yn;
                dg[i][e] += D * (yn * p.w1[e]);
                dy[e] = da * p.w1[e];
                if (post) dy[e] = ry * (dy[e] - yn * c2);
            }
            if (d.d_residual) store_unit((T*)d.d_residual + row * width, u, width, narrow<T>(dh));
            if (d.d_update) store_unit((T*)d.d_update + row * width, u, width, narrow<T>(dy));
            if (gate_ends) {
#pragma unroll
                for (int e = 0; e < E; ++e) dg[i][e] *= act_slope(d.act, p.ga[e]);
                store_vec<T>((char*)d.d_gate + row / d.rows_per_gate * width * vec_bytes<T>(d.gate_dtype), d.gate_dtype, u, width, dg[i]);
#pragma unroll
                for (int e = 0; e < E; ++e) dg[i][e] = 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);   // one unit's numbers at a time
        }
    }
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const int64_t u = tid + i * NT;
        const auto put = [&](int which, const float (&v)[E]) {
            store_vec<T>(a.partial + ((int64_t)which * a.workers + worker) * a.padded, CRESSO_F32, u, width, v);
        };
        if (d.d_post) put(G_POST, d1[i]);
        if (d.d_pre) put(G_PRE, d2[i]);
        if (d.d_scale) put(G_SCALE, ds[i]);
        if (d.d_gate && a.workers_per_gate > 1) put(G_GATE, dg[i]);
    }
}

// Adds the workers' partial sums, 64 columns and one vector a block: the
// waves take equal runs of workers in order and their sums are added in order.
// Latency of a run's loads bounds it, so there are as many waves as a block
// has (512 workers x 1001: 5.4 us, with four waves 8.9).
template <typename T>
__global__ __launch_bounds__(RN_SUM_NT) void seam_reduce_kernel(SeamArgs a) {
    constexpr int W = RN_SUM_NT / kWave;
    __shared__ float part[W][kWave];
    const cresso_residual_norm_desc& d = a.d;
    const int which = blockIdx.y < 3 ? (int)blockIdx.y : (int)G_GATE;
    void* to = which == G_POST ? d.d_post : which == G_PRE ? d.d_pre : which == G_SCALE ? d.d_scale : d.d_gate;
    if (!to) return;
    const int32_t code = which == G_POST ? d.post_dtype : which == G_PRE ? d.pre_dtype : which == G_SCALE ? d.scale_dtype : d.gate_dtype;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t col = (int64_t)blockIdx.x * kWave + lane;
    const int64_t n = which == G_GATE ? a.workers_per_gate : a.workers, w0 = which == G_GATE ? (blockIdx.y - 3) * n : 0;
    const int64_t share = (n + W - 1) / W, k0 = min(n, wave * share), k1 = min(n, k0 + share);
    const float* p = a.partial + ((int64_t)which * a.workers + w0) * a.padded + col;
    float s = 0.0f;
    if (col < d.width) {
#pragma unroll 8
        for (int64_t k = k0; k < k1; ++k) s += p[k * a.padded];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= d.width) return;
    for (int w = 1; w < W; ++w) s += part[w][lane];
    int64_t at = col;
    if (which == G_GATE) {
        const int64_t g = blockIdx.y - 3;
        at += g * d.width;
        const int64_t from = g * d.gate_stride + col;
        const float v = sizeof(T) == 4 || d.gate_dtype == CRESSO_F32 ? ((const float*)d.gate)[from] : to_f(((const T*)d.gate)[from]);
        s *= act_slope(d.act, act_of(d.act, v));
    }
    if (sizeof(T) == 4 || code == CRESSO_F32) ((float*)to)[at] = s;
    else ((T*)to)[at] = from_w<T>(s);
}

// Calls fn<T, WPR, NU> for the row type and the units of a row.
template <typename F> void with_shape(int32_t dtype, int64_t width, F&& fn) {
    with_row_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t units = (width + Unit<T>::n - 1) / Unit<T>::n;
        const auto go = [&](auto wpr, auto nu) { fn(t, wpr, nu); };
        using std::integral_constant;
        if (units <= 64) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
        else if (units <= 128) go(integral_constant<int, 2>{}, integral_constant<int, 1>{});
        else if (units <= 256) go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
        else if (units <= 512) go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
        else if (units <= 1024) go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
        else if (units <= 2048) go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
        else if constexpr (sizeof(T) == 4) go(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    });
}
int slots_of(int wpr) { return wpr * 64 < RN_MIN_NT ? RN_MIN_NT / (wpr * 64) : 1; }

// Workers of the gradient, each with whole gates' rows or a part of one gate's.
// As many as are resident at once (8 waves to a CU, by the registers of a row,
// its gradients and what is summed): more would only write more partial sums
// (16384 x 4096 bf16: 175 us with the sums; 206 with more workers and without the
// next row's loads ahead).
SeamArgs plan_of(const cresso_residual_norm_desc& d) {
    SeamArgs a{};
    a.d = d;
    a.padded = (d.width + 63) / 64 * 64;
    const int64_t rpg = d.gate ? d.rows_per_gate : d.rows, gates = d.rows / rpg;
    int64_t resident = 256;
    if (d.width <= RN_WIDE) with_shape(d.dtype, d.width, [&](auto, auto wpr, auto) { resident = 256 * std::max(1, 8 / (int)decltype(wpr)::value); });
    const int64_t want = std::max<int64_t>(1, (d.rows + resident - 1) / resident);
    if (rpg > want) {
        a.worker_rows = want;
        a.workers_per_gate = (rpg + want - 1) / want;
        a.gates_per_worker = 1;
        a.workers = gates * a.workers_per_gate;
    } else {
        a.workers_per_gate = 1;
        a.gates_per_worker = want / rpg;
        a.worker_rows = a.gates_per_worker * rpg;
        a.workers = (gates + a.gates_per_worker - 1) / a.gates_per_worker;
    }
    return a;
}

int32_t check_seam(const char* what, const cresso_residual_norm_desc* d) {
    if (!d) return fail(CRESSO_E_INVALID, "%s: null argument", what);
    if (!row_dtype(d->dtype)) return fail(CRESSO_E_UNSUPPORTED, "%s: dtype %d not supported (f32, bf16, f16)", what, d->dtype);
    if (d->rows < 0 || d->width < 1) return fail(CRESSO_E_INVALID, "%s: %lld rows of width %lld", what, (long long)d->rows, (long long)d->width);
    if (d->width > RN_MAX_WIDTH)
        return fail(CRESSO_E_UNSUPPORTED, "%s: width %lld above %d", what, (long long)d->width, RN_MAX_WIDTH);
    if (d->rows == 0) return CRESSO_OK;
    if (!d->residual) return fail(CRESSO_E_INVALID, "%s: null argument", what);
    if ((d->gate || d->post) && !d->update) return fail(CRESSO_E_INVALID, "%s: a gate or a norm of an update that is not there", what);
    if (!(d->eps > 0.0f)) return fail(CRESSO_E_INVALID, "%s: eps must be positive", what);
    const struct { const void* p; int32_t code; const char* name; } vecs[] = {
        {d->gate, d->gate_dtype, "gate"}, {d->post, d->post_dtype, "post_weight"}, {d->pre, d->pre_dtype, "pre_weight"},
        {d->scale_vec, d->scale_dtype, "residual_scale"}};
    for (const auto& v : vecs)
        if (v.p && v.code != CRESSO_F32 && v.code != d->dtype)
            return fail(CRESSO_E_UNSUPPORTED, "%s: %s of dtype %d (f32 or the rows' own)", what, v.name, v.code);
    if (d->gate) {
        if (d->act != CRESSO_GATE_NONE && d->act != CRESSO_GATE_SIGMOID && d->act != CRESSO_GATE_TANH)
            return fail(CRESSO_E_INVALID, "%s: unknown gate activation %d", what, d->act);
        if (d->rows_per_gate < 1 || d->rows % d->rows_per_gate)
            return fail(CRESSO_E_INVALID, "%s: %lld rows are no multiple of %lld rows per gate", what, (long long)d->rows,
                        (long long)d->rows_per_gate);
    }
    const struct { const void* p; int64_t stride, rows; const char* name; } spans[] = {
        {d->residual, d->residual_stride, d->rows, "residual"}, {d->update, d->update_stride, d->rows, "update"},
        {d->gate, d->gate_stride, d->gate ? d->rows / d->rows_per_gate : 0, "gate"},
        {d->d_out, d->d_out_stride, d->rows, "gradient of out"}, {d->d_normed, d->d_normed_stride, d->rows, "gradient of normed"}};
    for (const auto& v : spans)
        if (!row_stride_ok(v.p, v.rows, d->width, v.stride))
            return fail(CRESSO_E_INVALID, "%s: row stride %lld of the %s below the width", what, (long long)v.stride, v.name);
    return CRESSO_OK;
}

}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" int32_t cresso_residual_norm_forward(const cresso_residual_norm_desc* desc, void* stream) {
    const int32_t rc = check_seam("residual norm", desc);
    if (rc != CRESSO_OK || desc->rows == 0) return rc;
    if (desc->pre ? !desc->normed : !desc->out) return fail(CRESSO_E_INVALID, "residual norm: null output");
    SeamArgs a{};
    a.d = *desc;
    if (!a.d.gate) a.d.rows_per_gate = a.d.rows;
    with_shape(desc->dtype, desc->width, [&](auto t, auto wpr, auto nu) {
        constexpr int WPR = decltype(wpr)::value, NU = decltype(nu)::value;
        const int slots = slots_of(WPR);
        const int64_t blocks = std::min<int64_t>((a.d.rows + slots - 1) / slots, RN_FWD_BLOCKS);
        hipLaunchKernelGGL((seam_forward_kernel<decltype(t), WPR, NU>), dim3((uint32_t)blocks), dim3(WPR * 64 * slots), 0,
                           (hipStream_t)stream, a);
    });
    return launched("residual norm");
}

extern "C" size_t cresso_residual_norm_backward_workspace_bytes(const cresso_residual_norm_desc* desc) {
    if (check_seam("residual norm gradient", desc) != CRESSO_OK) return 0;
    if (desc->rows == 0) return 256;
    const SeamArgs a = plan_of(*desc);
    return (size_t)4 * a.workers * a.padded * sizeof(float);
}

extern "C" int32_t cresso_residual_norm_backward(const cresso_residual_norm_desc* desc, void* workspace,
                                                 size_t workspace_bytes, void* stream) {
    const int32_t rc = check_seam("residual norm gradient", desc);
    if (rc != CRESSO_OK || desc->rows == 0) return rc;
    if (!desc->stats && (desc->post || desc->d_normed)) return fail(CRESSO_E_INVALID, "residual norm gradient: no stats of the forward pass");
    if (desc->d_normed && !desc->pre) return fail(CRESSO_E_INVALID, "residual norm gradient: a gradient of a norm that is not there");
    if ((desc->d_gate && !desc->gate) || (desc->d_post && !desc->post) || (desc->d_pre && !desc->pre) ||
        (desc->d_scale && !desc->scale_vec) || (desc->d_update && !desc->update))
        return fail(CRESSO_E_INVALID, "residual norm gradient: an output for an input that is not there");
    SeamArgs a = plan_of(*desc);
    if (!a.d.gate) a.d.rows_per_gate = a.d.rows;
    const size_t need = (size_t)4 * a.workers * a.padded * sizeof(float);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
        return fail(CRESSO_E_INVALID, "residual norm gradient: workspace of %zu bytes at %p, %zu at a multiple of 16 needed", workspace_bytes,
                    workspace, need);
    const int64_t gates = a.d.gate && a.workers_per_gate > 1 ? a.d.rows / a.d.rows_per_gate : 0;
    a.partial = (float*)workspace;
    const bool full = desc->d_normed && desc->post;
    if (desc->width > RN_WIDE) {
        with_row_dtype(desc->dtype, [&](auto t) {
            using T = decltype(t);
            const auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3((uint32_t)a.workers), dim3(512), 0, (hipStream_t)stream, a);
            };
            constexpr int PER = 512 * Unit<T>::n;
            if (desc->width <= 8192) full ? go(seam_backward_wide_kernel<T, 8192 / PER, true>) : go(seam_backward_wide_kernel<T, 8192 / PER, false>);
            else go(seam_backward_wide_kernel<T, 16384 / PER, false>);   // less of it in scratch: 4096 x 16384 bf16 695 us, 887 with true
        });
    } else {
        with_shape(desc->dtype, desc->width, [&](auto t, auto wpr, auto nu) {
            constexpr int WPR = decltype(wpr)::value, NU = decltype(nu)::value;
            if constexpr (WPR * NU * 64 * Unit<decltype(t)>::n <= RN_WIDE) {
                const int slots = slots_of(WPR);
                const int64_t blocks = (a.workers + slots - 1) / slots;
                const auto go = [&](auto kernel) {
                    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(WPR * 64 * slots), 0, (hipStream_t)stream, a);
                };
                full ? go(seam_backward_kernel<decltype(t), WPR, NU, true>) : go(seam_backward_kernel<decltype(t), WPR, NU, false>);
            }
        });
    }
    if (a.d.d_post || a.d.d_pre || a.d.d_scale || (a.d.d_gate && gates > 0)) {
        with_row_dtype(desc->dtype, [&](auto t) {
            hipLaunchKernelGGL(seam_reduce_kernel<decltype(t)>, dim3((uint32_t)(a.padded / 64), (uint32_t)(3 + gates)),
                               dim3(RN_SUM_NT), 0, (hipStream_t)stream, a);
        });
    }
    return launched("residual norm gradient");
}
