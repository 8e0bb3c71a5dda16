// The router of a layer of experts: the `top` experts of each token, their
// weights, the order that brings each expert's rows together, and the gradient
// of the logits.
//
//   key_j = z_j + bias_j (fp32);  chosen: the largest keys, ties to the lowest j, NaN above all, -inf never
//   softmax   w_k = s * exp(z_k) / sum over all (or, normalized, over the chosen) of exp(z)
//   sigmoid   w_k = s * sg(z_k), normalized: over the chosen ones' sum;  sg(z) = 1 / (1 + exp(-z))
// and with p = w / s and d the gradient that arrives
//   softmax     dz_j = s * P_j * ([j chosen] d_j - sum_k p_k d_k),  P = softmax over all
//   normalized  dz_k = w_k * (d_k - sum_j p_j d_j)
//   sigmoid     dz_k = w_k * d_k * (1 - sg(z_k)),  normalized: w_k * (d_k - sum_j p_j d_j) * (1 - sg(z_k))
//
// A wave takes a token: each lane holds the keys of every 64th expert as
// numbers that order as the keys do, and each of the `top` rounds takes their
// maximum over the wave (one instruction a step) and finds its lowest holder
// by a ballot.
//
// The order is a counting sort.  The choosing kernel counts its tokens' slots
// by expert (integer additions in LDS: their order changes nothing), a second
// kernel adds the counts up over the workgroups, expert by expert, and a third
// ranks each workgroup's slots among one another.  Few tokens take one launch
// of one workgroup for all of it.
//
// Bound by instructions: the rounds of the choice, each a maximum and a ballot that
// wait for the one before.  16384 x 64 fp32, top 8: 10.9 us for the choice, 3.6 for the sums over workgroups, 4.9 for the places, 7.9 for the
// gradient (floors of 0.8 to 1.8 at HBM's rate); 8 x 64 in one launch 3.7, which
// is the launch and a chain of eight rounds.
#include "row_ops.hpp"

#include <algorithm>
#include <cmath>

namespace cresso {
namespace {

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_TOP = 32;
constexpr int64_t RT_MAX_TOKENS = (1 << 26) - 16;   // a launch has fewer than 2^32 threads: 64 a token, in workgroups of 16 tokens or 4
constexpr int RT_NT = 256;
constexpr int RT_TOKENS = 16;          // of a workgroup
constexpr int RT_SMALL_NT = 512;       // one workgroup for everything
constexpr int RT_SMALL_TOKENS = 64;
constexpr int RT_SMALL_SLOTS = 512;    // one wave places them 64 at a time
constexpr uint32_t RT_ABSENT = 0x007fffffu;   // order_of(-inf): keys up to here are not taken

struct RouteArgs {
    const void* logits;
    const float* bias;
    float* weights;
    int32_t *experts, *order, *places, *offsets;
    uint32_t* counts;      // [experts + 1][blocks], then where each workgroup's slots begin among the expert's
    uint32_t* totals;      // [experts + 1]
    int64_t stride, tokens;
    int32_t n, top, softmax, normalize;
    float scale;
    uint32_t blocks;
};

// Numbers that order as the keys do; zeros of both signs are one key, NaN is the largest.
__device__ __forceinline__ uint32_t order_of(float k) {
    if (k != k) return 0xffffffffu;
    const uint32_t u = __builtin_bit_cast(uint32_t, k + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
template <int CTRL, int ROW_MASK> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {   // of all lanes, to all lanes
    v = dpp_max<0xB1, 0xF>(v);   // quad_perm [1,0,3,2]
    v = dpp_max<0x4E, 0xF>(v);   // quad_perm [2,3,0,1]
    v = dpp_max<0x124, 0xF>(v);  // row_ror:4
    v = dpp_max<0x128, 0xF>(v);  // row_ror:8
    v = dpp_max<0x142, 0xA>(v);  // row_bcast:15 -> rows 1, 3
    v = dpp_max<0x143, 0xC>(v);  // row_bcast:31 -> rows 2, 3
    return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1);
}
__device__ __forceinline__ float lane_of(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
template <int CTRL, int ROW_MASK> __device__ __forceinline__ float dpp_largest(float v) {   // lanes without a source: -inf
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp((int)0xff800000u, __builtin_bit_cast(int, v), CTRL, ROW_MASK, 0xF, false)));
}
__device__ __forceinline__ float wave_largest(float v) {
    v = dpp_largest<0xB1, 0xF>(v);
    v = dpp_largest<0x4E, 0xF>(v);
    v = dpp_largest<0x124, 0xF>(v);
    v = dpp_largest<0x128, 0xF>(v);
    v = dpp_largest<0x142, 0xA>(v);
    v = dpp_largest<0x143, 0xC>(v);
    return lane_of(v, kWave - 1);
}
__device__ __forceinline__ float route_sum(float v) { return lane_of(wave_total(v), kWave - 1); }

template <typename T, int J> __device__ __forceinline__ void route_load(const RouteArgs& a, int64_t token, float (&z)[J]) {
    const T* row = (const T*)a.logits + token * a.stride;
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int i = j * kWave + lane;
        z[j] = i < a.n ? to_f(row[i]) : -INFINITY;
    }
}

// One token's choice: lane k < top leaves with its k-th expert (n: absent) and that one's weight.
template <int J> __device__ __forceinline__ void route_choose(const RouteArgs& a, const float (&z)[J], int& expert, float& weight) {
    const int lane = threadIdx.x & (kWave - 1);
    uint32_t key[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int i = j * kWave + lane;
        key[j] = 0;
        if (i < a.n) key[j] = order_of(a.bias ? z[j] + a.bias[i] : z[j]);
    }
    expert = a.n;
    float mine = -INFINITY;
    for (int k = 0; k < a.top; ++k) {
        uint32_t m = key[0];
#pragma unroll
        for (int j = 1; j < J; ++j) m = max(m, key[j]);
        m = wave_max(m);
        if (m <= RT_ABSENT) break;
        bool found = false;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const uint64_t who = __ballot(key[j] == m);
            if (!found && who) {
                found = true;
                const int l = __builtin_ctzll(who);
                const float v = lane_of(z[j], l);
                if (lane == k) {
                    expert = j * kWave + l;
                    mine = v;
                }
                if (lane == l) key[j] = 0;
            }
        }
    }
    const bool there = expert < a.n;
    if (a.softmax) {
        float m = there ? mine : -INFINITY;
        if (!a.normalize) {
#pragma unroll
            for (int j = 0; j < J; ++j) m = fmaxf(m, z[j]);
        }
        m = wave_largest(m);
        const float e = there ? expf(mine - m) : 0.0f;
        float sum = 0.0f;
        if (a.normalize) sum = e;
        else {
#pragma unroll
            for (int j = 0; j < J; ++j) sum += j * kWave + lane < a.n ? expf(z[j] - m) : 0.0f;
        }
        sum = route_sum(sum);
        weight = there ? a.scale * (e / sum) : 0.0f;
    } else if (!a.normalize) {
        weight = there ? a.scale * (expf(fminf(mine, 0.0f)) / (1.0f + expf(-fabsf(mine)))) : 0.0f;
    } else {
        // the chosen ones' largest factor is taken out, so that their sum is at least a half whatever they are
        const float m = fminf(wave_largest(there ? mine : -INFINITY), 0.0f);
        const float q = there ? expf(fminf(mine, 0.0f) - m) / (1.0f + expf(-fabsf(mine))) : 0.0f;
        const float sum = route_sum(q);   // by all lanes
        weight = there ? a.scale * (q / sum) : 0.0f;
    }
}
__device__ __forceinline__ void route_store(const RouteArgs& a, int64_t token, int expert, float weight) {
    const int lane = threadIdx.x & (kWave - 1);
    if (lane < a.top) {
        a.experts[token * a.top + lane] = expert < a.n ? expert : -1;
        a.weights[token * a.top + lane] = weight;
    }
}

// ---------------------------------------------------------------------------
// the order
// ---------------------------------------------------------------------------
// The places of up to 64 slots, one a lane, whose expert is e (on: there is a
// slot): next[e] is the place of e's next one.  `bits` hold every e.
__device__ __forceinline__ int32_t place_of(uint32_t* next, uint32_t e, bool on, int bits) {
    uint64_t same = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const uint64_t m = __ballot((e >> b) & 1);
        same &= (e >> b) & 1 ? m : ~m;
    }
    const uint64_t below = (1ull << (threadIdx.x & (kWave - 1))) - 1;
    const uint32_t ahead = (uint32_t)__popcll(same & below);
    uint32_t first = 0;
    if (on) first = next[e];
    __builtin_amdgcn_wave_barrier();
    if (on && !ahead) next[e] = first + (uint32_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
    return (int32_t)(first + ahead);
}
template <int CTRL, int ROW_MASK> __device__ __forceinline__ uint32_t dpp_sum(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {   // inclusive
    v = dpp_sum<0x111, 0xF>(v);   // row_shr:1
    v = dpp_sum<0x112, 0xF>(v);   // row_shr:2
    v = dpp_sum<0x114, 0xF>(v);   // row_shr:4
    v = dpp_sum<0x118, 0xF>(v);   // row_shr:8
    v = dpp_sum<0x142, 0xA>(v);   // row_bcast:15 -> rows 1, 3
    return dpp_sum<0x143, 0xC>(v);   // row_bcast:31 -> rows 2, 3
}

// A wave a token where its registers allow that (16384 x 64 fp32, top 8: 10.9 us, with four
// tokens to a wave 13.1; 2777 x 37 bf16 4.1 and 6.9).
template <int J> constexpr int kRouteThreads = J <= 4 ? RT_TOKENS * kWave : RT_NT;
template <typename T, int J> __global__ __launch_bounds__(kRouteThreads<J>) void route_kernel(RouteArgs a) {
    constexpr int NT = kRouteThreads<J>, WAVES = NT / kWave;
    __shared__ uint32_t count[RT_MAX_EXPERTS + 1];
    for (int e = threadIdx.x; e <= a.n; e += NT) count[e] = 0;
    __syncthreads();
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t first = (int64_t)blockIdx.x * RT_TOKENS;
    float z[J];
    const int64_t t0 = first + wave;
    if (t0 < a.tokens) route_load<T, J>(a, t0, z);
    for (int i = wave; i < RT_TOKENS; i += WAVES) {
        const int64_t t = first + i;
        if (t >= a.tokens) break;
        float next[J];
        if (i + WAVES < RT_TOKENS && t + WAVES < a.tokens) route_load<T, J>(a, t + WAVES, next);
        int expert;
        float weight;
        route_choose(a, z, expert, weight);
        route_store(a, t, expert, weight);
        if (lane < a.top) atomicAdd(&count[expert], 1u);
#pragma unroll
        for (int j = 0; j < J; ++j) z[j] = next[j];
    }
    __syncthreads();
    for (int e = threadIdx.x; e <= a.n; e += NT) a.counts[(int64_t)e * a.blocks + blockIdx.x] = count[e];
}

// Expert blockIdx.x: where each workgroup's slots begin among the expert's, and how many there are.
__global__ __launch_bounds__(RT_NT) void route_scan_kernel(RouteArgs a) {
    __shared__ uint32_t part[RT_NT / kWave];
    uint32_t* column = a.counts + (int64_t)blockIdx.x * a.blocks;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.blocks; b0 += RT_NT) {
        const uint32_t b = b0 + threadIdx.x;
        const uint32_t v = b < a.blocks ? column[b] : 0;
        const uint32_t upto = wave_scan(v);
        __syncthreads();
        if (lane == kWave - 1) part[wave] = upto;
        __syncthreads();
        uint32_t ahead = before;
#pragma unroll
        for (int w = 0; w < RT_NT / kWave; ++w) {
            if (w < wave) ahead += part[w];
            before += part[w];
        }
        if (b < a.blocks) column[b] = ahead + upto - v;
    }
    if (threadIdx.x == 0) a.totals[blockIdx.x] = before;
}

// Where each expert's slots begin, from the totals: next[e] += that.  One wave.
__device__ __forceinline__ void route_begin(uint32_t* next, const uint32_t* totals, int n, int32_t* offsets) {
    const int lane = threadIdx.x & (kWave - 1);
    uint32_t before = 0;
    for (int e0 = 0; e0 <= n; e0 += kWave) {
        const int e = e0 + lane;
        const uint32_t v = e <= n ? totals[e] : 0, upto = wave_scan(v);
        if (e <= n) {
            next[e] += before + upto - v;
            if (offsets) offsets[e] = (int32_t)(before + upto - v);
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)upto, kWave - 1);
    }
}

__global__ __launch_bounds__(kWave) void route_place_kernel(RouteArgs a, int bits) {
    __shared__ uint32_t next[RT_MAX_EXPERTS + 1];
    const int lane = threadIdx.x;
    const int64_t slot0 = (int64_t)blockIdx.x * (RT_TOKENS * a.top);
    const int slots = (int)min((int64_t)(RT_TOKENS * a.top), a.tokens * a.top - slot0);
    int32_t e0 = lane < slots ? a.experts[slot0 + lane] : 0;
    for (int e = lane; e <= a.n; e += kWave) next[e] = a.counts[(int64_t)e * a.blocks + blockIdx.x];
    __builtin_amdgcn_wave_barrier();
    route_begin(next, a.totals, a.n, blockIdx.x == 0 ? a.offsets : nullptr);
    __builtin_amdgcn_wave_barrier();
    for (int s = 0; s < slots; s += kWave) {
        const int i = s + lane;
        const bool on = i < slots;
        const uint32_t e = e0 < 0 ? (uint32_t)a.n : (uint32_t)e0;
        if (i + kWave < slots) e0 = a.experts[slot0 + i + kWave];
        const int32_t place = place_of(next, e, on, bits);
        if (on) {
            a.places[slot0 + i] = place;
            a.order[place] = (int32_t)(slot0 + i);
        }
    }
}

// Everything for at most RT_SMALL_TOKENS tokens.
template <typename T, int J> __global__ __launch_bounds__(RT_SMALL_NT) void route_small_kernel(RouteArgs a, int bits) {
    __shared__ uint32_t count[RT_MAX_EXPERTS + 1], next[RT_MAX_EXPERTS + 1];
    __shared__ int32_t chosen[RT_SMALL_SLOTS];
    for (int e = threadIdx.x; e <= a.n; e += RT_SMALL_NT) {
        count[e] = 0;
        next[e] = 0;
    }
    __syncthreads();
    const int lane = threadIdx.x & (kWave - 1);
    for (int t = threadIdx.x / kWave; t < (int)a.tokens; t += RT_SMALL_NT / kWave) {
        float z[J];
        route_load<T, J>(a, t, z);
        int expert;
        float weight;
        route_choose(a, z, expert, weight);
        route_store(a, t, expert, weight);
        if (lane < a.top) {
            chosen[t * a.top + lane] = expert;
            atomicAdd(&count[expert], 1u);
        }
    }
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    route_begin(next, count, a.n, a.offsets);
    __builtin_amdgcn_wave_barrier();
    const int slots = (int)a.tokens * a.top;
    for (int s = 0; s < slots; s += kWave) {
        const int i = s + lane;
        const bool on = i < slots;
        const int32_t place = place_of(next, on ? (uint32_t)chosen[i] : 0u, on, bits);
        if (on) {
            a.places[i] = place;
            a.order[place] = i;
        }
    }
}

// ---------------------------------------------------------------------------
// the gradient: a wave a token (16384 x 64 fp32, top 8: 7.9 us)
// ---------------------------------------------------------------------------
template <typename T, int J> __global__ __launch_bounds__(RT_NT) void route_backward_kernel(RouteArgs a, const float* d_weights, T* d_logits) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t token = (int64_t)blockIdx.x * (RT_NT / kWave) + threadIdx.x / kWave;
    if (token >= a.tokens) return;
    int e = -1;
    float w = 0.0f, d = 0.0f;
    if (lane < a.top) {
        e = a.experts[token * a.top + lane];
        w = a.weights[token * a.top + lane];
        d = d_weights[token * a.top + lane];
    }
    const bool there = e >= 0 && e < a.n;
    const float p = there && a.scale != 0.0f ? w / a.scale : 0.0f;
    float g[J], z[J];
    const bool all = a.softmax && !a.normalize;
    float mean = 0.0f;
    if (a.softmax || a.normalize) mean = route_sum(there ? p * d : 0.0f);
    float mine = there ? w * (a.normalize ? d - mean : d) : 0.0f;
    if (!a.softmax) {   // times 1 - sigmoid(z)
        float zk = 0.0f;
        if (there) zk = to_f(((const T*)a.logits)[token * a.stride + e]);
        if (there) mine *= expf(-fmaxf(zk, 0.0f)) / (1.0f + expf(-fabsf(zk)));
    }
#pragma unroll
    for (int j = 0; j < J; ++j) g[j] = 0.0f;
    const bool some = __any(there);   // a token without experts has no weights that depend on anything
    if (all && some) {
        route_load<T, J>(a, token, z);
        float m = z[0];
#pragma unroll
        for (int j = 1; j < J; ++j) m = fmaxf(m, z[j]);
        m = wave_largest(m);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            z[j] = j * kWave + lane < a.n ? expf(z[j] - m) : 0.0f;
            sum += z[j];
        }
        const float by = -a.scale * mean / route_sum(sum);
#pragma unroll
        for (int j = 0; j < J; ++j) g[j] = z[j] * by;
    }
    for (int k = 0; k < a.top; ++k) {
        const int ek = __builtin_amdgcn_readlane(e, k);
        const float gk = lane_of(mine, k);
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (ek == j * kWave + lane) g[j] += gk;
    }
    T* row = d_logits + token * a.n;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int i = j * kWave + lane;
        if (i < a.n) row[i] = from_w<T>(g[j]);
    }
}

bool route_small(const cresso_route_desc& d) { return d.tokens <= RT_SMALL_TOKENS && d.tokens * d.top <= RT_SMALL_SLOTS; }
uint32_t route_blocks(const cresso_route_desc& d) { return (uint32_t)((d.tokens + RT_TOKENS - 1) / RT_TOKENS); }

int32_t check_route(const cresso_route_desc* d) {
    if (!d) return fail(CRESSO_E_INVALID, "router: null descriptor");
    if (!row_dtype(d->dtype)) return fail(CRESSO_E_UNSUPPORTED, "router: dtype %d not supported (f32, bf16, f16)", d->dtype);
    if (d->tokens < 0) return fail(CRESSO_E_INVALID, "router: negative size");
    if (d->num_experts < 1 || d->num_experts > RT_MAX_EXPERTS)
        return fail(CRESSO_E_UNSUPPORTED, "router: %d experts, 1 to %d are taken", d->num_experts, RT_MAX_EXPERTS);
    if (d->top < 1 || d->top > RT_MAX_TOP || d->top > d->num_experts)
        return fail(CRESSO_E_UNSUPPORTED, "router: top %d of %d experts, 1 to %d are taken", d->top, d->num_experts, RT_MAX_TOP);
    if (d->tokens > RT_MAX_TOKENS || d->tokens * d->top >= (int64_t)1 << 31)
        return fail(CRESSO_E_UNSUPPORTED, "router: %lld tokens are more than one call takes", (long long)d->tokens);
    if (d->score != CRESSO_SCORE_SOFTMAX && d->score != CRESSO_SCORE_SIGMOID) return fail(CRESSO_E_INVALID, "router: unknown score %d", d->score);
    if (!std::isfinite(d->scale)) return fail(CRESSO_E_INVALID, "router: scale must be finite");
    return CRESSO_OK;
}
RouteArgs route_args(const cresso_route_desc& d) {
    RouteArgs a{};
    a.logits = d.logits;
    a.bias = d.bias;
    a.weights = d.weights;
    a.experts = d.experts;
    a.order = d.order;
    a.places = d.places;
    a.offsets = d.offsets;
    a.stride = d.logits_stride;
    a.tokens = d.tokens;
    a.n = d.num_experts;
    a.top = d.top;
    a.softmax = d.score == CRESSO_SCORE_SOFTMAX;
    a.normalize = d.normalize != 0;
    a.scale = d.scale;
    a.blocks = route_blocks(d);
    return a;
}
size_t route_bytes(const cresso_route_desc& d) {
    if (route_small(d)) return 16;
    return ((size_t)(d.num_experts + 1) * ((size_t)route_blocks(d) + 1) * 4 + 15) / 16 * 16;
}
// fn(T{}, J) with 64 J >= experts
template <typename F> void with_route(const cresso_route_desc& d, F&& fn) {
    with_row_dtype(d.dtype, [&](auto t) {
        const int n = d.num_experts;
        if (n <= 64) fn(t, std::integral_constant<int, 1>{});
        else if (n <= 128) fn(t, std::integral_constant<int, 2>{});
        else if (n <= 256) fn(t, std::integral_constant<int, 4>{});
        else if (n <= 512) fn(t, std::integral_constant<int, 8>{});
        else fn(t, std::integral_constant<int, 16>{});
    });
}
}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" size_t cresso_route_workspace_bytes(const cresso_route_desc* d) {
    return check_route(d) == CRESSO_OK ? route_bytes(*d) : 0;
}

extern "C" int32_t cresso_route_forward(const cresso_route_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    const int32_t rc = check_route(d);
    if (rc != CRESSO_OK) return rc;
    if (!d->offsets || (d->tokens > 0 && (!d->logits || !d->weights || !d->experts || !d->order || !d->places)))
        return fail(CRESSO_E_INVALID, "router: null argument");
    if (!row_stride_ok(d->logits, d->tokens, d->num_experts, d->logits_stride))
        return fail(CRESSO_E_INVALID, "router: row stride %lld of %d logits", (long long)d->logits_stride, d->num_experts);
    if (!workspace || workspace_bytes < route_bytes(*d) || ((uintptr_t)workspace & 15))
        return fail(CRESSO_E_INVALID, "router: workspace of %zu bytes at %p, %zu at a multiple of 16 needed", workspace_bytes, workspace,
                    route_bytes(*d));
    RouteArgs a = route_args(*d);
    a.counts = (uint32_t*)workspace;
    a.totals = a.counts + (size_t)(a.n + 1) * a.blocks;
    hipStream_t st = (hipStream_t)stream;
    int bits = 0;
    while ((a.n >> bits) > 0) ++bits;
    with_route(*d, [&](auto t, auto j) {
        using T = decltype(t);
        constexpr int J = decltype(j)::value;
        if (route_small(*d)) {
            hipLaunchKernelGGL((route_small_kernel<T, J>), dim3(1), dim3(RT_SMALL_NT), 0, st, a, bits);
            return;
        }
        hipLaunchKernelGGL((route_kernel<T, J>), dim3(a.blocks), dim3(kRouteThreads<J>), 0, st, a);
        hipLaunchKernelGGL(route_scan_kernel, dim3(a.n + 1), dim3(RT_NT), 0, st, a);
        hipLaunchKernelGGL(route_place_kernel, dim3(a.blocks), dim3(kWave), 0, st, a, bits);
    });
    return launched("router");
}

extern "C" int32_t cresso_route_backward(const cresso_route_desc* d, const float* d_weights, void* d_logits, void* stream) {
    const int32_t rc = check_route(d);
    if (rc != CRESSO_OK) return rc;
    if (d->tokens == 0) return CRESSO_OK;
    if (!d->logits || !d->weights || !d->experts || !d_weights || !d_logits) return fail(CRESSO_E_INVALID, "router gradient: null argument");
    if (!row_stride_ok(d->logits, d->tokens, d->num_experts, d->logits_stride))
        return fail(CRESSO_E_INVALID, "router gradient: row stride %lld of %d logits", (long long)d->logits_stride, d->num_experts);
    const RouteArgs a = route_args(*d);
    with_route(*d, [&](auto t, auto j) {
        using T = decltype(t);
        const uint32_t blocks = (uint32_t)((a.tokens + RT_NT / kWave - 1) / (RT_NT / kWave));
        hipLaunchKernelGGL((route_backward_kernel<T, decltype(j)::value>), dim3(blocks), dim3(RT_NT), 0, (hipStream_t)stream, a, d_weights,
                           (T*)d_logits);
    });
    return launched("router gradient");
}
