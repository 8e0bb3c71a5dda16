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
//
// A block's scale is split into a power of two, which the conversion of w to
// bf16 applies exactly, and a factor f of magnitude 1 to 2.  The fp32
// accumulators are kept in units of the current block's f and multiplied by
// f_before / f_now where a block begins: one multiplication per accumulator
// and block, and no second set of accumulators for a block's own sum, which
// is what lets a wave hold 128 x 64 outputs.
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int BP = 128;            // block of a scale
constexpr int BP_NT = 256;
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
// rows padded to whole blocks and 16-byte pieces.  64 x 64 bytes a block.
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
    int64_t rows, cols, depth;          // m, n, k: depth is whole blocks
    int64_t r_stride, w_stride, out_stride;
    int64_t scale_n, scale_k;           // strides of the scales along n's and k's blocks
    uint32_t tiles_m, tiles_n;
};

// The tiles of a stage have rows of 64 of k: 128 bytes of r, 64 of w.  The
// 16-byte pieces of a row change places by the row's number, so that 16 lanes
// that read 16 bytes each in one cycle (0-3, 12-15, 20-23 and 24-27, and
// likewise on) find them in different banks.
constexpr int BK = 64;
__device__ __forceinline__ int r_turn(int row) { return ((row >> 1) & 7) ^ (row & 4); }
__device__ __forceinline__ int w_turn(int row) { return ((row >> 4) & 1) * 2 + ((row >> 1) & 1); }

// eight e4m3 values times a power of two as bf16
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi, float unit) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, unit, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, unit, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, unit, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, unit, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The scales of a wave's columns, one block of k after another: lane i holds
// that of block i of a run of 64.  s = unit * f: a power of two between 2^-100
// and 2^100, and the rest (1 to 2 in magnitude unless s is beyond those); by is
// the f before over this one.  A scale of 0 keeps f = 1 and is told by `zero`:
// its block counts as zeros.
struct BlockScale {
    float unit, f, by;
    uint32_t keep;   // 0 for a scale of 0, else all ones
};
struct BlockScales {
    float unit, f, by;
    uint32_t keep;
    __device__ __forceinline__ void load(const float* s, int64_t stride, int first, int blocks, float f_before) {
        const int lane = threadIdx.x & (kWave - 1);
        const float v = s[(int64_t)min(first + lane, blocks - 1) * stride];
        unit = f = 1.0f;
        keep = v == 0.0f ? 0u : ~0u;
        if (keep) {
            int e;
            frexpf(v, &e);
            e = min(max(e - 1, -100), 100);
            unit = ldexpf(1.0f, e);
            f = ldexpf(v, -e);
        }
        const float before = __shfl_up(f, 1, kWave);
        by = (lane ? before : first ? f_before : f) / f;
    }
    __device__ __forceinline__ BlockScale at(int b) const {
        const auto lane = [&](float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), b & 63)); };
        return {lane(unit), lane(f), lane(by), (uint32_t)__builtin_amdgcn_readlane((int)keep, b & 63)};
    }
};

// Tile of a workgroup.  Workgroups go to the 8 XCDs in turn; each XCD takes a
// run of tiles, in columns of 8 tiles of m, so that the tiles that run
// together on one XCD share rows of both operands in its L2.
__device__ __forceinline__ void tile_of(const ProductArgs& a, uint32_t& tm, uint32_t& tn) {
    const uint32_t total = a.tiles_m * a.tiles_n, per = total / 8, rest = total % 8;
    const uint32_t xcd = blockIdx.x % 8, i = blockIdx.x / 8;
    uint32_t t = xcd * per + min(xcd, rest) + i;
    const uint32_t group = 8 * a.tiles_n, g = t / group, in = t - g * group;
    const uint32_t height = min(8u, a.tiles_m - g * 8);
    tm = g * 8 + in % height;
    tn = in / height;
}

// 16 bytes a lane from a buffer to LDS: lane i's go to lds + 16 * i.
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t from, uint32_t lane_at, uint32_t at, uint8_t* lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)lds, 16, lane_at, at, 0, 0);
}
// Waits until at most N of the wave's loads are on their way and all its LDS
// reads have ended (the stage they read is filled anew), then for the other waves.
template <int N> __device__ __forceinline__ void stage_ready() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A group begins with its reads from LDS, whose data the next group needs.
template <int READS> __device__ __forceinline__ void group_order() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_barrier(0);
}

// WM x WN waves of FM x FN fragments of 16 x 16 each.  Three stages of LDS:
// while one is multiplied, the next two are on their way from memory.  A
// stage is multiplied in four groups (two steps of k, two halves of the rows),
// and each group's fragments are read from LDS while the group before is
// multiplied, also across the barrier between two stages.
template <typename T, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM* WN * 64, 2) void product_kernel(ProductArgs a) {
    constexpr int NT = WM * WN * 64, TM = WM * FM * 16, TN = WN * FN * 16, H = FM / 2;
    constexpr int RL = TM * 8 / NT, WL = TN * 4 / NT;   // 16-byte pieces a thread loads per stage
    static_assert(RL * NT == TM * 8 && WL * NT == TN * 4 && FN == 4, "tile");
    constexpr int STAGE = TM * 128 + TN * 64;
    __shared__ __align__(16) uint8_t lds[3 * STAGE];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    uint32_t tm, tn;
    tile_of(a, tm, tn);
    const int64_t m0 = (int64_t)tm * TM, n0 = (int64_t)tn * TN;
    const int wm = (wave % WM) * (FM * 16), wn = (wave / WM) * (FN * 16);
    const int l16 = lane & 15, quad = lane >> 4;
    f32x4 acc[FN][FM] = {};
    // A thread's piece of the tile is the one whose place in LDS it fills.
    // Rows beyond the end load the last row's numbers; what they give is not stored.
    const int64_t rrows = min((int64_t)TM, a.rows - m0), wrows = min((int64_t)TN, a.cols - n0);
    const __amdgpu_buffer_rsrc_t rbuf = make_rsrc(a.r + m0 * a.r_stride, (uint32_t)(rrows * a.r_stride * 2));
    const __amdgpu_buffer_rsrc_t wbuf = make_rsrc(a.w + n0 * a.w_stride, (uint32_t)((wrows - 1) * a.w_stride + a.depth));
    uint32_t ro[RL], wo[WL];   // byte offsets: a tile spans less than 2^32
#pragma unroll
    for (int i = 0; i < RL; ++i) {
        const int place = tid + i * NT, row = place >> 3, piece = (place & 7) ^ r_turn(row);
        ro[i] = (uint32_t)min((int64_t)row, rrows - 1) * (uint32_t)(a.r_stride * 2) + piece * 16;
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int place = tid + i * NT, row = place >> 2, piece = (place & 3) ^ w_turn(row);
        wo[i] = (uint32_t)min((int64_t)row, wrows - 1) * (uint32_t)a.w_stride + piece * 16;
    }
    const float* const sp = a.scales + min(n0 + wn, a.cols - 1) / BP * a.scale_n;
    const int blocks = (int)(a.depth / BP), stages = 2 * blocks;
    int to = wave * 1024;   // where the next stage goes
    int next = 0;           // the stage to load; past the last one that is loaded again, and not used
    const auto fetch = [&] {
#pragma unroll
        for (int i = 0; i < RL; ++i) load_lds(rbuf, ro[i], next * (BK * 2), lds + to + i * (NT * 16));
#pragma unroll
        for (int i = 0; i < WL; ++i) load_lds(wbuf, wo[i], next * BK, lds + to + TM * 128 + i * (NT * 16));
        next = min(next + 1, stages - 1);
        to = to >= 2 * STAGE ? to - 2 * STAGE : to + STAGE;
    };
    // a lane's k: 16 of its quarter of the stage, 8 for each of two steps; a
    // fragment's row r of w is column 16*(r/4) + 4*i + r%4, so that a lane ends
    // with 16 consecutive columns of a row of the result (i leaves w_turn as it is)
    const int wrow = wn + (l16 >> 2) * 16 + (l16 & 3), wat = TM * 128 + wrow * 64 + ((quad ^ w_turn(wrow)) * 16);
    const int rrow = wm + l16, rat[2] = {rrow * 128 + (((quad * 2) ^ r_turn(rrow)) * 16), rrow * 128 + (((quad * 2 + 1) ^ r_turn(rrow)) * 16)};
    int from = 0;           // the stage that is read
    u32x4 fw[FN];
    bf16x8 fr[2][H];
    const auto read_w = [&] {
#pragma unroll
        for (int i = 0; i < FN; ++i) fw[i] = *(const u32x4*)(lds + from + wat + i * 256);
    };
    const auto read_r = [&](int set, int s, int h) {
#pragma unroll
        for (int j = 0; j < H; ++j) fr[set][j] = *(const bf16x8*)(lds + from + rat[s] + (h * H + j) * 2048);
    };
    bf16x8 f[FN];
    const auto widen = [&](int s, const BlockScale& by) {
#pragma unroll
        for (int i = 0; i < FN; ++i) f[i] = widen8(fw[i][2 * s] & by.keep, fw[i][2 * s + 1] & by.keep, by.unit);
    };
    const auto multiply = [&](int set, int h) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j)
                acc[i][h * H + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[i], fr[set][j], acc[i][h * H + j], 0, 0, 0);
    };
    const auto rescale = [&](int h, float by) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][h * H + j][e] *= by;
    };
    // Multiplies a stage and reads the first fragments of the next.  Where a
    // block begins, the second half's accumulators are multiplied by `by` on
    // the way; where it ends, the first half's, for the next block.
    const auto stage = [&](const BlockScale& now, bool begins, float by) {
        read_r(1, 0, 1);
        if (begins) rescale(1, by);
        widen(0, now);
        multiply(0, 0);
        group_order<H>();
        read_r(0, 1, 0);
        multiply(1, 1);
        group_order<H>();
        read_r(1, 1, 1);
        widen(1, now);
        multiply(0, 0);
        group_order<H>();
        stage_ready<RL + WL>();
        fetch();
        from = from >= 2 * STAGE ? 0 : from + STAGE;
        read_w();
        read_r(0, 0, 0);
        if (!begins) rescale(0, by);
        multiply(1, 1);
        group_order<FN + H>();
    };
    BlockScale now{1.0f, 1.0f, 1.0f, 0u};
    if (blocks) {
        BlockScales scales;
        scales.load(sp, a.scale_k, 0, blocks, 1.0f);
        now = scales.at(0);
        fetch();
        fetch();
        fetch();
        stage_ready<2 * (RL + WL)>();
        read_w();
        read_r(0, 0, 0);
        for (int b = 0; b < blocks; ++b) {
            if (((b + 1) & 63) == 0) scales.load(sp, a.scale_k, b + 1, blocks, now.f);
            BlockScale next = now;
            next.by = 1.0f;
            if (b + 1 < blocks) next = scales.at(b + 1);
            stage(now, true, now.by);
            stage(now, false, next.by);
            now = next;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing is on its way to LDS when the workgroup ends
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t m = m0 + wm + j * 16 + l16;
        if (m >= a.rows) continue;
        constexpr int E = Unit<T>::n;
        T* to = (T*)a.out + m * a.out_stride;
        const int64_t n = n0 + wn + quad * 16;
#pragma unroll
        for (int u = 0; u < 16 / E; ++u) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = acc[(u * E + e) / 4][j][(u * E + e) % 4] * now.f;
            store_unit(to, (n + u * E) / E, a.cols, narrow<T>(v));
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
    o.w_stride = up(depth, BP);
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
    // the kernel takes whole blocks of k, aligned 16-byte pieces, and 32-bit places in a tile's rows
    return turned || depth % BP || w_stride % 16 || ((uintptr_t)w & 15) || w_stride >= (int64_t)1 << 23;
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
            // the laid-out rows' ends are written too
            const dim3 grid((uint32_t)((turned ? up(c, 64) : o.w_stride) / 64), (uint32_t)((turned ? o.w_stride : up(r, 64)) / 64));
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
        using T = decltype(t);
        const auto go = [&](auto kernel, int tm, int tn, int threads) {
            a.tiles_m = (uint32_t)((rows + tm - 1) / tm);
            a.tiles_n = (uint32_t)((cols + tn - 1) / tn);
            hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n), dim3(threads), 0, st, a);
        };
        if (((rows + 255) / 256) * ((cols + 255) / 256) >= 256)
            go(product_kernel<T, 2, 4, 8, 4>, 256, 256, 512);
        else
            go(product_kernel<T, 2, 2, 4, 4>, 128, 128, 256);
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
