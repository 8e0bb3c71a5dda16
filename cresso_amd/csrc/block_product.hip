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
//
// A block whose scale is 0 counts as zeros, whatever its values: who divides a
// block of zeros by its largest magnitude is left with that scale and NaN.
//
// 16384 x 2048 x 5632 bf16: 372 us, 1015 TFLOP/s, after 23 us for the rounding
// (a plain bf16 product of the library: 354 to 374 us); its gradient 325 us,
// 1163 TFLOP/s, after 62 us (the library: 246).  The matrix instructions are
// busy for 47 and 54 % of the time, without a conflict in LDS; beside each of 16
// cycles stand 2.1 other vector instructions of 4 (conversion, rescaling), the
// last of the rounds is half empty (8 %), and all waves of a workgroup pass a
// barrier a stage, so the two of a SIMD read and convert at the same time.  8 x 2048 x 5632: 6 to 7 us, 1.8 TB/s, latency; 333 x 1024 x
// 1536 5.4 + 7.7 us.
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
// x rounded to e4m3 times a power of two, as bf16
// ---------------------------------------------------------------------------
constexpr uint32_t BP_INF = 0x7f800000u;
__device__ __forceinline__ float float_of(uint32_t b) { return __builtin_bit_cast(float, b); }
__device__ __forceinline__ uint32_t bits_of(float v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ uint32_t raw_of(bf16x2 v) { return __builtin_bit_cast(uint32_t, v); }

// N values of a row's block, the rest of which other lanes hold; join(u) is
// the largest u among those lanes.  All lanes of the wave take part.
template <int N, typename Join>
__device__ __forceinline__ void round_block(float (&v)[N], uint32_t (&out)[N / 2], Join&& join) {
    uint32_t top = 0;   // largest magnitude, as bits: they order as the numbers do
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, bits_of(v[i]) & 0x7fffffffu);
    top = join(top);
    const bool odd = top >= BP_INF;
    if (__any(odd)) {   // of the finite ones
        top = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t u = bits_of(v[i]) & 0x7fffffffu;
            top = max(top, u < BP_INF ? u : 0u);
        }
        top = join(top);
    }
    // top = 1.m * 2^(E-127) <= 448 * 2^e = 1.75 * 2^(e+8)
    const int e = max(BP_MIN_EXP, (int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u));
    const float down = float_of((uint32_t)(127 - e) << 23), up = float_of((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= down;
    if (__any(odd || e == 120)) {   // no infinities in the format; 256 * 2^120 is beyond fp32
        const float most = e == 120 ? 240.0f : 448.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = fabsf(v[i]) < INFINITY ? fminf(fmaxf(v[i], -most), most) : __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
        out[i] = raw_of(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2 * i], v[2 * i + 1], 0, false), up, false));
}

// N values from column `at` of a row of `width` (0 beyond it); N is whole units
template <typename T, int N> __device__ __forceinline__ void load_values(const T* row, int64_t at, int64_t width, float (&v)[N]) {
    constexpr int E = Unit<T>::n;
#pragma unroll
    for (int u = 0; u < N / E; ++u) {
        float t[E];
        widen<T>(load_unit(row, at / E + u, width), t);
#pragma unroll
        for (int i = 0; i < E; ++i) v[u * E + i] = t[i];
    }
}

// ---------------------------------------------------------------------------
// The weight's other layout: along n for the gradient (TURN), or only with
// rows padded to whole blocks and 16-byte pieces.  64 x 64 bytes a workgroup,
// 16 a lane in and out; turned, a lane gathers 16 bytes of a column from LDS,
// whose rows are 17 words apart, so that a wave's four runs of 16 rows lie 16
// banks from one another.
// ---------------------------------------------------------------------------
__device__ __forceinline__ u32x4 load_bytes(const uint8_t* p, int64_t left) {
    if (left >= 16) return ((const CRESSO_GLOBAL Raw16h*)p)->v;
    u32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
        if (i < left) r[i / 4] |= (uint32_t)((const CRESSO_GLOBAL uint8_t*)p)[i] << (8 * (i & 3));
    return r;
}
struct LayOut {
    const uint8_t* w;
    int64_t rows, cols, stride;   // as the weight is held
    uint8_t* out;
    int64_t out_stride;
    uint32_t wide, high;          // workgroups; 0: the weight is taken as it is
    int32_t turn;
};
__device__ __forceinline__ void lay_out(const LayOut& l, uint32_t block) {
    __shared__ uint32_t tile[64][17];
    const int a = threadIdx.x >> 2, b = (threadIdx.x & 3) * 16;
    const int64_t r0 = (int64_t)(block / l.wide) * 64, c0 = (int64_t)(block % l.wide) * 64;
    u32x4 v = {0, 0, 0, 0};
    if (r0 + a < l.rows) v = load_bytes(l.w + (r0 + a) * l.stride + c0 + b, l.cols - c0 - b);
    if (!l.turn) {
        if (r0 + a < l.rows) *(u32x4*)(l.out + (r0 + a) * l.out_stride + c0 + b) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[a][b / 4 + i] = v[i];
    __syncthreads();
    if (c0 + a >= l.cols) return;
    const uint8_t* from = (const uint8_t*)tile + a;   // column a, rows b on
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i] |= (uint32_t)from[(b + 4 * i + k) * 68] << (8 * k);
    }
    *(u32x4*)(l.out + (c0 + a) * l.out_stride + r0 + b) = v;
}

// What comes before a product, in one launch: the first workgroups lay the
// weight out, where that is wanted, the others round the rows: 16 lanes hold
// one row's 128 elements.
template <typename T>
__global__ __launch_bounds__(BP_NT) void prepare_kernel(LayOut l, const T* x, int64_t rows, int64_t width, int64_t stride, uint16_t* q,
                                                        int64_t q_stride) {
    const uint32_t laying = l.wide * l.high;
    if (blockIdx.x < laying) {
        lay_out(l, blockIdx.x);
        return;
    }
    const int64_t blocks = q_stride / BP;
    const int64_t job = ((int64_t)(blockIdx.x - laying) * BP_NT + threadIdx.x) / 16;
    const bool on = job < rows * blocks;
    const int64_t row = on ? job / blocks : 0, at = on ? (job - row * blocks) * BP + (threadIdx.x & 15) * 8 : width;
    float v[8];
    load_values(x + row * stride, at, width, v);
    uint32_t r[4];
    round_block(v, r, [](uint32_t u) {
#pragma unroll
        for (int m = 8; m >= 1; m >>= 1) u = max(u, (uint32_t)__shfl_xor((int)u, m, kWave));
        return u;
    });
    if (on) *(u32x4*)(q + row * q_stride + at) = u32x4{r[0], r[1], r[2], r[3]};
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
// r of the 16 columns of a fragment of w: row of the tile of w
template <int FN> __device__ __forceinline__ int w_row(int r) { return (r >> 2) * (4 * FN) + (r & 3); }
template <int FN> __device__ __forceinline__ int w_turn(int row) {
    if constexpr (FN == 4) return ((row >> 4) & 1) * 2 + ((row >> 1) & 1);
    const int a = row / (4 * FN);
    return ((a ^ (a >> 1)) & 1) * 2 + ((a >> 1) & 1);
}

// eight e4m3 values times a power of two as bf16
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi, float unit) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, unit, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, unit, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, unit, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, unit, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// s = unit * f: a power of two between 2^-100 and 2^100, and the rest (1 to 2
// in magnitude unless s is 0 or beyond those).  With the power of two in w no
// sum of products overflows that does not in the result.
__device__ __forceinline__ void split_scale(float s, float& unit, float& f) {
    const int e = min(max((int)((bits_of(s) >> 23) & 255) - 127, -100), 100);
    unit = float_of((uint32_t)(127 + e) << 23);
    f = s * float_of((uint32_t)(127 - e) << 23);
}

// The scales of a wave's columns, one block of k after another: lane i holds
// that of block i of a run of 64; by is the f before over this one.  A scale of
// 0 has f = 1, and `keep` makes its block count as zeros.
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
        split_scale(v, unit, f);
        keep = v == 0.0f ? 0u : ~0u;
        if (!keep) f = 1.0f;
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
// while one is multiplied, the next two are on their way from memory.
// Fragments are read from LDS a group of matrix instructions before they are
// needed, also across the barrier between two stages.  A group is a quarter of
// a stage where a wave has many rows (FM = 8: one of two steps of k, one half of
// the rows), since there are no registers for more; a whole stage otherwise,
// as fewer instructions do not cover the latency of LDS.
template <typename T, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM* WN * 64, 2) void product_kernel(ProductArgs a) {
    constexpr int NT = WM * WN * 64, TM = WM * FM * 16, TN = WN * FN * 16;
    constexpr bool QUARTERS = FM > 4;
    constexpr int H = QUARTERS ? FM / 2 : FM, SETS = QUARTERS ? 1 : 2;
    constexpr int RL = TM * 8 / NT, WL = TN * 4 / NT;   // 16-byte pieces a thread loads per stage
    static_assert(RL * NT == TM * 8 && WL * NT == TN * 4, "tile");
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
        const int place = tid + i * NT, row = place >> 2, piece = (place & 3) ^ w_turn<FN>(row);
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
    // fragment's row r of w is column 4*FN*(r/4) + 4*i + r%4, so that a lane ends
    // with 4*FN consecutive columns of a row of the result (i leaves w_turn as it is)
    const int wrow = wn + w_row<FN>(l16), wat = TM * 128 + wrow * 64 + ((quad ^ w_turn<FN>(wrow)) * 16);
    const int rrow = wm + l16, rat[2] = {rrow * 128 + (((quad * 2) ^ r_turn(rrow)) * 16), rrow * 128 + (((quad * 2 + 1) ^ r_turn(rrow)) * 16)};
    int from = 0;           // the stage that is read
    u32x4 fw[SETS][FN];
    bf16x8 fr[2 * SETS][H], f[FN];
    const auto read_w = [&](int set) {
#pragma unroll
        for (int i = 0; i < FN; ++i) fw[set][i] = *(const u32x4*)(lds + from + wat + i * 256);
    };
    const auto read_r = [&](int set, int s, int h) {
#pragma unroll
        for (int j = 0; j < H; ++j) fr[set][j] = *(const bf16x8*)(lds + from + rat[s] + (h * H + j) * 2048);
    };
    const auto widen = [&](int set, int s, const BlockScale& by) {
#pragma unroll
        for (int i = 0; i < FN; ++i) f[i] = widen8(fw[set][i][2 * s] & by.keep, fw[set][i][2 * s + 1] & by.keep, by.unit);
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
    const auto turn = [&] {   // to the next stage
        stage_ready<RL + WL>();
        fetch();
        from = from >= 2 * STAGE ? 0 : from + STAGE;
    };
    // Multiplies a stage, the first or second of its block, and reads the first
    // fragments of the next.  The accumulators are multiplied by the block's
    // `by` on the way; in quarters the second half's where the block begins
    // and the first half's where the one before it ends.
    const auto stage = [&](const BlockScale& now, const BlockScale& next, int second) {
        if constexpr (QUARTERS) {
            read_r(1, 0, 1);
            if (!second) rescale(1, now.by);
            widen(0, 0, now);
            multiply(0, 0);
            group_order<H>();
            read_r(0, 1, 0);
            multiply(1, 1);
            group_order<H>();
            read_r(1, 1, 1);
            widen(0, 1, now);
            multiply(0, 0);
            group_order<H>();
            turn();
            read_w(0);
            read_r(0, 0, 0);
            if (second) rescale(0, next.by);
            multiply(1, 1);
            group_order<FN + H>();
        } else {
            turn();
            read_w(second ^ 1);
            read_r((second ^ 1) * 2, 0, 0);
            read_r((second ^ 1) * 2 + 1, 1, 0);
            if (!second) rescale(0, now.by);
            widen(second, 0, now);
            multiply(second * 2, 0);
            widen(second, 1, now);
            multiply(second * 2 + 1, 0);
            group_order<FN + 2 * H>();
        }
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
        read_w(0);
        read_r(0, 0, 0);
        if constexpr (!QUARTERS) read_r(1, 1, 0);
        for (int b = 0; b < blocks; ++b) {
            if (((b + 1) & 63) == 0) scales.load(sp, a.scale_k, b + 1, blocks, now.f);
            BlockScale next = now;
            next.by = 1.0f;
            if (b + 1 < blocks) next = scales.at(b + 1);
            stage(now, next, 0);
            stage(now, next, 1);
            now = next;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing is on its way to LDS when the workgroup ends
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t m = m0 + wm + j * 16 + l16;
        if (m >= a.rows) continue;
        T* to = (T*)a.out + m * a.out_stride;
        const int64_t n = n0 + wn + quad * (4 * FN);
        constexpr int E = Unit<T>::n;
        if constexpr (4 * FN < E) {   // half a unit
            const uint32_t lo = narrow2<T>(acc[0][j][0] * now.f, acc[0][j][1] * now.f), hi = narrow2<T>(acc[0][j][2] * now.f, acc[0][j][3] * now.f);
            if (n + 4 <= a.cols) store8(to + n, u32x2{lo, hi});
            else if (n < a.cols) store_part(to + n, u32x4{lo, hi, 0, 0}, (int)(a.cols - n));
        } else {
#pragma unroll
            for (int u = 0; u < 4 * FN / E; ++u) {
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = acc[(u * E + e) / 4][j][(u * E + e) % 4] * now.f;
                store_unit(to, (n + u * E) / E, a.cols, narrow<T>(v));
            }
        }
    }
}

// ---------------------------------------------------------------------------
// At most 16 rows: bound by the weight's bytes, and below some megabytes by
// latency.
//
// A workgroup takes 16 FN columns and all of k, its eight waves every eighth
// block of 128 each; the waves' sums are added in LDS in their order.  The
// weight goes from memory to registers, as it lies (any alignment); a lane's
// 32 bytes of a row's block are the operand of four matrix instructions.  Each
// wave rounds its part of the rows itself, in that same layout: repeated for
// every workgroup, but the whole product is one launch.  The rounding is most
// of the arithmetic, so wide weights take FN = 2 or 4, as long as that leaves a
// workgroup for about each CU (8 x 2048 x 2048: 5.4 us with 1, 6.5 with 2; x 5632: 8.6
// with 1, 7.3 with 2, 8.5 with 4; 8 x 4096 x 8192: 13.2, 11.6 and 13.4; x 11008:
// 18.9, 17.6 and 14.3).  The depth does not move the edges: of 45 products from 512
// x 1024 to 16384 x 32000 the columns alone chose the fastest but once (512 x 32000
// 8.4 with 4, 8.2 with 2); 512 x 4096 3.5 with 1 and 3.8 with 2, x 5632 4.0 and 3.8,
// 16384 x 4096 26.9 and 29.9, x 5632 39.6 and 34.2.  16 x 2048 x 5632 takes 7.3
// us, in tiles 4.8 + 8.9.
// ---------------------------------------------------------------------------
constexpr int FEW_WAVES = 8;
constexpr int FEW_ROWS = 16;

template <typename T, int FN>
__global__ __launch_bounds__(FEW_WAVES * 64) void few_rows_kernel(ProductArgs a, const T* x, int64_t x_stride) {
    __shared__ f32x4 sums[FEW_WAVES][FN][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, quad = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * FN);
    const int blocks = (int)((a.depth + BP - 1) / BP);
    const uint8_t* wp[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) wp[i] = a.w + min(n0 + i * 16 + l16, a.cols - 1) * a.w_stride;
    const float* sp = a.scales + n0 / BP * a.scale_n;   // 16 FN divides 128
    const T* xp = x + min((int64_t)l16, a.rows - 1) * x_stride;
    f32x4 acc[FN] = {};
    for (int b = wave; b < blocks; b += FEW_WAVES) {
        const int64_t k = (int64_t)b * BP + quad * 32;
        u32x4 w[FN][2];
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[i][h] = load_bytes(wp[i] + k + h * 16, a.depth - k - h * 16);
        const float scale = sp[b * a.scale_k];
        float v[32];
        load_values(xp, k, a.depth, v);
        uint32_t u[16];
        round_block(v, u, [](uint32_t t) {
            t = max(t, (uint32_t)__shfl_xor((int)t, 16, kWave));
            return max(t, (uint32_t)__shfl_xor((int)t, 32, kWave));
        });
        float unit, f;
        split_scale(scale, unit, f);
        if (scale == 0.0f) {   // the block counts as zeros, as in the tiles
#pragma unroll
            for (int i = 0; i < FN; ++i) w[i][0] = w[i][1] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            f32x4 p = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < 4; ++s)
                p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    widen8(w[i][s / 2][2 * (s & 1)], w[i][s / 2][2 * (s & 1) + 1], unit),
                    __builtin_bit_cast(bf16x8, u32x4{u[4 * s], u[4 * s + 1], u[4 * s + 2], u[4 * s + 3]}), p, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] += p[e] * f;
        }
    }
#pragma unroll
    for (int i = 0; i < FN; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= FN) return;   // a wave for each fragment
    f32x4 v = sums[0][wave][lane];
#pragma unroll
    for (int k = 1; k < FEW_WAVES; ++k) {
        const f32x4 o = sums[k][wave][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += o[e];
    }
    const int64_t n = n0 + wave * 16 + quad * 4;
    if (l16 < a.rows) {
        T* to = (T*)a.out + l16 * a.out_stride + n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < a.cols) to[e] = from_w<T>(v[e]);
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

// How a product is computed: up to 16 rows in one launch (tile 0), more of them
// rounded first and then multiplied in tiles.
//
// 256 x 256 tiles run one to a CU and 128 x 128 two, in rounds of 256 and 512;
// a round of the first takes 1.6 to 1.9 times as long as one of the second
// (16384 x 2048 x 5632 372 us in 6 rounds, 416 in 11; 4096 x 4096 x 4096 114 in
// one, 122 in two; but 4352 x 2048 x 4352, 289 tiles of 256 or 1156 of 128, 111
// us against 81).  Smaller tiles take over where
// too few would be left for all CUs: 64 x 64 below 192 tiles of 128 (512 x 2048
// x 5632 25.5 us against 26.9, but 1024 x 4096 x 4096 58 against 47), 32 x 64
// below 256 tiles of 64 (200 x 2048 x 2048 13.0 us against 15.1, but 333 x
// 4096 x 5632 38.7 against 36.9; all of these with the rounding before them).
struct ProductPlan {
    int tile;
    bool copy;   // the weight is laid out anew
    int64_t r, w, total, r_stride, w_stride;
};
ProductPlan product_plan(int64_t rows, int64_t cols, int64_t depth, const void* weight, int64_t w_stride, int32_t turned) {
    ProductPlan o{};
    if (rows > FEW_ROWS) {
        const auto tiles = [&](int64_t t) { return ((rows + t - 1) / t) * ((cols + t - 1) / t); };
        const int64_t rounds256 = (tiles(256) + 255) / 256, rounds128 = (tiles(128) + 511) / 512;
        if (50 * rounds256 <= 29 * rounds128) o.tile = 256;
        else o.tile = tiles(128) >= 192 ? 128 : tiles(64) >= 256 ? 64 : 32;
    }
    // tiles take whole blocks of k, aligned 16-byte pieces, and 32-bit places in a tile's rows
    o.copy = turned || (o.tile && (depth % BP || w_stride % 16 || ((uintptr_t)weight & 15) || w_stride >= (int64_t)1 << 23));
    int64_t off = 0;
    const auto take = [&](int64_t b) { const int64_t at = off; off = up(off + b, 256); return at; };
    o.r_stride = up(depth, BP);
    if (o.tile) o.r = take(rows * o.r_stride * 2);
    o.w_stride = up(depth, BP);
    if (o.copy) o.w = take(cols * o.w_stride);
    o.total = std::max<int64_t>(off, 256);
    return o;
}

int32_t check_product(const char* what, int64_t rows, int64_t cols, int64_t depth, int32_t dtype) {
    if (!row_dtype(dtype)) return fail(CRESSO_E_UNSUPPORTED, "%s: dtype %d not supported (f32, bf16, f16)", what, dtype);
    if (rows < 0 || cols < 0 || depth < 0) return fail(CRESSO_E_INVALID, "%s: negative size", what);
    // grids of up to 2^32 threads, 32-bit places in a tile's rows
    if (rows >= (int64_t)1 << 22 || cols >= (int64_t)1 << 21 || depth >= (int64_t)1 << 21 || rows * (depth / BP + 1) >= (int64_t)1 << 27 ||
        cols * depth >= (int64_t)1 << 34 || rows * cols >= (int64_t)1 << 38)
        return fail(CRESSO_E_UNSUPPORTED, "%s: %lld x %lld x %lld is more than one call takes", what, (long long)rows,
                    (long long)cols, (long long)depth);
    return CRESSO_OK;
}
}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" size_t cresso_block_product_workspace_bytes(int64_t rows, int64_t cols, int64_t depth, const void* w,
                                                       int64_t w_stride, int32_t turned) {
    if (check_product("block product", rows, cols, depth, CRESSO_F32) != CRESSO_OK) return 0;
    return (size_t)product_plan(rows, cols, depth, w, w_stride, turned).total;
}

extern "C" int32_t cresso_block_product(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols,
                                        int64_t depth, const void* w, int64_t w_stride, const float* scales,
                                        int64_t scale_stride, int32_t turned, void* out, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const int32_t rc = check_product("block product", rows, cols, depth, dtype);
    if (rc != CRESSO_OK) return rc;
    if (rows == 0 || cols == 0) return CRESSO_OK;
    if (!out || (depth > 0 && (!x || !w || !scales))) return fail(CRESSO_E_INVALID, "block product: null argument");
    const int64_t w_rows = turned ? depth : cols, w_cols = turned ? cols : depth;
    if (!row_stride_ok(x, rows, depth, x_stride)) return fail(CRESSO_E_INVALID, "block product: row stride %lld of x below the depth", (long long)x_stride);
    if (w_rows > 1 && w_stride < w_cols)
        return fail(CRESSO_E_INVALID, "block product: row stride %lld of a weight of %lld columns", (long long)w_stride, (long long)w_cols);
    if (w_rows > BP && scale_stride < up(w_cols, BP) / BP)
        return fail(CRESSO_E_INVALID, "block product: row stride %lld of the scales of %lld columns", (long long)scale_stride, (long long)w_cols);
    const ProductPlan o = product_plan(rows, cols, depth, w, w_stride, turned);
    if (!workspace || workspace_bytes < (size_t)o.total || ((uintptr_t)workspace & 15))
        return fail(CRESSO_E_INVALID, "block product: workspace of %zu bytes at %p, %lld at a multiple of 16 needed", workspace_bytes, workspace,
                    (long long)o.total);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    ProductArgs a{};
    a.r = (const uint16_t*)(ws + o.r);
    a.r_stride = o.r_stride;
    a.w = o.copy ? (uint8_t*)ws + o.w : (const uint8_t*)w;
    a.w_stride = o.copy ? o.w_stride : w_stride;
    a.scales = scales;
    a.scale_n = turned ? 1 : scale_stride;
    a.scale_k = turned ? scale_stride : 1;
    a.out = out;
    a.out_stride = cols;
    a.rows = rows;
    a.cols = cols;
    a.depth = o.copy ? o.w_stride : depth;
    LayOut l{};
    if (o.copy && depth > 0) {
        l = {(const uint8_t*)w, turned ? depth : cols, turned ? cols : depth, w_stride, (uint8_t*)ws + o.w, o.w_stride, 0, 0, turned};
        // the laid-out rows' ends are written too
        l.wide = (uint32_t)((turned ? up(cols, 64) : o.w_stride) / 64);
        l.high = (uint32_t)((turned ? o.w_stride : up(cols, 64)) / 64);
    }
    with_row_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        // 16 rows and fewer are rounded by the product itself
        const int64_t jobs = o.tile ? rows * (o.r_stride / BP) : 0;
        const uint32_t groups = l.wide * l.high + (uint32_t)((jobs * 16 + BP_NT - 1) / BP_NT);
        if (groups)
            hipLaunchKernelGGL(prepare_kernel<T>, dim3(groups), dim3(BP_NT), 0, st, l, (const T*)x, jobs ? rows : 0, depth, x_stride,
                               (uint16_t*)(ws + o.r), o.r_stride);
        if (!o.tile) {
            a.depth = depth;   // x itself is not padded
            const auto few = [&](auto kernel, int fn) {
                hipLaunchKernelGGL(kernel, dim3((uint32_t)((cols + 16 * fn - 1) / (16 * fn))), dim3(FEW_WAVES * 64), 0, st, a, (const T*)x,
                                   x_stride);
            };
            if (cols <= 4096) few(few_rows_kernel<T, 1>, 1);
            else if (cols <= 8192) few(few_rows_kernel<T, 2>, 2);
            else few(few_rows_kernel<T, 4>, 4);
            return;
        }
        const auto tiles = [&](auto kernel, int tm, int tn, int threads) {
            a.tiles_m = (uint32_t)((rows + tm - 1) / tm);
            a.tiles_n = (uint32_t)((cols + tn - 1) / tn);
            hipLaunchKernelGGL(kernel, dim3(a.tiles_m * a.tiles_n), dim3(threads), 0, st, a);
        };
        if (o.tile == 256) tiles(product_kernel<T, 2, 4, 8, 4>, 256, 256, 512);
        else if (o.tile == 128) tiles(product_kernel<T, 1, 4, 8, 2>, 128, 128, 256);
        else if (o.tile == 64) tiles(product_kernel<T, 1, 4, 4, 1>, 64, 64, 256);
        else tiles(product_kernel<T, 1, 4, 2, 1>, 32, 64, 256);
    });
    return launched("block product");
}

extern "C" int32_t cresso_block_quantize(const void* w, int64_t w_stride, int32_t dtype, int64_t rows, int64_t cols,
                                         void* values, float* scales, void* stream) {
    const int32_t rc = check_product("block quantization", rows, cols, 0, dtype);
    if (rc != CRESSO_OK) return rc;
    if (rows == 0 || cols == 0) return CRESSO_OK;
    if (!w || !values || !scales) return fail(CRESSO_E_INVALID, "block quantization: null argument");
    if (!row_stride_ok(w, rows, cols, w_stride)) return fail(CRESSO_E_INVALID, "block quantization: row stride %lld below the width", (long long)w_stride);
    with_row_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const dim3 grid((uint32_t)(up(cols, BP) / BP), (uint32_t)(up(rows, BP) / BP));
        hipLaunchKernelGGL(quantize_blocks_kernel<T>, grid, dim3(BP_NT), 0, (hipStream_t)stream, (const T*)w, rows, cols,
                           w_stride, (uint8_t*)values, scales);
    });
    return launched("block quantization");
}
