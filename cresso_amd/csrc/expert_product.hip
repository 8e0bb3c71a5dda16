// Grouped products: checks of the arguments and the choice of a kernel
// (expert_product.hpp has the kernels, one source file a dtype compiles them).
#include "expert_product.hpp"

#include <algorithm>

namespace cresso {
template <> void group_launch<float>(GroupArgs, bool, bool, GroupPlan, hipStream_t);
template <> void group_launch<__half>(GroupArgs, bool, bool, GroupPlan, hipStream_t);
template <> void group_launch<__hip_bfloat16>(GroupArgs, bool, bool, GroupPlan, hipStream_t);

namespace {
int32_t check_group(const char* what, int32_t dtype, int64_t rows, int64_t a, int64_t b, int32_t experts) {
    if (!row_dtype(dtype)) return fail(CRESSO_E_UNSUPPORTED, "%s: dtype %d not supported (f32, bf16, f16)", what, dtype);
    if (rows < 0 || a < 0 || b < 0 || experts < 0) return fail(CRESSO_E_INVALID, "%s: negative size", what);
    // offsets of 32 bits; fewer than 2^24 workgroups of 256 threads, the most of a launch, with the smallest tiles
    const auto tiles = [](int64_t n) { return (n + 63) / 64; };
    const int64_t most = ((int64_t)1 << 24) - 4096;
    if (rows >= (int64_t)1 << 31 || a >= (int64_t)1 << 22 || b >= (int64_t)1 << 22 || experts > 1 << 16 ||
        (rows / 32 + experts) * tiles(std::max(a, b)) >= most || experts * (tiles(a) * tiles(b)) >= most)
        return fail(CRESSO_E_UNSUPPORTED, "%s: %lld rows, %d matrices of %lld x %lld are more than one call takes", what, (long long)rows,
                    experts, (long long)a, (long long)b);
    return CRESSO_OK;
}
// Whether rows at p go to LDS in whole pieces of 16 bytes: so do their width and stride, and a
// stage's rows lie within 2^31 bytes.
bool near_rows(int64_t width, int64_t stride) { return stride >= width && stride < (int64_t)1 << 21 && width < (int64_t)1 << 21; }
bool whole_rows(const void* p, int64_t width, int64_t stride, int32_t dtype) {
    const int64_t e = dtype == CRESSO_F32 ? 4 : 8;
    return ((uintptr_t)p & 15) == 0 && width % e == 0 && stride % e == 0 && near_rows(width, stride);
}
// Whether rows of the result are whole pieces of 16 bytes of 16-bit numbers: others take the large tiles longer to store.
bool piece_rows(const void* out, int64_t n) { return ((uintptr_t)out & 15) == 0 && n % 8 == 0; }

// Which tiles, and whether k is split.
//
// A product's time is modelled from its tiles of each side, in us at a depth of
// 2048 and bf16 (measured from 16 to 16384 rows, 4 to 64 experts): 64 on a side
// 12 + 0.0245 each, 128 13 + 0.066, 256 0.25 each but 45 at least.  The fastest
// of 512 x 2048 -> 2048 by 8 experts are 64 (16.8 us, 23.5 and 22.1), of 2000
// by 32 with 1024 columns 128 (31.8, 26.1, 41.9), of 16384 by 8 256 (215, 151,
// 129).  With w across k, tiles of 128 take 12 + 0.075 and those of 64 are no
// faster anywhere; of rows that are not whole it is the other way round (2000 x 1501 -> 1001
// by 32: 47 us with tiles of 64, 70 with 128).  fp32 products take 32 x 64 at any size (kGroupHigh says why).
// Weight gradients take 256 from three rounds of them on, if they have rows
// enough to be more than a store (16384 rows by 64 experts of 2048 x 1024: 173 us,
// 196 with 128; 2000 by 32: 59 and 53; 8192 by 8 of 2048 x 2048: 75 and 72).
//
// Where the tiles leave CUs idle, k is split into parts of 8 stages or more: for
// 16 bits below 256 tiles (64 x 4096 -> 256 by 2: 19.6 us in one part, 11.4 in 8;
// 512 x 2048 -> 2048 by 8, 384 tiles, 15.7 and 21.5 in 2), for fp32, whose tiles
// take longer, below 768 (300 x 4097 -> 515 by 4, 102 tiles: 67.6 us in one part, 35.4
// in 3, 33.3 in 5 or 7).
GroupPlan group_plan(int64_t rows, int64_t m, int64_t n, int64_t depth, int32_t experts, int32_t dtype, bool weight, bool across, bool whole, bool large) {
    const bool wide = dtype == CRESSO_F32;
    const int64_t e = std::max(experts, 1);
    const auto tiles = [&](int64_t t) -> double {
        const double across = (double)((n + t - 1) / t);
        const int64_t high = wide && !weight ? kGroupHigh<float, false> : t;
        return across * (weight ? (double)e * (double)((m + t - 1) / t) : (double)rows / high + 0.5 * (double)std::min(e, rows));
    };
    GroupPlan p{64, 1, whole, false};
    if (weight) {
        const int64_t side = std::min(m, n);
        if (large && !wide && side >= 256 && tiles(256) >= 768.0 && rows >= 128 * e) p.tile = 256;
        else if (whole && side > 64) p.tile = 128;
    } else if (!wide) {
        const bool turn = across && whole;
        const double t64 = turn ? 1e30 : 12.0 + 0.0245 * tiles(64), t128 = turn ? 12.0 + 0.075 * tiles(128) : 13.0 + 0.066 * tiles(128);
        const double t256 = std::max(45.0, 0.25 * tiles(256));
        if (t128 < t64 && (whole || !across)) p.tile = 128;
        if (large && t256 < std::min(t64, t128)) p.tile = 256;
    }
    const int64_t stages = (weight ? rows / e : depth) / (wide ? 32 : 64);
    const double enough = wide ? 768.0 : 256.0;
    // no expert has no tiles to split: the rows are filled with zeros, by workgroups that products in parts do not have
    if (p.tile < 256 && experts > 0) p.splits = (uint32_t)std::min<int64_t>({16, (int64_t)(enough / std::max(1.0, tiles(p.tile))), stages / 8});
    p.splits = std::max(p.splits, 1u);
    return p;
}
size_t group_bytes(const GroupPlan& p, int64_t results) { return p.splits > 1 ? ((size_t)p.splits * (size_t)results * 4 + 15) / 16 * 16 : 16; }

// ---------------------------------------------------------------------------
// Rows of 16-bit numbers that are no whole pieces, laid out anew: in a workspace,
// with zeros behind each row's end.
// ---------------------------------------------------------------------------
struct PadArgs {
    const __half* from;
    __half* to;
    int64_t rows, width, stride;        // of all matrices
    int64_t matrix_rows, matrix_stride;
    int32_t lanes;                      // of a row: a power of two
};
__global__ __launch_bounds__(256) void group_pad_kernel(PadArgs a) {
    const int lane = threadIdx.x & (a.lanes - 1), per = 256 / a.lanes;
    const int64_t units = (a.width + 7) / 8;
    for (int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / a.lanes; r < a.rows; r += (int64_t)gridDim.x * per) {
        const int64_t e = r / a.matrix_rows;
        const __half* row = a.from + e * a.matrix_stride + (r - e * a.matrix_rows) * a.stride;
        for (int64_t u = lane; u < units; u += a.lanes) store16(a.to + (r * units + u) * 8, load_unit(row, u, a.width));
    }
}
int64_t padded(int64_t width) { return (width + 7) / 8 * 8; }
void group_pad(const void* from, void* to, int64_t matrices, int64_t matrix_rows, int64_t matrix_stride, int64_t width, int64_t stride, hipStream_t st) {
    PadArgs a{(const __half*)from, (__half*)to, matrices * matrix_rows, width, stride, matrix_rows, matrix_stride, 8};
    while (a.lanes < kWave && a.lanes * 8 < width) a.lanes *= 2;
    const int64_t per = 256 / a.lanes;
    if (a.rows == 0) return;
    hipLaunchKernelGGL(group_pad_kernel, dim3((uint32_t)std::min<int64_t>((a.rows + per - 1) / per, 1 << 16)), dim3(256), 0, st, a);
}
// Whether that is worth it: the copies take 0.5 to 0.85 us a million numbers and 8
// for two launches, and save, in us a GFLOP measured with and without them, 0.6 to
// 1.1 of a product along k, 1.7 to 2.2 of one across, 2.3 to 4 of a weight gradient.
// Without and with: 16384 x 2047 -> 4095 by 8 554 us and 407, 721 and 435, 1355 and 330; 8192 x 1001
// -> 1501 by 8 67 and 63, 101 and 68, 128 and 61; 4000 x 777 -> 1333 by 16 31 and 43, 46 and 53,
// 49 and 44; 2000 x 1001 -> 1501 by 32 34 and 63, 47 and 60, 80 and 57.
bool group_pads(int64_t rows, int64_t cols, int64_t depth, int64_t numbers, int32_t dtype, double gain) {
    if (dtype == CRESSO_F32) return false;
    const double gflop = 2e-9 * (double)rows * (double)cols * (double)depth;
    return gflop * gain > 8.0 + 0.6e-6 * (double)numbers;
}
constexpr int64_t kPadMost = ((int64_t)1 << 21) - 8;   // near_rows of the copies
constexpr double kPadAlong = 0.9, kPadAcross = 2.2, kPadWeight = 3.5;   // us a GFLOP: w along k, w across it, the weight gradient
}  // namespace
}  // namespace cresso

using namespace cresso;

// Numbers of the copies of x and w, where rows of `depth` or `w_cols` are no whole pieces.
static int64_t product_copies(int64_t rows, int64_t cols, int64_t depth, int32_t experts, int32_t dtype, bool turned) {
    const int64_t w_cols = turned ? cols : depth;
    if ((depth % 8 == 0 && w_cols % 8 == 0) || std::max(depth, w_cols) >= kPadMost) return 0;
    const int64_t numbers = rows * padded(depth) + experts * (turned ? depth : cols) * padded(w_cols);
    return group_pads(rows, cols, depth, numbers, dtype, turned ? kPadAcross : kPadAlong) ? numbers : 0;
}
static int64_t weight_copies(int64_t rows, int64_t p_width, int64_t q_width, int32_t dtype) {
    if ((p_width % 8 == 0 && q_width % 8 == 0) || std::max(p_width, q_width) >= kPadMost) return 0;
    const int64_t numbers = rows * (padded(p_width) + padded(q_width));
    return group_pads(rows, p_width, q_width, numbers, dtype, kPadWeight) ? numbers : 0;
}

// Bytes of the sums, where k is split, whatever the operands' layouts; copies come behind them.
static size_t product_sums(int64_t rows, int64_t cols, int64_t depth, int32_t experts, int32_t dtype) {
    size_t most = 0;
    for (int i = 0; i < 8; ++i)
        most = std::max(most, group_bytes(group_plan(rows, 0, cols, depth, experts, dtype, false, i & 1, i & 2, (i & 4) && (i & 2)), rows * cols));
    return most;
}
static size_t weight_sums(int64_t rows, int64_t p_width, int64_t q_width, int32_t experts, int32_t dtype) {
    size_t most = 0;
    for (int i = 0; i < 3; ++i)
        most = std::max(most, group_bytes(group_plan(rows, p_width, q_width, 0, experts, dtype, true, true, i > 0, i > 1), experts * p_width * q_width));
    return most;
}

extern "C" size_t cresso_expert_product_workspace_bytes(int64_t rows, int64_t cols, int64_t depth, int32_t experts, int32_t dtype) {
    if (check_group("expert product", dtype, rows, cols, depth, experts) != CRESSO_OK) return 0;
    return product_sums(rows, cols, depth, experts, dtype) +
           2 * (size_t)std::max(product_copies(rows, cols, depth, experts, dtype, false), product_copies(rows, cols, depth, experts, dtype, true));
}
extern "C" size_t cresso_expert_product_weight_workspace_bytes(int64_t rows, int64_t p_width, int64_t q_width, int32_t experts,
                                                               int32_t dtype) {
    if (check_group("expert product gradient", dtype, rows, p_width, q_width, experts) != CRESSO_OK) return 0;
    return weight_sums(rows, p_width, q_width, experts, dtype) + 2 * (size_t)weight_copies(rows, p_width, q_width, dtype);
}

extern "C" int32_t cresso_expert_product(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, int64_t depth,
                                         const void* w, int64_t w_expert_stride, int64_t w_stride, int32_t turned, int32_t experts,
                                         const int32_t* offsets, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "expert product";
    const int32_t rc = check_group(what, dtype, rows, cols, depth, experts);
    if (rc != CRESSO_OK) return rc;
    if (rows == 0 || cols == 0) return CRESSO_OK;
    if (!out || !offsets || (depth > 0 && (!x || (experts > 0 && !w)))) return fail(CRESSO_E_INVALID, "%s: null argument", what);
    if (!row_stride_ok(x, rows, depth, x_stride)) return fail(CRESSO_E_INVALID, "%s: row stride %lld of x below the depth", what, (long long)x_stride);
    const int64_t w_rows = turned ? depth : cols, w_cols = turned ? cols : depth;
    if (w_rows > 1 && w_stride < w_cols)
        return fail(CRESSO_E_INVALID, "%s: row stride %lld of a weight of %lld columns", what, (long long)w_stride, (long long)w_cols);
    if (w_expert_stride < 0) return fail(CRESSO_E_INVALID, "%s: negative stride between experts", what);
    if (!workspace || workspace_bytes < cresso_expert_product_workspace_bytes(rows, cols, depth, experts, dtype) || ((uintptr_t)workspace & 15))
        return fail(CRESSO_E_INVALID, "%s: workspace of %zu bytes at %p, %zu at a multiple of 16 needed", what, workspace_bytes, workspace,
                    cresso_expert_product_workspace_bytes(rows, cols, depth, experts, dtype));
    GroupArgs a{};
    a.a = x;
    a.b = w;
    a.out = out;
    a.offsets = offsets;
    a.rows = rows;
    a.n = cols;
    a.k = depth;
    a.a_stride = x_stride;
    a.b_stride = w_stride;
    a.b_expert = w_expert_stride;
    a.experts = experts;
    a.sums = (float*)workspace;
    a.k_along = depth;
    a.b_across = cols;
    bool whole = whole_rows(x, depth, x_stride, dtype) && whole_rows(w, w_cols, w_stride, dtype) && w_expert_stride % (dtype == CRESSO_F32 ? 4 : 8) == 0;
    if (!whole && product_copies(rows, cols, depth, experts, dtype, turned != 0)) {
        __half* const to = (__half*)((char*)workspace + product_sums(rows, cols, depth, experts, dtype));
        group_pad(x, to, 1, rows, 0, depth, x_stride, (hipStream_t)stream);
        a.a = to;
        a.a_stride = a.k_along = padded(depth);
        a.b = to + rows * a.a_stride;
        a.b_stride = padded(w_cols);
        group_pad(w, (void*)a.b, experts, w_rows, w_expert_stride, w_cols, w_stride, (hipStream_t)stream);
        a.b_expert = w_rows * a.b_stride;
        a.b_across = a.b_stride;
        whole = true;
    }
    a.out_pieces = piece_rows(out, cols);
    GroupPlan plan = group_plan(rows, 0, cols, depth, experts, dtype, false, turned != 0, whole, whole && cols < kPadMost);
    plan.words = dtype == CRESSO_F32 && near_rows(depth, x_stride) && near_rows(w_cols, w_stride);
    with_row_dtype(dtype, [&](auto t) { group_launch<decltype(t)>(a, false, turned != 0, plan, (hipStream_t)stream); });
    return launched(what);
}

extern "C" int32_t cresso_expert_product_weight(const void* p, int64_t p_stride, int64_t p_width, const void* q, int64_t q_stride,
                                                int64_t q_width, int32_t dtype, int64_t rows, int32_t experts, const int32_t* offsets,
                                                void* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "expert product gradient";
    const int32_t rc = check_group(what, dtype, rows, p_width, q_width, experts);
    if (rc != CRESSO_OK) return rc;
    if (experts == 0 || p_width == 0 || q_width == 0) return CRESSO_OK;
    if (!out || !offsets || (rows > 0 && (!p || !q))) return fail(CRESSO_E_INVALID, "%s: null argument", what);
    if (!row_stride_ok(p, rows, p_width, p_stride) || !row_stride_ok(q, rows, q_width, q_stride))
        return fail(CRESSO_E_INVALID, "%s: row strides %lld and %lld below the widths", what, (long long)p_stride, (long long)q_stride);
    if (!workspace || workspace_bytes < cresso_expert_product_weight_workspace_bytes(rows, p_width, q_width, experts, dtype) ||
        ((uintptr_t)workspace & 15))
        return fail(CRESSO_E_INVALID, "%s: workspace of %zu bytes at %p, %zu at a multiple of 16 needed", what, workspace_bytes, workspace,
                    cresso_expert_product_weight_workspace_bytes(rows, p_width, q_width, experts, dtype));
    GroupArgs a{};
    a.a = p;
    a.b = q;
    a.out = out;
    a.offsets = offsets;
    a.rows = rows;
    a.m = p_width;
    a.n = q_width;
    a.a_stride = p_stride;
    a.b_stride = q_stride;
    a.experts = experts;
    a.sums = (float*)workspace;
    a.a_across = p_width;
    a.b_across = q_width;
    bool whole = whole_rows(p, p_width, p_stride, dtype) && whole_rows(q, q_width, q_stride, dtype);
    if (!whole && weight_copies(rows, p_width, q_width, dtype)) {
        __half* const to = (__half*)((char*)workspace + weight_sums(rows, p_width, q_width, experts, dtype));
        a.a_stride = a.a_across = padded(p_width);
        a.b_stride = a.b_across = padded(q_width);
        a.a = to;
        a.b = to + rows * a.a_stride;
        group_pad(p, to, 1, rows, 0, p_width, p_stride, (hipStream_t)stream);
        group_pad(q, (void*)a.b, 1, rows, 0, q_width, q_stride, (hipStream_t)stream);
        whole = true;
    }
    a.out_pieces = piece_rows(out, q_width);
    GroupPlan plan = group_plan(rows, p_width, q_width, 0, experts, dtype, true, true, whole, whole && q_width < kPadMost);
    plan.words = dtype == CRESSO_F32 && near_rows(p_width, p_stride) && near_rows(q_width, q_stride);
    with_row_dtype(dtype, [&](auto t) { group_launch<decltype(t)>(a, true, true, plan, (hipStream_t)stream); });
    return launched(what);
}
