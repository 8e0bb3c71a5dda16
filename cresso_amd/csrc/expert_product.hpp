// Products of rows with the matrix of the expert that they belong to.
//
//   product         out[i][c] = sum over d of x[i][d] * w[e(i)][c][d]        (or w[e(i)][d][c])
//   weight gradient out[e][a][b] = sum over expert e's rows i of p[i][a] * q[i][b]
//
// Both are out(m, n) = sum over k of A(m, k) * B(n, k) in tiles; an operand is
// held along k (its rows are m or n, their elements k) or across it (its rows
// are k, their elements m or n):
//   product          A = x along k, B = w along k or, for the gradient of x and for a weight that is held the
//                    other way round, across k;  one expert's rows are cut into tiles of m
//   weight gradient  A = p, B = q, both across k, which are one expert's rows
//
// A stage of a tile is ROW bytes of k: at 128, 64 numbers of 16 bits or 32 of
// fp32.  The matrix instructions take 16 x 16 x 32 of 16 bits, or 16 x 16 x 4 of
// fp32 four times; a lane's operand is always 16 bytes of k, and which k the
// four quarters of a wave take is the same for both operands, so the order of k
// within a stage is free.  Operands across k are read from LDS transposed.
//
// Few rows are bound by HBM (16 by 16 experts, 2048 -> 5632 bf16: 44.2 us, 5.3 TB/s
// of the matrices that are met), many by the matrix instructions and the power
// that they draw (32768 by 8: 663 to 678 us, 661 to 677 for the gradient of x, 603 to 618
// for the weights', 1.1 to 1.26 PFLOP/s), odd sizes by tiles that are partly empty.
#pragma once

#include "row_ops.hpp"

#include <algorithm>
#include <type_traits>

namespace cresso {

struct GroupArgs {
    const void *a, *b;
    void* out;
    const int32_t* offsets;
    int64_t rows;                          // of all experts
    int64_t m, n, k;                       // product: n columns, k depth; weight gradient: m and n
    int64_t k_along, a_across, b_across;   // what rows hold of k, m and n where they end in zeros of a copy, else k, m and n
    int64_t a_stride, b_stride, b_expert;  // elements
    int32_t experts;
    uint32_t tiles_m, tiles_n;             // product: tiles_m is the most there can be
    uint32_t tiles;                        // workgroups of tiles; those behind them fill rows without an expert
    int32_t out_pieces;   // the result's rows are whole aligned pieces
    // where k is split: parts of it, each with workgroups for all tiles, and their sums [splits][result] in fp32
    uint32_t splits;
    float* sums;
};

constexpr int kFillBlocks = 64;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Group {
    static constexpr int E = 16 / (int)sizeof(T);    // elements of a piece
};

// ---------------------------------------------------------------------------
// LDS.  Pieces of 16 bytes change places by their row's number, so that the
// lanes that read in one cycle find theirs in different banks: 16 lanes at 16
// bytes (0-3, 12-15, 20-23, 24-27 and likewise on), 32 at 8, 64 at 4.
// ---------------------------------------------------------------------------
// Along k, rows of 8 or 4 pieces.  A's fragment (FN 0) has rows l16 of its 16, B's fragment i rows
// 4 FN (l16 / 4) + 4 i + l16 % 4, so that a lane ends with 4 FN consecutive columns.
template <int ROW, int FN> __device__ __forceinline__ int turn_along(int row) {
    constexpr int run = FN > 0 ? 4 * FN : 4;
    const int c = row / run;
    if constexpr (ROW == 128) {
        if constexpr (FN == 0) return ((row >> 1) & 7) ^ (row & 4);
        else return ((row >> 1) & 1) | (c & 1) << 1 | ((c ^ (c >> 1)) & 1) << 2;
    } else {
        return ((c ^ (c >> 1)) & 1) * 2 + ((c >> 1) & 1);
    }
}
// Across k, rows of TILE elements: the blocks of 16 elements change places.
template <typename T, int ROW, int TILE> __device__ __forceinline__ int turn_across(int k) {
    const int far = k >> (ROW == 128 ? 4 : 3);   // what lies in a wave's other quarters
    if constexpr (sizeof(T) == 4) return ROW == 128 ? (TILE >= 64 ? (k >> 3) & 3 : (k >> 3) & 1) : (k >> 2) & 3;
    else if constexpr (TILE >= 128) return (k & 3) | (far & 1) << 2;
    else if constexpr (TILE == 64) return ((k >> 1) & 1) | (far & 1) << 1;
    else return far & 1;
}
// Row (or, across k, k) and piece that lie at a place of a tile's stage.
template <typename T, bool ACROSS, int ROW, int TILE, int FN> __device__ __forceinline__ void at_place(int place, int& row, int& piece) {
    if constexpr (ACROSS) {
        constexpr int E = Group<T>::E, per = TILE / E, block = 16 / E;   // pieces of a row, of a block
        row = place / per;
        const int pos = place % per;
        piece = ((pos / block) ^ turn_across<T, ROW, TILE>(row)) * block + pos % block;
    } else {
        row = place / (ROW / 16);
        piece = (place % (ROW / 16)) ^ turn_along<ROW, FN>(row);
    }
}

// A tile's operand on its way from memory, through registers, to LDS.  It has
// `size` rows along k, or `size` elements a row across it; what is beyond
// those, and beyond k, is 0.
template <typename T, bool ACROSS, int ROW, int TILE, int NT, int FN /* 0: A */> struct Operand {
    static constexpr int E = Group<T>::E, P = TILE * (ROW / 16) / NT;
    static_assert(P * NT == TILE * (ROW / 16), "tile");
    const T* base;
    int64_t stride, size, depth;
    u32x4 held[P];

    __device__ __forceinline__ void load(int64_t k0) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            int row, piece;
            at_place<T, ACROSS, ROW, TILE, FN>((int)threadIdx.x + i * NT, row, piece);
            held[i] = u32x4{0, 0, 0, 0};
            if constexpr (ACROSS) {
                if (k0 + row < depth) held[i] = load_unit(base + (k0 + row) * stride, piece, size);
            } else {
                if (row < size) held[i] = load_unit(base + row * stride, k0 / E + piece, depth);
            }
        }
    }
    __device__ __forceinline__ void store(uint8_t* lds) const {
#pragma unroll
        for (int i = 0; i < P; ++i) *(u32x4*)(lds + ((int)threadIdx.x + i * NT) * 16) = held[i];
    }
};

// V bytes a lane from a buffer to LDS: lane i's go to lds + V * i.  Written out,
// since with the builtin the compiler waits for all of them before each
// transposed read of LDS, whichever part that reads (32768 x 5632 -> 2048, the
// gradient of x: 1341 us, so 841 with the same tiles).  It writes no register but
// m0, a reserved one: the compiler keeps nothing in it, sets it right before what
// reads it, and warns where it is named as clobbered.  group_ready waits for the
// loads.
template <int V> __device__ __forceinline__ void group_to_lds(u32x4 from, uint32_t lane_at, uint32_t at, uint32_t lds) {
    static_assert(V == 16 || V == 4, "bytes of a lane");
    if constexpr (V == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(lds), "v"(lane_at), "s"(from), "s"(at));
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" : : "s"(lds), "v"(lane_at), "s"(from), "s"(at));
}

// The same with the numbers going to LDS by themselves, V bytes a lane: 16 for
// rows, strides and sizes of whole aligned pieces, 4 for fp32 of any.  What lies
// beyond the buffer is 0 in LDS.
template <typename T, bool ACROSS, int ROW, int TILE, int NT, int FN /* 0: A */, int V = 16> struct Stream {
    static constexpr int E = Group<T>::E, P = TILE * (ROW / V) / NT, KS = ROW / (int)sizeof(T);
    static_assert(P * NT == TILE * (ROW / V) && V % (int)sizeof(T) == 0, "tile");
    // Row (or, across k, k) of a thread's i-th load, and its first element there.
    static __device__ __forceinline__ void at_load(int i, int& row, int& element) {
        const int part = (int)threadIdx.x + i * NT;
        at_place<T, ACROSS, ROW, TILE, FN>(part / (16 / V), row, element);
        element = element * E + part % (16 / V) * (V / (int)sizeof(T));
    }
    const T* base;
    int64_t stride, size, depth;
    uint32_t at[P];   // byte of a thread's load in a stage's part of the buffer
    u32x4 buffer;     // the descriptor of make_rsrc of the next stage, in words
    uint32_t step, stage_bytes;
    int left;         // k of the stages that are still to come
    uint32_t wrap;    // along k: where the first of them follows the last
    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            int row, element;
            at_load(i, row, element);
            at[i] = (uint32_t)row * (uint32_t)(stride * (int)sizeof(T)) + (uint32_t)element * (uint32_t)sizeof(T);
        }
        const auto scalar = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
        const uint64_t from = (uint64_t)(uintptr_t)base;
        const uint32_t row_bytes = scalar((uint32_t)(stride * (int)sizeof(T)));
        const uint32_t last = scalar((uint32_t)((ACROSS ? size : depth) * (int64_t)sizeof(T)));
        const uint32_t rows = ACROSS ? (uint32_t)KS : min((uint32_t)TILE, scalar((uint32_t)size));
        buffer = u32x4{scalar((uint32_t)from), scalar((uint32_t)(from >> 32)) & 0xffffu, (rows - 1) * row_bytes + last, 0x00020000u};
        stage_bytes = row_bytes * KS;
        left = (int)scalar((uint32_t)depth);
        step = 0;
        wrap = 0xffffffffu;
        ending();
    }
    // Along k, with whole stages: the first one is `stage`, those before it come last.
    __device__ __forceinline__ void turn(uint32_t stage) {
        step = stage * ROW;
        wrap = (uint32_t)left * (uint32_t)sizeof(T);
    }
    // Before a stage that is not whole, and before those behind the last: what is behind k is 0.
    __device__ __forceinline__ void ending() {
        if (left >= KS) return;
        if (left <= 0) {
            buffer[2] = 0;
        } else if constexpr (ACROSS) {
            buffer[2] -= (uint32_t)(KS - left) * (stage_bytes / KS);
        } else {   // a row's next numbers are another row's
#pragma unroll
            for (int i = 0; i < P; ++i) {
                int row, element;
                at_load(i, row, element);
                if (element >= left) at[i] = 0x80000000u;   // beyond every buffer
            }
        }
    }
    __device__ __forceinline__ void next() {
        left -= KS;
        if constexpr (ACROSS) {
            const uint64_t from = ((uint64_t)buffer[1] << 32 | buffer[0]) + stage_bytes;
            buffer[0] = (uint32_t)from;
            buffer[1] = (uint32_t)(from >> 32);
        } else {
            step += ROW;
            if (step == wrap) step = 0;
        }
        ending();
    }
    // The thread's i-th load to the buffer at `to`, which is the wave's part of it; more: bytes further along k.
    __device__ __forceinline__ void piece(int i, uint32_t to, uint32_t more = 0) const {
        group_to_lds<V>(buffer, at[i], step + more, to + i * (NT * V));
    }
    __device__ __forceinline__ void fetch(uint32_t to) {
#pragma unroll
        for (int i = 0; i < P; ++i) piece(i, to);
        next();
    }
};

// Fragments of a wave: 16 m (or n) from `first` on, for step s of a stage (64 bytes of k each).
template <typename T, bool ACROSS, int ROW, int TILE, int FN /* 0: A */> struct Fragments {
    static constexpr int STEPS = ROW / 64;
    int at[2];   // along: the byte of fragment 0 for each step; across: of the lane's row, and its turn
    __device__ __forceinline__ void begin(int first) {
        const int lane = threadIdx.x & (kWave - 1), l16 = lane & 15, quad = lane >> 4;
        if constexpr (ACROSS) {
            const int k = sizeof(T) == 2 ? quad * (8 * STEPS) + (l16 >> 2) : quad * (4 * STEPS);
            at[0] = k * (TILE * (int)sizeof(T)) + (sizeof(T) == 2 ? (l16 & 3) * 8 : l16 * 4);
            at[1] = turn_across<T, ROW, TILE>(k) ^ (first / 16);
        } else {
            const int row = first + (FN > 0 ? (l16 >> 2) * (4 * FN) + (l16 & 3) : l16);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) at[s] = row * ROW + ((quad * STEPS + s) ^ turn_along<ROW, FN>(row)) * 16;
        }
    }
    __device__ __forceinline__ u32x4 read(const uint8_t* lds, int s, int i) const {
        if constexpr (!ACROSS) {
            return *(const u32x4*)(lds + at[s] + i * (FN > 0 ? 4 * ROW : 16 * ROW));
        } else {
            constexpr int R = TILE * (int)sizeof(T);   // bytes of a row
            const uint8_t* from = lds + at[0] + ((at[1] ^ i) * (16 * (int)sizeof(T)));
            if constexpr (sizeof(T) == 2) {
                // 16 lanes give four rows of 16 numbers and get a column of four each
                typedef __attribute__((address_space(3))) i16x4* Lds;
                const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from + s * 8 * R));
                const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from + (s * 8 + 4) * R));
                const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
                return u32x4{l[0], l[1], h[0], h[1]};
            } else {
                u32x4 r;
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = *(const uint32_t*)(from + (s * 4 + j) * R);
                return r;
            }
        }
    }
};

template <typename T> __device__ __forceinline__ f32x4 group_mfma(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 group_mfma<__hip_bfloat16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 group_mfma<__half>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 group_mfma<float>(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t x = a[j], y = b[j];
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y), c, 0, 0, 0);
    }
    return c;
}

// The same with the sum held in one place: with the builtin the compiler moves
// 256 registers of sums about, since a result may lie elsewhere than what it is
// added to.  Who reads a sum by anything but these waits with group_mfma_done;
// the matrix instructions wait for one another where they name the same registers.
template <typename T> __device__ __forceinline__ void group_mfma_into(u32x4 a, u32x4 b, f32x4& c) {
    static_assert(sizeof(T) == 2, "16 bits");
    if constexpr (std::is_same<T, __half>::value) asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// Sums of zero, in their registers here and now: a zero that the compiler writes
// right in front of a matrix instruction, as it does with one that is only
// assigned, is not there yet when that reads it.
template <int N> __device__ __forceinline__ void group_zero(f32x4 (&c)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        c[i] = f32x4{0, 0, 0, 0};
        asm volatile("" : "+a"(c[i]));
    }
}
// After the last of them: more than the 18 cycles that a result of four passes takes to be there for others.
template <int N> __device__ __forceinline__ void group_mfma_done(f32x4 (&c)[N]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+a"(c[i]));   // read behind the wait
}

// ---------------------------------------------------------------------------
// the tiles of ragged groups
// ---------------------------------------------------------------------------
// Rows [first, end) of expert e.  Offsets that point outside the rows, or fall, are held within them.
__device__ __forceinline__ void group_rows(const GroupArgs& a, int e, int64_t& first, int64_t& end) {
    first = min(max((int64_t)a.offsets[e], (int64_t)0), a.rows);
    end = min(max((int64_t)a.offsets[e + 1], first), a.rows);
}
// Sums over the lanes up to each, by row operations of the vector unit.
template <int CTRL, int ROW_MASK> __device__ __forceinline__ uint32_t group_add(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xF, false);
}
__device__ __forceinline__ uint32_t group_upto(uint32_t v) {
    v = group_add<0x111, 0xF>(v);   // row_shr:1
    v = group_add<0x112, 0xF>(v);   // row_shr:2
    v = group_add<0x114, 0xF>(v);   // row_shr:4
    v = group_add<0x118, 0xF>(v);   // row_shr:8
    v = group_add<0x142, 0xA>(v);   // row_bcast:15 -> rows 1, 3
    return group_add<0x143, 0xC>(v);   // row_bcast:31 -> rows 2, 3
}
// The tiles of m rows of all experts, 64 experts at a time, one a lane.  By each wave.
struct GroupTiles {
    int first, end;         // the lane's expert's rows, below 2^31
    uint32_t count, upto;   // its tiles, and those of the experts up to it from `expert` on
    int expert;             // of lane 0
    uint32_t before, all;   // tiles of the experts before that one; of all experts
    __device__ __forceinline__ void load(const GroupArgs& a, int tile, int e0) {
        const int lane = threadIdx.x & (kWave - 1);
        expert = e0;
        int64_t from = 0, to = 0;
        if (e0 + lane < a.experts) group_rows(a, e0 + lane, from, to);
        first = (int)from;
        end = (int)to;
        count = ((uint32_t)(end - first) + (uint32_t)tile - 1) / (uint32_t)tile;
        upto = group_upto(count);
    }
    __device__ __forceinline__ uint32_t here() const { return (uint32_t)__builtin_amdgcn_readlane((int)upto, kWave - 1); }
    __device__ __forceinline__ void begin(const GroupArgs& a, int tile) {
        const uint32_t most = (uint32_t)(a.rows / tile) + (uint32_t)a.experts;   // more only where offsets fall
        all = 0;
        for (int e0 = (a.experts - 1) / kWave * kWave; e0 >= 0; e0 -= kWave) {
            load(a, tile, e0);
            all = min(all + here(), most);   // below 2^26 + 2^31
        }
        before = 0;
    }
    // Tile t of all: its expert and rows.
    __device__ __forceinline__ void find(const GroupArgs& a, int tile, uint32_t t, int& e, int64_t& from, int64_t& to) const {
        GroupTiles g = *this;
        while (g.before + g.here() <= t && g.expert + kWave < a.experts) {
            g.before += g.here();
            g.load(a, tile, g.expert + kWave);
        }
        const uint64_t past = __ballot(g.before + g.upto > t);
        const int l = past ? __builtin_ctzll(past) : 0;
        const uint32_t ahead = g.before + (uint32_t)__builtin_amdgcn_readlane((int)(g.upto - g.count), l);
        e = g.expert + l;
        from = __builtin_amdgcn_readlane(g.first, l) + (int64_t)(t - ahead) * tile;
        to = min((int64_t)__builtin_amdgcn_readlane(g.end, l), from + tile);
    }
};

// Which of `total` tiles a workgroup takes.  Workgroups go to the 8 XCDs in
// turn; each XCD takes a run of tiles.  total or more: none.
__device__ __forceinline__ uint32_t group_run(uint32_t block, uint32_t total) {
    const uint32_t per = total / 8, rest = total % 8, xcd = block % 8, i = block / 8;
    return i < per + (xcd < rest ? 1u : 0u) ? xcd * per + min(xcd, rest) + i : total;
}
// Tile t among `high` x `wide`, in columns of 8 tiles of m, so that the tiles that run together on one XCD share rows of
// both operands in its L2.
__device__ __forceinline__ void group_place(uint32_t t, uint32_t high, uint32_t wide, uint32_t& tm, uint32_t& tn) {
    const uint32_t group = 8 * wide, g = t / group, in = t - g * group;
    const uint32_t height = min(8u, high - g * 8);
    tm = g * 8 + in % height;
    tn = in / height;
}

// The expert whose rows are the i-th most (of the first 64, in their order behind those): a weight
// gradient's tiles take as long as their expert's rows are many, so the longest begin.
__device__ __forceinline__ int group_longest(const GroupArgs& a, uint32_t i) {
    if (i >= (uint32_t)kWave) return (int)i;
    const int lane = threadIdx.x & (kWave - 1), n = min(a.experts, kWave);
    int64_t first = 0, end = -1;
    if (lane < n) group_rows(a, lane, first, end);
    const int mine = (int)(end - first);
    uint32_t before = 0;
    for (int e = 0; e < n; ++e) {
        const int other = __builtin_amdgcn_readlane(mine, e);
        before += other > mine || (other == mine && e < lane) ? 1u : 0u;
    }
    return __builtin_ctzll(__ballot(lane < n && before == i));
}

// Zeros into the rows that are no expert's.
template <typename T> __device__ __forceinline__ void group_fill(const GroupArgs& a, int64_t part, int64_t parts) {
    const int64_t begin = min(max((int64_t)a.offsets[0], (int64_t)0), a.rows);
    const int64_t end = min(max((int64_t)a.offsets[a.experts], begin), a.rows);
    const int64_t units = (a.n + Group<T>::E - 1) / Group<T>::E;
    for (int64_t r = part; r < begin + a.rows - end; r += parts) {
        const int64_t row = r < begin ? r : r - begin + end;
        for (int64_t u = threadIdx.x; u < units; u += blockDim.x) store_unit((T*)a.out + row * a.n, u, a.n, u32x4{0, 0, 0, 0});
    }
}

// A tile of TM x TN or, from row m0 and column n0 of it on, a part of one: one
// expert's rows of A and of the result (product), or all its rows as k (weight gradient).
struct GroupWork {
    int expert;
    int64_t first, end;   // rows: of the tile, or of the expert
    int64_t m0, n0;
};
// Tile t of all; high and wide: tiles of m, over all experts (product) or one (weight gradient), and of n.
template <bool WEIGHT>
__device__ __forceinline__ GroupWork group_work(const GroupArgs& a, const GroupTiles& tiles, uint32_t t, uint32_t high, uint32_t wide, int TM, int TN) {
    GroupWork w;
    uint32_t tm, tn;
    if constexpr (WEIGHT) {   // each expert's tiles over all XCDs
        const uint32_t per = high * wide;
        w.expert = group_longest(a, t / per);
        group_place(group_run(t % per, per), high, wide, tm, tn);
        group_rows(a, w.expert, w.first, w.end);
        w.first = __builtin_amdgcn_readfirstlane((int)w.first);   // below 2^31, and the same for all lanes
        w.end = __builtin_amdgcn_readfirstlane((int)w.end);
        w.m0 = (int64_t)tm * TM;
    } else {
        group_place(t, high, wide, tm, tn);
        tiles.find(a, TM, tm, w.expert, w.first, w.end);
        w.m0 = 0;
    }
    w.n0 = (int64_t)tn * TN;
    return w;
}
// The operands of a tile's part that begins at m0, n0, and its result's rows from `out` on.
template <typename T, bool WEIGHT, bool ACROSS, typename A, typename B>
__device__ __forceinline__ void group_operands(const GroupArgs& a, const GroupWork& w, A& oa, B& ob, T*& out, int64_t& rows) {
    if constexpr (WEIGHT) {
        oa.base = (const T*)a.a + w.first * a.a_stride + w.m0;
        ob.base = (const T*)a.b + w.first * a.b_stride + w.n0;
        oa.size = a.a_across - w.m0;
        oa.depth = ob.depth = w.end - w.first;
        out = (T*)a.out + (int64_t)w.expert * a.m * a.n;
        rows = a.m;
    } else {
        oa.base = (const T*)a.a + (w.first + w.m0) * a.a_stride;
        ob.base = (const T*)a.b + w.expert * a.b_expert + (ACROSS ? w.n0 : w.n0 * a.b_stride);
        oa.size = w.end - w.first - w.m0;
        oa.depth = a.k_along;
        ob.depth = ACROSS ? a.k : a.k_along;
        out = (T*)a.out + w.first * a.n;
        rows = w.end - w.first;
    }
    ob.size = (ACROSS ? a.b_across : a.n) - w.n0;
    oa.stride = a.a_stride;
    ob.stride = a.b_stride;
}
// What a workgroup of a kernel with one size of tiles does.  false: nothing.
template <bool WEIGHT> __device__ __forceinline__ bool group_begin(const GroupArgs& a, int TM, int TN, GroupWork& w) {
    GroupTiles tiles;
    if (!WEIGHT) tiles.begin(a, TM);
    const uint32_t high = WEIGHT ? a.tiles_m : tiles.all, total = high * a.tiles_n, block = blockIdx.x % a.tiles;
    const uint32_t t = WEIGHT ? block : group_run(block, total);
    if (!WEIGHT && t >= total) return false;
    w = group_work<WEIGHT>(a, tiles, t, high, a.tiles_n, TM, TN);
    return true;
}
// The workgroup's part of k, where it is split: whole stages of KS.
template <bool WEIGHT, bool ACROSS, int KS, typename A, typename B> __device__ __forceinline__ void group_part(const GroupArgs& a, A& oa, B& ob) {
    if (a.splits < 2) return;
    const int64_t part = blockIdx.x / a.tiles, stages = (oa.depth + KS - 1) / KS;
    const int64_t k0 = stages * part / a.splits * KS, k1 = min(stages * (part + 1) / a.splits * KS, oa.depth);
    oa.base += WEIGHT ? k0 * oa.stride : k0;
    ob.base += ACROSS ? k0 * ob.stride : k0;
    oa.depth = max(k1 - k0, (int64_t)0);
    ob.depth = max(min(ob.depth, k1) - k0, (int64_t)0);
}
// A lane holds columns 4 quad to 4 quad + 3 of each fragment's 16, or with B
// along k 4 FN columns in one piece, of rows l16 of each of FM fragments from m on.
template <typename T, bool ACROSS, int FM, int FN>
__device__ __forceinline__ void group_store(const GroupArgs& a, T* out, int64_t rows, int64_t m0, int64_t n0, const f32x4 (&acc)[FN][FM]) {
    constexpr int E = Group<T>::E;
    const int lane = threadIdx.x & (kWave - 1), l16 = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t m = m0 + j * 16 + l16;
        if (m >= rows) continue;
        T* to = out + m * a.n;
        if constexpr (ACROSS || 4 * FN < E) {
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const int64_t n = n0 + (ACROSS ? i * 16 + quad * 4 : quad * (4 * FN) + i * 4);
                const f32x4 v = acc[i][j];
                if constexpr (sizeof(T) == 4) {
                    store_unit(to + n, 0, a.n - n, __builtin_bit_cast(u32x4, v));
                } else {
                    const uint32_t lo = narrow2<T>(v[0], v[1]), hi = narrow2<T>(v[2], v[3]);
                    if (n + 4 <= a.n) store8(to + n, u32x2{lo, hi});
                    else if (n < a.n) store_part(to + n, u32x4{lo, hi, 0, 0}, (int)(a.n - n));
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4 * FN / E; ++u) {
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = acc[(u * E + e) / 4][j][(u * E + e) % 4];
                store_unit(to, (n0 + quad * (4 * FN)) / E + u, a.n, narrow<T>(v));
            }
        }
    }
}

template <typename T, bool WEIGHT, bool ACROSS, int FM, int FN>
__device__ __forceinline__ void group_result(const GroupArgs& a, T* out, int64_t rows, int64_t m0, int64_t n0, const f32x4 (&acc)[FN][FM]) {
    if (a.splits < 2) return group_store<T, ACROSS, FM, FN>(a, out, rows, m0, n0, acc);
    const int64_t all = (WEIGHT ? (int64_t)a.experts * a.m : a.rows) * a.n;
    group_store<float, ACROSS, FM, FN>(a, a.sums + (blockIdx.x / a.tiles) * all + (out - (T*)a.out), rows, m0, n0, acc);
}
// The parts' sums, in their order; rows that are no expert's are zeros.  A unit of the result a thread.
template <typename T, bool WEIGHT> __global__ __launch_bounds__(256) void group_join_kernel(GroupArgs a) {
    constexpr int E = Unit<T>::n;
    const int64_t all = (WEIGHT ? (int64_t)a.experts * a.m : a.rows) * a.n;
    int64_t begin = 0, end = all;
    if constexpr (!WEIGHT) {
        begin = min(max((int64_t)a.offsets[0], (int64_t)0), a.rows) * a.n;
        end = min(max((int64_t)a.offsets[a.experts], (int64_t)0), a.rows) * a.n;
    }
    const int64_t units = (all + E - 1) / E;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (int64_t)gridDim.x * 256) {
        float sum[E] = {};
        for (uint32_t p = 0; p < a.splits; ++p) {
            const float* from = a.sums + p * all;
#pragma unroll
            for (int i = 0; i < E / 4; ++i) {
                const f32x4 v = __builtin_bit_cast(f32x4, load_unit(from, u * (E / 4) + i, all));
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[4 * i + e] += v[e];
            }
        }
        if constexpr (!WEIGHT) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (u * E + e < begin || u * E + e >= end) sum[e] = 0.0f;
        }
        store_unit((T*)a.out, u, all, narrow<T>(sum));
    }
}

// WM x WN waves of FM x FN fragments of 16 x 16 each; operands of any alignment, through registers, for
// rows that do not go to LDS by themselves: 16 bits at odd strides or addresses that are not laid out anew, fp32
// rows far apart.
template <typename T, bool WEIGHT, bool B_ACROSS, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM* WN * 64, 2) void group_any_kernel(GroupArgs a) {
    constexpr int NT = WM * WN * 64, TM = WM * FM * 16, TN = WN * FN * 16, ROW = 128;
    constexpr int KS = ROW / (int)sizeof(T), STAGE = (TM + TN) * ROW;
    constexpr bool ACROSS = WEIGHT || B_ACROSS;   // B
    __shared__ __align__(16) uint8_t lds[2 * STAGE];
    if (blockIdx.x >= a.tiles * a.splits) {
        group_fill<T>(a, blockIdx.x - a.tiles, gridDim.x - a.tiles);
        return;
    }
    Operand<T, WEIGHT, ROW, TM, NT, 0> oa;
    Operand<T, ACROSS, ROW, TN, NT, FN> ob;
    GroupWork w;
    if (!group_begin<WEIGHT>(a, TM, TN, w)) return;
    T* out;
    int64_t rows;
    group_operands<T, WEIGHT, ACROSS>(a, w, oa, ob, out, rows);
    group_part<WEIGHT, ACROSS, KS>(a, oa, ob);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = (wave % WM) * (FM * 16), wn = (wave / WM) * (FN * 16);
    Fragments<T, WEIGHT, ROW, TM, 0> fa;
    Fragments<T, ACROSS, ROW, TN, FN> fb;
    fa.begin(wm);
    fb.begin(wn);
    f32x4 acc[FN][FM] = {};
    const int64_t stages = (oa.depth + KS - 1) / KS;
    if (stages) {
        oa.load(0);
        ob.load(0);
        oa.store(lds);
        ob.store(lds + TM * ROW);
    }
    for (int64_t s = 0; s < stages; ++s) {
        uint8_t* const now = lds + (s & 1) * STAGE;
        uint8_t* const next = lds + (~s & 1) * STAGE;
        __syncthreads();   // this stage is there, and the one before it has been read
        if (s + 1 < stages) {
            oa.load((s + 1) * KS);
            ob.load((s + 1) * KS);
        }
#pragma unroll
        for (int h = 0; h < ROW / 64; ++h) {
            u32x4 b[FN];
#pragma unroll
            for (int i = 0; i < FN; ++i) b[i] = fb.read(now + TM * ROW, h, i);
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const u32x4 v = fa.read(now, h, j);
#pragma unroll
                for (int i = 0; i < FN; ++i) acc[i][j] = group_mfma<T>(b[i], v, acc[i][j]);
            }
        }
        if (s + 1 < stages) {
            oa.store(next);
            ob.store(next + TM * ROW);
        }
    }
    group_result<T, WEIGHT, ACROSS, FM, FN>(a, out, rows, w.m0 + wm, w.n0 + wn, acc);
}

// Waits until at most N of the wave's loads are on their way and all its LDS
// reads have ended (the stage they read is filled anew), then for the other waves.
template <int N> __device__ __forceinline__ void group_ready() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Both operands along k in whole stages: each of an expert's columns of tiles
// begins with another stage, in an order of its own, but the same on every run.
// Rows whose strides are powers of two begin in the same memory channels, and
// tiles that begin together would all ask the same ones for their first numbers,
// and so on (16 rows x 2048 -> 5632 by 16, weights from memory: 52.6 us so, 47.5 turned;
// 2000 x 2048 -> 1024 by 32 40.0 and 37.2; the large tiles gain nothing).
template <int KS, typename A, typename B> __device__ __forceinline__ void group_turn(const GroupWork& w, int TN, A& oa, B& ob) {
    const uint32_t stages = (uint32_t)oa.left / KS;
    if (stages == 0 || (uint32_t)oa.left % KS) return;
    const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(w.n0 / TN) * 2 + (uint32_t)w.expert * 3)) % stages;
    oa.turn(first);
    ob.turn(first);
}

// The same for operands that go to LDS by themselves, STAGES - 1 stages ahead of
// the one that is multiplied: V = 16 for whole aligned pieces, 4 for fp32 of any
// alignment (777 x 1001 -> 1500 by 9 in tiles of 64 x 64 41.8 us, through registers 54.9).
template <typename T, bool WEIGHT, bool B_ACROSS, int WM, int WN, int FM, int FN, int ROW, int STAGES, int V = 16>
__global__ __launch_bounds__(WM* WN * 64, 2) void group_kernel(GroupArgs a) {
    constexpr int NT = WM * WN * 64, TM = WM * FM * 16, TN = WN * FN * 16;
    constexpr int KS = ROW / (int)sizeof(T), STAGE = (TM + TN) * ROW;
    constexpr bool ACROSS = WEIGHT || B_ACROSS;   // B
    __shared__ __align__(16) uint8_t lds[STAGES * STAGE];
    if (blockIdx.x >= a.tiles * a.splits) {
        group_fill<T>(a, blockIdx.x - a.tiles, gridDim.x - a.tiles);
        return;
    }
    typedef Stream<T, WEIGHT, ROW, TM, NT, 0, V> StreamA;
    typedef Stream<T, ACROSS, ROW, TN, NT, FN, V> StreamB;
    constexpr int LOADS = StreamA::P + StreamB::P;
    StreamA oa;
    StreamB ob;
    GroupWork w;
    if (!group_begin<WEIGHT>(a, TM, TN, w)) return;
    T* out;
    int64_t rows;
    group_operands<T, WEIGHT, ACROSS>(a, w, oa, ob, out, rows);
    group_part<WEIGHT, ACROSS, KS>(a, oa, ob);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = (wave % WM) * (FM * 16), wn = (wave / WM) * (FN * 16);
    Fragments<T, WEIGHT, ROW, TM, 0> fa;
    Fragments<T, ACROSS, ROW, TN, FN> fb;
    fa.begin(wm);
    fb.begin(wn);
    oa.begin();
    ob.begin();
    if constexpr (!ACROSS) group_turn<KS>(w, TN, oa, ob);
    f32x4 acc[FN][FM] = {};
    const int stages = (int)((oa.depth + KS - 1) / KS);
    const uint32_t mine = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + (uint32_t)wave * (kWave * V);
    uint32_t to = 0;
    const auto fetch = [&] {
        oa.fetch(mine + to);
        ob.fetch(mine + to + TM * ROW);
        to = to == (STAGES - 1) * STAGE ? 0 : to + STAGE;
    };
    if (stages) {
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) fetch();
    }
    int from = 0;
    for (int s = 0; s < stages; ++s) {
        group_ready<(STAGES - 2) * LOADS>();
        fetch();
        const uint8_t* const now = lds + from;
#pragma unroll
        for (int h = 0; h < ROW / 64; ++h) {
            u32x4 b[FN];
#pragma unroll
            for (int i = 0; i < FN; ++i) b[i] = fb.read(now + TM * ROW, h, i);
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const u32x4 v = fa.read(now, h, j);
#pragma unroll
                for (int i = 0; i < FN; ++i) acc[i][j] = group_mfma<T>(b[i], v, acc[i][j]);
            }
        }
        from = from == (STAGES - 1) * STAGE ? 0 : from + STAGE;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing is on its way to LDS when the workgroup ends
    group_result<T, WEIGHT, ACROSS, FM, FN>(a, out, rows, w.m0 + wm, w.n0 + wn, acc);
}

// A tile of 32 FM x 32 FN of 16 bits by four waves of 16 FM x 16 FN, one to a
// SIMD.  A stage's fragments are read while the one before is multiplied, and
// the pieces of the stage STAGES further on are asked for in between.
template <typename T, bool WEIGHT, bool ACROSS, int FM, int FN, int STAGES>
__device__ __forceinline__ void group_large_tile(const GroupArgs& a, const GroupWork& w, uint8_t* const lds) {
    constexpr int NT = 256, TM = 32 * FM, TN = 32 * FN, ROW = 64;
    constexpr int KS = ROW / (int)sizeof(T), STAGE = (TM + TN) * ROW;
    static_assert(STAGES * STAGE >= TM * TN * (int)sizeof(T), "the result goes through the stages' memory");
    typedef Stream<T, WEIGHT, ROW, TM, NT, 0> StreamA;
    typedef Stream<T, ACROSS, ROW, TN, NT, FN> StreamB;
    constexpr int PA = StreamA::P, LOADS = PA + StreamB::P, STEPS = FM * FN;
    StreamA oa;
    StreamB ob;
    T* out;
    int64_t rows;
    group_operands<T, WEIGHT, ACROSS>(a, w, oa, ob, out, rows);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = (wave & 1) * (16 * FM), wn = (wave >> 1) * (16 * FN);
    Fragments<T, WEIGHT, ROW, TM, 0> fa;
    Fragments<T, ACROSS, ROW, TN, FN> fb;
    fa.begin(wm);
    fb.begin(wn);
    oa.begin();
    ob.begin();
    f32x4 acc[FM][FN];
#pragma unroll
    for (int j = 0; j < FM; ++j) group_zero(acc[j]);
    const int stages = (int)((oa.depth + KS - 1) / KS);
    const uint32_t mine = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + (uint32_t)wave * 1024;
    u32x4 ra[2][FM], rb[2][FN];
    const auto piece = [&](int i, int buffer) {
        if (i < PA) oa.piece(i, mine + buffer * STAGE);
        else if (i < LOADS) ob.piece(i - PA, mine + buffer * STAGE + TM * ROW);
    };
    // Multiplies the stage in buffer `now`, whose fragments are in set `set`; reads
    // the next one's into the other, early enough to be there when the stage ends,
    // and fills `now` anew.  A wave issues one instruction in 4 cycles and a matrix
    // instruction takes 16, so each of them is followed by at most three others.
    const auto stage = [&](int now, int set) {
        group_ready<(STAGES - 2) * LOADS>();
        const uint8_t* const then = lds + (now + 1) % STAGES * STAGE;
        constexpr int EVERY = STEPS * 3 / 4 / (FM + FN) > 0 ? STEPS * 3 / 4 / (FM + FN) : 1, APART = STEPS / LOADS;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            group_mfma_into<T>(rb[set][t % FN], ra[set][t / FN], acc[t / FN][t % FN]);
            const int r = t / EVERY;
            if (t % EVERY == 0 && r < FN) rb[set ^ 1][r] = fb.read(then + TM * ROW, 0, r);
            else if (t % EVERY == 0 && r < FM + FN) ra[set ^ 1][r - FN] = fa.read(then, 0, r - FN);
            if (t % APART == 1) piece(t / APART, now);
            __builtin_amdgcn_sched_barrier(0);
        }
        oa.next();
        ob.next();
    };
    if (stages) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
            oa.fetch(mine + i * STAGE);
            ob.fetch(mine + i * STAGE + TM * ROW);
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < FN; ++i) rb[0][i] = fb.read(lds + TM * ROW, 0, i);
#pragma unroll
        for (int j = 0; j < FM; ++j) ra[0][j] = fa.read(lds, 0, j);
        constexpr int ROUND = STAGES % 2 ? 2 * STAGES : STAGES;
        for (int s = 0; s < stages; s += ROUND) {
#pragma unroll
            for (int i = 0; i < ROUND; ++i) {
                if (s + i >= stages) break;
                stage(i % STAGES, i & 1);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing is on its way to LDS when it is used otherwise
#pragma unroll
    for (int j = 0; j < FM; ++j) group_mfma_done(acc[j]);
    // The result through LDS, so that a wave stores long pieces of rows: a lane
    // writes 4 numbers of a fragment, or 4 FN in a row, and reads 16 bytes of a row.
    // Pieces change places by the row's number.
    __syncthreads();
    const int lane = threadIdx.x & (kWave - 1), l16 = lane & 15, quad = lane >> 4;
    const auto place = [](int row, int piece) { return row * (TN * 2) + ((piece ^ (row & (TN / 8 < 16 ? TN / 8 - 1 : 15))) * 16); };
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int row = wm + j * 16 + l16;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const int n = wn + (ACROSS ? i * 16 + quad * 4 : quad * (4 * FN) + i * 4);
            *(u32x2*)(lds + place(row, n / 8) + (n & 4) * 2) = u32x2{narrow2<T>(acc[j][i][0], acc[j][i][1]), narrow2<T>(acc[j][i][2], acc[j][i][3])};
        }
    }
    __syncthreads();
    constexpr int PER = TN / 8;   // pieces of a row
    const int64_t high = min((int64_t)TM, rows - w.m0), at = (int)threadIdx.x % PER, n = w.n0 + at * 8;
    T* const to = out + w.m0 * a.n + n;
#pragma unroll 4
    for (int r = (int)threadIdx.x / PER; r < high; r += NT / PER) {
        const u32x4 v = *(const u32x4*)(lds + place(r, at));
        if (n + 8 <= a.n) store16(to + (int64_t)r * a.n, v);
        else if (n < a.n) store_part(to + (int64_t)r * a.n, v, (int)(a.n - n));
    }
}

// 256 x 256 of 16 bits, one workgroup to a CU, bound by power and the matrix unit
// (busy 65 to 73 % of the cycles at a clock that falls to 1.8 GHz): eight waves of
// 128 x 64 would read 96 KB of LDS a stage, as long as their matrix instructions
// take; four of 128 x 128 read 64.  A workgroup goes from tile to tile, and asks
// for the next one's first stages before it stores the one that it has done.
// What is left behind the last full round of 256 tiles goes in quarters of 128 x
// 128, if those take less than a round.
//
// A stage along k is 64 bytes of each row, half a line of the caches, and by the
// time of the other half the line has left the first of them: the second one
// is asked twice for each.  With PAIRS, for two operands along k in whole pairs of
// stages, both halves are asked for together, A's in even stages and B's in odd
// ones; they wait in five stages' memory, of which one holds the result while
// the next tile's first four arrive (32768 x 2048 -> 5632 by 8: 697 us, so 663).
// Where B lies across k it gains nothing (672 and 677), where both do it loses (605 and 633).
constexpr uint32_t kRound = 256;
template <typename T, bool WEIGHT, bool B_ACROSS, bool PAIRS> __global__ __launch_bounds__(256, 1) void group_large_kernel(GroupArgs a) {
    constexpr bool ACROSS = WEIGHT || B_ACROSS;   // B
    constexpr int NT = 256, F = 8, TILE = 32 * F, ROW = 64, STAGES = 4;   // ahead
    constexpr int KS = ROW / (int)sizeof(T), STAGE = 2 * TILE * ROW, OWN = 32 * 16 * F * (int)sizeof(T);   // of a wave: 32 of its rows
    static_assert(4 * OWN == STAGE && !(PAIRS && ACROSS), "a stage's memory holds 32 rows of each wave's result");
    __shared__ __align__(16) uint8_t lds[(STAGES + 1) * STAGE];
    if (blockIdx.x >= kRound) {
        group_fill<T>(a, blockIdx.x - kRound, gridDim.x - kRound);
        return;
    }
    GroupTiles tiles;
    if (!WEIGHT) tiles.begin(a, TILE);
    const uint32_t high = WEIGHT ? a.tiles_m : tiles.all, total = high * a.tiles_n * (WEIGHT ? (uint32_t)a.experts : 1u);
    uint32_t rest = total % kRound;
    if (rest > kRound / 2) rest = 0;
    const uint32_t full = total - rest;
    typedef Stream<T, WEIGHT, ROW, TILE, NT, 0> StreamA;
    typedef Stream<T, ACROSS, ROW, TILE, NT, F> StreamB;
    constexpr int PA = StreamA::P, LOADS = PA + StreamB::P, STEPS = F * F;
    const int lane = threadIdx.x & (kWave - 1), l16 = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = (wave & 1) * (16 * F), wn = (wave >> 1) * (16 * F);
    uint32_t cur = 0;   // PAIRS: where the stage lies that is multiplied, among five
    const auto before = [](uint32_t at) { return at == 0 ? STAGES * STAGE : at - STAGE; };
    const auto behind = [](uint32_t at) { return at == STAGES * STAGE ? 0 : at + STAGE; };
    const uint32_t mine = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + (uint32_t)wave * 1024;
    Fragments<T, WEIGHT, ROW, TILE, 0> fa;
    Fragments<T, ACROSS, ROW, TILE, F> fb;
    fa.begin(wm);
    fb.begin(wn);
    f32x4 acc[F][F];
#pragma unroll
    for (int j = 0; j < F; ++j) group_zero(acc[j]);
    StreamA oa;
    StreamB ob;
    T* out = nullptr;
    int64_t rows = 0, m0 = 0, n0 = 0;
    int stages = 0;
    const auto begin = [&](uint32_t u) __attribute__((always_inline)) {   // tile u: where it lies, and its first stages on their way
        // weight gradients' tiles fall in length: who had an early one in a round takes a late one in the next
        const uint32_t in = u % kRound, round = u - in;   // the last round may be short
        const uint32_t at = !WEIGHT ? group_run(u, full) : u / kRound % 2 && round + kRound <= full ? round + kRound - 1 - in : u;
        const GroupWork w = group_work<WEIGHT>(a, tiles, at, high, a.tiles_n, TILE, TILE);
        group_operands<T, WEIGHT, ACROSS>(a, w, oa, ob, out, rows);
        m0 = w.m0;
        n0 = w.n0;
        stages = (int)((oa.depth + KS - 1) / KS);
        oa.begin();
        ob.begin();
        uint32_t to = cur;
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
            oa.fetch(mine + (PAIRS ? to : i * STAGE));
            ob.fetch(mine + (PAIRS ? to : i * STAGE) + TILE * ROW);
            to = behind(to);
        }
    };
    u32x4 ra[2][F], rb[2][F];
    // Multiplies stage `now`, counted from one of the first to the last buffer (PAIRS:
    // even or odd), whose fragments are in set now % 2; reads the next one's into
    // the other, early enough to be there when the stage ends, and fills `now` anew
    // (PAIRS: A's parts of the buffers of this stage and the one before, or B's of
    // the two before).  A wave issues one instruction in 4 cycles and a matrix
    // instruction takes 16, so each of them is followed by at most three others.
    // wait: loads and stores that came after the pieces of the next stage.
    const auto stage = [&](auto now, auto wait) __attribute__((always_inline)) {
        constexpr int N = decltype(now)::value, set = N & 1;
        group_ready<decltype(wait)::value>();
        const uint32_t next = PAIRS ? behind(cur) : (N + 1) % STAGES * STAGE;
        const uint32_t one = PAIRS ? (set == 0 ? before(cur) : before(before(cur))) : N * STAGE, other = set == 0 ? cur : before(cur);
        const uint8_t* const then = lds + next;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            group_mfma_into<T>(rb[set][t % F], ra[set][t / F], acc[t / F][t % F]);
            const int r = t / 3;
            if (t % 3 == 0 && r < F) rb[set ^ 1][r] = fb.read(then + TILE * ROW, 0, r);
            else if (t % 3 == 0 && r < 2 * F) ra[set ^ 1][r - F] = fa.read(then, 0, r - F);
            if (t % 8 == 1) {
                const int i = t / 8, half = i % 2;
                if (!PAIRS && i < PA) oa.piece(i, mine + one);
                else if (!PAIRS) ob.piece(i - PA, mine + one + TILE * ROW);
                else if (set == 0) oa.piece(i / 2, mine + (half ? other : one), half * ROW);
                else ob.piece(i / 2, mine + (half ? other : one) + TILE * ROW, half * ROW);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (!PAIRS || set == 0) oa.next();
        if (!PAIRS || set == 1) ob.next();
        if (PAIRS && set == 0) oa.next();
        if (PAIRS && set == 1) ob.next();
        cur = next;
    };
    constexpr std::integral_constant<int, 4 * F> STORES{};
    constexpr std::integral_constant<int, 0> NONE{}, S0{};
    constexpr std::integral_constant<int, 1> S1{};
    constexpr std::integral_constant<int, 2> S2{};
    constexpr std::integral_constant<int, 3> S3{};
    constexpr std::integral_constant<int, 2 * LOADS> TWO{};             // two stages' loads, or a pair's of A and of B
    constexpr std::integral_constant<int, (PAIRS ? 1 : 2) * LOADS> LAST{};   // before odd stages: a pair's of A
    const auto first = [&](auto later) __attribute__((always_inline)) {   // later: stores that came after the first stages' pieces
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS + decltype(later)::value) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint8_t* const from = lds + (PAIRS ? cur : 0);
#pragma unroll
        for (int i = 0; i < F; ++i) rb[0][i] = fb.read(from + TILE * ROW, 0, i);
#pragma unroll
        for (int j = 0; j < F; ++j) ra[0][j] = fa.read(from, 0, j);
        constexpr std::integral_constant<int, 2 * LOADS + decltype(later)::value> BOTH{};
        stage(S0, BOTH);
        stage(S1, BOTH);
        stage(S2, BOTH);
        stage(S3, LAST);
    };
    uint32_t u = blockIdx.x;
    if (u < full) {
        begin(u);
        first(NONE);
    }
    while (u < full) {
        for (int s = STAGES; s < stages; s += PAIRS ? 2 : STAGES) {   // 256 sums leave no registers for several ways out: stages behind the last are zeros
            stage(S0, TWO);
            stage(S1, LAST);
            if constexpr (!PAIRS) {
                stage(S2, TWO);
                stage(S3, LAST);
            }
        }
        group_ready<0>();   // nothing is on its way to LDS, and all waves have read it
        const int64_t left = rows - (m0 + wm);   // rows from the wave's first on
        const uint64_t to = (uint64_t)(uintptr_t)(out + (m0 + wm) * a.n + n0 + wn);
        const u32x4 result = {(uint32_t)to, (uint32_t)(to >> 32) & 0xffffu, left > 0 && n0 + wn < a.n ? (uint32_t)(((min(left, (int64_t)128) - 1) * a.n + a.n - n0 - wn) * (int64_t)sizeof(T)) : 0u, 0x00020000u};
        const int wide = (int)min(a.n - n0 - wn, (int64_t)128);   // columns from the wave's first on
        const uint32_t column = n0 + wn + l16 * 8 < a.n ? (uint32_t)l16 * 16 : 0x80000000u;   // beyond the result
        uint8_t* const own = lds + (PAIRS ? before(cur) : STAGES * STAGE) + wave * OWN;
        u += kRound;
        if (u < full) begin(u);
#pragma unroll
        for (int j = 0; j < F; ++j) group_mfma_done(acc[j]);
        // The result, 32 rows of the wave's at a time, through LDS of its own: a lane
        // writes 4 numbers of a fragment, or 32 in a row, and reads 16 bytes of a row.
        // Pieces change places by the row's number.
#pragma unroll
        for (int p = 0; p < F / 2; ++p) {
#pragma unroll
            for (int j = 2 * p; j < 2 * p + 2; ++j) {
#pragma unroll
                for (int i = 0; i < F; ++i) {
                    const int n = ACROSS ? i * 16 + quad * 4 : quad * (4 * F) + i * 4;
                    const f32x4 v = acc[j][i];
                    *(u32x2*)(own + ((j & 1) * 16 + l16) * 256 + (((n / 8) ^ l16) * 16) + (n & 4) * 2) = u32x2{narrow2<T>(v[0], v[1]), narrow2<T>(v[2], v[3])};
                    __builtin_amdgcn_sched_barrier(0);
                }
                group_zero(acc[j]);
            }
            __builtin_amdgcn_wave_barrier();
            if (!a.out_pieces) {
                T* const rest = (T*)(uintptr_t)((uint64_t)result[1] << 32 | result[0]) + l16 * 8;
                for (int row = quad; row < 32; row += 4) {
                    if (p * 32 + row >= left) break;
                    const u32x4 v = *(const u32x4*)(own + row * 256 + ((l16 ^ (row & 15)) * 16));
                    T* const to = rest + (p * 32 + row) * a.n;
                    if (l16 * 8 + 8 <= wide) store16(to, v);
                    else if (l16 * 8 < wide) store_part(to, v, wide - l16 * 8);
                }
                if (p == F / 2 - 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // they are no fixed number, which `first` counts on
            } else {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int row = r * 4 + quad;
                    const u32x4 v = *(const u32x4*)(own + row * 256 + ((l16 ^ (row & 15)) * 16));
                    const uint32_t at = column + (uint32_t)(p * 32 + row) * (uint32_t)(a.n * (int64_t)sizeof(T));
                    __builtin_amdgcn_raw_buffer_store_b128(v, __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)((uint64_t)result[1] << 32 | result[0]), (short)0, (int)result[2], 0x00020000), at, 0, 0);
                }
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
        if (u < full) first(STORES);
    }
    for (; u - full < 4 * rest; u += kRound) {
        const uint32_t i = u - full;
        GroupWork w = group_work<WEIGHT>(a, tiles, full + i / 4, high, a.tiles_n, 256, 256);
        w.m0 += (i & 1) * 128;
        w.n0 += (i & 2) * 64;
        if (w.n0 >= a.n || w.m0 >= (WEIGHT ? a.m : w.end - w.first)) continue;
        __syncthreads();
        group_large_tile<T, WEIGHT, ACROSS, 4, 4, 8>(a, w, lds);
    }
}

// Smaller tiles of 16 bits in the same manner, several workgroups to a CU, for a
// B across k (weight gradients of 16 rows by 16 experts of 2048 x 5632: 104 us, with
// group_kernel 133; the gradient of x 46 and 68).  Along k group_kernel's
// rows of 128 bytes are better than these of 64 (16 x 2048 -> 5632 by 16: 46 us, 49).
template <typename T, bool WEIGHT, bool B_ACROSS, int F, int STAGES, int BLOCKS> __global__ __launch_bounds__(256, BLOCKS) void group_small_kernel(GroupArgs a) {
    __shared__ __align__(16) uint8_t lds[STAGES * 64 * F * 64];
    if (blockIdx.x >= a.tiles) {
        group_fill<T>(a, blockIdx.x - a.tiles, gridDim.x - a.tiles);
        return;
    }
    GroupWork w;
    if (group_begin<WEIGHT>(a, 32 * F, 32 * F, w)) group_large_tile<T, WEIGHT, WEIGHT || B_ACROSS, F, F, STAGES>(a, w, lds);
}

// The rows of a tile that is 64 wide.  fp32 products take 32: experts' last tiles are
// emptier where they are higher, and 256 CUs share the others more evenly (777 x
// 1001 -> 1500 by 9: 36.5 us, 43.0 with 64 rows, the gradient of x 39.5 and 52; 777 x
// 1024 -> 1536 32.7 and 40.2; 2500 rows an expert lose 3 %).
template <typename T, bool WEIGHT> constexpr int kGroupHigh = sizeof(T) == 4 && !WEIGHT ? 32 : 64;
// How a product is computed: the side of its tiles, and into how many parts k is split.
struct GroupPlan {
    int tile;     // 64, 128 or 256; 64 stands for kGroupHigh x 64
    uint32_t splits;
    bool whole;   // aligned, whole pieces
    bool words;   // fp32 of any alignment whose rows lie apart, near enough for a buffer
};
// One dtype's kernels, each in a source file of its own.
template <typename T> void group_launch(GroupArgs a, bool weight, bool across, GroupPlan plan, hipStream_t st);

#define CRESSO_GROUP_LAUNCH(T)                                                                                          \
    template <> void group_launch<T>(GroupArgs a, bool weight, bool across, GroupPlan plan, hipStream_t st) {           \
        const auto run = [&](auto kernel, int high, int wide) {                                                         \
            a.tiles_n = (uint32_t)((a.n + wide - 1) / wide);                                                            \
            a.tiles_m = (uint32_t)(weight ? (a.m + high - 1) / high : a.rows / high + a.experts);                       \
            a.tiles = a.tiles_m * a.tiles_n * (weight ? (uint32_t)a.experts : 1u);                                      \
            a.splits = plan.splits;                                                                                     \
            hipLaunchKernelGGL(kernel, dim3(a.tiles * a.splits + (weight || a.splits > 1 ? 0 : kFillBlocks)),           \
                               dim3(256), 0, st, a);                                                                    \
        };                                                                                                              \
        const auto size = [&](auto w, auto x) {                                                                         \
            constexpr bool W = decltype(w)::value, X = decltype(x)::value;                                              \
            if constexpr (sizeof(T) == 2) {                                                                             \
                if (plan.whole && plan.tile == 256) {                                                                   \
                    a.tiles_n = (uint32_t)((a.n + 255) / 256);                                                          \
                    a.tiles_m = (uint32_t)((a.m + 255) / 256);                                                          \
                    a.splits = 1;                                                                                       \
                    const dim3 grid(kRound + (W ? 0 : kFillBlocks));                                                    \
                    if constexpr (!X) {                                                                                 \
                        if (a.k_along % 64 == 0) {                                                                           \
                            hipLaunchKernelGGL((group_large_kernel<T, W, X, true>), grid, dim3(256), 0, st, a);         \
                            return;                                                                                     \
                        }                                                                                               \
                    }                                                                                                   \
                    hipLaunchKernelGGL((group_large_kernel<T, W, X, false>), grid, dim3(256), 0, st, a);                \
                    return;                                                                                             \
                }                                                                                                       \
                if constexpr (X)                                                                                        \
                    if (plan.whole && plan.tile == 128 && plan.splits < 2) return run(group_small_kernel<T, W, X, 4, 4, 2>, 128, 128);\
                if constexpr (W)                                                                                        \
                    if (plan.whole && plan.tile == 64 && plan.splits < 2) return run(group_small_kernel<T, W, X, 2, 4, 4>, 64, 64);\
            }                                                                                                           \
            constexpr int FM = kGroupHigh<T, W> / 16, STAGES = FM == 2 ? 2 : 3;                                         \
            if (plan.whole && plan.tile >= 128) {                                                                       \
                if constexpr (W || sizeof(T) == 2) run(group_kernel<T, W, X, 1, 4, 8, 2, 128, 2>, 128, 128);            \
            } else if (plan.whole) {                                                                                    \
                if constexpr (W || !X || sizeof(T) == 4) run(group_kernel<T, W, X, 1, 4, FM, 1, 128, STAGES>, 16 * FM, 64);\
            } else if (plan.words) {                                                                                    \
                if constexpr (sizeof(T) == 4) run(group_kernel<T, W, X, 1, 4, FM, 1, 128, STAGES, 4>, 16 * FM, 64);     \
            } else if (plan.tile >= 128) {                                                                              \
                if constexpr (!X && sizeof(T) == 2) run(group_any_kernel<T, W, X, 1, 4, 8, 2>, 128, 128);               \
            } else {                                                                                                    \
                run(group_any_kernel<T, W, X, 1, 4, FM, 1>, 16 * FM, 64);                                               \
            }                                                                                                           \
            if (a.splits < 2) return;                                                                                   \
            const int64_t units = ((W ? (int64_t)a.experts * a.m : a.rows) * a.n + Unit<T>::n - 1) / Unit<T>::n;        \
            hipLaunchKernelGGL((group_join_kernel<T, W>), dim3((uint32_t)std::min<int64_t>((units + 255) / 256, 4096)), \
                               dim3(256), 0, st, a);                                                                    \
        };                                                                                                              \
        if (weight) size(std::true_type{}, std::true_type{});                                                           \
        else if (across) size(std::false_type{}, std::true_type{});                                                     \
        else size(std::false_type{}, std::false_type{});                                                                \
    }

}  // namespace cresso
