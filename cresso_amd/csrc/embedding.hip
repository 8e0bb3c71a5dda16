// Embedding lookup with a scale, and the gradient of its table.
//
//   out[t] = scale * table[id_t]                       (0 where id_t is outside the table)
//   dtable[v] = scale * sum of grad[t] over t with id_t = v, in the order of t;  0 for rows that no token names
//
// Forward: one read and one write of each token's row, 16 bytes per lane.
//
// Gradient: the tokens are sorted by id (stable, so a row's terms keep the
// order of the tokens and the result does not depend on timing), then the
// sorted list is cut into equal chunks, whatever the ids: a word that is a
// tenth of the text is shared by many waves as evenly as rare ones are.  Sums
// are fp32.  A segment (the tokens of one id) that ends inside its chunk is
// written to the table at once; one that goes on is kept as fp32 partial
// sums, which a second kernel adds in chunk order.  Rows without a token are
// filled by further waves of the first kernel, so the table is written once.
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

constexpr int EM_NT = 256;
constexpr int EM_CHUNK = 32;       // sorted tokens per wave (at most a wave's lanes)
constexpr int EM_MAX_BLOCKS = 1 << 20;   // of the lookup; more tokens are looped over
constexpr int EM_ZROWS = 8;        // table rows per wave of the fill
constexpr int SO_NT = 1024;        // threads of the sort: 16 waves
constexpr int SO_WAVES = SO_NT / kWave;
constexpr int SO_BITS = 9;         // digit
constexpr int SO_DIGITS = 1 << SO_BITS;
constexpr int SO_ROUNDS = 16;      // keys per thread
constexpr int SO_TILE = SO_NT * SO_ROUNDS;

template <typename I> __device__ __forceinline__ int64_t id_at(const void* ids, int64_t t) {
    return (int64_t)((const CRESSO_GLOBAL I*)ids)[t];
}
__device__ __forceinline__ int64_t load_id(const void* ids, int32_t id_bytes, int64_t t) {
    return id_bytes == 8 ? id_at<int64_t>(ids, t) : id_at<int32_t>(ids, t);
}

template <typename T>
__global__ __launch_bounds__(EM_NT) void embed_forward_kernel(const void* ids, int32_t id_bytes, int64_t tokens,
                                                              const T* table, int64_t rows, int64_t row_stride,
                                                              int64_t width, uint32_t units, uint32_t tokens_per_block,
                                                              float scale, T* out) {
    for (int64_t t0 = (int64_t)blockIdx.x * tokens_per_block; t0 < tokens; t0 += (int64_t)gridDim.x * tokens_per_block) {
        const uint32_t here = (uint32_t)min((int64_t)tokens_per_block, tokens - t0);
        for (uint32_t i = threadIdx.x; i < here * units; i += EM_NT) {
            const uint32_t k = i / units, u = i - k * units;
            const int64_t t = t0 + k, id = load_id(ids, id_bytes, t);
            u32x4 r = {0, 0, 0, 0};
            if (id >= 0 && id < rows) {
                r = load_unit(table + id * row_stride, u, width);
                float v[Unit<T>::n];
                widen<T>(r, v);
#pragma unroll
                for (int e = 0; e < Unit<T>::n; ++e) v[e] *= scale;
                r = narrow<T>(v);
            }
            store_unit(out + t * width, u, width, r);
        }
    }
}

// ---------------------------------------------------------------------------
// Stable sort of (id, token) by id, least significant digit first.
//
// A tile of up to 16384 keys is ranked by one workgroup: each wave takes a
// contiguous part, 64 keys a round, finds the lanes with its key's digit by
// one ballot per digit bit, and keeps a running count per digit in LDS.
// ---------------------------------------------------------------------------
struct SortTile {
    uint32_t key[SO_TILE];
    uint16_t from[SO_TILE];
    uint32_t count[SO_WAVES][SO_DIGITS];   // per wave and digit; then the first place of each
    uint32_t scan[SO_DIGITS / kWave];
};

__device__ __forceinline__ uint32_t digit_of(uint32_t key, int shift) { return (key >> shift) & (SO_DIGITS - 1); }

// Ranks the keys of a wave's part among the wave's keys of the same digit.
// Thread-held: key[r], rank[r] for round r; `mine` keys in this wave's part.
__device__ __forceinline__ void rank_wave(SortTile& s, const uint32_t (&key)[SO_ROUNDS], uint32_t (&rank)[SO_ROUNDS],
                                          int mine, int shift) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int d = lane; d < SO_DIGITS; d += kWave) s.count[wave][d] = 0;
    __builtin_amdgcn_wave_barrier();
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int r = 0; r < SO_ROUNDS; ++r) {
        if (r * kWave < mine) {
            const bool on = r * kWave + lane < mine;
            const uint32_t d = digit_of(key[r], shift);
            uint64_t same = __ballot(on);
#pragma unroll
            for (int b = 0; b < SO_BITS; ++b) {
                const uint64_t m = __ballot((d >> b) & 1);
                same &= ((d >> b) & 1) ? m : ~m;
            }
            if (on) {
                const uint32_t before = s.count[wave][d], ahead = (uint32_t)__popcll(same & below);
                rank[r] = before + ahead;
                __builtin_amdgcn_wave_barrier();
                if (ahead == 0) s.count[wave][d] = before + (uint32_t)__popcll(same);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Exclusive prefix of count[][] in digit order, then wave order.  All threads.
__device__ __forceinline__ void scan_counts(SortTile& s) {
    const int t = threadIdx.x, lane = t & (kWave - 1);
    uint32_t total = 0;
    if (t < SO_DIGITS)
        for (int w = 0; w < SO_WAVES; ++w) total += s.count[w][t];
    uint32_t upto = total;
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
        const uint32_t v = __shfl_up(upto, m, kWave);
        if (lane >= m) upto += v;
    }
    if (t < SO_DIGITS && lane == kWave - 1) s.scan[t / kWave] = upto;
    __syncthreads();
    if (t < SO_DIGITS) {
        uint32_t at = upto - total;
        for (int w = 0; w < t / kWave; ++w) at += s.scan[w];
        for (int w = 0; w < SO_WAVES; ++w) {
            const uint32_t n = s.count[w][t];
            s.count[w][t] = at;
            at += n;
        }
    }
    __syncthreads();
}

// The part of a tile of n keys that a wave ranks: [first, first + mine).
__device__ __forceinline__ void wave_part(int n, int wave, int& first, int& mine) {
    const int part = ((n + SO_WAVES - 1) / SO_WAVES + kWave - 1) / kWave * kWave;
    first = wave * part;
    mine = max(0, min(part, n - first));
}

__device__ __forceinline__ uint32_t key_of(const void* ids, int32_t id_bytes, int64_t t, int64_t rows) {
    const int64_t id = load_id(ids, id_bytes, t);
    return (uint32_t)(id >= 0 && id < rows ? id : rows);   // ids outside the table go last
}

// The whole sort of up to SO_TILE tokens in one workgroup.
__global__ __launch_bounds__(SO_NT) void embed_sort_tile_kernel(const void* ids, int32_t id_bytes, int32_t tokens,
                                                                int64_t rows, int32_t bits, uint32_t* sorted_ids,
                                                                uint32_t* sorted_tokens) {
    extern __shared__ __align__(16) char lds[];
    SortTile& s = *reinterpret_cast<SortTile*>(lds);
    const int lane = threadIdx.x & (kWave - 1);
    int first, mine;
    wave_part(tokens, threadIdx.x / kWave, first, mine);
    uint32_t key[SO_ROUNDS], rank[SO_ROUNDS], from[SO_ROUNDS];
#pragma unroll
    for (int r = 0; r < SO_ROUNDS; ++r) {
        const int i = r * kWave + lane;
        key[r] = i < mine ? key_of(ids, id_bytes, first + i, rows) : 0;
        from[r] = (uint32_t)(first + i);
        rank[r] = 0;
    }
    for (int shift = 0; shift < bits; shift += SO_BITS) {
        rank_wave(s, key, rank, mine, shift);
        __syncthreads();
        scan_counts(s);
#pragma unroll
        for (int r = 0; r < SO_ROUNDS; ++r)
            if (r * kWave + lane < mine) {
                const uint32_t at = s.count[threadIdx.x / kWave][digit_of(key[r], shift)] + rank[r];
                s.key[at] = key[r];
                s.from[at] = (uint16_t)from[r];
            }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SO_ROUNDS; ++r) {
            const int i = r * kWave + lane;
            if (i < mine) {
                key[r] = s.key[first + i];
                from[r] = s.from[first + i];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < SO_ROUNDS; ++r) {
        const int i = r * kWave + lane;
        if (i < mine) {
            sorted_ids[first + i] = key[r];
            sorted_tokens[first + i] = from[r];
        }
    }
}

// One digit of the sort of more tokens: counts of each tile, their places, the move.
struct SortPass {
    const void* ids;             // first pass: the tokens' ids; later passes: in_ids, in_tokens
    const uint32_t *in_ids, *in_tokens;
    uint32_t *out_ids, *out_tokens;
    uint32_t* places;            // [digit][tile]
    int64_t tokens, rows;
    uint32_t tiles;
    int32_t id_bytes, shift, first_pass;
};
__device__ __forceinline__ uint32_t pass_key(const SortPass& p, int64_t t) {
    return p.first_pass ? key_of(p.ids, p.id_bytes, t, p.rows) : p.in_ids[t];
}
__global__ __launch_bounds__(SO_NT) void embed_sort_count_kernel(SortPass p) {
    __shared__ uint32_t count[SO_DIGITS];
    for (int d = threadIdx.x; d < SO_DIGITS; d += SO_NT) count[d] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * SO_TILE;
    const int n = (int)min((int64_t)SO_TILE, p.tokens - t0);
    for (int i = threadIdx.x; i < n; i += SO_NT) atomicAdd(&count[digit_of(pass_key(p, t0 + i), p.shift)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < SO_DIGITS; d += SO_NT) p.places[(size_t)d * p.tiles + blockIdx.x] = count[d];
}
// Exclusive prefix over [digit][tile], one workgroup.
__global__ __launch_bounds__(SO_NT) void embed_sort_scan_kernel(uint32_t* places, size_t n) {
    __shared__ uint32_t part[SO_WAVES];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    uint32_t before = 0;
    for (size_t i0 = 0; i0 < n; i0 += SO_NT) {
        const size_t i = i0 + threadIdx.x;
        const uint32_t v = i < n ? places[i] : 0;
        uint32_t upto = v;
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) {
            const uint32_t w = __shfl_up(upto, m, kWave);
            if (lane >= m) upto += w;
        }
        if (lane == kWave - 1) part[wave] = upto;
        __syncthreads();
        uint32_t lead = before, all = 0;
        for (int w = 0; w < SO_WAVES; ++w) {
            if (w < wave) lead += part[w];
            all += part[w];
        }
        if (i < n) places[i] = lead + upto - v;
        before += all;
        __syncthreads();
    }
}
__global__ __launch_bounds__(SO_NT) void embed_sort_move_kernel(SortPass p) {
    extern __shared__ __align__(16) char lds[];
    SortTile& s = *reinterpret_cast<SortTile*>(lds);
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t t0 = (int64_t)blockIdx.x * SO_TILE;
    const int n = (int)min((int64_t)SO_TILE, p.tokens - t0);
    int first, mine;
    wave_part(n, wave, first, mine);
    uint32_t key[SO_ROUNDS], rank[SO_ROUNDS];
#pragma unroll
    for (int r = 0; r < SO_ROUNDS; ++r) {
        const int i = r * kWave + lane;
        key[r] = i < mine ? pass_key(p, t0 + first + i) : 0;
        rank[r] = 0;
    }
    rank_wave(s, key, rank, mine, p.shift);
    __syncthreads();
    // each digit's keys of this tile go to its place, wave after wave
    if (threadIdx.x < SO_DIGITS) {
        uint32_t at = p.places[(size_t)threadIdx.x * p.tiles + blockIdx.x];
        for (int w = 0; w < SO_WAVES; ++w) {
            const uint32_t c = s.count[w][threadIdx.x];
            s.count[w][threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SO_ROUNDS; ++r) {
        const int i = r * kWave + lane;
        if (i < mine) {
            const uint32_t at = s.count[wave][digit_of(key[r], p.shift)] + rank[r];
            const int64_t t = t0 + first + i;
            p.out_ids[at] = key[r];
            p.out_tokens[at] = p.first_pass ? (uint32_t)t : p.in_tokens[t];
        }
    }
}

// ---------------------------------------------------------------------------
// Sums over the sorted tokens
// ---------------------------------------------------------------------------
struct EmbedSum {
    const uint32_t *ids, *from;   // sorted
    uint32_t tokens, chunks, tiles, rows;   // tiles: column tiles of 64 units
    int64_t width, grad_stride;
    float scale;
    float* partial;               // [chunk][head, tail][tile][64 units] fp32
    uint32_t sum_blocks;
};

// first place in ids[lo, hi) whose id is >= v
__device__ __forceinline__ uint32_t lower_bound(const uint32_t* ids, uint32_t lo, uint32_t hi, uint32_t v) {
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (ids[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ float* partial_at(const EmbedSum& a, uint32_t chunk, int tail, uint32_t tile) {
    return a.partial + (((size_t)chunk * 2 + tail) * a.tiles + tile) * (kWave * Unit<T>::n) +
           (threadIdx.x & (kWave - 1)) * Unit<T>::n;
}
template <typename T>
__device__ __forceinline__ void write_row(const EmbedSum& a, T* out, uint32_t v, uint32_t unit, float (&s)[Unit<T>::n]) {
    if (v >= a.rows) return;   // ids outside the table
#pragma unroll
    for (int e = 0; e < Unit<T>::n; ++e) s[e] *= a.scale;
    store_unit(out + (int64_t)v * a.width, unit, a.width, narrow<T>(s));
}

template <typename T>
__global__ __launch_bounds__(EM_NT) void embed_sum_kernel(EmbedSum a, const T* grad, T* out) {
    constexpr int E = Unit<T>::n;
    const int lane = threadIdx.x & (kWave - 1);
    const uint32_t wave = threadIdx.x / kWave;
    if (blockIdx.x >= a.sum_blocks) {   // rows without a token
        const uint64_t v0 = ((uint64_t)(blockIdx.x - a.sum_blocks) * (EM_NT / kWave) + wave) * EM_ZROWS;
        if (v0 >= a.rows) return;
        const int n = (int)min((uint64_t)EM_ZROWS, a.rows - v0);
        bool empty = false;
        if (lane < n) {
            const uint32_t v = (uint32_t)v0 + lane, at = lower_bound(a.ids, 0, a.tokens, v);
            empty = at == a.tokens || a.ids[at] != v;
        }
        uint64_t todo = __ballot(empty);
        while (todo) {
            const int k = __builtin_ctzll(todo);
            todo &= todo - 1;
            T* row = out + (int64_t)(v0 + k) * a.width;
            for (int64_t u = lane; u * E < a.width; u += kWave) store_unit(row, u, a.width, u32x4{0, 0, 0, 0});
        }
        return;
    }
    const uint64_t job = (uint64_t)blockIdx.x * (EM_NT / kWave) + wave;
    const uint32_t chunk = (uint32_t)(job / a.tiles), tile = (uint32_t)(job - (uint64_t)chunk * a.tiles);
    if (chunk >= a.chunks) return;
    const uint32_t unit = tile * kWave + lane;
    const uint32_t p0 = chunk * EM_CHUNK, n = min((uint32_t)EM_CHUNK, a.tokens - p0);
    const uint32_t my_id = a.ids[p0 + min((uint32_t)lane, n - 1)], my_from = a.from[p0 + min((uint32_t)lane, n - 1)];
    const bool from_before = p0 > 0 && a.ids[p0 - 1] == __builtin_amdgcn_readfirstlane(my_id);
    const bool goes_on = p0 + n < a.tokens && a.ids[p0 + n] == a.ids[p0 + n - 1];
    float s[E] = {};
    uint32_t current = __builtin_amdgcn_readfirstlane(my_id);
    bool head = from_before;   // the current segment began in an earlier chunk
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t v = __builtin_amdgcn_readlane(my_id, i);
        if (v != current) {
            if (head) {
                float* q = partial_at<T>(a, chunk, 0, tile);
#pragma unroll
                for (int e = 0; e < E; ++e) q[e] = s[e];
            } else {
                write_row(a, out, current, unit, s);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] = 0.0f;
            head = false;
            current = v;
        }
        if (v < a.rows) {
            float g[E];
            widen<T>(load_unit(grad + (int64_t)__builtin_amdgcn_readlane(my_from, i) * a.grad_stride, unit, a.width), g);
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] += g[e];
        }
    }
    if (head || goes_on) {
        float* q = partial_at<T>(a, chunk, head ? 0 : 1, tile);
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = s[e];
    } else {
        write_row(a, out, current, unit, s);
    }
}

// Adds the partial sums of each segment that began in one chunk and went on in
// the next: a workgroup for its first chunk and a column tile.  The chunks
// are shared out over the waves in order, and the waves' sums added in order.
template <typename T>
__global__ __launch_bounds__(EM_NT) void embed_join_kernel(EmbedSum a, T* out) {
    constexpr int E = Unit<T>::n, W = EM_NT / kWave;
    __shared__ float part[W][kWave][E + 1];
    const uint32_t chunk = blockIdx.x / a.tiles, tile = blockIdx.x - chunk * a.tiles;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t p0 = chunk * EM_CHUNK, p1 = p0 + EM_CHUNK;   // there is a next chunk
    const uint32_t v = a.ids[p1 - 1];
    if (a.ids[p1] != v || v >= a.rows) return;
    if (p0 > 0 && a.ids[p0 - 1] == v) return;   // began earlier
    const uint32_t end = lower_bound(a.ids, p1, a.tokens, v + 1);
    const uint32_t heads = (end - 1) / EM_CHUNK - chunk;        // chunks after this one
    const uint32_t share = (heads + W - 1) / W;
    const uint32_t k0 = min(heads, wave * share), k1 = min(heads, k0 + share);
    float s[E] = {};
    if (wave == 0) {
        const float* q = partial_at<T>(a, chunk, 1, tile);
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] = q[e];
    }
#pragma unroll 4
    for (uint32_t k = k0; k < k1; ++k) {
        const float* q = partial_at<T>(a, chunk + 1 + k, 0, tile);
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += q[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) part[wave][lane][e] = s[e];
    __syncthreads();
    if (wave != 0) return;
    for (int w = 1; w < W; ++w)
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += part[w][lane][e];
    write_row(a, out, v, tile * kWave + lane, s);
}

int64_t al256(int64_t v) { return (v + 255) & ~(int64_t)255; }

struct EmbedLayout {
    int64_t ids, tokens, ids2, tokens2, places, partial, total;
    uint32_t chunks, tiles, sort_tiles;
};
EmbedLayout embed_layout(int64_t tokens, int64_t width, int32_t dtype) {
    EmbedLayout o{};
    const int64_t e = dtype == CRESSO_F32 ? 4 : 8;
    o.chunks = (uint32_t)((tokens + EM_CHUNK - 1) / EM_CHUNK);
    o.tiles = (uint32_t)((width + kWave * e - 1) / (kWave * e));
    o.sort_tiles = (uint32_t)((tokens + SO_TILE - 1) / SO_TILE);
    int64_t off = 0;
    auto take = [&](int64_t b) { const int64_t at = off; off = al256(off + b); return at; };
    o.ids = take(tokens * 4);
    o.tokens = take(tokens * 4);
    if (o.sort_tiles > 1) {
        o.ids2 = take(tokens * 4);
        o.tokens2 = take(tokens * 4);
        o.places = take((int64_t)SO_DIGITS * o.sort_tiles * 4);
    }
    if (o.chunks > 1) o.partial = take((int64_t)o.chunks * 2 * o.tiles * kWave * e * 4);
    o.total = std::max<int64_t>(off, 256);
    return o;
}

int32_t check_embedding(const char* what, const void* ids, int32_t id_bytes, int64_t tokens, int64_t rows, int64_t width,
                        int32_t dtype) {
    if (id_bytes != 4 && id_bytes != 8) return fail(CRESSO_E_INVALID, "%s: ids of %d bytes (4 or 8)", what, id_bytes);
    if (!row_dtype(dtype)) return fail(CRESSO_E_UNSUPPORTED, "%s: dtype %d not supported (f32, bf16, f16)", what, dtype);
    if (tokens < 0 || rows < 0 || width < 0) return fail(CRESSO_E_INVALID, "%s: negative size", what);
    // grids of up to 2^32 threads; 32-bit places in the sorted list
    if (tokens >= (int64_t)1 << 28 || rows >= (int64_t)1 << 28 || width >= (int64_t)1 << 28 ||
        tokens * (width / 256 + 1) >= (int64_t)1 << 29)
        return fail(CRESSO_E_UNSUPPORTED, "%s: %lld tokens, %lld rows, width %lld are more than one call takes", what,
                    (long long)tokens, (long long)rows, (long long)width);
    if (tokens > 0 && !ids) return fail(CRESSO_E_INVALID, "%s: null argument", what);
    return CRESSO_OK;
}

}  // namespace
}  // namespace cresso

using namespace cresso;

extern "C" int32_t cresso_embedding_forward(const void* ids, int32_t id_bytes, int64_t tokens, const void* table,
                                            int64_t rows, int64_t width, int64_t row_stride, int32_t dtype, double scale,
                                            void* out, void* stream) {
    const int32_t rc = check_embedding("embedding", ids, id_bytes, tokens, rows, width, dtype);
    if (rc != CRESSO_OK) return rc;
    if (tokens == 0 || width == 0) return CRESSO_OK;
    if (!out || (rows > 0 && !table)) return fail(CRESSO_E_INVALID, "embedding: null argument");
    if (rows > 1 && row_stride < width) return fail(CRESSO_E_INVALID, "embedding: row stride below the width");
    with_row_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const uint32_t units = (uint32_t)((width + Unit<T>::n - 1) / Unit<T>::n);
        const uint32_t per = std::max<uint32_t>(1, EM_NT / units);
        const int64_t blocks = std::min<int64_t>((tokens + per - 1) / per, EM_MAX_BLOCKS);
        hipLaunchKernelGGL(embed_forward_kernel<T>, dim3((uint32_t)blocks), dim3(EM_NT), 0, (hipStream_t)stream,
                           ids, id_bytes, tokens, (const T*)table, rows, row_stride, width, units, per, (float)scale,
                           (T*)out);
    });
    return launched("embedding");
}

extern "C" size_t cresso_embedding_backward_workspace_bytes(int64_t tokens, int64_t width, int32_t dtype) {
    if (tokens < 0 || width < 0 || tokens >= (int64_t)1 << 31 || width >= (int64_t)1 << 31 || !row_dtype(dtype)) return 0;
    return (size_t)embed_layout(tokens, width, dtype).total;
}

extern "C" int32_t cresso_embedding_backward(const void* ids, int32_t id_bytes, int64_t tokens, const void* grad,
                                             int64_t grad_stride, int64_t rows, int64_t width, int32_t dtype, double scale,
                                             void* grad_table, void* workspace, size_t workspace_bytes, void* stream) {
    const int32_t rc = check_embedding("embedding gradient", ids, id_bytes, tokens, rows, width, dtype);
    if (rc != CRESSO_OK) return rc;
    if (rows == 0 || width == 0) return CRESSO_OK;
    if (!grad_table || (tokens > 0 && !grad)) return fail(CRESSO_E_INVALID, "embedding gradient: null argument");
    if (tokens > 1 && grad_stride < 0) return fail(CRESSO_E_INVALID, "embedding gradient: negative row stride");
    const EmbedLayout o = embed_layout(tokens, width, dtype);
    if (!workspace || workspace_bytes < (size_t)o.total)
        return fail(CRESSO_E_INVALID, "embedding gradient: workspace of %zu bytes, %lld needed", workspace_bytes,
                    (long long)o.total);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    uint32_t *sid = (uint32_t*)(ws + o.ids), *sfrom = (uint32_t*)(ws + o.tokens);
    int bits = 1;   // of the largest key, `rows`
    while (((int64_t)1 << bits) <= rows) ++bits;
    if (o.sort_tiles == 1) {
        hipLaunchKernelGGL(embed_sort_tile_kernel, dim3(1), dim3(SO_NT), sizeof(SortTile), st, ids, id_bytes,
                           (int32_t)tokens, rows, bits, sid, sfrom);
    } else if (o.sort_tiles > 1) {
        uint32_t *a_ids = sid, *a_tok = sfrom, *b_ids = (uint32_t*)(ws + o.ids2), *b_tok = (uint32_t*)(ws + o.tokens2);
        SortPass p{};
        p.ids = ids;
        p.places = (uint32_t*)(ws + o.places);
        p.tokens = tokens;
        p.rows = rows;
        p.tiles = o.sort_tiles;
        p.id_bytes = id_bytes;
        for (p.shift = 0; p.shift < bits; p.shift += SO_BITS) {
            p.first_pass = p.shift == 0;
            p.in_ids = a_ids;
            p.in_tokens = a_tok;
            p.out_ids = b_ids;
            p.out_tokens = b_tok;
            hipLaunchKernelGGL(embed_sort_count_kernel, dim3(o.sort_tiles), dim3(SO_NT), 0, st, p);
            hipLaunchKernelGGL(embed_sort_scan_kernel, dim3(1), dim3(SO_NT), 0, st, p.places,
                               (size_t)SO_DIGITS * o.sort_tiles);
            hipLaunchKernelGGL(embed_sort_move_kernel, dim3(o.sort_tiles), dim3(SO_NT), sizeof(SortTile), st, p);
            std::swap(a_ids, b_ids);
            std::swap(a_tok, b_tok);
        }
        sid = a_ids;
        sfrom = a_tok;
    }
    with_row_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        EmbedSum a{};
        a.ids = sid;
        a.from = sfrom;
        a.tokens = (uint32_t)tokens;
        a.chunks = o.chunks;
        a.tiles = o.tiles;
        a.rows = (uint32_t)rows;
        a.width = width;
        a.grad_stride = grad_stride;
        a.scale = (float)scale;
        a.partial = (float*)(ws + o.partial);
        constexpr int W = EM_NT / kWave;
        a.sum_blocks = (uint32_t)(((uint64_t)o.chunks * o.tiles + W - 1) / W);
        const uint32_t zero_blocks = (uint32_t)((rows + EM_ZROWS * W - 1) / (EM_ZROWS * W));
        hipLaunchKernelGGL(embed_sum_kernel<T>, dim3(a.sum_blocks + zero_blocks), dim3(EM_NT), 0, st, a, (const T*)grad,
                           (T*)grad_table);
        if (o.chunks > 1)
            hipLaunchKernelGGL(embed_join_kernel<T>, dim3((o.chunks - 1) * o.tiles), dim3(EM_NT), 0, st, a, (T*)grad_table);
    });
    return launched("embedding gradient");
}
