// Embedding lookup with a scale, and the gradient of its table.
//
//   out[t] = scale * table[id_t]                       (0 where id_t is outside the table)
//   dtable[v] = scale * sum of grad[t] over t with id_t = v, in the order of t;  0 for rows that no token names
//
// Forward: one read and one write of each token's row, 16 bytes per lane;
// bound by HBM (16384 x 4096 bf16 of 32000 rows: 43 to 48 us, 134 MB written and
// 110 read, 5.1 to 5.7 TB/s) or, for a few tokens, by the launch and the two
// loads that wait for one another (8 x 2048: 2.7 us).
//
// Gradient: the tokens are sorted by id (stable, so a row's terms keep the
// order of the tokens and the result does not depend on timing), then the
// sorted list is cut into equal chunks, whatever the ids: a word that is a
// tenth of the text is shared by many waves as evenly as rare ones are.  Sums
// are fp32.  A segment (the tokens of one id) that ends inside its chunk is
// written to the table at once; one that goes on is kept as fp32 partial
// sums, which a second kernel adds in chunk order.  Rows without a token are
// filled by further waves of the first kernel, so the table is written once.
//
// 16384 x 4096 bf16 into 32000 rows: sort 6.0 + 8.8 us (latency of its steps in
// LDS, 16 workgroups), sums 83 us (134 MB in, 262 MB out: 4.8 TB/s), joins
// 6.8 us.  2777 x 768 fp32 into 50257 rows: sort 6.1 + 4.1, sums 29 us (163 MB,
// 5.6 TB/s), joins 4.0.
#include "row_ops.hpp"

#include <algorithm>

namespace cresso {
namespace {

constexpr int EM_NT = 256;
constexpr int EM_CHUNK = 32;       // sorted tokens per wave (at most a wave's lanes)
constexpr uint32_t EM_AHEAD = 8;   // of them whose loads are on their way together
constexpr int EM_MAX_BLOCKS = 1 << 20;   // of the lookup; more tokens are looped over
constexpr int EM_ZROWS = 8;        // table rows per wave of the fill
constexpr int SO_NT = 1024;        // threads of the sort: 16 waves
constexpr int SO_WAVES = SO_NT / kWave;
constexpr int SO_BITS = 9;         // digit
constexpr int SO_DIGITS = 1 << SO_BITS;
constexpr int SO_ROUNDS = 4;       // keys per thread of the counting sort
constexpr int SO_TILE = SO_NT * SO_ROUNDS;
constexpr int SO_MERGE = 32;       // tiles of SO_NT keys that are merged in one step

template <typename I> __device__ __forceinline__ int64_t id_at(const void* ids, int64_t t) {
    return (int64_t)((const CRESSO_GLOBAL I*)ids)[t];
}
__device__ __forceinline__ int64_t load_id(const void* ids, int32_t id_bytes, int64_t t) {
    return id_bytes == 8 ? id_at<int64_t>(ids, t) : id_at<int32_t>(ids, t);
}

// K units a thread: their ids, then their rows' units are on their way together.
template <typename T, int K>
__global__ __launch_bounds__(EM_NT) void embed_forward_kernel(const void* ids, int32_t id_bytes, int64_t tokens,
                                                              const T* table, int64_t rows, int64_t row_stride,
                                                              int64_t width, uint32_t units, float scale, T* out) {
    const uint64_t total = (uint64_t)tokens * units;
    for (uint64_t i0 = (uint64_t)blockIdx.x * (EM_NT * K); i0 < total; i0 += (uint64_t)gridDim.x * (EM_NT * K)) {
        const uint64_t t0 = i0 / units;   // the first token; the others by 32-bit steps from it
        const uint32_t u0 = (uint32_t)(i0 - t0 * units) + threadIdx.x;
        int64_t t[K], id[K];
        uint32_t u[K];
        u32x4 r[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const uint32_t at = u0 + k * EM_NT, step = at / units;
            t[k] = (int64_t)(t0 + step);
            u[k] = at - step * units;
            id[k] = t[k] < tokens ? load_id(ids, id_bytes, t[k]) : -1;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            r[k] = u32x4{0, 0, 0, 0};
            if (id[k] >= 0 && id[k] < rows) r[k] = load_unit(table + id[k] * row_stride, u[k], width);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (t[k] >= tokens) continue;
            const bool there = id[k] >= 0 && id[k] < rows;
            float v[Unit<T>::n];
            widen<T>(r[k], v);
#pragma unroll
            for (int e = 0; e < Unit<T>::n; ++e) v[e] = there ? v[e] * scale : 0.0f;   // a scale may be infinite
            store_unit(out + t[k] * width, u[k], width, narrow<T>(v));
        }
    }
}

// ---------------------------------------------------------------------------
// Stable sort of (id, token) by id.
//
// A tile of 1024 R keys is ranked by one workgroup, least significant digit
// first: each wave takes a contiguous part, 64 keys a round, finds the lanes
// with its key's digit by one ballot per digit bit, and keeps a running count
// per digit in LDS.  Up to 32 tiles of 1024 are sorted side by side and then
// merged in one step: a key's place is its own in its tile plus, for each other
// tile, the number of keys there that go before it, by binary search in LDS
// (which holds all tiles: 128 KB at 32).  More tokens go through one counting
// sort per digit, in tiles of 4096.  Ids of 15 bits, merged or in two passes of
// three kernels: 16384 tokens 15 us or 36, 32768 22 us or 37.
// ---------------------------------------------------------------------------
template <int R> struct SortTile {
    uint32_t key[SO_NT * R];
    uint16_t from[SO_NT * R];
    uint32_t count[SO_WAVES][SO_DIGITS];   // per wave and digit; then the first place of each
    uint32_t scan[SO_DIGITS / kWave];
};

__device__ __forceinline__ uint32_t digit_of(uint32_t key, int shift) { return (key >> shift) & (SO_DIGITS - 1); }

// Ranks the keys of a wave's part among the wave's keys of the same digit.
// Thread-held: key[r], rank[r] for round r; `mine` keys in this wave's part.
template <int R>
__device__ __forceinline__ void rank_wave(SortTile<R>& s, const uint32_t (&key)[R], uint32_t (&rank)[R], int mine, int shift) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int d = lane; d < SO_DIGITS; d += kWave) s.count[wave][d] = 0;
    __builtin_amdgcn_wave_barrier();
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int r = 0; r < R; ++r) {
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
template <int R> __device__ __forceinline__ void scan_counts(SortTile<R>& s) {
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

// Sorts each SO_NT tokens.  The last tile is filled up with the largest number.
__global__ __launch_bounds__(SO_NT) void embed_sort_tile_kernel(const void* ids, int32_t id_bytes, int32_t tokens,
                                                                int64_t rows, int32_t bits, uint32_t* sorted_ids,
                                                                uint32_t* sorted_tokens) {
    __shared__ SortTile<1> s;
    const int t0 = blockIdx.x * SO_NT, n = min(SO_NT, tokens - t0);
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int first, mine;
    wave_part(n, wave, first, mine);
    const bool on = lane < mine;
    uint32_t key[1] = {on ? key_of(ids, id_bytes, t0 + first + lane, rows) : 0}, rank[1] = {0}, from = first + lane;
    for (int shift = 0; shift < bits; shift += SO_BITS) {
        rank_wave(s, key, rank, mine, shift);
        __syncthreads();
        scan_counts(s);
        if (on) {
            const uint32_t at = s.count[wave][digit_of(key[0], shift)] + rank[0];
            s.key[at] = key[0];
            s.from[at] = (uint16_t)from;
        }
        __syncthreads();
        if (on) {
            key[0] = s.key[first + lane];
            from = s.from[first + lane];
        }
    }
    // one wave's part after another, filled up behind the last key
    const int i = threadIdx.x;
    sorted_ids[t0 + i] = i < n ? s.key[i] : ~0u;
    sorted_tokens[t0 + i] = i < n ? (uint32_t)t0 + s.from[i] : 0u;
}
// The place of each key of a sorted tile among all tiles.
__global__ __launch_bounds__(SO_NT) void embed_merge_kernel(const uint32_t* ids, const uint32_t* from, int32_t tokens, int32_t tiles,
                                                            uint32_t* sorted_ids, uint32_t* sorted_tokens) {
    extern __shared__ __align__(16) uint32_t keys[];   // [tiles][SO_NT]
    const int mine = blockIdx.x, i = threadIdx.x, t = mine * SO_NT + i;
    for (int c = 0; c < tiles; ++c) keys[c * SO_NT + i] = ids[c * SO_NT + i];
    __syncthreads();
    if (t >= tokens) return;
    const uint32_t key = keys[t], token = from[t];
    uint32_t place = i;
#pragma unroll 4
    for (int c = 0; c < tiles; ++c) {
        // of the tiles before, equal keys go before, too: keys < key + 1
        const uint32_t bound = c < mine ? key + 1 : key;
        const uint32_t* k = keys + c * SO_NT;
        uint32_t n = 0;
#pragma unroll
        for (int step = SO_NT / 2; step >= 1; step /= 2) n += k[n + step - 1] < bound ? step : 0;
        n += k[n] < bound;
        place += c == mine ? 0 : n;
    }
    sorted_ids[place] = key;
    sorted_tokens[place] = token;
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
    __shared__ SortTile<SO_ROUNDS> s;
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

// A wave takes a chunk and a column tile of 64 units.  The rows' loads wait for
// nothing but the list, which lies in the lanes, and eight of them are on
// their way together (2777 x 768 fp32: 29 us, with four 34).  The fill uses
// ordinary stores (nontemporal ones: 93 us instead of 83 for 16384 x 4096).
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
    for (uint32_t i0 = 0; i0 < n; i0 += EM_AHEAD) {
        u32x4 raw[EM_AHEAD];
#pragma unroll
        for (uint32_t k = 0; k < EM_AHEAD; ++k) {
            raw[k] = u32x4{0, 0, 0, 0};
            if (i0 + k < n && (uint32_t)__builtin_amdgcn_readlane(my_id, i0 + k) < a.rows)
                raw[k] = load_unit(grad + (int64_t)__builtin_amdgcn_readlane(my_from, i0 + k) * a.grad_stride, unit, a.width);
        }
#pragma unroll
        for (uint32_t k = 0; k < EM_AHEAD; ++k) {
            if (i0 + k >= n) break;
            const uint32_t v = __builtin_amdgcn_readlane(my_id, i0 + k);
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
                widen<T>(raw[k], g);
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] += g[e];
            }
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
    uint32_t chunks, tiles;
    uint32_t merge_tiles, count_tiles;   // of the sort: tiles of SO_NT, or of SO_TILE if there are too many of those
};
EmbedLayout embed_layout(int64_t tokens, int64_t width, int32_t dtype) {
    EmbedLayout o{};
    const int64_t e = dtype == CRESSO_F32 ? 4 : 8;
    o.chunks = (uint32_t)((tokens + EM_CHUNK - 1) / EM_CHUNK);
    o.tiles = (uint32_t)((width + kWave * e - 1) / (kWave * e));
    o.merge_tiles = (uint32_t)((tokens + SO_NT - 1) / SO_NT);
    if (o.merge_tiles > SO_MERGE) {
        o.merge_tiles = 0;
        o.count_tiles = (uint32_t)((tokens + SO_TILE - 1) / SO_TILE);
    }
    int64_t off = 0;
    auto take = [&](int64_t b) { const int64_t at = off; off = al256(off + b); return at; };
    const int64_t held = std::max<int64_t>(tokens, (int64_t)o.merge_tiles * SO_NT);   // tiles are filled up
    o.ids = take(held * 4);
    o.tokens = take(held * 4);
    if (o.merge_tiles != 1 && tokens > 0) {
        o.ids2 = take(held * 4);
        o.tokens2 = take(held * 4);
    }
    if (o.count_tiles) o.places = take((int64_t)SO_DIGITS * o.count_tiles * 4);
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
        // four units a thread once that leaves enough workgroups for all CUs
        // (16384 x 4096 bf16 43 us, 46 with one; 512 x 2048 4.9, 4.2 with one)
        const int64_t total = tokens * units;
        const auto go = [&](auto kernel, int k) {
            const int64_t blocks = std::min<int64_t>((total + EM_NT * k - 1) / (EM_NT * k), EM_MAX_BLOCKS);
            hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(EM_NT), 0, (hipStream_t)stream, ids, id_bytes, tokens, (const T*)table,
                               rows, row_stride, width, units, (float)scale, (T*)out);
        };
        if (total >= (int64_t)EM_NT * 4 * 1024) go(embed_forward_kernel<T, 4>, 4);
        else go(embed_forward_kernel<T, 1>, 1);
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
    if (!row_stride_ok(grad, tokens, width, grad_stride)) return fail(CRESSO_E_INVALID, "embedding gradient: row stride below the width");
    const EmbedLayout o = embed_layout(tokens, width, dtype);
    if (!workspace || workspace_bytes < (size_t)o.total || ((uintptr_t)workspace & 15))
        return fail(CRESSO_E_INVALID, "embedding gradient: workspace of %zu bytes at %p, %lld at a multiple of 16 needed", workspace_bytes,
                    workspace, (long long)o.total);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    uint32_t *sid = (uint32_t*)(ws + o.ids), *sfrom = (uint32_t*)(ws + o.tokens);
    int bits = 1;   // of the largest key, `rows`
    while (((int64_t)1 << bits) <= rows) ++bits;
    uint32_t *a_ids = sid, *a_tok = sfrom, *b_ids = (uint32_t*)(ws + o.ids2), *b_tok = (uint32_t*)(ws + o.tokens2);
    if (o.merge_tiles) {
        hipLaunchKernelGGL(embed_sort_tile_kernel, dim3(o.merge_tiles), dim3(SO_NT), 0, st, ids, id_bytes, (int32_t)tokens, rows, bits,
                           a_ids, a_tok);
        if (o.merge_tiles > 1) {
            hipLaunchKernelGGL(embed_merge_kernel, dim3(o.merge_tiles), dim3(SO_NT), o.merge_tiles * SO_NT * 4, st, a_ids, a_tok,
                               (int32_t)tokens, (int32_t)o.merge_tiles, b_ids, b_tok);
            sid = b_ids;
            sfrom = b_tok;
        }
    } else if (o.count_tiles) {
        SortPass p{};
        p.ids = ids;
        p.places = (uint32_t*)(ws + o.places);
        p.tokens = tokens;
        p.rows = rows;
        p.tiles = o.count_tiles;
        p.id_bytes = id_bytes;
        for (p.shift = 0; p.shift < bits; p.shift += SO_BITS) {
            p.first_pass = p.shift == 0;
            p.in_ids = a_ids;
            p.in_tokens = a_tok;
            p.out_ids = b_ids;
            p.out_tokens = b_tok;
            hipLaunchKernelGGL(embed_sort_count_kernel, dim3(o.count_tiles), dim3(SO_NT), 0, st, p);
            hipLaunchKernelGGL(embed_sort_scan_kernel, dim3(1), dim3(SO_NT), 0, st, p.places, (size_t)SO_DIGITS * o.count_tiles);
            hipLaunchKernelGGL(embed_sort_move_kernel, dim3(o.count_tiles), dim3(SO_NT), 0, st, p);
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
