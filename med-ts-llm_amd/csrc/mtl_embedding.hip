// Token table: lookup with scaling (mtl_embedding_fwd) and the table's gradient (mtl_embedding_bwd).
//
//   out[i, :]  = s table[id_i, :]
//   grad[v, :] = s sum over {i : id_i = v} dout[i, :]
//
// Both are HBM-bound (one multiply or add per element moved). The gradient is a scatter-add; atomics would make it depend on the order in which workgroups run, so
// the tokens are first SORTED by id (stable least-significant-digit radix sort of (id, position)) and every table row is then summed in position order:
//   1. sort: up to 8192 tokens in ONE workgroup's LDS, more in tiles of 4096 (two launches per digit: count, scatter). The dense gradient's zero rows are written by the other
//      workgroups of the first launch: the fill (V d elements, most of the traffic for a large vocabulary) hides the sort.
//   2. sum: a wave owns a WINDOW of consecutive sorted tokens and a chunk of columns, walks the window with the running sum of the current id in registers and writes a row
//      whenever the id changes: balanced whatever the distribution of the ids is, and no list of runs is needed. A run that crosses a window border leaves an fp32 partial per window
//      (one slot for a run that came in, one for a run that goes out).
//   3. join: the windows in which a crossing run starts have put themselves on a list; each such run's partials are added in window order.
#include "mtl_common.h"

namespace {

// Tokens that one workgroup sorts in its LDS: 4096 14 us, 8192 24 us (16 keys per thread spill: 16384 tokens 117 us, against 29 us and three more launches in tiles).
constexpr int SORT_MAX = 8192;
constexpr int TILE = 4096;               // tokens per workgroup of the tiled sort
constexpr int JOIN_SHORT = 16;           // windows behind its first one up to which a crossing run is joined by one wave
constexpr unsigned SELF_TILES = 256;     // tiles up to which each sums all tiles' counts itself
constexpr int MAX_BINS = 512;            // digits of up to 9 bits: two passes for every vocabulary up to 262143

// ---------------------------------------------------------------- element access
// Vectors of up to 16 bytes at any element's address (global accesses need no more alignment than their type's elements have): rows of odd width take the same path as others. A
// lane whose W columns would reach beyond the row starts earlier instead (Cols) and computes the columns it shares with its neighbour a second time: the same bits.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

// W consecutive elements as loaded: held like this until they are used, so that many rows are in flight in few registers
template <typename T, int W>
struct Raw {
    static constexpr int WORDS = (W * (int)sizeof(T) + 3) / 4;
    uint32_t w[WORDS];
    template <bool STREAM, typename V>
    static __device__ __forceinline__ V get(const void* p) {
        const V* v = reinterpret_cast<const V*>(p);
        return STREAM ? __builtin_nontemporal_load(v) : *v;
    }
    // STREAM: read once, past the caches
    template <bool STREAM>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (sizeof(T) * W >= 16) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const u32x4_any v = get<STREAM, u32x4_any>(reinterpret_cast<const uint32_t*>(p) + i);
                w[i] = v[0]; w[i + 1] = v[1]; w[i + 2] = v[2]; w[i + 3] = v[3];
            }
        } else if constexpr (sizeof(T) * W == 8) {
            const u32x2_any v = get<STREAM, u32x2_any>(p);
            w[0] = v[0]; w[1] = v[1];
        } else if constexpr (sizeof(T) == 4) w[0] = get<STREAM, uint32_t>(p);
        else w[0] = get<STREAM, uint16_t>(p);
    }
    __device__ __forceinline__ float at(int j) const {
        if (sizeof(T) == 4) return __uint_as_float(w[j]);
        return __uint_as_float((j & 1) ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    }
};
template <typename T, int W>
__device__ __forceinline__ void load_w(const T* p, float (&x)[W]) {
    Raw<T, W> r;
    r.template load<false>(p);
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = r.at(j);
}
__device__ __forceinline__ void store_1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_1(bf16_t* p, float x) { *p = f32_to_bf16(x); }
template <typename T, int W>
__device__ __forceinline__ void store_w(T* p, const float (&x)[W]) {
    if constexpr (W == 1) store_1(p, x[0]);
    else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < W; j += 4)
            *reinterpret_cast<u32x4_any*>(p + j) = (u32x4_any){__float_as_uint(x[j]), __float_as_uint(x[j + 1]), __float_as_uint(x[j + 2]), __float_as_uint(x[j + 3])};
    } else if constexpr (W == 4) *reinterpret_cast<u32x2_any*>(p) = (u32x2_any){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    else *reinterpret_cast<u32x4_any*>(p) = (u32x4_any){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

// a lane's columns at .. at + W - 1 of a row of d >= W; the first `skip` of them are its neighbour's as well; not `in`: it has none (and reads the row's first)
struct Cols { int64_t at; int skip; bool in; };
template <int W>
__device__ __forceinline__ Cols cols_of(int64_t c, int64_t d) {
    Cols k;
    k.in = c < d;
    k.at = !k.in ? 0 : (c <= d - W ? c : d - W);
    k.skip = k.in ? (int)(c - k.at) : 0;
    return k;
}

__device__ __forceinline__ int64_t load_id(const void* ids, int ids_i64, int64_t i) {
    return ids_i64 ? reinterpret_cast<const int64_t*>(ids)[i] : (int64_t)reinterpret_cast<const int32_t*>(ids)[i];
}

// ---------------------------------------------------------------- lookup
// rows narrower than a wave: 64 / LPR rows per wave (LPR lanes per row, W columns per lane and step)
template <typename TT, typename OT, int W>
__global__ __launch_bounds__(256) void embedding_fwd_narrow_kernel(const void* __restrict__ ids, int ids_i64, int64_t N, const TT* __restrict__ table, int64_t V, int64_t d, int64_t ld_table,
                                                                   float scale, OT* __restrict__ out, int64_t ld_out, int lpr_log2) {
    const int lpr = 1 << lpr_log2;
    const int rows_per_block = 256 >> lpr_log2;
    const Cols k = cols_of<W>((int64_t)(threadIdx.x & (lpr - 1)) * W, d);
    if (!k.in) return;
    for (int64_t i = (int64_t)blockIdx.x * rows_per_block + (threadIdx.x >> lpr_log2); i < N; i += (int64_t)gridDim.x * rows_per_block) {
        const int64_t id = load_id(ids, ids_i64, i);
        const bool in = id >= 0 && id < V;
        float x[W];
        load_w<TT, W>(table + (in ? id : 0) * ld_table + k.at, x);
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = in ? x[j] * scale : 0.f;
        store_w<OT, W>(out + i * ld_out + k.at, x);
    }
}

// a wave owns ROWS consecutive tokens and walks their columns: ROWS loads are in flight per step. `split` > 1: a row's columns are spread over that many waves.
template <typename TT, typename OT, int W, int ROWS>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* __restrict__ ids, int ids_i64, int64_t N, const TT* __restrict__ table, int64_t V, int64_t d, int64_t ld_table, float scale,
                                                            OT* __restrict__ out, int64_t ld_out, int split) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t group = item / split;
    const int64_t i0 = group * ROWS;
    if (i0 >= N) return;
    const int n = N - i0 < ROWS ? (int)(N - i0) : ROWS;
    int64_t mine = -1;
    if (lane < n) mine = load_id(ids, ids_i64, i0 + lane);
    const int lo = (int)mine, hi = (int)(mine >> 32);
    const TT* src[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int64_t id = (int64_t)(uint32_t)__builtin_amdgcn_readlane(lo, r) | ((int64_t)__builtin_amdgcn_readlane(hi, r) << 32);
        const bool in = id >= 0 && id < V;
        src[r] = in ? table + id * ld_table : nullptr;
    }
    for (int64_t c = ((item - group * split) * 64 + lane) * W; c < d; c += (int64_t)64 * W * split) {
        const int64_t at = cols_of<W>(c, d).at;
        Raw<TT, W> x[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (src[r]) x[r].template load<false>(src[r] + at);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (r >= n) break;
            float y[W];
#pragma unroll
            for (int j = 0; j < W; ++j) y[j] = src[r] ? x[r].at(j) * scale : 0.f;
            store_w<OT, W>(out + (i0 + r) * ld_out + at, y);
        }
    }
}

// ---------------------------------------------------------------- zero rows of the dense gradient
// rows of row_bytes each, ld_bytes apart (one row where the gradient is contiguous), stores of `width` (16, 4 or 2) bytes and a row's last ones of 2. A contiguous gradient of 144 MiB and more
// (`once`): one store per thread and workgroups that end with it, so that the chip writes one narrow front of addresses, in which each of eight neighbouring workgroups (of eight XCDs) has every eighth
// 4 KB. 2.1 GB with the sort and sum of 1 / 8192 tokens: 310 / 362 us (torch's fill alone 308); 16 KB in a row per workgroup 335 / 387, runs of 1, 2, 8 KB 315 / 366, 342 / 400, 340 / 385; four stores
// per thread from 512 workgroups 377 / 423. 154 MB 26.5 / 41.2 against 28.5 / 42.0, 134 MB 26.8 / 42.5 against 26.2 / 42.5. Non-temporal stores spare the sum behind them the eviction of dirty lines and take that longer themselves.
struct Fill { char* p; int64_t rows, row_bytes, ld_bytes; int width; bool once; };

__device__ __forceinline__ void fill_zero(const Fill& f, int64_t block, int64_t blocks) {
    const u32x4 zero = {0, 0, 0, 0};
    const bool flat = f.rows == 1;
    if (f.once) {                                                // (flat, 16 bytes wide; blocks: a multiple of 8 that covers the row)
        const int64_t i = (((block >> 3) * 4 + (threadIdx.x >> 8)) * 8 + (block & 7)) * 256 + (threadIdx.x & 255), n = f.row_bytes / 16, tail = n * 16 + threadIdx.x * 2;
        if (i < n) reinterpret_cast<u32x4*>(f.p)[i] = zero;
        if (block == 0 && tail < f.row_bytes) *reinterpret_cast<uint16_t*>(f.p + tail) = 0;
        return;
    }
    for (int64_t r = flat ? 0 : block; r < f.rows; r += flat ? 1 : blocks) {
        char* row = f.p + r * f.ld_bytes;
        const int64_t n = f.row_bytes / f.width, first = flat ? block * 4096 : 0, step = flat ? blocks * 4096 : 4096;      // (1024 threads, four stores each)
        for (int64_t i = first + threadIdx.x; i < n; i += step) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = i + u * 1024;
                if (at >= n) break;
                if (f.width == 16) reinterpret_cast<u32x4*>(row)[at] = zero;
                else if (f.width == 4) reinterpret_cast<uint32_t*>(row)[at] = 0;
                else reinterpret_cast<uint16_t*>(row)[at] = 0;
            }
        }
        const int64_t tail = n * f.width + threadIdx.x * 2;
        if ((!flat || block == 0) && tail < f.row_bytes) *reinterpret_cast<uint16_t*>(row + tail) = 0;
    }
}

// ---------------------------------------------------------------- sort
// key of a token: its id, or V (sorted behind every row) where it has no gradient
__device__ __forceinline__ uint32_t token_key(const void* ids, int ids_i64, int64_t i, int64_t V, int64_t pad) {
    const int64_t id = load_id(ids, ids_i64, i);
    return (id >= 0 && id < V && id != pad) ? (uint32_t)id : (uint32_t)V;
}

// 1024 threads rank E keys each by the digit (key >> shift) & (2^bits - 1): element (wave, e, lane) precedes (wave, e', lane') in that order, and the rank counts the elements of
// smaller digit plus the preceding ones of the same digit (stable). cnt: LDS [16][MAX_BINS]. On return cnt[w][dgt] = first rank of wave w's elements of digit dgt and rank[e] =
// the element's rank among its wave's elements of its digit. Lanes beyond the data (valid bit clear) take part in nothing.
template <int E>
__device__ __forceinline__ void rank_digits(const uint32_t (&key)[E], uint32_t valid, int shift, int bits, uint32_t* cnt, uint32_t (&rank)[E], int n_e) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t mask = (1u << bits) - 1u;
    for (int i = threadIdx.x; i < 16 * MAX_BINS; i += 1024) cnt[i] = 0;
    __syncthreads();
    uint32_t* mine = cnt + wave * MAX_BINS;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (e < n_e) {                                        // (uniform)
            const bool ok = (valid >> e) & 1u;
            const uint32_t dgt = (key[e] >> shift) & mask;
            uint64_t peers = __ballot(ok);
            for (int b = 0; b < bits; ++b) {
                const bool one = (dgt >> b) & 1u;
                const uint64_t with = __ballot(one);
                peers &= one ? with : ~with;
            }
            const uint64_t below = peers & ((1ull << lane) - 1ull);
            uint32_t first = 0;
            if (ok) first = mine[dgt];
            __builtin_amdgcn_wave_barrier();                  // every peer has read the counter before its first lane moves it (LDS accesses of a wave keep their order)
            rank[e] = first + (uint32_t)__popcll(below);
            if (ok && below == 0) mine[dgt] = first + (uint32_t)__popcll(peers);
            __builtin_amdgcn_wave_barrier();
        }
    }
    __syncthreads();
}

// exclusive prefix sum of one value per thread over 1024 threads; tot: LDS [16]. Returns the prefix; every thread gets the total.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t* tot, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(s, o, 64);
        if (lane >= o) s += up;
    }
    if (lane == 63) tot[wave] = s;
    __syncthreads();
    uint32_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const uint32_t x = tot[w];
        if (w < wave) before += x;
        sum += x;
    }
    __syncthreads();
    total = sum;
    return before + s - v;
}

// cnt[16][MAX_BINS] counts -> first ranks, digit major and wave minor: thread t owns digit t / 2, waves 8 (t % 2) .. + 7
__device__ __forceinline__ void scan_counts(uint32_t* cnt, uint32_t* tot) {
    const int dgt = threadIdx.x >> 1, w0 = (threadIdx.x & 1) * 8;
    uint32_t c[8], sum = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) { c[w] = cnt[(w0 + w) * MAX_BINS + dgt]; sum += c[w]; }
    uint32_t total;
    uint32_t at = block_exclusive(sum, tot, total);
#pragma unroll
    for (int w = 0; w < 8; ++w) { cnt[(w0 + w) * MAX_BINS + dgt] = at; at += c[w]; }
    __syncthreads();
}

// workgroup 0 sorts up to 1024 E tokens (E per thread), the others write the zero rows
template <int E>
__global__ __launch_bounds__(1024) void embedding_sort_small_kernel(const void* __restrict__ ids, int ids_i64, int N, int64_t V, int64_t pad, int passes, int bits, uint32_t* __restrict__ sid,
                                                                    uint32_t* __restrict__ spos, uint32_t* __restrict__ list_n, const Fill f) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    if (blockIdx.x > 0) {
        fill_zero(f, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    uint32_t* cnt = reinterpret_cast<uint32_t*>(smem);                       // [16][MAX_BINS]
    uint32_t* lkey = cnt + 16 * MAX_BINS;                                    // [max(N, 16)]
    uint32_t* tot = lkey;                                                    // [16]: in use between the keys' reading and the next writing of them only
    uint16_t* lpos = reinterpret_cast<uint16_t*>(lkey + (N > 16 ? N : 16)); // [N]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n_e = (N + 1023) >> 10;                                        // elements per thread: wave w owns [w n_e 64, (w + 1) n_e 64)
    const int i0 = wave * n_e * 64 + lane;
    const uint32_t mask = (1u << bits) - 1u;
    if (threadIdx.x < 2) list_n[threadIdx.x] = 0;
    uint32_t key[E], rank[E], valid = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        key[e] = 0;
        const int i = i0 + e * 64;
        if (e < n_e && i < N) { key[e] = token_key(ids, ids_i64, i, V, pad); valid |= 1u << e; }
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * bits;
        rank_digits<E>(key, valid, shift, bits, cnt, rank, n_e);
        scan_counts(cnt, tot);
        uint32_t pos[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            pos[e] = (uint32_t)(i0 + e * 64);
            if (p > 0 && ((valid >> e) & 1u)) pos[e] = lpos[i0 + e * 64];
        }
        __syncthreads();
        const bool last = p == passes - 1;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if ((valid >> e) & 1u) {
                const uint32_t at = cnt[wave * MAX_BINS + ((key[e] >> shift) & mask)] + rank[e];
                if (last) { sid[at] = key[e]; spos[at] = pos[e]; }
                else { lkey[at] = key[e]; lpos[at] = (uint16_t)pos[e]; }
            }
        if (last) break;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e)
            if ((valid >> e) & 1u) key[e] = lkey[i0 + e * 64];
    }
}

// tiled sort, digit counts of each tile: hist[tile][digit]. Workgroups behind the last tile write the zero rows.
__global__ __launch_bounds__(1024) void embedding_sort_count_kernel(const void* __restrict__ ids, int ids_i64, int64_t N, int64_t V, int64_t pad, const uint32_t* __restrict__ keys, int shift, int bits,
                                                                    int tiles, uint32_t* __restrict__ hist, uint32_t* __restrict__ list_n, const Fill f) {
    if ((int)blockIdx.x >= tiles) {
        fill_zero(f, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    __shared__ uint32_t cnt[MAX_BINS];
    if (list_n && blockIdx.x == 0 && threadIdx.x < 2) list_n[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < MAX_BINS; i += 1024) cnt[i] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < TILE / 1024; ++e) {
        const int64_t i = (int64_t)blockIdx.x * TILE + e * 1024 + threadIdx.x;
        if (i < N) {
            const uint32_t k = keys ? keys[i] : token_key(ids, ids_i64, i, V, pad);
            atomicAdd(&cnt[(k >> shift) & ((1u << bits) - 1u)], 1u);           // (a count: the order of the additions does not show)
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (1 << bits); i += 1024) hist[((int64_t)blockIdx.x << bits) + i] = cnt[i];
}

// More than SELF_TILES tiles: hist[tile][digit] becomes the number of the digit's tokens in earlier tiles, totals[digit] all of them. A workgroup per 64 digits, 16 waves over the tiles.
__global__ __launch_bounds__(1024) void embedding_sort_scan_kernel(uint32_t* __restrict__ hist, int tiles, int bits, uint32_t* __restrict__ totals) {
    __shared__ uint32_t sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dgt = blockIdx.x * 64 + lane;
    const bool in = dgt < (1 << bits);
    const int t0 = (int)((int64_t)tiles * wave / 16), t1 = (int)((int64_t)tiles * (wave + 1) / 16);
    uint32_t s = 0;
    if (in) {
#pragma unroll 8
        for (int t = t0; t < t1; ++t) s += hist[((int64_t)t << bits) + dgt];
    }
    sums[wave][lane] = s;
    __syncthreads();
    uint32_t at = 0;
    for (int w = 0; w < wave; ++w) at += sums[w][lane];
    if (!in) return;
    if (wave == 15) totals[dgt] = at + s;
    for (int t = t0; t < t1; t += 8) {
        uint32_t h[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) h[u] = t + u < t1 ? hist[((int64_t)(t + u) << bits) + dgt] : 0u;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (t + u < t1) hist[((int64_t)(t + u) << bits) + dgt] = at;
            at += h[u];
        }
    }
}

// The first rank of a tile's elements of every digit: tokens of smaller digits plus those of the same digit in earlier tiles. Up to SELF_TILES tiles each tile sums them up itself from
// all tiles' counts (totals == NULL); above that the work would grow with the square of the tiles, and the scan kernel has done it. Per digit of 50257 ids, scan + scatter against
// scatter alone: 100 000 tokens 15.1 / 12.1 us, 400 000 17.2 / 13.9, 1 M 22.5 / 20.9, 2 M 33 / 41, and a launch.
__global__ __launch_bounds__(1024) void embedding_sort_scatter_kernel(const void* __restrict__ ids, int ids_i64, int64_t N, int64_t V, int64_t pad, const uint32_t* __restrict__ keys,
                                                                      const uint32_t* __restrict__ poss, int shift, int bits, int tiles, const uint32_t* __restrict__ hist,
                                                                      const uint32_t* __restrict__ totals, uint32_t* __restrict__ sid, uint32_t* __restrict__ spos) {
    __shared__ uint32_t cnt[16 * MAX_BINS];
    __shared__ uint32_t sums[2 * 1024];
    __shared__ uint32_t tot[16];
    constexpr int E = TILE / 1024;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t key[E], pos[E], rank[E], valid = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int64_t i = (int64_t)blockIdx.x * TILE + (wave * E + e) * 64 + lane;
        key[e] = 0; pos[e] = 0;
        if (i < N) {
            key[e] = keys ? keys[i] : token_key(ids, ids_i64, i, V, pad);
            pos[e] = keys ? poss[i] : (uint32_t)i;
            valid |= 1u << e;
        }
    }
    // counts of digit threadIdx.x % bins: over every `groups`-th tile, all of them and the earlier ones
    const int bins = 1 << bits, groups = 1024 >> bits, dgt = threadIdx.x & (bins - 1);
    uint32_t all = 0, earlier = 0;
    if (totals) {
        if ((int)threadIdx.x < bins) { all = totals[dgt]; earlier = hist[((int64_t)blockIdx.x << bits) + dgt]; }
    } else {
#pragma unroll 8
        for (int t = threadIdx.x >> bits; t < tiles; t += groups) {
            const uint32_t h = hist[((int64_t)t << bits) + dgt];
            all += h;
            earlier += t < (int)blockIdx.x ? h : 0u;
        }
    }
    sums[threadIdx.x] = all;
    sums[1024 + threadIdx.x] = earlier;
    rank_digits<E>(key, valid, shift, bits, cnt, rank, E);
    all = earlier = 0;
    if ((int)threadIdx.x < bins)
        for (int g = 0; g < groups; ++g) { all += sums[g * bins + threadIdx.x]; earlier += sums[1024 + g * bins + threadIdx.x]; }
    uint32_t total;
    uint32_t at = block_exclusive(all, tot, total) + earlier;
    if ((int)threadIdx.x < bins) {
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const uint32_t c = cnt[w * MAX_BINS + threadIdx.x];
            cnt[w * MAX_BINS + threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if ((valid >> e) & 1u) {
            const uint32_t to = cnt[wave * MAX_BINS + ((key[e] >> shift) & (bins - 1))] + rank[e];
            sid[to] = key[e];
            spos[to] = pos[e];
        }
}

// ---------------------------------------------------------------- sum over windows
struct SumArgs {
    const uint32_t* sid; const uint32_t* spos;
    int64_t N, V, d, ld_dout, ld_grad;
    const void* dout; void* grad;
    float* part;                 // [windows][2][d]: 0 = the run that came into the window, 1 = the run that goes out of it (and started in it)
    uint32_t* list; uint32_t* list_n;      // [windows]: short runs from the front, long ones from the back; their two counts
    float scale;
    int accumulate, S, chunks;
    int64_t windows;
};

template <typename GT, int W>
__device__ __forceinline__ void write_row(const SumArgs& a, uint32_t id, const Cols& k, const float (&acc)[W]) {
    GT* to = reinterpret_cast<GT*>(a.grad) + (int64_t)id * a.ld_grad + k.at;
    float y[W];
#pragma unroll
    for (int j = 0; j < W; ++j) y[j] = acc[j] * a.scale;
    if (a.accumulate) {
        if (W > 1 && k.skip) {                                  // columns shared with a neighbour are added once: by it
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (j >= k.skip) {
                    float old[1];
                    load_w<GT, 1>(to + j, old);
                    store_1(to + j, y[j] + old[0]);
                }
            return;
        }
        float old[W];
        load_w<GT, W>(to, old);
#pragma unroll
        for (int j = 0; j < W; ++j) y[j] += old[j];
    }
    store_w<GT, W>(to, y);
}

// dout is read once and past the caches: 200 003 rows of 2 KB 94 us, through the caches 133 (the loads evict what the launches before left dirty there).
// A wave holds its window's ids and positions in its lanes (one load each), picks them by lane number, and keeps two groups of GROUP rows: one being added, the next one in flight.
template <typename DT, typename GT, int W>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const SumArgs a) {
    constexpr int GROUP = 8;
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = item / a.chunks;
    if (w >= a.windows) return;
    const int64_t chunk = item - w * a.chunks;
    const Cols k = cols_of<W>(chunk * (64 * W) + lane * W, a.d);
    const int64_t i0 = w * a.S, i1 = i0 + a.S < a.N ? i0 + a.S : a.N;
    const uint32_t none = (uint32_t)a.V;
    uint32_t ids = none, poss = 0;
    if (i0 + lane < i1) { ids = a.sid[i0 + lane]; poss = a.spos[i0 + lane]; }
    const uint32_t before = i0 > 0 ? a.sid[i0 - 1] : none, after = i1 < a.N ? a.sid[i1] : none;
    const int n = (int)__popcll(__ballot(ids != none));         // (sorted: the tokens without a gradient are the last ones)
    if (n == 0) return;
    const DT* dout = reinterpret_cast<const DT*>(a.dout) + k.at;
    uint32_t cur = (uint32_t)__builtin_amdgcn_readlane((int)ids, 0);
    bool came_in = before == cur;
    float acc[W];
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j] = 0.f;
    float* part = a.part + w * 2 * a.d + k.at;
    Raw<DT, W> now[GROUP], next[GROUP];
    auto fetch = [&](Raw<DT, W>(&x)[GROUP], int i) {
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            const int at = i + u < n ? i + u : n - 1;            // (beyond the end: the last token again, not used)
            x[u].template load<true>(dout + (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)poss, at) * a.ld_dout);
        }
    };
    auto add = [&](const Raw<DT, W>(&x)[GROUP], int i) {
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            if (i + u >= n) break;
            const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)ids, i + u);
            if (id != cur) {                                     // (uniform) the run of `cur` ends here, inside the window
                if (k.in) {
                    if (came_in) store_w<float, W>(part, acc);
                    else write_row<GT, W>(a, cur, k, acc);
                }
                cur = id;
                came_in = false;
#pragma unroll
                for (int j = 0; j < W; ++j) acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < W; ++j) acc[j] += x[u].at(j);
        }
    };
    fetch(now, 0);
    for (int i = 0; i < n; i += 2 * GROUP) {
        if (i + GROUP < n) fetch(next, i + GROUP);
        add(now, i);
        if (i + GROUP >= n) break;
        if (i + 2 * GROUP < n) fetch(now, i + 2 * GROUP);
        add(next, i + GROUP);
    }
    const bool goes_on = after == cur;
    if (k.in) {
        if (came_in) store_w<float, W>(part, acc);
        else if (goes_on) store_w<float, W>(part + a.d, acc);
        else write_row<GT, W>(a, cur, k, acc);
    }
    // the window in which a crossing run starts goes on a list (whose order shows nowhere: each entry is a whole run): LONG of runs that cover more than JOIN_SHORT windows behind it
    if (goes_on && !came_in && chunk == 0 && lane == 0) {
        const int64_t far = i1 + (int64_t)JOIN_SHORT * a.S;
        if (far < a.N && a.sid[far] == cur) a.list[a.windows - 1 - atomicAdd(a.list_n + 1, 1u)] = (uint32_t)w;
        else a.list[atomicAdd(a.list_n, 1u)] = (uint32_t)w;
    }
}

// number of windows behind w that the run of `id` reaches into, given that it goes on behind w: 64 windows looked at per step
__device__ __forceinline__ int64_t run_windows(const SumArgs& a, int64_t w, uint32_t id) {
    const int lane = threadIdx.x & 63;
    for (int64_t n = 1;; n += 64) {
        const int64_t end = (w + n + lane + 1) * a.S;             // does the run go on behind window w + n + lane?
        const uint64_t stops = __ballot(!(end < a.N && a.sid[end] == id));
        if (stops) return n + __ffsll((unsigned long long)stops) - 1;
    }
}

// The runs that cross window borders: tail partial of the window where the run starts, then the head partials of the following windows, in order. Short runs: a wave each per 256
// columns. Long ones: a workgroup per 64 columns, its 16 waves take a sixteenth of the windows each and are joined in order.
template <typename GT, int W>
__global__ __launch_bounds__(1024) void embedding_join_kernel(const SumArgs a, int long_blocks) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x >= long_blocks) {
        const int chunks = (int)((a.d + 64 * W - 1) / (64 * W));
        const int64_t items = (int64_t)a.list_n[0] * chunks, step = (int64_t)(gridDim.x - long_blocks) * 16;
        for (int64_t item = (int64_t)(blockIdx.x - long_blocks) * 16 + wave; item < items; item += step) {
            const int64_t w = a.list[item / chunks];
            const Cols k = cols_of<W>((item % chunks) * (64 * W) + lane * W, a.d);
            const uint32_t id = a.sid[(w + 1) * a.S];
            const int n = (int)run_windows(a, w, id);
            if (!k.in) continue;
            const float* part = a.part + w * 2 * a.d + k.at;
            float s[W];
            load_w<float, W>(part + a.d, s);
#pragma unroll 4
            for (int i = 1; i <= n; ++i) {
                float x[W];
                load_w<float, W>(part + (int64_t)i * 2 * a.d, x);
#pragma unroll
                for (int j = 0; j < W; ++j) s[j] += x[j];
            }
            write_row<GT, W>(a, id, k, s);
        }
        return;
    }
    const int chunks = (int)((a.d + 63) / 64);
    const int64_t items = (int64_t)a.list_n[1] * chunks;
    for (int64_t item = blockIdx.x; item < items; item += long_blocks) {
        const int64_t w = a.list[a.windows - 1 - item / chunks];
        const int64_t c = (item % chunks) * 64 + lane;
        const bool in = c < a.d;
        const uint32_t id = a.sid[(w + 1) * a.S];
        const int64_t n = run_windows(a, w, id);
        const int64_t k0 = w + 1 + n * wave / 16, k1 = w + 1 + n * (wave + 1) / 16;
        float s = wave == 0 && in ? a.part[w * 2 * a.d + a.d + c] : 0.f;
        if (in) {
#pragma unroll 8
            for (int64_t k = k0; k < k1; ++k) s += a.part[k * 2 * a.d + c];
        }
        sums[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && in) {
            float t[1] = {sums[0][lane]};
#pragma unroll
            for (int v = 1; v < 16; ++v) t[0] += sums[v][lane];
            write_row<GT, 1>(a, id, cols_of<1>(c, a.d), t);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side
inline int bits_for(int64_t V) { int b = 1; while (b < 31 && ((int64_t)1 << b) <= V) ++b; return b; }      // values 0 .. V
inline int passes_for(int64_t V) { return (bits_for(V) + 8) / 9; }
inline int bits_per_pass(int64_t V) { const int p = passes_for(V); return (bits_for(V) + p - 1) / p; }
inline int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// Window length: as long as about 2400 (window, column chunk) waves are left, at most 64 tokens; a longer window writes and joins fewer partial rows (2 / S of the rows read), a shorter one
// shortens the chain of a wave. Gradient as a whole, windows of 8 / 16 / 32 / 64: 2000 x 768 bf16 18.3 / 19.7 / 22.6 / 28.9 us (8 taken); 8192 x 4096 fp32 67 / 63 / 60 / 64 (32);
// 40 000 x 768 bf16 68 / 62 / 58 / 62 (32); 200 003 x 64 bf16 126 / 94 / 74 / 66 (64); 200 003 x 1024 bf16 199 / 160 / 145 / 141 (64).
inline int window_of(int64_t N, int64_t chunks) {
    int s = 8;
    while (s < 64 && N / (2 * s) * chunks >= 2400) s *= 2;
    return s;
}
inline int64_t chunks_of(int64_t d, int W) { return (d + 64 * W - 1) / (64 * W); }

// Four columns per lane; one where a row is narrower than a wave (200 003 x 64 bf16: 65.3 us, with four 67). Eight of bf16 (16 bytes) halve the waves in flight: 8192 x 2048 41.9 us against
// 38.5 with four, 200 003 x 1024 141.5 against 139.9.
inline int columns_of(int64_t d) { return d > 64 ? 4 : 1; }
// ids and positions are 32 bits; the sum is one grid of less than 2^32 threads
inline bool too_large(int64_t N, int64_t V, int64_t d) {
    if (N > 0x7fffffff || V >= 0x7fffffff) return true;
    const int64_t chunks = chunks_of(d, columns_of(d)), S = window_of(N, chunks);
    return chunks >= 1 << 26 || (N + S - 1) / S * chunks > (1 << 26) - 4;      // (four waves per workgroup, and 2^24 workgroups would be 2^32 threads)
}

struct Plan { int64_t sid, spos, sid2, spos2, hist, list, part, total; };
inline Plan plan_for(int64_t N, int64_t V, int64_t d) {
    Plan p;
    int64_t at = 8 + 4 * MAX_BINS;                                // two list counts, the scan's digit totals
    at = up(at, 256);
    auto take = [&](int64_t bytes) { const int64_t here = at; at += up(bytes, 256); return here; };
    const bool small = N <= SORT_MAX;
    const int64_t tiles = (N + TILE - 1) / TILE, windows = (N + 7) / 8;      // (8: the shortest window)
    p.sid = take(4 * N); p.spos = take(4 * N);
    p.sid2 = small ? 0 : take(4 * N); p.spos2 = small ? 0 : take(4 * N);
    p.hist = small ? 0 : take(4 * tiles * MAX_BINS);
    p.list = take(4 * windows);
    // partials: the window length depends on the columns per wave (64 or 256): the longer list of the two
    int64_t most = 0;
    for (int W : {1, 4}) { const int64_t s = window_of(N, chunks_of(d, W)); const int64_t w = (N + s - 1) / s; most = w > most ? w : most; }
    p.part = take(8 * most * d);
    p.total = at;
    return p;
}

template <int E>
void launch_sort_small(const void* ids, int ids_i64, int N, int64_t V, int64_t pad, int passes, int bits, uint32_t* sid, uint32_t* spos, uint32_t* list_n, const Fill& f, unsigned fill_blocks,
                       hipStream_t st) {
    const size_t fixed = 16 * MAX_BINS * 4;                       // (8192 tokens: 80 KB, two workgroups per CU write zeros)
    (void)hipFuncSetAttribute((const void*)embedding_sort_small_kernel<E>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)(fixed + E * 1024 * 6));
    hipLaunchKernelGGL(embedding_sort_small_kernel<E>, dim3(1 + fill_blocks), dim3(1024), fixed + (size_t)(N > 16 ? N : 16) * 6, st, ids, ids_i64, N, V, pad, passes, bits, sid, spos, list_n, f);
}

template <typename DT, typename GT>
void launch_sum(const SumArgs& a, int W, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.windows * a.chunks + 3) / 4);
    if (W == 4) hipLaunchKernelGGL((embedding_sum_kernel<DT, GT, 4>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((embedding_sum_kernel<DT, GT, 1>), dim3(blocks), dim3(256), 0, st, a);
}

template <typename TT, typename OT, int W>
void launch_fwd_w(const void* ids, int ids_i64, int64_t N, const void* table, int64_t V, int64_t d, int64_t ld_table, float scale, void* out, int64_t ld_out, hipStream_t st) {
    if (d <= 32 * W) {
        int lpr = 0;
        while (((int64_t)W << lpr) < d) ++lpr;
        const int64_t rows = 256 >> lpr, want = (N + rows - 1) / rows;
        hipLaunchKernelGGL((embedding_fwd_narrow_kernel<TT, OT, W>), dim3((unsigned)(want < 65536 ? want : 65536)), dim3(256), 0, st, ids, ids_i64, N, (const TT*)table, V, d, ld_table, scale, (OT*)out,
                           ld_out, lpr);
        return;
    }
    // Few tokens: a row's columns go to several waves, up to 8192 in all. 133 x 768 fp32 2.4 us (one wave per row 2.8), 1000 x 4096 5.8 (9.3); up to 16384 waves: 6.4, and 4096 x 768 5.7 against 5.0.
    // A row of more than four waves keeps three or four, one workgroup that writes 4 KB in a row per step: 8192 x 4096 fp32 41.6 us, one wave per row 47; 131 072 x 4096 bf16 297 against 333.
    const int64_t full = (d + 64 * W - 1) / (64 * W);
    int64_t split = full;
    while (split > (full > 4 ? 4 : 1) && N * split > 8192) split = (split + 1) / 2;
    // many tokens of rows up to four waves wide: as many waves as the row has, each with its columns of several rows. 65 536 x 1024 fp32 76.5 us with four rows, 81.9 with two, 91 with one, one wave
    // per row 86; 200 003 x 1024 bf16 115.3 with eight, 119.0 with four, one wave per two rows 119.8; of 1001 columns 137 against 154; below 16 384 tokens the loop above (8192 x 768 fp32 7.6 against 7.7)
    if (full <= 4 && N >= 16384) {
        const int rows = N >= 131072 ? 8 : 4;
        const unsigned blocks = (unsigned)(((N + rows - 1) / rows * full + 3) / 4);
        if (rows == 8) hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, W, 8>), dim3(blocks), dim3(256), 0, st, ids, ids_i64, N, (const TT*)table, V, d, ld_table, scale, (OT*)out, ld_out, (int)full);
        else hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, W, 4>), dim3(blocks), dim3(256), 0, st, ids, ids_i64, N, (const TT*)table, V, d, ld_table, scale, (OT*)out, ld_out, (int)full);
        return;
    }
    hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, W, 1>), dim3((unsigned)((N * split + 3) / 4)), dim3(256), 0, st, ids, ids_i64, N, (const TT*)table, V, d, ld_table, scale, (OT*)out, ld_out, (int)split);
}
template <typename TT, typename OT>
void launch_fwd(const void* ids, int ids_i64, int64_t N, const void* table, int64_t V, int64_t d, int64_t ld_table, float scale, void* out, int64_t ld_out, int W, hipStream_t st) {
    if (W == 8 && sizeof(TT) == 2 && sizeof(OT) == 2) launch_fwd_w<TT, OT, (sizeof(TT) == 2 && sizeof(OT) == 2) ? 8 : 4>(ids, ids_i64, N, table, V, d, ld_table, scale, out, ld_out, st);
    else if (W == 4) launch_fwd_w<TT, OT, 4>(ids, ids_i64, N, table, V, d, ld_table, scale, out, ld_out, st);
    else launch_fwd_w<TT, OT, 1>(ids, ids_i64, N, table, V, d, ld_table, scale, out, ld_out, st);
}

inline bool dtype_ok(int t) { return t == MTL_F32 || t == MTL_BF16; }
inline int size_of(int t) { return t == MTL_BF16 ? 2 : 4; }
}  // namespace

extern "C" int mtl_embedding_fwd(const void* ids, int ids_i64, int64_t N, const void* table, int table_dtype, int64_t V, int64_t d, int64_t ld_table, float scale, void* out, int out_dtype,
                                 int64_t ld_out, void* stream) {
    if (N < 0 || V <= 0 || d <= 0 || !dtype_ok(table_dtype) || !dtype_ok(out_dtype) || ld_table < d || ld_out < d) return MTL_ERR_ARG;
    if (N == 0) return MTL_OK;
    if (!ids || !table || !out) return MTL_ERR_ARG;
    if (((uintptr_t)ids & (ids_i64 ? 7 : 3)) || ((uintptr_t)table & (size_of(table_dtype) - 1)) || ((uintptr_t)out & (size_of(out_dtype) - 1))) return MTL_ERR_ALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    // 16-byte accesses of the wider type (8 columns only where both are bf16), one column where the row is shorter
    const int W = table_dtype == MTL_BF16 && out_dtype == MTL_BF16 && d >= 8 ? 8 : (d >= 4 ? 4 : 1);
    // (a launch holds less than 2^32 threads: up to 256 per token)
    for (int64_t done = 0, n; done < N; done += n) {
        n = N - done < (int64_t)1 << 23 ? N - done : (int64_t)1 << 23;
        const void* at = reinterpret_cast<const char*>(ids) + done * (ids_i64 ? 8 : 4);
        void* to = reinterpret_cast<char*>(out) + done * ld_out * size_of(out_dtype);
        if (table_dtype == MTL_F32 && out_dtype == MTL_F32) launch_fwd<float, float>(at, ids_i64, n, table, V, d, ld_table, scale, to, ld_out, W, st);
        else if (table_dtype == MTL_F32) launch_fwd<float, bf16_t>(at, ids_i64, n, table, V, d, ld_table, scale, to, ld_out, W, st);
        else if (out_dtype == MTL_F32) launch_fwd<bf16_t, float>(at, ids_i64, n, table, V, d, ld_table, scale, to, ld_out, W, st);
        else launch_fwd<bf16_t, bf16_t>(at, ids_i64, n, table, V, d, ld_table, scale, to, ld_out, W, st);
        MTL_CHECK_LAUNCH();
    }
    return MTL_OK;
}

extern "C" size_t mtl_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t d) {
    if (N <= 0 || V <= 0 || d <= 0) return 256;
    if (too_large(N, V, d)) return 0;
    return (size_t)plan_for(N, V, d).total;
}

extern "C" int mtl_embedding_bwd(const void* ids, int ids_i64, int64_t N, const void* dout, int dout_dtype, int64_t ld_dout, int64_t V, int64_t d, int64_t padding_idx, float scale, void* grad,
                                 int grad_dtype, int64_t ld_grad, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
    if (N < 0 || V <= 0 || d <= 0 || !dtype_ok(dout_dtype) || !dtype_ok(grad_dtype) || ld_grad < d || (N > 0 && ld_dout < d)) return MTL_ERR_ARG;
    if (too_large(N, V, d)) return MTL_ERR_UNSUPPORTED;
    if (!grad || (N > 0 && (!ids || !dout || !workspace))) return MTL_ERR_ARG;
    if (N == 0 && accumulate) return MTL_OK;
    const int gs = size_of(grad_dtype);
    if (((uintptr_t)grad & (gs - 1)) || (N > 0 && (((uintptr_t)ids & (ids_i64 ? 7 : 3)) || ((uintptr_t)dout & (size_of(dout_dtype) - 1)) || ((uintptr_t)workspace & 15)))) return MTL_ERR_ALIGN;
    if (N > 0 && workspace_bytes < mtl_embedding_bwd_workspace_bytes(N, V, d)) return MTL_ERR_WORKSPACE;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (padding_idx < 0) padding_idx = -1;
    Fill f = {(char*)grad, accumulate ? 0 : V, d * gs, ld_grad * gs, 2, false};
    if (!accumulate && ld_grad == d) { f.rows = 1; f.row_bytes = V * d * gs; }
    for (int w : {4, 16})
        if (((uintptr_t)grad & (w - 1)) == 0 && (f.rows == 1 || f.ld_bytes % w == 0)) f.width = w;
    f.once = f.rows == 1 && f.width == 16 && f.row_bytes >= (int64_t)144 << 20 && f.row_bytes < (int64_t)1 << 35;      // (2^32 threads per launch)
    const int64_t fill_want = f.once ? (f.row_bytes + (1 << 17) - 1) / (1 << 17) * 8 : f.rows == 1 ? (f.row_bytes / f.width + 4095) / 4096 : f.rows;
    const unsigned fill_blocks = (unsigned)(f.once || fill_want < 512 ? (f.rows > 0 && fill_want < 1 ? 1 : fill_want) : 512);
    char* ws = reinterpret_cast<char*>(workspace);
    if (N == 0) {
        // no token: zeros only (no tile to count)
        hipLaunchKernelGGL(embedding_sort_count_kernel, dim3(fill_blocks), dim3(1024), 0, st, ids, ids_i64, N, V, padding_idx, (const uint32_t*)nullptr, 0, 1, 0, (uint32_t*)nullptr, (uint32_t*)nullptr, f);
        MTL_CHECK_LAUNCH();
        return MTL_OK;
    }
    const int W = columns_of(d);
    const int64_t chunks = chunks_of(d, W);
    const int S = window_of(N, chunks);
    const int64_t windows = (N + S - 1) / S;
    const Plan p = plan_for(N, V, d);
    uint32_t* list_n = reinterpret_cast<uint32_t*>(ws);
    uint32_t* sid = reinterpret_cast<uint32_t*>(ws + p.sid);
    uint32_t* spos = reinterpret_cast<uint32_t*>(ws + p.spos);
    const int passes = passes_for(V), bits = bits_per_pass(V);
    if (N <= SORT_MAX) {
        if (N <= 4096) launch_sort_small<4>(ids, ids_i64, (int)N, V, padding_idx, passes, bits, sid, spos, list_n, f, fill_blocks, st);
        else launch_sort_small<8>(ids, ids_i64, (int)N, V, padding_idx, passes, bits, sid, spos, list_n, f, fill_blocks, st);
        MTL_CHECK_LAUNCH();
    } else {
        uint32_t* hist = reinterpret_cast<uint32_t*>(ws + p.hist);
        uint32_t* other_id = reinterpret_cast<uint32_t*>(ws + p.sid2);
        uint32_t* other_pos = reinterpret_cast<uint32_t*>(ws + p.spos2);
        const unsigned tiles = (unsigned)((N + TILE - 1) / TILE);
        const uint32_t *kin = nullptr, *pin = nullptr;
        for (int q = 0; q < passes; ++q) {
            const bool to_first = ((passes - 1 - q) & 1) == 0;                 // the last pass ends in sid / spos
            uint32_t* ko = to_first ? sid : other_id;
            uint32_t* po = to_first ? spos : other_pos;
            hipLaunchKernelGGL(embedding_sort_count_kernel, dim3(tiles + (q == 0 ? fill_blocks : 0)), dim3(1024), 0, st, ids, ids_i64, N, V, padding_idx, kin, q * bits, bits, (int)tiles, hist, list_n, f);
            uint32_t* totals = tiles > SELF_TILES ? list_n + 2 : nullptr;          // (MAX_BINS words behind the two list counts)
            if (totals) hipLaunchKernelGGL(embedding_sort_scan_kernel, dim3(((1u << bits) + 63) / 64), dim3(1024), 0, st, hist, (int)tiles, bits, totals);
            hipLaunchKernelGGL(embedding_sort_scatter_kernel, dim3(tiles), dim3(1024), 0, st, ids, ids_i64, N, V, padding_idx, kin, pin, q * bits, bits, (int)tiles, hist, totals, ko, po);
            MTL_CHECK_LAUNCH();
            kin = ko; pin = po;
        }
    }
    SumArgs a;
    a.sid = sid; a.spos = spos; a.N = N; a.V = V; a.d = d; a.ld_dout = ld_dout; a.ld_grad = ld_grad; a.dout = dout; a.grad = grad;
    a.part = reinterpret_cast<float*>(ws + p.part); a.list = reinterpret_cast<uint32_t*>(ws + p.list); a.list_n = list_n;
    a.scale = scale; a.accumulate = accumulate ? 1 : 0;
    a.chunks = (int)chunks; a.S = S; a.windows = windows;
    const bool d16 = dout_dtype == MTL_BF16, g16 = grad_dtype == MTL_BF16;
    if (d16 && g16) launch_sum<bf16_t, bf16_t>(a, W, st);
    else if (d16) launch_sum<bf16_t, float>(a, W, st);
    else if (g16) launch_sum<float, bf16_t>(a, W, st);
    else launch_sum<float, float>(a, W, st);
    MTL_CHECK_LAUNCH();
    if (a.windows > 1) {
        const int64_t most = ((a.windows - 1) * chunks_of(d, W > 1 ? 4 : 1) + 15) / 16;      // waves of 16 short runs' column chunks
        const int64_t most_long = (a.windows / (JOIN_SHORT + 1)) * chunks_of(d, 1);           // a long run takes at least that many windows
        const unsigned lb = (unsigned)(most_long < 256 ? most_long : 256), sb = (unsigned)(most < 256 ? most : 256);
        if (W > 1 && g16) hipLaunchKernelGGL((embedding_join_kernel<bf16_t, 4>), dim3(lb + sb), dim3(1024), 0, st, a, (int)lb);
        else if (W > 1) hipLaunchKernelGGL((embedding_join_kernel<float, 4>), dim3(lb + sb), dim3(1024), 0, st, a, (int)lb);
        else if (g16) hipLaunchKernelGGL((embedding_join_kernel<bf16_t, 1>), dim3(lb + sb), dim3(1024), 0, st, a, (int)lb);
        else hipLaunchKernelGGL((embedding_join_kernel<float, 1>), dim3(lb + sb), dim3(1024), 0, st, a, (int)lb);
        MTL_CHECK_LAUNCH();
    }
    return MTL_OK;
}
