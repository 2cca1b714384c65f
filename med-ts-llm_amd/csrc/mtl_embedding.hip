// Token table: lookup with scaling (mtl_embedding_fwd) and the table's gradient (mtl_embedding_bwd).
//
//   out[i, :]  = s table[id_i, :]
//   grad[v, :] = s sum over {i : id_i = v} dout[i, :]
//
// Both are HBM-bound (one multiply or add per element moved). The gradient is a scatter-add; atomics would make it depend on the order in which workgroups run, so
// the tokens are first SORTED by id (stable least-significant-digit radix sort of (id, position)) and every table row is then summed in position order:
//   1. sort: up to 16384 tokens in ONE workgroup's LDS, more in tiles of 4096 (count, scan, scatter per digit). The dense gradient's zero rows are written by the other workgroups
//      of the first launch that has a single busy workgroup: the fill (V d elements, most of the traffic for a large vocabulary) hides the sort.
//   2. sum: a wave owns a WINDOW of consecutive sorted tokens and a chunk of columns, walks the window with the running sum of the current id in registers and writes a row
//      whenever the id changes: balanced whatever the distribution of the ids is, and no list of runs is needed. A run that crosses a window border leaves an fp32 partial per window
//      (one slot for a run that came in, one for a run that goes out).
//   3. join: the windows in which a crossing run starts have put themselves on a list; each such run's partials are added in window order.
#include "mtl_common.h"

namespace {

constexpr int SORT_MAX = 16384;          // tokens that one workgroup sorts in its LDS
constexpr int TILE = 4096;               // tokens per workgroup of the tiled sort
constexpr int MAX_BINS = 512;            // digits of up to 9 bits: two passes for every vocabulary up to 262143

// ---------------------------------------------------------------- element access: W consecutive elements <-> fp32
template <typename T, int W>
struct Io;
template <>
struct Io<float, 1> {
    static __device__ __forceinline__ void load(const void* p, int64_t i, float (&x)[1]) { x[0] = reinterpret_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&x)[1]) { reinterpret_cast<float*>(p)[i] = x[0]; }
};
template <>
struct Io<bf16_t, 1> {
    static __device__ __forceinline__ void load(const void* p, int64_t i, float (&x)[1]) { x[0] = bf16_to_f32(reinterpret_cast<const bf16_t*>(p)[i]); }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&x)[1]) { reinterpret_cast<bf16_t*>(p)[i] = f32_to_bf16(x[0]); }
};
template <int W>
struct Io<float, W> {
    static __device__ __forceinline__ void load(const void* p, int64_t i, float (&x)[W]) {
#pragma unroll
        for (int j = 0; j < W; j += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i + j);
            x[j] = v[0]; x[j + 1] = v[1]; x[j + 2] = v[2]; x[j + 3] = v[3];
        }
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&x)[W]) {
#pragma unroll
        for (int j = 0; j < W; j += 4) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i + j) = (f32x4){x[j], x[j + 1], x[j + 2], x[j + 3]};
    }
};
template <int W>
struct Io<bf16_t, W> {
    static __device__ __forceinline__ void load(const void* p, int64_t i, float (&x)[W]) {
        uint32_t w[W / 2];
        const bf16_t* s = reinterpret_cast<const bf16_t*>(p) + i;
        if (W == 8) { const u32x4 v = *reinterpret_cast<const u32x4*>(s); w[0] = v[0]; w[1] = v[1]; w[W / 2 - 2] = v[2]; w[W / 2 - 1] = v[3]; }
        else { const u32x2 v = *reinterpret_cast<const u32x2*>(s); w[0] = v[0]; w[1] = v[1]; }
#pragma unroll
        for (int j = 0; j < W / 2; ++j) { x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&x)[W]) {
        bf16_t* d = reinterpret_cast<bf16_t*>(p) + i;
        if (W == 8) *reinterpret_cast<u32x4*>(d) = (u32x4){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[W - 4], x[W - 3]), pack_bf16x2(x[W - 2], x[W - 1])};
        else *reinterpret_cast<u32x2*>(d) = (u32x2){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    }
};

__device__ __forceinline__ int64_t load_id(const void* ids, int ids_i64, int64_t i) {
    return ids_i64 ? reinterpret_cast<const int64_t*>(ids)[i] : (int64_t)reinterpret_cast<const int32_t*>(ids)[i];
}

// ---------------------------------------------------------------- lookup
// a wave holds 64 / LPR rows (LPR lanes per row, W columns per lane and step): narrow tables fill the wave too
template <typename TT, typename OT, int W>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* __restrict__ ids, int ids_i64, int64_t N, const TT* __restrict__ table, int64_t V, int64_t d, int64_t ld_table,
                                                            float scale, OT* __restrict__ out, int64_t ld_out, int lpr_log2) {
    const int lpr = 1 << lpr_log2;
    const int rows_per_block = 256 >> lpr_log2;
    const int l = threadIdx.x & (lpr - 1);
    for (int64_t i = (int64_t)blockIdx.x * rows_per_block + (threadIdx.x >> lpr_log2); i < N; i += (int64_t)gridDim.x * rows_per_block) {
        const int64_t id = load_id(ids, ids_i64, i);
        const bool in = id >= 0 && id < V;
        const TT* src = table + (in ? id : 0) * ld_table;
        OT* dst = out + i * ld_out;
#pragma unroll 4
        for (int64_t c = (int64_t)l * W; c < d; c += (int64_t)lpr * W) {
            float x[W];
            Io<TT, W>::load(src, c, x);
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = in ? x[j] * scale : 0.f;
            Io<OT, W>::store(dst, c, x);
        }
    }
}

// ---------------------------------------------------------------- zero rows of the dense gradient
struct Fill { char* p; int64_t rows, row_bytes, ld_bytes; int width; };      // width: 16, 4 or 2 bytes per store

__device__ __forceinline__ void fill_zero(const Fill& f, int64_t block, int64_t blocks) {
    const int64_t per_row = f.row_bytes / f.width, total = f.rows * per_row;
    const bool flat = f.row_bytes == f.ld_bytes;
    for (int64_t i = block * blockDim.x + threadIdx.x; i < total; i += blocks * blockDim.x) {
        int64_t at = i * f.width;
        if (!flat) { const int64_t r = i / per_row; at = r * f.ld_bytes + (i - r * per_row) * f.width; }
        if (f.width == 16) *reinterpret_cast<u32x4*>(f.p + at) = (u32x4){0, 0, 0, 0};
        else if (f.width == 4) *reinterpret_cast<uint32_t*>(f.p + at) = 0;
        else *reinterpret_cast<uint16_t*>(f.p + at) = 0;
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
    uint32_t* tot = cnt + 16 * MAX_BINS;                                     // [16]
    uint32_t* lkey = tot + 16;                                               // [N]
    uint16_t* lpos = reinterpret_cast<uint16_t*>(lkey + N);                  // [N]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n_e = (N + 1023) >> 10;                                        // elements per thread: wave w owns [w n_e 64, (w + 1) n_e 64)
    const int i0 = wave * n_e * 64 + lane;
    const uint32_t mask = (1u << bits) - 1u;
    if (threadIdx.x == 0) *list_n = 0;
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

// tiled sort, digit counts of each tile: hist[digit][tile]
__global__ __launch_bounds__(1024) void embedding_sort_count_kernel(const void* __restrict__ ids, int ids_i64, int64_t N, int64_t V, int64_t pad, const uint32_t* __restrict__ keys, int shift, int bits,
                                                                    uint32_t* __restrict__ hist) {
    __shared__ uint32_t cnt[MAX_BINS];
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
    for (int i = threadIdx.x; i < (1 << bits); i += 1024) hist[(int64_t)i * gridDim.x + blockIdx.x] = cnt[i];
}

// exclusive prefix over all entries of hist in place (workgroup 0); the others write the zero rows
__global__ __launch_bounds__(1024) void embedding_sort_scan_kernel(uint32_t* __restrict__ hist, int64_t n, uint32_t* __restrict__ list_n, const Fill f) {
    __shared__ uint32_t tot[16];
    if (blockIdx.x > 0) {
        fill_zero(f, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    if (list_n && threadIdx.x == 0) *list_n = 0;
    uint32_t carry = 0;
    for (int64_t base = 0; base < n; base += 8192) {
        uint32_t c[8], sum = 0;
        const int64_t at = base + threadIdx.x * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) { c[j] = at + j < n ? hist[at + j] : 0u; sum += c[j]; }
        uint32_t total;
        uint32_t x = carry + block_exclusive(sum, tot, total);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (at + j < n) hist[at + j] = x;
            x += c[j];
        }
        carry += total;
    }
}

__global__ __launch_bounds__(1024) void embedding_sort_scatter_kernel(const void* __restrict__ ids, int ids_i64, int64_t N, int64_t V, int64_t pad, const uint32_t* __restrict__ keys,
                                                                      const uint32_t* __restrict__ poss, int shift, int bits, const uint32_t* __restrict__ hist, uint32_t* __restrict__ sid,
                                                                      uint32_t* __restrict__ spos) {
    __shared__ uint32_t cnt[16 * MAX_BINS];
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
    rank_digits<E>(key, valid, shift, bits, cnt, rank, E);
    // counts per wave -> the tile's first rank of each digit plus the waves before
    if (threadIdx.x < (1 << bits)) {
        uint32_t at = hist[(int64_t)threadIdx.x * gridDim.x + blockIdx.x];
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
            const uint32_t at = cnt[wave * MAX_BINS + ((key[e] >> shift) & ((1u << bits) - 1u))] + rank[e];
            sid[at] = key[e];
            spos[at] = pos[e];
        }
}

// ---------------------------------------------------------------- sum over windows
struct SumArgs {
    const uint32_t* sid; const uint32_t* spos;
    int64_t N, V, d, ld_dout, ld_grad;
    const void* dout; void* grad;
    float* part;                 // [windows][2][d]: 0 = the run that came into the window, 1 = the run that goes out of it (and started in it)
    uint32_t* list; uint32_t* list_n;
    float scale;
    int accumulate, S, chunks;
    int64_t windows;
};

template <typename GT, int W>
__device__ __forceinline__ void write_row(const SumArgs& a, uint32_t id, int64_t c, const float (&acc)[W]) {
    const int64_t at = (int64_t)id * a.ld_grad + c;
    float y[W];
#pragma unroll
    for (int j = 0; j < W; ++j) y[j] = acc[j] * a.scale;
    if (a.accumulate) {
        float old[W];
        Io<GT, W>::load(a.grad, at, old);
#pragma unroll
        for (int j = 0; j < W; ++j) y[j] += old[j];
    }
    Io<GT, W>::store(a.grad, at, y);
}

template <typename DT, typename GT, int W>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const SumArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = item / a.chunks;
    if (w >= a.windows) return;
    const int64_t c = (item - w * a.chunks) * (64 * W) + lane * W;
    const bool in = c < a.d;                                    // (d % W == 0 wherever W > 1)
    const int64_t i0 = w * a.S, i1 = i0 + a.S < a.N ? i0 + a.S : a.N;
    const uint32_t none = (uint32_t)a.V;
    uint32_t cur = a.sid[i0];
    bool came_in = i0 > 0 && a.sid[i0 - 1] == cur;
    float acc[W];
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j] = 0.f;
    float* part = a.part + w * 2 * a.d + c;
    for (int64_t i = i0; i < i1 && cur != none; i += 8) {
        uint32_t id[8];
        float x[8][W];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t at = i + u < i1 ? i + u : i1 - 1;      // (beyond the window: the last token again, not used)
            id[u] = i + u < i1 ? a.sid[at] : none;
            if (in) Io<DT, W>::load(a.dout, (int64_t)a.spos[at] * a.ld_dout + c, x[u]);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (i + u >= i1) break;
            if (id[u] != cur) {                                  // (uniform) the run of `cur` ends here, inside the window
                if (in) {
                    if (came_in) Io<float, W>::store(part, 0, acc);
                    else write_row<GT, W>(a, cur, c, acc);
                }
                cur = id[u];
                came_in = false;
#pragma unroll
                for (int j = 0; j < W; ++j) acc[j] = 0.f;
                if (cur == none) break;
            }
#pragma unroll
            for (int j = 0; j < W; ++j) acc[j] += x[u][j];
        }
    }
    if (cur == none) return;
    const bool goes_on = i1 < a.N && a.sid[i1] == cur;
    if (!in) return;
    if (came_in) Io<float, W>::store(part, 0, acc);
    else if (goes_on) {
        Io<float, W>::store(part, a.d, acc);
        if (c == 0) a.list[atomicAdd(a.list_n, 1u)] = (uint32_t)w;      // (the list's order shows nowhere: each entry is a whole run)
    } else write_row<GT, W>(a, cur, c, acc);
}

// the run that starts in window list[k] and goes on: tail partial of that window, then the head partials of the following ones up to the window where it ends. Four waves take a
// quarter of the windows each, in order, and are joined in order.
template <typename GT>
__global__ __launch_bounds__(256) void embedding_join_kernel(const SumArgs a, int chunks) {
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t items = (int64_t)*a.list_n * chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t w = a.list[item / chunks];
        const int64_t c = (item % chunks) * 64 + lane;
        const bool in = c < a.d;
        const uint32_t id = a.sid[(w + 1) * a.S];
        int64_t last = w + 1;                                     // the window in which the run ends
        for (;;) {                                                // 64 windows at a time: does the run go on behind window last + lane?
            const int64_t k = last + lane;
            const int64_t end = (k + 1) * a.S;
            const bool on = end < a.N && a.sid[end] == id;
            const uint64_t stops = __ballot(!on);
            if (stops) { last += __ffsll((unsigned long long)stops) - 1; break; }
            last += 64;
        }
        const int64_t n = last - w;                               // head partials of windows w + 1 .. last
        const int64_t k0 = w + 1 + n * wave / 4, k1 = w + 1 + n * (wave + 1) / 4;
        float s = wave == 0 && in ? a.part[w * 2 * a.d + a.d + c] : 0.f;
        if (in) {
#pragma unroll 8
            for (int64_t k = k0; k < k1; ++k) s += a.part[k * 2 * a.d + c];
        }
        sums[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && in) {
            const float t[1] = {((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane]};
            write_row<GT, 1>(a, id, c, t);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side
inline int bits_for(int64_t V) { int b = 1; while (b < 31 && ((int64_t)1 << b) <= V) ++b; return b; }      // values 0 .. V
inline int passes_for(int64_t V) { return (bits_for(V) + 8) / 9; }
inline int bits_per_pass(int64_t V) { const int p = passes_for(V); return (bits_for(V) + p - 1) / p; }
inline int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// window length: enough (window, column chunk) waves to fill the chip, at most 64 tokens (a partial row per window border costs 2 / S of the rows read)
inline int window_of(int64_t N, int64_t chunks) {
    int s = 8;
    while (s < 64 && N / (2 * s) * chunks >= 8192) s *= 2;
    return s;
}
inline int64_t chunks_of(int64_t d, int W) { return (d + 64 * W - 1) / (64 * W); }

struct Plan { int64_t sid, spos, sid2, spos2, hist, list, part, total; };
inline Plan plan_for(int64_t N, int64_t V, int64_t d) {
    Plan p;
    int64_t at = 256;                                             // list_n
    auto take = [&](int64_t bytes) { const int64_t here = at; at += up(bytes, 256); return here; };
    const bool small = N <= SORT_MAX;
    const int64_t tiles = (N + TILE - 1) / TILE, windows = (N + 7) / 8;      // (8: the shortest window)
    p.sid = take(4 * N); p.spos = take(4 * N);
    p.sid2 = small ? 0 : take(4 * N); p.spos2 = small ? 0 : take(4 * N);
    p.hist = small ? 0 : take(4 * tiles * MAX_BINS);
    p.list = take(4 * windows);
    // partials: the window length depends on the columns per wave (64, 256 or 512): the longest list of the three
    int64_t most = 0;
    for (int W : {1, 4, 8}) { const int64_t s = window_of(N, chunks_of(d, W)); const int64_t w = (N + s - 1) / s; most = w > most ? w : most; }
    p.part = take(8 * most * d);
    p.total = at;
    return p;
}

template <int E>
void launch_sort_small(const void* ids, int ids_i64, int N, int64_t V, int64_t pad, int passes, int bits, uint32_t* sid, uint32_t* spos, uint32_t* list_n, const Fill& f, unsigned fill_blocks,
                       hipStream_t st) {
    const size_t fixed = (16 * MAX_BINS + 16) * 4;
    (void)hipFuncSetAttribute((const void*)embedding_sort_small_kernel<E>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)(fixed + E * 1024 * 6));
    hipLaunchKernelGGL(embedding_sort_small_kernel<E>, dim3(1 + fill_blocks), dim3(1024), fixed + (size_t)N * 6, st, ids, ids_i64, N, V, pad, passes, bits, sid, spos, list_n, f);
}

template <typename DT, typename GT>
void launch_sum(const SumArgs& a, int W, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.windows * a.chunks + 3) / 4);
    if (W == 8) hipLaunchKernelGGL((embedding_sum_kernel<DT, GT, 8>), dim3(blocks), dim3(256), 0, st, a);
    else if (W == 4) hipLaunchKernelGGL((embedding_sum_kernel<DT, GT, 4>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((embedding_sum_kernel<DT, GT, 1>), dim3(blocks), dim3(256), 0, st, a);
}

template <typename TT, typename OT>
void launch_fwd(const void* ids, int ids_i64, int64_t N, const void* table, int64_t V, int64_t d, int64_t ld_table, float scale, void* out, int64_t ld_out, int W, hipStream_t st) {
    int lpr = 0;
    while (lpr < 6 && ((int64_t)W << lpr) < d) ++lpr;
    const int64_t rows = 256 >> lpr, want = (N + rows - 1) / rows;
    const unsigned blocks = (unsigned)(want < 65536 ? want : 65536);
    if (W == 8) hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, 8>), dim3(blocks), dim3(256), 0, st, ids, ids_i64, N, (const TT*)table, V, d, ld_table, scale, (OT*)out, ld_out, lpr);
    else if (W == 4) hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, 4>), dim3(blocks), dim3(256), 0, st, ids, ids_i64, N, (const TT*)table, V, d, ld_table, scale, (OT*)out, ld_out, lpr);
    else hipLaunchKernelGGL((embedding_fwd_kernel<TT, OT, 1>), dim3(blocks), dim3(256), 0, st, ids, ids_i64, N, (const TT*)table, V, d, ld_table, scale, (OT*)out, ld_out, lpr);
}

inline bool dtype_ok(int t) { return t == MTL_F32 || t == MTL_BF16; }
inline int size_of(int t) { return t == MTL_BF16 ? 2 : 4; }
// W columns per lane are possible for this operand: W * size <= 16 B accesses, aligned
inline bool fits(const void* p, int64_t ld, int dtype, int64_t d, int W) {
    const int64_t a = (int64_t)W * size_of(dtype) < 16 ? (int64_t)W * size_of(dtype) : 16;
    return d % W == 0 && (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0 && (ld * size_of(dtype)) % a == 0;
}

}  // namespace

extern "C" int mtl_embedding_fwd(const void* ids, int ids_i64, int64_t N, const void* table, int table_dtype, int64_t V, int64_t d, int64_t ld_table, float scale, void* out, int out_dtype,
                                 int64_t ld_out, void* stream) {
    if (N < 0 || V <= 0 || d <= 0 || !dtype_ok(table_dtype) || !dtype_ok(out_dtype) || ld_table < d || ld_out < d) return MTL_ERR_ARG;
    if (N == 0) return MTL_OK;
    if (!ids || !table || !out) return MTL_ERR_ARG;
    if (((uintptr_t)ids & (ids_i64 ? 7 : 3)) || ((uintptr_t)table & (size_of(table_dtype) - 1)) || ((uintptr_t)out & (size_of(out_dtype) - 1))) return MTL_ERR_ALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    // 16-byte accesses of the wider operand's type where both allow it
    int W = 1;
    for (int c : {4, 8})
        if (fits(table, ld_table, table_dtype, d, c) && fits(out, ld_out, out_dtype, d, c) && (c == 4 || (table_dtype == MTL_BF16 && out_dtype == MTL_BF16))) W = c;
    if (table_dtype == MTL_F32 && out_dtype == MTL_F32) launch_fwd<float, float>(ids, ids_i64, N, table, V, d, ld_table, scale, out, ld_out, W, st);
    else if (table_dtype == MTL_F32) launch_fwd<float, bf16_t>(ids, ids_i64, N, table, V, d, ld_table, scale, out, ld_out, W, st);
    else if (out_dtype == MTL_F32) launch_fwd<bf16_t, float>(ids, ids_i64, N, table, V, d, ld_table, scale, out, ld_out, W, st);
    else launch_fwd<bf16_t, bf16_t>(ids, ids_i64, N, table, V, d, ld_table, scale, out, ld_out, W, st);
    MTL_CHECK_LAUNCH();
    return MTL_OK;
}

extern "C" size_t mtl_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t d) {
    if (N <= 0 || V <= 0 || d <= 0) return 256;
    return (size_t)plan_for(N, V, d).total;
}

extern "C" int mtl_embedding_bwd(const void* ids, int ids_i64, int64_t N, const void* dout, int dout_dtype, int64_t ld_dout, int64_t V, int64_t d, int64_t padding_idx, float scale, void* grad,
                                 int grad_dtype, int64_t ld_grad, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
    if (N < 0 || V <= 0 || d <= 0 || !grad || !dtype_ok(dout_dtype) || !dtype_ok(grad_dtype) || ld_grad < d || (N > 0 && (!ids || !dout || ld_dout < d || !workspace))) return MTL_ERR_ARG;
    if (N > 0x7fffffff || V >= 0x7fffffff) return MTL_ERR_UNSUPPORTED;
    if (N == 0 && accumulate) return MTL_OK;
    const int gs = size_of(grad_dtype);
    if (((uintptr_t)grad & (gs - 1)) || (N > 0 && (((uintptr_t)ids & (ids_i64 ? 7 : 3)) || ((uintptr_t)dout & (size_of(dout_dtype) - 1)) || ((uintptr_t)workspace & 15)))) return MTL_ERR_ALIGN;
    if (N > 0 && workspace_bytes < mtl_embedding_bwd_workspace_bytes(N, V, d)) return MTL_ERR_WORKSPACE;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (padding_idx < 0) padding_idx = -1;
    Fill f = {(char*)grad, accumulate ? 0 : V, d * gs, ld_grad * gs, 2};
    for (int w : {4, 16})
        if (f.row_bytes % w == 0 && f.ld_bytes % w == 0 && ((uintptr_t)grad & (w - 1)) == 0) f.width = w;
    const int64_t fill_items = f.rows * (f.row_bytes / f.width);
    const unsigned fill_blocks = (unsigned)(fill_items == 0 ? 0 : ((fill_items + 1023) / 1024 < 1024 ? (fill_items + 1023) / 1024 : 1024));
    char* ws = reinterpret_cast<char*>(workspace);
    if (N == 0) {
        // no token: zeros only, through the scan kernel with an empty histogram (its counter lives in a workspace that may be NULL here)
        hipLaunchKernelGGL(embedding_sort_scan_kernel, dim3(1 + fill_blocks), dim3(1024), 0, st, (uint32_t*)nullptr, (int64_t)0, (uint32_t*)nullptr, f);
        MTL_CHECK_LAUNCH();
        return MTL_OK;
    }
    const Plan p = plan_for(N, V, d);
    uint32_t* list_n = reinterpret_cast<uint32_t*>(ws);
    uint32_t* sid = reinterpret_cast<uint32_t*>(ws + p.sid);
    uint32_t* spos = reinterpret_cast<uint32_t*>(ws + p.spos);
    const int passes = passes_for(V), bits = bits_per_pass(V);
    if (N <= SORT_MAX) {
        if (N <= 4096) launch_sort_small<4>(ids, ids_i64, (int)N, V, padding_idx, passes, bits, sid, spos, list_n, f, fill_blocks, st);
        else if (N <= 8192) launch_sort_small<8>(ids, ids_i64, (int)N, V, padding_idx, passes, bits, sid, spos, list_n, f, fill_blocks, st);
        else launch_sort_small<16>(ids, ids_i64, (int)N, V, padding_idx, passes, bits, sid, spos, list_n, f, fill_blocks, st);
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
            hipLaunchKernelGGL(embedding_sort_count_kernel, dim3(tiles), dim3(1024), 0, st, ids, ids_i64, N, V, padding_idx, kin, q * bits, bits, hist);
            const Fill none = {nullptr, 0, 16, 16, 16};
            hipLaunchKernelGGL(embedding_sort_scan_kernel, dim3(1 + (q == 0 ? fill_blocks : 0)), dim3(1024), 0, st, hist, (int64_t)tiles << bits, list_n, q == 0 ? f : none);
            hipLaunchKernelGGL(embedding_sort_scatter_kernel, dim3(tiles), dim3(1024), 0, st, ids, ids_i64, N, V, padding_idx, kin, pin, q * bits, bits, hist, ko, po);
            MTL_CHECK_LAUNCH();
            kin = ko; pin = po;
        }
    }
    int W = 1;
    for (int c : {4, 8})
        if (d > 64 * (c / 4) && fits(dout, ld_dout, dout_dtype, d, c) && fits(grad, ld_grad, grad_dtype, d, c) && (c == 4 || d % 512 == 0 || d >= 2048)) W = c;
    SumArgs a;
    a.sid = sid; a.spos = spos; a.N = N; a.V = V; a.d = d; a.ld_dout = ld_dout; a.ld_grad = ld_grad; a.dout = dout; a.grad = grad;
    a.part = reinterpret_cast<float*>(ws + p.part); a.list = reinterpret_cast<uint32_t*>(ws + p.list); a.list_n = list_n;
    a.scale = scale; a.accumulate = accumulate ? 1 : 0;
    a.chunks = (int)chunks_of(d, W);
    a.S = window_of(N, a.chunks);
    a.windows = (N + a.S - 1) / a.S;
    if (a.windows * a.chunks > (int64_t)0x7fffffff * 4) return MTL_ERR_UNSUPPORTED;
    const bool d16 = dout_dtype == MTL_BF16, g16 = grad_dtype == MTL_BF16;
    if (d16 && g16) launch_sum<bf16_t, bf16_t>(a, W, st);
    else if (d16) launch_sum<bf16_t, float>(a, W, st);
    else if (g16) launch_sum<float, bf16_t>(a, W, st);
    else launch_sum<float, float>(a, W, st);
    MTL_CHECK_LAUNCH();
    if (a.windows > 1) {
        const int jc = (int)chunks_of(d, 1);
        const int64_t most = (a.windows - 1) * jc;
        const unsigned blocks = (unsigned)(most < 2048 ? most : 2048);
        if (g16) hipLaunchKernelGGL(embedding_join_kernel<bf16_t>, dim3(blocks), dim3(256), 0, st, a, jc);
        else hipLaunchKernelGGL(embedding_join_kernel<float>, dim3(blocks), dim3(256), 0, st, a, jc);
        MTL_CHECK_LAUNCH();
    }
    return MTL_OK;
}
