// RMS norm of every query and key head and the rotary embedding behind it in one pass (mtl_qk_norm_rope_fwd), and its backward pass.
//
//   r = 1 / sqrt(mean_j x_j^2 + eps),  n = r x,  y = Rot(n w)            Rot: half-split rotation of the first R of D elements by the row's position (pairs j, j + R/2)
//   u = Rot^T dy,  dw = sum u n,  a = u w,  dx = r (a - n mean_j(a_j n_j))
//
// HBM-bound: the forward reads and writes (Hq + Hkv) D elements per row, the backward reads two and writes one (r is recomputed from x, which it reads anyway: nothing is saved).
// Layout: a wave owns the queries OR the keys of a row (one token; blockIdx.y says which: with both, the two weights and their gradients double the registers and halve the waves in
// flight) and walks their heads; a group of LPH lanes owns a head, each lane W consecutive PAIRS, i.e. W elements of each half: the rotation needs no exchange between lanes, the two
// sums take log2(LPH) DPP steps, and what the heads of a row share (cos, sin, the weight) is loaded once per row or wave and stays in registers.
// Pairs beyond R/2 (elements R .. D-1, split in halves the same way) are rotated by angle 0. All arithmetic fp32, one rounding at the store.
#include "mtl_common.h"

namespace {

constexpr int WAVES = 4;

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// sum over groups of L lanes, in every lane of the group (all 64 lanes active)
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    v = dpp_add<0xB1>(v);                       // quad_perm: neighbours
    v = dpp_add<0x4E>(v);                       // quad_perm: pairs
    if (L >= 8) v = dpp_add<0x141>(v);          // row_half_mirror: the other quad of 8
    if (L >= 16) v = dpp_add<0x140>(v);         // row_mirror: the other half of 16
    if (L >= 32) v += __shfl_xor(v, 16, 64);
    if (L >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

// vectors at any element's address (global accesses need no more alignment than their elements have)
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
// NT: the data pass the cache by (vectors of bf16 only)
template <typename T, int W, bool NT = false>
__device__ __forceinline__ void load_w(const T* p, float (&x)[W]) {
    if constexpr (W == 1) {
        if constexpr (sizeof(T) == 4) x[0] = *p;
        else x[0] = bf16_to_f32(*p);
    } else if constexpr (sizeof(T) == 4) {
        const u32x4_any a = reinterpret_cast<const u32x4_any*>(p)[0], b = reinterpret_cast<const u32x4_any*>(p)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = __uint_as_float(a[j]); x[4 + j] = __uint_as_float(b[j]); }
    } else {
        u32x4_any a;
        if constexpr (NT) a = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
        else a = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[2 * j] = __uint_as_float(a[j] << 16); x[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u); }
    }
}
template <typename T, int W>
__device__ __forceinline__ void store_w(T* p, const float (&x)[W]) {
    if constexpr (W == 1) {
        if constexpr (sizeof(T) == 4) *p = x[0];
        else *p = f32_to_bf16(x[0]);
    } else if constexpr (sizeof(T) == 4) {
        reinterpret_cast<u32x4_any*>(p)[0] = (u32x4_any){__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
        reinterpret_cast<u32x4_any*>(p)[1] = (u32x4_any){__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])};
    } else *reinterpret_cast<u32x4_any*>(p) = (u32x4_any){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

// Where a lane's C chunks of W pairs sit: lo[c] / hi[c] = the elements of the two halves, turn[c] = index of the first pair in the cos / sin row or -1 (not rotated), on[c] = in the head.
// The rotated pairs and the others are cut into chunks apart. SHIFT: a number of pairs that W does not divide; the last chunk starts earlier and computes skip[c] of its neighbour's pairs a
// second time (the same bits), which then count in no sum.
template <int W, int LPH, int C, bool SHIFT>
struct Lane {
    int lo[C], hi[C], turn[C], skip[C];
    bool on[C];
    __device__ __forceinline__ Lane(int D, int R) {
        const int l = threadIdx.x & (LPH - 1), rp = R >> 1, rest = (D - R) >> 1, nrot = (rp + W - 1) / W, nrest = (rest + W - 1) / W;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            int i = c * LPH + l;
            on[c] = i < nrot + nrest;
            if (!on[c]) i = 0;
            const bool rot = i < nrot;
            const int j = (rot ? i : i - nrot) * W, pairs = rot ? rp : rest;
            const int at = SHIFT && j > pairs - W ? pairs - W : j;
            skip[c] = j - at;
            lo[c] = rot ? at : R + at;
            hi[c] = lo[c] + pairs;
            turn[c] = rot ? at : -1;
        }
    }
    // x where pair j of chunk c counts, 0 where it is a neighbour's
    __device__ __forceinline__ float own(int c, int j, float x) const { return SHIFT && j < skip[c] ? 0.f : x; }
};

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
    return dtype == MTL_BF16 ? bf16_to_f32(reinterpret_cast<const bf16_t*>(w)[i]) : reinterpret_cast<const float*>(w)[i];
}
template <int W, int LPH, int C, bool S>
__device__ __forceinline__ void load_weights(const void* w, int dtype, const Lane<W, LPH, C, S>& L, float (&lo)[C][W], float (&hi)[C][W]) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            lo[c][j] = L.on[c] ? weight_at(w, dtype, L.lo[c] + j) : 0.f;
            hi[c][j] = L.on[c] ? weight_at(w, dtype, L.hi[c] + j) : 0.f;
        }
}

// cos / sin of a row's pairs; a position outside the table turns every element of the row into NaN
template <int W, int LPH, int C, bool S>
__device__ __forceinline__ void load_turn(const mtl_qk_norm_rope_args& a, int64_t b, int64_t t, const Lane<W, LPH, C, S>& L, float (&cs)[C][W], float (&sn)[C][W]) {
    int64_t pos = a.pos0 + t;
    if (a.positions) pos = a.pos_i64 ? reinterpret_cast<const int64_t*>(a.positions)[b * a.pos_bs + t] : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[b * a.pos_bs + t];
    const bool in = pos >= 0 && pos < a.n_pos;
    const float nan = __uint_as_float(0x7fc00000u);
    const float* cr = a.cos_t + (in ? pos : 0) * a.R;
    const float* sr = a.sin_t + (in ? pos : 0) * a.R;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (L.turn[c] >= 0) {
            load_w<float, W>(cr + L.turn[c], cs[c]);
            load_w<float, W>(sr + L.turn[c], sn[c]);
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) { cs[c][j] = 1.f; sn[c][j] = 0.f; }
        }
        if (!in)
#pragma unroll
            for (int j = 0; j < W; ++j) cs[c][j] = sn[c][j] = nan;
    }
}

// heads [h0, h1) of one row: forward
template <typename T, int W, int LPH, int C, bool S, bool NT>
__device__ __forceinline__ void heads_fwd(const T* x, T* y, int h0, int h1, int D, float eps, float inv_d, const Lane<W, LPH, C, S>& L, const float (&wl)[C][W], const float (&wh)[C][W],
                                          const float (&cs)[C][W], const float (&sn)[C][W]) {
    constexpr int G = 64 / LPH, U = W == 8 ? 2 : 1;      // heads per step of the wave, steps whose loads are in flight together
    const int g = (threadIdx.x & 63) / LPH;
    for (int h = h0; h < h1; h += G * U) {
        float lo[U][C][W], hi[U][C][W];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int hh = h + u * G + g;
                if (hh < h1 && L.on[c]) {
                    load_w<T, W, NT>(x + (int64_t)hh * D + L.lo[c], lo[u][c]);
                    load_w<T, W, NT>(x + (int64_t)hh * D + L.hi[c], hi[u][c]);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) lo[u][c][j] = hi[u][c][j] = 0.f;
                }
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int hh = h + u * G + g;
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < W; ++j) ss += L.own(c, j, lo[u][c][j]) * lo[u][c][j] + L.own(c, j, hi[u][c][j]) * hi[u][c][j];
            ss = group_sum<LPH>(ss);
            const float r = 1.0f / __builtin_sqrtf(ss * inv_d + eps);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float yl[W], yh[W];
#pragma unroll
                for (int j = 0; j < W; ++j) rope_pair(lo[u][c][j] * r * wl[c][j], hi[u][c][j] * r * wh[c][j], cs[c][j], sn[c][j], yl[j], yh[j]);
                if (hh < h1 && L.on[c]) {
                    store_w(y + (int64_t)hh * D + L.lo[c], yl);
                    store_w(y + (int64_t)hh * D + L.hi[c], yh);
                }
            }
        }
    }
}

// one side of a call: the queries (0) or the keys (1)
struct Side {
    const void *x, *dy, *w;
    void* y;
    int64_t x_bs, x_ts, dy_bs, dy_ts, y_bs, y_ts;
    int H;
};
__device__ __forceinline__ Side side_of(const mtl_qk_norm_rope_args& a, bool keys) {
    Side s;
    s.x = keys ? a.k : a.q; s.x_bs = keys ? a.k_bs : a.q_bs; s.x_ts = keys ? a.k_ts : a.q_ts;
    s.dy = keys ? a.dk_out : a.dq_out; s.dy_bs = keys ? a.dko_bs : a.dqo_bs; s.dy_ts = keys ? a.dko_ts : a.dqo_ts;
    s.y = keys ? a.k_out : a.q_out; s.y_bs = keys ? a.ko_bs : a.qo_bs; s.y_ts = keys ? a.ko_ts : a.qo_ts;
    s.w = keys ? a.wk : a.wq;
    s.H = (int)(keys ? a.Hkv : a.Hq);
    return s;
}

template <typename T, int W, int LPH, int C, bool S, bool NT>
__global__ __launch_bounds__(WAVES * 64) void qk_norm_rope_fwd_kernel(const mtl_qk_norm_rope_args a, int hq_per, int hk_per) {
    const Lane<W, LPH, C, S> L((int)a.D, (int)a.R);
    const int64_t rows = a.B * a.T;
    const float inv_d = 1.0f / (float)a.D;
    const Side s = side_of(a, blockIdx.y == 1);
    const int per = blockIdx.y ? hk_per : hq_per;                 // few rows: a row's heads are spread over gridDim.z waves
    const int h0 = blockIdx.z * per, h1 = h0 + per < s.H ? h0 + per : s.H;
    if (h0 >= h1) return;
    float wl[C][W], wh[C][W];
    load_weights(s.w, a.w_dtype, L, wl, wh);
    for (int64_t row = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * WAVES) {
        const int64_t b = row / a.T, t = row - b * a.T;
        float cs[C][W], sn[C][W];
        load_turn(a, b, t, L, cs, sn);
        heads_fwd<T, W, LPH, C, S, NT>((const T*)s.x + b * s.x_bs + t * s.x_ts, (T*)s.y + b * s.y_bs + t * s.y_ts, h0, h1, (int)a.D, a.eps, inv_d, L, wl, wh, cs, sn);
    }
}

// all heads of one row: backward; gl / gh accumulate dw
template <typename T, int W, int LPH, int C, bool S, bool NT, bool DW>
__device__ __forceinline__ void heads_bwd(const T* x, const T* dy, T* dx, int h1, int D, float eps, float inv_d, const Lane<W, LPH, C, S>& L, const float (&wl)[C][W],
                                          const float (&wh)[C][W], const float (&cs)[C][W], const float (&sn)[C][W], float (&gl)[C][W], float (&gh)[C][W]) {
    constexpr int G = 64 / LPH;
    const int g = (threadIdx.x & 63) / LPH;
    for (int h = 0; h < h1; h += G) {
        const int hh = h + g;
        float lo[C][W], hi[C][W], al[C][W], ah[C][W];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (hh < h1 && L.on[c]) {
                load_w<T, W, NT>(x + (int64_t)hh * D + L.lo[c], lo[c]);
                load_w<T, W, NT>(x + (int64_t)hh * D + L.hi[c], hi[c]);
                load_w<T, W, NT>(dy + (int64_t)hh * D + L.lo[c], al[c]);
                load_w<T, W, NT>(dy + (int64_t)hh * D + L.hi[c], ah[c]);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) lo[c][j] = hi[c][j] = al[c][j] = ah[c][j] = 0.f;
            }
        }
        float ss = 0.f, sa = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float ul, uh;
                rope_pair(al[c][j], ah[c][j], cs[c][j], -sn[c][j], ul, uh);          // the inverse rotation
                al[c][j] = ul; ah[c][j] = uh;
                const float xl = L.own(c, j, lo[c][j]), xh = L.own(c, j, hi[c][j]);
                ss += xl * lo[c][j] + xh * hi[c][j];
                sa += ul * wl[c][j] * xl + uh * wh[c][j] * xh;
            }
        ss = group_sum<LPH>(ss);
        sa = group_sum<LPH>(sa);
        const float r = 1.0f / __builtin_sqrtf(ss * inv_d + eps);
        const float m = sa * r * r * inv_d;                     // n mean(a n) = x r mean(a x r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float yl[W], yh[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (DW && hh < h1) { gl[c][j] += al[c][j] * (lo[c][j] * r); gh[c][j] += ah[c][j] * (hi[c][j] * r); }
                yl[j] = r * (al[c][j] * wl[c][j] - lo[c][j] * m);
                yh[j] = r * (ah[c][j] * wh[c][j] - hi[c][j] * m);
            }
            if (hh < h1 && L.on[c]) {
                store_w(dx + (int64_t)hh * D + L.lo[c], yl);
                store_w(dx + (int64_t)hh * D + L.hi[c], yh);
            }
        }
    }
}

// part [2][gridDim.x][D] (DW): every workgroup's weight gradient, summed over its waves and lane groups in a fixed order
template <typename T, int W, int LPH, int C, bool S, bool NT, bool DW>
__global__ __launch_bounds__(WAVES * 64) void qk_norm_rope_bwd_kernel(const mtl_qk_norm_rope_args a, float* __restrict__ part) {
    const Lane<W, LPH, C, S> L((int)a.D, (int)a.R);
    const int64_t rows = a.B * a.T;
    const float inv_d = 1.0f / (float)a.D;
    const Side s = side_of(a, blockIdx.y == 1);
    float wl[C][W], wh[C][W], gl[C][W], gh[C][W];
    load_weights(s.w, a.w_dtype, L, wl, wh);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < W; ++j) gl[c][j] = gh[c][j] = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * WAVES) {
        const int64_t b = row / a.T, t = row - b * a.T;
        float cs[C][W], sn[C][W];
        load_turn(a, b, t, L, cs, sn);
        heads_bwd<T, W, LPH, C, S, NT, DW>((const T*)s.x + b * s.x_bs + t * s.x_ts, (const T*)s.dy + b * s.dy_bs + t * s.dy_ts, (T*)s.y + b * s.y_bs + t * s.y_ts, s.H, (int)a.D, a.eps, inv_d, L, wl, wh, cs, sn,
                                    gl, gh);
    }
    if (!DW) return;
    constexpr int G = 64 / LPH;
    __shared__ float sums[WAVES * G * 2 * LPH * C * W];           // [waves * lane groups][D]
    const int slot = (threadIdx.x >> 6) * G + (threadIdx.x & 63) / LPH, D = (int)a.D;
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (L.on[c])
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (S && j < L.skip[c]) continue;               // (its neighbour has it)
                sums[slot * D + L.lo[c] + j] = gl[c][j];
                sums[slot * D + L.hi[c] + j] = gh[c][j];
            }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += WAVES * 64) {
        float x = 0.f;
#pragma unroll 8
        for (int k = 0; k < WAVES * G; ++k) x += sums[k * D + i];
        part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * D + i] = x;
    }
}

// dw[which][i] = sum over the workgroups of the backward: 16 waves take a sixteenth each, in order
__global__ __launch_bounds__(1024) void qk_norm_rope_dw_kernel(const float* __restrict__ part, int n, int D, float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = blockIdx.x * 64 + lane, which = blockIdx.y;
    float s = 0.f;
    if (i < D) {
        const int k0 = n * wave / 16, k1 = n * (wave + 1) / 16;
#pragma unroll 8
        for (int k = k0; k < k1; ++k) s += part[((int64_t)which * n + k) * D + i];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && i < D) {
        s = sums[0][lane];
#pragma unroll
        for (int w = 1; w < 16; ++w) s += sums[w][lane];
        (which ? dwk : dwq)[i] = s;
    }
}

// Workgroups per side; more rows are walked by the same ones. Forward 1024 / 2048: 29.2 / 30.8 us at 6656 x (32 + 8) heads of 128 in bf16, 14.2 / 16.4 at 8192 x 24 of 64, 57.6 / 55.8 at 8224 x 64 of 128.
// Backward 512 / 768 / 1536: 102 / 90 / 96 us at 8224 x 64 heads, 50 / 51 / 57 at 6656 x 40 (three of its workgroups fit a CU). Two of a wave's head steps in flight in the forward: 49 us, four
// 50 (without the loads below that pass the cache: 50, one step 57, four 55).
inline unsigned fwd_blocks(int64_t rows) { const int64_t b = (rows + WAVES - 1) / WAVES; return (unsigned)(b < 1024 ? b : 1024); }
inline unsigned bwd_blocks(int64_t rows) { const int64_t b = (rows + WAVES - 1) / WAVES; return (unsigned)(b < 768 ? b : 768); }

template <typename T, int W, int LPH, int C, bool S, bool NT>
int launch_with(const mtl_qk_norm_rope_args& a, bool bwd, hipStream_t st) {
    const int64_t rows = a.B * a.T;
    if (!bwd) {
        // One wave per row and side; where that leaves the chip empty, a row's heads go to several waves (each a whole number of the wave's head groups), up to 512 in all. 32 + 8 heads of 128:
        // 1 row 3.6 us (one wave 4.6), 32 rows 3.9 (5.3), 256 rows 4.6 (5.6); up to 4096 waves: 512 rows 7.5 against 5.9, 4000 rows 20.3 against 18.8.
        constexpr int G = 64 / LPH;
        int parts = 1;
        const int64_t steps = ((a.Hq > a.Hkv ? a.Hq : a.Hkv) + G - 1) / G;
        while (parts < steps && rows * parts < 512) parts *= 2;
        if (parts > steps) parts = (int)steps;
        const int hq = (int)(((a.Hq + parts - 1) / parts + G - 1) / G * G), hk = (int)(((a.Hkv + parts - 1) / parts + G - 1) / G * G);
        hipLaunchKernelGGL((qk_norm_rope_fwd_kernel<T, W, LPH, C, S, NT>), dim3(fwd_blocks(rows), 2, parts), dim3(WAVES * 64), 0, st, a, hq, hk);
        MTL_CHECK_LAUNCH();
        return MTL_OK;
    }
    const unsigned blocks = bwd_blocks(rows);
    float* part = reinterpret_cast<float*>(a.workspace);
    if (!a.dwq) {
        hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T, W, LPH, C, S, NT, false>), dim3(blocks, 2), dim3(WAVES * 64), 0, st, a, part);
        MTL_CHECK_LAUNCH();
        return MTL_OK;
    }
    hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T, W, LPH, C, S, NT, true>), dim3(blocks, 2), dim3(WAVES * 64), 0, st, a, part);
    MTL_CHECK_LAUNCH();
    hipLaunchKernelGGL(qk_norm_rope_dw_kernel, dim3((unsigned)((a.D + 63) / 64), 2), dim3(1024), 0, st, part, (int)blocks, (int)a.D, a.dwq, a.dwk);
    MTL_CHECK_LAUNCH();
    return MTL_OK;
}

// Queries and keys of 64 MiB and more (the backward reads dy's as much again) do not stay in the 256 MB cache behind what is written: their loads pass it by and leave it to the outputs, which are read
// next. Without / with, us, bf16 heads of 128: forward 42 MB 18.6 / 21.4, 67 MB 27.8 / 27.5, 101 MB 43.4 / 40.1, 135 MB 57.6 / 49.2, 270 MB 109 / 106; backward 42 MB 35.4 / 35.7, 67 MB 48.9 / 45.4,
// 101 MB 68.7 / 62.9, 135 MB 86.4 / 78.6, 270 MB 160 / 156. Between a projection and the attention: 67 MB 126 / 122, 135 MB 286 / 273. Only where every half of a head is whole lines of 128 bytes and a
// load takes 16 of each lane's: a line that two loads share comes twice (heads of 64, 101 MB: forward 51 / 52, backward 77 / 81; of 100: 78 / 83, 112 / 115; fp32, 135 MB: no gain). Stores that pass the
// cache by gain 6 % alone and lose up to 20 % with the kernel that reads them.
template <typename T, int W, int LPH, int C, bool S>
int launch(const mtl_qk_norm_rope_args& a, bool bwd, hipStream_t st) {
    if constexpr (W == 8 && LPH >= 8 && !S && sizeof(T) == 2)
        if (a.R % 128 == 0 && (a.D - a.R) % 128 == 0 && a.B * a.T * (a.Hq + a.Hkv) * a.D * 2 >= (int64_t)64 << 20) return launch_with<T, W, LPH, C, S, true>(a, bwd, st);
    return launch_with<T, W, LPH, C, S, false>(a, bwd, st);
}

// 8 pairs per lane where the rotated pairs and the others are at least 8 (or none); else one pair per lane and chunk
template <typename T, bool S>
int dispatch_wide(const mtl_qk_norm_rope_args& a, int chunks, bool bwd, hipStream_t st) {
    if (chunks <= 4) return launch<T, 8, 4, 1, S>(a, bwd, st);
    if (chunks <= 8) return launch<T, 8, 8, 1, S>(a, bwd, st);
    if (chunks <= 16) return launch<T, 8, 16, 1, S>(a, bwd, st);
    return launch<T, 8, 32, 1, S>(a, bwd, st);
}

template <typename T>
int dispatch(const mtl_qk_norm_rope_args& a, bool bwd, hipStream_t st) {
    const int rp = (int)(a.R / 2), rest = (int)((a.D - a.R) / 2), pairs = rp + rest;
    const int chunks = (rp + 7) / 8 + (rest + 7) / 8;
    if (rp >= 8 && (rest == 0 || rest >= 8) && chunks <= 32)
        return rp % 8 == 0 && rest % 8 == 0 ? dispatch_wide<T, false>(a, chunks, bwd, st) : dispatch_wide<T, true>(a, chunks, bwd, st);
    if (pairs <= 64) return launch<T, 1, 64, 1, false>(a, bwd, st);
    if (pairs <= 128) return launch<T, 1, 64, 2, false>(a, bwd, st);
    return launch<T, 1, 64, 4, false>(a, bwd, st);
}

int check_args(const mtl_qk_norm_rope_args* a, bool bwd) {
    if (!a || a->B < 0 || a->T < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D < 2 || a->R < 2 || a->D % 2 || a->R % 2 || a->R > a->D || a->n_pos < 0 || !(a->eps >= 0.f)) return MTL_ERR_ARG;
    if (a->D > 512 || a->Hq > 65536 || a->Hkv > 65536) return MTL_ERR_UNSUPPORTED;
    if ((a->dtype != MTL_F32 && a->dtype != MTL_BF16) || (a->w_dtype != MTL_F32 && a->w_dtype != MTL_BF16)) return MTL_ERR_ARG;
    if (bwd && !a->dwq != !a->dwk) return MTL_ERR_ARG;
    if (a->B == 0 || a->T == 0) return MTL_OK;
    if (!a->q || !a->k || !a->q_out || !a->k_out || !a->wq || !a->wk || !a->cos_t || !a->sin_t || a->n_pos == 0) return MTL_ERR_ARG;
    if (bwd && (!a->dq_out || !a->dk_out)) return MTL_ERR_ARG;
    const uintptr_t e = a->dtype == MTL_BF16 ? 1 : 3, w = a->w_dtype == MTL_BF16 ? 1 : 3;
    if ((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->q_out | (uintptr_t)a->k_out) & e) || (((uintptr_t)a->wq | (uintptr_t)a->wk) & w) || (((uintptr_t)a->cos_t | (uintptr_t)a->sin_t) & 3) ||
        ((uintptr_t)a->positions & (a->pos_i64 ? 7 : 3)))
        return MTL_ERR_ALIGN;
    if (bwd && ((((uintptr_t)a->dq_out | (uintptr_t)a->dk_out) & e) || (((uintptr_t)a->dwq | (uintptr_t)a->dwk | (uintptr_t)a->workspace) & 3))) return MTL_ERR_ALIGN;
    return MTL_OK;
}

__global__ void zero_pair_kernel(float* a, float* b, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) a[i] = b[i] = 0.f;
}

}  // namespace

extern "C" int mtl_qk_norm_rope_fwd(const mtl_qk_norm_rope_args* a, void* stream) {
    const int rc = check_args(a, false);
    if (rc) return rc;
    if (a->B == 0 || a->T == 0) return MTL_OK;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return a->dtype == MTL_BF16 ? dispatch<bf16_t>(*a, false, st) : dispatch<float>(*a, false, st);
}

extern "C" size_t mtl_qk_norm_rope_bwd_workspace_bytes(int64_t B, int64_t T, int64_t D) {
    if (B <= 0 || T <= 0 || D <= 0) return 16;
    return (size_t)bwd_blocks(B * T) * 2 * (size_t)D * 4;
}

extern "C" int mtl_qk_norm_rope_bwd(const mtl_qk_norm_rope_args* a, void* stream) {
    const int rc = check_args(a, true);
    if (rc) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (a->B == 0 || a->T == 0) {
        if (a->dwq) {
            hipLaunchKernelGGL(zero_pair_kernel, dim3((unsigned)((a->D + 255) / 256)), dim3(256), 0, st, a->dwq, a->dwk, (int)a->D);
            MTL_CHECK_LAUNCH();
        }
        return MTL_OK;
    }
    if (a->dwq && (!a->workspace || a->workspace_bytes < mtl_qk_norm_rope_bwd_workspace_bytes(a->B, a->T, a->D))) return MTL_ERR_WORKSPACE;
    return a->dtype == MTL_BF16 ? dispatch<bf16_t>(*a, true, st) : dispatch<float>(*a, true, st);
}
