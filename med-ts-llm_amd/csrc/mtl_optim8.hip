// Adam / AdamW step with the two moments held in 8 bits (mtl_adam8_step), their read-back (mtl_adam8_moments) and their packing (mtl_adam8_quantize).
//
// Blocks of 64 consecutive elements (flat index) share two power-of-two scales, one signed byte each:
//   m = e4m3(cm) 2^em       em = floor(log2 max |m|) - 7: the block's largest value lands in [128, 256] of e4m3's 448
//   r = u44(cr) 2^er        the ROOT of the second moment (v = r^2: half of v's exponent range), unsigned, 4 exponent and 4 mantissa bits:
//                           u44(c) = c for c < 16, else (16 + c % 16) 2^(c / 16 - 1); er = floor(log2 max r) - 17, so codes end at 240; 254 is infinity, 255 NaN
// Both formats are floating, so a power-of-two scale costs no precision, multiplies exactly, and a block whose scale changes keeps every value on its grid.
// r is rounded up or down by a threshold u(i, t) = frac(i a1 + t a2), (a1, a2) = the 2-D additive recurrence of the plastic number (1 / 1.3247.., 1 / 1.3247..^2):
// equidistributed over the elements of a step and over the steps of an element. Rounding to nearest would freeze r: with beta2 = 0.999 a step moves it by
// about 1 / 2000 of its value, half a grid step is 1 / 64 .. 1 / 32. No generator state: the step number and the element's index are all of it.
// |m| is rounded up or down by a threshold as well (MTL_ADAM8_M_THRESHOLD; 16 hashed bits of (step, index): m moves by 1 - beta1 of its distance to g, up to a whole grid step at a time, too
// fast for a recurrence to be independent of what it meets). To nearest, which a step without that flag does, is the closest code for ONE step, but over a run m stands still wherever
// (1 - beta1) |g - m| is below half a grid step: a constant gradient is held at 0.78 / 0.54 / 0.20 of its value (beta1 0.9 / 0.95 / 0.99), and what is left of a gradient that has
// stopped never goes, while r under it decays: a step of lr and more for ever. The thresholds cost nothing measurable of the fp32 step at
// 512 M elements (1304 / 1308 us), 16 % at 73 M (239 / 205), and 8 - 20 % of the bf16 step, whose arithmetic shows (56 M: 151 / 126 us). mtl_adam8_quantize, which rounds once and feeds nothing back, takes the nearest code.
// r > 0 never gets code 0 (m / (0 + eps) would explode); what is not finite becomes the NaN code of that element alone, but for a second moment that a finite gradient takes beyond
// fp32's range (|g| > 1.8e19): infinity, as with 32-bit moments (its parameter stands still).
//
// Every operation is ONE fp32 operation, rounded to nearest, in the order written (no contraction into fma, exact division and square root): a change in the last bit moves
// a value that sits at a rounding border to the next code, and this way the codes are a function of the inputs that any IEEE machine reproduces bit for bit.
#include "mtl_common.h"

#pragma clang fp contract(off)

namespace {

constexpr int MAX_T = MTL_ADAM8_MAX_TENSORS;
constexpr int THREADS = 256;
constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;      // 2^32 threads per launch: 17 G elements in fp32, 34 G in bf16
// 4 elements per lane and iteration; all loads of a workgroup's iterations are in flight before the first use. Iterations, measured at 512 M elements: fp32 step 1 / 2 / 4: 1351 / 1475 /
// 1413 us (6.1 TB/s); bf16 step 1066 / 968 / 1046 (5.3 TB/s: half of the bytes per element, the arithmetic shows). At 410 M elements, outputs not reused: read-back in fp32 659 / 689 / 737, in bf16
// 465 / 389 / 422, packing 934 / 966 / -. What these have in common: a workgroup moves 4 KB in a row of each wide array.
constexpr int ITERS_F32 = 1, ITERS_B16 = 2;
constexpr int chunk_of(int iters) { return THREADS * 4 * iters; }      // elements per workgroup: a whole number of 64-element blocks
inline __host__ __device__ int dtype_chunk(int64_t dtype) { return chunk_of(dtype == MTL_BF16 ? ITERS_B16 : ITERS_F32); }

struct Adam8Table {
    mtl_adam8_tensor t[MAX_T];
    int first_block[MAX_T + 1];
    int count;
};
struct Adam8Hyper { float om_b1, b2, om_b2, eps, wd, decay, inv_bc2, step_size; uint32_t t_thr, m_base; int mode; };   // mode: 0 no decay, 1 L2, 2 decoupled

struct State8Table {
    mtl_adam8_state t[MAX_T];
    int first_block[MAX_T + 1];
    int count;
};

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// largest of 16 lanes (one DPP row = one 64-element block at 4 elements per lane), in every one of them
template <int CTRL>
__device__ __forceinline__ uint32_t row_max_step(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
    return o > v ? o : v;
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = row_max_step<0x121>(v);       // row_ror 1, 2, 4, 8
    v = row_max_step<0x122>(v);
    v = row_max_step<0x124>(v);
    return row_max_step<0x128>(v);
}
__device__ __forceinline__ uint32_t max4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { const uint32_t x = a > b ? a : b, y = c > d ? c : d; return x > y ? x : y; }
__device__ __forceinline__ uint32_t min4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { const uint32_t x = a < b ? a : b, y = c < d ? c : d; return x < y ? x : y; }
constexpr uint32_t INF_BITS = 0x7f800000u;
// bits of |x|, 0 where it is not finite: ordered like the values
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < INF_BITS ? b : 0u;
}
__device__ __forceinline__ int scale_exp(uint32_t top_bits, int below) {
    const int e = (int)(top_bits >> 23) - 127 - below;
    return e < -126 ? -126 : e;                                // (the largest is 127 - 7)
}
__device__ __forceinline__ bool has_zero_byte(uint32_t x) { return ((x - 0x01010101u) & ~x & 0x80808080u) != 0; }

// The general forms of decoding and encoding handle every value; the step is bound by its arithmetic with them (bf16: 180 vector operations per element, 4.2 TB/s). What almost every wave
// meets are finite values within 2^13 of their block's largest, and for those the codes are fields of the fp32 numbers: u44(c) 2^er = bits (c + 2080 + 16 er) << 19 for c >= 16, and
// the threshold is added below the four mantissa bits that stay. A wave takes that path where all its values allow it (a uniform branch), with the same bits.
__device__ __forceinline__ void decode4(uint32_t cm, uint32_t cr, int em, int er, float (&m)[4], float (&r)[4]) {
    const float sm = pow2i(em);
    m[0] = __builtin_amdgcn_cvt_f32_fp8((int)cm, 0) * sm; m[1] = __builtin_amdgcn_cvt_f32_fp8((int)cm, 1) * sm;
    m[2] = __builtin_amdgcn_cvt_f32_fp8((int)cm, 2) * sm; m[3] = __builtin_amdgcn_cvt_f32_fp8((int)cm, 3) * sm;
    if (!__any(has_zero_byte(cr & 0xf0f0f0f0u) || has_zero_byte(~cr & 0xfefefefeu))) {      // no code below 16, no 254 or 255
        const uint32_t k = (uint32_t)(130 * 16 + 16 * er);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = __uint_as_float((((cr >> (8 * e)) & 0xffu) + k) << 19);
        return;
    }
    const float sr = pow2i(er);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t c = (cr >> (8 * e)) & 0xffu;
        float v = c < 16u ? (float)c : __uint_as_float((c + 130u * 16u) << 19);
        v = c >= 254u ? __uint_as_float(c == 254u ? INF_BITS : 0x7fc00000u) : v;
        r[e] = v * sr;
    }
}

__device__ __forceinline__ uint32_t encode_root(float r, float m, float inv, uint32_t u) {
    const float y = r * inv;
    const uint32_t large = ((__float_as_uint(y) + (u >> 13)) >> 19) - 130u * 16u;
    const uint32_t small = (uint32_t)__builtin_floorf(y + (float)(u >> 8) * 0x1p-24f);
    uint32_t c = y >= 16.0f ? large : small;
    c = (r > 0.f && c < 1u) ? 1u : c;
    if ((__float_as_uint(r) & INF_BITS) != INF_BITS) return c;
    return __float_as_uint(r) == INF_BITS && (__float_as_uint(m) & INF_BITS) != INF_BITS ? 254u : 255u;
}

// square root, rounded to nearest, of 0 and of x >= 2^-96: the hardware's estimate is off by at most one unit in the last place, and Tuckerman's test says which of it and its two neighbours
// it is: s is the rounded root of x where s pred(s) < x <= s succ(s) (Agarwal et al., New scalar and vector elementary functions for the IBM System/370, IBM J. Res. Dev. 30, 1986).
__device__ __forceinline__ float sqrt_near(float x) {
    float s = __builtin_amdgcn_sqrtf(x);
    const float down = __uint_as_float(__float_as_uint(s) - 1u), up = __uint_as_float(__float_as_uint(s) + 1u);
    const float rd = __builtin_fmaf(-down, s, x), ru = __builtin_fmaf(-up, s, x);
    s = rd <= 0.f ? down : s;
    return ru > 0.f ? up : s;
}

constexpr uint32_t DITHER_I = 0xC13FA9A9u;
constexpr uint32_t M_STREAM = 0x6D38u;          // the first moment's words of the counter hash

// e4m3 code of y, |y| <= 256, its magnitude rounded up where the fraction of a grid step and field / 2^16 (the middle of field's interval) reach one
__device__ __forceinline__ uint32_t encode_m(float y, uint32_t field) {
    const uint32_t b = __float_as_uint(y), a = b & 0x7fffffffu, u = field * 16u + 8u;
    const uint32_t normal = ((a + u) >> 20) - 120u * 8u;                                                                        // 2^-6 and more: three mantissa bits stay
    const uint32_t small = (uint32_t)__builtin_floorf(__uint_as_float(a) * 512.0f + (float)u * 0x1p-20f);                          // multiples of 2^-9
    return ((a >= 0x3c800000u ? normal : small) & 0x7fu) | ((b >> 24) & 0x80u);
}

// Codes of 4 elements and the block's exponents (the same in the 16 lanes of a block) from m and v; r[] receives sqrt(v). Every lane of the wave is active. M_THR: m against thresholds.
template <bool M_THR>
__device__ __forceinline__ void encode4(const float (&m)[4], const float (&v)[4], float (&r)[4], int64_t e0, uint32_t t_thr, uint32_t m_base, uint32_t& cm, uint32_t& cr, uint32_t& ex) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = sqrt_near(v[e]);
    uint32_t mb[4], rb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { mb[e] = __float_as_uint(m[e]) & 0x7fffffffu; rb[e] = __float_as_uint(r[e]); }
    uint32_t tm = row_max(max4(mb[0], mb[1], mb[2], mb[3])), tr = row_max(max4(rb[0], rb[1], rb[2], rb[3]));
    int em = scale_exp(tm, 7), er = scale_exp(tr, 17);
    const uint32_t u0 = (uint32_t)e0 * DITHER_I + t_thr;
    // 16 in the block's scale, and 2^-48: smaller roots come from v < 2^-96, for which sqrt_near is not exact
    const uint32_t least = (uint32_t)(131 + er) << 23, lo = least > 0x27800000u ? least : 0x27800000u;
    if (__any(tm >= INF_BITS || tr >= INF_BITS || min4(rb[0], rb[1], rb[2], rb[3]) < lo)) {
        tm = tr = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r[e] = __builtin_sqrtf(v[e]);
            const uint32_t a = finite_bits(m[e]), b = finite_bits(r[e]);
            tm = a > tm ? a : tm;
            tr = b > tr ? b : tr;
        }
        em = scale_exp(row_max(tm), 7); er = scale_exp(row_max(tr), 17);
        cr = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) cr |= encode_root(r[e], m[e], pow2i(-er), u0 + (uint32_t)e * DITHER_I) << (8 * e);
    } else {
        const uint32_t k = (uint32_t)(130 * 16 + 16 * er);
        cr = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) cr |= (((rb[e] + ((u0 + (uint32_t)e * DITHER_I) >> 13)) >> 19) - k) << (8 * e);
    }
    const float im = pow2i(-em);
    if constexpr (M_THR) {
        const uint64_t quad = (uint64_t)e0 >> 2;                // (the hash takes 24 bits of each of its two coordinates)
        const uint2 w = drop_quad(m_base, (uint32_t)(quad >> 24), (uint32_t)quad & 0xffffffu);
        cm = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) cm |= encode_m(m[e] * im, drop_field(w, (uint32_t)e)) << (8 * e);
    } else {
        int pk = __builtin_amdgcn_cvt_pk_fp8_f32(m[0] * im, m[1] * im, 0, false);
        pk = __builtin_amdgcn_cvt_pk_fp8_f32(m[2] * im, m[3] * im, pk, true);
        cm = (uint32_t)pk;
    }
    if (__any(max4(mb[0], mb[1], mb[2], mb[3]) >= INF_BITS))
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (mb[e] >= INF_BITS) cm = (cm & ~(0xffu << (8 * e))) | (0x7fu << (8 * e));
    ex = ((uint32_t)em & 0xffu) | (((uint32_t)er & 0xffu) << 8);
}

// 4 code bytes at p, nv of them in range
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int nv, bool vec) {
    if (vec && nv == 4) return *reinterpret_cast<const uint32_t*>(p);
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < nv) c |= (uint32_t)p[e] << (8 * e);
    return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint32_t c, int nv, bool vec) {
    if (vec && nv == 4) { *reinterpret_cast<uint32_t*>(p) = c; return; }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < nv) p[e] = (uint8_t)(c >> (8 * e));
}

// new moments (v: the second moment itself), and the update once their root is known
__device__ __forceinline__ void adam8_moments_of(float& p, float g, float& m, float r, float& v, const Adam8Hyper& h) {
    v = r * r;
    if (h.mode == 2) p = p * h.decay;
    else if (h.mode == 1) g = g + p * h.wd;
    m = m + (g - m) * h.om_b1;
    v = v * h.b2 + (g * g) * h.om_b2;
}
__device__ __forceinline__ float adam8_update(float p, float m, float r, const Adam8Hyper& h) { return p - (m / (r * h.inv_bc2 + h.eps)) * h.step_size; }

// HBM-bound: fp32 16 + 4/64 B per element (p read and written, g read, two code bytes read and written, two exponent bytes per 64 elements each way), bf16 10 + 4/64.
template <bool P16, bool M_THR>
__device__ __forceinline__ void adam8_chunk(const mtl_adam8_tensor& t, int64_t base, const Adam8Hyper& h) {
    float* p32 = reinterpret_cast<float*>(t.p);
    const float* g32 = reinterpret_cast<const float*>(t.g);
    bf16_t* p16 = reinterpret_cast<bf16_t*>(t.p);
    const bf16_t* g16 = reinterpret_cast<const bf16_t*>(t.g);
    const bool vec = (((uintptr_t)t.p | (uintptr_t)t.g) & (P16 ? 7 : 15)) == 0;
    const bool vec8 = (((uintptr_t)t.m8 | (uintptr_t)t.r8) & 3) == 0;
    constexpr int ITERS = P16 ? ITERS_B16 : ITERS_F32;
    float pp[ITERS][4], gg[ITERS][4];
    uint32_t cm[ITERS], cr[ITERS], ex[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int64_t e0 = base + ((int64_t)i * THREADS + threadIdx.x) * 4;
        const int64_t left = t.n - e0;
        const int nv = left >= 4 ? 4 : (left > 0 ? (int)left : 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) pp[i][e] = gg[i][e] = 0.f;
        cm[i] = cr[i] = ex[i] = 0;
        if (nv > 0) {
            ex[i] = *reinterpret_cast<const uint16_t*>(t.ex + (e0 >> 6) * 2);
            cm[i] = load_codes(t.m8 + e0, nv, vec8);
            cr[i] = load_codes(t.r8 + e0, nv, vec8);
            if (P16) {
                if (vec && nv == 4) {
                    const u32x2 a = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p16 + e0)), b = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(g16 + e0));
                    pp[i][0] = __uint_as_float(a[0] << 16); pp[i][1] = __uint_as_float(a[0] & 0xffff0000u); pp[i][2] = __uint_as_float(a[1] << 16); pp[i][3] = __uint_as_float(a[1] & 0xffff0000u);
                    gg[i][0] = __uint_as_float(b[0] << 16); gg[i][1] = __uint_as_float(b[0] & 0xffff0000u); gg[i][2] = __uint_as_float(b[1] << 16); gg[i][3] = __uint_as_float(b[1] & 0xffff0000u);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < nv) { pp[i][e] = bf16_to_f32(p16[e0 + e]); gg[i][e] = bf16_to_f32(g16[e0 + e]); }
                }
            } else if (vec && nv == 4) {
                const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p32 + e0)), b = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(g32 + e0));
#pragma unroll
                for (int e = 0; e < 4; ++e) { pp[i][e] = a[e]; gg[i][e] = b[e]; }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < nv) { pp[i][e] = p32[e0 + e]; gg[i][e] = g32[e0 + e]; }
            }
        }
    }
    bf16_t* sh = reinterpret_cast<bf16_t*>(t.shadow);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int64_t e0 = base + ((int64_t)i * THREADS + threadIdx.x) * 4;
        const int64_t left = t.n - e0;
        const int nv = left >= 4 ? 4 : (left > 0 ? (int)left : 0);
        float m[4], r[4], v[4];
        decode4(cm[i], cr[i], (int8_t)(ex[i] & 0xffu), (int8_t)(ex[i] >> 8), m, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            adam8_moments_of(pp[i][e], gg[i][e], m[e], r[e], v[e], h);
            if (e >= nv) m[e] = v[e] = 0.f;                     // (elements behind the tensor's end have no part in their block's scales)
        }
        uint32_t nm, nr, nx;
        encode4<M_THR>(m, v, r, e0, h.t_thr, h.m_base, nm, nr, nx);
#pragma unroll
        for (int e = 0; e < 4; ++e) pp[i][e] = adam8_update(pp[i][e], m[e], r[e], h);
        if (nv == 0) continue;                                  // (no cross-lane operation below)
        store_codes(t.m8 + e0, nm, nv, vec8);
        store_codes(t.r8 + e0, nr, nv, vec8);
        if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint16_t*>(t.ex + (e0 >> 6) * 2) = (uint16_t)nx;
        if (P16) {
            const u32x2 pk = {pack_bf16x2(pp[i][0], pp[i][1]), pack_bf16x2(pp[i][2], pp[i][3])};      // one rounding of the updated parameter
            if (vec && nv == 4) __builtin_nontemporal_store(pk, reinterpret_cast<u32x2*>(p16 + e0));
            else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < nv) p16[e0 + e] = f32_to_bf16(pp[i][e]);
            }
        } else if (vec && nv == 4) {
            __builtin_nontemporal_store((f32x4){pp[i][0], pp[i][1], pp[i][2], pp[i][3]}, reinterpret_cast<f32x4*>(p32 + e0));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < nv) p32[e0 + e] = pp[i][e];
        }
        if (sh) {                                               // bf16 copy [n / cols, ld_shadow] of the updated weight
            const uint32_t cols = (uint32_t)t.cols;
            uint32_t row = (uint32_t)e0 / cols, col = (uint32_t)e0 - row * cols;
            if (nv == 4 && col + 4 <= cols) {                   // one 8-byte store wherever the four sit in one row (2-byte aligned where cols is odd)
                typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
                *reinterpret_cast<u32x2_any*>(sh + (int64_t)row * t.ld_shadow + col) = (u32x2_any){pack_bf16x2(pp[i][0], pp[i][1]), pack_bf16x2(pp[i][2], pp[i][3])};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (e < nv) sh[(int64_t)row * t.ld_shadow + col] = f32_to_bf16(pp[i][e]);
                    if (++col == cols) { col = 0; ++row; }
                }
            }
        }
    }
}

template <bool M_THR>
__global__ __launch_bounds__(THREADS) void adam8_step_kernel(const Adam8Table tab, const Adam8Hyper h) {
    int ti = 0;
    const int b = blockIdx.x;
    while (ti + 1 < tab.count && b >= tab.first_block[ti + 1]) ++ti;
    const mtl_adam8_tensor t = tab.t[ti];
    const int64_t at = b - tab.first_block[ti];
    if (t.param_dtype == MTL_BF16) adam8_chunk<true, M_THR>(t, at * chunk_of(ITERS_B16), h);
    else adam8_chunk<false, M_THR>(t, at * chunk_of(ITERS_F32), h);
}

template <bool NT, typename V>
__device__ __forceinline__ void store_vec(V x, void* p) {
    if constexpr (NT) __builtin_nontemporal_store(x, reinterpret_cast<V*>(p));
    else *reinterpret_cast<V*>(p) = x;
}
template <bool B16, bool NT>
__device__ __forceinline__ void store_moment(void* dst, int64_t e0, int nv, const float (&x)[4]) {
    if (!dst) return;
    if constexpr (B16) {
        bf16_t* d = reinterpret_cast<bf16_t*>(dst) + e0;
        if (nv == 4 && ((uintptr_t)d & 7) == 0) return store_vec<NT>((u32x2){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])}, d);
        for (int e = 0; e < nv; ++e) d[e] = f32_to_bf16(x[e]);
    } else {
        float* d = reinterpret_cast<float*>(dst) + e0;
        if (nv == 4 && ((uintptr_t)d & 15) == 0) return store_vec<NT>((f32x4){x[0], x[1], x[2], x[3]}, d);
        for (int e = 0; e < nv; ++e) d[e] = x[e];
    }
}

template <bool B16, bool NT>
__device__ __forceinline__ void moments_chunk(const mtl_adam8_state& t, int64_t at) {
    constexpr int ITERS = B16 ? ITERS_B16 : ITERS_F32;
    const int64_t base = at * chunk_of(ITERS);
    const bool vec8 = (((uintptr_t)t.m8 | (uintptr_t)t.r8) & 3) == 0;
    uint32_t cm[ITERS], cr[ITERS], ex[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int64_t e0 = base + ((int64_t)i * THREADS + threadIdx.x) * 4, left = t.n - e0;
        const int nv = left >= 4 ? 4 : (left > 0 ? (int)left : 0);
        cm[i] = cr[i] = ex[i] = 0;
        if (nv > 0) {
            ex[i] = *reinterpret_cast<const uint16_t*>(t.ex + (e0 >> 6) * 2);
            cm[i] = load_codes(t.m8 + e0, nv, vec8);
            cr[i] = load_codes(t.r8 + e0, nv, vec8);
        }
    }
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int64_t e0 = base + ((int64_t)i * THREADS + threadIdx.x) * 4, left = t.n - e0;
        const int nv = left >= 4 ? 4 : (left > 0 ? (int)left : 0);
        if (nv == 0) break;
        float m[4], r[4], v[4];
        decode4(cm[i], cr[i], (int8_t)(ex[i] & 0xffu), (int8_t)(ex[i] >> 8), m, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = r[e] * r[e];
        store_moment<B16, NT>(t.m, e0, nv, m);
        store_moment<B16, NT>(t.v, e0, nv, v);
    }
}

// read-back of the codes: 2 B read, 4 (bf16) or 8 B written per element. NT: the written moments pass the cache by; where a call writes 192 MiB and more they would not stay in it for their reader.
// Without / with, us, alone and with a copy behind it: 76 M elements fp32 (612 MB) 128 / 107, 302 / 278; 59 M bf16 (235 MB) 60 / 50, 154 / 148; but 17 M fp32 (134 MB) 26.9 / 25.3, 57 / 63.
template <bool NT>
__global__ __launch_bounds__(THREADS) void adam8_moments_kernel(const State8Table tab) {
    int ti = 0;
    const int b = blockIdx.x;
    while (ti + 1 < tab.count && b >= tab.first_block[ti + 1]) ++ti;
    const mtl_adam8_state t = tab.t[ti];
    if (t.dtype == MTL_BF16) moments_chunk<true, NT>(t, b - tab.first_block[ti]);
    else moments_chunk<false, NT>(t, b - tab.first_block[ti]);
}

// packing of fp32 moments (taking over a run whose moments are held in 32 bits)
__global__ __launch_bounds__(THREADS) void adam8_quantize_kernel(const State8Table tab, uint32_t t_thr) {
    int ti = 0;
    const int b = blockIdx.x;
    while (ti + 1 < tab.count && b >= tab.first_block[ti + 1]) ++ti;
    const mtl_adam8_state t = tab.t[ti];
    const int64_t base = (int64_t)(b - tab.first_block[ti]) * chunk_of(ITERS_F32);
    const bool vec8 = (((uintptr_t)t.m8 | (uintptr_t)t.r8) & 3) == 0;
    const float* ms = reinterpret_cast<const float*>(t.m);
    const float* vs = reinterpret_cast<const float*>(t.v);
    const bool vec = (((uintptr_t)ms | (uintptr_t)vs) & 15) == 0;
#pragma unroll
    for (int i = 0; i < ITERS_F32; ++i) {
        const int64_t e0 = base + ((int64_t)i * THREADS + threadIdx.x) * 4;
        const int64_t left = t.n - e0;
        const int nv = left >= 4 ? 4 : (left > 0 ? (int)left : 0);
        float m[4], v[4], r[4];
        if (nv == 4 && vec) {
            const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(ms + e0)), b = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(vs + e0));
#pragma unroll
            for (int e = 0; e < 4; ++e) { m[e] = a[e]; v[e] = b[e]; }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = e < nv ? ms[e0 + e] : 0.f;
                v[e] = e < nv ? vs[e0 + e] : 0.f;
            }
        }
        uint32_t nm, nr, nx;
        encode4<false>(m, v, r, e0, t_thr, 0u, nm, nr, nx);
        if (nv == 0) continue;
        store_codes(t.m8 + e0, nm, nv, vec8);
        store_codes(t.r8 + e0, nr, nv, vec8);
        if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint16_t*>(t.ex + (e0 >> 6) * 2) = (uint16_t)nx;
    }
}

int check_state(const mtl_adam8_state& t, bool read_back) {
    if (t.n < 0 || (t.n > 0 && (!t.m8 || !t.r8 || !t.ex))) return MTL_ERR_ARG;
    if (t.n > 0 && !read_back && (!t.m || !t.v)) return MTL_ERR_ARG;
    if ((uintptr_t)t.ex & 1) return MTL_ERR_ALIGN;
    if (t.dtype != MTL_F32 && !(read_back && t.dtype == MTL_BF16)) return MTL_ERR_ARG;
    if (t.n > MAX_BLOCKS * dtype_chunk(t.dtype)) return MTL_ERR_UNSUPPORTED;
    return ((uintptr_t)t.m | (uintptr_t)t.v) & (t.dtype == MTL_F32 ? 3 : 1) ? MTL_ERR_ALIGN : MTL_OK;
}

template <typename Launch>
int for_tables(const mtl_adam8_state* states, int count, bool read_back, Launch launch) {
    for (int i = 0; i < count; ++i)
        if (const int rc = check_state(states[i], read_back)) return rc;
    for (int i = 0; i < count;) {
        State8Table tab;
        tab.count = 0;
        int64_t blocks = 0;
        for (; i < count && tab.count < MAX_T; ++i) {
            if (states[i].n == 0) continue;
            const int64_t nb = (states[i].n + dtype_chunk(states[i].dtype) - 1) / dtype_chunk(states[i].dtype);
            if (blocks + nb > MAX_BLOCKS) break;                // (this one goes into the next launch)
            tab.t[tab.count] = states[i];
            tab.first_block[tab.count++] = (int)blocks;
            blocks += nb;
        }
        tab.first_block[tab.count] = (int)blocks;
        if (blocks == 0) continue;
        launch(tab, (unsigned)blocks);
        MTL_CHECK_LAUNCH();
    }
    return MTL_OK;
}

}  // namespace

extern "C" int mtl_adam8_step(const mtl_adam8_tensor* tensors, int count, double lr, double beta1, double beta2, double eps, double weight_decay, int flags, int64_t step, void* stream) {
    if (count < 0 || (count > 0 && !tensors) || step < 1 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0) || (flags & ~(MTL_ADAM8_DECOUPLED | MTL_ADAM8_M_THRESHOLD))) return MTL_ERR_ARG;
    for (int i = 0; i < count; ++i) {
        const mtl_adam8_tensor& t = tensors[i];
        if (t.n < 0 || (t.param_dtype != MTL_F32 && t.param_dtype != MTL_BF16)) return MTL_ERR_ARG;
        if (t.n == 0) continue;
        if (!t.p || !t.g || !t.m8 || !t.r8 || !t.ex) return MTL_ERR_ARG;
        if (t.n > MAX_BLOCKS * dtype_chunk(t.param_dtype)) return MTL_ERR_UNSUPPORTED;
        if ((((uintptr_t)t.p | (uintptr_t)t.g) & (t.param_dtype == MTL_BF16 ? 1 : 3)) || ((uintptr_t)t.ex & 1) || ((uintptr_t)t.shadow & 1)) return MTL_ERR_ALIGN;
        if (t.shadow && (t.cols <= 0 || t.ld_shadow < t.cols || t.n % t.cols != 0 || t.n >= ((int64_t)1 << 32))) return MTL_ERR_ARG;
    }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    Adam8Hyper h;
    h.om_b1 = (float)(1.0 - beta1); h.b2 = (float)beta2; h.om_b2 = (float)(1.0 - beta2); h.eps = (float)eps; h.wd = (float)weight_decay;
    h.decay = (float)(1.0 - lr * weight_decay);
    h.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    h.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
    h.t_thr = (uint32_t)step * 0x91E10DA5u;
    h.m_base = drop_base((uint32_t)step, M_STREAM);
    h.mode = weight_decay == 0.0 ? 0 : (flags & MTL_ADAM8_DECOUPLED ? 2 : 1);
    for (int i = 0; i < count;) {
        Adam8Table tab;
        tab.count = 0;
        int64_t blocks = 0;
        double bytes = 0;
        for (; i < count && tab.count < MAX_T; ++i) {
            const mtl_adam8_tensor& t = tensors[i];
            if (t.n == 0) continue;
            const int64_t nb = (t.n + dtype_chunk(t.param_dtype) - 1) / dtype_chunk(t.param_dtype);
            if (blocks + nb > MAX_BLOCKS) break;
            tab.t[tab.count] = t;
            tab.first_block[tab.count++] = (int)blocks;
            blocks += nb;
            bytes += (double)t.n * ((t.param_dtype == MTL_BF16 ? 10.0 : 16.0) + 4.0 / 64 + (t.shadow ? 2.0 : 0.0));
        }
        tab.first_block[tab.count] = (int)blocks;
        if (blocks == 0) continue;
        if (flags & MTL_ADAM8_M_THRESHOLD) MTL_LAUNCH("adam8_step_kernel", bytes, 1, adam8_step_kernel<true>, dim3((unsigned)blocks), dim3(THREADS), 0, st, tab, h);
        else MTL_LAUNCH("adam8_step_kernel", bytes, 1, adam8_step_kernel<false>, dim3((unsigned)blocks), dim3(THREADS), 0, st, tab, h);
        MTL_CHECK_LAUNCH();
    }
    return MTL_OK;
}

extern "C" int mtl_adam8_moments(const mtl_adam8_state* states, int count, void* stream) {
    if (count < 0 || (count > 0 && !states)) return MTL_ERR_ARG;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return for_tables(states, count, true, [&](const State8Table& tab, unsigned blocks) {
        int64_t bytes = 0;
        for (int i = 0; i < tab.count; ++i) bytes += tab.t[i].n * (tab.t[i].dtype == MTL_BF16 ? 2 : 4) * ((tab.t[i].m != nullptr) + (tab.t[i].v != nullptr));
        if (bytes >= (int64_t)192 << 20) hipLaunchKernelGGL(adam8_moments_kernel<true>, dim3(blocks), dim3(THREADS), 0, st, tab);
        else hipLaunchKernelGGL(adam8_moments_kernel<false>, dim3(blocks), dim3(THREADS), 0, st, tab);
    });
}

extern "C" int mtl_adam8_quantize(const mtl_adam8_state* states, int count, int64_t step, void* stream) {
    if (count < 0 || (count > 0 && !states) || step < 0) return MTL_ERR_ARG;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return for_tables(states, count, false, [&](const State8Table& tab, unsigned blocks) {
        hipLaunchKernelGGL(adam8_quantize_kernel, dim3(blocks), dim3(THREADS), 0, st, tab, (uint32_t)step * 0x91E10DA5u);
    });
}
