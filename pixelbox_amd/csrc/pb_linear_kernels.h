// pb_linear_kernels.h -- kernels of the linear layers on device buffers (pb_quantize_rows, pb_linear_i8, pb_group_rows,
// pb_linear_grouped): y = act(x w^T * scales + bias), both operands with the summed axis contiguous.
//
// One byte layout serves every type.  A matrix instruction of 16 x 16 outputs takes 16 bytes per lane from each operand -- lane l
// holds bytes [16 (l / 16), + 16) of a 64-byte piece of row l % 16 --, which is 16 k of i8, 8 of bf16 / f16 and 4 of f32 (four
// v_mfma_f32_16x16x4_f32, one per element: the order of k inside a piece is the same for both operands, so the sum is over the
// same pairs).  The 32 x 32 forms take 32-byte pieces of 32 rows.  Kernels therefore move bytes and only the instruction knows the
// type.  The weights are the first operand: a lane then holds four CONSECUTIVE output channels of one row.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "pb_embed_common.h"

namespace pbl {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum { F32 = PB_TYPE_F32, BF16 = PB_TYPE_BF16, F16 = PB_TYPE_F16, I8 = PB_TYPE_I8 };

__host__ __device__ constexpr int type_bytes(int t) { return t == F32 ? 4 : t == I8 ? 1 : 2; }

// ---- one matrix step --------------------------------------------------------------------------------------------------------------
template <int T> struct Acc {
    typedef f32x4 q4;
    typedef f32x16 q16;
    typedef float e;
};
template <> struct Acc<I8> {
    typedef i32x4 q4;
    typedef i32x16 q16;
    typedef int e;
};

template <int T>
__device__ __forceinline__ void mma16(typename Acc<T>::q4 &c, const u32x4 &a, const u32x4 &b) {
    if constexpr (T == I8) c = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    else if constexpr (T == BF16) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (T == F16) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else {
        const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(af[e], bf[e], c, 0, 0, 0);
    }
}
template <int T>
__device__ __forceinline__ void mma32(typename Acc<T>::q16 &c, const u32x4 &a, const u32x4 &b) {
    if constexpr (T == I8) c = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    else if constexpr (T == BF16) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (T == F16) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else {
        const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(af[e], bf[e], c, 0, 0, 0);
    }
}

// ---- loads and stores of any alignment ---------------------------------------------------------------------------------------------------
// global_load / store_dwordx4 take any address; what that costs depends on the bound.  Tiles load a byte once for many products: on
// 4 bytes or less they lose what the way through registers costs (4096^3 i8 66 us aligned, 100 on 4 bytes, 134 odd).  The few forms live on
// loads, which go at full rate on 4 bytes and at a third off them (41 x 217 x 3903 f16: 26.6 us, with 3904 values 10.1): there (DW false)
// the aligned words around the 16 bytes are read -- only such as hold at least one of them -- and shifted into place (12.9 us; in
// tiles that costs more than it saves: 777 x 1003 x 1289 i8 with the operands in the caches 12.6 us, plain 11.2).
template <bool DW>
__device__ __forceinline__ u32x4 load16(const uint8_t *p) {
    u32x4 v;
    if constexpr (DW) {
        __builtin_memcpy(&v, p, 16);
        return v;
    } else {
        const uint32_t sh = (uint32_t)(uintptr_t)p & 3u;
        const uint8_t *d = p - sh;
        __builtin_memcpy(&v, __builtin_assume_aligned(d, 4), 16);
        const uint32_t e = *reinterpret_cast<const uint32_t *>(d + (sh ? 16 : 12));
        return u32x4{__builtin_amdgcn_alignbyte(v.y, v.x, sh), __builtin_amdgcn_alignbyte(v.z, v.y, sh), __builtin_amdgcn_alignbyte(v.w, v.z, sh),
                     __builtin_amdgcn_alignbyte(e, v.w, sh)};
    }
}
__device__ __forceinline__ void store16(uint8_t *p, const u32x4 &v) { __builtin_memcpy(p, &v, 16); }
// bytes [at, at + 16) of a row of `len` bytes, zero behind its end; reads nothing outside [0, len).  Without a branch for rows of 16
// bytes and more, so that several such loads are on their way together: the row's last 16 bytes, shifted down.
template <bool DW>
__device__ __forceinline__ u32x4 load16_tail(const uint8_t *row, int at, int len) {
    if (len >= 16) {
        const int off = min(at, len - 16), s = 8 * (at - off);
        const u32x4 t = load16<DW>(row + off);
        const uint64_t lo = ((uint64_t)t.y << 32) | t.x, hi = ((uint64_t)t.w << 32) | t.z;
        const uint64_t l2 = s == 0 ? lo : s < 64 ? (lo >> s) | (hi << (64 - s)) : s < 128 ? hi >> (s - 64) : 0;
        const uint64_t h2 = s < 64 ? hi >> s : 0;
        return u32x4{(uint32_t)l2, (uint32_t)(l2 >> 32), (uint32_t)h2, (uint32_t)(h2 >> 32)};
    }
    uint64_t half[2] = {0, 0};  // rows shorter than one piece
#pragma unroll 1
    for (int i = 0; at + i < len; ++i) {
        const uint64_t b = (uint64_t)row[at + i] << (8 * (i & 7));
        half[0] |= i < 8 ? b : 0;
        half[1] |= i < 8 ? 0 : b;
    }
    return u32x4{(uint32_t)half[0], (uint32_t)(half[0] >> 32), (uint32_t)half[1], (uint32_t)(half[1] >> 32)};
}

// ---- arguments of a product -----------------------------------------------------------------------------------------------------------
struct LinearArgs {
    const uint8_t *x, *w;
    const float *x_scale, *w_scale, *bias;
    const int32_t *offsets, *x_rows, *y_rows;
    uint8_t *y;
    long ldx, ldw, ldy;      // bytes between rows
    int kb;                  // bytes summed over (k <= 2^28)
    int m, n, groups;
    int nt0, n_tiles;        // this launch's tiles of output channels
    int x_total, y_total;    // rows of x and y: an index outside them is no row
    int act, y_type;
};

// ---- which rows a workgroup works on ----------------------------------------------------------------------------------------------------
// Groups are cut into tiles of BM rows; tile numbers run over the groups in order.  Every wave finds its tile by itself: lanes
// look at 64 groups at a time and add up their tile counts.  Offsets are data of the device: they are clamped to [0, m], a group
// that runs backwards is empty, so that nothing outside the buffers is touched whatever they hold.
struct Tile {
    int g, r0, r1;  // rows [r0, r1) of the order; r0 >= r1: nothing to do
    int nt;         // tile of output channels
};

// inclusive prefix sum over the wave's 64 lanes
__device__ __forceinline__ int wave_prefix(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // lane 15 of rows 0 and 2 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
    return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {  // in lane 63
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
    return v;
}

template <int BM, int BAND>
__device__ __forceinline__ Tile find_tile(const LinearArgs &a) {
    const int lane = threadIdx.x & 63;
    // group g0 + lane: its rows, and how many tiles the groups g0 .. g0 + lane have
    int lo = 0, hi = 0, c = 0, inc = 0;
    auto look = [&](int g0) {
        lo = hi = 0;
        if (g0 + lane < a.groups) {
            lo = min(max(a.offsets[g0 + lane], 0), a.m);
            hi = max(lo, min(a.offsets[g0 + lane + 1], a.m));
        }
        c = (hi - lo + BM - 1) / BM;
        inc = wave_prefix(c);
    };
    long m_tiles = 0;
    if (a.offsets) {
        for (int g0 = 0; g0 < a.groups; g0 += 64) {
            look(g0);
            m_tiles += __builtin_amdgcn_readlane(inc, 63);
        }
    } else m_tiles = (a.m + BM - 1) / BM;
    Tile t = {0, 0, 0, 0};
    // workgroups go round robin over the 8 XCDs: XCD x takes a contiguous eighth of the tiles, so that its L2 sees few panels.  A
    // group's tiles follow one another; inside it, BAND row tiles go through the channel tiles together.
    const long total = m_tiles * a.n_tiles, per = (total + 7) / 8;
    const long b = blockIdx.x, in = b >> 3;
    long id = (b & 7) * per + in;
    if (in >= per || id >= total) return t;
    int lo_g = 0, hi_g = a.m, tiles_g = (int)m_tiles;
    if (a.offsets) {
        for (int g0 = 0; g0 < a.groups; g0 += 64) {
            if (a.groups > 64) look(g0);
            const uint64_t past = __ballot((long)inc * a.n_tiles > id);
            if (past) {
                const int l = __builtin_ctzll(past);
                t.g = g0 + l;
                lo_g = __builtin_amdgcn_readlane(lo, l);
                hi_g = __builtin_amdgcn_readlane(hi, l);
                tiles_g = __builtin_amdgcn_readlane(c, l);
                id -= (long)(__builtin_amdgcn_readlane(inc, l) - tiles_g) * a.n_tiles;
                break;
            }
            id -= (long)__builtin_amdgcn_readlane(inc, 63) * a.n_tiles;
        }
    }
    const int band = (int)(id / ((long)BAND * a.n_tiles));
    const int rest = (int)(id - (long)band * BAND * a.n_tiles), bh = min(BAND, tiles_g - band * BAND);
    t.nt = a.nt0 + rest / bh;
    t.r0 = lo_g + (band * BAND + rest % bh) * BM;
    t.r1 = t.r0 < lo_g ? t.r0 : min(t.r0 + BM, hi_g);  // offsets that do not ascend may count more tiles than an int holds: none then
    return t;
}

// ---- epilogue: scales, bias, activation, one rounding, store ------------------------------------------------------------------------------
// tanh: from 1 on 1 - 2 t with t = e / (1 + e), e = exp(-2 |x|), and x's sign; below, where that loses digits, x + x^3 P(x^2) with P of degree
// 6, fitted to tanh so that the largest relative error over (0, 1] is least (0.08 units of 2^-24).  Within 4 units: t is off by (4 |x| + 2)
// / (1 + e) units from the exponential (its argument's two roundings and its own), 4 from the sum, the reciprocal and the product, of which the
// result takes 2 t / tanh x, at most 0.31 (at 1), and the last step is one more; below 1 the cubic part is off by 5 units, of which the result
// takes as much, and the last step is one more.  Measured over 3.2 million values: 1.74 units at worst, 0.40 in
// the mean square.  14 of the 57 us of 4330 x 7218 x 64; the library's tanhf took 26 of 63.
__device__ __forceinline__ float tanh_f(float x) {
    const float a = fabsf(x), e = __builtin_amdgcn_exp2f(a * -2.8853900817779268f), t = e * __builtin_amdgcn_rcpf(1.0f + e), z = x * x;
    float p = __builtin_fmaf(z, -0.0003584913210943341f, 0.0023015032056719065f);
    p = __builtin_fmaf(z, p, -0.007946296595036983f);
    p = __builtin_fmaf(z, p, 0.021486785262823105f);
    p = __builtin_fmaf(z, p, -0.05387984588742256f);
    p = __builtin_fmaf(z, p, 0.13332344591617584f);
    p = __builtin_fmaf(z, p, -0.33333295583724976f);
    return a < 1.0f ? __builtin_fmaf(x * z, p, x) : copysignf(__builtin_fmaf(t, -2.0f, 1.0f), x);
}
__device__ __forceinline__ float act_f(float v, int act) {
    if (act == PB_ACT_SILU) return pbe::silu_f(v);
    if (act == PB_ACT_TANH) return tanh_f(v);
    return v;
}
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// two values rounded to the nearest bf16 / f16 (halves to even), packed
__device__ __forceinline__ uint32_t pack2(float x, float y, int type) {
    const f32x2 v = {x, y};
    return type == BF16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2)) : __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// W consecutive channels [c0, ..) of y row yr
template <int W>
__device__ __forceinline__ void store_row(const LinearArgs &a, int yr, int c0, const float (&v)[W]) {
    if (c0 >= a.n) return;
    uint8_t *row = a.y + (long)yr * a.ldy;
    const bool whole = c0 + W <= a.n;
    if (a.y_type == F32) {
        float *p = reinterpret_cast<float *>(row) + c0;
        if (whole) __builtin_memcpy(p, v, 4 * W);
        else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (c0 + i < a.n) p[i] = v[i];
        }
    } else {
        uint16_t *p = reinterpret_cast<uint16_t *>(row) + c0;
        uint32_t h[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) h[i] = pack2(v[2 * i], v[2 * i + 1], a.y_type);
        if (whole) __builtin_memcpy(p, h, 2 * W);
        else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (c0 + i < a.n) p[i] = (uint16_t)(h[i / 2] >> (16 * (i & 1)));
        }
    }
}

// what a lane needs of its W output channels
template <int T, int W> struct Chan {
    float scale[W], bias[W];
    __device__ __forceinline__ void load(const LinearArgs &a, int g, int c0) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const bool in = c0 + i < a.n;
            const long at = (long)g * a.n + c0 + i;
            scale[i] = T == I8 && in ? a.w_scale[at] : 1.0f;
            bias[i] = a.bias && in ? a.bias[at] : 0.0f;
        }
    }
    // PLAIN: no activation, whole vectors of a known type YT -- what the large products mostly are, without a branch per row
    template <bool PLAIN = false, int YT = 0>
    __device__ __forceinline__ void finish(const LinearArgs &a, const typename Acc<T>::e (&s)[W], float row_scale, int yr, int c0) const {
        float v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = (float)s[i];
        if constexpr (T == I8) {
            // the sum times the row's scale leaves the range of f32 where the result need not: rows of values beyond 10^31 (a sum has up to 31
            // bits), and scales near the smallest ones.  There a power of two is taken out and put back
            if (row_scale >= 0x1p-100f && row_scale <= 0x1p96f) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] = v[i] * row_scale * scale[i];
            } else {
                const float out = row_scale > 1.0f ? 0x1p-64f : 0x1p64f, back = row_scale > 1.0f ? 0x1p64f : 0x1p-64f;
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] = v[i] * (row_scale * out) * scale[i] * back;
            }
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            v[i] += bias[i];
            if constexpr (!PLAIN) v[i] = act_f(v[i], a.act);
        }
        if constexpr (!PLAIN) store_row<W>(a, yr, c0, v);
        else if constexpr (YT == F32) __builtin_memcpy(reinterpret_cast<float *>(a.y + (long)yr * a.ldy) + c0, v, 4 * W);
        else {
            static_assert(W == 8, "");
            store16(a.y + (long)yr * a.ldy + 2 * c0, u32x4{pack2(v[0], v[1], YT), pack2(v[2], v[3], YT), pack2(v[4], v[5], YT), pack2(v[6], v[7], YT)});
        }
    }
};

// the x row and the y row of order position r (-1: no such row)
__device__ __forceinline__ int x_row_of(const LinearArgs &a, int r) {
    const int v = a.x_rows ? a.x_rows[r] : r;
    return (unsigned)v < (unsigned)a.x_total ? v : -1;
}
__device__ __forceinline__ int y_row_of(const LinearArgs &a, int r) {
    const int v = a.y_rows ? a.y_rows[r] : r;
    return (unsigned)v < (unsigned)a.y_total ? v : -1;
}

// the tile's rows of x and y, and the scales of its x rows
template <int T, int BM, int NTHR>
__device__ __forceinline__ void rows_to_lds(const LinearArgs &a, const Tile &t, int tid, int *xrows, int *yrows, float *scales) {
    for (int i = tid; i < BM; i += NTHR) {
        const int r = t.r0 + i;
        int xr = -1, yr = -1;
        if (r < t.r1) {
            xr = x_row_of(a, r);
            yr = xr < 0 ? -1 : y_row_of(a, r);
        }
        xrows[i] = xr;
        yrows[i] = yr;
        if constexpr (T == I8) scales[i] = xr < 0 ? 0.0f : a.x_scale[xr];
    }
}

// A wave's sums -> y, 32 rows x WN channels at a time: image(img, i) puts the sums of rows 32 i .. + 32 into LDS as the matrix
// instruction left them (4 consecutive channels per lane), and they come back as 8 consecutive channels per lane, whole rows by
// consecutive lanes.  s_mem: 32 (WN + 4) sums for each wave.
template <int T, int R, int WN, bool PLAIN, int YT, class Image>
__device__ __forceinline__ void store_rows(const LinearArgs &a, const Chan<T, 8> &ch, Image &&image, uint8_t *s_mem, const int *yrows, const float *scales,
                                           int wave, int lane, int c0, int valid) {
    typedef typename Acc<T>::e E;
    typedef typename Acc<T>::q4 Q;
    constexpr int PITCH = WN + 4;
    E *img = reinterpret_cast<E *>(s_mem) + wave * 32 * PITCH;
    constexpr int LPR = WN / 8, RPI = 64 / LPR;  // lanes per row, rows per instruction
    const int c8 = (lane % LPR) * 8;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i * 32 >= valid) break;
        image(img, i);
        __builtin_amdgcn_wave_barrier();  // one wave's LDS accesses are in order
#pragma unroll
        for (int r = 0; r < 32; r += RPI) {
            const int at = r + lane / LPR, yr = yrows[i * 32 + at];
            const Q lo = *reinterpret_cast<const Q *>(img + at * PITCH + c8), up = *reinterpret_cast<const Q *>(img + at * PITCH + c8 + 4);
            const E s[8] = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
            if (yr >= 0) ch.template finish<PLAIN, YT>(a, s, T == I8 ? scales[i * 32 + at] : 1.0f, yr, c0);
        }
        __builtin_amdgcn_wave_barrier();
    }
}
template <int T, int R, int WN, class Image>
__device__ __forceinline__ void store_tile(const LinearArgs &a, const Chan<T, 8> &ch, Image &&image, uint8_t *s_mem, const int *yrows, const float *scales,
                                           int wave, int lane, int c_wave, int valid) {
    const int c0 = c_wave + (lane % (WN / 8)) * 8;
    const bool plain = a.act == PB_ACT_NONE && c_wave + WN <= a.n;  // of the whole wave
    if (plain && a.y_type == BF16) store_rows<T, R, WN, true, BF16>(a, ch, image, s_mem, yrows, scales, wave, lane, c0, valid);
    else if (plain && a.y_type == F16) store_rows<T, R, WN, true, F16>(a, ch, image, s_mem, yrows, scales, wave, lane, c0, valid);
    else if (plain) store_rows<T, R, WN, true, F32>(a, ch, image, s_mem, yrows, scales, wave, lane, c0, valid);
    else store_rows<T, R, WN, false, F32>(a, ch, image, s_mem, yrows, scales, wave, lane, c0, valid);
}

// What the tile kernels share: K goes in steps of 128 bytes through NST LDS stages.  A row sits in LDS at a pitch of 128 bytes with its
// eight 16-byte pieces permuted, so that the fragment reads -- 16 bytes from each of 32 (or of 16 x 4) places -- are free of bank
// conflicts: with 32-row fragments piece c at c ^ (row / 2 & 7): 242 bytes a clock and CU, against 123 with c ^ (row & 7) and 32
// unpermuted; with 16-row fragments c ^ (row & 7): 232, unpermuted 63 (LDS reads alone, 256 workgroups of eight waves).  The permutation is done by
// the lanes' GLOBAL addresses, so a wave's eight rows of 128 bytes are still whole lines.  DMA: the
// loads go straight into LDS (16-byte aligned rows); otherwise through registers, which takes any alignment.  The last, partial step always goes through registers.
template <int T, int BM, int BN, int NTHR, int NST, bool ROWS16>
struct Loader {
    static constexpr int TAIL = BM > 128 ? 2 : 4;
    static constexpr int STAGE = (BM + BN) * 128, JA = BM * 8 / NTHR, J = (BM + BN) * 8 / NTHR;  // 16-byte pieces per thread and step: of x, in all
    static_assert(BM * 8 % NTHR == 0 && BN * 8 % NTHR == 0 && NTHR / 8 % 16 == 0 && (NST == 2 || NST == 4), "");
    const uint8_t *pp[J];  // this thread's rows: JA of x, the others of w
    uint8_t *mem;
    int tid, wave, lc, kb, full, steps;

    __device__ __forceinline__ Loader(const LinearArgs &a, const Tile &t, uint8_t *s_mem, const int *xrows, int tid_, int wave_) {
        mem = s_mem;
        tid = tid_;
        wave = wave_;
        kb = a.kb;
        full = kb >> 7;
        steps = (kb + 127) >> 7;
        lc = ((tid & 7) ^ ((tid >> (ROWS16 ? 3 : 4)) & 7)) * 16;  // the piece this thread moves in every row it touches
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int row = (tid + j * NTHR) >> 3;
            pp[j] = (j < JA ? a.x + (long)max(xrows[j < JA ? row : 0], 0) * a.ldx : a.w + ((long)t.g * a.n + min(t.nt * BN + row - BM, a.n - 1)) * a.ldw) + lc;
        }
    }
    __device__ __forceinline__ uint8_t *stage(int i) const { return mem + (i & (NST - 1)) * STAGE; }
    __device__ __forceinline__ void dma(int i, int j) const {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(pp[j] + (long)i * 128),
                                         (__attribute__((address_space(3))) void *)(stage(i) + wave * 1024 + j * NTHR * 16), 16, 0, 0);
    }
    __device__ __forceinline__ void load(int i, u32x4 (&to)[J]) const {
#pragma unroll
        for (int j = 0; j < J; ++j) to[j] = load16<true>(pp[j] + (long)i * 128);
    }
    __device__ __forceinline__ void put(int i, const u32x4 (&from)[J]) const {
#pragma unroll
        for (int j = 0; j < J; ++j) *reinterpret_cast<u32x4 *>(stage(i) + (tid + j * NTHR) * 16) = from[j];
    }
    __device__ __forceinline__ void tail(int i) const {  // the partial step behind the full ones
#pragma unroll
        for (int j0 = 0; j0 < J; j0 += TAIL) {  // a few loads on their way at a time
            u32x4 v[TAIL];
#pragma unroll
            for (int j = 0; j < TAIL && j0 + j < J; ++j) v[j] = load16_tail<true>(pp[j0 + j] - lc, i * 128 + lc, kb);
#pragma unroll
            for (int j = 0; j < TAIL && j0 + j < J; ++j) *reinterpret_cast<u32x4 *>(stage(i) + (tid + (j0 + j) * NTHR) * 16) = v[j];
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // steps [0, n) before the walk
    __device__ __forceinline__ void first(int n, bool by_dma) const {
        for (int i = 0; i < n; ++i) {
            if (i < full) {
                if (by_dma) {
#pragma unroll
                    for (int j = 0; j < J; ++j) dma(i, j);
                } else {
                    u32x4 r[J];
                    load(i, r);
                    put(i, r);
                }
            } else if (i < steps) tail(i);
        }
    }
    // this wave's loads of step i are in LDS; those of younger steps, at most NST - 2 of them, may still be on their way
    __device__ __forceinline__ void landed(int i) const {
        const int younger = min(NST - 2, full - 1 - i);
        if (NST > 3 && younger >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * J) : "memory");
        else if (NST > 2 && younger == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(J) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    static __device__ __forceinline__ void barrier() {  // this wave's LDS reads have come back, its LDS writes are done
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
};

// ---- k_linear_tile: small tiles -- 64 x 64 or 128 x 128, waves of 32 x 32 or 64 x 32 ---------------------------------------------------------
// For products with few tiles, where a step is short: a wave has one or two 32 x 32 matrix instructions to a 32-byte piece, and would
// wait out an LDS read for each piece, so it reads a step's four pieces at once behind the step's one barrier; four LDS stages give
// the loads three steps to arrive.  777 x 1003 x 1289 i8 12.5 us (rows of 1296 bytes 9.2), 1024 x 1024 x 1008 7.4.  (By these tiles with 4
// pieces one after the other 64 x 4096 x 4096 13.3 us instead of 12.8; two stages: weights out of HBM, 128 x 8192 x 8192, 33.7 us instead
// of 22.0.)
template <int T, int BM, int BN, int WM, int WN, int NST, bool DMA>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void k_linear_tile(const LinearArgs a) {
    constexpr int NWM = BM / WM, NWN = BN / WN, NTHR = 64 * NWM * NWN, MT = WM / 32, NT = WN / 32;
    constexpr int EPI = NWM * NWN * 32 * (WN + 4) * 4;
    typedef Loader<T, BM, BN, NTHR, NST, false> L;
    constexpr int J = L::J;
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[(NST * L::STAGE > EPI ? NST * L::STAGE : EPI)];
    __shared__ int s_xrow[BM], s_yrow[BM];
    __shared__ float s_scale[T == I8 ? BM : 1];
    const Tile t = find_tile<BM, 4>(a);
    if (t.r0 >= t.r1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    rows_to_lds<T, BM, NTHR>(a, t, tid, s_xrow, s_yrow, s_scale);
    __syncthreads();
    const L l(a, t, s_mem, s_xrow, tid, wave);
    const int wm = wave / NWN * WM, wn = wave % NWN * WN, li = lane & 31, hi = lane >> 5, c_wave = t.nt * BN + wn;
    Chan<T, 8> ch;  // on their way under the product
    ch.load(a, t.g, c_wave + (lane % (WN / 8)) * 8);
    typename Acc<T>::q16 acc[NT][MT] = {};
    const uint8_t *sa = s_mem + (wm + li) * 128, *sb = s_mem + (BM + wn + li) * 128;
    // MV: the 32-row pieces of this wave that hold rows -- a group's last tile is seldom full, and matrix instructions on nothing
    // would cost as much as others
    auto product = [&](auto MV, int i) {
        u32x4 fa[4][MT], fb[4][NT];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int c = (i & (NST - 1)) * L::STAGE + ((ks * 2 + hi) ^ ((li >> 1) & 7)) * 16;
            if constexpr (MV.value > 0) {
#pragma unroll
                for (int j = 0; j < NT; ++j) fb[ks][j] = *reinterpret_cast<const u32x4 *>(sb + j * 4096 + c);
            }
#pragma unroll
            for (int m = 0; m < MV.value; ++m) fa[ks][m] = *reinterpret_cast<const u32x4 *>(sa + m * 4096 + c);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int m = 0; m < MV.value; ++m) mma32<T>(acc[j][m], fb[ks][j], fa[ks][m]);
        __builtin_amdgcn_sched_barrier(0);
    };
    l.first(DMA ? NST : 1, DMA);
    auto walk = [&](auto MV) {
        if constexpr (DMA) {
            for (int i = 0; i < l.steps; ++i) {
                l.landed(i);
                L::barrier();  // step i is in LDS, everyone has read step i - 1
                const int next = i - 1 + NST;
                if (i > 0 && next < l.full) {
#pragma unroll
                    for (int j = 0; j < J; ++j) l.dma(next, j);
                } else if (i > 0 && next == l.full && l.full < l.steps) l.tail(l.full);
                product(MV, i);
            }
        } else {
            // step i + 2's registers are loaded while step i is multiplied, step i + 1's go to LDS behind it
            u32x4 even[J], odd[J];
            if (1 < l.full) l.load(1, even);
            auto half = [&](int i, const u32x4 (&now)[J], u32x4 (&later)[J]) {
                L::barrier();  // step i is in LDS, everyone has read step i - 1
                if (i + 2 < l.full) l.load(i + 2, later);
                product(MV, i);
                if (i + 1 < l.full) l.put(i + 1, now);
                else if (i + 1 == l.full && l.full < l.steps) l.tail(l.full);
            };
            for (int i = 0; i < l.steps; i += 2) {
                half(i, even, odd);
                if (i + 1 < l.steps) half(i + 1, odd, even);
            }
        }
    };
    const int valid = t.r1 - t.r0 - wm;  // rows of this wave's part
    if (valid <= 0) walk(std::integral_constant<int, 0>{});
    else if (MT > 1 && valid <= WM / 2) walk(std::integral_constant<int, (MT > 1 ? MT / 2 : MT)>{});
    else walk(std::integral_constant<int, MT>{});
    __syncthreads();  // the stages become the waves' epilogue images
    // 32 x 32 sums: lane l has row l % 32, channels 8 q + 4 (l / 32) + 0 .. 3
    auto image = [&](auto *img, int i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<typename Acc<T>::q4 *>(img + li * (WN + 4) + j * 32 + q * 8 + hi * 4) =
                    typename Acc<T>::q4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
    };
    store_tile<T, MT, WN>(a, ch, image, s_mem, s_yrow + wm, s_scale + (T == I8 ? wm : 0), wave, lane, c_wave, valid);
}

// ---- k_linear_wide: large tiles -- 256 x 256 with waves of 128 x 64, 128 x 128 with waves of 64 x 64 -------------------------------------------
// For products that fill the chip with such tiles.  16 x 16 matrix instructions: they read and write their sums half as often per
// multiplication as the 32 x 32 ones, and run faster (bare, without loads: i8 4.09 against 3.38 P/s).  On the same data 8192^3 took i8 423 us
// instead of 475, f16 794 instead of 892, bf16 745 instead of 846; on evenly spread codes 439, on normally
// distributed values 825 and 792.  The matrix units
// are busy 59 % of the cycles (i8; f16 over 32 experts 42 %) at 2.0 GHz (the bare loop: all of them at 1.95); on zeros i8 takes 393 us
// and f16 662.
// A step is 2 MT slots, one 16-row fragment of x each (MT pieces of the first 64 bytes, then of the second) against the wave's NT
// channel fragments.  Fragments of x are read PF slots ahead into a ring of PF + 1, the channels' a half step ahead.  The one
// barrier of a step stands PF slots before its end, where all that is left of the step is in registers: behind it the step's stage is
// free, so the loads of step i + NST leave there, among the matrix instructions, and have NST - 1 steps to arrive, and the first
// fragments of step i + 1 are read -- the matrix pipe has work across the barrier.  A partial step comes behind them, by itself.
template <int T, int BM, int BN, int WM, int WN, int NST, int PF, bool DMA>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void k_linear_wide(const LinearArgs a) {
    constexpr int NWM = BM / WM, NWN = BN / WN, NTHR = 64 * NWM * NWN, MT = WM / 16, NT = WN / 16, SLOTS = 2 * MT, X = SLOTS - PF;
    constexpr int EPI = NWM * NWN * 32 * (WN + 4) * 4;
    typedef Loader<T, BM, BN, NTHR, NST, true> L;
    constexpr int J = L::J;
    static_assert(SLOTS % (PF + 1) == 0 && X >= MT && NT <= MT && PF >= 1, "");
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[(NST * L::STAGE > EPI ? NST * L::STAGE : EPI)];
    __shared__ int s_xrow[BM], s_yrow[BM];
    __shared__ float s_scale[T == I8 ? BM : 1];
    const Tile t = find_tile<BM, 4>(a);
    if (t.r0 >= t.r1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    rows_to_lds<T, BM, NTHR>(a, t, tid, s_xrow, s_yrow, s_scale);
    __syncthreads();
    const L l(a, t, s_mem, s_xrow, tid, wave);
    const int wm = wave / NWN * WM, wn = wave % NWN * WN, li = lane & 15, q = lane >> 4, c_wave = t.nt * BN + wn;
    typename Acc<T>::q4 acc[NT][MT] = {};
    const uint8_t *sa = s_mem + (wm + li) * 128, *sb = s_mem + (BM + wn + li) * 128;
    const int piece[2] = {(q ^ (li & 7)) * 16, ((4 + q) ^ (li & 7)) * 16};
    u32x4 fa[PF + 1], fb[2][NT];
    auto read_x = [&](int i, int f) { fa[f % (PF + 1)] = *reinterpret_cast<const u32x4 *>(sa + (i & (NST - 1)) * L::STAGE + (f % MT) * 2048 + piece[f / MT]); };
    auto read_w = [&](int i, int half, int j) { fb[half][j] = *reinterpret_cast<const u32x4 *>(sb + (i & (NST - 1)) * L::STAGE + j * 2048 + piece[half]); };
    const int valid = t.r1 - t.r0 - wm;           // rows of this wave's part, and the 16-row fragments that hold some: a group's last
    const int pieces = (max(valid, 0) + 15) / 16;  // tile is seldom full, and matrix instructions on nothing would cost as much as others
    u32x4 regs[DMA ? 1 : J];
    l.first(min(NST, l.full), DMA);
    l.landed(0);
    L::barrier();
    if (l.full > 0) {
#pragma unroll
        for (int j = 0; j < NT; ++j) read_w(0, 0, j);
#pragma unroll
        for (int f = 0; f < PF; ++f) read_x(0, f);
    }
    auto walk = [&](auto ALL) {
        for (int i = 0; i < l.full; ++i) {
#pragma unroll
            for (int f = 0; f < SLOTS; ++f) {
                if (f + PF < SLOTS) read_x(i, f + PF);
                if (f < NT) read_w(i, 1, f);
                if (f == X) {
                    if constexpr (!DMA) {
                        if (i > 0 && i - 1 + NST < l.full) l.put(i - 1 + NST, regs);
                    }
                    l.landed(i + 1);
                    L::barrier();  // the rest of step i is in registers everywhere, step i + 1 is in LDS
                    if constexpr (!DMA) {
                        if (i + NST < l.full) l.load(i + NST, regs);
                    }
                    if (i + 1 < l.full) {
#pragma unroll
                        for (int j = 0; j < NT; ++j) read_w(i + 1, 0, j);
                    }
                }
                if (f >= X && i + 1 < l.full) read_x(i + 1, f - X);
                if (ALL.value || f % MT < pieces) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) mma16<T>(acc[j][f % MT], fb[f / MT][j], fa[f % (PF + 1)]);
                }
                if constexpr (DMA) {
                    constexpr int PER = (J + PF - 1) / PF;
                    if (f >= X && i + NST < l.full) {
#pragma unroll
                        for (int j = (f - X) * PER; j < (f - X + 1) * PER && j < J; ++j) l.dma(i + NST, j);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    if (pieces >= MT) walk(std::true_type{});  // a branch at every slot costs 7 %
    else walk(std::false_type{});
    if (l.full < l.steps) {  // the partial step, by itself
        L::barrier();
        l.tail(l.full);
        L::barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NT; ++j) read_w(l.full, h, j);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                read_x(l.full, h * MT + m);
#pragma unroll
                for (int j = 0; j < NT; ++j) mma16<T>(acc[j][m], fb[h][j], fa[(h * MT + m) % (PF + 1)]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    Chan<T, 8> ch;
    ch.load(a, t.g, c_wave + (lane % (WN / 8)) * 8);
    __syncthreads();  // the stages become the waves' epilogue images
    // 16 x 16 sums: lane l has row l % 16, channels 4 (l / 16) + 0 .. 3
    auto image = [&](auto *img, int i) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j) *reinterpret_cast<typename Acc<T>::q4 *>(img + (h * 16 + li) * (WN + 4) + j * 16 + q * 4) = acc[j][2 * i + h];
    };
    store_tile<T, WM / 32, WN>(a, ch, image, s_mem, s_yrow + wm, s_scale + (T == I8 ? wm : 0), wave, lane, c_wave, valid);
}

// ---- k_linear_few: 16 MT rows x 16 NT channels per workgroup, K split over its NW waves ----------------------------------------------------
// For few rows (or little work): the weights are read once, straight into registers, 64 U bytes of a row per wave and turn; the
// waves' partial sums meet in LDS and are added in wave order, so that a sum's order goes with k and U alone.  Bound by the weights out of
// HBM: 32 rows over 64 groups, 2048 x 2048 bf16 (210 MB of 25 groups in use) 42 us, 5.0 TB/s (a plain read 5.76, a copy 5.48); with weights in the
// caches by the way from a load to the last sum (16 x 4096 x 4096 i8 6.4 us, 1 x 256 x 1280 3.1 of which 1.5 are any launch's).  Loads a
// turn ahead would cost registers and with them waves: 40 us instead of 32 (evenly filled groups).
template <int T, int MT, int NT, int NW, int U, bool DW>
__global__ __launch_bounds__(64 * NW) void k_linear_few(const LinearArgs a) {
    typedef typename Acc<T>::e E;
    typedef typename Acc<T>::q4 Q;
    constexpr int BM = 16 * MT, BN = 16 * NT;
    constexpr int PITCH = BN + 4;
    __shared__ __attribute__((aligned(16))) E s_sum[NW][BM * PITCH];
    __shared__ float s_xscale[BM], s_wscale[BN], s_bias[BN];
    __shared__ int s_xrow[BM], s_yrow[BM];
    const Tile t = find_tile<BM, 1>(a);
    if (t.r0 >= t.r1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, kq = (lane >> 4) * 16;
    const int c_base = t.nt * BN;
    const uint8_t *px[MT], *pw[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) px[i] = a.x + (long)max(x_row_of(a, min(t.r0 + i * 16 + li, t.r1 - 1)), 0) * a.ldx + kq;
#pragma unroll
    for (int j = 0; j < NT; ++j) pw[j] = a.w + ((long)t.g * a.n + min(c_base + j * 16 + li, a.n - 1)) * a.ldw + kq;
    // what the end needs is on its way to LDS ahead of the operands: behind the sums it would cost two more trips to memory (512 rows
    // over 8 groups, 256 x 1280 f32: 18.3 us instead of 17.4 with its group_rows)
    auto to_lds = [](const float *from, float *to) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 4, 0, 0);
    };
    if (wave == NW - 1 && lane < BM) {
        const bool in = t.r0 + lane < t.r1;
        const int xr = in ? x_row_of(a, t.r0 + lane) : -1, yr = in ? y_row_of(a, t.r0 + lane) : -1;
        s_xrow[lane] = xr;
        s_yrow[lane] = yr;
        if constexpr (T == I8) to_lds(a.x_scale + max(xr, 0), s_xscale);
    } else if (wave == NW - 2 && lane < BN) {
        const long c = (long)t.g * a.n + min(c_base + lane, a.n - 1);
        if constexpr (T == I8) to_lds(a.w_scale + c, s_wscale);
        if (a.bias) to_lds(a.bias + c, s_bias);
    }
    Q acc[NT][MT] = {};
    const int kb1 = a.kb;
    for (int kb = wave * 64 * U; kb < kb1; kb += 64 * U * NW) {
        u32x4 fw[U][NT], fx[U][MT];
        if (kb + 64 * U <= kb1) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < NT; ++j) fw[u][j] = load16<DW>(pw[j] + kb + u * 64);
#pragma unroll
                for (int i = 0; i < MT; ++i) fx[u][i] = load16<DW>(px[i] + kb + u * 64);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = kb + u * 64;
                if (at + 64 <= kb1) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) fw[u][j] = load16<DW>(pw[j] + at);
#pragma unroll
                    for (int i = 0; i < MT; ++i) fx[u][i] = load16<DW>(px[i] + at);
                } else if (at < kb1) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) fw[u][j] = load16_tail<DW>(pw[j] - kq, at + kq, kb1);
#pragma unroll
                    for (int i = 0; i < MT; ++i) fx[u][i] = load16_tail<DW>(px[i] - kq, at + kq, kb1);
                } else {
#pragma unroll
                    for (int j = 0; j < NT; ++j) fw[u][j] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < MT; ++i) fx[u][i] = u32x4{0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) mma16<T>(acc[j][i], fw[u][j], fx[u][i]);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<Q *>(&s_sum[wave][(i * 16 + li) * PITCH + j * 16 + (lane >> 4) * 4]) = acc[j][i];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the loads into LDS
    __syncthreads();
    for (int q = tid; q < BM * BN / 4; q += 64 * NW) {
        const int r = q / (BN / 4), c = (q % (BN / 4)) * 4;
        const int yr = s_yrow[r];
        if (s_xrow[r] < 0 || yr < 0) continue;
        Q s = *reinterpret_cast<const Q *>(&s_sum[0][r * PITCH + c]);
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const Q o = *reinterpret_cast<const Q *>(&s_sum[w][r * PITCH + c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += o[i];
        }
        Chan<T, 4> ch;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ch.scale[i] = T == I8 ? s_wscale[c + i] : 1.0f;
            ch.bias[i] = a.bias ? s_bias[c + i] : 0.0f;
        }
        const E e[4] = {s[0], s[1], s[2], s[3]};
        ch.finish(a, e, T == I8 ? s_xscale[r] : 1.0f, yr, c_base + c);
    }
}

// ---- k_quantize_rows ------------------------------------------------------------------------------------------------------------------------
// scale = max(max |x| / 127, 2^-126); code = x / scale to the nearest whole number, halves to the even one.  Without a division per
// value, and exactly: x * (1 / scale) + 1.5 * 2^23, one fused multiply-add, is the whole number in the low bits (1 / scale is off by
// half a unit in the last place, the quotient by less than 7.7e-6).  Only where it lies within 1e-5 of a half -- one value in 50 000 -- the
// remainder x - r * scale decides, which a fused multiply-add gives exactly near scale / 2.  Bound by HBM: 8192 x 1280 f32 (52 MB) 10.0
// us, 5.2 TB/s (a copy 5.5); 8192 x 8192 bf16 41.2.  A row with an infinity or a NaN gets
// scale = NaN and codes 0, so that what is computed from it shows.
constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23
__device__ __forceinline__ uint32_t code_exact(float x, float inv, float scale, float half) {
    float r = rintf(x * inv);  // off by one at most
    const float d = __builtin_fmaf(-r, scale, x), ad = fabsf(d);
    const bool odd = ((int)r & 1) != 0;
    if (ad > half || (ad == half && odd)) r += d > 0.0f ? 1.0f : -1.0f;
    return (uint32_t)(int)r;
}
// V codes, packed four to a word
template <int V>
__device__ __forceinline__ void codes_of(const float (&x)[V], float inv, float scale, float half, uint32_t (&word)[V / 4]) {
    uint32_t q[V];
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float r = __builtin_fmaf(x[i], inv, MAGIC);
        q[i] = __float_as_uint(r);
        far = fmaxf(far, fabsf(__builtin_fmaf(x[i], inv, MAGIC - r)));
    }
    if (far > 0.49999f) {
#pragma unroll 1
        for (int i = 0; i < V; ++i) {
            float v = x[0];
#pragma unroll
            for (int j = 1; j < V; ++j) v = i == j ? x[j] : v;
            const uint32_t c = code_exact(v, inv, scale, half);
#pragma unroll
            for (int j = 0; j < V; ++j) q[j] = i == j ? c : q[j];
        }
    }
#pragma unroll
    for (int w = 0; w < V / 4; ++w) {
        const uint32_t lo = __builtin_amdgcn_perm(q[4 * w + 1], q[4 * w], 0x0c0c0400u), up = __builtin_amdgcn_perm(q[4 * w + 3], q[4 * w + 2], 0x0c0c0400u);
        word[w] = lo | (up << 16);
    }
}

template <int T> __device__ __forceinline__ float elem(const uint8_t *row, long i) {
    if constexpr (T == F32) return reinterpret_cast<const float *>(row)[i];
    else if constexpr (T == BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(row)[i] << 16);
    else return (float)reinterpret_cast<const _Float16 *>(row)[i];
}

// NTHR threads per row (a wave or a workgroup of four), V values per thread and turn; rows of up to NTHR * V * TURNS values stay in
// registers between the maximum and the codes, longer ones are read a second time.
template <int T, int NTHR, int TURNS>
__global__ __launch_bounds__(256) void k_quantize_rows(const uint8_t *__restrict__ x, int m, int k, long ldx, int8_t *__restrict__ codes, long ldc,
                                                       float *__restrict__ scale) {
    constexpr int V = T == F32 ? 4 : 8, RPB = 256 / NTHR;
    __shared__ uint32_t s_max[4];
    const int tid = threadIdx.x % NTHR;
    const int row = blockIdx.x * RPB + (RPB > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    if (row >= m) return;
    const uint8_t *px = x + (long)row * ldx;
    int8_t *pc = codes + (long)row * ldc;
    const uint32_t INF = 0x7f800000u;
    auto load = [&](int c, float (&v)[V]) {
        if (c + V <= k) {
            const u32x4 q = load16<true>(px + (long)c * type_bytes(T));
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if constexpr (T == F32) v[i] = __uint_as_float(q[i]);
                else if constexpr (T == BF16) v[i] = __uint_as_float(i & 1 ? q[i >> 1] & 0xffff0000u : q[i >> 1] << 16);
                else v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(q[i >> 1] >> (16 * (i & 1))));
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = c + i < k ? elem<T>(px, c + i) : 0.0f;
        }
    };
    float v[TURNS][V];
    uint32_t top = 0;  // |x| as bits: the order of non-negative floats, infinities and NaN above all of them
#pragma unroll
    for (int t = 0; t < TURNS; ++t) load((t * NTHR + tid) * V, v[t]);
#pragma unroll
    for (int t = 0; t < TURNS; ++t)
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(v[t][i]) & 0x7fffffffu);
    for (int c = (TURNS * NTHR + tid) * V; c < k; c += NTHR * V) {
        float u[V];
        load(c, u);
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(u[i]) & 0x7fffffffu);
    }
    top = (uint32_t)__builtin_amdgcn_readlane((int)wave_max(top), 63);
    if constexpr (NTHR > 64) {
        if ((tid & 63) == 0) s_max[tid >> 6] = top;
        __syncthreads();
        top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    }
    const bool bad = top >= INF;
    const float sc = fmaxf(__uint_as_float(top) / 127.0f, 1.17549435e-38f);
    if (tid == 0) scale[row] = bad ? __uint_as_float(0x7fc00000u) : sc;
    const float inv = bad ? 0.0f : 1.0f / sc, half = 0.5f * sc;
    auto put = [&](int c, float (&u)[V]) {
        if (c >= k) return;
        if (bad) {
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] = 0.0f;
        }
        uint32_t w[V / 4];
        codes_of<V>(u, inv, sc, half, w);
        if (c + V <= k) __builtin_memcpy(pc + c, w, V);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < k) pc[c + i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
        }
    };
#pragma unroll
    for (int t = 0; t < TURNS; ++t) put((t * NTHR + tid) * V, v[t]);
    for (int c = (TURNS * NTHR + tid) * V; c < k; c += NTHR * V) {
        float u[V];
        load(c, u);
        put(c, u);
    }
}

// ---- k_group_rows ---------------------------------------------------------------------------------------------------------------------------
// Workgroup g < groups counts the rows of smaller groups (its offset) and lists its own rows in ascending order; workgroup `groups`
// lists the rows without a group behind all others.  Every workgroup reads the whole array instead of meeting the others: no scratch
// memory, no atomics, one launch, one possible result.  The work is rows x (groups + 1): up to a million rows the array sits in each XCD's
// L2 (4 MB), beyond that it comes from the cache behind them, and lists of more than one LDS map are read twice (131073 rows of 256 groups
// 28 us, a million of 64 108, of 1024 417, 30 million of 1024 20 ms).  A first walk, four consecutive rows per lane, turns each
// comparison into a lane mask: the counts come from the scalar unit's bit counts, the masks of matching rows go to LDS -- four
// vector instructions for 64 rows, which is what bounds it (131072 rows, 256 groups: 27 us with a bit per lane put together by vector
// instructions).  Then every lane takes words of 32 rows, learns by prefix sums over the bit counts where its rows go, and lists
// them in LDS, from where the wave writes whole lines: rows written straight from the lanes that found them go to lines apart (131072
// rows of one group: 74 us).  Where half of a wave's 2048 rows and more are the group's, 64 rows' worth are written at once instead
// (one group 21 us, 8 groups 13, 256 groups 15; 256 groups of uneven sizes and a tenth of the rows without one 17.8: the workgroup with
// the most rows is the last).  Rows beyond one LDS map's 8192 per wave are walked a second time, map by map.
// As unsigned numbers, rows of no group are >= groups: a row is before group g if it is < g.
// v with the wave-uniform `value` in one lane: v_writelane_b32 as the compiler's intrinsic, which has no builtin of its own (as inline
// asm the compiler leaves out the two wait states between the comparison that writes the scalar register and this read of it)
extern "C" __device__ __attribute__((const)) int pb_writelane(int value, int lane, int v) __asm("llvm.amdgcn.writelane.i32");

template <int WAVES>
__global__ __launch_bounds__(64 * WAVES, 8) void k_group_rows(const int32_t *__restrict__ group, int m, int groups, int vec, int32_t *__restrict__ offsets,
                                                              int32_t *__restrict__ order) {
    constexpr int NTHR = 64 * WAVES, CHUNK = WAVES * 8192, STAGE = 1024;
    __shared__ uint32_t s_mask[CHUNK / 32];  // per 256 rows eight words: rows 4 l + i of lane l at bit l of pair i
    __shared__ uint16_t s_rows[WAVES][STAGE];
    __shared__ int s_lt[WAVES], s_eq[WAVES];
    const unsigned g = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunks = (int)(((long)m + CHUNK - 1) / CHUNK);  // m = 0: none
    int lt = 0;  // rows before this group, of this wave's 256s
    auto walk = [&](auto LAST, int c) {  // a wave takes every WAVES-th 256 rows
        const int32_t *p = group + (long)c * CHUNK;
        const int n = (int)min((long)CHUNK, (long)m - (long)c * CHUNK);
        int turn = wave;
        if (vec) {
            for (; (turn + 7 * WAVES + 1) * 256 <= n; turn += 8 * WAVES) {
                i32x4 q[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = *reinterpret_cast<const i32x4 *>(p + (turn + j * WAVES) * 256 + lane * 4);
                int words = 0;  // lane 8 j + 2 i + h: half h of turn j's mask i
#pragma unroll
                for (int j = 0; j < 8; ++j) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint64_t less = __ballot((unsigned)q[j][i] < g);
                        const uint64_t own = LAST.value ? ~less : __ballot((unsigned)q[j][i] == g);
                        lt += __builtin_popcountll(less);
                        words = pb_writelane((int)(uint32_t)own, 8 * j + 2 * i, words);
                        words = pb_writelane((int)(uint32_t)(own >> 32), 8 * j + 2 * i + 1, words);
                    }
                    __builtin_amdgcn_sched_barrier(0);  // all 64 masks at once would not fit the scalar registers
                }
                s_mask[(turn + (lane >> 3) * WAVES) * 8 + (lane & 7)] = (uint32_t)words;
            }
        }
#pragma unroll 1
        for (; turn * 256 < n; turn += WAVES) {
            const int at = turn * 256 + lane * 4;
            i32x4 q = {-1, -1, -1, -1};
            if (vec && at + 4 <= n) q = *reinterpret_cast<const i32x4 *>(p + at);
            else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + i < n) q[i] = p[at + i];
            }
            int words = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t less = __ballot((unsigned)q[i] < g);
                const uint64_t own = LAST.value ? ~less & __ballot(at + i < n) : __ballot((unsigned)q[i] == g);
                lt += __builtin_popcountll(less);
                words = pb_writelane((int)(uint32_t)own, 2 * i, words);
                words = pb_writelane((int)(uint32_t)(own >> 32), 2 * i + 1, words);
            }
            if (lane < 8) s_mask[turn * 8 + lane] = (uint32_t)words;
        }
        return n;
    };
    auto run = [&](auto LAST) {
        int n = 0;
        for (int c = 0; c < chunks; ++c) n = walk(LAST, c);
        if (lane == 0) s_lt[wave] = lt;
        __syncthreads();
        int first = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) first += s_lt[w];
        if (tid == 0) offsets[g] = first;  // workgroup `groups`: the number of rows that have a group
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) {
                __syncthreads();  // the words and counts before these have been read
                n = walk(LAST, c);
                __syncthreads();
            }
            const int words = (n + 31) >> 5, each = words <= NTHR ? 1 : words <= 2 * NTHR ? 2 : 4;  // for a thread
            auto word = [&](int w) {  // lanes 8 (w % 8) .. + 8 of turn w / 8, a bit of each of the four masks in turn
                const uint32_t *mask = s_mask + (w >> 3) * 8 + ((w >> 2) & 1);
                uint32_t bits = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t x = (mask[2 * k] >> (8 * (w & 3))) & 255u;
                    x = (x | x << 12) & 0x000f000fu;
                    x = (x | x << 6) & 0x03030303u;
                    x = (x | x << 3) & 0x11111111u;
                    bits |= x << k;
                }
                return bits;
            };
            const int w0 = wave * 64 * each;  // the wave's words: 64 at a time, one a lane
            uint32_t b[4];
            int inc[4], in_wave = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int w = w0 + i * 64 + lane;
                b[i] = i < each && w < words ? word(w) : 0u;
                inc[i] = wave_prefix(__builtin_popcount(b[i]));
                in_wave += __builtin_amdgcn_readlane(inc[i], 63);
            }
            if (lane == 63) s_eq[wave] = in_wave;
            __syncthreads();
            int to = first, all = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                if (w < wave) to += s_eq[w];
                all += s_eq[w];
            }
            first += all;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= each) break;
                const int n_in = __builtin_amdgcn_readlane(inc[i], 63);
                int row = c * CHUNK + (w0 + i * 64) * 32;
                if (n_in <= STAGE) {  // every lane lists its own rows, and the wave writes them
                    int at = inc[i] - __builtin_popcount(b[i]);
                    for (uint32_t left = b[i]; left; left &= left - 1) s_rows[wave][at++] = (uint16_t)(lane * 32 + __builtin_ctz(left));
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // LDS keeps a wave's order
                    for (int j = lane; j < n_in; j += 64) order[to + j] = row + s_rows[wave][j];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    to += n_in;
                } else {  // 64 rows at a time, a lane each
                    row += lane;
#pragma unroll 4
                    for (int l = 0; l < 64; l += 2) {
                        const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)b[i], l), high = (uint32_t)__builtin_amdgcn_readlane((int)b[i], l + 1);
                        const uint64_t in = (uint64_t)high << 32 | low;
                        const int at = to + __builtin_amdgcn_mbcnt_hi(high, __builtin_amdgcn_mbcnt_lo(low, 0u));
                        if (__builtin_amdgcn_inverse_ballot_w64(in)) order[at] = row;
                        to += __builtin_popcountll(in);
                        row += 64;
                    }
                }
            }
        }
    };
    if (g == (unsigned)groups) run(std::true_type{});
    else run(std::false_type{});
}

}  // namespace pbl
