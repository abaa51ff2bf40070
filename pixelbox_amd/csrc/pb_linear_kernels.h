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

// ---- loads ------------------------------------------------------------------------------------------------------------------------
template <bool ALIGNED>
__device__ __forceinline__ u32x4 load16(const uint8_t *p) {
    u32x4 v;
    if constexpr (ALIGNED) v = *reinterpret_cast<const u32x4 *>(p);
    else __builtin_memcpy(&v, p, 16);  // global_load_dwordx4 takes any address
    return v;
}
// bytes [at, at + 16) of a row of `len` bytes, zero behind its end; reads nothing outside [0, len)
template <bool ALIGNED>
__device__ __forceinline__ u32x4 load16_tail(const uint8_t *row, long at, long len) {
    if (at + 16 <= len) return load16<ALIGNED>(row + at);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (at >= len) return v;
    if (len >= 16) {  // the row's last 16 bytes, shifted down
        const u32x4 t = load16<false>(row + len - 16);
        const int s = 8 * (int)(at + 16 - len);  // 8 .. 120 bits
        const uint64_t lo = ((uint64_t)t.y << 32) | t.x, hi = ((uint64_t)t.w << 32) | t.z;
        const uint64_t l2 = s >= 64 ? hi >> (s - 64) : (lo >> s) | (hi << (64 - s));
        const uint64_t h2 = s >= 64 ? 0 : hi >> s;
        v = {(uint32_t)l2, (uint32_t)(l2 >> 32), (uint32_t)h2, (uint32_t)(h2 >> 32)};
        return v;
    }
    uint64_t half[2] = {0, 0};  // rows shorter than one piece
#pragma unroll 1
    for (int i = 0; at + i < len; ++i) {
        const uint64_t b = (uint64_t)row[at + i] << (8 * (i & 7));
        half[0] |= i < 8 ? b : 0;
        half[1] |= i < 8 ? 0 : b;
    }
    v = {(uint32_t)half[0], (uint32_t)(half[0] >> 32), (uint32_t)half[1], (uint32_t)(half[1] >> 32)};
    return v;
}

// ---- arguments of a product -----------------------------------------------------------------------------------------------------------
struct LinearArgs {
    const uint8_t *x, *w;
    const float *x_scale, *w_scale, *bias;
    const int32_t *offsets, *x_rows, *y_rows;
    uint8_t *y;
    long ldx, ldw, ldy;      // bytes between rows
    long kb;                 // bytes summed over
    int m, n, groups, n_tiles;
    int x_total, y_total;    // rows of x and y: an index outside them is no row
    int act, y_type;
    int y_vec;               // rows of y start on 16 bytes
};

// ---- which rows a workgroup works on ----------------------------------------------------------------------------------------------------
// Groups are cut into tiles of BM rows; tile numbers run over the groups in order.  Every wave finds its tile by itself: lanes
// look at 64 groups at a time and add up their tile counts.  Offsets are data of the device: they are clamped to [0, m], a group
// that runs backwards is empty, so that nothing outside the buffers is touched whatever they hold.
struct Tile {
    int g, r0, r1;  // rows [r0, r1) of the order; r0 >= r1: nothing to do
    int nt;         // tile of output channels
};

template <int BM, int BAND>
__device__ __forceinline__ Tile find_tile(const LinearArgs &a) {
    const int lane = threadIdx.x & 63;
    auto rows_of = [&](int g, int &lo, int &hi) {
        lo = 0;
        hi = a.m;
        if (a.offsets) {
            lo = min(max(a.offsets[g], 0), a.m);
            hi = min(max(a.offsets[g + 1], 0), a.m);
            hi = max(lo, hi);
        }
    };
    long m_tiles = 0;
    if (a.offsets) {
        for (int g0 = 0; g0 < a.groups; g0 += 64) {
            int lo = 0, hi = 0;
            if (g0 + lane < a.groups) rows_of(g0 + lane, lo, hi);
            int c = (hi - lo + BM - 1) / BM;
#pragma unroll
            for (int s = 32; s; s >>= 1) c += __shfl_xor(c, s);
            m_tiles += c;
        }
    } else m_tiles = (a.m + BM - 1) / BM;
    Tile t = {0, 0, 0, 0};
    // workgroups go round robin over the 8 XCDs: XCD x takes a contiguous eighth of the tiles, so that its L2 sees few panels.
    // Inside it, BAND row tiles go through the channel tiles together.
    const long total = m_tiles * a.n_tiles, per = (total + 7) / 8;
    const long b = blockIdx.x, in = b >> 3, id = (b & 7) * per + in;
    if (in >= per || id >= total) return t;
    const long band = id / ((long)BAND * a.n_tiles), rest = id - band * BAND * a.n_tiles;
    const int bh = (int)min((long)BAND, m_tiles - band * BAND);
    t.nt = (int)(rest / bh);
    int mt = (int)(band * BAND + rest % bh);
    if (!a.offsets) {
        t.r0 = mt * BM;
        t.r1 = min(t.r0 + BM, a.m);
        return t;
    }
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
        int lo = 0, hi = 0;
        if (g0 + lane < a.groups) rows_of(g0 + lane, lo, hi);
        const int c = (hi - lo + BM - 1) / BM;
        int inc = c;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o = __shfl_up(inc, s);
            if (lane >= s) inc += o;
        }
        const uint64_t past = __ballot(inc > mt);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            t.g = g0 + l;
            const int first = __shfl(inc - c, l);
            t.r0 = __shfl(lo, l) + (mt - first) * BM;
            t.r1 = min(t.r0 + BM, __shfl(hi, l));
            t.g = __builtin_amdgcn_readfirstlane(t.g);
            t.r0 = __builtin_amdgcn_readfirstlane(t.r0);
            t.r1 = __builtin_amdgcn_readfirstlane(t.r1);
            return t;
        }
        mt -= __shfl(inc, 63);
    }
    return t;
}

// ---- epilogue: scales, bias, activation, one rounding, store ------------------------------------------------------------------------------
__device__ __forceinline__ float act_f(float v, int act) {
    if (act == PB_ACT_SILU) return pbe::silu_f(v);
    if (act == PB_ACT_TANH) return tanhf(v);
    return v;
}
__device__ __forceinline__ uint16_t bits_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ uint16_t bits_f16(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

// W consecutive channels [c0, ..) of y row yr
template <int W>
__device__ __forceinline__ void store_row(const LinearArgs &a, int yr, int c0, const float (&v)[W]) {
    if (c0 >= a.n) return;
    uint8_t *row = a.y + (long)yr * a.ldy;
    const bool whole = a.y_vec && c0 + W <= a.n;
    if (a.y_type == F32) {
        float *p = reinterpret_cast<float *>(row) + c0;
        if (whole) {
#pragma unroll
            for (int i = 0; i < W; i += 4) *reinterpret_cast<f32x4 *>(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (c0 + i < a.n) p[i] = v[i];
        }
    } else {
        uint16_t *p = reinterpret_cast<uint16_t *>(row) + c0;
        uint16_t h[W];
#pragma unroll
        for (int i = 0; i < W; ++i) h[i] = a.y_type == BF16 ? bits_bf16(v[i]) : bits_f16(v[i]);
        if (whole) {
            if constexpr (W == 8) {
                u32x4 q;
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
                *reinterpret_cast<u32x4 *>(p) = q;
            } else {
                const u32x2 q = {h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16)};
                *reinterpret_cast<u32x2 *>(p) = q;
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (c0 + i < a.n) p[i] = h[i];
        }
    }
}

// what a lane needs of its W output channels
template <int T, int W> struct Chan {
    float scale[W], bias[W];
    __device__ __forceinline__ Chan(const LinearArgs &a, int g, int c0) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const bool in = c0 + i < a.n;
            const long at = (long)g * a.n + c0 + i;
            scale[i] = T == I8 && in ? a.w_scale[at] : 1.0f;
            bias[i] = a.bias && in ? a.bias[at] : 0.0f;
        }
    }
    __device__ __forceinline__ void finish(const LinearArgs &a, const typename Acc<T>::e (&s)[W], float row_scale, int yr, int c0) const {
        float v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
            v[i] = (float)s[i];
            if constexpr (T == I8) v[i] = v[i] * row_scale * scale[i];
            v[i] = act_f(v[i] + bias[i], a.act);
        }
        store_row<W>(a, yr, c0, v);
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

// A wave's sums -> y, 32 rows x WN channels at a time: they go to LDS as the matrix instruction left them (4 consecutive channels per
// lane) and come back as 8 consecutive channels per lane, whole rows by consecutive lanes.  s_mem: 32 (WN + 4) sums for each wave.
template <int T, int MT, int NT, int WN>
__device__ __forceinline__ void store_tile(const LinearArgs &a, int g, const typename Acc<T>::q16 (&acc)[NT][MT], uint8_t *s_mem, const int *yrows,
                                           const float *scales, int wave, int lane, int c_wave) {
    typedef typename Acc<T>::e E;
    typedef typename Acc<T>::q4 Q;
    constexpr int PITCH = WN + 4;
    E *img = reinterpret_cast<E *>(s_mem) + wave * 32 * PITCH;
    constexpr int LPR = WN / 8, RPI = 64 / LPR;  // lanes per row, rows per instruction
    const int li = lane & 31, hi = lane >> 5;
    const int c8 = (lane % LPR) * 8, c0 = c_wave + c8;
    const Chan<T, 8> ch(a, g, c0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const Q v = {acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
                *reinterpret_cast<Q *>(img + li * PITCH + j * 32 + q * 8 + hi * 4) = v;
            }
        __builtin_amdgcn_wave_barrier();  // one wave's LDS accesses are in order
#pragma unroll
        for (int r = lane / LPR; r < 32; r += RPI) {
            const int yr = yrows[i * 32 + r];
            const Q lo = *reinterpret_cast<const Q *>(img + r * PITCH + c8), up = *reinterpret_cast<const Q *>(img + r * PITCH + c8 + 4);
            const E s[8] = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
            if (yr >= 0) ch.finish(a, s, T == I8 ? scales[i * 32 + r] : 1.0f, yr, c0);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- k_linear_tile: a tile of BM rows x BN channels per workgroup, K in steps of 128 bytes through LDS ------------------------------------
// A step has four pieces of 32 bytes of K; a piece's fragments are read from LDS while the one before is multiplied.  The one barrier
// of a step stands before its LAST piece, whose fragments are in registers by then: behind it the step's stage is free, so the loads
// of step i + NST leave there (NST LDS stages) and have NST - 1 steps to arrive, and the first fragments of step i + 1 are read while
// the last piece of step i is multiplied -- the matrix pipe has work across the barrier.  Waves with one or two matrix instructions
// to a piece (FLAT) would wait out an LDS read for each piece: they read all four at once behind the barrier.
// Rows sit in LDS at a pitch of 128 bytes with their eight 16-byte pieces permuted (piece c at c ^ (row / 2 & 7)), which makes the
// fragment reads (16 bytes from each of 32 rows) free of bank conflicts: 249 bytes a clock and CU, against 121 with c ^ (row & 7)
// and 32 unpermuted (LDS reads alone, 256 workgroups of eight waves); the permutation is done by the lanes' GLOBAL addresses, so a
// wave's eight rows of 128 bytes are still whole lines.  DMA: the loads go straight into LDS (16-byte aligned rows); otherwise
// through registers, which takes any alignment.  The last, partial step always goes through registers.
template <int T, int BM, int BN, int WM, int WN, int NST, bool DMA>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void k_linear_tile(const LinearArgs a) {
    constexpr int NWM = BM / WM, NWN = BN / WN, NTHR = 64 * NWM * NWN;
    constexpr int MT = WM / 32, NT = WN / 32;
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int JA = BM * 8 / NTHR, J = (BM + BN) * 8 / NTHR;  // 16-byte pieces per thread and step: of x, in all
    constexpr int PITCH = WN + 4;                                // epilogue image of a wave: 32 rows of WN sums
    constexpr int EPI = NWM * NWN * 32 * PITCH * 4;
    constexpr bool FLAT = MT * NT <= 2;
    constexpr int NF = FLAT ? 4 : 2;  // pieces held in registers
    static_assert(BM * 8 % NTHR == 0 && BN * 8 % NTHR == 0 && NTHR / 8 % 16 == 0 && (NST == 2 || NST == 4), "");
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[(NST * STAGE > EPI ? NST * STAGE : EPI)];
    __shared__ int s_xrow[BM], s_yrow[BM];
    __shared__ float s_scale[T == I8 ? BM : 1];
    const Tile t = find_tile<BM, 4>(a);
    if (t.r0 >= t.r1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    rows_to_lds<T, BM, NTHR>(a, t, tid, s_xrow, s_yrow, s_scale);
    __syncthreads();
    const int lc = ((tid & 7) ^ ((tid >> 4) & 7)) * 16;  // the 16-byte piece this thread moves in every row it touches
    const int c_base = t.nt * BN;
    const uint8_t *pp[J];  // its rows: JA of x, the others of w
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int row = ((tid + j * NTHR) >> 3);
        pp[j] = (j < JA ? a.x + (long)max(s_xrow[j < JA ? row : 0], 0) * a.ldx : a.w + ((long)t.g * a.n + min(c_base + row - BM, a.n - 1)) * a.ldw) + lc;
    }
    const int full = (int)(a.kb >> 7), steps = (int)((a.kb + 127) >> 7);
    auto stage = [&](int i) { return s_mem + (i & (NST - 1)) * STAGE; };
    auto dma = [&](int i, int j) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(pp[j] + (long)i * 128),
                                         (__attribute__((address_space(3))) void *)(stage(i) + wave * 1024 + j * NTHR * 16), 16, 0, 0);
    };
    auto copy_tail = [&](int i) {  // the partial step behind the full ones
#pragma unroll 1
        for (int j = 0; j < J; ++j) {
            const uint8_t *row = j < JA ? a.x + (long)max(s_xrow[(tid + j * NTHR) >> 3], 0) * a.ldx
                                        : a.w + ((long)t.g * a.n + min(c_base + ((tid + j * NTHR) >> 3) - BM, a.n - 1)) * a.ldw;
            *reinterpret_cast<u32x4 *>(stage(i) + (tid + j * NTHR) * 16) = load16_tail<DMA>(row, (long)i * 128 + lc, a.kb);
        }
    };
    u32x4 regs[DMA ? 1 : J];
    auto load_regs = [&](int i) {
#pragma unroll
        for (int j = 0; j < J; ++j) regs[DMA ? 0 : j] = load16<false>(pp[j] + (long)i * 128);
    };
    auto put_regs = [&](int i) {
#pragma unroll
        for (int j = 0; j < J; ++j) *reinterpret_cast<u32x4 *>(stage(i) + (tid + j * NTHR) * 16) = regs[DMA ? 0 : j];
    };
    const int wm = wave / NWN * WM, wn = wave % NWN * WN, li = lane & 31, hi = lane >> 5;
    typename Acc<T>::q16 acc[NT][MT] = {};
    const uint8_t *sa = s_mem + (wm + li) * 128, *sb = s_mem + (BM + wn + li) * 128;
    u32x4 fa[NF][MT], fb[NF][NT];
    auto read = [&](int i, int ks, int to) {
        const int c = (i & (NST - 1)) * STAGE + ((ks * 2 + hi) ^ ((li >> 1) & 7)) * 16;
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[to][j] = *reinterpret_cast<const u32x4 *>(sb + j * 4096 + c);
#pragma unroll
        for (int m = 0; m < MT; ++m) fa[to][m] = *reinterpret_cast<const u32x4 *>(sa + m * 4096 + c);
    };
    // a piece; `send`: the loads of step i among its matrix instructions
    auto multiply = [&](int from, bool send, int i) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int m = 0; m < MT; ++m) mma32<T>(acc[j][m], fb[from][j], fa[from][m]);
            if constexpr (DMA) {
                if (send) {
#pragma unroll
                    for (int l = j * J / NT; l < (j + 1) * J / NT; ++l) dma(i, l);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // this wave's loads of step i are in LDS; those of younger steps may still be on their way
    auto landed = [&](int i) {
        const int younger = min(NST - 2, full - 1 - i);
        if (NST > 3 && younger >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * J) : "memory");
        else if (NST > 2 && younger == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(J) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    for (int i = 0; i < NST; ++i) {
        if (i < full) {
            if constexpr (DMA) {
#pragma unroll
                for (int j = 0; j < J; ++j) dma(i, j);
            } else {
                load_regs(i);
                put_regs(i);
            }
        } else if (i < steps) copy_tail(i);
    }
    auto barrier = [&] {  // this wave's LDS reads have come back, its LDS writes are done
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (FLAT) {
        for (int i = 0; i < steps; ++i) {
            landed(i);
            barrier();  // step i is in LDS, everyone has read step i - 1
            const int next = i - 1 + NST;
            const bool more = i > 0 && next < full;
            if (more) {
                if constexpr (DMA) {
#pragma unroll
                    for (int j = 0; j < J; ++j) dma(next, j);
                } else load_regs(next);
            } else if (i > 0 && next == full && full < steps) copy_tail(full);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) read(i, ks, ks);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) multiply(ks, false, 0);
            if constexpr (!DMA) {
                if (more) put_regs(next);
            }
        }
    } else {
        landed(0);
        barrier();
        if (steps > 0) read(0, 0, 0);
        for (int i = 0; i < steps; ++i) {
            const bool more = !DMA && i > 0 && i + NST - 1 < full;
            if (more) load_regs(i + NST - 1);
            read(i, 1, 1);
            multiply(0, false, 0);
            read(i, 2, 0);
            multiply(1, false, 0);
            read(i, 3, 1);
            multiply(0, false, 0);
            if (more) put_regs(i + NST - 1);
            landed(i + 1);
            barrier();  // the last piece's fragments are in registers everywhere, step i + 1 is in LDS
            if (i + NST == full && full < steps) copy_tail(full);
            if (i + 1 < steps) read(i + 1, 0, 0);
            multiply(1, DMA && i + NST < full, i + NST);
        }
    }
    __syncthreads();  // the stages become the waves' epilogue images
    store_tile<T, MT, NT, WN>(a, t.g, acc, s_mem, s_yrow + wm, s_scale + (T == I8 ? wm : 0), wave, lane, c_base + wn);
}

// ---- k_linear_few: 16 MT rows x 16 NT channels per workgroup, K split over its NW waves ----------------------------------------------------
// For few rows (or little work): the weights are read once, straight into registers, 256 bytes of a row per wave and turn; the
// waves' partial sums meet in LDS and are added in wave order.
template <int T, int MT, int NT, int NW, int U, bool ALIGNED>
__global__ __launch_bounds__(64 * NW) void k_linear_few(const LinearArgs a) {
    typedef typename Acc<T>::e E;
    typedef typename Acc<T>::q4 Q;
    constexpr int BM = 16 * MT, BN = 16 * NT;
    constexpr int PITCH = BN + 4;
    __shared__ __attribute__((aligned(16))) E s_sum[NW][BM * PITCH];
    const Tile t = find_tile<BM, 1>(a);
    if (t.r0 >= t.r1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, kq = (lane >> 4) * 16;
    const int c_base = t.nt * BN;
    const uint8_t *px[MT], *pw[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) px[i] = a.x + (long)max(x_row_of(a, min(t.r0 + i * 16 + li, t.r1 - 1)), 0) * a.ldx;
#pragma unroll
    for (int j = 0; j < NT; ++j) pw[j] = a.w + ((long)t.g * a.n + min(c_base + j * 16 + li, a.n - 1)) * a.ldw;
    Q acc[NT][MT] = {};
    for (long kb = (long)wave * 64 * U; kb < a.kb; kb += 64 * U * NW) {
        u32x4 fw[U][NT], fx[U][MT];
        if (kb + 64 * U <= a.kb) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < NT; ++j) fw[u][j] = load16<ALIGNED>(pw[j] + kb + u * 64 + kq);
#pragma unroll
                for (int i = 0; i < MT; ++i) fx[u][i] = load16<ALIGNED>(px[i] + kb + u * 64 + kq);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < NT; ++j) fw[u][j] = load16_tail<ALIGNED>(pw[j], kb + u * 64 + kq, a.kb);
#pragma unroll
                for (int i = 0; i < MT; ++i) fx[u][i] = load16_tail<ALIGNED>(px[i], kb + u * 64 + kq, a.kb);
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
    __syncthreads();
    for (int q = tid; q < BM * BN / 4; q += 64 * NW) {
        const int r = q / (BN / 4), c = (q % (BN / 4)) * 4;
        if (t.r0 + r >= t.r1) continue;
        Q s = *reinterpret_cast<const Q *>(&s_sum[0][r * PITCH + c]);
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const Q o = *reinterpret_cast<const Q *>(&s_sum[w][r * PITCH + c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += o[i];
        }
        const int xr = x_row_of(a, t.r0 + r), yr = y_row_of(a, t.r0 + r);
        if (xr < 0 || yr < 0) continue;
        const Chan<T, 4> ch(a, t.g, c_base + c);
        const E e[4] = {s[0], s[1], s[2], s[3]};
        ch.finish(a, e, T == I8 ? a.x_scale[xr] : 1.0f, yr, c_base + c);
    }
}

// ---- k_quantize_rows ------------------------------------------------------------------------------------------------------------------------
// scale = max(max |x| / 127, 2^-126); code = x / scale to the nearest whole number, halves to the even one.  The code is decided
// exactly without a division per value: r = rint(x * (1 / scale)) is off by at most one, and x - r * scale, which one fused
// multiply-add gives exactly wherever it is near scale / 2, says on which side of the half x lies.  A row with an infinity or a
// NaN gets scale = NaN and codes 0, so that what is computed from it shows.
__device__ __forceinline__ int code_of(float x, float inv, float scale, float half) {
    float r = rintf(x * inv);
    const float d = __builtin_fmaf(-r, scale, x), ad = fabsf(d);
    const float up = d > 0.0f ? 1.0f : -1.0f;
    const bool odd = ((int)r & 1) != 0;
    if (ad > half || (ad == half && odd)) r += up;
    return (int)r;
}

template <int T> __device__ __forceinline__ float elem(const uint8_t *row, long i) {
    if constexpr (T == F32) return reinterpret_cast<const float *>(row)[i];
    else if constexpr (T == BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(row)[i] << 16);
    else return (float)reinterpret_cast<const _Float16 *>(row)[i];
}

// A workgroup of NTHR threads per row, V values per thread and turn; rows of up to NTHR * V * TURNS values stay in registers between
// the maximum and the codes, longer ones are read a second time.  VEC: 16-byte loads (rows start on 16 bytes, codes on V).
template <int T, int NTHR, int TURNS, bool VEC>
__global__ __launch_bounds__(NTHR) void k_quantize_rows(const uint8_t *__restrict__ x, long m, int k, long ldx, int8_t *__restrict__ codes, long ldc,
                                                        float *__restrict__ scale) {
    constexpr int V = T == F32 ? 4 : 8;
    __shared__ uint32_t s_max[NTHR / 64];
    const int tid = threadIdx.x;
    const long row = blockIdx.x;
    const uint8_t *px = x + row * ldx;
    int8_t *pc = codes + row * ldc;
    const uint32_t INF = 0x7f800000u;
    auto load = [&](long c, float (&v)[V]) {
        if (VEC && c + V <= k) {
            const u32x4 q = *reinterpret_cast<const u32x4 *>(px + c * type_bytes(T));
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
    for (int t = 0; t < TURNS; ++t) {
        load(((long)t * NTHR + tid) * V, v[t]);
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(v[t][i]) & 0x7fffffffu);
    }
    for (long c = ((long)TURNS * NTHR + tid) * V; c < k; c += (long)NTHR * V) {
        float u[V];
        load(c, u);
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(u[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if constexpr (NTHR > 64) {
        if ((tid & 63) == 0) s_max[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NTHR / 64; ++w) top = max(top, s_max[w]);
    }
    const bool bad = top >= INF;
    const float sc = bad ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(top) / 127.0f, 1.17549435e-38f);
    if (tid == 0) scale[row] = sc;
    const float inv = 1.0f / sc, half = 0.5f * sc;
    auto put = [&](long c, const float (&u)[V]) {
        if (c >= k) return;
        int8_t q[V];
#pragma unroll
        for (int i = 0; i < V; ++i) q[i] = bad ? (int8_t)0 : (int8_t)code_of(u[i], inv, sc, half);
        if (VEC && c + V <= k) __builtin_memcpy(__builtin_assume_aligned(pc + c, V), q, V);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < k) pc[c + i] = q[i];
        }
    };
#pragma unroll
    for (int t = 0; t < TURNS; ++t) put(((long)t * NTHR + tid) * V, v[t]);
    for (long c = ((long)TURNS * NTHR + tid) * V; c < k; c += (long)NTHR * V) {
        float u[V];
        load(c, u);
        put(c, u);
    }
}

// ---- k_group_rows ---------------------------------------------------------------------------------------------------------------------------
// Workgroup g < groups counts the rows of smaller groups (its offset) and lists its own rows in ascending order; workgroup `groups`
// lists the rows without a group behind all others.  Every workgroup reads the whole array (it sits in L2) instead of meeting the
// others: no scratch memory, no atomics, one launch, one possible result.  A wave owns a contiguous segment, a lane four
// consecutive rows of each 256, and remembers its matches as bits, so that up to 131 072 rows are read once.
constexpr int GR_WAVES = 16, GR_TURNS = 32, GR_CHUNK = GR_WAVES * GR_TURNS * 256;

__global__ __launch_bounds__(64 * GR_WAVES) void k_group_rows(const int32_t *__restrict__ group, int m, int groups, int vec, int32_t *__restrict__ offsets,
                                                              int32_t *__restrict__ order) {
    __shared__ int s_lt[GR_WAVES], s_eq[GR_WAVES];
    const int g = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunks = (m + GR_CHUNK - 1) / GR_CHUNK;  // m = 0: none
    int seg = 0;
    uint32_t bits[GR_TURNS / 8];  // 4 bits for each turn
    int lt = 0, eq = 0;
    auto look = [&](long at, int n, uint32_t &eq4, int &lt4) {  // rows [at, at + 4) of the n below the segment's end
        int id[4];
        if (vec && at + 4 <= n) {
            const i32x4 q = *reinterpret_cast<const i32x4 *>(group + at);
            id[0] = q.x; id[1] = q.y; id[2] = q.z; id[3] = q.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) id[i] = at + i < n ? group[at + i] : -2;
        }
        eq4 = 0;
        lt4 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = at + i < n, has = (unsigned)id[i] < (unsigned)groups;
            const int key = has ? id[i] : groups;
            eq4 |= (in && key == g ? 1u : 0u) << i;
            lt4 += in && key < g ? 1 : 0;
        }
    };
    auto scan_chunk = [&](int c) {  // fills bits and eq of this wave's segment of chunk c, adds to lt
        const long base = (long)c * GR_CHUNK;
        const int n = (int)min((long)GR_CHUNK, (long)m - base);
        seg = ((n + GR_WAVES - 1) / GR_WAVES + 255) & ~255;
        eq = 0;
#pragma unroll
        for (int w = 0; w < GR_TURNS / 8; ++w) {
            bits[w] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int t = w * 8 + j;
                if (t * 256 >= seg) break;
                const long at = base + (long)wave * seg + t * 256 + lane * 4;
                uint32_t e4;
                int l4;
                look(at, (int)min((long)m, base + n), e4, l4);
                bits[w] |= e4 << (4 * j);
                lt += l4;
            }
            eq += __builtin_popcount(bits[w]);
        }
    };
    auto wave_sum = [&](int v) {
#pragma unroll
        for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
        return v;
    };
    for (int c = 0; c < chunks; ++c) scan_chunk(c);
    const int wl = wave_sum(lt);
    if (lane == 0) s_lt[wave] = wl;
    __syncthreads();
    int first = 0;
#pragma unroll
    for (int w = 0; w < GR_WAVES; ++w) first += s_lt[w];
    if (threadIdx.x == 0) offsets[g] = first;  // workgroup `groups`: the number of rows that have a group
    for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) scan_chunk(c);
        const int we = wave_sum(eq);
        __syncthreads();  // the last chunk's counts have been read
        if (lane == 0) s_eq[wave] = we;
        __syncthreads();
        int at = first;
#pragma unroll
        for (int w = 0; w < GR_WAVES; ++w) {
            if (w < wave) at += s_eq[w];
            first += s_eq[w];
        }
        const long base = (long)c * GR_CHUNK + (long)wave * seg;
#pragma unroll
        for (int w = 0; w < GR_TURNS / 8; ++w) {
            if (__ballot(bits[w] != 0) == 0) continue;
            for (int j = 0; j < 8; ++j) {
                const uint32_t e4 = (bits[w] >> (4 * j)) & 15u;
                int before = 0, all = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint64_t b = __ballot((e4 >> i) & 1u);
                    before += __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0u));
                    all += __builtin_popcountll(b);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((e4 >> i) & 1u) order[at + before + __builtin_popcount(e4 & ((1u << i) - 1u))] = (int32_t)(base + (w * 8 + j) * 256 + lane * 4 + i);
                at += all;
            }
        }
    }
}

}  // namespace pbl
