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

// ---- k_linear_tile: a tile of BM rows x BN channels per workgroup, K in steps of 128 bytes through LDS ------------------------------------
// Two LDS stages: the loads of step i + 1 run under the matrix instructions of step i, one barrier per step.  Rows sit in LDS at a
// pitch of 128 bytes with their eight 16-byte pieces permuted by the row number's low three bits (piece c at c ^ (row & 7)), which
// makes the fragment reads (16 bytes from each of 32 rows) free of bank conflicts; the permutation is done by the lanes' GLOBAL
// addresses, so a wave's eight rows of 128 bytes are still whole lines.  DMA: the loads go straight into LDS (16-byte aligned
// rows); otherwise through registers, which takes any alignment.  The last, partial step always goes through registers.
template <int T, int BM, int BN, int WM, int WN, bool DMA>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void k_linear_tile(const LinearArgs a) {
    constexpr int NWM = BM / WM, NWN = BN / WN, NTHR = 64 * NWM * NWN;
    constexpr int MT = WM / 32, NT = WN / 32;
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int JA = BM * 8 / NTHR, JB = BN * 8 / NTHR;  // 16-byte pieces per thread and step
    constexpr int PITCH = WN + 4;                          // epilogue image of a wave: 32 rows of WN sums
    constexpr int EPI = NWM * NWN * 32 * PITCH * 4;
    static_assert(BM * 8 % NTHR == 0 && BN * 8 % NTHR == 0 && NTHR / 8 % 8 == 0, "");
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[(2 * STAGE > EPI ? 2 * STAGE : EPI)];
    __shared__ int s_xrow[BM], s_yrow[BM];
    const Tile t = find_tile<BM, 4>(a);
    if (t.r0 >= t.r1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = tid; i < BM; i += NTHR) {
        const int r = t.r0 + i;
        s_xrow[i] = r < t.r1 ? x_row_of(a, r) : -1;
        s_yrow[i] = r < t.r1 ? y_row_of(a, r) : -1;
    }
    __syncthreads();
    const int lc = (tid & 7) ^ ((tid >> 3) & 7);  // the 16-byte piece this thread moves in every row it touches
    const uint8_t *pa[JA], *pb[JB];
#pragma unroll
    for (int j = 0; j < JA; ++j) pa[j] = a.x + (long)max(s_xrow[(tid + j * NTHR) >> 3], 0) * a.ldx;
    const int c_base = t.nt * BN;
#pragma unroll
    for (int j = 0; j < JB; ++j) pb[j] = a.w + ((long)t.g * a.n + min(c_base + ((tid + j * NTHR) >> 3), a.n - 1)) * a.ldw;
    const long full = a.kb >> 7, steps = (a.kb + 127) >> 7;

    u32x4 ra[JA], rb[JB];
    auto load_regs = [&](long i) {
        const long at = i * 128 + lc * 16;
        if (i < full) {
#pragma unroll
            for (int j = 0; j < JA; ++j) ra[j] = load16<DMA>(pa[j] + at);
#pragma unroll
            for (int j = 0; j < JB; ++j) rb[j] = load16<DMA>(pb[j] + at);
        } else {
#pragma unroll
            for (int j = 0; j < JA; ++j) ra[j] = load16_tail<DMA>(pa[j], at, a.kb);
#pragma unroll
            for (int j = 0; j < JB; ++j) rb[j] = load16_tail<DMA>(pb[j], at, a.kb);
        }
    };
    auto put_regs = [&](int buf) {
        uint8_t *s = s_mem + buf * STAGE;
#pragma unroll
        for (int j = 0; j < JA; ++j) *reinterpret_cast<u32x4 *>(s + (tid + j * NTHR) * 16) = ra[j];
#pragma unroll
        for (int j = 0; j < JB; ++j) *reinterpret_cast<u32x4 *>(s + BM * 128 + (tid + j * NTHR) * 16) = rb[j];
    };
    auto dma = [&](long i, int buf) {
        uint8_t *s = s_mem + buf * STAGE + wave * 1024;  // a wave's 64 lanes fill 1 KiB from here
        const long at = i * 128 + lc * 16;
#pragma unroll
        for (int j = 0; j < JA; ++j)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(pa[j] + at),
                                             (__attribute__((address_space(3))) void *)(s + j * NTHR * 16), 16, 0, 0);
#pragma unroll
        for (int j = 0; j < JB; ++j)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(pb[j] + at),
                                             (__attribute__((address_space(3))) void *)(s + BM * 128 + j * NTHR * 16), 16, 0, 0);
    };
    const int wm = wave / NWN * WM, wn = wave % NWN * WN;
    const int li = lane & 31, hi = lane >> 5;
    typename Acc<T>::q16 acc[NT][MT] = {};
    auto compute = [&](int buf) {
        const uint8_t *sa = s_mem + buf * STAGE + (wm + li) * 128, *sb = s_mem + buf * STAGE + (BM + wn + li) * 128;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int c = ((ks * 2 + hi) ^ (li & 7)) * 16;
            u32x4 fa[MT], fb[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[j] = *reinterpret_cast<const u32x4 *>(sb + j * 4096 + c);
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[i] = *reinterpret_cast<const u32x4 *>(sa + i * 4096 + c);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) mma32<T>(acc[j][i], fb[j], fa[i]);
        }
    };
    if constexpr (DMA) {
        auto fetch = [&](long i, int buf) {
            if (i < full) dma(i, buf);
            else {
                load_regs(i);
                put_regs(buf);
            }
        };
        if (steps > 0) fetch(0, 0);
        for (long i = 0; i < steps; ++i) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of step i have landed in LDS
            __syncthreads();                                  // everyone's have, and everyone is done with the other stage
            if (i + 1 < steps) fetch(i + 1, (int)(i + 1) & 1);
            compute((int)i & 1);
        }
    } else {
        if (steps > 0) {
            load_regs(0);
            put_regs(0);
        }
        for (long i = 0; i < steps; ++i) {
            __syncthreads();
            if (i + 1 < steps) load_regs(i + 1);
            compute((int)i & 1);
            if (i + 1 < steps) put_regs((int)(i + 1) & 1);
        }
    }
    __syncthreads();  // the stages become the waves' epilogue images
    // a wave turns 32 rows x WN channels at a time: its sums go to LDS as the matrix instruction left them (4 consecutive channels
    // per lane) and come back as 8 consecutive channels per lane, whole rows by consecutive lanes
    typedef typename Acc<T>::e E;
    E *img = reinterpret_cast<E *>(s_mem) + wave * 32 * PITCH;
    constexpr int LPR = WN / 8, RPI = 64 / LPR;  // lanes per row, rows per instruction
    const int c8 = (lane % LPR) * 8, c0 = c_base + wn + c8;
    const Chan<T, 8> ch(a, t.g, c0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                typename Acc<T>::q4 v = {acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
                *reinterpret_cast<typename Acc<T>::q4 *>(img + li * PITCH + j * 32 + q * 8 + hi * 4) = v;
            }
        __builtin_amdgcn_wave_barrier();  // one wave's LDS accesses are in order
#pragma unroll
        for (int r = lane / LPR; r < 32; r += RPI) {
            const int at = wm + i * 32 + r, yr = s_yrow[at], xr = s_xrow[at];
            const typename Acc<T>::q4 lo = *reinterpret_cast<const typename Acc<T>::q4 *>(img + r * PITCH + c8);
            const typename Acc<T>::q4 up = *reinterpret_cast<const typename Acc<T>::q4 *>(img + r * PITCH + c8 + 4);
            const E s[8] = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
            if (yr >= 0 && xr >= 0) ch.finish(a, s, T == I8 ? a.x_scale[xr] : 1.0f, yr, c0);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- k_linear_few: 16 MT rows x 16 NT channels per workgroup, K split over its NW waves ----------------------------------------------------
// For few rows (or little work): the weights are read once, straight into registers, 256 bytes of a row per wave and turn; the
// waves' partial sums meet in LDS and are added in wave order.
template <int T, int MT, int NT, int NW, bool ALIGNED>
__global__ __launch_bounds__(64 * NW) void k_linear_few(const LinearArgs a) {
    typedef typename Acc<T>::e E;
    typedef typename Acc<T>::q4 Q;
    constexpr int BM = 16 * MT, BN = 16 * NT, U = 4;
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
