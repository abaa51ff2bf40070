// The rates behind the floors of the linear layers: matrix instructions without loads, LDS reads of the tile kernels' fragments with and without
// the permutation of a row's 16-byte pieces, HBM reads and copies, an empty launch.
//   hipcc --offload-arch=gfx950 -O3 -Xclang -target-feature -Xclang -packed-fp32-ops profiles/micro/linear_rates.hip -o linear_rates
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../include/pixelbox_hip.h"
#include "../../pixelbox_amd/csrc/pb_linear_kernels.h"

using namespace pbl;
#define CK(x)                                                     \
    do {                                                          \
        hipError_t e_ = (x);                                      \
        if (e_ != hipSuccess) {                                   \
            printf("%s: %s\n", #x, hipGetErrorString(e_));        \
            exit(1);                                              \
        }                                                         \
    } while (0)

// random bits; type BF16, F16, F32: values of either sign from 0.5 to 1 (or 2)
__global__ void k_fill(uint32_t *p, long n, int type) {
    for (long i = blockIdx.x * 256l + threadIdx.x; i < n; i += gridDim.x * 256l) {
        uint32_t h = (uint32_t)i * 2654435761u + 17u;
        h = (h ^ h >> 15) * 2246822519u;
        h = (h ^ h >> 13) * 3266489917u;
        h ^= h >> 16;
        p[i] = type == BF16 ? (h & 0x807f807fu) | 0x3f003f00u : type == F16 ? (h & 0x83ff83ffu) | 0x38003800u : type == F32 ? (h & 0x807fffffu) | 0x3f000000u : h;
    }
}

// eight independent sums a wave (or sixteen of 16 x 16), two waves a SIMD
template <int T, bool WIDE> __global__ __launch_bounds__(512) void k_mfma(float *out, int n, const uint8_t *src) {
    u32x4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = *reinterpret_cast<const u32x4 *>(src + (threadIdx.x * 8 + i) * 16);
        b[i] = *reinterpret_cast<const u32x4 *>(src + (threadIdx.x * 8 + 4 + i) * 16);
    }
    float s = 0;
    if constexpr (WIDE) {
        typename Acc<T>::q16 c[8] = {};
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) mma32<T>(c[j], a[j & 3], b[(j >> 1) & 3]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) s += (float)c[j][e];
    } else {
        typename Acc<T>::q4 c[16] = {};
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) mma16<T>(c[j], a[j & 3], b[(j >> 2) & 3]);
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += (float)c[j][e];
    }
    if (s == 1.2345f) out[threadIdx.x] = s;
}

// 16-byte reads of 32-row (mode 0: pieces in order, 1: c ^ (row & 7), 2: c ^ (row / 2 & 7)) and of 16-row fragments (3: in order, 4: c ^ (row & 7)),
// rows 128 bytes apart
__global__ __launch_bounds__(512) void k_lds(float *out, int n, int mode) {
    __shared__ __attribute__((aligned(16))) uint32_t s[16384];
    for (int i = threadIdx.x; i < 16384; i += 512) s[i] = i * 7;
    __syncthreads();
    const int l = threadIdx.x & 63, r32 = l & 31, h = l >> 5, r16 = l & 15, q = l >> 4;
    const int off = mode == 0 ? r32 * 128 + h * 16 : mode == 1 ? r32 * 128 + (h ^ (r32 & 7)) * 16 : mode == 2 ? r32 * 128 + (h ^ ((r32 >> 1) & 7)) * 16
                    : mode == 3 ? r16 * 128 + q * 16 : r16 * 128 + (q ^ (r16 & 7)) * 16;
    const uint8_t *p = reinterpret_cast<const uint8_t *>(s) + off;
    u32x4 a = {0, 0, 0, 0};
    for (int i = 0; i < n; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a ^= *reinterpret_cast<const u32x4 *>(p + ((j * 8192) & 65535));
        asm volatile("" ::: "memory");
    }
    if (a.x == 12345) out[threadIdx.x] = (float)a.y;
}

// n is a multiple of 4 * 256 * gridDim.x
template <bool COPY> __global__ __launch_bounds__(256) void k_stream(const u32x4 *x, u32x4 *y, long n) {
    u32x4 a = {0, 0, 0, 0};
    for (long i = blockIdx.x * 256l + threadIdx.x; i < n; i += gridDim.x * 1024l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x4 v = x[i + j * gridDim.x * 256l];
            if constexpr (COPY) y[i + j * gridDim.x * 256l] = v;
            else a ^= v;
        }
    if constexpr (!COPY)
        if (a.x == 0x12345678u) y[threadIdx.x] = a;
}
__global__ void k_nothing() {}

template <class F> float us_of(F f, int n) {
    hipEvent_t a, b;
    CK(hipEventCreate(&a));
    CK(hipEventCreate(&b));
    for (int i = 0; i < 3; ++i) f();
    CK(hipDeviceSynchronize());
    std::vector<float> v;
    for (int r = 0; r < 7; ++r) {
        CK(hipEventRecord(a));
        for (int i = 0; i < n; ++i) f();
        CK(hipEventRecord(b));
        CK(hipEventSynchronize(b));
        float ms;
        CK(hipEventElapsedTime(&ms, a, b));
        v.push_back(ms * 1000 / n);
    }
    std::sort(v.begin(), v.end());
    return v[3];
}

template <int T> void mfma(const char *name, float *out, uint8_t *x, int n, double ops) {
    k_fill<<<64, 256>>>(reinterpret_cast<uint32_t *>(x), 1 << 18, T);
    const float w = us_of([&] { hipLaunchKernelGGL((k_mfma<T, true>), dim3(256), dim3(512), 0, 0, out, n, x); }, 3);
    const float s = us_of([&] { hipLaunchKernelGGL((k_mfma<T, false>), dim3(256), dim3(512), 0, 0, out, n, x); }, 3);
    printf("matrix instructions, %s: 32 x 32 %.0f, 16 x 16 %.0f T/s\n", name, 256.0 * 8 * 8 * n * ops / w * 1e-6, 256.0 * 8 * 16 * n * ops / 2 / s * 1e-6);
    fflush(stdout);
}

int main() {
    float *out;
    uint8_t *x;
    CK(hipMalloc(&out, 8192));
    CK(hipMalloc(&x, 1 << 20));
    mfma<I8>("i8", out, x, 4000, 2.0 * 32 * 32 * 32);
    mfma<BF16>("bf16", out, x, 4000, 2.0 * 32 * 32 * 16);
    mfma<F16>("f16", out, x, 4000, 2.0 * 32 * 32 * 16);
    mfma<F32>("f32", out, x, 1000, 2.0 * 32 * 32 * 8);
    const char *modes[] = {"32 rows, in order", "32 rows, c ^ (row & 7)", "32 rows, c ^ (row / 2 & 7)", "16 rows, in order", "16 rows, c ^ (row & 7)"};
    for (int m = 0; m < 5; ++m) {
        const float t = us_of([&] { hipLaunchKernelGGL(k_lds, dim3(256), dim3(512), 0, 0, out, 5000, m); }, 1);
        printf("LDS reads, %s: %.0f bytes a clock and CU at 2.4 GHz\n", modes[m], 512.0 * 16 * 8 * 5000 / t / 2400);
        fflush(stdout);
    }
    u32x4 *a, *b;
    const long n = 1l << 27;  // 2 GB of 16 bytes
    CK(hipMalloc(&a, n * 16));
    CK(hipMalloc(&b, n * 16));
    k_fill<<<1024, 256>>>(reinterpret_cast<uint32_t *>(a), n * 4, I8);
    for (int grid : {1024, 2048, 4096, 8192}) {
        const float r = us_of([&] { hipLaunchKernelGGL((k_stream<false>), dim3(grid), dim3(256), 0, 0, a, b, n); }, 3);
        const float c = us_of([&] { hipLaunchKernelGGL((k_stream<true>), dim3(grid), dim3(256), 0, 0, a, b, n); }, 3);
        printf("%d workgroups: read 2 GB %.2f TB/s, copy %.2f TB/s\n", grid, n * 16 / r * 1e-6, n * 32 / c * 1e-6);
        fflush(stdout);
    }
    printf("an empty launch, back to back: %.2f us\n", us_of([&] { hipLaunchKernelGGL(k_nothing, dim3(1), dim3(64), 0, 0); }, 500));
    return 0;
}
