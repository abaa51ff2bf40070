// pb_linear.hip -- C entry points of the linear layers on device buffers (kernels: pb_linear_kernels.h).
//
// Each call checks its arguments on the host, queues one kernel on the caller's stream (quantize_rows one for each 8 or 33 million
// rows, the heads' product one for as many channels as a launch takes) and returns.  Nothing is allocated, no
// state outlives a call: calls on any number of streams and from any number of threads are independent, and a captured graph
// holds nothing that another one shares.
#include <algorithm>
#include <climits>
#include <cmath>

#include "pb_common.h"
#include "pb_linear_kernels.h"

using namespace pbl;

namespace {

// the caller's device for the duration of a call; the device is left alone where it is the current one already
struct Device {
    int prev = -1;
    bool ok = true;
    explicit Device(int dev) {
        int cur = -1;
        ok = hipGetDevice(&cur) == hipSuccess;
        if (ok && cur != dev) {
            ok = hipSetDevice(dev) == hipSuccess;
            prev = cur;
        }
    }
    ~Device() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

// rows of `len` bytes, `pitch` bytes apart
struct Rows {
    const void *p;
    uint64_t rows, pitch, len;
};
Rows rows_of(const void *p, uint64_t rows, uint64_t ld, uint64_t n, int size) { return {p, rows, ld * size, n * size}; }
Rows vector_of(const void *p, uint64_t n) { return {p, 1, n * 4, n * 4}; }
// whether some byte may be in both: exact for rows at one pitch (column ranges of one wider tensor are apart), and for a single row
// between others; rows at different pitches count as one where the spans from first to last byte meet
bool overlap(const Rows &a, const Rows &b) {
    if (!a.p || !b.p || !a.rows || !b.rows || !a.len || !b.len) return false;
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    if (x >= y + (b.rows - 1) * b.pitch + b.len || y >= x + (a.rows - 1) * a.pitch + a.len) return false;
    if (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) return true;
    const uint64_t pitch = a.rows > 1 ? a.pitch : b.pitch, d = y >= x ? (y - x) % pitch : (pitch - (x - y) % pitch) % pitch;
    return d < a.len || d + b.len > pitch;
}
bool bad_type(int t) { return t != PB_TYPE_F32 && t != PB_TYPE_BF16 && t != PB_TYPE_F16; }
bool misaligned(const void *p, int size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) != 0; }

constexpr uint64_t MAX_LD = 1ull << 40, MAX_ROWS = INT_MAX - 256;  // a tile's end stays an int
// rows at a stride of ld elements: row * ld * 4 stays far inside 64 bits
bool fits(uint64_t rows, uint64_t ld) { return rows <= 1 || ld <= (1ull << 50) / rows; }

// The forms of a product.  A launch is taken to cost a start-up time, plus the number of rounds of workgroups it takes times (a form's
// own fixed time + its time per 4096 summed bytes), whatever the type's size, or the time of its bytes at the copy rate if that is more.
// Dense products, us:
//                 4096 channels by 4096 bytes of K, so many workgroups        4330 x 7218 by 64   4096 x 4096 by 4096 bytes, rows
//                 (rows on 16 bytes)                                          bytes               on 16 bytes    on 4   odd
//   few 16 x 16   256: 6.4   512: 10.4  1024: 17.8                            441                 909           1076   1566
//   few 32 x 16   256: 8.3   512: 13.7  1024: 25.1                            404                 720            832   1304
//   few 32 x 32   256: 10.4  512: 17.6  1024: 31.7                            127                 454            499    726
//   tile 64       256: 12.9  512: 19.2  1024: 34.6  2048: 68.0                 86                 132            171    205
//   tile 128      256: 26.4  512: 51.3 (one workgroup per CU)                  66                  94            127    158
//   wide 128      256: 30.5  512: 40.6  1024: 76.5 (two per CU)                57                  83             94    125
//   wide 256      128: 55    256: 60    512: 123                               52                  62
// A tile that holds next to no rows costs less (`thin`: its loads of x are of one row); f32 runs at the f32 matrix rate, a sixteenth of
// the others', and larger tiles gain less there; a longer program starts later when it is not in the instruction caches.  The figures
// below start from these and are fitted, all together, to the times of all forms on 1410 products, dense and grouped, of all types and
// alignments, 1 to 16384 rows, 32 to 8192 channels and values, launched back to back and after other work: the form with the least such
// cost, which is taken, ran 2.3 and 1.2 % longer than the best one there in the geometric mean.  The sum is what was fitted; a single figure
// need not be that form's time (16 x 16 is costed less on 4 bytes than on 16, tiles of 64 and 128 more on 4 than off them), and beyond
// those sizes the rule is only a guess between forms that all give the answer.  Sums of 8-bit products are the same by every form; sums
// of floats are added in an order that goes with the form.
enum Form { FEW11, FEW21, FEW22, TILE64, TILE128, WIDE128, WIDE256, FORMS };
struct FormCost {
    int bm, bn, threads, slots;  // tile, workgroup, workgroups per round
    float start, fixed, cost, cost4, cost_odd, cost_f32, thin;  // costs: rows on 16 bytes, on 4, on less; f32 rows
};
constexpr FormCost FORM[FORMS] = {
    {16, 16, 512, 256, 5.8f, 1.1f, 3.2f, 1.8f, 3.8f, 3.0f, 0.66f},   {32, 16, 512, 256, 6.1f, 0.9f, 4.1f, 4.1f, 4.3f, 5.4f, 0.98f},
    {32, 32, 512, 256, 6.0f, 1.0f, 5.3f, 5.9f, 6.1f, 7.2f, 1.f},     {64, 64, 256, 256, 6.8f, 1.9f, 9.2f, 14.4f, 13.6f, 17.5f, 0.7f},
    {128, 128, 512, 256, 5.9f, 7.1f, 18.9f, 42.f, 28.7f, 67.f, 0.72f}, {128, 128, 256, 512, 8.7f, 8.3f, 28.f, 41.f, 41.8f, 122.f, 0.75f},
    {256, 256, 512, 256, 10.2f, 15.f, 31.8f, 0.f, 0.f, 0.f, 0.72f}};  // rows on 16 bytes only: in registers its loads do not fit

// the workgroups of a launch: what the groups' rows can take in tiles at most (every group but one may end inside a tile) ...
long row_tiles(const LinearArgs &a, const FormCost &f) {
    const long full = ((long)a.m + f.bm - 1) / f.bm;
    return a.offsets ? std::min<long>(full + a.groups - 1, a.m) : full;
}
long workgroups(const LinearArgs &a, const FormCost &f) { return (row_tiles(a, f) * (((long)a.n + f.bn - 1) / f.bn) + 7) / 8 * 8; }

// FORMS where no form's launch stays below 2^32 threads; last: the largest form to choose from
Form pick_form(const LinearArgs &a, bool f32, int align, Form last = WIDE256) {
    // ... and will take: the lengths are not known here.  So many groups have rows if the rows fall evenly; a group's last tile is half
    // full in the middle, and so is the last round
    const bool many = a.offsets && a.groups > 1;
    const float groups = many ? a.groups * (1.f - std::exp(-(float)a.m / a.groups)) : 1.f, rows = (float)a.m / groups;
    const float bytes = ((groups * a.n + a.m) * (float)a.kb + 2.f * a.m * a.n) / 5.1e6f;
    int best = FORMS;
    float least = 3.4e38f;
    for (int i = 0; i <= last; ++i) {
        const FormCost &f = FORM[i];
        if (workgroups(a, f) > UINT32_MAX / f.threads || (i == WIDE256 && (f32 || align < 16))) continue;
        const float per_group = many ? std::max(1.f, rows / (float)f.bm + 0.5f) : (float)(((long)a.m + f.bm - 1) / f.bm);
        const float all = groups * per_group * (float)((a.n + f.bn - 1) / f.bn) / (float)f.slots;
        const float rounds = many ? std::max(1.f, all + 0.5f) : std::ceil(all);
        const float thin = f.thin + (1.f - f.thin) * std::min(1.f, rows / (float)f.bm);
        const float cost = f32 ? f.cost_f32 : align == 16 ? f.cost : align == 4 ? f.cost4 : f.cost_odd;
        const float c = f.start + std::max(bytes, rounds * thin * (f.fixed + cost * (float)a.kb / 4096.f));
        if (c < least) {
            least = c;
            best = i;
        }
    }
    return (Form)best;
}

// AL: every row of x and w starts on so many bytes (16: loads straight into LDS; 4; less)
template <int T, int AL>
int launch_form(const LinearArgs &a, Form f, dim3 grid, hipStream_t s) {
    constexpr bool DW = AL >= 4;
    // pieces of 64 bytes per wave and turn.  f32: the same in all three few forms, so that they add in one order (up to 1024 rows over 8
    // groups, 256 x 1280: 16 x 16 and 32 x 16 outputs 2 % faster to 1 % slower than with 4, 32 x 32 with 4 pieces 3 to 8 % slower)
    constexpr int U = T == F32 ? 2 : 4;
    switch (f) {
        case FEW11: hipLaunchKernelGGL((k_linear_few<T, 1, 1, 8, U, DW>), grid, dim3(512), 0, s, a); break;
        case FEW21: hipLaunchKernelGGL((k_linear_few<T, 2, 1, 8, U, DW>), grid, dim3(512), 0, s, a); break;
        case FEW22: hipLaunchKernelGGL((k_linear_few<T, 2, 2, 8, 2, DW>), grid, dim3(512), 0, s, a); break;
        case TILE64: hipLaunchKernelGGL((k_linear_tile<T, 64, 64, 32, 32, AL == 16 ? 4 : 2, AL == 16>), grid, dim3(256), 0, s, a); break;
        case TILE128: hipLaunchKernelGGL((k_linear_tile<T, 128, 128, 64, 32, 4, AL == 16>), grid, dim3(512), 0, s, a); break;
        case WIDE128: hipLaunchKernelGGL((k_linear_wide<T, 128, 128, 64, 64, 2, 3, AL == 16>), grid, dim3(256), 0, s, a); break;
        default:
            if constexpr (T != F32 && AL == 16) hipLaunchKernelGGL((k_linear_wide<T, 256, 256, 128, 64, 2, 7, true>), grid, dim3(512), 0, s, a);
            break;
    }
    PB_HIP(hipGetLastError());
    return PB_OK;
}
// one_order (f32): every sum is added in an order that depends on k alone -- by the few forms, in as many launches as the channels need
template <int T, int AL>
int launch(LinearArgs a, bool one_order, hipStream_t s) {
    Form f = pick_form(a, T == F32, AL, one_order ? FEW22 : WIDE256);
    if (one_order && f == FORMS) f = FEW22;
    PB_CHECK(f != FORMS, PB_ERR_INVALID, "linear: %d x %d is more than one launch takes", a.m, a.n);
    const long rows = row_tiles(a, FORM[f]), most = (UINT32_MAX / FORM[f].threads - 8) / rows;
    const int tiles = (a.n + FORM[f].bn - 1) / FORM[f].bn, each = one_order ? (int)std::min<long>(tiles, std::max(1l, most)) : tiles;
    for (a.nt0 = 0; a.nt0 < tiles; a.nt0 += each) {
        a.n_tiles = std::min(each, tiles - a.nt0);
        const int rc = launch_form<T, AL>(a, f, dim3((unsigned)((rows * a.n_tiles + 7) / 8 * 8)), s);
        if (rc) return rc;
    }
    return PB_OK;
}
template <int T>
int launch(const LinearArgs &a, bool one_order, hipStream_t s) {
    const uint64_t low = (uint64_t)(uintptr_t)a.x | (uint64_t)(uintptr_t)a.w | (uint64_t)a.ldx | (uint64_t)a.ldw;
    if (low % 16 == 0) return launch<T, 16>(a, one_order, s);
    if constexpr (T != F32) {
        if (low % 4 != 0) return launch<T, 1>(a, one_order, s);
    }
    return launch<T, 4>(a, one_order, s);
}

// what pb_linear_i8 and pb_linear_grouped have in common
int linear(const char *who, int device, void *stream, int type, const void *x, uint64_t x_total, uint64_t ldx, const float *x_scale, const void *w,
           uint64_t ldw, const float *w_scale, const float *bias, const int32_t *offsets, uint32_t groups, const int32_t *x_rows,
           const int32_t *y_rows, int act, void *y, int y_type, uint64_t y_total, uint64_t ldy, uint64_t m, uint32_t n, uint32_t k, bool one_order = false) {
    const bool i8 = type == PB_TYPE_I8;
    PB_CHECK(i8 || !bad_type(type), PB_ERR_INVALID, "%s: unknown type %d", who, type);
    PB_CHECK(!bad_type(y_type), PB_ERR_INVALID, "%s: unknown output type %d (f32, bf16, f16)", who, y_type);
    PB_CHECK(act >= PB_ACT_NONE && act <= PB_ACT_TANH, PB_ERR_INVALID, "%s: unknown activation %d", who, act);
    PB_CHECK(m <= MAX_ROWS && x_total <= MAX_ROWS && y_total <= MAX_ROWS, PB_ERR_INVALID, "%s: more than 2^31 - 257 rows", who);
    PB_CHECK(n <= (uint32_t)INT_MAX / 2 && k <= 1u << 28, PB_ERR_INVALID, "%s: n = %u, k = %u is out of range", who, n, k);
    PB_CHECK(!i8 || k <= PB_LINEAR_I8_MAX_K, PB_ERR_INVALID, "%s: k = %u would overflow 32-bit sums (at most %u)", who, k, PB_LINEAR_I8_MAX_K);
    PB_CHECK(groups >= 1 && groups <= PB_MAX_GROUPS, PB_ERR_INVALID, "%s: groups = %u (1 .. %u)", who, groups, PB_MAX_GROUPS);
    PB_CHECK(ldx >= k && ldw >= k && ldy >= n && ldx <= MAX_LD && ldw <= MAX_LD && ldy <= MAX_LD && fits(x_total, ldx) && fits((uint64_t)groups * n, ldw) && fits(y_total, ldy), PB_ERR_INVALID,
             "%s: rows of %u inputs and %u outputs do not fit their strides, or these the memory", who, k, n);
    if (m == 0 || n == 0) return PB_OK;
    const int size = type_bytes(type), y_size = type_bytes(y_type);
    PB_CHECK(y && (k == 0 || (x && w)), PB_ERR_INVALID, "%s: null buffer", who);
    PB_CHECK(!i8 || (x_scale && w_scale), PB_ERR_INVALID, "%s: 8-bit operands need x_scale and w_scale", who);
    PB_CHECK(x_total > 0 && y_total > 0, PB_ERR_INVALID, "%s: no rows to read or to write", who);
    PB_CHECK(x_rows || m <= x_total, PB_ERR_INVALID, "%s: m = %llu rows of an x of %llu", who, (unsigned long long)m, (unsigned long long)x_total);
    PB_CHECK(y_rows || m <= y_total, PB_ERR_INVALID, "%s: m = %llu rows of a y of %llu", who, (unsigned long long)m, (unsigned long long)y_total);
    PB_CHECK(!misaligned(x, size) && !misaligned(w, size) && !misaligned(y, y_size), PB_ERR_INVALID, "%s: a buffer is not aligned to its type", who);
    PB_CHECK(!misaligned(x_scale, 4) && !misaligned(w_scale, 4) && !misaligned(bias, 4) && !misaligned(offsets, 4) && !misaligned(x_rows, 4) &&
                 !misaligned(y_rows, 4),
             PB_ERR_INVALID, "%s: a scale, bias or index array is not aligned to 4 bytes", who);
    const Rows ys = rows_of(y, y_total, ldy, n, y_size);
    const uint64_t channels = (uint64_t)groups * n;
    PB_CHECK(!overlap(ys, rows_of(x, x_total, ldx, k, size)) && !overlap(ys, rows_of(w, channels, ldw, k, size)), PB_ERR_INVALID, "%s: y overlaps an operand", who);
    PB_CHECK(!(i8 && (overlap(ys, vector_of(x_scale, x_total)) || overlap(ys, vector_of(w_scale, channels)))) && !overlap(ys, vector_of(bias, channels)) &&
                 !overlap(ys, vector_of(offsets, groups + 1ull)) && !overlap(ys, vector_of(x_rows, m)) && !overlap(ys, vector_of(y_rows, m)),
             PB_ERR_INVALID, "%s: y overlaps a scale, the bias or an index array", who);
    Device dev(device);
    PB_CHECK(dev.ok, PB_ERR_HIP, "%s: no HIP device %d", who, device);
    LinearArgs a;
    a.x = static_cast<const uint8_t *>(x);
    a.w = static_cast<const uint8_t *>(w);
    a.x_scale = x_scale;
    a.w_scale = w_scale;
    a.bias = bias;
    a.offsets = offsets;
    a.x_rows = x_rows;
    a.y_rows = y_rows;
    a.y = static_cast<uint8_t *>(y);
    a.ldx = (long)ldx * size;
    a.ldw = (long)ldw * size;
    a.ldy = (long)ldy * y_size;
    a.kb = (int)k * size;
    a.m = (int)m;
    a.n = (int)n;
    a.groups = (int)groups;
    a.n_tiles = a.nt0 = 0;
    a.x_total = (int)x_total;
    a.y_total = (int)y_total;
    a.act = act;
    a.y_type = y_type;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (type) {
        case PB_TYPE_F32: return launch<F32>(a, one_order, s);
        case PB_TYPE_BF16: return launch<BF16>(a, false, s);
        case PB_TYPE_F16: return launch<F16>(a, false, s);
        default: return launch<I8>(a, false, s);
    }
}

// a wave per row where the row fits its registers and there are rows for every CU, else a workgroup of four; launches of fewer than
// 2^32 threads
template <int T>
void launch_quantize(const void *x, uint64_t m, uint32_t k, uint64_t ldx, void *codes, uint64_t ldc, float *scale, hipStream_t s) {
    constexpr uint32_t V = T == F32 ? 4 : 8;
    const long lx = (long)ldx * type_bytes(T), lc = (long)ldc;
    const bool waves = m >= 1024 && k <= 64 * V * 8;
    const uint64_t most = waves ? 4ull << 23 : 1ull << 23;
    for (uint64_t r = 0; r < m; r += most) {
        const uint8_t *px = static_cast<const uint8_t *>(x) + r * lx;
        int8_t *pc = static_cast<int8_t *>(codes) + r * lc;
        const int rows = (int)std::min(most, m - r);
        if (waves) hipLaunchKernelGGL((k_quantize_rows<T, 64, 8>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, px, rows, (int)k, lx, pc, lc, scale + r);
        else hipLaunchKernelGGL((k_quantize_rows<T, 256, 4>), dim3((unsigned)rows), dim3(256), 0, s, px, rows, (int)k, lx, pc, lc, scale + r);
    }
}

}  // namespace

int pb::linear_heads(int device, void *stream, int type, const void *x, const float *x_scale, const void *w, const float *w_scale, const float *bias,
                     const int *offsets, uint32_t heads, const int *order, float *y, uint32_t n, uint32_t d, uint32_t k) {
    return linear("pb_embed_heads_device", device, stream, type, x, n, k, x_scale, w, k, w_scale, bias, offsets, heads, order, order, PB_ACT_TANH, y,
                  PB_TYPE_F32, n, d, n, d, k, true);
}

extern "C" {

int pb_quantize_rows(int device, void *stream, const void *x, int x_type, uint64_t m, uint32_t k, uint64_t ldx, void *codes, uint64_t ldc, float *scale) {
    const char *who = "pb_quantize_rows";
    PB_CHECK(!bad_type(x_type), PB_ERR_INVALID, "%s: unknown type %d (f32, bf16, f16)", who, x_type);
    PB_CHECK(m <= MAX_ROWS && k <= 1u << 28, PB_ERR_INVALID, "%s: m = %llu, k = %u is out of range", who, (unsigned long long)m, k);
    PB_CHECK(ldx >= k && ldc >= k && ldx <= MAX_LD && ldc <= MAX_LD && fits(m, ldx) && fits(m, ldc), PB_ERR_INVALID, "%s: rows of %u values do not fit their strides, or these the memory", who, k);
    if (m == 0) return PB_OK;
    const int size = type_bytes(x_type);
    PB_CHECK(scale && (k == 0 || (x && codes)), PB_ERR_INVALID, "%s: null buffer", who);
    PB_CHECK(!misaligned(x, size) && !misaligned(scale, 4), PB_ERR_INVALID, "%s: a buffer is not aligned to its type", who);
    const Rows xr = rows_of(x, m, ldx, k, size), cr = rows_of(codes, m, ldc, k, 1), sr = vector_of(scale, m);
    PB_CHECK(!overlap(cr, xr) && !overlap(sr, xr) && !overlap(sr, cr), PB_ERR_INVALID, "%s: buffers overlap", who);
    Device dev(device);
    PB_CHECK(dev.ok, PB_ERR_HIP, "%s: no HIP device %d", who, device);
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (x_type) {
        case PB_TYPE_F32: launch_quantize<F32>(x, m, k, ldx, codes, ldc, scale, s); break;
        case PB_TYPE_BF16: launch_quantize<BF16>(x, m, k, ldx, codes, ldc, scale, s); break;
        default: launch_quantize<F16>(x, m, k, ldx, codes, ldc, scale, s); break;
    }
    PB_HIP(hipGetLastError());
    return PB_OK;
}

int pb_linear_i8(int device, void *stream, const void *x, uint64_t ldx, const float *x_scale, const void *w, uint64_t ldw, const float *w_scale,
                 const float *bias, int act, void *y, int y_type, uint64_t ldy, uint64_t m, uint32_t n, uint32_t k) {
    return linear("pb_linear_i8", device, stream, PB_TYPE_I8, x, m, ldx, x_scale, w, ldw, w_scale, bias, nullptr, 1, nullptr, nullptr, act, y, y_type, m, ldy,
                  m, n, k);
}

int pb_group_rows(int device, void *stream, const int *group, uint64_t m, uint32_t groups, int *offsets, int *order) {
    const char *who = "pb_group_rows";
    PB_CHECK(m <= MAX_ROWS, PB_ERR_INVALID, "%s: more than 2^31 - 257 rows", who);
    PB_CHECK(groups >= 1 && groups <= PB_MAX_GROUPS, PB_ERR_INVALID, "%s: groups = %u (1 .. %u)", who, groups, PB_MAX_GROUPS);
    PB_CHECK(offsets && (m == 0 || (group && order)), PB_ERR_INVALID, "%s: null buffer", who);
    PB_CHECK(!misaligned(group, 4) && !misaligned(offsets, 4) && !misaligned(order, 4), PB_ERR_INVALID, "%s: a buffer is not aligned to 4 bytes", who);
    const Rows gr = vector_of(group, m), orr = vector_of(order, m), fr = vector_of(offsets, groups + 1ull);
    PB_CHECK(!overlap(gr, orr) && !overlap(gr, fr) && !overlap(orr, fr), PB_ERR_INVALID, "%s: buffers overlap", who);
    Device dev(device);
    PB_CHECK(dev.ok, PB_ERR_HIP, "%s: no HIP device %d", who, device);
    const int vec = !misaligned(group, 16);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (m <= 4096) hipLaunchKernelGGL((k_group_rows<4>), dim3(groups + 1), dim3(256), 0, s, group, (int)m, (int)groups, vec, offsets, order);
    else hipLaunchKernelGGL((k_group_rows<16>), dim3(groups + 1), dim3(1024), 0, s, group, (int)m, (int)groups, vec, offsets, order);
    PB_HIP(hipGetLastError());
    return PB_OK;
}

int pb_linear_form(int type, uint64_t m, uint32_t n, uint32_t k, uint32_t groups, uint32_t align, int *form) {
    const char *who = "pb_linear_form";
    PB_CHECK(type == PB_TYPE_I8 || !bad_type(type), PB_ERR_INVALID, "%s: unknown type %d", who, type);
    PB_CHECK(m >= 1 && m <= MAX_ROWS && n >= 1 && n <= (uint32_t)INT_MAX / 2 && k <= 1u << 28 && groups <= PB_MAX_GROUPS, PB_ERR_INVALID,
             "%s: m = %llu, n = %u, k = %u, groups = %u is out of range", who, (unsigned long long)m, n, k, groups);
    PB_CHECK(align >= 1 && align <= 16 && (align & (align - 1)) == 0 && form, PB_ERR_INVALID, "%s: align = %u (1, 2, 4, 8, 16), or no room for the form", who, align);
    LinearArgs a = {};
    const int32_t some = 0;
    a.offsets = groups ? &some : nullptr;  // never followed
    a.kb = (int)k * type_bytes(type);
    a.m = (int)m;
    a.n = (int)n;
    a.groups = groups ? (int)groups : 1;
    *form = pick_form(a, type == PB_TYPE_F32, align == 16 ? 16 : align >= 4 || type == PB_TYPE_F32 ? 4 : 1);
    PB_CHECK(*form != FORMS, PB_ERR_INVALID, "%s: %d x %d is more than one launch takes", who, a.m, a.n);
    return PB_OK;
}

int pb_linear_grouped(int device, void *stream, int type, const void *x, uint64_t x_total, uint64_t ldx, const float *x_scale, const void *w, uint64_t ldw,
                      const float *w_scale, const float *bias, const int *offsets, uint32_t groups, const int *x_rows, const int *y_rows, int act,
                      void *y, int y_type, uint64_t y_total, uint64_t ldy, uint64_t m, uint32_t n, uint32_t k) {
    PB_CHECK(offsets || m == 0, PB_ERR_INVALID, "pb_linear_grouped: null offsets");
    return linear("pb_linear_grouped", device, stream, type, x, x_total, ldx, x_scale, w, ldw, w_scale, bias, offsets, groups, x_rows, y_rows, act, y, y_type,
                  y_total, ldy, m, n, k);
}

}  // extern "C"
