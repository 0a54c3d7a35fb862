// Quantisation to FP8 blocks (hif8_fp8_dev.h): codes and scale bytes of a matrix, of its transpose, or of
// both from one read, with the sums of its columns on the way (a linear's bias gradient).
//
// Everything here is bound by memory: 2 bytes read and 1 written per bf16 value (2 with the transpose).
#include "hif8_fp8_dev.h"

namespace hif8 {
namespace fp8 {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr int kThreads = 256;

// Codes along the rows.  16 lanes hold a block, 8 values each; a workgroup does 16 blocks at a time.
// Unit u is block u % S of row u / S; the units past a row's last block write its padding bytes.
// 75600 x 5120 bf16: 200-212 us, 5.5-5.8 TB/s; fp32: 335 us, 5.8 TB/s.
template <int DT, int FMT>
__global__ __launch_bounds__(kThreads) void k_fp8_rows(const uint8_t *__restrict__ x, int64_t ld, int64_t cols,
                                                       uint32_t units, uint32_t S, uint32_t nblk,
                                                       uint8_t *__restrict__ codes, uint8_t *__restrict__ scales)
{
    const uint32_t sub = threadIdx.x & 15u;
    for (uint32_t u = blockIdx.x * 16u + (threadIdx.x >> 4); u < units; u += gridDim.x * 16u) {
        const uint32_t row = u / S, b = u - row * S;
        if (b >= nblk) {
            if (sub == 0) scales[u] = 127;
            continue;
        }
        const int64_t c = int64_t(b) * kBlock + sub * 8u;
        const Eight<DT> v = load8<DT>(x + int64_t(row) * ld * size_of<DT>(), c, cols);
        const uint32_t amax = row16_max(amax8(v));
        const uint32_t byte = scale_byte<FMT>(amax);
        *(uint2 *)(codes + int64_t(row) * nblk * kBlock + c) = codes8<DT, FMT>(v, byte, amax);
        if (sub == 0) scales[u] = uint8_t(byte);
    }
}

// Codes along the rows and along the columns of one 128 x 128 tile.  Thread (g, s) = (tid / 16, tid % 16)
// holds rows 8g .. 8g + 7 at columns 8s .. 8s + 7: a wave reads 4 rows of 256 bytes per load, and the 8
// codes of a column that a thread makes are 8 consecutive bytes of the transpose, which goes out through
// LDS.  TILE: one scale for the whole tile.  The transpose's LDS rows are 128 bytes in 16 words of 8,
// word w of column c at w ^ (c >> 3 & 15): the 16 columns that a row of lanes writes at once then lie in
// different banks.  Four waves a SIMD (without the limit the compiler keeps one or two, 2.5 against 4.5 TB/s).
// Maxima of 16-bit values are taken two at a time, the codes by the conversions with a scale, and the codes go
// out past the caches (32760 x 8960 with sums: 281 us, in fp32 and by cached stores 311).
// bf16: 75600 x 5120 both 300-310 us, 5.0-5.1 TB/s; 32000 x 8960 with sums 235 us, 4.9 TB/s, but 32760 x 8960 276-281,
// 4.2 TB/s (also with padded rows of the transpose; columns of tiles first 264, and 255 at 32000); 13824 x 5120 tiles
// 45 us.  fp32 (what the self-attention hands its o projection): 75600 x 5120 both 432 us, 5.4 TB/s; 32760 x 1536 50 us,
// 6.1 TB/s.
template <int DT, int FMT, bool TILE>
__global__ __launch_bounds__(kThreads, DT == HIF8_DTYPE_F32 ? 3 : 4)
void k_fp8_both(const uint8_t *__restrict__ x, int64_t ld, int64_t rows, int64_t cols, uint8_t *__restrict__ codes,
                uint8_t *__restrict__ scales, uint8_t *__restrict__ codes_t, uint8_t *__restrict__ scales_t,
                float *__restrict__ colsum)
{
    constexpr bool kPacked = DT != HIF8_DTYPE_F32;    // 16-bit types: two values a word
    constexpr int kWords = kPacked ? 4 : 8;           // of 8 values
    __shared__ __attribute__((aligned(16))) uint8_t tr[128 * 128];
    __shared__ __attribute__((aligned(16))) uint32_t cmax[16][16 * kWords];
    __shared__ float csum[16][128];
    const int g = threadIdx.x >> 4, s = threadIdx.x & 15;
    const int64_t r0 = int64_t(blockIdx.y) * 128, c0 = int64_t(blockIdx.x) * 128;
    const int64_t c = c0 + s * 8;
    const int64_t cp = blocks_of(cols) * 128, rp = blocks_of(rows) * 128;
    const int64_t Sc = scale_row(cols), Sr = scale_row(rows);
    Eight<DT> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + g * 8 + i;
        v[i] = r < rows ? load8<DT>(x + r * ld * size_of<DT>(), c, cols) : Eight<DT>{};
    }
    // maxima of the thread's rows and columns
    uint32_t rm[8], cm[8] = {};
    auto larger = [](uint32_t a, uint32_t b) { return kPacked ? pk_umax(a, b) : umax(a, b); };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rm[i] = amax8(v[i]);
        if (!TILE) rm[i] = row16_max(rm[i]);
#pragma unroll
        for (int j = 0; j < kWords; ++j) cm[j] = larger(cm[j], v[i].w[j] & (kPacked ? 0x7FFF7FFFu : 0x7FFFFFFFu));
    }
    if (colsum) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) t += v[i].get(j);
            csum[g][s * 8 + j] = t;
        }
    }
    if (TILE) {
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) t = umax(t, rm[i]);
        t = row16_max(t);
        if (s == 0) cmax[0][g] = t;
    } else {
#pragma unroll
        for (int j = 0; j < kWords; j += 4) *(uint4 *)&cmax[g][s * kWords + j] = uint4{cm[j], cm[j + 1], cm[j + 2], cm[j + 3]};
    }
    __syncthreads();
    if (TILE) {
        uint32_t t = 0;
        for (int i = 0; i < 16; ++i) t = umax(t, cmax[0][i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) rm[i] = cm[i] = t;
    } else {
#pragma unroll 4
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int j = 0; j < kWords; j += 4) {
                const uint4 a = *(const uint4 *)&cmax[i][s * kWords + j];
                cm[j] = larger(cm[j], a.x), cm[j + 1] = larger(cm[j + 1], a.y);
                cm[j + 2] = larger(cm[j + 2], a.z), cm[j + 3] = larger(cm[j + 3], a.w);
            }
        if constexpr (kPacked) {
            const uint32_t w[4] = {cm[0], cm[1], cm[2], cm[3]};
#pragma unroll
            for (int j = 0; j < 8; ++j) cm[j] = widen<DT>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu);
        }
    }
    if (colsum && threadIdx.x < 128 && c0 + threadIdx.x < cols) {
        float t = 0.0f;
        for (int i = 0; i < 16; ++i) t += csum[i][threadIdx.x];
        colsum[int64_t(blockIdx.y) * cols + c0 + threadIdx.x] = t;
    }
    if (codes) {
        uint8_t *to = codes + (r0 + g * 8) * cp + c, *sc = scales + (r0 + g * 8) * Sc + blockIdx.x;
        const int left = rows - r0 - g * 8 < 8 ? int(rows - r0) - g * 8 : 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < left) {
                const uint32_t byte = scale_byte<FMT>(rm[i]);
                const uint2 o = codes8<DT, FMT>(v[i], byte, rm[i]);
                __builtin_nontemporal_store(u32x2{o.x, o.y}, (u32x2 *)(to + i * cp));
                if (s == 0) sc[i * Sc] = uint8_t(byte);
            }
        }
        if (s == 0 && blockIdx.x + 1 == gridDim.x)
            for (int i = 0; i < left; ++i)
                for (int64_t p = 1; p < Sc - blockIdx.x; ++p) sc[i * Sc + p] = 127;
    }
    if (!codes_t) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t byte = scale_byte<FMT>(cm[j]);
        Eight<DT> col;          // the column's 8 values, as a row holds them
        if constexpr (kPacked) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                col.w[i] = __builtin_amdgcn_perm(v[2 * i + 1].w[j >> 1], v[2 * i].w[j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) col.w[i] = v[i].w[j];
        }
        *(uint2 *)(tr + (s * 8 + j) * 128 + ((g ^ s) << 3)) = codes8<DT, FMT>(col, byte, cm[j]);
        if (g == 0 && c + j < cols) {
            scales_t[(c + j) * Sr + blockIdx.y] = uint8_t(byte);
            if (blockIdx.y + 1 == gridDim.y)
                for (int64_t p = gridDim.y; p < Sr; ++p) scales_t[(c + j) * Sr + p] = 127;
        }
    }
    __syncthreads();
    // 16 lanes write the 128 bytes of one column's row
    uint8_t *to = codes_t + (c0 + g) * rp + r0 + s * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int col = i * 16 + g;
        if (c0 + col < cols)
            __builtin_nontemporal_store(*(const u32x2 *)(tr + col * 128 + ((s ^ (col >> 3)) << 3)), (u32x2 *)(to + i * 16 * rp));
    }
}

// Column sums: 64 columns a workgroup, each wave every 16th tile's partial sums in order with 8 loads under way,
// then the waves' sums in order.
template <int DT>
__global__ __launch_bounds__(1024) void k_colsum(const float *__restrict__ part, int tiles, int64_t cols, void *__restrict__ out)
{
    __shared__ float s[16][64];
    const int64_t c = int64_t(blockIdx.x) * 64 + (threadIdx.x & 63);
    const int wave = threadIdx.x >> 6;
    const float *p = part + (c < cols ? c : 0);
    float t = 0.0f;
    for (int i = wave; i < tiles; i += 128) {
        float u[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = i + 16 * k < tiles ? p[int64_t(i + 16 * k) * cols] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += u[k];
    }
    s[wave][threadIdx.x & 63] = t;
    __syncthreads();
    if (wave == 0 && c < cols) {
        t = 0.0f;
        for (int k = 0; k < 16; ++k) t += s[k][threadIdx.x];
        if (DT == HIF8_DTYPE_F32) ((float *)out)[c] = t;
        else if (DT == HIF8_DTYPE_F16) ((_Float16 *)out)[c] = _Float16(t);
        else ((__bf16 *)out)[c] = __bf16(t);
    }
}

template <int DT, int FMT>
void launch(const uint8_t *x, int64_t ld, int64_t rows, int64_t cols, bool tile, uint8_t *codes, uint8_t *scales,
            uint8_t *codes_t, uint8_t *scales_t, float *colsum, hipStream_t st)
{
    if (!tile && !codes_t && !colsum) {
        const uint32_t S = uint32_t(scale_row(cols)), units = uint32_t(rows * S);
        const uint32_t wgs = units < (1u << 27) ? (units + 15) / 16 : 1u << 23;    // a grid has less than 2^32 threads
        k_fp8_rows<DT, FMT><<<wgs, kThreads, 0, st>>>(x, ld, cols, units, S, uint32_t(blocks_of(cols)), codes, scales);
        return;
    }
    const dim3 grid{uint32_t(blocks_of(cols)), uint32_t(blocks_of(rows))};
    if (tile) k_fp8_both<DT, FMT, true><<<grid, kThreads, 0, st>>>(x, ld, rows, cols, codes, scales, codes_t, scales_t, colsum);
    else k_fp8_both<DT, FMT, false><<<grid, kThreads, 0, st>>>(x, ld, rows, cols, codes, scales, codes_t, scales_t, colsum);
}

template <int DT>
void launch_dt(const void *x, int64_t ld, int64_t rows, int64_t cols, int fmt, bool tile, uint8_t *codes,
               uint8_t *scales, uint8_t *codes_t, uint8_t *scales_t, float *colsum, hipStream_t st)
{
    const uint8_t *p = (const uint8_t *)x;
    if (fmt == kE4M3) launch<DT, kE4M3>(p, ld, rows, cols, tile, codes, scales, codes_t, scales_t, colsum, st);
    else launch<DT, kE5M2>(p, ld, rows, cols, tile, codes, scales, codes_t, scales_t, colsum, st);
}

bool float_dtype(int dt) { return dt == HIF8_DTYPE_BF16 || dt == HIF8_DTYPE_F32 || dt == HIF8_DTYPE_F16; }

}  // namespace
}  // namespace fp8
}  // namespace hif8

using namespace hif8;

extern "C" {

int64_t hif8_fp8_scale_row(int64_t cols) { return cols > 0 ? fp8::scale_row(cols) : 0; }

int64_t hif8_fp8_quantize_workspace_bytes(int64_t rows, int64_t cols)
{
    return rows > 0 && cols > 0 ? fp8::blocks_of(rows) * cols * 4 : 0;
}

int hif8_fp8_quantize(const void *x, int dtype, int64_t rows, int64_t cols, int64_t ld, int format, int tile,
                      uint8_t *codes, uint8_t *scales, uint8_t *codes_t, uint8_t *scales_t, void *colsum,
                      int colsum_dtype, void *workspace, int64_t workspace_bytes, hif8_stream_t stream)
{
    if (!x || rows <= 0 || cols <= 0 || ld < cols || !fp8::float_dtype(dtype)) return HIF8_ERR_ARG;
    if (format != HIF8_FP8_E4M3 && format != HIF8_FP8_E5M2) return HIF8_ERR_ARG;
    if ((!codes && !codes_t) || !codes != !scales || !codes_t != !scales_t) return HIF8_ERR_ARG;
    if (colsum && (!fp8::float_dtype(colsum_dtype) || !workspace ||
                   workspace_bytes < hif8_fp8_quantize_workspace_bytes(rows, cols)))
        return HIF8_ERR_ARG;
    // a grid's first dimension has less than 2^32 threads, its second 2^16 workgroups; unit numbers in 32 bits
    if (fp8::blocks_of(rows) > 65535 || fp8::blocks_of(cols) > (1 << 23) || fp8::scale_row(cols) * rows >= (int64_t(1) << 31)) return HIF8_ERR_SHAPE;
    if ((uint64_t(codes) | uint64_t(codes_t) | uint64_t(workspace)) % 16) return HIF8_ERR_ALIGN;
    if (uint64_t(x) % (dtype == HIF8_DTYPE_F32 ? 4 : 2)) return HIF8_ERR_ALIGN;
    hipStream_t st = (hipStream_t)stream;
    float *part = colsum ? (float *)workspace : nullptr;
    if (dtype == HIF8_DTYPE_BF16)
        fp8::launch_dt<HIF8_DTYPE_BF16>(x, ld, rows, cols, format, tile != 0, codes, scales, codes_t, scales_t, part, st);
    else if (dtype == HIF8_DTYPE_F16)
        fp8::launch_dt<HIF8_DTYPE_F16>(x, ld, rows, cols, format, tile != 0, codes, scales, codes_t, scales_t, part, st);
    else
        fp8::launch_dt<HIF8_DTYPE_F32>(x, ld, rows, cols, format, tile != 0, codes, scales, codes_t, scales_t, part, st);
    if (colsum) {
        const dim3 grid{uint32_t((cols + 63) / 64)};
        const int tiles = int(fp8::blocks_of(rows));
        if (colsum_dtype == HIF8_DTYPE_F32) fp8::k_colsum<HIF8_DTYPE_F32><<<grid, 1024, 0, st>>>(part, tiles, cols, colsum);
        else if (colsum_dtype == HIF8_DTYPE_F16) fp8::k_colsum<HIF8_DTYPE_F16><<<grid, 1024, 0, st>>>(part, tiles, cols, colsum);
        else fp8::k_colsum<HIF8_DTYPE_BF16><<<grid, 1024, 0, st>>>(part, tiles, cols, colsum);
    }
    return hipGetLastError() == hipSuccess ? HIF8_OK : HIF8_ERR_HIP;
}

}  // extern "C"
