// LayerNorm of rows of D values, forward and backward, with the weight's and bias's gradients.
//
//   n = (x - mean) * rstd        y = n * w + b        w = weight, or 1 + scale for a modulated norm
//   h = dy * w                   dx = rstd * (h - mean(h) - n * mean(h * n))
//   dw = sum over rows of dy * n                      db = sum over rows of dy
//
// Weights may differ between groups of consecutive rows (the batch entries of a modulation), and their
// gradients are one row per group.  Statistics, sums and gradients are fp32, each output rounded once.
//
// Everything here is bound by memory: x is read once and y written once, and backward reads x and dy and
// writes dx once (75600 x 5120 bf16: forward 285-298 us, 5.2-5.4 TB/s, backward 430 us, 5.4 TB/s).  A row stays in
// the registers of its threads, E values each; a workgroup walks a strip of rows of one group with the group's weights
// in registers too, and backward keeps the strip's column sums there, one partial row of each per strip, which a
// second kernel adds up in order.
#include "hif8_fp8_dev.h"

namespace hif8 {
namespace ln {
namespace {

using fp8::Eight;
using fp8::load8;
using fp8::load_loose;
using fp8::u32x4;
using fp8::size_of;

constexpr int kThreads = 256;

struct Args {
    const uint8_t *x, *dy;
    uint8_t *y;               // forward: y; backward: dx
    float *stats;             // [rows][2]: mean, rstd
    const uint8_t *w, *b;     // [groups][ld_w], NULL: 1 and 0
    int64_t ld_w;
    float *part;              // [groups][strips][2][D], NULL: no gradients of w and b
    int64_t rows_per_group;
    int D, strips, w_dt;
    float eps, plus;          // plus: 1 for a modulation (w = 1 + scale)
};

__device__ __forceinline__ void put(void *p, int64_t i, int dt, float v)
{
    if (dt == HIF8_DTYPE_F32) ((float *)p)[i] = v;
    else if (dt == HIF8_DTYPE_F16) ((_Float16 *)p)[i] = _Float16(v);
    else ((__bf16 *)p)[i] = __bf16(v);
}

// N bytes at whatever address a row has, past the L2.
template <typename T> struct __attribute__((packed, aligned(2))) Loose {
    T v;
};
template <typename T> __device__ __forceinline__ void store_loose(uint8_t *p, T v)
{
    __builtin_nontemporal_store(v, &((Loose<T> *)p)->v);
}

// E values of a row in W threads, 8 consecutive ones in 16 bytes (fp32: twice).  KIND: kWhole, D is a multiple of 8;
// kTail, the thread with the row's end takes the row's last 8 values, some of which its neighbour has too: both
// compute and store the same of them, and only the sums leave them out; kShort, rows of less than 8 values.
enum Kind { kWhole, kTail, kShort };
template <int DT, int E, Kind KIND> struct Frag {
    Eight<DT> c[E / 8];
    static constexpr int kSize = size_of<DT>();
    // the first of the 8 columns of chunk k, and how many of them are a neighbour's (8: the thread has none)
    static __device__ __forceinline__ int start(int k, int t, int W, int D)
    {
        const int at = (k * W + t) * 8;
        return KIND == kTail && at > D - 8 ? D - 8 : at;
    }
    static __device__ __forceinline__ int skip(int k, int t, int W, int D)
    {
        const int at = (k * W + t) * 8;
        return at >= D ? 8 : at - start(k, t, W, D);
    }
    // whether value i counts in sums
    static __device__ __forceinline__ bool counts(int i, int t, int W, int D)
    {
        return KIND == kShort ? t == 0 && i < D : i % 8 >= skip(i / 8, t, W, D);
    }
    __device__ __forceinline__ void load(const uint8_t *row, int t, int W, int D)
    {
#pragma unroll
        for (int k = 0; k < E / 8; ++k) {
            c[k] = Eight<DT>{};
            if (KIND == kShort) c[k] = load8<DT>(row, (k * W + t) * 8, D);
            else if ((k * W + t) * 8 < D) {
                const uint8_t *p = row + start(k, t, W, D) * kSize;
                four(c[k], 0, load_loose<u32x4>(p));
                if constexpr (DT == HIF8_DTYPE_F32) four(c[k], 4, load_loose<u32x4>(p + 16));
            }
        }
    }
    static __device__ __forceinline__ void four(Eight<DT> &c, int i, const u32x4 &v)
    {
        c.w[i] = v.x, c.w[i + 1] = v.y, c.w[i + 2] = v.z, c.w[i + 3] = v.w;
    }
    __device__ __forceinline__ float get(int i) const { return c[i / 8].get(i % 8); }
    static __device__ __forceinline__ void store(uint8_t *row, int t, int W, int D, const float (&v)[E])
    {
        typedef float f8 __attribute__((ext_vector_type(8)));
        typedef _Float16 h8 __attribute__((ext_vector_type(8)));
        typedef __bf16 b8 __attribute__((ext_vector_type(8)));
        typedef float f4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < E / 8; ++k) {
            if ((k * W + t) * 8 >= D) continue;
            if (KIND == kShort) {
                for (int j = 0; j < 8; ++j)
                    if (j < D) put(row, j, DT, v[j]);
                continue;
            }
            uint8_t *p = row + start(k, t, W, D) * kSize;
            f8 o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = v[k * 8 + j];
            if constexpr (DT == HIF8_DTYPE_F32) {
                store_loose(p, __builtin_bit_cast(u32x4, f4{o[0], o[1], o[2], o[3]}));
                store_loose(p + 16, __builtin_bit_cast(u32x4, f4{o[4], o[5], o[6], o[7]}));
            } else if constexpr (DT == HIF8_DTYPE_F16)
                store_loose(p, __builtin_bit_cast(u32x4, __builtin_convertvector(o, h8)));
            else
                store_loose(p, __builtin_bit_cast(u32x4, __builtin_convertvector(o, b8)));
        }
    }
};

template <int CTRL> __device__ __forceinline__ float dpp_add(float v)
{
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float wave_sum(float v)
{
    v = dpp_add<0xB1>(v);      // the neighbour, the other pair of four, the other half of eight, of sixteen
    v = dpp_add<0x4E>(v);
    v = dpp_add<0x141>(v);
    v = dpp_add<0x140>(v);
    // rows of 16 lanes, then halves of the wave, change places with a copy's
    uint32_t a = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    a = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1));
    const auto q = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    const uint32_t q0 = q[0], q1 = q[1];
    return __builtin_bit_cast(float, q0) + __builtin_bit_cast(float, q1);
}
// Sums over the W threads of a row.  WIDE (more than a wave): through LDS, two buffers in turn, so that one barrier
// a call is enough.
template <bool WIDE> struct Sums {
    float (*buf)[2][16];
    int waves, at = 0;
    __device__ __forceinline__ float operator()(float a)
    {
        a = wave_sum(a);
        if (WIDE) {
            if ((threadIdx.x & 63) == 0) buf[at][0][threadIdx.x >> 6] = a;
            __syncthreads();
            a = 0.0f;
            for (int i = 0; i < waves; ++i) a += buf[at][0][i];
            at ^= 1;
        }
        return a;
    }
    __device__ __forceinline__ void operator()(float &a, float &b)
    {
        a = wave_sum(a);
        b = wave_sum(b);
        if (WIDE) {
            if ((threadIdx.x & 63) == 0) {
                buf[at][0][threadIdx.x >> 6] = a;
                buf[at][1][threadIdx.x >> 6] = b;
            }
            __syncthreads();
            a = b = 0.0f;
            for (int i = 0; i < waves; ++i) {
                a += buf[at][0][i];
                b += buf[at][1][i];
            }
            at ^= 1;
        }
    }
};

// Strip s of a group takes `rows` rows of every rows * strips: all workgroups walk through the group's memory
// together (rows next to each other in one strip: 5-10 % slower on 774 MB).
__device__ __forceinline__ void strip_rows(const Args &A, int s, int rows, int64_t &r0, int64_t &step)
{
    r0 = int64_t(s) * rows;
    step = int64_t(rows) * A.strips;
}

// A weight's row as the threads hold x's; its type is its own.
template <int WT, int E, Kind KIND> __device__ __forceinline__ void load_row(const uint8_t *p, int t, int W, int D, float add, float (&w)[E])
{
    Frag<WT, E, KIND> f;
    f.load(p, t, W, D);
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = add + f.get(i);
}
template <int E, Kind KIND>
__device__ __forceinline__ void load_weight(const uint8_t *base, const Args &A, int64_t group, int t, int W, float add, float (&w)[E])
{
    const uint8_t *p = base + group * A.ld_w * (A.w_dt == HIF8_DTYPE_F32 ? 4 : 2);
    if (A.w_dt == HIF8_DTYPE_F32) load_row<HIF8_DTYPE_F32, E, KIND>(p, t, W, A.D, add, w);
    else if (A.w_dt == HIF8_DTYPE_F16) load_row<HIF8_DTYPE_F16, E, KIND>(p, t, W, A.D, add, w);
    else load_row<HIF8_DTYPE_BF16, E, KIND>(p, t, W, A.D, add, w);
}

// WIDE: the workgroup has one row in hand, blockDim.x threads for it; otherwise one a wave.
template <int DT, int E, Kind KIND, bool WIDE> __global__ __launch_bounds__(WIDE ? 512 : kThreads) void k_ln_fwd(const Args A)
{
    typedef Frag<DT, E, KIND> F;
    __shared__ float buf[2][2][16];
    const int W = WIDE ? int(blockDim.x) : 64, rows = WIDE ? 1 : kThreads / 64;
    Sums<WIDE> sums{buf, W / 64};
    const int t = WIDE ? threadIdx.x : threadIdx.x & 63, sub = WIDE ? 0 : threadIdx.x >> 6;
    const int64_t group = blockIdx.y;
    const int64_t row_bytes = int64_t(A.D) * size_of<DT>(), base = group * A.rows_per_group;
    int64_t r0, step;
    const int64_t r1 = A.rows_per_group;
    strip_rows(A, blockIdx.x, rows, r0, step);
    F next;
    if (r0 + sub < r1) next.load(A.x + (base + r0 + sub) * row_bytes, t, W, A.D);
    float w[E], b[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        w[i] = 1.0f;
        b[i] = 0.0f;
    }
    if (A.w) load_weight<E, KIND>(A.w, A, group, t, W, A.plus, w);
    if (A.b) load_weight<E, KIND>(A.b, A, group, t, W, 0.0f, b);
    const float inv = 1.0f / float(A.D);
    for (int64_t r = r0 + sub; r < r1; r += step) {
        const F x = next;
        if (r + step < r1) next.load(A.x + (base + r + step) * row_bytes, t, W, A.D);
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += KIND != kTail || F::counts(i, t, W, A.D) ? x.get(i) : 0.0f;
        const float mean = sums(s) / float(A.D);     // a quotient: the mean of equal values is that value
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float d = F::counts(i, t, W, A.D) ? x.get(i) - mean : 0.0f;
            q += d * d;
        }
        const float rstd = 1.0f / sqrtf(sums(q) * inv + A.eps);
        if (t == 0 && A.stats) *(float2 *)(A.stats + 2 * (base + r)) = float2{mean, rstd};
        float y[E];
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = (x.get(i) - mean) * rstd * w[i] + b[i];
        F::store(A.y + (base + r) * row_bytes, t, W, A.D, y);
    }
}

template <int DT, int E, Kind KIND, bool WIDE> __global__ __launch_bounds__(WIDE ? 512 : kThreads) void k_ln_bwd(const Args A)
{
    typedef Frag<DT, E, KIND> F;
    __shared__ float buf[2][2][16];
    __shared__ float col[WIDE ? 1 : 2 * 64 * E];
    const int W = WIDE ? int(blockDim.x) : 64, rows = WIDE ? 1 : kThreads / 64;
    Sums<WIDE> sums{buf, W / 64};
    const int t = WIDE ? threadIdx.x : threadIdx.x & 63, sub = WIDE ? 0 : threadIdx.x >> 6;
    const int64_t group = blockIdx.y;
    const int64_t row_bytes = int64_t(A.D) * size_of<DT>(), base = group * A.rows_per_group;
    int64_t r0, step;
    const int64_t r1 = A.rows_per_group;
    strip_rows(A, blockIdx.x, rows, r0, step);
    F nx, nd;
    float2 ns{};
    auto fetch = [&](int64_t r) {
        nx.load(A.x + (base + r) * row_bytes, t, W, A.D);
        nd.load(A.dy + (base + r) * row_bytes, t, W, A.D);
        ns = *(const float2 *)(A.stats + 2 * (base + r));
    };
    if (r0 + sub < r1) fetch(r0 + sub);
    float w[E], dw[E] = {}, db[E] = {};
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = 1.0f;
    if (A.w) load_weight<E, KIND>(A.w, A, group, t, W, A.plus, w);
    const float inv = 1.0f / float(A.D);
    for (int64_t r = r0 + sub; r < r1; r += step) {
        const F x = nx, d = nd;
        const float mean = ns.x, rstd = ns.y;
        if (r + step < r1) fetch(r + step);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float g = d.get(i), n = (x.get(i) - mean) * rstd, h = g * w[i];
            if (KIND != kTail || F::counts(i, t, W, A.D)) {      // elsewhere g is 0 where it does not count
                s1 += h;
                s2 += h * n;
            }
            db[i] += g;
            dw[i] += g * n;
        }
        sums(s1, s2);
        s1 *= inv;
        s2 *= inv;
        float o[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float n = (x.get(i) - mean) * rstd;
            o[i] = rstd * (d.get(i) * w[i] - s1 - n * s2);
        }
        F::store(A.y + (base + r) * row_bytes, t, W, A.D, o);
    }
    if (!A.part) return;
    if (!WIDE) {       // the waves' column sums, one after the other
        for (int k = rows - 1; k > 0; --k) {
            __syncthreads();
            if (sub == k) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    col[i * 64 + t] = dw[i];
                    col[(E + i) * 64 + t] = db[i];
                }
            }
            __syncthreads();
            if (sub == k - 1) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    dw[i] += col[i * 64 + t];
                    db[i] += col[(E + i) * 64 + t];
                }
            }
        }
    }
    if (sub == 0) {
        float *p = A.part + (group * A.strips + blockIdx.x) * 2 * A.D;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (F::counts(i, t, W, A.D)) {
                const int c = F::start(i / 8, t, W, A.D) + i % 8;
                p[c] = dw[i];
                p[A.D + c] = db[i];
            }
    }
}

// dw and db of a group from its strips' partial rows: 64 columns a workgroup, each wave every 16th strip in order
// with 8 loads under way, then the waves' sums in order.
__global__ __launch_bounds__(1024) void k_ln_cols(const float *__restrict__ part, int strips, int D, void *dw, void *db, int dt)
{
    __shared__ float s[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
    const int64_t group = blockIdx.z;
    void *out = blockIdx.y ? db : dw;
    if (!out) return;
    const float *p = part + group * strips * 2 * D + int64_t(blockIdx.y) * D + (c < D ? c : 0);
    float v = 0.0f;
    for (int i = wave; i < strips; i += 128) {
        float u[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = i + 16 * k < strips ? p[int64_t(i + 16 * k) * 2 * D] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += u[k];
    }
    s[wave][threadIdx.x & 63] = v;
    __syncthreads();
    if (wave == 0 && c < D) {
        v = 0.0f;
        for (int k = 0; k < 16; ++k) v += s[k][threadIdx.x];
        put(out, group * D + c, dt, v);
    }
}

// Rows of up to 1536 values stay in one wave, four rows a workgroup and no barrier; longer ones take 16 values a
// thread in as many waves as they need.  Forward / backward in microseconds, one wave of 24 values a thread against two
// of 16: 4681 x 1536 bf16 6.0 / 17.5 and 9.0 / 27.5, 32760 x 1536 31.6 / 53.9 and 33.5 / 63.3, 32760 x 1032 24.0 / 41.0
// and 29.2 / 57.8, 512 x 1536 3.9 / 9.4 and 4.1 / 13.6; fp32 32760 x 1536 74.6 / 120 and 73.7 / 128.
constexpr int kOneWave = 1536;
template <int DT, int E, Kind KIND, bool WIDE> void launch(bool fwd, const Args &A, uint32_t groups, hipStream_t st)
{
    const dim3 grid{uint32_t(A.strips), groups};
    const int threads = WIDE ? (A.D + 64 * E - 1) / (64 * E) * 64 : kThreads;
    if (fwd) k_ln_fwd<DT, E, KIND, WIDE><<<grid, threads, 0, st>>>(A);
    else k_ln_bwd<DT, E, KIND, WIDE><<<grid, threads, 0, st>>>(A);
}
template <int DT, Kind KIND> void launch_size(bool fwd, const Args &A, uint32_t groups, hipStream_t st)
{
    if (A.D <= 512) launch<DT, 8, KIND, false>(fwd, A, groups, st);
    else if (A.D <= 1024) launch<DT, 16, KIND, false>(fwd, A, groups, st);
    else if (A.D <= kOneWave) launch<DT, 24, KIND, false>(fwd, A, groups, st);
    else launch<DT, 16, KIND, true>(fwd, A, groups, st);
}
template <int DT> void launch_dt(bool fwd, const Args &A, uint32_t groups, hipStream_t st)
{
    if (A.D % 8 == 0) launch_size<DT, kWhole>(fwd, A, groups, st);
    else if (A.D > 8) launch_size<DT, kTail>(fwd, A, groups, st);
    else launch<DT, 8, kShort, false>(fwd, A, groups, st);
}
void launch_all(bool fwd, int dt, const Args &A, uint32_t groups, hipStream_t st)
{
    if (dt == HIF8_DTYPE_BF16) launch_dt<HIF8_DTYPE_BF16>(fwd, A, groups, st);
    else if (dt == HIF8_DTYPE_F16) launch_dt<HIF8_DTYPE_F16>(fwd, A, groups, st);
    else launch_dt<HIF8_DTYPE_F32>(fwd, A, groups, st);
}

constexpr int64_t kMaxDim = 8192;
bool float_dtype(int dt) { return dt == HIF8_DTYPE_BF16 || dt == HIF8_DTYPE_F32 || dt == HIF8_DTYPE_F16; }
int value_bytes(int dt) { return dt == HIF8_DTYPE_F32 ? 4 : 2; }

// Strips of a group.  Forward: up to 40960 waves in all (75600 rows of 5120: 302 us; 1024 workgroups 332), but not
// less than 4 rows a wave, whose weights take as long to load as a row, unless that leaves CUs idle.  Backward:
// about 10 waves a CU, every CU the same (5120 columns: 512 workgroups 424 us, 409 or 614 of them 487 and 503),
// since each strip leaves two partial rows.  Backward in microseconds with 5 / 10 / 15 / 20 waves a CU: 75600 x 5120 412 /
// 430 / 438 / 451, 512 x 5120 19 / 27 / 27 / 27, 20000 x 4096 104 / 99 / 105 / 117, 20000 x 8192 192 / 185 / 185 / 201,
// 32760 x 2048 86 / 84 / 99 / 101, 32760 x 1536 51 / 54 / 57 / 61; fp32 20000 x 4096 198 / 214 / 211 / 216.
int strips_of(bool fwd, int64_t groups, int64_t rows_per_group, int64_t D)
{
    const int64_t at_once = D <= kOneWave ? 4 : 1, waves = D <= kOneWave ? 4 : (D + 1023) / 1024;
    const int64_t most = (rows_per_group + at_once - 1) / at_once;
    int64_t s;
    if (fwd) {
        const int64_t full = (1024 + groups - 1) / groups, cap = (40960 / waves + groups - 1) / groups;
        s = (most + 3) / 4 > full ? (most + 3) / 4 : full;
        s = s < cap ? s : cap;
    } else {
        s = (256 * (waves < 10 ? 10 / waves : 1) + groups - 1) / groups;
    }
    s = s < most ? s : most;
    return int(s > 0 ? s : 1);
}

int check(int64_t rows, int64_t D, int64_t groups, int dt, const void *x, const void *y, const void *w, const void *b,
          int w_dt, int64_t ld_w, float eps)
{
    if (!x || !y || rows <= 0 || D <= 0 || groups <= 0 || rows % groups || !float_dtype(dt) || !(eps >= 0.0f)) return HIF8_ERR_ARG;
    if ((w || b) && (!float_dtype(w_dt) || (groups > 1 && ld_w < D))) return HIF8_ERR_ARG;
    if (D > kMaxDim || groups > 65535) return HIF8_ERR_SHAPE;
    const uint64_t m = uint64_t(value_bytes(dt)) - 1, wmask = uint64_t(value_bytes(w_dt)) - 1;
    if ((uint64_t(x) | uint64_t(y)) & m || (uint64_t(w) | uint64_t(b)) & wmask) return HIF8_ERR_ALIGN;
    return HIF8_OK;
}

}  // namespace
}  // namespace ln
}  // namespace hif8

using namespace hif8;

extern "C" {

int hif8_layer_norm_fwd(const void *x, int dtype, int64_t rows, int64_t dim, int64_t groups, const void *weight,
                        const void *bias, int weight_dtype, int64_t ld_weight, int plus_one, float eps, void *y,
                        float *stats, hif8_stream_t stream)
{
    const int rc = ln::check(rows, dim, groups, dtype, x, y, weight, bias, weight_dtype, ld_weight, eps);
    if (rc != HIF8_OK) return rc;
    if (uint64_t(stats) % 8) return HIF8_ERR_ALIGN;
    ln::Args A{};
    A.x = (const uint8_t *)x, A.y = (uint8_t *)y, A.stats = stats, A.w = (const uint8_t *)weight, A.b = (const uint8_t *)bias;
    A.ld_w = ld_weight, A.rows_per_group = rows / groups, A.D = int(dim), A.w_dt = weight_dtype, A.eps = eps;
    A.plus = plus_one ? 1.0f : 0.0f;
    A.strips = ln::strips_of(true, groups, A.rows_per_group, dim);
    ln::launch_all(true, dtype, A, uint32_t(groups), (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? HIF8_OK : HIF8_ERR_HIP;
}

int64_t hif8_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t dim, int64_t groups)
{
    if (rows <= 0 || dim <= 0 || groups <= 0 || rows % groups) return 0;
    return groups * ln::strips_of(false, groups, rows / groups, dim) * 2 * dim * 4;
}

int hif8_layer_norm_bwd(const void *dy, const void *x, int dtype, int64_t rows, int64_t dim, int64_t groups,
                        const void *weight, int weight_dtype, int64_t ld_weight, int plus_one, const float *stats,
                        void *dx, void *dweight, void *dbias, void *workspace, int64_t workspace_bytes,
                        hif8_stream_t stream)
{
    const int rc = ln::check(rows, dim, groups, dtype, x, dx, weight, nullptr, weight_dtype, ld_weight, 0.0f);
    if (rc != HIF8_OK) return rc;
    const bool cols = dweight || dbias;
    if (!dy || !stats || (cols && !ln::float_dtype(weight_dtype))) return HIF8_ERR_ARG;
    if (cols && (!workspace || workspace_bytes < hif8_layer_norm_bwd_workspace_bytes(rows, dim, groups))) return HIF8_ERR_ARG;
    const uint64_t m = uint64_t(ln::value_bytes(dtype)) - 1, wm = uint64_t(ln::value_bytes(weight_dtype)) - 1;
    if (uint64_t(dy) & m || uint64_t(stats) % 8 || uint64_t(workspace) % 16 || (uint64_t(dweight) | uint64_t(dbias)) & wm)
        return HIF8_ERR_ALIGN;
    ln::Args A{};
    A.x = (const uint8_t *)x, A.dy = (const uint8_t *)dy, A.y = (uint8_t *)dx, A.stats = const_cast<float *>(stats);
    A.w = (const uint8_t *)weight, A.ld_w = ld_weight, A.rows_per_group = rows / groups, A.D = int(dim);
    A.w_dt = weight_dtype, A.plus = plus_one ? 1.0f : 0.0f;
    A.strips = ln::strips_of(false, groups, A.rows_per_group, dim);
    A.part = cols ? (float *)workspace : nullptr;
    hipStream_t st = (hipStream_t)stream;
    ln::launch_all(false, dtype, A, uint32_t(groups), st);
    if (cols)
        ln::k_ln_cols<<<dim3{uint32_t((dim + 63) / 64), 2, uint32_t(groups)}, 1024, 0, st>>>(A.part, A.strips, A.D, dweight,
                                                                                             dbias, weight_dtype);
    return hipGetLastError() == hipSuccess ? HIF8_OK : HIF8_ERR_HIP;
}

}  // extern "C"
