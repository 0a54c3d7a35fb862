// AdamW over many tensors in few launches, with moments in fp32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g              v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8 bits: m and r = sqrt(v) as e4m3 codes with a power-of-two scale for each 128 elements (hif8_fp8_dev.h).
// m is rounded to nearest.  With b2 near 1, r moves by less than half a step of its code, and to nearest it
// would stand still for good; it is rounded up with the probability of the fraction instead, by 16 bits of a
// number that the step, the tensor and the element's place decide.  r > 0 never becomes 0, which would leave
// an update over eps alone.
//
// Each element is read and written once, and every rounding is fp32's own (no contraction: the moments' codes
// go by the last bit), so that the kernel is bound by memory: 28 bytes an element in fp32, 28 with fp32 moments,
// fp32 master weights and a bf16 parameter, 16 with those in 8 bits, 10 without the masters too.  37 million bf16
// parameters with masters: 195 us, 5.3 TB/s; 246 million with 8-bit moments and masters: 718 us, 5.5 TB/s.
//
// The tensors' addresses travel in the kernel's arguments, up to kTensors a launch: nothing is kept between
// calls.  A launch's workgroups take consecutive chunks of its tensors in order.
#include "hif8_fp8_dev.h"

#include <algorithm>
#include <new>
#include <vector>

namespace hif8 {
namespace adamw {
namespace {

using fp8::Eight;

constexpr int kThreads = 256;
constexpr int kChunk = kThreads * 8;      // elements a workgroup handles at a time: 16 blocks of 128
constexpr int kTensors = 48;              // 48 * 72 bytes of arguments and the rest stay below 4 KB
constexpr int64_t kMost = int64_t(1) << 34;    // elements of a launch: a grid has less than 2^32 threads

struct Tensor {
    void *p;
    const void *g;
    void *m, *v;              // fp32, or codes
    uint8_t *ms, *vs;         // scale bytes of codes
    float *master;
    int64_t n;
};
struct Coefficients {         // of one step, from k_prepare
    float step_size, root;    // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    uint32_t key;             // of the step's dither
    uint32_t pad;
};
struct Args {
    Tensor t[kTensors];
    uint32_t chunk_end[kTensors];     // chunks of the tensors up to this one
    uint32_t index[kTensors];         // the tensors' numbers, for the dither
    int count;
    float b1, one_b1, b2, one_b2, eps, keep;
    const Coefficients *co;
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

__device__ __forceinline__ uint32_t mix(uint32_t h)
{
    h = (h ^ (h >> 16)) * 0x6A09E667u;
    h = (h ^ (h >> 15)) * 0xBB67AE85u;
    return h ^ (h >> 16);
}

__global__ void k_prepare(int64_t *step, int advance, double lr, double b1, double b2, uint32_t seed, Coefficients *co)
{
    const int64_t t = *step + advance;
    *step = t;
    co->step_size = float(lr / (1.0 - pow(b1, double(t))));
    co->root = float(1.0 / sqrt(1.0 - pow(b2, double(t))));
    co->key = seed + uint32_t(t) * 0x9E3779B9u;
}

// Values i .. i + 7 of a tensor of n as floats, at whatever address it has; zeros past its end.
template <int DT> __device__ __forceinline__ void read8(const void *p, int64_t i, int64_t n, float (&v)[8])
{
    const Eight<DT> e = fp8::load8<DT>((const uint8_t *)p, i, n);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = e.get(k);
}
template <typename T> __device__ __forceinline__ void store_loose(void *p, T v) { __builtin_memcpy(p, &v, sizeof(T)); }
template <int DT> __device__ __forceinline__ void write8(void *p, int64_t i, int left, const float (&v)[8])
{
    typedef float f4 __attribute__((ext_vector_type(4)));
    typedef float f8 __attribute__((ext_vector_type(8)));
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    f8 o;
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = v[k];
    if (DT == HIF8_DTYPE_F32) {
        float *q = (float *)p + i;
        if (left >= 8) {
            store_loose(q, f4{v[0], v[1], v[2], v[3]});
            store_loose(q + 4, f4{v[4], v[5], v[6], v[7]});
        } else
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < left) q[k] = v[k];
    } else {
        const uint4 w = DT == HIF8_DTYPE_F16 ? __builtin_bit_cast(uint4, __builtin_convertvector(o, h8))
                                             : __builtin_bit_cast(uint4, __builtin_convertvector(o, b8));
        uint16_t *q = (uint16_t *)p + i;
        if (left >= 8) store_loose(q, fp8::u32x4{w.x, w.y, w.z, w.w});
        else {
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < left) q[k] = uint16_t(u[k >> 1] >> (16 * (k & 1)));
        }
    }
}
// the same of codes: 8 bytes
__device__ __forceinline__ uint2 read_codes(const void *p, int64_t i, int left)
{
    const uint8_t *q = (const uint8_t *)p + i;
    uint2 w{0u, 0u};
    if (left >= 8) __builtin_memcpy(&w, q, 8);
    else
        for (int k = 0; k < 8; ++k)
            if (k < left) (k < 4 ? w.x : w.y) |= uint32_t(q[k]) << (8 * (k & 3));
    return w;
}
__device__ __forceinline__ void write_codes(void *p, int64_t i, int left, uint2 w)
{
    uint8_t *q = (uint8_t *)p + i;
    if (left >= 8) __builtin_memcpy(q, &w, 8);
    else
        for (int k = 0; k < 8; ++k)
            if (k < left) q[k] = uint8_t((k < 4 ? w.x : w.y) >> (8 * (k & 3)));
}
__device__ __forceinline__ void decode8(uint2 w, float scale, float (&v)[8])
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w.x), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w.x), true);
    const f2 c = __builtin_amdgcn_cvt_pk_f32_fp8(int(w.y), false), d = __builtin_amdgcn_cvt_pk_f32_fp8(int(w.y), true);
    v[0] = a.x * scale, v[1] = a.y * scale, v[2] = b.x * scale, v[3] = b.y * scale;
    v[4] = c.x * scale, v[5] = c.y * scale, v[6] = d.x * scale, v[7] = d.y * scale;
}
__device__ __forceinline__ uint32_t amax_of(const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fp8::umax(m, __builtin_bit_cast(uint32_t, v[k]) & 0x7FFFFFFFu);
    return fp8::row16_max(m);
}
// a >= 0 (at most 448) on e4m3's grid, up with the probability of the fraction
__device__ __forceinline__ float dithered(float a, uint32_t bits16)
{
    const int e = int(__builtin_bit_cast(uint32_t, a) >> 23) - 127;
    const int q = (e > -6 ? e : -6) - 3;
    const float up = __builtin_bit_cast(float, uint32_t(127 - q) << 23), down = __builtin_bit_cast(float, uint32_t(127 + q) << 23);
    float k = floorf(a * up + float(bits16) * 0x1p-16f);
    k = a > 0.0f && k < 1.0f ? 1.0f : k;
    return k * down;
}

template <int DT, bool BITS8, bool MASTER> __global__ __launch_bounds__(kThreads) void k_adamw(const Args A)
{
    // the tensor of this chunk: the first whose chunks end behind it
    int lo = 0, hi = A.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (blockIdx.x < A.chunk_end[mid]) hi = mid;
        else lo = mid + 1;
    }
    const Tensor T = A.t[lo];
    const uint32_t chunk = blockIdx.x - (lo ? A.chunk_end[lo - 1] : 0u);
    const int64_t i = int64_t(chunk) * kChunk + threadIdx.x * 8;
    const Coefficients co = *A.co;
    const int64_t rest = T.n - i;
    const int left = rest > 8 ? 8 : int(rest);
    float p[8], g[8], m[8], v[8], r[8];
    read8<DT>(T.g, i, T.n, g);
    if (MASTER) read8<HIF8_DTYPE_F32>(T.master, i, T.n, p);
    else read8<DT>(T.p, i, T.n, p);
    if (BITS8) {
        const int64_t blk = i >> 7;
        uint32_t sm = 127, sv = 127;
        if (left > 0) {
            sm = T.ms[blk];
            sv = T.vs[blk];
        }
        decode8(read_codes(T.m, i, left), fp8::scale_value(sm), m);
        decode8(read_codes(T.v, i, left), fp8::scale_value(sv), v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = v[k] * v[k];
    } else {
        read8<HIF8_DTYPE_F32>(T.m, i, T.n, m);
        read8<HIF8_DTYPE_F32>(T.v, i, T.n, v);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        m[k] = m[k] * A.b1 + g[k] * A.one_b1;
        v[k] = v[k] * A.b2 + g[k] * g[k] * A.one_b2;
        r[k] = __builtin_sqrtf(v[k]);       // to nearest; __fsqrt_rn is the instruction alone, off by one in the last place
        p[k] = p[k] * A.keep - m[k] / (r[k] * co.root + A.eps) * co.step_size;
    }
    if (MASTER) write8<HIF8_DTYPE_F32>(T.master, i, left, p);
    write8<DT>(T.p, i, left, p);
    if (!BITS8) {
        write8<HIF8_DTYPE_F32>(T.m, i, left, m);
        write8<HIF8_DTYPE_F32>(T.v, i, left, v);
        return;
    }
    // 16 lanes hold a block of 128; values past the tensor's end are 0
    const uint32_t am = amax_of(m), ar = amax_of(r);
    const uint32_t bm = fp8::scale_byte<fp8::kE4M3>(am), br = fp8::scale_byte<fp8::kE4M3>(ar);
    const float im = fp8::inverse_scale(bm, am), ir = fp8::inverse_scale(br, ar);
    const uint32_t key = mix(co.key + A.index[lo] * 0xBB67AE85u);
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const uint32_t h = mix(uint32_t((i + k) >> 1) * 0x9E3779B9u + key);
        r[k] = dithered(r[k] * ir, h & 0xFFFFu);
        r[k + 1] = dithered(r[k + 1] * ir, h >> 16);
    }
    if (left <= 0) return;
    write_codes(T.m, i, left, uint2{fp8::pack4<fp8::kE4M3>(m[0] * im, m[1] * im, m[2] * im, m[3] * im),
                                    fp8::pack4<fp8::kE4M3>(m[4] * im, m[5] * im, m[6] * im, m[7] * im)});
    write_codes(T.v, i, left, uint2{fp8::pack4<fp8::kE4M3>(r[0], r[1], r[2], r[3]), fp8::pack4<fp8::kE4M3>(r[4], r[5], r[6], r[7])});
    if ((threadIdx.x & 15) == 0) {
        T.ms[i >> 7] = uint8_t(bm);
        T.vs[i >> 7] = uint8_t(br);
    }
}

// Whether no two of the tensors that a call writes share a byte, and no gradient one with any of them.
bool apart(const hif8_adamw_tensor *t, int64_t count, int64_t size, bool bits8)
{
    typedef std::pair<uint64_t, uint64_t> Span;
    std::vector<Span> r;
    r.reserve(size_t(count) * 6);
    auto add = [&](const void *p, int64_t bytes) {
        if (p) r.emplace_back(uint64_t(p), uint64_t(p) + uint64_t(bytes));
    };
    for (int64_t k = 0; k < count; ++k) {
        const int64_t n = t[k].n, moment = bits8 ? n : 4 * n;
        add(t[k].param, n * size);
        add(t[k].master, n * 4);
        add(t[k].exp_avg, moment);
        add(t[k].exp_avg_sq, moment);
        if (bits8) {
            add(t[k].exp_avg_scales, fp8::blocks_of(n));
            add(t[k].exp_avg_sq_scales, fp8::blocks_of(n));
        }
    }
    std::sort(r.begin(), r.end());
    for (size_t k = 1; k < r.size(); ++k)
        if (r[k].first < r[k - 1].second) return false;
    for (int64_t k = 0; k < count; ++k) {
        const uint64_t g0 = uint64_t(t[k].grad), g1 = g0 + uint64_t(t[k].n * size);
        // the last written tensor that begins before the gradient's end
        const auto at = std::lower_bound(r.begin(), r.end(), Span{g1, 0});
        if (at != r.begin() && (at - 1)->second > g0) return false;
    }
    return true;
}

template <int DT> void launch(const Args &A, uint32_t wgs, bool bits8, bool master, hipStream_t st)
{
    if (master) {
        if (bits8) k_adamw<DT, true, true><<<wgs, kThreads, 0, st>>>(A);
        else k_adamw<DT, false, true><<<wgs, kThreads, 0, st>>>(A);
    } else {
        if (bits8) k_adamw<DT, true, false><<<wgs, kThreads, 0, st>>>(A);
        else k_adamw<DT, false, false><<<wgs, kThreads, 0, st>>>(A);
    }
}

}  // namespace
}  // namespace adamw
}  // namespace hif8

using namespace hif8;

extern "C" {

int64_t hif8_adamw_workspace_bytes(void) { return 64; }

int hif8_adamw_step(const hif8_adamw_tensor *tensors, int64_t count, int dtype, int state_bits, int64_t *step, int advance,
                    double lr, double beta1, double beta2, double eps, double weight_decay, uint32_t seed, void *workspace,
                    int64_t workspace_bytes, hif8_stream_t stream)
{
    if (!tensors || count <= 0 || !step || !workspace || workspace_bytes < hif8_adamw_workspace_bytes()) return HIF8_ERR_ARG;
    if (dtype != HIF8_DTYPE_BF16 && dtype != HIF8_DTYPE_F16 && dtype != HIF8_DTYPE_F32) return HIF8_ERR_ARG;
    if (state_bits != 8 && state_bits != 32) return HIF8_ERR_ARG;
    // in this form, so that a NaN is refused
    if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0))
        return HIF8_ERR_ARG;
    if (uint64_t(step) % 8 || uint64_t(workspace) % 16) return HIF8_ERR_ALIGN;
    const bool bits8 = state_bits == 8, master = tensors[0].master != nullptr;
    const uint64_t mask = dtype == HIF8_DTYPE_F32 ? 3 : 1;
    for (int64_t k = 0; k < count; ++k) {
        const hif8_adamw_tensor &t = tensors[k];
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || t.n <= 0) return HIF8_ERR_ARG;
        if ((t.master != nullptr) != master || (bits8 && (!t.exp_avg_scales || !t.exp_avg_sq_scales))) return HIF8_ERR_ARG;
        if ((uint64_t(t.param) | uint64_t(t.grad)) & mask || uint64_t(t.master) % 4 ||
            (!bits8 && (uint64_t(t.exp_avg) | uint64_t(t.exp_avg_sq)) % 4))
            return HIF8_ERR_ALIGN;
        if (t.n > adamw::kMost) return HIF8_ERR_SHAPE;
    }
    try {
        if (!adamw::apart(tensors, count, dtype == HIF8_DTYPE_F32 ? 4 : 2, bits8)) return HIF8_ERR_ARG;
    } catch (const std::bad_alloc &) {
        return HIF8_ERR_HIP;
    }
    hipStream_t st = (hipStream_t)stream;
    adamw::Coefficients *co = (adamw::Coefficients *)workspace;
    adamw::k_prepare<<<1, 1, 0, st>>>(step, advance != 0, lr, beta1, beta2, seed, co);
    adamw::Args A{};
    A.b1 = float(beta1), A.one_b1 = float(1.0 - beta1), A.b2 = float(beta2), A.one_b2 = float(1.0 - beta2);
    A.eps = float(eps), A.keep = float(1.0 - lr * weight_decay), A.co = co;
    for (int64_t k0 = 0; k0 < count; k0 += A.count) {
        int64_t chunks = 0, elements = 0;
        for (A.count = 0; A.count < adamw::kTensors && k0 + A.count < count; ++A.count) {
            const int k = A.count;
            const hif8_adamw_tensor &t = tensors[k0 + k];
            elements += t.n;
            if (k && elements > adamw::kMost) break;
            A.t[k] = adamw::Tensor{t.param, t.grad, t.exp_avg, t.exp_avg_sq, (uint8_t *)t.exp_avg_scales,
                                   (uint8_t *)t.exp_avg_sq_scales, (float *)t.master, t.n};
            chunks += (t.n + adamw::kChunk - 1) / adamw::kChunk;
            A.chunk_end[k] = uint32_t(chunks);        // at most 2^23 + kTensors
            A.index[k] = uint32_t(t.index);
        }
        if (dtype == HIF8_DTYPE_BF16) adamw::launch<HIF8_DTYPE_BF16>(A, uint32_t(chunks), bits8, master, st);
        else if (dtype == HIF8_DTYPE_F16) adamw::launch<HIF8_DTYPE_F16>(A, uint32_t(chunks), bits8, master, st);
        else adamw::launch<HIF8_DTYPE_F32>(A, uint32_t(chunks), bits8, master, st);
    }
    return hipGetLastError() == hipSuccess ? HIF8_OK : HIF8_ERR_HIP;
}

}  // extern "C"
