// y[M, N] = a[M, K] b[N, K]^T + bias on FP8 blocks (hif8_fp8_dev.h), on the scaled matrix instruction.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies each 32 values of k by a power of two per row of either
// operand.  A block's 128 values take two instructions with the same scale byte, so a product costs the
// same as one without scales, and the accumulators hold the scaled sums in fp32 all along.  The instruction itself
// cuts the terms of 8 consecutive k off towards zero, 13 bits below the largest of them: an fp32 result is 1.1e-5 to
// 1.5e-5 of its norm away from the exact one, 4e-5 to 5e-5 where a few channels are 20 times the others (fp32 sums:
// 1e-7).  The codes' own rounding, up to 2^-4 of a value, is far above that.  Which of the 64 values of k lies in which
// of a lane's registers does not matter as long as both operands agree.
//
// What bounds it: 75600 x 13824 x 5120 takes 4.08-4.5 ms, 2.4-2.6 PFLOP/s (by the card and how warm it is), on random
// codes and 3.25 ms, 3.3 PFLOP/s, with one operand zero: the card's power.  A tile of 256 x 256 takes 2.4 thousand
// cycles a step of 128 k (the matrix instructions alone 2.0) and 14 thousand besides, for its first loads and its
// outputs, so that short k are slower: 32760 x 8960 x 1536 415-480 us, 1.9-2.15 PFLOP/s.  (Workgroups that stay and load
// the next tile's first stage before they write one's outputs are 1 % faster and need every register; they are not
// kept.)  Outputs in fp32 instead of bf16: 75600 x 5120 x 5120 1635 us against 1550, 32760 x 1536 x 1536 95 against 80.
#include "hif8_fp8_dev.h"

namespace hif8 {
namespace fp8 {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
template <int DT> struct Type {
    static constexpr int value = DT;
};
constexpr int kBK = 128;           // bytes of k a step: one block of either operand
constexpr uint32_t kRowBytes = 128;

#define ASMV asm volatile
template <int N> __device__ __forceinline__ void wait_vm() { ASMV("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { ASMV("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() { ASMV("s_barrier" ::: "memory"); }
// 64 lanes x 16 B from the buffer (voff per lane) into LDS at m0v + lane * 16
__device__ __forceinline__ void load_lds(uint32_t m0v, uint32_t voff, const u32x4 &rs)
{
    ASMV("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(m0v), "v"(voff), "s"(rs) : "m0");
}

// Chunks of 16 bytes in an LDS row of 128 are stored at c ^ swizzle(row): the 16-byte reads of one column of
// chunks in 16 consecutive rows then hit all 64 banks once.
__device__ __forceinline__ uint32_t swizzle(uint32_t row) { return (row & 7u) ^ ((row >> 3) & 1u); }

// t / d for t < 2^31 by a product: m = ceil(2^(31 + s) / d) with 2^(s - 1) < d <= 2^s, which fits 32 bits, and
// t (m d - 2^(31 + s)) < 2^31 2^s.
struct Quotient {
    uint32_t m, shift, d;
    void set(uint32_t v)
    {
        d = v;
        shift = 0;
        while ((uint64_t(1) << shift) < v) ++shift;
        m = uint32_t(((uint64_t(1) << (31 + shift)) + v - 1) / v);
        shift += 31;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t t) const { return uint32_t((uint64_t(t) * m) >> shift); }
};
struct Args {
    const uint8_t *a, *sa, *b, *sb;
    const void *bias;
    void *y;
    float *part;          // fp32 sums of k ranges, [splits][M][N]
    int64_t M, N;
    int kp, S;            // bytes of a row of codes, of scale bytes
    int nk, splits, per;  // k steps, k ranges and their steps
    // Tiles go in groups of 2^group_shift rows of them (the last group has by_rest.d), down the rows first:
    // by_group.d tiles a group, full_groups of them.
    Quotient by_group, by_rest;
    int full_groups, group_shift;
    // An item is a tile and a k range: all tiles of the first range, of the second, ...  chunked: each XCD takes
    // items that follow each other, so that its L2 holds one range or few columns of tiles; otherwise every eighth.
    Quotient by_tiles;
    uint32_t items;
    bool chunked;
    int bias_dt, y_dt;
};

__device__ __forceinline__ float load_bias(const void *p, int dt, int64_t n)
{
    if (dt == HIF8_DTYPE_F32) return ((const float *)p)[n];
    if (dt == HIF8_DTYPE_F16) return float(((const _Float16 *)p)[n]);
    return float(((const __bf16 *)p)[n]);
}
__device__ __forceinline__ uint2 pack16(const f32x4 &v, int dt)
{
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    return dt == HIF8_DTYPE_F16 ? __builtin_bit_cast(uint2, __builtin_convertvector(v, h4))
                                : __builtin_bit_cast(uint2, __builtin_convertvector(v, b4));
}
// four values from element `at` on, `left` of them there
__device__ __forceinline__ void store4(void *y, int dt, int64_t at, int64_t left, const f32x4 &v, bool vec)
{
    if (dt == HIF8_DTYPE_F32) {
        float *p = (float *)y + at;
        if (vec) *(f32x4 *)p = v;
        else
            for (int i = 0; i < 4; ++i)
                if (i < left) p[i] = v[i];
        return;
    }
    const uint2 o = pack16(v, dt);
    uint16_t *p = (uint16_t *)y + at;
    if (vec) *(uint2 *)p = o;
    else
        for (int i = 0; i < 4; ++i)
            if (i < left) p[i] = uint16_t((i & 2 ? o.y : o.x) >> (16 * (i & 1)));
}

// A workgroup of 4 waves, 2 x 2, each W x W tiles of 32 x 32 along the rows of a (the matrix instruction's
// columns) and the rows of b (its rows, so that a lane holds 4 consecutive n of one m).  NST stages of one k
// step each in LDS (W * NST > 4: more than half of a CU's).
template <int FA, int FB, int W, int NST>
__global__ __launch_bounds__(kThreads, W * NST > 4 ? 1 : 2) void k_fp8_gemm(const Args A)
{
    constexpr int T = 64 * W;                    // rows of a and of b
    constexpr uint32_t kStage = 2 * uint32_t(T) * kRowBytes;
    // loads of a wave and stage: 8 rows x 128 bytes each, whole lines (half lines at a time come twice)
    constexpr int L = 2 * W;                     // for either operand
    // two meetings a step: the first frees the stage's part of a half a step before that of b (see the loop)
    constexpr bool kTwo = W >= 4;
    // fragments of a whole step ahead in a second set of registers (see the loop)
    constexpr bool kAhead = NST > 2;
    constexpr int kSets = kAhead ? 2 : 1;
    constexpr int kInFlight = (NST - 2) * 2 * L + (kTwo ? L : 0);
    // scale bytes: 16 of each row (16 k steps) in one of two windows
    constexpr uint32_t kScales = kStage * NST, kWindow = 2 * uint32_t(T) * 16;
    constexpr int LS = (2 * T + 255) / 256;      // loads of a wave and window, 64 rows each
    // The one array of the kernel, so that it begins at LDS address 0: loads into LDS address from there.
    constexpr uint32_t kBias = kScales + 2 * kWindow;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kBias + T * sizeof(float)];
    float *bias = (float *)(smem + kBias);
    ASMV("; lds base %0" ::"v"(uint32_t(uintptr_t(smem))) : "memory");
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t r = lane & 31u, h = lane >> 5;
    const uint32_t wm = (wave & 1u) * (32u * W), wn = (wave >> 1) * (32u * W);

    // ---- the tile and k range
    uint32_t t = blockIdx.x;                     // workgroups go round the 8 XCDs
    if (A.chunked) {
        const uint32_t x = t & 7u, rest = A.items & 7u;
        t = x * (A.items >> 3) + (x < rest ? x : rest) + (t >> 3);
    }
    const int range = int(A.by_tiles(t)), kb = range * A.per, nk = A.nk - kb < A.per ? A.nk - kb : A.per;
    t -= uint32_t(range) * A.by_tiles.d;
    int64_t m0, n0;
    {
        const uint32_t group = A.by_group(t), within = t - group * A.by_group.d;
        const uint32_t n = int(group) < A.full_groups ? within >> A.group_shift : A.by_rest(within);
        const uint32_t m = within - n * (int(group) < A.full_groups ? 1u << A.group_shift : A.by_rest.d);
        m0 = int64_t((group << A.group_shift) + m) * T;
        n0 = int64_t(n) * T;
    }
    const uint32_t k0 = uint32_t(kb) & 3u;       // the first step's byte in its word of scale bytes
    auto resource = [](const uint8_t *p, uint32_t bytes) {
        u32x4 v = {uint32_t(uint64_t(p)), uint32_t(uint64_t(p) >> 32), bytes, 0x00020000u};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_readfirstlane(v[i]);
        return v;
    };
    // codes from k step kb of the tile's first row to its last row's end; scale bytes of the tile's rows
    const uint32_t rows_a = uint32_t(A.M - m0 < T ? A.M - m0 : T), rows_b = uint32_t(A.N - n0 < T ? A.N - n0 : T);
    const uint32_t kofs = uint32_t(kb) * kBK;
    const u32x4 ra = resource(A.a + m0 * A.kp + kofs, rows_a * uint32_t(A.kp) - kofs);
    const u32x4 rb = resource(A.b + n0 * A.kp + kofs, rows_b * uint32_t(A.kp) - kofs);
    const u32x4 rsa = resource(A.sa + m0 * A.S, rows_a * uint32_t(A.S));
    const u32x4 rsb = resource(A.sb + n0 * A.S, rows_b * uint32_t(A.S));

    // ---- loads.  Load i of a wave brings rows (wave * L + i) * 8 .. + 7 of an operand: lane / 8 is the row, and
    // lane % 8 the place in it, whose chunk is the place un-swizzled.
    uint32_t off[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const uint32_t row = (wave * L + i) * 8u + (lane >> 3);
        off[i] = row * uint32_t(A.kp) + (((lane & 7u) ^ swizzle(row)) << 4);
    }
    // load y of the stage of k step k (past the end: nothing is read)
    auto issue = [&](int k, uint32_t slot, int y) {
        const bool of_a = y < L;
        const int i = of_a ? y : y - L;
        u32x4 e = of_a ? ra : rb;
        e[2] = k < nk ? e[2] : 0u;
        load_lds(__builtin_amdgcn_readfirstlane(slot * kStage + (of_a ? 0u : T * kRowBytes) + (wave * L + i) * 1024u),
                 off[i] + uint32_t(k) * kBK, e);
    };
    // Scale bytes: load i of a wave brings 16 bytes of rows (wave * LS + i) * 64 + lane of the 2 T (the waves
    // past them repeat the first).  A row's bytes are far from the next row's, so that a load takes as many
    // requests as rows: once a step they took as long as the codes, hence 16 steps at once.  A window starts at a
    // multiple of 16 blocks from (kb & ~3) on; what it reads past a row's bytes is not used.
    auto issue_scales = [&](uint32_t window) {
#pragma unroll
        for (int i = 0; i < LS; ++i) {
            const uint32_t first = (wave * LS + i) * 64u % uint32_t(2 * T);
            const bool of_a = first < uint32_t(T);
            u32x4 e = of_a ? rsa : rsb;
#pragma unroll
            for (int q = 0; q < 4; ++q) e[q] = __builtin_amdgcn_readfirstlane(e[q]);
            const uint32_t row = (of_a ? first : first - T) + lane;
            load_lds(__builtin_amdgcn_readfirstlane(kScales + (window & 1u) * kWindow + first * 16u),
                     row * uint32_t(A.S) + (uint32_t(kb) & ~3u) + window * 16u, e);
        }
    };
    // ---- fragments, scales, products
    uint32_t xa[kSets][W], xb[kSets][W];         // scale bytes of the lane's rows, in the low byte
    auto read_scale_words = [&](int k, uint32_t (&wa)[W], uint32_t (&wb)[W]) {
        const uint32_t at = uint32_t(k) + k0;
        const uint8_t *ps = smem + kScales + ((at >> 4) & 1u) * kWindow + (at & 12u);
#pragma unroll
        for (int j = 0; j < W; ++j) wa[j] = *(const uint32_t *)(ps + (wm + 32u * j + r) * 16u);
#pragma unroll
        for (int i = 0; i < W; ++i) wb[i] = *(const uint32_t *)(ps + (T + wn + 32u * i + r) * 16u);
    };
    auto shift_scales = [&](int k, const uint32_t (&wa)[W], const uint32_t (&wb)[W], int set) {
        const uint32_t sh = ((uint32_t(k) + k0) & 3u) * 8u;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            xa[set][j] = wa[j] >> sh;
            xb[set][j] = wb[j] >> sh;
        }
    };
    // half p of k: chunks 4 p + 2 h and + 1 of rows wm + 32 j + r; swizzle(row) = swizzle(r)
    uint32_t fo[2][2];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int c = 0; c < 2; ++c) fo[p][c] = r * kRowBytes + (((4u * p + 2u * h + c) ^ swizzle(r)) << 4);
    i32x8 fa[kSets][2][W], fb[kSets][2][W];
    // read x of the 2 W of an operand's half: 16 bytes of a fragment
    auto read = [&](bool of_b, int p, uint32_t slot, int x, int set) {
        const int k = x >> 1, c = x & 1;
        const uint8_t *at = smem + slot * kStage + fo[p][c] + (of_b ? T * kRowBytes + wn * kRowBytes : wm * kRowBytes) + k * (32 * kRowBytes);
        const i32x4 v = *(const i32x4 *)at;
        i32x8 &f = of_b ? fb[set][p][k] : fa[set][p][k];
        f = c == 0 ? __builtin_shufflevector(v, __builtin_shufflevector(f, f, 4, 5, 6, 7), 0, 1, 2, 3, 4, 5, 6, 7)
                   : __builtin_shufflevector(__builtin_shufflevector(f, f, 0, 1, 2, 3), v, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    f32x16 acc[W][W];
    // product x of a phase: 2 x 2 blocks of tiles, so that each fragment feeds two products in a row
    auto multiply = [&](int p, int x, int set) {
        constexpr int B = W % 2 == 0 ? 2 : 1;
        const int q = x / (B * B), e = x % (B * B), bi = q / (W / B), bj = bi % 2 ? W / B - 1 - q % (W / B) : q % (W / B);
        const int i = B * bi + (B == 2 && (e == 1 || e == 2) ? 1 : 0), j = B * bj + (B == 2 && e >= 2 ? 1 : 0);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[set][p][i], fa[set][p][j], acc[i][j], FB, FA, 0,
                                                                  int(xb[set][i]), 0, int(xa[set][j]));
    };

    // the first stage and its scale bytes before all else
#pragma unroll
    for (int y = 0; y < 2 * L; ++y) issue(0, 0, y);
    issue_scales(0);
#pragma unroll
    for (int s = 1; s < NST; ++s)
#pragma unroll
        for (int y = 0; y < 2 * L; ++y) issue(s, s, y);
    issue_scales(1);
    for (int n = tid; n < T; n += kThreads)
        bias[n] = A.bias && A.splits == 1 && n0 + n < A.N ? load_bias(A.bias, A.bias_dt, n0 + n) : 0.0f;
    constexpr int NM = W * W;
    wait_vm<(NST - 1) * 2 * L + LS>();
    wait_lds();
    barrier();
    // the sums start from the bias: acc[i][j], lane (r, h), element 4 q + e: n = 32 i + 8 q + 4 h + e, m = 32 j + r
    // of the wave's part
#pragma unroll
    for (int i = 0; i < W; ++i) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 b = *(const f32x4 *)&bias[wn + 32 * i + 8 * q + 4 * h];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][0][4 * q + e] = b[e];
        }
#pragma unroll
        for (int j = 1; j < W; ++j) acc[i][j] = acc[i][0];
    }
#pragma unroll
    for (int x = 0; x < 2 * W; ++x)
#pragma unroll
        for (int p = 0; p < kSets; ++p) {
            read(true, p, 0, x, 0);
            read(false, p, 0, x, 0);
        }
    {
        uint32_t wa[W], wb[W];
        read_scale_words(0, wa, wb);
        shift_scales(0, wa, wb, 0);
    }
    // Half 0 of a step's k is multiplied while half 1 is read; then the next step's stage has to have arrived
    // (every wave waits for its own loads, the barrier for all), the stage of this step is free and takes the
    // loads of NST steps on, and half 1 is multiplied while the next half 0 is read.  With kTwo the waves meet
    // once more, when the fragments of a have been read: the loads of a then fall into the first phase and
    // those of b into the second (all in the second: 3.7 against 2.5 thousand cycles a step, since what
    // arrives keeps LDS from the reads).  Reads and loads lie in the gaps between the products, whose order
    // is held.  No branch lies among the products, behind which the compiler would gather them: a window of
    // scale bytes at a time.
    // kAhead: a whole step's fragments are read behind the products of the one before, since half a step of a small
    // tile is too short for it, and the waves meet once a step, when those have come and the next stage has arrived
    // (512 x 5120 x 5120 23.7 -> 21.7 us, 2048 x 2048 x 2048 13.3 -> 12.5; a step of 128 x 128 is 0.45 us then, its LDS
    // traffic alone 0.37).  With two stages that leaves their loads less time: 4680 x 1536 x 8960 66 -> 73.
    uint32_t slot = 0;
    int k = 0;
    auto step_ahead = [&](auto tag) {
        constexpr int cur = decltype(tag)::value, next = (cur + 1) % kSets;
        wait_lds();
        wait_vm<kInFlight>();
        barrier();
        const uint32_t freed = slot;
        slot = slot + 1 == NST ? 0 : slot + 1;
        uint32_t wa[W], wb[W];
#pragma unroll
        for (int x = 0; x < 2 * NM; ++x) {
            multiply(x / NM, x % NM, cur);
            if (x == 0) read_scale_words(k + 1, wa, wb);
#pragma unroll
            for (int y = 0; y < 8 * W; ++y)
                if (y * NM / (4 * W) == x) read(y / 2 % 2, y / (4 * W), slot, y / 4 % W * 2 + y % 2, next);
#pragma unroll
            for (int y = 0; y < 2 * L; ++y)
                if (y * NM / L == x) issue(k + NST, freed, y);
            __builtin_amdgcn_sched_barrier(0);
        }
        shift_scales(k + 1, wa, wb, next);
        ++k;
    };
    while (k < nk) {
        const int stop = (k + int(k0)) / 16 * 16 + 16 - int(k0), end = stop < nk ? stop : nk;
        if constexpr (kAhead) {
            while (k + 1 < end) {
                step_ahead(Type<0>{});
                step_ahead(Type<1>{});
            }
            if (k < end) {
                step_ahead(Type<0>{});
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    xa[0][j] = xa[kSets - 1][j], xb[0][j] = xb[kSets - 1][j];
#pragma unroll
                    for (int p = 0; p < 2; ++p) fa[0][p][j] = fa[kSets - 1][p][j], fb[0][p][j] = fb[kSets - 1][p][j];
                }
            }
        }
        for (; !kAhead && k < end; ++k) {
#pragma unroll
            for (int x = 0; x < NM; ++x) {
                multiply(0, x, 0);
                if (kTwo) {
                    if (x < 5) {             // 8 reads in 5 gaps
#pragma unroll
                        for (int y = 0; y < 2 * W; ++y)
                            if (y * 5 / (2 * W) == x) read(false, 1, slot, y, 0);
                    }
                    if (x == 5) {
                        wait_lds();
                        barrier();
                    }
                    if (x > 5) {             // 8 reads in 8, 8 loads in 9
#pragma unroll
                        for (int y = 0; y < 2 * W; ++y)
                            if (6 + y * 8 / (2 * W) == x) read(true, 1, slot, y, 0);
#pragma unroll
                        for (int y = 0; y < L; ++y)
                            if (6 + y * 9 / L == x) issue(k + NST, slot, y);
                    }
                } else {
#pragma unroll
                    for (int y = 0; y < 2 * W; ++y)
                        if (y * NM / (2 * W) == x) {
                            read(true, 1, slot, y, 0);
                            read(false, 1, slot, y, 0);
                        }
                }
                if (x == NM - 1) {
                    wait_lds();
                    wait_vm<kInFlight>();
                    barrier();
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            const uint32_t freed = slot;
            slot = slot + 1 == NST ? 0 : slot + 1;
            uint32_t wa[W], wb[W];
#pragma unroll
            for (int x = 0; x < NM; ++x) {
                multiply(1, x, 0);
                if (x == 0) read_scale_words(k + 1, wa, wb);
#pragma unroll
                for (int y = 0; y < 2 * W; ++y)
                    if (y * NM / (2 * W) == x) {
                        read(true, 0, slot, y, 0);
                        read(false, 0, slot, y, 0);
                    }
#pragma unroll
                for (int y = kTwo ? L : 0; y < 2 * L; ++y)
                    if (kTwo ? (y - L) * NM / L == x : y * NM / (2 * L) == x) issue(k + NST, freed, y);
                __builtin_amdgcn_sched_barrier(0);
            }
            shift_scales(k + 1, wa, wb, 0);
        }
        // the window just left takes the one after the next: these loads only make the waits for others
        // stricter (every wave has read its last scale bytes there before the last barrier)
        issue_scales(((uint32_t(k) + k0) >> 4) + 1u);
    }
    wait_lds();
    wait_vm<0>();        // no load may still write to LDS
    barrier();           // the stages are free

    // 32 rows of the wave's part at a time go through its part of LDS (two in turn), so that 16 lanes (fp32: 32)
    // store 16 bytes each of one row.  (Straight from the accumulators the lanes of a store lie in 32 rows, one
    // request each.)
    const bool split = A.splits > 1;
    uint8_t *out = split ? (uint8_t *)(A.part + int64_t(range) * A.M * A.N) : (uint8_t *)A.y;
    auto write_out = [&](auto tag) {
        constexpr int dt = decltype(tag)::value;
        constexpr uint32_t kSize = dt == HIF8_DTYPE_F32 ? 4 : 2, kLanes = 32 * W * kSize / 16, kRows = 64 / kLanes;
        constexpr uint32_t kPitch = 32 * W * kSize + 16, kPart = 32 * kPitch;
        static_assert(4 * 2 * kPart <= kBias, "the outputs fit");
        const uint32_t row_bytes = uint32_t(A.N) * kSize;
        uint8_t *to = out + m0 * int64_t(row_bytes);
        const bool vec = row_bytes % 16 == 0;
        // stores past the tile's last row, or sent past it, are dropped
        const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(to, 0, rows_a * row_bytes, 0x00020000);
        const uint32_t lrow = lane / kLanes, lcol = lane % kLanes * (16 / kSize);
        const int64_t n = n0 + wn + lcol;
        uint32_t at = n < A.N ? (wm + lrow) * row_bytes + uint32_t(n) * kSize : 0x80000000u;
        uint8_t *part = smem + wave * (2 * kPart), *put = part + r * kPitch + 4 * h * kSize, *get = part + lrow * kPitch + lcol * kSize;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            // out of the matrix cores' registers now, not all at once ahead
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if constexpr (W >= 4) ASMV("" : "+a"(acc[i][j]));
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
                    uint8_t *p = put + (j % 2) * kPart + (32 * i + 8 * q) * kSize;
                    if constexpr (kSize == 4) *(f32x4 *)p = v;
                    else *(uint2 *)p = pack16(v, dt);
                }
            }
            if (vec) {
                u32x4 v[32 / kRows];
#pragma unroll
                for (uint32_t x = 0; x < 32 / kRows; ++x) v[x] = *(const u32x4 *)(get + (j % 2) * kPart + x * kRows * kPitch);
#pragma unroll
                for (uint32_t x = 0; x < 32 / kRows; ++x) {
                    // non-temporal: the bursts of stores, all CUs at once, go by the L2 (3-7 %)
                    __builtin_amdgcn_raw_buffer_store_b128(v[x], ro, at, 0, 2);
                    at += kRows * row_bytes;
                }
            } else {       // rows that are no multiple of 16 bytes: single values
#pragma unroll 1
                for (uint32_t x = 0; x < 32 / kRows; ++x) {
                    const uint8_t *v = get + (j % 2) * kPart + x * kRows * kPitch;
                    const uint32_t m = wm + 32 * j + x * kRows + lrow;
                    uint8_t *p = to + m * int64_t(row_bytes) + n * kSize;
#pragma unroll 1
                    for (uint32_t e = 0; e < 16 / kSize; ++e)
                        if (m < rows_a && n + e < A.N) {
                            if constexpr (kSize == 4) ((uint32_t *)p)[e] = ((const uint32_t *)v)[e];
                            else ((uint16_t *)p)[e] = ((const uint16_t *)v)[e];
                        }
                }
            }
        }
    };
    if (split || A.y_dt == HIF8_DTYPE_F32) write_out(Type<HIF8_DTYPE_F32>{});
    else if (A.y_dt == HIF8_DTYPE_F16) write_out(Type<HIF8_DTYPE_F16>{});
    else write_out(Type<HIF8_DTYPE_BF16>{});
}

// y = the sum of the k ranges' partial sums in order, plus the bias.
__global__ __launch_bounds__(256) void k_fp8_reduce(const Args A)
{
    const int64_t total = A.M * A.N;
    for (int64_t at = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4; at < total; at += int64_t(gridDim.x) * 1024) {
        const bool vec = A.N % 4 == 0;
        f32x4 v = {};
        for (int s = 0; s < A.splits; ++s) {
            const float *p = A.part + int64_t(s) * total + at;
            if (vec) v += *(const f32x4 *)p;
            else
                for (int e = 0; e < 4; ++e)
                    if (at + e < total) v[e] += p[e];
        }
        if (A.bias)
            for (int e = 0; e < 4; ++e)
                if (at + e < total) v[e] += load_bias(A.bias, A.bias_dt, (at + e) % A.N);
        store4(A.y, A.y_dt, at, total - at, v, vec);
    }
}

enum Plan { kBig, kMid, kDeep, kSmall };      // kDeep: kMid with three stages, one workgroup a CU
struct Choice {
    Plan plan;
    int tile, splits;
};
// The plan that takes the least time by what the tiles were measured to take: a step of 128 k and the rest of a
// tile in microseconds, with one workgroup a CU and with as many as fit (256 CUs), and for k ranges a launch, a read
// after the other of each range's sums and 8 bytes of memory traffic a partial sum.  Each tile size has its place (M x
// N x K, microseconds with tiles of 256 / 128 / 64): 5120 x 5120 x 8192 191 / 215 / 333, 4680 x 1536 x 8960 87 / 63 /
// 105, 128 x 5120 x 5120 50 / 19 / 13; and so have ranges: 1536 x 1536 x 32760 in 7 of 256-wide tiles 84, unsplit 285;
// 16 x 1536 x 8960 in 7 of 64 11, in 14 15, unsplit 18; but 16 x 13824 x 5120 in 2 of 64 17, unsplit 14, and 128 x 5120 x
// 5120 in 3 15.  A 128-wide tile alone on its CU waits for its loads with two stages: with three 512 x 5120 x 5120 takes
// 21, with two 32; where two tiles fit a CU each fills the other's waits, and 4680 x 1536 x 8960 takes 63 with two
// stages and 69 with three.  Four are no better than three.  Over 130 products of 1 to 8960 rows the plan taken is within
// 10 % of the best of all plans, 0.5 % on average.
Choice choose(int64_t M, int64_t N, int64_t nk)
{
    struct Tile {
        Plan plan;
        int size, room;       // workgroups that run at once
        double step, full_step, rest;
    };
    constexpr Tile kinds[] = {{kBig, 256, 256, 1.15, 1.15, 7.0}, {kMid, 128, 512, 0.8, 0.95, 3.0}, {kDeep, 128, 256, 0.46, 0.46, 3.0},
                              {kSmall, 64, 512, 0.22, 0.48, 2.0}};
    Choice best{kBig, 256, 1};
    double least = 1e300;
    for (const Tile &t : kinds) {
        const int64_t tiles = ((M + t.size - 1) / t.size) * ((N + t.size - 1) / t.size);
        for (int64_t s = 1; s <= 16 && (s == 1 || (nk >= 4 * s && tiles * s <= t.room)); ++s) {
            const int64_t steps = (nk + s - 1) / s, rounds = (tiles * s + t.room - 1) / t.room;
            double us = double(rounds) * (double(steps) * (tiles * s <= 256 ? t.step : t.full_step) + t.rest);
            if (s > 1) us = 1.05 * (us + 3.5 + double(s) * (0.25 + double(M) * double(N) * 8.0 / 4e6));
            if (us < least) {
                least = us;
                best = Choice{t.plan, t.size, int(s)};
            }
        }
    }
    return best;
}

template <int FA, int FB, int W, int NST> void launch(const Args &A, hipStream_t st)
{
    k_fp8_gemm<FA, FB, W, NST><<<A.items, kThreads, 0, st>>>(A);
}
template <int FA, int FB> void launch_plan(Plan p, const Args &A, hipStream_t st)
{
    if (p == kBig) launch<FA, FB, 4, 2>(A, st);
    else if (p == kMid) launch<FA, FB, 2, 2>(A, st);
    else if (p == kDeep) launch<FA, FB, 2, 3>(A, st);
    else launch<FA, FB, 1, 4>(A, st);
}

bool float_dtype(int dt) { return dt == HIF8_DTYPE_BF16 || dt == HIF8_DTYPE_F32 || dt == HIF8_DTYPE_F16; }

}  // namespace
}  // namespace fp8
}  // namespace hif8

using namespace hif8;

extern "C" {

int64_t hif8_fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K)
{
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const fp8::Choice c = fp8::choose(M, N, fp8::blocks_of(K));
    return c.splits > 1 ? c.splits * M * N * 4 : 0;
}

int hif8_fp8_gemm(const uint8_t *a, const uint8_t *a_scales, int a_format, const uint8_t *b, const uint8_t *b_scales,
                  int b_format, const void *bias, int bias_dtype, void *y, int y_dtype, int64_t M, int64_t N, int64_t K,
                  void *workspace, int64_t workspace_bytes, hif8_stream_t stream)
{
    if (!a || !a_scales || !b || !b_scales || !y || M <= 0 || N <= 0 || K <= 0) return HIF8_ERR_ARG;
    if ((a_format != HIF8_FP8_E4M3 && a_format != HIF8_FP8_E5M2) || (b_format != HIF8_FP8_E4M3 && b_format != HIF8_FP8_E5M2))
        return HIF8_ERR_ARG;
    if (!fp8::float_dtype(y_dtype) || (bias && !fp8::float_dtype(bias_dtype))) return HIF8_ERR_ARG;
    // 256 rows of codes and of outputs in 32-bit offsets
    if (K > (int64_t(1) << 23) || M > (int64_t(1) << 31) || N > (int64_t(1) << 21)) return HIF8_ERR_SHAPE;
    if ((uint64_t(a) | uint64_t(b) | uint64_t(y) | uint64_t(workspace)) % 16 || (uint64_t(a_scales) | uint64_t(b_scales)) % 4 ||
        (bias && uint64_t(bias) % (bias_dtype == HIF8_DTYPE_F32 ? 4 : 2)))
        return HIF8_ERR_ALIGN;
    const int64_t nk = fp8::blocks_of(K);
    const fp8::Choice c = fp8::choose(M, N, nk);
    if (c.splits > 1 && (!workspace || workspace_bytes < hif8_fp8_gemm_workspace_bytes(M, N, K))) return HIF8_ERR_ARG;
    fp8::Args A{};
    A.a = a, A.sa = a_scales, A.b = b, A.sb = b_scales, A.bias = bias, A.y = y, A.part = (float *)workspace;
    A.M = M, A.N = N, A.kp = int(nk * 128), A.S = int(fp8::scale_row(K)), A.nk = int(nk);
    const int64_t tiles_m = (M + c.tile - 1) / c.tile, tiles_n = (N + c.tile - 1) / c.tile;
    if (tiles_m * tiles_n >= int64_t(1) << 24) return HIF8_ERR_SHAPE;      // a grid has less than 2^32 threads
    A.per = int((nk + c.splits - 1) / c.splits);
    A.splits = int((nk + A.per - 1) / A.per);       // 65 steps in 16 ranges of 5 are 13
    A.by_tiles.set(uint32_t(tiles_m * tiles_n));
    A.items = uint32_t(tiles_m * tiles_n * A.splits);
    // Microseconds chunked / not: 1536 x 1536 x 32760 in 7 ranges 85 / 103, 700 x 8960 x 1536 14 / 18, 512 x 5120 x
    // 5120 22 / 24 (with two meetings a step); but with the many rows of a large grid, whose groups every eighth item covers evenly,
    // 32760 x 8960 x 1536 474 / 441, 8960 x 1536 x 32760 440 / 414.
    A.chunked = A.splits > 1 || tiles_m <= 8;
    // Microseconds in groups of 16 / 32 / 64 / 128 rows of tiles.  54 columns of them, 75600 x 13824 x 5120: 4152 / 4100 /
    // 4080 / 4144; 35, 32760 x 8960 x 1536: 421 / 415 / 415 / 429; 20, 13824 x 5120 x 32760: 2022 / 1884 / 2096 / 2095;
    // 6, 8960 x 1536 x 32760: 361 / 358 / 423 / 422.
    A.group_shift = tiles_n >= 32 ? 6 : 5;
    A.full_groups = int(tiles_m >> A.group_shift);
    A.by_group.set(uint32_t(tiles_n << A.group_shift));
    A.by_rest.set(uint32_t(tiles_m - (int64_t(A.full_groups) << A.group_shift) + (tiles_m % (1 << A.group_shift) == 0)));
    A.bias_dt = bias_dtype, A.y_dt = y_dtype;
    hipStream_t st = (hipStream_t)stream;
    if (a_format == HIF8_FP8_E4M3)
        b_format == HIF8_FP8_E4M3 ? fp8::launch_plan<0, 0>(c.plan, A, st) : fp8::launch_plan<0, 1>(c.plan, A, st);
    else
        b_format == HIF8_FP8_E4M3 ? fp8::launch_plan<1, 0>(c.plan, A, st) : fp8::launch_plan<1, 1>(c.plan, A, st);
    if (A.splits > 1) {
        const int64_t want = (M * N + 1023) / 1024;
        fp8::k_fp8_reduce<<<uint32_t(want < 8192 ? want : 8192), 256, 0, st>>>(A);
    }
    return hipGetLastError() == hipSuccess ? HIF8_OK : HIF8_ERR_HIP;
}

}  // extern "C"
