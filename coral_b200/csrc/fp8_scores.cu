// Rows in 8-bit floating point, and dense scores of such rows on the tcgen05 tensor cores.
//
// A row keeps its columns as e4m3 codes with one power-of-two scale (e8m0: a byte, 2^(byte - 127))
// for each block of 128 columns: x ~ code * 2^e, e the least integer with max|x| <= 448 * 2^e.  A
// power of two costs nothing against a free scale: the codes are floating point, so their relative
// rounding (half a step, 2^-4) does not depend on where in the range a block sits, and scaling by
// 2^e is exact.  It is also the scale the tensor cores apply themselves
// (tcgen05.mma kind::mxf8f6f4.block_scale), so the accumulator needs no correction between blocks.
#include <cuda.h>

#include <mutex>
#include <type_traits>

#include "scores.cuh"

namespace coral {

namespace {

// ------------------------------------------------------------------------------- compression

// Least e in [-127, 127] with amax <= 448 * 2^e, 448 = 1.75 * 2^8, from the bits of amax: the
// exponent less 8, one more when the mantissa is above 1.75.  A subnormal or zero amax ends at -127.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -127 ? -127 : e;
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}

constexpr int kQuantThreads = 256;
constexpr int kQuantLoads = 8;    // 16-byte loads a lane has in flight

// The larger magnitude, lane by lane of 16 bytes; NaN counts as nothing.
template <typename T>
__device__ __forceinline__ float abs_max(uint4 v);
template <>
__device__ __forceinline__ float abs_max<float>(uint4 v) {
    return fmaxf(fmaxf(fabsf(__uint_as_float(v.x)), fabsf(__uint_as_float(v.y))),
                 fmaxf(fabsf(__uint_as_float(v.z)), fabsf(__uint_as_float(v.w))));
}
template <>
__device__ __forceinline__ float abs_max<__nv_bfloat16>(uint4 v) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(__habs2(p[0]), __habs2(p[1])), __hmax2(__habs2(p[2]), __habs2(p[3]))));
    return fmaxf(m.x, m.y);
}
template <>
__device__ __forceinline__ float abs_max<__half>(uint4 v) {
    const __half2* p = reinterpret_cast<const __half2*>(&v);
    const float2 m = __half22float2(__hmax2(__hmax2(__habs2(p[0]), __habs2(p[1])), __hmax2(__habs2(p[2]), __habs2(p[3]))));
    return fmaxf(m.x, m.y);
}

// What is not finite counts as nothing in a block's maximum and its code is NaN (e4m3 has no infinity):
// it shows in every score of its row and costs the rest of its block no precision.  A NaN takes this
// course by itself; a block whose maximum came out infinite or NaN is put right here, in the registers of
// its eight lanes.
template <typename T, int J>
__device__ __forceinline__ float drop_infinities(uint4 (&v)[J]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (sizeof(T) == 4) {
                if ((w[i] & 0x7fffffffu) == 0x7f800000u) w[i] = 0x7fffffffu;
            } else {
                const uint32_t inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
                if ((w[i] & 0x7fffu) == inf) w[i] |= 0x7fffu;
                if ((w[i] >> 16 & 0x7fffu) == inf) w[i] |= 0x7fff0000u;
            }
        }
        m = fmaxf(m, abs_max<T>(v[j]));
    }
    return m;
}

// A block of 128 columns belongs to G lanes, 16 columns each, in J loads of 16 bytes that the G lanes make
// of consecutive bytes; its maximum takes log2 G shuffles.  G is 8, or fewer for rows of one block of
// at most 64, 32 or 16 columns, which would leave the other lanes idle (800k x 14 bf16: 52 us with
// eight, 11 with one).  A warp takes kQuantLoads / J steps of 32 / G consecutive blocks, all loads before the first
// use, and writes the scales together.  Bound by memory: 1M x 512 fp32 takes 369 us, 2.56 GB at
// 6.95 TB/s; 100003 x 200 bf16, cut from rows of 256, 15 us, 61 MB at 4.0 TB/s.  (A block
// to a whole warp or half of one is bound by instructions instead, 435 and 22 us: the few values a
// lane then has carry the same addresses, bounds and exponents.)
template <typename T, bool VEC, int G>
__global__ void __launch_bounds__(kQuantThreads)
fp8_quantize_kernel(const T* __restrict__ x, int64_t rows, int dim, int64_t ld, uint8_t* __restrict__ codes,
                    uint8_t* __restrict__ scales, uint32_t inv_per_row) {
    constexpr int E = 16 / (int)sizeof(T), J = 16 / E, S = kQuantLoads / J, P = 32 / G, N = P * S;
    const int lane = threadIdx.x & 31, in_block = lane % G * E;
    const int per_row = (dim + kFp8Block - 1) / kFp8Block;
    const int code_pitch = (dim + 15) / 16 * 16, scale_pitch = (dim + 511) / 512 * 4;
    const int64_t total = rows * per_row;
    const int64_t first = ((int64_t)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5)) * N;
    if (first >= total) return;
    const int64_t row0 = total <= 0x7fffffff ? (int64_t)((uint32_t)first / (uint32_t)per_row) : first / per_row;
    const int b0 = (int)(first - row0 * per_row);
    const int left = (int)(total - first < N ? total - first : N);      // blocks of this warp
    const auto place = [&](int i, int64_t& row, int& b) {               // block first + i
        const int at = b0 + i, over = per_row == 1 ? at : (int)__umulhi((uint32_t)at, inv_per_row);
        row = row0 + over;
        b = at - over * per_row;
    };
    uint4 v[S][J];
#pragma unroll
    for (int u = 0; u < S; ++u) {
        const int i = u * P + lane / G;
        int64_t row;
        int b;
        place(i, row, b);
        const int c = b * kFp8Block + in_block;
        const T* from = x + row * ld + c;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int cols = dim - c - j * G * E;      // of the row from here on
            v[u][j] = make_uint4(0u, 0u, 0u, 0u);
            if (i < left && cols > 0) {
                if (VEC && cols >= E) {
                    v[u][j] = __ldcs(reinterpret_cast<const uint4*>(from + j * G * E));
                } else {
                    T* w = reinterpret_cast<T*>(&v[u][j]);
#pragma unroll
                    for (int k = 0; k < E; ++k)
                        if (k < cols) w[k] = from[j * G * E + k];
                }
            }
        }
    }
    int mine = 0;      // the exponent of block first + lane
#pragma unroll
    for (int u = 0; u < S; ++u) {
        const int i = u * P + lane / G;
        int64_t row;
        int b;
        place(i, row, b);
        float m = abs_max<T>(v[u][0]);
#pragma unroll
        for (int j = 1; j < J; ++j) m = fmaxf(m, abs_max<T>(v[u][j]));
        bool again = false;
        do {
#pragma unroll
            for (int o = 1; o < G; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            again = !again && __any_sync(0xffffffffu, !(m < __uint_as_float(0x7f800000u)));
            if (again) m = drop_infinities<T, J>(v[u]);
        } while (again);
        const int e = scale_exponent(__float_as_uint(m));
        const float f = __uint_as_float((uint32_t)(127 - e) << 23);     // 2^-e: e in [-127, 120], 2^-e never subnormal
        if constexpr (P <= 8) {      // a lane's own block's, of up to 32 blocks a warp
            const int got = __shfl_sync(0xffffffffu, e, lane % P * G);
            if (lane / P == u) mine = got;
        } else if (i < left && lane % G == 0) {
            *reinterpret_cast<uint32_t*>(scales + row * 4) = (uint32_t)(e + 127);      // one block a row
        }
        uint8_t* to = codes + row * code_pitch + b * kFp8Block + in_block;
        const int codes_left = i < left ? code_pitch - b * kFp8Block - in_block : 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const T* w = reinterpret_cast<const T*>(&v[u][j]);
            uint32_t q[E / 4];
#pragma unroll
            for (int k = 0; k < E; k += 4)
                q[k / 4] = pack_e4m3(to_f32<T>(w[k]) * f, to_f32<T>(w[k + 1]) * f, to_f32<T>(w[k + 2]) * f, to_f32<T>(w[k + 3]) * f);
            if (codes_left > j * G * E) {
                if (E == 4)
                    *reinterpret_cast<uint32_t*>(to + j * G * E) = q[0];
                else
                    *reinterpret_cast<uint2*>(to + j * G * E) = make_uint2(q[0], q[E / 4 - 1]);
            }
        }
    }
    if (P <= 8 && lane < left) {
        int64_t row;
        int b;
        place(lane, row, b);
        uint8_t* s = scales + row * scale_pitch + b;
        *s = (uint8_t)(mine + 127);
        if (b == per_row - 1)      // the scales that pad the row to a multiple of four
            for (int i = 1; b + i < scale_pitch; ++i) s[i] = 0;
    }
}

template <typename T, int G>
cudaError_t quantize_g(const void* x, int64_t rows, int dim, int64_t ld, uint8_t* codes, uint8_t* scales,
                       cudaStream_t stream) {
    const uint32_t per_row = (uint32_t)((dim + kFp8Block - 1) / kFp8Block);
    const int per_cta = kQuantThreads / G * kQuantLoads / (int)sizeof(T);
    const int64_t ctas = (rows * per_row + per_cta - 1) / per_cta;
    const bool vec = ((uintptr_t)x | (uintptr_t)(ld * sizeof(T))) % 16 == 0;
    auto kernel = vec ? fp8_quantize_kernel<T, true, G> : fp8_quantize_kernel<T, false, G>;
    kernel<<<(unsigned)ctas, kQuantThreads, 0, stream>>>(static_cast<const T*>(x), rows, dim, ld, codes, scales,
                                                    per_row == 1 ? 0u : (uint32_t)((0x100000000ull + per_row - 1) / per_row));
    return cudaGetLastError();
}

template <typename T>
cudaError_t quantize_t(const void* x, int64_t rows, int dim, int64_t ld, uint8_t* codes, uint8_t* scales,
                       cudaStream_t stream) {
    if (dim <= 16) return quantize_g<T, 1>(x, rows, dim, ld, codes, scales, stream);
    if (dim <= 32) return quantize_g<T, 2>(x, rows, dim, ld, codes, scales, stream);
    if (dim <= 64) return quantize_g<T, 4>(x, rows, dim, ld, codes, scales, stream);
    return quantize_g<T, 8>(x, rows, dim, ld, codes, scales, stream);
}

// ----------------------------------------------------------------------------------- product
//
// out[q][j] = alpha * sum_b 2^(eq_b + ej_b) * (codes of q, codes of j)_b + bias[j], accumulated in
// fp32 in tensor memory.  One persistent CTA of 12 warps per SM, tiles of 128 queries x 256 rows:
//   warp 0     one lane issues the tiles' TMA loads (128-byte swizzle, 128 columns a stage).  A query
//              tile of no more k-blocks than stages is kept while the next row tile meets it too: with few
//              k-blocks the tensor copies, which take their time per row, are what a tile waits for;
//   warp 1     one lane issues, per stage, four tcgen05.mma (M = 128, N = 256, K = 32) and, per four
//              stages, three tcgen05.cp (their scales to tensor memory);
//   warp 2     brings scales to a shared-memory ring of their own in the layout tcgen05.cp takes, with
//              asynchronous 4-byte copies, six groups of four stages ahead: with rows of one or two
//              stages the latency of a scale would otherwise be the time of a tile;
//   warps 4-11 read the finished accumulator (two warps to a quarter of its rows, turn by turn),
//              apply alpha and bias, and store: pieces of 32 rows x 128 bytes through shared memory
//              (128-byte swizzle) and TMA, two in flight a warp, or, where the output's rows do not
//              start at 16-byte boundaries, by coalesced plain stores.
// A scale word of four bytes covers 512 columns; an instruction's K = 32 lies inside one block, so
// all four instructions of a stage name the same byte of the word (the scale ids of the instruction
// descriptor), byte (k-block mod 4).
//
// What bounds it: the base's bytes with not too many queries (64 x 1M x 512 with its 256 MB of scores:
// 129 us, 6.0 TB/s); memory with many queries and short rows (4001 x 100003 x 256 bf16: 194 us, 800 MB
// written at 4.1 TB/s), and the load side where rows of codes lie an odd multiple of 16 bytes apart and
// every other one starts inside a 32-byte sector (200 columns: 243 us, 226 with rows 224 bytes apart; 192
// columns: 205); with many and long rows
// shared memory: a stage's 48 KB arrive in 384 cycles and are read in another 384, against 512 cycles
// of products (4096 x 8192 x 4096: 116 to 120 us alone, 2.3 to 2.4 PFLOP/s; 138 us under a power cap).  Pairs of SMs
// on one tile would halve the row tile's share of that; not built.
//
// Tensor memory: two accumulators of 256 columns that share 64 (0-255 and 192-447) and, from 448,
// four slots of 16 columns of scales.  A slot is written again four groups, so at least four stages,
// later; that stage's codes have landed, so the products of the stage S <= 4 before it are done, and
// with them the slot's old ones.  The epilogue reads the shared columns first and then
// lets the next tile's products start.

constexpr int kTileM = 128, kTileN = 256, kTileK = 128;
constexpr int kABytes = kTileM * kTileK, kBBytes = kTileN * kTileK;
constexpr int kScaleBytes = (kTileM + kTileN) * 4;
constexpr int kAccStep = 192, kShared = 64, kTmemScales = 448;
constexpr int kScaleSlots = 8, kScalesAhead = 6;                    // groups in the ring, and in flight
constexpr int kEpiWarps = 8;
// Shared memory of a kernel with S stages: three leave every epilogue warp two pieces of output in
// flight; the split kernel, which stores otherwise, has four.
template <int S>
struct Layout {
    static constexpr int kOffB = S * kABytes;                       // query tiles first, then row tiles
    static constexpr int kOffScales = S * (kABytes + kBBytes);
    static constexpr int kOffOut = kOffScales + kScaleSlots * kScaleBytes;
    static constexpr int kOutBytes = S == 3 ? kEpiWarps * 2 * 4096 : 0;
    static constexpr int kOffBias = kOffOut + kOutBytes;            // each warp the biases of its columns
    static constexpr int kOffBars = kOffBias + kEpiWarps * (kTileN / 2) * 4;
    static constexpr int kBytes = kOffBars + 256 + 1024;
    static_assert(S <= 4, "scale slots in tensor memory");
    static_assert(kOffOut % 1024 == 0, "swizzled staging");
    static_assert(kBytes <= 232448, "shared memory");
};
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int64_t kChunkBytes = 32ll << 20;      // base bytes per chunk of tiles: a quarter of L2

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t mbar_test_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok;
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok;
}
// Bounded wait for a phase that a test has not found over: gives up when `limit` clocks have gone by (0: at
// once; try_wait would itself wait for a while) or another role of the CTA gave up.
__device__ __forceinline__ bool mbar_wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, long long limit) {
    const long long t0 = clock64();
    for (uint32_t spins = 1; limit != 0; ++spins) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spins & 15u) == 0u) {
            if (*abort_flag) return false;
            if (clock64() - t0 > limit) break;
        }
    }
    *abort_flag = 1;
    *static_cast<volatile int*>(err) = 1;
    __threadfence_system();
    return false;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const Fp8ScoresArgs& a) {
    return mbar_test_wait(bar, parity) || mbar_wait_on(bar, parity, abort_flag, a.err, a.wait_clocks);
}
// The same with the loop out of line, for the kernel of few queries (1 x 4M x 128: 83.2 us, 84.0 with it inline;
// the query tiles lose by it: 4096 x 8192 x 4096 119.8 us for 117.6).
__device__ __noinline__ bool mbar_wait_apart(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, long long limit) {
    return mbar_wait_on(bar, parity, abort_flag, err, limit);
}
__device__ __forceinline__ bool mbar_wait_few(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const Fp8ScoresArgs& a) {
    return mbar_test_wait(bar, parity) || mbar_wait_apart(bar, parity, abort_flag, a.err, a.wait_clocks);
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar))
        : "memory");
}
// Issued by the leader lane of a converged warp.  Written once and not read here: the output leaves L2
// to the base.
__device__ __forceinline__ void tma_store_2d(uint32_t leads, const CUtensorMap* map, int c0, int c1, const void* src,
                                             uint64_t policy) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%1, %2}], [%3], %4;\n\t"
        "@q cp.async.bulk.commit_group;\n\t}" ::"l"(map), "r"(c0), "r"(c1), "r"(smem_u32(src)), "l"(policy), "r"(leads)
        : "memory");
}
// Shared-memory matrix descriptor, K-major rows of 128 bytes with the 128-byte swizzle: 8-row groups
// 1024 bytes apart, descriptor version 1, layout type 2.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The same for 32 unswizzled rows of 16 bytes (scales): 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t desc_rows16(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
// Instruction descriptor of kind::mxf8f6f4: e4m3 x e4m3 (type 0), both K-major, e8m0 scales (bit 23),
// N / 8 from bit 17, M / 128 from bit 27; the scale ids (A from bit 29, B from bit 4) are or-ed in.
constexpr uint32_t kInstrDesc = (1u << 23) | ((uint32_t)(kTileN >> 3) << 17) | ((uint32_t)(kTileM >> 7) << 27);

// The issuing warp runs converged, with every operand the same in all lanes (so that operands stay in
// uniform registers: moving them there from one diverged lane costs more than the product lasts), and
// its leader lane issues.
__device__ __forceinline__ uint32_t elect_leader() {
    uint32_t leads;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(leads));
    return leads;
}
__device__ __forceinline__ void umma_mxf8(uint32_t leads, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b,
                                          uint32_t idesc, uint32_t tmem_sa, uint32_t tmem_sb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate), "r"(leads)
        : "memory");
}
// 32 rows of 16 bytes to 4 columns of tensor memory, the same in each of the four lane groups.
__device__ __forceinline__ void scales_to_tmem(uint32_t leads, uint32_t taddr, uint64_t desc) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(leads)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t leads, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(leads)
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<float>(float lo, float) { return __float_as_uint(lo); }

// The order of the tiles: the base in chunks of `chunk_n` row tiles that stay in L2, per chunk all query
// tiles, per query tile the chunk's row tiles.  Neighbouring CTAs then write neighbouring pieces of the
// same output rows, which DRAM takes faster than the same bytes scattered over many rows (4001 x 100003
// x 128 bf16: 203 us, 254 with query tiles first; without the evict-first stores 233 and 277).
struct TileOrder {
    uint32_t tiles, tiles_m, tiles_n, chunk_n;
    __device__ __forceinline__ void at(uint32_t t, int64_t& m0, int64_t& n0) const {
        const uint32_t c = t / (chunk_n * tiles_m), left = tiles_n - c * chunk_n;
        const uint32_t width = left < chunk_n ? left : chunk_n, in_chunk = t - c * chunk_n * tiles_m;
        const uint32_t m = in_chunk / width;
        m0 = (int64_t)m * kTileM;
        n0 = (int64_t)(c * chunk_n + in_chunk - m * width) * kTileN;
    }
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 load_peer(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// How a CTA stores its scores.
constexpr int kPlain = 0;      // coalesced plain stores
constexpr int kTma = 1;        // tensor stores
constexpr int kTmaOdd = 2;     // the same, and the columns after a row's last whole 16 bytes plainly (apart
                               // from kTma: the few instructions cost 33 x 2M x 100 fp32 93 -> 102 us)
constexpr int kSplit = 3;      // the tile's k-blocks are split over the CTAs of a cluster, see below

// With fewer tiles than SMs and many k-blocks, a cluster of 2, 4 or 8 CTAs shares a tile: rank r takes a
// range of its k-blocks (whole groups of four).  Then every CTA lays its partial accumulator out in its
// stages' memory, and rank p adds, over distributed shared memory and in rank order, the parts of the
// columns it owns and stores them.  The same additions in every run.  (Reading a row's 16-byte pieces
// side by side: written to the owner by the threads that hold them, a piece of 32 rows each, the parts
// take five times as long.)
template <typename T, int OUT, int S>
__global__ void __launch_bounds__(kThreads, 1)
fp8_scores_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ CUtensorMap map_out, const Fp8ScoresArgs a, const TileOrder order,
                  const int a_rows, const bool keeps_a) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    using L = Layout<S>;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBars);   // [S] codes landed
    uint64_t* empty = full + S;                                      // [S] the products that read the stage are done
    uint64_t* sfull = empty + S;                                     // [kScaleSlots] a group's scales landed
    uint64_t* sempty = sfull + kScaleSlots;                          // [kScaleSlots] and are no longer needed
    uint64_t* afull = sempty + kScaleSlots;                          // a kept query tile landed
    uint64_t* aempty = afull + 1;                                    // the products that read it are done
    uint64_t* tfull = aempty + 1;                                    // accumulator complete
    uint64_t* tfree = tfull + 1;                                     // the columns the next tile shares are drained
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfree + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // known to be uniform
    const int k_blocks = (a.dim + kTileK - 1) / kTileK;
    const int scale_pitch = (a.dim + 511) / 512 * 4;
    constexpr bool TMA_OUT = OUT == kTma || OUT == kTmaOdd, SPLIT = OUT == kSplit;
    const uint32_t rank = SPLIT ? cluster_rank() : 0, parts = SPLIT ? cluster_size() : 1;
    const uint32_t t_first = SPLIT ? blockIdx.x / parts : blockIdx.x, t_step = SPLIT ? order.tiles : gridDim.x;
    const int groups = (k_blocks + 3) / 4;
    const int k_first = SPLIT ? (int)(groups * rank / parts) * 4 : 0;
    const int k_end = SPLIT ? min(k_blocks, (int)(groups * (rank + 1) / parts) * 4) : k_blocks;

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            mbar_init(&sfull[s], 1);
            mbar_init(&sempty[s], 1);
        }
        mbar_init(afull, 1);
        mbar_init(aempty, 1);
        mbar_init(tfull, 1);
        mbar_init(tfree, kEpiWarps);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    // Query rows that are not loaded stay zero: products with whatever lay there would be as wrong to
    // store, but cost power, and with it clock.
    for (int i = a_rows * kTileK + tid * 16; i < kTileM * kTileK; i += kThreads * 16)
#pragma unroll
        for (int s = 0; s < S; ++s) *reinterpret_cast<uint4*>(smem + s * kABytes + i) = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t par = 0;
            bool ok = true;
            int64_t kept = -1;          // first row of the query tile kept, how many were
            uint32_t kept_tiles = 0;
            for (uint32_t t = t_first; t < order.tiles && ok; t += t_step) {
                int64_t m0, n0;
                order.at(t, m0, n0);
                for (int kb = k_first; kb < k_end; ++kb) {
                    if (!(ok = mbar_wait(&empty[s], par ^ 1u, abort_flag, a))) break;
                    mbar_expect_tx(&full[s], ((keeps_a ? 0 : a_rows) + kTileN) * kTileK);
                    if (!keeps_a) tma_load_2d(smem + s * kABytes, &map_a, kb * kTileK, (int)m0, &full[s]);
                    tma_load_2d(smem + L::kOffB + s * kBBytes, &map_b, kb * kTileK, (int)n0, &full[s]);
                    if (++s == S) {
                        s = 0;
                        par ^= 1u;
                    }
                }
                if (keeps_a && ok && m0 != kept) {
                    // after the row tile's loads: it fits the ring, and need not wait for the kept tile's end
                    if (kept >= 0 && !(ok = mbar_wait(aempty, (kept_tiles - 1) & 1u, abort_flag, a))) break;
                    kept = m0;
                    ++kept_tiles;
                    mbar_expect_tx(afull, k_blocks * a_rows * kTileK);
                    for (int kb = 0; kb < k_blocks; ++kb)
                        tma_load_2d(smem + kb * kABytes, &map_a, kb * kTileK, (int)m0, afull);
                }
            }
        }
    } else if (warp == 1) {
        const uint32_t leads = elect_leader();
        const uint32_t codes = smem_u32(smem), scales = smem_u32(smem + L::kOffScales);
        uint32_t s = 0, par = 0, i = 0, group = 0;
        bool ok = true;
        int64_t kept = -1;
        uint32_t kept_tiles = 0;
        for (uint32_t t = t_first; t < order.tiles && ok; t += t_step, ++i) {
            bool last_of_kept = false;
            if (keeps_a) {
                int64_t m0, n0, m1 = -1;
                order.at(t, m0, n0);
                if (t + t_step < order.tiles) order.at(t + t_step, m1, n0);
                last_of_kept = m1 != m0;
                if (m0 != kept) {
                    kept = m0;
                    if (!__all_sync(0xffffffffu, mbar_wait(afull, kept_tiles & 1u, abort_flag, a))) break;
                    ++kept_tiles;
                }
            }
            if (i > 0 && !__all_sync(0xffffffffu, mbar_wait(tfree, (i - 1) & 1u, abort_flag, a))) break;
            const uint32_t acc = tmem + (i & 1u) * kAccStep;
            for (int kb = k_first; kb < k_end; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait(&full[s], par, abort_flag, a));
                if (!ok) break;
                const uint32_t slot = group % kScaleSlots, ta = tmem + kTmemScales + group % 4 * 16, tb = ta + 8;
                if ((kb & 3) == 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sfull[slot], group / kScaleSlots & 1u, abort_flag, a));
                    if (!ok) break;
                }
                tc_fence_after();
                if ((kb & 3) == 0) {
                    const uint64_t sc = desc_rows16(scales + slot * kScaleBytes);
                    scales_to_tmem(leads, ta, sc);
                    scales_to_tmem(leads, tb, sc + (512 >> 4));
                    scales_to_tmem(leads, tb + 4, sc + (1024 >> 4));
                }
                const uint64_t da = desc_sw128(codes + (keeps_a ? kb : s) * kABytes);
                const uint64_t db = desc_sw128(codes + L::kOffB + s * kBBytes);
                const uint32_t idesc = kInstrDesc | (uint32_t)(kb & 3) << 29 | (uint32_t)(kb & 3) << 4;
                const int slices = (min(a.dim - kb * kTileK, kTileK) + 31) / 32;
                if (slices == kTileK / 32) {
#pragma unroll
                    for (int j = 0; j < kTileK / 32; ++j)
                        umma_mxf8(leads, acc, da + j * 2, db + j * 2, idesc, ta, tb, kb != k_first || j != 0 ? 1u : 0u);
                } else {
                    for (int j = 0; j < slices; ++j)
                        umma_mxf8(leads, acc, da + j * 2, db + j * 2, idesc, ta, tb, kb != k_first || j != 0 ? 1u : 0u);
                }
                umma_commit(leads, &empty[s]);
                if ((kb & 3) == 3 || kb == k_end - 1) {
                    umma_commit(leads, &sempty[slot]);
                    ++group;
                }
                if (++s == S) {
                    s = 0;
                    par ^= 1u;
                }
            }
            if (ok && last_of_kept) umma_commit(leads, aempty);
            if (ok) umma_commit(leads, tfull);
        }
    } else if (warp == 2) {
        // A group: the words that cover four k-blocks of the tile's rows, lane l those of rows l, l + 32, ...
        // Its copies are waited for kScalesAhead groups later.
        uint32_t sent = 0, done = 0;
        bool ok = true;
        auto publish = [&]() {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sfull[done % kScaleSlots]);
            ++done;
        };
        auto copy = [&](uint32_t dst, const uint8_t* base, int64_t r, int64_t rows, int kb) {
            const bool there = r < rows;      // else four zero bytes
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst),
                         "l"(base + (there ? r * scale_pitch + kb : 0)), "r"(there ? 4 : 0)
                         : "memory");
        };
        for (uint32_t t = t_first; t < order.tiles && ok; t += t_step) {
            int64_t m0, n0;
            order.at(t, m0, n0);
            for (int kb = k_first; kb < k_end; kb += 4) {
                const uint32_t slot = sent % kScaleSlots;
                ok = __all_sync(0xffffffffu, mbar_wait(&sempty[slot], (sent / kScaleSlots & 1u) ^ 1u, abort_flag, a));
                if (!ok) break;
                const uint32_t dst = smem_u32(smem + L::kOffScales + slot * kScaleBytes) + lane * 16;
#pragma unroll
                for (int g = 0; g < 4; ++g) copy(dst + g * 4, a.q_scales, m0 + g * 32 + lane, a.Q, kb);
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    copy(dst + 512 + (g >> 2) * 512 + (g & 3) * 4, a.scales, n0 + g * 32 + lane, a.n, kb);
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (++sent - done > kScalesAhead) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kScalesAhead) : "memory");
                    publish();
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        while (ok && done < sent) publish();
    } else if (SPLIT) {
        if (warp >= 4) {
            __all_sync(0xffffffffu, mbar_wait(tfull, 0, abort_flag, a));
            tc_fence_after();
        }
    } else if (warp >= 4) {
        const int g = warp & 3, half = (warp - 4) >> 2;      // 32 lanes of tensor memory; which of their two warps
        constexpr int W = 128 / (int)sizeof(T);              // columns of a piece
        unsigned char* stage = smem + L::kOffOut + (warp - 4) * 2 * 4096;      // two pieces in flight a warp
        float* sbias = reinterpret_cast<float*>(smem + L::kOffBias) + (warp - 4) * (kTileN / 2);
        constexpr int kTurn = 64, kTurns = kTileN / kTurn / 2;   // columns read at once; turns of a warp
        const uint32_t leads = elect_leader();
        const int odd = a.n % (16 / (int)sizeof(T));      // columns after the last whole 16 bytes
        uint64_t policy;
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        uint32_t i = 0, sent = 0;
        int64_t m_next, n_next;
        order.at(t_first, m_next, n_next);
        // the biases of a tile's columns are fetched while the tile before is stored
        float next_bias[kTurns * kTurn / 32];
        const auto col_of = [&](uint32_t tile, int turn) {
            // turns from the accumulator's shared columns on: its last 64 or its first 64
            return ((tile & 1u ? 0 : kTileN - kShared) + (2 * turn + half) * kTurn) & (kTileN - 1);
        };
        const auto fetch_bias = [&](uint32_t tile, int64_t n0) {
#pragma unroll
            for (int j = 0; j < kTurns * kTurn / 32; ++j) {
                const int64_t n = n0 + col_of(tile, j * 32 / kTurn) + j * 32 % kTurn + lane;
                next_bias[j] = n < a.n ? a.bias[n] : 0.f;
            }
        };
        if (a.bias) fetch_bias(0, n_next);
        for (uint32_t t = t_first; t < order.tiles; t += t_step, ++i) {
            const int64_t m0 = m_next + g * 32, n0 = n_next;
            if (t + t_step < order.tiles) order.at(t + t_step, m_next, n_next);
            const int rows = (int)(a.Q - m0 < 32 ? a.Q - m0 : 32);      // this warp's, none or fewer past the end
            if (a.bias) {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < kTurns * kTurn / 32; ++j) sbias[j * 32 + lane] = next_bias[j];
                __syncwarp();
                if (t + t_step < order.tiles) fetch_bias(i + 1, n_next);
            }
            if (!__all_sync(0xffffffffu, mbar_wait(tfull, i & 1u, abort_flag, a))) break;
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(g * 32) << 16) + (i & 1u) * kAccStep;
#pragma unroll 1
            for (int turn = 0; turn < kTurns; ++turn) {
                const int col0 = col_of(i, turn);
                const bool used = rows > 0 && n0 + col0 < a.n;
                uint32_t r[kTurn / 32][32];
                if (used) {
                    tmem_ld32(acc + (uint32_t)col0, r[0]);
                    tmem_ld32(acc + (uint32_t)col0 + 32, r[1]);
                    tmem_ld_wait();
                }
                if (turn == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tfree);
                }
                if (!used) continue;
#pragma unroll
                for (int p = 0; p < kTurn / W; ++p) {
                    const int col = col0 + p * W;
                    if (n0 + col >= a.n) continue;
#pragma unroll
                    for (int j = 0; j < W; j += 4) {
                        uint32_t* x = &r[(p * W + j) / 32][(p * W + j) % 32];
                        float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (a.bias) b = *reinterpret_cast<const float4*>(sbias + turn * kTurn + p * W + j);
                        x[0] = __float_as_uint(fmaf(a.alpha, __uint_as_float(x[0]), b.x));
                        x[1] = __float_as_uint(fmaf(a.alpha, __uint_as_float(x[1]), b.y));
                        x[2] = __float_as_uint(fmaf(a.alpha, __uint_as_float(x[2]), b.z));
                        x[3] = __float_as_uint(fmaf(a.alpha, __uint_as_float(x[3]), b.w));
                    }
                    if (TMA_OUT) {
                        constexpr int E = 16 / (int)sizeof(T);
                        unsigned char* buf = stage + (sent++ & 1u) * 4096;
                        // the piece that used this buffer has left shared memory
                        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                        __syncwarp();
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            uint4 x;
                            const uint32_t* y = &r[(p * W + u * E) / 32][(p * W + u * E) % 32];
                            if (sizeof(T) == 4)
                                x = make_uint4(y[0], y[1], y[2], y[3]);
                            else
                                x = make_uint4(pack2<T>(__uint_as_float(y[0]), __uint_as_float(y[1])),
                                               pack2<T>(__uint_as_float(y[2]), __uint_as_float(y[3])),
                                               pack2<T>(__uint_as_float(y[E - 4]), __uint_as_float(y[E - 3])),
                                               pack2<T>(__uint_as_float(y[E - 2]), __uint_as_float(y[E - 1])));
                            *reinterpret_cast<uint4*>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) = x;
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        tma_store_2d(leads, &map_out, (int)(n0 + col), (int)m0, buf, policy);
                        if constexpr (OUT == kTmaOdd) {
                            const uint32_t at = (uint32_t)(a.n - odd) - (uint32_t)(n0 + col);      // in the piece, or beyond W
                            if (at < (uint32_t)W && lane < rows) {
                                const T* from = reinterpret_cast<const T*>(buf + lane * 128 + ((at / E ^ (lane & 7)) << 4));
                                T* to = static_cast<T*>(a.out) + (m0 + lane) * a.ld + (a.n - odd);
                                for (int e = 0; e < odd; ++e) to[e] = from[e];
                            }
                        }
                    } else {
                        float* tile = reinterpret_cast<float*>(stage);      // column j of row l at l * 32 + (j ^ l)
#pragma unroll
                        for (int w = 0; w < W / 32; ++w) {
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 32; ++j) tile[lane * 32 + (j ^ lane)] = __uint_as_float(r[p * W / 32 + w][j]);
                            __syncwarp();
                            const int64_t n = n0 + col + w * 32 + lane;
                            if (n < a.n) {
                                T* out = static_cast<T*>(a.out) + m0 * a.ld + n;
#pragma unroll 4
                                for (int j = 0; j < rows; ++j) out[j * a.ld] = from_f32<T>(tile[j * 32 + (lane ^ j)]);
                            }
                        }
                    }
                }
            }
        }
        if (TMA_OUT) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }

    if constexpr (SPLIT) {
        const int width = kTileN / (int)parts;      // columns a CTA owns
        int64_t m0, n0;
        order.at(t_first, m0, n0);
        const int rows = (int)(a.Q - m0 < kTileM ? a.Q - m0 : kTileM);
        // the accumulator as [row][column], 16-byte pieces permuted by the row; the products that read
        // the stages' memory are done
        const int g = warp & 3, half = (warp - 4) >> 2, held = g * 32 + lane;
        const bool sound = __all_sync(0xffffffffu, !*abort_flag);
        if (warp >= 4 && g * 32 < rows && sound) {
            const uint32_t acc = tmem + ((uint32_t)(g * 32) << 16);
#pragma unroll 1
            for (int col = half * 32; col < kTileN; col += 64) {
                uint32_t r[32];
                __syncwarp();
                tmem_ld32(acc + (uint32_t)col, r);
                tmem_ld_wait();
                uint4* to = reinterpret_cast<uint4*>(smem) + held * (kTileN / 4);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    to[(col / 4 + u) ^ (held & 7)] = make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]);
            }
            tc_fence_before();
        }
        __syncwarp();
        cluster_sync();
        if (warp >= 4 && sound) {
            // four columns a thread, the threads of a row side by side
            const int log_pieces = __ffs(width / 4) - 1;
            const bool whole = ((uintptr_t)a.out | (uintptr_t)(a.ld * sizeof(T))) % (4 * sizeof(T)) == 0;
#pragma unroll 2
            for (int i = (warp - 4) * 32 + lane; i < rows << log_pieces; i += kEpiWarps * 32) {
                const int row = i >> log_pieces, piece = i - (row << log_pieces);
                const uint32_t from = smem_u32(smem) + (row * (kTileN / 4) + (((int)rank * (width / 4) + piece) ^ (row & 7))) * 16;
                float4 part[8];
#pragma unroll
                for (uint32_t p = 0; p < 8; ++p)
                    if (p < parts) part[p] = load_peer(peer_smem(from, p));
                float4 sum = part[0];
#pragma unroll
                for (uint32_t p = 1; p < 8; ++p) {
                    if (p >= parts) break;
                    const float4 x = part[p];
                    sum.x += x.x;
                    sum.y += x.y;
                    sum.z += x.z;
                    sum.w += x.w;
                }
                const int64_t n = n0 + (int64_t)rank * width + piece * 4;
                T* out = static_cast<T*>(a.out) + (m0 + row) * a.ld + n;
                alignas(16) T v[4];
                const float y[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = from_f32<T>(fmaf(a.alpha, y[e], a.bias && n + e < a.n ? a.bias[n + e] : 0.f));
                if (whole && n + 4 <= a.n) {
                    if (sizeof(T) == 4)
                        *reinterpret_cast<uint4*>(out) = *reinterpret_cast<uint4*>(v);
                    else
                        *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(v);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + e < a.n) out[e] = v[e];
                }
            }
        }
        __syncwarp();
        cluster_sync();      // nobody reads a peer any more
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // a wait ran out: give copies and products in flight time to land (bounded)
        const long long t_end = clock64() + 20000000ll;
        while (clock64() < t_end) {
        }
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ------------------------------------------------------------------------- product, few queries
//
// Up to 32 queries: the base rows take the products' M and the queries their N, so a tile is 256 base
// rows (two products of M = 128, N = NQ).  The products then cost a fraction of what a query tile of
// mostly nothing would, and of its power (1 x 1M x 512 ran 97 us at the 1.5 GHz that it left), and a lane
// holds one base row's scores, so all eight epilogue warps have work and a warp stores a query's 32 scores
// side by side straight from its registers, at any alignment.  Bound by memory: 1 x 1M x 512 79 us,
// 6.6 TB/s; 32 x 1M x 512 fp32 98 us (a query tile: 100); 1 x 4M x 128 83 us (165); where rows are short,
// by the tensor copies, which take their time per row more than per byte (16 x 1M bf16: 64 columns 28 us, 128
// columns 32; 17 x 2M fp32: 53 and 71): 16 x 1000003 x 100 bf16 32 us, 32 x 300k x 128 17 us (21.5), 17 x 2M x
// 100 70 us (87); against the rule, 32 x 1M x 130 bf16 51.8 us (51).  The query tile is
// kept, if its k-blocks fit the stages: its rows copied with every row tile cost 16 x 1000003 x 100 47 us.
// 64 queries lose: 64 x 1M x 128 bf16 takes 50 us against 47 in query tiles.  (Scores through shared memory and tensor stores: 16.5 us for 32 x
// 300k x 128, but 76 for 17 x 2M x 100 and 84 for 1 x 1M x 512.)
//
// Four stages of 34 or 36 KB: with five 1 x 1M x 512 takes 83 us, with six 87; memory slows when more is
// asked for at once.  Tensor memory: two buffers of 2 NQ columns and, from 128, eight slots of 16 columns
// of scales (as many slots as stages or more: see above).  Roles as above, epilogue warp 4 + 4 h + g for
// rows 32 g .. 32 g + 31 of half h.
constexpr int kFewQueries = 32, kFewStages = 4, kFewSlots = 8;
constexpr int kFewBase = 256 * kTileK;
template <int NQ>
struct Few {
    static constexpr int kQ = NQ * kTileK;                          // bytes of a stage's queries
    static constexpr int kOffQ = kFewStages * kFewBase;
    static constexpr int kOffScales = kOffQ + kFewStages * kQ;
    static constexpr int kOffBars = kOffScales + kScaleSlots * kScaleBytes;
    static constexpr int kBytes = kOffBars + 256 + 1024;
    static constexpr uint32_t kInstr = (1u << 23) | ((uint32_t)(NQ >> 3) << 17) | ((uint32_t)(kTileM >> 7) << 27);
    static_assert(NQ <= 32 && kFewSlots >= kFewStages && kBytes <= 232448, "few queries");
};

template <typename T, int NQ>
__global__ void __launch_bounds__(kThreads, 1)
fp8_few_scores_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_b,
                      const Fp8ScoresArgs a, const uint32_t tiles, const int q_rows) {
    using F = Few<NQ>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::kOffBars);      // [kFewStages] codes landed
    uint64_t* empty = full + kFewStages;                                   // [kFewStages] the products that read them are done
    uint64_t* sfull = empty + kFewStages;                                  // [kScaleSlots] a group's scales landed
    uint64_t* sempty = sfull + kScaleSlots;                                // [kScaleSlots] and are no longer needed
    uint64_t* tfull = sempty + kScaleSlots;                                // [2] accumulator buffer complete
    uint64_t* tfree = tfull + 2;                                           // [2] and drained
    uint64_t* qfull = tfree + 2;                                           // the query tile landed, if it is kept
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(qfull + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // known to be uniform
    const int k_blocks = (a.dim + kTileK - 1) / kTileK;
    const int scale_pitch = (a.dim + 511) / 512 * 4;
    const bool keeps_q = k_blocks <= kFewStages;      // as above

    if (tid == 0) {
        for (int s = 0; s < kFewStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            mbar_init(&sfull[s], 1);
            mbar_init(&sempty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tfree[b], kEpiWarps);
        }
        mbar_init(qfull, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // query rows that are not loaded stay zero: their products are not stored, but cost power
    for (int i = q_rows * kTileK + tid * 16; i < F::kQ; i += kThreads * 16)
#pragma unroll
        for (int s = 0; s < kFewStages; ++s)
            *reinterpret_cast<uint4*>(smem + F::kOffQ + s * F::kQ + i) = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t par = 0;
            bool ok = true;
            if (keeps_q) {
                mbar_expect_tx(qfull, k_blocks * q_rows * kTileK);
                for (int kb = 0; kb < k_blocks; ++kb)
                    tma_load_2d(smem + F::kOffQ + kb * F::kQ, &map_q, kb * kTileK, 0, qfull);
            }
            for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x)
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!(ok = mbar_wait_few(&empty[s], par ^ 1u, abort_flag, a))) break;
                    mbar_expect_tx(&full[s], kFewBase + (keeps_q ? 0 : q_rows) * kTileK);
                    tma_load_2d(smem + s * kFewBase, &map_b, kb * kTileK, (int)((int64_t)t * 256), &full[s]);
                    if (!keeps_q) tma_load_2d(smem + F::kOffQ + s * F::kQ, &map_q, kb * kTileK, 0, &full[s]);
                    if (++s == kFewStages) {
                        s = 0;
                        par ^= 1u;
                    }
                }
        }
    } else if (warp == 1) {
        const uint32_t leads = elect_leader();
        const uint32_t codes = smem_u32(smem), scales = smem_u32(smem + F::kOffScales);
        uint32_t s = 0, par = 0, i = 0, group = 0;
        bool ok = !keeps_q || __all_sync(0xffffffffu, mbar_wait_few(qfull, 0, abort_flag, a));
        for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++i) {
            const uint32_t b = i & 1u;
            if (i >= 2 && !__all_sync(0xffffffffu, mbar_wait_few(&tfree[b], ((i >> 1) - 1) & 1u, abort_flag, a))) break;
            const uint32_t acc = tmem + b * 2 * NQ;
            for (int kb = 0; kb < k_blocks; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait_few(&full[s], par, abort_flag, a));
                if (!ok) break;
                const uint32_t slot = group % kScaleSlots, ta = tmem + 128 + group % kFewSlots * 16, tb = ta + 8;
                if ((kb & 3) == 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait_few(&sfull[slot], group / kScaleSlots & 1u, abort_flag, a));
                    if (!ok) break;
                }
                tc_fence_after();
                if ((kb & 3) == 0) {
                    const uint64_t sc = desc_rows16(scales + slot * kScaleBytes);
                    scales_to_tmem(leads, ta, sc);
                    scales_to_tmem(leads, ta + 4, sc + (512 >> 4));
                    scales_to_tmem(leads, tb, sc + (1024 >> 4));
                }
                const uint64_t d0 = desc_sw128(codes + s * kFewBase), d1 = d0 + (128 * kTileK >> 4);
                const uint64_t dq = desc_sw128(codes + F::kOffQ + (keeps_q ? kb : s) * F::kQ);
                const uint32_t idesc = F::kInstr | (uint32_t)(kb & 3) << 29 | (uint32_t)(kb & 3) << 4;
                const int slices = (min(a.dim - kb * kTileK, kTileK) + 31) / 32;
                for (int j = 0; j < slices; ++j) {
                    umma_mxf8(leads, acc, d0 + j * 2, dq + j * 2, idesc, ta, tb, (kb | j) != 0 ? 1u : 0u);
                    umma_mxf8(leads, acc + NQ, d1 + j * 2, dq + j * 2, idesc, ta + 4, tb, (kb | j) != 0 ? 1u : 0u);
                }
                umma_commit(leads, &empty[s]);
                if ((kb & 3) == 3 || kb == k_blocks - 1) {
                    umma_commit(leads, &sempty[slot]);
                    ++group;
                }
                if (++s == kFewStages) {
                    s = 0;
                    par ^= 1u;
                }
            }
            if (ok) umma_commit(leads, &tfull[b]);
        }
    } else if (warp == 2) {
        // as above: a group's words, base rows first, then the queries'
        uint32_t sent = 0, done = 0;
        bool ok = true;
        auto publish = [&]() {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sfull[done % kScaleSlots]);
            ++done;
        };
        auto copy = [&](uint32_t dst, const uint8_t* base, int64_t r, int64_t rows, int kb) {
            const bool there = r < rows;      // else four zero bytes
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst),
                         "l"(base + (there ? r * scale_pitch + kb : 0)), "r"(there ? 4 : 0)
                         : "memory");
        };
        for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x)
            for (int kb = 0; kb < k_blocks; kb += 4) {
                const uint32_t slot = sent % kScaleSlots;
                ok = __all_sync(0xffffffffu, mbar_wait_few(&sempty[slot], (sent / kScaleSlots & 1u) ^ 1u, abort_flag, a));
                if (!ok) break;
                const uint32_t dst = smem_u32(smem + F::kOffScales + slot * kScaleBytes) + lane * 16;
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    copy(dst + (g >> 2) * 512 + (g & 3) * 4, a.scales, (int64_t)t * 256 + g * 32 + lane, a.n, kb);
                copy(dst + 1024, a.q_scales, lane, a.Q, kb);      // rows from Q on: zero, and not used
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (++sent - done > kScalesAhead) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kScalesAhead) : "memory");
                    publish();
                }
            }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        while (ok && done < sent) publish();
    } else if (warp >= 4) {
        const int row = (warp - 4) * 32 + lane;      // of the tile: half (warp - 4) / 4, 32 lanes of tensor memory (warp & 3)
        const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)((warp - 4) >> 2) * NQ;
        uint32_t i = 0;
        int64_t n = (int64_t)blockIdx.x * 256 + row;
        float next_bias = a.bias && n < a.n ? a.bias[n] : 0.f;
        for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
            const float bias = next_bias;
            T* out = static_cast<T*>(a.out) + n;
            const bool there = n < a.n;
            n += (int64_t)gridDim.x * 256;
            if (a.bias) next_bias = n < a.n ? a.bias[n] : 0.f;
            const uint32_t b = i & 1u;
            if (!__all_sync(0xffffffffu, mbar_wait_few(&tfull[b], i >> 1 & 1u, abort_flag, a))) break;
            tc_fence_after();
            uint32_t r[NQ];
            if constexpr (NQ == 16)
                tmem_ld16(from + b * 2 * NQ, r);
            else
                tmem_ld32(from + b * 2 * NQ, r);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tfree[b]);
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                if (q >= a.Q) break;
                if (there) *out = from_f32<T>(fmaf(a.alpha, __uint_as_float(r[q]), bias));
                out += a.ld;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // a wait ran out: give copies and products in flight time to land (bounded)
        const long long t_end = clock64() + 20000000ll;
        while (clock64() < t_end) {
        }
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static std::mutex mu;
    static EncodeTiledFn fn = nullptr;
    std::lock_guard<std::mutex> lock(mu);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) != cudaSuccess ||
            res != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

// A matrix as a 2-D tensor (column, row).  Loads outside it read zeros, stores outside it are dropped.
bool matrix_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t rows, int64_t cols, int64_t row_bytes,
                int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t gdim[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t gstride[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return enc(map, type, 2, const_cast<void*>(base), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Clusters of `parts` CTAs of the split kernel that the current device holds at once (fewer than SMs /
// parts: a cluster stays inside one group of SMs); asked for once per device.
template <typename Kernel>
int clusters_at_once(Kernel* kernel, int parts) {
    static std::atomic<int> known[64][4];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    const int slot = parts == 2 ? 1 : parts == 4 ? 2 : 3;
    if (dev >= 0 && dev < 64)
        if (const int n = known[dev][slot].load(std::memory_order_relaxed)) return n - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)parts);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Layout<4>::kBytes;
    cudaLaunchAttribute cluster = {};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = (unsigned)parts;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    if (dev >= 0 && dev < 64) known[dev][slot].store(n + 1, std::memory_order_relaxed);
    return n;
}

// CTAs that share a tile: the count with the shortest time in k-blocks a CTA goes through, one after the
// other, a wave of shared tiles costing kSplitCost more for its start and its join.  Shared or not: 1 x
// 1000 x 4096 6.8 or 16.7 us, 64 x 4096 x 4096 10 or 17, 128 x 2048 x 2048 10 or 12, 16 x 16384 x 2048
// 12.5 or 14; against the rule, 200 x 3000 x 1000 12.9 or 11.
constexpr int kSplitCost = 5;
template <typename Kernel>
int split_of(Kernel* kernel, uint32_t tiles, int k_blocks, int sm_count) {
    int best = 1;
    int64_t least = (int64_t)((tiles + sm_count - 1) / sm_count) * k_blocks;
    for (int p = 2; p <= 8 && 4 * p <= k_blocks + 3; p *= 2) {
        const int at_once = clusters_at_once(kernel, p);
        if (at_once < 1) continue;
        const int64_t cost = (int64_t)((tiles + at_once - 1) / at_once) * (((k_blocks + 3) / 4 + p - 1) / p * 4 + kSplitCost);
        if (cost < least) {
            least = cost;
            best = p;
        }
    }
    return best;
}

template <typename T>
cudaError_t scores_t(const Fp8ScoresArgs& a, int sm_count, cudaStream_t stream) {
    const CUtensorMapDataType type = a.type == kTypeF32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : a.type == kTypeBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    // Tensor stores need rows that start at 16-byte boundaries, and write whole 16 bytes, past the
    // tensor's end, too: the tensor they see ends with the last whole ones.
    const int whole = a.n - a.n % (16 / (int)sizeof(T));
    const bool tma = whole > 0 && ((uintptr_t)a.out | (uintptr_t)(a.ld * sizeof(T))) % 16 == 0;
    // rows of a query tile that are loaded: the others' products are not stored, whatever they are
    // (a row outside the matrix costs the tensor copy more than one inside it)
    const int a_rows = a.Q >= kTileM ? kTileM : (a.Q + 7) / 8 * 8;
    alignas(64) CUtensorMap map_a, map_b, map_out;
    if (!matrix_map(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.q_codes, a.Q, a.dim, fp8_code_pitch(a.dim), kTileK, a_rows,
                    CU_TENSOR_MAP_SWIZZLE_128B) ||
        !matrix_map(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, a.n, a.dim, fp8_code_pitch(a.dim), kTileK, kTileN,
                    CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    TileOrder order;
    order.tiles_m = (uint32_t)(((int64_t)a.Q + kTileM - 1) / kTileM);
    order.tiles_n = (uint32_t)(((int64_t)a.n + kTileN - 1) / kTileN);
    order.tiles = order.tiles_m * order.tiles_n;
    const int64_t in_l2 = kChunkBytes / (kTileN * fp8_code_pitch(a.dim));
    order.chunk_n = (uint32_t)(in_l2 < sm_count ? sm_count : in_l2);
    if (order.chunk_n > order.tiles_n) order.chunk_n = order.tiles_n;
    const int k_blocks = (a.dim + kTileK - 1) / kTileK;
    static std::atomic<uint64_t> granted[6];
    int parts = 1;
    if (order.tiles <= (uint32_t)sm_count && k_blocks > 4) {
        auto split = fp8_scores_kernel<T, kSplit, 4>;
        cudaError_t e = grant_smem(split, Layout<4>::kBytes, granted[kSplit]);
        if (e != cudaSuccess) return e;
        parts = split_of(split, order.tiles, k_blocks, sm_count);
    }
    if (parts == 1 && a.Q <= kFewQueries) {
        const bool most = a.Q > 16;
        auto few = most ? fp8_few_scores_kernel<T, 32> : fp8_few_scores_kernel<T, 16>;
        const int bytes = most ? Few<32>::kBytes : Few<16>::kBytes;
        cudaError_t e = grant_smem(few, bytes, granted[most ? 5 : 4]);
        if (e != cudaSuccess) return e;
        few<<<order.tiles < (uint32_t)sm_count ? order.tiles : (uint32_t)sm_count, kThreads, bytes, stream>>>(
            map_a, map_b, a, order.tiles, a_rows);
        return cudaGetLastError();
    }
    if (!tma)
        map_out = map_a;      // not used
    else if (!matrix_map(&map_out, type, a.out, a.Q, whole, a.ld * (int64_t)sizeof(T), 128 / (int)sizeof(T), 32,
                         CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    const int stages = parts > 1 ? 4 : 3, smem = stages == 4 ? Layout<4>::kBytes : Layout<3>::kBytes;
    const int out = !tma ? kPlain : whole < a.n ? kTmaOdd : kTma;
    auto kernel = parts > 1         ? fp8_scores_kernel<T, kSplit, 4>
                  : out == kTma     ? fp8_scores_kernel<T, kTma, 3>
                  : out == kTmaOdd  ? fp8_scores_kernel<T, kTmaOdd, 3>
                                    : fp8_scores_kernel<T, kPlain, 3>;
    if (parts == 1) {
        cudaError_t e = grant_smem(kernel, smem, granted[out]);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts > 1 ? order.tiles * parts : order.tiles < (uint32_t)sm_count ? order.tiles : (uint32_t)sm_count);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute cluster = {};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = (unsigned)parts;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, map_out, a, order, a_rows, k_blocks <= stages);
}

}  // namespace

cudaError_t launch_fp8_quantize(const void* x, int type, int64_t rows, int dim, int64_t ld, uint8_t* codes,
                                uint8_t* scales, cudaStream_t stream) {
    if (type == kTypeF32) return quantize_t<float>(x, rows, dim, ld, codes, scales, stream);
    if (type == kTypeBf16) return quantize_t<__nv_bfloat16>(x, rows, dim, ld, codes, scales, stream);
    return quantize_t<__half>(x, rows, dim, ld, codes, scales, stream);
}

cudaError_t launch_fp8_scores(const Fp8ScoresArgs& a, int sm_count, cudaStream_t stream) {
    if (a.type == kTypeF32) return scores_t<float>(a, sm_count, stream);
    if (a.type == kTypeBf16) return scores_t<__nv_bfloat16>(a, sm_count, stream);
    return scores_t<__half>(a, sm_count, stream);
}

}  // namespace coral
