// Rules on score rows, one pass: for row q and column j, with c = how often j occurs in seen[q] and
// (rho, phi, pi) = penalties[q],
//     c > 0:  s <- (s > 0 ? s / rho : s * rho) - phi * c - pi
//     s <- s + (sum of row q's biases whose id is j, in list order)
//     excluded: s <- -inf
// in fp32, rounded once to the output's type.
//
// A CTA owns kCols columns of one row.  Its own scores and mask words are requested first and stay in
// flight while it turns the row's two id lists into tables over its columns in shared memory: counts
// by integer atomics (their order does not show), biases by one warp in list order, and one bit for
// every column that either list touches: a thread whose columns are untouched reads one word of bits
// and no table.  Then it applies the rules and stores.  No table in global memory, nothing to clear between calls, one launch.  The
// history is read once per CTA, from L2: wider columns would read it less often but leave fewer CTAs
// an SM, and latency, not that traffic, is what a CTA waits for.
#include <math_constants.h>

#include "scores.cuh"

namespace coral {

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 4096;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// v[i] of 16 bytes in registers, for an i known at run time only.
template <typename T, int V>
__device__ __forceinline__ T element(const T (&v)[V], int i) {
    T x = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j)
        if (i == j) x = v[j];
    return x;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) score_rules_kernel(const RulesArgs a, const int chunks) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int q = blockIdx.x / chunks;
    const int64_t c0 = (int64_t)(blockIdx.x % chunks) * kCols;
    const int cols = (int)(a.n - c0 < kCols ? a.n - c0 : kCols);
    const int tid = threadIdx.x, lane = tid & 31;
    const bool has_seen = a.n_seen > 0, has_bias = a.n_bias > 0;
    uint32_t* count = reinterpret_cast<uint32_t*>(smem);
    float* bias = reinterpret_cast<float*>(smem) + (has_seen ? kCols : 0);
    uint32_t* touched = reinterpret_cast<uint32_t*>(smem) + kCols * ((has_seen ? 1 : 0) + (has_bias ? 1 : 0));

    // the thread's scores: U vectors of V, vector u at column (u * kThreads + tid) * V
    constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
    constexpr int U = kCols / (kThreads * V);
    constexpr uint32_t kAll = (1u << V) - 1u;
    const T* in = static_cast<const T*>(a.in) + (size_t)q * a.ld + c0;
    T* out = static_cast<T*>(a.out) + (size_t)q * a.ld_out + c0;
    const uint32_t* ex = a.excluded ? a.excluded + (size_t)q * a.ld_excluded + c0 / 32 : nullptr;
    alignas(16) T v[U][V];
    uint32_t m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = (u * kThreads + tid) * V;
        m[u] = ex && j < cols ? ex[j >> 5] >> (j & 31) & kAll : 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = (u * kThreads + tid) * V;
        if (m[u] != kAll) {      // what is excluded altogether is not read
            if (VEC && j + V <= cols) {
                *reinterpret_cast<uint4*>(v[u]) = *reinterpret_cast<const uint4*>(in + j);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (j + i < cols) v[u][i] = in[j + i];
            }
        }
    }

    float rho = 1.f, phi = 0.f, pi = 0.f;
    if (has_seen || has_bias) {
        const int32_t* seen = has_seen ? a.seen + (size_t)q * a.n_seen : nullptr;
        constexpr int kAhead = 8;      // ids of the history in flight while the tables are cleared
        int32_t ids_ahead[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ids_ahead[i] = i * kThreads + tid < a.n_seen ? seen[i * kThreads + tid] : -1;
        if (has_seen) {
            rho = a.penalties[(size_t)q * 3];
            phi = a.penalties[(size_t)q * 3 + 1];
            pi = a.penalties[(size_t)q * 3 + 2];
        }
        const int words = (int)(touched - count) + kCols / 32;
        for (int i = tid * 4; i < words; i += kThreads * 4) *reinterpret_cast<uint4*>(count + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (has_seen) {
            auto add = [&](int32_t id) {
                const int64_t j = (int64_t)id - c0;
                if (j >= 0 && j < cols && atomicAdd(&count[j], 1u) == 0u) atomicOr(&touched[j >> 5], 1u << (j & 31));
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) add(ids_ahead[i]);
#pragma unroll 4
            for (int i = kAhead * kThreads + tid; i < a.n_seen; i += kThreads) add(seen[i]);
        }
        if (has_bias && tid < 32) {
            const int32_t* ids = a.bias_ids + (size_t)q * a.n_bias;
            const float* vals = a.bias + (size_t)q * a.n_bias;
            for (int i0 = 0; i0 < a.n_bias; i0 += 32) {
                const int i = i0 + lane;
                const int64_t j = i < a.n_bias ? (int64_t)ids[i] - c0 : -1;
                uint32_t todo = __ballot_sync(0xffffffffu, j >= 0 && j < cols);
                if (!todo) continue;
                const float val = i < a.n_bias ? vals[i] : 0.f;
                for (; todo; todo &= todo - 1) {      // in list order
                    const int src = __ffs(todo) - 1;
                    const int at = __shfl_sync(0xffffffffu, (int)j, src);
                    const float x = __shfl_sync(0xffffffffu, val, src);
                    if (lane == 0) {
                        bias[at] += x;
                        atomicOr(&touched[at >> 5], 1u << (at & 31));
                    }
                }
            }
        }
        __syncthreads();
    }

    auto rule = [&](float s, int j) {
        if (has_seen) {
            const uint32_t c = count[j];
            if (c) {
                s = s > 0.f ? s / rho : s * rho;
                s = s - phi * (float)c - pi;
            }
        }
        if (has_bias) {
            const float b = bias[j];
            if (b != 0.f) s += b;
        }
        return s;
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = (u * kThreads + tid) * V;
        uint32_t hit = 0;
        if ((has_seen || has_bias) && j < cols) hit = touched[j >> 5] >> (j & 31) & kAll & ~m[u];
        if (m[u]) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (m[u] >> i & 1u) v[u][i] = from_f32<T>(-CUDART_INF_F);
        }
        if (VEC && j + V <= cols) {
            *reinterpret_cast<uint4*>(out + j) = *reinterpret_cast<uint4*>(v[u]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (j + i < cols) out[j + i] = v[u][i];
        }
        for (; hit; hit &= hit - 1) {      // the few touched columns again
            const int i = __ffs(hit) - 1;
            out[j + i] = from_f32<T>(rule(to_f32<T>(element<T, V>(v[u], i)), j + i));
        }
    }
}

template <typename T>
cudaError_t launch_rules(const RulesArgs& a, cudaStream_t stream) {
    const int64_t chunks = (a.n + kCols - 1) / kCols;
    const size_t smem = (size_t)kCols * 4 * ((a.n_seen > 0) + (a.n_bias > 0)) + kCols / 8;
    const bool vec = ((uintptr_t)a.in | (uintptr_t)a.out | (uintptr_t)(a.ld * sizeof(T)) |
                      (uintptr_t)(a.ld_out * sizeof(T))) % 16 == 0;
    auto kernel = vec ? score_rules_kernel<T, true> : score_rules_kernel<T, false>;
    kernel<<<(unsigned)(chunks * a.Q), kThreads, smem, stream>>>(a, (int)chunks);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_score_rules(const RulesArgs& a, int, cudaStream_t stream) {
    if (a.type == kTypeF32) return launch_rules<float>(a, stream);
    if (a.type == kTypeBf16) return launch_rules<__nv_bfloat16>(a, stream);
    return launch_rules<__half>(a, stream);
}

}  // namespace coral
