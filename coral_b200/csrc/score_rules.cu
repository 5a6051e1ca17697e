// Rules on score rows, one pass: for row q and column j, with c = how often j occurs in seen[q] and
// (rho, phi, pi) = penalties[q],
//     c > 0:  s <- (s > 0 ? s / rho : s * rho) - phi * c - pi
//     s <- s + (sum of row q's biases whose id is j, in list order)
//     excluded: s <- -inf
// in fp32, rounded once to the output's type.
//
// A CTA owns kCols columns of one row.  It turns the row's two id lists into tables over its own
// columns in shared memory (integer counts, so the order of the atomics does not show; a bias is
// summed by the thread that holds the id's first entry), then streams its columns with 16-byte
// accesses.  No table in global memory, nothing to clear between calls, no second launch.
#include <math_constants.h>

#include "scores.cuh"

namespace coral {

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 8192;

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

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) score_rules_kernel(const RulesArgs a, const int chunks) {
    extern __shared__ unsigned char smem[];
    const int q = blockIdx.x / chunks;
    const int64_t c0 = (int64_t)(blockIdx.x % chunks) * kCols;
    const int cols = (int)(a.n - c0 < kCols ? a.n - c0 : kCols);
    const int tid = threadIdx.x;
    const bool has_seen = a.n_seen > 0, has_bias = a.n_bias > 0;
    uint32_t* count = reinterpret_cast<uint32_t*>(smem);
    float* bias = reinterpret_cast<float*>(smem) + (has_seen ? kCols : 0);
    float rho = 1.f, phi = 0.f, pi = 0.f;
    if (has_seen) {
        rho = a.penalties[(size_t)q * 3];
        phi = a.penalties[(size_t)q * 3 + 1];
        pi = a.penalties[(size_t)q * 3 + 2];
        for (int i = tid; i < kCols; i += kThreads) count[i] = 0u;
    }
    if (has_bias)
        for (int i = tid; i < kCols; i += kThreads) bias[i] = 0.f;
    if (has_seen || has_bias) __syncthreads();
    if (has_seen) {
        const int32_t* seen = a.seen + (size_t)q * a.n_seen;
        for (int i = tid; i < a.n_seen; i += kThreads) {
            const int64_t j = (int64_t)seen[i] - c0;
            if (j >= 0 && j < cols) atomicAdd(&count[j], 1u);
        }
    }
    if (has_bias) {
        const int32_t* ids = a.bias_ids + (size_t)q * a.n_bias;
        const float* vals = a.bias + (size_t)q * a.n_bias;
        for (int i = tid; i < a.n_bias; i += kThreads) {
            const int32_t id = ids[i];
            const int64_t j = (int64_t)id - c0;
            if (j < 0 || j >= cols) continue;
            bool first = true;
            for (int p = 0; p < i && first; ++p) first = ids[p] != id;
            if (!first) continue;
            float s = vals[i];
            for (int p = i + 1; p < a.n_bias; ++p)
                if (ids[p] == id) s += vals[p];
            bias[j] = s;
        }
    }
    if (has_seen || has_bias) __syncthreads();

    const T* in = static_cast<const T*>(a.in) + (size_t)q * a.ld + c0;
    T* out = static_cast<T*>(a.out) + (size_t)q * a.ld_out + c0;
    const uint32_t* ex = a.excluded ? a.excluded + (size_t)q * a.ld_excluded + c0 / 32 : nullptr;
    auto rule = [&](float s, int j, bool out_of) {
        if (has_seen) {
            const uint32_t c = count[j];
            if (c) {
                s = s > 0.f ? s / rho : s * rho;
                s = s - phi * (float)c - pi;
            }
        }
        if (has_bias) s += bias[j];
        return from_f32<T>(out_of ? -CUDART_INF_F : s);
    };
    constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
    int j0 = tid * V;
    if (VEC) {
        for (; j0 + V <= cols; j0 += kThreads * V) {
            const uint32_t m = ex ? (ex[j0 >> 5] >> (j0 & 31)) & ((1u << V) - 1u) : 0u;
            alignas(16) T v[V];
            // a fully excluded vector is not read
            if (m != (1u << V) - 1u) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(in + j0);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = rule(to_f32<T>(v[i]), j0 + i, (m >> i) & 1u);
            *reinterpret_cast<uint4*>(out + j0) = *reinterpret_cast<uint4*>(v);
        }
        j0 = cols / V * V + tid;    // the ragged end, element by element
    }
    for (; j0 < cols; j0 += kThreads) {
        const bool m = ex && ((ex[j0 >> 5] >> (j0 & 31)) & 1u);
        out[j0] = rule(m ? 0.f : to_f32<T>(in[j0]), j0, m);
    }
}

template <typename T>
cudaError_t launch_rules(const RulesArgs& a, cudaStream_t stream) {
    const int64_t chunks = (a.n + kCols - 1) / kCols;
    const size_t smem = (size_t)kCols * 4 * ((a.n_seen > 0) + (a.n_bias > 0));
    const bool vec = ((uintptr_t)a.in | (uintptr_t)a.out | (uintptr_t)(a.ld * sizeof(T)) |
                      (uintptr_t)(a.ld_out * sizeof(T))) % 16 == 0;
    auto kernel = vec ? score_rules_kernel<T, true> : score_rules_kernel<T, false>;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
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
