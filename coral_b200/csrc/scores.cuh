// Operators on score rows: rows compressed to 8-bit floating point, dense products of compressed
// rows, rules applied to scores, and the choice of the k best (fp8_scores.cu, score_rules.cu,
// score_topk.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace coral {

// Element types of the C ABI (CORAL_F32, CORAL_BF16, CORAL_F16).
constexpr int kTypeF32 = 0, kTypeBf16 = 1, kTypeF16 = 2;
inline int type_bytes(int type) { return type == kTypeF32 ? 4 : 2; }

// Elements and fp32, to nearest even on the way back.
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

constexpr int kFp8Block = 128;        // columns that share one scale
constexpr int kFp8MaxDim = 1 << 16;
constexpr int kTopkMax = 1024;        // k of the selection
constexpr int kRulesMaxBias = 1024;   // biased ids per row
constexpr int kRulesMaxSeen = 1 << 24;   // history per row: counts are exact in fp32

// Bytes of one compressed row: codes are padded to 16 (tensor copies), scales to 4 (one word read
// covers 512 columns).
inline int64_t fp8_code_pitch(int dim) { return ((int64_t)dim + 15) / 16 * 16; }
inline int64_t fp8_scale_pitch(int dim) { return ((int64_t)dim + 511) / 512 * 4; }

cudaError_t launch_fp8_quantize(const void* x, int type, int64_t rows, int dim, int64_t ld, uint8_t* codes,
                                uint8_t* scales, cudaStream_t stream);

// Opt-in shared memory of a kernel, asked for once per kernel and device.
template <typename Kernel>
inline cudaError_t grant_smem(Kernel* kernel, int bytes, std::atomic<uint64_t>& granted) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (granted.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) granted.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

struct Fp8ScoresArgs {
    const uint8_t *q_codes, *q_scales, *codes, *scales;
    int Q, n, dim;
    float alpha;
    const float* bias;   // [n] or null
    void* out;
    int type;
    int64_t ld;          // elements between rows of out
    int* err;            // set when a bounded wait ran out
    long long wait_clocks;   // what a wait may take
};
cudaError_t launch_fp8_scores(const Fp8ScoresArgs& a, int sm_count, cudaStream_t stream);

struct RulesArgs {
    const void* in;
    void* out;
    int type, Q;
    int64_t n, ld, ld_out;
    const int32_t* seen;        // [Q][n_seen], ids outside [0, n) are skipped
    int n_seen;
    const float* penalties;     // [Q][3]
    const int32_t* bias_ids;    // [Q][n_bias], ids outside [0, n) are skipped
    const float* bias;          // [Q][n_bias]
    int n_bias;
    const uint32_t* excluded;   // rows of words, ld_excluded apart (0: one row for all)
    int64_t ld_excluded;
};
cudaError_t launch_score_rules(const RulesArgs& a, cudaStream_t stream);

struct TopkArgs {
    const void* in;
    int type, Q;
    int64_t n, ld;
    int k;
    int32_t id_base;
    int32_t* ids_out;
    float* scores_out;
    uint64_t* ws;               // topk_workspace_bytes
};
int64_t topk_workspace_bytes(int Q, int64_t n, int k, int sm_count);
cudaError_t launch_topk(const TopkArgs& a, int sm_count, cudaStream_t stream, int* launches);

}  // namespace coral
