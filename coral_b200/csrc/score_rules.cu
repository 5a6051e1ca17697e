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
// and no table.  Then it applies the rules and stores.  No table in global memory, nothing to clear
// between calls, one launch.  The history is read once per CTA, from L2: wider columns would read it
// less often but leave fewer CTAs an SM.
//
// Measured: 32 x 1M fp32 with a shared mask 42 us, 250 MB at 5.9 TB/s; 64 x 128000 bf16, histories of
// 2000, nine tenths excluded, 11.7 us (20 MB would take 3: each of a row's 32 CTAs reads the whole history and
// clears its tables, in three waves and a chain of mask, scores, tables and stores).  With tables read for every column, eight to a thread, the latter took
// 27 us, on bank conflicts.
#include <math_constants.h>

#include "scores.cuh"

namespace coral {

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 4096;

// v[i] of 16 bytes in registers, for an i known at run time only.
template <typename T, int V>
__device__ __forceinline__ T element(const T (&v)[V], int i) {
    T x = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j)
        if (i == j) x = v[j];
    return x;
}

// Where the rows lie: elements one by one; whole vectors from the first column on, a ragged end element
// by element; whole vectors from the first 16-byte boundary of each row on.
constexpr int kElements = 0, kAligned = 1, kShifted = 2;

template <typename T, int ROWS>
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

    // column of an id in the CTA, at least cols for one outside it (modulo 2^32; n is below 2^31)
    const auto column_of = [&](int32_t id) { return (uint32_t)id - (uint32_t)c0; };
    // the beginnings of the lists, in flight with the masks
    constexpr int kAhead = 8;
    const int32_t* seen = a.seen + (size_t)q * a.n_seen;
    const int32_t* bias_ids = a.bias_ids + (size_t)q * a.n_bias;
    const float* bias_vals = a.bias + (size_t)q * a.n_bias;
    int32_t ids_ahead[kAhead], bias_id = -1;
    float bias_val = 0.f, rho = 1.f, phi = 0.f, pi = 0.f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ids_ahead[i] = i * kThreads + tid < a.n_seen ? seen[i * kThreads + tid] : -1;
    if (tid < 32 && lane < a.n_bias) {
        bias_id = bias_ids[lane];
        bias_val = bias_vals[lane];
    }
    if (has_seen) {
        rho = a.penalties[(size_t)q * 3];
        phi = a.penalties[(size_t)q * 3 + 1];
        pi = a.penalties[(size_t)q * 3 + 2];
    }

    // The thread's scores: U vectors of V, vector u at column head + (u * kThreads + tid) * V, and, of
    // shifted rows, at most one of the columns before the first and after the last whole vector.
    constexpr bool VEC = ROWS != kElements, SHIFTED = ROWS == kShifted;
    constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
    constexpr int U = kCols / (kThreads * V);
    constexpr uint32_t kAll = (1u << V) - 1u;
    const T* in = static_cast<const T*>(a.in) + (size_t)q * a.ld + c0;
    T* out = static_cast<T*>(a.out) + (size_t)q * a.ld_out + c0;
    const uint32_t* ex = a.excluded ? a.excluded + (size_t)q * a.ld_excluded + c0 / 32 : nullptr;
    const int head = SHIFTED ? min(cols, (int)((16 - ((uintptr_t)in & 15)) % 16 / sizeof(T))) : 0;
    const int end = SHIFTED ? head + (cols - head) / V * V : cols;
    const int odd = !SHIFTED ? -1 : tid < head ? tid : tid >= 32 && end + tid - 32 < cols ? end + tid - 32 : -1;
    // V bits of a row of words from bit j on
    const auto bits_at = [&](const uint32_t* words, int j) {
        const int shift = j & 31;
        uint32_t b = words[j >> 5] >> shift;
        if (SHIFTED && shift + V > 32) b |= words[(j >> 5) + 1] << (32 - shift);
        return b & kAll;
    };
    alignas(16) T v[U][V];
    uint32_t m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = head + (u * kThreads + tid) * V;
        m[u] = SHIFTED && j >= end ? kAll : ex && j < end ? bits_at(ex, j) : 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = head + (u * kThreads + tid) * V;
        if (m[u] != kAll) {      // what is excluded altogether is not read
            if (SHIFTED || (VEC && j + V <= end)) {
                *reinterpret_cast<uint4*>(v[u]) = *reinterpret_cast<const uint4*>(in + j);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (j + i < end) v[u][i] = in[j + i];
            }
        }
    }
    const bool odd_out = odd >= 0 && ex && (ex[odd >> 5] >> (odd & 31) & 1u);
    T odd_in = from_f32<T>(-CUDART_INF_F);
    if (odd >= 0 && !odd_out) odd_in = in[odd];

    if (has_seen || has_bias) {
        const int words = (int)(touched - count) + kCols / 32 + 4;      // one word to spare behind the bits
        for (int i = tid * 4; i < words; i += kThreads * 4) *reinterpret_cast<uint4*>(count + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (has_seen) {
            auto add = [&](int32_t id) {
                const uint32_t j = column_of(id);
                if (j < (uint32_t)cols && atomicAdd(&count[j], 1u) == 0u) atomicOr(&touched[j >> 5], 1u << (j & 31));
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) add(ids_ahead[i]);
#pragma unroll 4
            for (int i = kAhead * kThreads + tid; i < a.n_seen; i += kThreads) add(seen[i]);
        }
        if (has_bias && tid < 32) {
            for (int i0 = 0; i0 < a.n_bias; i0 += 32) {
                const uint32_t j = column_of(bias_id);
                const float val = bias_val;
                if (i0 + 32 < a.n_bias) {      // the next ones in flight
                    const int i = i0 + 32 + lane;
                    bias_id = i < a.n_bias ? bias_ids[i] : -1;
                    bias_val = i < a.n_bias ? bias_vals[i] : 0.f;
                }
                const bool mine = j < (uint32_t)cols;
                if (!__any_sync(0xffffffffu, mine)) continue;
                // entries of one id take turns, in list order; different ids go together
                const uint32_t same = __match_any_sync(0xffffffffu, mine ? (int)j : -1 - lane);
                const uint32_t before = __popc(same & ((1u << lane) - 1u));
                const uint32_t turns = __reduce_max_sync(0xffffffffu, before);
                for (uint32_t turn = 0; turn <= turns; ++turn) {
                    if (mine && before == turn) bias[j] += val;
                    __syncwarp();
                }
                if (mine && before == 0) atomicOr(&touched[j >> 5], 1u << (j & 31));
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
        const int j = head + (u * kThreads + tid) * V;
        if (SHIFTED && j >= end) break;
        uint32_t hit = (has_seen || has_bias) && j < end ? bits_at(touched, j) & ~m[u] : 0u;
        if (m[u]) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (m[u] >> i & 1u) v[u][i] = from_f32<T>(-CUDART_INF_F);
        }
        if (SHIFTED || (VEC && j + V <= end)) {
            *reinterpret_cast<uint4*>(out + j) = *reinterpret_cast<uint4*>(v[u]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (j + i < end) out[j + i] = v[u][i];
        }
        for (; hit; hit &= hit - 1) {      // the few touched columns again
            const int i = __ffs(hit) - 1;
            out[j + i] = from_f32<T>(rule(to_f32<T>(element<T, V>(v[u], i)), j + i));
        }
    }
    if (odd >= 0) {
        if (!odd_out && (has_seen || has_bias) && (touched[odd >> 5] >> (odd & 31) & 1u))
            odd_in = from_f32<T>(rule(to_f32<T>(odd_in), odd));
        out[odd] = odd_in;
    }
}

template <typename T>
cudaError_t launch_rules(const RulesArgs& a, cudaStream_t stream) {
    const int64_t chunks = (a.n + kCols - 1) / kCols;
    const size_t smem = (size_t)kCols * 4 * ((a.n_seen > 0) + (a.n_bias > 0)) + kCols / 8 + 16;
    const uintptr_t lie = (uintptr_t)a.in | (uintptr_t)(a.ld * sizeof(T));
    const bool alike = ((uintptr_t)a.in - (uintptr_t)a.out) % 16 == 0 && (a.ld - a.ld_out) * (int64_t)sizeof(T) % 16 == 0;
    auto kernel = !alike          ? score_rules_kernel<T, kElements>
                  : lie % 16 == 0 ? score_rules_kernel<T, kAligned>
                                  : score_rules_kernel<T, kShifted>;
    kernel<<<(unsigned)(chunks * a.Q), kThreads, smem, stream>>>(a, (int)chunks);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_score_rules(const RulesArgs& a, cudaStream_t stream) {
    if (a.type == kTypeF32) return launch_rules<float>(a, stream);
    if (a.type == kTypeBf16) return launch_rules<__nv_bfloat16>(a, stream);
    return launch_rules<__half>(a, stream);
}

}  // namespace coral
