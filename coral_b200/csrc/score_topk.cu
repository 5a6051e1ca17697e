// The k best of every row of scores: ids and scores, best first, equal scores by the lower id.
//
// Keys: ord(score) in the high word (ord is monotone), the complement of the column in the low one,
// so keys are unique and a larger key is better.  -inf (an excluded row) and NaN never become a key;
// a row with fewer than k keys ends in padding (id -1).
//
// A CTA takes one slice of one row, in two passes.  The first keeps, in registers and without a
// barrier, the running maxima of fixed groups of columns (a thread's, or quarters of a thread's); the
// k-th largest of these maxima, rounded down to 16 bits, is a lower bound of the k-th best score.  The
// second reads the slice again, from L2 (slices are sized so that those at work fit), and collects what
// reaches the bound: k scores and a few more, unless many are equal.  A slice of one tile stays in
// registers between the passes.  If the buffer in shared memory overflows all the same, the slice is
// streamed a third time, the buffer cut to its k best by a radix selection (8-bit digits, from the top)
// whenever it might not take another tile; columns arrive in ascending order, so a score equal to the
// k-th has a higher id than the k keys it would have to beat and loses.
//
// Rows are cut into slices while there are fewer rows than CTAs to keep busy.  The k best of each
// slice then meet in a second launch, which selects among keys in the same way; it is launched before
// the first ends (programmatic dependent launch) and waits for it on the device.
#include <math_constants.h>

#include <type_traits>

#include "scores.cuh"

namespace coral {

namespace {

constexpr int kThreads = 512;
constexpr int kTile = 8192;                 // scores per step of a CTA
constexpr int kCap = kTile + kTopkMax;      // keys held in shared memory
constexpr int64_t kSliceBytes = 256 << 10;  // what two CTAs on every SM read twice fits L2

struct Shared {
    uint64_t keys[kCap];
    uint32_t hist[256];
    int cnt;
    int digit, above;     // the selection's current digit, keys above it
    float least;          // scores below it cannot be among the k best
};

template <typename T>
__device__ __forceinline__ float score_of(T v);
template <>
__device__ __forceinline__ float score_of<float>(float v) { return v; }
template <>
__device__ __forceinline__ float score_of<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float score_of<__half>(__half v) { return __half2float(v); }

__device__ __forceinline__ uint32_t ord_of(float s) {
    const uint32_t u = __float_as_uint(s + 0.f);      // one zero
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_ord(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
__device__ __forceinline__ float score_of_key(uint64_t k) { return of_ord((uint32_t)(k >> 32)); }

__device__ __forceinline__ uint64_t key_of(float s, uint32_t col) { return (uint64_t)ord_of(s) << 32 | (uint32_t)~col; }

// One step of a radix selection: warp 0 finds, from the histogram of a digit, the digit that holds
// the want-th largest key (sh.digit) and how many keys lie above it (sh.above).
__device__ __forceinline__ void pick_digit(Shared& sh, int want) {
    const int lane = threadIdx.x;     // lane l: digits 255 - 8 l .. 248 - 8 l, from the top
    uint32_t c[8], s = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += c[i] = sh.hist[255 - 8 * lane - i];
    uint32_t before = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
    }
    before -= s;          // keys with a digit above this lane's
    if (before < (uint32_t)want && before + s >= (uint32_t)want) {
        int i = 0;
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (i == j && before + c[j] < (uint32_t)want) {
                before += c[j];
                i = j + 1;
            }
        sh.digit = 255 - 8 * lane - i;
        sh.above = (int)before;
    }
}

template <typename T>
__device__ __forceinline__ T lowest_of();      // -inf
template <>
__device__ __forceinline__ float lowest_of<float>() { return -CUDART_INF_F; }
template <>
__device__ __forceinline__ __nv_bfloat16 lowest_of<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
template <>
__device__ __forceinline__ __half lowest_of<__half>() { return __ushort_as_half(0xfc00); }

// The larger of each of two pairs of 16-bit scores (NaN counts as nothing), and of the two of one.
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    } else {
        const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
}
template <typename T>
__device__ __forceinline__ float max_of(uint32_t m) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    else
        return fmaxf(__half2float(__ushort_as_half((unsigned short)m)), __half2float(__ushort_as_half((unsigned short)(m >> 16))));
}

// Cuts sh.keys[0..cnt) to its k largest (any order); all threads call it, cnt > k, keys distinct.
// Leaves k in sh.cnt and, in sh.least, the value just above the k-th largest's score.
__device__ void select_k(Shared& sh, int k) {
    const int tid = threadIdx.x, cnt = sh.cnt;
    uint64_t prefix = 0;          // digits of the k-th largest key found so far
    int want = k;                 // it is the want-th largest of the keys that share them
    int shift = 56;
    for (;; shift -= 8) {
        if (tid < 256) sh.hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < cnt; i += kThreads) {
            const uint64_t key = sh.keys[i];
            if (shift == 56 || (key >> (shift + 8)) == prefix) atomicAdd(&sh.hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid < 32) pick_digit(sh, want);
        __syncthreads();
        prefix = prefix << 8 | (uint64_t)sh.digit;
        want -= sh.above;
        const bool whole = sh.hist[sh.digit] == (uint32_t)want;   // the digit's keys are all wanted
        __syncthreads();
        if (whole || shift == 0) break;
    }
    // keys whose leading digits are >= prefix are exactly the k largest
    constexpr int kPer = (kCap + kThreads - 1) / kThreads;
    uint64_t mine[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine[i] = i * kThreads + tid < cnt ? sh.keys[i * kThreads + tid] : 0;
    if (tid == 0) sh.cnt = 0;
    __syncthreads();
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (mine[i] != 0 && (mine[i] >> shift) >= prefix) {
            sh.keys[atomicAdd(&sh.cnt, 1)] = mine[i];
            least = min(least, (uint32_t)(mine[i] >> 32));
        }
    least = __reduce_min_sync(0xffffffffu, least);
    if (tid < 256) sh.hist[tid] = 0xffffffffu;
    __syncthreads();
    if ((tid & 31) == 0) sh.hist[tid >> 5] = least;
    __syncthreads();
    if (tid < 32) {
        least = __reduce_min_sync(0xffffffffu, sh.hist[tid]);
        if (tid == 0) sh.least = of_ord(least + 1u);      // above +inf: NaN, which nothing reaches
    }
    __syncthreads();
}

// Writes the row's result, the k best of sh.keys[0..cnt): bitonic sort, descending.
__device__ void finish_row(Shared& sh, int q, const TopkArgs& a) {
    const int tid = threadIdx.x;
    if (sh.cnt > a.k && sh.cnt > 1024) select_k(sh, a.k);
    const int cnt = sh.cnt;
    int n2 = 32;
    while (n2 < cnt) n2 <<= 1;
    if (n2 <= kThreads) {      // a key a thread: partners nearer than a warp by shuffles
        uint64_t key = tid < cnt ? sh.keys[tid] : 0;
        for (int w = 2; w <= n2; w <<= 1)
            for (int j = w >> 1; j > 0; j >>= 1) {
                uint64_t other;
                if (j >= 32) {
                    __syncthreads();
                    sh.keys[tid] = key;
                    __syncthreads();
                    other = sh.keys[tid ^ j];
                } else {
                    other = __shfl_xor_sync(0xffffffffu, key, j);
                }
                const bool larger = ((tid & j) == 0) == ((tid & w) == 0);
                key = (key > other) == larger ? key : other;
            }
        __syncthreads();
        sh.keys[tid] = key;
    } else {
        for (int i = cnt + tid; i < n2; i += kThreads) sh.keys[i] = 0;
        __syncthreads();
        for (int w = 2; w <= n2; w <<= 1)
            for (int j = w >> 1; j > 0; j >>= 1) {
                for (int i = tid; i < n2; i += kThreads) {
                    const int p = i ^ j;
                    if (p > i) {
                        const uint64_t x = sh.keys[i], y = sh.keys[p];
                        if ((x < y) == ((i & w) == 0)) {
                            sh.keys[i] = y;
                            sh.keys[p] = x;
                        }
                    }
                }
                __syncthreads();
            }
    }
    __syncthreads();
    for (int i = tid; i < a.k; i += kThreads) {
        const bool there = i < cnt;
        const uint64_t key = there ? sh.keys[i] : 0;
        a.ids_out[(size_t)q * a.k + i] = there ? (int32_t)~(uint32_t)key + a.id_base : -1;
        a.scores_out[(size_t)q * a.k + i] = there ? score_of_key(key) : -3.402823466e+38f;
    }
}

// One tile in registers: U vectors of V scores a thread, vector u at column t0 + (u * kThreads + tid) * V.
// What lies past the slice's end reads -inf.
template <typename T, bool VEC>
struct Tile {
    static constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
    static constexpr int U = kTile / (kThreads * V);
    alignas(16) T v[U][V];

    __device__ __forceinline__ void load(const T* row, int64_t t0, int64_t c1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = t0 + (u * kThreads + threadIdx.x) * V;
            if (VEC && j + V <= c1) {
                *reinterpret_cast<uint4*>(v[u]) = *reinterpret_cast<const uint4*>(row + j);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[u][i] = j + i < c1 ? row[j + i] : lowest_of<T>();
            }
        }
    }
    __device__ __forceinline__ float best(int u) const {     // NaN counts as nothing
        if constexpr (VEC && sizeof(T) == 2) {
            const uint4 x = *reinterpret_cast<const uint4*>(v[u]);
            const uint32_t m = max2<T>(max2<T>(x.x, x.y), max2<T>(x.z, x.w));
            return max_of<T>(m);
        } else {
            float m = -CUDART_INF_F;
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, score_of<T>(v[u][i]));
            return m;
        }
    }
    // appends what reaches `least`; positions from kCap on are counted but not written
    __device__ __forceinline__ void collect(Shared& sh, float least, int64_t t0) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (best(u) >= least) {
                const int64_t j = t0 + (u * kThreads + threadIdx.x) * V;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float s = score_of<T>(v[u][i]);
                    if (s >= least) {
                        const int at = atomicAdd(&sh.cnt, 1);
                        if (at < kCap) sh.keys[at] = key_of(s, (uint32_t)(j + i));
                    }
                }
            }
    }
};

// Running maxima of four groups of a thread's columns: quarter g of its 16 scores of every tile.
template <typename T, bool VEC>
struct Maxima {
    static constexpr bool kPacked = VEC && sizeof(T) == 2;
    float m[kPacked ? 1 : 4];
    uint32_t p[kPacked ? 4 : 1];

    __device__ __forceinline__ Maxima() {
        if constexpr (kPacked) {
            const uint32_t none = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
            for (int g = 0; g < 4; ++g) p[g] = none;
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) m[g] = -CUDART_INF_F;
        }
    }
    __device__ __forceinline__ void add(const Tile<T, VEC>& t) {
        if constexpr (kPacked) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint4 x = *reinterpret_cast<const uint4*>(t.v[u]);
                p[2 * u] = max2<T>(p[2 * u], max2<T>(x.x, x.y));
                p[2 * u + 1] = max2<T>(p[2 * u + 1], max2<T>(x.z, x.w));
            }
        } else {
            constexpr int V = Tile<T, VEC>::V;
#pragma unroll
            for (int e = 0; e < 16; ++e) m[e / 4] = fmaxf(m[e / 4], score_of<T>(t.v[e / V][e % V]));
        }
    }
    __device__ __forceinline__ float group(int g) const {
        if constexpr (kPacked)
            return max_of<T>(p[g]);
        else
            return m[g];
    }
};

// Leaves in sh.least a lower bound of the k-th best score, from the maxima of all groups: the k-th
// largest, with the low 16 bits of its order cleared.  Two 8-bit digits of a radix selection.
template <typename T, bool VEC>
__device__ void first_threshold(Shared& sh, const Maxima<T, VEC>& maxima, int k) {
    const int tid = threadIdx.x;
    uint32_t o[4], top = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        o[g] = ord_of(maxima.group(g)) >> 16;
        top = max(top, o[g]);
    }
    const bool by_thread = k <= kThreads / 2;
    int want = k;
    uint32_t prefix = 0;
    for (int shift = 8; shift >= 0; shift -= 8) {
        if (tid < 256) sh.hist[tid] = 0;
        __syncthreads();
        if (by_thread) {
            if (shift == 8 || top >> 8 == prefix) atomicAdd(&sh.hist[(top >> shift) & 255], 1u);
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (shift == 8 || o[g] >> 8 == prefix) atomicAdd(&sh.hist[(o[g] >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid < 32) pick_digit(sh, want);
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)sh.digit;
        want -= sh.above;
        __syncthreads();
    }
    // never below the lowest finite score: -inf is not chosen
    if (tid == 0) sh.least = prefix <= ord_of(-3.402823466e+38f) >> 16 ? -3.402823466e+38f : of_ord(prefix << 16);
    __syncthreads();
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) topk_scan_kernel(const TopkArgs a, const int splits, const int64_t slice) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x;
    const int q = blockIdx.x / splits, part = blockIdx.x % splits;
    const int64_t c0 = part * slice;
    const int64_t c1 = c0 + slice < a.n ? c0 + slice : a.n;
    const T* row = static_cast<const T*>(a.in) + (size_t)q * a.ld;
    if (splits > 1) cudaTriggerProgrammaticLaunchCompletion();
    if (tid == 0) sh.cnt = 0;
    Tile<T, VEC> tile;
    if (c1 - c0 <= kTile) {
        tile.load(row, c0, c1);
        Maxima<T, VEC> maxima;
        maxima.add(tile);
        first_threshold(sh, maxima, a.k);
        tile.collect(sh, sh.least, c0);
    } else {
        Maxima<T, VEC> maxima;
#pragma unroll 2
        for (int64_t t0 = c0; t0 < c1; t0 += kTile) {
            tile.load(row, t0, c1);
            maxima.add(tile);
        }
        first_threshold(sh, maxima, a.k);
        const float least = sh.least;
#pragma unroll 2
        for (int64_t t0 = c0; t0 < c1; t0 += kTile) {
            tile.load(row, t0, c1);
            tile.collect(sh, least, t0);
        }
        __syncthreads();
        if (sh.cnt > kCap) {      // many equal scores
            __syncthreads();
            if (tid == 0) sh.cnt = 0;
            __syncthreads();
            for (int64_t t0 = c0; t0 < c1; t0 += kTile) {
                tile.load(row, t0, c1);
                tile.collect(sh, sh.least, t0);
                __syncthreads();
                const int cnt = sh.cnt;
                if (cnt > kCap - kTile) select_k(sh, a.k);     // no room for another tile
                else __syncthreads();
            }
        }
    }
    __syncthreads();
    if (splits == 1) {
        finish_row(sh, q, a);
    } else {
        if (sh.cnt > a.k) select_k(sh, a.k);
        uint64_t* mine = a.ws + ((size_t)q * splits + part) * a.k;
        for (int i = tid; i < a.k; i += kThreads) mine[i] = i < sh.cnt ? sh.keys[i] : 0;
    }
}

__global__ void __launch_bounds__(kThreads) topk_join_kernel(const TopkArgs a, const int splits) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x, q = blockIdx.x;
    const int total = splits * a.k;
    const uint64_t* keys = a.ws + (size_t)q * total;
    if (tid == 0) sh.cnt = 0;
    __syncthreads();
    cudaGridDependencySynchronize();
    for (int t0 = 0; t0 < total; t0 += kTile) {
        for (int i = t0 + tid; i < min(total, t0 + kTile); i += kThreads) {
            const uint64_t key = keys[i];
            if (key != 0) sh.keys[atomicAdd(&sh.cnt, 1)] = key;
        }
        __syncthreads();
        const int cnt = sh.cnt;
        __syncthreads();
        if (cnt > kCap - kTile) select_k(sh, a.k);
    }
    finish_row(sh, q, a);
}

int topk_splits(int Q, int64_t n, int k, int bytes, int sm_count) {
    const int64_t want = Q > 0 ? (int64_t)sm_count * 2 / Q : 1;
    const int64_t least = k > 256 ? 32 * (int64_t)k : kTile;     // a slice is worth its own selection
    int64_t s = (n + least - 1) / least;
    if (s > want) s = want;
    const int64_t fit = (n * bytes + kSliceBytes - 1) / kSliceBytes;
    if (s < fit) s = fit;
    return s < 1 ? 1 : (int)s;
}

template <typename T>
cudaError_t launch_topk_t(const TopkArgs& a, int splits, cudaStream_t stream) {
    const bool vec = ((uintptr_t)a.in | (uintptr_t)(a.ld * sizeof(T))) % 16 == 0;
    auto kernel = vec ? topk_scan_kernel<T, true> : topk_scan_kernel<T, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared));
    if (e != cudaSuccess) return e;
    // slices start at multiples of 8 scores, so 16-byte loads stay aligned
    const int64_t slice = ((a.n + splits - 1) / splits + 7) / 8 * 8;
    kernel<<<(unsigned)((int64_t)a.Q * splits), kThreads, sizeof(Shared), stream>>>(a, splits, slice);
    return cudaGetLastError();
}

}  // namespace

int64_t topk_workspace_bytes(int Q, int64_t n, int k, int sm_count) {
    const int s = topk_splits(Q, n, k, 4, sm_count);      // the wider the type, the more slices
    return s == 1 ? 0 : (int64_t)Q * s * k * 8;
}

cudaError_t launch_topk(const TopkArgs& a, int sm_count, cudaStream_t stream, int* launches) {
    const int splits = topk_splits(a.Q, a.n, a.k, type_bytes(a.type), sm_count);
    cudaError_t e = a.type == kTypeF32    ? launch_topk_t<float>(a, splits, stream)
                    : a.type == kTypeBf16 ? launch_topk_t<__nv_bfloat16>(a, splits, stream)
                                          : launch_topk_t<__half>(a, splits, stream);
    *launches = 1;
    if (e != cudaSuccess || splits == 1) return e;
    e = cudaFuncSetAttribute(topk_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.Q);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = stream;
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    *launches = 2;
    return cudaLaunchKernelEx(&cfg, topk_join_kernel, a, splits);
}

}  // namespace coral
