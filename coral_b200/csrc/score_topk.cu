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
// reaches the bound: k scores and a few more, unless many are equal.  It only notes the 16-byte vectors
// that hold such a score; the whole CTA then takes the noted ones apart at once.  A slice of one step (128 bytes a
// thread, all in flight at once) stays in registers between the passes.  If the buffer in shared memory
// overflows all the same, the second pass is repeated with the buffer cut to its k best by a radix
// selection (8-bit digits, from the top) whenever it might not take what comes next; columns arrive in
// ascending order, so a score equal to the k-th has a higher id than the k keys it would have to beat
// and loses.
//
// Rows are cut into slices while there are fewer rows than CTAs to keep busy.  What the slices collect
// then meets in a second launch, which finds its bound among keys in the same way; it is launched
// before the first ends (programmatic dependent launch) and waits for it on the device.
//
// Measured: 256 x 128000 bf16, k = 100: 20 us, of which the first pass takes 8 to 11 (65.5 MB at up to
// 6 TB/s), the bound 2, the second pass 4.5, the order 1.5; one pass against a running threshold, with
// the buffer cut now and then, took 45 us, because nearly every warp then held something to append.
// 1 x 1M fp32, k = 10: 7.4 us in two launches; k = 1000: 35 us (9 more with one key a thread in flight in
// the second).
#include <math_constants.h>

#include <type_traits>

#include "scores.cuh"

namespace coral {

namespace {

constexpr int kThreads = 512;
constexpr int kRoom = 8192;                 // keys that may arrive between two looks at the buffer
constexpr int kCap = kRoom + kTopkMax;      // keys held in shared memory
constexpr int kNotes = 4096;                // vectors noted
constexpr int64_t kSliceBytes = 256 << 10;  // what two CTAs on every SM read twice fits L2

struct Shared {
    uint64_t keys[kCap];
    uint32_t notes[kNotes];
    uint32_t hist[256];
    int cnt, noted;
    int digit, above;     // the selection's current digit, keys above it
    uint32_t top;         // the largest maximum
    float least;          // scores below it cannot be among the k best
};

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
__device__ __noinline__ void select_k(Shared& sh, int k) {
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

// Writes the row's result, the k best of sh.keys[0..cnt), in order.
__device__ void finish_row(Shared& sh, int q, const TopkArgs& a) {
    const int tid = threadIdx.x;
    if (sh.cnt > a.k && sh.cnt > 1024) select_k(sh, a.k);
    const int cnt = sh.cnt;
    auto write = [&](int rank, uint64_t key) {
        a.ids_out[(size_t)q * a.k + rank] = key ? (int32_t)~(uint32_t)key + a.id_base : -1;
        a.scores_out[(size_t)q * a.k + rank] = key ? score_of_key(key) : -3.402823466e+38f;
    };
    int n2 = 32;
    while (n2 < cnt) n2 <<= 1;
    if (n2 <= kThreads) {
        // a key's place is the number of larger keys; kThreads / n2 threads share the count of one
        const int mine = tid & (n2 - 1), part = tid / n2, parts = kThreads / n2;
        if (tid < n2) sh.notes[tid] = 0;
        const uint64_t key = mine < cnt ? sh.keys[mine] : 0;
        const int from = cnt * part / parts, to = cnt * (part + 1) / parts;
        int larger = 0;
#pragma unroll 8
        for (int i = from; i < to; ++i) larger += sh.keys[i] > key ? 1 : 0;
        __syncthreads();
        if (key) atomicAdd(&sh.notes[mine], (uint32_t)larger);
        __syncthreads();
        if (part == 0 && key && sh.notes[mine] < (uint32_t)a.k) write((int)sh.notes[mine], key);
    } else {
        // bitonic, descending; thread t holds keys 2 t and 2 t + 1, partners in its warp by shuffles
        __syncthreads();
        uint64_t x = 2 * tid < cnt ? sh.keys[2 * tid] : 0, y = 2 * tid + 1 < cnt ? sh.keys[2 * tid + 1] : 0;
        for (int w = 2; w <= 2 * kThreads; w <<= 1) {
            const bool down = (2 * tid & w) == 0;
            for (int j = w >> 1; j > 1; j >>= 1) {
                uint64_t ox, oy;
                if (j >= 64) {
                    __syncthreads();
                    sh.keys[2 * tid] = x;
                    sh.keys[2 * tid + 1] = y;
                    __syncthreads();
                    ox = sh.keys[2 * tid ^ j];
                    oy = sh.keys[(2 * tid + 1) ^ j];
                } else {
                    ox = __shfl_xor_sync(0xffffffffu, x, j >> 1);
                    oy = __shfl_xor_sync(0xffffffffu, y, j >> 1);
                }
                const bool larger = ((2 * tid & j) == 0) == down;
                x = (x > ox) == larger ? x : ox;
                y = (y > oy) == larger ? y : oy;
            }
            if ((x < y) == down) {
                const uint64_t z = x;
                x = y;
                y = z;
            }
        }
        if (2 * tid < min(cnt, a.k)) write(2 * tid, x);
        if (2 * tid + 1 < min(cnt, a.k)) write(2 * tid + 1, y);
    }
    for (int i = cnt + tid; i < a.k; i += kThreads) write(i, 0);
}

// Leaves in sh.least a lower bound of the k-th best score, from the maxima of disjoint groups of scores:
// o[0..4) are the high halves of the orders of four groups' maxima.  Bins of a histogram count maxima
// by their distance from the largest, at full resolution first, where nearly always at least k of them
// lie within its 255 bins, else 16 and 256 times coarser.
__device__ __forceinline__ void lower_bound_of_kth(Shared& sh, const uint32_t (&o)[4], int k) {
    const int tid = threadIdx.x;
    const uint32_t top = max(max(o[0], o[1]), max(o[2], o[3]));
    const bool by_thread = k <= kThreads / 2;      // else the quarters are needed
    if (tid == 0) sh.top = 0;
    if (tid < 256) sh.hist[tid] = 0;
    __syncthreads();
    const uint32_t warp_top = __reduce_max_sync(0xffffffffu, top);
    if ((tid & 31) == 0) atomicMax(&sh.top, warp_top);
    __syncthreads();
    const uint32_t hi = sh.top;
    uint32_t bound = 0;
    for (int shift = 0; shift <= 8; shift += 4) {
        if (by_thread) {
            const uint32_t d = (hi - top) >> shift;
            if (d < 255) atomicAdd(&sh.hist[255 - d], 1u);
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t d = (hi - o[g]) >> shift;
                if (d < 255) atomicAdd(&sh.hist[255 - d], 1u);
            }
        }
        if (tid == 0) sh.digit = 0;
        __syncthreads();
        if (tid < 32) pick_digit(sh, k);
        __syncthreads();
        const int digit = sh.digit;
        if (digit) {
            const uint32_t below = (uint32_t)(256 - digit) << shift;      // everything in the bin is nearer than this
            bound = hi >= below ? hi - below + 1 : 0;
            break;
        }
        if (tid < 256) sh.hist[tid] = 0;
        __syncthreads();
    }
    // never below the lowest finite score: -inf is not chosen
    if (tid == 0) sh.least = bound <= ord_of(-3.402823466e+38f) >> 16 ? -3.402823466e+38f : of_ord(bound << 16);
    __syncthreads();
}

// One step in registers: U vectors of V scores a thread, vector u at t0 + (u * kThreads + tid) * V of the
// slice's whole 16-byte vectors.  What lies past their end reads -inf.
template <typename T>
struct Step {
    static constexpr int V = 16 / (int)sizeof(T);
    static constexpr int U = 8;
    static constexpr int kScores = kThreads * U * V;
    static constexpr bool kPairs = sizeof(T) == 2;
    union {
        uint4 raw[U];
        T v[U][V];
    };

    __device__ __forceinline__ Step() {}
    __device__ __forceinline__ void load(const T* cols, int t0, int end) {
        constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = t0 + (u * kThreads + (int)threadIdx.x) * V;
            raw[u] = make_uint4(none, none, none, none);
            if (j < end) raw[u] = *reinterpret_cast<const uint4*>(cols + j);
        }
    }
    __device__ __forceinline__ float best(int u) const {     // NaN counts as nothing
        if constexpr (kPairs)
            return max_of<T>(max2<T>(max2<T>(raw[u].x, raw[u].y), max2<T>(raw[u].z, raw[u].w)));
        else
            return fmaxf(fmaxf(fmaxf(-CUDART_INF_F, v[u][0]), fmaxf(v[u][1], v[u][2])), v[u][3]);
    }
    __device__ __forceinline__ uint32_t reaching(float least) const {      // bit u: vector u holds such a score
        uint32_t hits = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) hits |= best(u) >= least ? 1u << u : 0u;
        return hits;
    }
};

__device__ __forceinline__ void append(Shared& sh, float s, uint32_t col) {      // counted, but not written, from kCap on
    const int at = atomicAdd(&sh.cnt, 1);
    if (at < kCap) sh.keys[at] = key_of(s, col);
}

// Notes the flagged vectors of a step by number; counted, but not written, from kNotes on.
template <typename T>
__device__ __forceinline__ void note(Shared& sh, uint32_t hits, int t0) {
    for (; hits; hits &= hits - 1) {
        const int at = atomicAdd(&sh.noted, 1);
        if (at < kNotes) sh.notes[at] = t0 / Step<T>::V + (__ffs(hits) - 1) * kThreads + threadIdx.x;
    }
}

// Appends the scores that reach `least` of the noted vectors, an element a thread.
template <typename T>
__device__ __forceinline__ void collect(Shared& sh, int noted, float least, const T* cols, uint32_t c0) {
    constexpr int V = Step<T>::V;
    for (int i = threadIdx.x; i < noted * V; i += kThreads) {
        const int j = (int)sh.notes[i / V] * V + i % V;
        const float s = to_f32<T>(cols[j]);
        if (s >= least) append(sh, s, c0 + (uint32_t)j);
    }
}

// Running maxima of four groups of a thread's columns: vectors g and g + 4 (g, g + 4, ...) of every step.
template <typename T>
struct Maxima {
    static constexpr bool kPairs = Step<T>::kPairs;
    float m[4];
    uint32_t p[4];

    __device__ __forceinline__ Maxima() {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            m[g] = -CUDART_INF_F;
            p[g] = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
        }
    }
    __device__ __forceinline__ void add(const Step<T>& t) {
#pragma unroll
        for (int u = 0; u < Step<T>::U; ++u) {
            if constexpr (kPairs)
                p[u & 3] = max2<T>(p[u & 3], max2<T>(max2<T>(t.raw[u].x, t.raw[u].y), max2<T>(t.raw[u].z, t.raw[u].w)));
            else
                m[u & 3] = fmaxf(m[u & 3], t.best(u));
        }
    }
    __device__ __forceinline__ uint32_t high(int g) const { return ord_of(kPairs ? fmaxf(m[g], max_of<T>(p[g])) : m[g]) >> 16; }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
topk_scan_kernel(const TopkArgs a, const int splits, const int64_t slice, const int slots) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    using Scores = Step<T>;
    const int tid = threadIdx.x;
    const int q = blockIdx.x / splits, part = blockIdx.x % splits;
    // Columns [c0, c0 + len) of the row: `head` of them up to a 16-byte boundary, whole vectors to `end`
    // (counted from the boundary), and what is left; a thread each for the odd ones.
    const int64_t row0 = part * slice;
    const int len = row0 < a.n ? (int)(row0 + slice < a.n ? slice : a.n - row0) : 0;
    const T* first = static_cast<const T*>(a.in) + (size_t)q * a.ld + row0;
    const int head = min(len, (int)((16 - ((uintptr_t)first & 15)) % 16 / sizeof(T)));
    const int end = (len - head) / Scores::V * Scores::V, left = len - head - end;
    const T* cols = first + head;
    const uint32_t c0 = (uint32_t)(row0 + head);
    if (splits > 1) cudaTriggerProgrammaticLaunchCompletion();
    if (tid == 0) sh.cnt = sh.noted = 0;
    const int odd = tid < head ? tid - head : end + tid - 32;      // from the boundary
    const bool has_odd = tid < head || (tid >= 32 && tid - 32 < left);
    const float rest = has_odd ? to_f32<T>(cols[odd]) : -CUDART_INF_F;
    Scores step;
    Maxima<T> maxima;
    for (int t0 = 0; t0 < end; t0 += Scores::kScores) {
        step.load(cols, t0, end);
        maxima.add(step);
    }
    maxima.m[0] = fmaxf(maxima.m[0], rest);
    const uint32_t high[4] = {maxima.high(0), maxima.high(1), maxima.high(2), maxima.high(3)};
    lower_bound_of_kth(sh, high, a.k);
    const float bound = sh.least;
    const bool in_registers = end <= Scores::kScores;
    for (int t0 = 0; t0 < end; t0 += Scores::kScores) {
        if (!in_registers) step.load(cols, t0, end);
        note<T>(sh, step.reaching(bound), t0);
    }
    __syncthreads();
    const int noted = sh.noted;
    if (noted <= kNotes) collect<T>(sh, noted, bound, cols, c0);
    if (has_odd && rest >= bound) append(sh, rest, c0 + (uint32_t)odd);
    __syncthreads();
    if (noted > kNotes || sh.cnt > kCap) {
        // many equal scores: a vector a thread at a time, the buffer cut whenever the next might not fit
        __syncthreads();
        if (tid == 0) sh.cnt = 0;
        __syncthreads();
        for (int t0 = 0; t0 < len; t0 += kThreads * Scores::V) {
            const float least = sh.least;
            for (int i = 0; i < Scores::V; ++i) {
                const int j = t0 + tid * Scores::V + i;
                const float s = j < len ? to_f32<T>(first[j]) : -CUDART_INF_F;
                if (s >= least) append(sh, s, (uint32_t)(row0 + j));
            }
            __syncthreads();
            const int cnt = sh.cnt;
            __syncthreads();
            if (cnt > kCap - kRoom) select_k(sh, a.k);
        }
    }
    __syncthreads();
    if (splits == 1) {
        finish_row(sh, q, a);
    } else {
        if (sh.cnt > slots) select_k(sh, a.k);
        uint64_t* mine = a.ws + ((size_t)q * splits + part) * slots;
        for (int i = tid; i < slots; i += kThreads) mine[i] = i < sh.cnt ? sh.keys[i] : 0;
    }
}

__global__ void __launch_bounds__(kThreads) topk_join_kernel(const TopkArgs a, const int splits, const int slots) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x, q = blockIdx.x;
    const int total = splits * slots;
    const uint64_t* keys = a.ws + (size_t)q * total;
    if (tid == 0) sh.cnt = 0;
    cudaGridDependencySynchronize();
    uint32_t high[4] = {0, 0, 0, 0};
#pragma unroll 2
    for (int i = tid; i < total; i += 4 * kThreads)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (i + g * kThreads < total) high[g] = max(high[g], (uint32_t)(keys[i + g * kThreads] >> 48));
    lower_bound_of_kth(sh, high, a.k);
    const uint32_t least = ord_of(sh.least);
    for (int careful = 0; careful < 2; ++careful) {
        for (int i0 = 0; i0 < total; i0 += kRoom) {
            constexpr int kTogether = 4;      // loads in flight
            static_assert(kRoom % (kTogether * kThreads) == 0, "rounds");
            for (int i1 = i0 + tid; i1 < min(total, i0 + kRoom); i1 += kTogether * kThreads) {
                uint64_t key[kTogether];
#pragma unroll
                for (int u = 0; u < kTogether; ++u) key[u] = i1 + u * kThreads < total ? keys[i1 + u * kThreads] : 0;
#pragma unroll
                for (int u = 0; u < kTogether; ++u)
                    if ((uint32_t)(key[u] >> 32) >= least) {
                        const int at = atomicAdd(&sh.cnt, 1);
                        if (at < kCap) sh.keys[at] = key[u];
                    }
            }
            if (careful) {
                __syncthreads();
                const int cnt = sh.cnt;
                __syncthreads();
                if (cnt > kCap - kRoom) select_k(sh, a.k);
            }
        }
        __syncthreads();
        const int cnt = sh.cnt;
        __syncthreads();
        if (cnt <= kCap) break;
        if (tid == 0) sh.cnt = 0;
        __syncthreads();
    }
    finish_row(sh, q, a);
}

// Keys a slice may leave: with some room above k, few slices need a selection of their own.  The bound is
// the looser the larger k (30 x 1M fp32, k = 1000: 68 us with a half, 73 with a quarter; 1 x 1M, k = 10:
// 0.2 us more with a half).
int slots_of(int k) { return k + (k > 256 ? k / 2 : k / 4) + 16; }

int topk_splits(int Q, int64_t n, int k, int bytes, int sm_count) {
    const int64_t want = Q > 0 ? (int64_t)sm_count * 2 / Q : 1;
    const int64_t least = k > 256 ? 48 * (int64_t)k : kRoom;     // a slice is worth its own selection (48 k
    // columns; 32 k: 1 x 1M fp32, k = 1000 38 us for 35; 64 k: 10 x 100k, k = 1000 25.7 for 24.1)
    int64_t s = (n + least - 1) / least;
    if (s > want) s = want;
    const int64_t fit = (n * bytes + kSliceBytes - 1) / kSliceBytes;
    if (s < fit) s = fit;
    return s < 1 ? 1 : (int)s;
}

template <typename T>
cudaError_t launch_topk_t(const TopkArgs& a, int splits, cudaStream_t stream) {
    auto kernel = topk_scan_kernel<T>;
    static std::atomic<uint64_t> granted;
    cudaError_t e = grant_smem(kernel, (int)sizeof(Shared), granted);
    if (e != cudaSuccess) return e;
    // slices start at multiples of 8 scores: as far from a 16-byte boundary as their row
    const int64_t slice = ((a.n + splits - 1) / splits + 7) / 8 * 8;
    kernel<<<(unsigned)((int64_t)a.Q * splits), kThreads, sizeof(Shared), stream>>>(a, splits, slice, slots_of(a.k));
    return cudaGetLastError();
}

}  // namespace

int64_t topk_workspace_bytes(int Q, int64_t n, int k, int sm_count) {
    const int s = topk_splits(Q, n, k, 4, sm_count);      // the wider the type, the more slices
    return s == 1 ? 0 : (int64_t)Q * s * slots_of(k) * 8;
}

cudaError_t launch_topk(const TopkArgs& a, int sm_count, cudaStream_t stream, int* launches) {
    const int splits = topk_splits(a.Q, a.n, a.k, type_bytes(a.type), sm_count);
    cudaError_t e = a.type == kTypeF32    ? launch_topk_t<float>(a, splits, stream)
                    : a.type == kTypeBf16 ? launch_topk_t<__nv_bfloat16>(a, splits, stream)
                                          : launch_topk_t<__half>(a, splits, stream);
    *launches = 1;
    if (e != cudaSuccess || splits == 1) return e;
    static std::atomic<uint64_t> granted;
    e = grant_smem(topk_join_kernel, (int)sizeof(Shared), granted);
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
    return cudaLaunchKernelEx(&cfg, topk_join_kernel, a, splits, slots_of(a.k));
}

}  // namespace coral
