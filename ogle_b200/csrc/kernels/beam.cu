// A step of a beam search: the best continuations over all beams and tokens of a group.
//
// One pass over the logits: a block has a range of one row, in batches of 4 x 16 bytes a thread. It sums exp(x - m) for some m near the
// largest logit and keeps, in shared memory, the logits that may be among its best: those above a border that `count` of them
// are known to reach. The first border comes from the threads' own maxima: in each of the 8 warps the (count / 8)-th largest, where all
// have logits, the least of them. After 1, 2, 4, 8, ... batches what has been kept is ranked, and the count-th is the new border. A second,
// small launch adds the ranges' sums and picks a group's best of the ranges' lists. What the first has no room or no numbers for - rising
// rows, NaN, infinities, logits beyond 10^6 - it leaves to the second, which goes over such a range again (a row of 128000 in some 0.5 ms).
//
// Measured: 48 x 8 rows of 128001 in bf16, 98 MB, 16 best: 35 us for the rows, 2.8 TB/s (43 % of a copy), and 5 for the rest. 10 instructions a
// logit, and 24 warps an SM that wait for one another's: neither memory nor the exponentials (43 % of their unit) are the bound. One
// request of 4 x 32000 in fp32 takes 10 us on the device, 5 for each launch. (Everything kept at once ranked anew in each batch:
// 128 us; a call of the rare cases' code from the first launch, whose registers it then took: 80.)
//
// Which of two beams' tokens comes first hangs on the logarithms of their sums, to all bits that are left. So the totals are
// of 64 bits, and the sums nearly: exponents in one rounding, exponentials in fp32 - but those of the kept logits, which are most of a
// peaked row's sum, are put right in 64 bits at the end, unless a later batch rose far above the first -, a batch's sum of a thread in fp32, all
// others in 64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "pairs.cuh"

namespace ogle {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVecs = 4;                         // of 16 bytes, a thread's share of a batch
constexpr int kMostCount = 128, kMostEnds = 1024;
constexpr int kKept = 1024;                      // logits that a block keeps at most ...
constexpr int kRankAt = kThreads;                // ... and how many of them are ranked, once there are more: one a thread
constexpr int kLook = 8;                         // batches between two looks at that, at most
constexpr float kLargest = 3.402823466e38f;
constexpr float kSpread = 1.375f;                // of x above m: exponents stay below 2, and are rounded by 2^-24
constexpr float kTame = 1e6f;                    // logits beyond it are left to the second launch: fp32 has no exponent for x log2(e) - c there
constexpr float kNear = 100.f;                   // what is further below a row's largest logit has no part in its sum: 2^30 of exp(-100) are 2^-114

// A logit and its token in one number: the larger logit is the larger number, of equal ones the lower token. 0: none.
typedef unsigned long long Key;
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ Key key_of(float x, int token) {
    x += 0.f;                                    // -0 is 0
    return x > -INFINITY ? (Key)ordered(x) << 32 | (uint32_t)~token : 0ull;
}
__device__ __forceinline__ float logit_of(Key k) { return unordered(uint32_t(k >> 32)); }
__device__ __forceinline__ int token_of(Key k) { return int(~uint32_t(k)); }

// What a block leaves behind - a sum of exp(x - m), or kAgain: the range is to be gone over again -, followed by its `count` best in falling
// order (0: none). The sum of logits that are all -kTame or less is left at 0.
struct __align__(16) Part { double sum, m; };
constexpr double kAgain = -1.;
// Whether a range's sum is wanting: beside a row's largest logit `top`, with `best` the range's first key.
__device__ __forceinline__ bool sum_is_wanting(double sum, Key best, float top) { return !(sum >= 0.) || sum == 0. && best && logit_of(best) >= top - kNear; }
__host__ __device__ inline size_t part_bytes(int count) { return sizeof(Part) + ((size_t)count + 1) / 2 * 16; }

struct BeamArgs {
    OgleBeamParams p;
    int range, ranges;                           // logits of a block; blocks of a row
    int token_bits, beam_shift;                  // of Total::at
    unsigned char* parts;
};

// 16 bytes of logits.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int kN = 4;
    static constexpr float kMost = kLargest;
    static constexpr uint32_t kNothing = 0xff800000u;              // minus infinity
    static __device__ __forceinline__ float at(const uint4& v, int l) { return __uint_as_float(reinterpret_cast<const uint32_t*>(&v)[l]); }
    static __device__ __forceinline__ float at_any(const uint4& v, int l) {       // l known at run time alone
        return __uint_as_float(l & 2 ? (l & 1 ? v.w : v.z) : (l & 1 ? v.y : v.x));
    }
    static __device__ __forceinline__ float largest(const uint4& v) {      // NaN where one is
        float r = __uint_as_float(v.x);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(r) : "f"(__uint_as_float(v.y)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(r) : "f"(__uint_as_float(v.z)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(r) : "f"(__uint_as_float(v.w)));
        return r;
    }
};
template <> struct Vec<__half> {
    static constexpr int kN = 8;
    static constexpr float kMost = 65504.f;
    static constexpr uint32_t kNothing = 0xfc00fc00u;
    static __device__ __forceinline__ float at(const uint4& v, int l) { return __half2float(reinterpret_cast<const __half*>(&v)[l]); }
    static __device__ __forceinline__ float at_any(const uint4& v, int l) {
        const uint32_t w = l & 4 ? (l & 2 ? v.w : v.z) : (l & 2 ? v.y : v.x), h = l & 1 ? w >> 16 : w & 0xffffu;
        return __half2float(__ushort_as_half((unsigned short)h));
    }
    static __device__ __forceinline__ float largest(const uint4& v) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
        const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static constexpr float kMost = 3.38953139e38f;
    static constexpr uint32_t kNothing = 0xff80ff80u;
    static __device__ __forceinline__ float at(const uint4& v, int l) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(&v)[l / 2];
        return __uint_as_float(l % 2 ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ float at_any(const uint4& v, int l) {
        const uint32_t w = l & 4 ? (l & 2 ? v.w : v.z) : (l & 2 ? v.y : v.x), h = l & 1 ? w >> 16 : w & 0xffffu;
        return __uint_as_float(h << 16);
    }
    static __device__ __forceinline__ float largest(const uint4& v) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
    }
};

__device__ __forceinline__ float max_nan(float x, float y) {       // NaN where one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
// The logits of range r: the row begins `shift` elements behind a 16-byte boundary; a range is whole vectors between such boundaries.
template <typename T>
__device__ __forceinline__ void range_of(const BeamArgs& a, const T* row, int r, int& begin, int& end) {
    const int shift = int(reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (Vec<T>::kN - 1);
    begin = r * a.range - shift;
    end = min(begin + a.range, a.p.vocab);
}

// exp(x - m) as the sums have it: 2^(x log2(e) - c) in one rounding of the exponent, which is small where the weight is large. c is an fp32
// number, m what it stands for; log2(e) in fp32 makes a weight wrong by 2^-26 of its distance from m. What a sum is off by is at most
// 2^-19 of it: 2^-20 ln 2 where nearly all of it comes of alike logits 11 to 22 below m, all rounded alike, 2^-26 of that distance, 2^-22
// for the exponentials and six roundings of 2^-24 in fp32. Those of logits that differ are not alike, and cancel.
constexpr float kLog2e = 1.442695022f;
__device__ __forceinline__ float weight(float x, float c) { return exp2_fast(fmaf(x, kLog2e, -c)); }

// The kept logits in order: keys[0 .. n) become the `count` largest of them, falling; returns how many there are. All threads; what has been
// written to keys is there, and so is the result.
__device__ __forceinline__ int rank_kept(Key* keys, int n, int count) {
    const int tid = threadIdx.x;
    constexpr int kMine = kKept / kThreads;
    Key mine[kMine];
    int rank[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        mine[i] = tid + i * kThreads < n ? keys[tid + i * kThreads] : 0ull;
        rank[i] = 0;
    }
    if (n <= kThreads) {
        if (mine[0]) {
            const ulonglong2* const two = reinterpret_cast<const ulonglong2*>(keys);
#pragma unroll 4
            for (int j = 0; j + 1 < n; j += 2) {
                const ulonglong2 k = two[j / 2];
                rank[0] += (k.x > mine[0]) + (k.y > mine[0]);
            }
            if (n & 1) rank[0] += keys[n - 1] > mine[0];
        }
    } else {
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const Key k = keys[j];
#pragma unroll
            for (int i = 0; i < kMine; ++i) rank[i] += k > mine[i];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (mine[i] && rank[i] < count) keys[rank[i]] = mine[i];
    __syncthreads();
    return min(n, count);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) beam_rows_kernel(BeamArgs a) {
    using V = Vec<T>;
    constexpr int N = V::kN, kBatch = kThreads * kVecs * N;
    __shared__ __align__(16) Key kept[kKept];
    __shared__ int n_kept, first_equal;
    __shared__ double warp_m[kWarps], warp_sum[kWarps];
    __shared__ uint32_t warp_border[kWarps];
    __shared__ int warp_have[kWarps];
    const OgleBeamParams& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.y;
    if (tid == 0) n_kept = 0;
    grid_dependency_trigger();
    grid_dependency_wait();
    unsigned char* const out = a.parts + ((size_t)row * a.ranges + blockIdx.x) * part_bytes(p.count);
    const T* const in = static_cast<const T*>(p.logits) + row * p.logits_stride;
    int begin, end;
    range_of<T>(a, in, blockIdx.x, begin, end);
    const auto load = [&](int t0, uint4 (&v)[kVecs]) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int t = t0 + (u * kThreads + tid) * N;
            v[u] = make_uint4(V::kNothing, V::kNothing, V::kNothing, V::kNothing);
            if (t >= 0 && t + N <= end) {
                v[u] = __ldcs(reinterpret_cast<const uint4*>(in + t));
            } else if (t + N > 0 && t < end) {                     // the row's ends
#pragma unroll
                for (int l = 0; l < N; ++l)
                    if (t + l >= 0 && t + l < end) reinterpret_cast<T*>(&v[u])[l] = in[t + l];
            }
        }
    };
    const float score = p.scores ? p.scores[row] : 0.f;
    uint4 v[kVecs];
    if (begin < end) load(begin, v);             // (under way while the score is)
    if (begin >= end || !(fabsf(score) <= kLargest)) {             // behind the row's end, or of a beam that is none
        if (tid == 0) *reinterpret_cast<Part*>(out) = Part{0., 0.};
        for (int i = tid; i < p.count; i += kThreads) reinterpret_cast<Key*>(out + sizeof(Part))[i] = 0ull;
        return;
    }

    // The first batch's largest logits of all threads: m, and a border that `count` logits reach. (A NaN is the largest, and its range is gone
    // over again.)
    float c, fine_to, limit;                                       // weights are 2^(x log2(e) - c), for logits up to fine_to; what is above limit is kept
    const auto refer_to = [&](float m) {
        c = m > -kTame ? m * kLog2e : INFINITY;                    // (else nothing but a mask's lowest so far: no weight, no reference, a sum of 0)
        fine_to = m > -kTame ? fminf(m + kSpread, kTame) : -kTame;
    };
    uint32_t border = ~0u;
    {
        float top = V::largest(v[0]);
#pragma unroll
        for (int u = 1; u < kVecs; ++u) top = max_nan(top, V::largest(v[u]));
        // The k-th largest of each warp, or of all its threads that have a logit: with the least such k of which that is `count` threads. A short row
        // ends in a warp most of whose threads have none, and whose largest says little: where the other warps suffice it is left
        // out. (Of 1289 logits such a warp's border lets up to all pass: 22 to 31 us, 5 without it.)
        const uint32_t nothing = ordered(-INFINITY);
        uint32_t mine = ordered(top + 0.f), nth = 0;
        const int have = __popc(__ballot_sync(~0u, mine > nothing));
        if (lane == 0) warp_have[tid / 32] = have;
        __syncthreads();
        int k = 0, all = 0, least = 0;                              // least: threads that have logits, in a warp that counts
#pragma unroll
        for (int w = 0; w < kWarps; ++w) least = max(least, (warp_have[w] + 1) / 2);
        while (all < p.count) {
            if (k == 32) {
                if (least <= 1) break;
                least = 1;
            } else {
                ++k;
            }
            all = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) all += warp_have[w] >= least ? min(warp_have[w], k) : 0;
        }
        uint32_t best = nothing;
        for (int i = 0; i < min(k, have); ++i) {
            nth = __reduce_max_sync(~0u, mine);
            if (i == 0) best = nth;
            const unsigned who = __ballot_sync(~0u, mine == nth);
            if (lane == __ffs(who) - 1) mine = 0;
        }
        if (lane == 0) {
            warp_m[tid / 32] = (double)unordered(best);
            warp_border[tid / 32] = have > 0 && have >= least ? nth : ~0u;
        }
        __syncthreads();
        double m = -kLargest;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            m = fmax(m, warp_m[w]);
            border = min(border, warp_border[w]);
        }
        // the number below the border (below 0 comes -0, which is not less)
        limit = all >= p.count ? unordered(border - (border == 0x80000000u ? 2 : 1)) : -INFINITY;
        refer_to(fminf(float(m), V::kMost));
    }
    const float c0 = c;
    double sum = 0.;
    int n = 0;
    bool full = false, again = false;
#pragma unroll 1
    for (int t0 = begin, batch = 0; t0 < end; t0 += kBatch, ++batch) {
        uint4 next[kVecs];
        const bool last = t0 + kBatch >= end;
        if (!last) load(t0 + kBatch, next);
        float top[kVecs], most;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            top[u] = V::largest(v[u]);
            most = u == 0 ? top[0] : max_nan(most, top[u]);
        }
        if (!(most <= fine_to)) {                                  // far above m, or a NaN: rare
            if (most <= kTame) {
                const float before = c;
                refer_to(most);
                sum = before < INFINITY ? sum * exp2((double)before - (double)c) : 0.;
            } else {
                again = true;
            }
        }
        unsigned long long s[kVecs];                               // (a sum to a vector: none waits for another)
        const unsigned long long log2e = pair(kLog2e, kLog2e), minus_c = pair(-c, -c);
#pragma unroll
        for (int l = 0; l < N; l += 2)
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                float e, f;
                unpair(fma2(pair(V::at(v[u], l), V::at(v[u], l + 1)), log2e, minus_c), e, f);
                const unsigned long long w = pair(exp2_fast(e), exp2_fast(f));
                s[u] = l == 0 ? w : add2(s[u], w);
            }
        float e, f;
        unpair(add2(add2(s[0], s[1]), add2(s[2], s[3])), e, f);
        sum += (double)(e + f);
        // Kept: what is above the limit. (The second time round - of the first batch, most of which equals the border - of those that equal it
        // the first 256 tokens', where there are enough of them.)
        const auto keep = [&](int below) {
#pragma unroll
            for (int u = 0; u < kVecs; ++u)
                if (top[u] > limit) {
                    unsigned who = 0;
#pragma unroll
                    for (int l = 0; l < N; ++l) who |= unsigned(V::at(v[u], l) > limit) << l;
                    while (who) {                                  // most often one
                        const int l = __ffs(who) - 1, token = t0 + (u * kThreads + tid) * N + l;
                        who &= who - 1;
                        const float x = V::at_any(v[u], l);
                        if (token >= below && ordered(x + 0.f) == border) continue;
                        const int at = atomicAdd(&n_kept, 1);
                        if (at < kKept) kept[at] = key_of(x, token);
                        full |= at >= kRankAt;
                    }
                }
        };
        keep(0x7fffffff);
        // The first batch's border is a guess: the next one is as high as can be. It is raised when there is twice as much to go by.
        const bool raise = (batch & (batch + 1)) == 0 || last;
        if (raise || batch % kLook == 0) {
            if (__syncthreads_or(full || raise)) {
                n = n_kept;
                if (n > kKept && batch == 0) {
                    // many equal logits: what 256 tokens have of the border or more
                    const int below = begin + kThreads * N / 8;
                    __syncthreads();
                    if (tid == 0) n_kept = first_equal = 0;
                    __syncthreads();
                    if (tid < kThreads / 8) {
                        int mine = 0;
#pragma unroll
                        for (int l = 0; l < N; ++l) mine += V::at(v[0], l) > limit;
                        atomicAdd(&first_equal, mine);
                    }
                    __syncthreads();
                    keep(first_equal >= p.count ? below : 0x7fffffff);
                    __syncthreads();
                    n = n_kept;
                }
                if (n > kKept) {                                   // no room: the range is gone over again
                    again = true;
                    limit = INFINITY;
                    n = 0;
                    __syncthreads();                               // everybody has seen the number
                } else {
                    n = rank_kept(kept, n, p.count);
                    // what equals the border later comes behind `count` that do, whose tokens are lower
                    if (limit < INFINITY) limit = n == p.count ? logit_of(kept[n - 1]) : -INFINITY;
                }
                if (tid == 0) n_kept = n;
                __syncthreads();
            }
            full = false;
        }
#pragma unroll
        for (int u = 0; u < kVecs; ++u) v[u] = next[u];
    }

    // logits just above -kTame: those below it, whose weight was taken for 0, would count beside them
    if (n > 0) {
        const float best = logit_of(kept[0]);
        again |= best > -kTame && best < kNear - kTame;
    }
    // the kept logits' part of the sum in 64 bits, where all threads have the same c
    const double inverse = 1. / (double)kLog2e;
    const bool same = __syncthreads_and(c == c0);
    double top = c < INFINITY ? (double)c * inverse : -INFINITY;
    if (same) {
        if (tid < n && c < INFINITY) {
            const float x = logit_of(kept[tid]);
            sum += exp((double)x - top) - (double)weight(x, c);
        }
    } else {
#pragma unroll
        for (int d = 16; d; d /= 2) top = fmax(top, __shfl_xor_sync(~0u, top, d));
        if (lane == 0) warp_m[tid / 32] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmax(top, warp_m[w]);
        sum = c < INFINITY ? sum * exp((double)c * inverse - top) : 0.;
    }
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0) warp_sum[tid / 32] = sum;
    const bool redo = __syncthreads_or(again);
    if (tid == 0) {
        double all = 0.;
        for (int w = 0; w < kWarps; ++w) all += warp_sum[w];
        *reinterpret_cast<Part*>(out) = Part{redo ? kAgain : all, top > -INFINITY ? top : 0.};
    }
    for (int i = tid; i < p.count; i += kThreads) reinterpret_cast<Key*>(out + sizeof(Part))[i] = i < n ? kept[i] : 0ull;
}

// ---- the groups
// A total as a whole number of the same order, and where it comes from, the lower the better: beam, logit (turned round), token. Beside a score or a
// logit of 10^20 64 bits have nothing left of a beam's other differences: the logits still tell. (Three numbers to a total: 2 us more.)
struct __align__(16) Total { unsigned long long value, at; };
// The bits are enough for all of the logit up to 2^32 beams x tokens; beyond that its last ones are left out.
__device__ __forceinline__ unsigned long long place_of(const BeamArgs& a, int beam, Key k) {
    const uint32_t logit = ~uint32_t(k >> 32) >> (32 + a.token_bits - a.beam_shift);
    return (unsigned long long)beam << a.beam_shift | (unsigned long long)logit << a.token_bits | (uint32_t)token_of(k);
}
__device__ __forceinline__ int beam_of(const BeamArgs& a, const Total& t) { return int(t.at >> a.beam_shift); }
__device__ __forceinline__ int token_of(const BeamArgs& a, const Total& t) { return int(t.at & ((1ull << a.token_bits) - 1)); }
__device__ __forceinline__ unsigned long long ordered(double x) {
    const unsigned long long u = __double_as_longlong(x + 0.);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double unordered(unsigned long long u) { return __longlong_as_double(u >> 63 ? u & ~(1ull << 63) : ~u); }
__device__ __forceinline__ bool better(const Total& x, const Total& y) { return x.value > y.value || x.value == y.value && x.at < y.at; }

constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 32, kPicked = 1024;
constexpr int kMostBeams = 1024;

// Goes over a range again, whatever its logits are: their sum in 64 bits; the count-th largest bit by bit, what is above it, and of those that
// equal it the first. All threads; `found` is theirs to use.
template <typename T>
__device__ __noinline__ void again(const BeamArgs& a, const T* row, int r, unsigned char* out, Total* found) {
    __shared__ double sums[kPickWarps];
    __shared__ int counts[2][kPickWarps];
    __shared__ int n_found, before[kPickWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, count = a.p.count;
    int begin, end;
    range_of(a, row, r, begin, end);
    begin = max(begin, 0);
    const auto at = [&](int t) {                                   // minus infinity for a NaN
        const float x = float(row[t]);
        return x == x ? fminf(x, Vec<T>::kMost) + 0.f : -INFINITY;
    };
    float top = -INFINITY;
#pragma unroll 8
    for (int t = begin + tid; t < end; t += kPickThreads) top = fmaxf(top, at(t));
#pragma unroll
    for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    __syncthreads();
    if (lane == 0) sums[warp] = (double)top;
    __syncthreads();
    for (int w = 0; w < kPickWarps; ++w) top = fmaxf(top, float(sums[w]));
    __syncthreads();
    double sum = 0.;
    if (top > -INFINITY)
#pragma unroll 4
        for (int t = begin + tid; t < end; t += kPickThreads) sum += exp((double)at(t) - (double)top);
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0) sums[warp] = sum;
    uint32_t border = 0;
    int more = 0;                                                  // above the border
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t next = border | 1u << bit;
        int c = 0;
#pragma unroll 8
        for (int t = begin + tid; t < end; t += kPickThreads) {
            const float x = at(t);
            c += x > -INFINITY && ordered(x) >= next;
        }
        c = __reduce_add_sync(~0u, c);
        if (lane == 0) counts[bit & 1][warp] = c;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < kPickWarps; ++w) all += counts[bit & 1][w];
        if (all >= count) border = next;
        else more = all;                                           // (the last one that is too high: the next number above the border)
    }
    // in the tokens' order, so that the first come first; at most count of them
    Key* const keys = reinterpret_cast<Key*>(found);
    if (tid == 0) n_found = 0;
    int equal = border ? count - more : 0;
    if (border == 0) equal = 0;
    __syncthreads();
    for (int t0 = begin; t0 < end; t0 += kPickThreads) {
        const int t = t0 + tid;
        const float x = t < end ? at(t) : -INFINITY;
        const uint32_t mine = x > -INFINITY ? ordered(x) : 0u;
        const bool is = border && mine == border;
        const unsigned who = __ballot_sync(~0u, is);
        if (lane == 0) before[warp] = __popc(who);
        __syncthreads();
        int place = __popc(who & ((1u << lane) - 1)), all = 0;
        for (int w = 0; w < kPickWarps; ++w) {
            if (w < warp) place += before[w];
            all += before[w];
        }
        if (mine > border || is && place < equal) keys[atomicAdd(&n_found, 1)] = key_of(x, t);
        equal = max(equal - all, 0);
        __syncthreads();
    }
    const int n = n_found;
    for (int i = tid; i < count; i += kPickThreads) {
        Key mine = 0ull;
        int rank = i;
        if (i < n) {
            mine = keys[i];
            rank = 0;
            for (int j = 0; j < n; ++j) rank += keys[j] > mine;
        }
        reinterpret_cast<Key*>(out + sizeof(Part))[rank] = mine;
    }
    if (tid == 0) {
        sum = 0.;
        for (int w = 0; w < kPickWarps; ++w) sum += sums[w];
        *reinterpret_cast<Part*>(out) = Part{sum, top > -INFINITY ? (double)top : 0.};
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(BeamArgs a) {
    extern __shared__ double2 beam_terms[];                        // of each beam: its largest logit m, and log sum exp(x - m); then score minus that
    __shared__ Total found[kPicked];
    __shared__ Total best[kMostCount];
    __shared__ unsigned warp_border[kPickWarps];
    __shared__ Total warp_best[kPickWarps];
    __shared__ int n_found;
    const OgleBeamParams& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = blockIdx.x;
    const size_t stride = part_bytes(p.count);
    if (tid == 0) n_found = 0;
    grid_dependency_trigger();
    grid_dependency_wait();
    unsigned char* const parts = a.parts + (size_t)g * p.beams * a.ranges * stride;
    const int lists = p.beams * a.ranges, all = lists * p.count;
    // Candidate i is the (i / lists)-th of list i % lists: the lists' best come first, and neighbours are of different lists.
    const auto key_at = [&](int i, int& list) {
        const int place = i / lists;
        list = i - place * lists;
        return reinterpret_cast<const Key*>(parts + list * stride + sizeof(Part))[place];
    };
    int my_list = 0;
    Key my_key = tid < all ? key_at(tid, my_list) : 0ull;          // under way while the sums are added
    for (int round = 0; round < 2; ++round) {
        bool redo = false;
        for (int b = warp; b < p.beams; b += kPickWarps) {
            const unsigned char* const mine = parts + (size_t)b * a.ranges * stride;
            float top = -INFINITY;
            Part part = {0., 0.};
            for (int r = lane; r < a.ranges; r += 32) {
                const Key k = *reinterpret_cast<const Key*>(mine + r * stride + sizeof(Part));
                if (r == lane) part = *reinterpret_cast<const Part*>(mine + r * stride);
                if (k) top = fmaxf(top, logit_of(k));
            }
#pragma unroll
            for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            double sum = 0.;
            for (int r = lane; r < a.ranges; r += 32) {
                if (r != lane) part = *reinterpret_cast<const Part*>(mine + r * stride);
                if (part.sum > 0.) sum += part.sum * exp(part.m - (double)top);
                else redo |= sum_is_wanting(part.sum, *reinterpret_cast<const Key*>(mine + r * stride + sizeof(Part)), top);
            }
#pragma unroll
            for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
            if (lane == 0) beam_terms[b] = make_double2(top, sum > 0. ? log(sum) : 0.);
        }
        if (!__syncthreads_or(redo) || round > 0) break;
        for (int list = 0; list < lists; ++list) {
            const int b = list / a.ranges;
            unsigned char* const part = parts + list * stride;
            if (sum_is_wanting(reinterpret_cast<const Part*>(part)->sum, *reinterpret_cast<const Key*>(part + sizeof(Part)), float(beam_terms[b].x))) {
                const size_t row = (size_t)(g * p.beams + b) * p.logits_stride;
                if (p.dtype == OGLE_F32) again(a, static_cast<const float*>(p.logits) + row, list - b * a.ranges, part, found);
                else if (p.dtype == OGLE_F16) again(a, static_cast<const __half*>(p.logits) + row, list - b * a.ranges, part, found);
                else again(a, static_cast<const __nv_bfloat16*>(p.logits) + row, list - b * a.ranges, part, found);
            }
        }
        __syncthreads();
        my_key = tid < all ? key_at(tid, my_list) : 0ull;
    }
    // Two beams of the same logits differ in their sums' errors, twice 2^-19 at most, where their rows lie differently to 16 bytes. They count as
    // the same, so that their totals are equal and come in the beams' order; so does what is as near by chance.
    constexpr int kMine = (kMostBeams + kPickThreads - 1) / kPickThreads;
    double minus[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int b = tid + i * kPickThreads;
        if (b >= p.beams) break;
        const double2 term = beam_terms[b];
        minus[i] = term.y;
        for (int o = 0; o < b; ++o)
            if (beam_terms[o].x == term.x && fabs(beam_terms[o].y - term.y) <= 0x1p-18) {
                minus[i] = beam_terms[o].y;
                break;
            }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int b = tid + i * kPickThreads;
        if (b < p.beams) beam_terms[b].y = (p.scores ? (double)p.scores[g * p.beams + b] : 0.) - minus[i];
    }
    __syncthreads();
    const auto total = [&](Key k, int list) {
        const int b = list / a.ranges;
        const double2 term = beam_terms[b];
        return Total{ordered(term.y + ((double)logit_of(k) - term.x)), place_of(a, b, k)};
    };
    // A border that `count` of them reach, by the upper half of the totals' bits: the count-th of the threads', among which the lists' best are,
    // bit by bit; or, where the threads have them all and a low border costs little, that of some warp's. (One request of four beams over
    // 32000 tokens, 256 candidates: 11.2 us on the device with the first, 9.6 with the second.)
    const Total my_total = my_key ? total(my_key, my_list) : Total{0ull, ~0ull};
    const unsigned upper = unsigned(my_total.value >> 32);
    unsigned border = 0;
    if (all > kPickThreads || p.count > 16) {
#pragma unroll 1
        for (unsigned bit = 1u << 31; bit; bit >>= 1)
            if (__syncthreads_count(upper >= (border | bit)) >= p.count) border |= bit;
    } else if (all > 32) {
        unsigned mine = upper, nth = 0;
        for (int i = 0; i < p.count; ++i) {
            nth = __reduce_max_sync(~0u, mine);
            const unsigned who = __ballot_sync(~0u, mine == nth);
            if (lane == __ffs(who) - 1) mine = 0;
        }
        if (lane == 0) warp_border[warp] = nth;
        __syncthreads();
        for (int w = 0; w < kPickWarps; ++w) border = max(border, warp_border[w]);
    }
    const auto offer = [&](const Total& t) {
        const bool in = unsigned(t.value >> 32) >= border;
        if (in) {
            const int at = atomicAdd(&n_found, 1);
            if (at < kPicked) found[at] = t;
        }
        return in;
    };
    if (my_key) offer(my_total);
    // what the threads have not looked at yet, a list to a thread: it falls, and ends where it has fallen below the border
    for (int list = tid; list < lists && all > kPickThreads; list += kPickThreads)
        for (int place = list < kPickThreads ? (kPickThreads - list + lists - 1) / lists : 0; place < p.count; ++place) {
            const Key k = reinterpret_cast<const Key*>(parts + list * stride + sizeof(Part))[place];
            if (!k || !offer(total(k, list))) break;
        }
    __syncthreads();
    int n = n_found;
    if (n <= kPicked) {
        for (int i = tid; i < n; i += kPickThreads) {
            const Total mine = found[i];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) rank += better(found[j], mine);
            if (rank < p.count) best[rank] = mine;
        }
        n = min(n, p.count);
    } else {
        // too many alike: the best, the best of the rest, ...
        Total last = {~0ull, 0ull};
        for (int k = 0; k < p.count; ++k) {
            Total mine = {0ull, ~0ull};
            for (int i = tid; i < all; i += kPickThreads) {
                int list;
                const Key key = key_at(i, list);
                if (!key) continue;
                const Total t = total(key, list);
                if (better(last, t) && better(t, mine)) mine = t;
            }
#pragma unroll
            for (int d = 16; d; d /= 2) {
                const Total o = {__shfl_xor_sync(~0u, mine.value, d), __shfl_xor_sync(~0u, mine.at, d)};
                if (better(o, mine)) mine = o;
            }
            if (lane == 0) warp_best[warp] = mine;
            __syncthreads();
            last = warp_best[0];
            for (int w = 1; w < kPickWarps; ++w)
                if (better(warp_best[w], last)) last = warp_best[w];
            __syncthreads();
            if (tid == 0) best[k] = last;
        }
        n = p.count;
    }
    __syncthreads();
    for (int i = tid; i < p.count; i += kPickThreads) {
        const bool there = i < n;
        p.out_score[(size_t)g * p.count + i] = there ? float(unordered(best[i].value)) : -INFINITY;
        p.out_beam[(size_t)g * p.count + i] = there ? beam_of(a, best[i]) : -1;
        p.out_token[(size_t)g * p.count + i] = there ? token_of(a, best[i]) : -1;
    }
    // the first of them that are no end token, in order: a warp looks at 32 at a time
    if (warp == 0) {
        int next = 0;
        for (int i0 = 0; i0 < n && next < p.beams; i0 += 32) {
            const int i = i0 + lane;
            bool goes_on = i < n;
            int beam = 0, token = 0;
            if (goes_on) {
                beam = beam_of(a, best[i]);
                token = token_of(a, best[i]);
                for (int e = 0; e < p.n_ends; ++e) goes_on &= __ldg(p.ends + e) != token;
            }
            const unsigned who = __ballot_sync(~0u, goes_on);
            const int at = next + __popc(who & ((1u << lane) - 1));
            if (goes_on && at < p.beams) {
                p.next_row[(size_t)g * p.beams + at] = g * p.beams + beam;
                p.next_token[(size_t)g * p.beams + at] = token;
                p.next_score[(size_t)g * p.beams + at] = float(unordered(best[i].value));
            }
            next += __popc(who);
        }
        for (int i = next + lane; i < p.beams; i += 32) {
            p.next_row[(size_t)g * p.beams + i] = p.next_token[(size_t)g * p.beams + i] = -1;
            p.next_score[(size_t)g * p.beams + i] = -INFINITY;
        }
    }
}

// ---- host
int check(const OgleBeamParams* p) {
    if (!p || p->n_groups < 0 || p->beams < 1 || p->vocab < 0 || p->count < 1 || p->n_ends < 0 || p->dtype < OGLE_F32 || p->dtype > OGLE_BF16) return OGLE_ERR_INVALID;
    if (p->count > kMostCount || p->beams > kMostBeams || p->n_ends > kMostEnds || p->vocab > (1 << 30) || (long long)p->n_groups * p->beams > 65535) return OGLE_ERR_UNSUPPORTED;
    if (p->n_groups * p->beams > 1 && p->logits_stride < p->vocab) return OGLE_ERR_INVALID;
    return OGLE_OK;
}
// A block's logits and how many blocks a row has: as many as one round of them (three to an SM) has for it, whole batches each.
void split(const OgleBeamParams* p, int& range, int& ranges) {
    const int n = p->dtype == OGLE_F32 ? 4 : 8, batch = kThreads * kVecs * n;
    const long batches = div_up((long)p->vocab + n - 1, batch), rows = (long)p->n_groups * p->beams;
    long blocks = rows > 0 ? 3L * kNumSMs / rows : 1;
    if (blocks < 1) blocks = 1;
    const long each = batches > 0 ? div_up(batches, blocks) : 1;
    range = int(each * batch);
    ranges = batches > 0 ? div_up(batches, each) : 1;
}

}  // namespace
}  // namespace ogle

using namespace ogle;

extern "C" {

size_t ogle_cuda_beam_step_workspace_bytes(const OgleBeamParams* p) {
    if (check(p) != OGLE_OK) return 0;
    int range, ranges;
    split(p, range, ranges);
    return (size_t)p->n_groups * p->beams * ranges * part_bytes(p->count);
}

int ogle_cuda_beam_step(const OgleBeamParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream) {
    const int rc = check(p);
    if (rc != OGLE_OK) return rc;
    if (p->n_groups == 0) return OGLE_OK;
    if ((!p->logits && p->vocab > 0) || (p->n_ends > 0 && !p->ends) || !p->out_score || !p->out_beam || !p->out_token || !p->next_row || !p->next_token || !p->next_score || !workspace)
        return OGLE_ERR_INVALID;
    if (!aligned16(workspace)) return OGLE_ERR_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(p->logits) % (p->dtype == OGLE_F32 ? 4 : 2) != 0) return OGLE_ERR_ALIGNMENT;
    if (workspace_bytes < ogle_cuda_beam_step_workspace_bytes(p)) return OGLE_ERR_INVALID;
    BeamArgs a = {};
    a.p = *p;
    split(p, a.range, a.ranges);
    int beam_bits = 0;
    while ((1LL << a.token_bits) < p->vocab) ++a.token_bits;
    while ((1 << beam_bits) < p->beams) ++beam_bits;
    a.beam_shift = 32 + a.token_bits < 64 - beam_bits ? 32 + a.token_bits : 64 - beam_bits;
    a.parts = static_cast<unsigned char*>(workspace);
    const dim3 grid(a.ranges, p->n_groups * p->beams);
    cudaError_t e;
    if (p->dtype == OGLE_F32) e = launch_overlapped(beam_rows_kernel<float>, grid, dim3(kThreads), 0, stream, a);
    else if (p->dtype == OGLE_F16) e = launch_overlapped(beam_rows_kernel<__half>, grid, dim3(kThreads), 0, stream, a);
    else e = launch_overlapped(beam_rows_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, stream, a);
    int done = OGLE_OK;
    if (e == cudaSuccess) {
        done = finish_launch();
        if (done != OGLE_OK) return done;
        e = launch_overlapped_if(overlapped_launches_enabled(true), beam_pick_kernel, dim3(p->n_groups), dim3(kPickThreads), p->beams * sizeof(double2), stream, a);
    }
    if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
    return finish_launch();
}

}  // extern "C"
