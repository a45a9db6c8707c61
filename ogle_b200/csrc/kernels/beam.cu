// A step of a beam search: the best continuations over all beams and tokens of a group.
//
// One pass over the logits: a block has a range of one row, in batches of 4 x 16 bytes a thread. It sums exp(x - m) for some m near the
// largest logit and keeps, in shared memory, the logits that may be among its best: those above a border that `count` of them
// are known to reach. The first border comes from the threads' own maxima: in each of the 8 warps the (count / 8)-th largest, the least of
// them. Whenever more than a few hundred have gathered, they are ranked and the count-th is the new border. A second, small launch
// adds the ranges' sums and picks a group's best of the ranges' lists.
//
// Which of two beams' tokens comes first hangs on the logarithms of their sums, to all bits that are left. So the totals are
// of 64 bits, and the sums nearly: x - m times log2(e) in two parts, exponentials in fp32 - but those of the kept logits, which are most of a
// peaked row's sum, are put right in 64 bits at the end -, a batch's sum of a thread in fp32, all others in 64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ogle {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVecs = 4;                         // of 16 bytes, a thread's share of a batch
constexpr int kMostCount = 128, kMostEnds = 1024;
constexpr int kKept = 1024;                      // logits that a block keeps at most ...
constexpr int kRankAt = 512;                     // ... and how many of them are ranked at the end of a batch
constexpr float kLargest = 3.402823466e38f;
static_assert(kRankAt + kMostCount <= kKept, "what the slow way adds to the kept");

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

// What a block leaves behind, followed by its `count` best in falling order (0: none).
struct __align__(16) Part { double sum; float m; int unused; };
__host__ __device__ inline size_t part_bytes(int count) { return sizeof(Part) + ((size_t)count + 1) / 2 * 16; }

struct BeamArgs {
    OgleBeamParams p;
    int range, ranges;                           // logits of a block; blocks of a row
    unsigned char* parts;
};

template <typename T> struct Vec { static constexpr int kN = 16 / sizeof(T); };
template <typename T> __device__ __forceinline__ float largest_of();
template <> __device__ __forceinline__ float largest_of<float>() { return kLargest; }
template <> __device__ __forceinline__ float largest_of<__half>() { return 65504.f; }
template <> __device__ __forceinline__ float largest_of<__nv_bfloat16>() { return 3.38953139e38f; }

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[Vec<T>::kN]) {
    const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int l = 0; l < Vec<T>::kN; ++l) x[l] = float(h[l]);
}
__device__ __forceinline__ float max_nan(float a, float b) {       // NaN where one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// exp(x - m) as the sums have it.
__device__ __forceinline__ float weight(float x, float m) {
    const float d = x - m, t = fmaf(d, 1.925963033e-8f, d * 1.442695022f);
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
    return y;
}

// The kept logits in order: keys[0 .. n) become the `count` largest of them, falling; returns how many there are. All threads.
__device__ __noinline__ int rank_kept(Key* keys, int n, int count, int* scratch) {
    const int tid = threadIdx.x;
    Key mine[kKept / kThreads];
    int rank[kKept / kThreads];
    int there = 0;
    __syncthreads();
    if (tid == 0) *scratch = 0;
#pragma unroll
    for (int i = 0; i < kKept / kThreads; ++i) {
        mine[i] = tid + i * kThreads < n ? keys[tid + i * kThreads] : 0ull;
        rank[i] = 0;
        there += mine[i] != 0;
    }
    __syncthreads();
    if (n <= kThreads) {
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank[0] += keys[j] > mine[0];
    } else {
        for (int j = 0; j < n; ++j) {
            const Key k = keys[j];
#pragma unroll
            for (int i = 0; i < kKept / kThreads; ++i) rank[i] += k > mine[i];
        }
    }
    if (there) atomicAdd(scratch, there);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKept / kThreads; ++i)
        if (mine[i] && rank[i] < count) keys[rank[i]] = mine[i];
    const int all = min(*scratch, count);
    __syncthreads();
    return all;
}

// The largest key that `count` keys of the batch reach, 0 where there are fewer: bit by bit. For batches most of which pass the border - many
// equal logits, or a rising row. All threads; `f` counts a thread's keys from a given one on.
template <typename F>
__device__ __forceinline__ Key border_of_batch(int count, int* sums, F f) {
    Key border = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
        const Key next = border | 1ull << bit;
        const int n = __reduce_add_sync(~0u, f(next));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sums[threadIdx.x / 32] = n;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) all += sums[w];
        if (all >= count) border = next;
    }
    return border;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) beam_rows_kernel(BeamArgs a) {
    constexpr int N = Vec<T>::kN, kBatch = kThreads * kVecs * N;
    __shared__ __align__(16) Key kept[kKept];
    __shared__ int n_kept, scratch, sums[kWarps];
    __shared__ float warp_m[kWarps];
    __shared__ uint32_t warp_border[kWarps];
    __shared__ double warp_sum[kWarps];
    const OgleBeamParams& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.y;
    if (tid == 0) n_kept = 0;
    grid_dependency_trigger();
    grid_dependency_wait();
    unsigned char* const out = a.parts + ((size_t)row * a.ranges + blockIdx.x) * part_bytes(p.count);
    const T* const in = static_cast<const T*>(p.logits) + row * p.logits_stride;
    // the row begins `shift` elements behind a 16-byte boundary; a range is whole vectors between such boundaries
    const int shift = int(reinterpret_cast<uintptr_t>(in) / sizeof(T)) & (N - 1);
    const int begin = blockIdx.x * a.range - shift, end = min(begin + a.range, p.vocab);
    const float score = p.scores ? p.scores[row] : 0.f;
    if (begin >= end || !(fabsf(score) <= kLargest)) {             // behind the row's end, or of a beam that is none
        if (tid == 0) *reinterpret_cast<Part*>(out) = Part{0., -INFINITY, 0};
        for (int i = tid; i < p.count; i += kThreads) reinterpret_cast<Key*>(out + sizeof(Part))[i] = 0ull;
        return;
    }
    const uint32_t nothing = sizeof(T) == 4 ? 0xff800000u : (largest_of<T>() < 1e5f ? 0xfc00fc00u : 0xff80ff80u);      // minus infinity
    const auto load = [&](int t0, uint4 (&v)[kVecs]) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int t = t0 + (u * kThreads + tid) * N;
            v[u] = make_uint4(nothing, nothing, nothing, nothing);
            if (t >= 0 && t + N <= end) {
                v[u] = __ldcs(reinterpret_cast<const uint4*>(in + t));
            } else if (t + N > 0 && t < end) {                     // the row's ends
#pragma unroll
                for (int l = 0; l < N; ++l)
                    if (t + l >= 0 && t + l < end) reinterpret_cast<T*>(&v[u])[l] = in[t + l];
            }
        }
    };

    const int of_warp = (p.count + kWarps - 1) / kWarps;
    uint4 v[kVecs];
    load(begin, v);
    float m = 0.f, m0 = 0.f, border = -INFINITY;
    double sum = 0.;
#pragma unroll 1
    for (int t0 = begin; t0 < end; t0 += kBatch) {
        uint4 next[kVecs];
        if (t0 + kBatch < end) load(t0 + kBatch, next);
        const auto largest = [&] {
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                float x[N];
                unpack<T>(v[u], x);
#pragma unroll
                for (int l = 0; l < N; ++l) top = max_nan(top, x[l]);
            }
            return top;
        };
        float top = largest();
        if (!(top <= kLargest)) {                                  // a NaN or an infinity: rare
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                T* const h = reinterpret_cast<T*>(&v[u]);
#pragma unroll
                for (int l = 0; l < N; ++l) {
                    const float x = float(h[l]);
                    if (x != x) h[l] = T(-INFINITY);
                    else if (x > kLargest) h[l] = T(largest_of<T>());
                }
            }
            top = largest();
        }
        const bool first = t0 == begin;
        if (first) {
            uint32_t mine = ordered(top + 0.f), best = 0, nth = 0;
            for (int i = 0; i < of_warp; ++i) {
                nth = __reduce_max_sync(~0u, mine);
                if (i == 0) best = nth;
                const unsigned who = __ballot_sync(~0u, mine == nth);
                if (lane == __ffs(who) - 1) mine = 0;
            }
            if (lane == 0) {
                warp_m[tid / 32] = unordered(best);
                warp_border[tid / 32] = of_warp <= 32 ? nth : 0;
            }
            __syncthreads();
            uint32_t least = ~0u;
            m = -kLargest;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                m = fmaxf(m, warp_m[w]);
                least = min(least, warp_border[w]);
            }
            m0 = m;
            // (below: a logit of minus infinity never passes)
            border = least > ordered(-INFINITY) ? unordered(least) : -INFINITY;
        }
        if (top - m > 40.f) {                                      // sums stay below 2^58 of 2^127
            sum *= exp((double)m - (double)top);
            m = top;
        }
        float s[kVecs];
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            float x[N];
            unpack<T>(v[u], x);
            s[u] = 0.f;
#pragma unroll
            for (int l = 0; l < N; ++l) s[u] += weight(x[l], m);
        }
        sum += (double)((s[0] + s[1]) + (s[2] + s[3]));
        bool full = false;
        // of a later batch what equals the border comes behind `count` that do and are of lower tokens
        const auto passes = [&](float x) { return x > border || first && x == border && x > -INFINITY; };
        if (passes(top)) {
#pragma unroll
            for (int u = 0; u < kVecs; ++u) {
                float x[N];
                unpack<T>(v[u], x);
#pragma unroll
                for (int l = 0; l < N; ++l)
                    if (passes(x[l])) {
                        const int at = atomicAdd(&n_kept, 1);
                        if (at < kKept) kept[at] = key_of(x[l], t0 + (u * kThreads + tid) * N + l);
                        full |= at >= kRankAt;
                    }
            }
        }
        if (__syncthreads_or(full)) {
            int n = n_kept;
            const bool lost = n > kKept;
            if (lost) {
                // the batch again: what came before it, then as many of it as can count
                for (int i = tid; i < kKept; i += kThreads)
                    if (token_of(kept[i]) >= t0) kept[i] = 0ull;
                n = rank_kept(kept, kKept, p.count, &scratch);
                if (tid == 0) n_kept = n;
                const auto each = [&](auto f) {
#pragma unroll
                    for (int u = 0; u < kVecs; ++u) {
                        float x[N];
                        unpack<T>(v[u], x);
#pragma unroll
                        for (int l = 0; l < N; ++l) f(key_of(x[l], t0 + (u * kThreads + tid) * N + l));
                    }
                };
                const Key from = border_of_batch(p.count, sums, [&](Key k) {
                    int c = 0;
                    each([&](Key mine) { c += mine >= k; });
                    return c;
                });
                each([&](Key mine) {
                    // (fewer than count in the batch: all that there are)
                    if (mine != 0 && mine >= from) {
                        const int at = atomicAdd(&n_kept, 1);
                        if (at < kKept) kept[at] = mine;
                    }
                });
                __syncthreads();
                n = n_kept;
            }
            n = rank_kept(kept, min(n, kKept), p.count, &scratch);
            if (tid == 0) n_kept = n;
            if (n == p.count) border = logit_of(kept[n - 1]);
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < kVecs; ++u) v[u] = next[u];
    }

    __syncthreads();
    const int n = rank_kept(kept, n_kept, p.count, &scratch);
    // the kept logits' part of the sum in 64 bits, where all threads have the same m
    const bool same = __syncthreads_and(m == m0);
    if (same && tid < n) {
        const float x = logit_of(kept[tid]);
        sum += exp((double)x - (double)m) - (double)weight(x, m);
    }
    float top = m;
#pragma unroll
    for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    if (lane == 0) warp_m[tid / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w]);
    if (top != m) sum *= exp((double)m - (double)top);
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0) warp_sum[tid / 32] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.;
        for (int w = 0; w < kWarps; ++w) sum += warp_sum[w];
        *reinterpret_cast<Part*>(out) = Part{sum, top, 0};
    }
    for (int i = tid; i < p.count; i += kThreads) reinterpret_cast<Key*>(out + sizeof(Part))[i] = i < n ? kept[i] : 0ull;
}

// ---- the groups
struct Total { double value; unsigned long long at; };             // at: beam * vocab + token
__device__ __forceinline__ bool better(const Total& x, const Total& y) { return x.value > y.value || x.value == y.value && x.at < y.at; }

constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 32, kPicked = 1024;
constexpr int kMostBeams = 1024;

__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(BeamArgs a) {
    extern __shared__ double2 beam_terms[];                        // of each beam: its largest logit m, and log sum exp(x - m)
    __shared__ Total found[kPicked];
    __shared__ Total best[kMostCount];
    __shared__ double warp_value[kPickWarps];
    __shared__ unsigned long long warp_at[kPickWarps];
    __shared__ int n_found;
    const OgleBeamParams& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = blockIdx.x;
    const size_t stride = part_bytes(p.count);
    if (tid == 0) n_found = 0;
    grid_dependency_trigger();
    grid_dependency_wait();
    const unsigned char* const parts = a.parts + (size_t)g * p.beams * a.ranges * stride;
    for (int b = warp; b < p.beams; b += kPickWarps) {
        const unsigned char* const mine = parts + (size_t)b * a.ranges * stride;
        float top = -INFINITY;
        for (int r = lane; r < a.ranges; r += 32) {
            const Key k = *reinterpret_cast<const Key*>(mine + r * stride + sizeof(Part));
            if (k) top = fmaxf(top, logit_of(k));
        }
#pragma unroll
        for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        double sum = 0.;
        for (int r = lane; r < a.ranges; r += 32) {
            const Part part = *reinterpret_cast<const Part*>(mine + r * stride);
            if (part.sum > 0.) sum += part.sum * exp((double)part.m - (double)top);
        }
#pragma unroll
        for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
        if (lane == 0) beam_terms[b] = make_double2(top, sum > 0. ? log(sum) : 0.);    // no sum: no kept logit either
    }
    __syncthreads();
    // Two beams of the same logits differ in the last bits of their sums where their rows lie differently to 16 bytes. They count as the same,
    // so that their totals are equal and come in the beams' order; so does what is as near by chance.
    constexpr int kMine = (kMostBeams + kPickThreads - 1) / kPickThreads;
    double minus[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int b = tid + i * kPickThreads;
        if (b >= p.beams) break;
        const double2 term = beam_terms[b];
        minus[i] = term.y;
        for (int o = 0; o < b; ++o)
            if (beam_terms[o].x == term.x && fabs(beam_terms[o].y - term.y) <= 0x1p-22) {
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
    const int lists = p.beams * a.ranges, all = lists * p.count;
    const auto total = [&](int i, Total& t) {                      // candidate i; false where there is none
        const int list = i / p.count, b = list / a.ranges;
        const Key k = reinterpret_cast<const Key*>(parts + list * stride + sizeof(Part))[i - list * p.count];
        if (!k) return false;
        const double2 term = beam_terms[b];
        t.value = term.y + ((double)logit_of(k) - term.x);
        t.at = (unsigned long long)b * p.vocab + token_of(k);
        return true;
    };
    // a border that `count` of them reach, from the threads' own best as above
    double border = -INFINITY;
    if (all > kPickThreads) {
        double mine = -INFINITY;
        Total t;
        for (int i = tid; i < all; i += kPickThreads)
            if (total(i, t)) mine = fmax(mine, t.value);
        double nth = -INFINITY;
        for (int i = 0; i < (p.count + kPickWarps - 1) / kPickWarps; ++i) {
            nth = mine;
#pragma unroll
            for (int d = 16; d; d /= 2) nth = fmax(nth, __shfl_xor_sync(~0u, nth, d));
            const unsigned who = __ballot_sync(~0u, mine == nth);
            if (lane == __ffs(who) - 1) mine = -INFINITY;
        }
        if (lane == 0) warp_value[warp] = nth;
        __syncthreads();
        border = warp_value[0];
        for (int w = 1; w < kPickWarps; ++w) border = fmin(border, warp_value[w]);
    }
    for (int i = tid; i < all; i += kPickThreads) {
        Total t;
        if (total(i, t) && t.value >= border) {
            const int at = atomicAdd(&n_found, 1);
            if (at < kPicked) found[at] = t;
        }
    }
    __syncthreads();
    int n = n_found;
    if (n <= kPicked) {
        for (int i = tid; i < n; i += kPickThreads) {
            const Total mine = found[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += better(found[j], mine);
            if (rank < p.count) best[rank] = mine;
        }
        n = min(n, p.count);
    } else {
        // too many equal ones: the best, the best of the rest, ...
        Total last = {INFINITY, 0ull};
        for (int k = 0; k < p.count; ++k) {
            Total mine = {-INFINITY, ~0ull}, t;
            for (int i = tid; i < all; i += kPickThreads)
                if (total(i, t) && better(last, t) && better(t, mine)) mine = t;
#pragma unroll
            for (int d = 16; d; d /= 2) {
                const Total o = {__shfl_xor_sync(~0u, mine.value, d), __shfl_xor_sync(~0u, mine.at, d)};
                if (better(o, mine)) mine = o;
            }
            if (lane == 0) { warp_value[warp] = mine.value; warp_at[warp] = mine.at; }
            __syncthreads();
            last = Total{warp_value[0], warp_at[0]};
            for (int w = 1; w < kPickWarps; ++w) {
                const Total o = {warp_value[w], warp_at[w]};
                if (better(o, last)) last = o;
            }
            __syncthreads();
            if (tid == 0) best[k] = last;
        }
        n = p.count;
    }
    __syncthreads();
    for (int i = tid; i < p.count; i += kPickThreads) {
        const bool there = i < n;
        p.out_score[(size_t)g * p.count + i] = there ? float(best[i].value) : -INFINITY;
        p.out_beam[(size_t)g * p.count + i] = there ? int(best[i].at / p.vocab) : -1;
        p.out_token[(size_t)g * p.count + i] = there ? int(best[i].at % p.vocab) : -1;
    }
    // the first of them that are no end token, in order: a warp looks at 32 at a time
    if (warp == 0) {
        int next = 0;
        for (int i0 = 0; i0 < n && next < p.beams; i0 += 32) {
            const int i = i0 + lane;
            bool goes_on = i < n;
            int beam = 0, token = 0;
            if (goes_on) {
                beam = int(best[i].at / p.vocab);
                token = int(best[i].at % p.vocab);
                for (int e = 0; e < p.n_ends; ++e) goes_on &= __ldg(p.ends + e) != token;
            }
            const unsigned who = __ballot_sync(~0u, goes_on);
            const int at = next + __popc(who & ((1u << lane) - 1));
            if (goes_on && at < p.beams) {
                p.next_row[(size_t)g * p.beams + at] = g * p.beams + beam;
                p.next_token[(size_t)g * p.beams + at] = token;
                p.next_score[(size_t)g * p.beams + at] = float(best[i].value);
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
