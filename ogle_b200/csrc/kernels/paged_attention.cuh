// What the forms of attention over the paged cache share.
#pragma once
#include "paged.cuh"
#include "tc_common.cuh"
#include "tma_host.h"

namespace ogle {
namespace paged {

constexpr int kChunk = 16;                       // keys of a warp's step; a page holds whole steps
constexpr int kGaveUp = 9;                       // in the library's device status word: a copy or a product did not come
constexpr float kHeadroom = 8.f;                 // a row's m moves only when an x exceeds it by more: w stays below 2^(8 + 7)
constexpr float kLift = 7.f;                     // of all weights, away from fp16's smallest numbers

struct AttnArgs {
    Batch b;
    const void* q;
    void* out;
    float* lse;
    long long q_row, q_head, out_row, out_head;
    float scale_log2;
    int causal, window;
    float* parts;                                // [ranges][2][kRows] x (DP + 2)
    struct Cut* cuts;                            // [ranges]
    int few_limit;                               // sequences of more rows x query heads of a group are the prompt form's; 0: all are one form's
    int by_segment;                              // tiles of rows a sequence can have, where cuts are kept by segment; else 0
    int cluster;                                 // blocks of a cluster that has one segment, or 0: ranges
    uint32_t spin_limit;
    int* error;
};

// What the join needs of a segment that was cut. rows 0: it was not. Kept by segment where there are fewer segments than
// ranges, else by the range that the segment begins in, its last.
struct __align__(16) Cut {
    int rows, row0, h, m0;         // rows of the tile; row of the sequence's first row; kv head; the tile's first row
    int first, last;               // ranges [first, last) have parts ...
    int gaps, unused;              // ... but for those that have no tile, where there are more ranges than tiles
    long long total;               // tiles of all segments
};

// A 64-bit division takes some hundred instructions, one in 32 bits twenty: nearly all are of small numbers.
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ int row_tiles(const Batch& a, int n, int rows) { return (n * a.group + rows - 1) / rows; }

// Keys that some row of the sequence attends: [lo, hi), lo down to a tile.
struct Span { int lo, hi; };
__device__ __forceinline__ Span span_of(const paged::Sequence& s, int first_row, int last_row, int causal, int window) {
    Span k;
    k.hi = causal ? min(s.len, s.first + last_row + 1) : s.len;
    k.lo = window > 0 ? max(0, max(s.first + first_row, 0) - window + 1) : 0;        // any window: the difference of two that are not negative
    k.hi = max(k.hi, 0);
    return k;
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int element, int token, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(element), "r"(token), "r"(head), "r"(page) : "memory");
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What rounding to fp16 left over, as fp16 again.
__device__ __forceinline__ uint32_t rest_bits(uint32_t rounded, float lo, float hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
    return half2_bits(lo - f.x, hi - f.y);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 numbers at a time.
__device__ __forceinline__ unsigned long long pair(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpair(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Four values of a row of the result from its weighted sum v, its m and its sum of weights; with the first four, its lse.
__device__ __forceinline__ void store_row(const AttnArgs& a, long long row, int head, int d, float4 v, float m, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;             // no weight: no token attended
    v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
    if (d < a.b.dim) {
        const long long y = row * a.out_row + head * a.out_head + d;
        if (a.b.dtype == OGLE_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + y) = v;
        } else {
            uint2 z;
            if (a.b.dtype == OGLE_F16) {
                z.x = half2_bits(v.x, v.y); z.y = half2_bits(v.z, v.w);
            } else {
                const __nv_bfloat162 e = __floats2bfloat162_rn(v.x, v.y), f = __floats2bfloat162_rn(v.z, v.w);
                z.x = *reinterpret_cast<const uint32_t*>(&e); z.y = *reinterpret_cast<const uint32_t*>(&f);
            }
            *reinterpret_cast<uint2*>(static_cast<unsigned short*>(a.out) + y) = z;
        }
    }
    if (d == 0 && a.lse) a.lse[row * a.b.q_heads + head] = sum == 0.f ? -INFINITY : (m - kLift + log2f(sum)) * 0.6931471805599453f;
}

// 16 values of a row from element d on, as fp32; zeros behind the head's end.
__device__ __forceinline__ void load16(const void* q, long long at, int d, int dim, int dtype, float* f) {
    if (d >= dim) {
#pragma unroll
        for (int l = 0; l < 16; ++l) f[l] = 0.f;
    } else if (dtype == OGLE_F32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at + d);
#pragma unroll
        for (int l = 0; l < 4; ++l) {
            const float4 v = p[l];
            f[4 * l] = v.x; f[4 * l + 1] = v.y; f[4 * l + 2] = v.z; f[4 * l + 3] = v.w;
        }
    } else {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(q) + at + d);
        const uint4 v[2] = {p[0], p[1]};
        const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
#pragma unroll
        for (int l = 0; l < 8; ++l) {
            const float2 g = dtype == OGLE_F16 ? __half22float2(*reinterpret_cast<const __half2*>(w + l)) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(w + l));
            f[2 * l] = g.x; f[2 * l + 1] = g.y;
        }
    }
}

// The join of parts (paged_attention.cu): tiles of `tile_rows` rows, of which at most `rows` exist; cuts kept for `entries` ranges or segments.
int launch_join(const AttnArgs& a, int dp, bool many, int entries, int ranges, int tile_rows, int rows, cudaStream_t stream);
// Map of the cache's bytes whose boxes are 16 tokens of one page and head.
bool cache_map(CUtensorMap* m, const Batch& b, const void* cache, int dp);

// The prompt form (paged_prompt.cu): sequences whose rows x query heads of a group are more than a.few_limit.
size_t prompt_workspace(const OglePagedBatch* b);
int launch_prompts(const OglePagedBatch* b, AttnArgs a, void* workspace, cudaStream_t stream);

}  // namespace paged
}  // namespace ogle
