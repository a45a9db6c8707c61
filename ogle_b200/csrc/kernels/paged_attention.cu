// Attention of the rows of a call over the paged 8-bit cache.
//
// o = sum_j w_j v_j / sum_j w_j with w_j = 2^(x_j - m), x_j = log2(e) scale (q . k_j), in one pass over the keys with a running m.
// For single tokens and drafts a key/value head is read for a few rows only - the query heads that share it - so the bytes of
// the cache are the bound, and what matters is that all of them are under way all the time: every warp has its own ring of
// copies and its own keys, and no barrier with the others until its part is done.
//
// Work: a segment is a tile of kRows rows (row of the sequence x query head of the group) of one sequence and kv head. All
// segments' tiles of 64 keys, laid end to end, are cut into equal ranges, one for each block, whatever the sequences' lengths are. A segment
// inside a block's range is finished there; parts of others go to the workspace, and paged_join_kernel adds them in order.
//
// The products run on 16-bit operands: an e4m3 value is an fp16 exactly; queries are scaled by a power of two so that their
// largest lies below 2^12 (11 bits of each, or 22 as two parts), weights lie below 2^15. kSplit keeps queries and weights as
// two parts, the high ones in rows 0-7 of the multiply and the low ones in rows 8-15: an accumulator's two halves of a row are
// then in the same thread, and up to 8 rows cost nothing more.
#include <type_traits>

#include "paged.cuh"

namespace ogle {
namespace {

using paged::Batch;

constexpr int kWarps = 4;
constexpr int kChunk = 16;                       // keys of a warp's step; a page holds whole steps
constexpr int kTileKeys = kWarps * kChunk;
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
    float* parts;                                // [blocks][2][kRows] x (DP + 2)
};

template <int DP, int MT, bool kSplit>
struct Form {
    static constexpr int kRows = MT * (kSplit ? 8 : 16);
    static constexpr int kStages = DP == 64 ? 6 : (DP == 128 ? 4 : 3);
    static constexpr int kStageBytes = 2 * kChunk * DP;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kJoin = kWarps * kRows * (DP + 4) * 4;
    static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
    static constexpr int kPart = kRows * (DP + 2);      // floats of a part: values, then m, then sums
    static constexpr int kBlocks = DP == 64 ? 4 : (DP == 128 && MT == 1 ? 3 : 2);   // that fit an SM at once
};

// ---- the ranges
struct Place { long long total, first; int b; };   // sum of all tiles; those of the sequences before b; the sequence of the position asked for

__device__ __forceinline__ int row_tiles(const Batch& a, int n, int rows) { return (n * a.group + rows - 1) / rows; }

// Keys that some row of the sequence attends: [lo, hi), lo down to a tile.
struct Span { int lo, hi; };
__device__ __forceinline__ Span span_of(const paged::Sequence& s, int first_row, int last_row, int causal, int window) {
    Span k;
    k.hi = causal ? min(s.len, s.len - s.n + last_row + 1) : s.len;
    k.lo = window > 0 ? max(0, s.len - s.n + first_row - window + 1) : 0;
    k.hi = max(k.hi, 0);
    return k;
}
__device__ __forceinline__ int tiles_of(const paged::Sequence& s, int causal, int window) {
    if (s.n <= 0) return 0;
    const Span k = span_of(s, 0, s.n - 1, causal, window);
    return k.hi > k.lo ? (k.hi - 1) / kTileKeys - k.lo / kTileKeys + 1 : 0;
}

// Sums the tiles of all sequences and finds the one that position total * num / den (or its end) falls in. All threads of a
// block of 128; `shared` holds 130 values.
template <typename F>
__device__ __forceinline__ Place locate(int n_seqs, int num, int den, long long* shared, F tiles) {
    const int tid = threadIdx.x, per = (n_seqs + 127) / 128;
    long long mine = 0;
    for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        if (b < n_seqs) mine += tiles(b);
    }
    long long sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long o = __shfl_up_sync(~0u, sum, d);
        if ((tid & 31) >= d) sum += o;
    }
    if ((tid & 31) == 31) shared[tid / 32] = sum;
    if (tid == 0) shared[5] = -1;
    __syncthreads();
    long long total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < tid / 32) before += shared[w];
        total += shared[w];
    }
    const long long at = total * num / den;
    sum += before;
    if (at >= sum - mine && at < sum) {
        long long first = sum - mine;
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            const long long t = b < n_seqs ? tiles(b) : 0;
            if (at < first + t) {
                shared[4] = first;
                shared[5] = b;
                break;
            }
            first += t;
        }
    }
    __syncthreads();
    Place p;
    p.total = total;
    p.first = shared[4];
    p.b = int(shared[5]);
    __syncthreads();
    return p;
}

// ---- copies and products
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    const int n = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
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

// Where unit u (16 bytes) of row r of a step lies: rows that are read together fall into different banks.
template <int DP>
__device__ __forceinline__ int key_at(int r, int u) { return r * DP + (DP == 64 ? u : u ^ ((r & 1) << 2)) * 16; }
template <int DP>
__device__ __forceinline__ int value_at(int r, int u) { return r * DP + (DP == 64 ? u ^ ((r >> 1) & 3) : u ^ (r & 7)) * 16; }

template <int DP, int MT, bool kSplit>
__global__ void __launch_bounds__(kWarps * 32, (Form<DP, MT, kSplit>::kBlocks)) paged_attention_kernel(AttnArgs a) {
    using F = Form<DP, MT, kSplit>;
    constexpr int kRows = F::kRows, NR = kSplit ? 1 : 2, KS = DP / 16, NB = DP / 8;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ long long shared[8];
    const Batch& B = a.b;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, c4 = lane & 3, r8 = lane >> 2;
    grid_dependency_trigger();
    grid_dependency_wait();
    const auto weight = [&](int b) {
        const paged::Sequence s = paged::sequence(B, b);
        return (long long)B.kv_heads * row_tiles(B, s.n, kRows) * tiles_of(s, a.causal, a.window);
    };
    const Place place = locate(B.n_seqs, blockIdx.x, gridDim.x, shared, weight);
    long long at = place.total * blockIdx.x / gridDim.x, first = place.first;
    const long long end = place.total * (blockIdx.x + 1) / gridDim.x;
    int b = place.b;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * F::kStages * F::kStageBytes;
    const uint32_t value_lane = (lane & 7) + ((lane >> 3) & 1) * 8;   // key of this lane's row of the transposed loads

    while (at < end && b < B.n_seqs) {
        paged::Sequence s = paged::sequence(B, b);
        int tiles = tiles_of(s, a.causal, a.window), rts = row_tiles(B, s.n, kRows);
        const long long all = (long long)B.kv_heads * rts * tiles;
        if (at >= first + all) { first += all; ++b; continue; }
        // segment: kv head, tile of rows; within it tiles [t0, t1)
        const long long seg = (at - first) / tiles;
        const int h = int(seg / rts), rt = int(seg % rts);
        const long long seg_first = first + seg * tiles;
        const int t0 = int(at - seg_first), t1 = int(min((long long)tiles, end - seg_first));
        const Span all_keys = span_of(s, 0, s.n - 1, a.causal, a.window);
        const int m0 = rt * kRows, m_end = min(s.n * B.group, m0 + kRows);
        const Span keys = span_of(s, m0 / B.group, (m_end - 1) / B.group, a.causal, a.window);
        const int inner_lo = span_of(s, (m_end - 1) / B.group, 0, a.causal, a.window).lo;
        const int inner_hi = span_of(s, 0, m0 / B.group, a.causal, a.window).hi;
        const int base = all_keys.lo / kTileKeys;
        int j_begin = max((base + t0) * kTileKeys, keys.lo / kChunk * kChunk), j_end = min((base + t1) * kTileKeys, keys.hi);
        const int steps = max(0, (j_end - j_begin + kChunk - 1) / kChunk);
        const int count = steps > warp ? (steps - warp + kWarps - 1) / kWarps : 0;   // of this warp: warp, warp + 4, ...

        // queries: this thread's parts of the rows it has
        uint32_t Q[MT][KS][4];
        float rs[MT][NR], m[MT][NR], l[MT][NR];
        int lo_row[MT][NR], hi_row[MT][NR];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int row = min(m0 + mt * (kSplit ? 8 : 16) + r * 8 + r8, m_end - 1);   // rows that are not there repeat the last
                const int i = row / B.group, g = row % B.group;
                const long long q0 = (s.row0 + i) * a.q_row + (h * B.group + g) * a.q_head;
                const Span k = span_of(s, i, i, a.causal, a.window);
                lo_row[mt][r] = k.lo;
                hi_row[mt][r] = k.hi;
                float top = 0.f;
                for (int d = c4; d < B.dim; d += 4) top = fmaxf(top, fabsf(paged::to_float(a.q, q0 + d, B.dtype)));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                // 2^e with |q| 2^-e below 2^12; an infinite or vanishing row stays as it is
                const int e = top > 1e-30f && top <= 3e38f ? int(__float_as_uint(top) >> 23) - 126 - 12 : 0;
                const float down = __uint_as_float(uint32_t(127 - e) << 23);
                rs[mt][r] = a.scale_log2 * __uint_as_float(uint32_t(127 + e) << 23);
                m[mt][r] = -INFINITY;
                l[mt][r] = 0.f;
#pragma unroll
                for (int t = 0; t < KS; ++t) {
                    // step t, this thread: word t % 4 of unit c4 + 4 (t / 4) - the order in which it reads keys
                    const int d = 16 * (c4 + 4 * (t / 4)) + 4 * (t % 4);
                    float f[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) f[x] = d < B.dim ? paged::to_float(a.q, q0 + d + x, B.dtype) * down : 0.f;
                    const uint32_t u = half2_bits(f[0], f[1]), v = half2_bits(f[2], f[3]);
                    if (kSplit) {
                        Q[mt][t][0] = u; Q[mt][t][1] = rest_bits(u, f[0], f[1]);
                        Q[mt][t][2] = v; Q[mt][t][3] = rest_bits(v, f[2], f[3]);
                    } else {
                        Q[mt][t][r] = u; Q[mt][t][2 + r] = v;
                    }
                }
            }
        float O[MT][NB][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) O[mt][n][x] = 0.f;
        float vref = 1.1754944e-38f;              // the unit of O: the largest value scale met

        // pages and scales of the warp's next 32 steps, a lane each; the 32 behind them are on their way
        int page[2] = {-1, -1};
        float ks[2] = {0.f, 0.f}, vs[2] = {0.f, 0.f};
        const auto look_up = [&](int which, int i) {
            page[which] = -1;
            ks[which] = vs[which] = 0.f;
            if (i < count) {
                page[which] = paged::page_of(B, b, (j_begin + (i * kWarps + warp) * kChunk) >> B.page_shift);
                if (page[which] >= 0) {
                    const long long o = (long long)page[which] * B.kv_heads + h;
                    ks[which] = __ldg(B.k_scale + o);
                    vs[which] = __ldg(B.v_scale + o);
                }
            }
        };
        look_up(0, lane);
        look_up(1, 32 + lane);
        const auto issue = [&](int i, int now) {
            if (i < count) {
                const int j0 = j_begin + (i * kWarps + warp) * kChunk;
                const int p0 = __shfl_sync(~0u, page[0], i & 31), p1 = __shfl_sync(~0u, page[1], i & 31);
                const int p = (i >> 5) == (now >> 5) ? p0 : p1;
                const long long o = (long long)max(p, 0) * B.page_stride + h * B.head_stride + (long long)(j0 & ((1 << B.page_shift) - 1)) * B.token_stride;
                const uint32_t dst = ring + (i % F::kStages) * F::kStageBytes;
#pragma unroll
                for (int x = 0; x < DP / 32; ++x) {
                    const int idx = x * 32 + lane, r = idx / (DP / 16), u = idx % (DP / 16);
                    const bool there = p >= 0 && j0 + r >= keys.lo && j0 + r < keys.hi && u * 16 < B.dim;
                    const long long from = there ? o + r * B.token_stride + u * 16 : 0;
                    copy16(dst + key_at<DP>(r, u), B.k_cache + from, there);
                    copy16(dst + kChunk * DP + value_at<DP>(r, u), B.v_cache + from, there);
                }
            }
            copies_commit();
        };
#pragma unroll
        for (int i = 0; i < F::kStages - 1; ++i) issue(i, 0);

        for (int i = 0; i < count; ++i) {
            if ((i & 31) == 0 && i > 0) {
                page[0] = page[1]; ks[0] = ks[1]; vs[0] = vs[1];
                look_up(1, i + 32 + lane);
            }
            copies_wait<F::kStages - 2>();
            __syncwarp();
            const uint32_t at_k = ring + (i % F::kStages) * F::kStageBytes, at_v = at_k + kChunk * DP;
            const int j0 = j_begin + (i * kWarps + warp) * kChunk;
            const float k_scale = __shfl_sync(~0u, ks[0], i & 31), v_scale = __shfl_sync(~0u, vs[0], i & 31);
            const bool no_page = __shfl_sync(~0u, page[0], i & 31) < 0;
            const bool edge = j0 < inner_lo || j0 + kChunk > inner_hi || no_page;
            // x = q . k
            float x[MT][2][NR * 2];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
                float S[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int y = 0; y < 4; ++y) S[mt][y] = 0.f;
#pragma unroll
                for (int u = 0; u < DP / 64; ++u) {
                    uint32_t w[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at_k + key_at<DP>(nb * 8 + r8, c4 + 4 * u)) : "memory");
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const uint32_t b0 = paged::e4m3x2_to_half2(uint16_t(w[y])), b1 = paged::e4m3x2_to_half2(uint16_t(w[y] >> 16));
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) mma(S[mt], Q[mt][4 * u + y], b0, b1);
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    if (kSplit) {
                        x[mt][nb][0] = (S[mt][0] + S[mt][2]) * (rs[mt][0] * k_scale);
                        x[mt][nb][1] = (S[mt][1] + S[mt][3]) * (rs[mt][0] * k_scale);
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; ++y) x[mt][nb][y % (2 * NR)] = S[mt][y] * (rs[mt][(y / 2) % NR] * k_scale);
                    }
                }
            }
            if (edge) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                        for (int y = 0; y < 2 * NR; ++y) {
                            const int j = j0 + nb * 8 + c4 * 2 + (y & 1);
                            if (no_page || j < lo_row[mt][y / 2] || j >= hi_row[mt][y / 2]) x[mt][nb][y] = -INFINITY;
                        }
            }
            // a larger unit for a row's weights or for the values: rare
            bool more = v_scale > vref;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                    for (int y = 0; y < 2 * NR; ++y) more |= x[mt][nb][y] > m[mt][y / 2] + kHeadroom;
            if (__any_sync(~0u, more)) {
                const float vnew = fmaxf(vref, v_scale), vratio = vref / vnew;
                vref = vnew;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float f[NR];
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        float top = fmaxf(fmaxf(x[mt][0][2 * r], x[mt][0][2 * r + 1]), fmaxf(x[mt][1][2 * r], x[mt][1][2 * r + 1]));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                        top = fmaxf(top, m[mt][r]);
                        f[r] = top == -INFINITY ? 1.f : exp2_fast(m[mt][r] - top);
                        m[mt][r] = top;
                        l[mt][r] *= f[r];
                        f[r] *= vratio;
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int y = 0; y < 4; ++y) O[mt][n][y] *= f[(y / 2) % NR];
                }
            }
            // weights, and with the values' scale as A operands of the second product
            const float v_unit = v_scale / vref;
            uint32_t P[MT][4];
            uint32_t seen[MT][4];                       // 1 where the row attends the key, for NaN among the values
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const float off = m[mt][r] == -INFINITY ? 0.f : m[mt][r] - kLift;
                        float p[2];
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            p[y] = exp2_fast(x[mt][nb][2 * r + y] - off);
                            l[mt][r] += p[y];
                            p[y] *= v_unit;
                        }
                        const uint32_t hi = half2_bits(p[0], p[1]);
                        const uint32_t see = (x[mt][nb][2 * r] == -INFINITY ? 0u : 0x3c00u) | (x[mt][nb][2 * r + 1] == -INFINITY ? 0u : 0x3c000000u);
                        if (kSplit) {
                            P[mt][2 * nb] = hi;
                            P[mt][2 * nb + 1] = rest_bits(hi, p[0], p[1]);
                            seen[mt][2 * nb] = see;
                            seen[mt][2 * nb + 1] = 0;
                        } else {
                            P[mt][2 * nb + r] = hi;
                            seen[mt][2 * nb + r] = see;
                        }
                    }
            // the stage's values, two units (32 elements) at a time
#pragma unroll
            for (int u = 0; u < DP / 32; ++u) {
                uint32_t w[4];
                ldmatrix_trans(w, at_v + value_at<DP>(value_lane, 2 * u + (lane >> 4)));
                uint32_t v[4][2];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const uint32_t t = __byte_perm(w[y], 0, 0x3120);   // (key, key + 1) of the even element, then of the odd one
                    v[y][0] = paged::e4m3x2_to_half2(uint16_t(t));
                    v[y][1] = paged::e4m3x2_to_half2(uint16_t(t >> 16));
                }
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int odd = 0; odd < 2; ++odd) {
                        uint32_t b0 = v[2 * y][odd], b1 = v[2 * y + 1][odd];
                        if (edge) {
                            // a row that does not attend a key has weight 0 for it, and 0 x NaN would still be NaN: NaNs are
                            // taken out, and counted for the rows that do attend them
                            const __half2 h0 = *reinterpret_cast<const __half2*>(&b0), h1 = *reinterpret_cast<const __half2*>(&b1);
                            const uint32_t n0 = __hneu2_mask(h0, h0), n1 = __hneu2_mask(h1, h1);
                            if (__any_sync(~0u, (n0 | n1) != 0)) {
                                b0 &= ~n0;
                                b1 &= ~n1;
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    float nan[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma(nan, seen[mt], n0 & 0x3c003c00u, n1 & 0x3c003c00u);
#pragma unroll
                                    for (int z = 0; z < 4; ++z)
                                        if (nan[z] > 0.f) O[mt][4 * u + 2 * y + odd][z] = NAN;
                                }
                            }
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) mma(O[mt][4 * u + 2 * y + odd], P[mt], b0, b1);
                    }
            }
            __syncwarp();
            issue(i + F::kStages - 1, i);
        }
        copies_wait<0>();
        __syncthreads();                          // every warp is through with its ring: the parts take its place

        // the warps' parts: values [kRows][DP + 4], then m and l
        float* const mine = reinterpret_cast<float*>(smem) + warp * kRows * (DP + 4);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float sum = l[mt][r];
                sum += __shfl_xor_sync(~0u, sum, 1);
                sum += __shfl_xor_sync(~0u, sum, 2);
                float* row = mine + (mt * (kSplit ? 8 : 16) + r * 8 + r8) * (DP + 4);
#pragma unroll
                for (int u = 0; u < DP / 16; ++u) {
                    float4 v;                     // the even block's two columns and the odd block's are four neighbours
                    if (kSplit) {
                        v.x = O[mt][2 * u][0] + O[mt][2 * u][2]; v.y = O[mt][2 * u + 1][0] + O[mt][2 * u + 1][2];
                        v.z = O[mt][2 * u][1] + O[mt][2 * u][3]; v.w = O[mt][2 * u + 1][1] + O[mt][2 * u + 1][3];
                    } else {
                        v.x = O[mt][2 * u][2 * r]; v.y = O[mt][2 * u + 1][2 * r];
                        v.z = O[mt][2 * u][2 * r + 1]; v.w = O[mt][2 * u + 1][2 * r + 1];
                    }
                    v.x *= vref; v.y *= vref; v.z *= vref; v.w *= vref;
                    *reinterpret_cast<float4*>(row + u * 16 + c4 * 4) = v;
                }
                if (c4 == 0) { row[DP] = m[mt][r]; row[DP + 1] = sum; }
            }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == tiles;
        float* const part = a.parts + ((long long)blockIdx.x * 2 + (t0 > 0 ? 0 : 1)) * F::kPart;
        for (int idx = tid; idx < kRows * (DP / 4); idx += kWarps * 32) {
            const int r = idx / (DP / 4), d = idx % (DP / 4) * 4, row = m0 + r;
            if (row >= m_end) continue;
            const float* p = reinterpret_cast<const float*>(smem) + r * (DP + 4);
            float top = -INFINITY, sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, p[w * kRows * (DP + 4) + DP]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float* q = p + w * kRows * (DP + 4);
                // a warp without a weight has nothing to give; one with a NaN does
                const float f = q[DP + 1] == 0.f ? 0.f : exp2_fast(q[DP] - top);
                if (q[DP + 1] == 0.f) continue;
                const float4 o = *reinterpret_cast<const float4*>(q + d);
                sum += q[DP + 1] * f;
                v.x += o.x * f; v.y += o.y * f; v.z += o.z * f; v.w += o.w * f;
            }
            if (!whole) {
                *reinterpret_cast<float4*>(part + r * DP + d) = v;
                if (d == 0) { part[kRows * DP + r] = top; part[kRows * DP + kRows + r] = sum; }
                continue;
            }
            store_row(a, s.row0 + row / B.group, h * B.group + row % B.group, d, v, top, sum);
        }
        __syncthreads();                          // the next segment's copies take the parts' place
        at = seg_first + t1;
    }
}

// Adds up the parts of segments that were cut, in the order of their ranges, and answers for sequences without a key. Block c
// stands for the boundary before range c + 1 and has the segment that this is the first boundary inside of.
template <int DP, int MT, bool kSplit>
__global__ void __launch_bounds__(kWarps * 32) paged_join_kernel(AttnArgs a, int ranges) {
    using F = Form<DP, MT, kSplit>;
    constexpr int kRows = F::kRows;
    __shared__ long long shared[8];
    const Batch& B = a.b;
    const int tid = threadIdx.x, c = blockIdx.x + 1;
    grid_dependency_trigger();
    grid_dependency_wait();
    for (int b = blockIdx.x; b < B.n_seqs; b += gridDim.x) {
        const paged::Sequence s = paged::sequence(B, b);
        if (s.n <= 0 || tiles_of(s, a.causal, a.window) > 0) continue;
        for (int idx = tid; idx < s.n * B.q_heads * (DP / 4); idx += blockDim.x) {
            const int row = idx / (B.q_heads * (DP / 4)), r = idx % (B.q_heads * (DP / 4));
            store_row(a, s.row0 + row, r / (DP / 4), r % (DP / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
        }
    }
    if (c >= ranges) return;
    const auto weight = [&](int b) {
        const paged::Sequence s = paged::sequence(B, b);
        return (long long)B.kv_heads * row_tiles(B, s.n, kRows) * tiles_of(s, a.causal, a.window);
    };
    const Place place = locate(B.n_seqs, c, ranges, shared, weight);
    if (place.b < 0) return;
    const paged::Sequence s = paged::sequence(B, place.b);
    const int tiles = tiles_of(s, a.causal, a.window), rts = row_tiles(B, s.n, kRows);
    const auto bound = [&](int k) { return place.total * k / ranges; };
    const long long x = bound(c), seg = (x - place.first) / tiles, begin = place.first + seg * tiles, end = begin + tiles;
    if (x == begin || bound(c - 1) > begin) return;
    const int h = int(seg / rts), m0 = int(seg % rts) * kRows, m_end = min(s.n * B.group, m0 + kRows);
    int last = c;                                 // ranges c - 1 .. last - 1 have parts
    while (last < ranges && bound(last) < end) ++last;
    for (int idx = tid; idx < kRows * (DP / 4); idx += kWarps * 32) {
        const int r = idx / (DP / 4), d = idx % (DP / 4) * 4, row = m0 + r;
        if (row >= m_end) continue;
        float top = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = c - 1; k < last; ++k) {
            if (bound(k) == bound(k + 1)) continue;             // more ranges than tiles
            const float* p = a.parts + ((long long)k * 2 + (k == c - 1 ? 1 : 0)) * F::kPart;
            const float m = p[kRows * DP + r], l = p[kRows * DP + kRows + r];
            if (l == 0.f) continue;
            const float4 o = *reinterpret_cast<const float4*>(p + r * DP + d);
            const float now = fmaxf(top, m), f = top == -INFINITY ? 0.f : exp2_fast(top - now), g = exp2_fast(m - now);
            sum = sum * f + l * g;
            v.x = v.x * f + o.x * g; v.y = v.y * f + o.y * g; v.z = v.z * f + o.z * g; v.w = v.w * f + o.w * g;
            top = now;
        }
        store_row(a, s.row0 + row / B.group, h * B.group + row % B.group, d, v, top, sum);
    }
}

// ---- host
struct Choice { int dp, mt; bool split; };

Choice choose(const OglePagedBatch* b) {
    Choice c;
    const long long rows = (long long)(b->max_rows < b->n_rows ? b->max_rows : b->n_rows) * (b->q_heads / b->kv_heads);
    c.dp = b->head_dim <= 64 ? 64 : (b->head_dim <= 128 ? 128 : 256);
    c.split = b->dtype == OGLE_F32 || rows <= 8;
    c.mt = c.dp == 256 || rows <= (c.split ? 8 : 16) ? 1 : 2;
    return c;
}

template <typename G>
auto with_form(const Choice& c, G g) {
    if (c.dp == 64) {
        if (c.split) return c.mt == 1 ? g(std::integral_constant<int, 64>(), std::integral_constant<int, 1>(), std::true_type())
                                      : g(std::integral_constant<int, 64>(), std::integral_constant<int, 2>(), std::true_type());
        return c.mt == 1 ? g(std::integral_constant<int, 64>(), std::integral_constant<int, 1>(), std::false_type())
                         : g(std::integral_constant<int, 64>(), std::integral_constant<int, 2>(), std::false_type());
    }
    if (c.dp == 128) {
        if (c.split) return c.mt == 1 ? g(std::integral_constant<int, 128>(), std::integral_constant<int, 1>(), std::true_type())
                                      : g(std::integral_constant<int, 128>(), std::integral_constant<int, 2>(), std::true_type());
        return c.mt == 1 ? g(std::integral_constant<int, 128>(), std::integral_constant<int, 1>(), std::false_type())
                         : g(std::integral_constant<int, 128>(), std::integral_constant<int, 2>(), std::false_type());
    }
    return c.split ? g(std::integral_constant<int, 256>(), std::integral_constant<int, 1>(), std::true_type())
                   : g(std::integral_constant<int, 256>(), std::integral_constant<int, 1>(), std::false_type());
}

// Ranges: as many blocks as fit the GPU at once, and no more than there can be tiles.
int ranges_of(const OglePagedBatch* b, int rows, int blocks) {
    const long long max_rows = b->max_rows < b->n_rows ? b->max_rows : b->n_rows;
    const long long tiles = (b->max_kv_len + kTileKeys - 1) / kTileKeys + 1;
    const long long most = (max_rows * (b->q_heads / b->kv_heads) + rows - 1) / rows * b->n_seqs;
    const double all = double(b->kv_heads) * double(most) * double(tiles);
    return all < double(kNumSMs * blocks) ? (all < 1 ? 1 : int(all)) : kNumSMs * blocks;
}

}  // namespace
}  // namespace ogle

using namespace ogle;

extern "C" {

size_t ogle_cuda_paged_attention_workspace_bytes(const OglePagedBatch* batch, const OgleAttentionParams* p) {
    Batch b;
    if (!p || paged::translate(batch, b) != OGLE_OK || b.n_seqs == 0) return 0;
    return with_form(choose(batch), [&](auto dp, auto mt, auto split) {
        using F = Form<decltype(dp)::value, decltype(mt)::value, decltype(split)::value>;
        return size_t(ranges_of(batch, F::kRows, F::kBlocks)) * 2 * F::kPart * sizeof(float);
    });
}

int ogle_cuda_paged_attention(const OglePagedBatch* batch, const OgleAttentionParams* p, void* workspace, size_t workspace_bytes,
                              ogle_stream_t stream) {
    AttnArgs a = {};
    int rc = paged::translate(batch, a.b);
    if (rc != OGLE_OK) return rc;
    if (!p || p->window < 0) return OGLE_ERR_INVALID;
    if (a.b.n_seqs == 0) return OGLE_OK;
    if (!p->q || !p->out || !workspace) return OGLE_ERR_INVALID;
    if (!paged::strides_ok(p->q, p->q_row, p->q_head, batch->dtype) || !paged::strides_ok(p->out, p->out_row, p->out_head, batch->dtype) || !aligned16(workspace))
        return OGLE_ERR_ALIGNMENT;
    if (workspace_bytes < ogle_cuda_paged_attention_workspace_bytes(batch, p)) return OGLE_ERR_INVALID;
    a.q = p->q; a.out = p->out; a.lse = p->lse;
    a.q_row = p->q_row; a.q_head = p->q_head; a.out_row = p->out_row; a.out_head = p->out_head;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.causal = p->causal; a.window = p->window;
    a.parts = static_cast<float*>(workspace);
    return with_form(choose(batch), [&](auto dp, auto mt, auto split) -> int {
        constexpr int DP = decltype(dp)::value, MT = decltype(mt)::value;
        constexpr bool kSplit = decltype(split)::value;
        using F = Form<DP, MT, kSplit>;
        const int ranges = ranges_of(batch, F::kRows, F::kBlocks);
        auto kernel = paged_attention_kernel<DP, MT, kSplit>;
        static std::atomic<uint64_t> sized{0};           // devices whose limit of shared memory is raised
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess && !(sized.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
            if (e == cudaSuccess) sized.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
        }
        if (e == cudaSuccess) e = launch_overlapped(kernel, dim3(ranges), dim3(kWarps * 32), F::kSmem, stream, a);
        if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
        int rc = finish_launch();
        if (rc != OGLE_OK) return rc;
        e = launch_overlapped_if(overlapped_launches_enabled(true), paged_join_kernel<DP, MT, kSplit>, dim3(ranges > 1 ? ranges - 1 : 1),
                                 dim3(kWarps * 32), 0, stream, a, ranges);
        if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
        return finish_launch();
    });
}

}  // extern "C"
