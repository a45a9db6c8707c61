// Which pages of the cache a query attends: bounds of the pages' keys, a score of every page for every query, the best of them.
//
// A page's bounds are the least and the largest key in every element, as whole numbers below 128 times a power of two of the page. A
// query is whole numbers below 128 as well (and a power of two that all pages share), so the largest product that any key within the bounds
// could have with it is a sum of products of whole numbers below 2^24: it does not depend on how it is summed, and two
// implementations of the score agree in every bit. The sum is a product of 8-bit matrices - the query's positive elements with the upper
// bounds, its negative ones with the lower - for which the cache's layout is the multiply's: a page is a column.
//
// Bound by latency: sequence, table, page, bounds, one look-up behind the other. 64 texts of up to 8000 tokens, pages of 64, 32 query heads to 8
// of 128: 7 us for the bounds of the new tokens' pages (4 MB) and 9 for scores and choice (10 MB). Twelve drafts over up to 150000 tokens, pages of 32:
// 5, 9 for the scores and 9 for the choice.
#include <atomic>

#include "paged.cuh"

namespace ogle {
namespace {

using paged::Batch;

// ---- bounds
struct BoundsArgs {
    Batch b;
    signed char* bounds;
    float* scale;
    int per_seq;                                 // pages that a sequence can have appended to
};

// The exponent of the smallest power of two t with amax <= 127 t, from the bits (0 for 0).
__device__ __forceinline__ int unit_exponent(float amax) {
    if (amax == 0.f) return 0;
    const bool small = amax < 0x1p-100f;
    const uint32_t u = __float_as_uint(small ? amax * 0x1p60f : amax);
    return int(u >> 23) - 126 - 7 - (small ? 60 : 0) + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);     // amax = f 2^(e + 7), f in [0.5, 1); 127 = 0.9921875 * 2^7
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }

constexpr int kBoundThreads = 128;

// A block has one page and head: a thread 16 elements of every so-many-th key.
__global__ void __launch_bounds__(kBoundThreads) page_bounds_kernel(BoundsArgs a) {
    __shared__ __half2 lowest[kBoundThreads * 8], highest[kBoundThreads * 8];
    __shared__ float tops[kBoundThreads / 32];
    const Batch& B = a.b;
    const int tid = threadIdx.x, h = blockIdx.y, b = blockIdx.x / a.per_seq, nth = blockIdx.x % a.per_seq;
    grid_dependency_trigger();
    grid_dependency_wait();
    const paged::Sequence s = paged::sequence(B, b);
    const int begin = max(s.first, 0), end = min(s.first + s.n, s.len), block = (begin >> B.page_shift) + nth;
    if (end <= begin || block > (end - 1) >> B.page_shift) return;
    const int page = paged::page_of(B, b, block);
    if (page < 0) return;
    const int tokens = min(s.len - (block << B.page_shift), 1 << B.page_shift), cols = B.dim / 16, lanes = kBoundThreads / cols;
    const int col = tid % cols, first = tid / cols;
    const unsigned char* const keys = B.k_cache + page * B.page_stride + h * B.head_stride + col * 16;
    const float inf = INFINITY;
    __half2 lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo[i] = __float2half2_rn(inf);
        hi[i] = __float2half2_rn(-inf);
    }
    if (first < lanes) {
#pragma unroll 4
        for (int t = first; t < tokens; t += lanes) {
            const uint4 v = *reinterpret_cast<const uint4*>(keys + t * B.token_stride);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t x, y;
                paged::e4m3x4_to_half2(w[i], x, y);
                const __half2 p = *reinterpret_cast<const __half2*>(&x), q = *reinterpret_cast<const __half2*>(&y);
                lo[2 * i] = __hmin2(lo[2 * i], p);         // (of a number and a NaN, the number)
                hi[2 * i] = __hmax2(hi[2 * i], p);
                lo[2 * i + 1] = __hmin2(lo[2 * i + 1], q);
                hi[2 * i + 1] = __hmax2(hi[2 * i + 1], q);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lowest[first * (cols * 8) + col * 8 + i] = lo[i];
            highest[first * (cols * 8) + col * 8 + i] = hi[i];
        }
    }
    __syncthreads();
    // pair `tid` of the elements
    const int pairs = B.dim / 2;
    float l[2] = {0.f, 0.f}, u[2] = {0.f, 0.f}, top = 0.f;
    if (tid < pairs) {
        __half2 least = lowest[tid], most = highest[tid];
        for (int i = 1; i < lanes; ++i) {
            least = __hmin2(least, lowest[i * pairs + tid]);
            most = __hmax2(most, highest[i * pairs + tid]);
        }
        const float2 f = __half22float2(least), g = __half22float2(most);
        if (f.x <= g.x) { l[0] = f.x; u[0] = g.x; }        // else: nothing but NaN
        if (f.y <= g.y) { l[1] = f.y; u[1] = g.y; }
#pragma unroll
        for (int i = 0; i < 2; ++i) top = fmaxf(top, fmaxf(fabsf(l[i]), fabsf(u[i])));
    }
#pragma unroll
    for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    if ((tid & 31) == 0) tops[tid / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBoundThreads / 32; ++w) top = fmaxf(top, tops[w]);
    const int exponent = unit_exponent(top);     // of e4m3 values: -15 to 2
    const float unit = power_of_two(exponent), by = power_of_two(-exponent);
    const long long at = (long long)page * B.kv_heads + h;
    if (tid < pairs) {
        signed char* const out = a.bounds + at * 2 * B.dim + tid * 2;
        *reinterpret_cast<char2*>(out) = make_char2((signed char)floorf(l[0] * by), (signed char)floorf(l[1] * by));
        *reinterpret_cast<char2*>(out + B.dim) = make_char2((signed char)ceilf(u[0] * by), (signed char)ceilf(u[1] * by));
    }
    if (tid == 0) a.scale[at] = unit * B.k_scale[at];
}

// ---- scores
struct ChooseArgs {
    Batch b;
    const void* q;
    long long q_row, q_head;
    const signed char* bounds;
    const float* scale;
    int* chosen;
    long long chosen_row, chosen_head;
    int count, first, last;
    unsigned* keys;                              // [rows][kv heads][stride]
    long long stride;
    int row0, rows;                              // rows of this launch
    int tiles, chunks, chunk_pages;              // tiles of rows that a sequence can have; chunks of pages
};

constexpr int kWarps = 4;
constexpr int kStepPages = 8;
constexpr int kMostSteps = 8;                    // of a warp
constexpr unsigned kAlways = ~0u;

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A page's score as a number that orders the same way: 0 for what is not chosen, 1 for what has no size.
__device__ __forceinline__ unsigned ordered_score(float x) {
    x += 0.f;
    if (x != x) return 1u;
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Rows of a tile: as many as have their query heads of a group in the 16 rows of a multiply, at least one.
__device__ __forceinline__ int rows_of_tile(int group) { return group >= 16 ? 1 : 16 / group; }

// Eight values of a row, as fp32, infinities and NaN as 0.
__device__ __forceinline__ void load8(const void* q, long long at, int dtype, float (&f)[8]) {
    if (dtype == OGLE_F32) {
        const float4* const p = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at);
        const float4 x = __ldg(p), y = __ldg(p + 1);
        f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(q) + at));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int l = 0; l < 4; ++l) {
            const float2 g = dtype == OGLE_F16 ? __half22float2(*reinterpret_cast<const __half2*>(w + l)) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(w + l));
            f[2 * l] = g.x; f[2 * l + 1] = g.y;
        }
    }
#pragma unroll
    for (int l = 0; l < 8; ++l)
        if (!(fabsf(f[l]) <= 3.402823466e38f)) f[l] = 0.f;
}

// A block has a tile of rows of one sequence, one kv head and a chunk of pages. The queries lie in shared memory as the multiply takes
// them: of 64 bytes of a head's elements, lane c4 of four has bytes [16 c4, 16 c4 + 16) - the order in which pages are read -, the
// lower bounds' first, then the upper bounds'. A warp's pages are looked up at once, before anything else, and the bounds of its next
// eight pages are under way while it multiplies.
// kFew: rows of few pages, whose keys stay in shared memory and are picked from at once.
constexpr int kRanked = 256;                     // keys whose ranks are counted one against all
constexpr int kFewRows = 4;
__device__ __forceinline__ void pick_by_rank(const unsigned* ranked, int* sums, int n, int* out, int count);

template <int kScoreWarps, bool kFew>
__global__ void __launch_bounds__(kScoreWarps * 32) choose_score_kernel(ChooseArgs a) {
    extern __shared__ __align__(16) unsigned char queries[];
    __shared__ int tile_score[kScoreWarps][16][kStepPages + 1];
    __shared__ unsigned tops[16];
    __shared__ __align__(16) unsigned ranked[kFew ? kFewRows : 1][kRanked];
    __shared__ int sums[kScoreWarps];
    const Batch& B = a.b;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, c4 = lane & 3, r8 = lane >> 2;
    if (tid < 16) tops[tid] = 0;
    grid_dependency_trigger();
    grid_dependency_wait();
    const int chunk = blockIdx.x % a.chunks, rest = blockIdx.x / a.chunks, h = rest % B.kv_heads, tile = rest / B.kv_heads % a.tiles, b = rest / B.kv_heads / a.tiles;
    const paged::Sequence s = paged::sequence(B, b);
    const int per = rows_of_tile(B.group);
    // rows of the tile that belong to this launch
    const int r0 = max(tile * per, a.row0 - s.row0), r1 = min(min(tile * per + per, s.n), a.row0 + a.rows - s.row0);
    if (r0 >= r1) return;
    const int last_place = min(s.first + r1 - 1, s.len - 1), blocks = last_place >= 0 ? (last_place >> B.page_shift) + 1 : 0;
    const int first_page = chunk * a.chunk_pages, end_page = min(first_page + a.chunk_pages, blocks);
    if (!kFew && first_page >= blocks) return;
    // lane l: page l % 8 of the warp's steps l / 8 and l / 8 + 4, ... (a chunk has kMostSteps of them at most)
    int page[kMostSteps / 4];
    float unit[kMostSteps / 4];
#pragma unroll
    for (int i = 0; i < kMostSteps / 4; ++i) {
        const int block = first_page + ((i * 4 + lane / kStepPages) * kScoreWarps + warp) * kStepPages + lane % kStepPages;
        page[i] = block < end_page ? paged::page_of(B, b, block) : -1;
    }
#pragma unroll
    for (int i = 0; i < kMostSteps / 4; ++i) unit[i] = page[i] >= 0 ? __ldg(a.scale + (long long)page[i] * B.kv_heads + h) : 0.f;
    const int n_rows = r1 - r0, heads = n_rows * B.group, m_tiles = (heads + 15) / 16, words = (B.dim + 63) / 64;
    const int bytes = 2 * B.dim;
    uint4 v[8];                                  // words of the lower and of the upper bounds in turn
    const auto load = [&](int step) {
        const int p = __shfl_sync(~0u, page[0], step % 4 * kStepPages + r8), q = __shfl_sync(~0u, page[1], step % 4 * kStepPages + r8);
        static_assert(kMostSteps == 8, "two pages a lane");
        const int mine = step < 4 ? p : q;
        const signed char* const from = a.bounds + ((long long)max(mine, 0) * B.kv_heads + h) * bytes;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                const int d = w * 64 + c4 * 16;
                v[2 * w + side] = w < words && d < B.dim && mine >= 0 ? __ldg(reinterpret_cast<const uint4*>(from + side * B.dim + d)) : make_uint4(0, 0, 0, 0);
            }
    };
    load(0);

    // the queries' whole numbers: a row's heads share a unit
    const int vecs = B.dim / 8, padded = words * 8, per_row = B.group * vecs;
    const long long q0 = (long long)(s.row0 + r0) * a.q_row + (long long)h * B.group * a.q_head;
    __syncthreads();
    for (int i = tid; i < n_rows * per_row; i += kScoreWarps * 32) {
        const int m = i / vecs, r = m / B.group;
        float f[8], top = 0.f;
        load8(a.q, q0 + r * a.q_row + (m - r * B.group) * a.q_head + (i - m * vecs) * 8, B.dtype, f);
#pragma unroll
        for (int l = 0; l < 8; ++l) top = fmaxf(top, fabsf(f[l]));
        atomicMax(tops + r, __float_as_uint(top));
    }
    __syncthreads();
    for (int i = tid; i < m_tiles * 16 * padded; i += kScoreWarps * 32) {
        const int m = i / padded, d = (i - m * padded) * 8, r = m / B.group;
        uint32_t low[2] = {0u, 0u}, high[2] = {0u, 0u};
        if (m < heads && d < B.dim) {
            float f[8];
            load8(a.q, q0 + r * a.q_row + (m - r * B.group) * a.q_head + d, B.dtype, f);
            const int exponent = unit_exponent(__uint_as_float(tops[r])), half = -exponent / 2;
            const float by = power_of_two(half), by_rest = power_of_two(-exponent - half);     // their product can be above the largest number
#pragma unroll
            for (int l = 0; l < 8; ++l) {
                const int x = min(max(__float2int_rn(f[l] * by * by_rest), -127), 127);
                low[l / 4] |= uint32_t(min(x, 0) & 255) << l % 4 * 8;
                high[l / 4] |= uint32_t(max(x, 0)) << l % 4 * 8;
            }
        }
        // eight elements are a step's two words of lane d % 64 / 16: row r8 bytes 0-3, row r8 + 8 the same, row r8 bytes 4-7, row r8 + 8 the same
        const int mt = m / 16, row = m % 16, w = d / 64;
        uint32_t* const to = reinterpret_cast<uint32_t*>(queries + ((mt * 2 * words + w) * 2 + d % 16 / 8) * 512 + ((row & 7) * 4 + d % 64 / 16) * 16) + row / 8;
        to[0] = low[0];
        to[2] = low[1];
        to[words * 256] = high[0];
        to[words * 256 + 2] = high[1];
    }
    __syncthreads();

    for (int step = 0; first_page + (step * kScoreWarps + warp) * kStepPages < end_page; ++step) {
        const int p0 = first_page + (step * kScoreWarps + warp) * kStepPages;
        uint4 z[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) z[w] = v[w];
        if (step + 1 < kMostSteps) load(step + 1);
        for (int mt = 0; mt < m_tiles; ++mt) {
            int c[4] = {0, 0, 0, 0}, e[4] = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; ++w)
                if (w < words)
#pragma unroll
                    for (int side = 0; side < 2; ++side) {
                        const uint4* const q = reinterpret_cast<const uint4*>(queries) + ((mt * 2 + side) * words + w) * 2 * 32 + lane;
                        const uint4 x = q[0], y = q[32], b8 = z[2 * w + side];
                        mma_s8(c, x.x, x.y, x.z, x.w, b8.x, b8.y);
                        mma_s8(e, y.x, y.y, y.z, y.w, b8.z, b8.w);
                    }
            tile_score[warp][r8][c4 * 2] = c[0] + e[0];
            tile_score[warp][r8][c4 * 2 + 1] = c[1] + e[1];
            tile_score[warp][r8 + 8][c4 * 2] = c[2] + e[2];
            tile_score[warp][r8 + 8][c4 * 2 + 1] = c[3] + e[3];
            __syncwarp();
            // the best of a row's heads: of a whole row, or of 16 of its heads more. Lane l has page l % 8, whose number and unit lie with it for
            // this step, of every fourth row.
            const int n = lane % kStepPages, blk = p0 + n;
            const int pg0 = __shfl_sync(~0u, page[0], step % 4 * kStepPages + n), pg1 = __shfl_sync(~0u, page[1], step % 4 * kStepPages + n);
            const float u0 = __shfl_sync(~0u, unit[0], step % 4 * kStepPages + n), u1 = __shfl_sync(~0u, unit[1], step % 4 * kStepPages + n);
            const int pg = step < 4 ? pg0 : pg1;
            const float u = step < 4 ? u0 : u1;
            for (int r = lane / kStepPages; r < n_rows && blk < end_page; r += 4) {
                const int from = B.group <= 16 ? r * B.group : 0, to = B.group <= 16 ? from + B.group : min(16, B.group - mt * 16);
                int best = tile_score[warp][from][n];
                for (int g = from + 1; g < to; ++g) best = max(best, tile_score[warp][g][n]);
                const int place = s.first + r0 + r, own = min(place, s.len - 1) >> B.page_shift;
                unsigned key = 0;
                if (pg >= 0 && place >= 0 && blk <= own) key = blk < a.first || blk > own - a.last ? kAlways : ordered_score(float(best) * u);
                unsigned* const to_key = kFew ? ranked[kFew ? r : 0] + blk : a.keys + ((long long)(s.row0 + r0 + r - a.row0) * B.kv_heads + h) * a.stride + blk;
                *to_key = mt > 0 ? max(*to_key, key) : key;
            }
            __syncwarp();
        }
    }
    if constexpr (kFew) {
        static_assert(kMostSteps * kStepPages * kScoreWarps >= kRanked, "all pages in a chunk");
        __syncthreads();
        for (int r = 0; r < n_rows; ++r) {
            const int place = min(s.first + r0 + r, s.len - 1), n = place >= 0 ? (place >> B.page_shift) + 1 : 0, row = s.row0 + r0 + r;
            // behind the row's own page there are zeros up to whole fours
            if (tid < 4 && n + tid < (n + 3) / 4 * 4) ranked[r][n + tid] = 0;
            __syncthreads();
            pick_by_rank(ranked[r], sums, n, a.chosen + row * a.chosen_row + h * a.chosen_head, a.count);
        }
    }
}

// ---- the best
// Of at most kRanked keys, each one's rank. A block's work; sums: a number to a warp.
__device__ __forceinline__ void pick_by_rank(const unsigned* ranked, int* sums, int n, int* out, int count) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, threads = blockDim.x;
    int before = 0;
    for (int i0 = 0; i0 < n; i0 += threads) {
        const int i = i0 + tid;
        const unsigned mine = i < n ? ranked[i] : 0u;
        int rank = 0;
        if (mine)
#pragma unroll 4
            for (int j = 0; j < n; j += 4) {
                const uint4 k = *reinterpret_cast<const uint4*>(ranked + j);
                rank += (k.x > mine || k.x == mine && j < i) + (k.y > mine || k.y == mine && j + 1 < i) +
                        (k.z > mine || k.z == mine && j + 2 < i) + (k.w > mine || k.w == mine && j + 3 < i);
            }
        const unsigned who = __ballot_sync(~0u, mine && rank < count);
        if (lane == 0) sums[warp] = __popc(who);
        __syncthreads();
        int at = before + __popc(who & ((1u << lane) - 1));
        for (int w = 0; w < threads / 32; ++w) {
            if (w < warp) at += sums[w];
            before += sums[w];
        }
        if (who >> lane & 1) out[at] = i;
        __syncthreads();
    }
    for (int i = before + tid; i < count; i += threads) out[i] = -1;
}

constexpr int kHeld = 8;                         // keys that a thread holds
constexpr int kMostThreads = 1024;

// A block has one row and kv head. Few pages: each key's rank. Else the count-th largest key, two bits at a time from the top - how many
// keys reach each of three candidates is one sum over the block -; a thread has neighbouring pages, so that what is chosen comes out
// in order. (By histograms of 11 bits in shared memory, whose upper digits are all alike: 4690 pages 10 us, so 4.)
__global__ void __launch_bounds__(kMostThreads) choose_pick_kernel(ChooseArgs a) {
    __shared__ __align__(16) unsigned ranked[kRanked];
    __shared__ int sums[2][kMostThreads / 32][3];
    const Batch& B = a.b;
    const int tid = threadIdx.x, threads = blockDim.x, warps = threads / 32, lane = tid & 31, warp = tid / 32;
    grid_dependency_trigger();
    grid_dependency_wait();
    const int h = blockIdx.x % B.kv_heads, rest = blockIdx.x / B.kv_heads, r = rest % B.max_rows, b = rest / B.max_rows;
    const paged::Sequence s = paged::sequence(B, b);
    const int row = s.row0 + r;
    if (r >= s.n || row < a.row0 || row >= a.row0 + a.rows) return;
    int* const out = a.chosen + row * a.chosen_row + h * a.chosen_head;
    const int place = s.first + r, top = min(place, s.len - 1), n = top >= 0 ? (top >> B.page_shift) + 1 : 0;
    const unsigned* const keys = a.keys + ((long long)(row - a.row0) * B.kv_heads + h) * a.stride;      // 16-byte aligned
    if (n <= kRanked) {
        if (tid < kRanked) ranked[tid] = tid < n ? keys[tid] : 0u;
        __syncthreads();
        pick_by_rank(ranked, &sums[0][0][0], n, out, a.count);
        return;
    }
    // a thread's pages [i0, i1): kHeld of them in registers, or, of more, whole fours in memory
    const bool holds = n <= threads * kHeld;
    const int per = holds ? kHeld : (n + threads * 4 - 1) / (threads * 4) * 4, i0 = min(tid * per, n), i1 = min(i0 + per, n);
    unsigned held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; i += 4) {
        uint4 k = make_uint4(0u, 0u, 0u, 0u);
        if (holds && i0 + i < i1) k = *reinterpret_cast<const uint4*>(keys + i0 + i);       // (a row of keys has whole fours)
        held[i] = k.x;
        held[i + 1] = i0 + i + 1 < i1 ? k.y : 0u;
        held[i + 2] = i0 + i + 2 < i1 ? k.z : 0u;
        held[i + 3] = i0 + i + 3 < i1 ? k.w : 0u;
    }
    const auto each = [&](auto f) {              // f(number, key), 0 for none
        if (holds) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i) f(i0 + i, held[i]);
        } else {
            for (int i = i0; i < i1; ++i) f(i, keys[i]);
        }
    };
    unsigned border = 0;
#pragma unroll 1
    for (int shift = 30, side = 0; shift >= 0; shift -= 2, side ^= 1) {
        int c[3] = {0, 0, 0};
        each([&](int, unsigned k) {
#pragma unroll
            for (int x = 0; x < 3; ++x) c[x] += k >= (border | unsigned(x + 1) << shift);
        });
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            const int sum = __reduce_add_sync(~0u, c[x]);
            if (lane == 0) sums[side][warp][x] = sum;
        }
        __syncthreads();                         // (the other half of the sums is written next)
        unsigned digit = 0;
#pragma unroll
        for (int x = 0; x < 3; ++x) digit += __reduce_add_sync(~0u, lane < warps ? sums[side][lane][x] : 0) >= a.count;
        border |= digit << shift;
    }
    // what is above the border is chosen, and of what equals it - with a border of 0 none, there are fewer than count - the first
    int more = 0, same = 0;
    each([&](int, unsigned k) {
        more += k > border;
        same += border && k == border;
    });
    int m = more, e = same;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(~0u, m, d), q = __shfl_up_sync(~0u, e, d);
        if (lane >= d) { m += o; e += q; }
    }
    __syncthreads();
    if (lane == 31) { sums[0][warp][0] = m; sums[0][warp][1] = e; }
    __syncthreads();
    const int wm = lane < warps ? sums[0][lane][0] : 0, we = lane < warps ? sums[0][lane][1] : 0;
    const int all_more = __reduce_add_sync(~0u, wm), all_same = __reduce_add_sync(~0u, we), equal = a.count - all_more;
    int before_more = m - more + __reduce_add_sync(~0u, lane < warp ? wm : 0), before_same = e - same + __reduce_add_sync(~0u, lane < warp ? we : 0);
    each([&](int i, unsigned k) {
        const bool is = border && k == border;
        if (k > border || is && before_same < equal) out[before_more + min(before_same, equal)] = i;
        before_more += k > border;
        before_same += is;
    });
    for (int i = all_more + min(all_same, equal) + tid; i < a.count; i += threads) out[i] = -1;
}

constexpr long long kMostKeys = 64ll << 20;      // of a launch: 256 MB

long long key_stride(const Batch& b) { return b.max_kv_len > 0 ? ((((b.max_kv_len - 1) >> b.page_shift) + 1) + 3) / 4 * 4 : 4; }      // whole 16 bytes
long long rows_at_once(const Batch& b) {
    const long long n = kMostKeys / (key_stride(b) * b.kv_heads);
    return n < 1 ? 1 : (n < b.n_rows ? n : b.n_rows);
}
int tile_rows(const Batch& b) {
    const int per = b.group >= 16 ? 1 : 16 / b.group, rows = b.max_rows < b.n_rows ? b.max_rows : b.n_rows;
    return per < rows ? per : rows;
}
size_t query_bytes(const Batch& b) { return size_t(div_up(tile_rows(b) * b.group, 16)) * 2 * div_up(b.dim, 64) * 1024; }
// Few pages, and few rows to a block: one launch.
bool few_form(const Batch& b) { return key_stride(b) <= kRanked && tile_rows(b) <= kFewRows && query_bytes(b) <= (32u << 10); }
// Raises the kernel's limit of shared memory to what the largest group of heads takes, once for each device: another thread's call may be between its
// own raise and its launch.
constexpr int kMostGroup = 256, kMostQueries = kMostGroup / 16 * 2 * 4 * 1024;
template <typename Kernel>
cudaError_t allow_queries(Kernel kernel) {
    static std::atomic<uint64_t> sized{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && !(sized.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostQueries);
        if (e == cudaSuccess) sized.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
    }
    return e;
}
int failed(cudaError_t e) {
    set_last_error(e);
    (void)cudaGetLastError();
    return OGLE_ERR_CUDA;
}

}  // namespace
}  // namespace ogle

using namespace ogle;

extern "C" {

int ogle_cuda_page_bounds(const OglePagedBatch* batch, signed char* bounds, float* bounds_scale, ogle_stream_t stream) {
    BoundsArgs a = {};
    const int rc = paged::translate(batch, a.b);
    if (rc != OGLE_OK) return rc;
    if (a.b.n_seqs == 0) return OGLE_OK;
    if (!bounds || !bounds_scale) return OGLE_ERR_INVALID;
    if (!aligned16(bounds)) return OGLE_ERR_ALIGNMENT;
    if (a.b.max_rows == 0 || a.b.max_kv_len == 0) return OGLE_OK;
    a.bounds = bounds;
    a.scale = bounds_scale;
    const long long rows = a.b.max_rows < a.b.n_rows ? a.b.max_rows : a.b.n_rows;
    a.per_seq = rows == 1 ? 1 : int((rows + (1 << a.b.page_shift) - 2) >> a.b.page_shift) + 1;
    if ((long long)a.per_seq * a.b.n_seqs >= (1LL << 31)) return OGLE_ERR_UNSUPPORTED;
    const cudaError_t e = launch_overlapped(page_bounds_kernel, dim3(a.per_seq * a.b.n_seqs, a.b.kv_heads), dim3(kBoundThreads), 0, stream, a);
    return e == cudaSuccess ? finish_launch() : failed(e);
}

size_t ogle_cuda_choose_pages_workspace_bytes(const OglePagedBatch* batch, const OgleChooseParams* p) {
    Batch b;
    if (!p || paged::translate(batch, b) != OGLE_OK || b.n_seqs == 0 || b.max_rows == 0 || b.max_kv_len == 0 || few_form(b)) return 0;
    return size_t(rows_at_once(b) * b.kv_heads * key_stride(b)) * sizeof(unsigned);
}

int ogle_cuda_choose_pages(const OglePagedBatch* batch, const OgleChooseParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream) {
    ChooseArgs a = {};
    const int rc = paged::translate(batch, a.b);
    if (rc != OGLE_OK) return rc;
    if (!p || p->count < 1 || p->first < 0 || p->last < 1 || p->first > p->count || p->last > p->count - p->first) return OGLE_ERR_INVALID;
    Batch& B = a.b;
    if (B.n_seqs == 0) return OGLE_OK;
    if (!p->q || !p->bounds || !p->bounds_scale || !p->chosen) return OGLE_ERR_INVALID;
    if (p->chosen_head < p->count || p->chosen_row < p->count) return OGLE_ERR_INVALID;
    if (!paged::strides_ok(p->q, p->q_row, p->q_head, batch->dtype) || !aligned16(p->bounds)) return OGLE_ERR_ALIGNMENT;
    if (B.group > kMostGroup) return OGLE_ERR_UNSUPPORTED;
    if (B.max_rows == 0) return OGLE_OK;
    const size_t needed = ogle_cuda_choose_pages_workspace_bytes(batch, p);
    if (needed > 0 && (!workspace || workspace_bytes < needed)) return OGLE_ERR_INVALID;
    if (!aligned16(workspace)) return OGLE_ERR_ALIGNMENT;
    a.q = p->q; a.q_row = p->q_row; a.q_head = p->q_head;
    a.bounds = p->bounds; a.scale = p->bounds_scale;
    a.chosen = p->chosen; a.chosen_row = p->chosen_row; a.chosen_head = p->chosen_head;
    a.count = p->count; a.first = p->first; a.last = p->last;
    a.keys = static_cast<unsigned*>(workspace);
    a.stride = key_stride(B);
    if (B.max_rows > B.n_rows) B.max_rows = B.n_rows;
    const int per = B.group >= 16 ? 1 : 16 / B.group;
    a.tiles = div_up(B.max_rows, per);
    // A chunk is one to eight steps of a block: as many as leave the GPU four blocks an SM.
    constexpr int kScoreWarps = kWarps;
    const long long tiles = (long long)B.n_seqs * a.tiles * B.kv_heads, steps = div_up(a.stride, kScoreWarps * kStepPages);
    long long each = tiles * steps / (4 * kNumSMs);
    each = each < 1 ? 1 : (each > kMostSteps ? kMostSteps : each);
    a.chunk_pages = int(each) * kScoreWarps * kStepPages;
    a.chunks = div_up(a.stride, a.chunk_pages);
    const long long blocks = (long long)B.n_seqs * a.tiles * B.kv_heads * a.chunks, picks = (long long)B.n_seqs * B.max_rows * B.kv_heads;
    if (blocks >= (1LL << 31) || picks >= (1LL << 31)) return OGLE_ERR_UNSUPPORTED;
    const size_t queries = query_bytes(B);
    int threads = div_up(a.stride, kHeld * 32) * 32;
    threads = threads < kRanked ? kRanked : (threads > kMostThreads ? kMostThreads : threads);
    if (few_form(B)) {
        if (tiles >= (1LL << 31)) return OGLE_ERR_UNSUPPORTED;
        a.rows = B.n_rows;
        a.chunks = 1;
        a.chunk_pages = kRanked;
        const cudaError_t e = launch_overlapped(choose_score_kernel<kWarps, true>, dim3(unsigned(tiles)), dim3(kWarps * 32), queries, stream, a);
        return e == cudaSuccess ? finish_launch() : failed(e);
    }
    const auto score = choose_score_kernel<kWarps, false>;
    if (queries > (44u << 10)) {
        const cudaError_t e = allow_queries(score);
        if (e != cudaSuccess) return failed(e);
    }
    const long long at_once = rows_at_once(B);
    for (long long row0 = 0; row0 < B.n_rows; row0 += at_once) {
        a.row0 = int(row0);
        a.rows = int(B.n_rows - row0 < at_once ? B.n_rows - row0 : at_once);
        cudaError_t e = launch_overlapped(score, dim3(unsigned(blocks)), dim3(kScoreWarps * 32), queries, stream, a);
        if (e != cudaSuccess) return failed(e);
        int done = finish_launch();
        if (done != OGLE_OK) return done;
        e = launch_overlapped_if(overlapped_launches_enabled(true), choose_pick_kernel, dim3(unsigned(picks)), dim3(threads), 0, stream, a);
        if (e != cudaSuccess) return failed(e);
        done = finish_launch();
        if (done != OGLE_OK) return done;
    }
    return OGLE_OK;
}

}  // extern "C"
