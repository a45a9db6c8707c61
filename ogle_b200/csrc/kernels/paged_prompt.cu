// Attention over the paged 8-bit cache for many rows of a sequence: prompts, on the tensor cores (tcgen05).
//
// A block has 256 rows (row of the sequence x query head of the group) of one sequence and kv head, as two tiles of 128, and goes
// through the keys 128 at a time:
//   four warps    read a tile of keys and of values ahead into registers and turn them into fp16 operands: e4m3 is exact in fp16, and
//                 a page's scale relative to the largest of the item is a power of two that is multiplied in on the way (exact
//                 down to 2^-15 of the largest), so that scores and weights know nothing of pages. Where an item's pages lie
//                 further apart, bytes alone are converted and the rows multiply by their pages' scales (see `apart`; the
//                 prompts below take 715 us then)
//   one thread    issues the products: S = Q K^T per tile, O += P V per tile, P taken from tensor memory
//   2 x 4 warps   a row a thread: maximum, weights 2^(x - off), their sum; P in fp16 over S; O rescaled when a row's maximum
//                 has grown by more than 2^8
// While one tile of rows is being weighted, the other's products run. Weights are handed over in two steps of 64 keys, so that the
// first sums run while the second half is being weighted. P lies over S in tensor memory (2 x 128 columns for S, 2 x DP for O), so
// the next S of a tile of rows is asked for once its P V is through.
// Shared memory has the products' operands to deliver beside the conversion's traffic; two S of 64 keys a tile of rows, which
// overlap more, read the queries twice as often and were slower (3.2 us a tile of keys, so 2.1). The tensor pipe and the special
// function units are each busy for half of the time where texts are long (2048 rows over 30000 tokens: 1011 us, 1029 TFLOP/s, 51 % both
// by the counters); taking a quarter of the exponentials off the latter, by a polynomial, made it slower. Six prompts of 2000 rows over 2500 earlier tokens: 326 us, 546 TFLOP/s - an item's beginning and end
// (queries, the first scores, the last sums, results: 10 us) take as long as its tiles there.
//
// Work: items (sequence, tile of 256 rows, kv head) laid end to end by their tiles of keys, cut into one range a block; parts
// of items that were cut go to the workspace and are joined as in the form for few rows (paged_attention.cu). The ranges'
// beginnings are found by a launch of one block (paged_plan_kernel).
#include "paged_attention.cuh"

namespace ogle {
namespace {

using namespace paged;

constexpr int kKeys = 128;                       // of a tile
constexpr int kStep = 64;                        // of a step: half a tile
constexpr int kTileRows = 128, kItemRows = 2 * kTileRows;
constexpr int kItemCost = 10;                    // tiles that an item's beginning and end take as long as: 20000 cycles, a tile 2000 to 4000
constexpr int kThreads = 16 * 32;                // 8 warps of rows, 4 of conversion, one for products and three that fill up its group
// Registers of a thread: a row has its 128 scores in them. (2 x 176 + 112 + 48) x 128 = the 128 of 512 threads at launch.
constexpr int kRowRegisters = 176, kConvertRegisters = 112, kIssueRegisters = 48;
constexpr int kConvertWarp = 8, kProductWarp = 12;
// Spread, as a power of two, up to which an item's scales are multiplied into its operands. Keys: all are exact fp16 numbers then. Values, too,
// but weights end at 2^-25 against a largest of 2^7 at least, and one that counts as 0 loses 2^-32 of a value 2^8 times the row's: 2^12 of
// them lose 2^-12, as much as a weight's own rounding.
constexpr int kKeySpread = 15, kValueSpread = 8;
constexpr float kLargeScore = 4194304.f;         // 2^22: larger ones leave the fused sums
constexpr int kNanKeys = 8192;                   // pieces of 16 values with a NaN that an item's edges can have: 1024 keys x 8

// A piece of 16 values of a token at an item's edge: which of them are NaN.
struct NanPiece { int key; uint16_t bits, unit; };

struct Start { int b, rt, h, off; };             // where a range begins: sequence, tile of rows, kv head, what of the item lies before; b -1: nowhere
struct Plan { long long total; int ranges, cost; };   // what all items count; ranges that it is cut into; what an item's ends count of it

struct PromptArgs {
    AttnArgs a;
    const Plan* plan;
    const Start* starts;
    NanPiece* nans;                              // [ranges][kNanKeys]
    int max_tiles;                               // tiles of rows that a sequence can have
};

template <int DP>
struct Layout {
    static constexpr int kHalf = kTileRows * 128;                 // 64 elements of 128 rows
    static constexpr int kTile = DP / 64 * kHalf;                 // a tile of fp16
    static constexpr int kQ = 0, kK = kQ + 2 * kTile, kV = kK + 2 * kTile;
    static constexpr int kSmem = kV + 2 * kTile + 1024;
    static constexpr int kPart = kItemRows * (DP + 2);
    static constexpr int kO = 256;                                // first column of O in tensor memory
};

__device__ __forceinline__ Sequence prompt_sequence(const AttnArgs& a, int b) {
    Sequence s = sequence(a.b, b);
    if ((long long)s.n * a.b.group <= a.few_limit) s.n = 0;
    return s;
}

// Tiles of keys that rows [m0, m_end) of the sequence attend.
__device__ __forceinline__ int key_tiles(const Span& k) { return k.hi > k.lo ? (k.hi - (k.lo & ~(kChunk - 1)) + kKeys - 1) / kKeys : 0; }
__device__ __forceinline__ Span item_span(const AttnArgs& a, const Sequence& s, int rt) {
    const int m0 = rt * kItemRows, m_end = min(s.n * a.b.group, m0 + kItemRows);
    return span_of(s, m0 / a.b.group, (m_end - 1) / a.b.group, a.causal, a.window);
}
// Tiles of keys of tile rt of a sequence's rows; -1 where there is no such item, or no key for the whole sequence.
__device__ __forceinline__ int item_tiles(const AttnArgs& a, const Sequence& s, int rt) {
    if (s.n <= 0 || rt >= row_tiles(a.b, s.n, kItemRows)) return -1;
    const Span all = span_of(s, 0, s.n - 1, a.causal, a.window);
    return all.hi > all.lo ? key_tiles(item_span(a, s, rt)) : -1;
}

// One block: sums all items, and each range's thread looks up which of them it begins in. An item's ends count as kItemCost tiles, but as
// a quarter of a range at most (and 1 at least: an item whose rows attend nothing is somebody's, too), so that short ranges are not
// spent on them.
__global__ void __launch_bounds__(1024) paged_plan_kernel(AttnArgs a, int max_tiles, int ranges, Plan* plan, Start* starts) {
    __shared__ long long sums[2][32], ends[1024];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long n = (long long)a.b.n_seqs * max_tiles;
    grid_dependency_trigger();
    grid_dependency_wait();
    const auto tiles_at = [&](long long i, int& b, int& rt) {
        b = int(quotient(i, max_tiles));
        rt = int(i - (long long)b * max_tiles);
        return i < n ? item_tiles(a, prompt_sequence(a, b), rt) : -1;
    };
    long long tiles = 0, items = 0;
    for (long long i = tid; i < n; i += 1024) {
        int b, rt;
        const int t = tiles_at(i, b, rt);
        if (t >= 0) { tiles += t; ++items; }
    }
#pragma unroll
    for (int d = 16; d; d /= 2) {
        tiles += __shfl_xor_sync(~0u, tiles, d);
        items += __shfl_xor_sync(~0u, items, d);
    }
    if (lane == 0) { sums[0][warp] = tiles; sums[1][warp] = items; }
    __syncthreads();
    tiles = sums[0][lane];
    items = sums[1][lane];
#pragma unroll
    for (int d = 16; d; d /= 2) {
        tiles += __shfl_xor_sync(~0u, tiles, d);
        items += __shfl_xor_sync(~0u, items, d);
    }
    const int heads = a.b.kv_heads, cost = int(max(1LL, min((long long)kItemCost, quotient(tiles * heads, 4LL * ranges))));
    const long long total = (tiles + items * cost) * heads;
    const int used = int(min((long long)ranges, total));
    if (tid == 0) *plan = Plan{total, used, cost};
    const long long at = tid < used ? quotient(total * tid, used) : -1;    // a thread to a range: there are no more than threads
    if (tid < ranges && tid >= used) starts[tid].b = -1;
    long long before = 0;
    for (long long i0 = 0; i0 < n; i0 += 1024) {
        int b, rt;
        const int t = tiles_at(i0 + tid, b, rt);
        long long sum = t < 0 ? 0 : (long long)(t + cost) * heads;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const long long u = __shfl_up_sync(~0u, sum, d);
            if (lane >= d) sum += u;
        }
        __syncthreads();
        if (lane == 31) sums[0][warp] = sum;
        __syncthreads();
        long long all = sums[0][lane];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const long long u = __shfl_up_sync(~0u, all, d);
            if (lane >= d) all += u;
        }
        const long long ahead = __shfl_sync(~0u, all, max(warp - 1, 0));
        all = __shfl_sync(~0u, all, 31);
        ends[tid] = before + sum + (warp > 0 ? ahead : 0);
        __syncthreads();
        if (at >= before && at < before + all) {
            int lo = 0, hi = 1023;                 // the first item that ends behind the range's beginning
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (ends[mid] > at) hi = mid;
                else lo = mid + 1;
            }
            const int c = tiles_at(i0 + lo, b, rt) + cost;
            const long long x = at - (ends[lo] - (long long)c * heads), h = quotient(x, c);
            starts[tid] = Start{b, rt, int(h), int(x - h * c)};
        }
        before += all;
    }
}

// A block's place in its range, and the item that it has.
struct Walk { long long at, end, total; int ranges, cost, b, rt, h, off; };
struct Item {
    Sequence s;
    int b, h, m0, m_end;
    int c0, c1, cost;
    int j0, tiles;                               // first key of its first tile; tiles of this part
    Span keys;
    int inner_lo, inner_hi;                      // keys that every row attends
};

__device__ __forceinline__ bool next_item(const PromptArgs& p, Walk& w, Item& g) {
    const AttnArgs& a = p.a;
    const Batch& B = a.b;
    while (w.at < w.end && w.b < B.n_seqs) {
        g.s = prompt_sequence(a, w.b);
        const int tiles = item_tiles(a, g.s, w.rt);
        g.cost = tiles + w.cost;
        if (tiles < 0) {
            w.rt = w.h = w.off = 0;
            ++w.b;
            continue;
        }
        g.b = w.b;
        g.h = w.h;
        g.m0 = w.rt * kItemRows;
        g.m_end = min(g.s.n * B.group, g.m0 + kItemRows);
        g.keys = item_span(a, g.s, w.rt);
        g.inner_lo = span_of(g.s, (g.m_end - 1) / B.group, 0, a.causal, a.window).lo;
        g.inner_hi = span_of(g.s, 0, g.m0 / B.group, a.causal, a.window).hi;
        g.c0 = w.off;
        g.c1 = int(min((long long)g.cost, w.off + (w.end - w.at)));
        const int t0 = max(g.c0 - w.cost, 0), t1 = max(g.c1 - w.cost, 0);
        g.j0 = (g.keys.lo & ~(kChunk - 1)) + t0 * kKeys;
        g.tiles = t1 - t0;
        if (g.c0 == 0 && g.c1 < g.cost) {
            const long long item_end = w.at + g.cost;
            const int last = min(int(quotient(item_end * w.ranges + w.total - 1, w.total)), w.ranges);
            a.cuts[blockIdx.x] = Cut{g.m_end - g.m0, g.s.row0, g.h, g.m0, int(blockIdx.x), last, 0, 0, w.total};
        }
        w.at += g.c1 - g.c0;
        w.off = 0;
        if (++w.h == B.kv_heads) { w.h = 0; ++w.rt; }
        return true;
    }
    return false;
}

// ---- tensor memory
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// Nothing that uses the loaded values may come before this.
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
          "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
          "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
          "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Operand whose rows run along the multiply's row or column side, 64 of them side by side in 128 bytes of the 128-byte swizzle
// (values: a token's elements): 8 tokens are 1024 bytes on, the next 64 elements `next` bytes.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t next) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(next >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// The four products of 64 elements of the reduction, issued from one block of instructions: the descriptors of the later ones
// are sums with constants, and the issuing thread does nothing in between. Queries by keys: 32 bytes on for each.
__device__ __forceinline__ void products_scores(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 q, 0, 0;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\t"
        "add.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
        "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, q;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, q;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, q;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Weights (in tensor memory, 8 columns for 16 keys) by values: 16 tokens, 2048 bytes, on for each.
__device__ __forceinline__ void products_sums(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 q, 0, 0;\n\t"
        "add.u32 a1, %1, 8;\n\tadd.s64 b1, %2, 128;\n\t"
        "add.u32 a2, %1, 16;\n\tadd.s64 b2, %2, 256;\n\t"
        "add.u32 a3, %1, 24;\n\tadd.s64 b3, %2, 384;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, q;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, q;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, q;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

struct Bars {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t q_full, s_full[2], p_full[2][2], pv_done[2][2], drain;      // [tile of rows][step of the tile of keys]
};

// A row's scores and weights where the item's pages lie apart, or scores are too large for the fused sums of the first loop, for its tiles
// from `state.tile` on; false where scores did not come.
// Scores are read twice, 32 at a time: this runs rarely, and needs few registers so. x = s rk is rounded before `off` is taken
// away - the row's largest x comes to kLift however large it is -, and O is of w 2^(log2 scale + up), with the row's largest w x scale
// near 2^kLift (as in the form for few rows).
struct RowState { int tile; float off, up, l; };
template <int DP>
__device__ __noinline__ bool rows_apart(const AttnArgs& a, const Item& item, Bars& bars, volatile int* abort, int q, Span k, float rs, bool apart, int j_first, int tiles,
                                        uint32_t my_tiles, uint32_t s_at, uint32_t o_at, RowState& state) {
    float off = state.off, up = state.up, l = state.l;
    const Batch& B = a.b;
    const int lane = threadIdx.x % 32, h = item.h;
    for (int t = state.tile; t < tiles; ++t) {
        const bool came = tc::wait_turn(&bars.s_full[q], (my_tiles + t) & 1, abort, a.spin_limit);
        if (!__all_sync(~0u, came)) {
            if (!came && !*abort) {
                *abort = 1;
                tc::record_error(a.error, kGaveUp);
            }
            return false;
        }
        after_sync();
        // factors of the tile's eight chunks, a lane each; no page: no key
        const int j0 = j_first + t * kKeys, j = j0 + (lane & 7) * kChunk, page = j < item.keys.hi ? page_of(B, item.b, j >> B.page_shift) : -1;
        const float ks = page < 0 ? -1.f : (apart ? __ldg(B.k_scale + (long long)page * B.kv_heads + h) : 1.f);
        const float vs = page < 0 ? 0.f : (apart ? __ldg(B.v_scale + (long long)page * B.kv_heads + h) : 1.f);
        const float v_log = vs > 0.f ? float(int(__float_as_uint(vs) >> 23) - 127) : -INFINITY;
        const auto read = [&](int c, uint32_t (&s)[32]) {
            tmem_load32(s, s_at + c * 32);
            tmem_loaded(s);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int key = j0 + c * 32 + i;
                const float k_scale = __shfl_sync(~0u, ks, c * 2 + i / kChunk);
                const float x = __fmul_rn(__uint_as_float(s[i]), fmaxf(rs * k_scale, 1e-37f));
                s[i] = key < k.lo || key >= k.hi || k_scale < 0.f ? 0xff800000u : __float_as_uint(x);
            }
        };
        float x[kKeys / kChunk], top = -INFINITY, high = INFINITY;       // of each chunk the largest
        bool more = false;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            read(c, s);
#pragma unroll
            for (int g = 2 * c; g < 2 * c + 2; ++g) {
                x[g] = __uint_as_float(s[g % 2 * kChunk]);
#pragma unroll
                for (int i = 1; i < kChunk; ++i) x[g] = fmaxf(x[g], __uint_as_float(s[g % 2 * kChunk + i]));
                top = fmaxf(top, x[g]);
                more |= x[g] - off + fmaxf(__shfl_sync(~0u, v_log, g) + up, 0.f) > kHeadroom + kLift;
            }
        }
        if (__any_sync(~0u, more)) {
            const float now = fmaxf(off, top - kLift), move = off - now;
#pragma unroll
            for (int g = 0; g < kKeys / kChunk; ++g) high = fminf(high, kLift - (x[g] - now) - __shfl_sync(~0u, v_log, g));
            high = fminf(high, up - move);
            const float f = exp2_fast(move + (high - up));
            if (t > 0)
#pragma unroll 1
                for (int c = 0; c < DP / 16; ++c) {
                    uint32_t o[16];
                    tmem_load16(o, o_at + c * 16);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tc::tmem_st16(o_at + c * 16, o);
                }
            l *= exp2_fast(move);
            off = now;
            up = high;
        }
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            uint32_t s[32], w[16];
            read(c, s);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const float by = exp2_fast(fminf(__shfl_sync(~0u, v_log, c * 2 + i / kChunk) + up, 126.f));
                const float e = exp2_fast(__uint_as_float(s[i]) - off), f = exp2_fast(__uint_as_float(s[i + 1]) - off);
                l += e + f;
                w[i / 2] = half2_bits(e * by, f * by);
            }
            tc::tmem_st16(s_at + c / 2 * kStep + c % 2 * 16, w);
            if (c & 1) {
                tmem_stored();
                before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bars.p_full[q][c / 2]);
            }
        }
    }
    state = RowState{tiles, off, up, l};
    return true;
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
paged_prompt_kernel(const __grid_constant__ PromptArgs p) {
    using L = Layout<DP>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ __align__(8) Bars bars;
    __shared__ Walk walk;
    __shared__ Item item;
    __shared__ uint32_t tmem_slot, top_scale[2], low_scale[2];    // bits of the item's largest and smallest scales of keys and values
    __shared__ float row_scale[2][kTileRows];      // 2^e that a row's queries were divided by
    __shared__ int more_items, odd_pages, nan_count;
    __shared__ volatile int gave_up;
    unsigned char* const smem = dynamic + ((1024 - (tc::smem_u32(dynamic) & 1023)) & 1023);
    const uint32_t base = tc::smem_u32(smem);
    const AttnArgs& a = p.a;
    const Batch& B = a.b;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&bars.k_full[i], 4); tc::mbar_init(&bars.v_full[i], 4);
            tc::mbar_init(&bars.k_empty[i], 1); tc::mbar_init(&bars.v_empty[i], 1);
            tc::mbar_init(&bars.s_full[i], 1);
            for (int j = 0; j < 2; ++j) { tc::mbar_init(&bars.p_full[i][j], 4); tc::mbar_init(&bars.pv_done[i][j], 1); }
        }
        tc::mbar_init(&bars.q_full, 8);
        tc::mbar_init(&bars.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        gave_up = 0;
        top_scale[0] = top_scale[1] = 0;
        low_scale[0] = low_scale[1] = ~0u;
        odd_pages = nan_count = 0;
    }
    if (warp == kProductWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    grid_dependency_trigger();
    grid_dependency_wait();
    if (tid == 0) {
        a.cuts[blockIdx.x].rows = 0;
        const Start s = p.starts[blockIdx.x];
        const Plan plan = *p.plan;
        more_items = 0;
        if (s.b >= 0) {                            // else: no such range
            walk = Walk{quotient(plan.total * blockIdx.x, plan.ranges), quotient(plan.total * (blockIdx.x + 1), plan.ranges), plan.total,
                        plan.ranges, plan.cost, s.b, s.rt, s.h, s.off};
            more_items = next_item(p, walk, item);
        }
    }
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tmem = tmem_slot;
    const uint32_t limit = a.spin_limit;
    volatile int* const abort = &gave_up;
    // tiles that this thread's role has been through, whatever item they were of
    uint32_t kv_tiles = 0, q_items = 0, my_tiles = 0, second_tiles = 0;
    bool failed = false;
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!failed && !tc::wait_turn(bar, parity & 1, abort, limit)) {
            failed = true;
            if (!*abort) {
                *abort = 1;
                tc::record_error(a.error, kGaveUp);
            }
        }
        return !failed;
    };

    // Every role goes through the items together: all threads look at the item's scales before it, and meet behind it.
    int j_first = 0, tiles = 0, halves = 0;        // first key, tiles of keys, tiles of rows that exist
    float k_unit = 1.f, v_unit = 1.f;              // the largest scales
    bool with_holes = false;                       // some of its tokens have no page
    // Its pages' scales lie too far apart for operands relative to the largest, or some of its values are zeros throughout (a row that
    // attends little else would keep nothing of the rest): operands are bytes, rows know of pages
    bool apart = false;
    const auto begin_item = [&]() {
        j_first = item.j0;
        tiles = item.tiles;
        const int j_last = min(item.keys.hi, j_first + tiles * kKeys);
        if (tiles > 0) {
            uint32_t top_k = 0, top_v = 0, low_k = ~0u, low_v = ~0u;
            int odd = 0;
            for (int i = (j_first >> B.page_shift) + tid; i <= (j_last - 1) >> B.page_shift; i += kThreads) {
                const int page = page_of(B, item.b, i);
                if (page < 0) { odd |= 1; continue; }
                const long long o = (long long)page * B.kv_heads + item.h;
                const uint32_t k = __float_as_uint(__ldg(B.k_scale + o)) & 0x7fffffffu, v = __float_as_uint(__ldg(B.v_scale + o)) & 0x7fffffffu;
                top_k = max(top_k, k);
                top_v = max(top_v, v);
                low_k = min(low_k, k ? k : ~0u);
                low_v = min(low_v, v ? v : ~0u);
                if (v == 0) odd |= 2;
            }
            if (top_k) { atomicMax(&top_scale[0], top_k); atomicMin(&low_scale[0], low_k); }
            if (top_v) { atomicMax(&top_scale[1], top_v); atomicMin(&low_scale[1], low_v); }
            if (odd) atomicOr(&odd_pages, odd);
        }
        __syncthreads();
        const auto spread = [&](int i) { return top_scale[i] ? int(top_scale[i] >> 23) - int(low_scale[i] >> 23) : 0; };
        apart = spread(0) > kKeySpread || spread(1) > kValueSpread || (odd_pages & 2);
        k_unit = top_scale[0] && !apart ? __uint_as_float(top_scale[0]) : 1.f;
        v_unit = top_scale[1] && !apart ? __uint_as_float(top_scale[1]) : 1.f;
        halves = item.m_end - item.m0 > kTileRows ? 2 : 1;
        with_holes = odd_pages & 1;
    };
    const auto end_item = [&]() {                  // false: no item is left, or a wait has run out
        before_sync();
        __syncthreads();
        after_sync();
        if (gave_up) return false;
        if (tid == 0) {
            top_scale[0] = top_scale[1] = 0;
            low_scale[0] = low_scale[1] = ~0u;
            odd_pages = nan_count = 0;
            more_items = next_item(p, walk, item);
        }
        __syncthreads();
        return more_items != 0;
    };

    if (warp < kConvertWarp) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
        const int q = warp / 4, r = tid & 127;           // tile, row of it
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lanes + q * kKeys, o_at = tmem + lanes + L::kO + q * DP;
        for (bool more = more_items != 0; more; more = end_item()) {
            begin_item();
            const int h = item.h;
            const bool mine = q < halves;
            const int row = min(item.m0 + q * kTileRows + r, item.m_end - 1);
            const int seq_row = row / B.group, head = h * B.group + row % B.group;
            const Span k = span_of(item.s, seq_row, seq_row, a.causal, a.window);
            if (tiles > 0 && mine) {
                // queries of the warp's 32 rows, 16 values a lane: rows side by side are read together, two rounds before the first is used (what
                // runs once an item is short code: with all eight rounds, and the results' four parts below, unrolled, its instructions took
                // longer to fetch - six prompts 359 us, so 331)
                constexpr int kLanes = DP / 16, kTogether = 32 / kLanes, kRounds = 32 / kTogether, kAtOnce = kRounds < 2 ? kRounds : 2;
                const int d = lane % kLanes * 16;
                const long long mine_at = (item.s.row0 + seq_row) * a.q_row + head * a.q_head;
                const bool back = a.scale_log2 < 0.f;        // the largest product is then the largest x
#pragma unroll 1
                for (int x0 = 0; x0 < kRounds; x0 += kAtOnce) {
                    uint4 raw[kAtOnce][2];
#pragma unroll
                    for (int x = 0; x < kAtOnce; ++x) {
                        const long long from = __shfl_sync(~0u, mine_at, (x0 + x) * kTogether + lane / kLanes);
                        const uint4* g = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.q) + from + d);
                        raw[x][0] = raw[x][1] = make_uint4(0, 0, 0, 0);
                        if (d < B.dim) { raw[x][0] = g[0]; raw[x][1] = g[1]; }
                    }
#pragma unroll
                    for (int x = 0; x < kAtOnce; ++x) {
                        const int at = (warp & 3) * 32 + (x0 + x) * kTogether + lane / kLanes;
                        const uint32_t* w = reinterpret_cast<const uint32_t*>(raw[x]);
                        float f[16], top = 0.f;
#pragma unroll
                        for (int y = 0; y < 8; ++y) {
                            const float2 g = B.dtype == OGLE_F16 ? __half22float2(*reinterpret_cast<const __half2*>(w + y)) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(w + y));
                            f[2 * y] = g.x;
                            f[2 * y + 1] = g.y;
                            top = fmaxf(top, fmaxf(fabsf(g.x), fabsf(g.y)));
                        }
#pragma unroll
                        for (int y = 1; y < kLanes; y *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, y));
                        const int e = top > 1e-30f && top <= 3e38f ? int(__float_as_uint(top) >> 23) - 126 - 12 : 0;
                        const float down = __uint_as_float(uint32_t(127 - e) << 23 | (back ? 0x80000000u : 0u));
                        if (lane % kLanes == 0) row_scale[q][at] = __uint_as_float(uint32_t(127 + e) << 23);
                        uint32_t y[8];
#pragma unroll
                        for (int z = 0; z < 8; ++z) y[z] = half2_bits(f[2 * z] * down, f[2 * z + 1] * down);
                        unsigned char* to = smem + L::kQ + q * L::kTile + (d / 64) * L::kHalf + at * 128;
                        const int c = d % 64 / 8;
                        *reinterpret_cast<uint4*>(to + (c ^ (at & 7)) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<uint4*>(to + ((c + 1) ^ (at & 7)) * 16) = make_uint4(y[4], y[5], y[6], y[7]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            __syncwarp();
            if (tiles > 0 && lane == 0) tc::mbar_arrive(&bars.q_full);
            // scores scaled by 0 are alike, hidden ones are not
            const float rs = mine && tiles > 0 ? fmaxf(fabsf(a.scale_log2) * row_scale[q][r] * k_unit, 1e-37f) : 0.f;

            float off = 0.f, bar_x = -INFINITY, l = 0.f, up = 0.f;
            int t = 0;
            for (; mine && !apart && t < tiles; ++t) {
                wait(&bars.s_full[q], my_tiles + t);
                if (__any_sync(~0u, failed)) { failed = true; break; }
                after_sync();
                const int j0 = j_first + t * kKeys;
                const bool edge = with_holes || j0 < item.inner_lo || j0 + kKeys > item.inner_hi;
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_load32(s[c], s_at + c * 32);
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_loaded(s[c]);
                if (edge) {
                    // keys that the row does not attend
                    const int lo = k.lo - j0, hi = k.hi - j0;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int x = 0; x < 32; ++x) if (c * 32 + x < lo || c * 32 + x >= hi) s[c][x] = 0xff800000u;
                    if (with_holes) {
#pragma unroll
                        for (int g = 0; g < kKeys / kChunk; ++g) {
                            const int j = j0 + g * kChunk;
                            if (j < item.keys.hi && page_of(B, item.b, j >> B.page_shift) < 0)
#pragma unroll
                                for (int x = 0; x < kChunk; ++x) s[g / 2][g % 2 * kChunk + x] = 0xff800000u;
                        }
                    }
                }
                float m[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    m[c] = __uint_as_float(s[c][0]);
#pragma unroll
                    for (int x = 1; x < 32; ++x) m[c] = fmaxf(m[c], __uint_as_float(s[c][x]));
                }
                const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * rs;
                if (__any_sync(~0u, top > bar_x)) {
                    const float old = bar_x - kHeadroom, now = fmaxf(top, old);
                    // fp32 numbers lie up to 1/4 apart below this, and further where weights would notice: the other loop's
                    if (__any_sync(~0u, top > kLargeScore || top < -kLargeScore && top > -INFINITY)) break;
                    float f = 1.f;
                    if (now > -INFINITY) {
                        f = exp2_fast(old - now);
                        off = now - kLift;
                        bar_x = now + kHeadroom;
                    }
                    l *= f;
                    if (t > 0) {
#pragma unroll 1
                        for (int c = 0; c < DP / 16; ++c) {
                            uint32_t o[16];
                            tmem_load16(o, o_at + c * 16);
#pragma unroll
                            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                            tc::tmem_st16(o_at + c * 16, o);
                        }
                    }
                }
                const unsigned long long rs2 = pair(rs, rs), off2 = pair(-off, -off);
                unsigned long long sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        float e, f;
                        unpair(fma2(pair(__uint_as_float(s[c][x]), __uint_as_float(s[c][x + 1])), rs2, off2), e, f);
                        e = exp2_fast(e);
                        f = exp2_fast(f);
                        sum[x / 2 & 1] = add2(sum[x / 2 & 1], pair(e, f));
                        w[x / 2] = half2_bits(e, f);
                    }
                    tc::tmem_st16(s_at + c / 2 * kStep + c % 2 * 16, w);          // over scores, all of which have been read
                    if (c & 1) {                          // a step's weights
                        tmem_stored();
                        before_sync();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&bars.p_full[q][c / 2]);
                    }
                }
                float e, f;
                unpair(add2(sum[0], sum[1]), e, f);
                l += e + f;
            }
            if (mine && t < tiles && !failed) {
                RowState state = {t, bar_x > -INFINITY ? off : -3e38f, 0.f, l};
                if (!rows_apart<DP>(a, item, bars, abort, q, k, rs, apart, j_first, tiles, my_tiles, s_at, o_at, state)) failed = true;
                bar_x = state.off + (kLift + kHeadroom);
                up = state.up;
                l = state.l;
            }
            if (mine && tiles > 0) {
                wait(&bars.pv_done[q][1], my_tiles + tiles - 1);
                if (__any_sync(~0u, failed)) failed = true;
                after_sync();
            }
            asm volatile("bar.sync 1, 384;" ::: "memory");    // the conversion's notes of NaNs
            if (mine && !failed) {
                uint32_t nan[4] = {0, 0, 0, 0};
                const int n = min(*(volatile int*)&nan_count, kNanKeys);
                for (int i = 0; i < n; ++i) {
                    const NanPiece* g = p.nans + (long long)blockIdx.x * kNanKeys + i;
                    const int key = *(volatile const int*)&g->key;
                    const uint32_t bits = *(volatile const uint16_t*)&g->bits, unit = *(volatile const uint16_t*)&g->unit;
                    if (key >= k.lo && key < k.hi)
#pragma unroll
                        for (int x = 0; x < 4; ++x) if (x == int(unit / 2)) nan[x] |= bits << (16 * (unit & 1));
                }
                const bool whole = item.c0 == 0 && item.c1 == item.cost, exists = item.m0 + q * kTileRows + r < item.m_end;
                // A row is a thread's; its values go through shared memory - where the tile's queries were - so that a warp stores
                // whole lines: 64 bytes of each of its rows at a time, pieces of 16 bytes turned by the row.
                unsigned char* const turn = smem + L::kQ + q * L::kTile + (warp & 3) * 32 * (DP * 2);
                // of O; in two factors where it can be near the smallest fp32 number
                const float more = exp2_fast(-0.5f * up), unit = more * v_unit;
                const float inv = !whole ? unit : (l == 0.f ? 0.f : unit / l);
#pragma unroll 1
                for (int c = 0; c < DP / 32; ++c) {
                    const uint32_t bad = c & 2 ? (c & 1 ? nan[3] : nan[2]) : (c & 1 ? nan[1] : nan[0]);
                    uint32_t o[32];
                    if (tiles > 0) {
                        tmem_load32(o, o_at + c * 32);
                        tmem_loaded(o);
                    } else {
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = 0;
                    }
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = bad >> x & 1 ? 0x7fc00000u : __float_as_uint(__uint_as_float(o[x]) * more * inv);
                    if (!whole) {                  // 128 bytes of each row
                        __syncwarp();
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            *reinterpret_cast<uint4*>(turn + lane * 128 + (x ^ (lane & 7)) * 16) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
                        __syncwarp();
                        float* const to = a.parts + ((long long)blockIdx.x * 2 + (item.c0 > 0 ? 0 : 1)) * L::kPart + (q * kTileRows + (warp & 3) * 32) * DP + c * 32;
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const int at = x * 4 + lane / 8;
                            *reinterpret_cast<uint4*>(to + at * DP + (lane & 7) * 4) = *reinterpret_cast<const uint4*>(turn + at * 128 + ((lane & 7) ^ (at & 7)) * 16);
                        }
                        continue;
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t w[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const float u = __uint_as_float(o[x * 8 + y * 2]), v = __uint_as_float(o[x * 8 + y * 2 + 1]);
                            const __nv_bfloat162 z = __floats2bfloat162_rn(u, v);
                            w[y] = B.dtype == OGLE_F16 ? half2_bits(u, v) : *reinterpret_cast<const uint32_t*>(&z);
                        }
                        *reinterpret_cast<uint4*>(turn + lane * (DP * 2) + ((c * 4 + x) ^ (lane & 7)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                if (whole) {
                    __syncwarp();
                    constexpr int kPieces = DP / 8, kTogether = 32 / kPieces;
                    const int piece = lane % kPieces, n_rows = item.m_end - item.m0 - q * kTileRows - (warp & 3) * 32;
                    const long long mine_at = (item.s.row0 + seq_row) * a.out_row + head * a.out_head;
#pragma unroll 2
                    for (int x = 0; x < 32; x += kTogether) {
                        const int at = x + lane / kPieces;
                        const long long to = __shfl_sync(~0u, mine_at, at);
                        const uint4 z = *reinterpret_cast<const uint4*>(turn + at * (DP * 2) + (piece ^ (at & 7)) * 16);
                        if (at < n_rows && piece * 8 < B.dim) *reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.out) + to + piece * 8) = z;
                    }
                    if (exists && a.lse)
                        a.lse[(long long)(item.s.row0 + seq_row) * B.q_heads + head] = l == 0.f ? -INFINITY : (bar_x - kHeadroom - kLift + log2f(l)) * 0.6931471805599453f;
                } else if (exists) {
                    float* const part = a.parts + ((long long)blockIdx.x * 2 + (item.c0 > 0 ? 0 : 1)) * L::kPart + kItemRows * DP + q * kTileRows + r;
                    part[0] = bar_x - kHeadroom;
                    part[kItemRows] = l;
                }
            }
            if (mine) my_tiles += tiles;
        }
    } else if (warp < kProductWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegisters));
        // a piece is 16 values of a token; eight lanes that store together have two tokens' four pieces: different banks. A warp has 32
        // tokens of a tile: two groups of 16, each in one page
        constexpr int kHalves = DP / 64, kRounds = 4;
        const int piece = lane & 3, row8 = lane >> 2, cw = warp - kConvertWarp;
        for (bool more = more_items != 0; more; more = end_item()) {
            begin_item();
            const int h = item.h, in_page = (1 << B.page_shift) - 1;
            const float k_inverse = apart ? 1.7014118e38f : 1.f / k_unit, v_inverse = apart ? 1.7014118e38f : 1.f / v_unit;
            int page[2];                           // of the tile whose values are asked for next
            float rk[2], rv[2];                    // scales of the tile that has been asked for, against the largest
            uint4 k_raw[kRounds][kHalves], v_raw[kRounds][kHalves];
            const auto look_up = [&](int t) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int j = j_first + t * kKeys + cw * 32 + g * kChunk;
                    page[g] = t < tiles && j < item.keys.hi ? page_of(B, item.b, j >> B.page_shift) : -1;
                }
            };
            const auto ask = [&](int t, const unsigned char* cache, const float* scales, float inverse, uint4 (&raw)[kRounds][kHalves], float (&ratio)[2]) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    ratio[g] = 0.f;
                    const int slot = (j_first + t * kKeys + cw * 32 + g * kChunk) & in_page;
                    const unsigned char* from = cache + (long long)page[g] * B.page_stride + h * B.head_stride + (long long)(slot + row8) * B.token_stride + piece * 16;
                    if (page[g] >= 0) {
                        const float scale = __ldg(scales + (long long)page[g] * B.kv_heads + h);
                        ratio[g] = fminf(scale * inverse, 1.f);       // (apart: 1, or 0)
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int half = 0; half < kHalves; ++half) {
                            raw[g * 2 + x][half] = make_uint4(0, 0, 0, 0);
                            if (page[g] >= 0 && half * 64 + piece * 16 < B.dim)
                                raw[g * 2 + x][half] = __ldg(reinterpret_cast<const uint4*>(from + x * 8 * B.token_stride + half * 64));
                        }
                }
            };
            const auto store = [&](int j0, bool clean, unsigned char* to, const uint4 (&raw)[kRounds][kHalves], const float (&ratio)[2]) {
#pragma unroll
                for (int x = 0; x < kRounds; ++x) {
                    const int r = cw * 32 + x * 8 + row8;
                    const __half2 f = __float2half2_rn(ratio[x / 2]);
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        uint32_t y[8];
                        const uint32_t w[4] = {raw[x][half].x, raw[x][half].y, raw[x][half].z, raw[x][half].w};
#pragma unroll
                        for (int z = 0; z < 4; ++z) e4m3x4_to_half2(w[z], y[2 * z], y[2 * z + 1]);
                        if (clean) {
                            // a NaN of a token that some row does not attend: out of the operand, its rows get it at the end
                            uint32_t bits = 0;
#pragma unroll
                            for (int z = 0; z < 8; ++z) {
                                const __half2 g = *reinterpret_cast<const __half2*>(&y[z]);
                                const uint32_t n = __hneu2_mask(g, g);
                                y[z] &= ~n;
                                bits |= ((n & 1) | (n >> 30 & 2)) << (2 * z);
                            }
                            const int key = j0 + r;
                            if (bits && key >= item.keys.lo && key < item.keys.hi) {
                                const int at = atomicAdd(&nan_count, 1);
                                if (at < kNanKeys) p.nans[(long long)blockIdx.x * kNanKeys + at] = NanPiece{key, uint16_t(bits), uint16_t(half * 4 + piece)};
                            }
                        }
#pragma unroll
                        for (int z = 0; z < 8; ++z) {
                            const __half2 g = __hmul2(*reinterpret_cast<const __half2*>(&y[z]), f);
                            y[z] = *reinterpret_cast<const uint32_t*>(&g);
                        }
                        unsigned char* row = to + half * L::kHalf + r * 128;
                        *reinterpret_cast<uint4*>(row + ((2 * piece) ^ (r & 7)) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<uint4*>(row + ((2 * piece + 1) ^ (r & 7)) * 16) = make_uint4(y[4], y[5], y[6], y[7]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            };
            if (tiles > 0) {
                look_up(0);
                ask(0, B.k_cache, B.k_scale, k_inverse, k_raw, rk);
                ask(0, B.v_cache, B.v_scale, v_inverse, v_raw, rv);
                look_up(1);
            }
            for (int t = 0; t < tiles; ++t) {
                const uint32_t st = kv_tiles & 1, use = kv_tiles >> 1;
                const int j0 = j_first + t * kKeys;
                const bool edge = j0 < item.inner_lo || j0 + kKeys > item.inner_hi;
                wait(&bars.k_empty[st], use + 1);
                if (__any_sync(~0u, failed)) { failed = true; break; }
                store(j0, false, smem + L::kK + st * L::kTile, k_raw, rk);
                if (lane == 0) tc::mbar_arrive(&bars.k_full[st]);
                ask(t + 1, B.k_cache, B.k_scale, k_inverse, k_raw, rk);
                wait(&bars.v_empty[st], use + 1);
                if (__any_sync(~0u, failed)) { failed = true; break; }
                if (edge) store(j0, true, smem + L::kV + st * L::kTile, v_raw, rv);
                else store(j0, false, smem + L::kV + st * L::kTile, v_raw, rv);
                if (lane == 0) tc::mbar_arrive(&bars.v_full[st]);
                ask(t + 1, B.v_cache, B.v_scale, v_inverse, v_raw, rv);
                look_up(t + 2);
                ++kv_tiles;
            }
            asm volatile("bar.sync 1, 384;" ::: "memory");
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegisters));
        for (bool more = more_items != 0; more; more = end_item()) {
            begin_item();
            if (warp == kProductWarp) {
                if (tiles > 0 && tc::elect_one()) {
                    constexpr uint32_t kF16 = (1u << 4) | ((uint32_t)(kTileRows >> 4) << 24);     // fp16 x fp16 into fp32, 128 rows
                    constexpr uint32_t kScores = kF16 | ((uint32_t)(kKeys >> 3) << 17);
                    constexpr uint32_t kSums = kF16 | (1u << 16) | ((uint32_t)(DP >> 3) << 17);   // values: elements side by side
                    const auto scores = [&](int q, int t) {     // S = Q K^T of tile t
                        const uint64_t qd = tc::umma_desc(base + L::kQ + q * L::kTile), kd = tc::umma_desc(base + L::kK + ((kv_tiles + t) & 1) * L::kTile);
#pragma unroll
                        for (int k = 0; k < DP / 64; ++k) products_scores(tmem + q * kKeys, qd + k * (L::kHalf >> 4), kd + k * (L::kHalf >> 4), kScores, k);
                        tc::umma_commit(&bars.s_full[q]);
                    };
                    const auto sums = [&](int q, int t, int step) {     // O += P V of a step of tile t; false: its weights did not come
                        if (!wait(&bars.p_full[q][step], (q ? second_tiles : my_tiles) + t)) return false;
                        after_sync();
                        products_sums(tmem + L::kO + q * DP, tmem + q * kKeys + step * kStep, desc_mn(base + L::kV + ((kv_tiles + t) & 1) * L::kTile + step * kStep * 128, L::kHalf),
                                      kSums, t + step);
                        tc::umma_commit(&bars.pv_done[q][step]);
                        return true;
                    };
                    const auto next = [&](int q, int t) {               // the next S of a tile of rows lies where its P is read
                        if (!wait(&bars.pv_done[q][1], (q ? second_tiles : my_tiles) + t)) return false;
                        after_sync();
                        scores(q, t + 1);
                        return true;
                    };
                    bool ok = wait(&bars.q_full, q_items) && wait(&bars.k_full[kv_tiles & 1], kv_tiles >> 1);
                    if (ok) {
                        after_sync();
                        for (int q = 0; q < halves; ++q) scores(q, 0);
                        tc::umma_commit(&bars.k_empty[kv_tiles & 1]);
                    }
                    for (int t = 0; ok && t < tiles; ++t) {
                        const uint32_t now = kv_tiles + t;
                        const bool last = t + 1 == tiles;
                        ok = wait(&bars.v_full[now & 1], now >> 1) && sums(0, t, 0) && sums(0, t, 1);
                        if (ok && !last) ok = wait(&bars.k_full[(now + 1) & 1], (now + 1) >> 1) && next(0, t);
                        if (ok && halves == 2) ok = sums(1, t, 0) && sums(1, t, 1) && (last || next(1, t));
                        if (ok) {
                            tc::umma_commit(&bars.v_empty[now & 1]);
                            if (!last) tc::umma_commit(&bars.k_empty[(now + 1) & 1]);
                        }
                    }
                }
                __syncwarp();
                kv_tiles += tiles;
                my_tiles += tiles;
                if (halves == 2) second_tiles += tiles;
                if (tiles > 0) ++q_items;
            }
        }
    }
    // Products under way end before tensor memory is given back, whichever role gave up (the rows wait for the last ones otherwise). The
    // thread elected is the one that issued them: for one mask it is always the same.
    if (gave_up && warp == kProductWarp && tc::elect_one()) {
        tc::umma_commit(&bars.drain);
        tc::mbar_wait(&bars.drain, 0);
    }
    __syncwarp();
    before_sync();
    __syncthreads();
    after_sync();
    if (warp == kProductWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

constexpr int kPromptRanges = kNumSMs;           // at most: a block to an SM
long long prompt_tiles(const OglePagedBatch* b) {
    const long long rows = b->max_rows < b->n_rows ? b->max_rows : b->n_rows;
    return (rows * (b->q_heads / b->kv_heads) + kItemRows - 1) / kItemRows;
}
size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

template <int DP>
int launch_form(const OglePagedBatch* b, PromptArgs p, void* workspace, cudaStream_t stream) {
    using L = Layout<DP>;
    constexpr int ranges = kPromptRanges;
    unsigned char* w = static_cast<unsigned char*>(workspace);
    p.a.parts = reinterpret_cast<float*>(w); w += up16(size_t(ranges) * 2 * L::kPart * sizeof(float));
    p.a.cuts = reinterpret_cast<Cut*>(w); w += up16(ranges * sizeof(Cut));
    Plan* plan = reinterpret_cast<Plan*>(w); w += sizeof(Plan);
    Start* starts = reinterpret_cast<Start*>(w); w += ranges * sizeof(Start);
    p.nans = reinterpret_cast<NanPiece*>(w);
    p.plan = plan; p.starts = starts;
    p.max_tiles = int(prompt_tiles(b));
    auto kernel = paged_prompt_kernel<DP>;
    static std::atomic<uint64_t> sized{0};               // devices whose limit of shared memory is raised
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && !(sized.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
        if (e == cudaSuccess) sized.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
    }
    if (e == cudaSuccess) e = launch_overlapped(paged_plan_kernel, dim3(1), dim3(1024), 0, stream, p.a, p.max_tiles, ranges, plan, starts);
    if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
    int rc = finish_launch();
    if (rc != OGLE_OK) return rc;
    e = launch_overlapped_if(overlapped_launches_enabled(true), kernel, dim3(ranges), dim3(kThreads), L::kSmem, stream, p);
    if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
    rc = finish_launch();
    if (rc != OGLE_OK) return rc;
    p.a.by_segment = 0;
    return launch_join(p.a, DP, false, ranges, ranges, kItemRows, kItemRows, stream);
}

}  // namespace

namespace paged {

size_t prompt_workspace(const OglePagedBatch* b) {
    constexpr int ranges = kPromptRanges;
    const size_t part = b->head_dim <= 64 ? Layout<64>::kPart : Layout<128>::kPart;
    return up16(size_t(ranges) * 2 * part * sizeof(float)) + up16(ranges * sizeof(Cut)) + sizeof(Plan) + ranges * sizeof(Start) +
           size_t(ranges) * kNanKeys * sizeof(NanPiece);
}

int launch_prompts(const OglePagedBatch* b, AttnArgs a, void* workspace, cudaStream_t stream) {
    PromptArgs p = {};
    p.a = a;
    return b->head_dim <= 64 ? launch_form<64>(b, p, workspace, stream) : launch_form<128>(b, p, workspace, stream);
}

}  // namespace paged
}  // namespace ogle
