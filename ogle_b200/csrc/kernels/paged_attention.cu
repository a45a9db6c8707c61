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
// Where there are few segments, none of them long, the blocks of a cluster have one segment instead and add their parts
// through each other's shared memory: one launch, no workspace.
//
// Measured: 64 sequences of up to 8000 tokens, 32 query heads to 8 of 128, 570 MB: 112 to 118 us, 74 to 78 % of what a copy reaches. 3 sequences
// of up to 200000 tokens, 16 query heads to one: 51 us, 3.9 TB/s with the join - 500 instructions a step of 16 keys, each warp
// waiting 2 of 8 cycles for the one before (four blocks an SM, the queries in shared memory; three, in registers: 56). What is short is bound
// by latency: one sequence of 700 tokens takes 9 us on the device.
//
// The products run on 16-bit operands: an e4m3 value is an fp16 exactly; queries are scaled by a power of two so that their
// largest lies below 2^12 (11 bits of each, or 22 as two parts), weights lie below 2^15. kSplit keeps queries and weights as
// two parts, the high ones in rows 0-7 of the multiply and the low ones in rows 8-15: an accumulator's two halves of a row are
// then in the same thread, and up to 8 rows cost nothing more.
#include <type_traits>

#include "paged_attention.cuh"

namespace ogle {
namespace {

using namespace paged;

constexpr int kWarps = 4;
constexpr int kTileKeys = kWarps * kChunk;
constexpr int kSegmentCost = 8;                  // tiles that a segment's beginning and end take as long as (64 sequences: 0 139 us, 2 124, 8 114)
template <int DP, int MT, bool kSplit>
struct Form {
    static constexpr int kRows = MT * (kSplit ? 8 : 16);
    static constexpr int kStages = DP == 64 ? 5 : 3;
    static constexpr int kBoxBytes = kChunk * (DP == 64 ? 64 : 128);                // of one copy
    static constexpr int kBoxes = DP == 256 ? 2 : 1;                                // to a step's keys, or values
    static constexpr int kStageBytes = 2 * kChunk * DP;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kJoin = kWarps * kRows * (DP + 4) * 4;
    static constexpr int kQueries = (kRing > kJoin ? kRing : kJoin);                // behind both: the queries as A operands, a lane's 16 bytes a step
    static constexpr int kSmem = kQueries + MT * (DP / 16) * 512 + 1024;            // the ring begins on a swizzle's boundary
    static constexpr int kPart = kRows * (DP + 2);      // floats of a part: values, then m, then sums
    static constexpr int kBlocks = DP == 64 ? (MT == 1 ? 5 : 3) : (DP == 128 ? (MT == 1 ? 4 : 2) : 2);   // that fit an SM at once
};

// ---- the ranges
__device__ __forceinline__ Sequence few_sequence(const AttnArgs& a, int b) {
    Sequence s = sequence(a.b, b);
    if (a.few_limit && (long long)s.n * a.b.group > a.few_limit) s.n = 0;
    return s;
}

struct Place { long long total, first; int b, cost; };   // sum of all; what comes before b; the sequence of the position asked for; of a segment

__device__ __forceinline__ int tiles_of(const paged::Sequence& s, int causal, int window) {
    if (s.n <= 0) return 0;
    const Span k = span_of(s, 0, s.n - 1, causal, window);
    return k.hi > k.lo ? (k.hi - 1) / kTileKeys - k.lo / kTileKeys + 1 : 0;
}
// What a segment of so many tiles counts in the ranges, its beginning and end being worth `cost` tiles.
__device__ __forceinline__ int counts(int tiles, int cost) { return tiles > 0 ? tiles + cost : 0; }

// Sums what all segments count and finds the sequence that range `num` of `den` begins in. A block of 128 threads; `shared`
// holds 10 values. A segment's beginning and end - queries, the first copies, the sum over warps - take a block as long as some
// tiles; they count as a quarter of a range at most, so that short ranges are not spent on them.
__device__ __forceinline__ Place locate(const AttnArgs& a, int rows, int num, int den, long long* shared) {
    const Batch& B = a.b;
    const int tid = threadIdx.x, per = (B.n_seqs + 127) / 128;
    const auto segments = [&](int b, int& tiles) {
        const Sequence s = few_sequence(a, b);
        tiles = tiles_of(s, a.causal, a.window);
        return tiles > 0 ? (long long)B.kv_heads * row_tiles(B, s.n, rows) : 0LL;
    };
    long long my_tiles = 0, my_segments = 0;
    for (int i = 0; i < per && tid * per + i < B.n_seqs; ++i) {
        int tiles;
        const long long n = segments(tid * per + i, tiles);
        my_tiles += n * tiles;
        my_segments += n;
    }
    long long t = my_tiles, n = my_segments;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long u = __shfl_up_sync(~0u, t, d), m = __shfl_up_sync(~0u, n, d);
        if ((tid & 31) >= d) { t += u; n += m; }
    }
    if ((tid & 31) == 31) { shared[tid / 32] = t; shared[4 + tid / 32] = n; }
    if (tid == 0) shared[9] = -1;
    __syncthreads();
    long long tiles = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < tid / 32) { t += shared[w]; n += shared[4 + w]; }
        tiles += shared[w];
        all += shared[4 + w];
    }
    Place p;
    p.cost = int(min((long long)kSegmentCost, quotient(tiles, 4LL * den)));
    p.total = tiles + all * p.cost;
    const long long at = quotient(p.total * num, den), sum = t + n * p.cost;
    long long first = sum - my_tiles - my_segments * p.cost;
    if (at >= first && at < sum) {
        for (int i = 0; i < per && tid * per + i < B.n_seqs; ++i) {
            int k;
            const long long m = segments(tid * per + i, k), c = m * (k + p.cost);
            if (at < first + c) {
                shared[8] = first;
                shared[9] = tid * per + i;
                break;
            }
            first += c;
        }
    }
    __syncthreads();
    p.first = shared[8];
    p.b = int(shared[9]);
    return p;
}

// ---- copies and products
__device__ __forceinline__ bool wait_copy(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t spin = 0; spin < limit; ++spin) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Where unit u (16 bytes) of row r of a step's keys or values lies: as the copies' swizzle puts it.
template <int DP>
__device__ __forceinline__ int unit_at(int r, int u) {
    return DP == 64 ? r * 64 + (u ^ ((r >> 1) & 3)) * 16 : (u >> 3) * (kChunk * 128) + r * 128 + ((u & 7) ^ (r & 7)) * 16;
}
// The key (of eight) that stands for column n of a product's block: eight lanes that read together get rows in different banks.
template <int DP>
__device__ __forceinline__ int key_of(int n) { return DP == 64 ? n : (n >> 1) + (n & 1) * 4; }

// A block's place in its range and the segment that it has: in shared memory, so that no thread keeps them in registers
// while it goes through keys.
struct Walk { long long at, first, end, total; int b, cost; };
struct Segment {
    paged::Sequence s;
    int b, h, m0, m_end;                          // sequence, kv head, rows of the tile
    int c0, c1, cost;                             // of what the segment counts, the range has [c0, c1)
    int j_begin, steps;                           // the range's keys in steps
    Span keys;                                    // that some row attends
    int inner_lo, inner_hi;                       // that every row attends
    const int* blocks;                            // chosen pages: of the one row, or ...
    const int2* list;                             // ... of the tile's rows
    int first_row, entries;
    unsigned all_rows;                            // bits of the tile's rows
};

// One thread: the next segment of the range; false where there is none.
template <int kRows>
__device__ __forceinline__ bool next_segment(const AttnArgs& a, Walk& w, Segment& g) {
    const Batch& B = a.b;
    for (; w.at < w.end && w.b < B.n_seqs; ++w.b) {
        g.s = few_sequence(a, w.b);
        const int tiles = tiles_of(g.s, a.causal, a.window), rts = row_tiles(B, g.s.n, kRows);
        g.cost = counts(tiles, w.cost);
        const long long all = (long long)B.kv_heads * rts * g.cost;
        if (w.at >= w.first + all) { w.first += all; continue; }
        const long long seg = quotient(w.at - w.first, g.cost), seg_first = w.first + seg * g.cost;
        g.b = w.b;
        g.h = int(quotient(seg, rts));
        const int rt = int(seg - (long long)g.h * rts);
        g.c0 = int(w.at - seg_first);
        g.c1 = int(min((long long)g.cost, w.end - seg_first));
        g.m0 = rt * kRows;
        g.m_end = min(g.s.n * B.group, g.m0 + kRows);
        const int first_row = g.m0 / B.group, last_row = (g.m_end - 1) / B.group;
        g.keys = span_of(g.s, first_row, last_row, a.causal, a.window);
        g.inner_lo = span_of(g.s, last_row, 0, a.causal, a.window).lo;
        g.inner_hi = span_of(g.s, 0, first_row, a.causal, a.window).hi;
        // its tiles come behind the segment's cost
        const int base = span_of(g.s, 0, g.s.n - 1, a.causal, a.window).lo / kTileKeys;
        const int t0 = max(g.c0 - w.cost, 0), t1 = max(g.c1 - w.cost, 0);
        g.j_begin = max((base + t0) * kTileKeys, g.keys.lo / kChunk * kChunk);
        g.steps = max(0, (min((base + t1) * kTileKeys, g.keys.hi) - g.j_begin + kChunk - 1) / kChunk);
        if (g.c0 == 0 && (a.by_segment || g.c1 < g.cost)) {
            // up to the first range that begins at or behind the segment's end
            const long long seg_end = seg_first + g.cost;
            const int last = min(int(quotient(seg_end * gridDim.x + w.total - 1, w.total)), int(gridDim.x));
            a.cuts[a.by_segment ? ((long long)g.b * B.kv_heads + g.h) * a.by_segment + rt : blockIdx.x] =
                Cut{g.c1 < g.cost ? g.m_end - g.m0 : 0, g.s.row0, g.h, g.m0, int(blockIdx.x), last, w.total < gridDim.x, 0, w.total};
        }
        w.at = seg_first + g.c1;
        return true;
    }
    return false;
}

// One thread: the cluster's segment, and this block's share of its tiles; false where there is no such tile of rows.
template <int kRows, bool kChosen>
__device__ __forceinline__ bool cluster_segment(const AttnArgs& a, Segment& g) {
    const Batch& B = a.b;
    const int c = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster, rt = c % a.by_segment;
    g.b = c / (a.by_segment * B.kv_heads);
    g.h = c / a.by_segment % B.kv_heads;
    g.s = few_sequence(a, g.b);
    const int tile_rows = kChosen ? a.tile_rows : kRows;
    g.m0 = rt * tile_rows;
    if (g.m0 >= g.s.n * B.group) return false;
    g.m_end = min(g.s.n * B.group, g.m0 + tile_rows);
    const int first_row = g.m0 / B.group, last_row = (g.m_end - 1) / B.group;
    g.keys = span_of(g.s, first_row, last_row, a.causal, a.window);
    g.inner_lo = span_of(g.s, last_row, 0, a.causal, a.window).lo;
    g.inner_hi = span_of(g.s, 0, first_row, a.causal, a.window).hi;
    int lo = g.keys.lo & ~(kChunk - 1), chunks = g.keys.hi > lo ? (g.keys.hi - lo + kChunk - 1) / kChunk : 0;
    if constexpr (kChosen) {
        // keys by their place in the list of pages
        g.first_row = first_row;
        g.all_rows = ~0u >> (31 - (last_row - first_row));
        g.list = a.lists ? a.lists + (long long)c * a.list_stride : nullptr;
        g.blocks = a.chosen + (g.s.row0 + first_row) * a.chosen_row + g.h * a.chosen_head;
        // (a row's choice may be shorter still: what is behind its end names no page)
        g.entries = a.lists ? a.list_len[c] : min(a.count, g.keys.hi > 0 ? ((g.keys.hi - 1) >> B.page_shift) + 1 : 0);
        lo = 0;
        chunks = g.entries << B.page_shift >> 4;
        static_assert(kChunk == 16, "");
    }
    const int c0 = chunks * rank / a.cluster, c1 = chunks * (rank + 1) / a.cluster;
    g.j_begin = lo + c0 * kChunk;
    g.steps = c1 - c0;
    g.c0 = g.c1 = g.cost = 0;
    return true;
}

__device__ __forceinline__ float4 remote_load4(uint32_t addr, int rank) {
    uint32_t r;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(r) : "memory");
    return v;
}
__device__ __forceinline__ float2 remote_load2(uint32_t addr, int rank) {
    uint32_t r;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(r) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Each block of the cluster has every so-many-th row and adds the blocks' parts in their order.
template <int DP>
__device__ __noinline__ void cluster_join(const AttnArgs& a, const Segment& g, const unsigned char* parts, const float2* sums, int rows) {
    const int size = a.cluster, rank = blockIdx.x % size;
#pragma unroll 1
    for (int idx = threadIdx.x; idx < rows * (DP / 4); idx += kWarps * 32) {
        const int r = idx / (DP / 4), d = idx % (DP / 4) * 4, row = g.m0 + r;
        if (row >= g.m_end || r % size != rank) continue;
        float top = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < size; ++k) {
            const float2 q = remote_load2(tc::smem_u32(sums + r), k);
            if (q.y != 0.f) top = fmaxf(top, q.x);
        }
        for (int k = 0; k < size; ++k) {
            const float2 q = remote_load2(tc::smem_u32(sums + r), k);
            if (q.y == 0.f) continue;
            const float f = exp2_fast(q.x - top);
            const float4 o = remote_load4(tc::smem_u32(parts) + (r * (DP + 4) + d) * 4, k);
            sum += q.y * f;
            v.x += o.x * f; v.y += o.y * f; v.z += o.z * f; v.w += o.w * f;
        }
        store_row(a, g.s.row0 + row / a.b.group, g.h * a.b.group + row % a.b.group, d, v, top, sum);
    }
}

// kChosen: over the pages that rows have chosen, a segment to a cluster (of one block or more). A place in the segment's list of pages
// stands for a key until it is looked up.
template <int DP, int MT, bool kSplit, bool kChosen>
__global__ void __launch_bounds__(kWarps * 32, (Form<DP, MT, kSplit>::kBlocks))
paged_attention_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using F = Form<DP, MT, kSplit>;
    constexpr int kRows = F::kRows, NR = kSplit ? 1 : 2, KS = DP / 16, NB = DP / 8;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ long long shared[10];
    __shared__ __align__(8) uint64_t bars[kWarps][F::kStages];
    __shared__ int gave_up, more_segments;
    __shared__ float row_scale[kRows];
    __shared__ __align__(8) float2 block_sum[kRows];      // cluster: m and sum of weights of a row in this block
    __shared__ Walk walk;
    __shared__ Segment segment;
    unsigned char* const smem = dynamic + ((1024 - (tc::smem_u32(dynamic) & 1023)) & 1023);
    const Batch& B = a.b;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, c4 = lane & 3, r8 = lane >> 2;
    if (tid < kWarps * F::kStages) {
        tc::mbar_init(&bars[0][0] + tid, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");       // by each thread that has initialised one
    }
    if (tid == 0) gave_up = 0;
    grid_dependency_trigger();
    grid_dependency_wait();
    if (kChosen || a.cluster) {
        if (tid == 0) more_segments = cluster_segment<kRows, kChosen>(a, segment);
        __syncthreads();
        if (!more_segments) return;
    } else {
        const Place place = locate(a, kRows, blockIdx.x, gridDim.x, shared);
        if (tid == 0) {
            if (!a.by_segment) a.cuts[blockIdx.x].rows = 0;
            walk = Walk{quotient(place.total * blockIdx.x, gridDim.x), place.first, quotient(place.total * (blockIdx.x + 1), gridDim.x), place.total, place.b, place.cost};
            more_segments = place.b >= 0 && next_segment<kRows>(a, walk, segment);
        }
        __syncthreads();
    }
    const unsigned char* const my_ring = smem + warp * F::kStages * F::kStageBytes;
    const uint32_t ring = tc::smem_u32(my_ring), bar0 = tc::smem_u32(&bars[warp][0]);
    const int nowhere = max(B.n_pages, 1);
    int put = 0, get = 0;                         // stages of the ring: the next to fill, the next to read
    uint32_t parity = 0;                          // of the next to read
    // this lane's rows of the two kinds of loads, as offsets into a step
    const uint32_t value_row = key_of<DP>(lane & 7) + ((lane >> 3) & 1) * 8;

    while (more_segments) {
        const int j_begin = segment.j_begin, h = segment.h, inner_lo = segment.inner_lo, inner_hi = segment.inner_hi;
        const int count = segment.steps > warp ? (segment.steps - warp + kWarps - 1) / kWarps : 0;   // of this warp: warp, warp + 4, ...

        // pages and scales of the warp's next 32 steps, a lane each; the 32 behind them are on their way
        int page[2] = {nowhere, nowhere};         // where there is no page: the copies find themselves outside and bring zeros
        float ks[2] = {0.f, 0.f}, vs[2] = {0.f, 0.f};
        const int in_page = (1 << B.page_shift) - 1;
        int start[2] = {0, 0};                    // chosen pages: a step's first key
        unsigned seen_by[2] = {0u, 0u};           // and the rows that have chosen its page; none where there is no page
        const auto look_up = [&](int which, int i) {
            int p = -1;
            if (i < count) {
                const int at = j_begin + (i * kWarps + warp) * kChunk;
                int block = at >> B.page_shift;
                if constexpr (kChosen) {
                    seen_by[which] = segment.all_rows;
                    if (segment.list) {
                        const int2 e = segment.list[block];
                        block = e.x;
                        seen_by[which] = unsigned(e.y);
                    } else {
                        block = __ldg(segment.blocks + block);
                    }
                    // none, or one behind the text
                    if (block < 0 || block > (segment.s.len - 1) >> B.page_shift) block = -1;
                    start[which] = block < 0 ? 0 : (block << B.page_shift) + (at & in_page);
                    if (block >= 0) p = paged::page_of(B, segment.b, block);
                    if (p < 0) seen_by[which] = 0u;
                } else {
                    p = paged::page_of(B, segment.b, block);
                }
            }
            page[which] = p >= 0 ? p : nowhere;
            ks[which] = vs[which] = 0.f;
            if (p >= 0) {
                const long long o = (long long)p * B.kv_heads + h;
                ks[which] = __ldg(B.k_scale + o);
                vs[which] = __ldg(B.v_scale + o);
            }
        };
        look_up(0, lane);
        look_up(1, 32 + lane);
        const auto issue = [&](int i, int p) {    // step i, whose page is p
            if (lane == 0) {
                const uint32_t dst = ring + put * F::kStageBytes, bar = bar0 + put * 8;
                const int token = (j_begin + (i * kWarps + warp) * kChunk) & in_page;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(F::kStageBytes) : "memory");
#pragma unroll
                for (int x = 0; x < F::kBoxes; ++x) {
                    copy_box(dst + x * F::kBoxBytes, &k_map, bar, x * 128, token, h, p);
                    copy_box(dst + kChunk * DP + x * F::kBoxBytes, &v_map, bar, x * 128, token, h, p);
                }
            }
            put = put + 1 == F::kStages ? 0 : put + 1;
        };
#pragma unroll
        for (int i = 0; i < F::kStages - 1; ++i) {
            const int p = __shfl_sync(~0u, page[0], i);
            if (i < count) issue(i, p);
        }

        // queries, once for all warps: in shared memory as the products take them (registers for them would leave room for a block less)
        uint4* const queries = reinterpret_cast<uint4*>(smem + F::kQueries) + lane;
        const float kDown = -3e38f;               // m of a row that has not met a key
        // weight w = 2^(s rs + noff) of product s; noff = kLift - m. (The product is rounded before the sum: so is m, and the largest x of a
        // row comes near kLift however large it is, where a fused sum would be off by what m was rounded by.) Sums of weights are of w; the
        // values' sums O are of w 2^(log2 scale + up), so that the row's largest w x scale, not its largest w, lies near 2^kLift: what a page's
        // scale is to other rows, or to a key that hardly counts, takes no bits from this row's weights
        float rs[MT][NR], noff[MT][NR], up[MT][NR], l[MT][NR];
        // (one copy of the code: it runs once a segment, and fetching a second took longer than running it - drafts of 5 rows 62 us, so 60)
#pragma unroll 1
        for (int i = 0; i < MT * NR; ++i) {
            const int mt = i / NR, r = i % NR;
            if (i % kWarps != warp || segment.steps == 0) continue;     // steps 0: a range that has the segment's cost alone
            // rows that are not there repeat the last
            const int tile_row = mt * (kSplit ? 8 : 16) + r * 8 + r8, row = min(segment.m0 + tile_row, segment.m_end - 1);
            const long long q0 = (segment.s.row0 + row / B.group) * a.q_row + (h * B.group + row % B.group) * a.q_head;
            float f[DP / 4], top = 0.f;
#pragma unroll
            for (int u = 0; u < DP / 64; ++u) load16(a.q, q0, 16 * (c4 + 4 * u), B.dim, B.dtype, f + 16 * u);
#pragma unroll
            for (int x = 0; x < DP / 4; ++x) top = fmaxf(top, fabsf(f[x]));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            // 2^e with |q| 2^-e below 2^12; an infinite or vanishing row stays as it is. A negative scale turns the queries' signs
            const int e = top > 1e-30f && top <= 3e38f ? int(__float_as_uint(top) >> 23) - 126 - 12 : 0;
            const float down = __uint_as_float(uint32_t(127 - e) << 23 | (a.scale_log2 < 0.f ? 0x80000000u : 0u));
            if (c4 == 0) row_scale[tile_row] = fabsf(a.scale_log2) * __uint_as_float(uint32_t(127 + e) << 23);
#pragma unroll
            for (int x = 0; x < DP / 4; ++x) f[x] *= down;
#pragma unroll
            for (int t = 0; t < KS; ++t) {        // step t: word t % 4 of unit c4 + 4 (t / 4) - the order in which keys are read
                const uint32_t u = half2_bits(f[4 * t], f[4 * t + 1]), v = half2_bits(f[4 * t + 2], f[4 * t + 3]);
                uint4* const to = queries + (mt * KS + t) * 32;
                if (kSplit) {
                    *to = make_uint4(u, rest_bits(u, f[4 * t], f[4 * t + 1]), v, rest_bits(v, f[4 * t + 2], f[4 * t + 3]));
                } else {
                    reinterpret_cast<uint32_t*>(to)[r] = u;
                    reinterpret_cast<uint32_t*>(to)[2 + r] = v;
                }
            }
        }
        __syncthreads();
        // Chosen pages: most steps are some row's edge, and hardly ever are there NaNs among the values. So a warp goes over its keys without a look for
        // them; where sums come out NaN it does so once more, with care (1000 rows: 197 us with a look at every step's bytes, 161 so).
        bool careful = !kChosen, lost = false;
    [[maybe_unused]] over:
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                noff[mt][r] = kLift - kDown;
                up[mt][r] = 0.f;
                l[mt][r] = 0.f;
                rs[mt][r] = row_scale[mt * (kSplit ? 8 : 16) + r * 8 + r8];
            }
        float O[MT][NB][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) O[mt][n][x] = 0.f;

        // chosen pages: of this lane's rows, the number in the tile and the first key that is hidden
        int row_bit[MT][NR], row_hi[MT][NR];
        if constexpr (kChosen) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const int row = min(segment.m0 + mt * (kSplit ? 8 : 16) + r * 8 + r8, segment.m_end - 1) / B.group;
                    row_bit[mt][r] = row - segment.first_row;
                    row_hi[mt][r] = span_of(segment.s, row, row, 1, 0).hi;
                }
        }

        for (int i = 0; i < count; ++i) {
            if ((i & 31) == 0 && i > 0) {
                page[0] = page[1]; ks[0] = ks[1]; vs[0] = vs[1];
                if constexpr (kChosen) { start[0] = start[1]; seen_by[0] = seen_by[1]; }
                look_up(1, i + 32 + lane);
            }
            const unsigned char* const step = my_ring + get * F::kStageBytes;
            const uint32_t at_v = ring + get * F::kStageBytes + kChunk * DP;
            const bool came = wait_copy(bar0 + get * 8, parity, a.spin_limit);
            if (!__all_sync(~0u, came)) {
                // nothing more is asked for; the copies under way are waited for, this one's among them
                for (int j = i; j < min(count, i + F::kStages - 1); ++j) {
                    wait_copy(bar0 + get * 8, parity, tc::kSpinLimit);
                    if (++get == F::kStages) { get = 0; parity ^= 1; }
                }
                if (lane == 0) {
                    gave_up = 1;
                    tc::record_error(a.error, kGaveUp);
                }
                lost = true;
                break;
            }
            if (++get == F::kStages) { get = 0; parity ^= 1; }
            const int j0 = kChosen ? __shfl_sync(~0u, start[0], i & 31) : j_begin + (i * kWarps + warp) * kChunk;
            const unsigned rows_here = kChosen ? __shfl_sync(~0u, seen_by[0], i & 31) : 0u;
            const float k_scale = __shfl_sync(~0u, ks[0], i & 31), v_scale = __shfl_sync(~0u, vs[0], i & 31);
            const bool edge = j0 < inner_lo || j0 + kChunk > inner_hi || k_scale == 0.f || kChosen && rows_here != segment.all_rows;       // 0: no page, or one of zeros
            // products of queries and keys; rows of parts are put together
            float S[2][MT][4];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int y = 0; y < 4; ++y) S[nb][mt][y] = 0.f;
#pragma unroll
            for (int u = 0; u < DP / 64; ++u) {
                uint4 w[2];
#pragma unroll
                for (int nb = 0; nb < 2; ++nb) w[nb] = *reinterpret_cast<const uint4*>(step + unit_at<DP>(nb * 8 + key_of<DP>(r8), c4 + 4 * u));
#pragma unroll
                for (int y = 0; y < 4; ++y) {     // the two blocks in turn: neither waits for its own last product
                    uint32_t q[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<uint4*>(q[mt]) = queries[(mt * KS + 4 * u + y) * 32];
#pragma unroll
                    for (int nb = 0; nb < 2; ++nb) {
                        uint32_t b0, b1;
                        paged::e4m3x4_to_half2(reinterpret_cast<const uint32_t*>(&w[nb])[y], b0, b1);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) mma(S[nb][mt], q[mt], b0, b1);
                    }
                }
            }
            if (kSplit)
#pragma unroll
                for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        S[nb][mt][0] += S[nb][mt][2];
                        S[nb][mt][1] += S[nb][mt][3];
                    }
            if (kChosen && edge) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const int end = rows_here >> row_bit[mt][r] & 1 ? row_hi[mt][r] - j0 : 0;
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                            for (int y = 0; y < 2; ++y)
                                if (nb * 8 + key_of<DP>(c4 * 2 + y) >= end) S[nb][mt][2 * r + y] = -INFINITY;
                    }
            } else if (edge) {
                const bool no_page = __shfl_sync(~0u, page[0], i & 31) == nowhere;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const int row = min(segment.m0 + mt * (kSplit ? 8 : 16) + r * 8 + r8, segment.m_end - 1) / B.group;
                        const Span k = span_of(segment.s, row, row, a.causal, a.window);
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int j = j0 + nb * 8 + key_of<DP>(c4 * 2 + y);
                                if (no_page || j < k.lo || j >= k.hi) S[nb][mt][2 * r + y] = -INFINITY;
                            }
                    }
            }
            // weights 2^(s rk + noff), and times the values' scale as A operands of the second product
            const float v_log = v_scale > 0.f ? float(int(__float_as_uint(v_scale) >> 23) - 127) : -INFINITY;     // a power of two, or no value
            float e[MT][2][2 * NR], rk[MT][NR];
            bool more = false;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    rk[mt][r] = fmaxf(rs[mt][r] * k_scale, 1e-37f);    // never 0: a hidden key's minus infinity stays one
                    const float most = kHeadroom + kLift - fmaxf(v_log + up[mt][r], 0.f);      // of w, and of w x scale
#pragma unroll
                    for (int nb = 0; nb < 2; ++nb)
                    {
                        float* const x = &e[mt][nb][2 * r];
                        unpair(add2(mul2(pair(S[nb][mt][2 * r], S[nb][mt][2 * r + 1]), pair(rk[mt][r], rk[mt][r])), pair(noff[mt][r], noff[mt][r])), x[0], x[1]);
                        more |= x[0] > most || x[1] > most;
                    }
                }
            if (__any_sync(~0u, more)) {
                // a larger unit for a row's weights or for its values: rare
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float f[NR];
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const float* s0 = &S[0][mt][2 * r];
                        const float* s1 = &S[1][mt][2 * r];
                        float top = __fmul_rn(fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s1[0], s1[1])), rk[mt][r]);
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                        const float now = fminf(noff[mt][r], kLift - top), move = now - noff[mt][r];
                        // what brings the largest w x scale to kLift: less with this step's, or as much more as m
                        const float high = fminf(up[mt][r] - move, kLift - (top + now) - v_log);
                        f[r] = exp2_fast(move + (high - up[mt][r]));
                        up[mt][r] = high;
                        noff[mt][r] = now;
                        l[mt][r] *= exp2_fast(move);
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                            for (int y = 0; y < 2; ++y) e[mt][nb][2 * r + y] = __fadd_rn(__fmul_rn(S[nb][mt][2 * r + y], rk[mt][r]), noff[mt][r]);
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int y = 0; y < 4; ++y) O[mt][n][y] *= f[(y / 2) % NR];
                }
            }
            uint32_t P[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float by = exp2_fast(fminf(v_log + up[mt][r], 126.f));    // beyond that w is 0
#pragma unroll
                    for (int nb = 0; nb < 2; ++nb) {
                        float p0 = exp2_fast(e[mt][nb][2 * r]), p1 = exp2_fast(e[mt][nb][2 * r + 1]);
                        l[mt][r] += p0 + p1;
                        p0 *= by;
                        p1 *= by;
                        const uint32_t hi = half2_bits(p0, p1);
                        if (kSplit) {
                            P[mt][2 * nb] = hi;
                            P[mt][2 * nb + 1] = rest_bits(hi, p0, p1);
                        } else {
                            P[mt][2 * nb + r] = hi;
                        }
                    }
                }
            // the step's values, two units (32 elements) at a time
            const auto values = [&](auto at_edge) {
                constexpr bool kEdge = decltype(at_edge)::value;
                uint32_t seen[MT][4];             // 1 where the row attends the key
                if (kEdge) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float* s = &S[nb][mt][2 * (r % NR)];
                                seen[mt][2 * nb + r] = r >= NR ? 0u : (s[0] == -INFINITY ? 0u : 0x3c00u) | (s[1] == -INFINITY ? 0u : 0x3c000000u);
                            }
                }
#pragma unroll
                for (int u = 0; u < DP / 32; ++u) {
                    uint32_t w[4];
                    ldmatrix_trans(w, at_v + unit_at<DP>(value_row, 2 * u + (lane >> 4)));
                    uint32_t v[4][2];
#pragma unroll
                    for (int y = 0; y < 4; ++y)   // (a key, the next) of the even element, then of the odd one
                        paged::e4m3x4_to_half2(__byte_perm(w[y], 0, 0x3120), v[y][0], v[y][1]);
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int odd = 0; odd < 2; ++odd) {
                            uint32_t b0 = v[2 * y][odd], b1 = v[2 * y + 1][odd];
                            if (kEdge) {
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
            };
            if (edge && careful) values(std::true_type());
            else values(std::false_type());
            __syncwarp();
            const int n = i + F::kStages - 1;
            const int p0 = __shfl_sync(~0u, page[0], n & 31), p1 = __shfl_sync(~0u, page[1], n & 31);
            if (n < count) issue(n, (n ^ i) >> 5 ? p1 : p0);
        }
        if constexpr (kChosen) {
            bool nan = false;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int y = 0; y < 4; ++y) nan |= O[mt][n][y] != O[mt][n][y];
            if (__any_sync(~0u, nan) && !careful && !lost) {
                careful = true;
                look_up(0, lane);
                look_up(1, 32 + lane);
#pragma unroll
                for (int i = 0; i < F::kStages - 1; ++i) {
                    const int p = __shfl_sync(~0u, page[0], i);
                    if (i < count) issue(i, p);
                }
                goto over;
            }
        }
        __syncthreads();                          // every warp is through with its ring: the parts take its place
        if (kChosen && gave_up && a.cluster <= 1) return;
        if (!kChosen && gave_up && !a.cluster) {
            // the segments that the rest of the range begins get their notes all the same: the join follows whatever stands there
            if (tid == 0 && a.by_segment)
                while (next_segment<kRows>(a, walk, segment)) {}
            return;
        }

        // the warps' parts: values [kRows][DP + 4], then m and l
        float* const mine = reinterpret_cast<float*>(smem) + warp * kRows * (DP + 4);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float sum = l[mt][r];
                sum += __shfl_xor_sync(~0u, sum, 1);
                sum += __shfl_xor_sync(~0u, sum, 2);
                const float unit = exp2_fast(-0.5f * up[mt][r]);        // applied twice: its square can be below the smallest fp32 number
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
                    v.x = v.x * unit * unit; v.y = v.y * unit * unit; v.z = v.z * unit * unit; v.w = v.w * unit * unit;
                    *reinterpret_cast<float4*>(row + u * 16 + c4 * 4) = v;
                }
                if (c4 == 0) { row[DP] = kLift - noff[mt][r]; row[DP + 1] = sum; }
            }
        __syncthreads();
        const bool whole = segment.c0 == 0 && segment.c1 == segment.cost;
        float* const part = a.parts + ((long long)blockIdx.x * 2 + (segment.c0 > 0 ? 0 : 1)) * F::kPart;
        for (int idx = tid; idx < kRows * (DP / 4); idx += kWarps * 32) {
            const int r = idx / (DP / 4), d = idx % (DP / 4) * 4, row = segment.m0 + r;
            if (row >= segment.m_end) continue;
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
            if (a.cluster > 1) {                  // where the first warp's were: no other thread reads them
                *reinterpret_cast<float4*>(smem + (r * (DP + 4) + d) * 4) = v;
                if (d == 0) block_sum[r] = make_float2(top, sum);
                continue;
            }
            if (!whole) {
                *reinterpret_cast<float4*>(part + r * DP + d) = v;
                if (d == 0) { part[kRows * DP + r] = top; part[kRows * DP + kRows + r] = sum; }
                continue;
            }
            store_row(a, segment.s.row0 + row / B.group, segment.h * B.group + row % B.group, d, v, top, sum);
        }
        if (a.cluster > 1) {
            cluster_meet();
            if (!gave_up) cluster_join<DP>(a, segment, smem, block_sum, kRows);
            cluster_meet();                       // nobody reads this block's part any more
            return;
        }
        if (kChosen) return;
        // the next segment's copies take the parts' place
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (tid == 0) more_segments = next_segment<kRows>(a, walk, segment);
        __syncthreads();
    }
}

// Adds up the parts of segments that were cut, in the order of their ranges, and answers for sequences without a key. Block
// (c, y) has segment c, or the one that begins in range c and goes on in the next; of its rows y, y + gridDim.y, ... a warp has one.
constexpr int kJoinWarps = 8;
template <int DP>
__global__ void __launch_bounds__(kJoinWarps * 32, 6) paged_join_kernel(AttnArgs a, int ranges, int rows_of_tile) {
    constexpr int kVecs = DP / 4, kPerLane = (kVecs + 31) / 32;
    const Batch& B = a.b;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, c = blockIdx.x;
    grid_dependency_trigger();
    grid_dependency_wait();
    Cut cut = a.cuts[c];
    if (a.by_segment) {
        // what nobody has written of: tiles of rows that the sequence does not have, sequences without a key
        const Sequence s = few_sequence(a, c / (B.kv_heads * a.by_segment));
        if (c % a.by_segment >= row_tiles(B, s.n, rows_of_tile) || tiles_of(s, a.causal, a.window) == 0) cut.rows = 0;
    }
    if (blockIdx.y == 0) {
        for (int b = blockIdx.x; b < B.n_seqs; b += gridDim.x) {
            const paged::Sequence s = paged::sequence(B, b);
            if (s.n <= 0 || tiles_of(s, a.causal, a.window) > 0) continue;
            for (int idx = tid; idx < s.n * B.q_heads; idx += blockDim.x)
                for (int d = 0; d < B.dim; d += 4)
                    store_row(a, s.row0 + idx / B.q_heads, idx % B.q_heads, d, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
        }
    }
    const int part_floats = rows_of_tile * (DP + 2);
    const auto part = [&](int k) { return a.parts + ((long long)k * 2 + (k == cut.first ? 1 : 0)) * part_floats; };
    const auto none = [&](int k) { return cut.gaps && quotient(cut.total * k, ranges) == quotient(cut.total * (k + 1), ranges); };
    for (int r = blockIdx.y * kJoinWarps + warp; r < cut.rows; r += gridDim.y * kJoinWarps) {
        float top = -INFINITY, sum = 0.f;
        float4 v[kPerLane];
#pragma unroll
        for (int u = 0; u < kPerLane; ++u) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = cut.first + lane; k < cut.last; k += 32)
            if (!none(k)) {
                const float* p = part(k) + rows_of_tile * DP + r;
                if (p[rows_of_tile] != 0.f) top = fmaxf(top, p[0]);
            }
#pragma unroll
        for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
#pragma unroll 2
        for (int k = cut.first; k < cut.last; ++k) {
            if (none(k)) continue;
            const float* p = part(k);
            const float m = p[rows_of_tile * DP + r], l = p[rows_of_tile * DP + rows_of_tile + r];
            const float f = l == 0.f ? 0.f : exp2_fast(m - top);    // a part without a weight has zeros
            sum += l * f;
#pragma unroll
            for (int u = 0; u < kPerLane; ++u)
                if (u * 32 + lane < kVecs) {
                    const float4 o = *reinterpret_cast<const float4*>(p + r * DP + (u * 32 + lane) * 4);
                    v[u].x += o.x * f; v[u].y += o.y * f; v[u].z += o.z * f; v[u].w += o.w * f;
                }
        }
        const int row = cut.m0 + r;
#pragma unroll
        for (int u = 0; u < kPerLane; ++u)
            if (u * 32 + lane < kVecs)
                store_row(a, cut.row0 + row / B.group, cut.h * B.group + row % B.group, (u * 32 + lane) * 4, v[u], top, sum);
    }
}

// The same for segments of many parts: a block has one row, looks at all its parts' maxima and sums at once, and its warps take
// every sixteenth part each.
constexpr int kManyWarps = 16, kMostRanges = 8 * kNumSMs;
template <int DP>
__global__ void __launch_bounds__(kManyWarps * 32) paged_join_many_kernel(AttnArgs a, int ranges, int rows_of_tile) {
    constexpr int kVecs = DP / 4, kPerLane = (kVecs + 31) / 32;
    __shared__ float factor[kMostRanges];
    __shared__ float4 sums[kManyWarps][kVecs];
    __shared__ float tops[kManyWarps], weights[kManyWarps];
    const Batch& B = a.b;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, c = blockIdx.x, r = blockIdx.y;
    grid_dependency_trigger();
    grid_dependency_wait();
    // what nobody has written of: tiles of rows that the sequence does not have, sequences without a key
    const Cut cut = a.cuts[c];
    const Sequence s = few_sequence(a, c / (B.kv_heads * a.by_segment));
    const int tiles = tiles_of(s, a.causal, a.window);
    if (r == 0 && s.n > 0 && tiles == 0 && c % (B.kv_heads * a.by_segment) == 0)
        for (int idx = tid; idx < s.n * B.q_heads; idx += blockDim.x)
            for (int d = 0; d < B.dim; d += 4)
                store_row(a, s.row0 + idx / B.q_heads, idx % B.q_heads, d, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
    if (c % a.by_segment >= row_tiles(B, s.n, rows_of_tile) || tiles == 0 || r >= cut.rows) return;
    const int part_floats = rows_of_tile * (DP + 2), n = cut.last - cut.first;
    const auto part = [&](int k) { return a.parts + ((long long)(cut.first + k) * 2 + (k == 0 ? 1 : 0)) * part_floats; };
    const auto none = [&](int k) { return cut.gaps && quotient(cut.total * (cut.first + k), ranges) == quotient(cut.total * (cut.first + k + 1), ranges); };
    constexpr int kMine = (kMostRanges + kManyWarps * 32 - 1) / (kManyWarps * 32);
    float m[kMine], l[kMine], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int k = tid + i * kManyWarps * 32;
        m[i] = l[i] = 0.f;
        if (k < n && !none(k)) {
            const float* p = part(k) + rows_of_tile * DP + r;
            m[i] = p[0];
            l[i] = p[rows_of_tile];
            if (l[i] != 0.f) top = fmaxf(top, m[i]);
        }
    }
#pragma unroll
    for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kManyWarps; ++w) top = fmaxf(top, tops[w]);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int k = tid + i * kManyWarps * 32;
        const float f = l[i] == 0.f ? 0.f : exp2_fast(m[i] - top);       // a part without a weight has zeros, a range without a tile no part
        if (k < n) factor[k] = l[i] == 0.f ? -1.f : f;
        sum += l[i] * f;
    }
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0) weights[warp] = sum;
    __syncthreads();
    float4 v[kPerLane];
#pragma unroll
    for (int u = 0; u < kPerLane; ++u) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = warp; k < n; k += kManyWarps) {
        const float f = factor[k];
        if (f == -1.f) continue;
        const float* p = part(k) + r * DP;
#pragma unroll
        for (int u = 0; u < kPerLane; ++u)
            if (u * 32 + lane < kVecs) {
                const float4 o = *reinterpret_cast<const float4*>(p + (u * 32 + lane) * 4);
                v[u].x += o.x * f; v[u].y += o.y * f; v[u].z += o.z * f; v[u].w += o.w * f;
            }
    }
#pragma unroll
    for (int u = 0; u < kPerLane; ++u)
        if (u * 32 + lane < kVecs) sums[warp][u * 32 + lane] = v[u];
    __syncthreads();
    if (tid >= kVecs) return;
    sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kManyWarps; ++w) {
        const float4 q = sums[w][tid];
        sum += weights[w];
        o.x += q.x; o.y += q.y; o.z += q.z; o.w += q.w;
    }
    const int row = cut.m0 + r;
    store_row(a, cut.row0 + row / B.group, cut.h * B.group + row % B.group, tid * 4, o, top, sum);
}

// The pages that some row of a tile has chosen, in order, with the rows that have: a warp to a segment. The rows' choices become bits, 1024
// pages at a time, a lane's word of them 32 pages. (A lane to a row, the least of their next pages in turn: 1000 rows of 24 pages 13 us, 4 so.)
constexpr int kMergeWarps = 4, kTileRows = 33;   // rows that a tile can have a part of, at most
__global__ void __launch_bounds__(kMergeWarps * 32) merge_choices_kernel(AttnArgs a, int tile_rows, int segments) {
    __shared__ unsigned bits[kMergeWarps][kTileRows][32];
    const Batch& B = a.b;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, c = blockIdx.x * kMergeWarps + warp;
    grid_dependency_trigger();
    grid_dependency_wait();
    if (c >= segments) return;
    const int b = c / (a.by_segment * B.kv_heads), h = c / a.by_segment % B.kv_heads, m0 = c % a.by_segment * tile_rows;
    const Sequence s = sequence(B, b);
    const int m_end = min(s.n * B.group, m0 + tile_rows), first_row = m0 / B.group, rows = m0 < m_end ? (m_end - 1) / B.group - first_row + 1 : 0;
    const int* const mine = a.chosen + (s.row0 + first_row) * a.chosen_row + h * a.chosen_head;
    const int pages = s.len > 0 ? ((s.len - 1) >> B.page_shift) + 1 : 0, entries = rows * a.count;
    int2* const list = a.lists + (long long)c * a.list_stride;
    int n = 0;
    for (int p0 = 0; p0 < pages; p0 += 1024) {
        for (int r = 0; r < rows; ++r) bits[warp][r][lane] = 0;
        __syncwarp();
        bool some = false;
        for (int i = lane; i < entries; i += 32) {
            const int r = i / a.count, block = __ldg(mine + r * a.chosen_row + (i - r * a.count)), at = block - p0;
            if (at >= 0 && at < 1024 && block < pages) {
                atomicOr(&bits[warp][r][at / 32], 1u << (at & 31));
                some = true;
            }
        }
        __syncwarp();
        if (!__any_sync(~0u, some)) continue;
        unsigned all = 0;
        for (int r = 0; r < rows; ++r) all |= bits[warp][r][lane];
        int sum = __popc(all);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int o = __shfl_up_sync(~0u, sum, d);
            if (lane >= d) sum += o;
        }
        int at = n + sum - __popc(all);
        while (all) {
            const int k = __ffs(all) - 1;
            all &= all - 1;
            unsigned who = 0;
            for (int r = 0; r < rows; ++r) who |= (bits[warp][r][lane] >> k & 1) << (r & 31);
            list[at++] = make_int2(p0 + lane * 32 + k, int(who));
        }
        n += __shfl_sync(~0u, sum, 31);
        __syncwarp();
    }
    if (lane == 0) a.list_len[c] = n;
}

// ---- host
struct Choice { int dp, mt; bool split; };

int few_limit(const OglePagedBatch* b);

Choice choose(const OglePagedBatch* b) {
    Choice c;
    long long rows = (long long)(b->max_rows < b->n_rows ? b->max_rows : b->n_rows) * (b->q_heads / b->kv_heads);
    const int limit = few_limit(b);
    if (limit && rows > limit) rows = limit;
    c.dp = b->head_dim <= 64 ? 64 : (b->head_dim <= 128 ? 128 : 256);
    c.split = b->dtype == OGLE_F32 || rows <= 8;
    c.mt = c.dp == 256 || rows <= (c.split ? 8 : 16) ? 1 : 2;
    return c;
}

// Over chosen pages: 32 rows of a tile only where a sequence has no more than that. A tile goes over what any of its rows has chosen, so
// that a larger one saves fewer reads of a page than it adds pages that few of its rows want (1000 rows, 24 pages each of which neighbours
// share half: 177 us with tiles of 32, 161 with tiles of 16).
Choice choose_sparse(const OglePagedBatch* b) {
    Choice c = choose(b);
    const long long rows = (long long)(b->max_rows < b->n_rows ? b->max_rows : b->n_rows) * (b->q_heads / b->kv_heads);
    if (rows > (c.split ? 16 : 32)) c.mt = 1;
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

// Tiles of rows that a sequence can have in this form, and segments of the whole call.
long long row_tiles_of(const OglePagedBatch* b, int rows) {
    long long most = (long long)(b->max_rows < b->n_rows ? b->max_rows : b->n_rows) * (b->q_heads / b->kv_heads);
    const int limit = few_limit(b);
    if (limit && most > limit) most = limit;
    return (most + rows - 1) / rows;
}
long long row_tiles_of_all(const OglePagedBatch* b, int rows) {
    const long long most = (long long)(b->max_rows < b->n_rows ? b->max_rows : b->n_rows) * (b->q_heads / b->kv_heads);
    return (most + rows - 1) / rows;
}
constexpr int kMostCluster = 16;                  // over chosen pages; 8 are what any GPU can have
// Raises the kernel's limits of shared memory and of a cluster's blocks, once for each device.
template <int DP, int MT, bool kSplit, bool kChosen = false>
cudaError_t prepare() {
    static std::atomic<uint64_t> sized{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && !(sized.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
        e = cudaFuncSetAttribute(paged_attention_kernel<DP, MT, kSplit, kChosen>, cudaFuncAttributeMaxDynamicSharedMemorySize, Form<DP, MT, kSplit>::kSmem);
        if (kChosen && e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<DP, MT, kSplit, kChosen>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) sized.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
    }
    return e;
}

// Clusters of so many blocks that the GPU runs at once. Asked once for all devices: two of them may differ by a few, which costs time at most.
template <int DP, int MT, bool kSplit, bool kChosen = false>
int most_clusters(int size) {
    static std::atomic<int> known[kMostCluster + 1] = {};      // one more than the number
    int n = known[size].load(std::memory_order_relaxed);
    if (n == 0) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(size);
        cfg.blockDim = dim3(kWarps * 32);
        cfg.dynamicSmemBytes = Form<DP, MT, kSplit>::kSmem;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (prepare<DP, MT, kSplit, kChosen>() != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, paged_attention_kernel<DP, MT, kSplit, kChosen>, &cfg) != cudaSuccess) {
            (void)cudaGetLastError();
            return 0;
        }
        known[size].store(++n, std::memory_order_relaxed);
    }
    return n - 1;
}

// Blocks of a cluster that has one segment, or 0: ranges. A call over clusters saves the second launch and the search for ranges, about
// 3 us, but takes as long as the longest sequence's share, and blocks that the clusters do not use stay idle. us over ranges / clusters,
// one query row each, 32 query heads to 8 of 128 elements: one sequence of 700 tokens 10.8 / 9.4, of 4000 13.6 / 13.6, of 8000 15.1 /
// 19.8; 4 of 2000 14.7 / 11.7, of 8000 23.1 / 22.7, of 16000 33.4 / 38.9; 16 of up to 4000 35.7 / 23.9, of up to 8000 35.4 / 38.2.
// So the tiles of 64 keys that pay a block go from 6, where few blocks of the GPU are used, to about 30, where all are.
// A cluster has to fit into a part of the GPU with all its blocks, so the sizes are those of which the runtime says that all run at once:
// of 96 clusters of 3 with 256 elements, two blocks an SM, 93 do (288 of 296 slots): 24 drafts of 5 over 4096 tokens each 83 us, 58 in ranges,
// and over 1000 40, 29 in clusters of 2. Where lengths differ the last three come as the shortest end - up to 20000 tokens in a window of
// 4096 59 us, 61 in ranges; one row each over up to 2000 26, 29 in clusters of 2 -, but lengths are the device's.
template <int DP, int MT, bool kSplit>
int cluster_of(const OglePagedBatch* b, const OgleAttentionParams* p) {
    using F = Form<DP, MT, kSplit>;
    constexpr long long slots = kNumSMs * F::kBlocks;
    const long long segments = row_tiles_of(b, F::kRows) * b->n_seqs * b->kv_heads;
    if (segments < 1 || segments * 2 > slots) return 0;
    int size = slots / segments < 8 ? int(slots / segments) : 8;
    while (size > 1 && most_clusters<DP, MT, kSplit>(size) < segments) --size;
    if (size < 2) return 0;
    long long keys = b->max_kv_len;
    if (p->window > 0 && keys > (long long)p->window + b->max_rows) keys = (long long)p->window + b->max_rows;
    return keys <= kTileKeys * size * (6 + 25 * segments * size / slots) ? size : 0;
}

// Ranges: as many blocks as fit the GPU at once, and no more than there can be tiles.
int ranges_of(const OglePagedBatch* b, int rows, int blocks) {
    const long long max_rows = b->max_rows < b->n_rows ? b->max_rows : b->n_rows;
    const long long tiles = (b->max_kv_len + kTileKeys - 1) / kTileKeys + 1;
    const long long most = (max_rows * (b->q_heads / b->kv_heads) + rows - 1) / rows * b->n_seqs;
    const double all = double(b->kv_heads) * double(most) * double(tiles);
    return all < double(kNumSMs * blocks) ? (all < 1 ? 1 : int(all)) : kNumSMs * blocks;
}

// Rows x query heads of a group above which a sequence is the prompt form's, or 0: every sequence is taken here. The prompt form reads a
// key once for 256 rows, where this one reads it for 16 or 32, but has three launches and the tensor cores' latencies to begin and end
// with. us here / there, 32 query heads to 8 of 128 elements: 64 and 80 rows of 8 sequences over 20000 tokens 174 / 187 and 249 / 188,
// over 3000 46 / 56 and 58 / 57; 128 rows of 32 sequences over 300 70 / 63; of one sequence, 128 rows over 20000 58 / 56, 256 over 3000
// 32 / 42, over 300 21 / 31. So 64 rows, and more where the call has few keys to go through.
// fp32 and heads above 128 stay here whatever their rows are, far from what the tensor cores could do: six prompts of about 2000 rows over about
// 2500 tokens, 32 query heads to 8, take 1896 us in fp32 (94 TFLOP/s; heads of 64 1103), 2336 in bf16 with heads of 256. The prompt form holds one
// fp16 part of queries and weights, and sums of two tiles of 256 columns would fill the tensor memory that the scores need.
int few_limit(const OglePagedBatch* b) {
    if (b->dtype == OGLE_F32 || b->head_dim > 128) return 0;
    const long long rows = (long long)(b->max_rows < b->n_rows ? b->max_rows : b->n_rows) * (b->q_heads / b->kv_heads);
    const double keys = double(b->n_seqs) * b->kv_heads * b->max_kv_len * (b->head_dim <= 64 ? 0.5 : 1.0);
    const int limit = 64 + int(5e6 / (keys > 5e3 ? keys : 5e3));
    return rows > limit ? limit : 0;
}
// Whether to launch the form for few rows, too: not where n_rows is max_rows of every sequence.
bool some_few(const OglePagedBatch* b) { return !few_limit(b) || (long long)b->n_seqs * b->max_rows != b->n_rows; }

size_t few_workspace(const OglePagedBatch* b, const OgleAttentionParams* p) {
    if (!some_few(b)) return 0;
    return with_form(choose(b), [&](auto dp, auto mt, auto split) {
        using F = Form<decltype(dp)::value, decltype(mt)::value, decltype(split)::value>;
        // with clusters it is not touched, but a caller without a workspace finds out at every size
        static_assert(sizeof(Cut) <= OGLE_ATTENTION_NO_WORKSPACE && 2 * F::kPart * sizeof(float) > OGLE_ATTENTION_NO_WORKSPACE, "");
        if (cluster_of<decltype(dp)::value, decltype(mt)::value, decltype(split)::value>(b, p)) return sizeof(Cut);
        return size_t(ranges_of(b, F::kRows, F::kBlocks)) * (2 * F::kPart * sizeof(float) + sizeof(Cut));
    });
}

// Attention over chosen pages: rows of a tile, segments, blocks to a segment, and what is kept of the tiles' lists where several rows share a
// tile.
struct ChosenShape { long long segments; int tile_rows, tiles, in_tile, cluster, list_stride; size_t lists; };      // in_tile: rows that one can have a part of
constexpr int kListsCost = 7;                    // tiles that the lists' launch takes as long as (a tile 0.7 us)
// What is longest is the number of rounds of blocks, each as long as its share of the segment's tiles of 64 keys and what a segment's
// beginning, end and join are worth. r rows are taken to choose r^0.45 times the pages of one (neighbours that share half: 4 rows 46 pages
// of 24 each, 8 rows 60), so that few rows with many pages are spread over more blocks than one tile of them could use.
// A cluster lies in one part of the chip, so that large ones leave places over; the runtime says how many run at once: of 592 places clusters
// of 3 have 561, of 7 546. (80 segments of 33 pages: in clusters of 7, which do not all fit, 26 to 30 us, of 6 16 to 23; 40 of 9
// pages and 296 places: 20 and 11. Clusters of 16, 8: 4 segments of 79 pages of 128 17 and 24 us, 8 of 64 pages of 64 13 and 14.5.)
template <typename MostClusters>
ChosenShape chosen_shape(const OglePagedBatch* b, int most_rows, int slots, int count, MostClusters most_clusters) {
    const int group = b->q_heads / b->kv_heads, rows = b->max_rows < b->n_rows ? b->max_rows : b->n_rows;
    const long long pages = ((long long)b->max_kv_len + b->page_tokens - 1) / b->page_tokens;
    ChosenShape best = {};
    double least = 0;
    double union_of = 1;                          // r^0.45 for r = 1, 2, 4, ...
    for (int r = 1; ; r *= 2, union_of *= 1.366) {
        if (r > 1 && (r * group > most_rows || r / 2 >= rows)) break;
        const int tile_rows = r * group < most_rows ? r * group : most_rows;
        ChosenShape c = {};
        c.tile_rows = tile_rows;
        c.tiles = int(row_tiles_of_all(b, tile_rows));
        c.segments = (long long)c.tiles * b->n_seqs * b->kv_heads;
        c.in_tile = rows <= 1 ? 1 : tile_rows % group == 0 ? tile_rows / group : (tile_rows + group - 2) / group + 1;
        const double wanted = count * union_of < double(pages) ? count * union_of : double(pages), tiles = wanted * b->page_tokens / kTileKeys;
        for (int size = 1; size <= kMostCluster; size += size < 8 ? 1 : 8) {
            long long fit = size == 1 ? slots : (long long)most_clusters(size) * size;
            if (fit == 0 && size > 8) break;
            if (fit == 0) fit = slots;            // (nothing to ask)
            const double rounds = double((c.segments * size + fit - 1) / fit);
            const double cost = rounds * (tiles / size + kSegmentCost + (size > 8 ? 4 : size > 1 ? 2 : 0)) + (c.in_tile > 1 ? kListsCost : 0);
            if (least == 0 || cost < least) {
                best = c;
                best.cluster = size;
                least = cost;
            }
        }
    }
    best.list_stride = (best.in_tile < rows ? best.in_tile : rows) * count;
    // (one row to every tile, none cut: its choice is the list)
    best.lists = best.in_tile > 1 ? size_t(best.segments) * (best.list_stride * sizeof(int2) + sizeof(int)) : 0;
    return best;
}

}  // namespace

namespace paged {

// Map of the cache's bytes whose boxes are 16 tokens of one page and head, swizzled as unit_at says. Elements behind the head's
// end and pages behind the last read zero.
bool cache_map(CUtensorMap* m, const Batch& b, const void* cache, int dp) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)b.dim, (cuuint64_t)1 << b.page_shift, (cuuint64_t)b.kv_heads, (cuuint64_t)(b.n_pages > 0 ? b.n_pages : 1)};
    const cuuint64_t strides[3] = {(cuuint64_t)b.token_stride, (cuuint64_t)b.head_stride, (cuuint64_t)b.page_stride};
    const cuuint32_t box[4] = {dp == 64 ? 64u : 128u, kChunk, 1, 1}, es[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(cache), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              dp == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_join(const AttnArgs& a, int dp, bool many, int entries, int ranges, int tile_rows, int rows, cudaStream_t stream) {
    const auto run = [&](auto kernel, int y, int warps) {
        const cudaError_t e = launch_overlapped_if(overlapped_launches_enabled(true), kernel, dim3(unsigned(entries), unsigned(y)),
                                                   dim3(warps * 32), 0, stream, a, ranges, tile_rows);
        if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return int(OGLE_ERR_CUDA); }
        return finish_launch();
    };
    if (many) {
        const auto kernel = dp == 64 ? paged_join_many_kernel<64> : (dp == 128 ? paged_join_many_kernel<128> : paged_join_many_kernel<256>);
        return run(kernel, rows, kManyWarps);
    }
    return run(dp == 64 ? paged_join_kernel<64> : (dp == 128 ? paged_join_kernel<128> : paged_join_kernel<256>), div_up(rows, kJoinWarps), kJoinWarps);
}

}  // namespace paged
}  // namespace ogle

using namespace ogle;

extern "C" {

size_t ogle_cuda_paged_attention_workspace_bytes(const OglePagedBatch* batch, const OgleAttentionParams* p) {
    Batch b;
    if (!p || paged::translate(batch, b) != OGLE_OK || b.n_seqs == 0) return 0;
    // the forms run one after the other: what one has left there the other may overwrite
    const size_t few = few_workspace(batch, p), prompts = few_limit(batch) ? prompt_workspace(batch) : 0;
    return few > prompts ? few : prompts;
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
    if (a.b.max_rows == 0) return OGLE_OK;       // no row of any sequence counts: there would be no segment to launch for
    a.q = p->q; a.out = p->out; a.lse = p->lse;
    a.q_row = p->q_row; a.q_head = p->q_head; a.out_row = p->out_row; a.out_head = p->out_head;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.causal = p->causal; a.window = p->window;
    a.parts = static_cast<float*>(workspace);
    a.spin_limit = tc::role_wait_limit();
    a.error = error_flag_ptr();
    if (!a.error) return OGLE_ERR_CUDA;
    const int limit = few_limit(batch);
    if (limit) {
        // where the host sees no sequence of few rows, the prompt form takes those that the device has all the same: row_start may hold fewer
        // rows than n_rows
        const bool few = some_few(batch);
        a.few_limit = few ? limit : 0;
        rc = launch_prompts(batch, a, workspace, stream);
        if (rc != OGLE_OK || !few) return rc;
    }
    return with_form(choose(batch), [&](auto dp, auto mt, auto split) -> int {
        constexpr int DP = decltype(dp)::value, MT = decltype(mt)::value;
        constexpr bool kSplit = decltype(split)::value;
        using F = Form<DP, MT, kSplit>;
        const int ranges = ranges_of(batch, F::kRows, F::kBlocks);
        auto kernel = paged_attention_kernel<DP, MT, kSplit, false>;
        const long long max_tiles = row_tiles_of(batch, F::kRows), segments = max_tiles * a.b.n_seqs * a.b.kv_heads;
        a.cluster = cluster_of<DP, MT, kSplit>(batch, p);
        a.by_segment = a.cluster || segments < ranges ? int(max_tiles) : 0;
        a.cuts = reinterpret_cast<Cut*>(a.parts + size_t(ranges) * 2 * F::kPart);
        cudaError_t e = prepare<DP, MT, kSplit>();
        CUtensorMap k_map, v_map;
        if (e == cudaSuccess && (!cache_map(&k_map, a.b, a.b.k_cache, DP) || !cache_map(&v_map, a.b, a.b.v_cache, DP))) {
            set_last_error("paged_attention: no tensor map of the cache");
            return OGLE_ERR_CUDA;
        }
        if (e == cudaSuccess) {
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            // behind the prompt form's launches it is this call's own affair
            attr[0].val.programmaticStreamSerializationAllowed = overlapped_launches_enabled(a.few_limit > 0) ? 1 : 0;
            attr[1].id = cudaLaunchAttributeClusterDimension;
            attr[1].val.clusterDim.x = a.cluster ? a.cluster : 1;
            attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(a.cluster ? unsigned(segments * a.cluster) : ranges);
            cfg.blockDim = dim3(kWarps * 32);
            cfg.dynamicSmemBytes = F::kSmem;
            cfg.stream = stream;
            cfg.attrs = attr;
            cfg.numAttrs = a.cluster ? 2 : 1;
            e = cudaLaunchKernelEx(&cfg, kernel, a, k_map, v_map);
        }
        if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
        int rc = finish_launch();
        if (rc != OGLE_OK || a.cluster) return rc;
        // a warp to a row, or sixteen where few segments are cut into many parts
        const long long rows = (long long)(a.b.max_rows < a.b.n_rows ? a.b.max_rows : a.b.n_rows) * a.b.group;
        const int tile = int(rows < F::kRows ? (rows < 1 ? 1 : rows) : F::kRows);
        // us by warps / by sixteen a row: one segment of 100000 keys 273 / 28, 32 of 60000 78 / 66, 72 of 60000 107 / 100, 96 of
        // 40000 99 / 94, 144 of 30000 105 / 104, 288 of 16000 99 / 102; of 16 rows each, 40 of 60000 81 / 72, 80 of 30000 73 / 73
        const bool many = ranges > 8 * segments;
        return launch_join(a, DP, many, a.by_segment ? int(segments < 1 ? 1 : segments) : ranges, ranges, F::kRows, tile, stream);
    });
}

size_t ogle_cuda_sparse_attention_workspace_bytes(const OglePagedBatch* batch, const OgleAttentionParams* p, const OgleChosenPages* c) {
    Batch b;
    if (!p || !c || c->count < 1 || paged::translate(batch, b) != OGLE_OK || b.n_seqs == 0 || b.max_rows == 0) return 0;
    return with_form(choose_sparse(batch), [&](auto dp, auto mt, auto split) {
        constexpr int DP = decltype(dp)::value, MT = decltype(mt)::value;
        using F = Form<DP, MT, decltype(split)::value>;
        return chosen_shape(batch, F::kRows, kNumSMs * F::kBlocks, c->count, most_clusters<DP, MT, decltype(split)::value, true>).lists;
    });
}

int ogle_cuda_sparse_attention(const OglePagedBatch* batch, const OgleAttentionParams* p, const OgleChosenPages* c, void* workspace,
                               size_t workspace_bytes, ogle_stream_t stream) {
    AttnArgs a = {};
    int rc = paged::translate(batch, a.b);
    if (rc != OGLE_OK) return rc;
    if (!p || !c || p->causal != 1 || p->window != 0 || c->count < 1) return OGLE_ERR_INVALID;
    if (a.b.n_seqs == 0) return OGLE_OK;
    if (!p->q || !p->out || !c->chosen || c->chosen_row < c->count || c->chosen_head < c->count) return OGLE_ERR_INVALID;
    if (!paged::strides_ok(p->q, p->q_row, p->q_head, batch->dtype) || !paged::strides_ok(p->out, p->out_row, p->out_head, batch->dtype) || !aligned16(workspace))
        return OGLE_ERR_ALIGNMENT;
    // a tile's keys are counted in 32 bits
    if ((long long)c->count * batch->page_tokens * 33 >= (1LL << 31)) return OGLE_ERR_UNSUPPORTED;
    if (a.b.max_rows == 0) return OGLE_OK;
    const size_t needed = ogle_cuda_sparse_attention_workspace_bytes(batch, p, c);
    if (needed > 0 && (!workspace || workspace_bytes < needed)) return OGLE_ERR_INVALID;
    a.q = p->q; a.out = p->out; a.lse = p->lse;
    a.q_row = p->q_row; a.q_head = p->q_head; a.out_row = p->out_row; a.out_head = p->out_head;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.causal = 1;
    a.spin_limit = tc::role_wait_limit();
    a.error = error_flag_ptr();
    if (!a.error) return OGLE_ERR_CUDA;
    a.chosen = c->chosen; a.chosen_row = c->chosen_row; a.chosen_head = c->chosen_head; a.count = c->count;
    return with_form(choose_sparse(batch), [&](auto dp, auto mt, auto split) -> int {
        constexpr int DP = decltype(dp)::value, MT = decltype(mt)::value;
        constexpr bool kSplit = decltype(split)::value;
        using F = Form<DP, MT, kSplit>;
        const ChosenShape shape = chosen_shape(batch, F::kRows, kNumSMs * F::kBlocks, c->count, most_clusters<DP, MT, kSplit, true>);
        a.tile_rows = shape.tile_rows;
        a.by_segment = shape.tiles;
        a.cluster = shape.cluster;
        if (shape.segments * a.cluster >= (1LL << 31)) return OGLE_ERR_UNSUPPORTED;
        cudaError_t e = prepare<DP, MT, kSplit, true>();
        CUtensorMap k_map, v_map;
        if (e == cudaSuccess && (!cache_map(&k_map, a.b, a.b.k_cache, DP) || !cache_map(&v_map, a.b, a.b.v_cache, DP))) {
            set_last_error("sparse_attention: no tensor map of the cache");
            return OGLE_ERR_CUDA;
        }
        if (e == cudaSuccess && shape.lists) {
            a.list_stride = shape.list_stride;
            a.lists = static_cast<int2*>(workspace);
            a.list_len = reinterpret_cast<int*>(a.lists + size_t(shape.segments) * shape.list_stride);
            e = launch_overlapped(merge_choices_kernel, dim3(unsigned((shape.segments + kMergeWarps - 1) / kMergeWarps)), dim3(kMergeWarps * 32), 0, stream, a,
                                  shape.tile_rows, int(shape.segments));
            if (e == cudaSuccess) {
                const int done = finish_launch();
                if (done != OGLE_OK) return done;
            }
        }
        if (e == cudaSuccess) {
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            // behind the lists' launch it is this call's own affair
            attr[0].val.programmaticStreamSerializationAllowed = overlapped_launches_enabled(shape.lists > 0) ? 1 : 0;
            attr[1].id = cudaLaunchAttributeClusterDimension;
            attr[1].val.clusterDim.x = a.cluster;
            attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(unsigned(shape.segments * a.cluster));
            cfg.blockDim = dim3(kWarps * 32);
            cfg.dynamicSmemBytes = F::kSmem;
            cfg.stream = stream;
            cfg.attrs = attr;
            cfg.numAttrs = 2;
            auto kernel = paged_attention_kernel<DP, MT, kSplit, true>;
            e = cudaLaunchKernelEx(&cfg, kernel, a, k_map, v_map);
        }
        if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
        return finish_launch();
    });
}

}  // extern "C"
