// The pages of the paged cache between two steps: who has which, copies of those that two texts would write to, compaction.
//
// References are counted: refs[page] is how often tables name the page, 0 where it is free. Every result is determined by its inputs -
// the k-th page asked for is the k-th lowest free one - so nothing depends on which block comes first, and atomics add whole numbers.
//
// What there is to read and write is small (64 x 8 sequences of 40 blocks and 8000 pages: 230 KB), so the launches are what it costs:
// one that looks at all pages and all sequences side by side, and one that writes. A bit for each free page and a count for each
// 1024 of them lead from a request's number to its page in one binary search and one warp's look at 32 words. Where there are few sequences
// and pages a cluster of blocks does it all in one launch.
#include "common.cuh"

namespace ogle {
namespace {

constexpr int kThreads = 256;
constexpr int kChunkPages = kThreads * 4;        // pages that a block looks at at a time
constexpr int kMostChunks = 1024;
constexpr int kMostPages = 1 << 26;

// Pages in chunks: one count for each, one bit for each page.
struct Pool {
    int n_pages, chunk, chunks;                  // pages of a chunk: a multiple of kChunkPages
    unsigned* bits;
    int* counts;
};

struct AdvanceArgs {
    OgleAdvanceParams p;
    Pool pool;                                   // of the free pages
    int *children, *first_child;                 // of each old sequence: texts that go on from it; the first of them
    int* base;                                   // of each new one: requests of those before it; then all of them
    int page_shift;
};

__device__ __forceinline__ bool is_page(int page, int n_pages) { return (unsigned)page < (unsigned)n_pages; }

// A block's part of the pool: bits and count of the pages for which `wanted` holds, the counts copied on the way.
template <typename F>
__device__ __forceinline__ void scan_chunk(const Pool& pool, int chunk, const int* refs, int* out, F wanted) {
    __shared__ int sums[kThreads / 32];
    const int tid = threadIdx.x, first = chunk * pool.chunk, end = min(first + pool.chunk, pool.n_pages);
    int mine = 0;
    for (int p0 = first; p0 < end; p0 += kChunkPages) {
        int r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int p = p0 + u * kThreads + tid;
            r[u] = p < end ? __ldg(refs + p) : 1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int p = p0 + u * kThreads + tid;
            const unsigned b = __ballot_sync(~0u, p < end && wanted(r[u]));
            if (p < end) out[p] = r[u];
            if ((tid & 31) == 0 && p < end) {
                pool.bits[p / 32] = b;
                mine += __popc(b);
            }
        }
    }
    if ((tid & 31) == 0) sums[tid / 32] = mine;
    __syncthreads();
    if (tid == 0) {
        int all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) all += sums[w];
        pool.counts[chunk] = all;
    }
}

// Exclusive sums of the chunks' counts, in shared memory, and their total. A whole block of 32 * kWarps threads.
template <int kWarps>
__device__ __forceinline__ int sum_chunks(const Pool& pool, int* before) {
    __shared__ int sums[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, per = (pool.chunks + kWarps * 32 - 1) / (kWarps * 32);
    int mine = 0;
    for (int i = 0; i < per; ++i) {
        const int c = tid * per + i;
        if (c < pool.chunks) mine += pool.counts[c];
    }
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += o;
    }
    if (lane == 31) sums[tid / 32] = sum;
    __syncthreads();
    int total = 0, at = sum - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < tid / 32) at += sums[w];
        total += sums[w];
    }
    for (int i = 0; i < per; ++i) {
        const int c = tid * per + i;
        if (c < pool.chunks) {
            before[c] = at;
            at += pool.counts[c];
        }
    }
    __syncthreads();
    return total;
}

// The k-th page whose bit is set, of more than k: a warp's work.
__device__ __forceinline__ int kth_page(const Pool& pool, const int* before, int k) {
    int lo = 0, hi = pool.chunks;                // the last chunk that begins at or before k
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (before[mid] <= k) lo = mid;
        else hi = mid;
    }
    const int lane = threadIdx.x & 31, words = (pool.n_pages + 31) / 32;
    int left = k - before[lo];
    for (int w0 = lo * (pool.chunk / 32); w0 < words; w0 += 32) {
        const unsigned b = w0 + lane < words ? pool.bits[w0 + lane] : 0u;
        int sum = __popc(b);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int o = __shfl_up_sync(~0u, sum, d);
            if (lane >= d) sum += o;
        }
        const int n = __popc(b);
        const unsigned here = __ballot_sync(~0u, left < sum);
        if (here) {
            const int l = __ffs(here) - 1;
            int page = -1;
            if (lane == l) page = (w0 + lane) * 32 + __fns(b, 0, left - (sum - n) + 1);
            return __shfl_sync(~0u, page, l);
        }
        left -= __shfl_sync(~0u, sum, 31);
    }
    return -1;
}

// What becomes of a new text's blocks.
struct Text {
    int parent, length, full;                    // blocks [0, full) are shared with the parent
    int half;                                    // the parent's page of the block that is half full, -1: none
    bool half_full, keeps;                       // there is such a block; its page goes on with this text
    int first_wanted, end;                       // blocks that ask for a page
};

__device__ __forceinline__ Text text_of(const AdvanceArgs& a, int i) {
    const OgleAdvanceParams& p = a.p;
    Text t;
    t.parent = __ldg(p.parent + i);
    if ((unsigned)t.parent >= (unsigned)p.n_old) t.parent = -1;
    t.length = t.parent >= 0 ? max(__ldg(p.kv_len + t.parent), 0) : 0;
    const int more = max(p.tokens ? __ldg(p.tokens + i) : p.new_tokens, 0), part = t.length & ((1 << a.page_shift) - 1);
    t.full = t.length >> a.page_shift;
    t.half_full = part > 0;
    t.half = -1;
    t.keeps = false;
    if (t.half_full && t.full < p.old_blocks && t.full < p.new_blocks) {
        const int page = __ldg(p.table + t.parent * p.old_stride + t.full);
        if (is_page(page, p.n_pages)) {
            t.half = page;
            t.keeps = __ldg(p.refs + page) == 1 && __ldcg(a.first_child + t.parent) == i;
        }
    }
    t.first_wanted = t.full + (t.half_full && (t.half < 0 || t.keeps));
    const long long blocks = ((long long)t.length + more + (1 << a.page_shift) - 1) >> a.page_shift;
    t.end = int(min(blocks, (long long)p.new_blocks));
    t.first_wanted = min(t.first_wanted, t.end);
    return t;
}

// The blocks of a cluster meet; what each has written is there for the others.
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Who has which parent, and how many pages the texts before each ask for. A block's work.
__device__ __forceinline__ void plan_texts(const AdvanceArgs& a) {
    const OgleAdvanceParams& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < 2) p.state[tid] = 0;
    for (int i = tid; i < p.n_old; i += kThreads) {
        a.children[i] = 0;
        a.first_child[i] = 0x7fffffff;
    }
    __syncthreads();
    for (int i = tid; i < p.n_new; i += kThreads) {
        const int parent = __ldg(p.parent + i);
        if ((unsigned)parent < (unsigned)p.n_old) {
            atomicAdd(a.children + parent, 1);
            atomicMin(a.first_child + parent, i);
        }
    }
    __syncthreads();
    __shared__ int sums[kThreads / 32];
    int before = 0;
    for (int i0 = 0; i0 < p.n_new; i0 += kThreads) {
        const int i = i0 + tid;
        int wanted = 0;
        if (i < p.n_new) {
            const Text t = text_of(a, i);
            wanted = t.end - t.first_wanted;
        }
        int sum = wanted;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int o = __shfl_up_sync(~0u, sum, d);
            if (lane >= d) sum += o;
        }
        if (lane == 31) sums[tid / 32] = sum;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < tid / 32) sum += sums[w];
            all += sums[w];
        }
        if (i < p.n_new) a.base[i] = before + sum - wanted;
        before += all;
        __syncthreads();
    }
    if (tid == 0) a.base[p.n_new] = before;
}

// The table's row of new text i, and what the old sequence i gives back. A block's work.
template <int kRowWarps>
__device__ __forceinline__ void advance_row(const AdvanceArgs& a, int i) {
    __shared__ int before[kMostChunks];
    __shared__ int freed;
    const OgleAdvanceParams& p = a.p;
    const int tid = threadIdx.x;
    if (tid == 0) freed = 0;
    if (i < p.n_new) {
        const Text t = text_of(a, i);
        const int base = __ldcg(a.base + i), wanted = t.end - t.first_wanted;
        int free_pages = 0;
        if (wanted > 0 || i == 0) free_pages = sum_chunks<kRowWarps>(a.pool, before);
        int* row = p.new_table + i * p.new_stride;
        for (int c = tid; c < p.new_blocks; c += kRowWarps * 32) {
            int page = -1;
            if (t.parent >= 0 && c < p.old_blocks && (c < t.full || c == t.full && t.keeps)) page = __ldg(p.table + t.parent * p.old_stride + c);
            if (c < t.first_wanted || c >= t.end) row[c] = page;
        }
        for (int k = tid / 32; k < wanted; k += kRowWarps) {
            const int page = base + k < free_pages ? kth_page(a.pool, before, base + k) : -1;
            if ((tid & 31) == 0) {
                row[t.first_wanted + k] = page;
                if (page >= 0) atomicAdd(p.new_refs + page, 1);
            }
            if (k == 0 && (tid & 31) == 0) {
                const bool copied = t.half >= 0 && !t.keeps && page >= 0;
                p.copies[3 * i] = copied ? t.half : -1;
                p.copies[3 * i + 1] = copied ? page : -1;
                p.copies[3 * i + 2] = copied ? t.length & ((1 << a.page_shift) - 1) : 0;
            }
        }
        if (tid == 0) {
            if (wanted <= 0) { p.copies[3 * i] = p.copies[3 * i + 1] = -1; p.copies[3 * i + 2] = 0; }
            p.new_len[i] = int(min((long long)t.length + max(p.tokens ? __ldg(p.tokens + i) : p.new_tokens, 0), 0x7fffffffLL));
            if (i == 0) {
                const int all = __ldcg(a.base + p.n_new), granted = min(all, free_pages);
                atomicAdd(p.state, free_pages - granted);
                atomicAdd(p.state + 1, all - granted);
            }
        }
    }
    if (i < p.n_old) {
        const int children = __ldcg(a.children + i), length = max(__ldg(p.kv_len + i), 0), full = length >> a.page_shift;
        const bool half_full = (length & ((1 << a.page_shift) - 1)) > 0;
        int mine = 0;
        for (int c = tid; c < p.old_blocks; c += kRowWarps * 32) {
            const int page = __ldg(p.table + i * p.old_stride + c);
            if (!is_page(page, p.n_pages)) continue;
            int n = 0;                           // of the new texts that name it here
            if (c < p.new_blocks) {
                if (c < full) n = children;
                else if (c == full && half_full) n = children > 0 && __ldg(p.refs + page) == 1;
            }
            if (n != 1) mine += atomicAdd(p.new_refs + page, n - 1) + n - 1 == 0;
        }
        __syncthreads();
        if (mine) atomicAdd(&freed, mine);
        __syncthreads();
        if (tid == 0 && freed) atomicAdd(p.state, freed);
    }
    if (i == 0 && p.n_new == 0 && tid < 32) {    // nobody above has counted the free pages
        int n = 0;
        for (int c = tid; c < a.pool.chunks; c += 32) n += a.pool.counts[c];
#pragma unroll
        for (int d = 16; d; d /= 2) n += __shfl_xor_sync(~0u, n, d);
        if (tid == 0) atomicAdd(p.state, n);
    }
}

constexpr int kRowWarps = 4, kFewRows = 24, kFewChunks = 8;

// Blocks [0, chunks): the pool. The last block: the sequences.
__global__ void __launch_bounds__(kThreads) advance_plan_kernel(AdvanceArgs a) {
    grid_dependency_trigger();
    grid_dependency_wait();
    if (int(blockIdx.x) < a.pool.chunks) scan_chunk(a.pool, blockIdx.x, a.p.refs, a.p.new_refs, [](int r) { return r == 0; });
    else plan_texts(a);
}
__global__ void __launch_bounds__(kRowWarps * 32) advance_rows_kernel(AdvanceArgs a) {
    grid_dependency_trigger();
    grid_dependency_wait();
    advance_row<kRowWarps>(a, blockIdx.x);
}
// Both, by a cluster of kFewChunks blocks: a launch less, 2 us of the host's 18 for a call with 4 texts, and on the device 7 us instead of 8.
__global__ void __launch_bounds__(kThreads) advance_few_kernel(AdvanceArgs a) {
    const int rank = blockIdx.x, rows = max(max(a.p.n_new, a.p.n_old), 1);
    grid_dependency_trigger();
    grid_dependency_wait();
    if (rank < a.pool.chunks) scan_chunk(a.pool, rank, a.p.refs, a.p.new_refs, [](int r) { return r == 0; });
    if (rank == kFewChunks - 1) plan_texts(a);
    cluster_meet();
    for (int i = rank; i < rows; i += kFewChunks) {
        advance_row<kThreads / 32>(a, i);
        __syncthreads();
    }
}

// ---- compaction
struct CompactArgs {
    OgleCompactParams p;
    Pool pool;                                   // of the used pages
    int* rank;                                   // of a used page behind the border: its number among those
    int* used;                                   // the border: pages in use
};

__global__ void __launch_bounds__(kThreads) compact_scan_kernel(CompactArgs a) {
    grid_dependency_trigger();
    grid_dependency_wait();
    scan_chunk(a.pool, blockIdx.x, a.p.refs, a.p.new_refs, [](int r) { return r != 0; });
}

// Pages in use below `page`: the sums of the chunks before it, and of the words before it in its chunk. A warp's work.
__device__ __forceinline__ int used_below(const Pool& pool, const int* before, int total, int page) {
    const int lane = threadIdx.x & 31;
    if (page >= pool.n_pages) return total;
    const int chunk = page / pool.chunk;
    int n = 0;
    for (int w = chunk * (pool.chunk / 32) + lane; w <= page / 32; w += 32) {
        const unsigned b = pool.bits[w];
        n += __popc(w < page / 32 ? b : b & ((1u << (page & 31)) - 1));
    }
#pragma unroll
    for (int d = 16; d; d /= 2) n += __shfl_xor_sync(~0u, n, d);
    return before[chunk] + n;
}

// The k-th used page behind the border and the k-th free one before it get copy k. A block's work, for the pages of a chunk.
__device__ __forceinline__ void pair_chunk(const CompactArgs& a, int chunk) {
    __shared__ int before[kMostChunks];
    __shared__ int below_border;
    const OgleCompactParams& p = a.p;
    const Pool& pool = a.pool;
    const int tid = threadIdx.x, lane = tid & 31;
    const int used = sum_chunks<kThreads / 32>(pool, before);
    if (tid < 32) {
        const int n = used_below(pool, before, used, used);
        if (tid == 0) below_border = n;
    }
    __syncthreads();
    const int moves = used - below_border;       // used behind the border, and free before it
    if (chunk == 0) {
        if (tid == 0) {
            *a.used = used;
            p.state[0] = used;
            p.state[1] = moves - min(moves, p.n_copies);
        }
        for (int k = moves + tid; k < p.n_copies; k += kThreads) {
            p.copies[3 * k] = p.copies[3 * k + 1] = -1;
            p.copies[3 * k + 2] = 0;
        }
    }
    const int first = chunk * pool.chunk, end = min(first + pool.chunk, pool.n_pages);
    if (first >= end) return;
    int sum = before[chunk];                // used pages below the warp's word, kept by each warp for itself
    const int words = (end - first + 31) / 32;
    for (int w0 = 0; w0 < words; w0 += 32) {     // 32 words: every warp sums them, each then has every eighth
        const unsigned b = w0 + lane < words ? pool.bits[first / 32 + w0 + lane] : 0u;
        int in = __popc(b);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int o = __shfl_up_sync(~0u, in, d);
            if (lane >= d) in += o;
        }
        const int ex = in - __popc(b);
        for (int w = tid / 32; w < 32; w += kThreads / 32) {
            const unsigned word = __shfl_sync(~0u, b, w);
            const int page = first + (w0 + w) * 32 + lane, n = sum + __shfl_sync(~0u, ex, w) + __popc(word & ((1u << lane) - 1));
            if (page >= end) continue;
            const bool is_used = word >> lane & 1;
            if (is_used && page >= used) {
                const int k = n - below_border;
                a.rank[page] = k;
                if (k < p.n_copies) {
                    p.copies[3 * k] = page;
                    p.copies[3 * k + 2] = p.page_tokens;
                }
            } else if (!is_used && page < used) {
                const int k = page - n;
                if (k < p.n_copies) p.copies[3 * k + 1] = page;
            }
        }
        sum += __shfl_sync(~0u, in, 31);
    }
}

// New numbers in the table, and the counts' places. All blocks' work.
__device__ __forceinline__ void rename_pages(const CompactArgs& a) {
    const OgleCompactParams& p = a.p;
    const int used = *a.used;
    const long long entries = (long long)p.n_seqs * p.blocks, all = entries + p.n_copies;
    for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < all; i += (long long)gridDim.x * kThreads) {
        if (i < entries) {
            const int row = int(i / p.blocks), c = int(i % p.blocks);
            int page = p.table[row * p.table_stride + c];        // (not a read-only load: new_table may be table)
            if (is_page(page, p.n_pages) && page >= used && __ldg(p.refs + page) != 0) {
                const int k = a.rank[page];
                if (k < p.n_copies) page = p.copies[3 * k + 1];
            }
            p.new_table[row * p.new_stride + c] = page;
        } else {
            const int k = int(i - entries), src = p.copies[3 * k], dst = p.copies[3 * k + 1];
            if (src >= 0) {
                p.new_refs[dst] = __ldg(p.refs + src);
                p.new_refs[src] = 0;
            }
        }
    }
}

__global__ void __launch_bounds__(kThreads) compact_pair_kernel(CompactArgs a) {
    grid_dependency_trigger();
    grid_dependency_wait();
    pair_chunk(a, blockIdx.x);
}
__global__ void __launch_bounds__(kThreads) compact_table_kernel(CompactArgs a) {
    grid_dependency_trigger();
    grid_dependency_wait();
    rename_pages(a);
}
// All three, by a cluster of kFewChunks blocks: 7 us on the device, as in three launches, and 14 us of the host's instead of 18.
constexpr int kFewItems = 1 << 15;               // of the table and of the copies
__global__ void __launch_bounds__(kThreads) compact_few_kernel(CompactArgs a) {
    const int rank = blockIdx.x;
    grid_dependency_trigger();
    grid_dependency_wait();
    if (rank < a.pool.chunks) scan_chunk(a.pool, rank, a.p.refs, a.p.new_refs, [](int r) { return r != 0; });
    cluster_meet();
    if (rank < a.pool.chunks) pair_chunk(a, rank);
    cluster_meet();
    rename_pages(a);
}

// ---- copies
// A window of copies is shared out among the blocks (., y): each adds up how many units its copies have - many have nothing to copy, others a
// token or a page -, and its warps take every so-many-th unit. (A warp to every unit that there could be: 512 texts with 200 copies of
// half a page in four layers, 107 MB: 35 us, 14 so.)
constexpr int kMostLayers = 64;                  // of a launch
constexpr int kWindow = 1024;                    // copies that a block looks over, most
constexpr int kDeal = 8;                         // copies next to each other in a window: the windows are dealt them in turn, as lists often end early
                                                 // (733 moves of 128 KB in four layers in a list for 3921: 120 us, 65 so)
struct CopyArgs {
    int n_copies, n_layers, kv_heads, dim, page_tokens, n_pages;
    long long page_stride, head_stride, token_stride;
    const int* copies;
    int unit_rows;                               // rows (a token of a head) of a unit
    int packed;                                  // a page's bytes lie in one piece
    OglePageTensors layer[kMostLayers];
};
struct Entry { int src, dst, tokens; };
__device__ __forceinline__ Entry entry_at(const CopyArgs& a, int c) {
    const int* const e = a.copies + 3LL * c;
    Entry x = {__ldg(e), __ldg(e + 1), min(max(__ldg(e + 2), 0), a.page_tokens)};
    if (!is_page(x.src, a.n_pages) || !is_page(x.dst, a.n_pages) || x.src == x.dst) x.src = -1;
    return x;
}

// The window's copies; first[i]: units of those before the i-th; returns all copies'. A whole block of kN threads.
template <int kN, typename F>
__device__ __forceinline__ int sum_units(const CopyArgs& a, int* first, Entry* entries, F units) {
    __shared__ int sums[kN / 32];
    constexpr int kMine = kWindow / kN;
    const int tid = threadIdx.x, lane = tid & 31, windows = gridDim.y, window = blockIdx.y;
    int mine[kMine], all_mine = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {            // (neighbours read neighbours: thread t has entries t, t + kN, ...)
        const int c = i * kN + tid, copy = (c / kDeal * windows + window) * kDeal + c % kDeal;
        mine[i] = 0;
        if (copy < a.n_copies) {
            const Entry e = entry_at(a, copy);
            entries[c] = e;
            if (e.src >= 0) mine[i] = units(e);
        }
        first[c] = mine[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        mine[i] = first[tid * kMine + i];
        all_mine += mine[i];
    }
    int sum = all_mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += o;
    }
    if (lane == 31) sums[tid / 32] = sum;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kN / 32; ++w) {
        if (w < tid / 32) sum += sums[w];
        total += sums[w];
    }
    int at = sum - all_mine;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        first[tid * kMine + i] = at;
        at += mine[i];
    }
    __syncthreads();
    return total;
}
__device__ __forceinline__ int copy_of(const int* first, int unit) {       // the last copy that begins at or before it
    int lo = 0, hi = kWindow;
#pragma unroll 1
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A warp has a unit of one page's keys or values in one layer, by loads and stores of 16 bytes; that of a page's first unit takes its scales,
// too. 8192 pages of 3 KB in four layers, 403 MB: 71 us, 87 % of what a copy reaches. (Runs of up to 4 KB through shared memory by the copy
// engine, 48 of an SM under way: 80 to 100; half a unit loaded while the last one is stored, in 64 registers: 150.)
constexpr int kUnit = 4096;                      // bytes of a unit: 8 x 16 a lane
constexpr int kCopyBlocks = 2;                   // that fit an SM at once (three, in 85 registers, keep a unit's places in memory: 100 us)
__global__ void __launch_bounds__(kThreads, kCopyBlocks) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    __shared__ int first[kWindow];
    __shared__ Entry entries[kWindow];
    const int tid = threadIdx.x, lane = tid & 31;
    grid_dependency_trigger();
    grid_dependency_wait();
    const int total = sum_units<kThreads>(a, first, entries, [&](const Entry& e) { return max((a.kv_heads * e.tokens + a.unit_rows - 1) / a.unit_rows, 1); });
    const int all = total * a.n_layers * 2, step = gridDim.x * (kThreads / 32), vecs = a.dim / 16;
    const float by_vecs = 1.f / float(vecs);
    for (int u = blockIdx.x * (kThreads / 32) + tid / 32; u < all; u += step) {
        const int which = u / total, kind = which & 1, of = u - which * total;
        const int c = copy_of(first, of);
        const Entry e = entries[c];
        const int src = e.src, dst = e.dst, tokens = e.tokens, unit = of - first[c];
        const OglePageTensors& t = a.layer[which >> 1];
        unsigned char* const base = static_cast<unsigned char*>(kind ? t.v : t.k);
        const unsigned char* const from = base + src * a.page_stride;
        unsigned char* const to = base + dst * a.page_stride;
        // a head's scale to a lane, under way with the rest
        float* const scales = kind ? t.v_scale : t.k_scale;
        float scale = 0.f;
        if (unit == 0 && lane < a.kv_heads) scale = scales[(long long)src * a.kv_heads + lane];
        const int rows = min(a.kv_heads * tokens - unit * a.unit_rows, a.unit_rows), n_vecs = rows * vecs;
        const bool whole = a.packed && tokens == a.page_tokens;
        // places in the page, in 16 bytes
        constexpr int U = kUnit / 512;
        const uint4* const in = reinterpret_cast<const uint4*>(from);
        uint4* const out = reinterpret_cast<uint4*>(to);
        if (whole) {
            const uint4* const mine = in + (size_t)unit * a.unit_rows * vecs + lane;
            uint4* const yours = out + (size_t)unit * a.unit_rows * vecs + lane;
            uint4 v[U];
#pragma unroll
            for (int x = 0; x < U; ++x)
                if (x * 32 + lane < n_vecs) v[x] = mine[x * 32];
#pragma unroll
            for (int x = 0; x < U; ++x)
                if (x * 32 + lane < n_vecs) yours[x * 32] = v[x];
        } else {
            // quotients by reciprocals: of i below 256 exactly, of rows (2^22 at most) within one
            const float by_tokens = 1.f / float(max(tokens, 1));
            const uint32_t per_head = uint32_t(a.head_stride >> 4), per_token = uint32_t(a.token_stride >> 4);
            uint32_t at[U];
            uint4 v[U];
#pragma unroll
            for (int x = 0; x < U; ++x) {
                const int i = x * 32 + lane;
                const int r = int((float(i) + 0.5f) * by_vecs), row = unit * a.unit_rows + r;
                int h = int((float(row) + 0.5f) * by_tokens), t = row - h * tokens;
                if (t < 0) { --h; t += tokens; }
                if (t >= tokens) { ++h; t -= tokens; }
                at[x] = h * per_head + t * per_token + (i - r * vecs);
                if (i < n_vecs) v[x] = in[at[x]];
            }
#pragma unroll
            for (int x = 0; x < U; ++x)
                if (x * 32 + lane < n_vecs) out[at[x]] = v[x];
        }
        if (unit > 0) continue;
        if (lane < a.kv_heads) scales[(long long)dst * a.kv_heads + lane] = scale;
        for (int h = lane + 32; h < a.kv_heads; h += 32) scales[(long long)dst * a.kv_heads + h] = scales[(long long)src * a.kv_heads + h];
        if (kind == 0 && t.bounds) {
            const long long bytes = 2LL * a.kv_heads * a.dim;
            const uint4* const f = reinterpret_cast<const uint4*>(t.bounds + src * bytes);
            uint4* const g = reinterpret_cast<uint4*>(t.bounds + dst * bytes);
            for (int i = lane; i < bytes / 16; i += 32) g[i] = f[i];
            for (int h = lane; h < a.kv_heads; h += 32) t.bounds_scale[(long long)dst * a.kv_heads + h] = t.bounds_scale[(long long)src * a.kv_heads + h];
        }
    }
}

Pool pool_of(int n_pages) {
    Pool pool = {};
    pool.n_pages = n_pages;
    pool.chunk = kChunkPages;
    while (div_up(n_pages, pool.chunk) > kMostChunks) pool.chunk *= 2;
    pool.chunks = div_up(n_pages, pool.chunk);
    return pool;
}
size_t pool_words(const Pool& pool) { return size_t(pool.n_pages + 31) / 32 + pool.chunks; }
bool page_size_ok(int tokens) { return tokens >= 16 && tokens <= 1024 && (tokens & (tokens - 1)) == 0; }
int failed(cudaError_t e) {
    set_last_error(e);
    (void)cudaGetLastError();
    return OGLE_ERR_CUDA;
}

// A launch of one cluster of kFewChunks blocks.
template <typename Args>
cudaError_t launch_few(void (*kernel)(Args), const Args& a, cudaStream_t stream) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlapped_launches_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kFewChunks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kFewChunks);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

int check_advance(const OgleAdvanceParams* p) {
    if (!p || p->n_old < 0 || p->n_new < 0 || p->old_blocks < 0 || p->new_blocks < 0 || p->n_pages < 0 || !page_size_ok(p->page_tokens)) return OGLE_ERR_INVALID;
    if (p->n_pages > kMostPages || p->n_old > (1 << 24) || p->n_new > (1 << 24) || p->new_blocks > (1 << 24) || p->old_blocks > (1 << 24)) return OGLE_ERR_UNSUPPORTED;
    if ((long long)p->n_new * p->new_blocks >= (1LL << 31)) return OGLE_ERR_UNSUPPORTED;      // requests are counted in 32 bits
    if ((p->n_old > 1 && p->old_stride < p->old_blocks) || (p->n_new > 1 && p->new_stride < p->new_blocks)) return OGLE_ERR_INVALID;
    return OGLE_OK;
}
int check_compact(const OgleCompactParams* p) {
    if (!p || p->n_seqs < 0 || p->blocks < 0 || p->n_pages < 0 || p->n_copies < 0 || !page_size_ok(p->page_tokens)) return OGLE_ERR_INVALID;
    if (p->n_pages > kMostPages || p->n_copies > (1 << 28)) return OGLE_ERR_UNSUPPORTED;
    if (p->n_seqs > 1 && (p->table_stride < p->blocks || p->new_stride < p->blocks)) return OGLE_ERR_INVALID;
    return OGLE_OK;
}

}  // namespace
}  // namespace ogle

using namespace ogle;

extern "C" {

size_t ogle_cuda_advance_pages_workspace_bytes(const OgleAdvanceParams* p) {
    if (check_advance(p) != OGLE_OK) return 0;
    return (pool_words(pool_of(p->n_pages)) + 2 * size_t(p->n_old) + p->n_new + 1) * 4;
}

int ogle_cuda_advance_pages(const OgleAdvanceParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream) {
    const int rc = check_advance(p);
    if (rc != OGLE_OK) return rc;
    if (!p->state || (p->n_pages > 0 && (!p->refs || !p->new_refs)) || (p->n_old > 0 && (!p->table || !p->kv_len)) ||
        (p->n_new > 0 && (!p->parent || !p->new_table || !p->new_len || !p->copies)) || !workspace)
        return OGLE_ERR_INVALID;
    // the rows of several texts read the row of one
    if ((p->n_pages > 0 && p->refs == p->new_refs) || (p->n_new > 0 && (p->table == p->new_table || p->kv_len == p->new_len))) return OGLE_ERR_INVALID;
    if (workspace_bytes < ogle_cuda_advance_pages_workspace_bytes(p)) return OGLE_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(workspace) & 3) return OGLE_ERR_ALIGNMENT;
    AdvanceArgs a = {};
    a.p = *p;
    a.pool = pool_of(p->n_pages);
    a.pool.bits = static_cast<unsigned*>(workspace);
    a.pool.counts = reinterpret_cast<int*>(a.pool.bits + (p->n_pages + 31) / 32);
    a.children = a.pool.counts + a.pool.chunks;
    a.first_child = a.children + p->n_old;
    a.base = a.first_child + p->n_old;
    a.page_shift = 4;
    while ((1 << a.page_shift) < p->page_tokens) ++a.page_shift;
    const int rows = p->n_new > p->n_old ? p->n_new : p->n_old;
    cudaError_t e;
    if (a.pool.chunks <= kFewChunks && rows <= kFewRows) {
        e = launch_few(advance_few_kernel, a, stream);
        return e == cudaSuccess ? finish_launch() : failed(e);
    }
    e = launch_overlapped(advance_plan_kernel, dim3(a.pool.chunks + 1), dim3(kThreads), 0, stream, a);
    if (e != cudaSuccess) return failed(e);
    const int done = finish_launch();
    if (done != OGLE_OK) return done;
    e = launch_overlapped_if(overlapped_launches_enabled(true), advance_rows_kernel, dim3(rows < 1 ? 1 : rows), dim3(kRowWarps * 32), 0, stream, a);
    return e == cudaSuccess ? finish_launch() : failed(e);
}

size_t ogle_cuda_compact_pages_workspace_bytes(const OgleCompactParams* p) {
    if (check_compact(p) != OGLE_OK) return 0;
    return (pool_words(pool_of(p->n_pages)) + size_t(p->n_pages) + 1) * 4;
}

int ogle_cuda_compact_pages(const OgleCompactParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream) {
    const int rc = check_compact(p);
    if (rc != OGLE_OK) return rc;
    const bool table = p->n_seqs > 0 && p->blocks > 0;
    if (!p->state || (p->n_pages > 0 && (!p->refs || !p->new_refs)) || (table && (!p->table || !p->new_table)) || (p->n_copies > 0 && !p->copies) || !workspace)
        return OGLE_ERR_INVALID;
    if (p->n_pages > 0 && p->refs == p->new_refs) return OGLE_ERR_INVALID;
    if (workspace_bytes < ogle_cuda_compact_pages_workspace_bytes(p)) return OGLE_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(workspace) & 3) return OGLE_ERR_ALIGNMENT;
    CompactArgs a = {};
    a.p = *p;
    a.pool = pool_of(p->n_pages);
    a.pool.bits = static_cast<unsigned*>(workspace);
    a.pool.counts = reinterpret_cast<int*>(a.pool.bits + (p->n_pages + 31) / 32);
    a.rank = a.pool.counts + a.pool.chunks;
    a.used = a.rank + p->n_pages;
    const bool overlapped = overlapped_launches_enabled(true);
    cudaError_t e = cudaSuccess;
    int done = OGLE_OK;
    const long items = (table ? (long)p->n_seqs * p->blocks : 0) + p->n_copies;
    if (!table) a.p.n_seqs = a.p.blocks = 0;
    if (a.pool.chunks >= 1 && a.pool.chunks <= kFewChunks && items <= kFewItems) {
        e = launch_few(compact_few_kernel, a, stream);
        return e == cudaSuccess ? finish_launch() : failed(e);
    }
    if (p->n_pages > 0) {
        e = launch_overlapped(compact_scan_kernel, dim3(a.pool.chunks), dim3(kThreads), 0, stream, a);
        if (e != cudaSuccess) return failed(e);
        done = finish_launch();
        if (done != OGLE_OK) return done;
    }
    e = launch_overlapped_if(overlapped && p->n_pages > 0, compact_pair_kernel, dim3(a.pool.chunks > 0 ? a.pool.chunks : 1), dim3(kThreads), 0, stream, a);
    if (e != cudaSuccess) return failed(e);
    done = finish_launch();
    if (done != OGLE_OK || items == 0) return done;
    e = launch_overlapped_if(overlapped, compact_table_kernel, dim3(grid_for(items, kThreads)), dim3(kThreads), 0, stream, a);
    return e == cudaSuccess ? finish_launch() : failed(e);
}

int ogle_cuda_copy_pages(const OgleCopyPagesParams* p, const OglePageTensors* layers_host_array, ogle_stream_t stream) {
    if (!p || p->n_copies < 0 || p->n_layers < 0 || p->n_pages < 0 || p->kv_heads < 1 || p->kv_heads > 4096 || !page_size_ok(p->page_tokens)) return OGLE_ERR_INVALID;
    if (p->head_dim < 16 || p->head_dim % 16 != 0) return OGLE_ERR_INVALID;
    if (p->head_dim > 256) return OGLE_ERR_UNSUPPORTED;
    if ((p->page_stride | p->head_stride | p->token_stride) & 15) return OGLE_ERR_ALIGNMENT;
    if (p->page_stride < 1 || p->head_stride < 1 || p->token_stride < p->head_dim) return OGLE_ERR_INVALID;
    if (p->n_copies == 0 || p->n_layers == 0 || p->n_pages == 0) return OGLE_OK;
    if (!p->copies || !layers_host_array) return OGLE_ERR_INVALID;
    for (int l = 0; l < p->n_layers; ++l) {
        const OglePageTensors& t = layers_host_array[l];
        if (!t.k || !t.v || !t.k_scale || !t.v_scale || (t.bounds && !t.bounds_scale)) return OGLE_ERR_INVALID;
        if (!aligned16(t.k) || !aligned16(t.v) || !aligned16(t.bounds)) return OGLE_ERR_ALIGNMENT;
    }
    CopyArgs a;
    a.n_copies = p->n_copies; a.kv_heads = p->kv_heads; a.dim = p->head_dim; a.page_tokens = p->page_tokens; a.n_pages = p->n_pages;
    a.page_stride = p->page_stride; a.head_stride = p->head_stride; a.token_stride = p->token_stride;
    a.copies = p->copies;
    a.unit_rows = kUnit / p->head_dim;
    a.packed = p->token_stride == p->head_dim && p->head_stride == p->token_stride * p->page_tokens;
    // places in a page are counted in 32 bits, in 16 bytes each
    if ((p->kv_heads - 1) * (p->head_stride >> 4) + (p->page_tokens - 1) * (p->token_stride >> 4) >= (1LL << 32) - 16) return OGLE_ERR_UNSUPPORTED;
    const long most_units = div_up((long)p->kv_heads * p->page_tokens, a.unit_rows);
    // a window's units are counted in 32 bits, its windows in a grid's second dimension
    if (most_units * kWindow * kMostLayers * 2 >= (1L << 31) || p->n_copies > 65535 * kWindow) return OGLE_ERR_UNSUPPORTED;
    for (int first = 0; first < p->n_layers; first += kMostLayers) {
        a.n_layers = p->n_layers - first < kMostLayers ? p->n_layers - first : kMostLayers;
        for (int l = 0; l < a.n_layers; ++l) a.layer[l] = layers_host_array[first + l];
        // one round of blocks for all windows
        const long windows = div_up(p->n_copies, kWindow), units = (long)(p->n_copies < kWindow ? p->n_copies : kWindow) * a.n_layers * 2 * most_units;
        const long at_once = windows < kNumSMs * kCopyBlocks ? kNumSMs * kCopyBlocks / windows : 1;
        long blocks = div_up(units, kThreads / 32);
        if (blocks > at_once) blocks = at_once;
        const cudaError_t e = launch_overlapped(copy_pages_kernel, dim3((unsigned)blocks, (unsigned)windows), dim3(kThreads), 0, stream, a);
        if (e != cudaSuccess) return failed(e);
        const int rc = finish_launch();
        if (rc != OGLE_OK) return rc;
    }
    return OGLE_OK;
}

}  // extern "C"
