// Appending to the paged 8-bit cache: rotation by position, one power-of-two scale for each page and head, e4m3.
//
// A block has one page of one sequence and either one head of the keys, one of the values, or a few heads of the queries: the
// page's scale depends on all rows that come to it, and nothing else does, so no block waits for another and no sum has an
// order to depend on. The rows' values stay in registers between the maximum and the rounding.
//
// Bound by memory where prompts are appended: 26000 rows of 32 + 2 x 8 heads of 128 in bf16, 855 MB, 190 us, 69 % of what a copy
// reaches (three blocks an SM, 80 registers a thread; two blocks 221 us). Single tokens are bound by latency - row, maximum, page: 5 us
// on the device for 1 or 96 of them, 14 us a call.
#include <type_traits>

#include "paged.cuh"

namespace ogle {
namespace {

using paged::Batch;

struct AppendArgs {
    Batch b;
    const void *k, *v, *q;
    void* q_out;
    long long k_row, k_head, v_row, v_head, q_row, q_head, qo_row, qo_head;
    const float* rotary;
    int rotary_dim, interleaved;
    int q_blocks;                 // blocks of kQHeads query heads
};

constexpr int kQHeads = 4;        // query heads of a block: they share a row's angles
constexpr int kHoldValues = 32;   // values a thread keeps
constexpr int kMaxThreads = 256;

// A piece is 2 W values of a head in two vectors of W: at `at` and at `at2`. Inside the rotated part, with pairs rotary_dim / 2
// apart, they are both halves of W pairs; every other piece is neighbours.
struct Piece { int at, at2, angle; };  // angle: first column of the table's cosines, -1: not rotated

template <int W>
__device__ __forceinline__ Piece piece_of(int i, int rotary_dim, bool interleaved) {
    Piece p;
    p.at = i * 2 * W;
    p.at2 = p.at + W;
    p.angle = -1;
    if (p.at < rotary_dim) {
        p.angle = i * W;
        if (!interleaved) {
            p.at = i * W;
            p.at2 = p.at + rotary_dim / 2;
        }
    }
    return p;
}

// W values as they lie: one vector of 16 bytes, or of 8.
template <typename T, int W>
struct Raw { uint32_t w[W * sizeof(T) / 4]; };
template <typename T, int W>
__device__ __forceinline__ Raw<T, W> load_raw(const T* p) {
    Raw<T, W> r;
    if constexpr (W * sizeof(T) == 16) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    }
    return r;
}
template <typename T, int W>
__device__ __forceinline__ void unpack(const Raw<T, W>& r, float* x) {
    const T* h = reinterpret_cast<const T*>(r.w);
#pragma unroll
    for (int l = 0; l < W; ++l) x[l] = float(h[l]);
}
template <typename T, int W>
__device__ __forceinline__ void store_values(T* p, const float* x) {
    Raw<T, W> r;
    T* h = reinterpret_cast<T*>(r.w);
#pragma unroll
    for (int l = 0; l < W; ++l) h[l] = T(x[l]);
    if constexpr (W * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
}

template <int W>
__device__ __forceinline__ void load_angles(const float* p, float (&c)[W]) {
#pragma unroll
    for (int l = 0; l < W; l += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + l));
        c[l] = v.x; c[l + 1] = v.y; c[l + 2] = v.z; c[l + 3] = v.w;
    }
}

// Products and sums are rounded one by one (no fused multiply-add): what is stored in 8 bits is then the same as from any other
// evaluation of the formula in fp32, where a fused one crosses a rounding boundary now and then.
template <int W>
__device__ __forceinline__ void rotate(float (&x)[2 * W], const float (&c)[W], const float (&s)[W], bool interleaved) {
#pragma unroll
    for (int l = 0; l < W; ++l) {
        float& a = interleaved ? x[2 * l] : x[l];
        float& b = interleaved ? x[2 * l + 1] : x[W + l];
        const float u = __fsub_rn(__fmul_rn(a, c[l]), __fmul_rn(b, s[l]));
        const float v = __fadd_rn(__fmul_rn(b, c[l]), __fmul_rn(a, s[l]));
        a = u;
        b = v;
    }
}

template <typename T, int W>
__device__ __forceinline__ void load_piece(const T* row, const Piece& p, const float* cs, int half, bool interleaved, float (&x)[2 * W]) {
    const Raw<T, W> lo = load_raw<T, W>(row + p.at), hi = load_raw<T, W>(row + p.at2);
    if (p.angle >= 0) {
        float c[W], s[W];
        load_angles<W>(cs + p.angle, c);
        load_angles<W>(cs + half + p.angle, s);
        unpack<T, W>(lo, x);
        unpack<T, W>(hi, x + W);
        if (interleaved) rotate<W>(x, c, s, true);
        else rotate<W>(x, c, s, false);
    } else {
        unpack<T, W>(lo, x);
        unpack<T, W>(hi, x + W);
    }
}

// The smallest power of two s with amax <= 448 s, from the bits: 448 = 0.875 * 2^9. At least 2^-120, so that 1 / s is a normal number.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = int(u >> 23) - 126 - 9 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);     // amax = f * 2^(e + 9), f in [0.5, 1)
    return __uint_as_float(uint32_t(max(e, -120) + 127) << 23);
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
}

// Zeros in `vecs` x 16 bytes of each head of the rows. (Out of line and behind all else, and still 1.6 us of the 26000 rows' 190: it takes
// registers.)
__device__ __noinline__ void clear_rows(void* out, long long row_bytes, long long head_bytes, int rows, int heads, int vecs) {
    for (int i = threadIdx.x; i < rows * heads * vecs; i += blockDim.x) {
        const int row = i / (heads * vecs), h = i / vecs % heads;
        *reinterpret_cast<uint4*>(static_cast<unsigned char*>(out) + row * row_bytes + h * head_bytes + i % vecs * 16) = make_uint4(0, 0, 0, 0);
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(kMaxThreads, 3) paged_append_kernel(AppendArgs a) {
    __shared__ int where[4];
    __shared__ float warp_max[kMaxThreads / 32];
    const Batch& B = a.b;
    const int tid = threadIdx.x, page_tokens = 1 << B.page_shift;
    grid_dependency_trigger();
    grid_dependency_wait();
    // which sequence, and which of the pages that it appends to
    int b = blockIdx.x, nth = 0;
    if (B.max_rows > 1) {
        if (tid < 32) {
            int before = 0, found = -1;
            for (int b0 = 0; b0 < B.n_seqs; b0 += 32) {
                int pages = 0;
                if (b0 + tid < B.n_seqs) {
                    const paged::Sequence s = paged::sequence(B, b0 + tid);
                    const int p0 = max(s.first, 0), p1 = min(s.first + s.n, s.len);
                    pages = p1 > p0 ? ((p1 - 1) >> B.page_shift) - (p0 >> B.page_shift) + 1 : (s.n > 0 && s.first < 0);
                }
                int sum = pages;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int o = __shfl_up_sync(~0u, sum, d);
                    if (tid >= d) sum += o;
                }
                const int at = int(blockIdx.x) - before;
                const unsigned hit = __ballot_sync(~0u, at >= sum - pages && at < sum);
                if (hit) {
                    const int l = __ffs(hit) - 1;
                    found = b0 + l;
                    nth = at - (__shfl_sync(~0u, sum, l) - __shfl_sync(~0u, pages, l));
                    break;
                }
                before += __shfl_sync(~0u, sum, 31);
            }
            if (tid == 0) { where[0] = found; where[1] = nth; }
        }
        __syncthreads();
        b = where[0];
        nth = where[1];
        if (b < 0) return;
    }
    const paged::Sequence s = paged::sequence(B, b);
    const int begin = max(s.first, 0), end = min(s.first + s.n, s.len);          // the new tokens
    const bool clears = s.first < 0 && nth == 0 && int(blockIdx.y) >= 2 * B.kv_heads;    // rows before the text: their queries are 0
    if (end <= begin && !clears) return;
    const int block = (begin >> B.page_shift) + nth;             // of the sequence's blocks of tokens
    const int t0 = max(begin, block << B.page_shift), t1 = min(end, (block + 1) << B.page_shift);
    const int row0 = s.row0 - s.first;                           // row of token t: row0 + t
    // a thread has one piece of every `stride`-th token
    const int pieces = B.dim / (2 * W), half = a.rotary_dim / 2, stride = int(blockDim.x) / pieces, my_piece = tid % pieces;
    const int my_t = tid / pieces < stride ? t0 + tid / pieces : t1;
    const bool inter = a.interleaved != 0;

    if (int(blockIdx.y) >= 2 * B.kv_heads) {                     // queries: rotated and stored as they came
        const int h0 = (blockIdx.y - 2 * B.kv_heads) * kQHeads, heads = min(kQHeads, B.q_heads - h0);
        const Piece p = piece_of<W>(my_piece, a.rotary_dim, inter);
        for (int t = my_t; t < t1; t += stride) {
            const T* x0 = static_cast<const T*>(a.q) + (row0 + t) * a.q_row + h0 * a.q_head;
            T* y0 = static_cast<T*>(a.q_out) + (row0 + t) * a.qo_row + h0 * a.qo_head;
            Raw<T, W> lo[kQHeads], hi[kQHeads];
#pragma unroll
            for (int h = 0; h < kQHeads; ++h)
                if (h < heads) {
                    lo[h] = load_raw<T, W>(x0 + h * a.q_head + p.at);
                    hi[h] = load_raw<T, W>(x0 + h * a.q_head + p.at2);
                }
            float c[W], s[W];
            if (p.angle >= 0) {
                const float* cs = a.rotary + (long long)t * a.rotary_dim + p.angle;
                load_angles<W>(cs, c);
                load_angles<W>(cs + half, s);
            }
#pragma unroll
            for (int h = 0; h < kQHeads; ++h)
                if (h < heads) {
                    float x[2 * W];
                    unpack<T, W>(lo[h], x);
                    unpack<T, W>(hi[h], x + W);
                    if (p.angle >= 0) {
                        if (inter) rotate<W>(x, c, s, true);
                        else rotate<W>(x, c, s, false);
                    }
                    store_values<T, W>(y0 + h * a.qo_head + p.at, x);
                    store_values<T, W>(y0 + h * a.qo_head + p.at2, x + W);
                }
        }
        if (clears) {
            const paged::Sequence before = paged::sequence(B, b);
            clear_rows(static_cast<T*>(a.q_out) + before.row0 * a.qo_row + h0 * a.qo_head, a.qo_row * sizeof(T), a.qo_head * sizeof(T),
                       min(before.n, -before.first), heads, B.dim * sizeof(T) / 16);
        }
        return;
    }
    const int page = paged::page_of(B, b, block);
    if (page < 0) return;
    const bool keys = int(blockIdx.y) < B.kv_heads;
    const int h = keys ? blockIdx.y : blockIdx.y - B.kv_heads;
    const T* x0 = static_cast<const T*>(keys ? a.k : a.v) + h * (keys ? a.k_head : a.v_head);
    const long long x_row = keys ? a.k_row : a.v_row;
    unsigned char* out = (keys ? B.k_cache : B.v_cache) + page * B.page_stride + h * B.head_stride;
    float* scale = (keys ? B.k_scale : B.v_scale) + (long long)page * B.kv_heads + h;
    const int rotary_dim = keys ? a.rotary_dim : 0, slot0 = t0 & (page_tokens - 1);
    const Piece p = piece_of<W>(my_piece, rotary_dim, inter);

    constexpr int kHold = kHoldValues / (2 * W);
    float x[kHold][2 * W], top = 0.f;
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
        const int t = my_t + u * stride;
        if (t < t1) load_piece<T, W>(x0 + (row0 + t) * x_row, p, a.rotary + (long long)t * rotary_dim, half, inter, x[u]);
    }
#pragma unroll
    for (int u = 0; u < kHold; ++u)
        if (my_t + u * stride < t1) {
#pragma unroll
            for (int l = 0; l < 2 * W; ++l) top = fmaxf(top, finite_abs(x[u][l]));
        }
    for (int t = my_t + kHold * stride; t < t1; t += stride) {    // pages of more than the registers hold
        float z[2 * W];
        load_piece<T, W>(x0 + (row0 + t) * x_row, p, a.rotary + (long long)t * rotary_dim, half, inter, z);
#pragma unroll
        for (int l = 0; l < 2 * W; ++l) top = fmaxf(top, finite_abs(z[l]));
    }
#pragma unroll
    for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const float old = slot0 > 0 ? *scale : 0.f;                  // read by every thread before one of them writes it
    if (blockDim.x > 32) {
        if ((tid & 31) == 0) warp_max[tid / 32] = top;
        __syncthreads();
        for (int w = 0; w < int(blockDim.x) / 32; ++w) top = fmaxf(top, warp_max[w]);
    } else {
        __syncwarp();
    }
    const float now = fmaxf(old, top > 0.f ? scale_for(top) : 0.f);      // 0: nothing but zeros so far (and infinities and NaN)
    const float inverse = now > 0.f ? 1.f / now : 1.f;           // a power of two: exact

    auto store = [&](int t, const float (&z)[2 * W]) {
        unsigned char* y = out + (long long)(t & (page_tokens - 1)) * B.token_stride;
        uint32_t w[W / 2];
#pragma unroll
        for (int l = 0; l < W / 2; ++l)
            w[l] = paged::e4m3x2(z[4 * l] * inverse, z[4 * l + 1] * inverse) | paged::e4m3x2(z[4 * l + 2] * inverse, z[4 * l + 3] * inverse) << 16;
        if constexpr (W == 8) {
            *reinterpret_cast<uint2*>(y + p.at) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2*>(y + p.at2) = make_uint2(w[2], w[3]);
        } else {
            *reinterpret_cast<uint32_t*>(y + p.at) = w[0];
            *reinterpret_cast<uint32_t*>(y + p.at2) = w[1];
        }
    };
#pragma unroll
    for (int u = 0; u < kHold; ++u)
        if (my_t + u * stride < t1) store(my_t + u * stride, x[u]);
    for (int t = my_t + kHold * stride; t < t1; t += stride) {
        float z[2 * W];
        load_piece<T, W>(x0 + (row0 + t) * x_row, p, a.rotary + (long long)t * rotary_dim, half, inter, z);
        store(t, z);
    }
    if (slot0 > 0 && 0.f < old && old < now) {                   // what the page has already moves to the new scale (under 0 it has no size)
        const float ratio = old * inverse;
        const int words = B.dim / 4, slots = page_tokens - (t1 - t0);
        for (int i = tid; i < slots * words; i += blockDim.x) {
            int slot = i / words;
            if (slot >= slot0) slot += t1 - t0;
            uint32_t* w = reinterpret_cast<uint32_t*>(out + (long long)slot * B.token_stride) + i % words;
            const uint32_t v = *w, l2 = paged::e4m3x2_to_half2(uint16_t(v)), h2 = paged::e4m3x2_to_half2(uint16_t(v >> 16));
            const float2 fl = __half22float2(*reinterpret_cast<const __half2*>(&l2)), fh = __half22float2(*reinterpret_cast<const __half2*>(&h2));
            *w = paged::e4m3x2(fl.x * ratio, fl.y * ratio) | paged::e4m3x2(fh.x * ratio, fh.y * ratio) << 16;
        }
    }
    if (tid == 0 && (slot0 == 0 || old != now)) *scale = now;
}

}  // namespace
}  // namespace ogle

using namespace ogle;

extern "C" int ogle_cuda_kv_append(const OglePagedBatch* batch, const OgleAppendParams* p, ogle_stream_t stream) {
    AppendArgs a = {};
    int rc = paged::translate(batch, a.b);
    if (rc != OGLE_OK) return rc;
    if (!p) return OGLE_ERR_INVALID;
    if (p->rotary && (p->rotary_dim < 8 || p->rotary_dim % 8 != 0 || p->rotary_dim > batch->head_dim || p->rotary_rows < batch->max_kv_len))
        return OGLE_ERR_INVALID;
    if (!aligned16(p->rotary)) return OGLE_ERR_ALIGNMENT;
    if (p->q && !p->q_out) return OGLE_ERR_INVALID;
    if (a.b.n_seqs == 0) return OGLE_OK;
    if (!p->k || !p->v) return OGLE_ERR_INVALID;
    const int dt = batch->dtype;
    if (!paged::strides_ok(p->k, p->k_row, p->k_head, dt) || !paged::strides_ok(p->v, p->v_row, p->v_head, dt) ||
        !paged::strides_ok(p->q, p->q_row, p->q_head, dt) || !paged::strides_ok(p->q_out, p->q_out_row, p->q_out_head, dt))
        return OGLE_ERR_ALIGNMENT;
    const Batch& B = a.b;
    if (B.max_rows == 0 || B.max_kv_len == 0) return OGLE_OK;
    a.k = p->k; a.v = p->v; a.q = p->q; a.q_out = p->q_out;
    a.k_row = p->k_row; a.k_head = p->k_head; a.v_row = p->v_row; a.v_head = p->v_head;
    a.q_row = p->q_row; a.q_head = p->q_head; a.qo_row = p->q_out_row; a.qo_head = p->q_out_head;
    a.rotary = p->rotary;
    a.rotary_dim = p->rotary ? p->rotary_dim : 0;
    a.interleaved = p->interleaved;
    a.q_blocks = p->q ? div_up(B.q_heads, kQHeads) : 0;
    // pages appended to: at most one a row, and at most two that it shares with what a sequence has already or will have
    long pages = B.max_rows == 1 ? B.n_seqs : (long)(B.n_rows >> B.page_shift) + 2L * B.n_seqs;
    if (B.max_rows > 1 && pages > B.n_rows) pages = B.n_rows;
    const int tokens = B.max_rows < (1 << B.page_shift) ? B.max_rows : 1 << B.page_shift;
    // 16 bytes of 16-bit values at a time where the rotated part is whole pieces of that (the 26000 rows: 221 us so, 338 by 8 bytes, when
    // both had their first form)
    const bool wide = dt != OGLE_F32 && a.rotary_dim % 16 == 0;
    const int pieces = B.dim / (wide ? 16 : 8), hold = kHoldValues / (wide ? 16 : 8);
    int threads = (div_up(tokens, hold) * pieces + 31) / 32 * 32;
    if (threads > kMaxThreads) threads = kMaxThreads;
    const dim3 grid((unsigned)pages, unsigned(2 * B.kv_heads + a.q_blocks));
    const auto run = [&](auto kernel) { return launch_overlapped(kernel, grid, dim3(threads), 0, stream, a); };
    cudaError_t e;
    if (dt == OGLE_F32) e = run(paged_append_kernel<float, 4>);
    else if (dt == OGLE_F16) e = wide ? run(paged_append_kernel<__half, 8>) : run(paged_append_kernel<__half, 4>);
    else e = wide ? run(paged_append_kernel<__nv_bfloat16, 8>) : run(paged_append_kernel<__nv_bfloat16, 4>);
    if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
    return finish_launch();
}
