// Logits before a token is chosen: repeated-token penalties, sparse biases, grammar masks, in one pass.
//
// A block has a slice of one row's vocabulary. It counts the row's tokens that fall into its slice in shared memory (whole
// numbers: their order does not matter) and notes for each the last bias named for it; then every logit is read and written
// once, 16 bytes at a time where the row's address allows it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ogle {
namespace {

constexpr int kThreads = 256;
constexpr unsigned kSeen = 0x80000000u;          // the token is in the prompt; the other bits count it behind it

struct LogitsArgs { OgleLogitsParams p; };

template <typename T> struct Vec { static constexpr int kN = 16 / sizeof(T); };

template <typename T>
__device__ __forceinline__ float as_float(T v) { return float(v); }

template <typename To, int N>
__device__ __forceinline__ void store_vec(To* p, const float (&x)[N]) {
    constexpr int kWords = N * sizeof(To) / 4;
    uint32_t w[kWords];
    To* h = reinterpret_cast<To*>(w);
#pragma unroll
    for (int l = 0; l < N; ++l) h[l] = To(x[l]);
#pragma unroll
    for (int q = 0; q < kWords; q += 4) *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + q) = make_uint4(w[q], w[q + 1], w[q + 2], w[q + 3]);
}

struct RowTerms { float repetition, presence, frequency; };

__device__ __forceinline__ float adjusted(float x, unsigned count, int bias, const float* bias_value, bool allowed, const RowTerms& t) {
    if (count) {
        x = x > 0.f ? __fdiv_rn(x, t.repetition) : __fmul_rn(x, t.repetition);
        const unsigned n = count & ~kSeen;
        if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(t.frequency, float(n))), t.presence);
    }
    if (bias) x = __fadd_rn(x, __ldg(bias_value + bias - 1));
    return allowed ? x : -INFINITY;
}

// U: vectors of 16 bytes a thread has of the slice; they are on their way while the tokens are counted.
template <typename Ti, typename To, int U>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(LogitsArgs a) {
    constexpr int N = Vec<Ti>::kN, kSlice = kThreads * N * U;
    extern __shared__ __align__(16) unsigned counts[];           // [kSlice], and as many last biases behind them
    const OgleLogitsParams& p = a.p;
    const int r = blockIdx.y, tid = threadIdx.x;
    const Ti* in = static_cast<const Ti*>(p.logits) + r * p.logits_stride;
    To* out = static_cast<To*>(p.out) + r * p.out_stride;
    // the row begins `shift` elements behind a 16-byte boundary; a slice is whole vectors between such boundaries
    const int shift = int(reinterpret_cast<uintptr_t>(in) / sizeof(Ti)) & (N - 1);
    const bool vectors = (reinterpret_cast<uintptr_t>(in) % sizeof(Ti)) == 0 && ((reinterpret_cast<uintptr_t>(out) - shift * sizeof(To)) & 15) == 0;
    const int s0 = blockIdx.x * kSlice - shift, s1 = min(s0 + kSlice, p.vocab), first = max(s0, 0);
    if (first >= s1) return;
    unsigned* const last_bias = counts + kSlice;
    const bool biased = p.bias_token != nullptr;
    grid_dependency_trigger();
    grid_dependency_wait();
    uint4 v[U];
    if (vectors) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = s0 + (u * kThreads + tid) * N;
            if (t >= 0 && t + N <= p.vocab) v[u] = *reinterpret_cast<const uint4*>(in + t);
        }
    }
    const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < N * U / 4; ++i) {
        reinterpret_cast<uint4*>(counts)[i * kThreads + tid] = none;
        if (biased) reinterpret_cast<uint4*>(last_bias)[i * kThreads + tid] = none;
    }
    __syncthreads();
    const unsigned width = s1 - first, at0 = first - s0;
    if (p.tokens) {
        const int t0 = max(p.token_start[r], 0), n = min(p.token_start[r + 1], p.n_tokens) - t0, prompt = p.prompt_len ? p.prompt_len[r] : 0;
        const int* tokens = p.tokens + t0;
#pragma unroll 4
        for (int i = tid; i < n; i += kThreads) {
            const unsigned t = unsigned(__ldg(tokens + i) - first);
            if (t < width) {
                if (i < prompt) atomicOr(&counts[t + at0], kSeen);
                else atomicAdd(&counts[t + at0], 1u);
            }
        }
    }
    const int bias0 = biased ? max(p.bias_start[r], 0) : 0;
    if (biased) {
        const int n = min(p.bias_start[r + 1], p.n_biases) - bias0;
        for (int i = tid; i < n; i += kThreads) {
            const unsigned t = unsigned(__ldg(p.bias_token + bias0 + i) - first);
            if (t < width) atomicMax(&last_bias[t + at0], unsigned(i + 1));
        }
    }
    const float* bias_value = biased ? p.bias_value + bias0 : nullptr;
    const RowTerms terms = {p.repetition ? p.repetition[r] : 1.f, p.presence ? p.presence[r] : 0.f, p.frequency ? p.frequency[r] : 0.f};
    const unsigned* allowed = p.allowed ? p.allowed + r * p.allowed_stride : nullptr;
    __syncthreads();
    const auto one = [&](int t) {
        const bool ok = !allowed || (__ldg(allowed + t / 32) >> (t % 32) & 1);
        out[t] = To(adjusted(as_float(in[t]), counts[t - s0], biased ? int(last_bias[t - s0]) : 0, bias_value, ok, terms));
    };
    if (!vectors) {
        for (int t = first + tid; t < s1; t += kThreads) one(t);
        return;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = s0 + (u * kThreads + tid) * N;
        if (t >= s1) continue;
        if (t < 0 || t + N > p.vocab) {          // a vector that hangs over an end of the row
            for (int l = 0; l < N; ++l)
                if (t + l >= 0 && t + l < s1) one(t + l);
            continue;
        }
        const Ti* h = reinterpret_cast<const Ti*>(&v[u]);
        unsigned bits = ~0u;
        if (allowed) {
            const int w = t / 32, s = t % 32;
            bits = __ldg(allowed + w) >> s;
            if (s + N > 32) bits |= __ldg(allowed + w + 1) << (32 - s);
        }
        float x[N];
        unsigned c[N], any = 0;
#pragma unroll
        for (int l = 0; l < N; ++l) x[l] = as_float(h[l]);
#pragma unroll
        for (int l = 0; l < N; l += 4) {
            const uint4 q = *reinterpret_cast<const uint4*>(counts + t - s0 + l);
            c[l] = q.x; c[l + 1] = q.y; c[l + 2] = q.z; c[l + 3] = q.w;
            any |= q.x | q.y | q.z | q.w;
        }
        // most vectors have no token of the text and no bias
        if (any) {
#pragma unroll
            for (int l = 0; l < N; ++l) x[l] = adjusted(x[l], c[l], 0, nullptr, true, terms);
        }
        if (biased) {
#pragma unroll
            for (int l = 0; l < N; l += 4) {
                const uint4 q = *reinterpret_cast<const uint4*>(last_bias + t - s0 + l);
                if (q.x | q.y | q.z | q.w) {
                    const unsigned i[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) if (i[k]) x[l + k] = __fadd_rn(x[l + k], __ldg(bias_value + i[k] - 1));
                }
            }
        }
#pragma unroll
        for (int l = 0; l < N; ++l) x[l] = bits >> l & 1 ? x[l] : -INFINITY;
        store_vec<To, N>(out + t, x);
    }
}

template <typename Ti, typename To, int U>
cudaError_t launch(const LogitsArgs& a, cudaStream_t s) {
    constexpr int kSlice = kThreads * Vec<Ti>::kN * U;
    const size_t smem = size_t(kSlice) * 4 * (a.p.bias_token ? 2 : 1);
    auto kernel = adjust_logits_kernel<Ti, To, U>;
    if (smem > 48 * 1024) {
        static std::atomic<uint64_t> sized{0};                   // devices whose limit of shared memory is raised
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return e;
        if (!(sized.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlice * 8);
            if (e != cudaSuccess) return e;
            sized.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
        }
    }
    return launch_overlapped(kernel, dim3(div_up(a.p.vocab + Vec<Ti>::kN - 1, kSlice), a.p.rows), dim3(kThreads), smem, s, a);
}

template <typename Ti, typename To>
cudaError_t launch(const LogitsArgs& a, cudaStream_t s) {
    // Slices of four vectors a thread, which count the row's tokens a quarter as often, where they still fill the GPU.
    const long blocks = (long)div_up(a.p.vocab, kThreads * Vec<Ti>::kN * 4) * a.p.rows;
    return blocks >= 2 * kNumSMs ? launch<Ti, To, 4>(a, s) : launch<Ti, To, 1>(a, s);
}

}  // namespace
}  // namespace ogle

using namespace ogle;

extern "C" int ogle_cuda_adjust_logits(const OgleLogitsParams* p, ogle_stream_t stream) {
    if (!p || p->rows < 0 || p->vocab < 0 || p->n_tokens < 0 || p->n_biases < 0 || p->dtype < OGLE_F32 || p->dtype > OGLE_BF16) return OGLE_ERR_INVALID;
    if (p->out_dtype != p->dtype && p->out_dtype != OGLE_F32) return OGLE_ERR_INVALID;
    if (p->rows == 0 || p->vocab == 0) return OGLE_OK;
    if (p->rows > 65535 || p->vocab > (1 << 30)) return OGLE_ERR_UNSUPPORTED;
    if (!p->logits || !p->out || (p->tokens && !p->token_start) || (p->bias_token && (!p->bias_value || !p->bias_start))) return OGLE_ERR_INVALID;
    if (p->logits_stride < p->vocab || p->out_stride < p->vocab || (p->allowed && p->allowed_stride != 0 && p->allowed_stride < (p->vocab + 31) / 32)) return OGLE_ERR_INVALID;
    if (p->out == p->logits && (p->out_dtype != p->dtype || p->out_stride != p->logits_stride)) return OGLE_ERR_INVALID;
    const LogitsArgs a = {*p};
    cudaError_t e;
    if (p->dtype == OGLE_F32) e = launch<float, float>(a, stream);
    else if (p->dtype == OGLE_F16) e = p->out_dtype == OGLE_F16 ? launch<__half, __half>(a, stream) : launch<__half, float>(a, stream);
    else e = p->out_dtype == OGLE_BF16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, stream) : launch<__nv_bfloat16, float>(a, stream);
    if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
    return finish_launch();
}
