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

struct LogitsArgs {
    OgleLogitsParams p;
    int slice;                                   // tokens of a block
};

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

template <typename Ti, typename To>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(LogitsArgs a) {
    constexpr int N = Vec<Ti>::kN;
    extern __shared__ __align__(16) unsigned counts[];           // [slice + N], and as many last biases behind them
    const OgleLogitsParams& p = a.p;
    const int r = blockIdx.y, tid = threadIdx.x;
    const Ti* in = static_cast<const Ti*>(p.logits) + r * p.logits_stride;
    To* out = static_cast<To*>(p.out) + r * p.out_stride;
    // the row begins `shift` elements behind a 16-byte boundary; a slice is whole vectors between such boundaries
    const int shift = int(reinterpret_cast<uintptr_t>(in) / sizeof(Ti)) & (N - 1);
    const bool vectors = (reinterpret_cast<uintptr_t>(in) % sizeof(Ti)) == 0 && ((reinterpret_cast<uintptr_t>(out) - shift * sizeof(To)) & 15) == 0;
    const int s0 = blockIdx.x * a.slice - shift, s1 = min(s0 + a.slice, p.vocab), first = max(s0, 0);
    if (first >= s1) return;
    unsigned* const last_bias = counts + a.slice;
    const int used = s1 - s0;
    grid_dependency_trigger();
    grid_dependency_wait();
    for (int i = tid; i < used; i += kThreads) counts[i] = 0;
    const bool biased = p.bias_token != nullptr;
    if (biased) for (int i = tid; i < used; i += kThreads) last_bias[i] = 0;
    __syncthreads();
    if (p.tokens) {
        const int t0 = max(p.token_start[r], 0), n = min(p.token_start[r + 1], p.n_tokens) - t0, prompt = p.prompt_len ? p.prompt_len[r] : 0;
        for (int i = tid; i < n; i += kThreads) {
            const int t = p.tokens[t0 + i];
            if (t < first || t >= s1) continue;
            if (i < prompt) atomicOr(&counts[t - s0], kSeen);
            else atomicAdd(&counts[t - s0], 1u);
        }
    }
    const int bias0 = biased ? max(p.bias_start[r], 0) : 0;
    if (biased) {
        const int t0 = bias0, n = min(p.bias_start[r + 1], p.n_biases) - t0;
        for (int i = tid; i < n; i += kThreads) {
            const int t = p.bias_token[t0 + i];
            if (t >= first && t < s1) atomicMax(&last_bias[t - s0], unsigned(i + 1));
        }
    }
    __syncthreads();
    const float* bias_value = biased ? p.bias_value + bias0 : nullptr;
    const RowTerms terms = {p.repetition ? p.repetition[r] : 1.f, p.presence ? p.presence[r] : 0.f, p.frequency ? p.frequency[r] : 0.f};
    const unsigned* allowed = p.allowed ? p.allowed + r * p.allowed_stride : nullptr;
    const auto one = [&](int t) {
        const bool ok = !allowed || (__ldg(allowed + t / 32) >> (t % 32) & 1);
        out[t] = To(adjusted(as_float(in[t]), counts[t - s0], biased ? int(last_bias[t - s0]) : 0, bias_value, ok, terms));
    };
    if (!vectors) {
        for (int t = first + tid; t < s1; t += kThreads) one(t);
        return;
    }
    for (int t = s0 + tid * N; t < s1; t += kThreads * N) {
        if (t < 0 || t + N > p.vocab) {          // a vector that hangs over an end of the row
            for (int l = 0; l < N; ++l)
                if (t + l >= 0 && t + l < s1) one(t + l);
            continue;
        }
        const uint4 v = *reinterpret_cast<const uint4*>(in + t);
        const Ti* h = reinterpret_cast<const Ti*>(&v);
        unsigned bits = ~0u;
        if (allowed) {
            const int w = t / 32, s = t % 32;
            bits = __ldg(allowed + w) >> s;
            if (s + N > 32) bits |= __ldg(allowed + w + 1) << (32 - s);
        }
        float x[N];
#pragma unroll
        for (int l = 0; l < N; ++l)
            x[l] = adjusted(as_float(h[l]), counts[t - s0 + l], biased ? int(last_bias[t - s0 + l]) : 0, bias_value, bits >> l & 1, terms);
        store_vec<To, N>(out + t, x);
    }
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
    LogitsArgs a = {*p, 0};
    a.slice = 4096;
    const size_t smem = size_t(a.slice) * 4 * (p->bias_token ? 2 : 1);
    const dim3 grid(div_up(p->vocab + 7, a.slice), p->rows);
    cudaError_t e;
    if (p->dtype == OGLE_F32) e = launch_overlapped(adjust_logits_kernel<float, float>, grid, dim3(kThreads), smem, stream, a);
    else if (p->dtype == OGLE_F16) e = launch_overlapped(p->out_dtype == OGLE_F16 ? adjust_logits_kernel<__half, __half> : adjust_logits_kernel<__half, float>, grid, dim3(kThreads), smem, stream, a);
    else e = launch_overlapped(p->out_dtype == OGLE_BF16 ? adjust_logits_kernel<__nv_bfloat16, __nv_bfloat16> : adjust_logits_kernel<__nv_bfloat16, float>, grid, dim3(kThreads), smem, stream, a);
    if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
    return finish_launch();
}
