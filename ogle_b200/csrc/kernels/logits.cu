// Logits before a token is chosen: repeated-token penalties, sparse biases, grammar masks, in one pass.
//
// A block has a range of one row's vocabulary. It writes every logit, masked, once - 16 bytes at a time where the row's address
// allows it - and mends those that a token of the text or a bias names: tokens are counted in shared memory (whole numbers:
// their order does not matter), the last bias named for a token is noted beside its count, and each such logit is computed
// anew. A row has some hundred of them, not worth a look-up for each of the others (which took 17 of 25 instructions a logit:
// 400 x 150000 93 us). Few tokens and biases go into a hash table at once; where they turn out to be too many for it, they are counted
// slice by slice of the range.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ogle {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 8192;                     // words of shared memory
constexpr int kEntries = kSlice / 2, kMostHashed = kEntries * 3 / 4;      // of the table: a token and its word each
constexpr int kText = 2048;                      // tokens of the text that are kept in shared memory
constexpr unsigned kEmpty = ~0u;
// A token's word in shared memory: how often it is behind the prompt (17 bits), the last bias named for it (13 bits, 0: none),
// whether it is in the prompt. Rows with more tokens or biases than that go through half a slice at a time, with 31 bits to count
// and a table of their own for biases.
constexpr unsigned kSeen = 0x80000000u;
constexpr int kBiasShift = 17;
constexpr int kMaxTokens = (1 << kBiasShift) - 1, kMaxBiases = (1 << 13) - 1;

struct LogitsArgs {
    OgleLogitsParams p;
    int range;                                   // tokens of a block
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

// word: kSeen and the count alone; bias: the last one's number + 1, or 0.
__device__ __forceinline__ float adjusted(float x, unsigned word, unsigned bias, const float* bias_value, const RowTerms& t) {
    if (word) {
        x = x > 0.f ? __fdiv_rn(x, t.repetition) : __fmul_rn(x, t.repetition);
        const unsigned n = word & ~kSeen;
        if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(t.frequency, float(n))), t.presence);
    }
    return bias ? __fadd_rn(x, __ldg(bias_value + bias - 1)) : x;
}

// (Loops over tokens are not unrolled: they run once in a block's life, and fetching their instructions took longer than what they do - one
// row of 32000: 16 us with all of them unrolled, 7 so.)
template <typename Ti, typename To>
__global__ void __launch_bounds__(kThreads, 4) adjust_logits_kernel(LogitsArgs a) {
    constexpr int N = Vec<Ti>::kN, U = 4;
    __shared__ __align__(16) unsigned words[kSlice];
    __shared__ int text[kText];
    __shared__ uint16_t taken[kMostHashed];
    __shared__ int n_taken;
    const OgleLogitsParams& p = a.p;
    const int r = blockIdx.y, tid = threadIdx.x;
    const Ti* in = static_cast<const Ti*>(p.logits) + r * p.logits_stride;
    To* out = static_cast<To*>(p.out) + r * p.out_stride;
    // the row begins `shift` elements behind a 16-byte boundary; a range is whole vectors between such boundaries
    const int shift = int(reinterpret_cast<uintptr_t>(in) / sizeof(Ti)) & (N - 1);
    const bool vectors = (reinterpret_cast<uintptr_t>(in) % sizeof(Ti)) == 0 && ((reinterpret_cast<uintptr_t>(out) - shift * sizeof(To)) & 15) == 0;
    const int begin = blockIdx.x * a.range - shift, end = min(begin + a.range, p.vocab), first = max(begin, 0);
    grid_dependency_trigger();
    grid_dependency_wait();
    // The grid has pieces for the row that begins farthest behind its boundary: of another row the last block may be past the vocabulary.
    if (begin >= end) return;
    const unsigned* allowed = p.allowed ? p.allowed + r * p.allowed_stride : nullptr;
    const int last_word = (p.vocab - 1) / 32;
    const int token0 = p.tokens ? max(p.token_start[r], 0) : 0, n_tokens = p.tokens ? min(p.token_start[r + 1], p.n_tokens) - token0 : 0;
    const int bias0 = p.bias_token ? max(p.bias_start[r], 0) : 0, n_biases = p.bias_token ? min(p.bias_start[r + 1], p.n_biases) - bias0 : 0;
    const bool named = n_tokens > 0 || n_biases > 0;
    if (named) {
#pragma unroll 4
        for (int i = tid; i < min(n_tokens, kText); i += kThreads) text[i] = __ldg(p.tokens + token0 + i);
        if (tid == 0) n_taken = 0;
    }
    const auto allows = [&](int t) { return !allowed || (__ldg(allowed + t / 32) >> (t % 32) & 1); };

    // every logit, masked (before the counting: where all blocks counted first, the memory had nothing to do meanwhile - 400 x 150000
    // 80 us, 57 so)
    int edge = first, edge_end = end;            // what is not whole vectors
    if (vectors) {
        for (int t0 = begin + tid * N; t0 < end; t0 += U * kThreads * N) {
            uint4 v[U];
            unsigned bits[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = t0 + u * kThreads * N;
                if (t >= 0 && t + N <= end) v[u] = *reinterpret_cast<const uint4*>(in + t);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {        // two words whether or not the bits lie in both: no branch between the loads
                const int t = min(max(t0 + u * kThreads * N, 0), p.vocab - 1), w = t / 32;
                bits[u] = allowed ? __funnelshift_r(__ldg(allowed + w), __ldg(allowed + min(w + 1, last_word)), t) : ~0u;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = t0 + u * kThreads * N;
                if (t >= 0 && t + N <= end) {
                    const Ti* h = reinterpret_cast<const Ti*>(&v[u]);
                    float x[N];
#pragma unroll
                    for (int l = 0; l < N; ++l) x[l] = bits[u] >> l & 1 ? as_float(h[l]) : -INFINITY;
                    store_vec<To, N>(out + t, x);
                }
            }
        }
        edge_end = begin < 0 ? min(begin + N, end) : first;
    }
    for (int k = 0; k < 2; ++k) {                // its head, or all of it; its tail
        for (int t = edge + tid; t < edge_end; t += kThreads) out[t] = To(allows(t) ? as_float(in[t]) : -INFINITY);
        edge = vectors ? max(begin + (end - begin) / N * N, edge_end) : end;
        edge_end = end;
    }
    if (!named) return;

    const int prompt = p.tokens && p.prompt_len ? p.prompt_len[r] : 0;
    const float* bias_value = p.bias_value + bias0;
    const RowTerms terms = {p.repetition ? p.repetition[r] : 1.f, p.presence ? p.presence[r] : 0.f, p.frequency ? p.frequency[r] : 0.f};
    // f(number, token), for biases or for the text's tokens: those in [s0, s0 + width). (Collecting them first, until a warp's lanes have one
    // each, took 1 us from 64 x 128001 with texts of 4000 and added 3 to 400 x 150000, whose blocks have whole rows.)
    const auto each = [&](bool biases, int s0, unsigned width, auto f) {
        const int n = biases ? n_biases : n_tokens;
#pragma unroll 1
        for (int i = tid; i < n; i += kThreads) {
            const int token = biases ? __ldg(p.bias_token + bias0 + i) : (i < kText ? text[i] : __ldg(p.tokens + token0 + i));
            if (token >= 0 && unsigned(token - s0) < width) f(i, token);
        }
    };
    // (in place, `in` has the logit still: what the mask let through is as it was)
    const auto mend = [&](int token, unsigned word, unsigned bias) {
        const float x = as_float(in[token]);
        if (allows(token)) out[token] = To(adjusted(x, word, bias, bias_value, terms));
    };
    const bool is_long = n_tokens > kMaxTokens || n_biases > kMaxBiases;
    const unsigned range = end - first;
    unsigned* const keys = words + kEntries;

    // a hash table, where the text's tokens and biases that fall into the range are few
    for (int i = tid; i < kEntries / 4; i += kThreads) {
        reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(keys)[i] = make_uint4(kEmpty, kEmpty, kEmpty, kEmpty);
    }
    __syncthreads();                             // all logits of the range are written, too
    if (!is_long) {
        // Its place in the table. Three quarters of it are for use; where more tokens come than that, no thread begins another, and
        // what was in hand - one a thread - finds a place still.
        const auto entry = [&](int token) {
            unsigned h = unsigned(token) * 2654435761u >> 20;
            for (;;) {
                const unsigned k = atomicCAS(&keys[h], kEmpty, unsigned(token));
                if (k == kEmpty) {               // a warp's new entries go on the list together
                    const unsigned with = __activemask(), lane = tid & 31, leader = __ffs(with) - 1;
                    int at = 0;
                    if (lane == leader) at = atomicAdd(&n_taken, __popc(with));
                    at = __shfl_sync(with, at, leader);
                    at += __popc(with & ((1u << lane) - 1));
                    if (at < kMostHashed) taken[at] = uint16_t(h);
                }
                if (k == kEmpty || k == unsigned(token)) return h;
                h = (h + 1) & (kEntries - 1);
            }
        };
        static_assert(kEntries == 4096 && kMostHashed + kThreads < kEntries, "20 bits off a hash of 32");
        const auto full = [&] { return *static_cast<volatile int*>(&n_taken) > kMostHashed; };
        // biases first: a word then has nothing else, and its largest value is the last of them
        if (n_biases > 0) {
            each(true, first, range, [&](int i, int token) {
                if (!full()) atomicMax(&words[entry(token)], unsigned(i + 1) << kBiasShift);
            });
            __syncthreads();
        }
        each(false, first, range, [&](int i, int token) {
            if (full()) return;
            const unsigned h = entry(token);
            if (i < prompt) atomicOr(&words[h], kSeen);
            else atomicAdd(&words[h], 1u);
        });
        __syncthreads();
        if (n_taken <= kMostHashed) {
#pragma unroll 1
            for (int i = tid; i < n_taken; i += kThreads) {
                const unsigned h = taken[i], w = words[h];
                mend(int(keys[h]), w & (kSeen | kMaxTokens), w << 1 >> (kBiasShift + 1));
            }
            return;
        }
        for (int i = tid; i < kEntries / 4; i += kThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    }
    // a word for each token of a slice, or two: counts and biases
    const unsigned slice = is_long ? kSlice / 2 : kSlice, step = is_long ? 2 : 1;
    for (int i = tid; i < kEntries / 4; i += kThreads) reinterpret_cast<uint4*>(keys)[i] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
    for (int s0 = first; s0 < end; s0 += slice) {
        const unsigned width = min(int(slice), end - s0);
        __syncthreads();                         // the words are 0
        each(true, s0, width, [&](int i, int token) {
            atomicMax(&words[(token - s0) * step + step - 1], is_long ? unsigned(i + 1) : unsigned(i + 1) << kBiasShift);
        });
        if (!is_long) __syncthreads();
        each(false, s0, width, [&](int i, int token) {
            if (i < prompt) atomicOr(&words[(token - s0) * step], kSeen);
            else atomicAdd(&words[(token - s0) * step], 1u);
        });
        __syncthreads();
        for (int k = 0; k < 2; ++k)              // the first to take a token's word out has the token
            each(k, s0, width, [&](int, int token) {
                if (is_long) {
                    const unsigned long long w = atomicExch(reinterpret_cast<unsigned long long*>(words) + (token - s0), 0ull);
                    if (w) mend(token, unsigned(w), unsigned(w >> 32));
                } else {
                    const unsigned w = atomicExch(&words[token - s0], 0u);
                    if (w) mend(token, w & (kSeen | kMaxTokens), w << 1 >> (kBiasShift + 1));
                }
            });
    }
}

template <typename Ti, typename To>
cudaError_t launch(LogitsArgs a, cudaStream_t s) {
    constexpr int N = Vec<Ti>::kN, kPiece = kThreads * N;
    // A block's range: whole pieces of a vector a thread. As many blocks to a row as one round of them (four to an SM) has
    // for it; at least one for every 2000 tokens of a row's text, so that those of a range fit the hash table. (400 x 150000, a row a
    // block: 16 pieces a block 71 us, so 56. One for every 500 / 1000 / 2000 / 4000 / without, us: 400 x 150000, texts of up to 8000,
    // 194 / 226 / 283 / 397 / 610; 150 x 50000, 16000, 165 / 122 / 162 / 204 / 230; 64 x 128001, 40000, 346 / 357 / 326 / 417 / 417;
    // 592 x 32000, 2500, 54 / 50 / 48 / 48 / 48; 400 x 150000, 2000, 64 / 74 / 71 / 71 / 71.)
    const long pieces = div_up(a.p.vocab + N - 1, kPiece), text = div_up(long(a.p.n_tokens) + a.p.n_biases, a.p.rows);
    long blocks = 4L * kNumSMs / a.p.rows;
    if (blocks < div_up(text, 2000)) blocks = div_up(text, 2000);
    const long each = div_up(pieces, blocks > 1 ? blocks : 1);
    a.range = int(each * kPiece);
    return launch_overlapped(adjust_logits_kernel<Ti, To>, dim3(div_up(pieces, each), a.p.rows), dim3(kThreads), 0, s, a);
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
    const LogitsArgs a = {*p, 1};
    cudaError_t e;
    if (p->dtype == OGLE_F32) e = launch<float, float>(a, stream);
    else if (p->dtype == OGLE_F16) e = p->out_dtype == OGLE_F16 ? launch<__half, __half>(a, stream) : launch<__half, float>(a, stream);
    else e = p->out_dtype == OGLE_BF16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, stream) : launch<__nv_bfloat16, float>(a, stream);
    if (e != cudaSuccess) { set_last_error(e); (void)cudaGetLastError(); return OGLE_ERR_CUDA; }
    return finish_launch();
}
