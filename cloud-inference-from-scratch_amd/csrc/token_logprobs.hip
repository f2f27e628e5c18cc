// What the model itself gave a token: out[r] = (l_t - max l) - log sum_i exp(l_i - max l) over row r of float32 logits, t the
// row's token.  One pass: every thread keeps the largest logit it has seen and the sum of exponentials relative to it, and
// rescales the sum when a larger one comes; the threads' pairs are joined the same way.  A token outside the vocabulary gives
// NaN, a row of -inf alone or with a +inf or a NaN gives NaN, as the formula does.
#include "common.h"

namespace {

constexpr int kThreads = 256;

struct Tally {
    float best, sum;  // the largest so far, and the sum of exp(l - best)
};

__device__ __forceinline__ Tally joined(Tally a, Tally b) {
    if (b.best > a.best) {
        const Tally c = a;
        a = b;
        b = c;
    }
    if (b.best == -INFINITY) {  // (nothing seen there, or only -inf and NaN)
        a.sum += b.sum;
        return a;
    }
    a.sum += b.sum * expf(b.best - a.best);
    return a;
}

__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, float* __restrict__ out, int vocab, long ld) {
    __shared__ Tally s[kThreads / kWave];
    const float* row = logits + static_cast<size_t>(blockIdx.x) * ld;
    Tally t = {-INFINITY, 0.f};
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
        const float l = row[i];
        if (l > t.best) {
            t.sum = t.best == -INFINITY ? t.sum + 1.f : t.sum * expf(t.best - l) + 1.f;
            t.best = l;
        } else if (l != -INFINITY) {
            t.sum += expf(l - t.best);  // (a NaN stays one)
        }
    }
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1)
        t = joined(t, Tally{__shfl_xor(t.best, offset, kWave), __shfl_xor(t.sum, offset, kWave)});
    if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = t;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < kThreads / kWave; ++w) t = joined(t, s[w]);
    const int token = tokens[blockIdx.x];
    const bool known = token >= 0 && token < vocab && t.best < INFINITY;
    out[blockIdx.x] = known ? (row[token] - t.best) - logf(t.sum) : NAN;
}

}  // namespace

CIE_API int cie_token_logprobs(void* stream, const float* logits, const int* tokens, float* out, int rows, int vocab, long ld) {
    if (rows < 0 || vocab <= 0 || ld < vocab || !logits || !tokens || !out) return CIE_BAD_ARGUMENT;
    if (rows == 0) return CIE_OK;
    token_logprobs_kernel<<<rows, kThreads, 0, static_cast<hipStream_t>(stream)>>>(logits, tokens, out, vocab, ld);
    return cie_after_launch();
}
