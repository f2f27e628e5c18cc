// What the model itself gave a token: out[r] = (l_t - max l) - log sum_i exp(l_i - max l) over row r of float32 logits, t the
// row's token.  The logits are read once: every thread keeps the largest logit it has seen and the sum of exponentials relative
// to it, and rescales the sum when a larger one comes (once in 16 numbers at most); pairs are joined the same way.  Many rows have
// a workgroup each; a row of few is cut in parts, whose pairs a second launch joins in order.  A token outside the vocabulary
// gives NaN, a row of -inf alone or with a +inf or a NaN gives NaN, as the formula does.
//
// What bounds it is the reading: 2,048 rows of 151,936 take 210 us, 5.9 TB/s (a plain reading of 1 GiB 5.6).  8 rows take 7 us for
// 4.9 MB, two launches' latency; a workgroup for each whole row takes 31.
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kTurn = kThreads * 16;  // numbers that a workgroup takes at a time: a thread four times four neighbours
constexpr float kLog2E = 1.44269504088896340736f;

struct Tally {
    float best, sum;  // the largest so far, and the sum of exp(l - best)
};

// (the product's rounding is off by x 2^-24 of the term, and x e^x is at most 0.37: less than the sum's own rounding)
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2E); }

__device__ __forceinline__ Tally joined(Tally a, Tally b) {
    if (b.best > a.best) {
        const Tally c = a;
        a = b;
        b = c;
    }
    a.sum += b.best == -INFINITY ? b.sum : b.sum * exp_of(b.best - a.best);  // (nothing there but -inf, or NaN in the sum)
    return a;
}

__device__ __forceinline__ Tally joined_wave(Tally t) {
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1)
        t = joined(t, Tally{__shfl_xor(t.best, offset, kWave), __shfl_xor(t.sum, offset, kWave)});
    return t;
}

__device__ __forceinline__ void finish(Tally t, const float* row, int token, int vocab, float* out) {
    const bool known = token >= 0 && token < vocab && t.best < INFINITY;
    *out = known ? (row[token] - t.best) - logf(t.sum) : NAN;
}

// grid: (parts, rows).  One part: the row is finished here.
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, Tally* __restrict__ tallies,
                      float* __restrict__ out, int vocab, long ld, int part) {
    __shared__ Tally s[kThreads / kWave];
    const int r = blockIdx.y, end = min(vocab, (static_cast<int>(blockIdx.x) + 1) * part);
    const float* row = logits + static_cast<size_t>(r) * ld;
    const bool lines = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    Tally t = {-INFINITY, 0.f};
    for (int begin = blockIdx.x * part; begin < end; begin += kTurn) {
        float l[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = begin + (q * kThreads + threadIdx.x) * 4;
            if (lines && at + 3 < end) {
                const float4 v = *reinterpret_cast<const float4*>(row + at);
                l[q * 4] = v.x;
                l[q * 4 + 1] = v.y;
                l[q * 4 + 2] = v.z;
                l[q * 4 + 3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) l[q * 4 + e] = at + e < end ? row[at + e] : -INFINITY;
            }
        }
        float most = l[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, l[i]);
        if (most > t.best) {
            t.sum = t.best == -INFINITY ? t.sum : t.sum * exp_of(t.best - most);
            t.best = most;
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += l[i] == -INFINITY ? 0.f : exp_of(l[i] - t.best);  // (a NaN stays one)
        t.sum += sum;
    }
    t = joined_wave(t);
    if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = t;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < kThreads / kWave; ++w) t = joined(t, s[w]);
    if (gridDim.x == 1)
        finish(t, row, tokens[r], vocab, out + r);
    else
        tallies[static_cast<size_t>(r) * gridDim.x + blockIdx.x] = t;
}

// One wave a row.
__global__ void __launch_bounds__(kWave)
token_logprobs_join_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, const Tally* __restrict__ tallies,
                           float* __restrict__ out, int vocab, long ld, int parts) {
    const int r = blockIdx.x;
    Tally t = {-INFINITY, 0.f};
    for (int p = threadIdx.x; p < parts; p += kWave) t = joined(t, tallies[static_cast<size_t>(r) * parts + p]);
    t = joined_wave(t);
    if (threadIdx.x == 0) finish(t, logits + static_cast<size_t>(r) * ld, tokens[r], vocab, out + r);
}

}  // namespace

// part: numbers of a row that a workgroup takes, a multiple of 4,096; tallies: rows * ceil(vocab / part) * 8 bytes, none for one part.
CIE_API int cie_token_logprobs(void* stream, const float* logits, const int* tokens, float* tallies, float* out, int rows, int vocab,
                               long ld, int part) {
    if (rows < 0 || rows > 65535 || vocab <= 0 || vocab > (1 << 30) || ld < vocab || part <= 0 || part % kTurn || part > (1 << 30) ||
        !logits || !tokens || !out || (part < vocab && !tallies))
        return CIE_BAD_ARGUMENT;
    if (rows == 0) return CIE_OK;
    const int parts = (vocab + part - 1) / part;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Tally* const kept = reinterpret_cast<Tally*>(tallies);
    token_logprobs_kernel<<<dim3(parts, rows), kThreads, 0, s>>>(logits, tokens, kept, out, vocab, ld, part);
    if (parts == 1 || cie_after_launch() != CIE_OK) return parts == 1 ? cie_after_launch() : CIE_LAUNCH_FAILED;
    token_logprobs_join_kernel<<<rows, kWave, 0, s>>>(logits, tokens, kept, out, vocab, ld, parts);
    return cie_after_launch();
}
