// Low-rank adapters of many requests beside a shared projection:
//   out[t, c] = into[t, c] + scale[a] * sum_r up[a][c, r] * h[t, p(c) R + r],   h[t, j] = sum_k down[a][j, k] x[t, k],
// a = adapter[t]; a row whose adapter is none (negative, or one that there is not) keeps its numbers.  A site stacks P
// projections that read the same rows (q, k and v; gate and up): `down` [A, P R, K] has R rows for each, the columns of `out`
// fall into P pieces, and p(c) is the piece of column c.
//
// The sums are float32, the result is rounded once.
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPieces = 4;

struct Pieces {
    int count;
    int begin[kMaxPieces + 1];  // first column of each, and the end
};

// h[t, j], one wave a number.
template <typename T>
__global__ void __launch_bounds__(kThreads)
adapter_down_plain(const T* __restrict__ x, long ldx, const T* __restrict__ down, const int* __restrict__ adapter,
                   float* __restrict__ h, int rows, int inner, int k, int adapters) {
    const int j = blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave, t = blockIdx.y;
    const int a = adapter[t];
    if (j >= inner || a < 0 || a >= adapters) return;
    const T* row = x + static_cast<size_t>(t) * ldx;
    const T* w = down + (static_cast<size_t>(a) * inner + j) * k;
    float sum = 0.f;
    for (int i = threadIdx.x % kWave; i < k; i += kWave) sum += to_float(row[i]) * to_float(w[i]);
    sum = wave_sum(sum);
    if (threadIdx.x % kWave == 0) h[static_cast<size_t>(t) * inner + j] = sum;
}

template <typename T, typename S>
__global__ void __launch_bounds__(kThreads)
adapter_up_plain(const float* __restrict__ h, const T* __restrict__ up, const float* __restrict__ scale,
                 const int* __restrict__ adapter, const S* into, long ld_into, S* out, long ld_out, int rows, int inner, int n,
                 int rank, int adapters, Pieces pieces) {
    const int c = blockIdx.x * kThreads + threadIdx.x, t = blockIdx.y;
    if (c >= n) return;
    const S old = into[static_cast<size_t>(t) * ld_into + c];
    S* place = out + static_cast<size_t>(t) * ld_out + c;
    const int a = adapter[t];
    if (a < 0 || a >= adapters) {
        *place = old;
        return;
    }
    int p = 0;
    while (p + 1 < pieces.count && c >= pieces.begin[p + 1]) ++p;
    const float* row = h + static_cast<size_t>(t) * inner + p * rank;
    const T* w = up + (static_cast<size_t>(a) * n + c) * rank;
    float sum = 0.f;
    for (int r = 0; r < rank; ++r) sum += row[r] * to_float(w[r]);
    *place = from_float<S>(to_float(old) + scale[a] * sum);
}

template <typename T, typename S>
int run_plain(hipStream_t s, const void* x, long ldx, const void* down, const void* up, const float* scale, const int* adapter,
              const void* into, long ld_into, void* out, long ld_out, float* h, int rows, int k, int n, int rank, int adapters,
              const Pieces& pieces) {
    const int inner = pieces.count * rank;
    adapter_down_plain<T><<<dim3((inner + 3) / 4, rows), kThreads, 0, s>>>(static_cast<const T*>(x), ldx, static_cast<const T*>(down),
                                                                          adapter, h, rows, inner, k, adapters);
    if (cie_after_launch() != CIE_OK) return CIE_LAUNCH_FAILED;
    adapter_up_plain<T, S><<<dim3((n + kThreads - 1) / kThreads, rows), kThreads, 0, s>>>(
        h, static_cast<const T*>(up), scale, adapter, static_cast<const S*>(into), ld_into, static_cast<S*>(out), ld_out, rows, inner, n,
        rank, adapters, pieces);
    return cie_after_launch();
}

}  // namespace

// dtype: of x, down and up; out_dtype: of into and out (dtype, or float32).  c1, c2, c3: where the second and later pieces begin
// (n where there is none).  h: rows * pieces * rank floats.  out may be into.
CIE_API int cie_lora_add(void* stream, int dtype, int out_dtype, const void* x, long ldx, const void* down, const void* up,
                         const float* scale, const int* adapter, const void* into, long ld_into, void* out, long ld_out, float* h,
                         int rows, int k, int n, int rank, int adapters, int piece_count, int c1, int c2, int c3) {
    if (rows < 0 || rows > 65535 || k <= 0 || n <= 0 || rank <= 0 || adapters <= 0 || piece_count < 1 || piece_count > kMaxPieces ||
        ldx < k || ld_into < n || ld_out < n || !x || !down || !up || !scale || !adapter || !into || !out || !h)
        return CIE_BAD_ARGUMENT;
    if (rows == 0) return CIE_OK;
    Pieces pieces = {piece_count, {0, c1, c2, c3, n}};
    for (int p = piece_count; p <= kMaxPieces; ++p) pieces.begin[p] = n;
    for (int p = 0; p < piece_count; ++p)
        if (pieces.begin[p + 1] <= pieces.begin[p]) return CIE_BAD_ARGUMENT;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == CIE_F32 && out_dtype == CIE_F32)
        return run_plain<float, float>(s, x, ldx, down, up, scale, adapter, into, ld_into, out, ld_out, h, rows, k, n, rank, adapters, pieces);
    if (dtype == CIE_BF16 && out_dtype == CIE_F32)
        return run_plain<bf16_t, float>(s, x, ldx, down, up, scale, adapter, into, ld_into, out, ld_out, h, rows, k, n, rank, adapters, pieces);
    if (dtype == CIE_BF16 && out_dtype == CIE_BF16)
        return run_plain<bf16_t, bf16_t>(s, x, ldx, down, up, scale, adapter, into, ld_into, out, ld_out, h, rows, k, n, rank, adapters, pieces);
    return CIE_BAD_ARGUMENT;
}
