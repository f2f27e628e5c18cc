// Drawing a token under top-k, top-p and min-p from a given number; one workgroup per row.
//
// Row r has float32 logits l, a temperature T, k, p, m and a number u in [0, 1).
//   T <= 0 (or NaN): the first index of the largest logit; nothing else counts.
//   w_i = exp((l_i - max l) / T), 1 where l_i = max l; NaN and -inf weigh nothing.
//   order: the larger logit first, of equal ones the lower index.
//   top-k (0 < k < vocab): the first k of the order.  top-p (p < 1): of these, the tokens in front of which less than
//   p of their weight lies (the first one always).  min-p (m > 0): tokens with w_i >= m (the largest always).
//   The token is the first kept one, in the order of the indices, whose running sum of w passes u times the sum of all kept.
// A row in which nothing weighs anything gives index 0.
//
// Every rule keeps a prefix of one order, so what is kept is said by one cut: a logit, and of the tokens that are equal to it
// the last index.
//
// Weights are summed as whole numbers, w times a power of two that lets a whole row fit 63 bits (2^44 for 152,000 tokens).
// Such sums do not depend on their order: threads add with atomics and a row's token is the same in any layout.  Rounding a
// weight to 2^-45 leaves a sum of 152,000 of them off by some 6e-12 of the largest weight; with float32 sums (1e-7) every
// few dozen rows without a rule would draw the neighbour of the token that the definition names.
#include "common.h"

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;

// Larger for a larger logit; 0 for NaN.  (-0 and +0 are equal.)
__device__ __forceinline__ uint32_t order_of(float l) {
    if (l != l) return 0u;
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kOrderOfMinusInf = 0x007fffffu;  // (whatever is not above it weighs nothing)

struct Row {
    const float* logits;
    int vocab;
    float best;      // the largest logit
    double inv_t;
    double unit;     // what a weight of 1 counts
    double least;    // min-p; 0: off

    __device__ __forceinline__ u64 weight(float l) const {
        if (order_of(l) <= kOrderOfMinusInf) return 0;
        const double w = l == best ? 1.0 : exp((static_cast<double>(l) - static_cast<double>(best)) * inv_t);
        if (!(w >= least)) return 0;
        return static_cast<u64>(w * unit + 0.5);
    }
};

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, kWave);
    return v;
}

__device__ __forceinline__ u64 wave_running_u64(u64 v) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int offset = 1; offset < kWave; offset <<= 1) {
        const u64 below = __shfl_up(v, offset, kWave);
        if (lane >= offset) v += below;
    }
    return v;
}

// The first index of [0, n) whose running sum of f(i) passes the target (u times the whole sum if `of_whole`), or the last
// index with any f if none does; -1 if the sum is 0.  Each of the workgroup's waves sums a stretch; the stretch that holds
// the target is cut again, until one wave's lanes hold an index each.  All threads call it and get the result.
template <typename F>
__device__ int seek(int n, double target, bool of_whole, u64* s_sum, F f) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int begin = 0, end = n;
    u64 before = 0;
    for (bool first = true; first || end - begin > kWave; first = false) {
        const int stretch = ((end - begin + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
        const int from = min(end, begin + wave * stretch), to = min(end, from + stretch);
        u64 sum = 0;
        for (int i = from + lane; i < to; i += kWave) sum += f(i);
        sum = wave_sum_u64(sum);
        __syncthreads();
        if (lane == 0) s_sum[wave] = sum;
        __syncthreads();
        if (first) {
            u64 total = 0;
            for (int w = 0; w < kWaves; ++w) total += s_sum[w];
            if (total == 0) return -1;
            if (of_whole) target *= static_cast<double>(total);
        }
        int owner = 0;
        u64 running = before, before_owner = before;
        for (int w = 0; w < kWaves; ++w) {
            if (s_sum[w] == 0) continue;
            owner = w;
            before_owner = running;
            running += s_sum[w];
            if (static_cast<double>(running) > target) break;
        }
        before = before_owner;
        begin = min(end, begin + owner * stretch);
        end = min(end, begin + stretch);
    }
    const u64 own = begin + lane < end ? f(begin + lane) : 0;
    const u64 running = before + wave_running_u64(own);
    const u64 passed = __ballot(own > 0 && static_cast<double>(running) > target);
    const u64 any = __ballot(own > 0);
    return begin + (passed ? __ffsll(passed) - 1 : 63 - __clzll(any));
}

struct Histogram {
    u64 weight[kBins];
    int count[kBins];
    u64 wave_weight[kWaves];
    int wave_count[kWaves];
    int bin;
    u64 above_weight;
    int above_count;
};

// The bin, from the largest digit down, in which the running count reaches `need` (by_count), or the running weight `limit`;
// the last bin that holds anything if none does.  The sums of the bins in front of it are left in `h`.
__device__ void cross(Histogram& h, bool by_count, int need, double limit) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    // thread t has bins kBins - 1 - 2 t and the next lower one
    const int hi = kBins - 1 - 2 * threadIdx.x, lo = hi - 1;
    const u64 own_w = h.weight[hi] + h.weight[lo];
    const int own_c = h.count[hi] + h.count[lo];
    u64 run_w = wave_running_u64(own_w);
    int run_c = own_c;
#pragma unroll
    for (int offset = 1; offset < kWave; offset <<= 1) {
        const int below = __shfl_up(run_c, offset, kWave);
        if (lane >= offset) run_c += below;
    }
    if (lane == kWave - 1) {
        h.wave_weight[wave] = run_w;
        h.wave_count[wave] = run_c;
    }
    if (threadIdx.x == 0) h.bin = -1;
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        run_w += h.wave_weight[w];
        run_c += h.wave_count[w];
    }
    u64 before_w = run_w - own_w;
    int before_c = run_c - own_c;
    for (int i = 0; i < 2; ++i) {
        const int bin = i == 0 ? hi : lo;
        const u64 after_w = before_w + h.weight[bin];
        const int after_c = before_c + h.count[bin];
        const bool reached = by_count ? after_c >= need : static_cast<double>(after_w) >= limit;
        if (reached && h.count[bin] > 0) atomicMax(&h.bin, bin);
        before_w = after_w;
        before_c = after_c;
    }
    __syncthreads();
    int found = h.bin;
    __syncthreads();
    if (found < 0) {  // (a limit that rounding left out of reach)
        if (h.count[lo] > 0 || h.count[hi] > 0) atomicMax(&h.bin, kBins - (h.count[lo] > 0 ? lo : hi));
        __syncthreads();
        found = kBins - h.bin;
    }
    if (found == hi || found == lo) {
        h.bin = found;
        h.above_weight = run_w - own_w + (found == lo ? h.weight[hi] : 0);
        h.above_count = run_c - own_c + (found == lo ? h.count[hi] : 0);
    }
    __syncthreads();
}

struct Cut {
    uint32_t key;    // the order of the last kept token
    int ties;        // how many tokens of that order are kept
    int equal;       // ... and how many there are
    u64 above;       // the weight of what lies in front of them
    u64 each;        // the weight of one of them
};

// The cut after `need` tokens (by_count), or where `limit` of the weight is reached, among the tokens not under `floor`.
// Three histograms of the order's 11, 11 and 10 bits, from the top.
__device__ Cut find_cut(const Row& row, Histogram& h, bool by_count, int need, double limit, uint32_t floor) {
    Cut cut = {0u, need, 0, 0, 0};
    for (int step = 0; step < 3; ++step) {
        const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bits = step == 2 ? 10 : 11;
        const uint32_t known = step == 0 ? 0u : 0xffffffffu << (shift + bits);
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            h.weight[b] = 0;
            h.count[b] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < row.vocab; i += kThreads) {
            const float l = row.logits[i];
            const uint32_t key = order_of(l);
            if ((key & known) != cut.key || key < floor) continue;
            const int bin = (key >> shift) & ((1 << bits) - 1);
            atomicAdd(&h.count[bin], 1);
            const u64 w = row.weight(l);
            if (w) atomicAdd(&h.weight[bin], w);
        }
        __syncthreads();
        cross(h, by_count, cut.ties, limit - static_cast<double>(cut.above));
        cut.key |= static_cast<uint32_t>(h.bin) << shift;
        cut.above += h.above_weight;
        if (by_count) cut.ties -= h.above_count;
        cut.equal = h.count[h.bin];
        cut.each = h.weight[h.bin];
    }
    cut.each /= max(1, cut.equal);  // (equal logits weigh the same)
    if (!by_count) {
        // the j-th of the equal ones is kept while less than the limit lies in front of it
        const double left = cut.each ? ceil((limit - static_cast<double>(cut.above)) / static_cast<double>(cut.each)) : 1.0;
        cut.ties = left < 1.0 ? 1 : left < cut.equal ? static_cast<int>(left) : cut.equal;
    }
    return cut;
}

__global__ void __launch_bounds__(kThreads)
sample_rules_kernel(const float* __restrict__ logits, const float* __restrict__ temperature, const float* __restrict__ uniform,
                    const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p,
                    int* __restrict__ out, int vocab, long ld, double unit) {
    __shared__ Histogram h;
    __shared__ u64 s_sum[kWaves];
    const int r = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    Row row;
    row.logits = logits + static_cast<size_t>(r) * ld;
    row.vocab = vocab;
    row.unit = unit;

    // the largest logit and its first index
    uint32_t best_key = 0;
    int best_idx = 0x7fffffff;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
        const uint32_t key = order_of(row.logits[i]);
        if (key > best_key) {
            best_key = key;
            best_idx = i;
        }
    }
    u64 first = (static_cast<u64>(best_key) << 32) | (0x7fffffffu - best_idx);
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) {
        const u64 other = __shfl_xor(first, offset, kWave);
        first = other > first ? other : first;
    }
    if (lane == 0) s_sum[wave] = first;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) first = s_sum[w] > first ? s_sum[w] : first;
    __syncthreads();
    best_key = static_cast<uint32_t>(first >> 32);
    best_idx = best_key > kOrderOfMinusInf ? 0x7fffffff - static_cast<int>(first & 0xffffffffu) : 0;
    const float temp = temperature[r];
    if (!(temp > 0.f) || best_key <= kOrderOfMinusInf) {
        if (threadIdx.x == 0) out[r] = best_idx;
        return;
    }
    row.best = row.logits[best_idx];
    row.inv_t = 1.0 / static_cast<double>(temp);
    row.least = 0.0;
    const int k = top_k ? top_k[r] : 0;
    const double p = top_p ? static_cast<double>(top_p[r]) : 1.0;
    const double m = min_p ? static_cast<double>(min_p[r]) : 0.0;

    Cut cut = {0u, vocab, vocab, 0, 0};  // everything
    u64 total = 0;
    const bool by_count = k > 0 && k < vocab;
    if (by_count) {
        cut = find_cut(row, h, true, k, 0.0, 0u);
        total = cut.above + cut.each * cut.ties;
    }
    if (p < 1.0) {
        if (!by_count) {
            u64 sum = 0;
            for (int i = threadIdx.x; i < vocab; i += kThreads) sum += row.weight(row.logits[i]);
            sum = wave_sum_u64(sum);
            if (lane == 0) s_sum[wave] = sum;
            __syncthreads();
            for (int w = 0; w < kWaves; ++w) total += s_sum[w];
            __syncthreads();
        }
        const Cut nucleus = find_cut(row, h, false, 0, p * static_cast<double>(total), cut.key);
        if (nucleus.key > cut.key) {
            cut = nucleus;
        } else if (nucleus.ties < cut.ties) {
            cut.ties = nucleus.ties;
            cut.equal = nucleus.equal;
        }
    }
    int last_tie = vocab;
    if (cut.ties < cut.equal) {  // which of the equal ones: the first by index
        const uint32_t key = cut.key;
        last_tie = seek(vocab, cut.ties - 0.5, false, s_sum, [&](int i) -> u64 { return order_of(row.logits[i]) == key; });
    }
    row.least = m > 1.0 ? 1.0 : m;  // (the largest always stays; NaN: off)
    if (!(row.least > 0.0)) row.least = 0.0;
    const uint32_t key = cut.key;
    const int picked = seek(vocab, static_cast<double>(uniform[r]), true, s_sum, [&](int i) -> u64 {
        const float l = row.logits[i];
        const uint32_t mine = order_of(l);
        return mine > key || (mine == key && i <= last_tie) ? row.weight(l) : 0;
    });
    if (threadIdx.x == 0) out[r] = picked < 0 ? best_idx : picked;
}

}  // namespace

// top_k, top_p and min_p may each be null: that rule is off in every row.
CIE_API int cie_sample_rules(void* stream, const float* logits, const float* temperature, const float* uniform, const int* top_k,
                             const float* top_p, const float* min_p, int* out, int rows, int vocab, long ld) {
    if (rows < 0 || vocab <= 0 || ld < vocab || rows > 65535 || vocab > (1 << 30) || !logits || !temperature || !uniform || !out)
        return CIE_BAD_ARGUMENT;
    if (rows == 0) return CIE_OK;
    int bits = 0;
    while ((1L << bits) < vocab) ++bits;
    const double unit = static_cast<double>(1L << (62 - bits < 51 ? 62 - bits : 51));
    sample_rules_kernel<<<rows, kThreads, 0, static_cast<hipStream_t>(stream)>>>(logits, temperature, uniform, top_k, top_p, min_p,
                                                                               out, vocab, ld, unit);
    return cie_after_launch();
}
