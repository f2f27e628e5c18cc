// Drawing a token under top-k, top-p and min-p from a given number.
//
// Row r has float32 logits l, a temperature T, k, p, m and a number u in [0, 1).
//   T <= 0 (or NaN): the first index of the largest logit; nothing else counts.
//   w_i = exp((l_i - max l) / T), 1 where l_i = max l; NaN and -inf weigh nothing.
//   order: the larger logit first, of equal ones the lower index.
//   top-k (0 < k < vocab): the first k of the order.  top-p (p < 1): of these, the tokens in front of which less than
//   p of their weight lies (the first one always).  min-p (m > 0): tokens with w_i >= m (the largest always).
//   The token is the first kept one, in the order of the indices, whose running sum of w passes u times the sum of all kept.
//   (A token of less than 2^-45 of the largest weight, for 152,000 tokens, is not drawn: see below.)
// A row in which nothing weighs anything gives index 0.
//
// The first launch reads the logits once, in parts that fill the GPU: the largest of each part, of each 16 numbers (a chunk), and,
// for rows without top-k, the part's sum of weights.  The last has a workgroup for each row.
//   top-k: the k-th largest of the chunks' largest is a bound that the k largest logits reach; what passes it, from the few
//     chunks whose largest does, is gathered, ranked, cut and drawn from in LDS.
//   top-p or min-p without top-k: a share p of the weight cannot reach down to tokens that weigh less than (1 - p) / vocab of
//     the sum, and min-p names its bound itself.  Two launches between the others go through the chunks that pass the bound: one adds
//     the weights to the row's histogram over equal bins of (max - l) / T, the other finds the bin that holds the cut, sums the
//     weights in front of it part by part and lists the bin's numbers.  The last one sorts these, and walks the part it draws from.
//   no rule: the parts' sums say which part is walked.
// Rows that defeat this (more than kList logits that pass a k's bound, or in the cut's bin) are cut by the bits of their logits.
//
// One reading of the logits is what this has to cost; what few rows take beyond it are the launches' chains of small steps (find the
// largest, add up, sort, add up, cut).  Measured, the kernels' own times: one row of 151,936 under top-k and top-p 18 us (0.6 MB; the
// draw alone 10.6); 8 rows under top-p alone 41 us (4.9 MB; parts 7, tally 9, collect 11, draw 14); 64 rows of all kinds 64 us
// (38.9 MB; 17, 9, 11, 28); 256 rows of 152,064 under all three rules 65 us (156 MB; parts 27 at 5.8 TB/s, draw 30).  One workgroup
// a row for all of it took 282, 400, 459 and 562 us.
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

// exp(x) for x <= 0, to some 1e-14 of it: x = n ln 2 + r with |r| <= ln 2 / 2, and 2^n times the series of e^r up to r^11, behind
// which r^12 / 12! = 6e-15 is left.  (18 instructions; a row without top-k takes one for each of its numbers.)
__device__ __forceinline__ double exp_below(double x) {
    x = fmax(x, -745.0);  // (2^-1074, no weight; NaN too)
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, x));
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, static_cast<int>(n));
}

struct Row {
    const float* logits;
    int vocab;
    float best;      // the largest logit
    double inv_t;
    double unit;     // what a weight of 1 counts
    double least;    // min-p; 0: off

    __device__ __forceinline__ double share(float l) const {
        if (!(l > -INFINITY)) return 0.0;
        return l == best ? 1.0 : exp_below((static_cast<double>(l) - static_cast<double>(best)) * inv_t);
    }
    __device__ __forceinline__ u64 weight(float l) const {
        const double w = share(l);
        return w >= least ? static_cast<u64>(w * unit + 0.5) : 0;
    }
};

// 64-bit sums over a wave without a round trip through LDS a step (a dozen of them were most of what a row's last launch took).
__device__ __forceinline__ u64 joined(uint32_t lo, uint32_t hi) { return static_cast<u64>(hi) << 32 | lo; }
template <int kControl, int kRows>
__device__ __forceinline__ u64 moved(u64 v) {  // (0 where a lane has no source, or lies in a row of 16 that is left out)
    const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v & 0xffffffffu), kControl, kRows, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), kControl, kRows, 0xf, false);
    return joined(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}
// The sum of the lanes up to each one: 1, 2, 4 and 8 lanes on within rows of 16, then a row's last lane to the next row, and the
// second row's to the upper half.
__device__ __forceinline__ u64 wave_running_u64(u64 v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    return v + moved<0x143, 0xc>(v);
}
__device__ __forceinline__ u64 last_lane(u64 v) {
    return joined(__builtin_amdgcn_readlane(static_cast<int>(v & 0xffffffffu), kWave - 1),
                  __builtin_amdgcn_readlane(static_cast<int>(v >> 32), kWave - 1));
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) { return last_lane(wave_running_u64(v)); }
// (0 is no number's better)
__device__ __forceinline__ u64 larger(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 wave_most_u64(u64 v) {
    v = larger(v, moved<0x111, 0xf>(v));
    v = larger(v, moved<0x112, 0xf>(v));
    v = larger(v, moved<0x114, 0xf>(v));
    v = larger(v, moved<0x118, 0xf>(v));
    v = larger(v, moved<0x142, 0xa>(v));
    return last_lane(larger(v, moved<0x143, 0xc>(v)));
}
// A lane's partner, N (a power of two) lanes off by exclusive or.
template <int N>
__device__ __forceinline__ uint32_t partner(uint32_t v) {
    if constexpr (N == 16) {
        const swap_pair_t both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return both[0] ^ both[1] ^ v;
    } else if constexpr (N == 32) {
        const swap_pair_t both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return both[0] ^ both[1] ^ v;
    } else if constexpr (N == 4) {  // 7 (a half row mirrored), then 3 (quads mirrored)
        const int half = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xf, 0xf, true);
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, half, 0x1b, 0xf, 0xf, true));
    } else {  // quads, or a row turned by half
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), N == 1 ? 0xb1 : N == 2 ? 0x4e : 0x128, 0xf, 0xf, true));
    }
}
template <int N>
__device__ __forceinline__ u64 partner_u64(u64 v) {
    return joined(partner<N>(static_cast<uint32_t>(v)), partner<N>(static_cast<uint32_t>(v >> 32)));
}

__device__ __forceinline__ double wave_sum_f64(double v) {  // (all lanes the same)
    const auto with = [&](u64 other) { v += __builtin_bit_cast(double, other); };
    with(partner_u64<1>(__builtin_bit_cast(u64, v)));
    with(partner_u64<2>(__builtin_bit_cast(u64, v)));
    with(partner_u64<4>(__builtin_bit_cast(u64, v)));
    with(partner_u64<8>(__builtin_bit_cast(u64, v)));
    with(partner_u64<16>(__builtin_bit_cast(u64, v)));
    with(partner_u64<32>(__builtin_bit_cast(u64, v)));
    return v;
}

// What the waves of a workgroup left in `s` (kCount of them): the sum of those in front of this one, and of all.
template <int kCount>
__device__ __forceinline__ void across_waves(const u64* s, u64& front, u64& total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const u64 own = lane < kCount ? s[lane] : 0;
    front = wave_sum_u64(lane < wave ? own : 0);
    total = wave_sum_u64(own);
}

// The first index of [begin, end) whose running sum of f(i), with `before` in front of it, passes the target (u times the whole
// sum if `of_whole`), or the last index with any f if none does; -1 if the sum is 0.  Each of the workgroup's waves sums a stretch; the stretch that holds
// the target is cut again, until one wave's lanes hold an index each.  All threads call it and get the result.
template <typename F>
__device__ int seek(int begin, int end, u64 before, double target, bool of_whole, u64* s_sum, F f) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
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
            if (of_whole) target *= static_cast<double>(before + total);
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
    u64 wave[kWaves];
    int bin;
    u64 above;
};

// The bin, from the largest digit down, in which the running count reaches `need` (by_count), or the running weight `limit`;
// the last bin that counts (weighs) anything if none does, -1 if all are empty.  The sum of the bins in front of it is left in
// h.above, the bin in h.bin.
template <bool kByCount>
__device__ void cross(Histogram& h, int need, double limit) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    // thread t has bins kBins - 1 - 2 t and the next lower one
    const int hi = kBins - 1 - 2 * threadIdx.x, lo = hi - 1;
    const u64 in_hi = kByCount ? static_cast<u64>(h.count[hi]) : h.weight[hi], in_lo = kByCount ? static_cast<u64>(h.count[lo]) : h.weight[lo];
    const u64 running = wave_running_u64(in_hi + in_lo);
    if (lane == kWave - 1) h.wave[wave] = running;
    if (threadIdx.x == 0) h.bin = -1;
    __syncthreads();
    u64 front, total;
    across_waves<kWaves>(h.wave, front, total);
    front += running - in_hi - in_lo;
    // (one bin: what lies in front of it does not reach, or is nothing, and with it the sum does)
    const double wanted = fmin(kByCount ? static_cast<double>(need) : limit, static_cast<double>(total));
    const bool in_first = in_hi && (front == 0 || static_cast<double>(front) < wanted) && static_cast<double>(front + in_hi) >= wanted;
    const bool in_second = in_lo && (front + in_hi == 0 || static_cast<double>(front + in_hi) < wanted) &&
                           static_cast<double>(front + in_hi + in_lo) >= wanted;
    if (in_first || in_second) {
        h.bin = in_first ? hi : lo;
        h.above = front + (in_first ? 0 : in_hi);
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
        if (by_count)
            cross<true>(h, cut.ties, 0.0);
        else
            cross<false>(h, 0, limit - static_cast<double>(cut.above));
        cut.key |= static_cast<uint32_t>(h.bin) << shift;
        if (by_count) {  // (what the larger bins weigh: the sum that decided is their count)
            u64 above = 0;
            for (int b = threadIdx.x; b < kBins; b += kThreads) above += b > h.bin ? h.weight[b] : 0;
            above = wave_sum_u64(above);
            if (threadIdx.x % kWave == 0) h.wave[threadIdx.x / kWave] = above;
            __syncthreads();
            u64 front;
            across_waves<kWaves>(h.wave, front, above);
            cut.above += above;
            cut.ties -= static_cast<int>(h.above);
        } else {
            cut.above += h.above;
        }
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

// The draw by the logits' bits: any row, several walks over it.
__device__ int draw_by_bits(Row& row, Histogram& h, u64* s_sum, int k, double p, double m, double u) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    Cut cut = {0u, row.vocab, row.vocab, 0, 0};  // everything
    u64 total = 0;
    const bool by_count = k > 0 && k < row.vocab;
    row.least = 0.0;
    if (by_count) {
        cut = find_cut(row, h, true, k, 0.0, 0u);
        total = cut.above + cut.each * cut.ties;
    }
    if (p < 1.0) {
        if (!by_count) {
            u64 sum = 0;
            for (int i = threadIdx.x; i < row.vocab; i += kThreads) sum += row.weight(row.logits[i]);
            sum = wave_sum_u64(sum);
            __syncthreads();
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
    int last_tie = row.vocab;
    const uint32_t key = cut.key;
    if (cut.ties < cut.equal)  // which of the equal ones: the first by index
        last_tie = seek(0, row.vocab, 0, cut.ties - 0.5, false, s_sum, [&](int i) -> u64 { return order_of(row.logits[i]) == key; });
    row.least = m;
    return seek(0, row.vocab, 0, u, true, s_sum, [&](int i) -> u64 {
        const float l = row.logits[i];
        const uint32_t mine = order_of(l);
        return mine > key || (mine == key && i <= last_tie) ? row.weight(l) : 0;
    });
}

// ---------------------------------------------------------------- first launch
constexpr int kPartThreads = 256;
constexpr int kPart = kPartThreads * 16;  // numbers of a part: a thread has four times four neighbours, 1,024 numbers apart

constexpr int kList = 4096;
constexpr int kMaxParts = 1024;

struct PartOf {
    struct Largest {
        u64 best;    // order << 32 | (0x7fffffff - index)
        double sum;  // of exp((l - the part's largest) / T), where the row asks for it
    };
    Largest* part;   // [rows, parts]
    float* chunk;    // [rows, parts * kPartThreads] the largest of each thread's 16; -inf where there is none
    // of rows under top-p or min-p without top-k:
    u64* kept;       // [rows, parts] weight of what lies in front of the cut's bin
    u64* histogram;  // [rows, kBins]
    u64* list;       // [rows, kList] the numbers of the cut's bin
    u64* head;       // [rows, 2] how many these are; what lies in front of them
};

__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// The rules of a row as they count: k = 0, p = 1 and m = 0 are off (NaN too).
struct Rules {
    float temp;
    int k;
    double p, m;
    __device__ __forceinline__ Rules(const float* temperature, const int* top_k, const float* top_p, const float* min_p, int r, int vocab) {
        temp = temperature[r];
        k = top_k && top_k[r] > 0 && top_k[r] < vocab ? top_k[r] : 0;
        p = top_p && top_p[r] < 1.f ? (top_p[r] > 0.f ? static_cast<double>(top_p[r]) : 0.0) : 1.0;
        m = min_p && min_p[r] > 0.f ? (min_p[r] < 1.f ? static_cast<double>(min_p[r]) : 1.0) : 0.0;  // (the largest stays)
    }
    __device__ __forceinline__ bool draws() const { return temp > 0.f; }
    __device__ __forceinline__ bool shares() const { return temp > 0.f && k == 0; }          // needs the parts' sums
    __device__ __forceinline__ bool tallied() const { return shares() && (p < 1.0 || m > 0.0); }
};

__global__ void __launch_bounds__(kPartThreads)
rules_parts_kernel(const float* __restrict__ logits, const float* __restrict__ temperature, const int* __restrict__ top_k,
                   const float* __restrict__ top_p, const float* __restrict__ min_p, PartOf of, int vocab, long ld) {
    constexpr int kPartWaves = kPartThreads / kWave;
    __shared__ u64 s_best[kPartWaves];
    __shared__ double s_sum[kPartWaves];
    const int r = blockIdx.y, part = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const float* row = logits + static_cast<size_t>(r) * ld;
    const int first = part * kPart + threadIdx.x * 4;
    float l[16];
    const bool lines = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int at = first + q * kPartThreads * 4;
        if (lines && at + 3 < vocab) {
            const float4 v = *reinterpret_cast<const float4*>(row + at);
            l[q * 4] = v.x;
            l[q * 4 + 1] = v.y;
            l[q * 4 + 2] = v.z;
            l[q * 4 + 3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) l[q * 4 + e] = at + e < vocab ? row[at + e] : -INFINITY;
        }
    }
    const Rules rules(temperature, top_k, top_p, min_p, r, vocab);
    uint32_t key = 0;
    int where = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // (in the order of the indices: the first of equal ones stays)
        const uint32_t mine = order_of(l[i]);
        if (mine > key) {
            key = mine;
            where = first + i / 4 * kPartThreads * 4 + i % 4;
        }
    }
    u64 best = (static_cast<u64>(key) << 32) | static_cast<uint32_t>(0x7fffffff - where);
    // the order's float (a chunk of NaN alone counts as -inf)
    const float largest = key <= kOrderOfMinusInf ? -INFINITY : logit_of(key);
    of.chunk[(static_cast<size_t>(r) * gridDim.x + part) * kPartThreads + threadIdx.x] = largest;
    best = wave_most_u64(best);
    if (lane == 0) s_best[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPartWaves; ++w) best = s_best[w] > best ? s_best[w] : best;
    PartOf::Largest* const mine = of.part + static_cast<size_t>(r) * gridDim.x + part;
    if (threadIdx.x == 0) mine->best = best;
    if (!rules.shares()) return;
    if (rules.tallied()) {  // (the launches behind this one add to them)
        for (int b = part * kPartThreads + threadIdx.x; b < kBins; b += gridDim.x * kPartThreads) of.histogram[static_cast<size_t>(r) * kBins + b] = 0;
        if (part == 0 && threadIdx.x == 0) of.head[2 * r] = 0;
    }
    key = static_cast<uint32_t>(best >> 32);
    double sum = 0.0;
    if (key > kOrderOfMinusInf) {
        const Row scaled = {row, vocab, logit_of(key), 1.0 / static_cast<double>(rules.temp), 1.0, 0.0};
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += scaled.share(l[i]);
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int w = 0; w < kPartWaves; ++w) sum += s_sum[w];
        mine->sum = sum;
    }
}

// What the parts say of a row: its largest logit, and the sum of its weights where the row asks for it.
template <int kBlock>
struct Whole {
    static constexpr int kBlockWaves = kBlock / kWave;
    u64 best[kBlockWaves];
    double sum[kMaxParts];  // what each part weighs

    __device__ __forceinline__ u64 find_best(const PartOf::Largest* part, int parts, const PartOf::Largest& own) {
        u64 found = own.best;
        for (int q = threadIdx.x + kBlock; q < parts; q += kBlock) found = larger(found, part[q].best);
        found = wave_most_u64(found);
        if (threadIdx.x % kWave == 0) best[threadIdx.x / kWave] = found;
        __syncthreads();
        return wave_most_u64(best[threadIdx.x % kBlockWaves]);
    }
    // (`own`: the thread's first part, asked for before anything waits)
    static __device__ __forceinline__ PartOf::Largest first_of(const PartOf::Largest* part, int parts) {
        return static_cast<int>(threadIdx.x) < parts ? part[threadIdx.x] : PartOf::Largest{0, 0.0};
    }
    // (every wave the same: lanes take the parts in turn, and are added in one order)
    __device__ __forceinline__ double find_total(const Row& row, const PartOf::Largest* part, int parts, const PartOf::Largest& own) {
        for (int q = threadIdx.x; q < parts; q += kBlock) {
            PartOf::Largest its = own;
            if (q >= kBlock) its = part[q];
            const uint32_t key = static_cast<uint32_t>(its.best >> 32);
            sum[q] = key > kOrderOfMinusInf ? its.sum * row.share(logit_of(key)) : 0.0;
        }
        __syncthreads();
        double total = 0.0;
        for (int q = threadIdx.x % kWave; q < parts; q += kWave) total += sum[q];
        return wave_sum_f64(total);
    }
};

// ---------------------------------------------------------------- rows under top-p or min-p without top-k
// What weighs less than (1 - p) / vocab of the sum, or less than m, is not kept however the rest is shared out.
// (In 32 bits, a little too far: the logarithm is off by some 1e-6 and 1e-7 of itself, the difference of two logits by 6e-8 of
// itself.  In 64 bits 8 rows' tally took 9.2 us, not 8.8.)
struct Reach {
    float best, distance, bins;  // (bins: how many of the histogram's a unit of distance has; they share the reach evenly)
    __device__ __forceinline__ Reach(const Row& row, const Rules& rules, double total) {
        best = row.best;
        const float least = fmaxf(rules.p < 1.0 ? static_cast<float>((1.0 - rules.p) * total) / static_cast<float>(row.vocab) : 0.f,
                                  static_cast<float>(rules.m));
        distance = (2e-6f - logf(fminf(least, 1.f))) * rules.temp * 1.000002f + 1e-30f;
        bins = (kBins - 1) / distance;
    }
    __device__ __forceinline__ bool operator()(float l) const { return l > -INFINITY && (l == best || best - l <= distance); }
};

// The larger the nearer to the largest.
__device__ __forceinline__ int bin_of(const Reach& reach, float l) {
    const float at = l == reach.best ? 0.f : (reach.best - l) * reach.bins;
    return kBins - 1 - (at < kBins - 1 ? static_cast<int>(at) : kBins - 1);
}

// What a row's numbers are sorted by: the larger logit first, then the lower index.
__device__ __forceinline__ u64 place_of(float l, int i) { return (static_cast<u64>(~order_of(l)) << 32) | static_cast<uint32_t>(i); }

// Runs f(l, index) over the thread's chunk of a part, if its largest passes.
template <typename F>
__device__ __forceinline__ void walk_chunk(const Row& row, float largest, int part, const Reach& reach, F f) {
    if (!reach(largest)) return;
    const int first = part * kPart + threadIdx.x * 4;
    float l[16];
    const bool lines = (reinterpret_cast<uintptr_t>(row.logits) & 15) == 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int at = first + q * kPartThreads * 4;
        if (lines && at + 3 < row.vocab) {
            const float4 v = *reinterpret_cast<const float4*>(row.logits + at);
            l[q * 4] = v.x;
            l[q * 4 + 1] = v.y;
            l[q * 4 + 2] = v.z;
            l[q * 4 + 3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) l[q * 4 + e] = at + e < row.vocab ? row.logits[at + e] : -INFINITY;
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (reach(l[i])) f(l[i], first + i / 4 * kPartThreads * 4 + i % 4);
}

// grid: (some workgroups, rows)
__global__ void __launch_bounds__(kPartThreads)
rules_tally_kernel(const float* __restrict__ logits, const float* __restrict__ temperature, const int* __restrict__ top_k,
                   const float* __restrict__ top_p, const float* __restrict__ min_p, PartOf of, int vocab, long ld, int parts, double unit) {
    __shared__ Whole<kPartThreads> whole;
    __shared__ u64 s_weight[kBins];
    const int r = blockIdx.y;
    const Rules rules(temperature, top_k, top_p, min_p, r, vocab);
    if (!rules.tallied() || !(rules.p < 1.0)) return;
    const PartOf::Largest* of_parts = of.part + static_cast<size_t>(r) * parts;
    // (what the launches before this one left is asked for at once: 8 rows' four launches 39 us, not 40)
    const PartOf::Largest own = whole.first_of(of_parts, parts);
    const float* chunks = of.chunk + static_cast<size_t>(r) * parts * kPartThreads + threadIdx.x;
    float largest = chunks[blockIdx.x * kPartThreads];
    for (int b = threadIdx.x; b < kBins; b += kPartThreads) s_weight[b] = 0;
    const uint32_t key = static_cast<uint32_t>(whole.find_best(of_parts, parts, own) >> 32);
    if (key <= kOrderOfMinusInf) return;
    const Row row = {logits + static_cast<size_t>(r) * ld, vocab, logit_of(key), 1.0 / static_cast<double>(rules.temp), unit, 0.0};
    const Reach reach(row, rules, whole.find_total(row, of_parts, parts, own));
    for (int part = blockIdx.x; part < parts; part += gridDim.x) {
        const int next = part + gridDim.x < parts ? part + gridDim.x : part;
        const float now = largest;
        largest = chunks[next * kPartThreads];
        walk_chunk(row, now, part, reach, [&](float l, int) {
            const u64 w = row.weight(l);
            if (w) atomicAdd(&s_weight[bin_of(reach, l)], w);
        });
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kPartThreads)
        if (s_weight[b]) atomicAdd(&of.histogram[static_cast<size_t>(r) * kBins + b], s_weight[b]);
}

// grid: (some workgroups, rows)
__global__ void __launch_bounds__(kPartThreads)
rules_collect_kernel(const float* __restrict__ logits, const float* __restrict__ temperature, const int* __restrict__ top_k,
                     const float* __restrict__ top_p, const float* __restrict__ min_p, PartOf of, int vocab, long ld, int parts, double unit) {
    constexpr int kOwn = kBins / kPartThreads, kPartWaves = kPartThreads / kWave;
    __shared__ Whole<kPartThreads> whole;
    __shared__ u64 s_sum[kPartWaves];
    __shared__ int s_bin, s_count;
    __shared__ u64 s_above, s_at, s_list[kPart];
    const int r = blockIdx.y, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const Rules rules(temperature, top_k, top_p, min_p, r, vocab);
    if (!rules.tallied()) return;
    const PartOf::Largest* of_parts = of.part + static_cast<size_t>(r) * parts;
    const PartOf::Largest own = whole.first_of(of_parts, parts);
    const float* chunks = of.chunk + static_cast<size_t>(r) * parts * kPartThreads + threadIdx.x;
    float largest = chunks[blockIdx.x * kPartThreads];
    if (threadIdx.x == 0) {
        s_bin = -1;
        s_above = 0;
    }
    const uint32_t key = static_cast<uint32_t>(whole.find_best(of_parts, parts, own) >> 32);
    if (key <= kOrderOfMinusInf) return;
    const Row row = {logits + static_cast<size_t>(r) * ld, vocab, logit_of(key), 1.0 / static_cast<double>(rules.temp), unit, 0.0};
    const double total = whole.find_total(row, of_parts, parts, own);
    const Reach reach(row, rules, total);
    if (rules.p < 1.0) {
        // the bin in which p of the weight is reached (without any, the lowest that has weight), and what lies in front of it
        u64 bins[kOwn], mine = 0;
        const u64* histogram = of.histogram + static_cast<size_t>(r) * kBins;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            bins[i] = histogram[kBins - 1 - static_cast<int>(threadIdx.x) * kOwn - i];
            mine += bins[i];
        }
        const u64 running = wave_running_u64(mine);
        if (lane == kWave - 1) s_sum[wave] = running;
        __syncthreads();
        u64 front, all;
        across_waves<kPartWaves>(s_sum, front, all);
        front += running - mine;
        const double limit = fmin(rules.p * total * unit, static_cast<double>(all));
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            // (one bin: what lies in front of it is below the limit, or nothing, and with it the limit is reached)
            if (bins[i] && (front == 0 || static_cast<double>(front) < limit) && static_cast<double>(front + bins[i]) >= limit) {
                s_bin = kBins - 1 - static_cast<int>(threadIdx.x) * kOwn - i;
                s_above = front;
            }
            front += bins[i];
        }
        __syncthreads();
    }
    const int cut_bin = s_bin;  // (-1: all are kept that min-p keeps)
    if (blockIdx.x == 0 && threadIdx.x == 0) of.head[2 * r + 1] = s_above;
    u64* list = of.list + static_cast<size_t>(r) * kList;
    for (int part = blockIdx.x; part < parts; part += gridDim.x) {
        if (threadIdx.x == 0) s_count = 0;
        __syncthreads();
        u64 sum = 0;
        const int next = part + gridDim.x < parts ? part + gridDim.x : part;
        const float now = largest;
        largest = chunks[next * kPartThreads];
        walk_chunk(row, now, part, reach, [&](float l, int i) {
            const int bin = bin_of(reach, l);
            if (bin < cut_bin) return;
            const u64 w = row.weight(l);
            if (w == 0) return;
            if (bin > cut_bin) {
                if (!(rules.m > 0.0 && row.share(l) < rules.m)) sum += w;
            } else {
                s_list[atomicAdd(&s_count, 1)] = place_of(l, i);
            }
        });
        sum = wave_sum_u64(sum);
        if (lane == 0) s_sum[wave] = sum;
        __syncthreads();
        u64 front;
        across_waves<kPartWaves>(s_sum, front, sum);
        const int count = s_count;
        if (threadIdx.x == 0) {
            of.kept[static_cast<size_t>(r) * parts + part] = sum;
            if (count) s_at = atomicAdd(&of.head[2 * r], static_cast<u64>(count));  // (the order in the list changes nothing)
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += kPartThreads)
            if (s_at + i < kList) list[s_at + i] = s_list[i];
    }
}

// ---------------------------------------------------------------- last launch
// The steps of a sorting network in which a wave's numbers, kOwn neighbours of each lane, are compared with those kApart places on and
// then half as far each time, down to the next one: in registers.  (Written out: a loop's branches took longer than its steps.)
template <int kOwn, int kApart>
__device__ __forceinline__ void merge_steps(uint32_t (&own)[kOwn], int first, int run) {
    uint32_t other[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        if constexpr (kApart < kOwn)
            other[i] = own[i ^ kApart];
        else
            other[i] = partner<kApart / kOwn>(own[i]);
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const bool smaller = (((first + i) & kApart) == 0) == (((first + i) & run) == 0);
        own[i] = smaller ? min(own[i], other[i]) : max(own[i], other[i]);
    }
    if constexpr (kApart > 1) merge_steps<kOwn, kApart / 2>(own, first, run);
}
template <int kOwn, int kRun>
__device__ __forceinline__ void sort_steps(uint32_t (&own)[kOwn], int first) {
    merge_steps<kOwn, kRun / 2>(own, first, kRun);
    if constexpr (kRun < kOwn * kWave) sort_steps<kOwn, kRun * 2>(own, first);
}

// keys[0 .. n) in ascending order; n up to kList, the room up to the next power of two (64 at least) is written.  Runs longer than a
// wave's numbers pass through LDS until they are not.  (Orders alone: equal logits are told apart by their index only at the cut.)
template <int kOwn>
__device__ void sort_held(uint32_t* keys, int n, int size) {
    uint32_t own[kOwn];
    const int first = threadIdx.x * kOwn;
    const bool idle = threadIdx.x / kWave * kWave * kOwn >= size;  // (a wave without numbers)
    if (!idle) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) own[i] = first + i < n ? keys[first + i] : ~0u;
        sort_steps<kOwn, 2>(own, first);
    }
    for (int run = 2 * kOwn * kWave; run <= size; run <<= 1) {
        for (int apart = run >> 1; apart >= kOwn * kWave; apart >>= 1) {
            __syncthreads();
            if (!idle) {
#pragma unroll
                for (int i = 0; i < kOwn; ++i) keys[first + i] = own[i];
            }
            __syncthreads();
            if (!idle) {
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    const uint32_t other = keys[(first + i) ^ apart];
                    const bool smaller = (((first + i) & apart) == 0) == (((first + i) & run) == 0);
                    own[i] = smaller ? min(own[i], other) : max(own[i], other);
                }
            }
        }
        if (!idle) merge_steps<kOwn, kOwn * kWave / 2>(own, first, run);
    }
    __syncthreads();
    if (!idle) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) keys[first + i] = own[i];
    }
    __syncthreads();
}
__device__ void sort_keys(uint32_t* keys, int n) {
    int size = kWave;
    while (size < n) size <<= 1;
    __syncthreads();
    if (size <= kThreads)
        sort_held<1>(keys, n, size);
    else if (size <= 2 * kThreads)
        sort_held<2>(keys, n, size);
    else
        sort_held<4>(keys, n, size);
}

// One wave's 64 numbers in ascending order.
template <int kRun, int kApart>
__device__ __forceinline__ void wave_sort_steps(u64& v) {
    const int lane = threadIdx.x % kWave;
    const u64 other = partner_u64<kApart>(v);
    const bool smaller = ((lane & kApart) == 0) == ((lane & kRun) == 0);
    v = (other < v) == smaller ? other : v;
    if constexpr (kApart > 1)
        wave_sort_steps<kRun, kApart / 2>(v);
    else if constexpr (kRun < kWave)
        wave_sort_steps<kRun * 2, kRun>(v);
}
__device__ __forceinline__ u64 wave_sort(u64 v) {
    wave_sort_steps<2, 1>(v);
    return v;
}

// Running sums in front of places: thread t has kPlaces of them, from t * kPlaces on.
constexpr int kPlaces = kList / kThreads;
__device__ __forceinline__ u64 sums_in_front(const u64 (&own)[kPlaces], u64* s_sum, u64& total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) mine += own[i];
    const u64 running = wave_running_u64(mine);
    __syncthreads();
    if (lane == kWave - 1) s_sum[wave] = running;
    __syncthreads();
    u64 front;
    across_waves<kWaves>(s_sum, front, total);
    return front + running - mine;
}
__device__ __forceinline__ u64 block_sum_u64(u64 v, u64* s_sum) {
    v = wave_sum_u64(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) s_sum[threadIdx.x / kWave] = v;
    __syncthreads();
    u64 front, total;
    across_waves<kWaves>(s_sum, front, total);
    return total;
}

// How far down a logit lies, in bins of 1/64 of a power of two: for distances of any scale.
__device__ __forceinline__ int octave_bin(float distance) {
    const int bin = static_cast<int>(__float_as_uint(distance) >> 17) - ((127 - 16) << 6);
    return bin < 0 ? 0 : bin < kBins - 1 ? bin : kBins - 1;
}

struct Shared {
    union {
        Histogram h;
        int hits[kList];             // chunks that pass
        struct {
            u64 segment[kMaxParts];  // the parts' weight
            uint32_t keys[kList];    // of the list, by size
        } cut;
    };
    union {
        u64 list[kList];
        Whole<kThreads> whole;
    };
    u64 sum[kWaves];
    int count, hit_count;
    int picked;  // what one wave draws alone (not in `count`, which the other waves may still have to read then)
};

// The smallest of the threads' first choices (kNone: none), the largest of their second ones (-1) if there is none.
constexpr int kNone = 0x7fffffff;
__device__ __forceinline__ int choose(int first, int second, Shared& s) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    // one number for both: a first choice counts more than any second one, and more the smaller it is
    u64 mine = first != kNone ? (1ull << 32) + static_cast<uint32_t>(kNone - first) : static_cast<uint32_t>(second + 1);
    mine = wave_most_u64(mine);
    __syncthreads();
    if (lane == 0) s.sum[wave] = mine;
    __syncthreads();
    mine = wave_most_u64(s.sum[lane % kWaves]);
    return mine >> 32 ? kNone - static_cast<int>(mine & 0xffffffffu) : static_cast<int>(mine) - 1;
}

// The place whose running sum passes the target, of thread t's kPlaces from t * kPlaces on (`front` in front of them); the last
// with any weight if none does, -1 without any.
__device__ __forceinline__ int pick_place(const u64 (&own)[kPlaces], u64 front, double target, Shared& s) {
    int mine = kNone, last = -1;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) {
        if (own[i] == 0) continue;
        last = threadIdx.x * kPlaces + i;
        front += own[i];
        if (mine == kNone && static_cast<double>(front) > target) mine = last;
    }
    return choose(mine, last, s);
}

// The draw from one part of the row, of what lies up to `cut` in its order; -1 without any weight.
__device__ int draw_from_part(const Row& row, Shared& s, int part, u64 before, double target, u64 cut) {
    u64 own[kPlaces], total;
    const int first = part * kPart + threadIdx.x * kPlaces;
    static_assert(kPart == kThreads * kPlaces, "a thread has four neighbours of a part");
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) {
        const float l = first + i < row.vocab ? row.logits[first + i] : -INFINITY;
        own[i] = place_of(l, first + i) <= cut ? row.weight(l) : 0;
    }
    const u64 front = before + sums_in_front(own, s.sum, total);
    const int place = pick_place(own, front, target, s);
    return place < 0 ? -1 : part * kPart + place;
}

// The part in which the running sum of s.cut.segment passes u times the whole, and its draw.  (A part whose numbers each round to no
// weight, though their sum has one, has nothing to draw: the next one then.)
__device__ int draw_from_segments(const Row& row, Shared& s, int parts, double u, u64 cut) {
    // every wave the same
    const int lane = threadIdx.x % kWave;
    u64 all = 0;
    for (int q = lane; q < parts; q += kWave) all += s.cut.segment[q];
    const double target = u * static_cast<double>(wave_sum_u64(all));
    int owner = 0;
    u64 before = 0, running = 0;
    for (int base = 0; base < parts; base += kWave) {
        const u64 own = base + lane < parts ? s.cut.segment[base + lane] : 0;
        const u64 sum = running + wave_running_u64(own);
        const u64 passed = __ballot(own && static_cast<double>(sum) > target), any = __ballot(own > 0);
        if (any) {
            const int which = passed ? __ffsll(passed) - 1 : 63 - __clzll(any);
            owner = base + which;
            const u64 front = sum - own;
            before = joined(__builtin_amdgcn_readlane(static_cast<int>(front & 0xffffffffu), which),
                            __builtin_amdgcn_readlane(static_cast<int>(front >> 32), which));
        }
        if (passed) break;
        running = last_lane(sum);
    }
    int picked = draw_from_part(row, s, owner, before, target, cut);
    for (int q = owner + 1; q < parts && picked < 0; ++q) picked = draw_from_part(row, s, q, 0, -1.0, cut);
    return picked;
}

// Which of a wave's weights, in the order of the lanes, passes u times their sum: its lane, or the last with any weight, or -1.
__device__ __forceinline__ int pick_lane(u64 weight, double u) {
    const u64 running = wave_running_u64(weight);
    const double target = u * static_cast<double>(last_lane(running));
    const u64 passed = __ballot(weight && static_cast<double>(running) > target), any = __ballot(weight > 0);
    return passed ? __ffsll(passed) - 1 : any ? 63 - __clzll(any) : -1;
}

// The cut of a list: of its n numbers by size the first k, of these the ones in front of which less than `limit` lies (p of what
// the k weigh, of_list; `above` lies in front of the list), of these the ones that weigh at least m (but never none).  The last
// kept place comes back (all threads; `front` of nothing: none is kept only with something above).
__device__ u64 cut_list(const Row& row, Shared& s, int n, int k, bool nucleus, bool of_list, double p_or_limit, double m, u64 above) {
    for (int i = threadIdx.x; i < n; i += kThreads) s.cut.keys[i] = static_cast<uint32_t>(s.list[i] >> 32);
    sort_keys(s.cut.keys, n);
    const int count = min(n, k), first = threadIdx.x * kPlaces;
    u64 own[kPlaces], total;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) own[i] = first + i < count ? row.weight(logit_of(~s.cut.keys[first + i])) : 0;
    u64 front = above + sums_in_front(own, s.sum, total);
    const double limit = of_list ? p_or_limit * static_cast<double>(total) : p_or_limit;
    int mine = 0;  // (what is kept is a prefix of all places, so the threads' numbers add up to it)
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) {
        if (first + i >= count) continue;
        const bool very_first = first + i == 0 && above == 0;
        const bool in_p = very_first || !nucleus || static_cast<double>(front) < limit;
        const bool in_m = very_first || !(m > 0.0) || row.share(logit_of(~s.cut.keys[first + i])) >= m;
        mine += in_p && in_m;
        front += own[i];
    }
    const int kept = static_cast<int>(block_sum_u64(mine, s.sum));
    if (kept == 0) return (static_cast<u64>(s.cut.keys[0]) << 32) - 1;
    // of the numbers equal to the last kept one only the first by index, if not all
    const uint32_t key = s.cut.keys[kept - 1];
    u64 counts = 0;  // the larger ones, and the equal ones
    for (int i = threadIdx.x; i < n; i += kThreads) counts += s.cut.keys[i] < key ? 1ull : s.cut.keys[i] == key ? 1ull << 32 : 0;
    counts = block_sum_u64(counts, s.sum);
    const int equal = static_cast<int>(counts >> 32), wanted = kept - static_cast<int>(counts & 0xffffffffu);
    if (wanted >= equal) return (static_cast<u64>(key) << 32) | 0xffffffffu;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 place = s.list[i];
        if (static_cast<uint32_t>(place >> 32) != key) continue;
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s.list[j] < place && static_cast<uint32_t>(s.list[j] >> 32) == key;
        if (rank == wanted - 1) s.sum[0] = place;
    }
    __syncthreads();
    const u64 cut = s.sum[0];
    __syncthreads();
    return cut;
}

// The draw from a list that holds the first of the row's order.
__device__ int draw_from_list(const Row& row, Shared& s, int n, int parts, const Rules& rules, double u) {
    if (n <= kWave) {  // one wave, a number to a lane: without a barrier
        if (threadIdx.x < kWave) {
            const int lane = threadIdx.x;
            const u64 place = wave_sort(lane < n ? s.list[lane] : ~0ull);
            const float l = logit_of(~static_cast<uint32_t>(place >> 32));
            const double share = lane < min(n, rules.k) ? row.share(l) : 0.0;
            u64 weight = static_cast<u64>(share * row.unit + 0.5);
            const u64 running = wave_running_u64(weight);
            const double limit = rules.p * static_cast<double>(last_lane(running));
            if (lane > 0 && ((rules.p < 1.0 && !(static_cast<double>(running - weight) < limit)) || (rules.m > 0.0 && share < rules.m))) weight = 0;
            const u64 kept = wave_sort(weight ? place << 32 | place >> 32 : ~0ull);  // by index
            weight = kept != ~0ull ? row.weight(logit_of(~static_cast<uint32_t>(kept))) : 0;
            const int which = pick_lane(weight, u);
            if (lane == max(0, which)) s.picked = which < 0 ? -1 : static_cast<int>(kept >> 32);
        }
        __syncthreads();
        return s.picked;
    }
    const u64 cut = cut_list(row, s, n, rules.k, rules.p < 1.0, true, rules.p, rules.m, 0);
    // where the kept ones lie: the parts' sums
    for (int q = threadIdx.x; q < parts; q += kThreads) s.cut.segment[q] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 place = s.list[i];
        if (place <= cut) atomicAdd(&s.cut.segment[static_cast<uint32_t>(place) / kPart], row.weight(logit_of(~static_cast<uint32_t>(place >> 32))));
    }
    __syncthreads();
    return draw_from_segments(row, s, parts, u, cut);
}

// The draw under top-k; -2: too many numbers pass the bound.
__device__ int draw_of_k(const Row& row, Shared& s, const float* chunks, int chunk_count, const Rules& rules, double u) {
    constexpr int kRound = 16;  // chunks of a thread that are read at once (all of them, up to 262,144 tokens)
    const auto bin_of = [&](float l) { return kBins - 1 - octave_bin(l == row.best ? 0.f : row.best - l); };
    const int rounds = (chunk_count + kRound * kThreads - 1) / (kRound * kThreads);
    float largest[kRound];
    const auto read = [&](int round) {
#pragma unroll
        for (int j = 0; j < kRound; ++j) {
            const int c = (round * kRound + j) * kThreads + threadIdx.x;
            largest[j] = c < chunk_count ? chunks[c] : -INFINITY;
        }
    };
    read(0);
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
        s.h.weight[b] = 0;
        s.h.count[b] = 0;
    }
    if (threadIdx.x == 0) s.count = s.hit_count = 0;
    __syncthreads();
    for (int round = 0; round < rounds; ++round) {
        if (round) read(round);
#pragma unroll
        for (int j = 0; j < kRound; ++j)
            if (largest[j] > -INFINITY) atomicAdd(&s.h.count[bin_of(largest[j])], 1);
    }
    __syncthreads();
    cross<true>(s.h, rules.k, 0.0);  // (fewer chunks than k: the last bin that has any, and then all below it)
    const int found = s.h.above + s.h.count[s.h.bin] >= static_cast<u64>(rules.k) ? s.h.bin : -1;
    __syncthreads();
    const auto passes = [&](float l) { return l > -INFINITY && bin_of(l) >= found; };
    for (int round = 0; round < rounds; ++round) {
        if (rounds > 1) read(round);
#pragma unroll
        for (int j = 0; j < kRound; ++j)
            if (passes(largest[j])) {
                const int at = atomicAdd(&s.hit_count, 1);
                if (at < kList) s.hits[at] = (round * kRound + j) * kThreads + threadIdx.x;
            }
    }
    __syncthreads();
    const int hits = s.hit_count;
    if (hits > kList) return -2;  // (each has a number that passes)
    const bool lines = (reinterpret_cast<uintptr_t>(row.logits) & 15) == 0;
    for (int item = threadIdx.x; item < hits * 4; item += kThreads) {
        const int c = s.hits[item / 4], first = c / kPartThreads * kPart + c % kPartThreads * 4 + item % 4 * kPartThreads * 4;
        float l[4];
        if (lines && first + 3 < row.vocab) {
            const float4 v = *reinterpret_cast<const float4*>(row.logits + first);
            l[0] = v.x;
            l[1] = v.y;
            l[2] = v.z;
            l[3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) l[e] = first + e < row.vocab ? row.logits[first + e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (passes(l[e])) {
                const int at = atomicAdd(&s.count, 1);
                if (at < kList) s.list[at] = place_of(l[e], first + e);
            }
    }
    __syncthreads();
    const int n = s.count;
    if (n > kList) return -2;
    return draw_from_list(row, s, n, chunk_count / kPartThreads, rules, u);
}

// What the launches before left of a tallied row, asked for before anything waits.
struct Tallied {
    u64 listed, above, list[kPlaces];
    __device__ __forceinline__ void ask(Shared& s, const PartOf& of, int r, int parts) {
        listed = of.head[2 * r];
        above = of.head[2 * r + 1];
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) list[i] = of.list[static_cast<size_t>(r) * kList + i * kThreads + threadIdx.x];  // (the first `listed` count)
        for (int q = threadIdx.x; q < parts; q += kThreads) s.cut.segment[q] = of.kept[static_cast<size_t>(r) * parts + q];
    }
};

// The draw of a row that was tallied; -2: the cut's bin holds more than its list.
__device__ int draw_of_tally(Row& row, Shared& s, const Tallied& tallied, int parts, const Rules& rules, double total, double u) {
    if (rules.p < 1.0 && tallied.listed > kList) return -2;
    const int n = rules.p < 1.0 ? static_cast<int>(tallied.listed) : 0;
    const double limit = rules.p * total * row.unit;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i)
        if (i * kThreads + static_cast<int>(threadIdx.x) < n) s.list[i * kThreads + threadIdx.x] = tallied.list[i];
    u64 cut = ~0ull;  // the last kept place
    __syncthreads();
    if (n > 0) {
        cut = cut_list(row, s, n, n, true, false, limit, rules.m, tallied.above);
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 place = s.list[i];
            if (place <= cut) atomicAdd(&s.cut.segment[static_cast<uint32_t>(place) / kPart], row.weight(logit_of(~static_cast<uint32_t>(place >> 32))));
        }
        __syncthreads();
    }
    row.least = rules.m;
    return draw_from_segments(row, s, parts, u, cut);
}

__global__ void __launch_bounds__(kThreads)
rules_draw_kernel(const float* __restrict__ logits, const float* __restrict__ temperature, const float* __restrict__ uniform,
                  const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p, PartOf of,
                  int* __restrict__ out, int vocab, long ld, int parts, double unit) {
    __shared__ Shared s;
    const int r = blockIdx.x;
    const PartOf::Largest* of_parts = of.part + static_cast<size_t>(r) * parts;
    const Rules rules(temperature, top_k, top_p, min_p, r, vocab);
    const PartOf::Largest own = s.whole.first_of(of_parts, parts);
    Tallied tallied;
    if (rules.tallied()) tallied.ask(s, of, r, parts);
    const u64 best = s.whole.find_best(of_parts, parts, own);
    const uint32_t best_key = static_cast<uint32_t>(best >> 32);
    const int best_idx = best_key > kOrderOfMinusInf ? 0x7fffffff - static_cast<int>(best & 0xffffffffu) : 0;
    if (!rules.draws() || best_key <= kOrderOfMinusInf) {
        if (threadIdx.x == 0) out[r] = best_idx;
        return;
    }
    Row row = {logits + static_cast<size_t>(r) * ld, vocab, logit_of(best_key), 1.0 / static_cast<double>(rules.temp), unit, 0.0};
    const double u = static_cast<double>(uniform[r]);
    __syncthreads();
    int picked = -2;
    if (rules.k > 0) {
        picked = draw_of_k(row, s, of.chunk + static_cast<size_t>(r) * parts * kPartThreads, parts * kPartThreads, rules, u);
    } else {
        const double total = s.whole.find_total(row, of_parts, parts, own);
        if (rules.tallied()) {
            __syncthreads();
            picked = draw_of_tally(row, s, tallied, parts, rules, total, u);
        } else {
            __syncthreads();
            for (int q = threadIdx.x; q < parts; q += kThreads) s.cut.segment[q] = static_cast<u64>(s.whole.sum[q] * unit + 0.5);
            __syncthreads();
            picked = draw_from_segments(row, s, parts, u, ~0ull);
        }
    }
    if (picked == -2) {
        __syncthreads();
        row.least = 0.0;
        picked = draw_by_bits(row, s.h, s.sum, rules.k, rules.p, rules.m, u);
    }
    if (threadIdx.x == 0) out[r] = picked < 0 ? best_idx : picked;
}

}  // namespace

// top_k, top_p and min_p may each be null: that rule is off in every row.  work, aligned to 8 bytes: rows * ceil(vocab / 4096) * 1,048
// bytes, and rows * 49,168 behind them where top_p or min_p is given.  spread: the workgroups that share a row under these.
CIE_API int cie_sample_rules(void* stream, const float* logits, const float* temperature, const float* uniform, const int* top_k,
                             const float* top_p, const float* min_p, int* out, void* work, int rows, int vocab, long ld, int spread) {
    if (rows < 0 || vocab <= 0 || ld < vocab || rows > 65535 || vocab > kMaxParts * kPart || spread < 1 || !logits || !temperature ||
        !uniform || !out || !work)
        return CIE_BAD_ARGUMENT;
    if (rows == 0) return CIE_OK;
    int bits = 0;
    while ((1L << bits) < vocab) ++bits;
    const double unit = static_cast<double>(1L << (62 - bits < 51 ? 62 - bits : 51));
    const int parts = (vocab + kPart - 1) / kPart;
    const size_t all = static_cast<size_t>(rows) * parts;
    PartOf of;
    of.part = static_cast<PartOf::Largest*>(work);
    of.kept = reinterpret_cast<u64*>(of.part + all);
    of.chunk = reinterpret_cast<float*>(of.kept + all);
    of.histogram = reinterpret_cast<u64*>(of.chunk + all * kPartThreads);
    of.list = of.histogram + static_cast<size_t>(rows) * kBins;
    of.head = of.list + static_cast<size_t>(rows) * kList;
    hipStream_t s = static_cast<hipStream_t>(stream);
    rules_parts_kernel<<<dim3(parts, rows), kPartThreads, 0, s>>>(logits, temperature, top_k, top_p, min_p, of, vocab, ld);
    if (cie_after_launch() != CIE_OK) return CIE_LAUNCH_FAILED;
    if (top_p || min_p) {
        const dim3 grid(spread < parts ? spread : parts, rows);
        if (top_p) {
            rules_tally_kernel<<<grid, kPartThreads, 0, s>>>(logits, temperature, top_k, top_p, min_p, of, vocab, ld, parts, unit);
            if (cie_after_launch() != CIE_OK) return CIE_LAUNCH_FAILED;
        }
        rules_collect_kernel<<<grid, kPartThreads, 0, s>>>(logits, temperature, top_k, top_p, min_p, of, vocab, ld, parts, unit);
        if (cie_after_launch() != CIE_OK) return CIE_LAUNCH_FAILED;
    }
    rules_draw_kernel<<<rows, kThreads, 0, s>>>(logits, temperature, uniform, top_k, top_p, min_p, of, out, vocab, ld, parts, unit);
    return cie_after_launch();
}
