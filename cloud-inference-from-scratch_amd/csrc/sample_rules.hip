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
// Two launches.  The first reads the logits once, in parts that fill the GPU: the largest of each part, of each 16 numbers (a
// chunk), and, for rows that draw from all tokens or from a share of all weight, the part's sum of weights.  The second has a
// workgroup for each row, which with that rarely needs the row again: the k-th largest of the chunks' largest is a bound
// that the k largest logits reach, a share p of the weight cannot reach down to tokens that weigh less than (1 - p) / vocab of
// the sum, min-p names its bound itself.  It gathers what passes the bound from the few chunks whose largest does, sorts it, and
// cuts and draws in LDS.  Where more than kList numbers pass (flat rows), the row is walked: a histogram of its weights, then
// the numbers of the one bin that holds the cut.  Rows that defeat that too (thousands of equal logits at the cut) are cut by the
// bits of their logits.
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

    __device__ __forceinline__ double share(float l) const {
        if (!(l > -INFINITY)) return 0.0;
        const double w = l == best ? 1.0 : exp((static_cast<double>(l) - static_cast<double>(best)) * inv_t);
        return w >= 0.0 ? w : 0.0;  // (an infinite temperature and an infinite distance: none)
    }
    __device__ __forceinline__ u64 weight(float l) const {
        const double w = share(l);
        return w >= least ? static_cast<u64>(w * unit + 0.5) : 0;
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
    u64 wave_weight[kWaves];
    int wave_count[kWaves];
    int bin;
    u64 above_weight;
    int above_count;
};

// The bin, from the largest digit down, in which the running count reaches `need` (by_count), or the running weight `limit`;
// the last bin that counts (weighs) anything if none does.  The sums of the bins in front of it are left in `h`.
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
        if (reached && (by_count ? h.count[bin] > 0 : h.weight[bin] > 0)) atomicMax(&h.bin, bin);
        before_w = after_w;
        before_c = after_c;
    }
    __syncthreads();
    int found = h.bin;
    __syncthreads();
    if (found < 0) {  // (a limit that rounding left out of reach)
        const bool low = by_count ? h.count[lo] > 0 : h.weight[lo] > 0, high = by_count ? h.count[hi] > 0 : h.weight[hi] > 0;
        if (low || high) atomicMax(&h.bin, kBins - (low ? lo : hi));
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

struct PartOf {
    u64* best;       // [rows, parts] order << 32 | (0x7fffffff - index) of the largest
    double* sum;     // [rows, parts] sum of exp((l - the part's largest) / T), where the row asks for it
    float* chunk;    // [rows, parts * kPartThreads] the largest of each thread's 16; -inf where there is none
};

__device__ __forceinline__ bool wants_sum(float temp, int k, int vocab) { return temp > 0.f && !(k > 0 && k < vocab); }

__global__ void __launch_bounds__(kPartThreads)
rules_parts_kernel(const float* __restrict__ logits, const float* __restrict__ temperature, const int* __restrict__ top_k, PartOf of,
                   int vocab, long ld) {
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
    const float largest = key <= kOrderOfMinusInf ? -INFINITY : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    of.chunk[(static_cast<size_t>(r) * gridDim.x + part) * kPartThreads + threadIdx.x] = largest;
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) {
        const u64 other = __shfl_xor(best, offset, kWave);
        best = other > best ? other : best;
    }
    if (lane == 0) s_best[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPartWaves; ++w) best = s_best[w] > best ? s_best[w] : best;
    if (threadIdx.x == 0) of.best[static_cast<size_t>(r) * gridDim.x + part] = best;
    const float temp = temperature[r];
    if (!wants_sum(temp, top_k ? top_k[r] : 0, vocab)) return;
    key = static_cast<uint32_t>(best >> 32);
    double sum = 0.0;
    if (key > kOrderOfMinusInf) {
        const Row scaled = {row, vocab, __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key), 1.0 / static_cast<double>(temp), 1.0, 0.0};
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += scaled.share(l[i]);
    }
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset, kWave);
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int w = 0; w < kPartWaves; ++w) sum += s_sum[w];
        of.sum[static_cast<size_t>(r) * gridDim.x + part] = sum;
    }
}

// ---------------------------------------------------------------- second launch
constexpr int kList = 4096;

// What a row's numbers are sorted by: the larger logit first, then the lower index.
__device__ __forceinline__ u64 place_of(float l, int i) { return (static_cast<u64>(~order_of(l)) << 32) | static_cast<uint32_t>(i); }
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// list[0 .. n) in ascending order; n up to kList, the list's room up to the next power of two is written.
__device__ void sort_list(u64* list, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = ~0ull;
    __syncthreads();
    for (int run = 2; run <= size; run <<= 1)
        for (int apart = run >> 1; apart > 0; apart >>= 1) {
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int i = 2 * t - (t & (apart - 1)), j = i + apart;
                const u64 a = list[i], b = list[j];
                if ((a > b) == ((i & run) == 0)) {
                    list[i] = b;
                    list[j] = a;
                }
            }
            __syncthreads();
        }
}

// Running sums in front of list places: thread t has the kList / kThreads places from t * 4 on.
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
    u64 front = running - mine;
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) front += s_sum[w];
        total += s_sum[w];
    }
    return front;
}

// How far down a logit lies, in bins of 1/64 of a power of two: for distances of any scale.
__device__ __forceinline__ int octave_bin(float distance) {
    const int bin = static_cast<int>(__float_as_uint(distance) >> 17) - ((127 - 16) << 6);
    return bin < 0 ? 0 : bin < kBins - 1 ? bin : kBins - 1;
}

struct Shared {
    Histogram h;
    u64 list[kList];
    u64 sum[kWaves], segment[kWaves];
    int count, kept;
    int picked;
};

// The numbers of the row that `passes` takes (it takes all that are larger than one it takes), from the chunks whose largest
// does; more than kList: as many as there are, and no list.
template <typename F>
__device__ int gather_list(const Row& row, const float* chunks, int chunk_count, Shared& s, F passes) {
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    for (int c = threadIdx.x; c < chunk_count; c += kThreads) {
        if (!passes(chunks[c])) continue;
        const int first = c / kPartThreads * kPart + c % kPartThreads * 4;
        for (int q = 0; q < 4; ++q)
            for (int e = 0; e < 4; ++e) {
                const int i = first + q * kPartThreads * 4 + e;
                if (i >= row.vocab) continue;
                const float l = row.logits[i];
                if (!passes(l)) continue;
                const int at = atomicAdd(&s.count, 1);
                if (at < kList) s.list[at] = place_of(l, i);
            }
    }
    __syncthreads();
    return s.count;
}

// The draw from a list that holds the first n of the row's order: the first k of them (k = 0: all), then those in front of which
// less than `limit` lies (or p of what the k weigh, of_list), then min-p.
__device__ int draw_from_list(const Row& row, Shared& s, int n, int k, bool nucleus, bool of_list, double p_or_limit, double m, double u) {
    sort_list(s.list, n);
    if (k > 0 && k < n) n = k;
    u64 own[kPlaces], total;
    const int first = threadIdx.x * kPlaces;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i)
        own[i] = first + i < n ? row.weight(logit_of(~static_cast<uint32_t>(s.list[first + i] >> 32))) : 0;
    u64 front = sums_in_front(own, s.sum, total);
    const double limit = of_list ? p_or_limit * static_cast<double>(total) : p_or_limit;
    if (threadIdx.x == 0) s.kept = 0;
    __syncthreads();
    int kept = 0;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) {
        if (first + i >= n) break;
        const float l = logit_of(~static_cast<uint32_t>(s.list[first + i] >> 32));
        if (first + i > 0 && nucleus && !(static_cast<double>(front) < limit)) break;
        if (first + i > 0 && m > 0.0 && row.share(l) < m) break;
        front += own[i];
        kept = first + i + 1;
    }
    if (kept) atomicMax(&s.kept, kept);
    __syncthreads();
    n = s.kept;
    // the kept ones by index, their logits' order beside it
    u64 turned[kPlaces];
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) turned[i] = first + i < n ? s.list[first + i] << 32 | s.list[first + i] >> 32 : 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPlaces; ++i)
        if (first + i < n) s.list[first + i] = turned[i];
    sort_list(s.list, n);
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) own[i] = first + i < n ? row.weight(logit_of(~static_cast<uint32_t>(s.list[first + i]))) : 0;
    front = sums_in_front(own, s.sum, total);
    const double target = u * static_cast<double>(total);
    if (threadIdx.x == 0) s.picked = -1;
    __syncthreads();
    // the first place whose running sum passes the target, else the last with any weight
    int mine = -1, last = -1;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) {
        if (own[i] == 0) continue;
        last = first + i;
        front += own[i];
        if (mine < 0 && static_cast<double>(front) > target) mine = first + i;
    }
    if (mine >= 0) atomicMax(&s.picked, 2 * kList - mine);
    if (last >= 0) atomicMax(&s.picked, last);
    __syncthreads();
    const int place = s.picked >= kList ? 2 * kList - s.picked : s.picked;
    return place < 0 ? -1 : static_cast<int>(s.list[place] >> 32);
}

// The draw from a share of all weight that is too many tokens for a list: a histogram of the weights over equal bins of
// (max - l) / T, of which the one that holds the cut goes to the list.  -2: it holds more than the list.
__device__ int draw_from_row(Row& row, Shared& s, double limit, double m, double u) {
    constexpr double kBinsOfUnit = 64.0;  // (beyond 32 units, where 2 million tokens weigh less than the least 1 - p, all is one bin)
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const auto bin_of = [&](float l) {
        const double at = l == row.best ? 0.0 : (static_cast<double>(row.best) - static_cast<double>(l)) * row.inv_t * kBinsOfUnit;
        return kBins - 1 - (at < kBins - 1 ? static_cast<int>(at) : kBins - 1);
    };
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
        s.h.weight[b] = 0;
        s.h.count[b] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < row.vocab; i += kThreads) {
        const float l = row.logits[i];
        const u64 w = row.weight(l);
        if (w) atomicAdd(&s.h.weight[bin_of(l)], w);
    }
    __syncthreads();
    cross(s.h, false, 0, limit);
    const int cut_bin = s.h.bin;
    const double above = static_cast<double>(s.h.above_weight);
    if (threadIdx.x == 0) s.count = 0;
    if (threadIdx.x < kWaves) s.segment[threadIdx.x] = 0;
    __syncthreads();
    const int stretch = ((row.vocab + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
    u64 sum = 0;
    const int to = min(row.vocab, (wave + 1) * stretch);
    for (int i = wave * stretch + lane; i < to; i += kWave) {
        const float l = row.logits[i];
        const u64 w = row.weight(l);
        if (w == 0) continue;
        const int bin = bin_of(l);
        if (bin > cut_bin) {
            if (!(m > 0.0 && row.share(l) < m)) sum += w;
        } else if (bin == cut_bin) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kList) s.list[at] = place_of(l, i);
        }
    }
    sum = wave_sum_u64(sum);
    if (lane == 0) s.segment[wave] = sum;
    __syncthreads();
    const int n = s.count;
    if (n > kList) return -2;
    sort_list(s.list, n);
    u64 own[kPlaces], total;
    const int first = threadIdx.x * kPlaces;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i)
        own[i] = first + i < n ? row.weight(logit_of(~static_cast<uint32_t>(s.list[first + i] >> 32))) : 0;
    u64 front = sums_in_front(own, s.sum, total);
    if (threadIdx.x == 0) s.kept = 0;
    __syncthreads();
    row.least = m;
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) {
        if (first + i >= n || !(first + i == 0 && above == 0.0) && !(above + static_cast<double>(front) < limit)) break;
        front += own[i];
        atomicMax(&s.kept, first + i + 1);
        const u64 w = row.weight(logit_of(~static_cast<uint32_t>(s.list[first + i] >> 32)));
        if (w) atomicAdd(&s.segment[static_cast<uint32_t>(s.list[first + i]) / stretch], w);
    }
    __syncthreads();
    // (nothing of the bin is kept only if rounding says so: then the cut lies in front of it)
    const u64 last = s.kept > 0 ? s.list[s.kept - 1] : n > 0 ? s.list[0] - 1 : 0;
    u64 all = 0;
    for (int w = 0; w < kWaves; ++w) all += s.segment[w];
    const double target = u * static_cast<double>(all);
    int owner = 0;
    u64 running = 0, before = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (s.segment[w] == 0) continue;
        owner = w;
        before = running;
        running += s.segment[w];
        if (static_cast<double>(running) > target) break;
    }
    return seek(owner * stretch, min(row.vocab, (owner + 1) * stretch), before, target, false, s.sum, [&](int i) -> u64 {
        const float l = row.logits[i];
        return place_of(l, i) <= last ? row.weight(l) : 0;
    });
}

__global__ void __launch_bounds__(kThreads)
rules_draw_kernel(const float* __restrict__ logits, const float* __restrict__ temperature, const float* __restrict__ uniform,
                  const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p, PartOf of,
                  int* __restrict__ out, int vocab, long ld, int parts, double unit) {
    __shared__ Shared s;
    const int r = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const u64* part_best = of.best + static_cast<size_t>(r) * parts;
    const double* part_sum = of.sum + static_cast<size_t>(r) * parts;
    const float* chunks = of.chunk + static_cast<size_t>(r) * parts * kPartThreads;

    // the largest logit and its first index
    u64 best = 0;
    for (int p = threadIdx.x; p < parts; p += kThreads) best = part_best[p] > best ? part_best[p] : best;
#pragma unroll
    for (int offset = kWave / 2; offset > 0; offset >>= 1) {
        const u64 other = __shfl_xor(best, offset, kWave);
        best = other > best ? other : best;
    }
    if (lane == 0) s.sum[wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) best = s.sum[w] > best ? s.sum[w] : best;
    __syncthreads();
    const uint32_t best_key = static_cast<uint32_t>(best >> 32);
    const int best_idx = best_key > kOrderOfMinusInf ? 0x7fffffff - static_cast<int>(best & 0xffffffffu) : 0;
    const float temp = temperature[r];
    if (!(temp > 0.f) || best_key <= kOrderOfMinusInf) {
        if (threadIdx.x == 0) out[r] = best_idx;
        return;
    }
    Row row = {logits + static_cast<size_t>(r) * ld, vocab, logit_of(best_key), 1.0 / static_cast<double>(temp), unit, 0.0};
    const int k = top_k && top_k[r] > 0 && top_k[r] < vocab ? top_k[r] : 0;
    const double p = top_p && top_p[r] < 1.f ? (top_p[r] > 0.f ? static_cast<double>(top_p[r]) : 0.0) : 1.0;  // (NaN: off)
    const double m = min_p && min_p[r] > 0.f ? (min_p[r] < 1.f ? static_cast<double>(min_p[r]) : 1.0) : 0.0;  // (the largest stays)
    const double u = static_cast<double>(uniform[r]);
    const int chunk_count = parts * kPartThreads;

    int picked = -2;
    if (k > 0) {
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            s.h.weight[b] = 0;
            s.h.count[b] = 0;
        }
        __syncthreads();
        const auto bin_of = [&](float l) { return kBins - 1 - octave_bin(l == row.best ? 0.f : row.best - l); };
        for (int c = threadIdx.x; c < chunk_count; c += kThreads)
            if (chunks[c] > -INFINITY) atomicAdd(&s.h.count[bin_of(chunks[c])], 1);
        __syncthreads();
        cross(s.h, true, k, 0.0);  // (fewer chunks than k: the last bin that has any, and then all below it)
        const int found = s.h.bin;
        const bool enough = s.h.above_count + s.h.count[found] >= k;
        const int n = gather_list(row, chunks, chunk_count, s, [&](float l) { return l > -INFINITY && (!enough || bin_of(l) >= found); });
        if (n <= kList) picked = draw_from_list(row, s, n, k, p < 1.0, true, p, m, u);
    } else {
        double total = 0.0, owner_before = 0.0;
        int owner = 0;
        double* const part = reinterpret_cast<double*>(s.list);  // what each part weighs
        for (int q = threadIdx.x; q < parts; q += kThreads) {
            const uint32_t key = static_cast<uint32_t>(part_best[q] >> 32);
            part[q] = key > kOrderOfMinusInf ? part_sum[q] * row.share(logit_of(key)) : 0.0;
        }
        __syncthreads();
        for (int q = 0; q < parts; ++q) total += part[q];  // (in order, in every thread)
        // what weighs less than this is not kept, however it is shared out; as a distance from the largest, a little rounded up
        const double least = p < 1.0 ? fmax((1.0 - p) * total / vocab, m) : m;
        if (least > 0.0) {
            const double reach = -log(least) * static_cast<double>(temp) * (1.0 + 1e-9) + 1e-30;
            const auto passes = [&](float l) {
                return l > -INFINITY && (l == row.best || static_cast<double>(row.best) - static_cast<double>(l) <= reach);
            };
            const int n = gather_list(row, chunks, chunk_count, s, passes);
            if (n <= kList)
                picked = draw_from_list(row, s, n, 0, p < 1.0, false, p * total * unit, m, u);
            else if (p < 1.0)
                picked = draw_from_row(row, s, p * total * unit, m, u);
            else {
                row.least = m;
                picked = seek(0, vocab, 0, u, true, s.sum, [&](int i) -> u64 { return row.weight(row.logits[i]); });
            }
        } else {
            const double target = u * total;
            double running = 0.0;
            for (int q = 0; q < parts; ++q) {
                if (part[q] * unit < 0.5) continue;
                owner = q;
                owner_before = running;
                running += part[q];
                if (running > target) break;
            }
            // (a part whose numbers each round to no weight has nothing to draw: the next one then)
            picked = -1;
            for (int q = owner; q < parts && picked < 0; ++q)
                picked = seek(q * kPart, min(vocab, (q + 1) * kPart), 0, q == owner ? (target - owner_before) * unit : -1.0, false, s.sum,
                              [&](int i) -> u64 { return row.weight(row.logits[i]); });
        }
    }
    if (picked == -2) picked = draw_by_bits(row, s.h, s.sum, k, p, m, u);
    if (threadIdx.x == 0) out[r] = picked < 0 ? best_idx : picked;
}

}  // namespace

// top_k, top_p and min_p may each be null: that rule is off in every row.  work: rows * ceil(vocab / 4096) * 1040 bytes, aligned to 8.
CIE_API int cie_sample_rules(void* stream, const float* logits, const float* temperature, const float* uniform, const int* top_k,
                             const float* top_p, const float* min_p, int* out, void* work, int rows, int vocab, long ld) {
    if (rows < 0 || vocab <= 0 || ld < vocab || rows > 65535 || vocab > kList * kPart || !logits || !temperature || !uniform || !out || !work)
        return CIE_BAD_ARGUMENT;
    if (rows == 0) return CIE_OK;
    int bits = 0;
    while ((1L << bits) < vocab) ++bits;
    const double unit = static_cast<double>(1L << (62 - bits < 51 ? 62 - bits : 51));
    const int parts = (vocab + kPart - 1) / kPart;
    const size_t all = static_cast<size_t>(rows) * parts;
    PartOf of;
    of.best = static_cast<u64*>(work);
    of.sum = reinterpret_cast<double*>(of.best + all);
    of.chunk = reinterpret_cast<float*>(of.sum + all);
    hipStream_t s = static_cast<hipStream_t>(stream);
    rules_parts_kernel<<<dim3(parts, rows), kPartThreads, 0, s>>>(logits, temperature, top_k, of, vocab, ld);
    if (cie_after_launch() != CIE_OK) return CIE_LAUNCH_FAILED;
    rules_draw_kernel<<<rows, kThreads, 0, s>>>(logits, temperature, uniform, top_k, top_p, min_p, of, out, vocab, ld, parts, unit);
    return cie_after_launch();
}
