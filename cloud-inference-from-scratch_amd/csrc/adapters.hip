// Low-rank adapters of many requests beside a shared projection:
//   out[t, c] = into[t, c] + scale[a] * sum_r up[a][c, r] * h[t, p(c) R + r],   h[t, j] = sum_k down[a][j, k] x[t, k],
// a = adapter[t]; a row whose adapter is none (negative, or one that there is not) keeps its numbers.  A site stacks P
// projections that read the same rows (q, k and v; gate and up): `down` [A, P R, K] has R rows for each, the columns of `out`
// fall into P pieces, and p(c) is the piece of column c.
//
// The sums are float32, the result is rounded once (h on its way onto rows of bfloat16 keeps 16 bits).  Two launches: `down` (K
// long, few columns; K cut into parts whose float32 sums lie side by side, so that few rows still fill the GPU) and `up` (R long, many
// columns; it adds the parts in order).  Rows are taken in tiles of consecutive ones; what a tile does is done once for each
// adapter that its rows have, on these rows alone, gathered into matrix-core tiles of 16.  So no plan of who has which adapter is
// made on the host, a row's sums do not depend on its neighbours, and a prompt (one adapter) and 64 requests (16 of them) run
// through the same code.
//
// Measured in captured chains of calls, both products, with what has to be read and written: one row of 2,048 and 2,560 columns, rank
// 16: 8.2 us (0.3 MB); 64 rows of 16 adapters, 2,048 and 22,016, rank 16: 12.4 us (19 MB); 24 rows of 8, 18,944 and 3,584, rank 32:
// 11.1 us (11.5 MB); 2,048 rows of two, 3,584 and 37,888, rank 64: 100 us (339 MB), onto the float32 stream 18,944 and 3,584 94 us.
// (A kernel's own time under the profiler, which the comments at the kernels give, is some half a us longer, of the last ones a tenth.)
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

// ---------------------------------------------------------------- tiles
typedef unsigned long long u64;
typedef float quad_t __attribute__((ext_vector_type(4)));
typedef __bf16 octet_t __attribute__((ext_vector_type(8)));
typedef __bf16 half_octet_t __attribute__((ext_vector_type(4)));

// What a lane hands to a matrix instruction: 16 bytes, `kLane` numbers of one row (lane % 16) that lie together (place
// lane / 16).  Both operands take their k in the same order, so which k an instruction calls which does not matter.
template <typename T>
struct Operand;
template <>
struct Operand<bf16_t> {
    typedef octet_t type;
    static constexpr int kLane = 8;
    static __device__ __forceinline__ quad_t mac(type a, type b, quad_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Operand<float> {
    typedef quad_t type;
    static constexpr int kLane = 4;
    static __device__ __forceinline__ quad_t mac(type a, type b, quad_t c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};
constexpr int kQuarters = 4;  // a wave's lanes hold 4 stretches of kLane k
constexpr int kWaves = kThreads / kWave;
constexpr int kTile = 16;
constexpr int kGroup = 4;
constexpr int kXcds = 8;

// Which lanes' rows have the adapter of this one's (those without an adapter belong together): a ballot for each bit of the numbers.
// (One adapter after the other, with a ballot and a readlane for each, took 2 of 8 us where 64 rows have 16.)
__device__ __forceinline__ u64 rows_of_same(int id, bool present, int adapters) {
    const u64 with = __ballot(present && id >= 0), without = __ballot(present && id < 0);
    u64 same = id >= 0 ? with : without;
    const int numbers = with & (with - 1) ? adapters - 1 : 0;  // (a row alone needs none)
    for (int bit = 0; numbers >> bit; ++bit) {
        const bool set = (id >> bit) & 1;
        const u64 ones = __ballot(set);
        same &= set ? ones : ~ones;
    }
    return present ? same : 0;
}
__device__ __forceinline__ u64 lanes_below() { return (1ull << (threadIdx.x % kWave)) - 1; }
// The sum of the lanes up to each one.
template <int kControl, int kRows>
__device__ __forceinline__ int moved(int v) {
    return __builtin_amdgcn_update_dpp(0, v, kControl, kRows, 0xf, false);
}
__device__ __forceinline__ int wave_running(int v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    return v + moved<0x143, 0xc>(v);
}

// The rows of a tile that have one adapter: lane i learns the i-th of them.
struct Gathered {
    int adapter, count, row;
};
__device__ __forceinline__ Gathered gather(int id, u64 mine) {
    const int lane = threadIdx.x % kWave;
    Gathered g;
    g.adapter = __builtin_amdgcn_readlane(id, __ffsll(mine) - 1);
    g.count = __popcll(mine);
    // (the others go behind them, so that every lane is sent exactly one row)
    const int place = (mine >> lane) & 1 ? __popcll(mine & lanes_below()) : g.count + __popcll(~mine & lanes_below());
    g.row = __builtin_amdgcn_ds_permute(place * 4, lane);
    return g;
}

// h_part[s, t, j]: the sums of part s of K.  grid: (parts, row tiles, column groups x slots).  A workgroup takes every
// `slots`-th of its tile's adapters.  K falls into chunks whose length depends on K alone; four waves share a chunk's k and join
// their sums through LDS, chunks are added one after the other in groups of kGroup, and the groups one after the other.  A part is
// one chunk (few rows: as many workgroups as there are) or a group of them (many rows: fewer sums to write and read): either
// way h is the same sum in the same order, whatever rows are beside it.  Few rows are bound by the way to their first result (one row
// of 2,048 at rank 16 x 3: 4.0 us; 24 rows of 8 adapters, K 18,944: 6.1 us for 11 MB of weights); 2,048 rows of 3,584 at rank 64 x 2,
// 22.6 us, by the waits of the one workgroup that each CU has (59 MB through L2: the rows for two column groups, the weights for
// 32 row tiles; 83 TFLOP/s).  More workgroups would mean more parts to write and to add, which costs the second product more.
template <typename T, int C, int R>
__device__ __forceinline__ void down_rows(const Gathered& g, const T* __restrict__ x, long ldx, const T* __restrict__ down,
                                          float* __restrict__ part, int row0, int inner, int j0, int k, int k_begin, int k_end,
                                          int chunk, quad_t (*s_sum)[kWaves][C][kWave]) {
    typedef Operand<T> Op;
    constexpr int kStep = Op::kLane * kQuarters, kOwn = (C + kWaves - 1) / kWaves;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, place = lane / kTile * Op::kLane;
    const T* rows[R];
    const T* weights[C];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int which = i * kTile + lane % kTile;
        rows[i] = x + static_cast<size_t>(row0 + __shfl(g.row, which < g.count ? which : 0, kWave)) * ldx;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int j = j0 + c * kTile + lane % kTile;
        weights[c] = down + (static_cast<size_t>(g.adapter) * inner + (j < inner ? j : inner - 1)) * k;
    }
    quad_t total[R][kOwn], acc[R][C];
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int o = 0; o < kOwn; ++o) total[i][o] = quad_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) acc[i][c] = quad_t{0.f, 0.f, 0.f, 0.f};
    }
    // a round is U steps of every wave (U of 1: 2,048 rows 24 us, not 22); the next round is under way while one is multiplied, also
    // across the end of a chunk
    constexpr int U = 2, kRound = kStep * kWaves * U;
    const int rounds = (k_end - k_begin + kRound - 1) / kRound, rounds_of_chunk = chunk / kRound;
    typename Op::type a[U][R], b[U][C];
    const auto ask = [&](int round) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = k_begin + (round * U + u) * (kStep * kWaves) + wave * kStep + place;
            const int from = at < k_end ? at : 0;
#pragma unroll
            for (int c = 0; c < C; ++c) b[u][c] = *reinterpret_cast<const typename Op::type*>(weights[c] + from);
#pragma unroll
            for (int i = 0; i < R; ++i) a[u][i] = *reinterpret_cast<const typename Op::type*>(rows[i] + from);
            if (at >= k_end) {  // (k is a multiple of kLane)
#pragma unroll
                for (int c = 0; c < C; ++c) b[u][c] = typename Op::type{};
#pragma unroll
                for (int i = 0; i < R; ++i) a[u][i] = typename Op::type{};
            }
        }
    };
    ask(0);
    int turn = 0;
    for (int round = 0, of_chunk = 1; round < rounds; ++round, ++of_chunk) {
        typename Op::type a_now[U][R], b_now[U][C];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < R; ++i) a_now[u][i] = a[u][i];
#pragma unroll
            for (int c = 0; c < C; ++c) b_now[u][c] = b[u][c];
        }
        if (round + 1 < rounds) ask(round + 1);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int c = 0; c < C; ++c) acc[i][c] = Op::mac(a_now[u][i], b_now[u][c], acc[i][c]);
        if (of_chunk < rounds_of_chunk && round + 1 < rounds) continue;
        of_chunk = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            // (two buffers in turn: a wave writes one again only behind the barrier of the other)
            quad_t(*s)[C][kWave] = s_sum[turn];
            turn ^= 1;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                s[wave][c][lane] = acc[i][c];
                acc[i][c] = quad_t{0.f, 0.f, 0.f, 0.f};
            }
            __syncthreads();
#pragma unroll
            for (int o = 0; o < kOwn; ++o) {
                const int c = wave + o * kWaves;
                if (c < C) total[i][o] += (s[0][c][lane] + s[1][c][lane]) + (s[2][c][lane] + s[3][c][lane]);
            }
        }
    }
    __syncthreads();  // (whoever comes next begins with the first buffer)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
            const int c = wave + o * kWaves, j = j0 + c * kTile + lane % kTile;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int which = i * kTile + lane / kTile * 4 + e;
                const int row = __shfl(g.row, which < g.count ? which : 0, kWave);
                if (c < C && which < g.count && j < inner) part[static_cast<size_t>(row0 + row) * inner + j] = total[i][o][e];
            }
        }
}

template <typename T, int C, bool kOneTile>  // kOneTile: tile_rows is 16 (a third of the registers: the form for many rows)
__global__ void __launch_bounds__(kThreads)
adapter_down_tiles(const T* __restrict__ x, long ldx, const T* __restrict__ down, const int* __restrict__ adapter,
                   float* __restrict__ h_part, int rows, int inner, int k, int adapters, int tile_rows, int slots, int chunk,
                   int part_k) {
    __shared__ quad_t s_sum[2][kWaves][C][kWave];
    const int lane = threadIdx.x % kWave, row0 = blockIdx.y * tile_rows;
    const int slot = blockIdx.z % slots, j0 = blockIdx.z / slots * (C * kTile);
    int id = lane < tile_rows && row0 + lane < rows ? adapter[row0 + lane] : -1;
    id = id < adapters ? id : -1;
    const int k_begin = blockIdx.x * part_k, k_end = min(k, k_begin + part_k);
    float* part = h_part + static_cast<size_t>(blockIdx.x) * rows * inner;
    const u64 same = rows_of_same(id, id >= 0, adapters);
    const bool first = same && __ffsll(same) - 1 == lane;
    const int running = wave_running(first), groups = __builtin_amdgcn_readlane(running, kWave - 1);
    const int group = __shfl(running, same ? __ffsll(same) - 1 : 0, kWave) - 1;  // (in the order of their first rows)
    for (int number = slot; number < groups; number += slots) {
        const Gathered g = gather(id, __ballot(same && group == number));
        if (kOneTile || g.count <= kTile)
            down_rows<T, C, 1>(g, x, ldx, down, part, row0, inner, j0, k, k_begin, k_end, chunk, s_sum);
        else if constexpr (!kOneTile) {
            if (g.count <= 2 * kTile)
                down_rows<T, C, 2>(g, x, ldx, down, part, row0, inner, j0, k, k_begin, k_end, chunk, s_sum);
            else
                down_rows<T, C, 4>(g, x, ldx, down, part, row0, inner, j0, k, k_begin, k_end, chunk, s_sum);
        }
    }
}

// The rows of h on their way into the second product, whose result is of type S.  In bfloat16 a number is the sum of several: its
// rounding, the rounding of what that left out, and so on, 8 bits each, and the product runs once for each.  A float32 stream has all
// three that a float32 number holds (with two 92.9 us of 94 for 2,048 rows of 18,944 and 3,584 at rank 64, 0.1 to 0.5 less of smaller
// ones); rows of bfloat16, which keep 8 bits of the sum, two (2^-17 of the number).
template <typename T, typename S>
struct Inner;
template <typename S>
struct Inner<bf16_t, S> {
    static constexpr int kTerms = sizeof(S) == 4 ? 3 : 2;
    typedef __bf16 store_t;
    static __device__ __forceinline__ void put(store_t* at, int apart, float v) {
#pragma unroll
        for (int i = 0; i < kTerms; ++i) {
            const __bf16 term = static_cast<__bf16>(v);
            const float kept = static_cast<float>(term);
            at[i * apart] = term;
            v = fabsf(kept) < INFINITY ? v - kept : 0.f;  // (exact)
        }
    }
};
template <>
struct Inner<float, float> {
    static constexpr int kTerms = 1;
    typedef float store_t;
    static __device__ __forceinline__ void put(store_t* at, int, float v) { at[0] = v; }
};

// kLane numbers of a row of `up` from place k on (rank is a multiple of 4; what lies behind it counts as 0).
__device__ __forceinline__ octet_t up_numbers(const bf16_t* row, int k, int rank) {
    if (rank % 8 == 0) return k < rank ? *reinterpret_cast<const octet_t*>(row + k) : octet_t{};
    half_octet_t lo = {}, hi = {};
    if (k < rank) lo = *reinterpret_cast<const half_octet_t*>(row + k);
    if (k + 4 < rank) hi = *reinterpret_cast<const half_octet_t*>(row + k + 4);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ quad_t up_numbers(const float* row, int k, int rank) {
    return k < rank ? *reinterpret_cast<const quad_t*>(row + k) : quad_t{};
}

// 16 bytes of a row of `into`, and what is added to them.
typedef uint32_t words_t __attribute__((ext_vector_type(4)));
template <typename S>
struct Piece {
    static constexpr int kNumbers = 16 / sizeof(S);
    static __device__ __forceinline__ words_t sum(words_t old, const float (&more)[kNumbers]);
};
template <>
__device__ __forceinline__ words_t Piece<float>::sum(words_t old, const float (&more)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) old[i] = __float_as_uint(__uint_as_float(old[i]) + more[i]);
    return old;
}
template <>
__device__ __forceinline__ words_t Piece<bf16_t>::sum(words_t old, const float (&more)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        old[i] = pack_bf16(__uint_as_float(old[i] << 16) + more[2 * i], __uint_as_float(old[i] & 0xffff0000u) + more[2 * i + 1]);
    return old;
}

// Four numbers of h: the parts, `apart` floats from each other, in the one order (chunks: by groups).
__device__ __forceinline__ quad_t sum_of_parts(const float* at, size_t apart, int parts, bool chunks) {
    quad_t sum = {0.f, 0.f, 0.f, 0.f};
    if (!chunks) {
#pragma unroll 4
        for (int s = 0; s < parts; ++s) sum += *reinterpret_cast<const quad_t*>(at + s * apart);
        return sum;
    }
#pragma unroll 2
    for (int s = 0; s < parts; s += kGroup) {
        quad_t part[kGroup] = {};
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
            if (s + i < parts) part[i] = *reinterpret_cast<const quad_t*>(at + (s + i) * apart);
        sum += ((part[0] + part[1]) + part[2]) + part[3];
    }
    return sum;
}

// A lane's numbers of its row of h (`at`), ready for the second product.
template <typename T, typename S, int kSteps, int kTerms>
__device__ __forceinline__ void ask_inner(typename Operand<T>::type (&h)[kTerms][kSteps], const float* at, size_t apart, int parts, bool chunks,
                                          float factor, int rank) {
    typedef Operand<T> Op;
    static_assert(kTerms == Inner<T, S>::kTerms, "room for all terms");
    const int quarter = threadIdx.x % kWave / kTile;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int r = (s * kQuarters + quarter) * Op::kLane;
        typename Inner<T, S>::store_t terms[kTerms][Op::kLane];
#pragma unroll
        for (int e = 0; e < Op::kLane; e += 4) {
            quad_t sum = {0.f, 0.f, 0.f, 0.f};
            if (r + e < rank) sum = sum_of_parts(at + r + e, apart, parts, chunks) * factor;
#pragma unroll
            for (int i = 0; i < 4; ++i) Inner<T, S>::put(&terms[0][e + i], Op::kLane, sum[i]);
        }
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int e = 0; e < Op::kLane; ++e) h[term][s][e] = terms[term][e];
    }
}

// Who of a row tile has which adapter.
struct Order {
    int id[kWave], order[kWave];  // the rows' adapters (-1: none); the rows by adapter,
    int group[kWave + 1], count;  // where each adapter's rows begin, and how many adapters there are

    // (rows without an adapter count as one more where they are to be copied)
    __device__ __forceinline__ void sort_rows(const int* adapter, int row0, int rows, int adapters, bool copies) {
        const int lane = threadIdx.x % kWave;
        if (threadIdx.x < kWave) {
            int mine = row0 + lane < rows ? adapter[row0 + lane] : -1;
            mine = mine >= 0 && mine < adapters ? mine : -1;
            const u64 same = rows_of_same(mine, row0 + lane < rows && (mine >= 0 || copies), adapters);
            const int place = __popcll(same & lanes_below());
            const bool first = same && place == 0;
            // the groups and rows in front of this lane's group, which come in the order of their first rows
            const int own = first ? 1 << 16 | __popcll(same) : 0, running = wave_running(own);
            const int front = __shfl(running - own, same ? __ffsll(same) - 1 : 0, kWave), all = __builtin_amdgcn_readlane(running, kWave - 1);
            if (same) order[(front & 0xffff) + place] = lane;
            if (first) group[front >> 16] = front & 0xffff;
            if (lane == 0) {
                group[all >> 16] = all & 0xffff;
                count = all >> 16;
            }
            id[lane] = mine;
        }
        __syncthreads();
    }
};

// The same for few rows: the rows of an adapter 16 at a time, of which a workgroup has every `slots`-th sixteen.  (In bytes where they
// do: beside three terms of ranks above 64 three workgroups then share a CU's LDS.  601 rows of 2,048 and 2,048 columns of the float32
// stream at rank 72 take 18.1 us, 23.0 with two of them.)
struct Sixteens {
    int adapter[kWave], count;
    uint8_t rows[kWave], order[kWave][kTile];

    __device__ __forceinline__ void sort_rows(const int* adapter_of, int row0, int rows_in_all, int adapters, int slots, int slot, bool copies) {
        const int lane = threadIdx.x % kWave;
        if (threadIdx.x < kWave) {
            int mine = row0 + lane < rows_in_all ? adapter_of[row0 + lane] : -1;
            mine = mine >= 0 && mine < adapters ? mine : -1;
            const u64 same = rows_of_same(mine, row0 + lane < rows_in_all && (mine >= 0 || copies), adapters);
            const int in_all = __popcll(same), place = __popcll(same & lanes_below());
            const int own = same && place == 0 ? (in_all + kTile - 1) / kTile : 0, running = wave_running(own);
            const int which = __shfl(running - own, same ? __ffsll(same) - 1 : 0, kWave) + place / kTile;
            if (same && which % slots == slot) {
                order[which / slots][place % kTile] = static_cast<uint8_t>(lane);
                if (place % kTile == 0) {
                    rows[which / slots] = static_cast<uint8_t>(min(kTile, in_all - place));
                    adapter[which / slots] = mine;
                }
            }
            const int number = __builtin_amdgcn_readlane(running, kWave - 1);
            if (lane == 0) count = number > slot ? (number - 1 - slot) / slots + 1 : 0;
        }
        __syncthreads();
    }
};

// The tile's rows of h in LDS: the parts added in order, times the adapter's scale.
template <typename T, typename S, int kSteps>
struct Rows {
    typedef typename Inner<T, S>::store_t store_t;
    static constexpr int kWidth = kSteps * Operand<T>::kLane * kQuarters, kTerms = Inner<T, S>::kTerms;
    static constexpr int kLd = kWidth + 16 / sizeof(store_t);  // (rows a little apart, so that 16 of them do not share their banks)
    store_t number[kTerms][kWave][kLd];

    // of(i, a): the tile's row of number i below `count`, and its adapter; -1: none
    template <typename Of>
    __device__ __forceinline__ void add_parts(int count, Of of, const float* h_part, int parts, bool chunks, const float* scale, int row0,
                                              int rows, int inner, int from, int rank) {
        constexpr int kFours = kWidth / 4;
        for (int item = threadIdx.x; item < count * kFours; item += kThreads) {
            const int r = item % kFours * 4;
            int a = -1;
            const int row = of(item / kFours, a);
            if (a < 0) continue;
            quad_t sum = {0.f, 0.f, 0.f, 0.f};
            if (r < rank)
                sum = sum_of_parts(h_part + static_cast<size_t>(row0 + row) * inner + from + r, static_cast<size_t>(rows) * inner, parts, chunks) *
                      scale[a];
#pragma unroll
            for (int e = 0; e < 4; ++e) Inner<T, S>::put(&number[0][row][r + e], kWave * kLd, sum[e]);
        }
        __syncthreads();
    }
};

// A wave's share of the second product for few rows: up to 16 rows of one adapter and a strip of columns.  h is the first operand,
// the strip's columns the second, dealt to the instructions so that a lane's results are 16 bytes of neighbouring columns (in
// four rows), and 16 lanes have 256 bytes of a row in one piece.
template <typename T, typename S, int kSteps>
struct Share {
    typedef Operand<T> Op;
    static constexpr int kOwn = Piece<S>::kNumbers, kStrip = kTile * kOwn, kTerms = Inner<T, S>::kTerms;
    typename Op::type weights[kSteps][kOwn];
    words_t old[4];
    int row[4], adapter, first;  // the rows of the lane's results (-1: none) and the first of its columns
    int mine;                    // the row that the lane brings to the product
    bool whole;

    __device__ __forceinline__ void ask(const Sixteens& tile, int which, int c0, int end, const T* up, int n, int rank, const S* into,
                                        long ld_into, bool wide) {
        const int lane = threadIdx.x % kWave, quarter = lane / kTile, count = tile.rows[which];
        adapter = tile.adapter[which];
        mine = tile.order[which][min(lane % kTile, count - 1)];
        first = c0 + lane % kTile * kOwn;
        whole = wide && first + kOwn <= end;
        if (adapter >= 0) {
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                const int c = first + j < end ? first + j : end - 1;
                const T* from = up + (static_cast<size_t>(adapter) * n + c) * rank;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) weights[s][j] = up_numbers(from, (s * kQuarters + quarter) * Op::kLane, rank);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            row[i] = quarter * 4 + i < count ? tile.order[which][quarter * 4 + i] : -1;
            if (whole && row[i] >= 0) old[i] = *reinterpret_cast<const words_t*>(into + static_cast<size_t>(row[i]) * ld_into + first);
        }
    }

    __device__ __forceinline__ void finish(const Rows<T, S, kSteps>& h, int end, const S* into, long ld_into, S* out, long ld_out) {
        const int quarter = threadIdx.x % kWave / kTile;
        quad_t acc[kOwn] = {};
        if (adapter >= 0) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    const typename Op::type its =
                        *reinterpret_cast<const typename Op::type*>(&h.number[term][mine][(s * kQuarters + quarter) * Op::kLane]);
#pragma unroll
                    for (int j = 0; j < kOwn; ++j) acc[j] = Op::mac(its, weights[s][j], acc[j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (row[i] < 0) continue;
            S* to = out + static_cast<size_t>(row[i]) * ld_out + first;
            if (whole) {
                float more[kOwn];
#pragma unroll
                for (int j = 0; j < kOwn; ++j) more[j] = acc[j][i];
                *reinterpret_cast<words_t*>(to) = adapter >= 0 ? Piece<S>::sum(old[i], more) : old[i];
                continue;
            }
            const S* from = into + static_cast<size_t>(row[i]) * ld_into + first;
#pragma unroll
            for (int j = 0; j < kOwn; ++j)
                if (first + j < end) to[j] = adapter >= 0 ? from_float<S>(to_float(from[j]) + acc[j][i]) : from[j];
        }
    }
};

// Which piece, and which of its columns, the block of that number has.
struct Columns {
    int piece, begin, end;
    __device__ __forceinline__ Columns(const Pieces& pieces, int number, int block) {
        piece = 0;
        for (; piece + 1 < pieces.count; ++piece) {
            const int blocks = (pieces.begin[piece + 1] - pieces.begin[piece] + block - 1) / block;
            if (number < blocks) break;
            number -= blocks;
        }
        begin = pieces.begin[piece] + number * block;
        end = min(pieces.begin[piece + 1], begin + block);
    }
};

// Few rows.  grid: (row tiles, column blocks of the pieces, slots): a workgroup has every `slots`-th of its tile's sixteens, a wave
// one of them and a strip of columns at a time.  A wave's first weights and rows of `into` are under way while the parts of h are
// added.  (h through LDS: a wave that adds its own 16 rows' parts, without a barrier, took 20 us for 64 rows of 22,016 columns where
// this took 12.8.)  What bounds it is the way to the first result: the adapters' numbers, the parts, the weights and the barrier between
// them; one row takes 5.3 us, 64 rows of 16 adapters 10.6 (6 MB of rows and 11 MB of weights at 1.6 TB/s).
template <typename T, typename S, int kSteps>
__global__ void __launch_bounds__(kThreads, kSteps == 1 ? 4 : kSteps == 2 ? 3 : 2)
adapter_up_rows(const float* __restrict__ h_part, int parts, bool chunks, const T* __restrict__ up, const float* __restrict__ scale,
                const int* __restrict__ adapter, const S* into, long ld_into, S* out, long ld_out, int rows, int inner, int n, int rank,
                int adapters, Pieces pieces, int block, int slots, bool wide) {
    __shared__ Sixteens tile;
    __shared__ __align__(16) Rows<T, S, kSteps> h;
    const int wave = threadIdx.x / kWave, row0 = blockIdx.x * kWave;
    const Columns columns(pieces, blockIdx.y, block);
    tile.sort_rows(adapter, row0, rows, adapters, slots, blockIdx.z, static_cast<const void*>(into) != static_cast<const void*>(out));
    if (tile.count == 0) return;
    into += static_cast<size_t>(row0) * ld_into;
    out += static_cast<size_t>(row0) * ld_out;
    constexpr int kStrip = Share<T, S, kSteps>::kStrip;
    const int strips = (columns.end - columns.begin + kStrip - 1) / kStrip, shares = tile.count * strips;
    Share<T, S, kSteps> share;
    const auto ask = [&](int number) {
        share.ask(tile, number / strips, columns.begin + number % strips * kStrip, columns.end, up, n, rank, into, ld_into, wide);
    };
    int number = wave;
    if (number < shares) ask(number);
    h.add_parts(
        tile.count * kTile,
        [&](int i, int& a) {
            if (i % kTile < tile.rows[i / kTile]) a = tile.adapter[i / kTile];
            return tile.order[i / kTile][i % kTile];
        },
        h_part, parts, chunks, scale, row0, rows, inner, columns.piece * rank, rank);
    while (number < shares) {
        share.finish(h, columns.end, into, ld_into, out, ld_out);
        number += kWaves;
        if (number < shares) ask(number);
    }
}

// Many rows.  grid: row tiles x column blocks of the pieces, rounded up to whole turns of the XCDs: each XCD has a run of them in
// which the row tiles of a column block follow each other, so that its L2 holds the block's weights.  A workgroup goes through its
// strips of columns, and in each through its tile's adapters (of a prompt there is one); each of its four waves has 16 of the
// adapter's rows, whose h it keeps in registers.  The strip's weights pass through LDS, which all four read, a strip ahead of
// its use.
//
// The loop over whole strips has no branch around a load or store: rows that are not there have an offset behind their buffer's end,
// which drops them.  The wait for a strip's weights then leaves the rows and stores behind them under way; with branches the
// compiler has to wait for all of them, once a strip.  2,048 rows of 37,888 columns at rank 64, two prompts: 88 us (with the branches
// 107) for 310 MB of rows read and written, 3.6 TB/s where a plain copy of this size reaches 5.1.
template <typename T, typename S, int kSteps, bool kEven>  // kEven: the rank is a multiple of a lane's numbers
__global__ void __launch_bounds__(kThreads, 4)
adapter_up_strips(const float* __restrict__ h_part, int parts, bool chunks, const T* __restrict__ up, const float* __restrict__ scale,
                  const int* __restrict__ adapter, const S* into, long ld_into, S* out, long ld_out, int rows, int inner, int n, int rank,
                  int adapters, Pieces pieces, int block, int row_tiles, int blocks, bool wide) {
    typedef Operand<T> Op;
    typedef typename Inner<T, S>::store_t store_t;
    constexpr int kOwn = Piece<S>::kNumbers, kStrip = kTile * kOwn, kLoads = kSteps * kQuarters, kMine = kStrip * kLoads / kThreads;
    typedef Rows<T, S, kSteps> RowsT;
    constexpr int kLd = RowsT::kLd, kTerms = RowsT::kTerms;
    static_assert(kStrip * kLoads % kThreads == 0, "every thread stages as many pieces");
    __shared__ Order tile;
    // Two buffers of weights in turn.  A tile of several adapters has them one after the other in the first, with a barrier more,
    // and its rows of h in place of the second.
    struct Weights {
        store_t number[kStrip][kLd];
    };
    constexpr size_t kSecond = sizeof(Weights) > sizeof(RowsT) ? sizeof(Weights) : sizeof(RowsT);
    __shared__ __align__(16) char lds[sizeof(Weights) + kSecond];
    Weights* const s_w = reinterpret_cast<Weights*>(lds);
    RowsT& s_h = *reinterpret_cast<RowsT*>(lds + sizeof(Weights));
    const int number_of_all = blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds;
    if (number_of_all >= row_tiles * blocks) return;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, quarter = lane / kTile, row0 = number_of_all % row_tiles * kWave;
    const Columns columns(pieces, number_of_all / row_tiles, block);
    tile.sort_rows(adapter, row0, rows, adapters, static_cast<const void*>(into) != static_cast<const void*>(out));
    if (tile.count == 0) return;
    into += static_cast<size_t>(row0) * ld_into;
    out += static_cast<size_t>(row0) * ld_out;
    // (wide: the last row of a tile ends below 2 GB)
    const unsigned last = min(kWave, rows - row0) - 1;
    constexpr int kNowhere = static_cast<int>(0x80000000u);
    const __amdgpu_buffer_rsrc_t of_into = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<S*>(into), 0, wide ? (last * static_cast<unsigned>(ld_into) + n) * static_cast<unsigned>(sizeof(S)) : 0, 0x00027000);
    const __amdgpu_buffer_rsrc_t of_out = __builtin_amdgcn_make_buffer_rsrc(
        out, 0, wide ? (last * static_cast<unsigned>(ld_out) + n) * static_cast<unsigned>(sizeof(S)) : 0, 0x00027000);
    const int groups = tile.count, total = (columns.end - columns.begin + kStrip - 1) / kStrip * groups;
    const int whole = wide ? (columns.end - columns.begin) / kStrip * groups : 0;
    const bool many = groups > 1;

    typename Op::type staged[kMine], h[kTerms][kSteps];
    words_t old[4];
    const auto ask_weights = [&](int number) {
        const int a = max(0, tile.id[tile.order[tile.group[number % groups]]]);  // (rows without an adapter: not used)
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int item = i * kThreads + threadIdx.x, c = min(columns.begin + number / groups * kStrip + item / kLoads, columns.end - 1);
            const int from = item % kLoads * Op::kLane;
            const T* row = up + (static_cast<size_t>(a) * n + c) * rank;
            if constexpr (kEven) {
                staged[i] = *reinterpret_cast<const typename Op::type*>(row + (from < rank ? from : 0));
                if (from >= rank) staged[i] = typename Op::type{};
            } else {
                staged[i] = up_numbers(row, from, rank);
            }
        }
    };
    // (column c lies where the lane that computes it reads without sharing banks)
    const auto put_weights = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int item = i * kThreads + threadIdx.x, c = item / kLoads;
            *reinterpret_cast<typename Op::type*>(&s_w[buffer].number[c % kOwn * kTile + c / kOwn][item % kLoads * Op::kLane]) = staged[i];
        }
    };
    const auto offset = [&](int number, int i, long ld) {
        const int from = tile.group[number % groups], which = wave * kTile + quarter * 4 + i;
        const int first = columns.begin + number / groups * kStrip + lane % kTile * kOwn;
        return which < tile.group[number % groups + 1] - from
                   ? (tile.order[from + which] * static_cast<int>(ld) + first) * static_cast<int>(sizeof(S))
                   : kNowhere;
    };
    const auto ask_rows = [&](int number) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            old[i] = __builtin_bit_cast(words_t, __builtin_amdgcn_raw_buffer_load_b128(of_into, offset(number, i, ld_into), 0, 0));
    };
    const auto ask_h = [&]() {  // of a tile's one adapter
        const int row = tile.order[min(wave * kTile + lane % kTile, tile.group[1] - 1)], a = tile.id[row];
        if (a < 0) return;
        ask_inner<T, S, kSteps>(h, h_part + static_cast<size_t>(row0 + row) * inner + columns.piece * rank, static_cast<size_t>(rows) * inner,
                                parts, chunks, scale[a], rank);
    };
    // the strip's weights are in LDS, the next ones are asked for: what the wave's 16 rows gain
    const auto gains = [&](int number, quad_t(&acc)[kOwn]) {
        const int buffer = many ? 0 : number & 1;
        if (many) __syncthreads();  // (the buffer has been read by all)
        put_weights(buffer);
        __syncthreads();  // (and the other buffer has been read by all)
        ask_weights(min(number + 1, total - 1));
        const int from = tile.group[number % groups], count = tile.group[number % groups + 1] - from;
        if (wave * kTile >= count) return;
        if (many) {
            const int row = tile.order[from + min(wave * kTile + lane % kTile, count - 1)];
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                    h[term][s] = *reinterpret_cast<const typename Op::type*>(&s_h.number[term][row][(s * kQuarters + quarter) * Op::kLane]);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                const typename Op::type weights =
                    *reinterpret_cast<const typename Op::type*>(&s_w[buffer].number[j * kTile + lane % kTile][(s * kQuarters + quarter) * Op::kLane]);
#pragma unroll
                for (int term = 0; term < kTerms; ++term) acc[j] = Op::mac(h[term][s], weights, acc[j]);
            }
    };
    ask_weights(0);
    ask_rows(0);
    if (many)
        s_h.add_parts(kWave, [&](int i, int& a) { a = tile.id[i]; return i; }, h_part, parts, chunks, scale, row0, rows, inner,
                      columns.piece * rank, rank);
    else
        ask_h();
    int number = 0;
    for (; number < whole; ++number) {
        quad_t acc[kOwn] = {};
        gains(number, acc);
        const bool has = tile.id[tile.order[tile.group[number % groups]]] >= 0;
        words_t now[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float more[kOwn];
#pragma unroll
            for (int j = 0; j < kOwn; ++j) more[j] = acc[j][i];
            const words_t sum = Piece<S>::sum(old[i], more);
#pragma unroll
            for (int w = 0; w < 4; ++w) now[i][w] = has ? sum[w] : old[i][w];
        }
        ask_rows(min(number + 1, total - 1));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(int __attribute__((ext_vector_type(4))), now[i]), of_out,
                                                   offset(number, i, ld_out), 0, 0);
    }
    // the columns behind the last whole strip, or rows that 16-byte pieces do not take
    for (; number < total; ++number) {
        quad_t acc[kOwn] = {};
        gains(number, acc);
        const int from = tile.group[number % groups], count = tile.group[number % groups + 1] - from, a = tile.id[tile.order[from]];
        const int first = columns.begin + number / groups * kStrip + lane % kTile * kOwn;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int which = wave * kTile + quarter * 4 + i;
            if (which >= count) continue;
            const int row = tile.order[from + which];
            const S* source = into + static_cast<size_t>(row) * ld_into + first;
            S* to = out + static_cast<size_t>(row) * ld_out + first;
#pragma unroll
            for (int j = 0; j < kOwn; ++j)
                if (first + j < columns.end) to[j] = a >= 0 ? from_float<S>(to_float(source[j]) + acc[j][i]) : source[j];
        }
    }
}

struct Plan {
    int chunk, parts, tile_rows, slots, block, up_slots;
    bool chunks(int k) const { return parts == (k + chunk - 1) / chunk; }
};

template <typename T, int C>
int launch_down(hipStream_t s, const T* x, long ldx, const T* down, const int* adapter, float* h, int rows, int k, int inner, int adapters,
                const Plan& plan) {
    const int part_k = plan.chunks(k) ? plan.chunk : kGroup * plan.chunk;
    const int groups = (inner + C * kTile - 1) / (C * kTile);
    const dim3 grid(plan.parts, (rows + plan.tile_rows - 1) / plan.tile_rows, groups * plan.slots);
    if (plan.tile_rows == kTile)
        adapter_down_tiles<T, C, true><<<grid, kThreads, 0, s>>>(x, ldx, down, adapter, h, rows, inner, k, adapters, plan.tile_rows,
                                                                plan.slots, plan.chunk, part_k);
    else
        adapter_down_tiles<T, C, false><<<grid, kThreads, 0, s>>>(x, ldx, down, adapter, h, rows, inner, k, adapters, plan.tile_rows,
                                                                 plan.slots, plan.chunk, part_k);
    return cie_after_launch();
}

template <typename T, typename S>
int run_tiles(hipStream_t s, const void* x_, long ldx, const void* down_, const void* up_, const float* scale, const int* adapter,
              const void* into_, long ld_into, void* out_, long ld_out, float* h, int rows, int k, int n, int rank, int adapters,
              const Pieces& pieces, const Plan& plan) {
    const T *x = static_cast<const T*>(x_), *down = static_cast<const T*>(down_), *up = static_cast<const T*>(up_);
    const S* into = static_cast<const S*>(into_);
    S* out = static_cast<S*>(out_);
    const int inner = pieces.count * rank;
    int code = inner <= kTile ? launch_down<T, 1>(s, x, ldx, down, adapter, h, rows, k, inner, adapters, plan)
               : inner <= 2 * kTile ? launch_down<T, 2>(s, x, ldx, down, adapter, h, rows, k, inner, adapters, plan)
                                    : launch_down<T, 4>(s, x, ldx, down, adapter, h, rows, k, inner, adapters, plan);
    if (code != CIE_OK) return code;
    int blocks = 0;
    bool wide = ld_into * sizeof(S) % 16 == 0 && ld_out * sizeof(S) % 16 == 0 && reinterpret_cast<uintptr_t>(into) % 16 == 0 &&
                reinterpret_cast<uintptr_t>(out) % 16 == 0;
    for (int p = 0; p < pieces.count; ++p) {
        blocks += (pieces.begin[p + 1] - pieces.begin[p] + plan.block - 1) / plan.block;
        wide = wide && pieces.begin[p] * sizeof(S) % 16 == 0;
    }
    const unsigned row_tiles = (rows + kWave - 1) / kWave;
    constexpr int kStep = Operand<T>::kLane * kQuarters;
    if (plan.up_slots > 0) {
#define CIE_UP(STEPS)                                                                                                              \
    adapter_up_rows<T, S, STEPS><<<dim3(row_tiles, blocks, plan.up_slots), kThreads, 0, s>>>(                                          \
        h, plan.parts, plan.chunks(k), up, scale, adapter, into, ld_into, out, ld_out, rows, inner, n, rank, adapters, pieces, plan.block,  \
        plan.up_slots, wide)
        if (rank <= kStep)
            CIE_UP(1);
        else if (rank <= 2 * kStep)
            CIE_UP(2);
        else if (rank <= 4 * kStep)
            CIE_UP(4);
        else if constexpr (kStep * 4 < 128)
            CIE_UP(8);
#undef CIE_UP
    } else {
        const bool near = (static_cast<double>(kWave) * (ld_into > ld_out ? ld_into : ld_out) + n) * sizeof(S) < 2147483648.0;
        const dim3 grid((row_tiles * blocks + kXcds - 1) / kXcds * kXcds);
#define CIE_UP_OF(STEPS, EVEN)                                                                                                    \
    adapter_up_strips<T, S, STEPS, EVEN><<<grid, kThreads, 0, s>>>(h, plan.parts, plan.chunks(k), up, scale, adapter, into, ld_into, out,    \
                                                                   ld_out, rows, inner, n, rank, adapters, pieces, plan.block,           \
                                                                   static_cast<int>(row_tiles), blocks, wide && near)
#define CIE_UP(STEPS)                            \
    if (rank % Operand<T>::kLane == 0)           \
        CIE_UP_OF(STEPS, true);                  \
    else if constexpr (Operand<T>::kLane > 4)    \
    CIE_UP_OF(STEPS, false)
        if (rank <= kStep) {
            CIE_UP(1);
        } else if (rank <= 2 * kStep) {
            CIE_UP(2);
        } else if constexpr (kStep * 2 < 64) {
            CIE_UP(4);
        }
#undef CIE_UP
#undef CIE_UP_OF
    }
    return cie_after_launch();
}

}  // namespace

// dtype: of x, down and up; out_dtype: of into and out (dtype, or float32).  c1, c2, c3: where the second and later pieces begin
// (n where there is none).  out may be into.  parts = 0: the kernels that take any shape (h: rows * pieces * rank floats).  Else the
// tiles, which take a rank that is a multiple of 4 and rows of x and down in 16-byte pieces: K in chunks of `chunk`, each of them
// a part or each four (h: as many floats for each part), `down` in tiles of tile_rows (16 to 64) rows and `slots` workgroups
// for a tile's adapters, `up` in blocks of `block` columns; up_slots > 0: in the form for few
// rows, with so many workgroups for the adapters of a tile of 64 rows, 0: in the form for many (a rank of up to 64).
CIE_API int cie_lora_add(void* stream, int dtype, int out_dtype, const void* x, long ldx, const void* down, const void* up,
                         const float* scale, const int* adapter, const void* into, long ld_into, void* out, long ld_out, float* h,
                         int rows, int k, int n, int rank, int adapters, int piece_count, int c1, int c2, int c3, int chunk,
                         int parts, int tile_rows, int slots, int block, int up_slots) {
    if (rows < 0 || rows > 65535 || k <= 0 || k > (1 << 28) || n <= 0 || n > (1 << 28) || rank <= 0 || rank > 128 || adapters <= 0 || piece_count < 1 ||
        piece_count > kMaxPieces || ldx < k || ld_into < n || ld_out < n || !x || !down || !up || !scale || !adapter || !into || !out || !h)
        return CIE_BAD_ARGUMENT;
    if (rows == 0) return CIE_OK;
    Pieces pieces = {piece_count, {0, c1, c2, c3, n}};
    for (int p = piece_count; p <= kMaxPieces; ++p) pieces.begin[p] = n;
    for (int p = 0; p < piece_count; ++p)
        if (pieces.begin[p + 1] <= pieces.begin[p]) return CIE_BAD_ARGUMENT;
    const Plan plan = {chunk, parts, tile_rows, slots, block, up_slots};
    if (parts != 0) {
        const int size = dtype == CIE_BF16 ? 2 : 4;
        const bool lines = k * size % 16 == 0 && ldx * size % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                           reinterpret_cast<uintptr_t>(down) % 16 == 0 && reinterpret_cast<uintptr_t>(up) % 16 == 0 &&
                           reinterpret_cast<uintptr_t>(h) % 16 == 0;
        const int share = 256 / size;  // (the k that a workgroup's four waves take at a time)
        if (!lines || rank % 4 || chunk < 2 * share || chunk % (2 * share) ||
            (!plan.chunks(k) && parts != (k + kGroup * chunk - 1) / (kGroup * chunk)) || tile_rows < 16 || tile_rows > kWave ||
            tile_rows % kTile || slots < 1 || slots > kWave || block < kWave || block % kWave || up_slots < 0 || up_slots > kWave ||
            (up_slots == 0 && rank > 64))
            return CIE_BAD_ARGUMENT;
        long blocks = 0;
        for (int p = 0; p < piece_count; ++p) blocks += (pieces.begin[p + 1] - pieces.begin[p] + block - 1) / block;
        if (up_slots > 0 && blocks > 65535) return CIE_BAD_ARGUMENT;  // (a grid's second dimension)
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
#define CIE_RUN(T, S)                                                                                                              \
    return parts == 0 ? run_plain<T, S>(s, x, ldx, down, up, scale, adapter, into, ld_into, out, ld_out, h, rows, k, n, rank, adapters,  \
                                        pieces)                                                                                     \
                      : run_tiles<T, S>(s, x, ldx, down, up, scale, adapter, into, ld_into, out, ld_out, h, rows, k, n, rank, adapters,  \
                                        pieces, plan)
    if (dtype == CIE_F32 && out_dtype == CIE_F32) CIE_RUN(float, float);
    if (dtype == CIE_BF16 && out_dtype == CIE_F32) CIE_RUN(bf16_t, float);
    if (dtype == CIE_BF16 && out_dtype == CIE_BF16) CIE_RUN(bf16_t, bf16_t);
#undef CIE_RUN
    return CIE_BAD_ARGUMENT;
}
