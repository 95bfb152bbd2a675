// experts.hip -- samples sorted by the expert (block field) each goes to, and back with weights; forward and gradient.
//
// A choice i = t * k + j sends sample t to expert ids[i]; an id outside [0, E) drops the choice.  The plan is a stable
// counting sort: offsets[e] choices lie before expert e, slot[i] is choice i's row in the sorted order, order[row] = i.
// Everything after the sort is a gather: no kernel here adds with atomics across workgroups, so results do not depend on
// the order in which workgroups run.
#include <algorithm>
#include <initializer_list>

#include "operators.h"

namespace sng {

// ---- stable counting sort -----------------------------------------------------------------------------------------
// A wave ranks 64 choices at a time: the lanes that hold the same expert find one another with one ballot per id bit,
// the lowest of them adds their number to the wave's counter of that expert in LDS, and a lane's rank is the counter's
// old value plus the peers below it.  Waves own contiguous pieces and counters of their own, so ranks follow the
// choices' order.  (An LDS counter per lane would need no ballots but 64 times the LDS.)
template <int ROUNDS>
__device__ __forceinline__ void wave_ranks(const int32_t* __restrict__ ids, uint32_t begin, uint32_t total, uint32_t n_experts, int id_bits, uint32_t* cnt,
                                           int lane, uint32_t (&key)[ROUNDS], uint32_t (&rank)[ROUNDS]) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = begin + r * 64 + lane;
        const uint32_t id = i < total ? (uint32_t)ids[i] : 0xffffffffu;
        key[r] = id < n_experts ? id : 0xffffffffu;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool kept = key[r] != 0xffffffffu;
        unsigned long long peers = __ballot(kept);
        for (int b = 0; b < id_bits; ++b) {
            const bool bit = (key[r] >> b) & 1u;
            const unsigned long long m = __ballot(bit);
            peers &= bit ? m : ~m;
        }
        uint32_t old = 0;
        const int leader = kept ? __ffsll(peers) - 1 : lane;
        if (kept && leader == lane) old = atomicAdd(&cnt[key[r]], (uint32_t)__popcll(peers));
        old = __shfl(old, leader, 64);
        rank[r] = old + (uint32_t)__popcll(peers & ((1ull << lane) - 1ull));
    }
}

// exclusive scan of one value per thread over a workgroup of NW waves; `all` receives the sum
template <int NW>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* wave_sums, uint32_t& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t u = __shfl_up(incl, d, 64);
        if (lane >= d) incl += u;
    }
    if (lane == 63) wave_sums[wave] = incl;
    __syncthreads();
    uint32_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const uint32_t u = wave_sums[w];
        before += w < wave ? u : 0u;
        sum += u;
    }
    __syncthreads();
    all = sum;
    return before + incl - v;
}

// Everything in one workgroup: ranks, the scan over waves and experts, the plan.  One launch instead of three for the
// small calls, where launches are the time.
template <int NW, int ROUNDS>
__global__ __launch_bounds__(NW * 64) void expert_sort_one_kernel(SortArgs a, int id_bits) {
    extern __shared__ uint32_t cnt[];   // [NW][n_experts]
    __shared__ uint32_t wave_sums[NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t e_n = a.n_experts;
    for (uint32_t i = threadIdx.x; i < NW * e_n; i += NW * 64) cnt[i] = 0;
    __syncthreads();
    uint32_t key[ROUNDS], rank[ROUNDS];
    const uint32_t begin = wave * (ROUNDS * 64);
    wave_ranks<ROUNDS>(a.experts, begin, a.total, e_n, id_bits, cnt + wave * e_n, lane, key, rank);
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < e_n; e0 += NW * 64) {
        const uint32_t e = e0 + threadIdx.x;
        uint32_t sum = 0;
        if (e < e_n)
            for (int w = 0; w < NW; ++w) sum += cnt[w * e_n + e];
        uint32_t all;
        uint32_t at = base + block_scan<NW>(sum, wave_sums, all);
        if (e < e_n) {
            a.offsets[e] = (int32_t)at;
            for (int w = 0; w < NW; ++w) {
                const uint32_t c = cnt[w * e_n + e];
                cnt[w * e_n + e] = at;
                at += c;
            }
        }
        base += all;
    }
    if (threadIdx.x == 0) a.offsets[e_n] = (int32_t)base;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = begin + r * 64 + lane;
        if (i >= a.total) continue;
        const bool kept = key[r] != 0xffffffffu;
        const uint32_t at = kept ? cnt[wave * e_n + key[r]] + rank[r] : 0;
        a.slot[i] = kept ? (int32_t)at : -1;
        if (kept) a.order[at] = (int32_t)i;
        if (i >= base) a.order[i] = -1;
    }
}

// Three launches: counts per (workgroup, expert); their exclusive sums down the workgroups; ranks and the plan.
__global__ __launch_bounds__(256) void expert_count_kernel(SortArgs a) {
    extern __shared__ uint32_t cnt[];
    for (uint32_t e = threadIdx.x; e < a.n_experts; e += 256) cnt[e] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * SORT_CHUNK;
#pragma unroll
    for (int r = 0; r < (int)(SORT_CHUNK / 256); ++r) {
        const uint32_t i = begin + r * 256 + threadIdx.x;
        const uint32_t id = i < a.total ? (uint32_t)a.experts[i] : 0xffffffffu;
        if (id < a.n_experts) atomicAdd(&cnt[id], 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.n_experts; e += 256) a.counts[(size_t)blockIdx.x * a.n_experts + e] = cnt[e];
}

// 64 experts per workgroup, 16 runs of workgroup counts each: a run's sum, the runs' exclusive scan in LDS, the prefixes
__global__ __launch_bounds__(1024) void expert_scan_kernel(SortArgs a, uint32_t blocks) {
    __shared__ uint32_t sums[16][64];
    const uint32_t e = blockIdx.x * 64 + (threadIdx.x & 63), run = threadIdx.x >> 6;
    const uint32_t per = (blocks + 15) / 16, b0 = min(blocks, run * per), b1 = min(blocks, b0 + per);
    const bool on = e < a.n_experts;
    uint32_t sum = 0;
    if (on)
#pragma unroll 8
        for (uint32_t b = b0; b < b1; ++b) sum += a.counts[(size_t)b * a.n_experts + e];
    sums[run][threadIdx.x & 63] = sum;
    __syncthreads();
    uint32_t at = 0;
    for (uint32_t r = 0; r < run; ++r) at += sums[r][threadIdx.x & 63];
    if (!on) return;
    if (run == 15) a.counts[(size_t)blocks * a.n_experts + e] = at + sum;
#pragma unroll 8
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t c = a.counts[(size_t)b * a.n_experts + e];
        a.counts[(size_t)b * a.n_experts + e] = at;
        at += c;
    }
}

__global__ __launch_bounds__(256) void expert_place_kernel(SortArgs a, uint32_t blocks, int id_bits) {
    extern __shared__ uint32_t cnt[];   // [4][n_experts]
    __shared__ uint32_t wave_sums[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t e_n = a.n_experts;
    constexpr int ROUNDS = SORT_CHUNK / 256;
    for (uint32_t i = threadIdx.x; i < 4 * e_n; i += 256) cnt[i] = 0;
    __syncthreads();
    uint32_t key[ROUNDS], rank[ROUNDS];
    const uint32_t begin = blockIdx.x * SORT_CHUNK + wave * (ROUNDS * 64);
    wave_ranks<ROUNDS>(a.experts, begin, a.total, e_n, id_bits, cnt + wave * e_n, lane, key, rank);
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < e_n; e0 += 256) {
        const uint32_t e = e0 + threadIdx.x;
        uint32_t all;
        const uint32_t first = base + block_scan<4>(e < e_n ? a.counts[(size_t)blocks * e_n + e] : 0u, wave_sums, all);
        if (e < e_n) {
            if (blockIdx.x == 0) a.offsets[e] = (int32_t)first;
            uint32_t at = first + a.counts[(size_t)blockIdx.x * e_n + e];
            for (int w = 0; w < 4; ++w) {
                const uint32_t c = cnt[w * e_n + e];
                cnt[w * e_n + e] = at;
                at += c;
            }
        }
        base += all;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[e_n] = (int32_t)base;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = begin + r * 64 + lane;
        if (i >= a.total) continue;
        const bool kept = key[r] != 0xffffffffu;
        const uint32_t at = kept ? cnt[wave * e_n + key[r]] + rank[r] : 0;
        a.slot[i] = kept ? (int32_t)at : -1;
        if (kept) a.order[at] = (int32_t)i;
        if (i >= base) a.order[i] = -1;
    }
}

void launch_expert_sort(const SortArgs& a, hipStream_t s) {
    int id_bits = 0;
    while ((1u << id_bits) < a.n_experts) ++id_bits;
    if (a.total <= 1024 && a.n_experts <= SORT_ONE_EXPERTS)
        expert_sort_one_kernel<4, 4><<<1, 256, 4 * a.n_experts * 4, s>>>(a, id_bits);
    else if (sort_in_one(a.total, a.n_experts))
        expert_sort_one_kernel<16, 16><<<1, 1024, 16 * a.n_experts * 4, s>>>(a, id_bits);
    else {
        const uint32_t blocks = sort_blocks(a.total);
        expert_count_kernel<<<blocks, 256, a.n_experts * 4, s>>>(a);
        expert_scan_kernel<<<(a.n_experts + 63) / 64, 1024, 0, s>>>(a, blocks);
        expert_place_kernel<<<blocks, 256, 4 * a.n_experts * 4, s>>>(a, blocks, id_bits);
    }
}

// ---- rows there and back ------------------------------------------------------------------------------------------
template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// HIP counts a grid's threads in 32 bits: larger grids loop
static uint32_t grid_of(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, 1u << 22); }

// a thread's elements per memory access: the widest of 16, 8, 4 bytes or one element that the row length, both
// strides and the addresses allow
static int vector_bytes(int elem, uint32_t d, std::initializer_list<uint64_t> addresses_and_strides) {
    uint64_t all = (uint64_t)d * elem;
    for (uint64_t v : addresses_and_strides) all |= v;
    for (int b : {16, 8, 4, 2})
        if (b > elem && all % b == 0) return b;
    return elem;
}

// Rows of the sorted order gathered from the samples: consecutive threads take consecutive pieces of consecutive rows,
// so the stores are whole lines also for 28-byte rows.
template <typename T>
__global__ __launch_bounds__(256) void expert_gather_kernel(const T* __restrict__ x, uint64_t ld_x, const int32_t* __restrict__ order, uint32_t total, FastDiv k,
                                                            uint32_t rows_per_block, FastDiv pieces, T* __restrict__ out, uint64_t ld_out) {
    for (uint32_t b = blockIdx.x; b * (uint64_t)rows_per_block < total; b += gridDim.x) {
        const uint32_t p0 = b * rows_per_block, rows = min(rows_per_block, total - p0);
        for (uint32_t i = threadIdx.x; i < rows * pieces.d; i += 256) {
            const uint32_t r = pieces.div(i), c = i - r * pieces.d;
            const uint32_t from = (uint32_t)order[p0 + r];
            if (from < total) out[(uint64_t)(p0 + r) * ld_out + c] = x[(uint64_t)k.div(from) * ld_x + c];
        }
    }
}

template <typename T>
static void gather(const RowsArgs& a, int elem, hipStream_t s) {
    const uint32_t per = sizeof(T) / elem, pieces = a.d / per, total = a.n * a.k;
    const uint32_t rows = std::max(1u, 1024u / pieces);
    expert_gather_kernel<T><<<grid_of((total + rows - 1) / rows), 256, 0, s>>>((const T*)a.src, a.ld_src / per, a.order, total, FastDiv(a.k), rows, FastDiv(pieces), (T*)a.dst,
                                                                     a.ld_dst / per);
}

void launch_expert_dispatch(const RowsArgs& a, hipStream_t s) {
    const int elem = a.dtype == DT_F32 ? 4 : a.dtype == DT_I8 ? 1 : 2;
    switch (vector_bytes(elem, a.d, {(uint64_t)a.src, (uint64_t)a.dst, a.ld_src * elem, a.ld_dst * elem})) {
        case 16: gather<uint4>(a, elem, s); break;
        case 8: gather<uint2>(a, elem, s); break;
        case 4: gather<uint32_t>(a, elem, s); break;
        case 2: gather<uint16_t>(a, elem, s); break;
        default: gather<uint8_t>(a, elem, s); break;
    }
}

// y[t] = sum_j w[t,j] rows[slot[t,j]], f32 in the order of j, rounded once.
template <typename T, int N>
__global__ __launch_bounds__(256) void expert_combine_kernel(RowsArgs a, uint32_t rows_per_block, FastDiv pieces) {
    using V = vec<T, N>;
    const uint32_t total = a.n * a.k;
    const V* __restrict__ src = (const V*)a.src;
    V* __restrict__ dst = (V*)a.dst;
    const uint64_t ld_src = a.ld_src / N, ld_dst = a.ld_dst / N;
    for (uint32_t b = blockIdx.x; b * (uint64_t)rows_per_block < a.n; b += gridDim.x)
    for (uint32_t i = threadIdx.x, t0 = b * rows_per_block, rows = min(rows_per_block, a.n - t0); i < rows * pieces.d; i += 256) {
        const uint32_t r = pieces.div(i), c = i - r * pieces.d;
        const uint32_t first = (t0 + r) * a.k;
        float sum[N] = {};
        for (uint32_t j = 0; j < a.k; ++j) {
            const uint32_t at = (uint32_t)a.slot[first + j];
            if (at >= total) continue;
            const V v = src[(uint64_t)at * ld_src + c];
            const float w = a.weights ? a.weights[first + j] : 1.0f;
#pragma unroll
            for (int q = 0; q < N; ++q) sum[q] = fmaf(w, (float)v[q], sum[q]);
        }
        V y;
#pragma unroll
        for (int q = 0; q < N; ++q) y[q] = (T)sum[q];
        dst[(uint64_t)(t0 + r) * ld_dst + c] = y;
    }
}

template <typename T, int N>
static void combine(const RowsArgs& a, hipStream_t s) {
    const uint32_t pieces = a.d / N, rows = std::max(1u, 256u / pieces);
    expert_combine_kernel<T, N><<<grid_of((a.n + rows - 1) / rows), 256, 0, s>>>(a, rows, FastDiv(pieces));
}

template <typename T>
static void combine_by_width(const RowsArgs& a, hipStream_t s) {
    const int elem = sizeof(T);
    const int b = vector_bytes(elem, a.d, {(uint64_t)a.src, (uint64_t)a.dst, a.ld_src * elem, a.ld_dst * elem});
    if (b == 16) combine<T, 16 / sizeof(T)>(a, s);
    else if (b == 8) combine<T, 8 / sizeof(T)>(a, s);
    else if (b == 4) combine<T, 4 / sizeof(T)>(a, s);
    else combine<T, 1>(a, s);
}

void launch_expert_combine(const RowsArgs& a, hipStream_t s) {
    if (a.dtype == DT_F16) combine_by_width<_Float16>(a, s);
    else if (a.dtype == DT_BF16) combine_by_width<__bf16>(a, s);
    else combine_by_width<float>(a, s);
}

// The gradient of the combine, sample by sample: G threads share one sample, so dy's row is read once for all its
// choices, each row of the sorted order is read and its gradient written once, and a choice's weight gradient is one
// reduction over the G threads (f32 sums, one per thread, then a tree).
template <typename T, int N, int G>
__global__ __launch_bounds__(256) void expert_combine_backward_kernel(RowsArgs a) {
    using V = vec<T, N>;
    constexpr int J = 4;   // choices per pass over dy
    __shared__ float part[4][J];
    const uint32_t total = a.n * a.k, pieces = a.d / N;
    const uint32_t g = threadIdx.x % G;
    const V* __restrict__ src = (const V*)a.src;
    const V* __restrict__ dy = (const V*)a.dy;
    V* __restrict__ dst = (V*)a.dst;
    const uint64_t ld_src = a.ld_src / N, ld_dst = a.ld_dst / N, ld_dy = a.ld_dy / N;
    // a group's lanes leave the loop together; with G = 256 the whole workgroup does
    for (uint64_t t = blockIdx.x * (uint64_t)(256 / G) + threadIdx.x / G; t < a.n; t += gridDim.x * (uint64_t)(256 / G))
    for (uint32_t j0 = 0; j0 < a.k; j0 += J) {
        uint32_t at[J];
        float w[J], dot[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const bool on = j0 + j < a.k;
            at[j] = on ? (uint32_t)a.slot[t * a.k + j0 + j] : 0xffffffffu;
            w[j] = on && a.weights ? a.weights[t * a.k + j0 + j] : 1.0f;
            dot[j] = 0.0f;
        }
        for (uint32_t c = g; c < pieces; c += G) {
            const V gv = dy[t * ld_dy + c];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (at[j] >= total) continue;
                if (a.dweights) {
                    const V v = src[(uint64_t)at[j] * ld_src + c];
#pragma unroll
                    for (int q = 0; q < N; ++q) dot[j] = fmaf((float)gv[q], (float)v[q], dot[j]);
                }
                if (dst) {
                    V o;
#pragma unroll
                    for (int q = 0; q < N; ++q) o[q] = (T)(w[j] * (float)gv[q]);
                    dst[(uint64_t)at[j] * ld_dst + c] = o;
                }
            }
        }
        if (!a.dweights) continue;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int m = (G < 64 ? G : 64) / 2; m > 0; m >>= 1) dot[j] += __shfl_xor(dot[j], m, 64);
        if constexpr (G == 256) {
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int j = 0; j < J; ++j) part[threadIdx.x >> 6][j] = dot[j];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < J; ++j) dot[j] = (part[0][j] + part[1][j]) + (part[2][j] + part[3][j]);
            __syncthreads();
        }
        if (g == 0)
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (j0 + j < a.k) a.dweights[t * a.k + j0 + j] = dot[j];
    }
}

template <typename T, int N>
static void combine_backward(const RowsArgs& a, hipStream_t s) {
    const uint32_t pieces = a.d / N;
    const auto blocks = [&](uint32_t g) { return grid_of(((uint64_t)a.n * g + 255) / 256); };
    if (pieces <= 1) expert_combine_backward_kernel<T, N, 1><<<blocks(1), 256, 0, s>>>(a);
    else if (pieces <= 4) expert_combine_backward_kernel<T, N, 4><<<blocks(4), 256, 0, s>>>(a);
    else if (pieces <= 16) expert_combine_backward_kernel<T, N, 16><<<blocks(16), 256, 0, s>>>(a);
    else if (pieces <= 128) expert_combine_backward_kernel<T, N, 64><<<blocks(64), 256, 0, s>>>(a);
    else expert_combine_backward_kernel<T, N, 256><<<grid_of(a.n), 256, 0, s>>>(a);
}

template <typename T>
static void combine_backward_by_width(const RowsArgs& a, hipStream_t s) {
    const int elem = sizeof(T);
    const int b = vector_bytes(elem, a.d, {(uint64_t)a.src, (uint64_t)a.dst, (uint64_t)a.dy, a.ld_src * elem, a.ld_dst * elem, a.ld_dy * elem});
    if (b == 16) combine_backward<T, 16 / sizeof(T)>(a, s);
    else if (b >= 4) combine_backward<T, 4 / sizeof(T)>(a, s);
    else combine_backward<T, 1>(a, s);
}

void launch_expert_combine_backward(const RowsArgs& a, hipStream_t s) {
    if (a.dtype == DT_F16) combine_backward_by_width<_Float16>(a, s);
    else if (a.dtype == DT_BF16) combine_backward_by_width<__bf16>(a, s);
    else combine_backward_by_width<float>(a, s);
}

}  // namespace sng
