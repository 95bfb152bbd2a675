// experts.hip -- samples sorted by the expert (block field) each goes to, and back with weights; forward and gradient.
//
// A choice i = t * k + j sends sample t to expert ids[i]; an id outside [0, E) drops the choice.  The plan is a stable
// counting sort: offsets[e] choices lie before expert e, slot[i] is choice i's row in the sorted order, order[row] = i.
// Behind the sort rows are scattered (dispatch, the rows' gradient: each has one source) or gathered (combine): no kernel
// here adds with atomics across workgroups, so results do not depend on the order in which workgroups run.
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
    // the counters' answers are asked for in all rounds before the first is waited for
    unsigned long long peers[ROUNDS];
    uint32_t old[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool kept = key[r] != 0xffffffffu;
        peers[r] = __ballot(kept);
        for (int b = 0; b < id_bits; ++b) {
            const bool bit = (key[r] >> b) & 1u;
            const unsigned long long m = __ballot(bit);
            peers[r] &= bit ? m : ~m;
        }
        old[r] = 0;
        if (kept && (peers[r] & ((1ull << lane) - 1ull)) == 0) old[r] = atomicAdd(&cnt[key[r]], (uint32_t)__popcll(peers[r]));
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        rank[r] = __shfl(old[r], key[r] != 0xffffffffu ? __ffsll(peers[r]) - 1 : lane, 64) + (uint32_t)__popcll(peers[r] & ((1ull << lane) - 1ull));
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

// Everything in one workgroup: ranks, the scan over waves and experts, the plan.  One launch instead of two or three for the
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
    // a thread's experts: a run of `per`, so that one scan over the workgroup does for all of them
    const uint32_t per = (e_n + NW * 64 - 1) / (NW * 64), e0 = min(e_n, threadIdx.x * per), e1 = min(e_n, e0 + per);
    uint32_t sum = 0, base;
    for (uint32_t e = e0; e < e1; ++e)
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += cnt[w * e_n + e];
    uint32_t at = block_scan<NW>(sum, wave_sums, base);
    for (uint32_t e = e0; e < e1; ++e) {
        a.offsets[e] = (int32_t)at;
        uint32_t c[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) c[w] = cnt[w * e_n + e];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            cnt[w * e_n + e] = at;
            at += c[w];
        }
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

// Bound by launches and by the chain of steps in a workgroup, not by its 12 bytes a choice: 2^21 choices of 64 experts take
// 5 + 5 + 13 us, 17000 take 11.
// Two launches or three: counts per (workgroup, expert); where they are many, their exclusive sums down the workgroups; ranks
// and the plan.
__global__ __launch_bounds__(256) void expert_count_kernel(SortArgs a, int copies) {
    extern __shared__ uint32_t cnt[];   // [copies][n_experts]: a wave's own counters where they fit, so that fewer adds meet
    for (uint32_t e = threadIdx.x; e < copies * a.n_experts; e += 256) cnt[e] = 0;
    const uint32_t begin = blockIdx.x * SORT_CHUNK;
    uint32_t id[SORT_CHUNK / 256];
#pragma unroll
    for (int r = 0; r < (int)(SORT_CHUNK / 256); ++r) {
        const uint32_t i = begin + r * 256 + threadIdx.x;
        id[r] = i < a.total ? (uint32_t)a.experts[i] : 0xffffffffu;
    }
    __syncthreads();
    uint32_t* mine = cnt + ((threadIdx.x >> 6) & (copies - 1)) * a.n_experts;
#pragma unroll
    for (int r = 0; r < (int)(SORT_CHUNK / 256); ++r)
        if (id[r] < a.n_experts) atomicAdd(&mine[id[r]], 1u);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.n_experts; e += 256) {
        uint32_t sum = cnt[e];
        for (int c = 1; c < copies; ++c) sum += cnt[c * a.n_experts + e];
        a.counts[(size_t)blockIdx.x * a.n_experts + e] = sum;
    }
}

// 64 experts per workgroup, 16 runs of workgroup counts each: a run's sum, the runs' exclusive scan in LDS, the prefixes.
// Up to HELD counts of a run stay in registers, all of them asked for at once; longer runs are read twice.
__global__ __launch_bounds__(1024) void expert_scan_kernel(SortArgs a, uint32_t blocks) {
    constexpr uint32_t HELD = 32;
    __shared__ uint32_t sums[16][64];
    const uint32_t column = threadIdx.x & 63, e = min(blockIdx.x * 64 + column, a.n_experts - 1), run = threadIdx.x >> 6;
    const uint32_t per = (blocks + 15) / 16, b0 = min(blocks, run * per), b1 = min(blocks, b0 + per);
    const bool on = blockIdx.x * 64 + column < a.n_experts;
    uint32_t* __restrict__ counts = a.counts + e;
    uint32_t held[HELD], sum = 0;
    if (per <= HELD) {
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i) held[i] = counts[(size_t)min(b0 + i, blocks - 1) * a.n_experts];
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i) {
            if (b0 + i >= b1) held[i] = 0;
            sum += held[i];
        }
    } else
#pragma unroll 8
        for (uint32_t b = b0; b < b1; ++b) sum += counts[(size_t)b * a.n_experts];
    sums[run][column] = sum;
    __syncthreads();
    uint32_t at = 0;
    for (uint32_t r = 0; r < run; ++r) at += sums[r][column];
    if (!on) return;
    if (run == 15) counts[(size_t)blocks * a.n_experts] = at + sum;
    if (per <= HELD) {
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i) {
            if (b0 + i < b1) counts[(size_t)(b0 + i) * a.n_experts] = at;
            at += held[i];
        }
    } else
#pragma unroll 8
        for (uint32_t b = b0; b < b1; ++b) {
            const uint32_t c = counts[(size_t)b * a.n_experts];
            counts[(size_t)b * a.n_experts] = at;
            at += c;
        }
}

// The rows' order goes out through LDS: a wave's lanes hold choices of as many experts as there are, and a store of theirs
// would touch as many lines; in the workgroup's own sorted order consecutive lanes write consecutive places.
// MANY: up to EXPERTS_MAX experts, in static LDS (launches take 64 KiB of the other kind).  ADDS: the counts are as
// expert_count_kernel left them, and every workgroup adds up those before its own: that is quicker than a launch while they
// are few.
template <int NW, bool MANY, bool ADDS>
__global__ __launch_bounds__(NW * 64) void expert_place_kernel(SortArgs a, uint32_t blocks, int id_bits) {
    extern __shared__ uint32_t cnt_of_call[];
    __shared__ uint32_t cnt_of_many[MANY ? (NW + 1) * EXPERTS_MAX : 1];
    uint32_t* const cnt = MANY ? cnt_of_many : cnt_of_call;   // [NW][n_experts], then [n_experts]: what to add to a place in the workgroup for the place in all
    __shared__ uint32_t wave_sums[NW];
    __shared__ uint32_t sorted[SORT_CHUNK];   // choice in the chunk (12 bits), expert
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t e_n = a.n_experts;
    constexpr int ROUNDS = SORT_CHUNK / (NW * 64);
    uint32_t* shift = cnt + NW * e_n;
    uint32_t *all = shift + e_n, *before = all + e_n;   // ADDS: of each expert, in all workgroups and in those before this one
    // a thread's experts: a run of `per`, so that one scan over the workgroup does for all of them.  Their counts are asked
    // for long before they are wanted (the first one's stay in registers).
    const uint32_t per = (e_n + NW * 64 - 1) / (NW * 64), e0 = min(e_n, threadIdx.x * per), e1 = min(e_n, e0 + per);
    const uint32_t* totals = ADDS ? all : a.counts + (size_t)blocks * e_n;
    const uint32_t* befores = ADDS ? before : a.counts + (size_t)blockIdx.x * e_n;
    uint32_t total0 = 0, before0 = 0;
    if (!ADDS && e0 < e1) {
        total0 = totals[e0];
        before0 = befores[e0];
    }
    for (uint32_t i = threadIdx.x; i < (ADDS ? NW + 3 : NW) * e_n; i += NW * 64) cnt[i] = 0;
    __syncthreads();
    if constexpr (ADDS) {   // consecutive threads take the experts of one workgroup's counts, as many times as there is room
        const uint32_t width = min(1u << id_bits, (uint32_t)(NW * 64)), parts = NW * 64 / width, part = threadIdx.x / width;
        for (uint32_t e = threadIdx.x % width; e < e_n; e += width) {
            uint32_t sum = 0, lower = 0;
#pragma unroll 8
            for (uint32_t b = part; b < blocks; b += parts) {
                const uint32_t c = a.counts[(size_t)b * e_n + e];
                sum += c;
                lower += b < blockIdx.x ? c : 0u;
            }
            atomicAdd(&all[e], sum);
            atomicAdd(&before[e], lower);
        }
    }
    uint32_t key[ROUNDS], rank[ROUNDS];
    const uint32_t chunk = blockIdx.x * SORT_CHUNK, begin = chunk + wave * (ROUNDS * 64);
    wave_ranks<ROUNDS>(a.experts, begin, a.total, e_n, id_bits, cnt + wave * e_n, lane, key, rank);
    __syncthreads();
    if (ADDS && e0 < e1) {
        total0 = totals[e0];
        before0 = befores[e0];
    }
    uint32_t here = 0, total = total0, base, local_base;
    for (uint32_t e = e0; e < e1; ++e) {
        if (e > e0) total += totals[e];
#pragma unroll
        for (int w = 0; w < NW; ++w) here += cnt[w * e_n + e];
    }
    uint32_t local = block_scan<NW>(here, wave_sums, local_base), first = block_scan<NW>(total, wave_sums, base);
    for (uint32_t e = e0; e < e1; ++e) {
        if (blockIdx.x == 0) a.offsets[e] = (int32_t)first;
        shift[e] = first + (e > e0 ? befores[e] : before0) - local;
        first += e > e0 ? totals[e] : total0;
        uint32_t c[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) c[w] = cnt[w * e_n + e];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            cnt[w * e_n + e] = local;
            local += c[w];
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[e_n] = (int32_t)base;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = begin + r * 64 + lane;
        if (i >= a.total) continue;
        const bool kept = key[r] != 0xffffffffu;
        const uint32_t at = kept ? cnt[wave * e_n + key[r]] + rank[r] : 0;
        a.slot[i] = kept ? (int32_t)(at + shift[key[r]]) : -1;
        if (kept) sorted[at] = key[r] << 12 | (i - chunk);
        if (i >= base) a.order[i] = -1;
    }
    __syncthreads();
    for (uint32_t l = threadIdx.x; l < local_base; l += NW * 64) a.order[l + shift[sorted[l] >> 12]] = (int32_t)(chunk + (sorted[l] & 4095u));
}
static_assert(SORT_CHUNK == 4096 && EXPERTS_MAX <= 1 << 20, "a choice of the chunk and its expert share 32 bits");

// (64 experts: 400000 choices, 6272 counts, 14.5 us for 15.7 with the scan's launch; 2^20 choices, 16384 counts, 20.5 for 16.8;
// 16 experts, 2^20: 4096 counts, 13.8 for 16.1)
constexpr uint64_t SORT_ADD_COUNTS = 1 << 13;

void launch_expert_sort(const SortArgs& a, hipStream_t s) {
    int id_bits = 0;
    while ((1u << id_bits) < a.n_experts) ++id_bits;
    if (a.total <= 1024 && a.n_experts <= SORT_ONE_EXPERTS)
        expert_sort_one_kernel<4, 4><<<1, 256, 4 * a.n_experts * 4, s>>>(a, id_bits);
    else if (a.total <= 4096 && a.n_experts <= SORT_ONE_EXPERTS)
        expert_sort_one_kernel<8, 8><<<1, 512, 8 * a.n_experts * 4, s>>>(a, id_bits);
    else if (sort_in_one(a.total, a.n_experts))
        expert_sort_one_kernel<16, 16><<<1, 1024, 16 * a.n_experts * 4, s>>>(a, id_bits);
    else {
        const uint32_t blocks = sort_blocks(a.total);
        const int copies = a.n_experts <= 1024 ? 4 : 1;
        expert_count_kernel<<<blocks, 256, copies * a.n_experts * 4, s>>>(a, copies);
        if (a.n_experts <= 1024 && (uint64_t)blocks * a.n_experts <= SORT_ADD_COUNTS) {
            expert_place_kernel<8, false, true><<<blocks, 512, 11 * a.n_experts * 4, s>>>(a, blocks, id_bits);
            return;
        }
        expert_scan_kernel<<<(a.n_experts + 63) / 64, 1024, 0, s>>>(a, blocks);
        if (a.n_experts <= 1024) expert_place_kernel<8, false, false><<<blocks, 512, 9 * a.n_experts * 4, s>>>(a, blocks, id_bits);
        else expert_place_kernel<4, true, false><<<blocks, 256, 0, s>>>(a, blocks, id_bits);
    }
}

// ---- rows there and back ------------------------------------------------------------------------------------------
template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// HIP counts a grid's threads in 32 bits: larger grids loop
static uint32_t grid_of(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, 1u << 22); }

// A row of d elements in pieces of N, each one memory access of up to 16 bytes: the last piece ends with the row and may
// repeat elements of the one before it (the same values, written twice).  Pieces lie at any multiple of an element, which
// the card's loads and stores take; d = 45 in f16 goes in 6 pieces and not in 45.
struct Pieces {
    FastDiv count;
    uint32_t d, n;
    Pieces(uint32_t d, uint32_t n) : count((d + n - 1) / n), d(d), n(n) {}
    __device__ __forceinline__ uint32_t start(uint32_t c) const { return min(c * n, d - n); }
};
static int piece_bytes(int elem, uint32_t d) {
    for (int b : {16, 8, 4, 2})
        if (b > elem && (uint64_t)d * elem >= (uint64_t)b) return b;
    return elem;
}
template <typename V>
__device__ __forceinline__ V get_piece(const void* p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <typename V>
__device__ __forceinline__ void put_piece(void* p, const V& v) { __builtin_memcpy(p, &v, sizeof(V)); }

// Each sample's row to all its places: x is read once and in order, and a row's pieces go out together.  (The other way
// round, rows of the sorted order gathered, reads a cache line of x for each 28-byte row: 2^20 x 2 such rows 45 us, this way
// 23, or 27 with nothing in the card's caches.)  Bound by memory, there by the parts of lines that its writes touch: 4.1 TB/s.
// Two choices are asked for together with the pieces: 2^20 x 2 rows of 28 bytes 26.8 us, in the loop over k 27.8; 2^18 x 2 of
// 68 bytes 20.9 and 23.4, of 252 bytes 57 and 60.
template <typename T, int K>   // a piece's bytes; K > 0: k, whose places are asked for together with the pieces
__global__ __launch_bounds__(256) void expert_scatter_kernel(RowsArgs a, uint32_t elem, uint32_t samples_per_block, Pieces pieces) {
    constexpr int U = 4;
    const uint32_t total = a.n * a.k;
    const char* __restrict__ x = (const char*)a.src;
    char* __restrict__ out = (char*)a.dst;
    for (uint64_t t0 = blockIdx.x * (uint64_t)samples_per_block; t0 < a.n; t0 += gridDim.x * (uint64_t)samples_per_block) {
        const uint32_t samples = min((uint64_t)samples_per_block, a.n - t0), count = samples * pieces.count.d;
        for (uint32_t i0 = threadIdx.x; i0 < count; i0 += 256 * U) {
            uint32_t t[U], c[U];
            T v[U];
            uint32_t places[U][K ? K : 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = min(i0 + u * 256, count - 1);
                t[u] = pieces.count.div(i);
                c[u] = pieces.start(i - t[u] * pieces.count.d);
                v[u] = get_piece<T>(x + ((t0 + t[u]) * a.ld_src + c[u]) * elem);
                if constexpr (K > 0) __builtin_memcpy(places[u], a.slot + (t0 + t[u]) * K, sizeof(places[u]));
            }
            if constexpr (K > 0) {
#pragma unroll
                for (int j = 0; j < K; ++j)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (places[u][j] < total && i0 + u * 256 < count) put_piece(out + ((uint64_t)places[u][j] * a.ld_dst + c[u]) * elem, v[u]);
            } else {
                for (uint32_t j = 0; j < a.k; ++j) {
                    uint32_t to[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) to[u] = (uint32_t)a.slot[(t0 + t[u]) * a.k + j];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (to[u] < total && i0 + u * 256 < count) put_piece(out + ((uint64_t)to[u] * a.ld_dst + c[u]) * elem, v[u]);
                }
            }
        }
    }
}

template <typename T>
static void scatter(const RowsArgs& a, uint32_t elem, hipStream_t s) {
    const Pieces pieces(a.d, sizeof(T) / elem);
    // Rows of half a line and less: one workgroup a CU, with a run of samples each, so that the parts of a line that its steps
    // write one after the other meet in the die's cache.  (Nothing in the caches: 2^20 x 2 rows of 28 bytes 26.8 us, 38.1 in as many
    // workgroups as fit; 2^18 x 4 of them 17.4 and 22.9; 2^18 x 2 rows of 64 bytes 14.4 and 15.0, of 128 bytes 23.9 and 22.1;
    // 16384 x 2 of 4096 bytes 41.7 and 39.1.)
    const uint32_t few = a.d * elem <= 64 ? (a.n + 255) / 256 : 1, samples = std::max(std::max(1u, 1024u / pieces.count.d), few);
    const uint32_t grid = grid_of((a.n + samples - 1) / samples);
    if (a.k == 2) expert_scatter_kernel<T, 2><<<grid, 256, 0, s>>>(a, elem, samples, pieces);
    else expert_scatter_kernel<T, 0><<<grid, 256, 0, s>>>(a, elem, samples, pieces);
}

void launch_expert_dispatch(const RowsArgs& a, hipStream_t s) {
    const int elem = a.dtype == DT_F32 ? 4 : a.dtype == DT_I8 ? 1 : 2;
    switch (piece_bytes(elem, a.d)) {
        case 16: scatter<uint4>(a, elem, s); break;
        case 8: scatter<uint2>(a, elem, s); break;
        case 4: scatter<uint32_t>(a, elem, s); break;
        case 2: scatter<uint16_t>(a, elem, s); break;
        default: scatter<uint8_t>(a, elem, s); break;
    }
}

// y[t] = sum_j w[t,j] rows[slot[t,j]], f32 in the order of j, rounded once.  The places and weights of J choices are asked
// for together, then their J pieces, so that a thread waits twice for J choices and not twice for each.  Bound by memory:
// 4099 x 8 rows of 4096 bf16, 302 MB, 64 us (4.7 TB/s); 2^20 x 2 rows of 4 f16, 42 MB, 9.0 us where the rows are in the card's
// caches (4.7), 13.9 from memory (3.0).
template <typename T, int N, int J>
__global__ __launch_bounds__(256) void expert_combine_kernel(RowsArgs a, uint32_t rows_per_block, Pieces pieces) {
    using V = vec<T, N>;
    const uint32_t total = a.n * a.k;
    const T* __restrict__ src = (const T*)a.src;
    T* __restrict__ dst = (T*)a.dst;
    for (uint32_t b = blockIdx.x; b * (uint64_t)rows_per_block < a.n; b += gridDim.x)
#pragma unroll J <= 2 ? 2 : 1
        for (uint32_t i = threadIdx.x, t0 = b * rows_per_block, rows = min(rows_per_block, a.n - t0); i < rows * pieces.count.d; i += 256) {
            const uint32_t r = pieces.count.div(i), c = pieces.start(i - r * pieces.count.d);
            const uint32_t first = (t0 + r) * a.k;
            float sum[N] = {};
            for (uint32_t j0 = 0; j0 < a.k; j0 += J) {
                uint32_t at[J];
                float w[J];
                V v[J];
                if (J <= 2 || a.k == J) {   // all of a sample's choices in one load (2^18 x 8 rows of 8 f16 14.4 us, one by one 17.1)
                    __builtin_memcpy(at, a.slot + first, sizeof(at));
                    if (a.weights) __builtin_memcpy(w, a.weights + first, sizeof(w));
                    else
#pragma unroll
                        for (int j = 0; j < J; ++j) w[j] = 1.0f;
                } else
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const uint32_t i = first + min(j0 + j, a.k - 1);
                        at[j] = (uint32_t)a.slot[i];
                        w[j] = a.weights ? a.weights[i] : 1.0f;
                    }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (j0 + j >= a.k) at[j] = total;
                    v[j] = at[j] < total ? get_piece<V>(src + (uint64_t)at[j] * a.ld_src + c) : V(0);
                }
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (at[j] < total)
#pragma unroll
                        for (int q = 0; q < N; ++q) sum[q] = fmaf(w[j], (float)v[j][q], sum[q]);
            }
            V y;
#pragma unroll
            for (int q = 0; q < N; ++q) y[q] = (T)sum[q];
            put_piece(dst + (uint64_t)(t0 + r) * a.ld_dst + c, y);
        }
}

template <typename T, int N>
static void combine(const RowsArgs& a, hipStream_t s) {
    const Pieces pieces(a.d, N);
    // four pieces a thread where there is work for the chip in that, and a sample's choices are one load (rows in the caches, as a
    // layer that has just written them leaves them: 2^20 x 2 rows of 4 f16 9.0 us, one piece a thread 11.9; 2^18 x 4 rows 6.1 and
    // 5.3, 2^18 x 2 rows of 128 28.2 and 27.6; from memory one piece is ahead: 13.9 and 13.2, 2^18 x 2 rows of 16 10.0 and 8.6)
    const bool four = a.k <= 2 && pieces.count.d <= 8 && (uint64_t)a.n * pieces.count.d >= 1u << 19;
    const uint32_t rows = std::max(1u, (four ? 1024u : 256u) / pieces.count.d), grid = grid_of((a.n + rows - 1) / rows);
    if (a.k == 1) expert_combine_kernel<T, N, 1><<<grid, 256, 0, s>>>(a, rows, pieces);
    else if (a.k == 2) expert_combine_kernel<T, N, 2><<<grid, 256, 0, s>>>(a, rows, pieces);
    else if (a.k <= 4) expert_combine_kernel<T, N, 4><<<grid, 256, 0, s>>>(a, rows, pieces);
    else expert_combine_kernel<T, N, 8><<<grid, 256, 0, s>>>(a, rows, pieces);
}

template <typename T>
static void combine_by_width(const RowsArgs& a, hipStream_t s) {
    const int n = piece_bytes(sizeof(T), a.d) / sizeof(T);
    if constexpr (sizeof(T) == 2) {
        if (n == 8) return combine<T, 8>(a, s);
    }
    if (n == 4) combine<T, 4>(a, s);
    else if (n == 2) combine<T, 2>(a, s);
    else combine<T, 1>(a, s);
}

void launch_expert_combine(const RowsArgs& a, hipStream_t s) {
    if (a.dtype == DT_F16) combine_by_width<_Float16>(a, s);
    else if (a.dtype == DT_BF16) combine_by_width<__bf16>(a, s);
    else combine_by_width<float>(a, s);
}

// The gradient of the combine, sample by sample: G threads share one sample, so dy's row is read once for four of its
// choices, each row of the sorted order is read and its gradient written once, and a choice's weight gradient is one
// reduction over the G threads (f32 sums, one per thread, then a tree).  Bound by memory: 16384 x 2 rows of 2048 f16,
// 336 MB, 63 us (5.3 TB/s, a large copy's rate).
template <typename T, int N, int G>
__global__ __launch_bounds__(256) void expert_combine_backward_kernel(RowsArgs a) {
    using V = vec<T, N>;
    constexpr int J = 4;   // choices per pass over dy
    __shared__ float part[4][J];
    const uint32_t total = a.n * a.k, pieces = (a.d + N - 1) / N;
    const uint32_t g = threadIdx.x % G;
    const T* __restrict__ src = (const T*)a.src;
    const T* __restrict__ dy = (const T*)a.dy;
    T* __restrict__ dst = (T*)a.dst;
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
            const uint32_t at_c = min(c * N, a.d - N), seen = c * N - at_c;   // (the last piece's elements that the one before has: not summed again)
            const V gv = get_piece<V>(dy + t * a.ld_dy + at_c);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (at[j] >= total) continue;
                if (a.dweights) {
                    const V v = get_piece<V>(src + (uint64_t)at[j] * a.ld_src + at_c);
#pragma unroll
                    for (int q = 0; q < N; ++q) dot[j] = (uint32_t)q >= seen ? fmaf((float)gv[q], (float)v[q], dot[j]) : dot[j];
                }
                if (dst) {
                    V o;
#pragma unroll
                    for (int q = 0; q < N; ++q) o[q] = (T)(w[j] * (float)gv[q]);
                    put_piece(dst + (uint64_t)at[j] * a.ld_dst + at_c, o);
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
    const uint32_t pieces = (a.d + N - 1) / N;
    const auto blocks = [&](uint32_t g) { return grid_of(((uint64_t)a.n * g + 255) / 256); };
    if (pieces <= 1) expert_combine_backward_kernel<T, N, 1><<<blocks(1), 256, 0, s>>>(a);
    else if constexpr (N * sizeof(T) < 16) {   // pieces below 16 bytes: the row is shorter than two of them (one element: one)
        if constexpr (N > 1) expert_combine_backward_kernel<T, N, 4><<<blocks(4), 256, 0, s>>>(a);
    } else if (pieces <= 4) expert_combine_backward_kernel<T, N, 4><<<blocks(4), 256, 0, s>>>(a);
    else if (pieces <= 16) expert_combine_backward_kernel<T, N, 16><<<blocks(16), 256, 0, s>>>(a);
    else if (pieces <= 128) expert_combine_backward_kernel<T, N, 64><<<blocks(64), 256, 0, s>>>(a);
    else expert_combine_backward_kernel<T, N, 256><<<grid_of(a.n), 256, 0, s>>>(a);
}

template <typename T>
static void combine_backward_by_width(const RowsArgs& a, hipStream_t s) {
    const int n = piece_bytes(sizeof(T), a.d) / sizeof(T);
    if constexpr (sizeof(T) == 2) {
        if (n == 8) return combine_backward<T, 8>(a, s);
    }
    if (n == 4) combine_backward<T, 4>(a, s);
    else if (n == 2) combine_backward<T, 2>(a, s);
    else combine_backward<T, 1>(a, s);
}

void launch_expert_combine_backward(const RowsArgs& a, hipStream_t s) {
    if (a.dtype == DT_F16) combine_backward_by_width<_Float16>(a, s);
    else if (a.dtype == DT_BF16) combine_backward_by_width<__bf16>(a, s);
    else combine_backward_by_width<float>(a, s);
}

}  // namespace sng
