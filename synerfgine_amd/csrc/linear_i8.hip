// linear_i8.hip -- the linear layer in 8-bit integers: rows brought to 8 bits with a scale each, times 8-bit weights with
// a scale for each output channel, on the int8 matrix instructions; dense, or by expert for rows sorted by expert.
//
//   y[r,c] = act( (sum_k q[r,k] w[c,k]) * ws[c] * s[r] + b[c] )
//
// The sum is exact (int32; n_in <= 131071), the rest is f32 and is rounded once, to y's type.
#include "linear_i8.h"

namespace sng {

// ---- rows to 8 bits: the kernel --------------------------------------------------------------------------------------
// G threads share a row and hold up to C pieces of 16 bytes each (of PB = 16; one element where the row's place or length
// allows no more) between the two passes; longer rows are read again.  Consecutive threads take consecutive pieces.  Bound
// by memory: 8192 x 4096 bf16, 100 MB, 22 us (4.6 TB/s).
template <int DT, int PB, int G>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
    constexpr int XB = bytes_of(DT), N = PB / XB, C = 8;
    using Bytes = Raw<DT, N < 4 / XB ? 4 / XB : N>;   // (one 16-bit element: a word with a zero beside it)
    __shared__ uint32_t part[4];
    const uint32_t g = threadIdx.x % G, pieces = a.cols / N;
    for (uint64_t r = blockIdx.x * (uint64_t)(256 / G) + threadIdx.x / G; r < a.rows; r += gridDim.x * (uint64_t)(256 / G)) {
        const char* __restrict__ x = (const char*)a.x + r * a.ld_x * XB;
        int8_t* __restrict__ out = a.q + r * a.ld_q;
        const auto get = [&](uint32_t c) {
            Bytes w = {};
            __builtin_memcpy(&w, __builtin_assume_aligned(x + (uint64_t)c * PB, PB), PB);
            return w;
        };
        Bytes held[C];
#pragma unroll
        for (int i = 0; i < C; ++i) held[i] = get(min(g + i * G, pieces - 1));   // (a piece twice does not change the maximum)
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < C; ++i) top = max(top, top_bits(held[i]));
        for (uint32_t c = g + C * G; c < pieces; c += G) top = max(top, top_bits(get(c)));
#pragma unroll
        for (int m = (G < 64 ? G : 64) / 2; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
        if constexpr (G == 256) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
            __syncthreads();
            top = max(max(part[0], part[1]), max(part[2], part[3]));
            __syncthreads();
        }
        const RowScale rs = row_scale(top);
        if (g == 0) a.scale[r] = rs.scale;
        const auto put = [&](uint32_t c, const Bytes& w) {
            if constexpr (N == 1) out[c] = (int8_t)(rs.finite ? quantize_careful(element(w, 0), rs.inv, rs.a) : 0);
            else {
                auto q = quantize_n(w, rs);
                if (!rs.finite) q = q ^ q;
                ((decltype(q)*)out)[c] = q;
            }
        };
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (g + i * G < pieces) put(g + i * G, held[i]);
        for (uint32_t c = g + C * G; c < pieces; c += G) put(c, get(c));
        for (uint32_t c = a.cols + g; c < a.cols_written; c += G) out[c] = 0;
    }
}

// The same for rows at any place and of any length, to rows padded and aligned as the tiles want them: units of 16 values.
template <int DT, int G>
__global__ __launch_bounds__(256) void quantize_units_kernel(QuantArgs a) {
    constexpr int XB = bytes_of(DT), C = 4;
    __shared__ uint32_t part[4];
    const uint32_t g = threadIdx.x % G, units = a.cols_written / 16, n = a.cols;
    for (uint64_t r = blockIdx.x * (uint64_t)(256 / G) + threadIdx.x / G; r < a.rows; r += gridDim.x * (uint64_t)(256 / G)) {
        const char* __restrict__ x = (const char*)a.x + r * a.ld_x * XB;
        Raw<DT, 16> held[C];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < C; ++i) held[i] = load_row16<DT>(x, (g + i * G) * 16, n);   // (past the end: the row's last 16 again)
#pragma unroll
        for (int i = 0; i < C; ++i) top = max(top, top_bits(held[i]));
        for (uint32_t u = g + C * G; u < units; u += G) top = max(top, top_bits(load_row16<DT>(x, u * 16, n)));
#pragma unroll
        for (int m = (G < 64 ? G : 64) / 2; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
        if constexpr (G == 256) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
            __syncthreads();
            top = max(max(part[0], part[1]), max(part[2], part[3]));
            __syncthreads();
        }
        const RowScale rs = row_scale(top);
        if (g == 0) a.scale[r] = rs.scale;
        const auto put = [&](Raw<DT, 16> v, uint32_t u) {
            v = inside<DT>(v, u * 16, n);
            i4 q = quantize_n(v, rs);
            if (!rs.finite) q = i4{0, 0, 0, 0};
            *(i4*)(a.q + r * a.ld_q + u * 16) = q;
        };
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (g + i * G < units) put(held[i], g + i * G);
        for (uint32_t u = g + C * G; u < units; u += G) put(load_row16<DT>(x, u * 16, n), u);
    }
}

// 8-bit rows (weights) to padded and aligned ones, `rows_per_block` rows a workgroup
__global__ __launch_bounds__(256) void pad_rows_kernel(const int8_t* __restrict__ w, uint64_t ld_w, uint32_t n, uint64_t rows, FastDiv units, uint32_t rows_per_block,
                                                       int8_t* __restrict__ to) {
    for (uint64_t r0 = blockIdx.x * (uint64_t)rows_per_block; r0 < rows; r0 += gridDim.x * (uint64_t)rows_per_block) {
        const uint32_t count = (uint32_t)min((uint64_t)rows_per_block, rows - r0) * units.d;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < count; i += 256) {
            const uint32_t r = units.div(i), u = i - r * units.d;
            Raw<DT_I8, 16> v = whole(load_odd16((const char*)w + (r0 + r) * ld_w, u * 16, n));
            v = inside<DT_I8>(v, u * 16, n);
            *(i4*)(to + (r0 * units.d + i) * 16) = as_fragment(v);
        }
    }
}

static uint32_t grid_of(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, 1u << 22); }

template <int DT, int PB>
static void quantize_by_length(const QuantArgs& a, hipStream_t s) {
    const uint32_t pieces = a.cols / (PB / bytes_of(DT));
    const auto blocks = [&](uint32_t g) { return grid_of(((uint64_t)a.rows * g + 255) / 256); };
    if (pieces <= 32) quantize_rows_kernel<DT, PB, 4><<<blocks(4), 256, 0, s>>>(a);
    else if (pieces <= 128) quantize_rows_kernel<DT, PB, 16><<<blocks(16), 256, 0, s>>>(a);
    else if (pieces <= 512 && a.rows >= 2048) quantize_rows_kernel<DT, PB, 64><<<blocks(64), 256, 0, s>>>(a);   // no barrier; fewer rows: more waves a row
    else quantize_rows_kernel<DT, PB, 256><<<blocks(256), 256, 0, s>>>(a);
}

template <int DT>
static void quantize(const QuantArgs& a, hipStream_t s) {
    constexpr int XB = bytes_of(DT), N = 16 / XB;
    const bool wide = a.cols % N == 0 && ((uint64_t)a.x | (a.ld_x * XB)) % 16 == 0 && ((uint64_t)a.q | a.ld_q) % N == 0;
    if (wide) quantize_by_length<DT, 16>(a, s);
    else if (((uint64_t)a.q | a.ld_q | a.cols_written) % 16 == 0 && a.cols >= 16) {
        const uint32_t units = a.cols_written / 16;
        const auto blocks = [&](uint32_t g) { return grid_of(((uint64_t)a.rows * g + 255) / 256); };
        if (units <= 64) quantize_units_kernel<DT, 16><<<blocks(16), 256, 0, s>>>(a);
        else if (units <= 256 && a.rows >= 2048) quantize_units_kernel<DT, 64><<<blocks(64), 256, 0, s>>>(a);
        else quantize_units_kernel<DT, 256><<<blocks(256), 256, 0, s>>>(a);
    } else quantize_by_length<DT, XB>(a, s);
}

void launch_pad_rows(const int8_t* w, uint64_t ld_w, uint32_t n, uint64_t rows, uint32_t padded, int8_t* to, hipStream_t s) {
    const uint32_t per = std::max(1u, 1024 / (padded / 16));   // 4 units a thread
    pad_rows_kernel<<<grid_of((rows + per - 1) / per), 256, 0, s>>>(w, ld_w, n, rows, FastDiv(padded / 16), per, to);
}

void launch_quantize_rows(const QuantArgs& a, hipStream_t s) {
    if (a.dtype == DT_F16) quantize<DT_F16>(a, s);
    else if (a.dtype == DT_BF16) quantize<DT_BF16>(a, s);
    else quantize<DT_F32>(a, s);
}

template <typename T, int N>
__device__ __forceinline__ void store_channels(T* __restrict__ y, const float (&v)[N], uint32_t left, bool aligned) {
    if (aligned && left >= N) {
        constexpr int P = 16 / sizeof(T);
#pragma unroll
        for (int p = 0; p < N / P; ++p) {
            vec<T, P> o;
#pragma unroll
            for (int q = 0; q < P; ++q) o[q] = (T)v[p * P + q];
            ((vec<T, P>*)y)[p] = o;
        }
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q)
            if ((uint32_t)q < left) y[q] = (T)v[q];
    }
}

// ---- tiles ------------------------------------------------------------------------------------------------------------
// For 8-bit rows or weights given at places or with strides that the tiles below do not take; 4 to 10 times their time.
// The matrix instruction's rows are output channels and its columns input rows, so a lane's accumulators are channels of
// one row; tile t's row 4g + i is channel 16 g + 4 t + i of the wave's 64, which makes a lane's 16 values one piece of y.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void linear_i8_tile_kernel(LinearArgs a) {
    constexpr int BK = 128, XT = BM / 32, CHUNKS = (BM + BN) * 8 / 256;
    static_assert(BN == 128, "two waves of 64 channels");
    __shared__ __align__(16) int8_t lds[(BM + BN) * BK];
    const RowTile tile = row_tile(a, blockIdx.x, BM == 128 ? 7 : 8);
    if (tile.begin >= tile.end) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t n0 = blockIdx.y * BN;
    const int8_t* __restrict__ w = a.w + (uint64_t)tile.expert * a.n_out * a.ld_w;
    const int wm = (wave & 1) * (BM / 2), wn = (wave >> 1) * 64;
    i4 acc[4][XT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int u = 0; u < XT; ++u) acc[t][u] = i4{0, 0, 0, 0};
    // rows of the LDS tile: [0, BM) input rows, [BM, BM + BN) channels; 16-byte pieces of a row are placed by key(row) so
    // that the lanes of a fragment read hit different banks
    const auto key = [](uint32_t row) { return (row & 3u) | ((row >> 2) & 4u); };
    const auto keyx = [](uint32_t row) { return row & 7u; };
    Raw<DT_I8, 16> next[CHUNKS];
    const auto load = [&](uint32_t k0) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t c = threadIdx.x + i * 256, row = c >> 3, k = k0 + (c & 7) * 16;
            const int8_t* from = row < BM ? (const int8_t*)a.x + (uint64_t)min(tile.begin + row, tile.end - 1) * a.ld_x : w + (uint64_t)min(n0 + row - BM, a.n_out - 1) * a.ld_w;
            next[i] = load_row16<DT_I8>((const char*)from, k, a.n_in);
        }
    };
    load(0);
    for (uint32_t k0 = 0; k0 < a.n_in; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t c = threadIdx.x + i * 256, row = c >> 3, piece = c & 7;
            i4 v = as_fragment(next[i]);
            if (k0 + BK > a.n_in) v = new_bytes(v, k0 + piece * 16, a.n_in);
            *(i4*)(lds + row * BK + ((piece ^ (row < BM ? keyx(row) : key(row - BM))) * 16)) = v;
        }
        __syncthreads();
        if (k0 + BK < a.n_in) load(k0 + BK);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t piece = h * 4 + (lane >> 4);
            i4 fx[XT], fw[4];
#pragma unroll
            for (int u = 0; u < XT; ++u) {
                const uint32_t row = wm + u * 16 + (lane & 15);
                fx[u] = *(const i4*)(lds + row * BK + ((piece ^ keyx(row)) * 16));
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t row = wn + ((lane >> 2) & 3) * 16 + t * 4 + (lane & 3);
                fw[t] = *(const i4*)(lds + (BM + row) * BK + ((piece ^ key(row)) * 16));
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int u = 0; u < XT; ++u) acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[t], fx[u], acc[t][u], 0, 0, 0);
        }
    }
    const uint32_t c0 = n0 + wn + (lane >> 4) * 16;
    if (c0 >= a.n_out) return;
    const uint32_t left = a.n_out - c0;
    const bool aligned = (((uint64_t)a.y | (a.ld_y * sizeof(T))) & 15) == 0;
    float ws[16], b[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const bool on = (uint32_t)q < left;
        ws[q] = on ? a.w_scale[(uint64_t)tile.expert * a.n_out + c0 + q] : 0.0f;
        b[q] = on && a.bias ? a.bias[(uint64_t)tile.expert * a.n_out + c0 + q] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < XT; ++u) {
        const uint32_t row = tile.begin + wm + u * 16 + (lane & 15);
        if (row >= tile.end) continue;
        const float s = a.x_scale[row];
        float v[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            v[q] = finish(acc[q >> 2][u][q & 3], ws[q], s, b[q], lowest(a));
        }
        store_channels<T, 16>((T*)a.y + (uint64_t)row * a.ld_y + c0, v, left, aligned);
    }
}

// The same product with both tiles brought straight into LDS (global_load_lds, 16 bytes a lane): no registers and no
// instructions stand between memory and the matrix units.  Steps of 128 bytes of n_in (whole cache lines), a stage of LDS
// each, in halves: while one half is multiplied from registers the next is read from LDS.  Once a step's second half is in
// registers its stage is free: the one barrier of the step, behind which the loads of STAGES steps ahead refill it.  Loads and
// reads are spread between the matrix instructions: behind the barrier every wave would else queue its loads first and
// the matrix units would wait for the queue.  A lane fetches the piece of its row that belongs at its place in LDS, which
// keeps the lanes of a fragment read on different banks.
// Wants n_in, both strides and both addresses in multiples of 16 bytes.
// 8192 x 4096 -> 8192: 237 us, 2.3 * 10^15 operations a second (torch's int8 product into int32: 281 us).  What bounds it is
// the card's power: an earlier form took 290 us of random values and 203 of zeros.  By expert (16384 rows on 16, 2048 -> 4096) 179 us: row tiles that an
// expert fills in part (an eighth of the work) and 4.5 rounds of tiles that take the time of 5.
__device__ const int8_t zeros16[16] __attribute__((aligned(16))) = {};

// workgroups go round the 8 dies one by one: each die gets a run of neighbouring tiles, in columns of 4 row tiles, so
// that its cache sees the same rows and channels again
struct TilePlace { uint32_t row, col; };
__device__ __forceinline__ TilePlace tile_place(uint32_t id, uint32_t col_tiles, uint32_t tiles) {
    const uint32_t group = id / (4 * col_tiles), in = id - group * 4 * col_tiles, high = min(4u, tiles / col_tiles - group * 4);
    return {group * 4 + in % high, in / high};
}
// The sums of a wave's XT fragments of rows from row0 on by 64 channels from c0 on, to y
template <int XT, bool WIDE>
__device__ __forceinline__ void finish_tile(const LinearArgs& a, const RowTile& tile, uint32_t row0, uint32_t c0, uint32_t g, uint32_t r, const i4 (&acc)[4][XT]) {
    if (c0 >= a.n_out) return;
    float ws[16], b[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const uint32_t c = c0 + channel_of(q >> 2, g, WIDE) + (q & 3);
        const uint64_t at = (uint64_t)tile.expert * a.n_out + min(c, a.n_out - 1);
        ws[q] = a.w_scale[at];
        b[q] = a.bias ? a.bias[at] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < XT; ++u) {
        const uint32_t row = row0 + u * 16 + r;
        if (row >= tile.end) continue;
        const float s = a.x_scale[row];
        float v[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) v[q] = finish(acc[q >> 2][u][q & 3], ws[q], s, b[q], lowest(a));
        store_block(a, row, c0, g, v, a.n_out - c0);
    }
}

// A wave holds BM / WR rows by 64 channels.  SPLIT: a workgroup takes one of a.splits runs of the steps and leaves its sums
// in a.partial; linear_i8_join_kernel adds them.
template <int BM, int BN, int WR, int STAGES, bool WIDE, bool SPLIT = false>
__global__ __launch_bounds__(BN * WR) void linear_i8_stream_kernel(LinearArgs a, uint32_t col_tiles, uint32_t tiles) {
    constexpr int WC = BN / 64, WAVES = WR * WC, XT = BM / WR / 16, BK = 128, STAGE = (BM + BN) * BK;
    constexpr int LOADS = (BM + BN) / 8 / WAVES;   // each brings 8 rows of 128 bytes
    __shared__ __align__(16) int8_t lds[STAGES * STAGE];
    const uint32_t all = SPLIT ? tiles * a.splits : tiles, per = (all + 7) / 8, place = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (place >= all) return;
    const uint32_t split = SPLIT ? place / tiles : 0, id = place - split * tiles;
    const TilePlace at = tile_place(id, col_tiles, tiles);
    const RowTile tile = row_tile(a, at.row, BM == 256 ? 8 : BM == 128 ? 7 : 6);
    if (tile.begin >= tile.end) return;
    const uint32_t all_steps = (a.n_in + BK - 1) / BK, first = SPLIT ? all_steps * split / a.splits : 0;
    const uint32_t steps = (SPLIT ? all_steps * (split + 1) / a.splits : all_steps) - first, n_in = min(steps * BK, a.n_in - first * BK);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15, n0 = at.col * BN;
    const uint32_t wm = wave / WC * (BM / WR), wn = wave % WC * 64;
    // this lane's loads: tile rows (wave + i * WAVES) * 8 + lane / 8.  Place p of fragment row r holds piece p ^ (r / 2 & 7):
    // the 16 lanes that LDS serves at a time (0-3, 12-15, 20-23, 24-27 and so on) then cover its 64 banks
    static_assert(WAVES % 4 == 0, "the bits of a row that its place depends on are the same for all of a lane's loads");
    const uint32_t row8 = lane >> 3, piece_x = ((lane & 7) ^ (row8 >> 1 | (wave & 1) << 2)) * 16;
    const uint32_t piece_w = WIDE ? piece_x : ((lane & 7) ^ ((row8 >> 1 & 1) | (wave & 3) << 1)) * 16;
    const int8_t* from[LOADS];
    uint32_t piece[LOADS];   // (the compiler keeps one of each kind)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const uint32_t row = (wave + i * WAVES) * 8 + row8;   // (8 rows are all of x or all of w)
        const bool of_x = (wave + i * WAVES) * 8 < BM;
        piece[i] = of_x ? piece_x : piece_w;
        if (of_x) from[i] = (const int8_t*)a.x + (uint64_t)min(tile.begin + row, tile.end - 1) * a.ld_x + first * BK + piece_x;
        else from[i] = a.w + ((uint64_t)tile.expert * a.n_out + min(n0 + row - BM, a.n_out - 1)) * a.ld_w + first * BK + piece_w;
    }
    // (pieces past the end are zeros; steps past the last are loaded too, so that the number of loads on their way is the
    // same in every step)
    const auto load = [&](uint32_t step, int i) {
        const int8_t* p = step * BK + piece[i] < n_in ? from[i] + step * BK : zeros16;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                         (__attribute__((address_space(3))) void*)(lds + step % STAGES * STAGE + (wave + i * WAVES) * 1024), 16, 0, 0);
    };
    i4 acc[4][XT] = {};
    const uint32_t key = r >> 1;
    const uint32_t at_x = (wm + r) * BK + (g ^ key) * 16, at_w = (BM + wn + channel_of(0, r >> 2, WIDE) + (r & 3)) * BK + (g ^ key) * 16;
    struct Fragments { i4 x[XT], w[4]; };   // of 64 bytes
    const auto read_w = [&](uint32_t step, int h, Fragments& f, int t) { f.w[t] = *(const i4*)(lds + step % STAGES * STAGE + (at_w ^ (h * 64)) + channel_of(t, 0, WIDE) * BK); };
    const auto read_x = [&](uint32_t step, int h, Fragments& f, int u) { f.x[u] = *(const i4*)(lds + step % STAGES * STAGE + (at_x ^ (h * 64)) + u * 16 * BK); };
    // all but the newest `left` of this wave's loads have come, its own reads of LDS too, and the same holds for every wave
    const auto meet = [&](auto left) { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(left)::value) : "memory"); };
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load(s, i);
    Fragments f[2];
    meet(std::integral_constant<int, (STAGES - 1) * LOADS>{});
#pragma unroll
    for (int t = 0; t < 4; ++t) read_w(0, 0, f[0], t);
#pragma unroll
    for (int u = 0; u < XT; ++u) read_x(0, 0, f[0], u);
    for (uint32_t step = 0; step < steps; ++step) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h == 1) meet(std::integral_constant<int, (STAGES - 2) * LOADS>{});   // this step's stage has been read, the next step's has come
            // XT pieces: four matrix instructions, a row fragment, and their share of the channel fragments and of the loads
#pragma unroll
            for (int u = 0; u < XT; ++u) {
#pragma unroll
                for (int q = u * 4 / XT; q < (u + 1) * 4 / XT; ++q) read_w(step + h, h ^ 1, f[h ^ 1], q);
                read_x(step + h, h ^ 1, f[h ^ 1], u);
                if (h == 1)
#pragma unroll
                    for (int q = u * LOADS / XT; q < (u + 1) * LOADS / XT; ++q) load(step + STAGES, q);
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[t][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[h].w[t], f[h].x[u], acc[t][u], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load may reach LDS after the workgroup has left it
    if constexpr (SPLIT) {
        i4* to = (i4*)a.partial + (uint64_t)(split * tiles + id) * (4 * XT * BN * WR) + threadIdx.x;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < XT; ++u) to[(t * XT + u) * BN * WR] = acc[t][u];
    } else finish_tile<XT, WIDE>(a, tile, tile.begin + wm, n0 + wn, g, r, acc);
}

// The sums that SPLIT left, added (exact: any order is the same) and finished; a workgroup a tile, its threads as there.
template <int BM, int BN, int WR, bool WIDE>
__global__ __launch_bounds__(BN * WR) void linear_i8_join_kernel(LinearArgs a, uint32_t col_tiles, uint32_t tiles) {
    constexpr int XT = BM / WR / 16, WC = BN / 64;
    const TilePlace at = tile_place(blockIdx.x, col_tiles, tiles);
    const RowTile tile = row_tile(a, at.row, BM == 256 ? 8 : BM == 128 ? 7 : 6);
    if (tile.begin >= tile.end) return;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    i4 acc[4][XT] = {};
#pragma unroll 4
    for (uint32_t split = 0; split < a.splits; ++split) {
        const i4* from = (const i4*)a.partial + (uint64_t)(split * tiles + blockIdx.x) * (4 * XT * BN * WR) + threadIdx.x;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < XT; ++u) acc[t][u] += from[(t * XT + u) * BN * WR];
    }
    finish_tile<XT, WIDE>(a, tile, tile.begin + wave / WC * (BM / WR), at.col * BN + wave % WC * 64, g, r, acc);
}

template <typename T>
static void linear(const LinearArgs& a, hipStream_t s) {
    linear_i8_tile_kernel<T, 128, 128><<<dim3(row_tiles(a, 7), (a.n_out + 127) / 128), 256, 0, s>>>(a);
}

template <int BM, int BN, int WR, int STAGES>
static void linear_stream(const LinearArgs& a, hipStream_t s) {
    const uint32_t cols = (a.n_out + BN - 1) / BN, tiles = row_tiles(a, BM == 256 ? 8 : BM == 128 ? 7 : 6) * cols, grid = (tiles + 7) / 8 * 8;
    if (a.y_dtype == DT_F32) linear_i8_stream_kernel<BM, BN, WR, STAGES, true><<<grid, BN * WR, 0, s>>>(a, cols, tiles);
    else linear_i8_stream_kernel<BM, BN, WR, STAGES, false><<<grid, BN * WR, 0, s>>>(a, cols, tiles);
}

static void linear_split(const LinearArgs& a, hipStream_t s) {
    const uint32_t cols = (a.n_out + 63) / 64, tiles = row_tiles(a, 6) * cols, grid = (tiles * a.splits + 7) / 8 * 8;
    if (a.y_dtype == DT_F32) {
        linear_i8_stream_kernel<64, 64, 4, 4, true, true><<<grid, 256, 0, s>>>(a, cols, tiles);
        linear_i8_join_kernel<64, 64, 4, true><<<tiles, 256, 0, s>>>(a, cols, tiles);
    } else {
        linear_i8_stream_kernel<64, 64, 4, 4, false, true><<<grid, 256, 0, s>>>(a, cols, tiles);
        linear_i8_join_kernel<64, 64, 4, false><<<tiles, 256, 0, s>>>(a, cols, tiles);
    }
}

bool linear_i8_quantizes(uint32_t rows, uint32_t n_in, uint32_t n_out, uint32_t n_experts) {
    const LinearKernel k = linear_i8_kernel(rows, n_in, n_out, n_experts);
    return k == LinearKernel::Rows || (k == LinearKernel::Few && linear_few_quantizes(rows, n_in, n_experts));
}

void launch_linear_i8(const LinearArgs& a, hipStream_t s) {
    switch (a.kernel) {
        case LinearKernel::Rows: launch_linear_rows(a, s); return;
        case LinearKernel::Few: launch_linear_few(a, s); return;
        case LinearKernel::Tile: break;
    }
    if (((uint64_t)a.x | a.ld_x | (uint64_t)a.w | a.ld_w | a.n_in) % 16 == 0) {
        if (a.splits > 1) linear_split(a, s);
        else switch (linear_i8_tile(a.rows, a.n_out, a.n_experts, a.offsets != nullptr)) {
            case LinearTile::T64: linear_stream<64, 64, 4, 4>(a, s); break;
            case LinearTile::T64x128: linear_stream<64, 128, 2, 4>(a, s); break;
            case LinearTile::T128: linear_stream<128, 128, 2, 2>(a, s); break;
            case LinearTile::T256: linear_stream<256, 256, 2, 2>(a, s); break;
        }
        return;
    }
    if (a.y_dtype == DT_F16) linear<_Float16>(a, s);
    else if (a.y_dtype == DT_BF16) linear<__bf16>(a, s);
    else linear<float>(a, s);
}

}  // namespace sng
