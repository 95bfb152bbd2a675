// linear_i8.hip -- the linear layer in 8-bit integers: rows brought to 8 bits with a scale each, times 8-bit weights with
// a scale for each output channel, on the int8 matrix instructions; dense, or by expert for rows sorted by expert.
//
//   y[r,c] = act( (sum_k q[r,k] w[c,k]) * ws[c] * s[r] + b[c] )
//
// The sum is exact (int32; n_in <= 131071), the rest is f32 and is rounded once, to y's type.
#include <algorithm>

#include "operators.h"

namespace sng {

typedef int i4 __attribute__((ext_vector_type(4)));
template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// ---- rows to 8 bits -------------------------------------------------------------------------------------------------
// q = round-half-even(127 x / a) with a = max(|x|'s largest, 2^-100), the quotient taken exactly.  v = x * fl(127 / a) is
// within 127 * 2^-23 < 2^-15 of it, so only values that close to a half need more: there 127 |x| and (m + 1/2) a are
// compared in double, where both products and their difference are exact (31, 32 bits and near one another).
__device__ __forceinline__ int quantize_one(float x, float inv, float a) {
    const float v = x * inv, f = rintf(v);
    if (fabsf(v - f) > 0.5f - 0x1p-15f) {
        const float m = floorf(fabsf(v));
        const double d = 127.0 * (double)fabsf(x) - ((double)m + 0.5) * (double)a;
        const int up = d > 0.0 ? 1 : d < 0.0 ? 0 : ((int)m & 1);
        const int q = (int)m + up;
        return x < 0.0f ? -q : q;
    }
    return (int)f;
}
// (m can also be the neighbour below when |v| rounds onto the half from above: floor is the same on both sides of m + 1/2)

__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// G threads share a row; up to C vectors a thread stay in registers between the two passes, longer rows are read again.
template <typename T, int N, int G>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
    using V = vec<T, N>;
    using Q = vec<int8_t, N>;
    constexpr int C = 4;
    __shared__ uint32_t part[4];
    const uint32_t g = threadIdx.x % G, pieces = a.cols / N;
    for (uint64_t r = blockIdx.x * (uint64_t)(256 / G) + threadIdx.x / G; r < a.rows; r += gridDim.x * (uint64_t)(256 / G)) {
        const V* __restrict__ x = (const V*)((const T*)a.x + r * a.ld_x);
        V held[C];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const uint32_t c = g + i * G;
            if (c < pieces) {
                held[i] = x[c];
#pragma unroll
                for (int q = 0; q < N; ++q) top = max(top, abs_bits((float)held[i][q]));
            }
        }
        for (uint32_t c = g + C * G; c < pieces; c += G) {
            const V v = x[c];
#pragma unroll
            for (int q = 0; q < N; ++q) top = max(top, abs_bits((float)v[q]));
        }
#pragma unroll
        for (int m = (G < 64 ? G : 64) / 2; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
        if constexpr (G == 256) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
            __syncthreads();
            top = max(max(part[0], part[1]), max(part[2], part[3]));
            __syncthreads();
        }
        const bool finite = top < 0x7f800000u;   // an infinity or NaN makes the row's scale, and so its results, NaN
        const float amax = fmaxf(__builtin_bit_cast(float, finite ? top : 0u), 0x1p-100f), inv = 127.0f / amax;
        if (g == 0) a.scale[r] = finite ? amax / 127.0f : __builtin_nanf("");
        int8_t* __restrict__ out = a.q + r * a.ld_q;
        const auto put = [&](uint32_t c, const V& v) {
            Q o;
#pragma unroll
            for (int q = 0; q < N; ++q) o[q] = (int8_t)(finite ? quantize_one((float)v[q], inv, amax) : 0);
            ((Q*)out)[c] = o;
        };
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (g + i * G < pieces) put(g + i * G, held[i]);
        for (uint32_t c = g + C * G; c < pieces; c += G) put(c, x[c]);
        for (uint32_t c = a.cols + g; c < a.cols_written; c += G) out[c] = 0;
    }
}

// 8-bit rows to the workspace's padded ones
__global__ __launch_bounds__(256) void pad_rows_kernel(QuantArgs a) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < (uint64_t)a.rows * a.cols_written; i += gridDim.x * 256ull) {
        const uint64_t r = i / a.cols_written;
        const uint32_t c = (uint32_t)(i - r * a.cols_written);
        a.q[r * a.ld_q + c] = c < a.cols ? ((const int8_t*)a.x)[r * a.ld_x + c] : 0;
    }
}

static uint32_t grid_of(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, 1u << 22); }

template <typename T, int N>
static void quantize_by_width(const QuantArgs& a, hipStream_t s) {
    const uint32_t pieces = a.cols / N;
    const auto blocks = [&](uint32_t g) { return grid_of(((uint64_t)a.rows * g + 255) / 256); };
    if (pieces <= 16) quantize_rows_kernel<T, N, 4><<<blocks(4), 256, 0, s>>>(a);
    else if (pieces <= 64) quantize_rows_kernel<T, N, 16><<<blocks(16), 256, 0, s>>>(a);
    else if (pieces <= 256) quantize_rows_kernel<T, N, 64><<<blocks(64), 256, 0, s>>>(a);
    else quantize_rows_kernel<T, N, 256><<<blocks(256), 256, 0, s>>>(a);
}

template <typename T>
static void quantize(const QuantArgs& a, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const bool wide = a.cols % N == 0 && ((uint64_t)a.x | (a.ld_x * sizeof(T))) % 16 == 0 && ((uint64_t)a.q | a.ld_q) % N == 0;
    if (wide) quantize_by_width<T, N>(a, s);
    else quantize_by_width<T, 1>(a, s);
}

void launch_quantize_rows(const QuantArgs& a, hipStream_t s) {
    if (a.dtype == DT_F16) quantize<_Float16>(a, s);
    else if (a.dtype == DT_BF16) quantize<__bf16>(a, s);
    else if (a.dtype == DT_F32) quantize<float>(a, s);
    else pad_rows_kernel<<<grid_of(((uint64_t)a.rows * a.cols_written + 255) / 256), 256, 0, s>>>(a);
}

// ---- which expert a row tile belongs to -----------------------------------------------------------------------------
// Expert e's tiles of B rows start at tile offsets[e] / B + e: that is monotonic and leaves room for
// ceil((offsets[e + 1] - offsets[e]) / B) of them, with at most one empty tile an expert (which returns at once), so no
// workgroup has to add up the experts before its own.  The 64 lanes look for the tile's expert in two steps of 64.
struct RowTile { uint32_t expert, begin, end; };   // rows [begin, end); begin >= end: nothing to do
template <uint32_t B>
__device__ __forceinline__ RowTile row_tile(const LinearArgs& a, uint32_t tile) {
    if (!a.offsets) {
        const uint32_t begin = tile * B;
        return {0, begin, min(begin + B, a.rows)};
    }
    const uint32_t lane = threadIdx.x & 63, step = (a.n_experts + 63) / 64;
    uint32_t e = lane * step;
    unsigned long long m = __ballot(e < a.n_experts && (uint32_t)a.offsets[min(e, a.n_experts)] / B + e <= tile);
    if (!m) return {0, 0, 0};
    uint32_t first = (uint32_t)(__popcll(m) - 1) * step;
    if (step > 1) {
        e = first + lane;
        m = __ballot(lane < step && e < a.n_experts && (uint32_t)a.offsets[min(e, a.n_experts)] / B + e <= tile);
        if (!m) return {0, 0, 0};
        first += (uint32_t)__popcll(m) - 1;
    }
    const uint32_t e0 = (uint32_t)a.offsets[first], end = min((uint32_t)a.offsets[first + 1], a.rows);
    const uint64_t begin = e0 + (uint64_t)(tile - (e0 / B + first)) * B;
    if (begin >= end) return {0, 0, 0};
    return {first, (uint32_t)begin, min((uint32_t)begin + B, end)};
}
static uint32_t row_tiles(const LinearArgs& a, uint32_t b) { return a.offsets ? a.rows / b + a.n_experts : (a.rows + b - 1) / b; }

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

// 16 bytes of a row from byte k on; bytes from n on are 0 (any alignment)
__device__ __forceinline__ i4 load_bytes(const int8_t* __restrict__ row, uint32_t k, uint32_t n) {
    i4 v = {0, 0, 0, 0};
    if (k + 16 <= n) __builtin_memcpy(&v, row + k, 16);
    else if (k < n) {
        uint32_t word[4] = {0, 0, 0, 0};
        for (uint32_t b = 0; b < 16; ++b)
            if (k + b < n) word[b >> 2] |= (uint32_t)(uint8_t)row[k + b] << (8 * (b & 3));
        v = i4{(int)word[0], (int)word[1], (int)word[2], (int)word[3]};
    }
    return v;
}

// ---- tiles ------------------------------------------------------------------------------------------------------------
// The matrix instruction's rows are output channels and its columns input rows, so a lane's accumulators are channels of
// one row; tile t's row 4g + i is channel 16 g + 4 t + i of the wave's 64, which makes a lane's 16 values one piece of y.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void linear_i8_tile_kernel(LinearArgs a) {
    constexpr int BK = 128, XT = BM / 32, CHUNKS = (BM + BN) * 8 / 256;
    static_assert(BN == 128, "two waves of 64 channels");
    __shared__ __align__(16) int8_t lds[(BM + BN) * BK];
    const RowTile tile = row_tile<BM>(a, blockIdx.x);
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
    i4 next[CHUNKS];
    const auto load = [&](uint32_t k0) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t c = threadIdx.x + i * 256, row = c >> 3, k = k0 + (c & 7) * 16;
            if (row < BM) next[i] = tile.begin + row < tile.end ? load_bytes(a.x + (uint64_t)(tile.begin + row) * a.ld_x, k, a.n_in) : i4{0, 0, 0, 0};
            else next[i] = n0 + row - BM < a.n_out ? load_bytes(w + (uint64_t)(n0 + row - BM) * a.ld_w, k, a.n_in) : i4{0, 0, 0, 0};
        }
    };
    load(0);
    for (uint32_t k0 = 0; k0 < a.n_in; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t c = threadIdx.x + i * 256, row = c >> 3, piece = c & 7;
            *(i4*)(lds + row * BK + ((piece ^ (row < BM ? keyx(row) : key(row - BM))) * 16)) = next[i];
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
            v[q] = (float)acc[q >> 2][u][q & 3] * ws[q] * s + b[q];   // (the row's scale last: it has the type's whole range)
            if (a.relu) v[q] = v[q] < 0.0f ? 0.0f : v[q];   // (keeps NaN)
        }
        store_channels<T, 16>((T*)a.y + (uint64_t)row * a.ld_y + c0, v, left, aligned);
    }
}

template <typename T>
static void linear(const LinearArgs& a, hipStream_t s) {
    linear_i8_tile_kernel<T, 128, 128><<<dim3(row_tiles(a, 128), (a.n_out + 127) / 128), 256, 0, s>>>(a);
}

void launch_linear_i8(const LinearArgs& a, hipStream_t s) {
    if (a.y_dtype == DT_F16) linear<_Float16>(a, s);
    else if (a.y_dtype == DT_BF16) linear<__bf16>(a, s);
    else linear<float>(a, s);
}

}  // namespace sng
