// linear_i8.hip -- the linear layer in 8-bit integers: rows brought to 8 bits with a scale each, times 8-bit weights with
// a scale for each output channel, on the int8 matrix instructions; dense, or by expert for rows sorted by expert.
//
//   y[r,c] = act( (sum_k q[r,k] w[c,k]) * ws[c] * s[r] + b[c] )
//
// The sum is exact (int32; n_in <= 131071), the rest is f32 and is rounded once, to y's type.
#include <algorithm>
#include <type_traits>

#include "operators.h"

namespace sng {

typedef int i4 __attribute__((ext_vector_type(4)));
template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// ---- rows to 8 bits -------------------------------------------------------------------------------------------------
// q = round-half-even(127 x / a) with a = max(|x|'s largest, 2^-100), the quotient taken exactly.  With inv = fl(127 / a)
// the product x * inv is within 127 * 2^-24 of it, so adding it to 1.5 * 2^23 in one fused operation rounds it rightly
// (q is then the sum's low byte) unless it lies within 2^-15 of a half.  Only those values need more: 127 |x| and
// (m + 1/2) a are compared in double, where both products and their difference are exact.
constexpr float ROUNDER = 12582912.0f;
__device__ __forceinline__ float quantize_fast(float x, float inv, float& near) {   // near: the largest distance from a whole number
    const float t = fmaf(x, inv, ROUNDER);
    near = fmaxf(near, fabsf(fmaf(x, inv, ROUNDER - t)));
    return t;
}
constexpr float NEAR_HALF = 0.5f - 0x1p-15f;
__device__ __noinline__ int quantize_half(float x, float inv, float a) {
    const float m = floorf(fabsf(x) * inv);   // the same whole number on both sides of m + 1/2
    const double d = 127.0 * (double)fabsf(x) - ((double)m + 0.5) * (double)a;
    const int q = (int)m + (d > 0.0 ? 1 : d < 0.0 ? 0 : ((int)m & 1));
    return x < 0.0f ? -q : q;
}
__device__ __forceinline__ int quantize_one(float x, float inv, float a) {
    float near = 0.0f;
    const float t = quantize_fast(x, inv, near);
    return near > NEAR_HALF ? quantize_half(x, inv, a) : (int)(int8_t)__builtin_bit_cast(uint32_t, t);
}
// 16 values to 16 bytes
__device__ __forceinline__ i4 quantize_16(const float (&x)[16], float inv, float a) {
    float near = 0.0f, t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = quantize_fast(x[i], inv, near);
    uint32_t b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = __builtin_bit_cast(uint32_t, t[i]);
    if (near > NEAR_HALF)
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = (uint32_t)quantize_one(x[i], inv, a);
    i4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x0c0c0400u);
        q[i] = (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
    return q;
}

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
__device__ __forceinline__ RowTile row_tile(const LinearArgs& a, uint32_t tile, uint32_t shift) {   // B = 1 << shift
    if (!a.offsets) {
        const uint32_t begin = tile << shift;
        return {0, begin, min(begin + (1u << shift), a.rows)};
    }
    const uint32_t lane = threadIdx.x & 63, step = (a.n_experts + 63) / 64;
    uint32_t e = lane * step;
    unsigned long long m = __ballot(e < a.n_experts && ((uint32_t)a.offsets[min(e, a.n_experts)] >> shift) + e <= tile);
    if (!m) return {0, 0, 0};
    uint32_t first = (uint32_t)(__popcll(m) - 1) * step;
    if (step > 1) {
        e = first + lane;
        m = __ballot(lane < step && e < a.n_experts && ((uint32_t)a.offsets[min(e, a.n_experts)] >> shift) + e <= tile);
        if (!m) return {0, 0, 0};
        first += (uint32_t)__popcll(m) - 1;
    }
    first = __builtin_amdgcn_readfirstlane(first);
    const uint32_t e0 = (uint32_t)a.offsets[first], end = min((uint32_t)a.offsets[first + 1], a.rows);
    const uint64_t begin = e0 + ((uint64_t)(tile - ((e0 >> shift) + first)) << shift);
    if (begin >= end) return {0, 0, 0};
    return {first, (uint32_t)begin, min((uint32_t)begin + (1u << shift), end)};
}
static uint32_t row_tiles(const LinearArgs& a, uint32_t shift) {
    return a.offsets ? (a.rows >> shift) + a.n_experts : (uint32_t)(((uint64_t)a.rows + (1u << shift) - 1) >> shift);
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

// ---- short rows -------------------------------------------------------------------------------------------------------
// n_in <= 256: a row is at most 4 fragments of 64 bytes, so a wave loads 16 rows, finds their scales, brings them to 8 bits
// and multiplies them without leaving its registers: x is read once and y written once, the floor of a layer this small.
// A lane holds the 16 consecutive values of one row that the matrix instruction wants of it; the four lanes of a row share
// their maximum with two shuffles.  The weights of up to 256 channels lie in LDS in fragment order (one linear
// ds_read_b128 a fragment, no bank conflicts), staged once for the workgroup's rows, which belong to one expert.
template <int XB>
struct RawRow { i4 v[XB]; };   // 16 elements of XB bytes

template <int XB>
__device__ __forceinline__ RawRow<XB> load_row16(const char* __restrict__ row, uint32_t k, uint32_t n) {
    RawRow<XB> r;
#pragma unroll
    for (int i = 0; i < XB; ++i) r.v[i] = i4{0, 0, 0, 0};
    if (k + 16 <= n) __builtin_memcpy(&r, row + (uint64_t)k * XB, 16 * XB);
    else
#pragma unroll
        for (int i = 0; i < 16; ++i)   // (static places only: the words have to stay in registers)
            if (k + i < n) {
                uint32_t e = 0;
                __builtin_memcpy(&e, row + (uint64_t)(k + i) * XB, XB);
                r.v[i * XB / 16][(i * XB / 4) & 3] |= (int)(e << (8 * ((i * XB) & 3)));
            }
    return r;
}

// the largest |x| of 16 values as f32 bits (those of an infinity or NaN are the largest)
template <int XB>
__device__ __forceinline__ uint32_t top_bits(const RawRow<XB>& r, int dtype) {
    uint32_t top = 0;
    if constexpr (XB == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, (uint32_t)r.v[i >> 2][i & 3] & 0x7fffffffu);
    } else if constexpr (XB == 2) {
        using u2 = uint16_t __attribute__((ext_vector_type(2)));
        u2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u2, (uint32_t)r.v[i >> 2][i & 3] & 0x7fff7fffu));
        const uint16_t h = max(m[0], m[1]);
        top = dtype == DT_BF16 ? (uint32_t)h << 16 : __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, h)) & 0x7fffffffu;
    }
    return top;
}
template <int XB>
__device__ __forceinline__ void to_floats(const RawRow<XB>& r, int dtype, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if constexpr (XB == 4) x[i] = __builtin_bit_cast(float, (uint32_t)r.v[i >> 2][i & 3]);
        else {
            const uint32_t w = (uint32_t)r.v[i >> 3][(i >> 1) & 3], h = (i & 1) ? w >> 16 : w & 0xffffu;
            x[i] = dtype == DT_BF16 ? __builtin_bit_cast(float, h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
        }
    }
}

struct RowScale { float scale, inv, amax; bool finite; };
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
    RowScale r;
    r.finite = top < 0x7f800000u;   // an infinity or NaN makes the row's scale, and so its results, NaN
    r.amax = fmaxf(__builtin_bit_cast(float, r.finite ? top : 0u), 0x1p-100f);
    r.inv = 127.0f / r.amax;
    r.scale = r.finite ? r.amax / 127.0f : __builtin_nanf("");
    return r;
}

// Which of a wave's 64 channels a lane's accumulator (t, i) is: a lane's 16-byte piece of y is next to those of the other
// three lanes of its row, so a store writes 64 consecutive bytes a row: 8 channels of f16 (two accumulators), 4 of f32.
__device__ __forceinline__ uint32_t channel_of(int t, uint32_t g, bool wide) { return wide ? t * 16 + g * 4 : (t >> 1) * 32 + g * 8 + (t & 1) * 4; }

// 16 bytes of y: 4 f32 or 8 16-bit channels of a row from channel c on, `left` of them inside
template <int N>
__device__ __forceinline__ void store_piece(const LinearArgs& a, uint32_t row, uint32_t c, const float (&v)[N], uint32_t left, bool aligned) {
    const uint64_t at = (uint64_t)row * a.ld_y + c;
    if constexpr (N == 4) {
        float* y = (float*)a.y + at;
        if (aligned && left >= 4) *(vec<float, 4>*)y = vec<float, 4>{v[0], v[1], v[2], v[3]};
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if ((uint32_t)i < left) y[i] = v[i];
    } else {
        uint16_t* y = (uint16_t*)a.y + at;
        vec<uint16_t, 8> o;
        if (a.y_dtype == DT_F16)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __builtin_bit_cast(uint16_t, (_Float16)v[i]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __builtin_bit_cast(uint16_t, (__bf16)v[i]);
        if (aligned && left >= 8) *(vec<uint16_t, 8>*)y = o;
        else
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((uint32_t)i < left) y[i] = o[i];
    }
}
// One row's 16 channels of a 64-channel block (v[4 t + i], channels as channel_of says), `left` channels from the block's first on
__device__ __forceinline__ void store_block(const LinearArgs& a, uint32_t row, uint32_t c0, uint32_t g, const float (&v)[16], uint32_t left, bool aligned) {
    if (a.y_dtype == DT_F32) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t c = channel_of(t, g, true);
            store_piece(a, row, c0 + c, {v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]}, left - min(left, c), aligned);
        }
    } else
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const uint32_t c = channel_of(2 * p, g, false);
            store_piece(a, row, c0 + c, {v[8 * p], v[8 * p + 1], v[8 * p + 2], v[8 * p + 3], v[8 * p + 4], v[8 * p + 5], v[8 * p + 6], v[8 * p + 7]}, left - min(left, c), aligned);
        }
}
__device__ __forceinline__ bool y_aligned(const LinearArgs& a) { return (((uint64_t)a.y | (a.ld_y * (a.y_dtype == DT_F32 ? 4 : 2))) & 15) == 0; }

// XB bytes an element of x; KC fragments of 64 a row; NB blocks of 64 channels
template <int XB, int KC, int NB>
__global__ __launch_bounds__(256) void linear_i8_rows_kernel(LinearArgs a, uint32_t shift) {
    constexpr int U = KC == 1 ? 2 : 1;   // groups of 16 rows in flight a wave
    __shared__ i4 lw[NB * 4 * KC * 64];
    __shared__ __align__(16) float lscale[NB * 64], lbias[NB * 64];
    const RowTile tile = row_tile(a, blockIdx.x, shift);
    if (tile.begin >= tile.end) return;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n0 = blockIdx.y * (NB * 64);
    const bool wide = a.y_dtype == DT_F32, aligned = y_aligned(a);
    const int8_t* __restrict__ w = (const int8_t*)a.w + (uint64_t)tile.expert * a.n_out * a.ld_w;
#pragma unroll
    for (int i = 0; i < NB * KC; ++i) {
        const uint32_t f = i * 256 + threadIdx.x, l = f & 63, kc = (f >> 6) % KC, t = (f >> 6) / KC & 3, nb = (f >> 6) / (4 * KC);
        const uint32_t c = n0 + nb * 64 + channel_of(t, (l >> 2) & 3, wide) + (l & 3);
        lw[f] = c < a.n_out ? load_bytes(w + (uint64_t)c * a.ld_w, kc * 64 + (l >> 4) * 16, a.n_in) : i4{0, 0, 0, 0};
    }
    if (threadIdx.x < NB * 64) {
        const uint32_t c = n0 + threadIdx.x;
        const uint64_t at = (uint64_t)tile.expert * a.n_out + c;
        lscale[threadIdx.x] = c < a.n_out ? a.w_scale[at] : 0.0f;
        lbias[threadIdx.x] = c < a.n_out && a.bias ? a.bias[at] : 0.0f;
    }
    __syncthreads();
    for (uint32_t r0 = tile.begin + wave * (16 * U); r0 < tile.end; r0 += 64 * U) {
        RawRow<XB> raw[U][KC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t row = r0 + u * 16 + (lane & 15);
#pragma unroll
            for (int kc = 0; kc < KC; ++kc)
                raw[u][kc] = load_row16<XB>((const char*)a.x + (uint64_t)min(row, tile.end - 1) * a.ld_x * XB, kc * 64 + g * 16, a.n_in);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t row = r0 + u * 16 + (lane & 15);
            i4 q[KC];
            float scale;
            if constexpr (XB == 1) {
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) q[kc] = raw[u][kc].v[0];
                scale = a.x_scale[min(row, tile.end - 1)];
            } else {
                uint32_t top = 0;
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) top = max(top, top_bits<XB>(raw[u][kc], a.x_dtype));
                top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
                top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
                const RowScale rs = row_scale(top);
                scale = rs.scale;
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    float x[16];
                    to_floats<XB>(raw[u][kc], a.x_dtype, x);
                    q[kc] = quantize_16(x, rs.inv, rs.amax);
                    if (!rs.finite) q[kc] = i4{0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                if (n0 + nb * 64 >= a.n_out) break;
                float v[16];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    i4 acc = {0, 0, 0, 0};
#pragma unroll
                    for (int kc = 0; kc < KC; ++kc) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(lw[((nb * 4 + t) * KC + kc) * 64 + lane], q[kc], acc, 0, 0, 0);
                    const uint32_t c = nb * 64 + channel_of(t, g, wide);
                    const vec<float, 4> ws = *(const vec<float, 4>*)(lscale + c), b = *(const vec<float, 4>*)(lbias + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float y = (float)acc[i] * ws[i] * scale + b[i];   // (the row's scale last: it has the type's whole range)
                        v[4 * t + i] = a.relu && y < 0.0f ? 0.0f : y;           // (keeps NaN)
                    }
                }
                if (row < tile.end) store_block(a, row, n0 + nb * 64, g, v, a.n_out - (n0 + nb * 64), aligned);
            }
        }
    }
}

template <int XB, int KC>
static void linear_rows(const LinearArgs& a, hipStream_t s) {
    // Rows a workgroup: few where there are few, so that the chip is filled; up to 512, where staging the weights is small
    // beside the rows.
    uint32_t shift = 6;
    while (shift < 9 && (a.rows >> shift) > 2048) ++shift;
    const uint32_t nb = a.n_out <= 64 ? 1 : a.n_out <= 128 ? 2 : 4;
    const dim3 grid(row_tiles(a, shift), (a.n_out + nb * 64 - 1) / (nb * 64));
    if (nb == 1) linear_i8_rows_kernel<XB, KC, 1><<<grid, 256, 0, s>>>(a, shift);
    else if (nb == 2) linear_i8_rows_kernel<XB, KC, 2><<<grid, 256, 0, s>>>(a, shift);
    else linear_i8_rows_kernel<XB, KC, 4><<<grid, 256, 0, s>>>(a, shift);
}
template <int XB>
static void linear_rows_by_length(const LinearArgs& a, hipStream_t s) {
    if (a.n_in <= 64) linear_rows<XB, 1>(a, s);
    else if (a.n_in <= 128) linear_rows<XB, 2>(a, s);
    else linear_rows<XB, 4>(a, s);
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// Bound by reading the weights once.  A workgroup takes 16 channels of one matrix and splits n_in over its NW waves, so
// that a whole chip of waves is loading also for one row; each wave's sums meet in LDS.  x (up to 16 rows at a time) is
// brought to 8 bits on the way: every wave reads its own part of the rows, the waves share the rows' maxima in LDS, and
// the first weights are on their way meanwhile.
template <int XB, int NW>
__global__ __launch_bounds__(NW * 64) void linear_i8_few_kernel(LinearArgs a) {
    constexpr int H = 4;   // fragments of 64 bytes of the weights in flight
    __shared__ uint32_t tops[NW][16];
    __shared__ i4 sums[NW][64];
    const uint32_t expert = blockIdx.y;
    uint32_t begin = 0, end = a.rows;
    if (a.offsets) {
        begin = (uint32_t)a.offsets[expert];
        end = min((uint32_t)a.offsets[expert + 1], a.rows);
        if (begin >= end) return;
    }
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const uint32_t n0 = blockIdx.x * 16, steps = (a.n_in + 63) / 64, per = (steps + NW - 1) / NW;
    const uint32_t s0 = min(steps, wave * per), s1 = min(steps, s0 + per);
    const int8_t* __restrict__ w = (const int8_t*)a.w + ((uint64_t)expert * a.n_out + min(n0 + r, a.n_out - 1)) * a.ld_w;
    for (uint32_t row0 = begin; row0 < end; row0 += 16) {
        const uint32_t row = row0 + r;
        const bool on = row < end;
        const char* __restrict__ x = (const char*)a.x + (uint64_t)(on ? row : row0) * a.ld_x * XB;
        i4 fw[H];
#pragma unroll
        for (int h = 0; h < H; ++h) fw[h] = s0 + h < s1 ? load_bytes(w, (s0 + h) * 64 + g * 16, a.n_in) : i4{0, 0, 0, 0};
        RowScale rs = {};
        if constexpr (XB > 1) {
            uint32_t top = 0;
            if (on)
#pragma unroll 4
                for (uint32_t s = s0; s < s1; ++s) top = max(top, top_bits<XB>(load_row16<XB>(x, s * 64 + g * 16, a.n_in), a.x_dtype));
            top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            if (g == 0) tops[wave][r] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NW; ++i) top = max(top, tops[i][r]);
            rs = row_scale(top);
        }
        i4 acc = {0, 0, 0, 0};
        for (uint32_t s = s0; s < s1; s += H) {
            i4 q[H];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                q[h] = i4{0, 0, 0, 0};
                if (on && s + h < s1) {
                    const RawRow<XB> raw = load_row16<XB>(x, (s + h) * 64 + g * 16, a.n_in);
                    if constexpr (XB == 1) q[h] = raw.v[0];
                    else if (rs.finite) {
                        float f[16];
                        to_floats<XB>(raw, a.x_dtype, f);
                        q[h] = quantize_16(f, rs.inv, rs.amax);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < H; ++h) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[h], q[h], acc, 0, 0, 0);
            if (s + H < s1)
#pragma unroll
                for (int h = 0; h < H; ++h) fw[h] = s + H + h < s1 ? load_bytes(w, (s + H + h) * 64 + g * 16, a.n_in) : i4{0, 0, 0, 0};
        }
        sums[wave][lane] = acc;
        __syncthreads();
        // 256 results, one a thread: row tid & 15, channel tid >> 4 (lane 16 (c / 4) + row held sum c % 4)
        for (uint32_t i = threadIdx.x; i < 256; i += NW * 64) {
            const uint32_t rr = i >> 4, c = i & 15;
            int sum = 0;
#pragma unroll
            for (int k = 0; k < NW; ++k) sum += ((const int*)&sums[k][(c >> 2) * 16 + rr])[c & 3];
            if (row0 + rr < end && n0 + c < a.n_out) {
                float scale;
                if constexpr (XB == 1) scale = a.x_scale[row0 + rr];
                else {
                    uint32_t top = 0;
#pragma unroll
                    for (int k = 0; k < NW; ++k) top = max(top, tops[k][rr]);
                    scale = row_scale(top).scale;
                }
                const uint64_t at = (uint64_t)expert * a.n_out + n0 + c;
                const float y = (float)sum * a.w_scale[at] * scale + (a.bias ? a.bias[at] : 0.0f), v = a.relu && y < 0.0f ? 0.0f : y;
                const uint64_t to = (uint64_t)(row0 + rr) * a.ld_y + n0 + c;
                if (a.y_dtype == DT_F16) ((_Float16*)a.y)[to] = (_Float16)v;
                else if (a.y_dtype == DT_BF16) ((__bf16*)a.y)[to] = (__bf16)v;
                else ((float*)a.y)[to] = v;
            }
        }
        __syncthreads();
    }
}

template <int XB>
static void linear_few(const LinearArgs& a, hipStream_t s) {
    const dim3 grid((a.n_out + 15) / 16, a.offsets ? a.n_experts : 1);
    if (a.n_in <= 1024) linear_i8_few_kernel<XB, 4><<<grid, 256, 0, s>>>(a);
    else linear_i8_few_kernel<XB, 8><<<grid, 512, 0, s>>>(a);
}

// ---- tiles ------------------------------------------------------------------------------------------------------------
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
    i4 next[CHUNKS];
    const auto load = [&](uint32_t k0) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t c = threadIdx.x + i * 256, row = c >> 3, k = k0 + (c & 7) * 16;
            if (row < BM) next[i] = tile.begin + row < tile.end ? load_bytes((const int8_t*)a.x + (uint64_t)(tile.begin + row) * a.ld_x, k, a.n_in) : i4{0, 0, 0, 0};
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

// The same product with both tiles brought straight into LDS (global_load_lds, 16 bytes a lane): no registers and no
// instructions stand between memory and the matrix units.  Steps of 128 bytes of n_in (whole cache lines), a stage of LDS
// each, in halves: while one half is multiplied from registers the next is read from LDS.  Once a step's second half is in
// registers its stage is free: the one barrier of the step, behind which the loads of STAGES steps ahead refill it.  Loads and
// reads are spread between the matrix instructions: behind the barrier every wave would else queue its loads first and
// the matrix units would wait for the queue.  A lane fetches the piece of its row that belongs at its place in LDS, which
// keeps the lanes of a fragment read on different banks.
// Wants n_in, both strides and both addresses in multiples of 16 bytes.
__device__ const int8_t zeros16[16] __attribute__((aligned(16))) = {};

// A wave holds BM / WR rows by 64 channels.
template <int BM, int BN, int WR, int STAGES, bool WIDE>
__global__ __launch_bounds__(BN * WR) void linear_i8_stream_kernel(LinearArgs a, uint32_t col_tiles, uint32_t tiles) {
    constexpr int WC = BN / 64, WAVES = WR * WC, XT = BM / WR / 16, BK = 128, STAGE = (BM + BN) * BK;
    constexpr int LOADS = (BM + BN) / 8 / WAVES;   // each brings 8 rows of 128 bytes
    __shared__ __align__(16) int8_t lds[STAGES * STAGE];
    // workgroups go round the 8 dies one by one: each die gets a run of neighbouring tiles, in columns of 4 row tiles, so
    // that its cache sees the same rows and channels again
    const uint32_t per = (tiles + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= tiles) return;
    const uint32_t row_tiles = tiles / col_tiles, group = id / (4 * col_tiles), in = id - group * 4 * col_tiles, high = min(4u, row_tiles - group * 4);
    const RowTile tile = row_tile(a, group * 4 + in % high, BM == 256 ? 8 : BM == 128 ? 7 : 6);
    if (tile.begin >= tile.end) return;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15, n0 = in / high * BN;
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
        if (of_x) from[i] = (const int8_t*)a.x + (uint64_t)min(tile.begin + row, tile.end - 1) * a.ld_x + piece_x;
        else from[i] = a.w + ((uint64_t)tile.expert * a.n_out + min(n0 + row - BM, a.n_out - 1)) * a.ld_w + piece_w;
    }
    // (pieces past the end are zeros; steps past the last are loaded too, so that the number of loads on their way is the
    // same in every step)
    const auto load = [&](uint32_t step, int i) {
        const int8_t* p = step * BK + piece[i] < a.n_in ? from[i] + step * BK : zeros16;
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
    const uint32_t steps = (a.n_in + BK - 1) / BK;
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
    const uint32_t c0 = n0 + wn;
    if (c0 >= a.n_out) return;
    const bool aligned = y_aligned(a);
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
        const uint32_t row = tile.begin + wm + u * 16 + r;
        if (row >= tile.end) continue;
        const float s = a.x_scale[row];
        float v[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const float y = (float)acc[q >> 2][u][q & 3] * ws[q] * s + b[q];
            v[q] = a.relu && y < 0.0f ? 0.0f : y;
        }
        store_block(a, row, c0, g, v, a.n_out - c0, aligned);
    }
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

LinearKernel linear_i8_kernel(uint32_t rows, uint32_t n_in, uint32_t n_out, uint32_t n_experts) {
    if (n_in <= 256) return LinearKernel::Rows;
    if (rows <= 16u * n_experts) return LinearKernel::Few;
    return LinearKernel::Tile;
}
bool linear_i8_quantizes(LinearKernel k, uint32_t rows, uint32_t n_experts) { return k != LinearKernel::Tile; }

void launch_linear_i8(const LinearArgs& a, hipStream_t s) {
    const int xb = a.x_dtype == DT_I8 ? 1 : a.x_dtype == DT_F32 ? 4 : 2;
    switch (linear_i8_kernel(a.rows, a.n_in, a.n_out, a.n_experts)) {
        case LinearKernel::Rows:
            if (xb == 1) linear_rows_by_length<1>(a, s);
            else if (xb == 2) linear_rows_by_length<2>(a, s);
            else linear_rows_by_length<4>(a, s);
            return;
        case LinearKernel::Few:
            if (xb == 1) linear_few<1>(a, s);
            else if (xb == 2) linear_few<2>(a, s);
            else linear_few<4>(a, s);
            return;
        case LinearKernel::Tile: break;
    }
    if (((uint64_t)a.x | a.ld_x | (uint64_t)a.w | a.ld_w | a.n_in) % 16 == 0) {
        // the largest tile that still gives most of the 256 CUs one: 256 x 256 reads each operand least often
        const uint64_t cells = (uint64_t)a.rows * a.n_out;
        if (cells >= 192ull * 256 * 256) linear_stream<256, 256, 2, 2>(a, s);
        else if (cells >= 192ull * 128 * 128) linear_stream<128, 128, 2, 2>(a, s);
        else linear_stream<64, 128, 2, 4>(a, s);
        return;
    }
    if (a.y_dtype == DT_F16) linear<_Float16>(a, s);
    else if (a.y_dtype == DT_BF16) linear<__bf16>(a, s);
    else linear<float>(a, s);
}

}  // namespace sng
