// linear_i8.h -- what the kernels of the 8-bit linear layer share: rows brought to 8 bits, fragment loads, row tiles by expert,
// results.  linear_i8.hip describes the layer.
#pragma once
#include <algorithm>
#include <type_traits>

#include "operators.h"

namespace sng {

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));
using i4 = vec<int, 4>;

// ---- rows to 8 bits -------------------------------------------------------------------------------------------------
// q = round-half-even(127 x / a) with a = max(|x|'s largest, 2^-100), the quotient taken exactly.  inv is 127 / a, or within
// 2^-22 of it from above; one fused operation adds x * inv to 1.5 * 2^23 and rounds once, and q is the sum's low byte.  Where
// that can differ from the exact quotient's rounding:
//   * x with 11 or fewer significant bits (f16, bf16): x = mx 2^s, a = ma 2^t with whole mx, ma < 2^11, so 127 x / a that is
//     not a half itself is at least 1/254 2^-11 of its value away from one, much more than inv's error.  A half means
//     254 mx = (odd <= 255) ma 2^n, so 127 divides either the odd number, then it is 127, the quotient 63.5, and rounding up
//     is right; or ma, then an inexact inv rounds halves up that belong to the even number below.  Only rows with such an a
//     (7 of 1024 in f16) take the careful way.
//   * f32: any value within 2^-14 of a half takes the careful way.
// The careful way takes the sign of 127 |x| - (m + 1/2) a, each product as a rounded value and its exact remainder (one
// fused operation each).  The two products are within 2^-13 of one another, so their difference is exact, and the
// remainders decide only where it is no larger than they are.  (Both sides taken 2^-8 times: neither product overflows,
// and with a >= 2^-100 no remainder is below f32's range.)
constexpr float ROUNDER = 12582912.0f;
constexpr float NEAR_HALF = 0.5f - 0x1p-14f;

struct RowScale {
    float scale, inv, a;
    bool finite, careful;
};
// a / 127 rounded once: the reciprocal's product corrected by its remainder (every mantissa checked against the division)
__device__ __forceinline__ float scale_of(uint32_t top) {
    const float a = fmaxf(__builtin_bit_cast(float, top), 0x1p-100f), r = 1.0f / 127.0f, q = a * r;
    return top < 0x7f800000u ? fmaf(fmaf(-127.0f, q, a), r, q) : __builtin_nanf("");   // an infinity or NaN makes the row's results NaN
}
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
    RowScale r;
    r.finite = top < 0x7f800000u;
    r.scale = scale_of(top);
    r.a = fmaxf(__builtin_bit_cast(float, r.finite ? top : 0u), 0x1p-100f);
    const float as = r.a * 0x1p-16f, rcp = __builtin_amdgcn_rcpf(as), rough = 127.0f * rcp;   // (scaled: the reciprocal of a large a is no normal number)
    float inv = fmaf(fmaf(-rough, as, 127.0f), rcp, rough);
    float over = fmaf(inv, as, -127.0f);
    if (over < 0.0f) {
        inv = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, inv) + 1u);
        over = 1.0f;
    }
    r.inv = inv * 0x1p-16f;
    const uint32_t mantissa = (__builtin_bit_cast(uint32_t, r.a) & 0x7fffffu) | 0x800000u;
    r.careful = over != 0.0f && mantissa * 0xefdfbf7fu <= 0xffffffffu / 127u;   // 127 divides it (times the inverse of 127 mod 2^32)
    return r;
}

__device__ __forceinline__ uint32_t quantize_careful(float x, float inv, float a) {
    const float v = x * inv, f = rintf(v), m = floorf(fabsf(v)), h = m + 0.5f;   // m: the same whole number on both sides of m + 1/2
    const float xs = fabsf(x) * 0x1p-8f, as = a * 0x1p-8f, p = 127.0f * xs, q = h * as;
    const float d = (p - q) + (fmaf(127.0f, xs, -p) - fmaf(h, as, -q));
    const int up = (int)m + (d > 0.0f ? 1 : d < 0.0f ? 0 : ((int)m & 1));
    return (uint32_t)(fabsf(v - f) > NEAR_HALF ? (x < 0.0f ? -up : up) : (int)f);
}

// N elements as they lie in memory
constexpr int bytes_of(int dtype) { return dtype == DT_F32 ? 4 : dtype == DT_I8 ? 1 : 2; }
template <int DT, int N>
struct Raw { uint32_t w[N * bytes_of(DT) / 4]; };
// the largest |x| as f32 bits (those of an infinity or NaN are the largest)
template <int DT, int N>
__device__ __forceinline__ uint32_t top_bits(const Raw<DT, N>& r) {
    uint32_t top = 0;
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int i = 0; i < N; ++i) top = max(top, r.w[i] & 0x7fffffffu);
    } else if constexpr (DT != DT_I8) {
        using u2 = vec<uint16_t, 2>;
        u2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < N / 2; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u2, r.w[i] & 0x7fff7fffu));
        const uint16_t h = max(m[0], m[1]);
        top = DT == DT_BF16 ? (uint32_t)h << 16 : __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, h)) & 0x7fffffffu;
    }
    return top;
}
template <int DT, int N>
__device__ __forceinline__ float element(const Raw<DT, N>& r, int i) {
    if constexpr (DT == DT_F32) return __builtin_bit_cast(float, r.w[i]);
    const uint32_t h = (i & 1) ? r.w[i >> 1] >> 16 : r.w[i >> 1] & 0xffffu;
    return DT == DT_BF16 ? __builtin_bit_cast(float, h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// N values of a row to N bytes (a row that is not finite: anything; a product's NaN scale hides it, where q itself is the
// result the caller puts zeros)
template <int DT, int N>
__device__ __forceinline__ vec<int, N / 4> quantize_n(const Raw<DT, N>& r, const RowScale& rs) {
    float near = 0.0f;
    uint32_t b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float x = element(r, i), t = fmaf(x, rs.inv, ROUNDER);
        if constexpr (DT == DT_F32) near = fmaxf(near, fabsf(fmaf(x, rs.inv, ROUNDER - t)));
        b[i] = __builtin_bit_cast(uint32_t, t);
    }
    if (__any(DT == DT_F32 ? near > NEAR_HALF : rs.careful)) {
        asm volatile("");   // (else the compiler takes the branch away and computes both ways for every value: 64 -> 64 layer 92 us for 60)
#pragma unroll
        for (int i = 0; i < N; ++i) b[i] = quantize_careful(element(r, i), rs.inv, rs.a);
    }
    vec<int, N / 4> q;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x0c0c0400u);
        q[i] = (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
    return q;
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

// 16 elements of a row of n >= 16 from element k on (a multiple of 16), at any alignment and without reading behind the
// row: the row's last 16 are read where fewer are left.  Some of those belong to the 16 before, which does no harm to a
// maximum, and none to a product if new_bytes() clears them in one of its two factors: nothing has to be moved.  Where the
// row is kept, inside() moves them to their places.  Loads and what corrects them are apart, so that all of a thread's loads
// are on their way before it waits for the first.
template <int DT>
__device__ __forceinline__ Raw<DT, 16> load_row16(const char* __restrict__ row, uint32_t k, uint32_t n) {
    Raw<DT, 16> r;
    __builtin_memcpy(&r, row + (uint64_t)min(k, n - 16) * bytes_of(DT), sizeof(r));
    return r;
}
// The same for bytes at odd places: whole words that hold them (4 and the one of the last byte, none without a byte of the
// 16), shifted together when they are wanted.  A 16-byte load that is not aligned to words takes several times as
// long (a row times 4097 -> 4096: 15.2 us, 9.5 this way, 6.8 for 4096; 1025 -> 2048: 6.7 and 4.8).
struct OddBytes { uint32_t w[5], shift; };
__device__ __forceinline__ OddBytes load_odd16(const char* __restrict__ row, uint32_t k, uint32_t n) {
    const char* p = row + min(k, n - 16);
    OddBytes r;
    __builtin_memcpy(r.w, __builtin_assume_aligned((const char*)((uint64_t)p & ~3ull), 4), 16);
    __builtin_memcpy(r.w + 4, __builtin_assume_aligned((const char*)((uint64_t)(p + 15) & ~3ull), 4), 4);
    r.shift = ((uint32_t)(uint64_t)p & 3) * 8;
    return r;
}
__device__ __forceinline__ Raw<DT_I8, 16> whole(const OddBytes& o) {
    Raw<DT_I8, 16> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __builtin_amdgcn_alignbit(o.w[i + 1], o.w[i], o.shift);
    return r;
}
__device__ __forceinline__ Raw<DT_I8, 16> whole(const Raw<DT_I8, 16>& r) { return r; }
__device__ __forceinline__ i4 new_bytes(i4 v, uint32_t k, uint32_t n) {
    const int had = (int)min(max(k + 16, n) - n, 16u);   // of the 16
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = had >= 4 * i + 4 ? 0 : v[i] & (int)(0xffffffffu << (max(had - 4 * i, 0) * 8));
    return v;
}
template <int DT>
__device__ __forceinline__ Raw<DT, 16> inside(Raw<DT, 16> r, uint32_t k, uint32_t n) {
    constexpr int XB = bytes_of(DT), W = 4 * XB;
    const uint32_t move = (k - min(k, n - 16)) * XB;   // bytes; 16 elements and more: nothing is left
#pragma unroll
    for (int by = W / 2; by > 0; by >>= 1)
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = move & (by * 4) ? (i + by < W ? r.w[i + by] : 0u) : r.w[i];
    if constexpr (XB < 4)
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = __builtin_amdgcn_alignbit(i + 1 < W ? r.w[i + 1] : 0u, r.w[i], (move & 3) * 8);
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = move >= 16 * XB ? 0u : r.w[i];
    return r;
}
// A whole row of n < 16
template <int DT>
__device__ __forceinline__ Raw<DT, 16> load_short_row(const char* __restrict__ row, uint32_t k, uint32_t n) {
    constexpr int XB = bytes_of(DT), W = 4 * XB;
    Raw<DT, 16> r = {};
    if (k == 0)
#pragma unroll 1
        for (uint32_t i = 0; i < n; ++i) {
            uint32_t e = 0;
            __builtin_memcpy(&e, row + (uint64_t)i * XB, XB);
            e <<= i * XB % 4 * 8;
#pragma unroll
            for (int j = 0; j < W; ++j) r.w[j] |= i * XB / 4 == (uint32_t)j ? e : 0u;
        }
    return r;
}
__device__ __forceinline__ i4 as_fragment(const Raw<DT_I8, 16>& r) { return i4{(int)r.w[0], (int)r.w[1], (int)r.w[2], (int)r.w[3]}; }

// Which of a wave's 64 channels a lane's accumulator (t, i) is: a lane's 16-byte piece of y is next to those of the other
// three lanes of its row, so a store writes 64 consecutive bytes a row: 8 channels of f16 (two accumulators), 4 of f32.
__device__ __forceinline__ uint32_t channel_of(int t, uint32_t g, bool wide) { return wide ? t * 16 + g * 4 : (t >> 1) * 32 + g * 8 + (t & 1) * 4; }

// 16 bytes of y at any place, of which `left` bytes (2 or 4 in all an element) lie inside the row
__device__ __forceinline__ void put_piece(char* p, const i4& v, uint32_t left) {
    if (left >= 16) __builtin_memcpy(p, &v, 16);
    else {   // 8, 4 and 2 bytes of it: a few instructions, where a store an element is a page of them
        if (left & 8) {
            const vec<int, 2> lo = {v[0], v[1]};
            __builtin_memcpy(p, &lo, 8);
        }
        if (left & 4) {
            const int w = left & 8 ? v[2] : v[0];
            __builtin_memcpy(p + (left & 8), &w, 4);
        }
        if (left & 2) {
            const uint16_t h = (uint16_t)(left & 8 ? (left & 4 ? v[3] : v[2]) : (left & 4 ? v[1] : v[0]));
            __builtin_memcpy(p + (left & 12), &h, 2);
        }
    }
}
template <typename T>
__device__ __forceinline__ i4 to_half(const float* v) {
    vec<T, 8> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (T)v[i];
    return __builtin_bit_cast(i4, o);
}
// One row's 16 channels of a 64-channel block from channel c0 on (v[4 t + i], channels as channel_of says), `left` > 0 of the
// 64 inside; YT: y's type, or -1: as a.y_dtype says
template <int YT = -1>
__device__ __forceinline__ void store_block(const LinearArgs& a, uint32_t row, uint32_t c0, uint32_t g, const float (&v)[16], uint32_t left) {
    const uint64_t at = (uint64_t)row * a.ld_y + c0;
    if (YT == DT_F32 || (YT < 0 && a.y_dtype == DT_F32)) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t c = channel_of(t, g, true);
            const vec<float, 4> o = {v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]};
            if (left >= 64) __builtin_memcpy((char*)a.y + (at + c) * 4, &o, 16);   // (the same for all lanes: no look at each piece)
            else if (c < left) put_piece((char*)a.y + (at + c) * 4, __builtin_bit_cast(i4, o), (left - c) * 4);
        }
    } else
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const uint32_t c = channel_of(2 * p, g, false);
            const i4 o = YT == DT_F16 || (YT < 0 && a.y_dtype == DT_F16) ? to_half<_Float16>(v + 8 * p) : to_half<__bf16>(v + 8 * p);
            if (left >= 64) __builtin_memcpy((char*)a.y + (at + c) * 2, &o, 16);
            else if (c < left) put_piece((char*)a.y + (at + c) * 2, o, (left - c) * 2);
        }
}
// A sum to its result: the row's scale last, since it has the type's whole range; low = 0 (ReLU) or -infinity.  NaN stays.
__device__ __forceinline__ float finish(int sum, float w_scale, float x_scale, float bias, float low) {
    return __builtin_elementwise_maximum(fmaf((float)sum * w_scale, x_scale, bias), low);
}
__device__ __forceinline__ float lowest(const LinearArgs& a) { return a.relu ? 0.0f : -__builtin_inff(); }

void launch_linear_rows(const LinearArgs& a, hipStream_t s);   // n_in <= 256
void launch_linear_few(const LinearArgs& a, hipStream_t s);
bool linear_few_quantizes(uint32_t rows, uint32_t n_in, uint32_t n_experts);

// f(the x type as a constant)
template <typename F>
inline void by_type(int dtype, F&& f) {
    if (dtype == DT_F16) f(std::integral_constant<int, DT_F16>{});
    else if (dtype == DT_BF16) f(std::integral_constant<int, DT_BF16>{});
    else if (dtype == DT_F32) f(std::integral_constant<int, DT_F32>{});
    else f(std::integral_constant<int, DT_I8>{});
}

}  // namespace sng
