// linear_i8_rows.hip -- the 8-bit linear layer for short rows (linear_i8.hip describes the layer)
#include "linear_i8.h"

namespace sng {

// n_in <= 256: a row is at most 4 fragments of 64 bytes, so a wave loads 16 rows, finds their scales, brings them to 8 bits
// and multiplies them without leaving its registers: x is read once and y written once, the floor of a layer this small.
// A lane holds the 16 consecutive values of one row that the matrix instruction wants of it; the four lanes of a row share
// their maximum with two shuffles.  The weights of up to 256 channels lie in LDS in fragment order (one linear
// ds_read_b128 a fragment, no bank conflicts), staged once for the workgroup's rows, which belong to one expert.
// x of type DT; KC fragments of 64 a row; NB blocks of 64 channels.  YT: y's type, or -1: any, at more registers and so fewer
// waves; -2: any, and n_in below 16.  What hides the memory's latency here is waves, in small workgroups.  2^20 x 64 -> 64
// f16: 268 MB, 53 us (5.1 TB/s, a large copy's rate); by expert, 2^19 rows on 512 experts, 32 -> 64: 31.5 us (3.2 TB/s: 32
// values fill half of the matrix instruction).
template <int DT, int YT, int KC, int NB>
__global__ __launch_bounds__(256) void linear_i8_rows_kernel(LinearArgs a, uint32_t shift) {
    constexpr int XB = bytes_of(DT);
    constexpr bool TINY = YT == -2;
    __shared__ i4 lw[NB * 4 * KC * 64];
    __shared__ __align__(16) float lscale[NB * 64], lbias[NB * 64];
    const RowTile tile = row_tile(a, blockIdx.x, shift);
    if (tile.begin >= tile.end) return;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n0 = blockIdx.y * (NB * 64), n = a.n_in;
    const bool wide = YT >= 0 ? YT == DT_F32 : a.y_dtype == DT_F32;
    const auto fetch = [&](uint32_t r0, Raw<DT, 16> (&raw)[KC]) {
        const char* row = (const char*)a.x + (uint64_t)min(r0 + (lane & 15), tile.end - 1) * a.ld_x * XB;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) raw[kc] = TINY ? load_short_row<DT>(row, kc * 64 + g * 16, n) : load_row16<DT>(row, kc * 64 + g * 16, n);
    };
    Raw<DT, 16> raw[KC];
    uint32_t r0 = tile.begin + wave * 16;
    if (r0 < tile.end) fetch(r0, raw);
    {   // the scales' and the first weights' loads before any of them is waited for
        const int8_t* __restrict__ w = (const int8_t*)a.w + (uint64_t)tile.expert * a.n_out * a.ld_w;
        const uint64_t c = (uint64_t)tile.expert * a.n_out + min(n0 + threadIdx.x, a.n_out - 1);   // (past the last channel: not used)
        const float scale = a.w_scale[c], bias = a.bias ? a.bias[c] : 0.0f;
        const auto w_row = [&](int i) {   // the channel and place in it of fragment lane i * 256 + tid
            const uint32_t f = i * 256 + threadIdx.x, t = (f >> 6) / KC & 3, nb = (f >> 6) / (4 * KC);
            return (const char*)w + (uint64_t)min(n0 + nb * 64 + channel_of(t, (f >> 2) & 3, wide) + (f & 3), a.n_out - 1) * a.ld_w;
        };
        const auto w_k = [&](int i) { return ((i * 256 + threadIdx.x) >> 6) % KC * 64 + ((threadIdx.x & 63) >> 4) * 16; };
#pragma unroll
        for (int i0 = 0; i0 < NB * KC; i0 += 4) {   // (up to four loads at a time: registers)
            constexpr int I = NB * KC < 4 ? NB * KC : 4;
            Raw<DT_I8, 16> fw[I];
#pragma unroll
            for (int i = 0; i < I; ++i) fw[i] = TINY ? load_short_row<DT_I8>(w_row(i0 + i), w_k(i0 + i), n) : load_row16<DT_I8>(w_row(i0 + i), w_k(i0 + i), n);
#pragma unroll
            for (int i = 0; i < I; ++i) lw[(i0 + i) * 256 + threadIdx.x] = as_fragment(fw[i]);   // (channels past the last: multiplied, not stored)
        }
        if (threadIdx.x < NB * 64) {
            lscale[threadIdx.x] = scale;
            lbias[threadIdx.x] = bias;
        }
    }
    __syncthreads();
    const float low = lowest(a);
    for (; r0 < tile.end; r0 += 64) {
        asm volatile("" ::: "memory");   // (else the scales are kept over the loop, in the registers of several waves)
        const uint32_t row = r0 + (lane & 15);
        i4 q[KC];
        float scale;
        if constexpr (DT == DT_I8) {
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) q[kc] = as_fragment(raw[kc]);
            scale = a.x_scale[min(row, tile.end - 1)];
        } else {
            uint32_t top = 0;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) top = max(top, top_bits(raw[kc]));
            top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            const RowScale rs = row_scale(top);
            scale = rs.scale;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) q[kc] = quantize_n(raw[kc], rs);
        }
        if (!TINY && n != KC * 64) {
            uint32_t k = g * 16;
            asm volatile("" : "+v"(k));   // (masks made ahead of the loop would stay in registers)
#pragma unroll
            for (int kc = KC / 2; kc < KC; ++kc) q[kc] = new_bytes(q[kc], kc * 64 + k, n);   // (n is above KC / 2 fragments)
        }
        if (r0 + 64 < tile.end) fetch(r0 + 64, raw);   // before the stores: a wait for loads is one for the stores before them too
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const uint32_t c0 = n0 + nb * 64;
            if (c0 >= a.n_out) break;
            const uint32_t left = a.n_out - c0;
            float v[16];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                i4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(lw[((nb * 4 + t) * KC + kc) * 64 + lane], q[kc], acc, 0, 0, 0);
                const uint32_t c = nb * 64 + channel_of(t, g, wide);
                const vec<float, 4> ws = *(const vec<float, 4>*)(lscale + c), b = *(const vec<float, 4>*)(lbias + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * t + i] = finish(acc[i], ws[i], scale, b[i], low);
            }
            if (row >= tile.end) continue;
            store_block<YT>(a, row, c0, g, v, left);
        }
    }
}

template <int DT, int YT, int KC>
static void linear_rows(const LinearArgs& a, hipStream_t s) {
    // Rows a workgroup: few where there are few, so that the chip is filled; else 128 (2^20 x 64 -> 64: 52.8 us; with 256 rows 55.7, with 512
    // 61.8).
    uint32_t shift = 6;
    if ((a.rows >> shift) > 2048) ++shift;
    // Channels a workgroup: 64 where there are few rows (staging 256 channels of 256 weights took 7 us of a 3.5 us call);
    // more where the rows fill the chip, since x is read and brought to 8 bits again for each of them.
    const uint32_t tiles = row_tiles(a, shift), nb = a.n_out <= 64 || tiles < 256 ? 1 : a.n_out <= 128 && YT >= 0 ? 2 : 4;
    const dim3 grid(tiles, (a.n_out + nb * 64 - 1) / (nb * 64));
    if (nb == 1) linear_i8_rows_kernel<DT, YT, KC, 1><<<grid, 256, 0, s>>>(a, shift);
    else if constexpr (YT >= 0) {
        if (nb == 2) linear_i8_rows_kernel<DT, YT, KC, 2><<<grid, 256, 0, s>>>(a, shift);
    }
    if (nb == 4) linear_i8_rows_kernel<DT, YT, KC, 4><<<grid, 256, 0, s>>>(a, shift);
}
template <int DT, int YT>
static void linear_rows_of(const LinearArgs& a, hipStream_t s) {
    if (a.n_in < 16) linear_rows<DT, -2, 1>(a, s);
    else if (a.n_in <= 64) linear_rows<DT, YT, 1>(a, s);
    else if (a.n_in <= 128) linear_rows<DT, YT, 2>(a, s);
    else linear_rows<DT, YT, 4>(a, s);
}
template <int DT>
static void linear_rows_by_type(const LinearArgs& a, hipStream_t s) {
    if constexpr (DT == DT_I8) {
        if (a.y_dtype == DT_F16) linear_rows_of<DT, DT_F16>(a, s);
        else if (a.y_dtype == DT_BF16) linear_rows_of<DT, DT_BF16>(a, s);
        else linear_rows_of<DT, DT_F32>(a, s);
    } else if (a.y_dtype == DT) linear_rows_of<DT, DT>(a, s);   // (a layer's output is its input's type; others: the general one)
    else linear_rows_of<DT, -1>(a, s);
}

void launch_linear_rows(const LinearArgs& a, hipStream_t s) {
    by_type(a.x_dtype, [&](auto t) { linear_rows_by_type<decltype(t)::value>(a, s); });
}

}  // namespace sng
