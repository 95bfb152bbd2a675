// linear_i8_few.hip -- the 8-bit linear layer for few rows (linear_i8.hip describes the layer)
#include "linear_i8.h"

namespace sng {

// Bound by reading the weights once, and for the smallest by the chain of waits.  A workgroup takes 16 CT channels of one
// matrix and splits n_in over its NW waves, so that a whole chip of waves is loading also for one row; each wave's sums meet
// in LDS.  x (up to 16 rows at a time) is brought to 8 bits on the way: every wave reads its own part of the rows, the
// waves share the rows' maxima in LDS.  Everything that a wave of up to H fragments needs is on its way before it waits for
// the first time: weights, rows, scales.
template <int DT, int NW, int H, int CT>   // H fragments of 64 bytes at a time
__global__ __launch_bounds__(NW * 64) void linear_i8_few_kernel(LinearArgs a) {
    constexpr int XB = bytes_of(DT), RESULTS = CT * 256 / (NW * 64) > 0 ? CT * 256 / (NW * 64) : 1;
    __shared__ uint32_t tops[NW][16];
    __shared__ i4 sums[NW][CT][64];
    const uint32_t expert = blockIdx.y;
    uint32_t begin = 0, end = a.rows;
    if (a.offsets) {
        begin = (uint32_t)a.offsets[expert];
        end = min((uint32_t)a.offsets[expert + 1], a.rows);
        if (begin >= end) return;
    }
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const uint32_t n0 = blockIdx.x * (16 * CT), steps = (a.n_in + 63) / 64, per = (steps + NW - 1) / NW;
    const uint32_t s0 = min(steps, wave * per), s1 = min(steps, s0 + per);
    const int8_t* w[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) w[t] = a.w + ((uint64_t)expert * a.n_out + min(n0 + t * 16 + r, a.n_out - 1)) * a.ld_w;
    // steps past this wave's last are read as its last and not multiplied; fragments are cleared past the row's end
    const auto load_w = [&](uint32_t s, Raw<DT_I8, 16> (&f)[H][CT]) {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int t = 0; t < CT; ++t) f[h][t] = load_row16<DT_I8>((const char*)w[t], min(s + h, s1 - 1) * 64 + g * 16, a.n_in);
    };
    const bool ragged = a.n_in % 64 != 0;
    // this thread's results: row (i / 16) % 16, channel i / 256 * 16 + i % 16 for i = tid + k NW 64
    float w_scale[RESULTS], bias[RESULTS];
    const auto channel = [&](int k) { return n0 + (threadIdx.x + k * NW * 64) / 256 * 16 + (threadIdx.x & 15); };
#pragma unroll
    for (int k = 0; k < RESULTS; ++k) {
        const uint64_t at = (uint64_t)expert * a.n_out + min(channel(k), a.n_out - 1);
        w_scale[k] = a.w_scale[at];
        bias[k] = a.bias ? a.bias[at] : 0.0f;
    }
    const float low = lowest(a);
    for (uint32_t row0 = begin; row0 < end; row0 += 16) {
        const uint32_t row = row0 + r;
        const bool on = row < end;
        const char* __restrict__ x = (const char*)a.x + (uint64_t)(on ? row : row0) * a.ld_x * XB;
        const auto load_x = [&](uint32_t s, Raw<DT, 16> (&f)[H]) {
#pragma unroll
            for (int h = 0; h < H; ++h) f[h] = load_row16<DT>(x, min(s + h, s1 - 1) * 64 + g * 16, a.n_in);
        };
        Raw<DT_I8, 16> fw[H][CT];
        Raw<DT, 16> fx[H];
        i4 acc[CT] = {};
        if (s0 < s1) {   // (a wave without a part only meets the others)
            if (on) load_x(s0, fx);
            load_w(s0, fw);
        }
        RowScale rs = {};
        if constexpr (DT != DT_I8) {
            uint32_t top = 0;
            if (on && s0 < s1) {   // (elements read for others' places are the row's own too)
#pragma unroll
                for (int h = 0; h < H; ++h) top = max(top, top_bits(fx[h]));
                for (uint32_t s = s0 + H; s < s1; ++s) top = max(top, top_bits(load_row16<DT>(x, s * 64 + g * 16, a.n_in)));
            }
            top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            if (g == 0) tops[wave][r] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NW; ++i) top = max(top, tops[i][r]);
            rs = row_scale(top);
        }
        for (uint32_t s = s0; s < s1; s += H) {
            if (s > s0) {
                if (on) load_x(s, fx);
                load_w(s, fw);
            }
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const uint32_t k = min(s + h, s1 - 1) * 64 + g * 16;
                i4 q = {0, 0, 0, 0};
                if (on) {   // (most lanes have no row when there are few)
                    if (ragged) keep_inside<DT>(fx[h], k, a.n_in);
                    if constexpr (DT == DT_I8) q = as_fragment(fx[h]);
                    else q = quantize_n(fx[h], rs);
                }
                if (s + h < s1)
#pragma unroll
                    for (int t = 0; t < CT; ++t) {
                        if (ragged) keep_inside<DT_I8>(fw[h][t], k, a.n_in);
                        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(as_fragment(fw[h][t]), q, acc[t], 0, 0, 0);
                    }
            }
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) sums[wave][t][lane] = acc[t];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < RESULTS; ++k) {
            const uint32_t i = threadIdx.x + k * NW * 64, rr = (i >> 4) & 15, c = i & 15;
            if (i < CT * 256 && row0 + rr < end && channel(k) < a.n_out) {   // lane 16 (c / 4) + row held sum c % 4
                int sum = 0;
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < NW; ++j) {
                    sum += ((const int*)&sums[j][i >> 8][(c >> 2) * 16 + rr])[c & 3];
                    if constexpr (DT != DT_I8) top = max(top, tops[j][rr]);
                }
                const float v = finish(sum, w_scale[k], DT == DT_I8 ? a.x_scale[row0 + rr] : scale_of(top), bias[k], low);
                const uint64_t to = (uint64_t)(row0 + rr) * a.ld_y + channel(k);
                if (a.y_dtype == DT_F16) ((_Float16*)a.y)[to] = (_Float16)v;
                else if (a.y_dtype == DT_BF16) ((__bf16*)a.y)[to] = (__bf16)v;
                else ((float*)a.y)[to] = v;
            }
        }
        __syncthreads();
    }
}

template <int DT>
static void linear_few(const LinearArgs& a, hipStream_t s) {
    const uint32_t experts = a.offsets ? a.n_experts : 1;
    constexpr int H8 = DT == DT_F32 ? 4 : 8;   // (registers)
    if ((uint64_t)a.n_out * experts > 1024 * 16) {   // more workgroups than the chip holds at once: twice the channels each
        const dim3 grid((a.n_out + 31) / 32, experts);
        if (a.n_in <= 1024) linear_i8_few_kernel<DT, 4, 4, 2><<<grid, 256, 0, s>>>(a);
        else linear_i8_few_kernel<DT, 8, 4, 2><<<grid, 512, 0, s>>>(a);
    } else {
        const dim3 grid((a.n_out + 15) / 16, experts);
        if (a.n_in <= 1024) linear_i8_few_kernel<DT, 4, 4, 1><<<grid, 256, 0, s>>>(a);
        else linear_i8_few_kernel<DT, 8, H8, 1><<<grid, 512, 0, s>>>(a);
    }
}

void launch_linear_few(const LinearArgs& a, hipStream_t s) {
    by_type(a.x_dtype, [&](auto t) { linear_few<decltype(t)::value>(a, s); });
}

}  // namespace sng
