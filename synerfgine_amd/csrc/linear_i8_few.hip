// linear_i8_few.hip -- the 8-bit linear layer for few rows (linear_i8.hip describes the layer)
#include "linear_i8.h"

namespace sng {

// Bound by reading the weights once (16 experts of 1024 -> 2048, 48 rows: 33.5 MB, 10.6 us, 3.2 TB/s), and for the smallest by
// the chain of waits (one row, 4096 -> 4096: 6.8 us from memory, 5.2 from the dies' caches).  A workgroup takes 16 CT channels of one
// matrix and splits n_in over its NW waves, so that a whole chip of waves is loading also for one row; each wave's sums meet
// in LDS.  x (up to 16 rows at a time) in floating point is brought to 8 bits on the way, by all waves together, into LDS,
// where the fragments are read from: with few rows most lanes of a fragment would have none to work on.  Every workgroup does
// that again, which is little beside its weights.  The rows are asked for first and the first weights right behind them:
// loads come back in their order, and the weights have the time that the rows' way to 8 bits takes.
//
// A call runs every instruction about once, out of a cold instruction cache: what is repeated is a loop, and the weights of
// a row's end are taken as load_row16 gives them.  (4097 -> 4096, one row, 8 waves, before ODD: 18 us; 20.5 us with code between
// the matrix instructions that moves them to their places, each jump over it a miss.  ODD: weights at odd places, 9.2 us
// with 16 waves.)  The figures of the rules below are of calls on the same buffers again, the weights in the card's caches.
constexpr uint32_t FEW_LDS = 60 * 1024;   // for x's rows
static uint32_t few_stride(uint32_t n_in) { return (n_in + 63) / 64 * 64 + 16; }   // (+ 16: the rows of a fragment read lie on different banks)

template <int DT, int NW, int H, int CT, bool ODD>   // H fragments of 64 bytes at a time
__global__ __launch_bounds__(NW * 64) void linear_i8_few_kernel(LinearArgs a, uint32_t group, uint32_t stride) {
    constexpr int XB = bytes_of(DT), T = NW * 64, RESULTS = CT * 256 / T > 0 ? CT * 256 / T : 1;
    extern __shared__ __align__(16) int8_t lq[];   // [group][stride]
    __shared__ uint32_t tops[16][NW];
    __shared__ i4 sums[NW][CT][64];
    const uint32_t expert = blockIdx.y;
    uint32_t begin = 0, end = a.rows;
    if (a.offsets) {
        begin = (uint32_t)a.offsets[expert];
        end = min((uint32_t)a.offsets[expert + 1], a.rows);
        if (begin >= end) return;
    }
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, r = lane & 15, n = a.n_in;
    const uint32_t n0 = blockIdx.x * (16 * CT), steps = (n + 63) / 64, per = (steps + NW - 1) / NW;
    const uint32_t s0 = min(steps, wave * per), s1 = min(steps, s0 + per);
    const char* w[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) w[t] = (const char*)a.w + ((uint64_t)expert * a.n_out + min(n0 + t * 16 + r, a.n_out - 1)) * a.ld_w;
    // steps past this wave's last are read as its last and not multiplied
    using Weights = std::conditional_t<ODD, OddBytes, Raw<DT_I8, 16>>;
    const auto load_w = [&](uint32_t s, Weights (&f)[H][CT]) {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const uint32_t k = min(s + h, s1 - 1) * 64 + g * 16;
                if constexpr (ODD) f[h][t] = load_odd16(w[t], k, n);
                else f[h][t] = load_row16<DT_I8>(w[t], k, n);
            }
    };
    // x's units of 16 values: a row's lie on WPR waves (several a thread where it has more), RPP rows a pass
    const uint32_t units = steps * 4, wpr = min((units + 63) / 64, (uint32_t)NW), rpp = NW / wpr, my_row = wave / wpr, my_unit = (wave % wpr) * 64 + lane;
    // this thread's results: row (i / 16) % 16, channel i / 256 * 16 + i % 16 for i = tid + k T
    float w_scale[RESULTS], bias[RESULTS];
    const auto channel = [&](int k) { return n0 + (threadIdx.x + k * T) / 256 * 16 + (threadIdx.x & 15); };
#pragma unroll
    for (int k = 0; k < RESULTS; ++k) {
        const uint64_t at = (uint64_t)expert * a.n_out + min(channel(k), a.n_out - 1);
        w_scale[k] = a.w_scale[at];
        bias[k] = a.bias ? a.bias[at] : 0.0f;
    }
    for (uint32_t row0 = begin; row0 < end; row0 += group) {
        const uint32_t rows = min(group, end - row0);
        Weights fw[H][CT];
        if constexpr (DT == DT_I8) {
            if (s0 < s1) load_w(s0, fw);   // (a wave without a part only meets the others)
        } else {
            const auto get = [&](uint32_t row, uint32_t u) { return load_row16<DT>((const char*)a.x + (uint64_t)(row0 + row) * a.ld_x * XB, u * 16, n); };
            const bool one = rows <= rpp && units <= wpr * 64;   // one unit a thread: it stays in registers
            Raw<DT, 16> held = {};
            if (my_row < rows && my_unit < units) held = get(my_row, my_unit);
            if (s0 < s1) load_w(s0, fw);
            // (a wave without a row of its own in a pass: none)
#pragma unroll 1
            for (uint32_t row = my_row < rpp ? my_row : rows; row < rows; row += rpp) {
                uint32_t top = 0;
#pragma unroll 1
                for (uint32_t u = my_unit; u < units; u += wpr * 64) {
                    if (!one) held = get(row, u);
                    top = max(top, top_bits(held));
                }
#pragma unroll
                for (int m = 32; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
                if (lane == 0) tops[row][wave % wpr] = top;
            }
            __syncthreads();
#pragma unroll 1
            for (uint32_t row = my_row < rpp ? my_row : rows; row < rows; row += rpp) {
                uint32_t top = 0;
#pragma unroll 1
                for (uint32_t i = 0; i < wpr; ++i) top = max(top, tops[row][i]);
                const RowScale rs = row_scale(top);
#pragma unroll 1
                for (uint32_t u = my_unit; u < units; u += wpr * 64) {
                    if (!one) held = get(row, u);
                    *(i4*)(lq + row * stride + u * 16) = new_bytes(quantize_n(held, rs), u * 16, n);
                }
            }
            __syncthreads();
        }
        i4 acc[CT] = {};
        for (uint32_t s = s0; s < s1; s += H) {
            Raw<DT_I8, 16> fx[H];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const uint32_t k = min(s + h, s1 - 1) * 64 + g * 16, row = min(r, rows - 1);
                if constexpr (DT == DT_I8) fx[h] = load_row16<DT_I8>((const char*)a.x + (uint64_t)(row0 + row) * a.ld_x, k, n);
                else __builtin_memcpy(&fx[h], __builtin_assume_aligned(lq + row * stride + k, 16), 16);
            }
            if (s > s0) load_w(s, fw);
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (s + h >= s1) break;
                const uint32_t k = (s + h) * 64 + g * 16;
                i4 x = as_fragment(fx[h]);
                if (DT == DT_I8 && (s + h + 1) * 64 > n) x = new_bytes(x, k, n);
#pragma unroll
                for (int t = 0; t < CT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(as_fragment(whole(fw[h][t])), x, acc[t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) sums[wave][t][lane] = acc[t];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < RESULTS; ++k) {
            const uint32_t i = threadIdx.x + k * T, rr = (i >> 4) & 15, c = i & 15;
            if (i < CT * 256 && rr < rows && channel(k) < a.n_out) {   // lane 16 (c / 4) + row held sum c % 4
                int sum = 0;
#pragma unroll
                for (int j = 0; j < NW; ++j) sum += ((const int*)&sums[j][i >> 8][(c >> 2) * 16 + rr])[c & 3];
                float scale;
                if constexpr (DT == DT_I8) scale = a.x_scale[row0 + rr];
                else {
                    uint32_t top = 0;
#pragma unroll 1
                    for (uint32_t j = 0; j < wpr; ++j) top = max(top, tops[rr][j]);
                    scale = scale_of(top);
                }
                const float v = finish(sum, w_scale[k], scale, bias[k], lowest(a));
                const uint64_t to = (uint64_t)(row0 + rr) * a.ld_y + channel(k);
                if (a.y_dtype == DT_F16) ((_Float16*)a.y)[to] = (_Float16)v;
                else if (a.y_dtype == DT_BF16) ((__bf16*)a.y)[to] = (__bf16)v;
                else ((float*)a.y)[to] = v;
            }
        }
        if (row0 + group < end) __syncthreads();
    }
}

template <int DT, int CT, bool ODD>
static void linear_few_of(const LinearArgs& a, hipStream_t s) {
    const uint32_t stride = few_stride(a.n_in), group = DT == DT_I8 ? 16 : std::min(16u, FEW_LDS / stride), lds = DT == DT_I8 ? 0 : group * stride;
    const dim3 grid((a.n_out + 16 * CT - 1) / (16 * CT), a.offsets ? a.n_experts : 1);
    // short sums: 8 waves where they all find room, so that more rows are brought to 8 bits at a time (1024 -> 1024: 8 rows 4.2 us,
    // 5.0 with 4 waves; 16 experts of 1024 -> 2048, 4 rows each: 9.5 and 8.6)
    if constexpr (CT > 1) {
        if (a.n_in <= 1024) linear_i8_few_kernel<DT, 4, 4, CT, ODD><<<grid, 256, lds, s>>>(a, group, stride);
        else linear_i8_few_kernel<DT, 8, 4, CT, ODD><<<grid, 512, lds, s>>>(a, group, stride);
    } else if (a.n_in <= 1024) linear_i8_few_kernel<DT, 8, 2, 1, ODD><<<grid, 512, lds, s>>>(a, group, stride);
    // longer ones: 16 waves where every workgroup has a CU of its own (8192 -> 1024: a row 6.8 us, 7.8 with 8; 2048 -> 8192: 7.1 and 6.8)
    else if (grid.x * grid.y <= 256) linear_i8_few_kernel<DT, 16, 4, 1, ODD><<<grid, 1024, lds, s>>>(a, group, stride);
    else linear_i8_few_kernel<DT, 8, 8, 1, ODD><<<grid, 512, lds, s>>>(a, group, stride);
}

template <int DT>
static void linear_few(const LinearArgs& a, hipStream_t s) {
    // more workgroups than the chip holds at once: twice the channels each
    const bool many = (uint64_t)a.n_out * (a.offsets ? a.n_experts : 1) > 1024 * 16, odd = ((uint64_t)a.w | a.ld_w | a.n_in) % 4 != 0;
    if (odd) many ? linear_few_of<DT, 2, true>(a, s) : linear_few_of<DT, 1, true>(a, s);
    else many ? linear_few_of<DT, 2, false>(a, s) : linear_few_of<DT, 1, false>(a, s);
}

// Whether x is brought to 8 bits by every workgroup or before, by a launch of its own (which costs the host 3 us too): up to
// 24576 values an expert's rows (4096 -> 4096, f32: 5 rows 9.9 us, 8 rows 8.9 us with the launch; bf16: 6 rows 7.7, 8 rows 9.0;
// 8192 -> 1024, bf16: 2 rows 8.0, 4 rows 10.6)
bool linear_few_quantizes(uint32_t rows, uint32_t n_in, uint32_t n_experts) { return (uint64_t)rows * n_in <= 24576ull * n_experts && few_stride(n_in) <= FEW_LDS / 2; }
void launch_linear_few(const LinearArgs& a, hipStream_t s) {
    by_type(a.x_dtype, [&](auto t) { linear_few<decltype(t)::value>(a, s); });
}

}  // namespace sng
