// linear_i8_rule.h -- which kernel of the 8-bit linear layer (linear_i8.hip) a call takes, by its sizes alone, so that the
// workspace's size is known before the call.  Plain host code.  Figures: calls on the same buffers again.
#pragma once
#include <algorithm>
#include <stdint.h>

namespace sng {

enum class LinearKernel { Rows, Few, Tile };
inline LinearKernel linear_i8_kernel(uint32_t rows, uint32_t n_in, uint32_t n_out, uint32_t n_experts) {
    // above 128 the rows' registers leave few waves, and every 256 channels bring x to 8 bits again (256 -> 4096: 20000 rows
    // 85 us, 64 in tiles; 512 rows 7.1 and 9.2; 256 -> 1024, 20000 rows 28 and 32)
    if (n_in <= 128 || (n_in <= 256 && (n_out <= 1024 || (uint64_t)rows * n_out <= 1u << 22))) return LinearKernel::Rows;
    // a fragment's 16 rows; by expert 12, since some have more (128 experts of 768 -> 1024: 12 rows 36 us, 34 in tiles; 8 rows 31, 33)
    if (n_in > 256 && rows <= (n_experts == 1 ? 16u : 12u * n_experts)) return LinearKernel::Few;
    return LinearKernel::Tile;
}

// Into how many parts the sums over n_in are split where there are few tiles, and the bytes of the parts' sums.
// Up to 128 tiles of 64 x 64 leave half of the CUs or more without one; parts of at least 4 steps, up to two workgroups a CU.  (32 x
// 8192 -> 1024: 15.7 us of 24.8, 17 x 2092 -> 321: 14.9 of 23.7; below 16 steps the join's launch is the larger part.)
struct LinearSplit { uint32_t splits; uint64_t bytes; };
inline LinearSplit linear_i8_split(uint32_t rows, uint32_t n_in, uint32_t n_out, uint32_t n_experts) {
    const uint64_t tiles = (((uint64_t)rows >> 6) + n_experts) * ((n_out + 63) / 64), steps = (n_in + 127) / 128;
    if (linear_i8_kernel(rows, n_in, n_out, n_experts) != LinearKernel::Tile || tiles > 128 || steps < 16) return {1, 0};
    const uint32_t splits = (uint32_t)std::min<uint64_t>(steps / 4, 512 / tiles);
    return {splits, splits * tiles * (64 * 64 * sizeof(int32_t))};
}

// The tile, rows by channels, of a call that is not split and whose rows and weights lie in multiples of 16 bytes.
// (Measured: 4096 -> 4096, 512 rows: 64 x 128 22 us, 128 x 128 31, 256 x 256 50; 2048 rows: 69, 45, 53; 8192: 256, 158, 130;
// 128 experts of 100 rows, 768 -> 1024: 73, 49, 58)
enum class LinearTile { T64, T64x128, T128, T256 };
inline LinearTile linear_i8_tile(uint32_t rows, uint32_t n_out, uint32_t n_experts, bool by_expert) {
    // tiles with rows in them; by expert as if all had the same number, since the host does not know the offsets
    const auto likely = [&](uint32_t high, uint32_t wide) {
        const uint64_t e = by_expert ? n_experts : 1, of_one = (rows + e - 1) / e;
        return e * ((of_one + high - 1) / high) * ((n_out + wide - 1) / wide);
    };
    const uint32_t slots = 256;   // CUs: a round of workgroups of 64 x 128 and 256 x 256, half a round of 128 x 128
    const uint64_t t128 = likely(128, 128), t256 = likely(256, 256);
    if (likely(64, 64) <= slots / 2) return LinearTile::T64;
    if (likely(64, 128) <= (by_expert ? slots * 7 / 8 : slots)) return LinearTile::T64x128;
    if (t128 <= 2 * slots || t128 * 17 <= (t256 + slots - 1) / slots * slots * 40) return LinearTile::T128;
    return LinearTile::T256;
}

}  // namespace sng
