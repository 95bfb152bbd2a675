"""Sizes for each tile of the 8-bit linear layer: (tile, rows, n_in, n_out, experts); 0 experts: one matrix, no offsets.
test_linear_i8_rule.py holds them against the product's rule, test_gpu_linear_i8_tiles.py runs them."""
TILES = [("64x64", 500, 400, 1000, 0), ("64x128", 530, 272, 1103, 0), ("128x128", 1301, 261, 2100, 0), ("256x256", 2309, 272, 4099, 0),
         ("64x64", 200, 300, 300, 8), ("64x128", 700, 272, 1101, 5), ("128x128", 2001, 272, 2102, 5), ("256x256", 2405, 261, 4100, 3)]
