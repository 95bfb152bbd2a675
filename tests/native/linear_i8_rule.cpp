// Prints, for each line "rows n_in n_out experts" of its input (0 experts: one matrix, no offsets), the kernel and the tile that
// the product's rule (synerfgine_amd/csrc/linear_i8_rule.h) gives the 8-bit linear layer.  Compiled by
// tests/test_linear_i8_rule.py as plain host code.
#include "linear_i8_rule.h"
#include <cstdio>
using namespace sng;

int main() {
    unsigned rows, n_in, n_out, experts;
    while (std::scanf("%u %u %u %u", &rows, &n_in, &n_out, &experts) == 4) {
        const unsigned e = experts ? experts : 1;
        const LinearKernel k = linear_i8_kernel(rows, n_in, n_out, e);
        const LinearSplit s = linear_i8_split(rows, n_in, n_out, e);
        const LinearTile t = linear_i8_tile(rows, n_out, e, experts != 0);
        const char* tile = t == LinearTile::T64 ? "64x64" : t == LinearTile::T64x128 ? "64x128" : t == LinearTile::T128 ? "128x128" : "256x256";
        std::printf("%s\n", k == LinearKernel::Rows ? "rows" : k == LinearKernel::Few ? "few" : s.splits > 1 ? "split" : tile);
    }
    return 0;
}
