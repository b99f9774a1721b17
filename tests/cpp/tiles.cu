// The tiles of a ragged batch as the attention kernels find them, on the host:
// reads g, rows of a tile, n_seq, n_tokens and q_start[n_seq + 1] from the
// command line and prints, for every tile of the launch, its sequence and its
// first row in it (-1: no tile).
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../hesa-llm_b200/csrc/paged.h"

int main(int argc, char** argv) {
    using namespace hesa_cuda;
    const int g = std::atoi(argv[1]), r = std::atoi(argv[2]), n_seq = std::atoi(argv[3]), n_tokens = std::atoi(argv[4]);
    std::vector<int32_t> starts;
    for (int i = 5; i < argc; ++i) starts.push_back(std::atoi(argv[i]));
    const BatchView b{nullptr, starts.data(), n_seq, n_tokens, n_tokens, n_tokens};
    const int64_t tiles = tile_bound(n_tokens, n_seq, g, r);
    for (int idx = 0; idx < tiles; ++idx) {
        int seq = 0, tile = 0;
        const bool some = locate_tile(b, g, r, 0, idx, seq, tile);
        std::printf("%d %d\n", seq, some ? tile * r : -1);
    }
    return 0;
}
