// tree_sm100_d64.cu -- the tcgen05 tree attention at head dims up to 64.
#include "tree_sm100.cuh"

namespace bfa {

int tree_sm100_d64(const TreeParams& p, int dtype, cudaStream_t st) { return launch_d<64>(p, dtype, st); }

}  // namespace bfa
