// tree_sm100_d256.cu -- the tcgen05 tree attention at head dims up to 256.
#include "tree_sm100.cuh"

namespace bfa {

int tree_sm100_d256(const TreeParams& p, int dtype, cudaStream_t st) { return launch_d<256>(p, dtype, st); }

}  // namespace bfa
