// tree_sm100_d128.cu -- the tcgen05 tree attention at head dims up to 128.
#include "tree_sm100.cuh"

namespace bfa {

int tree_sm100_d128(const TreeParams& p, int dtype, cudaStream_t st) { return launch_d<128>(p, dtype, st); }

}  // namespace bfa
