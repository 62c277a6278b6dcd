// tree_sm100.cu -- which problems the tcgen05 tree attention takes, and its tile.
#include <climits>

#include "sm100_host.h"
#include "tree_common.cuh"

namespace bfa {

int tree_sm100_d64(const TreeParams& p, int dtype, cudaStream_t st);
int tree_sm100_d128(const TreeParams& p, int dtype, cudaStream_t st);
int tree_sm100_d256(const TreeParams& p, int dtype, cudaStream_t st);

// Rows per block: 32 (stored four times), 128, or 256 (two tiles; O of two
// tiles does not fit TMEM at head dim 256). Joining the four quarters costs
// more the wider O is: at head dim 256 it pays only where the softmax is the
// longer part, with a soft-cap (device times with and without the four copies:
// B=16, 8 KV heads, one node: head dim 64, L=4096 45 and 57 us, head dim 128,
// L=8192 95 and 104 us; head dim 256, B=8, L=4096 61 and 58 us, and 67 against
// 69 us with a soft-cap, 15 nodes and a window).
TreeTile tree_sm100_tile(int64_t rows, int D, bool cap) {
  const bool four = rows <= 32 && (D <= 128 || cap);
  return {four ? 32 : rows > 128 && D <= 128 ? 256 : 128, D > 128 ? 64 : 128, 1};
}

bool tree_sm100_layout(const bfa_tree_args* a) {
  return device_is_sm100() && a->head_dim % 8 == 0 && a->page_size % 8 == 0 && a->num_pages > 0 && a->num_pages < INT32_MAX &&
         a->max_pages > 0 && vector_rows(a->q, 2) && vector_rows(a->o, 2) && tma_layout_ok(a->k.data, a->k.stride, 2) &&
         tma_layout_ok(a->v.data, a->v.stride, 2) && tma_layout_ok(a->k_pages.data, a->k_pages.stride, 2) &&
         tma_layout_ok(a->v_pages.data, a->v_pages.stride, 2);
}

int tree_sm100(const TreeParams& p, int dtype, cudaStream_t st) {
  if (p.D <= 64) return tree_sm100_d64(p, dtype, st);
  if (p.D <= 128) return tree_sm100_d128(p, dtype, st);
  return tree_sm100_d256(p, dtype, st);
}

}  // namespace bfa
