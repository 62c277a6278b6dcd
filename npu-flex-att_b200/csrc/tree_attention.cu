// tree_attention.cu -- the entry points of tree attention: checks, the choice
// of kernel and grid, the workspace and the merge of partial results.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "tree_common.cuh"

namespace bfa {
namespace {

// Joins the partial (O, LSE) of items that several blocks worked on, one warp
// per row, partials in the order of their keys:
//   lse = log2 sum_i 2^lse_i,  O = sum_i O_i·2^(lse_i - lse).
// Rows of an item that one block did whole are already final.
template <typename T>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int GN = p.G * p.N;
  if (row >= (int64_t)p.B * p.Hkv * GN) return;
  const int r_all = (int)(row % GN), hkv = (int)(row / GN % p.Hkv), b = (int)(row / GN / p.Hkv);
  const int rbk = r_all / p.rb, r = r_all - rbk * p.rb;
  const int64_t T_all = tree_chunks_before(p, p.B);
  const int len = tree_len(p, b), n_chunks = tree_chunks_of(p, len);
  const int64_t s0 = tree_chunks_before(p, b) + (int64_t)(hkv * p.n_rb + rbk) * n_chunks;
  const int blocks = tree_blocks(p, T_all);
  const int i0 = tree_owner(T_all, blocks, s0), i1 = tree_owner(T_all, blocks, s0 + n_chunks - 1);
  if (i0 == i1) return;
  auto slot = [&](int i) { return ((int64_t)i * 2 + (i == i0 ? 1 : 0)) * p.rb + r; };
  float m = neg_inf();
  for (int i = i0 + lane; i <= i1; i += 32) m = fmaxf(m, p.part_lse[slot(i)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  int hq, n;
  tree_row(p, hkv, r_all, &hq, &n);
  T* out = static_cast<T*>(p.o) + b * p.so[0] + hq * p.so[1] + n * p.so[2];
  float total = 0.f, acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = 0.f;
  if (m != neg_inf()) {
    for (int i = i0; i <= i1; ++i) {
      const int64_t at = slot(i);
      const float w = exp2f(p.part_lse[at] - m);
      total += w;
      const float* po = p.part_o + at * p.D;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (lane + 32 * c < p.D) acc[c] = fmaf(w, po[lane + 32 * c], acc[c]);
    }
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (lane + 32 * c < p.D) out[lane + 32 * c] = from_f32<T>(acc[c] * inv);
  if (lane == 0 && p.lse) {
    float l = neg_inf();
    if (total > 0.f) {
      l = (m + log2f(total)) * kLn2;
      if (p.alibi) {  // the row's depth, by the way up to the root
        int depth = 0;
        for (int x = n; x > 0; ++depth) {
          const int up = p.parents ? p.parents[b * p.parents_stride + x] : x - 1;
          if (up < 0 || up >= x) break;
          x = up;
        }
        l += tree_row_shift(p, hq, len + depth);
      }
    }
    p.lse[((int64_t)b * p.Hq + hq) * p.N + n] = l;
  }
}

int check_tree(const bfa_tree_args* a) {
  if (!a || a->batch < 0 || a->heads_q < 0 || a->heads_kv < 1 || a->nodes < 1 || a->num_pages < 0 || a->page_size < 1 ||
      a->max_pages < 0 || a->sliding_window < 0 || !(a->soft_cap >= 0))
    return BFA_ERR_INVALID_ARGUMENT;
  if (a->heads_q % a->heads_kv != 0) return BFA_ERR_SHAPE;
  if (a->head_dim < 1 || a->head_dim > 256 || a->nodes > kTreeNodes || a->dtype != (int)a->dtype ||
      dtype_bytes((int)a->dtype) == 0)
    return BFA_ERR_UNSUPPORTED;
  // Positions, rows per KV head and items are counted in 32 bits.
  if (a->batch > (1 << 24) || a->heads_q > (1 << 20) || a->page_size > INT32_MAX / 2 ||
      a->max_pages > (INT32_MAX / 2 - 128) / a->page_size || a->batch * a->heads_q > INT32_MAX / kTreeNodes)
    return BFA_ERR_UNSUPPORTED;
  return BFA_OK;
}

struct Plan {
  int rb, n_rb, chunk, tree_chunks, grid;
  size_t lse_at, bytes;
};

// Row block, chunk and grid of a problem: a function of sizes and type alone.
Plan make_plan(const bfa_tree_args* a) {
  Plan pl{};
  const int64_t rows = a->heads_q / a->heads_kv * a->nodes;
  const TreeTile tile = a->dtype == BFA_DTYPE_F32 ? TreeTile{kTreeSimtRows, kTreeSimtChunk, a->head_dim > 128 ? 1 : 2}
                                                  : tree_mma_tile(rows, (int)a->head_dim);
  pl.rb = tile.rb;
  pl.chunk = tile.chunk;
  pl.n_rb = (int)((rows + pl.rb - 1) / pl.rb);
  pl.tree_chunks = (int)((a->nodes + pl.chunk - 1) / pl.chunk);
  // At most one stretch per chunk that the tables could hold.
  int64_t seen = a->max_pages * a->page_size;
  if (a->sliding_window > 0) seen = std::min(seen, a->sliding_window);
  const int64_t chunks = ((seen + pl.chunk - 1) / pl.chunk + pl.tree_chunks) * a->batch * a->heads_kv * pl.n_rb;
  pl.grid = (int)std::min<int64_t>(chunks, (int64_t)sm_count() * tile.per_sm);
  const size_t rows_ws = (size_t)pl.grid * 2 * pl.rb;
  pl.lse_at = (rows_ws * a->head_dim * 4 + 255) / 256 * 256;
  pl.bytes = pl.lse_at + (rows_ws * 4 + 255) / 256 * 256;
  return pl;
}

template <typename T>
int launch_merge(const TreeParams& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.B * p.Hkv * p.G * p.N;
  tree_merge_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(p);
  note_launch();
  return launch_status("tree merge launch");
}

}  // namespace
}  // namespace bfa

extern "C" size_t bfa_tree_workspace_bytes(const bfa_tree_args* a) {
  using namespace bfa;
  if (check_tree(a) || a->batch * a->heads_q == 0) return 0;
  return make_plan(a).bytes;
}

extern "C" int bfa_tree_fwd(const bfa_tree_args* a, void* stream) {
  using namespace bfa;
  const int bad = check_tree(a);
  if (bad) return bad;
  if (a->batch * a->heads_q == 0) return BFA_OK;
  if (!a->q.data || !a->k.data || !a->v.data || !a->o.data || !a->lens ||
      (a->max_pages > 0 && (!a->page_table || (a->num_pages > 0 && (!a->k_pages.data || !a->v_pages.data)))))
    return BFA_ERR_INVALID_ARGUMENT;
  const bfa_tensor* unit[] = {&a->q, &a->k, &a->v, &a->o, &a->k_pages, &a->v_pages};
  for (const bfa_tensor* t : unit)
    if (t->data && a->head_dim > 1 && t->stride[3] != 1) return BFA_ERR_UNSUPPORTED;
  const Plan pl = make_plan(a);
  if (!a->workspace || a->workspace_bytes < (int64_t)pl.bytes || ((uintptr_t)a->workspace & 255u) != 0)
    return BFA_ERR_WORKSPACE;
  TreeParams p{};
  p.q = a->q.data; p.k = a->k.data; p.v = a->v.data; p.o = a->o.data;
  p.lse = a->lse;
  p.kp = a->k_pages.data; p.vp = a->v_pages.data;
  for (int i = 0; i < 4; ++i) {
    p.sq[i] = a->q.stride[i]; p.sk[i] = a->k.stride[i]; p.sv[i] = a->v.stride[i]; p.so[i] = a->o.stride[i];
    p.skp[i] = a->k_pages.stride[i]; p.svp[i] = a->v_pages.stride[i];
  }
  p.table = a->page_table; p.table_stride = a->page_table_stride;
  p.lens = a->lens;
  p.parents = a->parents; p.parents_stride = a->parents_stride;
  p.alibi = a->alibi_slopes;
  p.status = a->status;
  p.num_pages = a->num_pages;
  p.B = (int)a->batch; p.Hq = (int)a->heads_q; p.Hkv = (int)a->heads_kv; p.G = p.Hq / p.Hkv;
  p.N = (int)a->nodes; p.D = (int)a->head_dim; p.page = (int)a->page_size;
  p.cap_tokens = (int)(a->max_pages * a->page_size);
  p.window = (int)std::min<int64_t>(a->sliding_window, INT32_MAX / 2);
  p.scale = (float)a->scale;
  p.soft_cap = (float)a->soft_cap;
  p.grid = pl.grid; p.rb = pl.rb; p.n_rb = pl.n_rb; p.chunk = pl.chunk; p.tree_chunks = pl.tree_chunks;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_lse = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + pl.lse_at);
  cudaStream_t st = (cudaStream_t)stream;
  const int rc = a->dtype == BFA_DTYPE_F32 ? tree_simt(p, st) : tree_mma(p, (int)a->dtype, st);
  if (rc) return rc;
  switch (a->dtype) {
    case BFA_DTYPE_F32: return launch_merge<float>(p, st);
    case BFA_DTYPE_F16: return launch_merge<__half>(p, st);
    default: return launch_merge<__nv_bfloat16>(p, st);
  }
}
