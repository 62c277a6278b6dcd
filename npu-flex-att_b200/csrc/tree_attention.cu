// tree_attention.cu -- the entry points of tree attention: checks, the choice
// of kernel and grid, the workspace and the merge of partial results.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdlib>

#include "tree_common.cuh"

namespace bfa {
namespace {


// Joins the partial (O, LSE) of items that several blocks worked on, partials
// in the order of their keys:
//   lse = log2 sum_i 2^lse_i,  O = sum_i O_i·2^(lse_i - lse).
// An item that one block did whole is already final, and its merge blocks
// leave at once. A block has kMergeRows rows of an item, kWarps warps take a row: each sums every kWarps-th partial,
// eight loads in flight, and the first adds the warps' sums in order. One warp
// where an item has few partials (many items), four where a few items are
// spread over the GPU. kVec: columns per lane and load (4 where D allows it,
// else 1). Launched to start under the attention kernel's tail: what it needs
// of the inputs alone comes before it waits for the partials.
template <typename T, int kWarps, int kVec, int kMergeRows>
__global__ void __launch_bounds__(128, 7) tree_merge_kernel(const TreeParams p) {
  constexpr int kLoads = kVec == 4 ? 2 : 8;  // of 32·kVec columns: 256
  __shared__ float part[4][kVec * kLoads * 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % kWarps;
  const int GN = p.G * p.N;
  const int per_item = (min(p.rb, GN) + kMergeRows - 1) / kMergeRows;
  const int item_all = blockIdx.x / per_item, row0 = (blockIdx.x - item_all * per_item) * kMergeRows;
  const int b = item_all / (p.Hkv * p.n_rb), item = item_all - b * p.Hkv * p.n_rb;
  const int hkv = item / p.n_rb, rb0 = (item - hkv * p.n_rb) * p.rb;
  const int len = tree_len(p, b), n_chunks = tree_chunks_of(p, len);
  int i0, i1;
  auto owners = [&](auto zero) {
    using I = decltype(zero);
    I s0;
    const I T_all = tree_total<I>(p, b, &s0);
    s0 += (I)item * n_chunks;
    const I blocks = tree_blocks<I>(p, T_all);
    i0 = tree_owner<I>(T_all, blocks, s0);
    i1 = tree_owner<I>(T_all, blocks, s0 + n_chunks - 1);
  };
  if (p.small) owners(uint32_t{0});
  else owners(int64_t{0});
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (i0 == i1) return;
  for (int rr = warp / kWarps; rr < kMergeRows; rr += 4 / kWarps) {
    const int r = row0 + rr;
    if (r >= p.rb || rb0 + r >= GN) break;  // alike for the warps of a row
    auto slot = [&](int i) { return ((int64_t)i * 2 + (i == i0 ? 1 : 0)) * p.rb + r; };
    // kBatch partial results in flight, those past the last predicated off (an
    // item mostly has two to six; a loop that only unrolls would take them one
    // after another: one token over 4095 14.4 -> 13.1 us), the first ones beside
    // the LSEs.
    constexpr int kBatch = kWarps > 1 ? 4 : 2;
    float f[kBatch][kLoads][kVec];
    auto fetch = [&](int j0, int j, int n) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k, j += kWarps)
#pragma unroll
        for (int c = 0; c < kLoads; ++c) {
          const int d = (lane + 32 * c) * kVec;
          if (j >= n || d >= p.D) continue;
          const float* po = p.part_o + slot(j0 + j) * p.D + d;
          if constexpr (kVec == 4) *reinterpret_cast<float4*>(f[k][c]) = *reinterpret_cast<const float4*>(po);
          else f[k][c][0] = *po;
        }
    };
    fetch(i0, sub, min(32, i1 - i0 + 1));
    float m = neg_inf();
    bool nan = false;
    for (int i = i0 + lane; i <= i1; i += 32) {
      const float x = p.part_lse[slot(i)];
      nan |= x != x;
      m = fmaxf(m, x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // A NaN among them, which the maximum leaves out, makes the sums NaN.
    if (__any_sync(0xffffffffu, nan) && m == neg_inf()) m = 0.f;
    float total = 0.f, acc[kLoads][kVec];
#pragma unroll
    for (int c = 0; c < kLoads; ++c)
#pragma unroll
      for (int e = 0; e < kVec; ++e) acc[c][e] = 0.f;
    if (m != neg_inf()) {
      for (int j0 = i0; j0 <= i1; j0 += 32) {
        const float w = j0 + lane <= i1 ? exp2f(p.part_lse[slot(j0 + lane)] - m) : 0.f;
        float sum = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        total += sum;
        const int n = min(32, i1 - j0 + 1);
        for (int j = sub; j < n; j += kBatch * kWarps) {
          if (j0 > i0 || j > sub) fetch(j0, j, n);
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            if (j + k * kWarps >= n) break;
            const float wj = __shfl_sync(0xffffffffu, w, j + k * kWarps);
#pragma unroll
            for (int c = 0; c < kLoads; ++c) {
              if ((lane + 32 * c) * kVec >= p.D) continue;
#pragma unroll
              for (int e = 0; e < kVec; ++e) acc[c][e] = fmaf(wj, f[k][c][e], acc[c][e]);
            }
          }
        }
      }
    }
    if constexpr (kWarps > 1) {
      __syncthreads();  // the last row's sums have been read
#pragma unroll
      for (int c = 0; c < kLoads; ++c)
#pragma unroll
        for (int e = 0; e < kVec; ++e) part[warp][(c * kVec + e) * 32 + lane] = acc[c][e];
      __syncthreads();
      if (sub != 0) continue;
#pragma unroll
      for (int c = 0; c < kLoads; ++c)
#pragma unroll
        for (int e = 0; e < kVec; ++e)
#pragma unroll
          for (int k = 1; k < kWarps; ++k) acc[c][e] += part[warp + k][(c * kVec + e) * 32 + lane];
    }
    int hq, n;
    tree_row(p, hkv, rb0 + r, &hq, &n);
    T* out = static_cast<T*>(p.o) + b * p.so[0] + hq * p.so[1] + n * p.so[2];
    const float inv = total != 0.f ? 1.f / total : 0.f;  // 0: no part of the row saw anything
#pragma unroll
    for (int c = 0; c < kLoads; ++c)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int d = (lane + 32 * c) * kVec + e;
        if (d < p.D) out[d] = from_f32<T>(acc[c][e] * inv);
      }
    if (lane == 0 && p.lse) {
      float l = neg_inf();
      if (total != 0.f) {
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
}

int check_tree(const bfa_tree_args* a) {
  if (!a || a->batch < 0 || a->heads_q < 0 || a->heads_kv < 1 || a->nodes < 1 || a->num_pages < 0 || a->page_size < 1 ||
      a->max_pages < 0 || a->sliding_window < 0 || !(a->soft_cap >= 0))
    return BFA_ERR_INVALID_ARGUMENT;
  if (a->heads_q % a->heads_kv != 0) return BFA_ERR_SHAPE;
  if (a->head_dim < 1 || a->head_dim > 256 || a->nodes > kTreeNodes || a->dtype != (int)a->dtype ||
      dtype_bytes((int)a->dtype) == 0)
    return BFA_ERR_UNSUPPORTED;
  // Positions, rows per KV head, items, and the chunks of a sequence's items
  // are counted in 32 bits.
  if (a->batch > (1 << 24) || a->heads_q > (1 << 20) || a->page_size > INT32_MAX / 2 ||
      a->max_pages > (INT32_MAX / 2 - 128) / a->page_size || a->batch * a->heads_q > INT32_MAX / kTreeNodes ||
      a->heads_q * ((a->max_pages * a->page_size + 64) / 32 + 4) > INT32_MAX / 4)
    return BFA_ERR_UNSUPPORTED;
  return BFA_OK;
}

// The window in 32 bits. Positions stay below INT32_MAX / 2, so that a window of
// that size, or of any larger one, sees everything.
int window_of(const bfa_tree_args* a) { return (int)std::min<int64_t>(a->sliding_window, INT32_MAX / 2); }

// Row block, chunk and grid of a problem.
struct Plan {
  int rb, n_rb, chunk, tree_chunks, grid;
  size_t lse_at, bytes;
  bool small;
};

Plan make_plan(const bfa_tree_args* a, const TreeTile& tile) {
  Plan pl{};
  const int64_t rows = a->heads_q / a->heads_kv * a->nodes;
  pl.rb = tile.rb;
  pl.chunk = tile.chunk;
  pl.n_rb = (int)((rows + pl.rb - 1) / pl.rb);
  pl.tree_chunks = (int)((a->nodes + pl.chunk - 1) / pl.chunk);
  // At most one stretch per chunk that the tables could hold.
  int64_t seen = a->max_pages * a->page_size;
  if (a->sliding_window > 0) seen = std::min<int64_t>(seen, (int64_t)window_of(a) + pl.chunk);
  const int64_t chunks = ((seen + pl.chunk - 1) / pl.chunk + pl.tree_chunks) * a->batch * a->heads_kv * pl.n_rb;
  pl.grid = (int)std::min<int64_t>(chunks, (int64_t)sm_count() * tile.per_sm);
  pl.small = chunks < ((int64_t)1 << 31) / (pl.grid + 1);
  const size_t rows_ws = (size_t)pl.grid * 2 * pl.rb;
  pl.lse_at = (rows_ws * a->head_dim * 4 + 255) / 256 * 256;
  pl.bytes = pl.lse_at + (rows_ws * 4 + 255) / 256 * 256;
  return pl;
}

TreeTile simt_tile(const bfa_tree_args* a) { return {kTreeSimtRows, kTreeSimtChunk, a->head_dim > 128 ? 1 : 2}; }

bool tcgen05_on() {  // BFA_TREE_TCGEN05=0 keeps bf16/fp16 on the mma.sync kernel
  const char* e = std::getenv("BFA_TREE_TCGEN05");
  return !(e && e[0] == '0');
}

// Workspace for either 16-bit kernel: which one runs depends on the layouts,
// the workspace on the sizes alone.
size_t workspace_bytes(const bfa_tree_args* a) {
  if (a->dtype == BFA_DTYPE_F32) return make_plan(a, simt_tile(a)).bytes;
  const int64_t rows = a->heads_q / a->heads_kv * a->nodes;
  return std::max(make_plan(a, tree_mma_tile(rows, (int)a->head_dim)).bytes,
                  make_plan(a, tree_sm100_tile(rows, (int)a->head_dim, a->soft_cap > 0)).bytes);
}

template <typename T>
int launch_merge(const TreeParams& p, cudaStream_t st) {
  const int64_t items = (int64_t)p.B * p.Hkv * p.n_rb;
  // Four warps per row where an item is spread over at least four blocks on
  // average and all rows' blocks are resident at once (7 per SM; 4096 rows with
  // 5 partial results each 30 us with a warp per row, 37 with four, the
  // attention included, 512 rows 38 against 41); else a warp per row, or four
  // rows a warp where there are so many that the blocks' own start costs more
  // (16384 rows: 1.2 to 2 us less with a warp per row, 32768: alike, 65536: 9 us
  // more).
  const int64_t all = items * std::min(p.rb, p.G * p.N);
  const bool wide = p.grid >= 4 * items && all <= (int64_t)sm_count() * 7;
  const int rows = wide ? 1 : all <= (int64_t)sm_count() * 128 ? 4 : 16;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(items * ((std::min(p.rb, p.G * p.N) + rows - 1) / rows)));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  auto kernel = p.D % 4 == 0
                    ? (wide ? tree_merge_kernel<T, 4, 4, 1> : rows == 4 ? tree_merge_kernel<T, 1, 4, 4> : tree_merge_kernel<T, 1, 4, 16>)
                    : (wide ? tree_merge_kernel<T, 4, 1, 1> : rows == 4 ? tree_merge_kernel<T, 1, 1, 4> : tree_merge_kernel<T, 1, 1, 16>);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_fail("tree merge launch", e);
  }
  note_launch();
  return BFA_OK;
}

}  // namespace
}  // namespace bfa

extern "C" size_t bfa_tree_workspace_bytes(const bfa_tree_args* a) {
  using namespace bfa;
  if (check_tree(a) || a->batch * a->heads_q == 0) return 0;
  return workspace_bytes(a);
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
  if (!a->workspace || a->workspace_bytes < (int64_t)workspace_bytes(a) || ((uintptr_t)a->workspace & 255u) != 0)
    return BFA_ERR_WORKSPACE;
  const int64_t rows = a->heads_q / a->heads_kv * a->nodes;
  const bool f32 = a->dtype == BFA_DTYPE_F32;
  // tcgen05 wherever TMA can read the layouts: it was the faster one at every
  // size tried (B=16, L=8192, 8 KV heads of 128: 4 rows a KV head 90 against
  // 120 us, 64 rows 103 against 175, 256 rows 173 against 551).
  const bool tc = !f32 && tcgen05_on() && tree_sm100_layout(a);
  const Plan pl = make_plan(a, f32  ? simt_tile(a)
                               : tc ? tree_sm100_tile(rows, (int)a->head_dim, a->soft_cap > 0)
                                    : tree_mma_tile(rows, (int)a->head_dim));
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
  p.window = window_of(a);
  p.scale = (float)a->scale;
  p.soft_cap = (float)a->soft_cap;
  p.grid = pl.grid; p.rb = pl.rb; p.n_rb = pl.n_rb; p.chunk = pl.chunk; p.tree_chunks = pl.tree_chunks;
  p.page_log2 = -1;
  for (int i = 0; i < 31; ++i)
    if (p.page == 1 << i) p.page_log2 = i;
  p.chunk_log2 = pl.chunk == 128 ? 7 : pl.chunk == 64 ? 6 : 5;
  p.small = pl.small;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_lse = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + pl.lse_at);
  cudaStream_t st = (cudaStream_t)stream;
  const int rc = f32 ? tree_simt(p, st) : tc ? tree_sm100(p, (int)a->dtype, st) : tree_mma(p, (int)a->dtype, st);
  if (rc) return rc;
  switch (a->dtype) {
    case BFA_DTYPE_F32: return launch_merge<float>(p, st);
    case BFA_DTYPE_F16: return launch_merge<__half>(p, st);
    default: return launch_merge<__nv_bfloat16>(p, st);
  }
}
