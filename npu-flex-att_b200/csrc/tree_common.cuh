// tree_common.cuh -- what the tree-attention kernels share: parameters, the
// split of the work, the walk over chunks of keys and the tree's ancestor sets.
//
// A work item is (sequence b, KV head, row block): the rows r = g·N + n of the
// KV head's G query heads and N nodes, in blocks of `rb` rows. Its keys are the
// visible cached tokens in chunks of `chunk`, then one chunk with the tree's
// own N <= 64 keys (`tree_chunks` chunks where chunk < 64). The chunks of all items, in
// order, form one list; each block (at most `grid`, at least a chunk each) takes an equal stretch of it, so
// sequences of any mix of lengths load the GPU evenly and a single long one
// spreads over all of it. Where a stretch ends inside an item, the block
// leaves a partial (O, LSE) in the workspace and tree_merge_kernel joins an
// item's partials in the order of its keys: results do not depend on
// scheduling.
#pragma once

#include "bfa_internal.h"

namespace bfa {

constexpr int kTreeNodes = 64;

struct TreeParams {
  const void* q; const void* k; const void* v; void* o;
  float* lse;  // may be null
  const void* kp; const void* vp;
  int64_t sq[4], sk[4], sv[4], so[4], skp[4], svp[4];
  const int32_t* table; int64_t table_stride;
  const int32_t* lens;
  const int32_t* parents; int64_t parents_stride;
  const float* alibi;
  int32_t* status;
  int64_t num_pages;
  int B, Hq, Hkv, G, N, D, page, cap_tokens;  // cap_tokens: max_pages·page_size
  int page_log2;  // -1: no power of two
  int window;
  float scale, soft_cap;
  int grid, rb, n_rb, chunk, chunk_log2, tree_chunks;
  bool small;  // grid times the number of chunks fits 32 bits (a bound of the host's)
  float* part_o;    // [grid][2][rb][D]: slot 0 an item begun by an earlier block, slot 1 one left to a later
  float* part_lse;  // [grid][2][rb], base 2, without the ALiBi row constant
};

__device__ __forceinline__ int tree_len(const TreeParams& p, int b) {
  return min(max(p.lens[b], 0), p.cap_tokens);
}
// First cached token that is read: with a window the root, at position len,
// sees keys j >= len - W (deeper nodes see less), rounded down to a whole
// chunk, so that chunks start at multiples of their length.
__device__ __forceinline__ int tree_lo(const TreeParams& p, int len) {
  return p.window > 0 ? max(0, len - p.window) >> p.chunk_log2 << p.chunk_log2 : 0;
}
__device__ __forceinline__ int tree_chunks_of(const TreeParams& p, int len) {
  return ((len - tree_lo(p, len) + p.chunk - 1) >> p.chunk_log2) + p.tree_chunks;
}

// Counts of chunks: 32 bits (p.small) or 64.
// Of `grid` blocks, those that have work: every one of them at least a chunk.
template <typename I>
__device__ __forceinline__ I tree_blocks(const TreeParams& p, I T) {
  return T < (I)p.grid ? T : (I)p.grid;
}
// Where block i's stretch of T chunks begins, and which block holds chunk x.
template <typename I>
__device__ __forceinline__ I tree_start(I T, I blocks, I i) {
  return i * T / blocks;
}
template <typename I>
__device__ __forceinline__ int tree_owner(I T, I blocks, I x) {
  return (int)(((x + 1) * blocks - 1) / T);
}

// A position in the list of chunks.
struct TreeCursor {
  int b, item, c;  // sequence, KV head·n_rb + row block, chunk of the item
  int len, lo, n;  // of the sequence: cached tokens, first visible one, chunks of an item
  __device__ __forceinline__ void load(const TreeParams& p) {
    if (b < p.B) {
      len = tree_len(p, b);
      lo = tree_lo(p, len);
      n = tree_chunks_of(p, len);
    }
  }
  // On by k chunks of the same item (k >= 1; past its end: to the next item).
  __device__ __forceinline__ void next(const TreeParams& p, int k = 1) {
    c += k;
    if (c < n) return;
    c = 0;
    if (++item < p.Hkv * p.n_rb) return;
    item = 0;
    ++b;
    load(p);
  }
  __device__ __forceinline__ bool in_tree(const TreeParams& p) const { return c >= n - p.tree_chunks; }
  // First key of the chunk: a cached token, or a node of the tree.
  __device__ __forceinline__ int key0(const TreeParams& p) const {
    return in_tree(p) ? (c - (n - p.tree_chunks)) * p.chunk : lo + c * p.chunk;
  }
};

// Chunks of all sequences' items, and of those before sequence b; every lane
// of a warp calls it.
template <typename I>
__device__ __forceinline__ I tree_total(const TreeParams& p, int b, I* before) {
  I n = 0, m = 0;
  for (int i = threadIdx.x & 31; i < p.B; i += 32) {
    const int c = tree_chunks_of(p, tree_len(p, i));
    n += c;
    if (i < b) m += c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    n += __shfl_xor_sync(0xffffffffu, n, o);
    m += __shfl_xor_sync(0xffffffffu, m, o);
  }
  const I per = p.Hkv * p.n_rb;
  *before = m * per;
  return n * per;
}

template <typename I>
__device__ __forceinline__ int tree_stretch_in(const TreeParams& p, TreeCursor& cur) {
  const int lane = threadIdx.x & 31;
  const I per = p.Hkv * p.n_rb;
  I T = 0, before = 0, x = 0, end = 0;
  for (int pass = p.B > 32 ? 0 : 1; pass < 2; ++pass) {
    // Pass 0 (more than 32 sequences): the total. Pass 1: 32 sequences at a
    // time, a prefix sum over the warp finds the sequence of chunk x.
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int len = b0 + lane < p.B ? tree_len(p, b0 + lane) : 0;
      const I mine = b0 + lane < p.B ? (I)tree_chunks_of(p, len) * per : 0;
      I sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const I y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const I all = __shfl_sync(0xffffffffu, sum, 31);
      if (pass == 0) {
        T += all;
        continue;
      }
      if (b0 == 0) {
        if (p.B <= 32) T = all;
        const I blocks = tree_blocks<I>(p, T);
        if ((I)blockIdx.x >= blocks) return 0;
        x = tree_start<I>(T, blocks, blockIdx.x);
        end = tree_start<I>(T, blocks, blockIdx.x + 1);
      }
      const unsigned m = __ballot_sync(0xffffffffu, before + sum > x);
      if (m) {
        const int l = __ffs(m) - 1;
        cur.b = b0 + l;
        cur.len = __shfl_sync(0xffffffffu, len, l);
        before += __shfl_sync(0xffffffffu, sum - mine, l);
        break;
      }
      before += all;
    }
  }
  cur.lo = tree_lo(p, cur.len);
  cur.n = tree_chunks_of(p, cur.len);
  const int in = (int)(x - before);  // within one sequence: fits 32 bits (checked by the host)
  cur.item = in / cur.n;
  cur.c = in - cur.item * cur.n;
  return (int)(end - x);
}

// This block's stretch: `cur` at its first chunk, returns its number of chunks
// (0: none). Every lane of a warp calls it; one pass over the lengths where a
// lane each holds them.
__device__ __forceinline__ int tree_stretch(const TreeParams& p, TreeCursor& cur) {
  return p.small ? tree_stretch_in<uint32_t>(p, cur) : tree_stretch_in<int64_t>(p, cur);
}

// The rows of K and V that key j of a chunk lies in (null reads as zeros: past
// the keys, and before a window, where pages may have been given back).
// Reports a bad page. Rows of absent nodes are read like the others: their
// logits are masked, and the kernels keep values that a row does not see out
// of its sum even where they are not finite.
template <int kBytes>
__device__ __forceinline__ void tree_key_rows(const TreeParams& p, const TreeCursor& cur, int j, const char** kr, const char** vr) {
  *kr = *vr = nullptr;
  const int hkv = cur.item / p.n_rb;
  const int key = cur.key0(p) + j;
  if (cur.in_tree(p)) {
    if (key >= p.N) return;
    *kr = static_cast<const char*>(p.k) + (cur.b * p.sk[0] + hkv * p.sk[1] + key * p.sk[2]) * kBytes;
    *vr = static_cast<const char*>(p.v) + (cur.b * p.sv[0] + hkv * p.sv[1] + key * p.sv[2]) * kBytes;
    return;
  }
  if (key >= cur.len || (p.window > 0 && key < cur.len - p.window)) return;
  const int pg = p.page_log2 >= 0 ? key >> p.page_log2 : key / p.page, slot = key - pg * p.page;
  const int32_t page = p.table[cur.b * p.table_stride + pg];
  if (page < 0 || page >= p.num_pages) {
    if (p.status) *p.status = BFA_ERR_INDEX;
    return;
  }
  *kr = static_cast<const char*>(p.kp) + (page * p.skp[0] + hkv * p.skp[1] + slot * p.skp[2]) * kBytes;
  *vr = static_cast<const char*>(p.vp) + (page * p.svp[0] + hkv * p.svp[1] + slot * p.svp[2]) * kBytes;
}

// Ancestor sets of sequence b's nodes (bit m of anc[n]: m is n or above it; 0
// for an absent node) and their depths, by one warp: every round doubles the
// climbed distance.
struct TreeMasks {
  uint64_t anc[kTreeNodes];
  int32_t depth[kTreeNodes];
  int32_t up[kTreeNodes];
};
__device__ __forceinline__ void tree_masks(const TreeParams& p, int b, TreeMasks& m) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = lane + 32 * h;
    int up = -1;
    if (n < p.N && n > 0) {
      up = p.parents ? p.parents[b * p.parents_stride + n] : n - 1;
      if (up < -1 || up >= n) {
        up = -1;
        if (p.status) *p.status = BFA_ERR_INDEX;
      }
    }
    m.up[n] = up;
    m.anc[n] = n < p.N ? 1ull << n : 0ull;
  }
  __syncwarp();
#pragma unroll 1
  for (int r = 0; r < 6; ++r) {  // 2^6 >= the deepest climb
    uint64_t a[2];
    int u[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = lane + 32 * h;
      a[h] = m.anc[n];
      u[h] = m.up[n];
      if (u[h] >= 0) {
        a[h] |= m.anc[u[h]];
        u[h] = m.up[u[h]];
      }
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m.anc[lane + 32 * h] = a[h];
      m.up[lane + 32 * h] = u[h];
    }
    __syncwarp();
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = lane + 32 * h;
    if (!(m.anc[n] & 1)) m.anc[n] = 0;  // does not hang under the root
    m.depth[n] = max(0, __popcll(m.anc[n]) - 1);
  }
  __syncwarp();
}

// The ALiBi bias of pair (i, j) is slope·(i - j). For slope > 0 the kernels
// form it as slope·(g0 - j), g0 the first key the row can see, so that the
// logits that carry the softmax stay small, and add slope·(i - g0) to the LSE
// alone; for slope <= 0 it is largest at the row itself and g0 = i.
__device__ __forceinline__ int tree_alibi_ref(const TreeParams& p, float slope, int i) {
  if (!(slope > 0.f)) return i;
  return p.window > 0 ? max(0, i - p.window) : 0;
}

// cap·tanh(s/cap), by tanh x = 1 - 2/(1 + e^2x): absolute error near 1e-7·cap.
__device__ __forceinline__ float tree_cap(float s, float cap, float inv_cap) {
  return cap * (1.f - 2.f / (1.f + __expf(2.f * s * inv_cap)));
}

// Final O / LSE row address of row r of item (b, hkv).
__device__ __forceinline__ void tree_row(const TreeParams& p, int hkv, int r, int* hq, int* n) {
  const int g = r / p.N;
  *hq = hkv * p.G + g;
  *n = r - g * p.N;
}
__device__ __forceinline__ float tree_row_shift(const TreeParams& p, int hq, int pos) {
  if (!p.alibi) return 0.f;
  const float slope = p.alibi[hq];
  return slope * (float)(pos - tree_alibi_ref(p, slope, pos));
}

// How a kernel cuts a problem: rows per block, keys per chunk, resident blocks
// per SM.
struct TreeTile {
  int rb, chunk, per_sm;
};

// tree_simt.cu: CUDA cores, the fp32 path.
int tree_simt(const TreeParams& p, cudaStream_t st);
constexpr int kTreeSimtRows = 32, kTreeSimtChunk = 32;

// tree_mma.cu: bf16 / fp16 on mma.sync.
TreeTile tree_mma_tile(int64_t rows, int D);
int tree_mma(const TreeParams& p, int dtype, cudaStream_t st);

// tree_sm100.cu: bf16 / fp16 on tcgen05, pages by TMA.
TreeTile tree_sm100_tile(int64_t rows, int D, bool cap);
// Whether its layouts allow it (the sizes are the caller's rule).
bool tree_sm100_layout(const bfa_tree_args* a);
int tree_sm100(const TreeParams& p, int dtype, cudaStream_t st);

}  // namespace bfa
