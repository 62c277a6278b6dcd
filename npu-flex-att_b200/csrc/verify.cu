// verify.cu -- verification of a tree of drafted tokens against the target's
// probabilities, and the draw of the next token, in one launch.
//
// Mathematics. At a node with target law p and draft law q, children are
// independent draws from q, tested in order. The residual after c rejections
// is r_c = norm(max(r_{c-1} - q, 0)), r_0 = p. Written out,
//   r_c ∝ max(p - a_c·q, 0),  a_0 = 0, W_0 = 1,
//   a_{c+1} = a_c + W_c,  W_c = sum_v max(p(v) - a_c·q(v), 0),
// so a rejection needs one scalar pair and one sum over the vocabulary, and no
// residual is ever stored: child x is accepted when
//   u·W_c·q(x) < max(p(x) - a_c·q(x), 0).
// Without q (candidates that are no draws) r_c is p without the rejected
// tokens, and its mass 1 - sum of their p. The next token is
// argmax_v r(v)/e(v) with e ~ Exp(1): the minimum of independent exponentials
// e(v)/r(v) falls on v with probability r(v)/sum r, so the residual needs no
// normalising sum and the draw no prefix sum whose rounding would decide it.
//
// Bound: latency of the walk for few sequences, HBM for many: the final node's
// p and q rows and the noise row (V·(2e + 4) bytes a sequence), and once more
// the p and q rows of a node for each rejection that has a sibling left (from
// L2 after the first).
//
// Split. One cluster of 1 to 8 blocks per sequence, the vocabulary cut between
// them; every block gathers the N nodes' p(x) and q(x) at once and then walks
// the tree in shared memory, all blocks alike. Sums and maxima cross the
// cluster through distributed shared memory in a fixed order, so every block
// takes the same decisions and results do not depend on scheduling.
// Measured: one sequence, five nodes, 32768 entries 5.5 us, nearly all latency
// (gather, walk, one pass); 64 sequences of 15 nodes, 131072 entries in fp32
// 30 us for the 119 MB that the accepted paths read (59% of the copy rate:
// sequences end their walks at different times and leave SMs idle).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "bfa_internal.h"

namespace bfa {
namespace {

constexpr int kMaxNodes = 64;
constexpr int kVerifyThreads = 512;
constexpr int kVerifyPerSm = 2;  // resident blocks per SM: 64 registers a thread
constexpr int kMaxCluster = 8;
constexpr int kVerifyStep = 16 * kVerifyThreads;  // the most entries that a thread's loop counter moves by

struct VerifyParams {
  const void* target; const void* draft;
  int64_t st[2], sd[2];
  const void* tokens; int64_t tokens_stride; int token_bytes;
  const int32_t* parents; int64_t parents_stride;
  const float* uniforms; int64_t uniforms_stride;
  const float* noise; int64_t noise_stride;
  int32_t* path; int32_t* count; int32_t* next; int32_t* status;
  int N, V, slice;  // slice: vocabulary entries per block, a multiple of 8
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Store to the same shared variable of block `rank` of the cluster.
__device__ __forceinline__ void store_remote(uint64_t* p, uint32_t rank, uint64_t v) {
  const uint32_t local = (uint32_t)__cvta_generic_to_shared(p);
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(v) : "memory");
}

struct Shared {
  uint64_t slot[2][kMaxCluster];  // the cluster's partial results, two rounds
  uint64_t warp[kVerifyThreads / 32];
  float px[kMaxNodes], qx[kMaxNodes], u[kMaxNodes];
  int32_t parent[kMaxNodes], token[kMaxNodes];
  int32_t gone[kMaxNodes];        // rejected tokens (no draft law), a slot of its own for each rejection
};

// Combines one value per thread over the block and the cluster: `add` fp32
// sums (low word) in a fixed order, else the largest 64-bit key.
template <bool add>
__device__ __forceinline__ uint64_t combine(Shared& sh, uint64_t x, int round) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto join = [](uint64_t a, uint64_t b) -> uint64_t {
    if constexpr (add)
      return __float_as_uint(__uint_as_float((uint32_t)a) + __uint_as_float((uint32_t)b));
    else
      return a > b ? a : b;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = join(x, __shfl_xor_sync(0xffffffffu, x, o));
  if (lane == 0) sh.warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    x = lane < kVerifyThreads / 32 ? sh.warp[lane] : 0;
#pragma unroll
    for (int o = kVerifyThreads / 64; o > 0; o >>= 1) x = join(x, __shfl_xor_sync(0xffffffffu, x, o));
    const uint32_t n = cluster_size();
    x = __shfl_sync(0xffffffffu, x, 0);
    if (lane < n) store_remote(&sh.slot[round & 1][cluster_rank()], lane, x);
  }
  cluster_sync();  // also the block's own barrier
  const uint32_t n = cluster_size();
  x = sh.slot[round & 1][0];
  for (uint32_t i = 1; i < n; ++i) x = join(x, sh.slot[round & 1][i]);
  return x;
}

template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T x[V];
};
// Entries p[0, V) as they are stored (converted where they are used: fewer
// registers in flight).
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  Vec<T, V> t;
  if constexpr (V == 1) {
    t.x[0] = *p;
  } else {
    constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < V / kPer; ++i) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(p) + i);
      const Vec<T, kPer> u = *reinterpret_cast<const Vec<T, kPer>*>(&w);
#pragma unroll
      for (int j = 0; j < kPer; ++j) t.x[i * kPer + j] = u.x[j];
    }
  }
  return t;
}

// Entries per access: 16 bytes of T where every row allows it, else one.
template <typename T, int E>
__global__ void __launch_bounds__(kVerifyThreads, kVerifyPerSm) verify_kernel(const VerifyParams p) {
  // Accesses of a thread in flight together. One entry per access: those past
  // the slice's end are predicated off, since a loop that only unrolls leaves
  // its last, partial round to loads one after another (16 sequences of 50021
  // entries in bf16 12.7 -> 10.7 us). Vectors have few rounds, and predicated
  // ones were slower (64 sequences of 131072 30 -> 34 us): unrolled.
  constexpr int kSumBatch = E == 1 ? 16 : 1, kDrawBatch = E == 1 ? 8 : 1;
  constexpr int kSumUnroll = E == 1 ? 1 : 4, kDrawUnroll = E == 1 ? 1 : 2;
  constexpr int kStep = kVerifyThreads * E;
  static_assert(kStep * kSumBatch <= kVerifyStep && kStep * kDrawBatch <= kVerifyStep, "bound of the vocabulary");
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const uint32_t rank = cluster_rank();
  const int b = blockIdx.x / cluster_size();
  const int lo = (int)min((int64_t)rank * p.slice, (int64_t)p.V), hi = (int)min((int64_t)lo + p.slice, (int64_t)p.V);
  const T* target = static_cast<const T*>(p.target) + b * p.st[0];
  const T* draft = p.draft ? static_cast<const T*>(p.draft) + b * p.sd[0] : nullptr;
  const float* noise = p.noise + b * p.noise_stride;

  // The noise row is needed however the walk goes: on its way to L2 meanwhile.
  if (E > 1 && tid == 0 && hi > lo)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(noise + lo), "r"((uint32_t)(hi - lo) * 4u) : "memory");
  if (tid < p.N) {
    int32_t up = tid == 0 ? -1 : p.parents ? p.parents[b * p.parents_stride + tid] : tid - 1;
    const int64_t at = b * p.tokens_stride + tid;
    const int64_t x = p.token_bytes == 8 ? static_cast<const int64_t*>(p.tokens)[at] : (int64_t) static_cast<const int32_t*>(p.tokens)[at];
    const float u = p.uniforms[b * p.uniforms_stride + tid];
    float px = 0.f, qx = 0.f;
    if (tid > 0 && (up < -1 || up >= tid)) {
      up = -1;
      if (p.status) *p.status = BFA_ERR_INDEX;
    }
    if (up >= 0) {
      if (x >= 0 && x < p.V) {
        px = to_f32<T>(target[up * p.st[1] + x]);
        if (draft) qx = to_f32<T>(draft[up * p.sd[1] + x]);
      } else {
        up = -1;  // never a candidate
        if (p.status) *p.status = BFA_ERR_INDEX;
      }
    }
    sh.parent[tid] = up;
    sh.token[tid] = (int32_t)x;
    sh.px[tid] = px;
    sh.qx[tid] = qx;
    sh.u[tid] = u;
  }
  __syncthreads();
  if (cluster_size() > 1) cluster_sync();  // every block is there before a remote store

  int cur = 0, n_path = 1, round = 0;
  int gone0 = 0, gone1 = 0;  // sh.gone[gone0, gone1): the current node's
  float a = 0.f, w = 1.f, removed = 0.f;
  bool stale = false;  // w has to be summed before the next test
  int32_t* path = p.path + (int64_t)b * p.N;
  const bool writer = rank == 0 && tid == 0;
  if (writer) path[0] = 0;

  for (int n = 1; n < p.N; ++n) {
    if (sh.parent[n] != cur) continue;
    bool accept;
    if (draft) {
      if (stale) {
        const T* pr = target + cur * p.st[1];
        const T* qr = draft + cur * p.sd[1];
        float sum = 0.f;
#pragma unroll kSumUnroll
        for (int v0 = lo + tid * E; v0 < hi; v0 += kStep * kSumBatch) {
          Vec<T, E> pv[kSumBatch], qv[kSumBatch];
#pragma unroll
          for (int j = 0; j < kSumBatch; ++j)
            if (v0 + j * kStep < hi) {
              pv[j] = load_vec<T, E>(pr + v0 + j * kStep);
              qv[j] = load_vec<T, E>(qr + v0 + j * kStep);
            }
#pragma unroll
          for (int j = 0; j < kSumBatch; ++j)
            if (v0 + j * kStep < hi)
#pragma unroll
              for (int i = 0; i < E; ++i) sum += fmaxf(to_f32<T>(pv[j].x[i]) - a * to_f32<T>(qv[j].x[i]), 0.f);
        }
        w = __uint_as_float((uint32_t)combine<true>(sh, __float_as_uint(sum), round++));
        stale = false;
      }
      accept = sh.u[n] * (w * sh.qx[n]) < fmaxf(sh.px[n] - a * sh.qx[n], 0.f);
      if (!accept) {
        a += w;
        stale = true;
      }
    } else {
      bool again = false;
      for (int i = gone0; i < gone1; ++i) again |= sh.gone[i] == sh.token[n];
      accept = !again && sh.u[n] * (1.f - removed) < sh.px[n];
      if (!accept && !again) {
        removed += sh.px[n];
        // Every thread writes every slot, all with the same value, and reads
        // back only what it has written; no slot is used twice.
        sh.gone[gone1++] = sh.token[n];
      }
    }
    if (accept) {
      cur = n;
      a = removed = 0.f;
      w = 1.f;
      stale = false;
      gone0 = gone1;
      if (writer) path[n_path] = n;
      ++n_path;
    }
  }
  __syncthreads();

  const T* pr = target + cur * p.st[1];
  const T* qr = draft ? draft + cur * p.sd[1] : nullptr;
  uint64_t best = 0;
  for (int pass = 0; pass < 2; ++pass) {  // the second: an empty residual
    const bool use_q = pass == 0 && a > 0.f;
    const int use_gone = pass == 0 ? gone1 : gone0;
    float top = -1.f;
    int at = lo;
#pragma unroll kDrawUnroll
    for (int v0 = lo + tid * E; v0 < hi; v0 += kStep * kDrawBatch) {
      Vec<T, E> pv[kDrawBatch], qv[kDrawBatch];
      Vec<float, E> ev[kDrawBatch];
#pragma unroll
      for (int j = 0; j < kDrawBatch; ++j)
        if (v0 + j * kStep < hi) {
          pv[j] = load_vec<T, E>(pr + v0 + j * kStep);
          ev[j] = load_vec<float, E>(noise + v0 + j * kStep);
          if (use_q) qv[j] = load_vec<T, E>(qr + v0 + j * kStep);
        }
#pragma unroll
      for (int j = 0; j < kDrawBatch; ++j) {
        if (v0 + j * kStep >= hi) break;
        float r[E], most = -1.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float x = to_f32<T>(pv[j].x[i]);
          if (use_q) x -= a * to_f32<T>(qv[j].x[i]);
          r[i] = x > 0.f ? x / ev[j].x[i] : 0.f;
          r[i] = r[i] >= 0.f ? r[i] : 0.f;
          most = fmaxf(most, r[i]);
        }
        if (most > top) {  // a few times per thread: only here the rejected tokens matter
#pragma unroll
          for (int i = 0; i < E; ++i) {
            bool out = !(r[i] > top);
            for (int g = gone0; g < use_gone && !out; ++g) out = sh.gone[g] == v0 + j * kStep + i;
            if (!out) {
              top = r[i];
              at = v0 + j * kStep + i;
            }
          }
        }
      }
    }
    // Larger values first, then lower indices (values are >= 0 here, or the
    // thread had no entry).
    const uint64_t key = top < 0.f ? 0 : ((uint64_t)__float_as_uint(top) << 32) | (uint32_t)~(uint32_t)at;
    best = combine<false>(sh, key, round++);
    if ((best >> 32) != 0) break;
  }
  if (writer) {
    p.next[b] = best ? (int32_t) ~(uint32_t)best : 0;
    p.count[b] = n_path;
  }
  if (rank == 0)
    for (int i = n_path + tid; i < p.N; i += kVerifyThreads) path[i] = -1;
}

template <typename T, int E>
int launch_verify(VerifyParams& p, int B, cudaStream_t st) {
  // The largest cluster whose blocks are all resident at once and keep at
  // least 2048 entries each.
  int cluster = 1;
  while (cluster < kMaxCluster && (int64_t)B * cluster * 2 <= (int64_t)sm_count() * kVerifyPerSm && p.V / (cluster * 2) >= 2048) cluster *= 2;
  p.slice = ((p.V + cluster - 1) / cluster + 7) / 8 * 8;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)B * cluster);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T, E>, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_fail("verify kernel launch", e);
  }
  note_launch();
  return BFA_OK;
}

template <typename T>
int launch_typed(VerifyParams& p, int B, cudaStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  auto rows = [&](const void* d, const int64_t* s) {
    return ((uintptr_t)d & 15u) == 0 && s[0] % E == 0 && s[1] % E == 0;
  };
  const bool vec = p.V % E == 0 && rows(p.target, p.st) && (!p.draft || rows(p.draft, p.sd)) &&
                   ((uintptr_t)p.noise & 15u) == 0 && p.noise_stride % 4 == 0;
  return vec ? launch_verify<T, E>(p, B, st) : launch_verify<T, 1>(p, B, st);
}

}  // namespace
}  // namespace bfa

extern "C" int bfa_verify_tree(const bfa_verify_args* a, void* stream) {
  using namespace bfa;
  if (!a || a->batch < 0 || a->nodes < 1 || a->vocab < 1) return BFA_ERR_INVALID_ARGUMENT;
  if (a->nodes > kMaxNodes || a->vocab > INT32_MAX - kVerifyStep || a->batch > INT32_MAX / kMaxCluster ||
      a->dtype != (int)a->dtype || dtype_bytes((int)a->dtype) == 0)
    return BFA_ERR_UNSUPPORTED;
  if (a->batch == 0) return BFA_OK;
  if (!a->target || !a->tokens || !a->uniforms || !a->noise || !a->path || !a->count || !a->next_token ||
      (a->tokens_bytes != 4 && a->tokens_bytes != 8))
    return BFA_ERR_INVALID_ARGUMENT;
  VerifyParams p{};
  p.target = a->target; p.draft = a->draft;
  for (int i = 0; i < 2; ++i) {
    p.st[i] = a->target_stride[i];
    p.sd[i] = a->draft_stride[i];
  }
  p.tokens = a->tokens; p.tokens_stride = a->tokens_stride; p.token_bytes = (int)a->tokens_bytes;
  p.parents = a->parents; p.parents_stride = a->parents_stride;
  p.uniforms = a->uniforms; p.uniforms_stride = a->uniforms_stride;
  p.noise = a->noise; p.noise_stride = a->noise_stride;
  p.path = a->path; p.count = a->count; p.next = a->next_token; p.status = a->status;
  p.N = (int)a->nodes; p.V = (int)a->vocab;
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case BFA_DTYPE_F32: return launch_typed<float>(p, (int)a->batch, st);
    case BFA_DTYPE_F16: return launch_typed<__half>(p, (int)a->batch, st);
    default: return launch_typed<__nv_bfloat16>(p, (int)a->batch, st);
  }
}
