// tree_simt.cu -- attention of a tree of drafted tokens over a paged cache on
// the CUDA cores: the fp32 path.
//
// Online softmax in base 2 over chunks of 32 keys for blocks of 32 rows (the
// rows r = g·N + n of one KV head share its keys). Per chunk:
//   S: warp w forms rows 4w..4w+3, lane = key, from fp32 rows in shared memory
//      (5 vector reads for 16 multiply-adds);
//   softmax: in the same registers, row maxima and sums by shuffles;
//   P·V: thread = 2 or 4 columns x 4 or 8 rows, P read as vectors of 4 rows.
// Bound: shared-memory reads and FMA issue from about 8 rows per KV head on,
// HBM below. 13.5 TFLOP/s with 32 rows per KV head (B=4, L=4096, 4 KV heads of
// 128: 78 us, 13% of the HBM floor; 68 us with 4 rows, whose warps are mostly
// idle). The next chunk's rows come by cp.async while a chunk is worked on.
#include <cuda_runtime.h>

#include "tree_common.cuh"

namespace bfa {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = kTreeSimtRows, kKeys = kTreeSimtChunk;
static_assert(kRows == 4 * (kThreads / 32) && kKeys == 32, "warp w owns rows 4w..4w+3, a lane a key");

struct SimtShared {
  TreeMasks masks;
  const char* krow[2][kKeys];
  const char* vrow[2][kKeys];
  alignas(16) float p[kKeys][kRows];  // probabilities, row index innermost
  alignas(16) float alpha[kRows];
};

__device__ __forceinline__ void copy_row_piece(float* dst, const char* src, int d, int D, bool vec) {
  // 4 elements of a row; zeros past D and for a missing row.
  if (vec && src && d < D) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(src + (int64_t)d * 4) : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = (src && d + i < D) ? reinterpret_cast<const float*>(src)[d + i] : 0.f;
}

template <int D>  // head dim rounded up to 64, 128 or 256
__global__ void __launch_bounds__(kThreads) tree_simt_kernel(const TreeParams p, bool vec) {
  constexpr int kPitch = D + 4;  // floats; 16-byte rows shifted against each other
  constexpr int kPieces = D / 4;                    // 16-byte pieces of a row
  constexpr int kC = D == 64 ? 2 : 4;               // columns per thread in P·V
  constexpr int kCols = D / kC;                     // column groups
  constexpr int kRowTeams = kThreads / kCols;       // threads per column group
  constexpr int kQuads = kRows / kRowTeams / 4;     // groups of four rows per thread
  static_assert(kQuads * 4 * kRowTeams == kRows, "rows in fours");
  extern __shared__ __align__(16) uint8_t smem[];
  SimtShared& sh = *reinterpret_cast<SimtShared*>(smem);
  float* qs = reinterpret_cast<float*>(smem + (sizeof(SimtShared) + 15) / 16 * 16);
  float* ks = qs + kRows * kPitch;        // [2][kKeys][kPitch]
  float* vs = ks + 2 * kKeys * kPitch;    // [2][kKeys][kPitch]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  TreeCursor cur;
  const int n_x = tree_stretch(p, cur);
  if (n_x == 0) return;
  TreeCursor ahead = cur;  // the chunk whose rows are looked up next
  int masks_of = -1;

  const float inv_cap = p.soft_cap > 0.f ? 1.f / p.soft_cap : 0.f;
  const int pg = tid % kCols, team = tid / kCols;
  float acc[kQuads][4][kC];  // [quad][row][column]
  float row_m[4], row_l[4];  // rows 4w + i; l is this lane's part of the sum
  float slope[4];
  int pos[4];
  uint64_t anc[4];
  bool fresh = true;  // an item starts (or a stretch that begins inside one)
  int seg_c0 = 0;

  auto lookup = [&](int buf) {  // fills the row addresses of chunk `ahead`
    if (tid < kKeys) {
      const char *kr, *vr;
      tree_key_rows<4>(p, ahead, tid, &kr, &vr);
      sh.krow[buf][tid] = kr;
      sh.vrow[buf][tid] = vr;
    }
    ahead.next(p);
  };
  auto load = [&](int buf) {
    for (int i = tid; i < kKeys * kPieces; i += kThreads) {
      const int n = i / kPieces, d = (i % kPieces) * 4;
      copy_row_piece(ks + (buf * kKeys + n) * kPitch + d, sh.krow[buf][n], d, p.D, vec);
      copy_row_piece(vs + (buf * kKeys + n) * kPitch + d, sh.vrow[buf][n], d, p.D, vec);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  lookup(0);
  __syncthreads();
  load(0);
  if (n_x > 1) lookup(1);

  for (int x = 0; x < n_x; ++x) {
    const int buf = x & 1;
    const int hkv = cur.item / p.n_rb, rb0 = (cur.item - hkv * p.n_rb) * kRows;
    const int R = min(kRows, p.G * p.N - rb0);
    __syncthreads();  // the other buffer's readers and this chunk's addresses are done
    if (x + 1 < n_x) load(buf ^ 1);
    if (fresh) {
      fresh = false;
      seg_c0 = cur.c;
      if (masks_of != cur.b) {
        masks_of = cur.b;
        // A clamped length is an error of the caller's.
        if (tid == 0 && p.status && p.lens[cur.b] != cur.len) *p.status = BFA_ERR_INDEX;
        if (warp == 0) tree_masks(p, cur.b, sh.masks);
      }
      for (int i = tid; i < kRows * D; i += kThreads) {
        const int r = i / D, d = i - r * D;
        float x_ = 0.f;
        if (r < R && d < p.D) {
          int hq, n;
          tree_row(p, hkv, rb0 + r, &hq, &n);
          x_ = static_cast<const float*>(p.q)[cur.b * p.sq[0] + hq * p.sq[1] + n * p.sq[2] + d];
        }
        qs[r * kPitch + d] = x_;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * warp + i;
        int hq = 0, n = 0;
        if (r < R) tree_row(p, hkv, rb0 + r, &hq, &n);
        anc[i] = r < R ? sh.masks.anc[n] : 0ull;
        pos[i] = cur.len + sh.masks.depth[n];
        slope[i] = p.alibi ? p.alibi[hq] : 0.f;
        row_m[i] = neg_inf();
        row_l[i] = 0.f;
      }
#pragma unroll
      for (int a = 0; a < kQuads; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < kC; ++c) acc[a][i][c] = 0.f;
    }
    if (x + 1 < n_x) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (x + 2 < n_x) lookup(buf);  // this chunk's own addresses have been used

    {  // S and softmax: rows 4·warp + i, key = lane
      const float* kr = ks + (buf * kKeys + lane) * kPitch;
      const float* qr = qs + 4 * warp * kPitch;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        const float4 kv = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 qv = *reinterpret_cast<const float4*>(qr + i * kPitch + d);
          s[i] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[i]))));
        }
      }
      const bool tree = cur.in_tree(p);
      const int key = cur.key0(p) + lane;
      const bool exists = tree ? key < p.N : key < cur.len;
      const int kpos = tree ? cur.len + (key < kTreeNodes ? sh.masks.depth[key] : 0) : key;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x_ = s[i] * p.scale;
        if (p.soft_cap > 0.f) x_ = p.soft_cap * tanhf(x_ * inv_cap);
        if (p.alibi) x_ += slope[i] * (float)(tree_alibi_ref(p, slope[i], pos[i]) - kpos);
        bool keep = exists && anc[i] != 0;
        if (tree) keep = keep && ((anc[i] >> (key & 63)) & 1);
        if (p.window > 0) keep = keep && pos[i] - kpos <= p.window;
        x_ = keep ? x_ * kLog2e : neg_inf();
        float mx = x_;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m_new = fmaxf(row_m[i], mx);
        const float m_use = m_new == neg_inf() ? 0.f : m_new;
        const float alpha = exp2f(row_m[i] - m_use);
        const float pr = exp2f(x_ - m_use);
        row_l[i] = row_l[i] * alpha + pr;
        row_m[i] = m_new;
        sh.p[lane][4 * warp + i] = pr;
        if (lane == 0) sh.alpha[4 * warp + i] = alpha;
      }
    }
    __syncthreads();
    {  // P·V: columns 4·pg.., rows (team·kQuads + a)·4 + i
#pragma unroll
      for (int a = 0; a < kQuads; ++a) {
        const float4 al = *reinterpret_cast<const float4*>(&sh.alpha[(team * kQuads + a) * 4]);
        const float f[4] = {al.x, al.y, al.z, al.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < kC; ++c) acc[a][i][c] *= f[i];
      }
      // Whether rows differ in what they see of this chunk: the tree's, and the
      // cached ones that begin before the key from which on every row sees all.
      const bool differ = cur.in_tree(p) || (p.window > 0 && cur.key0(p) < cur.len + p.N - 1 - p.window);
#pragma unroll 4
      for (int n = 0; n < kKeys; ++n) {
        float vx[kC];
        const float* vr = vs + (buf * kKeys + n) * kPitch + pg * kC;
        if constexpr (kC == 4) *reinterpret_cast<float4*>(vx) = *reinterpret_cast<const float4*>(vr);
        else *reinterpret_cast<float2*>(vx) = *reinterpret_cast<const float2*>(vr);
#pragma unroll
        for (int a = 0; a < kQuads; ++a) {
          const float4 p4 = *reinterpret_cast<const float4*>(&sh.p[n][(team * kQuads + a) * 4]);
          const float f[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // A key that a row does not see leaves the row alone even where
            // its values are not finite.
            if (differ && f[i] == 0.f) continue;
#pragma unroll
            for (int c = 0; c < kC; ++c) acc[a][i][c] = fmaf(f[i], vx[c], acc[a][i][c]);
          }
        }
      }
    }
    const TreeCursor done = cur;
    cur.next(p);
    if (cur.c != 0 && x + 1 < n_x) continue;

    // The item, or this block's stretch of it, ends.
    fresh = true;
    const bool whole = seg_c0 == 0 && done.c == done.n - 1;
    __syncthreads();  // sh.p / sh.alpha are free
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float l = row_l[i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (lane == 0) {
        // l = 0: the row saw nothing and is empty. NaN (a logit that it saw was
        // NaN or +inf) goes on into O and LSE.
        sh.alpha[4 * warp + i] = l != 0.f ? 1.f / l : 0.f;
        sh.p[0][4 * warp + i] = l != 0.f ? row_m[i] + log2f(l) : neg_inf();
      }
    }
    __syncthreads();
    const int slot = seg_c0 > 0 ? 0 : 1;
    const int64_t prow = ((int64_t)blockIdx.x * 2 + slot) * p.rb;
#pragma unroll
    for (int a = 0; a < kQuads; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (team * kQuads + a) * 4 + i;
        if (r >= R) continue;
        const float inv = sh.alpha[r], l2 = sh.p[0][r];
        int hq, n;
        tree_row(p, hkv, rb0 + r, &hq, &n);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const int d = pg * kC + c;
          if (d >= p.D) continue;
          const float o = inv != 0.f ? acc[a][i][c] * inv : 0.f;
          if (whole)
            static_cast<float*>(p.o)[done.b * p.so[0] + hq * p.so[1] + n * p.so[2] + d] = o;
          else
            p.part_o[(prow + r) * p.D + d] = o;
        }
        if (pg == 0) {
          if (!whole) p.part_lse[prow + r] = l2;
          else if (p.lse)
            p.lse[((int64_t)done.b * p.Hq + hq) * p.N + n] =
                l2 == neg_inf() ? l2 : l2 * kLn2 + tree_row_shift(p, hq, done.len + sh.masks.depth[n]);
        }
      }
    __syncthreads();
  }
}

template <int D>
int launch(const TreeParams& p, cudaStream_t st) {
  const int bytes = (int)(sizeof(SimtShared) + 15) / 16 * 16 + (kRows + 4 * kKeys) * (D + 4) * 4;
  auto kernel = tree_simt_kernel<D>;
  static std::atomic<uint64_t> done;
  const int rc = allow_shared(kernel, bytes, done, "tree attention shared memory");
  if (rc) return rc;
  auto rows = [](const void* d, const int64_t* s) {
    return ((uintptr_t)d & 15u) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
  };
  const bool vec = p.D % 4 == 0 && rows(p.k, p.sk) && rows(p.v, p.sv) && rows(p.kp, p.skp) && rows(p.vp, p.svp);
  kernel<<<p.grid, kThreads, bytes, st>>>(p, vec);
  note_launch();
  return launch_status("tree attention launch");
}

}  // namespace

int tree_simt(const TreeParams& p, cudaStream_t st) {
  if (p.D <= 64) return launch<64>(p, st);
  if (p.D <= 128) return launch<128>(p, st);
  return launch<256>(p, st);
}

}  // namespace bfa
