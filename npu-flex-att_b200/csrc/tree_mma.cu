// tree_mma.cu -- attention of a tree of drafted tokens over a paged cache in
// bf16 / fp16, both products on mma.sync m16n8k16 (fp32 accumulate): the path
// of layouts that TMA cannot read (page sizes that are no multiple of 8, head
// dims that are none of 8, rows off the 16-byte grid). B=16, L=8192, 8 KV heads
// of 128: 4 rows a KV head 120 us, 256 rows 551 us.
//
// Mathematics: online softmax in base 2 over chunks of 64 keys. Rows r = g·N + n
// of one KV head are stacked, so its K/V cross HBM once per block of rows.
// P is rounded to the input type for P·V, the row sum takes it unrounded.
//
// Bound: HBM (K/V read once) while a KV head has few rows; from about 64 rows
// per KV head the products (mma.sync runs at a fraction of the tcgen05 rate).
//
// Split. A block has RW·KW warps: warp (rw, kw) owns 16 rows and 64/KW of a
// chunk's keys, so few rows still occupy four warps, and keeps its own running
// (m, l, O) in registers, with no exchange between warps until the block's
// stretch of an item ends, when the KW parts are joined through shared memory.
// S is the A operand of P·V as it stands in registers.
//
// Loads: cp.async into a ring of chunks (rows padded by 16 bytes: ldmatrix
// without bank conflicts). The row addresses of a chunk (page table, slot) are
// looked up once per chunk by 64 threads, one iteration before its loads, and
// the ring runs on across items, so a block streams without a gap.
#include <cuda_runtime.h>

#include <type_traits>

#include "tree_common.cuh"

namespace bfa {
namespace {

constexpr int kKeys = 64;  // keys per chunk

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Whether a 16-bit value's exponent is all ones (infinity or NaN).
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t x) {
  constexpr uint32_t e = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return (x & e) == e;
}

// D: head dim rounded up to 64, 128 or 256; the columns past it are zero in
// shared memory.
template <int D, int RW, int KW>
struct Tile {
  static constexpr int kThreads = 32 * RW * KW;
  static constexpr int kRows = 16 * RW;
  static constexpr int kRowBytes = D * 2 + 16;
  static constexpr int kTileBytes = kKeys * kRowBytes;
  // Three chunks in the ring; two at D = 256, where a chunk is 66 KB.
  static constexpr int kStages = D == 256 ? 2 : 3;
  // Registers hold q's fragments up to D = 128; at 256 they come from shared memory.
  static constexpr bool kQShared = D == 256;
  static constexpr int kJoinCols = 32;  // columns joined at a time over the KW parts
  static constexpr int kOffRows = 2 * kStages * kTileBytes;          // krow, vrow [2][64]
  static constexpr int kOffMasks = kOffRows + 2 * 2 * kKeys * 8;
  static constexpr int kOffBad = kOffMasks + (int)sizeof(TreeMasks);  // nodes whose values are not finite
  static constexpr int kOffMl = (kOffBad + 8 + 15) / 16 * 16;        // (m, l) [KW][rows]
  static constexpr int kOffJoin = kOffMl + (KW > 1 ? KW * kRows * 8 : 0);
  static constexpr int kOffQ = kOffJoin + (KW > 1 ? kRows * kJoinCols * 4 : 0);
  static constexpr int kBytes = kOffQ + (kQShared ? kRows * kRowBytes : 0);
  static constexpr int kPerSm = kBytes <= 115200 && kThreads <= 128 ? 2 : 1;
  static_assert(kBytes <= 232448, "shared memory");
};

struct Flags {
  bool vec;   // 16-byte rows of K/V and pages
  bool pair;  // 4-byte accesses of q, o and the partials
};

template <typename T, int D, int RW, int KW, bool PLAIN>
__global__ void __launch_bounds__(32 * RW * KW, (Tile<D, RW, KW>::kPerSm)) tree_mma_kernel(const TreeParams p, const Flags fl) {
  using L = Tile<D, RW, KW>;
  constexpr int kThreads = L::kThreads;
  constexpr int kMine = kKeys / KW;  // keys of a warp per chunk
  constexpr int NT = kMine / 8;      // its 8-key tiles
  constexpr int DT = D / 8;          // 8-column tiles of O
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t sbase = (uint32_t)__cvta_generic_to_shared(smem);
  const char** krow = reinterpret_cast<const char**>(smem + L::kOffRows);
  const char** vrow = krow + 2 * kKeys;
  TreeMasks& masks = *reinterpret_cast<TreeMasks*>(smem + L::kOffMasks);
  unsigned long long* bad = reinterpret_cast<unsigned long long*>(smem + L::kOffBad);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rw = warp % RW, kw = warp / RW;
  const int g = lane >> 2, t = lane & 3;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  TreeCursor cur;
  const int n_x = tree_stretch(p, cur);
  if (n_x == 0) return;
  TreeCursor ahead = cur;  // the next chunk to look up

  // Columns past the head dim are never loaded.
  if (p.D < D) {
    const int pad0 = p.D / 8 * 8;
    for (int i = tid; i < 2 * L::kStages * kKeys * (D - pad0); i += kThreads) {
      const int r = i / (D - pad0), c = pad0 + i % (D - pad0);
      *reinterpret_cast<uint16_t*>(smem + r * L::kRowBytes + c * 2) = 0;
    }
  }

  auto lookup = [&](int buf) {
    if (tid < kKeys) {
      const char *kr, *vr;
      tree_key_rows<2>(p, ahead, tid, &kr, &vr);
      krow[buf * kKeys + tid] = kr;
      vrow[buf * kKeys + tid] = vr;
    }
    ahead.next(p);
  };
  constexpr int kPieces = D / 8;
  constexpr int kRowsPerPass = kThreads / kPieces;
  static_assert(kThreads % kPieces == 0 && kKeys % kRowsPerPass == 0, "piece map");
  auto load = [&](int buf, int stage) {
    if (fl.vec) {
      const int n0 = tid / kPieces, pc = tid % kPieces;
      if (pc * 8 < p.D) {
        const uint32_t dst = sbase + (uint32_t)(2 * stage * L::kTileBytes + n0 * L::kRowBytes + pc * 16);
#pragma unroll
        for (int i = 0; i < kKeys / kRowsPerPass; ++i) {
          const char* kr = krow[buf * kKeys + n0 + i * kRowsPerPass];
          const char* vr = vrow[buf * kKeys + n0 + i * kRowsPerPass];
          const uint32_t d = dst + (uint32_t)(i * kRowsPerPass * L::kRowBytes);
          // No row: zeros, from an address that is on the 16-byte grid like the
          // others (the copy asks for that even where it reads nothing).
          cp_async16(d, kr ? kr + pc * 16 : static_cast<const char*>(p.k), kr ? 16 : 0);
          cp_async16(d + L::kTileBytes, vr ? vr + pc * 16 : static_cast<const char*>(p.k), vr ? 16 : 0);
        }
      }
    } else {
      for (int i = tid; i < 2 * kKeys * p.D; i += kThreads) {
        const int which = i / (kKeys * p.D), rem = i - which * kKeys * p.D;
        const int n = rem / p.D, d = rem - n * p.D;
        const char* r = (which ? vrow : krow)[buf * kKeys + n];
        *reinterpret_cast<uint16_t*>(smem + (2 * stage + which) * L::kTileBytes + n * L::kRowBytes + d * 2) =
            r ? reinterpret_cast<const uint16_t*>(r)[d] : (uint16_t)0;
      }
    }
    cp_async_commit();
  };
  lookup(0);
  __syncthreads();
  load(0, 0);
  if (n_x > 1) lookup(1);
  if (L::kStages == 3) {
    __syncthreads();
    if (n_x > 1) load(1, 1);
    else cp_async_commit();
    if (n_x > 2) lookup(0);
  }

  const float sl2 = p.scale * kLog2e;
  const float inv_cap = p.soft_cap > 0.f ? 1.f / p.soft_cap : 0.f;
  float o[DT][4];
  uint32_t qa[L::kQShared ? 1 : D / 16][4];
  float m[2], l[2], slope[2] = {0.f, 0.f};
  uint64_t anc[2];
  int pos[2], ref[2] = {0, 0};
  int seg_c0 = 0, R = 0, hkv = 0, rb0 = 0, all_from = 0;
  bool fresh = true;

  for (int x = 0; x < n_x; ++x) {
    const int stage = x % L::kStages;
    cp_async_wait<L::kStages - 2>();
    __syncthreads();  // chunk x is there; its slot's last readers and the looked-up rows are done
    {
      const int nx = x + L::kStages - 1;
      if (nx < n_x) load(nx & 1, nx % L::kStages);
      else cp_async_commit();
      if (nx + 1 < n_x) lookup((nx + 1) & 1);
    }
    if (fresh) {
      fresh = false;
      seg_c0 = cur.c;
      hkv = cur.item / p.n_rb;
      rb0 = (cur.item - hkv * p.n_rb) * L::kRows;
      R = min(L::kRows, p.G * p.N - rb0);
      if (warp == 0) tree_masks(p, cur.b, masks);
      if (tid == 0 && p.status && p.lens[cur.b] != cur.len) *p.status = BFA_ERR_INDEX;
      const uint16_t* qg = static_cast<const uint16_t*>(p.q) + cur.b * p.sq[0];
      if constexpr (L::kQShared) {
        for (int i = tid; i < L::kRows * (D / 2); i += kThreads) {
          const int r = i / (D / 2), c = (i - r * (D / 2)) * 2;
          uint32_t w = 0;
          if (r < R && c < p.D) {
            int hq, n;
            tree_row(p, hkv, rb0 + r, &hq, &n);
            const uint16_t* at = qg + hq * p.sq[1] + n * p.sq[2] + c;
            if (fl.pair) w = *reinterpret_cast<const uint32_t*>(at);
            else w = at[0] | (c + 1 < p.D ? (uint32_t)at[1] << 16 : 0u);
          }
          *reinterpret_cast<uint32_t*>(smem + L::kOffQ + r * L::kRowBytes + c * 2) = w;
        }
      } else {
        // A fragments: rows g and g + 8 of the warp, columns 16ks + 2t and + 8.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = rw * 16 + g + 8 * h;
          int hq, n;
          tree_row(p, hkv, rb0 + min(r, R - 1), &hq, &n);
          const uint16_t* at = qg + hq * p.sq[1] + n * p.sq[2];
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int c = 16 * ks + 8 * e + 2 * t;
              uint32_t w = 0;
              if (r < R && c < p.D) {
                if (fl.pair) w = *reinterpret_cast<const uint32_t*>(at + c);
                else w = at[c] | (c + 1 < p.D ? (uint32_t)at[c + 1] << 16 : 0u);
              }
              qa[ks][h + 2 * e] = w;
            }
        }
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = rw * 16 + g + 8 * h;
        int hq = 0, n = 0;
        if (r < R) tree_row(p, hkv, rb0 + r, &hq, &n);
        anc[h] = r < R ? masks.anc[n] : 0ull;
        pos[h] = cur.len + masks.depth[n];
        if (!PLAIN && p.alibi) {
          slope[h] = p.alibi[hq];
          ref[h] = tree_alibi_ref(p, slope[h], pos[h]);
        }
        m[h] = neg_inf();
        l[h] = 0.f;
      }
      // From this key on every row sees every cached token.
      all_from = p.window > 0 ? cur.len + p.N - 1 - p.window : 0;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    }

    const bool tree = cur.in_tree(p);
    const int key0 = cur.key0(p);
    const bool masked = tree || key0 + kKeys > cur.len || key0 < all_from;
    const uint32_t kt = sbase + (uint32_t)(2 * stage * L::kTileBytes), vt = kt + L::kTileBytes;
    const int mine0 = kw * kMine;

    // S = q·kᵀ of the warp's rows and keys.
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
    {
      const uint32_t ka = kt + (uint32_t)((mine0 + (lane >> 4) * 8 + (lane & 7)) * L::kRowBytes + ((lane >> 3) & 1) * 16);
      const uint32_t qaddr = sbase + (uint32_t)(L::kOffQ + (rw * 16 + (lane & 15)) * L::kRowBytes + (lane >> 4) * 16);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t af[4];
        if constexpr (L::kQShared) {
          ldsm_x4(qaddr + ks * 32, af);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) af[e] = qa[ks][e];
        }
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) {
          uint32_t bf[4];
          ldsm_x4(ka + (uint32_t)(i * 16 * L::kRowBytes) + ks * 32, bf);
          mma16816<T>(s[2 * i], af, bf[0], bf[1]);
          mma16816<T>(s[2 * i + 1], af, bf[2], bf[3]);
        }
      }
    }

    // Logits in base 2, masked; element (h, i, e): row g + 8h, key 8i + 2t + e.
    if (PLAIN && !masked) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] *= sl2;
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1;
          const int key = key0 + mine0 + 8 * i + 2 * t + (e & 1);
          float y = s[i][e];
          int kpos = key;
          if (tree) kpos = cur.len + masks.depth[key & (kTreeNodes - 1)];
          if (PLAIN) {
            y *= sl2;
          } else {
            y *= p.scale;
            if (p.soft_cap > 0.f) y = tree_cap(y, p.soft_cap, inv_cap);
            if (p.alibi) y += slope[h] * (float)(ref[h] - kpos);
            y *= kLog2e;
          }
          if (masked) {
            bool keep = tree ? key < p.N && ((anc[h] >> (key & 63)) & 1) : key < cur.len;
            if (p.window > 0) keep = keep && pos[h] - kpos <= p.window;
            y = keep ? y : neg_inf();
          }
          s[i][e] = y;
        }
    }

    // Values that are not finite must not reach rows that do not see them
    // (0·inf): in the chunks where rows differ in what they see, such rows of
    // V are zeroed for the product and added by hand below.
    uint64_t bad_keys = 0;
    if (tree || (p.window > 0 && masked)) {
      __syncthreads();
      if (tid == 0) *bad = 0ull;
      __syncthreads();
      for (int i = tid; i < kKeys * (D / 8); i += kThreads) {
        const int n = i / (D / 8);
        const uint4 w = *reinterpret_cast<const uint4*>(smem + (2 * stage + 1) * L::kTileBytes + n * L::kRowBytes + (i % (D / 8)) * 16);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
        bool b_ = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) b_ |= not_finite<T>(ws[e]) || not_finite<T>(ws[e] >> 16);
        if (b_) atomicOr(bad, 1ull << n);
      }
      __syncthreads();
      bad_keys = *bad;
    }

    // Online softmax; l is this lane's part of the row sum.
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = neg_inf();
#pragma unroll
      for (int i = 0; i < NT; ++i) mx = fmaxf(mx, fmaxf(s[i][2 * h], s[i][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m[h], mx);
      const float m_use = m_new == neg_inf() ? 0.f : m_new;
      alpha[h] = ex2(m[h] - m_use);
      m[h] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float pr = ex2(s[i][2 * h + e] - m_use);
          s[i][2 * h + e] = pr;
          sum += pr;
        }
      l[h] = l[h] * alpha[h] + sum;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        o[i][0] *= alpha[0];
        o[i][1] *= alpha[0];
        o[i][2] *= alpha[1];
        o[i][3] *= alpha[1];
      }
    }
    if (bad_keys != 0) {
      // By hand, before the rows are zeroed: O += p·v for the warp's bad keys.
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll 1
        for (int n = 0; n < 8; ++n) {
          if (!((bad_keys >> (mine0 + 8 * i + n)) & 1)) continue;
          float pr[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float mine = (n & 1) ? s[i][2 * h + 1] : s[i][2 * h];
            pr[h] = to_f32<T>(from_f32<T>(__shfl_sync(0xffffffffu, mine, (lane & 28) + (n >> 1))));
          }
          const T* vr = reinterpret_cast<const T*>(smem + (2 * stage + 1) * L::kTileBytes + (mine0 + 8 * i + n) * L::kRowBytes);
#pragma unroll
          for (int c = 0; c < DT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (pr[e >> 1] != 0.f) o[c][e] += pr[e >> 1] * to_f32<T>(vr[8 * c + 2 * t + (e & 1)]);
        }
      }
      __syncthreads();
      for (int i = tid; i < kKeys * (D / 8); i += kThreads)
        if ((bad_keys >> (i / (D / 8))) & 1)
          *reinterpret_cast<uint4*>(smem + (2 * stage + 1) * L::kTileBytes + (i / (D / 8)) * L::kRowBytes + (i % (D / 8)) * 16) =
              make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
    }

    // O += P·V.
    {
      const uint32_t va = vt + (uint32_t)((mine0 + (lane & 15)) * L::kRowBytes + (lane >> 4) * 16);
#pragma unroll
      for (int j = 0; j < kMine / 16; ++j) {
        uint32_t pf[4];
        pf[0] = pack2<T>(s[2 * j][0], s[2 * j][1]);
        pf[1] = pack2<T>(s[2 * j][2], s[2 * j][3]);
        pf[2] = pack2<T>(s[2 * j + 1][0], s[2 * j + 1][1]);
        pf[3] = pack2<T>(s[2 * j + 1][2], s[2 * j + 1][3]);
#pragma unroll
        for (int i = 0; i < DT / 2; ++i) {
          uint32_t bf[4];
          ldsm_x4_trans(va + (uint32_t)(j * 16 * L::kRowBytes) + i * 32, bf);
          mma16816<T>(o[2 * i], pf, bf[0], bf[1]);
          mma16816<T>(o[2 * i + 1], pf, bf[2], bf[3]);
        }
      }
    }

    const bool last = cur.c == cur.n - 1;
    const int seq = cur.b, len = cur.len;
    cur.next(p);
    if (!last && x + 1 < n_x) continue;

    // The item, or this block's stretch of it, ends.
    fresh = true;
    const bool whole = seg_c0 == 0 && last;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (anc[h] == 0) {  // an absent node: chunks that are not masked were summed for it too
        l[h] = 0.f;
        m[h] = neg_inf();  // which an infinite logit may have made infinite
      }
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    if constexpr (KW > 1) {
      float2* ml = reinterpret_cast<float2*>(smem + L::kOffMl);
      if (t == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) ml[kw * L::kRows + rw * 16 + g + 8 * h] = make_float2(m[h], l[h]);
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = rw * 16 + g + 8 * h;
        float top = neg_inf(), sum = 0.f;
#pragma unroll
        for (int i = 0; i < KW; ++i) top = fmaxf(top, ml[i * L::kRows + r].x);
        const float use = top == neg_inf() ? 0.f : top;
#pragma unroll
        for (int i = 0; i < KW; ++i) sum += ml[i * L::kRows + r].y * ex2(ml[i * L::kRows + r].x - use);
        const float f = ex2(m[h] - use);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          o[i][2 * h] *= f;
          o[i][2 * h + 1] *= f;
        }
        m[h] = top;
        l[h] = sum;
      }
      // Joined in the order of kw, kJoinCols columns at a time; the last part
      // ends up with the sums in its registers.
      float* join = reinterpret_cast<float*>(smem + L::kOffJoin);
#pragma unroll
      for (int c0 = 0; c0 < DT; c0 += L::kJoinCols / 8) {
#pragma unroll 1
        for (int k = 0; k < KW; ++k) {
          if (kw == k) {
#pragma unroll
            for (int i = 0; i < L::kJoinCols / 8; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float2* at = reinterpret_cast<float2*>(join + (rw * 16 + g + 8 * h) * L::kJoinCols + 8 * i + 2 * t);
                if (k > 0) {
                  const float2 y = *at;
                  o[c0 + i][2 * h] += y.x;
                  o[c0 + i][2 * h + 1] += y.y;
                }
                if (k < KW - 1) *at = make_float2(o[c0 + i][2 * h], o[c0 + i][2 * h + 1]);
              }
          }
          __syncthreads();
        }
      }
    }
    if (kw == KW - 1) {
      const int64_t prow = ((int64_t)blockIdx.x * 2 + (seg_c0 > 0 ? 0 : 1)) * p.rb;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = rw * 16 + g + 8 * h;
        if (r >= R) continue;
        // l = 0: the row saw nothing and is empty. NaN (a logit that it saw was
        // NaN or +inf) goes on into O and LSE.
        const float inv = l[h] != 0.f ? 1.f / l[h] : 0.f;
        int hq, n;
        tree_row(p, hkv, rb0 + r, &hq, &n);
        uint16_t* og = static_cast<uint16_t*>(p.o) + seq * p.so[0] + hq * p.so[1] + n * p.so[2];
        float* pg = p.part_o + (prow + r) * p.D;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const int c = 8 * i + 2 * t;
          if (c >= p.D) continue;
          // An empty row is zero even where the values it does not see are not finite.
          const float a = inv != 0.f ? o[i][2 * h] * inv : 0.f, b = inv != 0.f ? o[i][2 * h + 1] * inv : 0.f;
          if (whole) {
            const uint32_t w = pack2<T>(a, b);
            if (fl.pair) {
              *reinterpret_cast<uint32_t*>(og + c) = w;
            } else {
              og[c] = (uint16_t)w;
              if (c + 1 < p.D) og[c + 1] = (uint16_t)(w >> 16);
            }
          } else if (fl.pair) {
            *reinterpret_cast<float2*>(pg + c) = make_float2(a, b);
          } else {
            pg[c] = a;
            if (c + 1 < p.D) pg[c + 1] = b;
          }
        }
        if (t == 0) {
          const float l2 = l[h] != 0.f ? m[h] + __log2f(l[h]) : neg_inf();
          if (!whole) p.part_lse[prow + r] = l2;
          else if (p.lse)
            p.lse[((int64_t)seq * p.Hq + hq) * p.N + n] =
                l2 == neg_inf() ? l2 : l2 * kLn2 + tree_row_shift(p, hq, len + masks.depth[n]);
        }
      }
    }
    // The next segment rewrites the masks (and ml, q): the top-of-loop barrier
    // of the next chunk comes first.
  }
}

template <typename T, int D, int RW, int KW>
int launch_k(const TreeParams& p, const Flags& fl, cudaStream_t st) {
  using L = Tile<D, RW, KW>;
  const bool plain = p.soft_cap == 0.f && !p.alibi;
  auto kernel = plain ? tree_mma_kernel<T, D, RW, KW, true> : tree_mma_kernel<T, D, RW, KW, false>;
  static std::atomic<uint64_t> done[2];
  const int rc = allow_shared(kernel, L::kBytes, done[plain], "tree attention shared memory");
  if (rc) return rc;
  kernel<<<p.grid, L::kThreads, L::kBytes, st>>>(p, fl);
  note_launch();
  return launch_status("tree attention launch");
}

// Row warps for a KV head's rows: the least that hold them, up to 64 rows a
// block at D = 256 (O fills the registers) and 128 below.
int row_warps(int64_t rows, int D) {
  if (rows <= 16) return 1;
  if (rows <= 32) return 2;
  if (rows <= 64 || D > 128) return 4;
  return 8;
}

template <typename T, int D>
int launch_d(const TreeParams& p, const Flags& fl, cudaStream_t st) {
  switch (p.rb / 16) {
    case 1: return launch_k<T, D, 1, 4>(p, fl, st);
    case 2: return launch_k<T, D, 2, 2>(p, fl, st);
    case 4:
      if constexpr (D == 256) return launch_k<T, D, 4, 2>(p, fl, st);
      else return launch_k<T, D, 4, 1>(p, fl, st);
    default:
      if constexpr (D <= 128) return launch_k<T, D, 8, 1>(p, fl, st);
      return BFA_ERR_UNSUPPORTED;
  }
}

template <typename T>
int launch_t(const TreeParams& p, const Flags& fl, cudaStream_t st) {
  if (p.D <= 64) return launch_d<T, 64>(p, fl, st);
  if (p.D <= 128) return launch_d<T, 128>(p, fl, st);
  return launch_d<T, 256>(p, fl, st);
}

template <int D>
int per_sm(int rw) {
  switch (rw) {
    case 1: return Tile<D, 1, 4>::kPerSm;
    case 2: return Tile<D, 2, 2>::kPerSm;
    case 4: return D == 256 ? Tile<D, 4, 2>::kPerSm : Tile<D, 4, 1>::kPerSm;
    default: return 1;
  }
}

}  // namespace

TreeTile tree_mma_tile(int64_t rows, int D) {
  const int rw = row_warps(rows, D);
  return {16 * rw, kKeys, D <= 64 ? per_sm<64>(rw) : D <= 128 ? per_sm<128>(rw) : per_sm<256>(rw)};
}

int tree_mma(const TreeParams& p, int dtype, cudaStream_t st) {
  auto grid = [](const void* d, const int64_t* s, int bytes) {
    return ((uintptr_t)d & (bytes - 1)) == 0 && s[0] * 2 % bytes == 0 && s[1] * 2 % bytes == 0 && s[2] * 2 % bytes == 0;
  };
  Flags fl;
  fl.vec = p.D % 8 == 0 && grid(p.k, p.sk, 16) && grid(p.v, p.sv, 16) && grid(p.kp, p.skp, 16) && grid(p.vp, p.svp, 16);
  fl.pair = p.D % 2 == 0 && grid(p.q, p.sq, 4) && grid(p.o, p.so, 4);
  return dtype == BFA_DTYPE_F16 ? launch_t<__half>(p, fl, st) : launch_t<__nv_bfloat16>(p, fl, st);
}

}  // namespace bfa
