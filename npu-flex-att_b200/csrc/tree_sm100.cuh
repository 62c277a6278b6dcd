// tree_sm100.cuh -- attention of a tree of drafted tokens over a paged cache in
// bf16 / fp16 on tcgen05, K/V pages by TMA.
//
// Mathematics: the online softmax of the other forwards (base 2; P rounded to
// the input type and kept in TMEM as the A operand of P·V; O rescaled only when
// a row's maximum grows by more than 2^8). The rows r = g·N + n of one KV head
// are stacked into tiles of 128, so its K/V cross HBM once per block of rows.
//
// Bound: HBM (K/V read once) up to about 256 rows per KV head, the tensor cores
// above. Measured with its merge, bf16, 8 KV heads of 128, B=16, L=8192 (537 MB
// of K/V): 4 to 32 rows per KV head 90 to 95 us (91 to 87% of the HBM floor),
// 64 rows 103, 128 rows 113; 256 rows 173 us, where one tile's chain of softmax
// and products sets the pace (2.4 us per 128 keys for 1.1 us of products). Head
// dim 64, L=8192, 16 rows (268 MB): 62 us, the softmax's chain of latencies, 0.85
// us per chunk. A call that reads next to nothing takes 13 us: launch, work
// split, page table, one chunk, merge, each waiting for the one before.
//
// Split. Persistent blocks, one per SM, each with an equal stretch of the list
// of chunks (tree_common.cuh). Warp roles:
//   warps 0, 2  producers of K and of V: find a chunk's pages and load it by
//               TMA, a lane per box, into a ring that runs on across items
//   warp 1      MMA issuer
//   warp 2      also allocates TMEM
//   warp 3      the tree's ancestor sets, one item ahead; REP = 4: items whose O
//               holds columns that are not finite
//   warps 4..   softmax, 8 warps per 128-row tile: two threads share a row (TMEM
//               lane), each with half of the chunk's keys and of O's columns;
//               they agree on the row's maximum through shared memory. P (16-bit)
//               takes the first half of each thread's own columns of S
// Few rows (REP = 4: up to 32 per KV head). One row per TMEM lane would leave
// three quarters of the softmax warps without rows, and the one quarter's
// exponentials would set the pace (0.7 us a chunk, twice what HBM takes for
// it). So the rows are stored four times, once per quarter of the lanes, and
// each quarter forms P for its quarter of every half's keys, zeros elsewhere:
// the quarters' O are sums over different keys, joined like other partial
// results when the item ends.
// With two tiles (NT = 2) one tile's softmax runs under the other's products:
// S_0(j), S_1(j), then PV_0(j), S_0(j+1), PV_1(j), S_1(j+1). With one tile S is
// double-buffered: S(j+1) is formed before PV(j), and the softmax warps go from
// chunk to chunk without waiting for a product. (Tried and slower: P·V in two
// halves of the keys, each as soon as its P is stored, 1 to 3% by the second
// wait of the one issuing thread; two tiles with chunks of 64 and double-
// buffered S, 557 against 428 us on 512 rows over 10.5k tokens of 16 sequences.)
//
// A box is gcd(page_size, chunk) tokens of one page, so any page size that is a
// multiple of 8 works (8 rows of 128 bytes are the swizzle's atom). A lane per
// box issues. B=16, L=8192, 4 rows per KV head: pages of 64 and more 92 us, of
// 16 95, of 8 110 (121 with one elected lane for all boxes); head dim 64, 16
// rows: 63, 64 and 76. Tokens past a
// sequence's end arrive as whatever the page holds: their logits are masked,
// P·V stops at the last 16 keys that hold one, and the softmax warps clear the
// rest of those 16 in V before the product may read it.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <climits>
#include <numeric>
#include <type_traits>

#include "sm100_host.h"
#include "sm100_ptx.cuh"
#include "tree_common.cuh"

namespace bfa {
namespace {

using namespace sm100;

constexpr int kBM = 128;
constexpr float kRescaleThreshold = 8.0f;

// CH keys per chunk: 128, or 64 at D = 256 (64 KB of K and V either way).
template <int D, int NT, int REP>
struct TreeLayout {
  static constexpr int kCH = D == 256 ? 64 : 128;
  static constexpr int kSub = D / 64;
  static constexpr int kSeg = kCH / 2 / REP;
  static constexpr int kGroup = kSeg < 32 ? kSeg : 32;
  static constexpr uint32_t kQTile = kBM * D * 2;
  static constexpr uint32_t kKV = kCH * D * 2;
  static constexpr uint32_t kMisc = 10240;
  static constexpr int kFit = (int)((232448u - 1024u - kMisc - NT * kQTile) / kKV);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr uint32_t kOffKV = NT * kQTile;
  static constexpr uint32_t kOffMisc = kOffKV + kStages * kKV;
  static constexpr uint32_t kBytes = kOffMisc + kMisc + 1024;  // 1024: alignment of the tiles
  // TMEM columns: S (two buffers, or one per tile), O, and with one tile P (two
  // buffers of 16-bit pairs); with two tiles P takes columns of S.
  static constexpr uint32_t kTmemO = 2 * kCH;
  static constexpr uint32_t kTmemP = kTmemO + NT * D;
  static constexpr int kThreads = 128 + 256 * NT;
  static_assert(kStages >= 4, "K and V of two chunks");
  static_assert(kTmemP + (NT == 1 ? kCH : 0) <= 512, "TMEM");
  static_assert(REP == 1 || (REP == 4 && NT == 1), "rows");
  static_assert(REP == 1 || 4 * 2 * 32 * (D / 4) * 4 <= kQTile, "the quarters' O are joined in q's tile");
  static_assert(kBytes <= 232448, "shared memory");
};

struct TreeMisc {
  uint64_t bar[40];
  uint32_t tmem;
  int abort;
  unsigned long long bad[3][2];  // by the chunk's number mod 3: its keys whose values are not finite
  float top[2][2][2][kBM];       // row maxima: chunk's parity, tile, half of the keys, row
  float sum[2][2][kBM];          // row sums at an item's end: tile, half, row
  float quarter[kBM];            // REP = 4: maxima of the quarters, their sums by the item's parity,
  float total[2][kBM];
  int odd[2];                    // whether its O holds columns that are not finite,
  TreeCursor item[2];            // and its place, with the chunks of it that are this block's
  int count[2];
  TreeMasks masks[2];            // by the item's parity
};
static_assert(sizeof(TreeMisc) <= 10240, "misc");

// One column (32 bits per lane) of TMEM.
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  return r;
}

// N columns, 8 of S to 4 of P.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 32) tmem_ld32(taddr, r);
  else if constexpr (N == 16) tmem_ld16(taddr, r);
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t taddr, const uint32_t (&r)[N]) {
  if constexpr (N == 32) tmem_st32(taddr, r);
  else if constexpr (N == 16) tmem_st16(taddr, r);
  else if constexpr (N == 8)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  else
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}

// One lane of a converged warp. The compiler knows that a branch on it holds one
// thread, and issues tcgen05 and TMA instructions without a loop over the lanes
// that may be active (a branch on lane 0: 72 against 61 us at head dim 64, B=16,
// L=8192; 320 against 303 us on 512 rows).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// tanh by sign(x)·(1 - 2/(1 + e^{2|x|})). Where tanh_any keeps its exponent below
// 126, e^{2|x|} may run to infinity here (the quotient is 0 either way): the
// bound would turn NaN into 1.
__device__ __forceinline__ float tanh_of(float x) {
  return copysignf(1.0f - 2.0f * rcp(1.0f + ex2(2.0f * kLog2e * fabsf(x))), x);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return BF16 ? pack_bf16(a, b) : pack_f16(a, b);
}
template <bool BF16>
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
  const uint32_t h = hi ? w >> 16 : w & 0xffffu;
  return BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}
template <bool BF16>
__device__ __forceinline__ bool any_not_finite(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// With the rows stored four times, a value of V that is not finite meets the
// zeros that P holds for three of the quarters, and comes out as NaN in place of
// infinity. So where columns of an item's rows are not finite, they are formed
// again: the sum of the values of V there that are not finite, over this
// block's keys that the row sees (a positive weight changes none of them). Only
// broken inputs come here. Called by the warp of the ancestor sets once the item
// is stored: one token over 4095 takes 13.4 us with it and 13.1 without (called
// by the softmax warps 14.0, inlined into that warp's part 14.2).
// `cur`: the item and the first of `count` chunks; sums: the quarters' row sums.
template <int D, bool BF16>
__device__ __noinline__ void sum_not_finite(const TreeParams& p, const TreeMasks& masks, const float* sums, TreeCursor cur, int count) {
  const int lane = threadIdx.x & 31;
  const int hkv = cur.item / p.n_rb, r = (cur.item - hkv * p.n_rb) * p.rb + lane, end = cur.c + count;
  auto finite = [](float x) { return fabsf(x) < __int_as_float(0x7f800000); };
  auto row_of = [&](int key) -> int64_t {  // of a cached key in v_pages, -1: a bad page
    const int page = p.table[cur.b * p.table_stride + key / p.page];
    return page >= 0 && page < p.num_pages ? page * p.svp[0] + hkv * p.svp[1] + key % p.page * p.svp[2] : -1;
  };
  // Cached keys [from, some): in chunks where rows differ in what they see;
  // [some, to): seen by all. Of those, a lane collects which signs (NaN: both)
  // its 8 columns hold.
  const int from = cur.lo + cur.c * p.chunk, to = min(cur.len, cur.lo + end * p.chunk);
  const int all_from = p.window > 0 ? cur.len + p.N - 1 - p.window : 0;
  const int some = min(to, max(from, cur.lo + (max(all_from - cur.lo, 0) + p.chunk - 1) / p.chunk * p.chunk));
  uint32_t up = 0, down = 0;
#pragma unroll 1
  for (int key = some; key < to; ++key) {
    const int64_t at = row_of(key);
    if (at < 0 || lane * 8 >= p.D) continue;
    const uint4 w4 = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.vp) + at + lane * 8);
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = half_of<BF16>(w[e >> 1], e & 1);
      if (!finite(x)) {
        if (!(x < 0.f)) up |= 1u << e;
        if (!(x > 0.f)) down |= 1u << e;
      }
    }
  }
  // Then a lane per row.
  const float all = (sums[lane] + sums[32 + lane]) + (sums[64 + lane] + sums[96 + lane]);
  const bool live = r < p.G * p.N && all == all;  // a row sum that is NaN: the logits were no numbers, and O stays NaN
  int hq, node;
  tree_row(p, hkv, live ? r : 0, &hq, &node);
  const int depth = masks.depth[node];
  const int low = p.window > 0 ? max(from, cur.len + depth - p.window) : from;
  const bool whole = cur.c == 0 && count == cur.n;
#pragma unroll 1
  for (int d = 0; d < p.D; ++d) {
    const bool pos = (__shfl_sync(0xffffffffu, up, d >> 3) >> (d & 7)) & 1, neg = (__shfl_sync(0xffffffffu, down, d >> 3) >> (d & 7)) & 1;
    uint16_t* out = static_cast<uint16_t*>(p.o) + cur.b * p.so[0] + hq * p.so[1] + node * p.so[2] + d;
    float* part = p.part_o + (((int64_t)blockIdx.x * 2 + (cur.c > 0 ? 0 : 1)) * p.rb + lane) * p.D + d;
    if (!live || finite(whole ? half_of<BF16>(*out, 0) : *part)) continue;
    float sum = (pos ? __int_as_float(0x7f800000) : 0.f) + (neg ? __int_as_float(0xff800000) : 0.f);
    auto add = [&](const void* v, int64_t at) {
      const float x = half_of<BF16>(static_cast<const uint16_t*>(v)[at + d], 0);
      if (!finite(x)) sum += x;
    };
#pragma unroll 1
    for (int key = low; key < some; ++key) {
      const int64_t at = row_of(key);
      if (at >= 0) add(p.vp, at);
    }
    if (end > cur.n - p.tree_chunks)
#pragma unroll 1
      for (int n = 0; n < p.N; ++n)
        if (((masks.anc[node] >> n) & 1) && (p.window == 0 || depth - masks.depth[n] <= p.window))
          add(p.v, cur.b * p.sv[0] + hkv * p.sv[1] + n * p.sv[2]);
    if (sum == 0.f) continue;
    if (whole) *out = (uint16_t)pack2<BF16>(sum, 0.f);
    else *part = sum;
  }
  __syncwarp();
}

template <int D, int NT, int REP, bool BF16, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(TreeLayout<D, NT, REP>::kThreads, 1)
    tree_kernel(const __grid_constant__ CUtensorMap tmKp, const __grid_constant__ CUtensorMap tmVp,
                const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ TreeParams p, int box,
                uint64_t timeout_ns) {
  using L = TreeLayout<D, NT, REP>;
  constexpr int CH = L::kCH, NS = L::kStages;
  constexpr int HC = CH / 2;    // keys of a half
  constexpr int SEG = L::kSeg, GW = L::kGroup;  // keys of a softmax thread per chunk, and of them at a time
  using Group = uint32_t[L::kGroup];
  // With one tile a softmax thread holds its S row in registers from the
  // maximum to the exponentials. Two tiles' 512 softmax threads have 96
  // registers each: they read S twice, 32 columns at a time (holding it
  // spilled to local memory).
  constexpr bool kHold = NT == 1;
  constexpr int kGroups = SEG / GW, kUnroll = kHold ? kGroups : 1;
  enum {
    kQFull = 0,
    kKVFull = 1,
    kKVEmpty = kKVFull + NS,
    kMask = kKVEmpty + NS,   // the item's ancestor sets, by its parity
    kMaskFree = kMask + 2,   // an item's softmax is done with them
    // Two of each: NT = 2: of tile t, a phase a chunk; NT = 1: of the chunk's
    // parity (its S buffer), a phase every second chunk.
    kSFull = kMaskFree + 2,  // S formed
    kPFull = kSFull + 2,     // P, and an O that may be added to, in TMEM
    kODone = kPFull + 2,     // P·V done
    kDrain = kODone + 2,
    kNumBars = kDrain + 1
  };
  static_assert(kNumBars <= 40, "barriers");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  TreeMisc& mi = *reinterpret_cast<TreeMisc*>(smem + L::kOffMisc);
  auto bar = [&](int i) -> uint32_t { return sbase + L::kOffMisc + 8u * (uint32_t)i; };
  auto phase = [](int x) { return (NT == 2 ? x : x >> 1) & 1; };  // of chunk x's barriers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tmKp);
    tma_prefetch_desc(&tmVp);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int i = 0; i < kNumBars; ++i)
      mbar_init(bar(i), i == kQFull || i == kMaskFree || i == kMaskFree + 1 ? 8u * NT : i >= kPFull && i < kODone ? 8u : 1u);
    mi.abort = 0;
    mi.odd[0] = mi.odd[1] = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(&mi.tmem), 512);
    tmem_relinquish();
  }
  TreeCursor cur;
  const int n_x = tree_stretch(p, cur);  // 0 in a block without work: it only passes through
  WaitCtl ctl{(volatile int*)&mi.abort, p.status, timeout_ns};
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = mi.tmem;

  // P of a half of the keys.
  auto p_at = [&](int buf, int half) -> uint32_t {
    return tmem + (NT == 2 ? buf * CH + half * HC : L::kTmemP + buf * (CH / 2) + half * (HC / 2));
  };
  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------ producers
    const int kv = warp >> 1;
    // Lane i·kSub + s: columns [64s, 64s + 64) of box i, tokens [key0 + i·box,
    // + box) of one page (the tree's chunk: one box of 64 nodes).
    const int my_box = lane / L::kSub, my_sub = lane % L::kSub;
    const int boxes = CH / box, per = 32 / boxes;  // powers of 2
    // The boxes of `per` chunks of an item from its chunk `c`, one per lane:
    // their pages (0 past the cache) and first tokens in them; -1 in a box that
    // lies before the window whole, whose page may have been given back: its
    // table entry is not read, and it is loaded as zeros.
    int page = 0, slot = 0, next_page = 0, next_slot = 0;
    auto lookup = [&](const TreeCursor& at, int c) {
      const int t = at.lo + c * CH + lane * box;
      const int pg = p.page_log2 >= 0 ? t >> p.page_log2 : t / p.page;
      const bool behind = p.window > 0 && t + box <= at.len - p.window;
      next_slot = behind ? -1 : t - pg * p.page;
      next_page = t < at.len && !behind ? p.table[at.b * p.table_stride + pg] : 0;
    };
    bool ok = true;
    int x = 0, st = kv, round = 0;  // the next load's slot and that slot's round
    auto begin = [&](uint32_t bytes) -> bool {
      if (round > 0) ok = warp_wait(bar(kKVEmpty + st), (uint32_t)((round & 1) ^ 1), ctl);
      if (ok && lane == 0) mbar_arrive_expect_tx(bar(kKVFull + st), bytes);
      __syncwarp();
      return ok;
    };
    auto end = [&]() {
      __syncwarp();
      ++x;
      st += 2;
      if (st >= NS) {
        st -= NS;
        ++round;
      }
    };
    if (n_x > 0) lookup(cur, cur.c);
    while (x < n_x && ok) {
      const TreeCursor here = cur;
      const int count = min(here.n - here.c, n_x - x);
      const int cached = min(max(here.n - p.tree_chunks - here.c, 0), count);
      const int hkv = here.item / p.n_rb;
      const bool more = x + count < n_x;
      // The next pages that will be needed, this item's or the next one's:
      // looked up as soon as the last ones are in use.
      auto ahead = [&](int it) {
        if (it < cached) {
          lookup(here, here.c + it);
        } else {
          cur.next(p, count);
          if (more) lookup(cur, cur.c);
        }
      };
      if (cached == 0) ahead(0);
      for (int it = 0; it < cached; ++it) {
        const int j = it & (per - 1);
        if (j == 0) {
          page = next_page;
          slot = next_slot;
          if (slot < 0 || page < 0 || page >= p.num_pages) {
            page = (int)p.num_pages;  // outside the tensor: reads as zeros
            if (slot >= 0 && p.status) *p.status = BFA_ERR_INDEX;
            slot = 0;
          }
        }
        const int pg = __shfl_sync(0xffffffffu, page, j * boxes + my_box);  // the lane is taken modulo 32
        const int sl = __shfl_sync(0xffffffffu, slot, j * boxes + my_box);
        const int left = here.len - (here.lo + (here.c + it) * CH);
        const bool mine = my_box < boxes && my_box * box < left;
        const uint32_t bytes = left >= CH ? L::kKV : (uint32_t)__popc(__ballot_sync(0xffffffffu, mine)) * box * 128u;
        if (!begin(bytes)) break;
        if (mine)
          tma_load_4d(sbase + L::kOffKV + st * L::kKV + my_sub * (CH * 128) + my_box * box * 128, kv ? &tmVp : &tmKp,
                      bar(kKVFull + st), my_sub * 64, sl, hkv, pg);
        end();
        if (j == 0) ahead(it + per);
      }
      if (ok && cached < count && begin(L::kSub * 64 * 128u)) {  // the tree
        if (my_box == 0)
          tma_load_4d(sbase + L::kOffKV + st * L::kKV + my_sub * (CH * 128), kv ? &tmV : &tmK, bar(kKVFull + st), my_sub * 64, 0, hkv,
                      here.b);
        end();
      }
    }
    const int n = 2 * x + kv;  // past the last load issued
    // This warp's loads among the block's last NS (one per slot; earlier ones
    // have been consumed, and their slots hold later loads of either producer)
    // have landed before the block may end.
    if (lane == 0)
      for (int i = n - 2; i >= 0 && i >= 2 * n_x - NS; i -= 2) drain_wait(bar(kKVFull + i % NS), (i / NS) & 1, timeout_ns);
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t idS = idesc_f16(kBM, CH, BF16, false);
      constexpr uint32_t idO = idesc_f16(kBM, D, BF16, true);
      auto kv_addr = [&](int idx) -> uint32_t { return sbase + L::kOffKV + (uint32_t)(idx % NS) * L::kKV; };
      auto issue_s = [&](int t, int buf, int idx) {
        const uint64_t dq = desc_kmajor(sbase + t * L::kQTile);
        const uint64_t dk = desc_kmajor(kv_addr(idx));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t offq = (kk >> 2) * (kBM * 128) + (kk & 3) * 32;
          const uint32_t offk = (kk >> 2) * (CH * 128) + (kk & 3) * 32;
          mma_ss(tmem + buf * CH, dq + (offq >> 4), dk + (offk >> 4), idS, kk > 0 ? 1u : 0u);
        }
        mma_commit(bar(kSFull + buf));
      };
      auto wait = [&](int i, int parity) {
        if (!mbar_wait(bar(i), (uint32_t)parity, ctl, BFA_ERR_DEVICE_TIMEOUT)) return false;
        tc_fence_after();
        return true;
      };
      auto wait_load = [&](int idx) { return wait(kKVFull + idx % NS, (idx / NS) & 1); };
      // P·V of chunk x over its first `steps`·16 keys. O is
      // zeroed by the softmax warps at an item's start: every product adds.
      auto pv = [&](int t, int buf, int x, int steps) {
        const uint64_t dv = desc_mnmajor(kv_addr(2 * x + 1), CH * 128);
        if (!wait(kPFull + buf, phase(x))) return false;
        if (steps == CH / 16) {  // nearly always: no branch per product
#pragma unroll
          for (int kk = 0; kk < CH / 16; ++kk)
            mma_ts(tmem + L::kTmemO + t * D, p_at(buf, kk / (CH / 32)) + kk % (CH / 32) * 8, dv + ((kk * 16 * 128) >> 4), idO, 1u);
        } else {
#pragma unroll 1
          for (int kk = 0; kk < steps; ++kk)
            mma_ts(tmem + L::kTmemO + t * D, p_at(buf, kk / (CH / 32)) + kk % (CH / 32) * 8, dv + ((kk * 16 * 128) >> 4), idO, 1u);
        }
        mma_commit(bar(kODone + buf));
        return true;
      };
      bool ok = true;
      int seg = 0;
      for (int x = 0; x < n_x && ok; ++seg) {
        const int count = min(cur.n - cur.c, n_x - x);  // chunks of this item that are this block's
        ok = wait(kQFull, seg & 1) && wait_load(2 * x);
        if (!ok) break;
        issue_s(0, NT == 2 ? 0 : x & 1, 2 * x);
        if constexpr (NT == 2) issue_s(1, 1, 2 * x);
        mma_commit(bar(kKVEmpty + (2 * x) % NS));
        for (int it = 0; it < count; ++it, ++x) {
          const int iv = 2 * x + 1, ik = 2 * x + 2;
          const bool more = it + 1 < count;
          const int c = cur.c + it;
          const int keys = c >= cur.n - p.tree_chunks ? p.N : min(CH, cur.len - (cur.lo + c * CH));
          const int steps = (keys + 15) / 16;
          if constexpr (NT == 2) {
            if (!(ok = wait_load(iv) && pv(0, 0, x, steps))) break;
            if (more) {
              if (!(ok = wait_load(ik))) break;
              issue_s(0, 0, ik);
            }
            if (!(ok = pv(1, 1, x, steps))) break;
            mma_commit(bar(kKVEmpty + iv % NS));
            if (more) {
              issue_s(1, 1, ik);
              mma_commit(bar(kKVEmpty + ik % NS));
            }
          } else {
            if (more) {
              if (!(ok = wait_load(ik))) break;
              issue_s(0, (x + 1) & 1, ik);
              mma_commit(bar(kKVEmpty + ik % NS));
            }
            if (!(ok = wait_load(iv) && pv(0, x & 1, x, steps))) break;
            mma_commit(bar(kKVEmpty + iv % NS));
          }
        }
        cur.next(p, count);
      }
      mma_commit(bar(kDrain));
      drain_wait(bar(kDrain), 0, timeout_ns);
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ ancestor sets
    bool ok = true;
    int seg = 0;
    for (int x = 0; x < n_x && ok; ++seg) {
      const int count = min(cur.n - cur.c, n_x - x);
      if (seg > 1) ok = warp_wait(bar(kMaskFree + (seg & 1)), (uint32_t)(((seg >> 1) - 1) & 1), ctl);
      if constexpr (REP == 4) {
        if (ok && mi.odd[seg & 1]) sum_not_finite<D, BF16>(p, mi.masks[seg & 1], mi.total[seg & 1], mi.item[seg & 1], mi.count[seg & 1]);
        if (lane == 0) mi.odd[seg & 1] = 0, mi.item[seg & 1] = cur, mi.count[seg & 1] = count;
      }
      tree_masks(p, cur.b, mi.masks[seg & 1]);
      if (lane == 0) {
        if (p.status && p.lens[cur.b] != cur.len) *p.status = BFA_ERR_INDEX;
        mbar_arrive(bar(kMask + (seg & 1)));
      }
      x += count;
      cur.next(p, count);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax
    const int t = NT == 2 ? (warp - 4) >> 3 : 0, h = ((warp - 4) >> 2) & 1, wq = warp & 3;
    const int trow = wq * 32 + lane;                  // TMEM lane: row of the tile
    const int row = REP == 4 ? lane : trow;           // the row it holds
    const int seg0 = h * HC + (REP == 4 ? wq * SEG : 0);  // its first key of a chunk
    const int sid = threadIdx.x - 128;  // among the softmax threads
    constexpr int kSoft = 256 * NT;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    const uint32_t tO = tmem + lane_base + L::kTmemO + t * D + h * (D / 2);  // this thread's half of O
    const float sl2 = p.scale * kLog2e;
    const float cap_in = CAP ? p.scale / p.soft_cap : 0.f, cap_out = CAP ? p.soft_cap * kLog2e : 0.f;
    bool ok = true;  // false: this block gave up on a wait; the flow goes on without waiting
    if (REP > 1) {  // P outside a quarter's keys stays zero
      uint32_t z[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) z[i] = 0u;
#pragma unroll
      for (int i = 0; i < HC / 32; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) tmem_st16(p_at(b, h) + lane_base + 16 * i, z);
      tmem_st_wait();
    }
    int seg = 0;
    for (int x = 0; x < n_x; ++seg) {
      // ---------------------------------------------------- an item begins
      // (`cur` stands at its first chunk of this block's. Little else is kept
      // over the loop: what only masked chunks and the end need is formed
      // again there, from values made opaque so that none stays in registers.)
      const int count = min(cur.n - cur.c, n_x - x);
      auto where = [&](int* hq, int* node) -> bool {  // the row's head and node; false past the rows
        int item = cur.item;
        asm volatile("" : "+r"(item));
        const int hkv = item / p.n_rb, r = (item - hkv * p.n_rb) * p.rb + t * kBM + row;
        const bool live = r < p.G * p.N;
        tree_row(p, hkv, live ? r : 0, hq, node);
        return live;
      };
      {
        // Half of q's rows of this warp into the swizzled tile (its readers, the
        // last item's S products, are done: their barrier was waited for). The
        // lanes take the 16-byte pieces of a row side by side: a lane per row
        // would touch 32 lines with every load, and the page table's loads
        // would queue behind them (5 us at the start of an item of 256 rows).
        int hq, node;
        const bool live = where(&hq, &node);
        const int64_t mine = live ? cur.b * p.sq[0] + hq * p.sq[1] + node * p.sq[2] : -1;
        uint8_t* dst = smem + t * L::kQTile;
        if (D == 64) named_sync(4 + 4 * t + wq, 64);  // the other half's rows of the last item have left these lines
        constexpr int kPer = D / 16;  // pieces of a half row
#pragma unroll 8
        for (int i = 0; i < kPer; ++i) {
          const int idx = i * 32 + lane, r = idx / kPer, c = h * kPer + idx % kPer;
          const int64_t at = __shfl_sync(0xffffffffu, mine, r);
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if (at >= 0 && c * 8 < p.D) w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at + c * 8);
          *reinterpret_cast<uint4*>(dst + (c >> 3) * (kBM * 128) + sw128_offset(wq * 32 + r, c & 7)) = w;
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kQFull));
        uint32_t z[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0u;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) tmem_st16(tO + 16 * c, z);
        tmem_st_wait();
      }
      TreeMasks& masks = mi.masks[seg & 1];
      ok = ok && warp_wait(bar(kMask + (seg & 1)), (uint32_t)((seg >> 1) & 1), ctl);
      const int all_from = p.window > 0 ? cur.len + p.N - 1 - p.window : 0;
      float m = neg_inf(), l = 0.f;  // l: of this thread's keys
      float slope2 = 0.f;            // ALiBi, times log2 e
      int ref = 0;
      if (ALIBI) {
        int hq, node;
        where(&hq, &node);
        slope2 = p.alibi[hq] * kLog2e;
        ref = tree_alibi_ref(p, slope2, cur.len + masks.depth[node]);
      }

      for (int it = 0; it < count; ++it, ++x) {
        const int c = cur.c + it;
        const bool tree = c >= cur.n - p.tree_chunks;
        const int key0 = tree ? 0 : cur.lo + c * CH;
        const int valid = tree ? p.N : min(CH, cur.len - key0);  // rows of the chunk that hold keys
        const bool masked = tree || valid < CH || key0 < all_from;
        const int buf = NT == 2 ? t : x & 1;
        const uint32_t tS = tmem + lane_base + buf * CH;

        // The last P·V's rows of V that no key holds are cleared (the tree's
        // come as zeros); where rows differ in what they see, values that are
        // not finite are looked for: 0·inf must not reach a row that does not
        // see the key.
        bool hold = false;
        const bool differ = (tree && p.N > 1) || key0 < all_from;
        if (differ || (!tree && (valid & 15))) {
          ok = ok && warp_wait(bar(kKVFull + (2 * x + 1) % NS), (uint32_t)(((2 * x + 1) / NS) & 1), ctl);
          uint8_t* vt = smem + L::kOffKV + ((2 * x + 1) % NS) * L::kKV;
          // A warp that clears this has seen S(x - 1), which is issued after
          // every warp has stored P of chunk x - 3 (the slot's last use); one of
          // chunk x - 2 may still be on its way to read its own slot.
          unsigned long long* bad = mi.bad[x % 3];
          if (sid < 2) bad[sid] = 0ull;
          named_sync(3, kSoft);
          // Piece i: 16 bytes of row i / 8 of a 64-column sub-tile.
          const int upto = (valid + 15) / 16 * 16;
          for (int i = (differ ? 0 : valid * 8) + sid; i < upto * 8; i += kSoft) {
            const int r = i >> 3;
#pragma unroll
            for (int sub = 0; sub < L::kSub; ++sub) {
              uint4* at = reinterpret_cast<uint4*>(vt + sub * (CH * 128) + r * 128 + (i & 7) * 16);
              if (r >= valid) {
                *at = make_uint4(0u, 0u, 0u, 0u);
              } else {
                const uint4 w = *at;
                if (any_not_finite<BF16>(w.x) || any_not_finite<BF16>(w.y) || any_not_finite<BF16>(w.z) || any_not_finite<BF16>(w.w))
                  atomicOr(&bad[r >> 6], 1ull << (r & 63));
              }
            }
          }
          fence_async_shared();
          named_sync(3, kSoft);
          hold = (bad[0] | bad[1]) != 0;
        }

        ok = ok && warp_wait(bar(kSFull + buf), (uint32_t)phase(x), ctl);
        tc_fence_after();
        // Groups of columns past the last 16 keys that hold one are left out:
        // P·V stops there.
        const int used = (valid + 15) / 16 * 16 - seg0;  // of this thread's columns
        const bool formed = CAP || ALIBI || masked || !(sl2 > 0.f);  // logits in r, else raw products
        // What masked chunks keep: columns [lo, hi) of cached tokens, or the seen nodes.
        int lo = 0, hi = 0;
        uint64_t seen = 0;
        if (masked && used > 0) {
          int hq, node;
          const bool live = where(&hq, &node);
          const int depth = masks.depth[node];
          seen = live ? masks.anc[node] : 0ull;
          lo = p.window > 0 ? max(0, cur.len + depth - p.window - key0) : 0;
          hi = seen ? valid : 0;
          if (tree && p.window > 0 && p.window < p.N)
            for (int i = 0; i < p.N; ++i)
              if (depth - masks.depth[i] > p.window) seen &= ~(1ull << i);
        }
        // Logits in base 2 of a group (cap's tanh: the series on the FMA pipe
        // where every |s/cap| of the warp is small, else the closed form).
        auto form = [&](Group& u, int k0, auto tier_tag) {
          constexpr int TIER = decltype(tier_tag)::value;
          const float abase = ALIBI ? slope2 * (float)(ref - key0 - k0) : 0.f;
#pragma unroll
          for (int e = 0; e < GW; e += 2) {
            const float2 raw = make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1]));
            float2 y, bias = make_float2(0.f, 0.f);
            if (ALIBI) {
              if (tree) {
                const int from = ref - cur.len;
                bias.x = slope2 * (float)(from - masks.depth[(k0 + e) & (kTreeNodes - 1)]);
                bias.y = slope2 * (float)(from - masks.depth[(k0 + e + 1) & (kTreeNodes - 1)]);
              } else {
                bias = __ffma2_rn(make_float2(-slope2, -slope2), make_float2((float)e, (float)(e + 1)), make_float2(abase, abase));
              }
            }
            if (CAP) {
              if constexpr (TIER == 0) {
                y = make_float2(cap_out * tanh_of(cap_in * raw.x), cap_out * tanh_of(cap_in * raw.y));
              } else {
                float2 th;
                y = cap_logit2x2<TIER>(raw, cap_in, cap_out, &th);
              }
              if (ALIBI) y = __fadd2_rn(y, bias);
            } else {
              y = __ffma2_rn(raw, make_float2(sl2, sl2), bias);
            }
            u[e] = __float_as_uint(y.x);
            u[e + 1] = __float_as_uint(y.y);
          }
        };
        Group r[kHold ? kGroups : 1];
        float m4[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
        if (kHold) {
#pragma unroll
          for (int ch = 0; ch < kGroups; ++ch)
            if (GW * ch < used) tmem_load<GW>(tS + seg0 + GW * ch, r[kHold ? ch : 0]);
          tmem_ld_wait();
        }
#pragma unroll kUnroll
        for (int ch = 0; ch < kGroups; ++ch) {
          if (GW * ch >= used) continue;
          Group& u = r[kHold ? ch : 0];
          const int k0 = seg0 + GW * ch;
          if (!kHold) {
            tmem_load<GW>(tS + k0, u);
            tmem_ld_wait();
          }
          if (formed) {
            const int tier = CAP ? cap_tier<GW>(u, cap_in) : 0;
            if (CAP && tier == 2) form(u, k0, std::integral_constant<int, 2>{});
            else if (CAP && tier == 1) form(u, k0, std::integral_constant<int, 1>{});
            else form(u, k0, std::integral_constant<int, 0>{});
            if (masked) {
              uint32_t keep = 0;  // bit e: column k0 + e
              if (tree) {
                keep = k0 < kTreeNodes ? (uint32_t)(seen >> (k0 & 63)) : 0u;
              } else {
                const int from = min(max(lo - k0, 0), GW), to = min(max(hi - k0, 0), GW);
                if (to > from) keep = (0xffffffffu >> (32 - (to - from))) << from;
              }
#pragma unroll
              for (int e = 0; e < GW; ++e) u[e] = (keep >> e) & 1u ? u[e] : 0xff800000u;
            }
            if (!kHold) {
              tmem_store<GW>(tS + k0, u);
              tmem_st_wait();
            }
          }
#pragma unroll
          for (int e = 0; e < GW; e += 2)
            m4[(e >> 1) & 3] = fmax3(m4[(e >> 1) & 3], __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
        }
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if (!formed) mx *= sl2;
        // The row's maximum over both halves.
        mi.top[x & 1][t][h][trow] = mx;
        named_sync(4 + 4 * t + wq, 64);  // the two warps of these lanes
        mx = fmaxf(mx, mi.top[x & 1][t][h ^ 1][trow]);
        const bool grow = (mx > m + kRescaleThreshold) || (m == neg_inf() && mx != neg_inf());
        float m_new = m;
        bool rescale = false;
        if (__any_sync(0xffffffffu, grow)) {  // alike in both halves: the same rows and maxima
          m_new = fmaxf(m, mx);
          rescale = it > 0;
        }
        const float m_use = m_new == neg_inf() ? 0.f : m_new;
        const float alpha = ex2(m - m_use);
        m = m_new;
        // O may be rescaled, or added to by hand (below), once the last P·V is
        // done. NT = 2: S of this chunk was issued after it, so it is. NT = 1: S
        // was issued before it, and only what touches O waits for it; every
        // chunk waits for the one before, long done, so that no phase of the
        // barriers is passed over.
        if (NT == 2) {
          if (it > 0) ok = ok && warp_wait(bar(kODone + buf), (uint32_t)phase(x - 1), ctl);
        } else {
          if (x > 1) ok = ok && warp_wait(bar(kODone + buf), (uint32_t)phase(x - 2), ctl);
          if (rescale || (hold && it > 0)) ok = ok && warp_wait(bar(kODone + (buf ^ 1)), (uint32_t)phase(x - 1), ctl);
        }
        tc_fence_after();
        if (rescale) {
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o16[16];
            tmem_ld16(tO + 16 * i, o16);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o16[e] = __float_as_uint(__uint_as_float(o16[e]) * alpha);
            tmem_st16(tO + 16 * i, o16);
          }
          tmem_st_wait();
        }
        {
          float2 s2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 xs2 = make_float2(formed ? 1.f : sl2, formed ? 1.f : sl2), nm2 = make_float2(-m_use, -m_use);
#pragma unroll kUnroll
          for (int ch = 0; ch < kGroups; ++ch) {
            if (GW * ch >= used) continue;
            Group& u = r[kHold ? ch : 0];
            if (!kHold) {
              tmem_load<GW>(tS + seg0 + GW * ch, u);
              tmem_ld_wait();
            }
            uint32_t pk[GW / 2];
#pragma unroll
            for (int e = 0; e < GW; e += 2) {
              const float2 y = __ffma2_rn(make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])), xs2, nm2);
              const float p0 = ex2(y.x), p1 = ex2(y.y);
              s2[(e >> 1) & 1] = __fadd2_rn(s2[(e >> 1) & 1], make_float2(p0, p1));
              pk[e / 2] = pack2<BF16>(p0, p1);
            }
            tmem_store<GW / 2>(p_at(buf, h) + lane_base + (seg0 - h * HC + GW * ch) / 2, pk);
          }
          l = l * alpha + ((s2[0].x + s2[0].y) + (s2[1].x + s2[1].y));
          tmem_st_wait();
        }
        if (hold) {
          // Values that are not finite: O += p·v by hand for the rows that see
          // them, then the rows of V are cleared for the product.
          uint8_t* vt = smem + L::kOffKV + ((2 * x + 1) % NS) * L::kKV;
          tc_fence_before();
          named_sync(3, kSoft);  // all of P is stored
          tc_fence_after();
#pragma unroll 1
          for (int n = 0; n < valid; ++n) {
            if (!((mi.bad[x % 3][n >> 6] >> (n & 63)) & 1)) continue;
            const uint32_t w = tmem_ld1(p_at(buf, n / HC) + lane_base + (n % HC >> 1));
            tmem_ld_wait();
            const float pr = half_of<BF16>(w, n & 1);
#pragma unroll 1
            for (int i = 0; i < D / 32; ++i) {
              const int col = h * (D / 2) + 16 * i;
              uint32_t o16[16];
              tmem_ld16(tO + 16 * i, o16);
              tmem_ld_wait();
#pragma unroll
              for (int e8 = 0; e8 < 2; ++e8) {
                const uint4 v = *reinterpret_cast<const uint4*>(vt + (col >> 6) * (CH * 128) + sw128_offset(n, ((col & 63) >> 3) + e8));
                const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (pr != 0.f)
                    o16[8 * e8 + e] = __float_as_uint(__uint_as_float(o16[8 * e8 + e]) + pr * half_of<BF16>(vw[e >> 1], e & 1));
              }
              tmem_st16(tO + 16 * i, o16);
              tmem_st_wait();
            }
          }
          named_sync(3, kSoft);
          for (int i = sid; i < valid * 8; i += kSoft)
            if ((mi.bad[x % 3][i >> 9] >> ((i >> 3) & 63)) & 1)
#pragma unroll
              for (int sub = 0; sub < L::kSub; ++sub)
                *reinterpret_cast<uint4*>(vt + sub * (CH * 128) + (i >> 3) * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_async_shared();
          named_sync(3, kSoft);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPFull + buf));
      }

      // ------------------------------------------------------ the item ends
      mi.sum[t][h][trow] = l;
      named_sync(4 + 4 * t + wq, 64);
      l = mi.sum[t][0][trow] + mi.sum[t][1][trow];
      ok = ok && warp_wait(bar(kODone + (NT == 2 ? t : (x - 1) & 1)), (uint32_t)phase(x - 1), ctl);
      tc_fence_after();
      {
        const bool whole = cur.c == 0 && count == cur.n;
        int hq, node;
        const bool live = where(&hq, &node);
        if (masks.anc[node] == 0) l = 0.f;  // absent: chunks that are not masked were summed for it too
        // Only a row that saw nothing has l = 0, and is empty; l is NaN where a
        // logit that the row saw was NaN or +inf, and stays so, in O and LSE.
        float scale = l != 0.f ? 1.f / l : 0.f;  // of this lane's O
        if constexpr (REP == 4) {
          // The quarters' maxima and sums: weights 2^(m - top) / sum.
          if (h == 0) {
            mi.quarter[trow] = l != 0.f ? m : neg_inf();
            mi.total[seg & 1][trow] = l;
          }
          named_sync(3, kSoft);
          float top = neg_inf(), sum = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) top = fmaxf(top, mi.quarter[q * 32 + lane]);
          const float use = top == neg_inf() ? 0.f : top;
#pragma unroll
          for (int q = 0; q < 4; ++q) sum += mi.total[seg & 1][q * 32 + lane] * ex2(mi.quarter[q * 32 + lane] - use);
          scale = l != 0.f ? ex2(m - use) / sum : 0.f;
          m = top;
          l = sum;
        }
        const int64_t prow0 = ((int64_t)blockIdx.x * 2 + (cur.c > 0 ? 0 : 1)) * p.rb + t * kBM;
        const int64_t prow = prow0 + row;
        // Where the row's half goes (elements), -1: not stored.
        const bool store = ok && live;
        const int64_t place = !store ? -1 : whole ? cur.b * p.so[0] + hq * p.so[1] + node * p.so[2] : prow * p.D;
        const int d0 = h * (D / 2);
        uint16_t* og = static_cast<uint16_t*>(p.o);
        // 16 columns of O, scaled (an empty row is zero even where the values
        // that it does not see are not finite).
        auto columns = [&](int c, float* f) {
          uint32_t r[16];
          tmem_ld16(tO + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = scale != 0.f ? __uint_as_float(r[e]) * scale : 0.f;
        };
        auto put8 = [&](int64_t at, int d, const float4& x, const float4& y) {
          if (at < 0 || d >= p.D) return;
          if (whole) {
            *reinterpret_cast<uint4*>(og + at + d) =
                make_uint4(pack2<BF16>(x.x, x.y), pack2<BF16>(x.z, x.w), pack2<BF16>(y.x, y.y), pack2<BF16>(y.z, y.w));
          } else {
            *reinterpret_cast<float4*>(p.part_o + at + d) = x;
            *reinterpret_cast<float4*>(p.part_o + at + d + 4) = y;
          }
        };
        if constexpr (REP == 4) {
          // Joined in q's tile (its readers are done), D / 4 columns of each half
          // at a time: [quarter][row][16-byte unit of the row's D / 2 columns,
          // swizzled]. Every thread then adds the quarters, in their order, of
          // 8 columns of a row; threads side by side store one row's pieces.
          constexpr int kU = D / 8;
          float4* join = reinterpret_cast<float4*>(smem);
          auto unit = [&](int q, int r, int u) { return join + (q * 32 + r) * kU + (u ^ (r & 7)); };
          bool odd = false;  // columns that are not finite
#pragma unroll 1
          for (int c0 = 0; c0 < D / 2; c0 += D / 4) {
#pragma unroll
            for (int c = 0; c < D / 4; c += 16) {
              float f[16];
              columns(c0 + c, f);
#pragma unroll
              for (int e = 0; e < 16; e += 4) *unit(wq, lane, h * (kU / 2) + (c + e) / 4) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            }
            named_sync(3, kSoft);
#pragma unroll
            for (int i = sid; i < 32 * (kU / 2); i += kSoft) {  // whole warps
              const int r = i / (kU / 2), u = i % (kU / 2) * 2;
              float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float4 a = *unit(q, r, u), b = *unit(q, r, u + 1);
                x.x += a.x, x.y += a.y, x.z += a.z, x.w += a.w;
                y.x += b.x, y.y += b.y, y.z += b.z, y.w += b.w;
              }
              const int64_t at = __shfl_sync(0xffffffffu, place, r);
              // 0·x is 0, or NaN where x is not finite.
              const float probe = ((x.x + x.y) + (x.z + x.w)) * 0.f + ((y.x + y.y) + (y.z + y.w)) * 0.f;
              odd |= probe != 0.f && at >= 0;
              put8(at, u / (kU / 2) * (D / 2) + c0 + u % (kU / 2) * 4, x, y);
            }
            named_sync(3, kSoft);
          }
          if (odd) mi.odd[seg & 1] = 1;
        } else {
          // Turned in shared memory, kW columns at a time, so that lanes side by
          // side store one row's pieces (a lane per row: 32 lines a store). The
          // place is this warp's own part of q's tile: no other warp reads it,
          // or writes it before the next item's q.
          constexpr int kW = D == 64 ? 16 : 32, kUnits = kW / 4;
          uint8_t* turn = smem + t * L::kQTile + (D == 64 ? wq * 4096 + h * 2048 : h * (D / 128) * (kBM * 128) + wq * 4096);
          auto unit = [&](int r, int u) { return reinterpret_cast<float4*>(turn + r * (kW * 4) + ((u ^ r) & (kUnits - 1)) * 16); };
#pragma unroll 1
          for (int c = 0; c < D / 2; c += kW) {
            float f[kW];
#pragma unroll
            for (int e = 0; e < kW; e += 16) columns(c + e, f + e);
#pragma unroll
            for (int u = 0; u < kUnits; ++u) *unit(lane, u) = make_float4(f[4 * u], f[4 * u + 1], f[4 * u + 2], f[4 * u + 3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kW / 8; ++i) {
              const int idx = i * 32 + lane, r = idx / (kW / 8), u = idx % (kW / 8) * 2;
              put8(__shfl_sync(0xffffffffu, place, r), d0 + c + 4 * u, *unit(r, u), *unit(r, u + 1));
            }
            __syncwarp();
          }
        }
        if (store && h == 0 && (REP == 1 || wq == 0)) {
          const float l2 = l != 0.f ? m + lg2(l) : neg_inf();
          if (!whole) p.part_lse[prow] = l2;
          else if (p.lse)
            p.lse[((int64_t)cur.b * p.Hq + hq) * p.N + node] =
                l2 == neg_inf() ? l2 : l2 * kLn2 + tree_row_shift(p, hq, cur.len + masks.depth[node]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kMaskFree + (seg & 1)));
      cur.next(p, count);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (REP == 4 && warp == 3 && (mi.odd[0] | mi.odd[1]))  // the block's last two items
    for (int i = 0; i < 2; ++i)
      if (mi.odd[i]) sum_not_finite<D, BF16>(p, mi.masks[i], mi.total[i], mi.item[i], mi.count[i]);
}

constexpr uint64_t kTimeoutNs = 1000000000ull;

template <int D, int NT, int REP, bool BF16>
int launch(const TreeParams& p, int dtype, cudaStream_t st) {
  using L = TreeLayout<D, NT, REP>;
  const int box = std::gcd(p.page, L::kCH);
  CUtensorMap tm[4];
  if (!make_tmap_bhsd(&tm[0], p.kp, dtype, p.D, p.page, p.Hkv, (int)p.num_pages, p.skp, box) ||
      !make_tmap_bhsd(&tm[1], p.vp, dtype, p.D, p.page, p.Hkv, (int)p.num_pages, p.svp, box) ||
      !make_tmap_bhsd(&tm[2], p.k, dtype, p.D, p.N, p.Hkv, p.B, p.sk, 64) ||
      !make_tmap_bhsd(&tm[3], p.v, dtype, p.D, p.N, p.Hkv, p.B, p.sv, 64))
    return BFA_ERR_CUDA;
  const bool cap = p.soft_cap > 0.f, alibi = p.alibi != nullptr;
  auto kernel = cap ? (alibi ? tree_kernel<D, NT, REP, BF16, true, true> : tree_kernel<D, NT, REP, BF16, true, false>)
                    : (alibi ? tree_kernel<D, NT, REP, BF16, false, true> : tree_kernel<D, NT, REP, BF16, false, false>);
  static std::atomic<uint64_t> done[4];
  const int rc = allow_shared(kernel, (int)L::kBytes, done[2 * cap + alibi], "tree attention shared memory");
  if (rc) return rc;
  kernel<<<p.grid, L::kThreads, L::kBytes, st>>>(tm[0], tm[1], tm[2], tm[3], p, box, kTimeoutNs);
  note_launch();
  return launch_status("tree attention launch");
}

template <int D>
int launch_d(const TreeParams& p, int dtype, cudaStream_t st) {
  const bool bf16 = dtype == BFA_DTYPE_BF16;
  if (p.rb == 32) return bf16 ? launch<D, 1, 4, true>(p, dtype, st) : launch<D, 1, 4, false>(p, dtype, st);
  if constexpr (D <= 128)
    if (p.rb == 2 * kBM) return bf16 ? launch<D, 2, 1, true>(p, dtype, st) : launch<D, 2, 1, false>(p, dtype, st);
  return bf16 ? launch<D, 1, 1, true>(p, dtype, st) : launch<D, 1, 1, false>(p, dtype, st);
}

}  // namespace
}  // namespace bfa
