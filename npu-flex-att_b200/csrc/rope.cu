// rope.cu -- rotary positions on q and k in one launch, forward and transposed.
//
// Mathematics. With t the position of row (b, s) and pair i < R/2,
//   (a, b) -> (a·cos[t,i] - b·sin[t,i], a·sin[t,i] + b·cos[t,i]),
// pairs (x[i], x[i + R/2]) or (x[2i], x[2i+1]); dims >= R are copied. The
// transposed rotation (the gradient) is the same with -sin, also where the
// table carries a factor. fp32 arithmetic, one rounding to the tensor's type.
//
// Bound: HBM. Every element is read and written once (3 flops each), the table
// row of a token once per group of heads.
//
// Split. A unit is what one thread holds of a row: two 16-byte vectors that
// make whole pairs (half layout), or one (interleaved, and the copied dims).
// A thread keeps its unit's cos/sin in registers and goes over a span of heads,
// one after another; what hides the memory's latency is many resident threads:
// one head at a time in 40 registers (six blocks of 256 an SM, 32 bytes in
// flight a thread) ran at 92% of the copy rate where four heads in flight in
// 111 registers ran at 70%, and four squeezed into 64 with spills at 47%.
// Interleaved, with one vector in flight, eight blocks (31 registers): 88%
// against 81% with six. (B=4, S=4096, 32 + 8 heads of 128, bf16.)
// Rows that 16-byte vectors cannot address (strides, alignment, R/2 not a
// multiple of the vector) take the element-wise form of the same kernel, bound by
// its 2-byte accesses: 100 of the 128 dims in the half layout 202 us, a strided
// innermost dim 227, where vectors take 58 (interleaved 60).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "bfa_internal.h"

namespace bfa {
namespace {

struct RopeParams {
  const void* q; const void* k; void* qo; void* ko;
  int64_t sq[4], sk[4], sqo[4], sko[4];
  const float* cos; const float* sin;
  int64_t rows, table_stride;
  const void* pos; const void* off;
  int64_t pos_s[2];
  int pos_bytes, off_bytes;
  int B, Hq, Hk, S, D, R, units;
  int span;  // heads of a thread
  float sign;  // of sin: -1 for the transposed rotation
  int32_t* status;
};

__device__ __forceinline__ int64_t load_index(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// One 16-byte vector of T (or one element: V = 1) as fp32 and back.
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T x[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V == 1) r.x[0] = *p;
  else *reinterpret_cast<uint4*>(r.x) = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r) {
  if constexpr (V == 1) *p = r.x[0];
  else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.x);
}

// kPairs consecutive table entries, in vectors where the rows allow it (V > 1).
template <int V, int kPairs>
__device__ __forceinline__ void load_table(float (&f)[kPairs], const float* p) {
  if constexpr (V > 1 && kPairs % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kPairs; i += 4) *reinterpret_cast<float4*>(f + i) = __ldg(reinterpret_cast<const float4*>(p + i));
  } else if constexpr (V > 1 && kPairs % 2 == 0) {
#pragma unroll
    for (int i = 0; i < kPairs; i += 2) *reinterpret_cast<float2*>(f + i) = __ldg(reinterpret_cast<const float2*>(p + i));
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) f[i] = __ldg(p + i);
  }
}

// V: elements per vector access (1: element-wise, any strides).
template <typename T, bool IL, int V>
__global__ void __launch_bounds__(256, IL ? 8 : 6) rope_kernel(const RopeParams p) {
  const int idx = (int)(blockIdx.x * blockDim.x + threadIdx.x);
  if (idx >= p.S * p.units) return;
  const int s = idx / p.units, u = idx - s * p.units;
  // Units: first the turning ones, then the copied dims.
  constexpr int kTurn = (IL && V > 1) ? V : 2 * V;  // dims of a turning unit
  const int n_turn = p.R / kTurn;
  const bool turn = u < n_turn;
  constexpr int kPairs = kTurn / 2;
  // Dims of the unit's first and second vector (the second only where a
  // turning unit has one).
  constexpr bool kTwo = !IL || V == 1;
  const int d0 = !turn ? p.R + (u - n_turn) * V : IL ? u * kTurn : u * V;
  const int d1 = IL ? d0 + 1 : d0 + p.R / 2;
  const int H = p.Hq + p.Hk;
  const int first = blockIdx.y * p.span, last = min(first + p.span, H);

  for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
    alignas(16) float c[kPairs], sn[kPairs];
    if (turn) {
      int64_t t = p.pos ? load_index(p.pos, p.pos_bytes, b * p.pos_s[0] + s * p.pos_s[1]) : s;
      if (p.off) t += load_index(p.off, p.off_bytes, b);
      const bool ok = t >= 0 && t < p.rows;
      if (!ok && p.status) *p.status = BFA_ERR_INDEX;
      const int64_t at = (ok ? t : 0) * p.table_stride + u * kPairs;
      load_table<V, kPairs>(c, p.cos + at);
      load_table<V, kPairs>(sn, p.sin + at);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        c[i] = ok ? c[i] : __int_as_float(0x7fc00000);
        sn[i] = ok ? sn[i] * p.sign : __int_as_float(0x7fc00000);
      }
    }
    // The unit's place in head 0 of each tensor (rows of V > 1 have unit stride).
    const int64_t dq = d0 * (V > 1 ? 1 : p.sq[3]), dk = d0 * (V > 1 ? 1 : p.sk[3]);
    const T* q = static_cast<const T*>(p.q) + b * p.sq[0] + s * p.sq[2] + dq;
    const T* k = static_cast<const T*>(p.k) + b * p.sk[0] + s * p.sk[2] + dk;
    T* qo = static_cast<T*>(p.qo) + b * p.sqo[0] + s * p.sqo[2] + d0 * (V > 1 ? 1 : p.sqo[3]);
    T* ko = static_cast<T*>(p.ko) + b * p.sko[0] + s * p.sko[2] + d0 * (V > 1 ? 1 : p.sko[3]);
    const int step = d1 - d0;  // to the second vector
    for (int h = first; h < last; ++h) {
      const bool isq = h < p.Hq;
      const T* from = isq ? q + h * p.sq[1] : k + (h - p.Hq) * p.sk[1];
      T* to = isq ? qo + h * p.sqo[1] : ko + (h - p.Hq) * p.sko[1];
      Pack<T, V> x0 = load_pack<T, V>(from), x1;
      if (kTwo && turn) x1 = load_pack<T, V>(from + step * (V > 1 ? 1 : isq ? p.sq[3] : p.sk[3]));
      if (turn) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          T& ra = kTwo ? x0.x[i] : x0.x[(2 * i) % V];
          T& rb = kTwo ? x1.x[i] : x0.x[(2 * i + 1) % V];
          const float a = to_f32(ra), bb = to_f32(rb);
          ra = from_f32<T>(a * c[i] - bb * sn[i]);
          rb = from_f32<T>(a * sn[i] + bb * c[i]);
        }
      }
      store_pack<T, V>(to, x0);
      if (kTwo && turn) store_pack<T, V>(to + step * (V > 1 ? 1 : isq ? p.sqo[3] : p.sko[3]), x1);
    }
  }
}

bool same_place(const bfa_tensor& a, const bfa_tensor& b) {
  if (a.data != b.data) return false;
  for (int i = 0; i < 4; ++i)
    if (a.stride[i] != b.stride[i]) return false;
  return true;
}

template <typename T, bool IL, int V>
int launch_rope(RopeParams& p, bool in_place, cudaStream_t st) {
  const int turn = (IL && V > 1) ? p.R / V : p.R / (2 * V);
  p.units = turn + (in_place ? 0 : (p.D - p.R) / V);
  const int64_t per_head = (int64_t)p.S * p.units;
  if (per_head > INT32_MAX - 256) return BFA_ERR_UNSUPPORTED;
  const int64_t H = (int64_t)p.Hq + p.Hk;
  // More heads per thread (the table's values stay in registers) while two
  // full waves of threads remain.
  const int64_t wave = (int64_t)sm_count() * 2048;
  p.span = 1;
  while (p.span < H && per_head * p.B * ((H + 2 * p.span - 1) / (2 * p.span)) >= 2 * wave) p.span *= 2;
  const int threads = (int)std::min<int64_t>(256, (per_head + 31) / 32 * 32);
  const int64_t heads = (H + p.span - 1) / p.span;
  if (heads > 65535) return BFA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((per_head + threads - 1) / threads), (unsigned)heads, (unsigned)std::min(p.B, kBatchPlanes));
  rope_kernel<T, IL, V><<<grid, threads, 0, st>>>(p);
  note_launch();
  return launch_status("rope kernel launch");
}

template <typename T>
int launch_typed(RopeParams& p, const bfa_rope_args& a, cudaStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool il = a.interleaved != 0;
  const bool in_place = same_place(a.q, a.q_out) && (a.heads_k == 0 || same_place(a.k, a.k_out));
  bool vec = p.R % (il ? E : 2 * E) == 0 && p.D % E == 0 && (((uintptr_t)a.cos | (uintptr_t)a.sin) & 15u) == 0 && a.table_stride % 4 == 0;
  if (a.heads_q > 0) vec = vec && vector_rows(a.q, sizeof(T)) && vector_rows(a.q_out, sizeof(T));
  if (a.heads_k > 0) vec = vec && vector_rows(a.k, sizeof(T)) && vector_rows(a.k_out, sizeof(T));
  if (il) return vec ? launch_rope<T, true, E>(p, in_place, st) : launch_rope<T, true, 1>(p, in_place, st);
  return vec ? launch_rope<T, false, E>(p, in_place, st) : launch_rope<T, false, 1>(p, in_place, st);
}

}  // namespace
}  // namespace bfa

extern "C" int bfa_rope(const bfa_rope_args* a, void* stream) {
  using namespace bfa;
  if (!a || a->batch < 0 || a->heads_q < 0 || a->heads_k < 0 || a->seqlen < 0 || a->head_dim < 1 || a->rotary_dim < 2 ||
      a->rotary_dim % 2 != 0 || a->table_rows < 0 || (a->interleaved & ~1) || (a->inverse & ~1))
    return BFA_ERR_INVALID_ARGUMENT;
  if (a->rotary_dim > a->head_dim) return BFA_ERR_SHAPE;
  if (dtype_bytes((int)a->dtype) == 0 || a->dtype != (int)a->dtype) return BFA_ERR_UNSUPPORTED;
  if (a->batch > kMaxBatch || a->heads_q > INT32_MAX / 2 || a->heads_k > INT32_MAX / 2 || a->seqlen > INT32_MAX ||
      a->head_dim > 65536)
    return BFA_ERR_UNSUPPORTED;
  const int64_t heads = a->heads_q + a->heads_k;
  if (a->batch == 0 || a->seqlen == 0 || heads == 0) return BFA_OK;
  if (!a->cos || !a->sin || a->table_rows < 1 || (a->heads_q > 0 && (!a->q.data || !a->q_out.data)) ||
      (a->heads_k > 0 && (!a->k.data || !a->k_out.data)))
    return BFA_ERR_INVALID_ARGUMENT;
  if ((a->positions && a->positions_bytes != 4 && a->positions_bytes != 8) ||
      (a->offsets && a->offsets_bytes != 4 && a->offsets_bytes != 8))
    return BFA_ERR_INVALID_ARGUMENT;
  RopeParams p{};
  p.q = a->q.data; p.k = a->k.data; p.qo = a->q_out.data; p.ko = a->k_out.data;
  for (int i = 0; i < 4; ++i) {
    p.sq[i] = a->q.stride[i]; p.sk[i] = a->k.stride[i];
    p.sqo[i] = a->q_out.stride[i]; p.sko[i] = a->k_out.stride[i];
  }
  p.cos = a->cos; p.sin = a->sin;
  p.rows = a->table_rows; p.table_stride = a->table_stride;
  p.pos = a->positions; p.off = a->offsets;
  p.pos_s[0] = a->positions_stride[0]; p.pos_s[1] = a->positions_stride[1];
  p.pos_bytes = (int)a->positions_bytes; p.off_bytes = (int)a->offsets_bytes;
  p.B = (int)a->batch; p.Hq = (int)a->heads_q; p.Hk = (int)a->heads_k; p.S = (int)a->seqlen;
  p.D = (int)a->head_dim; p.R = (int)a->rotary_dim;
  p.sign = a->inverse ? -1.f : 1.f;
  p.status = a->status;
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case BFA_DTYPE_F32: return launch_typed<float>(p, *a, st);
    case BFA_DTYPE_F16: return launch_typed<__half>(p, *a, st);
    default: return launch_typed<__nv_bfloat16>(p, *a, st);
  }
}
