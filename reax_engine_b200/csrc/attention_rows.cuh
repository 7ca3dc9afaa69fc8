// attention_rows.cuh -- what an attention row sees, and one row computed by one warp.
//
// Sequence b has query rows [cu_q[b], cu_q[b+1]) and own keys [cu_k[b], cu_k[b+1]) behind `prefix` shared keys. Row i of m
// stands at t = prefix + n - m + i of the virtual key axis (prefix, then the n own keys) and sees [lo, hi) of it: hi = t + 1
// (causal) or all, lo = t - window + 1 with a window, both cut to [0, prefix + n].
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace reaxmoe {
namespace attn {

struct RowKeys {
  int p_lo, p_hi;   // prefix keys seen
  int k_lo, k_hi;   // keys of the packed k / v seen (row numbers of the packed tensors)
};

// the last b of [b0, b1) with cu_q[b] <= t (sequences of no rows are passed over); t < cu_q[b1]
__device__ __forceinline__ int sequence_of(const reaxmoe_attention_args& a, int t, int b0, int b1) {
#pragma unroll 1
  while (b1 - b0 > 1) {
    const int mid = (b0 + b1) >> 1;
    if (__ldg(a.cu_q + mid) <= t) b0 = mid; else b1 = mid;
  }
  return b0;
}

// the same of all sequences by a whole warp, 32 at a time
__device__ __forceinline__ int sequence_by_warp(const reaxmoe_attention_args& a, int t) {
  const int lane = threadIdx.x & 31;
  int b0 = 0, len = a.seqs;
#pragma unroll 1
  while (len > 1) {
    const int step = (len + 31) / 32, i = lane * step;
    const bool le = i < len && __ldg(a.cu_q + b0 + i) <= t;
    const int c = max(__popc(__ballot_sync(0xffffffffu, le)), 1) - 1;
    b0 += min(c * step, len - 1);
    len = max(min(step, len - c * step), 1);
  }
  return b0;
}

// A sequence: its first own key, prefix and own keys together, and the token behind its last query row. The cumulative lengths
// are cut to the tensors, so that no value of theirs makes a later access leave them.
struct Sequence {
  int ks, all, q_end;
};
__device__ __forceinline__ Sequence sequence_at(const reaxmoe_attention_args& a, int b) {
  const int kt = (int)a.k_tokens;
  Sequence s;
  s.ks = min(max(__ldg(a.cu_k + b), 0), kt);
  s.all = (int)a.prefix + min(max(__ldg(a.cu_k + b + 1), s.ks), kt) - s.ks;
  s.q_end = __ldg(a.cu_q + b + 1);
  return s;
}

// Keys that its query token t sees.
__device__ __forceinline__ RowKeys row_keys_in(const reaxmoe_attention_args& a, const Sequence& s, int t) {
  const int P = (int)a.prefix;
  const int pos = s.all - (s.q_end - t);                         // prefix + n - m + i
  const int hi = a.causal ? min(max(pos, -1) + 1, s.all) : s.all;
  const int lo = a.window > 0 && pos >= a.window ? min(pos - a.window + 1, hi) : 0;
  RowKeys r;
  r.p_lo = min(lo, P);
  r.p_hi = min(hi, P);
  r.k_lo = s.ks + max(lo - P, 0);
  r.k_hi = s.ks + max(hi - P, 0);
  return r;
}
__device__ __forceinline__ RowKeys row_keys_of(const reaxmoe_attention_args& a, int b, int t) {
  return row_keys_in(a, sequence_at(a, b), t);
}
__device__ __forceinline__ RowKeys row_keys(const reaxmoe_attention_args& a, int t) {
  return row_keys_of(a, sequence_of(a, t, 0, a.seqs), t);
}

template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);    // one conversion instruction for the pair
    return *reinterpret_cast<const uint32_t*>(&b);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One row by one warp, lane l holding elements [l D/32, (l+1) D/32): scores in fp32, running maximum and sum, key by key. It
// reads the keys that the row sees and no others, which the tensor-core kernel cannot do where a tile of keys ends inside
// what a row sees: there a masked key has weight 0, and 0 x (an infinity or NaN of its value) would be NaN.
template <int D, bool BF>
__device__ __forceinline__ void row_by_warp(const reaxmoe_attention_args& a, int t, int head) {
  constexpr int W = D / 64;                      // 32-bit words per lane
  const int lane = threadIdx.x & 31;
  const int kvh = head / (a.q_heads / a.kv_heads);
  const RowKeys rk = row_keys(a, t);
  auto load = [&](const void* base, int64_t row, int64_t stride, int64_t hs, int h, float2 (&f)[W]) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(base) + row * stride + h * hs) + lane * W;
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = unpack2<BF>(__ldg(p + i));
  };
  float2 q[W], acc[W];
  load(a.q, t, a.q_stride, a.q_head_stride, head, q);
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = make_float2(0.0f, 0.0f);
  const float c = a.scale * 1.4426950408889634f;  // scores in units of log2
  float m = -INFINITY, l = 0.0f;
  auto keys = [&](const void* kb, int64_t ks, int64_t khs, const void* vb, int64_t vs, int64_t vhs, int lo, int hi) {
#pragma unroll 1
    for (int j = lo; j < hi; ++j) {
      float2 k[W], v[W];
      load(kb, j, ks, khs, kvh, k);
      load(vb, j, vs, vhs, kvh, v);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) s = fmaf(q[i].x, k[i].x, fmaf(q[i].y, k[i].y, s));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= c;
      // a NaN score stays one: fmaxf would drop it
      const float mn = (s != s) ? s : fmaxf(m, s);
      const float f = m == mn ? 1.0f : exp2f(m - mn);
      const float p = s == mn && fabsf(s) != INFINITY ? 1.0f : exp2f(s - mn);
      m = mn;
      l = l * f + p;
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] = make_float2(fmaf(acc[i].x, f, p * v[i].x), fmaf(acc[i].y, f, p * v[i].y));
    }
  };
  keys(a.prefix_k, a.prefix_k_stride, a.prefix_k_head_stride, a.prefix_v, a.prefix_v_stride, a.prefix_v_head_stride, rk.p_lo,
       rk.p_hi);
  keys(a.k, a.k_stride, a.k_head_stride, a.v, a.v_stride, a.v_head_stride, rk.k_lo, rk.k_hi);
  const bool none = rk.p_lo >= rk.p_hi && rk.k_lo >= rk.k_hi;
  const float inv = none ? 0.0f : 1.0f / l;
  uint32_t* po = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_stride + head * a.out_head_stride) + lane * W;
#pragma unroll
  for (int i = 0; i < W; ++i) po[i] = pack2<BF>(acc[i].x * inv, acc[i].y * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[(int64_t)t * a.q_heads + head] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace attn
}  // namespace reaxmoe
