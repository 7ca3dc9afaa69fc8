// attention_rows.cuh -- what an attention row sees, and one row computed by one warp.
//
// Sequence b has query rows [cu_q[b], cu_q[b+1]) and own keys [cu_k[b], cu_k[b+1]) behind `prefix` shared keys. Row i of m
// stands at t = prefix + n - m + i of the virtual key axis (prefix, then the n own keys) and sees [lo, hi) of it: hi = t + 1
// (causal) or all, lo = t - window + 1 with a window, both cut to [0, prefix + n].
#pragma once

#include <climits>

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
// are cut to the tensors here and a row's distance to its sequence's end to at least 1 below, so that no value of theirs (a first
// one that is not 0, falling or negative ones) makes a later access leave the tensors.
struct Sequence {
  int ks, all, q_end;
};
__device__ __forceinline__ Sequence sequence_at(const reaxmoe_attention_args& a, int b) {
  const int kt = (int)a.k_tokens;
  Sequence s;
  s.ks = min(max(__ldg(a.cu_k + b), 0), kt);
  s.all = (int)a.prefix + min(max(__ldg(a.cu_k + b + 1), s.ks), kt) - s.ks;
  s.q_end = min(max(__ldg(a.cu_q + b + 1), 0), (int)a.q_tokens);
  return s;
}

// Keys that its query token t sees.
__device__ __forceinline__ RowKeys row_keys_in(const reaxmoe_attention_args& a, const Sequence& s, int t) {
  const int P = (int)a.prefix;
  const int pos = s.all - max(s.q_end - t, 1);                   // prefix + n - m + i
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

// An output before it is rounded. It is an average of values, but weights that were rounded up to 16 bits before the product may
// lift it by 2^-11: past fp16's largest value (65504), it is that value. (bf16 ends where fp32 does.)
template <bool BF>
__device__ __forceinline__ float in_range(float v) {
  if constexpr (BF) return v;
  return fabsf(v) < 66000.0f ? fminf(fmaxf(v, -65504.0f), 65504.0f) : v;
}

// One row by one warp, 32 keys at a time: lane = key for the scores, lane l = elements [l D/32, (l+1) D/32) for the sums. It
// reads the keys that the row sees and no others, which tiles of keys cannot: there a key that a row does not see has weight
// 0, and 0 x (an infinity or NaN of its value) is NaN.
// all: the whole row; else only those elements of it whose value in `out` (already written) is not finite. These are done again
// until none of them can become finite any more: then the values that are not finite are of keys that the row does see, and
// `out` stays as it is (an infinity in a key that many rows see would take minutes otherwise).
// alive(): called by the whole warp every 32 keys.
struct NoSign {
  __device__ __forceinline__ void operator()() const {}
};
template <int D, bool BF, typename Alive = NoSign>
__device__ __forceinline__ void row_by_warp(const reaxmoe_attention_args& a, int t, int head, bool all, Alive alive = Alive()) {
  constexpr int W = D / 64;                      // 32-bit words per lane
  const int lane = threadIdx.x & 31;
  const int kvh = head / (a.q_heads / a.kv_heads);
  const RowKeys rk = row_keys(a, t);
  uint32_t* po = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_stride + head * a.out_head_stride) + lane * W;
  const uint4* pq = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (int64_t)t * a.q_stride + head * a.q_head_stride);
  bool again[2 * W];
  float acc[2 * W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    float2 v = make_float2(NAN, NAN);
    if (!all) v = unpack2<BF>(*reinterpret_cast<volatile uint32_t*>(po + i));
    again[2 * i] = !(fabsf(v.x) < INFINITY);
    again[2 * i + 1] = !(fabsf(v.y) < INFINITY);
    acc[2 * i] = acc[2 * i + 1] = 0.0f;
  }
  const float c = a.scale * 1.4426950408889634f;  // scores in units of log2
  float m = -INFINITY, l = 0.0f;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const uint16_t* kb = static_cast<const uint16_t*>(part == 0 ? a.prefix_k : a.k) + kvh * (part == 0 ? a.prefix_k_head_stride : a.k_head_stride);
    const uint16_t* vb = static_cast<const uint16_t*>(part == 0 ? a.prefix_v : a.v) + kvh * (part == 0 ? a.prefix_v_head_stride : a.v_head_stride);
    const int64_t ks = part == 0 ? a.prefix_k_stride : a.k_stride, vs = part == 0 ? a.prefix_v_stride : a.v_stride;
    const int lo = part == 0 ? rk.p_lo : rk.k_lo, hi = part == 0 ? rk.p_hi : rk.k_hi;
#pragma unroll 1
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int n = min(32, hi - j0);
      alive();
      float w;
      {
        float s = -INFINITY;
        if (lane < n) {
          const uint4* pk = reinterpret_cast<const uint4*>(kb + (int64_t)(j0 + lane) * ks);
          s = 0.0f;
#pragma unroll 4
          for (int i = 0; i < D / 8; ++i) {
            const uint4 q4 = __ldg(pq + i), k4 = __ldg(pk + i);
            const uint32_t qw[4] = {q4.x, q4.y, q4.z, q4.w}, kw[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 qf = unpack2<BF>(qw[e]), kf = unpack2<BF>(kw[e]);
              s = fmaf(qf.x, kf.x, fmaf(qf.y, kf.y, s));
            }
          }
          s *= c;
        }
        float top = s;                            // NaN where a score is
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float x = __shfl_xor_sync(0xffffffffu, top, o);
          top = (top != top || x != x) ? NAN : fmaxf(top, x);
        }
        const float mn = (top != top || m != m) ? NAN : fmaxf(m, top);
        const float base = mn == -INFINITY ? 0.0f : mn, f = m == mn ? 1.0f : exp2f(m - base);
        w = lane < n ? exp2f(s - base) : 0.0f;
        float sum = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        m = mn;
        l = l * f + sum;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) acc[i] *= f;
      }
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const uint32_t* pv = reinterpret_cast<const uint32_t*>(vb + (int64_t)(j0 + j) * vs) + lane * W;
        const float wj = __shfl_sync(0xffffffffu, w, j);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float2 v = unpack2<BF>(__ldg(pv + i));
          acc[2 * i] = fmaf(wj, v.x, acc[2 * i]);
          acc[2 * i + 1] = fmaf(wj, v.y, acc[2 * i + 1]);
        }
      }
      if (!all) {
        bool over = true;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) over &= !again[i] || !(fabsf(acc[i]) < INFINITY);
        if (__all_sync(0xffffffffu, over)) return;
      }
    }
  }
  const bool none = rk.p_lo >= rk.p_hi && rk.k_lo >= rk.k_hi;
  const float inv = none ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float2 old = all ? make_float2(0.0f, 0.0f) : unpack2<BF>(*reinterpret_cast<volatile uint32_t*>(po + i));
    po[i] = pack2<BF>(again[2 * i] ? acc[2 * i] * inv : old.x, again[2 * i + 1] ? acc[2 * i + 1] * inv : old.y);
  }
  if (all && a.lse != nullptr && lane == 0)
    a.lse[(int64_t)t * a.q_heads + head] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Of a warp's rows (lane = row, all of one KV head; bit = row) whose elements in `out` are not all finite: those where some element
// is not for another reason than a value that the row sees, so that row_by_warp may still find it finite. One pass over the
// values that the rows see together, in blocks of 1024 keys: for each element the first and the last key of the block that is
// not finite there; it ends when no row is left. (Where one infinity is seen by thousands of rows, row_by_warp would go over all
// keys up to it for each of them: a prompt of 8192 tokens with one in the middle took 97 ms at D = 128, 0.7 without it, and
// takes 2.4.)
template <int D, bool BF, typename Alive>
__device__ __forceinline__ uint32_t unexplained_rows(const reaxmoe_attention_args& a, uint32_t rows, int tok, int head, Alive alive) {
  constexpr int W = D / 64, BLOCK = 1024;        // 32-bit words per lane
  constexpr uint32_t EXP = BF ? 0x7F807F80u : 0x7C007C00u;      // exponent bits: all ones where not finite
  const int lane = threadIdx.x & 31;
  const int kvh = __shfl_sync(0xffffffffu, head, __ffs(rows) - 1) / (a.q_heads / a.kv_heads);
  RowKeys rk = {0, 0, 0, 0};
  if ((rows >> lane) & 1u) rk = row_keys(a, tok);
  uint32_t explained[2 * W];                     // this lane's elements of a row (bit)
#pragma unroll
  for (int i = 0; i < 2 * W; ++i) explained[i] = 0u;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const uint16_t* vb = static_cast<const uint16_t*>(part == 0 ? a.prefix_v : a.v) + kvh * (part == 0 ? a.prefix_v_head_stride : a.v_head_stride);
    const int64_t vs = part == 0 ? a.prefix_v_stride : a.v_stride;
    const int lo = part == 0 ? rk.p_lo : rk.k_lo, hi = part == 0 ? rk.p_hi : rk.k_hi;
    const int from = __reduce_min_sync(0xffffffffu, lo < hi ? lo : INT_MAX), to = __reduce_max_sync(0xffffffffu, lo < hi ? hi : 0);
#pragma unroll 1
    for (int j0 = from; j0 < to; j0 += BLOCK) {
      const int end = min(to - j0, BLOCK);       // behind the block's last key, from j0
      int first[2 * W], last[2 * W];
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) {
        first[i] = BLOCK;
        last[i] = -1;
      }
      bool some = false;
#pragma unroll 1
      for (int j = 0; j < end; j += 8) {
        if ((j & 31) == 0) alive();
        uint32_t v[8][W];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t* pv = reinterpret_cast<const uint32_t*>(vb + (int64_t)(j0 + min(j + x, end - 1)) * vs) + lane * W;
#pragma unroll
          for (int i = 0; i < W; ++i) v[x][i] = __ldg(pv + i) & EXP;
        }
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) {
            const int at = min(j + x, end - 1);
            if (((v[x][i / 2] >> (i % 2 * 16)) & 0xFFFFu) == (EXP & 0xFFFFu)) {
              first[i] = min(first[i], at);
              last[i] = at;
              some = true;
            }
          }
      }
      if (!__any_sync(0xffffffffu, some)) continue;
#pragma unroll 1
      for (uint32_t left = rows; left != 0u; left &= left - 1u) {
        const int r = __ffs(left) - 1;
        const int rlo = __shfl_sync(0xffffffffu, lo, r) - j0, rhi = __shfl_sync(0xffffffffu, hi, r) - j0;
        const int t = __shfl_sync(0xffffffffu, tok, r), h = __shfl_sync(0xffffffffu, head, r);
        const volatile uint32_t* po = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.out) + (int64_t)t * a.out_stride + h * a.out_head_stride) + lane * W;
        bool open = false;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          if ((first[i] >= rlo && first[i] < min(rhi, BLOCK)) || (last[i] >= max(rlo, 0) && last[i] < rhi)) explained[i] |= 1u << r;
          open |= ((po[i / 2] >> (i % 2 * 16)) & EXP & 0xFFFFu) == (EXP & 0xFFFFu) && ((explained[i] >> r) & 1u) == 0u;
        }
        if (!__any_sync(0xffffffffu, open)) rows &= ~(1u << r);
      }
      if (rows == 0u) return 0u;
    }
  }
  return rows;
}

}  // namespace attn
}  // namespace reaxmoe
