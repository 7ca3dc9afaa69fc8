// attention_few.cuh -- attention of a generation step: few query rows per sequence (group heads x its one or two tokens, at most
// 16), bound by reading the keys and values once.
//
// A tile of 256 rows would hold the rows of many sequences, of which a tile of keys concerns one: the tensor cores keep up with
// memory there, but the softmax chain of a tile (about 2400 clocks, whatever the number of rows that see it) does not. Here each
// warp takes a unit of its own: the keys that a chunk of C packed keys has of one sequence, for one KV head. Chunk c and sequence
// b that overlap have the number u = c + b (a staircase: there are at most chunks + sequences of them, and b is found from u by
// bisection), under which the unit's partial maximum, sum and output stand for join_kernel. Units do not wait for one another.
//
// A sequence may have more rows than a unit's 16 all the same (a batch with unused slots, a chunk of a prompt in one of the others).
// Its units then do not share out its keys but its rows: the i-th takes rows 16 i .. 16 i + 15 and all keys that these see.
// Rows behind the last unit's (only where there are far fewer keys than rows) are done one by one. 4 sequences of 60 tokens and
// 20000 keys each in 256 slots: 0.94 ms at D = 128 (32 / 8 heads), 1.87 at D = 256 (16 / 8); one by one all rows took 14.4 and
// 18.0, and without the unused slots, in tiles, it is 0.28 and 0.24.
//
// Per 16 keys, rows m = 16 (unused ones are zero): S = Q K^T and O += P V by mma.m16n8k16, Q in registers, K and V in a ring of
// 16-row slots that 16-byte asynchronous copies fill (rows are D * 2 bytes, 16 bytes of padding keep ldmatrix free of
// conflicts). One bulk copy per row instead took 20 to 30 clocks of the copy engine each: 3.3 TB/s at D = 128.
#pragma once

#include "attention_rows.cuh"
#include "attention_sm100.cuh"

namespace reaxmoe {
namespace attn {

constexpr int FEW_ROWS = 16, FEW_WARPS = 8, JOIN_WARPS = 8;

struct FewParams {
  reaxmoe_attention_args a;
  int group;
  int chunk;         // keys of a chunk, a multiple of 16
  int units;         // chunks + sequences
  float2* ml;        // [kv_heads][units][16]: maximum in units of log2, sum
  float* o;          // [kv_heads][units][16][D]
  // partial results over the prefix (pair_kernel's layout), or prefix_parts == 0
  int prefix_parts, prefix_rows;      // rows of one part and KV head
  const float2* prefix_ml;
  const float* prefix_o;
};

template <int D>
struct FewLayout {
  static constexpr int PITCH = D * 2 + 16;
  static constexpr int SLOT = 16 * PITCH;
  static constexpr int SLOTS = D == 256 ? 3 : 6;
  static constexpr int BLOCKS = D == 64 ? 2 : 1;            // per SM
  static constexpr int total = FEW_WARPS * SLOTS * SLOT;
  static_assert(BLOCKS * (total + 1024) <= 233472, "shared memory");
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A unit of work of one warp: keys [from, to) of one sequence for one KV head.
struct Unit {
  int u, head;
  int q0, row0, rows;        // the sequence's first query token; the unit's rows of it (for this head); rows == 0: nothing to do
  int from, to;
  int lo0, hi0, lo1, hi1;    // keys that this thread's two rows see
};

// Unit number `task`, found by the whole warp.
__device__ __forceinline__ Unit find_unit(const FewParams& p, int task, int ntok) {
  const int lane = threadIdx.x & 31, kt = (int)p.a.k_tokens;
  Unit w;
  w.u = task / p.a.kv_heads;
  w.head = task - w.u * p.a.kv_heads;
  w.row0 = w.rows = w.from = w.to = 0;
  // the last b whose first unit, cu_k[b] / chunk + b, is not beyond u
  int b = 0, len = p.a.seqs;
#pragma unroll 1
  while (len > 1) {
    const int step = (len + 31) / 32, i = lane * step;
    const bool le = i < len && min(max(__ldg(p.a.cu_k + b + i), 0), kt) / p.chunk + b + i <= w.u;
    const int n = max(__popc(__ballot_sync(0xffffffffu, le)), 1) - 1;
    const int skip = min(n * step, len - 1);
    b += skip;
    len = max(min(step, len - n * step), 1);
  }
  const int qa = __ldg(p.a.cu_q + b);
  const Sequence sq = sequence_at(p.a, b);
  const int ke = sq.ks + sq.all - (int)p.a.prefix, c = w.u - b;
  w.q0 = max(qa, 0);
  const int q1 = min(sq.q_end, ntok);
  if (sq.ks >= ke || c < sq.ks / p.chunk || c > (ke - 1) / p.chunk) return w;            // the staircase has none here
  if (w.q0 >= q1) return w;
  const int total = (q1 - w.q0) * p.group;
  const bool by_rows = total > FEW_ROWS;
  if (by_rows) w.row0 = (c - sq.ks / p.chunk) * FEW_ROWS;
  if (w.row0 >= total) return w;
  w.rows = min(total - w.row0, FEW_ROWS);
  auto token = [&](int r) { return w.q0 + (w.row0 + min(r, w.rows - 1)) / p.group; };      // of the unit's row r
  const RowKeys k0 = row_keys_in(p.a, sq, token(lane >> 2)), k1 = row_keys_in(p.a, sq, token((lane >> 2) + 8));
  w.from = row_keys_in(p.a, sq, token(0)).k_lo;
  w.to = row_keys_in(p.a, sq, token(FEW_ROWS)).k_hi;
  if (!by_rows) {
    w.from = max(c * p.chunk, w.from);
    w.to = (int)min((int64_t)(c + 1) * p.chunk, (int64_t)w.to);
  }
  w.lo0 = k0.k_lo;
  w.hi0 = min(k0.k_hi, w.to);
  w.lo1 = k1.k_lo;
  w.hi1 = min(k1.k_hi, w.to);
  return w;
}

template <int D, bool BF>
__global__ void __launch_bounds__(FEW_WARPS * 32, FewLayout<D>::BLOCKS) few_kernel(const __grid_constant__ FewParams p) {
  using L = FewLayout<D>;
  constexpr float THR = BF ? 64.0f : 11.0f;       // as in pair_kernel
  constexpr float SHIFT = BF ? 0.0f : 4.0f;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * L::SLOTS * L::SLOT;
  const int ntok = min(__ldg(p.a.cu_q + p.a.seqs), (int)p.a.q_tokens);
  const float c = p.a.scale * 1.4426950408889634f;
  int filled = 0, used = 0;                       // ring positions
  const int tasks = p.units * p.a.kv_heads;
  const int r0 = lane >> 2, r1 = r0 + 8;          // this thread's rows of the accumulators
  int task = warp * gridDim.x + blockIdx.x;
  Unit w;
  if (task < tasks) w = find_unit(p, task, ntok);
#pragma unroll 1
  while (task < tasks) {
    const int rows = w.rows, q0 = w.q0, row0 = w.row0, head = w.head, from = w.from, to = w.to;
    const int lo0 = w.lo0, hi0 = w.hi0, lo1 = w.lo1, hi1 = w.hi1;
    const int64_t at_row = ((int64_t)head * p.units + w.u) * FEW_ROWS;
    task += FEW_WARPS * gridDim.x;
    if (from >= to) {
      if (lane < rows) p.ml[at_row + lane] = make_float2(-INFINITY, 0.0f);
      if (task < tasks) w = find_unit(p, task, ntok);
      continue;
    }
    const uint16_t* kb = static_cast<const uint16_t*>(p.a.k) + head * p.a.k_head_stride;
    const uint16_t* vb = static_cast<const uint16_t*>(p.a.v) + head * p.a.v_head_stride;
    const int groups = (to - from + 15) / 16;
    // Copy i of this unit: keys (i even) or values (odd) of its 16-key group i / 2; rows behind `to` become zeros. One commit
    // group each, empty behind the last, so that SLOTS - 1 later ones may be under way when one is used.
    auto fill = [&](int i) {
      if (i < 2 * groups) {
        constexpr int PIECES = D / 8, PER = 32 / PIECES;       // 16-byte pieces of a row, rows per instruction
        const int first = from + (i >> 1) * 16 + lane / PIECES;
        const int64_t stride = (i & 1) ? p.a.v_stride : p.a.k_stride;
        const uint16_t* src = ((i & 1) ? vb : kb) + (int64_t)first * stride + (lane % PIECES) * 8;
        const uint32_t dst = ring + filled * L::SLOT + lane / PIECES * L::PITCH + lane % PIECES * 16;
#pragma unroll
        for (int x = 0; x < 16; x += PER) {
          const bool in = first + x < to;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + x * L::PITCH), "l"(in ? src : kb), "r"(in ? 16 : 0)
                       : "memory");
          src += PER * stride;
        }
      }
      if (++filled == L::SLOTS) filled = 0;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int next = 0;
#pragma unroll 1
    for (; next < L::SLOTS; ++next) fill(next);
    // Q fragments
    uint32_t q[D / 16][4];
    {
      const uint16_t* qb = static_cast<const uint16_t*>(p.a.q) + (int64_t)head * p.group * p.a.q_head_stride + (lane & 3) * 2;
      const int qr0 = row0 + r0, qr1 = row0 + r1;
      const uint16_t* qa = qb + (int64_t)(q0 + qr0 / p.group) * p.a.q_stride + (int64_t)(qr0 % p.group) * p.a.q_head_stride;
      const uint16_t* qc = qb + (int64_t)(q0 + qr1 / p.group) * p.a.q_stride + (int64_t)(qr1 % p.group) * p.a.q_head_stride;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        q[x][0] = r0 < rows ? __ldg(reinterpret_cast<const uint32_t*>(qa + x * 16)) : 0u;
        q[x][1] = r1 < rows ? __ldg(reinterpret_cast<const uint32_t*>(qc + x * 16)) : 0u;
        q[x][2] = r0 < rows ? __ldg(reinterpret_cast<const uint32_t*>(qa + x * 16 + 8)) : 0u;
        q[x][3] = r1 < rows ? __ldg(reinterpret_cast<const uint32_t*>(qc + x * 16 + 8)) : 0u;
      }
    }
    if (task < tasks) w = find_unit(p, task, ntok);      // the next one, while the first copies are under way
    float acc[D / 8][4];
#pragma unroll
    for (int x = 0; x < D / 8; ++x) acc[x][0] = acc[x][1] = acc[x][2] = acc[x][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    // the slot with the next operand, once it has landed
    auto take = [&]() {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::SLOTS - 1) : "memory");
      __syncwarp();
      const uint32_t at = ring + used * L::SLOT;
      if (++used == L::SLOTS) used = 0;
      return at;
    };
#pragma unroll 1
    for (int i = 0; i < groups; ++i) {
      uint32_t at = take();
      float s[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.0f;
        const uint32_t row = at + (h * 8 + (lane & 7)) * L::PITCH + (lane >> 3) * 16;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          uint32_t f[4];
          ldmatrix4(row + x * 64, f);
          mma16816<BF>(s[h], q[2 * x], f[0], f[1]);
          mma16816<BF>(s[h], q[2 * x + 1], f[2], f[3]);
        }
      }
      __syncwarp();
      fill(next++);
      // rows r0: s[.][0], s[.][1], r1: s[.][2], s[.][3]; keys first + 8 h + 2 (lane % 4) + {0, 1}
      const int first = from + i * 16 + (lane & 3) * 2;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = first + h * 8 + e;
          s[h][e] = j >= lo0 && j < hi0 ? s[h][e] : -INFINITY;
          s[h][2 + e] = j >= lo1 && j < hi1 ? s[h][2 + e] : -INFINITY;
        }
      float t0 = max_nan(max_nan(s[0][0], s[0][1]), max_nan(s[1][0], s[1][1]));
      float t1 = max_nan(max_nan(s[0][2], s[0][3]), max_nan(s[1][2], s[1][3]));
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        t0 = max_nan(t0, __shfl_xor_sync(0xffffffffu, t0, o));
        t1 = max_nan(t1, __shfl_xor_sync(0xffffffffu, t1, o));
      }
      t0 *= c;
      t1 *= c;
      const bool g0 = t0 - m0 > THR, g1 = t1 - m1 > THR;
      const bool x0 = g0 && m0 != -INFINITY, x1 = g1 && m1 != -INFINITY;
      if (__any_sync(0xffffffffu, x0 || x1)) {
        const float f0 = x0 ? ex2(m0 - t0) : 1.0f, f1 = x1 ? ex2(m1 - t1) : 1.0f;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          acc[x][0] *= f0;
          acc[x][1] *= f0;
          acc[x][2] *= f1;
          acc[x][3] *= f1;
        }
      }
      if (g0) m0 = t0;
      if (g1) m1 = t1;
      const float mc0 = (m0 == -INFINITY ? 0.0f : m0) - SHIFT, mc1 = (m1 == -INFINITY ? 0.0f : m1) - SHIFT;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[h][e] = ex2(fmaf(s[h][e], c, -mc0));
          s[h][2 + e] = ex2(fmaf(s[h][2 + e], c, -mc1));
        }
      l0 += (s[0][0] + s[0][1]) + (s[1][0] + s[1][1]);
      l1 += (s[0][2] + s[0][3]) + (s[1][2] + s[1][3]);
      const uint32_t pw[4] = {pack2<BF>(s[0][0], s[0][1]), pack2<BF>(s[0][2], s[0][3]), pack2<BF>(s[1][0], s[1][1]),
                             pack2<BF>(s[1][2], s[1][3])};
      at = take();
      const uint32_t row = at + (lane & 15) * L::PITCH + (lane >> 4) * 16;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        uint32_t f[4];
        ldmatrix4_trans(row + x * 32, f);
        mma16816<BF>(acc[2 * x], pw, f[0], f[1]);
        mma16816<BF>(acc[2 * x + 1], pw, f[2], f[3]);
      }
      __syncwarp();
      fill(next++);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    if ((lane & 3) == 0) {
      if (r0 < rows) p.ml[at_row + r0] = make_float2(m0, l0);
      if (r1 < rows) p.ml[at_row + r1] = make_float2(m1, l1);
    }
    float* o = p.o + at_row * D + (lane & 3) * 2;
#pragma unroll
    for (int x = 0; x < D / 8; ++x) {
      if (r0 < rows) *reinterpret_cast<float2*>(o + r0 * D + x * 8) = make_float2(acc[x][0], acc[x][1]);
      if (r1 < rows) *reinterpret_cast<float2*>(o + r1 * D + x * 8) = make_float2(acc[x][2], acc[x][3]);
    }
  }
}

// Joins the units (and the prefix's parts) of a row by JW warps: 8 (a block) where a row has many partial results, else one. The
// factors of up to 32 JW partial results are worked out together, then the warps add these up, whose loads do not depend on one
// another. (256 sequences with 6 results a row: 22.8 us with 8 warps a row.)
template <int D, bool BF, int JW>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const __grid_constant__ FewParams p) {
  static_assert(JW == 1 || JW == JOIN_WARPS, "a warp or a block a row");
  constexpr float SHIFT = BF ? 0.0f : 4.0f;
  constexpr int W = D / 32, N = JW * 32;
  __shared__ float red[JW == 1 ? 1 : JW][D + 2];
  __shared__ float factor[JOIN_WARPS * 32];
  const int lane = threadIdx.x & 31, warp = JW == 1 ? 0 : threadIdx.x >> 5;       // warp of the row
  const int t = JW == 1 ? lane : threadIdx.x;                                     // thread of the row
  float* const factors = factor + (JW == 1 ? (threadIdx.x >> 5) * 32 : 0);
  const int id = JW == 1 ? blockIdx.x * JOIN_WARPS + (threadIdx.x >> 5) : blockIdx.x;
  const int tok = id / p.a.q_heads, head = id - tok * p.a.q_heads;
  auto sync = [] {
    if constexpr (JW == 1) __syncwarp(); else __syncthreads();
  };
  const int ntok = min(__ldg(p.a.cu_q + p.a.seqs), (int)p.a.q_tokens);
  if (tok >= ntok) return;
  const int b = sequence_by_warp(p.a, tok);
  const Sequence sq = sequence_at(p.a, b);
  const int q0 = max(__ldg(p.a.cu_q + b), 0), q1 = min(sq.q_end, ntok);
  const int kvh = head / p.group, row = (tok - q0) * p.group + head - kvh * p.group;
  const int ke = sq.ks + sq.all - (int)p.a.prefix;
  const int first = sq.ks / p.chunk + b, units = sq.ks < ke ? (ke - 1) / p.chunk + b - first + 1 : 0;
  const bool inside = tok >= q0 && tok < q1;         // (not where the lengths do not rise from 0)
  const bool by_rows = inside && (q1 - q0) * p.group > FEW_ROWS;
  if (!inside || (by_rows && units > 0 && row / FEW_ROWS >= units)) {
    if (warp == 0) row_by_warp<D, BF>(p.a, tok, head, true);
    return;
  }
  const int own = by_rows ? min(units, 1) : units, unit = first + (by_rows ? row / FEW_ROWS : 0);
  const int n = own + p.prefix_parts;
  // partial result i of n: the units of the row's own keys, then the prefix's parts
  const int64_t unit0 = ((int64_t)kvh * p.units + unit) * FEW_ROWS + row % FEW_ROWS;
  const int64_t part0 = (int64_t)kvh * p.prefix_rows + (int64_t)tok * p.group + head - kvh * p.group;
  const int64_t part_step = (int64_t)p.a.kv_heads * p.prefix_rows;
  auto ml = [&](int i) { return i < own ? p.ml[unit0 + (int64_t)i * FEW_ROWS] : p.prefix_ml[part0 + (i - own) * part_step]; };
  auto o = [&](int i) { return (i < own ? p.o + (unit0 + (int64_t)i * FEW_ROWS) * D : p.prefix_o + (part0 + (i - own) * part_step) * D) + lane * 2; };
  float m = -INFINITY;
  for (int i = t; i < n; i += N) m = fmaxf(m, ml(i).x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  if constexpr (JW > 1) {
    if (lane == 0) red[warp][0] = m;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < JW; ++x) m = fmaxf(m, red[x][0]);
  }
  float l = 0.0f, acc[W];
#pragma unroll
  for (int x = 0; x < W; ++x) acc[x] = 0.0f;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += N) {
    sync();
    const int count = min(n - i0, N);
    if (t < count) {
      const float2 v = ml(i0 + t);
      // -1: none of the row's keys, or scores of -inf alone; its output is not read
      const bool empty = v.x == -INFINITY && v.y == 0.0f;
      const float f = empty ? -1.0f : (v.x == m ? 1.0f : ex2(v.x - m));
      factors[t] = f;
      if (!empty) l = fmaf(v.y, f, l);
    }
    sync();
    // four results at a time: all their loads, then the sums
#pragma unroll 1
    for (int i = warp; i < count; i += 4 * JW) {
      float2 y[4][W / 2];
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = i + e * JW;
        f[e] = at < count ? factors[at] : -1.0f;
        const float* src = o(i0 + min(at, count - 1));
#pragma unroll
        for (int x = 0; x < W / 2; ++x) {
          y[e][x] = make_float2(0.0f, 0.0f);
          if (f[e] != -1.0f) y[e][x] = *reinterpret_cast<const float2*>(src + x * 64);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < W / 2; ++x) {
          acc[2 * x] = fmaf(y[e][x].x, f[e], acc[2 * x]);
          acc[2 * x + 1] = fmaf(y[e][x].y, f[e], acc[2 * x + 1]);
        }
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  if constexpr (JW > 1) {
    __syncthreads();
#pragma unroll
    for (int x = 0; x < W; x += 2) {
      red[warp][lane * 2 + x * 32] = acc[x];
      red[warp][lane * 2 + x * 32 + 1] = acc[x + 1];
    }
    if (lane == 0) red[warp][D] = l;
    __syncthreads();
    if (warp != 0) return;
    auto sum = [&](int at) {
      float v = red[0][at];
#pragma unroll
      for (int x = 1; x < JW; ++x) v += red[x][at];
      return v;
    };
    l = sum(D);
#pragma unroll
    for (int x = 0; x < W; x += 2) {
      acc[x] = sum(lane * 2 + x * 32);
      acc[x + 1] = sum(lane * 2 + x * 32 + 1);
    }
  }
  const RowKeys rk = row_keys_in(p.a, sq, tok);
  const bool none = rk.p_lo >= rk.p_hi && rk.k_lo >= rk.k_hi;
  const float inv = none ? 0.0f : 1.0f / l;
  uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.a.out) + (int64_t)tok * p.a.out_stride + head * p.a.out_head_stride);
  bool bad = false;
  uint32_t packed[W / 2];
#pragma unroll
  for (int x = 0; x < W; x += 2) {
    const float y0 = none ? 0.0f : in_range<BF>(acc[x] * inv), y1 = none ? 0.0f : in_range<BF>(acc[x + 1] * inv);
    bad |= !(fabsf(y0) < INFINITY) || !(fabsf(y1) < INFINITY);
    packed[x / 2] = pack2<BF>(y0, y1);
  }
#pragma unroll
  for (int x = 0; x < W / 2; ++x) out[lane + x * 32] = packed[x];
  if (p.a.lse != nullptr && lane == 0)
    p.a.lse[(int64_t)tok * p.a.q_heads + head] = none ? -INFINITY : (m - SHIFT + __log2f(l)) * 0.6931471805599453f;
  __syncwarp();
  if (__any_sync(0xffffffffu, bad) && l == l) row_by_warp<D, BF>(p.a, tok, head, false);     // (pair_kernel)
}

}  // namespace attn
}  // namespace reaxmoe
