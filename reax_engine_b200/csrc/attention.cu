// attention.cu -- attention over packed sequences and over a prefix that a batch shares (reaxmoe_attention), on the tensor
// cores of CTA pairs.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(c s_ij - c m_i),  c = scale log2(e),  s_ij = q_i . k_j over the keys j that
//   row i sees, m_i a running maximum (one pass over the keys; o and the sum are rescaled when it grows).
//
// Rows. Query head h of KV head g reads the same keys as its group's other heads, so the rows of KV head g are (token, head of
// the group) pairs, row = token * group + h % group, over ALL packed tokens: a tile of 256 consecutive rows (128 in each CTA of
// a pair) may end one sequence, hold others whole and begin the next. What a row sees is two ranges of keys (of the prefix and
// of its own sequence), a tile goes over the union of its rows' ranges, and the mask of a row is two comparisons with its
// range. Packing rows across sequences is what computes a shared prefix once for a batch of short continuations, and it reads
// the keys of a batch of single tokens once per KV head; for long prompts it costs nothing over tiles that stop at a sequence's
// end (the union of two sequences' ranges is what two tiles would read).
//
// A pair multiplies M = 256 rows (cta_group::2): each CTA holds 128 rows of Q and all accumulator columns of its rows, and
// half of every K and V tile, which halves the bytes that shared memory and L2 have to deliver per product against a CTA
// alone. Per tile of 128 keys
//   S = Q K^T          [256 x 128], Q and K from shared memory (128-byte swizzle, K-major);
//   P = exp2(c S - c m) by 8 warps per CTA, packed to 16 bits over the first half of S's own TMEM columns;
//   O += P V           [256 x D], P from TMEM, V from shared memory as it lies in memory (MN-major).
// S is double-buffered (2 x 128 columns) beside O (D columns): the tensor core multiplies S(j + 1) while the softmax of tile j
// runs, and the next item's first two S while this item's O is written out.
//
//   warps 0..7    softmax: TMEM lane quarter w % 4 (thread = row), column half w / 4; the halves of a row meet in shared memory
//   warp 8        K / V producer: ring of slots, alternately half a K tile (64 keys x D) and half a V tile (128 keys x D / 2)
//   warp 9        allocates TMEM; in the leader CTA one thread issues all MMAs of the pair
//   warps 10..13  loader: takes the next item, works out its key ranges, copies its Q rows
// Items (row tile, KV head, part of the keys) are taken in order, the first by pair number, further ones from a counter.
// With few rows an item's keys are split over several pairs, which leave partial sums that combine_kernel joins.
// All waits are bounded (globaltimer); a timeout records REAXMOE_ERR_DEVICE_TIMEOUT and the CTA winds down.
#include <cstring>

#include "attention_rows.cuh"
#include "attention_sm100.cuh"
#include "kernels.cuh"

namespace reaxmoe {
namespace attn {

constexpr int ROWS = 128;                 // query rows per CTA
constexpr int KT = 128;                   // keys per tile
constexpr int SM_WARPS = 8;               // softmax warps
constexpr int LD_WARP0 = 10, LD_WARPS = 4;
constexpr int THREADS = (LD_WARP0 + LD_WARPS) * 32;
constexpr int O_COL = 2 * KT;             // TMEM columns: S0, S1, O

template <int D>
struct Layout {
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int SLOT = 64 * D * 2;                   // half a K tile or half a V tile
  static constexpr int SLOTS = D == 256 ? 5 : 8;
  static constexpr int ring = Q_BYTES;
  static constexpr int xchg = ring + SLOTS * SLOT;          // [2][2][ROWS] floats: what the column halves of a row exchange
  static constexpr int bars = xchg + 4 * ROWS * 4;
  static constexpr int total = bars + 1024;
  static_assert(total <= 232448, "shared memory");
};

struct ItemInfo {
  int row0;          // first row of the pair's tile; -1: no more items
  int head, part;    // KV head, part of the keys
  int p_lo, p_hi;    // prefix keys of this part
  int o_lo, o_hi;    // own keys of this part
  int gap;           // keys that no row sees may lie between those of two sequences
};

struct Params {
  CUtensorMap tmK, tmV, tmPK, tmPV;
  reaxmoe_attention_args a;
  int group;
  int tiles, parts, items;
  int* counter;      // items taken beyond the first of each pair (null when there are none)
  float* part_o;     // [parts][kv_heads][tiles * 256][D]
  float2* part_ml;   // [parts][kv_heads][tiles * 256]: maximum in units of log2, sum
  unsigned long long timeout_ns;
};

__device__ __forceinline__ int row_count(const Params& p) {
  const int t = min(__ldg(p.a.cu_q + p.a.seqs), (int)p.a.q_tokens);
  return max(t, 0) * p.group;
}

// The tiles of an item in order: prefix tiles, then own tiles, each 128 keys from `start`. Where own keys that no row sees may
// lie between (gap), tiles begin at the first key that some row still needs; that is found by walking the tile's sequences.
struct TileIter {
  int pc, ph, oc, oh;
  int b, b_end, t0, t1, lo, hi;
  bool gap;
  __device__ __forceinline__ void need(const reaxmoe_attention_args& a) {
    const int q0 = __ldg(a.cu_q + b), q1 = __ldg(a.cu_q + b + 1);
    const int f = max(t0, q0), l = min(t1, q1) - 1;
    lo = 0;
    hi = 0;
    if (f <= l) {
      lo = row_keys_of(a, b, f).k_lo;
      hi = row_keys_of(a, b, l).k_hi;
    }
  }
  __device__ __forceinline__ void init(const Params& p, const ItemInfo& it) {
    pc = it.p_lo;
    ph = it.p_hi;
    oc = it.o_lo;
    oh = it.o_hi;
    gap = it.gap != 0;
    if (gap) {
      t0 = it.row0 / p.group;
      t1 = (min(it.row0 + 2 * ROWS, row_count(p)) - 1) / p.group + 1;
      b = sequence_of(p.a, t0);
      b_end = sequence_of(p.a, t1 - 1);
      need(p.a);
    }
  }
  __device__ __forceinline__ bool next(const Params& p, int& start, bool& pre) {
    if (pc < ph) {
      start = pc;
      pre = true;
      pc += KT;
      return true;
    }
    pre = false;
    if (gap) {
      while (hi <= oc) {
        if (b >= b_end) return false;
        ++b;
        need(p.a);
      }
      oc = max(oc, lo);
    }
    if (oc >= oh) return false;
    start = oc;
    oc += KT;
    return true;
  }
};

// MN-major V tile: 128-byte swizzle with 64-dim blocks 16 KiB apart (LBO) and 8-key groups 1024 bytes apart (SBO); for D = 64 a
// CTA's half is 32 dims wide: 64-byte swizzle, 8-key groups 512 bytes apart.
template <int D>
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
  const uint64_t base = (uint64_t)((saddr >> 4) & 0x3FFF) | (1ull << 46);
  if constexpr (D == 64) return base | (1ull << 16) | ((uint64_t)(512 >> 4) << 32) | (4ull << 61);
  return base | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (2ull << 61);
}

template <int D, bool BF>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) pair_kernel(const __grid_constant__ Params p) {
  using L = Layout<D>;
  constexpr int NS = L::SLOTS;
  constexpr float THR = BF ? 8.0f : 3.0f;     // the maximum in use may lag behind by a factor of 2^THR before O is rescaled
  // fp16 weights are shifted up by 2^12 (at most 2^15 with the lag), so that weights down to 2^-26 of the largest keep all bits
  constexpr float SHIFT = BF ? 0.0f : 12.0f;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* xchg = reinterpret_cast<float*>(smem + L::xchg);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
  uint64_t* full = bars;               // [NS] (leader's) both CTAs' halves landed (tx)
  uint64_t* empty = full + NS;         // [NS] the slot's MMAs are done (commit to both CTAs)
  uint64_t* s_full = empty + NS;       // [2] S is in TMEM (commit to both)
  uint64_t* p_full = s_full + 2;       // [2] (leader's) P is in TMEM (16 warps of the pair)
  uint64_t* pv_done = p_full + 2;      // [2] a tile's P V is in O (commit to both)
  uint64_t* o_full = pv_done + 2;      // the item's O is complete (commit to both)
  uint64_t* o_empty = o_full + 1;      // (leader's) O has been read out (16 warps)
  uint64_t* q_full = o_empty + 1;      // (leader's) Q rows are in shared memory (8 loader warps)
  uint64_t* q_empty = q_full + 1;      // the item's Q K^T are done (commit to both)
  uint64_t* info_full = q_empty + 1;   // [2] item info is there
  uint64_t* info_empty = info_full + 2;// [2] item info has been read (producer, MMA, 8 softmax warps)
  uint64_t* item_full = info_empty + 2;// the next item's number arrived (tx)
  uint64_t* item_free = item_full + 1; // (leader's) both CTAs took it
  uint64_t* xb = item_free + 1;        // [4] the two warps of a lane quarter
  uint64_t* ldb = xb + 4;              // the loader warps
  uint64_t* drainb = ldb + 1;
  ItemInfo* info = reinterpret_cast<ItemInfo*>(smem + L::bars + 512);   // [2]
  int* ld_part = reinterpret_cast<int*>(info + 2);                      // [2][LD_WARPS][7]: reductions, by parity
  uint32_t* next_item = reinterpret_cast<uint32_t*>(ld_part + 2 * LD_WARPS * 7);
  uint32_t* tmem_holder = next_item + 1;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles start on 1024 bytes
    set_status(p.a.status, REAXMOE_ERR_UNSUPPORTED);
    return;
  }
  // every lane of a warp waits and all get the same answer
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, wait_bounded(smem_u32(bar), parity & 1u, abort_flag, p.a.status, p.timeout_ns)) != 0;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&s_full[b]), 1);
      mbar_init(smem_u32(&p_full[b]), 2 * SM_WARPS);
      mbar_init(smem_u32(&pv_done[b]), 1);
      mbar_init(smem_u32(&info_full[b]), 1);
      mbar_init(smem_u32(&info_empty[b]), SM_WARPS + 2);
    }
    mbar_init(smem_u32(o_full), 1);
    mbar_init(smem_u32(o_empty), 2 * SM_WARPS);
    mbar_init(smem_u32(q_full), 2 * LD_WARPS);
    mbar_init(smem_u32(q_empty), 1);
    mbar_init(smem_u32(item_full), 1);
    mbar_init(smem_u32(item_free), 2);
    for (int b = 0; b < 4; ++b) mbar_init(smem_u32(&xb[b]), 2);
    mbar_init(smem_u32(ldb), LD_WARPS);
    mbar_init(smem_u32(drainb), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_holder)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                       // both CTAs' barriers are ready, both allocations made
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 8) {
    // ------------------------------------------------------------------------------------------ K / V producer
    int n = 0;                          // slots filled
    bool ok = true;
    auto fill = [&](bool value, int start, bool pre, int head) {
      const int s = n % NS;
      if (n >= NS && !wait(&empty[s], (uint32_t)(n / NS - 1))) return false;
      const uint32_t bar = map_to_rank(smem_u32(&full[s]), 0);
      if (lane == 0) {
        const uint32_t dst = smem_u32(smem + L::ring + s * L::SLOT);
        if (rank == 0) mbar_expect_tx(smem_u32(&full[s]), 2 * L::SLOT);
        if (!value) {
          const CUtensorMap* tm = pre ? &p.tmPK : &p.tmK;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) tma_load_3d_pair(dst + c * 8192, tm, bar, c * 64, head, start + 64 * (int)rank);
        } else {
          const CUtensorMap* tm = pre ? &p.tmPV : &p.tmV;
          constexpr int W = D == 64 ? 32 : 64;
#pragma unroll
          for (int c = 0; c < D / 2 / W; ++c)
            tma_load_3d_pair(dst + c * (KT * W * 2), tm, bar, (int)rank * (D / 2) + c * W, head, start);
        }
      }
      __syncwarp();
      ++n;
      return true;
    };
    for (int i = 0; ok; ++i) {
      const int ib = i & 1;
      if (!(ok = wait(&info_full[ib], (uint32_t)(i >> 1)))) break;
      const ItemInfo it = info[ib];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&info_empty[ib]));
      if (it.row0 < 0) break;
      TileIter ti;
      ti.init(p, it);
      int cur, nxt;
      bool cpre, npre;
      if (!ti.next(p, cur, cpre)) continue;
      ok = fill(false, cur, cpre, it.head);
      bool more = true;
      while (ok && more) {
        more = ti.next(p, nxt, npre);
        if (more) ok = fill(false, nxt, npre, it.head);
        if (ok) ok = fill(true, cur, cpre, it.head);
        cur = nxt;
        cpre = npre;
      }
    }
    // let the last loads land before the CTA may exit (only matters after an abort)
    if (rank == 0)
      for (int f = n - 1; f >= 0 && f >= n - NS; --f) wait_drain(smem_u32(&full[f % NS]), (uint32_t)(f / NS) & 1u);
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------------------ MMA issuer (leader)
    constexpr uint32_t kFmt = (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(256 >> 4) << 24);
    constexpr uint32_t kQK = kFmt | ((uint32_t)(KT >> 3) << 17);
    constexpr uint32_t kPV = kFmt | (1u << 16) | ((uint32_t)(D >> 3) << 17);   // B (V) MN-major
    int n = 0, g = 0, items = 0;        // slots consumed, tiles, items with tiles
    bool ok = true;
    const uint32_t qs = smem_u32(smem);
    auto qk = [&](int tile) {
      const int s = n % NS;
      if (!wait(&full[s], (uint32_t)(n / NS))) return false;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t ks = smem_u32(smem + L::ring + s * L::SLOT);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_pair_ss(tmem + (tile & 1) * KT, desc_sw128(qs + c * 16384 + k * 32), desc_sw128(ks + c * 8192 + k * 32), kQK,
                        (c | k) != 0 ? 1u : 0u);
        commit_pair(smem_u32(&empty[s]));
        commit_pair(smem_u32(&s_full[tile & 1]));
      }
      __syncwarp();
      ++n;
      return true;
    };
    for (int i = 0; ok; ++i) {
      const int ib = i & 1;
      if (!(ok = wait(&info_full[ib], (uint32_t)(i >> 1)))) break;
      const ItemInfo it = info[ib];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&info_empty[ib]));
      if (it.row0 < 0) break;
      if (rank != 0) continue;
      TileIter ti;
      ti.init(p, it);
      int start;
      bool pre;
      if (!ti.next(p, start, pre)) continue;
      if (!(ok = wait(q_full, (uint32_t)items))) break;
      if (!(ok = qk(g))) break;
      bool more = true;
      for (int j = 0; more; ++j, ++g) {
        more = ti.next(p, start, pre);
        if (more && !(ok = qk(g + 1))) break;
        if (!more && lane == 0) commit_pair(smem_u32(q_empty));
        if (!(ok = wait(&p_full[g & 1], (uint32_t)(g >> 1)))) break;
        if (j == 0 && items > 0 && !(ok = wait(o_empty, (uint32_t)(items - 1)))) break;
        const int s = n % NS;
        if (!(ok = wait(&full[s], (uint32_t)(n / NS)))) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t vs = smem_u32(smem + L::ring + s * L::SLOT);
#pragma unroll
          for (int k = 0; k < KT / 16; ++k)
            mma_pair_ts(tmem + O_COL, tmem + (g & 1) * KT + k * 8, desc_v<D>(vs + k * (D == 64 ? 1024 : 2048)), kPV,
                        (j | k) != 0 ? 1u : 0u);
          commit_pair(smem_u32(&empty[s]));
          commit_pair(smem_u32(&pv_done[g & 1]));
          if (!more) commit_pair(smem_u32(o_full));
        }
        __syncwarp();
        ++n;
      }
      ++items;
    }
    // every issued MMA has completed before TMEM may be released (matters after an abort)
    if (rank == 0) {
      if (lane == 0)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(drainb)) : "memory");
      __syncwarp();
      wait_drain(smem_u32(drainb), 0);
    }
  } else if (warp >= LD_WARP0) {
    // ------------------------------------------------------------------------------------------ loader: items and Q rows
    const int lw = warp - LD_WARP0, tid = threadIdx.x - LD_WARP0 * 32;
    const int nrows = row_count(p);
    const uint32_t leader_q = map_to_rank(smem_u32(q_full), 0), leader_free = map_to_rank(smem_u32(item_free), 0);
    int items = 0, syncs = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      int item = i == 0 ? pair : p.items;
      if (i > 0 && p.counter != nullptr) {
        if (rank == 0 && tid == 0) {
          if (i <= 1 || wait_bounded(smem_u32(item_free), (uint32_t)(i - 2) & 1u, abort_flag, p.a.status, p.timeout_ns)) {
            const uint32_t v = (uint32_t)(pairs + atomicAdd(p.counter, 1));
            for (uint32_t r = 0; r < 2; ++r)
              st_async_u32(map_to_rank(smem_u32(next_item), r), v, map_to_rank(smem_u32(item_full), r));
          }
        }
        if (tid == 0) mbar_expect_tx(smem_u32(item_full), 4);
        if (!wait(item_full, (uint32_t)(i - 1))) break;
        item = (int)*reinterpret_cast<volatile uint32_t*>(next_item);
      }
      const int ib = i & 1;
      if (i > 1 && !wait(&info_empty[ib], (uint32_t)((i >> 1) - 1))) break;
      if (item >= p.items) {
        if (tid == 0) {
          info[ib].row0 = -1;
          mbar_arrive(smem_u32(&info_full[ib]));
        }
        break;
      }
      // later tiles first: of a causal sequence these are the long ones
      const int part = item % p.parts, head = (item / p.parts) % p.a.kv_heads;
      const int row0 = (p.tiles - 1 - item / p.parts / p.a.kv_heads) * 2 * ROWS;
      // the union of the 256 rows' ranges: thread = rows 2 tid, 2 tid + 1
      int plo = INT_MAX, phi = 0, klo = INT_MAX, khi = 0, gap = 0, first_lo = INT_MAX, last_hi = INT_MAX;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + 2 * tid + h;
        if (r < nrows) {
          const RowKeys rk = row_keys(p.a, r / p.group);
          if (rk.p_lo < rk.p_hi) {
            plo = min(plo, rk.p_lo);
            phi = max(phi, rk.p_hi);
          }
          if (rk.k_lo < rk.k_hi) {
            klo = min(klo, rk.k_lo);
            khi = max(khi, rk.k_hi);
          }
          if (h == 0) first_lo = rk.k_lo;
          else if (rk.k_lo - last_hi >= KT) gap = 1;
          last_hi = rk.k_hi;
        } else if (h == 0) {
          first_lo = -1;
        }
      }
      const int nx = __shfl_down_sync(0xffffffffu, first_lo, 1);
      if (lane < 31 && last_hi != INT_MAX && nx >= 0 && nx - last_hi >= KT) gap = 1;
      const int wfirst = __shfl_sync(0xffffffffu, first_lo, 0), wlast = __shfl_sync(0xffffffffu, last_hi, 31);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        plo = min(plo, __shfl_xor_sync(0xffffffffu, plo, o));
        phi = max(phi, __shfl_xor_sync(0xffffffffu, phi, o));
        klo = min(klo, __shfl_xor_sync(0xffffffffu, klo, o));
        khi = max(khi, __shfl_xor_sync(0xffffffffu, khi, o));
        gap |= __shfl_xor_sync(0xffffffffu, gap, o);
      }
      int* mine = ld_part + (syncs & 1) * LD_WARPS * 7 + lw * 7;
      if (lane == 0) {
        mine[0] = plo;
        mine[1] = phi;
        mine[2] = klo;
        mine[3] = khi;
        mine[4] = gap;
        mine[5] = wfirst;
        mine[6] = wlast;
        mbar_arrive(smem_u32(ldb));
      }
      if (!wait(ldb, (uint32_t)syncs)) break;
      const int* all = ld_part + (syncs & 1) * LD_WARPS * 7;
      ++syncs;
#pragma unroll
      for (int w = 0; w < LD_WARPS; ++w) {
        plo = min(plo, all[w * 7]);
        phi = max(phi, all[w * 7 + 1]);
        klo = min(klo, all[w * 7 + 2]);
        khi = max(khi, all[w * 7 + 3]);
        gap |= all[w * 7 + 4];
        if (w > 0 && all[w * 7 - 1] != INT_MAX && all[w * 7 + 5] >= 0 && all[w * 7 + 5] != INT_MAX &&
            all[w * 7 + 5] - all[w * 7 - 1] >= KT)
          gap = 1;
      }
      if (p.counter != nullptr && i > 0 && tid == 0) mbar_arrive_cluster(leader_free);   // all loader threads have read it
      // this part of the tiles (counted without gaps)
      const int np = plo < phi ? (phi - plo + KT - 1) / KT : 0, no = klo < khi ? (khi - klo + KT - 1) / KT : 0;
      const int a0 = (int)((int64_t)(np + no) * part / p.parts), a1 = (int)((int64_t)(np + no) * (part + 1) / p.parts);
      ItemInfo it;
      it.row0 = row0;
      it.head = head;
      it.part = part;
      it.p_lo = a0 < np ? plo + a0 * KT : 0;
      it.p_hi = a0 < np ? (a1 >= np ? phi : plo + a1 * KT) : 0;
      it.o_lo = a1 > np ? klo + max(a0 - np, 0) * KT : 0;
      it.o_hi = a1 > np ? (a1 == np + no ? khi : klo + (a1 - np) * KT) : 0;
      it.gap = gap;
      if (tid == 0) {
        info[ib] = it;
        mbar_arrive(smem_u32(&info_full[ib]));
      }
      TileIter ti;
      ti.init(p, it);
      int start;
      bool pre;
      if (!ti.next(p, start, pre)) continue;
      if (items > 0 && !wait(q_empty, (uint32_t)(items - 1))) break;
      // 8 threads copy 128 bytes (64 elements) of a row; 16 rows per pass
      const int piece = tid & 7;
#pragma unroll 1
      for (int j = 0; j < ROWS / 16; ++j) {
        const int r = j * 16 + (tid >> 3);
        const int row = row0 + (int)rank * ROWS + r;
        const uint32_t dst = smem_u32(smem) + r * 128 + ((piece ^ (r & 7)) << 4);
        if (row < nrows) {
          const int t = row / p.group;
          const uint16_t* src = static_cast<const uint16_t*>(p.a.q) + (int64_t)t * p.a.q_stride +
                                (int64_t)(head * p.group + row - t * p.group) * p.a.q_head_stride + piece * 8;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) cp_async_16(dst + c * 16384, src + c * 64);
        } else {
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + c * 16384), "r"(0) : "memory");
        }
      }
      cp_async_wait_all();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_q);
      ++items;
    }
  } else {
    // ------------------------------------------------------------------------------------------ softmax, output
    const int quarter = warp & 3, half = warp >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int nrows = row_count(p);
    const float c = p.a.scale * 1.4426950408889634f;
    const uint32_t leader_p[2] = {map_to_rank(smem_u32(&p_full[0]), 0), map_to_rank(smem_u32(&p_full[1]), 0)};
    const uint32_t leader_o = map_to_rank(smem_u32(o_empty), 0);
    int g = 0, items = 0, ex = 0;
    bool ok = true;
    // the value of the row's other column half (both warps of the quarter call it)
    auto exchange = [&](float mine, float& other) {
      float* buf = xchg + (ex & 1) * 2 * ROWS;
      buf[half * ROWS + r] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&xb[quarter]));
      const bool fine = wait(&xb[quarter], (uint32_t)ex);
      other = buf[(half ^ 1) * ROWS + r];
      ++ex;
      return fine;
    };
    for (int i = 0; ok; ++i) {
      const int ib = i & 1;
      if (!(ok = wait(&info_full[ib], (uint32_t)(i >> 1)))) break;
      const ItemInfo it = info[ib];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&info_empty[ib]));
      if (it.row0 < 0) break;
      const int row = it.row0 + (int)rank * ROWS + r;
      const bool live = row < nrows;
      const bool any_live = __any_sync(0xffffffffu, live);
      const int tok = live ? row / p.group : 0;
      // a row that is not there needs no mask (its sums are not read)
      RowKeys rk = {0, INT_MAX, 0, INT_MAX};
      if (live) rk = row_keys(p.a, tok);
      const bool none = rk.p_lo >= rk.p_hi && rk.k_lo >= rk.k_hi;
      float m = -INFINITY, l = 0.0f;       // the maximum in use (of scores times c) and this half's sum
      TileIter ti;
      ti.init(p, it);
      int start, j = 0;
      bool pre;
      for (; ti.next(p, start, pre); ++j, ++g) {
        // keys from the part's end on are the next part's, whose first tile may begin inside this one where there are gaps
        const int lo = pre ? rk.p_lo : rk.k_lo, hi = pre ? min(rk.p_hi, it.p_hi) : min(rk.k_hi, it.o_hi);
        const int a0 = max(lo - start, 0), a1 = hi - start;          // columns [a0, a1) are seen
        if (!(ok = wait(&s_full[g & 1], (uint32_t)(g >> 1)))) break;
        const uint32_t scol = tmem + lanes + (uint32_t)((g & 1) * KT);
        if (any_live) {
          tc_fence_after();
          const bool all = __all_sync(0xffffffffu, a0 == 0 && a1 >= KT);
          const bool nothing = __all_sync(0xffffffffu, a0 >= KT || a1 <= a0);
          uint32_t w[32];
          if (nothing) {
#pragma unroll
            for (int x = 0; x < 32; ++x) w[x] = 0u;
          } else {
            uint32_t s0[32], s1[32];
            tc_ld_32x32b_x32(scol + half * 64, s0);
            tc_ld_32x32b_x32(scol + half * 64 + 32, s1);
            tc_wait_ld();
            if (!all) {
              const int b0 = a0 - half * 64, b1 = a1 - half * 64;
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                if (x < b0 || x >= b1) s0[x] = 0xFF800000u;
                if (x + 32 < b0 || x + 32 >= b1) s1[x] = 0xFF800000u;
              }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              mx[0] = fmaxf(mx[0], __uint_as_float(s0[x]));
              mx[1] = fmaxf(mx[1], __uint_as_float(s0[x + 1]));
              mx[2] = fmaxf(mx[2], __uint_as_float(s1[x]));
              mx[3] = fmaxf(mx[3], __uint_as_float(s1[x + 1]));
            }
            float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), theirs;
            if (!(ok = exchange(top, theirs))) break;
            top = fmaxf(top, theirs) * c;
            const bool grow = top - m > THR;       // from -inf on the first key
            const bool rescale = grow && m != -INFINITY;
            const float f = rescale ? ex2(m - top) : 1.0f;
            if (grow) m = top;
            l *= f;
            if (j > 0 && __any_sync(0xffffffffu, rescale)) {
              if (!(ok = wait(&pv_done[(g - 1) & 1], (uint32_t)((g - 1) >> 1)))) break;
              tc_fence_after();
              constexpr int HC = D / 2;            // this half's columns of O
#pragma unroll 1
              for (int x = 0; x < HC; x += 32) {
                uint32_t o[32];
                tc_ld_32x32b_x32(tmem + lanes + O_COL + half * HC + x, o);
                tc_wait_ld();
#pragma unroll
                for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                tc_st_32x32b_x32(tmem + lanes + O_COL + half * HC + x, o);
              }
              tc_wait_st();
            }
            const float mc = (m == -INFINITY ? 0.0f : m) - SHIFT;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const float e0 = ex2(fmaf(__uint_as_float(s0[x]), c, -mc)), e1 = ex2(fmaf(__uint_as_float(s0[x + 1]), c, -mc));
              w[x / 2] = pack2<BF>(e0, e1);
              sum[0] += e0;
              sum[1] += e1;
            }
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const float e0 = ex2(fmaf(__uint_as_float(s1[x]), c, -mc)), e1 = ex2(fmaf(__uint_as_float(s1[x + 1]), c, -mc));
              w[16 + x / 2] = pack2<BF>(e0, e1);
              sum[2] += e0;
              sum[3] += e1;
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          }
          tc_st_32x32b_x32(scol + half * 32, w);
          tc_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_p[g & 1]);
      }
      if (!ok) break;
      // the item's rows: o = O / l, or the partial sums of this part
      float other = 0.0f;
      if (j > 0 && !(ok = wait(o_full, (uint32_t)items))) break;
      if (any_live) {
        if (!(ok = exchange(l, other))) break;
        l += other;
        constexpr int HC = D / 2;
        const int head = it.head * p.group + (row - tok * p.group);
        const int64_t part_row = ((int64_t)it.part * p.a.kv_heads + it.head) * ((int64_t)p.tiles * 2 * ROWS) + row;
        const float inv = none ? 0.0f : 1.0f / l;
        uint16_t* out = static_cast<uint16_t*>(p.a.out) + (int64_t)tok * p.a.out_stride + head * p.a.out_head_stride + half * HC;
        bool bad = false;
        if (j > 0) tc_fence_after();
#pragma unroll 1
        for (int x = 0; x < HC; x += 32) {
          uint32_t o[32];
          if (j > 0) {
            tc_ld_32x32b_x32(tmem + lanes + O_COL + half * HC + x, o);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = 0u;
          }
          if (live && p.parts > 1) {
            float4* dst = reinterpret_cast<float4*>(p.part_o + part_row * D + half * HC + x);
#pragma unroll
            for (int y = 0; y < 8; ++y)
              dst[y] = make_float4(__uint_as_float(o[4 * y]), __uint_as_float(o[4 * y + 1]), __uint_as_float(o[4 * y + 2]),
                                   __uint_as_float(o[4 * y + 3]));
          } else if (live) {
#pragma unroll
            for (int y = 0; y < 32; y += 8) {
              uint32_t v[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const float f0 = none ? 0.0f : __uint_as_float(o[y + 2 * z]) * inv;
                const float f1 = none ? 0.0f : __uint_as_float(o[y + 2 * z + 1]) * inv;
                bad |= !(fabsf(f0) < INFINITY) || !(fabsf(f1) < INFINITY);
                v[z] = pack2<BF>(f0, f1);
              }
              *reinterpret_cast<uint4*>(out + x + y) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (j > 0 && lane == 0) mbar_arrive_cluster(leader_o);
        if (p.parts > 1) {
          if (live && half == 0) p.part_ml[part_row] = make_float2(m, l);
        } else {
          if (live && half == 0 && p.a.lse != nullptr)
            p.a.lse[(int64_t)tok * p.a.q_heads + head] = none ? -INFINITY : (m - SHIFT + __log2f(l)) * 0.6931471805599453f;
          // 0 x (an infinity or NaN of a value that the row does not see) is NaN: such rows are done again key by key. A sum
          // that is NaN itself came from a key that the row does see.
          if (!(ok = exchange(bad && l == l ? 1.0f : 0.0f, other))) break;
          uint32_t again = __ballot_sync(0xffffffffu, live && ((bad && l == l) || other != 0.0f));
          while (half == 0 && again != 0u) {
            const int src = __ffs(again) - 1;
            again &= again - 1u;
            row_by_warp<D, BF>(p.a, __shfl_sync(0xffffffffu, tok, src), __shfl_sync(0xffffffffu, head, src));
          }
        }
      } else if (j > 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_o);
      }
      if (j > 0) ++items;
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();                       // neither CTA's shared memory nor TMEM is in use any more
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the parts of a row: one warp per row.
template <int D, bool BF>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ Params p) {
  constexpr float SHIFT = BF ? 0.0f : 12.0f;
  constexpr int W = D / 32;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int tok = (int)(id / p.a.q_heads), head = (int)(id - (int64_t)tok * p.a.q_heads);
  if ((int64_t)tok * p.group >= row_count(p)) return;
  const int kvh = head / p.group;
  const int64_t stride = (int64_t)p.tiles * 2 * ROWS;
  const int64_t first = (int64_t)kvh * stride + (int64_t)tok * p.group + (head - kvh * p.group);
  float m = -INFINITY;
  for (int s = 0; s < p.parts; ++s) m = fmaxf(m, p.part_ml[first + (int64_t)s * p.a.kv_heads * stride].x);
  float l = 0.0f, acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = 0.0f;
  for (int s = 0; s < p.parts; ++s) {
    const int64_t row = first + (int64_t)s * p.a.kv_heads * stride;
    const float2 ml = p.part_ml[row];
    if (ml.x == -INFINITY && ml.y == 0.0f) continue;     // this part has none of the row's keys, or scores of -inf alone
    const float f = ml.x == m ? 1.0f : ex2(ml.x - m);
    l = fmaf(ml.y, f, l);
    const float4* src = reinterpret_cast<const float4*>(p.part_o + row * D) + lane;
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const float4 v = __ldg(src + i * 32);
      acc[4 * i] = fmaf(v.x, f, acc[4 * i]);
      acc[4 * i + 1] = fmaf(v.y, f, acc[4 * i + 1]);
      acc[4 * i + 2] = fmaf(v.z, f, acc[4 * i + 2]);
      acc[4 * i + 3] = fmaf(v.w, f, acc[4 * i + 3]);
    }
    if constexpr (W == 2) {
      const float2 v = __ldg(reinterpret_cast<const float2*>(p.part_o + row * D) + lane);
      acc[0] = fmaf(v.x, f, acc[0]);
      acc[1] = fmaf(v.y, f, acc[1]);
    }
  }
  const RowKeys rk = row_keys(p.a, tok);
  const bool none = rk.p_lo >= rk.p_hi && rk.k_lo >= rk.k_hi;
  const float inv = none ? 0.0f : 1.0f / l;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    acc[i] = none ? 0.0f : acc[i] * inv;
    bad |= !(fabsf(acc[i]) < INFINITY);
  }
  if (__any_sync(0xffffffffu, bad) && l == l) {
    row_by_warp<D, BF>(p.a, tok, head);
    return;
  }
  uint16_t* out = static_cast<uint16_t*>(p.a.out) + (int64_t)tok * p.a.out_stride + head * p.a.out_head_stride;
  if constexpr (W == 2) {
    reinterpret_cast<uint32_t*>(out)[lane] = pack2<BF>(acc[0], acc[1]);
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
      reinterpret_cast<uint2*>(out)[lane + i * 32] =
          make_uint2(pack2<BF>(acc[4 * i], acc[4 * i + 1]), pack2<BF>(acc[4 * i + 2], acc[4 * i + 3]));
  }
  if (p.a.lse != nullptr && lane == 0)
    p.a.lse[(int64_t)tok * p.a.q_heads + head] = none ? -INFINITY : (m - SHIFT + __log2f(l)) * 0.6931471805599453f;
}

// Row tiles, parts of the keys, and the workspace: counter, partial maxima and sums, partial outputs.
struct Plan {
  int group, tiles, parts, items, pairs;
  size_t ml, o, total;
};

static Plan plan(const reaxmoe_attention_args& a, int num_sms) {
  Plan pl;
  pl.group = a.q_heads / a.kv_heads;
  const int64_t rows = a.q_tokens * pl.group;
  pl.tiles = (int)ceil_div64(rows, 2 * ROWS);
  const int64_t base = (int64_t)pl.tiles * a.kv_heads;
  const int pairs = num_sms / 2 > 0 ? num_sms / 2 : 1;
  const int64_t keys = a.prefix + a.k_tokens;
  // split the keys when the tiles leave half of the pairs idle, into parts of at least 512 keys
  int64_t parts = base > 0 && base * 2 <= pairs ? pairs / base : 1;
  const int64_t most = ceil_div64(keys, 512);
  if (parts > most) parts = most;
  pl.parts = (int)(parts < 1 ? 1 : parts);
  const int64_t items = base * pl.parts;
  pl.items = (int)items;
  pl.pairs = (int)(items < pairs ? items : pairs);
  pl.ml = 256;
  const size_t prow = pl.parts > 1 ? (size_t)pl.parts * a.kv_heads * pl.tiles * 2 * ROWS : 0;
  pl.o = pl.ml + ((prow * 8 + 255) & ~size_t(255));
  pl.total = pl.o + prow * a.head_dim * 4;
  return pl;
}

template <int D, bool BF>
static int launch_t(const AttentionLaunch& l, const Plan& pl, cudaStream_t s) {
  const reaxmoe_attention_args& a = l.a;
  Params p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.group = pl.group;
  p.tiles = pl.tiles;
  p.parts = pl.parts;
  p.items = pl.items;
  uint8_t* ws = static_cast<uint8_t*>(l.workspace);
  p.counter = pl.items > pl.pairs ? reinterpret_cast<int*>(ws) : nullptr;
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
  p.part_o = reinterpret_cast<float*>(ws + pl.o);
  p.timeout_ns = l.timeout_ns;
  constexpr int VB = D == 64 ? 32 : 64;
  if (a.k_tokens > 0 &&
      (make_map_heads(&p.tmK, a.k, a.k_tokens, a.k_stride, a.kv_heads, a.k_head_stride, D, 64, 64) ||
       make_map_heads(&p.tmV, a.v, a.k_tokens, a.v_stride, a.kv_heads, a.v_head_stride, D, VB, KT)))
    return REAXMOE_ERR_CUDA;
  if (a.prefix > 0 &&
      (make_map_heads(&p.tmPK, a.prefix_k, a.prefix, a.prefix_k_stride, a.kv_heads, a.prefix_k_head_stride, D, 64, 64) ||
       make_map_heads(&p.tmPV, a.prefix_v, a.prefix, a.prefix_v_stride, a.kv_heads, a.prefix_v_head_stride, D, VB, KT)))
    return REAXMOE_ERR_CUDA;
  auto kfn = pair_kernel<D, BF>;
  if (cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::total) != cudaSuccess)
    return REAXMOE_ERR_CUDA;
  if (p.counter != nullptr && cudaMemsetAsync(p.counter, 0, sizeof(int), s) != cudaSuccess) return REAXMOE_ERR_CUDA;
  kfn<<<2 * pl.pairs, THREADS, Layout<D>::total, s>>>(p);
  if (pl.parts > 1) combine_kernel<D, BF><<<(unsigned)ceil_div64(a.q_tokens * a.q_heads, 8), 256, 0, s>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? 0 : REAXMOE_ERR_CUDA;
}

}  // namespace attn

size_t attention_workspace(const reaxmoe_attention_args& a, int num_sms) { return attn::plan(a, num_sms).total; }

int launch_attention(const AttentionLaunch& l, cudaStream_t s) {
  const attn::Plan pl = attn::plan(l.a, l.num_sms);
  const bool bf = l.a.dtype == REAXMOE_BF16;
  switch (l.a.head_dim) {
    case 64: return bf ? attn::launch_t<64, true>(l, pl, s) : attn::launch_t<64, false>(l, pl, s);
    case 128: return bf ? attn::launch_t<128, true>(l, pl, s) : attn::launch_t<128, false>(l, pl, s);
    default: return bf ? attn::launch_t<256, true>(l, pl, s) : attn::launch_t<256, false>(l, pl, s);
  }
}

}  // namespace reaxmoe
