// attention.cu -- attention over packed sequences and over a prefix that a batch shares (reaxmoe_attention), on the tensor
// cores of CTA pairs.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(c s_ij - c m_i),  c = scale log2(e),  s_ij = q_i . k_j over the keys j that
//   row i sees, m_i a running maximum (one pass over the keys; o and the sum are rescaled when it grows).
//
// Rows. Query head h of KV head g reads the same keys as its group's other heads, so the rows of KV head g are (token, head of
// the group) pairs, row = token * group + h % group, over ALL packed tokens: a tile of up to 256 consecutive rows (the whole
// tokens that fit into 128 rows, in each CTA of a pair) may end one sequence, hold others whole and begin the next. What a row sees is two ranges of keys (of the prefix and
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
// P is rounded to 16 bits because the tensor core takes it in the type of V (in 32 bits it would be two products, of a high and a
// low part); the sum that divides adds the weights as they are before it. Each weight is so off by half a step at most, the
// outputs by 2.1e-3 to 2.3e-3 (bf16) and 2.8e-4 (fp16) relative to their norm, where rounding alone makes 1.65e-3 and 2.1e-4. On
// rows with one large weight the lagging maximum (below) shows: 1.78e-3 on the decision model's heads against 1.41e-3 of a
// kernel whose largest weight is always 1. Maxima, sums and O are held in 32 bits.
// S has 2 buffers of 128 columns beside O (D columns) for D = 256, 3 for D <= 128: the tensor core multiplies S(j + 1) (and
// S(j + 2)) while the softmax of tile j runs, and the next item's first S while this item's O is written out.
//
//   warps 0..7    softmax: TMEM lane quarter w % 4 (thread = row), column half w / 4; the halves of a row exchange maxima
//   warp 8        K / V producer: ring of slots, alternately half a K tile (64 keys x D) and half a V tile (128 keys x D / 2)
//   warp 9        allocates TMEM; in the leader CTA one thread issues all MMAs of the pair
//   warp 10       loader: takes the next item, works out its key ranges, loads its Q rows (TMA)
//   warps 12..15  output: O from TMEM, divided by the sums, while the softmax warps are at the next item's first tiles
// Items (row tile, KV head, part of the keys) are taken in order, the first by pair number, further ones from a counter.
// With few rows an item's keys are split over several pairs, which leave partial sums that combine_kernel joins.
// All waits are bounded (globaltimer, from the last sign of life of those who do long work); a timeout records
// REAXMOE_ERR_DEVICE_TIMEOUT and the CTA winds down.
#include <atomic>
#include <cstring>

#include "attention_few.cuh"
#include "attention_rows.cuh"
#include "attention_sm100.cuh"
#include "kernels.cuh"

namespace reaxmoe {
namespace attn {

constexpr int ROWS = 128;                 // query rows per CTA
constexpr int KT = 128;                   // keys per tile
constexpr int SM_WARPS = 8;               // softmax warps
constexpr int OUT_WARP0 = 12, OUT_WARPS = 4;
constexpr int THREADS = (OUT_WARP0 + OUT_WARPS) * 32;
// registers a thread: the kernel is launched with 128 x 512 of them, and the warp groups share these out (the sum stays 512)
constexpr int REGS_SOFTMAX = 168, REGS_CONTROL = 64, REGS_OUT = 112;
static_assert(2 * REGS_SOFTMAX + REGS_CONTROL + REGS_OUT == 4 * 128 && THREADS == 512, "register shares");

struct ItemInfo {
  int row0;          // first row of the pair's tile; -1: no more items
  int b0, b1;        // first and last sequence that has rows in it
  Sequence first;    // the first
  int head, part;    // KV head, part of the keys
  int p_lo, p_hi;    // prefix keys of this part
  int o_lo, o_hi;    // own keys of this part
  int gap;           // keys that no row sees lie between those of two sequences
  int tiles;         // of 128 keys each
};

// Shared memory: Q, the ring of K and V slots, words, barriers (8 bytes each, by index), and what follows them.
template <int D>
struct Layout {
  static constexpr int NB = D == 256 ? 2 : 3;               // S buffers; TMEM columns: S0, S1, (S2,) O
  static constexpr int O_COL = NB * KT;
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int SLOT = 64 * D * 2;                   // half a K tile or half a V tile
  static constexpr int SLOTS = D == 256 ? 5 : 12;
  static constexpr int ring = Q_BYTES;
  static constexpr int words = ring + SLOTS * SLOT;         // [2][2][ROWS]: what the column halves of a row exchange, by parity
  static constexpr int bars = words + 4 * ROWS * 4;
  enum Bar {
    FULL = 0,                          // [SLOTS] (leader's) both CTAs' halves landed (tx)
    EMPTY = FULL + SLOTS,              // [SLOTS] the slot's MMAs are done (commit to both CTAs)
    S_FULL = EMPTY + SLOTS,            // [NB] S is in TMEM (commit to both)
    P_FULL = S_FULL + NB,              // [NB] (leader's) P is in TMEM (16 warps of the pair)
    PV_DONE = P_FULL + NB,             // [2] a tile's P V is in O (commit to both)
    O_FULL = PV_DONE + 2,              // the item's O is complete (commit to both)
    O_EMPTY = O_FULL + 1,              // (leader's) O has been read out (8 warps of the pair)
    Q_FULL = O_EMPTY + 1,              // (leader's) both CTAs' Q rows landed (tx)
    Q_EMPTY = Q_FULL + 1,              // the item's Q K^T are done (commit to both)
    INFO_FULL = Q_EMPTY + 1,           // [2] item info is there
    INFO_EMPTY = INFO_FULL + 2,        // [2] item info has been read (producer, MMA, softmax and output warps)
    ITEM_FULL = INFO_EMPTY + 2,        // the next item's number arrived (tx)
    ITEM_FREE = ITEM_FULL + 1,         // (leader's) both CTAs took it
    L_FULL = ITEM_FREE + 1,            // the item's factors 1 / sum are in shared memory (4 softmax warps)
    L_EMPTY = L_FULL + 1,              // they have been read (4 output warps)
    DRAIN = L_EMPTY + 1,               // every MMA is done
    BARS = DRAIN + 1
  };
  static constexpr int inv_l = bars + BARS * 8;             // [ROWS] floats
  static constexpr int info = (inv_l + ROWS * 4 + 7) / 8 * 8;      // [2] ItemInfo
  static constexpr int state = info + 2 * (int)sizeof(ItemInfo);   // next_item, tmem_holder, abort_flag, beat
  static constexpr int total = bars + 1024;
  static_assert(alignof(ItemInfo) <= 8 && state + 4 * 4 <= total, "what follows the barriers");
  static_assert(total <= 232448, "shared memory");
};

struct Params {
  CUtensorMap tmQ, tmK, tmV, tmPK, tmPV;
  reaxmoe_attention_args a;
  int group;
  int rows;          // rows of a CTA's tile: group times the tokens that fit into 128
  int tiles, parts, items;
  int prefix_only;   // own keys are left to few_kernel
  int partial;       // partial sums are left for a joining kernel
  int wide_out;      // output rows start on 32 bytes
  int* counter;      // items taken beyond the first of each pair (null when there are none)
  float* part_o;     // [parts][kv_heads][tiles * 2 * rows][D]
  float2* part_ml;   // [parts][kv_heads][tiles * 2 * rows]: maximum in units of log2, sum
  unsigned long long timeout_ns;
};

__device__ __forceinline__ int row_count(const Params& p) {
  const int t = min(__ldg(p.a.cu_q + p.a.seqs), (int)p.a.q_tokens);
  return max(t, 0) * p.group;
}

// The tiles of an item in order: prefix tiles, then own tiles, each 128 keys from `start`. Where own keys that no row sees lie
// between two sequences' (gap), a tile begins at the first key that some row still needs, found by walking the sequences.
struct TileIter {
  int cur, end, o_lo, o_hi;
  int b, b1, t0, t1, lo, hi;
  bool pre, gap;
  __device__ __forceinline__ void need(const reaxmoe_attention_args& a) {    // own keys that the tile's rows of sequence b see
    const int f = max(t0, __ldg(a.cu_q + b)), l = min(t1, __ldg(a.cu_q + b + 1)) - 1;
    const Sequence s = sequence_at(a, b);
    lo = row_keys_in(a, s, f).k_lo;
    hi = row_keys_in(a, s, l).k_hi;
    if (f > l || lo >= hi) lo = hi = 0;
  }
  __device__ __forceinline__ void own() {
    pre = false;
    cur = o_lo;
    end = o_hi;
  }
  __device__ __forceinline__ void init(const Params& p, const ItemInfo& it) {
    o_lo = it.o_lo;
    o_hi = it.o_hi;
    gap = it.gap != 0;
    if (gap) {
      t0 = it.row0 / p.group;
      t1 = min(it.row0 + 2 * p.rows, row_count(p)) / p.group;
      b = it.b0;
      b1 = it.b1;
      need(p.a);
    }
    pre = true;
    cur = it.p_lo;
    end = it.p_hi;
    if (cur >= end) own();
  }
  // one of the item's tiles: called it.tiles times at most
  __device__ __forceinline__ int next(const Params& p) {
    if (gap && !pre) {
#pragma unroll 1
      while (hi <= cur && b < b1) {
        ++b;
        need(p.a);
      }
      cur = max(cur, lo);
    }
    const int start = cur;
    cur += KT;
    return start;
  }
  __device__ __forceinline__ void after() {        // after each tile
    if (pre && cur >= end) own();
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
  constexpr int NS = L::SLOTS, NB = L::NB, AHEAD = NB - 1;   // S tiles multiplied ahead of the softmax
  constexpr int O_COL = L::O_COL;
  // The maximum in use may lag behind by a factor of 2^THR before O is rescaled, which costs a wait for the product before.
  // Weights in bf16 keep their precision at any size, so only the range of the fp32 sums limits the lag. fp16 weights end at
  // 2^16; they are shifted up by 2^SHIFT, so that weights down to 2^-18 of the one at the maximum in use keep all bits, those
  // below lose some, and those under 2^-29 vanish from the product: at most 2^-12 of a row's weight for up to 2^17 keys (a lag
  // of 2^3 at SHIFT 12, which has 2^-26 and 2^-37, made rescaling so frequent that D = 64 took 4500 clocks a tile).
  constexpr float THR = BF ? 64.0f : 11.0f;
  constexpr float SHIFT = BF ? 0.0f : 4.0f;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
  uint64_t *full = bars + L::FULL, *empty = bars + L::EMPTY, *s_full = bars + L::S_FULL, *p_full = bars + L::P_FULL;
  uint64_t *pv_done = bars + L::PV_DONE, *o_full = bars + L::O_FULL, *o_empty = bars + L::O_EMPTY, *q_full = bars + L::Q_FULL;
  uint64_t *q_empty = bars + L::Q_EMPTY, *info_full = bars + L::INFO_FULL, *info_empty = bars + L::INFO_EMPTY;
  uint64_t *item_full = bars + L::ITEM_FULL, *item_free = bars + L::ITEM_FREE, *l_full = bars + L::L_FULL;
  uint64_t *l_empty = bars + L::L_EMPTY, *drainb = bars + L::DRAIN;
  float* inv_l = reinterpret_cast<float*>(smem + L::inv_l);
  ItemInfo* info = reinterpret_cast<ItemInfo*>(smem + L::info);
  uint32_t* next_item = reinterpret_cast<uint32_t*>(smem + L::state);
  uint32_t* tmem_holder = next_item + 1;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile uint32_t* beat = tmem_holder + 2;     // changes with every slot filled and every 32 keys of a row done key by key

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles start on 1024 bytes
    set_status(p.a.status, REAXMOE_ERR_UNSUPPORTED);
    return;
  }
  auto wait1 = [&](uint64_t* bar, uint32_t parity) {
    return wait_alive(smem_u32(bar), parity & 1u, abort_flag, beat, p.a.status, p.timeout_ns);
  };
  // every lane of a warp waits and all get the same answer
  auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait1(bar, parity)) != 0; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(smem_u32(&s_full[b]), 1);
      mbar_init(smem_u32(&p_full[b]), 2 * SM_WARPS);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&pv_done[b]), 1);
      mbar_init(smem_u32(&info_full[b]), 1);
      mbar_init(smem_u32(&info_empty[b]), SM_WARPS + OUT_WARPS + 2);
    }
    mbar_init(smem_u32(o_full), 1);
    mbar_init(smem_u32(o_empty), 2 * OUT_WARPS);
    mbar_init(smem_u32(q_full), 1);
    mbar_init(smem_u32(q_empty), 1);
    mbar_init(smem_u32(item_full), 1);
    mbar_init(smem_u32(item_free), 2);
    mbar_init(smem_u32(l_full), SM_WARPS / 2);
    mbar_init(smem_u32(l_empty), OUT_WARPS);
    mbar_init(smem_u32(drainb), 1);
    *abort_flag = 0;
    *beat = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = threadIdx.x; i < 4 * ROWS; i += THREADS) sts_volatile(smem_u32(smem + L::words) + i * 4, 1u);   // not the first use's
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_holder)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                       // both CTAs' barriers are ready, both allocations made
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp >= SM_WARPS && warp < OUT_WARP0) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONTROL));
  if (warp == 8) {
    // ------------------------------------------------------------------------------------------ K / V producer
    if (elect_one()) {
      int s = 0, n = 0;                   // ring position, slots filled
      uint32_t sphase = 1;                // the first round finds the slots empty
      bool ok = true;
      auto fill = [&](bool value, int start, bool pre, int head) {
        if (n >= NS && !wait1(&empty[s], sphase)) return false;
        const uint32_t bar = map_to_rank(smem_u32(&full[s]), 0);
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
        *beat = (uint32_t)++n;
        if (++s == NS) {
          s = 0;
          sphase ^= 1u;
        }
        return true;
      };
      for (int i = 0; ok; ++i) {
        const int ib = i & 1;
        if (!(ok = wait1(&info_full[ib], (uint32_t)(i >> 1)))) break;
        const ItemInfo it = info[ib];
        mbar_arrive(smem_u32(&info_empty[ib]));
        if (it.row0 < 0) break;
        // K tiles run AHEAD tiles before their V tiles
        TileIter ti;
        ti.init(p, it);
        int start[AHEAD + 1];
        bool pre[AHEAD + 1];
#pragma unroll 1
        for (int j = 0; ok && j < it.tiles + AHEAD; ++j) {
#pragma unroll
          for (int a = AHEAD; a > 0; --a) {
            start[a] = start[a - 1];
            pre[a] = pre[a - 1];
          }
          if (j < it.tiles) {
            start[0] = ti.next(p);
            pre[0] = ti.pre;
            ti.after();
            ok = fill(false, start[0], pre[0], it.head);
          }
          if (ok && j >= AHEAD) ok = fill(true, start[AHEAD], pre[AHEAD], it.head);
        }
      }
      // let the last loads that the leader knows of land before the CTAs may exit (only matters after an abort)
      if (rank == 0)
#pragma unroll 1
        for (int f = n - 1; f >= 0 && f >= n - NS; --f) wait_drain(smem_u32(&full[f % NS]), (uint32_t)(f / NS) & 1u);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------------------ MMA issuer (leader)
    if (rank == 0 && elect_one()) {
      constexpr uint32_t kFmt = (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(256 >> 4) << 24);
      constexpr uint32_t kQK = kFmt | ((uint32_t)(KT >> 3) << 17);
      constexpr uint32_t kPV = kFmt | (1u << 16) | ((uint32_t)(D >> 3) << 17);   // B (V) MN-major
      const uint64_t qd = desc_sw128(smem_u32(smem)), kd = desc_sw128(smem_u32(smem + L::ring));
      const uint64_t vd = desc_v<D>(smem_u32(smem + L::ring));
      int slot = 0, items = 0;            // ring position, items with tiles
      uint32_t sphase = 0;
      int kbuf = 0, vbuf = 0, gv = 0;     // S buffers written and weighed with; tiles multiplied with V
      uint32_t vphase = 0;
      bool ok = true;
      auto qk = [&]() {
        if (!wait1(&full[slot], sphase)) return false;
        tc_fence_after();
        const uint64_t b = kd + (uint64_t)(slot * (L::SLOT >> 4));
        const uint32_t d = tmem + (uint32_t)(kbuf * KT);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_pair_ss(d, qd + (uint64_t)((c * 16384 + k * 32) >> 4), b + (uint64_t)((c * 8192 + k * 32) >> 4), kQK,
                        (c | k) != 0 ? 1u : 0u);
        commit_pair(smem_u32(&empty[slot]));
        commit_pair(smem_u32(&s_full[kbuf]));
        if (++kbuf == NB) kbuf = 0;
        if (++slot == NS) {
          slot = 0;
          sphase ^= 1u;
        }
        return true;
      };
      for (int i = 0; ok; ++i) {
        const int ib = i & 1;
        if (!(ok = wait1(&info_full[ib], (uint32_t)(i >> 1)))) break;
        const ItemInfo it = info[ib];
        mbar_arrive(smem_u32(&info_empty[ib]));
        if (it.row0 < 0) break;
        if (it.tiles == 0) continue;
        if (!(ok = wait1(q_full, (uint32_t)items))) break;
#pragma unroll 1
        for (int j = 0; j < it.tiles + AHEAD; ++j) {
          if (j < it.tiles && !(ok = qk())) break;
          if (j == it.tiles - 1) commit_pair(smem_u32(q_empty));
          if (j < AHEAD) continue;
          if (!(ok = wait1(&full[slot], sphase))) break;
          if (j == AHEAD && items > 0 && !(ok = wait1(o_empty, (uint32_t)(items - 1)))) break;
          if (!(ok = wait1(&p_full[vbuf], vphase))) break;
          tc_fence_after();
          const uint64_t b = vd + (uint64_t)(slot * (L::SLOT >> 4));
          const uint32_t a = tmem + (uint32_t)(vbuf * KT);
#pragma unroll
          for (int k = 0; k < KT / 16; ++k)
            mma_pair_ts(tmem + O_COL, a + k * 8, b + (uint64_t)((k * (D == 64 ? 1024 : 2048)) >> 4), kPV,
                        j == AHEAD && k == 0 ? 0u : 1u);
          commit_pair(smem_u32(&empty[slot]));
          commit_pair(smem_u32(&pv_done[gv & 1]));
          if (j == it.tiles + AHEAD - 1) commit_pair(smem_u32(o_full));
          ++gv;
          if (++vbuf == NB) {
            vbuf = 0;
            vphase ^= 1u;
          }
          if (++slot == NS) {
            slot = 0;
            sphase ^= 1u;
          }
        }
        ++items;
      }
      // every issued MMA has completed before TMEM may be released (matters after an abort)
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(drainb)) : "memory");
      wait_drain(smem_u32(drainb), 0);
    } else if (rank != 0 && lane == 0) {
      for (int i = 0;; ++i) {
        if (!wait1(&info_full[i & 1], (uint32_t)(i >> 1))) break;
        const int row0 = info[i & 1].row0;
        mbar_arrive(smem_u32(&info_empty[i & 1]));
        if (row0 < 0) break;
      }
    }
  } else if (warp == 10) {
    // ------------------------------------------------------------------------------------------ loader: items and Q rows
    const int ntok = row_count(p) / p.group, per = p.rows / p.group;      // tokens; tokens of a CTA's tile
    int items = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      int item = i == 0 ? pair : p.items;
      if (i > 0 && p.counter != nullptr) {
        if (lane == 0) {
          if (rank == 0 && (i == 1 || wait1(item_free, (uint32_t)(i - 2)))) {
            const uint32_t v = (uint32_t)(pairs + atomicAdd(p.counter, 1));
            for (uint32_t r = 0; r < 2; ++r)
              st_async_u32(map_to_rank(smem_u32(next_item), r), v, map_to_rank(smem_u32(item_full), r));
          }
          mbar_expect_tx(smem_u32(item_full), 4);
        }
        __syncwarp();
        if (!wait(item_full, (uint32_t)(i - 1))) break;
        item = (int)lds_volatile(smem_u32(next_item));
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(item_free), 0));
      }
      const int ib = i & 1;
      if (i > 1 && !wait(&info_empty[ib], (uint32_t)((i >> 1) - 1))) break;
      if (item >= p.items) {
        if (lane == 0) {
          info[ib].row0 = -1;
          mbar_arrive(smem_u32(&info_full[ib]));
        }
        break;
      }
      // later tiles first: of a causal sequence these are the long ones
      const int part = item % p.parts, head = (item / p.parts) % p.a.kv_heads;
      const int t0 = (p.tiles - 1 - item / p.parts / p.a.kv_heads) * 2 * per, t1 = min(t0 + 2 * per, ntok);
      ItemInfo it;
      memset(&it, 0, sizeof(it));
      it.row0 = t0 * p.group;
      it.head = head;
      it.part = part;
      if (t0 < t1) {
        // the union of the rows' ranges, sequence by sequence: from its first row's first key to its last row's last
        it.b0 = sequence_by_warp(p.a, t0);
        it.b1 = sequence_by_warp(p.a, t1 - 1);
        it.first = sequence_at(p.a, it.b0);
        int plo = INT_MAX, phi = 0, klo = INT_MAX, khi = 0;
        unsigned sum = 0;
#pragma unroll 4
        for (int b = it.b0 + lane; b <= it.b1; b += 32) {
          const int f = max(t0, __ldg(p.a.cu_q + b)), l = min(t1, __ldg(p.a.cu_q + b + 1)) - 1;
          if (f > l) continue;
          const Sequence s = b == it.b0 ? it.first : sequence_at(p.a, b);
          const RowKeys kf = row_keys_in(p.a, s, f), kl = row_keys_in(p.a, s, l);
          if (kf.p_lo < kl.p_hi) {
            plo = min(plo, kf.p_lo);
            phi = max(phi, kl.p_hi);
          }
          if (kf.k_lo < kl.k_hi && !p.prefix_only) {
            klo = min(klo, kf.k_lo);
            khi = max(khi, kl.k_hi);
            sum += (unsigned)(kl.k_hi - kf.k_lo);
          }
        }
        plo = __reduce_min_sync(0xffffffffu, plo);
        phi = __reduce_max_sync(0xffffffffu, phi);
        klo = __reduce_min_sync(0xffffffffu, klo);
        khi = __reduce_max_sync(0xffffffffu, khi);
        sum = __reduce_add_sync(0xffffffffu, sum);
        // this part of the tiles (counted without gaps)
        const int np = plo < phi ? (phi - plo + KT - 1) / KT : 0, no = klo < khi ? (khi - klo + KT - 1) / KT : 0;
        // (tiles times parts fits: at most 2^24 tiles, and parts only where the items are fewer than the pairs)
        const int a0 = (int)((unsigned)(np + no) * (unsigned)part / (unsigned)p.parts);
        const int a1 = (int)((unsigned)(np + no) * (unsigned)(part + 1) / (unsigned)p.parts);
        it.p_lo = a0 < np ? plo + a0 * KT : 0;
        it.p_hi = a0 < np ? (a1 >= np ? phi : plo + a1 * KT) : 0;
        it.o_lo = a1 > np ? klo + max(a0 - np, 0) * KT : 0;
        it.o_hi = a1 > np ? (a1 == np + no ? khi : klo + (a1 - np) * KT) : 0;
        it.gap = klo < khi && (unsigned)(khi - klo) - sum >= (unsigned)KT ? 1 : 0;
        it.tiles = (it.p_hi - it.p_lo + KT - 1) / KT;
        if (!it.gap) {
          it.tiles += max(it.o_hi - it.o_lo + KT - 1, 0) / KT;
        } else {
          // as TileIter goes over them
          TileIter ti;
          ti.init(p, it);
          int cur = it.o_lo;
#pragma unroll 1
          while (cur < it.o_hi) {
            cur = max(cur, ti.lo);
            const int hi = min(ti.hi, it.o_hi);
            if (cur < hi) {
              const int n = (hi - cur + KT - 1) / KT;
              it.tiles += n;
              cur += n * KT;
            }
            if (ti.b >= ti.b1) break;
            ++ti.b;
            ti.need(p.a);
          }
        }
      }
      if (lane == 0) {
        info[ib] = it;
        mbar_arrive(smem_u32(&info_full[ib]));
      }
      __syncwarp();
      if (it.tiles == 0) continue;
      if (items > 0 && !wait(q_empty, (uint32_t)(items - 1))) break;
      if (lane == 0) {
        if (rank == 0) mbar_expect_tx(smem_u32(q_full), (uint32_t)(2 * D * 2 * p.rows));
        const uint32_t bar = map_to_rank(smem_u32(q_full), 0);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d_pair(smem_u32(smem + c * ROWS * 128), &p.tmQ, bar, c * 64, 0, head, t0 + (int)rank * per);
      }
      __syncwarp();
      ++items;
    }
    if (rank == 0 && lane == 0 && items > 0) wait_drain(smem_u32(q_full), (uint32_t)(items - 1) & 1u);     // as in warp 8
  }
  } else if (warp < SM_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // ------------------------------------------------------------------------------------------ softmax
    const int quarter = warp & 3, half = warp >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t ocol = tmem + lanes + O_COL;
    const int nrows = row_count(p);
    const float c = p.a.scale * 1.4426950408889634f;
    const f32x2 c2 = x2_pack(c, c);
    const uint32_t p_full0 = map_to_rank(smem_u32(&p_full[0]), 0);
    const uint32_t x_mine = smem_u32(smem + L::words) + (uint32_t)(half * ROWS + r) * 4;
    const uint32_t x_other = smem_u32(smem + L::words) + (uint32_t)((half ^ 1) * ROWS + r) * 4;
    int g = 0, buf = 0, x_n = 0;          // tiles done, S buffer, exchanges
    uint32_t sphase = 0;
    bool ok = true;

    ItemInfo it, it_next;
    RowKeys rk, rk_next;
    int tok = 0, tok_next = 0;
    // the next item, and what this thread's row of it sees. A row that is not there needs no mask: its sums are not read.
    auto fetch = [&](int i) {
      const int ib = i & 1;
      if (!wait(&info_full[ib], (uint32_t)(i >> 1))) return false;
      it_next = info[ib];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&info_empty[ib]));
      const int row = it_next.row0 + (int)rank * p.rows + r;
      rk_next = {0, INT_MAX, 0, INT_MAX};
      tok_next = 0;
      if (it_next.row0 >= 0 && r < p.rows && row < nrows) {
        tok_next = row / p.group;
        rk_next = row_keys_in(p.a, it_next.b0 == it_next.b1 ? it_next.first
                                       : sequence_at(p.a, sequence_of(p.a, tok_next, it_next.b0, it_next.b1 + 1)), tok_next);
      }
      return true;
    };
    // The halves of a row exchange a value (maximum, sum) through one word each, whose lowest bit says which use of the word it
    // is: a word is used every other time, and written again only after the other side has gone on to the next one.
    // A maximum gives up its lowest bit for it, on both sides: it only says what the weights are relative to, so nothing is lost.
    // A sum keeps all its bits: it has no sign, whose place the shift frees.
    auto post = [&](uint32_t bits) {
      sts_volatile(x_mine + (uint32_t)((x_n & 1) * 2 * ROWS * 4), bits | (uint32_t)((x_n >> 1) & 1));
    };
    auto receive = [&](uint32_t& other) {
      const uint32_t at = x_other + (uint32_t)((x_n & 1) * 2 * ROWS * 4), tag = (uint32_t)((x_n >> 1) & 1);
      ++x_n;
      uint32_t v = lds_volatile(at);
      uint64_t t0 = 0;
      uint32_t seen = 0;
#pragma unroll 1
      for (uint32_t n = 1; !__all_sync(0xffffffffu, (v & 1u) == tag); ++n) {
        if ((n & 63u) == 0u) {
          const uint32_t now = *beat;
          if (t0 == 0 || now != seen) t0 = globaltimer();
          seen = now;
          const bool late = globaltimer() - t0 > p.timeout_ns;
          if (__any_sync(0xffffffffu, late || *abort_flag != 0)) {
            if (late) set_status(p.a.status, REAXMOE_ERR_DEVICE_TIMEOUT);
            *abort_flag = 1;
            return false;
          }
        }
        v = lds_volatile(at);
      }
      other = v & ~1u;
      return true;
    };
    auto cut = [](float v) { return __uint_as_float(__float_as_uint(v) & ~1u); };   // as the other side gets it
    // 32 scores -> weights 2^(c s - mc), their sums, and the packed weights to 16 TMEM columns; any: some row of the warp sees
    // some of the columns
    auto weights = [&](const uint32_t (&s)[32], bool any, float mc, f32x2 (&sum)[2], uint32_t dst) {
      uint32_t w[16];
      if (any) {
        const f32x2 nm = x2_pack(-mc, -mc);
#pragma unroll
        for (int x = 0; x < 32; x += 2) {
          float e0, e1;
          const f32x2 y = x2_fma(x2_pack(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), c2, nm);
          x2_unpack(y, e0, e1);
          e0 = ex2(e0);
          e1 = ex2(e1);
          w[x / 2] = pack2<BF>(e0, e1);
          sum[(x / 2) & 1] = x2_add(sum[(x / 2) & 1], x2_pack(e0, e1));
        }
      } else {
#pragma unroll
        for (int x = 0; x < 16; ++x) w[x] = 0u;
      }
      tc_st_32x32b_x16(dst, w);
    };
    auto hide = [&](uint32_t (&s)[32], uint32_t seen) {          // scores that the row does not see: weight 0
#pragma unroll
      for (int x = 0; x < 32; ++x) s[x] = (seen >> x) & 1u ? s[x] : 0xFF800000u;
    };

    if (!fetch(0)) ok = false;
    for (int i = 0; ok; ++i) {
      it = it_next;
      rk = rk_next;
      tok = tok_next;
      if (it.row0 < 0) break;
      const int row = it.row0 + (int)rank * p.rows + r;
      const bool live = r < p.rows && row < nrows;
      const bool any_live = __any_sync(0xffffffffu, live);
      const bool none = rk.p_lo >= rk.p_hi && rk.k_lo >= rk.k_hi;
      float m = -INFINITY, l = 0.0f;             // the maximum in use (of scores times c), the sum of this half's weights
      // keys from the part's end on are the next part's, whose first tile may begin inside this one where there are gaps
      const int p_hi = min(rk.p_hi, it.p_hi), k_hi = min(rk.k_hi, it.o_hi);
      // without gaps, tile j < np is the prefix's from p_lo + 128 j, the others are from o_lo + 128 (j - np); all rows of the
      // warp see all of tiles [pf, pf + pn) and [kf, kf + kn)
      const int np = (it.p_hi - it.p_lo + KT - 1) / KT;
      int pf = 0, pn = 0, kf = 0, kn = 0;
      TileIter ti;
      if (it.gap) {
        ti.init(p, it);
      } else {
        if (np > 0) {
          pf = max(__reduce_max_sync(0xffffffffu, rk.p_lo) - it.p_lo + KT - 1, 0) / KT;
          pn = max((__reduce_min_sync(0xffffffffu, p_hi) - it.p_lo) / KT - pf, 0);
        }
        if (it.tiles > np) {
          kf = max(__reduce_max_sync(0xffffffffu, rk.k_lo) - it.o_lo + KT - 1, 0) / KT;
          kn = max((__reduce_min_sync(0xffffffffu, k_hi) - it.o_lo) / KT - kf, 0);
          kf += np;
        }
      }
      struct Tile {
        bool full, some;                         // all rows of the warp see all 128 keys; some row sees some key
        bool any0, any1;                         // some row sees some of this thread's first / last 32 columns
        uint32_t seen0, seen1;                   // if not full: which of this thread's 64 columns its row sees
      } cur;
      auto next = [&](Tile& t, int j) {
        t.full = (unsigned)(j - pf) < (unsigned)pn || (unsigned)(j - kf) < (unsigned)kn;
        t.some = t.any0 = t.any1 = true;
        if (!t.full) {
          int start = j < np ? it.p_lo + j * KT : it.o_lo + (j - np) * KT;
          bool pre = j < np;
          if (it.gap) {
            start = ti.next(p);
            pre = ti.pre;
            ti.after();
          }
          const int a0 = (pre ? rk.p_lo : rk.k_lo) - start, a1 = (pre ? p_hi : k_hi) - start;   // columns [a0, a1) are seen
          t.some = __any_sync(0xffffffffu, a0 < KT && a1 > max(a0, 0));
          t.full = __all_sync(0xffffffffu, a0 <= 0 && a1 >= KT);
          auto seen = [&](int col) {                                   // of columns col .. col + 31
            const int f = min(max(a0 - col, 0), 32), e = min(max(a1 - col, 0), 32);
            const uint32_t below_e = e == 32 ? 0xffffffffu : (1u << e) - 1u, below_f = f == 32 ? 0xffffffffu : (1u << f) - 1u;
            return below_e & ~below_f;
          };
          t.seen0 = seen(half * 64);
          t.seen1 = seen(half * 64 + 32);
          t.any0 = __any_sync(0xffffffffu, t.seen0 != 0u);
          t.any1 = __any_sync(0xffffffffu, t.seen1 != 0u);
        }
      };
      uint32_t s0[32], s1[32];
      float mine = -INFINITY;
      auto scol = [&]() { return tmem + lanes + (uint32_t)(buf * KT); };
      auto load = [&](uint32_t (&x0)[32], uint32_t (&x1)[32]) {            // of the tile's scores, this half's columns
        tc_fence_after();
        tc_ld_32x32b_x32(scol() + half * 64, x0);
        tc_ld_32x32b_x32(scol() + half * 64 + 32, x1);
      };
      auto find_max = [&](const Tile& t, uint32_t (&x0)[32], uint32_t (&x1)[32]) {
        tc_wait_ld(x0);
        loaded(x1);
        if (!t.full) {
          hide(x0, t.seen0);
          hide(x1, t.seen1);
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 32; x += 2) {
          mx[0] = max3_nan(mx[0], __uint_as_float(x0[x]), __uint_as_float(x0[x + 1]));
          mx[1] = max3_nan(mx[1], __uint_as_float(x1[x]), __uint_as_float(x1[x + 1]));
        }
        mine = cut(max_nan(mx[0], mx[1]));
        post(__float_as_uint(mine));
      };
      // the softmax of one tile whose scores are in registers and whose half maxima are posted
      auto weigh = [&](const Tile& t, uint32_t (&x0)[32], uint32_t (&x1)[32]) {
        uint32_t other;
        if (!receive(other)) return false;
        const float top = max_nan(__uint_as_float(other), mine) * c;
        if (!(top < INFINITY)) l = NAN;          // a score that is NaN or infinite: so are the row's weights
        const bool grow = top - m > THR;         // from -inf on the first key
        const bool rescale = grow && m != -INFINITY;
        if (__any_sync(0xffffffffu, rescale)) {
          const float f = rescale ? ex2(m - top) : 1.0f;
          l *= f;
          if (!wait(&pv_done[(g - 1) & 1], (uint32_t)((g - 1) >> 1))) return false;
          tc_fence_after();
          constexpr int HC = D / 2;              // this half's columns of O
#pragma unroll 1
          for (int x = 0; x < HC; x += 32) {
            uint32_t o[32];
            tc_ld_32x32b_x32(ocol + half * HC + x, o);
            tc_wait_ld(o);
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            tc_st_32x32b_x32(ocol + half * HC + x, o);
          }
        }
        if (grow) m = top;
        const float mc = (m == -INFINITY ? 0.0f : m) - SHIFT;
        f32x2 sum[2] = {0ull, 0ull};
        // P takes the place of the first 64 columns of S, which both halves have read
        weights(x0, t.any0, mc, sum, scol() + half * 32);
        weights(x1, t.any1, mc, sum, scol() + half * 32 + 16);
        float y0, y1;
        x2_unpack(x2_add(sum[0], sum[1]), y0, y1);
        l += y0 + y1;
        return true;
      };
      auto nothing = [&]() {                     // no row of the warp sees any key of the tile
        uint32_t z[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) z[x] = 0u;
        tc_st_32x32b_x16(scol() + half * 32, z);
        tc_st_32x32b_x16(scol() + half * 32 + 16, z);
      };
      auto done = [&]() {
        if (any_live) {
          tc_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(p_full0 + (uint32_t)(buf * 8));
        ++g;
        if (++buf == NB) {
          buf = 0;
          sphase ^= 1u;
        }
      };
      if (it.tiles > 0) next(cur, 0);
#pragma unroll 1
      for (int j = 0; j < it.tiles; ++j) {
        if (!(ok = wait(&s_full[buf], sphase))) break;
        if (any_live) {
          if (cur.some) {
            load(s0, s1);
            find_max(cur, s0, s1);
            if (!(ok = weigh(cur, s0, s1))) break;
          } else {
            nothing();
          }
        }
        done();
        if (j + 1 < it.tiles) next(cur, j + 1);
      }
      if (!ok) break;
      // the sums, for the output warps
      if (any_live) {
        uint32_t other;
        post(__float_as_uint(l) << 1);
        if (!(ok = receive(other))) break;
        l += __uint_as_float(other >> 1);
      }
      if (half == 0) {
        if (i > 0 && !(ok = wait(l_empty, (uint32_t)(i - 1)))) break;
        inv_l[r] = none ? 0.0f : 1.0f / l;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(l_full));
        if (live) {
          const int in_group = row - tok * p.group;
          if (p.partial)
            p.part_ml[((int64_t)it.part * p.a.kv_heads + it.head) * ((int64_t)p.tiles * 2 * p.rows) + row] = make_float2(m, l);
          else if (p.a.lse != nullptr)
            p.a.lse[(int64_t)tok * p.a.q_heads + it.head * p.group + in_group] =
                none ? -INFINITY : (m - SHIFT + __log2f(l)) * 0.6931471805599453f;
        }
      }
      if (!(ok = fetch(i + 1))) break;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OUT));
    // ------------------------------------------------------------------------------------------ output
    const int quarter = warp - OUT_WARP0, r = quarter * 32 + lane;
    const uint32_t ocol = tmem + ((uint32_t)(quarter * 32) << 16) + O_COL;
    const int nrows = row_count(p);
    const uint32_t leader_o = map_to_rank(smem_u32(o_empty), 0);
    int items = 0;
    for (int i = 0;; ++i) {
      const int ib = i & 1;
      if (!wait(&info_full[ib], (uint32_t)(i >> 1))) break;
      const ItemInfo it = info[ib];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&info_empty[ib]));
      if (it.row0 < 0) break;
      const bool tiles = it.tiles > 0;
      const int row = it.row0 + (int)rank * p.rows + r;
      const bool live = r < p.rows && row < nrows;
      const int tok = live ? row / p.group : 0, head = it.head * p.group + (live ? row - tok * p.group : 0);
      uint16_t* out = static_cast<uint16_t*>(p.a.out) + (int64_t)tok * p.a.out_stride + head * p.a.out_head_stride;
      float* part = p.part_o + (((int64_t)it.part * p.a.kv_heads + it.head) * ((int64_t)p.tiles * 2 * p.rows) + row) * D;
      if (!wait(l_full, (uint32_t)i)) break;
      const float inv = inv_l[r];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(l_empty));
      if (tiles && !wait(o_full, (uint32_t)items)) break;
      const f32x2 inv2 = x2_pack(inv, inv);
      f32x2 check = 0ull;                        // becomes NaN with the first value that is not finite
      if (__any_sync(0xffffffffu, live)) {
        tc_fence_after();
#pragma unroll 1
        for (int x = 0; x < D; x += 32) {
          uint32_t o[32];
          if (tiles) {
            tc_ld_32x32b_x32(ocol + x, o);
            tc_wait_ld(o);
          } else {
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = 0u;
          }
          if (p.partial) {
            if (live) {
#pragma unroll
              for (int y = 0; y < 8; ++y)
                reinterpret_cast<float4*>(part + x)[y] =
                    make_float4(__uint_as_float(o[4 * y]), __uint_as_float(o[4 * y + 1]), __uint_as_float(o[4 * y + 2]),
                                __uint_as_float(o[4 * y + 3]));
            }
          } else {
            uint32_t v[2][8];
#pragma unroll
            for (int y = 0; y < 32; y += 2) {
              const f32x2 z = x2_mul(x2_pack(__uint_as_float(o[y]), __uint_as_float(o[y + 1])), inv2);
              check = x2_fma(z, 0ull, check);
              float z0, z1;
              x2_unpack(z, z0, z1);
              v[y / 16][(y / 2) & 7] = pack2<BF>(in_range<BF>(z0), in_range<BF>(z1));
            }
            if (live) {
              if (p.wide_out) {
                st_global_v8(out + x, v[0]);
                st_global_v8(out + x + 16, v[1]);
              } else {
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  *reinterpret_cast<uint4*>(out + x + y * 8) =
                      make_uint4(v[y / 2][(y & 1) * 4], v[y / 2][(y & 1) * 4 + 1], v[y / 2][(y & 1) * 4 + 2], v[y / 2][(y & 1) * 4 + 3]);
              }
            }
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      __syncwarp();
      if (tiles) {
        if (lane == 0) mbar_arrive_cluster(leader_o);
        ++items;
      }
      // 0 x (an infinity or NaN of a value that the row does not see) is NaN: such rows are done again key by key. A sum that
      // is NaN itself came from a key that the row does see.
      float x0, x1;
      x2_unpack(check, x0, x1);
      uint32_t again = __ballot_sync(0xffffffffu, live && inv == inv && !(x0 + x1 == 0.0f));
      auto alive = [&]() {                       // the other warps of both CTAs may have to wait for this one
        if (lane < 2) st_cluster_u32(map_to_rank(smem_u32(const_cast<uint32_t*>(beat)), (uint32_t)lane), (uint32_t)globaltimer());
      };
      if (again != 0u) again = unexplained_rows<D, BF>(p.a, again, tok, head, alive);
#pragma unroll 1
      for (; again != 0u; again &= again - 1u) {
        const int src = __ffs(again) - 1;
        row_by_warp<D, BF>(p.a, __shfl_sync(0xffffffffu, tok, src), __shfl_sync(0xffffffffu, head, src), false, alive);
      }
    }
  }
  // After an abort the other CTA may have loads under way that count on the leader's barriers without the leader's knowledge,
  // and item numbers and arrivals may be on their way to the other CTA. Whatever a warp started before it comes here has the
  // time to land: the warp that set the flag comes here after it.
  if (*abort_flag != 0) settle();
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
  constexpr float SHIFT = BF ? 0.0f : 4.0f;      // as in pair_kernel
  constexpr int W = D / 32;
  const int id = (int)(blockIdx.x * 8 + (threadIdx.x >> 5));     // fits: the rows of fewer tiles than there are pairs
  const int lane = threadIdx.x & 31;
  const int tok = id / p.a.q_heads, head = id - tok * p.a.q_heads;
  if (tok * p.group >= row_count(p)) return;
  const int kvh = head / p.group;
  const int64_t stride = (int64_t)p.tiles * 2 * p.rows;
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
    acc[i] = none ? 0.0f : in_range<BF>(acc[i] * inv);
    bad |= !(fabsf(acc[i]) < INFINITY);
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
  __syncwarp();
  if (__any_sync(0xffffffffu, bad) && l == l) row_by_warp<D, BF>(p.a, tok, head, false);
}

// Row tiles, parts of the keys, and the workspace: counter, partial maxima and sums, partial outputs (of pair_kernel, of
// few_kernel).
struct Plan {
  int group, rows, tiles, parts, items, pairs;
  bool few;
  int chunk, units;
  size_t ml, o, few_ml, few_o, total;
};

static Plan plan(const reaxmoe_attention_args& a, int num_sms) {
  Plan pl;
  pl.group = a.q_heads / a.kv_heads;
  const int64_t rows = a.q_tokens * pl.group;
  pl.rows = ROWS / pl.group * pl.group;
  pl.tiles = (int)ceil_div64(rows, 2 * pl.rows);
  const int64_t base = (int64_t)pl.tiles * a.kv_heads;
  const int pairs = num_sms / 2 > 0 ? num_sms / 2 : 1;
  // A generation step (no more query tokens than sequences, with some keys each) goes to few_kernel: 64 sequences of 2304 keys
  // take 143 us there against 453 in tiles at D = 64 (16 KV heads), 137 against 217 at D = 128 (8), 250 against 241 at D = 256
  // (8); one of 100 keys is quicker in tiles (12 to 18 us against 10 to 14). With a prefix it is a launch more, which pays from
  // some own keys on at D = 64 (256 sequences of 100 behind 16384: 98 us against 138), at D = 128 from more (of 100 140
  // against 138, of 500 221 against 289), at D = 256 hardly ever (of 500 282 against 284, 64 of 2500 305 against 289).
  // Over 380 sizes (1 to 256 sequences of 16 to 2500 keys behind 0 to 16384, 1 to 16 KV heads) what the rule picks takes 3.2,
  // 1.3 and 1.0 % longer on the geometric average than the better of the two at D = 64, 128 and 256 (tiles alone 30, 12 and
  // 4 %), and 45 % at worst (256 sequences of 16 keys behind 512, D = 64, 2 KV heads: 33 us against 22).
  pl.few = pl.group <= FEW_ROWS && a.q_tokens <= a.seqs && a.k_tokens >= 16 * (int64_t)a.seqs && a.k_tokens > 0 &&
           (a.prefix == 0 || (a.head_dim == 64 && a.k_tokens >= 4096) || (a.head_dim == 128 && a.k_tokens >= 32768));
  const int64_t keys = a.prefix + (pl.few ? 0 : a.k_tokens);
  // split the keys when the tiles leave half of the pairs idle, into parts of at least 512 keys
  int64_t parts = base > 0 && base * 2 <= pairs ? pairs / base : 1;
  const int64_t most = ceil_div64(keys, 512);
  if (parts > most) parts = most;
  pl.parts = (int)(parts < 1 ? 1 : parts);
  const int64_t items = base * pl.parts;
  pl.items = (int)items;
  pl.pairs = (int)(items < pairs ? items : pairs);
  // units of few_kernel, of at least 64 keys: with few sequences one for every warp of the device (each sequence may have one
  // more than its share), else about five, so that the ends of sequences even out (64 sequences of 2304 keys, D = 256: 260 us
  // with two a warp, 252 with three and four, 250 with five and six, 251 with eight; D = 128: 139, 136, 139, 138, 140, 141;
  // 200 of 700, D = 256: 252, 240, 240, 234, 246, 233: more than two matters, how many does not)
  const int64_t warps = ceil_div64((int64_t)num_sms * FEW_WARPS, a.kv_heads);       // for each KV head
  int64_t chunk = ceil_div64(a.k_tokens, warps >= 8 * (int64_t)a.seqs ? warps - a.seqs : 5 * warps);
  chunk = chunk < 64 ? 64 : ceil_div64(chunk, 16) * 16;
  pl.chunk = (int)chunk;
  pl.units = pl.few ? (int)(ceil_div64(a.k_tokens, chunk) + a.seqs) : 0;
  auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
  const size_t prow = pl.parts > 1 || (pl.few && a.prefix > 0) ? (size_t)pl.parts * a.kv_heads * pl.tiles * 2 * pl.rows : 0;
  const size_t frow = (size_t)pl.units * a.kv_heads * FEW_ROWS;
  pl.ml = 256;
  pl.o = up(pl.ml + prow * 8);
  pl.few_ml = up(pl.o + prow * a.head_dim * 4);
  pl.few_o = up(pl.few_ml + frow * 8);
  pl.total = prow == 0 && frow == 0 && pl.items <= pl.pairs ? 16 : pl.few_o + frow * a.head_dim * 4;
  return pl;
}

// the kernel's dynamic shared memory, allowed once per device (bit = device; devices from 64 on every time)
template <typename K>
static int allow_smem(K kfn, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return REAXMOE_ERR_CUDA;
  const uint64_t bit = device < 64 ? 1ull << device : 0ull;
  if ((done.load(std::memory_order_acquire) & bit) != 0) return 0;
  if (cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return REAXMOE_ERR_CUDA;
  done.fetch_or(bit, std::memory_order_release);
  return 0;
}

template <int D, bool BF>
static int launch_few(const AttentionLaunch& l, const Plan& pl, const Params* prefix, cudaStream_t s) {
  const reaxmoe_attention_args& a = l.a;
  uint8_t* ws = static_cast<uint8_t*>(l.workspace);
  FewParams f;
  memset(&f, 0, sizeof(f));
  f.a = a;
  f.group = pl.group;
  f.chunk = pl.chunk;
  f.units = pl.units;
  f.ml = reinterpret_cast<float2*>(ws + pl.few_ml);
  f.o = reinterpret_cast<float*>(ws + pl.few_o);
  if (prefix != nullptr) {
    f.prefix_parts = pl.parts;
    f.prefix_rows = pl.tiles * 2 * pl.rows;
    f.prefix_ml = prefix->part_ml;
    f.prefix_o = prefix->part_o;
  }
  static std::atomic<uint64_t> allowed{0};
  if (allow_smem(few_kernel<D, BF>, FewLayout<D>::total, allowed)) return REAXMOE_ERR_CUDA;
  const int64_t tasks = (int64_t)pl.units * a.kv_heads;
  const int64_t blocks = (int64_t)l.num_sms * (l.whole_device ? FewLayout<D>::BLOCKS : 1);
  const int grid = (int)(tasks < blocks ? tasks : blocks);
  few_kernel<D, BF><<<grid, FEW_WARPS * 32, FewLayout<D>::total, s>>>(f);
  // partial results a row on the average: a warp joins up to about 32
  const int64_t rows = a.q_tokens * a.q_heads, results = pl.units / a.seqs + (prefix != nullptr ? pl.parts : 0);
  if (results <= 32)
    join_kernel<D, BF, 1><<<(unsigned)ceil_div64(rows, JOIN_WARPS), JOIN_WARPS * 32, 0, s>>>(f);
  else
    join_kernel<D, BF, JOIN_WARPS><<<(unsigned)rows, JOIN_WARPS * 32, 0, s>>>(f);
  return cudaPeekAtLastError() == cudaSuccess ? 0 : REAXMOE_ERR_CUDA;
}

template <int D, bool BF>
static int launch_t(const AttentionLaunch& l, const Plan& pl, cudaStream_t s) {
  const reaxmoe_attention_args& a = l.a;
  Params p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.group = pl.group;
  p.rows = pl.rows;
  p.tiles = pl.tiles;
  p.parts = pl.parts;
  p.items = pl.items;
  p.wide_out = ((reinterpret_cast<uintptr_t>(a.out) & 31u) == 0 && (a.out_stride & 15) == 0 && (a.out_head_stride & 15) == 0) ? 1 : 0;
  uint8_t* ws = static_cast<uint8_t*>(l.workspace);
  p.counter = pl.items > pl.pairs ? reinterpret_cast<int*>(ws) : nullptr;
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
  p.part_o = reinterpret_cast<float*>(ws + pl.o);
  p.timeout_ns = l.timeout_ns;
  p.prefix_only = pl.few ? 1 : 0;
  p.partial = pl.parts > 1 || pl.few ? 1 : 0;
  if (pl.few && a.prefix == 0) return launch_few<D, BF>(l, pl, nullptr, s);
  constexpr int VB = D == 64 ? 32 : 64;
  if (make_map_rows(&p.tmQ, a.q, a.q_tokens, a.q_stride, a.kv_heads, pl.group, a.q_head_stride, D, pl.rows / pl.group))
    return REAXMOE_ERR_CUDA;
  if (a.k_tokens > 0 && !pl.few &&
      (make_map_heads(&p.tmK, a.k, a.k_tokens, a.k_stride, a.kv_heads, a.k_head_stride, D, 64, 64) ||
       make_map_heads(&p.tmV, a.v, a.k_tokens, a.v_stride, a.kv_heads, a.v_head_stride, D, VB, KT)))
    return REAXMOE_ERR_CUDA;
  if (a.prefix > 0 &&
      (make_map_heads(&p.tmPK, a.prefix_k, a.prefix, a.prefix_k_stride, a.kv_heads, a.prefix_k_head_stride, D, 64, 64) ||
       make_map_heads(&p.tmPV, a.prefix_v, a.prefix, a.prefix_v_stride, a.kv_heads, a.prefix_v_head_stride, D, VB, KT)))
    return REAXMOE_ERR_CUDA;
  static std::atomic<uint64_t> allowed{0};
  if (allow_smem(pair_kernel<D, BF>, Layout<D>::total, allowed)) return REAXMOE_ERR_CUDA;
  if (p.counter != nullptr && cudaMemsetAsync(p.counter, 0, sizeof(int), s) != cudaSuccess) return REAXMOE_ERR_CUDA;
  pair_kernel<D, BF><<<2 * pl.pairs, THREADS, Layout<D>::total, s>>>(p);
  if (pl.few) return launch_few<D, BF>(l, pl, &p, s);
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
