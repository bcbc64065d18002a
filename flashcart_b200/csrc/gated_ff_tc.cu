// Gated feed-forward block on tcgen05 tensor cores, fed by TMA (sm_100a): float32 rows as
// 3xTF32 products, and the input gradient of bfloat16 rows that are too long for gated_ff_bf16.cu.
//
// Mathematics and row layout: gated_ff.cu. The scales s_l, s_g are folded into the split
// weights, so the accumulators hold v_k and z_l - b_l themselves.
//
// A work item is one rank l of 128 rows and 64 output channels: first the gate product
// x_0 Wg_l, kept by the epilogue warps in registers, then the 2l+1 value products, each
// multiplied by the gate's activation on its way out. So y is written once, and neither gates
// nor values touch memory. Three modes share the kernel:
//   FWD  y_k = a_l v_k
//   PRE  the backward's first half: z_l and v_k again; g comes in by TMA while they are
//        computed; dv_k = g a_l goes out, sum_m g v_k stays in registers until the rank is
//        done and dz_l goes out
//   DX   dx_k = dv_k Wv_l (+ sum_l dz_l Wg_l for k = 0): items are (128 rows, component)
//
// What bounds it: DRAM (x in, y out: 453 MB for 27,648 x 16 rows of 128 channels, 70 us at the
// copy rate), with the tensor cores close behind (66 us: three products at half the measured
// bfloat16 rate). Measured there: FWD 110 us (4.1 TB/s), PRE 157 us (736 MB, 4.7 TB/s), DX 114 us
// (510 MB, 4.5 TB/s); in a loop of seconds the power limit takes another sixth. A slab's MMAs take
// 385 cycles and its copy 220 of the 870 that it costs: what is left is the latency of the
// barriers between the roles.
// A ring whose stages held A and the weights' slabs together was three deep in shared memory and
// waited for its copies (FWD 149 us, DX 143 us: gated_ff_stream.cu, which still serves above 128
// channels). Here the item's two weight matrices stay in shared memory (64 output channels x 128 x
// hi, lo: 64 KB each), work lists are ordered by rank so that they are loaded a few times per
// launch, and the ring holds A slabs alone. The price is that x is read from L2 once per 64 output
// channels.
//
// A tensor-core accumulation truncates the running sum (measured relative error of one
// accumulator: 4.5e-7 after 12 instructions, 8.2e-7 after 24, 1.6e-6 after 48), so a slab's
// small products (Ahi Wlo, Alo Whi) go in before its Ahi Whi, the even and the odd slabs of a
// pass go to two accumulators, and the epilogue adds them.
//
// Roles of the 20 warps (one persistent CTA per SM):
//   warp 0       TMA producer of A slabs, and the CTA's draw from its work list
//   warps 1, 3   MMA issue
//   warp 2       TMA producer of the weights
//   warps 4-11   splitters: the slab (128 rows x 32 channels) to tf32 parts in tensor memory;
//                two groups of four take the slabs in turn
//   warps 12-19  epilogue: two per lane quarter, 32 columns each
// Waits are bounded: on expiry the CTA raises FC_DEV_TIMEOUT, all roles stop, copies and MMAs
// in flight are drained and tensor memory is freed.
#include "gated_ff_tc.cuh"

#ifndef FC_HOST_EMU

#include <algorithm>

namespace fc {
namespace gtc {

constexpr int BN = 64;
constexpr int W_LO = (BN * BK * 4) >> 4;  // descriptor step from a slab's Whi to its Wlo
constexpr int W_SLAB = 2 * BN * BK * 4;  // [Whi | Wlo] of one k slab: 128 K-major rows, 16 KB
constexpr int MAX_NK = 4;                // k slabs of a resident matrix
// Tensor memory: four A slots of hi | lo columns (an MMA's slot is refilled about 700 cycles
// after it is issued, two slabs' worth of MMAs) and two accumulators.
constexpr int NACC = 2 /* (the code flips between them) */, ACC_W = 2 * BN, A_COLS = 256;
constexpr int MAX_STAGES = 8;
constexpr int SMEM_MAX = 227 * 1024;
constexpr int SPLIT_WARP0 = 4, EPI_WARP0 = 12, EPI_WARPS = 8, TC_THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int TC_REGS = 96;  // per thread at launch; the epilogue takes what the first four warps leave

template <int MODE, typename T>
struct Cfg {
  static constexpr int TILE_A = BM * BK * 4;
  static constexpr int A_STAGE = 2 * BK;  // tensor-memory columns: hi and lo parts
  // Slots of the A ring. Even, so that a slot belongs to one splitter group and one MMA warp,
  // whose waits miss none of its barriers' phases. PRE keeps the gates' slopes behind them.
  static constexpr int A_RING = MODE == PRE ? 2 : 4, Z_COL = 192;
  static constexpr int BUFS = MODE == PRE ? 2 : 1;   // staging boxes per epilogue warp
  static constexpr int FIXED = EPI_WARPS * BUFS * EPI_BUF + BAR_BYTES + 1024;
  static_assert(A_RING * A_STAGE <= (MODE == PRE ? Z_COL : A_COLS) && A_COLS + NACC * ACC_W <= 512, "tensor memory");
  // even, so that a stage always belongs to the same splitter group: its waits tell one phase
  // of a stage's barrier from the next only if they miss none
  static int stages(int nk) { return std::min(MAX_STAGES, (SMEM_MAX - FIXED - 2 * nk * W_SLAB) / TILE_A) & ~1; }
  static int smem(int nk, int st) { return FIXED + 2 * nk * W_SLAB + st * TILE_A; }
};

// An item's product passes: FWD, PRE the gate, then a value product per component, by the
// rank's gate matrix (weight slot 0) and value matrix (slot 1), which stay until the rank
// changes. DX one pass per component by the rank's transposed value matrix (slot 0); component
// 0 adds up ranks + 1 passes, through all transposed gate matrices in alternating slots (with
// one rank both simply stay).
template <int MODE, typename T>
__global__ void __launch_bounds__(TC_THREADS, 1) gated_tc_kernel(const __grid_constant__ Maps mp, const Args a) {
  using C = Cfg<MODE, T>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = a.stages, nk = a.nk;
  uint8_t* wmem = smem;                          // two weight slots of nk slabs
  uint8_t* ring = wmem + 2 * nk * W_SLAB;        // A stages
  uint8_t* epi = ring + S * C::TILE_A;           // staging boxes
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + EPI_WARPS * C::BUFS * EPI_BUF);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* a_full = empty + MAX_STAGES;
  uint64_t* a_free = a_full + C::A_RING;
  uint64_t* w_full = a_free + C::A_RING;         // [slot][k slab]
  uint64_t* w_free = w_full + 2 * MAX_NK;
  uint64_t* acc_full = w_free + 2;
  uint64_t* acc_empty = acc_full + NACC;
  uint64_t* sched_full = acc_empty + NACC;
  uint64_t* sched_empty = sched_full + SCHED;
  uint64_t* drain = sched_empty + SCHED;
  uint64_t* aux = drain + 1;                     // per epilogue warp and box: g has landed
  int* sched = reinterpret_cast<int*>(aux + EPI_WARPS * C::BUFS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sched + SCHED);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * MAX_STAGES + 2 * C::A_RING + 2 * MAX_NK + 2 + 2 * NACC + 2 * SCHED + 1 + EPI_WARPS * C::BUFS) * 8 +
                        SCHED * 4 + 8 <=
                    BAR_BYTES,
                "barriers");

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 32) {
    auto init = [](uint64_t* b, int n) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n));
    };
    for (int s = 0; s < MAX_STAGES; ++s) {
      init(&full[s], 1);
      init(&empty[s], 4);
    }
    for (int b = 0; b < C::A_RING; ++b) {
      init(&a_full[b], 4);
      init(&a_free[b], 1);
    }
    for (int b = 0; b < 2 * MAX_NK; ++b) init(&w_full[b], 1);
    for (int b = 0; b < 2; ++b) init(&w_free[b], 2);
    for (int b = 0; b < NACC; ++b) {
      init(&acc_full[b], 2);
      init(&acc_empty[b], EPI_WARPS);
    }
    for (int b = 0; b < SCHED; ++b) {
      init(&sched_full[b], 1);
      init(&sched_empty[b], 3 + 8 + EPI_WARPS);  // MMA, weights, splitter and epilogue warps
    }
    init(drain, 2);
    for (int b = 0; b < EPI_WARPS * C::BUFS; ++b) init(&aux[b], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;
  const int ct = (int)blockIdx.x % a.n_ct;  // this CTA's 64 output channels
  const bool cycle = MODE == DX && a.ranks > 1;

  // the q-th item of this CTA (-1: no more, or a wait gave up), for one thread or a whole warp
  auto item_one = [&](int q) -> int {
    const int s = q % SCHED;
    if (!wait_phase(smem_u32(&sched_full[s]), (uint32_t)((q / SCHED) & 1), abort_flag)) return -1;
    const int it = *reinterpret_cast<volatile int*>(&sched[s]);
    arrive(smem_u32(&sched_empty[s]));
    return it;
  };
  auto item_warp = [&](int q) -> int {
    const int s = q % SCHED;
    if (!wait_warp(smem_u32(&sched_full[s]), (uint32_t)((q / SCHED) & 1), abort_flag)) return -1;
    const int it = *reinterpret_cast<volatile int*>(&sched[s]);
    __syncwarp();
    if (lane == 0) arrive(smem_u32(&sched_empty[s]));
    return it;
  };
  auto passes_of = [&](const WorkItem& w) { return MODE == DX ? (w.k0 == 0 ? a.ranks + 1 : w.nm) : 1 + w.nm; };

  if (warp < SPLIT_WARP0) {
    FC_SETMAXNREG_DEC(40);
    if (warp == 0 && elect_one()) {
      // ---------------------------------------------------------------- A producer, work list
      const int first = (int)blockIdx.x / a.n_ct, group = (int)gridDim.x / a.n_ct;
      int next = first;
      int s = 0;
      uint32_t lap = 0;  // of the ring
      int64_t g = 0;
      bool ok = true;
      for (int q = 0; ok; ++q) {
        const int s4 = q % SCHED;
        if (q >= SCHED &&
            !wait_phase(smem_u32(&sched_empty[s4]), (uint32_t)((q / SCHED - 1) & 1), abort_flag))
          break;
        const int it = next < a.items ? next : -1;
        *reinterpret_cast<volatile int*>(&sched[s4]) = it;
        arrive(smem_u32(&sched_full[s4]));
        if (it < 0) break;
        next = group + atomicAdd(a.counter + ct, 1);
        const WorkItem w = work_item(a, it);
        const int passes = passes_of(w);
        for (int p = 0; p < passes && ok; ++p) {
          const bool gates = MODE == DX && w.k0 == 0 && p > 0;
          const CUtensorMap* ma = gates ? &mp.a2 : &mp.a;
          const int z = gates ? p - 1 : MODE == DX ? w.k0 + p : (p == 0 ? 0 : w.k0 + p - 1);
          // have the next pass's operands in L2: the ring's stages alone do not cover DRAM
          if (p + 1 < passes && (MODE != DX || w.k0 > 0)) {
            const int zn = w.k0 + p + (MODE == DX ? 1 : 0);
            tma_prefetch_3d(&mp.ap, 0, w.tile * BM, zn);
            if (MODE == PRE) tma_prefetch_3d(&mp.gp, ct * BN, w.tile * BM, zn);
          } else if (p + 1 == passes && next < a.items) {
            const WorkItem wn = work_item(a, next);
            tma_prefetch_3d(&mp.ap, 0, wn.tile * BM, MODE == DX ? wn.k0 : 0);
          }
          for (int kt = 0; kt < nk; ++kt, ++g) {
            if (lap > 0 && !wait_phase(smem_u32(&empty[s]), (lap - 1) & 1u, abort_flag)) {
              ok = false;
              break;
            }
            const uint32_t fb = smem_u32(&full[s]);
            arrive_tx(fb, C::TILE_A);
            tma_load_3d(smem_u32(ring + s * C::TILE_A), ma, kt * BK, w.tile * BM, z, fb);
            if (++s == S) {
              s = 0;
              ++lap;
            }
          }
        }
      }
      // the last copy into every stage must have landed before the CTA exits
      for (int t = 0; t < S; ++t) {
        const int64_t uses = g > t ? (g - 1 - t) / S + 1 : 0;
        if (uses > 0) drain_bar(smem_u32(&full[t]), (uint32_t)((uses - 1) & 1));
      }
    } else if (warp == 2 && elect_one()) {
      // ---------------------------------------------------------------- weight producer
      int rank = -1, loads0 = 0, loads1 = 0;
      bool ok = true;
      auto load = [&](int slot, int mat, int& loads) {
        if (loads > 0 && !wait_phase(smem_u32(&w_free[slot]), (uint32_t)((loads - 1) & 1), abort_flag)) {
          ok = false;
          return;
        }
        for (int kt = 0; kt < nk; ++kt) {
          uint8_t* to = wmem + (slot * nk + kt) * W_SLAB;
          const uint32_t fb = smem_u32(&w_full[slot * MAX_NK + kt]);
          arrive_tx(fb, W_SLAB);
          tma_load_3d(smem_u32(to), &mp.b, kt * BK, ct * BN, mat, fb);
          tma_load_3d(smem_u32(to + W_SLAB / 2), &mp.b, kt * BK, ct * BN, mat + 2 * a.ranks, fb);
        }
        ++loads;
      };
      for (int q = 0; ok; ++q) {
        const int it = item_one(q);
        if (it < 0) break;
        const WorkItem w = work_item(a, it);
        if (cycle && w.k0 == 0) {
          for (int p = 0; p <= a.ranks && ok; ++p) {
            const int mat = p == 0 ? 0 : a.ranks + p - 1;
            if (p & 1) load(1, mat, loads1);
            else load(0, mat, loads0);
          }
          rank = -1;
        } else if (w.l != rank) {
          rank = w.l;
          load(0, MODE == DX ? w.l : a.ranks + w.l, loads0);
          if (!cycle && ok) load(1, MODE == DX ? a.ranks : w.l, loads1);
        }
      }
      for (int kt = 0; kt < nk; ++kt) {
        if (loads0 > 0) drain_bar(smem_u32(&w_full[kt]), (uint32_t)((loads0 - 1) & 1));
        if (loads1 > 0) drain_bar(smem_u32(&w_full[MAX_NK + kt]), (uint32_t)((loads1 - 1) & 1));
      }
    } else if (warp == 1 || warp == 3) {
      // ---------------------------------------------------------------- MMA issue
      // Two warps, one for the even slabs of the ring and one for the odd: a slab's MMAs take 385
      // cycles, and the barrier operations around them as long again, so each warp issues while
      // the other one asks. Their sums go to the two halves of the accumulator. A whole warp
      // walks the loop (its addresses and descriptors stay uniform) and one lane issues.
      const int mine = warp >> 1;
      const uint64_t desc = make_desc(smem_u32(wmem));
      const uint32_t slot_step = (uint32_t)(nk * (W_SLAB >> 4));
      int rank = -1;
      uint32_t w_phase = 3u, held = 0u, check = 0u;  // per slot: phase of its last load, unreleased, not yet seen
      int par = 0;  // parity of the pass's first slab
      uint32_t as = (uint32_t)mine, a_phase = 0, ab = 0, acc_phase = 0;  // own A slot in turn, accumulator
      bool ok = true;
      bool a_ready = false, acc_ready = false;  // answers about the next slab and accumulator
      auto fresh = [&](int slot) {  // the slot's next matrix: all that read its last one is issued
        const uint32_t bit = 1u << slot;
        if ((held & bit) && elect_one()) commit(smem_u32(&w_free[slot]));
        held |= bit;
        check |= bit;
        w_phase ^= bit;
      };
      for (int q = 0; ok; ++q) {
        const int it = item_warp(q);
        if (it < 0) break;
        const WorkItem w = work_item(a, it);
        const int passes = passes_of(w);
        const bool through = cycle && w.k0 == 0;
        if (through) {
          rank = -1;
        } else if (w.l != rank) {
          rank = w.l;
          fresh(0);
          if (!cycle) fresh(1);
        }
        for (int p = 0; p < passes; ++p) {
          const int slot = through ? (p & 1) : (cycle || p == 0) ? 0 : 1;
          if (through) fresh(slot);
          if (!acc_ready) ok = wait_warp(smem_u32(&acc_empty[ab]), acc_phase ^ 1u, abort_flag);
          acc_ready = false;
          const uint32_t d = tmem + (uint32_t)A_COLS + ab * (uint32_t)ACC_W + (uint32_t)(mine * BN);
          const uint32_t ab_next = ab ^ 1u, acc_next = acc_phase ^ ab;
          const uint64_t db0 = desc + (slot ? slot_step : 0u);
          const bool check_w = (check >> slot) & 1u;
          const int first = mine ^ par;
#pragma unroll 1
          for (int kt = first; kt < nk; kt += 2) {
            if (check_w)
              ok = ok && wait_warp(smem_u32(&w_full[slot * MAX_NK + kt]), (w_phase >> slot) & 1u, abort_flag);
            if (!a_ready) ok = ok && wait_warp(smem_u32(&a_full[as]), a_phase, abort_flag);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;");
            const bool wrap = as + 2 >= (uint32_t)C::A_RING;
            const uint32_t as_next = wrap ? (uint32_t)mine : as + 2, ph_next = a_phase ^ (wrap ? 1u : 0u);
            const bool peek_a = peek_parity(smem_u32(&a_full[as_next]), ph_next);
            const bool peek_acc = peek_parity(smem_u32(&acc_empty[ab_next]), acc_next ^ 1u);
            const uint64_t db = db0 + (uint64_t)(kt * (W_SLAB >> 4));
            const uint32_t tah = tmem + as * (uint32_t)C::A_STAGE, tal = tah + (uint32_t)BK;
            if (elect_one()) {
              // the small products first: the sum that each accumulation truncates is then small
#pragma unroll
              for (int kk = 0; kk < BK / 8; ++kk) {
                mma_ta<BN>(d, tah + kk * 8, db + W_LO + 2 * kk, (kt > first || kk > 0) ? 1u : 0u);
                mma_ta<BN>(d, tal + kk * 8, db + 2 * kk, 1u);
              }
#pragma unroll
              for (int kk = 0; kk < BK / 8; ++kk) mma_ta<BN>(d, tah + kk * 8, db + 2 * kk, 1u);
              commit(smem_u32(&a_free[as]));  // the A slot is free once these MMAs have completed
            }
            a_ready = __all_sync(0xffffffffu, peek_a);
            acc_ready = __all_sync(0xffffffffu, peek_acc);
            as = as_next;
            a_phase = ph_next;
          }
          if (ok && elect_one()) {
            commit(smem_u32(&acc_full[ab]));
            if (through) commit(smem_u32(&w_free[slot]));
          }
          __syncwarp();
          // an odd number of slabs swaps the warps' slabs from pass to pass: the other one's weights
          // have to be there as well before this warp's next pass
          if (check_w && (nk & 1))
            for (int kt = first ^ 1; kt < nk; kt += 2)
              ok = ok && wait_warp(smem_u32(&w_full[slot * MAX_NK + kt]), (w_phase >> slot) & 1u, abort_flag);
          par ^= nk & 1;
          if (!ok) break;
          check &= ~(1u << slot);
          if (through) held &= ~(1u << slot);
          ab = ab_next;
          acc_phase = acc_next;
        }
      }
      if (elect_one()) {
        commit(smem_u32(drain));  // every MMA completes before tensor memory is freed
        drain_bar(smem_u32(drain), 0);
      }
      __syncwarp();
    }
  } else if (warp < EPI_WARP0) {
    // ------------------------------------------------------------------ splitters
    const int mine = (warp - SPLIT_WARP0) >> 2;  // this group's slabs: g = mine mod 2
    const int r = (warp & 3) * 32 + lane;        // row of the slab, lane of tensor memory
    // stage and lap of the ring, and slot of the A ring, of this group's next slab (every second
    // one); `left` slabs of the current item remain, counted from the group's next one
    int s = mine, left = -mine;
    uint32_t lap = 0, as = (uint32_t)mine, as_lap = 0;
    bool ok = true, full_ready = false, slot_ready = false;
    for (int q = 0; ok; ++q) {
      const int it = item_warp(q);
      if (it < 0) break;
      left += passes_of(work_item(a, it)) * nk;
      for (; left > 0; left -= 2) {
        if (!full_ready) ok = wait_warp(smem_u32(&full[s]), lap & 1u, abort_flag);
        if (!ok) break;
        const uint8_t* slab = ring + s * C::TILE_A;
        const uint32_t ta = tmem + ((uint32_t)((warp & 3) * 32) << 16) + as * (uint32_t)C::A_STAGE;
        uint32_t x[32];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(&x[4 * c]) = *reinterpret_cast<const uint4*>(slab + chunk_at<float>(r, c));
        // the slab is in registers once these loads are done: then its stage may be refilled. The
        // arrival alone does not hold the copy that refills it behind loads still on their way (the
        // last 16 bytes of some rows came from the next slab, in one product of 10^5).
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&empty[s]));
        // (the first lap's wait is for the phase before the first and succeeds at once)
        if (!slot_ready) ok = wait_warp(smem_u32(&a_free[as]), (as_lap & 1u) ^ 1u, abort_flag);
        if (!ok) break;
        int s_next = s + 2;
        uint32_t lap_next = lap;
        if (s_next >= S) {
          s_next -= S;
          ++lap_next;
        }
        uint32_t as_next = as + 2, as_lap_next = as_lap;
        if (as_next >= (uint32_t)C::A_RING) {
          as_next -= (uint32_t)C::A_RING;
          ++as_lap_next;
        }
        const bool peek_full = peek_parity(smem_u32(&full[s_next]), lap_next & 1u);
        const bool peek_slot = peek_parity(smem_u32(&a_free[as_next]), (as_lap_next & 1u) ^ 1u);
        asm volatile("tcgen05.fence::after_thread_sync;");
        store_parts(ta, x);  // three operations an element: issue slots are short here
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&a_full[as]));
        full_ready = __all_sync(0xffffffffu, peek_full);
        slot_ready = __all_sync(0xffffffffu, peek_slot);
        s = s_next;
        lap = lap_next;
        as = as_next;
        as_lap = as_lap_next;
      }
    }
  } else {
    FC_SETMAXNREG_INC(120);
    // ------------------------------------------------------------------ epilogue
    // one warp per lane quarter and 32 columns; a thread holds its row's 32 columns
    const int quarter = warp & 3, half = (warp - EPI_WARP0) >> 2;
    uint8_t* boxes = epi + (warp - EPI_WARP0) * C::BUFS * EPI_BUF;
    uint64_t* landed = aux + (warp - EPI_WARP0) * C::BUFS;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(A_COLS + half * 32);
    const float sa = MODE == DX ? 0.f : __ldg(a.scales + a.ranks + 1);
    const int col = ct * BN + half * 32;
    const bool live = col < a.N;  // the warp has columns to write
    uint32_t ab = 0, acc_phase = 0;  // the accumulator in turn
    uint32_t par = 0;                // parity of the pass's first slab
    bool ok = true;
    auto wait_acc = [&]() {
      const bool done = wait_warp(smem_u32(&acc_full[ab]), acc_phase, abort_flag);
      asm volatile("tcgen05.fence::after_thread_sync;");
      return done;
    };
    auto free_acc = [&]() {
      asm volatile("tcgen05.fence::before_thread_sync;");
      __syncwarp();
      if (lane == 0) arrive(smem_u32(&acc_empty[ab]));
      par ^= (uint32_t)nk & 1u;
      if (++ab == NACC) {
        ab = 0;
        acc_phase ^= 1u;
      }
    };
    // columns c0 .. c0+15 of the row: both halves of the accumulator (a single slab fills the
    // half of its parity)
    auto load16 = [&](int c0, float* f) {
      const uint32_t t = lane_base + ab * (uint32_t)ACC_W + (uint32_t)c0;
      if (nk > 1) tmem_ld_sum<16>(t, t + BN, f);
      else tmem_ld<16>(t + par * BN, f);
    };
    // this warp's 32 x 32 box from staging to memory
    auto send = [&](const CUtensorMap* map, uint8_t* buf, int row, int z) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (elect_one()) {
        tma_store_3d(map, smem_u32(buf), col, row, z);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
      __syncwarp();
    };
    // earlier stores have read their boxes (the elected lane is the same every time)
    auto boxes_free = [&]() {
      if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
    };
    // PRE: the box in turn is free (the boxes send by turns, so at most the other one's store is
    // still reading)
    auto box_free = [&]() {
      if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      __syncwarp();
    };
    uint32_t box = 0, box_phase = 0;  // PRE: the box in turn; bit b: parity of landed[b]'s next completion
    for (int q = 0; ok; ++q) {
      const int it = item_warp(q);
      if (it < 0) break;
      const WorkItem w = work_item(a, it);
      const int row0 = w.tile * BM + quarter * 32;
      if constexpr (MODE == DX) {
        float acc[32];
        const bool sums = w.k0 == 0;
        const int passes = passes_of(w);
        for (int p = 0; p < passes; ++p) {
          if (!(ok = wait_acc())) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float f[16];
            load16(h * 16, f);
#pragma unroll
            for (int c = 0; c < 16; ++c) acc[h * 16 + c] = (sums && p > 0) ? acc[h * 16 + c] + f[c] : f[c];
          }
          free_acc();
          if (live && (!sums || p + 1 == passes)) {
            boxes_free();
            put_row<T>(boxes, lane, acc);
            send(&mp.o, boxes, row0, sums ? 0 : w.k0 + p);
          }
        }
      } else {
        // ask for component m's box of g
        int asked = 0, got = 0;
        auto ask = [&](int m, uint32_t b) {
          asked = m + 1;
          if (elect_one()) {
            const uint32_t fb = smem_u32(&landed[b]);
            arrive_tx(fb, 32 * 32 * sizeof(T));
            tma_load_3d(smem_u32(boxes + b * EPI_BUF), &mp.g, col, row0, w.k0 + m, fb);
          }
          __syncwarp();
        };
        if (MODE == PRE && live) {
          box_free();
          ask(0, box);
        }
        float z[32];  // pre-activations of this thread's row
        ok = wait_acc();
#pragma unroll
        for (int h = 0; h < 2; ++h) load16(h * 16, z + h * 16);
        free_acc();
        if (a.bias && live) {
          const T* b = (const T*)a.bias + (int64_t)w.l * a.N;
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (col + c < a.N) z[c] += Io<T>::get(b[col + c]);
        }
        if constexpr (MODE == FWD) {
#pragma unroll
          for (int c = 0; c < 32; ++c) z[c] = sa * fast_act(a.act, z[c]);
          for (int m = 0; m < w.nm && ok; ++m) {
            if (!(ok = wait_acc())) break;
            float f[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) load16(h * 16, f + h * 16);
            free_acc();
            if (live) {
#pragma unroll
              for (int c = 0; c < 32; ++c) f[c] *= z[c];
              boxes_free();
              put_row<T>(boxes, lane, f);
              send(&mp.o, boxes, row0, w.k0 + m);
            }
          }
        } else {
          // the gates stay here, their slopes wait in tensor memory until the rank is done
          const uint32_t z_at = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(C::Z_COL + half * 32);
          {
            float slope[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float sg = fast_sigmoid(z[c]), q = 1.f - sg;
              slope[c] = sa * (a.act == FC_GATE_SIGMOID ? sg * q : sg * fmaf(z[c], q, 1.f));
              z[c] = sa * (a.act == FC_GATE_SIGMOID ? sg : z[c] * sg);
            }
            tmem_st32(z_at, reinterpret_cast<const uint32_t*>(slope));
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          }
          float sum[32];  // over m of g v
#pragma unroll
          for (int c = 0; c < 32; ++c) sum[c] = 0.f;
          for (int m = 0; m < w.nm && ok; ++m) {
            if (!wait_acc()) ok = false;
            if (got < asked) {
              ++got;
              const uint32_t par = (box_phase >> box) & 1u;
              box_phase ^= 1u << box;
              if (!wait_warp(smem_u32(&landed[box]), par, abort_flag)) {
                drain_bar(smem_u32(&landed[box]), par);  // the copy may still land: let it
                __syncwarp();
                ok = false;
              }
              uint8_t* buf = boxes + box * EPI_BUF;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float v[16];
                load16(h * 16, v);
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4) {
                  float4* at = reinterpret_cast<float4*>(buf + chunk_at<float>(lane, h * 4 + c4));
                  const float4 t = *at;
                  const float gv[4] = {t.x, t.y, t.z, t.w};
                  float o[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int c = h * 16 + c4 * 4 + e;
                    sum[c] += gv[e] * v[c4 * 4 + e];
                    o[e] = gv[e] * z[c];
                  }
                  *at = make_float4(o[0], o[1], o[2], o[3]);
                }
              }
              if (m + 1 < w.nm && ok) {
                boxes_free();  // the other box: its store is a component old
                ask(m + 1, box ^ 1u);
              }
              send(&mp.o, buf, row0, w.k0 + m);
              box ^= 1u;
            }
            free_acc();
          }
          if (got < asked) {  // gave up: the box asked for may still land
            drain_bar(smem_u32(&landed[box]), (box_phase >> box) & 1u);
            __syncwarp();
          }
          if (ok && live) {
            box_free();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float zz[16];
              tmem_ld<16>(z_at + h * 16, zz);
#pragma unroll
              for (int c = 0; c < 16; ++c) sum[h * 16 + c] *= zz[c];
            }
            put_row<float>(boxes + box * EPI_BUF, lane, sum);
            send(&mp.o2, boxes + box * EPI_BUF, row0, w.l);
            box ^= 1u;
          }
        }
      }
    }
    if (elect_one()) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) fc_flag(a.status, FC_DEV_TIMEOUT);
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ---------------------------------------------------------------------------- operand layouts

constexpr int MAX_LISTS = 160;  // work lists of a launch: one per 64 output channels

// Scaled weights as tf32 hi | lo parts: matrix q (values 0 .. ranks-1, then gates) at q, its
// low part 2 ranks matrices behind; (out, k) rows of kp elements, zero behind K. fwd: out =
// hidden, k = input channel; dx: the transpose. Also zeroes the work lists' counters.
struct PrepArgs {
  GatedArgs g;
  float* fwd;      // or null
  float* dx;       // or null
  bf16_t* direct;  // or null: in place of fwd, the weights as they are, in rows padded with zeros
  bf16_t* direct_dx;
  int* counters;
};

template <typename T>
__global__ void __launch_bounds__(256) prep_kernel(const PrepArgs p) {
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < 2 * MAX_LISTS; i += 256) p.counters[i] = 0;
  const int ranks = p.g.L + 1, q = blockIdx.y, l = q < ranks ? q : q - ranks, C = p.g.C, H = p.g.H;
  const T* w = q < ranks ? (const T*)p.g.wv[l] : (const T*)p.g.wg + (int64_t)l * H * C;
  const float sc = ((const float*)p.g.scales)[q < ranks ? l : ranks];
  const int pad_f = p.direct ? 7 : 3, pad_d = p.direct_dx ? 7 : 3;
  const int cp = (C + pad_f) & ~pad_f, hp = (H + pad_d) & ~pad_d;
  const int64_t nf = p.direct || p.fwd ? (int64_t)H * cp : 0, nd = p.direct_dx || p.dx ? (int64_t)C * hp : 0;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < nf + nd; i += (int64_t)gridDim.x * 256) {
    const bool f = i < nf;
    const int64_t e = f ? i : i - nf, size = f ? nf : nd;
    const int kp = f ? cp : hp, r = (int)(e / kp), k = (int)(e - (int64_t)r * kp);
    if (bf16_t* plain = f ? p.direct : p.direct_dx) {
      plain[q * size + e] = Io<bf16_t>::put(
          k >= (f ? C : H) ? 0.f : (float)Io<T>::get(f ? w[(int64_t)r * C + k] : w[(int64_t)k * C + r]));
      continue;
    }
    float x = 0.f;
    if (k < (f ? C : H)) x = sc * Io<T>::get(f ? w[(int64_t)r * C + k] : w[(int64_t)k * C + r]);
    const float hi = round_tf32(x);
    float* out = f ? p.fwd : p.dx;
    out[q * size + e] = hi;
    out[(q + 2 * ranks) * size + e] = round_tf32(x - hi);
  }
}

// rows of `width` elements between row lengths (tensors whose rows TMA cannot address)
template <typename T>
__global__ void __launch_bounds__(256) repitch_kernel(const T* __restrict__ src, int64_t src_ld, T* __restrict__ dst,
                                                      int64_t dst_ld, int width, int64_t rows) {
  const int64_t total = rows * width;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = total < ((int64_t)1 << 32) ? (int64_t)((uint32_t)i / (uint32_t)width) : i / width;
    const int64_t c = i - r * width;
    dst[r * dst_ld + c] = src[r * src_ld + c];
  }
}

// ---------------------------------------------------------------------------- host

static EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

template <typename E>
bool encode_rows(CUtensorMap* map, const void* base, int64_t channels, int64_t rows, int64_t comps, int64_t ld,
                        int box_c, int box_r) {
  const cuuint64_t dims[3] = {(cuuint64_t)channels, (cuuint64_t)rows, (cuuint64_t)comps};
  const cuuint64_t strides[2] = {(cuuint64_t)(comps * ld) * sizeof(E), (cuuint64_t)ld * sizeof(E)};
  const cuuint32_t box[3] = {(cuuint32_t)box_c, (cuuint32_t)box_r, 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return encode_fn()(map, sizeof(E) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     const_cast<void*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     box_c * sizeof(E) == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                     : box_c * sizeof(E) == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                               : CU_TENSOR_MAP_SWIZZLE_NONE,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template bool encode_rows<float>(CUtensorMap*, const void*, int64_t, int64_t, int64_t, int64_t, int, int);
template bool encode_rows<bf16_t>(CUtensorMap*, const void*, int64_t, int64_t, int64_t, int64_t, int, int);

// (k, output channel, matrix) map of weights in 128-byte boxes.
template <typename E>
static bool encode_weights(CUtensorMap* map, const E* base, int kp, int out, int mats, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)kp, (cuuint64_t)out, (cuuint64_t)mats};
  const cuuint64_t strides[2] = {(cuuint64_t)kp * sizeof(E), (cuuint64_t)kp * out * sizeof(E)};
  const cuuint32_t box[3] = {128 / sizeof(E), (cuuint32_t)box_rows, 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return encode_fn()(map, sizeof(E) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     const_cast<E*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return sms[dev];
}

template <int MODE, typename T>
static int run_resident(const Maps& mp, Args a, int sms, cudaStream_t s) {
  using C = Cfg<MODE, T>;
  a.stages = C::stages(a.nk);
  static Ready state;
  if (int rc = ready(gated_tc_kernel<MODE, T>, SMEM_MAX, state, TC_REGS)) return rc;
  const int lists = (int)std::min<int64_t>(a.items, sms / a.n_ct);
  gated_tc_kernel<MODE, T><<<lists * a.n_ct, TC_THREADS, C::smem(a.nk, a.stages), s>>>(mp, a);
  return fc_launched(1);
}

// A column tile has its work list, and every list some CTAs.
static bool one_list_each(int N, int sms) { return (N + BN - 1) / BN <= std::min(sms, MAX_LISTS); }

// Whether the products of a reduction over K into N columns keep their weights in shared memory.
static bool resident(int K, int N, int sms) { return K <= MAX_NK * BK && one_list_each(N, sms); }

// Whether the products of a reduction over K into N columns multiply bfloat16 as it is.
template <typename T>
static bool direct(int K, int N, int sms) {
  return sizeof(T) == 2 && K <= DIRECT_K && one_list_each(N, sms);
}
// The backward does in all its products, or in none: its halves hand each other dv and dz.
template <typename T>
static bool direct_backward(int C, int H, int sms) {
  return direct<T>(C, H, sms) && direct<T>(H, C, sms);
}

template <int MODE, typename T>
static int run_products(const Maps& mp, const Args& a, int K, bool dir, int sms, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (dir) {
      if constexpr (MODE == DX) return run_direct_dx(mp, a, sms, s);
      else return run_direct<MODE>(mp, a, sms, s);
    }
  }
  if constexpr (sizeof(T) == 4 || MODE == DX)
    if (resident(K, a.N, sms)) return run_resident<MODE, T>(mp, a, sms, s);
  return run_stream<MODE, T>(mp, a, sms, s);
}

// Rows of dv and dz parts are whole 128-byte lines: with 200 channels in rows of 200 (208, 256) the
// backward's first half took 78 (72, 67) us for 100,003 rows.
constexpr int PARTS_PAD = 64;

// Layout of the workspace (bytes), the same for the size query and the call.
struct Ws {
  int64_t counters, fwd, dx, dv, dz, part, bias, x, y, gx, bytes;
};

static Ws layout(int L, int C, int H, int64_t n, int esize, bool backward, int sms) {
  const int64_t ranks = L + 1, comps = ranks * ranks, per = 16 / esize;
  const int64_t pad = esize == 2 ? PARTS_PAD : 4;  // (float rows have no parts)
  const int64_t cp = (C + 3) / 4 * 4, hp = (H + pad - 1) / pad * pad;
  const int64_t ce = (C + per - 1) / per * per, he = (H + per - 1) / per * per;
  Ws w{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += (bytes + 127) / 128 * 128;
    return p;
  };
  w.counters = take(2 * MAX_LISTS * 4);
  w.fwd = take(4 * ranks * H * cp * 4);
  if (backward) {
    const int64_t parts = wgrad_part_count((int)ranks, C, H, sms);
    w.dx = take(4 * ranks * C * hp * 4);
    w.dv = take(n * comps * hp * 4);
    w.dz = take(n * ranks * hp * 4);
    w.part = take(parts * BM * BM * 4);
    w.bias = take(parts * 2 * BM * 4);
  }
  // copies in rows of whole 16 bytes, where the caller's are not
  const bool copy_c = ce != C, copy_h = he != H;
  if (copy_c) w.x = take(n * comps * ce * esize);
  if (copy_h) w.y = take(n * comps * he * esize);  // y, or the output gradient
  if (copy_c && backward) w.gx = take(n * comps * ce * esize);
  w.bytes = at;
  return w;
}

// A tensor as TMA can address it: itself (16-byte aligned, the caller's check), or a copy with
// padded rows.
template <typename T>
struct Rows {
  const T* p;
  int64_t ld;
  bool copied;
};

template <typename T>
static Rows<T> rows_of(const void* p, int width, void* room) {
  constexpr int per = 16 / sizeof(T);
  if (width % per == 0) return {(const T*)p, width, false};
  return {(const T*)room, (width + per - 1) / per * per, true};
}

template <typename T>
static int repitch(const T* src, int64_t src_ld, T* dst, int64_t dst_ld, int width, int64_t rows, cudaStream_t s) {
  const int64_t b = (rows * width + 255) / 256;
  repitch_kernel<T><<<(unsigned)std::min<int64_t>(b, 148 * 32), 256, 0, s>>>(src, src_ld, dst, dst_ld, width, rows);
  return fc_launched(1);
}

template <typename T>
static Args product_args(const GatedArgs& g, int N, int K, int mode, bool dir, int sms) {
  Args a{};
  a.L = g.L;
  a.ranks = g.L + 1;
  a.comps = a.ranks * a.ranks;
  a.N = N;
  a.nk = dir ? (K + DIRECT_BK - 1) / DIRECT_BK : (K + BK - 1) / BK;
  a.tiles = (int)((g.n + BM - 1) / BM);
  const bool res = dir || (resident(K, N, sms) && (sizeof(T) == 4 || mode == DX));
  const int width = !res ? STREAM_BN : dir && mode == DX ? DIRECT_DX_BN : BN;
  a.n_ct = (N + width - 1) / width;
  // with fewer (tile, rank) groups than SMs the components are items of their own (the gate is
  // computed again for each); PRE needs a rank's components together
  a.per_comp = (mode == DX && !res) || (mode != PRE && (int64_t)a.tiles * a.ranks * a.n_ct < sms);
  a.items = (int64_t)a.tiles * (a.per_comp ? a.comps : a.ranks);
  if (!res) {
    a.items *= a.n_ct;
    // units of 64 products, added in registers. PRE's epilogue is the longer the more units there
    // are: above 192 channels they have 96 products (100,003 rows of 200 -> 200 channels, both kernels
    // of the input gradient: 353 us, with 64 products 381; its error 6.6e-7, with 64 4.5e-7)
    a.kg = mode == PRE && a.nk > STREAM_KG * STREAM_NACC ? STREAM_KG + 1 : STREAM_KG;
    a.nu = (a.nk + a.kg - 1) / a.kg;
    const int tail = (2 * sms + a.ranks * a.n_ct - 1) / (a.ranks * a.n_ct);
    a.main_tiles = std::max(0, a.tiles - tail);
  }
  a.act = g.act;
  a.bias = g.bias;
  a.scales = (const float*)g.scales;
  a.status = g.status;
  return a;
}

template <typename T>
static int run_prep(const GatedArgs& g, void* fwd, void* dx, bool dir, int* counters, cudaStream_t s) {
  const int64_t each = (int64_t)g.H * (g.C + 7) + (dx ? (int64_t)g.C * (g.H + 7) : 0);
  const PrepArgs p{g, dir ? nullptr : (float*)fwd, dir ? nullptr : (float*)dx, dir ? (bf16_t*)fwd : nullptr,
                   dir ? (bf16_t*)dx : nullptr, counters};
  prep_kernel<T><<<dim3((unsigned)std::min<int64_t>((each + 255) / 256, 256), 2 * (g.L + 1)), 256, 0, s>>>(p);
  return fc_launched(1);
}

// The maps of x and of the weights that the forward products read.
template <typename T>
static bool encode_forward(Maps& mp, const GatedArgs& g, const Rows<T>& x, const void* weights, bool dir, int sms) {
  const int ranks = g.L + 1, comps = ranks * ranks;
  if (dir)
    return encode_rows<T>(&mp.a, x.p, g.C, g.n, comps, x.ld, DIRECT_BK, BM) &&
           encode_rows<T>(&mp.ap, x.p, g.C, g.n, comps, x.ld, DIRECT_K, BM) &&
           encode_weights<bf16_t>(&mp.b, (const bf16_t*)weights, (g.C + 7) & ~7, g.H, 2 * ranks, BN);
  return encode_rows<T>(&mp.a, x.p, g.C, g.n, comps, x.ld, BK, BM) &&
         encode_rows<T>(&mp.ap, x.p, g.C, g.n, comps, x.ld, MAX_NK * BK, BM) &&
         encode_weights<float>(&mp.b, (const float*)weights, (g.C + 3) & ~3, g.H, 4 * ranks,
                               sizeof(T) == 4 && resident(g.C, g.H, sms) ? BN : STREAM_BN);
}

}  // namespace gtc

int64_t gated_tc_ws(int L, int C, int H, int64_t n, int dtype, int backward) {
  return gtc::layout(L, C, H, n, dtype == FC_BF16 ? 2 : 4, backward != 0, 148 * 2).bytes;
}

template <typename T>
int gated_tc_fwd(const GatedArgs& a, cudaStream_t s) {
  using namespace gtc;
  const int sms = sm_count();
  if (!sms || !encode_fn()) return FC_ERR_LAUNCH;
  const int ranks = a.L + 1, comps = ranks * ranks;
  const Ws w = layout(a.L, a.C, a.H, a.n, sizeof(T), false, sms);
  uint8_t* ws = (uint8_t*)a.ws;
  const Rows<T> x = rows_of<T>(a.x, a.C, ws + w.x), y = rows_of<T>(a.y, a.H, ws + w.y);
  if (x.copied)
    if (int rc = repitch<T>((const T*)a.x, a.C, const_cast<T*>(x.p), x.ld, a.C, a.n * comps, s)) return rc;
  int* counters = (int*)(ws + w.counters);
  const bool dir = direct<T>(a.C, a.H, sms);
  if (int rc = run_prep<T>(a, ws + w.fwd, nullptr, dir, counters, s)) return rc;
  Args args = product_args<T>(a, a.H, a.C, FWD, dir, sms);
  args.counter = counters;
  Maps mp;
  if (!encode_forward<T>(mp, a, x, ws + w.fwd, dir, sms) || !encode_rows<T>(&mp.o, y.p, a.H, a.n, comps, y.ld, 32, 32))
    return FC_ERR_UNSUPPORTED;
  mp.a2 = mp.g = mp.gp = mp.o2 = mp.o;  // not used
  if (int rc = run_products<FWD, T>(mp, args, a.C, dir, sms, s)) return rc;
  if (y.copied) return repitch<T>(y.p, y.ld, (T*)a.y, a.H, a.H, a.n * comps, s);
  return 0;
}

template <typename T>
int gated_tc_bwd(const GatedArgs& a, cudaStream_t s) {
  using namespace gtc;
  const int sms = sm_count();
  if (!sms || !encode_fn()) return FC_ERR_LAUNCH;
  const int ranks = a.L + 1, comps = ranks * ranks;
  const bool dir = direct_backward<T>(a.C, a.H, sms);
  const int64_t hp = dir ? (a.H + PARTS_PAD - 1) / PARTS_PAD * PARTS_PAD : (a.H + 3) / 4 * 4;  // row length of dv and dz
  const Ws w = layout(a.L, a.C, a.H, a.n, sizeof(T), true, sms);
  uint8_t* ws = (uint8_t*)a.ws;
  const Rows<T> x = rows_of<T>(a.x, a.C, ws + w.x), gy = rows_of<T>(a.gy, a.H, ws + w.y);
  int* counters = (int*)(ws + w.counters);
  void *dx = ws + w.dx, *dv = ws + w.dv, *dz = ws + w.dz;
  // dv and dz in boxes: floats, or two bfloat16 parts a component
  auto encode_between = [&](CUtensorMap* map, const void* p, int64_t planes, int box_c, int box_r) {
    return dir ? encode_rows<bf16_t>(map, p, a.H, a.n, 2 * planes, hp, box_c, box_r)
               : encode_rows<float>(map, p, a.H, a.n, planes, hp, box_c, box_r);
  };
  bool any = a.gwg || a.gbias;
  for (int l = 0; l < ranks; ++l) any = any || a.gwv[l];
  if (a.n > 0) {
    if (x.copied)
      if (int rc = repitch<T>((const T*)a.x, a.C, const_cast<T*>(x.p), x.ld, a.C, a.n * comps, s)) return rc;
    if (gy.copied)
      if (int rc = repitch<T>((const T*)a.gy, a.H, const_cast<T*>(gy.p), gy.ld, a.H, a.n * comps, s)) return rc;
    if (int rc = run_prep<T>(a, ws + w.fwd, a.gx ? dx : nullptr, dir, counters, s)) return rc;
    Maps mp;
    if (!encode_forward<T>(mp, a, x, ws + w.fwd, dir, sms) || !encode_between(&mp.o, dv, comps, 32, 32) ||
        !encode_rows<T>(&mp.g, gy.p, a.H, a.n, comps, gy.ld, 32, 32) ||
        !encode_rows<T>(&mp.gp, gy.p, a.H, a.n, comps, gy.ld, BN, BM) ||
        !encode_between(&mp.o2, dz, ranks, 32, 32))
      return FC_ERR_UNSUPPORTED;
    mp.a2 = mp.o2;  // not used
    Args args = product_args<T>(a, a.H, a.C, PRE, dir, sms);
    args.counter = counters;
    if (int rc = run_products<PRE, T>(mp, args, a.C, dir, sms, s)) return rc;
    if (a.gx) {
      const Rows<T> gx = rows_of<T>(a.gx, a.C, ws + w.gx);
      Maps md;
      const int box = dir ? DIRECT_BK : BK;
      if (!encode_between(&md.a, dv, comps, box, BM) || !encode_between(&md.a2, dz, ranks, box, BM) ||
          !(dir ? encode_weights<bf16_t>(&md.b, (const bf16_t*)dx, (a.H + 7) & ~7, a.C, 2 * ranks, DIRECT_DX_BN)
                : encode_weights<float>(&md.b, (const float*)dx, (int)hp, a.C, 4 * ranks,
                                        resident(a.H, a.C, sms) ? BN : STREAM_BN)) ||
          !encode_between(&md.ap, dv, comps, MAX_NK * BK, BM) ||
          !encode_rows<T>(&md.o, gx.p, a.C, a.n, comps, gx.ld, 32, 32))
        return FC_ERR_UNSUPPORTED;
      md.g = md.gp = md.o2 = md.o;  // not used
      Args dargs = product_args<T>(a, a.C, a.H, DX, dir, sms);
      dargs.counter = counters + MAX_LISTS;
      if (int rc = run_products<DX, T>(md, dargs, a.H, dir, sms, s)) return rc;
      if (gx.copied)
        if (int rc = repitch<T>(gx.p, gx.ld, (T*)a.gx, a.C, a.C, a.n * comps, s)) return rc;
    }
  }
  if (!any) return 0;
  WOut o{};
  for (int l = 0; l < ranks; ++l) {
    o.w[l] = a.gwv[l];
    o.w[ranks + l] = a.gwg;
  }
  o.bias = a.gbias;
  o.scales = (const float*)a.scales;
  return run_wgrad<T>(ranks, a.C, a.H, a.n, dv, dz, hp, dir, x.p, x.ld, (float*)(ws + w.part), (float*)(ws + w.bias), o,
                      a.status, sms, s);
}

template int gated_tc_fwd<float>(const GatedArgs&, cudaStream_t);
template int gated_tc_fwd<bf16_t>(const GatedArgs&, cudaStream_t);
template int gated_tc_bwd<float>(const GatedArgs&, cudaStream_t);
template int gated_tc_bwd<bf16_t>(const GatedArgs&, cudaStream_t);

}  // namespace fc

#endif  // FC_HOST_EMU
