// Gated feed-forward products with more than 128 channels to reduce over (bfloat16 rows: 256):
// weights streamed (gated_ff_tc.cu keeps them in shared memory below that; measured on 27,648 x 16
// rows of 128 channels: this kernel 149 us forward and 143 us for the input gradient, that one 110
// and 114).
//
// What bounds it: the tensor cores (three products: 58 us for 100,003 rows of 200 -> 200 channels);
// measured there 135 us forward, 217 us first half of the backward, 123 us input gradient. A stage
// carries 32 KB of weights beside 16 KB of rows, so copies, splitters and MMAs together keep shared
// memory busy for 900 cycles a slab where the MMAs alone take 770, and four splitter warps do not
// hide behind them. PRE computes a gate again for each of its rank's components: 64 gates beside 64
// sums are what its registers hold.
//
// A tensor-core accumulation truncates, so no accumulator runs over more than 64 products (96: PRE
// above 192 channels): the error does not grow with the channels (float32 gradients of 320 to 16,384
// channels: 7e-7 to 1e-6; 4e-5 at 16,384 when PRE's three accumulators shared all of them).
//
// One persistent CTA per SM, 16 warps:
//   warp 0       TMA producer, and the CTA's draw from the work list (an atomic counter)
//   warp 1       MMA issue
//   warps 4-7    splitters: the A slab (128 rows x 32 channels) to tf32 parts in tensor memory
//   warps 8-15   epilogue: two warps per lane quarter, 64 columns each
// Every stage of the operand ring holds an A slab and the matching slab of the weights' two
// parts. See gated_ff_tc.cu for the modes and the order of the products.
#include "gated_ff_tc.cuh"

#ifndef FC_HOST_EMU

#include <algorithm>

namespace fc {
namespace gtc {

constexpr int BN = STREAM_BN, NACC = STREAM_NACC;
constexpr int TILE_B = BN * BK * 4;
constexpr int EPI_WARPS = 8;
constexpr int A_COLS = 128;  // tensor-memory columns of the A parts' ring; the accumulators behind them

template <int MODE, typename T>
struct Cfg {
  static constexpr bool A32 = MODE == DX || sizeof(T) == 4;  // A in float32: hi and lo parts
  static constexpr int TILE_A = BM * BK * (A32 ? 4 : 2);
  static constexpr int STAGE = TILE_A + 2 * TILE_B;
  static constexpr int A_STAGE = A32 ? 2 * BK : BK;  // tensor-memory columns
  // staging boxes per epilogue warp: PRE holds g's two; the others do with one for a fourth stage
  static constexpr int BUFS = MODE == PRE ? 2 : 1, EPI_BYTES = EPI_WARPS * BUFS * EPI_BUF;
  static constexpr int STAGES = A32 && MODE == PRE ? 3 : 4;
  static constexpr int A_RING = A_COLS / A_STAGE;
  static constexpr int SMEM = STAGES * STAGE + EPI_BYTES + BAR_BYTES + 1024;
  static_assert(A_COLS + NACC * BN <= 512, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory per CTA");
};

// A work item: rows 128 tile.., columns 128 ct.., and rank l's components m0 .. m0+nm-1 (FWD,
// PRE) or component k (DX).
struct Item {
  int tile, ct, l, k0, nm;
};

template <int MODE>
__device__ __forceinline__ Item item_of(const Args& a, int it) {
  Item w;
  if (MODE == DX || a.per_comp) {
    const int per_tile = a.comps * a.n_ct;
    w.tile = it / per_tile;
    const int r = it - w.tile * per_tile;
    w.k0 = r / a.n_ct;
    w.ct = r - w.k0 * a.n_ct;
    w.l = gated_rank_of(w.k0);
    w.nm = 1;
    return w;
  }
  // ranks of a tile one after the other, high ranks (most work) first; the last tiles rank by
  // rank, so that the work list ends with its smallest items
  const int group = a.ranks * a.n_ct, split = a.main_tiles * group;
  if (it < split) {
    w.tile = it / group;
    const int r = it - w.tile * group;
    w.l = a.L - r / a.n_ct;
    w.ct = r % a.n_ct;
  } else {
    const int tail = (a.tiles - a.main_tiles) * a.n_ct, r0 = it - split, r = r0 % tail;
    w.l = a.L - r0 / tail;
    w.tile = a.main_tiles + r / a.n_ct;
    w.ct = r % a.n_ct;
  }
  w.k0 = w.l * w.l;
  w.nm = 2 * w.l + 1;
  return w;
}

// LONG (PRE): a component has more units than there are accumulators. A kernel of its own: that loop's
// registers cost the short reductions 3%.
template <int MODE, typename T, bool LONG>
__global__ void __launch_bounds__(THREADS, 1) gated_stream_kernel(const __grid_constant__ Maps mp, const Args a) {
  using C = Cfg<MODE, T>;
  constexpr int S = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + S * C::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + C::EPI_BYTES);
  uint64_t* split = full + S;
  uint64_t* empty = split + S;
  uint64_t* a_free = empty + S;  // the MMAs have read a slot of the A ring
  uint64_t* acc_full = a_free + C::A_RING;
  uint64_t* acc_empty = acc_full + NACC;
  uint64_t* sched_full = acc_empty + NACC;
  uint64_t* sched_empty = sched_full + SCHED;
  uint64_t* drain = sched_empty + SCHED;
  uint64_t* aux = drain + 1;  // per epilogue warp and buffer: the box of g has landed
  int* sched = reinterpret_cast<int*>(aux + 2 * EPI_WARPS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sched + SCHED);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((3 * S + C::A_RING + 2 * NACC + 2 * SCHED + 1 + 2 * EPI_WARPS) * 8 + SCHED * 4 + 8 <= BAR_BYTES, "barriers");

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
    for (int s = 0; s < S; ++s) {
      init(&full[s], 1);
      init(&split[s], 4);
      init(&empty[s], 1);
    }
    for (int b = 0; b < C::A_RING; ++b) init(&a_free[b], 1);
    for (int b = 0; b < NACC; ++b) {
      init(&acc_full[b], 1);
      init(&acc_empty[b], EPI_WARPS);
    }
    for (int b = 0; b < SCHED; ++b) {
      init(&sched_full[b], 1);
      init(&sched_empty[b], 1 + 4 + EPI_WARPS);
    }
    init(drain, 1);
    for (int b = 0; b < 2 * EPI_WARPS; ++b) init(&aux[b], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;

  // the q-th item of this CTA for a warp (-1: no more, or a wait gave up)
  auto next_item = [&](int q) -> int {
    const int s = q % SCHED;
    if (!wait_warp(smem_u32(&sched_full[s]), (uint32_t)((q / SCHED) & 1), abort_flag)) return -1;
    const int it = *reinterpret_cast<volatile int*>(&sched[s]);
    __syncwarp();
    if (lane == 0) arrive(smem_u32(&sched_empty[s]));
    return it;
  };
  auto segments = [&](const Item& w) { return MODE == DX && w.k0 == 0 ? a.ranks + 1 : 1; };
  auto substeps = [&](const Item& w) { return MODE == DX ? 1 : 1 + w.nm; };

  if (warp < 4) {
    FC_SETMAXNREG_DEC(48);
    if (warp == 0 && elect_one()) {
      // ---------------------------------------------------------------- TMA producer
      constexpr uint32_t bytes = C::TILE_A + 2 * TILE_B;
      int next = (int)blockIdx.x;
      int64_t g = 0;
      uint32_t s = 0, lap = 0;
      bool ok = true, free = true;  // (peeked: the next stage is free)
      for (int q = 0; ok; ++q) {
        const int s4 = q % SCHED;
        if (q >= SCHED &&
            !wait_phase(smem_u32(&sched_empty[s4]), (uint32_t)((q / SCHED - 1) & 1), abort_flag))
          break;
        const int it = next < a.items ? next : -1;
        *reinterpret_cast<volatile int*>(&sched[s4]) = it;
        arrive(smem_u32(&sched_full[s4]));
        if (it < 0) break;
        next = (int)gridDim.x + atomicAdd(a.counter, 1);
        const Item w = item_of<MODE>(a, it);
        const int subs = substeps(w), segs = segments(w);
        for (int sub = 0; sub < subs && ok; ++sub)
          for (int seg = 0; seg < segs && ok; ++seg) {
            const CUtensorMap* ma = &mp.a;
            int z = MODE == DX ? w.k0 : (sub == 0 ? 0 : w.k0 + sub - 1);
            int mat = w.l;
            if (MODE == DX) {
              if (seg > 0) {
                ma = &mp.a2;
                z = seg - 1;
                mat = a.ranks + seg - 1;
              }
            } else if (sub == 0) {
              mat = a.ranks + w.l;
            }
            for (int kt = 0; kt < a.nk; ++kt, ++g) {
              if (!free && !wait_phase(smem_u32(&empty[s]), (lap - 1) & 1u, abort_flag)) {
                ok = false;
                break;
              }
              const uint32_t s_next = (s + 1) % S, lap_next = s_next ? lap : lap + 1;
              free = lap_next == 0 || peek_parity(smem_u32(&empty[s_next]), (lap_next - 1) & 1u);
              uint8_t* st = smem + s * C::STAGE;
              const uint32_t fb = smem_u32(&full[s]);
              arrive_tx(fb, bytes);
              tma_load_3d(smem_u32(st), ma, kt * BK, w.tile * BM, z, fb);
              tma_load_3d(smem_u32(st + C::TILE_A), &mp.b, kt * BK, w.ct * BN, mat, fb);
              tma_load_3d(smem_u32(st + C::TILE_A + TILE_B), &mp.b, kt * BK, w.ct * BN, mat + 2 * a.ranks, fb);
              s = s_next;
              lap = lap_next;
            }
          }
      }
      // the last load issued into every stage must have landed before the CTA exits
      for (int s = 0; s < S; ++s) {
        const int64_t uses = g > s ? (g - 1 - s) / S + 1 : 0;
        if (uses > 0) drain_bar(smem_u32(&full[s]), (uint32_t)((uses - 1) & 1));
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issue
      uint32_t s = 0, phase = 0, slot = 0, b = 0, acc_phase = 0;
      bool ok = true, split_ready = false, acc_ready = false;  // answers about the next slab and accumulator
      for (int q = 0; ok; ++q) {
        const int it = next_item(q);
        if (it < 0) break;
        const Item w = item_of<MODE>(a, it);
        const int units = substeps(w) * segments(w) * a.nu;
        int kt = 0;
        for (int j = 0; j < units; ++j) {
          if (!acc_ready) ok = wait_warp(smem_u32(&acc_empty[b]), acc_phase ^ 1u, abort_flag);
          const uint32_t d = tmem + (uint32_t)A_COLS + b * (uint32_t)BN;
          const uint32_t b_next = b + 1 == (uint32_t)NACC ? 0u : b + 1, acc_next = acc_phase ^ (b_next ? 0u : 1u);
          const int n = min(a.kg, a.nk - kt);
#pragma unroll 1
          for (int i = 0; i < n; ++i) {
            if (!split_ready) ok = ok && wait_warp(smem_u32(&split[s]), phase, abort_flag);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;");
            const uint32_t s_next = s + 1 == (uint32_t)S ? 0u : s + 1, phase_next = phase ^ (s_next ? 0u : 1u);
            const bool peek = peek_parity(smem_u32(&split[s_next]), phase_next);
            const bool peek_acc = peek_parity(smem_u32(&acc_empty[b_next]), acc_next ^ 1u);
            const uint64_t dbh = make_desc(smem_u32(smem + s * C::STAGE + C::TILE_A)), dbl = dbh + (TILE_B >> 4);
            const uint32_t tah = tmem + slot * (uint32_t)C::A_STAGE, tal = tah + (uint32_t)BK;
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < BK / 8; ++kk) {
                mma_ta<BN>(d, tah + kk * 8, dbl + 2 * kk, (i > 0 || kk > 0) ? 1u : 0u);
                if (C::A32) mma_ta<BN>(d, tal + kk * 8, dbh + 2 * kk, 1u);
              }
#pragma unroll
              for (int kk = 0; kk < BK / 8; ++kk) mma_ta<BN>(d, tah + kk * 8, dbh + 2 * kk, 1u);
              // the stage and the A slot are free once these MMAs have completed
              commit(smem_u32(&empty[s]));
              commit(smem_u32(&a_free[slot]));
              if (i + 1 == n) commit(smem_u32(&acc_full[b]));
            }
            split_ready = __all_sync(0xffffffffu, peek);
            acc_ready = __all_sync(0xffffffffu, peek_acc);
            s = s_next;
            phase = phase_next;
            slot = slot + 1 == (uint32_t)C::A_RING ? 0u : slot + 1;
          }
          if (!ok) break;
          kt = kt + n == a.nk ? 0 : kt + n;
          b = b_next;
          acc_phase = acc_next;
        }
      }
      if (elect_one()) {
        commit(smem_u32(drain));  // every MMA completes before tensor memory is freed
        drain_bar(smem_u32(drain), 0);
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    FC_SETMAXNREG_DEC(96);
    // ------------------------------------------------------------------ splitters
    const int r = (warp & 3) * 32 + lane;  // row of the slab, lane of tensor memory
    uint32_t s = 0, phase = 0, slot = 0, slot_phase = 1;  // (slots are free at first)
    bool ok = true, full_ready = false, slot_ready = false;
    for (int q = 0; ok; ++q) {
      const int it = next_item(q);
      if (it < 0) break;
      const Item w = item_of<MODE>(a, it);
      for (int left = substeps(w) * segments(w) * a.nk; left > 0; --left) {
        if (!full_ready) ok = wait_warp(smem_u32(&full[s]), phase, abort_flag);
        if (!slot_ready) ok = ok && wait_warp(smem_u32(&a_free[slot]), slot_phase, abort_flag);
        if (!ok) break;
        const uint32_t s_next = s + 1 == (uint32_t)S ? 0u : s + 1, phase_next = phase ^ (s_next ? 0u : 1u);
        const uint32_t slot_next = slot + 1 == (uint32_t)C::A_RING ? 0u : slot + 1;
        const uint32_t slot_phase_next = slot_phase ^ (slot_next ? 0u : 1u);
        const bool peek_full = peek_parity(smem_u32(&full[s_next]), phase_next);
        const bool peek_slot = peek_parity(smem_u32(&a_free[slot_next]), slot_phase_next);
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint8_t* slab = smem + s * C::STAGE;
        const uint32_t ta = tmem + ((uint32_t)((warp & 3) * 32) << 16) + slot * (uint32_t)C::A_STAGE;
        if constexpr (C::A32) {
          uint32_t x[32];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(&x[4 * c]) = *reinterpret_cast<const uint4*>(slab + chunk_at<float>(r, c));
          store_parts(ta, x);
        } else {
          uint32_t h[32];  // bfloat16 is a tf32 value: its bits are the high half
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(slab + chunk_at<bf16_t>(r, c));
            const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              h[8 * c + 2 * e] = vs[e] << 16;
              h[8 * c + 2 * e + 1] = vs[e] & 0xFFFF0000u;
            }
          }
          tmem_st32(ta, h);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&split[s]));
        full_ready = __all_sync(0xffffffffu, peek_full);
        slot_ready = __all_sync(0xffffffffu, peek_slot);
        s = s_next;
        phase = phase_next;
        slot = slot_next;
        slot_phase = slot_phase_next;
      }
    }
  } else {
    FC_SETMAXNREG_INC(184);
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = (warp - 8) >> 2;
    uint8_t* stage0 = epi + (warp - 8) * C::BUFS * EPI_BUF;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(A_COLS + half * 64);
    const float sa = MODE == DX ? 0.f : __ldg(a.scales + a.ranks + 1);
    uint32_t u = 0;
    uint32_t aux_phase = 0;
    bool ok = true;
    // units u .. u+count-1 are complete (their accumulators are read and then given back)
    auto wait_unit = [&](uint32_t v) {
      const bool done = wait_warp(smem_u32(&acc_full[v % NACC]), (uint32_t)((v / NACC) & 1), abort_flag);
      asm volatile("tcgen05.fence::after_thread_sync;");
      return done;
    };
    auto free_unit = [&](uint32_t v) {
      asm volatile("tcgen05.fence::before_thread_sync;");
      __syncwarp();
      if (lane == 0) arrive(smem_u32(&acc_empty[v % NACC]));
    };
    // 32 columns of this warp's rows from the staging buffer to memory
    auto send = [&](const CUtensorMap* map, uint8_t* buf, int col, int row, int z) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (elect_one()) {
        tma_store_3d(map, smem_u32(buf), col, row, z);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
      __syncwarp();
    };
    for (int q = 0; ok; ++q) {
      const int it = next_item(q);
      if (it < 0) break;
      const Item w = item_of<MODE>(a, it);
      const int col0 = w.ct * BN + half * 64, row0 = w.tile * BM + quarter * 32;
      const int nch = max(0, min(2, (a.N - col0 + 31) / 32));
      if constexpr (MODE == DX) {
        float acc[64];
#pragma unroll
        for (int c = 0; c < 64; ++c) acc[c] = 0.f;
        const int units = segments(w) * a.nu;
        for (int j = 0; j < units && ok; ++j, ++u) {
          if (!(ok = wait_unit(u))) break;
#pragma unroll
          for (int cb = 0; cb < 2; ++cb) {
            float f[32];
            tmem_ld<32>(lane_base + (uint32_t)((u % NACC) * BN + cb * 32), f);
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[cb * 32 + c] += f[c];
          }
          free_unit(u);
        }
        if (!ok) break;
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
          if (cb < nch) {
            if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            put_row<T>(stage0, lane, acc + cb * 32);
            send(&mp.o, stage0, col0 + cb * 32, row0, w.k0);
          }
      } else {
        // the gate: pre-activations of this thread's row and 64 columns
        float z[64];
#pragma unroll
        for (int c = 0; c < 64; ++c) z[c] = 0.f;
        for (int j = 0; j < a.nu && ok; ++j, ++u) {
          if (!(ok = wait_unit(u))) break;
#pragma unroll
          for (int cb = 0; cb < 2; ++cb) {
            float f[32];
            tmem_ld<32>(lane_base + (uint32_t)((u % NACC) * BN + cb * 32), f);
#pragma unroll
            for (int c = 0; c < 32; ++c) z[cb * 32 + c] += f[c];
          }
          free_unit(u);
        }
        if (!ok) break;
        if (a.bias) {
          const T* b = (const T*)a.bias + (int64_t)w.l * a.N;
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (col0 + c < a.N) z[c] += Io<T>::get(b[col0 + c]);
        }
        if constexpr (MODE == FWD) {
#pragma unroll
          for (int c = 0; c < 64; ++c) z[c] = sa * fast_act(a.act, z[c]);
          for (int m = 0; m < w.nm && ok; ++m) {
            float acc[64];
#pragma unroll
            for (int c = 0; c < 64; ++c) acc[c] = 0.f;
            for (int j = 0; j < a.nu; ++j, ++u) {
              if (!(ok = wait_unit(u))) break;
#pragma unroll
              for (int cb = 0; cb < 2; ++cb) {
                float f[32];
                tmem_ld<32>(lane_base + (uint32_t)((u % NACC) * BN + cb * 32), f);
#pragma unroll
                for (int c = 0; c < 32; ++c) acc[cb * 32 + c] += f[c];
              }
              free_unit(u);
            }
            if (!ok) break;
#pragma unroll
            for (int c = 0; c < 64; ++c) acc[c] *= z[c];
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
              if (cb < nch) {
                if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
                put_row<T>(stage0, lane, acc + cb * 32);
                send(&mp.o, stage0, col0 + cb * 32, row0, w.k0 + m);
              }
          }
        } else {
          float sum[64];  // over m of g v
#pragma unroll
          for (int c = 0; c < 64; ++c) sum[c] = 0.f;
          for (int m = 0; m < w.nm && ok; ++m) {
            // the output gradient's boxes come in while the products are computed
            if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            if (lane == 0)
              for (int cb = 0; cb < nch; ++cb) {
                const uint32_t ab = smem_u32(&aux[(warp - 8) * 2 + cb]);
                arrive_tx(ab, 32 * 32 * sizeof(T));
                tma_load_3d(smem_u32(stage0 + cb * EPI_BUF), &mp.g, col0 + cb * 32, row0, w.k0 + m, ab);
              }
            for (int cb = 0; cb < nch; ++cb) {
              const uint32_t ab = smem_u32(&aux[(warp - 8) * 2 + cb]);
              const uint32_t par = (aux_phase >> cb) & 1u;
              aux_phase ^= 1u << cb;
              if (!wait_warp(ab, par, abort_flag)) {
                drain_bar(ab, par);  // the copy may still land: let it, before the buffer goes
                __syncwarp();
                ok = false;
              }
            }
            // g v is a sum over v's units: they are multiplied and given back a few at a time, as many as
            // there are accumulators, so that none of them runs longer than a unit (the first few are
            // what the later ones leave over: those are a full set)
            auto units16 = [&](int count, int c0, float* v) {  // 16 columns of the units from u on, added
              tmem_ld<16>(lane_base + (uint32_t)((u % NACC) * BN + c0), v);
              for (int j = 1; j < count; ++j) {
                float v2[16];
                tmem_ld<16>(lane_base + (uint32_t)(((u + j) % NACC) * BN + c0), v2);
#pragma unroll
                for (int c = 0; c < 16; ++c) v[c] += v2[c];
              }
            };
            int units = a.nu;
#pragma unroll 1
            while (LONG && units > NACC) {
              const int count = units % NACC ? units % NACC : NACC;
              for (int j = 0; j < count; ++j)
                if (!wait_unit(u + j)) ok = false;
#pragma unroll
              for (int q = 0; q < 4; ++q)  // 16 of the warp's 64 columns
                if (q / 2 < nch) {
                  float v[16];
                  units16(count, q * 16, v);
                  const uint8_t* buf = stage0 + q / 2 * EPI_BUF;
                  constexpr int PER = 16 / sizeof(T);
#pragma unroll
                  for (int c = 0; c < 16 / PER; ++c) {
                    Pack<T, PER> gp;
                    gp.raw = *reinterpret_cast<const uint4*>(buf + chunk_at<T>(lane, (q % 2) * (16 / PER) + c));
#pragma unroll
                    for (int k = 0; k < PER; ++k) sum[q * 16 + c * PER + k] += Io<T>::get(gp.at(k)) * v[c * PER + k];
                  }
                }
              for (int j = 0; j < count; ++j, ++u) free_unit(u);
              units -= count;
            }
            for (int j = 0; j < units; ++j)
              if (!wait_unit(u + j)) ok = false;
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
              if (cb < nch) {
                uint8_t* buf = stage0 + cb * EPI_BUF;
                uint4 raw[sizeof(T) == 2 ? 4 : 1];
                if constexpr (sizeof(T) == 2) {  // rows of g and of dv differ in width: all of g first
#pragma unroll
                  for (int c = 0; c < 4; ++c) raw[c] = *reinterpret_cast<const uint4*>(buf + chunk_at<T>(lane, c));
                  __syncwarp();
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  float v[16];
                  units16(units, cb * 32 + h * 16, v);
#pragma unroll
                  for (int c4 = 0; c4 < 4; ++c4) {
                    float4* at = reinterpret_cast<float4*>(buf + chunk_at<float>(lane, h * 4 + c4));
                    float gv[4];
                    if constexpr (sizeof(T) == 4) {
                      const float4 t = *at;
                      gv[0] = t.x, gv[1] = t.y, gv[2] = t.z, gv[3] = t.w;
                    } else {
                      const int e0 = h * 16 + c4 * 4;  // element of the row
                      const uint4 t = raw[e0 / 8];
                      const uint32_t lo = (e0 % 8) ? t.z : t.x, hi = (e0 % 8) ? t.w : t.y;
                      gv[0] = __uint_as_float(lo << 16), gv[1] = __uint_as_float(lo & 0xFFFF0000u);
                      gv[2] = __uint_as_float(hi << 16), gv[3] = __uint_as_float(hi & 0xFFFF0000u);
                    }
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      const int c = cb * 32 + h * 16 + c4 * 4 + e;
                      sum[c] += gv[e] * v[c4 * 4 + e];
                      o[e] = gv[e] * (sa * fast_act(a.act, z[c]));
                    }
                    *at = make_float4(o[0], o[1], o[2], o[3]);
                  }
                }
                send(&mp.o, buf, col0 + cb * 32, row0, w.k0 + m);
              }
            for (int j = 0; j < units; ++j, ++u) free_unit(u);
          }
          if (!ok) break;
          if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int cb = 0; cb < 2; ++cb)
            if (cb < nch) {
#pragma unroll
              for (int c = 0; c < 32; ++c) sum[cb * 32 + c] *= sa * fast_dact(a.act, z[cb * 32 + c]);
              uint8_t* buf = stage0 + cb * EPI_BUF;
              put_row<float>(buf, lane, sum + cb * 32);
              send(&mp.o2, buf, col0 + cb * 32, row0, w.l);
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


template <int MODE, typename T>
int run_stream(const Maps& mp, const Args& args, int sms, cudaStream_t s) {
  constexpr int smem = Cfg<MODE, T>::SMEM;
  const int grid = (int)std::min<int64_t>(args.items, sms);
  if constexpr (MODE == PRE)
    if (args.nu > NACC) {
      static Ready state;
      if (int rc = ready(gated_stream_kernel<MODE, T, true>, smem, state)) return rc;
      gated_stream_kernel<MODE, T, true><<<grid, THREADS, smem, s>>>(mp, args);
      return fc_launched(1);
    }
  static Ready state;
  if (int rc = ready(gated_stream_kernel<MODE, T, false>, smem, state)) return rc;
  gated_stream_kernel<MODE, T, false><<<grid, THREADS, smem, s>>>(mp, args);
  return fc_launched(1);
}
template int run_stream<FWD, float>(const Maps&, const Args&, int, cudaStream_t);
template int run_stream<PRE, float>(const Maps&, const Args&, int, cudaStream_t);
template int run_stream<DX, float>(const Maps&, const Args&, int, cudaStream_t);
template int run_stream<FWD, bf16_t>(const Maps&, const Args&, int, cudaStream_t);
template int run_stream<PRE, bf16_t>(const Maps&, const Args&, int, cudaStream_t);
template int run_stream<DX, bf16_t>(const Maps&, const Args&, int, cudaStream_t);

}  // namespace gtc
}  // namespace fc

#endif  // FC_HOST_EMU
