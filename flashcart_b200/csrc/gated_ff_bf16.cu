// Gated feed-forward block for bfloat16 rows on tcgen05 tensor cores (sm_100a): the forward and
// the backward's first half, both operands bfloat16.
//
// Mathematics and row layout: gated_ff.cu; modes, work items and lists: gated_ff_tc.cu. Rows and
// weights are bfloat16, so their products are exact in the float accumulator and one product a
// pass is enough; the scales s_l, s_g multiply accumulators, not weights. The tensor cores read
// both operands where the copies put them, so no warp splits anything and sixteen warps share
// the epilogue, in two groups that take the items in turn: one computes gates while the other
// one's products run. For scalars (component 0) the gate and value products share one pass over
// the slab.
//
// What bounds it: the epilogue. 100,003 rows of 96 -> 200 channels are 59 MB (9 us), but a
// gate costs about 25 instructions, two of them on the special-function units.
// Measured there: forward 32 us; the backward's first half 57 us (219 MB, 34 us at the copy rate).
// Rows widened to tf32 in tensor memory, times two tf32 parts of the scaled weights, with one
// group of eight epilogue warps, took 61 and 100 us.
//
// Roles of the 20 warps (one persistent CTA per SM):
//   warp 0       TMA producer of A slabs
//   warp 1       MMA issue
//   warp 2       TMA producer of the weights
//   warps 4-19   epilogue: two groups of two warps per lane quarter, 32 columns each
#include "gated_ff_tc.cuh"

#ifndef FC_HOST_EMU

#include <algorithm>

namespace fc {
namespace gtc {

namespace {

constexpr int BN = 64;
constexpr int W_SLAB = BN * 128;   // 64 output channels x 64 input channels
constexpr int TILE_A = BM * 128;   // 128 rows x 64 channels
constexpr int MAX_NK = DIRECT_K / DIRECT_BK;
constexpr int MAX_STAGES = 6;
constexpr int EPI_WARP0 = 4, EPI_WARPS = 16, D_THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int D_REGS = 96;  // per thread at launch: 640 x 96 = 128 x 40 + 512 x 104 (and 3,072 left)
constexpr int SMEM_MAX = 227 * 1024;
constexpr int Z_COL = 256;  // PRE, behind 2 x 2 accumulators: the groups' slopes, then gates (PRE)

template <int MODE>
struct DCfg {
  static constexpr int BUFS = MODE == PRE ? 2 : 1;  // staging boxes per epilogue warp
  static constexpr int BOX = MODE == PRE ? 4096 : 2048;
  // accumulators of a group: a scalar item takes two, so with four the next item's products run
  // while this one's are read (PRE keeps its gates in their place)
  static constexpr int NG = MODE == PRE ? 2 : 4;
  static constexpr int FIXED = EPI_WARPS * BUFS * BOX + BAR_BYTES + 1024;
  static int stages(int nk) { return std::min(MAX_STAGES, (SMEM_MAX - FIXED - 2 * nk * W_SLAB) / TILE_A); }
  static int smem(int nk, int st) { return FIXED + 2 * nk * W_SLAB + st * TILE_A; }
};

// D (+)= A x B of one 64-channel slab, both K-major in shared memory; N rows of B.
template <int N>
__device__ __forceinline__ void mma_slab(uint32_t d, uint64_t da, uint64_t db, bool more) {
  constexpr uint32_t idesc =
      (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(da + 2 * kk), "l"(db + 2 * kk), "r"(idesc), "r"((more || kk > 0) ? 1u : 0u));
}

// sigma(z) for results that are rounded to bfloat16 (unit roundoff 2^-8): the exponent -z log2(e)
// is rounded once, which moves 2^t by |t| 2^-24 of itself at most.
__device__ __forceinline__ float brief_sigmoid(float z) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.44269502f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}

template <int MODE>
__global__ void __launch_bounds__(D_THREADS, 1) gated_bf16_kernel(const __grid_constant__ Maps mp, const Args a) {
  using C = DCfg<MODE>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = a.stages, nk = a.nk;
  uint8_t* wmem = smem;                    // [slab][gate or value matrix of the rank]
  uint8_t* ring = wmem + 2 * nk * W_SLAB;  // A stages
  uint8_t* epi = ring + S * TILE_A;        // staging boxes
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + EPI_WARPS * C::BUFS * C::BOX);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* w_full = empty + MAX_STAGES;   // [slot][k slab]
  uint64_t* w_free = w_full + 2 * MAX_NK;
  uint64_t* acc_full = w_free + 2;         // [group][accumulator]
  uint64_t* acc_empty = acc_full + 2 * C::NG;
  uint64_t* drain = acc_empty + 2 * C::NG;
  uint64_t* aux = drain + 1;               // per epilogue warp and box: g has landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux + EPI_WARPS * C::BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * MAX_STAGES + 2 * MAX_NK + 2 + 4 * C::NG + 1 + EPI_WARPS * C::BUFS) * 8 + 8 <= BAR_BYTES,
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
      init(&empty[s], 1);
    }
    for (int b = 0; b < 2 * MAX_NK; ++b) init(&w_full[b], 1);
    for (int b = 0; b < 2; ++b) init(&w_free[b], 1);
    for (int b = 0; b < 2 * C::NG; ++b) {
      init(&acc_full[b], 1);
      init(&acc_empty[b], EPI_WARPS / 2);
    }
    init(drain, 1);
    for (int b = 0; b < EPI_WARPS * C::BUFS; ++b) init(&aux[b], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;
  const int ct = (int)blockIdx.x % a.n_ct;  // this CTA's 64 output channels

  // The CTA's items: every `lists`-th of its column tile's list. (Drawn from a shared counter and
  // handed to the warps through barriers, each item cost every warp a barrier's answer.)
  const int first = (int)blockIdx.x / a.n_ct, lists = (int)gridDim.x / a.n_ct, items = (int)a.items;

  if (warp < EPI_WARP0) {
    FC_SETMAXNREG_DEC(40);
    if (warp == 0 && elect_one()) {
      // ---------------------------------------------------------------- A producer, work list
      int s = 0;
      uint32_t lap = 0;  // of the ring
      int64_t g = 0;
      bool ok = true;
      for (int it = first; it < items && ok; it += lists) {
        const WorkItem w = work_item(a, it);
        const int lead = w.k0 == 0 ? 0 : 1;  // passes before the first component's
        for (int p = 0; p < lead + w.nm && ok; ++p) {
          const int z = p < lead ? 0 : w.k0 + p - lead;
          if (p + 1 < lead + w.nm) {
            tma_prefetch_3d(&mp.ap, 0, w.tile * BM, w.k0 + p + 1 - lead);
            if (MODE == PRE) tma_prefetch_3d(&mp.gp, ct * BN, w.tile * BM, w.k0 + p + 1 - lead);
          } else if (it + lists < items) {
            const WorkItem wn = work_item(a, it + lists);
            tma_prefetch_3d(&mp.ap, 0, wn.tile * BM, 0);
            if (MODE == PRE) tma_prefetch_3d(&mp.gp, ct * BN, wn.tile * BM, wn.k0);
          }
          for (int kt = 0; kt < nk; ++kt, ++g) {
            if (lap > 0 && !wait_phase(smem_u32(&empty[s]), (lap - 1) & 1u, abort_flag)) {
              ok = false;
              break;
            }
            const uint32_t fb = smem_u32(&full[s]);
            arrive_tx(fb, TILE_A);
            tma_load_3d(smem_u32(ring + s * TILE_A), &mp.a, kt * DIRECT_BK, w.tile * BM, z, fb);
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
      int rank = -1, loads[2] = {0, 0};
      bool ok = true;
      for (int it = first; it < items && ok; it += lists) {
        const WorkItem w = work_item(a, it);
        if (w.l == rank) continue;
        rank = w.l;
#pragma unroll
        for (int slot = 0; slot < 2; ++slot) {
          if (!ok || (loads[slot] > 0 &&
                      !wait_phase(smem_u32(&w_free[slot]), (uint32_t)((loads[slot] - 1) & 1), abort_flag))) {
            ok = false;
            break;
          }
          for (int kt = 0; kt < nk; ++kt) {
            const uint32_t fb = smem_u32(&w_full[slot * MAX_NK + kt]);
            arrive_tx(fb, W_SLAB);
            tma_load_3d(smem_u32(wmem + (2 * kt + slot) * W_SLAB), &mp.b, kt * DIRECT_BK, ct * BN,
                        slot == 0 ? a.ranks + w.l : w.l, fb);
          }
          ++loads[slot];
        }
      }
      for (int kt = 0; kt < nk; ++kt)
#pragma unroll
        for (int slot = 0; slot < 2; ++slot)
          if (loads[slot] > 0) drain_bar(smem_u32(&w_full[slot * MAX_NK + kt]), (uint32_t)((loads[slot] - 1) & 1));
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issue
      const uint64_t wdesc = make_desc(smem_u32(wmem)), adesc = make_desc(smem_u32(ring));
      int rank = -1, loads = 0;
      uint32_t s = 0, lap = 0, pc[2] = {0u, 0u};  // passes of each group so far
      bool ok = true, ready_a = false;  // (peeked: the next slab is there)
      int group = 1;
      for (int it = first; it < items && ok; it += lists) {
        const WorkItem w = work_item(a, it);
        group ^= 1;
        bool check = false;
        if (w.l != rank) {
          rank = w.l;
          if (loads > 0 && elect_one()) {
            commit(smem_u32(&w_free[0]));
            commit(smem_u32(&w_free[1]));
          }
          __syncwarp();
          ++loads;
          check = true;
        }
        const bool both = w.k0 == 0;  // gate and value products from the same slabs
        const int passes = both ? w.nm : 1 + w.nm;
        uint32_t n = group ? pc[1] : pc[0];
        for (int p = 0; p < passes && ok; ++p) {
          // a scalar item's two accumulators side by side, if the ring does not part them; the
          // epilogue frees the first one before the second
          const bool two = both && p == 0;
          const uint32_t n2 = n + (two ? 1u : 0u), b = group * C::NG + n % C::NG, b2 = group * C::NG + n2 % C::NG;
          ok = wait_warp(smem_u32(&acc_empty[b2]), (n2 / C::NG & 1u) ^ 1u, abort_flag);
          const uint32_t slot = p == 0 ? 0u : 1u;
          for (int kt = 0; kt < nk; ++kt) {
            if (check && p < 2) {
              const uint32_t wp = (uint32_t)((loads - 1) & 1);
              ok = ok && wait_warp(smem_u32(&w_full[slot * MAX_NK + kt]), wp, abort_flag);
              if (two) ok = ok && wait_warp(smem_u32(&w_full[MAX_NK + kt]), wp, abort_flag);
            }
            if (!ready_a) ok = ok && wait_warp(smem_u32(&full[s]), lap & 1u, abort_flag);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;");
            const uint32_t s_next = s + 1 == (uint32_t)S ? 0u : s + 1, lap_next = s_next ? lap : lap + 1;
            const bool peek = peek_parity(smem_u32(&full[s_next]), lap_next & 1u);
            if (elect_one()) {
              const uint64_t da = adesc + (uint64_t)(s * (TILE_A >> 4));
              const uint64_t db = wdesc + (uint64_t)((2 * kt + slot) * (W_SLAB >> 4));
              if (b2 == b + 1) {
                mma_slab<2 * BN>(tmem + b * BN, da, db, kt > 0);
              } else {
                mma_slab<BN>(tmem + b * BN, da, db, kt > 0);
                if (two) mma_slab<BN>(tmem + b2 * BN, da, db + (W_SLAB >> 4), kt > 0);
              }
              commit(smem_u32(&empty[s]));  // the stage is free once these MMAs have completed
            }
            ready_a = __all_sync(0xffffffffu, peek);
            s = s_next;
            lap = lap_next;
          }
          if (ok && elect_one()) {
            commit(smem_u32(&acc_full[b]));
            if (two) commit(smem_u32(&acc_full[b2]));
          }
          __syncwarp();
          n += two ? 2 : 1;
        }
        if (group) pc[1] = n;
        else pc[0] = n;
      }
      if (elect_one()) {
        commit(smem_u32(drain));  // every MMA completes before tensor memory is freed
        drain_bar(smem_u32(drain), 0);
      }
      __syncwarp();
    }
  } else {
    FC_SETMAXNREG_INC(104);
    // ------------------------------------------------------------------ epilogue
    // a thread holds its row's 32 columns
    const int e = warp - EPI_WARP0, group = e >> 3, quarter = warp & 3, half = (e >> 2) & 1;
    uint8_t* boxes = epi + e * C::BUFS * C::BOX;
    uint64_t* landed = aux + e * C::BUFS;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 32);
    const float sa = __ldg(a.scales + a.ranks + 1), sg = __ldg(a.scales + a.ranks);
    const int col = ct * BN + half * 32;
    const bool live = col < a.N;  // the warp has columns to write
    uint32_t n = 0;               // passes of this group so far
    bool ok = true;
    auto acc_at = [&]() { return lanes + (group * C::NG + n % C::NG) * BN; };
    // the accumulator `ahead` of the one in turn is done, and with it all before that
    auto wait_acc = [&](uint32_t ahead) {
      const uint32_t i = n + ahead;
      const bool done = wait_warp(smem_u32(&acc_full[group * C::NG + i % C::NG]), i / C::NG & 1u, abort_flag);
      asm volatile("tcgen05.fence::after_thread_sync;");
      return done;
    };
    auto free_acc = [&]() {
      asm volatile("tcgen05.fence::before_thread_sync;");
      __syncwarp();
      if (lane == 0) arrive(smem_u32(&acc_empty[group * C::NG + n % C::NG]));
      ++n;
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
    // earlier stores have read their boxes (box_free: all but the last one)
    auto boxes_free = [&]() {
      if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
    };
    auto box_free = [&]() {
      if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      __syncwarp();
    };
    uint32_t box = 0, box_phase = 0;  // PRE: the box in turn; bit b: parity of landed[b]'s next completion
    for (int it = first + group * lists; it < items && ok; it += 2 * lists) {
      const WorkItem w = work_item(a, it);
      const int row0 = w.tile * BM + quarter * 32;
      const float sv = __ldg(a.scales + w.l);
      // ask for component m's box of g
      int asked = 0, got = 0;
      auto ask = [&](int m, uint32_t b) {
        asked = m + 1;
        if (elect_one()) {
          const uint32_t fb = smem_u32(&landed[b]);
          arrive_tx(fb, 32 * 32 * 2);
          tma_load_3d(smem_u32(boxes + b * C::BOX), &mp.g, col, row0, w.k0 + m, fb);
        }
        __syncwarp();
      };
      if (MODE == PRE && live) {
        box_free();
        ask(0, box);
      }
      float z[32];  // pre-activations of this thread's row
      const bool two = w.k0 == 0;  // gate and value products were one pass
      ok = wait_acc(two ? 1u : 0u);
      // (every phase of a barrier has to be seen, or its parity would tell too little: the answer
      // about the one that was not waited for is looked at later)
      const uint32_t skipped = n;
      const bool seen = !two || peek_parity(smem_u32(&acc_full[group * C::NG + n % C::NG]), n / C::NG & 1u);
      tmem_ld<32>(acc_at(), z);
      free_acc();
      if (live) {
#pragma unroll
        for (int c = 0; c < 32; ++c) z[c] *= sg;
        if (a.bias) {
          const bf16_t* b = (const bf16_t*)a.bias + (int64_t)w.l * a.N + col;
          if (!((reinterpret_cast<uintptr_t>(b) | (uintptr_t)(2 * a.N)) & 15)) {
#pragma unroll
            for (int c8 = 0; c8 < 4; ++c8)
              if (col + 8 * c8 < a.N) {
                Pack<bf16_t, 8> v;
                v.load(b + 8 * c8);
#pragma unroll
                for (int k = 0; k < 8; ++k) z[8 * c8 + k] += Io<bf16_t>::get(v.at(k));
              }
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (col + c < a.N) z[c] += Io<bf16_t>::get(b[c]);
          }
        }
      }
      if (ok && !__all_sync(0xffffffffu, seen))
        ok = wait_warp(smem_u32(&acc_full[group * C::NG + skipped % C::NG]), skipped / C::NG & 1u, abort_flag);
      if constexpr (MODE == FWD) {
        if (live)
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float sig = brief_sigmoid(z[c]);
            z[c] = sa * sv * (a.act == FC_GATE_SIGMOID ? sig : z[c] * sig);
          }
        for (int m = 0; m < w.nm && ok; ++m) {
          if (!two && !(ok = wait_acc(0u))) break;
          float f[32];
          tmem_ld<32>(acc_at(), f);
          free_acc();
          if (live) {
#pragma unroll
            for (int c = 0; c < 32; ++c) f[c] *= z[c];
            boxes_free();
            put_row<bf16_t>(boxes, lane, f);
            send(&mp.o, boxes, row0, w.k0 + m);
          }
        }
      } else {
        // gates and slopes wait in tensor memory
        const uint32_t z_at = lanes + (uint32_t)(Z_COL + group * BN), gate_at = z_at + 2 * BN;
        if (live) {
          float slope[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float sig = brief_sigmoid(z[c]), r = 1.f - sig;
            slope[c] = sa * sv * (a.act == FC_GATE_SIGMOID ? sig * r : sig * fmaf(z[c], r, 1.f));
            z[c] = sa * (a.act == FC_GATE_SIGMOID ? sig : z[c] * sig);
          }
          tmem_st32(z_at, reinterpret_cast<const uint32_t*>(slope));
          tmem_st32(gate_at, reinterpret_cast<const uint32_t*>(z));
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        float sum[32];  // over m of g v / s_l
#pragma unroll
        for (int c = 0; c < 32; ++c) sum[c] = 0.f;
        for (int m = 0; m < w.nm && ok; ++m) {
          if (!two && !wait_acc(0u)) ok = false;
          if (got < asked) {
            ++got;
            const uint32_t par = (box_phase >> box) & 1u;
            box_phase ^= 1u << box;
            if (!wait_warp(smem_u32(&landed[box]), par, abort_flag)) {
              drain_bar(smem_u32(&landed[box]), par);  // the copy may still land: let it
              __syncwarp();
              ok = false;
            }
            uint8_t* buf = boxes + box * C::BOX;
            uint4 raw[4];  // rows of g and of dv differ in width: all of g first
#pragma unroll
            for (int c = 0; c < 4; ++c) raw[c] = *reinterpret_cast<const uint4*>(buf + chunk_at<bf16_t>(lane, c));
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float v[16], gate[16];
              tmem_ld<16>(acc_at() + h * 16, v);
              tmem_ld<16>(gate_at + h * 16, gate);
#pragma unroll
              for (int c4 = 0; c4 < 4; ++c4) {
                const int e0 = h * 16 + c4 * 4;  // element of the row
                const uint4 t = raw[e0 / 8];
                const uint32_t lo = (e0 % 8) ? t.z : t.x, hi = (e0 % 8) ? t.w : t.y;
                const float gv[4] = {__uint_as_float(lo << 16), __uint_as_float(lo & 0xFFFF0000u),
                                     __uint_as_float(hi << 16), __uint_as_float(hi & 0xFFFF0000u)};
                float o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const int c = e0 + k;
                  sum[c] += gv[k] * v[c4 * 4 + k];
                  o[k] = gv[k] * gate[c4 * 4 + k];
                }
                *reinterpret_cast<float4*>(buf + chunk_at<float>(lane, h * 4 + c4)) =
                    make_float4(o[0], o[1], o[2], o[3]);
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
          put_row<float>(boxes + box * C::BOX, lane, sum);
          send(&mp.o2, boxes + box * C::BOX, row0, w.l);
          box ^= 1u;
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

}  // namespace

template <int MODE>
int run_direct(const Maps& mp, Args a, int sms, cudaStream_t s) {
  using C = DCfg<MODE>;
  a.stages = C::stages(a.nk);
  static Ready state;
  if (int rc = ready(gated_bf16_kernel<MODE>, SMEM_MAX, state, D_REGS)) return rc;
  const int lists = (int)std::min<int64_t>(a.items, sms / a.n_ct);
  gated_bf16_kernel<MODE><<<lists * a.n_ct, D_THREADS, C::smem(a.nk, a.stages), s>>>(mp, a);
  return fc_check_launch();
}
template int run_direct<FWD>(const Maps&, Args, int, cudaStream_t);
template int run_direct<PRE>(const Maps&, Args, int, cudaStream_t);

}  // namespace gtc
}  // namespace fc

#endif  // FC_HOST_EMU
