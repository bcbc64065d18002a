// Gated feed-forward block for bfloat16 rows on tcgen05 tensor cores (sm_100a): the forward, the
// backward's first half and the input gradient, both operands bfloat16.
//
// Mathematics and row layout: gated_ff.cu; modes, work items and lists: gated_ff_tc.cu. Rows and
// weights are bfloat16, so their products are exact in the float accumulator and one product a
// pass is enough; the scales s_l, s_g multiply accumulators, not weights. The tensor cores read
// both operands where the copies put them, so no warp splits anything and sixteen warps share
// the epilogue, in two groups that take the items in turn: one computes gates while the other
// one's products run. For scalars (component 0) the gate and value products share one pass over
// the slab.
//
// What bounds it: the barriers between copy, issue and epilogue. 100,003 rows of 96 -> 200 channels
// are 59 MB (9 us) and their gates 12 us of the special-function units, but a scalar item costs 1.3
// us whatever columns its epilogue has. Measured there: forward 31 us; the backward's first half 64
// us (219 MB, 34 us at the copy rate).
// Rows widened to tf32 in tensor memory, times two tf32 parts of the scaled weights, with one
// group of eight epilogue warps, took 61 and 100 us. (With dv and dz as floats the first half took
// 57 us, and what reads them 46 us more.)
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

// Every step-th item of a list, without a division per item (what one thread does for an item bounds
// the short ones).
struct Walk {
  int tile, q, step, tiles, end;
  __device__ __forceinline__ Walk(const Args& a, int first, int step_)
      : q(first / a.tiles), step(step_), tiles(a.tiles), end(a.per_comp ? a.comps : a.ranks) {
    tile = first - q * a.tiles;
  }
  __device__ __forceinline__ bool more() const { return q < end; }
  __device__ __forceinline__ void next() {
    tile += step;
    while (tile >= tiles) {
      tile -= tiles;
      ++q;
    }
  }
  __device__ __forceinline__ WorkItem item(const Args& a) const { return work_item(a, tile, q); }
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

// Eight floats as two bfloat16 parts, the upper halves of their bits and the rest rounded (16
// significant bits in a float's size), the second PART bytes behind the first: what the
// backward's second half multiplies. dv and dz are sums in 32 bits; these parts are their rounding
// (2^-17) as operands of products whose results are rounded to 8 bits. It moves 0.5% of the stored
// gradients by one last place against the same sums from floats, and leaves their error against 64
// bits where that is (1.659e-3 both ways, 100,003 rows of 96 -> 200 channels).
constexpr int PART = 2048;
__device__ __forceinline__ void put_parts(uint8_t* at, const float* f) {
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t b0 = __float_as_uint(f[2 * k]), b1 = __float_as_uint(f[2 * k + 1]);
    const float r0 = f[2 * k] - __uint_as_float(b0 & 0xFFFF0000u);
    const float r1 = f[2 * k + 1] - __uint_as_float(b1 & 0xFFFF0000u);
    hi[k] = __byte_perm(b0, b1, 0x7632);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo[k]) : "f"(r1), "f"(r0));
  }
  *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  *reinterpret_cast<uint4*>(at + PART) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
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
  const int first = (int)blockIdx.x / a.n_ct, lists = (int)gridDim.x / a.n_ct;

  if (warp < EPI_WARP0) {
    FC_SETMAXNREG_DEC(40);
    if (warp == 0 && elect_one()) {
      // ---------------------------------------------------------------- A producer, work list
      int s = 0;
      uint32_t lap = 0;  // of the ring
      int64_t g = 0;
      bool ok = true, free = true;  // (peeked: the next stage is free)
      Walk at(a, first, lists);
      WorkItem w = at.item(a);
      for (bool more = at.more(); more && ok;) {
        at.next();
        more = at.more();
        const WorkItem wn = at.item(a);  // (used where there is more)
        const int lead = w.k0 == 0 ? 0 : 1;  // passes before the first component's
        for (int p = 0; p < lead + w.nm && ok; ++p) {
          const int z = p < lead ? 0 : w.k0 + p - lead;
          if (p + 1 < lead + w.nm) {
            tma_prefetch_3d(&mp.ap, 0, w.tile * BM, w.k0 + p + 1 - lead);
            if (MODE == PRE) tma_prefetch_3d(&mp.gp, ct * BN, w.tile * BM, w.k0 + p + 1 - lead);
          } else if (more) {
            tma_prefetch_3d(&mp.ap, 0, wn.tile * BM, 0);
            if (MODE == PRE) tma_prefetch_3d(&mp.gp, ct * BN, wn.tile * BM, wn.k0);
          }
          for (int kt = 0; kt < nk; ++kt, ++g) {
            if (!free && !wait_phase(smem_u32(&empty[s]), (lap - 1) & 1u, abort_flag)) {
              ok = false;
              break;
            }
            const int s_next = s + 1 == S ? 0 : s + 1;
            const uint32_t lap_next = s_next ? lap : lap + 1;
            free = lap_next == 0 || peek_parity(smem_u32(&empty[s_next]), (lap_next - 1) & 1u);
            const uint32_t fb = smem_u32(&full[s]);
            arrive_tx(fb, TILE_A);
            tma_load_3d(smem_u32(ring + s * TILE_A), &mp.a, kt * DIRECT_BK, w.tile * BM, z, fb);
            s = s_next;
            lap = lap_next;
          }
        }
        w = wn;
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
      for (Walk at(a, first, lists); at.more() && ok; at.next()) {
        const WorkItem w = at.item(a);
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
      bool acc_ready = false;  // (peeked: the next pass's accumulator is free)
      Walk at(a, first, lists);
      WorkItem w = at.item(a);
      for (bool more = at.more(); more && ok;) {
        at.next();
        more = at.more();
        const WorkItem wn = at.item(a);
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
          if (!acc_ready) ok = wait_warp(smem_u32(&acc_empty[b2]), (n2 / C::NG & 1u) ^ 1u, abort_flag);
          acc_ready = false;
          // the accumulator that the next pass waits for: this group's next one, or the other's
          const bool same = p + 1 < passes;
          const uint32_t nx = same ? n + 1 : (group ? pc[0] : pc[1]) + (wn.k0 == 0 ? 1u : 0u);
          const uint32_t bx = (same ? group : group ^ 1) * C::NG + nx % C::NG;
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
            const bool peek_acc = peek_parity(smem_u32(&acc_empty[bx]), (nx / C::NG & 1u) ^ 1u);
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
            acc_ready = __all_sync(0xffffffffu, peek_acc);
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
        w = wn;
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
    // the same of both parts' boxes
    auto send_parts = [&](const CUtensorMap* map, uint8_t* buf, int row, int z) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (elect_one()) {
        tma_store_3d(map, smem_u32(buf), col, row, z);
        tma_store_3d(map, smem_u32(buf + PART), col, row, z + 1);
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
    for (Walk at(a, first + group * lists, 2 * lists); at.more() && ok; at.next()) {
      const WorkItem w = at.item(a);
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
            // the rows of dv's high parts take the place of g's, chunk by chunk
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float v[16], gate[16];
              tmem_ld<16>(acc_at() + h * 16, v);
              tmem_ld<16>(gate_at + h * 16, gate);
#pragma unroll
              for (int c8 = 0; c8 < 2; ++c8) {
                uint8_t* at = buf + chunk_at<bf16_t>(lane, h * 2 + c8);
                Pack<bf16_t, 8> gp;
                gp.raw = *reinterpret_cast<const uint4*>(at);
                float o[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const float gv = Io<bf16_t>::get(gp.at(k));
                  sum[h * 16 + c8 * 8 + k] += gv * v[c8 * 8 + k];
                  o[k] = gv * gate[c8 * 8 + k];
                }
                put_parts(at, o);
              }
            }
            if (m + 1 < w.nm && ok) {
              boxes_free();  // the other box: its store is a component old
              ask(m + 1, box ^ 1u);
            }
            send_parts(&mp.o, buf, row0, 2 * (w.k0 + m));
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
#pragma unroll
            for (int c8 = 0; c8 < 2; ++c8)
              put_parts(boxes + box * C::BOX + chunk_at<bf16_t>(lane, h * 2 + c8), sum + h * 16 + c8 * 8);
          }
          send_parts(&mp.o2, boxes + box * C::BOX, row0, 2 * w.l);
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

// ---------------------------------------------------------------------------- input gradient
//
// dx_k = s_l dv_k Wv_l (+ s_g sum_l dz_l Wg_l for k = 0) from the two bfloat16 parts of dv and dz
// and the transposed weights, a component's products all in one accumulator (the gates' in a
// second one: their scale is another). An item is one rank of 128 rows and 128 input channels, so
// dv and dz, twice the size of everything else, are read once up to 128 channels.
//
// What bounds it: DRAM (179 MB for 100,003 rows of 96 <- 200 channels, 28 us at the copy rate), but
// a CTA's ring of 64 KB and 782 tiles on 148 CTAs keep it at 52 us; from float dv and dz (split by
// threads, gated_ff_stream.cu) it took 73 us.
//
// The 12 warps: 0 TMA producer of A slabs, 1 MMA issue, 2 TMA producer of the weights, 4-11
// epilogue (two per lane quarter, 64 columns each).
constexpr int X_BN = DIRECT_DX_BN, X_SLAB = X_BN * 128, X_NACC = 4, X_STAGES = 4, X_THREADS = 12 * 32, X_BOX = 2048;
constexpr int X_FIXED = 8 * 2 * X_BOX + X_STAGES * TILE_A + BAR_BYTES + 1024;
static_assert(X_FIXED + 2 * MAX_NK * X_SLAB <= SMEM_MAX, "shared memory per CTA");

// The matrix of an item's pass p and the weight slot that holds it. Slots: a matrix stays until
// the other one has been used and a third is wanted. What a scalar item of several ranks multiplies
// by (a value matrix, then every rank's gates) is used once and given back at once.
struct Slots {
  int held[2] = {-1, -1};
  int last = 1;
  // slot of matrix m; fresh: it has to be loaded
  __device__ __forceinline__ int of(int m, bool& fresh) {
    fresh = false;
    if (held[0] == m) return last = 0;
    if (held[1] == m) return last = 1;
    fresh = true;
    last ^= 1;
    if (last) held[1] = m;
    else held[0] = m;
    return last;
  }
  __device__ __forceinline__ void drop(int slot) {
    if (slot) held[1] = -1;
    else held[0] = -1;
  }
};

__global__ void __launch_bounds__(X_THREADS, 1) gated_bf16_dx_kernel(const __grid_constant__ Maps mp, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nk = a.nk;
  uint8_t* wmem = smem;                       // [slot][k slab]
  uint8_t* ring = wmem + 2 * nk * X_SLAB;     // A stages
  uint8_t* epi = ring + X_STAGES * TILE_A;    // staging boxes
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + 8 * 2 * X_BOX);
  uint64_t* empty = full + X_STAGES;
  uint64_t* w_full = empty + X_STAGES;        // per slot
  uint64_t* w_free = w_full + 2;
  uint64_t* acc_full = w_free + 2;
  uint64_t* acc_empty = acc_full + X_NACC;
  uint64_t* drain = acc_empty + X_NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * X_STAGES + 4 + 2 * X_NACC + 1) * 8 + 8 <= BAR_BYTES, "barriers");

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
    for (int s = 0; s < X_STAGES; ++s) {
      init(&full[s], 1);
      init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      init(&w_full[b], 1);
      init(&w_free[b], 1);
    }
    for (int b = 0; b < X_NACC; ++b) {
      init(&acc_full[b], 1);
      init(&acc_empty[b], 8);
    }
    init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;
  const int ct = (int)blockIdx.x % a.n_ct;
  const int first = (int)blockIdx.x / a.n_ct, lists = (int)gridDim.x / a.n_ct, items = (int)a.items;
  // Last rows first: what the backward's first half wrote last is in L2 still.
  auto item_at = [&](int it) {
    WorkItem w = work_item(a, it);
    w.tile = a.tiles - 1 - w.tile;
    return w;
  };
  auto passes_of = [&](const WorkItem& w) { return w.k0 == 0 ? a.ranks + 1 : w.nm; };
  auto matrix_of = [&](const WorkItem& w, int p) { return w.k0 > 0 ? w.l : p == 0 ? 0 : a.ranks + p - 1; };

  if (warp == 0) {
    if (elect_one()) {
      uint32_t s = 0, lap = 0;
      int64_t g = 0;
      bool ok = true, free = true;
      for (int it = first; it < items && ok; it += lists) {
        const WorkItem w = item_at(it);
        const int passes = passes_of(w);
        for (int p = 0; p < passes && ok; ++p) {
          const bool gates = w.k0 == 0 && p > 0;
          for (int i = 0; i < 2 * nk; ++i, ++g) {  // slab and part
            if (!free && !wait_phase(smem_u32(&empty[s]), (lap - 1) & 1u, abort_flag)) {
              ok = false;
              break;
            }
            const uint32_t s_next = (s + 1) % X_STAGES, lap_next = s_next ? lap : lap + 1;
            free = lap_next == 0 || peek_parity(smem_u32(&empty[s_next]), (lap_next - 1) & 1u);
            const uint32_t fb = smem_u32(&full[s]);
            arrive_tx(fb, TILE_A);
            tma_load_3d(smem_u32(ring + s * TILE_A), gates ? &mp.a2 : &mp.a, (i >> 1) * DIRECT_BK, w.tile * BM,
                        2 * (gates ? p - 1 : w.k0 + p) + (i & 1), fb);
            s = s_next;
            lap = lap_next;
          }
        }
      }
      for (int t = 0; t < X_STAGES; ++t) {
        const int64_t uses = g > t ? (g - 1 - t) / X_STAGES + 1 : 0;
        if (uses > 0) drain_bar(smem_u32(&full[t]), (uint32_t)((uses - 1) & 1));
      }
    }
  } else if (warp == 2) {
    if (elect_one()) {
      Slots slots;
      int loads[2] = {0, 0};
      bool ok = true;
      for (int it = first; it < items && ok; it += lists) {
        const WorkItem w = item_at(it);
        const int passes = w.k0 == 0 ? a.ranks + 1 : 1;
        for (int p = 0; p < passes && ok; ++p) {
          bool fresh;
          const int m = matrix_of(w, p), slot = slots.of(m, fresh);
          if (fresh) {
            const int before = slot ? loads[1] : loads[0];
            if (before > 0 && !wait_phase(smem_u32(&w_free[slot]), (uint32_t)((before - 1) & 1), abort_flag)) {
              ok = false;
              break;
            }
            const uint32_t fb = smem_u32(&w_full[slot]);
            arrive_tx(fb, (uint32_t)(nk * X_SLAB));
            for (int kt = 0; kt < nk; ++kt)
              tma_load_3d(smem_u32(wmem + (slot * nk + kt) * X_SLAB), &mp.b, kt * DIRECT_BK, ct * X_BN, m, fb);
            if (slot) ++loads[1];
            else ++loads[0];
          }
          if (w.k0 == 0 && a.ranks > 1) slots.drop(slot);
        }
      }
      if (loads[0] > 0) drain_bar(smem_u32(&w_full[0]), (uint32_t)((loads[0] - 1) & 1));
      if (loads[1] > 0) drain_bar(smem_u32(&w_full[1]), (uint32_t)((loads[1] - 1) & 1));
    }
  } else if (warp == 1) {
    const uint64_t wdesc = make_desc(smem_u32(wmem)), adesc = make_desc(smem_u32(ring));
    Slots slots;
    uint32_t w_phase = 3u, unfreed = 0u;  // bit per slot: phase of its last load; not given back
    uint32_t s = 0, lap = 0, n = 0;
    bool ok = true, ready_a = false;
    for (int it = first; it < items && ok; it += lists) {
      const WorkItem w = item_at(it);
      const int passes = passes_of(w);
      for (int p = 0; p < passes && ok; ++p) {
        bool fresh;
        const int slot = slots.of(matrix_of(w, p), fresh);
        const uint32_t bit = 1u << slot;
        if (fresh) {
          if ((unfreed & bit) && elect_one()) commit(smem_u32(&w_free[slot]));
          __syncwarp();
          unfreed |= bit;
          w_phase ^= bit;
        }
        // all gate matrices' products add up in the accumulator behind the values'
        const bool opens = w.k0 > 0 || p <= 1, closes = w.k0 > 0 || p == 0 || p == a.ranks;
        if (opens) ok = wait_warp(smem_u32(&acc_empty[n % X_NACC]), (n / X_NACC & 1u) ^ 1u, abort_flag);
        if (fresh) ok = ok && wait_warp(smem_u32(&w_full[slot]), (w_phase >> slot) & 1u, abort_flag);
        const uint32_t d = tmem + n % X_NACC * X_BN;
        for (int i = 0; i < 2 * nk; ++i) {
          if (!ready_a) ok = ok && wait_warp(smem_u32(&full[s]), lap & 1u, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;");
          const uint32_t s_next = (s + 1) % X_STAGES, lap_next = s_next ? lap : lap + 1;
          const bool peek = peek_parity(smem_u32(&full[s_next]), lap_next & 1u);
          if (elect_one()) {
            mma_slab<X_BN>(d, adesc + (uint64_t)(s * (TILE_A >> 4)),
                           wdesc + (uint64_t)((slot * nk + (i >> 1)) * (X_SLAB >> 4)), !opens || i > 0);
            commit(smem_u32(&empty[s]));
          }
          ready_a = __all_sync(0xffffffffu, peek);
          s = s_next;
          lap = lap_next;
        }
        if (ok && elect_one()) {
          if (closes) commit(smem_u32(&acc_full[n % X_NACC]));
          if (w.k0 == 0 && a.ranks > 1) commit(smem_u32(&w_free[slot]));
        }
        __syncwarp();
        if (w.k0 == 0 && a.ranks > 1) {
          slots.drop(slot);
          unfreed &= ~bit;
        }
        if (closes) ++n;
      }
    }
    if (elect_one()) {
      commit(smem_u32(drain));
      drain_bar(smem_u32(drain), 0);
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int e = warp - 4, quarter = warp & 3, half = e >> 2;
    uint8_t* boxes = epi + e * 2 * X_BOX;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 64);
    const float sg = __ldg(a.scales + a.ranks);
    const int col = ct * X_BN + half * 64;
    uint32_t n = 0, box = 0;
    bool ok = true;
    for (int it = first; it < items && ok; it += lists) {
      const WorkItem w = item_at(it);
      const float sv = __ldg(a.scales + w.l);
      const bool two = w.k0 == 0;
      for (int m = 0; m < w.nm; ++m) {
        ok = wait_warp(smem_u32(&acc_full[n % X_NACC]), n / X_NACC & 1u, abort_flag);
        if (two) ok = ok && wait_warp(smem_u32(&acc_full[(n + 1) % X_NACC]), (n + 1) / X_NACC & 1u, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (col + h * 32 >= a.N) break;
          float f[32];
          tmem_ld<32>(lanes + n % X_NACC * X_BN + h * 32, f);
#pragma unroll
          for (int c = 0; c < 32; ++c) f[c] *= sv;
          if (two) {
            float z[32];
            tmem_ld<32>(lanes + (n + 1) % X_NACC * X_BN + h * 32, z);
#pragma unroll
            for (int c = 0; c < 32; ++c) f[c] = fmaf(sg, z[c], f[c]);
          }
          // (the elected lane is the same every time; at most the other box's store still reads)
          if (elect_one()) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          __syncwarp();
          put_row<bf16_t>(boxes + box * X_BOX, lane, f);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (elect_one()) {
            tma_store_3d(&mp.o, smem_u32(boxes + box * X_BOX), col + h * 32, w.tile * BM + quarter * 32, w.k0 + m);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          __syncwarp();
          box ^= 1;
        }
        asm volatile("tcgen05.fence::before_thread_sync;");
        __syncwarp();
        if (lane == 0) {
          arrive(smem_u32(&acc_empty[n % X_NACC]));
          if (two) arrive(smem_u32(&acc_empty[(n + 1) % X_NACC]));
        }
        n += two ? 2 : 1;
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

int run_direct_dx(const Maps& mp, const Args& a, int sms, cudaStream_t s) {
  static Ready state;
  if (int rc = ready(gated_bf16_dx_kernel, SMEM_MAX, state, 0)) return rc;
  const int lists = (int)std::min<int64_t>(a.items, sms / a.n_ct);
  gated_bf16_dx_kernel<<<lists * a.n_ct, X_THREADS, X_FIXED + 2 * a.nk * X_SLAB, s>>>(mp, a);
  return fc_launched(1);
}

template <int MODE>
int run_direct(const Maps& mp, Args a, int sms, cudaStream_t s) {
  using C = DCfg<MODE>;
  a.stages = C::stages(a.nk);
  static Ready state;
  if (int rc = ready(gated_bf16_kernel<MODE>, SMEM_MAX, state, D_REGS)) return rc;
  const int lists = (int)std::min<int64_t>(a.items, sms / a.n_ct);
  gated_bf16_kernel<MODE><<<lists * a.n_ct, D_THREADS, C::smem(a.nk, a.stages), s>>>(mp, a);
  return fc_launched(1);
}
template int run_direct<FWD>(const Maps&, Args, int, cudaStream_t);
template int run_direct<PRE>(const Maps&, Args, int, cudaStream_t);

}  // namespace gtc
}  // namespace fc

#endif  // FC_HOST_EMU
