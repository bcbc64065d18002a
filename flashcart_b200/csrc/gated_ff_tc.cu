// Gated feed-forward block on tcgen05 tensor cores, fed by TMA (sm_100a): float32 rows as
// 3xTF32 products, bfloat16 rows (exact in tf32) times weights in two tf32 parts.
//
// Mathematics and row layout: gated_ff.cu. The scales s_l, s_g are folded into the split
// weights, so the accumulators hold v_k and z_l - b_l themselves.
//
// gated_tc_kernel, one persistent CTA per SM, 16 warps:
//   warp 0       TMA producer, and the CTA's draw from the work list (an atomic counter)
//   warp 1       MMA issue (one thread)
//   warps 4-7    splitters: the A slab (128 rows x 32 channels) to tf32 parts in tensor memory
//   warps 8-15   epilogue: two warps per lane quarter, 64 columns each
// A work item is one rank l of 128 rows (and 128 hidden channels): first the gate product
// x_0 Wg_l, whose activation the epilogue warps keep in registers (64 columns of their row),
// then the 2l+1 value products, each multiplied by the gate on its way out. So x is read
// once per component (x_0 once more per rank), y is written once, and neither gates nor
// values touch memory. Three modes share the pipeline:
//   FWD  y_k = a_l v_k
//   PRE  the backward's first half: z_l and v_k again; g comes in by TMA while they are
//        computed; dv_k = g a_l goes out, sum_m g v_k stays in registers until the rank is
//        done and dz_l goes out
//   DX   dx_k = dv_k Wv_l (+ sum_l dz_l Wg_l for k = 0): items are (128 rows, component)
// wgrad_kernel forms dWv_l and dWg_l: the rows are the reduction, so both operands have to be
// transposed; the splitters do that on the way (a lane of tensor memory or a row of the
// K-major B tile is one channel, and a thread gathers its 32 rows' values from the row-major
// slab without bank conflicts). Every CTA takes an equal share of the slabs of all weight
// matrices, and a second kernel adds the partial matrices in order.
//
// Waits are bounded: on expiry the CTA raises FC_DEV_TIMEOUT, all roles stop, copies and MMAs
// in flight are drained and tensor memory is freed.
#include "gated_ff.cuh"
#include "tc_common.cuh"

#ifndef FC_HOST_EMU

#include <algorithm>

namespace fc {
namespace gtc {

using namespace tma;

constexpr int BN = 128, BK = 32, THREADS = 512;
constexpr int EPI_WARPS = 8, EPI_BUF = 4096, EPI_BYTES = EPI_WARPS * 2 * EPI_BUF;
constexpr int BAR_BYTES = 512;
constexpr int TILE_B = BN * BK * 4;
constexpr int A_COLS = 128;  // tensor-memory columns of the A parts' ring
constexpr int NACC = 3;      // accumulators behind them
constexpr int SCHED = 4;
// Slabs per accumulation unit. A tensor-core accumulation truncates the running sum (measured
// relative error: 4.5e-7 after 12 instructions, 8.2e-7 after 24, 1.6e-6 after 48), so a unit
// is 64 products, its small terms (hi x lo, lo x hi) go in before the slab's hi x hi while
// the sum is small, and the units are added in fp32 registers.
constexpr int KG = 2;
enum { FWD = 0, PRE = 1, DX = 2 };

template <int MODE, typename T>
struct Cfg {
  static constexpr bool A32 = MODE == DX || sizeof(T) == 4;  // A in float32: hi and lo parts
  static constexpr int TILE_A = BM * BK * (A32 ? 4 : 2);
  static constexpr int STAGE = TILE_A + 2 * TILE_B;
  static constexpr int A_STAGE = A32 ? 2 * BK : BK;  // tensor-memory columns
  static constexpr int STAGES = A32 ? 3 : 4;
  static constexpr int A_RING = A_COLS / A_STAGE;
  static constexpr int SMEM = STAGES * STAGE + EPI_BYTES + BAR_BYTES + 1024;
  static_assert(A_COLS + NACC * BN <= 512, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory per CTA");
};

struct Args {
  int64_t items;
  int L, ranks, comps;
  int N;                  // output columns of a component: H (FWD, PRE), C (DX)
  int nk, kg, nu;         // 32-wide slabs of a segment, slabs per unit, units per segment
  int n_ct, tiles, main_tiles, per_comp;
  int act;
  const void* bias;       // T, or null
  const float* act_scale;
  int* counter;           // work list, zeroed before the launch
  int* status;
};

struct Maps {
  CUtensorMap a;   // x (FWD, PRE) or dv (DX): (channel, row, component)
  CUtensorMap a2;  // dz (DX): (channel, row, rank)
  CUtensorMap b;   // split weights: (k, output channel, matrix)
  CUtensorMap o;   // y, dv or dx, 32 x 32 boxes
  CUtensorMap g;   // g (PRE)
  CUtensorMap o2;  // dz (PRE)
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

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float* f);
template <>
__device__ __forceinline__ void tmem_ld<32>(uint32_t taddr, float* f) {
  uint32_t v[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < 32; ++c) f[c] = __uint_as_float(v[c]);
}
template <>
__device__ __forceinline__ void tmem_ld<16>(uint32_t taddr, float* f) {
  uint32_t v[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < 16; ++c) f[c] = __uint_as_float(v[c]);
}

// 32 floats -> the tf32 parts of a lane's 32 columns
template <bool LO>
__device__ __forceinline__ void store_parts(uint32_t ta, const float* x) {
  uint32_t p[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) p[e] = __float_as_uint(round_tf32(x[e]));
  tmem_st32(ta, p);
  if (LO) {
#pragma unroll
    for (int e = 0; e < 32; ++e) p[e] = __float_as_uint(round_tf32(x[e] - round_tf32(x[e])));
    tmem_st32(ta + BK, p);
  }
}

// wait_parity for a whole warp: one answer, so that no lane leaves a collective alone
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return __all_sync(0xffffffffu, wait_parity(bar, parity, abort_flag, status));
}

__device__ __forceinline__ void drain_bar(uint32_t bar, uint32_t parity) {
  for (long long it = 0; it < WAIT_LIMIT; ++it)
    if (test_parity(bar, parity)) break;
}

// A warp's 32 x 32 staging box: row r in 32 * sizeof(E) bytes, its 16-byte chunks swizzled as
// TMA does for that row width (128 bytes: c ^ (r & 7); 64 bytes: c ^ ((r >> 1) & 3)).
template <typename E>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return sizeof(E) == 4 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// one row of 32 floats into the staging box
template <typename E>
__device__ __forceinline__ void put_row(uint8_t* buf, int r, const float* f) {
  constexpr int PER = 16 / sizeof(E);
#pragma unroll
  for (int c = 0; c < 32 / PER; ++c) {
    Pack<E, PER> p;
#pragma unroll
    for (int k = 0; k < PER; ++k) p.set(k, Io<E>::put(f[c * PER + k]));
    p.store(reinterpret_cast<E*>(buf + chunk_at<E>(r, c)));
  }
}

#define FC_SETMAXNREG_DEC(n) asm volatile("setmaxnreg.dec.sync.aligned.u32 " #n ";")
#define FC_SETMAXNREG_INC(n) asm volatile("setmaxnreg.inc.sync.aligned.u32 " #n ";")

template <int MODE, typename T>
__global__ void __launch_bounds__(THREADS, 1) gated_tc_kernel(const __grid_constant__ Maps mp, const Args a) {
  using C = Cfg<MODE, T>;
  constexpr int S = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + S * C::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + EPI_BYTES);
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

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
      init(&split[s], 128);
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
    if (!wait_warp(smem_u32(&sched_full[s]), (uint32_t)((q / SCHED) & 1), abort_flag, a.status)) return -1;
    const int it = *reinterpret_cast<volatile int*>(&sched[s]);
    __syncwarp();
    if (lane == 0) arrive(smem_u32(&sched_empty[s]));
    return it;
  };
  auto segments = [&](const Item& w) { return MODE == DX && w.k0 == 0 ? a.ranks + 1 : 1; };
  auto substeps = [&](const Item& w) { return MODE == DX ? 1 : 1 + w.nm; };

  if (warp < 4) {
    FC_SETMAXNREG_DEC(48);
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      constexpr uint32_t bytes = C::TILE_A + 2 * TILE_B;
      int next = (int)blockIdx.x;
      int64_t g = 0;
      bool ok = true;
      for (int q = 0; ok; ++q) {
        const int s4 = q % SCHED;
        if (q >= SCHED &&
            !wait_parity(smem_u32(&sched_empty[s4]), (uint32_t)((q / SCHED - 1) & 1), abort_flag, a.status))
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
              const int s = (int)(g % S);
              if (g >= S && !wait_parity(smem_u32(&empty[s]), (uint32_t)(((g / S) - 1) & 1), abort_flag, a.status)) {
                ok = false;
                break;
              }
              uint8_t* st = smem + s * C::STAGE;
              const uint32_t fb = smem_u32(&full[s]);
              arrive_tx(fb, bytes);
              tma_load_3d(smem_u32(st), ma, kt * BK, w.tile * BM, z, fb);
              tma_load_3d(smem_u32(st + C::TILE_A), &mp.b, kt * BK, w.ct * BN, mat, fb);
              tma_load_3d(smem_u32(st + C::TILE_A + TILE_B), &mp.b, kt * BK, w.ct * BN, mat + 2 * a.ranks, fb);
            }
          }
      }
      // the last load issued into every stage must have landed before the CTA exits
      for (int s = 0; s < S; ++s) {
        const int64_t uses = g > s ? (g - 1 - s) / S + 1 : 0;
        if (uses > 0) drain_bar(smem_u32(&full[s]), (uint32_t)((uses - 1) & 1));
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------------- MMA issue
      int64_t g = 0, u = 0;
      bool ok = true;
      for (int q = 0; ok; ++q) {
        const int s4 = q % SCHED;
        if (!wait_parity(smem_u32(&sched_full[s4]), (uint32_t)((q / SCHED) & 1), abort_flag, a.status)) break;
        const int it = *reinterpret_cast<volatile int*>(&sched[s4]);
        arrive(smem_u32(&sched_empty[s4]));
        if (it < 0) break;
        const Item w = item_of<MODE>(a, it);
        const int passes = substeps(w) * segments(w);
        for (int p = 0; p < passes && ok; ++p)
          for (int j = 0; j < a.nu && ok; ++j, ++u) {
            const int b = (int)(u % NACC);
            const int64_t v = u / NACC;
            if (v >= 1 && !wait_parity(smem_u32(&acc_empty[b]), (uint32_t)((v - 1) & 1), abort_flag, a.status)) {
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;");
            const uint32_t d = tmem + (uint32_t)(A_COLS + b * BN);
            const int k_end = min(a.nk, (j + 1) * a.kg);
            for (int kt = j * a.kg; kt < k_end; ++kt, ++g) {
              const int s = (int)(g % S);
              if (!wait_parity(smem_u32(&split[s]), (uint32_t)((g / S) & 1), abort_flag, a.status)) {
                ok = false;
                break;
              }
              asm volatile("tcgen05.fence::after_thread_sync;");
              uint8_t* st = smem + s * C::STAGE;
              const uint64_t dbh = make_desc(smem_u32(st + C::TILE_A));
              const uint64_t dbl = make_desc(smem_u32(st + C::TILE_A + TILE_B));
              const int slot = (int)(g % C::A_RING);
              const uint32_t tah = tmem + (uint32_t)(slot * C::A_STAGE), tal = tah + (uint32_t)BK;
#pragma unroll
              for (int kk = 0; kk < BK / 8; ++kk) {
                const uint64_t off = (uint64_t)((kk * 32) >> 4);
                mma_ta<BN>(d, tah + kk * 8, dbl + off, (kt > j * a.kg || kk > 0) ? 1u : 0u);
                if (C::A32) mma_ta<BN>(d, tal + kk * 8, dbh + off, 1u);
              }
#pragma unroll
              for (int kk = 0; kk < BK / 8; ++kk) mma_ta<BN>(d, tah + kk * 8, dbh + (uint64_t)((kk * 32) >> 4), 1u);
              // the stage and the A slot are free once these MMAs have completed
              commit(smem_u32(&empty[s]));
              commit(smem_u32(&a_free[slot]));
            }
            if (ok) commit(smem_u32(&acc_full[b]));
          }
      }
      commit(smem_u32(drain));  // every MMA completes before tensor memory is freed
      drain_bar(smem_u32(drain), 0);
    }
  } else if (warp < 8) {
    FC_SETMAXNREG_DEC(96);
    // ------------------------------------------------------------------ splitters
    const int r = (warp & 3) * 32 + lane;  // row of the slab, lane of tensor memory
    int64_t g = 0;
    bool ok = true;
    for (int q = 0; ok; ++q) {
      const int it = next_item(q);
      if (it < 0) break;
      const Item w = item_of<MODE>(a, it);
      const int64_t end = g + (int64_t)substeps(w) * segments(w) * a.nk;
      for (; g < end; ++g) {
        const int s = (int)(g % S);
        if (!wait_warp(smem_u32(&full[s]), (uint32_t)((g / S) & 1), abort_flag, a.status)) {
          ok = false;
          break;
        }
        const int slot = (int)(g % C::A_RING);
        if (g >= C::A_RING &&
            !wait_warp(smem_u32(&a_free[slot]), (uint32_t)((g / C::A_RING - 1) & 1), abort_flag, a.status)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint8_t* slab = smem + s * C::STAGE;
        const uint32_t ta = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(slot * C::A_STAGE);
        if constexpr (C::A32) {
          float x[32];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<float4*>(&x[4 * c]) = *reinterpret_cast<const float4*>(slab + chunk_at<float>(r, c));
          store_parts<true>(ta, x);
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
        arrive(smem_u32(&split[s]));
      }
    }
  } else {
    FC_SETMAXNREG_INC(184);
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = (warp - 8) >> 2;
    uint8_t* stage0 = epi + (warp - 8) * 2 * EPI_BUF;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(A_COLS + half * 64);
    const float sa = MODE == DX ? 0.f : __ldg(a.act_scale);
    int64_t u = 0;
    int nbuf = 0;
    uint32_t aux_phase = 0;
    bool ok = true;
    // units u .. u+count-1 are complete (their accumulators are read and then given back)
    auto wait_unit = [&](int64_t v) {
      const bool done = wait_warp(smem_u32(&acc_full[v % NACC]), (uint32_t)((v / NACC) & 1), abort_flag, a.status);
      asm volatile("tcgen05.fence::after_thread_sync;");
      return done;
    };
    auto free_unit = [&](int64_t v) {
      asm volatile("tcgen05.fence::before_thread_sync;");
      __syncwarp();
      if (lane == 0) arrive(smem_u32(&acc_empty[v % NACC]));
    };
    // 32 columns of this warp's rows from the staging buffer to memory
    auto send = [&](const CUtensorMap* map, uint8_t* buf, int col, int row, int z) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(map, smem_u32(buf), col, row, z);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
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
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            __syncwarp();
            uint8_t* buf = stage0 + nbuf * EPI_BUF;
            put_row<T>(buf, lane, acc + cb * 32);
            send(&mp.o, buf, col0 + cb * 32, row0, w.k0);
            nbuf ^= 1;
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
          for (int c = 0; c < 64; ++c) z[c] = sa * gated_act<float>(a.act, z[c]);
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
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                __syncwarp();
                uint8_t* buf = stage0 + nbuf * EPI_BUF;
                put_row<T>(buf, lane, acc + cb * 32);
                send(&mp.o, buf, col0 + cb * 32, row0, w.k0 + m);
                nbuf ^= 1;
              }
          }
        } else {
          float sum[64];  // over m of g v
#pragma unroll
          for (int c = 0; c < 64; ++c) sum[c] = 0.f;
          for (int m = 0; m < w.nm && ok; ++m) {
            // the output gradient's boxes come in while the products are computed
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            if (lane == 0)
              for (int cb = 0; cb < nch; ++cb) {
                const uint32_t ab = smem_u32(&aux[(warp - 8) * 2 + cb]);
                arrive_tx(ab, 32 * 32 * sizeof(T));
                tma_load_3d(smem_u32(stage0 + cb * EPI_BUF), &mp.g, col0 + cb * 32, row0, w.k0 + m, ab);
              }
            for (int j = 0; j < a.nu; ++j)
              if (!wait_unit(u + j)) ok = false;
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
              if (cb < nch) {
                const uint32_t ab = smem_u32(&aux[(warp - 8) * 2 + cb]);
                const uint32_t par = (aux_phase >> cb) & 1u;
                aux_phase ^= 1u << cb;
                if (!wait_warp(ab, par, abort_flag, a.status)) {
                  drain_bar(ab, par);  // the copy may still land: let it, before the buffer goes
                  __syncwarp();
                  ok = false;
                }
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
                  tmem_ld<16>(lane_base + (uint32_t)((u % NACC) * BN + cb * 32 + h * 16), v);
                  for (int j = 1; j < a.nu; ++j) {
                    float v2[16];
                    tmem_ld<16>(lane_base + (uint32_t)(((u + j) % NACC) * BN + cb * 32 + h * 16), v2);
#pragma unroll
                    for (int c = 0; c < 16; ++c) v[c] += v2[c];
                  }
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
                      o[e] = gv[e] * (sa * gated_act<float>(a.act, z[c]));
                    }
                    *at = make_float4(o[0], o[1], o[2], o[3]);
                  }
                }
                send(&mp.o, buf, col0 + cb * 32, row0, w.k0 + m);
              }
            for (int j = 0; j < a.nu; ++j, ++u) free_unit(u);
          }
          if (!ok) break;
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int cb = 0; cb < 2; ++cb)
            if (cb < nch) {
#pragma unroll
              for (int c = 0; c < 32; ++c) sum[cb * 32 + c] *= sa * gated_dact<float>(a.act, z[cb * 32 + c]);
              uint8_t* buf = stage0 + cb * EPI_BUF;
              put_row<float>(buf, lane, sum + cb * 32);
              send(&mp.o2, buf, col0 + cb * 32, row0, w.l);
            }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ---------------------------------------------------------------------------- weight gradients

// Matrices 0 .. ranks-1: dWv_l (reduction over the 2l+1 components of n rows), ranks .. 2
// ranks - 1: dWg_l (n rows). Each is cut into 128 x 128 output tiles ("jobs"), a job's
// reduction into 32-row slabs; all slabs of all jobs form one line that the CTAs share out
// equally. CTA i's part of job j has the partial matrix i + j of the workspace.
struct WArgs {
  int ranks, H, Cn;
  int n_ht, n_ct;
  int64_t blocks;      // 32-row blocks
  int64_t width[8];    // slabs per job of a matrix
  int skip;            // bit per matrix that is not wanted: its slabs keep their place on the
                       // line, so what is wanted does not depend on what else is
  int64_t total;       // slabs in all
  int ctas;
  float* part;         // partial matrices, 128 x 128 each
  float* bias_part;    // partial bias gradients, 128 each (ct = 0 jobs of the gates), or null
  int* status;
};

struct WMaps {
  CUtensorMap dv, dz, x;  // (channel, row, component / rank), boxes of 128 channels x 32 rows
};

struct Job {
  int mat, ht, ct;
  int64_t index;        // job number
  int64_t first, last;  // its slabs on the line
};

__host__ __device__ inline Job job_at(const WArgs& a, int64_t slab) {
  Job j{0, 0, 0, 0, 0, 0};
  const int tiles = a.n_ht * a.n_ct;
  int64_t at = 0;
  for (int mat = 0; mat < 2 * a.ranks; ++mat) {
    const int64_t len = a.width[mat] * tiles;
    if (slab < at + len) {
      const int64_t t = (slab - at) / a.width[mat];
      j.mat = mat;
      j.ht = (int)(t / a.n_ct);
      j.ct = (int)(t - (int64_t)j.ht * a.n_ct);
      j.index = (int64_t)mat * tiles + t;
      j.first = at + t * a.width[mat];
      j.last = j.first + a.width[mat];
      return j;
    }
    at += len;
  }
  return j;
}
__host__ __device__ inline int64_t cta_begin(const WArgs& a, int64_t i) { return i * a.total / a.ctas; }

template <typename T>
struct WCfg {
  static constexpr bool X32 = sizeof(T) == 4;
  static constexpr int TILE_D = 32 * BM * 4;         // raw dv / dz slab
  static constexpr int TILE_X = 32 * BN * sizeof(T); // raw x slab
  static constexpr int STAGE = TILE_D + TILE_X + (X32 ? 2 : 1) * TILE_B;
  static constexpr int STAGES = X32 ? 3 : 4;
  static constexpr int SMEM = STAGES * STAGE + BAR_BYTES + 1024;
  static constexpr int NACC = 2, A_COLS = STAGES * 2 * BK;  // every stage has its A slot
  static_assert(A_COLS + NACC * BN <= 512, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory per CTA");
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 1) wgrad_kernel(const __grid_constant__ WMaps mp, const WArgs a) {
  using C = WCfg<T>;
  constexpr int S = C::STAGES, NACC = C::NACC, A_COLS = C::A_COLS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * C::STAGE);
  uint64_t* split = full + S;
  uint64_t* empty = split + S;
  uint64_t* acc_full = empty + S;
  uint64_t* acc_empty = acc_full + NACC;
  uint64_t* drain = acc_empty + NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // within a stage: the K-major B parts first (1024-byte aligned), then the raw slabs
  constexpr int D_OFF = (C::X32 ? 2 : 1) * TILE_B, X_OFF = D_OFF + C::TILE_D;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
      init(&split[s], 256);
      init(&empty[s], 1);
    }
    for (int b = 0; b < NACC; ++b) {
      init(&acc_full[b], 1);
      init(&acc_empty[b], 4);
    }
    init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;
  const int64_t begin = cta_begin(a, blockIdx.x), end = cta_begin(a, blockIdx.x + 1);

  if (warp < 4) {
    FC_SETMAXNREG_DEC(56);
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      int64_t g = 0;
      bool ok = true;
      for (int64_t p = begin; p < end && ok;) {
        const Job j = job_at(a, p);
        const bool gates = j.mat >= a.ranks;
        const int l = gates ? j.mat - a.ranks : j.mat, w = gates ? 1 : 2 * l + 1;
        const int64_t stop = min(end, j.last);
        if (a.skip >> j.mat & 1) {
          p = stop;
          continue;
        }
        for (; p < stop; ++p, ++g) {
          const int s = (int)(g % S);
          if (g >= S && !wait_parity(smem_u32(&empty[s]), (uint32_t)(((g / S) - 1) & 1), abort_flag, a.status)) {
            ok = false;
            break;
          }
          // rows of a node block one component after the other: they share DRAM pages
          const int64_t r = p - j.first, nb = r / w;
          const int m = (int)(r - nb * w);
          uint8_t* st = smem + s * C::STAGE;
          const uint32_t fb = smem_u32(&full[s]);
          arrive_tx(fb, C::TILE_D + C::TILE_X);
          tma_load_3d(smem_u32(st + D_OFF), gates ? &mp.dz : &mp.dv, j.ht * BM, (int)(nb * 32), gates ? l : l * l + m,
                      fb);
          tma_load_3d(smem_u32(st + X_OFF), &mp.x, j.ct * BN, (int)(nb * 32), gates ? 0 : l * l + m, fb);
        }
      }
      for (int s = 0; s < S; ++s) {
        const int64_t uses = g > s ? (g - 1 - s) / S + 1 : 0;
        if (uses > 0) drain_bar(smem_u32(&full[s]), (uint32_t)((uses - 1) & 1));
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------------- MMA issue
      int64_t g = 0, u = 0;
      bool ok = true;
      for (int64_t p = begin; p < end && ok;) {
        const Job j = job_at(a, p);
        const int64_t stop = min(end, j.last);
        if (a.skip >> j.mat & 1) p = stop;
        while (p < stop && ok) {
          const int b = (int)(u % NACC);
          const int64_t v = u / NACC;
          if (v >= 1 && !wait_parity(smem_u32(&acc_empty[b]), (uint32_t)((v - 1) & 1), abort_flag, a.status)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;");
          const uint32_t d = tmem + (uint32_t)(A_COLS + b * BN);
          const int64_t unit = min(stop, p + KG);
          bool fresh = true;
          for (; p < unit; ++p, ++g) {
            const int s = (int)(g % S);
            if (!wait_parity(smem_u32(&split[s]), (uint32_t)((g / S) & 1), abort_flag, a.status)) {
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;");
            uint8_t* st = smem + s * C::STAGE;
            const uint64_t dbh = make_desc(smem_u32(st)), dbl = make_desc(smem_u32(st + TILE_B));
            const uint32_t tah = tmem + (uint32_t)(s * 2 * BK), tal = tah + (uint32_t)BK;
#pragma unroll
            for (int kk = 0; kk < BK / 8; ++kk) {
              const uint64_t off = (uint64_t)((kk * 32) >> 4);
              mma_ta<BN>(d, tal + kk * 8, dbh + off, fresh && kk == 0 ? 0u : 1u);
              if (C::X32) mma_ta<BN>(d, tah + kk * 8, dbl + off, 1u);
            }
#pragma unroll
            for (int kk = 0; kk < BK / 8; ++kk) mma_ta<BN>(d, tah + kk * 8, dbh + (uint64_t)((kk * 32) >> 4), 1u);
            fresh = false;
            commit(smem_u32(&empty[s]));
          }
          if (ok) {
            commit(smem_u32(&acc_full[b]));
            ++u;
          }
        }
      }
      commit(smem_u32(drain));
      drain_bar(smem_u32(drain), 0);
    }
  } else if (warp < 12) {
    FC_SETMAXNREG_DEC(112);
    // ------------------------------------------------------------------ splitters
    const bool of_d = warp < 8;               // dv / dz into tensor memory, or x into K-major rows
    const int c = (warp & 3) * 32 + lane;     // channel: lane of tensor memory, or row of the B tile
    int64_t g = 0;
    bool ok = true;
    for (int64_t p = begin; p < end && ok;) {
      const Job j = job_at(a, p);
      const int64_t stop = min(end, j.last);
      if (a.skip >> j.mat & 1) {
        p = stop;
        continue;
      }
      const bool bias = of_d && a.bias_part && j.mat >= a.ranks && j.ct == 0;
      float bsum = 0.f;
      for (; p < stop; ++p, ++g) {
        const int s = (int)(g % S);
        if (!wait_warp(smem_u32(&full[s]), (uint32_t)((g / S) & 1), abort_flag, a.status)) {
          ok = false;
          break;
        }
        uint8_t* st = smem + s * C::STAGE;
        float x[32];
        if (of_d) {
          const float* raw = reinterpret_cast<const float*>(st + D_OFF) + c;
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = raw[k * BM];
          if (bias) {
            float t = 0.f;  // a slab's sum first: fewer roundings against the running sum
#pragma unroll
            for (int k = 0; k < 32; ++k) t += x[k];
            bsum += t;
          }
          store_parts<true>(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(s * 2 * BK), x);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        } else {
          const T* raw = reinterpret_cast<const T*>(st + X_OFF) + c;
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = Io<T>::get(raw[k * BN]);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = C::X32 ? round_tf32(x[4 * q + e]) : x[4 * q + e];
            *reinterpret_cast<float4*>(st + chunk_at<float>(c, q)) = make_float4(h[0], h[1], h[2], h[3]);
            if (C::X32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) h[e] = round_tf32(x[4 * q + e] - h[e]);
              *reinterpret_cast<float4*>(st + TILE_B + chunk_at<float>(c, q)) = make_float4(h[0], h[1], h[2], h[3]);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        arrive(smem_u32(&split[s]));
      }
      if (bias && ok) a.bias_part[(blockIdx.x + j.index) * BM + c] = bsum;
    }
  } else {
    FC_SETMAXNREG_INC(216);
    // ------------------------------------------------------------------ epilogue: unit sums
    const int quarter = warp & 3;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)A_COLS;
    int64_t u = 0;
    bool ok = true;
    for (int64_t p = begin; p < end && ok;) {
      const Job j = job_at(a, p);
      const int64_t stop = min(end, j.last);
      if (a.skip >> j.mat & 1) {
        p = stop;
        continue;
      }
      float acc[BN];
#pragma unroll
      for (int c = 0; c < BN; ++c) acc[c] = 0.f;
      for (; p < stop; p += KG, ++u) {
        const int b = (int)(u % NACC);
        if (!wait_warp(smem_u32(&acc_full[b]), (uint32_t)((u / NACC) & 1), abort_flag, a.status)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
        for (int cb = 0; cb < BN / 32; ++cb) {
          float f[32];
          tmem_ld<32>(lane_base + (uint32_t)(b * BN + cb * 32), f);
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[cb * 32 + c] += f[c];
        }
        asm volatile("tcgen05.fence::before_thread_sync;");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&acc_empty[b]));
      }
      p = stop;
      if (!ok) break;
      float4* out = reinterpret_cast<float4*>(a.part + ((blockIdx.x + j.index) * BM + quarter * 32 + lane) * BN);
#pragma unroll
      for (int c = 0; c < BN / 4; ++c)
        out[c] = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

struct WOut {
  void* w[8];     // gradient of each matrix (gates: rows l H .. of one matrix), or null
  void* bias;     // ((ranks) H) or null
  const float* scales;
};

// Partial matrices added in the order of the CTAs. One block per 8 rows of a job's tile; the
// bias by the blocks of the ct = 0 gate jobs.
template <typename T>
__global__ void __launch_bounds__(256) wgrad_sum_kernel(const WArgs a, const WOut o) {
  const int tiles = a.n_ht * a.n_ct;
  const int64_t job = blockIdx.x / (BM / 8);
  const int row = (int)(blockIdx.x % (BM / 8)) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int mat = (int)(job / tiles), t = (int)(job % tiles);
  const int64_t width = a.width[mat];
  const int h = (t / a.n_ct) * BM + row, c = (t % a.n_ct) * BN + lane * 4;
  const bool gates = mat >= a.ranks;
  const bool bias = gates && o.bias && t % a.n_ct == 0 && (threadIdx.x & 31) == 0;
  if (h >= a.H || (!o.w[mat] && !bias)) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float bsum = 0.f;
  if (width > 0 && a.total > 0) {
    int64_t first = 0;
    for (int m = 0; m < mat; ++m) first += a.width[m] * tiles;
    first += t * width;
    int64_t i0 = first * a.ctas / a.total;
    while (i0 > 0 && cta_begin(a, i0) > first) --i0;
    while (i0 + 1 < a.ctas && cta_begin(a, i0 + 1) <= first) ++i0;
#pragma unroll 4
    for (int64_t i = i0; i < a.ctas; ++i) {
      if (cta_begin(a, i) >= first + width) break;
      const float4 v = *reinterpret_cast<const float4*>(a.part + ((i + job) * BM + row) * BN + lane * 4);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      if (bias) bsum += a.bias_part[(i + job) * BM + row];
    }
  }
  const int l = gates ? mat - a.ranks : mat;
  const float sc = o.scales[gates ? a.ranks : l];
  if (o.w[mat]) {
    T* out = (T*)o.w[mat] + ((int64_t)(gates ? l * a.H : 0) + h) * a.Cn + c;
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < a.Cn) out[e] = Io<T>::put(sc * v[e]);
  }
  if (bias) ((T*)o.bias)[(int64_t)l * a.H + h] = Io<T>::put(bsum);
}

// ---------------------------------------------------------------------------- operand layouts

// Scaled weights as tf32 hi | lo parts: matrix q (values 0 .. ranks-1, then gates) at q, its
// low part 2 ranks matrices behind; (out, k) rows of kp elements, zero behind K. fwd: out =
// hidden, k = input channel; dx: the transpose. Also zeroes the work lists' counters.
struct PrepArgs {
  GatedArgs g;
  float* fwd;  // or null
  float* dx;   // or null
  int* counters;
};

template <typename T>
__global__ void __launch_bounds__(256) prep_kernel(const PrepArgs p) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 4) p.counters[threadIdx.x] = 0;
  const int ranks = p.g.L + 1, q = blockIdx.y, l = q < ranks ? q : q - ranks, C = p.g.C, H = p.g.H;
  const T* w = q < ranks ? (const T*)p.g.wv[l] : (const T*)p.g.wg + (int64_t)l * H * C;
  const float sc = ((const float*)p.g.scales)[q < ranks ? l : ranks];
  const int cp = (C + 3) & ~3, hp = (H + 3) & ~3;
  const int64_t nf = p.fwd ? (int64_t)H * cp : 0, nd = p.dx ? (int64_t)C * hp : 0;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < nf + nd; i += (int64_t)gridDim.x * 256) {
    const bool f = i < nf;
    const int64_t e = f ? i : i - nf, size = f ? nf : nd;
    const int kp = f ? cp : hp, r = (int)(e / kp), k = (int)(e - (int64_t)r * kp);
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

// (channel, row, component) map of a tensor of rows [comps][ld]; box_c channels x box_r rows.
// swizzled: 32-channel boxes with the 128- or 64-byte swizzle of their row width.
template <typename E>
static bool encode_rows(CUtensorMap* map, const void* base, int64_t channels, int64_t rows, int64_t comps, int64_t ld,
                        int box_c, int box_r) {
  const cuuint64_t dims[3] = {(cuuint64_t)channels, (cuuint64_t)rows, (cuuint64_t)comps};
  const cuuint64_t strides[2] = {(cuuint64_t)(comps * ld) * sizeof(E), (cuuint64_t)ld * sizeof(E)};
  const cuuint32_t box[3] = {(cuuint32_t)box_c, (cuuint32_t)box_r, 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return encode_fn()(map, sizeof(E) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     const_cast<void*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     box_c != 32        ? CU_TENSOR_MAP_SWIZZLE_NONE
                     : sizeof(E) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B
                                      : CU_TENSOR_MAP_SWIZZLE_64B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool encode_weights(CUtensorMap* map, const float* base, int kp, int out, int mats) {
  const cuuint64_t dims[3] = {(cuuint64_t)kp, (cuuint64_t)out, (cuuint64_t)mats};
  const cuuint64_t strides[2] = {(cuuint64_t)kp * 4, (cuuint64_t)kp * out * 4};
  const cuuint32_t box[3] = {32, BN, 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(base), dims, strides, box, unit,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return sms[dev];
}

// Shared-memory size, and the registers that setmaxnreg shares out: the block must be launched
// with 128 per thread (its roles' shares add up to exactly that).
struct Ready {
  bool done[64] = {};
};
template <typename K>
static int ready(K kernel, int smem, Ready& r) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FC_ERR_LAUNCH;
  if (r.done[dev]) return 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return FC_ERR_LAUNCH;
  cudaFuncAttributes at;
  if (cudaFuncGetAttributes(&at, kernel) != cudaSuccess) return FC_ERR_LAUNCH;
  if (at.numRegs != 128) return FC_ERR_UNSUPPORTED;
  r.done[dev] = true;
  return 0;
}

template <int MODE, typename T>
static int run_products(const Maps& mp, const Args& args, cudaStream_t s) {
  constexpr int smem = Cfg<MODE, T>::SMEM;
  static Ready state;
  if (int rc = ready(gated_tc_kernel<MODE, T>, smem, state)) return rc;
  const int grid = (int)std::min<int64_t>(args.items, sm_count());
  gated_tc_kernel<MODE, T><<<grid, THREADS, smem, s>>>(mp, args);
  return fc_check_launch();
}

// Layout of the workspace (bytes), the same for the size query and the call.
struct Ws {
  int64_t counters, fwd, dx, dv, dz, part, bias, x, y, gx, bytes;
};

static Ws layout(int L, int C, int H, int64_t n, int esize, bool backward, int sms) {
  const int64_t ranks = L + 1, comps = ranks * ranks, per = 16 / esize;
  const int64_t cp = (C + 3) / 4 * 4, hp = (H + 3) / 4 * 4;
  const int64_t ce = (C + per - 1) / per * per, he = (H + per - 1) / per * per;
  Ws w{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += (bytes + 127) / 128 * 128;
    return p;
  };
  w.counters = take(16);
  w.fwd = take(4 * ranks * H * cp * 4);
  if (backward) {
    const int64_t jobs = 2 * ranks * ((H + BM - 1) / BM) * ((C + BN - 1) / BN);
    w.dx = take(4 * ranks * C * hp * 4);
    w.dv = take(n * comps * hp * 4);
    w.dz = take(n * ranks * hp * 4);
    w.part = take((sms + jobs) * BM * BN * 4);
    w.bias = take((sms + jobs) * BM * 4);
  }
  // copies with 16-byte rows, used where the caller's rows are not (or are misaligned)
  w.x = take(n * comps * ce * esize);
  w.y = take(n * comps * he * esize);  // y, or the output gradient
  if (backward) w.gx = take(n * comps * ce * esize);
  w.bytes = at;
  return w;
}

// A tensor as TMA can address it: itself, or a copy with padded rows.
template <typename T>
struct Rows {
  const T* p;
  int64_t ld;
  bool copied;
};

template <typename T>
static Rows<T> rows_of(const void* p, int width, void* room) {
  constexpr int per = 16 / sizeof(T);
  if (width % per == 0 && !(reinterpret_cast<uintptr_t>(p) & 15)) return {(const T*)p, width, false};
  return {(const T*)room, (width + per - 1) / per * per, true};
}

template <typename T>
static int repitch(const T* src, int64_t src_ld, T* dst, int64_t dst_ld, int width, int64_t rows, cudaStream_t s) {
  const int64_t b = (rows * width + 255) / 256;
  repitch_kernel<T><<<(unsigned)std::min<int64_t>(b, 148 * 32), 256, 0, s>>>(src, src_ld, dst, dst_ld, width, rows);
  return fc_check_launch();
}

static Args product_args(const GatedArgs& g, int N, int K, int n_items_cols, int mode, int sms) {
  Args a{};
  a.L = g.L;
  a.ranks = g.L + 1;
  a.comps = a.ranks * a.ranks;
  a.N = N;
  a.nk = (K + BK - 1) / BK;
  // PRE holds a component's accumulators until its epilogue is done, so all its units have to
  // fit the ring; the others add units of 64 products in registers
  a.kg = mode == PRE ? std::max(KG, (a.nk + NACC - 1) / NACC) : KG;
  a.nu = (a.nk + a.kg - 1) / a.kg;
  a.n_ct = n_items_cols;
  a.tiles = (int)((g.n + BM - 1) / BM);
  // with fewer (tile, rank) groups than SMs the components are items of their own (the gate is
  // computed again for each); PRE needs a rank's components together
  const int64_t groups = (int64_t)a.tiles * a.ranks * a.n_ct;
  a.per_comp = mode == DX || (mode == FWD && groups < sms);
  a.items = (int64_t)a.tiles * a.n_ct * (a.per_comp ? a.comps : a.ranks);
  const int tail = (2 * sms + a.ranks * a.n_ct - 1) / (a.ranks * a.n_ct);
  a.main_tiles = std::max(0, a.tiles - tail);
  a.act = g.act;
  a.bias = g.bias;
  a.act_scale = (const float*)g.scales + a.ranks + 1;
  a.status = g.status;
  return a;
}

template <typename T>
static int run_prep(const GatedArgs& g, float* fwd, float* dx, int* counters, cudaStream_t s) {
  const int64_t cp = (g.C + 3) & ~3, hp = (g.H + 3) & ~3;
  const int64_t each = (fwd ? g.H * cp : 0) + (dx ? g.C * hp : 0);
  const PrepArgs p{g, fwd, dx, counters};
  prep_kernel<T><<<dim3((unsigned)std::min<int64_t>((each + 255) / 256, 256), 2 * (g.L + 1)), 256, 0, s>>>(p);
  return fc_check_launch();
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
  float* weights = (float*)(ws + w.fwd);
  if (int rc = run_prep<T>(a, weights, nullptr, counters, s)) return rc;
  Args args = product_args(a, a.H, a.C, (a.H + BN - 1) / BN, FWD, sms);
  args.counter = counters;
  Maps mp;
  if (!encode_rows<T>(&mp.a, x.p, a.C, a.n, comps, x.ld, BK, BM) ||
      !encode_weights(&mp.b, weights, (a.C + 3) & ~3, a.H, 4 * ranks) ||
      !encode_rows<T>(&mp.o, y.p, a.H, a.n, comps, y.ld, 32, 32))
    return FC_ERR_UNSUPPORTED;
  mp.a2 = mp.g = mp.o2 = mp.o;  // not used
  if (int rc = run_products<FWD, T>(mp, args, s)) return rc;
  if (y.copied) return repitch<T>(y.p, y.ld, (T*)a.y, a.H, a.H, a.n * comps, s);
  return 0;
}

template <typename T>
int gated_tc_bwd(const GatedArgs& a, cudaStream_t s) {
  using namespace gtc;
  const int sms = sm_count();
  if (!sms || !encode_fn()) return FC_ERR_LAUNCH;
  const int ranks = a.L + 1, comps = ranks * ranks;
  const int64_t hp = (a.H + 3) / 4 * 4;
  const Ws w = layout(a.L, a.C, a.H, a.n, sizeof(T), true, sms);
  uint8_t* ws = (uint8_t*)a.ws;
  const Rows<T> x = rows_of<T>(a.x, a.C, ws + w.x), gy = rows_of<T>(a.gy, a.H, ws + w.y);
  int* counters = (int*)(ws + w.counters);
  float *fwd = (float*)(ws + w.fwd), *dx = (float*)(ws + w.dx), *dv = (float*)(ws + w.dv), *dz = (float*)(ws + w.dz);
  bool any = a.gwg || a.gbias;
  WArgs wa{};
  wa.ranks = ranks;
  wa.H = a.H;
  wa.Cn = a.C;
  wa.n_ht = (a.H + BM - 1) / BM;
  wa.n_ct = (a.C + BN - 1) / BN;
  wa.blocks = (a.n + 31) / 32;
  for (int l = 0; l < ranks; ++l) {
    wa.width[l] = wa.blocks * (2 * l + 1);
    wa.width[ranks + l] = wa.blocks;
    if (!a.gwv[l]) wa.skip |= 1 << l;
    if (!a.gwg && !a.gbias) wa.skip |= 1 << (ranks + l);
    wa.total += (wa.width[l] + wa.width[ranks + l]) * wa.n_ht * wa.n_ct;
    any = any || a.gwv[l];
  }
  wa.part = (float*)(ws + w.part);
  wa.bias_part = a.gbias ? (float*)(ws + w.bias) : nullptr;
  wa.status = a.status;
  if (a.n > 0) {
    if (x.copied)
      if (int rc = repitch<T>((const T*)a.x, a.C, const_cast<T*>(x.p), x.ld, a.C, a.n * comps, s)) return rc;
    if (gy.copied)
      if (int rc = repitch<T>((const T*)a.gy, a.H, const_cast<T*>(gy.p), gy.ld, a.H, a.n * comps, s)) return rc;
    if (int rc = run_prep<T>(a, fwd, a.gx ? dx : nullptr, counters, s)) return rc;
    Maps mp;
    if (!encode_rows<T>(&mp.a, x.p, a.C, a.n, comps, x.ld, BK, BM) ||
        !encode_weights(&mp.b, fwd, (a.C + 3) & ~3, a.H, 4 * ranks) ||
        !encode_rows<float>(&mp.o, dv, a.H, a.n, comps, hp, 32, 32) ||
        !encode_rows<T>(&mp.g, gy.p, a.H, a.n, comps, gy.ld, 32, 32) ||
        !encode_rows<float>(&mp.o2, dz, a.H, a.n, ranks, hp, 32, 32))
      return FC_ERR_UNSUPPORTED;
    mp.a2 = mp.o2;  // not used
    Args args = product_args(a, a.H, a.C, (a.H + BN - 1) / BN, PRE, sms);
    args.counter = counters;
    if (int rc = run_products<PRE, T>(mp, args, s)) return rc;
    if (a.gx) {
      const Rows<T> gx = rows_of<T>(a.gx, a.C, ws + w.gx);
      Maps md;
      if (!encode_rows<float>(&md.a, dv, a.H, a.n, comps, hp, BK, BM) ||
          !encode_rows<float>(&md.a2, dz, a.H, a.n, ranks, hp, BK, BM) ||
          !encode_weights(&md.b, dx, (int)hp, a.C, 4 * ranks) ||
          !encode_rows<T>(&md.o, gx.p, a.C, a.n, comps, gx.ld, 32, 32))
        return FC_ERR_UNSUPPORTED;
      md.g = md.o2 = md.o;  // not used
      Args dargs = product_args(a, a.C, a.H, (a.C + BN - 1) / BN, DX, sms);
      dargs.counter = counters + 1;
      if (int rc = run_products<DX, T>(md, dargs, s)) return rc;
      if (gx.copied)
        if (int rc = repitch<T>(gx.p, gx.ld, (T*)a.gx, a.C, a.C, a.n * comps, s)) return rc;
    }
  }
  if (!any) return 0;
  if (wa.total > 0) {
    // at least four slabs per CTA: a partial matrix costs 128 KB of traffic
    wa.ctas = (int)std::min<int64_t>(sms, (wa.total + 3) / 4);
    WMaps wm;
    if (!encode_rows<float>(&wm.dv, dv, a.H, a.n, comps, hp, BM, 32) ||
        !encode_rows<float>(&wm.dz, dz, a.H, a.n, ranks, hp, BM, 32) ||
        !encode_rows<T>(&wm.x, x.p, a.C, a.n, comps, x.ld, BN, 32))
      return FC_ERR_UNSUPPORTED;
    constexpr int smem = WCfg<T>::SMEM;
    static Ready state;
    if (int rc = ready(wgrad_kernel<T>, smem, state)) return rc;
    wgrad_kernel<T><<<wa.ctas, THREADS, smem, s>>>(wm, wa);
    if (int rc = fc_check_launch()) return rc;
  }
  WOut o{};
  for (int l = 0; l < ranks; ++l) {
    o.w[l] = a.gwv[l];
    o.w[ranks + l] = a.gwg;
  }
  o.bias = a.gbias;
  o.scales = (const float*)a.scales;
  if (wa.ctas == 0) wa.ctas = 1;
  wgrad_sum_kernel<T><<<(unsigned)(2 * ranks * wa.n_ht * wa.n_ct * (BM / 8)), 256, 0, s>>>(wa, o);
  return fc_check_launch();
}

template int gated_tc_fwd<float>(const GatedArgs&, cudaStream_t);
template int gated_tc_fwd<bf16_t>(const GatedArgs&, cudaStream_t);
template int gated_tc_bwd<float>(const GatedArgs&, cudaStream_t);
template int gated_tc_bwd<bf16_t>(const GatedArgs&, cudaStream_t);

}  // namespace fc

#endif  // FC_HOST_EMU
