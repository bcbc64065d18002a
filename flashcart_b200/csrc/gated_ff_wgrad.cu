// Weight gradients of the gated feed-forward block on the tensor cores.
//
// Matrices 0 .. ranks-1: dWv_l (reduction over the 2l+1 components of n rows), ranks .. 2
// ranks - 1: dWg_l (n rows). Each is cut into 128 x 128 output tiles ("jobs"), a job's
// reduction into 32-row slabs; all slabs of all jobs form one line that the CTAs share out
// equally. CTA i's part of job j has the partial matrix i + j of the workspace.
//
// The rows are the reduction, so both operands have to be transposed; the splitters do that on
// the way: a lane of tensor memory (dv, dz) or a row of the K-major B tile (x) is one channel,
// and a thread gathers its 32 rows' values from the row-major slab without bank conflicts.
// (bfloat16 operands need neither: wgrad_parts_kernel.)
//
// What bounds it: DRAM (dv, dz, x, and x_0 again for each rank's gates: 566 MB for 27,648 x 16
// rows of 128 -> 128 channels, 88 us at the copy rate). Measured there: 121 us (4.7 TB/s).
#include "gated_ff_tc.cuh"

#ifndef FC_HOST_EMU

#include <algorithm>

namespace fc {
namespace gtc {

constexpr int BN = 128, TILE_B = BN * BK * 4;
constexpr int PF = 6;  // slabs between the L2 prefetches and the copies
constexpr int KG = 2;  // slabs per accumulation unit (see gated_ff_tc.cu)

struct WArgs {
  int ranks, H, Cn;
  int n_ht, n_ct;
  int64_t blocks;      // row blocks: 32 rows (64: bfloat16 parts)
  int64_t width[8];    // slabs per job of a matrix
  int skip;            // bit per matrix that is not wanted: its slabs keep their place on the
                       // line, so what is wanted does not depend on what else is
  int64_t total;       // slabs in all
  int ctas;
  float* part;         // partial matrices, 128 x 128 each
  float* bias_part;    // partial bias gradients, 2 x 128 each (ct = 0 jobs of the gates), or null
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

constexpr int W_SPLIT0 = 4, W_EPI0 = 20, W_THREADS = 28 * 32;
constexpr int W_REGS = 72;  // per thread at launch: 896 x 72 = 128 x 40 + 512 x 56 + 256 x 120
constexpr int RAW = 4, OPS = 2;  // stages of raw slabs, slots of split operands; even: each belongs
                                 // to one splitter group, which so sees every phase of its barriers

template <typename T>
struct WCfg {
  static constexpr bool X32 = sizeof(T) == 4;
  static constexpr int TILE_D = 32 * BM * 4;          // raw dv / dz slab
  static constexpr int TILE_X = 32 * BN * sizeof(T);  // raw x slab
  static constexpr int OPERAND = (X32 ? 2 : 1) * TILE_B;
  static constexpr int SMEM = OPS * OPERAND + RAW * (TILE_D + TILE_X) + BAR_BYTES + 1024;
  static constexpr int NACC = 2, A_COLS = OPS * 2 * BK;
  static_assert(A_COLS + NACC * BN <= 512, "tensor memory");
  static_assert(SMEM <= 227 * 1024, "shared memory per CTA");
};

// Roles of the 28 warps: 0 TMA producer, 1 MMA issue, 4-19 splitters (two groups that take the
// slabs in turn, each four warps for dv / dz and four for x), 20-27 epilogue (unit sums, two
// warps per lane quarter). Measured before the second group, the raw ring of its own and the
// early answers: 130 us for 27,648 x 16 rows of 128 -> 128 channels, a slab waiting for its
// splitters most of the time.
template <typename T>
__global__ void __launch_bounds__(W_THREADS, 1) wgrad_kernel(const __grid_constant__ WMaps mp, const WArgs a) {
  using C = WCfg<T>;
  constexpr int NACC = C::NACC, A_COLS = C::A_COLS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* raw = smem + OPS * C::OPERAND;
  uint64_t* full = reinterpret_cast<uint64_t*>(raw + RAW * (C::TILE_D + C::TILE_X));
  uint64_t* empty = full + RAW;
  uint64_t* op_full = empty + RAW;
  uint64_t* op_free = op_full + OPS;
  uint64_t* acc_full = op_free + OPS;
  uint64_t* acc_empty = acc_full + NACC;
  uint64_t* drain = acc_empty + NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

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
    for (int s = 0; s < RAW; ++s) {
      init(&full[s], 1);
      init(&empty[s], 8);
    }
    for (int s = 0; s < OPS; ++s) {
      init(&op_full[s], 8);
      init(&op_free[s], 1);
    }
    for (int b = 0; b < NACC; ++b) {
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
  const int64_t begin = cta_begin(a, blockIdx.x), end = cta_begin(a, blockIdx.x + 1);

  if (warp < W_SPLIT0) {
    FC_SETMAXNREG_DEC(40);
    if (warp == 0 && elect_one()) {
      // ---------------------------------------------------------------- TMA producer
      int64_t g = 0;
      uint32_t s = 0, lap = 0;
      bool ok = true, free = true;  // (peeked: the next stage is free)
      for (int64_t p = begin; p < end && ok;) {
        const Job j = job_at(a, p);
        const bool gates = j.mat >= a.ranks;
        const int l = gates ? j.mat - a.ranks : j.mat, w = gates ? 1 : 2 * l + 1;
        const int64_t stop = min(end, j.last);
        if (a.skip >> j.mat & 1) {
          p = stop;
          continue;
        }
        const CUtensorMap* md = gates ? &mp.dz : &mp.dv;
        const int zd = gates ? l : l * l, zx = gates ? 0 : l * l;
        // rows of a node block one component after the other: they share DRAM pages
        int nb = (int)((p - j.first) / w), m = (int)((p - j.first) - (int64_t)nb * w);
        int nbf = nb + PF / w, mf = m + PF % w;  // PF slabs on
        if (mf >= w) {
          mf -= w;
          ++nbf;
        }
        for (; p < stop; ++p, ++g) {
          if (!free && !wait_phase(smem_u32(&empty[s]), (lap - 1) & 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t s_next = (s + 1) % RAW, lap_next = s_next ? lap : lap + 1;
          free = lap_next == 0 || peek_parity(smem_u32(&empty[s_next]), (lap_next - 1) & 1u);
          if (p + PF < stop) {  // the ring's stages alone do not cover DRAM
            tma_prefetch_3d(md, j.ht * BM, nbf * 32, zd + mf);
            tma_prefetch_3d(&mp.x, j.ct * BN, nbf * 32, zx + mf);
            if (++mf == w) {
              mf = 0;
              ++nbf;
            }
          }
          uint8_t* st = raw + s * (C::TILE_D + C::TILE_X);
          const uint32_t fb = smem_u32(&full[s]);
          arrive_tx(fb, C::TILE_D + C::TILE_X);
          tma_load_3d(smem_u32(st), md, j.ht * BM, nb * 32, zd + m, fb);
          tma_load_3d(smem_u32(st + C::TILE_D), &mp.x, j.ct * BN, nb * 32, zx + m, fb);
          if (++m == w) {
            m = 0;
            ++nb;
          }
          s = s_next;
          lap = lap_next;
        }
      }
      for (int t = 0; t < RAW; ++t) {
        const int64_t uses = g > t ? (g - 1 - t) / RAW + 1 : 0;
        if (uses > 0) drain_bar(smem_u32(&full[t]), (uint32_t)((uses - 1) & 1));
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issue
      const uint64_t desc = make_desc(smem_u32(smem));
      uint32_t os = 0, op_phase = 0, ab = 0, acc_phase = 0;
      bool ok = true, op_ready = false, acc_ready = false;
      for (int64_t p = begin; p < end && ok;) {
        const Job j = job_at(a, p);
        const int slabs = (int)(min(end, j.last) - p);
        p += slabs;
        if (a.skip >> j.mat & 1) continue;
#pragma unroll 1
        for (int t = 0; t < slabs; ++t) {
          const bool first = t % KG == 0, last = t % KG == KG - 1 || t + 1 == slabs;  // of its unit
          if (first && !acc_ready) ok = wait_warp(smem_u32(&acc_empty[ab]), acc_phase ^ 1u, abort_flag);
          if (!op_ready) ok = ok && wait_warp(smem_u32(&op_full[os]), op_phase, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;");
          const uint32_t os_next = os ^ 1u, ph_next = op_phase ^ os, ab_next = ab ^ 1u, acc_next = acc_phase ^ ab;
          const bool peek_op = peek_parity(smem_u32(&op_full[os_next]), ph_next);
          const bool peek_acc = peek_parity(smem_u32(&acc_empty[ab_next]), acc_next ^ 1u);
          const uint32_t d = tmem + (uint32_t)A_COLS + ab * (uint32_t)BN;
          const uint32_t tah = tmem + os * (uint32_t)(2 * BK), tal = tah + (uint32_t)BK;
          const uint64_t dbh = desc + (uint64_t)os * (C::OPERAND >> 4), dbl = dbh + (uint64_t)(TILE_B >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / 8; ++kk) {
              mma_ta<BN>(d, tal + kk * 8, dbh + 2 * kk, first && kk == 0 ? 0u : 1u);
              if (C::X32) mma_ta<BN>(d, tah + kk * 8, dbl + 2 * kk, 1u);
            }
#pragma unroll
            for (int kk = 0; kk < BK / 8; ++kk) mma_ta<BN>(d, tah + kk * 8, dbh + 2 * kk, 1u);
            commit(smem_u32(&op_free[os]));
            if (last) commit(smem_u32(&acc_full[ab]));
          }
          op_ready = __all_sync(0xffffffffu, peek_op);
          const bool acc_next_ready = __all_sync(0xffffffffu, peek_acc);
          os = os_next;
          op_phase = ph_next;
          if (last) {
            acc_ready = acc_next_ready;
            ab = ab_next;
            acc_phase = acc_next;
          }
        }
      }
      if (elect_one()) {
        commit(smem_u32(drain));
        drain_bar(smem_u32(drain), 0);
      }
      __syncwarp();
    }
  } else if (warp < W_EPI0) {
    FC_SETMAXNREG_DEC(56);
    // ------------------------------------------------------------------ splitters
    const int mine = (warp - W_SPLIT0) >> 3;           // this group's slabs: g = mine mod 2
    const bool of_d = ((warp - W_SPLIT0) & 4) == 0;    // dv / dz into tensor memory, or x into K-major rows
    const int c = (warp & 3) * 32 + lane;              // channel: lane of tensor memory, or row of the B tile
    const uint32_t ta = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(mine * 2 * BK);
    uint8_t* ops = smem + mine * C::OPERAND;
    uint32_t s = (uint32_t)mine, lap = 0, op_phase = 1;  // own raw stage, own operand slot (free at first)
    int left = -mine;                                    // slabs of the part from this group's next one on
    bool ok = true, full_ready = false;
    for (int64_t p = begin; p < end && ok;) {
      const Job j = job_at(a, p);
      const int slabs = (int)(min(end, j.last) - p);
      p += slabs;
      if (a.skip >> j.mat & 1) continue;
      const bool bias = of_d && a.bias_part && j.mat >= a.ranks && j.ct == 0;
      float bsum = 0.f;
      for (left += slabs; left > 0; left -= 2) {
        if (!full_ready) ok = wait_warp(smem_u32(&full[s]), lap & 1u, abort_flag);
        ok = ok && wait_warp(smem_u32(&op_free[mine]), op_phase, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint8_t* st = raw + s * (C::TILE_D + C::TILE_X);
        const uint32_t s_next = s ^ 2u, lap_next = lap + (s >> 1);  // stages mine and mine + 2 in turn
        const bool peek_full = peek_parity(smem_u32(&full[s_next]), lap_next & 1u);
        // 16 rows at a time; hi = the upper 19 bits, lo = the exact rest, rounded where tf32 ends
        if (of_d) {
          const uint32_t* src = reinterpret_cast<const uint32_t*>(st) + c;
          float t = 0.f;  // a slab's sum first: fewer roundings against the running sum
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t x[16], q[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = src[(h * 16 + k) * BM];
            if (bias)
#pragma unroll
              for (int k = 0; k < 16; ++k) t += __uint_as_float(x[k]);
#pragma unroll
            for (int k = 0; k < 16; ++k) q[k] = x[k] & 0xFFFFE000u;
            tmem_st16(ta + h * 16, q);
#pragma unroll
            for (int k = 0; k < 16; ++k)
              q[k] = __float_as_uint(__uint_as_float(x[k]) - __uint_as_float(x[k] & 0xFFFFE000u)) + 0x1000u;
            tmem_st16(ta + BK + h * 16, q);
          }
          bsum += t;
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        } else {
          // hi rounded here: were both operands' lo parts of their values' sign, the product of
          // the two that is left out would not average out (2.4e-7 of the sum)
          const uint32_t r0 = C::X32 ? 0x1000u : 0u;
          const T* src = reinterpret_cast<const T*>(st + C::TILE_D) + c;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t x[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(Io<T>::get(src[(h * 16 + k) * BN]));
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 v;
              v.x = (x[4 * q] + r0) & 0xFFFFE000u, v.y = (x[4 * q + 1] + r0) & 0xFFFFE000u;
              v.z = (x[4 * q + 2] + r0) & 0xFFFFE000u, v.w = (x[4 * q + 3] + r0) & 0xFFFFE000u;
              *reinterpret_cast<uint4*>(ops + chunk_at<float>(c, h * 4 + q)) = v;
              if (C::X32) {
                uint4 r;
                r.x = __float_as_uint(__uint_as_float(x[4 * q]) - __uint_as_float(v.x)) + 0x1000u;
                r.y = __float_as_uint(__uint_as_float(x[4 * q + 1]) - __uint_as_float(v.y)) + 0x1000u;
                r.z = __float_as_uint(__uint_as_float(x[4 * q + 2]) - __uint_as_float(v.z)) + 0x1000u;
                r.w = __float_as_uint(__uint_as_float(x[4 * q + 3]) - __uint_as_float(v.w)) + 0x1000u;
                *reinterpret_cast<uint4*>(ops + TILE_B + chunk_at<float>(c, h * 4 + q)) = r;
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) {
          arrive(smem_u32(&empty[s]));
          arrive(smem_u32(&op_full[mine]));
        }
        full_ready = __all_sync(0xffffffffu, peek_full);
        s = s_next;
        lap = lap_next;
        op_phase ^= 1u;
      }
      // both groups' sums of the bias channel: the first group's in the first half of the slot
      if (bias && ok) a.bias_part[((blockIdx.x + j.index) * 2 + mine) * BM + c] = bsum;
    }
  } else {
    FC_SETMAXNREG_INC(120);
    // ------------------------------------------------------------------ epilogue: unit sums
    const int quarter = warp & 3, half = (warp - W_EPI0) >> 2;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(A_COLS + half * 64);
    uint32_t ab = 0, acc_phase = 0;
    bool ok = true;
    for (int64_t p = begin; p < end && ok;) {
      const Job j = job_at(a, p);
      const int slabs = (int)(min(end, j.last) - p);
      p += slabs;
      if (a.skip >> j.mat & 1) continue;
      float acc[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) acc[c] = 0.f;
#pragma unroll 1
      for (int t = 0; t < slabs; t += KG) {
        if (!wait_warp(smem_u32(&acc_full[ab]), acc_phase, abort_flag)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
        for (int cb = 0; cb < 4; ++cb) {
          float f[16];
          tmem_ld<16>(lane_base + ab * (uint32_t)BN + (uint32_t)(cb * 16), f);
#pragma unroll
          for (int c = 0; c < 16; ++c) acc[cb * 16 + c] += f[c];
        }
        asm volatile("tcgen05.fence::before_thread_sync;");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&acc_empty[ab]));
        acc_phase ^= ab;
        ab ^= 1u;
      }
      if (!ok) break;
      float4* out =
          reinterpret_cast<float4*>(a.part + ((blockIdx.x + j.index) * BM + quarter * 32 + lane) * BN + half * 64);
#pragma unroll
      for (int c = 0; c < 16; ++c)
        out[c] = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) fc_flag(a.status, FC_DEV_TIMEOUT);
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// The same from two bfloat16 parts of dv and dz and bfloat16 rows x: the tensor cores take both
// operands M- and N-major, as they lie in memory, so slabs of 64 rows go from DRAM to shared
// memory and nothing is transposed. dz's column sums (the bias) are a product with a tile of ones.
// Bound by DRAM (200 MB for 100,003 rows of 96 x 200 channels, 31 us at the copy rate; measured 41
// us, with float dv and dz split and transposed by threads 66).
// The 12 warps: 0 TMA producer, 1 MMA issue, 4-11 epilogue (unit sums).
constexpr int P_ROWS = 64, P_BOX = P_ROWS * 128;  // 64 channels of 64 rows
constexpr int P_STAGE = 6 * P_BOX, P_STAGES = 4;  // hi, lo and x, two boxes each
constexpr int P_KG = 4;                           // slabs per accumulation unit: 32 accumulations
constexpr int P_ONES = 2048, P_THREADS = 12 * 32;
constexpr int P_SMEM = P_STAGES * P_STAGE + P_ONES + BAR_BYTES + 1024;
static_assert(P_SMEM <= 227 * 1024, "shared memory per CTA");

// M- or N-major operand of 128-byte rows (64 channels): 8 KB to the next 64 channels, 1 KB to the
// next 8 rows of the reduction.
__device__ __forceinline__ uint64_t make_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)(P_BOX >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

template <int N, bool B_MN>
__device__ __forceinline__ void mma_parts(uint32_t d, uint64_t da, uint64_t db, uint32_t acc) {
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (B_MN ? 1u << 16 : 0u) |
                             ((uint32_t)(N >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc));
}

__global__ void __launch_bounds__(P_THREADS, 1)
    wgrad_parts_kernel(const __grid_constant__ WMaps mp, const WArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ones = smem + P_STAGES * P_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(ones + P_ONES);
  uint64_t* empty = full + P_STAGES;
  uint64_t* acc_full = empty + P_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  constexpr int B_COLS = 2 * BN;  // behind the accumulators: the bias's

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
    for (int s = 0; s < P_STAGES; ++s) {
      init(&full[s], 1);
      init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      init(&acc_full[b], 1);
      init(&acc_empty[b], 8);
    }
    init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = threadIdx.x; i < P_ONES / 4; i += P_THREADS) reinterpret_cast<uint32_t*>(ones)[i] = 0x3F803F80u;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;
  const int64_t begin = cta_begin(a, blockIdx.x), end = cta_begin(a, blockIdx.x + 1);

  if (warp == 0) {
    if (elect_one()) {
      int64_t g = 0;
      uint32_t s = 0, lap = 0;
      bool ok = true, free = true;  // (peeked: the next stage is free)
      for (int64_t p = begin; p < end && ok;) {
        const Job j = job_at(a, p);
        const bool gates = j.mat >= a.ranks;
        const int l = gates ? j.mat - a.ranks : j.mat, w = gates ? 1 : 2 * l + 1;
        const int64_t stop = min(end, j.last);
        if (a.skip >> j.mat & 1) {
          p = stop;
          continue;
        }
        const CUtensorMap* md = gates ? &mp.dz : &mp.dv;
        const int zd = gates ? l : l * l, zx = gates ? 0 : l * l;
        int nb = (int)((p - j.first) / w), m = (int)((p - j.first) - (int64_t)nb * w);
        for (; p < stop; ++p, ++g) {
          if (!free && !wait_phase(smem_u32(&empty[s]), (lap - 1) & 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t s_next = (s + 1) % P_STAGES, lap_next = s_next ? lap : lap + 1;
          free = lap_next == 0 || peek_parity(smem_u32(&empty[s_next]), (lap_next - 1) & 1u);
          const uint32_t st = smem_u32(smem + s * P_STAGE), fb = smem_u32(&full[s]);
          arrive_tx(fb, P_STAGE);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int h0 = j.ht * BM + half * 64, c0 = j.ct * BN + half * 64;
            tma_load_3d(st + half * P_BOX, md, h0, nb * P_ROWS, 2 * (zd + m), fb);
            tma_load_3d(st + (2 + half) * P_BOX, md, h0, nb * P_ROWS, 2 * (zd + m) + 1, fb);
            tma_load_3d(st + (4 + half) * P_BOX, &mp.x, c0, nb * P_ROWS, zx + m, fb);
          }
          if (++m == w) {
            m = 0;
            ++nb;
          }
          s = s_next;
          lap = lap_next;
        }
      }
      for (int t = 0; t < P_STAGES; ++t) {
        const int64_t uses = g > t ? (g - 1 - t) / P_STAGES + 1 : 0;
        if (uses > 0) drain_bar(smem_u32(&full[t]), (uint32_t)((uses - 1) & 1));
      }
    }
  } else if (warp == 1) {
    const uint64_t desc = make_desc_mn(smem_u32(smem)), desc_ones = make_desc(smem_u32(ones));
    uint32_t s = 0, lap = 0, ab = 0, acc_phase = 0;
    bool ok = true, ready_a = false;
    for (int64_t p = begin; p < end && ok;) {
      const Job j = job_at(a, p);
      const int slabs = (int)(min(end, j.last) - p);
      p += slabs;
      if (a.skip >> j.mat & 1) continue;
      const bool bias = a.bias_part && j.mat >= a.ranks && j.ct == 0;
#pragma unroll 1
      for (int t = 0; t < slabs; ++t) {
        const bool opens = t % P_KG == 0, closes = t % P_KG == P_KG - 1 || t + 1 == slabs;
        if (opens) ok = wait_warp(smem_u32(&acc_empty[ab]), acc_phase ^ 1u, abort_flag);
        if (!ready_a) ok = ok && wait_warp(smem_u32(&full[s]), lap & 1u, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint32_t s_next = (s + 1) % P_STAGES, lap_next = s_next ? lap : lap + 1;
        const bool peek = peek_parity(smem_u32(&full[s_next]), lap_next & 1u);
        if (elect_one()) {
          const uint32_t d = tmem + ab * (uint32_t)BN, db = tmem + (uint32_t)B_COLS + ab * 16u;
          const uint64_t st = desc + (uint64_t)(s * (P_STAGE >> 4)), x = st + (uint64_t)(4 * P_BOX >> 4);
#pragma unroll
          for (int part = 1; part >= 0; --part)  // the low parts first: a sum is truncated less while it is small
#pragma unroll
            for (int kk = 0; kk < P_ROWS / 16; ++kk) {
              const uint64_t da = st + (uint64_t)((part * 2 * P_BOX + kk * 2048) >> 4);
              const uint32_t more = opens && part == 1 && kk == 0 ? 0u : 1u;
              mma_parts<BN, true>(d, da, x + (uint64_t)(kk * 2048 >> 4), more);
              if (bias) mma_parts<16, false>(db, da, desc_ones, more);
            }
          commit(smem_u32(&empty[s]));
          if (closes) commit(smem_u32(&acc_full[ab]));
        }
        ready_a = __all_sync(0xffffffffu, peek);
        s = s_next;
        lap = lap_next;
        if (closes) {
          acc_phase ^= ab;
          ab ^= 1u;
        }
      }
    }
    if (elect_one()) {
      commit(smem_u32(drain));
      drain_bar(smem_u32(drain), 0);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue: unit sums
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    uint32_t ab = 0, acc_phase = 0;
    bool ok = true;
    for (int64_t p = begin; p < end && ok;) {
      const Job j = job_at(a, p);
      const int slabs = (int)(min(end, j.last) - p);
      p += slabs;
      if (a.skip >> j.mat & 1) continue;
      const bool bias = a.bias_part && j.mat >= a.ranks && j.ct == 0 && half == 0;
      float acc[64], bsum = 0.f;
#pragma unroll
      for (int c = 0; c < 64; ++c) acc[c] = 0.f;
#pragma unroll 1
      for (int t = 0; t < slabs; t += P_KG) {
        if (!wait_warp(smem_u32(&acc_full[ab]), acc_phase, abort_flag)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
        for (int cb = 0; cb < 4; ++cb) {
          float f[16];
          tmem_ld<16>(lanes + ab * (uint32_t)BN + (uint32_t)(half * 64 + cb * 16), f);
#pragma unroll
          for (int c = 0; c < 16; ++c) acc[cb * 16 + c] += f[c];
        }
        if (bias) {
          float f[16];
          tmem_ld<16>(lanes + (uint32_t)B_COLS + ab * 16u, f);
          bsum += f[0];
        }
        asm volatile("tcgen05.fence::before_thread_sync;");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&acc_empty[ab]));
        acc_phase ^= ab;
        ab ^= 1u;
      }
      if (!ok) break;
      const int64_t at = blockIdx.x + j.index;
      float4* out = reinterpret_cast<float4*>(a.part + (at * BM + quarter * 32 + lane) * BN + half * 64);
#pragma unroll
      for (int c = 0; c < 16; ++c)
        out[c] = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
      if (bias) {  // (a part's slot holds two sums)
        a.bias_part[at * 2 * BM + quarter * 32 + lane] = bsum;
        a.bias_part[(at * 2 + 1) * BM + quarter * 32 + lane] = 0.f;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) fc_flag(a.status, FC_DEV_TIMEOUT);
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Partial matrices added in the order of the CTAs. A block takes four rows of a job's tile: its
// warps 4 r + p add every fourth partial of row r from the p-th on, and the four sums are added
// in order. The bias goes with the ct = 0 gate jobs.
constexpr int SUM_ROWS = 4, SUM_PARTS = 4;
template <typename T>
__global__ void __launch_bounds__(SUM_ROWS * SUM_PARTS * 32) wgrad_sum_kernel(const WArgs a, const WOut o) {
  __shared__ float4 red[SUM_ROWS][SUM_PARTS][32];
  __shared__ float bred[SUM_ROWS][SUM_PARTS];
  const int tiles = a.n_ht * a.n_ct;
  const int job = (int)(blockIdx.x / (BM / SUM_ROWS)), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rr = warp / SUM_PARTS, part = warp % SUM_PARTS;
  const int row = (int)(blockIdx.x % (BM / SUM_ROWS)) * SUM_ROWS + rr;
  const int mat = job / tiles, t = job - mat * tiles, ht = t / a.n_ct, ct = t - ht * a.n_ct;
  const bool gates = mat >= a.ranks;
  const int l = gates ? mat - a.ranks : mat;
  const int h = ht * BM + row, c = ct * BN + lane * 4;
  const bool bias = gates && o.bias && ct == 0;
  if (ht * BM + (int)(blockIdx.x % (BM / SUM_ROWS)) * SUM_ROWS >= a.H || (!o.w[mat] && !bias)) return;  // whole block
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float bsum = 0.f;
  if (a.total > 0) {
    // the CTAs whose share [i total / ctas, (i + 1) total / ctas) meets the job's slabs
    int64_t first = 0;
    for (int m = 0; m < mat; ++m) first += a.width[m] * tiles;
    const int64_t last = first + (t + 1) * a.width[mat];
    first += t * a.width[mat];
    int64_t i0 = first * a.ctas / a.total, i1 = last * a.ctas / a.total;
    while (i0 > 0 && cta_begin(a, i0) > first) --i0;
    while (i0 + 1 < a.ctas && cta_begin(a, i0 + 1) <= first) ++i0;
    while (i1 > i0 && cta_begin(a, i1) >= last) --i1;
    if (i1 >= a.ctas) i1 = a.ctas - 1;
    const float* p = a.part + ((i0 + part + job) * BM + row) * BN + lane * 4;
    const float* q = a.bias_part + (i0 + part + job) * 2 * BM + row;
    const int n = (int)(i1 - i0) - part;
#pragma unroll 8
    for (int i = 0; i <= n; i += SUM_PARTS) {
      const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)i * BM * BN);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if (bias && lane == 0)
      for (int i = 0; i <= n; i += SUM_PARTS) bsum += q[(int64_t)i * 2 * BM] + q[(int64_t)i * 2 * BM + BM];
  }
  red[rr][part][lane] = sum;
  if (lane == 0) bred[rr][part] = bsum;
  __syncthreads();
  if (part != 0 || h >= a.H) return;
  for (int k = 1; k < SUM_PARTS; ++k) {
    const float4 v = red[rr][k][lane];
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    bsum += bred[rr][k];
  }
  const float sc = o.scales[gates ? a.ranks : l];
  if (o.w[mat]) {
    T* out = (T*)o.w[mat] + ((int64_t)(gates ? l * a.H : 0) + h) * a.Cn + c;
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < a.Cn) out[e] = Io<T>::put(sc * v[e]);
  }
  if (bias && lane == 0) ((T*)o.bias)[(int64_t)l * a.H + h] = Io<T>::put(bsum);
}

int64_t wgrad_part_count(int ranks, int C, int H, int sms) {
  return (int64_t)sms + 2 * ranks * ((H + BM - 1) / BM) * (int64_t)((C + BN - 1) / BN);
}

template <typename T>
int run_wgrad(int ranks, int C, int H, int64_t n, const void* dv, const void* dz, int64_t dv_ld, bool parts,
              const T* x, int64_t x_ld, float* part, float* bias_part, const WOut& o, int* status, int sms,
              cudaStream_t s) {
  WArgs wa{};
  wa.ranks = ranks;
  wa.H = H;
  wa.Cn = C;
  wa.n_ht = (H + BM - 1) / BM;
  wa.n_ct = (C + BN - 1) / BN;
  const int rows = parts ? P_ROWS : 32;
  wa.blocks = (n + rows - 1) / rows;
  for (int l = 0; l < ranks; ++l) {
    wa.width[l] = wa.blocks * (2 * l + 1);
    wa.width[ranks + l] = wa.blocks;
    if (!o.w[l]) wa.skip |= 1 << l;
    if (!o.w[ranks + l] && !o.bias) wa.skip |= 1 << (ranks + l);
    wa.total += (wa.width[l] + wa.width[ranks + l]) * wa.n_ht * wa.n_ct;
  }
  wa.part = part;
  wa.bias_part = o.bias ? bias_part : nullptr;
  wa.status = status;
  wa.ctas = 1;
  if (wa.total > 0) {
    // at least four slabs per CTA: a partial matrix costs 128 KB of traffic
    wa.ctas = (int)std::min<int64_t>(sms, (wa.total + 3) / 4);
    const int comps = ranks * ranks;
    WMaps wm;
    if (parts) {
      if (!encode_rows<bf16_t>(&wm.dv, dv, H, n, 2 * comps, dv_ld, 64, P_ROWS) ||
          !encode_rows<bf16_t>(&wm.dz, dz, H, n, 2 * ranks, dv_ld, 64, P_ROWS) ||
          !encode_rows<T>(&wm.x, x, C, n, comps, x_ld, 64, P_ROWS))
        return FC_ERR_UNSUPPORTED;
      static Ready state;
      if (int rc = ready(wgrad_parts_kernel, P_SMEM, state, 0)) return rc;
      wgrad_parts_kernel<<<wa.ctas, P_THREADS, P_SMEM, s>>>(wm, wa);
    } else {
      if (!encode_rows<float>(&wm.dv, dv, H, n, comps, dv_ld, BM, 32) ||
          !encode_rows<float>(&wm.dz, dz, H, n, ranks, dv_ld, BM, 32) ||
          !encode_rows<T>(&wm.x, x, C, n, comps, x_ld, BN, 32))
        return FC_ERR_UNSUPPORTED;
      constexpr int smem = WCfg<T>::SMEM;
      static Ready state;
      if (int rc = ready(wgrad_kernel<T>, smem, state, W_REGS)) return rc;
      wgrad_kernel<T><<<wa.ctas, W_THREADS, smem, s>>>(wm, wa);
    }
    if (int rc = fc_launched(1)) return rc;
  }
  wgrad_sum_kernel<T><<<(unsigned)(2 * ranks * wa.n_ht * wa.n_ct * (BM / SUM_ROWS)), SUM_ROWS * SUM_PARTS * 32, 0,
                        s>>>(wa, o);
  return fc_launched(1);
}
template int run_wgrad<float>(int, int, int, int64_t, const void*, const void*, int64_t, bool, const float*, int64_t,
                              float*, float*, const WOut&, int*, int, cudaStream_t);
template int run_wgrad<bf16_t>(int, int, int, int64_t, const void*, const void*, int64_t, bool, const bf16_t*, int64_t,
                               float*, float*, const WOut&, int*, int, cudaStream_t);

}  // namespace gtc
}  // namespace fc

#endif  // FC_HOST_EMU
