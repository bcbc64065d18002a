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
#include "gated_ff_tc.cuh"

#ifndef FC_HOST_EMU

#include <algorithm>

namespace fc {
namespace gtc {

constexpr int BN = 128, TILE_B = BN * BK * 4;
constexpr int KG = 2;  // slabs per accumulation unit (see gated_ff_tc.cu)

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
      init(&split[s], 8);
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
          if (g >= S && !wait_phase(smem_u32(&empty[s]), (uint32_t)(((g / S) - 1) & 1), abort_flag)) {
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
          if (v >= 1 && !wait_phase(smem_u32(&acc_empty[b]), (uint32_t)((v - 1) & 1), abort_flag)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;");
          const uint32_t d = tmem + (uint32_t)(A_COLS + b * BN);
          const int64_t unit = min(stop, p + KG);
          bool fresh = true;
          for (; p < unit; ++p, ++g) {
            const int s = (int)(g % S);
            if (!wait_phase(smem_u32(&split[s]), (uint32_t)((g / S) & 1), abort_flag)) {
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
        if (!wait_warp(smem_u32(&full[s]), (uint32_t)((g / S) & 1), abort_flag)) {
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
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&split[s]));
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
        if (!wait_warp(smem_u32(&acc_full[b]), (uint32_t)((u / NACC) & 1), abort_flag)) {
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
    const float* q = a.bias_part + (i0 + part + job) * BM + row;
    const int n = (int)(i1 - i0) - part;
#pragma unroll 8
    for (int i = 0; i <= n; i += SUM_PARTS) {
      const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)i * BM * BN);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if (bias && lane == 0)
      for (int i = 0; i <= n; i += SUM_PARTS) bsum += q[(int64_t)i * BM];
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
int run_wgrad(int ranks, int C, int H, int64_t n, const float* dv, const float* dz, int64_t dv_ld, const T* x,
              int64_t x_ld, float* part, float* bias_part, const WOut& o, int* status, int sms, cudaStream_t s) {
  WArgs wa{};
  wa.ranks = ranks;
  wa.H = H;
  wa.Cn = C;
  wa.n_ht = (H + BM - 1) / BM;
  wa.n_ct = (C + BN - 1) / BN;
  wa.blocks = (n + 31) / 32;
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
    if (!encode_rows<float>(&wm.dv, dv, H, n, comps, dv_ld, BM, 32) ||
        !encode_rows<float>(&wm.dz, dz, H, n, ranks, dv_ld, BM, 32) ||
        !encode_rows<T>(&wm.x, x, C, n, comps, x_ld, BN, 32))
      return FC_ERR_UNSUPPORTED;
    constexpr int smem = WCfg<T>::SMEM;
    static Ready state;
    if (int rc = ready(wgrad_kernel<T>, smem, state)) return rc;
    wgrad_kernel<T><<<wa.ctas, THREADS, smem, s>>>(wm, wa);
    if (int rc = fc_check_launch()) return rc;
  }
  wgrad_sum_kernel<T><<<(unsigned)(2 * ranks * wa.n_ht * wa.n_ct * (BM / SUM_ROWS)), SUM_ROWS * SUM_PARTS * 32, 0,
                        s>>>(wa, o);
  return fc_check_launch();
}
template int run_wgrad<float>(int, int, int, int64_t, const float*, const float*, int64_t, const float*, int64_t, float*,
                              float*, const WOut&, int*, int, cudaStream_t);
template int run_wgrad<bf16_t>(int, int, int, int64_t, const float*, const float*, int64_t, const bf16_t*, int64_t,
                               float*, float*, const WOut&, int*, int, cudaStream_t);

}  // namespace gtc
}  // namespace fc

#endif  // FC_HOST_EMU
