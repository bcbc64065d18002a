// Gated feed-forward block on the tensor cores: what its kernels share.
#pragma once
#include "gated_ff.cuh"
#include "tc_common.cuh"

#ifndef FC_HOST_EMU

namespace fc {
namespace gtc {

using namespace tma;

constexpr int BK = 32, THREADS = 512;
// Reductions of bfloat16 rows and weights up to this length take the kernel without splitting.
constexpr int DIRECT_K = 256, DIRECT_BK = 64, DIRECT_DX_BN = 128;
constexpr int EPI_BUF = 4096;  // a warp's 32 x 32 float staging box
constexpr int BAR_BYTES = 640;
constexpr int SCHED = 4;  // work items handed out ahead
enum { FWD = 0, PRE = 1, DX = 2 };

// What a launch of the product kernels needs beside its tensor maps.
struct Args {
  int64_t items;          // of the work list (of each column tile's list: resident kernel)
  int L, ranks, comps;
  int N;                  // output columns of a component: H (FWD, PRE), C (DX)
  int nk, kg, nu;         // 32-wide slabs of a segment; slabs per unit and units per segment (streaming kernel)
  int n_ct, tiles, main_tiles, per_comp;
  int stages;             // A stages (resident kernel)
  int act;
  const void* bias;       // of the rows' type, or null
  const float* scales;    // one per rank, the gate map's, the activation's
  int* counter;           // work lists, zeroed before the launch
  int* status;
};

struct Maps {
  CUtensorMap a;   // x (FWD, PRE) or dv (DX): (channel, row, component)
  CUtensorMap a2;  // dz (DX): (channel, row, rank)
  CUtensorMap b;   // split weights: (k, output channel, matrix)
  CUtensorMap o;   // y, dv or dx, 32 x 32 boxes
  CUtensorMap g;   // g (PRE)
  CUtensorMap ap;  // a in boxes of a pass's rows and channels, for L2 prefetches (PRE)
  CUtensorMap gp;  // g in boxes of an item's rows and channels, for L2 prefetches (PRE)
  CUtensorMap o2;  // dz (PRE)
};

// Work item: 128 rows, and rank l's components k0 .. k0+nm-1.
struct WorkItem {
  int tile, l, k0, nm;
};

// Lists run through the ranks (high ones first: most work), all tiles of one before the next.
__device__ __forceinline__ WorkItem work_item(const Args& a, int tile, int q) {
  WorkItem w;
  w.tile = tile;
  if (a.per_comp) {
    w.k0 = a.comps - 1 - q;
    w.l = gated_rank_of(w.k0);
    w.nm = 1;
  } else {
    w.l = a.L - q;
    w.k0 = w.l * w.l;
    w.nm = 2 * w.l + 1;
  }
  return w;
}
__device__ __forceinline__ WorkItem work_item(const Args& a, int it) {
  const int q = it / a.tiles;
  return work_item(a, it - q * a.tiles, q);
}

// N consecutive columns of this thread's lane (warp-collective), waited for in the same statement:
// nothing that uses the values can come before the wait.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float* f);
template <>
__device__ __forceinline__ void tmem_ld<32>(uint32_t taddr, float* f) {
  uint32_t v[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int c = 0; c < 32; ++c) f[c] = __uint_as_float(v[c]);
}
template <>
__device__ __forceinline__ void tmem_ld<16>(uint32_t taddr, float* f) {
  uint32_t v[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int c = 0; c < 16; ++c) f[c] = __uint_as_float(v[c]);
}

// The sum of two groups of N consecutive columns of this thread's lane (one wait for both).
template <int N>
__device__ __forceinline__ void tmem_ld_sum(uint32_t ta, uint32_t tb, float* f);
template <>
__device__ __forceinline__ void tmem_ld_sum<16>(uint32_t ta, uint32_t tb, float* f) {
  uint32_t v[16], w[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]), "=r"(w[8]), "=r"(w[9]), "=r"(w[10]), "=r"(w[11]), "=r"(w[12]), "=r"(w[13]), "=r"(w[14]), "=r"(w[15])
      : "r"(ta), "r"(tb)
      : "memory");
#pragma unroll
  for (int c = 0; c < 16; ++c) f[c] = __uint_as_float(v[c]) + __uint_as_float(w[c]);
}
// 16 consecutive tensor-memory columns of this thread's lane (warp-collective).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 32 floats -> the tf32 parts of a lane's 32 columns: hi, the upper 19 bits, and lo, the rest,
// exact in float and rounded where tf32 ends (its lower 13 bits do not reach the product). The
// other operand's hi is rounded, so that the left-out product of both lo parts averages out.
__device__ __forceinline__ void store_parts(uint32_t ta, const uint32_t* x) {
  uint32_t p[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) p[e] = x[e] & 0xFFFFE000u;
  tmem_st32(ta, p);
#pragma unroll
  for (int e = 0; e < 32; ++e)
    p[e] = __float_as_uint(__uint_as_float(x[e]) - __uint_as_float(x[e] & 0xFFFFE000u)) + 0x1000u;
  tmem_st32(ta + BK, p);
}

// One lane of a converged warp. tcgen05 and TMA instructions take their operands from uniform
// registers; behind elect.sync the compiler knows that one lane is active and moves them there
// at once (eight MMAs issue in 385 cycles, the rate of the tensor pipe; behind `lane == 0` in 611).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(p));
  return p != 0;
}

// Whether the phase of this parity is over, without waiting. A barrier operation's answer takes
// about 300 cycles while the tensor cores and copies keep shared memory busy, so the roles ask
// about their next barrier before they work on the current slab and look at the answer after.
__device__ __forceinline__ bool peek_parity(uint32_t mbar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(mbar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded wait for the phase of this parity. Gives up (returning false) after the limit or once
// another role has; the flag tells the others, and the kernel reports it at its end. Kept as
// short as it can be: the roles' loops share each scheduler's instruction cache, and code that
// is fetched again and again costs more than what it does (a wait written out with its error
// path in every place made the kernel 10-40% slower).
constexpr int WAIT_ROUNDS = 1 << 22;
__device__ __forceinline__ bool wait_phase(uint32_t mbar, uint32_t parity, volatile int* abort_flag) {
  bool done;
  int round = 0;
#pragma unroll 1
  do {
    done = test_parity(mbar, parity);
  } while (!done && ++round < WAIT_ROUNDS && !((round & 31) == 0 && *abort_flag));
  if (!done) *abort_flag = 1;
  return done;
}

// wait_phase for a whole warp: one answer, so that no lane leaves a collective alone
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait_phase(bar, parity, abort_flag));
}

__device__ __forceinline__ void drain_bar(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int round = 0; round < WAIT_ROUNDS; ++round)
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

// sigma(z) by the hardware's base-2 exponential and reciprocal. The exponent -z log2(e) is
// formed as a float and its remainder, 2^(t + r) = 2^t (1 + r ln 2), so its rounding does not
// grow with |z|; the power stays finite (the reciprocal of 2^127 is flushed to 0). Where t itself
// overflows (|z| > 2.36e38) there is no remainder to add. NaN stays NaN (through r). Every instruction counts: a rank's gates are computed between two passes of the
// tensor cores, with both accumulators taken.
__device__ __forceinline__ float fast_sigmoid(float z) {
  const float hi = 1.44269502f, lo = 1.92596303e-8f;  // log2(e)
  const float t = -z * hi;
  const float r = fmaf(-z, lo, fmaf(-z, hi, -t));
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fminf(t, 127.f)));
  e = fabsf(t) == __int_as_float(0x7f800000) ? e : fmaf(e, r * 0.693147181f, e);  // (r is no number there)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}
__device__ __forceinline__ float fast_act(int act, float z) {
  const float s = fast_sigmoid(z);
  return act == FC_GATE_SIGMOID ? s : z * s;
}
__device__ __forceinline__ float fast_dact(int act, float z) {
  const float s = fast_sigmoid(z);
  return act == FC_GATE_SIGMOID ? s * (1.f - s) : s * (1.f + z * (1.f - s));
}

#define FC_SETMAXNREG_DEC(n) asm volatile("setmaxnreg.dec.sync.aligned.u32 " #n ";")
#define FC_SETMAXNREG_INC(n) asm volatile("setmaxnreg.inc.sync.aligned.u32 " #n ";")

// Per device: shared-memory size set, and the registers that setmaxnreg shares out checked
// (the block must be launched with `regs` per thread: its roles' shares are counted on that; 0
// where nothing is shared out).
struct Ready {
  bool done[64] = {};
};
template <typename K>
static int ready(K kernel, int smem, Ready& r, int regs = 128) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FC_ERR_LAUNCH;
  if (r.done[dev]) return 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return FC_ERR_LAUNCH;
  cudaFuncAttributes at;
  if (cudaFuncGetAttributes(&at, kernel) != cudaSuccess) return FC_ERR_LAUNCH;
  if (regs && at.numRegs != regs) return FC_ERR_UNSUPPORTED;
  r.done[dev] = true;
  return 0;
}

// Launchers of the other files.
constexpr int STREAM_BN = 128;  // output columns of a tile: streaming kernel
constexpr int STREAM_KG = 2, STREAM_NACC = 3;
template <int MODE>
int run_direct(const Maps& mp, Args a, int sms, cudaStream_t s);
int run_direct_dx(const Maps& mp, const Args& a, int sms, cudaStream_t s);
template <int MODE, typename T>
int run_stream(const Maps& mp, const Args& a, int sms, cudaStream_t s);

struct WOut {
  void* w[8];     // gradient of each matrix (gates: one matrix, ranks by rows), or null
  void* bias;     // ((ranks) H) or null
  const float* scales;
};
int64_t wgrad_part_count(int ranks, int C, int H, int sms);  // 128 x 128 partial matrices of the workspace
// dv, dz: float rows, or (parts) two bfloat16 parts per component, rows of dv_ld elements.
template <typename T>
int run_wgrad(int ranks, int C, int H, int64_t n, const void* dv, const void* dz, int64_t dv_ld, bool parts,
              const T* x, int64_t x_ld, float* part, float* bias_part, const WOut& o, int* status, int sms,
              cudaStream_t s);

// (channel, row, component) map of a tensor of rows [comps][ld]; box_c channels x box_r rows,
// boxes of 128- or 64-byte rows with that swizzle.
template <typename E>
bool encode_rows(CUtensorMap* map, const void* base, int64_t channels, int64_t rows, int64_t comps, int64_t ld,
                 int box_c, int box_r);

}  // namespace gtc
}  // namespace fc

#endif  // FC_HOST_EMU
