// Irreps dropout from a counter-based generator: y = x * keep / (1 - p), the mask computed
// where it is used and never stored.
//
// A feature row holds rank blocks l = 0..L of (2l+1, C). keep is one decision per (row, l,
// channel), shared by the 2l+1 components of the rank, so the operator commutes with
// rotations (dropping single components would not). L = 0 is the usual elementwise dropout.
//
// Randomness: Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC11): four channels 4q..4q+3 of a (row, l) take the four
// words of the block with counter (i mod 2^32, i div 2^32, offset mod 2^32, offset div
// 2^32), i = (row (L+1) + l) ceil(C/4) + q, and key = seed. A channel is dropped where its
// word is below floor(p 2^32). The gradient is the same operator on the output gradient with
// the same (seed, offset); they are read from device memory, so a captured step can advance
// them in place. A dropped element is 0 whatever x holds there (infinities and NaN
// included).
//
// What bounds it: DRAM, one read and one write of every element (one 16-byte vector per
// thread and component). One generator block serves 4 (2l+1) elements. Measured: 27,648 x 16 rows
// of 128 float32 channels 70 us a pass (6.4 TB/s, the copy rate); 2^26 plain elements 86 us in
// float32 (6.2 TB/s) and 84 us in bfloat16 (3.2 TB/s), where instructions are the bound: 122 for four
// elements, of which the generator's wide products are 20 and its keys' steps 20 (issue slots 71% busy,
// integer pipe 57%, DRAM 32%); channel counts that are no fours (99) go element by element, 117 us in
// float32.
#include "fc_vec.cuh"

namespace fc {

FC_HD FC_INLINE void philox4x32(uint32_t c[4], uint32_t k0, uint32_t k1) {
#ifdef __CUDA_ARCH__
#pragma unroll
#endif
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0];
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[1] = (uint32_t)p1;
    c[3] = (uint32_t)p0;
    c[0] = n0;
    c[2] = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

struct DropArgs {
  int64_t units;       // n * (L+1) * quads: one unit = four channels of one rank of one row
  int C, quads;
  uint64_t threshold;  // floor(p 2^32), up to 2^32
  double scale;        // 1 / (1 - p); 0 for p = 1
};

// keep factors of unit u's four channels
template <typename A>
FC_HD FC_INLINE void drop_factors(const DropArgs& a, uint64_t u, uint64_t seed, uint64_t offset, A f[4]) {
  uint32_t c[4] = {(uint32_t)u, (uint32_t)(u >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
  philox4x32(c, (uint32_t)seed, (uint32_t)(seed >> 32));
#ifdef __CUDA_ARCH__
#pragma unroll
#endif
  for (int k = 0; k < 4; ++k) f[k] = (uint64_t)c[k] >= a.threshold ? (A)a.scale : A(0);
}

template <typename A>
FC_HD FC_INLINE A drop_apply(A x, A f) {
  return f != A(0) ? x * f : A(0);
}

#ifdef FC_HOST_EMU

template <typename T>
int dropout_dispatch(int L, const T* x, const int64_t* rng, T* y, const DropArgs& a, cudaStream_t) {
  using A = typename Io<T>::Acc;
  for (int64_t u = 0; u < a.units; ++u) {
    A f[4];
    drop_factors<A>(a, (uint64_t)u, (uint64_t)rng[0], (uint64_t)rng[1], f);
    const int64_t rl = u / a.quads, row = rl / (L + 1);
    const int q = (int)(u - rl * a.quads), l = (int)(rl - row * (L + 1));
    for (int m = 0; m < 2 * l + 1; ++m)
      for (int k = 0; k < 4 && 4 * q + k < a.C; ++k) {
        const int64_t e = (row * (L + 1) * (L + 1) + l * l + m) * a.C + 4 * q + k;
        y[e] = Io<T>::put(drop_apply<A>(Io<T>::get(x[e]), f[k]));
      }
  }
  return 0;
}

#else

// I: type of the unit index (32 bits where the units fit: its two divisions are then cheap).
// VEC: a unit's four channels move as one vector (channels in fours, aligned tensors).
// UN units per thread, a block apart, with all their loads issued before the generator runs.
template <typename T, int L, bool VEC, int UN, typename I>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, const int64_t* __restrict__ rng,
                                                      T* __restrict__ y, const DropArgs a) {
  using A = typename Io<T>::Acc;
  constexpr int NC = (L + 1) * (L + 1);
  const uint64_t seed = (uint64_t)__ldg(rng), offset = (uint64_t)__ldg(rng + 1);
  const I total = (I)a.units, quads = (I)a.quads;
  constexpr int NV = sizeof(T) == 8 ? 2 : 4, PARTS = 4 / NV;  // a 64-bit quad is two 16-byte vectors
  for (I u0 = (I)blockIdx.x * (256 * UN) + threadIdx.x; u0 < total; u0 += (I)gridDim.x * (256 * UN)) {
    if constexpr (L == 0 && VEC) {
      // plain rows of channels in fours are one run of quads
      Pack<T, NV> v[UN][PARTS];
#pragma unroll
      for (int j = 0; j < UN; ++j)
        if (u0 + j * 256 < total)
#pragma unroll
          for (int h = 0; h < PARTS; ++h) v[j][h].load_stream(x + ((int64_t)(u0 + j * 256) * 4 + h * NV));
#pragma unroll
      for (int j = 0; j < UN; ++j)
        if (u0 + j * 256 < total) {
          A f[4];
          drop_factors<A>(a, (uint64_t)(u0 + j * 256), seed, offset, f);
#pragma unroll
          for (int h = 0; h < PARTS; ++h) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
              v[j][h].set(k, Io<T>::put(drop_apply<A>(Io<T>::get(v[j][h].at(k)), f[h * NV + k])));
            v[j][h].store(y + ((int64_t)(u0 + j * 256) * 4 + h * NV));
          }
        }
    } else {
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        const I u = u0 + j * 256;
        if (u >= total) break;
        const I rl = u / quads, row = rl / (L + 1);
        const int q = (int)(u - rl * quads), l = (int)(rl - row * (L + 1));
        const int64_t base = ((int64_t)row * NC + l * l) * a.C + 4 * q;
        const int ms = 2 * l + 1;
        if constexpr (VEC) {
          Pack<T, NV> v[2 * L + 1][PARTS];
#pragma unroll
          for (int m = 0; m < 2 * L + 1; ++m)
            if (m < ms)
#pragma unroll
              for (int h = 0; h < PARTS; ++h) v[m][h].load_stream(x + base + (int64_t)m * a.C + h * NV);
          A f[4];
          drop_factors<A>(a, (uint64_t)u, seed, offset, f);
#pragma unroll
          for (int m = 0; m < 2 * L + 1; ++m)
            if (m < ms)
#pragma unroll
              for (int h = 0; h < PARTS; ++h) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
                  v[m][h].set(k, Io<T>::put(drop_apply<A>(Io<T>::get(v[m][h].at(k)), f[h * NV + k])));
                v[m][h].store(y + base + (int64_t)m * a.C + h * NV);
              }
        } else {
          A f[4];
          drop_factors<A>(a, (uint64_t)u, seed, offset, f);
          const int nk = min(4, a.C - 4 * q);
          for (int m = 0; m < ms; ++m)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (k < nk) {
                const int64_t e = base + (int64_t)m * a.C + k;
                y[e] = Io<T>::put(drop_apply<A>(Io<T>::get(x[e]), f[k]));
              }
        }
      }
    }
  }
}

template <typename T, int L, bool VEC>
static int dropout_launch(const T* x, const int64_t* rng, T* y, const DropArgs& a, cudaStream_t s) {
  constexpr int UN = (L == 0 && VEC) ? (sizeof(T) == 2 ? 4 : 2) : 1;
  const int64_t b = (a.units + 256 * UN - 1) / (256 * UN);
  const unsigned grid = (unsigned)(b < (1 << 20) ? b : (1 << 20));
  // the grid-stride index must not wrap: units plus one stride fit 32 bits
  if (a.units + (int64_t)grid * 256 * UN < ((int64_t)1 << 32))
    dropout_kernel<T, L, VEC, UN, uint32_t><<<grid, 256, 0, s>>>(x, rng, y, a);
  else
    dropout_kernel<T, L, VEC, UN, uint64_t><<<grid, 256, 0, s>>>(x, rng, y, a);
  return fc_launched(1);
}

template <typename T>
int dropout_dispatch(int L, const T* x, const int64_t* rng, T* y, const DropArgs& a, cudaStream_t s) {
  const uintptr_t mask = (sizeof(T) == 8 ? 16 : 4 * sizeof(T)) - 1;
  const bool vec = a.C % 4 == 0 && !((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & mask);
  switch (L * 2 + (vec ? 1 : 0)) {
    case 0: return dropout_launch<T, 0, false>(x, rng, y, a, s);
    case 1: return dropout_launch<T, 0, true>(x, rng, y, a, s);
    case 2: return dropout_launch<T, 1, false>(x, rng, y, a, s);
    case 3: return dropout_launch<T, 1, true>(x, rng, y, a, s);
    case 4: return dropout_launch<T, 2, false>(x, rng, y, a, s);
    case 5: return dropout_launch<T, 2, true>(x, rng, y, a, s);
    case 6: return dropout_launch<T, 3, false>(x, rng, y, a, s);
    default: return dropout_launch<T, 3, true>(x, rng, y, a, s);
  }
}

#endif

// p in [0, 1], sizes checked by the caller
template <typename T>
int irreps_dropout(int L, int features, const void* x, const int64_t* rng, double p, int64_t n, void* y,
                   cudaStream_t s) {
  DropArgs a;
  a.C = features;
  a.quads = (features + 3) / 4;
  a.units = n * (L + 1) * a.quads;
  a.threshold = (uint64_t)(p * 4294967296.0);
  a.scale = p < 1.0 ? 1.0 / (1.0 - p) : 0.0;
  return dropout_dispatch<T>(L, (const T*)x, rng, (T*)y, a, s);
}

template int irreps_dropout<float>(int, int, const void*, const int64_t*, double, int64_t, void*, cudaStream_t);
template int irreps_dropout<double>(int, int, const void*, const int64_t*, double, int64_t, void*, cudaStream_t);
template int irreps_dropout<bf16_t>(int, int, const void*, const int64_t*, double, int64_t, void*, cudaStream_t);

}  // namespace fc
