// Gated feed-forward block over Cartesian features: 64-bit rows, and the host emulation of
// every type (the tensor-core form of 32- and 16-bit rows is in gated_ff_tc.cu).
//
// For row n, rank l, component m (x_k: the C channels of component k = l^2 + m):
//   z_l = s_g x_0 Wg_l^T + b_l,   a_l = s_a act(z_l),   v_k = s_l x_k Wv_l^T,   y_k = a_l v_k
// and for an output gradient g:
//   dv_k = g_k a_l,   dz_l = s_a act'(z_l) sum_m g_k v_k,
//   dx_k = s_l dv_k Wv_l  (+ s_g sum_l dz_l Wg_l for k = 0),
//   dWv_l = s_l sum_{n,m} dv_k^T x_k,   dWg_l = s_g sum_n dz_l^T x_0,   db_l = sum_n dz_l.
// z and v are recomputed in the backward instead of being kept: they cost as much to write
// and read as x, and the block's activations are what a training step runs out of.
//
// These kernels are 64 x 64 tiles of plain multiply-adds with functors for the operands and
// the epilogue (Acc = float, or double for 64-bit rows). Sums over rows are cut into slices
// of fixed length whose partial results are added in order, so they do not depend on timing.
#include "gated_ff.cuh"

#ifndef FC_HOST_EMU
#include <algorithm>
#endif

namespace fc {

// rows of (n, m) per partial weight gradient: at most 256 slices
FC_HD FC_INLINE int64_t gated_slice(int64_t rows) { return rows > 2048 * 256 ? (rows + 255) / 256 : 2048; }

template <typename T>
struct GLoad {
  using A = typename Io<T>::Acc;
  FC_HD static FC_INLINE A at(const void* p, int64_t i) { return Io<T>::get(((const T*)p)[i]); }
};

// z: pre-activations, all ranks side by side: A = x_0 rows, B = Wg^T
template <typename T>
struct GateProduct {
  using A = typename Io<T>::Acc;
  GatedArgs a;
  A* out;  // (n, (L+1) H)
  int raw;  // 1: z itself, 0: s_a act(z)
  FC_HD FC_INLINE A lhs(int, int64_t r, int64_t k) const {
    return GLoad<T>::at(a.x, r * (a.L + 1) * (a.L + 1) * a.C + k);
  }
  FC_HD FC_INLINE A rhs(int, int64_t k, int c) const { return GLoad<T>::at(a.wg, (int64_t)c * a.C + k); }
  FC_HD FC_INLINE void put(int, int64_t r, int c, A v) const {
    const A* sc = (const A*)a.scales;
    const A z = sc[a.L + 1] * v + (a.bias ? GLoad<T>::at(a.bias, c) : A(0));
    out[r * (a.L + 1) * a.H + c] = raw ? z : sc[a.L + 2] * gated_act<A>(a.act, z);
  }
};

// v_k (grid z = k), times the gate where one is given
template <typename T>
struct ValueProduct {
  using A = typename Io<T>::Acc;
  GatedArgs a;
  const A* gate;  // (n, (L+1) H) or null
  A* out;         // null: a.y
  FC_HD FC_INLINE A lhs(int z, int64_t r, int64_t k) const {
    return GLoad<T>::at(a.x, (r * (a.L + 1) * (a.L + 1) + z) * a.C + k);
  }
  FC_HD FC_INLINE A rhs(int z, int64_t k, int c) const {
    return GLoad<T>::at(a.wv[gated_rank_of(z)], (int64_t)c * a.C + k);
  }
  FC_HD FC_INLINE void put(int z, int64_t r, int c, A v) const {
    const int l = gated_rank_of(z);
    A t = ((const A*)a.scales)[l] * v;
    const int64_t o = (r * (a.L + 1) * (a.L + 1) + z) * a.H + c;
    if (out) {
      out[o] = t;
    } else {
      t *= gate[(r * (a.L + 1) + l) * a.H + c];
      ((T*)a.y)[o] = Io<T>::put(t);
    }
  }
};

// dx_k: K = H products with Wv_l, and for k = 0 (L+1) H more with Wg
template <typename T>
struct InputGrad {
  using A = typename Io<T>::Acc;
  GatedArgs a;
  const A* dv;
  const A* dz;
  FC_HD FC_INLINE A lhs(int z, int64_t r, int64_t k) const {
    return k < a.H ? ((const A*)a.scales)[gated_rank_of(z)] * dv[(r * (a.L + 1) * (a.L + 1) + z) * a.H + k]
                   : ((const A*)a.scales)[a.L + 1] * dz[r * (a.L + 1) * a.H + k - a.H];
  }
  FC_HD FC_INLINE A rhs(int z, int64_t k, int c) const {
    return k < a.H ? GLoad<T>::at(a.wv[gated_rank_of(z)], k * a.C + c) : GLoad<T>::at(a.wg, (k - a.H) * a.C + c);
  }
  FC_HD FC_INLINE void put(int z, int64_t r, int c, A v) const {
    ((T*)a.gx)[(r * (a.L + 1) * (a.L + 1) + z) * a.C + c] = Io<T>::put(v);
  }
};

// one slice of a weight gradient: rows are hidden channels, the reduction runs over (n, m).
// grid z = (rank or gate rank) * slices + slice
template <typename T>
struct WeightGrad {
  using A = typename Io<T>::Acc;
  GatedArgs a;
  const A* d;  // dv (values) or dz (gates)
  int gates, slices;
  int64_t slice;  // rows per slice
  A* out;         // (ranks, slices, H, C)
  FC_HD FC_INLINE A lhs(int z, int64_t r, int64_t k) const { return d[atd(z, k) + r]; }
  FC_HD FC_INLINE A rhs(int z, int64_t k, int c) const { return GLoad<T>::at(a.x, atx(z, k) + c); }
  FC_HD FC_INLINE int64_t atd(int z, int64_t k) const {
    const int l = z / slices, comps = (a.L + 1) * (a.L + 1), m = 2 * l + 1;
    const int64_t q = (int64_t)(z % slices) * slice + k;
    return gates ? (q * (a.L + 1) + l) * a.H : ((q / m) * comps + l * l + q % m) * a.H;
  }
  FC_HD FC_INLINE int64_t atx(int z, int64_t k) const {
    const int l = z / slices, comps = (a.L + 1) * (a.L + 1), m = 2 * l + 1;
    const int64_t q = (int64_t)(z % slices) * slice + k;
    return gates ? q * comps * a.C : ((q / m) * comps + l * l + q % m) * a.C;
  }
  FC_HD FC_INLINE void put(int z, int64_t r, int c, A v) const { out[((int64_t)z * a.H + r) * a.C + c] = v; }
  // rows of (n, m) in slice z
  FC_HD FC_INLINE int64_t depth(int z) const {
    const int l = z / slices;
    const int64_t all = a.n * (gates ? 1 : 2 * l + 1), from = (int64_t)(z % slices) * slice;
    return all <= from ? 0 : (all - from < slice ? all - from : slice);
  }
};

#ifndef FC_HOST_EMU
constexpr int GT = 64, GK = 16;

// C(r, c) = sum_{k < K(z)} lhs(z, r, k) rhs(z, k, c) for r < R, c < N: 64 x 64 per block of 256
template <typename A, class F, class KF>
__global__ void __launch_bounds__(256) gated_gemm(const F f, const KF depth, int64_t R, int N) {
  __shared__ A as[GK][GT + 1], bs[GK][GT + 1];
  const int z = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t r0 = (int64_t)blockIdx.x * GT;
  const int64_t K = depth(z);
  // (the gates of 2^20 channels in four ranks have more column tiles than a grid is high)
  for (int c0 = blockIdx.y * GT; c0 < N; c0 += gridDim.y * GT) {
    A acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = A(0);
    for (int64_t k0 = 0; k0 < K; k0 += GK) {
#pragma unroll
      for (int t = 0; t < GT * GK / 256; ++t) {
        const int e = threadIdx.x + t * 256, k = e & (GK - 1), o = e >> 4;
        as[k][o] = (r0 + o < R && k0 + k < K) ? f.lhs(z, r0 + o, k0 + k) : A(0);
        bs[k][o] = (c0 + o < N && k0 + k < K) ? f.rhs(z, k0 + k, c0 + o) : A(0);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < GK; ++k) {
        A p[4], q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = as[k][ty + 16 * i];
          q[i] = bs[k][tx + 16 * i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += p[i] * q[j];
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r0 + ty + 16 * i < R && c0 + tx + 16 * j < N) f.put(z, r0 + ty + 16 * i, c0 + tx + 16 * j, acc[i][j]);
  }
}
#endif

struct FixedDepth {
  int64_t k, k0;  // depth for z > 0 and for z = 0
  FC_HD FC_INLINE int64_t operator()(int z) const { return z == 0 ? k0 : k; }
};
template <class F>
struct OwnDepth {
  F f;
  FC_HD FC_INLINE int64_t operator()(int z) const { return f.depth(z); }
};

template <typename A, class F, class KF>
static int run_gemm(const F& f, const KF& depth, int64_t R, int N, int zs, cudaStream_t s) {
  if (R <= 0 || N <= 0 || zs <= 0) return 0;
#ifndef FC_HOST_EMU
  const dim3 grid((unsigned)((R + GT - 1) / GT), (unsigned)std::min((N + GT - 1) / GT, 65535), (unsigned)zs);
  gated_gemm<A><<<grid, 256, 0, s>>>(f, depth, R, N);
  return fc_launched(1);
#else
  (void)s;
  for (int z = 0; z < zs; ++z) {
    const int64_t K = depth(z);
    for (int64_t r = 0; r < R; ++r)
      for (int c = 0; c < N; ++c) {
        A sum = A(0);
        for (int64_t k = 0; k < K; ++k) sum += f.lhs(z, r, k) * f.rhs(z, k, c);
        f.put(z, r, c, sum);
      }
  }
  return 0;
#endif
}

// v -> dv (in place), z -> dz (in place), for element e = (row, l, h)
template <typename T>
FC_HD FC_INLINE void gated_pointwise(const GatedArgs& a, typename Io<T>::Acc* v, typename Io<T>::Acc* z, int64_t e) {
  using A = typename Io<T>::Acc;
  const A* sc = (const A*)a.scales;
  const int64_t rl = e / a.H, row = rl / (a.L + 1);
  const int h = (int)(e - rl * a.H), l = (int)(rl - row * (a.L + 1));
  const A zz = z[e], gate = sc[a.L + 2] * gated_act<A>(a.act, zz);
  A sum = A(0);
  for (int m = 0; m < 2 * l + 1; ++m) {
    const int64_t o = (row * (a.L + 1) * (a.L + 1) + l * l + m) * a.H + h;
    const A g = GLoad<T>::at(a.gy, o);
    sum += g * v[o];
    v[o] = g * gate;
  }
  z[e] = sum * sc[a.L + 2] * gated_dact<A>(a.act, zz);
}

// sum of a weight gradient's slices, in order, scaled
template <typename T>
FC_HD FC_INLINE void gated_slices_one(const typename Io<T>::Acc* part, int slices, int64_t count,
                                      typename Io<T>::Acc scale, T* out, int64_t e) {
  using A = typename Io<T>::Acc;
  A sum = A(0);
  for (int t = 0; t < slices; ++t) sum += part[(int64_t)t * count + e];
  out[e] = Io<T>::put(scale * sum);
}

// a slice of the bias gradient
template <typename A>
FC_HD FC_INLINE void gated_bias_one(const A* dz, int64_t n, int64_t width, int64_t slice, int64_t t, int64_t c,
                                    A* part) {
  const int64_t r1 = n < (t + 1) * slice ? n : (t + 1) * slice;
  A sum = A(0);
  for (int64_t r = t * slice; r < r1; ++r) sum += dz[r * width + c];
  part[t * width + c] = sum;
}

#ifndef FC_HOST_EMU
template <typename T>
__global__ void __launch_bounds__(256) gated_pointwise_kernel(const GatedArgs a, typename Io<T>::Acc* v,
                                                              typename Io<T>::Acc* z, int64_t total) {
  for (int64_t e = blockIdx.x * (int64_t)256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256)
    gated_pointwise<T>(a, v, z, e);
}
template <typename T>
__global__ void __launch_bounds__(256) gated_slices_kernel(const typename Io<T>::Acc* part, int slices,
                                                           int64_t count, const typename Io<T>::Acc* scale, T* out) {
  const int64_t e = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (e < count) gated_slices_one<T>(part, slices, count, scale ? *scale : typename Io<T>::Acc(1), out, e);
}
template <typename A>
__global__ void __launch_bounds__(256) gated_bias_kernel(const A* dz, int64_t n, int64_t width, int64_t slice, A* part) {
  const int64_t c = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (c < width) gated_bias_one<A>(dz, n, width, slice, blockIdx.y, c, part);
}
#endif

template <typename T>
static int run_slices(const typename Io<T>::Acc* part, int slices, int64_t count, const typename Io<T>::Acc* scale,
                      T* out, cudaStream_t s) {
#ifndef FC_HOST_EMU
  gated_slices_kernel<T><<<(unsigned)((count + 255) / 256), 256, 0, s>>>(part, slices, count, scale, out);
  return fc_launched(1);
#else
  (void)s;
  for (int64_t e = 0; e < count; ++e)
    gated_slices_one<T>(part, slices, count, scale ? *scale : typename Io<T>::Acc(1), out, e);
  return 0;
#endif
}

struct SimpleWs {
  int64_t z, v, part, bytes;
  int64_t slice_v, slice_g;
  int slices_v, slices_g;
};

static SimpleWs simple_ws(int L, int C, int H, int64_t n, int64_t acc, int backward) {
  const int64_t comps = (int64_t)(L + 1) * (L + 1);
  SimpleWs w;
  w.slice_v = gated_slice(n * (2 * L + 1));
  w.slice_g = gated_slice(n);
  w.slices_v = (int)((n * (2 * L + 1) + w.slice_v - 1) / w.slice_v);
  w.slices_g = (int)((n + w.slice_g - 1) / w.slice_g);
  int64_t at = 0;
  auto take = [&](int64_t count) {
    const int64_t p = at;
    at += (count * acc + 15) & ~(int64_t)15;
    return p;
  };
  w.z = take(n * (L + 1) * H);
  w.v = backward ? take(n * comps * H) : 0;
  w.part = backward ? take((int64_t)(L + 1) * (w.slices_v > w.slices_g ? w.slices_v : w.slices_g) * H * C) : 0;
  w.bytes = at;
  return w;
}

int64_t gated_simple_ws(int L, int C, int H, int64_t n, int dtype, int backward) {
  return simple_ws(L, C, H, n, dtype == FC_F64 ? 8 : 4, backward).bytes;
}

template <typename T>
int gated_simple_fwd(const GatedArgs& a, cudaStream_t s) {
  using A = typename Io<T>::Acc;
  A* gate = (A*)a.ws;
  const FixedDepth depth{a.C, a.C};
  if (int rc = run_gemm<A>(GateProduct<T>{a, gate, 0}, depth, a.n, (a.L + 1) * a.H, 1, s)) return rc;
  return run_gemm<A>(ValueProduct<T>{a, gate, nullptr}, depth, a.n, a.H, (a.L + 1) * (a.L + 1), s);
}

template <typename T>
int gated_simple_bwd(const GatedArgs& a, cudaStream_t s) {
  using A = typename Io<T>::Acc;
  const int ranks = a.L + 1, comps = ranks * ranks;
  const SimpleWs w = simple_ws(a.L, a.C, a.H, a.n, sizeof(A), 1);
  A *z = (A*)((uint8_t*)a.ws + w.z), *v = (A*)((uint8_t*)a.ws + w.v), *part = (A*)((uint8_t*)a.ws + w.part);
  const A* sc = (const A*)a.scales;
  const FixedDepth depth{a.C, a.C};
  if (int rc = run_gemm<A>(GateProduct<T>{a, z, 1}, depth, a.n, ranks * a.H, 1, s)) return rc;
  if (int rc = run_gemm<A>(ValueProduct<T>{a, nullptr, v}, depth, a.n, a.H, comps, s)) return rc;
  const int64_t total = a.n * ranks * a.H;
#ifndef FC_HOST_EMU
  if (total > 0) {
    const int64_t b = (total + 255) / 256;
    gated_pointwise_kernel<T><<<(unsigned)std::min<int64_t>(b, 1 << 20), 256, 0, s>>>(a, v, z, total);
    if (int rc = fc_launched(1)) return rc;
  }
#else
  for (int64_t e = 0; e < total; ++e) gated_pointwise<T>(a, v, z, e);
#endif
  if (a.gx)
    if (int rc = run_gemm<A>(InputGrad<T>{a, v, z}, FixedDepth{a.H, (int64_t)(ranks + 1) * a.H}, a.n, a.C, comps, s))
      return rc;
  bool any = false;
  for (int l = 0; l < ranks; ++l) any = any || a.gwv[l];
  const int64_t count = (int64_t)a.H * a.C;
  if (any) {
    const WeightGrad<T> f{a, v, 0, w.slices_v, w.slice_v, part};
    if (int rc = run_gemm<A>(f, OwnDepth<WeightGrad<T>>{f}, a.H, a.C, ranks * w.slices_v, s)) return rc;
    for (int l = 0; l < ranks; ++l)
      if (a.gwv[l])
        if (int rc = run_slices<T>(part + (int64_t)l * w.slices_v * count, w.slices_v, count, sc + l, (T*)a.gwv[l], s))
          return rc;
  }
  if (a.gwg) {
    const WeightGrad<T> f{a, z, 1, w.slices_g, w.slice_g, part};
    if (int rc = run_gemm<A>(f, OwnDepth<WeightGrad<T>>{f}, a.H, a.C, ranks * w.slices_g, s)) return rc;
    for (int l = 0; l < ranks; ++l)
      if (int rc = run_slices<T>(part + (int64_t)l * w.slices_g * count, w.slices_g, count, sc + ranks,
                                 (T*)a.gwg + l * count, s))
        return rc;
  }
  if (a.gbias) {
    const int64_t width = (int64_t)ranks * a.H;
#ifndef FC_HOST_EMU
    if (w.slices_g > 0) {
      gated_bias_kernel<A><<<dim3((unsigned)((width + 255) / 256), (unsigned)w.slices_g), 256, 0, s>>>(z, a.n, width,
                                                                                                        w.slice_g, part);
      if (int rc = fc_launched(1)) return rc;
    }
#else
    for (int t = 0; t < w.slices_g; ++t)
      for (int64_t c = 0; c < width; ++c) gated_bias_one<A>(z, a.n, width, w.slice_g, t, c, part);
#endif
    if (int rc = run_slices<T>(part, w.slices_g, width, nullptr, (T*)a.gbias, s)) return rc;
  }
  return 0;
}

#define FC_GATED_INST(T)                                           \
  template int gated_simple_fwd<T>(const GatedArgs&, cudaStream_t); \
  template int gated_simple_bwd<T>(const GatedArgs&, cudaStream_t);
FC_GATED_INST(double)
#ifdef FC_HOST_EMU
FC_GATED_INST(float)
FC_GATED_INST(bf16_t)
#endif

}  // namespace fc
