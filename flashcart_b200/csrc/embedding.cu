// Embedding lookup with scaling, and its gradient by sorted tokens.
//
// Forward: out[i, :] = offset + scale * table[idx[i], :]. Bound by DRAM: the output write
// (element tables stay in L1 / L2). One 16-byte vector of the output per thread and step,
// four steps' loads in flight. Measured: 27,648 rows of 2,944 float32 channels 61 us (5.3 TB/s),
// 2^26 elements in rows of 64 62 us (4.4 TB/s).
//
// Backward: d_table[v, :] = scale * sum over {i : idx[i] = v} of grad[i, :], in an order
// fixed by the sizes alone (no atomics), so equal inputs give equal bits. The tokens are
// sorted once (stable least-significant-digit radix sort of (token, row) pairs, 8 bits a
// pass at most: one pass for up to 255 types), then the sorted positions are cut into
// chunks of Lc. A chunk's lane group walks its rows in order with the running sum in
// registers; a token whose rows lie inside one chunk is written at once, a token that spans
// chunks leaves one partial sum per chunk in the workspace, and a second kernel adds the
// partial sums. Bound by the one read of grad; the sort moves 8 to 16 bytes per row and
// pass. Sums are float (double for 64-bit tables), rounded once. Measured: 1,492,998 rows of 16
// float32 channels into 4 types 55 us (sort 18, sums 29, joining 9; 16 us for one read of grad at
// the copy rate); 65,537 rows of 512 bfloat16 channels into 50,000 types 76 us (sort 28, bounds and
// zero rows 14, sums 22, joining 12).
//
// An index outside [0, n_types) raises FC_DEV_BAD_INDEX; its output row is written as zeros
// and its gradient row is ignored (it sorts behind every token as key n_types).
#include <algorithm>
#include <atomic>
#include <cstring>

#include "fc_vec.cuh"

namespace fc {

template <typename T>
FC_HD FC_INLINE T embed_value(T t, typename Io<T>::Acc scale, typename Io<T>::Acc offset) {
  return Io<T>::put(offset + scale * Io<T>::get(t));
}

#ifdef FC_HOST_EMU

int64_t embed_bwd_workspace(int64_t, int64_t, int64_t, int) { return 16; }

template <typename T>
int embed_fwd(const void* table_, int64_t V, int64_t D, const int64_t* idx, int64_t R, double scale, double offset,
              void* out_, int* status, cudaStream_t) {
  const T* table = (const T*)table_;
  T* out = (T*)out_;
  using A = typename Io<T>::Acc;
  for (int64_t i = 0; i < R; ++i) {
    const bool ok = idx[i] >= 0 && idx[i] < V;
    if (!ok) fc_flag(status, FC_DEV_BAD_INDEX);
    for (int64_t d = 0; d < D; ++d)
      out[i * D + d] = ok ? embed_value<T>(table[idx[i] * D + d], (A)scale, (A)offset) : Io<T>::put(A(0));
  }
  return 0;
}

template <typename T>
int embed_bwd(const void* grad_, const int64_t* idx, int64_t R, int64_t V, int64_t D, double scale, void* ws,
              void* d_table, int* status, cudaStream_t) {
  (void)ws;
  using A = typename Io<T>::Acc;
  const T* grad = (const T*)grad_;
  for (int64_t i = 0; i < R; ++i)
    if (idx[i] < 0 || idx[i] >= V) fc_flag(status, FC_DEV_BAD_INDEX);
  for (int64_t v = 0; v < V; ++v)
    for (int64_t d = 0; d < D; ++d) {
      A s = A(0);
      for (int64_t i = 0; i < R; ++i)
        if (idx[i] == v) s += Io<T>::get(grad[i * D + d]);
      ((T*)d_table)[v * D + d] = Io<T>::put((A)scale * s);
    }
  return 0;
}

#else

// ------------------------------------------------------------------------------ forward

// Rows of whole, aligned 16-byte vectors: unit = one vector, per_row of them in a row. Four
// units per thread and step; the next step's indices are asked for before this step's rows are
// (the index comes from DRAM, the row from L1 or L2).
template <typename T, typename I>
__global__ void __launch_bounds__(256) embed_fwd_vec(const T* __restrict__ table, int64_t V, int per_row,
                                                     const int64_t* __restrict__ idx, int64_t units,
                                                     typename Io<T>::Acc scale, typename Io<T>::Acc offset,
                                                     T* __restrict__ out, int* status) {
  constexpr int NV = Io<T>::VEC, UN = 4;
  const I total = (I)units, step = (I)gridDim.x * (256 * UN);
  int64_t t[UN], at[UN];
  auto ask = [&](I u0, int64_t* tt, int64_t* cc) {
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      const I u = u0 + j * 256;
      tt[j] = -1;
      cc[j] = 0;
      if (u < total) {
        const I row = u / (I)per_row;
        cc[j] = (int64_t)(u - row * (I)per_row);
        tt[j] = __ldg(idx + row);
      }
    }
  };
  I u0 = (I)blockIdx.x * (256 * UN) + threadIdx.x;
  ask(u0, t, at);
  for (; u0 < total; u0 += step) {
    int64_t tn[UN], an[UN];
    ask(u0 + step, tn, an);
    Pack<T, NV> v[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j)
      if (u0 + j * 256 < total) {
        if (t[j] < 0 || t[j] >= V) {
          if (at[j] == 0) fc_flag(status, FC_DEV_BAD_INDEX);
          t[j] = -1;
        } else {
          v[j].load(table + (t[j] * per_row + at[j]) * NV);
        }
      }
#pragma unroll
    for (int j = 0; j < UN; ++j)
      if (u0 + j * 256 < total) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          v[j].set(k, t[j] >= 0 ? embed_value<T>(v[j].at(k), scale, offset) : Io<T>::put(0));
        v[j].store(out + (int64_t)(u0 + j * 256) * NV);
      }
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      t[j] = tn[j];
      at[j] = an[j];
    }
  }
}

// Rows of any length from a vector's on, of a table that has rows (a wrong index reads row 0, and what
// it reads is not written): a thread writes aligned vectors of the flat output, whose
// elements belong to one row or two, so every element is read from one of two places without a
// branch (a warp's lanes cross rows at different elements). Two vectors per thread and step. 67 M
// elements in rows of 63: 81 us in float32 and 69 in bfloat16 (with a row test per element, as
// embed_fwd_flat below has it, 154 and 133).
template <typename T>
__global__ void __launch_bounds__(256) embed_fwd_odd(const T* __restrict__ table, uint32_t V, uint32_t D,
                                                     const int64_t* __restrict__ idx, uint32_t R, uint32_t total,
                                                     typename Io<T>::Acc scale, typename Io<T>::Acc offset,
                                                     T* __restrict__ out, int* status) {
  constexpr int NV = Io<T>::VEC, UN = 2;
  const uint32_t units = (total + NV - 1) / NV, step = gridDim.x * (256 * UN);
  for (uint32_t u0 = blockIdx.x * (256 * UN) + threadIdx.x; u0 < units; u0 += step) {
    T v[UN][NV];
    bool ok0[UN], ok1[UN];
    uint32_t left[UN];  // elements of the vector in its first row
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      const uint32_t u = u0 + j * 256;
      if (u < units) {
        const uint32_t row = u * NV / D, col = u * NV - row * D;
        const int64_t t0 = __ldg(idx + row), t1 = __ldg(idx + min(row + 1, R - 1));
        left[j] = D - col;
        ok0[j] = t0 >= 0 && t0 < V;
        ok1[j] = t1 >= 0 && t1 < V;
        if (!ok0[j] || (!ok1[j] && left[j] < NV)) fc_flag(status, FC_DEV_BAD_INDEX);
        // both places as if the vector began there; a wrong index reads row 0
        const uint32_t at0 = (ok0[j] ? (uint32_t)t0 : 0u) * D + col, at1 = (ok1[j] ? (uint32_t)t1 : 0u) * D - left[j];
#pragma unroll
        for (int k = 0; k < NV; ++k)
          // (behind the last row nothing is written: such an element reads the row's last)
          v[j][k] = table[(uint32_t)k < left[j] ? at0 + k : row + 1 < R ? at1 + k : at0];
      }
    }
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      const uint32_t u = u0 + j * 256;
      if (u < units) {
        Pack<T, NV> w;
#pragma unroll
        for (int k = 0; k < NV; ++k)
          w.set(k, ((uint32_t)k < left[j] ? ok0[j] : ok1[j]) ? embed_value<T>(v[j][k], scale, offset) : Io<T>::put(0));
        if (u * NV + NV <= total) {
          w.store(out + (int64_t)u * NV);
        } else {
          for (int k = 0; k < NV && u * NV + k < total; ++k) out[(int64_t)u * NV + k] = w.at(k);
        }
      }
    }
  }
}

// Any row length and size: a thread writes one aligned vector of the flat output, whose elements may
// belong to several rows (NV = 1 where the output itself is not 16-byte aligned).
template <typename T, int NV>
__global__ void __launch_bounds__(256) embed_fwd_flat(const T* __restrict__ table, int64_t V, int64_t D,
                                                      const int64_t* __restrict__ idx, int64_t total,
                                                      typename Io<T>::Acc scale, typename Io<T>::Acc offset,
                                                      T* __restrict__ out, int* status) {
  const int64_t units = (total + NV - 1) / NV;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (int64_t)gridDim.x * 256) {
    const int64_t e0 = u * NV;
    int64_t row = total < ((int64_t)1 << 32) ? (int64_t)((uint32_t)e0 / (uint32_t)D) : e0 / D;
    int64_t col = e0 - row * D;
    Pack<T, NV> v;
    int64_t t = __ldg(idx + row);
    bool ok = t >= 0 && t < V;
    if (!ok) fc_flag(status, FC_DEV_BAD_INDEX);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (e0 + k < total) {
        if (col == D) {
          col = 0;
          t = __ldg(idx + ++row);
          ok = t >= 0 && t < V;
          if (!ok) fc_flag(status, FC_DEV_BAD_INDEX);
        }
        v.set(k, ok ? embed_value<T>(table[t * D + col], scale, offset) : Io<T>::put(0));
        ++col;
      }
    }
    if (e0 + NV <= total) {
      v.store(out + e0);
    } else {
      for (int k = 0; k < NV && e0 + k < total; ++k) out[e0 + k] = v.at(k);
    }
  }
}

template <typename T>
int embed_fwd(const void* table_, int64_t V, int64_t D, const int64_t* idx, int64_t R, double scale, double offset,
              void* out_, int* status, cudaStream_t s) {
  using A = typename Io<T>::Acc;
  constexpr int NV = Io<T>::VEC;
  const T* table = (const T*)table_;
  T* out = (T*)out_;
  const uintptr_t at = reinterpret_cast<uintptr_t>(table), ao = reinterpret_cast<uintptr_t>(out);
  if (D % NV == 0 && D / NV <= 0x7fffffff && !((at | ao) & 15)) {
    const int64_t units = R * (D / NV), b = (units + 1023) / 1024;
    const unsigned grid = (unsigned)(b < 148 * 4 ? b : 148 * 4);  // four blocks per SM stay and walk on
    if (units + 2 * (int64_t)grid * 1024 < ((int64_t)1 << 32))
      embed_fwd_vec<T, uint32_t><<<grid, 256, 0, s>>>(table, V, (int)(D / NV), idx, units, (A)scale, (A)offset, out,
                                                      status);
    else
      embed_fwd_vec<T, uint64_t><<<grid, 256, 0, s>>>(table, V, (int)(D / NV), idx, units, (A)scale, (A)offset, out,
                                                      status);
  } else if (V > 0 && D >= NV && !(ao & 15) && R * D < ((int64_t)1 << 31) && V * D < ((int64_t)1 << 31)) {
    const int64_t b = (R * D + 512 * NV - 1) / (512 * NV);
    const unsigned grid = (unsigned)(b < 148 * 16 ? b : 148 * 16);
    embed_fwd_odd<T><<<grid, 256, 0, s>>>(table, (uint32_t)V, (uint32_t)D, idx, (uint32_t)R, (uint32_t)(R * D),
                                          (A)scale, (A)offset, out, status);
  } else {
    const bool aligned = !(ao & 15);
    const int64_t units = aligned ? (R * D + NV - 1) / NV : R * D, b = (units + 255) / 256;
    const unsigned grid = (unsigned)(b < (1 << 20) ? b : (1 << 20));
    if (aligned)
      embed_fwd_flat<T, NV><<<grid, 256, 0, s>>>(table, V, D, idx, R * D, (A)scale, (A)offset, out, status);
    else
      embed_fwd_flat<T, 1><<<grid, 256, 0, s>>>(table, V, D, idx, R * D, (A)scale, (A)offset, out, status);
  }
  return fc_launched(1);
}

// ------------------------------------------------------------------------------ token sort

constexpr int SORT_THREADS = 256, SORT_ITEMS = 8, SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int SMALL_THREADS = 1024, SMALL_ROWS = 8192;  // one block sorts this many in shared memory

struct SortPlan {
  int passes, bits, digits;  // digits = values of one pass's digit
};

static SortPlan sort_plan(int64_t V) {
  int need = 1;
  while (((int64_t)1 << need) <= V) ++need;  // keys 0 .. V
  SortPlan p;
  p.passes = (need + 7) / 8;
  p.bits = (need + p.passes - 1) / p.passes;
  p.digits = p.passes == 1 ? (int)(V + 1) : 1 << p.bits;
  return p;
}

__device__ __forceinline__ int token_key(const int64_t* idx, int64_t i, int64_t V, int* status) {
  const int64_t t = __ldg(idx + i);
  if (t >= 0 && t < V) return (int)t;
  fc_flag(status, FC_DEV_BAD_INDEX);
  return (int)V;
}

// Pass over one digit, 1: digit counts of every tile. FIRST reads the caller's indices.
template <bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS) sort_count(const int64_t* __restrict__ idx,
                                                           const int* __restrict__ keys, int64_t R, int64_t V,
                                                           int shift, int bits, int digits, int* __restrict__ hist,
                                                           int* status) {
  __shared__ int h[256];
  for (int d = threadIdx.x; d < digits; d += SORT_THREADS) h[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * SORT_TILE;
#pragma unroll
  for (int j = 0; j < SORT_ITEMS; ++j) {
    const int64_t i = base + j * SORT_THREADS + threadIdx.x;
    const bool in = i < R;
    const int k = in ? (FIRST ? token_key(idx, i, V, status) : keys[i]) : 0;
    const int d = in ? (k >> shift) & ((1 << bits) - 1) : 256;
    // one shared-memory add per distinct digit of the warp: few types would otherwise
    // serialise on a few counters
    const unsigned same = __match_any_sync(0xffffffffu, d);
    if (in && (int)(threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&h[d], __popc(same));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += SORT_THREADS) hist[(int64_t)d * gridDim.x + blockIdx.x] = h[d];
}

// Exclusive sum of one value per thread of a block of WARPS warps (sh: WARPS ints); total in
// the second result. Ends with a block barrier.
template <int WARPS>
__device__ __forceinline__ int block_exclusive(int v, int* sh, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int t = sh[w];
    if (w < warp) before += t;
    total += t;
  }
  __syncthreads();
  return before + x - v;
}

// 2: block d turns digit d's counts into exclusive sums over the tiles, and writes its total.
__global__ void __launch_bounds__(256) sort_scan(int* __restrict__ hist, int tiles, int* __restrict__ totals) {
  __shared__ int sh[8];
  int* row = hist + (int64_t)blockIdx.x * tiles;
  int carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + threadIdx.x;
    int total;
    const int ex = block_exclusive<8>(t < tiles ? row[t] : 0, sh, total);
    if (t < tiles) row[t] = carry + ex;
    carry += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Stable ranks of a warp's next 32 digits among those before them in the warp's segment:
// counters[d] holds how many digits d the warp has passed. d = 256 marks no element.
__device__ __forceinline__ int warp_rank(int d, int* counters) {
  const unsigned lane = threadIdx.x & 31;
  const unsigned same = __match_any_sync(0xffffffffu, d);
  const int before = d < 256 ? counters[d] : 0;
  __syncwarp();
  if (d < 256 && (int)lane == __ffs(same) - 1) counters[d] = before + __popc(same);
  __syncwarp();
  return before + __popc(same & ((1u << lane) - 1u));
}

// 3: every (key, row) to its place. Warp w of a tile owns a contiguous eighth of it.
template <bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS)
    sort_scatter(const int64_t* __restrict__ idx, const int* __restrict__ keys, const int* __restrict__ order,
                 int64_t R, int64_t V, int shift, int bits, int digits, const int* __restrict__ hist,
                 const int* __restrict__ totals, int* __restrict__ keys_out, int* __restrict__ order_out,
                 int* __restrict__ start, int scanned) {
  __shared__ int counters[SORT_THREADS / 32][256];
  __shared__ int base[256];
  __shared__ int sh[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int j = threadIdx.x; j < (SORT_THREADS / 32) * 256; j += SORT_THREADS) (&counters[0][0])[j] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * SORT_TILE + warp * (SORT_TILE / 8) + lane;
  int key[SORT_ITEMS], loc[SORT_ITEMS];
#pragma unroll
  for (int j = 0; j < SORT_ITEMS; ++j) {
    const int64_t i = first + j * 32;
    key[j] = i < R ? (FIRST ? token_key(idx, i, V, nullptr) : keys[i]) : -1;
  }
#pragma unroll
  for (int j = 0; j < SORT_ITEMS; ++j)
    loc[j] = warp_rank(key[j] >= 0 ? (key[j] >> shift) & ((1 << bits) - 1) : 256, counters[warp]);
  int all, d0 = 0, ahead = 0;  // of this thread's digit: in all tiles, in the tiles before this one
  if (threadIdx.x < digits) {
    const int* row = hist + (int64_t)threadIdx.x * gridDim.x;
    if (scanned) {
      d0 = totals[threadIdx.x];
      ahead = row[blockIdx.x];
    } else {
      for (int t = 0; t < (int)gridDim.x; ++t) {
        const int c = row[t];
        d0 += c;
        if (t < (int)blockIdx.x) ahead += c;
      }
    }
  }
  const int before = block_exclusive<8>(d0, sh, all);  // its barriers also end the ranking
  // a sort of one pass: the digits are the tokens, and their totals place them
  if (start && blockIdx.x == 0 && threadIdx.x < digits) start[threadIdx.x] = before;
  if (threadIdx.x < digits) {
    base[threadIdx.x] = before + ahead;
    int sum = 0;
    for (int w = 0; w < SORT_THREADS / 32; ++w) {
      const int t = counters[w][threadIdx.x];
      counters[w][threadIdx.x] = sum;
      sum += t;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < SORT_ITEMS; ++j)
    if (key[j] >= 0) {
      const int64_t i = first + j * 32;
      const int d = (key[j] >> shift) & ((1 << bits) - 1);
      const int to = base[d] + counters[warp][d] + loc[j];
      keys_out[to] = key[j];
      order_out[to] = FIRST ? (int)i : order[i];
    }
}

// Bytes of sort_small's dynamic shared memory: two buffers of keys and of rows, the warps' counters.
static constexpr int small_bytes(int R) { return (4 * ((R + 31) & ~31) + (SMALL_THREADS / 32) * 256) * 4; }

// The whole sort of up to SMALL_ROWS tokens in one block: the same three steps a pass, with
// keys and rows ping-ponged in shared memory (one launch where latency is all that counts).
__global__ void __launch_bounds__(SMALL_THREADS) sort_small(const int64_t* __restrict__ idx, int R, int64_t V,
                                                            int passes, int bits, int* __restrict__ keys_out,
                                                            int* __restrict__ order_out, int* __restrict__ start,
                                                            int* status) {
  extern __shared__ int sm[];
  constexpr int WARPS = SMALL_THREADS / 32;
  __shared__ int sh[WARPS];
  __shared__ int base[256];
  const int cap = (R + 31) & ~31;
  int* kbuf[2] = {sm, sm + cap};
  int* obuf[2] = {sm + 2 * cap, sm + 3 * cap};
  int* counters = sm + 4 * cap;  // [WARPS][256]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_warp = ((R + WARPS - 1) / WARPS + 31) & ~31;
  const int lo = min(R, warp * per_warp), hi = min(R, lo + per_warp);
  for (int i = threadIdx.x; i < R; i += SMALL_THREADS) {
    kbuf[0][i] = token_key(idx, i, V, status);
    obuf[0][i] = i;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits, mask = (1 << bits) - 1;
    const int *ki = kbuf[p & 1], *oi = obuf[p & 1];
    const bool last = p == passes - 1;
    int* ko = last ? keys_out : kbuf[(p + 1) & 1];
    int* oo = last ? order_out : obuf[(p + 1) & 1];
    for (int j = threadIdx.x; j < WARPS * 256; j += SMALL_THREADS) counters[j] = 0;
    __syncthreads();
    int loc[SMALL_ROWS / SMALL_THREADS];
#pragma unroll
    for (int j = 0; j < SMALL_ROWS / SMALL_THREADS; ++j) {
      const int i = lo + j * 32 + lane;
      if (lo + j * 32 < hi) loc[j] = warp_rank(i < hi ? (ki[i] >> shift) & mask : 256, counters + warp * 256);
    }
    __syncthreads();
    int sum = 0;
    if (threadIdx.x < 256)
      for (int w = 0; w < WARPS; ++w) {
        const int t = counters[w * 256 + threadIdx.x];
        counters[w * 256 + threadIdx.x] = sum;
        sum += t;
      }
    int all;
    const int before = block_exclusive<WARPS>(sum, sh, all);
    if (threadIdx.x < 256) base[threadIdx.x] = before;
    if (passes == 1 && threadIdx.x <= V) start[threadIdx.x] = before;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SMALL_ROWS / SMALL_THREADS; ++j) {
      const int i = lo + j * 32 + lane;
      if (i < hi) {
        const int k = ki[i], d = (k >> shift) & mask;
        const int to = base[d] + counters[warp * 256 + d] + loc[j];
        ko[to] = k;
        oo[to] = oi[i];
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------ segment sums

__device__ __forceinline__ int lower_bound(const int* __restrict__ keys, int n, int v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(keys + mid) < v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// Zeros in row[0 .. D) by the lanes of a warp.
template <typename T>
__device__ __forceinline__ void zero_row(T* row, int64_t D, bool vec, int lane, int step) {
  if (vec) {
    Pack<T, Io<T>::VEC> z;
    z.raw = make_uint4(0, 0, 0, 0);
    for (int64_t d = (int64_t)lane * Io<T>::VEC; d < D; d += (int64_t)step * Io<T>::VEC) z.store(row + d);
  } else {
    for (int64_t d = lane; d < D; d += step) row[d] = Io<T>::put(0);
  }
}

// start[v] = first sorted position of token v (v <= V); zero rows for tokens without any.
template <typename T>
__global__ void __launch_bounds__(256) embed_bounds(const int* __restrict__ keys, int R, int64_t V, int64_t D,
                                                    int vec, int* __restrict__ start, T* __restrict__ d_table) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int lane = threadIdx.x & 31;
  int a = 0, b = 0;
  if (v <= V) {
    a = lower_bound(keys, R, (int)v);
    start[v] = a;
  }
  // the next token's start is the next lane's own
  b = __shfl_down_sync(0xffffffffu, a, 1);
  if (lane == 31 && v < V) b = lower_bound(keys, R, (int)v + 1);
  unsigned none = __ballot_sync(0xffffffffu, v < V && a == b);
  while (none) {
    const int l = __ffs(none) - 1;
    none &= none - 1;
    zero_row<T>(d_table + (v - lane + l) * D, D, vec, lane, 32);
  }
}

struct SumPlan {
  int per;         // columns per lane
  int lanes;       // lanes of a group, a power of two up to 32
  int col_tiles;   // groups side by side over a row
  int Lc;          // sorted positions per chunk
  int64_t chunks;
  int64_t Dp;      // elements of a partial row
};

template <typename T>
static SumPlan sum_plan(int64_t R, int64_t D, bool vec) {
  SumPlan p;
  p.per = vec ? Io<T>::VEC : 4;
  p.lanes = 1;
  while (p.lanes < 32 && (int64_t)p.lanes * p.per < D) p.lanes *= 2;
  p.col_tiles = (int)((D + (int64_t)p.lanes * p.per - 1) / ((int64_t)p.lanes * p.per));
  // chunks just long enough that the lane groups together are 512 threads per SM, which with
  // eight rows in flight each cover the memory latency: shorter chunks write and re-read more
  // partial sums, longer ones leave too few loads in flight
  const int64_t fill = R * p.lanes * p.col_tiles / (148 * 512);
  p.Lc = (int)(fill < 16 ? 16 : fill > 256 ? 256 : (fill + 7) / 8 * 8);
  p.chunks = (R + p.Lc - 1) / p.Lc;
  p.Dp = (D + 7) / 8 * 8;
  return p;
}

// Partial slots of a chunk: 0 for a run that began before the chunk, 1 for one that begins
// in it and goes on behind it.
template <typename T, int PER, bool VECT>
__global__ void __launch_bounds__(256)
    embed_sum(const T* __restrict__ grad, const int* __restrict__ keys, const int* __restrict__ order,
              const int* __restrict__ start, int R, int64_t V, int64_t D, int Lc, int64_t chunks, int lanes,
              int col_tiles, typename Io<T>::Acc scale, typename Io<T>::Acc* __restrict__ partial, int64_t Dp,
              T* __restrict__ d_table) {
  using A = typename Io<T>::Acc;
  constexpr int U = 8;  // rows in flight
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
  const int64_t chunk = group / col_tiles;
  if (chunk >= chunks) return;
  const int64_t col0 = (group - chunk * col_tiles) * (int64_t)lanes * PER + (VECT ? lane * PER : lane);
  const int p0 = (int)(chunk * Lc), p1 = (int)min((int64_t)R, chunk * Lc + Lc);
  A acc[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) acc[k] = A(0);
  auto flush = [&](int key, int a, int b) {
    if (key >= V) return;
    const bool left = a == p0 && __ldg(start + key) < p0;
    const bool right = b == p1 && __ldg(start + key + 1) > p1;
    if (!left && !right) {
      T* row = d_table + (int64_t)key * D;
      if constexpr (VECT) {
        if (col0 < D) {
          Pack<T, PER> v;
#pragma unroll
          for (int k = 0; k < PER; ++k) v.set(k, Io<T>::put(scale * acc[k]));
          v.store(row + col0);
        }
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (col0 + k * lanes < D) row[col0 + k * lanes] = Io<T>::put(scale * acc[k]);
      }
    } else {
      A* row = partial + (chunk * 2 + (left ? 0 : 1)) * Dp;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int64_t c = col0 + (VECT ? k : k * lanes);
        if (c < D) row[c] = acc[k];
      }
    }
  };
  int cur = __ldg(keys + p0), from = p0;
  int key[U], row[U], key_next[U], row_next[U];
  auto ask = [&](int p, int* k, int* r) {  // the next rows' numbers come while this batch is added
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = min(p + u, p1 - 1);
      k[u] = __ldg(keys + q);
      r[u] = __ldg(order + q);
    }
  };
  ask(p0, key_next, row_next);
  for (int p = p0; p < p1; p += U) {
    Pack<T, VECT ? PER : 1> v[U][VECT ? 1 : PER];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      key[u] = key_next[u];
      row[u] = row_next[u];
    }
    if (p + U < p1) ask(p + U, key_next, row_next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* g = grad + (int64_t)row[u] * D;
      if constexpr (VECT) {
        if (col0 < D) v[u][0].load_stream(g + col0);
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (col0 + k * lanes < D) v[u][k].load_stream(g + col0 + k * lanes);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u < p1) {
        if (key[u] != cur) {
          flush(cur, from, p + u);
          cur = key[u];
          from = p + u;
#pragma unroll
          for (int k = 0; k < PER; ++k) acc[k] = A(0);
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) acc[k] += Io<T>::get(VECT ? v[u][0].at(VECT ? k : 0) : v[u][VECT ? 0 : k].at(0));
      }
    }
  }
  flush(cur, from, p1);
}

constexpr int MAX_SLICES = 16;

// Tokens that span chunks: their partial sums added, a token at a time per block. The block
// looks at `per_block` candidates (tokens, or chunks in which such a token ends, whichever
// are fewer) and adds each one's partial rows with fixed strides and a fixed tree. With few
// types (slices > 1, one candidate per block) blockIdx.z takes a slice of the chunks and leaves
// its sum to embed_finish. Candidates without any row get their zeros here when they are tokens.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
    embed_combine(const typename Io<T>::Acc* __restrict__ partial, const int* __restrict__ keys,
                  const int* __restrict__ start, int R, int64_t V, int64_t D, int64_t Dp, int Lc, int64_t chunks,
                  int by_token, int per_block, int lanes, int slices, int vec, typename Io<T>::Acc scale,
                  typename Io<T>::Acc* __restrict__ sums, T* __restrict__ d_table) {
  using A = typename Io<T>::Acc;
  constexpr int PC = 16 / sizeof(A);
  __shared__ int list[THREADS][3];
  __shared__ int count;
  __shared__ A red[THREADS][PC];
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const int64_t cand = (int64_t)blockIdx.x * per_block + threadIdx.x;
  if (threadIdx.x < per_block && cand < (by_token ? V : chunks)) {
    const int64_t v = by_token ? cand : keys[cand * Lc];
    if (v < V) {
      const int a = start[v], b = start[v + 1];
      if (b > a) {
        const int cf = a / Lc, cl = (b - 1) / Lc;
        if (cf < cl && (by_token || cl == cand)) {
          const int at = atomicAdd(&count, 1);  // the order of the list does not reach the results
          list[at][0] = (int)v;
          list[at][1] = cf;
          list[at][2] = cl;
        }
      } else if (by_token) {
        const int at = atomicAdd(&count, 1);
        list[at][0] = (int)v;
        list[at][1] = 0;
        list[at][2] = -1;
      }
    }
  }
  __syncthreads();
  const int n = count, lane = threadIdx.x & (lanes - 1), g = threadIdx.x / lanes, groups = THREADS / lanes;
  const int64_t col_tiles = (Dp + (int64_t)lanes * PC - 1) / ((int64_t)lanes * PC);
  // (64-bit rows may have more tiles than a grid is high)
  for (int64_t tile = blockIdx.y; tile < col_tiles; tile += gridDim.y) {
    const int64_t col = (tile * lanes + lane) * PC;
    for (int e = 0; e < n; ++e) {
      const int64_t v = list[e][0];
      const int cf = list[e][1], cl = list[e][2];
      if (cl < 0) {
        if (tile == 0 && blockIdx.z == 0)
          zero_row<T>(d_table + v * D, D, vec, threadIdx.x, THREADS);
        continue;
      }
      const int len = cl - cf + 1, c0 = cf + (int)((int64_t)len * blockIdx.z / slices),
                c1 = cf + (int)((int64_t)len * (blockIdx.z + 1) / slices);
      A acc[PC];
#pragma unroll
      for (int k = 0; k < PC; ++k) acc[k] = A(0);
      if (col < Dp) {
#pragma unroll 8
        for (int c = c0 + g; c < c1; c += groups) {
          Pack<A, PC> q;
          q.load(partial + ((int64_t)c * 2 + (c == cf ? 1 : 0)) * Dp + col);
#pragma unroll
          for (int k = 0; k < PC; ++k) acc[k] += q.at(k);
        }
      }
#pragma unroll
      for (int k = 0; k < PC; ++k) red[threadIdx.x][k] = acc[k];
      for (int half = groups / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (g < half)
#pragma unroll
          for (int k = 0; k < PC; ++k) red[threadIdx.x][k] += red[threadIdx.x + half * lanes][k];
      }
      __syncthreads();
      if (g == 0)
#pragma unroll
        for (int k = 0; k < PC; ++k)
          if (col + k < D) {
            if (slices > 1) sums[(v * slices + blockIdx.z) * Dp + col + k] = red[threadIdx.x][k];
            else d_table[v * D + col + k] = Io<T>::put(scale * red[threadIdx.x][k]);
          }
      __syncthreads();
    }
  }
}

// The slices of tokens that span chunks, added in order.
template <typename T>
__global__ void __launch_bounds__(256) embed_finish(const typename Io<T>::Acc* __restrict__ sums,
                                                    const int* __restrict__ start, int64_t V, int64_t D, int64_t Dp,
                                                    int Lc, int slices, typename Io<T>::Acc scale,
                                                    T* __restrict__ d_table) {
  const int64_t v = blockIdx.x, col = (int64_t)blockIdx.y * 256 + threadIdx.x;
  const int a = start[v], b = start[v + 1];
  if (col >= D || b <= a || a / Lc == (b - 1) / Lc) return;
  typename Io<T>::Acc t = 0;
  for (int z = 0; z < slices; ++z) t += sums[(v * slices + z) * Dp + col];
  d_table[v * D + col] = Io<T>::put(scale * t);
}

// ------------------------------------------------------------------------------ host

struct EmbedWs {
  int64_t keys[2], order[2], hist, totals, start, partial, sums, bytes;
};

// The largest sort's shared memory is allowed once per device: the limit is the kernel's, not the
// call's, and other host threads launch it with other sizes.
static bool sort_small_ready() {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (done[dev].load(std::memory_order_acquire)) return true;
  if (cudaFuncSetAttribute(sort_small, cudaFuncAttributeMaxDynamicSharedMemorySize, small_bytes(SMALL_ROWS)) !=
      cudaSuccess)
    return false;
  done[dev].store(true, std::memory_order_release);
  return true;
}

// Blocks that share a token's chunks: several where the types alone would leave SMs idle, but
// at least 64 chunks each.
static int combine_slices(int64_t V, const SumPlan& sp) {
  if (V > sp.chunks) return 1;
  const int64_t blocks = V * ((sp.Dp + 127) / 128), most = sp.chunks / (V * 64);
  const int64_t z = 148 * 2 / blocks < most ? 148 * 2 / blocks : most;
  return (int)(z < 1 ? 1 : z > MAX_SLICES ? MAX_SLICES : z);
}

static int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }

template <typename T>
static EmbedWs embed_ws(int64_t R, int64_t V, int64_t D, const SumPlan& sp) {
  const SortPlan so = sort_plan(V);
  const int64_t tiles = (R + SORT_TILE - 1) / SORT_TILE;
  EmbedWs w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += up16(bytes);
    return p;
  };
  for (int k = 0; k < 2; ++k) {
    w.keys[k] = take(R * 4);
    w.order[k] = take(R * 4);
  }
  w.hist = take(tiles * so.digits * 4);
  w.totals = take(so.digits * 4);
  w.start = take((V + 1) * 4);
  w.partial = take(sp.chunks * 2 * sp.Dp * (int64_t)sizeof(typename Io<T>::Acc));
  w.sums = take(combine_slices(V, sp) > 1 ? V * MAX_SLICES * sp.Dp * (int64_t)sizeof(typename Io<T>::Acc) : 0);
  w.bytes = at;
  return w;
}

template <typename T>
static int64_t embed_ws_bytes(int64_t R, int64_t V, int64_t D) {
  // the larger of both column layouts: the choice depends on the tensors' alignment
  const int64_t a = embed_ws<T>(R, V, D, sum_plan<T>(R, D, true)).bytes;
  const int64_t b = embed_ws<T>(R, V, D, sum_plan<T>(R, D, false)).bytes;
  return a > b ? a : b;
}

int64_t embed_bwd_workspace(int64_t R, int64_t V, int64_t D, int dtype) {
  if (dtype == FC_F64) return embed_ws_bytes<double>(R, V, D);
  return dtype == FC_BF16 ? embed_ws_bytes<bf16_t>(R, V, D) : embed_ws_bytes<float>(R, V, D);
}

template <typename T>
int embed_bwd(const void* grad_, const int64_t* idx, int64_t R, int64_t V, int64_t D, double scale, void* ws,
              void* d_table_, int* status, cudaStream_t s) {
  using A = typename Io<T>::Acc;
  const T* grad = (const T*)grad_;
  T* d_table = (T*)d_table_;
  const bool vec = D % Io<T>::VEC == 0 && !((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(d_table)) & 15);
  const SumPlan sp = sum_plan<T>(R, D, vec);
  const SortPlan so = sort_plan(V);
  const EmbedWs w = embed_ws<T>(R, V, D, sp);
  uint8_t* p = (uint8_t*)ws;
  int* keys[2] = {(int*)(p + w.keys[0]), (int*)(p + w.keys[1])};
  int* order[2] = {(int*)(p + w.order[0]), (int*)(p + w.order[1])};
  int *hist = (int*)(p + w.hist), *totals = (int*)(p + w.totals), *start = (int*)(p + w.start);
  A* partial = (A*)(p + w.partial);
  int at = 0;  // which of the pair holds the sorted tokens
  int launches = 0;
  if (R > 0 && R <= SMALL_ROWS) {
    if (!sort_small_ready()) return FC_ERR_LAUNCH;
    sort_small<<<1, SMALL_THREADS, small_bytes((int)R), s>>>(idx, (int)R, V, so.passes, so.bits, keys[0], order[0], start, status);
    launches = 1;
  } else if (R > 0) {
    const unsigned tiles = (unsigned)((R + SORT_TILE - 1) / SORT_TILE);
    for (int pass = 0; pass < so.passes; ++pass) {
      const int shift = pass * so.bits, to = pass & 1, from = to ^ 1;
      if (pass == 0)
        sort_count<true><<<tiles, SORT_THREADS, 0, s>>>(idx, nullptr, R, V, shift, so.bits, so.digits, hist, status);
      else
        sort_count<false><<<tiles, SORT_THREADS, 0, s>>>(idx, keys[from], R, V, shift, so.bits, so.digits, hist,
                                                         status);
      // few tiles: every scatter block adds their counts itself (a launch less)
      const int scanned = tiles > 64;
      launches += 2 + scanned;
      if (scanned) sort_scan<<<so.digits, 256, 0, s>>>(hist, (int)tiles, totals);
      if (pass == 0)
        sort_scatter<true><<<tiles, SORT_THREADS, 0, s>>>(idx, nullptr, nullptr, R, V, shift, so.bits, so.digits, hist,
                                                          totals, keys[to], order[to], so.passes == 1 ? start : nullptr, scanned);
      else
        sort_scatter<false><<<tiles, SORT_THREADS, 0, s>>>(idx, keys[from], order[from], R, V, shift, so.bits,
                                                           so.digits, hist, totals, keys[to], order[to], nullptr, scanned);
      at = to;
    }
  }
  if (fc_launched(launches)) return FC_ERR_LAUNCH;
  launches = 0;
  // with one pass the sort has placed the tokens, and embed_combine writes the empty rows
  const int by_token = V <= sp.chunks;
  if (R == 0 || so.passes > 1 || !by_token || sp.chunks == 1) {
    embed_bounds<T><<<(unsigned)((V + 1 + 255) / 256), 256, 0, s>>>(keys[at], (int)R, V, D, vec, start, d_table);
    ++launches;
  }
  if (R > 0) {
    const unsigned grid = (unsigned)((sp.chunks * sp.col_tiles * sp.lanes + 255) / 256);
    ++launches;
    if (vec)
      embed_sum<T, Io<T>::VEC, true><<<grid, 256, 0, s>>>(grad, keys[at], order[at], start, (int)R, V, D, sp.Lc,
                                                          sp.chunks, sp.lanes, sp.col_tiles, (A)scale, partial, sp.Dp,
                                                          d_table);
    else
      embed_sum<T, 4, false><<<grid, 256, 0, s>>>(grad, keys[at], order[at], start, (int)R, V, D, sp.Lc, sp.chunks,
                                                  sp.lanes, sp.col_tiles, (A)scale, partial, sp.Dp, d_table);
    if (sp.chunks > 1) {
      constexpr int PC = 16 / (int)sizeof(A);
      int lanes = 1;
      while (lanes < 32 && (int64_t)lanes * PC < sp.Dp) lanes *= 2;
      const int slices = combine_slices(V, sp);
      launches += slices > 1 ? 2 : 1;
      const int64_t cands = by_token ? V : sp.chunks;
      int64_t per_block = (cands + 148 * 4 - 1) / (148 * 4);
      // few types: long spans, large blocks; else most spans are a few chunks
      const int threads = by_token ? 512 : 256;
      if (per_block > threads) per_block = threads;
      A* sums = (A*)(p + w.sums);
      const dim3 cgrid((unsigned)((cands + per_block - 1) / per_block),
                       (unsigned)std::min<int64_t>((sp.Dp + (int64_t)lanes * PC - 1) / ((int64_t)lanes * PC), 65535),
                       (unsigned)slices);
      const auto combine = by_token ? embed_combine<T, 512> : embed_combine<T, 256>;
      combine<<<cgrid, threads, 0, s>>>(partial, keys[at], start, (int)R, V, D, sp.Dp, sp.Lc, sp.chunks, by_token,
                                        (int)per_block, lanes, slices, vec, (A)scale, sums, d_table);
      if (slices > 1)
        embed_finish<T><<<dim3((unsigned)V, (unsigned)((D + 255) / 256)), 256, 0, s>>>(
            sums, start, V, D, sp.Dp, sp.Lc, slices, (A)scale, d_table);
    }
  }
  return fc_launched(launches);
}

#endif

#define FC_EMBED_INST(T)                                                                                        \
  template int embed_fwd<T>(const void*, int64_t, int64_t, const int64_t*, int64_t, double, double, void*, int*, \
                            cudaStream_t);                                                                      \
  template int embed_bwd<T>(const void*, const int64_t*, int64_t, int64_t, int64_t, double, void*, void*, int*, \
                            cudaStream_t);
FC_EMBED_INST(float)
FC_EMBED_INST(double)
FC_EMBED_INST(bf16_t)

}  // namespace fc
