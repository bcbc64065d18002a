// Gated feed-forward block: arguments shared by its kernels.
#pragma once
#include "fc_vec.cuh"

namespace fc {

// Rows of rank blocks l = 0..L, component k = l^2 + m of row r at (r (L+1)^2 + k) C.
struct GatedArgs {
  int L, C, H;        // ranks, input and hidden channels
  int act;            // FC_GATE_SILU / FC_GATE_SIGMOID
  int64_t n;          // rows
  const void* x;      // (n, (L+1)^2 C)
  const void* wv[4];  // per rank (H, C)
  const void* wg;     // ((L+1) H, C)
  const void* bias;   // ((L+1) H) or null
  const void* scales; // L+1 value scales, the gate scale, the activation scale (Acc type)
  // forward
  void* y;            // (n, (L+1)^2 H)
  // backward
  const void* gy;     // (n, (L+1)^2 H)
  void* gx;           // outputs, each null where not wanted
  void* gwv[4];
  void* gwg;
  void* gbias;
  void* ws;
  int* status;
};

FC_HD FC_INLINE int gated_rank_of(int k) { return k >= 9 ? 3 : k >= 4 ? 2 : k >= 1 ? 1 : 0; }

// sigma(z) without overflow for any z (NaN stays NaN)
FC_HD FC_INLINE float gated_sigmoid(float z) { return 1.f / (1.f + expf(-z)); }
FC_HD FC_INLINE double gated_sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

template <typename A>
FC_HD FC_INLINE A gated_act(int act, A z) {
  const A s = gated_sigmoid(z);
  return act == FC_GATE_SIGMOID ? s : z * s;
}
template <typename A>
FC_HD FC_INLINE A gated_dact(int act, A z) {
  const A s = gated_sigmoid(z);
  return act == FC_GATE_SIGMOID ? s * (A(1) - s) : s * (A(1) + z * (A(1) - s));
}

// Plain multiply-add tiles (gated_ff.cu): 64-bit rows, and every type in the host emulation.
int64_t gated_simple_ws(int L, int C, int H, int64_t n, int dtype, int backward);
template <typename T>
int gated_simple_fwd(const GatedArgs& a, cudaStream_t s);
template <typename T>
int gated_simple_bwd(const GatedArgs& a, cudaStream_t s);

#ifndef FC_HOST_EMU
// Tensor-core form of float and bfloat16 rows (gated_ff_tc.cu).
int64_t gated_tc_ws(int L, int C, int H, int64_t n, int dtype, int backward);
template <typename T>
int gated_tc_fwd(const GatedArgs& a, cudaStream_t s);
template <typename T>
int gated_tc_bwd(const GatedArgs& a, cudaStream_t s);
#endif

}  // namespace fc
