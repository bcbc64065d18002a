// Storage types of the training-block operators and their 16-byte vectors.
//
// Io<T> describes a storage type: its arithmetic type Acc (float for 16- and 32-bit
// storage, double for 64-bit), the elements of a 16-byte vector, and the conversions (one
// rounding to nearest even where storage is narrower than Acc).
#pragma once
#include "fc_base.cuh"
#ifndef FC_HOST_EMU
#include <cuda_bf16.h>
#endif

namespace fc {

// Kernels that this host thread has launched for the training blocks.
inline int64_t& fc_launch_count() {
  static thread_local int64_t n = 0;
  return n;
}
#ifndef FC_HOST_EMU
// Launcher epilogue behind n launches.
inline int fc_launched(int n) {
  fc_launch_count() += n;
  return fc_check_launch();
}
#endif

struct bf16_t {
  uint16_t bits;
};

FC_HD FC_INLINE float bf16_to_f32(uint16_t b) {
#if defined(__CUDA_ARCH__)
  return __uint_as_float((uint32_t)b << 16);
#else
  const uint32_t u = (uint32_t)b << 16;
  float f;
  memcpy(&f, &u, 4);
  return f;
#endif
}

FC_HD FC_INLINE uint16_t f32_to_bf16(float f) {
#if defined(__CUDA_ARCH__)
  return __bfloat16_as_ushort(__float2bfloat16_rn(f));
#else
  uint32_t u;
  memcpy(&u, &f, 4);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);  // NaN stays NaN
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
#endif
}

template <typename T>
struct Io;
template <>
struct Io<float> {
  using Acc = float;
  static constexpr int VEC = 4;
  FC_HD static FC_INLINE float get(float v) { return v; }
  FC_HD static FC_INLINE float put(float v) { return v; }
};
template <>
struct Io<double> {
  using Acc = double;
  static constexpr int VEC = 2;
  FC_HD static FC_INLINE double get(double v) { return v; }
  FC_HD static FC_INLINE double put(double v) { return v; }
};
template <>
struct Io<bf16_t> {
  using Acc = float;
  static constexpr int VEC = 8;
  FC_HD static FC_INLINE float get(bf16_t v) { return bf16_to_f32(v.bits); }
  FC_HD static FC_INLINE bf16_t put(float v) { return bf16_t{f32_to_bf16(v)}; }
};

#ifndef FC_HOST_EMU
// 16 (or B) bytes of storage to and from registers; the address is a multiple of B.
template <int B>
struct Raw;
template <>
struct Raw<16> {
  using type = uint4;
};
template <>
struct Raw<8> {
  using type = uint2;
};
template <>
struct Raw<4> {
  using type = uint32_t;
};
template <>
struct Raw<2> {
  using type = uint16_t;
};

template <typename T, int NV>
struct Pack {
  typename Raw<(int)sizeof(T) * NV>::type raw;
  __device__ __forceinline__ T at(int k) const { return reinterpret_cast<const T*>(&raw)[k]; }
  __device__ __forceinline__ void set(int k, T v) { reinterpret_cast<T*>(&raw)[k] = v; }
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const decltype(raw)*>(p); }
  // read once, not kept in L1
  __device__ __forceinline__ void load_stream(const T* p) { raw = __ldcs(reinterpret_cast<const decltype(raw)*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<decltype(raw)*>(p) = raw; }
};
#endif

}  // namespace fc
