// numeric.h -- element types of the transformer operators (fp32, fp16, bf16): loads and stores through registers as fp32.
#ifndef V3D_CSRC_NUMERIC_H_
#define V3D_CSRC_NUMERIC_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace v3d {

typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }  // round to nearest even

// N consecutive elements at an address that is aligned to ONE element only: gfx950 does unaligned vector accesses, so an
// odd row length costs no scalar loads.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Packed {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[N]) {
  const Packed<T, N> r = *reinterpret_cast<const Packed<T, N>*>(p);
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = to_f32(r.v[j]);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[N]) {
  Packed<T, N> r;
#pragma unroll
  for (int j = 0; j < N; ++j) r.v[j] = from_f32<T>(in[j]);
  *reinterpret_cast<Packed<T, N>*>(p) = r;
}

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Sum over WIDTH (16, 32 or 64) neighbouring lanes, the same bits in every lane: four DPP steps inside a row of 16 (no LDS
// traffic), the rest through ds_bpermute.
template <int WIDTH>
__device__ __forceinline__ float lanes_sum(float x) {
  x += dpp_f32<0xB1>(x);   // quad_perm [1,0,3,2]
  x += dpp_f32<0x4E>(x);   // quad_perm [2,3,0,1]
  x += dpp_f32<0x141>(x);  // row_half_mirror
  x += dpp_f32<0x140>(x);  // row_mirror
  if constexpr (WIDTH >= 32) x += __shfl_xor(x, 16, 64);
  if constexpr (WIDTH >= 64) x += __shfl_xor(x, 32, 64);
  return x;
}

}  // namespace v3d

#endif
