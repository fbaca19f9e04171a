// Loads and lane exchanges of the kernels that stream K/V rows through registers (included by .hip
// sources only).
#pragma once

#include <hip/hip_runtime.h>

#include "nva_device.h"

namespace nva {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// A non-temporal load (K/V rows are read once per step) from a wave-uniform base plus a 32-bit lane
// offset (floats), as a buffer load: the base stays in scalar registers, so no per-lane 64-bit address is formed
// (headline decode 2.160-2.162 against 2.166-2.171 ms with the pointer form).  The cache policy
// matters, the form little: without the non-temporal bit the same loads take 2.40 ms, and
// adding the L1-bypass (sc0) or device-scope (sc1) bits changes nothing.
template <int POLICY>
__device__ __forceinline__ float4 ld4_buffer(const float *base, uint32_t off) {
  const uint64_t b = (uint64_t)(size_t)base;
  const uint64_t u = ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) << 32) |
                     (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc((void *)(size_t)u, (short)0, 0x7fffffff, kBufferWord3);
  const f32x4 t = __builtin_amdgcn_raw_buffer_load_b128(r, off * 4, 0, POLICY);
  return make_float4(t.x, t.y, t.z, t.w);
}
__device__ __forceinline__ float4 ld4_stream_at(const float *base, uint32_t off) {
  constexpr int kNonTemporal = 2;  // the nt bit of the buffer instructions' cache policy
  return ld4_buffer<kNonTemporal>(base, off);
}
// An offset (floats) behind the range of the loads above, which they answer with zeros: the V of a
// masked key, whose weight of 0 must not meet an infinity.
constexpr uint32_t kOutside = 0x20000000;
// The same, cached.
__device__ __forceinline__ float4 ld4_at(const float *base, uint32_t off) {
  return ld4_buffer<0>(base, off);
}

// x[lane] + x[lane ^ 16] (resp. lane ^ 32) in every lane, by gfx950's row-swap instructions:
// the swap of x with itself leaves one of the two values in each output, and the sum of the
// two is the same bits in both lanes of a pair.  No LDS round trip, unlike ds_swizzle or
// ds_bpermute.
__device__ __forceinline__ float add_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Max and sum over the four lanes {l, l ^ 16, l ^ 32, l ^ 48}; every lane gets the same bits.
__device__ __forceinline__ float max4_lanes(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  const float m = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false,
                                                  false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float sum4_lanes(float x) { return add_xor32(add_xor16(x)); }

}  // namespace nva
