// Device helpers of the low-bit serving operators (gfx950): loads of 16- and 32-bit
// floats, powers of two as float32, and the hardware's e2m1 and e4m3 conversions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "cp_host.h"

namespace cp {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Element types by cp_dtype code.
template <int DT> struct Elem;
template <> struct Elem<CP_F32> { typedef float T; };
template <> struct Elem<CP_BF16> { typedef __bf16 T; };
template <> struct Elem<CP_F16> { typedef _Float16 T; };

// A launch holds under 2^32 work items in x: so many workgroups of that many threads at most.
inline int64_t most_workgroups(int threads) { return 0xFFFFFFFFll / threads; }

// Allows a kernel this much LDS on the current device. It is asked for once for each device (a
// bit of done); a failure is reported and asked for again by the next call.
inline int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>* done, const char* what) {
  int dev = 0;
  CP_HIP(hipGetDevice(&dev));
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (dev < 64 && (done->load(std::memory_order_relaxed) & bit)) return CP_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return hip_fail(e, what);
  if (dev < 64) done->fetch_or(bit, std::memory_order_relaxed);
  return CP_OK;
}

inline int dtype_bytes(int dt) { return dt == CP_F32 ? 4 : dt == CP_BF16 || dt == CP_F16 ? 2 : 0; }

// Eight consecutive values as they are stored.
template <int DT>
struct Raw8 {
  u32x4 w[DT == CP_F32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const typename Elem<DT>::T* p) {
  Raw8<DT> r;
  r.w[0] = *reinterpret_cast<const u32x4*>(p);
  if constexpr (DT == CP_F32) r.w[1] = *reinterpret_cast<const u32x4*>(p + 4);
  return r;
}

// ... and as float32.
template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& raw, float (&v)[8]) {
  if constexpr (DT == CP_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(raw.w[0][i]), v[i + 4] = __uint_as_float(raw.w[1][i]);
  } else {
    const u32x4 r = raw.w[0];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == CP_BF16) {
        v[2 * i] = __uint_as_float(r[i] << 16);
        v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
      } else {
        const uint32_t w = r[i];  // a bit cast of a vector's element itself reads element 0
        const f16x2 h = __builtin_bit_cast(f16x2, w);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      }
    }
  }
}

// Eight consecutive values as float32 (p 16-byte aligned).
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* p, float (&v)[8]) {
  widen8<DT>(load_raw8<DT>(p), v);
}

// Two float32 rounded to nearest even in a 16-bit type, packed.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == CP_BF16) {
    bf16x2 h;
    h[0] = (__bf16)a;
    h[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, h);
  } else {
    f16x2 h;
    h[0] = (_Float16)a;
    h[1] = (_Float16)b;
    return __builtin_bit_cast(uint32_t, h);
  }
}

// Eight consecutive values from float32 (p 16-byte aligned).
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::T* p, const float (&v)[8]) {
  if constexpr (DT == CP_F32) {
    f32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = v[i], b[i] = v[i + 4];
    *reinterpret_cast<f32x4*>(p) = a;
    *reinterpret_cast<f32x4*>(p + 4) = b;
  } else {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<u32x4*>(p) = r;
  }
}

// Exponent of a finite positive float32 as frexp gives it: a = m * 2^e, m in [0.5, 1).
__device__ __forceinline__ int frexp_e(float a) { return __builtin_amdgcn_frexp_expf(a); }
__device__ __forceinline__ float frexp_m(float a) { return __builtin_amdgcn_frexp_mantf(a); }

// 2^(b - 127) of an exponent byte b: 2^-127 (a subnormal) for 0, NaN for 255.
__device__ __forceinline__ float pow2_byte(int b) {
  return __uint_as_float(b == 255 ? 0x7FC00000u : b == 0 ? 0x00400000u : (uint32_t)b << 23);
}

// Eight e4m3 codes as float32, and back (round to nearest even; |v| <= 448 or NaN).
__device__ __forceinline__ void e4m3_decode8(u32x2 c, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
    v[4 * i] = a[0], v[4 * i + 1] = a[1], v[4 * i + 2] = b[0], v[4 * i + 3] = b[1];
  }
}

__device__ __forceinline__ u32x2 e4m3_encode8(const float (&v)[8]) {
  u32x2 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
    c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], w, true);
  }
  return c;
}

}  // namespace cp
