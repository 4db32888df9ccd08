// Element access shared by the vocabulary operators (embedding, distillation): eight consecutive
// elements of fp32, binary16 or bfloat16 per lane, widened to fp32 and narrowed back with one
// rounding.
//
// The wide accesses assume the element's own alignment only, because rows of an odd width start
// anywhere.  Measured on the rows of a 50257-column matrix (8192 rows, one workgroup each): reads
// of rows that start at a multiple of 16, 8 or 4 bytes run at 6.28 TB/s alike, of rows that start
// at an odd multiple of 2 bytes at 4.9 TB/s; a copy runs at 5.4, 5.1 and 4.8 TB/s.  So nothing is
// gained by aligning beyond 4 bytes, and code that streams long rows of 16-bit elements takes one
// element off the front of the odd ones.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "half_types.h"
#include "status.h"

namespace rafhip {

typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef f16x8 f16x8_any __attribute__((aligned(2)));
typedef u16x8 u16x8_any __attribute__((aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kWide = 8;  // elements per lane and access

template <typename T>
struct Wide;

template <>
struct Wide<float> {
  typedef f32x4_any Sixteen;  // what sixteen bytes hold
  struct Raw {
    f32x4 a, b;
  };
  static __device__ __forceinline__ Raw load(const float* p) {
    const RAFHIP_GLOBAL f32x4_any* q = (const RAFHIP_GLOBAL f32x4_any*)p;
    return Raw{q[0], q[1]};
  }
  static __device__ __forceinline__ Raw fill(float x) { return Raw{f32x4{x, x, x, x}, f32x4{x, x, x, x}}; }
  // The compiler may not carry widened values past this point (nothing to widen here).
  static __device__ __forceinline__ void keep_narrow(Raw&) {}
  static __device__ __forceinline__ float get(const Raw& r, int j) { return j < 4 ? r.a[j & 3] : r.b[j & 3]; }
  static __device__ __forceinline__ void store(float* p, const float (&v)[kWide]) {
    RAFHIP_GLOBAL f32x4_any* q = (RAFHIP_GLOBAL f32x4_any*)p;
    q[0] = f32x4{v[0], v[1], v[2], v[3]};
    q[1] = f32x4{v[4], v[5], v[6], v[7]};
  }
  static __device__ __forceinline__ float one(const float* p) { return *(const RAFHIP_GLOBAL float*)p; }
  static __device__ __forceinline__ void put(float* p, float x) { *(RAFHIP_GLOBAL float*)p = x; }
};

template <>
struct Wide<_Float16> {
  typedef f16x8_any Sixteen;
  typedef f16x8 Raw;
  static __device__ __forceinline__ Raw load(const _Float16* p) { return *(const RAFHIP_GLOBAL f16x8_any*)p; }
  static __device__ __forceinline__ Raw fill(float x) {
    const _Float16 h = (_Float16)x;
    return Raw{h, h, h, h, h, h, h, h};
  }
  static __device__ __forceinline__ void keep_narrow(Raw& r) { asm volatile("" : "+v"(r)); }
  static __device__ __forceinline__ float get(const Raw& r, int j) { return (float)r[j]; }
  static __device__ __forceinline__ void store(_Float16* p, const float (&v)[kWide]) {
    f16x8 r;
#pragma unroll
    for (int j = 0; j < kWide; ++j) r[j] = (_Float16)v[j];
    *(RAFHIP_GLOBAL f16x8_any*)p = r;
  }
  static __device__ __forceinline__ float one(const _Float16* p) { return (float)*(const RAFHIP_GLOBAL _Float16*)p; }
  static __device__ __forceinline__ void put(_Float16* p, float x) { *(RAFHIP_GLOBAL _Float16*)p = (_Float16)x; }
};

template <>
struct Wide<Bf16> {
  typedef u16x8_any Sixteen;
  typedef u16x8 Raw;
  static __device__ __forceinline__ Raw load(const Bf16* p) { return *(const RAFHIP_GLOBAL u16x8_any*)p; }
  static __device__ __forceinline__ Raw fill(float x) {
    const unsigned short h = bf16_narrow(x);
    return Raw{h, h, h, h, h, h, h, h};
  }
  static __device__ __forceinline__ void keep_narrow(Raw& r) { asm volatile("" : "+v"(r)); }
  static __device__ __forceinline__ float get(const Raw& r, int j) { return bf16_widen(r[j]); }
  // gfx950 narrows two at once, to nearest even as bf16_narrow does.
  static __device__ __forceinline__ void store(Bf16* p, const float (&v)[kWide]) {
    bf16x8 r;
#pragma unroll
    for (int j = 0; j < kWide; ++j) r[j] = (__bf16)v[j];
    *(RAFHIP_GLOBAL u16x8_any*)p = __builtin_bit_cast(u16x8, r);
  }
  static __device__ __forceinline__ float one(const Bf16* p) {
    return bf16_widen(*(const RAFHIP_GLOBAL unsigned short*)p);
  }
  static __device__ __forceinline__ void put(Bf16* p, float x) { *(RAFHIP_GLOBAL unsigned short*)p = bf16_narrow(x); }
};

template <typename T>
__device__ __forceinline__ void widen8(const typename Wide<T>::Raw& r, float (&v)[kWide]) {
#pragma unroll
  for (int j = 0; j < kWide; ++j) v[j] = Wide<T>::get(r, j);
}

// Calls f with a value of the element type of `dtype` (RAFHIP_F32, RAFHIP_F16 or RAFHIP_BF16, checked before).
template <typename F>
void with_element(int32_t dtype, F&& f) {
  if (dtype == 0)
    f(float{});
  else if (dtype == 1)
    f(_Float16{});
  else
    f(Bf16{});
}

// Calls f with a value of the index type of `index_bits` (32 or 64, checked before).
template <typename F>
void with_index(int32_t index_bits, F&& f) {
  if (index_bits == 32)
    f(int32_t{});
  else
    f(int64_t{});
}

inline int element_bytes(int32_t dtype) { return dtype == 0 ? 4 : dtype == 1 || dtype == 2 ? 2 : 0; }

// What a call reads or writes.  The kernels read their inputs while they write, so the entry points refuse
// an output that shares bytes with an input or another output.
struct Extent {
  const char* name;
  const void* at;
  int64_t bytes;
};
inline bool share_bytes(const Extent& a, const Extent& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.at && b.at && a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}
template <size_t kOuts, size_t kIns>
int check_apart(const char* who, const Extent (&outs)[kOuts], const Extent (&ins)[kIns]) {
  for (size_t i = 0; i < kOuts; ++i) {
    for (const Extent& in : ins)
      if (share_bytes(outs[i], in)) return fail(RAFHIP_ERR_INVALID_ARG, "%s: %s overlaps %s", who, outs[i].name, in.name);
    for (size_t j = 0; j < i; ++j)
      if (share_bytes(outs[i], outs[j]))
        return fail(RAFHIP_ERR_INVALID_ARG, "%s: %s overlaps %s", who, outs[i].name, outs[j].name);
  }
  return RAFHIP_OK;
}

inline bool is_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0; }

}  // namespace rafhip
