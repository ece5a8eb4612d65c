// rowvec.cuh - rows of logits read and written as 16-byte vectors whatever
// their start, type or length, and the packed masks over them.
//
// A row [vocab] of T starts anywhere T may start.  Its vectors are the aligned
// 16-byte groups that cover it: vector i holds the elements e0 .. e0 + VE - 1
// with e0 = i * VE - shift, shift = the row's start inside its group.  Only
// the first and the last vector of a row can be partial; those move element
// by element, so nothing outside the row is touched.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cnnue {
namespace rows {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLog2e = 1.44269504088896340736f;

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Element count of 16 bytes, and the conversions of one element and one vector.
template <typename T>
struct Vec;

template <>
struct Vec<float> {
  static constexpr int VE = 4;
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  // -inf where `ok` has no bit.
  static __device__ __forceinline__ uint4 only(uint4 r, uint32_t ok) {
    return make_uint4(ok & 1 ? r.x : 0xff800000u, ok & 2 ? r.y : 0xff800000u, ok & 4 ? r.z : 0xff800000u,
                      ok & 8 ? r.w : 0xff800000u);
  }
  // The largest element; a NaN if there is one.
  static __device__ __forceinline__ float top(const uint4& r) {
    return max_nan(max_nan(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z)), __uint_as_float(r.w));
  }
};

// Word i of a 16-bit vector with `low` in the halves that `ok` does not name.
__device__ __forceinline__ uint32_t only_word(uint32_t w, uint32_t ok, int i, uint32_t low) {
  const uint32_t keep = (ok >> 2 * i & 1 ? 0x0000ffffu : 0u) | (ok >> 2 * i & 2 ? 0xffff0000u : 0u);
  return (w & keep) | (low & ~keep);
}

template <>
struct Vec<__nv_bfloat16> {
  static constexpr int VE = 8;
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ uint4 only(const uint4& r, uint32_t ok) {
    return make_uint4(only_word(r.x, ok, 0, 0xff80ff80u), only_word(r.y, ok, 1, 0xff80ff80u),
                      only_word(r.z, ok, 2, 0xff80ff80u), only_word(r.w, ok, 3, 0xff80ff80u));
  }
  static __device__ __forceinline__ float top(const uint4& r) {
    __nv_bfloat162 a, b, c, d;
    memcpy(&a, &r.x, 4), memcpy(&b, &r.y, 4), memcpy(&c, &r.z, 4), memcpy(&d, &r.w, 4);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(a, b), __hmax2_nan(c, d));
    return max_nan(__bfloat162float(m.x), __bfloat162float(m.y));
  }
};

template <>
struct Vec<__half> {
  static constexpr int VE = 8;
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 f = __half22float2(h);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ uint4 only(const uint4& r, uint32_t ok) {
    return make_uint4(only_word(r.x, ok, 0, 0xfc00fc00u), only_word(r.y, ok, 1, 0xfc00fc00u),
                      only_word(r.z, ok, 2, 0xfc00fc00u), only_word(r.w, ok, 3, 0xfc00fc00u));
  }
  static __device__ __forceinline__ float top(const uint4& r) {
    __half2 a, b, c, d;
    memcpy(&a, &r.x, 4), memcpy(&b, &r.y, 4), memcpy(&c, &r.z, 4), memcpy(&d, &r.w, 4);
    const __half2 m = __hmax2_nan(__hmax2_nan(a, b), __hmax2_nan(c, d));
    return max_nan(__half2float(m.x), __half2float(m.y));
  }
};

// Elements of `row` before it in its 16-byte group.
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) {
  return (int)(((uintptr_t)row & 15) / sizeof(T));
}

// Vectors that cover a row, whatever its shift (host and device).
template <typename T>
__host__ __device__ constexpr int64_t max_vectors(int64_t vocab) {
  return (vocab + 2 * (Vec<T>::VE - 1)) / Vec<T>::VE;
}

template <int VE>
constexpr uint32_t kFull = (1u << VE) - 1;

// Bit i: element e0 + i lies inside the row.
template <int VE>
__device__ __forceinline__ uint32_t inside(int e0, int vocab) {
  uint32_t b = kFull<VE>;
  if (e0 < 0) b &= kFull<VE> << -e0;
  if (e0 + VE > vocab) b = e0 < vocab ? b & (kFull<VE> >> (e0 + VE - vocab)) : 0;
  return b;
}

// Bit i: the packed mask allows element e0 + i (bit j of word w = token
// 32 w + j).  Elements outside the row give 0; no word past the last one that
// holds a token is read.
template <int VE>
__device__ __forceinline__ uint32_t allowed(const uint32_t* __restrict__ mask, int e0, int vocab) {
  const uint32_t in = inside<VE>(e0, vocab);
  if (in == 0) return 0;
  if (e0 < 0) return (__ldg(mask) << -e0) & in;
  const int w = e0 >> 5, sh = e0 & 31;
  uint32_t b = __ldg(mask + w) >> sh;
  if (sh + VE > 32 && 32 * (w + 1) < vocab) b |= __ldg(mask + w + 1) << (32 - sh);
  return b & in;
}

// One 16-byte load past L1.  Not the read-only path: a row may be processed in
// place, and each vector is then read and written by one thread.
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// allowed() for a vector that lies inside the row.
template <int VE>
__device__ __forceinline__ uint32_t allowed_whole(const uint32_t* __restrict__ mask, int e0) {
  const int w = e0 >> 5, sh = e0 & 31;
  uint32_t b = __ldg(mask + w) >> sh;
  if (sh > 32 - VE) b |= __ldg(mask + w + 1) << (32 - sh);
  return b & kFull<VE>;
}

// The raw vector e0 with at least the elements of `want` in it (the others are
// whatever a whole load brings, or 0).
template <typename T>
__device__ __forceinline__ uint4 load_raw(const T* row, int e0, uint32_t in, uint32_t want) {
  constexpr int VE = Vec<T>::VE;
  if (in == kFull<VE>) return load16(row + e0);
  float x[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) x[i] = want >> i & 1 ? Vec<T>::up(row[e0 + i]) : 0.f;
  return Vec<T>::pack(x);
}

// x to the elements of vector e0 (of the input's vectors, VE of them) of an
// output row of TO.  `whole`: that vector's output starts on a 16-byte
// boundary; else, or at the row's edges, element by element.
template <typename TO, int VE>
__device__ __forceinline__ void store(TO* row, int e0, uint32_t in, bool whole, const float* x) {
  if (in == kFull<VE> && whole && VE % Vec<TO>::VE == 0) {
#pragma unroll
    for (int j = 0; j < VE / Vec<TO>::VE; ++j)
      *reinterpret_cast<uint4*>(row + e0 + j * Vec<TO>::VE) = Vec<TO>::pack(x + j * Vec<TO>::VE);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (in >> i & 1) row[e0 + i] = Vec<TO>::down(x[i]);
  }
}

// Whether vector stores of the output line up with the input's vectors.
template <typename TO>
__device__ __forceinline__ bool lines_up(const TO* out_row, int shift) {
  return ((uintptr_t)(out_row - shift) & 15) == 0;
}

// Token i of a list of 32-bit or 64-bit tokens; what does not fit 31 bits
// comes back as INT32_MAX (out of every range) or, when negative, as -1.
__device__ __forceinline__ int token_at(const void* list, int64_t i, bool wide) {
  if (!wide) return __ldg((const int*)list + i);
  const long long t = __ldg((const long long*)list + i);
  return t < 0 ? -1 : t > 0x7fffffff ? 0x7fffffff : (int)t;
}

// Two fp32 operations in one instruction, each rounded as its scalar form.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  asm("{.reg .b64 ra, rb, rc;\n\tmov.b64 ra, {%0, %1};\n\tmov.b64 rb, {%2, %3};\n\t"
      "add.rn.f32x2 rc, ra, rb;\n\tmov.b64 {%0, %1}, rc;}"
      : "+f"(a.x), "+f"(a.y)
      : "f"(b.x), "f"(b.y));
  return a;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  asm("{.reg .b64 ra, rb, rc;\n\tmov.b64 ra, {%0, %1};\n\tmov.b64 rb, {%2, %3};\n\t"
      "mul.rn.f32x2 rc, ra, rb;\n\tmov.b64 {%0, %1}, rc;}"
      : "+f"(a.x), "+f"(a.y)
      : "f"(b.x), "f"(b.y));
  return a;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  asm("{.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%0, %1};\n\tmov.b64 rb, {%2, %3};\n\tmov.b64 rc, {%4, %5};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;}"
      : "+f"(a.x), "+f"(a.y)
      : "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return a;
}

}  // namespace rows
}  // namespace cnnue
