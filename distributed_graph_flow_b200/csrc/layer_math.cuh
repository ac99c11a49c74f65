// Device helpers shared by the layer operators (gated dense, segment group
// norm, gated scan): activations with their derivatives, two values at a time,
// and 16-byte vectors of fp32 / bf16 as fp32 values.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace dgfx {

// e^x and 1 / x by the special function unit, subnormal numbers flushed (the
// plain intrinsics spend as many instructions again on keeping them).
__device__ __forceinline__ float exp_f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ float rcp_f(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// 1 / (1 + e^-z) without overflow at either end: e^-z = inf gives 0.
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  const float2 t = mul2(z, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  e = add2(e, make_float2(1.0f, 1.0f));
  return make_float2(rcp_f(e.x), rcp_f(e.y));
}

// Phi(z), the normal distribution function, and e^(-z^2 / 2). The tail
// Phi(-|z|) is e^(-z^2 / 2) t P(t) with t = 1 / (1 + 0.295 |z|): t P(t) follows
// erfcx(|z| / sqrt 2) / 2, which falls like 1 / |z|. P has degree 7, a weighted minimax fit (Lawson's
// iteration, 64 bits) that is off by at most 1.1e-8 (1 + z^2) of the tail's
// value: below the rounding of the exponent, which is z^2 2^-24. Phi is the tail below
// zero, one minus it above: no subtraction in the lower tail, and the
// exponential is the derivative's too. Together with the roundings and the
// intrinsics (rcp 2, ex2 4 units of 2^-24) the relative error stays below
// (25 + 1.4 z^2) 2^-24; in a product with z, weighted by the normal
// distribution, it is 2.8e-8, as of the erf form in fp32.
__device__ __forceinline__ float2 normal_cdf2(float2 z, float2* bell) {
  auto both = [](float v) { return make_float2(v, v); };
  const float2 a = fma2(make_float2(fabsf(z.x), fabsf(z.y)), both(0.295f), both(1.0f));
  const float2 t = make_float2(rcp_f(a.x), rcp_f(a.y));
  float2 poly = fma2(t, both(0.03697340515f), both(-0.1713015898f));
  poly = fma2(poly, t, both(0.2456400625f));
  poly = fma2(poly, t, both(-0.08772105514f));
  poly = fma2(poly, t, both(0.1458911895f));
  poly = fma2(poly, t, both(0.09342662252f));
  poly = fma2(poly, t, both(0.1195008056f));
  poly = fma2(poly, t, both(0.1175905649f));
  const float2 x = mul2(mul2(z, both(-0.5f * 1.4426950408889634f)), z);
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
  const float2 tail = mul2(mul2(poly, t), e), rest = fma2(tail, both(-1.0f), both(1.0f));
  *bell = e;
  return make_float2(z.x < 0.0f ? tail.x : rest.x, z.y < 0.0f ? tail.y : rest.y);
}

// Activations (DGFX_ACT_*) of two values in fp32. gelu is the form z Phi(z) =
// z (1 + erf(z / sqrt 2)) / 2. relu compares instead of taking a maximum, so
// that NaN passes through.
template <int ACT>
__device__ __forceinline__ float2 act2_f(float2 z) {
  if (ACT == DGFX_ACT_GELU) {
    float2 bell;
    return mul2(z, normal_cdf2(z, &bell));
  }
  if (ACT == DGFX_ACT_SILU) return mul2(z, sigmoid2(z));
  if (ACT == DGFX_ACT_SIGMOID) return sigmoid2(z);
  if (ACT == DGFX_ACT_RELU) return make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y);
  return z;
}

// act(z) and act'(z) together (they share the exponential). relu'(0) = 0.
template <int ACT>
__device__ __forceinline__ void act2_both_f(float2 z, float2* value, float2* slope) {
  const float2 one = make_float2(1.0f, 1.0f), minus = make_float2(-1.0f, -1.0f);
  if (ACT == DGFX_ACT_SILU) {
    const float2 s = sigmoid2(z);
    *value = mul2(z, s);
    *slope = mul2(s, fma2(z, fma2(s, minus, one), one));
  } else if (ACT == DGFX_ACT_SIGMOID) {
    const float2 s = sigmoid2(z);
    *value = s;
    *slope = mul2(s, fma2(s, minus, one));
  } else if (ACT == DGFX_ACT_GELU) {
    float2 bell;
    const float2 cdf = normal_cdf2(z, &bell);
    *value = mul2(z, cdf);
    *slope = fma2(mul2(z, make_float2(0.39894228040143268f, 0.39894228040143268f)), bell, cdf);
  } else if (ACT == DGFX_ACT_RELU) {
    *value = act2_f<ACT>(z);
    *slope = make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
  } else {
    *value = z;
    *slope = one;
  }
}

// 16 bytes of T as fp32 values.
template <class T>
struct Vec16;
template <>
struct Vec16<float> {
  __device__ static __forceinline__ void unpack(const uint4& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x);
    f[1] = __uint_as_float(r.y);
    f[2] = __uint_as_float(r.z);
    f[3] = __uint_as_float(r.w);
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Vec16<__nv_bfloat16> {
  __device__ static __forceinline__ void unpack(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f[2 * q] = __uint_as_float(w[q] << 16);
      f[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
    }
  }
};

// Four adjacent values of T (a quad) as fp32.
template <class T>
struct Quad;
template <>
struct Quad<float> {
  using raw = uint4;
  __device__ static __forceinline__ void unpack(const raw& r, float (&f)[4]) { Vec16<float>::unpack(r, f); }
  __device__ static __forceinline__ raw pack(const float (&f)[4]) { return Vec16<float>::pack(f); }
  __device__ static __forceinline__ raw zero() { return make_uint4(0, 0, 0, 0); }
};
template <>
struct Quad<__nv_bfloat16> {
  using raw = uint2;
  __device__ static __forceinline__ void unpack(const raw& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x << 16);
    f[1] = __uint_as_float(r.x & 0xFFFF0000u);
    f[2] = __uint_as_float(r.y << 16);
    f[3] = __uint_as_float(r.y & 0xFFFF0000u);
  }
  __device__ static __forceinline__ raw pack(const float (&f)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
  __device__ static __forceinline__ raw zero() { return make_uint2(0, 0); }
};

// Chains of kernels, each of which needs the one before it: a kernel launched
// by launch_after may be brought onto the SMs while its predecessor still
// runs, and waits in after_previous (its first statement) until all of that
// one's blocks have ended and their writes are visible. The predecessor allows
// it by let_next_start. What the chain itself has written is read by plain
// loads, which the compiler keeps behind the wait. The first kernel of a chain is
// launched as usual.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... P, class... A>
void launch_after(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(block);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);  // its error stays for cudaGetLastError
}

__host__ __device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) {
  return v < lo ? lo : (v > hi ? hi : v);
}

inline bool ptr_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace dgfx
