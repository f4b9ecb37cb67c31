// L2: activations held in 8 bits between forward and backward, and the gated activation that keeps its input so.
//
// Per 32 consecutive values of a row one exponent byte b and 32 signed codes: x ~ code * 2^(b - 127), with the smallest power of two of which
// round(amax / 2^e) <= 127 steps reach the block's largest magnitude, ties to even. amax = m 2^x with m in [1, 2): e = x - 6, one more from m =
// 255/128 on (127.5 would round to 128). Everything but the rounding to whole steps is exact: amax and e come from the bits, x / 2^e is a product
// with a power of two, code * 2^e has 7 bits and fits every type that x may have. b = 255 marks a block that holds an infinity or a NaN: all of it is
// restored as NaN, so that an overflow is not hidden. e is at least -126, which holds blocks below 2^-120 more coarsely.
// 33 bytes for 32 values. A power of two for 32 values costs what a 32-bit scale for 128 costs and is as near on normal values
// (the block's maximum is smaller by what the step is rounded up), nearer where single values stand out.
//
// All kernels are bound by memory: a thread takes 8 neighbouring values (16 bytes of a 16-bit type), four threads a block.
// Sums and functions are in 32 bits; this file is compiled without fast math, so that 32-bit inputs keep their small values.
#include <cuda_fp16.h>
#include "common.cuh"
#include "sx_api.h"

namespace sx {

template <typename T> struct Act8;
template <> struct Act8<__nv_bfloat16> {
  static __device__ __forceinline__ float in(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 out(float v) { return __float2bfloat16(v); }
};
template <> struct Act8<__half> {
  static __device__ __forceinline__ float in(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half out(float v) { return __float2half_rn(v); }
};
template <> struct Act8<float> {
  static __device__ __forceinline__ float in(float v) { return v; }
  static __device__ __forceinline__ float out(float v) { return v; }
};

// 8 values from column c of a row of `width`: whole 16-byte loads where VEC (width, pitch and base are multiples of 8 values then), else one by one.
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* row, int c, int width, float (&f)[8]) {
  if (VEC) {
    union { uint4 q[sizeof(T) / 2]; T t[8]; } v;
    if (c < width) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) v.q[i] = reinterpret_cast<const uint4*>(row + c)[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = Act8<T>::in(v.t[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = c + j < width ? Act8<T>::in(row[c + j]) : 0.f;
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* row, int c, int width, const float (&f)[8]) {
  if (VEC) {
    if (c < width) {
      union { uint4 q[sizeof(T) / 2]; T t[8]; } v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v.t[j] = Act8<T>::out(f[j]);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(row + c)[i] = v.q[i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < width) row[c + j] = Act8<T>::out(f[j]);
  }
}

// Codes and exponent byte of a block whose four threads hold 8 values each; all four are there and get the byte.
__device__ __forceinline__ uint2 encode8(const float (&f)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
  const uint32_t four = 0xfu << (threadIdx.y * blockDim.x + threadIdx.x & 28u);
  top = max(top, __shfl_xor_sync(four, top, 1));
  top = max(top, __shfl_xor_sync(four, top, 2));
  const bool finite = top < 0x7f800000u;
  byte = finite ? max((int)((top + 0x10000u) >> 23) - 6, 1) : 255u;
  const float inv = finite ? __uint_as_float((254u - byte) << 23) : 0.f;
  uint32_t k[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) k[j] = finite ? (uint32_t)__float2int_rn(f[j] * inv) : 0u;
  uint2 r;
  r.x = __byte_perm(__byte_perm(k[0], k[1], 0x0040), __byte_perm(k[2], k[3], 0x0040), 0x5410);
  r.y = __byte_perm(__byte_perm(k[4], k[5], 0x0040), __byte_perm(k[6], k[7], 0x0040), 0x5410);
  return r;
}
__device__ __forceinline__ void decode8(uint2 r, uint32_t byte, float (&f)[8]) {
  const float step = byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j] = (float)(signed char)(r.x >> (8 * j)) * step;
    f[4 + j] = (float)(signed char)(r.y >> (8 * j)) * step;
  }
}

// x [rows, width] (pitch ld) -> codes [rows, 32 nb], exps [rows, nb], nb = ceil(width / 32); codes behind the row are 0.
template <bool VEC, typename T>
__global__ void pack8_kernel(const T* __restrict__ x, signed char* __restrict__ codes, unsigned char* __restrict__ exps, unsigned rows, int width,
                             long long ld, int nb) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= nb * 4) return;     // pieces come by four, as the block's size does
  float f[8];
  load8<VEC>(x + row * ld, piece * 8, width, f);
  uint32_t byte;
  const uint2 k = encode8(f, byte);
  reinterpret_cast<uint2*>(codes)[(long long)row * (nb * 4) + piece] = k;
  if ((piece & 3) == 0) exps[(long long)row * nb + (piece >> 2)] = (unsigned char)byte;
}
template <bool VEC, typename T>
__global__ void unpack8_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ exps, T* __restrict__ x, unsigned rows, int width,
                               long long ld, int nb) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece * 8 >= width) return;
  float f[8];
  decode8(reinterpret_cast<const uint2*>(codes)[(long long)row * (nb * 4) + piece], exps[(long long)row * nb + (piece >> 2)], f);
  store8<VEC>(x + row * ld, piece * 8, width, f);
}

// Value and derivative of the gate's function: 0 silu, 1 gelu by tanh, 2 relu. 16-bit results need 2^-9 of it: the approximate exponential and
// quotient (a few 2^-22) do; 32-bit ones take the exact functions.
template <bool FAST>
__device__ __forceinline__ void gate8(float g, int act, float& a, float& da) {
  if (act == 0) {
    const float s = FAST ? __fdividef(1.f, 1.f + __expf(-g)) : 1.f / (1.f + expf(-g));
    a = FAST ? g * s : g / (1.f + expf(-g));
    da = s * (1.f + g * (1.f - s));
  } else if (act == 1) {
    const float k0 = 0.7978845608028654f, k1 = 0.044715f;
    const float th = tanhf(k0 * (g + k1 * g * g * g));
    a = 0.5f * g * (1.f + th);
    da = 0.5f * (1.f + th) + 0.5f * g * (1.f - th * th) * k0 * (1.f + 3.f * k1 * g * g);
  } else {
    a = fmaxf(g, 0.f);
    da = g > 0.f ? 1.f : 0.f;
  }
}

// gu [rows, 2 width] (gate | up): h = act(gate) * up, and gate and up in 8 bits: codes [rows, 2, 32 nb], exps [rows, 2, nb].
template <bool VEC, typename T>
__global__ void glu8_fwd_kernel(const T* __restrict__ gu, T* __restrict__ h, signed char* __restrict__ codes, unsigned char* __restrict__ exps,
                                unsigned rows, int width, long long ld, int nb, int act) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= nb * 4) return;
  float g[8], u[8];
  load8<VEC>(gu + row * ld, piece * 8, width, g);
  load8<VEC>(gu + row * ld + width, piece * 8, width, u);
  uint32_t gb, ub;
  const uint2 gk = encode8(g, gb), uk = encode8(u, ub);
  uint2* kr = reinterpret_cast<uint2*>(codes) + (long long)row * (nb * 8);
  kr[piece] = gk;
  kr[nb * 4 + piece] = uk;
  if ((piece & 3) == 0) {
    unsigned char* er = exps + (long long)row * (2 * nb);
    er[piece >> 2] = (unsigned char)gb;
    er[nb + (piece >> 2)] = (unsigned char)ub;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float a, da;
    gate8<sizeof(T) == 2>(g[j], act, a, da);
    g[j] = a * u[j];
  }
  store8<VEC>(h + (long long)row * width, piece * 8, width, g);
}
// dgu = (dh * up * act'(gate) | dh * act(gate)) with gate and up as their 8 bits say.
template <bool VEC, typename T>
__global__ void glu8_bwd_kernel(const T* __restrict__ dh, const signed char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                T* __restrict__ dgu, unsigned rows, int width, int nb, int act) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece * 8 >= width) return;
  float g[8], u[8], d[8], dg[8];
  const uint2* kr = reinterpret_cast<const uint2*>(codes) + (long long)row * (nb * 8);
  const unsigned char* er = exps + (long long)row * (2 * nb);
  load8<VEC>(dh + (long long)row * width, piece * 8, width, d);
  decode8(kr[piece], er[piece >> 2], g);
  decode8(kr[nb * 4 + piece], er[nb + (piece >> 2)], u);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float a, da;
    gate8<sizeof(T) == 2>(g[j], act, a, da);
    dg[j] = d[j] * u[j] * da;
    d[j] *= a;
  }
  T* o = dgu + (long long)row * (2 * (long long)width);
  store8<VEC>(o, piece * 8, width, dg);
  store8<VEC>(o + width, piece * 8, width, d);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool act8_args_ok(long long rows, int width, int dtype) { return rows > 0 && rows <= 0x7fffffffll && width > 0 && width <= (1 << 27) && dtype >= 0 && dtype <= 2; }

// dtype 0 bf16, 1 fp16, 2 fp32
template <typename F>
static int by_type(int dtype, F f) {
  if (dtype == 0) f(__nv_bfloat16());
  else if (dtype == 1) f(__half());
  else f(float());
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

}  // namespace sx
using namespace sx;

extern "C" int sx_pack8(const void* x, void* codes, void* exps, long long rows, int width, long long ld, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!act8_args_ok(rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  dim3 grid, block;
  token_grid(rows, nb * 4, &grid, &block);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern) { kern<<<grid, block, 0, st>>>((const T*)x, (signed char*)codes, (unsigned char*)exps, (unsigned)rows, width, ld, nb); };
    if (width % 8 == 0 && ld % 8 == 0 && aligned16(x)) run(pack8_kernel<true, T>);
    else run(pack8_kernel<false, T>);
  });
}
extern "C" int sx_unpack8(const void* codes, const void* exps, void* x, long long rows, int width, long long ld, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!act8_args_ok(rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  dim3 grid, block;
  token_grid(rows, nb * 4, &grid, &block);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern) { kern<<<grid, block, 0, st>>>((const signed char*)codes, (const unsigned char*)exps, (T*)x, (unsigned)rows, width, ld, nb); };
    if (width % 8 == 0 && ld % 8 == 0 && aligned16(x)) run(unpack8_kernel<true, T>);
    else run(unpack8_kernel<false, T>);
  });
}
extern "C" int sx_glu8_fwd(const void* gu, void* h, void* codes, void* exps, long long rows, int width, long long ld, int act, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!act8_args_ok(rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  dim3 grid, block;
  token_grid(rows, nb * 4, &grid, &block);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern) {
      kern<<<grid, block, 0, st>>>((const T*)gu, (T*)h, (signed char*)codes, (unsigned char*)exps, (unsigned)rows, width, ld, nb, act);
    };
    if (width % 8 == 0 && ld % 8 == 0 && aligned16(gu) && aligned16(h)) run(glu8_fwd_kernel<true, T>);
    else run(glu8_fwd_kernel<false, T>);
  });
}
extern "C" int sx_glu8_bwd(const void* dh, const void* codes, const void* exps, void* dgu, long long rows, int width, int act, int dtype,
                           cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!act8_args_ok(rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  dim3 grid, block;
  token_grid(rows, nb * 4, &grid, &block);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern) {
      kern<<<grid, block, 0, st>>>((const T*)dh, (const signed char*)codes, (const unsigned char*)exps, (T*)dgu, (unsigned)rows, width, nb, act);
    };
    if (width % 8 == 0 && aligned16(dh) && aligned16(dgu)) run(glu8_bwd_kernel<true, T>);
    else run(glu8_bwd_kernel<false, T>);
  });
}
