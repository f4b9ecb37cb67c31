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
// All kernels are bound by memory: a thread takes 16 neighbouring values, two threads a block, so that 32 to 64 bytes a thread are on their way.
// Rounding is an addition of 1.5 * 2^23 (the sum's low byte is the code), restoring a byte placed in the mantissa of 2^23: the conversion
// instructions run at an eighth of the rate. Sums and functions are in 32 bits; this file is compiled without fast math, so that 32-bit inputs keep
// their small values.
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

constexpr int PER = 16;      // values of a thread

// How rows are read and written: 32-byte accesses where base, pitch and width are whole multiples of a thread's values (16 of them: WIDE), 16-byte ones
// where they are multiples of 8 (PAIR; the block's two threads take its vectors in turn, so that they fill sectors together). Else one value at a time
// (SINGLE), and a warp then shares 512 values so that neighbouring threads touch
// neighbouring ones: value j of a thread is 32 j behind its first, in the j-th block of the warp's (4101 columns: packed and restored in 222 us with 16
// neighbouring values a thread, 74 so).
enum { SINGLE = 0, PAIR = 1, WIDE = 2 };
template <int MODE>
__host__ __device__ __forceinline__ int threads_of(int nb) { return MODE == SINGLE ? (nb + 15) / 16 * 32 : nb * 2; }   // of a row of nb blocks

__device__ __forceinline__ void ld32(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
__device__ __forceinline__ void st32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
               "r"(r[6]), "r"(r[7])
               : "memory");
}
template <typename T> union Row16 {
  uint32_t w[sizeof(T) / 2][8];
  uint4 q[sizeof(T)];
  T t[PER];
};
// c: 16 times the thread's place in the row
template <int MODE, typename T>
__device__ __forceinline__ void load16(const T* row, int c, int width, Row16<T>& v) {
  if (MODE == WIDE) {
    if (c < width) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) ld32(row + c + i * (32 / (int)sizeof(T)), v.w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) v.q[i] = make_uint4(0, 0, 0, 0);
    }
  } else if (MODE == PAIR) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) {
      const int at = (c & ~31) + (2 * i + (c >> 4 & 1)) * (16 / (int)sizeof(T));
      v.q[i] = at < width ? *reinterpret_cast<const uint4*>(row + at) : make_uint4(0, 0, 0, 0);
    }
  } else {
    const int first = (c & ~511) + ((c >> 4) & 31);
#pragma unroll
    for (int j = 0; j < PER; ++j) v.t[j] = first + 32 * j < width ? row[first + 32 * j] : Act8<T>::out(0.f);
  }
}
template <int MODE, typename T>
__device__ __forceinline__ void store16(T* row, int c, int width, const float (&f)[PER]) {
  Row16<T> v;
#pragma unroll
  for (int j = 0; j < PER; ++j) v.t[j] = Act8<T>::out(f[j]);
  if (MODE == WIDE) {
    if (c < width) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) st32(row + c + i * (32 / (int)sizeof(T)), v.w[i]);
    }
  } else if (MODE == PAIR) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) {
      const int at = (c & ~31) + (2 * i + (c >> 4 & 1)) * (16 / (int)sizeof(T));
      if (at < width) *reinterpret_cast<uint4*>(row + at) = v.q[i];
    }
  } else {
    const int first = (c & ~511) + ((c >> 4) & 31);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (first + 32 * j < width) row[first + 32 * j] = v.t[j];
  }
}
template <typename T>
__device__ __forceinline__ void widen(const Row16<T>& v, float (&f)[PER]) {
#pragma unroll
  for (int j = 0; j < PER; ++j) f[j] = Act8<T>::in(v.t[j]);
}

// A block's exponent byte from the bits of its largest magnitude, the factor that turns a value into steps, and the sum whose low byte is the code (to be
// masked out in a block that is not finite: infinity times 0 is a NaN whose low byte may be anything).
__device__ __forceinline__ uint32_t exponent_of(uint32_t top) { return top >= 0x7f800000u ? 255u : max((int)((top + 0x10000u) >> 23) - 6, 1); }
__device__ __forceinline__ float per_step(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ uint32_t code_of(float f, float inv) { return __float_as_uint(fmaf(f, inv, 12582912.f)); }
__device__ __forceinline__ uint32_t finite_mask(uint32_t byte) { return byte == 255u ? 0u : 0xffffffffu; }
// 2^(byte - 127); packing makes no byte below 1
__device__ __forceinline__ float step_of(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23); }
// PAIR: word j of four codes of a thread in its block, by vectors of 8 values (16-bit types) or 4.
template <typename T>
__device__ __forceinline__ int word_at(int j, int side) { return sizeof(T) == 2 ? (j >> 1) * 4 + side * 2 + (j & 1) : j * 2 + side; }
// Blocks of a row of nb, from the threads of whole warps (SINGLE) or pairs that hold them: codes and exponents of the row.
template <int MODE, typename T>
__device__ __forceinline__ void encode16(const float (&f)[PER], int place, int nb, signed char* codes, unsigned char* exps) {
  if (MODE == SINGLE) {
    const int lane = place & 31, first = (place >> 5) * 16;      // the warp's first block
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (first + j >= nb) break;                                // uniform across the warp
      const uint32_t byte = exponent_of(__reduce_max_sync(0xffffffffu, __float_as_uint(f[j]) & 0x7fffffffu));
      codes[(first + j) * 32 + lane] = (signed char)(code_of(f[j], per_step(byte)) & finite_mask(byte));
      if (lane == j) mine = byte;
    }
    if (lane < PER && first + lane < nb) exps[first + lane] = (unsigned char)mine;
    return;
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(3u << ((threadIdx.y * blockDim.x + threadIdx.x) & 30u), top, 1));
  const uint32_t byte = exponent_of(top);
  const float inv = per_step(byte);
  const uint32_t mask = finite_mask(byte);
  uint32_t k[PER], r[4];
#pragma unroll
  for (int j = 0; j < PER; ++j) k[j] = code_of(f[j], inv);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r[j] = __byte_perm(__byte_perm(k[4 * j], k[4 * j + 1], 0x0040), __byte_perm(k[4 * j + 2], k[4 * j + 3], 0x0040), 0x5410) & mask;
  if (MODE == WIDE) {
    reinterpret_cast<uint4*>(codes)[place] = make_uint4(r[0], r[1], r[2], r[3]);
  } else {
    uint32_t* at = reinterpret_cast<uint32_t*>(codes) + (place >> 1) * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) at[word_at<T>(j, place & 1)] = r[j];
  }
  if ((place & 1) == 0) exps[place >> 1] = (unsigned char)byte;
}
template <int MODE, typename T>
struct Held16 {                                                  // read first, restored when the other operands are there
  uint4 k;
  uint32_t byte;
  signed char c[MODE == SINGLE ? PER : 1];
  __device__ __forceinline__ void load(int place, int nb, const signed char* codes, const unsigned char* exps) {
    if (MODE == SINGLE) {
      const int lane = place & 31, first = (place >> 5) * 16;
      byte = lane < PER && first + lane < nb ? exps[first + lane] : 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) c[MODE == SINGLE ? j : 0] = first + j < nb ? codes[(first + j) * 32 + lane] : 0;
    } else {
      if (MODE == WIDE) {
        k = reinterpret_cast<const uint4*>(codes)[place];
      } else {
        const uint32_t* at = reinterpret_cast<const uint32_t*>(codes) + (place >> 1) * 8;
        const int side = place & 1;
        k = make_uint4(at[word_at<T>(0, side)], at[word_at<T>(1, side)], at[word_at<T>(2, side)], at[word_at<T>(3, side)]);
      }
      byte = exps[place >> 1];
    }
  }
  __device__ __forceinline__ void restore(float (&f)[PER]) const {
    if (MODE == SINGLE) {
#pragma unroll
      for (int j = 0; j < PER; ++j) f[j] = (float)c[MODE == SINGLE ? j : 0] * step_of(__shfl_sync(0xffffffffu, byte, j));
      return;
    }
    const float step = step_of(byte);
    const uint32_t r[4] = {k.x ^ 0x80808080u, k.y ^ 0x80808080u, k.z ^ 0x80808080u, k.w ^ 0x80808080u};
#pragma unroll
    for (int j = 0; j < PER; ++j) f[j] = (__uint_as_float(__byte_perm(r[j / 4], 0x4b000000u, 0x7440 | (j & 3))) - 8388736.f) * step;
  }
};

// x [rows, width] (pitch ld) -> codes [rows, 32 nb], exps [rows, nb], nb = ceil(width / 32); codes behind the row are 0.
template <int MODE, typename T>
__global__ void pack8_kernel(const T* __restrict__ x, signed char* __restrict__ codes, unsigned char* __restrict__ exps, unsigned rows, int width,
                             long long ld, int nb) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= threads_of<MODE>(nb)) return;     // by twos, or by whole warps, as the block's size is
  Row16<T> v;
  load16<MODE>(x + row * ld, piece * PER, width, v);
  float f[PER];
  widen(v, f);
  encode16<MODE, T>(f, piece, nb, codes + (long long)row * (nb * 32), exps + (long long)row * nb);
}
template <int MODE, typename T>
__global__ void unpack8_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ exps, T* __restrict__ x, unsigned rows, int width,
                               long long ld, int nb) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= threads_of<MODE>(nb)) return;
  float f[PER];
  Held16<MODE, T> x8;
  x8.load(piece, nb, codes + (long long)row * (nb * 32), exps + (long long)row * nb);
  x8.restore(f);
  store16<MODE>(x + row * ld, piece * PER, width, f);
}

// Value and derivative of the gate's function: 0 silu, 1 gelu by tanh, 2 relu. Both smooth ones by a logistic function s: gelu's (1 + tanh y) / 2 is
// s(2 y), which loses nothing for negative g. 16-bit results need 2^-9 of it: e^-x = 2^(-x log2 e) and a reciprocal by the approximate instructions (a few
// 2^-22) do, whose results below 2^-126 are 0 (forward at 8192 x 14336 150.5 us; 156 by __expf and __fdividef); 32-bit ones take the exact functions.
template <bool FAST>
__device__ __forceinline__ float logistic(float x) {
  if (!FAST) return 1.f / (1.f + expf(-x));
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}
template <bool FAST>
__device__ __forceinline__ void gate8(float g, int act, float& a, float& da) {
  if (act == 0) {
    const float s = logistic<FAST>(g);
    a = g * s;
    da = fmaf(a, 1.f - s, s);
  } else if (act == 1) {
    const float k0 = 0.7978845608028654f, k1 = 0.044715f;
    const float s = logistic<FAST>(2.f * k0 * g * fmaf(k1 * g, g, 1.f));
    a = g * s;
    da = fmaf(2.f * a * (1.f - s), k0 * fmaf(3.f * k1 * g, g, 1.f), s);
  } else {
    a = fmaxf(g, 0.f);
    da = g > 0.f ? 1.f : 0.f;
  }
}

// gu [rows, 2 width] (gate | up): h = act(gate) * up, and gate and up in 8 bits: codes [rows, 2, 32 nb], exps [rows, 2, nb].
// Blocks of up to 256 threads; 16-bit types forward in 48 registers and backward in 64: 8192 x 14336 bf16 forward 150.5 us, 158 in 64, and backward 147 us,
// 161 in 48 (both move 947 MB; 180 and 164 in blocks of 448 threads). 32-bit types have more on their way and keep the registers that the compiler takes (39
// and 38 us at 4096 x 4096; 41 and 42 with fewer).
template <int MODE, typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 5 : 1) glu8_fwd_kernel(const T* __restrict__ gu, T* __restrict__ h, signed char* __restrict__ codes, unsigned char* __restrict__ exps,
                                unsigned rows, int width, long long ld, int nb, int act) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= threads_of<MODE>(nb)) return;
  Row16<T> gv, uv;
  load16<MODE>(gu + row * ld, piece * PER, width, gv);
  load16<MODE>(gu + row * ld + width, piece * PER, width, uv);
  float g[PER], u[PER];
  widen(gv, g);
  widen(uv, u);
  signed char* kr = codes + (long long)row * (nb * 64);
  unsigned char* er = exps + (long long)row * (2 * nb);
  encode16<MODE, T>(g, piece, nb, kr, er);
  encode16<MODE, T>(u, piece, nb, kr + nb * 32, er + nb);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    float a, da;
    gate8<sizeof(T) == 2>(g[j], act, a, da);
    g[j] = a * u[j];
  }
  store16<MODE>(h + (long long)row * width, piece * PER, width, g);
}
// dgu = (dh * up * act'(gate) | dh * act(gate)) with gate and up as their 8 bits say.
template <int MODE, typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 1) glu8_bwd_kernel(const T* __restrict__ dh, const signed char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                T* __restrict__ dgu, unsigned rows, int width, int nb, int act) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= threads_of<MODE>(nb)) return;
  const signed char* kr = codes + (long long)row * (nb * 64);
  const unsigned char* er = exps + (long long)row * (2 * nb);
  Row16<T> dv;
  load16<MODE>(dh + (long long)row * width, piece * PER, width, dv);
  Held16<MODE, T> g8, u8;
  g8.load(piece, nb, kr, er);
  u8.load(piece, nb, kr + nb * 32, er + nb);
  float g[PER], u[PER], d[PER];
  g8.restore(g);
  u8.restore(u);
  widen(dv, d);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    float a, da;
    gate8<sizeof(T) == 2>(g[j], act, a, da);
    g[j] = d[j] * u[j] * da;
    d[j] *= a;
  }
  T* o = dgu + (long long)row * (2 * (long long)width);
  store16<MODE>(o, piece * PER, width, g);
  store16<MODE>(o + width, piece * PER, width, d);
}

// As token_grid, but rows of 128 threads and more in blocks of 128 at most: a block's registers are what limits how many run.
static void rows_grid(long long rows, int threads, dim3* grid, dim3* block) {
  if (threads < 128) return token_grid(rows, threads, grid, block);
  const int parts = (threads + 127) / 128;
  *block = dim3(((threads + parts - 1) / parts + 31) / 32 * 32);
  *grid = dim3((unsigned)rows, parts);
}
static int row_mode(int width, long long ld, const void* p, const void* q, int size) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q);
  if (width % PER == 0 && ld * size % 32 == 0 && at % 32 == 0) return WIDE;
  return width % 8 == 0 && ld * size % 16 == 0 && at % 16 == 0 ? PAIR : SINGLE;
}
static bool act8_args_ok(const void* codes, long long rows, int width, int dtype) {
  return rows > 0 && rows <= 0x7fffffffll && width > 0 && width <= (1 << 26) && dtype >= 0 && dtype <= 2 && (reinterpret_cast<uintptr_t>(codes) & 15) == 0;
}

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
  if (!act8_args_ok(codes, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern, dim3 grid, dim3 block) { kern<<<grid, block, 0, st>>>((const T*)x, (signed char*)codes, (unsigned char*)exps, (unsigned)rows, width, ld, nb); };
    const int mode = row_mode(width, ld, x, nullptr, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == SINGLE ? threads_of<SINGLE>(nb) : threads_of<WIDE>(nb), &grid, &block);
    mode == WIDE ? run(pack8_kernel<WIDE, T>, grid, block) : mode == PAIR ? run(pack8_kernel<PAIR, T>, grid, block) : run(pack8_kernel<SINGLE, T>, grid, block);
  });
}
extern "C" int sx_unpack8(const void* codes, const void* exps, void* x, long long rows, int width, long long ld, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!act8_args_ok(codes, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern, dim3 grid, dim3 block) { kern<<<grid, block, 0, st>>>((const signed char*)codes, (const unsigned char*)exps, (T*)x, (unsigned)rows, width, ld, nb); };
    const int mode = row_mode(width, ld, x, nullptr, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == SINGLE ? threads_of<SINGLE>(nb) : threads_of<WIDE>(nb), &grid, &block);
    mode == WIDE ? run(unpack8_kernel<WIDE, T>, grid, block) : mode == PAIR ? run(unpack8_kernel<PAIR, T>, grid, block) : run(unpack8_kernel<SINGLE, T>, grid, block);
  });
}
extern "C" int sx_glu8_fwd(const void* gu, void* h, void* codes, void* exps, long long rows, int width, long long ld, int act, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!act8_args_ok(codes, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern, dim3 grid, dim3 block) {
      kern<<<grid, block, 0, st>>>((const T*)gu, (T*)h, (signed char*)codes, (unsigned char*)exps, (unsigned)rows, width, ld, nb, act);
    };
    const int mode = row_mode(width, ld, gu, h, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == SINGLE ? threads_of<SINGLE>(nb) : threads_of<WIDE>(nb), &grid, &block);
    mode == WIDE ? run(glu8_fwd_kernel<WIDE, T>, grid, block) : mode == PAIR ? run(glu8_fwd_kernel<PAIR, T>, grid, block) : run(glu8_fwd_kernel<SINGLE, T>, grid, block);
  });
}
extern "C" int sx_glu8_bwd(const void* dh, const void* codes, const void* exps, void* dgu, long long rows, int width, int act, int dtype,
                           cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!act8_args_ok(codes, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto kern, dim3 grid, dim3 block) {
      kern<<<grid, block, 0, st>>>((const T*)dh, (const signed char*)codes, (const unsigned char*)exps, (T*)dgu, (unsigned)rows, width, nb, act);
    };
    const int mode = row_mode(width, width, dh, dgu, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == SINGLE ? threads_of<SINGLE>(nb) : threads_of<WIDE>(nb), &grid, &block);
    mode == WIDE ? run(glu8_bwd_kernel<WIDE, T>, grid, block) : mode == PAIR ? run(glu8_bwd_kernel<PAIR, T>, grid, block) : run(glu8_bwd_kernel<SINGLE, T>, grid, block);
  });
}
