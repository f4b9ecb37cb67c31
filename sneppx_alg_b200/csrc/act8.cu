// L2: activations held in 8 bits between forward and backward, and the gated activation that keeps its input so.
//
// Per 32 consecutive values of a row one exponent byte b and 32 signed codes: x ~ code * 2^(b - 127), with the smallest power of two of which
// round(amax / 2^e) <= 127 steps reach the block's largest magnitude, ties to even. amax = m 2^x with m in [1, 2): e = x - 6, one more from m =
// 255/128 on (127.5 would round to 128), but not where 64 of those steps would be the type's infinity: at the top of its range (65280 on in fp16, from
// 255/256 of 2^128 on in the others) e stays and codes end at 127, which is off by less than a step, half of the step that e + 1 would have.
// Everything but the rounding to whole steps is exact: amax and e come from the bits, x / 2^e is a product with a power of two, code * 2^e has 7 bits and
// fits the type of x. b = 255 marks a block that holds an infinity or a NaN: all of it is restored as NaN, so that an overflow is not hidden. e is at least
// -126, which holds blocks below 2^-120 more coarsely.
// 33 bytes for 32 values. A power of two for 32 values costs what a 32-bit scale for 128 costs and is as near on normal values
// (the block's maximum is smaller by what the step is rounded up), nearer where single values stand out.
//
// All kernels are bound by memory: a thread takes 16 neighbouring values, two threads a block, so that 32 to 64 bytes a thread are on their way.
// Rounding is an addition of 1.5 * 2^23 (the sum's low byte is the code), restoring a byte placed in the mantissa of 2^23: the conversion
// instructions run at an eighth of the rate. Sums and functions are in 32 bits; this file is compiled without fast math, so that 32-bit inputs keep
// their small values.
#include <cuda_fp16.h>
#include <type_traits>
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
// where they are multiples of 8 (PAIR; the block's two threads take its vectors in turn, so that they fill sectors together). Rows that begin anywhere (ODD)
// are read and written by a warp as whole aligned words, 32 next to each other, and turned into 16 neighbouring values a thread and back through shared
// memory; a word that two rows or two warps share is read and written by halves (8192 x 4101 in bf16: packed and restored in 57 us, gated with its gradient
// 167; 78 and 226 with values one by one, 32 apart; 33 and 89 for whole vectors). What bounds them is the issue of instructions, 70 % of the SMs' rate with
// a third of DRAM's: each value goes through shared memory and a shift. Where a row has two blocks at most, of which a warp would be empty otherwise, threads take their 16
// neighbours one by one, and a warp several rows (NEAR: 22222 x 45 packed and restored 11.8 us, 17.5 as ODD; gated 30 and 45; at 77 columns 11.4 and 11.9,
// 30 and 28).
enum { ODD = 0, PAIR = 1, WIDE = 2, NEAR = 3 };
template <int MODE>
__host__ __device__ __forceinline__ int threads_of(int nb) { return MODE == ODD ? (nb + 15) / 16 * 32 : nb * 2; }   // of a row of nb blocks

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
// A warp's part of a row in shared memory: a thread's 32 or 64 bytes and 16 more, so that neither access meets a bank twice.
template <typename T> constexpr int STAGED = 4 * (int)sizeof(T) + 4;                          // words of a thread
template <typename T>
__device__ __forceinline__ int staged(int k) { return sizeof(T) == 2 ? (k >> 3) * 12 + (k & 7) : (k >> 4) * 20 + (k & 15); }
template <int MODE, typename T>
__device__ __forceinline__ uint32_t* stage_of_warp() {
  __shared__ __align__(16) uint32_t stage[MODE == ODD ? 8 * 32 * STAGED<T> : 4];
  return stage + (MODE == ODD ? ((threadIdx.y * blockDim.x + threadIdx.x) >> 5) * 32 * STAGED<T> : 0);
}
__device__ __forceinline__ uint32_t bits16(const void* p) { return *reinterpret_cast<const uint16_t*>(p); }
// c: 16 times the thread's place in the row. ODD: words as they lie, to be settled; `tail` the last thread's word behind the warp's.
template <int MODE, typename T>
__device__ __forceinline__ void load16(const T* row, int c, int width, Row16<T>& v, uint32_t& tail) {
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
  } else if (MODE == NEAR) {
#pragma unroll
    for (int j = 0; j < PER; ++j) v.t[j] = c + j < width ? row[c + j] : Act8<T>::out(0.f);
  } else {
    const int lane = c >> 4 & 31, first = c & ~511, n = width - first;
    const T* p = row + first;
    if (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v.w[j >> 3 & (sizeof(T) / 2 - 1)][j & 7] = lane + 32 * j < n ? reinterpret_cast<const uint32_t*>(p)[lane + 32 * j] : 0u;
    } else {
      const int s = (int)(reinterpret_cast<uintptr_t>(p) >> 1 & 1);      // the first value is a word's second half
      auto word = [&](int k) {                                           // values 2 k - s and the next
        const int lo = 2 * k - s, hi = lo + 1;
        if (lo >= 0 && hi < n) return *reinterpret_cast<const uint32_t*>(p + lo);
        return (lo >= 0 && lo < n ? bits16(p + lo) : 0u) | (hi < n ? bits16(p + hi) << 16 : 0u);
      };
#pragma unroll
      for (int j = 0; j < 8; ++j) v.w[0][j] = word(lane + 32 * j);
      tail = s && lane == 31 ? word(256) : 0u;
    }
  }
}
template <int MODE, typename T>
__device__ __forceinline__ void settle16(const T* row, int c, Row16<T>& v, uint32_t tail, uint32_t* stage) {
  if (MODE != ODD) return;
  const int lane = c >> 4 & 31;
#pragma unroll
  for (int j = 0; j < 4 * (int)sizeof(T); ++j) stage[staged<T>(lane + 32 * j)] = v.w[j >> 3][j & 7];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) v.q[i] = *reinterpret_cast<const uint4*>(stage + lane * STAGED<T> + 4 * i);
  __syncwarp();
  if (sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(row) & 2)) {
    uint32_t next = __shfl_down_sync(0xffffffffu, v.w[0][0], 1);
    if (lane == 31) next = tail;
#pragma unroll
    for (int j = 0; j < 8; ++j) v.w[0][j] = __funnelshift_r(v.w[0][j], j < 7 ? v.w[0][j + 1] : next, 16);
  }
}
template <int MODE, typename T>
__device__ __forceinline__ void store16(T* row, int c, int width, const float (&f)[PER], uint32_t* stage) {
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
  } else if (MODE == NEAR) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (c + j < width) row[c + j] = v.t[j];
  } else {
    const int lane = c >> 4 & 31, first = c & ~511, n = width - first;
    T* p = row + first;
    const int s = sizeof(T) == 2 ? (int)(reinterpret_cast<uintptr_t>(p) >> 1 & 1) : 0;
    if (s) {
      if (lane == 31 && 511 < n) p[511] = v.t[15];
      const uint32_t before = __shfl_up_sync(0xffffffffu, v.w[0][7], 1);
#pragma unroll
      for (int j = 7; j >= 0; --j) v.w[0][j] = __funnelshift_l(j > 0 ? v.w[0][j - 1] : before, v.w[0][j], 16);
    }
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) *reinterpret_cast<uint4*>(stage + lane * STAGED<T> + 4 * i) = v.q[i];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4 * (int)sizeof(T); ++j) {
      const int k = lane + 32 * j;
      const uint32_t x = stage[staged<T>(k)];
      if (sizeof(T) == 4) {
        if (k < n) reinterpret_cast<uint32_t*>(p)[k] = x;
      } else {
        const int lo = 2 * k - s, hi = lo + 1;
        if (lo >= 0 && hi < n) {
          *reinterpret_cast<uint32_t*>(p + lo) = x;
        } else {
          if (lo >= 0 && lo < n) *reinterpret_cast<uint16_t*>(p + lo) = (uint16_t)x;
          if (hi < n) *reinterpret_cast<uint16_t*>(p + hi) = (uint16_t)(x >> 16);
        }
      }
    }
    __syncwarp();
  }
}
template <typename T>
__device__ __forceinline__ void widen(const Row16<T>& v, float (&f)[PER]) {
#pragma unroll
  for (int j = 0; j < PER; ++j) f[j] = Act8<T>::in(v.t[j]);
}

// A block's exponent byte from the bits of its largest magnitude, the factor that turns a value into steps, and the sum whose low byte is the code (to be
// masked out in a block that is not finite: infinity times 0 is a NaN whose low byte may be anything).
template <typename T> constexpr int TOP_BYTE = std::is_same<T, __half>::value ? 15 - 6 + 127 : 127 - 6 + 127;      // of the type's largest values
template <typename T>
__device__ __forceinline__ uint32_t exponent_of(uint32_t top) {
  return top >= 0x7f800000u ? 255u : min(max((int)((top + 0x10000u) >> 23) - 6, 1), TOP_BYTE<T>);
}
__device__ __forceinline__ float per_step(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ uint32_t code_of(float f, float inv) { return __float_as_uint(fmaf(f, inv, 12582912.f)); }
__device__ __forceinline__ uint32_t finite_mask(uint32_t byte) { return byte == 255u ? 0u : 0xffffffffu; }
// 2^(byte - 127); packing makes no byte below 1
__device__ __forceinline__ float step_of(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23); }
// PAIR: word j of four codes of a thread in its block, by vectors of 8 values (16-bit types) or 4.
template <typename T>
__device__ __forceinline__ int word_at(int j, int side) { return sizeof(T) == 2 ? (j >> 1) * 4 + side * 2 + (j & 1) : j * 2 + side; }
// Blocks of a row of nb, from the pairs of threads that hold them: codes and exponents of the row.
template <int MODE, typename T>
__device__ __forceinline__ void encode16(const float (&f)[PER], int place, int nb, signed char* codes, unsigned char* exps) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(3u << ((threadIdx.y * blockDim.x + threadIdx.x) & 30u), top, 1));
  const uint32_t byte = exponent_of<T>(top);
  const float inv = per_step(byte);
  const uint32_t mask = finite_mask(byte);
  uint32_t r[4];
  auto codes_of = [&](auto limited) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k[i] = code_of(f[4 * j + i], inv);
        if (limited) k[i] = min(max((int)k[i], 0x4b400000 - 127), 0x4b400000 + 127);
      }
      r[j] = __byte_perm(__byte_perm(k[0], k[1], 0x0040), __byte_perm(k[2], k[3], 0x0040), 0x5410) & mask;
    }
  };
  if (byte == TOP_BYTE<T>) codes_of(std::true_type());      // rare: 128 steps are 127 here. Apart, so that neither holds sixteen codes in registers at once
  else codes_of(std::false_type());
  if (MODE == ODD && place >= 2 * nb) return;          // the last warp of a row may have threads to spare
  if (MODE != PAIR) {
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
  __device__ __forceinline__ void load(int place, int nb, const signed char* codes, const unsigned char* exps) {
    k = make_uint4(0, 0, 0, 0);
    byte = 1;
    if (MODE == ODD && place >= 2 * nb) return;
    if (MODE != PAIR) {
      k = reinterpret_cast<const uint4*>(codes)[place];
    } else {
      const uint32_t* at = reinterpret_cast<const uint32_t*>(codes) + (place >> 1) * 8;
      const int side = place & 1;
      k = make_uint4(at[word_at<T>(0, side)], at[word_at<T>(1, side)], at[word_at<T>(2, side)], at[word_at<T>(3, side)]);
    }
    byte = exps[place >> 1];
  }
  __device__ __forceinline__ void restore(float (&f)[PER]) const {
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
  uint32_t tail;
  load16<MODE>(x + row * ld, piece * PER, width, v, tail);
  settle16<MODE>(x + row * ld, piece * PER, v, tail, stage_of_warp<MODE, T>());
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
  store16<MODE>(x + row * ld, piece * PER, width, f, stage_of_warp<MODE, T>());
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
    a = g < 0.f ? 0.f : g;                     // NaN stays: it stands for an overflow
    da = g > 0.f ? 1.f : g <= 0.f ? 0.f : g;
  }
}

// gu [rows, 2 width] (gate | up): h = act(gate) * up, and gate and up in 8 bits: codes [rows, 2, 32 nb], exps [rows, 2, nb].
// Blocks of up to 256 threads; 16-bit types forward in 48 registers (ODD 64: 84 us at 8192 x 4101, 87 in 48) and backward in 64: 8192 x 14336 bf16 forward
// 150.5 us, 158 in 64, and backward 147 us, 161 in 48 (both move 947 MB; 180 and 164 in blocks of 448 threads). 32-bit types have more on their way and keep
// the registers that the compiler takes (39 and 38 us at 4096 x 4096; 41 and 42 with fewer).
// HOLD: gate and up are packed; without a gradient to come nothing is (a template argument: a branch takes registers that these blocks do not have).
template <int MODE, bool HOLD, typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? (MODE == ODD ? 4 : 5) : 1)
    glu8_fwd_kernel(const T* __restrict__ gu, T* __restrict__ h, signed char* __restrict__ codes, unsigned char* __restrict__ exps, unsigned rows, int width,
                    long long ld, int nb, int act) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= threads_of<MODE>(nb)) return;
  Row16<T> gv, uv;
  uint32_t gt, ut, *stage = stage_of_warp<MODE, T>();
  load16<MODE>(gu + row * ld, piece * PER, width, gv, gt);
  load16<MODE>(gu + row * ld + width, piece * PER, width, uv, ut);
  settle16<MODE>(gu + row * ld, piece * PER, gv, gt, stage);
  settle16<MODE>(gu + row * ld + width, piece * PER, uv, ut, stage);
  float g[PER], u[PER];
  widen(gv, g);
  widen(uv, u);
  if (HOLD) {
    signed char* kr = codes + (long long)row * (nb * 64);
    unsigned char* er = exps + (long long)row * (2 * nb);
    encode16<MODE, T>(g, piece, nb, kr, er);
    encode16<MODE, T>(u, piece, nb, kr + nb * 32, er + nb);
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    float a, da;
    gate8<sizeof(T) == 2>(g[j], act, a, da);
    g[j] = a * u[j];
  }
  store16<MODE>(h + (long long)row * width, piece * PER, width, g, stage);
}
// dgu = (dh * up * act'(gate) | dh * act(gate)) with gate and up as their 8 bits say.
template <int MODE, typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 1)
    glu8_bwd_kernel(const T* __restrict__ dh, const signed char* __restrict__ codes, const unsigned char* __restrict__ exps, T* __restrict__ dgu,
                    unsigned rows, int width, int nb, int act) {
  const unsigned row = blockIdx.x * blockDim.y + threadIdx.y;
  const int piece = blockIdx.y * blockDim.x + threadIdx.x;
  if (row >= rows || piece >= threads_of<MODE>(nb)) return;
  const signed char* kr = codes + (long long)row * (nb * 64);
  const unsigned char* er = exps + (long long)row * (2 * nb);
  Row16<T> dv;
  uint32_t tail, *stage = stage_of_warp<MODE, T>();
  load16<MODE>(dh + (long long)row * width, piece * PER, width, dv, tail);
  Held16<MODE, T> g8, u8;
  g8.load(piece, nb, kr, er);
  u8.load(piece, nb, kr + nb * 32, er + nb);
  settle16<MODE>(dh + (long long)row * width, piece * PER, dv, tail, stage);
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
  store16<MODE>(o, piece * PER, width, g, stage);
  store16<MODE>(o + width, piece * PER, width, d, stage);
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
  if (width % 8 == 0 && ld * size % 16 == 0 && at % 16 == 0) return PAIR;
  return width <= 64 ? NEAR : ODD;
}
static bool act8_args_ok(const void* values, const void* codes, const void* exps, long long rows, int width, int dtype) {
  return values && !codes == !exps && rows > 0 && rows <= 0x7fffffffll && width > 0 && width <= (1 << 26) && dtype >= 0 && dtype <= 2 &&
         (reinterpret_cast<uintptr_t>(codes) & 15) == 0;
}

// dtype 0 bf16, 1 fp16, 2 fp32
template <typename F>
static int by_type(int dtype, F f) {
  if (dtype == 0) f(__nv_bfloat16());
  else if (dtype == 1) f(__half());
  else f(float());
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

template <typename F>
static void by_mode(int mode, F f) {
  if (mode == WIDE) f(std::integral_constant<int, WIDE>());
  else if (mode == PAIR) f(std::integral_constant<int, PAIR>());
  else if (mode == NEAR) f(std::integral_constant<int, NEAR>());
  else f(std::integral_constant<int, ODD>());
}

}  // namespace sx
using namespace sx;

extern "C" int sx_pack8(const void* x, void* codes, void* exps, long long rows, int width, long long ld, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!codes || !act8_args_ok(x, codes, exps, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int mode = row_mode(width, ld, x, nullptr, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == ODD ? threads_of<ODD>(nb) : threads_of<WIDE>(nb), &grid, &block);
    by_mode(mode, [&](auto m) {
      pack8_kernel<decltype(m)::value, T><<<grid, block, 0, st>>>((const T*)x, (signed char*)codes, (unsigned char*)exps, (unsigned)rows, width, ld, nb);
    });
  });
}
extern "C" int sx_unpack8(const void* codes, const void* exps, void* x, long long rows, int width, long long ld, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!codes || !act8_args_ok(x, codes, exps, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int mode = row_mode(width, ld, x, nullptr, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == ODD ? threads_of<ODD>(nb) : threads_of<WIDE>(nb), &grid, &block);
    by_mode(mode, [&](auto m) {
      unpack8_kernel<decltype(m)::value, T><<<grid, block, 0, st>>>((const signed char*)codes, (const unsigned char*)exps, (T*)x, (unsigned)rows, width, ld,
                                                                    nb);
    });
  });
}
extern "C" int sx_glu8_fwd(const void* gu, void* h, void* codes, void* exps, long long rows, int width, long long ld, int act, int dtype, cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!h || !act8_args_ok(gu, codes, exps, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int mode = row_mode(width, ld, gu, h, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == ODD ? threads_of<ODD>(nb) : threads_of<WIDE>(nb), &grid, &block);
    by_mode(mode, [&](auto m) {
      auto kernel = codes ? glu8_fwd_kernel<decltype(m)::value, true, T> : glu8_fwd_kernel<decltype(m)::value, false, T>;
      kernel<<<grid, block, 0, st>>>((const T*)gu, (T*)h, (signed char*)codes, (unsigned char*)exps, (unsigned)rows, width, ld, nb, act);
    });
  });
}
extern "C" int sx_glu8_bwd(const void* dh, const void* codes, const void* exps, void* dgu, long long rows, int width, int act, int dtype,
                           cudaStream_t st) {
  if (rows == 0 || width == 0) return 0;
  if (!codes || !dgu || !act8_args_ok(dh, codes, exps, rows, width, dtype)) return -1;
  const int nb = (width + 31) / 32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int mode = row_mode(width, width, dh, dgu, sizeof(T));
    dim3 grid, block;
    rows_grid(rows, mode == ODD ? threads_of<ODD>(nb) : threads_of<WIDE>(nb), &grid, &block);
    by_mode(mode, [&](auto m) {
      glu8_bwd_kernel<decltype(m)::value, T><<<grid, block, 0, st>>>((const T*)dh, (const signed char*)codes, (const unsigned char*)exps, (T*)dgu,
                                                                     (unsigned)rows, width, nb, act);
    });
  });
}
