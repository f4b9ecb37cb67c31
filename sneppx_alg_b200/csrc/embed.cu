// L3: embedding lookup with scaling, and its gradient by sorted tokens.
//
//   y[t] = scale * W[id_t]                       dW[v] = scale * sum over { t : id_t = v } of dy[t]
//
// Both are bound by memory. The gradient sorts the tokens by word (stable, so that a word's tokens keep their order), cuts the sorted list into
// pieces of equal length and sums each piece's runs of one word in 32 bits: work does not depend on how often a word occurs, and a batch that is mostly
// one word (padding that is trained on, "the") costs what any other does. A run that leaves its piece is left as a partial sum, and the piece in which
// it began adds the partial sums up in their order. No atomics on sums: the same inputs give the same bits.
// Words that do not occur are known without a table of flags that would have to be cleared: mark[v] holds the position of one token of word v, or
// whatever was there, and only counts if that token exists and is v's.
// Ids outside [0, V) give rows of zeros and no gradient, and ST_BAD_ARGUMENT in the status word.
#include <cuda_fp16.h>
#include <type_traits>
#include "common.cuh"
#include "sx_api.h"

namespace sx {

constexpr int EMB_BAD_ARGUMENT = 5;      // ST_BAD_ARGUMENT (tc_common.cuh)
constexpr int DIGIT_MAX = 9;             // bits of a sorting pass: 512 bins; vocabularies up to 2^18 take two passes
constexpr int TILE_THREADS = 512, TILE_ITEMS = 8, TILE = TILE_THREADS * TILE_ITEMS, TILE_WARPS = TILE_THREADS / 32;

template <typename T> __device__ __forceinline__ float emb_in(T v);
template <> __device__ __forceinline__ float emb_in<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float emb_in<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float emb_in<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T emb_out(float v);
template <> __device__ __forceinline__ __nv_bfloat16 emb_out<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half emb_out<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float emb_out<float>(float v) { return v; }

// Eight neighbouring values in 16-byte accesses (VEC) or one by one up to the row's end.
template <typename T> union Emb8 { uint4 q[sizeof(T) / 2]; T t[8]; };
template <bool VEC, typename T>
__device__ __forceinline__ void emb_load(const T* row, int c, int d, Emb8<T>& v) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v.q[i] = reinterpret_cast<const uint4*>(row + c)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v.t[j] = c + j < d ? row[c + j] : emb_out<T>(0.f);
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void emb_store(T* row, int c, int d, const Emb8<T>& v) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(row + c)[i] = v.q[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < d) row[c + j] = v.t[j];
  }
}

__device__ __forceinline__ long long emb_id(const void* ids, int wide, long long i) {
  return wide ? reinterpret_cast<const long long*>(ids)[i] : (long long)reinterpret_cast<const int*>(ids)[i];
}

template <bool VEC, typename T>
__global__ void embed_fwd_kernel(const void* __restrict__ ids, int wide, const T* __restrict__ w, long long ldw, T* __restrict__ y, unsigned tokens, int d,
                                 long long V, float scale, int* status) {
  const unsigned t = blockIdx.x * blockDim.y + threadIdx.y;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (t >= tokens || c >= d) return;
  const long long id = emb_id(ids, wide, t);
  const bool ok = id >= 0 && id < V;
  Emb8<T> v;
  if (ok) {
    emb_load<VEC>(w + id * ldw, c, d, v);
    if (scale != 1.f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v.t[j] = emb_out<T>(emb_in(v.t[j]) * scale);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v.t[j] = emb_out<T>(0.f);
    if (c == 0 && status) atomicCAS(status, 0, EMB_BAD_ARGUMENT);
  }
  emb_store<VEC>(y + (long long)t * d, c, d, v);
}

// ----------------------------------------------------------------------------- tokens sorted by word
// Radix sort from the lowest digit, each pass stable: counts of a tile's digits, their prefix over the tiles, placement.
// A token's key is its word; padding and ids out of range have the key V and end up behind the rest.
struct SortArgs {
  const void* ids;                  // first pass: the ids themselves
  const unsigned* key_in;           // later passes
  const unsigned* pos_in;
  unsigned* key_out;
  unsigned* pos_out;
  unsigned* counts;                 // [bins, tiles]
  unsigned* totals;                 // [bins]
  unsigned* mark;                   // [V] or null
  int* status;
  long long V, padding;
  unsigned n, tiles;
  int wide, shift, bits;
};

__device__ __forceinline__ unsigned sort_key(const SortArgs& a, unsigned i) {
  if (a.key_in) return a.key_in[i];
  const long long id = emb_id(a.ids, a.wide, i);
  if (id < 0 || id >= a.V) {
    if (a.status) atomicCAS(a.status, 0, EMB_BAD_ARGUMENT);
    return (unsigned)a.V;
  }
  return id == a.padding ? (unsigned)a.V : (unsigned)id;
}

// Ranks of a warp's keys among its own equal digits, in order; cnt: the warp's counters (zero before). Item r of lane l is the warp's (32 r + l)-th.
__device__ __forceinline__ void warp_ranks(const unsigned (&key)[TILE_ITEMS], unsigned first, unsigned n, int shift, unsigned mask, unsigned short* cnt,
                                           unsigned (&rank)[TILE_ITEMS]) {
  const unsigned lane = threadIdx.x & 31;
#pragma unroll
  for (int r = 0; r < TILE_ITEMS; ++r) {
    const bool live = first + r * 32 + lane < n;
    const unsigned digit = live ? (key[r] >> shift) & mask : 0xffffffffu;
    const unsigned same = __match_any_sync(0xffffffffu, digit);
    const unsigned before = live ? cnt[digit] : 0;
    __syncwarp();
    rank[r] = before + __popc(same & ((1u << lane) - 1));
    if (live && (same >> lane) == 1u) cnt[digit] = (unsigned short)(rank[r] + 1);      // the last of its digit
    __syncwarp();
  }
}

__global__ void __launch_bounds__(TILE_THREADS) sort_count_kernel(const SortArgs a) {
  __shared__ unsigned hist[1 << DIGIT_MAX];
  const unsigned bins = 1u << a.bits, mask = bins - 1;
  for (unsigned b = threadIdx.x; b < bins; b += TILE_THREADS) hist[b] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < TILE_ITEMS; ++r) {
    const unsigned i = blockIdx.x * TILE + r * TILE_THREADS + threadIdx.x;
    if (i < a.n) {
      const unsigned k = sort_key(a, i);
      atomicAdd(&hist[(k >> a.shift) & mask], 1u);
      if (a.mark && k < a.V) a.mark[k] = i;
    }
  }
  __syncthreads();
  for (unsigned b = threadIdx.x; b < bins; b += TILE_THREADS) a.counts[(size_t)b * a.tiles + blockIdx.x] = hist[b];
}
// One block a bin: exclusive prefix of its counts over the tiles, and its total.
__global__ void __launch_bounds__(256) sort_prefix_kernel(const SortArgs a) {
  __shared__ unsigned warp_total[8];
  unsigned* row = a.counts + (size_t)blockIdx.x * a.tiles;
  const unsigned lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  unsigned carry = 0;
  for (unsigned t0 = 0; t0 < a.tiles; t0 += 256) {
    const unsigned t = t0 + threadIdx.x, v = t < a.tiles ? row[t] : 0;
    unsigned s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= (unsigned)o) s += u;
    }
    if (lane == 31) warp_total[w] = s;
    __syncthreads();
    unsigned before = carry, all = 0;
#pragma unroll
    for (unsigned k = 0; k < 8; ++k) {
      if (k < w) before += warp_total[k];
      all += warp_total[k];
    }
    if (t < a.tiles) row[t] = before + s - v;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.totals[blockIdx.x] = carry;
}
__global__ void __launch_bounds__(TILE_THREADS) sort_place_kernel(const SortArgs a) {
  __shared__ unsigned short cnt[TILE_WARPS][1 << DIGIT_MAX];
  __shared__ unsigned base[1 << DIGIT_MAX];
  __shared__ unsigned warp_total[TILE_WARPS];
  const unsigned bins = 1u << a.bits, mask = bins - 1, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const unsigned first = blockIdx.x * TILE + w * (32 * TILE_ITEMS);
  unsigned key[TILE_ITEMS], pos[TILE_ITEMS], rank[TILE_ITEMS];
#pragma unroll
  for (int r = 0; r < TILE_ITEMS; ++r) {
    const unsigned i = first + r * 32 + lane;
    key[r] = i < a.n ? sort_key(a, i) : 0;
    pos[r] = i < a.n ? (a.pos_in ? a.pos_in[i] : i) : 0;
  }
  for (unsigned b = lane; b < bins; b += 32) cnt[w][b] = 0;
  __syncwarp();
  warp_ranks(key, first, a.n, a.shift, mask, cnt[w], rank);
  // first place of each bin: exclusive prefix of the bins' totals (512 threads, at most 512 bins), plus what earlier tiles hold
  unsigned v = threadIdx.x < bins ? a.totals[threadIdx.x] : 0, s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= (unsigned)o) s += u;
  }
  if (lane == 31) warp_total[w] = s;
  __syncthreads();
  if (threadIdx.x < bins) {
    unsigned before = s - v;
    for (unsigned k = 0; k < w; ++k) before += warp_total[k];
    base[threadIdx.x] = before + a.counts[(size_t)threadIdx.x * a.tiles + blockIdx.x];
    unsigned run = 0;
    for (int k = 0; k < TILE_WARPS; ++k) {
      const unsigned c = cnt[k][threadIdx.x];
      cnt[k][threadIdx.x] = (unsigned short)run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < TILE_ITEMS; ++r) {
    if (first + r * 32 + lane < a.n) {
      const unsigned digit = (key[r] >> a.shift) & mask;
      const unsigned to = base[digit] + cnt[w][digit] + rank[r];
      a.key_out[to] = key[r];
      a.pos_out[to] = pos[r];
    }
  }
}

// ----------------------------------------------------------------------------- sums of runs
// Thread (x, y): eight columns, piece y of the sorted list. part [pieces, 2, d8]: partial sums of the run that a piece begins in the middle of (0) and
// of the run that begins in it and goes on (1).
template <bool VEC, typename G>
__device__ __forceinline__ void emb_finish(G* grad, long long ldg, unsigned word, int c, int d, const float (&acc)[8], float scale, int add) {
  G* row = grad + (long long)word * ldg;
  Emb8<G> o;
  if (add) {
    emb_load<VEC>(row, c, d, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) o.t[j] = emb_out<G>(emb_in(o.t[j]) + acc[j] * scale);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) o.t[j] = emb_out<G>(acc[j] * scale);
  }
  emb_store<VEC>(row, c, d, o);
}
__device__ __forceinline__ void part_store(float* part, unsigned piece, int side, int d8, int c, const float (&acc)[8]) {
  float4* p = reinterpret_cast<float4*>(part + ((size_t)piece * 2 + side) * d8 + c);
  p[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  p[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
}
template <bool VEC, typename T, typename G>
__global__ void __launch_bounds__(256) embed_sum_kernel(const T* __restrict__ dy, const unsigned* __restrict__ key, const unsigned* __restrict__ pos, G* grad,
                                                        long long ldg, float* __restrict__ part, unsigned n, unsigned len, int d, int d8, unsigned V,
                                                        float scale, int add) {
  const unsigned piece = blockIdx.x * blockDim.y + threadIdx.y;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  const unsigned i0 = piece * len;
  if (i0 >= n || c >= d) return;
  const unsigned i1 = min(n, i0 + len);
  unsigned word = key[i0];
  if (word >= V) return;               // V and beyond stand at the end of the list
  bool open = i0 > 0 && key[i0 - 1] == word;
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  constexpr int U = 8;
  for (unsigned i = i0; i < i1 && word < V; i += U) {
    unsigned k[U];
    Emb8<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k[u] = i + u < i1 ? key[i + u] : 0xffffffffu;
      if (k[u] < V) emb_load<VEC>(dy + (long long)pos[i + u] * d, c, d, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= i1 || word >= V) continue;
      if (k[u] != word) {
        if (open) part_store(part, piece, 0, d8, c, acc);
        else emb_finish<VEC>(grad, ldg, word, c, d, acc, scale, add);
        open = false;
        word = k[u];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      }
      if (word < V) {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += emb_in(v[u].t[j]);
      }
    }
  }
  if (word >= V) return;
  if (open) part_store(part, piece, 0, d8, c, acc);
  else if (i1 < n && key[i1] == word) part_store(part, piece, 1, d8, c, acc);
  else emb_finish<VEC>(grad, ldg, word, c, d, acc, scale, add);
}
// Pieces whose last run begins in them and goes on: its sum over the pieces that it reaches.
template <bool VEC, typename G>
__global__ void __launch_bounds__(256) embed_join_kernel(const unsigned* __restrict__ key, G* grad, long long ldg, const float* __restrict__ part, unsigned n,
                                                         unsigned len, int d, int d8, unsigned V, float scale, int add) {
  const unsigned piece = blockIdx.x * blockDim.y + threadIdx.y;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  const unsigned i0 = piece * len;
  if (i0 >= n || n - i0 <= len || c >= d) return;
  const unsigned i1 = i0 + len, word = key[i1];
  if (word >= V || key[i1 - 1] != word || (key[i0] == word && i0 > 0 && key[i0 - 1] == word)) return;
  float acc[8];
  const float* p = part + ((size_t)piece * 2 + 1) * d8 + c;
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = p[j];
  for (unsigned q = piece + 1;; ++q) {
    p = part + (size_t)q * 2 * d8 + c;
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    acc[0] += a.x; acc[1] += a.y; acc[2] += a.z; acc[3] += a.w;
    acc[4] += b.x; acc[5] += b.y; acc[6] += b.z; acc[7] += b.w;
    const unsigned long long next = (unsigned long long)(q + 1) * len;
    if (next >= n || key[next] != word) break;
  }
  emb_finish<VEC>(grad, ldg, word, c, d, acc, scale, add);
}
// Rows of words that do not occur: 32 at a time a block, their marks read together.
template <bool VEC, typename G>
__global__ void __launch_bounds__(256) embed_zero_kernel(const void* __restrict__ ids, int wide, long long padding, const unsigned* __restrict__ mark, G* grad,
                                                         long long ldg, unsigned n, int d, unsigned V) {
  __shared__ unsigned absent;
  for (unsigned long long v0 = (unsigned long long)blockIdx.x * 32; v0 < V; v0 += (unsigned long long)gridDim.x * 32) {
    __syncthreads();
    if (threadIdx.x < 32) {
      const unsigned v = (unsigned)v0 + threadIdx.x;
      bool zero = v < V;
      if (zero && v != padding) {
        const unsigned m = mark[v];
        zero = m >= n || emb_id(ids, wide, m) != v;
      }
      const unsigned b = __ballot_sync(0xffffffffu, zero);
      if (threadIdx.x == 0) absent = b;
    }
    __syncthreads();
    Emb8<G> z;
#pragma unroll
    for (int j = 0; j < 8; ++j) z.t[j] = emb_out<G>(0.f);
    for (unsigned b = absent; b; b &= b - 1) {
      G* row = grad + (long long)(v0 + __ffs(b) - 1) * ldg;
      for (int c = threadIdx.x * 8; c < d; c += 256 * 8) emb_store<VEC>(row, c, d, z);
    }
  }
}

static bool emb_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static int bits_of(long long v) {
  int b = 1;
  while (b < 62 && (1ll << b) <= v) ++b;
  return b;
}
// Tokens of a piece: enough pieces for eight blocks of 256 threads an SM, 8 tokens at least (one group of loads), 128 at most.
static unsigned piece_len(long long n, int d) {
  const long long want = 148ll * 8 * 256, threads = (d + 7) / 8;
  unsigned len = 8;
  while (len < 128 && n * threads / len > want) len *= 2;
  return len;
}
struct EmbPlan {
  unsigned tiles, len, pieces;
  int passes, bits, d8;
  long long o_key[2], o_pos[2], o_counts, o_totals, o_mark, o_part, bytes;
};
static EmbPlan emb_plan(long long n, long long V, int d, int dense) {
  EmbPlan p;
  const int bits = bits_of(V);           // keys up to V
  p.passes = (bits + DIGIT_MAX - 1) / DIGIT_MAX;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.tiles = (unsigned)((n + TILE - 1) / TILE);
  p.len = piece_len(n, d);
  p.pieces = (unsigned)((n + p.len - 1) / p.len);
  p.d8 = (d + 7) / 8 * 8;
  long long o = 0;
  auto take = [&](long long bytes) {
    const long long at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  for (int i = 0; i < 2; ++i) {
    p.o_key[i] = take(4 * n);
    p.o_pos[i] = take(4 * n);
  }
  p.o_counts = take(4ll * p.tiles << p.bits);
  p.o_totals = take(4ll << p.bits);
  p.o_mark = take(dense ? 4 * V : 0);
  p.o_part = take(8ll * p.pieces * p.d8);
  p.bytes = o;
  return p;
}

}  // namespace sx
using namespace sx;

extern "C" int sx_embed_fwd(const void* ids, int ids_wide, const void* w, long long ldw, void* y, long long tokens, int d, long long V, float scale, int dtype,
                            int* status, cudaStream_t st) {
  if (tokens == 0 || d == 0) return 0;
  if (tokens < 0 || tokens > 0x7fffffffll || d < 0 || d > (1 << 25) || V <= 0 || dtype < 0 || dtype > 2) return -1;
  dim3 grid, block;
  token_grid(tokens, (d + 7) / 8, &grid, &block);
  auto run = [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kern) { kern<<<grid, block, 0, st>>>(ids, ids_wide, (const T*)w, ldw, (T*)y, (unsigned)tokens, d, V, scale, status); };
    if (d % 8 == 0 && ldw % 8 == 0 && emb_aligned(w) && emb_aligned(y)) go(embed_fwd_kernel<true, T>);
    else go(embed_fwd_kernel<false, T>);
  };
  if (dtype == 0) run(__nv_bfloat16());
  else if (dtype == 1) run(__half());
  else run(float());
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

extern "C" long long sx_embed_bwd_workspace(long long tokens, long long V, int d, int add) { return emb_plan(tokens, V, d, !add).bytes; }

extern "C" int sx_embed_bwd(const void* ids, int ids_wide, const void* dy, void* grad, long long ldg, long long tokens, int d, long long V, long long padding,
                            float scale, int add, int dtype, int grad_dtype, void* work, long long work_bytes, int* status, cudaStream_t st) {
  if (d == 0 || (tokens == 0 && add)) return 0;
  if (tokens < 0 || tokens > 0x7fffffffll || d < 0 || d > (1 << 25) || V <= 0 || V > 0x7ffffffell || dtype < 0 || dtype > 2) return -1;
  if (grad_dtype != dtype && grad_dtype != 2) return -2;
  const EmbPlan p = emb_plan(tokens, V, d, !add);
  if (work_bytes < p.bytes || !emb_aligned(work)) return -3;
  uint8_t* b = (uint8_t*)work;
  SortArgs a = {};
  a.ids = ids; a.wide = ids_wide; a.V = V; a.padding = padding; a.n = (unsigned)tokens; a.tiles = p.tiles; a.bits = p.bits;
  a.counts = (unsigned*)(b + p.o_counts); a.totals = (unsigned*)(b + p.o_totals); a.status = status;
  unsigned* mark = (unsigned*)(b + p.o_mark);
  int at = 0;
  for (int pass = 0; pass < p.passes && tokens > 0; ++pass, at ^= 1) {
    a.mark = pass == 0 && !add ? mark : nullptr;
    a.shift = pass * p.bits;
    a.key_out = (unsigned*)(b + p.o_key[at]);
    a.pos_out = (unsigned*)(b + p.o_pos[at]);
    sort_count_kernel<<<p.tiles, TILE_THREADS, 0, st>>>(a);
    sort_prefix_kernel<<<1u << p.bits, 256, 0, st>>>(a);
    sort_place_kernel<<<p.tiles, TILE_THREADS, 0, st>>>(a);
    a.key_in = a.key_out;
    a.pos_in = a.pos_out;
  }
  const unsigned *key = a.key_in, *pos = a.pos_in;
  float* part = (float*)(b + p.o_part);
  const int items = p.d8 / 8;
  dim3 block, grid;
  block.x = items >= 128 ? 128 : (items + 31) / 32 * 32;
  block.y = 256 / block.x;
  grid.x = (p.pieces + block.y - 1) / block.y;
  grid.y = (items + block.x - 1) / block.x;
  auto run = [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    auto go = [&](auto vec) {
      constexpr bool VEC = decltype(vec)::value;
      if (!add) {
        const unsigned blocks = (unsigned)((V + 31) / 32);
        embed_zero_kernel<VEC, G><<<blocks < 148 * 8 ? blocks : 148 * 8, 256, 0, st>>>(ids, ids_wide, padding, mark, (G*)grad, ldg, (unsigned)tokens, d,
                                                                                      (unsigned)V);
      }
      if (tokens == 0) return;
      embed_sum_kernel<VEC, T, G><<<grid, block, 0, st>>>((const T*)dy, key, pos, (G*)grad, ldg, part, (unsigned)tokens, p.len, d, p.d8, (unsigned)V, scale, add);
      if (p.pieces > 1)
        embed_join_kernel<VEC, G><<<grid, block, 0, st>>>(key, (G*)grad, ldg, part, (unsigned)tokens, p.len, d, p.d8, (unsigned)V, scale, add);
    };
    if (d % 8 == 0 && ldg % 8 == 0 && emb_aligned(dy) && emb_aligned(grad)) go(std::true_type());
    else go(std::false_type());
  };
  if (dtype == 2) run(float(), float());
  else if (dtype == 1 && grad_dtype == 1) run(__half(), __half());
  else if (dtype == 1) run(__half(), float());
  else if (grad_dtype == 0) run(__nv_bfloat16(), __nv_bfloat16());
  else run(__nv_bfloat16(), float());
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
