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
// This file is compiled without fast math, so that fp32 tables and gradients keep their values below 2^-126.
#include <cooperative_groups.h>
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

// A thread's place c, a multiple of 8, in a row of d values. VEC (whole 16-byte accesses: d, pitch and base allow them): the values c to c + 7. Else the 32
// threads of a warp share 256 values so that neighbours touch neighbouring ones: value j of a thread is 32 j behind its first (2049 columns: 385 us
// with eight neighbouring values a thread, 97 so). Such rows wait for their loads, of which two-byte ones bring little each: a lookup of 8192 rows of 2049
// in bf16 20.5 us with half of the warps that an SM holds (52 registers), 12.4 at 2048.
template <typename T> union Emb8 { uint4 q[sizeof(T) / 2]; uint32_t w[2 * sizeof(T)]; T t[8]; };
// Eight fp32 values are a sector: with accesses of 16 bytes each sector is touched twice (rows of zeros of [32000, 4096] fp32 128 -> 98 us, of [128256,
// 4096] 446 -> 338).
__device__ __forceinline__ bool emb_sector(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }
template <bool VEC>
__host__ __device__ __forceinline__ int emb_places(int d) { return VEC ? (d + 7) / 8 : (d + 255) / 256 * 32; }   // threads of a row
template <bool VEC>
__device__ __forceinline__ bool emb_has(int c, int d) { return VEC ? c < d : (c & ~255) < d; }
template <bool VEC>
__device__ __forceinline__ int emb_first(int c) { return VEC ? c : (c & ~255) + ((c >> 3) & 31); }
template <bool VEC, typename T>
__device__ __forceinline__ void emb_load(const T* row, int c, int d, Emb8<T>& v) {
  if (VEC && sizeof(T) == 4 && emb_sector(row + c)) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4 % (2 * sizeof(T))]), "=r"(v.w[5 % (2 * sizeof(T))]),
                   "=r"(v.w[6 % (2 * sizeof(T))]), "=r"(v.w[7 % (2 * sizeof(T))])
                 : "l"(row + c));
  } else if (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v.q[i] = reinterpret_cast<const uint4*>(row + c)[i];
  } else {
    const int first = emb_first<VEC>(c);
#pragma unroll
    for (int j = 0; j < 8; ++j) v.t[j] = first + 32 * j < d ? row[first + 32 * j] : emb_out<T>(0.f);
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void emb_store(T* row, int c, int d, const Emb8<T>& v) {
  if (VEC && sizeof(T) == 4 && emb_sector(row + c)) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + c), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]),
                 "r"(v.w[4 % (2 * sizeof(T))]), "r"(v.w[5 % (2 * sizeof(T))]), "r"(v.w[6 % (2 * sizeof(T))]), "r"(v.w[7 % (2 * sizeof(T))])
                 : "memory");
  } else if (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(row + c)[i] = v.q[i];
  } else {
    const int first = emb_first<VEC>(c);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (first + 32 * j < d) row[first + 32 * j] = v.t[j];
  }
}

__device__ __forceinline__ long long emb_id(const void* ids, int wide, long long i) {
  return wide ? reinterpret_cast<const long long*>(ids)[i] : (long long)reinterpret_cast<const int*>(ids)[i];
}

// U tokens of a thread: t0, t0 + step, ... Their ids are read together and then their rows, so that U row pieces are on their way. c0 is a place in the
// row; c_step: to the thread's next one, 0 where it has one only (a loop around it costs the overlap of the loads: 5003 rows of 4096 20.5 us instead
// of 16.3).
template <bool VEC, int U, typename T>
__device__ __forceinline__ void lookup(const void* ids, int wide, const T* __restrict__ w, long long ldw, T* __restrict__ y, unsigned long long t0,
                                       unsigned long long step, unsigned tokens, int c0, int c_step, int d, long long V, float scale, int* status) {
  long long id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned long long t = t0 + u * step;
    id[u] = t < tokens ? emb_id(ids, wide, t) : 0;
    if (id[u] < 0 || id[u] >= V) {
      id[u] = -1;
      if (c0 == 0 && status) atomicCAS(status, 0, EMB_BAD_ARGUMENT);
    }
  }
  int c = c0;
  do {
    Emb8<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (id[u] >= 0) {
        emb_load<VEC>(w + id[u] * ldw, c, d, v[u]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u].t[j] = emb_out<T>(0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned long long t = t0 + u * step;
      if (t >= tokens) break;
      if (scale != 1.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u].t[j] = emb_out<T>(emb_in(v[u].t[j]) * scale);
      }
      emb_store<VEC>(y + (long long)t * d, c, d, v[u]);
    }
    c += c_step;
  } while (c_step > 0 && emb_has<VEC>(c, d));
}
// Block (pieces of a row, tokens). Four tokens a thread where that leaves eight warps for each scheduler (8192 rows of 4096: 23 us with one, 18.8 with four).
template <bool VEC, int U, typename T>
__global__ void embed_fwd_kernel(const void* __restrict__ ids, int wide, const T* __restrict__ w, long long ldw, T* __restrict__ y, unsigned tokens, int d,
                                 long long V, float scale, int* status) {
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  const unsigned long long rows = (unsigned long long)gridDim.x * blockDim.y, t = blockIdx.x * (unsigned long long)blockDim.y + threadIdx.y;
  if (t >= tokens || !emb_has<VEC>(c, d)) return;
  lookup<VEC, U>(ids, wide, w, ldw, y, t, rows, tokens, c, 0, d, V, scale, status);
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
      if (a.mark && !a.key_in && k < a.V) a.mark[k] = i;
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

// The whole sort in one cluster of up to eight CTAs, which exchange counts and tokens through each other's shared memory: 1024 threads of up to eight
// tokens each, so up to 65536 tokens. Two passes over 8192 tokens are one launch instead of six (33 us of kernels, and the host's time for them).
constexpr int CS_THREADS = 1024, CS_WARPS = CS_THREADS / 32, CS_MAX = 8;
struct ClusterSort {
  unsigned long long item[CS_THREADS * TILE_ITEMS];          // key << 32 | position
  unsigned short cnt[CS_WARPS][1 << DIGIT_MAX];
  unsigned hist[1 << DIGIT_MAX];
  unsigned base[1 << DIGIT_MAX];
  unsigned warp_total[16];
};
__device__ __forceinline__ void cluster_sort(ClusterSort& sm, const SortArgs& a, int passes, unsigned* key_out, unsigned* pos_out) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const unsigned lane = threadIdx.x & 31, w = threadIdx.x >> 5, bins = 1u << a.bits, mask = bins - 1;
  const unsigned rounds = (a.n + ctas * CS_THREADS - 1) / (ctas * CS_THREADS), per = rounds * CS_THREADS;   // tokens of a thread, of a CTA
  const unsigned first = rank * per + w * (rounds * 32);
  unsigned key[TILE_ITEMS], pos[TILE_ITEMS], place[TILE_ITEMS];
#pragma unroll
  for (int r = 0; r < TILE_ITEMS; ++r) {
    const unsigned i = first + r * 32 + lane;
    const bool live = r < rounds && i < a.n;
    key[r] = live ? sort_key(a, i) : 0;
    pos[r] = i;
    if (live && a.mark && key[r] < a.V) a.mark[key[r]] = i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * a.bits;
    for (unsigned b = lane; b < bins; b += 32) sm.cnt[w][b] = 0;
    __syncwarp();
#pragma unroll
    for (int r = 0; r < TILE_ITEMS; ++r) {
      if (r >= rounds) break;
      const bool live = first + r * 32 + lane < a.n;
      const unsigned digit = live ? (key[r] >> shift) & mask : 0xffffffffu;
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      const unsigned before = live ? sm.cnt[w][digit] : 0;
      __syncwarp();
      place[r] = before + __popc(same & ((1u << lane) - 1));
      if (live && (same >> lane) == 1u) sm.cnt[w][digit] = (unsigned short)(place[r] + 1);
      __syncwarp();
    }
    __syncthreads();
    // a bin's counts over the CTA's warps: their prefix, and the CTA's count
    if (threadIdx.x < bins) {
      unsigned run = 0;
#pragma unroll 8
      for (int k = 0; k < CS_WARPS; ++k) {
        const unsigned c = sm.cnt[k][threadIdx.x];
        sm.cnt[k][threadIdx.x] = (unsigned short)run;
        run += c;
      }
      sm.hist[threadIdx.x] = run;
    }
    cluster.sync();
    unsigned all = 0, earlier = 0;
    if (threadIdx.x < bins) {
      for (unsigned c = 0; c < ctas; ++c) {
        const unsigned v = *cluster.map_shared_rank(&sm.hist[threadIdx.x], c);
        earlier += c < rank ? v : 0;
        all += v;
      }
    }
    unsigned s = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= (unsigned)o) s += u;
    }
    if (lane == 31 && w < 16) sm.warp_total[w] = s;
    __syncthreads();
    if (threadIdx.x < bins) {
      unsigned before = s - all + earlier;
      for (unsigned k = 0; k < w; ++k) before += sm.warp_total[k];
      sm.base[threadIdx.x] = before;
    }
    __syncthreads();
    const bool last = pass == passes - 1;
#pragma unroll
    for (int r = 0; r < TILE_ITEMS; ++r) {
      if (r >= rounds || first + r * 32 + lane >= a.n) break;
      const unsigned digit = (key[r] >> shift) & mask, to = sm.base[digit] + sm.cnt[w][digit] + place[r];
      if (last) {
        key_out[to] = key[r];
        pos_out[to] = pos[r];
      } else {
        const unsigned cta = to / per;
        *cluster.map_shared_rank(&sm.item[to - cta * per], cta) = (unsigned long long)key[r] << 32 | pos[r];
      }
    }
    cluster.sync();               // all tokens are where they belong, and nobody reads this CTA's counts any more
    if (last) return;
#pragma unroll
    for (int r = 0; r < TILE_ITEMS; ++r) {
      const unsigned i = w * (rounds * 32) + r * 32 + lane;
      if (r < rounds && rank * per + i < a.n) {
        const unsigned long long v = sm.item[i];
        key[r] = (unsigned)(v >> 32);
        pos[r] = (unsigned)v;
      }
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
  if (add) {       // nobody else writes this row in this launch. By whole sectors as fast as vector reductions at the cache, which make small sums 0
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
// Rows of words that do not occur, `words` of up to 32 at a time a block, their marks read together; narrow rows several at once.
template <bool VEC, typename G>
__device__ __forceinline__ void zero_rows(const SortArgs& a, G* grad, long long ldg, int d, unsigned words, unsigned block, unsigned blocks) {
  __shared__ unsigned row_of[32], rows;
  const unsigned threads = blockDim.x * blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
  const unsigned vecs = emb_places<VEC>(d), side = max(threads / vecs, 1u), mine = tid / vecs, c0 = (tid - mine * vecs) * 8;
  Emb8<G> z;
#pragma unroll
  for (int j = 0; j < 8; ++j) z.t[j] = emb_out<G>(0.f);
  for (unsigned long long v0 = (unsigned long long)block * words; v0 < (unsigned long long)a.V; v0 += (unsigned long long)blocks * words) {
    __syncthreads();
    if (tid < 32) {
      const unsigned long long v = v0 + tid;
      bool zero = tid < words && v < (unsigned long long)a.V;
      if (zero && (long long)v != a.padding) {
        const unsigned m = a.mark[v];
        zero = m >= a.n || emb_id(a.ids, a.wide, m) != (long long)v;
      }
      const unsigned b = __ballot_sync(0xffffffffu, zero);
      if (zero) row_of[__popc(b & ((1u << tid) - 1))] = (unsigned)v;
      if (tid == 0) rows = __popc(b);
    }
    __syncthreads();
    if (mine < side) {
      for (unsigned k = mine; k < rows; k += side) {
        G* row = grad + (long long)row_of[k] * ldg;
        for (int c = c0; emb_has<VEC>(c, d); c += threads * 8) emb_store<VEC>(row, c, d, z);
      }
    }
  }
}
// Keys and positions of 32 tokens are read by the lanes at once and passed round; a warp goes from run to run and asks for four rows of a run at a time.
// Most words occur a few times only: what keeps memory busy is many warps, not long loads (eight rows of several runs in registers: 103 of them, a quarter
// of the warps, 93 us instead of 65 for 32768 tokens of 2048). Four rows of eight fp32 values do not fit the 48 registers that five blocks leave (added to
// [32000, 1024] fp32: four blocks 43 us, five 57).
template <bool VEC, typename T, typename G>
__global__ void __launch_bounds__(256, VEC && sizeof(T) == 4 ? 4 : 5)
    embed_sum_kernel(const SortArgs a, const T* __restrict__ dy, G* grad, long long ldg, float* __restrict__ part, unsigned len, int d, int d8, float scale,
                     int add, unsigned blocks_x, unsigned blocks, unsigned words) {
  if (blockIdx.x >= blocks) {          // the gradient is written whole: rows that have no sum, beside those that have
    zero_rows<VEC>(a, grad, ldg, d, words, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const unsigned *key = a.key_out, *pos = a.pos_out, n = a.n, V = (unsigned)a.V;
  const unsigned by = blockIdx.x / blocks_x, piece = (blockIdx.x - by * blocks_x) * blockDim.y + threadIdx.y, lane = threadIdx.x & 31;
  const int c = (by * blockDim.x + threadIdx.x) * 8;
  const unsigned i0 = piece * len;
  if (i0 >= n) return;                 // a warp's threads have one piece
  const unsigned i1 = min(n, i0 + len);
  const unsigned before = i0 > 0 ? key[i0 - 1] : 0xffffffffu, after = i1 < n ? key[i1] : 0xffffffffu;
  const bool mine = emb_has<VEC>(c, d);
  unsigned word = 0xffffffffu;         // none yet
  bool open = false;
  float acc[8];
  for (unsigned base = i0; base < i1; base += 32) {
    const unsigned kl = base + lane < i1 ? key[base + lane] : 0xffffffffu, pl = base + lane < i1 ? pos[base + lane] : 0;
    const unsigned count = __popc(__ballot_sync(0xffffffffu, kl < V));           // V and beyond stand at the end of the list
    unsigned prev = __shfl_up_sync(0xffffffffu, kl, 1);
    if (lane == 0) prev = word;
    const unsigned heads = __ballot_sync(0xffffffffu, kl != prev && kl < V);
    for (unsigned j = 0; j < count;) {
      if (heads >> j & 1) {            // another word
        if (word < V && mine) {
          if (open) part_store(part, piece, 0, d8, c, acc);
          else emb_finish<VEC>(grad, ldg, word, c, d, acc, scale, add);
        }
        const bool none = word >= V;
        word = __shfl_sync(0xffffffffu, kl, j);
        open = none && word == before;
        // the row that the sum will be added to is on its way while the tokens are (68 -> 65 us); a thread whose values lie all behind the row asks for none
        if (add && emb_first<VEC>(c) < d) asm volatile("prefetch.global.L2 [%0];" ::"l"(grad + (long long)word * ldg + emb_first<VEC>(c)));
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = 0.f;
      }
      const unsigned rest = heads & ~((2u << j) - 1), end = rest ? __ffs(rest) - 1 : count;
      for (; j < end; j += 4) {
        Emb8<T> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const unsigned at = __shfl_sync(0xffffffffu, pl, j + u);
          if (j + u < end && mine) emb_load<VEC>(dy + (long long)at * d, c, d, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (j + u < end) {
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += emb_in(v[u].t[k]);
          }
        }
      }
      j = end;
    }
  }
  if (word >= V || !mine) return;
  if (open) {
    part_store(part, piece, 0, d8, c, acc);
  } else if (after == word) {
    part_store(part, piece, 1, d8, c, acc);
  } else {
    emb_finish<VEC>(grad, ldg, word, c, d, acc, scale, add);
  }
}
// Runs that go over several pieces. A block takes 256 columns of eight neighbouring pieces, a warp a piece: it adds up a run that begins there and reaches
// up to 16 more by itself. Longer ones are the whole block's, one after another: warp y every eighth of their partial sums, the eight added in order.
constexpr int JOIN_ALONE = 16;
__device__ __forceinline__ void add_part(float (&acc)[8], const float* part, unsigned piece, int side, int d8, int c) {
  const float4* p = reinterpret_cast<const float4*>(part + ((size_t)piece * 2 + side) * d8 + c);
  const float4 a = p[0], b = p[1];
  acc[0] += a.x; acc[1] += a.y; acc[2] += a.z; acc[3] += a.w;
  acc[4] += b.x; acc[5] += b.y; acc[6] += b.z; acc[7] += b.w;
}
template <bool VEC, typename G>
__global__ void __launch_bounds__(256) embed_join_kernel(const unsigned* __restrict__ key, G* grad, long long ldg, const float* __restrict__ part, unsigned n,
                                                         unsigned len, int d, int d8, unsigned V, float scale, int add) {
  __shared__ float s[8][32][9];
  __shared__ unsigned reach[8];        // pieces behind a warp's own that its run goes on into, where the block adds it up
  const unsigned lane = threadIdx.x, y = threadIdx.y, piece = blockIdx.x * 8 + y;
  const int c = (int)(blockIdx.y * 32 + lane) * 8;
  const bool mine = emb_has<VEC>(c, d);
  const unsigned long long i0 = (unsigned long long)piece * len, i1 = i0 + len;
  unsigned more = 0;
  if (i1 < n) {
    const unsigned word = key[i1], last = key[i1 - 1], head = key[i0], before = i0 > 0 ? key[i0 - 1] : 0xffffffffu;
    if (word < V && last == word && (head != word || before != word)) {
      // how many pieces behind begin with the word: 32 probes 32 pieces apart, then the 32 behind the last that has it
      auto probe = [&](unsigned apart) {
        const unsigned long long at = i1 + (unsigned long long)(more + lane * apart) * len;
        const unsigned b = __ballot_sync(0xffffffffu, at < n && key[at] == word);
        return b == 0xffffffffu ? 32 : __ffs(~b) - 1;
      };
      for (int found = 32; found == 32;) {
        found = probe(32);
        more += found > 0 ? 32 * (found - 1) : 0;
      }
      more += probe(1);
    }
    if (more > 0 && more <= JOIN_ALONE && mine) {
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      add_part(acc, part, piece, 1, d8, c);
#pragma unroll 4
      for (unsigned q = 1; q <= more; ++q) add_part(acc, part, piece + q, 0, d8, c);
      emb_finish<VEC>(grad, ldg, word, c, d, acc, scale, add);
    }
  }
  if (lane == 0) reach[y] = more > JOIN_ALONE ? more : 0;
  __syncthreads();
  for (unsigned k = 0; k < 8; ++k) {
    const unsigned long_more = reach[k];
    if (long_more == 0) continue;      // the same for the whole block
    const unsigned from = blockIdx.x * 8 + k;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (mine) {
#pragma unroll 8
      for (unsigned q = y; q <= long_more; q += 8) add_part(acc, part, from + q, q == 0, d8, c);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[y][lane][j] = acc[j];
    __syncthreads();
    if (y == 0 && mine) {
      for (int i = 1; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += s[i][lane][j];
      emb_finish<VEC>(grad, ldg, key[(unsigned long long)(from + 1) * len], c, d, acc, scale, add);
    }
    __syncthreads();
  }
}
// The first cluster sorts the tokens for the gradient while the other CTAs look the rows up (y null: nothing to look up): the sort, which takes a few
// SMs for 10 to 20 us, costs nothing behind the lookup.
template <bool VEC, typename T>
__global__ void __launch_bounds__(CS_THREADS) embed_sort_lookup_kernel(const SortArgs a, int passes, const T* __restrict__ w, long long ldw, T* __restrict__ y,
                                                                       int d, float scale) {
  extern __shared__ uint8_t smem[];
  const unsigned ctas = cooperative_groups::this_cluster().num_blocks();
  if (blockIdx.x < ctas) {
    cluster_sort(*reinterpret_cast<ClusterSort*>(smem), a, passes, a.key_out, a.pos_out);
    return;
  }
  const unsigned vecs = emb_places<VEC>(d), side = max(CS_THREADS / vecs, 1u), mine = threadIdx.x / vecs, c0 = (threadIdx.x - mine * vecs) * 8;
  if (mine >= side) return;
  const unsigned long long step = (unsigned long long)(gridDim.x - ctas) * side;
  for (unsigned long long t0 = (unsigned long long)(blockIdx.x - ctas) * side + mine; t0 < a.n; t0 += step * 4) {     // the sort reports bad ids
    if (vecs <= CS_THREADS) lookup<VEC, 4>(a.ids, a.wide, w, ldw, y, t0, step, a.n, c0, 0, d, a.V, scale, nullptr);
    else lookup<VEC, 4>(a.ids, a.wide, w, ldw, y, t0, step, a.n, c0, CS_THREADS * 8, d, a.V, scale, nullptr);
  }
}

static bool emb_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static int bits_of(long long v) {
  int b = 1;
  while (b < 62 && (1ll << b) <= v) ++b;
  return b;
}
// Tokens of a piece: as many blocks as run at once, so that none waits for a second round (32768 tokens of 2048, sums and joins: 72 us in one round, 76 in 1.4,
// 75 and 79 in two and three). 8 tokens at least, so that runs are not all cut; 128 at most.
static unsigned piece_len(long long n, int d) {
  const long long slots = 148ll * 5 * 256, threads = (d + 7) / 8, len = (n * threads + slots - 1) / slots;
  return (unsigned)(len < 8 ? 8 : len > 128 ? 128 : len);
}
constexpr long long ONE_CLUSTER = (long long)CS_MAX * CS_THREADS * TILE_ITEMS;
static long long up256(long long bytes) { return (bytes + 255) / 256 * 256; }
// Tokens in the order of their words: keys, positions, and the mark of every word.
struct EmbSorted {
  long long o_pos, o_mark, bytes;
  int passes, bits;
  EmbSorted(long long n, long long V) {
    const int all = bits_of(V);            // keys up to V
    passes = (all + DIGIT_MAX - 1) / DIGIT_MAX;
    bits = (all + passes - 1) / passes;
    o_pos = up256(4 * n);
    o_mark = 2 * o_pos;
    bytes = o_mark + up256(4 * V);
  }
};
// Scratch of the backward pass.
struct EmbWork {
  unsigned tiles, len, pieces;
  int d8;
  long long o_sorted, o_other, o_counts, o_totals, o_part, bytes;
  EmbWork(long long n, long long V, int d, bool presorted) {
    const EmbSorted s(n, V);
    len = piece_len(n, d);
    pieces = (unsigned)((n + len - 1) / len);
    tiles = (unsigned)((n + TILE - 1) / TILE);
    d8 = (d + 255) / 256 * 256;            // a partial sum's floats: places of either kind
    o_part = 0;
    o_sorted = up256(8ll * pieces * d8);
    o_other = o_sorted + (presorted ? 0 : s.bytes);
    o_counts = o_other + (presorted || n <= ONE_CLUSTER ? 0 : 2 * s.o_pos);
    o_totals = o_counts + (presorted || n <= ONE_CLUSTER ? 0 : up256(4ll * tiles << s.bits));
    bytes = o_totals + (presorted || n <= ONE_CLUSTER ? 0 : up256(4ll << s.bits));
  }
};

// One cluster that sorts, as wide as leaves a thread few tokens; with rows to look up, CTAs for them on the other SMs.
template <bool VEC, typename T>
static int launch_sort_lookup(const SortArgs& a, int passes, const T* w, long long ldw, T* y, int d, float scale, cudaStream_t st) {
  auto kern = embed_sort_lookup_kernel<VEC, T>;
  static int fits[64][4];      // clusters of 1, 2, 4, 8 CTAs that a device has room for at once
  int dev = 0, size = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -10;
  while (size < 3 && a.n > CS_THREADS << size) ++size;
  const unsigned ctas = 1u << size;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(CS_THREADS);
  cfg.dynamicSmemBytes = sizeof(ClusterSort);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int room = __atomic_load_n(&fits[dev][size], __ATOMIC_ACQUIRE);
  if (room == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ClusterSort)) != cudaSuccess) return -10;
    if (cudaOccupancyMaxActiveClusters(&room, kern, &cfg) != cudaSuccess || room < 1) return -10;
    __atomic_store_n(&fits[dev][size], room, __ATOMIC_RELEASE);
  }
  if (y) {                     // the tokens are dealt out evenly: no more clusters than run at once
    const long long want = (((long long)a.n * emb_places<VEC>(d) + CS_THREADS - 1) / CS_THREADS + ctas - 1) / ctas, most = room > 1 ? room - 1 : 1;
    cfg.gridDim = dim3(ctas * (unsigned)(1 + (want < most ? want : most)));
  }
  return cudaLaunchKernelEx(&cfg, kern, a, passes, w, ldw, y, d, scale) == cudaSuccess ? 0 : -11;
}
static SortArgs sort_args(const void* ids, int wide, long long tokens, long long V, long long padding, const EmbSorted& s, uint8_t* sorted, int* status) {
  SortArgs a = {};
  a.ids = ids; a.wide = wide; a.V = V; a.padding = padding; a.n = (unsigned)tokens; a.bits = s.bits; a.status = status;
  a.key_out = (unsigned*)sorted;
  a.pos_out = (unsigned*)(sorted + s.o_pos);
  a.mark = (unsigned*)(sorted + s.o_mark);
  return a;
}
static bool emb_args_ok(long long tokens, int d, long long V, int dtype) {
  return tokens >= 0 && tokens <= 0x7fffffffll && d >= 0 && d <= (1 << 25) && V > 0 && V <= 0x7ffffffell && dtype >= 0 && dtype <= 2;
}

}  // namespace sx
using namespace sx;

// Bytes of `sorted`, or 0: so many tokens are not sorted by the forward pass.
extern "C" long long sx_embed_sorted_bytes(long long tokens, long long V) { return tokens > 0 && tokens <= ONE_CLUSTER ? EmbSorted(tokens, V).bytes : 0; }

extern "C" int sx_embed_fwd(const void* ids, int ids_wide, const void* w, long long ldw, void* y, long long tokens, int d, long long V, float scale, int dtype,
                            long long padding, void* sorted, int* status, cudaStream_t st) {
  if (tokens == 0 || d == 0) return 0;
  if (!emb_args_ok(tokens, d, V, dtype) || !ids || !w || !y || (sorted && (tokens > ONE_CLUSTER || (reinterpret_cast<uintptr_t>(sorted) & 255)))) return -1;
  const bool vec = d % 8 == 0 && ldw % 8 == 0 && emb_aligned(w) && emb_aligned(y);
  auto run = [&](auto t, auto v) {
    using T = decltype(t);
    constexpr bool VEC = decltype(v)::value;
    if (sorted) {
      const EmbSorted s(tokens, V);
      return launch_sort_lookup<VEC, T>(sort_args(ids, ids_wide, tokens, V, padding, s, (uint8_t*)sorted, status), s.passes, (const T*)w, ldw, (T*)y, d, scale, st);
    }
    dim3 grid, block;
    const int vecs = emb_places<VEC>(d);
    token_grid(tokens, vecs, &grid, &block);
    if (tokens * vecs >= 4ll * 148 * 1024) {
      grid.x = (grid.x + 3) / 4;
      embed_fwd_kernel<VEC, 4, T><<<grid, block, 0, st>>>(ids, ids_wide, (const T*)w, ldw, (T*)y, (unsigned)tokens, d, V, scale, status);
    } else {
      embed_fwd_kernel<VEC, 1, T><<<grid, block, 0, st>>>(ids, ids_wide, (const T*)w, ldw, (T*)y, (unsigned)tokens, d, V, scale, status);
    }
    return cudaGetLastError() == cudaSuccess ? 0 : -11;
  };
  auto typed = [&](auto t) { return vec ? run(t, std::true_type()) : run(t, std::false_type()); };
  return dtype == 0 ? typed(__nv_bfloat16()) : dtype == 1 ? typed(__half()) : typed(float());
}

extern "C" long long sx_embed_bwd_workspace(long long tokens, long long V, int d, int presorted) { return EmbWork(tokens, V, d, presorted != 0).bytes; }

extern "C" int sx_embed_bwd(const void* ids, int ids_wide, const void* dy, void* grad, long long ldg, long long tokens, int d, long long V, long long padding,
                            float scale, int add, int dtype, int grad_dtype, const void* sorted, void* work, long long work_bytes, int* status,
                            cudaStream_t st) {
  if (d == 0 || (tokens == 0 && add)) return 0;
  if (!emb_args_ok(tokens, d, V, dtype) || !grad || (tokens > 0 && (!ids || !dy || !work))) return -1;
  if (grad_dtype != dtype && grad_dtype != 2) return -2;
  const EmbSorted s(tokens, V);
  const EmbWork p(tokens, V, d, sorted != nullptr);
  if (work_bytes < p.bytes || (reinterpret_cast<uintptr_t>(work) & 255)) return -3;
  uint8_t* b = (uint8_t*)work;
  const bool vec = d % 8 == 0 && ldg % 8 == 0 && emb_aligned(dy) && emb_aligned(grad);
  SortArgs a = sort_args(ids, ids_wide, tokens, V, padding, s, sorted ? (uint8_t*)sorted : b + p.o_sorted, status);
  if (!sorted && tokens > 0 && tokens <= ONE_CLUSTER) {
    const int rc = launch_sort_lookup<true, float>(a, s.passes, nullptr, 0, nullptr, 0, 1.f, st);
    if (rc) return rc;
  } else if (!sorted && tokens > 0) {
    a.tiles = p.tiles;
    a.counts = (unsigned*)(b + p.o_counts);
    a.totals = (unsigned*)(b + p.o_totals);
    for (int pass = 0; pass < s.passes; ++pass) {
      uint8_t* to = (s.passes - pass) % 2 ? b + p.o_sorted : b + p.o_other;        // the last pass ends in o_sorted
      a.shift = pass * s.bits;
      a.key_out = (unsigned*)to;
      a.pos_out = (unsigned*)(to + s.o_pos);
      sort_count_kernel<<<p.tiles, TILE_THREADS, 0, st>>>(a);
      sort_prefix_kernel<<<1u << s.bits, 256, 0, st>>>(a);
      sort_place_kernel<<<p.tiles, TILE_THREADS, 0, st>>>(a);
      a.key_in = a.key_out;
      a.pos_in = a.pos_out;
    }
  }
  const unsigned* key = a.key_out;
  float* part = (float*)(b + p.o_part);
  const int items = vec ? (d + 7) / 8 : p.d8 / 8;
  dim3 block, grid;
  block.x = items >= 128 ? 128 : (items + 31) / 32 * 32;
  block.y = 256 / block.x;
  grid.x = (p.pieces + block.y - 1) / block.y;
  grid.y = (items + block.x - 1) / block.x;
  auto run = [&](auto t, auto g, auto v) {
    using T = decltype(t);
    using G = decltype(g);
    constexpr bool VEC = decltype(v)::value;
    const unsigned sums = grid.x * grid.y;
    // rows of zeros: many short blocks, which fill up what the sums leave, of about 64 KB each ([32000, 4096] fp32 87 us, 96 by 32 words a block; bf16 53 and
    // 64, [128256, 4096] 185 and 196; rows of 128 bytes want all 32: a million of them 74 us, 105 by 16)
    const long long row = (long long)d * sizeof(G);
    const unsigned words = (unsigned)(row >= 16384 ? 4 : row <= 2048 ? 32 : 65536 / row);
    const long long groups = add ? 0 : (V + words - 1) / words;
    embed_sum_kernel<VEC, T, G><<<sums + (unsigned)(groups < 148 * 128 ? groups : 148 * 128), block, 0, st>>>(
        a, (const T*)dy, (G*)grad, ldg, part, p.len, d, p.d8, scale, add, grid.x > 0 ? grid.x : 1, sums, words);
    if (p.pieces > 1)
      embed_join_kernel<VEC, G><<<dim3((p.pieces + 7) / 8, (d + 255) / 256), dim3(32, 8), 0, st>>>(
          key, (G*)grad, ldg, part, (unsigned)tokens, p.len, d, p.d8, (unsigned)V, scale, add);
  };
  auto typed = [&](auto t, auto g) { vec ? run(t, g, std::true_type()) : run(t, g, std::false_type()); };
  if (dtype == 2) typed(float(), float());
  else if (dtype == 1 && grad_dtype == 1) typed(__half(), __half());
  else if (dtype == 1) typed(__half(), float());
  else if (grad_dtype == 0) typed(__nv_bfloat16(), __nv_bfloat16());
  else typed(__nv_bfloat16(), float());
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
