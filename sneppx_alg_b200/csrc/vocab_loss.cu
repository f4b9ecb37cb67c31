// L4: per-token losses of a vocabulary projection, in tiles of the vocabulary, without the logits ever being held.
//
//   z = h w^T, soft-capped: c tanh(z / c);   lse = log sum_v e^{z_v};   nll = lse - z_target
//   dz_v = ((g_nll + g_lse) e^{z_v - lse} - g_nll [v = target]) (1 - (z_v / c)^2)
//
// One kernel, two epilogues, on the CTA-pair GEMM (256 x 256 tiles, accumulators double-buffered in TMEM, operands by TMA):
//   forward  each row's maximum and sum of exponentials over half a tile's columns (128) leave the SM as one pair of numbers, the target's logit by
//            itself; a second kernel joins the pairs of a row. 8 bytes leave for 128 logits.
//   backward the tile is computed again and leaves as dz in bf16 (half a step, 2^-9, of each value: what the products that follow take), for one piece of the
//            vocabulary at a time; the products dh += dz w and dw = dz^T h run on the GEMM kernel.
// Eight epilogue warps (four TMEM quadrants, two halves of the columns) keep the exponentials behind the products of widths from 256 on.
// Takes the place of the reference's softmax / cross-entropy kernels (kernel/cuda/autodiff_cuda.cu:519-608).
#include "tc_common.cuh"
#include "tc_pair.cuh"
#include "common.cuh"
#include "tmap.h"
#include "sx_api.h"

namespace sx {

constexpr int VL_BK = 64;
constexpr int VL_STAGES = 6;
constexpr int VL_A_BYTES = 128 * VL_BK * 2;
constexpr int VL_STAGE_BYTES = 2 * VL_A_BYTES;       // this CTA's 128 rows of h and of w
constexpr int VL_SMEM = VL_STAGES * VL_STAGE_BYTES + 1024 + 256;
constexpr int VL_EPI_WARPS = 8;
constexpr int VL_THREADS = 64 + 32 * VL_EPI_WARPS;
constexpr float LOG2E = 1.4426950408889634f;

struct VocabLossParams {
  CUtensorMap tmA, tmB;       // h [T, d], w [V, d]
  const long long* target;
  long long ignore_index;
  float2* part;               // forward: [2 n_blks, T] maximum and sum
  float* zt;                  // forward: [T] the target's logit
  const float* lse;           // backward
  const float* g_nll;         // backward: [T] or null
  const float* g_lse;
  __nv_bfloat16* dz;          // backward: [rows, ld]
  long long ld;
  int* status;
  int T, V, rows, d, v0, v1;  // columns [v0, v1) of the vocabulary
  int m_blks, n_blks;
  float cap, inv_cap;         // 0: none
};

template <bool GRAD, bool CAP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(VL_THREADS, 1) vocab_loss_kernel(const __grid_constant__ VocabLossParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + VL_STAGES * VL_STAGE_BYTES);   // even CTA: both CTAs' loads complete on it
  uint64_t* empty_bar = full_bar + VL_STAGES;
  uint64_t* tfull_bar = empty_bar + VL_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;                                                  // even CTA: the epilogue warps of both
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* s_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < VL_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull_bar[i], 1);
      mbar_init(&tempty_bar[i], 2 * VL_EPI_WARPS);
    }
    *s_abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&p.tmA);
    tma_prefetch_desc(&p.tmB);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barriers of both CTAs are initialised before any remote arrive or TMA completion
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total_tiles = p.m_blks * p.n_blks;
  const int num_kb = (p.d + VL_BK - 1) / VL_BK;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = cluster_id; t < total_tiles && ok; t += n_clusters) {
        int b, m_blk, n_blk;
        tile_coords(t, p.m_blks, p.n_blks, b, m_blk, n_blk);
        const int arow = m_blk * 256 + (int)rank * 128, brow = p.v0 + n_blk * 256 + (int)rank * 128;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, s_abort, p.status, ST_TIMEOUT_PRODUCER)) { ok = false; break; }
          uint8_t* sa = smem + stage * VL_STAGE_BYTES;
          if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * VL_STAGE_BYTES);
          const uint32_t fb = smem_u32(&full_bar[stage]) & PEER_MASK;
          tma2_load_3d(sa, &p.tmA, fb, kb * VL_BK, arow, 0);
          tma2_load_3d(sa + VL_A_BYTES, &p.tmB, fb, kb * VL_BK, brow, 0);
          if (++stage == VL_STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA only)
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc_f16(256, 256, 1, 0, 0);
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      for (int t = cluster_id; t < total_tiles && ok; t += n_clusters, ++it) {
        const int acc = it & 1;
        if (!mbar_wait(&tempty_bar[acc], ((it >> 1) & 1) ^ 1, s_abort, p.status, ST_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, s_abort, p.status, ST_TIMEOUT_MMA)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * VL_STAGE_BYTES), sb = sa + VL_A_BYTES;
#pragma unroll
          for (int k = 0; k < VL_BK / 16; ++k)
            umma2_f16_ss(d_tmem, umma_desc_sw128(sa + k * 32, 16, 1024), umma_desc_sw128(sb + k * 32, 16, 1024), idesc, (kb | k) != 0 ? 1u : 0u);
          umma2_commit_pair(&empty_bar[stage]);
          if (++stage == VL_STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) umma2_commit_pair(&tfull_bar[acc]);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue: a row a lane, 128 columns a warp
    const int q = warp & 3, half = (warp - 2) >> 2;
    int it = 0;
    for (int t = cluster_id; t < total_tiles; t += n_clusters, ++it) {
      int b, m_blk, n_blk;
      tile_coords(t, p.m_blks, p.n_blks, b, m_blk, n_blk);
      const int acc = it & 1;
      const int row = m_blk * 256 + (int)rank * 128 + q * 32 + lane;
      const int first = p.v0 + n_blk * 256 + half * 128;          // this warp's first column
      // the target as a column of this warp's 128, or far from them
      int tgt = -1;
      float a = 0.f, gn = 0.f, off = 0.f;
      if (row < p.T) {
        const long long tv = p.target[row];
        if (tv != p.ignore_index && tv >= first && tv < first + 128 && tv < p.v1) tgt = (int)(tv - first);
        if (GRAD) {
          if (p.g_nll && tv != p.ignore_index && tv >= 0 && tv < p.V) gn = p.g_nll[row];
          a = gn + (p.g_lse ? p.g_lse[row] : 0.f);
          off = -p.lse[row] * LOG2E;
        }
      }
      if (!mbar_wait_warp(&tfull_bar[acc], (it >> 1) & 1, s_abort, p.status, ST_TIMEOUT_EPILOGUE)) break;
      tc_fence_after();
      float mx = -INFINITY, sum = 0.f, zt = 0.f;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const int col0 = first + c * 32;
        if (GRAD ? col0 - p.v0 >= p.ld : col0 >= p.v1) break;     // uniform across the warp
        uint32_t r[32];
        tmem_ld32(tmem_base + acc * 256 + half * 128 + c * 32 + (static_cast<uint32_t>(q * 32) << 16), r);
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = CAP ? softcap(__uint_as_float(r[j]), p.cap, p.inv_cap) : __uint_as_float(r[j]);
        const int left = p.v1 - col0;                             // columns that the vocabulary has here
        const bool mine = (tgt >> 5) == c;                        // -1 >> 5 is -1
        if (!GRAD) {
          if (left < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= left) v[j] = -INFINITY;
          }
          if (__any_sync(0xffffffffu, mine)) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (mine && (tgt & 31) == j) zt = v[j];
          }
          float top = v[0];
#pragma unroll
          for (int j = 1; j < 31; j += 2) top = fmax3(top, v[j], v[j + 1]);
          top = fmaxf(fmaxf(top, v[31]), mx);
          const float at = top == -INFINITY ? 0.f : top * LOG2E;
          sum *= exp2f(fmaf(mx, LOG2E, -at));
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            s0 += exp2f(fmaf(v[j], LOG2E, -at));
            s1 += exp2f(fmaf(v[j + 1], LOG2E, -at));
          }
          sum += s0 + s1;
          mx = top;
        } else {
          float g[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = a * exp2f(fmaf(v[j], LOG2E, off));
          if (__any_sync(0xffffffffu, mine)) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (mine && (tgt & 31) == j) g[j] -= gn;
          }
          if (CAP) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float u = v[j] * p.inv_cap;
              g[j] *= fmaf(-u, u, 1.f);
            }
          }
          if (left < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= left) g[j] = 0.f;
          }
          if (row < p.rows) {
            uint4* o = reinterpret_cast<uint4*>(p.dz + (long long)row * p.ld + (col0 - p.v0));
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              o[j / 8] = make_uint4(pack_bf16x2(g[j], g[j + 1]), pack_bf16x2(g[j + 2], g[j + 3]), pack_bf16x2(g[j + 4], g[j + 5]),
                                    pack_bf16x2(g[j + 6], g[j + 7]));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_even_cta(&tempty_bar[acc]);
      if (!GRAD && row < p.T) {
        p.part[(long long)(n_blk * 2 + half) * p.T + row] = make_float2(mx, sum);
        if (tgt >= 0) p.zt[row] = zt;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*s_abort) bounded_delay_ns(2000000);  // let copies in flight land before freeing
  cluster_sync_all();  // neither CTA leaves (or frees TMEM) while its peer may still read its memory or signal it
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

// Joins the parts of 32 rows a block, 16 threads a row. The last logarithm is taken in 64 bits: one a row.
__global__ void __launch_bounds__(512) vocab_loss_join_kernel(const float2* __restrict__ part, const float* __restrict__ zt,
                                                              const long long* __restrict__ target, float* __restrict__ nll, float* __restrict__ lse, int T,
                                                              int V, int parts, long long ignore_index, int* status) {
  __shared__ float2 s[16][33];
  const int row = blockIdx.x * 32 + threadIdx.x;
  float mx = -INFINITY, sum = 0.f;
  if (row < T) {
    for (int i = threadIdx.y; i < parts; i += 16) {
      const float2 v = part[(long long)i * T + row];
      const float top = fmaxf(mx, v.x), at = top == -INFINITY ? 0.f : top * LOG2E;
      sum = sum * exp2f(fmaf(mx, LOG2E, -at)) + v.y * exp2f(fmaf(v.x, LOG2E, -at));
      mx = top;
    }
  }
  s[threadIdx.y][threadIdx.x] = make_float2(mx, sum);
  __syncthreads();
  if (threadIdx.y != 0 || row >= T) return;
  for (int i = 1; i < 16; ++i) {
    const float2 v = s[i][threadIdx.x];
    const float top = fmaxf(mx, v.x), at = top == -INFINITY ? 0.f : top * LOG2E;
    sum = sum * exp2f(fmaf(mx, LOG2E, -at)) + v.y * exp2f(fmaf(v.x, LOG2E, -at));
    mx = top;
  }
  const float l = (float)((double)mx + log((double)sum));
  const long long t = target[row];
  const bool valid = t != ignore_index && t >= 0 && t < V;
  if (t != ignore_index && !valid && status) atomicCAS(status, 0, (int)ST_BAD_ARGUMENT);
  lse[row] = l;
  nll[row] = valid ? l - zt[row] : 0.f;
}

static int vocab_loss_map(CUtensorMap* tm, const void* ptr, int d, long long rows, long long ld) {
  uint64_t dims[3] = {(uint64_t)d, (uint64_t)rows, 1};
  uint64_t strides[2] = {(uint64_t)ld * 2, (uint64_t)ld * rows * 2};
  uint32_t box[3] = {VL_BK, 128, 1};
  return make_tmap(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, ptr, dims, strides, box);
}

static int vocab_loss_setup(VocabLossParams* p, const void* h, long long ldh, const void* w, long long ldw, long long T, long long V, int d, float cap) {
  if (T <= 0 || T > (1 << 30) || V <= 0 || V > (1 << 30) || d <= 0 || d > (1 << 30) || d % 8 || ldh % 8 || ldw % 8 || ldh < d || ldw < d) return -1;
  if ((reinterpret_cast<uintptr_t>(h) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) || !(cap >= 0.f)) return -1;
  p->T = (int)T;
  p->V = (int)V;
  p->d = d;
  p->cap = cap;
  p->inv_cap = cap > 0.f ? 1.f / cap : 0.f;
  int rc = vocab_loss_map(&p->tmA, h, d, T, ldh);
  return rc ? rc : vocab_loss_map(&p->tmB, w, d, V, ldw);
}

template <bool GRAD, bool CAP>
static int vocab_loss_launch(VocabLossParams& p, cudaStream_t st) {
  auto kern = vocab_loss_kernel<GRAD, CAP>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, VL_SMEM) != cudaSuccess) return -10;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long tiles = (long long)p.m_blks * p.n_blks;
  if (tiles > 0x7fffffffll) return -1;
  const int clusters = (int)(tiles < sms / 2 ? tiles : sms / 2);
  kern<<<2 * clusters, VL_THREADS, VL_SMEM, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

}  // namespace sx
using namespace sx;

extern "C" int sx_vocab_loss_fwd(const void* h, long long ldh, const void* w, long long ldw, const long long* target, long long T, long long V, int d,
                                 long long ignore_index, float cap, void* part, float* zt, float* nll, float* lse, int* status, cudaStream_t st) {
  VocabLossParams p = {};
  int rc = vocab_loss_setup(&p, h, ldh, w, ldw, T, V, d, cap);
  if (rc) return rc;
  p.target = target; p.ignore_index = ignore_index; p.part = (float2*)part; p.zt = zt; p.status = status;
  p.v0 = 0; p.v1 = (int)V;
  p.m_blks = (int)((T + 255) / 256); p.n_blks = (int)((V + 255) / 256);
  rc = cap > 0.f ? vocab_loss_launch<false, true>(p, st) : vocab_loss_launch<false, false>(p, st);
  if (rc) return rc;
  vocab_loss_join_kernel<<<(unsigned)((T + 31) / 32), dim3(32, 16), 0, st>>>(p.part, zt, target, nll, lse, (int)T, (int)V, 2 * p.n_blks, ignore_index, status);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

extern "C" int sx_vocab_loss_grad(const void* h, long long ldh, const void* w, long long ldw, const long long* target, long long T, long long V, int d,
                                  long long ignore_index, float cap, const float* lse, const float* g_nll, const float* g_lse, void* dz, long long ld,
                                  long long rows, long long v0, long long v1, int* status, cudaStream_t st) {
  VocabLossParams p = {};
  int rc = vocab_loss_setup(&p, h, ldh, w, ldw, T, V, d, cap);
  if (rc) return rc;
  if (v0 < 0 || v1 <= v0 || v1 > V || ld % 32 || ld < v1 - v0 || ld > (1 << 30) || rows < T || rows > T + 255 || (reinterpret_cast<uintptr_t>(dz) & 15)) return -2;
  p.target = target; p.ignore_index = ignore_index; p.status = status;
  p.lse = lse; p.g_nll = g_nll; p.g_lse = g_lse; p.dz = (__nv_bfloat16*)dz; p.ld = ld; p.rows = (int)rows;
  p.v0 = (int)v0; p.v1 = (int)v1;
  p.m_blks = (int)((rows + 255) / 256); p.n_blks = (int)((ld + 255) / 256);
  return cap > 0.f ? vocab_loss_launch<true, true>(p, st) : vocab_loss_launch<true, false>(p, st);
}
