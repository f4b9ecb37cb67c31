// L4: per-token losses of a vocabulary projection, in tiles of the vocabulary, without the logits ever being held.
//
//   z = h w^T, soft-capped: c tanh(z / c);   lse = log sum_v e^{z_v};   nll = lse - z_target
//   dz_v = ((g_nll + g_lse) e^{z_v - lse} - g_nll [v = target]) (1 - (z_v / c)^2),
//   and of the target, without a difference of near-equal numbers, (g_nll (e^{-nll} - 1) + g_lse e^{-nll}) (1 - (z / c)^2)
//
// One kernel, two epilogues, on the CTA-pair GEMM (256 x 256 tiles, accumulators double-buffered in TMEM, operands by TMA):
//   forward  each row's maximum and sum of exponentials over a tile's columns but the target leave the SM as one pair of numbers, the target's logit by
//            itself; a second kernel joins the pairs of a row. 8 bytes leave for 256 logits.
//   backward the tile is computed again and leaves as dz in bf16 (half a step, 2^-9, of each value: the products that follow take no other type at this
//            rate, and the logits of linear_cross_entropy's gradient are held so too; dh and dw are off by 2.4e-3 with it, 1.7e-3 by their own rounding
//            alone; up to 2.7e-3 where tokens are few and one value, the target's, makes most of a row), for one piece of the vocabulary at a time; the products dh += dz w and dw = dz^T h run on the GEMM kernel.
// Sixteen epilogue warps (four TMEM quadrants, four groups of 64 columns): the exponentials of a tile are behind the products from widths of 256 on only
// if four warps of each scheduler take turns.
// The tensor cores cut what they add to an accumulator: over 4096 products a logit of 14 loses 1e-4. The forward pass, whose losses are differences of
// logits, therefore takes the accumulator out after 768 products at most, in equal parts, and adds in registers, rounded: lse of 4088 tokens over [128256,
// 4096] is off by 1.4e-6 without that, by 3.7e-7 in parts of 1024 and by 2.3e-7 in these, in the same time; parts of 512 cost 3% more there and 20% over 768
// columns. Widths just above one part pay little for their second: 4095 tokens over [50280, 1024] 276 us in two, 275 in one, with the soft cap 299 and 281,
// at half the error (lse 2.3e-7 and 4.5e-7). Up to 256 tokens, one row of tiles, wait for the weights more than for their epilogue and take parts of 384: half
// the error (nll of 4 tokens over [16377, 640] with a soft cap 6.1e-7 -> 3.1e-7, of 64 over [128256, 4096] 6.1e-7 -> 3.1e-7) in 18.6 us as before and 203
// instead of 200.
// Backward leaves a logit in one accumulator: an error of 1e-4 in it is one of 1e-4 of its e^{z - lse}, a twentieth of what the rounding of dz to bf16 takes.
// The target's value alone would lose it against 1 - e^{z - lse}, which may be smaller, so that is computed from the forward pass's nll (64 tokens over
// [32000, 4096]: dw of a target that the model gives an nll of 1e-3 is off by 1.9e-3 of itself, 6.8e-2 by the difference; of 2.5e-5 by 2.5e-3, 0.46 by the
// difference).
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
constexpr int VL_GROUPS = 4;                         // epilogue warps of a TMEM quadrant
constexpr int VL_COLS = 256 / VL_GROUPS;             // columns of an epilogue warp
constexpr int VL_EPI_WARPS = 4 * VL_GROUPS;
constexpr int VL_THREADS = 64 + 32 * VL_EPI_WARPS;
constexpr int VL_CHUNK = 768 / VL_BK;                // forward: k-blocks that stay in one accumulator at most
constexpr int VL_FEW_CHUNK = 384 / VL_BK;            // and of up to 256 tokens
constexpr int VL_SLOTS = 4;                          // tiles whose pairs may wait to be joined (below)
constexpr int VL_OFF_PAIRS = VL_STAGES * VL_STAGE_BYTES;
constexpr int VL_PAIR_BYTES = VL_SLOTS * (VL_GROUPS - 1) * 128 * 8;
constexpr int VL_OFF_BAR = VL_OFF_PAIRS + VL_PAIR_BYTES;
constexpr int VL_SMEM = VL_OFF_BAR + 1024 + 512;
constexpr float LOG2E = 1.4426950408889634f;
// Up to this magnitude of a row's maximum (or lse) exponentials of differences are 2^(z log2 e - top log2 e) by one multiply-add, off by the rounding of top
// log2 e, 2^-13 of its exponent at most; beyond, the difference is taken first, or finite logits of 1e7 and more would overflow.
constexpr float VL_NEAR = 2048.f;

struct VocabLossParams {
  CUtensorMap tmA, tmB;       // h [T, d], w [V, d]
  const long long* target;
  long long ignore_index;
  float2* part;               // forward: [n_blks, T] maximum and sum
  float* zt;                  // forward: [T] the target's logit, in the place of which the joining kernel leaves nll
  const float* lse;           // backward
  const float* nll;           // backward: of tokens that have a target
  const float* g_nll;         // backward: [T] or null
  const float* g_lse;
  __nv_bfloat16* dz;          // backward: [rows, ld]
  long long ld;
  int* status;
  int T, V, rows, d, v0, v1;  // columns [v0, v1) of the vocabulary
  int m_blks, n_blks;
  float cap, inv_cap;         // 0: none
};

// cap * tanh(z / cap) of a row's values. Up to |z / cap| = 0.6 (logits of 18 under a cap of 30) a polynomial: tanh u / u in u^2, minimax in the relative
// error (2.5e-9, 1e-7 as evaluated). One exponential and one reciprocal less for each value, where the unit that computes them bounds the epilogue (4095 x
// 50280 logits of width 768: backward's tiles 563 -> 291 us with this and whole-sector stores). Which form is taken is each row's own matter, so that a
// token's loss does not depend on its neighbours.
// Two values an instruction, where the soft cap makes arithmetic what the epilogue waits for (4095 x 50280 of width 768: forward 226 -> 212 us, backward's
// tiles 256 -> 250).
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
template <int N>
__device__ __forceinline__ void softcap_row(float (&v)[N], float cap, float inv) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(v[j]));
  if (top * inv <= 0.6f) {
    auto both = [](float x) { return two(x, x); };
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const uint64_t x = two(v[j], v[j + 1]), u = mul2(x, both(inv)), s = mul2(u, u);
      uint64_t t = fma2(s, both(-0.005852168625497215f), both(0.020753628859718726f));
      t = fma2(s, t, both(-0.053768704695067476f));
      t = fma2(s, t, both(0.13331688960047147f));
      t = fma2(s, t, both(-0.33333283257370855f));
      apart(mul2(x, fma2(s, t, both(1.f))), v[j], v[j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = softcap(v[j], cap, inv);
  }
}
// Infinite maxima are not subtracted: a logit of infinity makes the sum infinite, as the definition has it, and not a NaN.
__device__ __forceinline__ float2 join_pairs(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x), at = isinf(top) ? 0.f : top;
  return make_float2(top, a.y * exp2f((a.x - at) * LOG2E) + b.y * exp2f((b.x - at) * LOG2E));      // the larger one's factor is 1, whatever it is
}
__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
               "r"(r[6]), "r"(r[7])
               : "memory");
}

template <bool GRAD, bool CAP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(VL_THREADS, 1) vocab_loss_kernel(const __grid_constant__ VocabLossParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + VL_OFF_BAR);                   // even CTA: both CTAs' loads complete on it
  uint64_t* empty_bar = full_bar + VL_STAGES;
  uint64_t* tfull_bar = empty_bar + VL_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;                                                  // even CTA: the epilogue warps of both
  uint64_t* pairs_bar = tempty_bar + 2;                                                  // [VL_SLOTS][4 quadrants]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pairs_bar + 4 * VL_SLOTS);
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
    for (int i = 0; i < 4 * VL_SLOTS; ++i) mbar_init(&pairs_bar[i], VL_GROUPS - 1);
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
  const int most = p.m_blks == 1 ? VL_FEW_CHUNK : VL_CHUNK;
  const int parts = (num_kb + most - 1) / most;
  const int chunk = GRAD ? num_kb : (num_kb + parts - 1) / parts;      // equal ones: what is cut grows with the longest

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
      int it = 0;               // accumulators handed over
      bool ok = true;
      for (int t = cluster_id; t < total_tiles && ok; t += n_clusters) {
        for (int k0 = 0; k0 < num_kb && ok; k0 += chunk, ++it) {
          const int acc = it & 1, k1 = min(num_kb, k0 + chunk);
          if (!mbar_wait(&tempty_bar[acc], ((it >> 1) & 1) ^ 1, s_abort, p.status, ST_TIMEOUT_MMA)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * 256;
          for (int kb = k0; kb < k1; ++kb) {
            if (!mbar_wait(&full_bar[stage], phase, s_abort, p.status, ST_TIMEOUT_MMA)) { ok = false; break; }
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + stage * VL_STAGE_BYTES), sb = sa + VL_A_BYTES;
#pragma unroll
            for (int k = 0; k < VL_BK / 16; ++k)
              umma2_f16_ss(d_tmem, umma_desc_sw128(sa + k * 32, 16, 1024), umma_desc_sw128(sb + k * 32, 16, 1024), idesc, (kb != k0 || k != 0) ? 1u : 0u);
            umma2_commit_pair(&empty_bar[stage]);
            if (++stage == VL_STAGES) { stage = 0; phase ^= 1; }
          }
          if (ok) umma2_commit_pair(&tfull_bar[acc]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue: a row a lane, 64 columns a warp
    const int q = warp & 3, group = (warp - 2) >> 2;
    const uint32_t tmem_mine = tmem_base + group * VL_COLS + (static_cast<uint32_t>(q * 32) << 16);
    float2* pairs = reinterpret_cast<float2*>(smem + VL_OFF_PAIRS);
    int it = 0, tile = 0;
    bool ok = true;
    for (int t = cluster_id; t < total_tiles && ok; t += n_clusters, ++tile) {
      int b, m_blk, n_blk;
      tile_coords(t, p.m_blks, p.n_blks, b, m_blk, n_blk);
      const int row = m_blk * 256 + (int)rank * 128 + q * 32 + lane;
      const int first = p.v0 + n_blk * 256 + group * VL_COLS;     // this warp's first column
      const int left = p.v1 - first;                              // columns that the vocabulary has from there on
      // the target as a column of this warp's, or none
      int tgt = -1;
      float a = 0.f, gn = 0.f, off = 0.f, at_target = 0.f;
      if (row < p.T) {
        const long long tv = p.target[row];
        if (tv != p.ignore_index && tv >= first && tv < first + VL_COLS && tv < p.v1) tgt = (int)(tv - first);
        if (GRAD) {
          const float gz = p.g_lse ? p.g_lse[row] : 0.f;
          if (p.g_nll && tv != p.ignore_index && tv >= 0 && tv < p.V) gn = p.g_nll[row];
          a = gn + gz;
          off = -p.lse[row] * LOG2E;
          if (tgt >= 0) {
            const float nll = p.nll[row];
            at_target = fmaf(gn, expm1f(-nll), gz * __expf(-nll));
          }
        }
      }
      if (!GRAD) {
        float v[VL_COLS];
        for (int k0 = 0; k0 < num_kb; k0 += chunk, ++it) {
          const int acc = it & 1;
          ok = mbar_wait_warp(&tfull_bar[acc], (it >> 1) & 1, s_abort, p.status, ST_TIMEOUT_EPILOGUE);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < VL_COLS / 8; ++c) {            // eight at a time: with sixteen the values that stay leave the registers
            uint32_t r[8];
            tmem_ld8(tmem_mine + acc * 256 + c * 8, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c * 8 + j] = k0 == 0 ? __uint_as_float(r[j]) : v[c * 8 + j] + __uint_as_float(r[j]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_even_cta(&tempty_bar[acc]);
        }
        if (!ok) break;
        if (CAP) softcap_row(v, p.cap, p.inv_cap);
        if (left < VL_COLS) {
#pragma unroll
          for (int j = 0; j < VL_COLS; ++j)
            if (j >= left) v[j] = -INFINITY;
        }
        if (__any_sync(0xffffffffu, tgt >= 0)) {
          float zt = 0.f;
#pragma unroll
          for (int j = 0; j < VL_COLS; ++j) {
            if (tgt == j) {
              zt = v[j];
              v[j] = -INFINITY;          // the pairs are of the other words
            }
          }
          if (tgt >= 0) p.zt[row] = zt;
        }
        float top = fmaxf(v[0], v[1]);
#pragma unroll
        for (int j = 2; j < VL_COLS; j += 2) top = fmax3(top, v[j], v[j + 1]);
        float at = top * LOG2E, off = fmaf(top, LOG2E, -at);         // top log2 e was rounded, by `off`: the exponentials are 2^off too large
        if (fabsf(top) > VL_NEAR) {                                  // rare: too far out for that
          const float from = isinf(top) ? 0.f : top;
#pragma unroll
          for (int j = 0; j < VL_COLS; ++j) v[j] -= from;
          at = off = 0.f;
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < VL_COLS; j += 2) {
          sum[j & 3] += exp2f(fmaf(v[j], LOG2E, -at));
          sum[(j & 3) + 1] += exp2f(fmaf(v[j + 1], LOG2E, -at));
        }
        const float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        float2 pair = make_float2(top, off == 0.f ? total : fmaf(total, off * -0.6931471805599453f, total));
        // The first warp of a quadrant joins the four. The others may be two tiles ahead of it at most: an accumulator is filled again when all
        // sixteen have read it. Four slots, each with a barrier that they arrive on, are enough.
        const int slot = tile % VL_SLOTS;
        float2* mine = pairs + slot * (VL_GROUPS - 1) * 128 + q * 32 + lane;
        if (group > 0) {
          mine[(group - 1) * 128] = pair;
          __syncwarp();
          if (lane == 0) mbar_arrive(&pairs_bar[slot * 4 + q]);
        } else {
          ok = mbar_wait_warp(&pairs_bar[slot * 4 + q], (tile / VL_SLOTS) & 1, s_abort, p.status, ST_TIMEOUT_EPILOGUE);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < VL_GROUPS - 1; ++i) pair = join_pairs(pair, mine[i * 128]);
          if (row < p.T) p.part[(long long)n_blk * p.T + row] = pair;
        }
      } else {
        const int acc = it & 1;
        ok = mbar_wait_warp(&tfull_bar[acc], (it >> 1) & 1, s_abort, p.status, ST_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        ++it;
#pragma unroll
        for (int c = 0; c < VL_COLS / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(tmem_mine + acc * 256 + c * 32, r);
          tmem_ld_wait();
          if (c == VL_COLS / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_even_cta(&tempty_bar[acc]);
          }
          if (first - p.v0 + c * 32 >= p.ld) continue;             // uniform across the warp
          float v[32], g[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (CAP) softcap_row(v, p.cap, p.inv_cap);
          if (CAP) {                                               // the slope, before v may be moved
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const uint64_t u = mul2(two(v[j], v[j + 1]), two(p.inv_cap, p.inv_cap)), w = mul2(u, two(-1.f, -1.f));
              apart(fma2(w, u, two(1.f, 1.f)), g[j], g[j + 1]);
            }
          }
          const bool hot = __any_sync(0xffffffffu, (tgt >> 5) == c);
          float own = at_target;
          if (CAP && hot) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (tgt == c * 32 + j) own *= g[j];
          }
          float at = off;
          if (fabsf(off) > VL_NEAR * LOG2E) {
            const float lse = p.lse[row];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] -= lse;
            at = 0.f;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float x, y;
            apart(fma2(two(v[j], v[j + 1]), two(LOG2E, LOG2E), two(at, at)), x, y);
            const uint64_t e = mul2(two(a, a), two(exp2f(x), exp2f(y)));
            apart(CAP ? mul2(two(g[j], g[j + 1]), e) : e, g[j], g[j + 1]);
          }
          if (hot) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (tgt == c * 32 + j) g[j] = own;
          }
          if (left < (c + 1) * 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c * 32 + j >= left) g[j] = 0.f;
          }
          if (row < p.rows) {
            __nv_bfloat16* o = p.dz + (long long)row * p.ld + (first - p.v0 + c * 32);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) w[j] = pack_bf16x2(g[h * 16 + 2 * j], g[h * 16 + 2 * j + 1]);
              st_global_32(o + h * 16, w);
            }
          }
        }
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

// Joins the pairs of eight rows a block, 64 threads a row. With d the logarithm of the other words' sum over the target's exponential, nll = log(1 + e^d),
// which is right to a few 2^-20 of itself also where the model is sure and nll small; lse - z would be right to as much of z. In 64 bits: one a row.
__global__ void __launch_bounds__(512) vocab_loss_join_kernel(const float2* __restrict__ part, float* __restrict__ zt,
                                                              const long long* __restrict__ target, float* __restrict__ nll, float* __restrict__ lse, int T,
                                                              int V, int parts, long long ignore_index, int* status) {
  __shared__ float2 s[64][8];
  const int row = blockIdx.x * 8 + threadIdx.x;
  float2 pair = make_float2(-INFINITY, 0.f);
  if (row < T) {
#pragma unroll 4
    for (int i = threadIdx.y; i < parts; i += 64) pair = join_pairs(pair, part[(long long)i * T + row]);
  }
  s[threadIdx.y][threadIdx.x] = pair;
  for (int n = 32; n > 0; n >>= 1) {
    __syncthreads();
    if (threadIdx.y < n) s[threadIdx.y][threadIdx.x] = pair = join_pairs(pair, s[threadIdx.y + n][threadIdx.x]);
  }
  if (threadIdx.y != 0 || row >= T) return;
  const double others = (double)pair.x + log((double)pair.y);          // -infinity where there are none
  const long long t = target[row];
  const bool valid = t != ignore_index && t >= 0 && t < V;
  if (t != ignore_index && !valid && status) atomicCAS(status, 0, (int)ST_BAD_ARGUMENT);
  if (valid) {
    const double z = zt[row], d = others - z, more = log1p(exp(d <= 0 ? d : -d));
    const bool over = z == INFINITY;           // lse and z infinite: no difference
    nll[row] = zt[row] = over ? NAN : (float)(d <= 0 ? more : d + more);
    lse[row] = over && others == others ? INFINITY : (float)((d <= 0 ? z : others) + more);
  } else {
    nll[row] = 0.f;
    lse[row] = (float)others;
  }
}

// dh of several sums over parts of the vocabulary (parts [n, count] fp32): their sum, rounded once. Eight values a thread; count is a multiple of 8.
__global__ void __launch_bounds__(256) vocab_loss_sum_kernel(const float4* __restrict__ parts, uint4* __restrict__ out, int n, long long count8) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= count8) return;
  float4 a = parts[2 * i], b = parts[2 * i + 1];
  for (int k = 1; k < n; ++k) {
    const float4 c = parts[2 * (k * count8 + i)], e = parts[2 * (k * count8 + i) + 1];
    a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
    b.x += e.x; b.y += e.y; b.z += e.z; b.w += e.w;
  }
  out[i] = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
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
  static int known[64];      // multiprocessors of the devices that the kernel has been set up on
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -10;
  int sms = __atomic_load_n(&known[dev], __ATOMIC_ACQUIRE);
  if (sms == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, VL_SMEM) != cudaSuccess) return -10;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 2) return -10;
    __atomic_store_n(&known[dev], sms, __ATOMIC_RELEASE);
  }
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
  if (!h || !w || !target || !part || !zt || !nll || !lse) return -1;
  VocabLossParams p = {};
  int rc = vocab_loss_setup(&p, h, ldh, w, ldw, T, V, d, cap);
  if (rc) return rc;
  p.target = target; p.ignore_index = ignore_index; p.part = (float2*)part; p.zt = zt; p.status = status;
  p.v0 = 0; p.v1 = (int)V;
  p.m_blks = (int)((T + 255) / 256); p.n_blks = (int)((V + 255) / 256);
  rc = cap > 0.f ? vocab_loss_launch<false, true>(p, st) : vocab_loss_launch<false, false>(p, st);
  if (rc) return rc;
  vocab_loss_join_kernel<<<(unsigned)((T + 7) / 8), dim3(8, 64), 0, st>>>(p.part, zt, target, nll, lse, (int)T, (int)V, p.n_blks, ignore_index, status);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

namespace sx {

// What backward does with its scratch and in which order, from the arguments alone.
struct VocabLossPlan {
  long long piece, ld;        // words of a piece, pitch of dz
  int splits;                 // parts of a piece whose sums of dh are apart
  bool sums;                  // dh goes through 32-bit sums in scratch
  long long o_dz, o_acc, bytes;
};
constexpr long long PIECE_BYTES = 256ll << 20;       // of dz, where the caller does not say how wide a piece is
// dh has T d results only, and for few tokens or narrow models these are too few tiles for the machine: the product is then split over the words into sums of
// their own (4095 tokens of 768: 48 tiles on 74 pairs of SMs; 3 x 48 fill two rounds, and 50280 words take 225 us instead of 321; 64 tokens of 4096: 16
// tiles on 148 SMs, 128256 words 152 us in nine parts, 693 in one). The split that takes least: the product at 1.4 PFLOP/s where every place has a
// tile, and the sums written, and read for each further piece and once more at the end, at 6 TB/s.
static int dh_splits(long long T, int d, long long words, long long pieces) {
  const int places = T < 256 ? 148 : 74;             // the GEMM takes pairs of SMs from 256 rows on
  const long long tiles = (T < 256 ? (T + 127) / 128 : (T + 255) / 256) * ((d + 255) / 256);
  const long long rows = T < 256 ? (T + 127) / 128 * 128 : (T + 255) / 256 * 256;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 16 && (s == 1 || words / s >= 1024); ++s) {
    const double use = (double)(tiles * s) / (double)(places * ((tiles * s + places - 1) / places));
    const double sums = s > 1 || pieces > 1 ? 4.0 * s * (double)T * d * (2 * pieces) : 0;
    const double cost = 2.0 * (double)rows * d * (double)(words * pieces) / use / 1.4e15 + sums / 6e12;
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}
static long long k_part(long long words, int splits) { return ((words + splits - 1) / splits + 63) / 64 * 64; }   // at most `splits` parts
static VocabLossPlan vocab_loss_plan(const SxVocabLossArgs* a) {
  VocabLossPlan p;
  long long piece = a->piece > 0 ? a->piece : PIECE_BYTES / (2 * a->T);
  if (a->piece <= 0 && piece < 1024) piece = 1024;
  piece = (piece + 255) / 256 * 256;
  if (piece > a->V) piece = a->V;
  p.splits = 1;
  if (a->dh) {
    const int s = dh_splits(a->T, a->d, piece, (a->V + piece - 1) / piece);
    p.splits = (int)((piece + k_part(piece, s) - 1) / k_part(piece, s));
  }
  p.piece = piece;
  p.ld = (piece + 63) / 64 * 64;
  p.sums = a->dh && (p.splits > 1 || piece < a->V);
  long long o = 0;
  auto take = [&](long long bytes) {
    const long long at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  p.o_dz = take(2 * a->T * p.ld);
  p.o_acc = take(p.sums ? 4ll * p.splits * a->T * a->d : 0);
  p.bytes = o;
  return p;
}
static bool vocab_loss_args_ok(const SxVocabLossArgs* a) {
  return a->T > 0 && a->T <= (1 << 30) && a->V > 0 && a->V <= (1 << 30) && a->d > 0 && a->d % 8 == 0 && a->piece >= 0;
}

}  // namespace sx

extern "C" long long sx_vocab_loss_bwd_workspace(const SxVocabLossArgs* a) { return vocab_loss_args_ok(a) ? vocab_loss_plan(a).bytes : -1; }

extern "C" int sx_vocab_loss_bwd(const SxVocabLossArgs* a, cudaStream_t st) {
  if (!vocab_loss_args_ok(a) || !a->h || !a->w || !a->target || !a->lse || !a->nll || !a->work) return -1;
  const VocabLossPlan plan = vocab_loss_plan(a);
  if (a->work_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(a->work) & 255)) return -3;
  VocabLossParams p = {};
  int rc = vocab_loss_setup(&p, a->h, a->ldh, a->w, a->ldw, a->T, a->V, a->d, a->cap);
  if (rc) return rc;
  uint8_t* work = (uint8_t*)a->work;
  __nv_bfloat16* dz = (__nv_bfloat16*)(work + plan.o_dz);
  float* acc = (float*)(work + plan.o_acc);
  p.target = a->target; p.ignore_index = a->ignore_index; p.status = a->status;
  p.lse = a->lse; p.nll = a->nll; p.g_nll = a->g_nll; p.g_lse = a->g_lse; p.dz = dz; p.rows = (int)a->T;
  p.m_blks = (int)((a->T + 255) / 256);
  for (long long v0 = 0; v0 < a->V; v0 += plan.piece) {
    const long long v1 = v0 + plan.piece < a->V ? v0 + plan.piece : a->V, n = v1 - v0;
    const bool first = v0 == 0, last = v1 == a->V;
    p.v0 = (int)v0; p.v1 = (int)v1; p.ld = (n + 63) / 64 * 64;
    p.n_blks = (int)((p.ld + 255) / 256);
    rc = a->cap > 0.f ? vocab_loss_launch<true, true>(p, st) : vocab_loss_launch<true, false>(p, st);
    if (rc) return rc;
    const __nv_bfloat16* w = (const __nv_bfloat16*)a->w + v0 * a->ldw;
    SxGemmArgs g = {};
    g.alpha = 1.f; g.status = a->status; g.batch = 1; g.flags = 2; g.b_mn = 1;
    g.A = dz; g.lda = p.ld;
    if (a->dh) {
      const int s = plan.splits;
      g.B = w; g.ldb = a->ldw;
      g.M = (int)a->T; g.N = a->d; g.K = (int)n;
      if (s > 1) {                    // a last piece may have fewer parts
        g.k_step = (int)k_part(n, s);
        g.batch = (int)((n + g.k_step - 1) / g.k_step);
        g.strideD = a->T * a->d;
      }
      g.ldd = a->d;
      const bool out = !plan.sums || (s == 1 && last);
      g.D = out ? a->dh : (void*)acc;
      g.out_fp32 = !out;
      if (!first) {
        g.C = acc; g.ldc = a->d; g.strideC = g.strideD; g.c_fp32 = 1; g.beta = 1.f;
      }
      if ((rc = sx_gemm_bf16(&g, st))) return rc;
    }
    if (a->dw) {
      g.a_mn = 1; g.B = a->h; g.ldb = a->ldh; g.batch = 1; g.k_step = 0; g.strideC = g.strideD = 0;
      g.M = (int)n; g.N = a->d; g.K = (int)a->T;
      g.D = (char*)a->dw + v0 * a->lddw * (a->dw_fp32 ? 4 : 2);
      g.ldd = a->lddw; g.out_fp32 = a->dw_fp32;
      g.C = a->dw_add ? g.D : nullptr; g.ldc = a->lddw; g.c_fp32 = a->dw_fp32; g.beta = a->dw_add ? 1.f : 0.f;
      if ((rc = sx_gemm_bf16(&g, st))) return rc;
    }
  }
  if (a->dh && plan.splits > 1) {
    const long long count8 = a->T * a->d / 8;
    vocab_loss_sum_kernel<<<(unsigned)((count8 + 255) / 256), 256, 0, st>>>((const float4*)acc, (uint4*)a->dh, plan.splits, count8);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
