// Log-probabilities of given tokens, entropy and log-sum-exp of an LM head's logits that are never stored:
//   z[n, v] = sum_k hidden[n, k] weight[v, k]   (bf16 / fp16 operands, fp32 in tensor memory)
//   y = z - c,  s = sum_v e^y,  t = sum_v e^y y    lse = c + log s   entropy = log s - t / s
// A product kernel writes (c, s, t) of every vocabulary tile and row, head_join_kernel joins them.
//
// More than 128 rows: head_stats_kernel, bound by the tensor cores and, from some 0.1 s of load on, by the GPU's power:
// 4096 x 4096 x 151936 took 3100 us, 1645 TFLOP/s, in six launches after a pause, and 3409 to 3481 us, 1465 to 1496
// TFLOP/s, after 0.3 s of load, where the library's product alone, in the same run, took 3473 to 3491 us; 1000 x 2880 x
// 201088 took 779 us and 884 us (883 us). Up to 128 rows: head_few_kernel, bound by the weights' stream: 16 x 4096 x
// 151936 took 219 us, 5.7 TB/s (the library's product: 211 us); at 129 rows the pair kernel takes 258 us, at 128 this one
// 243 us. A tiled weight arrives 16 (pair) or 32 (few) rows a load: 5495 us, 1321 us and, 33 x 2048 x 102400, 112 us
// against 88 us row-major.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include "../common.cuh"
#include "../tma_host.h"
#include <algorithm>
#include <tuple>

namespace {

constexpr int BM = 128;  // rows of hidden per CTA: its half of the pair's M = 256, one tensor-memory lane each
constexpr int BN = 256;  // most vocabulary entries per tile; each CTA of the pair holds half of their weights
constexpr int BK = 64;   // 16-bit elements per 128-byte swizzled row
constexpr int RING = 224 * 1024;  // operand bytes per CTA: 7 stages of the widest tiles, more of smaller ones
constexpr int MAX_STAGES = 16;
constexpr int SMEM = RING + 1024 + 512;
constexpr int A_BYTES = BM * BK * 2;
constexpr int THREADS = 192;
constexpr float LOG2E = 1.4426950408889634f;

SNB_DEVICE float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
SNB_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// One lane of a converged warp; what the branch uses stays in uniform registers, as the MMA's operands must.
SNB_DEVICE bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// ---- a pair of CTAs: one MMA over both, issued by the even one --------------------------------------------------
SNB_DEVICE void tmem_alloc_pair(uint32_t* at, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(snb::smem_u32(at)), "r"(cols));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
}
SNB_DEVICE void tmem_dealloc_pair(uint32_t t, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(cols));
}
SNB_DEVICE void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// Arrives on the barrier at this offset in both CTAs once the MMAs issued so far are done.
SNB_DEVICE void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          snb::smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Loads into this CTA's memory and counts the bytes on the even CTA's barrier (its shared::cluster address).
SNB_DEVICE void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(snb::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
SNB_DEVICE void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

struct HeadParams {
  const int64_t* ids;
  int64_t vocab_offset;
  float4* part;  // [vocabulary tiles][n_pad]: reference, sum, weighted sum, the given token's logit
  int N, V, K, n_pad, mt, units, w_tiled;
  int width;     // vocabulary entries per tile: a multiple of 32 up to BN
  int stage, stages;  // the ring: bytes of a stage, how many stages
  uint32_t idesc;
  int* status;
};

// A pair of CTAs multiplies 256 rows of hidden with 256 vocabulary entries per unit of work: every CTA loads its own
// 128 rows and its half of the weights, so an operand byte in shared memory serves twice the products of a lone CTA
// (which would need 128 bytes of shared memory and 96 of L2 a cycle, more than an SM gets). The pairs walk the units
// (vocabulary tile, row tile) with the row tile running fastest, all of them together: a weight tile is read from DRAM
// once and from L2 by the other row tiles, and hidden stays in L2. Two accumulators of 256 columns: the statistics of
// one unit are taken while the next one is multiplied.
__global__ void __launch_bounds__(THREADS)
    head_stats_kernel(const __grid_constant__ CUtensorMap tmap_h, const __grid_constant__ CUtensorMap tmap_w,
                      const __grid_constant__ HeadParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + RING);  // used in the even CTA
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* acc_full = empty + MAX_STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;   // [2], used in the even CTA
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* loads = reinterpret_cast<int*>(tmem_slot + 1);  // k blocks issued / multiplied (the latter in the even CTA)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = snb::cluster_ctarank();
  const int pairs = gridDim.x / 2, first = blockIdx.x / 2;
  const int nk = (p.K + BK - 1) / BK;
  // bytes that one stage of the ring takes from both CTAs
  const uint32_t stage_bytes = 2 * A_BYTES + p.width * BK * 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_STAGES; ++s) {
      snb::mbar_init(&full[s], 1);
      snb::mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      snb::mbar_init(&acc_full[i], 1);
      snb::mbar_init(&acc_empty[i], 8);  // four warps of each CTA
    }
    snb::mbar_init(drain, 1);
    loads[0] = loads[1] = 0;
    snb::fence_mbar_init();
    snb::prefetch_tmap(&tmap_h);
    snb::prefetch_tmap(&tmap_w);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  snb::tc_fence_before();
  __syncthreads();
  snb::cluster_sync();
  snb::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  snb::pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0, s = 0, ph = 0;
      bool ok = true;
      for (int u = first; ok && u < p.units; u += pairs) {
        const int m0 = (u % p.mt) * 2 * BM + rank * BM, vt = u / p.mt;
        const int v0 = vt * p.width + rank * (p.width / 2);
        for (int kb = 0; kb < nk; ++kb, ++it) {
          ok = snb::mbar_wait_bounded(&empty[s], ph ^ 1, p.status, SNB_ERR_TIMEOUT_TMA);
          if (!ok) break;
          uint8_t* sA = smem + s * p.stage;
          uint8_t* sB = sA + A_BYTES;
          const int k0 = kb * BK;
          // the even CTA's barrier takes the bytes of both
          if (rank == 0) snb::mbar_arrive_expect_tx(&full[s], stage_bytes);
          const uint32_t bar = snb::mapa_shared(snb::smem_u32(&full[s]), 0);
          tma_load_pair(sA, &tmap_h, bar, k0, m0);
          if (p.w_tiled) {  // 128 x 64 blocks, each contiguous: 16 rows never straddle two of them
            for (int v = v0; v < v0 + p.width / 2; v += 16)
              tma_load_pair(sB + (v - v0) * BK * 2, &tmap_w, bar, 0, (v / 128 * nk + k0 / BK) * 128 + v % 128);
          } else {
            tma_load_pair(sB, &tmap_w, bar, k0, v0);
          }
          if (++s == p.stages) s = 0, ph ^= 1;
        }
      }
      loads[0] = it;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint64_t ring = snb::smem_desc_sw128(snb::smem_u32(smem));
      int it = 0, n = 0, s = 0, ph = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, int parity) {
        const bool r = snb::mbar_wait_bounded(bar, parity, p.status, SNB_ERR_TIMEOUT_MMA);
        snb::tc_fence_after();
        return __all_sync(0xffffffffu, r) != 0;
      };
      for (int u = first; ok && u < p.units; u += pairs, ++n) {
        ok = wait(&acc_empty[n & 1], ((n >> 1) & 1) ^ 1);
        for (int kb = 0; ok && kb < nk; ++kb, ++it) {
          ok = wait(&full[s], ph);
          if (!ok) break;
          const uint64_t a = ring + s * (p.stage >> 4), b = a + (A_BYTES >> 4);  // descriptors count 16 bytes
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              mma_pair(tmem + (n & 1) * BN, a + k * 2, b + k * 2, p.idesc, (kb | k) != 0 ? 1u : 0u);
            commit_pair(&empty[s]);
          }
          if (++s == p.stages) s = 0, ph ^= 1;
        }
        if (ok && elect_one()) commit_pair(&acc_full[n & 1]);
      }
      if (lane == 0) loads[1] = it;
      if (!ok) {
        if (elect_one()) commit_pair(drain);
        snb::mbar_wait_bounded(drain, 0, p.status, SNB_ERR_TIMEOUT_MMA);
      }
    }
  } else {
    const int q = warp & 3;
    int n = 0;
    for (int u = first; u < p.units; u += pairs, ++n) {
      const int vt = u / p.mt, v0 = vt * p.width;
      const int row = (u % p.mt) * 2 * BM + rank * BM + q * 32 + lane;
      const int64_t id = row < p.N ? p.ids[row] - p.vocab_offset - v0 : -1;
      const bool r_ok = snb::mbar_wait_bounded(&acc_full[n & 1], (n >> 1) & 1, p.status, SNB_ERR_TIMEOUT_EPI);
      if (!__all_sync(0xffffffffu, r_ok)) break;
      snb::tc_fence_after();
      float c = -INFINITY, s = 0.f, t = 0.f, chosen = -INFINITY;
#pragma unroll 1
      for (int j = 0; j < p.width / 32; ++j) {
        __syncwarp();  // the rows part below; the tensor-memory load wants the whole warp
        uint32_t r[32];
        snb::tmem_ld_32x32b_x32(tmem + ((uint32_t)(q * 32) << 16) + (n & 1) * BN + j * 32, r);
        snb::tmem_ld_wait();
        const int left = p.V - v0 - j * 32;
        if (left < 32) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i >= left) r[i] = 0xff800000u;  // columns past the vocabulary
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; ++i) mx = max_nan(mx, __uint_as_float(r[i]));
        if (id >= j * 32 && id < j * 32 + 32) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (id == j * 32 + i) chosen = __uint_as_float(r[i]);
        }
        if (mx != -INFINITY) {
          if (!(mx <= c)) {
            const float f = ex2((c - mx) * LOG2E);
            t = f > 0.f ? f * (t + s * (c - mx)) : 0.f;
            s *= f;
            c = mx;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float y = max_nan(__uint_as_float(r[i]) - c, -1e30f);
            const float e = ex2(y * LOG2E);
            s += e;
            t = fmaf(e, y, t);
          }
        }
      }
      snb::tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(snb::mapa_shared(snb::smem_u32(&acc_empty[n & 1]), 0));
      if (row < p.N) p.part[(size_t)vt * p.n_pad + row] = make_float4(c, s, t, chosen);
    }
  }
  snb::tc_fence_before();
  __syncthreads();
  if (warp == 0 && lane == 0 && rank == 0) {
    // loads of a pair that stopped early still arrive (bounded) before the memory goes away
    for (int i = loads[1]; i < loads[0]; ++i)
      if (!snb::mbar_wait_bounded(&full[i % p.stages], (i / p.stages) & 1, p.status, SNB_ERR_TIMEOUT_TMA)) break;
  }
  __syncthreads();
  snb::cluster_sync();  // neither CTA leaves while the other can still reach its memory
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---- few rows: the weight's stream ------------------------------------------------------------------------------
// With at most 128 rows the weights are the MMA's 128-row operand and the rows its columns: a pair's 256 rows would be
// mostly padding, whose products cost power (the clock fell to 1.5 GHz) and more time than the weights take to arrive.
// Every CTA takes an equal run of the vocabulary in groups of 32, four groups a unit. A warp's 32 lanes hold 32
// vocabulary entries, so each token's statistics are sums over lanes: columns and lanes change places while they are
// summed (31 shuffles for 32 sums).
constexpr int FEW = 128;
constexpr int GROUP = 32;  // vocabulary entries per partial result

struct FewParams {
  const int64_t* ids;
  int64_t vocab_offset;
  float4* part;   // [vocabulary groups][N]: reference, sum, weighted sum
  float* chosen;  // [N] the given token's logit
  int N, V, K, cols, groups, w_tiled;  // cols: N rounded up to what an MMA takes
  int stage, stages;
  uint32_t idesc;
  int* status;
};

// v[i] of all lanes summed over the lanes: lane l gets the sum of v[l]
SNB_DEVICE float sum_columns(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = (lane & o) ? v[i] : v[i + o], keep = (lane & o) ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}
SNB_DEVICE float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

__global__ void __launch_bounds__(THREADS)
    head_few_kernel(const __grid_constant__ CUtensorMap tmap_h, const __grid_constant__ CUtensorMap tmap_w,
                    const __grid_constant__ CUtensorMap tmap_w32, const __grid_constant__ FewParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + RING);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* acc_full = empty + MAX_STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* loads = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nk = (p.K + BK - 1) / BK;
  const int g0 = (int)((int64_t)blockIdx.x * p.groups / gridDim.x);
  const int g1 = (int)((int64_t)(blockIdx.x + 1) * p.groups / gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_STAGES; ++s) {
      snb::mbar_init(&full[s], 1);
      snb::mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      snb::mbar_init(&acc_full[i], 1);
      snb::mbar_init(&acc_empty[i], 4);
    }
    snb::mbar_init(drain, 1);
    loads[0] = loads[1] = 0;
    snb::fence_mbar_init();
    snb::prefetch_tmap(&tmap_h);
    snb::prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    snb::tmem_alloc(tmem_slot, 2 * FEW);
    snb::tmem_relinquish();
  }
  snb::tc_fence_before();
  __syncthreads();
  snb::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  snb::pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      // Every CTA starts at another place of the contraction: the rows of hidden are few lines, which all of them
      // would ask for at the same time.
      const int turn = (int)((int64_t)blockIdx.x * nk / gridDim.x);
      int it = 0, s = 0, ph = 0;
      bool ok = true;
      for (int g = g0; ok && g < g1; g += 4) {
        const int n = min(4, g1 - g);
        for (int kb = 0; kb < nk; ++kb, ++it) {
          ok = snb::mbar_wait_bounded(&empty[s], ph ^ 1, p.status, SNB_ERR_TIMEOUT_TMA);
          if (!ok) break;
          uint8_t* sW = smem + s * p.stage;
          const int k = kb + turn < nk ? kb + turn : kb + turn - nk;
          snb::mbar_arrive_expect_tx(&full[s], (n * GROUP + p.cols) * BK * 2);
          if (n == 4 && !p.w_tiled) {
            snb::tma_load_2d(sW, &tmap_w, &full[s], k * BK, g * GROUP);
          } else {
            for (int i = 0; i < n; ++i) {
              const int v = (g + i) * GROUP;
              snb::tma_load_2d(sW + i * GROUP * BK * 2, &tmap_w32, &full[s], p.w_tiled ? 0 : k * BK,
                               p.w_tiled ? (v / 128 * nk + k) * 128 + v % 128 : v);
            }
          }
          snb::tma_load_2d(sW + A_BYTES, &tmap_h, &full[s], k * BK, 0);
          if (++s == p.stages) s = 0, ph ^= 1;
        }
      }
      loads[0] = it;
    }
  } else if (warp == 1) {
    const uint64_t ring = snb::smem_desc_sw128(snb::smem_u32(smem));
    int it = 0, n = 0, s = 0, ph = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, int parity) {
      const bool r = snb::mbar_wait_bounded(bar, parity, p.status, SNB_ERR_TIMEOUT_MMA);
      snb::tc_fence_after();
      return __all_sync(0xffffffffu, r) != 0;
    };
    for (int g = g0; ok && g < g1; g += 4, ++n) {
      ok = wait(&acc_empty[n & 1], ((n >> 1) & 1) ^ 1);
      for (int kb = 0; ok && kb < nk; ++kb, ++it) {
        ok = wait(&full[s], ph);
        if (!ok) break;
        const uint64_t a = ring + s * (p.stage >> 4), b = a + (A_BYTES >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            snb::mma_bf16_ss(tmem + (n & 1) * FEW, a + k * 2, b + k * 2, p.idesc, (kb | k) != 0 ? 1u : 0u);
          snb::mma_commit(&empty[s]);
        }
        if (++s == p.stages) s = 0, ph ^= 1;
      }
      if (ok && elect_one()) snb::mma_commit(&acc_full[n & 1]);
    }
    if (lane == 0) loads[1] = it;
    if (!ok) {
      if (elect_one()) snb::mma_commit(drain);
      snb::mbar_wait_bounded(drain, 0, p.status, SNB_ERR_TIMEOUT_MMA);
    }
  } else {
    const int q = warp & 3;
    int n = 0;
    for (int g = g0; g < g1; g += 4, ++n) {
      const bool r_ok = snb::mbar_wait_bounded(&acc_full[n & 1], (n >> 1) & 1, p.status, SNB_ERR_TIMEOUT_EPI);
      if (!__all_sync(0xffffffffu, r_ok)) break;
      snb::tc_fence_after();
      const int v = (g + q) * GROUP + lane;  // this lane's vocabulary entry
#pragma unroll 1
      for (int j = 0; j < p.cols; j += 32) {
        __syncwarp();
        uint32_t r[32];
        snb::tmem_ld_32x32b_x32(tmem + ((uint32_t)(q * 32) << 16) + (n & 1) * FEW + j, r);
        snb::tmem_ld_wait();
        if (g + q >= g1) continue;  // the run's last unit can have fewer than four groups
        const int tok = j + lane;
        const int64_t id = tok < p.N ? p.ids[tok] - p.vocab_offset - (int64_t)(g + q) * GROUP : -1;
        const int at = id >= 0 && id < GROUP ? (int)id : -1;
        float e[32], t[32], c = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float z = v < p.V ? __uint_as_float(r[i]) : -INFINITY;
          if (__shfl_sync(0xffffffffu, at, i) == lane) p.chosen[j + i] = z;
          const float m = warp_max_nan(z);
          if (lane == i) c = m;
          const float y = max_nan(z - (m == -INFINITY ? 0.f : m), -1e30f);
          e[i] = ex2(y * LOG2E);
          t[i] = e[i] * y;
        }
        const float se = sum_columns(e), st = sum_columns(t);
        if (tok < p.N) p.part[(size_t)(g + q) * p.N + tok] = make_float4(c, se, st, 0.f);
      }
      snb::tc_fence_before();
      __syncwarp();
      if (lane == 0) snb::mbar_arrive(&acc_empty[n & 1]);
    }
  }
  snb::tc_fence_before();
  __syncthreads();
  if (warp == 0 && lane == 0) {
    for (int i = loads[1]; i < loads[0]; ++i)
      if (!snb::mbar_wait_bounded(&full[i % p.stages], (i / p.stages) & 1, p.status, SNB_ERR_TIMEOUT_TMA)) break;
  }
  if (warp == 1) snb::tmem_dealloc(tmem, 2 * FEW);
}

// Joins a row's partial results. ROWS rows per CTA of 256 threads: 8 where the rows are many (their partial results
// lie side by side), 1 where a row has many partial results and there are few rows. Whole calls with 1 / 8 rows per
// CTA, 512 x 151936: 16 rows 42.1 / 72.2 us, 128 62.1 / 97.1, 256 50.1 / 50.6, 512 85.7 / 85.5, 1024 155 / 152, 4096
// 545 / 530; 512 x 32768: 512 24.8 / 23.8, 2048 72.6 / 65.9.
// Tried and slower: CTAs so small that they wait beside the product's for its end (33 x 2048 x 102400: 90.7 us against
// 85.1).
template <int ROWS>
__global__ void __launch_bounds__(256)
    head_join_kernel(const float4* __restrict__ part, const float* __restrict__ chosen, int pitch, int N, int V,
                     int tiles, int width, const int64_t* __restrict__ ids, int64_t vocab_offset,
                     float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ lse_out) {
  constexpr int EACH = 256 / ROWS;  // threads per row
  snb::pdl_wait();
  const int r = threadIdx.x % ROWS, g = threadIdx.x / ROWS;
  const int n = blockIdx.x * ROWS + r;
  __shared__ float sx[EACH][ROWS + 1], sy[EACH][ROWS + 1];
  // the maximum first, then the sums against it: loads in a row that do not wait for one another
  float c = -INFINITY;
  if (n < N) {
#pragma unroll 4
    for (int i = g; i < tiles; i += EACH) c = max_nan(c, part[(size_t)i * pitch + n].x);
  }
  sx[g][r] = c;
  __syncthreads();
  for (int o = EACH / 2; o > 0; o >>= 1) {
    if (g < o) sx[g][r] = max_nan(sx[g][r], sx[g + o][r]);
    __syncthreads();
  }
  c = sx[0][r];
  __syncthreads();
  float s = 0.f, t = 0.f;
  if (n < N && c != -INFINITY) {
#pragma unroll 4
    for (int i = g; i < tiles; i += EACH) {
      const float4 p = part[(size_t)i * pitch + n];
      const float d = max_nan(p.x - c, -1e30f);  // a tile of -inf has weight 0
      const float f = ex2(d * LOG2E);
      s = fmaf(p.y, f, s);
      t = fmaf(fmaf(p.y, d, p.z), f, t);
    }
  }
  sx[g][r] = s;
  sy[g][r] = t;
  __syncthreads();
  for (int o = EACH / 2; o > 0; o >>= 1) {
    if (g < o) {
      sx[g][r] += sx[g + o][r];
      sy[g][r] += sy[g + o][r];
    }
    __syncthreads();
  }
  if (g != 0 || n >= N) return;
  s = sx[0][r];
  t = sy[0][r];
  const bool none = c == -INFINITY;
  const float lg = logf(s);
  const float lse = none ? -INFINITY : c + lg;
  const int64_t id = ids[n] - vocab_offset;
  float lp = -INFINITY;
  if (id >= 0 && id < V && !none)
    lp = ((chosen != nullptr ? chosen[n] : part[(size_t)(id / width) * pitch + n].w) - c) - lg;
  logprobs[n] = lp;
  entropy[n] = none ? 0.f : lg - t / s;
  lse_out[n] = lse;
}

void join_parts(const at::Tensor& part, const float* chosen, int pitch, int N, int V, int tiles, int width,
                const int64_t* ids, int64_t vocab_offset, at::Tensor& stats, cudaStream_t st) {
  float* out = stats.data_ptr<float>();
  const bool one = N <= 512;
  C10_CUDA_CHECK(snb::launch_pdl(one ? head_join_kernel<1> : head_join_kernel<8>, dim3(one ? N : (N + 7) / 8),
                                 dim3(256), 0, st, reinterpret_cast<const float4*>(part.data_ptr<float>()), chosen,
                                 pitch, N, V, tiles, width, ids, vocab_offset, out, out + N, out + 2 * N));
}

cudaLaunchConfig_t pair_config(cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// Pairs of CTAs that run at the same time (one CTA per SM, both SMs of a pair in one cluster), per device
int resident_pairs(int device) {
  static int known[64] = {0};
  int& n = known[device & 63];
  if (n == 0) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(head_stats_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = pair_config(attr);
    cfg.gridDim = dim3(2 * (at::cuda::getCurrentDeviceProperties()->multiProcessorCount / 2));
    int most = 0;
    C10_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&most, head_stats_kernel, &cfg));
    TORCH_CHECK(most > 0, "head_logprobs: no pair of CTAs fits this GPU");
    n = most;
  }
  return n;
}

// Vocabulary entries per tile. The pairs finish a round of units together, so a tile's width should make the last
// round a full one; a narrow tile on the other hand reads hidden more often (the 32 entries added to its cost). With
// hidden rows of 2880, in us for the 32 entries / none added / always 256 wide: 300 x 32768 71 / 70 / 75, 300 x 151936
// 333 / 366 / 326, 1000 x 102400 449 / 475 / 439, 1000 x 151936 658 / 697 / 675, 3000 x 151936 1878 / 2430 / 1874.
int pick_width(int mt, int64_t V, int pairs) {
  int best = BN;
  int64_t least = INT64_MAX;
  for (int w = BN; w >= 128; w -= 32) {
    const int64_t units = (V + w - 1) / w * mt, cost = (units + pairs - 1) / pairs * (w + 32);
    if (cost < least) least = cost, best = w;
  }
  return best;
}

}  // namespace

// hidden [N, K], weight [F, K] (or its 128 x 64 tiles, `tiled`, with F given), both bf16 or both fp16, K a multiple of
// 8; the first V entries (V = 0: all) are the vocabulary. ids [N] int64 or int32. Returns fp32 [N] log-probability,
// entropy and log-sum-exp.
std::tuple<at::Tensor, at::Tensor, at::Tensor> head_stats(at::Tensor hidden, at::Tensor weight, int64_t F, bool tiled,
                                                          int64_t V, at::Tensor ids, int64_t vocab_offset,
                                                          at::Tensor status) {
  TORCH_CHECK(hidden.is_cuda() && hidden.dim() == 2 && weight.dim() == 2 &&
                  (tiled || hidden.size(1) == weight.size(1)),
              "head_logprobs: hidden [rows, size] does not fit the weight [vocabulary, size]");
  const int64_t N = hidden.size(0), K = hidden.size(1);
  if (!tiled) F = weight.size(0);
  if (V == 0) V = F;
  const auto type = hidden.scalar_type();
  TORCH_CHECK(type == weight.scalar_type() && weight.device() == hidden.device(),
              "head_logprobs: hidden and the weight differ in type or device");
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf, "head_logprobs: takes bf16 or fp16 on CUDA");
  TORCH_CHECK(K > 0 && K % 8 == 0, "head_logprobs: needs a hidden size that is a multiple of 8");
  TORCH_CHECK(V > 0 && V <= F && V < (int64_t(1) << 30), "head_logprobs: valid_vocab is outside the weight's rows");
  TORCH_CHECK(ids.dim() == 1 && ids.numel() == N && ids.device() == hidden.device() &&
                  (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
              "head_logprobs: ids must be one int64 or int32 per row on the rows' device");
  TORCH_CHECK(N < (int64_t(1) << 30), "head_logprobs: too many rows");
  const c10::cuda::CUDAGuard guard(hidden.device());
  auto stats = at::empty({3, N}, hidden.options().dtype(at::kFloat));
  const auto result = std::make_tuple(stats.select(0, 0), stats.select(0, 1), stats.select(0, 2));
  if (N == 0) return result;
  hidden = snb_host::mappable(hidden);
  weight = snb_host::mappable(weight);
  ids = ids.to(at::kLong).contiguous();
  const bool bf16 = hidden.scalar_type() == at::kBFloat16;
  const auto dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto st = at::cuda::getCurrentCUDAStream();
  if (N <= FEW) {
    const int cols = (int)((N + 15) / 16 * 16), groups = (int)((V + GROUP - 1) / GROUP);
    const CUtensorMap th = snb_host::make_tmap_2d(hidden.data_ptr(), dt, K, N, hidden.stride(0) * 2, BK, cols,
                                                  CU_TENSOR_MAP_SWIZZLE_128B);
    // a whole unit's 128 rows in one load (a load costs its thread some 180 cycles), a run's ragged end by groups
    auto weights = [&](int rows) {
      return tiled ? snb_host::make_tmap_2d(weight.data_ptr(), dt, BK, weight.size(0), BK * 2, BK, rows,
                                            CU_TENSOR_MAP_SWIZZLE_128B)
                   : snb_host::make_tmap_2d(weight.data_ptr(), dt, K, V, weight.stride(0) * 2, BK, rows,
                                            CU_TENSOR_MAP_SWIZZLE_128B);
    };
    const CUtensorMap tw = weights(4 * GROUP), tw32 = weights(GROUP);
    auto part = at::empty({((int64_t)groups * 4 + 1) * N}, hidden.options().dtype(at::kFloat));
    FewParams p;
    p.ids = ids.data_ptr<int64_t>();
    p.vocab_offset = vocab_offset;
    p.part = reinterpret_cast<float4*>(part.data_ptr<float>());
    p.chosen = part.data_ptr<float>() + (int64_t)groups * 4 * N;
    p.N = (int)N;
    p.V = (int)V;
    p.K = (int)K;
    p.cols = cols;
    p.groups = groups;
    p.w_tiled = tiled ? 1 : 0;
    p.stage = A_BYTES + (cols * BK * 2 + 1023) / 1024 * 1024;
    p.stages = std::min(MAX_STAGES, RING / p.stage);
    p.idesc = snb::idesc_bf16_f32(BM, cols) & ~(bf16 ? 0u : (1u << 7) | (1u << 10));
    p.status = status.data_ptr<int>();
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    C10_CUDA_CHECK(cudaFuncSetAttribute(head_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    C10_CUDA_CHECK(snb::launch_pdl(head_few_kernel, dim3(std::min(groups, sms)), dim3(THREADS), SMEM, st, th, tw, tw32, p));
    join_parts(part, p.chosen, (int)N, (int)N, (int)V, groups, GROUP, p.ids, vocab_offset, stats, st);
    return result;
  }
  const CUtensorMap th = snb_host::make_tmap_2d(hidden.data_ptr(), dt, K, N, hidden.stride(0) * 2, BK, BM,
                                                CU_TENSOR_MAP_SWIZZLE_128B);
  const int mt = (int)((N + 2 * BM - 1) / (2 * BM)), n_pad = mt * 2 * BM;
  const int pairs = resident_pairs(hidden.device().index());
  const int width = pick_width(mt, V, pairs), vt = (int)((V + width - 1) / width);
  const CUtensorMap tw =
      tiled ? snb_host::make_tmap_2d(weight.data_ptr(), dt, BK, weight.size(0), BK * 2, BK, 16,
                                     CU_TENSOR_MAP_SWIZZLE_128B)
            : snb_host::make_tmap_2d(weight.data_ptr(), dt, K, V, weight.stride(0) * 2, BK, width / 2,
                                     CU_TENSOR_MAP_SWIZZLE_128B);
  TORCH_CHECK((int64_t)mt * vt < (int64_t(1) << 31), "head_logprobs: too much work for one call");
  auto part = at::empty({(int64_t)vt * n_pad * 4}, hidden.options().dtype(at::kFloat));
  HeadParams p;
  p.ids = ids.data_ptr<int64_t>();
  p.vocab_offset = vocab_offset;
  p.part = reinterpret_cast<float4*>(part.data_ptr<float>());
  p.N = (int)N;
  p.V = (int)V;
  p.K = (int)K;
  p.n_pad = n_pad;
  p.mt = mt;
  p.units = mt * vt;
  p.w_tiled = tiled ? 1 : 0;
  p.width = width;
  p.stage = A_BYTES + width / 2 * BK * 2;
  p.stages = std::min(MAX_STAGES, RING / p.stage);
  p.idesc = snb::idesc_bf16_f32(2 * BM, width) & ~(bf16 ? 0u : (1u << 7) | (1u << 10));
  p.status = status.data_ptr<int>();
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pair_config(attr);
  cfg.gridDim = dim3(2 * std::min(p.units, pairs));
  cfg.stream = st;
  cfg.numAttrs = snb::pdl_enabled() ? 2 : 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, head_stats_kernel, th, tw, p));
  join_parts(part, nullptr, n_pad, (int)N, (int)V, vt, width, p.ids, vocab_offset, stats, st);
  return result;
}
