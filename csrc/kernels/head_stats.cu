// Log-probabilities of given tokens, entropy and log-sum-exp of an LM head's logits that are never stored:
//   z[n, v] = sum_k hidden[n, k] weight[v, k]   (bf16 / fp16 operands, fp32 in tensor memory)
//   y = z - c,  s = sum_v e^y,  t = sum_v e^y y    lse = c + log s   entropy = log s - t / s
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include "../common.cuh"
#include "../tma_host.h"
#include <algorithm>

namespace {

constexpr int BM = 128;  // rows of hidden per tile: the MMA's M, one tensor-memory lane each
constexpr int BN = 256;  // vocabulary entries per tile
constexpr int BK = 64;   // 16-bit elements per 128-byte swizzled row
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int STAGES = 4;
constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 256;
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

// Partial result of one (vocabulary tile, row): reference, sum, weighted sum, and the given token's logit.
__global__ void __launch_bounds__(192)
    head_stats_kernel(const __grid_constant__ CUtensorMap tmap_h, const __grid_constant__ CUtensorMap tmap_w, int N,
                      int V, int K, uint32_t idesc, const int64_t* __restrict__ ids, int64_t vocab_offset,
                      float4* __restrict__ part, int n_pad, int w_tiled, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + STAGES * B_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* accum = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);
  int* loads = reinterpret_cast<int*>(tmem_slot + 1);  // [0] issued, [1] consumed
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.x * BM, v0 = blockIdx.y * BN;
  const int nk = (K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      snb::mbar_init(&full[s], 1);
      snb::mbar_init(&empty[s], 1);
    }
    snb::mbar_init(accum, 1);
    loads[0] = loads[1] = 0;
    snb::fence_mbar_init();
  }
  if (warp == 1) {
    snb::tmem_alloc(tmem_slot, BN);
    snb::tmem_relinquish();
  }
  snb::tc_fence_before();
  __syncthreads();
  snb::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  snb::pdl_trigger();
  snb::pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int kb = 0;
      for (; kb < nk; ++kb) {
        const int s = kb % STAGES;
        if (!snb::mbar_wait_bounded(&empty[s], ((kb / STAGES) & 1) ^ 1, status, SNB_ERR_TIMEOUT_TMA)) break;
        snb::mbar_arrive_expect_tx(&full[s], STAGE_BYTES);
        snb::tma_load_2d(sA + s * A_BYTES, &tmap_h, &full[s], kb * BK, m0);
        for (int h = 0; h < 2; ++h)
          snb::tma_load_2d(sB + s * B_BYTES + h * (B_BYTES / 2), &tmap_w, &full[s], w_tiled ? 0 : kb * BK,
                           w_tiled ? ((v0 / 128 + h) * nk + kb) * 128 : v0 + h * 128);
      }
      loads[0] = kb;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      int kb = 0;
      for (; kb < nk; ++kb) {
        const int s = kb % STAGES;
        if (!snb::mbar_wait_bounded(&full[s], (kb / STAGES) & 1, status, SNB_ERR_TIMEOUT_MMA)) {
          ok = false;
          break;
        }
        snb::tc_fence_after();
        const uint32_t a = snb::smem_u32(sA + s * A_BYTES), b = snb::smem_u32(sB + s * B_BYTES);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          snb::mma_bf16_ss(tmem, snb::smem_desc_sw128(a + k * 32), snb::smem_desc_sw128(b + k * 32), idesc,
                           (kb | k) != 0 ? 1u : 0u);
        snb::mma_commit(&empty[s]);
      }
      loads[1] = kb;
      snb::mma_commit(accum);
      if (!ok) snb::mbar_wait_bounded(accum, 0, status, SNB_ERR_TIMEOUT_MMA);
    }
  } else {
    const int q = warp & 3, n = m0 + q * 32 + lane;
    const bool ok = snb::mbar_wait_bounded(accum, 0, status, SNB_ERR_TIMEOUT_EPI);
    snb::tc_fence_after();
    const int64_t id = n < N ? ids[n] - vocab_offset - v0 : -1;
    float c = -INFINITY, s = 0.f, t = 0.f, chosen = -INFINITY;
    if (ok) {
#pragma unroll 1
      for (int j = 0; j < BN / 32; ++j) {
        uint32_t r[32];
        snb::tmem_ld_32x32b_x32(tmem + ((uint32_t)(q * 32) << 16) + j * 32, r);
        snb::tmem_ld_wait();
        const int left = V - v0 - j * 32;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (i >= left) r[i] = 0xff800000u;  // columns past the vocabulary
          mx = max_nan(mx, __uint_as_float(r[i]));
          if (id == j * 32 + i) chosen = __uint_as_float(r[i]);
        }
        if (mx == -INFINITY) continue;
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
    if (n < N) part[(size_t)blockIdx.y * n_pad + n] = make_float4(c, s, t, chosen);
  }
  snb::tc_fence_before();
  __syncthreads();
  if (warp == 0 && lane == 0) {
    for (int i = loads[1]; i < loads[0]; ++i)
      if (!snb::mbar_wait_bounded(&full[i % STAGES], (i / STAGES) & 1, status, SNB_ERR_TIMEOUT_TMA)) break;
  }
  if (warp == 1) snb::tmem_dealloc(tmem, BN);
}

constexpr int JOIN_ROWS = 8, JOIN_GROUPS = 32;

// Joins a row's partial results: 8 rows per CTA, 32 threads of each walk the vocabulary tiles.
__global__ void __launch_bounds__(JOIN_ROWS* JOIN_GROUPS)
    head_join_kernel(const float4* __restrict__ part, int n_pad, int N, int V, int tiles,
                     const int64_t* __restrict__ ids, int64_t vocab_offset, float* __restrict__ logprobs,
                     float* __restrict__ entropy, float* __restrict__ lse_out) {
  snb::pdl_wait();
  snb::pdl_trigger();
  const int r = threadIdx.x % JOIN_ROWS, g = threadIdx.x / JOIN_ROWS;
  const int n = blockIdx.x * JOIN_ROWS + r;
  __shared__ float sc[JOIN_GROUPS][JOIN_ROWS + 1], ss[JOIN_GROUPS][JOIN_ROWS + 1], st[JOIN_GROUPS][JOIN_ROWS + 1];
  float c = -INFINITY, s = 0.f, t = 0.f;
  auto join = [&](float c2, float s2, float t2) {
    if (c2 == -INFINITY) return;
    if (c == -INFINITY) {
      c = c2, s = s2, t = t2;
      return;
    }
    const float C = max_nan(c, c2), f = ex2((c - C) * LOG2E), f2 = ex2((c2 - C) * LOG2E);
    t = (f > 0.f ? f * (t + s * (c - C)) : 0.f) + (f2 > 0.f ? f2 * (t2 + s2 * (c2 - C)) : 0.f);
    s = s * f + s2 * f2;
    c = C;
    if (!(C < INFINITY)) s = t = NAN;
  };
  if (n < N) {
#pragma unroll 4
    for (int i = g; i < tiles; i += JOIN_GROUPS) {
      const float4 p = part[(size_t)i * n_pad + n];
      join(p.x, p.y, p.z);
    }
  }
  sc[g][r] = c;
  ss[g][r] = s;
  st[g][r] = t;
  __syncthreads();
  if (g != 0 || n >= N) return;
  for (int i = 1; i < JOIN_GROUPS; ++i) join(sc[i][r], ss[i][r], st[i][r]);
  const bool none = c == -INFINITY;
  const float lg = logf(s);
  const float lse = none ? -INFINITY : c + lg;
  const int64_t id = ids[n] - vocab_offset;
  float lp = -INFINITY;
  if (id >= 0 && id < V && !none) lp = (part[(size_t)(id / BN) * n_pad + n].w - c) - lg;
  logprobs[n] = lp;
  entropy[n] = none ? 0.f : lg - t / s;
  lse_out[n] = lse;
}

}  // namespace

// hidden [N, K], weight [>= V, K] (or 128 x 64 tiles, `tiled`), both bf16 or both fp16; ids [N] int64; outputs [N].
void head_stats(at::Tensor hidden, at::Tensor weight, int64_t V, bool tiled, at::Tensor ids,
                int64_t vocab_offset, at::Tensor logprobs, at::Tensor entropy, at::Tensor lse,
                at::Tensor status) {
  const int64_t N = hidden.size(0), K = hidden.size(1);
  TORCH_CHECK(hidden.is_cuda() && hidden.stride(1) == 1 && weight.stride(1) == 1, "head_logprobs: row-major operands");
  TORCH_CHECK(hidden.scalar_type() == weight.scalar_type() &&
                  (hidden.scalar_type() == at::kBFloat16 || hidden.scalar_type() == at::kHalf),
              "head_logprobs: bf16 or fp16 operands of one type");
  TORCH_CHECK(ids.scalar_type() == at::kLong && ids.is_contiguous() && ids.numel() == N,
              "head_logprobs: one int64 id per row");
  TORCH_CHECK(K > 0 && V > 0 && V < (int64_t(1) << 30) && N < (int64_t(1) << 30), "head_logprobs: sizes");
  if (N == 0) return;
  const bool bf16 = hidden.scalar_type() == at::kBFloat16;
  const auto dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUtensorMap th = snb_host::make_tmap_2d(hidden.data_ptr(), dt, K, N, hidden.stride(0) * 2, BK, BM,
                                                CU_TENSOR_MAP_SWIZZLE_128B);
  const CUtensorMap tw =
      tiled ? snb_host::make_tmap_2d(weight.data_ptr(), dt, BK, weight.size(0), BK * 2, BK, 128,
                                     CU_TENSOR_MAP_SWIZZLE_128B)
            : snb_host::make_tmap_2d(weight.data_ptr(), dt, K, V, weight.stride(0) * 2, BK, 128,
                                     CU_TENSOR_MAP_SWIZZLE_128B);
  const int mt = (int)((N + BM - 1) / BM), vt = (int)((V + BN - 1) / BN);
  TORCH_CHECK(vt <= 65535, "head_logprobs: vocabulary too wide");
  const int n_pad = mt * BM;
  auto part = at::empty({(int64_t)vt * n_pad * 4}, hidden.options().dtype(at::kFloat));
  auto st = at::cuda::getCurrentCUDAStream();
  const uint32_t idesc = snb::idesc_bf16_f32(BM, BN) & ~(bf16 ? 0u : (1u << 7) | (1u << 10));
  C10_CUDA_CHECK(cudaFuncSetAttribute(head_stats_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
  C10_CUDA_CHECK(snb::launch_pdl(head_stats_kernel, dim3(mt, vt), dim3(192), SMEM, st, th, tw, (int)N, (int)V,
                                 (int)K, idesc, ids.data_ptr<int64_t>(), vocab_offset,
                                 reinterpret_cast<float4*>(part.data_ptr<float>()), n_pad, tiled ? 1 : 0,
                                 status.data_ptr<int>()));
  C10_CUDA_CHECK(snb::launch_pdl(head_join_kernel, dim3((N + JOIN_ROWS - 1) / JOIN_ROWS),
                                 dim3(JOIN_ROWS * JOIN_GROUPS), 0, st,
                                 reinterpret_cast<const float4*>(part.data_ptr<float>()), n_pad, (int)N, (int)V, vt,
                                 ids.data_ptr<int64_t>(), vocab_offset, logprobs.data_ptr<float>(),
                                 entropy.data_ptr<float>(), lse.data_ptr<float>()));
}
