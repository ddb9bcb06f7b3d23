// Log-probabilities of given tokens, entropy, log-sum-exp and the best alternatives of logits rows, in one pass.
//
// For a row x of V logits (y = x - c, c the running reference, the row's maximum in the end):
//   s = sum e^y,  t = sum e^y y      lse = c + log s    entropy = log s - t / s    logprob(i) = x_i - c - log s
// Two partial results (c, s, t) join by C = max(c): s' = s e^(c-C), t' = (t + s (c - C)) e^(c-C). c, s and t are
// fp32. The subtraction comes before the scaling to base 2: rows masked with the type's lowest value would overflow
// the other way round.
//
// The best K entries (value descending, ties to the lower id) come from the same pass: a warp reads 512 contiguous
// bytes per load (a segment) and keeps the segment's maximum, which the running reference needs anyway. The K-th
// best of the threads' maxima is a lower bound of the K-th best entry, so afterwards only the segments whose
// maximum reaches it are read again (they are in L2) and sorted in by (value, ~id) keys: about K segments for
// ordinary rows, all of them for a constant row.
//
// Bound: the logits' bytes at DRAM rate. Per logit the arithmetic is one exponential (16 a clock and SM, the
// nearest limit: a bf16 row at full DRAM rate asks for about 12) and six simple instructions.
// Split: one CTA of 256 threads per row, four resident per SM; fewer rows than that put a cluster of 2 to 8 CTAs
// on each row, whose partial results the first CTA joins through distributed shared memory.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include "../common.cuh"
#include <algorithm>

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int UNROLL = 4;       // segments in flight per warp
constexpr int MAX_TOP = 32;     // one entry per lane of a warp's sorted list
constexpr int MAX_CLUSTER = 8;  // the portable cluster size
constexpr float LOG2E = 1.4426950408889634f;

// max that keeps a NaN
SNB_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
SNB_DEVICE float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Unsigned keys in the order of the values: -inf lowest, -0 equal to +0, NaN above +inf; 0 is below every value.
SNB_DEVICE uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  if (v != v) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
SNB_DEVICE float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static SNB_DEVICE void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
  static SNB_DEVICE float one(float v) { return v; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static SNB_DEVICE void unpack(const uint4& u, float (&f)[8]) { snb::unpack_bf16x8(u, f); }
  static SNB_DEVICE float one(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static SNB_DEVICE void unpack(const uint4& u, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  static SNB_DEVICE float one(__half v) { return __half2float(v); }
};

struct Stats {
  float c, s, t;  // reference, sum of e^y, sum of e^y y
};

SNB_DEVICE Stats join(const Stats& a, const Stats& b) {
  if (a.c == -INFINITY) return b;  // nothing seen yet
  if (b.c == -INFINITY) return a;
  const float C = max_nan(a.c, b.c);
  const float fa = ex2((a.c - C) * LOG2E), fb = ex2((b.c - C) * LOG2E);
  Stats r;
  r.c = C;
  r.s = a.s * fa + b.s * fb;
  // the far side's weight is 0 when its distance is infinite or merely large: 0 * inf must not become NaN
  r.t = (fa > 0.f ? fa * (a.t + a.s * (a.c - C)) : 0.f) + (fb > 0.f ? fb * (b.t + b.s * (b.c - C)) : 0.f);
  if (C != C || C == INFINITY) r.s = r.t = NAN;
  return r;
}

// A row is cut into an unaligned head (fewer than one vector), `units` segments of 32 vectors, and a tail.
template <typename T>
struct RowCut {
  int head, nvec, units, tail0;
  SNB_DEVICE RowCut(const T* row, int V) {
    constexpr int N = Vec<T>::N;
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % N);
    head = min(V, mis ? N - mis : 0);
    nvec = (V - head) / N;
    units = (nvec + 31) / 32;
    tail0 = head + nvec * N;
  }
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, 4)
    logits_stats_kernel(const T* __restrict__ logits, int64_t stride, int V, const int64_t* __restrict__ ids,
                        int64_t vocab_offset, int K, float* __restrict__ logprobs, float* __restrict__ entropy,
                        float* __restrict__ lse_out, float* __restrict__ top_vals, int64_t* __restrict__ top_ids) {
  constexpr int N = Vec<T>::N;
  extern __shared__ uint32_t seg_key[];  // [units of this CTA + 1]: the segments' maxima, the ragged ends last
  __shared__ Stats warp_stats[WARPS];
  __shared__ Stats cta_stats[MAX_CLUSTER];
  __shared__ uint64_t cand[WARPS * MAX_TOP];
  __shared__ uint64_t best[MAX_CLUSTER * MAX_TOP];  // filled by every CTA of the cluster in the first one's memory
  __shared__ int cand_n, best_n[MAX_CLUSTER];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = gridDim.x, rank = blockIdx.x;  // the cluster spans the grid's x axis
  const int64_t row = blockIdx.y;
  if (TOP && threadIdx.x == 0) cand_n = 0;
  snb::pdl_wait();
  snb::pdl_trigger();
  const T* x = logits + row * stride;
  const RowCut<T> cut(x, V);
  const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
  const int u0 = (int)((int64_t)rank * cut.units / C), u1 = (int)((int64_t)(rank + 1) * cut.units / C);

  Stats st{-INFINITY, 0.f, 0.f};
  uint32_t best_key = 0;
  auto add = [&](const float* v, int n, float mx) {
    // mx: the maximum of v[0..n); -inf: nothing to add
    if (mx == -INFINITY) return;
    if (!(mx <= st.c)) {  // also when mx is NaN
      const float f = ex2((st.c - mx) * LOG2E);
      st.t = f > 0.f ? f * (st.t + st.s * (st.c - mx)) : 0.f;
      st.s *= f;
      st.c = mx;
    }
#pragma unroll
    for (int i = 0; i < n; ++i) {
      // a logit of -inf has weight 0: the floor keeps 0 * y finite
      const float y = max_nan(v[i] - st.c, -1e30f);
      const float e = ex2(y * LOG2E);
      st.s += e;
      st.t = fmaf(e, y, st.t);
    }
  };

  for (int u = u0 + warp; u < u1; u += WARPS * UNROLL) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int uj = u + j * WARPS, iv = uj * 32 + lane;
      if (uj < u1 && iv < cut.nvec) raw[j] = __ldg(body + iv);
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int uj = u + j * WARPS;
      if (uj >= u1) break;
      float v[N], mx = -INFINITY;
      const bool have = uj * 32 + lane < cut.nvec;
      if (have) {
        Vec<T>::unpack(raw[j], v);
        mx = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) mx = max_nan(mx, v[i]);
        add(v, N, mx);
      }
      if constexpr (TOP) {
        const uint32_t k = have ? order_key(mx) : 0u;
        best_key = max(best_key, k);
        const uint32_t seg = __reduce_max_sync(0xffffffffu, k);
        if (lane == 0) seg_key[uj - u0] = seg;
      }
    }
  }
  // the ragged ends (head and tail, fewer than two vectors) belong to the first CTA's first warp
  const int ends = cut.head + (V - cut.tail0);
  const bool mine = rank == 0 && warp == 0 && lane < ends;
  const int end_i = lane < cut.head ? lane : cut.tail0 + lane - cut.head;
  float end_v = -INFINITY;
  if (mine) {
    end_v = Vec<T>::one(x[end_i]);
    add(&end_v, 1, end_v);
    if (TOP) best_key = max(best_key, order_key(end_v));
  }

#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats b;
    b.c = __shfl_xor_sync(0xffffffffu, st.c, o);
    b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    b.t = __shfl_xor_sync(0xffffffffu, st.t, o);
    // both lanes of a pair join in the same order: every lane ends with the same bits
    st = (lane & o) ? join(b, st) : join(st, b);
  }
  if (lane == 0) warp_stats[warp] = st;

  if constexpr (TOP) {
    // the K-th largest of the threads' maxima, bit by bit (0 when fewer than K threads hold any entry)
    uint32_t thr = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = thr | (1u << b);
      if (__syncthreads_count(best_key >= t) >= K) thr = t;
    }
    // every warp sorts the entries >= thr of its own segments into a list held across its lanes
    uint64_t list = 0;
    auto offer = [&](uint64_t key) {
      const uint64_t kth = __shfl_sync(0xffffffffu, list, K - 1);
      unsigned hit = __ballot_sync(0xffffffffu, key > kth && (uint32_t)(key >> 32) >= thr);
      while (hit) {
        const int src = __ffs(hit) - 1;
        hit &= hit - 1;
        const uint64_t k = __shfl_sync(0xffffffffu, key, src);
        const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
        if (k > list) list = (lane > 0 && k > up) ? up : k;
      }
    };
    const int mine_n = u1 - u0 - warp > 0 ? (u1 - u0 - warp + WARPS - 1) / WARPS : 0;
#pragma unroll 1
    for (int j0 = 0; j0 < mine_n; j0 += 32) {
      const int j = j0 + lane;
      unsigned sel = __ballot_sync(0xffffffffu, j < mine_n && seg_key[warp + j * WARPS] >= thr);
      while (sel) {
        const int uj = u0 + warp + (j0 + __ffs(sel) - 1) * WARPS;
        sel &= sel - 1;
        const int iv = uj * 32 + lane;
        float v[N];
        const bool have = iv < cut.nvec;
        if (have) Vec<T>::unpack(__ldg(body + iv), v);
        const uint32_t i0 = (uint32_t)(cut.head + iv * N);
#pragma unroll
        for (int i = 0; i < N; ++i)
          offer(have ? ((uint64_t)order_key(v[i]) << 32) | (0xffffffffu - (i0 + i)) : 0ull);
      }
    }
    if (warp == 0) offer(mine ? ((uint64_t)order_key(end_v) << 32) | (0xffffffffu - (uint32_t)end_i) : 0ull);
    const bool valid = lane < K && list != 0;
    const unsigned vm = __ballot_sync(0xffffffffu, valid);
    int base = 0;
    if (lane == 0 && vm) base = atomicAdd(&cand_n, __popc(vm));
    base = __shfl_sync(0xffffffffu, base, 0);
    if (valid) cand[base + lane] = list;
  }
  __syncthreads();

  // this CTA's result, into the first CTA's shared memory
  uint32_t dst_rank = 0;
  if (warp == 0) {
    Stats a = lane < WARPS ? warp_stats[lane] : Stats{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
      Stats b;
      b.c = __shfl_xor_sync(0xffffffffu, a.c, o);
      b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
      b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
      a = (lane & o) ? join(b, a) : join(a, b);
    }
    if (lane == 0) {
      const uint32_t at = snb::mapa_shared(snb::smem_u32(&cta_stats[rank]), dst_rank);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(a.c) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(a.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(a.t) : "memory");
    }
  }
  if constexpr (TOP) {
    const int n = cand_n;
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const uint64_t k = cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += cand[j] > k;
      if (r < K) {
        const uint32_t at = snb::mapa_shared(snb::smem_u32(&best[rank * MAX_TOP + r]), dst_rank);
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(k) : "memory");
      }
    }
    if (threadIdx.x == 0) {
      const uint32_t at = snb::mapa_shared(snb::smem_u32(&best_n[rank]), dst_rank);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(min(n, K)) : "memory");
    }
  }
  if (C > 1) {
    __syncwarp();
    snb::cluster_sync();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // every thread of the first CTA joins the few partial results itself
  Stats a = cta_stats[0];
  for (int r = 1; r < C; ++r) a = join(a, cta_stats[r]);
  const bool none = a.c == -INFINITY;  // every logit is -inf
  const float lg = logf(a.s);
  const float lse = none ? -INFINITY : a.c + lg;
  if (threadIdx.x == 0) {
    const int64_t id = ids[row] - vocab_offset;
    float lp = -INFINITY;
    if (id >= 0 && id < V && !none) lp = (Vec<T>::one(x[id]) - a.c) - lg;
    logprobs[row] = lp;
    entropy[row] = none ? 0.f : lg - a.t / a.s;
    lse_out[row] = lse;
  }
  if constexpr (TOP) {
    for (int i = threadIdx.x; i < C * MAX_TOP; i += THREADS) {
      const int r = i / MAX_TOP, p = i % MAX_TOP;
      if (p >= best_n[r]) continue;
      const uint64_t k = best[i];
      int at = p;  // the lists are sorted and their keys differ: the place in the merged list is the sum of ranks
      for (int q = 0; q < C; ++q) {
        if (q == r) continue;
        for (int j = 0; j < best_n[q] && best[q * MAX_TOP + j] > k; ++j) ++at;
      }
      if (at < K) {
        top_vals[row * K + at] = none ? -INFINITY : (key_value((uint32_t)(k >> 32)) - a.c) - lg;
        top_ids[row * K + at] = vocab_offset + (int64_t)(0xffffffffu - (uint32_t)k);
      }
    }
  }
}

template <typename T>
void launch(const at::Tensor& logits, int V, const at::Tensor& ids, int64_t vocab_offset, int K,
            at::Tensor& logprobs, at::Tensor& entropy, at::Tensor& lse, at::Tensor& top_vals,
            at::Tensor& top_ids) {
  const int64_t rows = logits.size(0);
  const auto* prop = at::cuda::getCurrentDeviceProperties();
  auto st = at::cuda::getCurrentCUDAStream();
  const int units = (V / Vec<T>::N + 31) / 32;
  // CTAs per row: enough to fill four CTAs per SM, as long as each keeps a load per warp in flight
  int C = 1;
  while (C < MAX_CLUSTER && rows * C * 2 <= (int64_t)prop->multiProcessorCount * 4 && units >= C * 2 * WARPS) C *= 2;
  const size_t smem = K > 0 ? sizeof(uint32_t) * ((units + C - 1) / C + 2) : 0;
  TORCH_CHECK(smem <= 200 * 1024, "token_logprobs: vocabulary of ", V, " is too wide for top_k");
  // the grid's y axis holds 65535 rows: longer batches go in several launches
  for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
    const int n = (int)std::min<int64_t>(65535, rows - r0);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C, n);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = snb::pdl_enabled() ? 2 : 1;
    const T* x = reinterpret_cast<const T*>(logits.data_ptr()) + r0 * logits.stride(0);
    const int64_t* id = ids.data_ptr<int64_t>() + r0;
    float* tv = K > 0 ? top_vals.data_ptr<float>() + r0 * K : nullptr;
    int64_t* ti = K > 0 ? top_ids.data_ptr<int64_t>() + r0 * K : nullptr;
    auto kern = K > 0 ? logits_stats_kernel<T, true> : logits_stats_kernel<T, false>;
    if (smem > 16 * 1024)
      C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, x, logits.stride(0), V, id, vocab_offset, K,
                                      logprobs.data_ptr<float>() + r0, entropy.data_ptr<float>() + r0,
                                      lse.data_ptr<float>() + r0, tv, ti));
  }
}

}  // namespace

// logits: [N, >= V] bf16 / fp16 / fp32, any row stride; only the first V columns are read, whatever the rest holds.
// ids: [N] int64 (less vocab_offset outside [0, V): log-probability -inf). Outputs: [N] fp32, top [N, K].
void logits_stats(at::Tensor logits, int64_t V, at::Tensor ids, int64_t vocab_offset, int64_t K,
                  at::Tensor logprobs, at::Tensor entropy, at::Tensor lse, at::Tensor top_vals,
                  at::Tensor top_ids) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1),
              "token_logprobs: logits must be a CUDA matrix with contiguous rows");
  TORCH_CHECK(V > 0 && V <= logits.size(1) && V < (int64_t(1) << 30), "token_logprobs: valid_vocab ", V,
              " outside the logits' ", logits.size(1), " columns");
  TORCH_CHECK(K >= 0 && K <= MAX_TOP && K <= V, "token_logprobs: top_k ", K, " not in [0, ", MAX_TOP, "]");
  TORCH_CHECK(ids.scalar_type() == at::kLong && ids.is_contiguous() && ids.numel() == logits.size(0),
              "token_logprobs: one int64 id per row");
  if (logits.size(0) == 0) return;
  switch (logits.scalar_type()) {
    case at::kFloat:
      launch<float>(logits, (int)V, ids, vocab_offset, (int)K, logprobs, entropy, lse, top_vals, top_ids);
      break;
    case at::kBFloat16:
      launch<__nv_bfloat16>(logits, (int)V, ids, vocab_offset, (int)K, logprobs, entropy, lse, top_vals, top_ids);
      break;
    case at::kHalf:
      launch<__half>(logits, (int)V, ids, vocab_offset, (int)K, logprobs, entropy, lse, top_vals, top_ids);
      break;
    default:
      TORCH_CHECK(false, "token_logprobs: dtype ", logits.scalar_type());
  }
}
