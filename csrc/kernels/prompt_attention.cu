// Causal attention of packed whole prompts (no cache): every prompt's queries over its own keys and values.
//
//   out[t, h] = sum_j p_j v[j, h / G],   p_j = exp(scale q[t, h] . k[j, h / G] - m) / (exp(sink[h] - m) + sum_j ...)
//   over the tokens j <= t of the same prompt, t - j < window where a window is set.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include "../common.cuh"
#include "../tma_host.h"
#include <algorithm>

namespace {

constexpr float LOG2E = 1.4426950408889634f;

SNB_DEVICE float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T>
SNB_DEVICE float2 unpack2(uint32_t u);
template <>
SNB_DEVICE float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
SNB_DEVICE float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <typename T>
SNB_DEVICE uint32_t pack2(float lo, float hi);
template <>
SNB_DEVICE uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
SNB_DEVICE uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct PromptParams {
  const void *q, *k, *v;
  void* out;
  int64_t qs, ks, vs, os;  // row strides, in elements
  const int* indptr;
  const float* sinks;
  int T, B, heads, kv_heads, window;
  float scale;  // of the scores, in log2 units
};

SNB_DEVICE int seq_bound(const PromptParams& p, int b) { return min(max(__ldg(p.indptr + b), 0), p.T); }

// One output row by one warp, from global memory: exact about what is masked (a masked key or value is never
// touched).
template <typename T, int D, int DV>
__device__ __noinline__ void attend_row(const PromptParams& p, int first, int t, int h) {
  const int lane = threadIdx.x & 31;
  const int hk = h / (p.heads / p.kv_heads);
  const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)t * p.qs + (int64_t)h * D;
  const T* k = reinterpret_cast<const T*>(p.k) + (int64_t)hk * D;
  const T* v = reinterpret_cast<const T*>(p.v) + (int64_t)hk * DV;
  const int lo = p.window > 0 ? max(first, t - p.window + 1) : first;
  auto score = [&](int j) {
    float a = 0.f;
    const T* kr = k + (int64_t)j * p.ks;
#pragma unroll 4
    for (int d = 0; d < D; d += 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(q + d), y = *reinterpret_cast<const uint4*>(kr + d);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(xs[i]), g = unpack2<T>(ys[i]);
        a = fmaf(f.x, g.x, a);
        a = fmaf(f.y, g.y, a);
      }
    }
    return a * p.scale;
  };
  float m = -INFINITY;
  bool nan = false;
  for (int j = lo + lane; j <= t; j += 32) {
    const float s = score(j);
    nan |= s != s;
    m = fmaxf(m, s);
  }
  m = snb::warp_max(m);
  if (p.sinks != nullptr) m = fmaxf(m, p.sinks[h] * LOG2E);
  nan = __any_sync(0xffffffffu, nan);
  if (m == -INFINITY) m = 0.f;
  float l = 0.f, o[DV / 32];
#pragma unroll
  for (int i = 0; i < DV / 32; ++i) o[i] = 0.f;
  for (int j0 = lo; j0 <= t; j0 += 32) {
    const int j = j0 + lane;
    const float w = j <= t ? ex2(score(j) - m) : 0.f;
    l += w;
    const int n = min(32, t - j0 + 1);
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const T* vr = v + (int64_t)(j0 + i) * p.vs + lane * (DV / 32);
#pragma unroll
      for (int d = 0; d < DV / 32; d += 2) {
        const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(vr + d));
        o[d] = fmaf(wi, f.x, o[d]);
        o[d + 1] = fmaf(wi, f.y, o[d + 1]);
      }
    }
  }
  l = snb::warp_sum(l);
  if (p.sinks != nullptr) l += ex2(p.sinks[h] * LOG2E - m);
  const float r = nan ? NAN : l > 0.f ? 1.f / l : 0.f;
  T* dst = reinterpret_cast<T*>(p.out) + (int64_t)t * p.os + (int64_t)h * DV + lane * (DV / 32);
#pragma unroll
  for (int d = 0; d < DV / 32; d += 2) *reinterpret_cast<uint32_t*>(dst + d) = pack2<T>(o[d] * r, o[d + 1] * r);
}

template <typename T, int D, int DV>
__global__ void __launch_bounds__(128) prompt_attention_rows_kernel(const PromptParams p) {
  snb::pdl_wait();
  snb::pdl_trigger();
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(w / p.heads), h = (int)(w % p.heads);
  if (t >= p.T) return;
  int lo = 0, hi = p.B;  // the last b with bound(b) <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (seq_bound(p, mid) <= t) lo = mid;
    else hi = mid;
  }
  const int first = seq_bound(p, lo);
  if (t < first || t >= seq_bound(p, lo + 1)) return;
  attend_row<T, D, DV>(p, first, t, h);
}

template <typename T, int D, int DV>
void launch(const PromptParams& p, cudaStream_t st) {
  const int64_t warps = (int64_t)p.T * p.heads;
  C10_CUDA_CHECK(snb::launch_pdl(prompt_attention_rows_kernel<T, D, DV>, dim3((unsigned)((warps + 3) / 4)), dim3(128),
                                 0, st, p));
}

template <typename T>
void dispatch(const PromptParams& p, int64_t D, int64_t DV, cudaStream_t st) {
  if (D == 64 && DV == 64) launch<T, 64, 64>(p, st);
  else if (D == 128 && DV == 128) launch<T, 128, 128>(p, st);
  else if (D == 192 && DV == 128) launch<T, 192, 128>(p, st);
  else TORCH_CHECK(false, "prompt_attention: head dims ", D, " / ", DV, " (64 / 64, 128 / 128 or 192 / 128)");
}

void check_rows(const at::Tensor& x, int64_t T, int64_t width, at::ScalarType dt, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(0) == T && x.size(1) == width && x.scalar_type() == dt,
              "prompt_attention: ", name, " must be a CUDA matrix of ", T, " x ", width, " and the queries' type");
  TORCH_CHECK(x.stride(1) == 1 && x.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "prompt_attention: ", name, " needs contiguous rows on 16-byte boundaries");
}

}  // namespace

// q [T, heads * D], k [T, kv_heads * D], v [T, kv_heads * DV], out [T, heads * DV]: bf16 or fp16, any row stride
// that is a multiple of 8. indptr [B + 1] int32, ascending; rows outside every prompt are not written.
void prompt_attention(at::Tensor out, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor indptr,
                      int64_t heads, int64_t kv_heads, int64_t D, int64_t DV, int64_t window, double sm_scale,
                      std::optional<at::Tensor> sinks, at::Tensor status) {
  const int64_t T = q.size(0), B = indptr.numel() - 1;
  TORCH_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "prompt_attention: ", heads, " heads over ",
              kv_heads, " KV heads");
  const auto dt = q.scalar_type();
  check_rows(q, T, heads * D, dt, "q");
  check_rows(k, T, kv_heads * D, dt, "k");
  check_rows(v, T, kv_heads * DV, dt, "v");
  check_rows(out, T, heads * DV, dt, "out");
  TORCH_CHECK(indptr.is_cuda() && indptr.scalar_type() == at::kInt && indptr.is_contiguous() && B >= 0,
              "prompt_attention: indptr must be a CUDA int32 vector");
  TORCH_CHECK(T < (int64_t(1) << 30), "prompt_attention: too many tokens");
  if (sinks)
    TORCH_CHECK(sinks->is_cuda() && sinks->scalar_type() == at::kFloat && sinks->is_contiguous() &&
                    sinks->numel() == heads,
                "prompt_attention: sinks must be one fp32 value per head");
  if (T == 0 || B == 0) return;
  PromptParams p;
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.out = out.data_ptr();
  p.qs = q.stride(0);
  p.ks = k.stride(0);
  p.vs = v.stride(0);
  p.os = out.stride(0);
  p.indptr = indptr.data_ptr<int>();
  p.sinks = sinks ? sinks->data_ptr<float>() : nullptr;
  p.T = (int)T;
  p.B = (int)B;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.window = (int)std::min<int64_t>(std::max<int64_t>(window, 0), T);
  p.scale = (float)(sm_scale * 1.4426950408889634);
  auto st = at::cuda::getCurrentCUDAStream();
  if (dt == at::kBFloat16) dispatch<__nv_bfloat16>(p, D, DV, st);
  else if (dt == at::kHalf) dispatch<__half>(p, D, DV, st);
  else TORCH_CHECK(false, "prompt_attention: dtype ", dt);
}
