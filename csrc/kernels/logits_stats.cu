// Log-probabilities of given tokens, entropy, log-sum-exp and the best alternatives of logits rows, in one pass.
//
// For a row x of V logits (y = x - c, c the running reference, the row's maximum in the end):
//   s = sum e^y,  t = sum e^y y      lse = c + log s    entropy = log s - t / s    logprob(i) = x_i - c - log s
// Two partial results (c, s, t) join by C = max(c): s' = s e^(c-C), t' = (t + s (c - C)) e^(c-C). c, s and t are
// fp32. The subtraction comes before the scaling to base 2: rows masked with the type's lowest value would overflow
// the other way round.
//
// The best K entries (value descending, ties to the lower id) come from the same pass: a warp reads 512 contiguous
// bytes per load and keeps the maximum of every two loads (a segment), which the running reference needs anyway. The K-th
// best of 32 groups' maxima is a lower bound of the K-th best entry, so afterwards only the segments whose
// maximum reaches it are read again (they are in L2) and sorted in by (value, ~id) keys: about K segments for
// ordinary rows, all of them for a constant row. The CTAs of a cluster exchange the groups' maxima, so that a row has
// these K segments once, not once per CTA (64 x 201088 fp32 with twenty: 26.3 us without the exchange, 20.5 with it).
//
// Bound: the logits' bytes at DRAM rate. A bf16 row at that rate brings 12 logits a clock and SM, so a logit has one
// exponential (of 16 a clock) and few issue slots: two values go through each fp32 instruction (f32x2), y is taken in
// units of log 2 by one multiply-add, maximum and floor act on the 16-bit pairs as loaded. The reference is rounded
// before it is subtracted, which shifts y by up to 2^-25 of the reference; the end takes that out again, and up to 2^26
// the shift is at most 4. So logits count as at least -2^26 (fp16 -6e4), which weighs nothing beside a maximum above
// -2^25 and keeps 0 * y finite where a logit is masked; a CTA whose maximum is outside +-2^25 (LOWEST, HIGHEST) reads
// its part once more on a path that subtracts first.
// The row comes through a ring of three 16 KB bulk copies that one thread keeps full.
// Measured on a B200: 4096 x 151936 bf16 without alternatives 242 us (5.1 TB/s), with five 258 us, with twenty 301 us
// (choosing them takes a CTA some 5 us after its row); 1000 x 201088 fp32 with five 135 us (6.0 TB/s); 64 x 201088 fp32
// without alternatives 14.3 us, with twenty 20.5 to 21.1 us. Tried and slower: CTAs that stay and load the next row's
// first stages while they choose (280 us with five); the bound from 64 groups.
// Split: one CTA per row, four resident per SM; fewer rows than that put a cluster of 2 to 8 CTAs on each row, whose
// partial results the first CTA joins through distributed shared memory.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include "../common.cuh"
#include <algorithm>
#include <tuple>

namespace {

constexpr int WARPS = 8;        // that read the row; one more keeps the ring full
constexpr int THREADS = (WARPS + 1) * 32;
constexpr int STAGES = 3;
constexpr int PER = 4;                    // segments that a warp reads of a stage
constexpr int STAGE_UNITS = PER * WARPS;
constexpr int STAGE_BYTES = STAGE_UNITS * 512;
constexpr int MAX_TOP = 32;     // one entry per lane of a warp's sorted list
constexpr int MAX_CLUSTER = 8;  // the portable cluster size
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// max that keeps a NaN
SNB_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
SNB_DEVICE float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
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

// two fp32 values in a 64-bit register pair
SNB_DEVICE uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
SNB_DEVICE float2 split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
SNB_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SNB_DEVICE uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SNB_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A 16-byte vector of logits. maximum(): of all its values, a NaN stays one. floor(): with values below FLOOR (exact
// in the type) raised to it; that changes nothing where the maximum is above LOWEST. two(): values 2 i and 2 i + 1.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr float FLOOR = -0x1p26f, LOWEST = -0x1p25f, HIGHEST = 0x1p25f;
  static constexpr uint32_t NONE = 0xff800000u;
  static SNB_DEVICE float2 two(const uint4& u, int i) {
    return i == 0 ? make_float2(__uint_as_float(u.x), __uint_as_float(u.y))
                  : make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static SNB_DEVICE float maximum(const uint4& u) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)),
                   max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static SNB_DEVICE uint4 floor(const uint4& u) {
    return make_uint4(__float_as_uint(max_nan(__uint_as_float(u.x), FLOOR)),
                      __float_as_uint(max_nan(__uint_as_float(u.y), FLOOR)),
                      __float_as_uint(max_nan(__uint_as_float(u.z), FLOOR)),
                      __float_as_uint(max_nan(__uint_as_float(u.w), FLOOR)));
  }
  static SNB_DEVICE float one(float v) { return v; }
};
// the 16-bit types: two values in a word
template <typename T, typename T2>
struct Vec16 {
  static constexpr int N = 8;
  static SNB_DEVICE uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }
  static SNB_DEVICE T2 as(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
  static SNB_DEVICE uint32_t bits(T2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
  static SNB_DEVICE T2 most(const uint4& u) {
    return __hmax2_nan(__hmax2_nan(as(u.x), as(u.y)), __hmax2_nan(as(u.z), as(u.w)));
  }
  static SNB_DEVICE uint4 raise(const uint4& u, T2 f) {
    return make_uint4(bits(__hmax2_nan(as(u.x), f)), bits(__hmax2_nan(as(u.y), f)), bits(__hmax2_nan(as(u.z), f)),
                      bits(__hmax2_nan(as(u.w), f)));
  }
};
template <>
struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16, __nv_bfloat162> {
  static constexpr float FLOOR = -0x1p26f, LOWEST = -0x1p25f, HIGHEST = 0x1p25f;
  static constexpr uint32_t NONE = 0xff80ff80u;
  static SNB_DEVICE float2 two(const uint4& u, int i) {
    const uint32_t w = word(u, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static SNB_DEVICE float maximum(const uint4& u) {
    const uint32_t w = bits(most(u));
    return max_nan(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static SNB_DEVICE uint4 floor(const uint4& u) { return raise(u, __float2bfloat162_rn(FLOOR)); }
  static SNB_DEVICE float one(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <>
struct Vec<__half> : Vec16<__half, __half2> {
  static constexpr float FLOOR = -6e4f, LOWEST = -5.9e4f, HIGHEST = 0x1p16f;
  static constexpr uint32_t NONE = 0xfc00fc00u;
  static SNB_DEVICE float2 two(const uint4& u, int i) { return __half22float2(as(word(u, i))); }
  static SNB_DEVICE float maximum(const uint4& u) {
    const float2 m = __half22float2(most(u));
    return max_nan(m.x, m.y);
  }
  static SNB_DEVICE uint4 floor(const uint4& u) { return raise(u, __float2half2_rn(FLOOR)); }
  static SNB_DEVICE float one(__half v) { return __half2float(v); }
};

struct Stats {
  float c, s, t;  // reference, sum of e^y, sum of e^y y
};

// Sums over the first `W` lanes (a power of two), in every one of them
template <int W>
SNB_DEVICE float lane_sum(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
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
                        float* __restrict__ lse_out, float* __restrict__ top_vals, int64_t* __restrict__ top_ids,
                        int* status) {
  constexpr int N = Vec<T>::N;
  extern __shared__ __align__(128) uint8_t dyn[];  // the ring, then the segments' maxima
  float* seg_max = reinterpret_cast<float*>(dyn + STAGES * STAGE_BYTES);
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ float warp_s[WARPS], warp_t[WARPS], warp_best[WARPS + 1];
  __shared__ uint32_t best_keys[WARPS * 32];
  __shared__ float row_c, row_lg;
  __shared__ Stats cta_stats[MAX_CLUSTER];
  __shared__ uint64_t cand[WARPS * MAX_TOP];
  uint32_t* groups = reinterpret_cast<uint32_t*>(cand);  // before it: the groups' maxima of every CTA of the cluster
  static_assert(sizeof(cand) >= MAX_CLUSTER * 32 * 4, "");
  __shared__ uint64_t lists[MAX_CLUSTER * MAX_TOP];  // filled by every CTA of the cluster in the first one's memory
  __shared__ int cand_n, best_n[MAX_CLUSTER];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = gridDim.x, rank = blockIdx.x;  // the cluster spans the grid's x axis
  const uint32_t dst_rank = 0;
  const int64_t row = blockIdx.y;
  if (threadIdx.x == 0) {
    if (TOP) cand_n = 0;
    for (int i = 0; i < STAGES; ++i) {
      snb::mbar_init(&full[i], 1);
      snb::mbar_init(&empty[i], WARPS);
    }
    snb::fence_mbar_init();
  }
  // the first CTA's memory is written from the others: all of them have to be there by then
  __syncwarp();
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  __syncthreads();
  snb::pdl_wait();
  snb::pdl_trigger();
  const T* x = logits + row * stride;
  const RowCut<T> cut(x, V);
  const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
  const int u0 = (int)((int64_t)rank * cut.units / C), u1 = (int)((int64_t)(rank + 1) * cut.units / C);

  float cl = -INFINITY;  // the reference times log2 e; two partial sums each, in the halves of a pair
  uint64_t s2 = 0, t2 = 0;
  float best = -INFINITY;  // this thread's maximum
  bool any = false;        // this thread has seen a logit
  const uint64_t log2e2 = pair(LOG2E, LOG2E);
  auto take = [&](const uint4& a, const uint4& b, float mx) {
    const float ml = max_nan(mx, Vec<T>::FLOOR) * LOG2E;
    if (ml > cl || ml != ml) {  // a reference that has become NaN stays one
      const float f = ex2(cl - ml), d = cl - ml;
      const uint64_t f2 = pair(f, f);
      // sums that weigh nothing now must not meet an infinite distance
      t2 = f > 0.f ? mul2(fma2(s2, pair(d, d), t2), f2) : 0;
      s2 = mul2(s2, f2);
      cl = ml;
    }
    const uint64_t c2 = pair(-cl, -cl);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 r = Vec<T>::floor(h == 0 ? a : b);
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        const float2 v = Vec<T>::two(r, k);
        const uint64_t y2 = fma2(pair(v.x, v.y), log2e2, c2);
        const float2 y = split(y2);
        const uint64_t e2 = pair(ex2(y.x), ex2(y.y));
        s2 = add2(s2, e2);
        t2 = fma2(e2, y2, t2);
      }
    }
  };

  const int v0 = u0 * 32, v1 = min(u1 * 32, cut.nvec);  // this CTA's vectors
  const int stages = (u1 - u0 + STAGE_UNITS - 1) / STAGE_UNITS;
  bool given = false;  // the given token's logit, in the last warp's first lane
  float given_x = 0.f;
  if (warp == WARPS) {
    if (lane == 0) {
      int i = 0;
      for (; i < stages; ++i) {
        const int b = i % STAGES;
        if (!snb::mbar_wait_bounded(&empty[b], ((i / STAGES) & 1) ^ 1, status, SNB_ERR_TIMEOUT_TMA)) break;
        const int v = v0 + i * STAGE_UNITS * 32;
        const uint32_t bytes = min(STAGE_BYTES, (v1 - v) * 16);
        snb::mbar_arrive_expect_tx(&full[b], bytes);
        snb::bulk_load(dyn + b * STAGE_BYTES, body + v, bytes, &full[b]);
      }
      // nothing is in flight when the memory goes away, even if the readers gave up
      for (int d = max(0, i - STAGES); d < i; ++d)
        snb::mbar_wait_bounded(&full[d % STAGES], (d / STAGES) & 1, status, SNB_ERR_TIMEOUT_TMA);
      const int64_t id = ids[row] - vocab_offset;
      given = id >= 0 && id < V;
      if (given) given_x = Vec<T>::one(x[id]);
    }
    __syncwarp();
  } else {
    for (int i = 0; i < stages; ++i) {
      const int b = i % STAGES;
      const bool ok = snb::mbar_wait_bounded(&full[b], (i / STAGES) & 1, status, SNB_ERR_TIMEOUT_MMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      uint4 raw[PER];
      const int first = u0 + i * STAGE_UNITS + warp;
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        const int uj = first + h * WARPS;
        const bool have = uj < u1 && uj * 32 + lane < cut.nvec;
        raw[h] = make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);  // all -inf: adds nothing
        if (have) raw[h] = *reinterpret_cast<const uint4*>(dyn + b * STAGE_BYTES + ((h * WARPS + warp) * 32 + lane) * 16);
        any |= have;
      }
#pragma unroll
      for (int h = 0; h < PER; h += 2) {
        const float mx = max_nan(Vec<T>::maximum(raw[h]), Vec<T>::maximum(raw[h + 1]));
        best = max_nan(best, mx);
        take(raw[h], raw[h + 1], mx);
        if constexpr (TOP) {
          const float seg = warp_max_nan(mx);
          if (lane == 0 && first + h * WARPS < u1) seg_max[((i * PER + h) / 2) * WARPS + warp] = seg;
        }
      }
      __syncwarp();
      if (lane == 0) snb::mbar_arrive(&empty[b]);
    }
  }
  // the ragged ends (head and tail, fewer than two vectors) belong to the first CTA's first warp
  const int ends = cut.head + (V - cut.tail0);
  const bool mine = rank == 0 && warp == 0 && lane < ends;
  const int end_i = lane < cut.head ? lane : cut.tail0 + lane - cut.head;
  float end_v = -INFINITY;
  if (mine) {
    any = true;
    end_v = Vec<T>::one(x[end_i]);
    best = max_nan(best, end_v);
  }
  {
    const float m = warp_max_nan(best);
    if (lane == 0) warp_best[warp] = m;
  }
  __syncthreads();
  float most = warp_best[0];
#pragma unroll
  for (int i = 1; i <= WARPS; ++i) most = max_nan(most, warp_best[i]);

  // From here on against the CTA's maximum, in natural units. A sum that weighs nothing there must not meet an infinite
  // distance; where the maximum is NaN the row is NaN whatever the sums are.
  float st_s = 0.f, st_t = 0.f;
  auto exact = [&](float v) {
    const float y = max_nan(v - most, -1e30f), e = ex2(y * LOG2E);
    st_s += e;
    st_t = fmaf(e, y, st_t);
  };
  if (most <= Vec<T>::LOWEST || most > Vec<T>::HIGHEST) {
    if (warp < WARPS && most != -INFINITY)
      for (int u = u0 + warp; u < u1; u += WARPS) {
        if (u * 32 + lane >= cut.nvec) continue;
        const uint4 raw = __ldg(body + u * 32 + lane);
#pragma unroll 1
        for (int k = 0; k < N / 2; ++k) {
          const float2 v = Vec<T>::two(raw, k);
          exact(v.x);
          exact(v.y);
        }
      }
  } else {
    const float2 ss = split(s2), ts = split(t2);
    const float d = fmaf(-most, LOG2E, cl), f = ex2(d);
    if (f > 0.f) {
      st_s = (ss.x + ss.y) * f;
      st_t = fmaf(ss.x + ss.y, d, ts.x + ts.y) * f * LN2;
    }
  }
  if (mine && most != -INFINITY) exact(end_v);
  st_s = lane_sum<32>(st_s);
  st_t = lane_sum<32>(st_t);
  if (warp < WARPS) {
    if (lane == 0) warp_s[warp] = st_s, warp_t[warp] = st_t;
    if (TOP) best_keys[threadIdx.x] = any ? order_key(best) : 0u;
  }
  __syncthreads();

  // this CTA's sums into the first CTA's shared memory, its groups' maxima into every CTA's
  if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (warp == WARPS) {  // the warp that has the least to do
    Stats a;
    a.c = most;
    a.s = lane_sum<WARPS>(lane < WARPS ? warp_s[lane] : 0.f);
    a.t = lane_sum<WARPS>(lane < WARPS ? warp_t[lane] : 0.f);
    if (lane == 0) {
      const uint32_t at = snb::mapa_shared(snb::smem_u32(&cta_stats[rank]), dst_rank);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(a.c) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(a.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(a.t) : "memory");
    }
    __syncwarp();
  }
  // the maximum of a group: the threads of one lane number
  uint32_t g = 0;
  if constexpr (TOP) {
#pragma unroll
    for (int i = 0; i < WARPS; ++i) g = max(g, best_keys[i * 32 + lane]);
    if (C > 1 && warp < C)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(
                       snb::mapa_shared(snb::smem_u32(&groups[rank * 32 + lane]), warp)),
                   "r"(g)
                   : "memory");
  }
  if (C > 1) {
    snb::cluster_sync();
    if (!TOP && rank != 0) return;
  } else if (!TOP) {
    __syncthreads();
  }

  if constexpr (TOP) {
    // a lower bound of the row's K-th best entry: the K-th largest of 32 groups' maxima, over the whole cluster (0 when
    // fewer than K groups hold any entry); every warp finds it for itself
    if (C > 1) {
      for (int i = 0; i < C; ++i) g = max(g, groups[i * 32 + lane]);
      __syncthreads();
    }
    int above = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) above += __shfl_sync(0xffffffffu, g, i) > g;
    const uint32_t thr = __reduce_min_sync(0xffffffffu, above < K ? g : 0xffffffffu);
    // every warp sorts the entries >= thr of its own segments into a list held across its lanes
    uint64_t list = 0;
    auto insert = [&](uint32_t k32, uint32_t i) {  // the same arguments in every lane
      const uint64_t k = ((uint64_t)k32 << 32) | (0xffffffffu - i);
      const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
      if (k > list) list = (lane > 0 && k > up) ? up : k;
    };
    const int mine_n = warp < WARPS && u1 - u0 - warp > 0 ? (u1 - u0 - warp + 2 * WARPS - 1) / (2 * WARPS) : 0;
#pragma unroll 1
    for (int j0 = 0; j0 < mine_n; j0 += 32) {
      const int j = j0 + lane;
      unsigned sel = __ballot_sync(0xffffffffu, j < mine_n && order_key(seg_max[warp + j * WARPS]) >= thr);
#pragma unroll 1
      while (sel) {
        uint4 raw[4];  // two segments, each two of the warp's units
        int un[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          un[n] = sel ? u0 + warp + (2 * (j0 + __ffs(sel) - 1) + n % 2) * WARPS : u1;
          if (n % 2) sel &= sel - 1;
          raw[n] = make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);
          if (un[n] < u1 && un[n] * 32 + lane < cut.nvec) raw[n] = __ldg(body + un[n] * 32 + lane);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          if (un[n] >= u1) continue;
          // entries come in ascending order of their ids, so one that equals the K-th of a full list stays out
          const uint64_t kth = __shfl_sync(0xffffffffu, list, K - 1);
          const bool full_nan = (uint32_t)(kth >> 32) == 0xffffffffu;  // nothing orders above a NaN
          const uint32_t least = kth ? max(thr, (uint32_t)(kth >> 32) + 1u) : thr;
          unsigned bits = 0;
          if (un[n] * 32 + lane < cut.nvec && !full_nan) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
              const float2 v = Vec<T>::two(raw[n], i);
              bits |= (unsigned)(order_key(v.x) >= least) << (2 * i) | (unsigned)(order_key(v.y) >= least) << (2 * i + 1);
            }
          }
          unsigned from = __ballot_sync(0xffffffffu, bits != 0);
#pragma unroll 1
          while (from) {
            const int src = __ffs(from) - 1;
            from &= from - 1;
            unsigned m = __shfl_sync(0xffffffffu, bits, src);
            const uint4 r = make_uint4(__shfl_sync(0xffffffffu, raw[n].x, src), __shfl_sync(0xffffffffu, raw[n].y, src),
                                       __shfl_sync(0xffffffffu, raw[n].z, src), __shfl_sync(0xffffffffu, raw[n].w, src));
#pragma unroll 1
            for (; m; m &= m - 1) {
              const int i = __ffs(m) - 1;
              const float2 v = Vec<T>::two(r, i / 2);
              insert(order_key(i & 1 ? v.y : v.x), (uint32_t)(cut.head + (un[n] * 32 + src) * N + i));
            }
          }
        }
      }
    }
    if (warp == 0) {
      for (unsigned e = __ballot_sync(0xffffffffu, mine); e; e &= e - 1) {
        const int src = __ffs(e) - 1;
        insert(order_key(__shfl_sync(0xffffffffu, end_v, src)), (uint32_t)__shfl_sync(0xffffffffu, end_i, src));
      }
    }
    const bool valid = lane < K && list != 0;
    const unsigned vm = __ballot_sync(0xffffffffu, valid);
    int base = 0;
    if (lane == 0 && vm) base = atomicAdd(&cand_n, __popc(vm));
    base = __shfl_sync(0xffffffffu, base, 0);
    if (valid) cand[base + lane] = list;
    __syncthreads();
    // the CTA's best K of its warps' lists, into the first CTA's shared memory
    const int n = cand_n;  // at most WARPS * MAX_TOP
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const uint64_t k = cand[i];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) r += cand[j] > k;
      if (r < K) {
        const uint32_t at = snb::mapa_shared(snb::smem_u32(&lists[rank * MAX_TOP + r]), dst_rank);
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(k) : "memory");
      }
    }
    if (threadIdx.x == 0) {
      const uint32_t at = snb::mapa_shared(snb::smem_u32(&best_n[rank]), dst_rank);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(min(n, K)) : "memory");
    }
    if (C > 1) {
      __syncwarp();
      snb::cluster_sync();
      if (rank != 0) return;
    } else {
      __syncthreads();
    }
  }

  if (warp == WARPS) {
    // two partial results join by their maximum: s' = s e^(c - C), t' = (t + s (c - C)) e^(c - C)
    Stats a{-INFINITY, 0.f, 0.f};
    if (lane < C) a = cta_stats[lane];
    const float m = warp_max_nan(a.c), d = a.c - m, f = ex2(d * LOG2E);
    const float ws = lane_sum<MAX_CLUSTER>(f > 0.f ? a.s * f : 0.f);
    const float wt = lane_sum<MAX_CLUSTER>(f > 0.f ? (a.t + a.s * d) * f : 0.f);
    if (lane == 0) {
      const bool none = m == -INFINITY;  // every logit is -inf
      const bool bad = m != m || m == INFINITY;
      const float lg = bad ? NAN : logf(ws);
      float lp = -INFINITY;
      if (given && !none) lp = (given_x - m) - lg;
      logprobs[row] = lp;
      entropy[row] = none ? 0.f : lg - wt / ws;
      lse_out[row] = none ? -INFINITY : m + lg;
      row_c = m;
      row_lg = lg;
    }
  }
  if constexpr (TOP) {
    // the lists' entries differ: an entry's place is how many of all come before it
    const int i = threadIdx.x, r = i / MAX_TOP, p = i % MAX_TOP;
    uint64_t k = 0;
    int at = K;
    if (r < C && p < best_n[r]) {
      k = lists[i];
      at = p;
      for (int q = 0; q < C; ++q) {
        const int n = q == r ? 0 : best_n[q];
#pragma unroll 4
        for (int j = 0; j < n; ++j) at += lists[q * MAX_TOP + j] > k;
      }
    }
    __syncthreads();
    if (at < K) {
      top_vals[row * K + at] = row_c == -INFINITY ? -INFINITY : (key_value((uint32_t)(k >> 32)) - row_c) - row_lg;
      top_ids[row * K + at] = vocab_offset + (int64_t)(0xffffffffu - (uint32_t)k);
    }
  }
}

template <typename T>
void launch(const at::Tensor& logits, int V, const at::Tensor& ids, int64_t vocab_offset, int K,
            at::Tensor& logprobs, at::Tensor& entropy, at::Tensor& lse, at::Tensor& top_vals, at::Tensor& top_ids,
            int* status) {
  const int64_t rows = logits.size(0);
  const auto* prop = at::cuda::getCurrentDeviceProperties();
  auto st = at::cuda::getCurrentCUDAStream();
  const int units = (V / Vec<T>::N + 31) / 32;
  // CTAs per row: enough to fill four CTAs per SM, as long as each keeps a load per warp in flight
  int C = 1;
  while (C < MAX_CLUSTER && rows * C * 2 <= (int64_t)prop->multiProcessorCount * 4 && units >= C * 2 * WARPS) C *= 2;
  const size_t smem = STAGES * STAGE_BYTES + (K > 0 ? sizeof(float) * ((units + C - 1) / C + 2 * WARPS) : 0);
  TORCH_CHECK(smem <= 200 * 1024, "token_logprobs: the vocabulary is too wide for top_k");
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
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, x, logits.stride(0), V, id, vocab_offset, K,
                                      logprobs.data_ptr<float>() + r0, entropy.data_ptr<float>() + r0,
                                      lse.data_ptr<float>() + r0, tv, ti, status));
  }
}

}  // namespace

// logits: [N, >= V] bf16 / fp16 / fp32, any row stride; only the first V columns are read, whatever the rest holds
// (V = 0: all). ids: [N] int64 or int32 (less vocab_offset outside [0, V): log-probability -inf). Returns fp32 [N]
// log-probability, entropy and log-sum-exp, the K best log-probabilities [N, K] and their ids.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> logits_stats(
    at::Tensor logits, int64_t V, at::Tensor ids, int64_t vocab_offset, int64_t K, at::Tensor status) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "token_logprobs: logits must be [rows, vocabulary] on CUDA");
  const int64_t N = logits.size(0);
  if (V == 0) V = logits.size(1);
  TORCH_CHECK(V > 0 && V <= logits.size(1) && V < (int64_t(1) << 30),
              "token_logprobs: valid_vocab is outside the logits' columns");
  static_assert(MAX_TOP == 32, "the message names it");
  TORCH_CHECK(K >= 0 && K <= MAX_TOP && K <= V, "token_logprobs: top_k must be 0 to 32 and at most the vocabulary");
  TORCH_CHECK(ids.dim() == 1 && ids.numel() == N && ids.device() == logits.device() &&
                  (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
              "token_logprobs: ids must be one int64 or int32 per row on the logits' device");
  const auto dt = logits.scalar_type();
  TORCH_CHECK(dt == at::kFloat || dt == at::kBFloat16 || dt == at::kHalf,
              "token_logprobs: takes bf16, fp16 or fp32 on CUDA");
  const c10::cuda::CUDAGuard guard(logits.device());
  if (logits.stride(1) != 1 && logits.size(1) > 1) logits = logits.contiguous();
  if (ids.scalar_type() != at::kLong) ids = ids.to(at::kLong);
  ids = ids.contiguous();
  auto make = [&](at::IntArrayRef size, at::ScalarType type) {
    return at::Tensor(at::detail::empty_cuda(size, type, logits.device(), std::nullopt));
  };
  auto logprobs = make({N}, at::kFloat), entropy = make({N}, at::kFloat), lse = make({N}, at::kFloat);
  auto top_vals = make({N, K}, at::kFloat), top_ids = make({N, K}, at::kLong);
  int* st = status.data_ptr<int>();
  if (N > 0) {
    auto run = [&](auto kind) {
      launch<decltype(kind)>(logits, (int)V, ids, vocab_offset, (int)K, logprobs, entropy, lse, top_vals, top_ids, st);
    };
    if (dt == at::kFloat) run(float());
    else if (dt == at::kHalf) run(__half());
    else run(__nv_bfloat16());
  }
  return {logprobs, entropy, lse, top_vals, top_ids};
}
