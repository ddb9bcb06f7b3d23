// Causal attention of packed whole prompts (no cache): every prompt's queries over its own keys and values.
//
//   out[t, h] = sum_j p_j v[j, h / G],   p_j = exp(scale q[t, h] . k[j, h / G] - m) / (exp(sink[h] - m) + sum_j ...)
//   over the tokens j <= t of the same prompt, t - j < window where a window is set.
//
// One pass over the keys in blocks of 128 with a running reference m and sum. A persistent CTA per SM works on two
// query tiles of 128 rows that share their keys and values: scores S = Q K^T and output O += P V on tcgen05 with S, P
// and O in tensor memory (P over the S it came from: 2 x (128 + 128) columns at head width 128), Q, K and V by TMA.
// 16 softmax warps: two threads per row, 64 keys each.
//
// What bounds it: the softmax warps. A block of both tiles is 2048 cycles of tensor core at head width 128 and takes
// about 2600; per score they spend 0.75 exponentials of the special-function unit's 1/4 a cycle and scheduler (the rest
// runs on the FMA pipe), the packing to 16 bits and the sums. Measured on a B200, 30 launches after a pause: one
// 8192-token prompt, 32 / 8 heads of 128: 427 to 431 us, 1280 TFLOP/s (under a second's load, where power lowers the
// clock, 498 us, 1105 TFLOP/s); 64 / 8 heads of 64: 642 us, 857 TFLOP/s (the same scores at half the products); 16 heads
// of 192 / 128: 336 us, 1023 TFLOP/s; 4096 tokens, 64 / 8 heads of 64, window 128: 43.3 us.
// Registers: 18 warps leave a thread 96. In bytes of stores and loads, 192 / 128 spills 56 / 84 (fp16 44 / 68), bf16 of
// 128 / 128 8 / 12, bf16 of 64 / 64 8 / 4, the others nothing.
// The running maximum and sum are the online softmax (Milakov and Gimelshein 2018).
// Tried and slower: one thread per row (its chain of loads, maximum, exponentials is twice as long: 575 us); turns of
// the two tiles at the exponentials (with one thread per row 4 % faster, with two a loss); heads of 64 with one tile
// per CTA and two CTAs per SM (687 us against 650).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include "../common.cuh"
#include "../tma_host.h"
#include <algorithm>
#include <type_traits>

namespace {

// Of each 8 pairs of exponentials those with the last index of every EMULATE run on the FMA pipe. One 8192-token prompt
// with 4, 2 (EMULATE 3 and 4), 1 and none of 8 there: 32 / 8 heads of 128 465, 431, 421, 419 us; 64 / 8 heads of 64 742,
// 642, 633, 685 us; 16 heads of 192 / 128 339, 336, 338, 336 us.
constexpr int EMULATE = 4;
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

// two fp32 values in one 64-bit register pair: one issue slot for both
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
SNB_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
SNB_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SNB_DEVICE float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
SNB_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

SNB_DEVICE float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of two values on the FMA pipe: x = n + f with n the nearest integer (found by adding 1.5 * 2^23) and |f| <= 1/2,
// 2^f by the cubic with p(0) = 1 whose largest relative error on that interval is least (1.02e-4, by Remez exchange;
// weights are rounded to 2^-9 or 2^-12 next), n added to the exponent. At -127 and below, masked scores of -inf among
// them, the result is exactly 0 (p(0) = 1 has no mantissa, and the exponent is 0), so what is masked adds nothing; down
// to -126 it is a value below 2^-126. 128 and above (`HIGH`: x can get there) and NaN become values past every 16-bit
// type's range.
template <bool HIGH>
SNB_DEVICE float2 exp2_fma(uint64_t x) {
  float2 c = split(x);
  c.x = max_nan(c.x, -127.f);
  c.y = max_nan(c.y, -127.f);
  if (HIGH) {
    c.x = min_nan(c.x, 128.f);
    c.y = min_nan(c.y, 128.f);
  }
  x = pair(c.x, c.y);
  const uint64_t big = pair(12582912.f, 12582912.f), less = pair(-12582912.f, -12582912.f);
  const uint64_t n = add2(x, big);
  const uint64_t f = fma2(add2(n, less), pair(-1.f, -1.f), x);
  uint64_t y = fma2(pair(0.055009059607982635f, 0.055009059607982635f), f, pair(0.2422109693288803f, 0.2422109693288803f));
  y = fma2(y, f, pair(0.6932829022407532f, 0.6932829022407532f));
  y = fma2(y, f, pair(1.f, 1.f));
  const float2 ny = split(n), r = split(y);
  return make_float2(__int_as_float(__float_as_int(r.x) + (__float_as_int(ny.x) << 23)),
                     __int_as_float(__float_as_int(r.y) + (__float_as_int(ny.y) << 23)));
}

// Bits 0 .. n (none for n < 0, all for n > 31)
SNB_DEVICE uint32_t upto(int n) { return n < 0 ? 0u : 0xffffffffu >> (31 - min(n, 31)); }

struct PromptParams {
  const void *q, *k, *v;
  void* out;
  int64_t qs, ks, vs, os;  // row strides, in elements
  const int* indptr;
  const float* sinks;
  int T, B, heads, kv_heads, window;
  float scale;  // of the scores, in log2 units
  int pair_heads, pairs, items;
  int wide_out;  // output rows lie on 32-byte boundaries
  uint32_t idesc;  // the operands' type, for the MMA
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

// ---- tensor-core kernel ---------------------------------------------------------------------------------------
constexpr int BQ = 128;  // query rows of a tile: one tensor-memory lane and one softmax thread each
constexpr int BKV = 128;  // keys of a block
constexpr int CHUNK = 128 * 128;  // bytes of 128 rows x 64 16-bit elements (one swizzled TMA box)
constexpr int LOAD_WARP = 16, MMA_WARP = 17;
constexpr int THREADS = 18 * 32;  // 2 tiles x 2 halves of the keys x 4 softmax warps, a load warp, an MMA warp

template <int D, int DV>
struct Cfg {
  static constexpr int QB = D / 64 * CHUNK, KB = D / 64 * CHUNK, VB = DV / 64 * CHUNK;
  static constexpr int NK = D == 64 ? 4 : D == 128 ? 3 : 2, NV = D == 64 ? 4 : D == 128 ? 2 : 1;
  static constexpr int SMEM = 2 * QB + NK * KB + NV * VB + 2 * BQ * 4 + 1024 + 512;  // + exchange, alignment, barriers and items
};

// One lane of a converged warp; the compiler keeps what such a branch uses in uniform registers, which the MMA's
// operands have to be in (converting them costs more than the 64 cycles that an MMA takes).
SNB_DEVICE bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// D[tmem] (+)= A[tmem] B[smem]: A holds two 16-bit values per 32-bit column
SNB_DEVICE void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
SNB_DEVICE void tmem_st_x32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(at)
      : "memory");
}
SNB_DEVICE void tmem_st_x8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(at)
               : "memory");
}
SNB_DEVICE void tmem_ld_x16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
// Named barriers of the two warps that share a quarter of a tile's rows (64 threads)
SNB_DEVICE void bar_pair(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
SNB_DEVICE bool bar_or(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.or.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)v)
      : "memory");
  return r != 0;
}
// 32 bytes, a whole sector: a row belongs to a thread, so a warp's store touches 32 rows
SNB_DEVICE void st_global_v8(void* at, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
SNB_DEVICE void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// B operand whose rows (keys) are the contraction: 64-wide column chunks `CHUNK` bytes apart, 8-row groups 1024 apart
SNB_DEVICE uint64_t desc_v(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | (uint64_t)(CHUNK >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// A work item: two query tiles that share their keys and values. With an even group size they are two heads of one
// group over the same 128 tokens, otherwise 256 consecutive tokens of one head.
struct Item {
  int first, len;  // the prompt's first token and length
  int r0;          // first query row, counted from `first`
  int h0;          // head of the first tile
  int kb0, kb1;    // key blocks [kb0, kb1), counted from `first`; none: the list has ended
};

// How far the list has been counted: a CTA's items ascend, so it goes over the prompts' bounds once.
struct Cursor {
  int phase = 0, b0 = 0, before = 0;
};

// Item w of the list (tile, head pair): the prompts in order, each prompt's tiles from its last one down to the second,
// then the first tiles of all prompts, which see the fewest keys and even out the end. Called by whole warps with
// ascending w. False past the end.
SNB_DEVICE bool decode_item(const PromptParams& p, int w, Cursor& at, Item& it) {
  const int lane = threadIdx.x & 31;
  const int rows = p.pair_heads ? BQ : 2 * BQ;
  const int idx = w / p.pairs, pair = w % p.pairs;
  for (; at.phase < 2; ++at.phase, at.b0 = 0)
    for (; at.b0 < p.B; at.b0 += 32) {
      const int b = at.b0 + lane;
      int a = 0, n = 0;
      if (b < p.B) {
        a = seq_bound(p, b);
        n = max(0, seq_bound(p, b + 1) - a);
      }
      const int nt = (n + rows - 1) / rows;
      int incl = at.phase == 0 ? max(nt - 1, 0) : min(nt, 1);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const unsigned in = __ballot_sync(0xffffffffu, incl > idx - at.before);
      if (in) {
        const int src = __ffs(in) - 1;
        it.first = __shfl_sync(0xffffffffu, a, src);
        it.len = __shfl_sync(0xffffffffu, n, src);
        it.r0 = at.phase == 0 ? (__shfl_sync(0xffffffffu, incl, src) - (idx - at.before)) * rows : 0;
        it.h0 = p.pair_heads ? pair * 2 : pair;
        it.kb1 = (min(it.len, it.r0 + rows) + BKV - 1) / BKV;
        it.kb0 = p.window > 0 ? max(0, it.r0 - p.window + 1) / BKV : 0;
        return true;
      }
      at.before += __shfl_sync(0xffffffffu, incl, 31);
    }
  return false;
}

// This CTA's r-th item. The list's items mostly shrink slowly (a prompt's tiles come last tile first), so the CTAs take
// them in alternating order: 0..n-1, then n-1..0.
SNB_DEVICE bool next_item(const PromptParams& p, int r, Cursor& at, Item& it) {
  const int n = gridDim.x;
  const int64_t w = (int64_t)r * n + ((r & 1) ? n - 1 - blockIdx.x : blockIdx.x);
  return w < p.items && decode_item(p, (int)w, at, it);
}

template <typename T, int D, int DV>
__global__ void __launch_bounds__(THREADS, 1)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                            const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tq32,
                            const __grid_constant__ PromptParams p, int* status) {
  using C = Cfg<D, DV>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * C::QB;
  uint8_t* sV = sK + C::NK * C::KB;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sV + C::NV * C::VB);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + C::NK;
  uint64_t* v_full = k_empty + C::NK;
  uint64_t* v_empty = v_full + C::NV;
  uint64_t* s_full = v_empty + C::NV;  // [2] scores of a tile are in tensor memory
  uint64_t* p_full = s_full + 2;       // [2][2] the first / second half of a tile's weights are (its output rescaled)
  uint64_t* o_full = p_full + 4;       // [2] a tile's output has taken up a block
  uint64_t* i_full = o_full + 2;       // [2] a work item is in its slot
  uint64_t* i_empty = i_full + 2;      // [2] and has been read by the softmax warps and the MMA warp
  uint64_t* drain = i_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* issued = reinterpret_cast<int*>(tmem_slot + 1);  // loads issued: q, k, v
  int* taken = issued + 3;                              // and waited for
  float* sX = reinterpret_cast<float*>(taken + 3);      // [2][128] what the two halves of a row exchange
  Item* sItem = reinterpret_cast<Item*>(sX + 2 * BQ);   // [2]
  float* sSink = reinterpret_cast<float*>(sItem + 2);   // [4][2] the sinks of an item's two heads

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    snb::mbar_init(q_full, 1);
    snb::mbar_init(q_empty, 1);
    for (int i = 0; i < C::NK; ++i) snb::mbar_init(&k_full[i], 1), snb::mbar_init(&k_empty[i], 1);
    for (int i = 0; i < C::NV; ++i) snb::mbar_init(&v_full[i], 1), snb::mbar_init(&v_empty[i], 1);
    for (int j = 0; j < 2; ++j) {
      snb::mbar_init(&s_full[j], 1);
      snb::mbar_init(&p_full[2 * j], 8);
      snb::mbar_init(&p_full[2 * j + 1], 8);
      snb::mbar_init(&o_full[j], 1);
    }
    for (int i = 0; i < 2; ++i) snb::mbar_init(&i_full[i], 1), snb::mbar_init(&i_empty[i], 17);
    snb::mbar_init(drain, 1);
    for (int i = 0; i < 6; ++i) issued[i] = 0;
    snb::fence_mbar_init();
  }
  if (threadIdx.x == LOAD_WARP * 32) {
    snb::prefetch_tmap(&tq);
    snb::prefetch_tmap(&tq32);
    snb::prefetch_tmap(&tk);
    snb::prefetch_tmap(&tv);
  }
  if (warp == MMA_WARP) {
    snb::tmem_alloc(tmem_slot, 512);
    snb::tmem_relinquish();
  }
  snb::tc_fence_before();
  __syncthreads();
  snb::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  snb::pdl_trigger();
  snb::pdl_wait();
  const int G = p.heads / p.kv_heads;

  if (warp == LOAD_WARP) {
    int nq = 0, nk = 0, nv = 0;
    bool ok = true;
    Cursor cursor;
    // It alone works the items out (a few global reads and divisions) and hands them over one item ahead.
    auto publish = [&](int r, Item& it) {
      const bool have = next_item(p, r, cursor, it);
      if (!have) it.kb0 = it.kb1 = 0;
      if (lane == 0) {
        float sink[2] = {0.f, 0.f};
        if (have && p.sinks != nullptr) {
          sink[0] = __ldg(p.sinks + it.h0);
          sink[1] = __ldg(p.sinks + it.h0 + (p.pair_heads ? 1 : 0));
        }
        ok = snb::mbar_wait_bounded(&i_empty[r & 1], ((r >> 1) & 1) ^ 1, status, SNB_ERR_TIMEOUT_TMA);
        if (ok) {
          sItem[r & 1] = it;
          // read at the item's end, when the slot of the item itself may be taken: item r - 4 is over by now, since
          // every softmax warp has taken item r - 2
          sSink[(r & 3) * 2] = sink[0];
          sSink[(r & 3) * 2 + 1] = sink[1];
          snb::mbar_arrive(&i_full[r & 1]);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      return have;
    };
    Item it, next;
    int hk = 0;
    auto load_k = [&](int kb) {
      const int s = nk % C::NK;
      if (!snb::mbar_wait_bounded(&k_empty[s], ((nk / C::NK) & 1) ^ 1, status, SNB_ERR_TIMEOUT_TMA)) return false;
      snb::mbar_arrive_expect_tx(&k_full[s], C::KB);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        snb::tma_load_2d(sK + s * C::KB + c * CHUNK, &tk, &k_full[s], hk * D + c * 64, it.first + kb * BKV);
      ++nk;
      return true;
    };
    auto load_v = [&](int kb) {
      const int s = nv % C::NV;
      if (!snb::mbar_wait_bounded(&v_empty[s], ((nv / C::NV) & 1) ^ 1, status, SNB_ERR_TIMEOUT_TMA)) return false;
      snb::mbar_arrive_expect_tx(&v_full[s], C::VB);
#pragma unroll
      for (int c = 0; c < DV / 64; ++c)
        snb::tma_load_2d(sV + s * C::VB + c * CHUNK, &tv, &v_full[s], hk * DV + c * 64, it.first + kb * BKV);
      ++nv;
      return true;
    };
    auto load_q = [&]() {
      if (!snb::mbar_wait_bounded(q_empty, (nq & 1) ^ 1, status, SNB_ERR_TIMEOUT_TMA)) return false;
      snb::mbar_arrive_expect_tx(q_full, 2 * C::QB);
      // The second tile's quarters of 32 rows lie in the opposite order: a quarter belongs to one scheduler's warps, and
      // where a mask cuts blocks (the diagonal, a window) its rows leave some quarters whole and some empty. Four
      // prompts near 1024 tokens, 64 heads of 64, window 128: 54.8 us with both tiles in order, 50.8 us like this.
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        snb::tma_load_2d(sQ + c * CHUNK, &tq, q_full, it.h0 * D + c * 64, it.first + it.r0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          snb::tma_load_2d(sQ + C::QB + c * CHUNK + (3 - i) * (CHUNK / 4), &tq32, q_full,
                           (it.h0 + (p.pair_heads ? 1 : 0)) * D + c * 64,
                           it.first + it.r0 + (p.pair_heads ? 0 : BQ) + i * 32);
      }
      ++nq;
      return true;
    };
    bool have = publish(0, it);
    for (int r = 0; ok && have; ++r, it = next) {
      hk = it.h0 / G;
      if (lane == 0) ok = load_k(it.kb0) && load_q();
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      have = publish(r + 1, next);
      if (lane == 0)
        for (int kb = it.kb0; ok && kb < it.kb1; ++kb) ok = load_v(kb) && (kb + 1 == it.kb1 || load_k(kb + 1));
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (lane == 0) issued[0] = nq, issued[1] = nk, issued[2] = nv;
  } else if (warp == MMA_WARP) {
    int nq = 0, nk = 0, nv = 0, np = 0;
    bool ok = true;
    const uint32_t id_s = p.idesc | snb::idesc_bf16_f32(BQ, BKV) & ~(7u << 7 | 7u << 10);
    const uint32_t id_o = p.idesc | snb::idesc_bf16_f32(BQ, DV) & ~(7u << 7 | 7u << 10) | 1u << 16;
    const uint64_t q_desc = snb::smem_desc_sw128(snb::smem_u32(sQ)), k_desc = snb::smem_desc_sw128(snb::smem_u32(sK)),
                   v_desc = desc_v(snb::smem_u32(sV));
    auto wait = [&](uint64_t* bar, int parity) {
      const bool r = snb::mbar_wait_bounded(bar, parity, status, SNB_ERR_TIMEOUT_MMA);
      snb::tc_fence_after();
      return __all_sync(0xffffffffu, r) != 0;
    };
    // addresses in descriptors count 16-byte units
    auto scores = [&](int j, int s) {
      const uint64_t a = q_desc + j * (C::QB >> 4), b = k_desc + s * (C::KB >> 4);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int off = ((k / 4) * CHUNK + (k % 4) * 32) >> 4;
          snb::mma_bf16_ss(tmem + j * 128, a + off, b + off, id_s, k > 0);
        }
        snb::mma_commit(&s_full[j]);
      }
    };
    // Half `part` of a block's weights: keys 32 part .. 32 part + 31 of each half of the block
    auto output = [&](int j, int s, int part, bool more) {
      const uint64_t b = v_desc + s * (C::VB >> 4);
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < BKV / 32; ++i) {
          const int k = (i / 2) * 4 + part * 2 + i % 2;
          mma_ts(tmem + 256 + j * DV, tmem + j * 128 + (k / 4) * 64 + (k % 4) * 8, b + k * (2048 >> 4), id_o,
                 more || i > 0);
        }
        if (part) snb::mma_commit(&o_full[j]);
      }
    };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) snb::mma_commit(bar);
    };
    for (int r = 0; ok; ++r) {
      ok = wait(&i_full[r & 1], (r >> 1) & 1);
      if (!ok) break;
      const int nb = sItem[r & 1].kb1 - sItem[r & 1].kb0;
      __syncwarp();
      if (lane == 0) snb::mbar_arrive(&i_empty[r & 1]);
      if (nb == 0) break;
      ok = wait(q_full, nq & 1) && wait(&k_full[nk % C::NK], (nk / C::NK) & 1);
      if (ok) {
        scores(0, nk % C::NK);
        scores(1, nk % C::NK);
        commit(&k_empty[nk % C::NK]);
        ++nk;
        if (nb == 1) commit(q_empty);
      }
      for (int i = 0; ok && i < nb; ++i) {
        const bool next = i + 1 < nb;
        const int ks = nk % C::NK, vs = nv % C::NV;
        ok = (!next || wait(&k_full[ks], (nk / C::NK) & 1)) && wait(&v_full[vs], (nv / C::NV) & 1);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ok = ok && wait(&p_full[2 * j], np & 1);
          if (!ok) break;
          output(j, vs, 0, i > 0);
          ok = wait(&p_full[2 * j + 1], np & 1);
          if (!ok) break;
          output(j, vs, 1, true);
          if (next) scores(j, ks);
        }
        if (!ok) break;
        commit(&v_empty[vs]);
        ++nv;
        ++np;
        if (next) {
          commit(&k_empty[ks]);
          ++nk;
          if (i + 2 == nb) commit(q_empty);
        }
      }
      ++nq;
    }
    if (lane == 0) taken[0] = nq, taken[1] = nk, taken[2] = nv;
    if (!ok) {  // products in flight still read this CTA's memory
      commit(drain);
      snb::mbar_wait_bounded(drain, 0, status, SNB_ERR_TIMEOUT_MMA);
    }
  } else {
    // Softmax: a row belongs to two threads, each with 64 of a block's 128 keys, in two warps of the same quarter of
    // the tile's rows. Their scores lie in columns [64 h, 64 h + 64) of the tile's scores; their weights go over the
    // first half of those.
    const int j = warp >> 3, h = (warp >> 2) & 1, bar = 1 + j * 4 + (warp & 3);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + j * 128 + h * 64 + lanes, o_at = tmem + 256 + j * DV + h * (DV / 2) + lanes;
    const int quarter = (j == 0 ? warp & 3 : 3 - (warp & 3)) * 32;  // its first row, see load_q
    float* x = sX + j * BQ + (warp & 3) * 32 + lane;
    int ns = 0;  // blocks done by this tile, over all items
    bool ok = true;
    constexpr bool NARROW = std::is_same<T, __half>::value;
    auto wait = [&](uint64_t* b, int parity) {
      const bool r = snb::mbar_wait_bounded(b, parity, status, SNB_ERR_TIMEOUT_EPI);
      snb::tc_fence_after();
      return __all_sync(0xffffffffu, r) != 0;
    };
    // both halves get op(first half's v, second half's v)
    auto exchange = [&](float v, auto op) {
      if (h == 1) *x = v;
      bar_pair(bar);
      if (h == 0) *x = v = op(v, *x);
      bar_pair(bar);
      return h == 0 ? v : *x;
    };
    // A wait that ran out must end both warps of a pair at the same place: the pair agrees on `ok` at the barrier that
    // each block and each item has anyway.
    for (int r = 0; ok; ++r) {
      ok = wait(&i_full[r & 1], (r >> 1) & 1);
      if (bar_or(bar, !ok)) {
        ok = false;
        break;
      }
      const Item it = sItem[r & 1];
      __syncwarp();
      if (lane == 0) snb::mbar_arrive(&i_empty[r & 1]);
      if (it.kb0 == it.kb1) break;
      const int head = it.h0 + (p.pair_heads ? j : 0);
      const int r0 = it.r0 + (p.pair_heads ? 0 : j * BQ);
      const int rel = r0 + quarter + lane;  // this thread's query, counted from the prompt's first token
      const int rw = r0 + quarter;  // this warp's first query
      const int lo = p.window > 0 ? rel - p.window + 1 : 0;
      float m = -INFINITY, l = 0.f;  // the reference, in log2 units; the weights' sum over this thread's keys
      for (int kb = it.kb0; kb < it.kb1; ++kb, ++ns) {
        ok = wait(&s_full[j], ns & 1) && ok;
        // The scores are read 16 columns at a time with the next 16 under way: all 64 would not fit the 96 registers
        // that 18 warps leave a thread, and with this much shared memory a spill goes to L2.
        const int k0 = kb * BKV + h * 64;
        uint32_t s[2][16];
        // What this warp's 32 rows see of 16 keys: nothing (0), a part (1) or all of them (2)
        auto sight = [&](int c) {
          const int kc = k0 + c * 16;
          if (kc > rw + 31 || (p.window > 0 && kc + 15 <= rw - p.window)) return 0;
          return kc + 15 > rw || (p.window > 0 && kc <= rw + 31 - p.window) ? 1 : 2;
        };
        auto next_chunk = [&](auto cut, int c, bool more) {
          snb::tmem_ld_wait();
          if (more) tmem_ld_x16(s_at + ((c + 1) & 3) * 16, s[(c + 1) & 1]);
          if (cut.value && sight(c) == 1) {  // of those that no row sees the caller makes nothing
            const uint32_t seen = upto(rel - k0 - c * 16) & ~upto(lo - 1 - k0 - c * 16);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[c & 1][i] = (seen >> i & 1) ? s[c & 1][i] : 0xff800000u;
          }
        };
        // The output in tensor memory follows a change of the reference by 2^-d, after the product `phase`. The stores
        // have landed on return: after an item's last block the epilogue reads the same columns with nothing in between.
        auto rescale = [&](float f, int phase) {
          ok = wait(&o_full[j], phase & 1);
#pragma unroll 1
          for (int c = 0; c < DV / 64; ++c) {
            uint32_t o[32];
            snb::tmem_ld_32x32b_x32(o_at + c * 32, o);
            snb::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_x32(o_at + c * 32, o);
          }
          tmem_st_wait();
        };
        // Blocks that every row sees whole take a path without the tests: those cost as much as the exponentials.
        const bool ragged = kb * BKV + BKV - 1 > r0 || (p.window > 0 && kb * BKV < r0 + BQ - p.window);
        tmem_ld_x16(s_at, s[0]);
        // Before the exponentials: a row's first block sets its reference to that block's maximum. For bf16 that may
        // be the maximum of masked scores too: a reference far above what the row sees costs no precision, only range,
        // and a row that runs out of it is computed once more below. fp16 weights have to lie between 2^-14 and 2^16,
        // so there every block's maximum over what the row sees is looked at, and the reference follows once it has
        // risen by 2^8. (A row's two threads hold the same m: they agree on this branch.)
        if (NARROW || __any_sync(0xffffffffu, m == -INFINITY)) {
          float mx[2] = {-INFINITY, -INFINITY};
          auto maximum = [&](auto cut) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              next_chunk(cut, c, true);
              if (cut.value && sight(c) == 0) continue;
#pragma unroll
              for (int i = 0; i < 16; i += 2)
                mx[i / 2 & 1] = max3(mx[i / 2 & 1], __uint_as_float(s[c & 1][i]), __uint_as_float(s[c & 1][i + 1]));
            }
          };
          if (NARROW && ragged) maximum(std::true_type());
          else maximum(std::false_type());
          const float top = fmaxf(mx[0], mx[1]) * p.scale;
          const bool rise = m == -INFINITY ? top > m : top - m > 8.f;
          if (!NARROW || bar_or(bar, rise || !ok)) {
            if (bar_or(bar, !ok)) {
              ok = false;
              break;
            }
            const float mn = fmaxf(m, exchange(top, [](float a, float b) { return fmaxf(a, b); }));
            const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
            l *= f;
            m = mn;
            if (kb > it.kb0) rescale(f, ns - 1);
          }
        }
        const float ref = m == -INFINITY ? 0.f : -m;
        const uint64_t scale2 = pair(p.scale, p.scale), ref2 = pair(ref, ref);
        uint64_t sum[2] = {0, 0};
        auto weights = [&](auto cut) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w2[8];
            next_chunk(cut, c, c < 3);
            if (cut.value && sight(c) == 0) {
#pragma unroll
              for (int i = 0; i < 8; ++i) w2[i] = 0;
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint64_t y = fma2(pair(__uint_as_float(s[c & 1][2 * i]), __uint_as_float(s[c & 1][2 * i + 1])),
                                        scale2, ref2);
                float2 e;
                if (i % EMULATE == EMULATE - 1) {
                  e = exp2_fma<!NARROW>(y);
                } else {
                  e = split(y);
                  e.x = ex2(e.x);
                  e.y = ex2(e.y);
                }
                w2[i] = pack2<T>(e.x, e.y);
                // a row of few keys (it sees all of them in ragged blocks) sums the weights as rounded: what the
                // product uses then adds up to one
                if (cut.value) e = unpack2<T>(w2[i]);
                sum[i & 1] = add2(sum[i & 1], pair(e.x, e.y));
              }
            }
            tmem_st_x8(s_at + c * 8, w2);
            if (c & 1) {  // half of the weights: their product can start
              tmem_st_wait();
              snb::tc_fence_before();
              __syncwarp();
              if (lane == 0) snb::mbar_arrive(&p_full[2 * j + c / 2]);
              __syncwarp();  // the tensor-memory instructions want the whole warp
            }
          }
        };
        if (ragged) weights(std::true_type());
        else weights(std::false_type());
        const float2 total = split(add2(sum[0], sum[1]));
        const float block = total.x + total.y;
        l += block;
        // After them, off the critical path: bf16 weights have fp32's range, so a reference that lags costs no
        // precision. It follows when a block's weights have come to more than 2^16; a weight past 2^128 in one step
        // turns the row's output into an infinity, and such rows are computed once more below.
        if (!NARROW && bar_or(bar, block > 65536.f || !ok)) {
          if (bar_or(bar, !ok)) {
            ok = false;
            break;
          }
          const float most = exchange(block, [](float a, float b) { return fmaxf(a, b); });
          // 2^-126 is the least factor that is not flushed to 0
          const float up = most > 65536.f ? (float)min((__float_as_int(most) >> 23) - 126, 126) : 0.f;
          const float f = ex2(-up);
          l *= f;
          m += up;
          rescale(f, ns);
        }
      }
      if (!ok) break;
      ok = wait(&o_full[j], (ns - 1) & 1);
      if (bar_or(bar, !ok)) {
        ok = false;
        break;
      }
      l = exchange(l, [](float a, float b) { return a + b; });
      // NaN if the sum over the keys left its range or an output is not finite
      float zero = l > 0x1p-100f && l < 0x1p100f ? 0.f : NAN;
      if (p.sinks != nullptr) l += ex2(sSink[(r & 3) * 2 + j] * LOG2E - (m == -INFINITY ? 0.f : m));
      const float inv = m == -INFINITY ? 0.f : 1.f / l;  // only scores of -inf: nothing but the sink has weight
      const bool store = rel < it.len;
      const int t = it.first + rel;
      T* dst = reinterpret_cast<T*>(p.out) + (int64_t)t * p.os + (int64_t)head * DV + h * (DV / 2);
#pragma unroll
      for (int c = 0; c < DV / 64; ++c) {
        uint32_t o[32];
        snb::tmem_ld_32x32b_x32(o_at + c * 32, o);
        snb::tmem_ld_wait();
        uint32_t w2[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float a = __uint_as_float(o[2 * i]) * inv, b = __uint_as_float(o[2 * i + 1]) * inv;
          zero = fmaf(a, 0.f, zero);
          zero = fmaf(b, 0.f, zero);
          w2[i] = pack2<T>(a, b);
        }
        if (store) {
          if (p.wide_out) {
#pragma unroll
            for (int i = 0; i < 2; ++i) st_global_v8(dst + c * 32 + i * 16, w2 + i * 8);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(dst + c * 32 + i * 8) =
                  make_uint4(w2[4 * i], w2[4 * i + 1], w2[4 * i + 2], w2[4 * i + 3]);
          }
        }
        __syncwarp();
      }
      const bool odd = zero != 0.f;
      // A NaN or infinity in a masked value still meets a weight of 0 in the product (0 * inf = NaN), and a masked
      // score can have set the reference: rows that came out without a finite result are computed once more,
      // touching nothing that is masked.
      if (bar_or(bar, odd && store)) {
        const bool either = exchange(odd && store ? 1.f : 0.f, [](float a, float b) { return fmaxf(a, b); }) > 0.f;
        unsigned again = h == 0 ? __ballot_sync(0xffffffffu, either) : 0u;
        while (again) {
          const int src = __ffs(again) - 1;
          again &= again - 1;
          attend_row<T, D, DV>(p, it.first, it.first + r0 + quarter + src, head);
        }
      }
    }
  }
  snb::tc_fence_before();
  __syncthreads();
  if (warp == LOAD_WARP && lane == 0) {
    // a CTA that stopped early still waits (bounded) for the loads it issued
    if (taken[0] < issued[0]) snb::mbar_wait_bounded(q_full, taken[0] & 1, status, SNB_ERR_TIMEOUT_TMA);
    for (int i = taken[1]; i < issued[1]; ++i)
      if (!snb::mbar_wait_bounded(&k_full[i % C::NK], (i / C::NK) & 1, status, SNB_ERR_TIMEOUT_TMA)) break;
    for (int i = taken[2]; i < issued[2]; ++i)
      if (!snb::mbar_wait_bounded(&v_full[i % C::NV], (i / C::NV) & 1, status, SNB_ERR_TIMEOUT_TMA)) break;
  }
  if (warp == MMA_WARP) snb::tmem_dealloc(tmem, 512);
}

template <typename T, int D, int DV>
void launch(PromptParams p, int* status, cudaStream_t st) {
  using C = Cfg<D, DV>;
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const auto dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto map = [&](const void* base, int64_t width, int64_t stride, int rows = 128) {
    return snb_host::make_tmap_2d(base, dt, width, p.T, stride * 2, 64, rows, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  const CUtensorMap tq = map(p.q, (int64_t)p.heads * D, p.qs), tk = map(p.k, (int64_t)p.kv_heads * D, p.ks),
                    tv = map(p.v, (int64_t)p.kv_heads * DV, p.vs), tq32 = map(p.q, (int64_t)p.heads * D, p.qs, 32);
  p.idesc = bf16 ? 1u << 7 | 1u << 10 : 0u;
  p.pair_heads = (p.heads / p.kv_heads) % 2 == 0;
  p.pairs = p.pair_heads ? p.heads / 2 : p.heads;
  p.wide_out = reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.os % 16 == 0;
  const int rows = p.pair_heads ? BQ : 2 * BQ;
  const int64_t items = ((int64_t)p.T / rows + std::min(p.B, p.T)) * p.pairs;  // at most one ragged tile per prompt
  TORCH_CHECK(items < (int64_t(1) << 31), "prompt_attention: too much work for one call");
  p.items = (int)items;
  auto kern = prompt_attention_kernel<T, D, DV>;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  C10_CUDA_CHECK(snb::launch_pdl(kern, dim3(std::min(p.items, sms)), dim3(THREADS), C::SMEM, st, tq, tk, tv, tq32,
                                 p, status));
}

template <typename T>
void dispatch(const PromptParams& p, int64_t D, int64_t DV, int* status, cudaStream_t st) {
  if (D == 64 && DV == 64) launch<T, 64, 64>(p, status, st);
  else if (D == 128 && DV == 128) launch<T, 128, 128>(p, status, st);
  else if (D == 192 && DV == 128) launch<T, 192, 128>(p, status, st);
  else TORCH_CHECK(false, "prompt_attention: serves keys / values 64 / 64, 128 / 128 or 192 / 128 wide");
}

bool is_matrix(const at::Tensor& x, int64_t T, int64_t width, const at::Tensor& q) {
  return x.dim() == 2 && x.size(0) == T && x.size(1) == width && x.scalar_type() == q.scalar_type() &&
         x.device() == q.device();
}

}  // namespace

// q [T, heads * D], k [T, kv_heads * D], v [T, kv_heads * DV]: bf16 or fp16 (rows that are not contiguous, not on
// 16-byte boundaries or overlap are copied first); out [T, heads * DV] or none. indptr [B + 1] int32, ascending; rows
// outside every prompt are not written.
at::Tensor prompt_attention(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor indptr, int64_t heads,
                            int64_t kv_heads, int64_t D, int64_t DV, int64_t window, double sm_scale,
                            std::optional<at::Tensor> sinks, std::optional<at::Tensor> given, at::Tensor status) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 2, "prompt_attention: q must be a CUDA matrix");
  TORCH_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
              "prompt_attention: the heads do not divide over the KV heads");
  TORCH_CHECK(window >= 0 && sm_scale > 0,
              "prompt_attention: the window must be 0 (off) or more, sm_scale must be positive");
  const auto dt = q.scalar_type();
  TORCH_CHECK(dt == at::kBFloat16 || dt == at::kHalf, "prompt_attention: takes bf16 or fp16 on CUDA");
  const int64_t T = q.size(0), B = indptr.numel() - 1;
  TORCH_CHECK(is_matrix(q, T, heads * D, q), "prompt_attention: q must be [tokens, heads * head_dim]");
  TORCH_CHECK(is_matrix(k, T, kv_heads * D, q),
              "prompt_attention: k must be [tokens, KV heads * head_dim] of q's type and device");
  TORCH_CHECK(is_matrix(v, T, kv_heads * DV, q),
              "prompt_attention: v must be [tokens, KV heads * v_head_dim] of q's type and device");
  TORCH_CHECK(indptr.dim() == 1 && B >= 0 && indptr.scalar_type() == at::kInt && indptr.device() == q.device(),
              "prompt_attention: qo_indptr must be an int32 vector of prompt bounds on q's device");
  TORCH_CHECK(T < (int64_t(1) << 30), "prompt_attention: too many tokens");
  if (sinks)
    TORCH_CHECK(sinks->device() == q.device() && sinks->scalar_type() == at::kFloat && sinks->is_contiguous() &&
                    sinks->numel() == heads,
                "prompt_attention: sinks must be one fp32 value per head on q's device");
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = given ? *given : at::empty({T, heads * DV}, q.options());
  TORCH_CHECK(is_matrix(out, T, heads * DV, q),
              "prompt_attention: out must be [tokens, heads * v_head_dim] of q's type and device");
  // a single row's stride means nothing
  TORCH_CHECK(T == 0 || snb_host::is_mappable(T > 1 ? out : out.view({heads * DV}).unsqueeze(0)),
              "prompt_attention: out needs contiguous rows on 16-byte boundaries that do not overlap");
  if (T == 0 || B == 0) return out;
  q = snb_host::mappable(q);
  k = snb_host::mappable(k);
  v = snb_host::mappable(v);
  indptr = indptr.contiguous();
  PromptParams p;
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.out = out.data_ptr();
  p.qs = q.stride(0);
  p.ks = k.stride(0);
  p.vs = v.stride(0);
  p.os = T > 1 ? out.stride(0) : heads * DV;
  p.indptr = indptr.data_ptr<int>();
  p.sinks = sinks ? sinks->data_ptr<float>() : nullptr;
  p.T = (int)T;
  p.B = (int)B;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.window = (int)std::min<int64_t>(window, T);
  p.scale = (float)(sm_scale * 1.4426950408889634);
  auto st = at::cuda::getCurrentCUDAStream();
  if (dt == at::kBFloat16) dispatch<__nv_bfloat16>(p, D, DV, status.data_ptr<int>(), st);
  else dispatch<__half>(p, D, DV, status.data_ptr<int>(), st);
  return out;
}
