// One AdamW step over a list of tensors, moments in 32 or 8 bits (formulas and formats: bamboo_b200.h, bb_adamw_list).
//
// Memory bounds it: 16 bytes a parameter with moments in 8 bits, an fp32 master, a bf16 gradient and a bf16 working copy (28 in 32 bits).
// A warp works on one block of 256 values, eight per lane, which is also the unit of the 8-bit scales: a block's largest magnitude is a
// warp-wide maximum of bit patterns, under which NaN and infinity are the largest.  The list travels as a kernel argument.
//
// Codes are 6 to 12 % apart and one step changes a root by (1 - beta2) / 2 of itself, so codes rounded to nearest stand still from step to step (bamboo_b200.h).
// Codes rounded up or down at random keep the average: the conversion takes 16 random bits, two neighbouring values share them from either end, and they are
// hashed from seed, step, place and the parameter's new bits, so the same call gives the same codes.
#include "common.cuh"
#include "bamboo_b200.h"
#include <cuda_fp8.h>
#include <limits.h>
#include <math.h>
#include <algorithm>
#include <vector>

namespace {

int refuse(const char* msg) { bb_set_last_error_msg(msg); return BB_ERR_INVALID_ARG; }

constexpr int LIST = 64;                       // tensors of one launch
// Ten CTAs of four warps per SM: with moments in 8 bits a warp spends longer between its loads and its stores than in 32, and 48 registers let 40 of
// them cover that.  150 M parameters, bf16 gradients and working copies, us: 8 bits 367 (6.5 TB/s) with the nearest codes, 355 (6.8) with codes rounded at
// random, which four conversions make instead of eight; 32 bits 612 (6.9).  With eight CTAs 8 bits took 30 more, with twelve (which spill) 45.  Instructions are never
// far from memory's time here: at the clocks that a power cap leaves (1.3 GHz) 8 bits come to 5.5 TB/s.  Before, lanes with eight neighbouring values each, exact quotients and a tensor found by comparisons in all lanes (constant
// memory gives one address at a time): 498.
constexpr int BLOCK = 256, THREADS = 128, WARPS = THREADS / 32, CTAS = 10;
constexpr float TOP = 256.f, TINY = 0x1p-100f; // code of a block's largest value; scales up to TINY hold nothing
constexpr float CODE_MIN = 0x1p-9f;            // smallest e4m3 value above 0

struct AdamTable {
  bb_adamw_tensor t[LIST];
  int first[LIST + 1];                         // first block of each tensor
  unsigned char vec[LIST];                     // whether it lies on 16 bytes (codes: 8) everywhere
  int count;
};
// (lr is folded into the rest: p -= rate m / (root sqrt(v) + eps) + shrink p, rate = lr / (1 - beta1^step), root = 1 / sqrt(1 - beta2^step))
struct AdamArgs { float b1, omb1, b2, omb2, eps, rate, root, shrink, grad_scale; int zero_grad; const float* coef; uint32_t key; };
enum { BITS_32 = 0, NEAREST = 1, STOCHASTIC = 2 };           // moments in 32 bits, in 8 bits with the nearest codes, with codes rounded up or down at random

// One instruction each, within 2^-22 of the value; subnormal arguments count.  The update that they make is of the order of lr.
__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float over(float v) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float2 code_pair(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t pair_code(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }

// Multiplicative hashing, twice (odd multipliers: the golden ratio's and the square root of two's first 32 bits)
__host__ __device__ __forceinline__ uint32_t hashed(uint32_t x) {
  x ^= x >> 16; x *= 0x9e3779b9u;
  x ^= x >> 15; x *= 0xb504f333u;
  return x ^ (x >> 16);
}
// One more product each, with other odd numbers, makes several words of a hash
__device__ __forceinline__ uint32_t word(uint32_t hash, uint32_t odd) {
  const uint32_t w = hash * odd;
  return w ^ (w >> 16);
}
// Codes of a, b, c, d (in the bytes from the lowest), each the neighbour above or below with the probability that makes its mean the value, in steps of 2^-16
__device__ __forceinline__ uint32_t stochastic_codes(float a, float b, float c, float d, uint32_t random) {
  uint32_t q;
  asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;" : "=r"(q) : "f"(d), "f"(c), "f"(b), "f"(a), "r"(random));
  return q;
}

// Codes of a lane's eight values under the block's scale, which every lane receives; ROOT: see CODE_MIN.  Rounded at random, the largest value is put at 256 and
// a little more, where it cannot become the code below.
template <bool ROOT, int KIND> __device__ __forceinline__ uint2 encode(const float* v, float& scale, uint32_t random0, uint32_t random1) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  scale = __uint_as_float(top);
  if (top >= 0x7f800000u) { scale = __uint_as_float(0x7fc00000u); return make_uint2(0, 0); }
  if (scale <= TINY) return make_uint2(0, 0);
  const float f = (KIND == STOCHASTIC ? TOP * (1.f + 0x1p-21f) : TOP) * over(scale);
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = v[i] * f;
    if (ROOT && v[i] > 0.f) c[i] = fmaxf(c[i], CODE_MIN);
  }
  if (KIND == STOCHASTIC) return make_uint2(stochastic_codes(c[0], c[1], c[2], c[3], random0), stochastic_codes(c[4], c[5], c[6], c[7], random1));
  return make_uint2(pair_code(c[0], c[1]) | pair_code(c[2], c[3]) << 16, pair_code(c[4], c[5]) | pair_code(c[6], c[7]) << 16);
}
__device__ __forceinline__ void decode(uint2 q, float scale, float* v) {
  const float2 f = make_float2(scale * (1.f / TOP), scale * (1.f / TOP));
  const uint32_t two[4] = {q.x & 0xffffu, q.x >> 16, q.y & 0xffffu, q.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 c = bb::mul2(code_pair(two[i]), f);
    v[2 * i] = c.x; v[2 * i + 1] = c.y;
  }
}

// A lane's values: four in each half of the block, so that a warp's access is one run of memory; at once where the block is whole and the tensors lie
// on 16 bytes, one by one elsewhere (value i is the block's (i / 4) 128 + 4 lane + i % 4, of which n are there)
constexpr int HALF = BLOCK / 2;
__device__ __forceinline__ int place(int lane, int i) { return (i >> 2) * HALF + 4 * lane + (i & 3); }

template <bool VEC> __device__ __forceinline__ void load8(const float* p, int lane, int n, float* v) {
  if (VEC) {
    const float4 a = reinterpret_cast<const float4*>(p)[lane], b = reinterpret_cast<const float4*>(p + HALF)[lane];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = place(lane, i) < n ? p[place(lane, i)] : 0.f;
  }
}
template <bool VEC> __device__ __forceinline__ void load8(const __nv_bfloat16* p, int lane, int n, float* v) {
  if (VEC) {
    const uint2 a = reinterpret_cast<const uint2*>(p)[lane], b = reinterpret_cast<const uint2*>(p + HALF)[lane];
    v[0] = bb::bf16_lo(a.x); v[1] = bb::bf16_hi(a.x); v[2] = bb::bf16_lo(a.y); v[3] = bb::bf16_hi(a.y);
    v[4] = bb::bf16_lo(b.x); v[5] = bb::bf16_hi(b.x); v[6] = bb::bf16_lo(b.y); v[7] = bb::bf16_hi(b.y);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = place(lane, i) < n ? __bfloat162float(p[place(lane, i)]) : 0.f;
  }
}
template <bool VEC> __device__ __forceinline__ void store8(float* p, int lane, int n, const float* v) {
  if (VEC) {
    reinterpret_cast<float4*>(p)[lane] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p + HALF)[lane] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (place(lane, i) < n) p[place(lane, i)] = v[i];
  }
}
template <bool VEC> __device__ __forceinline__ void store8(__nv_bfloat16* p, int lane, int n, const float* v) {
  if (VEC) {
    reinterpret_cast<uint2*>(p)[lane] = make_uint2(bb::pack_bf16x2(v[0], v[1]), bb::pack_bf16x2(v[2], v[3]));
    reinterpret_cast<uint2*>(p + HALF)[lane] = make_uint2(bb::pack_bf16x2(v[4], v[5]), bb::pack_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (place(lane, i) < n) p[place(lane, i)] = __float2bfloat16(v[i]);
  }
}
template <bool VEC> __device__ __forceinline__ uint2 load_codes(const uint8_t* p, int lane, int n) {
  uint2 q = make_uint2(0, 0);
  if (VEC) {
    q = make_uint2(reinterpret_cast<const uint32_t*>(p)[lane], reinterpret_cast<const uint32_t*>(p + HALF)[lane]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (place(lane, i) < n) (i < 4 ? q.x : q.y) |= (uint32_t)p[place(lane, i)] << (8 * (i & 3));
  }
  return q;
}
template <bool VEC> __device__ __forceinline__ void store_codes(uint8_t* p, int lane, int n, uint2 q) {
  if (VEC) {
    reinterpret_cast<uint32_t*>(p)[lane] = q.x;
    reinterpret_cast<uint32_t*>(p + HALF)[lane] = q.y;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (place(lane, i) < n) p[place(lane, i)] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}

template <int KIND, bool VEC>
__device__ __forceinline__ void block_step(const bb_adamw_tensor& t, long long at, long long block, int n, int lane, const AdamArgs& a, float gs) {
  constexpr bool EIGHT = KIND != BITS_32;
  float p[8], g[8], m[8], v[8], sm = 0.f, sv = 0.f;
  const long long blocks = (t.numel + BLOCK - 1) / BLOCK;
  float* master = t.master ? t.master : reinterpret_cast<float*>(t.param);
  if (EIGHT) { sm = t.scales[block]; sv = t.scales[blocks + block]; }
  load8<VEC>(master + at, lane, n, p);
  if (t.grad_dtype == BB_DTYPE_F32) load8<VEC>(reinterpret_cast<const float*>(t.grad) + at, lane, n, g);
  else load8<VEC>(reinterpret_cast<const __nv_bfloat16*>(t.grad) + at, lane, n, g);
  if (EIGHT) {
    decode(load_codes<VEC>(reinterpret_cast<const uint8_t*>(t.exp_avg) + at, lane, n), sm, m);
    decode(load_codes<VEC>(reinterpret_cast<const uint8_t*>(t.exp_avg_sq) + at, lane, n), sv, v);
  } else {
    load8<VEC>(reinterpret_cast<const float*>(t.exp_avg) + at, lane, n, m);
    load8<VEC>(reinterpret_cast<const float*>(t.exp_avg_sq) + at, lane, n, v);
  }
  const float2 b1 = make_float2(a.b1, a.b1), b2 = make_float2(a.b2, a.b2), gs1 = make_float2(gs * a.omb1, gs * a.omb1), gs2 = make_float2(gs, gs);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 x = make_float2(g[i], g[i + 1]), y = bb::mul2(x, gs2), old = make_float2(v[i], v[i + 1]);
    const float2 m2 = bb::fma2(b1, make_float2(m[i], m[i + 1]), bb::mul2(x, gs1));
    const float2 v2 = bb::fma2(b2, EIGHT ? bb::mul2(old, old) : old, bb::mul2(bb::mul2(y, make_float2(a.omb2, a.omb2)), y));
    const float2 r = make_float2(root_of(v2.x), root_of(v2.y));
    const float2 d = bb::fma2(r, make_float2(a.root, a.root), make_float2(a.eps, a.eps));
    const float2 u = bb::mul2(bb::mul2(m2, make_float2(-a.rate, -a.rate)), make_float2(over(d.x), over(d.y)));
    const float2 w = make_float2(p[i], p[i + 1]), q = bb::add2(w, bb::fma2(w, make_float2(-a.shrink, -a.shrink), u));
    m[i] = m2.x; m[i + 1] = m2.y;
    v[i] = EIGHT ? r.x : v2.x; v[i + 1] = EIGHT ? r.y : v2.y;
    p[i] = q.x; p[i + 1] = q.y;
  }
  store8<VEC>(master + at, lane, n, p);
  if (t.master) store8<VEC>(reinterpret_cast<__nv_bfloat16*>(t.param) + at, lane, n, p);
  if (a.zero_grad) {
    const float zeros[8] = {};
    if (t.grad_dtype == BB_DTYPE_F32) store8<VEC>(reinterpret_cast<float*>(t.grad) + at, lane, n, zeros);
    else store8<VEC>(reinterpret_cast<__nv_bfloat16*>(t.grad) + at, lane, n, zeros);
  }
  if (EIGHT) {
    if (!VEC) {                                // what a partial block has beyond its end decides nothing
#pragma unroll
      for (int i = 0; i < 8; ++i) if (place(lane, i) >= n) { m[i] = 0.f; v[i] = 0.f; }
    }
    uint32_t h = 0;
    if (KIND == STOCHASTIC) h = hashed(((uint32_t)block * 32 + lane) ^ (t.seed * 0x9e3779b9u + a.key) ^ __float_as_uint(p[0]));
    const uint2 cm = encode<false, KIND>(m, sm, h, word(h, 0xbb67ae85u)), cv = encode<true, KIND>(v, sv, word(h, 0xc6ef3721u), word(h, 0xa54ff53bu));
    store_codes<VEC>(reinterpret_cast<uint8_t*>(t.exp_avg) + at, lane, n, cm);
    store_codes<VEC>(reinterpret_cast<uint8_t*>(t.exp_avg_sq) + at, lane, n, cv);
    if (lane == 0) { t.scales[block] = sm; t.scales[blocks + block] = sv; }
  } else {
    store8<VEC>(reinterpret_cast<float*>(t.exp_avg) + at, lane, n, m);
    store8<VEC>(reinterpret_cast<float*>(t.exp_avg_sq) + at, lane, n, v);
  }
}

template <int KIND>
__global__ void __launch_bounds__(THREADS, CTAS)
adamw_list_kernel(const __grid_constant__ AdamTable table, const AdamArgs a) {
  bb::pdl_sync();
  const int lane = threadIdx.x & 31;
  const int unit = (gridDim.x - 1 - blockIdx.x) * WARPS + bb::warp_index();         // last ones first: the norm read them last
  if (unit >= table.first[table.count]) return;
  int lo = 0;
#pragma unroll
  for (int step = LIST / 2; step; step >>= 1) if (table.first[lo + step] <= unit) lo += step;
  const bb_adamw_tensor& t = table.t[lo];
  const long long block = unit - table.first[lo], at = block * BLOCK, left = t.numel - at;
  const float gs = a.coef ? a.coef[0] * a.grad_scale : a.grad_scale;
  if (table.vec[lo] && left >= BLOCK) block_step<KIND, true>(t, at, block, BLOCK, lane, a, gs);
  else block_step<KIND, false>(t, at, block, left < BLOCK ? (int)left : BLOCK, lane, a, gs);
}

bool bad_tensor(const bb_adamw_tensor& t, bool eight) {
  return !t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || t.numel <= 0 || t.numel > (1LL << 38) || (eight != (t.scales != nullptr)) ||
         (t.grad_dtype != BB_DTYPE_BF16 && t.grad_dtype != BB_DTYPE_F32) || ((uintptr_t)t.grad & (t.grad_dtype == BB_DTYPE_F32 ? 3 : 1)) ||
         ((uintptr_t)t.param & (t.master ? 1 : 3)) || (((uintptr_t)t.master | (uintptr_t)t.scales) & 3) ||
         (!eight && (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 3));
}
bool aligned(const bb_adamw_tensor& t, bool eight) {
  return (((uintptr_t)t.param | (uintptr_t)t.master | (uintptr_t)t.grad) & 15) == 0 &&
         (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & (eight ? 7 : 15)) == 0;
}
struct Range { uintptr_t from, to; bool written; };
}  // namespace

extern "C" int bb_adamw_list_overlaps(const bb_adamw_tensor* tensors, int count, int zero_grad) {
  if (!tensors || count <= 0) return 0;
  try {
    static thread_local std::vector<Range> all;          // (52 tensors are looked through in 4 us)
    all.clear();
    auto add = [&](const void* at, long long bytes, bool written) { if (at && bytes > 0) all.push_back({(uintptr_t)at, (uintptr_t)at + (uintptr_t)bytes, written}); };
    for (int i = 0; i < count; ++i) {
      const bb_adamw_tensor& t = tensors[i];
      const long long n = t.numel, moment = t.scales ? n : 4 * n;
      add(t.param, t.master ? 2 * n : 4 * n, true);
      add(t.master, 4 * n, true);
      add(t.grad, t.grad_dtype == BB_DTYPE_F32 ? 4 * n : 2 * n, zero_grad != 0);
      add(t.exp_avg, moment, true);
      add(t.exp_avg_sq, moment, true);
      add(t.scales, 8 * ((n + BLOCK - 1) / BLOCK), true);
    }
    std::sort(all.begin(), all.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t written = 0, read = 0;                     // where those in front end
    for (const Range& r : all) {
      if (r.from < written || (r.written && r.from < read)) return 1;
      (r.written ? written : read) = std::max(r.written ? written : read, r.to);
    }
    return 0;
  } catch (...) {
    bb_set_last_error_msg("bb_adamw_list_overlaps: out of memory");
    return 1;
  }
}

extern "C" int bb_adamw_list(const bb_adamw_tensor* tensors, int count, double lr, double beta1, double beta2, double eps, long long step,
                             double weight_decay, double grad_scale, int zero_grad, double max_norm, const double* sumsq, float* norm, void* workspace,
                             long long workspace_bytes, void* stream) {
  if (!tensors || count <= 0 || step < 1 || !(max_norm >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0) ||
      (max_norm > 0.0 && (!norm || !workspace || ((uintptr_t)workspace & 7) || workspace_bytes < bb_grad_norm_workspace_bytes())))
    return refuse("bb_adamw_list: an empty list, step < 1, a beta outside [0, 1), a negative norm, or clipping without a place for the norm or with a workspace that is too small");
  const bool eight = tensors[0].scales != nullptr, at_random = eight && tensors[0].seed != 0;
  for (int i = 0; i < count; ++i)
    if (bad_tensor(tensors[i], eight) || at_random != (eight && tensors[i].seed != 0))
      return refuse("bb_adamw_list: a null or misaligned pointer, an empty tensor, a gradient that is neither bf16 nor fp32, or scales or seeds for a part of the list only");
  cudaStream_t s = (cudaStream_t)stream;
  AdamArgs a;
  a.b1 = (float)beta1; a.omb1 = (float)(1.0 - beta1); a.b2 = (float)beta2; a.omb2 = (float)(1.0 - beta2); a.eps = (float)eps;
  a.rate = (float)(lr / (1.0 - pow(beta1, (double)step))); a.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  a.shrink = (float)(lr * weight_decay); a.grad_scale = (float)grad_scale; a.zero_grad = zero_grad; a.coef = nullptr;
  a.key = hashed((uint32_t)step ^ hashed((uint32_t)(step >> 32) + 1));
  BackToBack overlap;
  if (max_norm > 0.0) {
    if (int rc = bb_list_clip_coef(tensors, count, sumsq, grad_scale, max_norm, norm, workspace, s)) return rc;
    a.coef = (const float*)((double*)workspace + 1);
  }
  for (int from = 0; from < count;) {
    AdamTable t;
    long long blocks = 0;
    int n = 0;
    for (; n < LIST && from + n < count; ++n) {
      const long long more = (tensors[from + n].numel + BLOCK - 1) / BLOCK;
      if (blocks + more > INT_MAX - 64) break;          // (a launch's blocks are counted in an int; one tensor's always are)
      t.t[n] = tensors[from + n];
      t.vec[n] = aligned(t.t[n], eight) ? 1 : 0;
      t.first[n] = (int)blocks;
      blocks += more;
    }
    t.count = n;
    t.first[n] = (int)blocks;
    for (int i = n + 1; i <= LIST; ++i) t.first[i] = INT_MAX;
    BB_CUDA_CHECK(bb_launch(!eight ? adamw_list_kernel<BITS_32> : at_random ? adamw_list_kernel<STOCHASTIC> : adamw_list_kernel<NEAREST>, dim3((unsigned)((blocks + WARPS - 1) / WARPS)), THREADS, 0, s, t, a));
    from += n;
  }
  return BB_OK;
}
