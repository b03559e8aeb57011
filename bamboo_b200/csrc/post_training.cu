// Post-training of the vocabulary models: log-probabilities of given tokens with their gradient, the paired preference loss, the
// clipped policy loss with a KL term, the global gradient norm over a list of tensors, clipping, and the Adam step that clips.
// Softmax sums as in softmax2.cuh.
#include "softmax2.cuh"
#include <atomic>
#include <limits.h>
#include <math.h>
#include <stdio.h>

namespace {

// 16-byte loads that a thread has in flight (GRAD_LOADS: in a gradient by 256 threads).  8192 rows of 50257 bf16 logits, a sixteenth of them
// ignored: sums 120 us with four (6.4 TB/s), gradient by 256 threads 249 us with four, 246 with eight and two thirds of the threads per SM, 252
// with two; by 512 with four 242 (6.6 TB/s).
constexpr int ROW_LOADS = 4, GRAD_LOADS = 8;
constexpr int MAX_PARTS = 8;              // CTAs of a cluster that share a row
// How many threads share a row: with its bytes a thread's loads, barriers and start are spread over more of them, and with few rows
// more of them are needed to fill the machine (TEAM_THREADS; 148 SMs hold 303104).  us, bf16, per row a warp | 64 | 128 | 256 threads:
//   sums      16384 rows of 8 KB 29 | 29 | 38 | 64, of 16 KB 52 | 49 | 50 | 73, of 49 KB 137 | 128 | 122 | 140;  1024 of 16 KB 17 | 9 | 7 | 9
//   gradient  16384 rows of 4 KB 28 | 32 | 44 | 76, of 16 KB 91 | 88 | 92 | 111, of 32 KB 176 | 173 | 165 | 176;  1024 of 16 KB 11 | 8 | 7 | 8
//   policy    16384 rows of 4 KB 41 | 44 | 61 | 86, of 12 KB 94 | 81 | 92 | 123, of 24 KB 187 | 178 | 145 | 172;  1024 of 16 KB 21 | 18 | 15 | 19
// (fp32 within 10 % of the same ratios.)
constexpr size_t TINY_ROW = 1024;
constexpr long long TEAM_THREADS = 131072;
struct Teams { size_t warp, two, four; };
constexpr Teams SUM_TEAMS = {8192, 16384, 65536}, GRAD_TEAMS = {4096, 16384, 40960}, POLICY_TEAMS = {4096, 12288, 32768};
// Gradients of many long rows: 512 threads with four loads instead of 256 with eight (bf16, us: 16384 rows of 65 KB 330 | 328, of 98 KB 490 | 499, of 196 KB
// 1009 | 1026; 2048 of 98 KB 67 | 70; 512 of 98 KB 23.5 | 21.7).
constexpr size_t GRAD_EIGHT = 81920;
constexpr int GRAD_EIGHT_ROWS = 2048;
// From here on the policy loss keeps a row in shared memory instead of reading it twice (16384 rows, us, twice | kept: bf16 of 38 KB 238 | 285, of
// 49 KB 284 | 334, of 63 KB 373 | 383; fp32 of 32 KB 204 | 232, of 38 KB 253 | 248, of 49 KB 313 | 289).
template <typename T> constexpr size_t LONG_ROW = sizeof(T) == 2 ? 65536 : 32768;
int team_of(size_t bytes, long long rows, const Teams& by) {
  if (bytes <= TINY_ROW) return 32;
  int threads = bytes <= by.warp ? 32 : bytes <= by.two ? 64 : bytes <= by.four ? 128 : 256;
  while (threads < 256 && threads * rows < TEAM_THREADS) threads *= 2;
  return threads;
}

// dynamic shared memory next to a kernel's few static bytes: of one CTA per SM, and of each of two
constexpr size_t MAX_RING = 226 * 1024, PAIR_RING = 112 * 1024;

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& q, float* f) {
    f[0] = bb::bf16_lo(q.x); f[1] = bb::bf16_hi(q.x); f[2] = bb::bf16_lo(q.y); f[3] = bb::bf16_hi(q.y);
    f[4] = bb::bf16_lo(q.z); f[5] = bb::bf16_hi(q.z); f[6] = bb::bf16_lo(q.w); f[7] = bb::bf16_hi(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(bb::pack_bf16x2(f[0], f[1]), bb::pack_bf16x2(f[2], f[3]), bb::pack_bf16x2(f[4], f[5]), bb::pack_bf16x2(f[6], f[7]));
  }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }   // -inf
};
template <> struct Elem<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint4& q, float* f) {
    f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y); f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u); }
};

using bb::expo;
using bb::expo2;
using bb::ex2;
using bb::row_logp;
using bb::soft_add;
using bb::soft_merge;

// A row of n elements as [0, lead) up to the first 16-byte boundary, nvec vectors, and the rest from `tail`.
template <typename T> struct Span {
  int lead, nvec, tail;
  __device__ __forceinline__ Span(const T* p, int n) {
    const int off = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
    lead = off < n ? off : n;
    nvec = (n - lead) / Elem<T>::VEC;
    tail = lead + nvec * Elem<T>::VEC;
  }
};

// A row is worked on by a block, by its first THREADS threads (a warp more feeds them), or (THREADS = 32) by a warp of its own
template <int THREADS> __device__ __forceinline__ int row_thread() { return THREADS == 32 ? (int)(threadIdx.x & 31) : (int)threadIdx.x; }
template <int THREADS> constexpr int ROWS_OF_BLOCK = THREADS == 32 ? 8 : 1;
template <int THREADS> constexpr int BLOCK = THREADS == 32 ? 256 : THREADS;

// (r, s) of a warp's lanes merged: the largest reference first, one scaling, then plain sums
__device__ __forceinline__ void soft_warp(float& r, float& s) {
  float top = r;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (r != top) s *= ex2(r - top);             // (-inf - -inf would be NaN)
  r = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
}
// Barrier of the block's first THREADS threads: the whole block, or all but a warp that feeds the others
template <int THREADS, bool FED = false> __device__ __forceinline__ void row_barrier() {
  if constexpr (FED) asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
  else __syncthreads();
}
// The same for a block that is fed; whether `v` holds in any of those threads, the same answer for all of them
template <int THREADS> __device__ __forceinline__ bool row_barrier_any(bool v) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred P, Q;\n\tsetp.ne.u32 P, %1, 0;\n\tbar.red.or.pred Q, 1, %2, P;\n\tselp.u32 %0, 1, 0, Q;\n\t}"
               : "=r"(any) : "r"((uint32_t)v), "n"(THREADS) : "memory");
  return any != 0;
}
// (r, s) of the block's threads merged; the first warp gets the result
template <int THREADS, bool FED = false> __device__ __forceinline__ void soft_block(float& r, float& s, float2* smem /*[THREADS/32]*/) {
  soft_warp(r, s);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = make_float2(r, s);
  row_barrier<THREADS, FED>();
  if (threadIdx.x < 32) {
    const float2 q = threadIdx.x < THREADS / 32 ? smem[threadIdx.x] : make_float2(-INFINITY, 0.f);
    r = q.x; s = q.y;
    soft_warp(r, s);
  }
}

// This thread's share of a row, chunk by chunk with the reference kept below the largest logit (the exact form)
template <typename T, int THREADS> __device__ __noinline__ float2 soft_share_exact(const uint4* v, int nvec, K2 k) {
  constexpr int VEC = Elem<T>::VEC;
  float r = -INFINITY, s = 0.f;
  for (int c = row_thread<THREADS>(); c < nvec; c += THREADS) {
    float f[VEC];
    Elem<T>::unpack(v[c], f);
    soft_add<VEC>(r, s, f, k, -bb::SOFT_FAR);
  }
  return make_float2(r, s);
}

// VEC logits added to sums whose reference stays (see soft_share)
template <int VEC> __device__ __forceinline__ void soft_chunk(float2& sum, const float* f, K2 k, float r) {
#pragma unroll
  for (int i = 0; i < VEC; i += 2) {
    const float2 t = expo2(make_float2(f[i], f[i + 1]), k, r);
    sum = bb::add2(sum, make_float2(ex2(t.x), ex2(t.y)));
  }
}
// the elements of a row in front of its first 16-byte boundary and behind its last
template <typename T, int THREADS> __device__ __forceinline__ void soft_edges(const T* x, const Span<T>& sp, int n, K2 k, float& r, float& s) {
  for (int j = row_thread<THREADS>(); j < sp.lead + n - sp.tail; j += THREADS) {
    const float f = Elem<T>::get(x + (j < sp.lead ? j : sp.tail + j - sp.lead));
    soft_add<1>(r, s, &f, k, -bb::SOFT_FAR);
  }
}

// (r, s) of this thread's share of a row's chunks.  The reference comes from the thread's first chunk and stays: a later logit may be larger,
// 2^(k x - r) is a float all the same, so the loop needs no maximum; a share whose sum reaches SHARE_MOST (above a first
// chunk that is masked, for one) is taken (again) in the exact form.  That bound keeps what the merges make of the shares: 8 x 512 of them add up to less than 2^76, far from
// overflow; a share that a difference of 127 between references flushes to zero was below 2^-63 of the sum; and 1 / s is no denormal
// number.  A share that is taken again comes from L2: 8192 bf16 rows of 50257 at temperatures of 1 and 0.2 125 us, at 0.1 and below 235 (randn x 2;
// nearly every share).  U loads are in flight per thread.
constexpr float SHARE_MOST = 0x1p64f;
template <typename T, int THREADS, int U>
__device__ __forceinline__ void soft_share(const uint4* v, int nvec, K2 k, float& r, float& s) {
  constexpr int VEC = Elem<T>::VEC;
  r = -INFINITY; s = 0.f;
  int c = row_thread<THREADS>();
  float2 sum = make_float2(0.f, 0.f);
  float f[VEC];
  if (c < nvec) {
    Elem<T>::unpack(v[c], f);
    soft_add<VEC>(r, s, f, k, -bb::SOFT_FAR);
    c += THREADS;
  }
  for (; c + (U - 1) * THREADS < nvec; c += U * THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = v[c + u * THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) { Elem<T>::unpack(q[u], f); soft_chunk<VEC>(sum, f, k, r); }
  }
  if (c < nvec) {             // up to U - 1 more
    uint4 q[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u) q[u] = c + u * THREADS < nvec ? v[c + u * THREADS] : Elem<T>::nothing();
#pragma unroll
    for (int u = 0; u < U - 1; ++u) { Elem<T>::unpack(q[u], f); soft_chunk<VEC>(sum, f, k, r); }
  }
  s += sum.x + sum.y;
  if (!(s < SHARE_MOST)) { const float2 e = soft_share_exact<T, THREADS>(v, nvec, k); r = e.x; s = e.y; }
}

// A row whose largest logit is so far from zero that integer references are too coarse (a row masked whole by a large negative value): kept as
// (largest, -sum of 2^(k (x - largest))), so that what is rounded is a difference; (NaN, NaN) with a NaN or +inf in the row, (-inf, 0)
// when every logit is -inf.  Called by the first warp.
template <typename T> __device__ __noinline__ float2 soft_row_far(const T* x, int n, K2 k) {
  float top = -INFINITY;
  int bad = 0;
  for (int j = threadIdx.x & 31; j < n; j += 32) {
    const float f = Elem<T>::get(x + j);
    bad |= f != f || f == INFINITY;
    top = fmaxf(top, f);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (__any_sync(0xffffffffu, bad)) return make_float2(NAN, NAN);
  if (top == -INFINITY) return make_float2(top, 0.f);
  float sum = 0.f;
  for (int j = threadIdx.x & 31; j < n; j += 32) sum += ex2(bb::expo_gap(Elem<T>::get(x + j) - top, k));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return make_float2(top, -sum);
}

__device__ __forceinline__ bool soft_far(float r) { return fabsf(r) >= bb::SOFT_FAR; }

// The row's (r, s), in the row's first warp
template <typename T, int THREADS, int U>
__device__ __forceinline__ void soft_whole_row(const T* x, int n, K2 k, float& r, float& s, float2* smem) {
  const Span<T> sp(x, n);
  soft_share<T, THREADS, U>(reinterpret_cast<const uint4*>(x + sp.lead), sp.nvec, k, r, s);
  soft_edges<T, THREADS>(x, sp, n, k, r, s);
  if constexpr (THREADS == 32) soft_warp(r, s);
  else soft_block<THREADS>(r, s, smem);
  if (row_thread<THREADS>() < 32 && soft_far(r)) { const float2 e = soft_row_far(x, n, k); r = e.x; s = e.y; }
}

// -g softmax_j = ng 2^(k x_j - r).  Here k rounded to 32 bits will do: with what the rounding took at the largest logit (about r / k) in
// the factor, an entry is off by 1.3e-8 of its distance from the largest, in units of the exponent.
struct GradRow { float k, r, ng; };
__device__ __forceinline__ GradRow grad_factors(float g, K2 k, float r, float s) {
  const float k1 = k.hi + k.lo;
  return {k1, r, -g / s * ex2(((k.hi - k1) + k.lo) * (r / k1))};
}
// The target's entry, g (1 - softmax_t): with the arithmetic of the sum, so that nothing is left of a certain target
__device__ __forceinline__ float grad_target(float g, float xt, K2 k, float r, float s) { return fmaf(-g / s, ex2(expo(xt, k, r)), g); }
__device__ __forceinline__ float grad_entry(const GradRow& w, float x) { return w.ng * ex2(fmaf(x, w.k, -w.r)); }
template <typename T> __device__ __forceinline__ void grad_chunk(uint4* d, const uint4& q, const GradRow& w) {
  constexpr int VEC = Elem<T>::VEC;
  float f[VEC];
  Elem<T>::unpack(q, f);
#pragma unroll
  for (int i = 0; i < VEC; i += 2) {
    const float2 e = bb::fma2(make_float2(f[i], f[i + 1]), make_float2(w.k, w.k), make_float2(-w.r, -w.r));
    const float2 m = bb::mul2(make_float2(ex2(e.x), ex2(e.y)), make_float2(w.ng, w.ng));
    f[i] = m.x; f[i + 1] = m.y;
  }
  *d = Elem<T>::pack(f);
}
// What follows the chunks [0, whole): the target's entry (xt its logit, read before d, which may be x, was written; by the thread
// that wrote its chunk), the chunk that the padding begins in, the padding, and the elements around the 16-byte boundaries
template <typename T, int THREADS>
__device__ __forceinline__ void grad_rest(const T* x, float xt, T* d, int lead, int whole, int V, int cols, int t, float g, K2 k, float s, const GradRow& w) {
  constexpr int VEC = Elem<T>::VEC;
  if (t >= lead) {
    const int tc = (t - lead) / VEC;
    if (tc < whole && tc % THREADS == row_thread<THREADS>()) Elem<T>::put(d + t, grad_target(g, xt, k, w.r, s));
  }
  auto one = [&](int j) {
    float v = 0.f;
    if (j < V) { const float f = Elem<T>::get(x + j); v = j == t ? grad_target(g, f, k, w.r, s) : grad_entry(w, f); }
    Elem<T>::put(d + j, v);
  };
  const int nvec = (cols - lead) / VEC, tail = lead + nvec * VEC;
  for (int c = whole + row_thread<THREADS>(); c < nvec; c += THREADS) {
    const int j0 = lead + c * VEC;
    if (j0 >= V) *reinterpret_cast<uint4*>(d + j0) = make_uint4(0, 0, 0, 0);
    else for (int i = 0; i < VEC; ++i) one(j0 + i);
  }
  for (int j = row_thread<THREADS>(); j < lead + cols - tail; j += THREADS) one(j < lead ? j : tail + j - lead);
}

// Rows element by element: those kept by differences, gradients of another alignment than the logits', and vocabularies of less than a vector, which
// may end before the first boundary
template <typename T, int THREADS>
__device__ __noinline__ void grad_row_slow(const T* x, T* d, int V, int cols, int t, float g, K2 k, float r, float s) {
  const GradRow w = grad_factors(g, k, s < 0.f ? 0.f : r, s);
  for (int j = row_thread<THREADS>(); j < cols; j += THREADS) {
    float v = 0.f;
    if (j < V) {
      const float f = Elem<T>::get(x + j);
      if (s < 0.f) v = fmaf(g / s, ex2(bb::expo_gap(f - r, k)), j == t ? g : 0.f);
      else v = j == t ? grad_target(g, f, k, r, s) : grad_entry(w, f);
    }
    Elem<T>::put(d + j, v);
  }
}

// d[j] = g * ([j == t] - softmax_j) for j < V, 0 in [V, cols); zeros throughout when g == 0 (nothing is read then).  FAR: the row comes
// from memory, not from a cache that has just seen it
template <typename T, int THREADS, int U, bool FAR = false>
__device__ __forceinline__ void grad_row(const T* x, T* d, int V, int cols, int t, float g, K2 k, float r, float s) {
  constexpr int VEC = Elem<T>::VEC;
  const int tid = row_thread<THREADS>();
  if (s == 0.f) g = 0.f;
  if (g == 0.f) {
    const Span<T> sp(d, cols);
    uint4* dv = reinterpret_cast<uint4*>(d + sp.lead);
    for (int c = tid; c < sp.nvec; c += THREADS) dv[c] = make_uint4(0, 0, 0, 0);
    for (int j = tid; j < sp.lead + cols - sp.tail; j += THREADS) Elem<T>::put(d + (j < sp.lead ? j : sp.tail + j - sp.lead), 0.f);
    return;
  }
  if (s < 0.f || V < VEC || (((uintptr_t)x ^ (uintptr_t)d) & 15) != 0) {
    grad_row_slow<T, THREADS>(x, d, V, cols, t, g, k, r, s);
    return;
  }
  const GradRow w = grad_factors(g, k, r, s);
  const Span<T> sp(x, V);
  const uint4* xv = reinterpret_cast<const uint4*>(x + sp.lead);
  uint4* dv = reinterpret_cast<uint4*>(d + sp.lead);
  const int whole = sp.nvec;                            // chunks of vocabulary entries only
  const float xt = t >= sp.lead && (t - sp.lead) / VEC % THREADS == tid ? Elem<T>::get(x + t) : 0.f;
  int c = tid;
  for (; c + (U - 1) * THREADS < whole; c += U * THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = xv[c + u * THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) grad_chunk<T>(dv + c + u * THREADS, q[u], w);
  }
  if constexpr (FAR) {        // up to U - 1 more, their loads together as well
    uint4 q[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u) if (c + u * THREADS < whole) q[u] = xv[c + u * THREADS];
#pragma unroll
    for (int u = 0; u < U - 1; ++u) if (c + u * THREADS < whole) grad_chunk<T>(dv + c + u * THREADS, q[u], w);
  } else {
    for (; c < whole; c += THREADS) grad_chunk<T>(dv + c, xv[c], w);
  }
  grad_rest<T, THREADS>(x, xt, d, sp.lead, whole, V, cols, t, g, k, s, w);
}

// ------------------------------------------------------------------ sums of a block
template <int THREADS> __device__ __forceinline__ double block_sum(double v, double* smem /*[THREADS/32]*/) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v += smem[w];
  return v;
}

// The same for N values at once; every thread gets the sums
template <int THREADS, int N> __device__ __forceinline__ void block_sums(double* v, double (*smem)[N] /*[THREADS/32]*/) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) smem[threadIdx.x >> 5][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) v[i] += smem[w][i];
  }
}

// loss = mean of pair_loss, in a fixed order; by a block
template <int THREADS> __device__ __forceinline__ void mean_of(const double* pair_loss, int pairs, float* loss) {
  __shared__ double smem[THREADS / 32];
  double sum = 0.0;
  for (int i = threadIdx.x; i < pairs; i += THREADS) sum += pair_loss[i];
  sum = block_sum<THREADS>(sum, smem);
  if (threadIdx.x == 0) loss[0] = (float)(sum / pairs);
}

// ------------------------------------------------------------------ token log-probabilities
// A log-probability, and in `rest` what its rounding to 32 bits leaves out (rms 2.8e-7 for values between 8 and 16): the rewards are
// differences of log-probabilities that agree in most bits where a policy is near its reference, and that rounding would be most of
// their error.
__device__ inline void put_logp(double lp, int row, float* logp, float* rest) {
  logp[row] = (float)lp;
  if (rest) rest[row] = isinf(lp) ? 0.f : (float)(lp - (double)(float)lp);
}

// Registers for a full SM (32 a thread): bf16 sums with 34 take 5 to 25 % longer (2048 rows of 32 KB 17.8 us, with 32 14.5).  fp32 rows of
// a warp have 32 unasked, and lose 12 % when asked.
template <typename T, int THREADS> constexpr int SUM_BLOCKS = THREADS == 32 && sizeof(T) == 4 ? 0 : 2048 / BLOCK<THREADS>;
template <typename T, int THREADS>
__global__ void __launch_bounds__(BLOCK<THREADS>, SUM_BLOCKS<T, THREADS>)
token_logprob_fwd_kernel(const T* logits, long long ld, const long long* targets, K2 k, float* logp, float* rest, float2* stats,
                         int rows, int V, long long ignore_index, int* status) {
  __shared__ float2 smem[BLOCK<THREADS> / 32];
  bb::pdl_sync();
  const int row = THREADS == 32 ? (int)blockIdx.x * ROWS_OF_BLOCK<THREADS> + (int)(threadIdx.x >> 5) : (int)blockIdx.x;
  if (row >= rows) return;
  const long long t = targets[row];
  if (t == ignore_index || t < 0 || t >= V) {
    if (row_thread<THREADS>() == 0) {
      if (t != ignore_index) atomicCAS(status, 0, BB_ERR_INVALID_ARG);
      put_logp(0.0, row, logp, rest);
      if (stats) stats[row] = make_float2(0.f, 0.f);
    }
    return;
  }
  const T* x = logits + (size_t)row * ld;
  float r, s;
  const float xt = row_thread<THREADS>() == 0 ? Elem<T>::get(x + t) : 0.f;
  soft_whole_row<T, THREADS, ROW_LOADS>(x, V, k, r, s, smem);
  if (row_thread<THREADS>() == 0) {
    put_logp(row_logp(xt, k, r, s), row, logp, rest);
    if (stats) stats[row] = make_float2(r, s);
  }
}

// Few rows: a cluster per row, the chunks dealt out in equal parts; the parts' sums meet in the first CTA.  Three rows of 50257 fp32
// logits in a graph 4.5 us (6.6 by a CTA per row).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
token_logprob_fwd_cluster_kernel(const T* logits, long long ld, const long long* targets, K2 k, float* logp, float* rest, float2* stats, int V, long long ignore_index,
                                 int* status) {
  __shared__ float2 smem[THREADS / 32];
  __shared__ float2 parts[MAX_PARTS];
  bb::cluster_arrive_relaxed();           // waited for in front of the stores to the first CTA; a part's way through memory is longer
  bb::pdl_sync();
  const int rank = (int)bb::cluster_ctarank(), size = (int)bb::cluster_nctarank(), row = blockIdx.x / size;
  const long long t = targets[row];
  const bool counted = t != ignore_index && t >= 0 && t < V;
  const T* x = logits + (size_t)row * ld;
  float r = -INFINITY, s = 0.f;
  float xt = 0.f;
  if (counted) {
    if (rank == 0 && threadIdx.x == 0) xt = Elem<T>::get(x + t);
    const Span<T> sp(x, V);
    const int per = (sp.nvec + size - 1) / size, first = rank * per, mine = first < sp.nvec ? min(per, sp.nvec - first) : 0;
    soft_share<T, THREADS, ROW_LOADS>(reinterpret_cast<const uint4*>(x + sp.lead) + first, mine, k, r, s);
    if (rank == 0) soft_edges<T, THREADS>(x, sp, V, k, r, s);
    soft_block<THREADS>(r, s, smem);
  }
  __syncwarp();
  bb::cluster_wait();
  if (counted && threadIdx.x == 0) {
    const uint32_t at = bb::mapa_shared(bb::smem_u32(&parts[rank]), 0);
    bb::st_shared_cluster_u32(at, __float_as_uint(r));
    bb::st_shared_cluster_u32(at + 4, __float_as_uint(s));
  }
  __syncwarp();
  bb::cluster_sync();
  if (rank != 0 || threadIdx.x >= 32) return;
  if (!counted) {
    if (threadIdx.x == 0) {
      if (t != ignore_index) atomicCAS(status, 0, BB_ERR_INVALID_ARG);
      put_logp(0.0, row, logp, rest);
      if (stats) stats[row] = make_float2(0.f, 0.f);
    }
    return;
  }
  const float2 q = (int)threadIdx.x < size ? parts[threadIdx.x] : make_float2(-INFINITY, 0.f);
  r = q.x; s = q.y;
  soft_warp(r, s);
  if (soft_far(r)) { const float2 e = soft_row_far(x, V, k); r = e.x; s = e.y; }
  if (threadIdx.x == 0) {
    put_logp(row_logp(xt, k, r, s), row, logp, rest);
    if (stats) stats[row] = make_float2(r, s);
  }
}

// Threads of an SM that the registers leave room for: short rows gain from more of them (16384 bf16 rows of 16 KB 92 us with 1024, 84 with
// 1536), long ones from the loads that they would hold in registers instead.
template <int THREADS> constexpr int GRAD_BLOCKS = (THREADS == 256 ? 1024 : THREADS == 128 ? 1280 : 1536) / BLOCK<THREADS>;
template <typename T, int THREADS>
__global__ void __launch_bounds__(BLOCK<THREADS>, GRAD_BLOCKS<THREADS>)
token_logprob_bwd_kernel(const T* logits, long long ld, const long long* targets, const float2* stats, const float* row_grad,
                         const float* gscale_dev, float gscale, K2 k, T* dlogits, long long ldd, int rows, int V, int cols,
                         long long ignore_index, const double* pair_loss, int pairs, float* loss) {
  bb::pdl_sync();
  if (pair_loss && blockIdx.x == 0) mean_of<BLOCK<THREADS>>(pair_loss, pairs, loss);     // (the preference loss: one launch less)
  const int block = gridDim.x - 1 - blockIdx.x;     // the rows that the forward pass read last may still be in L2
  const int row = THREADS == 32 ? block * ROWS_OF_BLOCK<THREADS> + (int)(threadIdx.x >> 5) : block;
  if (row >= rows) return;
  const long long t = targets[row];
  const float2 st = stats[row];
  const bool counted = t != ignore_index && t >= 0 && t < V;
  const float g = counted ? row_grad[row] * (gscale_dev ? gscale_dev[0] : 1.f) * gscale : 0.f;
  grad_row<T, THREADS, THREADS == 256 ? GRAD_LOADS : ROW_LOADS, true>(logits + (size_t)row * ld, dlogits + (size_t)row * ldd, V, cols, (int)t, g, k, st.x, st.y);
}

// Tokens [a, b) of sequence q: rows of `seq_len` tokens, or between two offsets.  Offsets that do not ascend within [0, tokens]
// are recorded and cut to it.
__device__ __forceinline__ void sequence(const long long* offsets, long long seq_len, long long tokens, int q, long long& a, long long& b,
                                         int* status) {
  a = offsets ? offsets[q] : q * seq_len;
  b = offsets ? offsets[q + 1] : a + seq_len;
  if (a < 0 || b < a || b > tokens) {
    if (threadIdx.x == 0) atomicCAS(status, 0, BB_ERR_INVALID_ARG);
    a = a < 0 ? 0 : a > tokens ? tokens : a;
    b = b < a ? a : b > tokens ? tokens : b;
  }
}

// Zeros for the tokens in front of the first sequence (first CTA) and behind the last (last CTA) of `sequences`
__device__ __forceinline__ void outside_zero(const long long* offsets, long long tokens, int sequences, float* out) {
  if (!offsets) return;
  if (blockIdx.x == 0)
    for (long long i = threadIdx.x; i < offsets[0] && i < tokens; i += 256) out[i] = 0.f;
  if (blockIdx.x == gridDim.x - 1) {
    const long long end = offsets[sequences];
    for (long long i = (end > 0 ? end : 0) + threadIdx.x; i < tokens; i += 256) out[i] = 0.f;
  }
}

// ------------------------------------------------------------------ preference loss
// One CTA per pair.  s_q = sum (or mean) over counted tokens of logp - ref; h = beta (s_2i - s_2i+1); pair_loss[i] = f(h);
// row_grad = +-beta f'(h) / pairs (/ count) on counted tokens, 0 elsewhere.
__global__ void __launch_bounds__(256)
preference_pair_kernel(const float* logp, const float* rest, const float* ref, const long long* targets, const long long* offsets, long long seq_len,
                       long long tokens, int pairs, int form, double beta, double smoothing, int average, long long ignore_index,
                       double* pair_loss, float* rewards, float* row_grad, int* status) {
  __shared__ double smem[8][4];
  bb::pdl_sync();
  const int pair = blockIdx.x;
  double score[2], length[2], sums[4] = {0.0, 0.0, 0.0, 0.0};
  long long a[2], b[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    sequence(offsets, seq_len, tokens, 2 * pair + w, a[w], b[w], status);
    int count = 0;
#pragma unroll 4
    for (long long i = a[w] + threadIdx.x; i < b[w]; i += 256) {
      // (read without waiting for the target: what stands at a place that does not count is dropped, whatever it is)
      const double d = (double)logp[i] - (ref ? (double)ref[i] : 0.0) + (rest ? (double)rest[i] : 0.0);
      const bool counted = targets[i] != ignore_index;
      sums[w] += counted ? d : 0.0;
      count += counted;
    }
    sums[2 + w] = (double)count;
  }
  block_sums<256, 4>(sums, smem);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    length[w] = average ? fmax(sums[2 + w], 1.0) : 1.0;
    score[w] = sums[w] / length[w];
  }
  const double h = beta * (score[0] - score[1]);
  double loss, slope;
  if (form == BB_PREFERENCE_SIGMOID) {
    // softplus(z) = max(z, 0) + log(1 + e^-|z|);  -log sig(h) = softplus(-h)
    const double tail = log1p(exp(-fabs(h)));
    loss = (1.0 - smoothing) * (fmax(-h, 0.0) + tail) + smoothing * (fmax(h, 0.0) + tail);
    const double sig = 1.0 / (1.0 + exp(-h));
    slope = sig - 1.0 + smoothing;
  } else if (form == BB_PREFERENCE_HINGE) {
    loss = fmax(0.0, 1.0 - h);
    slope = h < 1.0 ? -1.0 : 0.0;
    if (h != h) loss = slope = h;
  } else {
    const double gap = (h - 0.5) / beta;
    loss = gap * gap;
    slope = 2.0 * gap / beta;
  }
  if (threadIdx.x == 0) {
    pair_loss[pair] = loss;
    rewards[2 * pair] = (float)(beta * score[0]);
    rewards[2 * pair + 1] = (float)(beta * score[1]);
  }
  for (int w = 0; w < 2; ++w) {
    const float g = (float)((w ? -slope : slope) * beta / ((double)pairs * length[w]));
    for (long long i = a[w] + threadIdx.x; i < b[w]; i += 256) row_grad[i] = targets[i] == ignore_index ? 0.f : g;
  }
  outside_zero(offsets, tokens, 2 * pairs, row_grad);
}

__global__ void __launch_bounds__(256)
preference_mean_kernel(const double* pair_loss, int pairs, float* loss) {
  bb::pdl_sync();
  mean_of<256>(pair_loss, pairs, loss);
}

// ------------------------------------------------------------------ policy loss
struct PolicyParams {
  const float* old_logp;        // NULL: the tokens were sampled by this very policy (ratio 1)
  const float* advantages;      // index = row / adv_div
  const float* ref;             // NULL: no KL term
  const float* weight;          // per token (sequence reduction); NULL: 1 / number of counted tokens
  const int* counts; int num_counts;
  long long adv_div;
  float low, high, kl_coef;     // ratio bounds 1 - clip_low, 1 + clip_high
};
constexpr float LN2_HI = 0.693147181f, LN2_LO = -1.9046542e-9f;        // ln 2 in two floats
struct PolicyInput { float old, adv, ref; };
struct PolicyToken { float loss, kl, clipped, slope; };

__device__ __forceinline__ PolicyInput policy_input(const PolicyParams& p, long long row) {
  return {p.old_logp ? p.old_logp[row] : 0.f, p.advantages[p.adv_div == 1 ? row : row / p.adv_div], p.ref ? p.ref[row] : 0.f};
}
// e^gap - 1 - gap, e = e^gap - 1.  The difference of the two cancels near zero (at a gap of 1e-3 to 1e-4 of the result), so below a quarter it is the
// series up to gap^8 / 8!, 4e-10 of the result short.
__device__ __forceinline__ float kl_term(float gap, float e) {
  if (!(fabsf(gap) < 0.25f)) return e - gap;
  float c = 1.f / 8.f;
#pragma unroll
  for (int n = 7; n >= 3; --n) c = fmaf(c, gap, 1.f) * (1.f / (float)n);
  return 0.5f * gap * gap * fmaf(c, gap, 1.f);
}

// `decided`: whether the token is clipped, where its gradient was made already (< 0: not yet)
__device__ __forceinline__ PolicyToken policy_token(const PolicyParams& p, const PolicyInput& in, double lp, int decided = -1) {
  PolicyToken o;
  const float ratio = p.old_logp ? expf((float)(lp - (double)in.old)) : 1.f;
  // (an advantage of 0 has no part in the surrogate, whatever the ratio overflowed to)
  const float plain = in.adv == 0.f ? 0.f : ratio * in.adv, bounded = fminf(fmaxf(ratio, p.low), p.high) * in.adv;
  const bool cut = decided < 0 ? bounded < plain : decided != 0;
  o.clipped = cut ? 1.f : 0.f;
  o.loss = cut ? -bounded : -plain;
  o.slope = cut ? 0.f : -plain;
  o.kl = 0.f;
  if (p.ref) {
    const float gap = (float)((double)in.ref - lp), e = expm1f(gap);
    o.kl = kl_term(gap, e);
    o.loss += p.kl_coef * o.kl;
    o.slope -= p.kl_coef * e;
  }
  return o;
}

// What the row kernels wait for between their halves: the token's slope, and whether it is clipped, from the row's sums.  The gaps between the
// log-probability and those of the other policies are differences of numbers of any size whose rounding to 32 bits would show (1e-5 at -150), so they
// are kept in two floats each (k x - r - log2 s exactly but for the logarithm of the sum's mantissa, 6e-8): 64 bits cost 3 to 5 % of rows of 4 to 30 KB.
struct PolicySlope { float slope; bool cut; };
__device__ __forceinline__ PolicySlope policy_slope(const PolicyParams& p, const PolicyInput& in, float xt, K2 k, float r, float s) {
  float to_old, to_ref;
  const float a = __fmul_rn(xt, k.hi);                       // (a product that no sum below may take up)
  if (s > 0.f && fabsf(a) < INFINITY) {
    const int bits = __float_as_int(s);
    const float log2_m = log2f(__int_as_float((bits & 0x7FFFFF) | 0x3F800000)), whole = r + (float)((bits >> 23) - 127);
    const float b = a - whole, v = b - a, b_rest = (a - (b - v)) - (whole + v);      // (the sum's rounding, by Knuth)
    const float rest = (b_rest - log2_m) + fmaf(xt, k.lo, fmaf(xt, k.hi, -a));
    const float lp = __fmul_rn(b, LN2_HI), lp_rest = fmaf(rest, LN2_HI, fmaf(b, LN2_LO, fmaf(b, LN2_HI, -lp)));
    to_old = (lp - in.old) + lp_rest;
    to_ref = (in.ref - lp) - lp_rest;
  } else {
    const double lp = row_logp(xt, k, r, s);
    to_old = (float)(lp - (double)in.old);
    to_ref = (float)((double)in.ref - lp);
  }
  const float ratio = p.old_logp ? expf(to_old) : 1.f;
  const float plain = in.adv == 0.f ? 0.f : ratio * in.adv, bounded = fminf(fmaxf(ratio, p.low), p.high) * in.adv;
  PolicySlope o = {bounded < plain ? 0.f : -plain, bounded < plain};
  if (p.ref) o.slope -= p.kl_coef * expm1f(to_ref);
  return o;
}

// Counted tokens of each of `gridDim.x` pieces of the targets (sequences, or equal pieces when weight is NULL) and, per sequence,
// the weight 1 / (sequences * counted) of its tokens
__global__ void __launch_bounds__(256)
policy_count_kernel(const long long* targets, const long long* offsets, long long piece, long long tokens, long long ignore_index,
                    int* counts, float* weight, int* status) {
  __shared__ double smem[8];
  bb::pdl_sync();
  long long a, b;
  if (weight) {
    sequence(offsets, piece, tokens, blockIdx.x, a, b, status);
  } else {
    a = blockIdx.x * piece;
    b = a + piece < tokens ? a + piece : tokens;
  }
  int count = 0;
  for (long long i = a + threadIdx.x; i < b; i += 256) count += targets[i] != ignore_index;
  const double n = block_sum<256>((double)count, smem);
  if (threadIdx.x == 0) counts[blockIdx.x] = (int)n;
  // rows drawn by policy_ring_kernel, CTAs of policy_token_kernel that are done
  if (threadIdx.x == 0 && blockIdx.x == 0) counts[gridDim.x] = counts[gridDim.x + 1] = 0;
  if (!weight) return;
  const float w = (float)(1.0 / ((double)gridDim.x * (n > 1.0 ? n : 1.0)));
  for (long long i = a + threadIdx.x; i < b; i += 256) weight[i] = w;
  outside_zero(offsets, tokens, gridDim.x, weight);
}

__device__ __forceinline__ float policy_weight(const PolicyParams& p, long long row) {
  if (p.weight) return p.weight[row];
  double n = 0.0;
  for (int i = 0; i < p.num_counts; ++i) n += (double)p.counts[i];
  return (float)(1.0 / (n > 1.0 ? n : 1.0));
}

// Token by token: row_grad (from log-probabilities), or the log-probability (from rows: the softmax sums and the target's logit that a row
// kernel left, and whether its gradient is that of a clipped token).  The sums of a CTA's tokens - weighted loss, KL, clipped -
// meet in the CTA that finishes last, in the order of the CTAs: loss[0], and stats = mean KL and share of clipped among counted tokens.
struct PolicyRow { float r, s, xt; int kind; };
constexpr int ROW_IGNORED = 0, ROW_COUNTS = 1, ROW_CLIPPED = 2;
template <bool FROM_ROWS>
__global__ void __launch_bounds__(256)
policy_token_kernel(float* logp, const PolicyRow* row_sums, K2 k, const long long* targets, const PolicyParams p, long long tokens, long long ignore_index,
                    float* row_grad, double* partial, int* done, float* loss, float* stats) {
  __shared__ double smem[8][4];
  __shared__ int s_last;
  bb::pdl_sync();
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  const float whole = p.weight ? 0.f : policy_weight(p, 0);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < tokens; i += (long long)gridDim.x * 256) {
    const float w = p.weight ? p.weight[i] : whole;
    double lp;
    int decided = -1;
    if constexpr (FROM_ROWS) {
      const PolicyRow q = row_sums[i];
      lp = q.kind == ROW_IGNORED ? 0.0 : row_logp(q.xt, k, q.r, q.s);
      if (logp) logp[i] = (float)lp;
      if (q.kind == ROW_IGNORED) continue;
      decided = q.kind == ROW_CLIPPED;
    } else {
      if (targets[i] == ignore_index || w == 0.f) { row_grad[i] = 0.f; continue; }
      lp = (double)logp[i];
    }
    const PolicyToken o = policy_token(p, policy_input(p, i), lp, decided);
    if constexpr (!FROM_ROWS) row_grad[i] = o.slope * w;
    v[0] += (double)o.loss * w; v[1] += o.kl; v[2] += o.clipped;
  }
  if (gridDim.x > 1) {
    block_sums<256, 4>(v, smem);
    if (threadIdx.x == 0) {
      for (int c = 0; c < 3; ++c) __stcg(partial + 3 * blockIdx.x + c, v[c]);
      __threadfence();
      s_last = atomicAdd(done, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    for (int c = 0; c < 3; ++c) v[c] = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256)
      for (int c = 0; c < 3; ++c) v[c] += __ldcg(partial + 3 * i + c);
  }
  v[3] = 0.0;
  for (int i = threadIdx.x; i < p.num_counts; i += 256) v[3] += (double)p.counts[i];
  block_sums<256, 4>(v, smem);
  if (threadIdx.x == 0) {
    const double total = fmax(v[3], 1.0);
    loss[0] = (float)v[0]; stats[0] = (float)(v[1] / total); stats[1] = (float)(v[2] / total);
  }
}

// What thread 0 does between the two halves of a row; the token's loss follows in policy_token_kernel
__device__ __forceinline__ void policy_row_finish(const PolicyParams& p, const PolicyInput& in, int row, float xt, K2 k, float r, float s, float weight, float gscale,
                                                  float* s_row, PolicyRow* row_sums) {
  const PolicySlope o = policy_slope(p, in, xt, k, r, s);
  s_row[0] = r; s_row[1] = s; s_row[2] = o.slope * weight * gscale;
  row_sums[row] = {r, s, xt, o.cut ? ROW_CLIPPED : ROW_COUNTS};
}

// One CTA per row of logits: log-probability, the token's loss and, because a row's gradient needs nothing of the other rows (the
// weights follow from the targets), that gradient too.  For rows that are short, or too long for policy_ring_kernel: the second half reads
// the row again, from L1 or L2.
// Registers for 1536 threads of an SM where the compiler would take more (16384 bf16 rows of 8203: 118 us with 48, 116 with 40)
template <typename T, int THREADS> constexpr int POLICY_BLOCKS = sizeof(T) == 2 && THREADS >= 64 && THREADS <= 256 ? 1536 / THREADS : 0;
template <typename T, int THREADS>
__global__ void __launch_bounds__(BLOCK<THREADS>, POLICY_BLOCKS<T, THREADS>)
policy_row_kernel(const T* logits, long long ld, const long long* targets, const PolicyParams p, K2 k, float gscale,
                  T* dlogits, long long ldd, int rows, int V, int cols, long long ignore_index, PolicyRow* row_sums, int* status) {
  __shared__ float2 smem[BLOCK<THREADS> / 32];
  __shared__ float s_row[BLOCK<THREADS> / 32][3];
  bb::pdl_sync();
  const int row = THREADS == 32 ? (int)blockIdx.x * ROWS_OF_BLOCK<THREADS> + (int)(threadIdx.x >> 5) : (int)blockIdx.x;
  if (row >= rows) return;
  float* mine = s_row[THREADS == 32 ? threadIdx.x >> 5 : 0];
  const bool first = row_thread<THREADS>() == 0;
  const long long t = targets[row];
  const T* x = logits + (size_t)row * ld;
  const bool valid = t != ignore_index && t >= 0 && t < V, counted = valid && !(p.weight && p.weight[row] == 0.f);
  float r = 0.f, s = 0.f, g = 0.f;
  if (counted) {
    // (in flight while the row is read: one after the other their latencies would stand between the two halves)
    PolicyInput in = {};
    float xt = 0.f, weight = 0.f;
    if (first) { in = policy_input(p, row); xt = Elem<T>::get(x + t); weight = policy_weight(p, row); }
    soft_whole_row<T, THREADS, ROW_LOADS>(x, V, k, r, s, smem);
    if (first) policy_row_finish(p, in, row, xt, k, r, s, weight, gscale, mine, row_sums);
    // also: every thread is past its reads of the row before it may be overwritten
    if constexpr (THREADS == 32) __syncwarp();
    else __syncthreads();
    r = mine[0]; s = mine[1]; g = mine[2];
  } else if (first) {
    if (!valid && t != ignore_index) atomicCAS(status, 0, BB_ERR_INVALID_ARG);
    row_sums[row] = {0.f, 0.f, 0.f, ROW_IGNORED};
  }
  grad_row<T, THREADS, ROW_LOADS>(x, dlogits + (size_t)row * ldd, V, cols, (int)t, g, k, r, s);
}

// What the feeding warp of policy_ring_kernel hands over with a row; row < 0: no more
struct PolicyTurn { int row, t; PolicyInput in; float weight, xt; };
constexpr int TURNS = 4;

// The same for long rows, each read from memory once.  A row lands in shared memory (a ring of stages of four chunks per thread that
// holds one row; bulk copies by a warp of their own), stays there for its gradient, and as that consumes stage after stage the next row
// follows into them.  Two CTAs per SM fill each other's turns: a row takes a CTA (V = 50257, bf16) about 1.7 us of ex2
// for the sum and again for the gradient, most of one between them for the sum's barrier and the token's slope, and an SM's
// share of the memory rate is a row in 4.5 us.  Rows that do not count cost a CTA a fraction of the others and come in
// runs (prompts), so rows are drawn from a counter.  7777 tokens, 16 sequences: 246-260 us from call to call with the two small kernels around it, 5.4-5.7 TB/s
// (beside 241 us: a block per row, read twice, 349; ring with rows dealt out in advance 305; 512 threads 248, 256 threads 245-248).
constexpr int RING_THREADS = 384, RING_CHUNKS = 4, RING_STAGE = RING_THREADS * RING_CHUNKS * 16, RING_STAGES = (int)(MAX_RING + RING_STAGE - 1) / RING_STAGE;
template <typename T>
__global__ void __launch_bounds__(RING_THREADS + 32, 2)
policy_ring_kernel(const T* logits, long long ld, const long long* targets, const PolicyParams p, K2 k, float gscale,
                   T* dlogits, long long ldd, int rows, int V, int cols, long long ignore_index, PolicyRow* row_sums, int* status, int stages, int* ticket) {
  constexpr int VEC = Elem<T>::VEC, THREADS = RING_THREADS, U = RING_CHUNKS, STAGE = THREADS * U;
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ float2 smem[THREADS / 32];
  __shared__ float s_row[3];
  __shared__ PolicyTurn turns[TURNS];
  __shared__ uint64_t turn_full[TURNS], turn_empty[TURNS];
  __shared__ int s_abort;
  __shared__ uint64_t full[RING_STAGES], empty[RING_STAGES];
  volatile int* abort_flag = &s_abort;
  const int warp = bb::warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int j = 0; j < stages; ++j) { bb::mbar_init(&full[j], 1); bb::mbar_init(&empty[j], THREADS / 32); }
    for (int j = 0; j < TURNS; ++j) { bb::mbar_init(&turn_full[j], 1); bb::mbar_init(&turn_empty[j], THREADS / 32); }
    bb::fence_barrier_init();
  }
  __syncthreads();
  bb::pdl_sync();
  if (warp == THREADS / 32) {
    // ---- the warp that feeds: draws rows, fetches what their tokens bring along, and lets the chunks of a counted row follow the gradient
    // of the row before it into the same places
    const float whole = p.weight ? 0.f : policy_weight(p, 0);
    bool alive = true;
    uint32_t phase = 0;
    int row = blockIdx.x;
    for (int it = 0; alive; ++it) {
      const bool more = row < rows;
      // (the next draw is under way while this row's copies are issued)
      const int drawn = more && lane == 0 ? (int)gridDim.x + atomicAdd(ticket, 1) : 0;
      PolicyTurn turn = {-1, -1, {}, 0.f, 0.f};
      const T* x = logits;
      if (more) {
        x += (size_t)row * ld;
        const long long t = targets[row];
        const bool valid = t != ignore_index && t >= 0 && t < V;
        turn.row = row;
        turn.weight = p.weight ? p.weight[row] : whole;
        turn.in = policy_input(p, row);
        if (valid && turn.weight != 0.f) { turn.t = (int)t; turn.xt = Elem<T>::get(x + t); }
        if (!valid && t != ignore_index && lane == 0) atomicCAS(status, 0, BB_ERR_INVALID_ARG);
      }
      const int at = it % TURNS;
      alive = bb::mbar_wait_warp(&turn_empty[at], ((it / TURNS) & 1) ^ 1, abort_flag, status);
      if (!alive) break;
      if (lane == 0) { turns[at] = turn; bb::mbar_arrive(&turn_full[at]); }
      __syncwarp();
      if (!more) break;
      if (turn.t >= 0) {
        const Span<T> sp(x, V);
        for (int j = 0; j < stages; ++j) {
          alive = bb::mbar_wait_warp(&empty[j], phase ^ 1, abort_flag, status);
          if (!alive) break;
          const int left = (sp.nvec - j * STAGE) * 16, bytes = left <= 0 ? 0 : left < RING_STAGE ? left : RING_STAGE;
          if (bb::elect_one()) {
            bb::mbar_arrive_expect_tx(&full[j], bytes);
            if (bytes) bb::bulk_load(ring + j * STAGE, x + sp.lead + (size_t)j * STAGE * VEC, bytes, &full[j]);
          }
          __syncwarp();
        }
        phase ^= 1;
      }
      row = __shfl_sync(0xffffffffu, drawn, 0);
    }
    return;
  }
  bool alive = true;
  uint32_t phase = 0;
  for (int it = 0;; ++it) {
    const int at = it % TURNS;
    alive = alive && bb::mbar_wait_warp(&turn_full[at], (it / TURNS) & 1, abort_flag, status);
    const PolicyTurn turn = turns[at];         // (handed back when the row is done, for the same reason as the stages)
    auto turn_done = [&] {
      __syncwarp();
      if (lane == 0) bb::mbar_arrive(&turn_empty[at]);
    };
    const int row = turn.row, t = turn.t;
    // a wait that ran out in one warp ends the loop for all of them here, where their barriers match; the barrier itself says so (a flag beside it
    // could be set for the next row, where this one does not count, before a slow warp has read it for this one)
    if (row_barrier_any<THREADS>(!alive) || row < 0) break;
    const T* x = logits + (size_t)row * ld;
    T* d = dlogits + (size_t)row * ldd;
    if (t < 0) {
      if (threadIdx.x == 0) row_sums[row] = {0.f, 0.f, 0.f, ROW_IGNORED};
      grad_row<T, THREADS, ROW_LOADS>(x, d, V, cols, 0, 0.f, k, 0.f, 0.f);
      turn_done();
      continue;
    }
    // ---- sum
    const Span<T> sp(x, V);
    const float xt = turn.xt;
    float r = -INFINITY, s = 0.f;
    float2 sum = make_float2(0.f, 0.f);
    for (int j = 0; j < stages; ++j) {
      if (alive) alive = bb::mbar_wait_warp(&full[j], phase, abort_flag, status);
      const int c = j * STAGE + threadIdx.x;
      float f[VEC];
      if (c + (U - 1) * THREADS < sp.nvec) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = ring[c + u * THREADS];
        if (j == 0) { Elem<T>::unpack(q[0], f); soft_add<VEC>(r, s, f, k, -bb::SOFT_FAR); }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u > 0 || j > 0) { Elem<T>::unpack(q[u], f); soft_chunk<VEC>(sum, f, k, r); }
      } else {
        for (int u = 0; u < U; ++u) {
          if (c + u * THREADS >= sp.nvec) break;
          Elem<T>::unpack(ring[c + u * THREADS], f);
          if (j == 0 && u == 0) soft_add<VEC>(r, s, f, k, -bb::SOFT_FAR);
          else soft_chunk<VEC>(sum, f, k, r);
        }
      }
    }
    s += sum.x + sum.y;
    if (!(s < SHARE_MOST)) { const float2 e = soft_share_exact<T, THREADS>(ring, sp.nvec, k); r = e.x; s = e.y; }
    soft_edges<T, THREADS>(x, sp, V, k, r, s);
    soft_block<THREADS, true>(r, s, smem);
    if (threadIdx.x < 32 && soft_far(r)) { const float2 e = soft_row_far(x, V, k); r = e.x; s = e.y; }
    if (threadIdx.x == 0) policy_row_finish(p, turn.in, row, xt, k, r, s, turn.weight, gscale, s_row, row_sums);
    row_barrier<THREADS, true>();    // also: every thread is past its reads of the row before it may be overwritten
    r = s_row[0]; s = s_row[1];
    float g = s_row[2];
    if (s == 0.f) g = 0.f;
    // ---- gradient; a stage is handed back by the warps that have taken their chunks out of it, which is certain once what was made of them
    // is on its way: an arrival right behind the loads may pass them (they queue behind stores of earlier stages), and the next
    // row's first lines land in what is still to be read
    const bool plain = g == 0.f || s < 0.f || (((uintptr_t)x ^ (uintptr_t)d) & 15) != 0;
    const GradRow gw = grad_factors(g, k, plain ? 0.f : r, s);
    const int whole = plain ? 0 : (V - sp.lead) / VEC;         // chunks of vocabulary entries only
    uint4* dv = reinterpret_cast<uint4*>(d + sp.lead);
    for (int j = 0; j < stages; ++j) {
      const int c = j * STAGE + threadIdx.x;
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = c + u * THREADS < whole ? ring[c + u * THREADS] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < U; ++u) if (c + u * THREADS < whole) grad_chunk<T>(dv + c + u * THREADS, q[u], gw);
      __syncwarp();
      if (lane == 0) bb::mbar_arrive(&empty[j]);
    }
    if (plain) grad_row<T, THREADS, ROW_LOADS>(x, d, V, cols, t, g, k, r, s);
    else grad_rest<T, THREADS>(x, xt, d, sp.lead, whole, V, cols, t, g, k, s, gw);
    turn_done();
    phase ^= 1;
  }
  if (!alive) {
    // copies that may still be in flight land before the CTA's shared memory is released (bounded)
    const uint64_t t0 = bb::globaltimer_ns();
    while (bb::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
}

constexpr int RESCALE_THREADS = 256;
// A gradient that was made for an upstream gradient of `made_for`, times *grad / made_for: nothing to do where they are the same
template <typename T>
__global__ void __launch_bounds__(RESCALE_THREADS)
rescale_kernel(T* d, long long ld, int cols, const float* grad, float made_for) {
  constexpr int VEC = Elem<T>::VEC;
  bb::pdl_sync();
  if (grad[0] == made_for) return;
  const float c = grad[0] / made_for;
  T* x = d + (size_t)blockIdx.x * ld;
  const Span<T> sp(x, cols);
  uint4* v = reinterpret_cast<uint4*>(x + sp.lead);
  for (int i = threadIdx.x; i < sp.nvec; i += RESCALE_THREADS) {
    float f[VEC];
    Elem<T>::unpack(v[i], f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] *= c;
    v[i] = Elem<T>::pack(f);
  }
  for (int j = threadIdx.x; j < sp.lead + cols - sp.tail; j += RESCALE_THREADS) {
    T* at = x + (j < sp.lead ? j : sp.tail + j - sp.lead);
    Elem<T>::put(at, Elem<T>::get(at) * c);
  }
}

// ------------------------------------------------------------------ gradient norm, clipping
constexpr int LIST_TENSORS = 128;             // tensors of one launch: their table travels as a kernel argument
// Both passes deal the list out in small pieces, most of them one per CTA: a CTA that walks a grid's share of a large list keeps
// fewer requests in flight between its pieces.  153 M bf16 values: sum 52 us (5.9 TB/s), scaling 93 us (6.6 TB/s) in pieces of 16384
// elements, 108 in pieces of 8192 or with four CTAs per SM that walk.
constexpr int NORM_THREADS = 512, NORM_LOADS = 4, NORM_CTAS = 8192;
constexpr long long SUM_PIECE = 32768, CLIP_PIECE = 16384;
struct TensorTable {
  void* data[LIST_TENSORS];
  long long numel[LIST_TENSORS];
  int first[LIST_TENSORS + 1];                // first piece of each tensor, a piece being `piece` elements
  unsigned char dtype[LIST_TENSORS];
  int count, piece;
};

// tensor and element range of a piece
__device__ __forceinline__ int table_find(const TensorTable& t, int piece, long long& a, long long& n) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= piece) lo = mid; else hi = mid - 1;
  }
  a = (long long)(piece - t.first[lo]) * t.piece;
  n = t.numel[lo] - a < t.piece ? t.numel[lo] - a : t.piece;
  return lo;
}

template <typename T> __device__ __forceinline__ float sumsq_chunk(const uint4& q) {
  constexpr int VEC = Elem<T>::VEC;
  float f[VEC];
  float2 sum = make_float2(0.f, 0.f);
  Elem<T>::unpack(q, f);
#pragma unroll
  for (int i = 0; i < VEC; i += 2) sum = bb::fma2(make_float2(f[i], f[i + 1]), make_float2(f[i], f[i + 1]), sum);
  return sum.x + sum.y;
}
// A thread's share again with its squares in 64 bits, for values from 1.8e19 on (and infinities and NaN, which stay)
template <typename T> __device__ __noinline__ double sumsq_share_wide(const T* x, int n) {
  const Span<T> sp(x, n);
  constexpr int VEC = Elem<T>::VEC;
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.lead);
  double sum = 0.0;
  for (int c = threadIdx.x; c < sp.nvec; c += NORM_THREADS) {
    float f[VEC];
    Elem<T>::unpack(v[c], f);
    for (int i = 0; i < VEC; ++i) sum += (double)f[i] * (double)f[i];
  }
  for (int j = threadIdx.x; j < sp.lead + n - sp.tail; j += NORM_THREADS) {
    const double f = (double)Elem<T>::get(x + (j < sp.lead ? j : sp.tail + j - sp.lead));
    sum += f * f;
  }
  return sum;
}
// (a chunk's squares in 32 bits, everything above in 64)
template <typename T> __device__ __forceinline__ double sumsq_piece(const T* x, int n) {
  constexpr int U = NORM_LOADS;
  const Span<T> sp(x, n);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.lead);
  double sum = 0.0;
  int c = threadIdx.x;
  for (; c + (U - 1) * NORM_THREADS < sp.nvec; c += U * NORM_THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = v[c + u * NORM_THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) sum += (double)sumsq_chunk<T>(q[u]);
  }
  for (; c < sp.nvec; c += NORM_THREADS) sum += (double)sumsq_chunk<T>(v[c]);
  for (int j = threadIdx.x; j < sp.lead + n - sp.tail; j += NORM_THREADS) {
    const float f = Elem<T>::get(x + (j < sp.lead ? j : sp.tail + j - sp.lead));
    sum += (double)(f * f);
  }
  return isfinite(sum) ? sum : sumsq_share_wide(x, n);
}

// What a squared norm means for the gradients: norm = pre_scale * sqrt(sum of squares), coefficient = min(1, max_norm / (norm + 1e-6)), NaN
// for a NaN norm
struct ClipTo { double pre_scale, max_norm; float* coef; float* norm; };
__device__ __forceinline__ void clip_write(const ClipTo& c, double sumsq) {
  const double norm = c.pre_scale * sqrt(sumsq), coef = c.max_norm / (norm + 1e-6);
  c.norm[0] = (float)norm;
  c.coef[0] = coef >= 1.0 ? 1.f : (float)coef;
}
__global__ void clip_coef_kernel(const double* sumsq, const ClipTo c) {
  bb::pdl_sync();
  clip_write(c, sumsq[0]);
}

// total[0] (+)= sum of squares of the list: every CTA sums its pieces (each gridDim.x-th), the CTA that finishes last adds the CTAs' sums in
// their order, and writes the coefficient where that was asked for.  `done` returns to zero by itself.
__global__ void __launch_bounds__(NORM_THREADS)
grad_sumsq_kernel(const __grid_constant__ TensorTable t, double* partial, double* total, int add, unsigned int* done, const ClipTo clip) {
  __shared__ double smem[NORM_THREADS / 32];
  __shared__ int s_last;
  bb::pdl_sync();
  double sum = 0.0;
  for (int piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
    long long a, n;
    const int i = table_find(t, piece, a, n);
    sum += t.dtype[i] == BB_DTYPE_F32 ? sumsq_piece(reinterpret_cast<const float*>(t.data[i]) + a, (int)n)
                                      : sumsq_piece(reinterpret_cast<const __nv_bfloat16*>(t.data[i]) + a, (int)n);
  }
  sum = block_sum<NORM_THREADS>(sum, smem);
  if (threadIdx.x == 0) {
    __stcg(partial + blockIdx.x, sum);
    __threadfence();
    s_last = atomicInc(done, gridDim.x - 1) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  sum = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += NORM_THREADS) sum += __ldcg(partial + i);
  sum = block_sum<NORM_THREADS>(sum, smem);
  if (threadIdx.x == 0) {
    if (add) sum += total[0];
    total[0] = sum;
    if (clip.coef) clip_write(clip, sum);
  }
}

template <typename T> __device__ __forceinline__ uint4 scale_chunk(const uint4& q, float c) {
  constexpr int VEC = Elem<T>::VEC;
  float f[VEC];
  Elem<T>::unpack(q, f);
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] *= c;
  return Elem<T>::pack(f);
}
template <typename T> __device__ __forceinline__ void scale_piece(T* x, int n, float c) {
  constexpr int U = NORM_LOADS;
  const Span<T> sp(x, n);
  uint4* v = reinterpret_cast<uint4*>(x + sp.lead);
  int i = threadIdx.x;
  for (; i + (U - 1) * NORM_THREADS < sp.nvec; i += U * NORM_THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = v[i + u * NORM_THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) v[i + u * NORM_THREADS] = scale_chunk<T>(q[u], c);
  }
  for (; i < sp.nvec; i += NORM_THREADS) v[i] = scale_chunk<T>(v[i], c);
  for (int j = threadIdx.x; j < sp.lead + n - sp.tail; j += NORM_THREADS) {
    T* p = x + (j < sp.lead ? j : sp.tail + j - sp.lead);
    Elem<T>::put(p, Elem<T>::get(p) * c);
  }
}

// One piece per CTA
__global__ void __launch_bounds__(NORM_THREADS)
grad_clip_kernel(const __grid_constant__ TensorTable t, const float* coef) {
  bb::pdl_sync();
  const float c = coef[0];
  if (c == 1.f) return;                         // within the norm: the gradients stay as they are
  long long a, n;
  // last pieces first: the sum read them last, and what of them is still in L2 need not come from memory again (sum and scaling of
  // those 153 M values 156 -> 153 us)
  const int i = table_find(t, gridDim.x - 1 - blockIdx.x, a, n);
  if (t.dtype[i] == BB_DTYPE_F32) scale_piece(reinterpret_cast<float*>(t.data[i]) + a, (int)n, c);
  else scale_piece(reinterpret_cast<__nv_bfloat16*>(t.data[i]) + a, (int)n, c);
}

// Adam on the clipped gradient; what the host can fold is folded there in 64 bits (1 - beta, bias corrections).  102.9 M parameters:
// 513 us at 6.8 TB/s (34 bytes each) with four elements per thread and CTAs of 256, which all come and go; 590 us in CTAs that
// walk, six per SM.
struct AdamParams { float lr, b1, omb1, b2, omb2, eps, inv_bc1, inv_bc2, decay; int decoupled, zero_grad; };

__global__ void __launch_bounds__(256)
adam_clip_kernel(float* p, float* g, float* m, float* v, __nv_bfloat16* lp, long long n, const AdamParams a, const float* coef,
                 float pre_scale) {
  bb::pdl_sync();
  // four elements per thread, last ones first (see grad_clip_kernel)
  const long long i = (gridDim.x - 1 - blockIdx.x) * 256LL + threadIdx.x;
  if (i >= n >> 2) return;
  const float4 P = reinterpret_cast<float4*>(p)[i], G = reinterpret_cast<float4*>(g)[i];
  const float4 M = reinterpret_cast<float4*>(m)[i], W = reinterpret_cast<float4*>(v)[i];
  float pp[4] = {P.x, P.y, P.z, P.w}, gg[4] = {G.x, G.y, G.z, G.w}, mm[4] = {M.x, M.y, M.z, M.w}, vv[4] = {W.x, W.y, W.z, W.w};
  const float c = coef[0] * pre_scale;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = gg[e] * c;
    if (!a.decoupled) x = fmaf(a.decay, pp[e], x);
    mm[e] = fmaf(a.b1, mm[e], a.omb1 * x);
    vv[e] = fmaf(a.b2, vv[e], a.omb2 * x * x);
    float step = (mm[e] * a.inv_bc1) / (sqrtf(vv[e] * a.inv_bc2) + a.eps);
    if (a.decoupled) step = fmaf(a.decay, pp[e], step);
    pp[e] = fmaf(-a.lr, step, pp[e]);
  }
  reinterpret_cast<float4*>(p)[i] = make_float4(pp[0], pp[1], pp[2], pp[3]);
  reinterpret_cast<float4*>(m)[i] = make_float4(mm[0], mm[1], mm[2], mm[3]);
  reinterpret_cast<float4*>(v)[i] = make_float4(vv[0], vv[1], vv[2], vv[3]);
  if (a.zero_grad) reinterpret_cast<float4*>(g)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (lp) reinterpret_cast<uint2*>(lp)[i] = make_uint2(bb::pack_bf16x2(pp[0], pp[1]), bb::pack_bf16x2(pp[2], pp[3]));
}

// ------------------------------------------------------------------ host side
bool bad_logits(const char* who, const void* logits, int dtype, long long ld, const void* targets, long long rows, int vocab, double scale) {
  if (!logits || !targets || rows <= 0 || rows > INT_MAX || vocab <= 0 || ld < vocab || !(scale > 1e-30) || !(scale < 1e30) ||
      (dtype != BB_DTYPE_BF16 && dtype != BB_DTYPE_F32) || ((uintptr_t)logits & (dtype == BB_DTYPE_F32 ? 3 : 1))) {
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: null or misaligned pointer, a size that is not positive, ld < vocab, an unknown type or a scale outside (1e-30, 1e30)", who);
    bb_set_last_error_msg(msg);
    return true;
  }
  return false;
}

// Whether the gradient may be written where it is asked for: apart from the logits, or exactly over them
bool bad_output(const void* logits, long long ld, const void* dlogits, long long ldd, int dtype, long long rows, int vocab, int cols) {
  const size_t item = dtype == BB_DTYPE_F32 ? 4 : 2;
  if (!dlogits || cols < vocab || ldd < cols || ((uintptr_t)dlogits & (item - 1))) return true;
  if (dlogits == logits) return ldd != ld;
  const uintptr_t a = (uintptr_t)logits, b = (uintptr_t)dlogits;
  const size_t an = ((size_t)(rows - 1) * (size_t)ld + (size_t)vocab) * item, bn = ((size_t)(rows - 1) * (size_t)ldd + (size_t)cols) * item;
  return a < b + bn && b < a + an;
}

int refuse(const char* msg) { bb_set_last_error_msg(msg); return BB_ERR_INVALID_ARG; }

// counts of counted tokens, and the weights of the sequence reduction; both at the front of the workspace
struct PolicyPlan { int num_counts; long long piece; size_t weight_at, rows_at, partial_at, bytes; };
int policy_token_ctas(long long tokens) {
  const long long want = (tokens + 255) / 256, cap = 4LL * bb_num_sms();
  return (int)(want < cap ? want : cap);
}
PolicyPlan policy_plan(long long tokens, int n_seq, bool by_sequence) {
  PolicyPlan pl;
  // (64 pieces at most: every CTA of the next kernel adds them up)
  pl.piece = (tokens + 63) / 64 > 2048 ? (tokens + 63) / 64 : 2048;
  pl.num_counts = by_sequence ? n_seq : (int)((tokens + pl.piece - 1) / pl.piece);
  size_t at = ((size_t)(pl.num_counts + 2) * 4 + 15) & ~(size_t)15;       // (two more: counters)
  pl.weight_at = at; at += by_sequence ? (size_t)tokens * 4 : 0;
  at = (at + 15) & ~(size_t)15;
  pl.rows_at = at; at += (size_t)tokens * sizeof(PolicyRow);
  pl.partial_at = at; at += (size_t)policy_token_ctas(tokens) * 24;
  pl.bytes = at;
  return pl;
}
// The list's tensors in pieces of `piece` elements, more where there would be too many
int table_fill(TensorTable& t, const bb_grad_tensor* list, int count, long long piece) {
  long long total = 0;
  for (int i = 0; i < count; ++i) total += list[i].numel;
  while (total / piece + count > (1 << 24)) piece *= 2;
  t.piece = (int)piece;
  t.count = count;
  int pieces = 0;
  for (int i = 0; i < count; ++i) {
    t.data[i] = list[i].data; t.numel[i] = list[i].numel; t.dtype[i] = (unsigned char)list[i].dtype;
    t.first[i] = pieces;
    pieces += (int)((list[i].numel + piece - 1) / piece);
  }
  t.first[count] = pieces;
  return pieces;
}
// Pieces of the sum: enough for every SM, none below 4096 elements
long long sum_piece(const bb_grad_tensor* list, int count) {
  long long total = 0;
  for (int i = 0; i < count; ++i) total += list[i].numel;
  const long long piece = (total / (4LL * bb_num_sms()) + 4095) / 4096 * 4096;
  return piece < 4096 ? 4096 : piece > SUM_PIECE ? SUM_PIECE : piece;
}

// Counters of the CTAs that are done, one per launch in turn; each is zero again when its launch is over.  A launch that is being captured
// keeps its counter for good, so those have a half of their own: a graph's replay never meets a launch that came round to the same one.
constexpr unsigned DONE_SLOTS = 1u << 15;
__device__ unsigned int g_norm_done[2 * DONE_SLOTS];
unsigned int* norm_done(cudaStream_t stream) {
  static unsigned int* table[64] = {nullptr};
  static std::atomic<unsigned> next[2];
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &status) != cudaSuccess) (void)cudaGetLastError();
  const int half = status == cudaStreamCaptureStatusNone ? 0 : 1;
  const int dev = bb_current_device();
  if (dev < 0) return nullptr;
  if (!table[dev]) {
    void* ptr = nullptr;
    if (cudaGetSymbolAddress(&ptr, g_norm_done) != cudaSuccess) return nullptr;
    table[dev] = static_cast<unsigned int*>(ptr);
  }
  return table[dev] + half * DONE_SLOTS + next[half].fetch_add(1u) % DONE_SLOTS;
}

bool bad_list(const bb_grad_tensor* list, int count) {
  if (!list || count <= 0) return true;
  for (int i = 0; i < count; ++i) {
    const int d = list[i].dtype;
    if (!list[i].data || list[i].numel <= 0 || list[i].numel > (1LL << 40) || (d != BB_DTYPE_BF16 && d != BB_DTYPE_F32) ||
        ((uintptr_t)list[i].data & (d == BB_DTYPE_F32 ? 3 : 1)))
      return true;
  }
  return false;
}

template <typename T> struct FwdCall { const T* logits; long long ld; const long long* targets; K2 k; float *logp, *rest; float2* stats; int rows, V; long long ignore; int* status; cudaStream_t s; };
// Blocks of a launch whose rows are worked on by THREADS threads each
template <int THREADS> int row_blocks(int rows) { return (rows + ROWS_OF_BLOCK<THREADS> - 1) / ROWS_OF_BLOCK<THREADS>; }
template <typename T, int THREADS> int fwd_rows(const FwdCall<T>& c) {
  BB_CUDA_CHECK(bb_launch(token_logprob_fwd_kernel<T, THREADS>, row_blocks<THREADS>(c.rows), BLOCK<THREADS>, 0, c.s, c.logits, c.ld, c.targets, c.k, c.logp,
                          c.rest, c.stats, c.rows, c.V, c.ignore, c.status));
  return BB_OK;
}
// CTAs per row: as long as four per SM do not come together, and a part keeps a chunk per thread (50 rows of 50257 bf16 logits 3.5 us less than
// with one CTA per row, 100 rows 2.9, 200 rows 1.9, from 300 on the same)
template <typename T> int fwd_parts(int rows, int V) {
  int parts = 1;
  while (parts < MAX_PARTS && 2LL * parts * rows <= 4LL * bb_num_sms() && (size_t)V * sizeof(T) / (2 * parts) >= 256 * 16) parts *= 2;
  return parts;
}
template <typename T> int fwd_call(const FwdCall<T>& c) {
  const int parts = fwd_parts<T>(c.rows, c.V);
  if (parts == 1) {
    const int threads = team_of(c.V * sizeof(T), c.rows, SUM_TEAMS);
    return threads == 32 ? fwd_rows<T, 32>(c) : threads == 64 ? fwd_rows<T, 64>(c) : threads == 128 ? fwd_rows<T, 128>(c) : fwd_rows<T, 256>(c);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c.rows * parts); cfg.blockDim = dim3(256); cfg.stream = c.s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = bb_back_to_back > 0 ? 2 : 1;
  BB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, token_logprob_fwd_cluster_kernel<T, 256>, c.logits, c.ld, c.targets, c.k, c.logp, c.rest, c.stats, c.V, c.ignore, c.status));
  return BB_OK;
}
int logprob_fwd(const void* logits, int dtype, long long ld, const long long* targets, double scale, float* logp, float* rest, float* stats, long long rows, int vocab,
                long long ignore_index, cudaStream_t s) {
  const K2 k = split_k(scale);
  int* status = bb_device_status_word();
  if (dtype == BB_DTYPE_BF16) return fwd_call<__nv_bfloat16>({(const __nv_bfloat16*)logits, ld, targets, k, logp, rest, (float2*)stats, (int)rows, vocab, ignore_index, status, s});
  return fwd_call<float>({(const float*)logits, ld, targets, k, logp, rest, (float2*)stats, (int)rows, vocab, ignore_index, status, s});
}

template <typename T> struct BwdCall {
  const T* logits; long long ld; const long long* targets; const float2* stats; const float* row_grad; const float* gscale_dev; float gscale; K2 k; T* dlogits;
  long long ldd; int rows, V, cols; long long ignore; const double* pair_loss; int pairs; float* loss; cudaStream_t s;
};
template <typename T, int THREADS> int bwd_rows(const BwdCall<T>& c) {
  BB_CUDA_CHECK(bb_launch(token_logprob_bwd_kernel<T, THREADS>, row_blocks<THREADS>(c.rows), BLOCK<THREADS>, 0, c.s, c.logits, c.ld, c.targets, c.stats, c.row_grad,
                          c.gscale_dev, c.gscale, c.k, c.dlogits, c.ldd, c.rows, c.V, c.cols, c.ignore, c.pair_loss, c.pairs, c.loss));
  return BB_OK;
}
template <typename T> int bwd_call(const BwdCall<T>& c) {
  const size_t bytes = c.V * sizeof(T);
  if (bytes > GRAD_EIGHT && c.rows >= GRAD_EIGHT_ROWS) return bwd_rows<T, 512>(c);
  const int threads = team_of(bytes, c.rows, GRAD_TEAMS);
  return threads == 32 ? bwd_rows<T, 32>(c) : threads == 64 ? bwd_rows<T, 64>(c) : threads == 128 ? bwd_rows<T, 128>(c) : bwd_rows<T, 256>(c);
}
int logprob_bwd(const void* logits, int dtype, long long ld, const long long* targets, double scale, const float* stats, const float* row_grad,
                const float* grad_scale_dev, float grad_scale, void* dlogits, long long ldd, long long rows, int vocab, int cols, long long ignore_index,
                const double* pair_loss, int pairs, float* loss, cudaStream_t s) {
  const K2 k = split_k(scale);
  const float g = (float)(scale * grad_scale);
  if (dtype == BB_DTYPE_BF16)
    return bwd_call<__nv_bfloat16>({(const __nv_bfloat16*)logits, ld, targets, (const float2*)stats, row_grad, grad_scale_dev, g, k, (__nv_bfloat16*)dlogits, ldd, (int)rows,
                                    vocab, cols, ignore_index, pair_loss, pairs, loss, s});
  return bwd_call<float>({(const float*)logits, ld, targets, (const float2*)stats, row_grad, grad_scale_dev, g, k, (float*)dlogits, ldd, (int)rows, vocab, cols, ignore_index,
                          pair_loss, pairs, loss, s});
}

}  // namespace

extern "C" int bb_token_logprob_fwd(const void* logits, int dtype, long long ld, const long long* targets, double scale, float* logp,
                                    float* stats, long long rows, int vocab, long long ignore_index, void* stream) {
  if (bad_logits("bb_token_logprob_fwd", logits, dtype, ld, targets, rows, vocab, scale)) return BB_ERR_INVALID_ARG;
  if (!logp || ((uintptr_t)stats & 7)) return refuse("bb_token_logprob_fwd: logp is needed, and stats 8-byte aligned");
  return logprob_fwd(logits, dtype, ld, targets, scale, logp, nullptr, stats, rows, vocab, ignore_index, (cudaStream_t)stream);
}

extern "C" int bb_token_logprob_bwd(const void* logits, int dtype, long long ld, const long long* targets, double scale, const float* stats,
                                    const float* row_grad, const float* grad_scale_dev, float grad_scale, void* dlogits, long long ldd,
                                    long long rows, int vocab, int cols, long long ignore_index, void* stream) {
  if (bad_logits("bb_token_logprob_bwd", logits, dtype, ld, targets, rows, vocab, scale)) return BB_ERR_INVALID_ARG;
  if (!stats || ((uintptr_t)stats & 7) || !row_grad || bad_output(logits, ld, dlogits, ldd, dtype, rows, vocab, cols))
    return refuse("bb_token_logprob_bwd: null pointer, columns that do not cover the vocabulary, or a gradient that overlaps the logits without being in place");
  return logprob_bwd(logits, dtype, ld, targets, scale, stats, row_grad, grad_scale_dev, grad_scale, dlogits, ldd, rows, vocab, cols, ignore_index, nullptr, 0,
                     nullptr, (cudaStream_t)stream);
}

namespace {
int preference_check(const bb_preference_desc* d, const long long* targets, const long long* offsets, const float* loss, const float* rewards,
                     const void* workspace) {
  if (!d || !targets || !loss || !rewards || !workspace || ((uintptr_t)workspace & 15))
    return refuse("bb_preference_loss: null pointer, or a workspace that is not 16-byte aligned");
  if (d->tokens <= 0 || d->tokens > INT_MAX || d->sequences <= 0 || d->sequences % 2 || (!offsets && d->tokens % d->sequences))
    return refuse("bb_preference_loss: sequences come in pairs, and without offsets all have tokens / sequences tokens");
  if (d->form < BB_PREFERENCE_SIGMOID || d->form > BB_PREFERENCE_SQUARED || !(d->beta > 0.0) || !(d->label_smoothing >= 0.0 && d->label_smoothing <= 1.0))
    return refuse("bb_preference_loss: unknown form, beta that is not positive, or label smoothing outside [0, 1]");
  return BB_OK;
}
int preference_pairs(const bb_preference_desc* d, const float* logp, const float* rest, const float* ref, const long long* targets, const long long* offsets, float* rewards,
                     float* row_grad, double* pair_loss, cudaStream_t s) {
  const int pairs = d->sequences / 2;
  BB_CUDA_CHECK(bb_launch(preference_pair_kernel, pairs, 256, 0, s, logp, rest, ref, targets, offsets, d->tokens / d->sequences, d->tokens, pairs, d->form,
                          d->beta, d->label_smoothing, d->average, d->ignore_index, pair_loss, rewards, row_grad, bb_device_status_word()));
  return BB_OK;
}
}  // namespace

extern "C" int bb_preference_loss(const bb_preference_desc* d, const float* logp, const float* ref, const long long* targets,
                                  const long long* offsets, float* loss, float* rewards, float* row_grad, void* workspace,
                                  long long workspace_bytes, void* stream) {
  if (int rc = preference_check(d, targets, offsets, loss, rewards, workspace)) return rc;
  if (!logp || !row_grad) return refuse("bb_preference_loss: logp and row_grad are needed");
  if (workspace_bytes < bb_preference_workspace_bytes(d)) return refuse("bb_preference_loss: workspace smaller than bb_preference_workspace_bytes()");
  cudaStream_t s = (cudaStream_t)stream;
  double* pair_loss = (double*)workspace;
  BackToBack overlap;
  if (int rc = preference_pairs(d, logp, nullptr, ref, targets, offsets, rewards, row_grad, pair_loss, s)) return rc;
  BB_CUDA_CHECK(bb_launch(preference_mean_kernel, 1, 256, 0, s, (const double*)pair_loss, d->sequences / 2, loss));
  return BB_OK;
}

extern "C" int bb_preference_loss_logits(const bb_preference_desc* d, const void* logits, int dtype, long long ld, double scale, int vocab, int cols,
                                         const float* ref, const long long* targets, const long long* offsets, float* loss, float* rewards,
                                         float* stats, float* row_grad, void* dlogits, long long ldd, float grad_scale, void* workspace, long long workspace_bytes, void* stream) {
  if (int rc = preference_check(d, targets, offsets, loss, rewards, workspace)) return rc;
  if (bad_logits("bb_preference_loss_logits", logits, dtype, ld, targets, d->tokens, vocab, scale)) return BB_ERR_INVALID_ARG;
  if ((uintptr_t)stats & 7) return refuse("bb_preference_loss_logits: stats 8-byte aligned");
  if (dlogits && bad_output(logits, ld, dlogits, ldd, dtype, d->tokens, vocab, cols))
    return refuse("bb_preference_loss_logits: columns that do not cover the vocabulary, or a gradient that overlaps the logits without being in place");
  if (workspace_bytes < bb_preference_workspace_bytes(d)) return refuse("bb_preference_loss_logits: workspace smaller than bb_preference_workspace_bytes()");
  cudaStream_t s = (cudaStream_t)stream;
  // pair losses | softmax sums | log-probabilities | what their rounding left out | row gradients
  double* pair_loss = (double*)workspace;
  float* ws = (float*)(pair_loss + d->sequences / 2);
  float *logp = ws + 2 * d->tokens, *rest = logp + d->tokens;
  if (!stats) stats = ws;
  if (!row_grad) row_grad = rest + d->tokens;
  BackToBack overlap;
  if (int rc = logprob_fwd(logits, dtype, ld, targets, scale, logp, rest, stats, d->tokens, vocab, d->ignore_index, s)) return rc;
  if (int rc = preference_pairs(d, logp, rest, ref, targets, offsets, rewards, row_grad, pair_loss, s)) return rc;
  if (!dlogits) {
    BB_CUDA_CHECK(bb_launch(preference_mean_kernel, 1, 256, 0, s, (const double*)pair_loss, d->sequences / 2, loss));
    return BB_OK;
  }
  return logprob_bwd(logits, dtype, ld, targets, scale, stats, row_grad, nullptr, grad_scale, dlogits, ldd, d->tokens, vocab, cols, d->ignore_index, pair_loss,
                     d->sequences / 2, loss, s);
}
extern "C" long long bb_preference_workspace_bytes(const bb_preference_desc* d) {
  return d && d->sequences > 0 && d->tokens > 0 ? (long long)d->sequences * 4 + 8 + 20 * d->tokens : -1;
}

namespace {
int policy_check(const bb_policy_desc* d, const long long* targets, const long long* offsets, const float* advantages, const float* loss,
                 const float* stats, const void* workspace) {
  if (!d || !targets || !advantages || !loss || !stats || !workspace || ((uintptr_t)workspace & 15))
    return refuse("bb_policy_loss: null pointer, or a workspace that is not 16-byte aligned");
  if (d->tokens <= 0 || d->tokens > INT_MAX || d->sequences <= 0 || (!offsets && d->tokens % d->sequences))
    return refuse("bb_policy_loss: sizes have to be positive, and without offsets all sequences have tokens / sequences tokens");
  if (d->advantage_per_sequence && offsets) return refuse("bb_policy_loss: advantages per sequence go with sequences of one length");
  if (!(d->clip_low >= 0.0) || !(d->clip_high >= 0.0) || !(d->kl_coef >= 0.0) || (d->reduction != BB_POLICY_TOKEN && d->reduction != BB_POLICY_SEQUENCE))
    return refuse("bb_policy_loss: clipping bounds and the KL weight cannot be negative, the reduction is by token or by sequence");
  return BB_OK;
}
// Counts of counted tokens and weights into the workspace, and what the token functions take
int policy_front(const bb_policy_desc* d, const PolicyPlan& pl, const long long* targets, const long long* offsets, const float* old_logp,
                 const float* advantages, const float* ref, void* workspace, PolicyParams& p, cudaStream_t s) {
  char* ws = (char*)workspace;
  const bool by_sequence = d->reduction == BB_POLICY_SEQUENCE;
  int* counts = (int*)ws;
  float* weight = by_sequence ? (float*)(ws + pl.weight_at) : nullptr;
  const long long seq_len = d->tokens / d->sequences;
  p.old_logp = old_logp; p.advantages = advantages; p.ref = ref; p.weight = weight; p.counts = counts; p.num_counts = pl.num_counts;
  p.adv_div = d->advantage_per_sequence ? seq_len : 1;
  p.low = (float)(1.0 - d->clip_low); p.high = (float)(1.0 + d->clip_high); p.kl_coef = ref ? (float)d->kl_coef : 0.f;
  BB_CUDA_CHECK(bb_launch(policy_count_kernel, pl.num_counts, 256, 0, s, targets, offsets, by_sequence ? seq_len : pl.piece, d->tokens, d->ignore_index,
                          counts, weight, bb_device_status_word()));
  return BB_OK;
}
}  // namespace

namespace {
struct PolicyRowCall {
  long long ld; const long long* targets; PolicyParams p; K2 k; float gscale; long long ldd; int V, cols; long long ignore_index;
  PolicyRow* row_sums; int* status; int rows; int* ticket; cudaStream_t stream;
};
template <typename T, int THREADS> int policy_rows_as(const T* logits, T* dlogits, const PolicyRowCall& c) {
  BB_CUDA_CHECK(bb_launch(policy_row_kernel<T, THREADS>, row_blocks<THREADS>(c.rows), BLOCK<THREADS>, 0, c.stream, logits, c.ld, c.targets, c.p, c.k, c.gscale, dlogits, c.ldd, c.rows, c.V, c.cols,
                          c.ignore_index, c.row_sums, c.status));
  return BB_OK;
}
template <typename T> int policy_rows(const T* logits, T* dlogits, const PolicyRowCall& c) {
  const size_t bytes = (size_t)c.V * sizeof(T);
  if (bytes <= LONG_ROW<T>) {
    const int threads = team_of(bytes, c.rows, POLICY_TEAMS);
    return threads == 32 ? policy_rows_as<T, 32>(logits, dlogits, c) : threads == 64 ? policy_rows_as<T, 64>(logits, dlogits, c)
         : threads == 128 ? policy_rows_as<T, 128>(logits, dlogits, c) : policy_rows_as<T, 256>(logits, dlogits, c);
  }
  const size_t smem = bytes / 16 * 16;
  const int stages = (int)((smem + RING_STAGE - 1) / RING_STAGE);
  if (smem > MAX_RING) return policy_rows_as<T, 512>(logits, dlogits, c);
  BB_ONCE_PER_DEVICE(BB_CUDA_CHECK(cudaFuncSetAttribute(policy_ring_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_RING)));
  // as many CTAs as the machine holds
  const int per_sm = smem <= PAIR_RING ? 2 : 1, most = per_sm * bb_num_sms();
  BB_CUDA_CHECK(bb_launch(policy_ring_kernel<T>, c.rows < most ? c.rows : most, RING_THREADS + 32, smem, c.stream, logits, c.ld, c.targets, c.p, c.k, c.gscale, dlogits,
                          c.ldd, c.rows, c.V, c.cols, c.ignore_index, c.row_sums, c.status, stages, c.ticket));
  return BB_OK;
}
template <bool FROM_ROWS>
int policy_tokens(const bb_policy_desc* d, const PolicyPlan& pl, float* logp, K2 k, const long long* targets, const PolicyParams& p, float* row_grad, float* loss,
                  float* stats, void* workspace, cudaStream_t s) {
  char* ws = (char*)workspace;
  BB_CUDA_CHECK(bb_launch(policy_token_kernel<FROM_ROWS>, policy_token_ctas(d->tokens), 256, 0, s, logp, (const PolicyRow*)(ws + pl.rows_at), k, targets, p, d->tokens,
                          d->ignore_index, row_grad, (double*)(ws + pl.partial_at), (int*)ws + pl.num_counts + 1, loss, stats));
  return BB_OK;
}
}  // namespace

extern "C" long long bb_policy_workspace_bytes(const bb_policy_desc* d) {
  if (!d || d->tokens <= 0 || d->sequences <= 0) return -1;
  return (long long)policy_plan(d->tokens, d->sequences, d->reduction == BB_POLICY_SEQUENCE).bytes;
}

extern "C" int bb_policy_loss(const bb_policy_desc* d, const float* logp, const float* old_logp, const float* advantages, const float* ref,
                              const long long* targets, const long long* offsets, float* loss, float* stats, float* row_grad,
                              void* workspace, long long workspace_bytes, void* stream) {
  if (int rc = policy_check(d, targets, offsets, advantages, loss, stats, workspace)) return rc;
  if (!logp || !row_grad) return refuse("bb_policy_loss: logp and row_grad are needed");
  if (workspace_bytes < bb_policy_workspace_bytes(d)) return refuse("bb_policy_loss: workspace smaller than bb_policy_workspace_bytes()");
  cudaStream_t s = (cudaStream_t)stream;
  const PolicyPlan pl = policy_plan(d->tokens, d->sequences, d->reduction == BB_POLICY_SEQUENCE);
  PolicyParams p;
  BackToBack overlap;
  if (int rc = policy_front(d, pl, targets, offsets, old_logp, advantages, ref, workspace, p, s)) return rc;
  return policy_tokens<false>(d, pl, const_cast<float*>(logp), K2{}, targets, p, row_grad, loss, stats, workspace, s);
}

extern "C" int bb_policy_loss_logits(const bb_policy_desc* d, const void* logits, int dtype, long long ld, double scale, int vocab, int cols,
                                     const float* old_logp, const float* advantages, const float* ref, const long long* targets,
                                     const long long* offsets, float* loss, float* stats, float* logp, void* dlogits, long long ldd,
                                     float grad_scale, void* workspace, long long workspace_bytes, void* stream) {
  if (int rc = policy_check(d, targets, offsets, advantages, loss, stats, workspace)) return rc;
  if (bad_logits("bb_policy_loss_logits", logits, dtype, ld, targets, d->tokens, vocab, scale)) return BB_ERR_INVALID_ARG;
  if (bad_output(logits, ld, dlogits, ldd, dtype, d->tokens, vocab, cols))
    return refuse("bb_policy_loss_logits: columns that do not cover the vocabulary, or a gradient that overlaps the logits without being in place");
  if (workspace_bytes < bb_policy_workspace_bytes(d)) return refuse("bb_policy_loss_logits: workspace smaller than bb_policy_workspace_bytes()");
  cudaStream_t s = (cudaStream_t)stream;
  const PolicyPlan pl = policy_plan(d->tokens, d->sequences, d->reduction == BB_POLICY_SEQUENCE);
  const K2 k = split_k(scale);
  const float g = (float)(scale * grad_scale);
  int* status = bb_device_status_word();
  PolicyParams p;
  BackToBack overlap;
  if (int rc = policy_front(d, pl, targets, offsets, old_logp, advantages, ref, workspace, p, s)) return rc;
  const PolicyRowCall c = {ld, targets, p, k, g, ldd, vocab, cols, d->ignore_index, (PolicyRow*)((char*)workspace + pl.rows_at), status, (int)d->tokens, (int*)workspace + pl.num_counts, s};
  if (int rc = dtype == BB_DTYPE_BF16 ? policy_rows((const __nv_bfloat16*)logits, (__nv_bfloat16*)dlogits, c) : policy_rows((const float*)logits, (float*)dlogits, c))
    return rc;
  return policy_tokens<true>(d, pl, logp, k, targets, p, nullptr, loss, stats, workspace, s);
}

extern "C" int bb_rescale_grad(void* grad, int dtype, long long ld, long long rows, int cols, const float* upstream, float made_for, void* stream) {
  if (!grad || !upstream || rows <= 0 || rows > INT_MAX || cols <= 0 || ld < cols || made_for == 0.f || (dtype != BB_DTYPE_BF16 && dtype != BB_DTYPE_F32) ||
      ((uintptr_t)grad & (dtype == BB_DTYPE_F32 ? 3 : 1)))
    return refuse("bb_rescale_grad: null or misaligned pointer, a size that is not positive, an unknown type, or made_for = 0");
  if (dtype == BB_DTYPE_BF16)
    BB_CUDA_CHECK(bb_launch(rescale_kernel<__nv_bfloat16>, (int)rows, RESCALE_THREADS, 0, (cudaStream_t)stream, (__nv_bfloat16*)grad, ld, cols, upstream, made_for));
  else
    BB_CUDA_CHECK(bb_launch(rescale_kernel<float>, (int)rows, RESCALE_THREADS, 0, (cudaStream_t)stream, (float*)grad, ld, cols, upstream, made_for));
  return BB_OK;
}

// workspace: sum of squares | coefficient | sums of the CTAs
extern "C" long long bb_grad_norm_workspace_bytes(void) { return 8LL * (2 + NORM_CTAS); }

namespace {
// Sum of squares of the list into the workspace's first value
int list_sumsq(const bb_grad_tensor* tensors, int count, double* workspace, cudaStream_t s, const ClipTo& clip = {}, bool add = false) {
  for (int at = 0; at < count; at += LIST_TENSORS) {
    const int n = count - at < LIST_TENSORS ? count - at : LIST_TENSORS;
    TensorTable t;
    const int pieces = table_fill(t, tensors + at, n, sum_piece(tensors + at, n));
    unsigned int* done = norm_done(s);
    if (!done) { bb_set_last_error_msg("bb_grad_sumsq: counters unavailable on this device"); return BB_ERR_CUDA; }
    BB_CUDA_CHECK(bb_launch(grad_sumsq_kernel, pieces < NORM_CTAS ? pieces : NORM_CTAS, NORM_THREADS, 0, s, t, workspace + 2, workspace, add || at > 0 ? 1 : 0, done,
                            at + n < count ? ClipTo{} : clip));
  }
  return BB_OK;
}
// The coefficient, from a sum that is there or from the list's own
int clip_front(const bb_grad_tensor* tensors, int count, const double* sumsq, double* workspace, const ClipTo& clip, cudaStream_t s) {
  if (!sumsq) return list_sumsq(tensors, count, workspace, s, clip);
  BB_CUDA_CHECK(bb_launch(clip_coef_kernel, 1, 1, 0, s, sumsq, clip));
  return BB_OK;
}
bool bad_workspace(const void* workspace, long long bytes) { return !workspace || ((uintptr_t)workspace & 7) || bytes < bb_grad_norm_workspace_bytes(); }
}  // namespace

// The clipping coefficient for a list of parameters (bb_adamw_list): into the workspace's second value
int bb_list_clip_coef(const bb_adamw_tensor* tensors, int count, const double* sumsq, double grad_scale, double max_norm, float* norm, void* workspace,
                      cudaStream_t s) {
  double* ws = (double*)workspace;
  const ClipTo clip = {grad_scale, max_norm, (float*)(ws + 1), norm};
  if (sumsq) return clip_front(nullptr, 0, sumsq, ws, clip, s);
  for (int at = 0; at < count; at += LIST_TENSORS) {
    bb_grad_tensor list[LIST_TENSORS];
    const int n = count - at < LIST_TENSORS ? count - at : LIST_TENSORS;
    for (int i = 0; i < n; ++i) list[i] = {tensors[at + i].grad, tensors[at + i].numel, tensors[at + i].grad_dtype};
    if (int rc = list_sumsq(list, n, ws, s, at + n < count ? ClipTo{} : clip, at > 0)) return rc;
  }
  return BB_OK;
}

extern "C" int bb_grad_sumsq(const bb_grad_tensor* tensors, int count, void* workspace, long long workspace_bytes, void* stream) {
  if (bad_list(tensors, count) || bad_workspace(workspace, workspace_bytes))
    return refuse("bb_grad_sumsq: an empty tensor, a type other than bf16 and fp32, or a workspace smaller than bb_grad_norm_workspace_bytes()");
  return list_sumsq(tensors, count, (double*)workspace, (cudaStream_t)stream);
}

extern "C" int bb_grad_clip(const bb_grad_tensor* tensors, int count, const double* sumsq, double max_norm, float* norm, void* workspace,
                            long long workspace_bytes, void* stream) {
  if (bad_list(tensors, count) || !norm || !(max_norm > 0.0) || bad_workspace(workspace, workspace_bytes))
    return refuse("bb_grad_clip: an empty tensor, a type other than bf16 and fp32, a norm that is not positive, or a workspace that is too small");
  BackToBack overlap;
  float* coef = (float*)((double*)workspace + 1);
  if (int rc = clip_front(tensors, count, sumsq, (double*)workspace, {1.0, max_norm, coef, norm}, (cudaStream_t)stream)) return rc;
  for (int at = 0; at < count; at += LIST_TENSORS) {
    TensorTable t;
    const int pieces = table_fill(t, tensors + at, count - at < LIST_TENSORS ? count - at : LIST_TENSORS, CLIP_PIECE);
    BB_CUDA_CHECK(bb_launch(grad_clip_kernel, pieces, NORM_THREADS, 0, (cudaStream_t)stream, t, (const float*)coef));
  }
  return BB_OK;
}

extern "C" int bb_adam_step_clipped(float* master, float* grad, float* exp_avg, float* exp_avg_sq, void* param_bf16, long long n, double lr,
                                    double beta1, double beta2, double eps, int step, int adam_w_mode, int bias_correction,
                                    double weight_decay, double grad_scale, int zero_grad, const double* sumsq, double max_norm,
                                    float* norm, void* workspace, long long workspace_bytes, void* stream) {
  if (!master || !grad || !exp_avg || !exp_avg_sq || n <= 0 || (n & 3) || step < 1 || bad_workspace(workspace, workspace_bytes) || !norm || !(max_norm > 0.0) ||
      (((uintptr_t)master | (uintptr_t)grad | (uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) || ((uintptr_t)param_bf16 & 7))
    return refuse("bb_adam_step_clipped: null or unaligned pointer, n not a multiple of 4, step < 1, a norm that is not positive, or a workspace that is too small");
  AdamParams a;
  a.lr = (float)lr; a.b1 = (float)beta1; a.omb1 = (float)(1.0 - beta1); a.b2 = (float)beta2; a.omb2 = (float)(1.0 - beta2); a.eps = (float)eps;
  a.inv_bc1 = bias_correction ? (float)(1.0 / (1.0 - pow(beta1, step))) : 1.f;
  a.inv_bc2 = bias_correction ? (float)(1.0 / (1.0 - pow(beta2, step))) : 1.f;
  a.decay = (float)weight_decay; a.decoupled = adam_w_mode ? 1 : 0; a.zero_grad = zero_grad;
  BackToBack overlap;
  const bb_grad_tensor t = {grad, n, BB_DTYPE_F32};
  float* coef = (float*)((double*)workspace + 1);
  if (int rc = clip_front(&t, 1, sumsq, (double*)workspace, {grad_scale, max_norm, coef, norm}, (cudaStream_t)stream)) return rc;
  const long long ctas = ((n >> 2) + 255) / 256;
  if (ctas > INT_MAX) return refuse("bb_adam_step_clipped: more elements than one launch covers");
  BB_CUDA_CHECK(bb_launch(adam_clip_kernel, (int)ctas, 256, 0, (cudaStream_t)stream, master, grad, exp_avg, exp_avg_sq, (__nv_bfloat16*)param_bf16, n, a,
                          (const float*)coef, (float)grad_scale));
  return BB_OK;
}
