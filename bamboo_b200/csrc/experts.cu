// Routing of tokens to experts and the way of their rows there and back (declarations and formulas in bamboo_b200.h).
//
// Every operator here is bound by memory, and for a few thousand tokens by its launches.  Nothing depends on the order in which CTAs run:
// places are counted and not drawn, sums are taken in one order.
#include "common.cuh"
#include "bamboo_b200.h"
#include <limits.h>
#include <stdio.h>

namespace {

int refuse(const char* msg) { bb_set_last_error_msg(msg); return BB_ERR_INVALID_ARG; }

__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_value(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// ------------------------------------------------------------------ routing
constexpr int MAX_EXPERTS = 256, MAX_CHOSEN = 32;
constexpr int ROUTE_WARPS = 32, ROUTE_THREADS = 32 * ROUTE_WARPS;
constexpr int BWD_WARPS = 8;
constexpr int WIDEST = INT_MAX - 4096;                // values of a row are counted in 32 bits, up to some thousand beyond the last

struct RouteParams {
  int tokens, experts, k, normalize;
  long long ld;
  int vec;                      // rows can be read in runs of a lane's logits
  int chunk, blocks;            // consecutive tokens of a block, blocks
  float* weights; int* chosen; int* rows; int* slots; int* offsets; float* balance; float2* stats; float* load;
  int* counts;                  // [blocks][experts + 1]: slots of every expert, tokens that have any
  float* probs;                 // [blocks][experts]: sums of softmax
};

// A lane's PER consecutive logits (-inf behind the last)
template <typename T, int PER> __device__ __forceinline__ void load_run(const T* row, int first, int n, int vec, float* x) {
  if (vec) {
    if (first < n) {
      constexpr int BYTES = PER * sizeof(T);
      alignas(16) T v[PER];
      if constexpr (BYTES >= 16) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(row + first)[i];
      } else if constexpr (BYTES == 8) {
        *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(row + first);
      } else if constexpr (BYTES == 4) {
        *reinterpret_cast<uint32_t*>(v) = *reinterpret_cast<const uint32_t*>(row + first);
      } else {
        v[0] = row[first];
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = first + i < n ? value_of(v[i]) : -INFINITY;         // (a run may go on into the padding)
      return;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = -INFINITY;
    return;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = first + i < n ? value_of(row[first + i]) : -INFINITY;
}

// A logit as a number whose order is that of the choice: NaN above all, 0 for what is never chosen (-inf), both zeros alike
__device__ __forceinline__ uint32_t choice_key(float x) {
  if (x != x) return 0xffffffffu;
  if (x == -INFINITY) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// One instruction each besides a product: arguments are at most 0 where it matters (a probability of e^-30 is off by 2e-6 of itself), and quotients within
// 2^-22.  The instructions of these kernels are what bounds them.
__device__ __forceinline__ float exp_fast(float x) { return __expf(x); }
__device__ __forceinline__ float over(float v) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// A lane's logits in the order of the choice, the first in front, their numbers (0 .. PER - 1) in the bytes of `which`
template <int PER> __device__ __forceinline__ void sort_keys(uint32_t* key, uint64_t& which) {
  uint32_t at[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) at[i] = i;
  // (a key moves in front of another only where it is larger: equal ones keep their order)
#pragma unroll
  for (int i = 1; i < PER; ++i)
#pragma unroll
    for (int j = i; j > 0; --j) {
      const bool swap = key[j] > key[j - 1];
      const uint32_t a = key[j], b = at[j];
      key[j] = swap ? key[j - 1] : a; at[j] = swap ? at[j - 1] : b;
      key[j - 1] = swap ? a : key[j - 1]; at[j - 1] = swap ? b : at[j - 1];
    }
  which = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) which |= (uint64_t)at[i] << (8 * i);
}

// Over the G lanes that share a token
template <int G> __device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int d = G / 2; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
template <int G> __device__ __forceinline__ uint32_t team_max(uint32_t v) {
  if constexpr (G == 32) {
    v = __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int d = G / 2; d; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  }
  return v;
}

// Where every expert's places begin, from how many it has; by one warp
__device__ __forceinline__ void places_of(const int* total, int* base, int n, int lane) {
  int carry = 0;
  for (int at = 0; at < n; at += 32) {
    const int e = at + lane, c = e < n ? total[e] : 0;
    int v = c;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    if (e < n) base[e] = carry + v - c;
    carry += __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) base[n] = carry;
}
// Offsets, shares and the balance term, by a block; `sum` is the e-th thread's sum of softmax
__device__ __forceinline__ void put_shares(const RouteParams& p, const int* total, const int* base, double* part, double sum) {
  const int n = p.experts, e = threadIdx.x, lane = threadIdx.x & 31, tokens = max(total[n], 1), places = max(base[n], 1);
  if (e < n) {
    p.offsets[e] = base[e];
    p.load[e] = (float)total[e] / (float)places;
    part[e] = (double)total[e] * sum;
  }
  if (e == 0) { p.offsets[n] = base[n]; p.load[n] = (float)tokens; }
  __syncthreads();
  if (e < 32) {
    double all = 0.0;
    for (int i = lane; i < n; i += 32) all += part[i];
#pragma unroll
    for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
    if (lane == 0) p.balance[0] = (float)(n * all / ((double)places * (double)tokens));
  }
}

// A team of G lanes per token (8, 16 or the warp, 32 / G tokens at a time), PER consecutive logits a lane, sorted; k rounds of a team-wide maximum, which goes
// to the first lane that has it in front, the j-th choice to lane j.  Then the block's slots are ranked within their experts, in order: every warp counts a run of
// them, and ranks it behind the runs before.  Instructions bound it: both kernels, us, 65536 tokens, 2 of 8 experts 17 (a warp per token 36), 6 of 64 34 (64);
// 32768, 8 of 128 33 (with two tokens a warp and 8 logits a lane 32: sorting them costs what the rounds save).
// A block per SM with all its warps: few blocks, because each adds up the counts of all others in the next kernel.
template <typename T, int PER, int G>
__global__ void __launch_bounds__(ROUTE_THREADS)
route_choose_kernel(const T* logits, const RouteParams p) {
  constexpr int S = 32 / G;
  extern __shared__ int shared[];
  int* hist = shared;                                                        // [ROUTE_WARPS][experts]
  float* sums = reinterpret_cast<float*>(shared + ROUTE_WARPS * p.experts);  // [ROUTE_WARPS][experts]
  __shared__ int some_tokens, total_of[MAX_EXPERTS + 1], base[MAX_EXPERTS + 1];
  __shared__ double part[MAX_EXPERTS];
  const bool alone = p.blocks == 1;          // a block that has all tokens places them too
  bb::pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = p.experts, seat = lane & (G - 1), first = seat * PER;
  const unsigned team = G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1) << (lane & ~(G - 1));
  const int t0 = blockIdx.x * p.chunk, t1 = min(p.tokens, t0 + p.chunk);
  for (int i = threadIdx.x; i < ROUTE_WARPS * n; i += ROUTE_THREADS) hist[i] = 0;
  if (threadIdx.x == 0) some_tokens = 0;
  float prob[PER] = {};
  int some = 0;
  float x[PER];
  auto load = [&](int t) {
    if (t < t1) {
      load_run<T, PER>(logits + (long long)t * p.ld, first, n, p.vec, x);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = -INFINITY;
    }
  };
  int t = t0 + warp * S + lane / G;
  load(t);
  for (; t - lane / G < t1; t += ROUTE_WARPS * S) {
    uint32_t key[PER];
    float own[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) { key[i] = choice_key(x[i]); own[i] = x[i]; }
    load(t + ROUTE_WARPS * S);           // the next token's
    int mine = -1;
    uint32_t value = 0;
    uint64_t which;
    sort_keys<PER>(key, which);
    for (int j = 0; j < p.k; ++j) {
      const uint32_t top = team_max<G>(key[0]);
      const int from = __ffs(__ballot_sync(0xffffffffu, key[0] == top) & team) - 1;
      const int at = __shfl_sync(0xffffffffu, first + (int)(which & 0xff), from);
      if (seat == j && top != 0) { mine = at; value = top; }
      if (lane == from) {
#pragma unroll
        for (int i = 0; i + 1 < PER; ++i) key[i] = key[i + 1];
        key[PER - 1] = 0;
        which >>= 8;
      }
    }
    const uint32_t best = __shfl_sync(0xffffffffu, value, lane & ~(G - 1));          // 0: nothing to choose
    const bool any = best != 0;
    const float top = any ? key_value(best) : 0.f;
    float e[PER], sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      e[i] = any && first + i < n ? exp_fast(own[i] - top) : 0.f;
      sum += e[i];
    }
    sum = team_sum<G>(sum);
    const float share = mine >= 0 ? exp_fast(key_value(value) - top) : 0.f, each = over(sum);
    const float scale = p.normalize ? over(team_sum<G>(share)) : each;
    if (t >= t1) continue;               // (a whole team; nothing below is done together)
    const long long s = (long long)t * p.k + seat;
    if (seat < p.k) {
      p.chosen[s] = mine;
      p.weights[s] = mine >= 0 ? share * scale : 0.f;
    }
    if (seat == 0) p.stats[t] = make_float2(top, sum);
    if (any) {
      ++some;
#pragma unroll
      for (int i = 0; i < PER; ++i) prob[i] = fmaf(e[i], each, prob[i]);
    }
  }
  __syncwarp();
#pragma unroll
  for (int d = G; d < 32; d <<= 1) {
#pragma unroll
    for (int i = 0; i < PER; ++i) prob[i] += __shfl_xor_sync(0xffffffffu, prob[i], d);
    some += __shfl_xor_sync(0xffffffffu, some, d);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) if (lane < G && first + i < n) sums[warp * n + first + i] = prob[i];
  __syncthreads();
  if (lane == 0 && some) atomicAdd(&some_tokens, some);
  const int k = p.k, slot0 = t0 * k, count = (t1 - t0) * k;
  const int run = (count + 32 * ROUTE_WARPS - 1) / (32 * ROUTE_WARPS) * 32, a = min(count, warp * run), b = min(count, a + run);
  int* mine = hist + warp * n;
  for (int i = a + lane; i - lane < b; i += 32) {
    const int e = i < b ? p.chosen[slot0 + i] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && (same & ((1u << lane) - 1)) == 0) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  float mass = 0.f;
  if (threadIdx.x < n) {
    const int e = threadIdx.x;
    int total = 0;
#pragma unroll 8
    for (int w = 0; w < ROUTE_WARPS; ++w) { const int c = hist[w * n + e]; hist[w * n + e] = total; total += c; mass += sums[w * n + e]; }
    if (alone) {
      total_of[e] = total;
    } else {
      p.counts[(long long)blockIdx.x * (n + 1) + e] = total;
      p.probs[(long long)blockIdx.x * n + e] = mass;
    }
  }
  if (threadIdx.x == 0) {
    total_of[n] = some_tokens;
    if (!alone) p.counts[(long long)blockIdx.x * (n + 1) + n] = some_tokens;
  }
  __syncthreads();
  if (alone) {
    if (warp == 0) places_of(total_of, base, n, lane);
    __syncthreads();
  }
  for (int i = a + lane; i - lane < b; i += 32) {
    const int e = i < b ? p.chosen[slot0 + i] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const unsigned before = same & ((1u << lane) - 1);
    int at = 0;
    if (e >= 0) at = mine[e];
    __syncwarp();
    if (e >= 0 && before == 0) mine[e] = at + __popc(same);
    if (i < b) {
      const int place = e < 0 ? -1 : at + __popc(before) + (alone ? base[e] : 0);
      p.rows[slot0 + i] = place;
      if (alone && place >= 0) p.slots[place] = i;
    }
    __syncwarp();
  }
  if (alone) {
    for (int r = base[n] + threadIdx.x; r < count; r += ROUTE_THREADS) p.slots[r] = -1;
    put_shares(p, total_of, base, part, (double)mass);
  }
}

// Every block adds up what stands before its slots (the counts of all blocks, once more each) and places them; one more block makes what there is one of.
__global__ void __launch_bounds__(ROUTE_THREADS)
route_place_kernel(const RouteParams p) {
  __shared__ int total[MAX_EXPERTS + 1], before[MAX_EXPERTS + 1], base[MAX_EXPERTS + 1];
  __shared__ float mass[ROUTE_THREADS];
  __shared__ double part[MAX_EXPERTS];
  const bool extra = (int)blockIdx.x == p.blocks;
  bb::pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = p.experts, width = n + 1;
  for (int e = threadIdx.x; e < width; e += ROUTE_THREADS) { total[e] = 0; before[e] = 0; }
  __syncthreads();
  const int groups = ROUTE_THREADS / width, g = threadIdx.x / width, e0 = threadIdx.x - g * width;
  if (g < groups) {
    int all = 0, ahead = 0;
#pragma unroll 8
    for (int b = g; b < p.blocks; b += groups) {
      const int c = p.counts[(long long)b * width + e0];
      all += c;
      if (b < (int)blockIdx.x) ahead += c;
    }
    atomicAdd(&total[e0], all);
    atomicAdd(&before[e0], ahead);
  }
  __syncthreads();
  if (warp == 0) places_of(total, base, n, lane);
  __syncthreads();
  const int routed = base[n];
  if (!extra) {
    const int k = p.k, t0 = blockIdx.x * p.chunk, t1 = min(p.tokens, t0 + p.chunk), all = p.tokens * k;
    for (int i = t0 * k + threadIdx.x; i < t1 * k; i += ROUTE_THREADS) {
      const int e = p.chosen[i];
      if (e >= 0) {
        const int at = base[e] + before[e] + p.rows[i];
        p.rows[i] = at;
        p.slots[at] = i;
      }
    }
    for (long long r = (long long)routed + blockIdx.x * ROUTE_THREADS + threadIdx.x; r < all; r += (long long)p.blocks * ROUTE_THREADS) p.slots[r] = -1;
    return;
  }
  // sums of softmax: blocks b = g, g + groups, ... by one thread, then the threads of an expert in their order
  const int teams = ROUTE_THREADS / n, team = threadIdx.x / n, e = threadIdx.x - team * n;
  float m = 0.f;
  if (team < teams) {
#pragma unroll 8
    for (int b = team; b < p.blocks; b += teams) m += p.probs[(long long)b * n + e];
  }
  mass[threadIdx.x] = m;
  __syncthreads();
  double sum = 0.0;
  if (threadIdx.x < n) for (int i = 0; i < teams; ++i) sum += (double)mass[i * n + threadIdx.x];
  put_shares(p, total, base, part, sum);
}

// A lane's run in shared memory (on its size, 16 bytes at most)
template <int PER> __device__ __forceinline__ void put_run(float* to, const float* v) {
  if constexpr (PER >= 4) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) *reinterpret_cast<float4*>(to + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else if constexpr (PER == 2) {
    *reinterpret_cast<float2*>(to) = make_float2(v[0], v[1]);
  } else {
    to[0] = v[0];
  }
}
template <int PER> __device__ __forceinline__ void get_run(const float* from, float* v) {
  if constexpr (PER >= 4) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) { const float4 q = *reinterpret_cast<const float4*>(from + i); v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w; }
  } else if constexpr (PER == 2) {
    const float2 q = *reinterpret_cast<const float2*>(from);
    v[0] = q.x; v[1] = q.y;
  } else {
    v[0] = from[0];
  }
}

// dx_e = p_e (c_e - sum p c) + what arrives through the weights; a team of lanes per token as above.  What arrives goes to the lanes that own the experts
// through shared memory.
template <typename T, int PER, int G>
__global__ void __launch_bounds__(32 * BWD_WARPS)
route_bwd_kernel(const T* logits, const RouteParams p, const float* d_weights, const float* d_balance, T* out, long long ldd, int cols, int vec_out) {
  __shared__ alignas(16) float arrived[BWD_WARPS][32 * PER];
  bb::pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = p.experts, seat = lane & (G - 1), first = seat * PER;
  const int t = blockIdx.x * (BWD_WARPS * (32 / G)) + threadIdx.x / G;
  const bool there = t < p.tokens;
  float* mail = arrived[warp] + lane / G * (G * PER);
  const float g = d_balance ? d_balance[0] * (float)n / p.load[n] : 0.f;
  const long long s = (long long)t * p.k + seat;
  int mine = there && seat < p.k ? p.chosen[s] : -1;
  if (mine >= n) mine = -1;
  const float2 st = there ? p.stats[t] : make_float2(0.f, 1.f);
  float x[PER], push[PER], d[PER];
  if (there) {
    load_run<T, PER>(logits + (long long)t * p.ld, first, n, p.vec, x);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) push[i] = d_balance && first + i < n ? g * p.load[first + i] : 0.f;
  const float dw = mine >= 0 && d_weights ? d_weights[s] : 0.f;
  const bool any = __shfl_sync(0xffffffffu, mine, lane & ~(G - 1)) >= 0;
  const float scale = over(st.y);
  float prob[PER], mean = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    x[i] = first + i < n ? exp_fast(x[i] - st.x) : 0.f;
    prob[i] = x[i] * scale;
    mean = fmaf(prob[i], push[i], mean);
    d[i] = 0.f;
  }
  put_run<PER>(mail + first, x);
  __syncwarp();
  float w = mine >= 0 ? mail[mine] : 0.f;          // the chosen ones' exponentials come back the way their gradients go
  w *= p.normalize ? over(team_sum<G>(w)) : scale;
  if (mine < 0) w = 0.f;
  const float through = team_sum<G>(w * dw);
  if (d_balance) mean = team_sum<G>(mean);
  __syncwarp();
  put_run<PER>(mail + first, d);
  __syncwarp();
  if (mine >= 0) mail[mine] = p.normalize ? w * (dw - through) : w * dw;
  __syncwarp();
  if (!there) return;
  const float off = p.normalize ? mean : mean + through;
  get_run<PER>(mail + first, d);
#pragma unroll
  for (int i = 0; i < PER; ++i) d[i] = any ? fmaf(prob[i], push[i] - off, d[i]) : 0.f;
  T* to = out + (long long)t * ldd;
  if (vec_out) {
    if (first < n) {
      alignas(16) T v[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) put_value(&v[i], d[i]);
      constexpr int BYTES = PER * sizeof(T);
      if constexpr (BYTES >= 16) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(to + first)[i] = reinterpret_cast<uint4*>(v)[i];
      } else if constexpr (BYTES == 8) {
        *reinterpret_cast<uint2*>(to + first) = *reinterpret_cast<uint2*>(v);
      } else if constexpr (BYTES == 4) {
        *reinterpret_cast<uint32_t*>(to + first) = *reinterpret_cast<uint32_t*>(v);
      } else {
        to[first] = v[0];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) if (first + i < n) put_value(to + first + i, d[i]);
  }
  for (int c = n + seat; c < cols; c += G) put_value(to + c, 0.f);
}

// ------------------------------------------------------------------ rows there and back
// A team of threads per row (a warp, eight rows to a block; or a whole block where rows are long), 16 bytes at a time where
// pointers and strides allow it.
template <typename T, int BYTES> struct Pack;
template <> struct Pack<float, 16> {
  static constexpr int N = 4;
  typedef float4 raw;
  static __device__ __forceinline__ void get(const float* p, float* v) { const float4 q = *reinterpret_cast<const float4*>(p); v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
  static __device__ __forceinline__ void put(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
};
template <> struct Pack<__nv_bfloat16, 16> {
  static constexpr int N = 8;
  typedef uint4 raw;
  static __device__ __forceinline__ void get(const __nv_bfloat16* p, float* v) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    v[0] = bb::bf16_lo(q.x); v[1] = bb::bf16_hi(q.x); v[2] = bb::bf16_lo(q.y); v[3] = bb::bf16_hi(q.y);
    v[4] = bb::bf16_lo(q.z); v[5] = bb::bf16_hi(q.z); v[6] = bb::bf16_lo(q.w); v[7] = bb::bf16_hi(q.w);
  }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, const float* v) {
    *reinterpret_cast<uint4*>(p) = make_uint4(bb::pack_bf16x2(v[0], v[1]), bb::pack_bf16x2(v[2], v[3]), bb::pack_bf16x2(v[4], v[5]), bb::pack_bf16x2(v[6], v[7]));
  }
};
template <> struct Pack<float, 4> {
  static constexpr int N = 1;
  typedef float raw;
  static __device__ __forceinline__ void get(const float* p, float* v) { v[0] = *p; }
  static __device__ __forceinline__ void put(float* p, const float* v) { *p = v[0]; }
};
template <> struct Pack<__nv_bfloat16, 2> {
  static constexpr int N = 1;
  typedef unsigned short raw;
  static __device__ __forceinline__ void get(const __nv_bfloat16* p, float* v) { v[0] = __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, const float* v) { *p = __float2bfloat16(v[0]); }
};

constexpr int MOVE_THREADS = 256;
// An index of the routing: -1 (none) where it does not point at one of `count` rows, which sets the status word unless it is -1 already
__device__ __forceinline__ int checked(int i, int count, int* status) {
  if (i < -1 || i >= count) {
    if (status) atomicCAS(status, 0, BB_ERR_INVALID_ARG);
    return -1;
  }
  return i;
}
template <int TEAM> constexpr int TEAMS = MOVE_THREADS / TEAM;

template <typename T, int BYTES, int TEAM>
__global__ void __launch_bounds__(MOVE_THREADS)
dispatch_kernel(const T* x, long long ld, const int* slots, int k, T* out, int rows, int tokens, int h, int* status) {
  typedef Pack<T, BYTES> P;
  typedef typename P::raw raw;
  bb::pdl_sync();
  const int r = blockIdx.x * TEAMS<TEAM> + threadIdx.x / TEAM, i0 = threadIdx.x % TEAM;
  if (r >= rows) return;
  const int s = checked(slots[r], tokens * k, status), n = h / P::N;
  raw* to = reinterpret_cast<raw*>(out + (long long)r * h);
  if (s < 0) {
    const float zeros[P::N] = {};
    for (int i = i0; i < n; i += TEAM) P::put(reinterpret_cast<T*>(to + i), zeros);
    return;
  }
  const raw* from = reinterpret_cast<const raw*>(x + (long long)(s / k) * ld);
#pragma unroll 4
  for (int i = i0; i < n; i += TEAM) to[i] = from[i];
}

// A team goes through its token's row in runs of TEAM x U pieces: their loads are in flight together, those of two rows where neither is dropped; the residual's
// follow the rows' (8192 tokens of 1024, two rows and a residual each: 15.2 us, 4.4 TB/s).  Row numbers and weights wait in the lanes of each warp.
template <typename T, int BYTES, int TEAM>
__global__ void __launch_bounds__(MOVE_THREADS)
combine_kernel(const T* x, long long ld, const int* rows_of, const float* weights, const T* residual, long long ld_res, int k, T* out, int tokens, int rows, int h,
               int* status) {
  typedef Pack<T, BYTES> P;
  constexpr int U = BYTES == 16 ? 16 / P::N : 4;
  bb::pdl_sync();
  const int t = blockIdx.x * TEAMS<TEAM> + threadIdx.x / TEAM, i0 = threadIdx.x % TEAM, lane = threadIdx.x & 31;
  if (t >= tokens) return;
  const int n = h / P::N;
  const long long s = (long long)t * k;
  const int my_row = lane < k ? checked(rows_of[s + lane], rows, status) : -1;
  const float my_weight = weights && lane < k ? weights[s + lane] : 1.f;
  for (int run = 0; run < n; run += TEAM * U) {
    const int i = run + i0;
    float sum[U][P::N] = {};
#pragma unroll 2
    for (int j = 0; j < k; ++j) {
      const int r = __shfl_sync(0xffffffffu, my_row, j);
      const float w = __shfl_sync(0xffffffffu, my_weight, j);
      if (r < 0) continue;
      const T* from = x + (long long)r * ld;
      float v[U][P::N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * TEAM < n) {
          P::get(from + (i + u * TEAM) * P::N, v[u]);
        } else {
#pragma unroll
          for (int c = 0; c < P::N; ++c) v[u][c] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < P::N; ++c) sum[u][c] = fmaf(w, v[u][c], sum[u][c]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * TEAM >= n) break;
      if (residual) {
        float v[P::N];
        P::get(residual + (long long)t * ld_res + (i + u * TEAM) * P::N, v);
#pragma unroll
        for (int c = 0; c < P::N; ++c) sum[u][c] += v[c];
      }
      P::put(out + (long long)t * h + (i + u * TEAM) * P::N, sum[u]);
    }
  }
}

// The gradient of the sum is read once per run and token; a warp's share of the j-th product gathers in its lane j.
template <typename T, int BYTES, int TEAM>
__global__ void __launch_bounds__(MOVE_THREADS, 4)          // (72 registers and three blocks an SM: 26.6 us for 22.5, 8192 tokens of 1024 with two rows each)
combine_bwd_kernel(const T* dy, long long ld_dy, const T* x, long long ld, const int* rows_of, const int* slots, const float* weights, int k, T* dx,
                   float* d_weights, int tokens, int rows, int h, int* status) {
  typedef Pack<T, BYTES> P;
  constexpr int U = BYTES == 16 ? 32 / P::N : 4;
  __shared__ float part[TEAM > 32 ? TEAM / 32 : 1][32];
  bb::pdl_sync();
  const int t = blockIdx.x * TEAMS<TEAM> + threadIdx.x / TEAM, i0 = threadIdx.x % TEAM, lane = threadIdx.x & 31;
  if (t >= tokens) return;
  const int n = h / P::N;
  const long long s = (long long)t * k;
  const T* from = dy + (long long)t * ld_dy;
  // (rows and places as loaded: what stands outside is left out here and told at the end)
  const int row = lane < k ? rows_of[s + lane] : -1, my_row = row >= 0 && row < rows ? row : -1;
  const float my_weight = lane < k ? weights[s + lane] : 0.f;
  unsigned writing = 0, clearing = 0;
  bool wrong = row != my_row && row != -1;
  if (dx) {
    // Every place has one writer: the slot that it names, if that slot names the place, else (zeros) the slot of the place's own number
    const bool place = lane < k && s + lane < rows;
    const int slot = place ? slots[s + lane] : -1, named = my_row >= 0 ? slots[my_row] : 0;
    const bool known = slot >= 0 && slot < tokens * k;
    const int back = known ? rows_of[slot] : -1;
    writing = __ballot_sync(0xffffffffu, my_row >= 0 && named == s + lane);
    clearing = __ballot_sync(0xffffffffu, place && back != s + lane);
    wrong |= (my_row >= 0 && named != s + lane) || (!known && slot != -1);
  }
  float dot = 0.f;
  for (int run = 0; run < n; run += TEAM * U) {
    const int i = run + i0;
    float d[U][P::N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * TEAM < n) {
        P::get(from + (i + u * TEAM) * P::N, d[u]);
      } else {
#pragma unroll
        for (int c = 0; c < P::N; ++c) d[u][c] = 0.f;
      }
    }
    for (int j = 0; j < k; ++j) {
      const int r = __shfl_sync(0xffffffffu, my_row, j);
      const float w = __shfl_sync(0xffffffffu, my_weight, j);
      if (r >= 0) {
        if (d_weights) {
          float v[U][P::N], sum = 0.f;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (i + u * TEAM < n) {
              P::get(x + (long long)r * ld + (i + u * TEAM) * P::N, v[u]);
            } else {
#pragma unroll
              for (int c = 0; c < P::N; ++c) v[u][c] = 0.f;
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < P::N; ++c) sum = fmaf(d[u][c], v[u][c], sum);
          sum = warp_sum(sum);
          if (lane == j) dot += sum;
        }
        if (writing >> j & 1u) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (i + u * TEAM >= n) break;
            float v[P::N];
#pragma unroll
            for (int c = 0; c < P::N; ++c) v[c] = w * d[u][c];
            P::put(dx + (long long)r * h + (i + u * TEAM) * P::N, v);
          }
        }
      }
      if (clearing >> j & 1u) {
        const float zeros[P::N] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) if (i + u * TEAM < n) P::put(dx + (s + j) * h + (i + u * TEAM) * P::N, zeros);
      }
    }
  }
  if (wrong && status) atomicCAS(status, 0, BB_ERR_INVALID_ARG);
  if (!d_weights) return;
  if (TEAM > 32) {
    part[threadIdx.x / 32 % (TEAM / 32)][lane] = dot;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    dot = 0.f;
#pragma unroll
    for (int w = 0; w < TEAM / 32; ++w) dot += part[w][lane];
    if (lane < k) d_weights[s + lane] = dot;
  } else if (lane < k) {
    d_weights[s + lane] = dot;
  }
}

// ------------------------------------------------------------------ host side
bool bad_route(const bb_route_desc* d) {
  return !d || d->tokens <= 0 || d->experts <= 0 || d->experts > MAX_EXPERTS || d->k <= 0 || d->k > d->experts || d->k > MAX_CHOSEN || d->cols < d->experts || d->cols > WIDEST || d->ld < d->cols ||
         (d->dtype != BB_DTYPE_BF16 && d->dtype != BB_DTYPE_F32) || (long long)d->tokens * d->k > INT_MAX - 1024;
}

// Lanes of a token's team, as many as its choices at least, and logits a lane
struct Team { int lanes, per; };
Team team_of(int experts, int k) {
  if (experts <= 32 && k <= 8) return {8, experts <= 8 ? 1 : experts <= 16 ? 2 : 4};
  if (experts <= 64 && k <= 16) return {16, 4};
  return {32, experts <= 32 ? 1 : experts <= 64 ? 2 : experts <= 128 ? 4 : 8};
}
bool odd(const void* p, uintptr_t mask) { return ((uintptr_t)p & mask) != 0; }
// Rows in runs of a lane's values, that end inside the row's `cols` and begin on their size (16 bytes at most)
template <typename T> bool in_runs(const T* p, long long ld, int experts, int cols, int per) {
  const int bytes = per * (int)sizeof(T) < 16 ? per * (int)sizeof(T) : 16;
  return (experts + per - 1) / per * per <= cols && ld * (long long)sizeof(T) % bytes == 0 && !odd(p, bytes - 1);
}

RouteParams route_params(const bb_route_desc* d) {
  RouteParams p = {};
  p.tokens = d->tokens; p.experts = d->experts; p.k = d->k; p.normalize = d->normalize; p.ld = d->ld;
  const int sms = bb_num_sms(), most = d->max_ctas > 0 && d->max_ctas < sms ? d->max_ctas : sms;
  p.chunk = (d->tokens + most - 1) / most;
  if (p.chunk < ROUTE_WARPS) p.chunk = ROUTE_WARPS;
  // One block does it all, in one launch, where its teams have a token each: us, 128 tokens, 2 of 8 experts 7.9 -> 4.7; 64, 6 of 64, 7.9 -> 6.9; 32, 8 of 200, 12.4 ->
  // 9.7 (with two tokens each 12.4 -> 14.2)
  if (d->tokens <= ROUTE_THREADS / team_of(d->experts, d->k).lanes) p.chunk = d->tokens;
  p.blocks = (d->tokens + p.chunk - 1) / p.chunk;
  return p;
}

template <typename T> struct RouteCall {
  const T* logits; RouteParams p; cudaStream_t s;
  const float *dw, *db; T* out; long long ldd; int cols, vec_out;
};
template <typename T, int PER, int G> int route_fwd_as(const RouteCall<T>& c) {
  BB_ONCE_PER_DEVICE(BB_CUDA_CHECK(cudaFuncSetAttribute(route_choose_kernel<T, PER, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * ROUTE_WARPS * G * PER * 4)));
  BB_CUDA_CHECK(bb_launch(route_choose_kernel<T, PER, G>, c.p.blocks, ROUTE_THREADS, 2 * ROUTE_WARPS * c.p.experts * 4, c.s, c.logits, c.p));
  if (c.p.blocks > 1) BB_CUDA_CHECK(bb_launch(route_place_kernel, c.p.blocks + 1, ROUTE_THREADS, 0, c.s, c.p));
  return BB_OK;
}
template <typename T, int PER, int G> int route_bwd_as(const RouteCall<T>& c) {
  constexpr int TOKENS = BWD_WARPS * (32 / G);
  BB_CUDA_CHECK(bb_launch(route_bwd_kernel<T, PER, G>, (c.p.tokens + TOKENS - 1) / TOKENS, 32 * BWD_WARPS, 0, c.s, c.logits, c.p, c.dw, c.db, c.out, c.ldd, c.cols,
                          c.vec_out));
  return BB_OK;
}
template <typename T> int route(RouteCall<T> c, int logits_cols, bool backward) {
  const Team t = team_of(c.p.experts, c.p.k);
  c.p.vec = in_runs(c.logits, c.p.ld, c.p.experts, logits_cols, t.per);
  if (backward) c.vec_out = c.p.experts % t.per == 0 && in_runs(c.out, c.ldd, c.p.experts, c.cols, t.per);
#define ROUTE_AS(per, lanes) (backward ? route_bwd_as<T, per, lanes>(c) : route_fwd_as<T, per, lanes>(c))
  if (t.lanes == 8) return t.per == 1 ? ROUTE_AS(1, 8) : t.per == 2 ? ROUTE_AS(2, 8) : ROUTE_AS(4, 8);
  if (t.lanes == 16) return ROUTE_AS(4, 16);
  return t.per == 1 ? ROUTE_AS(1, 32) : t.per == 2 ? ROUTE_AS(2, 32) : t.per == 4 ? ROUTE_AS(4, 32) : ROUTE_AS(8, 32);
#undef ROUTE_AS
}

// 16-byte accesses: every pointer and row on 16 bytes
template <typename T> bool whole(const void* a, long long lda, const void* b, long long ldb, const void* c, long long ldc, const void* d, int h) {
  const long long item = sizeof(T);
  return !odd(a, 15) && !odd(b, 15) && !odd(c, 15) && !odd(d, 15) && lda * item % 16 == 0 && ldb * item % 16 == 0 && ldc * item % 16 == 0 && h * item % 16 == 0;
}
// Rows from 16 KB on, few rows from 4 KB on, fewer from 2 KB on, by a block each (bf16, 8 rows a token, us, a warp | a block a row, combine and its gradient: 160 tokens
// of 1024 6.7, 7.4 | 4.0, 6.9; 500 6.8, 7.4 | 5.2, 10.7; 160 of 1600 11.7, 12.3 | 4.2, 7.2; 900 11.6, 12.4 | 7.5, 16.9; dispatch, 200 rows of 1024 2.3 | 1.7, of
// 1600 2.9 | 1.7, 512 of 2048 6.3 | 2.6, 4096 of 8192 25.6 | 16.8)
bool long_rows(long long rows, long long bytes, int few = 256) { return bytes >= 16384 || (bytes >= 4096 && rows < 1024) || (bytes >= 2048 && rows < few); }

#define MOVE(kernel, T, vec, big, rows, ...)                                                                                        \
  do {                                                                                                                              \
    const long long blocks_ = (big) ? (rows) : ((rows) + TEAMS<32> - 1) / TEAMS<32>;                                                \
    if (blocks_ > INT_MAX) return refuse("more rows than one launch covers");                                                       \
    if (vec) BB_CUDA_CHECK(bb_launch((big) ? kernel<T, 16, MOVE_THREADS> : kernel<T, 16, 32>, (int)blocks_, MOVE_THREADS, 0, s, __VA_ARGS__)); \
    else BB_CUDA_CHECK(bb_launch((big) ? kernel<T, sizeof(T), MOVE_THREADS> : kernel<T, sizeof(T), 32>, (int)blocks_, MOVE_THREADS, 0, s, __VA_ARGS__)); \
    return BB_OK;                                                                                                                   \
  } while (0)

template <typename T> int dispatch(const T* x, long long ld, const int* slots, int k, T* out, int rows, int tokens, int h, cudaStream_t s) {
  const bool vec = whole<T>(x, ld, out, 0, nullptr, 0, nullptr, h), big = long_rows(rows, (long long)h * sizeof(T));
  MOVE(dispatch_kernel, T, vec, big, rows, x, ld, slots, k, out, rows, tokens, h, bb_device_status_word());
}
template <typename T>
int combine(const T* x, long long ld, const int* rows_of, const float* w, const T* res, long long ld_res, int k, T* out, int tokens, int rows, int h, cudaStream_t s) {
  const bool vec = whole<T>(x, ld, out, 0, res, res ? ld_res : 0, nullptr, h), big = long_rows(tokens, (long long)h * sizeof(T), 768);
  MOVE(combine_kernel, T, vec, big, tokens, x, ld, rows_of, w, res, ld_res, k, out, tokens, rows, h, bb_device_status_word());
}
template <typename T>
int combine_bwd(const T* dy, long long ld_dy, const T* x, long long ld, const int* rows_of, const int* slots, const float* w, int k, T* dx, float* dw,
                int tokens, int rows, int h, cudaStream_t s) {
  const bool vec = whole<T>(dy, ld_dy, dw ? x : nullptr, dw ? ld : 0, nullptr, 0, dx, h), big = long_rows(tokens, (long long)h * sizeof(T));
  MOVE(combine_bwd_kernel, T, vec, big, tokens, dy, ld_dy, x, ld, rows_of, slots, w, k, dx, dw, tokens, rows, h, bb_device_status_word());
}

bool bad_move(const void* x, long long ld, int dtype, const void* index, int k, long long rows, long long tokens, int h) {
  return k > MAX_CHOSEN || !x || tokens <= 0 || k > INT_MAX / tokens || !index || odd(index, 3) || k <= 0 || rows <= 0 || rows > INT_MAX || h <= 0 || h > WIDEST || ld < h || (dtype != BB_DTYPE_BF16 && dtype != BB_DTYPE_F32) ||
         odd(x, dtype == BB_DTYPE_F32 ? 3 : 1);
}
}  // namespace

extern "C" long long bb_route_workspace_bytes(const bb_route_desc* d) {
  if (bad_route(d)) return 0;
  const RouteParams p = route_params(d);
  return 4LL * p.blocks * (2 * p.experts + 1);
}

extern "C" int bb_route_fwd(const bb_route_desc* d, const void* logits, float* weights, int* experts_out, int* rows_out, int* slots_out, int* offsets,
                            float* balance, float* stats, float* load, void* workspace, long long workspace_bytes, void* stream) {
  if (bad_route(d) || !logits || odd(logits, d->dtype == BB_DTYPE_F32 ? 3 : 1) || !weights || !experts_out || !rows_out || !slots_out || !offsets || !balance || !stats ||
      odd(stats, 7) || !load || !workspace || odd(workspace, 3) || workspace_bytes < bb_route_workspace_bytes(d))
    return refuse("bb_route_fwd: null or misaligned pointer, no tokens, 1 to 256 experts of which 1 to 32 are chosen, cols < experts, ld < cols, an unknown type, or a workspace that "
                  "is too small");
  RouteParams p = route_params(d);
  p.weights = weights; p.chosen = experts_out; p.rows = rows_out; p.slots = slots_out; p.offsets = offsets; p.balance = balance; p.stats = (float2*)stats; p.load = load;
  p.counts = (int*)workspace; p.probs = (float*)((int*)workspace + (long long)p.blocks * (p.experts + 1));
  BackToBack overlap(d->max_ctas == 0);
  return d->dtype == BB_DTYPE_BF16 ? route(RouteCall<__nv_bfloat16>{(const __nv_bfloat16*)logits, p, (cudaStream_t)stream}, d->cols, false)
                                   : route(RouteCall<float>{(const float*)logits, p, (cudaStream_t)stream}, d->cols, false);
}

extern "C" int bb_route_bwd(const bb_route_desc* d, const void* logits, const int* experts_out, const float* stats, const float* load,
                            const float* d_weights, const float* d_balance, void* dlogits, long long ldd, int cols, void* stream) {
  if (bad_route(d) || !logits || odd(logits, d->dtype == BB_DTYPE_F32 ? 3 : 1) || !experts_out || !stats || odd(stats, 7) || !load || !dlogits ||
      odd(dlogits, d->dtype == BB_DTYPE_F32 ? 3 : 1) || cols < d->experts || cols > WIDEST || ldd < cols)
    return refuse("bb_route_bwd: null or misaligned pointer, a descriptor that bb_route_fwd refuses, cols < experts or ldd < cols");
  RouteParams p = route_params(d);
  p.chosen = const_cast<int*>(experts_out); p.stats = (float2*)stats; p.load = const_cast<float*>(load);
  return d->dtype == BB_DTYPE_BF16
             ? route(RouteCall<__nv_bfloat16>{(const __nv_bfloat16*)logits, p, (cudaStream_t)stream, d_weights, d_balance, (__nv_bfloat16*)dlogits, ldd, cols}, d->cols, true)
             : route(RouteCall<float>{(const float*)logits, p, (cudaStream_t)stream, d_weights, d_balance, (float*)dlogits, ldd, cols}, d->cols, true);
}

extern "C" int bb_dispatch_rows(const void* x, long long ld, int dtype, const int* slots, int k, void* out, long long rows, long long tokens, int h,
                                void* stream) {
  if (bad_move(x, ld, dtype, slots, k, rows, tokens, h) || !out || odd(out, dtype == BB_DTYPE_F32 ? 3 : 1))
    return refuse("bb_dispatch_rows: null or misaligned pointer, a size that is not positive, ld < h, or an unknown type");
  return dtype == BB_DTYPE_BF16 ? dispatch((const __nv_bfloat16*)x, ld, slots, k, (__nv_bfloat16*)out, (int)rows, (int)tokens, h, (cudaStream_t)stream)
                                : dispatch((const float*)x, ld, slots, k, (float*)out, (int)rows, (int)tokens, h, (cudaStream_t)stream);
}

extern "C" int bb_combine_rows(const void* x, long long ld, int dtype, const int* rows_of, const float* weights, const void* residual, long long ld_residual,
                               int k, void* out, long long tokens, long long rows, int h, void* stream) {
  const uintptr_t mask = dtype == BB_DTYPE_F32 ? 3 : 1;
  if (bad_move(x, ld, dtype, rows_of, k, rows, tokens, h) || !out || odd(out, mask) || odd(weights, 3) || odd(residual, mask) || (residual && ld_residual < h))
    return refuse("bb_combine_rows: null or misaligned pointer, a size that is not positive, ld < h, or an unknown type");
  return dtype == BB_DTYPE_BF16 ? combine((const __nv_bfloat16*)x, ld, rows_of, weights, (const __nv_bfloat16*)residual, ld_residual, k, (__nv_bfloat16*)out, (int)tokens, (int)rows, h, (cudaStream_t)stream)
                                : combine((const float*)x, ld, rows_of, weights, (const float*)residual, ld_residual, k, (float*)out, (int)tokens, (int)rows, h, (cudaStream_t)stream);
}

extern "C" int bb_combine_rows_bwd(const void* dy, long long ld_dy, int dtype, const void* x, long long ld, const int* rows_of, const int* slots,
                                   const float* weights, int k, void* dx, float* d_weights, long long tokens, long long rows, int h,
                                   void* stream) {
  const uintptr_t mask = dtype == BB_DTYPE_F32 ? 3 : 1;
  if (bad_move(dy, ld_dy, dtype, rows_of, k, rows, tokens, h) || rows > tokens * k || !slots || odd(slots, 3) || !weights || odd(weights, 3) || (!dx && !d_weights) || odd(dx, mask) ||
      odd(d_weights, 3) || (d_weights && (!x || odd(x, mask) || ld < h)))
    return refuse("bb_combine_rows_bwd: null or misaligned pointer, a size that is not positive, a leading dimension < h, or an unknown type");
  return dtype == BB_DTYPE_BF16
             ? combine_bwd((const __nv_bfloat16*)dy, ld_dy, (const __nv_bfloat16*)x, ld, rows_of, slots, weights, k, (__nv_bfloat16*)dx, d_weights, (int)tokens, (int)rows, h, (cudaStream_t)stream)
             : combine_bwd((const float*)dy, ld_dy, (const float*)x, ld, rows_of, slots, weights, k, (float*)dx, d_weights, (int)tokens, (int)rows, h, (cudaStream_t)stream);
}
