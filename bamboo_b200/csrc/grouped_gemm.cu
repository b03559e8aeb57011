// Matrix products grouped by expert on the 5th-generation tensor cores.  Rows are sorted by expert: expert e owns rows
// [offsets[e], offsets[e + 1]) of x and of y, and has a weight W_e [n, k] of its own.
//
//   rows (forward)    y[r] = W_e x[r] (+ b_e, GeLU)        A = x, B = W_e, reduction over k
//   rows (input)      dx[r] = W_e^T dy[r] (* GeLU')        A = dy, B = W_e turned, reduction over n
//   weight gradient   dW_e = sum over its rows of dy[r] x[r]^T   A = dy turned, B = x turned, reduction over the expert's rows
//
// The offsets are on the device and the host never reads them: a launch has as many CTAs as there may be tiles (at most one per SM),
// and every warp walks the experts' tiles in the same order, unit after unit of its CTA's share.  No tile spans two experts.  A row
// tile that overhangs its expert computes its neighbour's rows and does not store them.  In a weight gradient the overhang is part of
// the reduction: where an expert ends inside a group of 16 rows (the reduction of one MMA), the neighbour's rows of that group are
// overwritten with zeros in shared memory, in both operands, so that an infinity or NaN over there stays there.
//
// The main loop is that of the dense product (gemm_tcgen05.cu): two producer warps, one MMA warp, eight epilogue warps, six
// stages of 32 KiB, two accumulators; pairs of CTAs (cta_group::2) on 256 x 256 tiles where the experts are large enough.
// Where tiles are few and reductions long, CTAs share them: rows in clusters (grouped_split_kernel), weight gradients in parts (grouped_join_kernel).
#include "common.cuh"
#include "bamboo_b200.h"
#include "gemm_panels.cuh"
#include "tma_host.cuh"
#include <atomic>
#include <limits.h>
#include <math.h>

namespace {

constexpr int BM = 128, BK = 64, UMMA_K = 16;
constexpr int TMA_WARP_0 = 0, MMA_WARP = 1, TMA_WARP_1 = 2, EPI_WARP = 3, EPI_WARPS = 8;
constexpr int SUM_WARP = EPI_WARP + EPI_WARPS;        // weight gradients only
template <bool WEIGHT> constexpr int THREADS = 32 * (SUM_WARP + (WEIGHT ? 1 : 0));
constexpr int A_STAGE_BYTES = BM * BK * 2;
constexpr int SLAB_BYTES = 32 * 128;
constexpr int MAX_EXPERTS = 256;
constexpr int WIDEST = INT_MAX - 4096;                // columns are counted in 32 bits, up to a tile beyond the last

template <int BN, bool PAIR> struct Cfg {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int B_STAGE_BYTES = B_ROWS * BK * 2;
  static constexpr int STAGE_BYTES = A_STAGE_BYTES + B_STAGE_BYTES;
  static constexpr int STAGES = B_ROWS == 256 ? 4 : 6;
  static constexpr int TILE_M = PAIR ? 2 * BM : BM;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int BAR_BYTES = (5 * STAGES + 4) * 8 + 8;
  static constexpr int TABLE_BYTES = (MAX_EXPERTS + 1) * 4 + MAX_EXPERTS;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * SLAB_BYTES + 1024 /*align slack*/ + BAR_BYTES + TABLE_BYTES;
  static_assert(SMEM_BYTES <= 227 * 1024, "fits an SM");
};

struct GroupParams {
  int rows;                   // of x and y
  int n, k;                   // columns of the result, and the length of the reduction (weight gradient: rows and columns of dW_e)
  int experts;
  int epi;
  int stage_bytes;            // that the copies of one CTA bring
  int split, quarters;        // grouped_split_kernel: CTAs that share a tile's reduction, runs of 32 rows that an expert can have in a tile; weight
                              // gradient: parts of each reduction, every one a unit of its own
  int rotate;                 // column tile i begins its reduction with k-block i: of few rows all CTAs would ask for the same few lines at once
  const int* offsets;
  void* D; void* D2; const void* bias; const void* aux;
  __nv_bfloat16* bias_grad; float* bias_accum;            // weight gradient: where db_e goes (one of them, or none) ...
  float* bias_parts;          // ... by way of [parts][column tiles][experts][n], where these are more than one
  float* parts;               // weight gradient in parts: [parts][experts][n][k]
  long long ldd, ld_aux, expert_stride;       // expert_stride: values of one dW_e
  int* status;
};

struct Unit {
  int e, ni, m0, n0;          // first row (a row of x, or of dW_e) and column of the tile
  int end;                    // where its rows end
  int k0, num_kb, tail;       // weight gradient: first row of the reduction, rows of the last k-block
  int part;                   // ... and which part of it this is
};

// The units of a CTA (pair) one after the other: one of each `workers` in a row.  Those of a weight gradient, longest reductions first, are dealt out there and
// back - worker w gets the w-th of a round, then the w-th from the end of the next - so that shares come out alike (16384 rows of 8 unequal experts, 4096 x
// 1024: 16 % over the mean share when dealt in one direction, 7 % now).
// PARTS: a weight gradient in parts (p.split of them); the arithmetic for it would cost short units of the others half a microsecond each.
template <bool WGRAD, int BN, int TILE_M, bool PARTS = false> struct Walk {
  const GroupParams& p;
  const int* start;
  const unsigned char* order;
  int e, first, tiles, unit, step, back, turn, cols, m_tiles;
  __device__ __forceinline__ Walk(const GroupParams& p_, const int* s, const unsigned char* o, int worker, int workers)
      : p(p_), start(s), order(o), e(-1), first(0), tiles(0), unit(worker), step(0), back(workers), turn(0), cols((p_.n + BN - 1) / BN), m_tiles(0) {
    if constexpr (WGRAD) {
      m_tiles = (p.n + TILE_M - 1) / TILE_M;
      cols = (p.k + BN - 1) / BN;
      back = 2 * (workers - 1 - worker) + 1;          // from a place to that in the next round, and 2 workers less that to the one after
      turn = 2 * workers;
    }
  }
  __device__ __forceinline__ bool next(Unit& u) {
    unit += step;
    step = back;
    if constexpr (WGRAD) back = turn - back;
    while (unit >= first + tiles) {
      if (++e == p.experts) return false;
      first += tiles;
      if constexpr (!WGRAD) m_tiles = (start[e + 1] - start[e] + TILE_M - 1) / TILE_M;
      tiles = m_tiles * cols * (PARTS ? p.split : 1);
    }
    const int local = unit - first, col = local / m_tiles, mi = local - col * m_tiles, part = PARTS ? col / cols : 0, ni = col - part * cols;
    u.ni = ni; u.n0 = ni * BN;
    if constexpr (WGRAD) {
      u.e = order[e];
      const int n = start[u.e + 1] - start[u.e];
      u.m0 = mi * TILE_M; u.end = p.n;
      const int all = (n + BK - 1) / BK;
      int from = 0, to = all;
      if constexpr (PARTS) { from = part * all / p.split; to = (part + 1) * all / p.split; }        // (at most 2^21 k-blocks, 32 parts)
      u.part = part;
      u.k0 = start[u.e] + from * BK; u.num_kb = to - from; u.tail = to == all ? n - (all - 1) * BK : BK;
    } else {
      u.e = e;
      u.m0 = start[e] + mi * TILE_M; u.end = start[e + 1];
      u.k0 = 0; u.num_kb = (p.k + BK - 1) / BK; u.tail = BK;
    }
    return true;
  }
};

// Rows [from, to) of the reduction become zeros in `boxes` boxes of 64 columns (64 rows of 128 bytes each; the swizzle permutes 16-byte
// chunks inside a row), by a whole warp.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int boxes, int from, int to, int lane) {
  const int chunks = (to - from) * 8;
  for (int b = 0; b < boxes; ++b)
    for (int i = lane; i < chunks; i += 32) *reinterpret_cast<uint4*>(tile + b * 8192 + from * 128 + i * 16) = make_uint4(0, 0, 0, 0);
}

// Where every expert's rows begin, ascending within [0, rows]; by one warp.  Offsets that do not ascend set the status word and are cut.
__device__ __forceinline__ void read_offsets(const GroupParams& p, int* start, int lane) {
  int carry = 0;
  bool bad = false;
  for (int at = 0; at <= p.experts; at += 32) {
    const int i = at + lane, raw = i <= p.experts ? __ldca(p.offsets + i) : INT_MIN;
    int v = raw < 0 ? 0 : raw > p.rows ? p.rows : raw;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d && o > v) v = o;
    }
    if (v < carry) v = carry;
    if (i <= p.experts) { start[i] = v; bad |= v != raw; }
    carry = __shfl_sync(0xffffffffu, v, 31);
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0 && p.status) atomicCAS(p.status, 0, BB_ERR_INVALID_ARG);
}

enum { ROWS = 0, ROWS_T = 1, WGRAD = 2 };     // B as stored, B turned, weight gradient

// db_e along with dW_e: one warp adds up rows of dy that stand in shared memory anyway, behind the MMAs that read them (`read_bar`) and in front of the
// copies that replace them (`summed_bar`).  (Beside the MMAs, told by the warp that issues them when a stage has landed: pairs took 85 us for 52 even
// without a bias.)  It takes longer for a k-block than its MMAs (512 cycles), so the column tiles that share the rows take
// their k-blocks in turn - tile i the k-blocks i, i + tiles, ... - and `grouped_join_kernel` adds the tiles' sums in their order (16384 rows of 8 experts,
// 4096 x 1024, us: 116, of which 108 are the weight gradient's; by the tiles of the first columns alone 169, with a pass of its own 108 + 33).  A lane keeps eight columns of each
// box and every fourth row.
struct ColumnSums {
  float2 v[BM / 64][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int b = 0; b < BM / 64; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[b][i] = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void add(int b, const uint4& q) {
    v[b][0] = bb::add2(v[b][0], make_float2(bb::bf16_lo(q.x), bb::bf16_hi(q.x)));
    v[b][1] = bb::add2(v[b][1], make_float2(bb::bf16_lo(q.y), bb::bf16_hi(q.y)));
    v[b][2] = bb::add2(v[b][2], make_float2(bb::bf16_lo(q.z), bb::bf16_hi(q.z)));
    v[b][3] = bb::add2(v[b][3], make_float2(bb::bf16_lo(q.w), bb::bf16_hi(q.w)));
  }
  __device__ __forceinline__ void add(const uint8_t* tile, int rows, int lane) {
#pragma unroll
    for (int b = 0; b < BM / 64; ++b) {
      const uint8_t* box = tile + b * 8192;
      if (rows == BK) {
        uint4 q[BK / 4];
#pragma unroll
        for (int i = 0; i < BK / 4; ++i) q[i] = *reinterpret_cast<const uint4*>(box + slab_off((lane >> 3) + 4 * i, lane & 7));
#pragma unroll
        for (int i = 0; i < BK / 4; ++i) add(b, q[i]);
      } else {
        for (int r = lane >> 3; r < rows; r += 4) add(b, *reinterpret_cast<const uint4*>(box + slab_off(r, lane & 7)));
      }
    }
  }
  __device__ __forceinline__ void write(const GroupParams& p, int e, int tile, int m0, int lane) {
#pragma unroll
    for (int b = 0; b < BM / 64; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 s = v[b][i];
#pragma unroll
        for (int d = 8; d < 32; d <<= 1) {
          s.x += __shfl_xor_sync(0xffffffffu, s.x, d);
          s.y += __shfl_xor_sync(0xffffffffu, s.y, d);
        }
        const int c = m0 + b * 64 + (lane & 7) * 8 + i * 2;
        if (lane < 8 && c < p.n) {             // (n is even)
          const long long at = (long long)e * p.n + c;
          if (p.bias_parts) *reinterpret_cast<float2*>(p.bias_parts + (long long)tile * p.experts * p.n + at) = s;
          else if (p.bias_accum) { p.bias_accum[at] += s.x; p.bias_accum[at + 1] += s.y; }
          else { p.bias_grad[at] = __float2bfloat16(s.x); p.bias_grad[at + 1] = __float2bfloat16(s.y); }
        }
      }
  }
};

// A panel of 32 rows and 64 columns, its rows' sums in the lanes' `v` (and `aux`, where there is one, in the slab): through the epilogue and out
template <int MODE>
__device__ __forceinline__ void finish_panel(const GroupParams& p, uint8_t* slab, const __nv_bfloat16* bias, bool has_bias, bool dual, bool has_aux, long long base, int r0,
                                             int nb, int end, int cols, int lane, float (&v)[64]) {
  if (MODE == ROWS && has_bias) {
    if (nb + 64 <= cols) {
#pragma unroll
      for (int i = 0; i < 64; i += 8) {
        float f[8]; unpack8(__ldg(reinterpret_cast<const uint4*>(bias + nb + i)), f);
#pragma unroll
        for (int k = 0; k < 8; k += 2) set2(v + i + k, bb::add2(get2(v + i + k), make_float2(f[k], f[k + 1])));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 64; ++i) if (nb + i < cols) v[i] += __bfloat162float(bias[nb + i]);
    }
  }
  if (MODE == ROWS && dual) {
    panel_store_row_bf16(slab, lane, v);     // pre-activation first
    __syncwarp();
    slab_flush_bf16(slab, reinterpret_cast<__nv_bfloat16*>(p.D2), p.ldd, r0, nb, end, cols, lane);
    // (of the sum itself: its rounding above is for the backward pass alone)
#pragma unroll
    for (int i = 0; i < 64; i += 2) set2(v + i, bb::gelu_tanh2(get2(v + i)));
    __syncwarp();
  } else if (MODE == ROWS_T && has_aux) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[32];
#pragma unroll
      for (int c = 0; c < 4; ++c) unpack8(*reinterpret_cast<const uint4*>(slab + slab_off(lane, 4 * h + c)), x + 8 * c);
      apply_aux<32>(p.epi, v + 32 * h, x);
    }
    __syncwarp();
  }
  panel_store_row_bf16(slab, lane, v);
  __syncwarp();
  slab_flush_bf16(slab, reinterpret_cast<__nv_bfloat16*>(p.D) + base, p.ldd, r0, nb, end, cols, lane);
  __syncwarp();
}

// rows that belong to no expert
__device__ __forceinline__ void zero_the_rest(const GroupParams& p, const int* start, int threads) {
  const int before = start[0], after = p.rows - start[p.experts], chunks = p.n >> 3;
  for (long long i = (long long)blockIdx.x * threads + threadIdx.x; i < (long long)(before + after) * chunks; i += (long long)gridDim.x * threads) {
    const int r = (int)(i / chunks), c = (int)(i - (long long)r * chunks);
    reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.D) + (long long)(r < before ? r : start[p.experts] + r - before) * p.ldd)[c] =
        make_uint4(0, 0, 0, 0);
  }
}

template <int MODE, int BN, bool PAIR, bool PARTS = false>
__global__ void __launch_bounds__(THREADS<MODE == WGRAD>, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GroupParams p) {
  using C = Cfg<BN, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * A_STAGE_BYTES;
  uint8_t* panels = smem + C::STAGES * C::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(panels + EPI_WARPS * SLAB_BYTES);      // [STAGES]
  uint64_t* empty_bar = full_bar + C::STAGES;       // [STAGES]
  uint64_t* clean_bar = empty_bar + C::STAGES;      // [STAGES] pairs: the other CTA's overhanging rows are zeros
  uint64_t* read_bar = clean_bar + C::STAGES;     // [STAGES] weight gradient: the MMAs have read a stage that is to be summed
  uint64_t* summed_bar = read_bar + C::STAGES;      // [STAGES] ... and its rows are added up
  uint64_t* tmem_full = summed_bar + C::STAGES;     // [2]
  uint64_t* tmem_empty = tmem_full + 2;             // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 2);                                     // [experts + 1]
  unsigned char* order = reinterpret_cast<unsigned char*>(start + MAX_EXPERTS + 1);       // [experts]

  const int warp = bb::warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? bb::cluster_ctarank() : 0u;
  const int worker = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int workers = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < C::STAGES; ++s) { bb::mbar_init(&full_bar[s], 1); bb::mbar_init(&empty_bar[s], 1); bb::mbar_init(&clean_bar[s], 1); bb::mbar_init(&read_bar[s], 1); bb::mbar_init(&summed_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { bb::mbar_init(&tmem_full[a], 1); bb::mbar_init(&tmem_empty[a], (PAIR ? 2 : 1) * EPI_WARPS); }
    bb::fence_barrier_init();
    bb::tma_prefetch_desc(&tmA);
    bb::tma_prefetch_desc(&tmB);
  }
  if (warp == MMA_WARP) {
    if (PAIR) { bb::tmem_alloc_pair(tmem_slot, C::TMEM_COLS); bb::tmem_relinquish_pair(); }
    else { bb::tmem_alloc(tmem_slot, C::TMEM_COLS); bb::tmem_relinquish(); }
  }
  bb::pdl_sync();
  if (warp == EPI_WARP) read_offsets(p, start, lane);
  bb::tc_fence_before_sync();
  if (PAIR) bb::cluster_sync();     // the peer's barriers are initialised before anything signals them
  else __syncthreads();
  bb::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  if constexpr (MODE == WGRAD) {
    // longest reductions first: the last units of a launch are then the short ones
    for (int e = threadIdx.x; e < p.experts; e += THREADS<true>) {
      const int n = start[e + 1] - start[e];
      int at = 0;
      for (int i = 0; i < p.experts; ++i) {
        const int o = start[i + 1] - start[i];
        at += o > n || (o == n && i < e);
      }
      order[at] = (unsigned char)e;
    }
    __syncthreads();
  } else {
    zero_the_rest(p, start, THREADS<false>);
  }
  Walk<MODE == WGRAD, BN, C::TILE_M, PARTS> walk(p, start, order, worker, workers);
  Unit u;
  const bool with_bias = MODE == WGRAD && (p.bias_grad || p.bias_accum);

  if (warp == TMA_WARP_0 || warp == TMA_WARP_1) {
    // ------------------------------------------------ producers: the stages in turn
    static_assert(C::STAGES % 2 == 0, "the producers take the stages in turn");
    const int turn = warp == TMA_WARP_1 ? 1 : 0;
    int s = 0; uint32_t phase = 0, summing = 0, summed_phase = 0;       // summing: stages whose last rows are (or were) added up
    bool alive = true;
    auto wait_summed = [&]() {
      if (!(MODE == WGRAD && ((summing >> s) & 1u))) return true;
      const bool got = bb::mbar_wait_warp(&summed_bar[s], (summed_phase >> s) & 1u, abort_flag, p.status);
      summed_phase ^= 1u << s;
      summing &= ~(1u << s);
      return got;
    };
    while (alive && walk.next(u)) {
      const int m0 = u.m0 + (int)rank * BM, n0 = u.n0 + (int)rank * C::B_ROWS;
      int next_sum = with_bias ? u.ni : -1;
      for (int kb = 0; kb < u.num_kb; ++kb) {
        const bool sums = MODE == WGRAD && kb == next_sum;
        if (sums) next_sum += walk.cols;
        if ((s & 1) == turn) {
          if (!bb::mbar_wait_warp(&empty_bar[s], phase ^ 1, abort_flag, p.status) || !wait_summed()) { alive = false; break; }
          if (sums) summing |= 1u << s;
          uint8_t* a = sA + s * A_STAGE_BYTES;
          uint8_t* b = sB + s * C::B_STAGE_BYTES;
          int at = kb;
          if (MODE != WGRAD && p.rotate) {
            at += u.ni % u.num_kb;
            if (at >= u.num_kb) at -= u.num_kb;
          }
          const int k0 = u.k0 + at * BK;
          // a stage whose last rows are to be zeroed completes in each CTA of a pair for itself
          const bool own = !PAIR || (MODE == WGRAD && kb == u.num_kb - 1 && (u.tail & 15));
          if (bb::elect_one()) {
            uint32_t fb = bb::smem_u32(&full_bar[s]);
            if (own) bb::mbar_arrive_expect_tx(&full_bar[s], p.stage_bytes);
            else if (rank == 0) bb::mbar_arrive_expect_tx(&full_bar[s], 2 * p.stage_bytes);
            if constexpr (PAIR) fb = bb::mapa_shared(fb, own ? rank : 0u);
            auto load2 = [&](uint8_t* dst, const CUtensorMap* tm, int x, int y) {
              if constexpr (PAIR) bb::tma_load_2d_pair(dst, tm, fb, x, y);
              else bb::tma_load_2d(dst, tm, &full_bar[s], x, y);
            };
            auto load3 = [&](uint8_t* dst, const CUtensorMap* tm, int x, int y, int z) {
              if constexpr (PAIR) bb::tma_load_3d_pair(dst, tm, fb, x, y, z);
              else bb::tma_load_3d(dst, tm, &full_bar[s], x, y, z);
            };
            if constexpr (MODE == WGRAD) {
#pragma unroll
              for (int j = 0; j < BM / 64; ++j) load2(a + j * 8192, &tmA, m0 + 64 * j, k0);
#pragma unroll
              for (int j = 0; j < C::B_ROWS / 64; ++j) load2(b + j * 8192, &tmB, n0 + 64 * j, k0);
            } else {
              // (a CTA of a pair without rows of this expert multiplies zeros, which behind the last row come from nowhere)
              load2(a, &tmA, k0, PAIR && m0 >= u.end ? p.rows : m0);
              if constexpr (MODE == ROWS) {
                load3(b, &tmB, k0, n0, u.e);
              } else {
#pragma unroll
                for (int j = 0; j < C::B_ROWS / 64; ++j) load3(b + j * 8192, &tmB, n0 + 64 * j, k0, u.e);
              }
            }
          }
          __syncwarp();
        }
        if (++s == C::STAGES) { s = 0; phase ^= 1; }
      }
    }
    if constexpr (PAIR) {
      // rank 0's commits arrive on this CTA's barriers too: none may still be on its way when the CTA leaves
      for (int i = 0; i < C::STAGES && alive; ++i) {
        if ((s & 1) == turn && (!bb::mbar_wait_warp(&empty_bar[s], phase ^ 1, abort_flag, p.status) || !wait_summed())) alive = false;
        if (++s == C::STAGES) { s = 0; phase ^= 1; }
      }
    }
    if (!alive) {
      // copies still in flight get time to land (bounded)
      const uint64_t t0 = bb::globaltimer_ns();
      while (bb::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------ MMA issuer (pairs: rank 0; the other CTA's only cleans its stages)
    constexpr uint32_t A_MN = MODE == WGRAD, B_MN = MODE != ROWS;
    constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | (A_MN << 15) | (B_MN << 16) | ((uint32_t)(BN >> 3) << 17) |
                               ((uint32_t)(C::TILE_M >> 4) << 24);
    constexpr uint32_t A_LBO = A_MN ? 8192u : 16u, B_LBO = B_MN ? 8192u : 16u, A_STEP = A_MN ? 2048u : 32u, B_STEP = B_MN ? 2048u : 32u;
    int s = 0; uint32_t phase = 0, clean_phase = 0;
    int acc = 0; uint32_t acc_phase = 0;
    bool alive = true;
    auto clean = [&](int stage, int tail) {
      zero_rows(sA + stage * A_STAGE_BYTES, BM / 64, tail, (tail + 15) & ~15, lane);
      zero_rows(sB + stage * C::B_STAGE_BYTES, C::B_ROWS / 64, tail, (tail + 15) & ~15, lane);
      bb::fence_proxy_async();
      __syncwarp();
    };
    while (alive && walk.next(u)) {
      if (u.num_kb == 0) continue;             // an expert without rows: the epilogue writes its zeros
      const bool ragged = MODE == WGRAD && (u.tail & 15);
      if (PAIR && rank == 1) {
        if (ragged) {
          const int st = (s + u.num_kb - 1) % C::STAGES;
          if (!bb::mbar_wait_warp(&full_bar[st], (clean_phase >> st) & 1u, abort_flag, p.status)) { alive = false; break; }
          clean_phase ^= 1u << st;
          clean(st, u.tail);
          if (lane == 0) bb::mbar_arrive_cluster(bb::mapa_shared(bb::smem_u32(&clean_bar[st]), 0));
        }
        s = (s + u.num_kb) % C::STAGES;
        continue;
      }
      if (!bb::mbar_wait_warp(&tmem_empty[acc], acc_phase ^ 1, abort_flag, p.status)) { alive = false; break; }
      bb::tc_fence_after_sync();
      const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
      int next_sum = with_bias ? u.ni : -1;
      for (int kb = 0; kb < u.num_kb; ++kb) {
        const bool sums = MODE == WGRAD && kb == next_sum;
        if (sums) next_sum += walk.cols;
        if (!bb::mbar_wait_warp(&full_bar[s], phase, abort_flag, p.status)) { alive = false; break; }
        int steps = BK / UMMA_K;
        if (MODE == WGRAD && kb == u.num_kb - 1) {
          steps = (u.tail + 15) >> 4;
          if (ragged) {
            clean(s, u.tail);
            if constexpr (PAIR) {
              const bool got = bb::mbar_wait_cluster(&clean_bar[s], (clean_phase >> s) & 1u, abort_flag, p.status);
              if (!__all_sync(0xffffffffu, got)) { alive = false; break; }
              clean_phase ^= 1u << s;
            }
          }
        }
        bb::tc_fence_after_sync();
        if (bb::elect_one()) {
          const uint64_t ad0 = bb::make_smem_desc_sw128(bb::smem_u32(sA + s * A_STAGE_BYTES), A_LBO, 1024u);
          const uint64_t bd0 = bb::make_smem_desc_sw128(bb::smem_u32(sB + s * C::B_STAGE_BYTES), B_LBO, 1024u);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            if (MODE == WGRAD && k >= steps) break;
            const uint64_t ad = ad0 + (uint64_t)(k * (A_STEP >> 4)), bd = bd0 + (uint64_t)(k * (B_STEP >> 4));
            if (PAIR) bb::umma_f16_pair(d_tmem, ad, bd, IDESC, (kb > 0 || k > 0) ? 1u : 0u);
            else bb::umma_f16(d_tmem, ad, bd, IDESC, (kb > 0 || k > 0) ? 1u : 0u);
          }
          if (sums) {
            if (PAIR) bb::umma_commit_pair(&read_bar[s], 3);
            else bb::umma_commit(&read_bar[s]);
          }
          if (PAIR) {
            bb::umma_commit_pair(&empty_bar[s], 3);
            if (kb == u.num_kb - 1) bb::umma_commit_pair(&tmem_full[acc], 3);
          } else {
            bb::umma_commit(&empty_bar[s]);
            if (kb == u.num_kb - 1) bb::umma_commit(&tmem_full[acc]);
          }
        }
        __syncwarp();
        if (++s == C::STAGES) { s = 0; phase ^= 1; }
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  } else if (MODE == WGRAD && warp == SUM_WARP) {
    // ------------------------------------------------ bias gradient
    int s = 0; uint32_t read_phase = 0;
    bool alive = with_bias;
    while (alive && walk.next(u)) {
      ColumnSums sums;
      sums.clear();
      for (int kb = u.ni; kb < u.num_kb; kb += walk.cols) {
        const int st = (s + kb) % C::STAGES;
        if (!bb::mbar_wait_warp(&read_bar[st], (read_phase >> st) & 1u, abort_flag, p.status)) { alive = false; break; }
        read_phase ^= 1u << st;
        sums.add(sA + st * A_STAGE_BYTES, kb == u.num_kb - 1 ? u.tail : BK, lane);
        __syncwarp();
        if (lane == 0) bb::mbar_arrive(&summed_bar[st]);
      }
      s = (s + u.num_kb) % C::STAGES;
      if (alive) sums.write(p, u.e, PARTS ? u.part * walk.cols + u.ni : u.ni, u.m0 + (int)rank * BM, lane);
    }
  } else {
    // ------------------------------------------------ epilogue: eight warps, two per TMEM lane quarter, panels of 128 bytes in turn
    const int eg = (warp - EPI_WARP) >> 2, quarter = warp & 3;
    const bool f32 = MODE == WGRAD && (PARTS || p.epi == BB_EPI_ACCUM_F32);
    const bool dual = MODE == ROWS && p.epi == BB_EPI_BIAS_GELU;
    const bool has_aux = MODE == ROWS_T && p.epi == BB_EPI_MUL_DGELU, has_bias = MODE == ROWS && (p.epi == BB_EPI_BIAS || dual);
    const int cols = MODE == WGRAD ? p.k : p.n;
    uint8_t* slab = panels + (warp - EPI_WARP) * SLAB_BYTES;
    int acc = 0; uint32_t acc_phase = 0;
    bool alive = true;
    while (alive && walk.next(u)) {
      const int r0 = u.m0 + (int)rank * BM + quarter * 32, n0 = u.n0;
      const bool none = MODE == WGRAD && u.num_kb == 0;
      if (none && f32 && !PARTS) continue;  // nothing to add
      uint32_t t_row = 0;
      if (!none) {
        if (!bb::mbar_wait_warp(&tmem_full[acc], acc_phase, abort_flag, p.status)) { alive = false; break; }
        bb::tc_fence_after_sync();
        t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * BN);
      }
      const int width = f32 ? 32 : 64, npanels = BN / width;
      const long long base = MODE == WGRAD ? u.e * p.expert_stride : 0;
      const __nv_bfloat16* bias = has_bias ? reinterpret_cast<const __nv_bfloat16*>(p.bias) + (long long)u.e * p.n : nullptr;
#pragma unroll 1
      for (int pn = eg; pn < npanels; pn += 2) {
        const int nb = n0 + pn * width;
        const bool some = nb < cols && r0 < u.end;
        if (has_aux && some) {
          uint4 ax[8];
          slab_fetch_bf16(reinterpret_cast<const __nv_bfloat16*>(p.aux), p.ld_aux, r0, nb, u.end, cols, lane, ax);
          slab_put(slab, lane, ax);
        }
        float v[64];
        if (none) {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = 0.f;
        } else {
          uint32_t r[32];
          bb::tmem_ld_32x32b_x32(t_row + pn * width, r);
          bb::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
          if (!f32) {
            bb::tmem_ld_32x32b_x32(t_row + pn * width + 32, r);
            bb::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[32 + i] = __uint_as_float(r[i]);
          }
        }
        if (pn + 2 >= npanels && !none) {
          // this warp has read its share of the accumulator
          bb::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if (PAIR) bb::mbar_arrive_cluster_relaxed(bb::mapa_shared(bb::smem_u32(&tmem_empty[acc]), 0));
            else bb::mbar_arrive(&tmem_empty[acc]);
          }
        }
        if (!some) continue;
        if (f32) {
          panel_store_row_f32(slab, lane, v);
          __syncwarp();
          if (PARTS) slab_flush_f32<false>(slab, p.parts + (long long)u.part * p.experts * p.expert_stride + base, p.ldd, r0, nb, u.end, cols, lane);
          else slab_flush_f32<true>(slab, reinterpret_cast<float*>(p.D) + base, p.ldd, r0, nb, u.end, cols, lane);
          __syncwarp();
          continue;
        }
        finish_panel<MODE>(p, slab, bias, has_bias, dual, has_aux, base, r0, nb, u.end, cols, lane, v);
      }
      if (!none && ++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  }

  bb::tc_fence_before_sync();
  if (PAIR) {
    // neither CTA leaves (or frees TMEM) while the other may still signal its barriers
    __syncwarp();
    bb::cluster_sync();
    if (warp == MMA_WARP) bb::tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
  } else {
    __syncthreads();
    if (warp == MMA_WARP) bb::tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// Few tiles and a long reduction: a cluster of 2, 4 or 8 CTAs shares a tile's reduction, each over a run of its k-blocks (a k-block takes 0.28 us with
// 128 columns, 0.37 with 256, however idle the GPU is; its MMAs alone, of 128 rows whether they exist or not, 0.14 and 0.27).  Panels of 64 columns are dealt out to the CTAs; each sends its sums of the others' panels into their
// operand stages, by then unused, and adds what it received to its own in the order of the CTAs: the same bits every time.  A cluster has one tile.
// Received panels: [other CTA][run of 32 rows][16 bytes of a row][row], so that a warp's access is one run of memory.
template <int MODE, int BN>
__global__ void __launch_bounds__(THREADS<false>, 1)
grouped_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GroupParams p) {
  using C = Cfg<BN, false>;
  constexpr int NP = BN / 64, PART_BYTES = 32 * 64 * 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * A_STAGE_BYTES;
  uint8_t* panels = smem + C::STAGES * C::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(panels + EPI_WARPS * SLAB_BYTES);      // [STAGES]
  uint64_t* empty_bar = full_bar + C::STAGES;       // [STAGES]
  uint64_t* tmem_full = empty_bar + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 2);                                     // [experts + 1]

  const int warp = bb::warp_index(), lane = threadIdx.x & 31;
  const int S = p.split, ks = (int)bb::cluster_ctarank();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < C::STAGES; ++s) { bb::mbar_init(&full_bar[s], 1); bb::mbar_init(&empty_bar[s], 1); }
    bb::mbar_init(tmem_full, 1);
    bb::fence_barrier_init();
    bb::tma_prefetch_desc(&tmA);
    bb::tma_prefetch_desc(&tmB);
  }
  if (warp == MMA_WARP) { bb::tmem_alloc(tmem_slot, BN); bb::tmem_relinquish(); }
  bb::pdl_sync();
  if (warp == EPI_WARP) read_offsets(p, start, lane);
  bb::tc_fence_before_sync();
  __syncthreads();
  bb::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  zero_the_rest(p, start, THREADS<false>);
  Walk<false, BN, BM> walk(p, start, nullptr, (int)bb::cluster_id(), (int)gridDim.x / S);
  Unit u = {};
  const bool some = walk.next(u);
  const int kb0 = ks * u.num_kb / S, num_kb = (ks + 1) * u.num_kb / S - kb0;                       // (at least one: the host sees to it)

  const int eg = (warp - EPI_WARP) >> 2, quarter = warp & 3, r0 = u.m0 + quarter * 32, cols = p.n;
  const bool dual = MODE == ROWS && p.epi == BB_EPI_BIAS_GELU;
  const bool has_aux = MODE == ROWS_T && p.epi == BB_EPI_MUL_DGELU, has_bias = MODE == ROWS && (p.epi == BB_EPI_BIAS || dual);
  uint8_t* slab = panels + (warp - EPI_WARP) * SLAB_BYTES;
  const int own = ks + eg * S, nb_own = u.n0 + own * 64;    // this warp's panel
  bool summed = false;
  if (!some) {
  } else if (warp == TMA_WARP_0 || warp == TMA_WARP_1) {
    const int turn = warp == TMA_WARP_1 ? 1 : 0;
    int s = 0; uint32_t phase = 0;
    bool alive = true;
    int at = p.rotate ? u.ni % num_kb : 0;
    for (int kb = 0; kb < num_kb; ++kb) {
      if ((s & 1) == turn) {
        if (!bb::mbar_wait_warp(&empty_bar[s], phase ^ 1, abort_flag, p.status)) { alive = false; break; }
        uint8_t* a = sA + s * A_STAGE_BYTES;
        uint8_t* b = sB + s * C::B_STAGE_BYTES;
        const int k0 = (kb0 + at) * BK;
        if (bb::elect_one()) {
          bb::mbar_arrive_expect_tx(&full_bar[s], p.stage_bytes);
          bb::tma_load_2d(a, &tmA, &full_bar[s], k0, u.m0);
          if constexpr (MODE == ROWS) {
            bb::tma_load_3d(b, &tmB, &full_bar[s], k0, u.n0, u.e);
          } else {
#pragma unroll
            for (int j = 0; j < C::B_ROWS / 64; ++j) bb::tma_load_3d(b + j * 8192, &tmB, &full_bar[s], u.n0 + 64 * j, k0, u.e);
          }
        }
        __syncwarp();
      }
      if (++at == num_kb) at = 0;
      if (++s == C::STAGES) { s = 0; phase ^= 1; }
    }
    if (!alive) {
      // copies still in flight get time to land (bounded)
      const uint64_t t0 = bb::globaltimer_ns();
      while (bb::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
  } else if (warp == MMA_WARP) {
    constexpr uint32_t B_MN = MODE != ROWS;
    constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | (B_MN << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
    constexpr uint32_t B_LBO = B_MN ? 8192u : 16u, B_STEP = B_MN ? 2048u : 32u;
    int s = 0; uint32_t phase = 0;
    for (int kb = 0; kb < num_kb; ++kb) {
      if (!bb::mbar_wait_warp(&full_bar[s], phase, abort_flag, p.status)) break;
      bb::tc_fence_after_sync();
      if (bb::elect_one()) {
        const uint64_t ad0 = bb::make_smem_desc_sw128(bb::smem_u32(sA + s * A_STAGE_BYTES), 16u, 1024u);
        const uint64_t bd0 = bb::make_smem_desc_sw128(bb::smem_u32(sB + s * C::B_STAGE_BYTES), B_LBO, 1024u);
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k)
          bb::umma_f16(tmem_base, ad0 + (uint64_t)(k * (32u >> 4)), bd0 + (uint64_t)(k * (B_STEP >> 4)), IDESC, (kb > 0 || k > 0) ? 1u : 0u);
        bb::umma_commit(&empty_bar[s]);
        if (kb == num_kb - 1) bb::umma_commit(tmem_full);
      }
      __syncwarp();
      if (++s == C::STAGES) { s = 0; phase ^= 1; }
    }
  } else {
    // the pre-activation of the own panel comes under the main loop
    if (has_aux && own < NP && nb_own < cols && r0 < u.end) {
      uint4 ax[8];
      slab_fetch_bf16(reinterpret_cast<const __nv_bfloat16*>(p.aux), p.ld_aux, r0, nb_own, u.end, cols, lane, ax);
      slab_put(slab, lane, ax);
    }
    summed = bb::mbar_wait_warp(tmem_full, 0, abort_flag, p.status) && r0 < u.end;
    bb::tc_fence_after_sync();
  }
  __syncwarp();
  // every CTA's MMAs have retired, so its stages can receive (all of its copies have landed)
  bb::cluster_sync();
  const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
  if (summed) {
    int turn = 0;
    for (int i = 1; i < S; ++i) {                           // the CTAs start with different owners
      const int owner = ks + i < S ? ks + i : ks + i - S, slot = ks < owner ? ks : ks - 1;
      for (int pn = owner, from = slot; pn < NP; pn += S, from += S - 1) {
        if ((turn++ & 1) != eg || u.n0 + pn * 64 >= cols) continue;
        const uint32_t dst = bb::mapa_shared(bb::smem_u32(smem) + (from * p.quarters + quarter) * PART_BYTES + lane * 16, owner);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          bb::tmem_ld_32x32b_x32(t_row + pn * 64 + h * 32, r);
          bb::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) bb::st_shared_cluster_v4(dst + (h * 8 + j) * 512, r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        }
      }
    }
  }
  __syncwarp();
  bb::cluster_sync();
  if (summed && own < NP && nb_own < cols) {
    float v[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = 0.f;
    const uint8_t* part = smem + (eg * (S - 1) * p.quarters + quarter) * PART_BYTES + lane * 16;
    for (int t = 0; t < S; ++t) {
      if (t == ks) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          bb::tmem_ld_32x32b_x32(t_row + own * 64 + h * 32, r);
          bb::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[h * 32 + i] += __uint_as_float(r[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float4 q = *reinterpret_cast<const float4*>(part + j * 512);
          v[4 * j] += q.x; v[4 * j + 1] += q.y; v[4 * j + 2] += q.z; v[4 * j + 3] += q.w;
        }
        part += p.quarters * PART_BYTES;
      }
    }
    const __nv_bfloat16* bias = has_bias ? reinterpret_cast<const __nv_bfloat16*>(p.bias) + (long long)u.e * p.n : nullptr;
    finish_panel<MODE>(p, slab, bias, has_bias, dual, has_aux, 0, r0, nb_own, u.end, cols, lane, v);
  }
  bb::tc_fence_before_sync();
  __syncthreads();
  if (warp == MMA_WARP) bb::tmem_dealloc(tmem_base, BN);
}

// The sums of the parts, and of the column tiles for the bias (see ColumnSums), in their order; four weights a thread, one bias (with four, 16 tiles of 15000
// took 6 us longer)
struct Join { const float* parts; int count; long long values; __nv_bfloat16* out; float* accum; };
__global__ void __launch_bounds__(256)
grouped_join_kernel(const Join bias, const Join weight, int bias_blocks) {
  bb::pdl_sync();
  if ((int)blockIdx.x < bias_blocks) {
    const long long i = blockIdx.x * 256LL + threadIdx.x;
    if (i >= bias.values) return;
    float s = 0.f;
#pragma unroll 4
    for (int t = 0; t < bias.count; ++t) s += bias.parts[t * bias.values + i];
    if (bias.accum) bias.accum[i] += s;
    else bias.out[i] = __float2bfloat16(s);
    return;
  }
  const long long i = (((int)blockIdx.x - bias_blocks) * 256LL + threadIdx.x) * 4;
  if (i >= weight.values) return;            // (a multiple of 64)
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int t = 0; t < weight.count; ++t) {
    const float4 q = *reinterpret_cast<const float4*>(weight.parts + t * weight.values + i);
    s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
  }
  if (weight.accum) {
    float4* to = reinterpret_cast<float4*>(weight.accum + i);
    const float4 q = *to;
    *to = make_float4(q.x + s.x, q.y + s.y, q.z + s.z, q.w + s.w);
  } else {
    *reinterpret_cast<uint2*>(weight.out + i) = make_uint2(bb::pack_bf16x2(s.x, s.y), bb::pack_bf16x2(s.z, s.w));
  }
}

// ---------------------------------------------------------------- bias gradients
// db_e = sum of its rows of dy, where no weight gradient carries it along.  A cluster of CTAs shares an expert's rows for 128 columns: every CTA sums a run of them (16 rows of 256 bytes at a
// time, four such steps in flight), the first adds the CTAs' sums in their order through distributed shared memory.  16384 rows of 4096, 8 experts, 30 us
// (4.4 TB/s): a CTA's start and the two cluster barriers weigh on runs of 256 rows; longer ones leave SMs idle (four CTAs an expert 31, two 42).
constexpr int COLSUM_COLS = 128, COLSUM_MOST = 8, COLSUM_U = 4;

__device__ __forceinline__ int clamped(const int* offsets, int e, int rows) {
  const int v = __ldca(offsets + e);
  return v < 0 ? 0 : v > rows ? rows : v;
}

__global__ void __launch_bounds__(256)
grouped_colsum_kernel(const __nv_bfloat16* dy, long long ld, const int* offsets, int rows, int n, __nv_bfloat16* out, float* accum) {
  __shared__ float part[16][COLSUM_COLS], mine[COLSUM_COLS];
  __shared__ int range[2];
  bb::pdl_sync();
  const int rank = (int)bb::cluster_ctarank(), parts = (int)bb::cluster_nctarank(), e = blockIdx.z;
  const int lane16 = threadIdx.x & 15, line = threadIdx.x >> 4, col = blockIdx.y * COLSUM_COLS + lane16 * 8;
  if (threadIdx.x < 32) {
    // the expert's rows: offsets that do not ascend are cut as the products cut them
    int lo = 0;
    for (int i = threadIdx.x; i <= e; i += 32) lo = max(lo, clamped(offsets, i, rows));
    lo = __reduce_max_sync(0xffffffffu, lo);
    if (threadIdx.x == 0) { range[0] = lo; range[1] = max(lo, clamped(offsets, e + 1, rows)); }
  }
  __syncthreads();
  const int each = (range[1] - range[0] + parts - 1) / parts, from = min(range[1], range[0] + rank * each), to = min(range[1], from + each);
  float v[8] = {};
  if (col < n) {
    int r = from + line;
    for (; r + (COLSUM_U - 1) * 16 < to; r += COLSUM_U * 16) {
      uint4 q[COLSUM_U];
#pragma unroll
      for (int u = 0; u < COLSUM_U; ++u) q[u] = __ldca(reinterpret_cast<const uint4*>(dy + (long long)(r + u * 16) * ld + col));
#pragma unroll
      for (int u = 0; u < COLSUM_U; ++u) {
        float f[8];
        unpack8(q[u], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += f[i];
      }
    }
    for (; r < to; r += 16) {
      float f[8];
      unpack8(__ldca(reinterpret_cast<const uint4*>(dy + (long long)r * ld + col)), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += f[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[line][lane16 * 8 + i] = v[i];
  __syncthreads();
  if (threadIdx.x < COLSUM_COLS) {
    float s = 0.f;
#pragma unroll
    for (int l = 0; l < 16; ++l) s += part[l][threadIdx.x];
    mine[threadIdx.x] = s;
  }
  bb::cluster_sync();
  const int c = blockIdx.y * COLSUM_COLS + threadIdx.x;
  if (rank == 0 && threadIdx.x < COLSUM_COLS && c < n) {
    float s = 0.f;
    for (int p = 0; p < parts; ++p) {
      float o;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(bb::mapa_shared(bb::smem_u32(&mine[threadIdx.x]), p)) : "memory");
      s += o;
    }
    if (accum) accum[(long long)e * n + c] += s;
    else out[(long long)e * n + c] = __float2bfloat16(s);
  }
  bb::cluster_sync();               // no CTA leaves before its sums were read
}

// ---------------------------------------------------------------- host side
int refuse(const char* msg) { bb_set_last_error_msg(msg); return BB_ERR_INVALID_ARG; }

// Whether S CTAs can share a tile's reduction: each has a k-block at least, and what it receives fits its operand stages
int quarters_of(const bb_grouped_desc* d) { return d->rows < BM ? (d->rows + 31) / 32 : BM / 32; }
constexpr int MOST_PARTS = 32;
template <int BN> bool can_split(const bb_grouped_desc* d, int S, int num_kb) {
  const int owned = (BN / 64 + S - 1) / S;
  return num_kb >= S && num_kb < INT_MAX / 8 && owned * (S - 1) * quarters_of(d) * 8192 <= Cfg<BN, false>::STAGES * Cfg<BN, false>::STAGE_BYTES;
}
template <int BN> cudaLaunchConfig_t split_config(int S, long long tiles, cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles < 1 ? 1 : tiles) * S); cfg.blockDim = dim3(THREADS<false>); cfg.dynamicSmemBytes = Cfg<BN, false>::SMEM_BYTES;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cfg;
}
// Clusters of S CTAs that the device holds at the same time (of 2: 74, of 4: 33, of 8: 15); 0 when it cannot be asked
template <int MODE, int BN> int clusters_at_once(int S) {
  static std::atomic<int> cache[64][9];
  const int dev = bb_current_device();
  if (dev < 0) return 0;
  int n = cache[dev][S].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = split_config<BN>(S, 1, attr);
    if (cudaFuncSetAttribute(grouped_split_kernel<MODE, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN, false>::SMEM_BYTES) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, grouped_split_kernel<MODE, BN>, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    if (n <= 0) n = -1;
    cache[dev][S].store(n, std::memory_order_relaxed);
  }
  return n > 0 ? n : 0;
}

template <int MODE, int BN, bool PAIR, bool PARTS = false>
int launch(const bb_grouped_desc* d, cudaStream_t stream, int split = 1) {
  using C = Cfg<BN, PAIR>;
  CUtensorMap tmA, tmB;
  GroupParams p = {};
  p.rows = d->rows; p.experts = d->experts; p.epi = d->epilogue; p.offsets = d->offsets;
  p.D = d->out; p.D2 = d->out2; p.bias = d->bias; p.aux = d->aux;
  p.ldd = d->ld_out; p.ld_aux = d->ld_aux ? d->ld_aux : d->ld_out;
  const int bias_tiles = d->bias_grad || d->bias_accum ? (d->k + BN - 1) / BN * split : 0;
  p.bias_grad = (__nv_bfloat16*)d->bias_grad; p.bias_accum = d->bias_accum; p.bias_parts = bias_tiles > 1 ? d->bias_parts : nullptr;
  p.split = split;
  const long long bias_values = (long long)d->experts * d->n, weight_values = bias_values * d->k;
  if (PARTS) p.parts = d->bias_parts + bias_tiles * bias_values;
  p.status = bb_device_status_word();
  int rc;
  long long tiles;
  const long long row_tiles = (long long)d->rows / C::TILE_M + (d->rows < d->experts ? d->rows : d->experts);      // at most
  if (MODE == WGRAD) {
    p.stage_bytes = C::STAGE_BYTES;
    p.n = d->n; p.k = d->k; p.expert_stride = (long long)d->n * d->k; p.ldd = d->k;
    rc = bbhost::encode_2d(&tmA, d->x, d->rows, d->n, d->ld_x, 64, BK);
    if (!rc) rc = bbhost::encode_2d(&tmB, d->weight, d->rows, d->k, d->ld_weight, 64, BK);
    tiles = (long long)d->experts * ((d->n + C::TILE_M - 1) / C::TILE_M) * ((d->k + BN - 1) / BN) * split;
  } else {
    p.n = MODE == ROWS ? d->n : d->k; p.k = MODE == ROWS ? d->k : d->n;
    // no expert has more rows than there are: of few rows a tile loads those alone (what stands in shared memory below them makes rows that are
    // not stored).  14 rows of 8 experts, 4096 x 1024, from memory: 17.5 -> 15.4 us, with `rotate` 14.8.
    // (Tiles of 64 columns and 16 stages of 16 rows took 22.)
    const int box = d->rows < BM ? (d->rows + 7) & ~7 : BM;
    p.stage_bytes = box * BK * 2 + C::B_STAGE_BYTES;
    p.rotate = d->rows < BM;
    rc = bbhost::encode_2d(&tmA, d->x, d->rows, p.k, d->ld_x, BK, box);
    // (the third dimension ends every expert's weight: what a box reads beyond it is zeros)
    if (!rc) rc = bbhost::encode_seqs(&tmB, d->weight, d->experts, d->n, d->k, d->k, 64, MODE == ROWS ? C::B_ROWS : BK);
    tiles = row_tiles * ((p.n + BN - 1) / BN);
  }
  if (rc) return rc;
  if (tiles > INT_MAX / 2 / split) return refuse("bb_grouped_gemm: more tiles than one launch covers");
  if constexpr (MODE != WGRAD && !PAIR) {
    if (split > 1) {
      p.quarters = quarters_of(d);
      BB_ONCE_PER_DEVICE(BB_CUDA_CHECK(cudaFuncSetAttribute(grouped_split_kernel<MODE, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES)));
      cudaLaunchAttribute attr[2];
      cudaLaunchConfig_t cfg = split_config<BN>(split, tiles, attr);
      cfg.stream = stream;
      if (bb_back_to_back > 0) cfg.numAttrs = 2;
      BB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, grouped_split_kernel<MODE, BN>, tmA, tmB, p));
      return BB_OK;
    }
  }
  BB_ONCE_PER_DEVICE(BB_CUDA_CHECK(cudaFuncSetAttribute(grouped_gemm_kernel<MODE, BN, PAIR, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES)));
  int workers = PAIR ? bb_num_sms() / 2 : bb_num_sms();
  if (d->max_ctas > 0 && d->max_ctas / (PAIR ? 2 : 1) < workers) workers = d->max_ctas / (PAIR ? 2 : 1);
  if (workers < 1) workers = 1;
  if (d->max_ctas < 0 || tiles < workers) workers = tiles < 1 ? 1 : (int)tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((PAIR ? 2 : 1) * workers); cfg.blockDim = dim3(THREADS<MODE == WGRAD>); cfg.dynamicSmemBytes = C::SMEM_BYTES; cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 0;
  if (bb_back_to_back > 0) cfg.numAttrs = 1;
  if (PAIR) {
    if (!cfg.numAttrs) attr[0] = attr[1];
    ++cfg.numAttrs;
  }
  BackToBack overlap((bias_tiles > 1 || p.parts) && d->max_ctas == 0);
  BB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, grouped_gemm_kernel<MODE, BN, PAIR, PARTS>, tmA, tmB, p));
  if (bias_tiles > 1 || p.parts) {
    const Join bias = {p.bias_parts, bias_tiles, bias_values, p.bias_grad, p.bias_accum};
    const bool f32 = d->epilogue == BB_EPI_ACCUM_F32;
    const Join weight = {p.parts, split, weight_values, f32 ? nullptr : (__nv_bfloat16*)d->out, f32 ? (float*)d->out : nullptr};
    const long long bias_blocks = bias_tiles > 1 ? (bias_values + 255) / 256 : 0, weight_blocks = p.parts ? (weight_values + 1023) / 1024 : 0;
    BB_CUDA_CHECK(bb_launch(grouped_join_kernel, (unsigned)(bias_blocks + weight_blocks), 256, 0, stream, bias, weight, (int)bias_blocks));
  }
  return BB_OK;
}

// Floats of scratch of a weight gradient in `split` parts, with tiles of `bn` columns
long long part_values(int n, int k, int experts, int bn, int split, bool bias) {
  const long long values = (long long)experts * n;
  return (bias ? (long long)((k + bn - 1) / bn) * split * values : 0) + (split > 1 ? split * values * k : 0);
}

// The tile by the time that it is expected to take, as for stored products (gemm_tcgen05.cu), with the number of row tiles that evenly spread rows
// would make: the host does not know the offsets.  Every expert adds half a tile of overhang.  us, pairs | 128 x 256 | 128 x 128, without
// an epilogue: 16384 rows of 8 experts, 4096 x 1024, 103 | 116 | 144 (1.33 PFLOP/s); 16384 of 64, 1024 x 1024, 44 | 49 | 54; 4096 of 64,
// 2048 x 512, 33 | 31 | 31; 2000 of 16, 1416 x 776, 19 | 15 | 16; 1024 of 8, 1024 x 256, 9.2 | 8.3 | 6.8; 14 of 8, 4096 x 1024, 19 | 15 | 20.  Tiles of 64
// columns were never quicker (248 | 7.4 | 26 us).
// A shared reduction where one wave of clusters holds all tiles that there may be, every CTA has four k-blocks or more, and it is expected to be quicker by a
// twentieth; the exchange grows with the CTAs and with the rows.  us, whole | shared by 2 | 4 | 8, the quickest kinds: 14 rows of 8 experts, 1024 x 4096, 23 | 17 |
// 17 | 24; 2 rows of it 22 | 15 | 11 | 11; 1024 rows of 8, 512 x 2048, 14 | 12 | 13; 2000 of 8, 512 x 4096, 23 | 20 | 27; 1 row, 4096 x 4096, 22 | 15 | 12 | 20;
// 14 of 8, 4096 x 1024, 14.5 | 21 | 32.
struct Plan { int kind, split; };
struct Kind { int bn; bool pair; double kblock, wave, once, shared; };
constexpr Kind KINDS[3] = {{256, true, 0.32, 1.9, 5.0, 0}, {256, false, 0.375, 1.8, 3.7, 6.0}, {128, false, 0.283, 1.0, 3.7, 5.0}};
int workers_of(const bb_grouped_desc* d, const Kind& k) {
  int workers = bb_num_sms();
  if (d->max_ctas > 0 && d->max_ctas < workers) workers = d->max_ctas;
  return !k.pair ? workers : workers > 1 ? workers / 2 : 1;
}
bool allowed(const bb_grouped_desc* d, const Kind& k) { return !(d->tile_n && d->tile_n != k.bn) && !(d->cta_pair && (d->cta_pair > 0) != k.pair); }

template <int MODE> Plan plan(const bb_grouped_desc* d) {
  const double used = d->rows < d->experts ? d->rows : d->experts, each = d->rows / used;
  int best = 0, best_split = 1;
  double best_us = -1;
  for (int i = 0; i < 3; ++i) {
    const Kind& k = KINDS[i];
    if (!allowed(d, k)) continue;
    const int tm = k.pair ? 2 * BM : BM, n = MODE == ROWS ? d->n : d->k, num_kb = ((MODE == ROWS ? d->k : d->n) + BK - 1) / BK;
    const double per = each / tm + 0.5, tiles = used * (per > 1 ? per : 1) * ((n + k.bn - 1) / k.bn);
    const double whole = ceil(tiles / workers_of(d, k)) * (num_kb * k.kblock + k.wave) + k.once;
    if (d->split < 2 && (best_us < 0 || whole < best_us)) { best_us = whole; best = i; best_split = 1; }
    const long long most = ((long long)d->rows / BM + (long long)used) * ((n + k.bn - 1) / k.bn);
    for (int S = 2; S <= 8 && !k.pair && d->max_ctas == 0 && d->split != 1; S *= 2) {
      if (d->split > 1 && S != d->split) continue;
      if (!(k.bn == 128 ? can_split<128>(d, S, num_kb) : can_split<256>(d, S, num_kb))) continue;
      if (d->split < 2 && (num_kb < 4 * S || most > (k.bn == 128 ? clusters_at_once<MODE, 128>(S) : clusters_at_once<MODE, 256>(S)))) continue;
      const double us = 1.05 * ((num_kb + S - 1) / S * k.kblock + k.shared + 0.2 * quarters_of(d) * S);
      if (best_us < 0 || us < best_us) { best_us = us; best = i; best_split = S; }
    }
  }
  return {best_us < 0 ? -1 : best, best_split};
}

// A weight gradient of few tiles takes its reductions in parts, each a unit of its own, whose sums a second kernel adds up.  The time of one wave is that of the
// longest expert, k-blocks take up to half as long again when all SMs ask for them, and the warp that sums the bias 0.7 us for one; the join costs a launch, and
// the parts' way to memory and back.  Fitted to 90 sizes from 400 to 20000 rows, 1 to 64 experts, with and without a bias: whole reductions take 1.21 times
// the quickest tile and number of parts in the mean, these 1.02.  us, whole | in parts, with the bias: 12874 rows of 1 expert, 352 x 208, 74 | 17; 8520 of 1,
// 1056 x 672, 45 | 23; 17253 of 13, 88 x 536, 25 | 17; 9249 of 15, 120 x 72, 19 | 12.
template <> Plan plan<WGRAD>(const bb_grouped_desc* d) {
  static const int counts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24};
  const double used = d->rows < d->experts ? d->rows : d->experts, each = d->rows / used / BK, values = (double)d->experts * d->n * d->k;
  const bool bias = d->bias_grad || d->bias_accum;
  Plan best = {-1, 1};
  double best_us = -1;
  for (int i = 0; i < 3; ++i) {
    const Kind& k = KINDS[i];
    if (!allowed(d, k)) continue;
    const int tm = k.pair ? 2 * BM : BM, workers = workers_of(d, k), cols = (d->k + k.bn - 1) / k.bn;
    const double tiles = (double)d->experts * ((d->n + tm - 1) / tm) * cols;
    for (int at = 0; at < (int)(sizeof(counts) / sizeof(counts[0])); ++at) {
      const int S = d->split ? d->split : counts[at];
      if (!d->split && S > 1 && (tiles * S > 2 * workers || each < 2 * S)) break;
      if (S > 1 && d->bias_parts_bytes < 4 * part_values(d->n, d->k, d->experts, k.bn, S, bias)) break;
      double kblock = k.kblock * (1 + 0.5 * (tiles * S < workers ? tiles * S / workers : 1));
      if (bias && kblock < 0.7 / cols) kblock = 0.7 / cols;
      const double longest = tiles * S <= workers ? each * (1 + 0.8 * (1 - 1 / used)) : each;
      double us = ceil(tiles * S / workers) * ((longest / S + 0.5) * kblock + k.wave) + k.once;
      if (S > 1) us = 1.05 * (us + 1 + 0.1 * S + 0.8e-6 * S * values);
      if (best_us < 0 || us < best_us) { best_us = us; best = {i, S}; }
      if (d->split) break;
    }
  }
  return best;
}

template <int MODE> int choose(const bb_grouped_desc* d, cudaStream_t stream) {
  const Plan b = plan<MODE>(d);
  if (b.kind < 0) return refuse("bb_grouped_gemm: a reduction that cannot be split like this, or not with this scratch");
  if constexpr (MODE == WGRAD) {
    if (b.split > 1)
      return b.kind == 0 ? launch<MODE, 256, true, true>(d, stream, b.split) : b.kind == 1 ? launch<MODE, 256, false, true>(d, stream, b.split) : launch<MODE, 128, false, true>(d, stream, b.split);
  }
  return b.kind == 0 ? launch<MODE, 256, true>(d, stream, b.split) : b.kind == 1 ? launch<MODE, 256, false>(d, stream, b.split) : launch<MODE, 128, false>(d, stream, b.split);
}

bool bad_sizes(const bb_grouped_desc* d) {
  return d->rows <= 0 || d->rows > INT_MAX - 1024 || d->n <= 0 || d->n > WIDEST || d->k <= 0 || d->k > WIDEST || (d->n & 7) || (d->k & 7) || d->experts <= 0 || d->experts > MAX_EXPERTS;
}
bool too_wide(int n) { return n > 65535 * COLSUM_COLS; }
bool bad_matrix(const void* p, long long ld, int cols) { return !p || ((uintptr_t)p & 15) || ld < cols || (ld & 7); }
}  // namespace

extern "C" int bb_grouped_max_experts(void) { return MAX_EXPERTS; }

extern "C" long long bb_grouped_bias_bytes(int n, int k, int experts) {
  return n <= 0 || k <= 0 || experts <= 0 ? 0 : 4LL * ((k + 127LL) / 128) * experts * n;
}

extern "C" long long bb_grouped_weight_bytes(int rows, int n, int k, int experts, int with_bias) {
  if (n <= 0 || k <= 0 || experts <= 0) return 0;
  const long long least = with_bias ? bb_grouped_bias_bytes(n, k, experts) : 0;
  bb_grouped_desc d = {};
  d.mode = BB_GROUPED_WEIGHT; d.rows = rows; d.n = n; d.k = k; d.experts = experts; d.bias_parts_bytes = LLONG_MAX;
  float none;
  if (with_bias) d.bias_accum = &none;               // (not written to)
  if (bad_sizes(&d)) return least;
  const Plan b = plan<WGRAD>(&d);
  const long long bytes = b.split > 1 ? 4 * part_values(n, k, experts, b.kind == 2 ? 128 : 256, b.split, with_bias) : 0;
  return bytes > least ? bytes : least;
}

extern "C" int bb_grouped_gemm(const bb_grouped_desc* d, void* stream) {
  if (!d || !d->offsets || ((uintptr_t)d->offsets & 3) || bad_sizes(d))
    return refuse("bb_grouped_gemm: null pointer, a size that is not positive or close to 2^31, n or k not a multiple of 8, or more than 256 experts");
  const bool turned = d->mode == BB_GROUPED_INPUT, wgrad = d->mode == BB_GROUPED_WEIGHT;
  if (d->mode != BB_GROUPED_ROWS && !turned && !wgrad) return refuse("bb_grouped_gemm: an unknown mode");
  // (a tile of a weight gradient sums all of an expert's rows: about 0.3 us for 64 of them, and a wait inside the kernel has 2 s)
  if (wgrad && d->rows > (1 << 27)) { bb_set_last_error_msg("bb_grouped_gemm: a weight gradient over more than 2^27 rows"); return BB_ERR_TOO_LARGE; }
  if (bad_matrix(d->x, d->ld_x, d->mode == BB_GROUPED_ROWS ? d->k : d->n) || bad_matrix(d->weight, wgrad ? d->ld_weight : d->k, d->k) || !d->out ||
      ((uintptr_t)d->out & 15) || (!wgrad && bad_matrix(d->out, d->ld_out, turned ? d->k : d->n)))
    return refuse("bb_grouped_gemm: operands are 16-byte aligned, with rows of a multiple of 8 values that do not overlap");
  if ((d->tile_n != 0 && d->tile_n != 128 && d->tile_n != 256) || (d->cta_pair > 0 && d->tile_n == 128))
    return refuse("bb_grouped_gemm: tile_n is 128 or 256, of a CTA pair 256");
  if (d->split < 0 || (wgrad ? d->split > MOST_PARTS : d->split != 0 && d->split != 1 && d->split != 2 && d->split != 4 && d->split != 8) ||
      (d->split > 1 && (wgrad ? !d->bias_parts : d->cta_pair > 0 || d->max_ctas > 0)))
    return refuse("bb_grouped_gemm: split is 1, 2, 4 or 8, for single CTAs without max_ctas, or up to 32 parts of a weight gradient, which take scratch");
  if ((d->bias_grad || d->bias_accum) && (!wgrad || (d->bias_grad && d->bias_accum) || ((uintptr_t)d->bias_grad & 1) || ((uintptr_t)d->bias_accum & 3)))
    return refuse("bb_grouped_gemm: a bias gradient goes with a weight gradient, to one place");
  if (wgrad && (((uintptr_t)d->bias_parts & 15) || (!d->bias_parts && d->bias_parts_bytes != 0))) return refuse("bb_grouped_gemm: scratch that is null or not 16-byte aligned");
  if ((d->bias_grad || d->bias_accum) && (!d->bias_parts || d->bias_parts_bytes < bb_grouped_bias_bytes(d->n, d->k, d->experts)))
    return refuse("bb_grouped_gemm: a bias gradient takes bb_grouped_bias_bytes() of scratch");
  const int e = d->epilogue;
  if (wgrad ? (e != BB_EPI_STORE && e != BB_EPI_ACCUM_F32)
            : turned ? (e != BB_EPI_STORE && e != BB_EPI_MUL_DGELU) : (e != BB_EPI_STORE && e != BB_EPI_BIAS && e != BB_EPI_BIAS_GELU))
    return refuse("bb_grouped_gemm: an epilogue that this product does not have");
  if (!wgrad && !turned && e != BB_EPI_STORE && (!d->bias || ((uintptr_t)d->bias & 15)))
    return refuse("bb_grouped_gemm: the epilogue takes a bias, 16-byte aligned");
  if (e == BB_EPI_BIAS_GELU && (!d->out2 || ((uintptr_t)d->out2 & 15))) return refuse("bb_grouped_gemm: the epilogue takes a second output, 16-byte aligned");
  if (e == BB_EPI_MUL_DGELU && bad_matrix(d->aux, d->ld_aux ? d->ld_aux : d->ld_out, d->k))
    return refuse("bb_grouped_gemm: the epilogue takes the pre-activation, 16-byte aligned");
  if (int rc = bbhost::bind_context()) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  return wgrad ? choose<WGRAD>(d, s) : turned ? choose<ROWS_T>(d, s) : choose<ROWS>(d, s);
}

extern "C" int bb_grouped_colsum(const void* dy, long long ld, const int* offsets, int experts, void* out_bf16, float* accum, int rows, int n, void* stream) {
  if (rows <= 0 || n <= 0 || (n & 7) || experts <= 0 || experts > MAX_EXPERTS || !offsets || ((uintptr_t)offsets & 3) || bad_matrix(dy, ld, n) || (!out_bf16 == !accum) ||
      ((uintptr_t)out_bf16 & 1) || ((uintptr_t)accum & 3))
    return refuse("bb_grouped_colsum: null or misaligned pointer, a size that is not positive, n no multiple of 8, more than 256 experts, or not one output");
  if (too_wide(n)) return refuse("bb_grouped_colsum: more columns than one launch covers");
  int parts = 1;
  while (parts < COLSUM_MOST && rows / experts >= 64 * parts) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, (n + COLSUM_COLS - 1) / COLSUM_COLS, experts); cfg.blockDim = dim3(256); cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = bb_back_to_back > 0 ? 2 : 1;
  BB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, grouped_colsum_kernel, (const __nv_bfloat16*)dy, ld, offsets, rows, n, (__nv_bfloat16*)out_bf16, accum));
  return BB_OK;
}

// ---------------------------------------------------------------- two layers per expert
namespace {
bb_grouped_desc part_of(const bb_expert_mlp_desc* m, int mode, int n, int k, int epilogue) {
  bb_grouped_desc d = {};
  d.mode = mode; d.rows = m->rows; d.n = n; d.k = k; d.experts = m->experts; d.epilogue = epilogue; d.offsets = m->offsets; d.max_ctas = m->max_ctas;
  return d;
}
// (all that the later products of a call could refuse, before the first is launched)
bool bad_mlp(const bb_expert_mlp_desc* m) {
  return !m || m->rows <= 0 || m->rows > INT_MAX - 1024 || m->in <= 0 || m->in > WIDEST || m->inner <= 0 || m->inner > WIDEST || m->out <= 0 || m->out > WIDEST || ((m->in | m->inner | m->out) & 7) || m->experts <= 0 ||
         m->experts > MAX_EXPERTS || !m->offsets || ((uintptr_t)m->offsets & 3) || !m->w1 || !m->w2 || (((uintptr_t)m->w1 | (uintptr_t)m->w2) & 15);
}
bool bad_scratch(const bb_expert_mlp_desc* m, bool weight, bool bias, int n, int k) {
  return weight && (((uintptr_t)m->scratch & 15) || (!m->scratch && m->scratch_bytes != 0) ||
                    (bias && (!m->scratch || m->scratch_bytes < bb_grouped_bias_bytes(n, k, m->experts))));
}
// the weight's and the bias's gradient of one layer, each where it is asked for
int weight_and_bias(const bb_expert_mlp_desc* m, const void* dy, long long ld_dy, int n, const void* x, long long ld_x, int k, void* dw, float* g_w, void* db, float* g_b,
                    void* stream) {
  if (dw || g_w) {
    bb_grouped_desc d = part_of(m, BB_GROUPED_WEIGHT, n, k, g_w ? BB_EPI_ACCUM_F32 : BB_EPI_STORE);
    d.x = dy; d.ld_x = ld_dy; d.weight = x; d.ld_weight = ld_x; d.out = g_w ? (void*)g_w : dw;
    d.bias_accum = g_b; d.bias_grad = g_b ? nullptr : db; d.bias_parts = m->scratch; d.bias_parts_bytes = m->scratch_bytes;
    return bb_grouped_gemm(&d, stream);
  }
  if (db || g_b) return bb_grouped_colsum(dy, ld_dy, m->offsets, m->experts, g_b ? nullptr : db, g_b, m->rows, n, stream);
  return BB_OK;
}
}  // namespace

extern "C" int bb_expert_mlp_fwd(const bb_expert_mlp_desc* m, const void* x, long long ld_x, void* pre, void* act, void* y, void* stream) {
  if (bad_mlp(m) || bad_matrix(x, ld_x, m->in) || !m->b1 || !m->b2 || (((uintptr_t)m->b1 | (uintptr_t)m->b2) & 15) || !pre || !act || !y ||
      (((uintptr_t)pre | (uintptr_t)act | (uintptr_t)y) & 15))
    return refuse("bb_expert_mlp_fwd: null or misaligned pointer, a size that is not positive or no multiple of 8, rows that overlap, or more than 256 experts");
  BackToBack overlap(m->max_ctas == 0);
  bb_grouped_desc d = part_of(m, BB_GROUPED_ROWS, m->inner, m->in, BB_EPI_BIAS_GELU);
  d.x = x; d.ld_x = ld_x; d.weight = m->w1; d.bias = m->b1; d.out = act; d.ld_out = m->inner; d.out2 = pre;
  if (int rc = bb_grouped_gemm(&d, stream)) return rc;
  d = part_of(m, BB_GROUPED_ROWS, m->out, m->inner, BB_EPI_BIAS);
  d.x = act; d.ld_x = m->inner; d.weight = m->w2; d.bias = m->b2; d.out = y; d.ld_out = m->out;
  return bb_grouped_gemm(&d, stream);
}

extern "C" int bb_expert_mlp_bwd(const bb_expert_mlp_desc* m, const void* x, long long ld_x, const void* pre, const void* act, const void* dy, long long ld_dy, void* dpre,
                                 void* dx, void* stream) {
  if (bad_mlp(m) || bad_matrix(x, ld_x, m->in) || bad_matrix(dy, ld_dy, m->out) || !pre || !act || (((uintptr_t)pre | (uintptr_t)act | (uintptr_t)dpre | (uintptr_t)dx) & 15) ||
      (((uintptr_t)m->dw1 | (uintptr_t)m->dw2 | (uintptr_t)m->g_w1 | (uintptr_t)m->g_w2) & 15) ||
      (((uintptr_t)m->db1 | (uintptr_t)m->db2) & 1) || (((uintptr_t)m->g_b1 | (uintptr_t)m->g_b2) & 3))
    return refuse("bb_expert_mlp_bwd: null or misaligned pointer, a size that is not positive or no multiple of 8, rows that overlap, or more than 256 experts");
  const bool dw1 = m->dw1 || m->g_w1, db1 = m->db1 || m->g_b1, dw2 = m->dw2 || m->g_w2, db2 = m->db2 || m->g_b2;
  if (bad_scratch(m, dw1, db1, m->inner, m->in) || bad_scratch(m, dw2, db2, m->out, m->inner))
    return refuse("bb_expert_mlp_bwd: scratch that is null or not 16-byte aligned; a bias gradient that comes with a weight gradient takes bb_grouped_bias_bytes() of it");
  if ((db1 && !dw1 && too_wide(m->inner)) || (db2 && !dw2 && too_wide(m->out))) return refuse("bb_expert_mlp_bwd: more columns than a bias gradient alone covers");
  if (m->rows > (1 << 27) && (m->dw1 || m->g_w1 || m->dw2 || m->g_w2)) {
    bb_set_last_error_msg("bb_expert_mlp_bwd: a weight gradient over more than 2^27 rows");
    return BB_ERR_TOO_LARGE;
  }
  BackToBack overlap(m->max_ctas == 0);
  if (dpre) {
    bb_grouped_desc d = part_of(m, BB_GROUPED_INPUT, m->out, m->inner, BB_EPI_MUL_DGELU);
    d.x = dy; d.ld_x = ld_dy; d.weight = m->w2; d.out = dpre; d.ld_out = m->inner; d.aux = pre; d.ld_aux = m->inner;
    if (int rc = bb_grouped_gemm(&d, stream)) return rc;
  } else if (dx || m->dw1 || m->g_w1 || m->db1 || m->g_b1) {
    return refuse("bb_expert_mlp_bwd: gradients of the first layer go through dpre");
  }
  if (dx) {
    bb_grouped_desc d = part_of(m, BB_GROUPED_INPUT, m->inner, m->in, BB_EPI_STORE);
    d.x = dpre; d.ld_x = m->inner; d.weight = m->w1; d.out = dx; d.ld_out = m->in;
    if (int rc = bb_grouped_gemm(&d, stream)) return rc;
  }
  if (int rc = weight_and_bias(m, dpre, m->inner, m->inner, x, ld_x, m->in, m->dw1, m->g_w1, m->db1, m->g_b1, stream)) return rc;
  return weight_and_bias(m, dy, ld_dy, m->out, act, m->inner, m->inner, m->dw2, m->g_w2, m->db2, m->g_b2, stream);
}
