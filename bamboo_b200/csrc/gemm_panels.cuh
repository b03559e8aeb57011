// Epilogue helpers that the tensor-core products share: panels of an output tile between registers (one row per lane), a warp's
// staging slab in shared memory and coalesced global accesses, and the GeLU arithmetic between.
#pragma once
#include "common.cuh"
#include "bamboo_b200.h"

namespace {

__device__ __forceinline__ void unpack8(const uint4& q, float* f) {
  f[0] = bb::bf16_lo(q.x); f[1] = bb::bf16_hi(q.x); f[2] = bb::bf16_lo(q.y); f[3] = bb::bf16_hi(q.y);
  f[4] = bb::bf16_lo(q.z); f[5] = bb::bf16_hi(q.z); f[6] = bb::bf16_lo(q.w); f[7] = bb::bf16_hi(q.w);
}

// One output row's slice of a panel (128 bytes = 8 chunks of 16 bytes) into swizzled shared memory.
__device__ __forceinline__ void panel_store_row_bf16(uint8_t* panel, int row, const float* v /*64*/) {
  uint8_t* base = panel + row * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint4 q;
    q.x = bb::pack_bf16x2(v[8 * c + 0], v[8 * c + 1]); q.y = bb::pack_bf16x2(v[8 * c + 2], v[8 * c + 3]);
    q.z = bb::pack_bf16x2(v[8 * c + 4], v[8 * c + 5]); q.w = bb::pack_bf16x2(v[8 * c + 6], v[8 * c + 7]);
    *reinterpret_cast<uint4*>(base + ((c ^ (row & 7)) << 4)) = q;
  }
}
__device__ __forceinline__ void panel_store_row_f32(uint8_t* panel, int row, const float* v /*32*/) {
  uint8_t* base = panel + row * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4*>(base + ((c ^ (row & 7)) << 4)) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}

// ---- warp-private staging slab: 32 rows x 128 bytes, 16-byte chunks XOR-swizzled by the row.
// Row side: lane == row (panel_store_row_* / panel_load_row_bf16 with row = lane).
// Coalesced side: lane -> (row 4*i + lane/8, chunk lane%8), i = 0..7: one instruction moves four
// complete 128-byte row segments.
__device__ __forceinline__ uint32_t slab_off(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// Whether the 32 rows from r0 and `width` columns from nb all lie inside the matrix (the same for a whole warp): then the
// addresses are one base and a constant step and the accesses go out back to back.  With a test per row and chunk the
// eight stores of a panel took 950 cycles, the longest part of its epilogue.
__device__ __forceinline__ bool inside(int r0, int nb, int width, int M, int N) { return r0 + 32 <= M && nb + width <= N; }

__device__ __forceinline__ void slab_put(uint8_t* slab, int lane, const uint4* ax) {
#pragma unroll
  for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(slab + slab_off(4 * i + (lane >> 3), lane & 7)) = ax[i];
}
// rows r0.., columns nb.. of a bf16 matrix -> ax (zero outside the matrix)
__device__ __forceinline__ void slab_fetch_bf16(const __nv_bfloat16* src, long long ld, int r0, int nb, int M, int N, int lane, uint4* ax) {
  const int c = nb + (lane & 7) * 8;
  if (inside(r0, nb, 64, M, N)) {
    const __nv_bfloat16* g = src + (long long)(r0 + (lane >> 3)) * ld + c;
#pragma unroll
    for (int i = 0; i < 8; ++i, g += 4 * ld) ax[i] = __ldca(reinterpret_cast<const uint4*>(g));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 4 * i + (lane >> 3);
    uint4 q = make_uint4(0, 0, 0, 0);
    if (r < M) {
      const __nv_bfloat16* g = src + (long long)r * ld + c;
      if (c + 8 <= N) {
        q = __ldca(reinterpret_cast<const uint4*>(g));
      } else {
        unsigned short e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = (c + k < N) ? __bfloat16_as_ushort(g[k]) : (unsigned short)0;
        q.x = e[0] | ((uint32_t)e[1] << 16); q.y = e[2] | ((uint32_t)e[3] << 16);
        q.z = e[4] | ((uint32_t)e[5] << 16); q.w = e[6] | ((uint32_t)e[7] << 16);
      }
    }
    ax[i] = q;
  }
}
__device__ __forceinline__ void slab_flush_bf16(const uint8_t* slab, __nv_bfloat16* dst, long long ld, int r0, int nb, int M, int N, int lane) {
  const int c = nb + (lane & 7) * 8;
  if (inside(r0, nb, 64, M, N)) {
    __nv_bfloat16* g = dst + (long long)(r0 + (lane >> 3)) * ld + c;
    uint4 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = *reinterpret_cast<const uint4*>(slab + slab_off(4 * i + (lane >> 3), lane & 7));
#pragma unroll
    for (int i = 0; i < 8; ++i, g += 4 * ld) *reinterpret_cast<uint4*>(g) = q[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rl = 4 * i + (lane >> 3);
    const int r = r0 + rl;
    const uint4 q = *reinterpret_cast<const uint4*>(slab + slab_off(rl, lane & 7));
    if (r < M) {
      __nv_bfloat16* g = dst + (long long)r * ld + c;
      if (c + 8 <= N) {
        *reinterpret_cast<uint4*>(g) = q;
      } else {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) if (c + k < N) g[k] = __ushort_as_bfloat16((unsigned short)(w[k >> 1] >> (16 * (k & 1))));
      }
    }
  }
}
// Add-reductions go out back to back only into outputs of less than 16 MiB.  A large output is read and written in memory, and bursts
// of reductions slow that down: 4096 x 16384 x 333 141 us in bursts and 135 row by row, 8192 x 2048 x 333 35.3 and 33.5, 2048 x 2048 x 513
// 13.2 and 12.5 (outputs not in L2; from 2000 k on no difference); a small one of many splits stays in L2: 64 x 576 x 100352
// 25.7 and 26.9.
__device__ __forceinline__ bool small_output(int M, int N) { return (long long)M * N < (1LL << 22); }
template <bool ACCUM>
__device__ __forceinline__ void slab_flush_f32(const uint8_t* slab, float* dst, long long ld, int r0, int nb, int M, int N, int lane) {
  const int c = nb + (lane & 7) * 4;
  if ((!ACCUM || small_output(M, N)) && inside(r0, nb, 32, M, N)) {
    float* g = dst + (long long)(r0 + (lane >> 3)) * ld + c;
    float4 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = *reinterpret_cast<const float4*>(slab + slab_off(4 * i + (lane >> 3), lane & 7));
#pragma unroll
    for (int i = 0; i < 8; ++i, g += 4 * ld) {
      if (ACCUM) asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(g), "f"(q[i].x), "f"(q[i].y), "f"(q[i].z), "f"(q[i].w) : "memory");
      else *reinterpret_cast<float4*>(g) = q[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rl = 4 * i + (lane >> 3);
    const int r = r0 + rl;
    const float4 q = *reinterpret_cast<const float4*>(slab + slab_off(rl, lane & 7));
    if (r < M) {
      float* g = dst + (long long)r * ld + c;
      if (c + 4 <= N) {
        if (ACCUM) asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(g), "f"(q.x), "f"(q.y), "f"(q.z), "f"(q.w) : "memory");
        else *reinterpret_cast<float4*>(g) = q;
      } else {
        const float w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c + k < N) { if (ACCUM) atomicAdd(g + k, w[k]); else g[k] = w[k]; }
        }
      }
    }
  }
}

// ---- narrow variant (four epilogue warps per lane quarter): 32 rows x 64 bytes = 32 bf16
// columns per pass, 2 KiB per warp.  Chunk c of row r sits at c ^ ((r >> 1) & 3): eight
// consecutive rows cover all 32 banks once, on the row side (lane == row) and on the coalesced
// side (lane -> row 8*i + lane/4, chunk lane%4, i = 0..3).
__device__ __forceinline__ uint32_t slab64_off(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }

__device__ __forceinline__ void slab64_store_row(uint8_t* slab, int row, const float* v /*32*/) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint4 q;
    q.x = bb::pack_bf16x2(v[8 * c + 0], v[8 * c + 1]); q.y = bb::pack_bf16x2(v[8 * c + 2], v[8 * c + 3]);
    q.z = bb::pack_bf16x2(v[8 * c + 4], v[8 * c + 5]); q.w = bb::pack_bf16x2(v[8 * c + 6], v[8 * c + 7]);
    *reinterpret_cast<uint4*>(slab + slab64_off(row, c)) = q;
  }
}
// rows r0.., columns nb..nb+31 of a bf16 matrix -> slab (zero outside the matrix), coalesced
__device__ __forceinline__ void slab64_fetch(uint8_t* slab, const __nv_bfloat16* src, long long ld, int r0, int nb, int M, int N, int lane) {
  const int c = nb + (lane & 3) * 8;
  uint4 q[4];
  if (inside(r0, nb, 32, M, N)) {
    const __nv_bfloat16* g = src + (long long)(r0 + (lane >> 2)) * ld + c;
#pragma unroll
    for (int i = 0; i < 4; ++i, g += 8 * ld) q[i] = __ldca(reinterpret_cast<const uint4*>(g));
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(slab + slab64_off(8 * i + (lane >> 2), lane & 3)) = q[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 8 * i + (lane >> 2);
    q[i] = make_uint4(0, 0, 0, 0);
    if (r < M) {
      const __nv_bfloat16* g = src + (long long)r * ld + c;
      if (c + 8 <= N) {
        q[i] = __ldca(reinterpret_cast<const uint4*>(g));
      } else {
        unsigned short e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = (c + k < N) ? __bfloat16_as_ushort(g[k]) : (unsigned short)0;
        q[i].x = e[0] | ((uint32_t)e[1] << 16); q[i].y = e[2] | ((uint32_t)e[3] << 16);
        q[i].z = e[4] | ((uint32_t)e[5] << 16); q[i].w = e[6] | ((uint32_t)e[7] << 16);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(slab + slab64_off(8 * i + (lane >> 2), lane & 3)) = q[i];
}
__device__ __forceinline__ void slab64_flush(const uint8_t* slab, __nv_bfloat16* dst, long long ld, int r0, int nb, int M, int N, int lane) {
  const int c = nb + (lane & 3) * 8;
  if (inside(r0, nb, 32, M, N)) {
    __nv_bfloat16* g = dst + (long long)(r0 + (lane >> 2)) * ld + c;
    uint4 q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const uint4*>(slab + slab64_off(8 * i + (lane >> 2), lane & 3));
#pragma unroll
    for (int i = 0; i < 4; ++i, g += 8 * ld) *reinterpret_cast<uint4*>(g) = q[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rl = 8 * i + (lane >> 2);
    const int r = r0 + rl;
    const uint4 q = *reinterpret_cast<const uint4*>(slab + slab64_off(rl, lane & 3));
    if (r < M) {
      __nv_bfloat16* g = dst + (long long)r * ld + c;
      if (c + 8 <= N) {
        *reinterpret_cast<uint4*>(g) = q;
      } else {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) if (c + k < N) g[k] = __ushort_as_bfloat16((unsigned short)(w[k >> 1] >> (16 * (k & 1))));
      }
    }
  }
}

__device__ __forceinline__ float2 get2(const float* v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ void set2(float* v, float2 a) { v[0] = a.x; v[1] = a.y; }
// GeLU of the bf16-rounded pre-activation: forward and backward (which re-reads the stored pre-activation) see the same argument
template <int W> __device__ __forceinline__ void gelu_rounded(float* v) {
#pragma unroll
  for (int i = 0; i < W; i += 2) {
    const uint32_t q = bb::pack_bf16x2(v[i], v[i + 1]);
    set2(v + i, bb::gelu_tanh2(make_float2(bb::bf16_lo(q), bb::bf16_hi(q))));
  }
}
// v *= gelu'(x) or v += x
template <int W> __device__ __forceinline__ void apply_aux(int epi, float* v, const float* x) {
  if (epi == BB_EPI_MUL_DGELU) {
#pragma unroll
    for (int i = 0; i < W; i += 2) set2(v + i, bb::mul2(get2(v + i), bb::gelu_tanh_grad2(get2(x + i))));
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 2) set2(v + i, bb::add2(get2(v + i), get2(x + i)));
  }
}

}  // namespace
