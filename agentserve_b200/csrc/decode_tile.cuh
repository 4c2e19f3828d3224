// Warp-level building blocks of the decode attention kernels: one warp folds paged
// 16-token blocks of one KV head, staged in 128B-swizzled shared memory, into the
// online softmax of up to 8 query heads.
#pragma once

#include "common.cuh"
#include "host_util.h"

namespace asb {

constexpr int kTileTokens = 16;  // tokens of a paged block

// Fold n <= G paged blocks of one sequence at once (G independent S^T accumulator
// chains for instruction-level parallelism).  Block k's K/V tiles are at kb[k]/vb[k]
// and its first token at tok0 + k*tok_step.  The running max is lazy: scores are
// exponentiated against the current max m_run unless some score exceeds it by more
// than 2^8 (one warp vote); only then is the max reduced across the 8 lanes that
// share a head column and O, l rescaled.  p stays <= 256, well inside bf16/fp32
// range, and l, O, m stay mutually consistent, so the result is unchanged.  p is rounded to
// the pool's type for the product with V, as the matrix instruction takes it; l sums it
// unrounded.
constexpr float kLazyMaxSlack = 8.0f;  // log2 units

template <typename T, int D, int G>
__device__ __forceinline__ void fold_blocks(const uint32_t (&kb)[G], const uint32_t (&vb)[G], int n,
                                            const uint32_t (&qb)[D / 16][2], int tok0,
                                            int tok_step, int seq_len, float scale_log2,
                                            float (&m_run)[2], float (&l_run)[2],
                                            float (&o_acc)[D / 16][4], int lane,
                                            uint32_t sub_bytes) {
  constexpr int KT = D / 16;
  float sc[G][4];
#pragma unroll
  for (int k = 0; k < G; ++k) sc[k][0] = sc[k][1] = sc[k][2] = sc[k][3] = 0.f;
#pragma unroll
  for (int kk = 0; kk < KT; ++kk) {
    const int mi = lane >> 3;
    const int row = (lane & 7) + 8 * (mi & 1);
    const int chunk = 2 * (kk & 3) + (mi >> 1);
    const uint32_t off = (kk >> 2) * sub_bytes + row * 128 + ((chunk ^ (row & 7)) << 4);
#pragma unroll
    for (int k = 0; k < G; ++k) {
      if (k < n) {
        uint32_t a0, a1, a2, a3;
        ldmatrix_x4(kb[k] + off, a0, a1, a2, a3);
        mma_16816<T>(sc[k], a0, a1, a2, a3, qb[kk][0], qb[kk][1]);
      }
    }
  }
  const int gq = lane >> 2;
  float lm0 = -INFINITY, lm1 = -INFINITY;
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const int t = tok0 + k * tok_step + gq;
    const bool v0 = k < n && t < seq_len;
    const bool v1 = k < n && t + 8 < seq_len;
    sc[k][0] = v0 ? sc[k][0] * scale_log2 : -INFINITY;
    sc[k][1] = v0 ? sc[k][1] * scale_log2 : -INFINITY;
    sc[k][2] = v1 ? sc[k][2] * scale_log2 : -INFINITY;
    sc[k][3] = v1 ? sc[k][3] * scale_log2 : -INFINITY;
    lm0 = fmaxf(lm0, fmaxf(sc[k][0], sc[k][2]));
    lm1 = fmaxf(lm1, fmaxf(sc[k][1], sc[k][3]));
  }
  const bool grow = lm0 > m_run[0] + kLazyMaxSlack || lm1 > m_run[1] + kLazyMaxSlack;
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      lm0 = fmaxf(lm0, __shfl_xor_sync(0xffffffffu, lm0, o));
      lm1 = fmaxf(lm1, __shfl_xor_sync(0xffffffffu, lm1, o));
    }
    const float mn0 = fmaxf(m_run[0], lm0), mn1 = fmaxf(m_run[1], lm1);
    const float al0 = fast_exp2(m_run[0] - mn0), al1 = fast_exp2(m_run[1] - mn1);
    m_run[0] = mn0;
    m_run[1] = mn1;
    l_run[0] *= al0;
    l_run[1] *= al1;
#pragma unroll
    for (int mt = 0; mt < KT; ++mt) {
      o_acc[mt][0] *= al0;
      o_acc[mt][1] *= al1;
      o_acc[mt][2] *= al0;
      o_acc[mt][3] *= al1;
    }
  }
#pragma unroll
  for (int k = 0; k < G; ++k) {
    if (k < n) {
      const float p0 = fast_exp2(sc[k][0] - m_run[0]), p1 = fast_exp2(sc[k][1] - m_run[1]);
      const float p2 = fast_exp2(sc[k][2] - m_run[0]), p3 = fast_exp2(sc[k][3] - m_run[1]);
      l_run[0] += p0 + p2;
      l_run[1] += p1 + p3;
      const uint32_t pb0 = movmatrix_trans(pack2<T>(p0, p1));
      const uint32_t pb1 = movmatrix_trans(pack2<T>(p2, p3));
#pragma unroll
      for (int mt = 0; mt < KT; ++mt) {
        const int mi = lane >> 3;
        const int row = (lane & 7) + 8 * (mi >> 1);
        const int chunk = 2 * (mt & 3) + (mi & 1);
        uint32_t a0, a1, a2, a3;
        ldmatrix_x4_trans(vb[k] + (mt >> 2) * sub_bytes + row * 128 + ((chunk ^ (row & 7)) << 4),
                          a0, a1, a2, a3);
        mma_16816<T>(o_acc[mt], a0, a1, a2, a3, pb0, pb1);
      }
    }
  }
}

// Q^T of the GQA group of KV head g as B-fragments of S^T = K Q^T: column n = query
// head g*group + n (zero columns past the group).
template <typename T, int D>
__device__ __forceinline__ void load_q_frags(uint32_t (&qb)[D / 16][2], const T* __restrict__ q,
                                             int64_t q_stride, int b, int g, int group, int lane) {
  const int gq = lane >> 2, tq = lane & 3;
  const bool has_head = gq < group;
  const T* qrow = q + int64_t(b) * q_stride + int64_t(g * group + (has_head ? gq : 0)) * D;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    qb[kk][0] = has_head ? *reinterpret_cast<const uint32_t*>(qrow + 16 * kk + 2 * tq) : 0u;
    qb[kk][1] = has_head ? *reinterpret_cast<const uint32_t*>(qrow + 16 * kk + 2 * tq + 8) : 0u;
  }
}

template <typename T>
CUtensorMapDataType tma_dtype();
template <>
inline CUtensorMapDataType tma_dtype<__nv_bfloat16>() { return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }
template <>
inline CUtensorMapDataType tma_dtype<__half>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }

// 4-D map over one layer's K or V plane [NB, 16, Kh, D] viewed innermost-first as
// (D, Kh, 16, NB); box = 64 elements (128 B, swizzled) x 1 head x 16 tokens x 1 block.
template <typename T>
inline int make_pool_map(CUtensorMap* map, const void* base, int Kh, int D, int num_blocks) {
  const uint64_t es = sizeof(T);
  const uint64_t dims[4] = {uint64_t(D), uint64_t(Kh), uint64_t(kTileTokens), uint64_t(num_blocks)};
  const uint64_t strides[3] = {D * es, uint64_t(Kh) * D * es, uint64_t(kTileTokens) * Kh * D * es};
  const uint32_t box[4] = {64, 1, uint32_t(kTileTokens), 1};
  return encode_tensor_map(map, tma_dtype<T>(), 4, const_cast<void*>(base), dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace asb
