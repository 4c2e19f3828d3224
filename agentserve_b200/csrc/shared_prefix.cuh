// Shared-prefix decode attention: the plan's layout and the join of partial results.
//
// The softmax over a sequence's keys is split into parts: splits of the blocks its group
// shares (each computed once for all members) and splits of its own blocks.  A part of
// one (sequence, head) is (m, l, o): m = max of its scores, l = sum exp(s - m),
// o = sum exp(s - m) v.  Parts are joined by
//   M = max m_i,  out = sum exp(m_i - M) o_i / sum exp(m_i - M) l_i,
// all in fp32.  A part without keys is (-inf, 0, 0).
#pragma once

#include "common.cuh"

namespace asb {
namespace sp {

constexpr int kBS = 16;  // tokens per block
constexpr int kMagic = 0x53504c31;

// Plan: kHeader ints, then per batch row kRowInts, the members of all groups, the
// prefix items (kPrefixInts each) and the own items (kOwnInts each).
constexpr int kHeader = 32;
enum Header {
  kHMagic, kHSeqs, kHHeads, kHKvHeads, kHDim, kHDtype, kHPrefixItems, kHOwnItems, kHPrefixGrid,
  kHOwnGrid, kHOffRows, kHOffMembers, kHOffPrefix, kHOffOwn, kHPrefixParts, kHOwnParts,
  kHTileRows, kHInts, kHMostShared
};
constexpr int kRowInts = 8;
enum RowInfo {
  kRShared,       // shared blocks at the front of the row's table
  kRPrefixSplits, // parts those were split into
  kRPrefixPart,   // part index of the first of them (a part holds H heads)
  kRPrefixStep,   // part indexes from one split to the next
  kROwnSplits,
  kROwnPart
};
constexpr int kPrefixInts = 8;
enum PrefixItem { kPMembers, kPRow0, kPRows, kPBegin, kPEnd, kPPart };
constexpr int kOwnInts = 4;
enum OwnItem { kORow, kOSplit };

// Parts in the workspace: counters, then (m, l) and o of every (part, head); the prefix
// parts come first.
struct Parts {
  int32_t* counters;  // [B * H] arrivals of the own items, zero between calls
  float2* ml;         // [(prefix parts + own parts) * H]
  float* o;           // [(prefix parts + own parts) * H * D]
};

struct Args {
  const int32_t* plan;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* seq_lens;
  int64_t q_stride;
  int H, Kh, D, group;
  int num_blocks, max_blocks;
  float scale;
  int own_part0;  // index of the first own part
  int os_h, os_d; // output strides of a head and of a dimension
  int wait_first; // no prefix launch before this one: wait for the stream at the start
  Parts parts;
  int* status;
  uint64_t wait_limit;
};

// A row's own keys and what of its shared part counts.  A row shorter than its group's
// shared part takes nothing from it: all its keys are its own.
struct RowPlan {
  int shared, prefix_splits, prefix_part, prefix_step, own_splits, own_part;
  int len, blocks;
};
__device__ __forceinline__ RowPlan row_plan(const Args& a, int b, bool flag) {
  const int32_t* r = a.plan + a.plan[kHOffRows] + b * kRowInts;
  RowPlan p;
  p.shared = r[kRShared];
  p.prefix_splits = r[kRPrefixSplits];
  p.prefix_part = r[kRPrefixPart];
  p.prefix_step = r[kRPrefixStep];
  p.own_splits = r[kROwnSplits];
  p.own_part = a.own_part0 + r[kROwnPart];
  p.len = max(0, a.seq_lens[b]);
  p.blocks = (p.len + kBS - 1) / kBS;
  if (p.blocks > a.max_blocks) {
    if (flag) flag_status(a.status, kStatusBadLength);
    p.blocks = a.max_blocks;
    p.len = a.max_blocks * kBS;
  }
  if (p.len < p.shared * kBS) p.shared = p.prefix_splits = 0;
  return p;
}

// Exponentials of the parts' units: base 2 or e.
template <bool kBase2>
__device__ __forceinline__ float part_exp(float x) {
  return kBase2 ? fast_exp2(x) : expf(x);
}

// Ends an own item: rows [h0, h0 + nr) of sequence b, whose part of split s is in shared
// memory (o [nr][ld], m, l).  Joins it with the other parts of the row when it is the
// last to arrive, and writes the output.  All threads of the block call this.
template <typename T, bool kBase2>
__device__ void finish_own(const Args& a, const RowPlan& p, T* __restrict__ out, int b, int split,
                           int h0, int nr, const float* o, int ld, const float* m,
                           const float* l) {
  __shared__ int s_last;
  const int D = a.D, H = a.H;
  const bool alone = p.own_splits == 1;
  if (!alone) {
    for (int i = threadIdx.x; i < nr * D; i += blockDim.x) {
      const int r = i / D, d = i - r * D;
      const size_t at = size_t(p.own_part + split) * H + h0 + r;
      a.parts.o[at * D + d] = o[r * ld + d];
      if (d == 0) a.parts.ml[at] = make_float2(m[r], l[r]);
    }
    // the barrier orders this block's stores before thread 0's fence, which publishes
    // them before the arrival; the last arriver fences again before its reads
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      s_last = atomicAdd(a.parts.counters + b * H + h0, 1) == p.own_splits - 1;
      if (s_last) __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
  }
  if (p.prefix_splits > 0 && !a.wait_first) pdl_wait();  // the prefix parts are written
  for (int i = threadIdx.x; i < nr * D; i += blockDim.x) {
    const int r = i / D, d = i - r * D, h = h0 + r;
    float M = alone ? m[r] : -INFINITY;
    if (!alone)
      for (int s = 0; s < p.own_splits; ++s)
        M = fmaxf(M, __ldcg(&a.parts.ml[size_t(p.own_part + s) * H + h]).x);
    for (int s = 0; s < p.prefix_splits; ++s)
      M = fmaxf(M, __ldcg(&a.parts.ml[(size_t(p.prefix_part) + size_t(s) * p.prefix_step) * H + h]).x);
    float L = 0.f, O = 0.f;
    if (M != -INFINITY) {
      if (alone) {
        const float w = part_exp<kBase2>(m[r] - M);
        L = w * l[r];
        O = w * o[r * ld + d];
      } else {
        for (int s = 0; s < p.own_splits; ++s) {
          const size_t at = size_t(p.own_part + s) * H + h;
          const float2 ml = __ldcg(&a.parts.ml[at]);
          const float w = part_exp<kBase2>(ml.x - M);
          L += w * ml.y;
          O += w * __ldcg(&a.parts.o[at * D + d]);
        }
      }
      for (int s = 0; s < p.prefix_splits; ++s) {
        const size_t at = (size_t(p.prefix_part) + size_t(s) * p.prefix_step) * H + h;
        const float2 ml = __ldcg(&a.parts.ml[at]);
        const float w = part_exp<kBase2>(ml.x - M);
        L += w * ml.y;
        O += w * __ldcg(&a.parts.o[at * D + d]);
      }
    }
    out[size_t(b) * H * D + size_t(h) * a.os_h + size_t(d) * a.os_d] =
        Elem<T>::from_f32(L > 0.f ? O / L : 0.f);
  }
  if (!alone && threadIdx.x == 0) a.parts.counters[b * H + h0] = 0;  // for the next call
}

}  // namespace sp
}  // namespace asb
