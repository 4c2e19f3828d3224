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

// Plan: kHeader ints, then the members of all groups, the prefix items and the own
// items.  An item holds all that its block needs to start, so a block reaches its first
// K / V load after one plan read; an unused item is all zero.
constexpr int kHeader = 32;
enum Header {
  kHMagic, kHSeqs, kHHeads, kHKvHeads, kHDim, kHDtype, kHPrefixItems, kHOwnItems, kHPrefixGrid,
  kHOwnGrid, kHOffMembers, kHOffPrefix, kHOffOwn, kHPrefixParts, kHOwnParts, kHTileRows, kHInts,
  kHMostShared
};
constexpr int kItemInts = 8;
struct PrefixItem {
  int table_row;  // batch row whose table names the blocks (the group's first member)
  int members;    // its group's first entry in the members
  int row0, rows; // query rows (member, head of the KV head) of the group
  int begin, end; // blocks
  int part;       // part index of the group's first member (a part holds H heads)
  int unused;     // 0
};
struct OwnItem {
  int row, split;     // batch row, and which of its own_splits ranges
  int shared;         // shared blocks at the front of its table
  int prefix_splits;  // parts those were divided into,
  int prefix_part;    // the first one's index
  int prefix_step;    // and the distance to the next
  int own_splits;     // 0: unused item
  int own_part;
};

// Parts in the workspace: counters, then (m, l) and o of every (part, head); the prefix
// parts come first.
struct Parts {
  int32_t* counters;  // [B * H] arrivals of the own items, zero between calls
  float2* ml;         // [(prefix parts + own parts) * H]
  float* o;           // [(prefix parts + own parts) * H * D]
};

struct Args {
  const PrefixItem* prefix_items;
  const OwnItem* own_items;
  const int32_t* members;
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

template <typename Item>
__device__ __forceinline__ Item load_item(const Item* items, int i) {
  static_assert(sizeof(Item) == 4 * kItemInts, "item size");
  alignas(16) Item it;
  const int4* src = reinterpret_cast<const int4*>(items + i);
  reinterpret_cast<int4*>(&it)[0] = __ldg(src);
  reinterpret_cast<int4*>(&it)[1] = __ldg(src + 1);
  return it;
}

// A row's own keys and what of its shared part counts.  A row shorter than its group's
// shared part takes nothing from it: all its keys are its own.  So does every row of a group
// that shares more blocks than the table holds (a captured launch, whose plan was replaced):
// rows are cut to the table.
struct RowPlan {
  int shared, prefix_splits, prefix_part, prefix_step, own_splits, own_part;
  int len, begin, count;  // keys; this item's blocks
};
__device__ __forceinline__ RowPlan row_plan(const Args& a, const OwnItem& it, bool flag) {
  RowPlan p;
  p.shared = it.shared;
  p.prefix_splits = it.prefix_splits;
  p.prefix_part = it.prefix_part;
  p.prefix_step = it.prefix_step;
  p.own_splits = it.own_splits;
  p.own_part = a.own_part0 + it.own_part;
  p.len = max(0, a.seq_lens[it.row]);
  int blocks = p.len / kBS + (p.len % kBS != 0);  // any length: no sum past 31 bits
  if (blocks > a.max_blocks) {
    if (flag) flag_status(a.status, kStatusBadLength);
    blocks = a.max_blocks;
    p.len = a.max_blocks * kBS;
  }
  if (p.len < p.shared * kBS) p.shared = p.prefix_splits = 0;
  const int own = blocks - p.shared;
  const int per = (own + p.own_splits - 1) / p.own_splits;
  p.begin = p.shared + min(own, it.split * per);
  p.count = p.shared + min(own, (it.split + 1) * per) - p.begin;
  return p;
}

// Exponentials of the parts' units: base 2 or e.
template <bool kBase2>
__device__ __forceinline__ float part_exp(float x) {
  return kBase2 ? fast_exp2(x) : expf(x);
}

// Most parts a row has of either kind (the plan keeps to it), so that the weights of a
// join fit in shared memory.
constexpr int kMaxSplits = 64;

// Shared-memory floats a join works in.
constexpr int join_scratch(int rows, int threads) { return rows * 2 * kMaxSplits + 4 * threads; }

// Ends an own item: rows [h0, h0 + nr) of sequence b.  Its part of split `split` is in
// shared memory as kSub results over different keys (o [kSub][kRows][D], rows D apart
// by ld, m and l [kSub][kRows]).  Joins them with the other parts of the rows, when it is
// the last of the row's own items to arrive, and writes the output.  All threads of the
// block call this.  A warp per row turns the (m, l) into weights; then every thread sums
// its share of the parts for four dimensions of a row, eight loads in flight, as the
// parts come from L2.  scratch: join_scratch() floats of shared memory, 16-byte aligned,
// apart from o, m and l.
template <typename T, bool kBase2, int kRows, int kThreads, int kSub>
__device__ void finish_own(const Args& a, const RowPlan& p, T* __restrict__ out, int b, int split,
                           int h0, int nr, const float* o, int ld, const float* m, const float* l,
                           float* scratch) {
  __shared__ int s_last;
  auto s_w = reinterpret_cast<float(*)[2 * kMaxSplits]>(scratch + 4 * kThreads);
  float4* s_sum = reinterpret_cast<float4*>(scratch);
  const int D = a.D, H = a.H;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool alone = p.own_splits == 1;
  if (!alone) {
    // this item's part: its results relative to their common maximum
    for (int i = threadIdx.x; i < nr * D; i += kThreads) {
      const int r = i / D, d = i - r * D;
      float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < kSub; ++w) M = fmaxf(M, m[w * kRows + r]);
#pragma unroll
      for (int w = 0; w < kSub; ++w) {
        const float x = m[w * kRows + r];
        // no keys (l = o = 0), or NaN in all of them, which the sums keep
        const float e = x == -INFINITY ? 0.f : part_exp<kBase2>(x - M);
        L += e * l[w * kRows + r];
        O += e * o[(w * kRows + r) * ld + d];
      }
      const size_t at = size_t(p.own_part + split) * H + h0 + r;
      a.parts.o[at * D + d] = O;
      if (d == 0) a.parts.ml[at] = make_float2(M, L);
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
    if (threadIdx.x == 0) a.parts.counters[b * H + h0] = 0;  // for the next call
  }
  if (p.prefix_splits > 0 && !a.wait_first) pdl_wait();  // the prefix parts are written
  // parts in global memory, then (alone) this item's results in shared memory
  const int ng = p.prefix_splits + (alone ? 0 : p.own_splits);
  const int np = ng + (alone ? kSub : 0);
  const auto part = [&](int s) -> size_t {
    return s < p.prefix_splits ? size_t(p.prefix_part) + size_t(s) * p.prefix_step
                               : size_t(p.own_part + s - p.prefix_splits);
  };
  for (int r = warp; r < nr; r += kThreads / 32) {
    float2 ml[2 * kMaxSplits / 32];
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2 * kMaxSplits / 32; ++i) {
      const int s = lane + 32 * i;
      ml[i] = make_float2(-INFINITY, 0.f);
      if (s < ng)
        ml[i] = __ldcg(&a.parts.ml[part(s) * H + h0 + r]);
      else if (s < np)
        ml[i] = make_float2(m[(s - ng) * kRows + r], l[(s - ng) * kRows + r]);
      M = fmaxf(M, ml[i].x);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float L = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * kMaxSplits / 32; ++i) {
      ml[i].x = ml[i].x == -INFINITY ? 0.f : part_exp<kBase2>(ml[i].x - M);
      L += ml[i].x * ml[i].y;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int i = 0; i < 2 * kMaxSplits / 32; ++i)
      if (lane + 32 * i < np) s_w[r][lane + 32 * i] = ml[i].x * inv;
  }
  __syncthreads();
  if ((D & 3) == 0) {
    const int dv = D >> 2, nv = nr * dv;
    const bool packed =
        a.os_d == 1 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0;
    for (int v0 = 0; v0 < nv; v0 += kThreads) {
      // as many threads as there are vectors share out the parts
      const int here = min(nv - v0, kThreads), ways = kThreads / here;
      const int way = threadIdx.x / here;
      const int v = v0 + threadIdx.x - way * here;
      const int r = v / dv, d = (v - r * dv) * 4;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      const auto add = [&](float w, const float4& x) {
        acc.x += w * x.x;
        acc.y += w * x.y;
        acc.z += w * x.z;
        acc.w += w * x.w;
      };
      if (way < ways) {
        const float* base = a.parts.o + size_t(h0 + r) * D + d;
        for (int s0 = way; s0 < ng; s0 += 8 * ways) {
          float4 x[8];
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int s = s0 + e * ways;
            w[e] = s < ng ? s_w[r][s] : 0.f;
            x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (w[e] != 0.f)  // a part without keys holds no values
              x[e] = __ldcg(reinterpret_cast<const float4*>(base + part(s) * H * D));
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) add(w[e], x[e]);
        }
        for (int s = ng + way; s < np; s += ways) {
          const float w = s_w[r][s];
          if (w == 0.f) continue;
          add(w, *reinterpret_cast<const float4*>(o + ((s - ng) * kRows + r) * ld + d));
        }
      }
      if (ways > 1) {
        s_sum[threadIdx.x] = acc;
        __syncthreads();
        if (way == 0)
          for (int y = 1; y < ways; ++y) add(1.f, s_sum[threadIdx.x + y * here]);
      }
      if (way == 0) {
        T* dst = out + size_t(b) * H * D + size_t(h0 + r) * a.os_h + size_t(d) * a.os_d;
        T val[4] = {Elem<T>::from_f32(acc.x), Elem<T>::from_f32(acc.y), Elem<T>::from_f32(acc.z),
                    Elem<T>::from_f32(acc.w)};
        if (packed) {
          struct alignas(4 * sizeof(T)) Four {
            T v[4];
          };
          *reinterpret_cast<Four*>(dst) = Four{val[0], val[1], val[2], val[3]};
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[size_t(e) * a.os_d] = val[e];
        }
      }
      if (v0 + kThreads < nv) __syncthreads();
    }
    return;
  }
  for (int i = threadIdx.x; i < nr * D; i += kThreads) {
    const int r = i / D, d = i - r * D;
    float acc = 0.f;
    for (int s = 0; s < np; ++s) {
      const float w = s_w[r][s];
      if (w == 0.f) continue;
      acc += w * (s < ng ? __ldcg(&a.parts.o[(part(s) * H + h0 + r) * D + d])
                         : o[((s - ng) * kRows + r) * ld + d]);
    }
    out[size_t(b) * H * D + size_t(h0 + r) * a.os_h + size_t(d) * a.os_d] =
        Elem<T>::from_f32(acc);
  }
}

// Tensor-core launches (shared_prefix_tc.cu): 16-bit types, head_dim 64 or 128.
constexpr int kTcTileRows = 256;
inline bool tc_geometry(int D, int dtype) {
  return (dtype == AS_DTYPE_BF16 || dtype == AS_DTYPE_F16) && (D == 64 || D == 128);
}
int tc_launch(int prefix_grid, int own_grid, void* out, const void* q, const void* k_cache,
              const void* v_cache, const Args& a, int dtype, cudaStream_t stream);

}  // namespace sp
}  // namespace asb
