// (9) Decode attention for a batch whose sequences share leading blocks.
//
// The engine's prefix cache lets requests hold the same pool blocks
// (DeviceBlockAllocator.share_blocks); the reference copies the prefix per request and
// attends over every copy (agentserve/engine/engine.py:274-281, agentserve/model/
// llama.py:419-469).  Here a group's shared blocks are read and multiplied once: its
// members' query heads of one KV head are the rows of one matrix product with the
// shared keys.  Two launches: the prefix launch writes partial results per (split,
// member, head); the own launch attends over every sequence's remaining blocks and
// joins the parts (shared_prefix.cuh).  It is launched programmatically: its blocks
// start while the prefix launch runs and wait for it only before they join.
//
// A host-side plan divides both kinds of work over the GPU.  It holds for as long as the
// same sequences share the same blocks: lengths are read on the device at every call.
#include <algorithm>
#include <vector>

#include "common.cuh"
#include "host_util.h"
#include "shared_prefix.cuh"

namespace asb {
namespace sp {
namespace {

inline size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

// ===========================================================================
// CUDA-core kernels: any type, head_dim <= 256, any group.
// A block holds a tile of query rows and walks 32 * TG tokens at a time, K and V staged
// in shared memory as fp32.  Scores: one token per lane, so a dot product needs no
// shuffles and a K row read feeds RW query rows; products with V: one dimension per
// lane.  TG > 1 gives token groups to different warps when there are few rows.
// ===========================================================================
constexpr int kThreads = 256;
constexpr int kNWarps = kThreads / 32;

template <int DP, int RW, int TG>
struct GenCfg {
  static constexpr int kRowWarps = kNWarps / TG;
  static constexpr int kRows = kRowWarps * RW;
  static constexpr int kTokens = 32 * TG;
  static constexpr int kLdK = DP + 4;  // float4 reads of 8 lanes hit 32 different banks
  static constexpr int kFloats = kRows * DP + kTokens * kLdK + kTokens * DP + kNWarps * RW * 32;
  static constexpr int kJoin = TG * kRows * (DP + 2);  // reuses the K / V space
  static constexpr int kMerge = kJoin + join_scratch(kRows, kThreads);
  static constexpr int kSmemBytes = 4 * (kFloats > kMerge ? kFloats : kMerge);
};

template <typename T, int DP, int RW, int TG, bool kPrefix>
__global__ void __launch_bounds__(kThreads)
sp_generic_kernel(T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ k_cache,
                  const T* __restrict__ v_cache, const Args a) {
  using Cfg = GenCfg<DP, RW, TG>;
  constexpr int EPL = DP / 32;
  if (kPrefix || a.wait_first) {
    pdl_wait();
    pdl_trigger();
  }
  const int32_t* plan = a.plan;
  if (int(blockIdx.x) >= plan[kPrefix ? kHPrefixItems : kHOwnItems]) {
    if (!kPrefix) pdl_wait();
    return;
  }
  const int g = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.D, group = a.group;

  // this item's query rows and token range
  int b = 0, split = 0, row0 = 0, rows = 0, begin, end, part = 0, table_row;
  const int32_t* members = nullptr;
  RowPlan rp{};
  if (kPrefix) {
    const int32_t* it = plan + plan[kHOffPrefix] + blockIdx.x * kPrefixInts;
    members = plan + plan[kHOffMembers] + it[kPMembers];
    row0 = it[kPRow0] + blockIdx.z * Cfg::kRows;  // the plan's tiles may be larger
    rows = min(Cfg::kRows, it[kPRows] - int(blockIdx.z) * Cfg::kRows);
    if (rows <= 0) return;
    begin = it[kPBegin] * kBS;
    end = it[kPEnd] * kBS;
    part = it[kPPart];
    table_row = members[0];
  } else {
    const int32_t* it = plan + plan[kHOffOwn] + blockIdx.x * kOwnInts;
    b = it[kORow];
    split = it[kOSplit];
    row0 = blockIdx.z * Cfg::kRows;
    rows = min(Cfg::kRows, group - row0);
    rp = row_plan(a, b, threadIdx.x == 0 && split == 0 && g == 0 && row0 == 0);
    const int own = rp.blocks - rp.shared;
    const int per = (own + rp.own_splits - 1) / rp.own_splits;
    begin = (rp.shared + min(own, split * per)) * kBS;
    end = min(rp.len, (rp.shared + min(own, (split + 1) * per)) * kBS);
    table_row = b;
  }

  extern __shared__ __align__(16) float smem[];
  float* sq = smem;                                // [rows][DP]
  float* sk = sq + Cfg::kRows * DP;                // [tokens][kLdK]
  float* sv = sk + Cfg::kTokens * Cfg::kLdK;       // [tokens][DP]
  float* spr = sv + Cfg::kTokens * DP;             // [warps][RW][32] probabilities
  __shared__ int s_ok[Cfg::kTokens];
  for (int i = threadIdx.x; i < Cfg::kRows * DP; i += kThreads) {
    const int r = i / DP, d = i - r * DP;
    float x = 0.f;
    if (r < rows && d < D) {
      const int rr = row0 + r;
      const int seq = kPrefix ? members[rr / group] : b;
      const int h = g * group + (kPrefix ? rr % group : rr);
      x = Elem<T>::to_f32(q[int64_t(seq) * a.q_stride + int64_t(h) * D + d]);
    }
    sq[i] = x;
  }

  const int wr = warp % Cfg::kRowWarps, tg = warp / Cfg::kRowWarps;
  float m[RW], l[RW], o[RW][EPL];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[r][e] = 0.f;
  }
  for (int t0 = begin; t0 < end; t0 += Cfg::kTokens) {
    __syncthreads();
    if (threadIdx.x < Cfg::kTokens) {
      const int t = t0 + threadIdx.x;
      int id = -1;
      if (t < end) {
        id = a.bt[int64_t(table_row) * a.bt_stride + t / kBS];
        if (id < 0 || id >= a.num_blocks) {
          flag_status(a.status, kStatusBadBlockId);
          id = -1;
        }
      }
      s_ok[threadIdx.x] = id;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < Cfg::kTokens * DP; i += kThreads) {
      const int t = i / DP, d = i - t * DP;
      float kx = 0.f, vx = 0.f;
      if (s_ok[t] >= 0 && d < D) {
        const int64_t at =
            ((int64_t(s_ok[t]) * kBS + (t0 + t) % kBS) * a.Kh + g) * int64_t(D) + d;
        kx = Elem<T>::to_f32(k_cache[at]);
        vx = Elem<T>::to_f32(v_cache[at]);
      }
      sk[t * Cfg::kLdK + d] = kx;
      sv[i] = vx;
    }
    __syncthreads();
    const int tok = tg * 32 + lane;
    const bool ok = s_ok[tok] >= 0;
    float s[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) s[r] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      const float4 kv = *reinterpret_cast<const float4*>(sk + tok * Cfg::kLdK + d);
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        const float4 qv = *reinterpret_cast<const float4*>(sq + (wr * RW + r) * DP + d);
        s[r] += qv.x * kv.x;
        s[r] += qv.y * kv.y;
        s[r] += qv.z * kv.z;
        s[r] += qv.w * kv.w;
      }
    }
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const float x = ok ? s[r] * a.scale : -INFINITY;
      float mx = x;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float mn = fmaxf(m[r], mx);
      const float alpha = m[r] == -INFINITY ? 0.f : expf(m[r] - mn);
      const float p = x != -INFINITY ? expf(x - mn) : 0.f;  // also while mn is still -inf
      m[r] = mn;
      l[r] = l[r] * alpha + p;  // one lane's share; summed after the loop
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[r][e] *= alpha;
      spr[(warp * RW + r) * 32 + lane] = p;
    }
    __syncwarp();
#pragma unroll 2
    for (int t = 0; t < 32; t += 4) {
      float4 p[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r)
        p[r] = *reinterpret_cast<const float4*>(spr + (warp * RW + r) * 32 + t);
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float* vr = sv + (tg * 32 + t) * DP + lane + 32 * e;
        const float v0 = vr[0], v1 = vr[DP], v2 = vr[2 * DP], v3 = vr[3 * DP];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          o[r][e] += p[r].x * v0;
          o[r][e] += p[r].y * v1;
          o[r][e] += p[r].z * v2;
          o[r][e] += p[r].w * v3;
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RW; ++r)
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);

  // token groups joined in shared memory
  __syncthreads();
  float* ro = smem;                                  // [TG][rows][DP]
  float* rm = ro + TG * Cfg::kRows * DP;             // [TG][rows]
  float* rl = rm + TG * Cfg::kRows;
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const int at = tg * Cfg::kRows + wr * RW + r;
#pragma unroll
    for (int e = 0; e < EPL; ++e) ro[at * DP + lane + 32 * e] = o[r][e];
    if (lane == 0) {
      rm[at] = m[r];
      rl[at] = l[r];
    }
  }
  __syncthreads();
  if (TG > 1) {
    for (int r = warp; r < Cfg::kRows; r += kNWarps) {
      float M = -INFINITY, L = 0.f;
      for (int t = 0; t < TG; ++t) M = fmaxf(M, rm[t * Cfg::kRows + r]);
      float acc[EPL];
#pragma unroll
      for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
      if (M != -INFINITY) {
        for (int t = 0; t < TG; ++t) {
          const int at = t * Cfg::kRows + r;
          const float w = expf(rm[at] - M);
          L += w * rl[at];
#pragma unroll
          for (int e = 0; e < EPL; ++e) acc[e] += w * ro[at * DP + lane + 32 * e];
        }
      }
      __syncwarp();
#pragma unroll
      for (int e = 0; e < EPL; ++e) ro[r * DP + lane + 32 * e] = acc[e];
      if (lane == 0) {
        rm[r] = M;
        rl[r] = L;
      }
    }
    __syncthreads();
  }
  if (kPrefix) {
    for (int i = threadIdx.x; i < rows * D; i += kThreads) {
      const int r = i / D, d = i - r * D, rr = row0 + r;
      const size_t at = size_t(part + rr / group) * a.H + g * group + rr % group;
      a.parts.o[at * D + d] = ro[r * DP + d];
      if (d == 0) a.parts.ml[at] = make_float2(rm[r], rl[r]);
    }
    return;
  }
  finish_own<T, false, Cfg::kRows, kThreads>(a, rp, out, b, split, g * group + row0, rows, ro, DP,
                                             rm, rl, smem + Cfg::kJoin);
  pdl_wait();  // this launch ends after the prefix launch before it
}

constexpr int kGenericRows = 32;

template <typename T, int DP, int RW, int TG, bool kPrefix>
int launch_generic_one(dim3 grid, int tile_rows, T* out, const T* q, const T* k, const T* v, const Args& a,
                       cudaStream_t s) {
  using Cfg = GenCfg<DP, RW, TG>;
  auto kern = sp_generic_kernel<T, DP, RW, TG, kPrefix>;
  if (Cfg::kSmemBytes > 48 * 1024)
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
  grid.z = kPrefix ? (tile_rows + Cfg::kRows - 1) / Cfg::kRows
                   : (a.group + Cfg::kRows - 1) / Cfg::kRows;
  launch_pdl(kern, grid, dim3(kThreads), Cfg::kSmemBytes, s, out, q, k, v, a);
  return check_launch("as_shared_prefix_decode_attention");
}

template <typename T, int DP>
int launch_generic(int prefix_grid, int own_grid, int tile_rows, T* out, const T* q, const T* k, const T* v,
                   const Args& a, cudaStream_t s) {
  if (prefix_grid > 0) {
    const int rc = launch_generic_one<T, DP, 4, 1, true>(dim3(prefix_grid, a.Kh), tile_rows, out,
                                                         q, k, v, a, s);
    if (rc) return rc;
  }
  const dim3 grid(own_grid, a.Kh);
  // few heads per KV head: warps share the tokens instead
  if (a.group <= 4 && DP <= 128)
    return launch_generic_one<T, DP, 1, 2, false>(grid, tile_rows, out, q, k, v, a, s);
  if (a.group <= 8) return launch_generic_one<T, DP, 1, 1, false>(grid, tile_rows, out, q, k, v, a, s);
  return launch_generic_one<T, DP, 4, 1, false>(grid, tile_rows, out, q, k, v, a, s);
}

template <typename T>
int launch_generic_dim(int prefix_grid, int own_grid, int tile_rows, T* out, const T* q, const T* k, const T* v,
                       const Args& a, cudaStream_t s) {
  if (a.D <= 32) return launch_generic<T, 32>(prefix_grid, own_grid, tile_rows, out, q, k, v, a, s);
  if (a.D <= 64) return launch_generic<T, 64>(prefix_grid, own_grid, tile_rows, out, q, k, v, a, s);
  if (a.D <= 128) return launch_generic<T, 128>(prefix_grid, own_grid, tile_rows, out, q, k, v, a, s);
  return launch_generic<T, 256>(prefix_grid, own_grid, tile_rows, out, q, k, v, a, s);
}

// ===========================================================================
// Plan
// ===========================================================================
// Sizes that depend on the batch size and the geometry alone, so a captured graph and
// its workspace serve every plan of the same batch size.
struct Limits {
  int tile_rows;      // query rows of a prefix item
  int prefix_slots;   // prefix blocks (CTAs) aimed at, over all KV heads
  int own_slots;      // own CTAs aimed at
  int min_prefix;     // smallest prefix split, in 16-token blocks
  int min_own;
  int prefix_items, own_items;    // most items a plan can have
  int64_t prefix_parts, own_parts;  // most parts (of H heads each)
};

Limits limits(int B, int H, int Kh, int D, int dtype) {
  Limits n{};
  const int group = H / Kh;
  n.tile_rows = tc_geometry(D, dtype) ? kTcTileRows : kGenericRows;
  n.prefix_slots = 2 * sm_count();
  n.own_slots = 6 * sm_count();
  n.min_prefix = 8;
  n.min_own = 8;
  const int tiles = (int(int64_t(B) * group / n.tile_rows) + B / 2 + 1);
  n.prefix_items = (n.prefix_slots + Kh - 1) / Kh + tiles;
  n.own_items = (n.own_slots + Kh - 1) / Kh + B;
  n.prefix_parts = B + (int64_t(n.prefix_slots) * n.tile_rows + H - 1) / H;
  n.own_parts = n.own_items;
  return n;
}

int64_t plan_ints(const Limits& n, int B) {
  return kHeader + int64_t(B) * (kRowInts + 1) + int64_t(n.prefix_items) * kPrefixInts +
         int64_t(n.own_items) * kOwnInts;
}

bool sizes_ok(int B, int H, int Kh, int D, int dtype) {
  return B > 0 && B <= 65535 && H > 0 && Kh > 0 && H % Kh == 0 && H <= 65535 && D > 0 &&
         D <= 256 && dtype_size(dtype) > 0 && int64_t(B) * H < (int64_t(1) << 30);
}

}  // namespace
}  // namespace sp
}  // namespace asb

using namespace asb;
using namespace asb::sp;

extern "C" int64_t as_shared_prefix_plan_ints(int32_t num_seqs, int32_t num_heads,
                                              int32_t num_kv_heads, int32_t head_dim,
                                              int32_t dtype) {
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, dtype)) return 0;
  return plan_ints(limits(num_seqs, num_heads, num_kv_heads, head_dim, dtype), num_seqs);
}

extern "C" size_t as_shared_prefix_workspace_size(int32_t num_seqs, int32_t num_heads,
                                                  int32_t num_kv_heads, int32_t head_dim,
                                                  int32_t dtype) {
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, dtype)) return 0;
  const Limits n = limits(num_seqs, num_heads, num_kv_heads, head_dim, dtype);
  const size_t rows = size_t(n.prefix_parts + n.own_parts) * num_heads;
  return align256(size_t(num_seqs) * num_heads * sizeof(int32_t)) +
         align256(rows * sizeof(float2)) + align256(rows * head_dim * sizeof(float));
}

extern "C" int as_shared_prefix_plan(int32_t* plan, int64_t capacity,
                                     const int32_t* group_offsets, const int32_t* members,
                                     const int32_t* prefix_blocks, int32_t num_groups,
                                     const int32_t* row_blocks, int32_t num_seqs,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t dtype, int32_t full_grid) {
  const char* who = "as_shared_prefix_plan";
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, dtype) || num_groups < 0)
    return fail(AS_ERR_INVALID_ARG, "%s: bad sizes (B=%d H=%d Kh=%d D=%d groups=%d)", who,
                num_seqs, num_heads, num_kv_heads, head_dim, num_groups);
  if (!plan || !row_blocks || (num_groups && (!group_offsets || !members || !prefix_blocks)))
    return fail(AS_ERR_INVALID_ARG, "%s: null pointer", who);
  const int B = num_seqs, H = num_heads, Kh = num_kv_heads, group = H / Kh;
  const Limits n = limits(B, H, Kh, head_dim, dtype);
  if (capacity < plan_ints(n, B))
    return fail(AS_ERR_INVALID_ARG, "%s: the plan needs %lld ints", who,
                static_cast<long long>(plan_ints(n, B)));
  // C++ allocations below may throw; nothing may leave a C entry that way
  try {
    struct Group {
      int first, size, blocks, tiles, splits, chunk;
    };
    std::vector<Group> groups;
    std::vector<int> shared(B, 0), seen(B, 0);
    std::vector<int> list;
    if (num_groups && group_offsets[0] != 0)
      return fail(AS_ERR_INVALID_ARG, "%s: group_offsets must start at 0", who);
    for (int i = 0; i < num_groups; ++i) {
      const int lo = group_offsets[i], hi = group_offsets[i + 1];
      if (lo > hi || hi > B)
        return fail(AS_ERR_INVALID_ARG, "%s: group_offsets must rise to at most num_seqs", who);
      if (prefix_blocks[i] < 0)
        return fail(AS_ERR_INVALID_ARG, "%s: negative prefix_blocks", who);
      for (int j = lo; j < hi; ++j) {
        const int b = members[j];
        if (b < 0 || b >= B || seen[b]++)
          return fail(AS_ERR_INVALID_ARG,
                      "%s: members must be different rows of the batch (row %d)", who, b);
        if (row_blocks[b] < prefix_blocks[i])
          return fail(AS_ERR_INVALID_ARG, "%s: row %d holds fewer blocks than its group shares",
                      who, b);
      }
      // one member, or nothing shared: its keys are its own
      if (hi - lo < 2 || prefix_blocks[i] == 0) continue;
      Group g{int(list.size()), hi - lo, prefix_blocks[i], 0, 0, 0};
      g.tiles = int((int64_t(g.size) * group + n.tile_rows - 1) / n.tile_rows);
      for (int j = lo; j < hi; ++j) {
        list.push_back(members[j]);
        shared[members[j]] = g.blocks;
      }
      groups.push_back(g);
    }
    for (int b = 0; b < B; ++b)
      if (row_blocks[b] < 0) return fail(AS_ERR_INVALID_ARG, "%s: negative row_blocks", who);

    // prefix splits: about prefix_slots CTAs in all, and within the workspace's parts
    int64_t work = 0;
    for (const Group& g : groups) work += int64_t(g.tiles) * g.blocks * Kh;
    int64_t chunk = std::max<int64_t>(n.min_prefix, (work + n.prefix_slots - 1) / n.prefix_slots);
    for (;; chunk += chunk / 2) {
      int64_t parts = 0;
      for (Group& g : groups) {
        g.splits = int(std::min<int64_t>(kMaxSplits, (g.blocks + chunk - 1) / chunk));
        g.chunk = (g.blocks + g.splits - 1) / g.splits;
        g.splits = (g.blocks + g.chunk - 1) / g.chunk;
        parts += int64_t(g.splits) * g.size;
      }
      if (parts <= n.prefix_parts) break;
    }
    int64_t own_work = 0;
    for (int b = 0; b < B; ++b) own_work += int64_t(row_blocks[b] - shared[b]) * Kh;
    const int64_t own_chunk =
        std::max<int64_t>(n.min_own, (own_work + n.own_slots - 1) / n.own_slots);

    std::fill(plan, plan + kHeader, 0);
    int32_t* rows = plan + kHeader;
    std::fill(rows, rows + int64_t(B) * kRowInts, 0);
    int32_t* mem = rows + int64_t(B) * kRowInts;
    std::fill(mem, mem + B, 0);
    std::copy(list.begin(), list.end(), mem);
    int32_t* pre = mem + B;
    int32_t* own = pre + int64_t(n.prefix_items) * kPrefixInts;
    int n_pre = 0, n_own = 0, most = 0;
    int64_t part = 0;
    for (const Group& g : groups) {
      most = std::max(most, g.blocks);
      for (int i = 0; i < g.size; ++i) {
        int32_t* r = rows + int64_t(list[g.first + i]) * kRowInts;
        r[kRShared] = g.blocks;
        r[kRPrefixSplits] = g.splits;
        r[kRPrefixPart] = int32_t(part + i);
        r[kRPrefixStep] = g.size;
      }
      const int all_rows = g.size * group;
      for (int s = 0; s < g.splits; ++s)
        for (int t = 0; t < g.tiles; ++t) {
          int32_t* it = pre + int64_t(n_pre++) * kPrefixInts;
          std::fill(it, it + kPrefixInts, 0);
          it[kPMembers] = g.first;
          it[kPRow0] = t * n.tile_rows;
          it[kPRows] = std::min(n.tile_rows, all_rows - t * n.tile_rows);
          it[kPBegin] = s * g.chunk;
          it[kPEnd] = std::min(g.blocks, (s + 1) * g.chunk);
          it[kPPart] = int32_t(part + int64_t(s) * g.size);
        }
      part += int64_t(g.splits) * g.size;
    }
    // own items, the longest first so that the last to start are short
    struct Own {
      int row, split, blocks;
    };
    std::vector<Own> items;
    int64_t own_part = 0;
    for (int b = 0; b < B; ++b) {
      const int blocks = row_blocks[b] - shared[b];
      const int splits = std::clamp<int>(int((blocks + own_chunk - 1) / own_chunk), 1, kMaxSplits);
      int32_t* r = rows + int64_t(b) * kRowInts;
      r[kROwnSplits] = splits;
      r[kROwnPart] = int32_t(own_part);
      if (splits > 1) own_part += splits;
      for (int s = 0; s < splits; ++s) items.push_back({b, s, (blocks + splits - 1) / splits});
    }
    std::stable_sort(items.begin(), items.end(),
                     [](const Own& x, const Own& y) { return x.blocks > y.blocks; });
    for (const Own& x : items) {
      int32_t* it = own + int64_t(n_own++) * kOwnInts;
      std::fill(it, it + kOwnInts, 0);
      it[kORow] = x.row;
      it[kOSplit] = x.split;
    }
    plan[kHMagic] = kMagic;
    plan[kHSeqs] = B;
    plan[kHHeads] = H;
    plan[kHKvHeads] = Kh;
    plan[kHDim] = head_dim;
    plan[kHDtype] = dtype;
    plan[kHPrefixItems] = n_pre;
    plan[kHOwnItems] = n_own;
    plan[kHPrefixGrid] = full_grid ? n.prefix_items : n_pre;
    plan[kHOwnGrid] = full_grid ? n.own_items : n_own;
    plan[kHOffRows] = kHeader;
    plan[kHOffMembers] = int32_t(mem - plan);
    plan[kHOffPrefix] = int32_t(pre - plan);
    plan[kHOffOwn] = int32_t(own - plan);
    plan[kHPrefixParts] = int32_t(n.prefix_parts);
    plan[kHOwnParts] = int32_t(n.own_parts);
    plan[kHTileRows] = n.tile_rows;
    plan[kHInts] = int32_t((own - plan) + int64_t(n.own_items) * kOwnInts);
    plan[kHMostShared] = most;
  } catch (...) {
    return fail(AS_ERR_INVALID_ARG, "%s: out of host memory", who);
  }
  return AS_OK;
}

extern "C" int as_shared_prefix_decode_attention(
    void* out, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
    const int32_t* block_tables, int64_t bt_stride, const int32_t* seq_lens_k,
    const int32_t* plan_header, const int32_t* plan, int32_t num_seqs, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks,
    int32_t max_blocks, float scale, void* workspace, size_t workspace_bytes, int32_t out_layout,
    int32_t dtype, as_stream_t stream) {
  const char* who = "as_shared_prefix_decode_attention";
  if (!dtype_size(dtype)) return fail(AS_ERR_INVALID_ARG, "%s: unknown dtype", who);
  if (block_size != kBS)
    return fail(AS_ERR_UNSUPPORTED, "%s: block_size must be 16 (got %d)", who, block_size);
  if (num_seqs == 0) return AS_OK;
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, dtype) || num_blocks <= 0 ||
      max_blocks <= 0 || bt_stride < max_blocks || q_stride < int64_t(num_heads) * head_dim)
    return fail(AS_ERR_INVALID_ARG, "%s: bad sizes (B=%d H=%d Kh=%d D=%d NB=%d maxb=%d)", who,
                num_seqs, num_heads, num_kv_heads, head_dim, num_blocks, max_blocks);
  if (out_layout != AS_LAYOUT_HEAD_MAJOR && out_layout != AS_LAYOUT_DIM_MAJOR)
    return fail(AS_ERR_INVALID_ARG, "%s: unknown out_layout %d", who, out_layout);
  if (!(scale > 0.f) || scale > 3e38f)
    return fail(AS_ERR_INVALID_ARG, "%s: scale must be positive and finite", who);
  if (!out || !q || !k_cache || !v_cache || !block_tables || !seq_lens_k || !plan_header || !plan)
    return fail(AS_ERR_INVALID_ARG, "%s: null pointer", who);
  const int32_t* h = plan_header;
  if (h[kHMagic] != kMagic || h[kHSeqs] != num_seqs || h[kHHeads] != num_heads ||
      h[kHKvHeads] != num_kv_heads || h[kHDim] != head_dim || h[kHDtype] != dtype)
    return fail(AS_ERR_INVALID_ARG, "%s: the plan was made for another batch", who);
  if (h[kHMostShared] > max_blocks)
    return fail(AS_ERR_INVALID_ARG, "%s: the plan shares %d blocks, the table holds %d", who,
                h[kHMostShared], max_blocks);
  const Limits n = limits(num_seqs, num_heads, num_kv_heads, head_dim, dtype);
  if (h[kHPrefixParts] != n.prefix_parts || h[kHOwnParts] != n.own_parts)
    return fail(AS_ERR_INVALID_ARG, "%s: the plan was made for another GPU", who);
  const size_t need = as_shared_prefix_workspace_size(num_seqs, num_heads, num_kv_heads, head_dim,
                                                      dtype);
  if (!workspace || workspace_bytes < need)
    return fail(AS_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, need);
  if (reinterpret_cast<uintptr_t>(workspace) & 255)
    return fail(AS_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", who);

  Args a{};
  a.plan = plan;
  a.bt = block_tables;
  a.bt_stride = bt_stride;
  a.seq_lens = seq_lens_k;
  a.q_stride = q_stride;
  a.H = num_heads;
  a.Kh = num_kv_heads;
  a.D = head_dim;
  a.group = num_heads / num_kv_heads;
  a.num_blocks = num_blocks;
  a.max_blocks = max_blocks;
  a.scale = scale;
  a.own_part0 = int(n.prefix_parts);
  a.os_h = out_layout == AS_LAYOUT_HEAD_MAJOR ? head_dim : 1;
  a.os_d = out_layout == AS_LAYOUT_HEAD_MAJOR ? 1 : num_heads;
  a.wait_first = h[kHPrefixGrid] == 0;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const size_t rows = size_t(n.prefix_parts + n.own_parts) * num_heads;
  a.parts.counters = reinterpret_cast<int32_t*>(w);
  w += align256(size_t(num_seqs) * num_heads * sizeof(int32_t));
  a.parts.ml = reinterpret_cast<float2*>(w);
  w += align256(rows * sizeof(float2));
  a.parts.o = reinterpret_cast<float*>(w);
  a.status = device_status_ptr();
  a.wait_limit = wait_limit_ns();
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // TMA reads the planes from 16-byte boundaries; others take the CUDA-core kernels
  const bool aligned = ((reinterpret_cast<uintptr_t>(k_cache) |
                         reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0;
  if (tc_geometry(head_dim, dtype) && aligned)
    return tc_launch(h[kHPrefixGrid], h[kHOwnGrid], out, q, k_cache, v_cache, a, dtype, s);
  auto run = [&](auto tag) -> int {
    using T = decltype(tag);
    return launch_generic_dim<T>(h[kHPrefixGrid], h[kHOwnGrid], n.tile_rows, static_cast<T*>(out),
                                 static_cast<const T*>(q), static_cast<const T*>(k_cache),
                                 static_cast<const T*>(v_cache), a, s);
  };
  switch (dtype) {
    case AS_DTYPE_F32: return run(float());
    case AS_DTYPE_F16: return run(__half());
    default: return run(__nv_bfloat16());
  }
}
