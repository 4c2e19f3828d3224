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
#include <utility>
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
// lane.  TG > 1 gives token groups to different warps when there are few rows.  Bound, on
// short parts, by the round of each 32 * TG tokens: ids, then K / V with no load in flight over
// the arithmetic, and three block barriers (16 fp32 sequences in two groups on 1,024 tokens
// 26 us, of which FMAs are 2); on long ones by FMAs and shared-memory reads: 64 bf16 sequences
// on 4,096 tokens 209 us where the tensor-core launches take 20.
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
  static_assert(!kPrefix || TG == 1, "a prefix item leaves one result");
  constexpr int EPL = DP / 32;
  if (kPrefix || a.wait_first) {
    pdl_wait();
    pdl_trigger();
  }
  const int g = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.D, group = a.group;

  // this item's query rows and token range
  int b = 0, split = 0, row0, rows, begin, end, part = 0, table_row;
  const int32_t* members = nullptr;
  RowPlan rp{};
  if (kPrefix) {
    const PrefixItem it = load_item(a.prefix_items, blockIdx.x);
    members = a.members + it.members;
    row0 = it.row0 + blockIdx.z * Cfg::kRows;  // the plan's tiles may be larger
    rows = min(Cfg::kRows, it.rows - int(blockIdx.z) * Cfg::kRows);
    if (rows <= 0) return;
    if (it.end > a.max_blocks) {  // of a group that row_plan() attends alone: not in the table
      if (threadIdx.x == 0) flag_status(a.status, kStatusBadLength);
      return;
    }
    begin = it.begin * kBS;
    end = it.end * kBS;
    part = it.part;
    table_row = it.table_row;
  } else {
    const OwnItem it = load_item(a.own_items, blockIdx.x);
    if (it.own_splits == 0) {
      pdl_wait();
      return;
    }
    b = table_row = it.row;
    split = it.split;
    row0 = blockIdx.z * Cfg::kRows;
    rows = min(Cfg::kRows, group - row0);
    rp = row_plan(a, it, threadIdx.x == 0 && split == 0 && g == 0 && row0 == 0);
    begin = rp.begin * kBS;
    end = min(rp.len, (rp.begin + rp.count) * kBS);
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

  // the token groups' results in shared memory, for the join
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
  if (kPrefix) {
    for (int i = threadIdx.x; i < rows * D; i += kThreads) {
      const int r = i / D, d = i - r * D, rr = row0 + r;
      const size_t at = size_t(part + rr / group) * a.H + g * group + rr % group;
      a.parts.o[at * D + d] = ro[r * DP + d];
      if (d == 0) {
        a.parts.ml[at] = make_float2(rm[r], rl[r]);
      }
    }
    return;
  }
  finish_own<T, false, Cfg::kRows, kThreads, TG>(a, rp, out, b, split, g * group + row0, rows, ro, DP,
                                             rm, rl, smem + Cfg::kJoin);
  pdl_wait();  // this launch ends after the prefix launch before it
}

constexpr int kGenericRows = 32;
// Fixed costs of a block, in the units of its piece: halves of a 128-key tile, and blocks of
// 16 keys.  Measured, us per call (n sequences on their shared tokens): prefix 5, with 2 and
// with 10 the same within 1%; own 16, with 32 the same, with 6 64 on 4,096 26.5 instead of 19.9
// and on 14,336 39.3 instead of 33.3.
constexpr int64_t kPrefixOverhead = 5;
constexpr int64_t kOwnOverhead = 16;
// Least own blocks of an item, where a row has that many: with 4, 16 fp32 sequences on 1,024
// take 33.7 us instead of 25.8; with 16 as with 8.
constexpr int64_t kMinOwn = 8;
// Most blocks of a row: its keys are counted in 31 bits.
constexpr int kMostBlocks = (1 << 27) - 1;
static_assert(int64_t(kMostBlocks) * kBS < int64_t(1) << 31, "keys");

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
  bool tc;
  int tile_rows;     // most query rows of a prefix item
  int prefix_slots;  // prefix blocks (CTAs) that run at once, over all KV heads
  int own_slots;     // own CTAs that run at once
  int own_per_item;  // CTAs of an own item
  int prefix_items, own_items;      // most items a plan can have
  int64_t prefix_parts, own_parts;  // most parts (of H heads each)
};

Limits limits(int B, int H, int Kh, int D, int dtype) {
  Limits n{};
  const int group = H / Kh;
  n.tc = tc_geometry(D, dtype);
  n.tile_rows = n.tc ? kTcTileRows : kGenericRows;
  n.prefix_slots = (n.tc ? 1 : 2) * sm_count();
  n.own_slots = (n.tc && D == 64 ? 4 : 3) * sm_count();
  n.own_per_item = Kh * (n.tc ? (group + 7) / 8 : 1);
  const int per_tile = std::max(1, n.tile_rows / group) * group;  // rows, whole members
  const int tiles = int(int64_t(B) * group / std::min(per_tile, n.tile_rows)) + B + 1;
  n.prefix_items = 2 * n.prefix_slots / Kh + tiles;
  n.own_items = 4 * n.own_slots / n.own_per_item + B;
  // a prefix CTA leaves at most tile_rows rows of parts
  n.prefix_parts = int64_t(B) + 2 * int64_t(n.prefix_slots) * n.tile_rows / H;
  n.own_parts = n.own_items;
  return n;
}

// Least cost C such that pieces of at most C fit in `fit` CTAs, at most `waves` waves of
// them: tries one wave after the other, each with a fixed cost, and keeps the cheapest.
// count(C) falls as C grows.
template <typename F>
int64_t best_piece(int64_t least, int64_t most, int64_t slots, int max_waves, int64_t overhead,
                   F count) {
  int64_t best = -1, best_cost = 0;
  for (int waves = 1; waves <= max_waves; ++waves) {
    if (count(most) > slots * waves) continue;
    int64_t lo = least, hi = most;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (count(mid) <= slots * waves)
        hi = mid;
      else
        lo = mid + 1;
    }
    const int64_t cost = waves * (lo + overhead);
    if (best < 0 || cost < best_cost) {
      best = lo;
      best_cost = cost;
    }
  }
  return best < 0 ? most : best;
}

int64_t plan_ints(const Limits& n, int B) {
  return kHeader + (int64_t(B) + 3) / 4 * 4 +
         (int64_t(n.prefix_items) + n.own_items) * kItemInts;
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
      int first, size, blocks, tiles, tile_rows, splits, chunk;
    };
    std::vector<Group> groups;
    std::vector<int> shared(B, 0), seen(B, 0);
    std::vector<int> list;
    if (num_groups && group_offsets[0] != 0)
      return fail(AS_ERR_INVALID_ARG, "%s: group_offsets must start at 0", who);
    for (int b = 0; b < B; ++b) {
      if (row_blocks[b] < 0) return fail(AS_ERR_INVALID_ARG, "%s: negative row_blocks", who);
      if (row_blocks[b] > kMostBlocks)  // bounds the shared blocks too, checked below
        return fail(AS_ERR_INVALID_ARG, "%s: row_blocks past %d", who, kMostBlocks);
    }
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
      // whole members to a tile
      Group g{int(list.size()), hi - lo, prefix_blocks[i], 0, 0, 0, 0};
      g.tile_rows = group > n.tile_rows ? n.tile_rows : n.tile_rows / group * group;
      g.tiles = (g.size * group + g.tile_rows - 1) / g.tile_rows;
      for (int j = lo; j < hi; ++j) {
        list.push_back(members[j]);
        shared[members[j]] = g.blocks;
      }
      groups.push_back(g);
    }

    // prefix splits: pieces of about equal length, in units of 8 blocks (half units on
    // tensor cores, for the fixed cost)
    const int64_t cost = n.tc ? 2 : 1;
    auto split_prefix = [&](int64_t piece) -> int64_t {
      int64_t ctas = 0;
      for (Group& g : groups) {
        const int units = (g.blocks + 7) / 8;
        const int splits = int(std::min<int64_t>(kMaxSplits, (units * cost + piece - 1) / piece));
        g.chunk = (units + splits - 1) / splits * 8;
        g.splits = (g.blocks + g.chunk - 1) / g.chunk;
        ctas += int64_t(g.splits) * g.tiles * Kh;
      }
      return ctas;
    };
    if (!groups.empty()) {
      int64_t most = 2;
      for (const Group& g : groups) most = std::max(most, (g.blocks + 7) / 8 * cost);
      int64_t piece = best_piece(n.tc ? 2 : 1, most, n.prefix_slots, 2, n.tc ? kPrefixOverhead : 1,
                                 split_prefix);
      for (;; piece += (piece + 1) / 2) {  // and within the workspace's parts and the items
        const int64_t ctas = split_prefix(piece);
        int64_t parts = 0;
        for (const Group& g : groups) parts += int64_t(g.splits) * g.size;
        if (parts <= n.prefix_parts && ctas / Kh <= n.prefix_items) break;
      }
    }
    auto own_splits = [&](int b, int64_t piece) -> int {
      const int64_t blocks = row_blocks[b] - shared[b];
      return int(std::clamp<int64_t>((blocks + piece - 1) / piece, 1, kMaxSplits));
    };
    int64_t own_most = kMinOwn;
    for (int b = 0; b < B; ++b) own_most = std::max<int64_t>(own_most, row_blocks[b] - shared[b]);
    const int64_t own_piece =
        best_piece(kMinOwn, own_most, n.own_slots, 4, n.tc ? kOwnOverhead : 8,
                   [&](int64_t piece) {
          int64_t items = 0;
          for (int b = 0; b < B; ++b) items += own_splits(b, piece);
          return items * n.own_per_item;
        });

    std::fill(plan, plan + kHeader, 0);
    int32_t* mem = plan + kHeader;
    const int mem_ints = (B + 3) / 4 * 4;
    auto* pre = reinterpret_cast<PrefixItem*>(mem + mem_ints);
    auto* own = reinterpret_cast<OwnItem*>(pre + n.prefix_items);
    std::fill(mem, mem + (plan_ints(n, B) - kHeader), 0);
    std::copy(list.begin(), list.end(), mem);
    std::vector<OwnItem> row_items(B, OwnItem{});
    int n_pre = 0, n_own = 0, most = 0;
    int part = 0;
    for (const Group& g : groups) {
      most = std::max(most, g.blocks);
      for (int i = 0; i < g.size; ++i) {
        OwnItem& r = row_items[list[g.first + i]];
        r.shared = g.blocks;
        r.prefix_splits = g.splits;
        r.prefix_part = part + i;
        r.prefix_step = g.size;
      }
      const int all_rows = g.size * group;
      for (int s = 0; s < g.splits; ++s)
        for (int t = 0; t < g.tiles; ++t) {
          PrefixItem& it = pre[n_pre++];
          it.table_row = list[g.first];
          it.members = g.first;
          it.row0 = t * g.tile_rows;
          it.rows = std::min(g.tile_rows, all_rows - t * g.tile_rows);
          it.begin = s * g.chunk;
          it.end = std::min(g.blocks, (s + 1) * g.chunk);
          it.part = part + s * g.size;
        }
      part += g.splits * g.size;
    }
    // own items, the longest first so that the last to start are short
    std::vector<std::pair<int64_t, OwnItem>> items;
    int own_part = 0;
    for (int b = 0; b < B; ++b) {
      const int64_t blocks = row_blocks[b] - shared[b];
      OwnItem& r = row_items[b];
      r.row = b;
      r.own_splits = own_splits(b, own_piece);
      r.own_part = own_part;
      if (r.own_splits > 1) own_part += r.own_splits;
      for (r.split = 0; r.split < r.own_splits; ++r.split)
        items.push_back({(blocks + r.own_splits - 1) / r.own_splits, r});
    }
    std::stable_sort(items.begin(), items.end(),
                     [](const auto& x, const auto& y) { return x.first > y.first; });
    for (const auto& x : items) own[n_own++] = x.second;
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
    plan[kHOffMembers] = int32_t(mem - plan);
    plan[kHOffPrefix] = int32_t(reinterpret_cast<int32_t*>(pre) - plan);
    plan[kHOffOwn] = int32_t(reinterpret_cast<int32_t*>(own) - plan);
    plan[kHPrefixParts] = int32_t(n.prefix_parts);
    plan[kHOwnParts] = int32_t(n.own_parts);
    plan[kHTileRows] = n.tile_rows;
    plan[kHInts] = int32_t(plan_ints(n, B));
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
  if (reinterpret_cast<uintptr_t>(plan) & 15)
    return fail(AS_ERR_INVALID_ARG, "%s: the plan must be 16-byte aligned", who);
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
  a.members = plan + h[kHOffMembers];
  a.prefix_items = reinterpret_cast<const PrefixItem*>(plan + h[kHOffPrefix]);
  a.own_items = reinterpret_cast<const OwnItem*>(plan + h[kHOffOwn]);
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
