// (9) Shared-prefix decode attention on tensor cores: bf16 / fp16, head_dim 64 or 128.
//
// Prefix launch (sp_prefix_kernel).  A group's members' query heads of KV head g are the
// rows of a matrix: a tile of 128 of them attends over one range of the shared blocks
// with tcgen05.mma, S = Q K^T into TMEM, softmax by four warps (one row per thread),
// P back into TMEM as the A operand of O += P V.  K / V tiles arrive by TMA, block by
// block.  Roles: warp 0 loads, warp 1 issues MMAs, warps 2-5 softmax.  Two blocks share
// an SM (about 100 KB of shared memory and 256 TMEM columns each), so one's
// exponentials overlap the other's products and waits.
//
// Own launch (sp_own_kernel).  One sequence, up to 8 query heads of a KV head: too few
// rows for tcgen05, and bound by reading K / V once; the decode kernel's warp-level
// m16n8k16 fold over TMA-staged blocks (decode_tile.cuh).  Its blocks start while the
// prefix launch runs, and join the parts (shared_prefix.cuh) after it.
//
// Every wait is bounded: one that runs out sets status bit 4, the block stops issuing,
// lets its copies land, frees its TMEM and leaves an empty part.
#include <string.h>

#include <type_traits>

#include "common.cuh"
#include "decode_tile.cuh"
#include "f32x2.cuh"
#include "host_util.h"
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

namespace asb {
namespace sp {
namespace {

constexpr float kLazySlack = 8.0f;  // log2 units a row's scores may exceed its maximum by

// ===========================================================================
// Prefix
// ===========================================================================
template <int HD>
struct PreCfg {
  static constexpr int D = HD;
  static constexpr int kBN = D == 64 ? 128 : 64;  // keys per tile: 32 KB of K and V
  static constexpr int kBlocks = kBN / kBS;
  static constexpr int kSub = D / 64;             // 128-byte-wide swizzle sub-tiles
  static constexpr int kQSub = 128 * 128;
  static constexpr int kKVSub = kBN * 128;
  static constexpr int kQBytes = kSub * kQSub;
  static constexpr int kKVBytes = kSub * kKVSub;  // K (or V) of one tile
  static constexpr int kStages = 2;
  static constexpr int kOffKV = kQBytes;
  static constexpr int kOffBar = kOffKV + kStages * 2 * kKVBytes;
  static constexpr int kSmemBytes = kOffBar + 256;
  static constexpr int kThreads = 192;
  // TMEM columns: S [0, kBN), P (16-bit pairs) after it, O the last D of 256
  static constexpr int kCols = 256;
  static constexpr int kColP = kBN;
  static constexpr int kColO = kCols - D;
  static_assert(kBN + kBN / 2 + D <= kCols, "TMEM columns");
  static_assert(2 * (kSmemBytes + 1024) <= 227 * 1024, "two blocks per SM");
};

struct PreBars {
  uint64_t kv_full[2], kv_empty[2];
  uint64_t s_full, s_free, p_full, pv_done, drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(PreBars) <= 256, "barrier block");

__device__ __forceinline__ bool stopped(volatile int* flag) { return *flag != 0; }

template <typename T, int HD>
__global__ void __launch_bounds__(192, 2)
sp_prefix_kernel(const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const T* __restrict__ q,
                 const Args a, float scale_log2, int starve) {
  using Cfg = PreCfg<HD>;
  constexpr int D = Cfg::D, BN = Cfg::kBN, NS = Cfg::kStages, NB = Cfg::kBlocks;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescS = tc::idesc_f16(kBF16, 128, BN, false, false);
  constexpr uint32_t kIdescO = tc::idesc_f16(kBF16, 128, D, false, true);
  pdl_wait();
  pdl_trigger();  // every block of this launch has started: the own launch may start

  const int32_t* plan = a.plan;
  if (int(blockIdx.x) >= plan[kHPrefixItems]) return;
  const int32_t* it = plan + plan[kHOffPrefix] + blockIdx.x * kPrefixInts;
  const int32_t* members = plan + plan[kHOffMembers] + it[kPMembers];
  const int row0 = it[kPRow0], rows = it[kPRows];
  const int begin = it[kPBegin], end = it[kPEnd], part = it[kPPart];
  const int g = blockIdx.y, group = a.group;
  const int n_tiles = (end - begin + NB - 1) / NB;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  PreBars* bars = reinterpret_cast<PreBars*>(smem + Cfg::kOffBar);
  volatile int* abort_flag = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int active = (rows + 31) / 32;  // softmax warps with rows
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars->kv_full[s], 1);
      mbar_init(&bars->kv_empty[s], 1);
    }
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->s_free, active);
    mbar_init(&bars->p_full, active);
    mbar_init(&bars->pv_done, 1);
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(&bars->tmem, Cfg::kCols);
    tc::tmem_relinquish();
  }
  // Q rows (member, head) into the 128B-swizzled layout; rows past the tile are zero
  {
    const bool vec = ((reinterpret_cast<uintptr_t>(q) | uintptr_t(a.q_stride * 2)) & 15) == 0;
    for (int i = threadIdx.x; i < 128 * (D / 8); i += Cfg::kThreads) {
      const int r = i / (D / 8), c = i - r * (D / 8);
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        const int rr = row0 + r;
        const T* src = q + int64_t(members[rr / group]) * a.q_stride +
                       int64_t(g * group + rr % group) * D + c * 8;
        if (vec) {
          x = *reinterpret_cast<const uint4*>(src);
        } else {
          T* e = reinterpret_cast<T*>(&x);
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = src[j];
        }
      }
      *reinterpret_cast<uint4*>(smem + (c >> 3) * Cfg::kQSub + r * 128 +
                                (((c & 7) ^ (r & 7)) << 4)) = x;
    }
    fence_proxy_async_smem();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = bars->tmem;
  const uint32_t sQ = smem_u32(smem), sKV = smem_u32(smem + Cfg::kOffKV);

  int issued = 0;
  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (!starve) {
      if (lane == 0) {
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
      }
      const int32_t* row = a.bt + int64_t(members[0]) * a.bt_stride;
      // blocks past the range: any block of it (finite as the rest), masked below
      const int first = row[begin];
      const int fill = first >= 0 && first < a.num_blocks ? first : 0;
      auto load_id = [&](int j) -> int {
        const int blk = begin + NB * j + (lane & (NB - 1));
        int id = fill;
        if (blk < end) {
          id = __ldg(row + blk);
          if (id < 0 || id >= a.num_blocks) {
            flag_status(a.status, kStatusBadBlockId);
            id = fill;
          }
        }
        return id;
      };
      const uint64_t policy = l2_policy_evict_last();  // other row tiles read them too
      int id = load_id(0);
      for (int j = 0; j < n_tiles; ++j) {
        const int st = j % NS;
        const bool ready =
            !stopped(abort_flag) &&
            (j < NS || mbar_wait(&bars->kv_empty[st], ((j / NS) + 1) & 1, a.status, a.wait_limit));
        if (!__all_sync(0xffffffffu, ready)) {
          *abort_flag = 1;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&bars->kv_full[st], 2 * Cfg::kKVBytes);
        __syncwarp();
        uint8_t* stage = smem + Cfg::kOffKV + st * 2 * Cfg::kKVBytes;
        if (lane < NB) {
#pragma unroll
          for (int sb = 0; sb < Cfg::kSub; ++sb) {
            tma_load_4d(stage + sb * Cfg::kKVSub + lane * 2048, &tmap_k, &bars->kv_full[st],
                        sb * 64, g, 0, id, policy);
            tma_load_4d(stage + Cfg::kKVBytes + sb * Cfg::kKVSub + lane * 2048, &tmap_v,
                        &bars->kv_full[st], sb * 64, g, 0, id, policy);
          }
        }
        issued = j + 1;
        if (j + 1 < n_tiles) id = load_id(j + 1);
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMAs
    if (lane == 0) {
      auto issue_s = [&](int st) {
        const uint32_t k = sKV + st * 2 * Cfg::kKVBytes;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_f16(tmem,
                      tc::sdesc_sw128(sQ + (kk >> 2) * Cfg::kQSub + (kk & 3) * 32, 16, 1024),
                      tc::sdesc_sw128(k + (kk >> 2) * Cfg::kKVSub + (kk & 3) * 32, 16, 1024),
                      kIdescS, kk > 0 ? 1u : 0u);
      };
      auto wait = [&](uint64_t* bar, int parity) -> bool {
        return !stopped(abort_flag) && mbar_wait(bar, parity & 1, a.status, a.wait_limit);
      };
      bool ok = wait(&bars->kv_full[0], 0);
      if (ok) {
        issue_s(0);
        tc::commit(&bars->s_full);
      }
      for (int j = 0; ok && j < n_tiles; ++j) {
        if (j + 1 < n_tiles) {  // S of the next tile while the softmax works on this one
          ok = wait(&bars->kv_full[(j + 1) % NS], (j + 1) / NS) && wait(&bars->s_free, j);
          if (!ok) break;
          tc::fence_after_sync();
          issue_s((j + 1) % NS);
          tc::commit(&bars->s_full);
        }
        ok = wait(&bars->p_full, j);
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t v = sKV + (j % NS) * 2 * Cfg::kKVBytes + Cfg::kKVBytes;
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          tc::mma_f16_ts(tmem + Cfg::kColO, tmem + Cfg::kColP + kk * 8,
                         tc::sdesc_sw128(v + kk * 2048, Cfg::kKVSub, 1024), kIdescO,
                         (j > 0 || kk > 0) ? 1u : 0u);
        tc::commit(&bars->pv_done);
        tc::commit(&bars->kv_empty[j % NS]);
      }
      if (!ok) *abort_flag = 1;
      tc::commit(&bars->drain);
      mbar_wait(&bars->drain, 0, a.status, a.wait_limit);
    }
    __syncwarp();
  } else if ((warp & 3) < active) {
    // -------------------------------------------------------------- softmax
    const int quad = warp & 3;  // the TMEM lanes this warp may access
    const int r = quad * 32 + lane;
    const uint32_t tS = tmem + (uint32_t(quad * 32) << 16);
    const uint32_t tP = tS + Cfg::kColP, tO = tS + Cfg::kColO;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const bool go = !stopped(abort_flag) &&
                      mbar_wait(&bars->s_full, j & 1, a.status, a.wait_limit);
      if (!__all_sync(0xffffffffu, go)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      float x[BN];
      {
        uint32_t v[BN / 32][32];
#pragma unroll
        for (int u = 0; u < BN / 32; ++u) tc::ld_32x32b_x32(tS + 32 * u, v[u]);
        tc::wait_ld();
#pragma unroll
        for (int u = 0; u < BN / 32; ++u)
#pragma unroll
          for (int c = 0; c < 32; ++c) x[32 * u + c] = __uint_as_float(v[u][c]);
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->s_free);
      const int keys = (end - begin) * kBS - j * BN;  // of this tile
      if (keys < BN) {
#pragma unroll
        for (int c = 0; c < BN; ++c) x[c] = c < keys ? x[c] : -INFINITY;
      }
      float mp[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) mp[c] = fmaxf(x[c], x[8 + c]);
#pragma unroll
      for (int c = 16; c < BN; c += 16)
#pragma unroll
        for (int e = 0; e < 8; ++e) mp[e] = max3f(mp[e], x[c + e], x[c + 8 + e]);
      const float mx = fmaxf(fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])),
                             fmaxf(fmaxf(mp[4], mp[5]), fmaxf(mp[6], mp[7])));
      // lazy maximum: exponents stay below 2^8, within every type's range, unless a
      // score exceeds the current one by more; then O and l are rescaled
      float alpha = 1.f;
      if (mx * scale_log2 > m + kLazySlack) {
        const float m_new = mx * scale_log2;
        alpha = fast_exp2(m - m_new);
        m = m_new;
      }
      const float neg_m = m == -INFINITY ? 0.f : -m;
      const uint64_t sc2 = f2_pack(scale_log2, scale_log2);
      const uint64_t nm2 = f2_pack(neg_m, neg_m);
      uint64_t sum2[4] = {0, 0, 0, 0};
      uint32_t pk[BN / 2];
#pragma unroll
      for (int c = 0; c < BN / 2; ++c) {
        float e0, e1;
        f2_unpack(f2_fma(f2_pack(x[2 * c], x[2 * c + 1]), sc2, nm2), e0, e1);
        const float p0 = fast_exp2(e0), p1 = fast_exp2(e1);
        sum2[c & 3] = f2_add(sum2[c & 3], f2_pack(p0, p1));
        pk[c] = pack2<T>(p0, p1);
      }
      float s0, s1;
      f2_unpack(f2_add(f2_add(sum2[0], sum2[1]), f2_add(sum2[2], sum2[3])), s0, s1);
      if (j > 0) {  // the product with V of the last tile still reads P and writes O
        if (!__all_sync(0xffffffffu,
                        mbar_wait(&bars->pv_done, (j - 1) & 1, a.status, a.wait_limit))) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
      }
#pragma unroll
      for (int u = 0; u < BN / 64; ++u)
        tc::st_32x32b_x32(tP + 32 * u, *reinterpret_cast<const uint32_t(*)[32]>(&pk[32 * u]));
      l = l * alpha + (s0 + s1);
      if (j > 0 && __any_sync(0xffffffffu, alpha < 1.f)) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tc::ld_32x32b_x32(tO + c * 32, o);
          tc::wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tc::st_32x32b_x32(tO + c * 32, o);
        }
      }
      tc::wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full);
    }
    if (!ok) *abort_flag = 1;
    const bool done = ok && __all_sync(0xffffffffu, mbar_wait(&bars->pv_done, (n_tiles - 1) & 1,
                                                              a.status, a.wait_limit));
    if (ok && !done) *abort_flag = 1;
    const int rr = row0 + r;
    const size_t at = (size_t(part) + rr / group) * a.H + g * group + rr % group;
    if (done) {
      tc::fence_after_sync();
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tc::ld_32x32b_x32(tO + c * 32, o);
        tc::wait_ld();
        if (r < rows) {
          uint4* dst = reinterpret_cast<uint4*>(a.parts.o + at * D + c * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
    }
    if (r < rows) a.parts.ml[at] = done ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
    tc::fence_before_sync();
  }

  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, Cfg::kCols);
  }
  if (warp == 0 && lane == 0 && *abort_flag) {  // let the copies in flight land
    for (int j = max(0, issued - NS); j < issued; ++j)
      mbar_wait(&bars->kv_full[j % NS], (j / NS) & 1, a.status, a.wait_limit);
  }
}

// ===========================================================================
// Own blocks
// ===========================================================================
template <int D>
struct OwnCfg {
  static constexpr int kWarps = 4;  // consumers; one more warp loads
  static constexpr int kThreads = (kWarps + 1) * 32;
  static constexpr int kSub = D / 64;
  static constexpr int kSubBytes = kBS * 128;
  static constexpr int kTileBytes = kSub * kSubBytes;  // one block of K or V, one head
  static constexpr int kSlotBytes = 2 * kTileBytes;
  static constexpr int kStageBytes = kWarps * kSlotBytes;  // a block per consumer warp
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 2 * kStages * 8;
  static constexpr int kHeads = 8;
  static constexpr int kJoinFloats = kWarps * kHeads * (D + 2);
  static_assert(4 * (kJoinFloats + join_scratch(kHeads, kThreads)) <= kStages * kStageBytes,
                "the joins use the stages' space");
};

template <typename T, int D>
__global__ void __launch_bounds__(OwnCfg<D>::kThreads)
sp_own_kernel(const __grid_constant__ CUtensorMap tmap_k,
              const __grid_constant__ CUtensorMap tmap_v, T* __restrict__ out,
              const T* __restrict__ q, const Args a, float scale_log2, int starve) {
  using Cfg = OwnCfg<D>;
  constexpr int NS = Cfg::kStages, KT = D / 16, W = Cfg::kWarps;
  if (a.wait_first) {
    pdl_wait();
    pdl_trigger();
  }
  // Without the wait: everything read below was written before the prefix launch, whose
  // blocks let this launch start only after their own wait for it.
  const int32_t* plan = a.plan;
  if (int(blockIdx.x) >= plan[kHOwnItems]) {
    pdl_wait();
    return;
  }
  const int32_t* it = plan + plan[kHOffOwn] + blockIdx.x * kOwnInts;
  const int b = it[kORow], split = it[kOSplit];
  const int chunks = (a.group + Cfg::kHeads - 1) / Cfg::kHeads;
  const int g = blockIdx.y / chunks, chunk = blockIdx.y - g * chunks;
  const int h0 = g * a.group + chunk * Cfg::kHeads;
  const int heads = min(Cfg::kHeads, a.group - chunk * Cfg::kHeads);
  const RowPlan rp = row_plan(a, b, threadIdx.x == 0 && split == 0 && blockIdx.y == 0);
  const int own = rp.blocks - rp.shared;
  const int per = (own + rp.own_splits - 1) / rp.own_splits;
  const int begin = rp.shared + min(own, split * per);
  const int count = rp.shared + min(own, (split + 1) * per) - begin;
  const int n_iter = (count + W - 1) / W;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + NS * Cfg::kStageBytes);
  uint64_t* empty = full + NS;
  __shared__ int s_timeout;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], W);
    }
    s_timeout = 0;
    fence_mbarrier_init();
  }
  __syncthreads();

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[KT][4];
#pragma unroll
  for (int i = 0; i < KT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const int gq = lane >> 2, tq = lane & 3;
  int issued = 0;
  if (warp == W) {
    if (!starve) {
      if (lane == 0) {
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
      }
      const int32_t* row = a.bt + int64_t(b) * a.bt_stride + begin;
      const uint64_t policy = l2_policy_evict_first();
      auto load_id = [&](int i) -> int {  // lane j: the block of consumer warp j
        const int blk = i * W + lane;
        if (lane >= W || blk >= count) return 0;
        const int id = __ldg(row + blk);
        if (id >= 0 && id < a.num_blocks) return id;
        flag_status(a.status, kStatusBadBlockId);
        return 0;  // keeps the copy in bounds; the row's result is not meaningful
      };
      int id = n_iter > 0 ? load_id(0) : 0;
      for (int i = 0; i < n_iter; ++i) {
        const int st = i % NS;
        if (i >= NS &&
            !__all_sync(0xffffffffu, mbar_wait(&empty[st], ((i / NS) + 1) & 1, a.status,
                                               a.wait_limit))) {
          s_timeout = 1;
          break;
        }
        const int nb = min(W, count - i * W);
        if (lane == 0) mbar_arrive_expect_tx(&full[st], uint32_t(nb * Cfg::kSlotBytes));
        __syncwarp();
        if (lane < nb) {
          uint8_t* slot = smem + st * Cfg::kStageBytes + lane * Cfg::kSlotBytes;
#pragma unroll
          for (int sb = 0; sb < Cfg::kSub; ++sb) {
            tma_load_4d(slot + sb * Cfg::kSubBytes, &tmap_k, &full[st], sb * 64, g, 0, id, policy);
            tma_load_4d(slot + Cfg::kTileBytes + sb * Cfg::kSubBytes, &tmap_v, &full[st], sb * 64,
                        g, 0, id, policy);
          }
        }
        issued = i + 1;
        if (i + 1 < n_iter) id = load_id(i + 1);
        __syncwarp();
      }
    }
  } else {
    // Q^T as B fragments of S^T = K Q^T: column n = query head h0 + n
    uint32_t qb[KT][2];
    const T* qrow = q + int64_t(b) * a.q_stride + int64_t(h0 + min(gq, heads - 1)) * D;
    const bool words = ((reinterpret_cast<uintptr_t>(q) & 3) | (a.q_stride & 1)) == 0;
    auto pair = [&](int e) -> uint32_t {
      if (gq >= heads) return 0u;
      if (words) return *reinterpret_cast<const uint32_t*>(qrow + e);
      const T two[2] = {qrow[e], qrow[e + 1]};
      uint32_t v;
      memcpy(&v, two, 4);
      return v;
    };
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      qb[kk][0] = pair(16 * kk + 2 * tq);
      qb[kk][1] = pair(16 * kk + 2 * tq + 8);
    }
    for (int i = 0; i < n_iter; ++i) {
      const int st = i % NS;
      const int blk = i * W + warp;
      if (blk < count) {
        if (!__all_sync(0xffffffffu,
                        mbar_wait(&full[st], (i / NS) & 1, a.status, a.wait_limit))) {
          s_timeout = 1;
          break;
        }
        uint8_t* slot = smem + st * Cfg::kStageBytes + warp * Cfg::kSlotBytes;
        const int tok0 = (begin + blk) * kBS;
        if (tok0 + kBS > rp.len) {
          // rows past the sequence hold whatever was there: p = 0 does not undo a NaN
          // or an infinity in V (the last block: nothing is loaded over it again)
          for (int c = lane; c < Cfg::kTileBytes / 16; c += 32)
            if (tok0 + ((c >> 3) & (kBS - 1)) >= rp.len)
              *reinterpret_cast<uint4*>(slot + Cfg::kTileBytes + c * 16) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
        const uint32_t kb[1] = {smem_u32(slot)}, vb[1] = {smem_u32(slot + Cfg::kTileBytes)};
        fold_blocks<T, D, 1>(kb, vb, 1, qb, tok0, kBS, rp.len, scale_log2, m, l, o, lane,
                             Cfg::kSubBytes);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], off);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], off);
    }
  }
  __syncthreads();
  const bool failed = s_timeout != 0;
  if (failed && warp == W && lane == 0) {  // let the copies in flight land
    for (int i = max(0, issued - NS); i < issued; ++i)
      mbar_wait(&full[i % NS], (i / NS) & 1, a.status, a.wait_limit);
  }
  __syncthreads();

  // the warps' results joined in the stages' space: every copy has landed
  float* ro = reinterpret_cast<float*>(smem);        // [W][8][D]
  float* rm = ro + W * Cfg::kHeads * D;              // [W][8]
  float* rl = rm + W * Cfg::kHeads;
  if (warp < W) {
    float* ow = ro + warp * Cfg::kHeads * D;
#pragma unroll
    for (int mt = 0; mt < KT; ++mt) {
      const int d = 16 * mt + gq;
      ow[2 * tq * D + d] = failed ? 0.f : o[mt][0];
      ow[(2 * tq + 1) * D + d] = failed ? 0.f : o[mt][1];
      ow[2 * tq * D + d + 8] = failed ? 0.f : o[mt][2];
      ow[(2 * tq + 1) * D + d + 8] = failed ? 0.f : o[mt][3];
    }
    if (gq == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        rm[warp * Cfg::kHeads + 2 * tq + e] = failed ? -INFINITY : m[e];
        rl[warp * Cfg::kHeads + 2 * tq + e] = failed ? 0.f : l[e];
      }
    }
  }
  __syncthreads();
  float M[W], lw[W];  // this thread's row of the join
  for (int idx = threadIdx.x; idx < heads * D; idx += Cfg::kThreads) {
    const int h = idx / D, d = idx - h * D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, M[w] = rm[w * Cfg::kHeads + h]);
    float acc = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      lw[w] = M[w] == -INFINITY ? 0.f : fast_exp2(M[w] - top);
      if (lw[w] > 0.f) acc += lw[w] * ro[(w * Cfg::kHeads + h) * D + d];
    }
    ro[h * D + d] = acc;  // warp 0's value of this very element: read above by this thread
  }
  __syncthreads();
  if (threadIdx.x < heads) {
    const int h = threadIdx.x;
    float top = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, rm[w * Cfg::kHeads + h]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float x = rm[w * Cfg::kHeads + h];
      if (x != -INFINITY) L += fast_exp2(x - top) * rl[w * Cfg::kHeads + h];
    }
    rm[h] = top;
    rl[h] = L;
  }
  __syncthreads();
  finish_own<T, true, Cfg::kHeads, Cfg::kThreads>(a, rp, out, b, split, h0, heads, ro, D, rm, rl,
                                                  ro + Cfg::kJoinFloats);
  pdl_wait();  // this launch ends after the prefix launch before it
}

template <typename T, int D>
int launch(int prefix_grid, int own_grid, void* out, const void* q, const void* k_cache,
           const void* v_cache, const Args& a, cudaStream_t s) {
  CUtensorMap mk, mv;
  int rc = make_pool_map<T>(&mk, k_cache, a.Kh, D, a.num_blocks);
  if (!rc) rc = make_pool_map<T>(&mv, v_cache, a.Kh, D, a.num_blocks);
  if (rc) return rc;
  const float scale_log2 = a.scale * kLog2e;
  const int starve = take_starve_flag(AS_KERNEL_SHARED_PREFIX) ? 1 : 0;
  if (prefix_grid > 0) {
    using Cfg = PreCfg<D>;
    auto kern = sp_prefix_kernel<T, D>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes + 1024);
    launch_pdl(kern, dim3(prefix_grid, a.Kh), dim3(Cfg::kThreads), Cfg::kSmemBytes + 1024, s, mk,
               mv, static_cast<const T*>(q), a, scale_log2, starve);
    rc = check_launch("as_shared_prefix_decode_attention");
    if (rc) return rc;
  }
  using Cfg = OwnCfg<D>;
  auto kern = sp_own_kernel<T, D>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
  const int chunks = (a.group + Cfg::kHeads - 1) / Cfg::kHeads;
  launch_pdl(kern, dim3(own_grid, a.Kh * chunks), dim3(Cfg::kThreads), Cfg::kSmemBytes, s, mk, mv,
             static_cast<T*>(out), static_cast<const T*>(q), a, scale_log2, starve);
  return check_launch("as_shared_prefix_decode_attention");
}

}  // namespace

int tc_launch(int prefix_grid, int own_grid, void* out, const void* q, const void* k_cache,
              const void* v_cache, const Args& a, int dtype, cudaStream_t s) {
  if (dtype == AS_DTYPE_BF16)
    return a.D == 64
               ? launch<__nv_bfloat16, 64>(prefix_grid, own_grid, out, q, k_cache, v_cache, a, s)
               : launch<__nv_bfloat16, 128>(prefix_grid, own_grid, out, q, k_cache, v_cache, a, s);
  return a.D == 64 ? launch<__half, 64>(prefix_grid, own_grid, out, q, k_cache, v_cache, a, s)
                   : launch<__half, 128>(prefix_grid, own_grid, out, q, k_cache, v_cache, a, s);
}

}  // namespace sp
}  // namespace asb
