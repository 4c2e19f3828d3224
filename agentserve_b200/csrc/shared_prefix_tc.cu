// (9) Shared-prefix decode attention on tensor cores: bf16 / fp16, head_dim 64 or 128.
//
// Prefix launch (sp_prefix_kernel).  A group's members' query heads of KV head g are the
// rows of a matrix that attends over the shared blocks.  A block runs two softmax
// streams of 128 rows, the two halves of a tile of up to 256 rows, which share every
// K / V tile.  S = Q K^T by tcgen05.mma into TMEM, P back into TMEM as the A
// operand of O += P V; K / V arrive by TMA, paged block by paged block.  Roles (320
// threads, one block per SM): warp 0 loads K / V, warp 1 issues MMAs by polling which
// stream is ready, warps 2-5 and 6-9 the streams' softmax, one row per thread, the two
// warps of an SM sub-partition taking turns on its exponent unit.  Bound at head_dim 64 by
// that unit (2,770 cycles for two streams' 128 keys; 2,048 at its peak), at 128 by the tensor
// pipe (60% busy, S at N = 64) and the softmax's chain: 126 GFLOP in 162 us, 778 TFLOP/s.
//
// Own launch (sp_own_kernel).  One sequence, up to 8 query heads of a KV head: too few
// rows for tcgen05, and bound by reading K / V once; the decode kernel's warp-level
// m16n8k16 fold over TMA-staged blocks (decode_tile.cuh).  Its blocks start while the
// prefix launch runs, and join the parts (shared_prefix.cuh) after it.  300 MB of own K / V
// in 59 us, 5.1 TB/s.  The launches alone and cold, and both in a graph, us: 64 sequences on
// 4,096 tokens (head_dim 64) 12.3, 15.4, 19.9; on 14,336 20.9, 22.3, 33.4; 256 on 30,000 (128)
// 162, 59, 192.  Those are with the plan's own grid; full_grid adds blocks without work, which
// come before a later head's and hold their places: 29.8, 42.8 and 211 us in all.
//
// Scores, softmax sums, parts and joins are fp32.  Probabilities are rounded to the pool's type
// for the product with V, as the matrix instructions take them: by at most 2^-8 (bf16) or 2^-11
// (fp16) of each, and in fp16 by 2^-25 of a part's largest where they are smaller than 2^-14 of
// it.  The sums l take them unrounded.  Against 64 bits the output's error is 1.15 to 1.4 times
// (rms) that of a result rounded once.
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
  static constexpr int kBN = D == 64 ? 128 : 64;  // keys per tile
  static constexpr int kBlocks = kBN / kBS;
  static constexpr int kSub = D / 64;             // 128-byte-wide swizzle sub-tiles
  static constexpr int kQSub = 128 * 128;
  static constexpr int kKVSub = kBN * 128;
  static constexpr int kQBytes = kSub * kQSub;    // 128 rows
  static constexpr int kKVBytes = kSub * kKVSub;  // K (or V) of one tile
  static constexpr int kStages = 4;
  static constexpr int kOffKV = 2 * kQBytes;
  static constexpr int kOffBar = kOffKV + kStages * 2 * kKVBytes;
  static constexpr int kSmemBytes = kOffBar + 256;
  static constexpr int kThreads = 320;
  // TMEM columns of a stream, from 256 i: S, P (16-bit pairs), O the last D.  At D = 128
  // two S of 64 keys take turns, so that the next one is ready when a softmax ends, and P
  // overwrites the S it came from, by then in registers.  (Before that one S of 128 keys
  // under its P, the next issued after PV: 256 sequences on 30,000 tokens 227 us, then 209.)
  static constexpr int kCols = 512;
  static constexpr bool kAliasP = D == 128;
  static constexpr int kColP = kAliasP ? 0 : kBN;
  static constexpr int kColO = 256 - D;
  static_assert(kSmemBytes + 1024 <= 227 * 1024, "shared memory");
};

struct PreBars {
  uint64_t kv_full[4], kv_empty[4];
  uint64_t s_full[2][2], s_free[2], p_full[2], pv_done[2];  // [stream], S's place
  uint64_t turn[2][4];  // hand-off of the exponent unit between a sub-partition's warps
  uint64_t drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(PreBars) <= 256, "barrier block");

__device__ __forceinline__ bool stopped(volatile int* flag) { return *flag != 0; }

template <typename T, int HD>
__global__ void __launch_bounds__(320, 1)
sp_prefix_kernel(const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const T* __restrict__ q,
                 const Args a, float scale_log2, int starve) {
  using Cfg = PreCfg<HD>;
  constexpr int D = Cfg::D, BN = Cfg::kBN, NS = Cfg::kStages, NB = Cfg::kBlocks;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescS = tc::idesc_f16(kBF16, 128, BN, false, false);
  constexpr uint32_t kIdescO = tc::idesc_f16(kBF16, 128, D, false, true);

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  PreBars* bars = reinterpret_cast<PreBars*>(smem + Cfg::kOffBar);
  volatile int* abort_flag = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_wait();
  pdl_trigger();  // every block of this launch has started: the own launch may start
  const PrefixItem it = load_item(a.prefix_items, blockIdx.x);
  if (it.rows == 0) return;
  if (it.end > a.max_blocks) {  // of a group that row_plan() attends alone: not in the table
    if (threadIdx.x == 0) flag_status(a.status, kStatusBadLength);
    return;
  }
  const int g = blockIdx.y, group = a.group;
  const int n_tiles = (it.end - it.begin + NB - 1) / NB;
  // streams: rows and key tiles of each
  const int rows0 = min(it.rows, 128), rows1 = it.rows - rows0;
  const int n0 = n_tiles, n1 = rows1 > 0 ? n_tiles : 0;
  const int active0 = (rows0 + 31) / 32, active1 = (rows1 + 31) / 32;  // warps with rows

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars->kv_full[s], 1);
      mbar_init(&bars->kv_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      const int n = max(1, i ? active1 : active0);
      mbar_init(&bars->s_full[i][0], 1);
      mbar_init(&bars->s_full[i][1], 1);
      mbar_init(&bars->s_free[i], n);
      mbar_init(&bars->p_full[i], n);
      mbar_init(&bars->pv_done[i], 1);
      for (int w = 0; w < 4; ++w) mbar_init(&bars->turn[i][w], 1);
    }
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_mbarrier_init();
  }
  __syncthreads();  // the barriers are initialised

  int issued = 0;
  if (warp == 0) {
    // ------------------------------------------------- K / V loads, from now on
    if (!starve) {
      if (lane == 0) {
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
      }
      const int32_t* row = a.bt + int64_t(it.table_row) * a.bt_stride;
      // 32 block ids at a time, one per lane, read ahead of their use.  Blocks past the
      // range: its last one (finite as the rest), masked below; an id outside the pool is
      // flagged and block 0 read in its place.
      const auto load_ids = [&](int j) -> int {
        const int id = __ldg(row + min(it.begin + NB * j + lane, it.end - 1));
        if (id >= 0 && id < a.num_blocks) return id;
        flag_status(a.status, kStatusBadBlockId);
        return 0;
      };
      constexpr int kPer = 32 / NB;  // tiles per read
      const uint64_t policy = l2_policy_evict_last();  // other row tiles read them too
      int ids = load_ids(0), next = n_tiles > kPer ? load_ids(kPer) : 0;
      for (int j = 0; j < n_tiles; ++j) {
        const int st = j % NS;
        const bool ready =
            !stopped(abort_flag) &&
            (j < NS || mbar_wait(&bars->kv_empty[st], ((j / NS) + 1) & 1, a.status, a.wait_limit));
        if (!__all_sync(0xffffffffu, ready)) {
          *abort_flag = 1;
          break;
        }
        if (j > 0 && j % kPer == 0) {
          ids = next;
          if (j + kPer < n_tiles) next = load_ids(j + kPer);
        }
        const int id = __shfl_sync(0xffffffffu, ids, (j % kPer) * NB + (lane & (NB - 1)));
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
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    tc::tmem_alloc(&bars->tmem, Cfg::kCols);
    tc::tmem_relinquish();
  } else if (warp >= 2) {
    // Q rows (member, head) into the 128B-swizzled layout, a thread per row, all
    // copies in flight at once; rows past a tile are zero
    const int r = threadIdx.x - 64;
    uint8_t* dst = smem + (r >> 7) * Cfg::kQBytes + (r & 127) * 128;
    const auto chunk = [&](int c) -> uint8_t* {
      return dst + (c >> 3) * Cfg::kQSub + (((c & 7) ^ (r & 7)) << 4);
    };
    if (r < it.rows) {
      const int rr = it.row0 + r;
      const T* src = q + int64_t(__ldg(a.members + it.members + rr / group)) * a.q_stride +
                     int64_t(g * group + rr % group) * D;
      if (((reinterpret_cast<uintptr_t>(q) | uintptr_t(a.q_stride * 2)) & 15) == 0) {
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) cp_async_16(smem_u32(chunk(c)), src + c * 8);
        asm volatile("cp.async.wait_all;" ::: "memory");
      } else {
        for (int c = 0; c < D / 8; ++c) {
          T e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = src[c * 8 + j];
          memcpy(chunk(c), e, 16);
        }
      }
    } else {
      for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(chunk(c)) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  uint32_t tmem = 0;
  if (warp > 0) {  // Q and the TMEM address are there; the loads go on beside this
    tc::fence_before_sync();
    asm volatile("bar.sync 1, %0;" ::"n"(Cfg::kThreads - 32) : "memory");
    tc::fence_after_sync();
    tmem = bars->tmem;
  }
  const uint32_t sQ = smem_u32(smem), sKV = smem_u32(smem + Cfg::kOffKV);

  if (warp == 1) {
    // ----------------------------------------------------------------- MMAs
    // An MMA costs this thread 20 cycles; under a branch on lane == 0 it cost 77, and the
    // issue bound the launch (256 sequences on 30,000 tokens 243 us, by this alone 227).
    if (tc::elect_one()) {
      auto issue_s = [&](int i, int st, int place) {
        const uint32_t qi = sQ + i * Cfg::kQBytes;
        const uint32_t k = sKV + st * 2 * Cfg::kKVBytes;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_f16(tmem + 256 * i + place * BN,
                      tc::sdesc_sw128(qi + (kk >> 2) * Cfg::kQSub + (kk & 3) * 32, 16, 1024),
                      tc::sdesc_sw128(k + (kk >> 2) * Cfg::kKVSub + (kk & 3) * 32, 16, 1024),
                      kIdescS, kk > 0 ? 1u : 0u);
      };
      auto issue_pv = [&](int i, int st, int place, bool acc) {
        const uint32_t v = sKV + st * 2 * Cfg::kKVBytes + Cfg::kKVBytes;
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          tc::mma_f16_ts(tmem + 256 * i + Cfg::kColO, tmem + 256 * i + Cfg::kColP + place * BN + kk * 8,
                         tc::sdesc_sw128(v + kk * 2048, Cfg::kKVSub, 1024), kIdescO,
                         (acc || kk > 0) ? 1u : 0u);
      };
      const int nk[2] = {n0, n1};
      int js[2] = {0, 0}, jp[2] = {0, 0};  // next S and next PV of each stream
      bool ok = true;
      uint64_t t_idle = 0;
      uint32_t spin = 0;
      while (jp[0] < nk[0] || jp[1] < nk[1]) {
        if (stopped(abort_flag)) break;
        bool did = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = js[i];
          const int place = Cfg::kAliasP ? j & 1 : 0;
          if (j < nk[i] && mbar_test_wait(&bars->kv_full[j % NS], (j / NS) & 1) &&
              (Cfg::kAliasP ? jp[i] >= j - 1  // PV(j - 2), which reads P there, is issued
                            : j == 0 || mbar_test_wait(&bars->s_free[i], (j - 1) & 1))) {
            tc::fence_after_sync();
            issue_s(i, j % NS, place);
            tc::commit(&bars->s_full[i][place]);
            js[i] = j + 1;
            did = true;
          }
          const int jq = jp[i];
          if (jq < js[i] && mbar_test_wait(&bars->p_full[i], jq & 1)) {
            tc::fence_after_sync();
            issue_pv(i, jq % NS, Cfg::kAliasP ? jq & 1 : 0, jq > 0);
            tc::commit(&bars->pv_done[i]);
            jp[i] = jq + 1;
            did = true;
            // a stage is free once every stream that reads it has issued its PV
            if (jp[1 - i] > jq || jq >= nk[1 - i]) tc::commit(&bars->kv_empty[jq % NS]);
          }
        }
        if (did) {
          spin = 0;
        } else if ((++spin & 255u) == 0u) {  // the timer is slow to read: rarely
          const uint64_t now = global_timer_ns();
          if (spin == 256u) {
            t_idle = now;
          } else if (now - t_idle > a.wait_limit) {
            flag_status(a.status, kStatusWaitTimeout);
            ok = false;
            break;
          }
        }
      }
      if (!ok) *abort_flag = 1;
      tc::commit(&bars->drain);
      mbar_wait(&bars->drain, 0, a.status, a.wait_limit);
    }
    __syncwarp();
  } else if (warp > 1) {
    // -------------------------------------------------------------- softmax
    const int i = (warp - 2) >> 2;  // stream
    const int quad = warp & 3;      // the TMEM lanes this warp may access
    const int r = quad * 32 + lane;
    const int my_rows = i ? rows1 : rows0, n = i ? n1 : n0;
    if (quad < (i ? active1 : active0)) {
      const uint32_t row = tmem + 256 * i + (uint32_t(quad * 32) << 16);
      const uint32_t tO = row + Cfg::kColO;
      const bool partner = quad < (i ? active0 : active1);
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        const int place = Cfg::kAliasP ? j & 1 : 0;
        const uint32_t tS = row + place * BN, tP = tS + Cfg::kColP;
        const bool go = !stopped(abort_flag) &&
                        mbar_wait(&bars->s_full[i][place], (Cfg::kAliasP ? j >> 1 : j) & 1,
                                  a.status, a.wait_limit);
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
        if (!Cfg::kAliasP) {
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->s_free[i]);
        }
        const int keys = (it.end - it.begin) * kBS - j * BN;  // of this tile
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
        // lazy maximum: exponentials stay below 2^8, within every type's range, unless a
        // score exceeds the current one by more; then O and l are rescaled
        float alpha = 1.f;
        if (mx * scale_log2 > m + kLazySlack) {
          const float m_new = mx * scale_log2;
          alpha = fast_exp2(m - m_new);
          m = m_new;
        }
        const float neg_m = m == -INFINITY ? 0.f : -m;
        // a warp waits only for a hand-off that its partner will make
        if (partner && (i == 1 || j > 0)) {
          const bool mine = !stopped(abort_flag) &&
                            mbar_wait(&bars->turn[i][quad], (i == 0 ? j - 1 : j) & 1, a.status,
                                      a.wait_limit);
          if (!__all_sync(0xffffffffu, mine)) {
            ok = false;
            break;
          }
        }
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
          pk[c] = pack2<T>(p0, p1);  // rounded for the product with V: see the top
          if (c == BN / 4 - 1) {  // half-way: the partner's start overlaps the rest
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->turn[1 - i][quad]);
          }
        }
        float s0, s1;
        f2_unpack(f2_add(f2_add(sum2[0], sum2[1]), f2_add(sum2[2], sum2[3])), s0, s1);
        if (j > 0) {  // the product with V of the last tile still reads P and writes O
          if (!__all_sync(0xffffffffu,
                          mbar_wait(&bars->pv_done[i], (j - 1) & 1, a.status, a.wait_limit))) {
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
        if (lane == 0) mbar_arrive(&bars->p_full[i]);
      }
      if (!ok) *abort_flag = 1;
      const bool done =
          ok && n > 0 && __all_sync(0xffffffffu, mbar_wait(&bars->pv_done[i], (n - 1) & 1,
                                                           a.status, a.wait_limit));
      if (ok && n > 0 && !done) *abort_flag = 1;
      const int rr = it.row0 + 128 * i + r;
      const int part = it.part + rr / group;
      const size_t at = size_t(part) * a.H + g * group + rr % group;
      if (done) {
        // A row per thread in TMEM.  Of many rows, O goes by way of this warp's part of Q,
        // which no MMA of the stream reads any more, to global memory in whole lines: 64
        // sequences (256 rows) on 4,096 tokens 19.8 us, straight from the threads 20.6.  Of
        // few rows straight: 4 (16 rows) on 160 8.1 us, by way of Q 8.6; 16 (64 rows) on
        // 8,000 17.4 and 17.8; 32 (128 rows) on 14,336 22.6 and 22.2.
        const bool lines = it.rows > 64;
        tc::fence_after_sync();
        uint8_t* mine = smem + i * Cfg::kQBytes + quad * 4096;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tc::ld_32x32b_x32(tO + c * 32, o);
          tc::wait_ld();
          if (!lines) {
            if (r < my_rows) {
              uint4* dst = reinterpret_cast<uint4*>(a.parts.o + at * D + c * 32);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
            continue;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(mine + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int row = 4 * k + (lane >> 3), e = lane & 7;
            const size_t to = __shfl_sync(0xffffffffu, static_cast<unsigned long long>(at), row);
            if (quad * 32 + row < my_rows)
              *reinterpret_cast<uint4*>(a.parts.o + to * D + c * 32 + e * 4) =
                  *reinterpret_cast<const uint4*>(mine + row * 128 + ((e ^ (row & 7)) << 4));
          }
          __syncwarp();
        }
      }
      if (r < my_rows) a.parts.ml[at] = done ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
    }
    tc::fence_before_sync();
  }

  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, Cfg::kCols);
  }
  if (warp == 0 && lane == 0 && stopped(abort_flag)) {  // let the copies in flight land
    for (int j = max(0, issued - NS); j < issued; ++j)
      mbar_wait(&bars->kv_full[j % NS], (j / NS) & 1, a.status, a.wait_limit);
  }
}

// ===========================================================================
// Own blocks
// ===========================================================================
template <int D>
struct OwnCfg {
  // Consumers; one more warp loads.  At D = 128 three and one stage, so that a block fits
  // beside one of the prefix launch (256 sequences on 30,000 tokens, with four and two 209 us,
  // then 201).
  static constexpr int kWarps = D == 64 ? 4 : 3;
  static constexpr int kThreads = (kWarps + 1) * 32;
  static constexpr int kSub = D / 64;
  static constexpr int kSubBytes = kBS * 128;
  static constexpr int kTileBytes = kSub * kSubBytes;  // one block of K or V, one head
  static constexpr int kSlotBytes = 2 * kTileBytes;
  static constexpr int kStageBytes = kWarps * kSlotBytes;  // a block per consumer warp
  static constexpr int kStages = D == 64 ? 3 : 1;
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
  const OwnItem it = load_item(a.own_items, blockIdx.x);
  if (it.own_splits == 0) {
    pdl_wait();
    return;
  }
  const int b = it.row, split = it.split;
  const int chunks = (a.group + Cfg::kHeads - 1) / Cfg::kHeads;
  const int g = blockIdx.y / chunks, chunk = blockIdx.y - g * chunks;
  const int h0 = g * a.group + chunk * Cfg::kHeads;
  const int heads = min(Cfg::kHeads, a.group - chunk * Cfg::kHeads);
  const RowPlan rp = row_plan(a, it, threadIdx.x == 0 && split == 0 && blockIdx.y == 0);
  const int begin = rp.begin, count = rp.count;
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
        // Only after its own wait for the stage: a warp that runs ahead would else be counted
        // for a round that slower ones still read.  (A warp without a block is in the last
        // round, after which nothing is loaded.)
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
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

  // the warps' results in the stages' space: every copy has landed
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
  finish_own<T, true, Cfg::kHeads, Cfg::kThreads, W>(a, rp, out, b, split, h0, heads, ro, D, rm,
                                                     rl, ro + Cfg::kJoinFloats);
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
