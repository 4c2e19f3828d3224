// (8) Sampling with temperature, top-k, top-p and min-p from given uniform numbers
// (agentserve/engine/sampling.py's sampled branch: temperature, then top-k, then top-p;
// min-p is an addition), one token per row of logits.
//
// With x = nan_to_num(logit, 0, 1e4, -1e4) in fp32, m = max x and w = exp((x - m) / T),
// order the tokens by (x descending, index ascending).  The kept tokens are the first
// n = max(1, min(n_k, n_p, n_m)) of that order: n_k = top_k, n_p the least n whose
// weights sum to at least p times those of the first n_k, n_m the number with
// w >= min_p.  The row's token is the first kept one, in index order, at which the
// running sum of kept weights exceeds u times their total.
//
// No sort: every filter keeps a prefix of one order, so a cut (a value, and how many of
// the tokens equal to it) describes it.  A cut is found by histograms over the distance
// from the maximum: 1024 bins over 12 nats, then 1024 in the chosen bin, then (rarely)
// over the values' bits, until one value is left.
//
// Sums decide between neighbouring tokens, and a border token can weigh 1e-6 of the
// total: weights are computed in 64 bits and summed in fixed point (2^-45 at 128K
// tokens), which makes every sum exact and independent of the order of the atomics.
//
// A row is worked on by a cluster of 1 to 8 CTAs, each holding a run of indexes, its warps
// runs of that; they exchange totals over distributed shared memory.  Every decision
// follows from exchanged values, so all CTAs of a cluster take the same barriers.
#include <string.h>

#include <type_traits>

#include "common.cuh"
#include "host_util.h"

namespace asb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBinBits = 10;
constexpr int kBins = 1 << kBinBits;
constexpr float kWindow = 12.f;  // nats covered by the first histogram
constexpr int kTable = 512;      // 2^(i / 512)
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxRun = 1 << 17;  // tokens of a CTA
// A weight is at most 1 = 2^43 units: the sum of kMaxVocab of them fits 64 bits, and its
// three pieces of 15 bits, summed over a CTA's tokens, fit 32 bits each.
constexpr int kFrac = 43;
constexpr int kPiece = 15;
typedef unsigned long long u64;

__device__ __forceinline__ float sanitize(float v) {
  if (v != v) return 0.f;
  if (v == INFINITY) return 1e4f;
  if (v == -INFINITY) return -1e4f;
  return v;
}
// Order-preserving bits of an fp32 value; -0 as +0.
__device__ __forceinline__ uint32_t ord_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// ---- the cluster's shared memory -------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t peer_addr_of(const void* p, uint32_t rank) {
  return peer_addr(smem_u32(p), rank);
}
__device__ __forceinline__ uint32_t peer_load(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void peer_store64(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void cluster_sync(int C) {
  if (C == 1) {
    __syncthreads();
  } else {
    __syncwarp();  // the aligned form takes whole warps
    asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

struct Slot {
  u64 a, b, c;
};
struct Shared {
  double table[kTable];          // 2^(i / 512) in units of the fixed point
  uint32_t hist[3][kBins];       // pieces of the summed measure
  uint32_t kmin[kBins], kmax[kBins];
  Slot slot[2][kMaxCluster];     // exchanges, in turn
  u64 warp[kWarps];
  u64 warp2[kWarps];
  Slot found, found2;
  int holds;  // the chosen token is in this CTA's run
};

// bf16 rows: a histogram by value.  The 4096 values of magnitude 2^-9 to 128 have a
// bin each, in descending order; the few closer to zero are listed; those at or below
// -128 (masks) weigh nothing next to any maximum this path accepts.  The first pass then
// needs no maximum and no exponential, both cuts come from one merge, and the second
// pass looks the weights up.  Rows outside this (values of 128 and more, NaN, cuts among
// the listed values, u <= 0) take the general path.
constexpr int kValueLo = (127 - 9) << 7;  // bits of 2^-9
constexpr int kValues = 16 << 7;          // values of one sign
constexpr int kListed = 2048;
struct ByValue {
  u64 weight[2 * kValues];
  uint32_t count[2 * kValues];
  uint16_t list[kListed];
  uint32_t n_listed, refuse;
  u64 positive[2];  // (C = 1) count and weight of the positive bins
};
__device__ __forceinline__ int value_bin(uint32_t code) {  // of a magnitude within range
  return int(((code & 0x7fff) - kValueLo) ^ ((code & 0x8000) ? kValues : kValues - 1));
}
__device__ __forceinline__ float bin_value(int bin) {
  const uint32_t code = bin < kValues ? uint32_t(kValueLo + kValues - 1 - bin)
                                      : 0x8000u | uint32_t(kValueLo + bin - kValues);
  return __uint_as_float(code << 16);
}

struct Params {
  int64_t* out;
  float* logprobs;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t row_stride;
  int V, C, chunk;      // tokens, CTAs of a cluster, tokens of a CTA
};

// One CTA's view of its row.
template <typename T>
struct Row {
  Shared& s;
  const T* row;
  int C, rank, turn;  // turn: which slot buffer the next exchange uses
  int i0, i1;         // this warp's run of indexes
  bool vec;           // rows from 16-byte boundaries
  bool special;       // the row holds NaN or infinities
  float m;
  // weights
  double c, md;       // log2(e) / T, m
  const u64* by_value;  // weights by value (bf16), or null
  // distances from the maximum in units of a second-level bin
  float dscale;

  // f(x, index of x[0]) for this warp's tokens, 32 lanes x 16 bytes at a time; places past
  // the run hold -infinity, which no token is
  static constexpr int VEC = 16 / int(sizeof(T));
  template <typename F>
  __device__ __forceinline__ void visit(F f) const {
    const int lane = threadIdx.x & 31;
    for (int base = i0; base < i1; base += 32 * VEC) {  // the same trips for every lane
      const int i = base + lane * VEC;
      float x[VEC];
      if (vec && base + 32 * VEC <= i1) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + i));
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = Elem<T>::to_f32(e[j]);
        if (special) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[j] = sanitize(x[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          x[j] = i + j < i1 ? sanitize(Elem<T>::to_f32(row[i + j])) : -INFINITY;
      }
      f(x, i);
    }
  }

  // w in fixed point: 2^y, y = (x - m) log2(e) / T, as 2^(j / 512) from the table times
  // a cubic in the rest (|rest| <= 1/1024: relative error below 1e-14).  Adding 1.5 *
  // 2^43 rounds y to 512ths; adding 2^52 to the product rounds it to a whole number.
  __device__ __forceinline__ u64 fixed(float x) const {
    const uint32_t b = __float_as_uint(x);
    // fp32 to fp64 on the integer units (zeros and denormals become values below 1e-38)
    const double xd = __hiloint2double(int((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)),
                                       int(b << 29));
    const double d = xd - md;
    const double kRound = 6755399441055744.0 / 512.0;  // 1.5 * 2^52 / 512
    const double t = fma(d, c, kRound);
    const int j = __double2loint(t);
    const double whole = t - kRound;
    const double f = fma(d, c, -whole);
    double p = fma(f, 0.05550410866482158, 0.24022650695910072);  // ln2^3 / 6, ln2^2 / 2
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    const double tab = s.table[j & (kTable - 1)];
    const double scaled = __hiloint2double(__double2hiint(tab) + ((j >> 9) << 20), __double2loint(tab));
    const double v = fma(scaled, p, 4503599627370496.0);  // 2^52
    const u64 bits = u64(__double_as_longlong(v)) & 0xFFFFFFFFFFFFFull;
    return whole > -60.0 ? bits : 0ull;  // below half a unit (and out of the exponent's range)
  }
  // Four weights at a time, 0 where a test fails; nothing is computed where no lane's
  // passes, and else all four side by side: the chain of one is long.
  template <typename P, typename F>
  __device__ __forceinline__ void weigh(const float (&x)[VEC], P test, F f) const {
#pragma unroll
    for (int h = 0; h < VEC; h += 4) {
      bool ok[4], any = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) any |= ok[j] = test(x[h + j]);
      if (!__any_sync(0xffffffffu, any)) continue;
      u64 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fixed(x[h + j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) f(x[h + j], h + j, ok[j] ? v[j] : 0ull);
    }
  }
  // The weight of a token, looked up where the row has a table.
  __device__ __forceinline__ u64 weight(float x) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      if (by_value) {
        const uint32_t code = __float_as_uint(x) >> 16;
        if ((code & 0x7fff) - uint32_t(kValueLo) < uint32_t(kValues))
          return by_value[value_bin(code)];
      }
    }
    return fixed(x);
  }
  // f(index in x, weight) for the tokens above the cut.  Few are (or the weights are
  // looked up): one place at a time, where any lane's is.  All are: four side by side.
  template <typename F>
  __device__ __forceinline__ void above(const float (&x)[VEC], float cut, F f) const {
    if (cut == -INFINITY && !by_value) {
      weigh(x, [&](float v) { return v > cut; }, [&](float, int j, u64 v) { f(j, v); });
      return;
    }
    bool any = false;
#pragma unroll
    for (int j = 0; j < VEC; ++j) any |= x[j] > cut;
    if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (x[j] > cut) f(j, weight(x[j]));
  }
  // Distance from the maximum in second-level bins, -1 outside the window.
  __device__ __forceinline__ int dist(float x) const {
    const float d = (m - x) * dscale;
    return d < float(1 << (2 * kBinBits)) ? int(d) : -1;
  }

  // Slot `v` of every CTA, at every CTA.  One barrier; two buffers in turn, so a slot is
  // rewritten only after a barrier that follows its last reads.
  __device__ __forceinline__ const Slot* exchange(const Slot& v) {
    Slot* buf = s.slot[turn];
    turn ^= 1;
    if (threadIdx.x < C) {
      const uint32_t at = peer_addr_of(&buf[rank], threadIdx.x);
      peer_store64(at, v.a);
      peer_store64(at + 8, v.b);
      peer_store64(at + 16, v.c);
    }
    cluster_sync(C);
    return buf;
  }

  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.hist[0][i] = s.hist[1][i] = s.hist[2][i] = 0;
      s.kmin[i] = 0xffffffffu;
      s.kmax[i] = 0;
    }
    __syncthreads();
  }
  template <bool kCount>
  __device__ __forceinline__ void add(int bin, u64 v) {
    if (kCount) {
      atomicAdd(&s.hist[0][bin], uint32_t(v));
    } else {
      constexpr uint32_t mask = (1u << kPiece) - 1;
      atomicAdd(&s.hist[0][bin], uint32_t(v) & mask);
      atomicAdd(&s.hist[1][bin], uint32_t(v >> kPiece) & mask);
      const uint32_t top = uint32_t(v >> (2 * kPiece));
      if (top) atomicAdd(&s.hist[2][bin], top);
    }
  }

  struct Found {
    int bin;        // -1: the target lies beyond the histogram
    u64 before;     // sum above the bin (or of the whole histogram)
    uint32_t lo, hi;  // least and largest key in it, where those were kept
  };
  // Sums the cluster's histograms and finds the first bin at which acc + the running sum
  // reaches the target.  The histograms may be cleared afterwards.
  template <bool kCount>
  __device__ Found find(u64 acc, u64 target, bool keys) {
    cluster_sync(C);  // every CTA's histogram is complete
    const int S = kBins / C;  // bins of this CTA's slice
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    // thread t: bins [t * per, (t + 1) * per) of the slice
    const int per = S > kThreads ? S / kThreads : 1;  // 1 or 2
    u64 v[2] = {0, 0};
    if (C == 1) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int bin = 2 * t + e;
        v[e] = s.hist[0][bin];
        if (!kCount)
          v[e] += (u64(s.hist[1][bin]) << kPiece) + (u64(s.hist[2][bin]) << (2 * kPiece));
      }
    } else if (t < S) {
      const uint32_t at = smem_u32(&s.hist[0][rank * S + t]);
      uint32_t h[kMaxCluster][kCount ? 1 : 3];
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {  // all loads in flight
        const uint32_t from = peer_addr(at, q < C ? q : 0);
#pragma unroll
        for (int e = 0; e < (kCount ? 1 : 3); ++e) h[q][e] = peer_load(from + 4 * kBins * e);
      }
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {
        if (q < C) {
          v[0] += h[q][0];
          if (!kCount) v[0] += (u64(h[q][kCount ? 0 : 1]) << kPiece) + (u64(h[q][kCount ? 0 : 2]) << (2 * kPiece));
        }
      }
    }
    // running sums of the slice
    u64 inc = v[0] + v[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    if (lane == 31) s.warp[warp] = inc;
    __syncthreads();
    u64 base = 0, slice = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += s.warp[w];
      slice += s.warp[w];
    }
    const u64 e0 = base + inc - v[0] - v[1];  // of the slice, before this thread's bins
    const Slot* all = exchange(Slot{slice, 0, 0});
    u64 start = acc, whole = acc;
    for (int q = 0; q < C; ++q) {
      if (q < rank) start += all[q].a;
      whole += all[q].a;
    }
    if (whole < target) return Found{-1, whole, 0, 0};
    // the thread whose bin it is tells every CTA
    const u64 b0 = start + e0, b1 = b0 + v[0], b2 = b1 + v[1];
    if (b0 < target && b2 >= target) {
      const int e = b1 >= target ? 0 : 1;
      const int bin = rank * S + t * per + e;
      uint32_t lo = 0xffffffffu, hi = 0;
      if (keys) {
        for (int q = 0; q < C; ++q) {
          lo = min(lo, peer_load(peer_addr_of(&s.kmin[bin], q)));
          hi = max(hi, peer_load(peer_addr_of(&s.kmax[bin], q)));
        }
      }
      for (int q = 0; q < C; ++q) {
        const uint32_t at = peer_addr_of(&s.found, q);
        peer_store64(at, u64(bin));
        peer_store64(at + 8, e ? b1 : b0);
        peer_store64(at + 16, (u64(hi) << 32) | lo);
      }
    }
    cluster_sync(C);
    const Found f{int(s.found.a), s.found.b, uint32_t(s.found.c), uint32_t(s.found.c >> 32)};
    __syncthreads();  // read by all before it is written again
    return f;
  }

  // First pass of a bf16 row: counts by value, and the maximum.
  __device__ __forceinline__ void count_values(ByValue& bv, float& mx) {
    const int lane = threadIdx.x & 31;
    const auto one = [&](uint32_t code) {
      const uint32_t d = (code & 0x7fff) - uint32_t(kValueLo);
      if (d < uint32_t(kValues)) {
        atomicAdd(&bv.count[d ^ ((code & 0x8000) ? kValues : kValues - 1)], 1u);
      } else if (int(d) < 0) {
        const uint32_t at = atomicAdd(&bv.n_listed, 1u);
        if (at < kListed)
          bv.list[at] = uint16_t(code);
        else
          bv.refuse = 1;
      } else if (code < 0x8000 || code > 0xff80) {
        bv.refuse = 1;
      }
    };
    __nv_bfloat162 top = __float2bfloat162_rn(-INFINITY);
    for (int base = i0; base < i1; base += 32 * VEC) {
      const int i = base + lane * VEC;
      if (vec && base + 32 * VEC <= i1) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + i));
        const uint32_t wd[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          __nv_bfloat162 v;
          memcpy(&v, &wd[j], 4);
          top = __hmax2(top, v);
          one(wd[j] & 0xffff);
          one(wd[j] >> 16);
        }
      } else {
        for (int j = 0; j < VEC && i + j < i1; ++j) {
          const __nv_bfloat16 v = *reinterpret_cast<const __nv_bfloat16*>(row + i + j);
          top = __hmax2(top, __nv_bfloat162(v, v));
          one(__bfloat16_as_ushort(v));
        }
      }
    }
    mx = fmaxf(__bfloat162float(top.x), __bfloat162float(top.y));
  }

  // Both cuts of a bf16 row from the cluster's counts by value.  False: a cut lies among
  // the listed values.
  __device__ bool value_cuts(ByValue& bv, int k, float tp, float& cut, u64& ties) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    constexpr int kAll = 2 * kValues;
    for (int i = t; i < kAll; i += kThreads) bv.weight[i] = fixed(bin_value(i));
    u64 listed = 0;
    for (int i = t; i < int(bv.n_listed); i += kThreads)
      listed += fixed(__uint_as_float(uint32_t(bv.list[i]) << 16));
    by_value = bv.weight;
    // thread t: bins [rank * S + t * per, + per) summed over the cluster
    const int S = kAll / C, per = S / kThreads;  // 8, 4, 2 or 1
    const int first = rank * S + t * per;
    uint32_t n[kAll / kThreads];
#pragma unroll
    for (int e = 0; e < kAll / kThreads; ++e) n[e] = 0;
    if (C == 1) {
#pragma unroll
      for (int e = 0; e < kAll / kThreads; ++e) n[e] = bv.count[first + e];
    } else {
      const uint32_t at = smem_u32(&bv.count[first]);
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {
        const uint32_t from = peer_addr(at, q < C ? q : 0);
#pragma unroll
        for (int e = 0; e < kAll / kThreads / 2; ++e) {
          if (e < per && q < C) n[e] += peer_load(from + 4 * e);
        }
      }
    }
    __syncthreads();  // the weights are there
    u64 mass = 0, num = 0;
#pragma unroll
    for (int e = 0; e < kAll / kThreads; ++e) {
      if (n[e]) mass += n[e] * bv.weight[first + e];
      num += n[e];
    }
    u64 m_inc = mass, n_inc = num;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 a = __shfl_up_sync(0xffffffffu, m_inc, o);
      const uint32_t b = __shfl_up_sync(0xffffffffu, uint32_t(n_inc), o);
      if (lane >= o) {
        m_inc += a;
        n_inc += b;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) listed += __shfl_xor_sync(0xffffffffu, listed, o);
    if (lane == 31) {
      s.warp[warp] = m_inc;
      s.warp2[warp] = n_inc;
    }
    if (lane == 0) s.hist[0][warp] = uint32_t(listed), s.hist[1][warp] = uint32_t(listed >> 32);
    __syncthreads();
    u64 m_before = 0, n_before = 0, m_slice = 0, n_slice = 0;
    listed = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) {
        m_before += s.warp[i];
        n_before += s.warp2[i];
      }
      m_slice += s.warp[i];
      n_slice += s.warp2[i];
      listed += (u64(s.hist[1][i]) << 32) | s.hist[0][i];
    }
    m_before += m_inc - mass;
    n_before += n_inc - num;
    if (C == 1 && t == kThreads / 2) {  // the first thread of the negative values
      bv.positive[0] = n_before;
      bv.positive[1] = m_before;
    }
    const Slot* all = exchange(Slot{m_slice, (n_slice << 32) | bv.n_listed, listed});
    // running sums before this thread's bins; the listed values lie between the signs
    u64 m_pos = 0, n_pos = 0, m_list = 0, n_list = 0, m_all = 0, n_all = 0;
    for (int q = 0; q < C; ++q) {
      if (q < rank) {
        m_before += all[q].a;
        n_before += all[q].b >> 32;
      }
      if (2 * q < C) {
        m_pos += all[q].a;
        n_pos += all[q].b >> 32;
      }
      m_all += all[q].a;
      n_all += all[q].b >> 32;
      m_list += all[q].c;
      n_list += all[q].b & 0xffffffffull;
    }
    if (C == 1) {
      n_pos = bv.positive[0];
      m_pos = bv.positive[1];
    }
    m_all += m_list;
    n_all += n_list;
    if (first >= kValues) {
      m_before += m_list;
      n_before += n_list;
    }
    // The first bin at which the running count (or weight) reaches the target; the thread
    // whose it is tells every CTA the sums before it.
    // (One place per call: no barrier parts a CTA's read of the first from a peer's
    // write of the second.)
    const auto locate = [&](bool count, u64 target, Slot& place) -> Slot {
      u64 a = m_before, b = n_before;
#pragma unroll
      for (int e = 0; e < kAll / kThreads; ++e) {
        const u64 da = n[e] ? n[e] * bv.weight[first + e] : 0;
        const u64 run = count ? b : a, step = count ? n[e] : da;
        if (run < target && run + step >= target) {
          for (int q = 0; q < C; ++q) {
            const uint32_t at = peer_addr_of(&place, q);
            peer_store64(at, u64(first + e));
            peer_store64(at + 8, a);
            peer_store64(at + 16, b);
          }
        }
        a += da;
        b += n[e];
      }
      cluster_sync(C);
      return place;
    };
    u64 z = m_all, above = m_all, wcut = 0;
    if (k > 0 && u64(k) < n_all) {
      if (u64(k) > n_pos && u64(k) <= n_pos + n_list) return false;
      const Slot f = locate(true, u64(k), s.found);
      cut = bin_value(int(f.a));
      ties = u64(k) - f.c;
      wcut = bv.weight[f.a];
      above = f.b;
      z = above + ties * wcut;
    }
    if (tp < 1.f) {
      u64 target = u64(ceil(double(z) * double(tp)));
      if (target < 1) target = 1;
      if (target <= above) {
        if (target > m_pos && target <= m_pos + m_list) return false;
        const Slot f = locate(false, target, s.found2);
        cut = bin_value(int(f.a));
        const u64 wc = max(bv.weight[f.a], u64(1));
        ties = (target - f.b + wc - 1) / wc;
      } else if (wcut > 0) {
        ties = min(ties, (target - above + wcut - 1) / wcut);
      }
    }
    return true;
  }

  struct Cut {
    float x;    // values above it are kept, and the first ties of those equal to it
    u64 above;  // summed measure of the values above it
  };
  // The cut at which the running measure reaches the target.  The first histogram (over
  // the window) is filled; measure(x) is 0 for tokens out of the running.
  template <bool kCount, typename M>
  __device__ Cut select(u64 target, M measure) {
    Found f = find<kCount>(0, target, false);
    u64 acc = f.before;
    uint32_t lo = ord_key(-3.402823466e38f), hi = ord_key(m);
    int q = -1;  // second-level distance of the tokens left, -1: those beyond the window
    clear();
    if (f.bin >= 0) {
      const int b1 = f.bin;
      visit([&](const float(&x)[VEC], int) {
        bool in[VEC], any = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = (m - x[j]) * dscale;
          any |= in[j] = d >= float(b1 << kBinBits) && d < float((b1 + 1) << kBinBits);
        }
        if (!any) return;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (!in[j]) continue;
          const u64 v = measure(x[j]);
          if (!v) continue;
          const int sub = dist(x[j]) & (kBins - 1);
          add<kCount>(sub, v);
          atomicMin(&s.kmin[sub], ord_key(x[j]));
          atomicMax(&s.kmax[sub], ord_key(x[j]));
        }
      });
      f = find<kCount>(acc, target, true);
      q = (b1 << kBinBits) | max(f.bin, 0);
      acc = f.before;
      lo = f.lo;
      hi = f.hi;
      clear();
    }
    // the tokens left differ in their lowest bits only, or lie beyond the window: by key,
    // ten bits at a time
    for (int level = 0; lo < hi && level < 4; ++level) {
      int shift = 0;
      while (((hi - lo) >> shift) >= uint32_t(kBins)) ++shift;
      visit([&](const float(&x)[VEC], int) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint32_t k = ord_key(x[j]);
          if (k < lo || k > hi || dist(x[j]) != q) continue;
          const u64 v = measure(x[j]);
          if (v) add<kCount>(int((hi - k) >> shift), v);
        }
      });
      f = find<kCount>(acc, target, false);
      acc = f.before;
      const uint32_t top = hi - (uint32_t(max(f.bin, 0)) << shift);
      const uint32_t width = (1u << shift) - 1;
      lo = top - lo > width ? top - width : lo;
      hi = top;
      clear();
    }
    return Cut{key_value(hi), acc};
  }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Maximum of this warp's tokens (NaN ignored), and whether any is NaN or infinite.  Two
// 16-bit elements at a time: adding one to the exponent's lowest bit carries into the
// sign's place exactly when all its bits are set.
template <typename T>
__device__ __forceinline__ void scan_max(const T* row, int i0, int i1, bool vec, float& mx,
                                         uint32_t& special) {
  constexpr int VEC = 16 / int(sizeof(T));
  const int lane = threadIdx.x & 31;
  mx = -INFINITY;
  special = 0;
  for (int base = i0 + lane * VEC; base < i1; base += 32 * VEC) {
    if (vec && base + VEC <= i1) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + base));
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mx = fmaxf(mx, __uint_as_float(w[j]));
          special |= ((w[j] & 0x7fffffffu) + 0x00800000u) & 0x80000000u;
        }
      } else {
        constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
        constexpr uint32_t kInc = kBF16 ? 0x00800080u : 0x04000400u;
        using T2 = typename std::conditional<kBF16, __nv_bfloat162, __half2>::type;
        T2 v[4];
        memcpy(v, w, 16);
        const T2 a = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
        mx = fmaxf(mx, fmaxf(Elem<T>::to_f32(a.x), Elem<T>::to_f32(a.y)));
#pragma unroll
        for (int j = 0; j < 4; ++j) special |= ((w[j] & 0x7fff7fffu) + kInc) & 0x80008000u;
      }
    } else {
      for (int j = 0; j < VEC && base + j < i1; ++j) {
        const float x = Elem<T>::to_f32(row[base + j]);
        mx = fmaxf(mx, x);
        special |= ((__float_as_uint(x) & 0x7fffffffu) + 0x00800000u) & 0x80000000u;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_tokens_kernel(const T* __restrict__ logits, const Params p) {
  __shared__ Shared s;
  extern __shared__ __align__(16) uint8_t dynamic_smem[];  // bf16: ByValue
  constexpr bool kByValue = std::is_same<T, __nv_bfloat16>::value;
  ByValue& bv = *reinterpret_cast<ByValue*>(dynamic_smem);
  constexpr int VEC = Row<T>::VEC;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int r = blockIdx.x / p.C;
  Row<T> w{s};
  w.C = p.C;
  w.rank = p.C > 1 ? int(cluster_rank()) : 0;
  w.turn = 0;
  w.row = logits + int64_t(r) * p.row_stride;
  w.vec = (reinterpret_cast<uintptr_t>(w.row) & 15) == 0;
  w.by_value = nullptr;
  const int first = min(p.V, w.rank * p.chunk), last = min(p.V, first + p.chunk);
  // every warp owns one run of the CTA's run, in steps of a warp's 512 bytes
  const int per_warp = ((last - first + kWarps - 1) / kWarps + 255) / 256 * 256;
  w.i0 = min(last, first + warp * per_warp);
  w.i1 = min(last, w.i0 + per_warp);

  if (t == 0) s.holds = 0;
  for (int i = t; i < kTable; i += kThreads)
    s.table[i] = exp2(double(i) / kTable) * double(1ull << kFrac);
  if constexpr (kByValue) {
    for (int i = t; i < 2 * kValues; i += kThreads) bv.count[i] = 0;
    if (t == 0) bv.n_listed = bv.refuse = 0;
  }
  w.clear();
  pdl_wait();  // programmatic launch: the logits come from the kernel before
  pdl_trigger();

  // the row's settings, as one CTA reads them
  Slot mine{0, 0, 0};
  const float u = p.u[r];
  if (w.rank == 0) {
    mine.b = (u64(__float_as_uint(p.temperature[r])) << 32) |
             __float_as_uint(p.top_p ? p.top_p[r] : 1.f);
    mine.c = (u64(uint32_t(p.top_k ? p.top_k[r] : 0)) << 32) |
             __float_as_uint(p.min_p ? p.min_p[r] : 0.f);
  }
  float mx;
  uint32_t special = 0;
  if constexpr (kByValue)
    w.count_values(bv, mx);
  else
    scan_max(w.row, w.i0, w.i1, w.vec, mx, special);
  special = __reduce_or_sync(0xffffffffu, special);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) s.warp[warp] = (u64(special != 0) << 32) | ord_key(mx);
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) {
    mine.a = max(mine.a & 0xffffffffull, s.warp[i] & 0xffffffffull) |
             ((mine.a | s.warp[i]) & (1ull << 32));
  }
  if (kByValue && (bv.refuse || !(u > 0.f))) mine.a |= 1ull << 32;
  const Slot* all = w.exchange(mine);
  u64 top = 0;
  w.special = false;
  for (int q = 0; q < p.C; ++q) {
    top = max(top, all[q].a & 0xffffffffull);
    w.special |= (all[q].a >> 32) != 0;
  }
  w.m = key_value(uint32_t(top));
  const float T_ = __uint_as_float(uint32_t(all[0].b >> 32));
  const float tp = __uint_as_float(uint32_t(all[0].b));
  const int k = int(uint32_t(all[0].c >> 32));
  const float mp = __uint_as_float(uint32_t(all[0].c));
  // values of -128 and below weigh less than half a unit
  const bool by_value = kByValue && !w.special && (w.m + 128.f) > 45.f * T_;
  if (kByValue && !by_value) w.special = true;  // what the first pass saw is not known here
  if (w.special) {  // over the sanitised values
    float best = -INFINITY;
    w.visit([&](const float(&x)[VEC], int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) best = fmaxf(best, x[j]);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) s.warp[warp] = ord_key(best);
    __syncthreads();
    u64 key = 0;
    for (int i = 0; i < kWarps; ++i) key = max(key, s.warp[i]);
    all = w.exchange(Slot{key, 0, 0});
    key = 0;
    for (int q = 0; q < p.C; ++q) key = max(key, all[q].a);
    w.m = key_value(uint32_t(key));
  }
  const float m = w.m;

  // the least index that passes a test, over the cluster
  auto first_index = [&](auto test) -> int {
    uint32_t at = 0xffffffffu;
    w.visit([&](const float(&x)[VEC], int i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (test(x[j])) at = min(at, uint32_t(i + j));
    });
    at = __reduce_min_sync(0xffffffffu, at);
    __syncthreads();
    if (lane == 0) s.warp[warp] = at;
    __syncthreads();
    u64 least = 0xffffffffu;
    for (int i = 0; i < kWarps; ++i) least = min(least, s.warp[i]);
    const Slot* got = w.exchange(Slot{least, 0, 0});
    for (int q = 0; q < p.C; ++q) least = min(least, got[q].a);
    return int(least);
  };
  if (!(T_ > 1e-6f) || k == 1 || tp <= 0.f || mp > 1.f) {  // one token is kept: the first maximum
    const int at = first_index([&](float x) { return x == m; });
    if (w.rank == 0 && t == 0) {
      p.out[r] = at;
      if (p.logprobs) p.logprobs[r] = 0.f;
    }
    if (p.C > 1) cluster_sync(p.C);  // no CTA leaves while its slots may be written
    return;
  }
  const double T64 = double(T_);
  w.c = 1.4426950408889634 / T64;
  w.md = double(m);
  w.dscale = float(double(1 << (2 * kBinBits)) / double(kWindow) / T64);

  // -FLT_MAX - 1: everything is above the cut
  float cut = -INFINITY;
  u64 ties = ~0ull;
  bool cuts = false;  // found
  if constexpr (kByValue) {
    if (by_value && (tp < 1.f || (k > 0 && k < p.V) || !(mp > 0.f))) {
      cuts = w.value_cuts(bv, k, tp, cut, ties);
      if (!cuts) {
        cut = -INFINITY;
        ties = ~0ull;
        __syncthreads();
        w.clear();
      }
    }
  }
  if (!cuts && k > 0 && k < p.V) {
    w.visit([&](const float(&x)[VEC], int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int d = w.dist(x[j]);
        if (d >= 0) w.template add<true>(d >> kBinBits, 1);
      }
    });
    const auto c = w.template select<true>(u64(k), [](float) { return 1ull; });
    cut = c.x;
    ties = u64(k) - c.above;
  }
  if (!cuts && tp < 1.f) {
    // weights of the first n_k: all above the cut, and `ties` times the weight at it
    u64 z = 0;
    w.visit([&](const float(&x)[VEC], int) {
      w.weigh(x, [&](float v) { return v > cut; }, [&](float v, int, u64 f) {
        z += f;
        const int d = w.dist(v);
        if (d >= 0 && f) w.template add<false>(d >> kBinBits, f);
      });
    });
    z = warp_sum(z);
    __syncthreads();
    if (lane == 0) s.warp[warp] = z;
    __syncthreads();
    z = 0;
    for (int i = 0; i < kWarps; ++i) z += s.warp[i];
    all = w.exchange(Slot{z, 0, 0});
    z = 0;
    for (int q = 0; q < p.C; ++q) z += all[q].a;
    const u64 above = z;
    const u64 wcut = cut == -INFINITY ? 0 : w.fixed(cut);
    if (cut != -INFINITY) z += ties * wcut;
    u64 target = u64(ceil(double(z) * double(tp)));
    if (target < 1) target = 1;
    if (target <= above) {  // else the boundary lies among the ties at the cut
      const float old = cut;
      const auto c = w.template select<false>(
          target, [&](float x) { return x > old ? w.fixed(x) : 0ull; });
      cut = c.x;
      const u64 wc = max(w.fixed(cut), u64(1));
      ties = (target - c.above + wc - 1) / wc;
    } else if (wcut > 0) {
      ties = min(ties, (target - above + wcut - 1) / wcut);
    }
  }
  if (mp > 0.f) {
    // min-p is a threshold on the weight: the least value that passes, found by stepping
    // from its closed form
    auto pass = [&](float x) { return exp((double(x) - double(m)) / T64) >= double(mp); };
    const double at = double(m) + T64 * log(double(mp));
    if (at > -3e38) {
      uint32_t key = ord_key(float(at));
      for (int i = 0; i < 4 && pass(key_value(key - 1)); ++i) --key;
      for (int i = 0; i < 8 && !pass(key_value(key)); ++i) ++key;
      const float least = key_value(key);
      if (least > cut) {
        cut = least;
        ties = ~0ull;
      }
    }
  }
  // sums of the kept tokens above the cut and the number at it, by warp and CTA
  u64 sum = 0;
  uint32_t n_ties = 0, lowest = 0xffffffffu;
  w.visit([&](const float(&x)[VEC], int) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) n_ties += x[j] == cut;
    w.above(x, cut, [&](int, u64 f) { sum += f; });
  });
  if (!(u > 0.f))  // the first kept token of positive weight (in 64 bits: above 2^-1074)
    w.visit([&](const float(&x)[VEC], int i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (x[j] >= cut && (double(x[j]) - w.md) * w.c > -1074.0)
          lowest = min(lowest, uint32_t(i + j));
    });
  sum = warp_sum(sum);
  const u64 n_tie = __reduce_add_sync(0xffffffffu, n_ties);
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  __syncthreads();
  if (lane == 0) {
    s.warp[warp] = sum;
    s.warp2[warp] = (n_tie << 32) | lowest;
  }
  __syncthreads();
  Slot totals{0, 0, 0xffffffffu};
  for (int i = 0; i < kWarps; ++i) {
    totals.a += s.warp[i];
    totals.b += s.warp2[i] >> 32;
    totals.c = min(totals.c & 0xffffffffull, s.warp2[i] & 0xffffffffull);
  }
  if (w.rank == 0) totals.c |= u64(__float_as_uint(u)) << 32;
  all = w.exchange(totals);
  const float uu = __uint_as_float(uint32_t(all[0].c >> 32));
  const u64 wcut = cut == -INFINITY ? 0 : w.weight(cut);
  u64 before = 0, total = 0, t_before = 0, t_all = 0, low = 0xffffffffu;
  for (int q = 0; q < p.C; ++q) {
    if (q < w.rank) {
      before += all[q].a;
      t_before += all[q].b;
    }
    total += all[q].a;
    t_all += all[q].b;
    low = min(low, all[q].c & 0xffffffffull);
  }
  total += min(ties, t_all) * wcut;
  for (int i = 0; i < warp; ++i) {
    before += s.warp[i];
    t_before += s.warp2[i] >> 32;
  }
  before += min(ties, t_before) * wcut;
  u64 quota = ties > t_before ? min(ties - t_before, n_tie) : 0;  // this warp's ties
  const u64 here = sum + quota * wcut;
  const double one = double(1ull << kFrac);
  auto write = [&](int i, float x) {
    p.out[r] = i;
    if (p.logprobs)
      p.logprobs[r] = float((double(x) - double(m)) / T64 - log(double(total) / one));
  };
  if (p.C > 1) cluster_sync(p.C);  // every CTA has read its slots: none is used from here on
  if (!(uu > 0.f)) {
    if (w.rank == 0 && t == 0) {
      const float x = Elem<T>::to_f32(w.row[low]);
      write(int(low), sanitize(x));
    }
    return;
  }
  u64 target = u64(double(uu) * double(total));
  if (target >= total) target = total - 1;
  // The warp whose run holds the token divides its run among the CTA's warps, and the one
  // whose share holds it finds the token.
  __syncthreads();
  if (before <= target && target < before + here && lane == 0) {
    s.found = Slot{before, quota, (u64(uint32_t(w.i0)) << 32) | uint32_t(w.i1)};
    s.holds = 1;
  }
  __syncthreads();
  if (!s.holds) return;  // another CTA's run
  const int run0 = int(s.found.c >> 32), run1 = int(uint32_t(s.found.c));
  const int share = ((run1 - run0 + kWarps - 1) / kWarps + 32 * VEC - 1) / (32 * VEC) * (32 * VEC);
  w.i0 = min(run1, run0 + warp * share);
  w.i1 = min(run1, w.i0 + share);
  sum = 0;
  n_ties = 0;
  w.visit([&](const float(&x)[VEC], int) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) n_ties += x[j] == cut;
    w.above(x, cut, [&](int, u64 f) { sum += f; });
  });
  sum = warp_sum(sum);
  n_ties = __reduce_add_sync(0xffffffffu, n_ties);
  if (lane == 0) {
    s.warp[warp] = sum;
    s.warp2[warp] = n_ties;
  }
  __syncthreads();
  u64 c = s.found.a;
  quota = s.found.b;
  for (int i = 0; i < warp; ++i) {
    const u64 used = min(quota, s.warp2[i]);
    c += s.warp[i] + used * wcut;
    quota -= used;
  }
  if (!(c <= target && target < c + sum + min(quota, u64(n_ties)) * wcut)) return;
  bool done = false;
  w.visit([&](const float(&x)[VEC], int i) {
    if (done) return;
    uint32_t my_ties = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) my_ties += x[j] == cut;
    uint32_t ties_inc = my_ties;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t n = __shfl_up_sync(0xffffffffu, ties_inc, o);
      if (lane >= o) ties_inc += n;
    }
    uint32_t tie = ties_inc - my_ties;  // ties before this lane's tokens
    u64 v[VEC], mine_sum = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[j] = 0;
      if (x[j] == cut && u64(tie++) < quota) v[j] = wcut;
    }
    w.above(x, cut, [&](int j, u64 f) { v[j] += f; });
#pragma unroll
    for (int j = 0; j < VEC; ++j) mine_sum += v[j];
    u64 inc = mine_sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, c + inc > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        u64 run = c + inc - mine_sum;
        int at = 0;
        float chosen = x[0];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          run += v[j];
          if (run <= target && j + 1 < VEC) {
            at = j + 1;
            chosen = x[j + 1];
          }
        }
        write(i + at, chosen);
      }
      done = true;
    }
    c += __shfl_sync(0xffffffffu, inc, 31);
    const u64 used = __shfl_sync(0xffffffffu, ties_inc, 31);
    quota -= min(quota, used);
  });
}

// CTAs of a row's cluster: enough to fill the SMs (two CTAs each) when rows are few, at
// least 2048 tokens each so that the exchanges do not outweigh the work, and never more
// than kMaxRun each.
int cluster_size(int rows, int vocab) {
  int c = 1;
  while (c < kMaxCluster &&
         ((int64_t(rows) * c * 2 <= 2 * int64_t(sm_count()) && vocab / (2 * c) >= 2048) ||
          (vocab + c - 1) / c > kMaxRun - 256))
    c *= 2;
  return c;
}

}  // namespace
}  // namespace asb

using namespace asb;

extern "C" int as_sample_tokens(int64_t* out, float* logprobs, const void* logits,
                                int64_t row_stride, const float* u, const float* temperature,
                                const int32_t* top_k, const float* top_p, const float* min_p,
                                int32_t num_rows, int32_t vocab, int32_t dtype,
                                as_stream_t stream) {
  if (!dtype_size(dtype)) return fail(AS_ERR_INVALID_ARG, "as_sample_tokens: unknown dtype");
  if (num_rows < 0 || vocab <= 0 || row_stride < vocab)
    return fail(AS_ERR_INVALID_ARG, "as_sample_tokens: bad sizes");
  if (vocab > kMaxVocab)
    return fail(AS_ERR_UNSUPPORTED, "as_sample_tokens: vocab > %d", kMaxVocab);
  if (num_rows > (1 << 24)) return fail(AS_ERR_INVALID_ARG, "as_sample_tokens: too many rows");
  if (num_rows == 0) return AS_OK;
  if (!out || !logits || !u || !temperature)
    return fail(AS_ERR_INVALID_ARG, "as_sample_tokens: null pointer");
  if (reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype))
    return fail(AS_ERR_INVALID_ARG, "as_sample_tokens: logits are not aligned to their type");
  Params p{};
  p.out = out;
  p.logprobs = logprobs;
  p.u = u;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.row_stride = row_stride;
  p.V = vocab;
  p.C = cluster_size(num_rows, vocab);
  p.chunk = ((vocab + p.C - 1) / p.C + 255) / 256 * 256;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto tag) -> int {
    using T = decltype(tag);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(num_rows) * p.C);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    if (std::is_same<T, __nv_bfloat16>::value) {
      cfg.dynamicSmemBytes = sizeof(ByValue);
      cudaFuncSetAttribute(sample_tokens_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(sizeof(ByValue)));
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.C;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.C > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T>, static_cast<const T*>(logits), p);
    return check_launch("as_sample_tokens");
  };
  switch (dtype) {
    case AS_DTYPE_F32: return run(float());
    case AS_DTYPE_F16: return run(__half());
    default: return run(__nv_bfloat16());
  }
}
