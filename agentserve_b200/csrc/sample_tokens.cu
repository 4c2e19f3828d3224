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
// from the maximum: 1024 bins, then 1024 in the chosen bin, then (rarely) over the values'
// bits, until one value, or a list short enough to compare each token with all others, is
// left.
//
// Sums decide between neighbouring tokens, and a border token can weigh 1e-6 of the
// total: weights are computed in 64 bits and summed in fixed point (units of 2^-42 of
// the largest), which makes every sum exact and independent of the order of the atomics.
//
// Few rows are bound by latency (a cluster barrier or a pass of few tokens costs about 1K
// cycles: one bf16 row of 128,256 tokens, top-p, 19 us, of which the logits' bytes are 0.04),
// many by integer instructions and shared-memory atomics (256 rows 84 us, 66 MB read twice).
//
// A row is worked on by a cluster of 1 to 8 CTAs, each holding a run of indexes, its warps
// runs of that; they exchange totals over distributed shared memory.  Every decision
// follows from exchanged values, so all CTAs of a cluster take the same barriers.
#include <stddef.h>
#include <string.h>

#include <atomic>
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
constexpr float kWindow = 12.f;  // nats covered by the first histogram of weights
constexpr float kCountWindow = 24.f;  // units of the logits covered by that of counts
constexpr int kList = 256;       // tokens left at which a cut is found by comparing them all
constexpr int kTable = 512;      // 2^(i / 512)
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxRun = (1 << 17) + 256;  // tokens of a CTA
// A weight is at most 1 = 2^42 units: the sum of kMaxVocab of them fits 64 bits, and its
// three pieces of 14 bits, summed over a CTA's tokens, fit 32 bits each.
constexpr int kFrac = 42;
constexpr int kPiece = 14;
typedef unsigned long long u64;
// A weight is positive in 64 bits above 2^-1075, which rounds to 0.
constexpr double kLeastExponent = -1075.0;
static_assert(u64(kMaxRun) << kPiece < 1ull << 32 && kFrac - 2 * kPiece <= kPiece, "sums");
static_assert(kMaxVocab / kMaxCluster + 256 <= kMaxRun, "runs");

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
__device__ __forceinline__ uint4 peer_load4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
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

// The two halves of a first barrier: a CTA's shared memory may be written by others once it
// runs.
__device__ __forceinline__ void cluster_started(int C) {
  if (C == 1) return;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait_started(int C) {
  if (C == 1) return;
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Slot {
  u64 a, b, c;
};
struct alignas(16) Shared {
  double table[kTable];       // 2^(i / 512) in units of the fixed point
  uint32_t hist[3][kBins];    // pieces of the summed measure
  uint32_t kmin[kBins], kmax[kBins];
  Slot slot[2][kMaxCluster];  // exchanges, in turn
  Slot found, found2;
  u64 warp[kWarps];
  uint32_t flag;
  uint32_t n_list;     // tokens left in this CTA's run; the first of them
  float list[kList];
  float left[kList];   // the cluster's, and what each measures
  u64 measure[kList];
};
// Tokens waiting for their weight, per warp: one group of a visit past a full batch.
constexpr int kBatch = 64;
constexpr int kQueue = kBatch - 1 + 256;
struct Queue {
  float x[kWarps][kQueue + 1];
};
static_assert(sizeof(Queue) >= 3 * kBins * 4 && kThreads == kBins / 2, "find() stages over it");

// bf16 rows: a histogram by value.  The 4096 values of magnitude 2^-9 to 128 have a
// bin each; the few closer to zero are listed; those at or below -128 (masks) weigh
// nothing next to any maximum this path accepts.  The first pass then needs no maximum
// and no exponential, both cuts come from one merge, and the second pass looks the
// weights up.  Rows outside this (values of 128 and more, NaN, cuts among the listed
// values, u <= 0 or >= 1) take the general path.
//
// 64 rows of 128,256 tokens, top-p: 35 us, and 81 by the general path (fp16).  The passes
// are bound by integer instructions (half rate), so a value's place is two
// logic operations and a multiply-add away from its 16 bits: counts (4 bytes each) and
// weights (8) lie in ascending magnitude, those of the negative values 0x8000 bytes after
// those of the positive ones.
constexpr int kValueLo = (127 - 9) << 7;  // bits of 2^-9
constexpr int kValues = 16 << 7;          // values of one sign
constexpr int kListed = 2048;
struct ByValue {
  uint32_t positive[kValues];      // counts
  u64 weight_positive[kValues];
  uint16_t list[kListed];
  uint32_t n_listed, refuse, pad[(0x8000 - 28 * 1024) / 4 - 2];
  uint32_t negative[kValues];      // byte 0x8000
  u64 weight_negative[kValues];
};
static_assert(offsetof(ByValue, negative) - offsetof(ByValue, positive) == 0x8000 &&
                  offsetof(ByValue, weight_negative) - offsetof(ByValue, weight_positive) == 0x8000,
              "layout");
__device__ __forceinline__ bool has_bin(uint32_t code) {
  return (code & 0x7fff) - uint32_t(kValueLo) < uint32_t(kValues);
}
// Byte offsets of a value's count and weight from the (virtual) ones of +0.
__device__ __forceinline__ uint32_t count_offset(uint32_t code) {
  return (code & 0x7fff) * 4 + (code & 0x8000);
}
__device__ __forceinline__ uint32_t weight_offset(uint32_t code) {
  return (code & 0x7fff) * 8 + (code & 0x8000);
}
// Values in descending order: bin -> code.
__device__ __forceinline__ uint32_t bin_code(int bin) {
  return bin < kValues ? uint32_t(kValueLo + kValues - 1 - bin)
                       : 0x8000u | uint32_t(kValueLo + bin - kValues);
}
__device__ __forceinline__ float code_value(uint32_t code) { return __uint_as_float(code << 16); }

struct Params {
  int64_t* out;
  float* logprobs;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t row_stride;
  int V, C, chunk;  // tokens, CTAs of a cluster, tokens of a CTA
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, v, o);
    if (int(threadIdx.x & 31) >= o) v += n;
  }
  return v;
}
// Most of a call's time on a short row is the fetching of instructions that run once, so
// the steps that several stages share are functions of their own.
struct Scan {
  u64 before, total;  // of the threads before this one; of the block
};
__device__ __noinline__ Scan block_scan(Shared& s, u64 v) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const u64 inc = warp_scan(v);
  __syncthreads();  // s.warp is free
  if (lane == 31) s.warp[warp] = inc;
  __syncthreads();
  const u64 w = warp_scan(lane < kWarps ? s.warp[lane] : 0);
  const u64 base = __shfl_sync(0xffffffffu, w, warp == 0 ? 0 : warp - 1);
  return Scan{(warp ? base : 0) + inc - v, __shfl_sync(0xffffffffu, w, kWarps - 1)};
}

struct Found {
  int bin;          // -1: the target lies beyond the histogram
  u64 before;       // sum above the bin (or of the whole histogram)
  uint32_t lo, hi;  // least and largest key in it, where those were kept
};

// One CTA's view of its row.
template <typename T>
struct Row {
  Shared* sp;
  const T* row;
  Queue* queue;
  const ByValue* by_value;  // weights by value (bf16), or null
  int C, rank, turn;    // turn: which slot buffer the next exchange uses
  int i0, i1;           // this warp's run of indexes (from below 0: see visit)
  bool special;         // it holds NaN or infinities
  float m, dscale;      // maximum; distances from it in second-level bins
  double c, md;         // log2(e) / T; m

  static constexpr int VEC = 16 / int(sizeof(T));
  static constexpr int kGroup = 32 * VEC;
  __device__ __forceinline__ bool inside(int i) const { return uint32_t(i) < uint32_t(i1); }

  // f(x, index of x[0]) for this warp's tokens, 32 lanes x 16 bytes at a time, loads three
  // groups ahead; places outside the run hold -infinity, which no token is.  Every lane
  // makes the same trips.  Runs begin at 16-byte boundaries: that of a row which does not
  // begins at the one before it, at an index below 0, and its first group is read token by
  // token.
  template <typename F>
  __device__ __forceinline__ void visit(F f) const {
    const int first = i0 + int(threadIdx.x & 31) * VEC;
    const int full = (i1 - i0) / kGroup, groups = (i1 - i0 + kGroup - 1) / kGroup;
    const auto whole = [&](int g) { return g < full && (g > 0 || i0 >= 0); };
    const uint4* src = reinterpret_cast<const uint4*>(row + first);
    const auto load = [&](int g) -> uint4 {
      return whole(g) ? __ldg(src + g * 32) : make_uint4(0, 0, 0, 0);
    };
    uint4 r0 = load(0), r1 = load(1), r2 = load(2);
#pragma unroll 1
    for (int g = 0; g < groups; ++g) {
      const uint4 raw = r0;
      r0 = r1;
      r1 = r2;
      r2 = load(g + 3);
      const int i = first + g * kGroup;
      float x[VEC];
      if (whole(g)) {
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = Elem<T>::to_f32(e[j]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = inside(i + j) ? Elem<T>::to_f32(row[i + j]) : -INFINITY;
      }
      if (special) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          x[j] = inside(i + j) ? sanitize(x[j]) : -INFINITY;
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
    const double xd = __hiloint2double(
        int((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), int(b << 29));
    const double d = xd - md;
    const double kRound = 6755399441055744.0 / 512.0;  // 1.5 * 2^52 / 512
    const double t = fma(d, c, kRound);
    const int j = __double2loint(t);
    const double whole = t - kRound;
    const double f = fma(d, c, -whole);
    double p = fma(f, 0.05550410866482158, 0.24022650695910072);  // ln2^3 / 6, ln2^2 / 2
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    const double tab = sp->table[j & (kTable - 1)];
    const double scaled =
        __hiloint2double(__double2hiint(tab) + ((j >> 9) << 20), __double2loint(tab));
    const double v = fma(scaled, p, 4503599627370496.0);  // 2^52
    const u64 bits = u64(__double_as_longlong(v)) & 0xFFFFFFFFFFFFFull;
    return whole > -60.0 ? bits : 0ull;  // below half a unit (and out of the exponent's range)
  }
  // The weight of a token, looked up where the row has a table.
  __device__ __forceinline__ u64 weight(float x) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const uint32_t code = __float_as_uint(x) >> 16;
      if (by_value && has_bin(code))
        return *reinterpret_cast<const u64*>(
            reinterpret_cast<const uint8_t*>(by_value->weight_positive) +
            (weight_offset(code) - 8 * kValueLo));
    }
    return fixed(x);
  }
  // Distance from the maximum in second-level bins, -1 outside the window.
  __device__ __forceinline__ int dist(float x) const {
    const float d = (m - x) * dscale;
    return d < float(1 << (2 * kBinBits)) ? int(d) : -1;
  }

  // Slot `v` of every CTA, at every CTA.  One barrier; two buffers in turn, so a slot is
  // rewritten only after a barrier that follows its last reads.
  __device__ __forceinline__ const Slot* exchange(const Slot& v) {
    Slot* buf = sp->slot[turn];
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
  __device__ __forceinline__ void clear() const {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      sp->hist[0][i] = sp->hist[1][i] = sp->hist[2][i] = 0;
      sp->kmin[i] = 0xffffffffu;
      sp->kmax[i] = 0;
    }
    if (threadIdx.x == 0) sp->n_list = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add(int bin, u64 v) const {
    constexpr uint32_t mask = (1u << kPiece) - 1;
    atomicAdd(&sp->hist[0][bin], uint32_t(v) & mask);
    const uint32_t mid = uint32_t(v >> kPiece) & mask, top = uint32_t(v >> (2 * kPiece));
    if (mid) atomicAdd(&sp->hist[1][bin], mid);
    if (top) atomicAdd(&sp->hist[2][bin], top);
  }
};

// A weight outside the passes, where the code's size counts more than a call.
template <typename T>
__device__ __noinline__ u64 fixed_call(const Shared* sp, double md, double c, float x) {
  Row<T> w;
  w.sp = const_cast<Shared*>(sp);
  w.md = md;
  w.c = c;
  return w.fixed(x);
}

// Sums the cluster's histograms and finds the first bin at which acc + the running sum
// reaches the target, by way of one exchange.  The histograms may be cleared afterwards.
template <typename T>
__device__ __noinline__ Found find(Row<T> w, u64 acc, u64 target, bool keys) {
  Shared& s = *w.sp;
  const int C = w.C, t = threadIdx.x;
  cluster_sync(C);  // every CTA's histogram is complete
  const int S = kBins / C;  // bins of this CTA's slice; thread t has 2t, 2t + 1 or t
  const int per = S > kThreads ? 2 : 1, mine = t * per, bin0 = w.rank * S + mine;
  const uint32_t* from = &s.hist[0][0];
  if (C > 1) {
    // The slice of every CTA's three histograms, side by side, over the queue (not in use
    // now): 768 loads of 16 bytes, all in flight at once.  (Summed straight from the peers,
    // three words at a time: find() took 11.5K cycles of a call's 47K.)
    uint32_t* stage = reinterpret_cast<uint32_t*>(w.queue);
    const int r = (t & (kBins / 4 - 1)) * 4, e = t / (kBins / 4);  // e: 0 or 1
    const uint32_t at = peer_addr_of(&s.hist[0][w.rank * S + (r & (S - 1))], r / S);
    const uint4 x = peer_load4(at + 4 * kBins * e);
    if (e == 0) {
      const uint4 y = peer_load4(at + 4 * kBins * 2);
      *reinterpret_cast<uint4*>(stage + 2 * kBins + r) = y;
    }
    *reinterpret_cast<uint4*>(stage + kBins * e + r) = x;
    from = stage;
    __syncthreads();
  }
  u64 v[2] = {0, 0};
  if (mine < S) {
    const auto bin = [&](const uint32_t* h) -> u64 {
      return h[0] + (u64(h[kBins]) << kPiece) + (u64(h[2 * kBins]) << (2 * kPiece));
    };
    for (int q = 0; q < C; ++q) v[0] += bin(from + q * S + mine);
    if (per == 2) v[1] = bin(from + mine + 1);  // C = 1
  }
  const Scan sc = block_scan(s, v[0] + v[1]);
  const Slot* all = w.exchange(Slot{sc.total, 0, 0});
  u64 start = acc, whole = acc;
  for (int q = 0; q < C; ++q) {
    if (q < w.rank) start += all[q].a;
    whole += all[q].a;
  }
  if (whole < target) return Found{-1, whole, 0, 0};
  // the thread whose bin it is tells every CTA
  const u64 b0 = start + sc.before, b1 = b0 + v[0], b2 = b1 + v[1];
  if (b0 < target && b2 >= target) {
    const int e = b1 >= target ? 0 : 1;
    uint32_t lo = 0xffffffffu, hi = 0;
    if (keys) {
      for (int q = 0; q < C; ++q) {
        lo = min(lo, peer_load(peer_addr_of(&s.kmin[bin0 + e], q)));
        hi = max(hi, peer_load(peer_addr_of(&s.kmax[bin0 + e], q)));
      }
    }
    for (int q = 0; q < C; ++q) {
      const uint32_t at = peer_addr_of(&s.found, q);
      peer_store64(at, u64(bin0 + e));
      peer_store64(at + 8, e ? b1 : b0);
      peer_store64(at + 16, (u64(hi) << 32) | lo);
    }
  }
  cluster_sync(C);
  return Found{int(s.found.a), s.found.b, uint32_t(s.found.c), uint32_t(s.found.c >> 32)};
}

struct Cut {
  float x;    // values above it are kept, and the first ties of those equal to it
  u64 above;  // summed measure of the values above it
  int turn;
};
// The cut at which the running measure reaches the target: the number of tokens, or the
// weight of those above `over`.  The first histogram (over the window) is filled.
template <typename T>
__device__ __noinline__ Cut select_cut(Row<T> w, bool count, u64 target, float over) {
  constexpr int VEC = Row<T>::VEC;
  Shared& s = *w.sp;
  Found f = find(w, 0, target, false);
  w.turn ^= 1;
  u64 acc = f.before;
  uint32_t lo = ord_key(-3.402823466e38f), hi = ord_key(w.m);
  int q = -1;  // distance of the tokens left, -1: those beyond the window
  const bool in_window = f.bin >= 0;
  const float near = in_window ? float(f.bin << kBinBits) : 0.f;
  const float far = near + float(kBins);
  bool first = in_window;
  // The tokens left: those of the chosen bin, by distance; after that (or beyond the
  // window) those that differ in their lowest bits only, by key, ten bits at a time.
  for (int level = 0; first || (lo < hi && level < 5); ++level) {
    int shift = 0;
    while (((hi - lo) >> shift) >= uint32_t(kBins)) ++shift;
    __syncthreads();
    w.clear();
    w.visit([&](const float(&x)[VEC], int) {
      uint32_t in = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        bool mine;
        if (first) {
          const float d = (w.m - x[j]) * w.dscale;
          mine = d >= near && d < far;
        } else {
          const uint32_t k = ord_key(x[j]);
          mine = k >= lo && k <= hi && w.dist(x[j]) == q;
        }
        in |= uint32_t(mine) << j;
      }
      while (in) {  // few
        const int j = __ffs(in) - 1;
        in &= in - 1;
        float y = x[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) y = e == j ? x[e] : y;
        const u64 v = count ? 1 : (y > over ? w.fixed(y) : 0);
        if (!v) continue;
        const uint32_t at = atomicAdd(&s.n_list, 1u);
        if (at < kList) s.list[at] = y;
        const int bin = first ? w.dist(y) & (kBins - 1) : int((hi - ord_key(y)) >> shift);
        w.add(bin, v);
        if (first) {
          atomicMin(&s.kmin[bin], ord_key(y));
          atomicMax(&s.kmax[bin], ord_key(y));
        }
      }
    });
    __syncthreads();
    const Slot* all = w.exchange(Slot{s.n_list, 0, 0});
    uint32_t left = 0;
    for (int e = 0; e < w.C; ++e) left += uint32_t(all[e].a);
    if (left <= kList) {
      // Few: every CTA gathers them, and each token is compared with every other.
      uint32_t from = 0;
      for (int e = 0; e < w.C; ++e) {
        const uint32_t n = uint32_t(all[e].a);
        if (threadIdx.x < n) {
          const float y = __uint_as_float(peer_load(peer_addr_of(&s.list[threadIdx.x], e)));
          s.left[from + threadIdx.x] = y;
          s.measure[from + threadIdx.x] = count ? 1 : w.fixed(y);
        }
        from += n;
      }
      __syncthreads();
      if (threadIdx.x < left) {
        const float y = s.left[threadIdx.x];
        u64 above = acc, here = 0;
#pragma unroll 1
        for (uint32_t i = 0; i < left; ++i) {
          const float z = s.left[i];
          const u64 v = s.measure[i];
          above += z > y ? v : 0;
          here += z == y ? v : 0;
        }
        if (above < target && above + here >= target)  // equal tokens write the same
          s.found = Slot{__float_as_uint(y), above, 0};
      }
      __syncthreads();
      hi = ord_key(__uint_as_float(uint32_t(s.found.a)));
      acc = s.found.b;
      break;
    }
    const int b1 = f.bin;
    f = find(w, acc, target, first);
    w.turn ^= 1;
    acc = f.before;
    const uint32_t bin = uint32_t(max(f.bin, 0));
    if (first) {
      q = (b1 << kBinBits) | int(bin);
      lo = f.lo;
      hi = f.hi;
      first = false;
    } else {
      const uint32_t top = hi - (bin << shift), width = (1u << shift) - 1;
      lo = top - lo > width ? top - width : lo;
      hi = top;
    }
  }
  __syncthreads();
  w.clear();
  return Cut{key_value(hi), acc, w.turn};
}

// This warp's summed weight of the tokens above the cut, and its number of tokens at it;
// with `hist`, the first histogram by weight as well.  Tokens above the cut wait in a
// queue until two batches of 32 are there, so the long chain of a weight is walked by
// full warps, twice side by side.
struct Kept {
  u64 sum;
  uint32_t ties;
};
template <typename T>
__device__ __noinline__ Kept sum_above(Row<T> w, float cut, bool hist) {
  constexpr int VEC = Row<T>::VEC;
  const int lane = threadIdx.x & 31;
  float* q = w.queue->x[threadIdx.x >> 5];
  int n = 0;
  u64 sum = 0;
  uint32_t ties = 0;
  const auto batch = [&]() {
    __syncwarp();
    n -= kBatch;  // may be negative at the end
    const bool has_a = n + lane >= 0, has_b = n + 32 + lane >= 0;
    const float a = has_a ? q[n + lane] : w.m, b = has_b ? q[n + 32 + lane] : w.m;
    u64 va = w.fixed(a), vb = w.fixed(b);
    va = has_a ? va : 0;
    vb = has_b ? vb : 0;
    sum += va + vb;
    if (hist) {
#pragma unroll 1
      for (int e = 0; e < 2; ++e) {
        const int d = w.dist(e ? b : a);
        const u64 v = e ? vb : va;
        if (d >= 0 && v) w.add(d >> kBinBits, v);
      }
    }
    __syncwarp();
  };
  w.visit([&](const float(&x)[VEC], int) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      any |= x[j] > cut;
      ties += x[j] == cut;
    }
    if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const uint32_t mask = __ballot_sync(0xffffffffu, x[j] > cut);
      if (x[j] > cut) q[n + __popc(mask & ((1u << lane) - 1))] = x[j];
      n += __popc(mask);
    }
    while (n >= kBatch) batch();
  });
  if (n > 0) batch();
  return Kept{warp_sum(sum), __reduce_add_sync(0xffffffffu, ties)};
}

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) {
  __nv_bfloat162 v;
  memcpy(&v, &w, 4);
  return v;
}
// Whether a pair of values has one without a bin: bits 15 and 31.
__device__ __forceinline__ uint32_t unbinned(uint32_t w) {
  const uint32_t mag = w & 0x7fff7fffu;
  constexpr uint32_t kOver = 0x8000 - kValueLo - kValues, kUnder = 0x8000 - kValueLo;
  return ((mag + kOver * 0x10001u) | ~(mag + kUnder * 0x10001u)) & 0x80008000u;
}

// f(16 bytes) for a warp's run of a bf16 row, undecoded, as Row::visit reads it.  Plain
// arguments, so that nothing of the loop lives in memory.
template <typename F>
__device__ __forceinline__ void visit_bf16(const uint16_t* row, int i0, int i1, F f) {
  const int first = i0 + int(threadIdx.x & 31) * 8;
  const int full = (i1 - i0) / 256, groups = (i1 - i0 + 255) / 256;
  const auto whole = [&](int g) { return g < full && (g > 0 || i0 >= 0); };
  const uint4* src = reinterpret_cast<const uint4*>(row + first);
  const auto load = [&](int g) -> uint4 {
    return whole(g) ? __ldg(src + g * 32) : make_uint4(0, 0, 0, 0);
  };
  uint4 r0 = load(0), r1 = load(1), r2 = load(2);
#pragma unroll 1
  for (int g = 0; g < groups; ++g) {
    uint4 raw = r0;
    r0 = r1;
    r1 = r2;
    r2 = load(g + 3);
    if (!whole(g)) {
      uint32_t w[4] = {0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
      const int i = first + g * 256;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (uint32_t(i + j) < uint32_t(i1))
          w[j >> 1] = __byte_perm(w[j >> 1], row[i + j], j & 1 ? 0x5410 : 0x3254);
      raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
    f(raw);
  }
}

// sum_above() for a bf16 row with weights by value.
__device__ __noinline__ Kept sum_above_by_value(Row<__nv_bfloat16> w, float cut) {
  const __nv_bfloat162 cut2 = __float2bfloat162_rn(cut);  // exact: a bf16 value or a bound on them
  const uint8_t* weights =
      reinterpret_cast<const uint8_t*>(w.by_value->weight_positive) - 8 * kValueLo;
  u64 sum = 0;
  uint32_t ties = 0;
  visit_bf16(reinterpret_cast<const uint16_t*>(w.row), w.i0, w.i1,
             [&](const uint4& raw) {
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
    const __nv_bfloat162 top = __hmax2(__hmax2(as_bf162(word[0]), as_bf162(word[1])),
                                       __hmax2(as_bf162(word[2]), as_bf162(word[3])));
    if (!__any_sync(0xffffffffu, __hge2_mask(top, cut2) != 0)) return;
    uint32_t slow = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t bad = unbinned(word[j]);
      uint32_t up = __hgt2_mask(as_bf162(word[j]), cut2);
      ties += __popc(__heq2_mask(as_bf162(word[j]), cut2) & 0x10001u);
      slow |= bad & up;
      up &= ~bad;
      if (up & 0x8000)
        sum += *reinterpret_cast<const u64*>(weights + weight_offset(word[j]));
      if (int(up) < 0)
        sum += *reinterpret_cast<const u64*>(weights + weight_offset(word[j] >> 16));
    }
    if (slow) {  // closer to zero than the bins (or far below: no weight)
      uint32_t a = word[0], b = word[1], c = word[2], d = word[3];
#pragma unroll 1
      for (int j = 0; j < 8; ++j) {
        const float x = code_value(a & 0xffff);
        if (!has_bin(a) && x > cut) sum += w.fixed(x);
        a = __funnelshift_r(a, b, 16);
        b = __funnelshift_r(b, c, 16);
        c = __funnelshift_r(c, d, 16);
        d >>= 16;
      }
    }
  });
  return Kept{warp_sum(sum), __reduce_add_sync(0xffffffffu, ties)};
}

// First pass of a bf16 row: counts by value, and the maximum.
__device__ __noinline__ float count_values(const uint16_t* row, int i0, int i1, ByValue& bv) {
  uint8_t* counts = reinterpret_cast<uint8_t*>(bv.positive) - 4 * kValueLo;
  const auto count = [&](uint32_t code) {
    atomicAdd(reinterpret_cast<uint32_t*>(counts + count_offset(code)), 1u);
  };
  __nv_bfloat162 top = __float2bfloat162_rn(-INFINITY);
  visit_bf16(row, i0, i1, [&](const uint4& raw) {
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
    const uint32_t odd =
        unbinned(word[0]) | unbinned(word[1]) | unbinned(word[2]) | unbinned(word[3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __hmax2(top, as_bf162(word[j]));
    if (!odd) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        count(word[j]);
        count(word[j] >> 16);
      }
      return;
    }
    // few groups: token by token
    uint32_t a = word[0], b = word[1], c = word[2], d = word[3];
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      const uint32_t mag = a & 0x7fff;
      if (mag - uint32_t(kValueLo) < uint32_t(kValues)) {
        count(a);
      } else if (mag < uint32_t(kValueLo)) {
        const uint32_t at = atomicAdd(&bv.n_listed, 1u);
        if (at < kListed)
          bv.list[at] = uint16_t(a);
        else
          bv.refuse = 1;
      } else if (!(a & 0x8000) || mag > 0x7f80) {  // 128 and more, NaN
        bv.refuse = 1;
      }
      a = __funnelshift_r(a, b, 16);
      b = __funnelshift_r(b, c, 16);
      c = __funnelshift_r(c, d, 16);
      d >>= 16;
    }
  });
  return fmaxf(__bfloat162float(top.x), __bfloat162float(top.y));
}

// Both cuts of a bf16 row from the cluster's counts by value.  cut.turn < 0: one of them
// lies among the listed values.
struct Cuts {
  float x;
  u64 ties;
  int turn;
};
template <int C>
__device__ __noinline__ Cuts value_cuts(Row<__nv_bfloat16> w, ByValue& bv, int k, float tp) {
  Shared& s = *w.sp;
  const int t = threadIdx.x;
  constexpr int kAll = 2 * kValues, S = kAll / C, kPer = S / kThreads;  // 8, 4, 2 or 1
  // thread t: bins [rank * S + t * kPer, + kPer) summed over the cluster
  const int first = w.rank * S + t * kPer;
  const int step = first < kValues ? -1 : 1;  // from one bin's count to the next's
  const uint8_t* counts = reinterpret_cast<const uint8_t*>(bv.positive) - 4 * kValueLo;
  const auto weight_of = [&](int bin) -> u64& {
    return *reinterpret_cast<u64*>(reinterpret_cast<uint8_t*>(bv.weight_positive) - 8 * kValueLo +
                                   weight_offset(bin_code(bin)));
  };
  uint32_t n[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) n[e] = 0;
  uint32_t h[C][kPer];
#pragma unroll
  for (int q = 0; q < C; ++q) {
    const uint32_t from = peer_addr(smem_u32(counts + count_offset(bin_code(first))), q);
#pragma unroll
    for (int e = 0; e < kPer; ++e) h[q][e] = peer_load(from + 4 * step * e);
  }
  u64 wt[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) wt[e] = w.fixed(code_value(bin_code(first + e)));
  for (int i = t; i < int(bv.n_listed); i += kThreads)
    w.add(0, w.fixed(code_value(bv.list[i])));
#pragma unroll
  for (int q = 0; q < C; ++q)
#pragma unroll
    for (int e = 0; e < kPer; ++e) n[e] += h[q][e];
  __syncthreads();  // the listed values' sum is there
  const u64 listed = s.hist[0][0] + (u64(s.hist[1][0]) << kPiece) + (u64(s.hist[2][0]) << (2 * kPiece));
  u64 mass = 0, num = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (n[e]) mass += n[e] * wt[e];
    num += n[e];
  }
  const Scan ms = block_scan(s, mass), ns = k > 0 ? block_scan(s, num) : Scan{0, 0};
  u64 m_before = ms.before, n_before = ns.before;
  if (C == 1 && t == kThreads / 2) s.found2 = Slot{0, m_before, n_before};  // the positive values
  const Slot* all = w.exchange(Slot{ms.total, (ns.total << 32) | bv.n_listed, listed});
  // running sums before this thread's bins; the listed values lie between the signs
  u64 m_pos = 0, n_pos = 0, m_list = 0, n_list = 0, m_all = 0, n_all = 0;
#pragma unroll
  for (int q = 0; q < C; ++q) {
    if (q < w.rank) {
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
    m_pos = s.found2.b;
    n_pos = s.found2.c;
    __syncthreads();
  }
  m_all += m_list;
  n_all += n_list;
  if (first >= kValues) {
    m_before += m_list;
    n_before += n_list;
  }
  // The first bin at which the running count (or weight) reaches the target: the thread
  // whose it is tells every CTA the sums before it.  (One place per call: no barrier
  // parts a CTA's read of the first from a peer's write of the second.)
  const auto locate = [&](bool count, u64 target, Slot& place) -> Slot {
    u64 a = m_before, b = n_before;
#pragma unroll 1
    for (int e = 0; e < kPer; ++e) {
      uint32_t ne = n[0];
      u64 we = wt[0];
#pragma unroll
      for (int y = 1; y < kPer; ++y) {
        ne = y == e ? n[y] : ne;
        we = y == e ? wt[y] : we;
      }
      const u64 da = ne ? ne * we : 0;
      const u64 run = count ? b : a, step = count ? ne : da;
      if (run < target && run + step >= target) {
        for (int q = 0; q < C; ++q) {
          const uint32_t at = peer_addr_of(&place, q);
          peer_store64(at, u64(first + e));
          peer_store64(at + 8, a);
          peer_store64(at + 16, b);
        }
      }
      a += da;
      b += ne;
    }
    cluster_sync(C);
    return place;
  };
  Cuts r{-INFINITY, ~0ull, w.turn};
  int last = kAll - 1;  // the lowest kept value's bin
  u64 z = m_all, above = m_all, wcut = 0;
  if (k > 0 && u64(k) < n_all) {
    if (u64(k) > n_pos && u64(k) <= n_pos + n_list) return Cuts{0.f, 0, -1 - w.turn};
    const Slot f = locate(true, u64(k), s.found);
    r.x = code_value(bin_code(int(f.a)));
    r.ties = u64(k) - f.c;
    last = int(f.a);
    wcut = w.fixed(r.x);
    above = f.b;
    z = above + r.ties * wcut;
  }
  if (tp < 1.f) {
    u64 target = u64(ceil(double(z) * double(tp)));
    if (target < 1) target = 1;
    if (target <= above) {
      if (target > m_pos && target <= m_pos + m_list) return Cuts{0.f, 0, -1 - w.turn};
      const Slot f = locate(false, target, s.found2);
      r.x = code_value(bin_code(int(f.a)));
      last = int(f.a);
      const u64 wc = max(w.fixed(r.x), u64(1));
      r.ties = (target - f.b + wc - 1) / wc;
    } else if (wcut > 0) {
      r.ties = min(r.ties, (target - above + wcut - 1) / wcut);
    }
  }
  // the kept values' weights, for the second pass
#pragma unroll 2
  for (int i = t; i <= last; i += kThreads) weight_of(i) = w.fixed(code_value(bin_code(i)));
  __syncthreads();
  return r;
}

// The row's token for a u outside (0, 1): the first or last kept one whose weight is positive
// in 64 bits.  Of the tokens at the cut those are kept before which there are
// fewer than `ties` in index order; `seen` of them come before this warp's run.  s.flag is 0.
template <typename T>
__device__ __noinline__ int end_of_kept(Row<T> w, float cut, u64 ties, u64 seen, bool last) {
  constexpr int VEC = Row<T>::VEC;
  uint32_t best = 0;  // ~index or index + 1: the largest is wanted
  w.visit([&](const float(&x)[VEC], int i) {
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) n += x[j] == cut;
    const u64 upto = seen + warp_scan(n);  // with this lane's own
    u64 at = upto - n;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const bool kept = x[j] > cut || (x[j] == cut && at < ties);
      at += x[j] == cut;
      if (kept && (double(x[j]) - w.md) * w.c > kLeastExponent)
        best = max(best, last ? uint32_t(i + j) + 1 : ~uint32_t(i + j));
    }
    seen = __shfl_sync(0xffffffffu, upto, 31);
  });
  best = __reduce_max_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0) atomicMax(&w.sp->flag, best);
  __syncthreads();
  const Slot* all = w.exchange(Slot{w.sp->flag, 0, 0});
  best = 0;  // the maximum is kept: some warp has one
  for (int q = 0; q < w.C; ++q) best = max(best, uint32_t(all[q].a));
  return int(last ? best - 1 : ~best);
}

// The least value whose weight is at least min_p, by steps from its closed form.
__device__ __noinline__ float least_kept(float m, double T, double min_p) {
  const double at = double(m) + T * log(min_p);
  if (!(at > -3e38)) return -INFINITY;
  const auto pass = [&](uint32_t key) {
    return exp((double(key_value(key)) - double(m)) / T) >= min_p;
  };
  uint32_t key = ord_key(float(at)) - 4;
  for (int i = 0; i < 12 && !pass(key); ++i) ++key;
  return key_value(key);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_tokens_kernel(const T* __restrict__ logits, const Params p) {
  __shared__ Shared s;
  extern __shared__ __align__(16) uint8_t dynamic_smem[];  // Queue; bf16: or ByValue
  constexpr bool kByValue = std::is_same<T, __nv_bfloat16>::value;
  ByValue& bv = *reinterpret_cast<ByValue*>(dynamic_smem);
  constexpr int VEC = Row<T>::VEC;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int r = blockIdx.x / p.C;
  Row<T> w;
  w.sp = &s;
  w.queue = reinterpret_cast<Queue*>(dynamic_smem);
  w.by_value = nullptr;
  w.C = p.C;
  w.rank = p.C > 1 ? int(cluster_rank()) : 0;
  w.turn = 0;
  w.row = logits + int64_t(r) * p.row_stride;
  w.special = false;
  const int origin = -int((reinterpret_cast<uintptr_t>(w.row) & 15) / sizeof(T));
  const int first = min(p.V, origin + w.rank * p.chunk), last = min(p.V, first + p.chunk);
  // every warp owns one run of the CTA's run, in steps of a warp's 512 bytes
  const int per_warp = ((last - first + kWarps - 1) / kWarps + 255) / 256 * 256;
  w.i0 = min(last, first + warp * per_warp);
  w.i1 = min(last, w.i0 + per_warp);

  cluster_started(p.C);
  if (t == 0) {
    s.flag = 0;
    // Read where a running sum reaches its target, as every target here is at most the sum of
    // its tokens.  Equal in all CTAs whatever happens: they must take the same barriers.
    s.found = s.found2 = Slot{0, 0, 0};
  }
  for (int i = t; i < kTable; i += kThreads)
    s.table[i] = exp2(double(i) / kTable) * double(1ull << kFrac);
  if constexpr (kByValue) {
    for (int i = t; i < kValues; i += kThreads) bv.positive[i] = bv.negative[i] = 0;
    if (t == 0) bv.n_listed = bv.refuse = 0;
  }
  w.clear();
  pdl_wait();  // programmatic launch: the logits come from the kernel before
  pdl_trigger();

  // This CTA's run on its way to L2 at once: the passes' own loads are too few in flight
  // to stream it from HBM.  (Whole 16-byte words of the run, 4 KB to a thread.)
  {
    const uintptr_t lo = (reinterpret_cast<uintptr_t>(w.row + max(first, 0)) + 15) & ~uintptr_t(15);
    const uintptr_t hi = reinterpret_cast<uintptr_t>(w.row + last) & ~uintptr_t(15);
    for (uintptr_t a = lo + uintptr_t(t) * 4096; a < hi; a += kThreads * 4096) {
      const uint32_t bytes = uint32_t(min(hi - a, uintptr_t(4096)));
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a), "r"(bytes) : "memory");
    }
  }

  // the row's settings, as one CTA reads them
  Slot mine{0, 0, 0};
  const float u = p.u[r];
  if (w.rank == 0) {
    mine.b = (u64(__float_as_uint(p.temperature[r])) << 32) |
             __float_as_uint(p.top_p ? p.top_p[r] : 1.f);
    mine.c = (u64(uint32_t(p.top_k ? p.top_k[r] : 0)) << 32) |
             __float_as_uint(p.min_p ? p.min_p[r] : 0.f);
  }
  float mx = -INFINITY;
  uint32_t special = 0;
  if constexpr (kByValue) {
    mx = count_values(reinterpret_cast<const uint16_t*>(w.row), w.i0, w.i1, bv);
  } else {
    w.visit([&](const float(&x)[VEC], int i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        mx = fmaxf(mx, x[j]);
        // adding one to the exponent carries into the sign's place when it is all ones
        const uint32_t e = (__float_as_uint(x[j]) & 0x7fffffffu) + 0x00800000u;
        special |= w.inside(i + j) ? e : 0;
      }
    });
    special &= 0x80000000u;
  }
  // the block's maximum and flags
  const auto block_max = [&](uint32_t key, uint32_t flags) -> u64 {
    key = __reduce_max_sync(0xffffffffu, key);
    flags = __reduce_or_sync(0xffffffffu, flags);
    __syncthreads();
    if (lane == 0) s.warp[warp] = (u64(flags) << 32) | key;
    __syncthreads();
    const u64 v = lane < kWarps ? s.warp[lane] : 0;
    return (u64(__reduce_or_sync(0xffffffffu, uint32_t(v >> 32))) << 32) |
           __reduce_max_sync(0xffffffffu, uint32_t(v));
  };
  mine.a = block_max(ord_key(mx), special != 0);
  if (kByValue && (bv.refuse || !(u > 0.f && u < 1.f))) mine.a |= 1ull << 32;
  cluster_wait_started(p.C);
  const Slot* all = w.exchange(mine);
  uint32_t top = 0;
  for (int q = 0; q < p.C; ++q) {
    top = max(top, uint32_t(all[q].a));
    w.special |= (all[q].a >> 32) != 0;
  }
  const float T_ = __uint_as_float(uint32_t(all[0].b >> 32));
  const float tp = __uint_as_float(uint32_t(all[0].b));
  const int k = int(uint32_t(all[0].c >> 32));
  const float mp = __uint_as_float(uint32_t(all[0].c));
  w.m = key_value(top);
  // values of -128 and below weigh less than half a unit
  const bool by_value = kByValue && !w.special && (w.m + 128.f) > 45.f * T_;
  if (kByValue && !by_value) w.special = true;  // not known: as if
  if (w.special) {  // the maximum of the sanitised values
    mx = -INFINITY;
    w.visit([&](const float(&x)[VEC], int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) mx = fmaxf(mx, x[j]);
    });
    all = w.exchange(Slot{block_max(ord_key(mx), 0), 0, 0});
    top = 0;
    for (int q = 0; q < p.C; ++q) top = max(top, uint32_t(all[q].a));
    w.m = key_value(top);
  }
  const float m = w.m;

  // the least index that passes a test, over the cluster
  const auto first_index = [&](auto test) -> int {
    uint32_t at = 0xffffffffu;
    w.visit([&](const float(&x)[VEC], int i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (test(x[j])) at = min(at, uint32_t(i + j));
    });
    const uint32_t least = ~uint32_t(block_max(~at, 0));
    const Slot* got = w.exchange(Slot{least, 0, 0});
    at = 0xffffffffu;
    for (int q = 0; q < p.C; ++q) at = min(at, uint32_t(got[q].a));
    return int(at);
  };
  if (!(T_ > 1e-6f) || k == 1 || tp <= 0.f || mp > 1.f) {  // one token is kept: the first maximum
    const int at = first_index([&](float x) { return x == m; });
    if (w.rank == 0 && t == 0) {
      p.out[r] = at;
      if (p.logprobs) p.logprobs[r] = 0.f;
    }
    return;
  }
  const double T64 = double(T_);
  w.c = 1.4426950408889634 / T64;
  w.md = double(m);
  w.dscale = float(1 << (2 * kBinBits)) / kCountWindow;

  float cut = -INFINITY;  // everything is above it
  u64 ties = ~0ull;
  const bool by_k = k > 0 && k < p.V, by_p = tp < 1.f;
  bool found = !by_k && !by_p;
  if constexpr (kByValue) {
    if (by_value && (!found || !(mp > 0.f))) {
      const Cuts c = p.C == 1   ? value_cuts<1>(w, bv, k, tp)
                     : p.C == 2 ? value_cuts<2>(w, bv, k, tp)
                     : p.C == 4 ? value_cuts<4>(w, bv, k, tp)
                                : value_cuts<8>(w, bv, k, tp);
      if (c.turn >= 0) {
        w.turn = c.turn;
        w.by_value = &bv;
        cut = c.x;
        ties = c.ties;
        found = true;
      } else {
        w.turn = -1 - c.turn;
        // counts by value leave masks out, so a row with -infinities comes here unsanitised;
        // the passes below count every token
        w.special = true;
        cluster_sync(p.C);  // no peer reads the counts any more: the queue lies over them
        w.clear();
      }
    }
  }
  if (!found) {
    if (by_k) {
      w.visit([&](const float(&x)[VEC], int) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int d = w.dist(x[j]);
          if (d >= 0) atomicAdd(&s.hist[0][d >> kBinBits], 1u);
        }
      });
      const Cut c = select_cut(w, true, u64(k), 0.f);
      w.turn = c.turn;
      cut = c.x;
      ties = u64(k) - c.above;
    }
    if (by_p) {
      w.dscale = float(double(1 << (2 * kBinBits)) / double(kWindow) / T64);
      // weights of the first n_k: all above the cut, and `ties` times the weight at it
      const Kept kept = sum_above(w, cut, true);
      all = w.exchange(Slot{block_scan(s, lane == 0 ? kept.sum : 0).total, 0, 0});
      u64 above = 0;
      for (int q = 0; q < p.C; ++q) above += all[q].a;
      const u64 wcut = cut == -INFINITY ? 0 : w.fixed(cut);
      const u64 z = above + (cut == -INFINITY ? 0 : ties * wcut);
      u64 target = u64(ceil(double(z) * double(tp)));
      if (target < 1) target = 1;
      if (target <= above) {  // else the boundary lies among the ties at the cut
        const Cut c = select_cut(w, false, target, cut);
        w.turn = c.turn;
        cut = c.x;
        const u64 wc = max(w.fixed(cut), u64(1));
        ties = (target - c.above + wc - 1) / wc;
      } else if (wcut > 0) {
        ties = min(ties, (target - above + wcut - 1) / wcut);
      }
    }
  }
  if (mp > 0.f) {
    float least = least_kept(m, T64, double(mp));
    if (kByValue && w.by_value) {  // up to a bf16 value: the second pass compares in bf16
      const uint32_t b = __float_as_uint(least);
      if (b & 0xffff) least = __uint_as_float((b & 0xffff0000u) + ((b >> 31) ? 0 : 0x10000u));
    }
    if (least > cut) {
      cut = least;
      ties = ~0ull;
    }
  }

  // weights of the kept tokens above the cut and the number at it, by warp and CTA
  Kept kept;
  if constexpr (kByValue)
    kept = w.by_value ? sum_above_by_value(w, cut) : sum_above(w, cut, false);
  else
    kept = sum_above(w, cut, false);
  const Scan ws = block_scan(s, lane == 0 ? kept.sum : 0);
  const Scan wt = block_scan(s, lane == 0 ? kept.ties : 0);
  all = w.exchange(Slot{ws.total, wt.total, __float_as_uint(u)});
  const float uu = __uint_as_float(uint32_t(all[0].c));
  const u64 wcut = cut == -INFINITY ? 0 : w.weight(cut);
  u64 before = 0, total = 0, t_before = 0, t_all = 0;
  for (int q = 0; q < p.C; ++q) {
    if (q < w.rank) {
      before += all[q].a;
      t_before += all[q].b;
    }
    total += all[q].a;
    t_all += all[q].b;
  }
  total += min(ties, t_all) * wcut;
  // lane 0's: what comes before this warp's run, and what the run holds
  before += ws.before;
  t_before += wt.before;
  const u64 ahead = before + min(ties, t_before) * wcut;
  const u64 after = before + kept.sum + min(ties, t_before + kept.ties) * wcut;
  const auto write = [&](int i, float x) {
    p.out[r] = i;
    if (p.logprobs)
      p.logprobs[r] =
          float((double(x) - double(m)) / T64 - log(double(total) / double(1ull << kFrac)));
  };
  if (!(uu > 0.f && uu < 1.f)) {
    const u64 seen = __shfl_sync(0xffffffffu, t_before, 0);
    const int i = end_of_kept(w, cut, ties, seen, uu >= 1.f);
    if (w.rank == 0 && t == 0) write(i, sanitize(Elem<T>::to_f32(w.row[i])));
    return;
  }
  const u64 target = u64(double(uu) * double(total));  // u < 1: below the total
  const auto weight = [&](float x) -> u64 {  // of a token above the cut
    if constexpr (kByValue) {
      const uint32_t code = __float_as_uint(x) >> 16;
      if (w.by_value && has_bin(code))
        return *reinterpret_cast<const u64*>(
            reinterpret_cast<const uint8_t*>(w.by_value->weight_positive) +
            (weight_offset(code) - 8 * kValueLo));
    }
    return fixed_call<T>(&s, w.md, w.c, x);
  };
  const auto at = [&](u64 above, u64 t_seen) { return above + min(ties, t_seen) * wcut; };
  // the token among this thread's [j0, j1), which begin after `before` and `t_before`
  const auto pick = [&](int j0, int j1) {
#pragma unroll 1
    for (int i = j0; i < j1; ++i) {
      const float x = sanitize(Elem<T>::to_f32(w.row[i]));
      t_before += x == cut;
      if (x > cut) before += weight(x);
      if (at(before, t_before) > target) {
        write(i, x);
        return;
      }
    }
  };
  if (per_warp <= 512) {
    // A short run: the warp whose it is walks it, 32 lanes x 16 bytes at a time.  (Runs of 2048
    // walked so: 64 bf16 rows of 128256 tokens 42 us instead of 36, fp32 100 instead of 88.)
    if (!__shfl_sync(0xffffffffu, ahead <= target && target < after, 0)) return;
    before = __shfl_sync(0xffffffffu, before, 0);
    t_before = __shfl_sync(0xffffffffu, t_before, 0);
    bool done = false;
    w.visit([&](const float(&x)[VEC], int i) {
      if (done) return;
      u64 sum = 0;
      uint32_t n = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        n += x[j] == cut;
        if (x[j] > cut) sum += weight(x[j]);
      }
      const u64 s_inc = warp_scan(sum), n_inc = warp_scan(n);
      const uint32_t hit =
          __ballot_sync(0xffffffffu, at(before + s_inc, t_before + n_inc) > target);
      if (hit) {
        done = true;
        if (lane == __ffs(hit) - 1) {
          before += s_inc - sum;
          t_before += n_inc - n;
          pick(max(i, 0), min(i + VEC, w.i1));
        }
      } else {
        before += __shfl_sync(0xffffffffu, s_inc, 31);
        t_before += __shfl_sync(0xffffffffu, n_inc, 31);
      }
    });
    return;
  }
  // A long one goes to the whole CTA, a few tokens per thread.
  if (lane == 0 && ahead <= target && target < after) {
    s.found = Slot{before, t_before, (u64(uint32_t(w.i0)) << 32) | uint32_t(w.i1)};
    s.flag = 1;
  }
  __syncthreads();
  if (!s.flag) return;  // another CTA's run
  before = s.found.a;
  t_before = s.found.b;
  const int run0 = int(s.found.c >> 32), run1 = int(uint32_t(s.found.c));
  const int share = ((run1 - run0 + kThreads - 1) / kThreads + VEC - 1) / VEC * VEC;
  const int j0 = min(run1, run0 + t * share), j1 = min(run1, j0 + share);
  u64 sum = 0, n_ties = 0;
#pragma unroll 1
  for (int i = j0; i < j1; i += VEC) {
    T e[VEC];
    if (i >= 0 && i + VEC <= j1) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(w.row + i));
      memcpy(e, &raw, 16);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = w.row[max(0, min(i + j, j1 - 1))];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float x = sanitize(Elem<T>::to_f32(e[j]));
      if (uint32_t(i + j) < uint32_t(j1)) {
        n_ties += x == cut;
        if (x > cut) sum += weight(x);
      }
    }
  }
  t_before += block_scan(s, n_ties).before;
  before += block_scan(s, sum).before;
  if (at(before, t_before) <= target && target < at(before + sum, t_before + n_ties))
    pick(max(j0, 0), j1);
}

static_assert(sizeof(Queue) <= sizeof(ByValue), "the queue lies over the counts");

// Rows of at most kSmall tokens: one CTA sorts (value descending, index ascending), and
// every filter is a length of the sorted row.  Against the clusters, 64 rows, top-k and
// top-p: 256 tokens 7 us (bf16 15, fp32 21), 1,000 13 (16, 20), 2,048 23 (15, 20).
constexpr int kSmall = 1024;
struct SmallShared {
  Shared s;  // block_scan's
  u64 key[kSmall];
  u64 weight[kSmall];  // by index
  u64 z;
  int n;
  uint32_t low, high;  // first and last kept index of positive weight
};

static_assert(sizeof(SmallShared) + 1024 <= 64 * 1024, "shared memory");

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_small_kernel(const T* __restrict__ logits, const Params p) {
  extern __shared__ __align__(16) uint8_t dynamic_smem[];
  SmallShared& sm = *reinterpret_cast<SmallShared*>(dynamic_smem);
  const int t = threadIdx.x, r = blockIdx.x, V = p.V;
  int N = 2;
  while (N < V) N *= 2;
  const int per = (N + kThreads - 1) / kThreads;  // places of a thread, side by side
  pdl_wait();
  pdl_trigger();
  const T* row = logits + int64_t(r) * p.row_stride;
  const float T_ = p.temperature[r], tp = p.top_p ? p.top_p[r] : 1.f;
  const float mp = p.min_p ? p.min_p[r] : 0.f, u = p.u[r];
  const int k = p.top_k ? p.top_k[r] : 0;
  for (int i = t; i < N; i += kThreads) {
    sm.key[i] = i < V ? (u64(ord_key(sanitize(Elem<T>::to_f32(row[i])))) << 32) | ~uint32_t(i) : 0;
    sm.weight[i] = 0;
  }
  if (t == 0) {
    sm.low = 0xffffffffu;
    sm.high = 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int size = 2; size <= N; size *= 2) {
#pragma unroll 1
    for (int step = size / 2; step > 0; step /= 2) {
      for (int j = t; j < N / 2; j += kThreads) {
        const int a = 2 * j - (j & (step - 1)), b = a + step;
        const u64 x = sm.key[a], y = sm.key[b];
        if ((x < y) == ((a & size) == 0)) {  // descending runs first
          sm.key[a] = y;
          sm.key[b] = x;
        }
      }
      __syncthreads();
    }
  }
  const auto value = [&](int i) { return key_value(uint32_t(sm.key[i] >> 32)); };
  const auto index = [&](int i) { return int(~uint32_t(sm.key[i])); };
  const float m = value(0);
  if (!(T_ > 1e-6f) || k == 1 || tp <= 0.f || mp > 1.f) {
    if (t == 0) {
      p.out[r] = index(0);
      if (p.logprobs) p.logprobs[r] = 0.f;
    }
    return;
  }
  const double T64 = double(T_), c = 1.4426950408889634 / T64, one = double(1ull << kFrac);
  const int n_k = k > 0 && k < V ? k : V;
  // weights in the sorted order, and how many pass min-p
  u64 w[kSmall / kThreads] = {}, sum = 0, pass = 0;
  uint32_t positive = 0;
  for (int e = 0; e < per; ++e) {
    const int i = t * per + e;
    if (i >= n_k) break;
    const double d = double(value(i)) - double(m), x = exp(d / T64);
    w[e] = u64(__double2ll_rn(x * one));
    sum += w[e];
    pass += !(mp > 0.f) || x >= double(mp);
    positive |= uint32_t(d * c > kLeastExponent) << e;  // exp may give 0 for the smallest
  }
  const Scan ws = block_scan(sm.s, sum);
  int n = max(1, int(min(block_scan(sm.s, pass).total, u64(n_k))));
  if (tp < 1.f) {
    const u64 target = max(u64(ceil(double(ws.total) * double(tp))), u64(1));
    if (t == 0) sm.n = n_k;
    __syncthreads();
    u64 run = ws.before;
    for (int e = 0; e < per; ++e) {
      if (run < target && run + w[e] >= target) sm.n = t * per + e + 1;
      run += w[e];
    }
    __syncthreads();
    n = min(n, sm.n);
  }
  // the kept weights by index
  for (int e = 0; e < per; ++e) {
    const int i = t * per + e;
    if (i >= n) break;
    sm.weight[index(i)] = w[e];
    if (positive >> e & 1) {
      atomicMin(&sm.low, uint32_t(index(i)));
      atomicMax(&sm.high, uint32_t(index(i)));
    }
  }
  __syncthreads();
  sum = 0;
  for (int e = 0; e < per && t * per + e < V; ++e) sum += sm.weight[t * per + e];
  const Scan is = block_scan(sm.s, sum);
  const auto write = [&](int i) {
    const float x = sanitize(Elem<T>::to_f32(row[i]));
    p.out[r] = i;
    if (p.logprobs)
      p.logprobs[r] = float((double(x) - double(m)) / T64 - log(double(is.total) / one));
  };
  if (!(u > 0.f && u < 1.f)) {
    if (t == 0) write(int(u >= 1.f ? sm.high : sm.low));
    return;
  }
  const u64 target = u64(double(u) * double(is.total));  // u < 1: below the total
  if (!(is.before <= target && target < is.before + sum)) return;
  u64 run = is.before;
  for (int i = t * per; i < V; ++i) {
    run += sm.weight[i];
    if (run > target) {
      write(i);
      return;
    }
  }
}

template <typename T>
cudaLaunchConfig_t launch_config(int clusters, int C, cudaLaunchAttribute* attr,
                                 cudaStream_t stream = nullptr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(clusters) * C);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.dynamicSmemBytes = std::is_same<T, __nv_bfloat16>::value ? sizeof(ByValue) : sizeof(Queue);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  return cfg;
}

// Clusters of C CTAs that the device holds at once, asked for once (148 SMs: 148 of 2, 71 of
// 4, 33 of 8; fewer than the CTAs' own 296 would give).
template <typename T>
int resident_clusters(int C) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kMaxCluster + 1];
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (dev < kDevices && (n = known[dev][C].load(std::memory_order_relaxed)) > 0) return n;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = launch_config<T>(1, C, attr);
  if (cudaOccupancyMaxActiveClusters(&n, sample_tokens_kernel<T>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (dev < kDevices) known[dev][C].store(n, std::memory_order_relaxed);
  return n;
}

// CTAs of a row's cluster: as many as leave the rows' clusters all resident, with at least
// 2048 tokens each so that the exchanges do not outweigh the work, and at most kMaxRun.
// Rows in bf16, whose passes are short, keep an SM to each CTA.  Measured, us, top-p 0.9:
//   rows x tokens           C = 1   2    4    8
//   fp32  14 x 128256       188   107   64   43
//   fp32  36 x 128256       188   106   86   92
//   fp32  72 x 128256       188   107  133  145
//   bf16  14 x 128256        51    34   24   19
//   bf16  24 x 32003         24    19   17   18
//   bf16  64 x 128256        52    34   37   52
//   bf16 148 x 32003         25    26   50   79
template <typename T>
int cluster_size(int rows, int vocab) {
  const int share = std::is_same<T, __nv_bfloat16>::value ? 2 : 1;
  int c = 1;
  while (c < kMaxCluster &&
         ((vocab / (2 * c) >= 2048 && int64_t(rows) * share <= resident_clusters<T>(2 * c)) ||
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
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto tag) -> int {
    using T = decltype(tag);
    if (vocab <= kSmall) {
      cudaFuncSetAttribute(sample_small_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           int(sizeof(SmallShared)));
      launch_pdl(sample_small_kernel<T>, dim3(unsigned(num_rows)), dim3(kThreads),
                 sizeof(SmallShared), s, static_cast<const T*>(logits), p);
      return check_launch("as_sample_tokens");
    }
    cudaFuncSetAttribute(
        sample_tokens_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
        int(std::is_same<T, __nv_bfloat16>::value ? sizeof(ByValue) : sizeof(Queue)));
    p.C = cluster_size<T>(num_rows, vocab);
    const int lead = 16 / int(sizeof(T)) - 1;  // at most: from a boundary to the row
    p.chunk = ((vocab + lead + p.C - 1) / p.C + 255) / 256 * 256;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = launch_config<T>(num_rows, p.C, attr, s);
    cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T>, static_cast<const T*>(logits), p);
    return check_launch("as_sample_tokens");
  };
  switch (dtype) {
    case AS_DTYPE_F32: return run(float());
    case AS_DTYPE_F16: return run(__half());
    default: return run(__nv_bfloat16());
  }
}
