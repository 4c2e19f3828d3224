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
// No sort: every filter keeps a prefix of one order, so a threshold on (x, number of
// ties at x) describes it, and the threshold is found by histograms over a monotone
// integer distance from the maximum, refined until one value is left.
//
// Sums decide between neighbouring tokens, and a boundary token can weigh 1e-6 of the
// total: weights are computed in 64 bits and summed in 64-bit fixed point (2^-45 at
// 128K tokens), which also makes every sum independent of the order of the atomics.
#include "common.cuh"
#include "host_util.h"

namespace asb {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;           // two bins per thread
constexpr int kDistBits = 22;         // distance Q: two histogram levels of 11 bits
constexpr float kDistRange = 32.f;    // nats covered by Q before it saturates
constexpr int kMaxVocab = 1 << 24;

__device__ __forceinline__ float sanitize(float v) {
  if (v != v) return 0.f;
  if (v == INFINITY) return 1e4f;
  if (v == -INFINITY) return -1e4f;
  return v == 0.f ? 0.f : v;  // -0 ties with +0
}
// Order-preserving bits of an fp32 value.
__device__ __forceinline__ uint32_t ord_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// Calls f(x, index) for the elements [i0, i1) of a row, 32 lanes x 16 bytes at a time.
template <typename T, typename F>
__device__ __forceinline__ void visit(const T* __restrict__ row, int i0, int i1, bool vec, F f) {
  constexpr int VEC = 16 / int(sizeof(T));
  const int lane = threadIdx.x & 31;
  for (int base = i0 + lane * VEC; base < i1; base += 32 * VEC) {
    if (vec && base + VEC <= i1) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + base));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f(sanitize(Elem<T>::to_f32(e[j])), base + j);
    } else {
      for (int j = 0; j < VEC && base + j < i1; ++j)
        f(sanitize(Elem<T>::to_f32(row[base + j])), base + j);
    }
  }
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Shared {
  unsigned long long hist[kBins];
  unsigned long long warp[kWarps];
  unsigned long long before;  // sum of everything above the chosen bin
  uint32_t lo, hi;
  int bin;
};

// Sum over the block; every thread gets it.
__device__ unsigned long long block_sum(Shared& s, unsigned long long v) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long t = 0;
  for (int w = 0; w < kWarps; ++w) t += s.warp[w];
  return t;
}

// First bin at which acc + (sums of bins up to it) reaches target, and the sum before it.
__device__ void find_bin(Shared& s, unsigned long long acc, unsigned long long target) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  __syncthreads();
  const unsigned long long a = s.hist[2 * t], b = s.hist[2 * t + 1];
  unsigned long long inc = a + b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) s.warp[warp] = inc;
  if (t == 0) {
    s.bin = 0;
    s.before = acc;
  }
  __syncthreads();
  unsigned long long base = acc;
  for (int w = 0; w < warp; ++w) base += s.warp[w];
  const unsigned long long e0 = base + inc - a - b;  // before bin 2t
  if (e0 < target && e0 + a >= target) {
    s.bin = 2 * t;
    s.before = e0;
  } else if (e0 + a < target && e0 + a + b >= target) {
    s.bin = 2 * t + 1;
    s.before = e0 + a;
  }
  __syncthreads();
}

// The threshold of a filter: keys above `key` are kept, and of those equal to it the
// first `ties` in index order.
struct Cut {
  uint32_t key;
  unsigned long long above;  // summed measure of the keys above it
};

// Finds the key at which the running measure (count or weight, in the descending
// order) reaches `target`; the caller guarantees that the whole row's measure does.
// measure(x, key) is 0 for tokens out of the running.
template <typename T, typename M>
__device__ Cut select_cut(Shared& s, const T* row, int i0, int i1, bool vec, float m, float dscale,
                          unsigned long long target, M measure) {
  auto dist = [&](float x) -> int {
    const float y = (m - x) * dscale;
    return y >= float((1 << kDistBits) - 1) ? (1 << kDistBits) - 1 : int(y);
  };
  auto clear = [&]() {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.hist[i] = 0;
    __syncthreads();
  };
  unsigned long long acc = 0;
  clear();
  visit(row, i0, i1, vec, [&](float x, int) {
    const unsigned long long v = measure(x, ord_key(x));
    if (v) atomicAdd(&s.hist[dist(x) >> 11], v);
  });
  find_bin(s, acc, target);
  const int b1 = s.bin;
  acc = s.before;
  clear();
  visit(row, i0, i1, vec, [&](float x, int) {
    const int q = dist(x);
    if ((q >> 11) != b1) return;
    const unsigned long long v = measure(x, ord_key(x));
    if (v) atomicAdd(&s.hist[q & 2047], v);
  });
  find_bin(s, acc, target);
  const int q = (b1 << 11) | s.bin;
  acc = s.before;
  // keys at this distance
  __syncthreads();
  if (threadIdx.x == 0) {
    s.lo = 0xffffffffu;
    s.hi = 0;
  }
  __syncthreads();
  visit(row, i0, i1, vec, [&](float x, int) {
    if (dist(x) != q || !measure(x, ord_key(x))) return;
    atomicMin(&s.lo, ord_key(x));
    atomicMax(&s.hi, ord_key(x));
  });
  __syncthreads();
  uint32_t lo = s.lo, hi = s.hi;
  // a 32-bit key takes three levels of 11 bits at most (the bound also ends the loop
  // should another stream rewrite the logits meanwhile)
  for (int level = 0; lo < hi && level < 3; ++level) {
    int shift = 0;
    while (((hi - lo) >> shift) >= uint32_t(kBins)) ++shift;
    clear();
    visit(row, i0, i1, vec, [&](float x, int) {
      const uint32_t k = ord_key(x);
      if (k < lo || k > hi) return;
      const unsigned long long v = measure(x, k);
      if (v) atomicAdd(&s.hist[(hi - k) >> shift], v);
    });
    find_bin(s, acc, target);
    acc = s.before;
    const uint32_t top = hi - (uint32_t(s.bin) << shift);
    const uint32_t width = (1u << shift) - 1;
    lo = top - lo > width ? top - width : lo;
    hi = top;
  }
  return Cut{hi, acc};
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_tokens_kernel(int64_t* __restrict__ out, float* __restrict__ logprobs,
                     const T* __restrict__ logits, int64_t row_stride, int V,
                     const float* __restrict__ u, const float* __restrict__ temperature,
                     const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                     const float* __restrict__ min_p, int frac_bits) {
  __shared__ Shared s;
  const int r = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* row = logits + int64_t(r) * row_stride;
  const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
  // every warp owns one run of indexes, so sums per warp are sums in index order
  const int chunk = ((V + kWarps - 1) / kWarps + 255) / 256 * 256;
  const int i0 = min(V, warp * chunk), i1 = min(V, i0 + chunk);

  unsigned long long best = 0;
  visit(row, i0, i1, vec, [&](float x, int i) {
    const unsigned long long k =
        (static_cast<unsigned long long>(ord_key(x)) << 32) | (0xFFFFFFFFu - uint32_t(i));
    best = k > best ? k : best;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
    best = k > best ? k : best;
  }
  if (lane == 0) s.warp[warp] = best;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) best = s.warp[w] > best ? s.warp[w] : best;
  const float m = key_value(uint32_t(best >> 32));

  const float T_ = temperature[r];
  const int k = top_k ? top_k[r] : 0;
  const float p = top_p ? top_p[r] : 1.f;
  const float mp = min_p ? min_p[r] : 0.f;
  if (!(T_ > 1e-6f) || k == 1 || p <= 0.f || mp > 1.f) {  // only the first token is kept
    if (threadIdx.x == 0) {
      out[r] = int64_t(0xFFFFFFFFu - uint32_t(best & 0xFFFFFFFFull));
      if (logprobs) logprobs[r] = 0.f;
    }
    return;
  }
  const double inv_t = 1.0 / double(T_);
  const float dscale = float(double(1 << kDistBits) / double(kDistRange) * inv_t);
  const double one = double(1ull << frac_bits);
  auto weight = [&](float x) -> double { return exp((double(x) - double(m)) * inv_t); };
  // a token of positive weight counts at least one unit, so u = 0 can reach it
  auto fixed = [&](float x) -> unsigned long long {
    const double w = weight(x);
    const unsigned long long f = static_cast<unsigned long long>(__double2ll_rn(w * one));
    return f == 0 && w > 0.0 ? 1 : f;
  };

  uint32_t cut = 0;  // smallest key kept; of the tokens equal to it, `ties` are
  unsigned long long ties = ~0ull;
  if (k > 0 && k < V) {
    const Cut c = select_cut(s, row, i0, i1, vec, m, dscale, static_cast<unsigned long long>(k),
                             [&](float, uint32_t) { return 1ull; });
    cut = c.key;
    ties = static_cast<unsigned long long>(k) - c.above;
  }
  if (p < 1.f) {
    // weights of the first n_k: all above the cut, and `ties` times the weight at it
    unsigned long long z = 0;
    visit(row, i0, i1, vec, [&](float x, int) {
      if (ord_key(x) > cut) z += fixed(x);
    });
    z = block_sum(s, z);
    const unsigned long long wcut = cut ? fixed(key_value(cut)) : 0;
    if (cut) z += ties * wcut;
    const unsigned long long target =
        static_cast<unsigned long long>(ceil(double(z) * double(p)));
    const unsigned long long above_cut = cut ? z - ties * wcut : z;
    if (target <= above_cut) {  // else the boundary lies among the ties at the cut
      const Cut c = select_cut(s, row, i0, i1, vec, m, dscale, target > 0 ? target : 1,
                               [&](float x, uint32_t key) { return key > cut ? fixed(x) : 0ull; });
      cut = c.key;
      const unsigned long long w = fixed(key_value(cut));
      ties = (target - c.above + w - 1) / w;
    } else {
      const unsigned long long need = (target - above_cut + wcut - 1) / wcut;
      ties = need < ties ? need : ties;
    }
  }
  // min-p is a threshold on the weight alone
  const double mpd = double(mp);
  auto above = [&](float x) { return ord_key(x) > cut && (!(mp > 0.f) || weight(x) >= mpd); };
  const bool cut_kept = cut != 0 && (!(mp > 0.f) || weight(key_value(cut)) >= mpd);
  const unsigned long long wcut = cut_kept ? fixed(key_value(cut)) : 0;

  // how many of the ties lie before this warp's run
  unsigned long long tie_count = 0;
  if (cut_kept) {
    visit(row, i0, i1, vec, [&](float x, int) { tie_count += ord_key(x) == cut; });
    tie_count = warp_sum(tie_count);
  }
  __syncthreads();
  if (lane == 0) s.warp[warp] = tie_count;
  __syncthreads();
  unsigned long long ties_before = 0;
  for (int w = 0; w < warp; ++w) ties_before += s.warp[w];
  unsigned long long quota = ties > ties_before ? ties - ties_before : 0;
  if (quota > tie_count) quota = tie_count;

  unsigned long long sum = 0;
  visit(row, i0, i1, vec, [&](float x, int) {
    if (above(x)) sum += fixed(x);
  });
  sum = warp_sum(sum) + quota * wcut;
  __syncthreads();
  if (lane == 0) s.warp[warp] = sum;
  __syncthreads();
  unsigned long long before = 0, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s.warp[w];
    total += s.warp[w];
  }
  const float uu = u[r];
  // u outside [0, 1): the first / last kept token of positive weight
  unsigned long long target = uu > 0.f ? static_cast<unsigned long long>(double(uu) * double(total)) : 0;
  if (target >= total) target = total - 1;
  if (!(before <= target && target < before + sum)) return;
  // this warp's run holds the token: walk it 32 elements at a time
  unsigned long long c = before;
  for (int base = i0; base < i1; base += 32) {
    const int i = base + lane;
    const float x = i < i1 ? sanitize(Elem<T>::to_f32(row[i])) : 0.f;
    const bool in = i < i1;
    const bool tie = in && cut_kept && ord_key(x) == cut;
    const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
    const bool kept = in && (above(x) || (tie && __popc(tie_mask & ((1u << lane) - 1)) < quota));
    unsigned long long w = kept ? fixed(x) : 0;
    unsigned long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, c + inc > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        out[r] = i;
        if (logprobs) logprobs[r] = float((double(x) - double(m)) * inv_t - log(double(total) / one));
      }
      return;
    }
    c += __shfl_sync(0xffffffffu, inc, 31);
    const uint32_t n_tie = __popc(tie_mask);
    quota -= quota < n_tie ? quota : n_tie;
  }
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
  if (num_rows == 0) return AS_OK;
  if (!out || !logits || !u || !temperature)
    return fail(AS_ERR_INVALID_ARG, "as_sample_tokens: null pointer");
  if (reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype))
    return fail(AS_ERR_INVALID_ARG, "as_sample_tokens: logits are not aligned to their type");
  // the sum of `vocab` weights of at most 1 stays below 2^62
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  const int frac = 62 - bits;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto tag) -> int {
    using T = decltype(tag);
    sample_tokens_kernel<T><<<num_rows, kThreads, 0, s>>>(
        out, logprobs, static_cast<const T*>(logits), row_stride, vocab, u, temperature, top_k,
        top_p, min_p, frac);
    return check_launch("as_sample_tokens");
  };
  switch (dtype) {
    case AS_DTYPE_F32: return run(float());
    case AS_DTYPE_F16: return run(__half());
    default: return run(__nv_bfloat16());
  }
}
