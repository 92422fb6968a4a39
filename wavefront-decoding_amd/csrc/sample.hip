// Drawing tokens from logits: temperature, top-k, top-p, min-p, and a uniform
// number per row that the caller gives.
//
// With w_j = 2^((l_j - max l) log2(e) / T) and the tokens ordered by (l
// descending, j ascending), the kept tokens are a prefix of that order: the
// first k; of these the shortest prefix with sum w >= p * (their sum); of these
// the ones with w >= min_p (the first always). The token is the lowest kept j
// with sum of w over the kept tokens up to j > u * (their sum).
//
// Every comparison is between sums over up to the whole vocabulary, so how the
// sums are rounded decides tokens: w is computed in fp64 (which runs at the
// fp32 rate here) and held as an integer multiple of 2^-44. Integer sums do not
// depend on their order, so a token depends on its row alone -- not on the
// kernel's layout, the companions or the run -- and a border is off by 2^-45 per
// token. u, p and their products with the sums are exact (64 x 64 -> 128 bits).
//
// One workgroup per row. Where the kept tokens are few -- top-k, or a top-p whose
// tokens hold enough of the weight -- they are found without ordering the row: of
// the 1024 threads' largest logits, at least k are no smaller than the k-th, so
// every one of the first k tokens is at or above it, and few others are. Those go
// to a list in LDS, which is sorted (one entry a thread), and top-k, top-p and
// min_p are positions in it.
// Otherwise a histogram of the logits' distance from the largest says which of
// 1024 bins the last kept token lies in, by count or by weight, and a radix select
// over that bin's tokens (over the row, if they are too many) finds its key; ties
// with it are kept in index order.
#include "wfd_common.h"

namespace wfd {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmChunk = 4 * kSmThreads;  // logits per round of the workgroup, 4 consecutive ones a thread
constexpr int kSmMaxVocab = 1 << 19;      // sums of 2^19 weights of 2^44 fit 63 bits
constexpr double kSmOne = 17592186044416.0;  // 2^44

// Keys order as the logits do; -0 is +0; 0 is below every logit's key.
__device__ __forceinline__ uint32_t sm_key(float l) {
  const uint32_t b = __float_as_uint(l + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float sm_logit(uint32_t key) {
  return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
}

__device__ __forceinline__ uint64_t sm_shfl_xor(uint64_t v, int m) {
  return (uint64_t)__shfl_xor((unsigned long long)v, m, 64);
}
__device__ __forceinline__ uint64_t sm_shfl_up(uint64_t v, int m) {
  return (uint64_t)__shfl_up((unsigned long long)v, m, 64);
}

struct SmArgs {
  const float* logits;
  int64_t ld;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int64_t *out, *ring;
  const int32_t* ring_rows;
  int64_t ring_len;
  const int64_t* expect;
  int32_t* accept;
  int V;
};

constexpr int kSmBins = 1024;   // one per thread
constexpr int kSmList = 2048;
constexpr int kSmSort = kSmThreads;  // entries of a list that is sorted
constexpr int kSmGuess = 600;        // top-k up to which the list is tried: ~900 tokens are then above the k-th thread's
constexpr float kSmMasked = -1e4f;  // logits down to here spread the bins; the others share the last

__device__ __forceinline__ uint64_t sm_wave_sum(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += sm_shfl_xor(v, m);
  return v;
}

// 2^x for x <= 0 in units of 2^-44, rounded to nearest: x = m / 32 + r, 2^r by its
// series to r^5 (the rest is below 3e-15 of it), 2^(m / 32) from the table with
// the exponent added to its bits. Adding 1.5 2^52 (2^52) leaves the nearest integer
// in the low bits of the sum.
__device__ __forceinline__ uint64_t sm_exp2(double x, const double* __restrict__ tab) {
  x = fmax(x, -900.);  // also of NaN; far below the least weight
  const double t = fma(x, 32., 6755399441055744.);
  const int k = (int)(uint32_t)__double_as_longlong(t);
  const double r = fma(t - 6755399441055744., -0.03125, x);
  double p = fma(r, 0.0013333558146428443, 0.009618129107628477);
  p = fma(p, r, 0.05550410866482158);
  p = fma(p, r, 0.24022650695910072);
  p = fma(p, r, 0.6931471805599453);
  p = fma(p, r, 1.0);
  const double two = __longlong_as_double(__double_as_longlong(tab[k & 31]) + ((long long)((k >> 5) + 44) << 52));
  return (uint64_t)__double_as_longlong(fma(p, two, 4503599627370496.)) & 0xfffffffffffffull;
}

// floor(s f) for f in [0, 1), and whether anything was cut off
__device__ __forceinline__ uint64_t sm_mul_frac(uint64_t s, float f, bool& rest) {
  const uint64_t q = (uint64_t)((double)f * 18446744073709551616.0);
  rest = s * q != 0;
  return __umul64hi(s, q);
}

// CAP > 0: the row is kept in LDS (V <= CAP); 0: it is read again in every pass
// (from L2). In registers, 32 logits a thread, the passes' code spilled.
template <int CAP>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SmArgs a) {
  __shared__ unsigned long long hist[kSmBins];
  __shared__ unsigned long long seg[(CAP > 0 ? CAP : kSmMaxVocab) / 256];  // the running sums' steps, in index order
  __shared__ __align__(16) u32x4 keep[CAP > 0 ? CAP / 4 : 1];
  __shared__ uint32_t list_key[kSmList];
  __shared__ uint32_t list_idx[kSmList];
  __shared__ double tab[32];
  __shared__ float s_max[kSmWaves], s_min[kSmWaves];
  __shared__ unsigned long long s_sum[kSmWaves];
  __shared__ uint32_t s_lo[kSmWaves], s_hi[kSmWaves];
  __shared__ unsigned long long s_u64;
  __shared__ uint32_t s_u32, s_count;
  const int i = blockIdx.x;
  const int t = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int V = a.V;
  const float* row = a.logits + (int64_t)i * a.ld;
  const bool vec = ((uintptr_t)row & 15) == 0;
  // wave w holds the logits [w per_wave, (w + 1) per_wave): index order is wave, round, lane
  const int per_wave = (V + 63) / 64 * 4;
  const int w_end = min((wave + 1) * per_wave, V);
  const int nchunks = (per_wave + 255) / 256;
  auto first_of = [&](int c) { return wave * per_wave + 256 * c + 4 * lane; };

  auto fetch = [&](int c, float (&x)[4]) {  // 4 logits; -inf past the wave's
    const int e = first_of(c);
    if (vec && e + 4 <= w_end) {
      Elem<float>::unpack(ld16(row + e), x);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = e + k < w_end ? row[e + k] : -INFINITY;
    }
  };
  if constexpr (CAP > 0) {  // every load first; a thread reads back only what it stores
    float x[CAP / kSmChunk][4];
#pragma unroll
    for (int c = 0; c < CAP / kSmChunk; ++c) fetch(c, x[c]);
#pragma unroll
    for (int c = 0; c < CAP / kSmChunk; ++c) keep[c * kSmThreads + t] = Elem<float>::pack(x[c]);
  }
  if (t < 32) tab[t] = exp2((double)t * 0.03125);
  // f(first index, the 4 logits) over the row, in index order per thread; -inf fills the
  // places past the wave's share, which no weight, bin or key below counts
  auto each = [&](auto f) {
    float x[4];
    if constexpr (CAP > 0) {
      for (int c = 0; c < nchunks; ++c) {
        Elem<float>::unpack(keep[c * kSmThreads + t], x);
        f(first_of(c), x);
      }
    } else {
      fetch(0, x);
      for (int c = 0; c < nchunks; ++c) {  // a chunk ahead
        float y[4];
        fetch(min(c + 1, nchunks - 1), y);
        f(first_of(c), x);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = y[k];
      }
    }
  };

  // the largest logit (of the thread, of the row), whether there is a NaN, the range of the bins
  float mine = -INFINITY, low = INFINITY;
  bool nan = false;
  each([&](int, const float (&x)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      nan |= x[q] != x[q];
      mine = fmaxf(mine, x[q]);
      low = fminf(low, x[q] > kSmMasked ? x[q] : INFINITY);
    }
  });
  float best = mine;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    best = fmaxf(best, __shfl_xor(best, m, 64));
    low = fminf(low, __shfl_xor(low, m, 64));
  }
  nan = __ballot(nan) != 0;
  if (lane == 0) {
    s_max[wave] = nan ? __uint_as_float(0x7fc00000u) : best;
    s_min[wave] = low;
  }
  __syncthreads();
  nan = false;
#pragma unroll
  for (int w = 0; w < kSmWaves; ++w) {
    nan |= s_max[w] != s_max[w];
    best = fmaxf(best, s_max[w]);
    low = fminf(low, s_min[w]);
  }

  const float T = a.temperature ? a.temperature[i] : 1.f;
  if (nan || !(T > 0.f) || best == -INFINITY) {  // uniform
    // greedy rows: the first of the largest; a row with a NaN: its first, visibly, as
    // in wfd_argmax; a row without any possible token: 0
    int bi = 0x7fffffff;
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 3; q >= 0; --q)
        if (e + q < w_end && (nan ? x[q] != x[q] : x[q] == best)) bi = min(bi, e + q);
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) bi = min(bi, __shfl_xor(bi, m, 64));
    if (lane == 0) s_lo[wave] = (uint32_t)bi;
    __syncthreads();
    if (t == 0) {
      for (int w = 0; w < kSmWaves; ++w) bi = min(bi, (int)s_lo[w]);
      argmax_finish(i, bi, a.out, a.ring, a.ring_rows, a.ring_len, a.expect, a.accept);
    }
    return;
  }
  const double inv = fmin(1.4426950408889634 / (double)T, 1e300);  // finite: 0 times it is 0
  const bool endless = best == INFINITY;  // infinite logits share everything
  auto weight = [&](float l) -> uint64_t {
    if (endless) return l == best ? (uint64_t)kSmOne : 0;
    return sm_exp2(((double)l - (double)best) * inv, tab);  // of the largest itself: exactly one
  };
  const int k = a.top_k ? a.top_k[i] : 0;
  const bool has_k = k > 0 && k < V;
  const float p = a.top_p ? a.top_p[i] : 1.f;
  const bool has_p = p < 1.f;
  const float minp = a.min_p ? a.min_p[i] : 0.f;
  // min_p on the integer weights' scale: w >= min_p for w on or above it
  const uint64_t wmin = minp > 0.f ? (minp < 1.f ? (uint64_t)ceil((double)minp * kSmOne) : (uint64_t)kSmOne) : 0;
  float u = a.u[i];
  u = u > 0.f ? (u < 1.f ? u : 0.99999994f) : 0.f;

  auto block_sum = [&](uint64_t v) -> uint64_t {
    v = sm_wave_sum(v);
    __syncthreads();
    if (lane == 0) s_sum[wave] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int w = 0; w < kSmWaves; ++w) s += s_sum[w];
    return s;
  };
  // The sum of the threads' v before this one.
  auto block_scan = [&](uint64_t v) -> uint64_t {
    uint64_t inc = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const uint64_t o = sm_shfl_up(inc, m);
      if (lane >= m) inc += o;
    }
    __syncthreads();
    if (lane == 63) s_sum[wave] = inc;
    __syncthreads();
    uint64_t before = lane < wave ? (uint64_t)s_sum[lane] : 0;  // 16 waves
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) before += sm_shfl_xor(before, m);
    return (uint64_t)__shfl((unsigned long long)before, 0, 64) + inc - v;
  };
  // The bin (thread t holds bin t's sum v) in which base plus the running sum reaches need; before: the sum before it.
  auto find_bin = [&](uint64_t v, uint64_t base, uint64_t need, uint64_t& before) -> uint32_t {
    const uint64_t run = base + block_scan(v);
    if (run < need && run + v >= need) {
      s_u32 = t;
      s_u64 = run;
    }
    __syncthreads();
    before = s_u64;
    return s_u32;
  };

  // Kept so far: keys above kk, and the first `ties` tokens with key kk.
  uint32_t kk = 0;
  uint64_t ties = 0, ties_left = 0;  // and the ones with key kk that are not

  // The shortest prefix of the kept tokens whose measure (1 or the weight), on
  // top of base, reaches need. over(f) calls f(key) for tokens that include all
  // that may end it; equal keys may all be there, the kept ties count as ties.
  auto refine = [&](auto over, uint64_t base, uint64_t need, bool by_weight) {
    const uint32_t k0 = kk;
    const uint64_t t0 = ties;
    uint32_t lo = 0xffffffffu, hi = 0;
    over([&](uint32_t key) {
      if (key > k0 || (t0 && key == k0)) {
        lo = min(lo, key);
        hi = max(hi, key);
      }
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      lo = min(lo, (uint32_t)__shfl_xor((int)lo, m, 64));
      hi = max(hi, (uint32_t)__shfl_xor((int)hi, m, 64));
    }
    __syncthreads();
    if (lane == 0) {
      s_lo[wave] = lo;
      s_hi[wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSmWaves; ++w) {
      lo = min(lo, s_lo[w]);
      hi = max(hi, s_hi[w]);
    }
    // digits of hi - key, so that larger keys come first
    const int bits = 32 - __clz((int)((hi - lo) | 1u));
    int shift = bits;
    uint32_t prefix = 0;
    while (shift > 0) {  // uniform
      const int width = min(10, shift), next = shift - width;
      const uint32_t mask = (1u << width) - 1;
      __syncthreads();
      hist[t] = 0;
      __syncthreads();
      auto add = [&](uint32_t key, uint64_t m) {
        const uint32_t off = hi - key;
        if (shift == bits || off >> shift == prefix) atomicAdd(&hist[(off >> next) & mask], (unsigned long long)m);
      };
      over([&](uint32_t key) {
        if (key > k0 && key >= lo && key <= hi) {
          const uint64_t m = by_weight ? weight(sm_logit(key)) : 1;
          if (m) add(key, m);
        }
      });
      if (t == 0 && t0 && k0 >= lo && k0 <= hi) add(k0, t0 * (by_weight ? weight(sm_logit(k0)) : 1));
      __syncthreads();
      const uint32_t d = find_bin(hist[t], base, need, base);
      prefix = (prefix << width) | d;
      shift = next;
    }
    kk = hi - prefix;
    const uint64_t one = by_weight ? weight(sm_logit(kk)) : 1;
    ties = (need - base + one - 1) / one;  // >= 1; no more than there are, since they reach need
    uint64_t equal = 0;
    over([&](uint32_t key) { equal += key == kk; });
    ties_left = block_sum(equal) - ties;
  };

  const float scale = best > low ? (float)(kSmBins - 2) / (best - low) : 1.f;
  auto bin_of = [&](float l) -> int { return l == best ? 0 : (int)fminf((best - l) * scale, (float)(kSmBins - 1)); };
  // Tokens of bins [b0, b1] to the list; false if they are too many.
  int nlist = 0;
  auto collect = [&](int b0, int b1, uint32_t room = kSmList) -> bool {
    __syncthreads();
    if (t == 0) s_count = 0;
    __syncthreads();
    each([&](int e, const float (&x)[4]) {
      bool in[4];
      int n_in = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int b = bin_of(x[q]);
        in[q] = e + q < w_end && b >= b0 && b <= b1;
        n_in += in[q];
      }
      if (n_in) {
        uint32_t at = atomicAdd(&s_count, (uint32_t)n_in);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (in[q]) {
            if (at < kSmList) {
              list_key[at] = sm_key(x[q]);
              list_idx[at] = e + q;
            }
            ++at;
          }
      }
    });
    __syncthreads();
    nlist = (int)min(s_count, (uint32_t)kSmList);
    return s_count <= room;
  };
  auto over_list = [&](auto f) {
    for (int e = t; e < nlist; e += kSmThreads) f(list_key[e]);
  };
  auto over_row = [&](auto f) {
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < w_end) f(sm_key(x[q]));
    });
  };

  auto need_of = [&](uint64_t s) -> uint64_t {  // the weight that top-p asks of s, at least the least
    bool rest;
    const uint64_t need = sm_mul_frac(s, p > 0.f ? p : 0.f, rest);
    return rest || need == 0 ? need + 1 : need;
  };
  bool all_listed = false;  // every kept token is in the list
  int last_tie = 0x7fffffff;  // ties are kept up to this index
  bool selected = !has_k && !has_p;

  // the list of the first tokens, sorted, and the kept ones in it: of the k first
  // (k > 0, else of all), those that reach need(weight of these)
  auto from_list = [&](int kept_of, auto need) {
    // larger keys first, lower indexes first among equals; nothing behind the list
    uint64_t v = t < nlist ? ((uint64_t)list_key[t] << 32) | (uint32_t)~list_idx[t] : 0;
    unsigned long long* swap = hist;
#pragma unroll
    for (int size = 2; size <= kSmSort; size <<= 1) {
#pragma unroll
      for (int step = size >> 1; step > 0; step >>= 1) {
        uint64_t o;
        if (step < 64) {
          o = sm_shfl_xor(v, step);
        } else {
          __syncthreads();
          swap[t] = v;
          __syncthreads();
          o = swap[t ^ step];
        }
        const bool first = (t & step) == 0, falling = (t & size) == 0;
        v = (first == falling) == (v > o) ? v : o;
      }
    }
    __syncthreads();
    swap[t] = v;
    const uint64_t w = t < nlist ? weight(sm_logit((uint32_t)(v >> 32))) : 0;
    const uint64_t before = block_scan(w);
    if (t == kept_of - 1) s_u64 = before + w;
    __syncthreads();
    int n_kept = kept_of;
    if (has_p) {
      const uint64_t least = need((uint64_t)s_u64);
      if (before < least && before + w >= least) s_u32 = t;
      __syncthreads();
      n_kept = (int)s_u32 + 1;
    }
    const uint64_t last = swap[n_kept - 1];
    kk = (uint32_t)(last >> 32);
    last_tie = (int)~(uint32_t)last;
    all_listed = selected = true;
  };
  if (has_k && (V <= kSmSort || k <= min(kSmGuess, V / 4))) {  // V / 4 threads, or 960, hold logits
    uint32_t b = kSmBins - 1;
    if (V > kSmSort) {
      hist[t] = 0;
      __syncthreads();
      if (first_of(0) < w_end) atomicAdd(&hist[bin_of(mine)], 1ull);
      __syncthreads();
      uint64_t before;
      b = find_bin(hist[t], 0, (uint64_t)k, before);
    }
    if (collect(0, b, kSmSort)) from_list(k, need_of);
  }
  if (has_k && !selected) {
    hist[t] = 0;
    __syncthreads();
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < w_end) atomicAdd(&hist[bin_of(x[q])], 1ull);
    });
    __syncthreads();
    uint64_t before;
    const uint32_t b = find_bin(hist[t], 0, (uint64_t)k, before);
    const uint64_t upto = before + hist[b];
    all_listed = upto <= kSmList;
    if (all_listed) {
      collect(0, b);
      refine(over_list, 0, (uint64_t)k, false);
    } else if (collect(b, b)) {
      refine(over_list, before, (uint64_t)k, false);
    } else {
      refine(over_row, 0, (uint64_t)k, false);
    }
  }
  auto kept_sum = [&](auto over) -> uint64_t {
    uint64_t s = 0;
    over([&](uint32_t key) {
      if (key > kk) s += weight(sm_logit(key));
    });
    s = block_sum(s);
    return ties ? s + ties * weight(sm_logit(kk)) : s;
  };
  if (has_p && !selected) {
    if (all_listed) {
      refine(over_list, 0, need_of(kept_sum(over_list)), true);
    } else {
      const uint32_t k0 = kk;
      const uint64_t t0 = ties;
      __syncthreads();
      hist[t] = 0;
      __syncthreads();
      each([&](int, const float (&x)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint64_t w = weight(x[q]);
          if (w && sm_key(x[q]) > k0) atomicAdd(&hist[bin_of(x[q])], (unsigned long long)w);
        }
      });
      if (t == 0 && t0) atomicAdd(&hist[bin_of(sm_logit(k0))], (unsigned long long)(t0 * weight(sm_logit(k0))));
      __syncthreads();
      const uint64_t own = hist[t];
      const uint64_t need = need_of(block_sum(own));
      uint64_t before;
      const uint32_t b = find_bin(own, 0, need, before);
      uint64_t upto = 0;
      each([&](int e, const float (&x)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) upto += e + q < w_end && bin_of(x[q]) <= (int)b;
      });
      if (!has_k && block_sum(upto) <= kSmSort) {
        collect(0, b, kSmSort);
        from_list(nlist, [&](uint64_t) { return need; });
      } else if (collect(b, b)) {
        refine(over_list, before, need, true);
      } else {
        refine(over_row, 0, need, true);
      }
    }
  }

  // Lowest index of [from, to), in steps of 256 that seg has the sums of, whose
  // running sum of measure(index, logit), from base on, exceeds target.
  auto find_in = [&](int from, int to, uint64_t base, uint64_t target, auto measure) -> int {
    __syncthreads();
    if (wave == 0) {
      const int ns = (to - from + 255) / 256;
      for (int s0 = 0; s0 < ns; s0 += 64) {
        const uint64_t own = s0 + lane < ns ? (uint64_t)seg[s0 + lane] : 0;
        uint64_t inc = own;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
          const uint64_t o = sm_shfl_up(inc, m);
          if (lane >= m) inc += o;
        }
        const uint64_t run = base + inc - own;
        const uint64_t hit = __ballot(run <= target && run + own > target);
        if (hit) {
          const int b = __builtin_ctzll(hit);
          const uint64_t at = (uint64_t)__shfl((unsigned long long)run, b, 64);
          // the step's 256 logits again, 4 a lane
          const int e = from + (s0 + b) * 256 + 4 * lane;
          uint64_t v[4], sum = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            v[q] = e + q < to ? measure(e + q, row[e + q]) : 0;
            sum += v[q];
          }
          uint64_t in2 = sum;
#pragma unroll
          for (int m = 1; m < 64; m <<= 1) {
            const uint64_t o = sm_shfl_up(in2, m);
            if (lane >= m) in2 += o;
          }
          uint64_t r2 = at + in2 - sum;
          if (r2 <= target && r2 + sum > target) {
            int q = 0;
            while (q < 3 && r2 + v[q] <= target) r2 += v[q++];
            s_u32 = (uint32_t)(e + q);
          }
          break;
        }
        base += (uint64_t)__shfl((unsigned long long)inc, 63, 64);
      }
    }
    __syncthreads();
    return (int)s_u32;
  };
  // The same over the row, for the target that goal(sum over the row) gives: the
  // waves' sums say whose share it is in, the workgroup adds up that share's steps.
  auto find = [&](auto measure, auto goal) -> int {
    uint64_t sum = 0;
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) sum += e + q < w_end ? measure(e + q, x[q]) : 0;
    });
    const uint64_t target = goal(block_sum(sum));
    uint64_t base = 0, upto = 0;
    int w = -1;
    do {  // at most 16 waves; their sums exceed target
      base = upto;
      upto += s_sum[++w];
    } while (upto <= target && w < kSmWaves - 1);
    const int from = w * per_wave, to = min(from + per_wave, V);
    for (int c = wave; c * 256 < to - from; c += kSmWaves) {
      const int e = from + 256 * c + 4 * lane;
      uint64_t v = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) v += e + q < to ? measure(e + q, row[e + q]) : 0;
      v = sm_wave_sum(v);
      if (lane == 0) seg[c] = v;
    }
    return find_in(from, to, base, target, measure);
  };
  if (ties && ties_left) {
    const uint64_t nth = ties - 1;
    last_tie = find([&](int, float l) -> uint64_t { return sm_key(l) == kk ? 1 : 0; }, [&](uint64_t) { return nth; });
    __syncthreads();
  }
  auto kept = [&](int e, float l) -> uint64_t {
    const uint32_t key = sm_key(l);
    if (!(key > kk || (key == kk && e <= last_tie))) return 0;
    const uint64_t w = weight(l);
    return w >= wmin ? w : 0;
  };
  auto goal = [&](uint64_t total) -> uint64_t {
    bool rest;
    return sm_mul_frac(total, u, rest);
  };
  int id;
  if (all_listed) {
    const int ns = (V + 255) / 256;
    __syncthreads();
    for (int e = t; e < ns; e += kSmThreads) seg[e] = 0;
    __syncthreads();
    uint64_t sum = 0;
    for (int e = t; e < nlist; e += kSmThreads) {
      const uint64_t w = kept((int)list_idx[e], sm_logit(list_key[e]));
      sum += w;
      if (w) atomicAdd(&seg[list_idx[e] >> 8], (unsigned long long)w);
    }
    id = find_in(0, V, 0, goal(block_sum(sum)), kept);
  } else {
    id = find(kept, goal);
  }
  if (t == 0) argmax_finish(i, id, a.out, a.ring, a.ring_rows, a.ring_len, a.expect, a.accept);
}

}  // namespace wfd

extern "C" {

int wfd_sample(const float* logits, int64_t ld, const float* u, const float* temperature, const int32_t* top_k,
               const float* top_p, const float* min_p, int64_t* out, int64_t* ring, const int32_t* ring_rows,
               int64_t ring_len, const int64_t* expect, int32_t* accept, int n, int vocab, hipStream_t stream) {
  using namespace wfd;
  if (n < 0 || vocab <= 0 || ld < vocab) {
    set_error("wfd_sample: bad shape n=%d vocab=%d ld=%lld", n, vocab, (long long)ld);
    return kBadArg;
  }
  if (vocab > kSmMaxVocab) {
    set_error("wfd_sample: vocab=%d (at most %d)", vocab, kSmMaxVocab);
    return kUnsupported;
  }
  if (n == 0) return kOk;
  if (!logits || !u || !out || (ring && (!ring_rows || ring_len <= 0)) || (!expect != !accept)) {
    set_error("wfd_sample: null pointer argument (ring needs ring_rows and a length; expect and accept go together)");
    return kBadArg;
  }
  SmArgs a;
  a.logits = logits;
  a.ld = ld;
  a.u = u;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.out = out;
  a.ring = ring;
  a.ring_rows = ring_rows;
  a.ring_len = ring_len;
  a.expect = expect;
  a.accept = accept;
  a.V = vocab;
  if (vocab <= 2 * kSmChunk)
    hipLaunchKernelGGL(sample_kernel<2 * kSmChunk>, dim3(n), dim3(kSmThreads), 0, stream, a);
  else if (vocab <= 8 * kSmChunk)
    hipLaunchKernelGGL(sample_kernel<8 * kSmChunk>, dim3(n), dim3(kSmThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(sample_kernel<0>, dim3(n), dim3(kSmThreads), 0, stream, a);
  return launch_status("wfd_sample");
}

}  // extern "C"
