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
// One workgroup per row; no sort: the prefix is found by a radix select over
// the logits' order-preserving keys, 8 bits a pass from the top, with the count
// (top-k) or the weight (top-p) of each digit's tokens in LDS; only the tokens
// that share the digits found so far take part. Ties with the last kept key are
// kept in index order.
#include "wfd_common.h"

namespace wfd {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmChunk = 4 * kSmThreads;  // logits per round of the workgroup: 4 consecutive ones a thread
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

// NR > 0: the row's chunks live in registers (V <= NR * kSmChunk); 0: they are
// read again in every pass (from L2).
template <int NR>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SmArgs a) {
  __shared__ unsigned long long hist[256];
  __shared__ unsigned long long seg[kSmMaxVocab / 256];  // per 256 logits, in index order
  __shared__ float s_max[kSmWaves];
  __shared__ int s_idx[kSmWaves];
  __shared__ unsigned long long s_sum[kSmWaves];
  __shared__ unsigned long long s_u64[2];
  __shared__ uint32_t s_u32[2];
  const int i = blockIdx.x;
  const int t = threadIdx.x;
  const int wave = t >> 6, lane = t & 63;
  const int V = a.V;
  const float* row = a.logits + (int64_t)i * a.ld;
  const bool vec = ((uintptr_t)row & 15) == 0;
  const int nchunks = (V + kSmChunk - 1) / kSmChunk;

  auto fetch = [&](int c, float (&x)[4]) {  // logits 4096 c + 4 t ..; past the row: NaN-free filler, masked by index
    const int e = c * kSmChunk + 4 * t;
    if (vec && e + 4 <= V) {
      Elem<float>::unpack(ld16(row + e), x);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = e + k < V ? row[e + k] : -INFINITY;
    }
  };
  float reg[NR > 0 ? NR : 1][4];
  if constexpr (NR > 0) {
#pragma unroll
    for (int c = 0; c < NR; ++c) fetch(c, reg[c]);
  }
  // f(chunk, first index, the 4 logits) over the row, in index order per thread
  auto each = [&](auto f) {
    if constexpr (NR > 0) {
#pragma unroll
      for (int c = 0; c < NR; ++c)
        if (c < nchunks) f(c, c * kSmChunk + 4 * t, reg[c]);
    } else {
      for (int c = 0; c < nchunks; ++c) {
        float x[4];
        fetch(c, x);
        f(c, c * kSmChunk + 4 * t, x);
      }
    }
  };

  // the largest logit and its first index; a NaN ranks above everything, as in wfd_argmax
  float best = -INFINITY;
  int bi = 0x7fffffff;
  each([&](int, int e, const float (&x)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (e + k < V) argmax_merge(best, bi, x[k], e + k);
  });
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) argmax_merge(best, bi, __shfl_xor(best, m, 64), __shfl_xor(bi, m, 64));
  if (lane == 0) {
    s_max[wave] = best;
    s_idx[wave] = bi;
  }
  __syncthreads();
  best = s_max[0];
  bi = s_idx[0];
  for (int w = 1; w < kSmWaves; ++w) argmax_merge(best, bi, s_max[w], s_idx[w]);

  const float T = a.temperature ? a.temperature[i] : 1.f;
  // greedy rows; rows with a NaN (its index, visibly) or without any possible token (index 0)
  if (!(T > 0.f) || best != best || best == -INFINITY) {  // uniform
    if (t == 0) argmax_finish(i, bi, a.out, a.ring, a.ring_rows, a.ring_len, a.expect, a.accept);
    return;
  }
  const double mx = (double)best;
  const double inv = 1.4426950408889634 / (double)T;
  auto weight_of = [&](float l, float floor_w) -> uint64_t {
    if (l == best) return (uint64_t)kSmOne;  // also of infinite logits
    if (l == -INFINITY) return 0;
    const double w = exp2(((double)l - mx) * inv);
    if (floor_w > 0.f && w < (double)floor_w) return 0;
    return w > 0. ? (uint64_t)(w * kSmOne + 0.5) : 0;  // NaN (infinite temperature under an infinite logit): 0
  };
  auto weight = [&](float l) { return weight_of(l, 0.f); };

  auto block_sum = [&](uint64_t v) -> uint64_t {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += sm_shfl_xor(v, m);
    __syncthreads();
    if (lane == 0) s_sum[wave] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int w = 0; w < kSmWaves; ++w) s += s_sum[w];
    return s;
  };

  // Kept so far: keys above kk, and the first `ties` tokens with key kk.
  uint32_t kk = 0;
  uint64_t ties = 0;

  // The shortest prefix of the kept tokens whose measure (1 or the weight) reaches need > 0.
  auto select = [&](uint64_t need, bool by_weight) {
    const uint32_t k0 = kk;
    const uint64_t t0 = ties;
    uint32_t prefix = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (t < 256) hist[t] = 0;
      __syncthreads();
      each([&](int, int e, const float (&x)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t key = sm_key(x[k]);
          if (e + k < V && key > k0 && (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))) {
            const uint64_t m = by_weight ? weight(x[k]) : 1;
            if (m) atomicAdd(&hist[(key >> shift) & 255], (unsigned long long)m);
          }
        }
      });
      if (t == 0 && t0 && (shift == 24 || (k0 >> (shift + 8)) == (prefix >> (shift + 8)))) {
        // the kept ties, as one
        atomicAdd(&hist[(k0 >> shift) & 255], (unsigned long long)(t0 * (by_weight ? weight(sm_logit(k0)) : 1)));
      }
      __syncthreads();
      if (wave == 0) {  // lane b holds digits 255 - 4 b .. 252 - 4 b: the running sum from the top
        uint64_t v[4], own = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) own += v[k] = hist[255 - 4 * lane - k];
        uint64_t inc = own;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
          const uint64_t o = sm_shfl_up(inc, m);
          if (lane >= m) inc += o;
        }
        uint64_t run = above + inc - own;
        const uint64_t hit = __ballot(run < need && run + own >= need);  // one lane: the sums reach need
        if (hit >> lane & 1) {
          int d = 255 - 4 * lane;
#pragma unroll
          for (int k = 0; k < 3; ++k)
            if (run + v[k] < need && d == 255 - 4 * lane - k) {
              run += v[k];
              --d;
            }
          s_u32[0] = prefix | ((uint32_t)d << shift);
          s_u64[0] = run;
        }
      }
      __syncthreads();
      prefix = s_u32[0];
      above = s_u64[0];
    }
    kk = prefix;
    const uint64_t each_w = by_weight ? weight(sm_logit(kk)) : 1;
    ties = (need - above + each_w - 1) / each_w;  // >= 1; no more than there are, since they reach need
  };

  const int k = a.top_k ? a.top_k[i] : 0;
  if (k > 0 && k < V) select((uint64_t)k, false);

  auto mul_frac = [](uint64_t s, float f, uint64_t& lo) -> uint64_t {  // floor(s * f), f in [0, 1), and the rest
    const uint64_t q = (uint64_t)((double)f * 18446744073709551616.0);
    lo = s * q;
    return __umul64hi(s, q);
  };
  auto kept_sum = [&](float floor_w) -> uint64_t {
    uint64_t s = 0;
    each([&](int, int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < V && sm_key(x[q]) > kk) s += weight_of(x[q], floor_w);
    });
    s = block_sum(s);
    return ties ? s + ties * weight_of(sm_logit(kk), floor_w) : s;
  };
  const float p = a.top_p ? a.top_p[i] : 1.f;
  if (p < 1.f) {
    uint64_t lo;
    const uint64_t s = kept_sum(0.f);
    uint64_t need = mul_frac(s, p > 0.f ? p : 0.f, lo);
    if (lo || need == 0) ++need;
    select(need, true);
  }

  // the last kept tie's index, if some of the ties are left out
  auto find = [&](uint64_t target, auto measure) -> int {  // lowest index whose running sum exceeds target
    each([&](int c, int e, const float (&x)[4]) {
      uint64_t v = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < V) v += measure(e + q, x[q]);
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) v += sm_shfl_xor(v, m);
      if (lane == 0) seg[c * kSmWaves + wave] = v;
    });
    __syncthreads();
    if (wave == 0) {
      uint64_t base = 0;
      const int ns = nchunks * kSmWaves;
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
          // the segment's 256 logits again, 4 a lane
          const int e = (s0 + b) * 256 + 4 * lane;
          uint64_t v[4], mine = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            v[q] = e + q < V ? measure(e + q, row[e + q]) : 0;
            mine += v[q];
          }
          uint64_t in2 = mine;
#pragma unroll
          for (int m = 1; m < 64; m <<= 1) {
            const uint64_t o = sm_shfl_up(in2, m);
            if (lane >= m) in2 += o;
          }
          uint64_t r2 = at + in2 - mine;
          if (r2 <= target && r2 + mine > target) {
            int q = 0;
            while (q < 3 && r2 + v[q] <= target) r2 += v[q++];
            s_u32[0] = (uint32_t)(e + q);
          }
          break;
        }
        base = (uint64_t)__shfl((unsigned long long)inc, 63, 64) + base;
      }
    }
    __syncthreads();
    const int r = (int)s_u32[0];
    __syncthreads();
    return r;
  };
  int last_tie = -1;
  if (ties) last_tie = find(ties - 1, [&](int, float l) -> uint64_t { return sm_key(l) == kk ? 1 : 0; });
  const float minp = a.min_p ? a.min_p[i] : 0.f;
  const uint64_t total = kept_sum(minp);
  float u = a.u[i];
  u = u > 0.f ? (u < 1.f ? u : 0.99999994f) : 0.f;
  uint64_t lo;
  const uint64_t target = mul_frac(total, u, lo);
  const int id = find(target, [&](int e, float l) -> uint64_t {
    const uint32_t key = sm_key(l);
    return key > kk || (key == kk && e <= last_tie) ? weight_of(l, minp) : 0;
  });
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
    hipLaunchKernelGGL(sample_kernel<2>, dim3(n), dim3(kSmThreads), 0, stream, a);
  else if (vocab <= 8 * kSmChunk)
    hipLaunchKernelGGL(sample_kernel<8>, dim3(n), dim3(kSmThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(sample_kernel<0>, dim3(n), dim3(kSmThreads), 0, stream, a);
  return launch_status("wfd_sample");
}

}  // extern "C"
