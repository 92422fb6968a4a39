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
// Where top-k keeps few tokens they are found without ordering the row: of the 1024
// threads' largest logits, at least k are no smaller than the k-th, so every one of
// the first k tokens is at or above it, and few others are. Those go to a list in LDS,
// which is put in order (four threads an entry) if it is short, and top-k, top-p and
// min_p are positions in it. A top-p alone guesses the bin, of 1024 by the distance
// from the largest logit, that its last token lies in from 32-bit weights; one pass
// over the exact ones then gives the row's sum, the waves' sums of the bins before
// and the bin's tokens, in whose order the last one is found (the guess is checked
// against the exact sums; two exact passes took 100 rows a third longer). Otherwise a
// histogram says which bin the last kept token lies in, by count or by weight, and a
// radix select over that bin's tokens (over the row, if they are too many) finds its
// key; ties with it are kept in index order.
//
// Rows of up to 32768 logits are one workgroup's, which keeps them in LDS. Longer
// ones are cut into slabs of 8192, a workgroup each, in four launches that leave
// their results in the workspace: the slabs' largest logits; the k candidates or
// the histogram; the weights before the border's bin and its tokens; the row's
// token. What no slab could prepare (a top-k beyond kSmGuess, a list that
// overflows) the last launch does by itself as for a short row. Slabs for rows of
// 32000 took 32 top-p rows from 30.8 to 26.7 us, but 100 of them from 28.8 to 35, one
// as long, and one row with top-k from 13 to 19.
//
// Bound by the one CU a row has (the logits themselves are microseconds), there by
// instructions: 4 waves a SIMD issue one each 4 cycles apiece, so of 32000 logits the
// exact weights, ~45 instructions each, take 8 us, the 32-bit ones 6, the candidates 4,
// reading the row 3, and each step that waits for the workgroup 0.3. 1 x 32000 with
// top-k and top-p 13 us, 100 x 32000 mixed 28, 16 x 128000 top-p 33 (4 + 8 + 9 + 13 in
// four launches), 8 x 128000 with top-k 23.
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

// Wave-wide folds over neighbouring lanes' registers (DPP), a third of the latency of
// shuffles through LDS; every lane of the wave calls them. fold(lanes 0..l) in lane l.
constexpr int kSmQuad1 = 0xb1, kSmQuad2 = 0x4e;  // lane l ^ 1, l ^ 2
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sm_dpp(uint32_t v, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t sm_dpp_add(uint64_t v) {
  return v + (((uint64_t)sm_dpp<CTRL, ROWS>((uint32_t)(v >> 32), 0) << 32) | sm_dpp<CTRL, ROWS>((uint32_t)v, 0));
}
__device__ __forceinline__ uint64_t sm_row_scan(uint64_t v) {  // within rows of 16 lanes
  v = sm_dpp_add<0x111, 0xf>(v);  // from 1, 2, 4, 8 lanes before
  v = sm_dpp_add<0x112, 0xf>(v);
  v = sm_dpp_add<0x114, 0xf>(v);
  return sm_dpp_add<0x118, 0xf>(v);
}
__device__ __forceinline__ uint64_t sm_wave_scan(uint64_t v) {
  v = sm_dpp_add<0x142, 0xa>(sm_row_scan(v));  // a row's last lane to the next row, of each half
  return sm_dpp_add<0x143, 0xc>(v);            // lane 31 to the upper half
}
__device__ __forceinline__ uint64_t sm_lane(uint64_t v, int lane) {  // lane: uniform
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ uint64_t sm_last_lane(uint64_t v) { return sm_lane(v, 63); }
__device__ __forceinline__ uint64_t sm_wave_sum(uint64_t v) { return sm_last_lane(sm_wave_scan(v)); }
template <typename F>
__device__ __forceinline__ uint32_t sm_wave_fold(uint32_t v, uint32_t none, F f) {
  v = f(v, sm_dpp<0x111, 0xf>(v, none));
  v = f(v, sm_dpp<0x112, 0xf>(v, none));
  v = f(v, sm_dpp<0x114, 0xf>(v, none));
  v = f(v, sm_dpp<0x118, 0xf>(v, none));
  v = f(v, sm_dpp<0x142, 0xa>(v, none));
  v = f(v, sm_dpp<0x143, 0xc>(v, none));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t sm_wave_min(uint32_t v) {
  return sm_wave_fold(v, 0xffffffffu, [](uint32_t x, uint32_t y) { return min(x, y); });
}
__device__ __forceinline__ uint32_t sm_wave_max(uint32_t v) {
  return sm_wave_fold(v, 0u, [](uint32_t x, uint32_t y) { return max(x, y); });
}
__device__ __forceinline__ float sm_wave_max(float v) {
  return __uint_as_float(sm_wave_fold(__float_as_uint(v), 0xff800000u, [](uint32_t x, uint32_t y) {
    return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
  }));
}
__device__ __forceinline__ float sm_wave_min(float v) { return -sm_wave_max(-v); }

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
constexpr int kSmFew = kSmThreads / 4;  // entries of a list that is put in order
constexpr int kSmShort = 2048;       // slabs of so few logits are listed whole
constexpr int kSmLong = 32768;       // longest row of one workgroup
constexpr int kSmSlab = 8192;
constexpr int kSmSlabs = kSmMaxVocab / kSmSlab;
constexpr int kSmRowList = 8192;     // tokens that the slabs of a row may list
// Top-k to which the list is tried: ~900 tokens reach the 600th thread's. The slabs of a
// long row list as many each, and past kSmRowList in all the last launch draws the row
// alone, as it does for a larger top-k without having tried. 16 rows, top-k 50 / 200 / 300
// / 600 / 601 in us:  65536 logits 20 / 25 / 27 / 29 / 45;  128000 21 / 26 / 29 / 57 / 65;
// 262144 27 / 34 / 75 / 79 / 98;  524288 39 / 118 / 126 / 130 / 171. Tried to 200 only,
// top-k 300 of these takes 42 / 62 / 94 / 166; never, 50 takes 34 / 52 / 85 / 154.
constexpr int kSmGuess = 600;
constexpr float kSmMasked = -1e4f;  // logits down to here spread the bins; the others share the last

// 2^x for x <= 0 in units of 2^-44, rounded to an integer: x = m / 128 + r, 2^r by its
// series to r^4 (the rest is below 2e-15 of it), 2^(44 + m / 128) from the table with
// the exponent added to its bits. Adding 1.5 2^52 leaves the nearest integer in the
// low bits of the sum, adding and subtracting 2^52 rounds to it.
constexpr int kSmTable = 128;
__device__ __forceinline__ double sm_exp2(double x, const double* __restrict__ tab) {
  x = fmax(x, -900.);  // also of NaN; far below the least weight
  const double t = fma(x, (double)kSmTable, 6755399441055744.);
  const int k = (int)(uint32_t)__double_as_longlong(t);
  const double r = fma(t - 6755399441055744., -1. / kSmTable, x);
  double p = fma(r, 0.009618129107628477, 0.05550410866482158);
  p = fma(p, r, 0.24022650695910072);
  p = fma(p, r, 0.6931471805599453);
  p = fma(p, r, 1.0);
  const double two =
      __longlong_as_double(__double_as_longlong(tab[k & (kSmTable - 1)]) + ((long long)(k & -kSmTable) << 45));
  return fma(p, two, 4503599627370496.) - 4503599627370496.;
}

// floor(s f) for f in [0, 1), and whether anything was cut off
__device__ __forceinline__ uint64_t sm_mul_frac(uint64_t s, float f, bool& rest) {
  const uint64_t q = (uint64_t)((double)f * 18446744073709551616.0);
  rest = s * q != 0;
  return __umul64hi(s, q);
}

// What a long row's launches leave each other.
struct SmRowWs {
  unsigned long long hist[kSmBins];
  unsigned long long share[kSmSlabs * kSmWaves];  // weights kept in the waves' shares, slab after slab
  float max[kSmSlabs], min[kSmSlabs];
  uint32_t nan[kSmSlabs];
  uint32_t count;  // of the list; more than kSmRowList: it is incomplete
  uint32_t pad[3];
  uint32_t key[kSmRowList], idx[kSmRowList];
};

// CAP > 0: the logits at hand, at most CAP, are kept in LDS; < 0: at most -CAP, in
// registers, whose loads are in flight until the first use (for the slabs' 8 a thread;
// the one-workgroup kernel's code spilled with 8 too). 0: they are read again in every
// pass (from L2).
template <int CAP, int LIST>
struct SmShared {
  unsigned long long hist[kSmBins];
  unsigned long long seg[(CAP > 0 ? CAP : CAP < 0 ? -CAP : kSmMaxVocab) / 256];  // the running sums' steps
  u32x4 keep[CAP > 0 ? CAP / 4 : 1];
  uint32_t list_key[LIST], list_idx[LIST];
  double tab[kSmTable];
  float max[kSmWaves], min[kSmWaves];
  unsigned long long sum[4][kSmWaves];
  unsigned long long share[kSmWaves];  // kept weights of the waves' shares
  uint32_t lo[kSmWaves], hi[kSmWaves];
  unsigned long long u64;
  uint32_t u32, count;
};

// A workgroup's work on logits [begin, end) of a row: wave w holds [begin + w
// per_wave, begin + (w + 1) per_wave), 4 consecutive ones a lane and round, so
// that index order is wave, round, lane. Every method is called by all threads.
template <int CAP, int LIST>
struct Sm {
  const SmArgs& a;
  SmShared<CAP, LIST>& s;
  const int i, t, wave, lane, V, begin, end, per_wave, w_end, rounds;
  const float* row;
  const bool vec;
  // the row's largest logit and the bins' range, and the thread's own largest
  float best, low, mine;
  bool nan;
  // parameters
  float T, p, minp, u, scale;
  int k;
  bool has_k, has_p, endless;
  double inv;
  uint64_t wmin;
  // Kept: keys above kk, and the first `ties` tokens with key kk, of which ties_left
  // more are not kept; last_tie: the index of the last kept one.
  uint32_t kk = 0;
  uint64_t ties = 0, ties_left = 0;
  int last_tie = 0x7fffffff;
  float held[CAP < 0 ? -CAP / kSmChunk : 1][4];
  bool ties_listed = false;  // every token with key kk is in the list
  int nlist = 0;

  __device__ __forceinline__ Sm(const SmArgs& args, SmShared<CAP, LIST>& sh, int row_i, int lo, int hi)
      : a(args), s(sh), i(row_i), t(threadIdx.x), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
        lane(threadIdx.x & 63), V(args.V), begin(lo), end(hi), per_wave((hi - lo + 63) / 64 * 4),
        w_end(min(lo + (wave + 1) * per_wave, hi)), rounds((per_wave + 255) / 256),
        row(args.logits + (int64_t)row_i * args.ld), vec(((uintptr_t)(row + lo) & 15) == 0) {
    if constexpr (CAP < 0) {
#pragma unroll
      for (int c = 0; c < -CAP / kSmChunk; ++c) fetch(c, held[c]);
    }
    if (t < kSmTable) s.tab[t] = exp2((double)t * (1. / kSmTable)) * kSmOne;
  }

  __device__ __forceinline__ int first_of(int c) const { return begin + wave * per_wave + 256 * c + 4 * lane; }
  __device__ __forceinline__ void fetch(int c, float (&x)[4]) const {  // 4 logits; -inf past the wave's
    const int e = first_of(c);
    if (vec && e + 4 <= w_end) {
      Elem<float>::unpack(ld16(row + e), x);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = e + q < w_end ? row[e + q] : -INFINITY;
    }
  }
  // f(first index, 4 logits), in index order per thread; -inf fills the places past the
  // wave's share, which no weight, bin or key below counts
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    float x[4];
    if constexpr (CAP < 0) {
#pragma unroll
      for (int c = 0; c < -CAP / kSmChunk; ++c)
        if (c < rounds) f(first_of(c), held[c]);
    } else if constexpr (CAP > 0) {
      for (int c = 0; c < rounds; ++c) {
        Elem<float>::unpack(s.keep[c * kSmThreads + t], x);
        f(first_of(c), x);
      }
    } else {
      fetch(0, x);
      for (int c = 0; c < rounds; ++c) {  // a round ahead
        float y[4];
        fetch(min(c + 1, rounds - 1), y);
        f(first_of(c), x);
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = y[q];
      }
    }
  }

  // --- the workgroup's sums -------------------------------------------------
  // The waves' sums are 16 lanes of each wave, which adds them up for itself: 16 adds by
  // every wave took twice the time.
  __device__ __forceinline__ uint64_t block_sum(uint64_t v) {
    v = sm_wave_sum(v);
    __syncthreads();
    if (lane == 0) s.sum[0][wave] = v;
    __syncthreads();
    return sm_lane(sm_row_scan(s.sum[0][lane & 15]), 15);
  }
  __device__ __forceinline__ void block_sums(uint64_t (&v)[4]) {  // v[3] by waves is left in share
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = sm_wave_sum(v[q]);
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) s.sum[q][wave] = v[q];
      s.share[wave] = v[3];
    }
    __syncthreads();
    const uint64_t run = sm_row_scan(s.sum[lane >> 4][lane & 15]);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = sm_lane(run, 16 * q + 15);
  }
  // The sum of the threads' v before this one.
  __device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t& total) {
    const uint64_t inc = sm_wave_scan(v);
    __syncthreads();
    if (lane == 63) s.sum[0][wave] = inc;
    __syncthreads();
    const uint64_t run = sm_row_scan(s.sum[0][lane & 15]);
    total = sm_lane(run, 15);
    return (wave ? sm_lane(run, wave - 1) : 0) + inc - v;
  }
  // The shares' sum, for find_by_waves.
  __device__ __forceinline__ uint64_t share_sum(uint64_t v) {
    v = sm_wave_sum(v);
    __syncthreads();
    if (lane == 0) s.share[wave] = v;
    __syncthreads();
    return sm_lane(sm_row_scan(s.share[lane & 15]), 15);
  }
  // The bin (thread t holds bin t's sum v) in which base plus the running sum reaches need; before: the sum before it.
  __device__ __forceinline__ uint32_t find_bin(uint64_t v, uint64_t base, uint64_t need, uint64_t& before) {
    uint64_t total;
    return bin_at(v, base + block_scan(v, total), need, before);
  }
  __device__ __forceinline__ uint32_t bin_at(uint64_t v, uint64_t run, uint64_t need, uint64_t& before) {
    if (run < need && run + v >= need) {
      s.u32 = t;
      s.u64 = run;
    }
    __syncthreads();
    before = s.u64;
    return s.u32;
  }
  // The bin in which top-p of all bins' weight is reached.
  __device__ __forceinline__ uint32_t top_p_bin(uint64_t v, uint64_t& need, uint64_t& before) {
    uint64_t total;
    const uint64_t run = block_scan(v, total);
    need = need_of(total);
    return bin_at(v, run, need, before);
  }

  __device__ __forceinline__ void block_range(uint32_t& lo, uint32_t& hi) {
    lo = sm_wave_min(lo);
    hi = sm_wave_max(hi);
    __syncthreads();
    if (lane == 0) {
      s.lo[wave] = lo;
      s.hi[wave] = hi;
    }
    __syncthreads();
    lo = sm_wave_min(s.lo[lane & 15]);
    hi = sm_wave_max(s.hi[lane & 15]);
  }

  // --- the row's largest logit, whether there is a NaN, the range of the bins --
  __device__ __forceinline__ void largest() {
    mine = -INFINITY;
    float lo = INFINITY;
    bool bad = false;
    auto look = [&](int, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        bad |= x[q] != x[q];
        mine = fmaxf(mine, x[q]);
        lo = fminf(lo, x[q] > kSmMasked ? x[q] : INFINITY);
      }
    };
    if constexpr (CAP > 0) {  // on their way to LDS, every load first; a thread reads back only what it stores
      float x[CAP / kSmChunk][4];
#pragma unroll
      for (int c = 0; c < CAP / kSmChunk; ++c) fetch(c, x[c]);
#pragma unroll
      for (int c = 0; c < CAP / kSmChunk; ++c) {
        s.keep[c * kSmThreads + t] = Elem<float>::pack(x[c]);
        look(first_of(c), x[c]);
      }
    } else {
      each(look);
    }
    const float hi = sm_wave_max(mine);
    lo = sm_wave_min(lo);
    bad = __ballot(bad) != 0;
    if (lane == 0) {
      s.max[wave] = hi;
      s.min[wave] = lo;
      s.lo[wave] = bad;
    }
    __syncthreads();
    nan = __ballot(s.lo[lane & 15] != 0) != 0;
    best = sm_wave_max(s.max[lane & 15]);
    low = sm_wave_min(s.min[lane & 15]);
    __syncthreads();
  }
  // The same of a long row, from its slabs'.
  __device__ __forceinline__ void largest_of(const SmRowWs& ws, int slabs) {
    nan = false;
    best = -INFINITY;
    low = INFINITY;
    const int l = min(lane, slabs - 1);  // at most 64
    nan = __ballot(ws.nan[l] != 0) != 0;
    best = ws.max[l];
    low = ws.min[l];
    best = sm_wave_max(best);
    low = sm_wave_min(low);
  }
  // false: a row of one token, the first of its order (greedy ones), or with a NaN or without any possible token
  __device__ __forceinline__ bool parameters() {
    T = a.temperature ? a.temperature[i] : 1.f;
    if (nan || !(T > 0.f) || best == -INFINITY) return false;
    inv = fmin(1.4426950408889634 / (double)T, 1e300);  // finite: 0 times it is 0
    endless = best == INFINITY;                          // infinite logits share everything
    k = a.top_k ? a.top_k[i] : 0;
    has_k = k > 0 && k < V;
    p = a.top_p ? a.top_p[i] : 1.f;
    has_p = p < 1.f;
    minp = a.min_p ? a.min_p[i] : 0.f;
    if (minp > 1.f) return false;  // no weight reaches it: the first token alone, the greedy one
    // on the integer weights' scale: w >= min_p for w on or above it
    wmin = minp > 0.f ? (uint64_t)ceil((double)minp * kSmOne) : 0;
    u = a.u[i];
    u = u > 0.f ? (u < 1.f ? u : 0.99999994f) : 0.f;
    scale = best > low ? (float)(kSmBins - 2) / (best - low) : 1.f;
    return true;
  }
  // The first index of the largest logit, or of a NaN.
  __device__ __forceinline__ int first_best() {
    int bi = 0x7fffffff;
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 3; q >= 0; --q)
        if (e + q < w_end && (nan ? x[q] != x[q] : x[q] == best)) bi = min(bi, e + q);
    });
    bi = (int)sm_wave_min((uint32_t)bi);
    __syncthreads();
    if (lane == 0) s.lo[wave] = (uint32_t)bi;
    __syncthreads();
    for (int w = 0; w < kSmWaves; ++w) bi = min(bi, (int)s.lo[w]);
    return bi;
  }

  // --- weights and bins ------------------------------------------------------
  __device__ __forceinline__ double weight_d(float l) const {  // an integer
    if (endless) return l == best ? kSmOne : 0.;
    return sm_exp2(((double)l - (double)best) * inv, s.tab);  // of the largest itself: exactly one
  }
  __device__ __forceinline__ void weights(const float (&x)[4], double (&w)[4]) const {
    if (endless) {
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = x[q] == best ? kSmOne : 0.;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = sm_exp2(((double)x[q] - (double)best) * inv, s.tab);
    }
  }
  __device__ __forceinline__ uint64_t weight(float l) const {
    return (uint64_t)__double_as_longlong(weight_d(l) + 4503599627370496.) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ int bin_of(float l) const {  // by the distance from the largest
    return l == best ? 0 : (int)fminf((best - l) * scale, (float)(kSmBins - 1));
  }
  __device__ __forceinline__ bool above(int e, float l) const {
    const uint32_t key = sm_key(l);
    return key > kk || (key == kk && e <= last_tie);
  }
  __device__ __forceinline__ uint64_t kept(int e, float l) const {
    if (!above(e, l)) return 0;
    const uint64_t w = weight(l);
    return w >= wmin ? w : 0;
  }
  __device__ __forceinline__ uint64_t need_of(uint64_t sum) const {  // what top-p asks of sum, at least 1
    bool rest;
    const uint64_t need = sm_mul_frac(sum, p > 0.f ? p : 0.f, rest);
    return rest || need == 0 ? need + 1 : need;
  }
  __device__ __forceinline__ uint64_t goal(uint64_t total) const {
    bool rest;
    return sm_mul_frac(total, u, rest);
  }

  // The least logit of bins 0..b (bin_of falls as the logit rises): a 64-ary search over
  // the keys by one wave.
  __device__ __forceinline__ float least_of(int b) const {
    if (b < 0) return NAN;  // none compares at or above it
    if (b >= kSmBins - 1) return -INFINITY;
    uint32_t lo = 0, hi = sm_key(best);  // bin_of(best) is 0; keys below -inf's are NaN, in the last bin
    while (lo < hi) {
      const uint32_t step = (hi - lo) / 64 + 1;
      const uint32_t at = min(lo + lane * step, hi);
      const uint64_t in = __ballot(bin_of(sm_logit(at)) <= b);
      if (in == 0) {
        lo += 63 * step + 1;
      } else {
        const uint32_t f = __builtin_ctzll(in);
        hi = min(lo + f * step, hi);
        if (f) lo += (f - 1) * step + 1;
      }
    }
    return sm_logit(hi);
  }
  // The logits of bins [b0, b1] are x with x >= from and not x >= past; the list is empty then.
  __device__ __forceinline__ void bin_range(int b0, int b1, float& from, float& past) {
    __syncthreads();
    if (wave < 2) {
      const float l = least_of(wave == 0 ? b1 : b0 - 1);
      if (lane == 0) s.max[wave] = l;
    }
    if (t == 0) s.count = 0;
    __syncthreads();
    from = s.max[0];
    past = s.max[1];
  }
  __device__ __forceinline__ void list(int e, float l) {
    const uint32_t at = atomicAdd(&s.count, 1u);
    if (at < LIST) {
      s.list_key[at] = sm_key(l);
      s.list_idx[at] = e;
    }
  }
  // --- the list ----------------------------------------------------------------
  // Tokens of bins [b0, b1] to the list; false if they are more than room. With
  // `drawable`, without those whose weight is certainly 0 (masked ones, above all): they
  // are never drawn, come last in the order and add to no sum.
  __device__ __forceinline__ bool collect(int b0, int b1, uint32_t room, bool drawable) {
    const float reach = drawable ? (float)inv : 0.f;
    float from, past;
    bin_range(b0, b1, from, past);
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (x[q] >= from && !(x[q] >= past) && e + q < w_end && !((best - x[q]) * reach > 47.f)) list(e + q, x[q]);
    });
    __syncthreads();
    nlist = (int)min(s.count, (uint32_t)LIST);
    return s.count <= room;
  }
  // One pass over the weights: all of them, those of the bins before b, and of these what
  // min_p leaves; the tokens of bin b that weigh anything to the list, and their weight.
  // false: more than the list holds.
  struct Split {
    uint64_t all, before, kept, at;  // the thread's
  };
  __device__ __forceinline__ bool split(int b, Split& sp) {
    float from, past;
    bin_range(b, b, from, past);
    // integers up to 512 logits x 2^44 a thread: exact in 53 bits
    double all = 0., before = 0., at = 0., left_out = 0.;
    const double least = (double)wmin;
    each([&](int e, const float (&x)[4]) {
      double w[4];
      weights(x, w);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        all += w[q];
        before = fma(w[q], x[q] >= past ? 1. : 0., before);
      }
      if (wmin) {  // uniform
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (x[q] >= past && w[q] < least) left_out += w[q];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (x[q] >= from && !(x[q] >= past) && w[q] > 0.) {
          at += w[q];
          list(e + q, x[q]);
        }
    });
    sp.all = (uint64_t)all;
    sp.before = (uint64_t)before;
    sp.at = (uint64_t)at;
    sp.kept = (uint64_t)(before - left_out);
    __syncthreads();
    nlist = (int)min(s.count, (uint32_t)LIST);
    return s.count <= LIST;
  }
  // The bin in which top-p probably ends, by 32-bit weights in units of 2^-31.
  __device__ __forceinline__ int likely_bin() {
    if (endless) return 0;
    const float f = (float)fmin(inv, 1e30);
    __syncthreads();
    s.hist[t] = 0;
    __syncthreads();
    each([&](int, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float d = best - x[q];
        const uint32_t m = (uint32_t)__builtin_amdgcn_exp2f(fmaxf(fmaf(d, -f, 31.f), -1.f));  // inf * 0 is 0 here
        if (m) atomicAdd(&s.hist[(int)fminf(d * scale, (float)(kSmBins - 1))], (unsigned long long)m);
      }
    });
    __syncthreads();
    uint64_t need, before;
    return (int)top_p_bin(s.hist[t], need, before);
  }
  // The bin that holds the k-th of the threads' largest logits (of `mine`, of the threads
  // that hold any): every one of the first k tokens is in it or before.
  __device__ __forceinline__ int guess_bin(uint64_t of) {
    __syncthreads();
    s.hist[t] = 0;
    __syncthreads();
    if (first_of(0) < w_end) atomicAdd(&s.hist[bin_of(mine)], 1ull);
    __syncthreads();
    uint64_t before;
    return (int)find_bin(s.hist[t], 0, of, before);
  }
  template <typename F>
  __device__ __forceinline__ void over_list(F f) const {
    for (int e = t; e < nlist; e += kSmThreads) f(s.list_key[e]);
  }
  template <typename F>
  __device__ __forceinline__ void over_row(F f) {
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < w_end) f(sm_key(x[q]));
    });
  }
  // The token of a list of at most kSmFew: of its n_kept first -- larger logits first,
  // lower indexes first among equals -- those whose weight reaches need(weight of these),
  // with top-p; of these the ones min_p leaves, by index. An entry's place is the number
  // that come before it, the sum of the kept tokens of lower index likewise.
  __device__ __forceinline__ uint64_t entry(int e) const {
    return ((uint64_t)s.list_key[e] << 32) | (uint32_t)~s.list_idx[e];
  }
  __device__ __forceinline__ uint64_t ordered_few() {  // the thread's entry of the list in order; 0 past it
    __syncthreads();
    s.hist[t] = 0;
    __syncthreads();
    const int mine_e = t >> 2;  // four threads an entry, a quarter of the comparisons each
    const uint64_t own = mine_e < nlist ? entry(mine_e) : 0;
    uint32_t place = 0;
    if (mine_e < nlist) {
#pragma unroll 4
      for (int e = t & 3; e < nlist; e += 4) place += entry(e) > own;
    }
    place += sm_dpp<kSmQuad1, 0xf>(place, 0);
    place += sm_dpp<kSmQuad2, 0xf>(place, 0);
    if ((t & 3) == 0 && mine_e < nlist) s.hist[place] = own;
    __syncthreads();
    return s.hist[t];
  }
  template <typename N>
  __device__ __forceinline__ int token_of_few(int n_kept, N need) {
    const uint64_t v = ordered_few();
    const uint32_t key = (uint32_t)(v >> 32), idx = ~(uint32_t)v;
    uint64_t w = t < nlist ? weight(sm_logit(key)) : 0;
    if (has_p) {
      uint64_t all;
      const uint64_t before = block_scan(w, all);
      if (t == n_kept - 1) s.u64 = before + w;
      __syncthreads();
      const uint64_t least = need((uint64_t)s.u64);
      if (before < least && before + w >= least) s.u32 = t;
      __syncthreads();
      n_kept = (int)s.u32 + 1;
    }
    if (w < wmin || t >= n_kept) w = 0;
    __syncthreads();
    s.hist[t] = w;
    if (t < n_kept) s.list_idx[t] = idx;
    __syncthreads();
    const int e0 = t >> 2;
    const bool in = e0 < n_kept;
    const uint32_t idx0 = in ? s.list_idx[e0] : 0;
    uint64_t before = 0, total = 0;
    if (in) {
#pragma unroll 4
      for (int e = t & 3; e < n_kept; e += 4) {
        const uint64_t o = s.hist[e];
        total += o;
        before += s.list_idx[e] < idx0 ? o : 0;
      }
    }
    total = sm_dpp_add<kSmQuad2, 0xf>(sm_dpp_add<kSmQuad1, 0xf>(total));
    before = sm_dpp_add<kSmQuad2, 0xf>(sm_dpp_add<kSmQuad1, 0xf>(before));
    if (in && (t & 3) == 0) {
      const uint64_t target = goal(total);
      if (before <= target && before + (uint64_t)s.hist[e0] > target) s.u32 = idx0;
    }
    __syncthreads();
    return (int)s.u32;
  }

  // The shortest prefix of the kept tokens whose measure (1 or the weight), on top of
  // base, reaches need. over(f) calls f(key) for tokens that include all that may end
  // it; equal keys may all be there, the kept ties count as ties.
  template <typename O>
  __device__ __forceinline__ void refine(O over, uint64_t base, uint64_t need, bool by_weight) {
    const uint32_t k0 = kk;
    const uint64_t t0 = ties;
    uint32_t lo = 0xffffffffu, hi = 0;
    over([&](uint32_t key) {
      if (key > k0 || (t0 && key == k0)) {
        lo = min(lo, key);
        hi = max(hi, key);
      }
    });
    block_range(lo, hi);
    // digits of hi - key, so that larger keys come first
    const int bits = 32 - __clz((int)((hi - lo) | 1u));
    int shift = bits;
    uint32_t prefix = 0;
    while (shift > 0) {  // uniform
      const int width = min(10, shift), next = shift - width;
      const uint32_t mask = (1u << width) - 1;
      __syncthreads();
      s.hist[t] = 0;
      __syncthreads();
      auto add = [&](uint32_t key, uint64_t m) {
        const uint32_t off = hi - key;
        if (shift == bits || off >> shift == prefix) atomicAdd(&s.hist[(off >> next) & mask], (unsigned long long)m);
      };
      over([&](uint32_t key) {
        if (key > k0 && key >= lo && key <= hi) {
          const uint64_t m = by_weight ? weight(sm_logit(key)) : 1;
          if (m) add(key, m);
        }
      });
      if (t == 0 && t0 && k0 >= lo && k0 <= hi) add(k0, t0 * (by_weight ? weight(sm_logit(k0)) : 1));
      __syncthreads();
      const uint32_t d = find_bin(s.hist[t], base, need, base);
      prefix = (prefix << width) | d;
      shift = next;
    }
    kk = hi - prefix;
    const uint64_t one = by_weight ? weight(sm_logit(kk)) : 1;
    ties = (need - base + one - 1) / one;  // >= 1; no more than there are, since they reach need
    uint64_t equal = 0;
    over([&](uint32_t key) { equal += key == kk; });
    ties_left = block_sum(equal) - ties;
  }
  __device__ __forceinline__ void refine_list(uint64_t base, uint64_t need, bool by_weight) {
    refine([&](auto f) { over_list(f); }, base, need, by_weight);
    ties_listed = true;
  }
  // top-p's last kept token: the list (all of its bin's that weigh anything) in order,
  // on top of base, reaches need at it.
  __device__ __forceinline__ void border(uint64_t base, uint64_t need) {
    if (nlist > kSmFew) {
      refine_list(base, need, true);
      if (ties_left) last_listed_tie();
      return;
    }
    const uint64_t v = ordered_few();
    const uint64_t w = t < nlist ? weight(sm_logit((uint32_t)(v >> 32))) : 0;
    uint64_t all;
    const uint64_t before = base + block_scan(w, all);
    if (before < need && before + w >= need) s.u64 = v;
    __syncthreads();
    kk = (uint32_t)(s.u64 >> 32);
    last_tie = (int)~(uint32_t)s.u64;
  }
  __device__ __forceinline__ void refine_row(uint64_t need, bool by_weight) {
    refine([&](auto f) { over_row(f); }, 0, need, by_weight);
    ties_listed = false;
  }
  __device__ __forceinline__ uint64_t list_sum() {  // weight of the kept tokens, all of them listed
    uint64_t sum = 0;
    over_list([&](uint32_t key) {
      if (key > kk) sum += weight(sm_logit(key));
    });
    sum = block_sum(sum);
    return ties ? sum + ties * weight(sm_logit(kk)) : sum;
  }
  // The index of the last kept tie, from a list that holds all of them.
  __device__ __forceinline__ void last_listed_tie() {
    int lo = 0, hi = V - 1;
    while (lo < hi) {  // uniform: the least index up to which there are enough
      const int mid = (lo + hi) >> 1;
      uint64_t n = 0;
      for (int e = t; e < nlist; e += kSmThreads) n += s.list_key[e] == kk && (int)s.list_idx[e] <= mid;
      if (block_sum(n) >= ties) hi = mid;
      else lo = mid + 1;
    }
    last_tie = lo;
  }

  // --- the token ---------------------------------------------------------------
  // The lane's 4 logits of step c, of 256, of a share [from, to) of the row; in LDS if
  // it is wave `share`'s.
  __device__ __forceinline__ void step_of(int from, int to, int share, int c, float (&x)[4]) const {
    if constexpr (CAP > 0) {
      if (share >= 0) {
        Elem<float>::unpack(s.keep[c * kSmThreads + 64 * share + lane], x);
        return;
      }
    }
    const int e = from + 256 * c + 4 * lane;
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = e + q < to ? row[e + q] : 0.f;
  }
  // Lowest index of [from, to), in steps of 256 that seg has the sums of, whose
  // running sum of measure(index, logit), from base on, exceeds target.
  template <typename M>
  __device__ __forceinline__ int find_in(int from, int to, int share, uint64_t base, uint64_t target, M measure) {
    __syncthreads();
    if (wave == 0) {
      const int ns = (to - from + 255) / 256;
      for (int s0 = 0; s0 < ns; s0 += 64) {
        const uint64_t own = s0 + lane < ns ? (uint64_t)s.seg[s0 + lane] : 0;
        const uint64_t inc = sm_wave_scan(own);
        const uint64_t run = base + inc - own;
        const uint64_t hit = __ballot(run <= target && run + own > target);
        if (hit) {
          const int b = __builtin_ctzll(hit);
          const uint64_t at = (uint64_t)__shfl((unsigned long long)run, b, 64);
          // the step's 256 logits again, 4 a lane
          const int e = from + (s0 + b) * 256 + 4 * lane;
          float x[4];
          step_of(from, to, share, s0 + b, x);
          uint64_t v[4], sum = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            v[q] = e + q < to ? measure(e + q, x[q]) : 0;
            sum += v[q];
          }
          uint64_t r2 = at + sm_wave_scan(sum) - sum;
          if (r2 <= target && r2 + sum > target) {
            int q = 0;
            while (q < 3 && r2 + v[q] <= target) r2 += v[q++];
            s.u32 = (uint32_t)(e + q);
          }
          break;
        }
        base += sm_last_lane(inc);
      }
    }
    __syncthreads();
    return (int)s.u32;
  }
  // The same over one share [from, to), whose steps the workgroup adds up first.
  template <typename M>
  __device__ __forceinline__ int find_share(int from, int to, int share, uint64_t base, uint64_t target, M measure) {
    __syncthreads();  // other threads' logits
    for (int c = wave; c * 256 < to - from; c += kSmWaves) {
      const int e = from + 256 * c + 4 * lane;
      float x[4];
      step_of(from, to, share, c, x);
      uint64_t v = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) v += e + q < to ? measure(e + q, x[q]) : 0;
      v = sm_wave_sum(v);
      if (lane == 0) s.seg[c] = v;
    }
    return find_in(from, to, share, base, target, measure);
  }
  template <typename M>
  __device__ __forceinline__ uint64_t own_sum(M measure) {  // the thread's
    uint64_t sum = 0;
    each([&](int e, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) sum += e + q < w_end ? measure(e + q, x[q]) : 0;
    });
    return sum;
  }
  // The same over the row, for the target that aim(sum over the row) gives: the waves'
  // sums say whose share it is in.
  template <typename M, typename A>
  __device__ __forceinline__ int find(M measure, A aim) {
    return find_by_waves(measure, aim(share_sum(own_sum(measure))));
  }
  template <typename M>
  __device__ __forceinline__ int find_by_waves(M measure, uint64_t target) {  // from the waves' sums
    uint64_t base = 0, upto = 0;
    int w = -1;
    do {  // at most 16 waves; their sums exceed target
      base = upto;
      upto += s.share[++w];
    } while (upto <= target && w < kSmWaves - 1);
    const int from = begin + w * per_wave;
    return find_share(from, min(from + per_wave, end), w, base, target, measure);
  }
  __device__ __forceinline__ int listed_token() {  // every kept token is in the list
    const int ns = (V + 255) / 256;
    __syncthreads();
    for (int e = t; e < ns; e += kSmThreads) s.seg[e] = 0;
    __syncthreads();
    uint64_t sum = 0;
    for (int e = t; e < nlist; e += kSmThreads) {
      const uint64_t w = kept((int)s.list_idx[e], sm_logit(s.list_key[e]));
      sum += w;
      if (w) atomicAdd(&s.seg[s.list_idx[e] >> 8], (unsigned long long)w);
    }
    const uint64_t total = block_sum(sum);
    return find_in(0, V, -1, 0, goal(total), [&](int e, float l) { return kept(e, l); });
  }
  // Drops what no k-th token's bin reaches from a list that holds the first k tokens.
  __device__ __forceinline__ void thin_list() {
    __syncthreads();
    s.hist[t] = 0;
    __syncthreads();
    uint32_t key[LIST / kSmThreads], idx[LIST / kSmThreads];
#pragma unroll
    for (int c = 0; c < LIST / kSmThreads; ++c) {
      const int e = c * kSmThreads + t;
      key[c] = e < nlist ? s.list_key[e] : 0;
      idx[c] = e < nlist ? s.list_idx[e] : 0;
      if (e < nlist) atomicAdd(&s.hist[bin_of(sm_logit(key[c]))], 1ull);
    }
    if (t == 0) s.count = 0;
    __syncthreads();
    uint64_t before;
    const int b = (int)find_bin(s.hist[t], 0, (uint64_t)k, before);
#pragma unroll
    for (int c = 0; c < LIST / kSmThreads; ++c)
      if (c * kSmThreads + t < nlist && bin_of(sm_logit(key[c])) <= b) {
        const uint32_t at = atomicAdd(&s.count, 1u);
        s.list_key[at] = key[c];
        s.list_idx[at] = idx[c];
      }
    __syncthreads();
    nlist = (int)s.count;
  }
  // A list that holds the first k tokens, or all that can be drawn, and whatever else:
  // top-k, top-p and the token.
  __device__ __forceinline__ int token_of_list() {
    if (nlist > kSmFew && nlist > k) thin_list();
    if (nlist <= kSmFew) return token_of_few(min(k, nlist), [&](uint64_t sum) { return need_of(sum); });
    if (nlist > k) {
      refine_list(0, (uint64_t)k, false);
    } else {  // all of the list, and nothing that is not in it
      uint32_t lo = 0xffffffffu, hi = 0;
      over_list([&](uint32_t key) { lo = min(lo, key); });
      block_range(lo, hi);
      kk = lo - 1;
    }
    if (has_p) refine_list(0, need_of(list_sum()), true);
    if (ties_left) last_listed_tie();
    return listed_token();
  }

  // The row's token, by this workgroup alone; largest() and parameters() came before.
  __device__ __forceinline__ int token() {
    if (has_k) {
      // V / 4 threads, or 960 of the 1024, hold logits
      if (V <= LIST || k <= min(kSmGuess, V / 4)) {
        const int b = V <= LIST ? kSmBins - 1 : guess_bin((uint64_t)k);
        if (collect(0, b, LIST, true)) return token_of_list();
      }
      __syncthreads();
      s.hist[t] = 0;
      __syncthreads();
      each([&](int e, const float (&x)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (e + q < w_end) atomicAdd(&s.hist[bin_of(x[q])], 1ull);
      });
      __syncthreads();
      uint64_t before;
      const uint32_t b = find_bin(s.hist[t], 0, (uint64_t)k, before);
      const uint64_t upto = before + s.hist[b];
      if (upto <= LIST) {
        collect(0, b, LIST, true);
        return token_of_list();
      }
      if (collect(b, b, LIST, false)) refine_list(before, (uint64_t)k, false);
      else refine_row((uint64_t)k, false);
    }
    if (has_p && !has_k) {
      Split sp;
      const bool fits = split(likely_bin(), sp);
      uint64_t v[4] = {sp.all, sp.before, sp.at, sp.kept};
      block_sums(v);
      const uint64_t need = need_of(v[0]), before = v[1];
      if (fits && before < need && before + v[2] >= need) {
        border(before, need);
        uint64_t more = 0;  // kept ones of the listed tokens
        for (int e = t; e < nlist; e += kSmThreads) {
          const int idx = (int)s.list_idx[e];
          const uint64_t w = kept(idx, sm_logit(s.list_key[e]));
          if (w) atomicAdd(&s.share[(idx - begin) / per_wave], (unsigned long long)w);
          more += w;
        }
        return find_by_waves([&](int e, float l) { return kept(e, l); }, goal(v[3] + block_sum(more)));
      }
    }
    if (has_p) {  // behind a top-k, or with a bin of too many tokens, or at a bin's edge
      const uint64_t own = weigh_bins(s.hist);
      uint64_t need, before;
      const int b = (int)top_p_bin(own, need, before);
      if (collect(b, b, LIST, true)) refine_list(before, need, true);
      else refine_row(need, true);
    }
    if (!has_k && !has_p) {
      Split sp;
      split(kSmBins, sp);
      return find_by_waves([&](int e, float l) { return kept(e, l); }, goal(share_sum(sp.kept)));
    }
    if (ties && ties_left) {
      if (ties_listed) {
        last_listed_tie();
      } else {
        const uint64_t nth = ties - 1;
        last_tie = find([&](int, float l) -> uint64_t { return sm_key(l) == kk ? 1 : 0; },
                        [&](uint64_t) { return nth; });
        __syncthreads();
      }
    }
    return find([&](int e, float l) { return kept(e, l); }, [&](uint64_t sum) { return goal(sum); });
  }
  // The kept tokens' weights by bin, in LDS; the thread's bin.
  __device__ __forceinline__ uint64_t weigh_bins(unsigned long long* hist) {
    const uint32_t k0 = kk;
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
    if (t == 0 && ties) atomicAdd(&hist[bin_of(sm_logit(k0))], (unsigned long long)(ties * weight(sm_logit(k0))));
    __syncthreads();
    return hist[t];
  }
  __device__ __forceinline__ void finish(int id) {
    if (t == 0) argmax_finish(i, id, a.out, a.ring, a.ring_rows, a.ring_len, a.expect, a.accept);
  }
};

template <int CAP>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SmArgs a) {
  __shared__ __align__(16) SmShared<CAP, 2048> sh;
  Sm<CAP, 2048> m(a, sh, blockIdx.x, 0, a.V);
  m.largest();
  m.finish(m.parameters() ? m.token() : m.first_best());
}

// --- long rows: grid (slab, row) but for the last ------------------------------
using SmSlab = Sm<-kSmSlab, 2048>;
using SmSlabShared = SmShared<-kSmSlab, 2048>;

__global__ __launch_bounds__(kSmThreads) void sample_largest_kernel(SmArgs a, SmRowWs* wss) {
  __shared__ __align__(16) SmSlabShared sh;
  const int slab = blockIdx.x;
  SmSlab m(a, sh, blockIdx.y, slab * kSmSlab, min((slab + 1) * kSmSlab, a.V));
  SmRowWs& ws = wss[blockIdx.y];
  m.largest();
  if (m.t == 0) {
    ws.max[slab] = m.best;
    ws.min[slab] = m.low;
    ws.nan[slab] = m.nan;
  }
  if (slab == 0) {
    ws.hist[m.t] = 0;
    if (m.t == 0) ws.count = 0;
  }
}

// What the row's workgroup can do with the slabs' lists.
__device__ __forceinline__ bool sm_listed(const SmSlab& m) { return m.has_k && m.k <= kSmGuess; }

__device__ __forceinline__ void sm_append(SmSlab& m, SmRowWs& ws) {  // the slab's list to the row's
  const uint32_t n = m.s.count;
  if (m.t == 0) m.s.u32 = atomicAdd(&ws.count, n <= 2048 ? n : kSmRowList + 1);
  __syncthreads();
  const uint32_t at = m.s.u32;
  for (uint32_t e = m.t; e < (uint32_t)m.nlist && at + e < kSmRowList; e += kSmThreads) {
    ws.key[at + e] = m.s.list_key[e];
    ws.idx[at + e] = m.s.list_idx[e];
  }
}

// With top-k, the tokens that may be among the first k: each slab's first k and a few.
// With top-p alone, the weights by bin.
__global__ __launch_bounds__(kSmThreads) void sample_bins_kernel(SmArgs a, SmRowWs* wss) {
  __shared__ __align__(16) SmSlabShared sh;
  const int slab = blockIdx.x;
  SmSlab m(a, sh, blockIdx.y, slab * kSmSlab, min((slab + 1) * kSmSlab, a.V));
  SmRowWs& ws = wss[blockIdx.y];
  m.largest_of(ws, gridDim.x);
  if (!m.parameters()) return;
  __syncthreads();  // the table
  if (sm_listed(m)) {
    m.mine = -INFINITY;
    m.each([&](int, const float (&x)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) m.mine = fmaxf(m.mine, x[q]);
    });
    const int len = m.end - m.begin;
    const int b = len <= kSmShort || m.k > min(kSmGuess, len / 4) ? kSmBins - 1 : m.guess_bin((uint64_t)m.k);
    m.collect(0, b, 2048, true);
    sm_append(m, ws);
  } else if (m.has_p && !m.has_k) {
    const uint64_t own = m.weigh_bins(sh.hist);
    if (own) atomicAdd(&ws.hist[m.t], (unsigned long long)own);
  }
}

// Without top-k: the kept weight of each wave's share, with top-p up to the border's
// bin, whose tokens go to the list.
__global__ __launch_bounds__(kSmThreads) void sample_shares_kernel(SmArgs a, SmRowWs* wss) {
  __shared__ __align__(16) SmSlabShared sh;
  const int slab = blockIdx.x;
  SmSlab m(a, sh, blockIdx.y, slab * kSmSlab, min((slab + 1) * kSmSlab, a.V));
  SmRowWs& ws = wss[blockIdx.y];
  m.largest_of(ws, gridDim.x);
  if (!m.parameters() || m.has_k) return;
  __syncthreads();  // the table
  int b = kSmBins;
  if (m.has_p) {
    uint64_t need, before;
    b = (int)m.top_p_bin(ws.hist[m.t], need, before);
  }
  SmSlab::Split sp;
  m.split(b, sp);
  if (m.has_p) sm_append(m, ws);
  const uint64_t sum = sm_wave_sum(sp.kept);
  if (m.lane == 0) ws.share[slab * kSmWaves + m.wave] = sum;
}

__global__ __launch_bounds__(kSmThreads) void sample_row_kernel(SmArgs a, SmRowWs* wss, int slabs) {
  __shared__ __align__(16) SmShared<0, kSmRowList> sh;
  SmRowWs& ws = wss[blockIdx.x];
  Sm<0, kSmRowList> m(a, sh, blockIdx.x, 0, a.V);
  // what the launches before left, all loads at once
  const uint32_t count = ws.count;
  const uint64_t bin = ws.hist[m.t];
  uint64_t own = ws.share[min(m.t, slabs * kSmWaves - 1)];
  const uint32_t key0 = ws.key[m.t], idx0 = ws.idx[m.t];
  auto take_list = [&]() {
    m.nlist = (int)count;
    for (int e = m.t; e < m.nlist; e += kSmThreads) {
      sh.list_key[e] = e < kSmThreads ? key0 : ws.key[e];
      sh.list_idx[e] = e < kSmThreads ? idx0 : ws.idx[e];
    }
  };
  m.largest_of(ws, slabs);
  __syncthreads();  // the table
  if (!m.parameters()) {  // the first slab that has it
    const int l = min(m.lane, slabs - 1);
    const bool has = m.lane < slabs && (m.nan ? ws.nan[l] != 0 : ws.max[l] == m.best);
    const int slab = __builtin_ctzll(__ballot(has));
    Sm<0, kSmRowList> one(a, sh, blockIdx.x, slab * kSmSlab, min((slab + 1) * kSmSlab, a.V));
    one.best = m.best;
    one.nan = m.nan;
    m.finish(one.first_best());
    return;
  }
  const bool listed = m.has_k && m.k <= kSmGuess;
  if ((listed || (m.has_p && !m.has_k)) ? count > kSmRowList : m.has_k) {  // not prepared
    m.largest();
    m.finish(m.token());
    return;
  }
  if (listed) {
    take_list();
    __syncthreads();
    m.finish(m.token_of_list());
    return;
  }
  // the shares, at most 1024, one a thread; with top-p the kept ones of the listed tokens added
  if (m.t >= slabs * kSmWaves) own = 0;
  if (m.has_p) {
    take_list();
    uint64_t need, before;
    m.top_p_bin(bin, need, before);
    m.border(before, need);
    __syncthreads();
    sh.hist[m.t] = own;
    __syncthreads();
    for (int e = m.t; e < m.nlist; e += kSmThreads) {
      const int idx = (int)sh.list_idx[e], slab = idx / kSmSlab, lo = slab * kSmSlab;
      const uint64_t w = m.kept(idx, sm_logit(sh.list_key[e]));
      const int per_wave = (min(lo + kSmSlab, a.V) - lo + 63) / 64 * 4;
      if (w) atomicAdd(&sh.hist[slab * kSmWaves + (idx - lo) / per_wave], (unsigned long long)w);
    }
    __syncthreads();
    own = sh.hist[m.t];
  }
  uint64_t total;
  const uint64_t before = m.block_scan(own, total), target = m.goal(total);
  if (before <= target && before + own > target) {
    sh.u32 = m.t;
    sh.u64 = before;
  }
  __syncthreads();
  const int slab = (int)sh.u32 / kSmWaves, w = (int)sh.u32 % kSmWaves;
  const uint64_t base = sh.u64;
  const int lo = slab * kSmSlab, hi = min(lo + kSmSlab, a.V), per_wave = (hi - lo + 63) / 64 * 4;
  const int from = lo + w * per_wave;
  __syncthreads();
  m.finish(m.find_share(from, min(from + per_wave, hi), -1, base, target,
                        [&](int e, float l) { return m.kept(e, l); }));
}

}  // namespace wfd

extern "C" {

size_t wfd_sample_workspace_bytes(int n, int vocab) {
  return n <= 0 || vocab <= wfd::kSmLong || vocab > wfd::kSmMaxVocab ? 0 : (size_t)n * sizeof(wfd::SmRowWs);
}

int wfd_sample(const float* logits, int64_t ld, const float* u, const float* temperature, const int32_t* top_k,
               const float* top_p, const float* min_p, int64_t* out, int64_t* ring, const int32_t* ring_rows,
               int64_t ring_len, const int64_t* expect, int32_t* accept, int n, int vocab, void* workspace,
               size_t ws_bytes, hipStream_t stream) {
  using namespace wfd;
  if (n < 0 || vocab <= 0 || ld < vocab) {
    set_error("wfd_sample: bad shape n=%d vocab=%d ld=%lld", n, vocab, (long long)ld);
    return kBadArg;
  }
  if (vocab > kSmMaxVocab || n > 65535) {
    set_error("wfd_sample: vocab=%d n=%d (at most %d and 65535)", vocab, n, kSmMaxVocab);
    return kUnsupported;
  }
  if (n == 0) return kOk;
  const size_t need = wfd_sample_workspace_bytes(n, vocab);
  if (!logits || !u || !out || (ring && (!ring_rows || ring_len <= 0)) || (!expect != !accept) ||
      (need && !workspace)) {
    set_error("wfd_sample: null pointer argument (ring needs ring_rows and a length; expect and accept go together)");
    return kBadArg;
  }
  if (need && ((uintptr_t)workspace & 15)) {
    set_error("wfd_sample: workspace must be 16-byte aligned");
    return kBadArg;
  }
  if (ws_bytes < need) {
    set_error("wfd_sample: workspace %zu bytes < required %zu", ws_bytes, need);
    return kWorkspace;
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
  const dim3 block(kSmThreads);
  if (vocab <= 2 * kSmChunk) {
    hipLaunchKernelGGL(sample_kernel<2 * kSmChunk>, dim3(n), block, 0, stream, a);
  } else if (vocab <= kSmLong) {
    hipLaunchKernelGGL(sample_kernel<kSmLong>, dim3(n), block, 0, stream, a);
  } else {
    SmRowWs* ws = (SmRowWs*)workspace;
    const int slabs = (vocab + kSmSlab - 1) / kSmSlab;
    const dim3 grid(slabs, n);
    hipLaunchKernelGGL(sample_largest_kernel, grid, block, 0, stream, a, ws);
    if (top_k || top_p) hipLaunchKernelGGL(sample_bins_kernel, grid, block, 0, stream, a, ws);
    hipLaunchKernelGGL(sample_shares_kernel, grid, block, 0, stream, a, ws);
    hipLaunchKernelGGL(sample_row_kernel, dim3(n), block, 0, stream, a, ws, slabs);
  }
  return launch_status("wfd_sample");
}

}  // extern "C"
