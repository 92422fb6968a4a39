// Log probabilities of given tokens, the entropy of their distributions and the
// most probable tokens.
//
//   log p_t = (l_t - m) - log Z,   Z = sum_j e^(l_j - m),   m = max l
//   entropy = log Z - sum_j e^(l_j - m) (l_j - m) / Z
//
// The logits are read once: a workgroup holds up to 32768 of a row in registers, 32
// a thread, and goes over them there three times (largest, sums, candidates for the
// top); 256, 512 or 1024 threads by what the row needs. A workgroup asks for its next
// row before it ranks this one's candidates, which is why its barriers wait for LDS
// alone. Longer rows are cut into equal slabs, whose results a second launch joins; the
// cut follows from the vocabulary alone, so a row's bits do not depend on its fellows.
//
// Z is summed without its largest terms, which are counted instead: log Z is log1p of
// what is left, and that is all there is to a confident row's log probability. A factor
// that clamps to 0 for d = 0 and 1 for all others leaves them out, for one instruction.
//
// Top tokens: the a.top-th best of 256 groups of threads has at least a.top logits at or
// before its best, so what ranks before that are the candidates (74 of random logits for
// 64 tokens, with 64 groups 300); each counts those that rank before it, which is its
// place. A row with a NaN, or with more candidates than the list takes (equal logits by
// the thousand), finds its tokens one after the other instead.
//
// Bound by the row's bytes, for bf16 by the instructions, 17 a logit, 7 of them the sums'
// (the VALU is busy for 81 % of the time): 2048 rows of 32000 fp32 logits 58 us (4.5 TB/s)
// without tokens, 71 with the 20 best (66 with the card not at its power limit; 75 before
// the next row was asked for early), bf16 44 and 59; one row 7 and 11 us, most of it the
// way of its bytes and five exchanges through LDS. Rows of 128000: 512 fp32 57 and 71 us
// (4.6 TB/s), bf16 48 and 70, one fp32 row 10 and 16.
#include "wfd_common.h"

namespace wfd {

constexpr int kLpPer = 32;  // logits of a thread
constexpr int kLpMaxThreads = 1024;
constexpr int kLpSlab = kLpPer * kLpMaxThreads;
constexpr int kLpMaxTop = 64;
constexpr int kLpGroups = 256;
constexpr int kLpList = 2048;           // candidates
constexpr int kLpResident = 256 * 2048;  // threads that the card holds; rows past them wait for their turn
constexpr float kLpLog2e = 1.44269504088896340736f;

struct LpArgs {
  const void* logits;
  int64_t ld;
  const int64_t* ids;
  float *out, *entropy, *top_val;
  int64_t* top_id;
  float* sums;     // with several slabs: m, z, t of each
  uint64_t* tops;  // and its top tokens
  int n, V, top, parts, slab;
};

// Tokens in the order of the argmax (NaN first, equal ones by index) as falling numbers.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t j) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 is 0
  const uint32_t k = x != x ? ~0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (uint64_t)k << 32 | (uint32_t)~j;
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k ^ (~(uint32_t)((int32_t)k >> 31) | 0x80000000u));
}
__device__ __forceinline__ int lp_index(uint64_t key) { return (int)~(uint32_t)key; }

// LDS is all that a workgroup's waves exchange; loads of the next row are not waited for.
__device__ __forceinline__ void lp_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * kLpLog2e); }

template <int CTRL>
__device__ __forceinline__ uint32_t lp_dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
// Lanes' partners in aligned groups of 2, 4, 8, 16 lanes, whose halves agree.
template <int STEP>
__device__ __forceinline__ uint32_t lp_other(uint32_t x) {
  return STEP == 0 ? lp_dpp<0xB1>(x) : STEP == 1 ? lp_dpp<0x4E>(x) : STEP == 2 ? lp_dpp<0x141>(x) : lp_dpp<0x140>(x);
}
// The larger of three; a NaN, which the sums show, may or may not come through.
__device__ __forceinline__ float lp_max3(float a, float b, float c) {
  float x;  // fmaxf of loaded values costs an instruction more for each
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(x) : "v"(a), "v"(b), "v"(c));
  return x;
}
template <int STEP>
__device__ __forceinline__ int lp_other(int x) {
  return (int)lp_other<STEP>((uint32_t)x);
}
template <int STEP>
__device__ __forceinline__ float lp_other(float x) {
  return __uint_as_float(lp_other<STEP>(__float_as_uint(x)));
}
template <typename OP>
__device__ __forceinline__ float lp_wave(float x, OP op) {  // over the wave, the same in all lanes
  x = op(x, lp_other<0>(x));
  x = op(x, lp_other<1>(x));
  x = op(x, lp_other<2>(x));
  x = op(x, lp_other<3>(x));
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lp_wave_max(float x) {
  return lp_wave(x, [](float a, float b) { return lp_max3(a, b, b); });
}
__device__ __forceinline__ float lp_wave_sum(float x) {
  return lp_wave(x, [](float a, float b) { return a + b; });
}

// 16 bytes of a row that is aligned to its elements.
template <typename T>
struct LpChunk;
template <>
struct LpChunk<float> {
  static constexpr int N = 4;
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ void load(const float* p, float (&v)[N]) {
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = x[e];
  }
};
template <>
struct LpChunk<bf16_t> {
  static constexpr int N = 8;
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ void load(const bf16_t* p, float (&v)[N]) {
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = __uint_as_float(e & 1 ? x[e / 2] & 0xffff0000u : x[e / 2] << 16);
  }
};

// Z - 1, sum e d and the largest of two parts joined.
__device__ __forceinline__ void lp_join(float& m, float& z, float& t, float om, float oz, float ot) {
  if (om > m) {
    const float xm = m, xz = z, xt = t;
    m = om, z = oz, t = ot;
    om = xm, oz = xz, ot = xt;
  }
  if (om == -INFINITY) return;
  const float d = om - m, c = lp_exp(d);
  z += c * (1.f + oz);
  if (c != 0.f) t += c * fmaf(1.f + oz, d, ot);
}

// How many of a list rank before k; the list is read in eights.
__device__ __forceinline__ int lp_before(const uint64_t* list, int count, uint64_t k) {
  int before = 0;
  for (int o = 0; o < count; o += 8) {
    uint64_t x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = list[o + e];
#pragma unroll
    for (int e = 0; e < 8; ++e) before += o + e < count && x[e] > k;
  }
  return before;
}

__device__ __forceinline__ float lp_log_z(float m, float z) { return m - m == 0.f ? log1pf(z) : NAN; }

template <typename T>
__device__ __forceinline__ void lp_store(const LpArgs& a, int64_t i, float m, float z, float t, float logz) {
  if (a.ids) {
    const int64_t id = a.ids[i];
    a.out[i] = id >= 0 && id < a.V ? (Elem<T>::load((const T*)a.logits + i * a.ld + id) - m) - logz : NAN;
  }
  if (a.entropy) a.entropy[i] = logz - t / (1.f + z);
}

template <typename T, int TH>
__global__ __launch_bounds__(TH) __attribute__((amdgpu_waves_per_eu(8))) void logprobs_kernel(LpArgs a) {
  using Chunk = LpChunk<T>;
  constexpr int CH = Chunk::N, NC = kLpPer / CH, W = TH / 64;
  constexpr int PER = TH / kLpGroups;  // threads of a group
  __shared__ __align__(16) float max_lds[W], z_lds[W], t_lds[W];
  __shared__ int i_lds[W];
  __shared__ int ones_lds[W];
  __shared__ uint64_t group_lds[kLpGroups];
  __shared__ uint64_t least_lds;
  __shared__ int count_lds, best_lds;
  __shared__ __align__(16) uint64_t list_lds[kLpList];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t units = (int64_t)a.n * a.parts;
  float v[NC][CH];
  int64_t i;
  int first, len;
  const T* row;
  auto place = [&](int64_t u) {
    i = a.parts > 1 ? u / a.parts : u;
    first = (int)(u - i * a.parts) * a.slab;
    len = min(a.slab, a.V - first);
    row = (const T*)a.logits + i * a.ld + first;
  };
  auto load = [&](int64_t u) {
    place(u);
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < CH; ++e) v[c][e] = -INFINITY;
      const int j = CH * (tid + TH * c);
      if (j + CH <= len) Chunk::load(row + j, v[c]);
    }
    if (const int last = len / CH; len % CH && tid == last % TH) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (c == last / TH)
#pragma unroll
          for (int e = 0; e < CH; ++e)
            if (e < len % CH) v[c][e] = Elem<T>::load(row + CH * last + e);
    }
  };
  int64_t u = blockIdx.x;
  if (u < units) load(u);
  for (; u < units; u += gridDim.x) {  // uniform
    place(u);
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // or what follows from it stays in registers over the rows
    const int lane = tid & 63;
    // the largest, and the first chunk of the thread's with its largest
    auto chunk_max = [&](int c) {
      float x = lp_max3(v[c][0], v[c][1], v[c][2]);
#pragma unroll
      for (int e = 3; e < CH - 1; e += 2) x = lp_max3(x, v[c][e], v[c][e + 1]);
      return lp_max3(x, x, v[c][CH - 1]);
    };
    float lm = chunk_max(0);
    int lc = 0;
#pragma unroll
    for (int c = 1; c < NC; ++c) {
      const float x = chunk_max(c);
      lc = x > lm ? c : lc;
      lm = lp_max3(lm, lm, x);
    }
    const uint64_t lkey = lp_key(lm, lc * TH + tid);
    if (a.top > 1) {
      uint64_t k = lkey;
      auto step = [&](auto s) {
        constexpr int S = decltype(s)::value;
        const uint64_t o = (uint64_t)lp_other<S>((uint32_t)(k >> 32)) << 32 | lp_other<S>((uint32_t)k);
        k = o > k ? o : k;
      };
      if constexpr (PER > 1) step(std::integral_constant<int, 0>{});
      if constexpr (PER > 2) step(std::integral_constant<int, 1>{});
      if (tid % PER == 0) group_lds[tid / PER] = k;
    }
    if (const float x = lp_wave_max(lm); lane == 0) max_lds[wave] = x;
    if (tid == 0) {
      count_lds = 0;
      best_lds = INT_MAX;
    }
    lp_sync();
    // of the W waves' values, which the lanes of each 16 take
    auto over_waves = [&](auto x, auto op) {
      x = op(x, lp_other<0>(x));
      x = op(x, lp_other<1>(x));
      if constexpr (W > 4) x = op(x, lp_other<2>(x));
      if constexpr (W > 8) x = op(x, lp_other<3>(x));
      return x;
    };
    const auto add = [](auto x, auto y) { return x + y; };
    const float m = over_waves(max_lds[tid & (W - 1)], [](float x, float y) { return lp_max3(x, y, y); });
    const float mm = m == -INFINITY ? 0.f : m;
    float z = 0.f, t = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < CH; ++e) {
        const float d = v[c][e] - mm, p = lp_exp(d);
        // without the largest, whose p is 1: 0 x inf is a NaN, which clamps to 0, all other d go to 1
        z = fmaf(p, __builtin_amdgcn_fmed3f(d * -INFINITY, 0.f, 1.f), z);
        t = fmaf(p, fmaxf(d, -3e38f), t);  // 0, not NaN, where p is 0
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    int ones = 0;  // of the wave's logits, how many are the largest
    if (__builtin_amdgcn_ballot_w64(lm == m)) {  // uniform over the wave
      int best = INT_MAX;
#pragma unroll
      for (int c = NC - 1; c >= 0; --c)
#pragma unroll
        for (int e = CH - 1; e >= 0; --e) {
          ones += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[c][e] == m));
          best = v[c][e] == m ? CH * TH * c + e : best;
        }
      if (best != INT_MAX) atomicMin(&best_lds, best + CH * tid);
    }
    z = lp_wave_sum(z);
    t = lp_wave_sum(t);
    if (lane == 0) {
      z_lds[wave] = z;
      t_lds[wave] = t;
      ones_lds[wave] = ones;
    }
    if (a.top > 1 && wave == W - 1) {
      // the least number whose digits from the first on leave a.top groups or more, until they are
      // not many more (equal bf16 values would be told apart by their places, 20 digits on)
      uint64_t k[kLpGroups / 64], least = 0;
#pragma unroll
      for (int g = 0; g < kLpGroups / 64; ++g) k[g] = group_lds[64 * g + lane];
      for (int b = 63; b >= 0; --b) {  // uniform
        const uint64_t x = least | (uint64_t)1 << b;
        int in = 0;
#pragma unroll
        for (int g = 0; g < kLpGroups / 64; ++g) in += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k[g] >= x));
        if (in >= a.top) least = x;
        if (in >= a.top && in <= a.top + a.top / 4) break;
      }
      if (lane == 0) least_lds = least;
    }
    lp_sync();
    z = over_waves(z_lds[tid & (W - 1)], add);
    const bool nan = z != z;  // a NaN or +inf among the logits; uniform
    if (m != -INFINITY) z += (float)(over_waves(ones_lds[tid & (W - 1)], add) - 1);
    auto log_z = [&]() { return lp_log_z(m, z); };
    const uint64_t least = a.top > 1 ? least_lds : 0;
    auto store_top = [&](int k, uint64_t key) {  // key: of the index within the slab
      const int j = lp_index(key);
      if (a.parts > 1) {
        a.tops[u * a.top + k] = lp_key(lp_value(key), first + j);
      } else {
        a.top_val[u * a.top + k] = (lp_value(key) - m) - log_z();
        a.top_id[u * a.top + k] = j;
      }
    };
    // a slab of fewer logits than a.top leaves the rest as key 0, which ranks behind every logit
    if (a.parts > 1)
      for (int k = len + tid; k < a.top; k += TH) a.tops[u * a.top + k] = 0;
    if (wave == 0) t = over_waves(t_lds[tid & (W - 1)], add);
    if (tid == 0) {
      if (a.parts > 1) {
        a.sums[u * 3] = nan ? NAN : m;
        a.sums[u * 3 + 1] = z;
        a.sums[u * 3 + 2] = t;
      } else {
        lp_store<T>(a, i, m, z, t, log_z());
      }
    }
    if (a.top > 1 && !nan && lkey >= least) {
      // what ranks at or before the chunk of `least`; its value may lie between -inf and a NaN's
      const float tx = lp_value(max(least, (uint64_t)0x007fffff << 32));
      const uint32_t tc = ~(uint32_t)least;
      auto in = [&](float x, uint32_t chunk) { return x > tx || (x == tx && chunk <= tc); };
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t chunk = TH * c + tid;
        asm volatile("" : "+v"(chunk));  // not 32 indices for all rows
        if (in(chunk_max(c), chunk))
#pragma unroll
          for (int e = 0; e < CH; ++e)
            if (const int j = CH * (int)chunk + e; in(v[c][e], chunk) && j < len) {
              const int at = atomicAdd(&count_lds, 1);
              if (at < kLpList) list_lds[at] = lp_key(v[c][e], j);
            }
      }
    }
    if (u + gridDim.x < units) {  // uniform; on its way during the rest
      load(u + gridDim.x);
      place(u);
    }
    int count = 0;
    if (a.top > 1 && !nan) {
      lp_sync();
      count = count_lds;
      if (count <= kLpList)
        for (int s = tid; s < count; s += TH) {
          const uint64_t k = list_lds[s];
          const int before = lp_before(list_lds, count, k);
          if (before < a.top) store_top(before, k);
        }
    } else if (a.top == 1 && !nan) {
      if (tid == 0) store_top(0, lp_key(m, best_lds));
    }
    if (a.top && (nan || count > kLpList)) {  // uniform
      float lv = 0.f;
      int li = -1;
      for (int k = 0; k < min(a.top, len); ++k) {
        float bv = -INFINITY;
        int bi = INT_MAX;
        for (int j = tid; j < len; j += TH) {
          const float x = Elem<T>::load(row + j);
          float cv = lv;
          int ci = li;
          argmax_merge(cv, ci, x, j);  // (x, j) ranks before (lv, li): taken already
          if (li < 0 || ci != j) argmax_merge(bv, bi, x, j);
        }
#pragma unroll
        for (int s = 32; s >= 1; s >>= 1) argmax_merge(bv, bi, __shfl_xor(bv, s, 64), __shfl_xor(bi, s, 64));
        lp_sync();
        if (lane == 0) {
          max_lds[wave] = bv;
          i_lds[wave] = bi;
        }
        lp_sync();
        for (int w = 0; w < W; ++w) argmax_merge(bv, bi, max_lds[w], i_lds[w]);
        lv = bv;
        li = bi;
        if (tid == 0) store_top(k, lp_key(lv, li));
      }
    }
    lp_sync();  // the next row's writes
  }
}

// The slabs' results joined, a workgroup per row.
constexpr int kLpJoin = 256;
template <typename T>
__global__ __launch_bounds__(kLpJoin) void logprobs_join(LpArgs a) {
  __shared__ __align__(16) uint64_t list_lds[kLpList + kLpMaxTop];
  __shared__ uint64_t best_lds[kLpMaxTop];
  const int tid = threadIdx.x, lane = tid & 63;
  for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    float m = -INFINITY, z = 0.f, t = 0.f;
    bool nan = false;
    for (int p = lane; p < a.parts; p += 64) {
      const float* s = a.sums + (i * a.parts + p) * 3;
      nan |= s[0] != s[0];
      lp_join(m, z, t, s[0], s[1], s[2]);
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1)
      lp_join(m, z, t, __shfl_xor(m, s, 64), __shfl_xor(z, s, 64), __shfl_xor(t, s, 64));
    m = __builtin_amdgcn_ballot_w64(nan) ? NAN : __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(m)));
    z = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(z)));
    t = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(t)));
    const float logz = lp_log_z(m, z);
    if (tid == 0) lp_store<T>(a, i, m, z, t, logz);
    if (a.top) {
      const uint64_t* tops = a.tops + i * a.parts * a.top;
      const int64_t all = (int64_t)a.parts * a.top;
      int kept = 0;
      for (int64_t at = 0; at < all; at += kLpList) {  // the best so far, and as many more as the list takes
        const int more = (int)min(all - at, (int64_t)kLpList), count = kept + more;
        for (int s = tid; s < kept; s += kLpJoin) list_lds[s] = best_lds[s];
        for (int s = tid; s < more; s += kLpJoin) list_lds[kept + s] = tops[at + s];
        __syncthreads();
        for (int s = tid; s < count; s += kLpJoin) {
          const uint64_t k = list_lds[s];
          const int before = lp_before(list_lds, count, k);
          if (before < a.top) best_lds[before] = k;
        }
        kept = a.top;
        __syncthreads();
      }
      if (tid < a.top) {
        const uint64_t k = best_lds[tid];
        a.top_val[i * a.top + tid] = (lp_value(k) - m) - logz;
        a.top_id[i * a.top + tid] = lp_index(k);
      }
      __syncthreads();
    }
  }
}

// Equal slabs, of whole chunks of all lanes.
inline int lp_parts(int V) { return (V - 1) / kLpSlab + 1; }
inline int lp_slab(int V) {
  const int p = lp_parts(V);
  return p == 1 ? V : ((V - 1) / p + 512) / 512 * 512;
}

template <typename T>
void launch_logprobs(const LpArgs& a, hipStream_t st) {
  auto launch = [&](auto th) {
    constexpr int TH = decltype(th)::value;
    const int64_t units = (int64_t)a.n * a.parts;
    hipLaunchKernelGGL((logprobs_kernel<T, TH>), dim3((unsigned)std::min<int64_t>(units, kLpResident / TH)), dim3(TH), 0,
                       st, a);
  };
  if (a.slab <= kLpPer * 256)
    launch(std::integral_constant<int, 256>{});
  else if (a.slab <= kLpPer * 512)
    launch(std::integral_constant<int, 512>{});
  else
    launch(std::integral_constant<int, 1024>{});
  if (a.parts > 1)
    hipLaunchKernelGGL(logprobs_join<T>, dim3(std::min(a.n, kLpResident / kLpJoin)), dim3(kLpJoin), 0, st, a);
}

}  // namespace wfd

extern "C" {

size_t wfd_logprobs_workspace_bytes(int n, int vocab, int top) {
  using namespace wfd;
  if (n <= 0 || vocab <= kLpSlab || top < 0 || top > kLpMaxTop) return 0;
  const size_t units = (size_t)n * lp_parts(vocab);
  return (units * top * sizeof(uint64_t) + units * 3 * sizeof(float) + 15) / 16 * 16;
}

int wfd_logprobs(const void* logits, int64_t ld, const int64_t* ids, float* out, float* entropy, float* top_val,
                 int64_t* top_id, int top, int n, int vocab, int dtype, void* workspace, size_t ws_bytes,
                 hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_logprobs";
  if (n < 0 || vocab <= 0 || ld < vocab || top < 0 || top > vocab) {
    set_error("%s: bad shape n=%d vocab=%d ld=%lld top=%d", me, n, vocab, (long long)ld, top);
    return kBadArg;
  }
  if ((dtype != kBF16 && dtype != kF32) || top > kLpMaxTop) {
    set_error("%s: unsupported dtype=%d top=%d (up to %d)", me, dtype, top, kLpMaxTop);
    return kUnsupported;
  }
  if (n == 0) return kOk;
  if (!logits || (ids == nullptr) != (out == nullptr) || (top && (!top_val || !top_id))) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  if (!out && !entropy && !top) return kOk;
  const size_t need = wfd_logprobs_workspace_bytes(n, vocab, top);
  if (need && (!workspace || ws_bytes < need || (uintptr_t)workspace % 16)) {
    set_error("%s: workspace of %zu bytes at %p, needs %zu, 16-byte aligned", me, ws_bytes, workspace, need);
    return kWorkspace;
  }
  LpArgs a{logits, ld, ids, out, entropy, top_val, top_id, nullptr, nullptr, n, vocab, top, lp_parts(vocab), lp_slab(vocab)};
  a.tops = (uint64_t*)workspace;
  a.sums = (float*)(a.tops + (size_t)n * a.parts * top);
  if (dtype == kBF16)
    launch_logprobs<bf16_t>(a, stream);
  else
    launch_logprobs<float>(a, stream);
  return launch_status(me);
}

}  // extern "C"
