// Decode attention of rows that share a prefix: the rows of a group attend the
// group's prefix, computed for all of them together, and then keys of their own.
//
//   o_i = softmax over [prefix of i's group | i's own keys] of (q_i . k * scale), times V
//
// Softmax over a union is a merge of softmaxes over its parts: a part leaves its
// maximum m, sum l and unnormalised output o, and the row is sum o 2^(m - M) /
// sum l 2^(m - M) over its parts. The prefix is cut into chunks of keys, a
// workgroup computes one chunk for up to kShRows (query row, query head) pairs of
// a group and one kv head -- each key is read once for all of them -- and a row's
// own keys are cut likewise, for that row alone; attn_shared_combine merges a
// row's parts in the order of its keys.
//
// The chunks follow from the lengths and Hkv alone, and a row's arithmetic within
// a chunk from the chunk, so a row's bits do not depend on its group's other
// rows, on the launch, or on where the row sits.
#include "attn_combine.h"

namespace wfd {

constexpr int kShRows = 16;      // (query row, head) pairs per workgroup
constexpr int kShWaves = 4;      // key streams per workgroup
constexpr int kShMinChunk = 128;
constexpr int kShMaxChunk = 1024;
constexpr int kShOwnChunk = 512;
constexpr int kShTarget = 256;   // chunks x kv heads aimed at
constexpr int kShMaxG = 16;

// Keys per chunk of a prefix of P keys: enough chunks for a workgroup per CU over
// the kv heads while they are at least 128 keys; long prefixes take 1024, where
// the parts' traffic is small against the keys'.
__host__ __device__ inline int prefix_chunk(int P, int Hkv) {
  const int64_t c = ((int64_t)P * Hkv + kShTarget - 1) / kShTarget;
  const int64_t r = (c + kShMinChunk - 1) / kShMinChunk * kShMinChunk;
  return (int)(r < kShMinChunk ? kShMinChunk : (r > kShMaxChunk ? kShMaxChunk : r));
}

__host__ __device__ inline int div_up(int a, int b) { return a <= 0 ? 0 : (a + b - 1) / b; }

// The most chunks any prefix of up to P keys makes (a chunk has at least
// P Hkv / 256 keys unless it has 1024).
inline int max_prefix_chunks(int P, int Hkv) {
  const int few = div_up(P, kShMinChunk), target = div_up(kShTarget, Hkv), many = div_up(P, kShMaxChunk);
  const int b = few < target ? few : target;
  return b > many ? b : many;
}

struct ShArgs {
  const void *q, *kc, *vc;
  int64_t br;
  const int64_t* pbase;
  const int32_t *plen, *gfirst;
  const int64_t* rbase;
  const int32_t* rlen;
  void* out;
  float *po, *pml;
  int n, H, Hkv, ng, tiles, pchunks, ochunks, pmax, omax;
  float scale_log2;
};

template <typename T, int DH>
__global__ __launch_bounds__(64 * kShWaves) void attn_shared_kernel(ShArgs a) {
  constexpr int V = Elem<T>::kVec;
  constexpr int KSTEP = 4 * V;
  constexpr int NDS = DH / KSTEP;
  constexpr int NC = DH / 16;
  __shared__ float p_lds[kShWaves][16][17];
  __shared__ float o_lds[kShWaves][16][DH];
  __shared__ float m_lds[kShWaves][16];
  __shared__ float l_lds[kShWaves][16];
  const int G = a.H / a.Hkv;
  const int g = blockIdx.x % a.Hkv;
  int64_t item = blockIdx.x / a.Hkv;
  const int64_t nprefix = (int64_t)a.ng * a.pchunks * a.tiles;
  int row0, nr, k0, k1, part;  // first query row, pairs, keys, the part's place
  int64_t base;
  if (item < nprefix) {
    const int tile = (int)(item % a.tiles);
    item /= a.tiles;
    const int c = (int)(item % a.pchunks), j = (int)(item / a.pchunks);
    const int P = min(a.plen[j], a.pmax);
    const int first = a.gfirst[j];
    const int pairs = (min(a.gfirst[j + 1], a.n) - first) * G;
    const int ck = prefix_chunk(P, a.Hkv);
    k0 = c * ck;
    k1 = min(k0 + ck, P);
    if (k0 >= k1 || tile * kShRows >= pairs) return;  // uniform
    row0 = first;
    nr = pairs;
    part = c;
    base = a.pbase[j];
    // pairs tile * kShRows .. of the group
    item = tile * kShRows;
  } else {
    item -= nprefix;
    const int c = (int)(item % a.ochunks), i = (int)(item / a.ochunks);
    const int L = min(a.rlen[i], a.omax);
    k0 = c * kShOwnChunk;
    k1 = min(k0 + kShOwnChunk, L);
    if (k0 >= k1) return;
    row0 = i;
    nr = G;
    part = a.pchunks + c;
    base = a.rbase[i];
    item = 0;
  }
  const int p0 = (int)item;
  nr = min(nr - p0, kShRows);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int64_t hb = kv_offset(base, g, a.Hkv, DH, a.br);
  const int64_t rs = a.br > 1 ? (int64_t)DH : (int64_t)a.Hkv * DH;
  const T* kb = (const T*)a.kc + hb;
  const T* vb = (const T*)a.vc + hb;
  auto pair_row = [&](int r) { return (int64_t)(row0 + (p0 + r) / G) * a.H + g * G + (p0 + r) % G; };

  u32x4 qf[NDS];
#pragma unroll
  for (int s = 0; s < NDS; ++s)
    qf[s] = col < nr ? ld16((const T*)a.q + pair_row(col) * DH + grp * V + s * KSTEP) : zero16();

  float mrun[4], lrun[4];
  f32x4 o[NC];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    mrun[r] = -INFINITY;
    lrun[r] = 0.f;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int t0 = k0 + 16 * wave; t0 < k1; t0 += 16 * kShWaves) {
    const T* kp = kb + (int64_t)min(t0 + col, k1 - 1) * rs + grp * V;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NDS; ++s) acc = mfma_step<T>(qf[s], ld16(kp + s * KSTEP), acc);
    float corr[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float sv = t0 + col < k1 ? acc[r] * a.scale_log2 : -INFINITY;
      float mt = sv;
#pragma unroll
      for (int sh = 8; sh >= 1; sh >>= 1) mt = fmaxf(mt, __shfl_xor(mt, sh, 64));
      const float mnew = fmaxf(mrun[r], mt);
      corr[r] = mrun[r] == -INFINITY ? 0.f : exp2f(mrun[r] - mnew);
      mrun[r] = mnew;
      const float p = sv == -INFINITY ? 0.f : exp2f(sv - mnew);
      float lt = p;
#pragma unroll
      for (int sh = 8; sh >= 1; sh >>= 1) lt += __shfl_xor(lt, sh, 64);
      lrun[r] = fmaf(lrun[r], corr[r], lt);
      p_lds[wave][4 * grp + r][col] = p;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[c][r] *= corr[r];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const float p = p_lds[wave][col][4 * s + grp];
      const int key = t0 + 4 * s + grp;
      const T* vp = vb + (int64_t)min(key, k1 - 1) * rs + col;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float v = key < k1 ? Elem<T>::load(vp + 16 * c) : 0.f;
        o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(p, v, o[c], 0, 0, 0);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int c = 0; c < NC; ++c) o_lds[wave][4 * grp + r][16 * c + col] = o[c][r];
    if (col == 0) {
      m_lds[wave][4 * grp + r] = mrun[r];
      l_lds[wave][4 * grp + r] = lrun[r];
    }
  }
  __syncthreads();
  const int ms = a.pchunks + a.ochunks;
  for (int idx = threadIdx.x; idx < nr * DH; idx += 64 * kShWaves) {
    const int r = idx / DH, d = idx - r * DH;
    float M = -INFINITY, O = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) M = fmaxf(M, m_lds[w][r]);
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) {
      const float f = m_lds[w][r] == -INFINITY ? 0.f : exp2f(m_lds[w][r] - M);
      O = fmaf(o_lds[w][r][d], f, O);
      L = fmaf(l_lds[w][r], f, L);
    }
    const int64_t at = pair_row(r) * ms + part;
    a.po[at * DH + d] = O;
    if (d == 0) {
      a.pml[2 * at] = M;
      a.pml[2 * at + 1] = L;
    }
  }
}

// Group of row i (the last one that starts at or before it and ends after it), or -1.
__device__ __forceinline__ int row_group(const int32_t* __restrict__ gfirst, int ng, int i) {
  if (ng == 0 || i < gfirst[0] || i >= gfirst[ng]) return -1;
  int lo = 0, hi = ng;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (gfirst[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// One row's parts, prefix chunks then its own, merged in that order.
template <typename T, int DH>
__global__ __launch_bounds__(DH) void attn_shared_combine(ShArgs a) {
  constexpr int B = kCombineBatch;
  const int h = blockIdx.x, i = blockIdx.y, d = threadIdx.x;
  const int j = row_group(a.gfirst, a.ng, i);
  const int P = j < 0 ? 0 : min(a.plen[j], a.pmax);
  const int np = P > 0 ? div_up(P, prefix_chunk(P, a.Hkv)) : 0;
  const int ns = np + div_up(min(a.rlen[i], a.omax), kShOwnChunk);
  const int64_t base = ((int64_t)i * a.H + h) * (a.pchunks + a.ochunks);
  auto at = [&](int s) { return base + (s < np ? s : a.pchunks + s - np); };
  float M = -INFINITY;
  for (int s0 = 0; s0 < ns; s0 += B) {
    float mv[B];
#pragma unroll
    for (int b = 0; b < B; ++b) mv[b] = s0 + b < ns ? a.pml[2 * at(s0 + b)] : -INFINITY;
#pragma unroll
    for (int b = 0; b < B; ++b) M = fmaxf(M, mv[b]);
  }
  float O = 0.f, L = 0.f;
  for (int s0 = 0; s0 < ns; s0 += B) {
    float mv[B], lv[B], ov[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const bool ok = s0 + b < ns;
      const int64_t p = ok ? at(s0 + b) : base;
      mv[b] = ok ? a.pml[2 * p] : -INFINITY;
      lv[b] = ok ? a.pml[2 * p + 1] : 0.f;
      ov[b] = ok ? a.po[p * DH + d] : 0.f;
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (s0 + b < ns) {
        const float f = mv[b] == -INFINITY ? 0.f : exp2f(mv[b] - M);
        L = fmaf(lv[b], f, L);
        O = fmaf(ov[b], f, O);
      }
    }
  }
  Elem<T>::store((T*)a.out + ((int64_t)i * a.H + h) * DH + d, attn_finish_nan(O, L));
}

template <typename T, int DH>
static void launch_shared(const ShArgs& a, hipStream_t st) {
  const int64_t items = (int64_t)a.ng * a.pchunks * a.tiles + (int64_t)a.n * a.ochunks;
  if (items)
    hipLaunchKernelGGL((attn_shared_kernel<T, DH>), dim3((unsigned)(items * a.Hkv)), dim3(64 * kShWaves), 0, st, a);
  hipLaunchKernelGGL((attn_shared_combine<T, DH>), dim3(a.H, a.n), dim3(DH), 0, st, a);
}

}  // namespace wfd

extern "C" {

size_t wfd_attn_shared_workspace_bytes(int n, int H, int Hkv, int Dh, int prefix_len_max, int kv_len_max) {
  using namespace wfd;
  if (n <= 0 || H <= 0 || Hkv <= 0 || Dh <= 0 || prefix_len_max < 0 || kv_len_max < 0) return 0;
  const size_t parts = (size_t)n * H * (max_prefix_chunks(prefix_len_max, Hkv) + div_up(kv_len_max, kShOwnChunk));
  return align256(parts * Dh * sizeof(float)) + align256(parts * 2 * sizeof(float));
}

int wfd_attn_shared(const void* q, const void* k_cache, const void* v_cache, int64_t kv_block_rows,
                    const int64_t* prefix_row_base, const int32_t* prefix_len, const int32_t* group_first, int ngroups,
                    int group_max, const int64_t* kv_row_base, const int32_t* kv_len, void* out, int n, int H,
                    int Hkv, int Dh, int dtype, float scale, int prefix_len_max, int kv_len_max, void* workspace,
                    size_t ws_bytes, hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_attn_shared";
  if (n < 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || H > 65535 || ngroups < 0 || group_max < 0 || kv_block_rows < 0 ||
      prefix_len_max < 0 || kv_len_max < 0) {
    set_error("%s: bad shape n=%d H=%d Hkv=%d ngroups=%d group_max=%d prefix_len_max=%d kv_len_max=%d", me, n, H, Hkv,
              ngroups, group_max, prefix_len_max, kv_len_max);
    return kBadArg;
  }
  if (kv_block_rows > 1 && (prefix_len_max > kv_block_rows || kv_len_max > kv_block_rows)) {
    set_error("%s: prefix_len_max=%d kv_len_max=%d exceed a block, kv_block_rows=%lld", me, prefix_len_max, kv_len_max,
              (long long)kv_block_rows);
    return kBadArg;
  }
  const int G = H / Hkv;
  if ((dtype != kBF16 && dtype != kF32) || (Dh != 64 && Dh != 128) || G > kShMaxG) {
    set_error("%s: unsupported dtype=%d Dh=%d G=%d (Dh 64/128, H / Hkv up to %d)", me, dtype, Dh, G, kShMaxG);
    return kUnsupported;
  }
  if (n == 0) return kOk;
  if (!q || !k_cache || !v_cache || !kv_row_base || !kv_len || !out || !workspace ||
      (ngroups && (!prefix_row_base || !prefix_len || !group_first))) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) & 15) {
    set_error("%s: q, the caches, out and workspace must be 16-byte aligned", me);
    return kBadArg;
  }
  const size_t need = wfd_attn_shared_workspace_bytes(n, H, Hkv, Dh, prefix_len_max, kv_len_max);
  if (ws_bytes < need) {
    set_error("%s: workspace %zu bytes < required %zu", me, ws_bytes, need);
    return kWorkspace;
  }
  ShArgs a;
  a.q = q;
  a.kc = k_cache;
  a.vc = v_cache;
  a.br = kv_block_rows;
  a.pbase = prefix_row_base;
  a.plen = prefix_len;
  a.gfirst = group_first;
  a.rbase = kv_row_base;
  a.rlen = kv_len;
  a.out = out;
  a.n = n;
  a.H = H;
  a.Hkv = Hkv;
  a.ng = ngroups;
  const int64_t pairs = (int64_t)(group_max < n ? group_max : n) * G;
  const int64_t tiles = (pairs + kShRows - 1) / kShRows;
  a.pchunks = max_prefix_chunks(prefix_len_max, Hkv);
  a.ochunks = div_up(kv_len_max, kShOwnChunk);
  a.pmax = prefix_len_max;
  a.omax = kv_len_max;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.po = (float*)workspace;
  a.pml = (float*)((char*)workspace + align256((size_t)n * H * (a.pchunks + a.ochunks) * Dh * sizeof(float)));
  // in double: the product of four counts may pass 64 bits
  const double wgs = ((double)ngroups * a.pchunks * (double)tiles + (double)n * a.ochunks) * Hkv;
  if (wgs > 2147483647.0 || n > 65535) {
    set_error("%s: n=%d ngroups=%d group_max=%d prefix_len_max=%d kv_len_max=%d beyond the grid", me, n, ngroups,
              group_max, prefix_len_max, kv_len_max);
    return kUnsupported;
  }
  a.tiles = (int)tiles;
  if (a.pchunks == 0 || tiles == 0) a.ng = 0;
  if (dtype == kBF16)
    Dh == 64 ? launch_shared<bf16_t, 64>(a, stream) : launch_shared<bf16_t, 128>(a, stream);
  else
    Dh == 64 ? launch_shared<float, 64>(a, stream) : launch_shared<float, 128>(a, stream);
  return launch_status(me);
}

}  // extern "C"
