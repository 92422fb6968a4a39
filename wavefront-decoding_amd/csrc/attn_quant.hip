// Wavefront decode attention over 8-bit slot caches, read in place (quant.h has
// the format; wfd_attn_decode the operation):
//   o[i,h,:] = softmax_t(q[i,h,:] . K_t * scale) V_t,   K_t = kcode_t 2^(ke_t - 127), V_t likewise.
//
// Codes are exact in bf16 and the scales are powers of two, so the products are
// those of a cache that held the values themselves: q . kcode runs on MFMA in
// q's type (the codes converted, not q), the score takes its key's scale, and
// the probability its key's V scale before it multiplies V's codes in fp32 on
// the VALU. Statistics and sums are fp32; the one rounding is the output's.
//
// Bound by HBM: (Dh + 1) bytes of K and of V per key and kv head. Work split as
// in wfd_attn_decode: a workgroup of 8 waves owns one (1024-key split, kv head,
// query row), its waves take 64-key tiles round-robin, a split's waves merge
// through LDS in fixed order and a row's splits in attn_combine_kernel, all a
// function of kv_len only, so a row's bits do not depend on the launch.
#include "attn_combine.h"
#include "quant.h"

namespace wfd {

// Codes of a 16-byte piece as MFMA operand fragments: piece p of a key holds
// its values 16 p .. 16 p + 15; step t of its steps takes kVec of them.
template <typename T, int CODE>
__device__ __forceinline__ u32x4 code_frag(const u32x4& w, int t) {
  if constexpr (sizeof(T) == 2) {
    float f[8];
    decode4<CODE>(w[2 * t], f);
    decode4<CODE>(w[2 * t + 1], f + 4);
    return Elem<bf16_t>::pack(f);
  } else {
    float f[4];
    decode4<CODE>(w[t], f);
    return Elem<float>::pack(f);
  }
}

template <typename T, int CODE, int DH, int G>
__global__ __launch_bounds__(512) void attn_q_split_kernel(
    const T* __restrict__ q, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
    const uint8_t* __restrict__ ke, const uint8_t* __restrict__ ve, const int64_t* __restrict__ row_base,
    const int32_t* __restrict__ kv_len, float* __restrict__ part_o, float* __restrict__ part_ml, T* __restrict__ out,
    int H, int Hkv, int max_splits, float scale_log2, int64_t block_rows, int vsplit) {
  constexpr int NW = 8;
  constexpr int TK = 64;
  constexpr int V = Elem<T>::kVec;
  constexpr int NJ = TK / 16;       // 16-key blocks per tile
  constexpr int LPK = DH / 16;      // 16-byte pieces (lanes) per key row
  constexpr int KPI = 64 / LPK;     // key rows per load instruction
  constexpr int NLD = TK / KPI;     // load instructions per tile and tensor
  constexpr int NP = LPK / 4;       // pieces per lane of a fragment (its lane group's)
  constexpr int STEPS = 16 / V;     // MFMA steps per piece
  constexpr int SW = 16 / LPK;      // key rows per 256 bytes of LDS
  __shared__ __align__(16) u32x4 k_lds[NW][TK * LPK];
  __shared__ float p_lds[NW][G][TK];
  __shared__ float o_lds[NW][G][DH];
  __shared__ float m_lds[NW][G];
  __shared__ float l_lds[NW][G];

  const int split = blockIdx.x;
  const int g = blockIdx.y;
  const int nz = gridDim.z / vsplit;
  const int vp = blockIdx.z / nz;
  const int i = blockIdx.z - vp * nz;
  const int DV = DH / vsplit;
  const int d0 = vp * DV;  // output columns [d0, d0 + DV) are this workgroup's
  const int len = kv_len[i];
  if (split * kAttnSplit >= len) {  // uniform
    if (split == 0)                 // no keys: a zero row
      for (int idx = threadIdx.x; idx < G * DV; idx += 64 * NW)
        Elem<T>::store(out + ((int64_t)i * H + g * G + idx / DV) * DH + d0 + idx % DV, 0.f);
    return;
  }
  const int kend = min(len, (split + 1) * kAttnSplit);
  const int ntiles = (kend - split * kAttnSplit + TK - 1) / TK;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 15;
  const int grp = lane >> 4;
  const int vg = lane / LPK;    // V row of this lane within a load
  const int dseg = lane % LPK;  // its 16 columns
  const bool vmine = dseg * 16 >= d0 && dseg * 16 < d0 + DV;
  const int64_t hb = kv_offset(row_base[i], g, Hkv, DH, block_rows);
  const int64_t rs = block_rows > 1 ? (int64_t)DH : (int64_t)Hkv * DH;  // key stride, bytes
  const int64_t es = block_rows > 1 ? 1 : Hkv;                          // exponent stride
  const uint8_t* kb = kc + hb;
  const uint8_t* vb = vc + hb;
  const uint8_t* keb = ke + hb / DH;
  const uint8_t* veb = ve + hb / DH;

  // Q as the A operand, row = query head g G + col, in the codes' k order
  u32x4 qf[NP][STEPS];
  {
    const bool real = col < G;
    const T* qp = q + ((int64_t)i * H + g * G + (real ? col : 0)) * DH + 16 * grp;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int t = 0; t < STEPS; ++t) qf[p][t] = real ? ld16(qp + 64 * p + V * t) : zero16();
  }

  float mrun[G], lrun[G], o[G][16];
#pragma unroll
  for (int m = 0; m < G; ++m) {
    mrun[m] = -INFINITY;
    lrun[m] = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[m][e] = 0.f;
  }

  for (int t = wave; t < ntiles; t += NW) {  // uniform over the wave
    const int t0 = split * kAttnSplit + t * TK;
    u32x4 kf[NLD], vf[NLD];
    uint32_t kx[NJ], vx[NJ];
#pragma unroll
    for (int s = 0; s < NLD; ++s) {  // whole key rows; the piece order keeps the fragment reads off each other's banks
      const int r = KPI * s + lane / LPK;
      const int key = min(t0 + r, kend - 1);
      kf[s] = ld16(kb + (int64_t)key * rs + ((lane % LPK) ^ ((r / SW) % LPK)) * 16);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int key = min(t0 + 16 * j + col, kend - 1);
      kx[j] = keb[key * es];
      vx[j] = veb[key * es];
    }
#pragma unroll
    for (int s = 0; s < NLD; ++s) {
      const int key = min(t0 + KPI * s + vg, kend - 1);
      vf[s] = vmine ? ld16(vb + (int64_t)key * rs + dseg * 16) : zero16();
    }
    // the LDS executes one wave's accesses in order
    asm volatile("" ::: "memory");
#pragma unroll
    for (int s = 0; s < NLD; ++s) k_lds[wave][64 * s + lane] = kf[s];
    asm volatile("" ::: "memory");
    // scores: lane (grp, col) holds S[row 4 grp + r][key 16 j + col]
    f32x4 acc[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int r = 16 * j + col;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const u32x4 w = k_lds[wave][r * LPK + ((4 * p + grp) ^ ((r / SW) % LPK))];
#pragma unroll
        for (int st = 0; st < STEPS; ++st) acc[j] = mfma_step<T>(qf[p][st], code_frag<T, CODE>(w, st), acc[j]);
      }
    }
    // rows 0 .. G - 1 sit in lane group 0: it reduces them, the others follow
    float p4[NJ][4];
    float corr[G];
#pragma unroll
    for (int m = 0; m < G; ++m) {
      float mt = -INFINITY;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const bool valid = t0 + 16 * j + col < kend;
        const float sv = valid ? acc[j][m] * (scale_log2 * code_scale(kx[j])) : -INFINITY;
        p4[j][m] = sv;
        mt = fmaxf(mt, sv);
      }
#pragma unroll
      for (int sh = 8; sh >= 1; sh >>= 1) mt = fmaxf(mt, __shfl_xor(mt, sh, 64));
      mt = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(mt)));
      const float mnew = fmaxf(mrun[m], mt);
      corr[m] = (mrun[m] == -INFINITY) ? 0.f : exp2f(mrun[m] - mnew);
      mrun[m] = mnew;
      float lt = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float p = (p4[j][m] == -INFINITY) ? 0.f : exp2f(p4[j][m] - mnew);
        lt += p;
        // a key past the end contributes nothing whatever scale it was clamped to
        p4[j][m] = t0 + 16 * j + col < kend ? p * code_scale(vx[j]) : 0.f;
      }
#pragma unroll
      for (int sh = 8; sh >= 1; sh >>= 1) lt += __shfl_xor(lt, sh, 64);
      lt = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(lt)));
      lrun[m] = fmaf(lrun[m], corr[m], lt);
    }
    if (grp == 0) {
#pragma unroll
      for (int m = 0; m < G; ++m)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int kt = 16 * j + col;
          p_lds[wave][m][(kt % KPI) * NLD + kt / KPI] = p4[j][m];  // in the V lanes' key order
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int m = 0; m < G; ++m)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[m][e] *= corr[m];
#pragma unroll
    for (int s = 0; s < NLD; ++s) {
      float v[16];
#pragma unroll
      for (int w = 0; w < 4; ++w) decode4<CODE>(vf[s][w], v + 4 * w);
#pragma unroll
      for (int m = 0; m < G; ++m) {
        const float p = p_lds[wave][m][vg * NLD + s];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[m][e] = fmaf(p, v[e], o[m][e]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // the next tile rewrites P and K
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
#pragma unroll
  for (int m = 0; m < G; ++m) {
#pragma unroll
    for (int sh = LPK; sh < 64; sh <<= 1)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[m][e] += __shfl_xor(o[m][e], sh, 64);
    if (vg == 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o_lds[wave][m][dseg * 16 + e] = o[m][e];
    }
    if (lane == 0) {
      m_lds[wave][m] = mrun[m];
      l_lds[wave][m] = lrun[m];
    }
  }
  __syncthreads();

  // merge the waves in fixed order: the row itself if its keys fit one split,
  // this split's unnormalised partial otherwise
  const int ns = min((len + kAttnSplit - 1) / kAttnSplit, max_splits);
  for (int idx = threadIdx.x; idx < G * DV; idx += 64 * NW) {
    const int m = idx / DV;
    const int d = d0 + (idx - m * DV);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, m_lds[w][m]);
    float O = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = m_lds[w][m];
      const float f = (mw == -INFINITY) ? 0.f : exp2f(mw - M);
      O = fmaf(o_lds[w][m][d], f, O);
      L = fmaf(l_lds[w][m], f, L);
    }
    const int64_t row = (int64_t)i * H + g * G + m;
    if (ns == 1) {
      Elem<T>::store(out + row * DH + d, attn_finish_nan(O, L));
    } else {
      const int64_t pidx = row * max_splits + split;
      part_o[pidx * DH + d] = O;
      if (d == 0) {
        part_ml[pidx * 2] = M;
        part_ml[pidx * 2 + 1] = L;
      }
    }
  }
}

struct AttnQArgs {
  const void* q;
  const uint8_t *kc, *vc, *ke, *ve;
  const int64_t* rb;
  const int32_t* kl;
  void* out;
  float *po, *pml;
  int n, H, Hkv, ms;
  float scale_log2;
  int64_t br;
};

template <typename T, int CODE, int DH, int G>
static void launch_attn_q(const AttnQArgs& a, hipStream_t st) {
  const int vs = 1;
  hipLaunchKernelGGL((attn_q_split_kernel<T, CODE, DH, G>), dim3(a.ms, a.Hkv, a.n * vs), dim3(512), 0, st,
                     (const T*)a.q, a.kc, a.vc, a.ke, a.ve, a.rb, a.kl, a.po, a.pml, (T*)a.out, a.H, a.Hkv, a.ms,
                     a.scale_log2, a.br, vs);
  if (a.ms > 1)  // some query may span several splits
    hipLaunchKernelGGL((attn_combine_kernel<T, DH, true>), dim3(a.H, a.n), dim3(DH), 0, st, a.po, a.pml, a.kl, (T*)a.out,
                       a.H, a.ms);
}

template <typename T, int CODE>
static bool dispatch_attn_q(int Dh, int G, const AttnQArgs& a, hipStream_t st) {
#define WFD_ATTNQ_CASE(DHV, GV)             \
  if (Dh == DHV && G == GV) {               \
    launch_attn_q<T, CODE, DHV, GV>(a, st); \
    return true;                            \
  }
  WFD_ATTNQ_CASE(64, 1)
  WFD_ATTNQ_CASE(64, 2)
  WFD_ATTNQ_CASE(64, 4)
  WFD_ATTNQ_CASE(128, 1)
  WFD_ATTNQ_CASE(128, 2)
  WFD_ATTNQ_CASE(128, 4)
#undef WFD_ATTNQ_CASE
  return false;
}

}  // namespace wfd

extern "C" {

int wfd_attn_decode_q(const void* q, const void* k_codes, const void* v_codes, const uint8_t* k_exp,
                      const uint8_t* v_exp, int code, int64_t kv_block_rows, const int64_t* kv_row_base,
                      const int32_t* kv_len, void* out, int n, int H, int Hkv, int Dh, int dtype, float scale,
                      int kv_len_max, void* workspace, size_t ws_bytes, hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_attn_decode_q";
  if (int rc = check_qcache(me, n, Hkv, Dh, code, kv_block_rows)) return rc;
  if (H <= 0 || H > kMaxHeads || H % Hkv != 0 || kv_len_max < 1 ||
      (kv_block_rows > 1 && kv_len_max > kv_block_rows)) {
    set_error("%s: bad shape H=%d Hkv=%d kv_len_max=%d kv_block_rows=%lld", me, H, Hkv, kv_len_max,
              (long long)kv_block_rows);
    return kBadArg;
  }
  const int G = H / Hkv;
  if ((dtype != kBF16 && dtype != kF32) || (G != 1 && G != 2 && G != 4)) {
    set_error("%s: unsupported dtype=%d G=%d (G = H / Hkv 1/2/4)", me, dtype, G);
    return kUnsupported;
  }
  if (n > 32767) {
    set_error("%s: n=%d beyond the grid (32767 rows)", me, n);
    return kUnsupported;
  }
  if (n == 0) return kOk;
  if (!q || !k_codes || !v_codes || !k_exp || !v_exp || !kv_row_base || !kv_len || !out || !workspace) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  if (((uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)out | (uintptr_t)workspace) & 15) {
    set_error("%s: q, the codes, out and workspace must be 16-byte aligned", me);
    return kBadArg;
  }
  const size_t need = attn_ws_bytes(n, H, Dh, kv_len_max);
  if (ws_bytes < need) {
    set_error("%s: workspace %zu bytes < required %zu", me, ws_bytes, need);
    return kWorkspace;
  }
  AttnQArgs a;
  a.q = q;
  a.kc = (const uint8_t*)k_codes;
  a.vc = (const uint8_t*)v_codes;
  a.ke = k_exp;
  a.ve = v_exp;
  a.rb = kv_row_base;
  a.kl = kv_len;
  a.out = out;
  a.n = n;
  a.H = H;
  a.Hkv = Hkv;
  a.ms = max_splits_for(kv_len_max);
  a.po = (float*)workspace;
  a.pml = (float*)((char*)workspace + align256((size_t)n * H * a.ms * Dh * sizeof(float)));
  a.scale_log2 = scale * 1.4426950408889634f;
  a.br = kv_block_rows;
  if (dtype == kBF16)
    code == WFD_E4M3 ? dispatch_attn_q<bf16_t, WFD_E4M3>(Dh, G, a, stream)
                     : dispatch_attn_q<bf16_t, WFD_INT8>(Dh, G, a, stream);
  else
    code == WFD_E4M3 ? dispatch_attn_q<float, WFD_E4M3>(Dh, G, a, stream)
                     : dispatch_attn_q<float, WFD_INT8>(Dh, G, a, stream);
  return launch_status(me);
}

}  // extern "C"
