// Wavefront decode attention over 8-bit slot caches, read in place (quant.h has
// the format; wfd_attn_decode the operation):
//   o[i,h,:] = softmax_t(q[i,h,:] . K_t * scale) V_t,   K_t = kcode_t 2^(ke_t - 127), V_t likewise.
//
// Codes are exact in bf16 and the scales are powers of two, so the products are
// those of a cache that held the values themselves: a score takes its key's
// scale after q . kcode, a probability its key's V scale before it meets V's
// codes. Both products run on the 16x16x32 bf16 MFMA, S^T = K Q^T and O^T = V^T
// P^T, the query heads of the kv head as the 16 columns. fp32 queries are split
// into three bf16 terms, which hold all their bits; probabilities into two (a
// half step of 2^-16 of each) or, for fp32, three. Statistics and sums are fp32.
// A third term for bf16 outputs too moves their distance from the exact ones in the
// seventh digit (0.00166 of the norm, their own rounding): 64 rows x 32.7k keys 393 ->
// 424 us, 8 rows 10.5 -> 11.2.
//
// Bound by HBM: (Dh + 1) bytes of K and of V per key and kv head. P.V on the
// VALU, as in wfd_attn_decode, took 1600 vector instructions per 64 keys of four
// heads and held 64 rows over 32k keys at 3.3 TB/s; a tile here takes a fifth. 64
// rows x 4 kv heads x 32.7k e4m3 keys: 375-400 us, 5.4-5.7 TB/s (reads alone, so above
// the 4.9 of a copy); 112 rows x 16 heads x 128-1200 int8 keys 78-82 us, 3.8-4.0 TB/s
// (short rows' first loads and merges); 8 rows of 512-778 keys 10.4 us, one tile after
// another in 128 workgroups.
// Work split as there: a workgroup of 8 waves owns one (1024-key split, kv head,
// query row), its waves take 32-key tiles round-robin, each through LDS of its
// own a tile ahead; the waves merge through LDS in fixed order and a row's splits
// in attn_q_combine, all a function of kv_len only, so a row's bits do not
// depend on the launch.
#include "attn_combine.h"
#include "quant.h"

namespace wfd {

struct AttnQArgs {
  const void* q;
  const uint8_t *kc, *vc, *ke, *ve;
  const int64_t* rb;
  const int32_t* kl;
  void* out;
  float *po, *pml;
  int n, H, Hkv, ms, spw;
  float scale_log2;
  int64_t br;
};

constexpr int kAqWaves = 8;
constexpr int kAqMaxG = 16;        // columns of the MFMA
constexpr int kAqMaxHeads = 4096;  // a split's keys stay within 32-bit offsets of its first

// Eight codes (two dwords) as a bf16 operand fragment, exact.
template <int CODE>
__device__ __forceinline__ u32x4 code_frag(uint32_t w0, uint32_t w1) {
  if constexpr (CODE == WFD_E4M3) {
    // two codes an instruction; taken as the dword it is
    auto pair = [](uint32_t w, bool hi) {
      return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    };
    return u32x4{pair(w0, false), pair(w0, true), pair(w1, false), pair(w1, true)};
  } else {
    float f[8];
    decode4<CODE>(w0, f);
    decode4<CODE>(w1, f + 4);
    return Elem<bf16_t>::pack(f);
  }
}

// The next bf16 term of eight values: x's rounding, which x then loses.
__device__ __forceinline__ u32x4 take_term(float (&x)[8], bool last) {
  const u32x4 w = Elem<bf16_t>::pack(x);
  if (!last) {
    float r[8];
    Elem<bf16_t>::unpack(w, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] -= r[e];
  }
  return w;
}

template <typename T, int CODE, int DH>
__global__ __launch_bounds__(64 * kAqWaves) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 ? 4 : 2))) void
attn_q_split_kernel(AttnQArgs a) {
  constexpr int NW = kAqWaves;
  constexpr int TK = 32;
  constexpr int QT = sizeof(T) == 2 ? 1 : 3;  // bf16 terms of a query
  constexpr int PT = sizeof(T) == 2 ? 2 : 3;  // and of a probability
  constexpr int LPK = DH / 16;   // 16-byte pieces (lanes) per row of codes
  constexpr int RPI = 64 / LPK;  // rows per load instruction
  constexpr int NLD = TK / RPI;
  constexpr int NP = LPK / 4;    // pieces per lane of a K fragment, two MFMA steps each
  constexpr int NDB = DH / 16;
  constexpr int RP = DH + 16;    // LDS row pitch: 16 rows start on 16 different 16-byte bank groups
  constexpr int OP = DH + 4;
  constexpr int kTile = TK * RP;
  constexpr size_t kStage = (size_t)NW * 2 * kTile, kMerge = sizeof(float) * NW * kAqMaxG * OP;
  __shared__ __align__(16) uint8_t lds[kStage > kMerge ? kStage : kMerge];
  __shared__ __align__(16) float s_lds[NW][2 * TK];  // a tile's K and V scales
  __shared__ __align__(16) u32x4 q_lds[QT == 1 ? NP : 1][2][64];
  __shared__ float m_lds[NW][kAqMaxG];
  __shared__ float l_lds[NW][kAqMaxG];

  const int split0 = blockIdx.x * a.spw, g = blockIdx.y, i = blockIdx.z;
  const int G = a.H / a.Hkv;
  const int64_t row0 = (int64_t)i * a.H + g * G;
  const int len = min(a.kl[i], a.ms * kAttnSplit);
  if (split0 * kAttnSplit >= len) {  // uniform
    if (split0 == 0)                 // no keys: zero rows
      for (int idx = threadIdx.x; idx < G * DH; idx += 64 * NW) Elem<T>::store((T*)a.out + row0 * DH + idx, 0.f);
    return;
  }
  // keys from split0's first, nk of them: the workgroup's splits, nsp of them
  const int nk = min(len - split0 * kAttnSplit, a.spw * kAttnSplit);
  const int nsp = (nk + kAttnSplit - 1) / kAttnSplit;
  const int ns = (len + kAttnSplit - 1) / kAttnSplit;  // the row's
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  uint8_t* k_lds = lds + wave * 2 * kTile;
  uint8_t* v_lds = k_lds + kTile;

  // codes of this head from the first split's first key; the resources end with the
  // last one, so that later rows read as zeros
  const uint32_t rs = a.br > 1 ? DH : a.Hkv * DH;  // key stride, bytes
  const int64_t at = kv_offset(a.rb[i], g, a.Hkv, DH, a.br) + (int64_t)split0 * kAttnSplit * rs;
  const uint32_t span = (uint32_t)(nk - 1) * rs + DH;
  auto rsrc = [&](const uint8_t* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p + at), (short)0, span, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t kr = rsrc(a.kc), vr = rsrc(a.vc);
  const uint8_t* eb = (lane < TK ? a.ke : a.ve) + at / DH;  // lane: the K (V) scale of key lane % 32
  const uint32_t es = rs / DH;
  const int lr = lane / LPK, lp = lane % LPK;  // row within a load, piece
  uint32_t off[NLD];
#pragma unroll
  for (int s = 0; s < NLD; ++s) off[s] = (uint32_t)(TK * wave + RPI * s + lr) * rs + (uint32_t)lp * 16u;
  u32x4 kreg[NLD], vreg[NLD];
  uint32_t ereg;
  int t0 = TK * wave;
  auto fetch = [&](int t) {  // this wave's next tile
#pragma unroll
    for (int s = 0; s < NLD; ++s) {
      kreg[s] = buf_ld16(kr, off[s]);
      vreg[s] = buf_ld16(vr, off[s]);
      off[s] += (uint32_t)(TK * NW) * rs;
    }
    ereg = eb[(uint64_t)min(t + (lane % TK), nk - 1) * es];
  };
  fetch(t0);

  // Q as the B operand, column = query head, in the codes' k order: three terms in
  // registers, or bf16 in LDS, whose registers would cost a wave per SIMD. Columns
  // past the last head repeat it; nothing of theirs is kept.
  const T* qp = (const T*)a.q + (row0 + min(col, G - 1)) * DH + 16 * grp;
  u32x4 qf[QT][NP][2];
  if constexpr (QT == 1) {
    if (wave < NP)
#pragma unroll
      for (int st = 0; st < 2; ++st) q_lds[wave][st][lane] = ld16(qp + 64 * wave + 8 * st);
    __syncthreads();
  } else {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        float x[8], lo[4], hi[4];
        Elem<float>::unpack(ld16(qp + 64 * p + 8 * st), lo);
        Elem<float>::unpack(ld16(qp + 64 * p + 8 * st + 4), hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = lo[e];
          x[4 + e] = hi[e];
        }
#pragma unroll
        for (int c = 0; c < QT; ++c) qf[c][p][st] = take_term(x, c == QT - 1);
      }
  }
  // V^T fragment of 16 dims: the transposing read gives lane i of a 16-lane group byte
  // i % 8 of what lanes i / 8 + 2 e address, e < 8. Lane j addresses half j % 2 of the
  // piece in row key(j / 2), key(e) = 16 (e / 4) + 4 grp + e % 4: the keys whose scores the
  // group's lanes hold, in their order.
  const int vkey = 16 * (col >> 3) + 4 * grp + ((col >> 1) & 3);
  const uint32_t v_at = (uint32_t)(vkey * RP + 8 * (col & 1));
  auto vt_frag = [&](int db) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    typedef const __attribute__((address_space(3))) void* lds_ptr;
    const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (lds_i32x2*)(lds_ptr)(v_lds + v_at + 16 * db));
    return code_frag<CODE>((uint32_t)w[0], (uint32_t)w[1]);
  };

  // lane (grp, col): of query head col, the keys 16 j + 4 grp + r of a tile and the dims
  // 16 db + 4 grp + r of the output; lrun its share of the sum. mref is the head's
  // maximum when a tile last exceeded it by more than 2^8 (see attn_shared.hip).
  float* o_lds = reinterpret_cast<float*>(lds);
  for (int sp = 0; sp < nsp; ++sp) {  // uniform over the workgroup
  const int t_end = min((sp + 1) * kAttnSplit, nk);
  float mref = -INFINITY, lrun = 0.f;
  f32x4 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (; t0 < t_end; t0 += TK * NW) {  // uniform over the wave
#pragma unroll
    for (int s = 0; s < NLD; ++s) {
      *reinterpret_cast<u32x4*>(k_lds + (RPI * s + lr) * RP + 16 * lp) = kreg[s];
      *reinterpret_cast<u32x4*>(v_lds + (RPI * s + lr) * RP + 16 * lp) = vreg[s];
    }
    // a key past the end weighs nothing, whatever its clamped scale says
    const float sc = code_scale(ereg);
    s_lds[wave][lane] = lane < TK ? sc * a.scale_log2 : (t0 + (lane % TK) < nk ? sc : 0.f);
    fetch(t0 + TK * NW);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x4 acc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int r = 16 * j + col;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const u32x4 w =
            *reinterpret_cast<const u32x4*>(k_lds + r * RP + (4 * p + grp) * 16);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const u32x4 kf = code_frag<CODE>(w[2 * st], w[2 * st + 1]);
#pragma unroll
          for (int c = QT - 1; c >= 0; --c)
            acc[j] = mfma_step<bf16_t>(kf, QT == 1 ? q_lds[p][st][lane] : qf[c][p][st], acc[j]);
        }
      }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4 ks = *reinterpret_cast<const f32x4*>(&s_lds[wave][16 * j + 4 * grp]);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[j][r] *= ks[r];
    }
    if (t0 + TK > nk) {  // the last tile (uniform)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + 16 * j + 4 * grp + r >= nk) acc[j][r] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) mt = fmaxf(mt, acc[j][r]);
    if (__builtin_amdgcn_ballot_w64(mt > mref + 8.f)) {
      mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
      const float mnew = mt > mref + 8.f ? mt : mref;
      const float corr = mref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref - mnew);
      mref = mnew;
      lrun *= corr;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[db][r] *= corr;
    }
    const float ref = mref == -INFINITY ? 0.f : mref;
    float pv[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4 vs = *reinterpret_cast<const f32x4*>(&s_lds[wave][TK + 16 * j + 4 * grp]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f(acc[j][r] - ref);
        lrun += p;
        pv[4 * j + r] = p * vs[r];
      }
    }
    u32x4 pb[PT];
#pragma unroll
    for (int c = 0; c < PT; ++c) pb[c] = take_term(pv, c == PT - 1);
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const u32x4 vf = vt_frag(db);
#pragma unroll
      for (int c = PT - 1; c >= 0; --c) o[db] = mfma_step<bf16_t>(vf, pb[c], o[db]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // the next tile overwrites this one
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  lrun += __shfl_xor(lrun, 16, 64);
  lrun += __shfl_xor(lrun, 32, 64);

  __syncthreads();  // every wave's tiles are done: the merge takes their LDS
  if (col < G) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      *reinterpret_cast<f32x4*>(o_lds + (wave * kAqMaxG + col) * OP + 16 * db + 4 * grp) = o[db];
    if (grp == 0) {
      m_lds[wave][col] = mref;
      l_lds[wave][col] = lrun;
    }
  }
  __syncthreads();
  // merge the waves in fixed order: the row itself if its keys fit one split,
  // this split's unnormalised partial otherwise
  for (int idx = threadIdx.x; idx < G * (DH / 4); idx += 64 * NW) {
    const int m = idx / (DH / 4), d = 4 * (idx % (DH / 4));
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, m_lds[w][m]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = m_lds[w][m];
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
      const f32x4 ow = *reinterpret_cast<const f32x4*>(o_lds + (w * kAqMaxG + m) * OP + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(ow[e], f, O[e]);
      L = fmaf(l_lds[w][m], f, L);
    }
    if (ns == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) Elem<T>::store((T*)a.out + (row0 + m) * DH + d + e, attn_finish_nan(O[e], L));
    } else {
      const int64_t pidx = (row0 + m) * a.ms + split0 + sp;
      *reinterpret_cast<f32x4*>(a.po + pidx * DH + d) = O;
      if (d == 0) {
        a.pml[pidx * 2] = M;
        a.pml[pidx * 2 + 1] = L;
      }
    }
  }
  __syncthreads();  // the next split's tiles take the LDS; this one's partial is written
  }
  if (ns == 1 || nsp < ns) return;
  // a row whose splits were all this workgroup's: attn_merge_parts' sums, on
  // partials that this workgroup wrote
  for (int idx = threadIdx.x; idx < G * (DH / 4); idx += 64 * NW) {
    const int m = idx / (DH / 4), d = 4 * (idx % (DH / 4));
    const int64_t base = (row0 + m) * a.ms;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int sp = 0; sp < ns; ++sp) M = fmaxf(M, a.pml[(base + sp) * 2]);
    for (int sp = 0; sp < ns; ++sp) {
      const float mv = a.pml[(base + sp) * 2];
      const float f = mv == -INFINITY ? 0.f : exp2f(mv - M);
      const f32x4 ov = *reinterpret_cast<const f32x4*>(a.po + (base + sp) * DH + d);
      L = fmaf(a.pml[(base + sp) * 2 + 1], f, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(ov[e], f, O[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) Elem<T>::store((T*)a.out + (row0 + m) * DH + d + e, attn_finish_nan(O[e], L));
  }
}

template <typename T, int DH>
__global__ __launch_bounds__(kMergeThreads) void attn_q_combine(AttnQArgs a) {
  const int h = blockIdx.x, i = blockIdx.y;
  const int ns = (min(a.kl[i], a.ms * kAttnSplit) + kAttnSplit - 1) / kAttnSplit;
  if (ns <= 1) return;  // finished by its split's workgroup
  const int64_t row = (int64_t)i * a.H + h;
  attn_merge_parts<T, DH>(a.po, a.pml, ns, [&](int s) { return row * a.ms + s; }, (T*)a.out + row * DH);
}

// Splits a workgroup takes, one after the other. A row of up to four splits is one
// workgroup's where the rows alone make 1024 splits (two rounds of workgroups): it
// finishes the row itself, with the combine kernel's arithmetic, and neither that
// launch nor workgroups that find no keys are needed. 112 rows x 16 heads x 128-1200
// keys: 104 -> 82 us, 64 x 16 x 1100-2000: 88 -> 86. Longer rows keep a workgroup per
// split (64 rows x 4 heads x 32k keys, four splits each: 400 -> 410 us), and so do
// fewer rows, whose splits are what fills the chip (8 x 16 x 1100-2000: 18.0 -> 21.3).
constexpr int kAqRowSplits = 4;
constexpr int kAqFill = 1024;
static int splits_per_workgroup(int ms, int64_t rows) {
  return ms <= kAqRowSplits && ms * rows >= kAqFill ? ms : 1;
}

template <typename T, int CODE, int DH>
static void launch_attn_q(const AttnQArgs& a, hipStream_t st) {
  const int wgs = (a.ms + a.spw - 1) / a.spw;
  hipLaunchKernelGGL((attn_q_split_kernel<T, CODE, DH>), dim3(wgs, a.Hkv, a.n), dim3(64 * kAqWaves), 0, st, a);
  if (wgs > 1)  // some query may span several workgroups
    hipLaunchKernelGGL((attn_q_combine<T, DH>), dim3(a.H, a.n), dim3(kMergeThreads), 0, st, a);
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
  if (H <= 0 || H > kAqMaxHeads || H % Hkv != 0 || kv_len_max < 1 ||
      (kv_block_rows > 1 && kv_len_max > kv_block_rows)) {
    set_error("%s: bad shape H=%d Hkv=%d kv_len_max=%d kv_block_rows=%lld", me, H, Hkv, kv_len_max,
              (long long)kv_block_rows);
    return kBadArg;
  }
  const int G = H / Hkv;
  if ((dtype != kBF16 && dtype != kF32) || G > kAqMaxG) {
    set_error("%s: unsupported dtype=%d G=%d (G = H / Hkv up to %d)", me, dtype, G, kAqMaxG);
    return kUnsupported;
  }
  if (n > 65535 || kv_len_max > INT32_MAX - (kAttnSplit - 1)) {  // whole splits below 2^31
    set_error("%s: n=%d kv_len_max=%d beyond the grid (65535 rows, 2^31 - 1024 keys)", me, n, kv_len_max);
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
  a.spw = splits_per_workgroup(a.ms, (int64_t)n * Hkv);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.br = kv_block_rows;
#define WFD_ATTNQ_CASE(TT, DT, CODE)                            \
  if (dtype == DT && code == CODE) {                             \
    if (Dh == 64) launch_attn_q<TT, CODE, 64>(a, stream);        \
    else launch_attn_q<TT, CODE, 128>(a, stream);                \
  }
  WFD_ATTNQ_CASE(bf16_t, kBF16, WFD_E4M3)
  WFD_ATTNQ_CASE(bf16_t, kBF16, WFD_INT8)
  WFD_ATTNQ_CASE(float, kF32, WFD_E4M3)
  WFD_ATTNQ_CASE(float, kF32, WFD_INT8)
#undef WFD_ATTNQ_CASE
  return launch_status(me);
}

}  // extern "C"
