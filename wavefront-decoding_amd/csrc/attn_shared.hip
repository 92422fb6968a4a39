// Decode attention of rows that share a prefix: the rows of a group attend the
// group's prefix, computed for all of them together, and then keys of their own.
//
//   o_i = softmax over [prefix of i's group | i's own keys] of (q_i . k * scale), times V
//
// Softmax over a union is a merge of softmaxes over its parts: a part leaves its
// maximum m, sum l and unnormalised output o, and the row is sum o 2^(m - M) /
// sum l 2^(m - M) over its parts. The prefix is cut into chunks of keys, a
// workgroup computes one chunk for up to 32 (query row, query head) pairs
// of a group and one kv head -- each key is read once for all of them -- and a row's
// own keys are cut likewise, for that row alone; attn_shared_combine merges a
// row's parts.
//
// The chunks follow from the lengths and Hkv alone, and a row's arithmetic within
// a chunk from the chunk, so a row's bits do not depend on its group's other
// rows, on the launch, or on where the row sits.
#include "attn_combine.h"

namespace wfd {

constexpr int kShRows = 32;      // (query row, head) pairs per workgroup
constexpr int kShWaves = 4;      // key streams per workgroup
constexpr int kShMinChunk = 128;
constexpr int kShMaxChunk = 1024;
constexpr int kShOwnChunk = 512;
constexpr int kShTarget = 128;   // chunks x kv heads aimed at
constexpr int kShMaxG = 16;
constexpr int kShMaxRows = 65535;  // the merge's grid
constexpr int kShMaxHeads = 4096;  // a chunk's keys stay within 32-bit offsets of its first

// Keys per chunk of a prefix of P keys: 128 chunks over the kv heads, a workgroup
// each for every second CU, while they are at least 128 keys: the parts' traffic
// grows with the chunks, and a group's pairs and the other groups fill the rest.
// In us, with 64 / 128 / 256 chunks (rows x keys x kv heads):
//   few rows:  4 x 2000 x 16  14.1 / 12.6 / 13.8    4 x 8000 x 4    15.0 / 13.8 / 15.5
//              4 x 16000 x 2  16.0 / 14.9 / 18.2    16 x 4000 x 16  23.7 / 18.8 / 17.7
//              8 x 32000 x 4  27.5 / 27.5 / 27.4
//   many:      64 x 8000 x 16 56 / 56 / 59          64 over 4 x 2000 x 16  44 / 47 / 54
//              100 over 3 x 20-32k x 4  92-94 / 92-97 / 109
// At most 1024 keys (512: 58 for 64 x 8000, 105 for the 100 rows; 2048: 55, 95), and 512
// of a row's own (256: 60 and 98; 1024: 56 and 95).
__host__ __device__ inline int prefix_chunk(int P, int Hkv) {
  const int64_t c = ((int64_t)P * Hkv + kShTarget - 1) / kShTarget;
  const int64_t r = (c + kShMinChunk - 1) / kShMinChunk * kShMinChunk;
  return (int)(r < kShMinChunk ? kShMinChunk : (r > kShMaxChunk ? kShMaxChunk : r));
}

__host__ __device__ inline int div_up(int a, int b) { return a <= 0 ? 0 : (a - 1) / b + 1; }

// The most chunks any prefix of up to P keys makes (a chunk has at least
// P Hkv / kShTarget keys unless it has 1024).
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
  int n, H, Hkv, ng, gmax, tiles, pchunks, ochunks, pmax, omax;
  uint32_t items;
  float scale_log2;
};

// What one workgroup computes: keys [k0, k1) of the slot rows from `base`, for nr
// pairs from pair p0 of the query rows from row0 (pair r: query row row0 + r / G,
// head g G + r % G), left as the rows' part `part`.
struct ShItem {
  int g, row0, p0, nr, k0, k1, part;
  int64_t base;
};

// The workgroup's item; false if it has none (a shorter prefix, a smaller group).
// Prefix items first, RT pairs each. The items are the grid's workgroups in order, x first. The tiles of one (group, chunk, head) read
// the same keys: they are 8 workgroups apart, so they run on one XCD at about the
// same time, and one of them brings the keys to its L2.
template <int RT>
__device__ __forceinline__ bool sh_item(const ShArgs& a, ShItem& it) {
  const uint32_t G = a.H / a.Hkv;
  const uint32_t x = blockIdx.y * gridDim.x + blockIdx.x;  // the host keeps the items below 2^31
  if (x >= a.items) return false;  // the grid's last row
  const uint32_t nkeys = (uint32_t)a.ng * a.pchunks * a.Hkv;
  const uint32_t nprefix = (nkeys + 7) / 8 * 8 * a.tiles;
  if (x < nprefix) {
    const uint32_t q = x / 8;
    const uint32_t tile = q % a.tiles;
    const uint32_t kg = q / a.tiles * 8 + x % 8;
    if (kg >= nkeys) return false;
    it.g = (int)(kg % a.Hkv);
    const uint32_t jc = kg / a.Hkv;
    const int c = (int)(jc % a.pchunks), j = (int)(jc / a.pchunks);
    const int P = max(min(a.plen[j], a.pmax), 0);
    const int ck = prefix_chunk(P, a.Hkv);
    it.row0 = a.gfirst[j];
    it.p0 = tile * RT;
    it.nr = min((min(a.gfirst[j + 1], a.n) - it.row0) * (int)G - it.p0, RT);
    it.k0 = c * ck;  // below 2^31: there are at most 2^21 chunks of 1024
    it.k1 = it.k0 + min(ck, P - it.k0);
    it.part = c;
    it.base = a.pbase[j];
  } else {
    const uint32_t y = x - nprefix;
    it.g = (int)(y % a.Hkv);
    const uint32_t ic = y / a.Hkv;
    const int c = (int)(ic % a.ochunks);
    it.row0 = (int)(ic / a.ochunks);
    it.p0 = 0;
    it.nr = (int)G;
    it.k0 = c * kShOwnChunk;
    it.k1 = it.k0 + min(kShOwnChunk, max(min(a.rlen[it.row0], a.omax), 0) - it.k0);
    it.part = a.pchunks + c;
    it.base = a.rbase[it.row0];
  }
  return it.k0 < it.k1 && it.nr > 0;
}

__device__ __forceinline__ int64_t sh_pair(const ShArgs& a, const ShItem& it, int r) {
  const int G = a.H / a.Hkv;
  const int row = (it.p0 + r) / G;
  return (int64_t)(it.row0 + row) * a.H + it.g * G + (it.p0 + r - row * G);
}

// Merges the workgroup's key streams, one per wave, and leaves the part: o_lds
// [wave][pair][DH, pitch OP], m / l [wave][pair]. A thread first has one pair's
// weights and place (it would otherwise compute them for every value), then takes
// four columns of a pair at a time. With `again` it only replaces the NaN that it left
// before (a thread has the same values both times) where the streams now hold an infinity.
template <int DH, int OP, int RT>
__device__ __forceinline__ void sh_leave(const ShArgs& a, const ShItem& it, const float* o_lds, const float* m_lds,
                                         float* l_lds, int64_t* at_lds, bool again) {
  const int ms = a.pchunks + a.ochunks;
  if (threadIdx.x < it.nr) {
    const int r = threadIdx.x;
    float M = -INFINITY, L = 0.f, f[kShWaves];
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) M = fmaxf(M, m_lds[w * RT + r]);
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) {
      const float mw = m_lds[w * RT + r];
      f[w] = mw == -INFINITY ? 0.f : exp2f(mw - M);
      L = fmaf(l_lds[w * RT + r], f[w], L);
    }
    const int64_t at = sh_pair(a, it, r) * ms + it.part;
    a.pml[2 * at] = M;
    a.pml[2 * at + 1] = L;
    at_lds[r] = at;
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) l_lds[w * RT + r] = f[w];
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < it.nr * (DH / 4); idx += 64 * kShWaves) {
    const int r = idx / (DH / 4), d = 4 * (idx % (DH / 4));
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) {
      const float f = l_lds[w * RT + r];
      const f32x4 ow = *reinterpret_cast<const f32x4*>(o_lds + (w * RT + r) * OP + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(ow[e], f, O[e]);
    }
    f32x4* left = reinterpret_cast<f32x4*>(a.po + at_lds[r] * DH + d);
    if (again) {  // uniform
      const f32x4 was = *left;
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = was[e] != was[e] && fabsf(O[e]) == INFINITY ? O[e] : was[e];
    }
    *left = O;
  }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 sh_mfma32(const u32x4& x, const u32x4& y, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), acc, 0,
                                                 0, 0);
}

// The scale's size; zero is a tiny one, under which -inf stays -inf, and NaN is NaN.
__device__ __forceinline__ float sh_scale(const ShArgs& a) {
  return a.scale_log2 != a.scale_log2 ? a.scale_log2 : fmaxf(fabsf(a.scale_log2), 1e-37f);
}

// One tile's scores (of the lane's pair) to probabilities, under the pair's reference
// point: the maximum when it was last moved, which is when a tile exceeds it by more
// than 2^8. Probabilities up to 2^8 lose nothing in fp32 sums or bf16, and most tiles
// rescale nothing (with the running maximum itself some pair of the 32 moves in nearly
// every tile). It depends on the pair's own scores only.
template <int NDB>
__device__ __forceinline__ void sh_softmax(f32x16& sc, f32x16 (&o)[NDB], float& mref, float& lrun, float scale) {
  float mt = -INFINITY;
#pragma unroll
  for (int r = 0; r < 16; ++r) mt = fmaxf(mt, sc[r]);
  mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * scale;
  if (__builtin_amdgcn_ballot_w64(mt > mref + 8.f)) {
    const float mnew = mt > mref + 8.f ? mt : mref;
    const float corr = mref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref - mnew);
    mref = mnew;
    lrun *= corr;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= corr;
  }
  const float ref = mref == -INFINITY ? 0.f : mref;
  // v_exp_f32 flushes below 2^-126: far under what a sum that holds 2^-8 or more resolves
  float lt = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    sc[r] = __builtin_amdgcn_exp2f(fmaf(sc[r], scale, -ref));
    lt += sc[r];
  }
  lrun += lt + __shfl_xor(lt, 32, 64);
}

// A wave's stream to LDS for the merge: lane (col, hf) holds pair col's columns
// 32 db + 8 (r / 4) + 4 hf + r % 4.
template <int DH, int OP, int RT>
__device__ __forceinline__ void sh_keep(const ShItem& it, int wave, int col, int hf, const f32x16 (&o)[DH / 32],
                                        float mref, float lrun, float* o_lds, float* m_lds, float* l_lds) {
  if (col < it.nr) {
#pragma unroll
    for (int db = 0; db < DH / 32; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(o_lds + (wave * RT + col) * OP + 32 * db + 8 * r + 4 * hf) =
            f32x4{o[db][4 * r], o[db][4 * r + 1], o[db][4 * r + 2], o[db][4 * r + 3]};
    if (hf == 0) {
      m_lds[wave * RT + col] = mref;
      l_lds[wave * RT + col] = lrun;
    }
  }
}

// bf16: 32 pairs per workgroup, one per column of the 32x32x16 MFMA, and four
// waves that each stream 32-key tiles of the chunk (wave w tiles w, w + 4, ...)
// through LDS of their own: whole rows to registers a tile ahead, to LDS as
// loaded, no workgroup barrier before the merge. A wave computes S^T = K Q^T and
// O^T = V^T P^T; the K rows of a tile are taken in the order that makes a lane's
// S^T registers the 8 consecutive keys its P^T operand wants (result register r of
// lane half hf is key 16 (r / 8) + 8 hf + r % 8), so P never leaves its lane, and
// V^T comes out of the row-major tile by transposing LDS reads. Keys past the
// chunk read as zeros and score -inf.
//
// 64 rows x 8000 keys x 16 heads: 50 us and 5 for the merge (floor 41), of which the
// loads alone take 43; 100 rows x 20-32k x 4 kv heads: 84-88 + 8, loads alone 60: each
// tile of 32 pairs takes its prefix from the L2 again (740 MB, 12 TB/s), and products
// and exponentials only partly hide behind them at two waves per SIMD. 64 pairs a
// wave (57 -> 69 and 100 -> 129 us), eight waves sharing the tiles of 64 pairs (55 -> 56
// and 89 -> 94) and two chains of K Q^T (as one) were no faster, all with P in one term.
template <int DH>
__global__ __launch_bounds__(64 * kShWaves) __attribute__((amdgpu_waves_per_eu(2))) void attn_shared_bf16_kernel(
    ShArgs a) {
  constexpr int RT = kShRows;
  constexpr int TK = 32;
  constexpr int NDS = DH / 16;
  constexpr int NDB = DH / 32;
  constexpr int KP = DH + 8;    // LDS row pitches: K reads 16 bytes of 32 rows, V^T 64 bytes of 8 rows,
  constexpr int VP = DH + 32;   // each spread over all banks
  constexpr int CPR = DH / 8;   // 16-byte pieces per row
  constexpr int RPI = 64 / CPR;
  constexpr int NLD = TK / RPI;
  constexpr int OP = DH + 4;
  constexpr int kWaveEls = TK * (KP + VP);
  constexpr size_t kStage = sizeof(bf16_t) * kWaveEls * kShWaves, kMerge = sizeof(float) * kShWaves * RT * OP;
  __shared__ __align__(16) unsigned char lds[kStage > kMerge ? kStage : kMerge];
  __shared__ float m_lds[kShWaves * RT];
  __shared__ float l_lds[kShWaves * RT];
  __shared__ int64_t at_lds[RT];
  __shared__ int nan_lds;
  ShItem it;
  if (!sh_item<RT>(a, it)) return;  // uniform
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 31, hf = lane >> 5;
  bf16_t* k_lds = reinterpret_cast<bf16_t*>(lds) + wave * kWaveEls;
  bf16_t* v_lds = k_lds + TK * KP;

  // K / V of this head from key k0; the resources end with key k1 - 1
  const int64_t rs = a.br > 1 ? (int64_t)DH : (int64_t)a.Hkv * DH;
  const int64_t at = kv_offset(it.base, it.g, a.Hkv, DH, a.br) + it.k0 * rs;
  const int nk = it.k1 - it.k0;
  const uint32_t rsb = (uint32_t)(rs * sizeof(bf16_t));
  const uint32_t span = (uint32_t)(nk - 1) * rsb + DH * sizeof(bf16_t);
  auto rsrc = [&](const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>((const bf16_t*)p + at), (short)0, span, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t kr = rsrc(a.kc), vr = rsrc(a.vc);
  const int lr = lane / CPR, lp = lane % CPR;  // row within a load, piece
  u32x4 kreg[NLD], vreg[NLD];
  uint32_t off[NLD];
  auto first_tile = [&]() {
#pragma unroll
    for (int s = 0; s < NLD; ++s) off[s] = (uint32_t)(TK * wave + RPI * s + lr) * rsb + (uint32_t)lp * 16u;
  };
  auto fetch = [&]() {  // this wave's next tile; zeros past the chunk
#pragma unroll
    for (int s = 0; s < NLD; ++s) {
      kreg[s] = buf_ld16(kr, off[s]);
      vreg[s] = buf_ld16(vr, off[s]);
      off[s] += (uint32_t)(TK * kShWaves) * rsb;
    }
  };
  first_tile();
  fetch();

  // Q as the B operand; a negative scale's sign goes to q, so that scores order as
  // their products do
  const float scale = sh_scale(a);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  u32x4 qf[NDS];
  {
    const bf16_t* qp = (const bf16_t*)a.q + sh_pair(a, it, min(col, it.nr - 1)) * DH + 8 * hf;
#pragma unroll
    for (int s = 0; s < NDS; ++s) qf[s] = ld16(qp + 16 * s) ^ flip;
  }
  const int krow = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
  const int tg = lane >> 4, ti = lane & 15;
  const int v_lane = ((tg >> 1) * 8 + (ti >> 2)) * VP + 16 * (tg & 1) + 4 * (ti & 3);
  auto vt_frag = [&](int db, int s) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    typedef const __attribute__((address_space(3))) void* lds_ptr;
    const bf16_t* p = v_lds + v_lane + 16 * s * VP + 32 * db;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_ptr)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_ptr)(p + 4 * VP));
    const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
    return u32x4{x.x, x.y, y.x, y.y};
  };

  // A second pass over the chunk where the first left a NaN: the low terms below have
  // either sign, and zero, so that an infinity in V comes out as a NaN. With the high
  // term, of p's sign, in their place it is itself unless the sum is a NaN all the same.
  // Asking costs 0.3 us a launch (4 rows x 512 keys 10.2 -> 10.5), nothing past the noise
  // in the long cases.
  bool again = false;
  for (;;) {  // uniform over the workgroup
  float mref = -INFINITY, lrun = 0.f;
  f32x16 o[NDB];
#pragma unroll
  for (int c = 0; c < NDB; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[c][r] = 0.f;

  for (int t0 = TK * wave; t0 < nk; t0 += TK * kShWaves) {  // uniform over the wave
#pragma unroll
    for (int s = 0; s < NLD; ++s) {
      *reinterpret_cast<u32x4*>(k_lds + (RPI * s + lr) * KP + 8 * lp) = kreg[s];
      *reinterpret_cast<u32x4*>(v_lds + (RPI * s + lr) * VP + 8 * lp) = vreg[s];
    }
    fetch();
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x16 sc;
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
    for (int s = 0; s < NDS; ++s)
      sc = sh_mfma32(*reinterpret_cast<const u32x4*>(k_lds + krow * KP + 16 * s + 8 * hf), qf[s], sc);
    if (t0 + TK > nk) {  // the chunk's last tile (uniform)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (t0 + 16 * (r >> 3) + 8 * hf + (r & 7) >= nk) sc[r] = -INFINITY;
    }
    sh_softmax<NDB>(sc, o, mref, lrun, scale);
    // P meets V in two bf16 terms, half a step of 2^-16 of it. In one (2^-8, at random
    // signs) the output was 0.0023 of its norm off instead of 0.00166, which is its own
    // rounding, for 0-5 % less time; a third term changes that in the seventh digit and
    // costs 100 rows x 20-32k 90 -> 99 us; fp32 products take 8 times the MFMA time.
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = sc[8 * s + 2 * e], y = sc[8 * s + 2 * e + 1];
        hi[e] = f32x2_to_bf16x2_bits(x, y);
        lo[e] = f32x2_to_bf16x2_bits(x - __uint_as_float(hi[e] << 16), y - __uint_as_float(hi[e] & 0xffff0000u));
        lo[e] = again ? hi[e] : lo[e];
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const u32x4 vf = vt_frag(db, s);
        o[db] = sh_mfma32(vf, lo, o[db]);
        o[db] = sh_mfma32(vf, hi, o[db]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // the next tile overwrites this one
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  if (threadIdx.x == 0) nan_lds = 0;
  __syncthreads();  // every wave's tiles are done: the merge takes their LDS
  float* o_lds = reinterpret_cast<float*>(lds);
  sh_keep<DH, OP, RT>(it, wave, col, hf, o, mref, lrun, o_lds, m_lds, l_lds);
  float sum[NDB] = {};  // NaN if any of them is
#pragma unroll
  for (int r = 0; r < 16; ++r)
#pragma unroll
    for (int db = 0; db < NDB; ++db) sum[db] += o[db][r];
#pragma unroll
  for (int db = 1; db < NDB; ++db) sum[0] += sum[db];
  if (sum[0] != sum[0]) nan_lds = 1;
  __syncthreads();
  const bool more = !again && nan_lds;
  sh_leave<DH, OP, RT>(a, it, o_lds, m_lds, l_lds, at_lds, again);
  if (!more) break;
  again = true;
  __syncthreads();
  first_tile();
  fetch();
  }
}

// fp32: the same on the 32x32x2 MFMA. A lane's operands of K Q^T are four consecutive
// columns at a time (lane half hf takes columns 8 j + 4 hf + e at step 4 j + e), its
// S^T register r is key 8 (r / 4) + 4 hf + r % 4, which is also the key it supplies of
// P^T at step r. K goes through LDS; V^T comes straight from the cache, 32 consecutive
// values of a row to half of the lanes, loaded under the scores, and the next tile of K
// under P V, into the registers that V leaves. 64 rows x 8000 keys x 16 heads: 124-139
// us (floor 82; its products alone, by count, 55); V through LDS too, which leaves a wave per SIMD,
// 152; 16 pairs on the 16x16x4 form, operands straight from the cache, 371.
template <int DH>
__global__ __launch_bounds__(64 * kShWaves) __attribute__((amdgpu_waves_per_eu(2))) void attn_shared_f32_kernel(
    ShArgs a) {
  constexpr int RT = kShRows;
  constexpr int TK = 32;
  constexpr int NDB = DH / 32;
  constexpr int KP = DH + 4;    // LDS row pitch: 16 bytes of 16 rows are spread over all banks
  constexpr int CPR = DH / 4;   // 16-byte pieces per row
  constexpr int RPI = 64 / CPR;
  constexpr int NLD = TK / RPI;
  constexpr int OP = DH + 4;
  constexpr int kWaveEls = TK * KP;
  static_assert(kWaveEls >= RT * OP, "the merge takes the tiles' LDS");
  __shared__ __align__(16) float lds[kWaveEls * kShWaves];
  __shared__ float m_lds[kShWaves * RT];
  __shared__ float l_lds[kShWaves * RT];
  __shared__ int64_t at_lds[RT];
  ShItem it;
  if (!sh_item<RT>(a, it)) return;  // uniform
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 31, hf = lane >> 5;
  float* k_lds = lds + wave * kWaveEls;

  const int64_t rs = a.br > 1 ? (int64_t)DH : (int64_t)a.Hkv * DH;
  const int64_t at = kv_offset(it.base, it.g, a.Hkv, DH, a.br) + it.k0 * rs;
  const int nk = it.k1 - it.k0;
  const uint32_t rsb = (uint32_t)(rs * sizeof(float));
  const uint32_t span = (uint32_t)(nk - 1) * rsb + DH * sizeof(float);
  auto rsrc = [&](const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>((const float*)p + at), (short)0, span, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t kr = rsrc(a.kc), vr = rsrc(a.vc);
  const int lr = lane / CPR, lp = lane % CPR;
  u32x4 kreg[NLD];
  float vreg[16][NDB];
  uint32_t koff = (uint32_t)(TK * wave + lr) * rsb + (uint32_t)lp * 16u;
  uint32_t voff = (uint32_t)(TK * wave + 4 * hf) * rsb + (uint32_t)col * 4u;
  const uint32_t next = (uint32_t)(TK * kShWaves) * rsb;
  // zeros past the chunk
  auto fetch_k = [&](int q) {  // a quarter of this wave's next tile
#pragma unroll
    for (int s = q * NLD / 4; s < (q + 1) * NLD / 4; ++s) kreg[s] = buf_ld16(kr, koff + (uint32_t)(RPI * s) * rsb);
  };
  auto fetch_v = [&]() {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t row = voff + (uint32_t)(8 * (r >> 2) + (r & 3)) * rsb;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        vreg[r][db] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(vr, row + 128u * db, 0, 0));
    }
    voff += next;
  };
#pragma unroll
  for (int q = 0; q < 4; ++q) fetch_k(q);
  koff += next;

  const float scale = sh_scale(a);  // as in the bf16 kernel
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80000000u : 0u;
  u32x4 qf[DH / 8];
  {
    const float* qp = (const float*)a.q + sh_pair(a, it, min(col, it.nr - 1)) * DH + 4 * hf;
#pragma unroll
    for (int s = 0; s < DH / 8; ++s) qf[s] = ld16(qp + 8 * s) ^ flip;
  }
  float mref = -INFINITY, lrun = 0.f;
  f32x16 o[NDB];
#pragma unroll
  for (int c = 0; c < NDB; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[c][r] = 0.f;

  for (int t0 = TK * wave; t0 < nk; t0 += TK * kShWaves) {  // uniform over the wave
#pragma unroll
    for (int s = 0; s < NLD; ++s) *reinterpret_cast<u32x4*>(k_lds + (RPI * s + lr) * KP + 4 * lp) = kreg[s];
    fetch_v();
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x16 sc;
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
    for (int j = 0; j < DH / 8; ++j) {
      const f32x4 kf = *reinterpret_cast<const f32x4*>(k_lds + col * KP + 8 * j + 4 * hf);
      const f32x4 q4 = __builtin_bit_cast(f32x4, qf[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sc = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], q4[e], sc, 0, 0, 0);
    }
    if (t0 + TK > nk) {  // the chunk's last tile (uniform)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (t0 + 8 * (r >> 2) + 4 * hf + (r & 3) >= nk) sc[r] = -INFINITY;
    }
    sh_softmax<NDB>(sc, o, mref, lrun, scale);
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // the next tile of K takes the registers that V leaves
#pragma unroll
      for (int r = 4 * q; r < 4 * q + 4; ++r)
#pragma unroll
        for (int db = 0; db < NDB; ++db)
          o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(vreg[r][db], sc[r], o[db], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      fetch_k(q);
    }
    koff += next;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // the next tile overwrites this one
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  __syncthreads();  // every wave's tiles are done: the merge takes their LDS
  sh_keep<DH, OP, RT>(it, wave, col, hf, o, mref, lrun, lds, m_lds, l_lds);
  __syncthreads();
  sh_leave<DH, OP, RT>(a, it, lds, m_lds, l_lds, at_lds, false);
}

// One row's parts, prefix chunks then its own. The row's group is found by one
// wave-wide look at group_first per 64 groups. A row past the rows that the grid was
// sized for has no prefix parts: it is NaN, not a merge of what the workspace held.
template <typename T, int DH>
__global__ __launch_bounds__(kMergeThreads) void attn_shared_combine(ShArgs a) {
  const int h = blockIdx.x, i = blockIdx.y, lane = threadIdx.x & 63;
  const int own = div_up(min(a.rlen[i], a.omax), kShOwnChunk);
  int P = 0, at = 0;
  for (int j0 = 0; j0 < a.ng; j0 += 64) {  // uniform
    const int j = min(j0 + lane, a.ng - 1);
    const int first = a.gfirst[j];
    const uint64_t hit = __ballot(j0 + lane < a.ng && first <= i && i < a.gfirst[j + 1]);
    const int len = a.plen[j];
    if (hit) {
      P = __shfl(len, __builtin_ctzll(hit), 64);
      at = i - __shfl(first, __builtin_ctzll(hit), 64);
    }
  }
  P = min(P, a.pmax);
  const int np = P > 0 ? div_up(P, prefix_chunk(P, a.Hkv)) : 0;
  const int64_t row = (int64_t)i * a.H + h, base = row * (a.pchunks + a.ochunks);
  if (np && at >= a.gmax) {  // uniform
    if (threadIdx.x < DH) Elem<T>::store((T*)a.out + row * DH + threadIdx.x, NAN);
    return;
  }
  attn_merge_parts<T, DH>(a.po, a.pml, np + own, [&](int s) { return base + (s < np ? s : a.pchunks + s - np); },
                          (T*)a.out + row * DH);
}

// A launch has fewer than 2^32 threads in x. A multiple of 8, as sh_item's order wants.
constexpr uint32_t kShGridX = 1u << 23;

template <typename T, int DH>
static void launch_shared(ShArgs& a, hipStream_t st) {
  const int64_t nkeys = (int64_t)a.ng * a.pchunks * a.Hkv, own = (int64_t)a.n * a.ochunks * a.Hkv;
  a.items = (uint32_t)((nkeys + 7) / 8 * 8 * a.tiles + own);
  const dim3 grid(a.items < kShGridX ? a.items : kShGridX, (a.items + kShGridX - 1) / kShGridX), block(64 * kShWaves);
  if (a.items) {
    if constexpr (sizeof(T) == 4)
      hipLaunchKernelGGL((attn_shared_f32_kernel<DH>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((attn_shared_bf16_kernel<DH>), grid, block, 0, st, a);
    if (hipPeekAtLastError() != hipSuccess) return;  // no parts to merge
  }
  hipLaunchKernelGGL((attn_shared_combine<T, DH>), dim3(a.H, a.n), dim3(kMergeThreads), 0, st, a);
}

}  // namespace wfd

extern "C" {

size_t wfd_attn_shared_workspace_bytes(int n, int H, int Hkv, int Dh, int prefix_len_max, int kv_len_max) {
  using namespace wfd;
  // 0 for what the call refuses; the largest it takes is below 2^61
  if (n <= 0 || n > kShMaxRows || H <= 0 || H > kShMaxHeads || Hkv <= 0 || Dh <= 0 || Dh > 128 || prefix_len_max < 0 ||
      kv_len_max < 0)
    return 0;
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
  if (n < 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || H > kShMaxHeads || ngroups < 0 || group_max < 0 ||
      kv_block_rows < 0 || prefix_len_max < 0 || kv_len_max < 0) {
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
  a.gmax = group_max;
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
  const double most = (((double)ngroups * a.pchunks * Hkv + 8) * (double)tiles + (double)n * a.ochunks * Hkv);
  if (most > 2147483647.0 || n > kShMaxRows) {
    set_error("%s: n=%d ngroups=%d group_max=%d prefix_len_max=%d kv_len_max=%d beyond the grid", me, n, ngroups,
              group_max, prefix_len_max, kv_len_max);
    return kUnsupported;
  }
  a.tiles = (int)tiles;
  if (dtype == kBF16)
    Dh == 64 ? launch_shared<bf16_t, 64>(a, stream) : launch_shared<bf16_t, 128>(a, stream);
  else
    Dh == 64 ? launch_shared<float, 64>(a, stream) : launch_shared<float, 128>(a, stream);
  return launch_status(me);
}

}  // extern "C"
