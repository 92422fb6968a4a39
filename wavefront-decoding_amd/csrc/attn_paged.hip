// Attention of a sequence's newest tokens over a KV cache in pages (pages.h).
//
//   o = softmax over the visible keys of (q . k * scale), times V
//
// visible to the row at position p: keys j <= p, and with a window those with
// j > p - window or j < sinks. The rows of a sequence are dealt in tiles, whose
// (row, head) pairs of one kv head are the columns of the products; a tile's visible
// keys are a list of key blocks (the blocks with sinks, then those from the first
// row's window to the last row), which is cut into parts where the sequence alone
// would leave CUs idle, a workgroup each. Softmax over a union is a merge of
// softmaxes over its parts: a part leaves its maximum m, sum l and unnormalised
// output o, and attn_paged_combine adds them up.
//
// A sequence of few rows (up to kPaFewPairs pairs of a kv head) is cut at key positions
// that are the same for every row, and a wave of a part takes every fourth block of it by
// the block's place in the sequence. What a tile holds beside a row then adds hidden keys to
// it and nothing else, and a hidden key changes no bit: a row has the bits it has alone,
// as the next token of its context. A sequence of more rows is cut by its own rows and
// length, unless the caller asks for every row's own bits (wfd_attn_paged_by_row). In either
// case the rest of the call has no part in it.
#include <algorithm>
#include <type_traits>

#include "attn_combine.h"
#include "pages.h"

namespace wfd {

constexpr int kPaRows = 32;  // pairs of a wave: the columns of its 32x32 MFMA
constexpr int kPaWaves = 4;
constexpr int kPaMaxG = kPaRows;
// A sequence's pairs per kv head up to which its rows are "few": read by 32 pairs at a time, with
// no waiting for other waves. 16 rows of 4 heads over 1000 keys 18.1 us as few, 22.5 as many, 32
// sequences of them 28.4 and 28.7; 24 such rows 18.0 and 23.3, 32 sequences of these 37.4 and 31.7.
constexpr int kPaFewPairs = 64;
constexpr int kPaAllFew = 0x7fffffff;  // all of them, where every row is to have its own bits
constexpr int kPaManyRows = kPaRows * kPaWaves;
// Keys per block of the few-row kernels and of the many-row one. Blocks, parts and targets are
// powers of two and counted by shifts: each workgroup looks for its own item, and with 64-bit
// divisions in that 112 single rows took 141 us for 134.
constexpr int kPaLogBlock = 5, kPaBlock = 1 << kPaLogBlock;
constexpr int kPaManyLogBlock = 6, kPaManyBlock = 1 << kPaManyLogBlock;
// Few rows: parts of 512 keys up to key 32768 / Hkv, of 1024 behind it; under a window of 512. One
// row of 16 heads over 1000 keys takes 16.9 us, 8 over 511 to 777 18.3, 64 over 500 / 600 keys 45.6
// / 70, 8 of 4 kv heads over 1000 to 1200 17.1. With near parts of 256: 13.9, 18.4, 51 / 64, 15.2,
// and 16 drafts of 8 rows over 500 to 3000 keys 48.5 for 39.6. With 1024 throughout: 18.5, 16.6,
// 45.6 / 53, 23.6, and one row over 2000 keys 22.7 for 17.1, as with half as many near parts; with
// twice as many 64 rows over 32700 keys, 4 kv heads, 773 for 767 (1024: 746). Windows with parts
// of 1024: 64 rows, window 1024, 48.7 for 37.7, window 4096 122 for 117.
constexpr int kPaLogNear = 4, kPaLogFar = 5;  // blocks of either
constexpr int kPaNear = 64;                   // near parts x kv heads
// fp32 sequences of more pairs: parts x tiles x kv heads that are aimed at, and the least keys of a part.
constexpr int kPaTarget = 64;
constexpr int kPaMinPart = 256;
// Many rows: two workgroups a CU (512 rows behind 7600 keys 75 us, with half as many 91; with the
// parts' sizes rounded up to powers of two 80 behind 7700) of at least 512 keys: 128 rows of 16
// heads over 1000 keys 25 us (with 1024: 36, with 256: 22), 32 such sequences 133 (134, 172).
// Twice that for a sequence of 64 (tile, kv head)s, four times for one of 96: 500 rows of 16 heads
// over 2000 keys 42 us for 34, four such sequences 66 for 75; 700 rows (96) 58 us, with twice 44,
// once 40, four such sequences 76, 91, 99, eight 131, 162, 201.
constexpr int kPaManyMinPart = 512;
constexpr int kPaManyLogTarget = 9, kPaManyTarget = 1 << kPaManyLogTarget;
// Workgroups of a launch, which take the items in turn: of few rows those that the card holds
// at once (the host knows bounds of the items only; with four times as many 33 sequences' drafts
// take 33.7 us for 30.6), of many rows more, as their items differ in length.
constexpr int kPaResident = 512;
constexpr int kPaManyGrid = 8192;
constexpr int kPaMergeGrid = 2048;

// Where a sequence's blocks are cut: `near` parts of 2^kPaLogNear blocks from position 0 on, behind
// them parts of 2^lf.
struct PaCut {
  int near, lf;
  __host__ __device__ int of(int block) const {
    const int nb = near << kPaLogNear;
    return block < nb ? block >> kPaLogNear : near + ((block - nb) >> lf);
  }
  __host__ __device__ int start(int part) const {
    return part < near ? part << kPaLogNear : (near << kPaLogNear) + ((part - near) << lf);
  }
};

// window: the caller's, also where it covers all keys, so that kv_len_max does not decide on bits.
inline PaCut pa_few_cut(int Hkv, int window) {
  return window ? PaCut{0, kPaLogNear} : PaCut{(kPaNear + Hkv - 1) / Hkv, kPaLogFar};
}

struct PaArgs {
  const void *q, *kp, *vp;
  const int32_t *cu_q, *kv_len;
  void* out;
  PageMap m;
  float *po, *pml;       // the parts' slots
  int64_t seq_slots;     // slots kept per sequence; 0: row_per for every row and head
  int n, nseq, H, Hkv, G, qmax, kmax, window, sinks;
  int g_magic;           // x / G = x g_magic >> 16 for x < 128
  int few_tile, many_tile;  // rows of a tile
  int row_per;
  int few_pairs;         // kPaFewPairs, or kPaAllFew
  uint32_t many_wgs, many_lead;  // of a kv head
  PaCut cut;             // of few rows
  float scale_log2;
};

__host__ __device__ inline int pa_div_up(int64_t a, int b) { return (int)((a + b - 1) / b); }

// Blocks of 2^lb keys that a tile of `rows` rows sees at most of `len` positions.
__host__ __device__ inline int pa_blocks(int len, int rows, int window, int sinks, int lb) {
  auto up = [lb](uint32_t x) { return (int)((x + (1u << lb) - 1) >> lb); };
  const int all = up(len);
  if (!window) return all;
  const int some = up(sinks) + up((uint32_t)window + rows - 1) + 1;
  return some < all ? some : all;
}

// Blocks per part of many rows, the least number that leaves a sequence of `tiles` tiles of
// `blocks` blocks at most the target's parts.
__host__ __device__ inline int pa_part(int tiles, int blocks, int Hkv) {
  const int wide = tiles * Hkv;  // with many of them a part saves less than its merge costs
  const int more = wide >= 96 ? 4 : (wide >= 64 ? 2 : 1);
  const int least = more * kPaManyMinPart / kPaManyBlock;
  const int64_t p = ((int64_t)blocks * Hkv * tiles + kPaManyTarget - 1) >> kPaManyLogTarget;
  return (int)(p < least ? least : (p < (1 << 29) ? p : 1 << 29));
}
__host__ __device__ inline int pa_parts(int blocks, int part) {  // of a list of blocks
  return (int)(((uint32_t)blocks + (uint32_t)part - 1) / (uint32_t)part);
}

// Parts that a tile of `rows` rows sees at most of `len` positions.
__host__ __device__ inline int pa_most_parts(PaCut cut, int len, int rows, int window, int sinks) {
  if (len <= 0) return 1;
  const int all = cut.of((len - 1) >> kPaLogBlock) + 1;
  if (!window) return all;
  const int ls = cut.near && kPaLogNear < cut.lf ? kPaLogNear : cut.lf;
  const int run = (int)(((uint32_t)window + rows - 1 + kPaBlock - 1) >> kPaLogBlock) + 1;  // blocks in a row
  const int some = (sinks ? cut.of((sinks - 1) >> kPaLogBlock) + 1 : 0) + ((run - 2 + (1 << ls)) >> ls) + 1;
  return some < all ? some : all;
}

struct PaSeq {
  int b, q0, nq, ne;  // the sequence, its first row, its rows, those within the bound
  int pos0;           // the first row's position
  bool many;
  int tiles;
  int part;           // many: blocks per part of a tile
  PaCut cut;          // otherwise: of the sequence
  int parts;          // at most, of a tile
};

template <typename T>
__device__ __forceinline__ PaSeq pa_seq(const PaArgs& a, int b, int c0, int c1, int kv) {
  PaSeq s;
  s.b = b;
  s.q0 = c0;
  s.nq = min(c1, a.n) - c0;
  kv = max(kv, 0);
  s.pos0 = kv - (c1 - c0);
  s.ne = min(max(s.nq, 0), a.qmax);
  const bool large = s.ne * a.G > a.few_pairs;
  s.many = sizeof(T) == 2 && large;
  const int rows = s.many ? a.many_tile : a.few_tile, len = min(kv, a.kmax);
  s.tiles = s.ne <= rows ? min(s.ne, 1) : (int)((uint32_t)(s.ne - 1) / (uint32_t)rows) + 1;
  s.cut = a.cut;
  if (s.many) {
    const int blocks = pa_blocks(len, rows, a.window, a.sinks, kPaManyLogBlock);
    s.part = pa_part(s.tiles, blocks, a.Hkv);
    s.parts = max(pa_parts(blocks, s.part), 1);
    return s;
  }
  s.part = 0;
  if (sizeof(T) == 4 && large) {
    const int wide = s.tiles * a.Hkv;
    const int blocks = pa_blocks(len, rows, a.window, a.sinks, kPaLogBlock);
    const int p = wide >= kPaTarget ? 1 << 26 : max((int)(((uint32_t)blocks * wide + kPaTarget - 1) / kPaTarget), kPaMinPart / kPaBlock);
    s.cut = PaCut{0, 32 - __builtin_clz((unsigned)(p - 1))};
  }
  s.parts = pa_most_parts(s.cut, len, rows, a.window, a.sinks);
  if (a.window && len > 0) {  // uniform; the parts from the first row's window on, and the sinks'
    const int lo = max(max(s.pos0, 0) - a.window + 1, 0) >> kPaLogBlock;
    const int some = (a.sinks ? s.cut.of((a.sinks - 1) >> kPaLogBlock) + 1 : 0) +
                     max(s.cut.of((len - 1) >> kPaLogBlock) - s.cut.of(lo), 0) + 1;
    s.parts = min(s.parts, some);
  }
  return s;
}

// A tile of rows, and its visible blocks: those with sinks, and a run to its last row. Of many
// rows they are a list that is cut into parts; of few the parts are those of the sequence that
// hold any.
struct PaTile {
  int i0, nr;       // its first row in the sequence and the number of its pairs
  int pmin, pmax;   // first and last position, the last below kmax
  int ns, first, nt;  // blocks with sinks, the first block of the run, blocks in all
  int in0, in1;     // the blocks [in0, in1) that every row sees whole: many, of the list; few, of the sequence
  int sink_parts, first_part;  // few: parts with sinks, the run's first other part
  int parts;        // one at least
};

template <bool MANY>
__device__ __forceinline__ PaTile pa_tile(const PaArgs& a, const PaSeq& s, int tile) {
  constexpr int BLOCK = MANY ? kPaManyBlock : kPaBlock;
  const int rows = MANY ? a.many_tile : a.few_tile;
  PaTile t;
  t.i0 = tile * rows;
  const int count = min(s.ne - t.i0, rows);
  t.nr = count * a.G;
  t.pmin = s.pos0 + t.i0;
  t.pmax = min(t.pmin + count - 1, a.kmax - 1);
  t.ns = t.first = t.nt = t.in0 = t.in1 = t.sink_parts = t.first_part = 0;
  t.parts = 1;
  if (count <= 0 || t.pmax < 0) return t;
  const int lo = a.window ? max(max(t.pmin, 0) - a.window + 1, 0) : 0;
  t.ns = (min(a.sinks, lo) + BLOCK - 1) / BLOCK;
  t.first = max(min(lo, t.pmax) / BLOCK, t.ns);
  t.nt = t.ns + t.pmax / BLOCK + 1 - t.first;
  t.in0 = max(a.window ? max(t.pmax - a.window + BLOCK, 0) / BLOCK : 0, t.first);
  t.in1 = t.pmin + 1 > 0 ? (t.pmin + 1) / BLOCK : 0;
  if constexpr (MANY) {
    t.in0 += t.ns - t.first;
    t.in1 += t.ns - t.first;
    t.parts = pa_parts(t.nt, s.part);
  } else {
    t.sink_parts = t.ns ? s.cut.of(t.ns - 1) + 1 : 0;
    t.first_part = max(s.cut.of(t.first), t.sink_parts);
    t.parts = t.sink_parts + max(s.cut.of(t.pmax / BLOCK) - t.first_part + 1, 0);
  }
  return t;
}

// A wave's blocks of a part of few rows: every fourth of the sequence, `lead` of them with sinks.
struct PaBlocks {
  int sink, lead, run, count;
  __device__ __forceinline__ int at(int i) const { return i < lead ? sink + 4 * i : run + 4 * (i - lead); }
};
__device__ __forceinline__ PaBlocks pa_wave_blocks(const PaSeq& s, const PaTile& t, int part, int wave) {
  static_assert(kPaWaves == 4 && kPaLogNear >= 2 && kPaMinPart / kPaBlock >= 4, "a part's first block is wave 0's");
  const int q = part < t.sink_parts ? part : part - t.sink_parts + t.first_part;
  const int b0 = s.cut.start(q), b1 = s.cut.start(q + 1);
  PaBlocks w;
  w.sink = b0 + wave;
  w.lead = max((min(b1, t.ns) - w.sink + 3) >> 2, 0);
  const int from = max(b0, t.first);
  w.run = from + ((wave - from) & 3);
  w.count = w.lead + (t.nt > 0 ? max((min(b1, t.pmax / kPaBlock + 1) - w.run + 3) >> 2, 0) : 0);
  return w;
}

// The slot of part 0 of row q0 + i, head h.
__device__ __forceinline__ int64_t pa_slot(const PaArgs& a, const PaSeq& s, int i, int h) {
  if (a.seq_slots) return s.b * a.seq_slots + ((int64_t)i * a.H + h) * s.parts;
  return ((int64_t)(s.q0 + i) * a.H + h) * a.row_per;
}

// The sequence of unit u among the sequences' units(s), and the unit within it; false
// past the last. Wave-wide, 64 sequences a step.
template <typename T, typename F>
__device__ __forceinline__ bool pa_find(const PaArgs& a, uint32_t u, F units, PaSeq& s, int& local) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < a.nseq; b0 += 64) {  // uniform
    const int b = min(b0 + lane, a.nseq - 1);
    const int c0 = a.cu_q[b], c1 = a.cu_q[b + 1], kv = a.kv_len[b];
    const PaSeq t = pa_seq<T>(a, b, c0, c1, kv);
    // the host keeps a launch's sum below 2^31
    const uint32_t sum = wave_scan_add(b0 + lane < a.nseq && t.nq > 0 ? (uint32_t)units(t) : 0u);
    const int at = __popcll(__ballot(sum <= u));  // ascending: so many are before u's sequence
    if (at < 64) {
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      s = pa_seq<T>(a, b0 + at, of(c0), of(c1), of(kv));
      local = (int)(u - (at ? (uint32_t)__builtin_amdgcn_readlane((int)sum, at - 1) : 0u));
      return true;
    }
    u -= (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return false;
}

// The item of workgroup unit u of the few- or many-row kernel: a part of a tile. False
// past the last; a unit may be a part that its tile does not have.
template <typename T, bool MANY>
__device__ __forceinline__ bool pa_item(const PaArgs& a, uint32_t u, PaSeq& s, PaTile& t, int& part, bool& first) {
  int local;
  if (!pa_find<T>(a, u, [](const PaSeq& q) { return q.many == MANY ? max(q.tiles, 1) * q.parts : 0; }, s, local))
    return false;
  first = local == 0;
  int tile = 0;
  if (s.tiles > 1) {  // uniform
    tile = s.parts > 1 ? (int)((uint32_t)local / (uint32_t)s.parts) : local;
    local -= tile * s.parts;
  }
  part = local;
  t = pa_tile<MANY>(a, s, MANY ? max(s.tiles - 1 - tile, 0) : tile);  // many: the last tiles, which see most, first
  return true;
}

__device__ __forceinline__ bool pa_sees(const PaArgs& a, int key, int pos) {
  return key <= pos && (!a.window || pos - key < a.window || key < a.sinks);
}

// Rows past q_len_max are NaN; the sequence's first item writes them for its kv head.
template <typename T, int DH>
__device__ __forceinline__ void pa_rows_past(const PaArgs& a, const PaSeq& s, int g) {
  for (int p = threadIdx.x / DH; p < (s.nq - s.ne) * a.G; p += 64 * kPaWaves / DH) {
    const int i = p / a.G;
    Elem<T>::store((T*)a.out + ((int64_t)(s.q0 + s.ne + i) * a.H + g * a.G + p - i * a.G) * DH + threadIdx.x % DH, NAN);
  }
}

// What a row at position pos gets for O / L.
__device__ __forceinline__ float pa_finish(const PaArgs& a, int pos, float o, float l) {
  return pos < 0 ? 0.f : (pos >= a.kmax ? NAN : o / l);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 pa_mfma32(const u32x4& x, const u32x4& y, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), acc, 0,
                                                 0, 0);
}

// The scale's size; zero is a tiny one, under which -inf stays -inf, and NaN is NaN.
__device__ __forceinline__ float pa_scale(const PaArgs& a) {
  return a.scale_log2 != a.scale_log2 ? a.scale_log2 : fmaxf(fabsf(a.scale_log2), 1e-37f);
}

// A negative scale's sign goes to q. (Not as q is loaded: that would wait for it there.)
template <int N>
__device__ __forceinline__ void pa_flip(u32x4 (&q)[N], uint32_t flip) {
  if (flip) {  // uniform
#pragma unroll
    for (int k = 0; k < N; ++k) q[k] ^= flip;
  }
}

// Largest / sum of a lane's and lane ^ 32's values, in both.
__device__ __forceinline__ float pa_max_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float pa_add_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// A block's scores (of the lane's pair) to probabilities, under the pair's reference
// point: the maximum when it was last moved, which is when a block exceeds it by more
// than 2^8. Probabilities up to 2^8 lose nothing in fp32 sums or bf16, and most blocks
// rescale nothing. It depends on the pair's own scores only.
template <int NB, int NDB>
__device__ __forceinline__ void pa_softmax(f32x16 (&sc)[NB], f32x16 (&o)[NDB], float& mref, float& lrun, float scale) {
  float mt = -INFINITY;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, sc[b][r]);
  mt = pa_max_halves(mt) * scale;
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
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      sc[b][r] = __builtin_amdgcn_exp2f(fmaf(sc[b][r], scale, -ref));
      lt += sc[b][r];
    }
  lrun += lt;  // of this lane half's keys
}

// A probability of 0 times an infinity or a NaN in V would be a NaN, also in a row that
// does not see the key. Blocks that some row sees and another does not are therefore
// looked through as they are staged: what is not finite is replaced by 0, and the rows
// that see it get it added afterwards, from the page. (Blocks that all rows see need
// none of this.)
__device__ __forceinline__ bool pa_clean(u32x4& v) {  // 8 bf16; were any not finite?
  uint32_t odd = 0;  // an exponent of ones carries into its sign's place
#pragma unroll
  for (int e = 0; e < 4; ++e) odd |= (v[e] & 0x7f807f80u) + 0x00800080u;
  if (!(odd & 0x80008000u)) return false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((v[e] & 0x7f80u) == 0x7f80u) v[e] &= 0xffff0000u;
    if ((v[e] & 0x7f800000u) == 0x7f800000u) v[e] &= 0xffffu;
  }
  return true;
}

// The keys k0 + bit of `odd` (uniform) to the rows that see them: lane (col, hf) holds
// pair col's columns 32 db + 8 (r / 4) + 4 hf + r % 4.
template <typename T, int DH>
__device__ __forceinline__ void pa_add_odd(const PaArgs& a, const PaSeq& s, const PaTile& t, uint64_t odd, int k0,
                                           int64_t head, int pos, int hf, f32x16 (&o)[DH / 32]) {
#pragma unroll 1
  for (; odd; odd &= odd - 1) {
    const int key = k0 + __builtin_ctzll(odd);
    if (key > t.pmax) return;
    const bool see = pa_sees(a, key, pos);
    const uint32_t page = (uint32_t)a.m.table[(int64_t)s.b * a.m.ld + (key >> a.m.log2_rows)];
    if (page >= a.m.pages) continue;  // its scores are NaN
    const T* row = (const T*)a.vp + page * a.m.page_els + head +
                   (int64_t)(key & ((1 << a.m.log2_rows) - 1)) * a.m.row_els + 4 * hf;
#pragma unroll
    for (int db = 0; db < DH / 32; ++db) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = Elem<T>::load(row + 32 * db + 8 * i + e);
          if (see && x - x != 0.f) o[db][4 * i + e] += x;
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// What is added to the scores of 16-key group `group`: its page may be none of the pool.
__device__ __forceinline__ float pa_bad(int bad, int group) { return bad >> group & 1 ? NAN : 0.f; }

// What a block's 64 keys from k0 on (fewer of them in use) are to the lane's row: scores of
// those that it does not see become -inf. place(b, r): register r of product b is key
// k0 + lead + place. The keys are bits of a word, two instructions a score.
__device__ __forceinline__ uint64_t pa_keys_to(int x) {  // bits 0 .. x
  return x < 0 ? 0 : ~0ull >> (63 - min(x, 63));
}
__device__ __forceinline__ uint64_t pa_hidden(const PaArgs& a, int pos, int k0, int lead) {
  const int last = max(pos, -1) - k0;
  uint64_t see = pa_keys_to(last);
  if (a.window) see &= ~pa_keys_to(max(last, -1) - a.window) | pa_keys_to(a.sinks - k0 - 1);  // uniform
  return ~see >> lead;
}
template <int NB, typename F>
__device__ __forceinline__ void pa_hide(const PaArgs& a, f32x16 (&sc)[NB], int pos, int k0, int lead, F place) {
  const uint64_t hidden = pa_hidden(a, pos, k0, lead);
  uint32_t word[2] = {(uint32_t)hidden, (uint32_t)(hidden >> 32)};
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      uint32_t hide;  // written in C it becomes three instructions
      asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(hide) : "v"(word[place(b, r) >> 5]), "i"(place(b, r) & 31));
      sc[b][r] = __uint_as_float((hide & 0xff800000u) | (~hide & __float_as_uint(sc[b][r])));
    }
}

__device__ __forceinline__ void pa_wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where a wave's blocks are: lane l has 16-key group l of its next 64 / GPB blocks (GPB groups
// each; block(i) is the number of the i-th), as the byte offset of its first row from the
// pool's start. A group past the tile's last key counts as that key's, one in no page of the
// pool as page 0's.
struct PaPages {
  uint32_t lo, hi;
  uint64_t bad;  // groups in no page
  __device__ __forceinline__ const char* at(const void* pool, int group) const {  // uniform
    const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, group) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)lo, group);
    return (const char*)pool + o;
  }
};
template <typename T, int BLOCK, typename F>
__device__ __forceinline__ PaPages pa_pages(const PaArgs& a, const PaSeq& s, const PaTile& t, int64_t head, F block) {
  constexpr int GPB = BLOCK / 16;
  const int lane = threadIdx.x & 63;
  const int blk = min(block(lane / GPB), t.pmax / BLOCK);
  const int key = min(blk * BLOCK + 16 * (lane % GPB), t.pmax & ~15);
  const uint32_t id = (uint32_t)a.m.table[(int64_t)s.b * a.m.ld + (key >> a.m.log2_rows)];
  const bool bad = id >= a.m.pages;
  const uint64_t at = sizeof(T) * ((uint64_t)(bad ? 0 : id) * a.m.page_els + head +
                                   (uint64_t)(key & ((1 << a.m.log2_rows) - 1)) * a.m.row_els);
  PaPages p;
  p.lo = (uint32_t)at;
  p.hi = (uint32_t)(at >> 32);
  p.bad = __ballot(bad);
  return p;
}

// The last row that may be read of a group of a block: those past the tile's last key are that key's.
template <int BLOCK>
__device__ __forceinline__ int pa_last_row(const PaTile& t, bool last_block, int group) {
  const int last = t.pmax % BLOCK - 16 * group;
  return !last_block || last > 15 ? 15 : (last < 0 ? t.pmax & 15 : last);
}

// The transposed fragment of V from rows at a lane's place in a row-major block of LDS, rows VP elements apart.
template <int VP>
__device__ __forceinline__ u32x4 pa_vt_frag(const bf16_t* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  typedef const __attribute__((address_space(3))) void* lds_ptr;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_ptr)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_ptr)(p + 4 * VP));
  const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
  return u32x4{x.x, x.y, y.x, y.y};
}

// The workgroup's key streams, one per wave, merged: to the rows themselves, or as a
// part. o_lds [wave][pair][DH, pitch OP], m / l [wave][pair]. A thread first has one
// pair's weights and place, then takes four columns of a pair at a time.
template <typename T, int DH, int OP>
__device__ __forceinline__ void pa_leave(const PaArgs& a, const PaSeq& s, const PaTile& t, int g, int np, int part,
                                         const float* o_lds, const float* m_lds, float* l_lds, int64_t* at_lds,
                                         float* fin_lds) {
  constexpr int RT = kPaRows;
  if (threadIdx.x < t.nr) {
    const int r = threadIdx.x, j = r * a.g_magic >> 16, i = t.i0 + j, h = g * a.G + (r - j * a.G);
    float M = -INFINITY, L = 0.f, f[kPaWaves];
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) M = fmaxf(M, m_lds[w * RT + r]);
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) {
      const float mw = m_lds[w * RT + r];
      f[w] = mw == -INFINITY ? 0.f : exp2f(mw - M);
      L = fmaf(l_lds[w * RT + r], f[w], L);
    }
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) l_lds[w * RT + r] = f[w];
    if (np > 1) {
      const int64_t at = pa_slot(a, s, i, h) + part;
      a.pml[2 * at] = M;
      a.pml[2 * at + 1] = L;
      at_lds[r] = at;
    } else {
      at_lds[r] = (int64_t)(s.q0 + i) * a.H + h;
      fin_lds[r] = L;
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < t.nr * (DH / 4); idx += 64 * kPaWaves) {
    const int r = idx / (DH / 4), d = 4 * (idx % (DH / 4));
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) {
      const float f = l_lds[w * RT + r];
      const f32x4 ow = *reinterpret_cast<const f32x4*>(o_lds + (w * RT + r) * OP + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(ow[e], f, O[e]);
    }
    if (np > 1) {
      *reinterpret_cast<f32x4*>(a.po + at_lds[r] * DH + d) = O;
    } else {
      const int pos = t.pmin + (r * a.g_magic >> 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = pa_finish(a, pos, O[e], fin_lds[r]);
      T* out = (T*)a.out + at_lds[r] * DH + d;
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(out) = uint2{f32x2_to_bf16x2_bits(O[0], O[1]), f32x2_to_bf16x2_bits(O[2], O[3])};
      else
        *reinterpret_cast<f32x4*>(out) = O;
    }
  }
}

// A wave's stream to LDS for the merge: lane (col, hf) holds pair col's columns
// 32 db + 8 (r / 4) + 4 hf + r % 4.
template <int DH, int OP>
__device__ __forceinline__ void pa_keep(int nr, int wave, int col, int hf, const f32x16 (&o)[DH / 32], float mref,
                                        float lrun, float* o_lds, float* m_lds, float* l_lds) {
  if (col < nr) {
#pragma unroll
    for (int db = 0; db < DH / 32; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(o_lds + (wave * kPaRows + col) * OP + 32 * db + 8 * r + 4 * hf) =
            f32x4{o[db][4 * r], o[db][4 * r + 1], o[db][4 * r + 2], o[db][4 * r + 3]};
  }
  lrun = pa_add_halves(lrun);
  if (col < nr && hf == 0) {
    m_lds[wave * kPaRows + col] = mref;
    l_lds[wave * kPaRows + col] = lrun;
  }
}

// The block at a place of a tile's list.
__device__ __forceinline__ int pa_listed(const PaTile& t, int c) { return c < t.ns ? c : c - t.ns + t.first; }

// bf16, few rows: bound by the keys and values, each read once per tile of 32 pairs (64 rows of
// 4 heads x 4 over 32700 keys 765 us, 5.6 TB/s; 112 rows of 16 heads over 127 to 1199 keys 124
// us, 4.9 TB/s), and for few short sequences by a chain of launch, search, page numbers, keys,
// merge and, where any row may have more than 512 keys, a second launch that merges the parts
// (8 rows over 511 to 777 keys 18.6 us, 3.9 of them the second launch).
// Up to 32 pairs per workgroup, one per column of the 32x32x16 MFMA, and
// four waves that each stream 32-key blocks (pa_wave_blocks) through LDS of their own: whole rows to registers a block ahead, to LDS as loaded,
// no workgroup barrier before the merge. A wave computes S^T = K Q^T and O^T = V^T P^T;
// the K rows of a block are taken in the order that makes a lane's S^T registers the 8
// consecutive keys its P^T operand wants (result register r of lane half hf is key
// 16 (r / 8) + 8 hf + r % 8), so P never leaves its lane, and V^T comes out of the
// row-major block by transposing LDS reads.
template <int DH>
struct PaFewLds {
  static constexpr int KP = DH + 8;   // row pitches: K reads 16 bytes of 32 rows, V^T 64 bytes of 8 rows,
  static constexpr int VP = DH + 32;  // each spread over all banks
  static constexpr int OP = DH + 4;
  static constexpr int kWaveEls = kPaBlock * (KP + VP);
  union {
    bf16_t block[kPaWaves][kWaveEls];
    float o[kPaWaves * kPaRows * OP];  // of the merge, as what follows
  };
};
struct PaMergeLds {
  float m[kPaWaves * kPaRows];
  float l[kPaWaves * kPaRows];
  int64_t at[kPaRows];
  float fin[kPaRows];
};
// workgroup `wg` of `wgs` of a kv head
template <int DH>
__device__ __forceinline__ void pa_few_bf16(const PaArgs& a, PaFewLds<DH>& lds, PaMergeLds& merge, uint32_t wg,
                                            uint32_t wgs) {
  constexpr int TK = kPaBlock;
  constexpr int NDS = DH / 16;
  constexpr int NDB = DH / 32;
  constexpr int KP = PaFewLds<DH>::KP, VP = PaFewLds<DH>::VP, OP = PaFewLds<DH>::OP;
  constexpr int CPR = DH / 8;   // 16-byte pieces per row
  constexpr int RPI = 64 / CPR;
  constexpr int NLD = TK / RPI;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 31, hf = lane >> 5;
  bf16_t* k_lds = lds.block[wave];
  bf16_t* v_lds = k_lds + TK * KP;
  const float scale = pa_scale(a);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  const int lr = lane / CPR, lp = lane % CPR;  // row within a load, piece
  const uint32_t rsb = (uint32_t)a.m.row_els * sizeof(bf16_t);
  const int krow = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
  const int tg = lane >> 4, ti = lane & 15;
  const int v_lane = ((tg >> 1) * 8 + (ti >> 2)) * VP + 16 * (tg & 1) + 4 * (ti & 3);
  auto vt_frag = [&](int db, int s) { return pa_vt_frag<VP>(v_lds + v_lane + 16 * s * VP + 32 * db); };
  const int g = blockIdx.x;
  const int64_t head = g * a.m.head_els;

  for (uint32_t u = wg;; u += wgs) {  // uniform
    PaSeq s;
    PaTile t;
    int part;
    bool first;
    if (!pa_item<bf16_t, false>(a, u, s, t, part, first)) return;
    if (first && s.ne < s.nq) pa_rows_past<bf16_t, DH>(a, s, g);
    if (t.nr <= 0 || part >= t.parts) continue;
    const PaBlocks mine = pa_wave_blocks(s, t, part, wave);

    u32x4 kreg[NLD], vreg[NLD];
    PaPages pages;
    int bad = 0;
    auto fetch = [&](int c) {
      const int i = c & 31;
      if (i == 0) pages = pa_pages<bf16_t, TK>(a, s, t, head, [&](int x) { return mine.at(c + x); });
      const bool end = mine.at(c) == t.pmax / TK;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char *kb = pages.at(a.kp, 2 * i + h), *vb = pages.at(a.vp, 2 * i + h);
        const int last = pa_last_row<TK>(t, end, h);
#pragma unroll
        for (int e = 0; e < NLD / 2; ++e) {
          const uint32_t off = __umul24((uint32_t)min(RPI * e + lr, last), rsb) + (uint32_t)lp * 16u;
          kreg[h * (NLD / 2) + e] = ld16(kb + off);
          vreg[h * (NLD / 2) + e] = ld16(vb + off);
        }
      }
      bad = (int)(pages.bad >> (2 * i) & 3);
    };
    const int pr = min(col, t.nr - 1), qi = pr * a.g_magic >> 16;
    const int qpos = t.pmin + qi;
    u32x4 qf[NDS];
    {
      const bf16_t* qp = (const bf16_t*)a.q +
                         ((int64_t)(s.q0 + t.i0 + qi) * a.H + g * a.G + (pr - qi * a.G)) * DH + 8 * hf;
#pragma unroll
      for (int k = 0; k < NDS; ++k) qf[k] = ld16(qp + 16 * k);
    }
    if (mine.count > 0) fetch(0);
    pa_flip(qf, flip);
    float mref = -INFINITY, lrun = 0.f;
    f32x16 o[NDB];
#pragma unroll
    for (int c = 0; c < NDB; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[c][r] = 0.f;

    for (int c = 0; c < mine.count; ++c) {  // uniform over the wave
      const int blk = mine.at(c), k0 = blk * TK;
      const bool all = blk >= t.in0 && blk < t.in1;
      uint32_t odd = 0;  // keys whose V is not finite
      if (!all) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
          const uint64_t b = __builtin_amdgcn_ballot_w64(pa_clean(vreg[i]));
          if (b) {
#pragma unroll
            for (int r = 0; r < RPI; ++r)
              odd |= (b >> (CPR * r) & ((1ull << CPR) - 1) ? 1u : 0u) << (RPI * i + r);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        *reinterpret_cast<u32x4*>(k_lds + (RPI * i + lr) * KP + 8 * lp) = kreg[i];
        *reinterpret_cast<u32x4*>(v_lds + (RPI * i + lr) * VP + 8 * lp) = vreg[i];
      }
      const int bad_now = bad;
      if (c + 1 < mine.count) fetch(c + 1);
      pa_wave_fence();
      f32x16 sc[1];
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[0][r] = 0.f;
#pragma unroll
      for (int k = 0; k < NDS; ++k)
        sc[0] = pa_mfma32(*reinterpret_cast<const u32x4*>(k_lds + krow * KP + 16 * k + 8 * hf), qf[k], sc[0]);
      if (bad_now) {  // uniform
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[0][r] += pa_bad(bad_now, r >> 3);
      }
      if (!all) pa_hide(a, sc, qpos, k0, 8 * hf, [](int, int r) { return 16 * (r >> 3) + (r & 7); });  // uniform
      pa_softmax<1, NDB>(sc, o, mref, lrun, scale);
      // P meets V in two bf16 terms, half a step of 2^-15 of it: these rows are bound by the
      // loads. The first is cut off below P, so that both have its sign and an infinity in V
      // is itself.
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = sc[0][8 * k + 2 * e], y1 = sc[0][8 * k + 2 * e + 1];
          const uint32_t b0 = __float_as_uint(y0 * 0.998046875f), b1 = __float_as_uint(y1 * 0.998046875f);
          hi[e] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
          lo[e] = f32x2_to_bf16x2_bits(y0 - __uint_as_float(b0 & 0xffff0000u), y1 - __uint_as_float(b1 & 0xffff0000u));
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const u32x4 vf = vt_frag(db, k);
          o[db] = pa_mfma32(vf, lo, o[db]);
          o[db] = pa_mfma32(vf, hi, o[db]);
        }
      }
      if (odd) pa_add_odd<bf16_t, DH>(a, s, t, odd, k0, head, qpos, hf, o);
      pa_wave_fence();  // the next block overwrites this one
    }
    __syncthreads();  // every wave's blocks are done: the merge takes their LDS
    pa_keep<DH, OP>(t.nr, wave, col, hf, o, mref, lrun, lds.o, merge.m, merge.l);
    __syncthreads();
    pa_leave<bf16_t, DH, OP>(a, s, t, g, t.parts, part, lds.o, merge.m, merge.l, merge.at, merge.fin);
    __syncthreads();  // the next item's blocks take it again
  }
}

template <int DH>
__global__ __launch_bounds__(64 * kPaWaves) __attribute__((amdgpu_waves_per_eu(2))) void attn_paged_few_bf16(PaArgs a) {
  __shared__ __align__(16) PaFewLds<DH> lds;
  __shared__ PaMergeLds merge;
  pa_few_bf16<DH>(a, lds, merge, blockIdx.y, gridDim.y);
}

// fp32, all rows: the same on the 16x16x4 MFMA, with one column tile for up to 16 pairs and
// two for up to 32. Lane (i, kg) = (lane % 16, lane / 16) holds columns 16 j + 4 kg + e of its
// operands of K Q^T at step 4 j + e; its S^T register r of 16-key group h is key 16 h + 4 kg + r,
// which is also the key it supplies of P^T at step 4 h + r. The rows of V^T are taken in the
// order that makes a lane's 16-byte load of V its operand of four products (dimensions 64 q + 4 i
// + e), and its O^T registers are then dimensions 64 q + 16 kg + 4 r + e. V comes straight from
// its page, asked for before the scores; K goes straight to LDS, the next block's once the
// scores are done, its 16-byte pieces of row r exchanged (piece p at p ^ r % 16) so that a
// column of them is spread over all banks.
// Bound by the keys and values where there are enough of them (64 rows of 16 heads of 128 over
// 1000 to 4000 keys, 4 kv heads, 156 us, 131 at a copy's rate), by two trips to memory a block,
// K's and then V's, where a wave has few blocks: 127 rows of 33 sequences, 4 heads of 64 over 40
// to 2000 keys, 24.5 us (70 MB: 14), 4 of them the merge. On the 32x32x2 MFMA, K through
// registers and V in pieces of 4 bytes, 31 and 287.
template <int DH>
struct PaF32Lds {
  static constexpr int OP = DH + 4;
  union {
    float k[kPaWaves][kPaBlock * DH];
    float o[kPaWaves * kPaRows * OP];  // of the merge
  };
};
__device__ __forceinline__ float pa_max_groups(float x) {  // over a lane's i
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pa_max_halves(fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])));
}
__device__ __forceinline__ float pa_add_groups(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pa_add_halves(__uint_as_float(p[0]) + __uint_as_float(p[1]));
}

// x, but what follows from it is not kept in registers across the blocks.
__device__ __forceinline__ uint32_t pa_here(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A lane's 16 bytes of global memory (uniform base, lane offset) straight to LDS, at the
// wave's `to` + 16 times the lane. M0 holds the LDS address; one wait state separates its
// write from the load. In assembly, so that the compiler, which would put a wait for all
// loads before LDS reads, leaves the waits to where they are written.
__device__ __forceinline__ void pa_load_lds(const char* base, uint32_t off, const void* to) {
  const uint32_t m0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0), "v"(off), "s"(base)
               : "memory", "m0");
}

template <int DH, int NT>
__device__ __forceinline__ void pa_f32_part(const PaArgs& a, const PaSeq& s, const PaTile& t, int g, int part,
                                            PaF32Lds<DH>& lds, PaMergeLds& merge) {
  constexpr int TK = kPaBlock;
  constexpr int NJ = DH / 16;
  constexpr int NQ = DH / 64;
  constexpr int RB = DH * 4;    // bytes per row
  constexpr int CPR = DH / 4;   // 16-byte pieces per row
  constexpr int RPI = 64 / CPR;
  constexpr int NLD = TK / RPI;
  constexpr int OP = PaF32Lds<DH>::OP;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, i16 = lane & 15, kg = lane >> 4;
  float* k_lds = lds.k[wave];
  const float scale = pa_scale(a);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80000000u : 0u;
  const int lr = lane / CPR, lp = lane % CPR;  // row within a load of K, place in it
  const uint32_t piece = 16u * (lp ^ lr);      // that goes there, of load i this ^ 16 times its first row % 16
  const uint32_t k_lane = (uint32_t)(i16 * RB + 16 * (kg ^ i16));
  const uint32_t rsb = (uint32_t)a.m.row_els * sizeof(float);
  const int64_t head = g * a.m.head_els;
  const PaBlocks mine = pa_wave_blocks(s, t, part, wave);

  PaPages pages;
  int next = 0, bad = 0;
  int last[2];  // the last row to read of either group
  auto find = [&](int c) {
    next = c & 31;
    if (next == 0) pages = pa_pages<float, TK>(a, s, t, head, [&](int x) { return mine.at(c + x); });
    const bool end = mine.at(c) == t.pmax / TK;
    last[0] = pa_last_row<TK>(t, end, 0);
    last[1] = pa_last_row<TK>(t, end, 1);
    bad = (int)(pages.bad >> (2 * next) & 3);
  };
  auto fetch_k = [&]() {
    const uint32_t pc = pa_here(piece), r0 = pa_here(lr);
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const uint32_t row = min((RPI * i & 15) + r0, (uint32_t)last[i / (NLD / 2)]);
      pa_load_lds(pages.at(a.kp, 2 * next + i / (NLD / 2)), __umul24(row, rsb) + (pc ^ 16u * (RPI * i & 15)),
                  k_lds + RPI * i * DH);
    }
  };
  int qpos[NT];
  u32x4 qf[NT][NJ];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int pr = min(16 * n + i16, t.nr - 1), qi = pr * a.g_magic >> 16;
    qpos[n] = t.pmin + qi;
    const float* qp = (const float*)a.q + ((int64_t)(s.q0 + t.i0 + qi) * a.H + g * a.G + (pr - qi * a.G)) * DH + 4 * kg;
#pragma unroll
    for (int j = 0; j < NJ; ++j) qf[n][j] = ld16(qp + 16 * j);
  }
  if (mine.count > 0) {
    find(0);
    fetch_k();
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) pa_flip(qf[n], flip);
  float mref[NT], lrun[NT];
  f32x4 o[NT][NQ][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    mref[n] = -INFINITY;
    lrun[n] = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][q][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  for (int c = 0; c < mine.count; ++c) {  // uniform over the wave
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // K is there
    f32x4 v[8][NQ];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const char* vb = pages.at(a.vp, 2 * next + k / 4);
      const uint32_t off = __umul24((uint32_t)min(4 * kg + (k & 3), last[k / 4]), rsb) + 16u * i16;
#pragma unroll
      for (int q = 0; q < NQ; ++q) v[k][q] = *reinterpret_cast<const f32x4*>(vb + off + 256 * q);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int bad_now = bad;
    const uint32_t k_at = pa_here(k_lane);
    f32x4 kf[2][2];
    auto read_k = [&](int j) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        kf[j & 1][h] = *reinterpret_cast<const f32x4*>((const char*)k_lds + (k_at ^ 64 * j) + 16 * h * RB);
    };
    read_k(0);
    f32x4 sc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) sc[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (j + 1 < NJ) read_k(j + 1);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            sc[n][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j & 1][h][e], __uint_as_float(qf[n][j][e]), sc[n][h], 0,
                                                            0, 0);
    }
    const int blk = mine.at(c), k0 = blk * TK;
    const bool all = blk >= t.in0 && blk < t.in1;
    if (bad_now) {  // uniform
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) sc[n][h] += pa_bad(bad_now, h);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (!all) {  // uniform
        const uint32_t hidden = (uint32_t)pa_hidden(a, qpos[n], k0, 4 * kg);
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (hidden >> (16 * (x / 4) + x % 4) & 1) sc[n][x / 4][x % 4] = -INFINITY;
      }
      float mt = -INFINITY;
#pragma unroll
      for (int x = 0; x < 8; ++x) mt = fmaxf(mt, sc[n][x / 4][x % 4]);
      mt = pa_max_groups(mt) * scale;
      if (__builtin_amdgcn_ballot_w64(mt > mref[n] + 8.f)) {  // as in pa_softmax
        const float mnew = mt > mref[n] + 8.f ? mt : mref[n];
        const float corr = mref[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref[n] - mnew);
        mref[n] = mnew;
        lrun[n] *= corr;
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][q][e] *= corr;
      }
      const float ref = mref[n] == -INFINITY ? 0.f : mref[n];
      float lt = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float p = __builtin_amdgcn_exp2f(fmaf(sc[n][x / 4][x % 4], scale, -ref));
        sc[n][x / 4][x % 4] = p;
        lt += p;
      }
      lrun[n] += lt;  // of this lane's keys
    }
    uint32_t odd = 0;  // keys whose V is not finite
    if (!all) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        bool any = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool x = v[k][q][e] - v[k][q][e] != 0.f;
            any |= x;
            v[k][q][e] = x ? 0.f : v[k][q][e];
          }
        const uint64_t b = __builtin_amdgcn_ballot_w64(any);
        if (b) {  // uniform
#pragma unroll
          for (int x = 0; x < 4; ++x) odd |= (b >> 16 * x & 0xffff ? 1u : 0u) << (16 * (k / 4) + 4 * x + k % 4);
        }
      }
    }
    // V is there before the next loads go out, or each of its uses would wait for these too
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int q = 0; q < NQ; ++q) asm volatile("" : "+v"(v[k][q]));
    if (c + 1 < mine.count) {  // uniform
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this block's K is read
      find(c + 1);
      fetch_k();
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            o[n][q][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[k][q][e], sc[n][k / 4][k % 4], o[n][q][e], 0, 0, 0);
    // as pa_add_odd
#pragma unroll 1
    for (; odd; odd &= odd - 1) {
      const int key = k0 + __builtin_ctz(odd);
      if (key > t.pmax) break;
      const uint32_t page = (uint32_t)a.m.table[(int64_t)s.b * a.m.ld + (key >> a.m.log2_rows)];
      if (page >= a.m.pages) continue;  // its scores are NaN
      const float* row = (const float*)a.vp + page * a.m.page_els + head +
                         (int64_t)(key & ((1 << a.m.log2_rows) - 1)) * a.m.row_els + 16 * kg;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(row + 64 * q + 4 * r);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if (x[e] - x[e] != 0.f && pa_sees(a, key, qpos[n])) o[n][q][e][r] += x[e];
        }
    }
  }
  __syncthreads();  // every wave's blocks are done: the merge takes their LDS
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int pr = 16 * n + i16;
    lrun[n] = pa_add_groups(lrun[n]);
    if (pr < t.nr) {
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<f32x4*>(lds.o + (wave * kPaRows + pr) * OP + 64 * q + 16 * kg + 4 * r) =
              f32x4{o[n][q][0][r], o[n][q][1][r], o[n][q][2][r], o[n][q][3][r]};
      if (kg == 0) {
        merge.m[wave * kPaRows + pr] = mref[n];
        merge.l[wave * kPaRows + pr] = lrun[n];
      }
    }
  }
  __syncthreads();
  pa_leave<float, DH, OP>(a, s, t, g, t.parts, part, lds.o, merge.m, merge.l, merge.at, merge.fin);
  __syncthreads();  // the next item's blocks take it again
}

template <int DH>
__global__ __launch_bounds__(64 * kPaWaves) __attribute__((amdgpu_waves_per_eu(2))) void attn_paged_f32(PaArgs a) {
  __shared__ __align__(16) PaF32Lds<DH> lds;
  __shared__ PaMergeLds merge;
  const int g = blockIdx.x;
  PaSeq s;
  PaTile t;
  int part;
  bool first;
  for (uint32_t u = blockIdx.y; pa_item<float, false>(a, u, s, t, part, first); u += gridDim.y) {  // uniform
    if (first && s.ne < s.nq) pa_rows_past<float, DH>(a, s, g);
    if (t.nr <= 0 || part >= t.parts) continue;
    if (t.nr <= 16)
      pa_f32_part<DH, 1>(a, s, t, g, part, lds, merge);
    else
      pa_f32_part<DH, 2>(a, s, t, g, part, lds, merge);
  }
}

// bf16, many rows: up to 128 pairs per workgroup, 32 of each of four waves, which share
// the key blocks: 64 keys, staged by all of them in two LDS buffers, the next block's
// loads under way while one is computed, a barrier a block. S^T, P and O^T as in the
// few-row kernel, P in one bf16 term (half a step of 2^-8 of each probability: the error of
// an output is 0.0023 of it for 0.0017, which its own rounding leaves; a second term would
// double the products of P V). A wave skips the blocks that none of its rows sees.
//
// Two workgroups share a CU, two waves a SIMD, all its registers. 16384 causal rows of 16
// heads (4 kv heads): 920 to 970 TFLOP/s, three quarters of a large library product's rate,
// the MFMA busy for 37 % of the time, the VALU for 45 %; a workgroup alone on its CU takes
// 0.63 of that. Under a window of 1024 a tile is 18 blocks, of which 5 lie at an edge, and
// its first loads and its stores count: 16252 rows of 16 heads 228 to 240 us, 560 to 580 TFLOP/s.
// Measured and not better: eight waves with tiles of 256 pairs (the same, with a window 6 %
// slower), blocks straight to LDS with the products of the next block between the
// exponentials of this one (a window: 270 to 305 us), raised priority of one of the two
// waves (the same), the next item asked for before this one is stored (the same).
template <int DH>
struct PaManyLds {
  static constexpr int KP = DH + 8, VP = DH + 32;
  bf16_t k[2][kPaManyBlock * KP];
  bf16_t v[2][kPaManyBlock * VP];
  // keys of a block whose V is not finite: of the one computed, the one staged, and those before and behind, in turn
  uint32_t odd[4][2];
};
template <int DH>
__device__ __forceinline__ void pa_many_bf16(const PaArgs& a, PaManyLds<DH>& lds, uint32_t wg, uint32_t wgs) {
  constexpr int TK = kPaManyBlock;
  constexpr int NT = 64 * kPaWaves;
  constexpr int NDS = DH / 16;
  constexpr int NDB = DH / 32;
  constexpr int NKB = TK / 32;
  constexpr int NPS = TK / 16;
  constexpr int KP = PaManyLds<DH>::KP, VP = PaManyLds<DH>::VP;
  constexpr int CPR = DH / 8;
  constexpr int RPT = NT / CPR;       // rows of a piece of all threads
  constexpr int NLD = TK * CPR / NT;  // 16-byte pieces of K (and of V) per thread
  auto& k_lds = lds.k;
  auto& v_lds = lds.v;
  auto& odd_lds = lds.odd;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 31, hf = lane >> 5;
  const float scale = pa_scale(a);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  const int lr = threadIdx.x / CPR, lp = threadIdx.x % CPR;
  const uint32_t rsb = (uint32_t)a.m.row_els * sizeof(bf16_t);
  // the rows of this wave's piece i lie in one 16-key group
  auto group = [&](int i) { return RPT == 16 ? i : 2 * i + wave / 2; };
  const int krow = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
  const int tg = lane >> 4, ti = lane & 15;
  const int v_lane = ((tg >> 1) * 8 + (ti >> 2)) * VP + 16 * (tg & 1) + 4 * (ti & 3);
  auto vt_frag = [&](int b, int db, int k) { return pa_vt_frag<VP>(&v_lds[b][v_lane + 16 * k * VP + 32 * db]); };
  const int g = blockIdx.x;
  const int64_t head = g * a.m.head_els;

  for (uint32_t u = wg;; u += wgs) {  // uniform
    PaSeq s;
    PaTile t;
    int part;
    bool first;
    if (!pa_item<bf16_t, true>(a, u, s, t, part, first)) return;
    if (first && s.ne < s.nq) pa_rows_past<bf16_t, DH>(a, s, g);
    if (t.nr <= 0 || part >= t.parts) continue;
    const int c0 = part * s.part, c1 = min(c0 + s.part, t.nt);

    u32x4 kreg[NLD], vreg[NLD];
    PaPages pages;
    int bad = 0;
    auto fetch = [&](int c) {
      const int i16 = (c - c0) & 15;
      if (i16 == 0) pages = pa_pages<bf16_t, TK>(a, s, t, head, [&](int x) { return pa_listed(t, c + x); });
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        const uint32_t off = __umul24((uint32_t)min(lr & 15, pa_last_row<TK>(t, c == t.nt - 1, group(i))), rsb) +
                             (uint32_t)lp * 16u;
        kreg[i] = ld16(pages.at(a.kp, 4 * i16 + group(i)) + off);
        vreg[i] = ld16(pages.at(a.vp, 4 * i16 + group(i)) + off);
      }
      bad = (int)(pages.bad >> (4 * i16) & 15);
    };
    auto stage = [&](int c) {
      const int b = (c - c0) & 1;
      if (c < t.in0 || c >= t.in1) {  // uniform
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
          const int row = lr + i * RPT;
          if (pa_clean(vreg[i])) atomicOr(&odd_lds[(c - c0) & 3][row >> 5], 1u << (row & 31));
        }
      }
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        *reinterpret_cast<u32x4*>(&k_lds[b][(lr + i * RPT) * KP + 8 * lp]) = kreg[i];
        *reinterpret_cast<u32x4*>(&v_lds[b][(lr + i * RPT) * VP + 8 * lp]) = vreg[i];
      }
    };
    if (threadIdx.x < 8) odd_lds[threadIdx.x >> 1][threadIdx.x & 1] = 0;
    const int pr = min(kPaRows * wave + col, t.nr - 1), qi = pr * a.g_magic >> 16;
    const int qpos = t.pmin + qi;
    // the wave's first and last position
    const int w0 = t.pmin + (min(kPaRows * wave, t.nr - 1) * a.g_magic >> 16);
    const int w1 = t.pmin + ((min(kPaRows * wave + kPaRows, t.nr) - 1) * a.g_magic >> 16);
    const bool live = kPaRows * wave < t.nr;
    const int64_t qrow = (int64_t)(s.q0 + t.i0 + qi) * a.H + g * a.G + (pr - qi * a.G);
    u32x4 qf[NDS];
#pragma unroll
    for (int k = 0; k < NDS; ++k) qf[k] = ld16((const bf16_t*)a.q + qrow * DH + 8 * hf + 16 * k);
    if (c0 < c1) fetch(c0);
    pa_flip(qf, flip);

    float mref = -INFINITY, lrun = 0.f;
    f32x16 o[NDB];
#pragma unroll
    for (int c = 0; c < NDB; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[c][r] = 0.f;

    __syncthreads();  // odd_lds is clear
    int bad_now = 0;
    if (c0 < c1) {
      stage(c0);
      bad_now = bad;
      if (c0 + 1 < c1) fetch(c0 + 1);
    }
    __syncthreads();
    // a block that every row sees whole, or one at an edge of what they see
    auto block = [&](auto edge, int c) {
      constexpr bool EDGE = decltype(edge)::value;
      const int b = (c - c0) & 1;
      [[maybe_unused]] const int k0 = pa_listed(t, c) * TK;
      // some row of the wave sees some key (uniform over the wave)
      bool any = live;
      if constexpr (EDGE)
        any = any && k0 <= w1 && (!a.window || k0 + TK - 1 > w0 - a.window || k0 < a.sinks);
      if (any) {
        f32x16 sc[NKB];
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[kb][r] = 0.f;
        __builtin_amdgcn_s_setprio(1);
        // the operands of a step are read under the products of the one before
        u32x4 kf[4][NKB];
        auto read_k = [&](int k) {
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb)
            kf[k & 3][kb] = *reinterpret_cast<const u32x4*>(&k_lds[b][(32 * kb + krow) * KP + 16 * k + 8 * hf]);
        };
#pragma unroll
        for (int k = 0; k < 3; ++k) read_k(k);
#pragma unroll
        for (int k = 0; k < NDS; ++k) {
          if (k + 3 < NDS) read_k(k + 3);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) sc[kb] = pa_mfma32(kf[k & 3][kb], qf[k], sc[kb]);
        }
        __builtin_amdgcn_s_setprio(0);
        if (bad_now) {  // uniform
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[kb][r] += pa_bad(bad_now, 2 * kb + (r >> 3));
        }
        if constexpr (EDGE)
          pa_hide(a, sc, qpos, k0, 8 * hf, [](int kb, int r) { return 32 * kb + 16 * (r >> 3) + (r & 7); });
        u32x4 vf[2][NDB];
        auto read_v = [&](int k) {
#pragma unroll
          for (int db = 0; db < NDB; ++db) vf[k & 1][db] = vt_frag(b, db, k);
        };
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
        pa_softmax<NKB, NDB>(sc, o, mref, lrun, scale);
        u32x4 pb[NPS];
#pragma unroll
        for (int k = 0; k < NPS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            pb[k][e] = f32x2_to_bf16x2_bits(sc[k >> 1][8 * (k & 1) + 2 * e], sc[k >> 1][8 * (k & 1) + 2 * e + 1]);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k = 0; k < NPS; ++k) {
          if (k + 1 < NPS) read_v(k + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int db = 0; db < NDB; ++db) o[db] = pa_mfma32(vf[k & 1][db], pb[k], o[db]);
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (EDGE) {
          const uint32_t* w = odd_lds[(c - c0) & 3];
          const uint64_t odd = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)w[1]) << 32 |
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)w[0]);
          if (odd) pa_add_odd<bf16_t, DH>(a, s, t, odd, k0, head, qpos, hf, o);
        }
      }
      if (threadIdx.x < 2) odd_lds[(c - c0 + 3) & 3][threadIdx.x] = 0;  // of the block before, for the third from here
      if (c + 1 < c1) {  // uniform over the workgroup
        stage(c + 1);
        bad_now = bad;
        if (c + 2 < c1) fetch(c + 2);
      }
      __syncthreads();
    };
    int c = c0;
    for (const int e = min(t.in0, c1); c < e; ++c) block(std::true_type{}, c);
    for (const int e = min(t.in1, c1); c < e; ++c) block(std::false_type{}, c);
    for (; c < c1; ++c) block(std::true_type{}, c);
    lrun = pa_add_halves(lrun);
    if (kPaRows * wave + col < t.nr) {
      if (t.parts > 1) {
        const int64_t at = pa_slot(a, s, t.i0 + qi, g * a.G + (pr - qi * a.G)) + part;
        if (hf == 0) *reinterpret_cast<float2*>(a.pml + 2 * at) = float2{mref, lrun};
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(a.po + at * DH + 32 * db + 8 * i + 4 * hf) =
                f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
      } else {
        const float inv = pa_finish(a, qpos, 1.f, lrun);
        const bool none = qpos < 0;  // zero, whatever the sums
        bf16_t* op = (bf16_t*)a.out + qrow * DH + 4 * hf;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint2 w;
            w.x = f32x2_to_bf16x2_bits(o[db][4 * i] * inv, o[db][4 * i + 1] * inv);
            w.y = f32x2_to_bf16x2_bits(o[db][4 * i + 2] * inv, o[db][4 * i + 3] * inv);
            if (none) w.x = w.y = 0u;
            *reinterpret_cast<uint2*>(op + 32 * db + 8 * i) = w;
          }
      }
    }
    __syncthreads();  // odd_lds, before the next item clears it
  }
}

// Both kinds of rows in one launch, so that those bound by memory and those bound by
// products share the CUs (61 single rows and 3 pieces of prompts of 500 to 1100 rows, 4 kv
// heads: 270 us; when it was 275 one kernel after the other took 307):
// a.many_wgs of the workgroups of a kv head take many rows,
// a.many_lead of them (one per CU) before those that take few, the others behind.
template <int DH>
__global__ __launch_bounds__(64 * kPaWaves) __attribute__((amdgpu_waves_per_eu(2))) void attn_paged_both_bf16(
    PaArgs a) {
  __shared__ __align__(16) union Lds {
    PaFewLds<DH> few;
    PaManyLds<DH> many;
    __device__ Lds() {}
  } lds;
  __shared__ PaMergeLds merge;
  const uint32_t y = blockIdx.y, few = gridDim.y - a.many_wgs;
  if (y < a.many_lead || y >= a.many_lead + few)
    pa_many_bf16<DH>(a, lds.many, y < a.many_lead ? y : y - few, a.many_wgs);
  else
    pa_few_bf16<DH>(a, lds.few, merge, y - a.many_lead, few);
}

// The parts of the rows that have several, merged. A row that has keys in up to kPaWide of them
// takes DH / 4 threads of four columns, one fma per part in the parts' order on the largest
// maximum; a row of more a workgroup, whose slot x takes the parts of the sequence that are x
// modulo its slots, in their order, before the slots are merged in theirs. A part without a key
// that the row sees (its maximum is -inf) changes nothing in either, so a row's bits do not
// depend on the parts that its tile has beside its own. Bound by the parts' bytes: 2170 rows of
// 16 heads, up to 5 parts of those of prompts, 24 us; 8 rows of 2 parts 3.9, the launch and its search.
constexpr int kPaWide = 16;
constexpr int kPaMergeThreads = 256;

// Parts in which the row at position pos sees a key.
__device__ __forceinline__ int pa_own_parts(const PaArgs& a, const PaSeq& s, int pos) {
  const int lo = a.window ? max(pos - a.window + 1, 0) : 0, ns = (min(a.sinks, lo) + kPaBlock - 1) >> kPaLogBlock;
  const int sink_parts = ns ? s.cut.of(ns - 1) + 1 : 0;
  return sink_parts + max(s.cut.of(pos >> kPaLogBlock) - max(s.cut.of(lo >> kPaLogBlock), sink_parts) + 1, 0);
}

template <typename T, int DH>
__global__ __launch_bounds__(kPaMergeThreads) void attn_paged_combine(PaArgs a) {
  constexpr int TPP = DH / 4, PP = kPaMergeThreads / TPP, B = 4;
  __shared__ __align__(16) float o_lds[PP][DH];
  __shared__ float m_lds[PP], l_lds[PP];
  const int H = a.H, d = 4 * (threadIdx.x % TPP), slot = threadIdx.x / TPP;
  auto units = [&](const PaSeq& q) {
    return q.parts <= 1 ? 0 : (q.parts > kPaWide ? q.ne * H : (q.ne * H + PP - 1) / PP);
  };
  for (uint32_t u = blockIdx.x;; u += gridDim.x) {  // uniform
    PaSeq s;
    int pair;
    if (!pa_find<T>(a, u, units, s, pair)) return;
    const bool one = s.parts > kPaWide;  // pair of the workgroup
    if (!one) pair = pair * PP + slot;
    if (pair >= s.ne * H) continue;  // no barrier ahead unless the unit is one pair
    const int i = pair / H, h = pair - i * H, pos = s.pos0 + i;
    int np, sink_parts = 0, first_part = 0, own;
    if (s.many) {
      own = np = pa_tile<true>(a, s, i / a.many_tile).parts;
    } else {
      const PaTile t = pa_tile<false>(a, s, i / a.few_tile);
      np = t.parts;
      sink_parts = t.sink_parts;
      first_part = t.first_part;
      own = pa_own_parts(a, s, min(max(pos, 0), a.kmax - 1));
    }
    if (np <= 1) continue;  // finished by its workgroup
    const int64_t base = pa_slot(a, s, i, h);
    T* row = (T*)a.out + ((int64_t)(s.q0 + i) * H + h) * DH;
    const float2* ml = reinterpret_cast<const float2*>(a.pml) + base;
    const float* po = a.po + base * DH + d;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    if (one && own > kPaWide) {  // uniform
      const int lead = max((sink_parts - slot + PP - 1) / PP, 0);
      const int run = sink_parts + ((slot - first_part) & (PP - 1));
      const int count = lead + max((np - run + PP - 1) / PP, 0);
      auto place = [&](int e) { return e < lead ? slot + PP * e : run + PP * (e - lead); };
      for (int e0 = 0; e0 < count; e0 += B) {
        float2 w[B];
        f32x4 v[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
          const int p = place(min(e0 + b, count - 1));
          w[b] = ml[p];
          v[b] = *reinterpret_cast<const f32x4*>(po + (int64_t)p * DH);
        }
#pragma unroll
        for (int b = 0; b < B; ++b)
          if (e0 + b < count) {
            const float mn = fmaxf(M, w[b].x);
            const float corr = M == -INFINITY ? 1.f : exp2f(M - mn);  // nothing but zeros (or a NaN to keep) so far
            const float f = w[b].x == -INFINITY ? 0.f : exp2f(w[b].x - mn);
            M = mn;
            L = fmaf(w[b].y, f, L * corr);
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = fmaf(v[b][e], f, O[e] * corr);
          }
      }
      *reinterpret_cast<f32x4*>(&o_lds[slot][d]) = O;
      if (d == 0) {
        m_lds[slot] = M;
        l_lds[slot] = L;
      }
      __syncthreads();
      if (threadIdx.x < TPP) {
        M = -INFINITY;
        L = 0.f;
        O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < PP; ++x) M = fmaxf(M, m_lds[x]);
#pragma unroll
        for (int x = 0; x < PP; ++x) {
          const float f = m_lds[x] == -INFINITY ? 0.f : exp2f(m_lds[x] - M);
          L = fmaf(l_lds[x], f, L);
          const f32x4 v = *reinterpret_cast<const f32x4*>(&o_lds[x][d]);
#pragma unroll
          for (int e = 0; e < 4; ++e) O[e] = fmaf(v[e], f, O[e]);
        }
      }
      __syncthreads();  // before the next row's
    } else if (!one || slot == 0) {
      for (int p = 0; p < np; ++p) M = fmaxf(M, ml[p].x);
      for (int p0 = 0; p0 < np; p0 += B) {
        float2 w[B];
        f32x4 v[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
          w[b] = ml[min(p0 + b, np - 1)];
          v[b] = *reinterpret_cast<const f32x4*>(po + (int64_t)min(p0 + b, np - 1) * DH);
        }
#pragma unroll
        for (int b = 0; b < B; ++b)
          if (p0 + b < np) {
            const float f = w[b].x == -INFINITY ? 0.f : exp2f(w[b].x - M);
            L = fmaf(w[b].y, f, L);
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = fmaf(v[b][e], f, O[e]);
          }
      }
    }
    if (one && slot) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) O[e] = pa_finish(a, pos, O[e], L);
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(row + d) = uint2{f32x2_to_bf16x2_bits(O[0], O[1]), f32x2_to_bf16x2_bits(O[2], O[3])};
    else
      *reinterpret_cast<f32x4*>(row + d) = O;
  }
}

// How a launch is cut at most: what the host knows are bounds. Slots are kept per row for the
// most parts that any row has, or per sequence for what one has at most, whichever takes less.
struct PaPlan {
  bool many;
  int few_tile, many_tile, row_per;
  int64_t seq_slots, slots, few_units, many_units;
};
// Slots of one sequence that is not of few rows, where its tiles have several parts: pairs of a
// tile x tiles x kv heads x parts. Many rows: parts < target / (tiles Hkv) + 1, of which tiles Hkv
// is below the target. fp32: parts < target / (tiles Hkv) + 4, with a window's and its sinks' ends.
constexpr int64_t kPaManySlots = 2 * kPaManyTarget * kPaManyRows;
constexpr int64_t kPaF32Slots = 5 * kPaTarget * kPaRows;

// The most parts of a tile of many rows: of a sequence with more tiles they are fewer.
static int pa_most_many(int blocks, int Hkv) {
  const int p = pa_div_up(kPaManyTarget, Hkv), all = pa_div_up(blocks, kPaManyMinPart / kPaManyBlock);
  return p < all ? p : (all > 1 ? all : 1);
}

// The same in a sequence of fp32 rows that are not few: it has more than two tiles.
static int pa_most_f32(int kmax, int Hkv, int rows, int window, int sinks) {
  const int wide = 3 * Hkv;
  if (wide >= kPaTarget) return 1;
  const int p = pa_most_parts(PaCut{0, 3}, kmax, rows, window, sinks), most = kPaTarget / wide + 4;
  return p < most ? p : most;
}

static PaPlan pa_plan(int n, int nseq, int H, int Hkv, int dtype, int qmax, int kmax, PaCut cut, int window,
                      int sinks, int few_pairs) {
  PaPlan p{};
  const int G = H / Hkv;
  if (qmax > n) qmax = n;
  const bool large = (int64_t)qmax * G > few_pairs;
  p.many = dtype == kBF16 && large;
  p.few_tile = kPaRows / G;
  p.many_tile = kPaManyRows / G;
  const int few_rows = large ? few_pairs / G : qmax;  // of a sequence
  const int few = pa_most_parts(cut, kmax, p.few_tile, window, sinks);
  int most = 1;  // of a tile of the other sequences
  if (p.many) most = pa_most_many(pa_blocks(kmax, p.many_tile, window, sinks, kPaManyLogBlock), Hkv);
  else if (large) most = pa_most_f32(kmax, Hkv, p.few_tile, window, sinks);
  p.row_per = few > most ? few : most;
  if (p.row_per > 1) {
    int64_t one = few > 1 ? (int64_t)few_rows * H * few : 0;
    if (most > 1) one = std::max(one, p.many ? kPaManySlots : kPaF32Slots);
    const int64_t by_row = (int64_t)n * H * p.row_per;
    p.seq_slots = nseq * one < by_row ? one : 0;
    p.slots = p.seq_slots ? nseq * one : by_row;
  }
  const int64_t rows = std::min((int64_t)nseq * (p.many ? few_rows : qmax), (int64_t)n);
  p.few_units = (rows / p.few_tile + nseq) * (p.many ? few : p.row_per);
  if (p.many) p.many_units = ((int64_t)n / p.many_tile + nseq) * most;
  return p;
}

static unsigned pa_grid(int64_t units, int64_t most) {
  const int64_t m = most < 1 ? 1 : (most > 32767 ? 32767 : most);
  return (unsigned)(units < 1 ? 1 : (units < m ? units : m));
}

template <typename T, int DH>
static void launch_paged(PaArgs a, const PaPlan& p, hipStream_t st) {
  const dim3 block(64 * kPaWaves);
  const unsigned few = pa_grid(p.few_units, kPaResident / a.Hkv);
  if constexpr (sizeof(T) == 4) {
    hipLaunchKernelGGL((attn_paged_f32<DH>), dim3(a.Hkv, few), block, 0, st, a);
  } else if (p.many) {
    a.many_wgs = pa_grid(p.many_units, kPaManyGrid / a.Hkv);
    a.many_lead = pa_grid(a.many_wgs, kPaResident / 2 / a.Hkv);
    hipLaunchKernelGGL((attn_paged_both_bf16<DH>),
                       dim3(a.Hkv, a.many_wgs + pa_grid(p.few_units, kPaResident / 2 / a.Hkv)), block, 0, st, a);
  } else {
    hipLaunchKernelGGL((attn_paged_few_bf16<DH>), dim3(a.Hkv, few), block, 0, st, a);
  }
  if (hipPeekAtLastError() != hipSuccess) return;  // no parts to merge
  if (p.row_per > 1)
    hipLaunchKernelGGL((attn_paged_combine<T, DH>), dim3(pa_grid((int64_t)a.n * a.H, kPaMergeGrid)),
                       dim3(kPaMergeThreads), 0, st, a);
}

static size_t pa_workspace(int n, int nseq, int H, int Hkv, int Dh, int dtype, int q_len_max, int kv_len_max,
                           int window, int sinks, int few_pairs) {
  // 0 for what the call refuses
  if (n <= 0 || nseq <= 0 || H <= 0 || H > 4096 || Hkv <= 0 || H % Hkv || H / Hkv > kPaMaxG || Dh <= 0 || Dh > 128 ||
      q_len_max < 0 || kv_len_max <= 0 || window < 0 || sinks < 0)
    return 0;
  const PaCut cut = pa_few_cut(Hkv, window);
  if (window >= kv_len_max) window = 0;
  if (sinks > kv_len_max) sinks = kv_len_max;
  const PaPlan p = pa_plan(n, nseq, H, Hkv, dtype, q_len_max, kv_len_max, cut, window, sinks, few_pairs);
  const size_t slots = (size_t)p.slots;
  return slots ? align256(slots * Dh * sizeof(float)) + align256(slots * 2 * sizeof(float)) : 0;
}

static int pa_call(const char* me, const void* q, const void* k_pages, const void* v_pages, int64_t kv_block_rows,
                   const int32_t* page_table, int64_t ld_table, int pages_per_seq, int64_t num_pages, int page_rows,
                   const int32_t* cu_q, const int32_t* kv_len, int nseq, void* out, int n, int H, int Hkv, int Dh,
                   int dtype, float scale, int q_len_max, int kv_len_max, int window, int sinks, int few_pairs,
                   void* workspace, size_t ws_bytes, hipStream_t stream) {
  PaArgs a;
  const int rc = page_map(a.m, me, page_table, ld_table, pages_per_seq, num_pages, page_rows, kv_block_rows, nseq,
                          Hkv, Dh, dtype);
  if (rc != kOk) return rc;
  if (n < 0 || H <= 0 || H > 4096 || H % Hkv != 0 || q_len_max < 0 || kv_len_max < 0 || window < 0 || sinks < 0) {
    set_error("%s: bad shape n=%d H=%d Hkv=%d q_len_max=%d kv_len_max=%d window=%d sinks=%d", me, n, H, Hkv,
              q_len_max, kv_len_max, window, sinks);
    return kBadArg;
  }
  if (H / Hkv > kPaMaxG) {
    set_error("%s: unsupported H=%d Hkv=%d (H / Hkv up to %d)", me, H, Hkv, kPaMaxG);
    return kUnsupported;
  }
  if (kv_len_max > (int64_t)pages_per_seq * page_rows) {
    set_error("%s: kv_len_max=%d past pages_per_seq=%d of page_rows=%d", me, kv_len_max, pages_per_seq, page_rows);
    return kBadArg;
  }
  if (n == 0 || nseq == 0) return kOk;
  if (!q || !cu_q || !kv_len || !out || (kv_len_max && (!page_table || (num_pages && (!k_pages || !v_pages))))) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out | (uintptr_t)workspace) & 15) {
    set_error("%s: q, the pages, out and workspace must be 16-byte aligned", me);
    return kBadArg;
  }
  const size_t need = pa_workspace(n, nseq, H, Hkv, Dh, dtype, q_len_max, kv_len_max, window, sinks,
                                   few_pairs);
  if (need && (!workspace || ws_bytes < need)) {
    set_error("%s: workspace %zu bytes < required %zu", me, ws_bytes, need);
    return kWorkspace;
  }
  if (kv_len_max > 0x7fffffff - 1024 || (int64_t)n * (H / Hkv) > 0x7fffffff - 1024) {
    set_error("%s: kv_len_max=%d n=%d beyond 2^31 - 1024 (n times H / Hkv too)", me, kv_len_max, n);
    return kUnsupported;
  }
  a.q = q;
  a.kp = k_pages;
  a.vp = v_pages;
  a.cu_q = cu_q;
  a.kv_len = kv_len;
  a.out = out;
  a.n = n;
  a.nseq = nseq;
  a.H = H;
  a.Hkv = Hkv;
  a.G = H / Hkv;
  a.qmax = q_len_max < n ? q_len_max : n;
  a.kmax = num_pages ? kv_len_max : 0;  // an empty pool: every position is past it
  // no position is at kv_len_max or beyond: what covers all of them is none, and sums of these stay in 32 bits
  a.window = window < kv_len_max ? window : 0;
  a.sinks = sinks < kv_len_max ? sinks : kv_len_max;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.cut = pa_few_cut(Hkv, window);
  const PaPlan p = pa_plan(n, nseq, H, Hkv, dtype, a.qmax, kv_len_max, a.cut, a.window, a.sinks, few_pairs);
  if (p.few_units > 0x7fffffff - 65536 || p.many_units > 0x7fffffff - 65536) {
    set_error("%s: n=%d nseq=%d kv_len_max=%d beyond the grid", me, n, nseq, kv_len_max);
    return kUnsupported;
  }
  a.po = (float*)workspace;
  a.pml = (float*)((char*)workspace + align256((size_t)p.slots * Dh * sizeof(float)));
  a.seq_slots = p.seq_slots;
  a.g_magic = 65536 / a.G + 1;
  a.few_tile = p.few_tile;
  a.many_tile = p.many_tile;
  a.row_per = p.row_per;
  a.few_pairs = few_pairs;
  if (dtype == kBF16)
    Dh == 64 ? launch_paged<bf16_t, 64>(a, p, stream) : launch_paged<bf16_t, 128>(a, p, stream);
  else
    Dh == 64 ? launch_paged<float, 64>(a, p, stream) : launch_paged<float, 128>(a, p, stream);
  return launch_status(me);
}

}  // namespace wfd

extern "C" {

size_t wfd_attn_paged_workspace_bytes(int n, int nseq, int H, int Hkv, int Dh, int dtype, int q_len_max,
                                      int kv_len_max, int window, int sinks) {
  return wfd::pa_workspace(n, nseq, H, Hkv, Dh, dtype, q_len_max, kv_len_max, window, sinks, wfd::kPaFewPairs);
}

int wfd_attn_paged(const void* q, const void* k_pages, const void* v_pages, int64_t kv_block_rows,
                   const int32_t* page_table, int64_t ld_table, int pages_per_seq, int64_t num_pages,
                   int page_rows, const int32_t* cu_q, const int32_t* kv_len, int nseq, void* out, int n, int H,
                   int Hkv, int Dh, int dtype, float scale, int q_len_max, int kv_len_max, int window,
                   int sinks, void* workspace, size_t ws_bytes, hipStream_t stream) {
  return wfd::pa_call("wfd_attn_paged", q, k_pages, v_pages, kv_block_rows, page_table, ld_table, pages_per_seq,
                      num_pages, page_rows, cu_q, kv_len, nseq, out, n, H, Hkv, Dh, dtype, scale, q_len_max, kv_len_max,
                      window, sinks, wfd::kPaFewPairs, workspace, ws_bytes, stream);
}

size_t wfd_attn_paged_by_row_workspace_bytes(int n, int nseq, int H, int Hkv, int Dh, int dtype, int q_len_max,
                                             int kv_len_max, int window, int sinks) {
  return wfd::pa_workspace(n, nseq, H, Hkv, Dh, dtype, q_len_max, kv_len_max, window, sinks, wfd::kPaAllFew);
}

int wfd_attn_paged_by_row(const void* q, const void* k_pages, const void* v_pages, int64_t kv_block_rows,
                          const int32_t* page_table, int64_t ld_table, int pages_per_seq, int64_t num_pages,
                          int page_rows, const int32_t* cu_q, const int32_t* kv_len, int nseq, void* out, int n, int H,
                          int Hkv, int Dh, int dtype, float scale, int q_len_max, int kv_len_max, int window,
                          int sinks, void* workspace, size_t ws_bytes, hipStream_t stream) {
  return wfd::pa_call("wfd_attn_paged_by_row", q, k_pages, v_pages, kv_block_rows, page_table, ld_table, pages_per_seq,
                      num_pages, page_rows, cu_q, kv_len, nseq, out, n, H, Hkv, Dh, dtype, scale, q_len_max, kv_len_max,
                      window, sinks, wfd::kPaAllFew, workspace, ws_bytes, stream);
}

}  // extern "C"
