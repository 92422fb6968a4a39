// Keys and values appended to the pages of a KV cache (pages.h), k and q rotated
// on the way.
//
// A workgroup takes one row of the call. It asks for the row's values first, three
// 16-byte pieces a thread, then each wave finds the row's sequence by a look at cu_q (64
// entries a load), its position, its page, and the sines and cosines of that position,
// four (fp32: two) pairs a load. Bound by memory, every value read once and written once:
// 8332 rows of 16 + 2 * 16 heads of 128 bf16 39 us (5.2 TB/s, a large copy's rate; 51 us
// with the values asked for after the place is known and the table read number by
// number). 8 rows 3.5 us, the launch and that chain of loads (4.3).
#include "pages.h"

namespace wfd {

constexpr int kPgThreads = 256;
constexpr int kPgMaxRows = (1 << 24) - 1;  // a workgroup each: a launch has fewer than 2^32 threads
constexpr int kPgAhead = 3;  // pieces of a thread asked for before the row's place is known

struct PgRow {
  int64_t at;  // element offset of the row's kv head 0, -1: the row has no place
  int pos;
  bool mine;   // the row is one of a sequence
};

__device__ __forceinline__ PgRow pg_row(const PageMap& m, const int32_t* __restrict__ cu_q,
                                        const int32_t* __restrict__ kv_len, int nseq, int r) {
  PgRow o;
  const int b = seq_of_row(cu_q, nseq, r);
  o.mine = b >= 0;
  o.at = -1;
  o.pos = -1;
  if (b < 0) return o;
  o.pos = max(kv_len[b], 0) - (cu_q[b + 1] - r);
  const int j = o.pos >> m.log2_rows;
  if (o.pos < 0 || j >= m.per_seq) return o;
  const uint32_t page = (uint32_t)m.table[b * m.ld + j];
  if (page >= m.pages) return o;
  o.at = page * m.page_els + (int64_t)(o.pos & ((1 << m.log2_rows) - 1)) * m.row_els;
  return o;
}

// The rotation of wfd_qkv_rope_append, bit for bit.
__device__ __forceinline__ void pg_rotate(float& x0, float& x1, float c, float s) {
  const float y0 = fmaf(x0, c, -(x1 * s));
  const float y1 = fmaf(x0, s, x1 * c);
  x0 = y0;
  x1 = y1;
}

// qkv rows (H + 2 Hkv heads of DH): heads below H to q_out, the next Hkv to k, the last to v.
template <typename T, int DH>
__global__ __launch_bounds__(kPgThreads) void qkv_rope_append_paged_kernel(
    const T* __restrict__ qkv, int64_t ldq, const int32_t* __restrict__ cu_q, const int32_t* __restrict__ kv_len,
    int nseq, PageMap m, const float* __restrict__ cos_t, const float* __restrict__ sin_t, int tab_rows,
    T* __restrict__ q_out, T* __restrict__ kp, T* __restrict__ vp, int H, int Hkv) {
  constexpr int V = Elem<T>::kVec, CPR = DH / V;
  typedef float fvec __attribute__((ext_vector_type(V / 2)));
  const int r = blockIdx.x, chunks = (H + 2 * Hkv) * CPR;
  const T* src = qkv + r * ldq;
  u32x4 w[kPgAhead];
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kPgAhead; ++i) w[i] = ld16(src + min(c0 + kPgThreads * i, chunks - 1) * V);
  };
  load(threadIdx.x);
  const PgRow row = pg_row(m, cu_q, kv_len, nseq, r);
  if (!row.mine) return;  // uniform
  const bool turn = row.pos >= 0 && row.pos < tab_rows;
  // every chunk of a thread is at the same place of its head
  static_assert(kPgThreads % CPR == 0, "a thread's place in its heads");
  const int d = threadIdx.x % CPR * V;
  fvec cs, sn;
#pragma unroll
  for (int e = 0; e < V / 2; ++e) cs[e] = sn[e] = NAN;
  if (turn) {  // uniform
    cs = *reinterpret_cast<const fvec*>(cos_t + (int64_t)row.pos * (DH / 2) + d / 2);
    sn = *reinterpret_cast<const fvec*>(sin_t + (int64_t)row.pos * (DH / 2) + d / 2);
  }
  for (int c0 = threadIdx.x; c0 < chunks; c0 += kPgThreads * kPgAhead) {
    if (c0 >= kPgThreads) load(c0);
#pragma unroll
    for (int i = 0; i < kPgAhead; ++i) {
      const int c = c0 + kPgThreads * i, head = c / CPR;
      if (c >= chunks) break;
      if (head < H + Hkv) {
        float x[V];
        Elem<T>::unpack(w[i], x);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) pg_rotate(x[2 * e], x[2 * e + 1], cs[e], sn[e]);
        w[i] = Elem<T>::pack(x);
      }
      if (head < H)
        *reinterpret_cast<u32x4*>(q_out + ((int64_t)r * H + head) * DH + d) = w[i];
      else if (row.at >= 0 && turn) {
        const bool isv = head >= H + Hkv;
        T* p = isv ? vp : kp;
        *reinterpret_cast<u32x4*>(p + row.at + (head - H - (isv ? Hkv : 0)) * m.head_els + d) = w[i];
      }
    }
  }
}

template <typename T, int DH>
__global__ __launch_bounds__(kPgThreads) void kv_append_paged_kernel(
    const T* __restrict__ k, int64_t ldk, const T* __restrict__ v, int64_t ldv, const int32_t* __restrict__ cu_q,
    const int32_t* __restrict__ kv_len, int nseq, PageMap m, T* __restrict__ kp, T* __restrict__ vp, int Hkv) {
  constexpr int V = Elem<T>::kVec, CPR = DH / V;
  const int r = blockIdx.x, chunks = 2 * Hkv * CPR;
  u32x4 w[kPgAhead];
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kPgAhead; ++i) {
      const int c = min(c0 + kPgThreads * i, chunks - 1), vc = c - Hkv * CPR;
      w[i] = ld16(vc >= 0 ? v + r * ldv + vc * V : k + r * ldk + c * V);
    }
  };
  load(threadIdx.x);
  const PgRow row = pg_row(m, cu_q, kv_len, nseq, r);
  if (row.at < 0) return;  // uniform
  for (int c0 = threadIdx.x; c0 < chunks; c0 += kPgThreads * kPgAhead) {
    if (c0 >= kPgThreads) load(c0);
#pragma unroll
    for (int i = 0; i < kPgAhead; ++i) {
      const int c = c0 + kPgThreads * i, head = c / CPR;
      if (c >= chunks) break;
      const bool isv = head >= Hkv;
      *reinterpret_cast<u32x4*>((isv ? vp : kp) + row.at + (head - (isv ? Hkv : 0)) * m.head_els + c % CPR * V) = w[i];
    }
  }
}

}  // namespace wfd

extern "C" {

int wfd_qkv_rope_append_paged(const void* qkv, int64_t ldq, const int32_t* cu_q, const int32_t* kv_len, int nseq,
                              const int32_t* page_table, int64_t ld_table, int pages_per_seq, int64_t num_pages,
                              int page_rows, const float* rope_cos, const float* rope_sin, int rope_rows, void* q_out,
                              void* k_pages, void* v_pages, int64_t kv_block_rows, int n, int H, int Hkv, int Dh,
                              int dtype, hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_qkv_rope_append_paged";
  PageMap m;
  const int rc = page_map(m, me, page_table, ld_table, pages_per_seq, num_pages, page_rows, kv_block_rows, nseq, Hkv,
                          Dh, dtype);
  if (rc != kOk) return rc;
  const int vec = dtype == kBF16 ? 8 : 4;
  if (n < 0 || H <= 0 || H > 4096 || rope_rows <= 0 || ldq < (int64_t)(H + 2 * Hkv) * Dh || ldq % vec) {
    set_error("%s: bad shape n=%d H=%d Hkv=%d Dh=%d rope_rows=%d ldq=%lld", me, n, H, Hkv, Dh, rope_rows,
              (long long)ldq);
    return kBadArg;
  }
  if (n > kPgMaxRows) {
    set_error("%s: n=%d beyond the grid (up to %d rows)", me, n, kPgMaxRows);
    return kUnsupported;
  }
  if (n == 0 || nseq == 0) return kOk;
  if (!qkv || !cu_q || !kv_len || !rope_cos || !rope_sin || !q_out || (pages_per_seq && !page_table) ||
      (num_pages && (!k_pages || !v_pages))) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)rope_cos |
       (uintptr_t)rope_sin) & 15) {
    set_error("%s: qkv, q_out, the pages and the rope tables must be 16-byte aligned", me);
    return kBadArg;
  }
#define WFD_PG(TT, DHV)                                                                                              \
  hipLaunchKernelGGL((qkv_rope_append_paged_kernel<TT, DHV>), dim3(n), dim3(kPgThreads), 0, stream, (const TT*)qkv, \
                     ldq, cu_q, kv_len, nseq, m, rope_cos, rope_sin, rope_rows, (TT*)q_out, (TT*)k_pages,            \
                     (TT*)v_pages, H, Hkv)
  if (dtype == kBF16) {
    if (Dh == 64) WFD_PG(bf16_t, 64);
    else WFD_PG(bf16_t, 128);
  } else {
    if (Dh == 64) WFD_PG(float, 64);
    else WFD_PG(float, 128);
  }
#undef WFD_PG
  return launch_status(me);
}

int wfd_kv_append_paged(const void* k, int64_t ldk, const void* v, int64_t ldv, const int32_t* cu_q,
                        const int32_t* kv_len, int nseq, const int32_t* page_table, int64_t ld_table,
                        int pages_per_seq, int64_t num_pages, int page_rows, void* k_pages, void* v_pages,
                        int64_t kv_block_rows, int n, int Hkv, int Dh, int dtype, hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_kv_append_paged";
  PageMap m;
  const int rc = page_map(m, me, page_table, ld_table, pages_per_seq, num_pages, page_rows, kv_block_rows, nseq, Hkv,
                          Dh, dtype);
  if (rc != kOk) return rc;
  const int vec = dtype == kBF16 ? 8 : 4;
  if (n < 0 || ldk < (int64_t)Hkv * Dh || ldv < (int64_t)Hkv * Dh || ldk % vec || ldv % vec) {
    set_error("%s: bad shape n=%d Hkv=%d Dh=%d ldk=%lld ldv=%lld", me, n, Hkv, Dh, (long long)ldk, (long long)ldv);
    return kBadArg;
  }
  if (n > kPgMaxRows) {
    set_error("%s: n=%d beyond the grid (up to %d rows)", me, n, kPgMaxRows);
    return kUnsupported;
  }
  if (n == 0 || nseq == 0 || pages_per_seq == 0 || num_pages == 0) return kOk;
  if (!k || !v || !cu_q || !kv_len || !page_table || !k_pages || !v_pages) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) {
    set_error("%s: k, v and the pages must be 16-byte aligned", me);
    return kBadArg;
  }
#define WFD_PG(TT, DHV)                                                                                            \
  hipLaunchKernelGGL((kv_append_paged_kernel<TT, DHV>), dim3(n), dim3(kPgThreads), 0, stream, (const TT*)k, ldk, \
                     (const TT*)v, ldv, cu_q, kv_len, nseq, m, (TT*)k_pages, (TT*)v_pages, Hkv)
  if (dtype == kBF16) {
    if (Dh == 64) WFD_PG(bf16_t, 64);
    else WFD_PG(bf16_t, 128);
  } else {
    if (Dh == 64) WFD_PG(float, 64);
    else WFD_PG(float, 128);
  }
#undef WFD_PG
  return launch_status(me);
}

}  // extern "C"
