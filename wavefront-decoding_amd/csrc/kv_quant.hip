// The 8-bit slot cache written and read back (quant.h has the format).
//
// A row of one kv head is dealt to Dh / 8 lanes of 8 values each (16 bytes of
// bf16), so a wave covers 4 rows of 128 or 8 of 64; the row's largest |x| is a
// few shuffles within those lanes, the codes leave as 8 bytes a lane and the
// exponent as one byte from the row's first lane. Bound by memory: every value
// is read once and every code written once. 8192 bf16 rows of 16 heads x 128 take
// 20.6 us to write (4.9 TB/s, as a large copy) and 19.2 to read back, fp32 ones 34 and
// 29; the few rows of a decode step 2.7 us a launch, the launch itself.
#include <type_traits>

#include "quant.h"

namespace wfd {

constexpr int kQThreads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    Elem<T>::unpack(ld16(p), x);
  } else {
    float a[4], b[4];
    Elem<T>::unpack(ld16(p), a);
    Elem<T>::unpack(ld16(p + 4), b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<u32x4*>(p) = Elem<T>::pack(x);
  } else {
    *reinterpret_cast<u32x4*>(p) = u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                                         __float_as_uint(x[3])};
    *reinterpret_cast<u32x4*>(p + 4) = u32x4{__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]),
                                             __float_as_uint(x[7])};
  }
}

// Quantise one row held by LPR consecutive lanes (lane part `sub` its columns
// 8 sub ..) and store it at element offset `off` of the codes.
template <int CODE, int LPR>
__device__ __forceinline__ void write_row(const float (&x)[8], int sub, int64_t off, uint8_t* __restrict__ codes,
                                          uint8_t* __restrict__ exps) {
  uint32_t amax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
  for (int m = LPR / 2; m >= 1; m >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, m, 64));
  const uint32_t b = exp_byte<CODE>(amax);
  *reinterpret_cast<uint2*>(codes + off + 8 * sub) = encode8<CODE>(x, b);
  if (sub == 0) exps[off / (8 * LPR)] = (uint8_t)b;
}

// bf16 lanes take a K and a V row, 32 bytes of loads in flight as an fp32 lane has of
// one: the write of 8192 rows x 16 heads x 128 in 20.6 us where a row a lane group took
// 24.6; fp32 34 us (4.9 TB/s) either way, and with the read back 74 us against 75.5.
template <typename T>
constexpr bool kAppendPair = sizeof(T) == 2;

template <typename T, int CODE, int DH>
__global__ __launch_bounds__(kQThreads) void kv_append_q_kernel(const T* __restrict__ k, int64_t ldk,
                                                                const T* __restrict__ v, int64_t ldv,
                                                                uint8_t* __restrict__ kc, uint8_t* __restrict__ vc,
                                                                uint8_t* __restrict__ ke, uint8_t* __restrict__ ve,
                                                                int64_t block_rows,
                                                                const int64_t* __restrict__ flat_row, int n,
                                                                int Hkv) {
  constexpr int LPR = DH / 8;
  const int64_t unit = ((int64_t)blockIdx.x * kQThreads + threadIdx.x) / LPR;
  const int sub = threadIdx.x % LPR;
  if constexpr (kAppendPair<T>) {  // (token, head): K and V
    const int i = (int)(unit / Hkv);
    if (i >= n) return;
    const int h = (int)(unit - (int64_t)i * Hkv);
    float x[8], y[8];
    load8(k + i * ldk + h * DH + 8 * sub, x);
    load8(v + i * ldv + h * DH + 8 * sub, y);
    const int64_t off = kv_offset(flat_row[i], h, Hkv, DH, block_rows);
    write_row<CODE, LPR>(x, sub, off, kc, ke);
    write_row<CODE, LPR>(y, sub, off, vc, ve);
  } else {  // (token, K or V, head)
    const int i = (int)(unit / (2 * Hkv));
    if (i >= n) return;
    const int r = (int)(unit - (int64_t)i * 2 * Hkv);
    const bool isv = r >= Hkv;
    const int h = isv ? r - Hkv : r;
    float x[8];
    load8((isv ? v + i * ldv : k + i * ldk) + h * DH + 8 * sub, x);
    write_row<CODE, LPR>(x, sub, kv_offset(flat_row[i], h, Hkv, DH, block_rows), isv ? vc : kc, isv ? ve : ke);
  }
}

// y to the float on its side of zero, last bit set if anything was cut off:
// such a value compares with, and rounds to, anything of fewer bits exactly as
// y itself would, so a code made from it is one rounding of y.
__device__ __forceinline__ float round_odd(double y) {
  const float f = (float)y;
  const double d = (double)f;
  if (d == y) return f;
  uint32_t b = __float_as_uint(f);
  if (fabs(d) > fabs(y)) b -= 1;
  return __uint_as_float(b | 1u);
}

// The rotated rows: q as the unquantised path rotates it (fp32, one rounding to
// T; the same bits), k in 64 bits -- its products are exact there, and fp64 adds
// run at the fp32 rate -- so that its codes are one rounding of the rotation and
// do not depend on how the product is fused; v as it is.
template <typename T, int CODE, int DH>
__global__ __launch_bounds__(kQThreads) void qkv_rope_append_q_kernel(
    const T* __restrict__ qkv, int64_t ldq, const int32_t* __restrict__ pos, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, int tab_rows, const int64_t* __restrict__ flat_row, T* __restrict__ q_out,
    uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, uint8_t* __restrict__ ke, uint8_t* __restrict__ ve,
    int64_t block_rows, int n, int H, int Hkv) {
  constexpr int LPR = DH / 8;
  const int heads = H + 2 * Hkv;
  const int64_t unit = ((int64_t)blockIdx.x * kQThreads + threadIdx.x) / LPR;  // (token, head of q | k | v)
  const int sub = threadIdx.x % LPR;
  const int i = (int)(unit / heads);
  if (i >= n) return;
  const int head = (int)(unit - (int64_t)i * heads);
  float x[8];
  load8(qkv + i * ldq + head * DH + 8 * sub, x);
  if (head >= H + Hkv) {
    write_row<CODE, LPR>(x, sub, kv_offset(flat_row[i], head - H - Hkv, Hkv, DH, block_rows), vc, ve);
    return;
  }
  int p = pos[i];
  p = p < 0 ? 0 : (p >= tab_rows ? tab_rows - 1 : p);
  float c[4], s[4], y[8];
  Elem<float>::unpack(ld16(cos_t + (int64_t)p * (DH / 2) + 4 * sub), c);
  Elem<float>::unpack(ld16(sin_t + (int64_t)p * (DH / 2) + 4 * sub), s);
  if (head < H) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[2 * j] = fmaf(x[2 * j], c[j], -(x[2 * j + 1] * s[j]));
      y[2 * j + 1] = fmaf(x[2 * j], s[j], x[2 * j + 1] * c[j]);
    }
    store8(q_out + ((int64_t)i * H + head) * DH + 8 * sub, y);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double a = x[2 * j], b = x[2 * j + 1], cd = c[j], sd = s[j];
    y[2 * j] = round_odd(a * cd - b * sd);
    y[2 * j + 1] = round_odd(a * sd + b * cd);
  }
  write_row<CODE, LPR>(y, sub, kv_offset(flat_row[i], head - H, Hkv, DH, block_rows), kc, ke);
}

template <typename T, int CODE, int DH>
__global__ __launch_bounds__(kQThreads) void kv_read_q_kernel(const uint8_t* __restrict__ kc,
                                                              const uint8_t* __restrict__ vc,
                                                              const uint8_t* __restrict__ ke,
                                                              const uint8_t* __restrict__ ve, int64_t block_rows,
                                                              const int64_t* __restrict__ flat_row,
                                                              T* __restrict__ k_out, T* __restrict__ v_out, int n,
                                                              int Hkv) {
  constexpr int LPR = DH / 8;
  const int64_t unit = ((int64_t)blockIdx.x * kQThreads + threadIdx.x) / LPR;
  const int sub = threadIdx.x % LPR;
  const int i = (int)(unit / (2 * Hkv));
  if (i >= n) return;
  const int r = (int)(unit - (int64_t)i * 2 * Hkv);
  const bool isv = r >= Hkv;
  const int h = isv ? r - Hkv : r;
  const int64_t off = kv_offset(flat_row[i], h, Hkv, DH, block_rows);
  const uint2 w = *reinterpret_cast<const uint2*>((isv ? vc : kc) + off + 8 * sub);
  const float sc = code_scale((isv ? ve : ke)[off / DH]);
  float x[8];
  decode4<CODE>(w.x, x);
  decode4<CODE>(w.y, x + 4);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= sc;
  store8((isv ? v_out : k_out) + ((int64_t)i * Hkv + h) * DH + 8 * sub, x);
}

// Workgroups over `units` rows of Dh values; 0 if they are past the grid, whose threads
// in x stay below 2^32.
static unsigned q_grid(int64_t units, int Dh) {
  const int64_t wgs = (units * (Dh / 8) + kQThreads - 1) / kQThreads;
  return wgs * kQThreads <= 0xffffffffll ? (unsigned)wgs : 0u;
}

// Runs f<T, CODE, DH>() for the run-time type, code and head size (checked before).
template <typename F>
static void q_dispatch(int dtype, int code, int Dh, F f) {
#define WFD_Q_CASE(TT, DT, CODE)                                                                      \
  if (dtype == DT && code == CODE) {                                                                  \
    if (Dh == 64) f(TT{}, std::integral_constant<int, CODE>{}, std::integral_constant<int, 64>{});    \
    else f(TT{}, std::integral_constant<int, CODE>{}, std::integral_constant<int, 128>{});            \
  }
  WFD_Q_CASE(bf16_t, kBF16, WFD_E4M3)
  WFD_Q_CASE(bf16_t, kBF16, WFD_INT8)
  WFD_Q_CASE(float, kF32, WFD_E4M3)
  WFD_Q_CASE(float, kF32, WFD_INT8)
#undef WFD_Q_CASE
}

static int check_dtype(const char* what, int dtype) {
  if (dtype == kBF16 || dtype == kF32) return kOk;
  set_error("%s: unsupported dtype %d", what, dtype);
  return kUnsupported;
}

}  // namespace wfd

extern "C" {

int wfd_kv_append_q(const void* k, int64_t ldk, const void* v, int64_t ldv, void* k_codes, void* v_codes,
                    uint8_t* k_exp, uint8_t* v_exp, int code, int64_t kv_block_rows, const int64_t* flat_row, int n,
                    int Hkv, int Dh, int dtype, hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_kv_append_q";
  if (int rc = check_qcache(me, n, Hkv, Dh, code, kv_block_rows)) return rc;
  if (int rc = check_dtype(me, dtype)) return rc;
  if (ldk < (int64_t)Hkv * Dh || ldv < (int64_t)Hkv * Dh) {
    set_error("%s: row pitch ldk=%lld ldv=%lld below Hkv * Dh = %d", me, (long long)ldk, (long long)ldv, Hkv * Dh);
    return kBadArg;
  }
  if (n == 0) return kOk;
  if (!k || !v || !k_codes || !v_codes || !k_exp || !v_exp || !flat_row) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  const int esz = dtype == kBF16 ? 2 : 4;
  if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)(ldk * esz) | (uintptr_t)(ldv * esz)) & 15) ||
      (((uintptr_t)k_codes | (uintptr_t)v_codes) & 15)) {
    set_error("%s: k, v, their row pitches and the codes must be 16-byte aligned", me);
    return kBadArg;
  }
  const unsigned grid = q_grid((int64_t)n * Hkv * (dtype == kBF16 ? 1 : 2), Dh);
  if (!grid) {
    set_error("%s: n=%d Hkv=%d beyond the grid", me, n, Hkv);
    return kUnsupported;
  }
  q_dispatch(dtype, code, Dh, [&](auto t, auto c, auto d) {
    using T = decltype(t);
    hipLaunchKernelGGL((kv_append_q_kernel<T, decltype(c)::value, decltype(d)::value>), dim3(grid), dim3(kQThreads),
                       0, stream, (const T*)k, ldk, (const T*)v, ldv, (uint8_t*)k_codes, (uint8_t*)v_codes, k_exp,
                       v_exp, kv_block_rows, flat_row, n, Hkv);
  });
  return launch_status(me);
}

int wfd_qkv_rope_append_q(const void* qkv, int64_t ldq, const int32_t* pos, const float* rope_cos,
                          const float* rope_sin, int rope_rows, const int64_t* flat_row, void* q_out, void* k_codes,
                          void* v_codes, uint8_t* k_exp, uint8_t* v_exp, int code, int64_t kv_block_rows, int n, int H,
                          int Hkv, int Dh, int dtype, hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_qkv_rope_append_q";
  if (int rc = check_qcache(me, n, Hkv, Dh, code, kv_block_rows)) return rc;
  if (int rc = check_dtype(me, dtype)) return rc;
  if (H <= 0 || H > kMaxHeads || rope_rows <= 0 || ldq < ((int64_t)H + 2 * (int64_t)Hkv) * Dh) {
    set_error("%s: bad shape H=%d Hkv=%d Dh=%d rope_rows=%d ldq=%lld", me, H, Hkv, Dh, rope_rows, (long long)ldq);
    return kBadArg;
  }
  if (n == 0) return kOk;
  if (!qkv || !pos || !rope_cos || !rope_sin || !flat_row || !q_out || !k_codes || !v_codes || !k_exp || !v_exp) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  const int esz = dtype == kBF16 ? 2 : 4;
  if (((uintptr_t)qkv | (uintptr_t)(ldq * esz) | (uintptr_t)rope_cos | (uintptr_t)rope_sin | (uintptr_t)q_out |
       (uintptr_t)k_codes | (uintptr_t)v_codes) & 15) {
    set_error("%s: qkv, its row pitch, the tables, q_out and the codes must be 16-byte aligned", me);
    return kBadArg;
  }
  const unsigned grid = q_grid((int64_t)n * ((int64_t)H + 2 * (int64_t)Hkv), Dh);
  if (!grid) {
    set_error("%s: n=%d H=%d Hkv=%d beyond the grid", me, n, H, Hkv);
    return kUnsupported;
  }
  q_dispatch(dtype, code, Dh, [&](auto t, auto c, auto d) {
    using T = decltype(t);
    hipLaunchKernelGGL((qkv_rope_append_q_kernel<T, decltype(c)::value, decltype(d)::value>), dim3(grid),
                       dim3(kQThreads), 0, stream, (const T*)qkv, ldq, pos, rope_cos, rope_sin, rope_rows, flat_row,
                       (T*)q_out, (uint8_t*)k_codes, (uint8_t*)v_codes, k_exp, v_exp, kv_block_rows, n, H, Hkv);
  });
  return launch_status(me);
}

int wfd_kv_read_q(const void* k_codes, const void* v_codes, const uint8_t* k_exp, const uint8_t* v_exp, int code,
                  int64_t kv_block_rows, const int64_t* flat_row, void* k_out, void* v_out, int n, int Hkv, int Dh,
                  int dtype, hipStream_t stream) {
  using namespace wfd;
  const char* me = "wfd_kv_read_q";
  if (int rc = check_qcache(me, n, Hkv, Dh, code, kv_block_rows)) return rc;
  if (int rc = check_dtype(me, dtype)) return rc;
  if (n == 0) return kOk;
  if (!k_codes || !v_codes || !k_exp || !v_exp || !flat_row || !k_out || !v_out) {
    set_error("%s: null pointer argument", me);
    return kBadArg;
  }
  if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15) {
    set_error("%s: the codes, k_out and v_out must be 16-byte aligned", me);
    return kBadArg;
  }
  const unsigned grid = q_grid((int64_t)n * 2 * Hkv, Dh);
  if (!grid) {
    set_error("%s: n=%d Hkv=%d beyond the grid", me, n, Hkv);
    return kUnsupported;
  }
  q_dispatch(dtype, code, Dh, [&](auto t, auto c, auto d) {
    using T = decltype(t);
    hipLaunchKernelGGL((kv_read_q_kernel<T, decltype(c)::value, decltype(d)::value>), dim3(grid), dim3(kQThreads), 0,
                       stream, (const uint8_t*)k_codes, (const uint8_t*)v_codes, k_exp, v_exp, kv_block_rows,
                       flat_row, (T*)k_out, (T*)v_out, n, Hkv);
  });
  return launch_status(me);
}

}  // extern "C"
