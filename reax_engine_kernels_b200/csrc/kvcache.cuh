// Quantised key/value cache: rows are quantised as they are written (reax_kv_write) and read back (reax_kv_read), sm_100a.
//
// A row is the D values of one (token, key/value head).  With amax = max |x_d| and n the least integer >= -127 with
// amax <= 448 * 2^n (448 = the largest e4m3 value), it is stored as e4m3(x_d / 2^n) and the byte n + 127.  A power of two
// costs nothing in precision (e4m3 is a floating type) and makes both directions exact but for the one rounding to
// e4m3: x / 2^n and e4m3 * 2^n only move an exponent, and an e4m3 value fits bf16's 8 bits.  A row with a value that is
// not finite is stored as zeros with byte 255 and reads back as NaN, so no e4m3 NaN code is ever stored.
//
// Layout: values [pages][H][page][D] bytes, exponents [pages][H][page] bytes (both with any page and head stride), so that the
// rows of one page and head are contiguous for the attention kernel.
//
// HBM-bound: 2 D bytes read and D + 1 written per row (write), the reverse (read).  A thread owns 16 values (two 16-byte
// loads, one 16-byte store), D / 16 lanes share a row; a CTA handles consecutive tokens of one head, so that its stores
// fall in whole pages.  One row a thread; two in a large write (four: fewer CTAs fit, 73 us for the write below).  32768
// tokens x 8 heads of 256: written in 61 us, read back in 66, 6.4 and 6.0 TB/s.
#pragma once
#include "common.cuh"

namespace reax {

constexpr int KV_THREADS = 128;

struct KvArgs {
  const uint16_t *k, *v;  // write: source rows; read: unused
  uint16_t *ko, *vo;      // read: destination rows
  long long sT, sH, vT, vH;  // token / head strides of k and v (or ko and vo), elements
  uint8_t *kc, *ke, *vc, *ve;
  long long cP, cH, eP, eH;  // page / head strides of the values and of the exponents, bytes
  const long long* slots;
  long long rows;  // pages * page
  int T, page, shift;  // shift: log2(page), or -1 where page is not a power of two
};

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

// four fp32 -> four e4m3 bytes, round to nearest even (the inputs never exceed 448)
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
// two e4m3 bytes -> f16x2 (exact)
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint16_t b) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(b));
  return r;
}
// 2^(b - 127) of an exponent byte; 255 is NaN, 0 the subnormal 2^-127
__device__ __forceinline__ float pow2_byte(uint32_t b) {
  return __uint_as_float(b == 255u ? 0x7fc00000u : b == 0u ? 0x00400000u : b << 23);
}

// Row of a slot, or -1 where the row is skipped (a negative slot; one past the end, which is also reported).
__device__ __forceinline__ long long kv_slot(const KvArgs& a, int t) {
  const long long s = a.slots[t];
  if (s >= a.rows) {
    record_status(ST_BAD_SLOT);
    return -1;
  }
  return s;
}

// Page and offset of a slot.  A 64-bit division costs more than all else a thread does for a row.
__device__ __forceinline__ long long kv_page(const KvArgs& a, long long s, int& off) {
  const long long pg = a.shift >= 0 ? s >> a.shift : s / a.page;
  off = (int)(s - pg * a.page);
  return pg;
}

// grid (token tiles, H, 2: k / v)
template <int D, int R>
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(KvArgs a) {
  constexpr int LPR = D / 16, RPB = KV_THREADS / LPR;  // lanes per row, rows per CTA and pass
  const int sub = threadIdx.x % LPR, row = threadIdx.x / LPR, h = blockIdx.y;
  const bool is_v = blockIdx.z;
  const uint16_t* src = (is_v ? a.v : a.k) + h * (is_v ? a.vH : a.sH) + sub * 16;
  const long long sT = is_v ? a.vT : a.sT;
  const long long t0 = (long long)blockIdx.x * (RPB * R) + row;
  pdl_wait();
  uint4 x[R][2];
  long long at[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const long long t = t0 + i * RPB;
    at[i] = -1;
    x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
    if (t < a.T) {
      const uint4* p = reinterpret_cast<const uint4*>(src + t * sT);
      x[i][0] = *p;
      x[i][1] = p[1];
      at[i] = kv_slot(a, (int)t);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max_u16x2(m, w[e] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    // amax = 1.f * 2^(e - 127): n + 127 = e - 8, one more where 1.f > 1.75.  A subnormal amax has e = 0.
    const int e = (int)(m >> 7);
    const int byte = e == 255 ? 255 : max(0, e - 8 + ((m & 0x7fu) > 0x60u));
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);  // 2^-n
    uint4 y = make_uint4(0, 0, 0, 0);
    if (byte != 255) {
      uint32_t z[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        z[j] = pack_e4m3(bf_lo(w[2 * j]) * inv, bf_hi(w[2 * j]) * inv, bf_lo(w[2 * j + 1]) * inv, bf_hi(w[2 * j + 1]) * inv);
      y = make_uint4(z[0], z[1], z[2], z[3]);
    }
    if (at[i] >= 0) {
      int off;
      const long long pg = kv_page(a, at[i], off);
      __stcs(reinterpret_cast<uint4*>((is_v ? a.vc : a.kc) + pg * a.cP + h * a.cH + (long long)off * D + sub * 16), y);
      if (sub == 0) ((is_v ? a.ve : a.ke) + pg * a.eP + h * a.eH)[off] = (uint8_t)byte;
    }
  }
}

// bf16 bits of e4m3 * 2^n for two values
__device__ __forceinline__ uint32_t dequant2(uint32_t two, float scale) {
  const uint32_t f = e4m3x2_f16x2((uint16_t)two);
  float lo, hi;
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(lo), "=f"(hi) : "r"(f));
  return pack_bf16(lo * scale, hi * scale);
}

// grid (token tiles, H, 2: k / v)
template <int D>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(KvArgs a) {
  constexpr int LPR = D / 16, RPB = KV_THREADS / LPR;
  const int sub = threadIdx.x % LPR, h = blockIdx.y;
  const bool is_v = blockIdx.z;
  const long long t = (long long)blockIdx.x * RPB + threadIdx.x / LPR;
  pdl_wait();
  if (t >= a.T) return;
  const long long at = kv_slot(a, (int)t);
  uint4 x = make_uint4(0, 0, 0, 0);
  uint32_t ex = 0;
  if (at >= 0) {
    int off;
    const long long pg = kv_page(a, at, off);
    x = __ldcs(reinterpret_cast<const uint4*>((is_v ? a.vc : a.kc) + pg * a.cP + h * a.cH + (long long)off * D + sub * 16));
    ex = ((is_v ? a.ve : a.ke) + pg * a.eP + h * a.eH)[off];
  }
  const float s = pow2_byte(ex);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t y[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[2 * j] = dequant2(w[j] & 0xffffu, s);
    y[2 * j + 1] = dequant2(w[j] >> 16, s);
  }
  uint4* p = reinterpret_cast<uint4*>((is_v ? a.vo : a.ko) + t * (is_v ? a.vT : a.sT) + h * (is_v ? a.vH : a.sH) + sub * 16);
  __stcs(p, make_uint4(y[0], y[1], y[2], y[3]));
  __stcs(p + 1, make_uint4(y[4], y[5], y[6], y[7]));
}

}  // namespace reax

namespace reax_host {

inline int page_shift(int page) { return page > 0 && !(page & (page - 1)) ? __builtin_ctz(page) : -1; }

// 0, or the refusal's code: -3 head dimension, -2 page size, -1 pointers and strides
inline int kv_check(const reax::KvArgs& a, const void* x, const void* y, int H, int D, long long pages) {
  if (D != 128 && D != 256) return -3;
  if (a.page <= 0 || a.page % 16 || pages < 0 || pages > (1LL << 40) / a.page) return -2;
  if (a.T < 0 || H <= 0 || H > 65535) return -1;
  if (a.T > 0 && (!x || !y || !a.kc || !a.ke || !a.vc || !a.ve || !a.slots)) return -1;
  if (((uintptr_t)x | (uintptr_t)y | (uintptr_t)a.kc | (uintptr_t)a.vc) & 15) return -1;
  if ((a.sT | a.sH | a.vT | a.vH) & 7) return -1;
  if ((a.cP | a.cH) & 15) return -1;
  return 0;
}

template <bool WRITE, int D>
inline int kv_go(const reax::KvArgs& a, int H, cudaStream_t st) {
  if (a.T == 0) return 0;
  constexpr int RPB = reax::KV_THREADS / (D / 16);
  int dev = 0;
  cudaGetDevice(&dev);
  // The write takes two rows a thread from ten waves of CTAs on (16 fit an SM), where HBM is the bound: 32768 tokens x 8 heads of 256
  // in 61.4 us, 64.5 with one; 8192 x 8 heads of 128, which the L2 takes in, in 9.9 with one, 10.5 with two.
  const int r = WRITE && (long long)((a.T + RPB - 1) / RPB) * H * 2 > 160LL * device_sms(dev) ? 2 : 1;
  const dim3 grid((a.T + RPB * r - 1) / (RPB * r), H, 2);
  void (*kernel)(reax::KvArgs) = !WRITE ? reax::kv_read_kernel<D> : r == 1 ? reax::kv_write_kernel<D, 1> : reax::kv_write_kernel<D, 2>;
  return launch_dependent(kernel, grid, reax::KV_THREADS, 0, true, st, 1, a);
}

}  // namespace reax_host

#define REAX_DEFINE_KV_EXPORTS()                                                                                       \
  REAX_API int reax_kv_write(const void* k, long long ksT, long long ksH, const void* v, long long vsT, long long vsH,    \
                             void* kc, void* ke, void* vc, void* ve, long long csP, long long csH, long long esP,        \
                             long long esH, const long long* slots, int T, int H, int D, int page, long long pages,      \
                             void* stream) {                                                                            \
    reax::KvArgs a{(const uint16_t*)k, (const uint16_t*)v, nullptr, nullptr, ksT, ksH, vsT, vsH, (uint8_t*)kc,             \
                   (uint8_t*)ke, (uint8_t*)vc, (uint8_t*)ve, csP, csH, esP, esH, slots, pages * page, T, page,                    \
                   reax_host::page_shift(page)};                                                                          \
    if (int rc = reax_host::kv_check(a, k, v, H, D, pages)) return rc;                                                    \
    return D == 128 ? reax_host::kv_go<true, 128>(a, H, (cudaStream_t)stream)                                             \
                    : reax_host::kv_go<true, 256>(a, H, (cudaStream_t)stream);                                            \
  }                                                                                                                      \
  REAX_API int reax_kv_read(void* k, long long ksT, long long ksH, void* v, long long vsT, long long vsH, const void* kc, \
                            const void* ke, const void* vc, const void* ve, long long csP, long long csH, long long esP, \
                            long long esH, const long long* slots, int T, int H, int D, int page, long long pages,       \
                            void* stream) {                                                                             \
    reax::KvArgs a{nullptr, nullptr, (uint16_t*)k, (uint16_t*)v, ksT, ksH, vsT, vsH, (uint8_t*)kc, (uint8_t*)ke,           \
                   (uint8_t*)vc, (uint8_t*)ve, csP, csH, esP, esH, slots, pages * page, T, page,                                  \
                   reax_host::page_shift(page)};                                                                          \
    if (int rc = reax_host::kv_check(a, k, v, H, D, pages)) return rc;                                                    \
    return D == 128 ? reax_host::kv_go<false, 128>(a, H, (cudaStream_t)stream)                                            \
                    : reax_host::kv_go<false, 256>(a, H, (cudaStream_t)stream);                                           \
  }
