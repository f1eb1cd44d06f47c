// Host side of reax_fmha_paged: how the keys are cut, which kernels run, argument checks, the exported entry points.
#pragma once
#include "paged.cuh"
#include "prefix.cuh"

namespace reax_host {

struct PagedPlan {
  int chunk, splits, pchunk, psplits;
};
inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Whether the prefix goes to prefix_kernel (128 rows a CTA): from the second group of 16 rows on paged_kernel would read it twice.
inline bool prefix_tiled(int B, int M) { return (long long)B * M > 16; }

// Chunks of the keys, from the shapes alone (the lengths are on the device, and a captured launch replays with others): as
// many CTAs as keep every SM at its resident count about three times over when all sequences are full, but no chunk under 256
// keys, 64 for each of the four warps.
inline PagedPlan paged_plan(int B, int H, int M, int D, int P, int page, int Lp, int sms) {
  auto cut = [&](long long keys, long long units, int resident, int& chunk, int& splits) {
    const long long want = (3LL * sms * resident + units - 1) / units;
    long long c = (keys + want - 1) / want;
    c = (c + 63) / 64 * 64;
    chunk = (int)(c < 256 ? 256 : c);
    splits = keys ? ceil_div(keys, chunk) : 0;
  };
  const int rows = M <= 8 ? 8 : 16, resident = M <= 8 ? (D == 256 ? 3 : 4) : (D == 256 ? 2 : 3);
  PagedPlan p;
  cut((long long)P * page, (long long)B * H * ceil_div(M, rows), resident, p.chunk, p.splits);
  if (prefix_tiled(B, M)) {  // one CTA of 128 rows per SM; two tiles of 64 keys at least
    const long long units = (long long)H * ceil_div((long long)B * M, reax::PF_ROWS), want = units < sms ? sms / units : 1;
    const int c = ceil_div(ceil_div(Lp, want), reax::PF_BN) * reax::PF_BN;
    p.pchunk = c < 2 * reax::PF_BN ? 2 * reax::PF_BN : c;
    p.psplits = ceil_div(Lp, p.pchunk);
  } else {
    cut(Lp, (long long)H * ceil_div((long long)B * M, 16), D == 256 ? 2 : 3, p.pchunk, p.psplits);
  }
  if (p.splits == 0) p.splits = 1;  // no pages at all: one chunk without keys
  return p;
}

inline int paged_check(int B, int H, int M, int G, int D, int P, int page, int Lp) {
  if (D != 128 && D != 256) return -3;
  if (page <= 0 || page % 16) return -2;
  if (B < 0 || B > 65535 || H <= 0 || H > 65535 || M < 0 || G <= 0 || P < 0 || Lp < 0) return -1;
  if ((long long)P * page > (1LL << 30) || Lp > (1 << 30) || (long long)B * M > (1LL << 30) || (long long)B * H * M > 0x7fffffffLL)
    return -1;
  return 0;
}

template <int D, int RT, bool PRE>
inline int paged_launch(const reax::PagedArgs& a, cudaStream_t st) {
  using C = reax::PagedCfg<D, RT>;
  static SmemAttr attr;
  if (ensure_smem(attr, reax::paged_kernel<D, RT, PRE>, C::SMEM, true) != cudaSuccess) return -4;
  const long long x = PRE ? (long long)ceil_div((long long)a.B * a.M, C::ROWS) * a.psplits : (long long)ceil_div(a.M, C::ROWS) * a.splits;
  if (x > 0x7fffffffLL) return -1;
  return launch_dependent(reax::paged_kernel<D, RT, PRE>, dim3((unsigned)x, a.H, PRE ? 1 : a.B), 128, C::SMEM, !PRE && a.psplits, st, a);
}

template <int D>
inline int prefix_launch(const reax::PagedArgs& a, cudaStream_t st) {
  using C = reax::PrefixCfg<D>;
  static SmemAttr attr;
  if (ensure_smem(attr, reax::prefix_kernel<D>, C::SMEM, true) != cudaSuccess) return -4;
  const long long x = (long long)ceil_div((long long)a.B * a.M, reax::PF_ROWS) * a.psplits;
  if (x > 0x7fffffffLL) return -1;
  reax::prefix_kernel<D><<<dim3((unsigned)x, a.H), reax::PF_THREADS, C::SMEM, st>>>(a);
  return (int)cudaGetLastError();
}

// Up to 8 rows per (sequence, head), what a decode step has, go in one group of 8; more in CTAs of 16 rows.
template <int D>
inline int paged_go(const reax::PagedArgs& a, cudaStream_t st) {
  if (a.psplits)
    if (int rc = prefix_tiled(a.B, a.M) ? prefix_launch<D>(a, st) : paged_launch<D, 2, true>(a, st)) return rc;
  if (int rc = a.M <= 8 ? paged_launch<D, 1, false>(a, st) : paged_launch<D, 2, false>(a, st)) return rc;
  if (a.splits + a.psplits > 1) {
    const dim3 rows((unsigned)((long long)a.B * a.H * a.M));
    return launch_dependent(a.M <= 8 ? reax::paged_join_kernel<D, 8> : reax::paged_join_kernel<D, 16>, rows, 128, 0, true, st, a);
  }
  return 0;
}

}  // namespace reax_host

#define REAX_DEFINE_PAGED_EXPORTS()                                                                                      REAX_API int reax_fmha_paged_splits(int B, int H, int M, int D, int P, int page, int Lp) {                                  if (int rc = reax_host::paged_check(B, H, M, 1, D, P, page, Lp)) return rc;                                              int dev = 0;                                                                                                             if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;                                                                         const reax_host::PagedPlan p = reax_host::paged_plan(B > 0 ? B : 1, H, M > 0 ? M : 1, D, P, page, Lp,                                                                         reax_host::device_sms(dev));                                        return p.splits + p.psplits;                                                                                           }                                                                                                                        REAX_API int reax_fmha_paged(const void* q, long long qsB, long long qsH, long long qsM, const void* kc, const void* ke,                                const void* vc, const void* ve, long long csP, long long csH, long long esP,                                             long long esH, const int* table, long long tsB, const int* prefix, int prefix_len,                                       const int* qpos, int G, long long qpBs, void* o, long long osB, long long osH,                                           long long osM, void* ws, float scale, int B, int H, int M, int D, int P, int page,                                       long long pages, void* stream) {                                                              const int Lp = prefix_len;                                                                                               if (int rc = reax_host::paged_check(B, H, M, G, D, P, page, Lp)) return rc;                                              if (B == 0 || M == 0) return 0;                                                                                          if (!q || !qpos || !o || pages < 0 || (P > 0 && !table) || (Lp > 0 && !prefix)) return -1;                                if ((P > 0 || Lp > 0) && (!kc || !ke || !vc || !ve)) return -1;                                                           if (((uintptr_t)q | (uintptr_t)o | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)ke | (uintptr_t)ve | (uintptr_t)ws) & 15)       return -1;                                                                                                             if ((qsB | qsH | qsM | osB | osH | osM) & 7) return -1;                                                                  if ((csP | csH | esP | esH) & 15) return -1;                                                                             int dev = 0;                                                                                                             cudaGetDevice(&dev);                                                                                                     const reax_host::PagedPlan p = reax_host::paged_plan(B, H, M, D, P, page, Lp, reax_host::device_sms(dev));               const int splits = p.splits + p.psplits;                                                                                 if (splits > 1 && !ws) return -5;                                                                                        float* part = (float*)ws;                                                                                                reax::PagedArgs a{(const uint16_t*)q, qsB, qsH, qsM, (const uint8_t*)kc, (const uint8_t*)ke, (const uint8_t*)vc,                             (const uint8_t*)ve, csP, csH, esP, esH, table, tsB, qpos, qpBs, (uint16_t*)o, osB, osH, osM, part,                         part ? part + (long long)splits * B * H * M * D : nullptr, Lp ? prefix : nullptr,                                        scale * 1.4426950408889634f, B, H, M, G, P, page, reax_host::page_shift(page), Lp, p.chunk,                              p.splits, p.pchunk, p.psplits, pages};                                                                 return D == 128 ? reax_host::paged_go<128>(a, (cudaStream_t)stream) : reax_host::paged_go<256>(a, (cudaStream_t)stream);   }
