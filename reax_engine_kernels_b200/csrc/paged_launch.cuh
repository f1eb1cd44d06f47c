// Host side of reax_fmha_paged: how the keys are cut, which kernels run, argument checks, the exported entry points.
#pragma once
#include "paged.cuh"
#include "prefix.cuh"

namespace reax_host {

struct PagedPlan {
  int chunk, splits, cluster, pchunk, psplits;
};
inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Whether the prefix goes to prefix_kernel (128 rows a CTA): from the second group of 16 rows on paged_kernel would read it twice.
// A prefix of 32768 keys, 8 heads of 128, 4 rows a sequence, the whole call: 4 sequences (16 rows) 29 us by paged_kernel, 41 by
// prefix_kernel; 8: 50 and 44; 32: 124 and 48.  Of 1024 keys the two are within 0.5 us (head dim 256: paged_kernel 1 to 3 us ahead).
inline bool prefix_tiled(int B, int M) { return (long long)B * M > 16; }

// Chunks of the keys, from the shapes alone (the lengths are on the device, and a captured launch replays with others).
//  * Few CTAs: as many chunks, up to the 8 of a cluster, as fit the GPU twice over with 64 keys (16 for each warp) or more in
//    each, joined within the cluster; as long as a chunk then is no longer than 256 keys.  One sequence of 1024 keys (8 heads of
//    128): 6.3 us, against 8.5 with the join in a kernel of its own and 15.5 in one chunk; of 4096, where a chunk would be
//    512: 10.2 against 8.1.
//  * Otherwise fixed chunks, as many CTAs as make three waves when all sequences are full: short sequences then leave at once, and
//    long ones spread.  Even shares take 37 us where these take 25 (32 ragged sequences up to 2048 keys).  No chunk under D keys (heads of
//    128: 128 against 256 is 23.6 against 25.0 us for 32 sequences of up to 512 keys behind a prefix, 10.1 against 11.7 for a prefix of
//    1024 before 4 sequences, 20.6 against 20.0 for 8 of up to 4096; heads of 256, one sequence of 4096: 11.1 against 10.9);
//    none under 1024 where the sequences alone fill half the GPU (64 of up to 1024 keys: 26 -> 23 us), or under 256 behind a prefix,
//    where a join runs anyway (32 of up to 512 keys, heads of 256: 50.2 -> 45.5; 64 of up to 1024, heads of 128: 46.2 -> 42.8); no more than 32
//    chunks once they are two CTAs an SM (one sequence of 65536 keys: 42 us in 205 chunks, 32 in 32).
inline PagedPlan paged_plan(int B, int H, int M, int D, int P, int page, int Lp, int sms) {
  auto cut = [&](long long keys, long long units, int resident, int& chunk, int& splits) {
    const long long slots = (long long)sms * resident, floor = 2 * units > slots ? (Lp ? 256 : 1024) : D;
    const long long most = 2LL * sms > 32 * units ? (2LL * sms + units - 1) / units : 32;
    const long long three = (3 * slots + units - 1) / units, want = three < most ? three : most;
    const long long c = ((keys + want - 1) / want + 63) / 64 * 64;
    chunk = (int)(c < floor ? floor : c);
    splits = keys ? ceil_div(keys, chunk) : 0;
  };
  const int rows = M <= 8 ? 8 : 16, resident = M <= 8 ? (D == 256 ? 3 : 4) : (D == 256 ? 2 : 3);
  const long long keys = (long long)P * page, units = (long long)B * H * ceil_div(M, rows);
  PagedPlan p;
  cut(keys, units, resident, p.chunk, p.splits);
  if (p.splits == 0) p.splits = 1;  // no pages at all: one chunk without keys
  int s = 1;
  while (s < 8 && 2 * s * units <= 2LL * sms && keys >= 2 * s * 64) s *= 2;
  p.cluster = Lp == 0 && s > 1 && keys <= 256LL * s;
  if (p.cluster) p.splits = s;
  if (prefix_tiled(B, M)) {  // one CTA of 128 rows per SM; two tiles of 64 keys at least
    const long long tiles = (long long)H * ceil_div((long long)B * M, reax::PF_ROWS), want = tiles < sms ? sms / tiles : 1;
    const int c = ceil_div(ceil_div(Lp, want), reax::PF_BN) * reax::PF_BN;
    p.pchunk = c < 2 * reax::PF_BN ? 2 * reax::PF_BN : c;
    p.psplits = ceil_div(Lp, p.pchunk);
  } else {
    cut(Lp, (long long)H * ceil_div((long long)B * M, 16), D == 256 ? 2 : 3, p.pchunk, p.psplits);
  }
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
  const dim3 grid((unsigned)x, a.H, PRE ? 1 : a.B);
  return launch_dependent(reax::paged_kernel<D, RT, PRE>, grid, 128, C::SMEM, true, st, !PRE && a.cluster ? a.splits : 1, a);
}

template <int D>
inline int prefix_launch(const reax::PagedArgs& a, cudaStream_t st) {
  using C = reax::PrefixCfg<D>;
  static SmemAttr attr;
  if (ensure_smem(attr, reax::prefix_kernel<D>, C::SMEM, true) != cudaSuccess) return -4;
  const long long x = (long long)ceil_div((long long)a.B * a.M, reax::PF_ROWS) * a.psplits;
  if (x > 0x7fffffffLL) return -1;
  return launch_dependent(reax::prefix_kernel<D>, dim3((unsigned)x, a.H), reax::PF_THREADS, C::SMEM, true, st, 1, a);
}

// Up to 8 rows per (sequence, head), what a decode step has, go in one group of 8; more in CTAs of 16 rows.  With 16 for all:
// 8 sequences of 32768 keys, 4 rows, 8 heads of 256: 188 -> 227 us; 64 of up to 256 keys, heads of 128: 9.6 -> 15.3.
template <int D>
inline int paged_go(const reax::PagedArgs& a, cudaStream_t st) {
  if (a.psplits)
    if (int rc = prefix_tiled(a.B, a.M) ? prefix_launch<D>(a, st) : paged_launch<D, 2, true>(a, st)) return rc;
  if (int rc = a.M <= 8 ? paged_launch<D, 1, false>(a, st) : paged_launch<D, 2, false>(a, st)) return rc;
  if (a.splits + a.psplits > 1 && !a.cluster) {
    // Eight partial outputs ahead where all rows' CTAs fit the GPU at 64 registers (one sequence of 16384 keys, 32 rows: 15.9 us with
    // none, 15.5 with two, 14.3 with eight); two, in 32 registers, where they would not (64 sequences, 2048 rows: 21.2, 21.0 and 24.0)
    const long long rows = (long long)a.B * a.H * a.M;
    int dev = 0;
    cudaGetDevice(&dev);
    return launch_dependent(rows <= 8LL * device_sms(dev) ? reax::paged_join_kernel<D, 8> : reax::paged_join_kernel<D, 2>, dim3((unsigned)rows),
                            128, 0, true, st, 1, a);
  }
  return 0;
}

}  // namespace reax_host

// ------------------------------------------------------------------------------------------------
// exported entry points
// ------------------------------------------------------------------------------------------------
REAX_API int reax_fmha_paged_splits(int B, int H, int M, int D, int P, int page, int Lp) {
  if (int rc = reax_host::paged_check(B, H, M, 1, D, P, page, Lp)) return rc;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  const reax_host::PagedPlan p =
      reax_host::paged_plan(B > 0 ? B : 1, H, M > 0 ? M : 1, D, P, page, Lp, reax_host::device_sms(dev));
  return p.cluster ? 1 : p.splits + p.psplits;
}

REAX_API int reax_fmha_paged(const void* q, long long qsB, long long qsH, long long qsM, const void* kc, const void* ke,
                             const void* vc, const void* ve, long long csP, long long csH, long long esP, long long esH,
                             const int* table, long long tsB, const int* prefix, int prefix_len, const int* qpos, int G,
                             long long qpBs, void* o, long long osB, long long osH, long long osM, void* ws, float scale,
                             int B, int H, int M, int D, int P, int page, long long pages, void* stream) {
  const int Lp = prefix_len;
  if (int rc = reax_host::paged_check(B, H, M, G, D, P, page, Lp)) return rc;
  if (B == 0 || M == 0) return 0;
  if (!q || !qpos || !o || pages < 0 || (P > 0 && !table) || (Lp > 0 && !prefix)) return -1;
  if ((P > 0 || Lp > 0) && (!kc || !ke || !vc || !ve)) return -1;
  if (((uintptr_t)q | (uintptr_t)o | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)ke | (uintptr_t)ve | (uintptr_t)ws) & 15)
    return -1;
  if ((qsB | qsH | qsM | osB | osH | osM) & 7) return -1;
  if ((csP | csH | esP | esH) & 15) return -1;
  int dev = 0;
  cudaGetDevice(&dev);
  const reax_host::PagedPlan p = reax_host::paged_plan(B, H, M, D, P, page, Lp, reax_host::device_sms(dev));
  const int splits = p.cluster ? 1 : p.splits + p.psplits;  // partial results in the workspace
  if (splits > 1 && !ws) return -5;
  float* part = (float*)ws;
  reax::PagedArgs a{};
  a.q = (const uint16_t*)q, a.qB = qsB, a.qH = qsH, a.qM = qsM;
  a.kc = (const uint8_t*)kc, a.ke = (const uint8_t*)ke, a.vc = (const uint8_t*)vc, a.ve = (const uint8_t*)ve;
  a.cP = csP, a.cH = csH, a.eP = esP, a.eH = esH;
  a.table = table, a.tB = tsB, a.qpos = qpos, a.qpB = qpBs;
  a.o = (uint16_t*)o, a.oB = osB, a.oH = osH, a.oM = osM;
  a.part = part, a.lse = part ? part + (long long)splits * B * H * M * D : nullptr;
  a.prefix = Lp ? prefix : nullptr;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.B = B, a.H = H, a.M = M, a.G = G, a.P = P, a.page = page, a.shift = reax_host::page_shift(page), a.Lp = Lp;
  a.chunk = p.chunk, a.splits = p.splits, a.cluster = p.cluster, a.pchunk = p.pchunk, a.psplits = p.psplits;
  a.pages = pages;
  return D == 128 ? reax_host::paged_go<128>(a, (cudaStream_t)stream) : reax_host::paged_go<256>(a, (cudaStream_t)stream);
}
