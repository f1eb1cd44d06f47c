// Attention over the paged quantised cache (reax_fmha_paged): one or a few tokens per sequence, sm_100a.
//
//   o[b, h, r] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max),  over the keys j <= qpos[b, r / G]
//
// with k_j = e4m3 row * 2^nk_j and v_j = e4m3 row * 2^nv_j out of the sequence's pages (and, for positions below prefix_len, out
// of the pages that all sequences share).  Everything but the products' operands is fp32: scores,
// both running maxima, the sum and the accumulators.
//
// HBM-bound: every visible cache byte is read once per key/value head, for all of the head's rows together.  A CTA of four warps
// takes 8 or 16 rows of one (sequence, head) and a chunk of its keys; each warp takes every fourth group of 16 keys, streams them
// through its own cp.async ring (no barrier in the loop) and keeps its own sums; the four are merged through shared memory,
// up to eight chunks of a sequence through the distributed shared memory of their cluster, more (or a prefix) by
// paged_join_kernel.
//
// The products are transposed, S^T = K Q^T and O^T = V^T P^T, so that keys and value columns fill the 16 rows of an m16n8k16 and
// the 4 to 8 query rows of a decode step its 8 columns.  With query rows as the 16 (the first version of this kernel, 3.5 TB/s over
// a long cache of head dim 256) half of the products and accumulators were padding, and 8 warps fitted an SM.
//
// Operands are f16: every e4m3 value is exact in f16 (cvt.rn.f16x2.e4m3x2 runs at 128 values per clock per SM, the cache
// arrives at 22), q is scaled per row by a power of two so that its largest magnitude lies in [1, 2) (a bf16 has 8 bits, f16
// has 11, so a value loses bits only 2^-14 below the row's largest), and p keeps f16's 11 bits.  mma.sync is right here: the
// stream needs 180 of the 1024 multiply-adds per clock per SM that it sustains.
//
// The value row's power of two cannot be applied after the product, and p * 2^nv may leave f16's range, so p's partner
// carries it: with x_j the score in the log2 domain and p_j = 2^(x_j - m), P_j = p_j * 2^nv_j * 2^(m - m') feeds the product, while the
// sum takes p_j; the two references meet in one factor 2^(m' - m) at the end.  m and m' follow the maxima of x and x + nv lazily:
// they are raised to the maximum only when a p or P passes 2^8 (well within f16, and 2^-14 of the largest weight still is a
// normal number), which one vote per 16 keys finds out.  With both exponents taken for each score, and both references
// compared with it, a group of 16 keys took 373 instructions a warp at D = 128, a third of them for 4 scores a thread.
// A key's P is (p_j * 2^nv_j) * 2^(m - m') in that order: behind a best key with a row of zeros (nv = -127) the two powers' product
// is infinite, and p_j may be 0.  So keys with p_j under 2^-126 count as 0, and every other P that leaves the range raises m'.
//
// Fragments without shuffles: the k index of q . k may be permuted as long as q and k agree, so a thread takes 16 adjacent
// bytes of a key row (four k16 steps at once).  ldmatrix.m16n16.trans.b8 leaves four consecutive keys of a value column in a register,
// so the keys' order in P V is made to suit: row g of S^T is key 4 (g / 2) + g % 2 of its 16, row g + 8 the key two behind it.
// P^T goes from accumulator to B fragment by movmatrix.
#pragma once
#include <cuda_fp16.h>

#include "kvcache.cuh"

namespace reax {

struct PagedArgs {
  const uint16_t* q;
  long long qB, qH, qM;
  const uint8_t *kc, *ke, *vc, *ve;
  long long cP, cH, eP, eH;
  const int* table;  // [B][P]
  long long tB;
  const int* qpos;
  long long qpB;
  uint16_t* o;
  long long oB, oH, oM;
  float* part;   // [splits][rows][D] partial outputs, each divided by its own sum
  float* lse;    // [splits][rows] log2 of that sum, -inf where the chunk holds no visible key
  const int* prefix;  // page ids of the shared prefix, NULL without one
  float scale_log2;
  int B, H, M, G, P, page, shift, Lp;
  int chunk, splits;    // a sequence's own keys: keys per chunk, chunks
  int cluster;          // 1: the CTAs of one tile's chunks are a cluster and join their results themselves
  int pchunk, psplits;  // the prefix: keys per chunk, chunks
  long long pages;
};

// RT: groups of 8 query rows per CTA
template <int D, int RT>
struct PagedCfg {
  static constexpr int WARPS = 4, ROWS = 8 * RT, KT = 16;
  static constexpr int STAGES = D == 256 && RT == 1 ? 2 : 3;
  static constexpr int CTAS = RT == 1 ? (D == 256 ? 3 : 4) : (D == 256 ? 2 : 3);  // per SM
  static constexpr int TILE = KT * D;          // bytes of the K (or V) rows of one group of keys
  static constexpr int STAGE = 2 * TILE + 48;  // + both rows of exponents, + the validity word
  static constexpr int QP = 2 * D + 16;        // row pitch of q
  static constexpr int QBYTES = ROWS * QP;
  static constexpr int OP = D + 4;  // row pitch of a warp's merged accumulators, fp32
  static constexpr int RING = WARPS * STAGES * STAGE, MERGE = WARPS * ROWS * OP * 4;
  static constexpr int SMEM = QBYTES + (RING > MERGE ? RING : MERGE);
};

// 16-byte chunk of a row in shared memory.  Rows 4i and 4i + 1 (and the two behind them) must differ in bit 2 for the K reads (a
// quarter warp reads four chunks of each), all rows of a group of eight for ldmatrix.
__device__ __forceinline__ int paged_swz(int row) { return ((row & 1) << 2) | ((row >> 1) & 3); }

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// two 16 x 16 byte matrices (rows: lanes 0-15, 16-31), transposed: r[2 i] holds bytes 4 t .. + 3 of column g of the i-th, r[2 i + 1]
// of column g + 8
__device__ __forceinline__ void ldsm_b8_x2_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void cp_async16_full(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The reference of a row that has seen no key yet: anything passes it, and it weighs nothing beside a real one
constexpr float PAGED_NONE = -1e30f;
// A maximum for use as a subtrahend: -inf replaced
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// The keys of batch entry b that ROWS (8 or 16) rows from r0 on can see, over the sequence's own pages (positions from Lp on).
__device__ __forceinline__ int paged_limit(const PagedArgs& a, int b, int r) {
  return r < a.M ? max(a.qpos[b * a.qpB + r / a.G], -1) - a.Lp : -1 - a.Lp;
}
template <int ROWS>
__device__ __forceinline__ int paged_visible(const PagedArgs& a, int b, int r0, int lane) {
  int lim = paged_limit(a, b, r0 + (lane & (ROWS - 1)));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) lim = max(lim, __shfl_xor_sync(0xffffffffu, lim, o));
  return min(max(lim, -1), a.P * a.page - 1) + 1;
}

// Keys per chunk of a tile that sees n: fixed, or for a cluster even shares of 64 keys (16 for each warp) or more
__device__ __forceinline__ int paged_chunk(const PagedArgs& a, int n) {
  return a.cluster ? max(((n + a.splits - 1) / a.splits + 63) & ~63, 64) : a.chunk;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
  return x;
}

// q rows as f16 in shared memory, each scaled by a power of two; srow[r] takes it out again.  128 threads, 8 per row.
template <int D, int ROWS, int QP, typename RowPtr>
__device__ __forceinline__ void paged_load_q(char* sq, float* srow, RowPtr row_ptr, float scale_log2) {
  constexpr int LPR = 8, V = D / (8 * LPR);  // threads per row, 16-byte loads per thread
  const int row = threadIdx.x / LPR, sub = threadIdx.x % LPR;
  if (row >= ROWS) return;  // whole warps
  const uint16_t* p = row_ptr(row);
  uint4 x[V];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    x[i] = p ? *reinterpret_cast<const uint4*>(p + (i * LPR + sub) * 8) : make_uint4(0, 0, 0, 0);
    m = max_u16x2(m, max_u16x2(max_u16x2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                               max_u16x2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
  }
  m = max(m & 0xffffu, m >> 16);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  // 2^-e with e the exponent of the largest magnitude; rows that are zero, subnormal or not finite stay in a range
  // where the power of two is a normal number (an infinity or NaN stays one)
  const int e = min(max((int)(m >> 7), 2), 252);
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
  if (sub == 0) srow[row] = __uint_as_float((uint32_t)e << 23) * scale_log2;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = pack_f16(bf_lo(w[k]) * inv, bf_hi(w[k]) * inv);
    *reinterpret_cast<uint4*>(sq + row * QP + (i * LPR + sub) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

// Own keys (PRE = false): grid (row tiles * splits, H, B).  Prefix keys: grid (tiles of the batch's B * M rows * psplits, H).
template <int D, int RT, bool PRE>
__global__ void __launch_bounds__(128, PagedCfg<D, RT>::CTAS) paged_kernel(const __grid_constant__ PagedArgs a) {
  using C = PagedCfg<D, RT>;
  constexpr int ROWS = C::ROWS;
  constexpr bool QREG = RT == 1;  // q's fragments stay in registers
  extern __shared__ __align__(128) char smem[];
  __shared__ float srow[ROWS];
  __shared__ float sm[C::WARPS][3][ROWS];
  __shared__ float slse[ROWS];
  if (PRE || a.psplits == 0) pdl_wait();  // beside a prefix kernel, that one has waited
  if (PRE) pdl_launch();
  const int nsplit = PRE ? a.psplits : a.splits;
  const int h = blockIdx.y, split = blockIdx.x % nsplit, r0 = blockIdx.x / nsplit * ROWS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  // batch entry and row of the CTA's row i; r >= M: there is none
  auto row_of = [&](int i, int& b, int& r) {
    b = PRE ? (r0 + i) / a.M : blockIdx.z;
    r = PRE ? (r0 + i) % a.M : r0 + i;
    if (PRE && b >= a.B) b = 0, r = a.M;
  };
  const int n = PRE ? a.Lp : paged_visible<ROWS>(a, blockIdx.z, r0, lane);
  const int chunk = PRE ? a.pchunk : paged_chunk(a, n);
  const int c0 = min(split * chunk, n), c1 = min(n, c0 + chunk);
  const bool cluster = !PRE && a.cluster;
  const bool direct = !PRE && !cluster && a.psplits == 0 && n <= chunk;  // the only chunk writes the output itself
  if (c0 >= n && !(direct && split == 0) && !cluster) {
    if (!PRE) pdl_wait();
    return;
  }
  const int ntiles = (c1 - c0 + 15) >> 4;

  char* ring = smem + C::QBYTES + warp * (C::STAGES * C::STAGE);
  const uint32_t ring_u = smem_u32(ring);
  const int* table = PRE ? a.prefix : a.table + blockIdx.z * a.tB;
  const uint8_t *kb = a.kc + h * a.cH, *vb = a.vc + h * a.cH, *keb = a.ke + h * a.eH, *veb = a.ve + h * a.eH;

  // page of group i of this warp: its page id is loaded one group ahead of its use
  auto group_page = [&](int i, int& off) {
    const int j = c0 + (warp + C::WARPS * i) * 16;
    const int pi = a.shift >= 0 ? j >> a.shift : j / a.page;
    off = j - pi * a.page;
    return pi;
  };
  const int mine = ntiles > warp ? (ntiles - warp + C::WARPS - 1) / C::WARPS : 0;
  int next_id = 0, next_off = 0;
  if (mine > 0) next_id = table[group_page(0, next_off)];
  auto issue = [&](int i) {
    if (i < mine) {
      const long long pid = next_id;
      const int off = next_off;
      const bool ok = pid >= 0 && pid < a.pages;
      if (i + 1 < mine) next_id = table[group_page(i + 1, next_off)];
      const int valid = ok ? min(16, n - (c0 + (warp + C::WARPS * i) * 16)) : 0;
      const uint32_t st = ring_u + (i % C::STAGES) * C::STAGE;
      constexpr int CPR = D / 16;  // the 16 rows are contiguous in the page
      const long long base = (ok ? pid * a.cP + (long long)off * D : 0) + lane * 16;
      if (valid == 16) {
#pragma unroll
        for (int u = 0; u < CPR / 2; ++u) {
          const int idx = u * 32 + lane, row = idx / CPR, c = idx % CPR;
          const uint32_t dst = st + row * D + ((c ^ paged_swz(row)) << 4);
          cp_async16_full(dst, kb + base + u * 512);
          cp_async16_full(dst + C::TILE, vb + base + u * 512);
        }
      } else {
#pragma unroll
        for (int u = 0; u < CPR / 2; ++u) {
          const int idx = u * 32 + lane, row = idx / CPR, c = idx % CPR;
          const uint32_t dst = st + row * D + ((c ^ paged_swz(row)) << 4);
          cp_async16(dst, row < valid ? kb + base + u * 512 : kb, row < valid);
          cp_async16(dst + C::TILE, row < valid ? vb + base + u * 512 : vb, row < valid);
        }
      }
      if (lane < 2) {
        const long long es = ok ? pid * a.eP + off : 0;
        cp_async16(st + 2 * C::TILE + lane * 16, (lane ? veb : keb) + es, ok);
      }
      if (lane == 2) {
        *reinterpret_cast<int*>(ring + (i % C::STAGES) * C::STAGE + 2 * C::TILE + 32) = ok;
        if (!ok) record_status(ST_BAD_PAGE);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) issue(i);

  paged_load_q<D, ROWS, C::QP>(smem, srow,
                               [&](int r) -> const uint16_t* {
                                 int b, m;
                                 row_of(r, b, m);
                                 return m < a.M ? a.q + b * a.qB + h * a.qH + m * a.qM : nullptr;
                               },
                               a.scale_log2);
  __syncthreads();
  int lim[RT][2];  // rows 8 rt + 2 t, + 1
  float rs[RT][2];
  int least = 0x7fffffff;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      int b, m;
      row_of(rt * 8 + 2 * t + e, b, m);
      // rows past M see what there is, so that they do not make every group of keys a masked one
      lim[rt][e] = m < a.M ? min(paged_limit(a, b, m) + (PRE ? a.Lp : 0), n - 1) : n - 1;
      rs[rt][e] = srow[rt * 8 + 2 * t + e];
      least = min(least, lim[rt][e]);
    }
  // q's B fragments: thread (g, t) holds row g at 64 c + 16 t .. + 15, the k16 steps' words w at + 4 w
  uint4 qf[QREG ? D / 64 : 1][2];
  const char* qrow = smem + g * C::QP + t * 32;
  if (QREG) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) qf[c][x] = *reinterpret_cast<const uint4*>(qrow + c * 128 + x * 16);
  }

  float o[RT][D / 16][4];
  float m[RT][2], mv[RT][2], rho[RT][2], l[RT][2];  // rho = 2^(m - mv)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[rt][j][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) m[rt][e] = mv[rt][e] = PAGED_NONE, rho[rt][e] = 1.f, l[rt][e] = 0.f;
  }
  const int key = 4 * (g >> 1) + (g & 1);  // this thread's keys: key and key + 2
  // A row's chunk c ^ swz: the part of c that the unrolled loops count stays out of the XOR
  const int ksw = (t ^ (paged_swz(key) & 3)) << 4, kbit = (paged_swz(key) & 4) << 4;
  const int ksw2 = (t ^ (paged_swz(key + 2) & 3)) << 4, kbit2 = (paged_swz(key + 2) & 4) << 4;
  const int vrow = lane & 15, vsw = (lane >> 4) ^ paged_swz(vrow);
  int slot = 0;

  for (int i = 0; i < mine; ++i) {
    issue(i + C::STAGES - 1);
    cp_async_wait<C::STAGES - 1>();
    __syncwarp();
    const int j0 = c0 + (warp + C::WARPS * i) * 16;
    const char* st = ring + slot * C::STAGE;
    const bool ok = *reinterpret_cast<const int*>(st + 2 * C::TILE + 32);
    const char *kr0 = st + key * D + ksw, *kr1 = st + (key + 2) * D + ksw2;
    const uint32_t vr = ring_u + slot * C::STAGE + C::TILE + vrow * D;
    slot = slot + 1 == C::STAGES ? 0 : slot + 1;
    // ---- scores: 16 keys x 8 rows, two chains of k steps
    float s[RT][2][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[rt][0][e] = s[rt][1][e] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 k0 = *reinterpret_cast<const uint4*>(kr0 + ((c * 64) ^ kbit));
      const uint4 k1 = *reinterpret_cast<const uint4*>(kr1 + ((c * 64) ^ kbit2));
      const uint32_t kw0[4] = {k0.x, k0.y, k0.z, k0.w}, kw1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t ka[4] = {e4m3x2_f16x2((uint16_t)kw0[w]), e4m3x2_f16x2((uint16_t)kw1[w]),
                                e4m3x2_f16x2((uint16_t)(kw0[w] >> 16)), e4m3x2_f16x2((uint16_t)(kw1[w] >> 16))};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const uint4 q4 = QREG ? qf[QREG ? c : 0][w >> 1]
                                : *reinterpret_cast<const uint4*>(qrow + rt * 8 * C::QP + c * 128 + (w >> 1) * 16);
          mma_f16(s[rt][w & 1], ka, w & 1 ? q4.z : q4.x, w & 1 ? q4.w : q4.y);
        }
      }
    }
    // ---- weights; the exponent bytes of the thread's two keys (255, a NaN row, becomes an infinity)
    const char* meta = st + 2 * C::TILE;
    const uint32_t kx = *reinterpret_cast<const uint32_t*>(meta + (key & 12)) >> (8 * (g & 1));
    const uint32_t vx = *reinterpret_cast<const uint32_t*>(meta + 16 + (key & 12)) >> (8 * (g & 1));
    const float ks[2] = {__uint_as_float(max((kx << 23) & 0x7f800000u, 0x00400000u)), __uint_as_float(max((kx << 7) & 0x7f800000u, 0x00400000u))};
    const float vf[2] = {__uint_as_float(max((vx << 23) & 0x7f800000u, 0x00400000u)), __uint_as_float(max((vx << 7) & 0x7f800000u, 0x00400000u))};
    const bool rare = __any_sync(0xffffffffu, j0 + 15 > least || max3f(ks[0], ks[1], fmaxf(vf[0], vf[1])) == INFINITY) || !ok;
    const bool nan[2] = {fmaxf(ks[0], vf[0]) == INFINITY, fmaxf(ks[1], vf[1]) == INFINITY};
    float p[RT][2][2], pv[RT][2][2];  // [key][row]
    auto weigh = [&]() {  // returns whether a weight passes 2^8
      float top = 0.f;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = __fmaf_rn(s[rt][0][2 * r + e] + s[rt][1][2 * r + e], rs[rt][e] * ks[r], -m[rt][e]);
            p[rt][r][e] = ex2_approx(x);
            pv[rt][r][e] = (p[rt][r][e] * vf[r]) * rho[rt][e];  // vf * rho may pass fp32's range, and p be 0
          }
      if (rare) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!ok || j0 + key + 2 * r > lim[rt][e]) p[rt][r][e] = pv[rt][r][e] = 0.f;
              else if (nan[r]) p[rt][r][e] = pv[rt][r][e] = __uint_as_float(0x7fc00000u);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) top = max3f(top, p[rt][r][e], pv[rt][r][e]);
      return top > 256.f;
    };
    if (__any_sync(0xffffffffu, weigh())) {  // raise the references to the maxima
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float al[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = PAGED_NONE, my = PAGED_NONE;
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (!rare || (ok && !nan[r] && j0 + key + 2 * r <= lim[rt][e])) {
              const float x = (s[rt][0][2 * r + e] + s[rt][1][2 * r + e]) * (rs[rt][e] * ks[r]);
              mx = fmaxf(mx, x);
              my = fmaxf(my, x + __log2f(vf[r]));
            }
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
            my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, k));
          }
          mx = fmaxf(mx, m[rt][e]);
          my = fmaxf(fmaxf(my, mv[rt][e]), mx - 127.f);  // no less but by rounding; rho stays finite
          l[rt][e] *= ex2_approx(m[rt][e] - mx);
          al[e] = ex2_approx(mv[rt][e] - my);
          rho[rt][e] = ex2_approx(fminf(mx - my, 127.f));
          m[rt][e] = mx;
          mv[rt][e] = my;
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[rt][j][e] *= al[e & 1];
      }
      weigh();
    }
    uint32_t pb[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[rt][0] += p[rt][r][0];
        l[rt][1] += p[rt][r][1];
        pb[rt][r] = movmatrix(pack_f16(pv[rt][r][0], pv[rt][r][1]));
      }
    }
    // ---- o^T += V^T P^T
#pragma unroll
    for (int j = 0; j < D / 16; j += 2) {
      uint32_t v4[4];
      ldsm_b8_x2_trans(vr + ((j ^ vsw) << 4), v4);
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const uint32_t va[4] = {e4m3x2_f16x2((uint16_t)v4[2 * jj]), e4m3x2_f16x2((uint16_t)v4[2 * jj + 1]),
                                e4m3x2_f16x2((uint16_t)(v4[2 * jj] >> 16)), e4m3x2_f16x2((uint16_t)(v4[2 * jj + 1] >> 16))};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) mma_f16(o[rt][j + jj], va, pb[rt][0], pb[rt][1]);
      }
    }
    __syncwarp();  // the stage may be filled again
  }
  cp_async_wait<0>();
  if (!PRE) pdl_launch();

  // ---- merge the four warps
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) l[rt][e] += __shfl_xor_sync(0xffffffffu, l[rt][e], k);
      if (g == 0) {
        const int r = rt * 8 + 2 * t + e;
        sm[warp][0][r] = m[rt][e];
        sm[warp][1][r] = mv[rt][e];
        sm[warp][2][r] = l[rt][e];
      }
    }
  __syncthreads();  // all rings are drained: their space takes the accumulators, [warp][ROWS][OP] fp32
  float* so = reinterpret_cast<float*>(smem + C::QBYTES);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = rt * 8 + 2 * t + e;
      float top = PAGED_NONE;
#pragma unroll
      for (int w = 0; w < C::WARPS; ++w) top = fmaxf(top, sm[w][1][r]);
      const float f = ex2_approx(mv[rt][e] - top);
      // a NaN weight stays NaN; a warp without visible keys adds zeros
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        so[(warp * ROWS + r) * C::OP + 16 * j + g] = o[rt][j][e] * f;
        so[(warp * ROWS + r) * C::OP + 16 * j + 8 + g] = o[rt][j][2 + e] * f;
      }
    }
  __syncthreads();
  // The own keys' kernel runs beside the prefix's (none of its inputs come from there), and ends after it: so what is launched
  // behind it finds both results
  if (!PRE) pdl_wait();
  const int row = threadIdx.x >> 3, sub = threadIdx.x & 7;  // 8 threads a row
  const long long rows = (long long)a.B * a.H * a.M;
  if (row < ROWS) {
    int b, mr;
    row_of(row, b, mr);
    float top = PAGED_NONE, topv = PAGED_NONE, sum = 0.f;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) top = fmaxf(top, sm[w][0][row]), topv = fmaxf(topv, sm[w][1][row]);
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) sum += sm[w][2][row] * ex2_approx(sm[w][0][row] - top);
    const float half = ex2_approx(0.5f * (topv - top)), fac = half / sum;  // in two steps: 2^-127 is below what ex2 gives
    const float lse = sum == 0.f ? -INFINITY : top + log2f(sum);
    const long long at = (PRE ? a.splits + split : split) * rows + ((long long)b * a.H + h) * a.M + mr;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int d = (i * 8 + sub) * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = 0.f;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) v[e] += so[(w * ROWS + row) * C::OP + d + e];
        v[e] = sum == 0.f ? 0.f : v[e] * half * fac;
      }
      if (direct && mr < a.M)
        *reinterpret_cast<uint4*>(a.o + b * a.oB + h * a.oH + mr * a.oM + d) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      if (!direct && (cluster || mr < a.M)) {  // for the cluster in this CTA's shared memory, over the first warp's share
        float4* p = reinterpret_cast<float4*>(cluster ? so + row * C::OP + d : a.part + at * D + d);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
    if (sub == 0) {
      if (cluster) slse[row] = lse;
      else if (!direct && mr < a.M) a.lse[at] = lse;
    }
  }
  if (!cluster) return;

  // ---- join the cluster's chunks, four values of a row per thread
  cluster_sync_all();
  const uint32_t so_u = smem_u32(so), lse_u = smem_u32(slse);
  for (int x = split * 128 + threadIdx.x; x < ROWS * (D / 4); x += nsplit * 128) {
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    int b, mr;
    row_of(r, b, mr);
    if (mr >= a.M) continue;
    float w[8], top = -INFINITY, sum = 0.f;
    float4 p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < nsplit) {
        w[i] = ld_cluster_f32(mapa_shared(lse_u + r * 4, i));
        p[i] = ld_cluster_v4(mapa_shared(so_u + (r * C::OP + d) * 4, i));
        top = fmaxf(top, w[i]);
      }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < nsplit) {
        const float f = ex2_approx(w[i] - finite_or_zero(top));  // a NaN stays one
        sum += f;
        acc.x += f * p[i].x, acc.y += f * p[i].y, acc.z += f * p[i].z, acc.w += f * p[i].w;
      }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>(a.o + b * a.oB + h * a.oH + mr * a.oM + d) =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
  cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// Joins the chunks' partial outputs: one CTA per row; D / 4 threads take four values each, 128 / (D / 4) groups of them every other
// chunk.  AHEAD: partial outputs a thread asks for before the chunks' sums are compared.
template <int D, int AHEAD>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int TPG = D / 4, GROUPS = 128 / TPG;
  __shared__ float red[4], sum_s[GROUPS];
  __shared__ __align__(16) float acc_s[GROUPS][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = threadIdx.x / TPG, d = threadIdx.x % TPG * 4;
  const long long rows = (long long)a.B * a.H * a.M, R = blockIdx.x;
  const int r = (int)(R % a.M), h = (int)(R / a.M % a.H), b = (int)(R / a.M / a.H);
  const int n = paged_visible<16>(a, b, r & ~15, lane);  // the tile's, of 8 rows too: there are none behind them then
  pdl_wait();
  const int chunk = paged_chunk(a, n), mine = (n + chunk - 1) / chunk, total = mine + a.psplits;
  if (a.psplits == 0 && n <= chunk) return;  // written by its only chunk
  auto slot = [&](int i) { return (i < mine ? i : a.splits + i - mine) * rows + R; };
  // the first partial outputs, while the sums are compared
  float4 ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = grp + k * GROUPS;
    ahead[k] = i < total ? *reinterpret_cast<const float4*>(a.part + slot(i) * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float top = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x; i < total; i += 128) {
    const float x = a.lse[slot(i)];
    nan |= x != x;
    top = fmaxf(top, x);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  if (lane == 0) red[warp] = top;
  nan = __syncthreads_or(nan);
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ref = nan ? __uint_as_float(0x7fc00000u) : finite_or_zero(top);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = grp + k * GROUPS;
    const float w = i < total ? ex2_approx(a.lse[slot(i)] - ref) : 0.f;
    sum += w;
    acc.x += w * ahead[k].x, acc.y += w * ahead[k].y, acc.z += w * ahead[k].z, acc.w += w * ahead[k].w;
  }
#pragma unroll 8
  for (int i = grp + AHEAD * GROUPS; i < total; i += GROUPS) {
    const long long at = slot(i);
    const float w = ex2_approx(a.lse[at] - ref);
    const float4 x = *reinterpret_cast<const float4*>(a.part + at * D + d);
    sum += w;
    acc.x += w * x.x, acc.y += w * x.y, acc.z += w * x.z, acc.w += w * x.w;
  }
  *reinterpret_cast<float4*>(&acc_s[grp][d]) = acc;
  if (threadIdx.x % TPG == 0) sum_s[grp] = sum;
  __syncthreads();
  if (grp) return;
  sum = sum_s[0];
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float4 x = *reinterpret_cast<const float4*>(&acc_s[i][d]);
    acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
    sum += sum_s[i];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(a.o + b * a.oB + h * a.oH + r * a.oM + d) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

}  // namespace reax
