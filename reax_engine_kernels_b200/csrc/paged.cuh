// Attention over the paged quantised cache (reax_fmha_paged): one or a few tokens per sequence, sm_100a.
//
//   o[b, h, r] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max),  over the keys j <= qpos[b, r / G]
//
// with k_j = e4m3 row * 2^nk_j and v_j = e4m3 row * 2^nv_j out of the sequence's pages (and, for positions below prefix_len, out
// of the pages that all sequences share).  Everything but the products' operands is fp32: scores,
// both running maxima, the sum and the accumulators.
//
// HBM-bound: every visible cache byte is read once per key/value head, for all of the head's rows together.  A CTA of four warps
// takes 16 rows of one (sequence, head) and a chunk of its keys; each warp takes every fourth group of 16 keys, streams them
// through its own cp.async ring (no barrier in the loop) and keeps its own softmax; the four are merged through shared memory,
// the chunks by paged_join_kernel.  A sequence that fits one chunk is written by its only CTA.
//
// Operands are f16: every e4m3 value is exact in f16 (cvt.rn.f16x2.e4m3x2 runs at 128 values per clock per SM, the cache
// arrives at 22), q is scaled per row by a power of two so that its largest magnitude lies in [1, 2) (a bf16 has 8 bits, f16
// has 11, so a value loses bits only 2^-14 below the row's largest), and p keeps f16's 11 bits.  mma.sync is right here: with 16 rows the
// stream needs 360 of the 1024 multiply-adds per clock per SM that it sustains.
//
// The value row's power of two cannot be applied after the product, and p * 2^nv may leave f16's range, so p's partner
// carries it: with x_j the score in the log2 domain, P_j = 2^(x_j + nv_j - m'), m' the running maximum of x + nv, feeds the
// product, while the sum takes 2^(x_j - m); the two maxima meet in one factor 2^(m' - m) at the end.
//
// Fragments without shuffles: the k index of q . k may be permuted as long as q and k agree, so a thread takes 16 adjacent
// bytes of a key row (four k16 steps at once); and ldmatrix.trans on byte pairs leaves two adjacent value columns of two keys
// in a register, which one byte permute and two conversions turn into the fragments of the even and the odd column.
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
  int chunk, splits;    // the sequences' own keys: keys per chunk, chunks
  int pchunk, psplits;  // the same of the prefix
  long long pages;
};

template <int D>
struct PagedCfg {
  static constexpr int WARPS = 4, STAGES = 3, KT = 16;
  static constexpr int TILE = KT * D;                 // bytes of the K (or V) rows of one group of keys
  static constexpr int STAGE = 2 * TILE + 48;         // + both rows of exponents, + the validity word
  static constexpr int QBYTES = 16 * D * 2;
  static constexpr int SMEM = QBYTES + WARPS * STAGES * STAGE;
};

// 16-byte chunk of a row in shared memory.  Rows 2i and 2i + 1 must differ in bit 2 for the K reads (a quarter warp reads four
// chunks of each), all eight rows of a group for ldmatrix.
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
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Maximum of two rows' running values, -inf replaced for use as a subtrahend
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// The keys of batch entry b that 16 rows from r0 on can see, over the sequence's own pages (positions from Lp on).
__device__ __forceinline__ int paged_limit(const PagedArgs& a, int b, int r) {
  return r < a.M ? max(a.qpos[b * a.qpB + r / a.G], -1) - a.Lp : -1 - a.Lp;
}
__device__ __forceinline__ int paged_visible(const PagedArgs& a, int b, int r0, int lane) {
  int lim = paged_limit(a, b, r0 + (lane & 15));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) lim = max(lim, __shfl_xor_sync(0xffffffffu, lim, o));
  return min(max(lim, -1), a.P * a.page - 1) + 1;
}

// q rows as f16 A fragments in shared memory, [D / 64][4][32 lanes] x 16 bytes: thread (g, t) of block c and word w holds rows g
// and g + 8 at values 64 c + 16 t + 4 w .. + 3.  scale[r] takes the row's power of two out again.
template <int D, typename RowPtr>
__device__ __forceinline__ void paged_load_q(char* sq, float* srow, RowPtr row_ptr, float scale_log2) {
  constexpr int LPR = 8;  // threads per row, 128 threads
  const int row = threadIdx.x / LPR, sub = threadIdx.x % LPR;
  const uint16_t* p = row_ptr(row);
  constexpr int V = D / (8 * LPR);  // 16-byte loads per thread
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
    const int d = (i * LPR + sub) * 8;  // values d..d+3 are word w of thread t, d+4..d+7 the next word
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int dd = d + 4 * k, c = dd >> 6, t = (dd >> 4) & 3, wd = (dd >> 2) & 3;
      char* dst = sq + ((c * 4 + wd) * 32 + (row & 7) * 4 + t) * 16 + (row >> 3) * 4;
      *reinterpret_cast<uint32_t*>(dst) = pack_f16(bf_lo(w[2 * k]) * inv, bf_hi(w[2 * k]) * inv);            // a0 / a1
      *reinterpret_cast<uint32_t*>(dst + 8) = pack_f16(bf_lo(w[2 * k + 1]) * inv, bf_hi(w[2 * k + 1]) * inv);  // a2 / a3
    }
  }
}

// Own keys (PRE = false): grid (row tiles * splits, H, B).  Prefix keys: grid (tiles of the batch's B * M rows * psplits, H).
template <int D, bool PRE>
__global__ void __launch_bounds__(PagedCfg<D>::WARPS * 32, D == 256 ? 2 : 3) paged_kernel(const __grid_constant__ PagedArgs a) {
  using C = PagedCfg<D>;
  extern __shared__ __align__(128) char smem[];
  __shared__ float srow[16];
  __shared__ float sm[C::WARPS][3][16];
  const int nsplit = PRE ? a.psplits : a.splits, chunk = PRE ? a.pchunk : a.chunk;
  const int h = blockIdx.y, split = blockIdx.x % nsplit, r0 = blockIdx.x / nsplit * 16;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  // batch entry and row of the CTA's row i; r >= M: there is none
  auto row_of = [&](int i, int& b, int& r) {
    b = PRE ? (r0 + i) / a.M : blockIdx.z;
    r = PRE ? (r0 + i) % a.M : r0 + i;
    if (PRE && b >= a.B) b = 0, r = a.M;
  };
  const int n = PRE ? a.Lp : paged_visible(a, blockIdx.z, r0, lane);
  const int c0 = split * chunk, c1 = min(n, c0 + chunk);
  const bool direct = !PRE && a.psplits == 0 && n <= chunk;  // the only chunk writes the output itself
  if (c0 >= n && !(direct && split == 0)) return;
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
      const long long base = ok ? pid * a.cP + (long long)off * D : 0;
      constexpr int CPR = D / 16;
#pragma unroll
      for (int u = 0; u < CPR / 2; ++u) {
        const int idx = u * 32 + lane, row = idx / CPR, c = idx % CPR;
        const uint32_t dst = st + row * D + ((c ^ paged_swz(row)) << 4);
        const long long src = base + (row < valid ? row * D + c * 16 : 0);
        cp_async16(dst, kb + src, row < valid);
        cp_async16(dst + C::TILE, vb + src, row < valid);
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

  paged_load_q<D>(smem, srow,
                  [&](int r) -> const uint16_t* {
                    int b, m;
                    row_of(r, b, m);
                    return m < a.M ? a.q + b * a.qB + h * a.qH + m * a.qM : nullptr;
                  },
                  a.scale_log2);
  __syncthreads();
  int lim[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int b, m;
    row_of(g + 8 * i, b, m);
    lim[i] = paged_limit(a, b, m) + (PRE ? a.Lp : 0);
  }
  const float rs[2] = {srow[g], srow[g + 8]};

  float o[D / 16][2][4];
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][0][e] = o[j][1][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, mv[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int i = 0; i < mine; ++i) {
    issue(i + C::STAGES - 1);
    cp_async_wait<C::STAGES - 1>();
    __syncwarp();
    const int j0 = c0 + (warp + C::WARPS * i) * 16;
    const char* st = ring + (i % C::STAGES) * C::STAGE;
    // ---- scores of 16 keys: two n8 tiles, two chains of k steps each
    float s[2][2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][0][e] = s[nt][1][e] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      uint4 kx[2];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
        kx[nt] = *reinterpret_cast<const uint4*>(st + (nt * 8 + g) * D + (((c * 4 + t) ^ paged_swz(g)) << 4));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint4 qx = *reinterpret_cast<const uint4*>(smem + ((c * 4 + w) * 32 + lane) * 16);
        const uint32_t qa[4] = {qx.x, qx.y, qx.z, qx.w};
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const uint32_t kw = w == 0 ? kx[nt].x : w == 1 ? kx[nt].y : w == 2 ? kx[nt].z : kx[nt].w;
          mma_f16(s[nt][w & 1], qa, e4m3x2_f16x2((uint16_t)kw), e4m3x2_f16x2((uint16_t)(kw >> 16)));
        }
      }
    }
    // ---- scale, mask, both maxima
    const bool ok = *reinterpret_cast<const int*>(st + 2 * C::TILE + 32);
    float x[2][2][2], nv[2][2];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const uint32_t ek = *reinterpret_cast<const uint16_t*>(st + 2 * C::TILE + nt * 8 + 2 * t);
      const uint32_t ev = *reinterpret_cast<const uint16_t*>(st + 2 * C::TILE + 16 + nt * 8 + 2 * t);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ks = pow2_byte((ek >> (8 * e)) & 255u);
        const uint32_t vbyte = (ev >> (8 * e)) & 255u;
        nv[nt][e] = vbyte == 255u ? __uint_as_float(0x7fc00000u) : (float)((int)vbyte - 127);
        const int j = j0 + nt * 8 + 2 * t + e;
#pragma unroll
        for (int r = 0; r < 2; ++r)
          x[r][nt][e] = ok && j <= lim[r] && j < n ? (s[nt][0][2 * r + e] + s[nt][1][2 * r + e]) * (rs[r] * ks) : -INFINITY;
      }
    }
    float alpha[2];
    uint32_t pa[4];
    bool grew = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = fmaxf(fmaxf(x[r][0][0], x[r][0][1]), fmaxf(x[r][1][0], x[r][1][1]));
      float my = fmaxf(fmaxf(x[r][0][0] + nv[0][0], x[r][0][1] + nv[0][1]), fmaxf(x[r][1][0] + nv[1][0], x[r][1][1] + nv[1][1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 1));
      mx = fmaxf(m[r], fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)));
      my = fmaxf(mv[r], fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 2)));
      grew |= my != mv[r];
      const float ux = finite_or_zero(mx), uy = finite_or_zero(my);
      l[r] *= ex2_approx(m[r] - ux);
      alpha[r] = ex2_approx(mv[r] - uy);
      m[r] = mx;
      mv[r] = my;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        l[r] += ex2_approx(x[r][nt][0] - ux) + ex2_approx(x[r][nt][1] - ux);
        // a masked key's exponent may be any byte, NaN's too: its weight is 0, not 2^NaN
        const float p0 = x[r][nt][0] == -INFINITY ? 0.f : ex2_approx(x[r][nt][0] + nv[nt][0] - uy);
        const float p1 = x[r][nt][1] == -INFINITY ? 0.f : ex2_approx(x[r][nt][1] + nv[nt][1] - uy);
        pa[nt * 2 + r] = pack_f16(p0, p1);
      }
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[j][0][e] *= alpha[e >> 1];
          o[j][1][e] *= alpha[e >> 1];
        }
    }
    // ---- o += P V
    const uint32_t vrow = ring_u + (i % C::STAGES) * C::STAGE + C::TILE + (lane & 15) * D;
#pragma unroll
    for (int j = 0; j < D / 16; j += 2) {
      uint32_t v4[4];
      ldsm_x4_trans(vrow + (((j + (lane >> 4)) ^ paged_swz(lane & 7)) << 4), v4);
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const uint32_t lo = __byte_perm(v4[2 * jj], 0, 0x3120), hi = __byte_perm(v4[2 * jj + 1], 0, 0x3120);
        mma_f16(o[j + jj][0], pa, e4m3x2_f16x2((uint16_t)lo), e4m3x2_f16x2((uint16_t)hi));
        mma_f16(o[j + jj][1], pa, e4m3x2_f16x2((uint16_t)(lo >> 16)), e4m3x2_f16x2((uint16_t)(hi >> 16)));
      }
    }
    __syncwarp();  // the stage may be filled again
  }
  cp_async_wait<0>();

  // ---- merge the four warps
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (t == 0) {
      sm[warp][0][g + 8 * r] = m[r];
      sm[warp][1][g + 8 * r] = mv[r];
      sm[warp][2][g + 8 * r] = l[r];
    }
  }
  __syncthreads();  // all rings are drained: their space takes the accumulators, [warp][16][D + 4] fp32
  constexpr int OP = D + 4;
  float* so = reinterpret_cast<float*>(smem);
  static_assert(C::WARPS * 16 * OP * 4 <= C::SMEM, "the accumulators fit the ring");
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) top = fmaxf(top, sm[w][1][g + 8 * r]);
    const float f = ex2_approx(mv[r] - finite_or_zero(top));
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
      *reinterpret_cast<float4*>(so + (warp * 16 + g + 8 * r) * OP + 16 * j + 4 * t) =
          make_float4(o[j][0][2 * r] * f, o[j][1][2 * r] * f, o[j][0][2 * r + 1] * f, o[j][1][2 * r + 1] * f);
  }
  __syncthreads();
  const int row = threadIdx.x >> 3, sub = threadIdx.x & 7;  // 8 threads a row
  int b, mr;
  row_of(row, b, mr);
  if (mr >= a.M) return;
  float top = -INFINITY, topv = -INFINITY, sum = 0.f;
#pragma unroll
  for (int w = 0; w < C::WARPS; ++w) top = fmaxf(top, sm[w][0][row]), topv = fmaxf(topv, sm[w][1][row]);
#pragma unroll
  for (int w = 0; w < C::WARPS; ++w) sum += sm[w][2][row] * ex2_approx(sm[w][0][row] - finite_or_zero(top));
  const float fac = sum == 0.f ? 0.f : ex2_approx(finite_or_zero(topv) - finite_or_zero(top)) / sum;
  const long long R = ((long long)b * a.H + h) * a.M + mr, rows = (long long)a.B * a.H * a.M;
  const long long at = (PRE ? a.splits + split : split) * rows + R;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int d = (i * 8 + sub) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int w = 0; w < C::WARPS; ++w) v[e] += so[(w * 16 + row) * OP + d + e];
      v[e] = sum == 0.f ? 0.f : v[e] * fac;
    }
    if (direct) {
      *reinterpret_cast<uint4*>(a.o + b * a.oB + h * a.oH + mr * a.oM + d) =
          make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
      float4* p = reinterpret_cast<float4*>(a.part + at * D + d);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
  if (!direct && sub == 0) a.lse[at] = sum == 0.f ? -INFINITY : top + log2f(sum);
}

// Joins the chunks' partial outputs: one warp per row.
template <int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedArgs a) {
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.B * a.H * a.M, R = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (R >= rows) return;
  const int r = (int)(R % a.M), h = (int)(R / a.M % a.H), b = (int)(R / a.M / a.H);
  const int n = paged_visible(a, b, r & ~15, lane);
  if (a.psplits == 0 && n <= a.chunk) return;  // written by its only chunk
  const int mine = (n + a.chunk - 1) / a.chunk, total = mine + a.psplits;
  auto slot = [&](int i) { return i < mine ? i : a.splits + i - mine; };
  float top = -INFINITY;
  bool nan = false;
  for (int i = lane; i < total; i += 32) {
    const float x = a.lse[slot(i) * rows + R];
    nan |= x != x;
    top = fmaxf(top, x);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  if (__any_sync(0xffffffffu, nan)) top = __uint_as_float(0x7fc00000u);
  const float ref = finite_or_zero(top);
  constexpr int V = D / 32;
  float acc[V], sum = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < total; ++i) {
    const long long at = slot(i) * rows + R;
    const float w = ex2_approx(a.lse[at] - ref);
    sum += w;
    const float4* p = reinterpret_cast<const float4*>(a.part + at * D + lane * V);
#pragma unroll
    for (int e = 0; e < V / 4; ++e) {
      const float4 x = p[e];
      acc[4 * e] += w * x.x, acc[4 * e + 1] += w * x.y, acc[4 * e + 2] += w * x.z, acc[4 * e + 3] += w * x.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t y[V / 2];
#pragma unroll
  for (int e = 0; e < V / 2; ++e) y[e] = pack_bf16(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  uint16_t* out = a.o + b * a.oB + h * a.oH + r * a.oM + lane * V;
  if (V == 8) *reinterpret_cast<uint4*>(out) = make_uint4(y[0], y[1], y[V / 2 - 2], y[V / 2 - 1]);
  else *reinterpret_cast<uint2*>(out) = make_uint2(y[0], y[1]);
}

}  // namespace reax

namespace reax_host {

struct PagedPlan {
  int chunk, splits, pchunk, psplits;
};
inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Chunks of the keys, from the shapes alone (the lengths are on the device, and a captured launch replays with others): as
// many CTAs as keep every SM at its resident count about three times over when all sequences are full, but no chunk under 256
// keys, 64 for each of the four warps.
inline PagedPlan paged_plan(int B, int H, int M, int D, int P, int page, int Lp, int sms) {
  const int resident = D == 256 ? 2 : 3;
  auto cut = [&](long long keys, long long units, int& chunk, int& splits) {
    const long long want = (3LL * sms * resident + units - 1) / units;
    long long c = (keys + want - 1) / want;
    c = (c + 63) / 64 * 64;
    chunk = (int)(c < 256 ? 256 : c);
    splits = keys ? ceil_div(keys, chunk) : 0;
  };
  PagedPlan p;
  cut((long long)P * page, (long long)B * H * ceil_div(M, 16), p.chunk, p.splits);
  cut(Lp, (long long)H * ceil_div((long long)B * M, 16), p.pchunk, p.psplits);
  if (p.splits == 0) p.splits = 1;  // no pages at all: one chunk without keys
  return p;
}

inline int paged_check(int B, int H, int M, int G, int D, int P, int page, int Lp) {
  if (D != 128 && D != 256) return -3;
  if (page <= 0 || page % 16) return -2;
  if (B < 0 || B > 65535 || H <= 0 || H > 65535 || M < 0 || G <= 0 || P < 0 || Lp < 0) return -1;
  if ((long long)P * page > (1LL << 30) || Lp > (1 << 30) || (long long)B * M > (1LL << 30)) return -1;
  return 0;
}

template <int D>
inline int paged_go(const reax::PagedArgs& a, cudaStream_t st) {
  using C = reax::PagedCfg<D>;
  static SmemAttr own, pre;
  if (ensure_smem(own, reax::paged_kernel<D, false>, C::SMEM, true) != cudaSuccess) return -4;
  if (ensure_smem(pre, reax::paged_kernel<D, true>, C::SMEM, true) != cudaSuccess) return -4;
  const long long tiles = ceil_div(a.M, 16), ptiles = ceil_div((long long)a.B * a.M, 16);
  if (tiles * a.splits > 0x7fffffffLL || ptiles * a.psplits > 0x7fffffffLL) return -1;
  if (a.psplits)
    reax::paged_kernel<D, true><<<dim3((unsigned)(ptiles * a.psplits), a.H), C::WARPS * 32, C::SMEM, st>>>(a);
  reax::paged_kernel<D, false><<<dim3((unsigned)(tiles * a.splits), a.H, a.B), C::WARPS * 32, C::SMEM, st>>>(a);
  if (a.splits + a.psplits > 1) {
    const long long rows = (long long)a.B * a.H * a.M;
    reax::paged_join_kernel<D><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(a);
  }
  return (int)cudaGetLastError();
}

}  // namespace reax_host

#define REAX_DEFINE_PAGED_EXPORTS()                                                                                      REAX_API int reax_fmha_paged_splits(int B, int H, int M, int D, int P, int page, int Lp) {                                  if (int rc = reax_host::paged_check(B, H, M, 1, D, P, page, Lp)) return rc;                                              int dev = 0;                                                                                                             if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;                                                                         const reax_host::PagedPlan p = reax_host::paged_plan(B > 0 ? B : 1, H, M > 0 ? M : 1, D, P, page, Lp,                                                                         reax_host::device_sms(dev));                                        return p.splits + p.psplits;                                                                                           }                                                                                                                        REAX_API int reax_fmha_paged(const void* q, long long qsB, long long qsH, long long qsM, const void* kc, const void* ke,                                const void* vc, const void* ve, long long csP, long long csH, long long esP,                                             long long esH, const int* table, long long tsB, const int* prefix, int prefix_len,                                       const int* qpos, int G, long long qpBs, void* o, long long osB, long long osH,                                           long long osM, void* ws, float scale, int B, int H, int M, int D, int P, int page,                                       long long pages, void* stream) {                                                              const int Lp = prefix_len;                                                                                               if (int rc = reax_host::paged_check(B, H, M, G, D, P, page, Lp)) return rc;                                              if (B == 0 || M == 0) return 0;                                                                                          if (!q || !qpos || !o || pages < 0 || (P > 0 && !table) || (Lp > 0 && !prefix)) return -1;                                if ((P > 0 || Lp > 0) && (!kc || !ke || !vc || !ve)) return -1;                                                           if (((uintptr_t)q | (uintptr_t)o | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)ke | (uintptr_t)ve | (uintptr_t)ws) & 15)       return -1;                                                                                                             if ((qsB | qsH | qsM | osB | osH | osM) & 7) return -1;                                                                  if ((csP | csH | esP | esH) & 15) return -1;                                                                             int dev = 0;                                                                                                             cudaGetDevice(&dev);                                                                                                     const reax_host::PagedPlan p = reax_host::paged_plan(B, H, M, D, P, page, Lp, reax_host::device_sms(dev));               const int splits = p.splits + p.psplits;                                                                                 if (splits > 1 && !ws) return -5;                                                                                        float* part = (float*)ws;                                                                                                reax::PagedArgs a{(const uint16_t*)q, qsB, qsH, qsM, (const uint8_t*)kc, (const uint8_t*)ke, (const uint8_t*)vc,                             (const uint8_t*)ve, csP, csH, esP, esH, table, tsB, qpos, qpBs, (uint16_t*)o, osB, osH, osM, part,                         part ? part + (long long)splits * B * H * M * D : nullptr, Lp ? prefix : nullptr,                                        scale * 1.4426950408889634f, B, H, M, G, P, page, reax_host::page_shift(page), Lp, p.chunk,                              p.splits, p.pchunk, p.psplits, pages};                                                                 return D == 128 ? reax_host::paged_go<128>(a, (cudaStream_t)stream) : reax_host::paged_go<256>(a, (cudaStream_t)stream);   }
