// Gated delta rule with a carried state over 32-token chunks, for sequences longer than a few tokens (see delta_state.cuh for the
// recurrence, the arguments and the kernel for short ones), sm_100a.
//
// With G_i the log2 decay from the chunk's start through token i, and h the state before the chunk, the chunk's updates solve
//   u_i = beta_i (v_i - 2^G_i h k_i - sum_{j<i} 2^(G_i - G_j) (k_i . k_j) u_j)
// that is, u = T r with T = (1 + L)^-1 diag(beta), L_ij = beta_i 2^(G_i - G_j) (k_i . k_j) below the diagonal, r_j = v_j - 2^G_j h k_j;
//   o_i = scale (2^G_i h q_i + sum_{j<=i} 2^(G_i - G_j) (q_i . k_j) u_j),  h <- 2^G_last h + sum_j 2^(G_last - G_j) u_j k_j^T.
//
// Precision.  The state is fp32 and stays so: k and q are bf16 and enter the matrix products as they are; an fp32 operand (h, r, u,
// T) enters as the sum of three bf16 numbers, which hold its 24 bits, one product each (of products of two such operands the six
// that reach 2^-24).  What only feeds o, which is rounded to bf16, takes two.  The products accumulate in fp32.  G is summed in 64-bit
// fixed point (32 bits behind the point): in fp32 a difference of sums of strong decays would lose its low bits, and fp64 arithmetic
// took a third of the preparation's time.  An infinity or NaN in a token's inputs may reach the outputs of all tokens of its chunk.
//
// Bound: the tensor pipe of mma.sync.  A warp owns 16 rows of h in accumulator fragments (64 registers), which are at once
// the layout of the A operand of h k, so the state never leaves the registers; 310 m16n8k16 per warp and chunk, 8 cycles
// each.  (tcgen05 would want 128 rows and the state in tensor memory, to be read, split and written back each chunk; three
// bf16 terms at 16 rows keep it in place.)  A CTA is 64 rows of one (sequence, head): four such warps, and four that
// prepare the next chunk (the two Gram matrices, decays, the triangular inverse) while the four work on this one, with one
// barrier per chunk for all.  The two groups of four split the registers 168 / 88 (setmaxnreg), and two CTAs fit an SM.
// With two preparing warps, each with a whole Gram matrix and its own decays, the preparation took 8000 cycles a chunk
// against the products' 4000 to 5800.
#pragma once
#include "delta_state.cuh"

namespace reax {

constexpr int DC_T = 32;                 // tokens per chunk
constexpr int DC_THREADS = 256;
constexpr int DC_KP = 272, DC_VP = 144;  // row pitches in bytes of k, q and of v: 16 past a multiple of 128, so that eight rows of an
constexpr int DC_MP = 80;                // ldmatrix fall in different banks; of T and of P (32 bf16)
struct DcIn {                            // a chunk's inputs
  uint8_t k[DC_T * DC_KP], q[DC_T * DC_KP], v[DC_T * DC_VP];
};
struct DcPrep {  // what is prepared of them
  uint8_t T[3][DC_T * DC_MP], P[2][DC_T * DC_MP];
};
struct DcSmem {
  DcIn in[3];
  DcPrep prep[2];
  struct {
    int whole[DC_T];   // G_i = whole + frac, 0 <= frac < 1
    float frac[DC_T], beta[DC_T];
    float grow[DC_T], left[DC_T];  // 2^G_i, 2^(G_last - G_i)
  } G[3];                          // chunk c's in c % 3
  float L[DC_T][DC_T + 4];  // -(strictly lower part) column by column
  float X[DC_T][DC_T + 4];  // (1 + it)^-1 row by row (only blocks on and below the diagonal)
  float Y[16][20];
  uint8_t o[4][DC_T * 48];  // per warp: 32 tokens x 16 rows
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void stsm_x4_t(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
// x, y as sums of N bf16 numbers: s[i] holds the i-th terms of both (8, 16 or 24 bits in all)
template <int N>
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = pack_bf16(x, y);
    if (i + 1 < N) {
      x -= bf_lo(s[i]);
      y -= bf_hi(s[i]);
    }
  }
}
// accumulator fragments of two n8 tiles -> the A fragment of one k16 step, in N terms
template <int N>
__device__ __forceinline__ void split_frag(const float (&c0)[4], const float (&c1)[4], uint32_t (&a)[N][4]) {
  uint32_t s[N];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float(&c)[4] = r < 2 ? c0 : c1;
    split_bf16<N>(c[(r & 1) * 2], c[(r & 1) * 2 + 1], s);
#pragma unroll
    for (int i = 0; i < N; ++i) a[i][r] = s[i];
  }
}

// copies of the 32 tokens from t on into `in`, zeros past the sequence's end; the 128 preparing threads
__device__ __forceinline__ void dc_load(const DeltaArgs& a, DcIn& in, long long t, long long e, int hk, int hv, int row0, int pt) {
  const int kT = a.H * 128, vT = a.HV * 128, left = (int)min(e - t, (long long)DC_T);
  const uint16_t *k = a.k + t * kT + hk * 128, *q = a.q + t * kT + hk * 128, *v = a.v + t * vT + hv * 128 + row0;
#pragma unroll
  for (int i = 0; i < DC_T * 16 / 128; ++i) {
    const int x = pt + i * 128, r = x >> 4, c = x & 15;
    const int off = (r < left ? r : 0) * kT + c * 8;
    cp_async16(smem_u32(in.k + r * DC_KP + c * 16), k + off, r < left);
    cp_async16(smem_u32(in.q + r * DC_KP + c * 16), q + off, r < left);
  }
#pragma unroll
  for (int i = 0; i < DC_T * 8 / 128; ++i) {
    const int x = pt + i * 128, r = x >> 3, c = x & 7;
    cp_async16(smem_u32(in.v + r * DC_VP + c * 16), v + (r < left ? r : 0) * vT + c * 8, r < left);
  }
}

// 2^(whole + frac) for whole < 2^23, |frac| < 1, the whole part into ex2's exponent: 0 where it would pass 2^-126, not above 2^126
__device__ __forceinline__ float exp2_parts(int whole, float frac) {
  return __uint_as_float(__float_as_uint(ex2_approx(frac)) + ((uint32_t)min(max(whole, -125), 125) << 23)) * (whole < -125 ? 0.f : 1.f);
}

// The decays of a chunk, a token per lane: G and beta for the Gram matrices, 2^G_i and 2^(G_last - G_i) for the products.
__device__ __forceinline__ void dc_decays(DcSmem& s, int slot, int lane, float g, float beta) {
  // Past +-2^9 a token's decay is 0 or infinite in fp32 anyway; a NaN one makes its beta NaN
  long long G = __float2ll_rn(fminf(fmaxf(g, -512.f), 512.f) * 0x1p32f);
  if (g != g) beta = g;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, G, o);
    if (lane >= o) G += x;
  }
  const int whole = (int)(G >> 32);
  const float frac = (float)((uint32_t)G >> 8) * 0x1p-24f;  // 24 bits are exact
  s.G[slot].whole[lane] = whole;
  s.G[slot].frac[lane] = frac;
  s.G[slot].beta[lane] = beta;
  s.G[slot].grow[lane] = exp2_parts(whole, frac);
  s.G[slot].left[lane] = exp2_parts(__shfl_sync(0xffffffffu, whole, 31) - whole, __shfl_sync(0xffffffffu, frac, 31) - frac);
}

// A third of both Gram matrices: w = 0 rows 0-15 by columns 0-15, 1 rows 16-31 by columns 0-15, 2 rows 16-31 by columns 16-31.
// s.L = -(strictly lower beta_i 2^(G_i - G_j) k_i . k_j), P = lower 2^(G_i - G_j) q_i . k_j in two terms.
__device__ __forceinline__ void dc_gram(DcSmem& s, const DcIn& in, int slot, DcPrep& out, int w, int lane) {
  const int gq = lane >> 2, t = lane & 3, i0 = w ? 16 : 0, j0 = w == 2 ? 16 : 0;
  const uint32_t ka = smem_u32(in.k), qa = smem_u32(in.q);
  float acc[2][2][4];  // k . k, q . k; column tiles
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;
  const uint32_t arow = (i0 + (lane & 15)) * DC_KP + (lane >> 4) * 16, brow = (j0 + (lane & 7) + (lane >> 4) * 8) * DC_KP + ((lane >> 3) & 1) * 16;
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    uint32_t x[2][4], b[4];
    ldsm_x4(ka + arow + ks * 32, x[0]);
    ldsm_x4(qa + arow + ks * 32, x[1]);
    ldsm_x4(ka + brow + ks * 32, b);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      mma_bf16(acc[m][0], x[m], b[0], b[1]);
      mma_bf16(acc[m][1], x[m], b[2], b[3]);
    }
  }
  int Wi[2], Wj[2][2];
  float Fi[2], Fj[2][2], bi[2];  // all read before the first store below, which the compiler would not move them across
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = i0 + gq + 8 * r, j = j0 + 8 * r + 2 * t;
    Wi[r] = s.G[slot].whole[i], Fi[r] = s.G[slot].frac[i], bi[r] = -s.G[slot].beta[i];
    const int2 wj = *reinterpret_cast<const int2*>(&s.G[slot].whole[j]);
    const float2 fj = *reinterpret_cast<const float2*>(&s.G[slot].frac[j]);
    Wj[r][0] = wj.x, Wj[r][1] = wj.y, Fj[r][0] = fj.x, Fj[r][1] = fj.y;
  }
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = i0 + gq + 8 * r, j = j0 + n * 8 + 2 * t;
      float d[2], p[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = exp2_parts(Wi[r] - Wj[n][e], Fi[r] - Fj[n][e]);
        d[e] = j + e < i ? bi[r] * (acc[0][n][2 * r + e] * x) : 0.f;
        p[e] = j + e <= i ? acc[1][n][2 * r + e] * x : 0.f;
      }
      s.L[j][i] = d[0];
      s.L[j + 1][i] = d[1];
      uint32_t y[2];
      split_bf16<2>(p[0], p[1], y);
      *reinterpret_cast<uint32_t*>(out.P[0] + i * DC_MP + j * 2) = y[0];
      *reinterpret_cast<uint32_t*>(out.P[1] + i * DC_MP + j * 2) = y[1];
    }
}

// X = (1 - N)^-1 for N = s.L, in fp32, by the four preparing warps.  The 8 x 8 blocks on the diagonal by forward substitution, a
// column to a lane; then twice [[A, 0], [C, B]]^-1 = [[A', 0], [B' C A', B']] of inverses A', B', first to 16 x 16, then to 32 x 32.
// One warp's substitution over all 32 rows is a chain of 31 steps with 496 multiply-adds a lane, 4300 cycles at 88 registers.
__device__ __forceinline__ void dc_inverse(DcSmem& s, int pt) {
  if (pt < 32) {
    const int b = pt & 24, col = pt & 7;
    float l[7][8], x[8];
#pragma unroll
    for (int j = 0; j < 7; ++j)
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&s.L[b + j][b + i]);
        l[j][i] = v.x, l[j][i + 1] = v.y, l[j][i + 2] = v.z, l[j][i + 3] = v.w;
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i == col ? 1.f : 0.f;
#pragma unroll
    for (int j = 0; j < 7; ++j)
#pragma unroll
      for (int i = j + 1; i < 8; ++i) x[i] = __fmaf_rn(l[j][i], x[j], x[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s.X[b + i][b + col] = x[i];
  }
  named_bar_sync<1, 128>();
  {
    const int j0 = pt >> 6 << 4, i0 = j0 + 8, r = (pt >> 3) & 7, c = pt & 7;
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) y = __fmaf_rn(s.L[j0 + k][i0 + r], s.X[j0 + k][j0 + c], y);
    s.Y[(pt >> 6 << 3) + r][c] = y;
    s.X[j0 + r][i0 + c] = 0.f;
    named_bar_sync<1, 128>();
    float z = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) z = __fmaf_rn(s.X[i0 + r][i0 + k], s.Y[(pt >> 6 << 3) + k][c], z);
    s.X[i0 + r][j0 + c] = z;
  }
  named_bar_sync<1, 128>();
  {
    const int r = pt >> 3, c = (pt & 7) * 2;
    float y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 x = *reinterpret_cast<const float2*>(&s.X[k][c]);
      const float n = s.L[k][16 + r];
      y0 = __fmaf_rn(n, x.x, y0), y1 = __fmaf_rn(n, x.y, y1);
    }
    *reinterpret_cast<float2*>(&s.Y[r][c]) = make_float2(y0, y1);
    named_bar_sync<1, 128>();
    float z0 = 0.f, z1 = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 y = *reinterpret_cast<const float2*>(&s.Y[k][c]);
      const float x = s.X[16 + r][16 + k];
      z0 = __fmaf_rn(x, y.x, z0), z1 = __fmaf_rn(x, y.y, z1);
    }
    *reinterpret_cast<float2*>(&s.X[16 + r][c]) = make_float2(z0, z1);
  }
  named_bar_sync<1, 128>();
}

// T = inverse * beta_j in three terms; thread pt of the 128 takes 8 columns of a row
__device__ __forceinline__ void dc_terms(const DcSmem& s, int slot, DcPrep& out, int pt) {
  const int i = pt >> 2, j = (pt & 3) * 8;
  uint32_t y[3][4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float2 x = *reinterpret_cast<const float2*>(&s.X[i][j + 2 * c]), b = *reinterpret_cast<const float2*>(&s.G[slot].beta[j + 2 * c]);
    uint32_t z[3];
    split_bf16<3>(x.x * b.x, x.y * b.y, z);
#pragma unroll
    for (int k = 0; k < 3; ++k) y[k][c] = z[k];
  }
#pragma unroll
  for (int k = 0; k < 3; ++k)
    *reinterpret_cast<uint4*>(out.T[k] + i * DC_MP + j * 2) = make_uint4(y[k][0], y[k][1], y[k][2], y[k][3]);
}

// The four preparing warps, chunk c (its decays are there already), and warp 3 the decays of c + 1
template <typename Decays>
__device__ __forceinline__ void dc_prepare(DcSmem& s, int c, int w, int lane, Decays decays) {
  DcPrep& out = s.prep[c & 1];
  if (w < 3) dc_gram(s, s.in[c % 3], c % 3, out, w, lane);
  named_bar_sync<1, 128>();
  dc_inverse(s, w * 32 + lane);
  dc_terms(s, c % 3, out, w * 32 + lane);
  if (w == 3) decays();
}

// The sequence of this CTA: the longest first (they are the last to end), in their order past a length that one pass can sort.
__device__ __forceinline__ int dc_sequence(const DeltaArgs& a) {
  __shared__ long long len[DC_THREADS];
  __shared__ int mine;
  if (a.N > DC_THREADS) return blockIdx.z;
  const int i = threadIdx.x;
  if (i < a.N) {
    long long b, e;
    delta_range(a, i, b, e);
    len[i] = e - b;
  }
  __syncthreads();
  if (i < a.N) {
    int before = 0;
    for (int k = 0; k < a.N; ++k) before += len[k] > len[i] || (len[k] == len[i] && k < i);
    if (before == (int)blockIdx.z) mine = i;
  }
  __syncthreads();
  return mine;
}

// grid (2, HV, N): 64 rows of one (sequence, value head) per CTA; sequences of at most DS_MOST tokens are the step kernel's
__global__ void __launch_bounds__(DC_THREADS, 2) delta_chunk_kernel(DeltaArgs a) {
  extern __shared__ __align__(128) uint8_t dc_raw[];
  DcSmem& s = *reinterpret_cast<DcSmem*>(dc_raw);
  pdl_wait();
  pdl_launch();  // the step kernel's sequences are others
  const int n = dc_sequence(a), hv = blockIdx.y, lane = threadIdx.x & 31, warp = warp_id();
  const int gq = lane >> 2, t4 = lane & 3, row0 = blockIdx.x * 64;
  long long t0, e;
  delta_range(a, n, t0, e);
  if (e - t0 <= DS_MOST) return;
  const int slot = delta_slot(a, n);
  if (slot < 0) return;
  const long long oT = (long long)a.HV * 128;
  if (!delta_slot_ok(a, n, slot)) {  // the rows of a sequence that cannot run are NaN
    uint16_t* o = a.o + (long long)hv * 128 + row0;
    for (long long i = threadIdx.x; i < (e - t0) * 64; i += DC_THREADS) o[(t0 + (i >> 6)) * oT + (i & 63)] = 0x7fff;
    return;
  }
  const int hk = hv / (a.HV / a.H);
  const int chunks = (int)((e - t0 + DC_T - 1) / DC_T);
  // The two roles' loops meet at one barrier per chunk: chunk c + 1 is prepared while the products of c run
  if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int pt = threadIdx.x - 128;
    // warp 7: its lanes' token's decay and beta of chunk c, asked for well before the decays are computed
    float gw = 0.f;
    uint16_t bw = 0;  // still as bits: a conversion would wait for it
    auto scalars = [&](int c) {
      const long long t = t0 + (long long)c * DC_T + lane;
      gw = t < e ? a.g[t * a.HV + hv] : 0.f;
      bw = t < e ? a.beta[t * a.HV + hv] : (uint16_t)0;
    };
    dc_load(a, s.in[0], t0, e, hk, hv, row0, pt);
    cp_async_commit();
    if (warp == 7) {
      scalars(0);
      dc_decays(s, 0, lane, gw, bf_lo(bw));
      scalars(1);
    }
    cp_async_wait<0>();
    named_bar_sync<1, 128>();
    for (int c = -1; c < chunks; ++c) {
      if (c + 2 < chunks) dc_load(a, s.in[(c + 2) % 3], t0 + (long long)(c + 2) * DC_T, e, hk, hv, row0, pt);
      cp_async_commit();
      if (c + 1 < chunks)
        dc_prepare(s, c + 1, warp - 4, lane, [&] {
          dc_decays(s, (c + 2) % 3, lane, gw, bf_lo(bw));
          scalars(c + 3);
        });
      cp_async_wait<0>();
      named_bar_sync<2, DC_THREADS>();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    float h[16][4];
    float* st = a.state + slot * a.sS + ((long long)hv * 128 + row0 + warp * 16 + gq) * 128 + 2 * t4;
    const bool fresh = a.fresh && a.fresh[n];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float2 x = fresh ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2*>(st + r * 8 * 128 + j * 8);
        h[j][2 * r] = x.x;
        h[j][2 * r + 1] = x.y;
      }
    named_bar_sync<2, DC_THREADS>();
    for (int c = 0; c < chunks; ++c) {
      const DcIn& in = s.in[c % 3];
      const DcPrep& pr = s.prep[c & 1];
      const auto& dec = s.G[c % 3];
      const uint32_t ka = smem_u32(in.k), qa = smem_u32(in.q), va = smem_u32(in.v);
      // ---- h k (three terms) and h q (two)
      float sk[4][4], sq[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) sk[j][x] = sq[j][x] = 0.f;
      const uint32_t brow = ((lane & 7) + (lane >> 4) * 8) * DC_KP + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t ha[3][4];
        split_frag<3>(h[2 * ks], h[2 * ks + 1], ha);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t b[4];
          ldsm_x4(ka + brow + p * 16 * DC_KP + ks * 32, b);
#pragma unroll
          for (int i = 2; i >= 0; --i) {
            mma_bf16(sk[2 * p], ha[i], b[0], b[1]);
            mma_bf16(sk[2 * p + 1], ha[i], b[2], b[3]);
          }
          ldsm_x4(qa + brow + p * 16 * DC_KP + ks * 32, b);
#pragma unroll
          for (int i = 1; i >= 0; --i) {
            mma_bf16(sq[2 * p], ha[i], b[0], b[1]);
            mma_bf16(sq[2 * p + 1], ha[i], b[2], b[3]);
          }
        }
      }
      // ---- r = v - 2^G (h k); o starts as 2^G (h q)
      const uint32_t vaddr = va + ((lane & 7) + (lane >> 4) * 8) * DC_VP + warp * 32 + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t vv[4];  // (tokens 0-7, rows 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
        ldsm_x4_t(vaddr + p * 16 * DC_VP, vv);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 gr = *reinterpret_cast<const float2*>(&dec.grow[(2 * p + x) * 8 + 2 * t4]);
          float(&k4)[4] = sk[2 * p + x];
          float(&q4)[4] = sq[2 * p + x];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            k4[2 * r] = __fmaf_rn(-gr.x, k4[2 * r], bf_lo(vv[2 * x + r]));
            k4[2 * r + 1] = __fmaf_rn(-gr.y, k4[2 * r + 1], bf_hi(vv[2 * x + r]));
            q4[2 * r] *= gr.x;
            q4[2 * r + 1] *= gr.y;
          }
        }
      }
      // ---- u = T r: the six products of three terms by three
      float u[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) u[j][x] = 0.f;
      const uint32_t mrow = ((lane & 7) + (lane >> 4) * 8) * DC_MP + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t ra[3][4];
        split_frag<3>(sk[2 * ks], sk[2 * ks + 1], ra);
#pragma unroll
        for (int p = ks; p < 2; ++p)
#pragma unroll
          for (int y = 2; y >= 0; --y) {
            uint32_t b[4];
            ldsm_x4(smem_u32(pr.T[y]) + mrow + p * 16 * DC_MP + ks * 32, b);
#pragma unroll
            for (int i = 2 - y; i >= 0; --i) {
              mma_bf16(u[2 * p], ra[i], b[0], b[1]);
              mma_bf16(u[2 * p + 1], ra[i], b[2], b[3]);
            }
          }
      }
      // ---- o += P u
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t ua[2][4];
        split_frag<2>(u[2 * ks], u[2 * ks + 1], ua);
#pragma unroll
        for (int p = ks; p < 2; ++p)
#pragma unroll
          for (int y = 1; y >= 0; --y) {
            uint32_t b[4];
            ldsm_x4(smem_u32(pr.P[y]) + mrow + p * 16 * DC_MP + ks * 32, b);
#pragma unroll
            for (int i = 1 - y; i >= 0; --i) {
              mma_bf16(sq[2 * p], ua[i], b[0], b[1]);
              mma_bf16(sq[2 * p + 1], ua[i], b[2], b[3]);
            }
          }
      }
      const uint32_t so = smem_u32(s.o[warp]);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t y[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          y[x] = pack_bf16(sq[2 * p + (x >> 1)][(x & 1) * 2] * a.scale, sq[2 * p + (x >> 1)][(x & 1) * 2 + 1] * a.scale);
        stsm_x4_t(so + (p * 16 + (lane & 7) + (lane >> 4) * 8) * 48 + ((lane >> 3) & 1) * 16, y);
      }
      __syncwarp();
      const long long t = t0 + (long long)c * DC_T + lane;
      if (t < e) {
        uint4* dst = reinterpret_cast<uint4*>(a.o + t * oT + hv * 128 + row0 + warp * 16);
        dst[0] = *reinterpret_cast<const uint4*>(s.o[warp] + lane * 48);
        dst[1] = *reinterpret_cast<const uint4*>(s.o[warp] + lane * 48 + 16);
      }
      // ---- h <- 2^G_last h + (2^(G_last - G_j) u_j) k_j^T
      const float last = dec.grow[DC_T - 1];
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) h[j][x] *= last;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 le = *reinterpret_cast<const float2*>(&dec.left[(2 * ks + x) * 8 + 2 * t4]);
          float(&u4)[4] = u[2 * ks + x];
          u4[0] *= le.x, u4[1] *= le.y, u4[2] *= le.x, u4[3] *= le.y;
        }
        uint32_t ua[3][4];
        split_frag<3>(u[2 * ks], u[2 * ks + 1], ua);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          uint32_t b[4];  // (tokens 0-7, keys 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
          ldsm_x4_t(ka + (ks * 16 + (lane & 15)) * DC_KP + j * 16 + (lane >> 4) * 16, b);
#pragma unroll
          for (int i = 2; i >= 0; --i) {
            mma_bf16(h[j], ua[i], b[0], b[1]);
            mma_bf16(h[j + 1], ua[i], b[2], b[3]);
          }
        }
      }
      named_bar_sync<2, DC_THREADS>();
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *reinterpret_cast<float2*>(st + r * 8 * 128 + j * 8) = make_float2(h[j][2 * r], h[j][2 * r + 1]);
  }
}

}  // namespace reax

namespace reax_host {

inline int delta_go(const reax::DeltaArgs& a, cudaStream_t st) {
  if (int rc = delta_check(a)) return rc;
  if (a.N == 0 || a.T == 0) return 0;
  const dim3 grid(2, a.HV, a.N);
  // Each kernel takes the sequences of its lengths, which are on the device.  T = N is taken for a decode batch and T <= DS_MOST
  // leaves no long sequence: the step kernel alone then takes every length.  (64 sequences of one token, 32 heads: 45 us; with the
  // chunk kernel, which finds nothing to do, beside it 73.)
  if (a.T == a.N || a.T <= reax::DS_MOST)
    return launch_dependent(reax::delta_step_kernel, grid, reax::DS_THREADS, 0, true, st, 1, a, 0x7fffffffffffffffLL, true);
  static SmemAttr attr;
  if (ensure_smem(attr, reax::delta_chunk_kernel, (int)sizeof(reax::DcSmem), true) != cudaSuccess) return -4;
  // setmaxnreg's shares (four warps of 168 registers a thread, four of 88) come out of the registers of the launch: with fewer
  // than 128 a thread the kernel would wait for the rest for good
  static std::atomic<int> regs{0};
  if (!regs) {
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, reax::delta_chunk_kernel) != cudaSuccess) return -4;
    regs = at.numRegs;
  }
  if (regs < 128) return -4;
  if (int rc = launch_dependent(reax::delta_chunk_kernel, grid, reax::DC_THREADS, (int)sizeof(reax::DcSmem), true, st, 1, a)) return rc;
  return launch_dependent(reax::delta_step_kernel, grid, reax::DS_THREADS, 0, true, st, 1, a, reax::DS_MOST, false);
}

}  // namespace reax_host

#define REAX_DEFINE_DELTA_STATE_EXPORT()                                                                               \
  REAX_API int reax_delta_state(const void* q, const void* k, const void* v, const void* g, const void* beta,             \
                                const long long* cu, void* state, long long ssS, const int* slots, const void* fresh,     \
                                void* o, float scale, long long T, long long S, int N, int H, int HV, void* stream) {     \
    reax::DeltaArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (const uint16_t*)beta, (const float*)g,  \
                      cu, (float*)state, ssS, slots, (const uint8_t*)fresh, (uint16_t*)o, scale, T, S, N, H, HV};          \
    return reax_host::delta_go(a, (cudaStream_t)stream);                                                                  \
  }
