// Attention of a whole batch over the prefix that its sequences share (reax_fmha_paged with a prefix), sm_100a tcgen05.
//
// The B * M query rows of a key/value head are one matrix: with 64 sequences of 4 rows each it is 256 rows against the same
// keys, and the prefix is read (and dequantised) once per 128 rows instead of once per sequence.  The result is a partial output
// and the log2 of its sum for each row and chunk of the prefix, as paged_kernel leaves them; paged_join_kernel joins all.
//
// One CTA per SM takes 128 rows of one head and a chunk of the keys, 64 at a time.  15 warps:
//   0..3    softmax, a thread per row (TMEM lane): S out of TMEM, P (f16) back over it;
//   4..7    dequantisation of K: 16 cache bytes -> 16 f16 in 128-byte-swizzled shared memory, each warp sixteen rows of a tile;
//   8..11   of V.  (All eight on K, then on V: each waits on both sides of either, and 126 us where these take 123.)
//   13, 14  bulk copies of the bytes of K, of V, as many rows at a time as surely lie in one page (16 to 64), three tiles ahead (four
//           at D = 128).  (Loads into registers by the dequantising warps took longer to issue than the conversion; one warp for both
//           copies is late with pages of 16: 70 us for a call that takes 62, 32 questions on 32768 tokens in heads of 256.)
//   12      issues S_j = Q K_j^T (M = 128, N = 64, K = D), then O += P_{j-1} V_{j-1} (N = D, K = 64).
// K and V have two buffers each, S two, freed by tcgen05.commit.
//
// At D = 256 a tile takes 2150 cycles, what the softmax's four warps take from S to P (750 to read it and for the maximum, 1050 for 64
// exponents a thread and P, the rest waits); the products 530 and 510 (the tensor core's rate), the conversions 1500 each, side by side.
// What they share is the shared-memory port, where the f16 rows are written and read once (1024 cycles) and the cache's bytes pass; so q
// and P are operands out of tensor memory.  64 questions on a shared document of 32768 tokens: 119 us, 78 of them here.  Measured
// slower (in a call of then 123): a branch of one lane to issue the products (137 us), tiles of 128 keys, whose f16 rows leave room for one buffer each; S
// as two chains side by side, which leaves q no room in tensor memory; a half to an eighth of the exponents as polynomials on the FMA
// pipe (128 to 123.5).
//
// The rows' powers of two go into the f16 values, relative to the tile's largest (nk, nv): e4m3 has 4 bits, f16 11, and a row stays
// exact down to 2^-15 of the tile's largest row.  What is left is one factor per tile, so a score costs one multiply-add and one
// exponent: P = 2^(x + nv - mv + 7), with two lazy references per query: no x passes m by more than 8, no x + nv passes mv by more
// (P < 2^15).  The 7 keeps f16's full precision down to 2^-21 of the largest.  (Raising a reference costs a pass over O in tensor memory: with
// 2 in place of the 8 most tiles did.  Both powers of two applied to the scores, with two exponents each, took twice the
// softmax's time.)  O carries 2^(7 - mv) until the end, the sum 2^-m.
// What decides is a key's own weight: a large row that a query does not see, or that weighs nothing, must not cost the others bits.
// So a tile whose rows of K lie more than 2^15 apart, or those of V more than 2^7, keeps its e4m3 values as they are, and each score
// takes its key's two powers and two exponents, as in paged_kernel.  (2^7: mv may lie that far above the largest x_j + nv_j, and the 7 takes
// it back: a weight below f16's range is off by 2^-25 of the largest, as there.)  Such a tile costs two of the common ones: the call above
// takes 204 us with one small value row in every tile.  Rows of zeros count as 2^-127.
// A row whose K or V is NaN becomes a NaN key and a zero value, which reaches the queries that see it and no others.
#pragma once
#include "paged.cuh"

namespace reax {

constexpr int PF_BN = 64, PF_ROWS = 128, PF_THREADS = 15 * 32;

template <int D>
struct PrefixCfg {
  static constexpr uint32_t KV_BYTES = PF_BN * D * 2;
  static constexpr uint32_t Q_COL = 128, O_COL = 256, TMEM_COLS = 512;  // S (then P) at columns 0 and 64
  static constexpr int RAW = PF_BN * D, EXP = 2 * PF_BN;  // a tile's rows of K (or V) as they lie in the cache; both exponents
  // Of those in flight, K and V in turn.  Even, so that a buffer's full barrier always has the same warps waiting: others could take
  // the parity of the phase before theirs for it.
  static constexpr int NR = D == 256 ? 6 : 8;
  static_assert(NR % 2 == 0 && NR <= 8);
  static constexpr int SMEM = 1024 + 4 * KV_BYTES + NR * (RAW + EXP);
};

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int b_mn_major = 0) {
  return idesc_bf16(M, N, b_mn_major) & ~((1u << 7) | (1u << 10));  // format 0 of A and B: f16
}

// bytes (a multiple of 16, both addresses 16-byte aligned) from global to shared memory; they count on the mbarrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}

// One lane of the warp, always the same
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}\n" : "=r"(x));
  return x;
}
// The whole warp comes here, the lane with `lead` issues.  With the warp together the compiler keeps descriptors and addresses in uniform
// registers, which is where the instruction takes them from: a product of N = 64 every 33 cycles (the tensor core's rate), in a
// branch of one lane every 50.
__device__ __forceinline__ void mma_ts_lead(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accum, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accum), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_commit_lead(uint32_t bar, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar),
      "r"(lead)
      : "memory");
}

__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t addr) {
  uint16_t x;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(addr) : "memory");
  return x;
}

// grid (tiles of 128 rows * chunks of the prefix, H)
template <int D>
__global__ void __launch_bounds__(PF_THREADS, 1) prefix_kernel(const __grid_constant__ PagedArgs a) {
  using C = PrefixCfg<D>;
  extern __shared__ uint8_t pf_raw[];
  __shared__ __align__(8) uint64_t bars[12 + 2 * C::NR];
  __shared__ uint32_t sgran[C::NR];  // which of a raw buffer's four groups of 16 keys were copied
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  // a tile's largest nk and nv (bytes; + 256: its rows lie too far apart for that, the keys' own are in sown), its even and odd keys that exist
  __shared__ uint4 stile[4];
  __shared__ uint4 sown[4][PF_BN / 8];  // 16 bits a key: nk and, above it, nv
  pdl_wait();
  pdl_launch();  // the own keys' kernel needs nothing from here
  const uint32_t base = (smem_u32(pf_raw) + 1023u) & ~1023u;
  const uint32_t sk = base, sv = sk + 2 * C::KV_BYTES, sraw = sv + 2 * C::KV_BYTES, sexp = sraw + C::NR * C::RAW;
  const int split = blockIdx.x % a.psplits, R0 = blockIdx.x / a.psplits * PF_ROWS, h = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = warp_id();
  const int c0 = split * a.pchunk, c1 = min(a.Lp, c0 + a.pchunk), ntiles = (c1 - c0 + PF_BN - 1) / PF_BN;
  const int rows = a.B * a.M;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  // kfull 0,1  vfull 2,3  s_done 4,5  pv_done 6,7  p_ready 8,9  drain 10  q_ready 11  raw_full 12..  raw_empty 12 + NR..
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(bar(i), 4), mbar_init(bar(4 + i), 1);
    mbar_init(bar(8), 4);
    mbar_init(bar(9), 4);
    mbar_init(bar(10), 1);
    mbar_init(bar(11), 4);
    for (int i = 0; i < C::NR; ++i) mbar_init(bar(12 + i), 1), mbar_init(bar(12 + C::NR + i), 4);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(&tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* abort = &abort_flag;

  if (warp >= 4 && warp < 12) {  // ---------------------------------------------------------------- dequantisation
    // A load of a warp covers whole rows, two (D = 256) or four, 64 bytes to four lanes.  Neighbouring groups of four lanes take
    // neighbouring rows and different 64-byte parts, so that eight lanes' loads and stores fall in different banks.
    constexpr int RPU = 512 / D, U = 16 / RPU, NQ = D / 64;
    const bool is_v = warp >= 8;
    const int w = warp & 3, row = w * 16 + (lane & 15), grp = lane >> 2;
    const int ur = 2 * ((grp >> 1) / NQ) + (grp & 1), quad = ((grp >> 1) + (grp & 1)) % NQ;
    // scale: of row w * 16 + (lane & 15); all ones: a row without values, filled with `fill`
    auto put = [&](uint32_t buf, uint32_t raw, uint32_t scale, uint32_t fill) {
      uint4 x[U];
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = ld_shared_v4(raw + (w * 16 + i * RPU + ur) * D + quad * 64 + (lane & 3) * 16);
      const bool some = __any_sync(0xffffffffu, scale == 0xffffffffu);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int r = i * RPU + ur;
        const uint32_t sc = __shfl_sync(0xffffffffu, scale, r);
        const uint32_t y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        const uint32_t dst = buf + quad * (PF_BN * 128) + (w * 16 + r) * 128;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t z[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const uint32_t v = e4m3x2_f16x2((uint16_t)(n & 1 ? y[2 * k + (n >> 1)] >> 16 : y[2 * k + (n >> 1)]));
            asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(z[n]) : "r"(v), "r"(sc));
          }
          if (some && sc == 0xffffffffu) z[0] = z[1] = z[2] = z[3] = fill;
          st_shared_v4(dst + (((2 * (lane & 3) + k) ^ (r & 7)) << 4), make_uint4(z[0], z[1], z[2], z[3]));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    // f16x2 of 2^(n - top), which is -15 at least
    auto scale_of = [&](int n, int top) {
      const int e = n - top;
      const uint32_t b = e >= -14 ? (uint32_t)(e + 15) << 10 : 1u << (e + 24);
      return b | (b << 16);
    };
    int rs = is_v;
    uint32_t phase = 0;
    for (int j = 0; j < ntiles; ++j) {
      const int s = j & 1;
      const uint32_t par = ((j >> 1) & 1) ^ 1;  // the buffer's previous use, done; the first two pass at once
      const uint32_t raw = sraw + rs * C::RAW, ex = sexp + rs * C::EXP;
      if (!mbar_wait_warp(bar(12 + rs), phase, abort, ST_TIMEOUT_ATTN)) break;
      // exponents of keys 2 lane, 2 lane + 1; NaN rows and keys that do not exist take no part in the maxima
      const bool even_ok = (sgran[rs] >> (lane >> 3)) & 1u && c0 + j * PF_BN + 2 * lane < c1;
      const bool odd_ok = even_ok && c0 + j * PF_BN + 2 * lane + 1 < c1;
      const uint32_t kb = ld_shared_u16(ex + 2 * lane), vb = ld_shared_u16(ex + PF_BN + 2 * lane);
      const int k2[2] = {(int)(kb & 255u), (int)(kb >> 8)}, v2[2] = {(int)(vb & 255u), (int)(vb >> 8)};
      int kn = 0, vn = 0, kl = 255, vl = 255;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if ((e ? odd_ok : even_ok) && k2[e] != 255 && v2[e] != 255)
          kn = max(kn, k2[e]), vn = max(vn, v2[e]), kl = min(kl, k2[e]), vl = min(vl, v2[e]);
      kn = __reduce_max_sync(0xffffffffu, kn);
      vn = __reduce_max_sync(0xffffffffu, vn);
      const bool wide = __any_sync(0xffffffffu, kl < kn - 15 || vl < vn - 7);
      const uint32_t even = __ballot_sync(0xffffffffu, even_ok), odd = __ballot_sync(0xffffffffu, odd_ok);
      const uint32_t kp = __shfl_sync(0xffffffffu, kb, row >> 1), vp = __shfl_sync(0xffffffffu, vb, row >> 1);
      const int nk = row & 1 ? kp >> 8 : kp & 255u, nv = row & 1 ? vp >> 8 : vp & 255u;
      const bool none = nk == 255 || nv == 255 || !(((row & 1 ? odd : even) >> (row >> 1)) & 1u);
      if (!mbar_wait_warp(bar((is_v ? 6 : 4) + s), par, abort, ST_TIMEOUT_ATTN)) break;
      const uint32_t scale = none ? 0xffffffffu : wide ? 0x3c003c00u : is_v ? scale_of(nv, vn) : scale_of(nk, kn);
      if (warp == 4 && wide) reinterpret_cast<uint32_t*>(sown[j & 3])[lane] = (kb & 255u) | (vb & 255u) << 8 | (kb >> 8) << 16 | (vb >> 8) << 24;
      // a key's NaN where there is no key either: masked
      put((is_v ? sv : sk) + s * C::KV_BYTES, raw, scale, is_v ? 0u : 0x7e007e00u);
      // For the softmax, which reads it after S_j.  Four of them: this one's place was read by the softmax of j - 4, which was done
      // before S_{j-2} was issued, whose end K_j's buffer waited for.
      if (warp == 4 && lane == 0) {
        stile[j & 3] = make_uint4(kn, vn + (wide ? 256 : 0), even, odd);
      }
      if (lane == 0) {
        mbar_arrive(bar((is_v ? 2 : 0) + s));
        mbar_arrive(bar(12 + C::NR + rs));
      }
      rs += 2;
      if (rs >= C::NR) rs -= C::NR, phase ^= 1;
    }
  } else if (warp >= 13) {  // --------------------------------------------------------------------- copies
    // lanes 0-3: rows of a group of 16 keys, 4-7 and 8-11: their exponents (both, for K and for V: a NaN in one leaves out the other)
    // rows of a copy: what of a tile surely lies in one page
    const int piece = a.page % 64 == 0 ? 64 : a.page % 32 == 0 ? 32 : 16;
    const int gr = lane & 3, what = lane >> 2, first = gr * 16 & ~(piece - 1);
    const bool mine = first == gr * 16;
    const bool is_v = warp == 14;
    const uint8_t *rows_of = (is_v ? a.vc : a.kc) + h * a.cH, *exps = (what == 1 ? a.ke : a.ve) + h * a.eH;
    CopyLedger ledger;
    int off = 0;
    auto page_of = [&](int j) {
      const int key = c0 + j * PF_BN + first, pi = a.shift >= 0 ? key >> a.shift : key / a.page;
      off = key - pi * a.page;
      return key < c1 ? a.prefix[pi] : -1;
    };
    int id = page_of(0), rs = is_v;
    uint32_t phase = 0;
    for (int j = 0; j < ntiles; ++j) {
      const bool ok = id >= 0 && id < a.pages;
      if (!ok && c0 + j * PF_BN + first < c1) record_status(ST_BAD_PAGE);
      const uint8_t* from = what ? exps + (ok ? id * a.eP + off : 0) : rows_of + (ok ? id * a.cP + (long long)off * D : 0);
      if (j + 1 < ntiles) id = page_of(j + 1);
      const uint32_t groups = __ballot_sync(0xffffffffu, ok) & 15u;
      if (!mbar_wait_warp(bar(12 + C::NR + rs), phase ^ 1, abort, ST_TIMEOUT_ATTN)) break;
      if (lane == 0) {
        sgran[rs] = groups;
        ledger.arm(rs, phase);
        mbar_arrive_expect_tx(bar(12 + rs), __popc(groups) * 16 * (D + 2));
      }
      __syncwarp();
      if (ok && mine && what < 3)
        bulk_load(what ? sexp + rs * C::EXP + (what - 1) * PF_BN + first : sraw + rs * C::RAW + first * D, from, what ? piece : piece * D,
                  bar(12 + rs));
      rs += 2;
      if (rs >= C::NR) rs -= C::NR, phase ^= 1;
    }
    if (lane == 0) ledger.drain([&](int i) { return bar(12 + i); });  // no copy outlives the CTA
    __syncwarp();
  } else if (warp == 12) {  // --------------------------------------------------------------------- MMA issue
    constexpr uint32_t IDESC_S = idesc_f16(PF_ROWS, PF_BN), IDESC_PV = idesc_f16(PF_ROWS, D, /*b_mn_major=*/1);
    const uint32_t lead = elect_lane();
    for (int j = 0; j <= ntiles; ++j) {
      if (j < ntiles) {
        const int s = j & 1;
        if (j == 0 && !mbar_wait_warp(bar(11), 0, abort, ST_TIMEOUT_ATTN)) break;
        if (!mbar_wait_warp(bar(s), (j >> 1) & 1, abort, ST_TIMEOUT_ATTN)) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ts_lead(tmem + s * 64, tmem + C::Q_COL + kk * 8,
                      sw128_desc(sk + s * C::KV_BYTES + (kk >> 2) * (PF_BN * 128) + (kk & 3) * 32), IDESC_S, kk > 0, lead);
        mma_commit_lead(bar(4 + s), lead);
      }
      if (j > 0) {
        const int i = j - 1, s = i & 1;
        if (!mbar_wait_warp(bar(8 + s), (i >> 1) & 1, abort, ST_TIMEOUT_ATTN)) break;
        if (!mbar_wait_warp(bar(2 + s), (i >> 1) & 1, abort, ST_TIMEOUT_ATTN)) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < PF_BN / 16; ++kk)
          mma_ts_lead(tmem + C::O_COL, tmem + s * 64 + kk * 8,
                      sw128_desc(sv + s * C::KV_BYTES + kk * 2048, /*lbo=*/PF_BN * 128, /*sbo=*/1024), IDESC_PV, i > 0 || kk > 0, lead);
        mma_commit_lead(bar(6 + s), lead);
      }
    }
    // whatever was issued ends before the CTA gives its memory back
    mma_commit_lead(bar(10), lead);
    const long long t0 = clock64();
    while (!mbar_try_wait(bar(10), 0))
      if (clock64() - t0 > REAX_DRAIN_LIMIT) {
        record_status(ST_TIMEOUT_DRAIN);
        break;
      }
    __syncwarp();
  } else if (warp < 4) {  // ----------------------------------------------------------------------- softmax
    const int row = warp * 32 + lane, R = R0 + row;
    const bool real = R < rows;
    int lim = a.Lp - 1;
    if (real) lim = max(min(a.qpos[R / a.M * a.qpB + R % a.M / a.G], lim), -1);  // a difference to it stays in 32 bits
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    // q: the row scaled by its power of two (and by the scale's sign), f16, into tensor memory
    const uint16_t* qrow = a.q + (real ? R / a.M * a.qB + R % a.M * a.qM : 0) + h * a.qH;
    uint32_t top = 0;
#pragma unroll 8
    for (int c = 0; c < D / 8; ++c) {
      const uint4 x = real ? *reinterpret_cast<const uint4*>(qrow + c * 8) : make_uint4(0, 0, 0, 0);
      top = max_u16x2(top, max_u16x2(max_u16x2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), max_u16x2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
    }
    const int e = min(max((int)(max(top & 0xffffu, top >> 16) >> 7), 2), 252);
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23) * (a.scale_log2 < 0.f ? -1.f : 1.f);
    const float rs = __uint_as_float((uint32_t)e << 23) * fabsf(a.scale_log2);
#pragma unroll 4
    for (int c = 0; c < D / 16; ++c) {
      uint32_t y[8];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 x = real ? *reinterpret_cast<const uint4*>(qrow + c * 16 + k * 8) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) y[4 * k + i] = pack_f16(bf_lo(w[i]) * inv, bf_hi(w[i]) * inv);
      }
      tmem_st8_nowait(lanes + C::Q_COL + c * 8, y);
    }
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(11));
    float m = PAGED_NONE, mv = PAGED_NONE, l = 0.f;
    bool live = true;
    // raises the references to a tile's maxima and rescales what there is
    auto raise = [&](int j, float mx, float my) {
      const float up = fmaxf(mx, m), upv = fmaxf(my, mv);
      l *= ex2_approx(m - up);
      m = up;
      if (j > 0) {
        const float ao = ex2_approx(mv - upv);
        live = mbar_wait_warp(bar(7 - (j & 1)), ((j - 1) >> 1) & 1, abort, ST_TIMEOUT_ATTN);
        if (!live) return;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(lanes + C::O_COL + c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * ao);
          tmem_st32_nowait(lanes + C::O_COL + c, o);
        }
        tmem_wait_st();
      }
      mv = upv;
    };
    auto factor = [&](uint32_t nk) {  // not 0: a masked score is -inf; nor infinite: a score may be 0
      return fminf(fmaxf(rs * pow2_byte(nk), 0x1p-126f), 0x1.fffffep127f);
    };
    for (int j = 0; j < ntiles; ++j) {
      const int s = j & 1, k0 = c0 + j * PF_BN;
      live = mbar_wait_warp(bar(4 + s), (j >> 1) & 1, abort, ST_TIMEOUT_ATTN);
      if (!live) break;
      tc_fence_after();
      const uint4 tile = ld_shared_v4(smem_u32(&stile[j & 3]));
      if (tile.y < 256u) {
        // What needs nothing of S comes before it.  P = 2^(x - m + at + 7), at = nv - (mv - m): the values of a tile 2^60 smaller than
        // what counts add nothing, but its weights still count in the sum
        const float vn = (float)((int)tile.y - 127), c1s = factor(tile.x), most = fminf(m, mv - vn) + 8.f;
        float at = fmaxf(vn - (mv - m), -60.f), c0s = at + 7.f - m;
        uint32_t x[64];
        tmem_ld64(lanes + s * 64, x);
        if (__any_sync(0xffffffffu, k0 + PF_BN - 1 > lim || (tile.z & tile.w) != 0xffffffffu)) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (k0 + i > lim || !(((i & 1 ? tile.w : tile.z) >> (i >> 1)) & 1u)) x[i] = 0xff800000u;  // -inf
        }
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          t0 = max3f(t0, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          t1 = max3f(t1, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
        }
        const float mx = fmaxf(t0, t1) * c1s;
        if (__any_sync(0xffffffffu, mx > most)) {
          raise(j, mx, mx + vn);
          if (!live) break;
          at = fmaxf(vn - (mv - m), -60.f);
          c0s = at + 7.f - m;
        }
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p0 = ex2_approx(__fmaf_rn(__uint_as_float(x[c * 16 + 2 * i]), c1s, c0s));
            const float p1 = ex2_approx(__fmaf_rn(__uint_as_float(x[c * 16 + 2 * i + 1]), c1s, c0s));
            sum += p0 + p1;
            y[i] = pack_f16(p0, p1);
          }
          tmem_st8_nowait(lanes + s * 64 + c * 8, y);
        }
        l = __fmaf_rn(sum, ex2_approx(-at - 7.f), l);
      } else {
        // The keys' own powers of two, 16 keys at a time in two passes: as variants of the code above they took its registers and 4 us
        // of 87 in calls without such a tile.  The first pass puts the scores back over S, the second P's chunk c over S's chunks up to c
        auto value_n = [&](const uint4* own, int i) {  // nv + 127 of key i of the 16
          const uint32_t w = reinterpret_cast<const uint32_t*>(own)[i >> 1];
          return __uint_as_float(__byte_perm(w, 0x4b000000u, i & 1 ? 0x7653u : 0x7651u)) - 0x1p23f;
        };
        const int seen = lim - k0;
        float mx = -INFINITY, my = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t x[16];
          tmem_ld16_nowait(lanes + s * 64 + c * 16, x);
          const uint4 own[2] = {sown[j & 3][2 * c], sown[j & 3][2 * c + 1]};
          const uint32_t even = tile.z >> 8 * c, odd = tile.w >> 8 * c;
          tmem_wait_ld16(x);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(own)[i >> 1];
            const float nk = __uint_as_float(max((i & 1 ? w << 7 : w << 23) & 0x7f800000u, 0x00400000u));
            const float f = fminf(fmaxf(rs * nk, 0x1p-126f), 0x1.fffffep127f);
            const bool is = (16 * c + i <= seen) & (((i & 1 ? odd : even) & (1u << (i >> 1))) != 0);
            const float y = is ? __uint_as_float(x[i]) * f : -INFINITY;
            mx = fmaxf(mx, y);
            my = fmaxf(my, y + value_n(own, i));
            x[i] = __float_as_uint(y);
          }
          tmem_st16_nowait(lanes + s * 64 + c * 16, x);
        }
        my -= 127.f;
        tmem_wait_st();
        if (__any_sync(0xffffffffu, mx > m + 8.f || my > mv + 8.f)) {
          raise(j, mx, my);
          if (!live) break;
        }
        const float cv = 7.f - 127.f - mv;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t x[16], y[8];
          tmem_ld16_nowait(lanes + s * 64 + c * 16, x);
          const uint4 own[2] = {sown[j & 3][2 * c], sown[j & 3][2 * c + 1]};
          tmem_wait_ld16(x);
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float x0 = __uint_as_float(x[i]), x1 = __uint_as_float(x[i + 1]);
            sum += ex2_approx(x0 - m) + ex2_approx(x1 - m);
            y[i >> 1] = pack_f16(ex2_approx(x0 + (value_n(own, i) + cv)), ex2_approx(x1 + (value_n(own, i + 1) + cv)));
          }
          l += sum;
          tmem_st8_nowait(lanes + s * 64 + c * 8, y);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(8 + s));
    }
    if (live) live = mbar_wait_warp(bar(6 + ((ntiles - 1) & 1)), ((ntiles - 1) >> 1) & 1, abort, ST_TIMEOUT_ATTN);
    const long long out = (long long)(a.splits + split) * a.B * a.H * a.M + ((long long)(R / a.M) * a.H + h) * a.M + R % a.M;
    if (live) {
      tc_fence_after();
      const float half = ex2_approx(0.5f * (mv - m)), fac = half * 0x1p-7f / l;  // in two steps, as in paged_kernel
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld32(lanes + C::O_COL + c, o);
        if (real) {
          float4* p = reinterpret_cast<float4*>(a.part + out * D + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = l == 0.f ? 0.f : __uint_as_float(o[4 * e + k]) * half * fac;
            p[e] = make_float4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
    // after a wait that ran out the rows are NaN, not what the workspace held
    if (real) a.lse[out] = !live ? __uint_as_float(0x7fc00000u) : l == 0.f ? -INFINITY : m + log2f(l);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

}  // namespace reax
