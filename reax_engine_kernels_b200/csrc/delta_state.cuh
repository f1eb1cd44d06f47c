// Gated delta rule with a carried state: token by token, one token per sequence to long runs, sm_100a.
//
// Per sequence and value head, with h [value 128][key 128] fp32 (the transpose of the state that the chunked kernels carry):
//   h <- 2^g h;  u = beta (v - h k);  h <- h + u k^T;  o = scale * h q
// Both products are taken of the old state, hk = h k and hq = h q, so that one reduction serves a token:
//   u = beta (v - 2^g hk),  o = scale (2^g hq + u (k . q)),  h <- 2^g h + u k^T
// All of it in fp32; only o is rounded (to bf16, its type).
//
// One token: HBM-bound, 64 KB of state read and written per (sequence, head).  The rows of h are independent, so a warp
// owns 16 of them and a CTA of four warps 64: every load of a warp (8 KB) is in flight at once, in registers, and there
// is no shared memory and no barrier.  16 lanes share a row, each with 8 keys; a lane keeps row r ^ (lane / 2) of its half
// warp's 8 rows in register slot r, so that each step of the reduction sends the upper half of the slots and keeps the
// lower half without a select (16 shuffles for the 16 sums of a half warp instead of 64), and the new u come back by
// seven shuffles.
#pragma once
#include "common.cuh"

namespace reax {

struct DeltaArgs {
  const uint16_t *q, *k, *v, *beta;
  const float* g;
  const long long* cu;
  float* state;
  long long sS;  // slot stride of the state, elements
  const int* slots;      // NULL: sequence n uses slot n
  const uint8_t* fresh;  // NULL: no sequence starts from zeros
  uint16_t* o;
  float scale;
  long long T, S;
  int N, H, HV;
};

constexpr int DS_THREADS = 128;
// Longest sequence that goes token by token beside longer ones.  64 sequences x 32 heads of 9 tokens: 113 us by this kernel, 152 by
// the chunk kernel; of 16 tokens: 166 and 154.  16 sequences of 12: 37 and 41.
constexpr long long DS_MOST = 14;

// The sequence's token range, cut to the T rows there are.
__device__ __forceinline__ void delta_range(const DeltaArgs& a, int n, long long& b, long long& e) {
  b = min(max(a.cu[n], 0LL), a.T);
  e = min(max(a.cu[n + 1], b), a.T);
}

// The slot that sequence n asks for; negative: it is left alone
__device__ __forceinline__ int delta_slot(const DeltaArgs& a, int n) { return a.slots ? a.slots[n] : n; }

// Whether sequence n may run on slot s: not past the end, nor named by an earlier sequence with tokens (two CTAs would race on it).
// Every thread of the CTA calls it.
__device__ __forceinline__ bool delta_slot_ok(const DeltaArgs& a, int n, int s) {
  int bad = s >= a.S;
  if (a.slots)
    for (int i = threadIdx.x; i < n; i += blockDim.x)
      if (a.slots[i] == s) {
        long long b, e;
        delta_range(a, i, b, e);
        bad |= e > b;
      }
  if (!__syncthreads_or(bad)) return true;
  if (threadIdx.x == 0) record_status(ST_BAD_STATE);
  return false;
}

// grid (2, HV, N): 64 rows of one (sequence, value head) per CTA; sequences of more than `most` tokens are the chunk kernel's
__global__ void __launch_bounds__(DS_THREADS, 4) delta_step_kernel(DeltaArgs a, long long most, bool first) {
  if (first) pdl_wait();
  const int n = blockIdx.z, hv = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & 15, half = lane >> 4, own = sub >> 1;
  const int row0 = blockIdx.x * 64 + warp * 16 + half * 8;
  long long t, e;
  delta_range(a, n, t, e);
  const int slot = delta_slot(a, n);
  const bool zero = a.fresh && a.fresh[n];
  if (t >= e || e - t > most || slot < 0) {
    pdl_wait();
    return;
  }
  // The state and the first token are asked for before the slots of the sequences before this one are looked at: 64 sequences of
  // one token, 32 heads, in 45.5 us, 48.7 with the slots first.  (An earlier sequence may be writing the slot: then this one stops.)
  float* st = a.state + slot * a.sS + ((long long)hv * 128 + row0) * 128 + sub * 8;
  uint64_t h[8][4];
  if (zero || slot >= a.S) {
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) h[r][j] = 0;
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const ulonglong2* p = reinterpret_cast<const ulonglong2*>(st + (r ^ own) * 128);
      const ulonglong2 x = __ldcs(p), y = __ldcs(p + 1);
      h[r][0] = x.x, h[r][1] = x.y, h[r][2] = y.x, h[r][3] = y.y;
    }
  }
  // the token's rows; from one token to the next by 32-bit steps
  const int hk = hv / (a.HV / a.H), kT = a.H * 128, oT = a.HV * 128;
  const uint16_t *kp = a.k + t * kT + hk * 128 + sub * 8, *qp = a.q + t * kT + hk * 128 + sub * 8;
  const uint16_t *vp = a.v + t * oT + hv * 128 + row0 + own, *bp = a.beta + t * a.HV + hv;
  const float* gp = a.g + t * a.HV + hv;
  uint16_t* o = a.o + t * oT + hv * 128 + row0 + own;
  uint4 kw = *reinterpret_cast<const uint4*>(kp), qw = *reinterpret_cast<const uint4*>(qp);
  uint16_t vw = *vp, bw = *bp;
  float gw = *gp;
  if (!delta_slot_ok(a, n, slot)) {  // the rows of a sequence that cannot run are NaN
    if (!(lane & 1))
      for (; t < e; ++t, o += oT) *o = 0x7fff;
    pdl_wait();
    return;
  }
  for (; t < e; ++t) {
    const uint32_t kb[4] = {kw.x, kw.y, kw.z, kw.w}, qb[4] = {qw.x, qw.y, qw.z, qw.w};
    const float vt = bf_lo(vw), bt = bf_lo(bw), at = exp2f(gw);
    if (t + 1 < e) {  // the next token's operands, while this one is computed
      kp += kT, qp += kT, vp += oT, bp += a.HV, gp += a.HV;
      kw = *reinterpret_cast<const uint4*>(kp), qw = *reinterpret_cast<const uint4*>(qp);
      vw = *vp, bw = *bp, gw = *gp;
    }
    uint64_t k2[4], q2[4], s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k2[j] = f2(bf_lo(kb[j]), bf_hi(kb[j]));
      q2[j] = f2(bf_lo(qb[j]), bf_hi(qb[j]));
      s = f2fma(k2[j], q2[j], s);
    }
    float dk[8], dq[8], x, y;
    f2get(s, x, y);
    float kq = x + y;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      uint64_t p = f2mul(h[r][0], k2[0]), u = f2mul(h[r][0], q2[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) p = f2fma(h[r][j], k2[j], p), u = f2fma(h[r][j], q2[j], u);
      f2get(p, x, y);
      dk[r] = x + y;
      f2get(u, x, y);
      dq[r] = x + y;
    }
#pragma unroll
    for (int m = 4; m > 0; m >>= 1)
#pragma unroll
      for (int r = 0; r < m; ++r) {
        dk[r] += __shfl_xor_sync(0xffffffffu, dk[r + m], 2 * m);
        dq[r] += __shfl_xor_sync(0xffffffffu, dq[r + m], 2 * m);
      }
    const float sk = dk[0] + __shfl_xor_sync(0xffffffffu, dk[0], 1), sq = dq[0] + __shfl_xor_sync(0xffffffffu, dq[0], 1);
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, m);
    const float u = bt * (vt - at * sk);
    const float ot = a.scale * (at * sq + u * kq);
    if (!(lane & 1)) *o = __bfloat16_as_ushort(__float2bfloat16_rn(ot));
    o += oT;
    const uint64_t a2 = f2(at, at);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float ur = r ? __shfl_xor_sync(0xffffffffu, u, 2 * r) : u;
      const uint64_t u2 = f2(ur, ur);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[r][j] = f2fma(u2, k2[j], f2mul(a2, h[r][j]));
    }
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    ulonglong2* p = reinterpret_cast<ulonglong2*>(st + (r ^ own) * 128);
    __stcs(p, make_ulonglong2(h[r][0], h[r][1]));
    __stcs(p + 1, make_ulonglong2(h[r][2], h[r][3]));
  }
  pdl_wait();  // beside the chunk kernel this one may be through first: what is launched next finds both results
}

}  // namespace reax

namespace reax_host {

inline int delta_check(const reax::DeltaArgs& a) {
  if (a.H <= 0 || a.HV <= 0 || a.HV % a.H || a.HV > 65535) return -2;
  if (a.N < 0 || a.N > 65535 || a.T < 0 || a.S < 0) return -1;
  if (a.N == 0 || a.T == 0) return 0;
  if (!a.q || !a.k || !a.v || !a.beta || !a.g || !a.cu || !a.state || !a.o) return -1;
  if (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.o | (uintptr_t)a.state) & 15) return -1;
  if (a.sS % 4) return -1;
  if (!a.slots && a.N > a.S) return -1;
  return 0;
}

}  // namespace reax_host
