// rgp_ssm.h -- plan of the selective state-space scan, shared by its forward (rgp_ssm_fwd.hip), backward (rgp_ssm_bwd.hip) and host
// side (rgp_ssm.hip).
#pragma once
#include "rgp_seq.h"


// Steps between the states that a training forward pass leaves for the backward pass, and the steps whose states and decays the backward
// kernel holds in registers.  At N = 16 their bytes per (row, channel) are 8 in 32 bits; 16 steps would halve that but need 64 registers
// more, and the kernel is bound by the latency of one wave per SIMD then.
#define SSM_CK_LG 3
#define SSM_CK (1 << SSM_CK_LG)
// A step behind the end of a block has dt = u = gp = 0 and changes nothing: its decay is exp(0 A) = 1.  For that A must be finite:
// minus infinity (forget everything) is held as a value whose product with the dt of any real step still decays to 0, likewise plus
// infinity (2e38 log2 e is still finite in 32 bits).
template <typename A> static __device__ __forceinline__ A ssm_finite(A a) {
  const A most = sizeof(A) == 4 ? (A)2.0e38f : (A)1.0e308;
  return a < -most ? -most : a > most ? most : a;
}

// What a block with decay e makes of the state s that enters it.  Where A is positive the product of many decays may be infinite: a state of zero
// stays zero all the same.
template <typename A> static __device__ __forceinline__ A ssm_through(A e, A s) { return s == (A)0 ? (A)0 : e * s; }

// Where channel c of a tile's row stands in LDS.  A thread writes V neighbouring channels, so at any one of its writes the wave's lanes are V
// entries apart and would meet in the same banks; the place is c with its low bits exchanged by the number of the 128-byte line, which puts
// those lanes side by side and leaves neighbouring channels in one line for the recurrence.
template <int V, int BYTES>
static __device__ __forceinline__ int ssm_place(int c) {
  constexpr int SH = BYTES == 8 ? 4 : BYTES == 16 ? 3 : 2;
  return V == 1 ? c : c ^ ((c >> SH) & (V - 1));
}

// Elements of a thread's vector in the element role: 16 bytes, fewer where a tile's vectors would not go round the CH K threads (CH TL / V = CH K):
// 4096 x 1024 bf16, N = 32, backward 179 us with 16 bytes and a quarter of the threads at work, 152 with 8 and all of them.
constexpr int ssm_vec(int bytes, int TL, int K) { return TL / K < 16 / bytes ? (TL > K ? TL / K : 1) : 16 / bytes; }
constexpr int ssm_fwd_tile(int bytes, int K) { return bytes == 8 || K <= 2 ? 16 : 32; }
constexpr int ssm_bwd_tile(int bytes, int K, int CH) { return bytes == 8 ? 8 : bytes == 2 && CH * K == 256 && (K == 4 || K == 8) ? 32 : 16; }

struct SsmShape { int K, R, CH; };   // lanes a channel, states a lane, channels a workgroup

struct SsmDev {
  rgp_ssm_scan a;
  SeqGeo g;
  int lg;                            // the time split has blocks of L = 2^lg steps
  int64_t L;
  int64_t nslot;                     // blocks
  int join;                          // every block joins the sums of the blocks before it (behind it) by itself
  int Dg, ncb;                       // channels per group, channel blocks per group
  int wide;                          // activations in 16-byte vectors, at any element's address: no workgroup has fewer channels than a vector
  void* part;                        // state (forward) or adjoint (backward) that every block starts from [nslot][D][N]
  void* sumdt;                       // sum of dt over a block [nslot][D]
  void *pA, *pD, *pBC;               // partial sums of the backward pass: [nslot][D][N], [nslot][2][D], [ncb][rows][2][G][N]
};

// What enters block b: s (the initial state, or zero) through the sums that the first walk left of the blocks before it -- behind it for the
// adjoint.  R states of one channel from n0 on; decay(sum of dt, r) is a block's.
template <bool BACK, int R, typename A, typename F>
static __device__ __forceinline__ void ssm_enter(const SsmDev& d, const SeqBlock& b, int ch, int n0, A (&s)[R], F decay) {
  constexpr int U = 4;
  const int64_t DN = (int64_t)d.a.D * d.a.N, last = ((b.len + d.L - 1) >> d.lg) - 1, step = (d.g.off ? 1 : (int64_t)d.g.n_seq) * (BACK ? -1 : 1);
  const int64_t slot = seq_slot(d.g, b.seq, b.start, d.lg, BACK ? last : 0), dp = step * DN, dq = step * d.a.D;
  const A* p = (const A*)d.part + slot * DN + (int64_t)ch * d.a.N + n0;
  const A* q = (const A*)d.sumdt + slot * d.a.D + ch;
  for (int left = (int)(BACK ? last - b.j : b.j); left > 0; left -= U, p += U * dp, q += U * dq) {
    A h[U][R], t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {                                  // read together
      const int k = u < left ? u : 0;
      t[u] = q[k * dq];
#pragma unroll
      for (int r = 0; r < R; ++r) h[u][r] = n0 + r < d.a.N ? p[k * dp + r] : (A)0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < left) {
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = ssm_through(decay(t[u], r), s[r]) + h[u][r];
      }
  }
}

// fwd: mode 0 = the whole operator, 1 = what a block adds to the state and its sum of dt; bwd likewise with the adjoint
hipError_t ssm_fwd_launch(const SsmDev& d, SsmShape p, int mode, hipStream_t s);
hipError_t ssm_bwd_launch(const SsmDev& d, SsmShape p, int mode, hipStream_t s);
