// rgp_ssm.h -- plan of the selective state-space scan, shared by its forward (rgp_ssm_fwd.hip), backward (rgp_ssm_bwd.hip) and host
// side (rgp_ssm.hip).
#pragma once
#include "rgp_seq.h"

#define SSM_R 4                      // states per lane

// Steps between the states that a training forward pass leaves for the backward pass, and the steps the backward kernel holds in
// registers.  Their bytes per (row, channel) are N * sizeof(acc) / CK: 4 at N = 16 for 32-bit states, against 6 to 14 that the activations
// cost; 8 steps for 64-bit ones, whose registers are twice as wide.
template <typename A> struct SsmCk { static constexpr int n = 16; };
template <> struct SsmCk<double> { static constexpr int n = 8; };

struct SsmDev {
  rgp_ssm_scan a;
  SeqGeo g;
  int64_t L;                         // steps per block of the time split
  int64_t nslot;                     // blocks
  int Dg, ncb;                       // channels per group, channel blocks per group
  int wu, wd, wz, wgy, wout;         // 16-byte accesses possible: u, delta, z, gy, outputs
  void* part;                        // state (forward) or adjoint (backward) that every block starts from [nslot][D][N]
  void* sumdt;                       // sum of dt over a block [nslot][D]
  void *pA, *pD, *pBC;               // partial sums of the backward pass: [nslot][D][N], [nslot][2][D], [ncb][rows][2][G][N]
};

// fwd: mode 0 = the whole operator, 1 = what a block adds to the state and its sum of dt; bwd likewise with the adjoint
hipError_t ssm_fwd_launch(const SsmDev& d, int K, int CH, int mode, hipStream_t s);
hipError_t ssm_bwd_launch(const SsmDev& d, int K, int CH, int mode, hipStream_t s);
