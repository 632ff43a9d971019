// rgp_ssm_bwd.hip -- backward kernel of the selective state-space scan.  With gp = dL/dp (gy times silu(z)), a = exp(dt A) and the adjoint
//     lam_t[n] = C_t[n] gp_t + a_{t+1}[n] lam_{t+1}[n]
// the gradients are
//     gu = dt sum_n lam B + skip gp;   gdelta = sigmoid(delta + bias) (u sum_n lam B + sum_n lam a s_{t-1} A);
//     gB[n] = sum_d lam dt u;  gC[n] = sum_d gp s;  gA[n] = sum_t lam a s_{t-1} dt;  gskip = sum_t gp u;  gz = gy p silu'(z).
// The work is laid out as in the forward pass.  A tile is walked in pieces of CK steps: each starts from a state that the forward pass left
// there, keeps the piece's states and decays in registers, then walks back.  Running the recurrence backwards instead (s_{t-1} = (s_t - dt u B)
// / a) would lose everything for small a.  The sums over channels in gB and gC fold 2 R values over the wave's channels with half-wave and
// 16-lane register swaps, then over the waves through LDS; what crosses workgroups is written once and summed in a fixed order.
//
// Bound by the vector unit: a step of a wave takes 86 instructions in the recurrence (13 for each of a lane's states, 17 for the sums over
// channels, 6 for those over states) and about 28 for the elements, tiles and partial sums; SQ_ACTIVE_INST_VALU is 0.88 of the busy cycles.
// 8191 x 1024 bf16, N = 16: 139 us, and 39 for the walk that only sums the blocks (MODE 1); 32 x 4096 x 64 fp32: 148 and 38; 8 x 512 x 40
// fp64 in blocks of 16 steps: 21 and 11.  fp64 that fills the card (32 x 4096 x 64: 429 and 186) is bound the same way, by 172 and 85 instructions a
// step of a wave with 8 channels (issue ratios 0.80 and 0.89).  Two waves a SIMD: a tile of 32 steps fits their LDS for 16-bit types with 4 lanes a
// channel, 16 steps elsewhere (with 2 lanes 64 instead of 71 us at 4096 x 1024, N = 8); one lane a channel, and 4 states a lane in fp64, need the
// registers of two.
#include "rgp_ssm.h"

template <typename T, int K, int R, int CH, int MODE, int V>
static __global__ void __launch_bounds__(CH* K, (sizeof(T) == 8 && R == 4) || K == 1 ? 1 : 2) ssm_bwd_kernel(SsmDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  constexpr int THREADS = CH * K, NV = CH / V, RPI = THREADS / NV, CK = SSM_CK, NP = R * K, WAVES = THREADS / 64;
  constexpr int TL = ssm_bwd_tile(sizeof(T), K, CH), SUB = TL / CK;
  constexpr int NI = RPI >= TL ? 1 : TL / RPI, NB = (TL * NP + THREADS - 1) / THREADS;
  struct alignas(4 * sizeof(A)) Four { A x, y, z, w; };
  struct alignas(16) Quad { A v[R]; };
  __shared__ Four pl[TL][CH];                          // in: dt, u, gp, sigmoid(delta + bias); out: gu, gdelta, p
  __shared__ A zf[MODE == 0 ? NI * V : 1][THREADS];     // gy silu'(z), each thread its own
  __shared__ Quad Bl[MODE == 0 ? TL : 1][K];
  __shared__ Quad Cl[TL][K];
  __shared__ A red[MODE == 0 ? WAVES : 1][MODE == 0 ? TL : 1][2 * NP];
  const rgp_ssm_scan& a = d.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t slot = blockIdx.x;
  const int grp = (int)blockIdx.y / d.ncb, cig = (int)blockIdx.y - grp * d.ncb, c0 = cig * CH;
  const SeqBlock b = seq_find(d.g, blockIdx.x, d.lg);
  const int N = a.N, chn = d.Dg - c0 < CH ? d.Dg - c0 : CH, ch0 = grp * d.Dg + c0;
  const int ev = tid % NV, et = tid / NV;               // roles as in the forward kernel
  const bool here = ev * V < chn && et < TL;
  const int el = !here || ev * V + V <= chn ? ev * V : chn - V, ech = ch0 + (here ? el : 0);
  const int ch = tid / K, k = tid % K, cp = ssm_place<V, sizeof(Four)>(ch);
  const bool live = ch < chn;
  if (!b.ok) {                                        // an empty block still owns a row of the partial sums
    if (MODE == 0) {
      if (live)
        for (int r = 0; r < R; ++r)
          if (k * R + r < N) ((A*)d.pA)[(slot * a.D + ch0 + ch) * N + k * R + r] = (A)0;
      if (tid < chn) {
        ((A*)d.pD)[slot * 2 * a.D + ch0 + tid] = (A)0;
        ((A*)d.pD)[(slot * 2 + 1) * a.D + ch0 + tid] = (A)0;
      }
    }
    return;
  }
  if (MODE == 1 && b.j == 0) return;                              // nothing precedes the first block of a sequence
  const int64_t t0 = b.j * d.L, t1 = t0 + d.L < b.len ? t0 + d.L : b.len;
  A bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) bias[i] = a.bias ? ((const A*)a.bias)[ech + i] : (A)0;
  const A skip = MODE == 0 && a.skip && live ? ((const A*)a.skip)[ch0 + ch] : (A)0;
  A gD = (A)0, gbias = (A)0;
  A Ar[R], carry[R], gA[R], sum = (A)0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool ok = live && k * R + r < N;
    Ar[r] = ok ? ssm_finite(((const A*)a.A)[(int64_t)(ch0 + ch) * N + k * R + r]) : (A)0;
    carry[r] = MODE == 0 && d.part && !d.join && ok ? ((const A*)d.part)[(slot * a.D + ch0 + ch) * N + k * R + r] : (A)0;
    gA[r] = (A)0;
  }
  const A* const ckpt = MODE == 0 ? (const A*)a.states + (seq_slot(d.g, b.seq, b.start, SSM_CK_LG, t0 >> SSM_CK_LG) * a.D + ch0 + ch) * N + k * R : nullptr;
  const int64_t cks = (d.g.off ? 1 : (int64_t)d.g.n_seq) * a.D * N;
  const SeqStride su{a.u_st, a.u_sb}, sd{a.delta_st, a.delta_sb}, sz{a.z_st, a.z_sb}, sB{a.B_st, a.B_sb}, sC{a.C_st, a.C_sb}, sg{a.gy_st, a.gy_sb};
  auto decay = [&](A dt, int r) {
    return sizeof(A) == 4 ? (A)seq_exp2((float)(dt * (Ar[r] * (A)1.44269504088896341))) : seq_exp(dt * Ar[r]);
  };
  if (MODE == 0 && d.join && live) ssm_enter<true>(d, b, ch0 + ch, k * R, carry, decay);

  Vec ru[NI], rd[NI], rz[NI], rg[NI];
  T rB[NB], rC[NB];
  auto fetch = [&](int64_t tt) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t at = tt + et + i * RPI, t = at < t1 ? at : t1 - 1;
      if (MODE == 0) ru[i] = *(const Vec*)(seq_row((const T*)a.u, d.g, b, su, t) + ech);
      rd[i] = *(const Vec*)(seq_row((const T*)a.delta, d.g, b, sd, t) + ech);
      rg[i] = *(const Vec*)(seq_row((const T*)a.gy, d.g, b, sg, t) + ech);
      if (a.z) rz[i] = *(const Vec*)(seq_row((const T*)a.z, d.g, b, sz, t) + ech);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, n = e % NP < N ? e % NP : 0;
      const int64_t at = tt + e / NP, t = at < t1 ? at : t1 - 1;
      if (MODE == 0) rB[i] = seq_row((const T*)a.B, d.g, b, sB, t)[(int64_t)grp * N + n];
      rC[i] = seq_row((const T*)a.C, d.g, b, sC, t)[(int64_t)grp * N + n];
    }
  };
  const int64_t last = t0 + (t1 - t0 - 1) / TL * TL;
  fetch(last);
  for (int64_t tt = last; tt >= t0; tt -= TL) {
    const int nt = t1 - tt < TL ? (int)(t1 - tt) : TL;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int tl = et + i * RPI;
      if (et < TL) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          Four p;
          const A dt = seq_softplus((A)rd[i].e[j] + bias[j], p.w);
          p.x = dt;
          p.y = MODE == 0 ? (A)ru[i].e[j] : (A)0;
          A gp = (A)rg[i].e[j];
          if (a.z) {
            const A z = (A)rz[i].e[j], q = gp * seq_sigmoid(z);
            if (MODE == 0) zf[i * V + j][tid] = q + (gp - q) * (z * seq_sigmoid(z));
            gp = z * q;
          }
          p.z = gp;
          pl[tl][ssm_place<V, sizeof(Four)>(el + j)] = p;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
      if (TL * NP % THREADS == 0 || tl < TL) {
        if (MODE == 0) Bl[tl][n / R].v[n % R] = (A)rB[i];
        Cl[tl][n / R].v[n % R] = (A)rC[i];
      }
    }
    if (nt < TL || N < NP || chn < CH) {                           // the same threads take back what is behind the end: all lanes' values are folded below
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int tl = et + i * RPI;
        if (et < TL) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const Four none{(A)0, (A)0, (A)0, (A)0};
            if (tl >= nt) pl[tl][ssm_place<V, sizeof(Four)>(el + j)] = none;
            if (ev * V + j >= chn) pl[tl][ssm_place<V, sizeof(Four)>(ev * V + j)] = none;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
        if ((TL * NP % THREADS == 0 || tl < TL) && (n >= N || tl >= nt)) {
          if (MODE == 0) Bl[tl][n / R].v[n % R] = (A)0;
          Cl[tl][n / R].v[n % R] = (A)0;
        }
      }
    }
    __syncthreads();
    if (tt > t0) fetch(tt - TL);
    if (MODE == 1) {
#pragma unroll
      for (int t = TL - 1; t >= 0; --t) {                         // steps behind the end change nothing
        const Four p = pl[t][cp];
        const Quad C = Cl[t][k];
        sum += p.x;
#pragma unroll
        for (int r = 0; r < R; ++r) carry[r] = (C.v[r] * p.z + carry[r]) * decay(p.x, r);
      }
    } else {
#pragma unroll 1
      for (int sub = SUB - 1; sub >= 0; --sub) {
        const int tb = sub * CK;
        if (tb >= nt) continue;
        A s0[R], s[CK][R], e[CK][R];
#pragma unroll
        for (int r = 0; r < R; ++r) s0[r] = live && k * R + r < N ? ckpt[(int)((tt + tb - t0) >> SSM_CK_LG) * cks + r] : (A)0;
        // operands of a step are read from LDS while the step before is computed
        Four p = pl[tb][cp];
        Quad B = Bl[tb][k], C;
#pragma unroll
        for (int i = 0; i < CK; ++i) {
          const int tn = tb + (i + 1 < CK ? i + 1 : i);
          const Four pn = pl[tn][cp];
          const Quad Bn = Bl[tn][k];
          const A w = p.x * p.y;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            e[i][r] = decay(p.x, r);
            s[i][r] = e[i][r] * (i ? s[i ? i - 1 : 0][r] : s0[r]) + w * B.v[r];
          }
          p = pn;
          B = Bn;
          if (i + 1 == CK) C = Cl[tb + CK - 1][k];
        }
#pragma unroll
        for (int i = CK - 1; i >= 0; --i) {
          const int t = tb + i, tn = t - (i ? 1 : 0);
          const Four pn = pl[tn][cp];
          const Quad Bn = Bl[tn][k], Cn = Cl[tn][k];
          const A w = p.x * p.y;
          A g1 = (A)0, g2 = (A)0, yd = (A)0, vB[R], vC[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const A lam = C.v[r] * p.z + carry[r];
            vC[r] = p.z * s[i][r];
            vB[r] = lam * w;
            g1 += lam * B.v[r];
            yd += C.v[r] * s[i][r];
            carry[r] = lam * e[i][r];
            const A q = carry[r] * (i ? s[i ? i - 1 : 0][r] : s0[r]);
            g2 += q * Ar[r];
            gA[r] += q * p.x;
          }
          g1 = seq_sum<K>(g1);
          g2 = seq_sum<K>(g2);
          yd = seq_sum<K>(yd);
          // the same in all K lanes; lane k writes the k-th (every lane all of them where K < 4), without a branch around the store
          const A o0 = p.x * g1 + skip * p.z, o1 = (p.y * g1 + g2) * p.w, o2 = yd + skip * p.y;
          gD += p.z * p.y;
          gbias += o1;
          if constexpr (K >= 4) {
            ((A*)&pl[t][cp])[k & 3] = (k & 3) == 0 ? o0 : (k & 3) == 1 ? o1 : o2;
          } else {
            Four o;
            o.x = o0; o.y = o1; o.z = o2; o.w = (A)0;
            pl[t][cp] = o;
          }
          // over the wave's channels: lane bit 5 selects gB / gC, bit 4 and (4 states a lane) bit 3 the state
          A* const f_to = &red[wave][t][(lane >> 5) * NP + k * R + ((lane >> 4) & 1) * (R / 2)];
          if constexpr (R == 2) {
            A f = seq_fold<false>(seq_fold<true>(vB[0], vC[0]), seq_fold<true>(vB[1], vC[1]));
            if constexpr (K <= 8) f += seq_dpp<0x128>(f);                  // row_ror:8
            if constexpr (K <= 4) f += seq_xor4(f);
            if constexpr (K <= 2) f += seq_dpp<0x4E>(f);
            f_to[0] = f;                                           // lanes that hold the same sum write it to the same place
          } else {
            const bool b3 = (lane & 8) != 0;
            A f0 = seq_fold<true>(vB[0], vC[0]), f1 = seq_fold<true>(vB[1], vC[1]), f2 = seq_fold<true>(vB[2], vC[2]), f3 = seq_fold<true>(vB[3], vC[3]);
            f0 = seq_fold<false>(f0, f2);
            f1 = seq_fold<false>(f1, f3);
            if constexpr (K == 16) {
              f_to[0] = f0;
              f_to[1] = f1;
            } else {
              A f = seq_fold8(f0, f1, b3);
              if constexpr (K <= 4) f += seq_xor4(f);
              if constexpr (K <= 2) f += seq_dpp<0x4E>(f);
              if constexpr (K == 1) f += seq_dpp<0xB1>(f);
              f_to[b3] = f;
            }
          }
          p = pn;
          B = Bn;
          C = Cn;
        }
      }
    }
    __syncthreads();
    if (MODE == 0) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int tl = et + i * RPI;
        if (here && tl < nt) {
          Vec ou, od, oz;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const Four p = pl[tl][ssm_place<V, sizeof(Four)>(el + j)];
            ou.e[j] = (T)p.x;
            od.e[j] = (T)p.y;
            if (a.z) oz.e[j] = (T)(zf[i * V + j][tid] * p.z);
          }
          const int64_t o = seq_row_index(d.g, b, tt + tl) * a.D + ech;
          *(Vec*)((T*)a.gu + o) = ou;
          *(Vec*)((T*)a.gdelta + o) = od;
          if (a.z) *(Vec*)((T*)a.gz + o) = oz;
        }
      }
      for (int e = tid; e < nt * 2 * NP; e += THREADS) {
        const int tl = e / (2 * NP), w = e % (2 * NP), n = w % NP;
        if (n < N) {
          A v = (A)0;
#pragma unroll
          for (int q = 0; q < WAVES; ++q) v += red[q][tl][w];
          const int64_t row = seq_row_index(d.g, b, tt + tl);
          if (d.ncb == 1) {
            T* const o = (T*)(w < NP ? a.gB : a.gC);
            o[(row * a.G + grp) * N + n] = (T)v;
          } else {
            ((A*)d.pBC)[(((int64_t)cig * 2 + (w >= NP)) * a.rows + row) * a.G * N + (int64_t)grp * N + n] = v;
          }
        }
      }
      __syncthreads();
    }
  }
  if (MODE == 1) {
    if (live) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (k * R + r < N) ((A*)d.part)[(slot * a.D + ch0 + ch) * N + k * R + r] = carry[r];
      if (k == 0) ((A*)d.sumdt)[slot * a.D + ch0 + ch] = sum;
    }
    return;
  }
  if (live) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (k * R + r < N) ((A*)d.pA)[(slot * a.D + ch0 + ch) * N + k * R + r] = gA[r];
  }
  if (live && k == 0) {
    ((A*)d.pD)[slot * 2 * a.D + ch0 + ch] = gD;
    ((A*)d.pD)[(slot * 2 + 1) * a.D + ch0 + ch] = gbias;
  }
}

template <typename T, int K, int R, int CH>
static hipError_t go(const SsmDev& d, int mode, hipStream_t s) {
  constexpr int V = ssm_vec(sizeof(T), ssm_bwd_tile(sizeof(T), K, CH), K);
  const dim3 g((unsigned)d.nslot, (unsigned)(d.a.G * d.ncb)), t(CH * K);
  if (mode == 0 && d.wide) hipLaunchKernelGGL((ssm_bwd_kernel<T, K, R, CH, 0, V>), g, t, 0, s, d);
  else if (mode == 0) hipLaunchKernelGGL((ssm_bwd_kernel<T, K, R, CH, 0, 1>), g, t, 0, s, d);
  else if (d.wide) hipLaunchKernelGGL((ssm_bwd_kernel<T, K, R, CH, 1, V>), g, t, 0, s, d);
  else hipLaunchKernelGGL((ssm_bwd_kernel<T, K, R, CH, 1, 1>), g, t, 0, s, d);
  return hipGetLastError();
}
template <typename T>
static hipError_t pick(const SsmDev& d, SsmShape p, int mode, hipStream_t s) {
  if constexpr (sizeof(T) == 8) {
    switch (p.K) {
      case 2: return go<T, 2, 2, 64>(d, mode, s);
      case 4: return p.CH == 16 ? go<T, 4, 2, 16>(d, mode, s) : go<T, 4, 2, 64>(d, mode, s);
      case 8: return p.CH == 8 ? go<T, 8, 2, 8>(d, mode, s) : go<T, 8, 2, 32>(d, mode, s);
      default: return p.R == 2 ? go<T, 16, 2, 16>(d, mode, s) : go<T, 16, 4, 16>(d, mode, s);
    }
  } else {
    switch (p.K) {
      case 1: return go<T, 1, 4, 64>(d, mode, s);
      case 2: return go<T, 2, 4, 64>(d, mode, s);
      case 4: return p.CH == 16 ? go<T, 4, 4, 16>(d, mode, s) : go<T, 4, 4, 64>(d, mode, s);
      case 8: return go<T, 8, 4, 32>(d, mode, s);
      default: return go<T, 16, 4, 16>(d, mode, s);
    }
  }
}
hipError_t ssm_bwd_launch(const SsmDev& d, SsmShape p, int mode, hipStream_t s) {
  switch (d.a.dtype) {
    case RGP_F64: return pick<double>(d, p, mode, s);
    case RGP_F32: return pick<float>(d, p, mode, s);
    case RGP_BF16: return pick<__bf16>(d, p, mode, s);
    default: return pick<_Float16>(d, p, mode, s);
  }
}
