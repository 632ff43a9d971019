// rgp_ssm_bwd.hip -- backward kernel of the selective state-space scan.  With gp = dL/dp (gy times silu(z)), a = exp(dt A) and the adjoint
//     lam_t[n] = C_t[n] gp_t + a_{t+1}[n] lam_{t+1}[n]
// the gradients are
//     gu = dt sum_n lam B + skip gp;   gdelta = sigmoid(delta + bias) (u sum_n lam B + sum_n lam a s_{t-1} A);
//     gB[n] = sum_d lam dt u;  gC[n] = sum_d gp s;  gA[n] = sum_t lam a s_{t-1} dt;  gskip = sum_t gp u;  gz = gy p silu'(z).
// The work is laid out as in the forward pass.  A tile is CK steps: it starts from a state that the forward pass left every CK steps, keeps
// the tile's states and decays in registers, then walks back.  Running the recurrence backwards instead (s_{t-1} = (s_t - dt u B) / a) would
// lose everything for small a.  The sums over channels in gB and gC fold 2 SSM_R values over the wave's channels with half-wave and
// 16-lane register swaps, then over the waves through LDS; what crosses workgroups is written once and summed in a fixed order.
#include "rgp_ssm.h"

template <typename T, int K, int CH, int MODE>
static __global__ void __launch_bounds__(CH* K) ssm_bwd_kernel(SsmDev d) {
  typedef typename SeqAcc<T>::type A;
  constexpr int THREADS = CH * K, V = SeqVec<T>::V, NV = CH / V, CK = SsmCk<A>::n, TL = CK, NP = SSM_R * K, R = SSM_R, WAVES = THREADS / 64;
  constexpr int ITEMS = TL * NV, NI = (ITEMS + THREADS - 1) / THREADS, NB = (TL * NP + THREADS - 1) / THREADS;
  struct alignas(4 * sizeof(A)) Four { A x, y, z, w; };
  struct alignas(16) Quad { A v[R]; };
  __shared__ Four pl[TL][CH];                          // in: dt, u, gp; out: sum lam B, sum lam a s A, sum C s
  __shared__ Quad Bl[MODE == 0 ? TL : 1][K];
  __shared__ Quad Cl[TL][K];
  __shared__ A red[MODE == 0 ? WAVES : 1][MODE == 0 ? TL : 1][2 * NP];
  const rgp_ssm_scan& a = d.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t nchb = (int64_t)a.G * d.ncb;
  const int64_t slot = blockIdx.x / nchb;
  const int cb = (int)(blockIdx.x - slot * nchb), grp = cb / d.ncb, cig = cb - grp * d.ncb, c0 = cig * CH;
  const SeqBlock b = seq_find(d.g, slot, d.L);
  const int N = a.N, chn = d.Dg - c0 < CH ? d.Dg - c0 : CH, ch0 = grp * d.Dg + c0;
  const int ev = tid % NV, et = tid / NV, eval = chn - ev * V < 0 ? 0 : (chn - ev * V < V ? chn - ev * V : V);
  const int ech = ch0 + ev * V;
  const int ch = tid / K, k = tid % K;
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
  const int64_t t0 = b.j * d.L, t1 = t0 + d.L < b.len ? t0 + d.L : b.len;
  A bias[V], skip[V], gD[V], gbias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias && i < eval ? ((const A*)a.bias)[ech + i] : (A)0;
    skip[i] = MODE == 0 && a.skip && i < eval ? ((const A*)a.skip)[ech + i] : (A)0;
    gD[i] = gbias[i] = (A)0;
  }
  A Ar[R], carry[R], gA[R], sum = (A)0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool ok = live && k * R + r < N;
    Ar[r] = ok ? ((const A*)a.A)[(int64_t)(ch0 + ch) * N + k * R + r] : (A)0;
    carry[r] = MODE == 0 && d.part && ok ? ((const A*)d.part)[(slot * a.D + ch0 + ch) * N + k * R + r] : (A)0;
    gA[r] = (A)0;
  }
  const A* const ckpt = MODE == 0 ? (const A*)a.states + (seq_slot0(d.g, b.seq, b.start, CK) * a.D + ch0 + ch) * N + k * R : nullptr;
  const SeqStride su{a.u_st, a.u_sb}, sd{a.delta_st, a.delta_sb}, sz{a.z_st, a.z_sb}, sB{a.B_st, a.B_sb}, sC{a.C_st, a.C_sb}, sg{a.gy_st, a.gy_sb};
  auto decay = [&](A dt, int r) {
    return sizeof(A) == 4 ? (A)seq_exp2((float)(dt * (Ar[r] * (A)1.44269504088896341))) : seq_exp(dt * Ar[r]);
  };

  SeqVec<T> ru[NI], rd[NI], rz[NI], rg[NI];
  T rB[NB], rC[NB];
  A rs[R];
  auto fetch = [&](int64_t tt) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int tl = et + i * (THREADS / NV);
      const int n = tl < TL && tt + tl < t1 ? eval : 0;
      const int64_t t = n ? tt + tl : t0;
      if (MODE == 0) ru[i] = seq_load(seq_row((const T*)a.u, d.g, b, su, t) + ech, n, d.wu);
      rd[i] = seq_load(seq_row((const T*)a.delta, d.g, b, sd, t) + ech, n, d.wd);
      rg[i] = seq_load(seq_row((const T*)a.gy, d.g, b, sg, t) + ech, n, d.wgy);
      if (a.z) rz[i] = seq_load(seq_row((const T*)a.z, d.g, b, sz, t) + ech, n, d.wz);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
      const bool ok = tl < TL && n < N && tt + tl < t1;
      const int64_t t = ok ? tt + tl : t0;
      if (MODE == 0) rB[i] = ok ? seq_row((const T*)a.B, d.g, b, sB, t)[(int64_t)grp * N + n] : (T)0;
      rC[i] = ok ? seq_row((const T*)a.C, d.g, b, sC, t)[(int64_t)grp * N + n] : (T)0;
    }
    if (MODE == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) rs[r] = live && k * R + r < N ? ckpt[tt / CK * ((int64_t)a.D * N) + r] : (A)0;
    }
  };
  const int64_t last = t0 + (t1 - t0 - 1) / TL * TL;
  fetch(last);
  for (int64_t tt = last; tt >= t0; tt -= TL) {
    const int nt = t1 - tt < TL ? (int)(t1 - tt) : TL;
    SeqVec<T> cu[NI], cz[NI], cg[NI];
    A sig[NI][V], dts[NI][V];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int tl = et + i * (THREADS / NV);
      cu[i] = ru[i];
      cz[i] = rz[i];
      cg[i] = rg[i];
      if (tl < TL) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          Four p;
          p.x = dts[i][j] = seq_softplus((A)rd[i].e[j] + bias[j], sig[i][j]);
          p.y = MODE == 0 ? (A)ru[i].e[j] : (A)0;
          p.z = (A)rg[i].e[j];
          p.w = (A)0;
          if (a.z) {
            A comp;
            const A z = (A)rz[i].e[j];
            p.z *= z * seq_sigmoid(z, comp);
          }
          if (MODE == 0) {
            gD[j] += p.z * p.y;
          }
          pl[tl][ev * V + j] = p;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
      if (tl < TL) {
        if (MODE == 0) Bl[tl][n / R].v[n % R] = (A)rB[i];
        Cl[tl][n / R].v[n % R] = (A)rC[i];
      }
    }
    A s0[R];
    if (MODE == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) s0[r] = rs[r];
    }
    __syncthreads();
    if (tt > t0) fetch(tt - TL);
    if (MODE == 1) {
#pragma unroll
      for (int t = TL - 1; t >= 0; --t) {
        if (t < nt) {
          const Four p = pl[t][ch];
          const Quad C = Cl[t][k];
          sum += p.x;
#pragma unroll
          for (int r = 0; r < R; ++r) carry[r] = (C.v[r] * p.z + carry[r]) * decay(p.x, r);
        }
      }
    } else {
      A s[TL][R], e[TL][R];
#pragma unroll
      for (int t = 0; t < TL; ++t) {
        if (t < nt) {
          const Four p = pl[t][ch];
          const Quad B = Bl[t][k];
          const A w = p.x * p.y;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            e[t][r] = decay(p.x, r);
            s[t][r] = e[t][r] * (t ? s[t ? t - 1 : 0][r] : s0[r]) + w * B.v[r];
          }
        }
      }
#pragma unroll
      for (int t = TL - 1; t >= 0; --t) {
        if (t < nt) {
          const Four p = pl[t][ch];
          const Quad B = Bl[t][k], C = Cl[t][k];
          const A w = p.x * p.y;
          A g1 = (A)0, g2 = (A)0, yd = (A)0, vB[R], vC[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const A lam = C.v[r] * p.z + carry[r];
            vC[r] = p.z * s[t][r];
            vB[r] = lam * w;
            g1 += lam * B.v[r];
            yd += C.v[r] * s[t][r];
            carry[r] = lam * e[t][r];
            const A q = carry[r] * (t ? s[t ? t - 1 : 0][r] : s0[r]);
            g2 += q * Ar[r];
            gA[r] += q * p.x;
          }
          g1 = seq_sum<K>(g1);
          g2 = seq_sum<K>(g2);
          yd = seq_sum<K>(yd);
          if (k == 0) {
            Four o;
            o.x = g1; o.y = g2; o.z = yd; o.w = (A)0;
            pl[t][ch] = o;
          }
          // over the wave's channels: lane bit 5 selects gB / gC, bit 4 and bit 3 the state
          const bool b3 = (lane & 8) != 0;
          A f0 = seq_fold<true>(vB[0], vC[0]), f1 = seq_fold<true>(vB[1], vC[1]), f2 = seq_fold<true>(vB[2], vC[2]), f3 = seq_fold<true>(vB[3], vC[3]);
          f0 = seq_fold<false>(f0, f2);
          f1 = seq_fold<false>(f1, f3);
          A* const o = &red[wave][t][(lane >> 5) * NP + k * R + ((lane >> 4) & 1) * 2];
          if constexpr (K == 16) {
            o[0] = f0;
            o[1] = f1;
          } else {
            A f = seq_fold8(f0, f1, b3);
            if constexpr (K <= 4) f += seq_xor4(f);
            if constexpr (K <= 2) f += seq_dpp<0x4E>(f);
            if constexpr (K == 1) f += seq_dpp<0xB1>(f);
            if ((lane & 7) == k) o[b3] = f;
          }
        }
      }
    }
    __syncthreads();
    if (MODE == 0) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int tl = et + i * (THREADS / NV);
        if (tl < nt && eval > 0) {
          SeqVec<T> ou, od, oz;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const Four p = pl[tl][ev * V + j];
            const A u = (A)cu[i].e[j], gy = (A)cg[i].e[j];
            A gp = gy;
            if (a.z) {
              A comp;
              const A z = (A)cz[i].e[j], sg_ = seq_sigmoid(z, comp);
              gp = gy * (z * sg_);
              oz.e[j] = (T)(gy * (p.z + skip[j] * u) * (sg_ + z * sg_ * comp));
            }
            ou.e[j] = (T)(dts[i][j] * p.x + skip[j] * gp);
            const A graw = (u * p.x + p.y) * sig[i][j];
            gbias[j] += graw;
            od.e[j] = (T)graw;
          }
          const int64_t o = seq_row_index(d.g, b, tt + tl) * a.D + ech;
          seq_store((T*)a.gu + o, ou, eval, d.wout);
          seq_store((T*)a.gdelta + o, od, eval, d.wout);
          if (a.z) seq_store((T*)a.gz + o, oz, eval, d.wout);
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
  // gskip and gbias: the threads that share a vector of channels, through the tile's LDS; only threads below QR saw a row of the tile
  constexpr int QR = THREADS / NV < TL ? THREADS / NV : TL;
  A* const buf = (A*)&pl[0][0];
  static_assert(QR * CH <= TL * CH * 4, "one value per contributing thread and channel of a vector");
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (et < QR) {
#pragma unroll
      for (int j = 0; j < V; ++j) buf[et * CH + ev * V + j] = which ? gbias[j] : gD[j];
    }
    __syncthreads();
    if (tid < chn) {
      A v = (A)0;
      for (int q = 0; q < QR; ++q) v += buf[q * CH + tid];
      ((A*)d.pD)[(slot * 2 + which) * a.D + ch0 + tid] = v;
    }
    __syncthreads();
  }
}

template <typename T, int K, int CH>
static hipError_t go(const SsmDev& d, int mode, hipStream_t s) {
  const int64_t grid = d.nslot * d.a.G * d.ncb;
  if (mode == 0) hipLaunchKernelGGL((ssm_bwd_kernel<T, K, CH, 0>), dim3((unsigned)grid), dim3(CH * K), 0, s, d);
  else hipLaunchKernelGGL((ssm_bwd_kernel<T, K, CH, 1>), dim3((unsigned)grid), dim3(CH * K), 0, s, d);
  return hipGetLastError();
}
template <typename T>
static hipError_t pick(const SsmDev& d, int K, int CH, int mode, hipStream_t s) {
  switch (K) {
    case 1: return go<T, 1, 64>(d, mode, s);
    case 2: return go<T, 2, 64>(d, mode, s);
    case 4: return CH == 16 ? go<T, 4, 16>(d, mode, s) : go<T, 4, 64>(d, mode, s);
    case 8: return go<T, 8, 32>(d, mode, s);
    default: return go<T, 16, 16>(d, mode, s);
  }
}
hipError_t ssm_bwd_launch(const SsmDev& d, int K, int CH, int mode, hipStream_t s) {
  switch (d.a.dtype) {
    case RGP_F64: return pick<double>(d, K, CH, mode, s);
    case RGP_F32: return pick<float>(d, K, CH, mode, s);
    case RGP_BF16: return pick<__bf16>(d, K, CH, mode, s);
    default: return pick<_Float16>(d, K, CH, mode, s);
  }
}
