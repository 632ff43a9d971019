// rgp_ssm_fwd.hip -- forward kernel of the selective state-space scan
//     dt = softplus(delta + bias);  s[n] = exp(dt A[n]) s[n] + dt u B[n];  y = (sum_n C[n] s[n] + skip u) silu(z).
// K lanes hold one channel's states, SSM_R each; a workgroup holds CH channels of one group of B / C and walks its block of time in tiles
// of TL steps.  What is elementwise over (step, channel) -- softplus, silu, the loads and stores, 16 bytes a lane -- runs with the lanes
// over the tile's elements; between them the recurrence reads (dt, dt u) and the rows of B and C from LDS and leaves y there.  The next
// tile's loads are in flight while a tile is walked.
#include "rgp_ssm.h"

template <typename T, int K, int CH, int MODE>
static __global__ void __launch_bounds__(CH* K) ssm_fwd_kernel(SsmDev d) {
  typedef typename SeqAcc<T>::type A;
  constexpr int THREADS = CH * K, V = SeqVec<T>::V, NV = CH / V, TL = sizeof(A) == 8 ? 16 : 32, NP = SSM_R * K, R = SSM_R;
  constexpr int ITEMS = TL * NV, NI = (ITEMS + THREADS - 1) / THREADS, NB = (TL * NP + THREADS - 1) / THREADS, CK = SsmCk<A>::n;
  struct alignas(2 * sizeof(A)) Pair { A dt, w; };
  struct alignas(16) Quad { A v[R]; };
  __shared__ Pair pl[TL][CH];
  __shared__ Quad Bl[TL][K];
  __shared__ Quad Cl[MODE == 0 ? TL : 1][K];
  const rgp_ssm_scan& a = d.a;
  const int tid = threadIdx.x;
  const int64_t nchb = (int64_t)a.G * d.ncb;
  const int64_t slot = blockIdx.x / nchb;
  const int cb = (int)(blockIdx.x - slot * nchb), grp = cb / d.ncb, c0 = (cb - grp * d.ncb) * CH;      // first channel, inside the group
  const SeqBlock b = seq_find(d.g, slot, d.L);
  if (!b.ok) {
    if (MODE == 0 && a.last && b.len == 0 && b.j == 0) {         // a sequence without steps hands its state on
      const int c = c0 + (int)threadIdx.x / K, n0 = (int)threadIdx.x % K * R;
      if (c < d.Dg)
        for (int r = n0; r < n0 + R && r < a.N; ++r) {
          const int64_t at = (b.seq * a.D + grp * d.Dg + c) * a.N + r;
          ((A*)a.last)[at] = a.init ? ((const A*)a.init)[at] : (A)0;
        }
    }
    return;
  }
  const int64_t t0 = b.j * d.L, t1 = t0 + d.L < b.len ? t0 + d.L : b.len;
  const int N = a.N, chn = d.Dg - c0 < CH ? d.Dg - c0 : CH;      // channels of this block
  const int ch0 = grp * d.Dg + c0;                               // first channel

  // elementwise role: vector v of the rows tid / NV, tid / NV + THREADS / NV, ...
  const int ev = tid % NV, et = tid / NV, eval = chn - ev * V < 0 ? 0 : (chn - ev * V < V ? chn - ev * V : V);
  const int ech = ch0 + ev * V;
  A bias[V], skip[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias && i < eval ? ((const A*)a.bias)[ech + i] : (A)0;
    skip[i] = MODE == 0 && a.skip && i < eval ? ((const A*)a.skip)[ech + i] : (A)0;
  }
  // recurrence role: states k R .. k R + R - 1 of channel ch
  const int ch = tid / K, k = tid % K;
  const bool live = ch < chn;
  A Ar[R], s[R], sum = (A)0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool ok = live && k * R + r < N;
    Ar[r] = ok ? ((const A*)a.A)[(int64_t)(ch0 + ch) * N + k * R + r] : (A)0;
    if (sizeof(A) == 4) Ar[r] *= (A)1.44269504088896341;          // exp(dt A) = 2^(dt A log2 e)
    s[r] = (A)0;
    if (MODE == 0 && ok) {
      if (d.part) s[r] = ((const A*)d.part)[(slot * a.D + ch0 + ch) * N + k * R + r];
      else if (a.init) s[r] = ((const A*)a.init)[(b.seq * a.D + ch0 + ch) * N + k * R + r];
    }
  }
  A* const ckpt = MODE == 0 && a.states ? (A*)a.states + ((seq_slot0(d.g, b.seq, b.start, CK)) * a.D + ch0 + ch) * N + k * R : nullptr;
  const SeqStride su{a.u_st, a.u_sb}, sd{a.delta_st, a.delta_sb}, sz{a.z_st, a.z_sb}, sB{a.B_st, a.B_sb}, sC{a.C_st, a.C_sb};

  SeqVec<T> ru[NI], rd[NI], rz[NI];
  T rB[NB], rC[NB];
  auto fetch = [&](int64_t tt) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int tl = et + i * (THREADS / NV);
      const int n = tl < TL && tt + tl < t1 ? eval : 0;
      const int64_t t = n ? tt + tl : t0;                        // an address inside the block even where nothing is read
      ru[i] = seq_load(seq_row((const T*)a.u, d.g, b, su, t) + ech, n, d.wu);
      rd[i] = seq_load(seq_row((const T*)a.delta, d.g, b, sd, t) + ech, n, d.wd);
      if (MODE == 0 && a.z) rz[i] = seq_load(seq_row((const T*)a.z, d.g, b, sz, t) + ech, n, d.wz);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
      const bool ok = tl < TL && n < N && tt + tl < t1;
      const int64_t t = ok ? tt + tl : t0;
      rB[i] = ok ? seq_row((const T*)a.B, d.g, b, sB, t)[(int64_t)grp * N + n] : (T)0;
      if (MODE == 0) rC[i] = ok ? seq_row((const T*)a.C, d.g, b, sC, t)[(int64_t)grp * N + n] : (T)0;
    }
  };
  fetch(t0);
  for (int64_t tt = t0; tt < t1; tt += TL) {
    const int nt = t1 - tt < TL ? (int)(t1 - tt) : TL;
    SeqVec<T> cu[NI], cz[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int tl = et + i * (THREADS / NV);
      cu[i] = ru[i];
      if (MODE == 0) cz[i] = rz[i];
      if (tl < TL) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          A sig;
          const A dt = seq_softplus((A)rd[i].e[j] + bias[j], sig);
          Pair p;
          p.dt = dt;
          p.w = dt * (A)ru[i].e[j];
          pl[tl][ev * V + j] = p;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
      if (tl < TL) {
        Bl[tl][n / R].v[n % R] = (A)rB[i];
        if (MODE == 0) Cl[tl][n / R].v[n % R] = (A)rC[i];
      }
    }
    __syncthreads();
    if (tt + TL < t1) fetch(tt + TL);
    for (int tb = 0; tb < nt; tb += CK) {
      if (MODE == 0 && ckpt && live) {
        A* const c = ckpt + (tt + tb) / CK * ((int64_t)a.D * N);
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (k * R + r < N) c[r] = s[r];
      }
#pragma unroll
      for (int i = 0; i < CK; ++i) {
        const int t = tb + i;
        if (t < nt) {
          const Pair p = pl[t][ch];
          const Quad B = Bl[t][k];
          A acc = (A)0;
          if (MODE == 1) sum += p.dt;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const A e = sizeof(A) == 4 ? (A)seq_exp2((float)(p.dt * Ar[r])) : seq_exp(p.dt * Ar[r]);
            s[r] = e * s[r] + p.w * B.v[r];
            if (MODE == 0) acc += s[r] * Cl[t][k].v[r];
          }
          if (MODE == 0) {
            acc = seq_sum<K>(acc);
            if (k == 0) pl[t][ch].dt = acc;
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
          SeqVec<T> o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            A y = pl[tl][ev * V + j].dt + skip[j] * (A)cu[i].e[j];
            if (a.z) {
              A comp;
              const A z = (A)cz[i].e[j];
              y *= z * seq_sigmoid(z, comp);
            }
            o.e[j] = (T)y;
          }
          seq_store((T*)a.y + seq_row_index(d.g, b, tt + tl) * a.D + ech, o, eval, d.wout);
        }
      }
    }
  }
  if (MODE == 0 && a.last && t1 == b.len && live) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (k * R + r < N) ((A*)a.last)[(b.seq * a.D + ch0 + ch) * N + k * R + r] = s[r];
  }
  if (MODE == 1 && live) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (k * R + r < N) ((A*)d.part)[(slot * a.D + ch0 + ch) * N + k * R + r] = s[r];
    if (k == 0) ((A*)d.sumdt)[slot * a.D + ch0 + ch] = sum;
  }
}

template <typename T, int K, int CH>
static hipError_t go(const SsmDev& d, int mode, hipStream_t s) {
  const int64_t grid = d.nslot * d.a.G * d.ncb;
  if (mode == 0) hipLaunchKernelGGL((ssm_fwd_kernel<T, K, CH, 0>), dim3((unsigned)grid), dim3(CH * K), 0, s, d);
  else hipLaunchKernelGGL((ssm_fwd_kernel<T, K, CH, 1>), dim3((unsigned)grid), dim3(CH * K), 0, s, d);
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
hipError_t ssm_fwd_launch(const SsmDev& d, int K, int CH, int mode, hipStream_t s) {
  switch (d.a.dtype) {
    case RGP_F64: return pick<double>(d, K, CH, mode, s);
    case RGP_F32: return pick<float>(d, K, CH, mode, s);
    case RGP_BF16: return pick<__bf16>(d, K, CH, mode, s);
    default: return pick<_Float16>(d, K, CH, mode, s);
  }
}
