// rgp_ssm_fwd.hip -- forward kernel of the selective state-space scan
//     dt = softplus(delta + bias);  s[n] = exp(dt A[n]) s[n] + dt u B[n];  y = (sum_n C[n] s[n] + skip u) silu(z).
// K lanes hold one channel's states, R each; a workgroup holds CH channels of one group of B / C and walks its block of time in tiles
// of TL steps.  What is elementwise over (step, channel) -- softplus, silu, the loads and stores -- runs with the lanes over the tile's
// elements, a vector of V (16 bytes) each, the last one moved back to end with the channels; single elements, in every workgroup, where the last
// one has fewer channels than a vector.  Between them the recurrence reads (dt, dt u) and the rows of B and C from LDS and leaves y there.  The next tile's
// loads are in flight while a tile is walked.
// Bound by the vector unit: a step of a wave (64 / K channels) takes 22.6 instructions in the recurrence, 4 of them exponentials at a quarter of
// the rate, and 12 for the elements; the unit is busy 96 % of the kernel's time (SQ_ACTIVE_INST_VALU).  8191 x 1024 bf16, N = 16, training: 49 us,
// and 33 for the walk that only sums the blocks (MODE 1).  8 x 65536 x 64 fp32: 170 us, 3.5 TB/s, and 119.  32 x 4096 x 64 fp64: 200 and 154, the unit
// busy all the time, 99 and 74 instructions a step of a wave with 8 channels.  What else was tried: 8 states a lane
// (fewer lane sums, but half the waves): 58 instead of 49 us.  Registers allow 4 waves a SIMD, which that takes (3: 188 instead of 174 us); with
// one or two lanes a channel, tiles of 16 steps keep the element role in registers (8192 x 2000 fp32, N = 4: 64 us, with 32 steps 110).
#include "rgp_ssm.h"

template <typename T, int K, int R, int CH, int MODE, int V>
static __global__ void __launch_bounds__(CH* K, sizeof(T) < 8 && (K == 4 || K == 8) && CH * K == 256 && V > 1 ? 4 : 1) ssm_fwd_kernel(SsmDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  constexpr int THREADS = CH * K, NV = CH / V, TL = ssm_fwd_tile(sizeof(T), K), NP = R * K, RPI = THREADS / NV;
  constexpr int NI = RPI >= TL ? 1 : TL / RPI, NB = (TL * NP + THREADS - 1) / THREADS, CK = SSM_CK;
  struct alignas(2 * sizeof(A)) Pair { A dt, w; };
  struct alignas(16) Quad { A v[R]; };
  __shared__ Pair pl[TL][CH + (V > 1 ? 4 : 0)];
  __shared__ Quad Bl[TL][K];
  __shared__ Quad Cl[MODE == 0 ? TL : 1][K];
  const rgp_ssm_scan& a = d.a;
  const int tid = threadIdx.x;
  const int64_t slot = blockIdx.x;
  const int grp = (int)blockIdx.y / d.ncb, c0 = ((int)blockIdx.y - grp * d.ncb) * CH;       // group, first channel inside the group
  const SeqBlock b = seq_find(d.g, blockIdx.x, d.lg);
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
  if (MODE == 1 && (b.j + 1) * d.L >= b.len) return;              // nothing follows the last block of a sequence
  const int64_t t0 = b.j * d.L, t1 = t0 + d.L < b.len ? t0 + d.L : b.len;
  const int N = a.N, chn = d.Dg - c0 < CH ? d.Dg - c0 : CH;      // channels of this block
  const int ch0 = grp * d.Dg + c0;                               // first channel

  // Elementwise role: vector ev of the rows et, et + RPI, ... of a tile.  Rows behind the end and channels behind the last one read the
  // last row and the first channel there are, and count as zero.
  const int ev = tid % NV, et = tid / NV;
  const bool here = ev * V < chn && et < TL;
  const int el = !here || ev * V + V <= chn ? ev * V : chn - V, ech = ch0 + (here ? el : 0);       // first channel in the tile, in all
  A bias[V], skip[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias ? ((const A*)a.bias)[ech + i] : (A)0;
    skip[i] = MODE == 0 && a.skip ? ((const A*)a.skip)[ech + i] : (A)0;
  }
  // recurrence role: states k R .. k R + R - 1 of channel ch
  const int ch = tid / K, k = tid % K, cp = ssm_place<V, sizeof(Pair)>(ch);
  const bool live = ch < chn;
  A Ar[R], s[R], sum = (A)0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool ok = live && k * R + r < N;
    Ar[r] = ok ? ((const A*)a.A)[(int64_t)(ch0 + ch) * N + k * R + r] : (A)0;
    Ar[r] = ssm_finite(Ar[r]);
    if (sizeof(A) == 4) Ar[r] *= (A)1.44269504088896341;          // exp(dt A) = 2^(dt A log2 e)
    s[r] = (A)0;
    if (MODE == 0 && ok) {
      if (d.part && !d.join) s[r] = ((const A*)d.part)[(slot * a.D + ch0 + ch) * N + k * R + r];
      else if (a.init) s[r] = ((const A*)a.init)[(b.seq * a.D + ch0 + ch) * N + k * R + r];
    }
  }
  auto decay = [&](A dt, int r) { return sizeof(A) == 4 ? (A)seq_exp2((float)(dt * Ar[r])) : seq_exp(dt * Ar[r]); };
  if (MODE == 0 && d.join && live) ssm_enter<false>(d, b, ch0 + ch, k * R, s, decay);
  // the states of the block: every CK steps, a stride of cks values apart
  A* const ckpt = MODE == 0 && a.states ? (A*)a.states + (seq_slot(d.g, b.seq, b.start, SSM_CK_LG, t0 >> SSM_CK_LG) * a.D + ch0 + ch) * N + k * R : nullptr;
  const int64_t cks = (d.g.off ? 1 : (int64_t)d.g.n_seq) * a.D * N;
  const SeqStride su{a.u_st, a.u_sb}, sd{a.delta_st, a.delta_sb}, sz{a.z_st, a.z_sb}, sB{a.B_st, a.B_sb}, sC{a.C_st, a.C_sb};

  Vec ru[NI], rd[NI], rz[NI];
  T rB[NB], rC[NB];
  auto fetch = [&](int64_t tt) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t at = tt + et + i * RPI, t = at < t1 ? at : t1 - 1;
      ru[i] = *(const Vec*)(seq_row((const T*)a.u, d.g, b, su, t) + ech);
      rd[i] = *(const Vec*)(seq_row((const T*)a.delta, d.g, b, sd, t) + ech);
      if (MODE == 0 && a.z) rz[i] = *(const Vec*)(seq_row((const T*)a.z, d.g, b, sz, t) + ech);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, n = e % NP < N ? e % NP : 0;
      const int64_t at = tt + e / NP, t = at < t1 ? at : t1 - 1;
      rB[i] = seq_row((const T*)a.B, d.g, b, sB, t)[(int64_t)grp * N + n];
      if (MODE == 0) rC[i] = seq_row((const T*)a.C, d.g, b, sC, t)[(int64_t)grp * N + n];
    }
  };
  fetch(t0);
  for (int64_t tt = t0; tt < t1; tt += TL) {
    const int nt = t1 - tt < TL ? (int)(t1 - tt) : TL;
    Vec cu[NI], cz[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int tl = et + i * RPI;
      cu[i] = ru[i];
      if (MODE == 0) cz[i] = rz[i];
      if (et < TL) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          A sig;
          const A dt = seq_softplus((A)rd[i].e[j] + bias[j], sig);
          Pair p;
          p.dt = dt;
          p.w = dt * (A)ru[i].e[j];
          pl[tl][ssm_place<V, sizeof(Pair)>(el + j)] = p;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
      if (TL * NP % THREADS == 0 || tl < TL) {
        Bl[tl][n / R].v[n % R] = (A)rB[i];
        if (MODE == 0) Cl[tl][n / R].v[n % R] = (A)rC[i];
      }
    }
    if (nt < TL || N < NP) {                                       // the same threads take back what is behind the end
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int tl = et + i * RPI;
        if (et < TL && tl >= nt) {
#pragma unroll
          for (int j = 0; j < V; ++j) pl[tl][ssm_place<V, sizeof(Pair)>(el + j)] = Pair{(A)0, (A)0};
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int e = tid + i * THREADS, tl = e / NP, n = e % NP;
        if ((TL * NP % THREADS == 0 || tl < TL) && (n >= N || tl >= nt)) {
          Bl[tl][n / R].v[n % R] = (A)0;
          if (MODE == 0) Cl[tl][n / R].v[n % R] = (A)0;
        }
      }
    }
    __syncthreads();
    if (tt + TL < t1) fetch(tt + TL);
    for (int tb = 0; tb < nt; tb += CK) {
      if (MODE == 0 && ckpt && live) {
        A* const c = ckpt + (int)((tt + tb - t0) >> SSM_CK_LG) * cks;
        if (N == NP) {
#pragma unroll
          for (int r = 0; r < R; ++r) c[r] = s[r];
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (k * R + r < N) c[r] = s[r];
        }
      }
#pragma unroll
      for (int i = 0; i < CK; ++i) {
        const int t = tb + i;                                     // steps behind the end change nothing
        const Pair p = pl[t][cp];
        const Quad B = Bl[t][k];
        A acc = (A)0;
        if (MODE == 1) sum += p.dt;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[r] = decay(p.dt, r) * s[r] + p.w * B.v[r];
          if (MODE == 0) acc += s[r] * Cl[t][k].v[r];
        }
        if (MODE == 0) {
          acc = seq_sum<K>(acc);
          pl[t][cp].dt = acc;                                     // all K lanes, the same value
        }
      }
    }
    __syncthreads();
    if (MODE == 0) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int tl = et + i * RPI;
        if (here && tl < nt) {
          Vec o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            A y = pl[tl][ssm_place<V, sizeof(Pair)>(el + j)].dt + skip[j] * (A)cu[i].e[j];
            if (a.z) {
              const A z = (A)cz[i].e[j];
              y *= z * seq_sigmoid(z);
            }
            o.e[j] = (T)y;
          }
          *(Vec*)((T*)a.y + seq_row_index(d.g, b, tt + tl) * a.D + ech) = o;
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

template <typename T, int K, int R, int CH>
static hipError_t go(const SsmDev& d, int mode, hipStream_t s) {
  constexpr int V = ssm_vec(sizeof(T), ssm_fwd_tile(sizeof(T), K), K);
  const dim3 g((unsigned)d.nslot, (unsigned)(d.a.G * d.ncb)), t(CH * K);
  if (mode == 0 && d.wide) hipLaunchKernelGGL((ssm_fwd_kernel<T, K, R, CH, 0, V>), g, t, 0, s, d);
  else if (mode == 0) hipLaunchKernelGGL((ssm_fwd_kernel<T, K, R, CH, 0, 1>), g, t, 0, s, d);
  else if (d.wide) hipLaunchKernelGGL((ssm_fwd_kernel<T, K, R, CH, 1, V>), g, t, 0, s, d);
  else hipLaunchKernelGGL((ssm_fwd_kernel<T, K, R, CH, 1, 1>), g, t, 0, s, d);
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
hipError_t ssm_fwd_launch(const SsmDev& d, SsmShape p, int mode, hipStream_t s) {
  switch (d.a.dtype) {
    case RGP_F64: return pick<double>(d, p, mode, s);
    case RGP_F32: return pick<float>(d, p, mode, s);
    case RGP_BF16: return pick<__bf16>(d, p, mode, s);
    default: return pick<_Float16>(d, p, mode, s);
  }
}
