// rgp_ssm.hip -- host side of the selective state-space scan (argument checks, split over time, work buffer), the kernels that join the
// blocks of the split, the sums over partial results, the scan's form for one step, and the short causal convolution.
#include "rgp_ssm.h"

// ---- sums of partial results in a fixed order -----------------------------------------------------------------------------------------
// 64 outputs a workgroup, 4 threads for each: thread q adds partials q, q + 4, ..., four at a time into separate sums so that the loads
// overlap; the order depends on P alone.
template <typename A, typename O>
static __global__ void __launch_bounds__(256) seq_reduce_kernel(const A* part, int64_t P, int64_t stride, int64_t n, O* out) {
  __shared__ A sh[4][64];
  const int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int q = threadIdx.x >> 6;
  A s0 = (A)0, s1 = (A)0, s2 = (A)0, s3 = (A)0;
  if (i < n) {
    int64_t p = q;
    for (; p + 12 < P; p += 16) {
      s0 += part[p * stride + i];
      s1 += part[(p + 4) * stride + i];
      s2 += part[(p + 8) * stride + i];
      s3 += part[(p + 12) * stride + i];
    }
    for (; p < P; p += 4) s0 += part[p * stride + i];
  }
  sh[q][threadIdx.x & 63] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (q == 0 && i < n) {
    const int l = threadIdx.x;
    out[i] = (O)((sh[0][l] + sh[1][l]) + (sh[2][l] + sh[3][l]));
  }
}
template <typename A, typename O>
static rgp_status reduce_go(rgp_handle h, hipStream_t s, const void* part, int64_t P, int64_t stride, int64_t n, void* out) {
  if (n < 1) return RGP_OK;
  hipLaunchKernelGGL((seq_reduce_kernel<A, O>), dim3((unsigned)((n + 63) / 64)), dim3(256), 0, s, (const A*)part, P, stride, n, (O*)out);
  return seq_launched(h, "sum of partial results");
}
rgp_status seq_reduce(rgp_handle h, hipStream_t s, int acc, int dt, const void* part, int64_t P, int64_t stride, int64_t n, void* out) {
  if (acc == RGP_F64) return reduce_go<double, double>(h, s, part, P, stride, n, out);
  if (dt == RGP_F32) return reduce_go<float, float>(h, s, part, P, stride, n, out);
  if (dt == RGP_BF16) return reduce_go<float, __bf16>(h, s, part, P, stride, n, out);
  return reduce_go<float, _Float16>(h, s, part, P, stride, n, out);
}

// ---- joining the blocks of the time split -----------------------------------------------------------------------------------------------
// part[block] holds what a block adds to the state that enters it; a thread walks one (sequence, channel, state) over the blocks and
// leaves the entering state there.  A whole block multiplies it by exp(A sum dt): the decays of a diagonal recurrence commute.
// back: the same for the adjoint, from the last block to the first.
template <typename A>
static __global__ void __launch_bounds__(256) ssm_join_kernel(SsmDev d, int back) {
  const rgp_ssm_scan& a = d.a;
  const int64_t DN = (int64_t)a.D * a.N, idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t seq = idx / DN, dn = idx - seq * DN, ch = dn / a.N;
  if (seq >= a.n_seq) return;
  int64_t start = seq * d.g.T, len = d.g.T;
  if (d.g.off) {
    start = seq_off(d.g, seq);
    const int64_t end = seq_off(d.g, seq + 1);
    len = end > start ? end - start : 0;
  }
  const int64_t nb = (len + d.L - 1) / d.L, slot0 = seq_slot0(d.g, seq, start, d.L);
  const A Av = ((const A*)a.A)[dn];
  A* const part = (A*)d.part + slot0 * DN + dn;
  const A* const sum = (const A*)d.sumdt + slot0 * a.D + ch;
  A s = !back && a.init ? ((const A*)a.init)[seq * DN + dn] : (A)0;
  constexpr int U = 8;
  for (int64_t j = 0; j < nb; j += U) {
    A p[U], q[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t jj = j + i < nb ? j + i : nb - 1, at = back ? nb - 1 - jj : jj;
      p[i] = part[at * DN];
      q[i] = seq_exp(Av * sum[at * a.D]);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (j + i < nb) {
        part[(back ? nb - 1 - (j + i) : j + i) * DN] = s;
        s = q[i] * s + p[i];
      }
    }
  }
}

// ---- host side of the scan --------------------------------------------------------------------------------------------------------------
static const char* scan_bad(const rgp_ssm_scan* a) {
  if (!a) return "null arguments";
  if (a->dtype < 0 || a->dtype > 3) return "dtype must be RGP_F64, RGP_F32, RGP_BF16 or RGP_F16";
  if (a->n_seq < 1 || a->D < 1 || a->N < 1 || a->G < 1 || a->rows < 0 || a->T < 0) return "empty problem";
  if (a->N > 64) return "at most 64 states per channel";
  if (a->D % a->G) return "D must be a multiple of G";
  if (!a->off && (a->T < 1 || a->T * a->n_seq != a->rows)) return "rows must be T * n_seq, T >= 1";
  return nullptr;
}

struct ScanPlan {
  SsmDev d;
  int K, CH, acc;
  bool split;
  int64_t part_bytes, sum_bytes, pA_bytes, pD_bytes, pBC_bytes, bytes;
};
static int64_t up256(int64_t b) { return (b + 255) & ~(int64_t)255; }

static void scan_plan(const rgp_ssm_scan* a, bool back, ScanPlan& p) {
  SsmDev& d = p.d;
  d = SsmDev{};
  d.a = *a;
  d.g = SeqGeo{a->off, a->T, a->rows, a->n_seq, a->reverse};
  d.Dg = a->D / a->G;
  p.acc = a->dtype == RGP_F64 ? 8 : 4;
  p.K = a->N <= 4 ? 1 : a->N <= 8 ? 2 : a->N <= 16 ? 4 : a->N <= 32 ? 8 : 16;
  p.CH = p.K <= 4 ? 64 : 256 / p.K;
  if (p.K == 4 && (d.Dg + 15) / 16 * 16 < (d.Dg + 63) / 64 * 64) p.CH = 16;
  d.ncb = (d.Dg + p.CH - 1) / p.CH;
  const int64_t longest = a->off ? (a->max_len > 0 && a->max_len < a->rows ? a->max_len : a->rows) : a->T;
  // Split over time where whole sequences would leave most of the card's 1024 SIMDs without a wave: a split walks every step twice.
  const int64_t waves = (int64_t)a->n_seq * a->G * d.ncb * (p.CH * p.K / 64);
  const double mean = (double)a->rows / a->n_seq;
  int64_t L = 0;
  const double want = 2048.0;
  if (longest >= 256) {
    const double one = (double)longest + (double)waves * mean / 2048.0;           // steps of the longest sequence, and of the whole work
    int64_t l = (int64_t)(waves * mean / want);
    l = (l + 63) / 64 * 64;
    if (l < 64) l = 64;
    const double two = 1.8 * ((double)l + (double)waves * mean / 2048.0) + 100.0;
    if (two < one) L = l;
  }
  p.split = L > 0;
  d.L = p.split ? L : (a->off ? (a->rows + 63) / 64 * 64 : (a->T + 63) / 64 * 64);
  if (d.L < 64) d.L = 64;
  d.nslot = seq_blocks(d.g, d.L);
  const int64_t DN = (int64_t)a->D * a->N;
  p.part_bytes = p.split ? up256(d.nslot * DN * p.acc) : 0;
  p.sum_bytes = p.split ? up256(d.nslot * a->D * p.acc) : 0;
  p.pA_bytes = back ? up256(d.nslot * DN * p.acc) : 0;
  p.pD_bytes = back ? up256(d.nslot * 2 * a->D * p.acc) : 0;
  p.pBC_bytes = back && d.ncb > 1 ? up256((int64_t)d.ncb * 2 * a->rows * a->G * a->N * p.acc) : 0;
  p.bytes = p.part_bytes + p.sum_bytes + p.pA_bytes + p.pD_bytes + p.pBC_bytes;
}

extern "C" int64_t rgp_ssm_scan_workspace(const rgp_ssm_scan* a, int backward) {
  if (scan_bad(a)) return -1;
  ScanPlan p;
  scan_plan(a, backward != 0, p);
  return p.bytes;
}
extern "C" int64_t rgp_ssm_scan_states_bytes(const rgp_ssm_scan* a) {
  if (scan_bad(a)) return -1;
  const SeqGeo g{a->off, a->T, a->rows, a->n_seq, a->reverse};
  const int ck = a->dtype == RGP_F64 ? SsmCk<double>::n : SsmCk<float>::n;
  return seq_blocks(g, ck) * a->D * a->N * (a->dtype == RGP_F64 ? 8 : 4);
}

static rgp_status scan_run(rgp_handle h, hipStream_t s, const rgp_ssm_scan* a, bool back) {
  const char* const what = back ? "ssm scan backward: " : "ssm scan forward: ";
  if (const char* bad = scan_bad(a)) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + bad);
  const bool some = a->rows > 0;                       // without rows the activations may have no memory
  if (!a->A || (some && (!a->u || !a->delta || !a->B || !a->C))) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "u, delta, A, B and C are required");
  if (!back && some && !a->y) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "y is required");
  if (back && (!a->gA || (some && (!a->gy || !a->states || !a->gu || !a->gdelta || !a->gB || !a->gC || (a->z && !a->gz)))))
    return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "gy, states and the gradients' buffers are required");
  ScanPlan p;
  scan_plan(a, back, p);
  SsmDev& d = p.d;
  if (p.bytes > a->work_bytes || (p.bytes && !a->work) || ((uintptr_t)a->work & 15))
    return rgp_fail(h, RGP_ERR_WORKSPACE, std::string(what) + "work buffer too small or not 16-byte aligned");
  const int e = seq_dtype_bytes(a->dtype), V = 16 / e;
  const bool groups = a->G == 1 || d.Dg % V == 0;
  d.wu = groups && seq_aligned(a->u, a->u_st, a->u_sb, e);
  d.wd = groups && seq_aligned(a->delta, a->delta_st, a->delta_sb, e);
  d.wz = groups && a->z && seq_aligned(a->z, a->z_st, a->z_sb, e);
  d.wgy = groups && back && seq_aligned(a->gy, a->gy_st, a->gy_sb, e);
  d.wout = groups && a->D % V == 0 && (back ? seq_aligned(a->gu, 0, 0, e) && seq_aligned(a->gdelta, 0, 0, e) && (!a->z || seq_aligned(a->gz, 0, 0, e))
                                             : seq_aligned(a->y, 0, 0, e));
  char* w = (char*)a->work;
  auto take = [&](int64_t bytes) { void* r = bytes ? (void*)w : nullptr; w += bytes; return r; };
  d.part = take(p.part_bytes);
  d.sumdt = take(p.sum_bytes);
  d.pA = take(p.pA_bytes);
  d.pD = take(p.pD_bytes);
  d.pBC = take(p.pBC_bytes);
  if ((double)d.nslot * a->G * d.ncb * p.CH * p.K > 4294967295.0 || (double)a->n_seq * a->D * a->N > 1.0e12)
    return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "more than 2^32 work items");
  const int64_t DN = (int64_t)a->D * a->N;
  const unsigned join = (unsigned)((a->n_seq * DN + 255) / 256);
  hipError_t err = hipSuccess;
  if (d.nslot > 0) {
    if (p.split) {
      err = back ? ssm_bwd_launch(d, p.K, p.CH, 1, s) : ssm_fwd_launch(d, p.K, p.CH, 1, s);
      if (err == hipSuccess) {
        if (p.acc == 8) hipLaunchKernelGGL(ssm_join_kernel<double>, dim3(join), dim3(256), 0, s, d, back ? 1 : 0);
        else hipLaunchKernelGGL(ssm_join_kernel<float>, dim3(join), dim3(256), 0, s, d, back ? 1 : 0);
        err = hipGetLastError();
      }
    }
    if (err == hipSuccess) err = back ? ssm_bwd_launch(d, p.K, p.CH, 0, s) : ssm_fwd_launch(d, p.K, p.CH, 0, s);
    if (err != hipSuccess) return rgp_fail(h, RGP_ERR_HIP, std::string(what) + hipGetErrorString(err));
  }
  if (!back) return RGP_OK;
  const int acc = a->dtype == RGP_F64 ? RGP_F64 : RGP_F32;
  rgp_status st = seq_reduce(h, s, acc, acc, d.pA, d.nslot, DN, DN, a->gA);
  if (!st && a->gskip) st = seq_reduce(h, s, acc, acc, d.pD, d.nslot, 2 * (int64_t)a->D, a->D, a->gskip);
  if (!st && a->gbias) st = seq_reduce(h, s, acc, acc, (char*)d.pD + (int64_t)a->D * p.acc, d.nslot, 2 * (int64_t)a->D, a->D, a->gbias);
  if (!st && d.ncb > 1) {
    const int64_t n = a->rows * a->G * a->N;
    st = seq_reduce(h, s, acc, a->dtype, d.pBC, d.ncb, 2 * n, n, a->gB);
    if (!st) st = seq_reduce(h, s, acc, a->dtype, (char*)d.pBC + n * p.acc, d.ncb, 2 * n, n, a->gC);
  }
  return st;
}
extern "C" rgp_status rgp_ssm_scan_forward(rgp_handle h, void* stream, const rgp_ssm_scan* a) {
  SEQ_ENTRY(h, "ssm scan", { return scan_run(h, (hipStream_t)stream, a, false); })
}
extern "C" rgp_status rgp_ssm_scan_backward(rgp_handle h, void* stream, const rgp_ssm_scan* a) {
  SEQ_ENTRY(h, "ssm scan", { return scan_run(h, (hipStream_t)stream, a, true); })
}

// ---- one step -----------------------------------------------------------------------------------------------------------------------------
// Bound by reading and writing the state: K lanes a channel, 16 bytes of state a lane (32 in fp64), as in the kernels over time.
template <typename T, int K>
static __global__ void __launch_bounds__(256) ssm_step_kernel(rgp_ssm_scan a, int Dg) {
  typedef typename SeqAcc<T>::type A;
  constexpr int R = SSM_R;
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) / K;
  const int k = threadIdx.x % K, N = a.N;
  const bool live = e < (int64_t)a.n_seq * a.D;
  const int64_t row = live ? e / a.D : 0;
  const int ch = live ? (int)(e - row * a.D) : 0, grp = ch / Dg;
  A sig;
  const A u = (A)((const T*)a.u)[row * a.u_sb + ch];
  const A dt = seq_softplus((A)((const T*)a.delta)[row * a.delta_sb + ch] + (a.bias ? ((const A*)a.bias)[ch] : (A)0), sig);
  const A w = dt * u;
  A acc = (A)0;
  if (live) {
    A* const st = (A*)a.last + (row * a.D + ch) * N + k * R;
    const A* const Ar = (const A*)a.A + (int64_t)ch * N + k * R;
    const T* const B = (const T*)a.B + row * a.B_sb + (int64_t)grp * N + k * R;
    const T* const C = (const T*)a.C + row * a.C_sb + (int64_t)grp * N + k * R;
    A s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = k * R + r < N ? st[r] : (A)0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (k * R + r < N) {
        s[r] = seq_exp(dt * Ar[r]) * s[r] + w * (A)B[r];
        acc += s[r] * (A)C[r];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (k * R + r < N) st[r] = s[r];
  }
  acc = seq_sum<K>(acc);
  if (live && k == 0) {
    A y = acc + (a.skip ? ((const A*)a.skip)[ch] : (A)0) * u;
    if (a.z) {
      A comp;
      const A z = (A)((const T*)a.z)[row * a.z_sb + ch];
      y *= z * seq_sigmoid(z, comp);
    }
    ((T*)a.y)[row * a.D + ch] = (T)y;
  }
}
template <typename T>
static hipError_t step_pick(const rgp_ssm_scan& a, hipStream_t s) {
  const int K = a.N <= 4 ? 1 : a.N <= 8 ? 2 : a.N <= 16 ? 4 : a.N <= 32 ? 8 : 16;
  const unsigned grid = (unsigned)(((int64_t)a.n_seq * a.D * K + 255) / 256);
  const int Dg = a.D / a.G;
  switch (K) {
    case 1: hipLaunchKernelGGL((ssm_step_kernel<T, 1>), dim3(grid), dim3(256), 0, s, a, Dg); break;
    case 2: hipLaunchKernelGGL((ssm_step_kernel<T, 2>), dim3(grid), dim3(256), 0, s, a, Dg); break;
    case 4: hipLaunchKernelGGL((ssm_step_kernel<T, 4>), dim3(grid), dim3(256), 0, s, a, Dg); break;
    case 8: hipLaunchKernelGGL((ssm_step_kernel<T, 8>), dim3(grid), dim3(256), 0, s, a, Dg); break;
    default: hipLaunchKernelGGL((ssm_step_kernel<T, 16>), dim3(grid), dim3(256), 0, s, a, Dg); break;
  }
  return hipGetLastError();
}
extern "C" rgp_status rgp_ssm_scan_step(rgp_handle h, void* stream, const rgp_ssm_scan* a) {
  SEQ_ENTRY(h, "ssm scan step", {
    if (const char* bad = scan_bad(a)) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string("ssm scan step: ") + bad);
    if (a->off || a->T != 1) return rgp_fail(h, RGP_ERR_BAD_ARG, "ssm scan step: one row per sequence (T = 1, no offsets)");
    if (!a->u || !a->delta || !a->B || !a->C || !a->A || !a->y || !a->last || a->init != a->last)
      return rgp_fail(h, RGP_ERR_BAD_ARG, "ssm scan step: u, delta, A, B, C, y and the state (init = last) are required");
    if ((double)a->n_seq * a->D * 16 > 4294967295.0) return rgp_fail(h, RGP_ERR_BAD_ARG, "ssm scan step: more than 2^32 work items");
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a->dtype == RGP_F64 ? step_pick<double>(*a, s) : a->dtype == RGP_F32 ? step_pick<float>(*a, s)
                       : a->dtype == RGP_BF16 ? step_pick<__bf16>(*a, s) : step_pick<_Float16>(*a, s);
    if (e != hipSuccess) return rgp_fail(h, RGP_ERR_HIP, std::string("ssm scan step: ") + hipGetErrorString(e));
    return RGP_OK;
  })
}

// ---- short causal convolution ---------------------------------------------------------------------------------------------------------------
// v_t = silu(bias + sum_j w_j x_{t-W+1+j}) reads x once and writes v once: bound by memory.  A thread holds V channels (16 bytes) and walks a
// run of CONV_RUN steps with the last W - 1 inputs in registers; the W - 1 rows before a run are read again (from cache).
#define CONV_RUN 16
#define CONV_FLY 8
struct ConvDev {
  rgp_ssm_conv a;
  SeqGeo g;
  int64_t nrun, nvec;
  int wx, wgv, wout, lanes;        // 16-byte accesses; vectors side by side in a workgroup (backward)
  void* part;
};

// x at step t of the sequence, in walking order; before the first step the state, behind the last one zero
template <typename T, int W>
static __device__ __forceinline__ SeqVec<T> conv_x(const ConvDev& d, const SeqBlock& b, int64_t t, int64_t c, int n) {
  const rgp_ssm_conv& a = d.a;
  if (t < 0) {
    SeqVec<T> z = seq_load((const T*)a.x, 0, false);
    if (!a.init) return z;
    return seq_load((const T*)a.init + ((b.seq * (W - 1) + W - 1 + t) * a.D + c), n, false);
  }
  return seq_load(seq_row((const T*)a.x, d.g, b, SeqStride{a.x_st, a.x_sb}, t) + c, n, d.wx);
}

template <typename T, int W>
static __global__ void __launch_bounds__(256) conv_fwd_kernel(ConvDev d) {
  typedef typename SeqAcc<T>::type A;
  constexpr int V = SeqVec<T>::V;
  const rgp_ssm_conv& a = d.a;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, run = idx / d.nvec, c = (idx - run * d.nvec) * V;
  if (run >= d.nrun) return;
  const SeqBlock b = seq_find(d.g, run, CONV_RUN);
  if (!b.ok) return;
  const int n = a.D - c < V ? (int)(a.D - c) : V;
  const int64_t t0 = b.j * CONV_RUN;
  const int nt = b.len - t0 < CONV_RUN ? (int)(b.len - t0) : CONV_RUN;
  A w[W][V], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias && i < n ? ((const A*)a.bias)[c + i] : (A)0;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][i] = i < n ? ((const A*)a.w)[(c + i) * W + j] : (A)0;
  }
  A x[W][V];                                       // the window, in the arithmetic type
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const SeqVec<T> r = conv_x<T, W>(d, b, t0 - (W - 1) + j, c, n);
#pragma unroll
    for (int i = 0; i < V; ++i) x[j][i] = (A)r.e[i];
  }
  for (int tb = 0; tb < nt; tb += CONV_FLY) {
    SeqVec<T> r[CONV_FLY];                         // this many rows are in flight at once
#pragma unroll
    for (int k = 0; k < CONV_FLY; ++k) r[k] = conv_x<T, W>(d, b, t0 + (tb + k < nt ? tb + k : nt - 1), c, n);
#pragma unroll
    for (int k = 0; k < CONV_FLY; ++k) {
      if (tb + k < nt) {
        SeqVec<T> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[W - 1][i] = (A)r[k].e[i];
          A p = bias[i], comp;
#pragma unroll
          for (int j = 0; j < W; ++j) p += w[j][i] * x[j][i];
          o.e[i] = (T)(p * seq_sigmoid(p, comp));
        }
        seq_store((T*)a.v + seq_row_index(d.g, b, t0 + tb + k) * a.D + c, o, n, d.wout);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) x[j][i] = x[j + 1][i];
      }
    }
  }
}
// the W - 1 inputs before the step behind the last one
template <typename T, int W>
static __global__ void __launch_bounds__(256) conv_last_kernel(ConvDev d) {
  constexpr int V = SeqVec<T>::V;
  const rgp_ssm_conv& a = d.a;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, seq = idx / d.nvec, c = (idx - seq * d.nvec) * V;
  if (seq >= a.n_seq) return;
  SeqBlock b;
  b.seq = seq;
  b.start = seq * d.g.T;
  b.len = d.g.T;
  if (d.g.off) {
    b.start = seq_off(d.g, seq);
    const int64_t end = seq_off(d.g, seq + 1);
    b.len = end > b.start ? end - b.start : 0;
  }
  const int n = a.D - c < V ? (int)(a.D - c) : V;
  SeqVec<T> x[W - 1];                              // all read before any is written: last may be init
#pragma unroll
  for (int j = 0; j < W - 1; ++j) x[j] = conv_x<T, W>(d, b, b.len - (W - 1) + j, c, n);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) seq_store((T*)a.last + (seq * (W - 1) + j) * a.D + c, x[j], n, false);
}

// Backward: gp = gv silu'(pre), gx_t = sum_j w_j gp_{t+W-1-j}, gw_j = sum_t gp_t x_{t-W+1+j}, gbias = sum gp.  pre is formed again from x
// (one more read would cost more than W multiply-adds).  A thread walks its run and W - 1 steps behind it; the parameter sums of the
// threads with the same channels go through LDS, then from all workgroups through `part`.
template <typename T, int W>
static __global__ void __launch_bounds__(256) conv_bwd_kernel(ConvDev d) {
  typedef typename SeqAcc<T>::type A;
  constexpr int V = SeqVec<T>::V;
  __shared__ A sh[256 * V];
  const rgp_ssm_conv& a = d.a;
  const int lane = threadIdx.x % d.lanes, rl = threadIdx.x / d.lanes, nr = 256 / d.lanes;
  const int64_t nvb = (d.nvec + d.lanes - 1) / d.lanes;                  // workgroups side by side over the channels
  const int64_t rb = blockIdx.x / nvb, vb = blockIdx.x - rb * nvb, nrb = gridDim.x / nvb;
  const int64_t vec = vb * d.lanes + lane, c = vec * V;
  const int n = vec < d.nvec ? (a.D - c < V ? (int)(a.D - c) : V) : 0;
  A w[W][V], bias[V], gw[W][V], gb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias && i < n ? ((const A*)a.bias)[c + i] : (A)0;
    gb[i] = (A)0;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      w[j][i] = i < n ? ((const A*)a.w)[(c + i) * W + j] : (A)0;
      gw[j][i] = (A)0;
    }
  }
  if (n > 0)
    for (int64_t run = rb * nr + rl; run < d.nrun; run += nrb * nr) {
      const SeqBlock b = seq_find(d.g, run, CONV_RUN);
      if (!b.ok) continue;
      const int64_t t0 = b.j * CONV_RUN, t1 = t0 + CONV_RUN < b.len ? t0 + CONV_RUN : b.len;
      A x[W][V], gp[W][V];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const SeqVec<T> r = conv_x<T, W>(d, b, t0 - (W - 1) + (j < W - 1 ? j : 0), c, n);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[j][i] = (A)r.e[i];
          gp[j][i] = (A)0;
        }
      }
      const int nt = (int)(t1 - t0) + W - 1;                             // gp of step t0 + k; gx of step t0 + k - W + 1 is then complete
      for (int kb = 0; kb < nt; kb += CONV_FLY) {
        SeqVec<T> rx[CONV_FLY], rg[CONV_FLY];
#pragma unroll
        for (int k = 0; k < CONV_FLY; ++k) {
          const int64_t t = t0 + kb + k < b.len ? t0 + kb + k : b.len - 1;
          rx[k] = conv_x<T, W>(d, b, t, c, n);
          rg[k] = seq_load(seq_row((const T*)a.gv, d.g, b, SeqStride{a.gv_st, a.gv_sb}, t) + c, n, d.wgv);
        }
#pragma unroll
        for (int k = 0; k < CONV_FLY; ++k) {
          if (kb + k < nt) {
            const int64_t t = t0 + kb + k;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              x[W - 1][i] = (A)rx[k].e[i];
              A p = bias[i], comp;
#pragma unroll
              for (int j = 0; j < W; ++j) p += w[j][i] * x[j][i];
              const A sg = seq_sigmoid(p, comp);
              const A q = t < b.len ? (A)rg[k].e[i] * (sg + p * sg * comp) : (A)0;
              gp[W - 1][i] = q;
              if (t < t1) {
                gb[i] += q;
#pragma unroll
                for (int j = 0; j < W; ++j) gw[j][i] += q * x[j][i];
              }
            }
            const int64_t to = t - (W - 1);
            if (to >= t0) {
              SeqVec<T> o;
#pragma unroll
              for (int i = 0; i < V; ++i) {
                A v = (A)0;
#pragma unroll
                for (int j = 0; j < W; ++j) v += w[W - 1 - j][i] * gp[j][i];      // gp[j] is step to + j, whose tap W - 1 - j reads x_to
                o.e[i] = (T)v;
              }
              seq_store((T*)a.gx + seq_row_index(d.g, b, to) * a.D + c, o, n, d.wout);
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
              for (int i = 0; i < V; ++i) {
                x[j][i] = x[j + 1][i];
                gp[j][i] = gp[j + 1][i];
              }
          }
        }
      }
    }
  A* const part = (A*)d.part + rb * (W + 1) * a.D;                       // [W][D] taps, then [D] bias
#pragma unroll
  for (int j = 0; j <= W; ++j) {
#pragma unroll
    for (int i = 0; i < V; ++i) sh[threadIdx.x * V + i] = j < W ? gw[j < W ? j : 0][i] : gb[i];
    __syncthreads();
    for (int e = threadIdx.x; e < d.lanes * V; e += 256) {
      A v = (A)0;
      for (int q = 0; q < nr; ++q) v += sh[q * d.lanes * V + e];
      const int64_t ch = vb * d.lanes * V + e;
      if (ch < a.D) part[j * a.D + ch] = v;
    }
    __syncthreads();
  }
}
// gw [D][W] and gbias [D] from part [P][W + 1][D]
template <typename A>
static __global__ void __launch_bounds__(256) conv_sum_kernel(const A* part, int64_t P, int D, int W, A* gw, A* gbias) {
  __shared__ A sh[4][64];
  const int64_t n = (int64_t)(W + 1) * D, i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int q = threadIdx.x >> 6;
  A s0 = (A)0, s1 = (A)0;
  if (i < n) {
    int64_t p = q;
    for (; p + 4 < P; p += 8) {
      s0 += part[p * n + i];
      s1 += part[(p + 4) * n + i];
    }
    for (; p < P; p += 4) s0 += part[p * n + i];
  }
  sh[q][threadIdx.x & 63] = s0 + s1;
  __syncthreads();
  if (q == 0 && i < n) {
    const A v = (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
    const int64_t j = i / D, ch = i - j * D;
    if (j < W) gw[ch * W + j] = v;
    else if (gbias) gbias[ch] = v;
  }
}

template <typename T, int W>
static __global__ void __launch_bounds__(256) conv_step_kernel(ConvDev d) {
  typedef typename SeqAcc<T>::type A;
  constexpr int V = SeqVec<T>::V;
  const rgp_ssm_conv& a = d.a;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, seq = idx / d.nvec, c = (idx - seq * d.nvec) * V;
  if (seq >= a.n_seq) return;
  const int n = a.D - c < V ? (int)(a.D - c) : V;
  T* const st = (T*)a.last + seq * (W - 1) * a.D + c;
  SeqVec<T> x[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) x[j] = seq_load((const T*)st + (int64_t)j * a.D, n, d.wout);
  x[W - 1] = seq_load((const T*)a.x + seq * a.x_sb + c, n, d.wx);
  SeqVec<T> o;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    A p = a.bias && i < n ? ((const A*)a.bias)[c + i] : (A)0, comp;
#pragma unroll
    for (int j = 0; j < W; ++j) p += (i < n ? ((const A*)a.w)[(c + i) * W + j] : (A)0) * (A)x[j].e[i];
    o.e[i] = (T)(p * seq_sigmoid(p, comp));
  }
  seq_store((T*)a.v + seq * a.D + c, o, n, d.wgv);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) seq_store(st + (int64_t)j * a.D, x[j + 1], n, d.wout);
}

static const char* conv_bad(const rgp_ssm_conv* a) {
  if (!a) return "null arguments";
  if (a->dtype < 0 || a->dtype > 3) return "dtype must be RGP_F64, RGP_F32, RGP_BF16 or RGP_F16";
  if (a->n_seq < 1 || a->D < 1 || a->rows < 0 || a->T < 0) return "empty problem";
  if (a->W < 2 || a->W > 8) return "2 to 8 taps";
  if (!a->off && (a->T < 1 || a->T * a->n_seq != a->rows)) return "rows must be T * n_seq, T >= 1";
  return nullptr;
}
static void conv_plan(const rgp_ssm_conv* a, ConvDev& d, int64_t& grid, int64_t& nrb) {
  d = ConvDev{};
  d.a = *a;
  d.g = SeqGeo{a->off, a->T, a->rows, a->n_seq, a->reverse};
  const int V = 16 / seq_dtype_bytes(a->dtype);
  d.nvec = (a->D + V - 1) / V;
  d.nrun = seq_blocks(d.g, CONV_RUN);
  d.lanes = 1;
  while (d.lanes < 64 && d.lanes < d.nvec) d.lanes *= 2;
  const int64_t nvb = (d.nvec + d.lanes - 1) / d.lanes, nr = 256 / d.lanes;
  nrb = (d.nrun + nr - 1) / nr;
  const int64_t most = nvb > 2048 ? 1 : 2048 / nvb;                      // eight workgroups a CU; more only lengthens the sum over them
  if (nrb > most) nrb = most;
  if (nrb < 1) nrb = 1;
  grid = nrb * nvb;
}
extern "C" int64_t rgp_ssm_conv_workspace(const rgp_ssm_conv* a, int backward) {
  if (conv_bad(a)) return -1;
  if (!backward) return 0;
  ConvDev d;
  int64_t grid, nrb;
  conv_plan(a, d, grid, nrb);
  return nrb * (a->W + 1) * a->D * (a->dtype == RGP_F64 ? 8 : 4);
}

enum { CONV_FWD, CONV_LAST, CONV_BWD, CONV_STEP };
template <typename T, int W>
static hipError_t conv_go(const ConvDev& d, int what, int64_t grid, hipStream_t s) {
  if (grid < 1) return hipSuccess;
  if (what == CONV_FWD) hipLaunchKernelGGL((conv_fwd_kernel<T, W>), dim3((unsigned)grid), dim3(256), 0, s, d);
  else if (what == CONV_LAST) hipLaunchKernelGGL((conv_last_kernel<T, W>), dim3((unsigned)grid), dim3(256), 0, s, d);
  else if (what == CONV_BWD) hipLaunchKernelGGL((conv_bwd_kernel<T, W>), dim3((unsigned)grid), dim3(256), 0, s, d);
  else hipLaunchKernelGGL((conv_step_kernel<T, W>), dim3((unsigned)grid), dim3(256), 0, s, d);
  return hipGetLastError();
}
template <typename T>
static hipError_t conv_taps(const ConvDev& d, int what, int64_t grid, hipStream_t s) {
  switch (d.a.W) {
    case 2: return conv_go<T, 2>(d, what, grid, s);
    case 3: return conv_go<T, 3>(d, what, grid, s);
    case 4: return conv_go<T, 4>(d, what, grid, s);
    case 5: return conv_go<T, 5>(d, what, grid, s);
    case 6: return conv_go<T, 6>(d, what, grid, s);
    case 7: return conv_go<T, 7>(d, what, grid, s);
    default: return conv_go<T, 8>(d, what, grid, s);
  }
}
static hipError_t conv_launch(const ConvDev& d, int what, int64_t grid, hipStream_t s) {
  switch (d.a.dtype) {
    case RGP_F64: return conv_taps<double>(d, what, grid, s);
    case RGP_F32: return conv_taps<float>(d, what, grid, s);
    case RGP_BF16: return conv_taps<__bf16>(d, what, grid, s);
    default: return conv_taps<_Float16>(d, what, grid, s);
  }
}
static rgp_status conv_run(rgp_handle h, hipStream_t s, const rgp_ssm_conv* a, int what) {
  const std::string name = what == CONV_BWD ? "ssm conv backward: " : what == CONV_STEP ? "ssm conv step: " : "ssm conv forward: ";
  if (const char* bad = conv_bad(a)) return rgp_fail(h, RGP_ERR_BAD_ARG, name + bad);
  const bool some = a->rows > 0;
  if (!a->w || (some && !a->x)) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "x and w are required");
  ConvDev d;
  int64_t grid, nrb;
  conv_plan(a, d, grid, nrb);
  const int e = seq_dtype_bytes(a->dtype), V = 16 / e;
  if ((double)d.nrun * d.nvec > 4294967295.0 || (double)a->n_seq * d.nvec > 4294967295.0 || (double)grid * 256 > 4294967295.0)
    return rgp_fail(h, RGP_ERR_BAD_ARG, name + "more than 2^32 work items");
  d.wx = seq_aligned(a->x, a->x_st, a->x_sb, e);
  const int64_t seqs = ((int64_t)a->n_seq * d.nvec + 255) / 256;
  hipError_t err = hipSuccess;
  if (what == CONV_BWD) {
    if (!a->gw || (some && (!a->gv || !a->gx))) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "gv, gx and gw are required");
    if (rgp_ssm_conv_workspace(a, 1) > a->work_bytes || !a->work || ((uintptr_t)a->work & 15))
      return rgp_fail(h, RGP_ERR_WORKSPACE, name + "work buffer too small or not 16-byte aligned");
    d.wgv = seq_aligned(a->gv, a->gv_st, a->gv_sb, e);
    d.wout = a->D % V == 0 && seq_aligned(a->gx, 0, 0, e);
    d.part = a->work;
    err = conv_launch(d, CONV_BWD, grid, s);
    if (err == hipSuccess) {
      const unsigned sg = (unsigned)(((int64_t)(a->W + 1) * a->D + 63) / 64);
      if (a->dtype == RGP_F64) hipLaunchKernelGGL(conv_sum_kernel<double>, dim3(sg), dim3(256), 0, s, (const double*)d.part, nrb, a->D, a->W, (double*)a->gw, (double*)a->gbias);
      else hipLaunchKernelGGL(conv_sum_kernel<float>, dim3(sg), dim3(256), 0, s, (const float*)d.part, nrb, a->D, a->W, (float*)a->gw, (float*)a->gbias);
      err = hipGetLastError();
    }
  } else if (what == CONV_STEP) {
    if (a->off || a->T != 1) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "one row per sequence (T = 1, no offsets)");
    if (!a->v || !a->last || a->init != a->last) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "v and the state (init = last) are required");
    d.wx = seq_aligned(a->x, 0, a->x_sb, e);
    d.wout = a->D % V == 0 && seq_aligned(a->last, 0, 0, e);
    d.wgv = a->D % V == 0 && seq_aligned(a->v, 0, 0, e);
    err = conv_launch(d, CONV_STEP, seqs, s);
  } else {
    if (some && !a->v) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "v is required");
    if (a->last && a->last == a->init) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "last must not be init");
    d.wout = a->D % V == 0 && seq_aligned(a->v, 0, 0, e);
    err = conv_launch(d, CONV_FWD, (d.nrun * d.nvec + 255) / 256, s);
    if (err == hipSuccess && a->last) err = conv_launch(d, CONV_LAST, seqs, s);
  }
  return err == hipSuccess ? RGP_OK : rgp_fail(h, RGP_ERR_HIP, name + hipGetErrorString(err));
}
extern "C" rgp_status rgp_ssm_conv_forward(rgp_handle h, void* stream, const rgp_ssm_conv* a) {
  SEQ_ENTRY(h, "ssm conv", { return conv_run(h, (hipStream_t)stream, a, CONV_FWD); })
}
extern "C" rgp_status rgp_ssm_conv_backward(rgp_handle h, void* stream, const rgp_ssm_conv* a) {
  SEQ_ENTRY(h, "ssm conv", { return conv_run(h, (hipStream_t)stream, a, CONV_BWD); })
}
extern "C" rgp_status rgp_ssm_conv_step(rgp_handle h, void* stream, const rgp_ssm_conv* a) {
  SEQ_ENTRY(h, "ssm conv", { return conv_run(h, (hipStream_t)stream, a, CONV_STEP); })
}
