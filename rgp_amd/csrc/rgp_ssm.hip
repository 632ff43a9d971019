// rgp_ssm.hip -- host side of the selective state-space scan (argument checks, split over time, work buffer), the kernels that join the
// blocks of the split, the sums over partial results, the scan's form for one step, and the short causal convolution.
#include "rgp_ssm.h"

#include <type_traits>

// ---- sums of partial results in a fixed order -----------------------------------------------------------------------------------------
// A workgroup forms W outputs of one of up to five sums, Q = 1024 / W threads for each: thread q adds partials q, q + Q, ... in eight
// interleaved sums (that many loads are in flight), then the Q are added in LDS.  W = 64, 16 where there are many partials (2048 of 1024 outputs:
// 9 us with 64), and up to SEQ_FEW partials are added by one thread an output.  The order depends on the count of partials alone.  5 to 8 us for
// all sums of a backward pass.  Beyond SEQ_HUGE partials (many short sequences) rows r, r + SEQ_MANY, ... are first added into row r.
#define SEQ_FEW 32
#define SEQ_MANY 512
#define SEQ_HUGE 8192
#define SEQ_SUMS_GRID 65536          // workgroups of a launch, which go on to further outputs (a launch holds fewer than 2^32 threads)
static __host__ __device__ inline int64_t seq_sums_width(int64_t P) { return P <= SEQ_FEW ? 1024 : P <= SEQ_MANY ? 64 : 16; }
template <typename A>
static __device__ __forceinline__ void seq_sums_store(const SeqSum& j, int64_t i, A v) {
  const int64_t o = j.turn > 1 ? (i % (j.n / j.turn)) * j.turn + i / (j.n / j.turn) : i;
  switch (j.dt) {
    case RGP_F64: ((double*)j.out)[o] = (double)v; break;
    case RGP_F32: ((float*)j.out)[o] = (float)v; break;
    case RGP_BF16: ((__bf16*)j.out)[o] = (__bf16)(float)v; break;
    default: ((_Float16*)j.out)[o] = (_Float16)(float)v; break;
  }
}
template <typename A>
static __global__ void __launch_bounds__(1024) seq_sums_kernel(SeqSums g) {
  __shared__ A sh[1024];
  for (int64_t at = blockIdx.x; at < g.blocks; at += gridDim.x) {
    int k = 0;
    while (k + 1 < g.count && at >= g.job[k + 1].block0) ++k;
    const SeqSum& j = g.job[k];
    const A* const part = (const A*)j.part;
    const int64_t o0 = (at - j.block0) * seq_sums_width(j.P);
    int64_t n = j.n;
    if (j.end && j.end[0] * j.per < n) n = j.end[0] < 0 ? 0 : j.end[0] * j.per;
    if (j.P <= SEQ_FEW) {                                  // uniform over the workgroup
      const int64_t i = o0 + threadIdx.x;
      if (i < n) {
        A v = (A)0;
#pragma unroll 8
        for (int64_t p = 0; p < j.P; ++p) v += part[p * j.stride + i];
        seq_sums_store(j, i, v);
      }
      continue;
    }
    const int W = (int)seq_sums_width(j.P), Q = 1024 / W, G = W == 64 ? 4 : 8, l = threadIdx.x % W, q = threadIdx.x / W;       // Q = G G
    const int64_t i = o0 + l;
    A v8[8] = {};
    if (i < n) {
      const A* p = part + q * j.stride + i;
      int64_t left = j.P > q ? (j.P - q + Q - 1) / Q : 0;
      const int64_t step = Q * j.stride;
      for (; left >= 8; left -= 8, p += 8 * step) {
#pragma unroll
        for (int u = 0; u < 8; ++u) v8[u] += p[u * step];
      }
#pragma unroll
      for (int u = 0; u < 7; ++u)
        if (u < left) v8[u] += p[u * step];
    }
    __syncthreads();                                       // the outputs before these are out of sh
    sh[threadIdx.x] = ((v8[0] + v8[1]) + (v8[2] + v8[3])) + ((v8[4] + v8[5]) + (v8[6] + v8[7]));
    __syncthreads();
    A v = (A)0;
    if (q < G) {                                            // G groups of G threads' sums
      v = sh[q * G * W + l];
      for (int r = 1; r < G; ++r) v += sh[(q * G + r) * W + l];
    }
    __syncthreads();
    if (q < G) sh[q * W + l] = v;
    __syncthreads();
    if (q == 0 && i < n) {
      for (int r = 1; r < G; ++r) v += sh[r * W + l];
      seq_sums_store(j, i, v);
    }
  }
}
template <typename A>
static __global__ void __launch_bounds__(256) seq_gather_kernel(A* part, int64_t P, int64_t stride, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  A v8[8] = {};
  int64_t r = blockIdx.y;                                 // this thread alone reads and writes column i of these rows
  for (; r + 7 * SEQ_MANY < P; r += 8 * SEQ_MANY) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v8[u] += part[(r + u * SEQ_MANY) * stride + i];
  }
  for (; r < P; r += SEQ_MANY) v8[0] += part[r * stride + i];
  part[blockIdx.y * stride + i] = ((v8[0] + v8[1]) + (v8[2] + v8[3])) + ((v8[4] + v8[5]) + (v8[6] + v8[7]));
}
void SeqSums::add(void* part, int64_t P, int64_t stride, int64_t n, void* out, int dt, int turn, const int64_t* end, int64_t per) {
  if (!out || n < 1) return;
  SeqSum& j = job[count++];
  j.part = part; j.P = P; j.stride = stride; j.n = n; j.out = out; j.dt = dt; j.turn = turn; j.end = end; j.per = per;
}
rgp_status SeqSums::run(rgp_handle h, hipStream_t s, int acc) {
  if (!count) return RGP_OK;
  for (int k = 0; k < count; ++k) {
    SeqSum& j = job[k];
    if (j.P <= SEQ_HUGE) continue;
    const dim3 g((unsigned)((j.n + 255) / 256), SEQ_MANY);
    if (acc == RGP_F64) hipLaunchKernelGGL(seq_gather_kernel<double>, g, dim3(256), 0, s, (double*)j.part, j.P, j.stride, j.n);
    else hipLaunchKernelGGL(seq_gather_kernel<float>, g, dim3(256), 0, s, (float*)j.part, j.P, j.stride, j.n);
    const rgp_status st = seq_launched(h, "sum of partial results");
    if (st) return st;
    j.P = SEQ_MANY;
  }
  blocks = 0;
  for (int k = 0; k < count; ++k) {
    job[k].block0 = blocks;
    blocks += (job[k].n + seq_sums_width(job[k].P) - 1) / seq_sums_width(job[k].P);
  }
  const dim3 grid((unsigned)(blocks < SEQ_SUMS_GRID ? blocks : SEQ_SUMS_GRID));
  if (acc == RGP_F64) hipLaunchKernelGGL(seq_sums_kernel<double>, grid, dim3(1024), 0, s, *this);
  else hipLaunchKernelGGL(seq_sums_kernel<float>, grid, dim3(1024), 0, s, *this);
  return seq_launched(h, "sum of partial results");
}

// ---- joining the blocks of the time split -----------------------------------------------------------------------------------------------
// part[block] holds what a block adds to the state that enters it, and is left holding that entering state.  A whole block multiplies the
// state by exp(A sum dt): the decays of a diagonal recurrence commute.  back: the same for the adjoint, from the last block to the first.
// 64 lanes take neighbouring (channel, state) pairs of one sequence, Q threads a pair: each walks its part of the blocks twice, first for
// what that stretch does as a whole, then with the state that enters it (Q = 1: once).  The walk waits for memory, JOIN_U blocks at a time;
// with Q = 16 for 1024 blocks of 8 sequences x 64 channels it takes 14 us where one thread a pair took 479; for many short sequences Q = 1 takes
// 14 us where Q = 16 took 98, and for 13 sequences x 1024 channels x 32 states 6.4 where Q = 4 took 16.
#define JOIN_U 8
template <typename A, int Q>
static __global__ void __launch_bounds__(Q == 1 ? 256 : Q * 64) ssm_join_kernel(SsmDev d, int back) {
  __shared__ A shP[Q][64], shH[Q][64];
  const rgp_ssm_scan& a = d.a;
  const int l = threadIdx.x & 63, q = Q == 1 ? 0 : threadIdx.x >> 6, wide = Q == 1 ? 256 : 64;
  const int64_t DN = (int64_t)a.D * a.N, per = (DN + wide - 1) / wide, seq = blockIdx.x / per;
  const int64_t dn = (blockIdx.x - seq * per) * wide + (Q == 1 ? threadIdx.x : l);
  const bool ok = dn < DN;
  int64_t start = seq * d.g.T, len = d.g.T;
  if (d.g.off) {
    start = seq_off(d.g, seq);
    const int64_t end = seq_off(d.g, seq + 1);
    len = end > start ? end - start : 0;
  }
  const int64_t nb = (len + d.L - 1) >> d.lg, slot0 = seq_slot(d.g, seq, start, d.lg, 0), step = d.g.off ? 1 : d.g.n_seq;
  const int64_t each = (nb + Q - 1) / Q, j0 = q * each < nb ? q * each : nb, j1 = !ok ? j0 : (j0 + each < nb ? j0 + each : nb);
  const int64_t at0 = ok ? dn : 0, ch = at0 / a.N;
  const A Av = ssm_finite(((const A*)a.A)[at0]);
  A* const part = (A*)d.part + slot0 * DN + at0;
  const A* const sum = (const A*)d.sumdt + slot0 * a.D + ch;
  A P = (A)1, H = (A)0, s = (A)0;
  if (Q == 1) s = !back && a.init && ok ? ((const A*)a.init)[seq * DN + dn] : (A)0;
  const int64_t dp = (back ? -step : step) * DN, ds = (back ? -step : step) * a.D;
  // up to n of the `left` blocks from pp / ps on: their sums are read together, then walked.  (The block that nothing follows has left no
  // sums: what is read there goes unused.)
  auto walk = [&](A* pp, const A* ps, int left, auto n, int pass) {
    A p[n()], e[n()];
#pragma unroll
    for (int i = 0; i < n(); ++i) {
      const int k = i < left ? i : 0;
      p[i] = pp[k * dp];
      e[i] = seq_exp(Av * ps[k * ds]);
    }
#pragma unroll
    for (int i = 0; i < n(); ++i) {
      if (i < left) {
        if (pass == 0) {
          P *= e[i];
          H = ssm_through(e[i], H) + p[i];
        } else {
          pp[i * dp] = s;
          s = ssm_through(e[i], s) + p[i];
        }
      }
    }
  };
  for (int pass = Q == 1 ? 1 : 0; pass < 2; ++pass) {
    A* pp = part + (back ? nb - 1 - j0 : j0) * step * DN;
    const A* ps = sum + (back ? nb - 1 - j0 : j0) * step * a.D;
    int left = (int)(j1 - j0);
    for (; left >= JOIN_U; left -= JOIN_U, pp += JOIN_U * dp, ps += JOIN_U * ds) walk(pp, ps, JOIN_U, std::integral_constant<int, JOIN_U>(), pass);
    if (left > 3) walk(pp, ps, left, std::integral_constant<int, JOIN_U>(), pass);
    else if (left > 1) walk(pp, ps, left, std::integral_constant<int, 3>(), pass);
    else if (left > 0) walk(pp, ps, left, std::integral_constant<int, 1>(), pass);
    if (pass == 0) {
      shP[q][l] = P;
      shH[q][l] = H;
      __syncthreads();                                    // also: every block's sums are read before the states replace them
      s = !back && a.init && ok ? ((const A*)a.init)[seq * DN + dn] : (A)0;
      for (int r = 0; r < q; ++r) s = ssm_through(shP[r][l], s) + shH[r][l];
    }
  }
}

template <typename A>
static void join_launch(const SsmDev& d, int Q, unsigned grid, int back, hipStream_t s) {
  if (Q == 1) hipLaunchKernelGGL((ssm_join_kernel<A, 1>), dim3(grid), dim3(256), 0, s, d, back);
  else if (Q == 4) hipLaunchKernelGGL((ssm_join_kernel<A, 4>), dim3(grid), dim3(256), 0, s, d, back);
  else hipLaunchKernelGGL((ssm_join_kernel<A, 16>), dim3(grid), dim3(1024), 0, s, d, back);
}

// ---- host side of the scan --------------------------------------------------------------------------------------------------------------
static const char* scan_bad(const rgp_ssm_scan* a) {
  if (!a) return "null arguments";
  if (a->dtype < 0 || a->dtype > 3) return "dtype must be RGP_F64, RGP_F32, RGP_BF16 or RGP_F16";
  if (a->n_seq < 1 || a->D < 1 || a->N < 1 || a->G < 1 || a->rows < 0 || a->T < 0) return "empty problem";
  if (a->N > 64) return "at most 64 states per channel";
  if (a->rows > SEQ_MOST || a->T > SEQ_MOST) return "more than 2^40 rows";
  if (a->D % a->G) return "D must be a multiple of G";
  if (!a->off && (a->T < 1 || a->T * a->n_seq != a->rows)) return "rows must be T * n_seq, T >= 1";
  return nullptr;
}

// Up to so many blocks a sequence each block's workgroup joins for itself, which saves a launch: training steps of 32 x 300 x 64 fp32 take 81 us
// of kernels with the launch and 75 without, of 16 x 100 x 64 fp64 73 and 67; with 16 blocks (8 x 1000 x 300 fp32) 177 and 180, with 32 (4 x 256 x
// 40 fp32) 54 and 64.
#define JOIN_SELF 12
struct ScanPlan {
  SsmDev d;
  SsmShape sh;
  int acc, Q;                      // Q: threads that walk the blocks of one state in the join
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
  // States a lane: 4; 2 in fp64, where an exponential takes dozens of instructions: more lanes a channel shorten a step where the waves are few
  // (training steps of 8 x 64 x 1000: 131 -> 105 us, 8 x 40 x 300: 83 -> 71) and the backward kernel gets two waves a SIMD (8191 x 512: N = 8 555 ->
  // 463 us, N = 16 714 -> 708, N = 32 627 -> 653).
  const bool f64 = a->dtype == RGP_F64;
  SsmShape& h = p.sh;
  h.R = f64 && a->N <= 32 ? 2 : 4;
  h.K = f64 ? 2 : 1;
  while (h.K * h.R < a->N) h.K *= 2;
  h.CH = h.K <= 4 ? 64 : 256 / h.K;
  const int few = 64 / h.K;                                         // channels of a single wave, where that leaves fewer lanes idle
  if ((h.K == 4 || (f64 && h.K == 8)) && (d.Dg + few - 1) / few * few < (d.Dg + h.CH - 1) / h.CH * h.CH) h.CH = few;
  d.ncb = (d.Dg + h.CH - 1) / h.CH;
  const int64_t longest = a->off ? (a->max_len > 0 && a->max_len < a->rows ? a->max_len : a->rows) : a->T;
  // Split over time.  In units of the time in which a SIMD with several waves walks one wave's step (about 80 ns forward, 260 ns backward, four
  // times that in fp64): unsplit, the whole work spread over 1024 SIMDs, but no less than the longest sequence at twice that time (a lone wave
  // waits for its own results); split, the work, a walk over one block, the first walk (0.65 of the forward one, 0.3 of the backward one), and
  // the join.  Measured backward: 8 x 1024 x 1024 bf16, N = 32, 445 us unsplit; N = 16 in 16 blocks, 186 split.  Forward, 4 x 64 x 64 fp64: 37 us
  // unsplit, 24 split.
  // Blocks of 64 steps, longer ones where the waves get many (they leave the join and the sums of the backward pass less to read), shorter ones
  // where that leaves SIMDs idle: training steps of 8 x 512 x 40 fp64 take 122 us of kernels with 32 steps a block, 96 with 16, 107 with 8; of 4 x
  // 256 x 40 fp64 111, 81 and 72; of 8 x 4096 x 32 fp32 111 with 64 and 105 with 32 (backward alone; forward loses with them).
  const double waves = (double)a->G * d.ncb * (h.CH * h.K / 64.0), work = waves * a->rows / 1024.0, most = back ? 12288.0 : 24576.0;
  auto count = [&](int g) { return waves * ((double)(a->rows >> g) + a->n_seq); };
  int lg = 6;
  if (count(6) < (back || f64 ? 2048.0 : 1024.0)) lg = count(5) < (f64 ? 2048.0 : 1024.0) ? 4 : 5;
  if (lg == 4 && count(4) < 512.0) lg = 3;
  while (lg < 20 && count(lg) > most) ++lg;
  const double one = work > 2.0 * longest ? work : 2.0 * longest, block = 2.0 * ((int64_t)1 << lg);
  const double two = back ? 1.3 * (work + block) + (f64 ? 25.0 : 80.0) : 1.65 * (work + block) + (f64 ? 40.0 : 130.0);
  if (!(two < one)) lg = 0;
  p.split = lg > 0;
  if (!p.split)
    for (lg = 6; ((int64_t)1 << lg) < (a->off ? a->rows : a->T); ++lg) {}
  d.lg = lg;
  d.L = (int64_t)1 << lg;
  const int64_t deep = (longest + d.L - 1) >> d.lg;
  p.Q = deep <= 8 || (double)a->n_seq * a->D * a->N >= 131072.0 ? 1 : deep <= 128 ? 4 : 16;      // one where the pairs alone give two waves a SIMD
  d.nslot = seq_blocks(d.g, d.lg);
  d.join = p.split && deep <= JOIN_SELF;
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
  return seq_blocks(g, SSM_CK_LG) * a->D * a->N * (a->dtype == RGP_F64 ? 8 : 4);
}

static rgp_status scan_run(rgp_handle h, hipStream_t s, const rgp_ssm_scan* a, bool back) {
  const char* const what = back ? "ssm scan backward: " : "ssm scan forward: ";
  if (const char* bad = scan_bad(a)) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + bad);
  const bool some = a->rows > 0;                       // without rows the activations may have no memory
  if (!a->A || (some && (!a->u || !a->delta || !a->B || !a->C))) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "u, delta, A, B and C are required");
  if (!back && some && !a->y) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "y is required");
  // every block of time may read init while the last one writes last
  if (!back && seq_overlap(a->last, a->init, (int64_t)a->n_seq * a->D * a->N * (a->dtype == RGP_F64 ? 8 : 4)))
    return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "last must not share memory with init");
  if (back && (!a->gA || (some && (!a->gy || !a->states || !a->gu || !a->gdelta || !a->gB || !a->gC || (a->z && !a->gz)))))
    return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "gy, states and the gradients' buffers are required");
  ScanPlan p;
  scan_plan(a, back, p);
  SsmDev& d = p.d;
  if (p.bytes > a->work_bytes || (p.bytes && !a->work) || ((uintptr_t)a->work & 15))
    return rgp_fail(h, RGP_ERR_WORKSPACE, std::string(what) + "work buffer too small or not 16-byte aligned");
  // Vectors need as many channels as they have elements in every workgroup; where the last one has fewer, all take the kernels of single elements
  // (training steps of 512 x 16 x 1025 bf16 take 382 us, x 1032 332, x 1024 237; of 4096 x 32 x 65 fp32 525, x 68 505, x 64 279).
  const int V = 16 / seq_dtype_bytes(a->dtype), rest = d.Dg % p.sh.CH;
  d.wide = rest == 0 || rest >= V;
  char* w = (char*)a->work;
  auto take = [&](int64_t bytes) { void* r = bytes ? (void*)w : nullptr; w += bytes; return r; };
  d.part = take(p.part_bytes);
  d.sumdt = take(p.sum_bytes);
  d.pA = take(p.pA_bytes);
  d.pD = take(p.pD_bytes);
  d.pBC = take(p.pBC_bytes);
  const int64_t DN = (int64_t)a->D * a->N;
  const int64_t join = p.split && !d.join ? (int64_t)a->n_seq * (p.Q == 1 ? (DN + 255) / 256 : (DN + 63) / 64) : 0;      // workgroups, where it is a launch
  const double join_threads = (double)join * (p.Q == 1 ? 256 : p.Q * 64);
  if ((double)d.nslot * p.sh.CH * p.sh.K > 4294967295.0 || (int64_t)a->G * d.ncb > 65535 || seq_blocks(d.g, SSM_CK_LG) > 4294967295 || join_threads > 4294967295.0)
    return rgp_fail(h, RGP_ERR_BAD_ARG, std::string(what) + "more than 2^32 work items");
  hipError_t err = hipSuccess;
  if (d.nslot > 0) {
    if (p.split) {
      err = back ? ssm_bwd_launch(d, p.sh, 1, s) : ssm_fwd_launch(d, p.sh, 1, s);
      if (err == hipSuccess && !d.join) {
        if (p.acc == 8) join_launch<double>(d, p.Q, (unsigned)join, back ? 1 : 0, s);
        else join_launch<float>(d, p.Q, (unsigned)join, back ? 1 : 0, s);
        err = hipGetLastError();
      }
    }
    if (err == hipSuccess) err = back ? ssm_bwd_launch(d, p.sh, 0, s) : ssm_fwd_launch(d, p.sh, 0, s);
    if (err != hipSuccess) return rgp_fail(h, RGP_ERR_HIP, std::string(what) + hipGetErrorString(err));
  }
  if (!back) return RGP_OK;
  const int acc = a->dtype == RGP_F64 ? RGP_F64 : RGP_F32;
  SeqSums sums;
  sums.add(d.pA, d.nslot, DN, DN, a->gA, acc);
  sums.add(d.pD, d.nslot, 2 * (int64_t)a->D, a->D, a->gskip, acc);
  sums.add((char*)d.pD + (int64_t)a->D * p.acc, d.nslot, 2 * (int64_t)a->D, a->D, a->gbias, acc);
  if (d.ncb > 1) {
    const int64_t per = (int64_t)a->G * a->N, n = a->rows * per, *end = a->off ? a->off + a->n_seq : nullptr;
    sums.add(d.pBC, d.ncb, 2 * n, n, a->gB, a->dtype, 1, end, per);
    sums.add((char*)d.pBC + n * p.acc, d.ncb, 2 * n, n, a->gC, a->dtype, 1, end, per);
  }
  return sums.run(h, s, acc);
}
extern "C" rgp_status rgp_ssm_scan_forward(rgp_handle h, void* stream, const rgp_ssm_scan* a) {
  SEQ_ENTRY(h, "ssm scan", { return scan_run(h, (hipStream_t)stream, a, false); })
}
extern "C" rgp_status rgp_ssm_scan_backward(rgp_handle h, void* stream, const rgp_ssm_scan* a) {
  SEQ_ENTRY(h, "ssm scan", { return scan_run(h, (hipStream_t)stream, a, true); })
}

// ---- one step -----------------------------------------------------------------------------------------------------------------------------
// Bound by reading and writing the state: K lanes a channel, 16 bytes of state a lane (32 in fp64), as in the kernels over time.  256 x 2048
// bf16, N = 16: 17.8 us for 67 MB of state and 8 MB beside it, 4.2 TB/s; one sequence of 40 channels 3.8 us, the launch.
#define STEP_R 4                     // states a lane
template <typename T, int K>
static __global__ void __launch_bounds__(256) ssm_step_kernel(rgp_ssm_scan a, int Dg, int whole) {
  typedef typename SeqAcc<T>::type A;
  constexpr int R = STEP_R;
  const uint32_t e = (blockIdx.x * 256u + threadIdx.x) / K;              // host-checked: below 2^32
  const int k = threadIdx.x % K, N = a.N;
  const bool live = e < (uint32_t)a.n_seq * (uint32_t)a.D;
  const int64_t row = live ? e / (uint32_t)a.D : 0;
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
    struct alignas(16) Quad { A v[R]; };
    Quad s, Aq, Bq, Cq;
    if (whole) {
      s = *(const Quad*)st;
      Aq = *(const Quad*)Ar;
      const SeqVec<T, R> b = *(const SeqVec<T, R>*)B, c = *(const SeqVec<T, R>*)C;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        Bq.v[r] = (A)b.e[r];
        Cq.v[r] = (A)c.e[r];
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool in = k * R + r < N;
        s.v[r] = in ? st[r] : (A)0;
        Aq.v[r] = in ? Ar[r] : (A)0;
        Bq.v[r] = in ? (A)B[r] : (A)0;
        Cq.v[r] = in ? (A)C[r] : (A)0;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s.v[r] = seq_exp(dt * ssm_finite(Aq.v[r])) * s.v[r] + w * Bq.v[r];
      acc += s.v[r] * Cq.v[r];
    }
    if (whole) *(Quad*)st = s;
    else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (k * R + r < N) st[r] = s.v[r];
    }
  }
  acc = seq_sum<K>(acc);
  if (live && k == 0) {
    A y = acc + (a.skip ? ((const A*)a.skip)[ch] : (A)0) * u;
    if (a.z) {
      const A z = (A)((const T*)a.z)[row * a.z_sb + ch];
      y *= z * seq_sigmoid(z);
    }
    ((T*)a.y)[row * a.D + ch] = (T)y;
  }
}
static int step_lanes(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }       // lanes a channel
template <typename T>
static hipError_t step_pick(const rgp_ssm_scan& a, hipStream_t s) {
  const int K = step_lanes(a.N);
  const unsigned grid = (unsigned)(((int64_t)a.n_seq * a.D * K + 255) / 256);
  const int Dg = a.D / a.G;
  const int whole = a.N == STEP_R * K && ((uintptr_t)a.last & 15) == 0 && ((uintptr_t)a.A & 15) == 0 &&
                    seq_aligned(a.B, a.B_sb, (int)sizeof(T), STEP_R) && seq_aligned(a.C, a.C_sb, (int)sizeof(T), STEP_R);
  switch (K) {
    case 1: hipLaunchKernelGGL((ssm_step_kernel<T, 1>), dim3(grid), dim3(256), 0, s, a, Dg, whole); break;
    case 2: hipLaunchKernelGGL((ssm_step_kernel<T, 2>), dim3(grid), dim3(256), 0, s, a, Dg, whole); break;
    case 4: hipLaunchKernelGGL((ssm_step_kernel<T, 4>), dim3(grid), dim3(256), 0, s, a, Dg, whole); break;
    case 8: hipLaunchKernelGGL((ssm_step_kernel<T, 8>), dim3(grid), dim3(256), 0, s, a, Dg, whole); break;
    default: hipLaunchKernelGGL((ssm_step_kernel<T, 16>), dim3(grid), dim3(256), 0, s, a, Dg, whole); break;
  }
  return hipGetLastError();
}
extern "C" rgp_status rgp_ssm_scan_step(rgp_handle h, void* stream, const rgp_ssm_scan* a) {
  SEQ_ENTRY(h, "ssm scan step", {
    if (const char* bad = scan_bad(a)) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string("ssm scan step: ") + bad);
    if (a->off || a->T != 1) return rgp_fail(h, RGP_ERR_BAD_ARG, "ssm scan step: one row per sequence (T = 1, no offsets)");
    if (!a->u || !a->delta || !a->B || !a->C || !a->A || !a->y || !a->last || a->init != a->last)
      return rgp_fail(h, RGP_ERR_BAD_ARG, "ssm scan step: u, delta, A, B, C, y and the state (init = last) are required");
    if ((double)a->n_seq * a->D * step_lanes(a->N) > 4294967295.0 - 255.0) return rgp_fail(h, RGP_ERR_BAD_ARG, "ssm scan step: more than 2^32 work items");
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a->dtype == RGP_F64 ? step_pick<double>(*a, s) : a->dtype == RGP_F32 ? step_pick<float>(*a, s)
                       : a->dtype == RGP_BF16 ? step_pick<__bf16>(*a, s) : step_pick<_Float16>(*a, s);
    if (e != hipSuccess) return rgp_fail(h, RGP_ERR_HIP, std::string("ssm scan step: ") + hipGetErrorString(e));
    return RGP_OK;
  })
}

// ---- short causal convolution ---------------------------------------------------------------------------------------------------------------
// v_t = silu(bias + sum_j w_j x_{t-W+1+j}) reads x once and writes v once: bound by memory.  A thread holds V = 2 channels (1 where there
// is only one, and in a step of an odd width) and walks a run of 8 or 16 steps with the last W - 1 inputs in registers, CONV_FLY rows in flight; the W - 1 rows
// before a run are read again (from cache).  Wider vectors have fewer waves to wait with: backward over 8191 x 1024 bf16 46 us with 8 channels
// a thread, 31 with 4, 26 with 2; runs of 8 steps 36 (4 channels), of 32 29 (2 channels); 8 rows in flight change nothing.  Forward, 8 x 65536 x
// 64 fp32: 49 us, 5.5 TB/s; in 16 bits a thread's two channels make accesses of 4 bytes, and 8191 x 1024 takes 11 us, 3.0 TB/s: the waves wait
// 0.63 of their cycles (SQ_WAIT_ANY), the vector unit issues 0.58 of the time.
#define CONV_FLY 4
#define CONV_V 2
struct ConvDev {
  rgp_ssm_conv a;
  SeqGeo g;
  int64_t nrun, nvec;
  int lg;                          // a run has 2^lg steps
  int wide, same, lanes;           // pairs of channels; a wave's lanes are in one run; vectors side by side in a workgroup (backward)
  void* part;
};

// first channel of a vector: the last one of an odd width is moved back by one
template <int V>
static __device__ __forceinline__ int64_t conv_at(int64_t vec, int D) { return vec * V + V <= D ? vec * V : D - V; }

// x at step t of the sequence, in walking order; before the first step the state
template <typename T, int W, int V>
static __device__ __forceinline__ SeqAny<T, V> conv_x(const ConvDev& d, const SeqBlock& b, int64_t t, int64_t c) {
  const rgp_ssm_conv& a = d.a;
  if (t >= 0) return *(const SeqAny<T, V>*)(seq_row((const T*)a.x, d.g, b, SeqStride{a.x_st, a.x_sb}, t) + c);
  SeqAny<T, V> z;
#pragma unroll
  for (int i = 0; i < V; ++i) z.e[i] = a.init ? ((const T*)a.init)[(b.seq * (W - 1) + W - 1 + t) * a.D + c + i] : (T)0;
  return z;
}

template <typename T, int W, int V>
static __global__ void __launch_bounds__(256) conv_fwd_kernel(ConvDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  const rgp_ssm_conv& a = d.a;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x, run = idx / (uint32_t)d.nvec;
  const int64_t c = conv_at<V>(idx - run * (uint32_t)d.nvec, a.D);
  if (run >= d.nrun) return;
  const SeqBlock b = seq_find(d.g, d.same ? (uint32_t)__builtin_amdgcn_readfirstlane(run) : run, d.lg);
  if (!b.ok) return;
  const int64_t t0 = b.j << d.lg;
  const int L = 1 << d.lg, nt = b.len - t0 < L ? (int)(b.len - t0) : L;
  A w[W][V], bias[V], x[W - 1 + CONV_FLY][V];      // x: the W - 1 rows before a batch of steps and the batch's, in the arithmetic type
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias ? ((const A*)a.bias)[c + i] : (A)0;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][i] = ((const A*)a.w)[(c + i) * W + j];
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const Vec r = conv_x<T, W, V>(d, b, t0 - (W - 1) + j, c);
#pragma unroll
    for (int i = 0; i < V; ++i) x[j][i] = (A)r.e[i];
  }
  const T* px = seq_row((const T*)a.x, d.g, b, SeqStride{a.x_st, a.x_sb}, t0) + c;
  T* pv = (T*)a.v + seq_row_index(d.g, b, t0) * a.D + c;
  const int64_t sx = d.g.reverse ? -a.x_st : a.x_st, vrow = (d.g.off ? 1 : (int64_t)a.n_seq) * a.D, sv = d.g.reverse ? -vrow : vrow;
  for (int tb = 0; tb < nt; tb += CONV_FLY) {
#pragma unroll
    for (int k = 0; k < CONV_FLY; ++k) {           // behind the end the last row again
      const Vec r = *(const Vec*)px;
      px += tb + k + 1 < nt ? sx : 0;
#pragma unroll
      for (int i = 0; i < V; ++i) x[W - 1 + k][i] = (A)r.e[i];
    }
#pragma unroll
    for (int k = 0; k < CONV_FLY; ++k) {
      Vec o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        A p = bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) p += w[j][i] * x[k + j][i];
        o.e[i] = (T)(p * seq_sigmoid(p));
      }
      if (tb + k < nt) *(Vec*)pv = o;
      pv += sv;
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) x[j][i] = x[j + CONV_FLY][i];
  }
}
// the W - 1 inputs before the step behind the last one
template <typename T, int W, int V>
static __global__ void __launch_bounds__(256) conv_last_kernel(ConvDev d) {
  const rgp_ssm_conv& a = d.a;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, seq = idx / d.nvec, c = conv_at<V>(idx - seq * d.nvec, a.D);
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
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const SeqAny<T, V> x = conv_x<T, W, V>(d, b, b.len - (W - 1) + j, c);
#pragma unroll
    for (int i = 0; i < V; ++i) ((T*)a.last)[(seq * (W - 1) + j) * a.D + c + i] = x.e[i];
  }
}

// Backward (8191 x 1024 bf16 26 us, 1.9 TB/s, 32 x 4096 x 64 fp32 30, 3.3 TB/s: the waves wait 0.66 of their cycles, the vector unit issues 0.55 of
// the time): gp = gv silu'(pre), gx_t
// = sum_j w_j gp_{t+W-1-j}, gw_j = sum_t gp_t x_{t-W+1+j}, gbias = sum gp.  pre is formed again from x (one more read would cost more than W
// multiply-adds).  A thread walks its runs and W - 1 steps behind each; the parameter sums of the threads with the same channels go through
// LDS, then from all workgroups through `part`.
template <typename T, int W, int V>
static __global__ void __launch_bounds__(256) conv_bwd_kernel(ConvDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  __shared__ A sh[256 * V];
  const rgp_ssm_conv& a = d.a;
  const int lane = threadIdx.x % d.lanes, rl = threadIdx.x / d.lanes, nr = 256 / d.lanes;
  const int64_t vec = (int64_t)blockIdx.y * d.lanes + lane, c = conv_at<V>(vec, a.D);
  const bool live = vec < d.nvec;
  const int twice = live ? (int)(vec * V - c) : 0;                       // channels that the vector before counts
  A w[W][V], bias[V], gw[W][V], gb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias && live ? ((const A*)a.bias)[c + i] : (A)0;
    gb[i] = (A)0;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      w[j][i] = live ? ((const A*)a.w)[(c + i) * W + j] : (A)0;
      gw[j][i] = (A)0;
    }
  }
  if (live)
    for (int64_t run = (int64_t)blockIdx.x * nr + rl; run < d.nrun; run += (int64_t)gridDim.x * nr) {
      const SeqBlock b = seq_find(d.g, d.lanes == 64 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)run) : (uint32_t)run, d.lg);
      if (!b.ok) continue;
      const int64_t t0 = b.j << d.lg, L = (int64_t)1 << d.lg, t1 = t0 + L < b.len ? t0 + L : b.len;
      // x and gp: the W - 1 steps before a batch and the batch's.  Steps past the end are computed like the others, with gp = 0: branches
      // around them would keep the windows from being renamed instead of moved.
      A x[W - 1 + CONV_FLY][V], gp[W - 1 + CONV_FLY][V];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        const Vec r = conv_x<T, W, V>(d, b, t0 - (W - 1) + j, c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[j][i] = (A)r.e[i];
          gp[j][i] = (A)0;
        }
      }
      const int nt = (int)(t1 - t0) + W - 1;                             // gp of step t0 + k; gx of step t0 + k - W + 1 is then complete
      const int in = (int)(t1 - t0), have = b.len - t0 < nt ? (int)(b.len - t0) : nt;
      const T* px = seq_row((const T*)a.x, d.g, b, SeqStride{a.x_st, a.x_sb}, t0) + c;
      const T* pg = seq_row((const T*)a.gv, d.g, b, SeqStride{a.gv_st, a.gv_sb}, t0) + c;
      T* po = (T*)a.gx + seq_row_index(d.g, b, t0) * a.D + c;
      const int64_t orow = (d.g.off ? 1 : (int64_t)a.n_seq) * a.D;
      const int64_t sx = d.g.reverse ? -a.x_st : a.x_st, sg = d.g.reverse ? -a.gv_st : a.gv_st, so = d.g.reverse ? -orow : orow;
      po -= (W - 1) * so;                                                // moves with gp's step, W - 1 steps ahead of gx's
      for (int kb = 0; kb < nt; kb += CONV_FLY) {
        Vec rg[CONV_FLY];
#pragma unroll
        for (int k = 0; k < CONV_FLY; ++k) {
          const Vec r = *(const Vec*)px;                                 // behind the end the last row again
          rg[k] = *(const Vec*)pg;
          px += kb + k + 1 < have ? sx : 0;
          pg += kb + k + 1 < have ? sg : 0;
#pragma unroll
          for (int i = 0; i < V; ++i) x[W - 1 + k][i] = (A)r.e[i];
        }
#pragma unroll
        for (int k = 0; k < CONV_FLY; ++k) {
          Vec o;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            A p = bias[i];
#pragma unroll
            for (int j = 0; j < W; ++j) p += w[j][i] * x[k + j][i];
            const A sg_ = seq_sigmoid(p);
            const A q = kb + k < have ? (A)rg[k].e[i] * (sg_ + p * sg_ * ((A)1 - sg_)) : (A)0;
            gp[W - 1 + k][i] = q;
            const A own = kb + k < in ? q : (A)0;                        // the W - 1 steps behind the run count in the next one
            gb[i] += own;
#pragma unroll
            for (int j = 0; j < W; ++j) gw[j][i] += own * x[k + j][i];
            A v = (A)0;
#pragma unroll
            for (int j = 0; j < W; ++j) v += w[W - 1 - j][i] * gp[k + j][i];      // gp[k + j] is j steps on, and its tap W - 1 - j reads this x
            o.e[i] = (T)v;
          }
          if (kb + k >= W - 1 && kb + k < nt) *(Vec*)po = o;
          po += so;
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            x[j][i] = x[j + CONV_FLY][i];
            gp[j][i] = gp[j + CONV_FLY][i];
          }
      }
    }
  A* const part = (A*)d.part + (int64_t)blockIdx.x * (W + 1) * a.D;      // [W][D] taps, then [D] bias
#pragma unroll
  for (int j = 0; j <= W; ++j) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i >= twice) sh[threadIdx.x * V + i - twice] = j < W ? gw[j < W ? j : 0][i] : gb[i];
    __syncthreads();
    for (int e = threadIdx.x; e < d.lanes * V; e += 256) {
      A v = (A)0;
      for (int q = 0; q < nr; ++q) v += sh[q * d.lanes * V + e];
      const int64_t ch = (int64_t)blockIdx.y * d.lanes * V + e;
      if (ch < a.D) part[j * a.D + ch] = v;
    }
    __syncthreads();
  }
}

template <typename T, int W, int V>
static __global__ void __launch_bounds__(256) conv_step_kernel(ConvDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  const rgp_ssm_conv& a = d.a;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x, seq = idx / (uint32_t)d.nvec;
  const int64_t c = (int64_t)(idx - seq * (uint32_t)d.nvec) * V;
  if (seq >= (uint32_t)a.n_seq) return;
  T* const st = (T*)a.last + (int64_t)seq * (W - 1) * a.D + c;
  Vec x[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) x[j] = *(const Vec*)(st + (int64_t)j * a.D);
  x[W - 1] = *(const Vec*)((const T*)a.x + seq * a.x_sb + c);
  A w[V][W];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) w[i][j] = ((const A*)a.w)[(c + i) * W + j];
  Vec o;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    A p = a.bias ? ((const A*)a.bias)[c + i] : (A)0;
#pragma unroll
    for (int j = 0; j < W; ++j) p += w[i][j] * (A)x[j].e[i];
    o.e[i] = (T)(p * seq_sigmoid(p));
  }
  *(Vec*)((T*)a.v + (int64_t)seq * a.D + c) = o;
#pragma unroll
  for (int j = 0; j < W - 1; ++j) *(Vec*)(st + (int64_t)j * a.D) = x[j + 1];
}

static const char* conv_bad(const rgp_ssm_conv* a) {
  if (!a) return "null arguments";
  if (a->dtype < 0 || a->dtype > 3) return "dtype must be RGP_F64, RGP_F32, RGP_BF16 or RGP_F16";
  if (a->n_seq < 1 || a->D < 1 || a->rows < 0 || a->T < 0) return "empty problem";
  if (a->W < 2 || a->W > 8) return "2 to 8 taps";
  if (a->rows > SEQ_MOST || a->T > SEQ_MOST) return "more than 2^40 rows";
  if (!a->off && (a->T < 1 || a->T * a->n_seq != a->rows)) return "rows must be T * n_seq, T >= 1";
  return nullptr;
}
static void conv_plan(const rgp_ssm_conv* a, bool wide, ConvDev& d, int64_t& nrb, int64_t& nvb) {
  d = ConvDev{};
  d.a = *a;
  d.g = SeqGeo{a->off, a->T, a->rows, a->n_seq, a->reverse};
  d.wide = wide;
  const int V = wide ? CONV_V : 1;
  d.nvec = (a->D + V - 1) / V;
  d.same = d.nvec % 64 == 0;
  // runs of 16 steps unless that leaves fewer than two waves a SIMD
  for (d.lg = 4; d.lg > 3 && seq_blocks(d.g, d.lg) * d.nvec < 131072; --d.lg) {}
  d.nrun = seq_blocks(d.g, d.lg);
  d.lanes = 1;
  while (d.lanes < 64 && d.lanes < d.nvec) d.lanes *= 2;
  nvb = (d.nvec + d.lanes - 1) / d.lanes;
  const int64_t nr = 256 / d.lanes, most = nvb > 2048 ? 1 : 2048 / nvb;  // eight workgroups a CU; more only lengthens the sum over them
  nrb = (d.nrun + nr - 1) / nr;
  if (nrb > most) nrb = most;
  if (nrb < 1) nrb = 1;
}
extern "C" int64_t rgp_ssm_conv_workspace(const rgp_ssm_conv* a, int backward) {
  if (conv_bad(a)) return -1;
  if (!backward) return 0;
  ConvDev d;
  int64_t nrb, nvb;
  conv_plan(a, a->D >= CONV_V, d, nrb, nvb);
  return nrb * (a->W + 1) * a->D * (a->dtype == RGP_F64 ? 8 : 4);
}

enum { CONV_FWD, CONV_LAST, CONV_BWD, CONV_STEP };
template <typename T, int W, int V>
static hipError_t conv_go(const ConvDev& d, int what, dim3 grid, hipStream_t s) {
  if (grid.x < 1) return hipSuccess;
  if (what == CONV_FWD) hipLaunchKernelGGL((conv_fwd_kernel<T, W, V>), grid, dim3(256), 0, s, d);
  else if (what == CONV_LAST) hipLaunchKernelGGL((conv_last_kernel<T, W, V>), grid, dim3(256), 0, s, d);
  else if (what == CONV_BWD) hipLaunchKernelGGL((conv_bwd_kernel<T, W, V>), grid, dim3(256), 0, s, d);
  else hipLaunchKernelGGL((conv_step_kernel<T, W, V>), grid, dim3(256), 0, s, d);
  return hipGetLastError();
}
template <typename T, int W>
static hipError_t conv_wide(const ConvDev& d, int what, dim3 grid, hipStream_t s) {
  return d.wide ? conv_go<T, W, CONV_V>(d, what, grid, s) : conv_go<T, W, 1>(d, what, grid, s);
}
template <typename T>
static hipError_t conv_taps(const ConvDev& d, int what, dim3 grid, hipStream_t s) {
  switch (d.a.W) {
    case 2: return conv_wide<T, 2>(d, what, grid, s);
    case 3: return conv_wide<T, 3>(d, what, grid, s);
    case 4: return conv_wide<T, 4>(d, what, grid, s);
    case 5: return conv_wide<T, 5>(d, what, grid, s);
    case 6: return conv_wide<T, 6>(d, what, grid, s);
    case 7: return conv_wide<T, 7>(d, what, grid, s);
    default: return conv_wide<T, 8>(d, what, grid, s);
  }
}
static hipError_t conv_launch(const ConvDev& d, int what, dim3 grid, hipStream_t s) {
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
  const bool some = a->rows > 0;                       // without rows the activations may have no memory
  if (!a->w || (some && !a->x)) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "x and w are required");
  if (what == CONV_BWD && (!a->gw || (some && (!a->gv || !a->gx)))) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "gv, gx and gw are required");
  if (what == CONV_STEP && (a->off || a->T != 1)) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "one row per sequence (T = 1, no offsets)");
  if (what == CONV_STEP && (!a->v || !a->last || a->init != a->last)) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "v and the state (init = last) are required");
  if (what == CONV_FWD && some && !a->v) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "v is required");
  if (what == CONV_FWD && seq_overlap(a->last, a->init, (int64_t)a->n_seq * (a->W - 1) * a->D * seq_dtype_bytes(a->dtype)))
    return rgp_fail(h, RGP_ERR_BAD_ARG, name + "last must not share memory with init");
  const bool wide = what == CONV_STEP ? a->D % CONV_V == 0 : a->D >= CONV_V;      // a step changes its state in place: no channel twice
  ConvDev d;
  int64_t nrb, nvb;
  conv_plan(a, wide, d, nrb, nvb);
  const int64_t seqs = ((int64_t)a->n_seq * d.nvec + 255) / 256;
  if ((double)d.nrun * d.nvec > 4294967295.0 - 256.0 || (double)a->n_seq * d.nvec > 4294967295.0 - 256.0 || nvb > 65535 || (double)nrb * 256 > 4294967295.0)
    return rgp_fail(h, RGP_ERR_BAD_ARG, name + "more than 2^32 work items");
  hipError_t err = hipSuccess;
  if (what == CONV_BWD) {
    if (rgp_ssm_conv_workspace(a, 1) > a->work_bytes || !a->work || ((uintptr_t)a->work & 15))
      return rgp_fail(h, RGP_ERR_WORKSPACE, name + "work buffer too small or not 16-byte aligned");
    d.part = a->work;
    err = conv_launch(d, CONV_BWD, dim3((unsigned)nrb, (unsigned)nvb), s);
    if (err == hipSuccess) {
      const int acc = a->dtype == RGP_F64 ? RGP_F64 : RGP_F32;
      const int64_t n = (int64_t)a->W * a->D, per = n + a->D;
      SeqSums sums;
      sums.add(d.part, nrb, per, n, a->gw, acc, a->W);
      sums.add((char*)d.part + n * (acc == RGP_F64 ? 8 : 4), nrb, per, a->D, a->gbias, acc);
      return sums.run(h, s, acc);
    }
  } else if (what == CONV_STEP) {
    err = conv_launch(d, CONV_STEP, dim3((unsigned)seqs), s);
  } else {
    err = conv_launch(d, CONV_FWD, dim3((unsigned)((d.nrun * d.nvec + 255) / 256)), s);
    if (err == hipSuccess && a->last) err = conv_launch(d, CONV_LAST, dim3((unsigned)seqs), s);
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
