// rgp_norm.hip -- root-mean-square norm of x + residual and its gradient; global norm of many gradient tensors and their clipping.
// All of it is bound by memory: every kernel reads its operands once, 16 bytes a lane, and keeps a row in registers between the sum of
// squares and the product.  Norm of 16384 x 2048 bf16: forward 52 us, 5.2 TB/s, backward 72 us, 4.7 TB/s (a large copy reaches 5.07); rows of 300 or
// 1001 elements the same to 6 %; 5 x 2048: 3.6 us, the launch.  Clipping of 400 M bf16 elements: 193 us for the norm (4.1 TB/s), 283 for the scaling
// (5.7 TB/s, helped by what the norm left in the memory-side cache); 84 211 fp64 elements in 39 tensors: 4.6 + 5.1 us.
#include "rgp_seq.h"

struct NormDev {
  rgp_rms_norm a;
  void* part;
};

// sum over the TPR threads of a row; TPR <= 64: lanes of one wave, else the whole workgroup of TPR threads
template <int TPR, typename A>
static __device__ __forceinline__ A row_sum(A v, A* sh) {
  if constexpr (TPR <= 64) {
    return seq_sum_wide<TPR>(v);
  } else {
    v = seq_sum_wide<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    A s = (A)0;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) s += sh[i];
    return s;
  }
}

// TPR threads a row, NE vectors of V elements each (16 bytes; V = 1 for rows shorter than that); rows of TPR * NE * V >= C elements. WHOLE: C
// is a multiple of V, otherwise the row's last vector is moved back and its first elements belong to the one before.  A workgroup takes every
// gridDim-th group of rows and keeps w; the next rows are loaded while these are normed.  hid is rounded to its type where it is written; the
// norm uses the sum before that rounding.
template <typename T, int TPR, int NE, int V, bool WHOLE>
static __global__ void __launch_bounds__(256) rms_fwd_kernel(NormDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  constexpr int RPB = 256 / TPR;
  __shared__ A sh[4];
  const rgp_rms_norm& a = d.a;
  const int l = threadIdx.x % TPR, rg = threadIdx.x / TPR;
  A w[NE][V];
  int64_t col[NE];
  bool in[NE];
  int own[NE];                                       // first element that this lane counts
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int64_t c = (int64_t)(l + i * TPR) * V;
    in[i] = c < a.C;
    col[i] = !in[i] ? 0 : WHOLE || c + V <= a.C ? c : a.C - V;
    own[i] = in[i] ? (int)(c - col[i]) : V;
#pragma unroll
    for (int j = 0; j < V; ++j) w[i][j] = in[i] ? ((const A*)a.w)[col[i] + j] : (A)0;
  }
  Vec x[NE], r[NE];
  auto fetch = [&](int64_t row) {                    // rows behind the last one read the last one
    const int64_t rr = row < a.rows ? row : a.rows - 1;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      x[i] = *(const Vec*)((const T*)a.x + rr * a.x_st + col[i]);
      if (a.residual) r[i] = *(const Vec*)((const T*)a.residual + rr * a.residual_st + col[i]);
    }
  };
  int64_t r0 = (int64_t)blockIdx.x * RPB;
  if (r0 < a.rows) fetch(r0 + rg);
  for (; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + rg;
    A h[NE][V], q = (A)0;
#pragma unroll
    for (int i = 0; i < NE; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = (A)x[i].e[j] + (a.residual ? (A)r[i].e[j] : (A)0);
        q += (WHOLE ? in[i] : j >= own[i]) ? h[i][j] * h[i][j] : (A)0;
      }
    if (r0 + (int64_t)gridDim.x * RPB < a.rows) fetch(row + (int64_t)gridDim.x * RPB);
    q = row_sum<TPR>(q, sh);
    const A rs = seq_rsqrt(q / (A)a.C + (A)a.eps);
    if (row < a.rows) {
      if (a.rstd && l == 0) ((A*)a.rstd)[row] = rs;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        if (in[i]) {
          Vec y, o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            o.e[j] = (T)h[i][j];
            y.e[j] = (T)(h[i][j] * rs * w[i][j]);
          }
          *(Vec*)((T*)a.y + row * a.C + col[i]) = y;
          if (a.hid) *(Vec*)((T*)a.hid + row * a.C + col[i]) = o;
        }
      }
    }
  }
}
// rows longer than a workgroup's registers: the sum of squares, then the row once more
template <typename T, int V>
static __global__ void __launch_bounds__(256) rms_fwd_long_kernel(NormDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  __shared__ A sh[4];
  const rgp_rms_norm& a = d.a;
  const int64_t row = blockIdx.x;
  A q = (A)0, rs = (A)0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 256 * V) {
      const Vec x = *(const Vec*)((const T*)a.x + row * a.x_st + c);
      Vec r, y, o;
      if (a.residual) r = *(const Vec*)((const T*)a.residual + row * a.residual_st + c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const A h = (A)x.e[j] + (a.residual ? (A)r.e[j] : (A)0);
        if (pass == 0) q += h * h;
        o.e[j] = (T)h;
        y.e[j] = (T)(h * rs * ((const A*)a.w)[c + j]);
      }
      if (pass == 1) {
        *(Vec*)((T*)a.y + row * a.C + c) = y;
        if (a.hid) *(Vec*)((T*)a.hid + row * a.C + c) = o;
      }
    }
    if (pass == 0) {
      q = row_sum<256>(q, sh);
      rs = seq_rsqrt(q / (A)a.C + (A)a.eps);
      if (a.rstd && threadIdx.x == 0) ((A*)a.rstd)[row] = rs;
    }
  }
}

// gx = ghid + r (gy w - hid r^2 mean(gy w hid)); gw = sum over rows of gy hid r.  hid is x + residual again, before its rounding to a 16-bit
// storage type: gw is a sum over many rows in 32 bits, and that rounding (2^-9 relative) would be its largest error by far.  A workgroup
// takes every gridDim-th group of rows, sums gw in registers and adds its row groups through LDS; the workgroups' sums are added in a fixed
// order afterwards.
template <typename T, int TPR, int NE, int V, bool WHOLE>
static __global__ void __launch_bounds__(256, NE * V * sizeof(typename SeqAcc<T>::type) > 128 ? 1 : 2) rms_bwd_kernel(NormDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  constexpr int RPB = 256 / TPR;
  __shared__ A sh[4];
  __shared__ A acc[256 * V];
  const rgp_rms_norm& a = d.a;
  const int l = threadIdx.x % TPR, rg = threadIdx.x / TPR;
  A gw[NE][V], w[NE][V];
  int64_t col[NE];
  bool in[NE];
  int own[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int64_t c = (int64_t)(l + i * TPR) * V;
    in[i] = c < a.C;
    col[i] = !in[i] ? 0 : WHOLE || c + V <= a.C ? c : a.C - V;
    own[i] = in[i] ? (int)(c - col[i]) : V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      gw[i][j] = (A)0;
      w[i][j] = in[i] ? ((const A*)a.w)[col[i] + j] : (A)0;
    }
  }
  const A inv = (A)1 / (A)a.C;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + rg;
    const bool live = row < a.rows;
    const int64_t rr = live ? row : a.rows - 1;
    Vec x[NE], r[NE], g[NE], gh[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      x[i] = *(const Vec*)((const T*)a.x + rr * a.x_st + col[i]);
      if (a.residual) r[i] = *(const Vec*)((const T*)a.residual + rr * a.residual_st + col[i]);
      g[i] = *(const Vec*)((const T*)a.gy + rr * a.gy_st + col[i]);
      if (a.ghid) gh[i] = *(const Vec*)((const T*)a.ghid + rr * a.ghid_st + col[i]);
    }
    const A rs = ((const A*)a.rstd)[rr];
    A hid[NE][V], q = (A)0;
#pragma unroll
    for (int i = 0; i < NE; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        hid[i][j] = (A)x[i].e[j] + (a.residual ? (A)r[i].e[j] : (A)0);
        q += (WHOLE ? in[i] : j >= own[i]) ? (A)g[i].e[j] * w[i][j] * hid[i][j] : (A)0;
      }
    q = row_sum<TPR>(q, sh) * inv * rs * rs;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      if (in[i] && live) {
        Vec o;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const A gy = (A)g[i].e[j], h = hid[i][j];
          A v = rs * (gy * w[i][j] - h * q);
          if (a.ghid) v += (A)gh[i].e[j];
          o.e[j] = (T)v;
          gw[i][j] += gy * h * rs;
        }
        *(Vec*)((T*)a.gx + rr * a.C + col[i]) = o;
      }
    }
  }
  A* const part = (A*)d.part + (int64_t)blockIdx.x * a.C;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (WHOLE || j >= own[i]) acc[threadIdx.x * V + j - (WHOLE ? 0 : own[i])] = gw[i][j];       // what is left out lies behind the row's end
    __syncthreads();
    for (int e = threadIdx.x; e < TPR * V; e += 256) {
      A v = (A)0;
#pragma unroll
      for (int q = 0; q < RPB; ++q) v += acc[q * TPR * V + e];
      const int64_t c = (int64_t)i * TPR * V + e;
      if (c < a.C) part[c] = v;
    }
  }
}
// rows longer than a workgroup's registers: gw goes through memory, one row of the partial sums per workgroup
template <typename T, int V>
static __global__ void __launch_bounds__(256) rms_bwd_long_kernel(NormDev d) {
  typedef typename SeqAcc<T>::type A;
  typedef SeqAny<T, V> Vec;
  __shared__ A sh[4];
  const rgp_rms_norm& a = d.a;
  A* const part = (A*)d.part + (int64_t)blockIdx.x * a.C;
  for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 256 * V)      // the elements that this thread adds to below
#pragma unroll
    for (int j = 0; j < V; ++j) part[c + j] = (A)0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const A rs = ((const A*)a.rstd)[row];
    A q = (A)0;
    for (int pass = 0; pass < 2; ++pass) {
      for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 256 * V) {
        const Vec x = *(const Vec*)((const T*)a.x + row * a.x_st + c);
        const Vec g = *(const Vec*)((const T*)a.gy + row * a.gy_st + c);
        Vec r, gh, o;
        if (a.residual) r = *(const Vec*)((const T*)a.residual + row * a.residual_st + c);
        if (pass == 1 && a.ghid) gh = *(const Vec*)((const T*)a.ghid + row * a.ghid_st + c);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const A w = ((const A*)a.w)[c + j], gy = (A)g.e[j], h = (A)x.e[j] + (a.residual ? (A)r.e[j] : (A)0);
          if (pass == 0) {
            q += gy * w * h;
          } else {
            o.e[j] = (T)((a.ghid ? (A)gh.e[j] : (A)0) + rs * (gy * w - h * q));
            part[c + j] += gy * h * rs;
          }
        }
        if (pass == 1) *(Vec*)((T*)a.gx + row * a.C + c) = o;
      }
      if (pass == 0) q = row_sum<256>(q, sh) / (A)a.C * rs * rs;
    }
  }
}

// Threads a row and vectors a thread: of the shapes that hold a row, the one that leaves the fewest lanes idle, and of those the one with the
// fewest threads a row -- unless the rows are few, where more threads a row finish it sooner.
struct RmsShape { int tpr, ne; };
static RmsShape rms_shape(const rgp_rms_norm* a) {
  const int V = 16 / seq_dtype_bytes(a->dtype);
  if (a->C < V) return RmsShape{8, 1};                                        // single elements, at most 7 of them
  const int64_t nv = (a->C + V - 1) / V, rows = a->rows;
  static const int tprs[5] = {8, 16, 32, 64, 256}, nes[5] = {1, 2, 3, 4, 8};
  RmsShape best{0, 0};
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < 5; ++j) {
      const int64_t hold = (int64_t)tprs[i] * nes[j];
      if (hold < nv || (nes[j] == 8 && tprs[i] < 256) || (tprs[i] == 32 && nes[j] != 3)) continue;       // 32 threads fill the gap between 64 and 128
      const bool few = rows * tprs[i] <= 65536;                          // fewer threads than the card has lanes: the wider shape is free
      if (!best.tpr || hold < (int64_t)best.tpr * best.ne || (few && tprs[i] > best.tpr && hold <= 2 * (int64_t)best.tpr * best.ne))
        best = RmsShape{tprs[i], nes[j]};
    }
  return best;
}
static int64_t rms_blocks(const rgp_rms_norm* a, RmsShape s, int64_t most) {
  const int64_t rpb = s.tpr ? 256 / s.tpr : 1, want = (a->rows + rpb - 1) / rpb;
  return want < most ? (want < 1 ? 1 : want) : most;
}
// Backward: as many workgroups as are resident at once, two a CU (their sums of gw have to be joined, and a second round of a few is as long as
// the first: 599 instead of 512 for 4793 x 7000 bf16 take 117 us instead of 83).  Short rows, of which a thread holds little, have room for
// more, as long as each keeps eight groups of rows: 838860 x 40 takes 75 us with 2048, 116 with 512.
#define RMS_FWD_BLOCKS 2048
static int64_t rms_bwd_blocks(const rgp_rms_norm* a, RmsShape s) {
  const int64_t eight = s.tpr == 8 && s.ne <= 2 ? rms_blocks(a, s, INT64_MAX) / 8 : 0;
  return rms_blocks(a, s, eight < 512 ? 512 : eight > 2048 ? 2048 : eight);
}
static const char* rms_bad(const rgp_rms_norm* a) {
  if (!a) return "null arguments";
  if (a->dtype < 0 || a->dtype > 3) return "dtype must be RGP_F64, RGP_F32, RGP_BF16 or RGP_F16";
  if (a->rows < 0 || a->C < 1) return "empty rows";
  if (a->rows > SEQ_MOST || a->C > SEQ_MOST) return "more than 2^40 rows or columns";
  if (!(a->dtype == RGP_F64 ? a->eps > 0.0 : (float)a->eps > 0.0f)) return "eps must be positive in the arithmetic type";
  return nullptr;
}
extern "C" int64_t rgp_rms_norm_workspace(const rgp_rms_norm* a, int backward) {
  if (rms_bad(a)) return -1;
  if (!backward) return 0;
  return rms_bwd_blocks(a, rms_shape(a)) * a->C * (a->dtype == RGP_F64 ? 8 : 4);
}
template <typename T, int TPR, int NE, int V>
static hipError_t rms_go(const NormDev& d, bool back, int64_t blocks, hipStream_t s) {
  const dim3 g((unsigned)blocks), t(256);
  if (V == 1 || d.a.C % V == 0) {
    if (back) hipLaunchKernelGGL((rms_bwd_kernel<T, TPR, NE, V, true>), g, t, 0, s, d);
    else hipLaunchKernelGGL((rms_fwd_kernel<T, TPR, NE, V, true>), g, t, 0, s, d);
  } else if constexpr (V > 1) {
    if (back) hipLaunchKernelGGL((rms_bwd_kernel<T, TPR, NE, V, false>), g, t, 0, s, d);
    else hipLaunchKernelGGL((rms_fwd_kernel<T, TPR, NE, V, false>), g, t, 0, s, d);
  }
  return hipGetLastError();
}
template <typename T, int TPR>
static hipError_t rms_ne(const NormDev& d, int ne, bool back, int64_t blocks, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  switch (ne) {
    case 1: return rms_go<T, TPR, 1, V>(d, back, blocks, s);
    case 2: return rms_go<T, TPR, 2, V>(d, back, blocks, s);
    case 3: return rms_go<T, TPR, 3, V>(d, back, blocks, s);
    case 4: return rms_go<T, TPR, 4, V>(d, back, blocks, s);
    default:
      if constexpr (TPR == 256) return rms_go<T, TPR, 8, V>(d, back, blocks, s);
      return hipErrorInvalidValue;
  }
}
template <typename T, int V>
static hipError_t rms_long(const NormDev& d, bool back, int64_t blocks, hipStream_t s) {
  if (back) hipLaunchKernelGGL((rms_bwd_long_kernel<T, V>), dim3((unsigned)blocks), dim3(256), 0, s, d);
  else hipLaunchKernelGGL((rms_fwd_long_kernel<T, V>), dim3((unsigned)d.a.rows), dim3(256), 0, s, d);
  return hipGetLastError();
}
template <typename T>
static hipError_t rms_pick(const NormDev& d, RmsShape sh, bool back, int64_t blocks, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (d.a.C < V) return rms_go<T, 8, 1, 1>(d, back, blocks, s);                 // the shape of up to 8 single elements
  switch (sh.tpr) {
    case 8: return rms_ne<T, 8>(d, sh.ne, back, blocks, s);
    case 16: return rms_ne<T, 16>(d, sh.ne, back, blocks, s);
    case 32: return rms_go<T, 32, 3, V>(d, back, blocks, s);
    case 64: return rms_ne<T, 64>(d, sh.ne, back, blocks, s);
    case 256: return rms_ne<T, 256>(d, sh.ne, back, blocks, s);
    default: return d.a.C % V == 0 ? rms_long<T, V>(d, back, blocks, s) : rms_long<T, 1>(d, back, blocks, s);
  }
}
static rgp_status rms_run(rgp_handle h, hipStream_t s, const rgp_rms_norm* a, bool back) {
  const std::string name = back ? "rms norm backward: " : "rms norm: ";
  if (const char* bad = rms_bad(a)) return rgp_fail(h, RGP_ERR_BAD_ARG, name + bad);
  if (!a->w || (back && !a->gw) || (a->rows > 0 && (!a->x || (!back && !a->y) || (back && (!a->gy || !a->gx || !a->rstd)))))
    return rgp_fail(h, RGP_ERR_BAD_ARG, name + "a required buffer is null");
  if (!back && a->rows > 0 && (a->residual != nullptr) != (a->hid != nullptr)) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "residual and hid go together");
  NormDev d{};
  d.a = *a;
  const RmsShape sh = rms_shape(a);
  // a workgroup a row; more of such rows would fill over 500 GB
  if (!back && !sh.tpr && a->rows > 16777215) return rgp_fail(h, RGP_ERR_BAD_ARG, name + "more than 2^24 - 1 rows of more than 32 KB");
  const int64_t blocks = back ? rms_bwd_blocks(a, sh) : rms_blocks(a, sh, RMS_FWD_BLOCKS);
  if (back && (rgp_rms_norm_workspace(a, 1) > a->work_bytes || !a->work || ((uintptr_t)a->work & 15)))
    return rgp_fail(h, RGP_ERR_WORKSPACE, name + "work buffer too small or not 16-byte aligned");
  d.part = a->work;
  if (!back && a->rows == 0) return RGP_OK;
  hipError_t err = a->dtype == RGP_F64 ? rms_pick<double>(d, sh, back, blocks, s) : a->dtype == RGP_F32 ? rms_pick<float>(d, sh, back, blocks, s)
                 : a->dtype == RGP_BF16 ? rms_pick<__bf16>(d, sh, back, blocks, s) : rms_pick<_Float16>(d, sh, back, blocks, s);
  if (err != hipSuccess) return rgp_fail(h, RGP_ERR_HIP, name + hipGetErrorString(err));
  if (!back) return RGP_OK;
  const int acc = a->dtype == RGP_F64 ? RGP_F64 : RGP_F32;
  SeqSums sums;
  sums.add(d.part, blocks, a->C, a->C, a->gw, acc);
  return sums.run(h, s, acc);
}
extern "C" rgp_status rgp_rms_norm_forward(rgp_handle h, void* stream, const rgp_rms_norm* a) {
  SEQ_ENTRY(h, "rms norm", { return rms_run(h, (hipStream_t)stream, a, false); })
}
extern "C" rgp_status rgp_rms_norm_backward(rgp_handle h, void* stream, const rgp_rms_norm* a) {
  SEQ_ENTRY(h, "rms norm", { return rms_run(h, (hipStream_t)stream, a, true); })
}

// ---- global gradient norm and clipping ---------------------------------------------------------------------------------------------------------
// The tensors of a launch travel in the kernel's arguments (GT of them), so nothing is uploaded and a captured launch keeps its table.
// A workgroup takes one piece of one tensor -- 64 KB, or 8 KB where all of them are little and a longer walk would only add latency; its sum
// of squares, in double, goes to its own place, and the places are added in a fixed order: by a workgroup of their own, or, up to GFEW of
// them, by every workgroup of the clipping (which saves a launch where launches are what counts).
#define GT 128
#define GFEW 1024
struct GradTable {
  void* p[GT];
  int64_t n[GT];
  int first[GT + 1];             // first piece of each tensor, counted inside the launch
  uint8_t dt[GT];
  int count, bytes;              // tensors, bytes of a piece
};
static inline int grad_piece_bytes(int n, const int64_t* numel, const int32_t* dtype) {
  int64_t all = 0;
  for (int i = 0; i < n; ++i) all += numel[i] * seq_dtype_bytes(dtype[i]);
  return all <= (4 << 20) ? 8192 : 65536;
}
static inline int64_t grad_pieces(int64_t n, int dt, int bytes) { return (n * seq_dtype_bytes(dt) + bytes - 1) / bytes; }

static __device__ __forceinline__ int grad_find(const GradTable& t, int piece) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= piece) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// calls f(pointer, n, wide) for the elements of one piece: single elements up to a 16-byte boundary, vectors, single elements
template <typename T, typename F>
static __device__ __forceinline__ void grad_walk(T* p, int64_t n, F f) {
  constexpr int V = SeqVec<T>::V;
  int64_t head = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
  if (head > n) head = n;
  const int64_t nv = (n - head) / V, tail = n - head - nv * V;
  if ((int64_t)threadIdx.x < head) f(p + threadIdx.x, 1, false);
  T* const q = p + head;
  for (int64_t v = threadIdx.x; v < nv; v += 256) f(q + v * V, V, true);
  if ((int64_t)threadIdx.x < tail) f(q + nv * V + threadIdx.x, 1, false);
}
template <typename T>
static __device__ __forceinline__ double grad_sum(T* p, int64_t n) {
  double s = 0.0;
  grad_walk(p, n, [&](T* q, int k, bool wide) {
    const SeqVec<T> v = seq_load((const T*)q, k, wide);
#pragma unroll
    for (int i = 0; i < SeqVec<T>::V; ++i) {
      const double x = (double)(typename SeqAcc<T>::type)v.e[i];
      s = fma(x, x, s);
    }
  });
  return s;
}
static __global__ void __launch_bounds__(256) grad_sumsq_kernel(GradTable t, double* part) {
  __shared__ double sh[16];
  const int i = grad_find(t, blockIdx.x);
  const int es = t.dt[i] == RGP_F64 ? 8 : t.dt[i] == RGP_F32 ? 4 : 2;
  const int64_t per = t.bytes / es, o = (int64_t)((int)blockIdx.x - t.first[i]) * per, n = t.n[i] - o < per ? t.n[i] - o : per;
  double s;
  switch (t.dt[i]) {
    case RGP_F64: s = grad_sum((double*)t.p[i] + o, n); break;
    case RGP_F32: s = grad_sum((float*)t.p[i] + o, n); break;
    case RGP_BF16: s = grad_sum((__bf16*)t.p[i] + o, n); break;
    default: s = grad_sum((_Float16*)t.p[i] + o, n); break;
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}
static __device__ __forceinline__ double grad_add(const double* part, int64_t n, double* sh) {
  const int step = blockDim.x;
  double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
  int64_t i = threadIdx.x;
  for (; i + 3 * step < n; i += 4 * step) {
    s0 += part[i];
    s1 += part[i + step];
    s2 += part[i + 2 * step];
    s3 += part[i + 3 * step];
  }
  for (; i < n; i += step) s0 += part[i];
  return block_sum((s0 + s1) + (s2 + s3), sh);
}
static __global__ void __launch_bounds__(1024) grad_total_kernel(const double* part, int64_t n, double* out) {
  __shared__ double sh[16];
  const double s = grad_add(part, n, sh);
  if (threadIdx.x == 0) out[0] = s;
}
template <typename T>
static __device__ __forceinline__ void grad_scale(T* p, int64_t n, double c) {
  typedef typename SeqAcc<T>::type A;
  auto each = [&](auto f) {
    grad_walk(p, n, [&](T* q, int k, bool wide) {
      SeqVec<T> v = seq_load((const T*)q, k, wide);
#pragma unroll
      for (int i = 0; i < SeqVec<T>::V; ++i) v.e[i] = (T)(A)((A)v.e[i] * f);
      seq_store(q, v, k, wide);
    });
  };
  if (sizeof(A) == 4 && c < 1.17549435082228751e-38) each(c);      // below the normal numbers of 32 bits the factor itself would be rounded away
  else each((A)c);
}
// sum: nsum places to add (1: the sum itself).  Walks tensors and pieces from the last to the first: what the norm read last is still in the
// memory-side cache.  The first workgroup of the launch that says so writes the norm.
static __global__ void __launch_bounds__(256) grad_clip_kernel(GradTable t, const double* sum, int nsum, double max_norm, double* norm_out) {
  __shared__ double sh[16];
  const double norm = sqrt(nsum == 1 ? sum[0] : grad_add(sum, nsum, sh)), c = max_norm / (norm + 1e-6);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = norm;
  if (t.count == 0 || !(c < 1.0) || !(norm < 1.7976931348623157e308)) return;           // nothing to clip, or a norm that is no number
  const int i = grad_find(t, blockIdx.x);
  const int es = t.dt[i] == RGP_F64 ? 8 : t.dt[i] == RGP_F32 ? 4 : 2;
  const int64_t per = t.bytes / es, o = (int64_t)(t.first[i + 1] - 1 - (int)blockIdx.x) * per, n = t.n[i] - o < per ? t.n[i] - o : per;
  switch (t.dt[i]) {
    case RGP_F64: grad_scale((double*)t.p[i] + o, n, c); break;
    case RGP_F32: grad_scale((float*)t.p[i] + o, n, c); break;
    case RGP_BF16: grad_scale((__bf16*)t.p[i] + o, n, c); break;
    default: grad_scale((_Float16*)t.p[i] + o, n, c); break;
  }
}

static const char* grad_bad(int n, const int64_t* numel, const int32_t* dtype) {
  if (n < 0 || (n > 0 && (!numel || !dtype))) return "null arguments";
  for (int i = 0; i < n; ++i) {
    if (numel[i] < 0) return "a negative element count";
    if (dtype[i] < 0 || dtype[i] > 3) return "dtype must be RGP_F64, RGP_F32, RGP_BF16 or RGP_F16";
  }
  return nullptr;
}
extern "C" int64_t rgp_grad_workspace(int n, const int64_t* numel, const int32_t* dtype) {
  if (grad_bad(n, numel, dtype)) return -1;
  const int bytes = grad_piece_bytes(n, numel, dtype);
  int64_t p = 0;
  for (int i = 0; i < n; ++i) p += grad_pieces(numel[i], dtype[i], bytes);
  return (p < 1 ? 1 : p) * (int64_t)sizeof(double);
}
// calls f(table, pieces, pieces before) for groups of up to GT tensors; back: from the last tensor to the first
template <typename F>
static rgp_status grad_tables(rgp_handle h, int n, void* const* ptr, const int64_t* numel, const int32_t* dtype, bool back, F f) {
  GradTable t;
  t.bytes = grad_piece_bytes(n, numel, dtype);
  int64_t before = 0;
  for (int k = 0; k < n;) {                              // a group: the next GT tensors that have elements, fewer where the grid would grow too long
    int64_t pieces = 0;
    t.count = 0;
    for (; k < n && t.count < GT; ++k) {
      const int i = back ? n - 1 - k : k;
      if (numel[i] == 0) continue;
      const int64_t add = grad_pieces(numel[i], dtype[i], t.bytes);
      if (add > 8000000) return rgp_fail(h, RGP_ERR_BAD_ARG, "gradient norm: a tensor of more than 500 GB");
      if (pieces + add > 8000000) break;
      t.p[t.count] = ptr[i];
      t.n[t.count] = numel[i];
      t.dt[t.count] = (uint8_t)dtype[i];
      t.first[t.count++] = (int)pieces;
      pieces += add;
    }
    if (!t.count) continue;
    t.first[t.count] = (int)pieces;
    const rgp_status st = f(t, (unsigned)pieces, before);
    if (st) return st;
    before += pieces;
  }
  return RGP_OK;
}
static rgp_status grad_check(rgp_handle h, int n, void* const* ptr, const int64_t* numel, const int32_t* dtype) {
  if (const char* bad = grad_bad(n, numel, dtype)) return rgp_fail(h, RGP_ERR_BAD_ARG, std::string("gradient norm: ") + bad);
  if (n > 0 && !ptr) return rgp_fail(h, RGP_ERR_BAD_ARG, "gradient norm: null arguments");
  for (int i = 0; i < n; ++i)
    if (numel[i] > 0 && (!ptr[i] || (uintptr_t)ptr[i] % seq_dtype_bytes(dtype[i]))) return rgp_fail(h, RGP_ERR_BAD_ARG, "gradient norm: a null or misaligned tensor");
  return RGP_OK;
}
// the pieces' sums in `work`; their number
static rgp_status grad_sums(rgp_handle h, hipStream_t s, int n, void* const* ptr, const int64_t* numel, const int32_t* dtype, void* work,
                            int64_t work_bytes, int64_t& total) {
  if (!work || ((uintptr_t)work & 7) || rgp_grad_workspace(n, numel, dtype) > work_bytes)
    return rgp_fail(h, RGP_ERR_WORKSPACE, "gradient norm: work buffer too small");
  total = 0;
  return grad_tables(h, n, ptr, numel, dtype, false, [&](const GradTable& t, unsigned pieces, int64_t before) {
    hipLaunchKernelGGL(grad_sumsq_kernel, dim3(pieces), dim3(256), 0, s, t, (double*)work + before);
    total = before + pieces;
    return seq_launched(h, "gradient norm");
  });
}
extern "C" rgp_status rgp_grad_sumsq(rgp_handle h, void* stream, int n, void* const* ptr, const int64_t* numel, const int32_t* dtype,
                                     double* sumsq, void* work, int64_t work_bytes) {
  SEQ_ENTRY(h, "gradient norm", {
    rgp_status st = grad_check(h, n, ptr, numel, dtype);
    if (st) return st;
    if (!sumsq) return rgp_fail(h, RGP_ERR_BAD_ARG, "gradient norm: sumsq is required");
    int64_t total = 0;
    st = grad_sums(h, (hipStream_t)stream, n, ptr, numel, dtype, work, work_bytes, total);
    if (st) return st;
    hipLaunchKernelGGL(grad_total_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const double*)work, total, sumsq);
    return seq_launched(h, "gradient norm");
  })
}
extern "C" rgp_status rgp_grad_clip(rgp_handle h, void* stream, int n, void* const* ptr, const int64_t* numel, const int32_t* dtype,
                                    const double* sumsq, double max_norm, double* norm, void* work, int64_t work_bytes) {
  SEQ_ENTRY(h, "gradient clip", {
    rgp_status st = grad_check(h, n, ptr, numel, dtype);
    if (st) return st;
    if (!norm || norm == sumsq || !(max_norm > 0.0)) return rgp_fail(h, RGP_ERR_BAD_ARG, "gradient clip: norm, apart from sumsq, and a positive max_norm are required");
    const hipStream_t s = (hipStream_t)stream;
    const double* sum = sumsq;
    int64_t nsum = 1;
    if (!sumsq) {
      st = grad_sums(h, s, n, ptr, numel, dtype, work, work_bytes, nsum);
      if (st) return st;
      sum = (const double*)work;
      if (nsum > GFEW || nsum == 0) {                    // into the first place, which only this workgroup reads
        hipLaunchKernelGGL(grad_total_kernel, dim3(1), dim3(1024), 0, s, (const double*)work, nsum, (double*)work);
        nsum = 1;
        st = seq_launched(h, "gradient clip");
        if (st) return st;
      }
    }
    bool first = true;
    st = grad_tables(h, n, ptr, numel, dtype, true, [&](const GradTable& t, unsigned pieces, int64_t) {
      hipLaunchKernelGGL(grad_clip_kernel, dim3(pieces), dim3(256), 0, s, t, sum, (int)nsum, max_norm, first ? norm : nullptr);
      first = false;
      return seq_launched(h, "gradient clip");
    });
    if (st || !first) return st;
    GradTable none;                                      // no elements at all: the norm alone
    none.count = 0;
    hipLaunchKernelGGL(grad_clip_kernel, dim3(1), dim3(256), 0, s, none, sum, (int)nsum, max_norm, norm);
    return seq_launched(h, "gradient clip");
  })
}
