// rgp_seq.h -- what the sequence operators (state-space scan, short convolution, RMS norm, gradient clipping) share: storage types and
// their 32/64-bit arithmetic, 16-byte loads and stores with a scalar path, lane sums, the addressing of (T, batch, features) and packed rows.
#pragma once
#include <math.h>

#include <new>

#include "rgp_common.h"

// Storage type -> arithmetic type.  States, sums and statistics are held in the arithmetic type; only what is written as an activation
// (or its gradient) is rounded to the storage type, once.
template <typename T> struct SeqAcc { typedef float type; };
template <> struct SeqAcc<double> { typedef double type; };

template <typename T, int W = 16 / (int)sizeof(T)>
struct alignas(W * sizeof(T)) SeqVec {
  static constexpr int V = W;
  T e[V];
};

// The same at any address that an element may have: global memory takes 16-byte accesses at element boundaries at 94 % or more of the rate of
// aligned ones (measured on rows of 301 and 2047 two-byte elements), so odd widths and strides need no path of their own (less than a vector does). Where a row is not
// whole vectors the last one is moved back to end with the row: two lanes then write the same values to the elements they share, and only one
// of them may count these in a sum.
template <typename T, int W>
struct __attribute__((packed, aligned(sizeof(T)))) SeqAny {
  T e[W];
};

// V consecutive elements, n of them valid (0..V; the others read as zero / stay as they are in memory).  wide: the address is 16-byte
// aligned.  Both paths touch valid elements only.
template <typename T>
static __device__ __forceinline__ SeqVec<T> seq_load(const T* p, int n, bool wide) {
  SeqVec<T> r;
  if (wide && n == SeqVec<T>::V) return *reinterpret_cast<const SeqVec<T>*>(p);
#pragma unroll
  for (int i = 0; i < SeqVec<T>::V; ++i) r.e[i] = i < n ? p[i] : (T)0;
  return r;
}
template <typename T>
static __device__ __forceinline__ void seq_store(T* p, const SeqVec<T>& v, int n, bool wide) {
  if (wide && n == SeqVec<T>::V) {
    *reinterpret_cast<SeqVec<T>*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < SeqVec<T>::V; ++i)
    if (i < n) p[i] = v.e[i];
}

// ---- lane exchange of either arithmetic type ----------------------------------------------------------------------------------------
template <int CTRL>
static __device__ __forceinline__ float seq_dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
static __device__ __forceinline__ double seq_dpp(double x) { return dpp_f64<CTRL>(x); }

// sum over aligned groups of K lanes (K a power of two up to 16), in every lane of the group, in a fixed order
template <int K, typename A>
static __device__ __forceinline__ A seq_sum(A x) {
  if constexpr (K >= 2) x += seq_dpp<0xB1>(x);
  if constexpr (K >= 4) x += seq_dpp<0x4E>(x);
  if constexpr (K >= 8) x += seq_dpp<0x141>(x);
  if constexpr (K >= 16) x += seq_dpp<0x140>(x);
  return x;
}
template <int K, typename A>
static __device__ __forceinline__ A seq_sum_wide(A x) {       // K up to 64
  x = seq_sum<(K < 16 ? K : 16)>(x);
  if constexpr (K >= 32) x += __shfl_xor(x, 16);
  if constexpr (K >= 64) x += __shfl_xor(x, 32);
  return x;
}

// Two values a, b over the wave -> one: lanes of the lower half hold a[l] + a[l + 32], lanes of the upper half b[l - 32] + b[l]
// (v_permlane32_swap exchanges the upper half of its first register with the lower half of its second).  The 16-lane form does the
// same for neighbouring rows of 16: even rows hold a's sum, odd rows b's.
static __device__ __forceinline__ void seq_swap32(unsigned& a, unsigned& b) {
  auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0]; b = r[1];
}
static __device__ __forceinline__ void seq_swap16(unsigned& a, unsigned& b) {
  auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0]; b = r[1];
}
template <bool HALF>
static __device__ __forceinline__ float seq_fold(float a, float b) {
  unsigned x = __float_as_uint(a), y = __float_as_uint(b);
  if (HALF) seq_swap32(x, y); else seq_swap16(x, y);
  return __uint_as_float(x) + __uint_as_float(y);
}
template <bool HALF>
static __device__ __forceinline__ double seq_fold(double a, double b) {
  unsigned xl = (unsigned)__double2loint(a), xh = (unsigned)__double2hiint(a);
  unsigned yl = (unsigned)__double2loint(b), yh = (unsigned)__double2hiint(b);
  if (HALF) { seq_swap32(xl, yl); seq_swap32(xh, yh); } else { seq_swap16(xl, yl); seq_swap16(xh, yh); }
  return __hiloint2double((int)xh, (int)xl) + __hiloint2double((int)yh, (int)yl);
}
// the same over lanes 8 apart inside rows of 16: lanes with bit 3 clear hold a's sum, the others b's
template <typename A>
static __device__ __forceinline__ A seq_fold8(A a, A b, bool bit3) {
  const A mine = bit3 ? b : a, other = bit3 ? a : b;
  return mine + seq_dpp<0x128>(other);          // row_ror:8
}
template <typename A>
static __device__ __forceinline__ A seq_xor4(A x) { return seq_dpp<0x1B>(seq_dpp<0x141>(x)); }     // lanes 7 - l, then 3 - l in the quad

// ---- elementary functions -----------------------------------------------------------------------------------------------------------
static __device__ __forceinline__ float seq_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
static __device__ __forceinline__ float seq_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
static __device__ __forceinline__ double seq_exp(double x) { return exp(x); }
static __device__ __forceinline__ float seq_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
static __device__ __forceinline__ double seq_rcp(double x) { return 1.0 / x; }
static __device__ __forceinline__ float seq_rsqrt(float x) { return 1.0f / sqrtf(x); }
static __device__ __forceinline__ double seq_rsqrt(double x) { return 1.0 / sqrt(x); }
// exp(-|x|) keeps its relative accuracy for large |x| (the argument is split in two before the exponent of 2 is taken); a NaN counts as -200
static __device__ __forceinline__ float seq_exp_neg(float x) {
  const float a = fmaxf(-fabsf(x), -200.0f);
  const float hi = a * 1.44269504088896341f;
  const float lo = fmaf(a, 1.44269504088896341f, -hi) + a * 1.92596299e-8f;       // log2(e) = 1.44269502... + 1.9259e-8
  const float e = __builtin_amdgcn_exp2f(hi);
  return fmaf(e, lo * 0.693147181f, e);
}
static __device__ __forceinline__ double seq_exp_neg(double x) { return exp(-fabs(x)); }

// log(1 + e) for 0 <= e <= 1 as 2 atanh(s), s = e / (2 + e) <= 1/3: 2 s + 2 s q R(q) with q = s^2 keeps the RELATIVE accuracy of small e, which
// the step size dt = softplus(x) needs (biases put it at 1e-3).  R is the cubic whose largest relative error in the result is smallest over
// q <= 1/9 (4.5e-9, a thirteenth of a rounding; the series of atanh needs three terms more for that).
static __device__ __forceinline__ float seq_log1p01(float e) {
  const float s = e * seq_rcp(2.0f + e), q = s * s;
  float p = 0.14005993677f;
  p = fmaf(p, q, 0.14000902572f);
  p = fmaf(p, q, 0.20010763625f);
  p = fmaf(p, q, 0.33333208143f);
  return fmaf(s * 2.0f * q, p, 2.0f * s);
}
static __device__ __forceinline__ double seq_log1p01(double e) { return log1p(e); }

// softplus(x) and the sigmoid (its derivative); NaN passes through the first, and with dt through everything that the second multiplies
template <typename A>
static __device__ __forceinline__ A seq_softplus(A x, A& sig) {
  const A e = seq_exp_neg(x), big = seq_rcp((A)1 + e);
  sig = x >= (A)0 ? big : e * big;
  return (x < (A)0 ? (A)0 : x) + seq_log1p01(e);
}
// the sigmoid, off by at most |x| half steps relative to its value (what the argument of the exponential rounds by)
template <typename A>
static __device__ __forceinline__ A seq_sigmoid(A x) { return seq_rcp((A)1 + seq_exp(-x)); }

// ---- rows of sequences --------------------------------------------------------------------------------------------------------------
// off == nullptr: n_seq sequences of T steps, step t of sequence s at base + s * sb + t * st; otherwise packed rows, step t of sequence s at
// base + (off[s] + t) * st.  Sequences are cut into blocks of L = 2^lg steps that never cross a sequence; block j of sequence i is number j *
// n_seq + i (neighbours in number are neighbours in memory), or floor(off[i] / L) + i + j for packed rows: those numbers are increasing,
// distinct and below rows / L + n_seq without a table of block counts (some stay empty).  Offsets are clamped to the rows there are, so a wrong
// table cannot make a kernel touch memory outside its tensors.
struct SeqGeo {
  const int64_t* off;
  int64_t T, rows;
  int n_seq, reverse;
};
struct SeqBlock {
  int64_t start, len, seq, j;      // first row (packed) or seq * T, steps of the sequence, sequence, block
  bool ok;
};
static __host__ __device__ inline int64_t seq_blocks(const SeqGeo& g, int lg) {
  return g.off ? (g.rows >> lg) + g.n_seq : (int64_t)g.n_seq * ((g.T + ((int64_t)1 << lg) - 1) >> lg);
}
static __device__ __forceinline__ int64_t seq_off(const SeqGeo& g, int64_t i) {
  int64_t v = g.off[i];
  v = v < 0 ? 0 : v;
  return v > g.rows ? g.rows : v;
}
static __device__ __forceinline__ SeqBlock seq_find(const SeqGeo& g, uint32_t slot, int lg) {       // slot < 2^32, host-checked
  SeqBlock b;
  if (!g.off) {
    const uint32_t q = slot / (uint32_t)g.n_seq;
    b.seq = slot - q * (uint32_t)g.n_seq;
    b.j = q;
    b.start = b.seq * g.T;
    b.len = g.T;
    b.ok = (b.j << lg) < g.T;
    return b;
  }
  int lo = 0, hi = g.n_seq - 1;                         // the last i with floor(off[i] / L) + i <= slot
  while (lo < hi) {
    const int mid = (int)(((unsigned)lo + (unsigned)hi + 1) >> 1);
    if ((seq_off(g, mid) >> lg) + mid <= (int64_t)slot) lo = mid; else hi = mid - 1;
  }
  b.seq = lo;
  b.start = seq_off(g, lo);
  const int64_t end = seq_off(g, lo + 1);
  b.len = end > b.start ? end - b.start : 0;
  b.j = (int64_t)slot - ((b.start >> lg) + lo);
  b.ok = b.j >= 0 && (b.j << lg) < b.len;
  return b;
}
// the number of block j of a sequence
static __device__ __forceinline__ int64_t seq_slot(const SeqGeo& g, int64_t seq, int64_t start, int lg, int64_t j) {
  return g.off ? (start >> lg) + seq + j : j * g.n_seq + seq;
}
#define SEQ_MOST ((int64_t)1 << 40)            // rows: products of sizes stay below 2^63
struct SeqStride { int64_t st, sb; };
template <typename T>
static __device__ __forceinline__ T* seq_row(T* base, const SeqGeo& g, const SeqBlock& b, SeqStride s, int64_t t) {
  const int64_t r = g.reverse ? b.len - 1 - t : t;
  return base + (g.off ? (b.start + r) * s.st : b.seq * s.sb + r * s.st);
}
static __device__ __forceinline__ int64_t seq_row_index(const SeqGeo& g, const SeqBlock& b, int64_t t) {
  const int64_t r = g.reverse ? b.len - 1 - t : t;                 // row number in the contiguous layout of the outputs
  return g.off ? b.start + r : r * g.n_seq + b.seq;
}

// out[i] = sum over p < P of part[p * stride + i], i < n, rounded to type dt; up to five such sums in one launch, each in a fixed order (no
// atomics: results do not depend on timing).  turn > 1: the partials are [turn][n / turn], out is [n / turn][turn].  end: outputs from
// end[0] * per on stay as they are (rows behind the last packed sequence, whose partials nobody wrote).
struct SeqSum { void* part; int64_t P, stride, n; void* out; int dt, turn; int64_t block0; const int64_t* end; int64_t per; };
struct SeqSums {
  SeqSum job[5];
  int count = 0;
  int64_t blocks = 0;              // workgroups' worth of outputs
  void add(void* part, int64_t P, int64_t stride, int64_t n, void* out, int dt, int turn = 1, const int64_t* end = nullptr, int64_t per = 0);
  rgp_status run(rgp_handle h, hipStream_t s, int acc);
};

// the current device is the handle's for the length of a call
struct SeqDevice {
  int before = -1;
  hipError_t e;
  explicit SeqDevice(int want) {
    e = hipGetDevice(&before);
    if (e == hipSuccess && before != want) e = hipSetDevice(want); else before = -1;
  }
  ~SeqDevice() { if (before >= 0) (void)hipSetDevice(before); }
};
#define SEQ_ENTRY(h, what, body)                                                                      \
  if (!(h)) return RGP_ERR_BAD_ARG;                                                                   \
  try {                                                                                               \
    SeqDevice dev_((h)->device);                                                                      \
    if (dev_.e != hipSuccess) return rgp_fail(h, RGP_ERR_HIP, std::string(what ": ") + hipGetErrorString(dev_.e)); \
    body                                                                                              \
  } catch (const std::bad_alloc&) {                                                                   \
    return RGP_ERR_WORKSPACE;                                                                         \
  } catch (...) {                                                                                     \
    return RGP_ERR_HIP;                                                                               \
  }
static inline rgp_status seq_launched(rgp_handle h, const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RGP_OK : rgp_fail(h, RGP_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}
static inline bool seq_overlap(const void* a, const void* b, int64_t bytes) {                // two buffers of that size
  return a && b && (uintptr_t)a < (uintptr_t)b + bytes && (uintptr_t)b < (uintptr_t)a + bytes;
}
static inline int seq_dtype_bytes(int dt) { return dt == RGP_F64 ? 8 : dt == RGP_F32 ? 4 : 2; }
static inline bool seq_aligned(const void* p, int64_t stride, int elem, int v) {        // for vectors of v elements
  return (uintptr_t)p % (v * elem) == 0 && stride % v == 0;
}
