// Optimizer operators over all tensors of a model at once, gfx950: the global gradient norm and the scaling by it, the AdamW step
// with 32-bit moments and the AdamW step with moments held in 8 bits.
//
// Every entry point takes HOST arrays of n device pointers and element counts.  The pointers ride in the kernel arguments (kMax*
// tensors per launch, under 4 KiB): nothing is uploaded, nothing is kept between calls, and a captured graph holds them by value.
// A tensor is a dense run of memory in whatever order its dimensions lie; a workgroup owns one chunk of one tensor and finds it
// from the prefix sums of the tensors' workgroup counts.  All kernels stream: they are bound by HBM, so what they are measured
// against is bytes / bandwidth.
#include <math.h>
#include <stdlib.h>
#include <algorithm>
#include <type_traits>
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxNorm = 160;     // tensors per launch: 8 + 8 + 4 + 4 bytes each
constexpr int kMaxStep = 80;      // 5 * 8 + 4 bytes each
constexpr int kMaxStep8 = 72;     // 6 * 8 + 4
constexpr int kMaxPrepare = 280;  // 8 + 4 + 1, and kMaxRates different rates
constexpr int kMaxRates = 8;
constexpr int kNormWorkgroups = 2048;   // 8 on a CU: all resident at once
constexpr long kMaxNumel = 1L << 33;   // element / 8 fits the 32-bit hash input, a tensor's workgroups one launch
constexpr long kMaxWorkgroups = (1L << 24) - 1;   // a launch holds less than 2^32 work-items

enum { kF32 = 0, kBf16 = 1, kF16 = 2 };

// ------------------------------------------------------------------------------------------------ element types
// Vector accesses at ELEMENT alignment: views of a flat bucket start anywhere, and the memory pipe takes wide accesses at any
// element boundary (a line that is cut costs a second request, nothing else).  They are non-temporal: every byte of a step is used once,
// and lines that are not kept leave the memory-side cache to the gradients that the norm has just read (Res-101's clipped step 350 -> 316
// us).  Those alone are kept (KEEP) where there is something left of them when the next launch reads them: see kKeepBytes.
template <typename T, int N> struct Wide {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <typename T, int N, bool KEEP = false> __device__ __forceinline__ void load_f32(const T* p, float (&x)[N]) {
  typedef typename Wide<T, N>::type V;
  const V v = KEEP ? *reinterpret_cast<const V*>(p) : __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = (float)v[i];
}
template <typename T, int N> __device__ __forceinline__ void store_f32(T* p, const float (&x)[N]) {
  typedef typename Wide<T, N>::type V;
  V v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (T)x[i];   // round to nearest even
  __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
}

// index of the tensor that owns this workgroup: block0[0 .. n] are prefix sums in the kernel arguments.  The lanes compare 64
// entries at a time (one vector load each) instead of walking them by dependent scalar loads.
__device__ __forceinline__ int owner(const int* block0, int n, int b) {
  const int lane = threadIdx.x & 63;
  int i = 0;
  for (int k = 0; k < n; k += 64) {
    const bool before = k + lane < n && block0[k + lane] <= b;
    i += __popcll(__ballot(before));
  }
  return __builtin_amdgcn_readfirstlane(i) - 1;
}

// ------------------------------------------------------------------------------------------------ gradient norm
// norm = sqrt(sum of all g^2) and the factor min(1, max_norm / (norm + 1e-6)).  Squares and sums in 64 bits: no overflow for any
// fp32 gradient, and the order of the partial sums (fixed: chunks, then workgroups in index order) does not show in 32 bits.
// Gradients of up to kKeepBytes in all are read into the caches, for the launch that reads them again; larger ones pass by.  Clipping of
// fp32 (us, kept / passing by): 96 MB 49 / 54, 192 MB 93 / 105, 383 MB 194 / 211, 768 MB 404 / 415, 1151 MB 617 / 623; the norm alone of 2.4 GB
// 422 / 380 (6.4 TB/s).  Res-101's clipped step: 272 / 297.
constexpr long kKeepBytes = 1L << 30;
struct NormTable {
  const void* g[kMaxNorm];
  long numel[kMaxNorm];
  int block0[kMaxNorm];
  int dtype[kMaxNorm];
  long chunk;          // elements per workgroup, a multiple of kThreads * 8
  int n, keep;
};

template <typename T, int N, bool KEEP> __device__ __forceinline__ double square_sum(const T* g, long e0, long e1) {
  constexpr int kFly = 4;   // vectors on their way per thread
  double acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.0;
  long e = e0 + (long)threadIdx.x * N;
  for (; e + (kFly - 1) * kThreads * N + N <= e1; e += kFly * kThreads * N) {
    float x[kFly][N];
#pragma unroll
    for (int u = 0; u < kFly; ++u) load_f32<T, N, KEEP>(g + e + u * kThreads * N, x[u]);
#pragma unroll
    for (int u = 0; u < kFly; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = __builtin_fma((double)x[u][i], (double)x[u][i], acc[i]);
  }
  for (; e + N <= e1; e += kThreads * N) {
    float x[N];
    load_f32<T, N, KEEP>(g + e, x);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = __builtin_fma((double)x[i], (double)x[i], acc[i]);
  }
  for (; e < e1; ++e) {   // at most N - 1 elements, of one thread
    const double x = (double)(float)g[e];
    acc[0] = __builtin_fma(x, x, acc[0]);
  }
#pragma unroll
  for (int s = 1; s < N; s *= 2)
#pragma unroll
    for (int i = 0; i + s < N; i += 2 * s) acc[i] += acc[i + s];
  return acc[0];
}

template <int NW> __device__ __forceinline__ double workgroup_sum(double x) {
  __shared__ double part[NW];
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) x += __shfl_xor(x, s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) t += part[i];
  return t;
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(NormTable tab, double* __restrict__ partial) {
  const int i = owner(tab.block0, tab.n, blockIdx.x);
  const long e0 = (long)((int)blockIdx.x - tab.block0[i]) * tab.chunk;
  const long e1 = e0 + tab.chunk < tab.numel[i] ? e0 + tab.chunk : tab.numel[i];
  const auto sum = [&](auto keep) {
    constexpr bool KEEP = decltype(keep)::value;
    if (tab.dtype[i] == kF32) return square_sum<float, 4, KEEP>(static_cast<const float*>(tab.g[i]), e0, e1);
    if (tab.dtype[i] == kBf16) return square_sum<__bf16, 8, KEEP>(static_cast<const __bf16*>(tab.g[i]), e0, e1);
    return square_sum<_Float16, 8, KEEP>(static_cast<const _Float16*>(tab.g[i]), e0, e1);
  };
  double s = tab.keep ? sum(std::true_type{}) : sum(std::false_type{});
  s = workgroup_sum<kThreads / 64>(s);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The partial sums of all workgroups, in index order within a thread, then over the threads: norm and factor, in every thread.
constexpr int kFinish = 512;   // threads of the launches that do nothing else at length
template <int NT> __device__ __forceinline__ float2 finish_norm(const double* __restrict__ partial, int n, double max_norm) {
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += NT) s += partial[i];
  s = workgroup_sum<NT / 64>(s);
  const double norm = sqrt(s);
  // (an infinite limit asks for the norm alone; a norm that is not a number stays one in the factor, an infinite one gives 0)
  const double f = max_norm / (norm + 1e-6);
  return make_float2((float)norm, isinf(max_norm) ? 1.f : f < 1.0 || f != f ? (float)f : 1.f);
}

struct NormPart {
  const double* partial;   // NULL: the norm is not this call's to compute
  int n;
  double max_norm;
};

__global__ __launch_bounds__(kFinish) void grad_norm_finish_kernel(const double* __restrict__ partial, int n, double max_norm,
                                                                   float* __restrict__ out) {
  const float2 r = finish_norm<kFinish>(partial, n, max_norm);
  if (threadIdx.x == 0) { out[0] = r.x; out[1] = r.y; }
}

// ------------------------------------------------------------------------------------------------ scaling
struct ScaleTable {
  void* g[kMaxNorm];
  long numel[kMaxNorm];
  int block0[kMaxNorm];
  int dtype[kMaxNorm];
  long chunk;
  int n;
};

template <typename T, int N> __device__ __forceinline__ void scale_run(T* g, long e0, long e1, float f) {
  constexpr int kFly = 4;
  long e = e0 + (long)threadIdx.x * N;
  for (; e + (kFly - 1) * kThreads * N + N <= e1; e += kFly * kThreads * N) {
    float x[kFly][N];
#pragma unroll
    for (int u = 0; u < kFly; ++u) load_f32<T, N>(g + e + u * kThreads * N, x[u]);
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[u][i] *= f;
      store_f32<T, N>(g + e + u * kThreads * N, x[u]);
    }
  }
  for (; e + N <= e1; e += kThreads * N) {
    float x[N];
    load_f32<T, N>(g + e, x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= f;
    store_f32<T, N>(g + e, x);
  }
  for (; e < e1; ++e) g[e] = (T)((float)g[e] * f);
}

// Every workgroup joins the partial sums itself -- at most 2048 and one per tensor, 8 bytes each: 17 KiB of L2 for Res-101 -- because a
// launch of one workgroup in between would keep the device waiting for 7 us.  The reading grows with the square of the number of tensors:
// 10 000 of 500 elements are 10 000 workgroups that read 80 KB each (norm alone 591 us, with the scaling 842; 1000 of them 65 / 94).
__global__ __launch_bounds__(kThreads) void grad_clip_kernel(ScaleTable tab, NormPart part, float* __restrict__ out) {
  const float2 r = finish_norm<kThreads>(part.partial, part.n, part.max_norm);
  if (out && blockIdx.x == 0 && threadIdx.x == 0) { out[0] = r.x; out[1] = r.y; }
  const float f = r.y;
  if (f == 1.f) return;   // within the limit: the gradients are neither read nor written
  const int i = owner(tab.block0, tab.n, blockIdx.x);
  const long e0 = (long)((int)blockIdx.x - tab.block0[i]) * tab.chunk;
  const long e1 = e0 + tab.chunk < tab.numel[i] ? e0 + tab.chunk : tab.numel[i];
  if (tab.dtype[i] == kF32) scale_run<float, 4>(static_cast<float*>(tab.g[i]), e0, e1, f);
  else if (tab.dtype[i] == kBf16) scale_run<__bf16, 8>(static_cast<__bf16*>(tab.g[i]), e0, e1, f);
  else scale_run<_Float16, 8>(static_cast<_Float16*>(tab.g[i]), e0, e1, f);
}

// ------------------------------------------------------------------------------------------------ what a step needs per tensor
// One thread per tensor: t <- t + 1 in the tensor's step counter, and the step's factors in 64 bits, rounded once:
// keep = 1 - lr * decay, size = lr / (1 - beta1^t), root = 1 / sqrt(1 - beta2^t); for 8-bit moments the key of its rounding terms.
// Where the call clips, the same workgroup joins the norm's partial sums first (one launch less than a kernel of its own); a call of more
// than kMaxPrepare tensors or kMaxRates rates has several such launches, and each joins them again.
// The counters live on the device, so a captured step counts on with every replay.
struct Rate {
  double lr;
  const float* lr_device;   // learning rate in device memory (a schedule under a captured graph), or NULL
  double decay;
};
struct PrepareTable {
  float* step[kMaxPrepare];
  Rate rate[kMaxRates];
  unsigned id[kMaxPrepare];
  unsigned char which[kMaxPrepare];   // entry of rate
  int n;
  unsigned seed;
  double beta1, beta2;
};
struct Factors {
  float keep, size, root;
  unsigned key;
};

__host__ __device__ __forceinline__ unsigned mix32(unsigned x) {   // multiplicative (golden ratio, sqrt 2) with folded shifts
  x = (x ^ (x >> 16)) * 0x9E3779B9u;
  x = (x ^ (x >> 15)) * 0x6A09E667u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ bool skipped(const float* clip, int skip_nonfinite) {
  return skip_nonfinite && !isfinite(clip[0]);
}

__global__ __launch_bounds__(kFinish) void adamw_prepare_kernel(PrepareTable tab, NormPart part, float* __restrict__ clip, int skip_nonfinite,
                                                                Factors* __restrict__ factors) {
  bool skip = false;
  if (part.partial) {
    const float2 r = finish_norm<kFinish>(part.partial, part.n, part.max_norm);
    if (threadIdx.x == 0) { clip[0] = r.x; clip[1] = r.y; }
    skip = skip_nonfinite && !isfinite(r.x);
  } else if (clip) {
    skip = skipped(clip, skip_nonfinite);
  }
  const int i = threadIdx.x;
  if (i >= tab.n || skip) return;
  const Rate rate = tab.rate[tab.which[i]];
  const float t = *tab.step[i] + 1.f;   // (exact up to 2^24 steps)
  *tab.step[i] = t;
  const double lr = rate.lr_device ? (double)*rate.lr_device : rate.lr;
  Factors f;
  f.keep = (float)(1.0 - lr * rate.decay);
  f.size = (float)(lr / (1.0 - pow(tab.beta1, (double)t)));
  f.root = (float)(1.0 / sqrt(1.0 - pow(tab.beta2, (double)t)));
  f.key = mix32(mix32(tab.seed + 0x9E3779B9u * (tab.id[i] + 1u)) + (unsigned)t);
  factors[i] = f;
}

struct Consts {
  float beta1, one_beta1, beta2, one_beta2, eps;
};

// m <- beta1 m + (1 - beta1) g;  v <- beta2 v + (1 - beta2) g^2;  p <- keep p - size * m / (root sqrt(v) + eps)
// The step with 8-bit moments has about as many instructions as it has bytes: EXACT = false takes the quotient from v_sqrt and v_rcp, each
// off by one unit in the last place (2^-23 of the value) at most, and a product, in place of the exactly rounded sequences (302 M bf16: step
// and unpacking 985 -> 884 us); the tests' bounds count 2^-23 for each.  v_sqrt takes a v below 2^-126 for 0: beside
// eps >= 2^-39 / sqrt(1 - beta2), which is 2^-39 root or more, that is below 2^-24 of the denominator.  A smaller eps takes the exact
// sequences, which are built for one block per wave only.
template <bool EXACT> __device__ __forceinline__ void adamw_element(float& p, float g, float& m, float& v, const Consts& k, const Factors& f) {
  m = m * k.beta1 + g * k.one_beta1;
  v = v * k.beta2 + (g * g) * k.one_beta2;
  const float q = EXACT ? m / (sqrtf(v) * f.root + k.eps) : m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) * f.root + k.eps);
  p = p * f.keep - q * f.size;
}

// ------------------------------------------------------------------------------------------------ AdamW, 32-bit moments
struct StepTable {
  void* p[kMaxStep];
  const void* g[kMaxStep];
  float* m[kMaxStep];
  float* v[kMaxStep];
  long numel[kMaxStep];
  int block0[kMaxStep];
  int n;
};
// A thread takes four neighbours and nothing else: a wave's accesses are runs of 1 KiB of fp32, and the workgroups in flight walk one
// compact window of each buffer.  Measured on MI355X, clipped Res-101 fp32 / 604 M bf16, us: one group of four 297 / 2165 (6.1 TB/s);
// two groups, loads first, 299 / 2345; four 304 / 2299; four, each loaded behind the one before it, 324 / 2408.  Eight neighbours of
// bf16 (one 16-byte access, two of the moments 32 bytes apart): 2560.
constexpr int kStepElems = kThreads * 4;   // per workgroup
// Elements in front of the first 128-byte boundary of m: the first workgroup takes them one by one, so that the runs of a view into a
// flat buffer -- whose four tensors usually start alike -- do not cut lines.
__host__ __device__ __forceinline__ int step_head(const float* m, long numel) {
  const long h = (32 - (long)((reinterpret_cast<uintptr_t>(m) >> 2) & 31)) & 31;
  return (int)(h < numel ? h : numel);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void adamw_step_kernel(StepTable tab, const Factors* __restrict__ factors,
                                                              const float* __restrict__ clip, int skip_nonfinite, Consts k) {
  constexpr int N = 4;
  const int i = owner(tab.block0, tab.n, blockIdx.x);
  if (clip && skipped(clip, skip_nonfinite)) return;
  const float c = clip ? clip[1] : 1.f;
  const Factors f = factors[i];
  T* p = static_cast<T*>(tab.p[i]);
  const T* g = static_cast<const T*>(tab.g[i]);
  float* m = tab.m[i];
  float* v = tab.v[i];
  const long numel = tab.numel[i];
  const int head = step_head(m, numel);
  const int block = (int)blockIdx.x - tab.block0[i];
  const auto single = [&](long q) {
    float xp = (float)p[q], xm = m[q], xv = v[q];
    adamw_element<true>(xp, (float)g[q] * c, xm, xv, k, f);
    p[q] = (T)xp; m[q] = xm; v[q] = xv;
  };
  if (block == 0 && (int)threadIdx.x < head) single(threadIdx.x);
  const long e = head + (long)block * kStepElems + (long)threadIdx.x * N;
  if (e + N <= numel) {
    float xp[N], xg[N], xm[N], xv[N];
    load_f32<T, N>(g + e, xg);
    load_f32<float, N>(m + e, xm);
    load_f32<float, N>(v + e, xv);
    load_f32<T, N>(p + e, xp);
#pragma unroll
    for (int j = 0; j < N; ++j) adamw_element<true>(xp[j], xg[j] * c, xm[j], xv[j], k, f);
    store_f32<T, N>(p + e, xp);
    store_f32<float, N>(m + e, xm);
    store_f32<float, N>(v + e, xv);
  } else {
    for (long r = e; r < numel; ++r) single(r);   // the end of a tensor
  }
}

// ------------------------------------------------------------------------------------------------ moments in 8 bits
// The upper 12 bits of a non-negative fp32 (8 of the exponent, 3 of the mantissa) number a fixed grid of LEVELS, eight for each
// power of two.  256 elements in memory order share a base per moment; a code counts levels from it, code 0 is zero:
//   m: sign and 7 bits, levels base + 1 .. base + 126 (15.7 powers of two below the block's largest; what lies lower is 0)
//   v: 8 bits, levels base + 1 .. base + 254 (31.7 powers of two, the same span in |g|); a v that is not 0 keeps code 1 at least,
//      for a zero would turn the next m / sqrt(v) into m / eps.
// Why a fixed grid with dithered rounding: beta2 = 0.999 moves v by 0.1 % a step, the levels are 12.5 % apart, and to the nearest
// v would never move again.  x + u with u uniform below one spacing, cut off, is right on average; and since the grid does not
// move with the base, a value that does not change is not rounded again.
// Infinity and NaN stay in their element: the base counts finite levels only, bit 14 of the base says that the block holds such
// values, and the top code (127 / 255, which finite values never reach) is NaN there.
constexpr int kBlock = 256;
constexpr int kNanFlag = 0x4000;
constexpr int kInfLevel = 0x7F8;   // level of infinity; NaN lies above

__device__ __forceinline__ float decode_m(unsigned code, int base) {
  const unsigned level = code & 127u;
  unsigned bits = level ? (level + (unsigned)(base & 0x3FFF)) << 20 : 0u;
  if ((base & kNanFlag) && level == 127u) bits = 0x7FC00000u;
  return __uint_as_float(bits | (code & 128u) << 24);
}
__device__ __forceinline__ float decode_v(unsigned code, int base) {
  unsigned bits = code ? (code + (unsigned)(base & 0x3FFF)) << 20 : 0u;
  if ((base & kNanFlag) && code == 255u) bits = 0x7FC00000u;
  return __uint_as_float(bits);
}
// four codes each; base: the block's two, the same for the whole wave
__device__ __forceinline__ void decode4(unsigned cm, unsigned cv, int base, float (&m)[4], float (&v)[4]) {
  const unsigned bm = (unsigned)base & 0x3FFFu, bv = ((unsigned)base >> 16) & 0x3FFFu;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned a = (cm >> (8 * j)) & 127u, b = (cv >> (8 * j)) & 255u, sign = (cm << (24 - 8 * j)) & 0x80000000u;
    m[j] = __uint_as_float((a ? (a + bm) << 20 : 0u) | sign);
    v[j] = __uint_as_float(b ? (b + bv) << 20 : 0u);
  }
  if (__builtin_expect(base & (kNanFlag | kNanFlag << 16), 0)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = decode_m((cm >> (8 * j)) & 255u, base & 0xFFFF);
      v[j] = decode_v((cv >> (8 * j)) & 255u, base >> 16);
    }
  }
}

struct Step8Table {
  void* p[kMaxStep8];
  const void* g[kMaxStep8];
  unsigned char* m[kMaxStep8];
  unsigned char* v[kMaxStep8];
  int* base[kMaxStep8];   // per block: m in the low half, v in the high one
  long numel[kMaxStep8];
  int block0[kMaxStep8];
  int n;
};
// Blocks that a wave holds at a time: four share what a workgroup does first (finding its tensor, pointers, factors), which costs
// against the kernel's own instructions; a launch that would give the CUs less than four such workgroups each takes one block per wave
// instead.  302 M bf16, step and unpacking: four 884 us, two 905, one 1190; 1.1 M fp32: step 9.0 / 7.3 / 6.8 us, unpacking 5.5 / 5.1 / 5.3;
// 72 odd tensors of 1.2 M fp16 together: 10.4 / 7.5 / 6.3 us, unpacking 8.1 / 5.9 / 4.9.
template <int WB> struct Wave8 {
  static constexpr int kElems = kThreads / 64 * WB * kBlock;   // per workgroup
};

__device__ __forceinline__ unsigned max_halves(unsigned a, unsigned b) {
  typedef unsigned short Pair __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(Pair, a), __builtin_bit_cast(Pair, b)));
}
// both halves' maxima over the wave, as a scalar: within 16 lanes by lane swaps, then row by row into the last lane
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned max_dpp(unsigned x) {
  return max_halves(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ unsigned wave_max_halves(unsigned x) {
  x = max_dpp<0xB1, 0xF>(x);    // quad_perm 1 0 3 2
  x = max_dpp<0x4E, 0xF>(x);    // quad_perm 2 3 0 1
  x = max_dpp<0x141, 0xF>(x);   // row_half_mirror
  x = max_dpp<0x140, 0xF>(x);   // row_mirror
  x = max_dpp<0x142, 0xA>(x);   // row_bcast15 into rows 1, 3
  x = max_dpp<0x143, 0xC>(x);   // row_bcast31 into rows 2, 3
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}

// The levels of four elements with their dither (at most 0x800), m in the low half, v in the high one.  r: the first element's hash
// product, dr: its step to the next.
__device__ __forceinline__ void levels4(const float (&m)[4], const float (&v)[4], unsigned r, unsigned dr, unsigned (&q)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j, r += dr) {
    const unsigned um = ((r >> 12) & 0xFFFF0u) | 8u, uv = ((r << 4) & 0xFFFF0u) | 8u;
    const unsigned qm = ((__float_as_uint(m[j]) & 0x7FFFFFFFu) + um) >> 20, qv = ((__float_as_uint(v[j]) & 0x7FFFFFFFu) + uv) >> 20;
    q[j] = qm | qv << 16;
  }
}

// Bases of the block from the wave's largest levels, and the four elements' codes.
__device__ __forceinline__ int codes4(const float (&m)[4], const float (&v)[4], const unsigned (&q)[4], unsigned& cm, unsigned& cv) {
  unsigned top = wave_max_halves(max_halves(max_halves(q[0], q[1]), max_halves(q[2], q[3])));
  int flag = 0;
  if (__builtin_expect((top & 0xFFFFu) >= (unsigned)kInfLevel || (top >> 16) >= (unsigned)kInfLevel, 0)) {   // uniform, rare
    flag = kNanFlag;
    unsigned t = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      t = max_halves(t, ((q[j] & 0xFFFFu) < (unsigned)kInfLevel ? q[j] & 0xFFFFu : 0u) | ((q[j] >> 16) < (unsigned)kInfLevel ? q[j] & 0xFFFF0000u : 0u));
    top = wave_max_halves(t);
  }
  const int bm = max((int)(top & 0xFFFFu) - 126, 0), bv = max((int)(top >> 16) - 254, 0);
  cm = cv = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int qm = (int)(q[j] & 0xFFFFu), qv = (int)(q[j] >> 16);
    int lm = max(qm - bm, 0), lv = max(qv - bv, (int)min(__float_as_uint(v[j]), 1u));
    if (flag) {
      lm = qm >= kInfLevel ? 127 : lm;
      lv = qv >= kInfLevel ? 255 : lv;
    }
    cm |= ((unsigned)lm | ((__float_as_uint(m[j]) >> 24) & 128u)) << (8 * j);
    cv |= (unsigned)lv << (8 * j);
  }
  return bm | bv << 16 | flag | flag << 16;
}

typedef unsigned Word __attribute__((aligned(1)));   // four codes, at any address

// Codes of up to kKeepCodes bytes in a call are left in the caches for whoever reads them next (KEEP), more of them pass by: as lines that
// wait to be written back they would only be in the way.  The step itself takes as long either way; unpacking behind it, us, kept /
// passing by: 110 MB of codes 53 / 62, 604 MB 346 / 295.
constexpr long kKeepCodes = 256L << 20;

// A lane has four neighbours of each of the wave's blocks, so that all of the wave's accesses are runs of memory (1 KiB of fp32
// parameters, 256 bytes of codes), and all loads are on their way before the first is used.
template <typename T, int WB, bool EXACT, bool KEEP>
__global__ __launch_bounds__(kThreads) void adamw8_step_kernel(Step8Table tab, const Factors* __restrict__ factors,
                                                               const float* __restrict__ clip, int skip_nonfinite, Consts k) {
  const int i = owner(tab.block0, tab.n, blockIdx.x);
  if (clip && skipped(clip, skip_nonfinite)) return;
  const float c = clip ? clip[1] : 1.f;
  const Factors f = factors[i];
  T* p = static_cast<T*>(tab.p[i]);
  const T* g = static_cast<const T*>(tab.g[i]);
  unsigned char* cm = tab.m[i];
  unsigned char* cv = tab.v[i];
  const long numel = tab.numel[i];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const long e0 = (long)((int)blockIdx.x - tab.block0[i]) * Wave8<WB>::kElems + wave * (WB * kBlock);
  if (e0 >= numel) return;
  int* base = tab.base[i] + e0 / kBlock;
  const long e = e0 + lane * 4;
  if (e0 + WB * kBlock <= numel) {
    float xp[WB][4], xg[WB][4];
    unsigned um[WB], uv[WB];
    int b[WB];
#pragma unroll
    for (int u = 0; u < WB; ++u) {
      const Word* wm = reinterpret_cast<const Word*>(cm + e + u * kBlock);
      const Word* wv = reinterpret_cast<const Word*>(cv + e + u * kBlock);
      um[u] = KEEP ? *wm : __builtin_nontemporal_load(wm);
      uv[u] = KEEP ? *wv : __builtin_nontemporal_load(wv);
      load_f32<T, 4>(g + e + u * kBlock, xg[u]);
      load_f32<T, 4>(p + e + u * kBlock, xp[u]);
      b[u] = base[u];
    }
#pragma unroll
    for (int u = 0; u < WB; ++u) {
      float xm[4], xv[4];
      decode4(um[u], uv[u], b[u], xm, xv);
#pragma unroll
      for (int j = 0; j < 4; ++j) adamw_element<EXACT>(xp[u][j], xg[u][j] * c, xm[j], xv[j], k, f);
      store_f32<T, 4>(p + e + u * kBlock, xp[u]);
      const unsigned h = mix32((unsigned)((e + u * kBlock) >> 3) ^ f.key);
      unsigned q[4];
      levels4(xm, xv, (lane & 1) ? h * 9u : h, 2u * h, q);
      unsigned wm, wv;
      b[u] = codes4(xm, xv, q, wm, wv);
      if (KEEP) {
        *reinterpret_cast<Word*>(cm + e + u * kBlock) = wm;
        *reinterpret_cast<Word*>(cv + e + u * kBlock) = wv;
      } else {
        __builtin_nontemporal_store(wm, reinterpret_cast<Word*>(cm + e + u * kBlock));
        __builtin_nontemporal_store(wv, reinterpret_cast<Word*>(cv + e + u * kBlock));
      }
    }
    if (lane == 0) {
#pragma unroll
      for (int u = 0; u < WB; ++u) base[u] = b[u];
    }
    return;
  }
  // the end of a tensor: elements behind it count as zeros of the block
  for (int u = 0; u < WB && e0 + u * kBlock < numel; ++u) {
    const long e1 = e + u * kBlock;
    const int b = base[u];
    float xm[4], xv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      xm[j] = xv[j] = 0.f;
      if (e1 + j < numel) {
        xm[j] = decode_m(cm[e1 + j], b & 0xFFFF);
        xv[j] = decode_v(cv[e1 + j], b >> 16);
        float xp = (float)p[e1 + j];
        adamw_element<EXACT>(xp, (float)g[e1 + j] * c, xm[j], xv[j], k, f);
        p[e1 + j] = (T)xp;
      }
    }
    const unsigned h = mix32((unsigned)(e1 >> 3) ^ f.key);
    unsigned q[4];
    levels4(xm, xv, (lane & 1) ? h * 9u : h, 2u * h, q);
    unsigned wm, wv;
    const int nb = codes4(xm, xv, q, wm, wv);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e1 + j < numel) {
        cm[e1 + j] = (unsigned char)(wm >> (8 * j));
        cv[e1 + j] = (unsigned char)(wv >> (8 * j));
      }
    if (lane == 0) base[u] = nb;
  }
}

struct UnpackTable {
  const unsigned char* m[kMaxStep8];
  const unsigned char* v[kMaxStep8];
  const int* base[kMaxStep8];
  void* out_m[kMaxStep8];
  void* out_v[kMaxStep8];
  long numel[kMaxStep8];
  int block0[kMaxStep8];
  int n;
};

template <typename T, int WB> __global__ __launch_bounds__(kThreads) void unpack_moments_kernel(UnpackTable tab) {
  const int i = owner(tab.block0, tab.n, blockIdx.x);
  const long numel = tab.numel[i];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const long e0 = (long)((int)blockIdx.x - tab.block0[i]) * Wave8<WB>::kElems + wave * (WB * kBlock);
  if (e0 >= numel) return;
  const int* base = tab.base[i] + e0 / kBlock;
  const long e = e0 + lane * 4;
  const unsigned char* cm = tab.m[i] + e;
  const unsigned char* cv = tab.v[i] + e;
  T* out_m = static_cast<T*>(tab.out_m[i]) + e;
  T* out_v = static_cast<T*>(tab.out_v[i]) + e;
  if (e0 + WB * kBlock <= numel) {
    unsigned um[WB], uv[WB];
    int b[WB];
#pragma unroll
    for (int u = 0; u < WB; ++u) {
      um[u] = *reinterpret_cast<const Word*>(cm + u * kBlock);
      uv[u] = *reinterpret_cast<const Word*>(cv + u * kBlock);
      b[u] = base[u];
    }
#pragma unroll
    for (int u = 0; u < WB; ++u) {
      float xm[4], xv[4];
      decode4(um[u], uv[u], b[u], xm, xv);
      store_f32<T, 4>(out_m + u * kBlock, xm);
      store_f32<T, 4>(out_v + u * kBlock, xv);
    }
    return;
  }
  for (int u = 0; u < WB && e0 + u * kBlock < numel; ++u)
    for (int j = 0; j < 4 && e + u * kBlock + j < numel; ++j) {
      out_m[u * kBlock + j] = (T)decode_m(cm[u * kBlock + j], base[u] & 0xFFFF);
      out_v[u * kBlock + j] = (T)decode_v(cv[u * kBlock + j], base[u] >> 16);
    }
}

// ------------------------------------------------------------------------------------------------ host side
// (kernel arguments are 4 KiB at most; beside a table a launch passes under 100 bytes)
static_assert(sizeof(NormTable) <= 3968 && sizeof(ScaleTable) <= 3968 && sizeof(PrepareTable) <= 3968 && sizeof(StepTable) <= 3968 &&
              sizeof(Step8Table) <= 3968 && sizeof(UnpackTable) <= 3968, "tensors per launch");

int type_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

// Buffers that a call writes must not meet anything else that it reads or writes (the same parameter twice, a moment that is a
// view of another, a shared step counter, a learning rate inside a parameter): the workgroups run in no order.
struct Spans {
  struct Span {
    uintptr_t lo, hi;   // twice the addresses; hi's lowest bit says "written"
  };
  Span* s = nullptr;
  long n = 0;
  explicit Spans(long most) { s = static_cast<Span*>(malloc((size_t)(most > 0 ? most : 1) * sizeof(Span))); }
  ~Spans() { free(s); }
  Spans(const Spans&) = delete;
  void add(const void* p, long bytes, bool written) {
    if (bytes <= 0) return;
    s[n].lo = reinterpret_cast<uintptr_t>(p) * 2;
    s[n].hi = (reinterpret_cast<uintptr_t>(p) + (uintptr_t)bytes) * 2 + (written ? 1 : 0);
    ++n;
  }
  bool clash() {   // (the 1505 spans of 301 tensors: 7 us)
    std::sort(s, s + n, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    uintptr_t any = 0, written = 0;
    for (long i = 0; i < n; ++i) {
      const uintptr_t lo = s[i].lo, hi = s[i].hi & ~(uintptr_t)1;
      const bool w = s[i].hi & 1;
      if (lo < written || (w && lo < any)) return true;
      if (hi > any) any = hi;
      if (w && hi > written) written = hi;
    }
    return false;
  }
};

// how many of the next tensors go into one launch: `most` at most, and fewer where their workgroups (of 1024 elements or more) would be
// more than a launch may have
int fit(int n, int most, const long* numel) {
  long workgroups = 0;
  int k = 0;
  for (; k < n && k < most; ++k) {
    workgroups += numel[k] / 1024 + 2;
    if (k > 0 && workgroups > kMaxWorkgroups) break;
  }
  return k;
}

bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

long norm_chunk(int n, const long* numel) {
  long total = 0;
  for (int i = 0; i < n; ++i) total += numel[i];
  const long unit = kThreads * 8;
  long chunk = (total / kNormWorkgroups + unit - 1) / unit * unit;
  return chunk < 2 * unit ? 2 * unit : chunk;
}

int check_grads(const char* what, int n, const void* const* grads, const long* numel, const int* dtypes) {
  DTT_REQUIRE(n >= 0 && (n == 0 || (grads && numel && dtypes)), "%s: null pointer", what);
  for (int i = 0; i < n; ++i) {
    DTT_REQUIRE(numel[i] >= 0 && numel[i] <= kMaxNumel, "%s: tensor %d: bad element count", what, i);
    DTT_REQUIRE(dtypes[i] >= kF32 && dtypes[i] <= kF16, "%s: tensor %d: unknown element type %d", what, i, dtypes[i]);
    DTT_REQUIRE(numel[i] == 0 || (grads[i] && aligned_to(grads[i], type_bytes(dtypes[i]))), "%s: tensor %d: null or unaligned pointer", what, i);
  }
  return 1;
}

}  // namespace

extern "C" size_t dtt_grad_norm_workspace_bytes(int n, const long* numel) {
  if (n <= 0 || !numel) return sizeof(double);
  const long chunk = norm_chunk(n, numel);
  long blocks = 0;
  for (int i = 0; i < n; ++i) blocks += numel[i] > 0 ? (numel[i] + chunk - 1) / chunk : 0;
  return (size_t)(blocks > 0 ? blocks : 1) * sizeof(double);
}

namespace {

// the partial sums of all tensors; returns their number, -1 after a failed launch.  dtypes: one per tensor, or NULL (all `dtype`)
int norm_partials(int n, const void* const* grads, const long* numel, const int* dtypes, int dtype, double* partial, hipStream_t stream) {
  const long chunk = n > 0 ? norm_chunk(n, numel) : 1;
  int blocks = 0;
  long bytes = 0;
  for (int i = 0; i < n; ++i) bytes += numel[i] * type_bytes(dtypes ? dtypes[i] : dtype);
  NormTable tab;
  tab.keep = bytes <= kKeepBytes;
  for (int i = 0; i < n;) {
    tab.n = 0; tab.chunk = chunk;
    int here = 0;
    for (; i < n && tab.n < kMaxNorm; ++i) {
      if (numel[i] == 0) continue;
      const int j = tab.n++;
      tab.g[j] = grads[i]; tab.numel[j] = numel[i]; tab.dtype[j] = dtypes ? dtypes[i] : dtype; tab.block0[j] = here;
      here += (int)((numel[i] + chunk - 1) / chunk);
    }
    if (here == 0) break;
    hipLaunchKernelGGL(grad_norm_kernel, dim3((unsigned)here), dim3(kThreads), 0, stream, tab, partial + blocks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
      dtt_set_error("grad_norm_kernel: launch failed: %s", hipGetErrorString(e));
      return -1;
    }
    blocks += here;
  }
  return blocks;
}

}  // namespace

extern "C" int dtt_grad_norm(int n, const void* const* grads, const long* numel, const int* dtypes, double max_norm, float* out,
                             void* workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (!check_grads("grad_norm", n, grads, numel, dtypes)) return 0;
  DTT_REQUIRE(out && aligned_to(out, 4) && workspace && aligned_to(workspace, 8), "grad_norm: null or unaligned pointer");
  DTT_REQUIRE(max_norm >= 0.0, "grad_norm: max_norm must not be negative");
  const size_t need = dtt_grad_norm_workspace_bytes(n, numel);
  DTT_REQUIRE(workspace_bytes >= need, "grad_norm: workspace too small");
  Spans spans(n + 2L);
  DTT_REQUIRE(spans.s, "grad_norm: out of host memory");
  for (int i = 0; i < n; ++i) spans.add(grads[i], numel[i] * type_bytes(dtypes[i]), false);
  spans.add(out, 8, true);
  spans.add(workspace, (long)need, true);
  DTT_REQUIRE(!spans.clash(), "grad_norm: the result, the workspace or a gradient share memory");
  double* partial = static_cast<double*>(workspace);
  dtt_prof_begin("grad_norm", stream);
  const int blocks = norm_partials(n, grads, numel, dtypes, 0, partial, stream);
  if (blocks < 0) return 0;
  hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(kFinish), 0, stream, partial, blocks, max_norm, out);
  DTT_CHECK_LAUNCH("grad_norm_finish_kernel");
  dtt_prof_end("grad_norm", stream);
  return 1;
}

extern "C" int dtt_grad_clip(int n, void* const* grads, const long* numel, const int* dtypes, double max_norm, float* out, void* workspace,
                             size_t workspace_bytes, void* stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (!check_grads("grad_clip", n, grads, numel, dtypes)) return 0;
  DTT_REQUIRE(out && aligned_to(out, 4) && workspace && aligned_to(workspace, 8), "grad_clip: null or unaligned pointer");
  DTT_REQUIRE(max_norm >= 0.0, "grad_clip: max_norm must not be negative");
  const size_t need = dtt_grad_norm_workspace_bytes(n, numel);
  DTT_REQUIRE(workspace_bytes >= need, "grad_clip: workspace too small");
  Spans spans(n + 2L);
  DTT_REQUIRE(spans.s, "grad_clip: out of host memory");
  for (int i = 0; i < n; ++i) spans.add(grads[i], numel[i] * type_bytes(dtypes[i]), true);
  spans.add(out, 8, true);
  spans.add(workspace, (long)need, true);
  DTT_REQUIRE(!spans.clash(), "grad_clip: two of the gradients, the result or the workspace share memory");
  double* partial = static_cast<double*>(workspace);
  dtt_prof_begin("grad_clip", stream);
  NormPart part;
  part.partial = partial;
  part.max_norm = max_norm;
  part.n = norm_partials(n, grads, numel, dtypes, 0, partial, stream);
  if (part.n < 0) return 0;
  if (part.n == 0) {   // nothing but empty tensors: norm 0
    hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(kFinish), 0, stream, partial, 0, max_norm, out);
    DTT_CHECK_LAUNCH("grad_norm_finish_kernel");
  }
  const long chunk = n > 0 ? norm_chunk(n, numel) : 1;
  ScaleTable tab;
  float* to = out;
  for (int i = 0; i < n;) {
    tab.n = 0; tab.chunk = chunk;
    int here = 0;
    for (; i < n && tab.n < kMaxNorm; ++i) {
      if (numel[i] == 0) continue;
      const int j = tab.n++;
      tab.g[j] = grads[i]; tab.numel[j] = numel[i]; tab.dtype[j] = dtypes[i]; tab.block0[j] = here;
      here += (int)((numel[i] + chunk - 1) / chunk);
    }
    if (here == 0) break;
    hipLaunchKernelGGL(grad_clip_kernel, dim3((unsigned)here), dim3(kThreads), 0, stream, tab, part, to);
    DTT_CHECK_LAUNCH("grad_clip_kernel");
    to = nullptr;   // (the first launch has written norm and factor)
  }
  dtt_prof_end("grad_clip", stream);
  return 1;
}

extern "C" size_t dtt_adamw_workspace_bytes(int n, const long* numel) {
  return (size_t)(n > 0 ? n : 1) * sizeof(Factors) + dtt_grad_norm_workspace_bytes(n, numel);
}

namespace {

// The tensors of a step, of one element type (dtypes NULL) or of several; bases NULL: moments in fp32.
struct StepLists {
  int n;
  const int* dtypes;
  int dtype;
  void* const* params;
  const void* const* grads;
  const void* const* exp_avgs;
  const void* const* exp_avg_sqs;
  const short* const* bases;
  const long* numel;
  float* const* steps;
  const double* lr;
  const float* const* lr_device;
  const double* decay;
};

// what a step checks of its tensors, rates and norm; the buffers' spans are collected for the overlap check (spans_of(n) of them at most)
long spans_of(int n) { return 7L * (n > 0 ? n : 0) + 2; }
int check_lists(const char* what, const StepLists& l, bool in8bits, const float* clip, bool clip_written, Spans& spans) {
  DTT_REQUIRE(l.n >= 0 && (l.n == 0 || (l.params && l.grads && l.exp_avgs && l.exp_avg_sqs && l.numel && l.steps && l.lr && l.decay && (l.bases || !in8bits))),
              "%s: null pointer", what);
  DTT_REQUIRE(aligned_to(clip, 4), "%s: unaligned norm and factor", what);
  DTT_REQUIRE(spans.s, "%s: out of host memory", what);
  const int ms = in8bits ? 1 : 4;
  for (int i = 0; i < l.n; ++i) {
    const int dtype = l.dtypes ? l.dtypes[i] : l.dtype;
    DTT_REQUIRE(dtype >= kF32 && dtype <= kF16, "%s: unknown element type %d", what, dtype);
    const int es = type_bytes(dtype);
    DTT_REQUIRE(l.numel[i] >= 0 && l.numel[i] <= kMaxNumel, "%s: tensor %d: bad element count", what, i);
    DTT_REQUIRE(l.steps[i] && aligned_to(l.steps[i], 4), "%s: tensor %d: null or unaligned step counter", what, i);
    DTT_REQUIRE(!l.lr_device || aligned_to(l.lr_device[i], 4), "%s: tensor %d: unaligned learning rate", what, i);
    DTT_REQUIRE(l.lr[i] >= 0.0 && l.decay[i] >= 0.0, "%s: tensor %d: learning rate and weight decay must not be negative", what, i);
    DTT_REQUIRE(l.numel[i] == 0 || (l.params[i] && l.grads[i] && aligned_to(l.params[i], es) && aligned_to(l.grads[i], es)),
                "%s: tensor %d: null or unaligned pointer", what, i);
    DTT_REQUIRE(l.numel[i] == 0 || (l.exp_avgs[i] && l.exp_avg_sqs[i] && aligned_to(l.exp_avgs[i], ms) && aligned_to(l.exp_avg_sqs[i], ms) &&
                                    (!in8bits || (l.bases[i] && aligned_to(l.bases[i], 4)))),
                "%s: tensor %d: null or unaligned moment", what, i);
  }
  for (int i = 0; i < l.n; ++i) spans.add(l.params[i], l.numel[i] * type_bytes(l.dtypes ? l.dtypes[i] : l.dtype), true);
  for (int i = 0; i < l.n; ++i) spans.add(l.grads[i], l.numel[i] * type_bytes(l.dtypes ? l.dtypes[i] : l.dtype), false);
  for (int i = 0; i < l.n; ++i) spans.add(l.steps[i], 4, true);
  for (int i = 0; i < l.n; ++i) spans.add(l.exp_avgs[i], l.numel[i] * ms, true);
  for (int i = 0; i < l.n; ++i) spans.add(l.exp_avg_sqs[i], l.numel[i] * ms, true);
  for (int i = 0; in8bits && i < l.n; ++i) spans.add(l.bases[i], (l.numel[i] + kBlock - 1) / kBlock * 4, true);
  for (int i = 0; l.lr_device && i < l.n; ++i) spans.add(l.lr_device[i], l.lr_device[i] ? 4 : 0, false);
  spans.add(clip, clip ? 8 : 0, clip_written);
  return 1;
}

// what both steps check
int check_step(const char* what, const StepLists& l, bool in8bits, double beta1, double beta2, double eps, double max_norm, const float* clip,
               int skip_nonfinite, const void* workspace, size_t workspace_bytes) {
  DTT_REQUIRE(l.dtype >= kF32 && l.dtype <= kF16, "%s: unknown element type %d", what, l.dtype);
  DTT_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "%s: betas must lie in [0, 1)", what);
  DTT_REQUIRE(eps >= 0.0, "%s: eps must not be negative", what);
  DTT_REQUIRE(max_norm == max_norm, "%s: max_norm is not a number", what);
  DTT_REQUIRE(clip || (!skip_nonfinite && max_norm < 0.0), "%s: clipping and skip_nonfinite need a place for norm and factor", what);
  Spans spans(spans_of(l.n));
  if (!check_lists(what, l, in8bits, clip, max_norm >= 0.0, spans)) return 0;
  const size_t need = dtt_adamw_workspace_bytes(l.n, l.numel);
  DTT_REQUIRE(workspace && aligned_to(workspace, 16) && workspace_bytes >= need, "%s: workspace too small or unaligned", what);
  spans.add(workspace, (long)need, true);
  DTT_REQUIRE(!spans.clash(), "%s: two of the buffers share memory", what);
  return 1;
}

// the norm where the call clips, then counters and factors
int prepare(int n, int dtype, const void* const* grads, const long* numel, float* const* steps, const double* lr, const float* const* lr_device,
            const double* decay, const unsigned* ids, unsigned seed, double beta1, double beta2, double max_norm, float* clip, int skip_nonfinite,
            Factors* factors, hipStream_t stream) {
  NormPart part = {nullptr, 0, 0.0};
  if (max_norm >= 0.0) {
    double* partial = reinterpret_cast<double*>(factors + (n > 0 ? n : 1));
    part.n = norm_partials(n, grads, numel, nullptr, dtype, partial, stream);
    if (part.n < 0) return 0;
    part.partial = partial;
    part.max_norm = max_norm;
  }
  PrepareTable tab;
  tab.beta1 = beta1; tab.beta2 = beta2; tab.seed = seed;
  for (int i = 0; i < n;) {
    const int i0 = i;
    int rates = 0;
    for (tab.n = 0; i < n && tab.n < kMaxPrepare; ++i) {
      const float* dev = lr_device ? lr_device[i] : nullptr;
      int r = 0;
      while (r < rates && !(tab.rate[r].lr == lr[i] && tab.rate[r].lr_device == dev && tab.rate[r].decay == decay[i])) ++r;
      if (r == rates) {
        if (rates == kMaxRates) break;   // more rates than the table holds: another launch
        tab.rate[rates].lr = lr[i]; tab.rate[rates].lr_device = dev; tab.rate[rates].decay = decay[i];
        ++rates;
      }
      const int j = tab.n++;
      tab.step[j] = steps[i]; tab.which[j] = (unsigned char)r; tab.id[j] = ids ? ids[i] : (unsigned)i;
    }
    hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(kFinish), 0, stream, tab, part, clip, skip_nonfinite, factors + i0);
    DTT_CHECK_LAUNCH("adamw_prepare_kernel");
  }
  return 1;
}

// whether a launch over these tensors has waves hold four blocks (see Wave8)
bool four_blocks(int n, const long* numel) {
  long workgroups = 0;
  for (int i = 0; i < n; ++i) workgroups += (numel[i] + Wave8<4>::kElems - 1) / Wave8<4>::kElems;
  return workgroups >= 4L * dtt_device_cus();
}
int workgroups8(long numel, bool four) {
  const int per = four ? Wave8<4>::kElems : Wave8<1>::kElems;
  return (int)((numel + per - 1) / per);
}

Consts consts(double beta1, double beta2, double eps) {
  Consts k;
  k.beta1 = (float)beta1; k.one_beta1 = (float)(1.0 - beta1);
  k.beta2 = (float)beta2; k.one_beta2 = (float)(1.0 - beta2);
  k.eps = (float)eps;
  return k;
}

}  // namespace

extern "C" int dtt_adamw_check(int n, const int* dtypes, void* const* params, const void* const* grads, const void* const* exp_avgs,
                               const void* const* exp_avg_sqs, const short* const* bases, const long* numel, float* const* steps,
                               const double* lr, const float* const* lr_device, const double* weight_decay, const float* clip) {
  DTT_REQUIRE(n == 0 || dtypes, "adamw_check: null pointer");
  const StepLists lists = {n, dtypes, 0, params, grads, exp_avgs, exp_avg_sqs, bases, numel, steps, lr, lr_device, weight_decay};
  Spans spans(spans_of(n));
  if (!check_lists("adamw_check", lists, bases != nullptr, clip, false, spans)) return 0;
  DTT_REQUIRE(!spans.clash(), "adamw_check: two of the buffers share memory");
  return 1;
}

extern "C" int dtt_adamw_step(int n, int dtype, void* const* params, const void* const* grads, float* const* exp_avgs,
                              float* const* exp_avg_sqs, const long* numel, float* const* steps, const double* lr,
                              const float* const* lr_device, const double* weight_decay, double beta1, double beta2, double eps,
                              double max_norm, float* clip, int skip_nonfinite, void* workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const StepLists lists = {n, nullptr, dtype, params, grads, reinterpret_cast<const void* const*>(exp_avgs),
                           reinterpret_cast<const void* const*>(exp_avg_sqs), nullptr, numel, steps, lr, lr_device, weight_decay};
  if (!check_step("adamw", lists, false, beta1, beta2, eps, max_norm, clip, skip_nonfinite, workspace, workspace_bytes)) return 0;
  Factors* factors = static_cast<Factors*>(workspace);
  const Consts k = consts(beta1, beta2, eps);
  dtt_prof_begin("adamw", stream);
  if (!prepare(n, dtype, grads, numel, steps, lr, lr_device, weight_decay, nullptr, 0u, beta1, beta2, max_norm, clip, skip_nonfinite, factors,
               stream)) return 0;
  StepTable tab;
  for (int i0 = 0; i0 < n; i0 += tab.n) {
    tab.n = fit(n - i0, kMaxStep, numel + i0);
    int blocks = 0;
    for (int j = 0; j < tab.n; ++j) {
      const int i = i0 + j;
      tab.p[j] = params[i]; tab.g[j] = grads[i]; tab.m[j] = exp_avgs[i]; tab.v[j] = exp_avg_sqs[i]; tab.numel[j] = numel[i];
      tab.block0[j] = blocks;
      const long body = numel[i] - step_head(exp_avgs[i], numel[i]);
      const long nb = numel[i] == 0 ? 0 : body <= kStepElems ? 1 : (body + kStepElems - 1) / kStepElems;
      blocks += (int)nb;
    }
    if (blocks == 0) continue;
    const dim3 grid((unsigned)blocks), wg(kThreads);
    if (dtype == kF32) hipLaunchKernelGGL((adamw_step_kernel<float>), grid, wg, 0, stream, tab, factors + i0, clip, skip_nonfinite, k);
    else if (dtype == kBf16) hipLaunchKernelGGL((adamw_step_kernel<__bf16>), grid, wg, 0, stream, tab, factors + i0, clip, skip_nonfinite, k);
    else hipLaunchKernelGGL((adamw_step_kernel<_Float16>), grid, wg, 0, stream, tab, factors + i0, clip, skip_nonfinite, k);
    DTT_CHECK_LAUNCH("adamw_step_kernel");
  }
  dtt_prof_end("adamw", stream);
  return 1;
}

extern "C" int dtt_adamw8_step(int n, int dtype, void* const* params, const void* const* grads, unsigned char* const* exp_avgs,
                               unsigned char* const* exp_avg_sqs, short* const* bases, const long* numel, float* const* steps,
                               const double* lr, const float* const* lr_device, const double* weight_decay, const unsigned* ids,
                               unsigned seed, double beta1, double beta2, double eps, double max_norm, float* clip, int skip_nonfinite,
                               void* workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const StepLists lists = {n, nullptr, dtype, params, grads, reinterpret_cast<const void* const*>(exp_avgs),
                           reinterpret_cast<const void* const*>(exp_avg_sqs), bases, numel, steps, lr, lr_device, weight_decay};
  if (!check_step("adamw8", lists, true, beta1, beta2, eps, max_norm, clip, skip_nonfinite, workspace, workspace_bytes)) return 0;
  Factors* factors = static_cast<Factors*>(workspace);
  const Consts k = consts(beta1, beta2, eps);
  dtt_prof_begin("adamw8", stream);
  if (!prepare(n, dtype, grads, numel, steps, lr, lr_device, weight_decay, ids, seed, beta1, beta2, max_norm, clip, skip_nonfinite, factors,
               stream)) return 0;
  const bool exact = !(eps >= 0x1p-39 / sqrt(1.0 - beta2));
  long codes = 0;
  for (int i = 0; i < n; ++i) codes += 2 * numel[i];
  const bool keep = codes <= kKeepCodes;
  Step8Table tab;
  for (int i0 = 0; i0 < n; i0 += tab.n) {
    tab.n = fit(n - i0, kMaxStep8, numel + i0);
    const bool four = !exact && four_blocks(tab.n, numel + i0);
    int blocks = 0;
    for (int j = 0; j < tab.n; ++j) {
      const int i = i0 + j;
      tab.p[j] = params[i]; tab.g[j] = grads[i]; tab.m[j] = exp_avgs[i]; tab.v[j] = exp_avg_sqs[i]; tab.base[j] = reinterpret_cast<int*>(bases[i]);
      tab.numel[j] = numel[i]; tab.block0[j] = blocks;
      blocks += workgroups8(numel[i], four);
    }
    if (blocks == 0) continue;
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, tab, factors + i0, clip, skip_nonfinite, k);
    };
    const auto shape = [&](auto type) {
      using T = decltype(type);
      if (exact) launch(adamw8_step_kernel<T, 1, true, true>);
      else if (!four) launch(adamw8_step_kernel<T, 1, false, true>);
      else if (keep) launch(adamw8_step_kernel<T, 4, false, true>);
      else launch(adamw8_step_kernel<T, 4, false, false>);
    };
    if (dtype == kF32) shape(float());
    else if (dtype == kBf16) shape(__bf16());
    else shape(_Float16());
    DTT_CHECK_LAUNCH("adamw8_step_kernel");
  }
  dtt_prof_end("adamw8", stream);
  return 1;
}

extern "C" int dtt_adamw8_unpack(int n, const unsigned char* const* exp_avgs, const unsigned char* const* exp_avg_sqs,
                                 const short* const* bases, const long* numel, int out_dtype, void* const* out_avgs,
                                 void* const* out_avg_sqs, void* stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DTT_REQUIRE(n >= 0 && (n == 0 || (exp_avgs && exp_avg_sqs && bases && numel && out_avgs && out_avg_sqs)), "adamw8_unpack: null pointer");
  DTT_REQUIRE(out_dtype == kF32 || out_dtype == kBf16, "adamw8_unpack: the values come as fp32 or bf16 (fp16 lacks their range)");
  const int es = type_bytes(out_dtype);
  Spans spans(5L * (n > 0 ? n : 0));
  DTT_REQUIRE(spans.s, "adamw8_unpack: out of host memory");
  for (int i = 0; i < n; ++i) {
    DTT_REQUIRE(numel[i] >= 0 && numel[i] <= kMaxNumel, "adamw8_unpack: tensor %d: bad element count", i);
    DTT_REQUIRE(numel[i] == 0 || (exp_avgs[i] && exp_avg_sqs[i] && bases[i] && aligned_to(bases[i], 4) && out_avgs[i] && out_avg_sqs[i] &&
                                  aligned_to(out_avgs[i], es) && aligned_to(out_avg_sqs[i], es)),
                "adamw8_unpack: tensor %d: null or unaligned pointer", i);
  }
  for (int i = 0; i < n; ++i) spans.add(exp_avgs[i], numel[i], false);
  for (int i = 0; i < n; ++i) spans.add(exp_avg_sqs[i], numel[i], false);
  for (int i = 0; i < n; ++i) spans.add(bases[i], (numel[i] + kBlock - 1) / kBlock * 4, false);
  for (int i = 0; i < n; ++i) spans.add(out_avgs[i], numel[i] * es, true);
  for (int i = 0; i < n; ++i) spans.add(out_avg_sqs[i], numel[i] * es, true);
  DTT_REQUIRE(!spans.clash(), "adamw8_unpack: two of the tensors share memory");
  UnpackTable tab;
  for (int i0 = 0; i0 < n; i0 += tab.n) {
    tab.n = fit(n - i0, kMaxStep8, numel + i0);
    const bool four = four_blocks(tab.n, numel + i0);
    int blocks = 0;
    for (int j = 0; j < tab.n; ++j) {
      const int i = i0 + j;
      tab.m[j] = exp_avgs[i]; tab.v[j] = exp_avg_sqs[i]; tab.base[j] = reinterpret_cast<const int*>(bases[i]); tab.out_m[j] = out_avgs[i];
      tab.out_v[j] = out_avg_sqs[i]; tab.numel[j] = numel[i]; tab.block0[j] = blocks;
      blocks += workgroups8(numel[i], four);
    }
    if (blocks == 0) continue;
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, tab); };
    if (out_dtype == kF32) four ? launch(unpack_moments_kernel<float, 4>) : launch(unpack_moments_kernel<float, 1>);
    else four ? launch(unpack_moments_kernel<__bf16, 4>) : launch(unpack_moments_kernel<__bf16, 1>);
    DTT_CHECK_LAUNCH("unpack_moments_kernel");
  }
  return 1;
}
