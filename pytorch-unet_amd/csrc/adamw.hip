// Optimizer step over many tensors (include/unetk.h: "optimizer step over many tensors"): global gradient norm, clip,
// AdamW with fp32 moments or with e4m3 moments and one power-of-two scale per 256 elements.
//
// The tensors of a call travel as kernel arguments, a table of up to 4 KiB a launch: nothing is uploaded, kept or shared between
// calls, and a captured graph owns its copy.  Each tensor is cut into chunks of kChunk elements; a workgroup takes every
// gridDim.x-th chunk and finds its tensor with one compare per lane and a ballot over 64 tensors' first chunks.
//
// Everything here is bound by HBM (a copy of 2 GB reaches 5.0 TB/s on this card, a sum 4.0 to 6.3).  Measured, three sets of
// inputs in turn so that no step finds its own in the 256 MiB last-level cache; "U-Net": 31 M elements in 64 tensors, "wide":
// 124 M; bytes are what a step has to read and write once, the second read of the gradients not counted:
//                                   sums + counts    update                both
//   fp32, clip, U-Net                  22 us         139 us, 6.3 TB/s      161 us   (0.87 GB, 174 us at the copy's rate)
//   fp32, clip, wide                   80            596,    5.8           676      (3.48 GB, 695)
//   bf16, clip, 17 M elements           9             65,    5.8            74      (0.38 GB, 76)
//   8-bit moments, fp32, U-Net         23             75,    6.6            98      (0.50 GB, 99)
//   8-bit moments, bf16, wide          43            214,    5.8           257      (1.24 GB, 249)
// (profiles/adamw_kernels.txt; what other grids, chunks and cache policies take: profiles/adamw_sweeps.txt)
#include <algorithm>
#include <cfloat>
#include <new>

#include "common.h"

namespace {

constexpr int kGrads = 192;       // tensors a launch that needs their gradients alone: 20 bytes each
constexpr int kPrepare = 128;     // 28 bytes each
constexpr int kSteps = 256;       // a prepare without sums: 8 bytes and a thread each
constexpr int kUpdate = 64;       // 52 bytes each
constexpr int kChunk = 4096;      // elements, 16 per thread; 2048 / 8192: wide 672 / 693 us (678), wide bf16 in 8 bits 277 / 264
                                  // (262 to 270), 190 tensors 48 / 56 (48), clip of 130 bf16 tensors 37 / 35 (35)
constexpr int kBlock = 256;       // elements that share a scale: one wave, four per lane
// Workgroups at most.  The sums: every later workgroup adds up as many partials; with 512 / 1024 / 2048 a step takes 165 / 162 /
// 164 us for the U-Net and 684 / 678 / 694 for its wide form.  The clip does not mind (512 to 4096: 1 % for the U-Net).  The
// update wants few streams at once, 512 / 768 / 1024 / 2048 take 164 / 162 / 163 / 170 us for the U-Net, 671 / 678 / 686 / 725
// for its wide form, 80 / 75 / 76 / 78 in bf16.  The 8-bit one has arithmetic to hide and evens out its end with many: 2048 /
// 4096 / 8192 take 102 / 99 / 99 and 275 / 267 / 262 to 270 us.
constexpr int kSumsqGrid = 1024;
constexpr int kClipGrid = 2048;
constexpr int kUpdateGrid = 768;
constexpr int kUpdate8Grid = 8192;

template <int N> struct Chunks {
  int64_t numel[N];
  int first[N];                   // first chunk of each tensor; INT32_MAX behind the last tensor
  int total;
};
struct GradTable {
  Chunks<kGrads> c;
  void* grad[kGrads];
};
struct StepTable {
  float* step[kSteps];
};
struct PrepareTable {
  Chunks<kPrepare> c;
  const void* grad[kPrepare];
  float* step[kPrepare];
};
struct UpdateTable {
  Chunks<kUpdate> c;
  void* param[kUpdate];
  const void* grad[kUpdate];
  void* exp_avg[kUpdate];
  void* exp_avg_sq[kUpdate];
};
struct Update8Table : UpdateTable {
  void* scales[kUpdate];          // NULL: this tensor's moments are fp32
};

struct Clip {                     // where an update finds its clip coefficient
  const double* partials;
  int n_partials;
  float max_norm;
  const float* grad_scale;
  float* norm_out;
};
struct Coefs {                    // per tensor, written by the prepare kernel
  float step_size, root_correction, decay;
  unsigned key;
};
static_assert(sizeof(GradTable) <= 3900 && sizeof(PrepareTable) <= 3900 && sizeof(Update8Table) <= 3900,
              "with a launch's scalars under 4 KiB");
static_assert(kGrads % 64 == 0 && kPrepare % 64 == 0 && kPrepare <= 256 && kUpdate % 64 == 0, "lanes and threads");
static_assert(sizeof(Coefs) == 16, "unetk.h promises 16 bytes a tensor");

// Which tensor owns a chunk (wave-uniform).  Tensors without elements own none: their first chunk is the next one's.
template <int N> struct Owners {
  int first[N / 64];              // this lane's entries
  __device__ __forceinline__ explicit Owners(const Chunks<N>& c) {
#pragma unroll
    for (int k = 0; k < N / 64; ++k) first[k] = c.first[k * 64 + (threadIdx.x & 63)];
  }
  __device__ __forceinline__ int of(int chunk) const {
    int t = -1;
#pragma unroll
    for (int k = 0; k < N / 64; ++k) t += __popcll(__ballot(first[k] <= chunk));
    return __builtin_amdgcn_readfirstlane(t);
  }
};

// Four elements at any element-aligned address (global accesses of gfx950 need no more).
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32u __attribute__((aligned(1)));
typedef unsigned short u16u __attribute__((aligned(1)));
template <typename T> struct Raw4 { typedef u16x4u type; };
template <> struct Raw4<float> { typedef f32x4u type; };

// FULL: all four exist; otherwise those before n, zeros behind.  ONCE: nothing of this step reads them again, so they pass by
// the caches, as all stores do, and leave the gradients there between the sums and the update: the U-Net's step falls from 186
// to 162 us, the wide one's from 766 to 678; with the sums' reads passing by as well it is 181 and 714 to 721.
template <typename T, bool FULL, bool ONCE = false>
__device__ __forceinline__ typename Raw4<T>::type load4(const void* base, long i, long n) {
  typedef typename Raw4<T>::type V;
  const T* p = static_cast<const T*>(base) + i;
  if (FULL && ONCE) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  if (FULL || i + 4 <= n) return *reinterpret_cast<const V*>(p);
  V v = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (i + k < n) {
      if constexpr (sizeof(T) == 4) v[k] = p[k];
      else v[k] = __builtin_bit_cast(unsigned short, p[k]);
    }
  return v;
}
template <typename T> __device__ __forceinline__ float elem(const typename Raw4<T>::type& v, int k) {
  if constexpr (sizeof(T) == 4) return v[k];
  else return to_f32(__builtin_bit_cast(T, (unsigned short)v[k]));
}
template <typename T, bool FULL> __device__ __forceinline__ void store4(void* base, long i, long n, const float* in) {
  T* p = static_cast<T*>(base) + i;
  if (FULL || i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      __builtin_nontemporal_store(f32x4u{in[0], in[1], in[2], in[3]}, reinterpret_cast<f32x4u*>(p));
    } else {
      u16x4u v;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __builtin_bit_cast(unsigned short, from_f32<T>(in[k]));
      __builtin_nontemporal_store(v, reinterpret_cast<u16x4u*>(p));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (i + k < n) p[k] = from_f32<T>(in[k]);
  }
}

// Sum over the workgroup's 256 threads in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double s) {
  __shared__ double red[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// Squares are exact in fp64 (24-bit significands), so nothing overflows or is lost on the way to the norm.
template <typename T, bool FULL> __device__ __forceinline__ double chunk_sumsq(const void* grad, long base, long n) {
  typename Raw4<T>::type g[kChunk / 1024];
#pragma unroll
  for (int j = 0; j < kChunk / 1024; ++j) g[j] = load4<T, FULL>(grad, base + j * 1024, n);
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kChunk / 1024; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const double x = elem<T>(g[j], k);
      s += x * x;
    }
  return s;
}
// One read of the gradients: 124 MB that a kernel before wrote in 21 to 22 us (5.7 TB/s), by themselves or in a step; 31 us right
// behind the clip of other gradients, whose stores are still on their way to memory.  A workgroup's sum goes to a slot of its own,
// so that the norm does not depend on who comes first.
template <typename T, typename Table> __device__ __forceinline__ void write_partial(const Table& tb, double* partials) {
  const Owners owners(tb.c);
  double s = 0.0;
  for (int chunk = blockIdx.x; chunk < tb.c.total; chunk += gridDim.x) {
    const int t = owners.of(chunk);
    const long n = tb.c.numel[t], start = (long)(chunk - tb.c.first[t]) * kChunk;
    s += start + kChunk <= n ? chunk_sumsq<T, true>(tb.grad[t], start + threadIdx.x * 4, n)
                             : chunk_sumsq<T, false>(tb.grad[t], start + threadIdx.x * 4, n);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

template <typename T> __global__ __launch_bounds__(256) void grad_sumsq_kernel(GradTable tb, double* __restrict__ partials) {
  write_partial<T>(tb, partials);
}

// The finalizer of the 32-bit MurmurHash3: a published mixing in which every input bit flips every output bit about half of the
// time.
__device__ __forceinline__ unsigned mix32(unsigned h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

struct Schedule {
  double lr, beta1, beta2, weight_decay;
  const float* lr_dev;
  const float* found_inf;
  unsigned seed;
};
// Counts a tensor's step and writes its bias corrections.
__device__ __forceinline__ void count_step(float* step, const Schedule& h, Coefs* out) {
  if (h.found_inf && *h.found_inf != 0.f) return;
  const float t = *step + 1.f;
  *step = t;
  const double rate = h.lr_dev ? (double)*h.lr_dev : h.lr;
  Coefs c;
  c.step_size = (float)(rate / (1.0 - pow(h.beta1, (double)t)));
  c.root_correction = (float)(1.0 / sqrt(1.0 - pow(h.beta2, (double)t)));
  c.decay = (float)(1.0 - rate * h.weight_decay);
  c.key = mix32((unsigned)(long)t * 0x9E3779B9u + h.seed);
  *out = c;
}
__global__ __launch_bounds__(kSteps) void adamw_steps_kernel(StepTable tb, int n_tensors, Schedule h, Coefs* __restrict__ coefs) {
  if (threadIdx.x < n_tensors) count_step(tb.step[threadIdx.x], h, coefs + threadIdx.x);
}
template <typename T>
__global__ __launch_bounds__(256) void adamw_prepare_kernel(PrepareTable tb, int n_tensors, Schedule h, Coefs* __restrict__ coefs,
                                                            double* __restrict__ partials) {
  if (blockIdx.x == 0 && threadIdx.x < n_tensors) count_step(tb.step[threadIdx.x], h, coefs + threadIdx.x);
  write_partial<T>(tb, partials);
}

// What the gradient is multiplied by.  Every workgroup sums the partials in the same order, so all agree to the bit, and no
// launch in between has to (a kernel of one workgroup costs 3 us; for up to 128 tensors these sums do not show beside the read
// of the gradients).  Their cost grows with the number of partials times that of the launches: over 1000 / 2000 tensors of 0.5 M
// elements a step takes 9 / 130 us more than one without a clip and a read of the gradients at 6 TB/s (2.9 / 5.9 ms in all), with
// 8-bit moments and their larger grid 230 / 1260 us more (2.0 / 4.8 ms).  A norm that is not a number makes the coefficient one
// that is not either, as clip_grad_norm_ does.
__device__ __forceinline__ float grad_factor(const Clip& c) {
  const double inv_scale = c.grad_scale ? 1.0 / (double)*c.grad_scale : 1.0;
  if (!c.partials) return (float)inv_scale;
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < c.n_partials; i += 256) s += c.partials[i];
  const float norm = (float)(sqrt(block_sum(s)) * inv_scale);
  if (blockIdx.x == 0 && threadIdx.x == 0 && c.norm_out) *c.norm_out = norm;
  float coef = c.max_norm / (norm + 1e-6f);
  coef = coef > 1.f ? 1.f : coef;
  return (float)(coef * inv_scale);
}

// Second pass of the clip: 38 to 39 us for 124 MB of gradients (6.4 TB/s read and written, the read mostly from the last-level
// cache), from the last chunk the sums read to the first, as in the updates.
template <typename T, bool FULL> __device__ __forceinline__ void clip_chunk(void* grad, long base, long n, float coef) {
  typename Raw4<T>::type g[kChunk / 1024];
#pragma unroll
  for (int j = 0; j < kChunk / 1024; ++j) g[j] = load4<T, FULL>(grad, base + j * 1024, n);
#pragma unroll
  for (int j = 0; j < kChunk / 1024; ++j) {
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = elem<T>(g[j], k) * coef;
    store4<T, FULL>(grad, base + j * 1024, n, x);
  }
}
template <typename T> __global__ __launch_bounds__(256) void grad_clip_kernel(GradTable tb, Clip clip) {
  const Owners owners(tb.c);
  const float coef = grad_factor(clip);
  if (coef == 1.f) return;
  for (int chunk = tb.c.total - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const int t = owners.of(chunk);
    const long n = tb.c.numel[t], start = (long)(chunk - tb.c.first[t]) * kChunk;
    if (start + kChunk <= n) clip_chunk<T, true>(tb.grad[t], start + threadIdx.x * 4, n, coef);
    else clip_chunk<T, false>(tb.grad[t], start + threadIdx.x * 4, n, coef);
  }
}

struct Betas {
  float beta1, rest1, beta2, rest2, eps;
};

// One element: the moments in place, the new parameter returned.  Square root and quotient are the correctly rounded ones: at
// 28 bytes an element there is time for 200 vector instructions, and this takes about 60.
__device__ __forceinline__ float adamw_element(float p, float g, float& m, float& v, const Coefs& c, const Betas& b) {
  m = fmaf(b.rest1, g, b.beta1 * m);
  v = fmaf(b.rest2 * g, g, b.beta2 * v);
  return fmaf(-c.step_size, m / fmaf(sqrtf(v), c.root_correction, b.eps), p * c.decay);
}

template <typename T, bool FULL>
__device__ __forceinline__ void update_chunk(const UpdateTable& tb, int t, long start, long n, float factor, const Coefs& c,
                                             const Betas& b) {
#pragma unroll
  for (int j = 0; j < kChunk / 1024; ++j) {
    const long i = start + threadIdx.x * 4 + j * 1024;
    if (!FULL && i >= n) break;
    const auto pv = load4<T, FULL, true>(tb.param[t], i, n), gv = load4<T, FULL>(tb.grad[t], i, n);
    const auto mv = load4<float, FULL, true>(tb.exp_avg[t], i, n), vv = load4<float, FULL, true>(tb.exp_avg_sq[t], i, n);
    float p[4], m[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[k] = mv[k];
      v[k] = vv[k];
      p[k] = adamw_element(elem<T>(pv, k), elem<T>(gv, k) * factor, m[k], v[k], c, b);
    }
    store4<T, FULL>(tb.param[t], i, n, p);
    store4<float, FULL>(tb.exp_avg[t], i, n, m);
    store4<float, FULL>(tb.exp_avg_sq[t], i, n, v);
  }
}

// From the last chunk to the first: what the sums read last is still in the last-level cache (forwards: up to 6 % more).
template <typename T>
__global__ __launch_bounds__(256) void adamw_update_kernel(UpdateTable tb, Betas b, const Coefs* __restrict__ coefs,
                                                           const float* __restrict__ found_inf, Clip clip) {
  const Owners owners(tb.c);
  const float factor = grad_factor(clip);
  if (found_inf && *found_inf != 0.f) return;
  for (int chunk = tb.c.total - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const int t = owners.of(chunk);
    const Coefs c = coefs[t];
    const long n = tb.c.numel[t], start = (long)(chunk - tb.c.first[t]) * kChunk;
    if (start + kChunk <= n) update_chunk<T, true>(tb, t, start, n, factor, c, b);
    else update_chunk<T, false>(tb, t, start, n, factor, c, b);
  }
}

// ---- 8-bit moments.  A scale is 2^k, kept as the byte e = 127 + k.  Multiplying by a power of two is exact, so a value that
// fits e4m3 comes back as it went in, and x * 2^-(k + 120) has its e4m3 code in the top bits of its fp32 word: exponent field
// and three bits of mantissa from bit 20 on, subnormals included (fp32's subnormals begin where e4m3's do then).
constexpr unsigned kInfinity = 0x7f800000u;

// Largest of the wave's values, in a scalar register: DPP shifts within rows of 16, then row to row; zeros come in at the ends.
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#define UNETK_MAX_STEP(ctrl) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true))
  UNETK_MAX_STEP(0x111);          // row_shr:1, 2, 4, 8
  UNETK_MAX_STEP(0x112);
  UNETK_MAX_STEP(0x114);
  UNETK_MAX_STEP(0x118);
  UNETK_MAX_STEP(0x142);          // row_bcast:15, 31
  UNETK_MAX_STEP(0x143);
#undef UNETK_MAX_STEP
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
// 127 + the smallest k >= -127 with top <= 448 * 2^k = 1.75 * 2^(8 + k): the exponent goes up by one beyond a mantissa of 1.75
__device__ __forceinline__ int scale_byte(unsigned top) { return max((int)((top + 0x1fffffu) >> 23) - 8, 0); }

// Four codes of a block with scale byte e; carry[k]: 16 random bits in 4..19, which together with the half step in bit 3 push
// the word over the next code as often as it is near.  ROOT: not negative, and above zero stays above zero.
template <bool ROOT> __device__ __forceinline__ unsigned encode4(const float* x, int e, const unsigned* carry) {
  unsigned w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = __float_as_uint(__builtin_amdgcn_ldexpf(x[k], 7 - e)) + carry[k];
    if (ROOT) w[k] = max(w[k], min(__float_as_uint(x[k]), 0x100000u)) << 4;
    else w[k] = (w[k] & 0x80000000u) | (w[k] << 4 & 0x7fffffffu);
  }
  // the top bytes of the four words
  return __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0703u) | __builtin_amdgcn_perm(w[3], w[2], 0x07030c0cu);
}

// Rare: a value of the wave is not finite.  The scale is the finite ones', their codes are as ever, the others become NaN.
template <bool ROOT> __device__ __forceinline__ unsigned encode4_special(const float* x, int* e, const unsigned* carry) {
  float y[4];
  unsigned top = 0, nan = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned a = __float_as_uint(x[k]) & 0x7fffffffu;
    if (a >= kInfinity) nan |= 0xffu << 8 * k;
    y[k] = a >= kInfinity ? 0.f : x[k];
    top = max(top, a >= kInfinity ? 0u : a);
  }
  *e = scale_byte(wave_umax(top));
  return (encode4<ROOT>(y, *e, carry) & ~nan) | (nan & 0x7f7f7f7fu);
}

// A block of 256 elements, a wave's: four per lane, so that codes move as words, parameters as 8 or 16 bytes, and the block's
// maxima need six DPP steps and no LDS.  At 10 bytes an element (bf16) HBM leaves time for some 70 vector instructions; with
// correctly rounded roots and quotients, shuffles and checks at each element it took about 120 (373 us for 124 M elements),
// now about 60 (212 us, bound by HBM again): the scale's arithmetic is scalar, root and reciprocal are one instruction each
// (1 ulp, against a rounding to 3 bits of mantissa in the moments and 4 roundings in the update), and values that are not
// finite or squares that are subnormal (v_sqrt_f32 takes those for zero) are looked for once a wave.
template <typename T, bool FULL>
__device__ __forceinline__ void update_block(const Update8Table& tb, int t, long block, long n, float factor, const Coefs& c,
                                             const Betas& b) {
  const int lane = threadIdx.x & 63;
  const long i = block * kBlock + lane * 4;
  const auto pv = load4<T, FULL, true>(tb.param[t], i, n), gv = load4<T, FULL>(tb.grad[t], i, n);
  unsigned char* mp = static_cast<unsigned char*>(tb.exp_avg[t]) + i;
  unsigned char* rp = static_cast<unsigned char*>(tb.exp_avg_sq[t]) + i;
  unsigned mc = 0, rc = 0;
  if (FULL || i + 4 <= n) {
    mc = __builtin_nontemporal_load(reinterpret_cast<const u32u*>(mp));
    rc = __builtin_nontemporal_load(reinterpret_cast<const u32u*>(rp));
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (i + k < n) mc |= (unsigned)mp[k] << 8 * k, rc |= (unsigned)rp[k] << 8 * k;
  }
  u16u* sp = reinterpret_cast<u16u*>(static_cast<unsigned char*>(tb.scales[t]) + block * 2);
  const int old = __builtin_amdgcn_readfirstlane((int)*sp);
  const float ms = __builtin_amdgcn_ldexpf(1.f, (old & 255) - 127), rs = __builtin_amdgcn_ldexpf(1.f, (old >> 8) - 127);
  float m[4], r[4], p[4];
  {
    const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc, true);
    const auto r01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc, false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc, true);
    m[0] = m01[0] * ms; m[1] = m01[1] * ms; m[2] = m23[0] * ms; m[3] = m23[1] * ms;
    r[0] = r01[0] * rs; r[1] = r01[1] * rs; r[2] = r23[0] * rs; r[3] = r23[1] * rs;
  }
  // v, and whether one of the wave is so small that v_sqrt_f32 would take it for zero
  float v[4];
  unsigned mtop = 0, rtop = 0, least = ~0u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float g = elem<T>(gv, k) * factor;
    m[k] = fmaf(b.rest1, g, b.beta1 * m[k]);
    v[k] = fmaf(b.rest2 * g, g, b.beta2 * (r[k] * r[k]));
    least = min(least, __float_as_uint(v[k]) - 1u);                  // zero goes to the top
    mtop = max(mtop, __float_as_uint(m[k]) & 0x7fffffffu);
  }
  if (__any(least < 0x007fffffu)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = sqrtf(v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = __builtin_amdgcn_sqrtf(v[k]);
  }
  unsigned carry_m[4], carry_r[4];
  const unsigned place = (unsigned)i ^ (unsigned)(i >> 32) ^ c.key;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    rtop = max(rtop, __float_as_uint(r[k]) & 0x7fffffffu);
    // one ulp each of the root and the reciprocal; the denominator is no subnormal, which v_rcp_f32 would take for zero: a root
    // above zero exceeds 2^-75, and eps is zero or normal
    p[k] = fmaf(-c.step_size * m[k], __builtin_amdgcn_rcpf(fmaf(r[k], c.root_correction, b.eps)), elem<T>(pv, k) * c.decay);
    const unsigned h = mix32(place ^ k);
    carry_m[k] = (h << 4 & 0xffff0u) | 8u;
    carry_r[k] = (h >> 12 & 0xffff0u) | 8u;
  }
  store4<T, FULL>(tb.param[t], i, n, p);
  mtop = wave_umax(mtop);
  rtop = wave_umax(rtop);
  int me = scale_byte(mtop), re = scale_byte(rtop);
  if (__builtin_expect(max(mtop, rtop) < kInfinity, 1)) {
    mc = encode4<false>(m, me, carry_m);
    rc = encode4<true>(r, re, carry_r);
  } else {
    mc = encode4_special<false>(m, &me, carry_m);
    rc = encode4_special<true>(r, &re, carry_r);
  }
  if (FULL || i + 4 <= n) {
    __builtin_nontemporal_store(mc, reinterpret_cast<u32u*>(mp));
    __builtin_nontemporal_store(rc, reinterpret_cast<u32u*>(rp));
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (i + k < n) mp[k] = (unsigned char)(mc >> 8 * k), rp[k] = (unsigned char)(rc >> 8 * k);
  }
  if (lane == 0) *sp = (unsigned short)(me | re << 8);
}

// Tensors with 8-bit moments and, in the same launch, tensors with fp32 moments (a network's biases and BatchNorms: a launch of
// their own took 7 to 14 us).
template <typename T>
__global__ __launch_bounds__(256) void adamw8_update_kernel(Update8Table tb, Betas b, const Coefs* __restrict__ coefs,
                                                            const float* __restrict__ found_inf, Clip clip) {
  const Owners owners(tb.c);
  const float factor = grad_factor(clip);
  if (found_inf && *found_inf != 0.f) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int chunk = tb.c.total - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const int t = owners.of(chunk);
    const Coefs c = coefs[t];
    const long n = tb.c.numel[t], start = (long)(chunk - tb.c.first[t]) * kChunk;
    if (!tb.scales[t]) {
      if (start + kChunk <= n) update_chunk<T, true>(tb, t, start, n, factor, c, b);
      else update_chunk<T, false>(tb, t, start, n, factor, c, b);
      continue;
    }
    const long block = start / kBlock + wave;
    if (start + kChunk <= n) {
#pragma unroll
      for (int j = 0; j < kChunk / kBlock; j += 4) update_block<T, true>(tb, t, block + j, n, factor, c, b);
    } else {
      for (int j = 0; j < kChunk / kBlock && (block + j) * kBlock < n; j += 4)
        update_block<T, false>(tb, t, block + j, n, factor, c, b);
    }
  }
}

// ---- host side
// Fills the chunk map of n tensors; false if they have more chunks than a launch can count.
template <int N, typename Numel> bool fill_chunks(int n, Chunks<N>* c, const Numel& numel) {
  int64_t total = 0;
  for (int i = 0; i < N; ++i) {
    c->first[i] = INT32_MAX;
    if (i >= n) continue;
    c->numel[i] = numel(i);
    c->first[i] = (int)total;
    total += (c->numel[i] + kChunk - 1) / kChunk;
    if (total >= INT32_MAX) return false;
  }
  c->total = (int)total;
  return true;
}

int check_grad(const void* grad, int64_t numel, uintptr_t mask) {
  if (numel < 0) return UNETK_ERR_ARG;
  if (numel == 0) return UNETK_OK;
  if (numel >= (int64_t)(INT32_MAX - 1) * kChunk) return UNETK_ERR_SHAPE;
  if (!grad) return UNETK_ERR_ARG;
  return ((uintptr_t)grad & mask) ? UNETK_ERR_ALIGN : UNETK_OK;
}

int check_grads(void* const* grads, const int64_t* numel, int n, int dtype) {
  if (!grads || !numel || n <= 0) return UNETK_ERR_ARG;
  if (!unetk_dtype_ok(dtype)) return UNETK_ERR_DTYPE;
  for (int i = 0; i < n; ++i)
    if (const int rc = check_grad(grads[i], numel[i], unetk_esize(dtype) - 1)) return rc;
  return UNETK_OK;
}

struct Span {
  uintptr_t begin, end;
};
// Whether two of the spans share a byte; sorts them.
bool any_overlap(Span* spans, int n) {
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  for (int i = 1; i < n; ++i)
    if (spans[i].begin < spans[i - 1].end) return true;
  return false;
}

// Gradients that share memory would be scaled in any order, once or twice.  Those of one buffer or one allocation order (rising
// or falling) need no sorting, which takes 6 us for 130 in random order.
int check_apart(void* const* grads, const int64_t* numel, int n, int dtype) {
  const uintptr_t es = unetk_esize(dtype);
  const auto span = [&](int i) { return Span{(uintptr_t)grads[i], (uintptr_t)grads[i] + numel[i] * es}; };
  Span last{0, 0};
  bool rising = true, falling = true, first = true;
  for (int i = 0; i < n; ++i) {
    if (numel[i] == 0) continue;
    const Span s = span(i);
    rising &= first || s.begin >= last.end;
    falling &= first || s.end <= last.begin;
    last = s;
    first = false;
  }
  if (rising || falling) return UNETK_OK;
  Span* spans = new (std::nothrow) Span[n];
  if (!spans) return UNETK_ERR_TOO_LARGE;
  int k = 0;
  for (int i = 0; i < n; ++i)
    if (numel[i]) spans[k++] = span(i);
  const bool overlap = any_overlap(spans, k);
  delete[] spans;
  return overlap ? UNETK_ERR_ARG : UNETK_OK;
}

enum { kStep = 1, kMoments = 2 };                                    // what a call needs of a record
int check_tensors(const unetk_adamw_tensor* tensors, void* const* grads, int n, int dtype, int need) {
  if (!tensors || !grads || n <= 0) return UNETK_ERR_ARG;
  if (!unetk_dtype_ok(dtype)) return UNETK_ERR_DTYPE;
  const uintptr_t mask = unetk_esize(dtype) - 1;
  for (int i = 0; i < n; ++i) {
    const unetk_adamw_tensor& t = tensors[i];
    if (const int rc = check_grad(grads[i], t.numel, mask)) return rc;
    if ((need & kStep) && !t.step) return UNETK_ERR_ARG;
    if ((need & kStep) && ((uintptr_t)t.step & 3)) return UNETK_ERR_ALIGN;
    if (t.numel == 0 || !(need & kMoments)) continue;
    if (!t.param || !t.exp_avg || !t.exp_avg_sq) return UNETK_ERR_ARG;
    if ((uintptr_t)t.param & mask) return UNETK_ERR_ALIGN;
    if (!t.scales && (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 3)) return UNETK_ERR_ALIGN;
  }
  return UNETK_OK;
}

int check_clip(const double* partials, int64_t n_partials, double max_norm) {
  if (partials && !(max_norm >= 0.0)) return UNETK_ERR_ARG;
  if ((partials != nullptr) != (n_partials > 0) || n_partials < 0 || n_partials > INT32_MAX) return UNETK_ERR_ARG;
  return ((uintptr_t)partials & 7) ? UNETK_ERR_ALIGN : UNETK_OK;
}

inline int grid_of(int total, int most) { return total < 1 ? 1 : total < most ? total : most; }
inline int part_of(int n_tensors, int at, int most) { return n_tensors - at < most ? n_tensors - at : most; }

bool any_scales(const unetk_adamw_tensor* tensors, int n) {
  for (int i = 0; i < n; ++i)
    if (tensors[i].scales) return true;
  return false;
}

bool fill_update(const unetk_adamw_tensor* tensors, void* const* grads, int n, Update8Table* u) {
  for (int i = 0; i < n; ++i) {
    u->scales[i] = tensors[i].scales;
    u->param[i] = tensors[i].param;
    u->grad[i] = grads[i];
    u->exp_avg[i] = tensors[i].exp_avg;
    u->exp_avg_sq[i] = tensors[i].exp_avg_sq;
  }
  return fill_chunks(n, &u->c, [&](int i) { return tensors[i].numel; });
}

}  // namespace

extern "C" {

int64_t unetk_grad_partials(int n_tensors) {
  if (n_tensors <= 0) return UNETK_ERR_ARG;
  return ((int64_t)n_tensors + kPrepare - 1) / kPrepare * kSumsqGrid;      // of the smaller table
}

int64_t unetk_grad_sumsq(void* const* grads, const int64_t* numel, int n_tensors, int dtype, double* partials, void* stream) {
  int rc = check_grads(grads, numel, n_tensors, dtype);
  if (rc != UNETK_OK) return rc;
  if (!partials) return UNETK_ERR_ARG;
  if ((uintptr_t)partials & 7) return UNETK_ERR_ALIGN;
  if ((rc = check_apart(grads, numel, n_tensors, dtype)) != UNETK_OK) return rc;
  int64_t written = 0;
  for (int at = 0; at < n_tensors; at += kGrads) {
    const int n = part_of(n_tensors, at, kGrads);
    GradTable tb;
    if (!fill_chunks(n, &tb.c, [&](int i) { return numel[at + i]; })) return UNETK_ERR_SHAPE;
    for (int i = 0; i < n; ++i) tb.grad[i] = grads[at + i];
    const int grid = grid_of(tb.c.total, kSumsqGrid);
    UNETK_WITH_T(dtype, hipLaunchKernelGGL(grad_sumsq_kernel<T>, dim3(grid), dim3(256), 0, (hipStream_t)stream, tb,
                                           partials + written));
    UNETK_CHECK_LAUNCH();
    written += grid;
  }
  return written;
}

int unetk_grad_clip(void* const* grads, const int64_t* numel, int n_tensors, int dtype, const double* partials,
                    int64_t n_partials, double max_norm, float* norm_out, void* stream) {
  int rc = check_grads(grads, numel, n_tensors, dtype);
  if (rc == UNETK_OK) rc = check_clip(partials, n_partials, max_norm);
  if (rc != UNETK_OK) return rc;
  if (!partials) return UNETK_ERR_ARG;
  for (int at = (n_tensors - 1) / kGrads * kGrads; at >= 0; at -= kGrads) {
    const int n = part_of(n_tensors, at, kGrads);
    GradTable tb;
    if (!fill_chunks(n, &tb.c, [&](int i) { return numel[at + i]; })) return UNETK_ERR_SHAPE;
    for (int i = 0; i < n; ++i) tb.grad[i] = grads[at + i];
    const Clip clip{partials, (int)n_partials, (float)max_norm, nullptr, norm_out};
    UNETK_WITH_T(dtype, hipLaunchKernelGGL(grad_clip_kernel<T>, dim3(grid_of(tb.c.total, kClipGrid)), dim3(256), 0,
                                           (hipStream_t)stream, tb, clip));
    UNETK_CHECK_LAUNCH();
  }
  return UNETK_OK;
}

int64_t unetk_adamw_overlaps(const unetk_adamw_tensor* tensors, const uint8_t* element_size, int n_tensors) {
  if (!tensors || !element_size || n_tensors <= 0 || n_tensors > INT32_MAX / 5) return UNETK_ERR_ARG;
  Span* spans = new (std::nothrow) Span[5 * n_tensors];
  if (!spans) return UNETK_ERR_TOO_LARGE;
  int k = 0;
  const auto add = [&](const void* p, int64_t bytes) {
    if (bytes > 0) spans[k++] = Span{(uintptr_t)p, (uintptr_t)p + bytes};
  };
  for (int i = 0; i < n_tensors; ++i) {
    const unetk_adamw_tensor& t = tensors[i];
    add(t.step, sizeof(float));
    add(t.param, t.numel * element_size[i]);
    add(t.exp_avg, t.numel * (t.scales ? 1 : 4));
    add(t.exp_avg_sq, t.numel * (t.scales ? 1 : 4));
    if (t.scales) add(t.scales, (t.numel + kBlock - 1) / kBlock * 2);
  }
  const bool overlap = any_overlap(spans, k);
  delete[] spans;
  return overlap;
}

int64_t unetk_adamw_prepare(const unetk_adamw_tensor* tensors, void* const* grads, int n_tensors, int dtype, double lr,
                            const float* lr_dev, double beta1, double beta2, double weight_decay, int64_t seed,
                            const float* found_inf, float* coefs, double* partials, void* stream) {
  const int rc = check_tensors(tensors, grads, n_tensors, dtype, kStep);
  if (rc != UNETK_OK) return rc;
  if (!coefs) return UNETK_ERR_ARG;
  if (((uintptr_t)partials & 7) || ((uintptr_t)coefs & 15)) return UNETK_ERR_ALIGN;
  const Schedule h{lr, beta1, beta2, weight_decay, lr_dev, found_inf, (unsigned)seed};
  if (!partials) {
    for (int at = 0; at < n_tensors; at += kSteps) {
      const int n = part_of(n_tensors, at, kSteps);
      StepTable tb;
      for (int i = 0; i < n; ++i) tb.step[i] = tensors[at + i].step;
      hipLaunchKernelGGL(adamw_steps_kernel, dim3(1), dim3(kSteps), 0, (hipStream_t)stream, tb, n, h,
                         reinterpret_cast<Coefs*>(coefs) + at);
      UNETK_CHECK_LAUNCH();
    }
    return 0;
  }
  int64_t written = 0;
  for (int at = 0; at < n_tensors; at += kPrepare) {
    const int n = part_of(n_tensors, at, kPrepare);
    PrepareTable tb;
    if (!fill_chunks(n, &tb.c, [&](int i) { return tensors[at + i].numel; })) return UNETK_ERR_SHAPE;
    for (int i = 0; i < n; ++i) tb.grad[i] = grads[at + i], tb.step[i] = tensors[at + i].step;
    const int grid = grid_of(tb.c.total, kSumsqGrid);
    UNETK_WITH_T(dtype, hipLaunchKernelGGL(adamw_prepare_kernel<T>, dim3(grid), dim3(256), 0, (hipStream_t)stream, tb, n, h,
                                           reinterpret_cast<Coefs*>(coefs) + at, partials + written));
    UNETK_CHECK_LAUNCH();
    written += grid;
  }
  return written;
}

int unetk_adamw_update(const unetk_adamw_tensor* tensors, void* const* grads, int n_tensors, int dtype, double beta1,
                       double beta2, double eps, const float* grad_scale, const float* found_inf, const float* coefs,
                       const double* partials, int64_t n_partials, double max_norm, float* norm_out, void* stream) {
  int rc = check_tensors(tensors, grads, n_tensors, dtype, kMoments);
  if (rc == UNETK_OK) rc = check_clip(partials, n_partials, max_norm);
  if (rc != UNETK_OK) return rc;
  if (!coefs) return UNETK_ERR_ARG;
  if (eps > 0.0 && eps < FLT_MIN && any_scales(tensors, n_tensors)) return UNETK_ERR_ARG;        // see update_block
  const Betas b{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
  const Clip clip{partials, (int)n_partials, (float)max_norm, grad_scale, norm_out};
  for (int at = (n_tensors - 1) / kUpdate * kUpdate; at >= 0; at -= kUpdate) {
    const int n = part_of(n_tensors, at, kUpdate);
    Update8Table tb;
    if (!fill_update(tensors + at, grads + at, n, &tb)) return UNETK_ERR_SHAPE;
    const Coefs* co = reinterpret_cast<const Coefs*>(coefs) + at;
    const bool any8 = any_scales(tensors + at, n);
    const dim3 grid(grid_of(tb.c.total, any8 ? kUpdate8Grid : kUpdateGrid));
    if (any8)
      UNETK_WITH_T(dtype, hipLaunchKernelGGL(adamw8_update_kernel<T>, grid, dim3(256), 0, (hipStream_t)stream, tb, b, co,
                                             found_inf, clip));
    else
      UNETK_WITH_T(dtype, hipLaunchKernelGGL(adamw_update_kernel<T>, grid, dim3(256), 0, (hipStream_t)stream, tb, b, co,
                                             found_inf, clip));
    UNETK_CHECK_LAUNCH();
  }
  return UNETK_OK;
}

}  // extern "C"
