// Optimizer step over many tensors (include/unetk.h: "optimizer step over many tensors"): global gradient norm, clip,
// AdamW with fp32 moments or with e4m3 moments and one power-of-two scale per 256 elements.
//
// The tensors of a call travel as kernel arguments, up to kTable of them a launch: nothing is uploaded, kept or shared
// between calls, and a captured graph owns its copy.  Each tensor is cut into chunks of kChunk elements; a workgroup takes
// every gridDim.x-th chunk and finds its tensor with one compare per lane and a ballot over the tensors' first chunks.
#include "common.h"

namespace {

constexpr int kTable = 64;        // tensors a launch: one per lane of the search, < 4 KiB of arguments
constexpr int kChunk = 4096;      // elements: 16 per thread
constexpr int kBlock = 256;       // elements that share a scale: one wave, four per lane
constexpr int kSumsqGrid = 512;
constexpr int kUpdateGrid = 2048; // eight workgroups per CU

struct Chunks {
  int64_t numel[kTable];
  int first[kTable];              // first chunk of each tensor; INT32_MAX behind the last tensor
  int total;
};
struct GradTable {
  Chunks c;
  void* grad[kTable];
};
struct PrepareTable {
  Chunks c;
  const void* grad[kTable];
  float* step[kTable];
};
struct UpdateTable {
  Chunks c;
  void* param[kTable];
  const void* grad[kTable];
  void* exp_avg[kTable];
  void* exp_avg_sq[kTable];
};
struct Update8Table {
  UpdateTable u;
  void* scales[kTable];
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
static_assert(sizeof(Coefs) == 16, "unetk.h promises 16 bytes a tensor");

// The tensor that owns a chunk (wave-uniform).  Tensors without elements own none: their first chunk is the next one's.
__device__ __forceinline__ int owner_of(const Chunks& c, int chunk) {
  const unsigned long long below = __ballot(c.first[threadIdx.x & 63] <= chunk);
  return __builtin_amdgcn_readfirstlane(__popcll(below) - 1);
}

// Vectors of four elements at any element-aligned address (global accesses of gfx950 need no more).
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32u __attribute__((aligned(1)));
typedef unsigned short u16u __attribute__((aligned(1)));

template <typename T> __device__ __forceinline__ void load4(const void* base, long i, long n, float* out) {
  const T* p = static_cast<const T*>(base) + i;
  if (i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const f32x4u v = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = v[k];
    } else {
      const u16x4u v = *reinterpret_cast<const u16x4u*>(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = to_f32(__builtin_bit_cast(T, (unsigned short)v[k]));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = i + k < n ? to_f32(p[k]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store4(void* base, long i, long n, const float* in) {
  T* p = static_cast<T*>(base) + i;
  if (i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4u*>(p) = f32x4u{in[0], in[1], in[2], in[3]};
    } else {
      u16x4u v;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __builtin_bit_cast(unsigned short, from_f32<T>(in[k]));
      *reinterpret_cast<u16x4u*>(p) = v;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[k] = from_f32<T>(in[k]);
  }
}

// Sum over the workgroup's 256 threads in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double s, double* red) {
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  return red[0];
}

// Squares are exact in fp64 (24-bit significands), so nothing overflows or is lost on the way to the norm.
template <typename T, typename Table> __device__ double chunk_sumsq(const Table& tb) {
  double s = 0.0;
  for (int chunk = blockIdx.x; chunk < tb.c.total; chunk += gridDim.x) {
    const int t = owner_of(tb.c, chunk);
    const long n = tb.c.numel[t], base = (long)(chunk - tb.c.first[t]) * kChunk + threadIdx.x * 4;
#pragma unroll
    for (int j = 0; j < kChunk / 1024; ++j) {
      const long i = base + j * 1024;
      if (i >= n) break;
      float g[4];
      load4<T>(tb.grad[t], i, n, g);
#pragma unroll
      for (int k = 0; k < 4; ++k) s += (double)g[k] * g[k];
    }
  }
  return s;
}

template <typename T> __global__ __launch_bounds__(256) void grad_sumsq_kernel(GradTable tb, double* __restrict__ partials) {
  __shared__ double red[256];
  const double s = block_sum(chunk_sumsq<T>(tb), red);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ __forceinline__ unsigned mix32(unsigned h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// Counts the step and writes the bias corrections (workgroup 0, a thread per tensor); with SUM also the partial sums.
template <typename T, bool SUM>
__global__ __launch_bounds__(256) void adamw_prepare_kernel(PrepareTable tb, int n_tensors, double lr,
                                                            const float* __restrict__ lr_dev, double beta1, double beta2,
                                                            double weight_decay, unsigned seed,
                                                            const float* __restrict__ found_inf, Coefs* __restrict__ coefs,
                                                            double* __restrict__ partials) {
  if (blockIdx.x == 0 && threadIdx.x < n_tensors && !(found_inf && *found_inf != 0.f)) {
    const float t = *tb.step[threadIdx.x] + 1.f;
    *tb.step[threadIdx.x] = t;
    const double rate = lr_dev ? (double)*lr_dev : lr;
    Coefs c;
    c.step_size = (float)(rate / (1.0 - pow(beta1, (double)t)));
    c.root_correction = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
    c.decay = (float)(1.0 - rate * weight_decay);
    c.key = mix32((unsigned)(long)t * 0x9E3779B9u + seed);
    coefs[threadIdx.x] = c;
  }
  if constexpr (SUM) {
    __shared__ double red[256];
    const double s = block_sum(chunk_sumsq<T>(tb), red);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
  }
}

// What the gradient is multiplied by.  Every workgroup sums the partials in the same order, so all agree to the bit.  A norm
// that is not a number makes the coefficient one that is not either, as clip_grad_norm_ does.
__device__ __forceinline__ float grad_factor(const Clip& c) {
  const double inv_scale = c.grad_scale ? 1.0 / (double)*c.grad_scale : 1.0;
  if (!c.partials) return (float)inv_scale;
  __shared__ double red[256];
  double s = 0.0;
  for (int i = threadIdx.x; i < c.n_partials; i += 256) s += c.partials[i];
  const float norm = (float)(sqrt(block_sum(s, red)) * inv_scale);
  if (blockIdx.x == 0 && threadIdx.x == 0 && c.norm_out) *c.norm_out = norm;
  float coef = c.max_norm / (norm + 1e-6f);
  coef = coef > 1.f ? 1.f : coef;
  return (float)(coef * inv_scale);
}

template <typename T> __global__ __launch_bounds__(256) void grad_clip_kernel(GradTable tb, Clip clip) {
  const float coef = grad_factor(clip);
  if (coef == 1.f) return;
  for (int chunk = blockIdx.x; chunk < tb.c.total; chunk += gridDim.x) {
    const int t = owner_of(tb.c, chunk);
    const long n = tb.c.numel[t], base = (long)(chunk - tb.c.first[t]) * kChunk + threadIdx.x * 4;
#pragma unroll
    for (int j = 0; j < kChunk / 1024; ++j) {
      const long i = base + j * 1024;
      if (i >= n) break;
      float g[4];
      load4<T>(tb.grad[t], i, n, g);
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] *= coef;
      store4<T>(tb.grad[t], i, n, g);
    }
  }
}

struct Betas {
  float beta1, rest1, beta2, rest2, eps;
};

// One element: m and v in place, the new parameter returned; `root` is sqrt(v).
__device__ __forceinline__ float adamw_element(float p, float g, float& m, float& v, float& root, const Coefs& c, const Betas& b) {
  m = fmaf(b.rest1, g, b.beta1 * m);
  v = fmaf(b.rest2 * g, g, b.beta2 * v);
  root = sqrtf(v);
  return fmaf(-c.step_size, m / fmaf(root, c.root_correction, b.eps), p * c.decay);
}

template <typename T>
__global__ __launch_bounds__(256) void adamw_update_kernel(UpdateTable tb, Betas b, const Coefs* __restrict__ coefs,
                                                           const float* __restrict__ found_inf, Clip clip) {
  const float factor = grad_factor(clip);
  if (found_inf && *found_inf != 0.f) return;
  for (int chunk = blockIdx.x; chunk < tb.c.total; chunk += gridDim.x) {
    const int t = owner_of(tb.c, chunk);
    const Coefs c = coefs[t];
    const long n = tb.c.numel[t], base = (long)(chunk - tb.c.first[t]) * kChunk + threadIdx.x * 4;
#pragma unroll
    for (int j = 0; j < kChunk / 1024; ++j) {
      const long i = base + j * 1024;
      if (i >= n) break;
      float p[4], g[4], m[4], v[4];
      load4<T>(tb.param[t], i, n, p);
      load4<T>(tb.grad[t], i, n, g);
      load4<float>(tb.exp_avg[t], i, n, m);
      load4<float>(tb.exp_avg_sq[t], i, n, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float root;
        p[k] = adamw_element(p[k], g[k] * factor, m[k], v[k], root, c, b);
      }
      store4<T>(tb.param[t], i, n, p);
      store4<float>(tb.exp_avg[t], i, n, m);
      store4<float>(tb.exp_avg_sq[t], i, n, v);
    }
  }
}

// ---- 8-bit moments.  A scale is 2^k, kept as the byte e = 127 + k.  Multiplying by a power of two is exact, so a value that
// fits e4m3 comes back as it went in, and x * 2^-(k + 120) has its e4m3 code in the top bits of its fp32 word: exponent field
// and three bits of mantissa from bit 20 on, subnormals included (fp32's subnormals begin where e4m3's do then).
__device__ __forceinline__ unsigned finite_bits(float x) {          // |x| as an integer that orders like it; 0 unless finite
  const unsigned a = __float_as_uint(x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
  return v;
}
// 127 + the smallest k >= -127 with top <= 448 * 2^k = 1.75 * 2^(8 + k): the exponent goes up by one beyond a mantissa of 1.75
__device__ __forceinline__ int scale_byte(unsigned top) { return max((int)((top + 0x1fffffu) >> 23) - 8, 0); }

__device__ __forceinline__ unsigned encode(float x, int e, unsigned u16, unsigned lowest) {
  const unsigned w = __float_as_uint(__builtin_amdgcn_ldexpf(x, 7 - e));
  unsigned code = ((w & 0x7fffffffu) + (u16 << 4) + 8u) >> 20;
  if (x != 0.f) code = max(code, lowest);
  if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) code = 0x7fu;
  return code | (w >> 31 << 7);
}

template <typename T>
__global__ __launch_bounds__(256) void adamw8_update_kernel(Update8Table tb8, Betas b, const Coefs* __restrict__ coefs,
                                                            const float* __restrict__ found_inf, Clip clip) {
  const UpdateTable& tb = tb8.u;
  const float factor = grad_factor(clip);
  if (found_inf && *found_inf != 0.f) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int chunk = blockIdx.x; chunk < tb.c.total; chunk += gridDim.x) {
    const int t = owner_of(tb.c, chunk);
    const Coefs c = coefs[t];
    const long n = tb.c.numel[t];
    const long first_block = (long)(chunk - tb.c.first[t]) * (kChunk / kBlock) + wave;
#pragma unroll
    for (int j = 0; j < kChunk / kBlock / 4; ++j) {
      const long block = first_block + j * 4, i = block * kBlock + lane * 4;
      if (block * kBlock >= n) break;                               // wave-uniform
      float p[4], g[4], m[4], v[4], r[4];
      load4<T>(tb.param[t], i, n, p);
      load4<T>(tb.grad[t], i, n, g);
      unsigned char* mp = static_cast<unsigned char*>(tb.exp_avg[t]) + i;
      unsigned char* rp = static_cast<unsigned char*>(tb.exp_avg_sq[t]) + i;
      unsigned mc = 0, rc = 0;
      if (i + 4 <= n) {
        mc = *reinterpret_cast<const u32u*>(mp);
        rc = *reinterpret_cast<const u32u*>(rp);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k < n) mc |= (unsigned)mp[k] << 8 * k, rc |= (unsigned)rp[k] << 8 * k;
      }
      u16u* sp = reinterpret_cast<u16u*>(static_cast<unsigned char*>(tb8.scales[t]) + block * 2);
      const unsigned old = *sp;
      const float ms = __builtin_amdgcn_ldexpf(1.f, (int)(old & 255) - 127), rs = __builtin_amdgcn_ldexpf(1.f, (int)(old >> 8) - 127);
      {
        const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc, true);
        const auto r01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc, false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc, true);
        m[0] = m01[0] * ms; m[1] = m01[1] * ms; m[2] = m23[0] * ms; m[3] = m23[1] * ms;
        r[0] = r01[0] * rs; r[1] = r01[1] * rs; r[2] = r23[0] * rs; r[3] = r23[1] * rs;
      }
      unsigned mtop = 0, rtop = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = r[k] * r[k];
        p[k] = adamw_element(p[k], g[k] * factor, m[k], v[k], r[k], c, b);
        mtop = max(mtop, finite_bits(m[k]));
        rtop = max(rtop, finite_bits(r[k]));
      }
      const int me = scale_byte(wave_umax(mtop)), re = scale_byte(wave_umax(rtop));
      mc = rc = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned h = mix32((unsigned)(i + k) ^ (unsigned)((i + k) >> 32) ^ c.key);
        mc |= encode(m[k], me, h & 0xffffu, 0u) << 8 * k;
        rc |= encode(r[k], re, h >> 16, 1u) << 8 * k;
      }
      store4<T>(tb.param[t], i, n, p);
      if (i + 4 <= n) {
        *reinterpret_cast<u32u*>(mp) = mc;
        *reinterpret_cast<u32u*>(rp) = rc;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k < n) mp[k] = (unsigned char)(mc >> 8 * k), rp[k] = (unsigned char)(rc >> 8 * k);
      }
      if (lane == 0) *sp = (unsigned short)(me | re << 8);
    }
  }
}

// ---- host side
// Fills the chunk map of n tensors; false if they have more chunks than a launch can count.
template <typename Numel> bool fill_chunks(int n, Chunks* c, const Numel& numel) {
  int64_t total = 0;
  for (int i = 0; i < kTable; ++i) {
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

enum { kStep = 1, kMoments = 2, kScales = 4 };                       // what a call needs of a record
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
    if (!t.param || !t.exp_avg || !t.exp_avg_sq || ((need & kScales) && !t.scales)) return UNETK_ERR_ARG;
    if ((uintptr_t)t.param & mask) return UNETK_ERR_ALIGN;
    if (!(need & kScales) && (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 3)) return UNETK_ERR_ALIGN;
  }
  return UNETK_OK;
}

int check_clip(const double* partials, int64_t n_partials, double max_norm) {
  if (partials && !(max_norm >= 0.0)) return UNETK_ERR_ARG;
  if ((partials != nullptr) != (n_partials > 0) || n_partials < 0 || n_partials > INT32_MAX) return UNETK_ERR_ARG;
  return ((uintptr_t)partials & 7) ? UNETK_ERR_ALIGN : UNETK_OK;
}

inline int grid_of(int total, int most) { return total < 1 ? 1 : total < most ? total : most; }
inline int table_of(int n_tensors, int at) { return n_tensors - at < kTable ? n_tensors - at : kTable; }

bool fill_update(const unetk_adamw_tensor* tensors, void* const* grads, int n, UpdateTable* u) {
  for (int i = 0; i < n; ++i) {
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
  return ((int64_t)n_tensors + kTable - 1) / kTable * kSumsqGrid;
}

int64_t unetk_grad_sumsq(void* const* grads, const int64_t* numel, int n_tensors, int dtype, double* partials, void* stream) {
  const int rc = check_grads(grads, numel, n_tensors, dtype);
  if (rc != UNETK_OK) return rc;
  if (!partials) return UNETK_ERR_ARG;
  if ((uintptr_t)partials & 7) return UNETK_ERR_ALIGN;
  int64_t written = 0;
  for (int at = 0; at < n_tensors; at += kTable) {
    const int n = table_of(n_tensors, at);
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
  for (int at = 0; at < n_tensors; at += kTable) {
    const int n = table_of(n_tensors, at);
    GradTable tb;
    if (!fill_chunks(n, &tb.c, [&](int i) { return numel[at + i]; })) return UNETK_ERR_SHAPE;
    for (int i = 0; i < n; ++i) tb.grad[i] = grads[at + i];
    const Clip clip{partials, (int)n_partials, (float)max_norm, nullptr, norm_out};
    UNETK_WITH_T(dtype, hipLaunchKernelGGL(grad_clip_kernel<T>, dim3(grid_of(tb.c.total, kUpdateGrid)), dim3(256), 0,
                                           (hipStream_t)stream, tb, clip));
    UNETK_CHECK_LAUNCH();
  }
  return UNETK_OK;
}

int64_t unetk_adamw_prepare(const unetk_adamw_tensor* tensors, void* const* grads, int n_tensors, int dtype, double lr,
                            const float* lr_dev, double beta1, double beta2, double weight_decay, int64_t seed,
                            const float* found_inf, float* coefs, double* partials, void* stream) {
  const int rc = check_tensors(tensors, grads, n_tensors, dtype, kStep);
  if (rc != UNETK_OK) return rc;
  if (!coefs) return UNETK_ERR_ARG;
  if (((uintptr_t)partials & 7) || ((uintptr_t)coefs & 15)) return UNETK_ERR_ALIGN;
  int64_t written = 0;
  for (int at = 0; at < n_tensors; at += kTable) {
    const int n = table_of(n_tensors, at);
    PrepareTable tb;
    if (!fill_chunks(n, &tb.c, [&](int i) { return tensors[at + i].numel; })) return UNETK_ERR_SHAPE;
    for (int i = 0; i < n; ++i) tb.grad[i] = grads[at + i], tb.step[i] = tensors[at + i].step;
    Coefs* co = reinterpret_cast<Coefs*>(coefs) + at;
    if (partials) {
      const int grid = grid_of(tb.c.total, kSumsqGrid);
      UNETK_WITH_T(dtype, hipLaunchKernelGGL((adamw_prepare_kernel<T, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, tb, n,
                                             lr, lr_dev, beta1, beta2, weight_decay, (unsigned)seed, found_inf, co,
                                             partials + written));
      written += grid;
    } else {
      hipLaunchKernelGGL((adamw_prepare_kernel<float, false>), dim3(1), dim3(256), 0, (hipStream_t)stream, tb, n, lr, lr_dev,
                         beta1, beta2, weight_decay, (unsigned)seed, found_inf, co, (double*)nullptr);
    }
    UNETK_CHECK_LAUNCH();
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
  const Betas b{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
  const Clip clip{partials, (int)n_partials, (float)max_norm, grad_scale, norm_out};
  for (int at = 0; at < n_tensors; at += kTable) {
    UpdateTable tb;
    if (!fill_update(tensors + at, grads + at, table_of(n_tensors, at), &tb)) return UNETK_ERR_SHAPE;
    const Coefs* co = reinterpret_cast<const Coefs*>(coefs) + at;
    UNETK_WITH_T(dtype, hipLaunchKernelGGL(adamw_update_kernel<T>, dim3(grid_of(tb.c.total, kUpdateGrid)), dim3(256), 0,
                                           (hipStream_t)stream, tb, b, co, found_inf, clip));
    UNETK_CHECK_LAUNCH();
  }
  return UNETK_OK;
}

int unetk_adamw8_update(const unetk_adamw_tensor* tensors, void* const* grads, int n_tensors, int dtype, double beta1,
                        double beta2, double eps, const float* grad_scale, const float* found_inf, const float* coefs,
                        const double* partials, int64_t n_partials, double max_norm, float* norm_out, void* stream) {
  int rc = check_tensors(tensors, grads, n_tensors, dtype, kMoments | kScales);
  if (rc == UNETK_OK) rc = check_clip(partials, n_partials, max_norm);
  if (rc != UNETK_OK) return rc;
  if (!coefs) return UNETK_ERR_ARG;
  const Betas b{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
  const Clip clip{partials, (int)n_partials, (float)max_norm, grad_scale, norm_out};
  for (int at = 0; at < n_tensors; at += kTable) {
    const int n = table_of(n_tensors, at);
    Update8Table tb;
    if (!fill_update(tensors + at, grads + at, n, &tb.u)) return UNETK_ERR_SHAPE;
    for (int i = 0; i < n; ++i) tb.scales[i] = tensors[at + i].scales;
    const Coefs* co = reinterpret_cast<const Coefs*>(coefs) + at;
    UNETK_WITH_T(dtype, hipLaunchKernelGGL(adamw8_update_kernel<T>, dim3(grid_of(tb.u.c.total, kUpdateGrid)), dim3(256), 0,
                                           (hipStream_t)stream, tb, b, co, found_inf, clip));
    UNETK_CHECK_LAUNCH();
  }
  return UNETK_OK;
}

}  // extern "C"
