// Optimizer operators over lists of tensors: the gradient norm (and clipping by it) and the AdamW step, with moments in
// 32 bits or in 8.  One launch takes up to 84 tensors; their pointers travel in the kernel's arguments, so a call uploads
// nothing, keeps nothing from one call for the next, and can be captured into a graph.
//
//   g~ = g * grad_scale * coef                      coef = min(1, max_norm / (||g * grad_scale|| + 1e-6)), 1 without clipping
//   m' = b1 m + (1 - b1) g~,   v' = b2 v + (1 - b2) g~^2
//   w' = w (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// torch.optim.AdamW's update (decoupled decay); w is fp32, the parameter itself or the master copy of a half-precision one.
// This translation unit is built with -ffp-contract=off: the moments that become 8-bit codes are formed by separately
// rounded products and sums, so that the same operations anywhere else give the same codes.
#include "common.h"

#include <math.h>

#include <type_traits>

namespace oivae {

constexpr int kThreads = 256;
constexpr int kMomentBlock = OIVAE_ADAMW_BLOCK;   // a tensor's moments occupy whole blocks of 128 elements
constexpr int kSlots = 84;        // tensors of one AdamW launch: the argument struct stays below 4 KiB
constexpr int kOptions = 8;       // sets of (lr, decay, step) in one launch
constexpr int kChunk = 1024;      // elements of an AdamW workgroup: one vector of four a thread
constexpr int kGradSlots = 160;   // tensors of one norm / scaling launch
constexpr int kNormBlocks = 1024; // cap on the blocks of one norm launch (= its partial sums)
constexpr int kFewBlocks = 256;   // up to so many, the norm launch concludes the norm itself (grad_norm_one)
constexpr int kFewChunks = 2048;  // up to so many, the scaling blocks add the partial sums themselves (grad_clip_kernel)

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));        // parameters and gradients may start anywhere
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f2v __attribute__((vector_size(8)));

// ---- types of gradients and parameters ---------------------------------------------------------------------------------
__device__ __forceinline__ float half_to_float(uint16_t h, int type) {
  if (type == OIVAE_BF16) return __uint_as_float((uint32_t)h << 16);
  _Float16 x;
  __builtin_memcpy(&x, &h, 2);
  return (float)x;
}

// to nearest, ties to even: the copy a model computes with; the fp32 master keeps what this drops
__device__ __forceinline__ uint16_t float_to_half(float x, int type) {
  uint16_t h;
  if (type == OIVAE_BF16) {
    const __bf16 b = (__bf16)x;
    __builtin_memcpy(&h, &b, 2);
  } else {
    const _Float16 f = (_Float16)x;
    __builtin_memcpy(&h, &f, 2);
  }
  return h;
}

// four consecutive elements from i on; those at n and beyond are zero and not read
__device__ __forceinline__ f4 load4(const void* p, int type, int64_t i, int64_t n) {
  f4 x = {0.f, 0.f, 0.f, 0.f};
  if (type == OIVAE_F32) {
    const float* q = static_cast<const float*>(p) + i;
    if (i + 4 <= n) return *reinterpret_cast<const f4u*>(q);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (i + j < n) x[j] = q[j];
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    h4u h = {0, 0, 0, 0};
    if (i + 4 <= n) {
      h = *reinterpret_cast<const h4u*>(q);
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (i + j < n) h[j] = q[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = half_to_float(h[j], type);
  }
  return x;
}

__device__ __forceinline__ void store4(void* p, int type, int64_t i, int64_t n, f4 x) {
  if (type == OIVAE_F32) {
    float* q = static_cast<float*>(p) + i;
    if (i + 4 <= n) {
      *reinterpret_cast<f4u*>(q) = x;
      return;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (i + j < n) q[j] = x[j];
  } else {
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    h4u h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = float_to_half(x[j], type);
    if (i + 4 <= n) {
      *reinterpret_cast<h4u*>(q) = h;
      return;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (i + j < n) q[j] = h[j];
  }
}

// weights and moments: read once and written once a step, past the caches that the gradients -- just written by the backward
// pass -- may still be in
__device__ __forceinline__ f4 stream4(const float* p, int64_t i, int64_t n) {
  if (i + 4 <= n) return __builtin_nontemporal_load(reinterpret_cast<const f4u*>(p + i));
  return load4(p, OIVAE_F32, i, n);
}

__device__ __forceinline__ void stream4(float* p, int64_t i, int64_t n, f4 x) {
  if (i + 4 <= n) __builtin_nontemporal_store((f4u)x, reinterpret_cast<f4u*>(p + i));
  else store4(p, OIVAE_F32, i, n, x);
}

__device__ __forceinline__ void stream4_half(void* p, int type, int64_t i, int64_t n, f4 x) {
  if (i + 4 > n) {
    store4(p, type, i, n, x);
    return;
  }
  h4u h;
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = float_to_half(x[j], type);
  __builtin_nontemporal_store(h, reinterpret_cast<h4u*>(static_cast<uint16_t*>(p) + i));
}

// ---- gradient norm -----------------------------------------------------------------------------------------------------
struct GradSlot {
  void* g;
  int64_t n;
};
struct GradLaunch {
  GradSlot s[kGradSlots];
  uint32_t first[kGradSlots];   // a tensor's first chunk in the launch
  uint32_t info[kGradSlots];    // type | (index of its step counter + 1) << 2
  int32_t count;
  uint32_t chunks;
};

// elements of one chunk: 256 threads x four vectors of 16 bytes
__host__ __device__ inline int grad_chunk(int type) { return type == OIVAE_F32 || type == OIVAE_F32_WATCHED ? 4096 : 8192; }

// The last slot whose first chunk is not behind `chunk`, by bisection over scalar loads; the first chunks lie side by side, a few
// cache lines (within the slots: 0.7 us more of a 5 us launch).  A ballot over the lanes' comparisons saves 0.3 us there and
// costs 12 % of a large step.
template <class Launch>
__device__ __forceinline__ int find_slot(const Launch& a, uint32_t chunk) {
  int lo = 0, hi = a.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// the same sum in every thread, in an order of its own: within waves, then over waves
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[kThreads / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kThreads / 64; ++j) s += part[j];
  return s;
}

// eight 16-bit elements from i on; what lies at n and beyond is zero and not read
typedef uint16_t h8 __attribute__((ext_vector_type(8)));
typedef uint16_t h8u __attribute__((ext_vector_type(8), aligned(2)));
__device__ __forceinline__ h8 load8(const void* p, int64_t i, int64_t n) {
  const uint16_t* q = static_cast<const uint16_t*>(p) + i;
  if (i + 8 <= n) return *reinterpret_cast<const h8u*>(q);
  h8 x = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (i + j < n) x[j] = q[j];
  return x;
}

// Squares are formed and added in fp64 -- a large gradient's square leaves fp32's range -- in an order that depends on the
// sizes alone: per thread, per block, then over the blocks.  HBM-bound: 268M fp32 in 179 us with the sum over the blocks,
// 6.0 TB/s (2048 blocks 183, 4096 184); 67M bf16 in 29 us.
__device__ __forceinline__ double sum_of_squares(const GradLaunch& a) {
  double acc[2] = {0.0, 0.0};
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const int k = find_slot(a, c);
    const GradSlot& s = a.s[k];
    const int type = a.info[k] & 3;
    const int64_t base = (int64_t)(c - a.first[k]) * grad_chunk(type);
    if (type == OIVAE_F32 || type == OIVAE_F32_WATCHED) {
      f4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = load4(s.g, OIVAE_F32, base + (u * kThreads + threadIdx.x) * 4, s.n);
      if (type == OIVAE_F32_WATCHED) {   // zeros, which change no sum, or NaN where an element is not finite
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j & 1] += (double)(x[u][j] * 0.f);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j & 1] = fma((double)x[u][j], (double)x[u][j], acc[j & 1]);
      }
    } else {
      h8 h[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) h[u] = load8(s.g, base + (u * kThreads + threadIdx.x) * 8, s.n);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const double x = (double)half_to_float(h[u][j], type);
          acc[j & 1] = fma(x, x, acc[j & 1]);
        }
    }
  }
  return block_sum(acc[0] + acc[1]);
}

__device__ __forceinline__ float clip_coef(float norm, float max_norm) {
  const float limit = max_norm > 0.f ? max_norm / (norm + 1e-6f) : 1.f;
  return limit > 1.f ? 1.f : limit;   // NaN stays
}

struct Verdict {
  float grad_scale, max_norm;
  oivae_clip_t* clip;
  oivae_step_t* steps;
  double ln_b1, ln_b2;
  const uint32_t* bad;
};

// One block's work: the norm, the coefficient, whether the step is to be left out (a norm that is not finite, or a failed
// launch behind the gradients: common.h ErrWords), and -- unless it is -- the step counters of the launch's tensors, with
// their bias corrections.  `parts` < 0: the verdict stands already (further tensors of the same step).
__device__ __forceinline__ void conclude(const GradLaunch& a, const double* part, int parts, const Verdict& v) {
  int skip;
  if (parts >= 0) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const float norm = (float)(sqrt(block_sum(s)) * fabs((double)v.grad_scale));
    skip = (v.bad != nullptr && *v.bad != 0) || !(fabsf(norm) <= 3.402823466e38f);
    if (threadIdx.x == 0) {
      v.clip->norm = norm;
      v.clip->coef = clip_coef(norm, v.max_norm);
      v.clip->skip = skip;
      if (v.steps != nullptr) v.clip->skipped += skip;
    }
  } else {
    skip = v.clip->skip;
  }
  if (v.steps == nullptr || skip) return;
  for (int i = threadIdx.x; i < a.count; i += kThreads) {
    const uint32_t index = a.info[i] >> 2;
    if (index == 0) continue;
    oivae_step_t& q = v.steps[index - 1];
    const int t = q.t + 1;
    q.t = t;
    // 1 - b^t = -expm1(t ln b) keeps its digits where b^t is near 1 (t = 1, b2 = 0.999); in fp64, rounded once, as the host
    // does where it counts (run_adamw).  In fp32 the step of 136 tensors takes the same 22 us.
    q.inv_bc1 = (float)(1.0 / -expm1(t * v.ln_b1));
    q.inv_bc2_sqrt = (float)(1.0 / sqrt(-expm1(t * v.ln_b2)));
  }
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(GradLaunch a, double* __restrict__ part) {
  const double s = sum_of_squares(a);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(kThreads) void grad_norm_final(GradLaunch a, const double* __restrict__ part, int parts, Verdict v) {
  conclude(a, part, parts, v);
}

// Both in one launch, the last block to arrive concluding; clip->ticket is zero before and after.  For few blocks: their
// arrivals at one word take about 14 ns each, one after the other, a second launch about 4 us.
__global__ __launch_bounds__(kThreads) void grad_norm_one(GradLaunch a, double* part, Verdict v) {
  __shared__ int last;
  const double s = sum_of_squares(a);
  if (threadIdx.x == 0) {
    __hip_atomic_store(part + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t k = __hip_atomic_fetch_add(&v.clip->ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    last = k == gridDim.x - 1;
    if (last) __hip_atomic_store(&v.clip->ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (last) conclude(a, part, (int)gridDim.x, v);
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double* __restrict__ part, int parts, float* norm) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
  s = block_sum(s);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// g *= coef, one chunk a block.  With parts > 0 every block adds the partial sums itself, and the first one of the first launch
// leaves the norm: cheaper than a launch between for few chunks, the same or dearer for many.  Norm and scaling in us, every
// block / a launch between, fp32: 256 chunks 9.9 / 13.0, 800 12.5 / 14.6, 1500 15.6 / 17.4, 2048 17.9 / 19.6, 3000 28.5 / 28.6,
// 8264 80.7 / 80.6, 16384 152 / 149, 65600 605 / 589; bf16: 800 13.9 / 15.9, 2048 19.5 / 20.5, 3000 29.9 / 30.2, 16384 153 / 154.
// HBM-bound: 268M fp32 gradients in 410 us behind the norm
// (5.2 TB/s), 196 us with it when nothing has to be scaled.  One vector a thread scales them in 382 us, but then four times
// the waves start only to read that the coefficient is one (237 us with the norm).
__global__ __launch_bounds__(kThreads) void grad_clip_kernel(GradLaunch a, const double* __restrict__ part, int parts, float max_norm,
                                                             float* norm_out, int first) {
  float norm;
  if (parts > 0) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    norm = (float)sqrt(block_sum(s));
    if (first && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  } else {
    norm = *norm_out;
  }
  const float coef = clip_coef(norm, max_norm);
  if (coef == 1.f) return;   // a product with one
  const int k = find_slot(a, blockIdx.x);
  const GradSlot& s = a.s[k];
  const int type = a.info[k] & 3;
  const int64_t base = (int64_t)(blockIdx.x - a.first[k]) * grad_chunk(type), n = s.n;
  if (type == OIVAE_F32) {
    f4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = load4(s.g, OIVAE_F32, base + (u * kThreads + threadIdx.x) * 4, n);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = base + (u * kThreads + threadIdx.x) * 4;
      if (i < n) store4(s.g, OIVAE_F32, i, n, x[u] * coef);
    }
  } else {
    h8 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = load8(s.g, base + (u * kThreads + threadIdx.x) * 8, n);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = base + (u * kThreads + threadIdx.x) * 8;
      uint16_t* q = static_cast<uint16_t*>(s.g) + i;
      h8 y;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = float_to_half(half_to_float(x[u][j], type) * coef, type);
      if (i + 8 <= n) {
        *reinterpret_cast<h8u*>(q) = y;
      } else {
#pragma unroll
        for (int j = 0; j < 7; ++j)
          if (i + j < n) q[j] = y[j];
      }
    }
  }
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
struct AdamwSlot {
  void* p;
  const void* g;
  int64_t n;
  uint32_t at;      // its first moment block in the flat moment buffers
  uint32_t index;   // of its step counter, and of its random bits
  int32_t types;    // gradient | parameter << 8
  int32_t option;   // index into the launch's Options
};
struct Options {
  float lr, weight_decay;
  const float* lr_dev;
  float inv_bc1, inv_bc2_sqrt;
  int32_t step;     // t and its corrections, where no counters on the device are given
  int32_t pad;
};
struct AdamwLaunch {
  AdamwSlot s[kSlots];
  uint32_t first[kSlots];   // a tensor's first chunk in the launch
  Options opt[kOptions];
  oivae_adamw_state_t st;
  const oivae_clip_t* clip;
  const uint32_t* bad;
  float b1, omb1, b2, omb2, eps, gscale;
  uint32_t seed;
  int32_t count;
};
static_assert(sizeof(AdamwLaunch) <= 4096 && sizeof(GradLaunch) <= 4096, "kernel arguments of 4 KiB at most");

// What a workgroup needs of its tensor; everything uniform.  The two words that can call the step off are read here and
// looked at before the stores, so that the tensor's loads do not wait for them.
struct Tile {
  const void* g;
  void* p;
  int64_t n, flat, base;   // size; place in the moment buffers; the workgroup's first element
  uint32_t at, index, step, off;
  int gt, pt;
  float gscale, decay, step_size, inv_bc2_sqrt;
};

// a word behind a pointer of the argument struct, by a global load (the compiler takes such a pointer for a generic one)
template <class T>
__device__ __forceinline__ T word(const T* p) {
  return *(const __attribute__((address_space(1))) T*)p;
}

// Behind a norm the blocks run from the last element to the first: the caches still hold what the norm read last (268M bf16
// with clipping 1325 against 1378 us).
__device__ __forceinline__ Tile find_tile(const AdamwLaunch& a) {
  const uint32_t block = a.clip != nullptr ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const int k = find_slot(a, block);
  const AdamwSlot& s = a.s[k];
  const Options& q = a.opt[s.option];
  Tile r;
  r.off = (a.bad != nullptr ? word(a.bad) : 0u) | (a.clip != nullptr ? (uint32_t)word(&a.clip->skip) : 0u);
  r.g = s.g;
  r.p = s.p;
  r.n = s.n;
  r.at = s.at;
  r.flat = (int64_t)s.at * kMomentBlock;
  r.base = (int64_t)(block - a.first[k]) * kChunk;
  r.index = s.index;
  r.gt = s.types & 255;
  r.pt = s.types >> 8;
  float inv_bc1 = q.inv_bc1;
  r.inv_bc2_sqrt = q.inv_bc2_sqrt;
  r.step = (uint32_t)q.step;
  if (a.st.steps != nullptr) {
    const oivae_step_t* t = a.st.steps + s.index;
    inv_bc1 = word(&t->inv_bc1);
    r.inv_bc2_sqrt = word(&t->inv_bc2_sqrt);
    r.step = (uint32_t)word(&t->t);
  }
  const float lr = q.lr_dev != nullptr ? word(q.lr_dev) : q.lr;
  r.gscale = a.clip != nullptr ? a.gscale * word(&a.clip->coef) : a.gscale;
  r.decay = 1.f - lr * q.weight_decay;
  r.step_size = lr * inv_bc1;
  return r;
}

// One vector of four elements per thread and stream: the loads of a wave are 1 KiB pieces, and a small workgroup keeps its
// four streams short, so that many are in flight.  1024 elements a workgroup against 2048 / 4096 on 268M bf16 parameters:
// 1280 (5.9 TB/s) against 1364 / 1332 us; with weights and moments through the caches 1420 us.
__global__ __launch_bounds__(kThreads) void adamw32_kernel(AdamwLaunch a) {
  const Tile r = find_tile(a);
  const int64_t i = r.base + threadIdx.x * 4;
  if (i >= r.n) return;
  float* __restrict__ m = static_cast<float*>(a.st.m) + r.flat + i;   // moments occupy whole blocks: a vector that begins
  float* __restrict__ v = static_cast<float*>(a.st.v) + r.flat + i;   // inside the tensor ends inside its block
  float* __restrict__ w = r.pt == OIVAE_F32 ? static_cast<float*>(r.p) : a.st.master + r.flat;
  const f4 gi = load4(r.g, r.gt, i, r.n);
  f4 wi = stream4(w, i, r.n);
  f4 mi = __builtin_nontemporal_load(reinterpret_cast<const f4*>(m)), vi = __builtin_nontemporal_load(reinterpret_cast<const f4*>(v));
  if (r.off) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float g = gi[j] * r.gscale;
    mi[j] = fmaf(a.omb1, g, a.b1 * mi[j]);
    vi[j] = fmaf(a.omb2 * g, g, a.b2 * vi[j]);
    wi[j] = fmaf(-r.step_size, mi[j] / fmaf(sqrtf(vi[j]), r.inv_bc2_sqrt, a.eps), wi[j] * r.decay);
  }
  __builtin_nontemporal_store(mi, reinterpret_cast<f4*>(m));
  __builtin_nontemporal_store(vi, reinterpret_cast<f4*>(v));
  stream4(w, i, r.n, wi);
  if (r.pt != OIVAE_F32) stream4_half(r.p, r.pt, i, r.n, wi);
}

// ---- moments of 8 bits ----
// A block of 128 elements shares one power of two (scale byte b stands for 2^(b - 127), 255 for NaN); first moments are
// e4m3 codes (three digits, 17 binades: their sign and relative size matter), second moments e5m2 codes (31 binades of v:
// its root spans what m does).  Stochastic rounding: b2 = 0.999 moves v by a thousandth a step where a code's neighbours
// are an eighth or a quarter away -- to nearest, v would stand still; with random bits below the code's last place, cut
// off, its expectation moves as it should.  A v that is not zero keeps at least the smallest code, so that an element never
// divides a live first moment by eps alone.
//   The power of two brings the block's largest magnitude into [2^7, 2^8) (e4m3's largest is 448) or [2^14, 2^15) (57344),
// so rounding up never leaves the format.  v_cvt_sr_fp8_f32 / v_cvt_sr_bf8_f32 add the upper 20 or 21 of 32 random bits
// below the code's last place and cut off, subnormal codes included.
constexpr uint32_t kMix1 = 0x9E3779B1u, kMix2 = 0x6A09E667u, kMix3 = 0xBB67AE85u, kMix4 = 0x3C6EF373u;   // odd, with
// no pattern in their bits: a prime near 2^32 times the golden ratio's fraction, and 2^32 times the fractions of the roots of
// 2, 3 and 5

__device__ __forceinline__ uint32_t random_key(uint32_t seed, uint32_t step, uint32_t tensor) {
  uint32_t k = seed * kMix1 + step * kMix3 + tensor * kMix4;
  k = (k ^ (k >> 16)) * kMix2;
  k = (k ^ (k >> 15)) * kMix3;
  return k ^ (k >> 16);
}

// largest of 16 consecutive lanes' values, in each of them
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));    // lane ^ 1
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));    // lane ^ 2
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true));   // mirrored within 8
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, true));   // mirrored within 16
  return x;
}

// ... of 32
__device__ __forceinline__ uint32_t max32(uint32_t x) {
  x = max16(x);
  const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);   // rows 0, 0, 2, 2 and rows 1, 1, 3, 3
  return max((uint32_t)p[0], (uint32_t)p[1]);
}

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte << 23);
}

// 32 lanes hold one block, four elements each (one vector per thread and stream, as above).  With 16 lanes and 8 elements
// a lane the vectors of a wave are 32 bytes apart: 861 us on 268M bf16 parameters against 719.
//   kFast: hardware root and reciprocal (one unit in the last place each) instead of the correctly rounded ones, about a
// third of the instructions: 719 against 779 us (704 now, 6.1 TB/s).  The hardware root takes subnormals for zero: up to
// 1.1e-19, times 1 / sqrt(1 - b2) at most, in a denominator of at least eps.
template <bool kFast>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(AdamwLaunch a) {
  const Tile r = find_tile(a);
  const int64_t i = r.base + threadIdx.x * 4;
  const int64_t blk = i / kMomentBlock;
  if (blk >= (r.n + kMomentBlock - 1) / kMomentBlock) return;   // whole blocks, that is whole halves of a wave, leave together
  uint32_t* __restrict__ m = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.st.m) + r.flat + i);
  uint32_t* __restrict__ v = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.st.v) + r.flat + i);
  uint8_t* __restrict__ ms = a.st.m_scale + r.at + blk;
  uint8_t* __restrict__ vs = a.st.v_scale + r.at + blk;
  float* __restrict__ w = r.pt == OIVAE_F32 ? static_cast<float*>(r.p) : a.st.master + r.flat;
  const f4 gi = load4(r.g, r.gt, i, r.n);
  f4 wi = stream4(w, i, r.n);
  const int mc = (int)*m, vc = (int)*v;
  const float msc = scale_of(*ms), vsc = scale_of(*vs);
  if (r.off) return;
  const f2v m0 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, true);
  const f2v v0 = __builtin_amdgcn_cvt_pk_f32_bf8(vc, false), v1 = __builtin_amdgcn_cvt_pk_f32_bf8(vc, true);
  float mj[4] = {m0[0], m0[1], m1[0], m1[1]}, vj[4] = {v0[0], v0[1], v1[0], v1[1]};
  uint32_t mmax = 0, vmax = 0;   // magnitudes as bit patterns: a NaN is larger than everything and stays visible
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float g = gi[j] * r.gscale;
    mj[j] = (mj[j] * msc) * a.b1 + g * a.omb1;
    vj[j] = (vj[j] * vsc) * a.b2 + (g * g) * a.omb2;
    const float q = kFast ? mj[j] * __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(vj[j]), r.inv_bc2_sqrt, a.eps))
                          : mj[j] / fmaf(sqrtf(vj[j]), r.inv_bc2_sqrt, a.eps);
    wi[j] = fmaf(-r.step_size, q, wi[j] * r.decay);
    mmax = max(mmax, __float_as_uint(mj[j]) & 0x7FFFFFFFu);
    vmax = max(vmax, __float_as_uint(vj[j]) & 0x7FFFFFFFu);   // (a NaN may carry a sign)
  }
  const uint32_t me = max32(mmax) >> 23, ve = max32(vmax) >> 23;
  const uint32_t mb = me == 255u ? 255u : max(me, 8u) - 7u, vb = ve == 255u ? 255u : max(ve, 15u) - 14u;
  const uint32_t x0 = (uint32_t)i * kMix1 + (uint32_t)((uint64_t)i >> 32) * kMix4 + random_key(a.seed, r.step, r.index);
  int mq = 0, vq = 0;
  auto one = [&](auto J) {
    constexpr int j = decltype(J)::value;
    uint32_t x = x0 + (uint32_t)j * kMix1;
    x = (x ^ (x >> 14)) * kMix2;
    x ^= x >> 14;
    const float zm = __builtin_amdgcn_ldexpf(mj[j], 127 - (int)mb), zv = __builtin_amdgcn_ldexpf(vj[j], 127 - (int)vb);
    mq = __builtin_amdgcn_cvt_sr_fp8_f32(zm, (int)x, mq, j);
    vq = __builtin_amdgcn_cvt_sr_bf8_f32(vj[j] > 0.f ? fmaxf(zv, 0x1p-16f) : 0.f, (int)(x << 11), vq, j);
  };
  one(std::integral_constant<int, 0>{});
  one(std::integral_constant<int, 1>{});
  one(std::integral_constant<int, 2>{});
  one(std::integral_constant<int, 3>{});
  *m = (uint32_t)mq;
  *v = (uint32_t)vq;
  if ((threadIdx.x & 31) == 0) {
    *ms = (uint8_t)mb;
    *vs = (uint8_t)vb;
  }
  if (i >= r.n) return;
  stream4(w, i, r.n, wi);
  if (r.pt != OIVAE_F32) stream4_half(r.p, r.pt, i, r.n, wi);
}

// ---- host --------------------------------------------------------------------------------------------------------------
static bool aligned_to(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(a - 1)) == 0; }
static int size_of(int type) { return type == OIVAE_F32 || type == OIVAE_F32_WATCHED ? 4 : 2; }

constexpr uint32_t kMaxChunks = 0xFFFFFFu;   // workgroups of one launch: a grid's size in threads stays below 2^32
constexpr int64_t kMaxElements = (int64_t)kMaxChunks * kChunk;   // of one tensor

static int check_grad(const char* who, int32_t i, const void* g, int64_t n, int32_t type, int32_t last_type = OIVAE_F16) {
  if (n < 0) return fail(OIVAE_E_ARG, "%s: tensor %d has a negative size", who, i);
  if (type < OIVAE_F32 || type > last_type) return fail(OIVAE_E_ARG, "%s: tensor %d has unknown gradient type %d", who, i, type);
  if (n > 0 && !g) return fail(OIVAE_E_ARG, "%s: tensor %d has a null gradient", who, i);
  if (!aligned_to(g, size_of(type))) return fail(OIVAE_E_ARG, "%s: gradient %d is not aligned to its elements", who, i);
  if (n > kMaxElements) return fail(OIVAE_E_SHAPE, "%s: tensor %d has more than %lld elements", who, i, (long long)kMaxElements);
  return OIVAE_OK;
}

// gradients in launches of at most kGradSlots tensors and 2^22 chunks (64 GiB), in the caller's order
template <class F>
static int for_grad_launches(const oivae_grad_t* t, int32_t count, F&& launch) {
  GradLaunch a;
  a.count = 0;
  a.chunks = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (t[i].n == 0 && t[i].index < 0) continue;
    const int ck = grad_chunk(t[i].type);
    const uint32_t c = (uint32_t)((t[i].n + ck - 1) / ck);
    if (a.count == kGradSlots || (a.count > 0 && a.chunks + (uint64_t)c > (1u << 22))) {
      if (int rc = launch(a)) return rc;
      a.count = 0;
      a.chunks = 0;
    }
    a.s[a.count] = GradSlot{t[i].g, t[i].n};
    a.first[a.count] = a.chunks;
    a.info[a.count++] = (uint32_t)t[i].type | (uint32_t)(t[i].index + 1) << 2;
    a.chunks += c;
  }
  return a.count > 0 ? launch(a) : OIVAE_OK;
}

static int check_grads(const char* who, const oivae_grad_t* t, int32_t count, void* workspace, int64_t workspace_bytes,
                       int32_t last_type) {
  uint64_t seen[1024] = {0};   // indices below 65536: two threads would advance a counter named twice
  for (int32_t i = 0; i < count; ++i) {
    if (int rc = check_grad(who, i, t[i].g, t[i].n, t[i].type, last_type)) return rc;
    const int32_t k = t[i].index;
    if (k < -1 || k >= 1 << 29) return fail(OIVAE_E_ARG, "%s: tensor %d has index %d", who, i, k);
    if (k < 0 || k >= 65536) continue;
    if (seen[k >> 6] >> (k & 63) & 1) return fail(OIVAE_E_ARG, "%s: index %d appears twice", who, k);
    seen[k >> 6] |= (uint64_t)1 << (k & 63);
  }
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < oivae_grad_norm_workspace_bytes(count))
    return fail(OIVAE_E_WORKSPACE, "%s: workspace of %lld bytes (8-byte aligned) needed", who,
                (long long)oivae_grad_norm_workspace_bytes(count));
  return OIVAE_OK;
}

// the partial sums of all launches, one behind the other; their number into `parts`, that of the chunks into `chunks`
static int launch_partials(const char* who, const oivae_grad_t* t, int32_t count, double* part, int64_t room, int64_t* parts,
                           int64_t* chunks, hipStream_t st) {
  *parts = 0;
  *chunks = 0;
  return for_grad_launches(t, count, [&](const GradLaunch& a) -> int {
    if (a.chunks == 0) return OIVAE_OK;
    const unsigned blocks = a.chunks < (uint32_t)kNormBlocks ? a.chunks : (unsigned)kNormBlocks;
    if (*parts + blocks > room) return fail(OIVAE_E_WORKSPACE, "%s: workspace too small for gradients this large", who);
    hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(kThreads), 0, st, a, part + *parts);
    OIVAE_LAUNCH_CHECK();
    *parts += blocks;
    *chunks += a.chunks;
    return OIVAE_OK;
  });
}

static int run_adamw(const char* who, bool eight, const oivae_adamw_tensor_t* t, int32_t count, const oivae_adamw_group_t* groups,
                     int32_t n_groups, const oivae_adamw_state_t* st, double beta1, double beta2, double eps, float grad_scale,
                     uint32_t seed, const oivae_clip_t* clip, void* stream) {
  if (count < 0 || (count > 0 && (!t || !groups || !st))) return fail(OIVAE_E_ARG, "%s: bad argument", who);
  if (count == 0) return OIVAE_OK;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0))
    return fail(OIVAE_E_ARG, "%s: betas must be in [0, 1) and eps not negative", who);
  if (!st->m || !st->v || (eight && (!st->m_scale || !st->v_scale))) return fail(OIVAE_E_ARG, "%s: null moment buffer", who);
  if (!aligned_to(st->m, 16) || !aligned_to(st->v, 16) || !aligned_to(st->master, 16))
    return fail(OIVAE_E_ARG, "%s: moment and master buffers must be 16-byte aligned", who);
  int64_t place = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (int rc = check_grad(who, i, t[i].g, t[i].n, t[i].g_type)) return rc;
    if (t[i].p_type < OIVAE_F32 || t[i].p_type > OIVAE_F16) return fail(OIVAE_E_ARG, "%s: tensor %d has unknown type %d", who, i, t[i].p_type);
    if (t[i].n > 0 && !t[i].p) return fail(OIVAE_E_ARG, "%s: tensor %d is null", who, i);
    if (!aligned_to(t[i].p, size_of(t[i].p_type))) return fail(OIVAE_E_ARG, "%s: tensor %d is not aligned to its elements", who, i);
    if (t[i].p_type != OIVAE_F32 && !st->master) return fail(OIVAE_E_ARG, "%s: half-precision parameters need master weights", who);
    if (t[i].at < 0 || t[i].at % kMomentBlock != 0 || t[i].at / kMomentBlock > (int64_t)0xFFFFFFFFu)
      return fail(OIVAE_E_ARG, "%s: tensor %d's place in the moment buffers must be a multiple of %d", who, i, kMomentBlock);
    if (t[i].at < place) return fail(OIVAE_E_ARG, "%s: tensor %d's place in the moment buffers reaches into the one before it", who, i);
    place = t[i].at + t[i].n;
    if (t[i].group < 0 || t[i].group >= n_groups) return fail(OIVAE_E_ARG, "%s: tensor %d names group %d of %d", who, i, t[i].group, n_groups);
    if (t[i].index < 0) return fail(OIVAE_E_ARG, "%s: tensor %d has a negative index", who, i);
    if (!st->steps && t[i].step < 1) return fail(OIVAE_E_ARG, "%s: tensor %d is at step %d", who, i, t[i].step);
  }
  hipStream_t hs = (hipStream_t)stream;
  if (int rc = poll_error_word(who, hs)) return rc;
  AdamwLaunch a;
  a.st = *st;
  a.clip = clip;
  a.bad = bad_word_device();
  a.b1 = (float)beta1; a.omb1 = (float)(1.0 - beta1);   // the differences in double: 1 - 0.999f has lost five digits
  a.b2 = (float)beta2; a.omb2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.gscale = grad_scale;
  a.seed = seed;
  a.count = 0;
  const bool fast = eps * sqrt(1.0 - beta2) >= 3e-12;   // what the hardware root loses is under 2^-24 of the denominator
  struct { int32_t group, step; } names[kOptions];
  int32_t n_names = 0;
  uint32_t chunks = 0;
  auto launch = [&]() -> int {
    if (a.count == 0) return OIVAE_OK;
    if (!eight) hipLaunchKernelGGL(adamw32_kernel, dim3(chunks), dim3(kThreads), 0, hs, a);
    else if (fast) hipLaunchKernelGGL(adamw8_kernel<true>, dim3(chunks), dim3(kThreads), 0, hs, a);
    else hipLaunchKernelGGL(adamw8_kernel<false>, dim3(chunks), dim3(kThreads), 0, hs, a);
    OIVAE_LAUNCH_CHECK();
    a.count = 0;
    n_names = 0;
    chunks = 0;
    return OIVAE_OK;
  };
  for (int32_t i = 0; i < count; ++i) {
    if (t[i].n == 0) continue;
    const int32_t step = st->steps ? 0 : t[i].step;
    const uint64_t c = ((uint64_t)t[i].n + kChunk - 1) / kChunk;
    int32_t q = 0;
    while (q < n_names && (names[q].group != t[i].group || names[q].step != step)) ++q;
    if (a.count == kSlots || q == kOptions || (a.count > 0 && chunks + c > kMaxChunks)) {
      if (int rc = launch()) return rc;
      q = 0;
    }
    if (q == n_names) {
      names[n_names].group = t[i].group;
      names[n_names++].step = step;
      const oivae_adamw_group_t& g = groups[t[i].group];
      Options& o = a.opt[q];
      o.lr = g.lr; o.weight_decay = g.weight_decay; o.lr_dev = g.lr_dev;
      o.step = step;
      o.inv_bc1 = step ? (float)(1.0 / -expm1(step * log(beta1))) : 1.f;
      o.inv_bc2_sqrt = step ? (float)(1.0 / sqrt(-expm1(step * log(beta2)))) : 1.f;
    }
    a.first[a.count] = chunks;
    a.s[a.count++] = AdamwSlot{t[i].p, t[i].g, t[i].n, (uint32_t)(t[i].at / kMomentBlock), (uint32_t)t[i].index,
                               t[i].g_type | t[i].p_type << 8, q};
    chunks += (uint32_t)c;
  }
  return launch();
}

}  // namespace oivae

using namespace oivae;

// A launch takes kGradSlots tensors, fewer only where they would pass 64 GiB: eight more cover the 288 GB of a GPU.
extern "C" int64_t oivae_grad_norm_workspace_bytes(int32_t count) {
  return (int64_t)sizeof(double) * kNormBlocks * ((count <= 0 ? 0 : (count - 1) / kGradSlots) + 9);
}

extern "C" int oivae_grad_norm(const oivae_grad_t* grads, int32_t count, int32_t with_norm, float grad_scale, float max_norm,
                               oivae_clip_t* clip, oivae_step_t* steps, double beta1, double beta2, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  const char* who = "oivae_grad_norm";
  if (count < 0 || (count > 0 && !grads) || !clip) return fail(OIVAE_E_ARG, "%s: bad argument", who);
  if (steps && !(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
    return fail(OIVAE_E_ARG, "%s: betas must be in [0, 1)", who);
  if (int rc = check_grads(who, grads, count, workspace, workspace_bytes, OIVAE_F32_WATCHED)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (int rc = poll_error_word(who, st)) return rc;
  double* part = static_cast<double*>(workspace);
  const Verdict v{grad_scale, max_norm, clip, steps, steps ? log(beta1) : 0.0, steps ? log(beta2) : 0.0, bad_word_device()};
  int launches = 0;
  uint32_t chunks = 0;
  for_grad_launches(grads, count, [&](const GradLaunch& a) -> int {
    ++launches;
    chunks = a.chunks;
    return OIVAE_OK;
  });
  if (with_norm && launches == 1 && chunks > 0 && chunks <= (uint32_t)kFewBlocks)
    return for_grad_launches(grads, count, [&](const GradLaunch& a) -> int {
      hipLaunchKernelGGL(grad_norm_one, dim3(a.chunks), dim3(kThreads), 0, st, a, part, v);
      OIVAE_LAUNCH_CHECK();
      return OIVAE_OK;
    });
  int64_t parts = 0, all = 0;
  if (with_norm)
    if (int rc = launch_partials(who, grads, count, part, workspace_bytes / (int64_t)sizeof(double), &parts, &all, st)) return rc;
  bool first = true;
  auto conclude_launch = [&](const GradLaunch& a) -> int {
    if (!first && !steps) return OIVAE_OK;
    hipLaunchKernelGGL(grad_norm_final, dim3(1), dim3(kThreads), 0, st, a, (const double*)part, first ? (int)parts : -1, v);
    OIVAE_LAUNCH_CHECK();
    first = false;
    return OIVAE_OK;
  };
  if (launches > 0) return for_grad_launches(grads, count, conclude_launch);
  GradLaunch none;
  none.count = 0;
  none.chunks = 0;
  return conclude_launch(none);
}

extern "C" int oivae_clip_grad_norm(const oivae_grad_t* grads, int32_t count, float max_norm, float* norm, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const char* who = "oivae_clip_grad_norm";
  if (count < 0 || (count > 0 && !grads) || !norm) return fail(OIVAE_E_ARG, "%s: bad argument", who);
  if (int rc = check_grads(who, grads, count, workspace, workspace_bytes, OIVAE_F16)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (int rc = poll_error_word(who, st)) return rc;
  double* part = static_cast<double*>(workspace);
  int64_t parts = 0, chunks = 0;
  if (int rc = launch_partials(who, grads, count, part, workspace_bytes / (int64_t)sizeof(double), &parts, &chunks, st)) return rc;
  const bool scale = max_norm > 0.f && parts > 0;
  const bool few = scale && chunks <= kFewChunks;
  if (!few) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, (const double*)part, (int)parts, norm);
    OIVAE_LAUNCH_CHECK();
  }
  if (!scale) return OIVAE_OK;
  int first = 1;
  return for_grad_launches(grads, count, [&](const GradLaunch& a) -> int {
    if (a.chunks == 0) return OIVAE_OK;
    hipLaunchKernelGGL(grad_clip_kernel, dim3(a.chunks), dim3(kThreads), 0, st, a, (const double*)part, few ? (int)parts : 0, max_norm,
                       norm, first);
    OIVAE_LAUNCH_CHECK();
    first = 0;
    return OIVAE_OK;
  });
}

extern "C" int oivae_adamw_f32(const oivae_adamw_tensor_t* tensors, int32_t count, const oivae_adamw_group_t* groups, int32_t n_groups,
                               const oivae_adamw_state_t* state, double beta1, double beta2, double eps, float grad_scale,
                               const oivae_clip_t* clip, void* stream) {
  return run_adamw("oivae_adamw_f32", false, tensors, count, groups, n_groups, state, beta1, beta2, eps, grad_scale, 0, clip, stream);
}

extern "C" int oivae_adamw_f8(const oivae_adamw_tensor_t* tensors, int32_t count, const oivae_adamw_group_t* groups, int32_t n_groups,
                              const oivae_adamw_state_t* state, double beta1, double beta2, double eps, float grad_scale,
                              uint32_t seed, const oivae_clip_t* clip, void* stream) {
  return run_adamw("oivae_adamw_f8", true, tensors, count, groups, n_groups, state, beta1, beta2, eps, grad_scale, seed, clip, stream);
}
