// Optimizer operators over lists of tensors: the gradient norm (and clipping by it) and the AdamW step, with moments in
// 32 bits or in 8.  One launch takes up to 76 tensors; their pointers travel in the kernel's arguments, so a call uploads
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

namespace oivae {

constexpr int kThreads = 256;
constexpr int kMomentBlock = OIVAE_ADAMW_BLOCK;   // a tensor's moments occupy whole blocks of 128 elements
constexpr int kSlots = 76;        // tensors of one AdamW launch: the argument struct stays below 4 KiB
constexpr int kGroups = 8;        // (lr, decay) pairs of one launch
constexpr int kGradSlots = 160;   // tensors of one norm / scaling launch
constexpr int kNormBlocks = 1024; // cap on the blocks of one norm launch (= its partial sums)
constexpr int kAdvance = 896;     // step counters advanced by one launch

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));        // parameters and gradients may start anywhere
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
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

// ---- gradient norm -----------------------------------------------------------------------------------------------------
struct GradSlot {
  void* g;
  int64_t n;
  uint32_t first;   // its first chunk in the launch
  int32_t type;
};
struct GradLaunch {
  GradSlot s[kGradSlots];
  int32_t count;
  uint32_t chunks;
};
constexpr int kGradChunk = 4096;   // elements

// the last slot whose first chunk is not behind `chunk`
template <class Launch>
__device__ __forceinline__ int find_slot(const Launch& a, uint32_t chunk) {
  int lo = 0, hi = a.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.s[mid].first <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[kThreads / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kThreads / 64; ++j) s += part[j];
  return s;
}

// squares are formed and added in fp64 (a large fp32 gradient's square leaves fp32's range), in an order that depends on
// the sizes alone: per thread, per block, then grad_norm_final over the blocks
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(GradLaunch a, double* __restrict__ part) {
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const GradSlot& s = a.s[find_slot(a, c)];
    const int64_t base = (int64_t)(c - s.first) * kGradChunk + (int64_t)threadIdx.x * 4;
    const int type = s.type;
    f4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = load4(s.g, type, base + u * kThreads * 4, s.n);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = fma((double)x[u][j], (double)x[u][j], acc);
  }
  acc = block_sum(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

struct Advance {
  int32_t which[kAdvance];
  int32_t count;
};

// One block: the norm, the coefficient, whether the step is to be left out (a norm that is not finite, or a failed launch
// behind the gradients: common.h ErrWords), and -- unless it is -- the step counters of the tensors that take part.
// `parts` < 0: the verdict in `clip` stands already (further counters of the same step).
__global__ __launch_bounds__(kThreads) void grad_norm_final(const double* __restrict__ part, int parts, float grad_scale,
                                                            float max_norm, oivae_clip_t* clip, int32_t* steps, Advance adv,
                                                            const uint32_t* __restrict__ bad) {
  int skip;
  if (parts >= 0) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    s = block_sum(s);
    const float norm = (float)(sqrt(s) * fabs((double)grad_scale));
    const float limit = max_norm > 0.f ? max_norm / (norm + 1e-6f) : 1.f;
    skip = (bad != nullptr && *bad != 0) || !(fabsf(norm) <= 3.402823466e38f);
    if (threadIdx.x == 0) {
      clip->norm = norm;
      clip->coef = limit > 1.f ? 1.f : limit;   // NaN stays
      clip->skip = skip;
      if (steps != nullptr) clip->skipped += skip;
    }
  } else {
    skip = clip->skip;
  }
  if (steps == nullptr || skip) return;
  for (int i = threadIdx.x; i < adv.count; i += kThreads) steps[adv.which[i]] += 1;
}

__global__ __launch_bounds__(kThreads) void grad_clip_kernel(GradLaunch a, const oivae_clip_t* __restrict__ clip) {
  const float coef = clip->coef;
  if (coef == 1.f) return;   // nothing to scale
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const GradSlot& s = a.s[find_slot(a, c)];
    const int64_t base = (int64_t)(c - s.first) * kGradChunk + (int64_t)threadIdx.x * 4;
    const int type = s.type;
    f4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = load4(s.g, type, base + u * kThreads * 4, s.n);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (base + u * kThreads * 4 < s.n) store4(s.g, type, base + u * kThreads * 4, s.n, x[u] * coef);
  }
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
struct AdamwSlot {
  void* p;
  const void* g;
  int64_t n;
  uint32_t at;      // its first moment block in the flat moment buffers
  uint32_t first;   // its first chunk in the launch
  uint32_t key;     // its index: of its step counter, and of its random bits
  int32_t step;     // t, where no counters on the device are given
  int32_t types;    // gradient | parameter << 8
  int32_t group;
};
struct AdamwLaunch {
  AdamwSlot s[kSlots];
  oivae_adamw_group_t grp[kGroups];
  oivae_adamw_state_t st;
  const oivae_clip_t* clip;
  const uint32_t* bad;
  float ln_b1, ln_b2, b1, omb1, b2, omb2, eps, gscale;
  uint32_t seed;
  int32_t count;
};
static_assert(sizeof(AdamwLaunch) <= 4096 && sizeof(GradLaunch) <= 4096, "kernel arguments of 4 KiB at most");
constexpr int kChunk = 4096;   // elements of one workgroup

struct StepScalars {
  float gscale, decay, step_size, inv_bc2_sqrt;
};

// bias corrections from t itself: 1 - b^t = -expm1(t ln b) keeps its digits where b^t is near 1 (t = 1, b2 = 0.999)
__device__ __forceinline__ StepScalars step_scalars(const AdamwLaunch& a, const AdamwSlot& s) {
  const float t = (float)(a.st.steps != nullptr ? a.st.steps[s.key] : s.step);
  const oivae_adamw_group_t& q = a.grp[s.group];
  const float lr = q.lr_dev != nullptr ? *q.lr_dev : q.lr;
  StepScalars r;
  r.gscale = a.clip != nullptr ? a.gscale * a.clip->coef : a.gscale;
  r.decay = 1.f - lr * q.weight_decay;
  r.step_size = lr / -expm1f(t * a.ln_b1);
  r.inv_bc2_sqrt = 1.f / sqrtf(-expm1f(t * a.ln_b2));
  return r;
}

__device__ __forceinline__ bool left_out(const AdamwLaunch& a) {
  return (a.bad != nullptr && *a.bad != 0) || (a.clip != nullptr && a.clip->skip != 0);
}

__global__ __launch_bounds__(kThreads) void adamw32_kernel(AdamwLaunch a) {
  if (left_out(a)) return;
  const AdamwSlot& s = a.s[find_slot(a, blockIdx.x)];
  const StepScalars r = step_scalars(a, s);
  const int gt = s.types & 255, pt = s.types >> 8;
  const int64_t n = s.n, flat = (int64_t)s.at * kMomentBlock;
  float* __restrict__ m = static_cast<float*>(a.st.m) + flat;
  float* __restrict__ v = static_cast<float*>(a.st.v) + flat;
  float* __restrict__ w = pt == OIVAE_F32 ? static_cast<float*>(s.p) : a.st.master + flat;
  const int64_t base = (int64_t)(blockIdx.x - s.first) * kChunk + (int64_t)threadIdx.x * 4;
  f4 gi[4], wi[4], mi[4], vi[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = base + u * kThreads * 4;
    gi[u] = load4(s.g, gt, i, n);
    wi[u] = load4(w, OIVAE_F32, i, n);
    mi[u] = f4{0.f, 0.f, 0.f, 0.f};
    vi[u] = f4{0.f, 0.f, 0.f, 0.f};
    if (i < n) {   // moments occupy whole blocks: a vector that begins inside the tensor ends inside its block
      mi[u] = *reinterpret_cast<const f4*>(m + i);
      vi[u] = *reinterpret_cast<const f4*>(v + i);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = base + u * kThreads * 4;
    if (i >= n) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float g = gi[u][j] * r.gscale;
      const float mj = fmaf(a.omb1, g, a.b1 * mi[u][j]);
      const float vj = fmaf(a.omb2 * g, g, a.b2 * vi[u][j]);
      const float d = fmaf(sqrtf(vj), r.inv_bc2_sqrt, a.eps);
      wi[u][j] = fmaf(-r.step_size, mj / d, wi[u][j] * r.decay);
      mi[u][j] = mj;
      vi[u][j] = vj;
    }
    *reinterpret_cast<f4*>(m + i) = mi[u];
    *reinterpret_cast<f4*>(v + i) = vi[u];
    store4(w, OIVAE_F32, i, n, wi[u]);
    if (pt != OIVAE_F32) store4(s.p, pt, i, n, wi[u]);
  }
}

// ---- moments of 8 bits ----
// A block of 128 elements shares one power of two (scale byte b stands for 2^(b - 127), 255 for NaN); first moments are
// e4m3 codes (three digits, 17 binades: their sign and relative size matter), second moments e5m2 codes (31 binades of v:
// its root spans what m does).  Stochastic rounding: b2 = 0.999 moves v by a thousandth a step where a code's neighbours
// are an eighth or a quarter away -- to nearest, v would stand still; with random bits below the code's last place, cut
// off, its expectation moves as it should.  A v that is not zero keeps at least the smallest code, so that an element never
// divides a live first moment by eps alone.
//   The power of two brings the block's largest magnitude into [2^7, 2^8) (e4m3's largest is 448) or [2^14, 2^15) (57344),
// so rounding up never leaves the format; and a second exact scaling puts the code's subnormal spacing on fp32's own, where
// code = (fp32 bits + random bits) >> 20 or 21, subnormal codes included.
constexpr uint32_t kMix1 = 0x9E3779B1u, kMix2 = 0x6A09E667u, kMix3 = 0xBB67AE85u, kMix4 = 0x3C6EF373u;   // 2^32 times the
// fractions of the golden ratio and of the roots of 2, 3 and 5, made odd

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

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte << 23);
}

__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return (a & 255u) | (b & 255u) << 8 | (c & 255u) << 16 | d << 24;
}

// 16 lanes hold one block, 8 elements each
__global__ __launch_bounds__(kThreads) void adamw8_kernel(AdamwLaunch a) {
  if (left_out(a)) return;
  const AdamwSlot& s = a.s[find_slot(a, blockIdx.x)];
  const StepScalars r = step_scalars(a, s);
  const int gt = s.types & 255, pt = s.types >> 8;
  const int64_t n = s.n, flat = (int64_t)s.at * kMomentBlock;
  uint8_t* __restrict__ m = static_cast<uint8_t*>(a.st.m) + flat;
  uint8_t* __restrict__ v = static_cast<uint8_t*>(a.st.v) + flat;
  uint8_t* __restrict__ ms = a.st.m_scale + s.at;
  uint8_t* __restrict__ vs = a.st.v_scale + s.at;
  float* __restrict__ w = pt == OIVAE_F32 ? static_cast<float*>(s.p) : a.st.master + flat;
  const uint32_t key = random_key(a.seed, (uint32_t)(a.st.steps != nullptr ? a.st.steps[s.key] : s.step), s.key);
  const int64_t end = (n + kMomentBlock - 1) / kMomentBlock * kMomentBlock;
#pragma unroll 1
  for (int u = 0; u < kChunk / (kThreads * 8); ++u) {
    const int64_t i = (int64_t)(blockIdx.x - s.first) * kChunk + u * kThreads * 8 + (int64_t)threadIdx.x * 8;
    if (i >= end) break;   // whole blocks, that is whole rows of 16 lanes, leave together
    const int64_t blk = i / kMomentBlock;
    const f4 g0 = load4(s.g, gt, i, n), g1 = load4(s.g, gt, i + 4, n);
    f4 w0 = load4(w, OIVAE_F32, i, n), w1 = load4(w, OIVAE_F32, i + 4, n);
    const u2 mc = *reinterpret_cast<const u2*>(m + i), vc = *reinterpret_cast<const u2*>(v + i);
    const float msc = scale_of(ms[blk]), vsc = scale_of(vs[blk]);
    float g[8], wj[8], mj[8], vj[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[j] = g0[j] * r.gscale; g[4 + j] = g1[j] * r.gscale;
      wj[j] = w0[j]; wj[4 + j] = w1[j];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f2v ml = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[h], false), mh = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[h], true);
      const f2v vl = __builtin_amdgcn_cvt_pk_f32_bf8((int)vc[h], false), vh = __builtin_amdgcn_cvt_pk_f32_bf8((int)vc[h], true);
      mj[4 * h] = ml[0]; mj[4 * h + 1] = ml[1]; mj[4 * h + 2] = mh[0]; mj[4 * h + 3] = mh[1];
      vj[4 * h] = vl[0]; vj[4 * h + 1] = vl[1]; vj[4 * h + 2] = vh[0]; vj[4 * h + 3] = vh[1];
    }
    uint32_t mmax = 0, vmax = 0;   // magnitudes as bit patterns: a NaN is larger than everything and stays visible
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mj[j] = (mj[j] * msc) * a.b1 + g[j] * a.omb1;
      vj[j] = (vj[j] * vsc) * a.b2 + (g[j] * g[j]) * a.omb2;
      const float d = sqrtf(vj[j]) * r.inv_bc2_sqrt + a.eps;
      wj[j] = wj[j] * r.decay - r.step_size * (mj[j] / d);
      mmax = max(mmax, __float_as_uint(mj[j]) & 0x7FFFFFFFu);
      vmax = max(vmax, __float_as_uint(vj[j]) & 0x7FFFFFFFu);
    }
    const uint32_t me = max16(mmax) >> 23, ve = max16(vmax) >> 23;
    const uint32_t mb = me == 255u ? 255u : max(me, 8u) - 7u, vb = ve == 255u ? 255u : max(ve, 15u) - 14u;
    const int mshift = 127 - (int)mb - 120, vshift = 127 - (int)vb - 112;
    const uint64_t e0 = (uint64_t)i;
    const uint32_t x0 = (uint32_t)e0 * kMix1 + (uint32_t)(e0 >> 32) * kMix4 + key;
    uint32_t mq[8], vq[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t x = x0 + (uint32_t)j * kMix1;
      x = (x ^ (x >> 14)) * kMix2;
      x ^= x >> 14;
      const uint32_t zm = __float_as_uint(__builtin_amdgcn_ldexpf(mj[j], mshift));
      const uint32_t zv = __float_as_uint(__builtin_amdgcn_ldexpf(vj[j], vshift));
      mq[j] = ((zm & 0x7FFFFFFFu) + (x >> 12)) >> 20 | (zm >> 31) << 7;
      vq[j] = max((zv + (x & 0x1FFFFFu)) >> 21, vj[j] > 0.f ? 1u : 0u);
    }
    const u2 mo = {pack_bytes(mq[0], mq[1], mq[2], mq[3]), pack_bytes(mq[4], mq[5], mq[6], mq[7])};
    const u2 vo = {pack_bytes(vq[0], vq[1], vq[2], vq[3]), pack_bytes(vq[4], vq[5], vq[6], vq[7])};
    *reinterpret_cast<u2*>(m + i) = mo;
    *reinterpret_cast<u2*>(v + i) = vo;
    if ((threadIdx.x & 15) == 0) {
      ms[blk] = (uint8_t)mb;
      vs[blk] = (uint8_t)vb;
    }
    w0 = f4{wj[0], wj[1], wj[2], wj[3]};
    w1 = f4{wj[4], wj[5], wj[6], wj[7]};
    if (i < n) store4(w, OIVAE_F32, i, n, w0);
    if (i + 4 < n) store4(w, OIVAE_F32, i + 4, n, w1);
    if (pt != OIVAE_F32) {
      if (i < n) store4(s.p, pt, i, n, w0);
      if (i + 4 < n) store4(s.p, pt, i + 4, n, w1);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
static bool aligned_to(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(a - 1)) == 0; }
static int size_of(int type) { return type == OIVAE_F32 ? 4 : 2; }

static int check_grad(const char* who, int32_t i, const void* g, int64_t n, int32_t type) {
  if (n < 0) return fail(OIVAE_E_ARG, "%s: tensor %d has a negative size", who, i);
  if (type < OIVAE_F32 || type > OIVAE_F16) return fail(OIVAE_E_ARG, "%s: tensor %d has unknown gradient type %d", who, i, type);
  if (n > 0 && !g) return fail(OIVAE_E_ARG, "%s: tensor %d has a null gradient", who, i);
  if (!aligned_to(g, size_of(type))) return fail(OIVAE_E_ARG, "%s: gradient %d is not aligned to its elements", who, i);
  if (n > (int64_t)1 << 40) return fail(OIVAE_E_SHAPE, "%s: tensor %d has more than 2^40 elements", who, i);
  return OIVAE_OK;
}

// gradients in launches of at most kGradSlots tensors and 2^30 chunks, in the caller's order
template <class F>
static int for_grad_launches(const oivae_grad_t* t, int32_t count, F&& launch) {
  GradLaunch a;
  a.count = 0;
  a.chunks = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (t[i].n == 0) continue;
    const uint32_t c = (uint32_t)((t[i].n + kGradChunk - 1) / kGradChunk);
    if (a.count == kGradSlots || (a.count > 0 && a.chunks + (uint64_t)c > (1u << 30))) {
      if (int rc = launch(a)) return rc;
      a.count = 0;
      a.chunks = 0;
    }
    a.s[a.count++] = GradSlot{t[i].g, t[i].n, a.chunks, t[i].type};
    a.chunks += c;
  }
  return a.count > 0 ? launch(a) : OIVAE_OK;
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
  for (int32_t i = 0; i < count; ++i) {
    if (int rc = check_grad(who, i, t[i].g, t[i].n, t[i].g_type)) return rc;
    if (t[i].p_type < OIVAE_F32 || t[i].p_type > OIVAE_F16) return fail(OIVAE_E_ARG, "%s: tensor %d has unknown type %d", who, i, t[i].p_type);
    if (t[i].n > 0 && !t[i].p) return fail(OIVAE_E_ARG, "%s: tensor %d is null", who, i);
    if (!aligned_to(t[i].p, size_of(t[i].p_type))) return fail(OIVAE_E_ARG, "%s: tensor %d is not aligned to its elements", who, i);
    if (t[i].p_type != OIVAE_F32 && !st->master) return fail(OIVAE_E_ARG, "%s: half-precision parameters need master weights", who);
    if (t[i].at < 0 || t[i].at % kMomentBlock != 0 || t[i].at / kMomentBlock > (int64_t)0xFFFFFFFFu)
      return fail(OIVAE_E_ARG, "%s: tensor %d's place in the moment buffers must be a multiple of %d", who, i, kMomentBlock);
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
  a.ln_b1 = (float)log(beta1); a.ln_b2 = (float)log(beta2);
  a.b1 = (float)beta1; a.omb1 = (float)(1.0 - beta1);   // the differences in double: 1 - 0.999f has lost five digits
  a.b2 = (float)beta2; a.omb2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.gscale = grad_scale;
  a.seed = seed;
  int32_t names[kGroups], n_names = 0;
  uint32_t chunks = 0;
  a.count = 0;
  auto launch = [&]() -> int {
    if (a.count == 0) return OIVAE_OK;
    if (eight) hipLaunchKernelGGL(adamw8_kernel, dim3(chunks), dim3(kThreads), 0, hs, a);
    else hipLaunchKernelGGL(adamw32_kernel, dim3(chunks), dim3(kThreads), 0, hs, a);
    OIVAE_LAUNCH_CHECK();
    a.count = 0;
    n_names = 0;
    chunks = 0;
    return OIVAE_OK;
  };
  for (int32_t i = 0; i < count; ++i) {
    if (t[i].n == 0) continue;
    const uint32_t c = (uint32_t)((t[i].n + kChunk - 1) / kChunk);
    int32_t q = 0;
    while (q < n_names && names[q] != t[i].group) ++q;
    // a grid's size in threads stays below 2^32
    if (a.count == kSlots || q == kGroups || (a.count > 0 && chunks + (uint64_t)c > 0xFFFFFFu)) {
      if (int rc = launch()) return rc;
      q = 0;
    }
    if (c > 0xFFFFFFu) return fail(OIVAE_E_SHAPE, "%s: tensor %d has more than %lld elements", who, i, (long long)0xFFFFFF * kChunk);
    if (q == n_names) {
      names[n_names++] = t[i].group;
      a.grp[q] = groups[t[i].group];
    }
    a.s[a.count++] = AdamwSlot{t[i].p, t[i].g, t[i].n, (uint32_t)(t[i].at / kMomentBlock), chunks, (uint32_t)t[i].index, t[i].step,
                               t[i].g_type | t[i].p_type << 8, q};
    chunks += c;
  }
  return launch();
}

}  // namespace oivae

using namespace oivae;

extern "C" int64_t oivae_grad_norm_workspace_bytes(int32_t count) {
  const int64_t launches = count <= 0 ? 1 : count;   // a launch takes at least one tensor (at most kGradSlots)
  return (int64_t)sizeof(double) * kNormBlocks * ((launches + kGradSlots - 1) / kGradSlots + 1);
}

extern "C" int oivae_grad_norm(const oivae_grad_t* grads, int32_t count, float grad_scale, float max_norm, oivae_clip_t* clip,
                               int32_t* steps, const int32_t* which, int32_t n_which, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  const char* who = "oivae_grad_norm";
  if (count < 0 || (count > 0 && !grads) || !clip || n_which < 0 || (n_which > 0 && (!which || !steps)))
    return fail(OIVAE_E_ARG, "%s: bad argument", who);
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < oivae_grad_norm_workspace_bytes(count))
    return fail(OIVAE_E_WORKSPACE, "%s: workspace of %lld bytes (8-byte aligned) needed", who,
                (long long)oivae_grad_norm_workspace_bytes(count));
  for (int32_t i = 0; i < count; ++i)
    if (int rc = check_grad(who, i, grads[i].g, grads[i].n, grads[i].type)) return rc;
  for (int32_t i = 0; i < n_which; ++i)
    if (which[i] < 0) return fail(OIVAE_E_ARG, "%s: negative step counter index", who);
  hipStream_t st = (hipStream_t)stream;
  if (int rc = poll_error_word(who, st)) return rc;
  double* part = static_cast<double*>(workspace);
  const int64_t room = workspace_bytes / (int64_t)sizeof(double);
  int64_t parts = 0;
  if (int rc = for_grad_launches(grads, count, [&](const GradLaunch& a) -> int {
        const unsigned blocks = a.chunks < (uint32_t)kNormBlocks ? a.chunks : (unsigned)kNormBlocks;
        if (parts + blocks > room) return fail(OIVAE_E_WORKSPACE, "%s: workspace too small for tensors this large", who);
        hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(kThreads), 0, st, a, part + parts);
        OIVAE_LAUNCH_CHECK();
        parts += blocks;
        return OIVAE_OK;
      }))
    return rc;
  int32_t done = 0;
  do {
    Advance adv;
    adv.count = n_which - done < kAdvance ? n_which - done : kAdvance;
    for (int32_t i = 0; i < adv.count; ++i) adv.which[i] = which[done + i];
    hipLaunchKernelGGL(grad_norm_final, dim3(1), dim3(kThreads), 0, st, (const double*)part, done == 0 ? (int)parts : -1,
                       grad_scale, max_norm, clip, steps, adv, bad_word_device());
    OIVAE_LAUNCH_CHECK();
    done += adv.count;
  } while (done < n_which);
  return OIVAE_OK;
}

extern "C" int oivae_grad_clip(const oivae_grad_t* grads, int32_t count, const oivae_clip_t* clip, void* stream) {
  const char* who = "oivae_grad_clip";
  if (count < 0 || (count > 0 && !grads) || !clip) return fail(OIVAE_E_ARG, "%s: bad argument", who);
  for (int32_t i = 0; i < count; ++i)
    if (int rc = check_grad(who, i, grads[i].g, grads[i].n, grads[i].type)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (int rc = poll_error_word(who, st)) return rc;
  return for_grad_launches(grads, count, [&](const GradLaunch& a) -> int {
    const unsigned blocks = a.chunks < 8192u ? a.chunks : 8192u;
    hipLaunchKernelGGL(grad_clip_kernel, dim3(blocks), dim3(kThreads), 0, st, a, clip);
    OIVAE_LAUNCH_CHECK();
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
