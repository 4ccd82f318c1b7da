// adamw.hip -- AdamW (decoupled weight decay) over many tensors at once, with the moments in float32 or in 8 bits.
//
// Per element, in float32, g' = clip * g (clip: a device scalar, 1 without one):
//     m <- m + (1 - beta1) (g' - m)
//     v <- v beta2 + (1 - beta2) g' g'
//     p <- p (1 - lr wd) - (lr / (1 - beta1^t)) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// A clip factor that is NaN (gradients that are not finite) leaves parameters and moments as they were.
//
// 8-bit moments.  256 consecutive elements of a tensor (flat order) are a block; a block's m is held as e4m3 values and its v as
// e5m2 values, each times a power of two of its own (e8m0: one byte a block).  The powers are taken from the block's largest
// finite magnitude, so m spans 2^17 and v 2^31 of range below it.  Powers of two, so that an unchanged value keeps its place
// on the grid when the block's largest value moves: a moving scale would re-round every element at every step.
//   Rounding: stochastic, up with the probability of the part cut off.  To the nearest, beta2 = 0.999 moves v by less than
// half of a step (2^-3 relative) at every ordinary step, and v would never follow the gradients again; stochastic rounding
// keeps the mean of the moving average.  The parameters, where they are bfloat16, are rounded the same way and for the same
// reason: lr * m / sqrt(v) is below half of a bfloat16 step for most of them.  The random bits are a function of (seed, step,
// tensor's position, element), so a run repeats itself bit by bit.  A v above zero is never rounded to zero: m / (0 + eps)
// would throw its parameter away.  What is not finite stays so (e4m3 has no infinity: NaN) and is left out of the block's scale.
//
// What bounds both: HBM.  float32 moments move 28 B an element (bfloat16 parameters: 22), 8-bit ones 16 (10).
#include "common.h"

#include <cmath>

#pragma clang fp contract(off)      // (one rounding per operation: the 8-bit codes are then the formula's, not the compiler's)

namespace {

constexpr int AW_MAX = REPMODE_ADAMW_MAX;
constexpr int AW_BLOCK = REPMODE_ADAMW_BLOCK;       // elements of a block of 8-bit moments: one wave, 4 elements a lane
constexpr int AW_UNITS = 4;                         // blocks a wave has in flight
constexpr int AW_WAVES = 4;
constexpr int AW_CHUNK = AW_BLOCK * AW_UNITS * AW_WAVES;

struct AdamWHyper {
  float w1;          // 1 - beta1
  float beta2;
  float w2;          // 1 - beta2
  float bc2_sqrt;    // sqrt(1 - beta2^t)
  float eps;
  float step;        // lr / (1 - beta1^t)
  float decay;       // 1 - lr * weight_decay
  uint32_t base;     // of the random bits: a function of (seed, t)
};
static_assert(sizeof(AdamWHyper) == REPMODE_ADAMW_HYPER_FLOATS * sizeof(float), "hyper_dev holds an AdamWHyper");

// two multiply-xorshift rounds: a bijection of 32 bits whose output bits each depend on every input bit
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x455c2ed3u;
  x = (x ^ (x >> 15)) * 0x55a35cd1u;
  return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t noise_base(uint64_t seed, uint64_t step) {
  return mix32((uint32_t)step ^ mix32((uint32_t)(step >> 32) ^ mix32((uint32_t)seed ^ mix32((uint32_t)(seed >> 32) + 1u))));
}
constexpr uint32_t AW_PARAM_KEY = 0x6f002d25u;      // separates the parameter's random bits from the moments'

struct AdamWArgs {
  void* p[AW_MAX];
  const void* g[AW_MAX];
  void* m[AW_MAX];
  void* v[AW_MAX];
  uint8_t* ms[AW_MAX];           // 8-bit moments: the blocks' powers of two
  uint8_t* vs[AW_MAX];
  long numel[AW_MAX];
  int first[AW_MAX + 1];         // first workgroup of tensor i
  int nt;
  int position[AW_MAX];          // in the caller's whole list (random bits)
  AdamWHyper h;
  const AdamWHyper* hd;          // non-null: the step's constants come from device memory (a captured step)
  const float* clip;
};
static_assert(sizeof(AdamWArgs) <= 4096, "launch arguments");

template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, bool vec, long left) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      r = *reinterpret_cast<const f32x4*>(p);
    } else {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p);
      r = f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)};
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) r[k] = to_f32<T>(p[k]);
  }
  return r;
}

__device__ __forceinline__ uint32_t load4_bytes(const uint8_t* p, bool vec, long left) {
  if (vec && left >= 4) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t r = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) r |= (uint32_t)p[k] << (8 * k);
  return r;
}

__device__ __forceinline__ void store4(float* p, const f32x4& x, bool vec, long left) {
  if (vec && left >= 4) {
    *reinterpret_cast<f32x4*>(p) = x;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = x[k];
}

__device__ __forceinline__ void store4_bytes(uint8_t* p, uint32_t x, bool vec, long left) {
  if (vec && left >= 4) {
    *reinterpret_cast<uint32_t*>(p) = x;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = (uint8_t)(x >> (8 * k));
}

// float32 -> bfloat16, up with the probability of the 16 bits cut off
__device__ __forceinline__ bf16_t round_param(float x, uint32_t bits16) {
  uint32_t u = __float_as_uint(x);
  if ((u & 0x7f800000u) != 0x7f800000u) u += bits16;
  else if (u & 0x7fffffu) u |= 0x400000u;
  return (bf16_t)(u >> 16);
}

__device__ __forceinline__ void store4_param(float* p, const f32x4& x, bool vec, long left, uint32_t, uint32_t) { store4(p, x, vec, left); }
__device__ __forceinline__ void store4_param(bf16_t* p, const f32x4& x, bool vec, long left, uint32_t key, uint32_t index) {
  bf16_t r[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) r[k] = round_param(x[k], mix32((index + k) ^ key) & 0xffffu);
  if (vec && left >= 4) {
    *reinterpret_cast<u32x2*>(p) = u32x2{(uint32_t)r[0] | ((uint32_t)r[1] << 16), (uint32_t)r[2] | ((uint32_t)r[3] << 16)};
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = r[k];
}

__device__ __forceinline__ void update(const AdamWHyper& h, float clip, f32x4& p, const f32x4& grad, f32x4& m, f32x4& v) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float g = grad[k] * clip;
    m[k] = m[k] + h.w1 * (g - m[k]);
    v[k] = v[k] * h.beta2 + h.w2 * g * g;
    p[k] = p[k] * h.decay - h.step * (m[k] / (sqrtf(v[k]) / h.bc2_sqrt + h.eps));
  }
}

// the values of 4 e4m3 / e5m2 codes
__device__ __forceinline__ f32x4 decode_e4m3(uint32_t w) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return f32x4{a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ f32x4 decode_e5m2(uint32_t w) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_bf8(w, false), b = __builtin_amdgcn_cvt_pk_f32_bf8(w, true);
  return f32x4{a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ float power_of_two(uint32_t biased) { return __uint_as_float(biased << 23); }      // 2^(biased - 127), 1..254

// The largest finite magnitude's biased exponent over the wave's 256 elements, less `room`, at least 1: the block's power of two.
__device__ __forceinline__ uint32_t block_scale(const f32x4& x, int room) {
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t u = __float_as_uint(x[k]) & 0x7fffffffu;
    if (u < 0x7f800000u && u > most) most = u;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)most, off, 64);
    if (o > most) most = o;
  }
  const int e = (int)(most >> 23) - room;
  return (uint32_t)(e < 1 ? 1 : e);
}

// A magnitude x (already times the block's inverse power) as the code of a float with MAN mantissa bits and bias BIAS: `up`, of
// the 23 - MAN bits that are cut off, is added before the cut.  Below the smallest normal value the steps stay as they are
// there: adding that value puts them at the same place of the float32 mantissa.
template <int MAN, int BIAS, uint32_t INF, uint32_t NAN_>
__device__ __forceinline__ uint32_t encode(float x, uint32_t up) {
  const float least = __uint_as_float((uint32_t)(128 - BIAS) << 23);
  const bool low = x < least;
  const uint32_t u = __float_as_uint(low ? x + least : x);
  const uint32_t code = ((u + up) >> (23 - MAN)) - (low ? (uint32_t)(128 - BIAS) << MAN : (uint32_t)(127 - BIAS) << MAN);
  if ((u & 0x7f800000u) == 0x7f800000u) return (u & 0x7fffffu) ? NAN_ : INF;
  return code;
}

template <typename T, bool EIGHT>
__global__ __launch_bounds__(64 * AW_WAVES) void adamw_kernel(AdamWArgs a) {
  const float clip = a.clip ? *a.clip : 1.f;
  if (clip != clip) return;                                   // gradients that are not finite: the step is left out
  const AdamWHyper h = a.hd ? *a.hd : a.h;
  int i = 0;
  for (int lo = 0, hi = a.nt; hi - lo > 1;) {                  // the tensor of this workgroup: first[i] <= blockIdx.x < first[i + 1]
    const int mid = (lo + hi) >> 1;
    if ((int)blockIdx.x >= a.first[mid]) lo = mid;
    else hi = mid;
    i = lo;
  }
  const long n = a.numel[i];
  T* __restrict__ p = static_cast<T*>(a.p[i]);
  const T* __restrict__ g = static_cast<const T*>(a.g[i]);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long chunk = (long)((int)blockIdx.x - a.first[i]) * AW_CHUNK;
  // (a chunk never crosses a multiple of 2^32: the upper half of the element index is the workgroup's)
  uint32_t key = mix32(h.base + (uint32_t)a.position[i]);
  if (chunk >> 32) key = mix32(key + (uint32_t)(chunk >> 32));
  const bool vec_p = (((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) == 0;
  f32x4 P[AW_UNITS], G[AW_UNITS];
  if constexpr (!EIGHT) {
    float* __restrict__ m = static_cast<float*>(a.m[i]);
    float* __restrict__ v = static_cast<float*>(a.v[i]);
    const bool vec_s = (((uintptr_t)m | (uintptr_t)v) & 15) == 0;
    f32x4 M[AW_UNITS], V[AW_UNITS];
#pragma unroll
    for (int u = 0; u < AW_UNITS; ++u) {
      const long o = chunk + ((u * AW_WAVES + wave) * 64 + lane) * 4, left = n - o;
      P[u] = load4(p + o, vec_p, left);
      G[u] = load4(g + o, vec_p, left);
      M[u] = load4(m + o, vec_s, left);
      V[u] = load4(v + o, vec_s, left);
    }
#pragma unroll
    for (int u = 0; u < AW_UNITS; ++u) {
      const long o = chunk + ((u * AW_WAVES + wave) * 64 + lane) * 4, left = n - o;
      update(h, clip, P[u], G[u], M[u], V[u]);
      store4_param(p + o, P[u], vec_p, left, mix32(key ^ AW_PARAM_KEY), (uint32_t)o);
      store4(m + o, M[u], vec_s, left);
      store4(v + o, V[u], vec_s, left);
    }
  } else {
    uint8_t* __restrict__ m = static_cast<uint8_t*>(a.m[i]);
    uint8_t* __restrict__ v = static_cast<uint8_t*>(a.v[i]);
    uint8_t* __restrict__ ms = a.ms[i];
    uint8_t* __restrict__ vs = a.vs[i];
    const bool vec_s = (((uintptr_t)m | (uintptr_t)v) & 3) == 0;
    uint32_t M8[AW_UNITS], V8[AW_UNITS], ME[AW_UNITS], VE[AW_UNITS];
#pragma unroll
    for (int u = 0; u < AW_UNITS; ++u) {
      const long b = chunk / AW_BLOCK + u * AW_WAVES + wave, o = b * AW_BLOCK + lane * 4, left = n - o;
      ME[u] = VE[u] = 1;
      P[u] = load4(p + o, vec_p, left);
      G[u] = load4(g + o, vec_p, left);
      M8[u] = load4_bytes(m + o, vec_s, left);
      V8[u] = load4_bytes(v + o, vec_s, left);
      if (b * AW_BLOCK < n) { ME[u] = ms[b]; VE[u] = vs[b]; }
    }
#pragma unroll
    for (int u = 0; u < AW_UNITS; ++u) {
      const long b = chunk / AW_BLOCK + u * AW_WAVES + wave, o = b * AW_BLOCK + lane * 4, left = n - o;
      if (b * AW_BLOCK >= n) break;                            // (uniform over the wave)
      f32x4 M = decode_e4m3(M8[u]) * power_of_two(ME[u]), V = decode_e5m2(V8[u]) * power_of_two(VE[u]);
      update(h, clip, P[u], G[u], M, V);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k >= left) M[k] = V[k] = 0.f;                      // (behind the tensor's end: not of the block)
      const uint32_t me = block_scale(M, 7), ve = block_scale(V, 14);
      const float mi = power_of_two(254 - me), vi = power_of_two(254 - ve);
      uint32_t mw = 0, vw = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t r = mix32(((uint32_t)o + k) ^ key);
        uint32_t mc = encode<3, 7, 0x7fu, 0x7fu>(fabsf(M[k]) * mi, ((r & 0xffffu) << 4) + 8u);
        mc |= (__float_as_uint(M[k]) >> 24) & 0x80u;
        uint32_t vc = encode<2, 15, 0x7cu, 0x7eu>(V[k] * vi, ((r >> 16) << 5) + 16u);
        if (V[k] > 0.f && vc == 0) vc = 1;
        mw |= mc << (8 * k);
        vw |= vc << (8 * k);
      }
      store4_param(p + o, P[u], vec_p, left, mix32(key ^ AW_PARAM_KEY), (uint32_t)o);
      store4_bytes(m + o, mw, vec_s, left);
      store4_bytes(v + o, vw, vec_s, left);
      if (lane == 0) { ms[b] = (uint8_t)me; vs[b] = (uint8_t)ve; }
    }
  }
}

int check_hyper(double lr, double beta1, double beta2, double eps, double weight_decay) {
  RM_REQUIRE(lr >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && weight_decay >= 0 && std::isfinite(lr) &&
                 std::isfinite(eps) && std::isfinite(weight_decay), "adamw: bad hyper-parameters");
  return REPMODE_OK;
}

// one thread: *step_dev += 1, and the constants of that step in the host path's double arithmetic
__global__ void adamw_hyper_kernel(long* __restrict__ step_dev, AdamWHyper* __restrict__ out, double lr, const float* __restrict__ lr_dev,
                                   double beta1, double beta2, double eps, double weight_decay, uint64_t seed) {
  if (threadIdx.x != 0 || blockIdx.x != 0) return;
  const long t = *step_dev + 1;
  *step_dev = t;
  const double l = lr_dev ? (double)*lr_dev : lr;
  const double bc1 = 1.0 - pow(beta1, (double)t), bc2 = 1.0 - pow(beta2, (double)t);
  out->w1 = (float)(1.0 - beta1);
  out->beta2 = (float)beta2;
  out->w2 = (float)(1.0 - beta2);
  out->bc2_sqrt = (float)sqrt(bc2);
  out->eps = (float)eps;
  out->step = (float)(l / bc1);
  out->decay = (float)(1.0 - l * weight_decay);
  out->base = noise_base(seed, (uint64_t)t);
}

}  // namespace

extern "C" int repmode_adamw_hyper_dev(long* step_dev, float* hyper_dev, double lr, const float* lr_dev, double beta1, double beta2,
                                       double eps, double weight_decay, unsigned long seed, void* stream) {
  RM_REQUIRE(step_dev && hyper_dev, "adamw_hyper_dev: null pointer");
  RM_REQUIRE(((uintptr_t)step_dev & 7) == 0 && ((uintptr_t)hyper_dev & 15) == 0 && ((uintptr_t)lr_dev & 3) == 0, "adamw_hyper_dev: misaligned buffers");
  if (int rc = check_hyper(lr, beta1, beta2, eps, weight_decay)) return rc;
  hipLaunchKernelGGL(adamw_hyper_kernel, dim3(1), dim3(64), 0, static_cast<hipStream_t>(stream), step_dev, reinterpret_cast<AdamWHyper*>(hyper_dev),
                     lr, lr_dev, beta1, beta2, eps, weight_decay, (uint64_t)seed);
  RM_LAUNCH_CHECK("adamw_hyper_dev");
  return REPMODE_OK;
}

extern "C" int repmode_adamw_multi(int ntensors, int dtype, int state_bits, void* const* p, const void* const* g, void* const* m, void* const* m_scale,
                                   void* const* v, void* const* v_scale, const long* numel, const int* position, double lr, double beta1, double beta2,
                                   double eps, double weight_decay, long step, unsigned long seed, const float* hyper_dev, const float* clip,
                                   void* stream) {
  RM_REQUIRE(p && g && m && v && numel && position, "adamw_multi: null pointer");
  RM_REQUIRE(ntensors > 0 && ntensors <= AW_MAX, "adamw_multi: 1..%d tensors per call, got %d", AW_MAX, ntensors);
  RM_REQUIRE(dtype == REPMODE_F32 || dtype == REPMODE_BF16, "adamw_multi: bad dtype %d", dtype);
  RM_REQUIRE(state_bits == 32 || state_bits == 8, "adamw_multi: moments in 32 or 8 bits, got %d", state_bits);
  RM_REQUIRE(state_bits == 32 || (m_scale && v_scale), "adamw_multi: null pointer");
  const bool eight = state_bits == 8;
  AdamWArgs a{};
  a.clip = clip;
  if (hyper_dev) {
    a.hd = reinterpret_cast<const AdamWHyper*>(hyper_dev);
  } else {
    RM_REQUIRE(step >= 1, "adamw: step count starts at 1 (got %ld)", step);
    if (int rc = check_hyper(lr, beta1, beta2, eps, weight_decay)) return rc;
    const double bc1 = 1.0 - std::pow(beta1, (double)step), bc2 = 1.0 - std::pow(beta2, (double)step);
    a.h.w1 = (float)(1.0 - beta1);
    a.h.beta2 = (float)beta2;
    a.h.w2 = (float)(1.0 - beta2);
    a.h.bc2_sqrt = (float)std::sqrt(bc2);
    a.h.eps = (float)eps;
    a.h.step = (float)(lr / bc1);
    a.h.decay = (float)(1.0 - lr * weight_decay);
    a.h.base = noise_base(seed, (uint64_t)step);
  }
  a.nt = ntensors;
  long total = 0;
  const uintptr_t psize = dtype == REPMODE_F32 ? 4 : 2;
  for (int i = 0; i < ntensors; ++i) {
    RM_REQUIRE(p[i] && g[i] && m[i] && v[i] && numel[i] > 0 && (!eight || (m_scale[i] && v_scale[i])), "adamw_multi: bad tensor %d", i);
    RM_REQUIRE((((uintptr_t)p[i] | (uintptr_t)g[i]) & (psize - 1)) == 0 && (eight || (((uintptr_t)m[i] | (uintptr_t)v[i]) & 3) == 0),
               "adamw_multi: tensor %d is not aligned to its elements", i);
    a.p[i] = p[i]; a.g[i] = g[i]; a.m[i] = m[i]; a.v[i] = v[i]; a.numel[i] = numel[i]; a.position[i] = position[i];
    if (eight) { a.ms[i] = static_cast<uint8_t*>(m_scale[i]); a.vs[i] = static_cast<uint8_t*>(v_scale[i]); }
    a.first[i] = (int)total;
    total += (numel[i] + AW_CHUNK - 1) / AW_CHUNK;
    RM_REQUIRE(total < (1L << 31), "adamw_multi: grid too large");
  }
  a.first[ntensors] = (int)total;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)total), block(64 * AW_WAVES);
  if (dtype == REPMODE_F32 && !eight) hipLaunchKernelGGL((adamw_kernel<float, false>), grid, block, 0, s, a);
  else if (dtype == REPMODE_F32) hipLaunchKernelGGL((adamw_kernel<float, true>), grid, block, 0, s, a);
  else if (!eight) hipLaunchKernelGGL((adamw_kernel<bf16_t, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((adamw_kernel<bf16_t, true>), grid, block, 0, s, a);
  RM_LAUNCH_CHECK("adamw_multi");
  return REPMODE_OK;
}
