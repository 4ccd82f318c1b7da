// adamw.hip -- AdamW (decoupled weight decay) over many tensors at once, with the moments in float32 or in 8 bits.
//
// Per element, in float32, g' = clip * g (clip: a device scalar, 1 without one):
//     m <- m + (1 - beta1) (g' - m)
//     v <- v beta2 + (1 - beta2) g' g'
//     p <- p (1 - lr wd) - (lr / (1 - beta1^t)) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// A clip factor that is NaN (gradients that are not finite) leaves parameters, moments and a count on the device as they were.
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
// What bounds both: HBM.  float32 moments move 28 B an element (bfloat16 parameters: 22), 8-bit ones 16 (10).  108.6 M float32 parameters
// 517 us (5.9 TB/s; four reads and three writes without arithmetic reach that too) and, 8-bit moments, 283 us (6.1); 201 M bfloat16
// ones 750 us (5.9), 402.8 M with 8-bit moments 682 us (5.9).  With bfloat16 parameters and 8-bit moments the vector units are next:
// hence one first hash multiplication for four elements, and the hardware's stochastic conversions.
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
  float root;        // 1 / sqrt(1 - beta2^t)
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

// ---- four elements of a lane.  AW_WHOLE: all of them lie in the tensor and the address suits one access, which goes past the
// caches: nothing but the gradients can be there from what ran before, and what is written is next read a whole pass later
// (4 / 32 / 128 M float32 parameters, float32 moments: 24.6 / 162 / 640 us, through the caches 32.0 / 184 / 706; right after the norm
// of the same gradients 20.7 / 144 / 603 and 25.0 / 160 / 663.  Only a list of tens of MB that is updated again and again with nothing
// in between would gain by the caches: 28.3 and 26.1 at 4 M.)
// AW_PART: element by element, `left` of them in the tensor; every load is made -- past the end the last element again, left > 0 or not --
// so that one wait does for all of a lane's.
enum { AW_PART = 0, AW_WHOLE = 1, AW_SOME = 2 };
template <typename E>
__device__ __forceinline__ void load_part(const E* p, int left, E (&e)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) e[k] = p[min(k, left - 1)];
}
template <typename V>
__device__ __forceinline__ V fetch(const V* p) { return __builtin_nontemporal_load(p); }
template <typename V>
__device__ __forceinline__ void put(V* p, const V& x) { __builtin_nontemporal_store(x, p); }
template <int HOW>
__device__ __forceinline__ f32x4 load4(const float* p, int left) {
  if constexpr (HOW != AW_PART) return fetch(reinterpret_cast<const f32x4*>(p));
  float e[4];
  load_part(p, left, e);
  return f32x4{e[0], e[1], e[2], e[3]};
}
template <int HOW>
__device__ __forceinline__ f32x4 load4(const bf16_t* p, int left) {
  if constexpr (HOW != AW_PART) {
    const u32x2 w = fetch(reinterpret_cast<const u32x2*>(p));
    return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)};
  }
  bf16_t e[4];
  load_part(p, left, e);
  return f32x4{bf16_to_f32(e[0]), bf16_to_f32(e[1]), bf16_to_f32(e[2]), bf16_to_f32(e[3])};
}
template <int HOW>
__device__ __forceinline__ uint32_t load4(const uint8_t* p, int left) {
  if constexpr (HOW != AW_PART) return fetch(reinterpret_cast<const uint32_t*>(p));
  uint8_t e[4];
  load_part(p, left, e);
  return (uint32_t)e[0] | (uint32_t)e[1] << 8 | (uint32_t)e[2] << 16 | (uint32_t)e[3] << 24;
}
template <int HOW>
__device__ __forceinline__ void store4(float* p, const f32x4& x, int left) {
  if constexpr (HOW != AW_PART) {
    put(reinterpret_cast<f32x4*>(p), x);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = x[k];
}
template <int HOW>
__device__ __forceinline__ void store4(uint8_t* p, uint32_t x, int left) {
  if constexpr (HOW != AW_PART) {
    put(reinterpret_cast<uint32_t*>(p), x);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = (uint8_t)(x >> (8 * k));
}

// The random bits mix32(index ^ key) of a lane's four elements, j = 0, 4, .. of a chunk that starts at a multiple of AW_CHUNK (a power
// of two below 2^16).  There the first round's x ^ (x >> 16) is s ^ j with one s for the whole chunk, and its product
// with the odd factor differs between the four elements by multiples of that factor which are the chunk's too: one multiplication
// instead of four.  (held(): the compiler is not to see where a value comes from.  It would undo this, and make a product that is shifted
// afterwards a second product; integer products take several times an addition's time.)
__device__ __forceinline__ uint32_t held(uint32_t x) {
  asm("" : "+v"(x));
  return x;
}
struct Noise {
  uint32_t s, c[4];
  __device__ __forceinline__ Noise(uint32_t chunk, uint32_t key) {
    const uint32_t x = chunk ^ key, t = x ^ (x >> 16);
    s = t & ~3u;
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = ((t & 3u) ^ k) * 0x455c2ed3u;
  }
  __device__ __forceinline__ void operator()(uint32_t j, uint32_t (&h)[4]) const {
    const uint32_t product = held((s ^ j) * 0x455c2ed3u);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t z = product + c[k];
      z = held((z ^ (z >> 15)) * 0x55a35cd1u);
      h[k] = z ^ (z >> 16);
    }
  }
};
static_assert((AW_CHUNK & (AW_CHUNK - 1)) == 0 && AW_CHUNK <= (1 << 16), "Noise");

// parameters: float32 as they are; bfloat16 up with the probability of the 16 bits cut off
template <int HOW>
__device__ __forceinline__ void store4_param(float* p, const f32x4& x, int left, const Noise&, uint32_t) { store4<HOW>(p, x, left); }
template <int HOW>
__device__ __forceinline__ void store4_param(bf16_t* p, const f32x4& x, int left, const Noise& noise, uint32_t j) {
  uint32_t h[4], r[4];
  noise(j, h);
#pragma unroll
  for (int k = 0; k < 4; ++k)                                  // (a NaN's bits must not run over into the sign)
    r[k] = x[k] == x[k] ? __float_as_uint(x[k]) + (h[k] & 0xffffu) : 0x7fc00000u;
  if constexpr (HOW != AW_PART) {
    put(reinterpret_cast<u32x2*>(p), u32x2{(r[0] >> 16) | (r[1] & 0xffff0000u), (r[2] >> 16) | (r[3] & 0xffff0000u)});
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = (bf16_t)(r[k] >> 16);
}

// m, v: one rounding per operation.  p: square root and reciprocal of the hardware (1 ulp each; they take numbers below 2^-126 for zero,
// so such a v goes through a square root of 2^100 v).
// Returns the bits, less one, of the smallest v above zero.
__device__ __forceinline__ uint32_t update(const AdamWHyper& h, float clip, f32x4& p, const f32x4& grad, f32x4& m, f32x4& v, float v_scale) {
  const float b = h.beta2 * v_scale;
  uint32_t least = ~0u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float g = grad[k] * clip;
    m[k] = m[k] + h.w1 * (g - m[k]);
    v[k] = v[k] * b + h.w2 * g * g;
    const uint32_t u = __float_as_uint(v[k]) - 1u;            // (zero: the largest)
    least = u < least ? u : least;
  }
  f32x4 root;
#pragma unroll
  for (int k = 0; k < 4; ++k) root[k] = __builtin_amdgcn_sqrtf(v[k]);
  if (least < 0x0d800000u) {                                   // 2^-100
#pragma unroll
    for (int k = 0; k < 4; ++k) root[k] = v[k] < 0x1p-100f ? __builtin_amdgcn_sqrtf(v[k] * 0x1p100f) * 0x1p-50f : root[k];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) p[k] = fmaf(-(h.step * m[k]), __builtin_amdgcn_rcpf(fmaf(root[k], h.root, h.eps)), p[k] * h.decay);
  return least;
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

// the largest over the wave, in a scalar register: rows of 16 lanes by shifts, then the rows by two broadcasts
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  auto step = [&](uint32_t o) { x = o > x ? o : x; };
  step(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));      // row_shr:1
  step(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
  step(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
  step(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
  step(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));     // row_bcast:15 into rows 1 and 3
  step(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));     // row_bcast:31 into rows 2 and 3
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ uint32_t largest(const f32x4& x, uint32_t below) {      // of the bits of |x| that are less than `below`
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t u = __float_as_uint(x[k]) & 0x7fffffffu;
    most = u > most && u < below ? u : most;
  }
  return wave_max(most);
}
// the block's power of two (biased): brings its largest magnitude to [2^room, 2^(room + 1))
__device__ __forceinline__ uint32_t block_power(uint32_t most, int room) {
  const int e = (int)(most >> 23) - room;
  return (uint32_t)(e < 1 ? 1 : e);
}

// What is not finite, among values that may be: NaN for NaN (and for infinity in e4m3, which has none), infinity in e5m2.
__device__ __forceinline__ uint32_t encode_special(float x, uint32_t code, bool e5m2) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  if (u < 0x7f800000u) return code;
  return (__float_as_uint(x) >> 24 & 0x80u) | (!e5m2 ? 0x7fu : u > 0x7f800000u ? 0x7eu : 0x7cu);
}

// A block's m and v as codes.  The conversions round stochastically by adding the upper 20 (e4m3) or 21 (e5m2) bits of their second
// operand to the part cut off -- also below the smallest normal value -- which is this file's rounding with 16 random bits and a half.
// least_v: at most the bits, less one, of the lane's smallest v above zero.  RARE: a v that would be rounded to zero is looked for before
// all are guarded against it (with bfloat16 parameters, where the vector units are as busy as HBM: 402.8 M of them 711 us, without the
// branch 737; with float32 ones they are not, and the branch costs: 108.6 M 287 us, without 283).
template <bool RARE>
__device__ __forceinline__ void encode4(const f32x4& m, const f32x4& v, uint32_t least_v, const uint32_t (&h)[4], uint32_t& mw, uint32_t& vw,
                                        uint32_t& me, uint32_t& ve) {
  uint32_t most_m = largest(m, ~0u), most_v = largest(v, ~0u);
  const bool finite = most_m < 0x7f800000u && most_v < 0x7f800000u;           // (of the whole block)
  if (!finite) { most_m = largest(m, 0x7f800000u); most_v = largest(v, 0x7f800000u); }
  me = block_power(most_m, 7);
  ve = block_power(most_v, 14);
  const float mi = power_of_two(254 - me), vi = power_of_two(254 - ve);
  float x[4], y[4];
  uint32_t a[4], b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = m[k] * mi;
    y[k] = v[k] * vi;
    a[k] = (h[k] << 16) | 0x8000u;
    b[k] = (h[k] & 0xffff0000u) | 0x8000u;
  }
  if (!RARE || __any(ve <= 16 || least_v < ((ve - 16) << 23))) {             // (above zero: not rounded to zero)
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = fmaxf(y[k], v[k] > 0.f ? 0x1p-16f : 0.f);
  }
  int p = 0, q = 0;
  p = __builtin_amdgcn_cvt_sr_fp8_f32(x[0], a[0], p, 0);
  p = __builtin_amdgcn_cvt_sr_fp8_f32(x[1], a[1], p, 1);
  p = __builtin_amdgcn_cvt_sr_fp8_f32(x[2], a[2], p, 2);
  p = __builtin_amdgcn_cvt_sr_fp8_f32(x[3], a[3], p, 3);
  q = __builtin_amdgcn_cvt_sr_bf8_f32(y[0], b[0], q, 0);
  q = __builtin_amdgcn_cvt_sr_bf8_f32(y[1], b[1], q, 1);
  q = __builtin_amdgcn_cvt_sr_bf8_f32(y[2], b[2], q, 2);
  q = __builtin_amdgcn_cvt_sr_bf8_f32(y[3], b[3], q, 3);
  mw = (uint32_t)p;
  vw = (uint32_t)q;
  if (!finite) {
    uint32_t mc = 0, vc = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mc |= encode_special(m[k], (mw >> (8 * k)) & 0xffu, false) << (8 * k);
      vc |= encode_special(v[k], (vw >> (8 * k)) & 0xffu, true) << (8 * k);
    }
    mw = mc;
    vw = vc;
  }
}

// UNITS blocks of each wave (AW_SOME: those of them that lie in the tensor as a whole); all their loads are under way before the first
// is used.
template <typename T, bool EIGHT, int HOW, int UNITS>
__device__ __forceinline__ void adamw_units(const AdamWArgs& a, int i, const AdamWHyper& h, float clip, uint32_t key, long chunk, int unit, int wave,
                                            int lane, long n) {
  using S = std::conditional_t<EIGHT, uint8_t, float>;
  using W = std::conditional_t<EIGHT, uint32_t, f32x4>;
  const Noise state_noise((uint32_t)chunk, key), param_noise((uint32_t)chunk, mix32(key ^ AW_PARAM_KEY));
  f32x4 P[UNITS], G[UNITS];
  W M[UNITS], V[UNITS];
  uint32_t ME[UNITS], VE[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const long o = chunk + ((unit + u) * AW_WAVES + wave) * AW_BLOCK;         // of the wave's block; uniform
    const int left = HOW != AW_PART ? 4 : (int)(n - o < AW_BLOCK ? n - o : AW_BLOCK) - lane * 4;
    if (HOW == AW_SOME && o + AW_BLOCK > n) break;
    P[u] = load4<HOW>(static_cast<const T*>(a.p[i]) + o + lane * 4, left);
    G[u] = load4<HOW>(static_cast<const T*>(a.g[i]) + o + lane * 4, left);
    M[u] = load4<HOW>(static_cast<const S*>(a.m[i]) + o + lane * 4, left);
    V[u] = load4<HOW>(static_cast<const S*>(a.v[i]) + o + lane * 4, left);
    if constexpr (EIGHT) {
      ME[u] = a.ms[i][o / AW_BLOCK];
      VE[u] = a.vs[i][o / AW_BLOCK];
    }
  }
  if (clip != clip) return;                                    // gradients that are not finite: the step is left out
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int j = ((unit + u) * AW_WAVES + wave) * AW_BLOCK + lane * 4;
    const long o = chunk + ((unit + u) * AW_WAVES + wave) * AW_BLOCK;
    const int left = HOW != AW_PART ? 4 : (int)(n - o < AW_BLOCK ? n - o : AW_BLOCK) - lane * 4;
    if (HOW == AW_SOME && o + AW_BLOCK > n) break;
    T* p = static_cast<T*>(a.p[i]) + o + lane * 4;
    S* m = static_cast<S*>(a.m[i]) + o + lane * 4;
    S* v = static_cast<S*>(a.v[i]) + o + lane * 4;
    if constexpr (EIGHT) {
      const uint32_t me0 = __builtin_amdgcn_readfirstlane(ME[u]), ve0 = __builtin_amdgcn_readfirstlane(VE[u]);
      f32x4 m4 = decode_e4m3(M[u]) * power_of_two(me0), v4 = decode_e5m2(V[u]);
      const uint32_t least_v = update(h, clip, P[u], G[u], m4, v4, power_of_two(ve0));
      if constexpr (HOW == AW_PART) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k >= left) m4[k] = v4[k] = 0.f;                                  // (behind the tensor's end: not of the block)
      }
      uint32_t r[4], mw, vw, me, ve;
      state_noise(j, r);
      encode4<sizeof(T) == 2>(m4, v4, least_v, r, mw, vw, me, ve);
      store4_param<HOW>(p, P[u], left, param_noise, j);
      store4<HOW>(m, mw, left);
      store4<HOW>(v, vw, left);
      if (lane == 0) {
        a.ms[i][o / AW_BLOCK] = (uint8_t)me;
        a.vs[i][o / AW_BLOCK] = (uint8_t)ve;
      }
    } else {
      update(h, clip, P[u], G[u], M[u], V[u], 1.f);
      store4_param<HOW>(p, P[u], left, param_noise, j);
      store4<HOW>(m, M[u], left);
      store4<HOW>(v, V[u], left);
    }
  }
}

template <typename T, bool EIGHT>
__global__ __launch_bounds__(64 * AW_WAVES) void adamw_kernel(AdamWArgs a) {
  float clip = 1.f;
  if (a.clip) clip = *a.clip;
  AdamWHyper h = a.h;
  if (a.hd) h = *a.hd;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int i = 0;
  for (int hi = a.nt; hi - i > 1;) {                           // the tensor of this workgroup: first[i] <= blockIdx.x < first[i + 1]
    const int mid = (i + hi) >> 1;
    if ((int)blockIdx.x >= a.first[mid]) i = mid;
    else hi = mid;
  }
  const long n = a.numel[i];
  const long chunk = (long)((int)blockIdx.x - a.first[i]) * AW_CHUNK;
  // (a chunk never crosses a multiple of 2^32: the upper half of the element index is the workgroup's)
  uint32_t key = mix32(h.base + (uint32_t)a.position[i]);
  if (chunk >> 32) key = mix32(key + (uint32_t)(chunk >> 32));
  constexpr uintptr_t PA = 4 * sizeof(T) - 1, SA = EIGHT ? 3 : 15;
  const bool aligned = (((uintptr_t)a.p[i] | (uintptr_t)a.g[i]) & PA) == 0 && (((uintptr_t)a.m[i] | (uintptr_t)a.v[i]) & SA) == 0;
  if (!aligned) {
#pragma unroll 1
    for (int u = 0; u < AW_UNITS; ++u)
      if (chunk + (u * AW_WAVES + wave) * AW_BLOCK < n) adamw_units<T, EIGHT, AW_PART, 1>(a, i, h, clip, key, chunk, u, wave, lane, n);
    return;
  }
  if (chunk + AW_CHUNK <= n) {
    adamw_units<T, EIGHT, AW_WHOLE, AW_UNITS>(a, i, h, clip, key, chunk, 0, wave, lane, n);
    return;
  }
  adamw_units<T, EIGHT, AW_SOME, AW_UNITS>(a, i, h, clip, key, chunk, 0, wave, lane, n);
  const int whole = (int)((n - chunk) / AW_BLOCK);             // the block behind them, if the tensor ends inside it
  if ((n - chunk) % AW_BLOCK && whole % AW_WAVES == wave) adamw_units<T, EIGHT, AW_PART, 1>(a, i, h, clip, key, chunk, whole / AW_WAVES, wave, lane, n);
}

int check_hyper(double lr, double beta1, double beta2, double eps, double weight_decay) {
  RM_REQUIRE(lr >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && weight_decay >= 0 && std::isfinite(lr) &&
                 std::isfinite(eps) && std::isfinite(weight_decay), "adamw: bad hyper-parameters");
  return REPMODE_OK;
}

// (an eps above zero stays so: the reciprocal takes what is below 2^-126 for zero)
__host__ __device__ __forceinline__ float float_eps(double eps) { return eps > 0 && eps < 0x1p-126 ? 0x1p-126f : (float)eps; }

// one thread: *step_dev += 1 unless the step is left out, and the constants of that step in the host path's double arithmetic
__global__ void adamw_hyper_kernel(long* __restrict__ step_dev, AdamWHyper* __restrict__ out, double lr, const float* __restrict__ lr_dev,
                                   double beta1, double beta2, double eps, double weight_decay, uint64_t seed,
                                   const float* __restrict__ clip) {
  if (threadIdx.x != 0 || blockIdx.x != 0) return;
  const long t = *step_dev + 1;
  if (!clip || *clip == *clip) *step_dev = t;
  const double l = lr_dev ? (double)*lr_dev : lr;
  const double bc1 = 1.0 - pow(beta1, (double)t), bc2 = 1.0 - pow(beta2, (double)t);
  out->w1 = (float)(1.0 - beta1);
  out->beta2 = (float)beta2;
  out->w2 = (float)(1.0 - beta2);
  out->root = (float)(1.0 / sqrt(bc2));
  out->eps = float_eps(eps);
  out->step = (float)(l / bc1);
  out->decay = (float)(1.0 - l * weight_decay);
  out->base = noise_base(seed, (uint64_t)t);
}

}  // namespace

extern "C" int repmode_adamw_hyper_clip_dev(long* step_dev, float* hyper_dev, double lr, const float* lr_dev, double beta1, double beta2,
                                            double eps, double weight_decay, unsigned long seed, const float* clip, void* stream) {
  RM_REQUIRE(step_dev && hyper_dev, "adamw_hyper_dev: null pointer");
  RM_REQUIRE(((uintptr_t)step_dev & 7) == 0 && ((uintptr_t)hyper_dev & 15) == 0 && (((uintptr_t)lr_dev | (uintptr_t)clip) & 3) == 0,
             "adamw_hyper_dev: misaligned buffers");
  if (int rc = check_hyper(lr, beta1, beta2, eps, weight_decay)) return rc;
  hipLaunchKernelGGL(adamw_hyper_kernel, dim3(1), dim3(64), 0, static_cast<hipStream_t>(stream), step_dev, reinterpret_cast<AdamWHyper*>(hyper_dev),
                     lr, lr_dev, beta1, beta2, eps, weight_decay, (uint64_t)seed, clip);
  RM_LAUNCH_CHECK("adamw_hyper_dev");
  return REPMODE_OK;
}
extern "C" int repmode_adamw_hyper_dev(long* step_dev, float* hyper_dev, double lr, const float* lr_dev, double beta1, double beta2,
                                       double eps, double weight_decay, unsigned long seed, void* stream) {
  return repmode_adamw_hyper_clip_dev(step_dev, hyper_dev, lr, lr_dev, beta1, beta2, eps, weight_decay, seed, nullptr, stream);
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
    a.h.root = (float)(1.0 / std::sqrt(bc2));
    a.h.eps = float_eps(eps);
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
  auto launch = [&](auto t, auto e) {
    hipLaunchKernelGGL((adamw_kernel<decltype(t), decltype(e)::value>), grid, block, 0, s, a);
  };
  if (dtype == REPMODE_F32) eight ? launch(float{}, std::true_type{}) : launch(float{}, std::false_type{});
  else eight ? launch(bf16_t{}, std::true_type{}) : launch(bf16_t{}, std::false_type{});
  RM_LAUNCH_CHECK("adamw_multi");
  return REPMODE_OK;
}
