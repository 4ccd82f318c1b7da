// balance.hip -- the load-balance loss of a router (or of a mixture's gates) with its per-expert counts, forward and backward.
//
// Logits x[g][n][e], any strides: G groups (sequences, or 1) of N rows over E experts, float32 or bfloat16.  For the rows of a
// group that count -- not masked, not all -inf; there are N_g of them --
//     p_n = softmax(x_n)                C_n = the top_k largest of x_n (ties: the lowest index first; never a -inf)
//     f_ge = |{n : e in C_n}| / (top_k N_g)          P_ge = (1 / N_g) sum_n p_ne
//     loss = coef E (1 / G') sum_g sum_e f_ge P_ge    G': the groups with N_g > 0
// and, the counts being constants,
//     dx_ne = up * p_ne (w_ge - sum_j w_gj p_nj),     w_ge = coef E f_ge / (G' N_g).
//
// A row's E values live in the registers of LPR lanes, 8 (E > 512: 16) a lane, so a row is read once and softmax, choice and
// the lane's share of the column sums (probabilities in float32, counts as integers) need no memory.  A workgroup walks many
// rows and writes one partial per expert; one launch adds the partials of a group's columns in a fixed order in float64, one
// more makes the loss of them where there are several such workgroups.  No float atomics: a run repeats itself bit by bit.
// The backward pass reads the logits again and needs nothing of a row but its logits.
// What bounds it: HBM for the backward pass (one read, one write), the choice's rounds for wide forward passes.
#include "common.h"

#include <cmath>

namespace {

constexpr int BL_WAVES = 4;
constexpr int BL_MAX_E = REPMODE_BALANCE_MAX_EXPERTS;
constexpr int BL_FINISH = 256;           // threads of the finish: 64 columns, 4 shares of the partials

struct BalanceArgs {
  const void* x;
  const uint8_t* mask;
  void* dx;                  // backward
  const float* weight;       // backward: w_ge but for 1 / G', which stands behind them
  const float* up;           // backward
  long sg, sn, se;           // strides of x (elements)
  long mg, mn;               // strides of the mask
  long dg, dn, de;           // strides of dx
  long rows;
  int groups, experts, top_k;
  int blocks;                // workgroups per group
  float* psum;               // forward: [groups][blocks][experts]
  int* count;                //          the same shape
  int* valid;                //          [groups][blocks]
};

// e^x for x <= 0, NaN and -inf: 2^t with t = x log2(e) in two parts (t's rounding alone would cost |x| 2^-24 of the result)
__device__ __forceinline__ float exp_neg(float x) {
  const float t = x * 1.44269504f, lo = fmaf(x, 1.44269504f, -t) + x * 1.92596303e-8f;
  const float r = __builtin_amdgcn_exp2f(t);
  return x < -104.f ? 0.f : fmaf(r, lo * 0.693147181f, r);
}

template <int LPR>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// expert of element j of lane `sub` of a row: pieces of V consecutive experts, the lanes' pieces next to each other
template <int LPR, int V>
__device__ __forceinline__ int expert_of(int j, int sub) { return (j / V) * (LPR * V) + sub * V + j % V; }

template <typename T, int LPR, int EPL, int V>
__device__ __forceinline__ void load_row(const BalanceArgs& a, const T* row, int sub, float (&x)[EPL]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < EPL; j += V) {
      const int e = expert_of<LPR, V>(j, sub);
      if (e < a.experts) {                                  // (V divides the experts here)
        const u32x4 w = *reinterpret_cast<const u32x4*>(row + e);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (sizeof(T) == 4) {
            x[j + k] = __uint_as_float(w[k]);
          } else {
            x[j + 2 * k] = __uint_as_float(w[k] << 16);
            x[j + 2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) x[j + k] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = expert_of<LPR, 1>(j, sub);
      x[j] = e < a.experts ? to_f32<T>(row[(long)e * a.se]) : -INFINITY;
    }
  }
}

template <typename T, int LPR, int EPL, int V>
__global__ __launch_bounds__(64 * BL_WAVES) void balance_fwd_kernel(BalanceArgs a) {
  constexpr int RPW = 64 / LPR;                             // rows a wave works on at once
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPR, slot = lane / LPR;
  const int g = blockIdx.y;
  const T* x0 = static_cast<const T*>(a.x) + (long)g * a.sg;
  const uint8_t* mask = a.mask ? a.mask + (long)g * a.mg : nullptr;
  float psum[EPL];
  int cnt[EPL], valid = 0;
#pragma unroll
  for (int j = 0; j < EPL; ++j) { psum[j] = 0.f; cnt[j] = 0; }
  const long step = (long)a.blocks * BL_WAVES * RPW;
  for (long n0 = ((long)blockIdx.x * BL_WAVES + wave) * RPW; n0 < a.rows; n0 += step) {
    const long n = n0 + slot;
    bool on = n < a.rows && (!mask || mask[n * a.mn]);
    float x[EPL];
    if (on) {
      load_row<T, LPR, EPL, V>(a, x0 + n * a.sn, sub, x);
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) top = fmaxf(top, x[j]);
    top = row_max<LPR>(top);
    const float from = top == -INFINITY ? 0.f : top;
    float y[EPL], sum = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) { y[j] = exp_neg(x[j] - from); sum += y[j]; }
    sum = row_sum<LPR>(sum);
    on = on && sum != 0.f;                                  // (all -inf: the row does not count; a NaN does)
    const float inv = on ? 1.f / sum : 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) psum[j] += on ? y[j] * inv : 0.f;
    valid += on && sub == 0;
    // the choice, one expert a round: the largest value that is left, the lowest index where several have it
    for (int k = 0; k < a.top_k; ++k) {
      float best = -INFINITY;
      int at = BL_MAX_E;
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (x[j] > best) { best = x[j]; at = expert_of<LPR, V>(j, sub); }
#pragma unroll
      for (int off = LPR / 2; off > 0; off >>= 1) {
        const float ob = __shfl_xor(best, off, 64);
        const int oa = __shfl_xor(at, off, 64);
        if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (expert_of<LPR, V>(j, sub) == at) { ++cnt[j]; x[j] = -INFINITY; }
    }
  }
  // the wave's rows, then the workgroup's waves
#pragma unroll
  for (int off = 32; off >= LPR; off >>= 1) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      psum[j] += __shfl_xor(psum[j], off, 64);
      cnt[j] += __shfl_xor(cnt[j], off, 64);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) valid += __shfl_xor(valid, off, 64);
  __shared__ float sp[BL_WAVES][LPR * EPL];
  __shared__ int sc[BL_WAVES][LPR * EPL], sv[BL_WAVES];
  if (slot == 0) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      sp[wave][expert_of<LPR, V>(j, sub)] = psum[j];
      sc[wave][expert_of<LPR, V>(j, sub)] = cnt[j];
    }
  }
  if (lane == 0) sv[wave] = valid;
  __syncthreads();
  const long at = (long)g * a.blocks + blockIdx.x;
  for (int e = threadIdx.x; e < a.experts; e += 64 * BL_WAVES) {
    float p = 0.f;
    int c = 0;
#pragma unroll
    for (int w = 0; w < BL_WAVES; ++w) { p += sp[w][e]; c += sc[w][e]; }
    a.psum[at * a.experts + e] = p;
    a.count[at * a.experts + e] = c;
  }
  if (threadIdx.x == 0) {
    int v = 0;
#pragma unroll
    for (int w = 0; w < BL_WAVES; ++w) v += sv[w];
    a.valid[at] = v;
  }
}

struct FinishArgs {
  const float* psum;
  const int* count;
  const int* valid;
  int groups, experts, top_k, blocks;
  double coef;
  double* term;              // [groups][column workgroups]: sum_e f P of the columns
  float* loss;
  long* counts;              // [groups][experts]
  float* prob;               // [groups][experts]
  float* weight;             // [groups][experts] and, last, 1 / G'
};

// a group's 64 columns: counts, mean probabilities, weights (but for 1 / G') and this part of sum_e f_e P_e
__global__ __launch_bounds__(BL_FINISH) void balance_columns_kernel(FinishArgs a) {
  const int g = blockIdx.y, col = threadIdx.x & 63, share = threadIdx.x >> 6, e = blockIdx.x * 64 + col;
  constexpr int SHARES = BL_FINISH / 64;
  __shared__ double sp[SHARES][64];
  __shared__ long sc[SHARES][64], sn[BL_FINISH];
  double p = 0;
  long c = 0, n = 0;
  if (e < a.experts)
    for (int b = share; b < a.blocks; b += SHARES) {
      const long at = ((long)g * a.blocks + b) * a.experts + e;
      p += a.psum[at];
      c += a.count[at];
    }
  for (int b = threadIdx.x; b < a.blocks; b += BL_FINISH) n += a.valid[(long)g * a.blocks + b];
  sp[share][col] = p;
  sc[share][col] = c;
  sn[threadIdx.x] = n;
  __syncthreads();
  if (share != 0) return;
  p = 0; c = 0; n = 0;
  for (int s = 0; s < SHARES; ++s) { p += sp[s][col]; c += sc[s][col]; }
  for (int t = col; t < BL_FINISH; t += 64) n += sn[t];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  double term = 0;
  if (e < a.experts) {
    const double some = n > 0 ? (double)n : 1.0, f = (double)c / (some * a.top_k), mean = p / some;
    term = f * mean;
    a.counts[(long)g * a.experts + e] = c;
    a.prob[(long)g * a.experts + e] = (float)mean;
    a.weight[(long)g * a.experts + e] = (float)(a.coef * a.experts * f / some);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) term += __shfl_xor(term, off, 64);
  if (col == 0) {
    a.term[(long)g * gridDim.x + blockIdx.x] = term;
    if (blockIdx.x == 0) a.term[(long)a.groups * gridDim.x + g] = n > 0 ? 1.0 : 0.0;
  }
}

__global__ __launch_bounds__(BL_FINISH) void balance_loss_kernel(FinishArgs a, int parts) {
  double sum = 0, some = 0;
  for (long i = threadIdx.x; i < (long)a.groups * parts; i += BL_FINISH) sum += a.term[i];
  for (int g = threadIdx.x; g < a.groups; g += BL_FINISH) some += a.term[(long)a.groups * parts + g];
  __shared__ double ss[BL_FINISH / 64], sn[BL_FINISH / 64];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) { sum += __shfl_xor(sum, off, 64); some += __shfl_xor(some, off, 64); }
  if ((threadIdx.x & 63) == 0) { ss[threadIdx.x >> 6] = sum; sn[threadIdx.x >> 6] = some; }
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = some = 0;
  for (int w = 0; w < BL_FINISH / 64; ++w) { sum += ss[w]; some += sn[w]; }
  const double share = some > 0 ? 1.0 / some : 0.0;
  *a.loss = (float)(a.coef * a.experts * sum * share);
  a.weight[(long)a.groups * a.experts] = (float)share;
}

template <typename T, int LPR, int EPL, int V>
__global__ __launch_bounds__(64 * BL_WAVES) void balance_bwd_kernel(BalanceArgs a) {
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPR, slot = lane / LPR;
  const int g = blockIdx.y;
  const T* x0 = static_cast<const T*>(a.x) + (long)g * a.sg;
  T* d0 = static_cast<T*>(a.dx) + (long)g * a.dg;
  const uint8_t* mask = a.mask ? a.mask + (long)g * a.mg : nullptr;
  const float scale = *a.up * a.weight[(long)a.groups * a.experts];
  float w[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = expert_of<LPR, V>(j, sub);
    w[j] = e < a.experts ? scale * a.weight[(long)g * a.experts + e] : 0.f;
  }
  const long step = (long)a.blocks * BL_WAVES * RPW;
  for (long n0 = ((long)blockIdx.x * BL_WAVES + wave) * RPW; n0 < a.rows; n0 += step) {
    const long n = n0 + slot;
    const bool in = n < a.rows, on = in && (!mask || mask[n * a.mn]);
    float x[EPL];
    if (on) {
      load_row<T, LPR, EPL, V>(a, x0 + n * a.sn, sub, x);
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) top = fmaxf(top, x[j]);
    top = row_max<LPR>(top);
    const float from = top == -INFINITY ? 0.f : top;
    float sum = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) { x[j] = exp_neg(x[j] - from); sum += x[j]; }
    sum = row_sum<LPR>(sum);
    const float inv = on && sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) { x[j] *= inv; dot += x[j] * w[j]; }
    dot = row_sum<LPR>(dot);
#pragma unroll
    for (int j = 0; j < EPL; ++j) x[j] = sum != 0.f ? x[j] * (w[j] - dot) : 0.f;      // (a row that does not count: 0 whatever w is)
    if (!in) continue;
    T* row = d0 + n * a.dn;
    if constexpr (V > 1) {
#pragma unroll
      for (int j = 0; j < EPL; j += V) {
        const int e = expert_of<LPR, V>(j, sub);
        if (e < a.experts) {
          u32x4 o;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 4) o[k] = __float_as_uint(x[j + k]);
            else o[k] = pack_bf16x2(x[j + 2 * k], x[j + 2 * k + 1]);
          }
          *reinterpret_cast<u32x4*>(row + e) = o;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = expert_of<LPR, 1>(j, sub);
        if (e < a.experts) {
          if constexpr (sizeof(T) == 4) row[(long)e * a.de] = x[j];
          else row[(long)e * a.de] = f32_to_bf16(x[j]);
        }
      }
    }
  }
}

int lanes_per_row(int experts) {
  int lpr = 1;
  while (lpr < 64 && lpr * 8 < experts) lpr *= 2;
  return lpr;
}

// workgroups per group: enough rows to fill them, and eight to a CU over all groups
int blocks_for(long groups, long rows, int experts) {
  const long per = (long)BL_WAVES * (64 / lanes_per_row(experts));
  const long want = (rows + per - 1) / per, most = groups >= 2048 ? 1 : 2048 / groups;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, bool BWD, int LPR, int EPL, int V>
void launch_one(const BalanceArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.blocks, (unsigned)a.groups), block(64 * BL_WAVES);
  if constexpr (BWD) hipLaunchKernelGGL((balance_bwd_kernel<T, LPR, EPL, V>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((balance_fwd_kernel<T, LPR, EPL, V>), grid, block, 0, s, a);
}

template <typename T, bool BWD, int V>
void launch(const BalanceArgs& a, hipStream_t s) {
  switch (lanes_per_row(a.experts)) {
    case 1: return launch_one<T, BWD, 1, 8, V>(a, s);
    case 2: return launch_one<T, BWD, 2, 8, V>(a, s);
    case 4: return launch_one<T, BWD, 4, 8, V>(a, s);
    case 8: return launch_one<T, BWD, 8, 8, V>(a, s);
    case 16: return launch_one<T, BWD, 16, 8, V>(a, s);
    case 32: return launch_one<T, BWD, 32, 8, V>(a, s);
    default: return a.experts <= 512 ? launch_one<T, BWD, 64, 8, V>(a, s) : launch_one<T, BWD, 64, 16, V>(a, s);
  }
}

template <bool BWD>
void dispatch(const BalanceArgs& a, int dtype, hipStream_t s) {
  // 16-byte pieces where every row has them: consecutive experts, rows that start at 16 bytes and hold whole pieces
  const int per = dtype == REPMODE_F32 ? 4 : 8;
  auto whole = [&](const void* p, long sg, long sn, long se) {
    return ((uintptr_t)p & 15) == 0 && se == 1 && sn % per == 0 && (a.groups == 1 || sg % per == 0);
  };
  const bool vec = a.experts % per == 0 && whole(a.x, a.sg, a.sn, a.se) && (!BWD || whole(a.dx, a.dg, a.dn, a.de));
  if (dtype == REPMODE_F32) vec ? launch<float, BWD, 4>(a, s) : launch<float, BWD, 1>(a, s);
  else vec ? launch<bf16_t, BWD, 8>(a, s) : launch<bf16_t, BWD, 1>(a, s);
}

int check_shape(const char* who, const void* x, int dtype, long groups, long rows, int experts) {
  RM_REQUIRE(dtype == REPMODE_F32 || dtype == REPMODE_BF16, "%s: bad dtype %d", who, dtype);
  RM_REQUIRE(groups > 0 && groups <= 65535 && rows >= 0 && experts > 0 && experts <= BL_MAX_E,
             "%s: 1..65535 groups, 1..%d experts; got %ld groups of %ld rows over %d experts", who, BL_MAX_E, groups, rows, experts);
  RM_REQUIRE(x || rows == 0, "%s: null pointer", who);
  return REPMODE_OK;
}

}  // namespace

extern "C" int repmode_balance_plan(long groups, long rows, int experts, long* ws_bytes) {
  RM_REQUIRE(ws_bytes, "balance_plan: null pointer");
  if (int rc = check_shape("balance_plan", ws_bytes, REPMODE_F32, groups, rows, experts)) return rc;
  const long blocks = blocks_for(groups, rows, experts);
  *ws_bytes = groups * ((experts + 63) / 64 + 1) * 8 + groups * blocks * experts * 8 + groups * blocks * 4;
  return REPMODE_OK;
}

extern "C" int repmode_balance_fwd(const void* x, int dtype, long groups, long rows, int experts, long sg, long sn, long se,
                                   const unsigned char* mask, long mg, long mn, int top_k, double coef, void* ws, long ws_bytes,
                                   float* loss, long* counts, float* prob, float* weight, void* stream) {
  if (int rc = check_shape("balance_fwd", x, dtype, groups, rows, experts)) return rc;
  RM_REQUIRE(ws && loss && counts && prob && weight, "balance_fwd: null pointer");
  RM_REQUIRE(top_k >= 1 && top_k <= experts, "balance_fwd: top_k must be 1..%d, got %d", experts, top_k);
  RM_REQUIRE(rows * (long)top_k < (1L << 31), "balance_fwd: too many rows in a group");
  long need = 0;
  if (int rc = repmode_balance_plan(groups, rows, experts, &need)) return rc;
  RM_REQUIRE(ws_bytes >= need && ((uintptr_t)ws & 7) == 0, "balance_fwd: workspace of %ld bytes (8-byte aligned) needed, got %ld", need, ws_bytes);
  const int parts = (experts + 63) / 64;
  BalanceArgs a{};
  a.x = x; a.mask = mask;
  a.sg = sg; a.sn = sn; a.se = se; a.mg = mg; a.mn = mn;
  a.rows = rows; a.groups = (int)groups; a.experts = experts; a.top_k = top_k;
  a.blocks = blocks_for(groups, rows, experts);
  double* term = static_cast<double*>(ws);
  a.psum = reinterpret_cast<float*>(term + groups * (parts + 1));
  a.count = reinterpret_cast<int*>(a.psum + groups * a.blocks * experts);
  a.valid = a.count + groups * a.blocks * experts;
  hipStream_t s = static_cast<hipStream_t>(stream);
  dispatch<false>(a, dtype, s);
  RM_LAUNCH_CHECK("balance_fwd");
  FinishArgs f{a.psum, a.count, a.valid, a.groups, experts, top_k, a.blocks, coef, term, loss, counts, prob, weight};
  hipLaunchKernelGGL(balance_columns_kernel, dim3(parts, (unsigned)groups), dim3(BL_FINISH), 0, s, f);
  RM_LAUNCH_CHECK("balance_columns");
  hipLaunchKernelGGL(balance_loss_kernel, dim3(1), dim3(BL_FINISH), 0, s, f, parts);
  RM_LAUNCH_CHECK("balance_loss");
  return REPMODE_OK;
}

extern "C" int repmode_balance_bwd(const void* x, int dtype, long groups, long rows, int experts, long sg, long sn, long se,
                                   const unsigned char* mask, long mg, long mn, const float* weight, const float* up, void* dx, long dg,
                                   long dn, long de, void* stream) {
  if (int rc = check_shape("balance_bwd", x, dtype, groups, rows, experts)) return rc;
  if (rows == 0) return REPMODE_OK;
  RM_REQUIRE(weight && up && dx, "balance_bwd: null pointer");
  BalanceArgs a{};
  a.x = x; a.mask = mask; a.dx = dx; a.weight = weight; a.up = up;
  a.sg = sg; a.sn = sn; a.se = se; a.mg = mg; a.mn = mn; a.dg = dg; a.dn = dn; a.de = de;
  a.rows = rows; a.groups = (int)groups; a.experts = experts;
  a.blocks = blocks_for(groups, rows, experts);
  dispatch<true>(a, dtype, static_cast<hipStream_t>(stream));
  RM_LAUNCH_CHECK("balance_bwd");
  return REPMODE_OK;
}
