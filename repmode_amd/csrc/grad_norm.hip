// grad_norm.hip -- the 2-norm of many tensors together and the factor that clips it, without a host synchronisation:
//     norm = sqrt(sum_i sum_e x_ie^2)          clip = min(1, max_norm / (norm + 1e-6)), NaN where a value is not finite
//
// Products and sums are float64: the square of a float32 (or bfloat16) value is exact there and cannot overflow or vanish, so
// gradients of 1e-30 and of 1e30 count for what they are; the float64 units keep up with HBM (one conversion and one fused
// multiply-add an element).  The sum's order is fixed -- a workgroup per GN_CHUNK bytes of a tensor, one partial each, the
// partials added by one workgroup in a fixed order -- so a run repeats itself bit by bit.
// What bounds it: HBM, one read of the tensors, past the caches: 64 / 256 M float32 values 47 / 165 us (5.7 / 6.5 TB/s), through them 91 /
// 246 us -- and an update that reads the gradients next gains less by finding a part of them there than the norm loses (norm and
// update of 128 M float32 values 716 and 739 us).
#include "common.h"

#include <cmath>

namespace {

constexpr int GN_MAX = REPMODE_GRAD_NORM_MAX;
constexpr int GN_CHUNK = REPMODE_GRAD_NORM_CHUNK;         // bytes of a tensor per workgroup
constexpr int GN_THREADS = 256;

struct NormArgs {
  const void* x[GN_MAX];
  long numel[GN_MAX];
  int first[GN_MAX + 1];         // first workgroup of tensor i
  int nt;
};
static_assert(sizeof(NormArgs) + 16 <= 4096, "launch arguments");

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off, 64);
  return v;
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {          // in thread 0
  __shared__ double part[THREADS / 64];
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < THREADS / 64; ++w) v += part[w];
  return v;
}

template <typename T>
__global__ __launch_bounds__(GN_THREADS) void grad_norm_kernel(NormArgs a, double* __restrict__ partial) {
  constexpr int VEC = 16 / sizeof(T), ITEMS = GN_CHUNK / 16 / GN_THREADS;
  int i = 0;
  for (int hi = a.nt; hi - i > 1;) {                           // the tensor of this workgroup: first[i] <= blockIdx.x < first[i + 1]
    const int mid = (i + hi) >> 1;
    if ((int)blockIdx.x >= a.first[mid]) i = mid;
    else hi = mid;
  }
  const long base = (long)((int)blockIdx.x - a.first[i]) * (GN_CHUNK / sizeof(T)), n = a.numel[i];
  const T* __restrict__ x = static_cast<const T*>(a.x[i]);
  double sum = 0;
  auto add = [&](float f) { sum = fma((double)f, (double)f, sum); };
  const long end = base + (long)(GN_CHUNK / sizeof(T)) < n ? base + (long)(GN_CHUNK / sizeof(T)) : n;
  long rest = base;                                             // what is left to take one by one
  if (((uintptr_t)x & 15) == 0) {
    const int pieces = (int)(end - base) / VEC;                 // of 16 bytes; all loads are under way before the first is used
    const u32x4* q = reinterpret_cast<const u32x4*>(x + base) + threadIdx.x;
    u32x4 w[ITEMS];
    if (pieces == ITEMS * GN_THREADS) {
#pragma unroll
      for (int u = 0; u < ITEMS; ++u) w[u] = __builtin_nontemporal_load(q + u * GN_THREADS);
    } else {
#pragma unroll
      for (int u = 0; u < ITEMS; ++u) w[u] = u * GN_THREADS + (int)threadIdx.x < pieces ? q[u * GN_THREADS] : u32x4{0, 0, 0, 0};
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < ITEMS; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (VEC == 4) {
          add(__uint_as_float(w[u][k]));
        } else {
          add(__uint_as_float(w[u][k] << 16));
          add(__uint_as_float(w[u][k] & 0xffff0000u));
        }
      }
    rest += (long)pieces * VEC;
  }
  constexpr int AHEAD = 8;
  for (long o = rest + threadIdx.x; o < end; o += AHEAD * GN_THREADS) {         // (every load is made, behind the last value that again)
    T v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) v[u] = x[o + u * GN_THREADS < end ? o + u * GN_THREADS : end - 1];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (o + u * GN_THREADS < end) add(to_f32<T>(v[u]));
  }
  sum = block_sum<GN_THREADS>(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

constexpr int GF_THREADS = 1024;
__global__ __launch_bounds__(GF_THREADS) void grad_norm_finish_kernel(const double* __restrict__ partial, long n, double max_norm,
                                                                    float* __restrict__ norm, float* __restrict__ clip) {
  constexpr int AHEAD = 8;                                      // loads under way
  double sum = 0;
  long i = threadIdx.x;
  for (; i + (AHEAD - 1) * GF_THREADS < n; i += AHEAD * GF_THREADS) {
    double v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) v[u] = partial[i + u * GF_THREADS];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) sum += v[u];
  }
  for (; i < n; i += GF_THREADS) sum += partial[i];
  sum = block_sum<GF_THREADS>(sum);
  if (threadIdx.x == 0) {
    const double r = sqrt(sum);
    *norm = (float)r;
    const double c = max_norm / (r + 1e-6);
    *clip = !(sum < INFINITY) ? __uint_as_float(0x7fc00000u) : c < 1.0 ? (float)c : 1.f;
  }
}

}  // namespace

extern "C" int repmode_grad_norm_partial(int ntensors, int dtype, const void* const* x, const long* numel, double* partial, long capacity,
                                         long* used, void* stream) {
  RM_REQUIRE(x && numel && partial && used, "grad_norm: null pointer");
  RM_REQUIRE(ntensors > 0 && ntensors <= GN_MAX, "grad_norm: 1..%d tensors per call, got %d", GN_MAX, ntensors);
  RM_REQUIRE(dtype == REPMODE_F32 || dtype == REPMODE_BF16, "grad_norm: bad dtype %d", dtype);
  const long per = GN_CHUNK / (dtype == REPMODE_F32 ? 4 : 2);
  NormArgs a{};
  a.nt = ntensors;
  long total = 0;
  for (int i = 0; i < ntensors; ++i) {
    RM_REQUIRE(x[i] && numel[i] > 0, "grad_norm: bad tensor %d", i);
    RM_REQUIRE(((uintptr_t)x[i] & (dtype == REPMODE_F32 ? 3 : 1)) == 0, "grad_norm: tensor %d is not aligned to its elements", i);
    a.x[i] = x[i]; a.numel[i] = numel[i];
    a.first[i] = (int)total;
    total += (numel[i] + per - 1) / per;
    RM_REQUIRE(total < (1L << 31), "grad_norm: grid too large");
  }
  RM_REQUIRE(total <= capacity, "grad_norm: %ld partial sums needed, room for %ld", total, capacity);
  a.first[ntensors] = (int)total;
  if (dtype == REPMODE_F32) hipLaunchKernelGGL(grad_norm_kernel<float>, dim3((unsigned)total), dim3(GN_THREADS), 0, static_cast<hipStream_t>(stream), a, partial);
  else hipLaunchKernelGGL(grad_norm_kernel<bf16_t>, dim3((unsigned)total), dim3(GN_THREADS), 0, static_cast<hipStream_t>(stream), a, partial);
  RM_LAUNCH_CHECK("grad_norm");
  *used = total;
  return REPMODE_OK;
}

extern "C" int repmode_grad_norm_finish(const double* partial, long n, double max_norm, float* norm, float* clip, void* stream) {
  RM_REQUIRE(norm && clip && n >= 0 && (partial || n == 0), "grad_norm_finish: null pointer");
  RM_REQUIRE(max_norm >= 0, "grad_norm_finish: max_norm must not be negative or NaN");
  hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(GF_THREADS), 0, static_cast<hipStream_t>(stream), partial, n, max_norm, norm, clip);
  RM_LAUNCH_CHECK("grad_norm_finish");
  return REPMODE_OK;
}
