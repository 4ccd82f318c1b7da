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
// the lane's share of the column sums (probabilities in float32, counts as integers) need no memory.
//   The choice needs no order, only the k-th largest value: each lane sorts its values once (a network of 2- and 3-sorters), then top_k rounds take the
// row's largest head and move the list of the lane that holds it up by one; what is at least the last round's value is chosen.
// The first round's value is the softmax's maximum.  All of it on integers that are ordered as the values are; bfloat16
// values carry their index in the lower half, so no two are equal; float32 rows where more than top_k values
// reach the last one (equal values) are chosen again one by one, value and index.
//   A workgroup walks many rows and writes one partial per expert; one launch adds the partials of a group's columns in a fixed
// order in float64, one more makes the loss of them; where one workgroup has seen all rows it does both itself.  No float atomics: a
// run repeats itself bit by bit.  The backward pass reads the logits again and needs nothing of a row but its logits.
// What bounds it: the backward pass HBM (one read, one write: 262144 x 256 float32 logits 82 us, 6.5 TB/s), the forward pass the
// instructions of exponential and choice (the same logits 69 us for the top 8 and 5 for the columns, where a read takes 40; the top 1
// some 20 us less).
#include "common.h"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace {

constexpr int BL_WAVES = 8;
constexpr int BL_MAX_E = REPMODE_BALANCE_MAX_EXPERTS;
constexpr int BL_TILE_BYTES = 72 << 10;  // of a tile: two workgroups share a CU's LDS
constexpr int BL_JOIN = BL_WAVES * (sizeof(float) + sizeof(int));      // bytes a column of a row takes where a workgroup's waves are joined
constexpr int BL_FINISH = 256;           // threads of the finish
constexpr int BL_COLUMNS = 4;            // columns of a workgroup of it; the other threads share the partials
constexpr int BL_BLOCKS = 512;           // workgroups of a pass: two to a CU, which registers leave room for
constexpr long BL_ROWS = 1024;           // rows that a lane adds in float32, at most about (equal ones are off by half as many roundings); in
                                         // many long groups, where 512 workgroups would leave more to each, there are more workgroups

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
  int tile_rows, pitch;      // tiled: rows of a tile, floats from one of them to the next in LDS
  float* psum;               // forward: [groups][blocks][experts]
  int* count;                //          the same shape
  int* valid;                //          [groups][blocks]
};

// ---- over the LPR neighbouring lanes of a row, the result in each of them.  Up to 16 lanes by DPP (inside a row of 16: quads, then
// mirrors, which do because the quads' lanes agree by then), rows and halves by swaps.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true); }
template <int LPR, typename T, typename Op>
__device__ __forceinline__ T over_row(T v, Op op) {
  auto with = [&](uint32_t o) { v = op(v, __builtin_bit_cast(T, o)); };
  auto bits = [&]() { return __builtin_bit_cast(uint32_t, v); };
  if constexpr (LPR >= 2) with(dpp<0xB1>(bits()));          // quad_perm 1 0 3 2
  if constexpr (LPR >= 4) with(dpp<0x4E>(bits()));          // quad_perm 2 3 0 1
  if constexpr (LPR >= 8) with(dpp<0x141>(bits()));         // row_half_mirror
  if constexpr (LPR >= 16) with(dpp<0x140>(bits()));        // row_mirror
  if constexpr (LPR >= 32) {
    const auto w = __builtin_amdgcn_permlane16_swap(bits(), bits(), false, false);
    v = op(__builtin_bit_cast(T, (uint32_t)w[0]), __builtin_bit_cast(T, (uint32_t)w[1]));
  }
  if constexpr (LPR >= 64) {
    const auto w = __builtin_amdgcn_permlane32_swap(bits(), bits(), false, false);
    v = op(__builtin_bit_cast(T, (uint32_t)w[0]), __builtin_bit_cast(T, (uint32_t)w[1]));
  }
  return v;
}
template <int LPR>
__device__ __forceinline__ int row_max(int v) { return over_row<LPR>(v, [](int a, int b) { return a > b ? a : b; }); }
template <int LPR, typename T>
__device__ __forceinline__ T row_sum(T v) { return over_row<LPR>(v, [](T a, T b) { return a + b; }); }

// Integers in the order of the floats: a negative float's is its magnitude's, negated, so -0 and 0 have one key.  What lies below
// not_lowest is -inf (or a NaN with its sign bit); a NaN without it lies above all.  The same step leads back.
__device__ __forceinline__ int turn(int u) { return u < 0 ? (int)0x80000000 - u : u; }
// (a bfloat16 value's key leaves the lower half to the index)
template <typename T>
constexpr int not_lowest = sizeof(T) == 2 ? (int)0x80810000 : (int)0x80800001;
// the softmax's shift of a row whose largest key this is
template <typename T>
__device__ __forceinline__ float top_of(int key) {
  if (key < not_lowest<T>) return 0.f;                       // (nothing but -inf)
  return __int_as_float(turn(sizeof(T) == 2 ? key & (int)0xffff0000 : key));
}

// y_j = e^(x_j - top) of a row (y may be x), and its sum.  As 2^(x_j L - top L), L = log2(e), in one fused step: the rounding of
// top L is the whole row's and goes out with the sum, so a probability is off by |x_j - top| 2^-24 like that of a rounded
// difference.  From 2^20 on, where that rounding would grow to 2^-4 and more (at last to a sum of 0 or infinity), the difference is
// taken first.
template <int LPR, int EPL>
__device__ __forceinline__ float row_exp(float top, const float (&x)[EPL], float (&y)[EPL]) {
  constexpr float L = 1.44269504f;
  const float shift = top * L;
  const bool far = fabsf(top) >= 0x1p20f;
  if (__any(far)) {                                           // (row by row: what a row gives does not go by the rows beside it)
#pragma unroll
    for (int j = 0; j < EPL; ++j) y[j] = __builtin_amdgcn_exp2f(far ? (x[j] - top) * L : fmaf(x[j], L, -shift));
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) y[j] = __builtin_amdgcn_exp2f(fmaf(x[j], L, -shift));
  }
  float sum = y[0];
#pragma unroll
  for (int j = 1; j < EPL; ++j) sum += y[j];
  return row_sum<LPR>(sum);
}

__device__ __forceinline__ void sort2(int& a, int& b) {
  const int x = a, y = b;
  a = max(x, y);
  b = min(x, y);
}
// One instruction for each of the three.  (Spelled with minima and maxima the median would share their first steps with the others, and
// none of the three be one instruction.  No lane shift reads its result: the rounds below shift what a selection or a maximum made.)
__device__ __forceinline__ void sort3(int& a, int& b, int& c) {
  const int x = a, y = b, z = c;
  a = max(max(x, y), z);
  asm("v_med3_i32 %0, %1, %2, %3" : "=v"(b) : "v"(x), "v"(y), "v"(z));
  c = min(min(x, y), z);
}
// Eight values, descending: as the columns (0 1 2) (3 4 5) (6 7) of a square whose columns and then rows are sorted (which keeps the
// columns so).  0 is the largest then.  Of its diagonal 2 4 6, sorted, two at least lie below both of 1 and 3 (4, and one's neighbour), so
// only the largest may lie above the smaller of those; 5 and 7 likewise.  27 instructions, where pairs alone take 38.
__device__ __forceinline__ void sort8(int* s) {
  sort3(s[0], s[1], s[2]);
  sort3(s[3], s[4], s[5]);
  sort2(s[6], s[7]);
  sort3(s[0], s[3], s[6]);
  sort3(s[1], s[4], s[7]);
  sort2(s[2], s[5]);
  sort3(s[2], s[4], s[6]);
  sort2(s[1], s[3]);
  sort2(s[5], s[7]);
  sort2(s[3], s[2]);
  sort2(s[6], s[5]);
  const int third = s[3], fourth = s[2], fifth = s[4], sixth = s[6], seventh = s[5];
  s[2] = third; s[3] = fourth; s[4] = fifth; s[5] = sixth; s[6] = seventh;
}
// descending: eights, then Batcher's odd-even merges
template <int N>
__device__ __forceinline__ void sort_descending(int (&s)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 8) sort8(s + j);
#pragma unroll
  for (int p = 8; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if ((i + j) / (2 * p) == (i + j + k) / (2 * p) && i + j + k < N) sort2(s[i + j], s[i + j + k]);
}

// the lane whose head is t moves its list up by one, as far as N values of it are looked at afterwards
template <int N, int EPL>
__device__ __forceinline__ void pop(int (&s)[EPL], int t) {
  const bool mine = s[0] == t;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int here = s[j], next = j + 1 < EPL ? s[j + 1] : (int)0x80000000;
    s[j] = mine ? +next : +here;
  }
}
// rounds K + 1 .. top_k of at most EPL: after the K-th, EPL - K values of a list can still count
template <int LPR, int K, int EPL>
__device__ __forceinline__ int rounds_from(int (&s)[EPL], int t, int top_k) {
  if constexpr (K < EPL) {
    if (K < top_k) {
      pop<EPL - K>(s, t);
      return rounds_from<LPR, K + 1>(s, row_max<LPR>(s[0]), top_k);
    }
  }
  return t;
}

// the k-th largest of a row (equal heads of several lanes count once); s: the lane's keys, sorted; top: the row's largest
template <int LPR, int EPL>
__device__ __forceinline__ int row_kth(int (&s)[EPL], int top, int top_k) {
  int t = top;
  if constexpr (LPR == 1) {
#pragma unroll
    for (int j = 1; j < EPL; ++j) t = j < top_k ? +s[j] : t;
  } else if (__builtin_expect(top_k <= EPL, 1)) {
    t = rounds_from<LPR, 1>(s, t, top_k);
  } else {
    for (int k = 1; k < top_k; ++k) {
      pop<EPL>(s, t);
      t = row_max<LPR>(s[0]);
    }
  }
  return t;
}

// expert of element j of lane `sub` of a row: pieces of V consecutive experts, the lanes' pieces next to each other
template <int LPR, int V>
__device__ __forceinline__ int expert_of(int j, int sub) { return (j / V) * (LPR * V) + sub * V + j % V; }

// A lane's values of a row as they are in memory.  Every load is made, in a straight line -- past the row's last value that again -- since
// behind loads that may or may not have been made there is one wait for all that are under way, and behind each of them one where
// its value is converted.
template <typename T, int EPL, int V>
struct RawRow {
  std::conditional_t<V == 1, T, u32x4> w[EPL / V];
};
template <typename T, int LPR, int EPL, int V>
__device__ __forceinline__ void fetch_row(const BalanceArgs& a, const T* row, int sub, RawRow<T, EPL, V>& r) {
#pragma unroll
  for (int q = 0; q < EPL / V; ++q) {
    const int e = min(expert_of<LPR, V>(q * V, sub), a.experts - V);          // (V divides the experts)
    if constexpr (V == 1) r.w[q] = row[(long)e * a.se];
    else r.w[q] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + e));
  }
}
// as floats; -inf where there is none, and everywhere in a row that does not count
template <typename T, int LPR, int EPL, int V>
__device__ __forceinline__ void row_values(const BalanceArgs& a, const RawRow<T, EPL, V>& r, bool on, int sub, float (&x)[EPL]) {
#pragma unroll
  for (int q = 0; q < EPL / V; ++q) {
    if constexpr (V == 1) {
      x[q] = to_f32<T>(r.w[q]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          x[q * V + k] = __uint_as_float(r.w[q][k]);
        } else {
          x[q * V + 2 * k] = __uint_as_float(r.w[q][k] << 16);
          x[q * V + 2 * k + 1] = __uint_as_float(r.w[q][k] & 0xffff0000u);
        }
      }
    }
  }
  if (a.experts == LPR * EPL && __all(on)) return;
#pragma unroll
  for (int j = 0; j < EPL; ++j) x[j] = on && expert_of<LPR, V>(j, sub) < a.experts ? x[j] : -INFINITY;
}

// Logits whose rows, not experts, are neighbours in memory: a tile of rows is read along them into LDS, [row][expert] with an odd
// pitch, and the rows taken from there.  (Read directly a wave would use 4 RPW bytes of each cache line it asks for.)
template <typename T>
__device__ __forceinline__ void load_tile(const BalanceArgs& a, const T* x0, const uint8_t* mask, long n0, float* tile) {
  constexpr int AHEAD = 8;
  const int r = threadIdx.x % a.tile_rows, e0 = threadIdx.x / a.tile_rows, step = 64 * BL_WAVES / a.tile_rows;
  const long n = min(n0 + r, a.rows - 1);
  const bool on = n == n0 + r && (!mask || mask[n * a.mn]);
  const T* x = x0 + n * a.sn;
  int e = e0;
  for (; e - e0 + AHEAD * step <= a.experts; e += AHEAD * step) {
    const T* from = x + (long)e * a.se;
    T v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) v[u] = from[(long)(u * step) * a.se];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) tile[r * a.pitch + e + u * step] = on ? to_f32<T>(v[u]) : -INFINITY;
  }
  if (e - e0 < a.experts) {
    T v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) v[u] = x[(long)min(e + u * step, a.experts - 1) * a.se];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (e + u * step < a.experts) tile[r * a.pitch + e + u * step] = on ? to_f32<T>(v[u]) : -INFINITY;
  }
}
template <int LPR, int EPL>
__device__ __forceinline__ void row_of_tile(const BalanceArgs& a, const float* tile, int r, int sub, float (&x)[EPL]) {
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = expert_of<LPR, 1>(j, sub);
    x[j] = e < a.experts ? tile[r * a.pitch + e] : -INFINITY;
  }
}

// cnt += the lane's chosen values of a row: those of at least the k-th largest key t
template <typename T, int LPR, int EPL, int V>
__device__ __forceinline__ void choose(const int (&key)[EPL], int t, int sub, int top_k, int (&cnt)[EPL]) {
  const int from = max(t, not_lowest<T>);
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) cnt[j] += key[j] >= from;
  } else {
    // A row with top_k values or more has at least top_k of t or more, and equal ones only if it has more.  Over the wave's rows by
    // ballots; where a row has fewer, row by row.
    bool in[EPL];
    int n = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      in[j] = key[j] >= from;
      n += __popcll(__ballot(in[j]));
    }
    bool equal = n != 64 / LPR * top_k || __any(t < not_lowest<T>);
    if (equal) {
      int own = 0;
#pragma unroll
      for (int j = 0; j < EPL; ++j) own += in[j];
      equal = __any(row_sum<LPR>(own) > top_k);
    }
    if (equal) {                                              // one by one, the largest that is left, the lowest index first
      int s[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) s[j] = key[j];
      for (int k = 0; k < top_k; ++k) {
        int best = s[0];
#pragma unroll
        for (int j = 1; j < EPL; ++j) best = max(best, s[j]);
        best = row_max<LPR>(best);
        int at = -BL_MAX_E;
#pragma unroll
        for (int j = EPL - 1; j >= 0; --j)
          if (s[j] == best && best >= not_lowest<T>) at = -expert_of<LPR, V>(j, sub);
        at = -row_max<LPR>(at);
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (expert_of<LPR, V>(j, sub) == at) { ++cnt[j]; s[j] = (int)0x80000000; }
      }
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) cnt[j] += in[j];
    }
  }
}

struct FinishArgs {
  const float* psum;
  const int* count;
  const int* valid;
  int groups, experts, top_k, blocks;
  double coef;
  double* term;              // [groups][column workgroups]: sum_e f P of the columns; behind them, [groups]: 1 where the group has rows
  float* loss;
  long* counts;              // [groups][experts]
  float* prob;               // [groups][experts]
  float* weight;             // [groups][experts] but for 1 / G', and, last, 1 / G'
};

// an expert's outputs, n: the group's rows; returns f P
__device__ __forceinline__ double finish_expert(const FinishArgs& a, int g, int e, double p, long c, long n) {
  const double some = n > 0 ? (double)n : 1.0, f = (double)c / (some * a.top_k), mean = p / some;
  a.counts[(long)g * a.experts + e] = c;
  a.prob[(long)g * a.experts + e] = (float)mean;
  a.weight[(long)g * a.experts + e] = (float)(a.coef * a.experts * f / some);
  return f * mean;
}
__device__ __forceinline__ void finish_loss(const FinishArgs& a, double sum, double some) {
  const double share = some > 0 ? 1.0 / some : 0.0;
  *a.loss = (float)(a.coef * a.experts * sum * share);
  a.weight[(long)a.groups * a.experts] = (float)share;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

template <typename T, int LPR, int EPL, int V, bool TILED>
__global__ __launch_bounds__(64 * BL_WAVES) void balance_fwd_kernel(BalanceArgs a, FinishArgs f) {
  constexpr int RPW = 64 / LPR;                             // rows a wave works on at once
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane % LPR, slot = lane / LPR;
  const int g = blockIdx.y;
  const T* x0 = static_cast<const T*>(a.x) + (long)g * a.sg;
  const uint8_t* mask = a.mask ? a.mask + (long)g * a.mg : nullptr;
  float psum[EPL];
  int cnt[EPL], valid = 0;
#pragma unroll
  for (int j = 0; j < EPL; ++j) { psum[j] = 0.f; cnt[j] = 0; }
  auto work = [&](float (&x)[EPL]) {
    int key[EPL], s[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      key[j] = turn(__float_as_int(x[j]));
      if constexpr (sizeof(T) == 2) key[j] |= 0xffff - expert_of<LPR, V>(j, sub);
      s[j] = key[j];
    }
    sort_descending(s);
    const int top = row_max<LPR>(s[0]);
    const float sum = row_exp<LPR>(top_of<T>(top), x, x);
    const bool counts = sum != 0.f;                         // (all -inf: the row does not count; a NaN does)
    const float inv = counts ? __builtin_amdgcn_rcpf(sum) : 0.f;         // (1 ulp; 1 <= sum <= experts)
#pragma unroll
    for (int j = 0; j < EPL; ++j) psum[j] = fmaf(x[j], inv, psum[j]);
    valid += __popcll(__ballot(counts));                    // (the wave's, LPR for each row)
    choose<T, LPR, EPL, V>(key, row_kth<LPR>(s, top, a.top_k), sub, a.top_k, cnt);
  };
  if constexpr (TILED) {
    extern __shared__ float tile[];
    for (long n0 = (long)blockIdx.x * a.tile_rows; n0 < a.rows; n0 += (long)a.blocks * a.tile_rows) {
      load_tile(a, x0, mask, n0, tile);
      __syncthreads();
      for (int r = wave * RPW; r < a.tile_rows; r += BL_WAVES * RPW) {
        float x[EPL];
        row_of_tile<LPR>(a, tile, r + slot, sub, x);
        work(x);
      }
      __syncthreads();
    }
  } else {
    // Rows are fetched while those before them are worked on, into two sets of registers that take turns; behind the last rows the last
    // again.
    const unsigned step = a.blocks * BL_WAVES * RPW, end = (unsigned)a.rows;          // (rows < 2^31, step <= 2^18)
    unsigned n0 = (blockIdx.x * BL_WAVES + wave) * RPW;
    const long slot_at = slot * a.sn;
    const T* rows = x0 + (long)n0 * a.sn;
    auto walk = [&](auto has_mask) {
      constexpr bool MASKED = decltype(has_mask)::value;
      struct Rows {
        RawRow<T, EPL, V> row;
        uint8_t on;
      };
      auto fetch = [&](Rows& to, unsigned n, const T* from) {
        long at = slot_at;
        unsigned in = slot;
        if (n + RPW > end) {
          in = min(in, end - 1 - n);
          at = in * a.sn;
        }
        fetch_row<T, LPR, EPL, V>(a, from + at, sub, to.row);
        if constexpr (MASKED) to.on = mask[(long)(n + in) * a.mn];
      };
      auto turn_of = [&](Rows& now, Rows& then) {             // whether there are more
        const bool more = n0 + step < end;
        const unsigned n = n0;
        n0 += more ? step : 0;
        rows += more ? step * a.sn : 0;
        fetch(then, n0, rows);
        float x[EPL];
        bool on = n + slot < end;
        if constexpr (MASKED) on = on && now.on;
        row_values<T, LPR, EPL, V>(a, now.row, on, sub, x);
        work(x);
        return more;
      };
      Rows even, odd;
      fetch(even, n0, rows);
      while (turn_of(even, odd) && turn_of(odd, even)) {}
    };
    if (n0 < end) {
      if (mask) walk(std::true_type{});
      else walk(std::false_type{});
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
  __shared__ int sv[BL_WAVES];
  __shared__ double st[BL_WAVES];
  __shared__ __align__(16) char own[TILED ? 1 : BL_JOIN * LPR * EPL];
  extern __shared__ float tile[];                           // (of a tiled pass, whose rows are done with)
  float(*sp)[LPR * EPL] = reinterpret_cast<float(*)[LPR * EPL]>(TILED ? reinterpret_cast<char*>(tile) : own);
  int(*sc)[LPR * EPL] = reinterpret_cast<int(*)[LPR * EPL]>(sp + BL_WAVES);
  if (slot == 0) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      sp[wave][expert_of<LPR, V>(j, sub)] = psum[j];
      sc[wave][expert_of<LPR, V>(j, sub)] = cnt[j];
    }
  }
  if (lane == 0) sv[wave] = valid / LPR;
  __syncthreads();
  int rows = 0;
#pragma unroll
  for (int w = 0; w < BL_WAVES; ++w) rows += sv[w];
  const bool alone = gridDim.x == 1 && gridDim.y == 1;      // this workgroup has seen all rows: it finishes
  const long at = (long)g * a.blocks + blockIdx.x;
  double term = 0;
  for (int e = threadIdx.x; e < a.experts; e += 64 * BL_WAVES) {
    double p = 0;
    int c = 0;
#pragma unroll
    for (int w = 0; w < BL_WAVES; ++w) { p += sp[w][e]; c += sc[w][e]; }
    if (alone) {
      term += finish_expert(f, 0, e, p, c, rows);
    } else {
      a.psum[at * a.experts + e] = (float)p;
      a.count[at * a.experts + e] = c;
    }
  }
  if (!alone) {
    if (threadIdx.x == 0) a.valid[at] = rows;
    return;
  }
  term = wave_sum(term);
  if (lane == 0) st[wave] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    term = 0;
    for (int w = 0; w < BL_WAVES; ++w) term += st[w];
    finish_loss(f, term, rows > 0 ? 1.0 : 0.0);
  }
}

// BL_COLUMNS columns of a group: counts, mean probabilities, weights (but for 1 / G') and this part of sum_e f_e P_e
__global__ __launch_bounds__(BL_FINISH) void balance_columns_kernel(FinishArgs a) {
  constexpr int SHARES = BL_FINISH / BL_COLUMNS, AHEAD = 8;
  static_assert(64 % BL_COLUMNS == 0, "a wave holds whole shares");
  const int g = blockIdx.y, col = threadIdx.x % BL_COLUMNS, share = threadIdx.x / BL_COLUMNS, e = blockIdx.x * BL_COLUMNS + col;
  __shared__ double sp[BL_FINISH / 64][BL_COLUMNS];
  __shared__ long sc[BL_FINISH / 64][BL_COLUMNS], sn[BL_FINISH / 64];
  double p = 0;
  long c = 0, n = 0;
  const long at = (long)g * a.blocks * a.experts + min(e, a.experts - 1);
  for (int b0 = 0; b0 < a.blocks; b0 += AHEAD * SHARES) {      // (every load is made: behind the last partial the last again)
    float v[AHEAD];
    int w[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const long b = at + (long)min(b0 + u * SHARES + share, a.blocks - 1) * a.experts;
      v[u] = a.psum[b];
      w[u] = a.count[b];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const bool in = b0 + u * SHARES + share < a.blocks;
      p += in ? v[u] : 0.f;
      c += in ? w[u] : 0;
    }
  }
  for (int b = threadIdx.x; b < a.blocks; b += BL_FINISH) n += a.valid[(long)g * a.blocks + b];
#pragma unroll
  for (int off = 32; off >= BL_COLUMNS; off >>= 1) {          // the wave's shares of a column
    p += __shfl_xor(p, off, 64);
    c += __shfl_xor(c, off, 64);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  if ((threadIdx.x & 63) < BL_COLUMNS) {
    sp[threadIdx.x >> 6][col] = p;
    sc[threadIdx.x >> 6][col] = c;
  }
  if ((threadIdx.x & 63) == 0) sn[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  p = 0; c = 0; n = 0;
#pragma unroll
  for (int w = 0; w < BL_FINISH / 64; ++w) { p += sp[w][col]; c += sc[w][col]; n += sn[w]; }
  const double term = wave_sum(share == 0 && e < a.experts ? finish_expert(a, g, e, p, c, n) : 0.0);
  if (threadIdx.x == 0) {
    a.term[(long)g * gridDim.x + blockIdx.x] = term;
    if (blockIdx.x == 0) a.term[(long)a.groups * gridDim.x + g] = n > 0 ? 1.0 : 0.0;
  }
}

__global__ __launch_bounds__(BL_FINISH) void balance_loss_kernel(FinishArgs a, int parts) {
  double sum = 0, some = 0;
  for (long i = threadIdx.x; i < (long)a.groups * parts; i += BL_FINISH) sum += a.term[i];
  for (int g = threadIdx.x; g < a.groups; g += BL_FINISH) some += a.term[(long)a.groups * parts + g];
  __shared__ double ss[BL_FINISH / 64], sn[BL_FINISH / 64];
  sum = wave_sum(sum);
  some = wave_sum(some);
  if ((threadIdx.x & 63) == 0) { ss[threadIdx.x >> 6] = sum; sn[threadIdx.x >> 6] = some; }
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = some = 0;
  for (int w = 0; w < BL_FINISH / 64; ++w) { sum += ss[w]; some += sn[w]; }
  finish_loss(a, sum, some);
}

template <typename T, int LPR, int EPL, int V, bool TILED>
__global__ __launch_bounds__(64 * BL_WAVES) void balance_bwd_kernel(BalanceArgs a) {
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane % LPR, slot = lane / LPR;
  const int g = blockIdx.y;
  const T* x0 = static_cast<const T*>(a.x) + (long)g * a.sg;
  T* d0 = static_cast<T*>(a.dx) + (long)g * a.dg;
  const uint8_t* mask = a.mask ? a.mask + (long)g * a.mg : nullptr;
  const float scale = *a.up * a.weight[(long)a.groups * a.experts];
  float w[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) w[j] = a.weight[(long)g * a.experts + min(expert_of<LPR, V>(j, sub), a.experts - 1)];
#pragma unroll
  for (int j = 0; j < EPL; ++j) w[j] = expert_of<LPR, V>(j, sub) < a.experts ? scale * w[j] : 0.f;
  auto work = [&](float (&x)[EPL]) {                        // logits in, gradients out
    int top = turn(__float_as_int(x[0]));
#pragma unroll
    for (int j = 1; j < EPL; ++j) top = max(top, turn(__float_as_int(x[j])));
    const float sum = row_exp<LPR>(top_of<float>(row_max<LPR>(top)), x, x);
    const float inv = sum != 0.f ? __builtin_amdgcn_rcpf(sum) : 0.f;
    // w_e - d with d = sum_j w_j p_j, which is (w_e - r) - sum_j (w_j - r) p_j for any r, the sum of the p_j being 1.  With d's first
    // value for r the second sum is what that value was off by, and neither the rounding of the p_j's sum nor that of a p_j near 1
    // is left in the differences: for a row that one expert has nearly to itself they are as small as what the others have.
    float r = 0.f, d = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) { x[j] *= inv; r = fmaf(x[j], w[j], r); }
    r = row_sum<LPR>(r);
#pragma unroll
    for (int j = 0; j < EPL; ++j) d = fmaf(x[j], w[j] - r, d);
    d = row_sum<LPR>(d);
#pragma unroll
    for (int j = 0; j < EPL; ++j) x[j] = sum != 0.f ? x[j] * ((w[j] - r) - d) : 0.f;      // (a row that does not count: 0 whatever w is)
  };
  if constexpr (TILED) {
    extern __shared__ float tile[];
    const int r = threadIdx.x % a.tile_rows, e0 = threadIdx.x / a.tile_rows, estep = 64 * BL_WAVES / a.tile_rows;
    for (long n0 = (long)blockIdx.x * a.tile_rows; n0 < a.rows; n0 += (long)a.blocks * a.tile_rows) {
      load_tile(a, x0, mask, n0, tile);
      __syncthreads();
      for (int q = wave * RPW; q < a.tile_rows; q += BL_WAVES * RPW) {
        float x[EPL];
        row_of_tile<LPR>(a, tile, q + slot, sub, x);
        work(x);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const int e = expert_of<LPR, 1>(j, sub);
          if (e < a.experts) tile[(q + slot) * a.pitch + e] = x[j];
        }
      }
      __syncthreads();
      if (n0 + r < a.rows) {
        T* d = d0 + (n0 + r) * a.dn;
        for (int e = e0; e < a.experts; e += estep) {
          if constexpr (sizeof(T) == 4) d[(long)e * a.de] = tile[r * a.pitch + e];
          else d[(long)e * a.de] = f32_to_bf16(tile[r * a.pitch + e]);
        }
      }
      __syncthreads();
    }
    return;
  }
  const long step = (long)a.blocks * BL_WAVES * RPW;
  for (long n0 = ((long)blockIdx.x * BL_WAVES + wave) * RPW; n0 < a.rows; n0 += step) {
    const long n = min(n0 + slot, a.rows - 1);
    const bool in = n == n0 + slot;
    RawRow<T, EPL, V> raw;
    float x[EPL];
    fetch_row<T, LPR, EPL, V>(a, x0 + n * a.sn, sub, raw);
    row_values<T, LPR, EPL, V>(a, raw, in && (!mask || mask[n * a.mn]), sub, x);
    work(x);
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

// workgroups per group: enough rows to fill them, two to a CU over all groups (they walk the rows that are left), more for BL_ROWS.  One
// group whose rows a workgroup has done in four rounds stays with one: that saves the two launches that join partials.
long rounds(long rows, int experts) {
  const long per = (long)BL_WAVES * (64 / lanes_per_row(experts));
  return (rows + per - 1) / per;
}
int walkers(long groups, long rows, int experts) {
  const long want = rounds(rows, experts), most = groups >= BL_BLOCKS ? 1 : BL_BLOCKS / groups;
  return (int)std::max(std::min(std::max(want, 1L), most), (want + BL_ROWS - 1) / BL_ROWS);
}
int blocks_for(long groups, long rows, int experts) {
  return groups == 1 && rounds(rows, experts) <= 4 ? 1 : walkers(groups, rows, experts);
}

template <typename T, bool BWD, int LPR, int EPL, int V, bool TILED>
int launch_one(const BalanceArgs& a, const FinishArgs& f, hipStream_t s) {
  const dim3 grid((unsigned)a.blocks, (unsigned)a.groups), block(64 * BL_WAVES);
  const size_t lds = TILED ? std::max((size_t)a.tile_rows * a.pitch * sizeof(float), (size_t)(BWD ? 0 : BL_JOIN * LPR * EPL)) : 0;
  if constexpr (TILED) {
    static std::atomic<unsigned long> allowed{0};           // per device: the tile may take more than 64 KiB
    int dev = 0;
    RM_HIP(hipGetDevice(&dev));
    if (!(allowed.load() >> (dev & 63) & 1)) {
      const void* kernel;
      if constexpr (BWD) kernel = reinterpret_cast<const void*>(&balance_bwd_kernel<T, LPR, EPL, V, TILED>);
      else kernel = reinterpret_cast<const void*>(&balance_fwd_kernel<T, LPR, EPL, V, TILED>);
      RM_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, BL_TILE_BYTES));
      allowed.fetch_or(1ul << (dev & 63));
    }
  }
  if constexpr (BWD) hipLaunchKernelGGL((balance_bwd_kernel<T, LPR, EPL, V, TILED>), grid, block, lds, s, a);
  else hipLaunchKernelGGL((balance_fwd_kernel<T, LPR, EPL, V, TILED>), grid, block, lds, s, a, f);
  RM_LAUNCH_CHECK(BWD ? "balance_bwd" : "balance_fwd");
  return REPMODE_OK;
}

template <typename T, bool BWD, int V, bool TILED>
int launch(const BalanceArgs& a, const FinishArgs& f, hipStream_t s) {
  switch (lanes_per_row(a.experts)) {
    case 1: return launch_one<T, BWD, 1, 8, V, false>(a, f, s);
    case 2: return launch_one<T, BWD, 2, 8, V, false>(a, f, s);
    case 4: return launch_one<T, BWD, 4, 8, V, TILED && BWD>(a, f, s);
    case 8: return launch_one<T, BWD, 8, 8, V, TILED>(a, f, s);
    case 16: return launch_one<T, BWD, 16, 8, V, TILED>(a, f, s);
    case 32: return launch_one<T, BWD, 32, 8, V, TILED>(a, f, s);
    default: return a.experts <= 512 ? launch_one<T, BWD, 64, 8, V, TILED>(a, f, s) : launch_one<T, BWD, 64, 16, V, TILED>(a, f, s);
  }
}

// A pass with the form its strides ask for:
//   16-byte pieces where every row has them: consecutive experts, rows that start at 16 bytes and hold whole pieces;
//   tiles where the rows are neighbours and a row takes so many lanes that a wave's loads along the experts would leave most of a cache
// line -- forward from 8 (2^26 float32 logits, 32 / 64 / 128 / 512 experts, tiles and without, top 1: 92 / 86 / 84 / 87 us and 86 / 135 /
// 235 / 446; bfloat16 73 / 71 / 70 / 78 and 59 / 103 / 148 / 515), backward, which would leave the lines it writes too, from 4 (16 / 24 /
// 64 / 512 experts: 154 / 153 / 137 / 146 and 142 / 247 / 255 / 997; bfloat16 127 / 133 / 110 / 131 and 120 / 180 / 236 / 1132);
//   else element by element.
template <bool BWD>
int dispatch(BalanceArgs a, FinishArgs* finish, int dtype, hipStream_t s) {
  FinishArgs f{};
  if (finish) f = *finish;
  const int per = dtype == REPMODE_F32 ? 4 : 8;
  auto whole = [&](const void* p, long sg, long sn, long se) {
    return ((uintptr_t)p & 15) == 0 && se == 1 && sn % per == 0 && (a.groups == 1 || sg % per == 0);
  };
  if (a.experts % per == 0 && whole(a.x, a.sg, a.sn, a.se) && (!BWD || whole(a.dx, a.dg, a.dn, a.de)))
    return dtype == REPMODE_F32 ? launch<float, BWD, 4, false>(a, f, s) : launch<bf16_t, BWD, 8, false>(a, f, s);
  if (a.se != 1 && a.sn == 1 && lanes_per_row(a.experts) >= (BWD ? 4 : 8)) {
    a.pitch = a.experts | 1;
    a.tile_rows = 64 * BL_WAVES;
    while ((size_t)a.tile_rows * a.pitch * sizeof(float) > BL_TILE_BYTES) a.tile_rows /= 2;
    const long tiles = (a.rows + a.tile_rows - 1) / a.tile_rows;
    // (a tile is rows for at least two rounds of the workgroup, so there are never more workgroups than the plan has)
    if (tiles < a.blocks) a.blocks = (int)(tiles < 1 ? 1 : tiles);
    if (finish) finish->blocks = f.blocks = a.blocks;
    return dtype == REPMODE_F32 ? launch<float, BWD, 1, true>(a, f, s) : launch<bf16_t, BWD, 1, true>(a, f, s);
  }
  return dtype == REPMODE_F32 ? launch<float, BWD, 1, false>(a, f, s) : launch<bf16_t, BWD, 1, false>(a, f, s);
}

int check_shape(const char* who, const void* x, int dtype, long groups, long rows, int experts) {
  RM_REQUIRE(dtype == REPMODE_F32 || dtype == REPMODE_BF16, "%s: bad dtype %d", who, dtype);
  RM_REQUIRE(groups > 0 && groups <= 65535 && rows >= 0 && experts > 0 && experts <= BL_MAX_E,
             "%s: 1..65535 groups, 1..%d experts; got %ld groups of %ld rows over %d experts", who, BL_MAX_E, groups, rows, experts);
  RM_REQUIRE(rows < (1L << 31), "%s: too many rows in a group", who);
  RM_REQUIRE(x || rows == 0, "%s: null pointer", who);
  return REPMODE_OK;
}

}  // namespace

extern "C" int repmode_balance_plan(long groups, long rows, int experts, long* ws_bytes) {
  RM_REQUIRE(ws_bytes, "balance_plan: null pointer");
  if (int rc = check_shape("balance_plan", ws_bytes, REPMODE_F32, groups, rows, experts)) return rc;
  const long blocks = blocks_for(groups, rows, experts);
  *ws_bytes = groups * ((experts + BL_COLUMNS - 1) / BL_COLUMNS + 1) * 8 + groups * blocks * experts * 8 + groups * blocks * 4;
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
  const int parts = (experts + BL_COLUMNS - 1) / BL_COLUMNS;
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
  FinishArgs f{a.psum, a.count, a.valid, a.groups, experts, top_k, a.blocks, coef, term, loss, counts, prob, weight};
  if (int rc = dispatch<false>(a, &f, dtype, s)) return rc;
  if (groups == 1 && f.blocks == 1) return REPMODE_OK;
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
  a.blocks = walkers(groups, rows, experts);
  return dispatch<true>(a, nullptr, dtype, static_cast<hipStream_t>(stream));
}
