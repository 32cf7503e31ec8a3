// The softmax loss of latent factors over the whole catalogue, with its gradients (blp_softmax_loss*).
//
//   z_ij = scale x_i . w_j        lse_i = log sum_j exp z_ij        loss_i = lse_i - z_{i, t_i}
//   dS_ij = g_i (exp(z_ij - lse_i) - [j = t_i])       dX = scale dS W       dW = scale dS^T X
//
// x_i are the rows scored (users), w_j every row of the catalogue, t_i the row's target. The scores are
// never kept. Wide factors: the forward pass reduces each tile of them to a (reference, sum) pair a row, and the backward
// pass recomputes them piece by piece of the catalogue into a workspace of dS, from which the two products of the
// gradient are taken. Narrow factors: k_narrow_lse and k_narrow_grads, and no dS in memory.
//
// The matrix instructions take halves, and dS is no half: rounded to one it would add 2^-8 (bfloat16) of each term to
// gradients that are themselves rounded to 2^-8. It is held as a sum of two, d1 = dS rounded and d2 = dS - d1 rounded, which
// leaves 2^-16 (float16: 2^-22), and both are multiplied: the gradients' products take twice the instructions, six products
// of 2 M N k operations in all (narrow factors: seven, as the scores are computed once more).
//
// Float factors go through the matrix cores as three halves each: x1 = x rounded to bfloat16, x2 = x - x1 rounded,
// x3 = x - x1 - x2, together all 24 bits; of the nine products of two such sums the six largest are taken (the others lie
// below 2^-25 of the product), each exact in the 32-bit accumulators. That is 6 matrix instructions of 16 cycles for
// 16 x 16 x 32 products where the float instructions take 256 cycles.
//
// float16 factors whose rows have gradients of their own are taken as floats ("T" the type they are multiplied as, "ST" the
// one they are stored as): a row's dS may be any times smaller than the largest row's, and float16 ends at 2^-24 where
// bfloat16 planes go on. Gradients 10^7 times below the largest would keep two digits, and lose all at 10^9.
//
// A row whose target lies outside [0, n_cols) is ignored: loss 0, gradient 0, and its x is never multiplied
// (it may hold anything, NaN too).
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "blp_internal.h"
#include "latent.h"

namespace {

using namespace blp::tile;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;

// The matrix instructions' type, and the planes a factor is held in.
constexpr int mma_type(int t) { return t == F32 ? BF16 : t; }
constexpr int planes_of(int t) { return t == F32 ? 3 : 1; }
constexpr int ds_planes_of(int t) { return t == F32 ? 3 : 2; }
// Products of planes that one of the scores (ROW) or of the gradients (COL) takes.
constexpr int segments_of(int t, int layout) { return t == F32 ? 6 : layout == COL ? 2 : 1; }
// float16 holds dS times this: its lowest step is then 2^-38, far below the 2^-24 of a 32-bit difference from 1.
constexpr float extra_of(int t) { return t == F16 ? 16384.f : 1.f; }

using blp::DeviceGuard;
using blp::div_up;
using blp::FastDiv;
using blp::up;
using Targets = blp::Ids;  // the target of row i, or -1 (ignored)

// ---------------------------------------------------------------- packing
// Rows as the tile engine takes them: whole granules of 8 halves (zeros past k), 16-byte aligned; with targets, the
// ignored rows as zeros. Floats go into three planes of halves, `plane` bytes apart; an infinite or NaN factor has nothing
// in the lower planes, one that would round to infinity is cut off. One granule a thread; bound by the copy. Both
// operands in one launch; `flag` (or null) is cleared.
struct PackArgs {
  const char* src;  // null: nothing to pack
  int64_t ld, rows;  // bytes
  Targets targets;
  char* dst;
  int64_t plane;
  unsigned blocks;
};

template <int T, int ST>
__device__ inline void pack_rows(const PackArgs& a, int k, FastDiv per, unsigned block) {
  const int64_t n = a.rows * per.d, step = (int64_t)a.blocks * 256;
  for (int64_t i = block * 256ll + threadIdx.x; i < n; i += step) {
    const int64_t r = n < (1ll << 31) ? (int64_t)per((uint32_t)i) : i / per.d;
    const int e0 = (int)(i - r * per.d) * 8;
    const bool keep = !a.targets.at || a.targets(r) >= 0;
    if constexpr (T == F32) {
      bf16x8 v[3];
      const char* s = a.src + r * a.ld + (int64_t)e0 * size_of(ST);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = keep && e0 + e < k ? load1<ST>(s + e * size_of(ST)) : 0.f;
        const bool finite = fabsf(x) <= 3.4028235e38f;
        __bf16 first = (__bf16)x;
        if (finite && !(fabsf((float)first) <= 3.4e38f)) first = __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(x) >> 16));
        const float rest = finite ? x - (float)first : 0.f;
        const __bf16 second = (__bf16)rest;
        v[0][e] = first;
        v[1][e] = second;
        v[2][e] = (__bf16)(rest - (float)second);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(a.dst + p * a.plane + i * 16) = v[p];
    } else {
      i32x4 v = {0, 0, 0, 0};
      if (keep) {
        const char* s = a.src + r * a.ld + (int64_t)e0 * 2;
        if (e0 + 8 <= k) {
          v = reinterpret_cast<const Unaligned16*>(s)->v;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (e0 + j < k) v[j >> 1] |= (int)((uint32_t)reinterpret_cast<const uint16_t*>(s)[j] << (16 * (j & 1)));
        }
      }
      reinterpret_cast<i32x4*>(a.dst)[i] = v;
    }
  }
}

template <int T, int ST>
__global__ __launch_bounds__(256) void k_pack(PackArgs x, PackArgs w, int k, FastDiv per, uint32_t* flag) {
  if (flag && blockIdx.x == 0 && threadIdx.x == 0) *flag = 0;
  if (blockIdx.x < x.blocks)
    pack_rows<T, ST>(x, k, per, blockIdx.x);
  else
    pack_rows<T, ST>(w, k, per, blockIdx.x - x.blocks);
}

// What the narrow gradients read of a row of x, in blocks of 64 rows: log2(e) lse - log2(extra) (infinite: ignored),
// g / max|g|, the target.
struct Rows {
  float* at;
  __device__ float* of(int64_t block) const { return at + block * 256; }
  __device__ void put(int64_t row, int64_t target, float lse, float extra, float g) const {
    float* to = of(row >> 6) + (row & 63);
    to[0] = target >= 0 ? fmaf(lse, LOG2E, -__builtin_amdgcn_logf(extra)) : INFINITY;
    to[64] = target >= 0 ? g : 0.f;
    reinterpret_cast<int*>(to)[128] = (int)target;
    to[192] = 0.f;
  }
};

// ---------------------------------------------------------------- forward
// Two pairs as one. fmaxf drops a NaN, the sum keeps it (exp2(NaN - base)); an infinite reference gives inf - inf = NaN.
__device__ inline void merge(float& top, float& sum, float t2, float s2) {
  const float t = fmaxf(top, t2);
  const float base = t == -INFINITY ? 0.f : t;
  sum = sum * __builtin_amdgcn_exp2f(top - base) + s2 * __builtin_amdgcn_exp2f(t2 - base);
  top = t;
}

// One (reference, sum of exp2(z - reference)) pair a row and wave tile, in base 2: part[tile * rows + row].
// Each lane takes its first score as its reference, which does as long as no sum grows past 2^60; only where one
// does (or a score is infinite or NaN) the maximum is taken: 16 cycles a 64 scores instead of 22 or more.
// 8,192 x 100,000 x 1,024 bf16: 1.71 ms, 980 TFLOP/s; the engine alone runs at 1,223 for this k.
template <int T>
struct EpiLse {
  float2* part;
  float* hit;  // z of the target
  Targets targets;
  int64_t n, m;
  float scale;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int tile, int, lds_char*) const {
    if (p0 >= n || q0 >= m) {
      const int64_t row = q0 + (threadIdx.x & 63);  // a wave past the catalogue's end still owns its pairs
      if (q0 < m && (int)(threadIdx.x & 63) < S::FQ * 16)
        for (int64_t r = row; r < min(m, q0 + S::FQ * 16); r += 64) part[(int64_t)tile * m + r] = make_float2(-INFINITY, 0.f);
      return;
    }
    const int lane = fresh_lane(), l = lane & 15, h = lane >> 4;
    const int left = (int)min(n - p0, (int64_t)(S::FP * 16)), rows = (int)min(m - q0, (int64_t)(S::FQ * 16));
    const float c = scale * LOG2E;
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      const int64_t row = q0 + min(j * 16 + l, rows - 1), t = targets(row) - p0;
      const bool here = j * 16 + l < rows && t >= 0 && t < left && ((t >> 2) & 3) == h;  // this lane holds the target's score
      if (left < S::FP * 16) {
#pragma unroll
        for (int i = 0; i < S::FP; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i * 16 + h * 4 + e >= left) acc[i][j][e] = scale < 0.f ? INFINITY : -INFINITY;
      }
      if (__any(here)) {
        const int at = here ? (int)t - h * 4 : -1;
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < S::FP; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) z = at == i * 16 + e ? acc[i][j][e] : z;
        if (here) hit[row] = z * scale;
      }
      float top = acc[0][j][0] * c, sum = 0.f;
#pragma unroll
      for (int i = 0; i < S::FP; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, -top));
      if (__any(!(sum < 0x1p60f))) {
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < S::FP; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool past = left < S::FP * 16 && i * 16 + h * 4 + e >= left;  // for a scale of 0: inf 0 is NaN
            acc[i][j][e] = past ? -INFINITY : acc[i][j][e] * c;
            top = fmaxf(top, acc[i][j][e]);
          }
        const float base = top == -INFINITY ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < S::FP; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(acc[i][j][e] - base);
      }
#pragma unroll
      for (int o = 16; o <= 32; o <<= 1) merge(top, sum, __shfl_xor(top, o, 64), __shfl_xor(sum, o, 64));
      if (h == 0 && j * 16 + l < rows) part[(int64_t)tile * m + row] = make_float2(top, sum);
    }
  }
};

// total[0] = the sum of the losses, or their mean over the rows not ignored; total[1] = their number. By one block, in
// fixed order and in 64 bits: the same result every time.
struct Total {
  float* at;
  int mean;
};
template <int THREADS>
__device__ inline void take_total(const float* loss, const Targets& targets, int64_t m, const Total& t) {
  __shared__ double s_sum[THREADS / 64];
  __shared__ int64_t s_n[THREADS / 64];
  double sum = 0.0;
  int64_t n = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < m; i += THREADS) {  // the losses of ignored rows are 0
    sum += loss[i];
    n += targets(i) >= 0;
  }
  for (int o = 32; o; o >>= 1) {
    sum += __shfl_xor(sum, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    s_sum[threadIdx.x >> 6] = sum;
    s_n[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 64; ++i) {
      sum += s_sum[i];
      n += s_n[i];
    }
    t.at[0] = (float)(t.mean ? sum / (double)max(n, (int64_t)1) : sum);
    t.at[1] = (float)max(n, (int64_t)1);
  }
}

__global__ __launch_bounds__(1024) void k_total(const float* __restrict__ loss, Targets targets, int64_t m, Total total) {
  take_total<1024>(loss, targets, m, total);
}

// R rows a block, 256 / R threads a row over the tiles' pairs: 32 rows read whole lines of pairs, 4 rows have 64 threads
// each where there are too few rows to fill the card. Leaves the rows' parameters of the narrow gradients (`rows`), and
// with `done` (0 before) the block that ends last takes the total. The rows from `row0` on.
template <int R>
__global__ __launch_bounds__(256) void k_join(const float2* __restrict__ part, int64_t tiles, int64_t m, int64_t row0,
                                              const float* __restrict__ hit, Targets targets, float* __restrict__ loss,
                                              float* __restrict__ lse, Rows rows, float extra, Total total, uint32_t* done) {
  constexpr int G = 256 / R;
  __shared__ float2 s_part[G][R];
  __shared__ int s_last;
  const int r = threadIdx.x & (R - 1), g = threadIdx.x / R;
  const int64_t row = row0 + blockIdx.x * (int64_t)R + r;
  float top = -INFINITY, sum = 0.f;
  if (row < m) {
    int64_t t = g;
    for (; t + 3 * G < tiles; t += 4 * G) {
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = part[(t + u * G) * m + row];
#pragma unroll
      for (int u = 0; u < 4; ++u) merge(top, sum, v[u].x, v[u].y);
    }
    for (; t < tiles; t += G) {
      const float2 v = part[t * m + row];
      merge(top, sum, v.x, v.y);
    }
  }
  s_part[g][r] = make_float2(top, sum);
  for (int half = G / 2; half; half >>= 1) {
    __syncthreads();
    if (g < half) {
      merge(top, sum, s_part[g + half][r].x, s_part[g + half][r].y);
      s_part[g][r] = make_float2(top, sum);
    }
  }
  if (g == 0 && row < m) {
    const float l = (top + __builtin_amdgcn_logf(sum)) * LN2;  // logf: base 2
    const int64_t t = targets(row);
    lse[row] = l;
    loss[row] = t >= 0 ? l - hit[row] : 0.f;
    if (rows.at) rows.put(row, t, l, extra, 1.f);
  } else if (g == 0 && rows.at && row < (m + 63) / 64 * 64) {
    rows.put(row, -1, 0.f, extra, 0.f);
  }
  if (!done) return;
  __threadfence();  // this block's losses are seen by the device before its mark is
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(done, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  take_total<256>(loss, targets, m, total);
}

// ---------------------------------------------------------------- backward
// What the gradient of row i is multiplied with: g_i / count. dS holds g_i / max|g| times the softmax
// difference, in [-1, 1] (halves keep 14 more bits below that), and the products' epilogues put the
// magnitude back in 32 bits.
struct RowGrad {
  const float* g;      // [rows] (stride 1), one value (stride 0), or null: 1
  int stride;
  const float* count;  // divide by this, or null
  const float* top;    // max |g| (stride 1), or null
  float extra;         // the halves' factor
  __device__ float row(int64_t i) const {  // in [-1, 1] times extra
    if (!g || !stride) return extra;
    const float t = *top, v = g[i];
    if (!(fabsf(v) <= FLT_MAX)) return v;  // an infinite or NaN gradient: its row's, and the catalogue's
    return t > 0.f ? v / t * extra : 0.f;
  }
  __device__ double all() const {  // in 64 bits: times a scale it may leave the floats' range where the gradient does not
    const double f = (g ? (stride ? *top : *g) : 1.f) / (double)extra;
    return count ? f / *count : f;
  }
};

// top = max |g| of the finite row gradients (1 if there is none).
__global__ __launch_bounds__(1024) void k_top_grad(const float* __restrict__ g, Targets targets, int64_t m,
                                                   float* __restrict__ top) {
  __shared__ float s_top[16];
  float t = -1.f;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < m; i += 1024) {
    const float v = fabsf(g[i]);
    t = targets(i) >= 0 && v <= FLT_MAX ? fmaxf(t, v) : t;
  }
  for (int o = 32; o; o >>= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
  if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) t = fmaxf(t, s_top[i]);
    *top = t < 0.f ? 1.f : t;
  }
}

// dS of one piece: ds[row * ld + p], zeros past the catalogue's end. A piece of 8,192 x 14,336 x 1,024 bf16 0.31 ms, 770
// TFLOP/s with 0.47 GB written; dX and dW of it, which read that, 0.45 and 0.49 ms (1,070 and 990).
template <int T>
struct EpiGrad {
  char* ds;
  int64_t ld;     // elements
  int64_t plane;  // bytes between the planes of dS
  const float* lse;
  RowGrad g;
  Targets targets;
  int64_t j0;  // the piece's first column
  int64_t n, m;
  float scale;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int, int, lds_char* scratch) const {
    if (p0 >= ld || q0 >= m) return;
    const int lane = fresh_lane(), l = lane & 15, h = lane >> 4;
    const float c = scale * LOG2E;
    const int left = (int)min(n - p0, (int64_t)(S::FP * 16)), rows = (int)min(m - q0, (int64_t)(S::FQ * 16));
    int hit[S::FQ];   // the target's place in the lane's block; far off: none
    bool any[S::FQ];  // in one of the wave's lanes
    float gr[S::FQ], l2[S::FQ];
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) {
      const int64_t row = q0 + min(j * 16 + l, rows - 1), t = targets(row), at = t - j0 - p0;
      hit[j] = t >= 0 && at >= 0 && at < S::FP * 16 ? (int)at - h * 4 : -1000;
      any[j] = __any(hit[j] != -1000);
      gr[j] = t >= 0 ? g.row(row) : 0.f;
      l2[j] = t >= 0 ? -lse[row] * LOG2E : -INFINITY;
    }
    constexpr int MT = mma_type(T);
    const int width = (int)min(ld - p0, (int64_t)(S::FP * 16));
    char* at = ds + (q0 * ld + p0) * size_of(MT);
    auto value = [&](int i, int j) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, l2[j]));
      if (any[j]) {  // rare
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (hit[j] == i * 16 + e) v[e] -= 1.f;
      }
      v *= gr[j];
      if (left < S::FP * 16) {  // the catalogue's last rows
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i * 16 + h * 4 + e >= left) v[e] = 0.f;
      }
      return v;
    };
#pragma unroll
    for (int i = 0; i < S::FP; ++i)
#pragma unroll
      for (int j = 0; j < S::FQ; ++j) acc[i][j] = value(i, j);
#pragma unroll 1
    for (int p = 0; p < ds_planes_of(T); ++p) {
      store_block<MT, S>(scratch, at + p * plane, ld * size_of(MT), width, rows, [&](int i, int j) { return acc[i][j]; });
      typedef std::conditional_t<MT == BF16, __bf16, _Float16> Half;
#pragma unroll
      for (int i = 0; i < S::FP; ++i)
#pragma unroll
        for (int j = 0; j < S::FQ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] -= (float)(Half)acc[i][j][e];  // what the plane left over
    }
  }
};

// out[q][p] = alpha acc, rounded once.
template <int T>
struct EpiOut {
  char* out;
  int64_t ld;  // bytes
  int64_t np, nq;
  RowGrad g;
  float scale;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int, int, lds_char* scratch) const {
    if (p0 >= np || q0 >= nq) return;
    const double alpha = scale * g.all();
    const int left = (int)min(np - p0, (int64_t)(S::FP * 16)), rows = (int)min(nq - q0, (int64_t)(S::FQ * 16));
    store_block<T, S>(scratch, out + q0 * ld + p0 * size_of(T), ld, left, rows, [&](int i, int j) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)(acc[i][j][e] * alpha);
      return v;
    });
  }
};

// part[slice][q][p] (+)= acc: the sums over slices of k and pieces of the catalogue, in 32 bits.
struct EpiPart {
  float* part;
  int64_t ld, np, nq;  // elements; ld a multiple of 4
  int add;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int, int slice, lds_char*) const {
    const int lane = fresh_lane(), h = lane >> 4;
    float* base = part + (int64_t)slice * nq * ld;
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) {
      const int64_t q = q0 + j * 16 + (lane & 15);
      if (q >= nq) continue;
#pragma unroll
      for (int i = 0; i < S::FP; ++i) {
        const int64_t p = p0 + i * 16 + h * 4;
        if (p >= ld) continue;
        f32x4* at = reinterpret_cast<f32x4*>(base + q * ld + p);
        *at = add ? *at + acc[i][j] : acc[i][j];
      }
    }
  }
};

// out = alpha sum_s part[s], always in the same order: G threads an output of four, thread g the slices g, g + G, ...,
// then the threads' sums. G = 16 where the slices are many and the outputs few. Two of them a launch.
struct SumArgs {
  const float* part;
  int slices;
  int64_t nq;
  char* out;
  int64_t ldo;  // bytes
  unsigned blocks;
};

template <int T, int G>
__device__ inline void sum_rows(const SumArgs& a, int64_t np, FastDiv per, double alpha, unsigned block, f32x4* s_sum) {
  constexpr int V = 256 / G;
  const int64_t n = a.nq * per.d;
  const int v = threadIdx.x & (V - 1), gr = threadIdx.x / V;
  for (int64_t i0 = block * (int64_t)V; i0 < n; i0 += (int64_t)a.blocks * V) {
    const int64_t i = i0 + v;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (i < n) {
      const float* at = a.part + i * 4;  // a row is per.d fours: rows follow one another
#pragma unroll 4
      for (int s = gr; s < a.slices; s += G) sum += *reinterpret_cast<const f32x4*>(at + s * (n * 4));
    }
    if constexpr (G > 1) {
      __syncthreads();
      s_sum[threadIdx.x] = sum;
      __syncthreads();
      if (gr > 0) continue;
      for (int k = 1; k < G; ++k) sum += s_sum[k * V + v];
    }
    if (i < n) {
      const int64_t q = n < (1ll << 31) ? (int64_t)per((uint32_t)i) : i / per.d, p = (i - q * per.d) * 4;
      for (int e = 0; e < 4; ++e)
        if (p + e < np) store1<T>(a.out + q * a.ldo + (p + e) * size_of(T), (float)(sum[e] * alpha));
    }
  }
}

template <int T, int G>
__global__ __launch_bounds__(256) void k_sum_parts(SumArgs a, SumArgs b, int64_t np, FastDiv per, RowGrad g, float scale) {
  __shared__ f32x4 s_sum[G > 1 ? 256 : 1];
  const double alpha = scale * g.all();
  if (blockIdx.x < a.blocks)
    sum_rows<T, G>(a, np, per, alpha, blockIdx.x, s_sum);
  else
    sum_rows<T, G>(b, np, per, alpha, blockIdx.x - a.blocks, s_sum);
}

// ---------------------------------------------------------------- narrow factors
// Halves with k up to 128, floats up to 64: the scores never leave the registers, in the backward pass either. A wave holds
// 32 rows of one side ("own") as fragments for the whole kernel and the other side ("stream") passes through LDS, 64 rows
// a stage:
//   LSE  own x, stream w: a running sum of exp2(score - reference) a lane, joined over the lanes at the end
//   DX   own x, stream w: dS of 32 stream rows at a time, as two halves each (floats: three), is the second product's
//        operand as it lies (the matrix instruction's k order is free, so its rows of w are read from LDS,
//        transposed, in the order in which the lanes hold dS); dx accumulates in registers
//   DW   own w, stream x: the same with the sides changed
// 64 scores at k = 64 need 8 (LSE) or 24 (DX, DW) cycles of a SIMD's matrix unit and about 17 (LSE) or 27 of its vector unit, 8
// of them exp2; two waves' shares of the two units overlap by half at most on this chip. 10,000 x 100,000 x 64: LSE 184 to
// 220 us (of the cycles that a compute unit is busy its vector unit is in 87%, the matrix unit in 32%, LDS in 16%), both
// gradients 730 to 840 us (77%, 53%, 20%). Computing the exponentials again in DX and DW costs less than writing dS once and
// reading it twice: that took 2.36 ms in all with one plane of it.
// Larger waves (64 rows: 275 us for LSE) hide less of each other's waits, one more stage ahead does not matter.
__global__ __launch_bounds__(64) void k_rows(const float* __restrict__ lse, RowGrad g, Targets targets, int64_t m, Rows rows) {
  const int64_t i = blockIdx.x * 64ll + threadIdx.x;
  const int64_t t = i < m ? targets(i) : -1;
  rows.put(i, t, t >= 0 ? lse[i] : 0.f, g.extra, t >= 0 ? g.row(i) / g.extra : 0.f);
}

enum NarrowMode { LSE, DX, DW };

struct NarrowArgs {
  Operand own, stream;
  int64_t own_plane, stream_plane;  // floats: bytes between the planes
  int kp;
  int64_t range;  // stream rows of a split, a multiple of 64
  int own_tiles, splits;
  float scale, extra;
  Targets targets;  // LSE
  float2* part;     // LSE
  float* hit;       // LSE
  Rows rows;        // DX, DW
};

template <int KS_, int FO_>
struct NarrowShape {  // the second product's accumulators, for the epilogues
  static constexpr int FP = 2 * KS_, FQ = FO_, SCRATCH = 16384;
};

// Two values as halves; `rest`: they become what that left over.
template <int T>
__device__ inline int pack2(float& a, float& b, bool rest) {
  if constexpr (T == BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const int both = __builtin_bit_cast(int, b2{(__bf16)a, (__bf16)b});
    if (rest) {
      a -= __uint_as_float((uint32_t)both << 16);
      b -= __uint_as_float((uint32_t)both & 0xffff0000u);
    }
    return both;
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 both = {(_Float16)a, (_Float16)b};
    if (rest) {
      a -= (float)both[0];
      b -= (float)both[1];
    }
    return __builtin_bit_cast(int, both);
  }
}

// LDS of a workgroup: a stage's rows, and three buffers of them (floats: two, a stage of theirs lasts longer).
template <int T, int KS>
struct NarrowLds {
  static constexpr int HALVES = KS > 2 ? 2 : 1;  // 128-byte parts of a row
  static constexpr int PART = 64 * STAGE;        // bytes of one part of a stage
  static constexpr int BUF = planes_of(T) * HALVES * PART;
  static constexpr bool THREE = T != F32;
};

template <int T, int ST, int KS, int MODE, bool PER_ROW, class Epi>
__device__ __attribute__((always_inline)) inline void narrow_body(const NarrowArgs& a, const Epi& epi, int block, char* s_a, char* s_b,
                                                                  char* s_c, char* s_ra, char* s_rb, char* s_rc) {
  constexpr int MT = mma_type(T), PL = planes_of(T), PD = ds_planes_of(T);
  constexpr int FO = 2;  // own fragments of 16 rows a wave
  constexpr int HALVES = NarrowLds<T, KS>::HALVES, PART = NarrowLds<T, KS>::PART, BUF = NarrowLds<T, KS>::BUF;
  constexpr bool THREE = NarrowLds<T, KS>::THREE;
  constexpr int COPIES = 2 * PL * HALVES + (MODE == DW);  // a wave issues for a stage
  // a die's workgroups take neighbouring own tiles of one split: the split's rows stay in its L2
  const int n_blocks = a.own_tiles * a.splits, per = n_blocks >> 3, more = n_blocks & 7, xcd = block & 7;
  if (block >= n_blocks) return;
  const int id = xcd * per + min(xcd, more) + (block >> 3);
  const int split = id / a.own_tiles, own_tile = id - split * a.own_tiles;
  const int lane = threadIdx.x & 63, l = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t own0 = (int64_t)own_tile * (64 * FO) + wave * (16 * FO);
  const int64_t s0 = split * a.range, s1 = min(a.stream.rows, s0 + a.range);
  const int stages = (int)((s1 - s0 + 63) >> 6);
  const float c = fabsf(a.scale) * LOG2E;
  const Operand stream = {a.stream.base, a.stream.ld, s1};

  frag_t own[PL][FO][KS];
#pragma unroll
  for (int p = 0; p < PL; ++p)
#pragma unroll
    for (int j = 0; j < FO; ++j) {
      const int64_t r = own0 + j * 16 + l;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        own[p][j][s] = frag_t{0, 0, 0, 0};
        if (r < a.own.rows && s * 32 + h * 8 < a.kp)
          own[p][j][s] = *reinterpret_cast<const frag_t*>(a.own.base + p * a.own_plane + r * a.own.ld + (s * 32 + h * 8) * 2);
        if (a.scale < 0.f) own[p][j][s] ^= (int)0x80008000;  // the scores' sign, so that c is positive
      }
    }
  // a lane's own rows: LSE: targets; DX: lse and targets; DW: w rows (nothing)
  int target[FO];
  float lane_l2[FO], lane_g[FO];
#pragma unroll
  for (int j = 0; j < FO; ++j) {
    const int64_t r = own0 + j * 16 + l;
    target[j] = -1;
    lane_l2[j] = INFINITY;
    lane_g[j] = 0.f;
    if constexpr (MODE == LSE) {
      if (r < a.own.rows) target[j] = (int)a.targets(r);
    } else if constexpr (MODE == DX) {
      if (r < a.own.rows) {
        const float* at = a.rows.of(r >> 6) + (r & 63);
        lane_l2[j] = at[0];
        lane_g[j] = at[64];
        target[j] = reinterpret_cast<const int*>(at)[128];
      }
    }
  }
  // LSE: the reference of the sum, a score or a maximum (not yet times c), its -top c (0 while it is infinite), the sum
  float top[FO], shift[FO], sum[FO];
  f32x4 out[2 * KS][FO];            // DX, DW
#pragma unroll
  for (int j = 0; j < FO; ++j) {
    top[j] = -INFINITY;
    shift[j] = 0.f;
    sum[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i) out[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t base_row = lane_base<MT, ROW, 64>();
  const uint32_t base_tr = (4 * h + (l >> 2)) * STAGE + (((l & 3) >> 1) ^ (4 * (h & 1) + (l >> 2))) * 16 + (l & 1) * 8;

  auto load = [&](char* buf, char* rbuf, int t) {
    const int64_t r0 = s0 + (int64_t)t * 64;
#pragma unroll
    for (int p = 0; p < PL; ++p)
#pragma unroll
      for (int s = 0; s < HALVES; ++s)
        load_stage<MT, ROW, 64, 4>((lds_char*)buf + (p * HALVES + s) * PART,
                                   Operand{stream.base + p * a.stream_plane, stream.ld, s1}, r0, s * 64, a.kp);
    if constexpr (MODE == DW)  // by every wave alike, so that their counts agree
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_at((const char*)a.rows.of(min(r0, a.stream.rows - 1) >> 6)),
                                               (__attribute__((address_space(3))) void*)(lds_char*)rbuf, 16, lane * 16, 0, 0, 0);
  };
  auto compute = [&](const char* buf, const char* rbuf, int t) {
    const lds_char* lds = (const lds_char*)buf;
    const int r0 = (int)(s0 + (int64_t)t * 64);  // stream rows fit 31 bits
    if (r0 >= (int)s1) return;
    // 32 stream rows' products with the own rows
    auto products = [&](int half, f32x4(&acc)[2][FO]) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int x = 0; x < PL; ++x) {
          frag_t p[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            p[i] = read_frag<MT, ROW, 64>(lds + (x * HALVES + (s >> 1)) * PART, base_row, half * 2 + i, s & 1);
#pragma unroll
          for (int y = 0; y < PL - x; ++y)  // floats: the six larger products of the planes
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int j = 0; j < FO; ++j)
                acc[i][j] = mma<MT>(p[i], own[y][j][s], s + x + y ? acc[i][j] : f32x4{0.f, 0.f, 0.f, 0.f});
        }
    };
    if constexpr (MODE == LSE) {
      bool here = false, slow = s1 - r0 < 64;
#pragma unroll
      for (int j = 0; j < FO; ++j) here |= (unsigned)(target[j] - r0) < 64u;
      const bool any = __any(here);
      if (!__any(slow)) {
        // Each lane's first score is its reference, and does as long as no sum grows past 2^60 (or is NaN): no maximum to take.
        float add[FO];
#pragma unroll
        for (int j = 0; j < FO; ++j) add[j] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          f32x4 acc[2][FO];
          products(half, acc);
          if (half == 0 && t == 0) {
#pragma unroll
            for (int j = 0; j < FO; ++j) {
              top[j] = acc[0][j][0];
              shift[j] = -top[j] * c;
            }
          }
          if (any) {  // the targets' scores: rare
            const int first = r0 + half * 32 + h * 4;
#pragma unroll
            for (int j = 0; j < FO; ++j) {
              const int at = target[j] - first;
              float z = 0.f;
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) z = at == i * 16 + e ? acc[i][j][e] : z;
              if ((unsigned)at < 32u && (at & 12) == 0) a.hit[own0 + j * 16 + l] = z * fabsf(a.scale);
            }
          }
#pragma unroll
          for (int j = 0; j < FO; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) add[j] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, shift[j]));
        }
#pragma unroll
        for (int j = 0; j < FO; ++j) slow |= !(add[j] < 0x1p60f);
        if (!__any(slow)) {
#pragma unroll
          for (int j = 0; j < FO; ++j) sum[j] += add[j];
          return;
        }
        if (t == 0) {  // no reference yet that holds
#pragma unroll
          for (int j = 0; j < FO; ++j) {
            top[j] = -INFINITY;
            shift[j] = 0.f;
          }
        }
      }
      // The range's last stage, and rows that rise far or hold a NaN: rare. A NaN keeps its wave's 32 rows here: 10,000 x 100,000
      // x 64 bf16 200 us without one, 250 with one, 510 with one in every 32 rows.
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        f32x4 acc[2][FO];
        products(half, acc);
        const int first = r0 + half * 32 + h * 4;  // the lane's stream rows: first + 16 i + e
#pragma unroll
        for (int j = 0; j < FO; ++j) {
          float high = top[j];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = first + i * 16 + e;
              if (r == target[j] && r < (int)s1) a.hit[own0 + j * 16 + l] = acc[i][j][e] * fabsf(a.scale);
              if (r < (int)s1) high = fmaxf(high, acc[i][j][e]);  // past the range's end: zeros in LDS
            }
          if (high > top[j]) {
            if (top[j] != -INFINITY) sum[j] *= __builtin_amdgcn_exp2f((top[j] - high) * c);
            top[j] = high;
            shift[j] = -high * c;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (first + i * 16 + e < (int)s1) sum[j] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, shift[j]));
        }
      }
    } else {
      const __attribute__((address_space(3))) float* rp = (const __attribute__((address_space(3))) float*)(const lds_char*)rbuf;
      bool mine = false;  // a target of these rows lies in this wave's block
      if constexpr (MODE == DX) {
#pragma unroll
        for (int j = 0; j < FO; ++j) mine |= (unsigned)(target[j] - r0) < 64u;
      } else {
        const int t64 = ((const __attribute__((address_space(3))) int*)rp)[128 + lane];
        mine = (unsigned)(t64 - (int)own0) < 16u * FO;
      }
      const bool any = __any(mine), cut = (int)s1 - r0 < 64;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x4 acc[2][FO];
        products(half, acc);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x4 l2, g;
          if constexpr (MODE == DW) {
            l2 = *(const __attribute__((address_space(3))) f32x4*)(rp + half * 32 + i * 16 + h * 4);
            if constexpr (PER_ROW) g = *(const __attribute__((address_space(3))) f32x4*)(rp + 64 + half * 32 + i * 16 + h * 4);
          }
#pragma unroll
          for (int j = 0; j < FO; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (MODE == DX)
                acc[i][j][e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, -lane_l2[j]));
              else
                acc[i][j][e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, -l2[e]));
            }
          if (MODE == DX && cut) {  // past the range's end: exp2(-lse) of any size, times rows of zeros
#pragma unroll
            for (int j = 0; j < FO; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (r0 + half * 32 + i * 16 + h * 4 + e >= (int)s1) acc[i][j][e] = 0.f;
          }
          if (any) {  // rare
            if constexpr (MODE == DX) {
#pragma unroll
              for (int j = 0; j < FO; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (target[j] == r0 + half * 32 + i * 16 + h * 4 + e) acc[i][j][e] -= a.extra;
            } else {
              const i32x4 t = *(const __attribute__((address_space(3))) i32x4*)(rp + 128 + half * 32 + i * 16 + h * 4);
#pragma unroll
              for (int j = 0; j < FO; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (t[e] == (int)own0 + j * 16 + l) acc[i][j][e] -= a.extra;
            }
          }
          if constexpr (MODE == DW && PER_ROW)
#pragma unroll
            for (int j = 0; j < FO; ++j) acc[i][j] *= g;
        }
        frag_t q[PD][FO];
#pragma unroll
        for (int p = 0; p < PD; ++p)
#pragma unroll
          for (int j = 0; j < FO; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                float a = acc[i][j][2 * w], b = acc[i][j][2 * w + 1];
                q[p][j][2 * i + w] = pack2<MT>(a, b, p + 1 < PD);
                acc[i][j][2 * w] = a;
                acc[i][j][2 * w + 1] = b;
              }
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
          for (int x = 0; x < PL; ++x) {
            const lds_char* at = lds + (base_tr ^ ((d & 3) << 5)) + (x * HALVES + (d >> 2)) * PART + half * 32 * STAGE;
            i32x4 v;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const s16x4 tr = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + s * 16 * STAGE));
              const i32x2 w = __builtin_bit_cast(i32x2, tr);
              v[2 * s] = w[0];
              v[2 * s + 1] = w[1];
            }
#pragma unroll
            for (int y = 0; y < PD - x; ++y)
#pragma unroll
              for (int j = 0; j < FO; ++j) out[d][j] = mma<MT>(v, q[y][j], out[d][j]);
          }
      }
    }
  };

  // Three buffers, two stages ahead (floats: two, one ahead). Stages past the range copy zeros and are not computed, so
  // every trip takes all buffers and the counts of outstanding copies stay the same.
  load(s_a, s_ra, 0);
  if constexpr (THREE) {
    load(s_b, s_rb, 1);
#pragma unroll 1
    for (int t = 0; t < stages; t += 3) {
      ring_barrier<COPIES>();
      load(s_c, s_rc, t + 2);
      compute(s_a, s_ra, t);
      ring_barrier<COPIES>();
      load(s_a, s_ra, t + 3);
      compute(s_b, s_rb, t + 1);
      ring_barrier<COPIES>();
      load(s_b, s_rb, t + 4);
      compute(s_c, s_rc, t + 2);
    }
  } else {
#pragma unroll 1
    for (int t = 0; t < stages; t += 2) {
      ring_barrier<0>();
      load(s_b, s_rb, t + 1);
      compute(s_a, s_ra, t);
      ring_barrier<0>();
      load(s_a, s_ra, t + 2);
      compute(s_b, s_rb, t + 1);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // nothing in flight towards LDS when the workgroup ends

  if constexpr (MODE == LSE) {
#pragma unroll
    for (int j = 0; j < FO; ++j) {
      float m = top[j] == -INFINITY ? top[j] : top[j] * c;
#pragma unroll
      for (int o = 16; o <= 32; o <<= 1) merge(m, sum[j], __shfl_xor(m, o, 64), __shfl_xor(sum[j], o, 64));
      const int64_t r = own0 + j * 16 + l;
      if (h == 0 && r < a.own.rows) a.part[(int64_t)split * a.own.rows + r] = make_float2(m, sum[j]);
    }
  } else {
    if constexpr (MODE == DX && PER_ROW)
#pragma unroll
      for (int j = 0; j < FO; ++j)
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d) out[d][j] *= lane_g[j];
    lds_char* scratch;
    {  // a wave's 32 rows of up to 128 halves: the ring's buffers in parts
      __syncthreads();
      constexpr int WAVE = 16 * FO * pow2_up(32 * KS * size_of(ST));
      if constexpr (WAVE * 4 <= BUF)
        scratch = (lds_char*)s_a + wave * WAVE;
      else
        scratch = wave < 2 ? (lds_char*)s_a + wave * WAVE : (lds_char*)s_b + (wave - 2) * WAVE;
      static_assert(WAVE * 2 <= BUF, "two waves a buffer");
    }
    epi.template run<NarrowShape<KS, FO>>(out, 0, own0, 0, split, scratch);
  }
}

template <int T, int KS>
__global__ __launch_bounds__(256, KS > 2 || T == F32 ? 3 : 4) void k_narrow_lse(NarrowArgs a) {
  using L = NarrowLds<T, KS>;
  __shared__ __attribute__((aligned(1024))) char s_a[L::BUF], s_b[L::BUF], s_c[L::THREE ? L::BUF : 16];
  narrow_body<T, T, KS, LSE, false>(a, 0, blockIdx.x, s_a, s_b, s_c, nullptr, nullptr, nullptr);
}

// A gradient's outputs: splits' partial sums, or rounded in place.
template <int T>
struct EpiGradient {
  bool parts;
  EpiPart part;
  EpiOut<T> out;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int tile, int slice, lds_char* scratch) const {
    if (parts)
      part.template run<S>(acc, p0, q0, tile, slice, scratch);
    else
      out.template run<S>(acc, p0, q0, tile, slice, scratch);
  }
};

// Both gradients in one launch: the workgroups of one fill the compute units that the other's leave (10,000 x 100,000
// x 64: 782 workgroups of dw alone keep three quarters of the card's slots busy).
template <int T, int ST, int KS, bool PER_ROW>
__global__ __launch_bounds__(256, KS > 2 || T == F32 ? 3 : 4) void k_narrow_grads(NarrowArgs w, EpiGradient<ST> ew, int w_blocks,
                                                                                  NarrowArgs x, EpiGradient<ST> ex) {
  using L = NarrowLds<T, KS>;
  __shared__ __attribute__((aligned(1024))) char s_a[L::BUF], s_b[L::BUF], s_c[L::THREE ? L::BUF : 16];
  __shared__ __attribute__((aligned(1024))) char s_ra[1024], s_rb[1024], s_rc[L::THREE ? 1024 : 16];
  if ((int)blockIdx.x < w_blocks)
    narrow_body<T, ST, KS, DW, PER_ROW>(w, ew, blockIdx.x, s_a, s_b, s_c, s_ra, s_rb, s_rc);
  else
    narrow_body<T, ST, KS, DX, PER_ROW>(x, ex, blockIdx.x - w_blocks, s_a, s_b, s_c, s_ra, s_rb, s_rc);
}

// ---------------------------------------------------------------- host side
// dS of one piece of the catalogue, all planes: 8,192 x 100,000 x 1,024 halves take 10.1 ms a step; 128 MiB 10.7, 256 MiB
// 10.3, 1 GiB 10.4 (smaller pieces pay for dx's sums, which each adds to, larger ones for dS leaving the last-level cache).
constexpr int64_t PIECE_BYTES = 512ll << 20;
constexpr int64_t JOINED = 1ll << 28;         // rows of a launch of k_join, 8 threads each: less than 2^32 threads
constexpr int64_t PAIR_BYTES = 256ll << 20;   // the forward pass's pairs of the rows taken at a time

enum ShapeId { BIG, MID, FLAT, THIN };
using Flat = Shape<4, 1, 4, 2>;  // 256 x 32, two: few rows
using Thin = Shape<4, 1, 1, 2>;  // 64 x 32, four: few tiles
constexpr int BP_OF[] = {256, 128, 256, 64}, BQ_OF[] = {256, 128, 32, 32}, WP_OF[] = {2, 2, 4, 4}, PER_CU[] = {1, 2, 2, 4};

int64_t tiles_of(int shape, int64_t np, int64_t nq) { return div_up(np, BP_OF[shape]) * div_up(nq, BQ_OF[shape]); }

// A stage of every tile, in us: 1.55 a round of the large shape and, two workgroups side by side, 1.2 of the middle one
// (8,192 x 100,000 x 1,024 halves: 980 and 860 TFLOP/s). Where there are few tiles a compute unit's way to memory counts, and
// small ones on many of them are faster: 80 x 267 x 1,728 halves, 75 us a step in tiles of 128 x 128 and 47 in 64 x 32; 15 x
// 3,344 x 240 floats, 75 us in 256 x 32 and 55; but 200 x 20,000 x 512 halves 92 and 121.
double stage_us(int shape, int64_t tiles) {
  const int64_t slots = 256 * PER_CU[shape], each = std::min<int64_t>(div_up(tiles, 256), PER_CU[shape]);
  static const double thin[] = {0.4, 0.55, 0.75, 1.0};
  return (double)div_up(tiles, slots) * (shape == BIG ? 1.55 : shape == THIN ? thin[each - 1] : each > 1 ? 1.2 : 0.8);
}
// Up to 32 rows: tiles of 32.
bool fits(int shape, int64_t nq) { return shape == THIN || (shape == FLAT) == (nq <= 32); }

// The shape whose rounds of tiles over the card cost least.
int shape_of(int64_t np, int64_t nq) {
  int best = FLAT;
  double least = -1;
  for (int shape : {BIG, MID, FLAT, THIN}) {
    if (!fits(shape, nq)) continue;
    const double cost = stage_us(shape, std::max<int64_t>(tiles_of(shape, np, nq), 1));
    if (least < 0 || cost < least) {
      least = cost;
      best = shape;
    }
  }
  return best;
}

struct Layout {
  int64_t bytes = 0;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
};

// One product's slices over k: enough workgroups, at least 4 stages a slice.
struct Slices {
  int shape, n;
  int stages;  // a slice
};
Slices slices_of(int64_t np, int64_t nq, int64_t k, int segments) {
  const int64_t stages = div_up(k, STAGE / 2) * segments;
  Slices best = {FLAT, 1, (int)stages};
  double least = -1;
  for (int shape : {BIG, MID, FLAT, THIN}) {
    if (!fits(shape, nq)) continue;
    const int64_t tiles = std::max<int64_t>(tiles_of(shape, np, nq), 1), slots = 256 * PER_CU[shape];
    int64_t n = std::min<int64_t>(std::max<int64_t>(std::min(slots / tiles, stages / 4), 1), 64);
    const int64_t each = std::max<int64_t>(div_up(stages, n), 1);
    n = std::max<int64_t>(div_up(stages, each), 1);
    // a tile's stages, and its outputs, which take about as long as 2 1/2 of them
    const double cost = ((double)each + 2.5) * stage_us(shape, tiles * n);
    if (least < 0 || cost < least) {
      least = cost;
      best = {shape, (int)n, (int)each};
    }
  }
  return best;
}

// The splits of the stream rows of a narrow kernel: r workgroups a compute unit for the r that costs least. A stage takes
// `us` of a compute unit when its workgroups hide each other's waits (three of them; two 1.15 times as long, one 1.8), a
// workgroup starts in about one stage, and a split's partial sums are written and read at 4 TB/s.
struct Splits {
  int own_tiles, n;
  int64_t range;
};
Splits splits_of(int64_t own, int64_t stream, int trip, double us, double part_bytes) {
  Splits best = {(int)div_up(own, 128), 1, 0};
  const int64_t tiles = std::max(best.own_tiles, 1), stages = std::max<int64_t>(div_up(stream, 64), 1);
  double least = -1;
  for (int r = 1; r <= 12; ++r) {
    const int64_t want = std::max<int64_t>(std::min(256 * r / tiles, stages), 1);
    const int64_t per = up(div_up(stages, want), trip), n = div_up(stages, per), each = div_up(tiles * n, 256);
    const double cost = (double)each * (double)(per + 1) * us * (each >= 3 ? 1.0 : each == 2 ? 1.15 : 1.8) +
                        (n > 1 ? (double)n * part_bytes * 2 / 4e6 : 0.0);
    if (least < 0 || cost < least) {
      least = cost;
      best.n = (int)n;
      best.range = per * 64;
    }
  }
  return best;
}

struct Plan {
  int type, es;         // the type that the factors are multiplied as, and the size of the one they are stored as
  int planes, kp;       // the engine's: planes of halves, kp of them a row
  int ds_planes;
  int64_t m, n;
  int k;
  bool grads, pack_w, pack_x;
  bool narrow;          // k_narrow
  int ks;
  Splits nl, nx, nw;
  int fwd;              // else k_product
  int64_t fwd_tiles, fwd_rows;
  int64_t piece, pieces;
  Slices sx, sw;
  int64_t o_x, o_w, o_part, o_hit, o_top, o_rows, o_ds, o_px, o_pw, bytes;
  int64_t x_plane() const { return m * kp * 2; }
  int64_t w_plane() const { return n * kp * 2; }
  int64_t ds_plane() const { return m * piece * 2; }
};
constexpr int KE = STAGE / 2;  // halves of k a stage

bool aligned(const void* p, int64_t ld_bytes, int64_t row_bytes) {
  return (((uintptr_t)p | (uintptr_t)ld_bytes | (uintptr_t)row_bytes) & 15) == 0;
}

// `pack_x`, `pack_w`: whether the rows have to be packed (they are not whole aligned granules)
Plan plan_of(int type, int es, int64_t m, int64_t n, int k, bool forward, bool grads, bool pack_x, bool pack_w) {
  Plan p;
  p.type = type;
  p.es = es;
  p.planes = planes_of(type);
  p.ds_planes = ds_planes_of(type);
  p.kp = (int)up(k, 8);
  p.m = m;
  p.n = n;
  p.k = k;
  p.grads = grads;
  p.pack_w = pack_w || type == F32;
  p.pack_x = grads || pack_x || type == F32;
  Layout l;
  p.o_x = l.take(p.pack_x ? p.planes * p.x_plane() : 0);
  p.o_w = l.take(p.pack_w ? p.planes * p.w_plane() : 0);
  p.narrow = p.kp <= (type == F32 ? 64 : 128);
  if (p.narrow) {
    p.ks = (p.kp + 31) / 32;
    const int trip = type == F32 ? 2 : 3;  // stages of a trip of k_narrow's loop
    // measured: halves 0.3 and 0.75 us a stage at k = 64, floats 0.8 and 2 at k = 50
    const double lse_us = type == F32 ? 0.4 * p.ks : 0.22 + 0.05 * p.ks, grad_us = type == F32 ? 1.0 * p.ks : 0.41 + 0.17 * p.ks;
    p.nl = splits_of(m, n, trip, lse_us, 8.0 * m);
    p.nx = splits_of(m, n, trip, grad_us, 4.0 * m * up(k, 4));
    p.nw = splits_of(n, m, trip, grad_us, 4.0 * n * up(k, 4));
    p.o_part = l.take(forward ? p.nl.n * m * 8 : 0);
    p.fwd_rows = m;
    p.o_hit = l.take(forward ? m * 4 : 0);
    p.o_top = l.take(16);
    p.o_rows = l.take(grads ? div_up(m, 64) * 1024 : 0);
    p.o_px = l.take(grads && p.nx.n > 1 ? p.nx.n * m * up(k, 4) * 4 : 0);
    p.o_pw = l.take(grads && p.nw.n > 1 ? p.nw.n * n * up(k, 4) * 4 : 0);
    p.bytes = std::max<int64_t>(l.bytes, 256);
    return p;
  }
  p.fwd = shape_of(n, m);
  p.fwd_tiles = div_up(n, BP_OF[p.fwd]) * WP_OF[p.fwd];
  // whole tiles of rows; at least 512, so that short lists are joined, and their total taken, in one launch
  p.fwd_rows = std::min(m, std::max<int64_t>(PAIR_BYTES / (p.fwd_tiles * 8) / 256 * 256, 512));
  p.o_part = l.take(forward ? p.fwd_tiles * p.fwd_rows * 8 : 0);
  p.o_hit = l.take(forward ? p.fwd_rows * 4 : 0);
  p.o_top = l.take(16);
  if (grads) {
    // whole tiles of columns within the budget, the pieces as equal as that allows
    const int64_t most = std::max<int64_t>(PIECE_BYTES / (std::max<int64_t>(m, 1) * 2 * p.ds_planes) / 256 * 256, 256);
    p.pieces = div_up(n, most);
    p.piece = std::min(up(div_up(n, p.pieces), 256), up(n, 64));
    p.pieces = div_up(n, p.piece);
    p.o_ds = l.take(p.ds_planes * p.ds_plane());
    p.sx = slices_of(k, m, std::min(p.piece, n), segments_of(type, COL));
    p.sw = slices_of(k, p.piece, m, segments_of(type, COL));
    p.o_px = l.take(p.sx.n > 1 || p.pieces > 1 ? (int64_t)p.sx.n * m * up(k, 4) * 4 : 0);
    p.o_pw = l.take(p.sw.n > 1 ? (int64_t)p.sw.n * p.piece * up(k, 4) * 4 : 0);
  }
  p.bytes = std::max<int64_t>(l.bytes, 256);
  return p;
}

template <int T, int LP, int LQ, class S, class Epi>
void launch(const Problem& a, dim3 grid, const Epi& epi, hipStream_t st) {
  k_product<mma_type(T), LP, LQ, segments_of(T, LP), S, Epi><<<grid, S::THREADS, 0, st>>>(a, epi);
}

// `stages`: of a slice (0: all)
template <int T, int LP, int LQ, class Epi>
int product(int shape, Problem a, int slices, int stages, Epi epi, hipStream_t st) {
  const int64_t tp = div_up(a.p.rows, BP_OF[shape]), tq = div_up(a.q.rows, BQ_OF[shape]);
  a.tiles_p = (int)tp;
  a.tiles_q = (int)tq;
  a.slice = stages ? stages : (int)div_up(a.k, KE) * segments_of(T, LP);
  // as many workgroups as fit the card, which take tile after tile
  const dim3 grid((unsigned)std::min<int64_t>(tp * tq, 256 * PER_CU[shape]), (unsigned)slices);
  if (shape == BIG)
    launch<T, LP, LQ, Big>(a, grid, epi, st);
  else if (shape == MID)
    launch<T, LP, LQ, Mid>(a, grid, epi, st);
  else if (shape == FLAT)
    launch<T, LP, LQ, Flat>(a, grid, epi, st);
  else
    launch<T, LP, LQ, Thin>(a, grid, epi, st);
  BLP_HIP(hipGetLastError());
  return 0;
}

// The sums of one or two sets of partial results (nq = 0: none).
template <int T>
int sum_parts(SumArgs a, SumArgs b, int64_t np, RowGrad g, float scale, hipStream_t st) {
  const FastDiv per((uint32_t)(up(np, 4) / 4));
  const int64_t na = a.nq * per.d, nb = b.nq * per.d;
  if (na + nb == 0) return 0;
  const bool many = std::max(na ? a.slices : 0, nb ? b.slices : 0) >= 16 && na + nb < 256 * 1024;
  const int64_t each = many ? 16 : 256;
  a.blocks = (unsigned)std::min<int64_t>(div_up(na, each), 8192);
  b.blocks = (unsigned)std::min<int64_t>(div_up(nb, each), 8192);
  if (many)
    k_sum_parts<T, 16><<<a.blocks + b.blocks, 256, 0, st>>>(a, b, np, per, g, scale);
  else
    k_sum_parts<T, 1><<<a.blocks + b.blocks, 256, 0, st>>>(a, b, np, per, g, scale);
  BLP_HIP(hipGetLastError());
  return 0;
}

struct Call {
  Plan p;
  hipStream_t st;
  Operand x, w;  // as the engine takes them
  Targets targets;
  float scale;
  char* ws;
};

template <int T, int ST>
int bind(Call& c, const void* x, int64_t ldx, const void* w, int64_t ldw, uint32_t* flag) {
  const Plan& p = c.p;
  c.x = {(const char*)x, ldx * p.es, p.m};
  c.w = {(const char*)w, ldw * p.es, p.n};
  const int64_t per = p.kp / 8;
  auto blocks = [&](int64_t rows) { return (unsigned)std::min<int64_t>(div_up(rows * per, 256), 4096); };
  PackArgs ax = {}, aw = {};
  if (p.pack_x) {
    ax = {c.x.base, c.x.ld, p.m, c.targets, c.ws + p.o_x, p.x_plane(), blocks(p.m)};
    if (!p.grads) ax.targets.at = nullptr;
    c.x = {ax.dst, (int64_t)p.kp * 2, p.m};
  }
  if (p.pack_w) {
    aw = {c.w.base, c.w.ld, p.n, Targets{nullptr, 0, 0}, c.ws + p.o_w, p.w_plane(), blocks(p.n)};
    c.w = {aw.dst, (int64_t)p.kp * 2, p.n};
  }
  if (ax.blocks + aw.blocks == 0) return 0;
  k_pack<T, ST><<<ax.blocks + aw.blocks, 256, 0, c.st>>>(ax, aw, p.k, FastDiv((uint32_t)per), flag);
  BLP_HIP(hipGetLastError());
  return 0;
}

template <int T, class F>
void with_steps(int ks, F f) {
  if (ks == 1) {
    f(std::integral_constant<int, 1>{});
  } else if (ks == 2) {
    f(std::integral_constant<int, 2>{});
  } else if constexpr (T != F32) {
    if (ks == 3)
      f(std::integral_constant<int, 3>{});
    else
      f(std::integral_constant<int, 4>{});
  }
}

template <int T>
int narrow_lse(const Call& c, float2* part, float* hit) {
  const Plan& p = c.p;
  const NarrowArgs a = {c.x, c.w, p.x_plane(), p.w_plane(), p.kp, p.nl.range, p.nl.own_tiles, p.nl.n, c.scale, 1.f, c.targets,
                        part, hit, Rows{nullptr}};
  const int64_t blocks = (int64_t)p.nl.own_tiles * p.nl.n;
  with_steps<T>(p.ks, [&](auto ks) { k_narrow_lse<T, decltype(ks)::value><<<(unsigned)blocks, 256, 0, c.st>>>(a); });
  BLP_HIP(hipGetLastError());
  return 0;
}

template <int T, int ST>
int narrow_grads(const Call& c, RowGrad g, void* dx, int64_t lddx, void* dw, int64_t lddw) {
  const Plan& p = c.p;
  const int64_t ldp = up(p.k, 4);
  float *px = (float*)(c.ws + p.o_px), *pw = (float*)(c.ws + p.o_pw);
  const Rows rows = {(float*)(c.ws + p.o_rows)};
  const NarrowArgs x = {c.x, c.w, p.x_plane(), p.w_plane(), p.kp, p.nx.range, dx ? p.nx.own_tiles : 0, p.nx.n, c.scale, g.extra,
                        c.targets, nullptr, nullptr, rows};
  const NarrowArgs w = {c.w, c.x, p.w_plane(), p.x_plane(), p.kp, p.nw.range, dw ? p.nw.own_tiles : 0, p.nw.n, c.scale, g.extra,
                        c.targets, nullptr, nullptr, rows};
  const EpiGradient<ST> ex = {p.nx.n > 1, {px, ldp, p.k, p.m, 0}, {(char*)dx, lddx * p.es, p.k, p.m, g, c.scale}};
  const EpiGradient<ST> ew = {p.nw.n > 1, {pw, ldp, p.k, p.n, 0}, {(char*)dw, lddw * p.es, p.k, p.n, g, c.scale}};
  const int64_t bw = up((int64_t)w.own_tiles * w.splits, 8), bx = (int64_t)x.own_tiles * x.splits;  // eights: x keeps its dies
  const bool per_row = g.g && g.stride;
  auto launch = [&](int64_t bw, int64_t bx) -> int {
    if (bw + bx == 0) return 0;
    with_steps<T>(p.ks, [&](auto ks) {
      constexpr int KS = decltype(ks)::value;
      if constexpr (T != F16) {  // row gradients of float16 are taken as floats
        if (per_row) k_narrow_grads<T, ST, KS, true><<<(unsigned)(bw + bx), 256, 0, c.st>>>(w, ew, (int)bw, x, ex);
      }
      if constexpr (T == ST) {
        if (!per_row) k_narrow_grads<T, ST, KS, false><<<(unsigned)(bw + bx), 256, 0, c.st>>>(w, ew, (int)bw, x, ex);
      }
    });
    BLP_HIP(hipGetLastError());
    return 0;
  };
  // a launch takes less than 2^32 threads: each gradient's workgroups do (a 128th of up to 2^31 - 2^16 rows), both's may not
  int rc = 0;
  if (bw + bx < 1 << 24) {
    rc = launch(bw, bx);
  } else {
    rc = launch(bw, 0);
    if (!rc) rc = launch(0, bx);
  }
  if (rc) return rc;
  const SumArgs sx = {px, p.nx.n, dx && p.nx.n > 1 ? p.m : 0, (char*)dx, lddx * p.es, 0};
  const SumArgs sw = {pw, p.nw.n, dw && p.nw.n > 1 ? p.n : 0, (char*)dw, lddw * p.es, 0};
  return sum_parts<ST>(sx, sw, p.k, g, c.scale, c.st);
}

template <int T>
int forward(const Call& c, float* loss, float* lse, Total total, uint32_t* done) {
  const Plan& p = c.p;
  if (p.m > 0) {
    float2* part = (float2*)(c.ws + p.o_part);
    float* hit = (float*)(c.ws + p.o_hit);
    // as many rows at a time as the pairs have room for (narrow factors: all)
    for (int64_t r0 = 0; r0 < p.m; r0 += p.fwd_rows) {
      const int64_t m = std::min(p.fwd_rows, p.m - r0);
      const Targets targets = {c.targets.from(r0), c.targets.wide, c.targets.rows};
      int rc;
      if (p.narrow) {
        rc = narrow_lse<T>(c, part, hit);
      } else {
        const Problem a = {c.w, {c.x.base + r0 * c.x.ld, c.x.ld, m}, p.kp, 0, 0, 0, p.w_plane(), p.x_plane()};
        rc = product<T, ROW, ROW>(p.fwd, a, 1, 0, EpiLse<T>{part, hit, targets, p.n, m, c.scale}, c.st);
      }
      if (rc) return rc;
      const int64_t pairs = p.narrow ? p.nl.n : p.fwd_tiles;
      const Rows rows = {p.narrow && p.grads ? (float*)(c.ws + p.o_rows) : nullptr};
      const int64_t all = rows.at ? up(m, 64) : m;
      for (int64_t j0 = 0; j0 < all; j0 += JOINED) {
        const int64_t n = std::min(JOINED, all - j0);
        if (m >= 4096)
          k_join<32><<<(unsigned)div_up(n, 32), 256, 0, c.st>>>(part, pairs, m, j0, hit, targets, loss + r0, lse + r0, rows,
                                                                extra_of(T), total, done);
        else
          k_join<4><<<(unsigned)div_up(n, 4), 256, 0, c.st>>>(part, pairs, m, j0, hit, targets, loss + r0, lse + r0, rows,
                                                              extra_of(T), total, done);
        BLP_HIP(hipGetLastError());
      }
    }
  }
  if (total.at && !(done && p.m > 0)) {
    k_total<<<1, 1024, 0, c.st>>>(loss, c.targets, p.m, total);
    BLP_HIP(hipGetLastError());
  }
  return 0;
}

template <int T, int ST>
int backward(const Call& c, bool fwd, const float* lse, RowGrad g, void* dx, int64_t lddx, void* dw, int64_t lddw) {
  const Plan& p = c.p;
  if (p.m == 0) {  // no rows: the catalogue's gradient is zero
    if (dw) {
      return sum_parts<ST>(SumArgs{nullptr, 0, p.n, (char*)dw, lddw * p.es, 0}, SumArgs{}, p.k, RowGrad{nullptr, 0, nullptr, nullptr, 1.f},
                          1.f, c.st);
    }
    return 0;
  }
  g.extra = extra_of(T);
  if (g.g && g.stride) {
    float* top = (float*)(c.ws + p.o_top);
    k_top_grad<<<1, 1024, 0, c.st>>>(g.g, c.targets, p.m, top);
    BLP_HIP(hipGetLastError());
    g.top = top;
  }
  if (p.narrow) {
    if (!fwd) {  // the forward pass's last step leaves them otherwise
      k_rows<<<(unsigned)div_up(p.m, 64), 64, 0, c.st>>>(lse, g, c.targets, p.m, Rows{(float*)(c.ws + p.o_rows)});
      BLP_HIP(hipGetLastError());
    }
    return narrow_grads<T, ST>(c, g, dx, lddx, dw, lddw);
  }
  char* ds = c.ws + p.o_ds;
  float *px = (float*)(c.ws + p.o_px), *pw = (float*)(c.ws + p.o_pw);
  const int64_t ldp = up(p.k, 4);
  const bool parts_x = p.sx.n > 1 || p.pieces > 1;
  int rc = 0;
  for (int64_t j0 = 0; j0 < p.n && !rc; j0 += p.piece) {
    const int64_t nj = std::min(p.piece, p.n - j0);
    const Operand wj = {c.w.base + j0 * c.w.ld, c.w.ld, nj};
    // the scores of the piece again, as dS. Its width is written up to the end of the last tile: zeros past the catalogue's
    const Problem as = {wj, c.x, p.kp, 0, 0, 0, p.w_plane(), p.x_plane()};
    const EpiGrad<T> eg = {ds, p.piece, p.ds_plane(), lse, g, c.targets, j0, nj, p.m, c.scale};
    rc = product<T, ROW, ROW>(shape_of(nj, p.m), as, 1, 0, eg, c.st);
    if (rc) break;
    const Operand dsr = {ds, p.piece * 2, p.m};
    if (dx) {
      const Problem ax = {{wj.base, wj.ld, p.k}, dsr, nj, 0, 0, 0, p.w_plane(), p.ds_plane()};
      // the last piece is narrower: its slices are those that have stages (the first piece, which is whole, has set them all)
      const int slices = (int)std::min<int64_t>(p.sx.n, div_up(div_up(nj, KE) * segments_of(T, COL), p.sx.stages));
      if (parts_x)
        rc = product<T, COL, ROW>(p.sx.shape, ax, slices, p.sx.stages, EpiPart{px, ldp, p.k, p.m, j0 > 0}, c.st);
      else
        rc = product<T, COL, ROW>(p.sx.shape, ax, 1, 0, EpiOut<ST>{(char*)dx, lddx * p.es, p.k, p.m, g, c.scale}, c.st);
      if (rc) break;
    }
    if (dw) {
      const Problem aw = {{c.x.base, c.x.ld, p.k}, {ds, p.piece * 2, nj}, p.m, 0, 0, 0, p.x_plane(), p.ds_plane()};
      char* out = (char*)dw + j0 * lddw * p.es;
      if (p.sw.n > 1) {
        rc = product<T, COL, COL>(p.sw.shape, aw, p.sw.n, p.sw.stages, EpiPart{pw, ldp, p.k, nj, 0}, c.st);
        if (rc) break;
        rc = sum_parts<ST>(SumArgs{pw, p.sw.n, nj, out, lddw * p.es, 0}, SumArgs{}, p.k, g, c.scale, c.st);
      } else {
        rc = product<T, COL, COL>(p.sw.shape, aw, 1, 0, EpiOut<ST>{out, lddw * p.es, p.k, nj, g, c.scale}, c.st);
      }
    }
  }
  if (rc) return rc;
  if (dx && parts_x) rc = sum_parts<ST>(SumArgs{px, p.sx.n, p.m, (char*)dx, lddx * p.es, 0}, SumArgs{}, p.k, g, c.scale, c.st);
  return rc;
}

constexpr int64_t MOST_ROWS = (1ll << 31) - (1 << 16);  // the row numbers of stages past the end fit 31 bits

int check_args(int type, int64_t rows, int64_t cols, int k) {
  BLP_CHECK(type >= 0 && type <= 2, BLP_E_ARG, "softmax loss: type must be BLP_F32, BLP_BF16 or BLP_F16");
  BLP_CHECK(rows >= 0 && rows <= MOST_ROWS, BLP_E_ARG, "softmax loss: rows must be in [0, 2^31 - 2^16]");
  BLP_CHECK(cols >= 1 && cols <= MOST_ROWS, BLP_E_ARG, "softmax loss: the catalogue must have 1 to 2^31 - 2^16 rows");
  BLP_CHECK(k >= 1 && k <= (1 << 20), BLP_E_ARG, "softmax loss: k must be in [1, 2^20]");
  // the gradients' tiles, 64 x 32 or larger, are counted in 31 bits; the scores' are fewer (pieces and pairs bound them)
  BLP_CHECK(std::max(rows, cols) <= (1ll << 41) / k, BLP_E_ARG, "softmax loss: rows x k and columns x k must be at most 2^41");
  return 0;
}

template <int T, int ST>
int run(Call& c, const void* x, int64_t ldx, const void* w, int64_t ldw, float* loss, float* lse, float* total, int mean,
        bool fwd, RowGrad g, void* dx, int64_t lddx, void* dw, int64_t lddw) {
  // With gradients the packing comes first and clears the mark by which the last block to end takes the total. Every
  // block's fence writes its die's cache back, so that pays for few of them (106 x 7,073 x 31 floats:
  // 31.4 -> 28.2 us a step; 1,590 x 7,073 x 31: 50 -> 75).
  uint32_t* done = fwd && total && c.p.grads && c.p.m > 0 && c.p.m <= 512 ? (uint32_t*)(c.ws + c.p.o_top) + 1 : nullptr;
  int rc = bind<T, ST>(c, x, ldx, w, ldw, done);
  if constexpr (T == ST) {
    if (!rc && fwd) rc = forward<T>(c, loss, lse, Total{total, mean}, done);
  }
  if (!rc && c.p.grads) rc = backward<T, ST>(c, fwd, lse, g, dx, lddx, dw, lddw);
  return rc;
}

int dispatch(int device, void* stream, int type, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* target,
             int target64, int64_t m, int64_t n, int k, float scale, float* loss, float* lse, float* total, int mean, bool fwd,
             RowGrad g, bool grads, void* dx, int64_t lddx, void* dw, int64_t lddw, void* ws, int64_t ws_bytes) {
  int rc = check_args(type, m, n, k);
  if (rc) return rc;
  const int es = size_of(type);
  BLP_CHECK(w && (m == 0 || (x && target && loss && lse)) && ws, BLP_E_ARG, "softmax loss: null pointer");
  BLP_CHECK(fabsf(scale) <= 3.4028235e38f, BLP_E_ARG, "softmax loss: scale must be finite");
  BLP_CHECK(fabsf(scale) <= 0x1p127f, BLP_E_ARG, "softmax loss: scale must be at most 2^127 (times log2 e it has to be a float)");
  BLP_CHECK(ldx >= k && ldw >= k && (!dx || lddx >= k) && (!dw || lddw >= k), BLP_E_ARG,
            "softmax loss: a row stride is smaller than k");
  BLP_CHECK(std::max(ldx, ldw) <= (1 << 20), BLP_E_ARG, "softmax loss: row strides must be at most 2^20 elements");
  Call c;
  const bool as_floats = type == F16 && g.g && g.stride;
  c.p = plan_of(as_floats ? F32 : type, es, m, n, k, fwd, grads, !aligned(x, ldx * es, (int64_t)k * es), !aligned(w, ldw * es, (int64_t)k * es));
  BLP_CHECK(ws_bytes >= c.p.bytes, BLP_E_ARG, "softmax loss: the workspace is too small (blp_softmax_loss_workspace)");
  BLP_CHECK(((uintptr_t)ws & 255) == 0, BLP_E_ARG, "softmax loss: the workspace must be 256-byte aligned");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  c.st = (hipStream_t)stream;
  c.targets = {target, target64, n};
  c.scale = scale;
  c.ws = (char*)ws;
  if (as_floats) return run<F32, F16>(c, x, ldx, w, ldw, loss, lse, total, mean, fwd, g, dx, lddx, dw, lddw);
  if (type == F32) return run<F32, F32>(c, x, ldx, w, ldw, loss, lse, total, mean, fwd, g, dx, lddx, dw, lddw);
  if (type == BF16) return run<BF16, BF16>(c, x, ldx, w, ldw, loss, lse, total, mean, fwd, g, dx, lddx, dw, lddw);
  return run<F16, F16>(c, x, ldx, w, ldw, loss, lse, total, mean, fwd, g, dx, lddx, dw, lddw);
}

}  // namespace

extern "C" int blp_softmax_loss_workspace(int type, const void* x, int64_t ldx, const void* table, int64_t ldt, int64_t rows,
                                          int64_t cols, int k, int forward, int grads, int64_t* bytes) {
  int rc = check_args(type, rows, cols, k);
  if (rc) return rc;
  BLP_CHECK(bytes, BLP_E_ARG, "softmax loss: null pointer");
  const int es = size_of(type);
  auto need = [&](int as) {
    return plan_of(as, es, rows, cols, k, forward != 0, grads != 0, !aligned(x, ldx * es, (int64_t)k * es),
                   !aligned(table, ldt * es, (int64_t)k * es))
        .bytes;
  };
  *bytes = need(type);
  if (type == F16 && !forward && grads) *bytes = std::max(*bytes, need(F32));  // row gradients, if it gets them
  return 0;
}

extern "C" int blp_softmax_loss(int device, void* stream, int type, const void* x, int64_t ldx, const void* table, int64_t ldt,
                                const void* target, int target64, int64_t rows, int64_t cols, int k, float scale, float* loss,
                                float* lse, float* total, int mean, int grads, void* dx, int64_t lddx, void* dtable,
                                int64_t lddt, void* ws, int64_t ws_bytes) {
  const RowGrad g = {nullptr, 0, total && mean ? total + 1 : nullptr, nullptr, 1.f};
  return dispatch(device, stream, type, x, ldx, table, ldt, target, target64, rows, cols, k, scale, loss, lse, total, mean, true,
                  g, grads != 0, dx, lddx, dtable, lddt, ws, ws_bytes);
}

extern "C" int blp_softmax_loss_backward(int device, void* stream, int type, const void* x, int64_t ldx, const void* table,
                                         int64_t ldt, const void* target, int target64, int64_t rows, int64_t cols, int k,
                                         float scale, const float* lse, const float* grad, int grad_stride, const float* count,
                                         void* dx, int64_t lddx, void* dtable, int64_t lddt, void* ws, int64_t ws_bytes) {
  BLP_CHECK(grad_stride == 0 || grad_stride == 1, BLP_E_ARG, "softmax loss: grad_stride must be 0 or 1");
  const RowGrad g = {grad, grad_stride, count, nullptr, 1.f};
  float* l = const_cast<float*>(lse);
  return dispatch(device, stream, type, x, ldx, table, ldt, target, target64, rows, cols, k, scale, l, l, nullptr, 0, false, g,
                  true, dx, lddx, dtable, lddt, ws, ws_bytes);
}
