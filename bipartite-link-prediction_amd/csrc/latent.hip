// The softmax loss of latent factors over the whole catalogue, with its gradients (blp_softmax_loss*).
//
//   z_ij = scale x_i . w_j        lse_i = log sum_j exp z_ij        loss_i = lse_i - z_{i, t_i}
//   dS_ij = g_i (exp(z_ij - lse_i) - [j = t_i])       dX = scale dS W       dW = scale dS^T X
//
// x_i are the rows scored (users), w_j every row of the catalogue, t_i the row's target. The scores are
// never kept: the forward pass reduces each tile of them to a (max, sum) pair a row, and the backward pass
// recomputes them piece by piece of the catalogue into a workspace of dS, from which the two products of
// the gradient are taken. Four products of 2 M N k operations in all; the workspace is bounded.
//
// A row whose target lies outside [0, n_cols) is ignored: loss 0, gradient 0, and its x is never multiplied
// (it may hold anything, NaN too).
#include <algorithm>

#include "blp_internal.h"
#include "latent.h"

namespace {

using namespace blp::tile;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;

using blp::DeviceGuard;
using Targets = blp::Ids;  // the target of row i, or -1 (ignored)

// ---------------------------------------------------------------- packing
// Rows as the tile engine takes them: `kp` elements a row (whole granules, zeros past k), 16-byte aligned;
// with targets, the ignored rows as zeros. One 16-byte granule a thread; bound by the copy.
template <int ES>
__global__ __launch_bounds__(256) void k_pack(const char* __restrict__ src, int64_t ld, int64_t rows, int k, int kp,
                                              Targets targets, char* __restrict__ dst) {
  constexpr int GE = 16 / ES;
  const int per = kp / GE;
  const bool aligned = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)ld) & 15) == 0;
  const int64_t n = rows * per, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t r = i / per;
    const int e0 = (int)(i - r * per) * GE;
    i32x4 v = {0, 0, 0, 0};
    if (!targets.at || targets(r) >= 0) {
      const char* s = src + r * ld + (int64_t)e0 * ES;
      if (aligned && e0 + GE <= k) {
        v = *reinterpret_cast<const i32x4*>(s);
      } else if constexpr (ES == 4) {
        for (int j = 0; j < GE; ++j)
          if (e0 + j < k) v[j] = reinterpret_cast<const int32_t*>(s)[j];
      } else {
        for (int j = 0; j < GE; ++j)
          if (e0 + j < k) v[j >> 1] |= (int)((uint32_t)reinterpret_cast<const uint16_t*>(s)[j] << (16 * (j & 1)));
      }
    }
    reinterpret_cast<i32x4*>(dst)[i] = v;
  }
}

// ---------------------------------------------------------------- forward
// One (max, sum of exp2) pair a row and wave tile, in base 2: part[tile * rows + row].
template <int T>
struct EpiLse {
  float2* part;
  float* hit;  // z of the target
  Targets targets;
  int64_t n, m;
  float scale;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int tile) const {
    const int lane = threadIdx.x & 63, h = lane >> 4;
    const float c = scale * LOG2E;
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) {
      const int64_t row = q0 + j * 16 + (lane & 15);
      const int64_t t = row < m ? targets(row) : -1;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < S::FP; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t p = p0 + i * 16 + h * 4 + e;
          if (p == t) hit[row] = acc[i][j][e] * scale;
          const float z = p < n ? acc[i][j][e] * c : -INFINITY;
          acc[i][j][e] = z;
          top = fmaxf(top, z);
        }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < S::FP; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(acc[i][j][e] - base);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (h == 0 && row < m) part[(int64_t)tile * m + row] = make_float2(top, sum);
    }
  }
};

// fmaxf drops a NaN, the sum keeps it (exp2(NaN - base)); an infinite max gives inf - inf = NaN.
__device__ inline void merge(float& top, float& sum, float t2, float s2) {
  const float t = fmaxf(top, t2);
  const float base = t == -INFINITY ? 0.f : t;
  sum = sum * __builtin_amdgcn_exp2f(top - base) + s2 * __builtin_amdgcn_exp2f(t2 - base);
  top = t;
}

// 32 rows a block, 8 threads a row over the tiles' pairs.
__global__ __launch_bounds__(256) void k_join(const float2* __restrict__ part, int64_t tiles, int64_t m,
                                              const float* __restrict__ hit, Targets targets, float* __restrict__ loss,
                                              float* __restrict__ lse) {
  __shared__ float2 s_part[8][32];
  const int r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t row = blockIdx.x * 32ll + r;
  float top = -INFINITY, sum = 0.f;
  if (row < m)
    for (int64_t t = g; t < tiles; t += 8) {
      const float2 v = part[t * m + row];
      merge(top, sum, v.x, v.y);
    }
  s_part[g][r] = make_float2(top, sum);
  __syncthreads();
  if (g == 0 && row < m) {
    for (int i = 1; i < 8; ++i) merge(top, sum, s_part[i][r].x, s_part[i][r].y);
    const float l = (top + __builtin_amdgcn_logf(sum)) * LN2;  // logf: base 2
    lse[row] = l;
    loss[row] = targets(row) >= 0 ? l - hit[row] : 0.f;
  }
}

// total[0] = the sum of the losses, or their mean over the rows not ignored; total[1] = their number.
// One block, fixed order, in 64 bits: the same result every time.
__global__ __launch_bounds__(1024) void k_total(const float* __restrict__ loss, Targets targets, int64_t m, int mean,
                                                float* __restrict__ total) {
  __shared__ double s_sum[16];
  __shared__ int64_t s_n[16];
  double sum = 0.0;
  int64_t n = 0;
  for (int64_t i = threadIdx.x; i < m; i += 1024)
    if (targets(i) >= 0) {
      sum += loss[i];
      ++n;
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
    for (int i = 1; i < 16; ++i) {
      sum += s_sum[i];
      n += s_n[i];
    }
    total[0] = (float)(mean ? sum / (double)max(n, (int64_t)1) : sum);
    total[1] = (float)max(n, (int64_t)1);
  }
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
    const float t = *top;
    return t > 0.f ? g[i] / t * extra : t != t ? t : 0.f;
  }
  __device__ float all() const {
    const float f = (g ? (stride ? *top : *g) : 1.f) / extra;
    return count ? f / *count : f;
  }
};

__global__ __launch_bounds__(1024) void k_top_grad(const float* __restrict__ g, Targets targets, int64_t m,
                                                   float* __restrict__ top) {
  __shared__ float s_top[16];
  float t = 0.f;
  bool nan = false;
  for (int64_t i = threadIdx.x; i < m; i += 1024)
    if (targets(i) >= 0) {
      const float v = fabsf(g[i]);
      nan |= !(v <= 3.0e38f);
      t = fmaxf(t, v);
    }
  if (nan) t = INFINITY;
  for (int o = 32; o; o >>= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
  if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) t = fmaxf(t, s_top[i]);
    *top = t <= 3.0e38f ? t : NAN;  // an infinite or NaN gradient: everything it reaches is NaN
  }
}

// dS of one piece: ds[row * ld + p - 0], zeros past the catalogue's end.
template <int T>
struct EpiGrad {
  char* ds;
  int64_t ld;  // elements
  const float* lse;
  RowGrad g;
  Targets targets;
  int64_t j0;  // the piece's first column
  int64_t n, m;
  float scale;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int) const {
    const int lane = threadIdx.x & 63, h = lane >> 4;
    const float c = scale * LOG2E;
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) {
      const int64_t row = q0 + j * 16 + (lane & 15);
      if (row >= m) continue;
      const int64_t t = targets(row) - j0;  // negative: not here or ignored
      const bool valid = targets(row) >= 0;
      const float gr = valid ? g.row(row) : 0.f, l2 = lse[row] * LOG2E;
      char* at = ds + row * ld * size_of(T);
#pragma unroll
      for (int i = 0; i < S::FP; ++i) {
        const int64_t p = p0 + i * 16 + h * 4;
        if (p >= ld) continue;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, -l2)) - (p + e == t ? 1.f : 0.f);
          v[e] = valid && p + e < n ? d * gr : 0.f;
        }
        store4<T>(at + p * size_of(T), v);
      }
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
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int) const {
    const int lane = threadIdx.x & 63, h = lane >> 4;
    const float alpha = scale * g.all();
    const bool whole = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)ld) & (4 * size_of(T) - 1)) == 0;
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) {
      const int64_t q = q0 + j * 16 + (lane & 15);
      if (q >= nq) continue;
#pragma unroll
      for (int i = 0; i < S::FP; ++i) {
        const int64_t p = p0 + i * 16 + h * 4;
        char* at = out + q * ld + p * size_of(T);
        if (whole && p + 4 <= np) {
          store4<T>(at, acc[i][j] * alpha);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (p + e < np) store1<T>(at + e * size_of(T), acc[i][j][e] * alpha);
        }
      }
    }
  }
};

// part[slice][q][p] (+)= acc: the sums over slices of k and pieces of the catalogue, in 32 bits.
struct EpiPart {
  float* part;
  int64_t ld, np, nq;  // elements; ld a multiple of 4
  int add;
  template <class S>
  __device__ void run(f32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int) const {
    const int lane = threadIdx.x & 63, h = lane >> 4;
    float* base = part + (int64_t)blockIdx.y * nq * ld;
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

// out = alpha sum_s part[s], in the slices' order.
template <int T>
__global__ __launch_bounds__(256) void k_sum_parts(const float* __restrict__ part, int slices, int64_t ld, int64_t np,
                                                   int64_t nq, RowGrad g, float scale, char* __restrict__ out, int64_t ldo) {
  const float alpha = scale * g.all();
  const int64_t per = ld / 4, n = nq * per, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t q = i / per, p = (i - q * per) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < slices; ++s) v += *reinterpret_cast<const f32x4*>(part + (s * nq + q) * ld + p);
    for (int e = 0; e < 4; ++e)
      if (p + e < np) store1<T>(out + q * ldo + (p + e) * size_of(T), v[e] * alpha);
  }
}

// ---------------------------------------------------------------- host side
constexpr int64_t PIECE_BYTES = 512ll << 20;  // dS of one piece of the catalogue
constexpr int64_t GOAL = 512;                 // workgroups a launch should have

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t div_up(int64_t v, int64_t by) { return (v + by - 1) / by; }

enum ShapeId { BIG, MID, NARROW_P, NARROW_Q };
using Big = Shape<2, 4, 8, 4>;       // 256 x 256
using Mid = Shape<2, 2, 4, 4>;       // 128 x 128
using NarrowP = Shape<1, 4, 4, 4>;   // 64 x 256
using NarrowQ = Shape<4, 1, 4, 2>;   // 256 x 32

int bp_of(int s) { return s == BIG || s == NARROW_Q ? 256 : s == MID ? 128 : 64; }
int bq_of(int s) { return s == BIG || s == NARROW_P ? 256 : s == MID ? 128 : 32; }
int wp_of(int s) { return s == BIG || s == MID ? 2 : s == NARROW_P ? 1 : 4; }

// Few rows: 32 of them a tile. Few outputs a row: 64. Else the large tile once it fills the card.
int shape_of(int64_t np, int64_t nq) {
  if (nq <= 32) return NARROW_Q;
  if (np <= 64) return NARROW_P;
  return div_up(np, 256) * div_up(nq, 256) >= 192 ? BIG : MID;
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
  int64_t k_slice;
};
Slices slices_of(int64_t np, int64_t nq, int64_t k, int ke) {
  Slices s;
  s.shape = shape_of(np, nq);
  const int64_t tiles = std::max<int64_t>(div_up(np, bp_of(s.shape)) * div_up(nq, bq_of(s.shape)), 1);
  const int64_t stages = div_up(k, ke);
  int64_t n = tiles >= GOAL / 2 ? 1 : std::min(GOAL / tiles, std::max<int64_t>(stages / 4, 1));
  n = std::min<int64_t>(std::max<int64_t>(n, 1), 64);
  const int64_t per = std::max<int64_t>(div_up(stages, n), 1);
  s.n = (int)std::max<int64_t>(div_up(stages, per), 1);
  s.k_slice = per * ke;
  return s;
}

struct Plan {
  int type, es, ge, ke, kp;
  int64_t m, n;
  int k;
  bool grads, pack_w, pack_x;
  int fwd;
  int64_t fwd_tiles;
  int64_t piece, pieces;
  Slices sx, sw;
  int64_t o_x, o_w, o_part, o_hit, o_top, o_ds, o_px, o_pw, bytes;
};

bool aligned(const void* p, int64_t ld_bytes, int64_t row_bytes) {
  return (((uintptr_t)p | (uintptr_t)ld_bytes | (uintptr_t)row_bytes) & 15) == 0;
}

// `pack_w`: whether the catalogue has to be packed (its rows are not whole aligned granules)
Plan plan_of(int type, int64_t m, int64_t n, int k, bool forward, bool grads, bool pack_x, bool pack_w) {
  Plan p;
  p.type = type;
  p.es = size_of(type);
  p.ge = 16 / p.es;
  p.ke = STAGE / p.es;
  p.kp = (int)up(k, p.ge);
  p.m = m;
  p.n = n;
  p.k = k;
  p.grads = grads;
  p.pack_w = pack_w;
  p.pack_x = grads || pack_x;
  Layout l;
  p.o_x = l.take(p.pack_x ? m * p.kp * p.es : 0);
  p.o_w = l.take(pack_w ? n * p.kp * p.es : 0);
  p.fwd = shape_of(n, m);
  p.fwd_tiles = div_up(n, bp_of(p.fwd)) * wp_of(p.fwd);
  p.o_part = l.take(forward ? p.fwd_tiles * m * 8 : 0);
  p.o_hit = l.take(forward ? m * 4 : 0);
  p.o_top = l.take(16);
  if (grads) {
    // whole tiles of columns within the budget, the pieces as equal as that allows
    const int64_t most = std::max<int64_t>(PIECE_BYTES / (std::max<int64_t>(m, 1) * p.es) / 256 * 256, 256);
    p.pieces = div_up(n, most);
    p.piece = std::min(up(div_up(n, p.pieces), 256), up(n, 64));
    p.pieces = div_up(n, p.piece);
    p.o_ds = l.take(m * p.piece * p.es);
    p.sx = slices_of(k, m, std::min(p.piece, n), p.ke);
    p.sw = slices_of(k, p.piece, m, p.ke);
    p.o_px = l.take(p.sx.n > 1 || p.pieces > 1 ? (int64_t)p.sx.n * m * up(k, 4) * 4 : 0);
    p.o_pw = l.take(p.sw.n > 1 ? (int64_t)p.sw.n * p.piece * up(k, 4) * 4 : 0);
  }
  p.bytes = std::max<int64_t>(l.bytes, 256);
  return p;
}

template <int T, int LP, int LQ, class Epi>
int product(int shape, Problem a, int slices, Epi epi, hipStream_t st) {
  const int64_t tp = div_up(a.p.rows, bp_of(shape)), tq = div_up(a.q.rows, bq_of(shape));
  BLP_CHECK(tp * tq <= 0x7fffffff, BLP_E_ARG, "softmax loss: too many tiles for one launch");
  a.tiles_p = (int)tp;
  a.tiles_q = (int)tq;
  const dim3 grid((unsigned)(tp * tq), (unsigned)slices);
  if (shape == BIG)
    k_product<T, LP, LQ, Big, Epi><<<grid, Big::THREADS, 0, st>>>(a, epi);
  else if (shape == MID)
    k_product<T, LP, LQ, Mid, Epi><<<grid, Mid::THREADS, 0, st>>>(a, epi);
  else if (shape == NARROW_P)
    k_product<T, LP, LQ, NarrowP, Epi><<<grid, NarrowP::THREADS, 0, st>>>(a, epi);
  else
    k_product<T, LP, LQ, NarrowQ, Epi><<<grid, NarrowQ::THREADS, 0, st>>>(a, epi);
  BLP_HIP(hipGetLastError());
  return 0;
}

int64_t grid_for(int64_t n) { return std::max<int64_t>(std::min<int64_t>(div_up(n, 256), 8192), 1); }

template <int T>
int pack(const char* src, int64_t ld, int64_t rows, int k, int kp, Targets t, char* dst, hipStream_t st) {
  if (rows == 0) return 0;
  k_pack<size_of(T)><<<grid_for(rows * (kp * size_of(T) / 16)), 256, 0, st>>>(src, ld, rows, k, kp, t, dst);
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

template <int T>
int bind(Call& c, const void* x, int64_t ldx, const void* w, int64_t ldw) {
  const Plan& p = c.p;
  c.x = {(const char*)x, ldx * p.es, p.m};
  c.w = {(const char*)w, ldw * p.es, p.n};
  int rc = 0;
  if (p.pack_x) {
    Targets t = c.targets;
    if (!p.grads) t.at = nullptr;
    rc = pack<T>(c.x.base, c.x.ld, p.m, p.k, p.kp, t, c.ws + p.o_x, c.st);
    c.x = {c.ws + p.o_x, (int64_t)p.kp * p.es, p.m};
  }
  if (!rc && p.pack_w) {
    rc = pack<T>(c.w.base, c.w.ld, p.n, p.k, p.kp, Targets{nullptr, 0, 0}, c.ws + p.o_w, c.st);
    c.w = {c.ws + p.o_w, (int64_t)p.kp * p.es, p.n};
  }
  return rc;
}

template <int T>
int forward(const Call& c, float* loss, float* lse, float* total, int mean) {
  const Plan& p = c.p;
  if (p.m > 0) {
    float2* part = (float2*)(c.ws + p.o_part);
    float* hit = (float*)(c.ws + p.o_hit);
    const Problem a = {c.w, c.x, p.kp, up(p.kp, p.ke), 0, 0};
    int rc = product<T, ROW, ROW>(p.fwd, a, 1, EpiLse<T>{part, hit, c.targets, p.n, p.m, c.scale}, c.st);
    if (rc) return rc;
    k_join<<<(unsigned)div_up(p.m, 32), 256, 0, c.st>>>(part, p.fwd_tiles, p.m, hit, c.targets, loss, lse);
    BLP_HIP(hipGetLastError());
  }
  if (total) {
    k_total<<<1, 1024, 0, c.st>>>(loss, c.targets, p.m, mean, total);
    BLP_HIP(hipGetLastError());
  }
  return 0;
}

template <int T>
int backward(const Call& c, const float* lse, RowGrad g, void* dx, int64_t lddx, void* dw, int64_t lddw) {
  const Plan& p = c.p;
  if (p.m == 0) {  // no rows: the catalogue's gradient is zero
    if (dw) {
      k_sum_parts<T><<<grid_for(p.n * up(p.k, 4) / 4), 256, 0, c.st>>>(nullptr, 0, up(p.k, 4), p.k, p.n,
                                                                      RowGrad{nullptr, 0, nullptr, nullptr, 1.f}, 1.f,
                                                                      (char*)dw, lddw * p.es);
      BLP_HIP(hipGetLastError());
    }
    return 0;
  }
  g.extra = T == F16 ? 16384.f : 1.f;  // halves: a probability below 2^-24 is not lost
  if (g.g && g.stride) {
    float* top = (float*)(c.ws + p.o_top);
    k_top_grad<<<1, 1024, 0, c.st>>>(g.g, c.targets, p.m, top);
    BLP_HIP(hipGetLastError());
    g.top = top;
  }
  char* ds = c.ws + p.o_ds;
  float *px = (float*)(c.ws + p.o_px), *pw = (float*)(c.ws + p.o_pw);
  const int64_t ldp = up(p.k, 4);
  const bool parts_x = p.sx.n > 1 || p.pieces > 1;
  int rc = 0;
  for (int64_t j0 = 0; j0 < p.n && !rc; j0 += p.piece) {
    const int64_t nj = std::min(p.piece, p.n - j0);
    const Operand wj = {c.w.base + j0 * c.w.ld, c.w.ld, nj};
    // the scores of the piece again, as dS. All of its width is written: zeros past the end
    const Problem as = {{wj.base, wj.ld, nj}, c.x, p.kp, up(p.kp, p.ke), 0, 0};
    EpiGrad<T> eg = {ds, p.piece, lse, g, c.targets, j0, nj, p.m, c.scale};
    rc = product<T, ROW, ROW>(shape_of(nj, p.m), as, 1, eg, c.st);
    if (rc) break;
    const Operand dsr = {ds, p.piece * p.es, p.m};
    if (dx) {
      const Problem ax = {{wj.base, wj.ld, p.k}, dsr, nj, p.sx.k_slice, 0, 0};
      if (parts_x)
        rc = product<T, COL, ROW>(p.sx.shape, ax, p.sx.n, EpiPart{px, ldp, p.k, p.m, j0 > 0}, c.st);
      else
        rc = product<T, COL, ROW>(p.sx.shape, ax, 1, EpiOut<T>{(char*)dx, lddx * p.es, p.k, p.m, g, c.scale}, c.st);
      if (rc) break;
    }
    if (dw) {
      const Problem aw = {{c.x.base, c.x.ld, p.k}, {ds, p.piece * p.es, nj}, p.m, p.sw.k_slice, 0, 0};
      char* out = (char*)dw + j0 * lddw * p.es;
      if (p.sw.n > 1) {
        rc = product<T, COL, COL>(p.sw.shape, aw, p.sw.n, EpiPart{pw, ldp, p.k, nj, 0}, c.st);
        if (rc) break;
        k_sum_parts<T><<<grid_for(nj * (ldp / 4)), 256, 0, c.st>>>(pw, p.sw.n, ldp, p.k, nj, g, c.scale, out, lddw * p.es);
        BLP_HIP(hipGetLastError());
      } else {
        rc = product<T, COL, COL>(p.sw.shape, aw, 1, EpiOut<T>{out, lddw * p.es, p.k, nj, g, c.scale}, c.st);
      }
    }
  }
  if (rc) return rc;
  if (dx && parts_x && p.m > 0) {
    k_sum_parts<T><<<grid_for(p.m * (ldp / 4)), 256, 0, c.st>>>(px, p.sx.n, ldp, p.k, p.m, g, c.scale, (char*)dx, lddx * p.es);
    BLP_HIP(hipGetLastError());
  }
  return 0;
}

int check_args(int type, int64_t rows, int64_t cols, int k) {
  BLP_CHECK(type >= 0 && type <= 2, BLP_E_ARG, "softmax loss: type must be BLP_F32, BLP_BF16 or BLP_F16");
  BLP_CHECK(rows >= 0 && rows < (1ll << 31), BLP_E_ARG, "softmax loss: rows must be in [0, 2^31)");
  BLP_CHECK(cols >= 1 && cols < (1ll << 31), BLP_E_ARG, "softmax loss: the catalogue must have 1 to 2^31 - 1 rows");
  BLP_CHECK(k >= 1 && k <= (1 << 20), BLP_E_ARG, "softmax loss: k must be in [1, 2^20]");
  return 0;
}

template <int T>
int run(Call& c, const void* x, int64_t ldx, const void* w, int64_t ldw, float* loss, float* lse, float* total, int mean,
        bool fwd, RowGrad g, void* dx, int64_t lddx, void* dw, int64_t lddw) {
  int rc = bind<T>(c, x, ldx, w, ldw);
  if (!rc && fwd) rc = forward<T>(c, loss, lse, total, mean);
  if (!rc && c.p.grads) rc = backward<T>(c, lse, g, dx, lddx, dw, lddw);
  return rc;
}

int dispatch(int device, void* stream, int type, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* target,
             int target64, int64_t m, int64_t n, int k, float scale, float* loss, float* lse, float* total, int mean, bool fwd,
             RowGrad g, bool grads, void* dx, int64_t lddx, void* dw, int64_t lddw, void* ws, int64_t ws_bytes) {
  int rc = check_args(type, m, n, k);
  if (rc) return rc;
  const int es = size_of(type);
  BLP_CHECK(w && (m == 0 || (x && target && loss && lse)) && ws, BLP_E_ARG, "softmax loss: null pointer");
  BLP_CHECK(ldx >= k && ldw >= k && (!dx || lddx >= k) && (!dw || lddw >= k), BLP_E_ARG,
            "softmax loss: a row stride is smaller than k");
  BLP_CHECK(std::max(ldx, ldw) <= (1 << 20) , BLP_E_ARG, "softmax loss: row strides must be at most 2^20 elements");
  Call c;
  c.p = plan_of(type, m, n, k, fwd, grads, !aligned(x, ldx * es, (int64_t)k * es), !aligned(w, ldw * es, (int64_t)k * es));
  BLP_CHECK(ws_bytes >= c.p.bytes, BLP_E_ARG, "softmax loss: the workspace is too small (blp_softmax_loss_workspace)");
  BLP_CHECK(((uintptr_t)ws & 255) == 0, BLP_E_ARG, "softmax loss: the workspace must be 256-byte aligned");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  c.st = (hipStream_t)stream;
  c.targets = {target, target64, n};
  c.scale = scale;
  c.ws = (char*)ws;
  if (type == F32) return run<F32>(c, x, ldx, w, ldw, loss, lse, total, mean, fwd, g, dx, lddx, dw, lddw);
  if (type == BF16) return run<BF16>(c, x, ldx, w, ldw, loss, lse, total, mean, fwd, g, dx, lddx, dw, lddw);
  return run<F16>(c, x, ldx, w, ldw, loss, lse, total, mean, fwd, g, dx, lddx, dw, lddw);
}

}  // namespace

extern "C" int blp_softmax_loss_workspace(int type, const void* x, int64_t ldx, const void* table, int64_t ldt, int64_t rows,
                                          int64_t cols, int k, int forward, int grads, int64_t* bytes) {
  int rc = check_args(type, rows, cols, k);
  if (rc) return rc;
  BLP_CHECK(bytes, BLP_E_ARG, "softmax loss: null pointer");
  const int es = size_of(type);
  *bytes = plan_of(type, rows, cols, k, forward != 0, grads != 0, !aligned(x, ldx * es, (int64_t)k * es),
                   !aligned(table, ldt * es, (int64_t)k * es))
               .bytes;
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
