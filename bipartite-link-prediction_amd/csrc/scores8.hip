// Scores of the catalogue from 8-bit factors (blp_quantize_rows, blp_scores8).
//
//   s_i = max_k |x_ik| / 127      q_ik = x_ik / s_i rounded to the nearest whole number, halves to the even one
//   C_ij = s_i t_j sum_k q_ik p_jk
//
// The sum of products is a whole number in 32 bits, exact for k < 2^17; it is scaled in 32-bit floats and
// rounded to the output's type once.
#include <algorithm>

#include "blp_internal.h"
#include "latent.h"

namespace {

using namespace blp::tile;
using namespace blp::rows;
using blp::DeviceGuard;
using blp::div_up;
using blp::up;
using blp::FastDiv;

struct __attribute__((packed, aligned(1))) Unaligned4 {
  uint32_t v;
};


// ---------------------------------------------------------------- quantising
// x / s rounded to nearest, halves to even -- of the true quotient, not of its 32-bit rounding: the first
// guess is off by one at most (a division: 1 / s may not be a number of 32 bits), and x - q s is exact in an fma (both are
// multiples of the smaller last place of x and s, and the difference is about s / 2 at most), so comparing it with s / 2
// settles the guess.
__device__ inline int to8(float x, float s) {
  float q = rintf(x / s);
  const float r = fmaf(-q, s, x), half = 0.5f * s;
  const bool odd = ((int)q & 1) != 0;
  if (r > half || (r == half && odd)) q += 1.f;
  if (r < -half || (r == -half && odd)) q -= 1.f;
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

// `lanes` (a power of two up to 64) lanes a row, one 16-byte vector each a step. HELD steps (1 or 8) stay in registers between
// the maximum and the rounding; longer rows (0) are read twice, the second time out of the cache. Bytes [k, kp) of a row are
// set to zero. A row with a NaN or an infinity gets the scale NaN and zeros, so its scores are NaN; a row of zeros the scale
// 0. 4,096 rows of 4,096 bf16 take 18 us: moving x and q would take 11 (4.68 TB/s), the arithmetic after the loads is not hidden.
template <int T, int HELD>
__global__ __launch_bounds__(256) void k_quantize(const char* __restrict__ x, int64_t ld, int64_t rows, int k, int kp, int lanes,
                                                  int8_t* __restrict__ q, int64_t ldq, float* __restrict__ s) {
  constexpr int ES = size_of(T), NE = Vec<T>::NE;
  const int64_t row = (blockIdx.x * 256ll + threadIdx.x) / lanes;
  const int l = threadIdx.x & (lanes - 1);
  if (row >= rows) return;
  const char* src = x + row * ld;
  uint32_t top = 0;
  auto largest = [&](const Vec<T>& v) {
#pragma unroll
    for (int e = 0; e < NE; ++e) top = max(top, __float_as_uint(fabsf(v.v[e >> 2][e & 3])));  // a NaN's bits are the largest
  };
  auto load = [&](int e0) { return e0 < k ? load_vec<T>(src + (int64_t)e0 * ES, k - e0) : Vec<T>{}; };
  Vec<T> held[HELD ? HELD : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int u = 0; u < HELD; ++u) held[u] = load((u * lanes + l) * NE);
#pragma unroll
    for (int u = 0; u < HELD; ++u) largest(held[u]);
  } else {
#pragma unroll 4
    for (int e0 = l * NE; e0 < k; e0 += lanes * NE) largest(load(e0));
  }
  for (int o = lanes >> 1; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  const bool bad = top >= 0x7f800000u;
  const float scale = bad ? NAN : __builtin_bit_cast(float, top) / 127.f;
  const bool none = bad || scale == 0.f;
  if (l == 0) s[row] = scale;
  // x / s by a product: a guess that lies within s / 2 of x is right (0 where 1 / s is no number of 32 bits: never)
  const float inverse = 1.f / scale, border = scale >= 0x1p-126f ? 0.5f * scale : 0.f;
  int8_t* dst = q + row * ldq;
  auto put = [&](const Vec<T>& v, int e0) {
    uint32_t w[NE / 4];
#pragma unroll
    for (int i = 0; i < NE / 4; ++i) w[i] = 0;
    if (!none) {
      float off = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const float at = v.v[e >> 2][e & 3], guess = rintf(at * inverse);
        off = fmaxf(off, fabsf(fmaf(-guess, scale, at)));
        w[e >> 2] |= ((uint32_t)(int)guess & 255u) << (8 * (e & 3));
      }
      if (!(off < border)) {  // one of them on or past a border: rare
#pragma unroll
        for (int i = 0; i < NE / 4; ++i) w[i] = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) w[e >> 2] |= ((uint32_t)to8(v.v[e >> 2][e & 3], scale) & 255u) << (8 * (e & 3));
      }
    }
    if (e0 + NE <= kp) {
#pragma unroll
      for (int i = 0; i < NE / 4; ++i) reinterpret_cast<Unaligned4*>(dst + e0)[i].v = w[i];
    } else {
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (e0 + e < kp) dst[e0 + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (int u = 0; u < HELD; ++u)
      if ((u * lanes + l) * NE < kp) put(held[u], (u * lanes + l) * NE);
  } else {
#pragma unroll 4
    for (int e0 = l * NE; e0 < kp; e0 += lanes * NE) put(load(e0), e0);
  }
}

template <int T>
int quantize(const void* x, int64_t ld, int64_t rows, int k, int kp, int8_t* q, int64_t ldq, float* s, hipStream_t st) {
  constexpr int NE = Vec<T>::NE;
  int lanes = 1;
  while (lanes < 64 && lanes * NE < kp) lanes <<= 1;
  const int64_t most = (1ll << 31) / lanes;  // rows of a launch, which takes less than 2^32 threads
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int64_t n = std::min(most, rows - r0);
    const unsigned grid = (unsigned)((n * lanes + 255) / 256);
    (lanes * NE >= kp ? k_quantize<T, 1> : lanes * NE * 8 >= kp ? k_quantize<T, 8> : k_quantize<T, 0>)<<<grid, 256, 0, st>>>(
        (const char*)x + r0 * ld * size_of(T), ld * size_of(T), n, k, kp, lanes, q + r0 * ldq, ldq, s + r0);
    BLP_HIP(hipGetLastError());
  }
  return 0;
}

// 8-bit rows as the tile engine takes them: whole granules, zeros past k.
__global__ __launch_bounds__(256) void k_pack8(const int8_t* __restrict__ src, int64_t ld, int64_t rows, int k, FastDiv per,
                                               int8_t* __restrict__ dst) {
  const int64_t n = rows * per.d, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t r = n < (1ll << 31) ? (int64_t)per((uint32_t)i) : i / per.d;
    const int e0 = (int)(i - r * per.d) * 16;
    const int8_t* s = src + r * ld + e0;
    i32x4 v = {0, 0, 0, 0};
    if (e0 + 16 <= k) {
      v = reinterpret_cast<const Unaligned16*>(s)->v;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (e0 + j < k) v[j >> 2] |= (int)((uint32_t)(uint8_t)s[j] << (8 * (j & 3)));
    }
    reinterpret_cast<i32x4*>(dst)[i] = v;
  }
}

// ---------------------------------------------------------------- scores
template <int TO, bool STREAM = false>  // past the caches
struct EpiScores {
  char* out;
  int64_t ld;  // bytes
  const float *s, *t;
  int64_t np, nq;
  template <class S>
  __device__ void run(i32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int, int, lds_char* scratch) const {
    if (p0 >= np || q0 >= nq) return;
    const int lane = fresh_lane(), l = lane & 15, h = lane >> 4;
    const int left = (int)min(np - p0, (int64_t)(S::FP * 16)), rows = (int)min(nq - q0, (int64_t)(S::FQ * 16));
    f32x4 tp[S::FP];
    float sq[S::FQ];
#pragma unroll
    for (int i = 0; i < S::FP; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) tp[i][e] = t[p0 + min(i * 16 + h * 4 + e, left - 1)];
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) sq[j] = s[q0 + min(j * 16 + l, rows - 1)];
    bool far = false;
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) far |= fabsf(sq[j]) > 0x1p96f;
    far = __any(far);
    store_block<TO, S, STREAM>(scratch, out + q0 * ld + p0 * size_of(TO), ld, left, rows, [&](int i, int j) {
      f32x4 v;
      if (far) {  // |sum| < 2^31, times s it may pass the largest float though the score does not: in 64 bits
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)((double)acc[i][j][e] * sq[j] * tp[i][e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j][e] * sq[j] * tp[i][e];
      }
      return v;
    });
  }
};

// A slice's sums of k as they are: part[slice][q][p].
struct EpiSums {
  int32_t* part;
  int64_t ld, nq;  // elements; ld a multiple of 4
  template <class S>
  __device__ void run(i32x4 (&acc)[S::FP][S::FQ], int64_t p0, int64_t q0, int, int slice, lds_char*) const {
    const int lane = fresh_lane(), h = lane >> 4;
    int32_t* base = part + (int64_t)slice * nq * ld;
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) {
      const int64_t q = q0 + j * 16 + (lane & 15);
      if (q >= nq) continue;
#pragma unroll
      for (int i = 0; i < S::FP; ++i) {
        const int64_t p = p0 + i * 16 + h * 4;
        if (p < ld) *reinterpret_cast<i32x4*>(base + q * ld + p) = acc[i][j];
      }
    }
  }
};

// The slices' sums as scores, four a thread.
template <int TO>
__global__ __launch_bounds__(256) void k_join8(const int32_t* __restrict__ part, int slices, int64_t ld, FastDiv per, EpiScores<TO> epi) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const int64_t row = per(i), p = ((int64_t)i - row * per.d) * 4;
  if (row >= epi.nq) return;
  i32x4 sum = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < slices; ++s) sum += *reinterpret_cast<const i32x4*>(part + ((int64_t)s * epi.nq + row) * ld + p);
  const double sq = epi.s[row];
  char* at = epi.out + row * epi.ld + p * size_of(TO);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (p + e < epi.np) {
      const float v = fabs(sq) > 0x1p96 ? (float)((double)sum[e] * sq * epi.t[p + e]) : (float)sum[e] * (float)sq * epi.t[p + e];
      store1<TO>(at + e * size_of(TO), v);
    }
}

// k up to 128: one stage, and the outputs are what counts. A workgroup of 8 waves, 16 rows and 16 FP columns each, in 32
// KiB of LDS, so that three of them share a compute unit and some load and multiply while others store. Bound by the
// stores: 10,000 x 100,000 bf16, 2.0 GB, 0.45 to 0.48 ms (4.2 to 4.4 TB/s; a fill reaches 6.8). Larger k go through
// k_product (4,096 x 16,384 x 4,096: 241 us, 2,278 TOP/s).
template <int FP_>
struct OuterShape : Shape<1, 8, FP_, 1> {
  static constexpr int SCRATCH = 4096;
};
template <int TO, bool STREAM>
__global__ __launch_bounds__(512, 6) void k_outer8(Problem a, EpiScores<TO, STREAM> epi) {
  using S = OuterShape<TO == F32 ? 4 : 8>;
  __shared__ __attribute__((aligned(1024))) char s_all[32768];
  int tp, tq;
  tile_of(a, blockIdx.x, &tp, &tq);
  const int64_t p0 = (int64_t)tp * S::BP, q0 = (int64_t)tq * S::BQ;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  lds_char *lp = (lds_char*)s_all, *lq = lp + S::BP * STAGE;
  load_stage<I8, ROW, S::BP, 8>(lp, a.p, p0, 0, a.k);
  load_stage<I8, ROW, S::BQ, 8>(lq, a.q, q0, 0, a.k);
  i32x4 acc[S::FP][1];
#pragma unroll
  for (int i = 0; i < S::FP; ++i) acc[i][0] = i32x4{0, 0, 0, 0};
  stage_barrier();
  const uint32_t bp = lane_base<I8, ROW, S::BP>(), bq = lane_base<I8, ROW, S::BQ>();
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    Frags<I8, ROW, ROW, S> f;
    f.read(lp, lq, bp, bq, 0, wave, kk);
    f.multiply(acc);
  }
  __syncthreads();
  epi.template run<S>(acc, p0, q0 + wave * 16, 0, 0, lp + wave * 4096);
}

// The same where many rows of outputs do not begin at whole vectors: k_outer8's stores of 16 bytes straddle lines, 10,000 x
// 99,998 take 0.95 ms past the caches, 0.67 through them and 0.62 here (float32: 1.87, 1.01 and 0.83). A workgroup passes
// along a strip of columns, W of them a step, with its 128 rows of q in registers; the scores go through LDS, where row r
// begins at its place within its line, so that LINES whole lines of
// every row leave, aligned, a step; what is left of the last one is carried to the next step. Only a strip's ends are
// partial lines.
template <int TO>
struct Strip {
  static constexpr int LINES = TO == F32 ? 2 : 1, W = LINES * 128 / size_of(TO), PITCH = (LINES + 1) * 128 + 16;
};
template <int TO, int KK>
__global__ __launch_bounds__(512) void k_strip8(Operand w, Operand x, int k, EpiScores<TO> epi, int strips, int steps) {
  constexpr int ES = size_of(TO), EG = 16 / ES, LINES = Strip<TO>::LINES, W = Strip<TO>::W, FP = W / 16, PITCH = Strip<TO>::PITCH;
  constexpr int GR = LINES * 8, RPI = 64 / GR;  // granules of a row a step, rows a store instruction
  __shared__ __attribute__((aligned(1024))) char s_p[W * STAGE], s_q[W * STAGE];
  __shared__ __attribute__((aligned(16))) char s_rows[8][16 * PITCH];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15, h = lane >> 4;
  // a die's workgroups take neighbouring rows of one strip: the strip's part of the catalogue stays in its L2
  const int n = gridDim.x, groups = n / strips, per = n >> 3, more = n & 7, xcd = blockIdx.x & 7;
  const int id = xcd * per + min(xcd, more) + (blockIdx.x >> 3);
  const int strip = id / groups;
  const int64_t q0 = ((int64_t)(id - strip * groups) * 8 + wave) * 16, c0 = (int64_t)strip * steps * W;
  const int total = (int)min((int64_t)steps * W, w.rows - c0), rows = (int)max(min(x.rows - q0, (int64_t)16), (int64_t)0);
  lds_char* const lds = (lds_char*)s_rows[wave];

  const int64_t qr = min(q0 + l, x.rows - 1);
  frag_t q[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    q[kk] = frag_t{0, 0, 0, 0};
    if (kk * 64 + h * 16 < k) q[kk] = *reinterpret_cast<const frag_t*>(x.base + qr * x.ld + kk * 64 + h * 16);
  }
  const float sq = epi.s[qr];
  const bool far = __any(fabsf(sq) > 0x1p96f);
  char* const out = epi.out + q0 * epi.ld + c0 * ES;  // row r's first output: out + r ld
  auto place = [&](int r) { return (int)((uintptr_t)(out + r * epi.ld) & 127); };
  lds_char* const mine = lds + l * PITCH + place(l) + h * 4 * ES;
  int at[16 / RPI];  // the granule's place among its row's outputs, in elements
  char* to[16 / RPI];
#pragma unroll
  for (int i = 0; i < 16 / RPI; ++i) {
    const int r = i * RPI + lane / GR;
    to[i] = r < rows ? out + r * epi.ld - place(r) + (lane & (GR - 1)) * 16 : nullptr;
    at[i] = (lane & (GR - 1)) * EG - place(r) / ES;
  }
  f32x4 t[FP];
  auto scales = [&](int c) {
#pragma unroll
    for (int f = 0; f < FP; ++f) {
      const int first = c + f * 16 + h * 4;
      if (c + W <= total) {
        struct __attribute__((packed, aligned(4))) Four {
          f32x4 v;
        };
        t[f] = reinterpret_cast<const Four*>(epi.t + c0 + first)->v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[f][e] = epi.t[c0 + min(first + e, total - 1)];
      }
    }
  };
  auto emit = [&](int c) {  // the outputs from column c on that lie in the first LINES lines
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
      const i32x4 v = *(const __attribute__((address_space(3))) i32x4*)(lds + (i * RPI + lane / GR) * PITCH + (lane & (GR - 1)) * 16);
      char* const o = to[i] + (int64_t)c * ES;
      const int first = at[i] + c;  // of the lane's granule
      if (to[i] && first >= 0 && first + EG <= total) {
        __builtin_nontemporal_store(v, reinterpret_cast<i32x4*>(o));
      } else if (to[i] && first + EG > 0 && first < total) {
#pragma unroll
        for (int e = 0; e < EG; ++e)
          if (first + e >= 0 && first + e < total) {
            if constexpr (ES == 4)
              reinterpret_cast<int*>(o)[e] = v[e];
            else
              reinterpret_cast<uint16_t*>(o)[e] = (uint16_t)((uint32_t)v[e >> 1] >> (16 * (e & 1)));
          }
      }
    }
  };
  const uint32_t base = lane_base<I8, ROW, W>();
  auto load = [&](char* buf, int c) { load_stage<I8, ROW, W, 8>((lds_char*)buf, w, c0 + c, 0, k); };
  auto step = [&](const char* buf, int c) {
    if (c >= total) return;
    i32x4 acc[FP];
#pragma unroll
    for (int f = 0; f < FP; ++f) {
      acc[f] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) acc[f] = mma<I8>(read_frag<I8, ROW, W>((const lds_char*)buf, base, f, kk), q[kk], acc[f]);
    }
#pragma unroll
    for (int f = 0; f < FP; ++f) {
      f32x4 v;
      if (far) {  // |sum| < 2^31, times s it may pass the largest float though the score does not: in 64 bits
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)((double)acc[f][e] * sq * t[f][e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)acc[f][e] * sq * t[f][e];
      }
      if constexpr (TO == F32) {
        struct __attribute__((packed, aligned(4))) Out {
          f32x4 v;
        };
        ((__attribute__((address_space(3))) Out*)(mine + f * 16 * ES))->v = v;
      } else {
        struct __attribute__((packed, aligned(2))) Out {
          i32x2 v;
        };
        i32x2 b;
        if constexpr (TO == BF16)
          b = __builtin_bit_cast(i32x2, __builtin_convertvector(v, bf16x4));
        else
          b = __builtin_bit_cast(i32x2, __builtin_convertvector(v, f16x4));
        ((__attribute__((address_space(3))) Out*)(mine + f * 16 * ES))->v = b;
      }
    }
    scales(min(c + W, total - 1));
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    emit(c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // the last line, not yet whole, becomes the first
      lds_char* const r = lds + (i * 8 + (lane >> 3)) * PITCH + (lane & 7) * 16;
      *(__attribute__((address_space(3))) i32x4*)r = *(const __attribute__((address_space(3))) i32x4*)(r + LINES * 128);
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  load(s_p, 0);
  scales(0);
  int c = 0;
  for (; c < total; c += 2 * W) {  // rows past the catalogue's end and steps past the strip's copy zeros, or are not taken
    stage_barrier();
    load(s_q, c + W);
    step(s_p, c);
    stage_barrier();
    load(s_p, c + 2 * W);
    step(s_q, c + W);
  }
  emit((total + W - 1) / W * W);  // what the carried line holds
  __builtin_amdgcn_s_waitcnt(0x0f70);  // nothing in flight towards LDS when the workgroup ends
}

using NarrowQ = Shape<4, 1, 4, 2>;  // 256 x 32

// The tiles of longer rows, and how many slices of k: a tile's stages take about 1 us each (large tiles: 1.8), its outputs
// 2.5 stages; slices take one more launch and their sums' way through memory. 10 x 1,266 x 6,462: 5 tiles of 51 stages,
// 52 us in one slice and 19 in 17, each with the packing of its rows.
enum Tiles { NARROW, MID, BIG };
struct Split {
  Tiles tiles;
  int n, stages;  // slices, stages of each
  int64_t bytes;  // of their sums
};
Split split_of(int64_t rows, int64_t cols, int k) {
  const int64_t stages = div_up(k, STAGE);
  Split best = {MID, 1, (int)stages, 0};
  // two stages of k: two small workgroups a compute unit, so that one's stores run beside the other's loads
  if (rows <= 32)
    best.tiles = NARROW;
  else if (k > 2 * STAGE && div_up(cols, 256) * div_up(rows, 256) >= 192)
    best.tiles = BIG;
  const int64_t tiles = div_up(cols, best.tiles == MID ? 128 : 256) * div_up(rows, best.tiles == NARROW ? 32 : best.tiles == MID ? 128 : 256);
  const int64_t slots = best.tiles == BIG ? 256 : 512;
  double least = -1;
  for (int64_t n = 1; n <= 32 && n * tiles <= slots && n <= std::max<int64_t>(stages / 2, 1); ++n) {
    const int64_t each = div_up(stages, n), slices = div_up(stages, each), bytes = slices * rows * up(cols, 4) * 4;
    const double cost = ((double)each + 2.5) * (best.tiles == BIG ? 1.8 : 1.0) + (slices > 1 ? 4.0 + 2.0 * bytes / 4e6 : 0.0);
    if (least < 0 || cost < least) {
      least = cost;
      best.n = (int)slices;
      best.stages = (int)each;
      best.bytes = slices > 1 ? bytes : 0;
    }
  }
  return best;
}

template <class S, class Epi>
int launch(Problem a, int slices, int stages, Epi epi, hipStream_t st) {
  const int64_t tp = div_up(a.p.rows, S::BP), tq = div_up(a.q.rows, S::BQ);
  a.tiles_p = (int)tp;
  a.tiles_q = (int)tq;
  a.slice = stages;
  const dim3 grid((unsigned)std::min<int64_t>(tp * tq, S::BP == 256 && S::BQ == 256 ? 256 : 512), (unsigned)slices);
  k_product<I8, ROW, ROW, 1, S, Epi><<<grid, S::THREADS, 0, st>>>(a, epi);
  BLP_HIP(hipGetLastError());
  return 0;
}
template <class Epi>
int launch(const Problem& a, const Split& s, Epi epi, hipStream_t st) {
  if (s.tiles == NARROW) return launch<NarrowQ>(a, s.n, s.stages, epi, st);
  if (s.tiles == BIG) return launch<Big>(a, s.n, s.stages, epi, st);
  return launch<Mid>(a, s.n, s.stages, epi, st);
}

constexpr int64_t MOST_BLOCKS = (1 << 23) - 1;  // of 512 threads: a launch takes less than 2^32 threads

template <int TO>
int scores(const Operand& w, const Operand& x, int k, const float* s, const float* t, void* out, int64_t ldo, char* ws, hipStream_t st) {
  const Problem a = {w, x, k, (int)div_up(k, STAGE), 0, 0, 0, 0};
  // Outputs that the last-level cache holds (256 MB) are written to it, and so are rows that do not begin at whole vectors,
  // whose lines meet there; others go past it. 3,000 x 20,001 x 500 bf16, 0.12 GB: 74 us, past it 89; 12,000 x 16,001 x 144,
  // 0.38 GB: 160 and 290; 10,000 x 100,000 x 64, 2 GB: 659 and 492.
  const bool vectors = (((uintptr_t)out | (uintptr_t)(ldo * size_of(TO))) & 15) == 0, large = x.rows * ldo * size_of(TO) > 256ll << 20;
  const EpiScores<TO> epi = {(char*)out, ldo * size_of(TO), s, t, w.rows, x.rows};
  const EpiScores<TO, true> past = {epi.out, epi.ld, s, t, w.rows, x.rows};
  if (k <= STAGE && x.rows > 32) {
    // 0.24 GB of bf16 take 81 us in strips and 62 without, 0.4 GB 134 and 150, 0.48 GB of float32 110 and 134
    if (!vectors && large) {
      constexpr int W = Strip<TO>::W;
      const int64_t groups = div_up(x.rows, 128), all = div_up(w.rows, W);
      const int64_t want = std::max<int64_t>(std::min<int64_t>(div_up(2560, groups), all / 4), 1);  // 10 workgroups a compute unit
      const int64_t steps = std::min<int64_t>(div_up(all, want), (1 << 29) / W);  // a strip's columns are counted in 31 bits
      const int64_t strips = div_up(all, steps);
      if (groups * strips <= MOST_BLOCKS) {
        (k <= 64 ? k_strip8<TO, 1> : k_strip8<TO, 2>)<<<(unsigned)(groups * strips), 512, 0, st>>>(w, x, k, epi, (int)strips, (int)steps);
        BLP_HIP(hipGetLastError());
        return 0;
      }
    }
    Problem o = a;
    o.tiles_p = (int)div_up(w.rows, TO == F32 ? 64 : 128);
    o.tiles_q = (int)div_up(x.rows, 128);
    if ((int64_t)o.tiles_p * o.tiles_q <= MOST_BLOCKS) {
      const unsigned grid = (unsigned)(o.tiles_p * o.tiles_q);
      if (large)
        k_outer8<TO, true><<<grid, 512, 0, st>>>(o, past);
      else
        k_outer8<TO, false><<<grid, 512, 0, st>>>(o, epi);
      BLP_HIP(hipGetLastError());
      return 0;
    }
  }
  // longer rows, and outputs of more than 2^37 scores: workgroups that take tile after tile
  const Split split = split_of(x.rows, w.rows, k);
  if (split.n == 1) return vectors && large ? launch(a, split, past, st) : launch(a, split, epi, st);
  const int64_t ld = up(w.rows, 4);
  const int rc = launch(a, split, EpiSums{(int32_t*)ws, ld, x.rows}, st);
  if (rc) return rc;
  k_join8<TO><<<(unsigned)div_up(x.rows * ld / 4, 256), 256, 0, st>>>((const int32_t*)ws, split.n, ld, FastDiv((uint32_t)(ld / 4)), epi);
  BLP_HIP(hipGetLastError());
  return 0;
}

// Which operands are packed: those whose rows do not begin at whole granules, and, where k ends inside a granule, one of
// them at least (the shorter): zeros past its k make what the other holds there count for nothing. (A granule that begins
// inside a row ends on the same page.)
struct Packed {
  bool x, w;
};
Packed packed(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t cols, int k) {
  Packed p = {(((uintptr_t)x | (uintptr_t)ldx) & 15) != 0, (((uintptr_t)w | (uintptr_t)ldw) & 15) != 0};
  if (k % 16 && !p.x && !p.w) (rows <= cols ? p.x : p.w) = true;
  return p;
}

int check_args(int64_t rows, int64_t cols, int k) {
  BLP_CHECK(rows >= 0 && rows < (1ll << 31) && cols >= 1 && cols < (1ll << 31), BLP_E_ARG,
            "scores8: rows must be in [0, 2^31), columns in [1, 2^31)");
  BLP_CHECK(k >= 1 && k < (1 << 17), BLP_E_ARG, "scores8: k must be in [1, 2^17)");
  BLP_CHECK(div_up(rows, 128) * div_up(cols, 128) < (1ll << 31), BLP_E_ARG, "scores8: rows x columns must be below 2^45");
  return 0;
}

int64_t workspace(const void* q, int64_t ldq, const void* p, int64_t ldp, int64_t rows, int64_t cols, int k) {
  const int64_t kp = up(k, 16);
  const Packed pack = packed(q, ldq, p, ldp, rows, cols, k);
  return (pack.x ? up(rows * kp, 256) : 0) + (pack.w ? up(cols * kp, 256) : 0) + split_of(rows, cols, k).bytes;
}

int pack(Operand& o, int k, char*& ws, hipStream_t st) {
  const int64_t kp = up(k, 16), n = o.rows * kp / 16;
  k_pack8<<<(unsigned)std::max<int64_t>(std::min<int64_t>(div_up(n, 256), 8192), 1), 256, 0, st>>>(
      (const int8_t*)o.base, o.ld, o.rows, k, FastDiv((uint32_t)(kp / 16)), (int8_t*)ws);
  BLP_HIP(hipGetLastError());
  o = {ws, kp, o.rows};
  ws += up(o.rows * kp, 256);
  return 0;
}

}  // namespace

extern "C" int blp_quantize_rows(int device, void* stream, int type, const void* x, int64_t ldx, int64_t rows, int k, int8_t* q,
                                 int64_t ldq, float* s) {
  BLP_CHECK(type >= 0 && type <= 2, BLP_E_ARG, "quantize_rows: type must be BLP_F32, BLP_BF16 or BLP_F16");
  BLP_CHECK(rows >= 0 && rows < (1ll << 31) && k >= 1 && k <= (1 << 20), BLP_E_ARG,
            "quantize_rows: rows must be in [0, 2^31), k in [1, 2^20]");
  if (rows == 0) return 0;
  BLP_CHECK(x && q && s, BLP_E_ARG, "quantize_rows: null pointer");
  BLP_CHECK(ldx >= k && ldq >= k, BLP_E_ARG, "quantize_rows: a row stride is smaller than k");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  hipStream_t st = (hipStream_t)stream;
  const int kp = (int)std::min<int64_t>(ldq, (k + 15) / 16 * 16);
  if (type == F32) return quantize<F32>(x, ldx, rows, k, kp, q, ldq, s, st);
  if (type == BF16) return quantize<BF16>(x, ldx, rows, k, kp, q, ldq, s, st);
  return quantize<F16>(x, ldx, rows, k, kp, q, ldq, s, st);
}

extern "C" int blp_scores8_workspace(const int8_t* q, int64_t ldq, const int8_t* table, int64_t ldt, int64_t rows, int64_t cols,
                                     int k, int64_t* bytes) {
  int rc = check_args(rows, cols, k);
  if (rc) return rc;
  BLP_CHECK(bytes, BLP_E_ARG, "scores8: null pointer");
  *bytes = workspace(q, ldq, table, ldt, rows, cols, k);
  return 0;
}

extern "C" int blp_scores8(int device, void* stream, const int8_t* q, int64_t ldq, const float* s, const int8_t* table, int64_t ldt,
                           const float* ts, int64_t rows, int64_t cols, int k, int out_type, void* out, int64_t ldo, void* ws,
                           int64_t ws_bytes) {
  int rc = check_args(rows, cols, k);
  if (rc) return rc;
  if (rows == 0) return 0;
  BLP_CHECK(out_type >= 0 && out_type <= 2, BLP_E_ARG, "scores8: type must be BLP_F32, BLP_BF16 or BLP_F16");
  BLP_CHECK(q && s && table && ts && out, BLP_E_ARG, "scores8: null pointer");
  BLP_CHECK(ldq >= k && ldt >= k && ldo >= cols, BLP_E_ARG, "scores8: a row stride is smaller than the row");
  BLP_CHECK((uintptr_t)out % size_of(out_type) == 0, BLP_E_ARG, "scores8: out must be aligned to its elements");
  BLP_CHECK(std::max(ldq, ldt) <= (1 << 22), BLP_E_ARG, "scores8: row strides must be at most 2^22");
  const int64_t need = workspace(q, ldq, table, ldt, rows, cols, k);
  BLP_CHECK(need == 0 || (ws && ws_bytes >= need), BLP_E_ARG,
            "scores8: the workspace is too small (blp_scores8_workspace)");
  BLP_CHECK(((uintptr_t)ws & 255) == 0, BLP_E_ARG, "scores8: the workspace must be 256-byte aligned");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  hipStream_t st = (hipStream_t)stream;
  char* at = (char*)ws;
  Operand x = {(const char*)q, ldq, rows}, w = {(const char*)table, ldt, cols};
  const Packed packs = packed(q, ldq, table, ldt, rows, cols, k);
  if (packs.x) rc = pack(x, k, at, st);
  if (!rc && packs.w) rc = pack(w, k, at, st);
  if (rc) return rc;
  const int kp = (int)up(k, 16);
  if (out_type == F32) return scores<F32>(w, x, kp, s, ts, out, ldo, at, st);
  if (out_type == BF16) return scores<BF16>(w, x, kp, s, ts, out, ldo, at, st);
  return scores<F16>(w, x, kp, s, ts, out, ldo, at, st);
}
