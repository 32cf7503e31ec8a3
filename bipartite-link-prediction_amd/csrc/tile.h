// The tile engine of the latent-factor products (latent.hip, scores8.hip): C[q][p] = sum_k P(p, k) Q(q, k)
// on the matrix cores, with the caller's epilogue over the accumulators. gfx950 only.
//
// A workgroup owns a tile of BP x BQ outputs and walks k in stages of 128 bytes (64 halves, 128 8-bit
// integers). A stage of each operand is copied from memory straight into LDS (16 bytes a lane, no register
// in between). A fragment is 16 bytes of a row: 8 halves or 16 8-bit integers, one 16-row matrix instruction.
// The next stage is in flight while this one is multiplied, in the other of two buffers, so a stage costs one
// barrier. A workgroup takes tile after tile, and the next one's first stage is on its way while this one is finished: with
// an odd number of stages while its outputs leave, with an even one it has landed before they do. A stage of 256 x 256 x 64 halves is 64 KiB of copies and 2,048 cycles of the matrix unit; 8,192 x
// 32,768 x 4,096 random halves run at 1,061 TFLOP/s, at 1,346 without the copies, and the copies alone take as long as
// 1,717 would (constant halves, which draw less power: 1,319): bound by power and the second-level cache together.
//
// Layouts of an operand: ROW -- k contiguous, element (p, k) at base + p ld + k size; COL -- p contiguous,
// element (p, k) at base + k ld + p size, whose halves are transposed on their way out of LDS
// (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 halves and get columns).
// LDS banks: ROW tiles hold 128 bytes a row, its 16-byte granule c stored at c ^ (row & 7), so the rows a
// fragment read touches together fall on different banks; COL tiles XOR the granule with bits of k.
//
// Bounds: an operand's granules outside its rows or its k are not read (the lane's buffer offset is set
// out of the buffer's range, which loads zeros). Bases and row strides are multiples of 16 bytes and rows
// are padded to whole granules (the callers pack what is not).
//
// The matrix instruction leaves lane l with q = l % 16 and the four p = 4 (l / 16) + 0..3 of a 16 x 16
// block: p is the contiguous dimension of what is written, and a row's reduction over p is in-lane first.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace blp {
namespace tile {

enum Type { F32 = 0, BF16 = 1, F16 = 2, I8 = 3 };
enum Layout { ROW = 0, COL = 1 };

typedef int frag_t __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int STAGE = 128;  // bytes of k a stage holds

__host__ __device__ constexpr int size_of(int t) { return t == F32 ? 4 : t == I8 ? 1 : 2; }

template <int T>
struct Acc {
  typedef f32x4 type;
};
template <>
struct Acc<I8> {
  typedef i32x4 type;
};

template <int T>
__device__ inline typename Acc<T>::type mma(frag_t p, frag_t q, typename Acc<T>::type c) {
  static_assert(T == BF16 || T == F16 || T == I8, "floats are multiplied as halves (latent.hip)");
  if constexpr (T == BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
  else if constexpr (T == F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(p, q, c, 0, 0, 0);
}

// One operand of a product: `ld` in bytes, `rows` the valid p in elements.
struct Operand {
  const char* base;
  int64_t ld;
  int64_t rows;
};

// Workgroup shape: WP x WQ waves, each FP x FQ blocks of 16 x 16.
template <int WP_, int WQ_, int FP_, int FQ_>
struct Shape {
  static constexpr int WP = WP_, WQ = WQ_, FP = FP_, FQ = FQ_;
  static constexpr int WAVES = WP * WQ, THREADS = WAVES * 64;
  static constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16;
  static constexpr int STAGE_BYTES = (BP + BQ) * 128;
  static constexpr int SHARE = STAGE_BYTES / WAVES, UNIT = SHARE < 4096 ? 1024 : 4096;
  static constexpr int SCRATCH = SHARE / UNIT * UNIT;  // LDS for a wave's outputs
};

using Big = Shape<2, 4, 8, 4>;  // 256 x 256, one workgroup a compute unit
using Mid = Shape<2, 2, 4, 4>;  // 128 x 128, two

typedef __attribute__((address_space(3))) char lds_char;

__device__ inline __amdgpu_buffer_rsrc_t rsrc_at(const char* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, 0x7fffffff, 0x00020000);
}
constexpr uint32_t OUT_OF_RANGE = 0x80000000u;

// COL tiles (halves): which granules of a row trade places, by k: the 16 lanes of a transposing read take 4 rows (k & 3)
// of 32 bytes, the next 16 the rows 8 further.
__device__ inline int col_swz(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) << 1; }

// Copy stage [k0, k0 + STAGE/size) of a tile of R rows starting at row r0 into LDS (asynchronous: counted
// by vmcnt). Every wave copies R / WAVES rows' worth of granules.
template <int T, int LAYOUT, int R, int WAVES>
__device__ inline void load_stage(lds_char* lds, const Operand& o, int64_t r0, int64_t k0, int64_t kend) {
  constexpr int ES = size_of(T), GE = 16 / ES;
  constexpr int PASS = WAVES * 64;                    // granules a pass of the workgroup copies
  constexpr int GRANULES = R * STAGE / 16;
  static_assert(GRANULES % PASS == 0, "tile too small for the workgroup");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if constexpr (LAYOUT == ROW) {
    const __amdgpu_buffer_rsrc_t rs = rsrc_at(o.base + r0 * o.ld + k0 * ES);
    const int row0 = wave * 8 + (lane >> 3);
    const int c = (lane & 7) ^ (row0 & 7);
    const bool k_ok = k0 + c * GE < kend;
    const uint32_t ld = (uint32_t)o.ld;
    const int64_t left = o.rows - r0;
    uint32_t off = (uint32_t)row0 * ld + c * 16;
#pragma unroll
    for (int i = 0; i < GRANULES / PASS; ++i) {
      const bool ok = k_ok && row0 + i * (PASS / 8) < left;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(lds + (i * PASS + wave * 64) * 16), 16,
          ok ? off : OUT_OF_RANGE, 0, 0, 0);
      off += (PASS / 8) * ld;
    }
  } else {
    constexpr int GR = R / GE;  // granules a k row
    const __amdgpu_buffer_rsrc_t rs = rsrc_at(o.base + k0 * o.ld + r0 * ES);
    const uint32_t ld = (uint32_t)o.ld;
    const int64_t left = o.rows - r0;
#pragma unroll
    for (int i = 0; i < GRANULES / PASS; ++i) {
      const int g = (i * WAVES + wave) * 64 + lane;
      const int k = g / GR, c = (g % GR) ^ (col_swz(k) & (GR - 1));
      const bool ok = k0 + k < kend && c * GE < left;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(lds + (i * PASS + wave * 64) * 16), 16,
          ok ? (uint32_t)k * ld + c * 16 : OUT_OF_RANGE, 0, 0, 0);
    }
  }
}

// Where this lane's part of fragment 0 of a stage lies (bytes). The others differ by constants and by an
// exclusive or with the fragment's number, so one register a stage addresses them all.
template <int T, int LAYOUT, int R>
__device__ inline uint32_t lane_base() {
  const int lane = threadIdx.x & 63, i = lane & 15, h = lane >> 4;
  if constexpr (LAYOUT == ROW) {
    return i * STAGE + (h ^ (i & 7)) * 16;
  } else {
    const int k = h * 8 + (i >> 2);
    return k * R * 2 + (((i & 3) >> 1) ^ (col_swz(k) & (R / 8 - 1))) * 16 + (i & 1) * 8;
  }
}

// Fragment f (rows 16 f ..) of the half stage kk: granules 4 kk + lane / 16 of k.
template <int T, int LAYOUT, int R>
__device__ inline frag_t read_frag(const lds_char* lds, uint32_t base, int f, int kk) {
  if constexpr (LAYOUT == ROW) {
    return *(const __attribute__((address_space(3))) frag_t*)(lds + (base ^ (kk * 64)) + f * 16 * STAGE);
  } else {
    static_assert(T == BF16 || T == F16, "column layout: halves");
    const lds_char* at = lds + (base ^ (f << 5)) + kk * 32 * R * 2;
    i32x4 v;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + s * 4 * R * 2));
      const i32x2 w = __builtin_bit_cast(i32x2, t);
      v[2 * s] = w[0];
      v[2 * s + 1] = w[1];
    }
    return v;
  }
}

template <int T, int LP, int LQ, class S>
struct Frags {
  frag_t p[S::FP], q[S::FQ];
  // half a stage (kk) out of LDS. The addresses are made anew each time: kept they would cost registers
  __device__ inline void read(const lds_char* lp, const lds_char* lq, uint32_t bp, uint32_t bq, int wp, int wq, int kk) {
    asm volatile("" : "+v"(bp), "+v"(bq));
#pragma unroll
    for (int j = 0; j < S::FQ; ++j) q[j] = read_frag<T, LQ, S::BQ>(lq, bq, wq * S::FQ + j, kk);
#pragma unroll
    for (int i = 0; i < S::FP; ++i) p[i] = read_frag<T, LP, S::BP>(lp, bp, wp * S::FP + i, kk);
  }
  __device__ inline void multiply(typename Acc<T>::type (&acc)[S::FP][S::FQ]) const {
#pragma unroll
    for (int i = 0; i < S::FP; ++i)
#pragma unroll
      for (int j = 0; j < S::FQ; ++j) acc[i][j] = mma<T>(p[i], q[j], acc[i][j]);
  }
};

// The lane, as a value that nothing computed from it is kept across the tiles (epilogues' addresses would cost the
// accumulators their registers).
__device__ inline int fresh_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

__device__ inline void stage_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies have landed (lgkmcnt, expcnt: any)
  __syncthreads();
}

// The same with this wave's last `LEFT` copies still in flight: a stage's copies have landed when only those of
// the LEFT issued after it are outstanding (they land in order). Every read of LDS issued before has returned.
template <int LEFT>
__device__ inline void ring_barrier() {
  static_assert(LEFT < 16, "the count's low bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | LEFT);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct Problem {
  Operand p, q;
  int64_t k;            // valid k, in elements
  int slice;            // stages of one slice (blockIdx.y) of all segments' stages; every slice launched has at least one
  int tiles_p, tiles_q;
  // Values held as sums of halves (x = x1 + x2 + ..., see latent.hip): products of the operands' planes, which lie this many
  // bytes apart, are segments of one sum over k. Six segments, three planes each: x1 w1, x1 w2, x2 w1, x2 w2, x1 w3, x3 w1,
  // one after the other. Two, of one plane of P and two of Q: p q1 and p q2 take turns, so that p's stage comes out of the
  // cache the second time.
  int64_t p_plane, q_plane;
};
__host__ __device__ constexpr int p_plane_of(int seg) { return (0x850 >> (2 * seg)) & 3; }
__host__ __device__ constexpr int q_plane_of(int seg) { return (0x244 >> (2 * seg)) & 3; }

// The workgroup's tile: consecutive workgroups go to the 8 dies in turn, so each die gets one contiguous
// range of tiles, and walks it in bands of 8 q tiles: the p tile stays in the die's L2 while they pass.
__device__ inline void tile_of(const Problem& a, int b, int* tp, int* tq) {
  const int n = a.tiles_p * a.tiles_q;
  const int per = n >> 3, extra = n & 7, xcd = b & 7, at = b >> 3;
  const int t = xcd * per + min(xcd, extra) + at;
  constexpr int BAND = 8;
  const int band = t / (BAND * a.tiles_p), in = t - band * BAND * a.tiles_p;
  const int width = min(BAND, a.tiles_q - band * BAND);
  *tp = in / width;
  *tq = band * BAND + in - *tp * width;
}

template <int T, int LP, int LQ, int SEGS, class S, class Epi>
__global__ __launch_bounds__(S::THREADS, 2) void k_product(Problem a, Epi epi) {
  constexpr int KE = STAGE / size_of(T);
  __shared__ __attribute__((aligned(1024))) char s_0[S::STAGE_BYTES], s_1[S::STAGE_BYTES];
  lds_char *l0 = (lds_char*)s_0, *l1 = (lds_char*)s_1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wp = wave % S::WP, wq = wave / S::WP;
  const uint32_t bp = lane_base<T, LP, S::BP>(), bq = lane_base<T, LQ, S::BQ>();
  const int per_seg = (int)((a.k + KE - 1) / KE), sb = blockIdx.y * a.slice;
  const int stages = min(a.slice, SEGS * per_seg - sb), tiles = a.tiles_p * a.tiles_q;
  auto load = [&](lds_char* to, int tp, int tq, int t) {
    int at = sb + t;
    Operand p = a.p, q = a.q;
    if constexpr (SEGS == 6) {
      const int seg = at / per_seg;
      at -= seg * per_seg;
      p.base += p_plane_of(seg) * a.p_plane;
      q.base += q_plane_of(seg) * a.q_plane;
    } else if constexpr (SEGS == 2) {
      q.base += (at & 1) * a.q_plane;
      at >>= 1;
    }
    load_stage<T, LP, S::BP, S::WAVES>(to, p, (int64_t)tp * S::BP, (int64_t)at * KE, a.k);
    load_stage<T, LQ, S::BQ, S::WAVES>(to + S::BP * STAGE, q, (int64_t)tq * S::BQ, (int64_t)at * KE, a.k);
  };
  auto landed = [] {  // this wave's copies, and its reads of LDS, are done; then every wave's
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  int tp, tq, np = 0, nq = 0;
  tile_of(a, blockIdx.x, &tp, &tq);
  load(l0, tp, tq, 0);
  for (int b = blockIdx.x; b < tiles; b += gridDim.x) {
    const bool more = b + (int)gridDim.x < tiles;
    if (more) tile_of(a, b + gridDim.x, &np, &nq);
    typename Acc<T>::type acc[S::FP][S::FQ];
#pragma unroll
    for (int i = 0; i < S::FP; ++i)
#pragma unroll
      for (int j = 0; j < S::FQ; ++j) acc[i][j] = 0;
    auto multiply = [&](lds_char* from) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        Frags<T, LP, LQ, S> f;
        f.read(from, from + S::BP * STAGE, bp, bq, wp, wq, kk);
        f.multiply(acc);
      }
    };
    int t = 0;
    for (; t + 2 <= stages; t += 2) {
      landed();
      load(l1, tp, tq, t + 1);
      multiply(l0);
      landed();
      if (t + 2 < stages)
        load(l0, tp, tq, t + 2);
      else if (more)
        load(l0, np, nq, 0);
      multiply(l1);
    }
    if (t < stages) {
      landed();
      multiply(l0);
    }
    __syncthreads();  // every wave's last reads are done, and its copies: the second buffer is free for the outputs
    if (t < stages && more) load(l0, np, nq, 0);
    epi.template run<S>(acc, (int64_t)tp * S::BP + wp * S::FP * 16, (int64_t)tq * S::BQ + wq * S::FQ * 16, tp * S::WP + wp, blockIdx.y,
                        l1 + wave * S::SCRATCH);
    tp = np;
    tq = nq;
  }
}

// round to the type once
template <int T>
__device__ inline void store1(char* at, float v) {
  if constexpr (T == F32) {
    *reinterpret_cast<float*>(at) = v;
  } else if constexpr (T == BF16) {
    *reinterpret_cast<__bf16*>(at) = (__bf16)v;
  } else {
    *reinterpret_cast<_Float16*>(at) = (_Float16)v;
  }
}
template <int T>
__device__ inline float load1(const char* at) {
  if constexpr (T == F32) {
    return *reinterpret_cast<const float*>(at);
  } else if constexpr (T == BF16) {
    return (float)*reinterpret_cast<const __bf16*>(at);
  } else {
    return (float)*reinterpret_cast<const _Float16*>(at);
  }
}

struct __attribute__((packed, aligned(2))) Unaligned16 {  // global memory takes any alignment
  i32x4 v;
};

// A wave's 16 FP x 16 FQ outputs, already values of the type (`value(i, j)`: the four of a lane in block (i, j)),
// into rows of `out` (row q of the block at out + q ld bytes; element p at p * size): by way of LDS, so that a row's
// elements leave as whole lines, 16 bytes a lane, instead of 8 bytes from 16 rows each. Rows from nq and elements
// from np on are not written. LDS rows are a power of two of bytes; their granules are swapped by the row's number,
// which spreads both the writes and the reads over the banks. NT: stores that do not stay in the cache.
__host__ __device__ constexpr int pow2_up(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}
template <int TO, class S, bool NT = false, class F>
__device__ inline void store_block(lds_char* scratch, char* out, int64_t ld, int64_t np, int64_t nq, F value) {
  constexpr int ES = size_of(TO), ROWB = pow2_up(S::FP * 16 * ES), GR = ROWB / 16;  // bytes, granules of an LDS row
  constexpr int FIT = S::SCRATCH / (16 * ROWB), J = FIT < S::FQ ? FIT : S::FQ;  // blocks of 16 rows a pass
  static_assert(J >= 1 && S::FQ % J == 0, "passes of whole blocks");
  constexpr int LANES = GR < 64 ? GR : 64, RPI = 64 / LANES;               // lanes a row, rows an instruction
  const int lane = fresh_lane(), l = lane & 15, h = lane >> 4;
#pragma unroll
  for (int j0 = 0; j0 < S::FQ; j0 += J) {
    if (j0) __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < S::FP; ++i) {
        if (i == 0) __builtin_amdgcn_sched_barrier(0);  // one row's values at a time: few registers
        const f32x4 v = value(i, j0 + j);
        const int row = j * 16 + l;
        if constexpr (TO == F32) {
          const int g = (i * 4 + h) ^ (row & (GR - 1) & 15);
          *(__attribute__((address_space(3))) f32x4*)(scratch + row * ROWB + g * 16) = v;
        } else {
          const int g = (i * 2 + (h >> 1)) ^ (row & (GR - 1) & 15);
          __attribute__((address_space(3))) i32x2* at =
              (__attribute__((address_space(3))) i32x2*)(scratch + row * ROWB + g * 16 + (h & 1) * 8);
          if constexpr (TO == BF16)
            *at = __builtin_bit_cast(i32x2, __builtin_convertvector(v, bf16x4));
          else
            *at = __builtin_bit_cast(i32x2, __builtin_convertvector(v, f16x4));
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int g = lane & (LANES - 1), p = g * (16 / ES);
#pragma unroll
    for (int r0 = 0; r0 < J * 16; r0 += RPI) {
      const int row = r0 + lane / LANES;
      const i32x4 v = *(const __attribute__((address_space(3))) i32x4*)(scratch + row * ROWB + (g ^ (row & (GR - 1) & 15)) * 16);
      const int64_t q = j0 * 16 + row;
      if (q >= nq) continue;
      char* at = out + q * ld + p * ES;
      if (p + 16 / ES <= np) {
        if constexpr (NT) __builtin_nontemporal_store(v, &reinterpret_cast<Unaligned16*>(at)->v); else reinterpret_cast<Unaligned16*>(at)->v = v;
      } else if (p < np) {
#pragma unroll
        for (int e = 0; e < 16 / ES; ++e)
          if (p + e < np) {
            if constexpr (ES == 4)
              reinterpret_cast<int*>(at)[e] = v[e];
            else
              reinterpret_cast<uint16_t*>(at)[e] = (uint16_t)((uint32_t)v[e >> 1] >> (16 * (e & 1)));
          }
      }
    }
  }
}

}  // namespace tile
}  // namespace blp
