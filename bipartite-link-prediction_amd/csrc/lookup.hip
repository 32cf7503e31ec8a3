// Rows of a factor table by id, scaled, and the gradient of that (blp_lookup*).
//
//   y_i = scale table[id_i] (an id outside the table: zeros)      dT_r = scale sum_{i : id_i = r} dy_i
//
// The gradient is a sum over each row's positions in ascending order, with no float atomics: the ids are
// sorted (stable, with their positions), chunks of CHUNK sorted entries are summed by one group of lanes
// each, a row's sum that lies inside a chunk is written at once and one that crosses chunks is left as
// partial sums, which a second kernel adds up in the chunks' order. Everything is read once and the result
// does not depend on timing. Bound by the reads of dy (one row per id) and the writes of dT.
#include <algorithm>

#include "blp_internal.h"
#include "latent.h"

namespace {

using namespace blp::tile;
using blp::DeviceGuard;
using blp::Ids;

// ---------------------------------------------------------------- vectors of a row
// NE elements of 16 bytes, wherever they start (global memory takes any alignment); the row's last
// vector may be short.
template <int T>
struct Vec {
  static constexpr int NE = 16 / size_of(T);
  f32x4 v[NE / 4];
};
struct __attribute__((packed, aligned(2))) Raw16 {
  i32x4 v;
};

template <int T>
__device__ inline Vec<T> load_vec(const char* at, int left) {
  constexpr int NE = Vec<T>::NE;
  Vec<T> r;
  if (left >= NE) {
    const i32x4 raw = reinterpret_cast<const Raw16*>(at)->v;
    if constexpr (T == F32) {
      r.v[0] = __builtin_bit_cast(f32x4, raw);
    } else if constexpr (T == BF16) {
      const bf16x8 b = __builtin_bit_cast(bf16x8, raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) r.v[e >> 2][e & 3] = (float)b[e];
    } else {
      const f16x8 b = __builtin_bit_cast(f16x8, raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) r.v[e >> 2][e & 3] = (float)b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e) r.v[e >> 2][e & 3] = e < left ? load1<T>(at + e * size_of(T)) : 0.f;
  }
  return r;
}

template <int T>
__device__ inline void store_vec(char* at, int left, const Vec<T>& r) {
  constexpr int NE = Vec<T>::NE;
  if (left >= NE) {
    Raw16 raw;
    if constexpr (T == F32) {
      raw.v = __builtin_bit_cast(i32x4, r.v[0]);
    } else if constexpr (T == BF16) {
      bf16x8 b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = (__bf16)r.v[e >> 2][e & 3];
      raw.v = __builtin_bit_cast(i32x4, b);
    } else {
      f16x8 b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = (_Float16)r.v[e >> 2][e & 3];
      raw.v = __builtin_bit_cast(i32x4, b);
    }
    *reinterpret_cast<Raw16*>(at) = raw;
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e)
      if (e < left) store1<T>(at + e * size_of(T), r.v[e >> 2][e & 3]);
  }
}

// ---------------------------------------------------------------- lookup
// One vector a thread, four rows in flight.
template <int T>
__global__ __launch_bounds__(256) void k_lookup(const char* __restrict__ table, int64_t ld, Ids ids, int64_t n, int k,
                                                float scale, char* __restrict__ out, int64_t ldo) {
  constexpr int NE = Vec<T>::NE, U = 4;
  const int per = (k + NE - 1) / NE;
  const int64_t total = n * per, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i0 = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i0 < total; i0 += step * U) {
    Vec<T> v[U];
    int64_t row[U];
    int e0[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * step;
      row[u] = i < total ? i / per : -1;
      e0[u] = i < total ? (int)(i - row[u] * per) * NE : 0;
      const int64_t id = row[u] >= 0 ? ids(row[u]) : -1;
      v[u] = Vec<T>{};
      if (id >= 0) v[u] = load_vec<T>(table + id * ld + (int64_t)e0[u] * size_of(T), k - e0[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] >= 0) {
#pragma unroll
        for (int j = 0; j < NE / 4; ++j) v[u].v[j] *= scale;
        store_vec<T>(out + row[u] * ldo + (int64_t)e0[u] * size_of(T), k - e0[u], v[u]);
      }
  }
}

// ---------------------------------------------------------------- sort
// Stable radix sort of (id, position), least significant digit first, BITS bits a pass. A block takes
// SORT_N consecutive entries; wave w of it the w-th quarter, 64 at a time in order. The entries of one
// digit are found with ballots (a lane's rank among them by counting the lanes below), so ranks follow
// positions; ids outside the table get the largest key and end up last.
constexpr int BITS = 10, BINS = 1 << BITS, SORT_WAVES = 4, SORT_ROUNDS = 8;
constexpr int SORT_N = SORT_WAVES * SORT_ROUNDS * 64;

// counts[digit * blocks + block]; with `zero`, also clears the gradient (16 bytes a thread).
struct Clear {
  char* out;
  int64_t ld, rows;  // bytes
  int row_bytes;
  __device__ void run(int64_t at, int64_t step) const {
    if (!out) return;
    const int per = (row_bytes + 15) / 16;
    for (int64_t i = at; i < rows * per; i += step) {
      const int64_t r = i / per;
      const int b = (int)(i - r * per) * 16;
      char* p = out + r * ld + b;
      if (b + 16 <= row_bytes) {
        reinterpret_cast<Raw16*>(p)->v = i32x4{0, 0, 0, 0};
      } else {
        for (int j = 0; j < row_bytes - b; j += 2) *reinterpret_cast<uint16_t*>(p + j) = 0;
      }
    }
  }
};

__device__ inline uint32_t key_at(const Ids& ids, const uint32_t* keys, int64_t i) {
  if (keys) return keys[i];
  const int64_t id = ids(i);
  return id >= 0 ? (uint32_t)id : (uint32_t)ids.rows;
}

__global__ __launch_bounds__(256) void k_digit_counts(Ids ids, const uint32_t* __restrict__ keys, int64_t n, int shift,
                                                      uint32_t* __restrict__ counts, Clear clear) {
  __shared__ uint32_t s_count[BINS];
  for (int i = threadIdx.x; i < BINS; i += 256) s_count[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * SORT_N;
  for (int r = 0; r < SORT_N / 256; ++r) {
    const int64_t i = base + r * 256 + threadIdx.x;
    if (i < n) atomicAdd(&s_count[(key_at(ids, keys, i) >> shift) & (BINS - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += 256) counts[(int64_t)i * gridDim.x + blockIdx.x] = s_count[i];
  clear.run(blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
}

// One wave a digit: its counts become the exclusive sums over the blocks; total[digit].
__global__ __launch_bounds__(64) void k_digit_sums(uint32_t* __restrict__ counts, int blocks, uint32_t* __restrict__ total) {
  uint32_t run = 0;
  for (int b0 = 0; b0 < blocks; b0 += 64) {
    const int b = b0 + threadIdx.x;
    const uint32_t c = b < blocks ? counts[(int64_t)blockIdx.x * blocks + b] : 0;
    uint32_t s = c;
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t t = __shfl_up(s, o, 64);
      if ((int)threadIdx.x >= o) s += t;
    }
    if (b < blocks) counts[(int64_t)blockIdx.x * blocks + b] = run + s - c;
    run += __shfl(s, 63, 64);
  }
  if (threadIdx.x == 0) total[blockIdx.x] = run;
}

__global__ __launch_bounds__(256) void k_scatter(Ids ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                 int64_t n, int shift, const uint32_t* __restrict__ counts,
                                                 const uint32_t* __restrict__ total, uint32_t* __restrict__ keys_out,
                                                 uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t s_base[BINS];
  __shared__ uint16_t s_wave[SORT_WAVES][BINS];
  __shared__ uint32_t s_sum[SORT_WAVES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < SORT_WAVES * BINS; i += 256) (&s_wave[0][0])[i] = 0;
  // where each digit starts: exclusive sums of the totals, four digits a thread
  uint32_t c[BINS / 256], sum = 0;
#pragma unroll
  for (int j = 0; j < BINS / 256; ++j) {
    c[j] = sum;
    sum += total[threadIdx.x * (BINS / 256) + j];
  }
  uint32_t s = sum;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = __shfl_up(s, o, 64);
    if (lane >= o) s += t;
  }
  if (lane == 63) s_sum[w] = s;
  __syncthreads();
  uint32_t before = s - sum;
  for (int i = 0; i < w; ++i) before += s_sum[i];
#pragma unroll
  for (int j = 0; j < BINS / 256; ++j) {
    const int d = threadIdx.x * (BINS / 256) + j;
    s_base[d] = before + c[j] + counts[(int64_t)d * gridDim.x + blockIdx.x];
  }
  // ranks within the wave
  const int64_t base = (int64_t)blockIdx.x * SORT_N + w * (SORT_ROUNDS * 64);
  uint32_t key[SORT_ROUNDS];
  uint16_t rank[SORT_ROUNDS];
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r) {
    const int64_t i = base + r * 64 + lane;
    const bool in = i < n;
    key[r] = in ? key_at(ids, keys, i) : 0;
    const uint32_t d = (key[r] >> shift) & (BINS - 1);
    unsigned long long same = __ballot(in);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
      const unsigned long long m = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? m : ~m;
    }
    const int below = __popcll(same & ((1ull << lane) - 1));
    if (in) rank[r] = (uint16_t)(s_wave[w][d] + below);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in && below == 0) s_wave[w][d] += (uint16_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < BINS / 256; ++j) {  // the waves' counts become exclusive sums over the waves
    const int d = threadIdx.x * (BINS / 256) + j;
    uint32_t run = 0;
    for (int i = 0; i < SORT_WAVES; ++i) {
      const uint32_t t = s_wave[i][d];
      s_wave[i][d] = (uint16_t)run;
      run += t;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r) {
    const int64_t i = base + r * 64 + lane;
    if (i < n) {
      const uint32_t d = (key[r] >> shift) & (BINS - 1);
      const uint32_t at = s_base[d] + s_wave[w][d] + rank[r];
      keys_out[at] = key[r];
      pos_out[at] = pos ? pos[i] : (uint32_t)i;
    }
  }
}

// Up to SMALL entries: one block, a bitonic sort of (id, position) pairs in LDS. The other blocks clear.
constexpr int SMALL = 2048;
__global__ __launch_bounds__(1024) void k_sort_small(Ids ids, int n, uint32_t* __restrict__ keys_out,
                                                     uint32_t* __restrict__ pos_out, Clear clear) {
  if (blockIdx.x > 0) {
    clear.run((blockIdx.x - 1) * 1024ll + threadIdx.x, (gridDim.x - 1) * 1024ll);
    return;
  }
  __shared__ unsigned long long s_v[SMALL];
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = threadIdx.x; i < size; i += 1024)
    s_v[i] = i < n ? (unsigned long long)key_at(ids, nullptr, i) << 32 | (uint32_t)i : ~0ull;
  __syncthreads();
  for (int k2 = 2; k2 <= size; k2 <<= 1)
    for (int j = k2 >> 1; j > 0; j >>= 1) {
      for (int t = threadIdx.x; t < size / 2; t += 1024) {
        const int a = ((t & ~(j - 1)) << 1) | (t & (j - 1)), b = a | j;
        const unsigned long long x = s_v[a], y = s_v[b];
        if ((x > y) == ((a & k2) == 0)) {
          s_v[a] = y;
          s_v[b] = x;
        }
      }
      __syncthreads();
    }
  for (int i = threadIdx.x; i < n; i += 1024) {
    keys_out[i] = (uint32_t)(s_v[i] >> 32);
    pos_out[i] = (uint32_t)s_v[i];
  }
}

// ---------------------------------------------------------------- sums
constexpr int CHUNK = 64;  // sorted entries a group of lanes adds up

template <int T>
__device__ inline void put(char* out, int64_t ldo, uint32_t key, int e0, int k, const Vec<T>& sum, float scale, int add) {
  Vec<T> r = sum;
  char* at = out + (int64_t)key * ldo + (int64_t)e0 * size_of(T);
#pragma unroll
  for (int j = 0; j < Vec<T>::NE / 4; ++j) r.v[j] *= scale;
  if (add) {
    const Vec<T> o = load_vec<T>(at, k - e0);
#pragma unroll
    for (int j = 0; j < Vec<T>::NE / 4; ++j) r.v[j] += o.v[j];
  }
  store_vec<T>(at, k - e0, r);
}

// A partial sum in 32 bits: part[(2 chunk + side) * kv + vector * NE], side 0: the chunk's first row when it
// began in an earlier chunk, side 1: its last row when it goes on in the next (and began in this one).
template <int T>
__device__ inline void put_part(float* part, int64_t slot, int64_t kv, int vec, const Vec<T>& sum) {
  f32x4* at = reinterpret_cast<f32x4*>(part + slot * kv + (int64_t)vec * Vec<T>::NE);
#pragma unroll
  for (int j = 0; j < Vec<T>::NE / 4; ++j) at[j] = sum.v[j];
}

// `lanes` (a power of two up to 64) lanes a chunk, blockIdx.y the column tile of lanes * NE elements.
template <int T>
__global__ __launch_bounds__(256) void k_chunk_sums(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t n,
                                                    uint32_t rows, const char* __restrict__ dy, int64_t ld, int k, int lanes,
                                                    float scale, char* __restrict__ out, int64_t ldo, int add,
                                                    float* __restrict__ part, int64_t kv) {
  constexpr int NE = Vec<T>::NE, U = 4;
  const int64_t chunk = (blockIdx.x * 256ll + threadIdx.x) / lanes;
  const int vec = blockIdx.y * lanes + (threadIdx.x & (lanes - 1)), e0 = vec * NE;
  const int64_t b = chunk * CHUNK, e = min(n, b + CHUNK);
  if (b >= n || e0 >= k) return;
  const char* src = dy + (int64_t)e0 * size_of(T);
  uint32_t cur = keys[b];
  bool head = b > 0 && keys[b - 1] == cur;  // the running row began in an earlier chunk
  Vec<T> sum{};
  for (int64_t i = b; i < e; i += U) {
    uint32_t key[U];
    Vec<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      key[u] = i + u < e ? keys[i + u] : rows;
      v[u] = Vec<T>{};
      if (key[u] < rows) v[u] = load_vec<T>(src + (int64_t)pos[i + u] * ld, k - e0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < e && key[u] != cur) {  // `cur` ended before this entry
        if (cur < rows) {
          if (head)
            put_part<T>(part, 2 * chunk, kv, vec, sum);
          else
            put<T>(out, ldo, cur, e0, k, sum, scale, add);
        }
        head = false;
        cur = key[u];
        sum = Vec<T>{};
      }
      if (i + u < e)
#pragma unroll
        for (int j = 0; j < NE / 4; ++j) sum.v[j] += v[u].v[j];
    }
  }
  if (cur >= rows) return;
  const bool goes_on = e < n && keys[e] == cur;
  if (head)
    put_part<T>(part, 2 * chunk, kv, vec, sum);
  else if (goes_on)
    put_part<T>(part, 2 * chunk + 1, kv, vec, sum);
  else
    put<T>(out, ldo, cur, e0, k, sum, scale, add);
}

// The rows that cross chunks: the block of the chunk in which such a row begins adds its partial sums, one
// group of lanes every (256 / lanes)-th of them in 64 bits, then the groups' in order.
template <int T>
__global__ __launch_bounds__(256) void k_join_chunks(const uint32_t* __restrict__ keys, int64_t n, uint32_t rows, int k, int lanes,
                                                     float scale, char* __restrict__ out, int64_t ldo, int add,
                                                     const float* __restrict__ part, int64_t kv) {
  constexpr int NE = Vec<T>::NE;
  __shared__ double s_sum[256 * NE];
  const int64_t chunk = blockIdx.x, e = (chunk + 1) * CHUNK;
  if (e >= n) return;
  const uint32_t key = keys[e - 1];
  if (key >= rows || keys[e] != key) return;
  if (chunk * CHUNK > 0 && keys[chunk * CHUNK] == key && keys[chunk * CHUNK - 1] == key) return;  // began earlier
  // the last chunk with this row: a search for the first entry behind it
  int64_t lo = e, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] == key)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int64_t last = (lo - 1) / CHUNK;
  const int groups = 256 / lanes, g = threadIdx.x / lanes, l = threadIdx.x & (lanes - 1);
  const int vec = blockIdx.y * lanes + l, e0 = vec * NE;
  double sum[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) sum[j] = 0.0;
  if (e0 < k)
    for (int64_t c = chunk + g; c <= last; c += groups) {
      const f32x4* at = reinterpret_cast<const f32x4*>(part + (2 * c + (c == chunk ? 1 : 0)) * kv + (int64_t)e0);
#pragma unroll
      for (int j = 0; j < NE; ++j) sum[j] += (double)at[j >> 2][j & 3];
    }
#pragma unroll
  for (int j = 0; j < NE; ++j) s_sum[j * 256 + threadIdx.x] = sum[j];
  __syncthreads();
  if (g == 0 && e0 < k) {
    Vec<T> r;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      for (int i = 1; i < groups; ++i) sum[j] += s_sum[j * 256 + i * lanes + l];
      r.v[j >> 2][j & 3] = (float)sum[j];
    }
    put<T>(out, ldo, key, e0, k, r, scale, add);
  }
}

// ---------------------------------------------------------------- host side
int64_t div_up(int64_t v, int64_t by) { return (v + by - 1) / by; }
int64_t up(int64_t v, int64_t to) { return div_up(v, to) * to; }

struct Plan {
  int passes;
  int64_t blocks, chunks, kv;
  int64_t o_keys[2], o_pos[2], o_counts, o_total, o_part, bytes;
};

Plan plan_of(int type, int64_t n, int64_t rows, int k) {
  Plan p;
  int64_t at = 0;
  auto take = [&](int64_t b) {
    const int64_t o = at;
    at += up(b, 256);
    return o;
  };
  int bits = 1;
  while (bits < 32 && (rows >> bits)) ++bits;
  p.passes = n <= SMALL ? 0 : (int)div_up(bits, BITS);
  p.blocks = div_up(n, SORT_N);
  p.chunks = div_up(n, CHUNK);
  p.kv = up(k, 16 / size_of(type));
  for (int i = 0; i < 2; ++i) {
    p.o_keys[i] = take(4 * n);
    p.o_pos[i] = take(4 * n);
  }
  p.o_counts = take(p.passes ? 4 * BINS * p.blocks : 0);
  p.o_total = take(4 * BINS);
  p.o_part = take(8 * p.chunks * p.kv);
  p.bytes = std::max<int64_t>(at, 256);
  return p;
}

template <int T>
int lookup(hipStream_t st, const void* table, int64_t ld, Ids ids, int64_t n, int k, float scale, void* out, int64_t ldo) {
  const int64_t total = n * div_up(k, 16 / size_of(T));
  const unsigned grid = (unsigned)std::min<int64_t>(div_up(total, 1024), 1 << 20);
  k_lookup<T><<<std::max(grid, 1u), 256, 0, st>>>((const char*)table, ld * size_of(T), ids, n, k, scale, (char*)out,
                                                  ldo * size_of(T));
  BLP_HIP(hipGetLastError());
  return 0;
}

template <int T>
int lookup_grad(hipStream_t st, const Plan& p, const void* dy, int64_t ld, Ids ids, int64_t n, int k, float scale, void* out,
                int64_t ldo, int add, char* ws) {
  const int ES = size_of(T);
  uint32_t* keys[2] = {(uint32_t*)(ws + p.o_keys[0]), (uint32_t*)(ws + p.o_keys[1])};
  uint32_t* pos[2] = {(uint32_t*)(ws + p.o_pos[0]), (uint32_t*)(ws + p.o_pos[1])};
  uint32_t *counts = (uint32_t*)(ws + p.o_counts), *total = (uint32_t*)(ws + p.o_total);
  const Clear none = {nullptr, 0, 0, 0}, clear = {add ? nullptr : (char*)out, ldo * ES, ids.rows, k * ES};
  int cur = 0;
  if (p.passes == 0) {
    const int64_t words = ids.rows * div_up((int64_t)k * ES, 16);
    const unsigned grid = 1 + (unsigned)std::min<int64_t>(add ? 1 : div_up(words, 4096), 1024);
    k_sort_small<<<grid, 1024, 0, st>>>(ids, (int)n, keys[0], pos[0], clear);
    BLP_HIP(hipGetLastError());
  }
  for (int s = 0; s < p.passes; ++s) {
    const uint32_t* kin = s ? keys[cur] : nullptr;
    const int to = s ? cur ^ 1 : 0;
    k_digit_counts<<<(unsigned)p.blocks, 256, 0, st>>>(ids, kin, n, s * BITS, counts, s ? none : clear);
    BLP_HIP(hipGetLastError());
    k_digit_sums<<<BINS, 64, 0, st>>>(counts, (int)p.blocks, total);
    BLP_HIP(hipGetLastError());
    k_scatter<<<(unsigned)p.blocks, 256, 0, st>>>(ids, kin, s ? pos[cur] : nullptr, n, s * BITS, counts, total, keys[to], pos[to]);
    BLP_HIP(hipGetLastError());
    cur = to;
  }
  if (n == 0) return 0;
  constexpr int NE = Vec<T>::NE;
  const int64_t vecs = div_up(k, NE);
  int lanes = 1;
  while (lanes < 64 && lanes < vecs) lanes <<= 1;
  const unsigned tiles = (unsigned)div_up(vecs, lanes);
  float* part = (float*)(ws + p.o_part);
  k_chunk_sums<T><<<dim3((unsigned)div_up(p.chunks * lanes, 256), tiles), 256, 0, st>>>(
      keys[cur], pos[cur], n, (uint32_t)ids.rows, (const char*)dy, ld * ES, k, lanes, scale, (char*)out, ldo * ES, add, part, p.kv);
  BLP_HIP(hipGetLastError());
  if (p.chunks > 1) {
    k_join_chunks<T><<<dim3((unsigned)(p.chunks - 1), tiles), 256, 0, st>>>(keys[cur], n, (uint32_t)ids.rows, k, lanes, scale,
                                                                            (char*)out, ldo * ES, add, part, p.kv);
    BLP_HIP(hipGetLastError());
  }
  return 0;
}

int check_args(int type, int64_t n, int64_t rows, int k) {
  BLP_CHECK(type >= 0 && type <= 2, BLP_E_ARG, "lookup: type must be BLP_F32, BLP_BF16 or BLP_F16");
  BLP_CHECK(n >= 0 && n < (1ll << 31), BLP_E_ARG, "lookup: the number of ids must be in [0, 2^31)");
  BLP_CHECK(rows >= 1 && rows < (1ll << 31), BLP_E_ARG, "lookup: the table must have 1 to 2^31 - 1 rows");
  BLP_CHECK(k >= 1 && k <= (1 << 20), BLP_E_ARG, "lookup: k must be in [1, 2^20]");
  return 0;
}

}  // namespace

extern "C" int blp_lookup(int device, void* stream, int type, const void* table, int64_t ldt, int64_t rows, int k, const void* ids,
                          int ids64, int64_t n, float scale, void* out, int64_t ldo) {
  int rc = check_args(type, n, rows, k);
  if (rc) return rc;
  if (n == 0) return 0;
  BLP_CHECK(table && ids && out, BLP_E_ARG, "lookup: null pointer");
  BLP_CHECK(ldt >= k && ldo >= k, BLP_E_ARG, "lookup: a row stride is smaller than k");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  const Ids at = {ids, ids64, rows};
  hipStream_t st = (hipStream_t)stream;
  if (type == F32) return lookup<F32>(st, table, ldt, at, n, k, scale, out, ldo);
  if (type == BF16) return lookup<BF16>(st, table, ldt, at, n, k, scale, out, ldo);
  return lookup<F16>(st, table, ldt, at, n, k, scale, out, ldo);
}

extern "C" int blp_lookup_grad_workspace(int type, int64_t n, int64_t rows, int k, int64_t* bytes) {
  int rc = check_args(type, n, rows, k);
  if (rc) return rc;
  BLP_CHECK(bytes, BLP_E_ARG, "lookup: null pointer");
  *bytes = plan_of(type, n, rows, k).bytes;
  return 0;
}

extern "C" int blp_lookup_grad(int device, void* stream, int type, const void* grad, int64_t ldg, const void* ids, int ids64,
                               int64_t n, int64_t rows, int k, float scale, void* out, int64_t ldo, int add, void* ws,
                               int64_t ws_bytes) {
  int rc = check_args(type, n, rows, k);
  if (rc) return rc;
  BLP_CHECK(out && ws && (n == 0 || (grad && ids)), BLP_E_ARG, "lookup: null pointer");
  BLP_CHECK((n == 0 || ldg >= k) && ldo >= k, BLP_E_ARG, "lookup: a row stride is smaller than k");
  const Plan p = plan_of(type, n, rows, k);
  BLP_CHECK(ws_bytes >= p.bytes, BLP_E_ARG, "lookup: the workspace is too small (blp_lookup_grad_workspace)");
  BLP_CHECK(((uintptr_t)ws & 255) == 0, BLP_E_ARG, "lookup: the workspace must be 256-byte aligned");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  const Ids at = {ids, ids64, rows};
  hipStream_t st = (hipStream_t)stream;
  if (type == F32) return lookup_grad<F32>(st, p, grad, ldg, at, n, k, scale, out, ldo, add, (char*)ws);
  if (type == BF16) return lookup_grad<BF16>(st, p, grad, ldg, at, n, k, scale, out, ldo, add, (char*)ws);
  return lookup_grad<F16>(st, p, grad, ldg, at, n, k, scale, out, ldo, add, (char*)ws);
}
