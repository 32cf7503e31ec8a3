// Rows of a factor table by id, scaled, and the gradient of that (blp_lookup*).
//
//   y_i = scale table[id_i] (an id outside the table: zeros)      dT_r = scale sum_{i : id_i = r} dy_i
//
// The gradient is a sum over each row's positions, in an order that is the same every time, with no float atomics: the ids
// are sorted (stable, with their positions), chunks of up to 64 sorted entries are summed in ascending order and 32 bits by one
// group of lanes each, a row's sum that lies inside a chunk is written at once and one that crosses chunks is left as
// partial sums, which a second kernel adds up in 64 bits: in the chunks' order, or, for rows of more than 8 chunks, those of
// each group of lanes in turn, then the groups'. Every row of dy is read once, every row of dT written once.
#include <algorithm>
#include <type_traits>

#include "blp_internal.h"
#include "latent.h"

namespace {

using namespace blp::tile;
using blp::DeviceGuard;
using blp::div_up;
using blp::up;
using namespace blp::rows;
using blp::FastDiv;
using blp::Ids;

// ---------------------------------------------------------------- lookup
// One vector a thread, four in flight: bound by memory. 2 M ids x 64 bf16 out of 1 M rows: 97 us; 0.34 GB have to move
// (3.5 TB/s), 0.53 GB do with the rows read more than once.
// `n` rows with n * per < 2^31 (the host takes longer lists in parts).
template <int T>
__global__ __launch_bounds__(256) void k_lookup(const char* __restrict__ table, int64_t ld, Ids ids, int64_t i0, uint32_t n,
                                                int k, FastDiv per, float scale, char* __restrict__ out, int64_t ldo) {
  constexpr int NE = Vec<T>::NE, U = 4;
  const uint32_t total = n * per.d, step = gridDim.x * blockDim.x;
  for (uint32_t at = blockIdx.x * blockDim.x + threadIdx.x; at < total; at += step * U) {
    Vec<T> v[U];
    int64_t id[U];
    uint32_t row[U], e0[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = at + u * step;
      row[u] = per(min(i, total - 1));
      e0[u] = (min(i, total - 1) - row[u] * per.d) * NE;
      id[u] = ids(i0 + row[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = Vec<T>{};
      if (id[u] >= 0) v[u] = load_vec<T>(table + id[u] * ld + (int64_t)e0[u] * size_of(T), k - (int)e0[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + u * step < total) {
#pragma unroll
        for (int j = 0; j < NE / 4; ++j) v[u].v[j] *= scale;
        store_vec<T>(out + (i0 + row[u]) * ldo + (int64_t)e0[u] * size_of(T), k - (int)e0[u], v[u]);
      }
  }
}

// ---------------------------------------------------------------- sort
// Stable radix sort of (id, position), least significant digit first, BITS (9 or 10) bits a pass. A block takes
// 512 ROUNDS consecutive entries; wave w of it the w-th eighth, 64 at a time in order. The entries of one
// digit are found with ballots (a lane's rank among them by counting the lanes below), so ranks follow
// positions; ids outside the table get the largest key and end up last. 1 M ids of 100,000 rows, two passes: counts 2 x 5 us,
// sums 2 x 5 us, entries 2 x 11 us (8 MB in, 8 MB out in scattered entries; keys and positions apart: 17 us).
constexpr int SORT_WAVES = 8, SORT_THREADS = 64 * SORT_WAVES, MOST_BITS = 10;

struct Entry {  // eight bytes together: a scattered entry is one write
  uint32_t key, pos;
};

__device__ inline uint32_t key_at(const Ids& ids, const Entry* in, int64_t i) {
  if (in) return in[i].key;
  const int64_t id = ids(i);
  return id >= 0 ? (uint32_t)id : (uint32_t)ids.rows;
}

// counts[block][digit]
template <int ROUNDS, int BITS>
__global__ __launch_bounds__(SORT_THREADS) void k_digit_counts(Ids ids, const Entry* __restrict__ in, int64_t n, int shift,
                                                               uint32_t* __restrict__ counts) {
  constexpr int BINS = 1 << BITS;
  __shared__ uint32_t s_count[BINS];
  for (int i = threadIdx.x; i < BINS; i += SORT_THREADS) s_count[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ROUNDS);
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = base + r * SORT_THREADS + threadIdx.x;
    if (i < n) atomicAdd(&s_count[(key_at(ids, in, i) >> shift) & (BINS - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += SORT_THREADS) counts[(int64_t)blockIdx.x * BINS + i] = s_count[i];
}

// 16 digits a block, 64 threads each over the blocks' rows: counts become exclusive sums over the blocks; total[digit].
template <int BITS>
__global__ __launch_bounds__(1024) void k_digit_sums(uint32_t* __restrict__ counts, int blocks, uint32_t* __restrict__ total) {
  constexpr int BINS = 1 << BITS;
  __shared__ uint32_t s_sum[64][17];
  const int c = threadIdx.x & 15, w = threadIdx.x >> 4, d = blockIdx.x * 16 + c;
  const int per = (blocks + 63) / 64, b0 = min(blocks, w * per), b1 = min(blocks, b0 + per);
  uint32_t sum = 0;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) sum += counts[(int64_t)b * BINS + d];
  s_sum[w][c] = sum;
  __syncthreads();
  if (threadIdx.x < 512) {  // a wave scans two digits' 64 sums, one after the other
    const int lane = threadIdx.x & 63, v = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t x = s_sum[lane][v * 2 + k];
      uint32_t s = x;
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t t = __shfl_up(s, o, 64);
        if (lane >= o) s += t;
      }
      s_sum[lane][v * 2 + k] = s - x;
      if (lane == 63) total[blockIdx.x * 16 + v * 2 + k] = s;
    }
  }
  __syncthreads();
  uint32_t run = s_sum[w][c];
#pragma unroll 8
  for (int b = b0; b < b1; ++b) {
    const uint32_t x = counts[(int64_t)b * BINS + d];
    counts[(int64_t)b * BINS + d] = run;
    run += x;
  }
}

template <int ROUNDS, int BITS>
__global__ __launch_bounds__(SORT_THREADS) void k_scatter(Ids ids, const Entry* __restrict__ in, int64_t n, int shift,
                                                          const uint32_t* __restrict__ counts,
                                                          const uint32_t* __restrict__ total, Entry* __restrict__ out) {
  constexpr int BINS = 1 << BITS;
  __shared__ uint32_t s_base[BINS];
  __shared__ uint16_t s_wave[SORT_WAVES][BINS];
  __shared__ uint32_t s_sum[SORT_WAVES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ROUNDS) + w * (64 * ROUNDS);
  Entry entry[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = min(base + r * 64 + lane, n - 1);
    entry[r] = in ? in[i] : Entry{key_at(ids, nullptr, i), (uint32_t)i};
  }
  for (int i = threadIdx.x; i < SORT_WAVES * BINS / 2; i += SORT_THREADS) reinterpret_cast<uint32_t*>(&s_wave[0][0])[i] = 0;
  // where each digit starts: exclusive sums of the totals, BINS / 512 digits a thread
  uint32_t c[BINS / SORT_THREADS], sum = 0;
#pragma unroll
  for (int j = 0; j < BINS / SORT_THREADS; ++j) {
    c[j] = sum;
    sum += total[threadIdx.x * (BINS / SORT_THREADS) + j];
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
  for (int j = 0; j < BINS / SORT_THREADS; ++j) {
    const int d = threadIdx.x * (BINS / SORT_THREADS) + j;
    s_base[d] = before + c[j] + counts[(int64_t)blockIdx.x * BINS + d];
  }
  // ranks within the wave
  uint16_t rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool ok = base + r * 64 + lane < n;
    const uint32_t d = (entry[r].key >> shift) & (BINS - 1);
    unsigned long long same = __ballot(ok);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
      const unsigned long long m = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? m : ~m;
    }
    const int below = __popcll(same & ((1ull << lane) - 1));
    if (ok) rank[r] = (uint16_t)(s_wave[w][d] + below);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (ok && below == 0) s_wave[w][d] += (uint16_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < BINS / SORT_THREADS; ++j) {  // the waves' counts become exclusive sums over the waves
    const int d = threadIdx.x * (BINS / SORT_THREADS) + j;
    uint32_t run = 0;
    for (int i = 0; i < SORT_WAVES; ++i) {
      const uint32_t t = s_wave[i][d];
      s_wave[i][d] = (uint16_t)run;
      run += t;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (base + r * 64 + lane < n) {
      const uint32_t d = (entry[r].key >> shift) & (BINS - 1);
      out[s_base[d] + s_wave[w][d] + rank[r]] = entry[r];
    }
  }
}

// Up to SMALL entries, in one launch: an entry's place is the number of entries with a smaller key, or with the same key
// before it. Every block has all keys in LDS; a wave places EACH entries, its lanes passing over the keys by vectors.
// n^2 comparisons: 2,000 entries take 6 us and 8,192 take 13, where the radix passes' six launches take 20 and more.
constexpr int SMALL = 8192, EACH = 4, PLACED = 8 * EACH;
__global__ __launch_bounds__(512) void k_place_small(Ids ids, int n, Entry* __restrict__ out) {
  extern __shared__ uint4 s_key[];  // n rounded up to 16, the rest the largest key
  uint32_t* const word = reinterpret_cast<uint32_t*>(s_key);
  const int quads = (n + 15) / 16 * 4;
  for (int i = threadIdx.x; i < quads * 4; i += 512) word[i] = i < n ? key_at(ids, nullptr, i) : 0xffffffffu;
  __syncthreads();
  const int lane = threadIdx.x & 63, first = blockIdx.x * PLACED + (threadIdx.x >> 6) * EACH;
  if (first >= n) return;
  uint32_t key[EACH];
  int place[EACH];
#pragma unroll
  for (int u = 0; u < EACH; ++u) {  // first is a multiple of four: the entries lie in one vector
    key[u] = word[first + u];
    place[u] = lane < u && word[first + lane] == key[u];  // within the vector
  }
#pragma unroll 2
  for (int q = lane; q < quads; q += 64) {
    const uint4 v = s_key[q];
    const uint32_t same = q < (first >> 2);  // before the entries the same key counts, too
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const uint32_t below = key[u] + same;
      place[u] += (v.x < below) + (v.y < below) + (v.z < below) + (v.w < below);
    }
  }
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) place[u] += __shfl_xor(place[u], o, 64);
    if (lane == u && first + u < n) out[place[u]] = Entry{key[u], (uint32_t)(first + u)};
  }
}

// ---------------------------------------------------------------- sums
constexpr int HEAVY = 8;  // chunks: a row that crosses more of them is added up by a whole block

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

struct Sums {
  const Entry* in;           // sorted
  int64_t n, chunk, chunks;  // entries, entries a chunk
  uint32_t rows;
  int k, lanes;              // lanes of a chunk: a power of two up to 64; blockIdx.y: their column tile
  float scale;
  char* out;
  int64_t ldo;
  int add;
  float* part;
  int64_t kv;  // floats of a partial sum
};

// Bound by reading dy, in whole rows but in sorted order: 1 M x 64 float32 0.28 GB in 60 us, 4.7
// TB/s; 16,384 x 1,024 bf16 0.09 GB in 20 us.
// The first `clear_blocks` blocks clear the rows without ids: 64 rows a wave, whose entries it looks up, 64 probes at
// a time.
template <int T>
__device__ void clear_rows(const Sums& a, int64_t wave) {
  const int lane = threadIdx.x & 63;
  const int64_t r0 = wave * 64;
  if (r0 >= a.rows) return;
  int64_t lo[2] = {0, 0}, hi[2] = {a.n, a.n};  // the first entries of row r0 and of row r0 + 64
  while (lo[0] < hi[0] || lo[1] < hi[1]) {
    unsigned long long less[2];
    int64_t step[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      step[i] = (hi[i] - lo[i] + 63) >> 6;
      const int64_t at = lo[i] + lane * step[i];
      less[i] = __ballot(at < hi[i] && a.in[at].key < (uint32_t)(r0 + i * 64));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = __popcll(less[i]);
      hi[i] = min(hi[i], lo[i] + c * step[i]);
      if (c) lo[i] += (c - 1) * step[i] + 1;
    }
  }
  uint32_t low = 0, high = 0;  // which of the 64 rows have entries
  if (lo[1] - lo[0] <= 512) {
    for (int64_t i = lo[0] + lane; i < lo[1]; i += 64) {
      const uint32_t r = a.in[i].key - (uint32_t)r0;
      (r < 32 ? low : high) |= 1u << (r & 31);
    }
    for (int o = 1; o < 64; o <<= 1) {
      low |= __shfl_xor(low, o, 64);
      high |= __shfl_xor(high, o, 64);
    }
  } else {
    const uint32_t r = (uint32_t)(r0 + lane);
    int64_t first = lo[0], end = lo[1];
    while (first < end) {
      const int64_t mid = (first + end) >> 1;
      if (a.in[mid].key < r)
        first = mid + 1;
      else
        end = mid;
    }
    const unsigned long long there = __ballot(first < lo[1] && a.in[first].key == r);
    low = (uint32_t)there;
    high = (uint32_t)(there >> 32);
  }
  unsigned long long left = ~((unsigned long long)high << 32 | low);
  if (a.rows - r0 < 64) left &= (1ull << (a.rows - r0)) - 1;
  const int vecs = (a.k + Vec<T>::NE - 1) / Vec<T>::NE;
  // short rows: several at a time
  const int each = a.lanes, groups = 64 / each, l = lane & (each - 1);
  char* at = a.out + (r0 + lane / each) * a.ldo;
  left >>= lane / each;
  for (int r = 0; r < 64; r += groups, at += groups * a.ldo, left >>= groups & 63)
    if (left & 1)
      for (int v = l; v < vecs; v += each) store_vec<T>(at + (int64_t)v * 16, a.k - v * Vec<T>::NE, Vec<T>{});
}

template <int T>
__global__ __launch_bounds__(256) void k_chunk_sums(Sums a, const char* __restrict__ dy, int64_t ld, unsigned clear_blocks) {
  constexpr int NE = Vec<T>::NE, U = 8;
  if (blockIdx.x < clear_blocks) {
    if (blockIdx.y == 0) clear_rows<T>(a, blockIdx.x * 4ll + (threadIdx.x >> 6));
    return;
  }
  const int64_t chunk = ((blockIdx.x - clear_blocks) * 256ll + threadIdx.x) / a.lanes;
  const int vec = blockIdx.y * a.lanes + (threadIdx.x & (a.lanes - 1)), e0 = vec * NE, k = a.k;
  const int64_t b = chunk * a.chunk, e = min(a.n, b + a.chunk);
  const uint32_t rows = a.rows;
  if (b >= a.n || e0 >= k) return;
  const char* src = dy + (int64_t)e0 * size_of(T);
  uint32_t cur = a.in[b].key;
  bool head = b > 0 && a.in[b - 1].key == cur;  // the running row began in an earlier chunk
  Vec<T> sum{};
  for (int64_t i = b; i < e; i += U) {
    Entry in[U];
    Vec<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) in[u] = i + u < e ? a.in[i + u] : Entry{rows, 0};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = Vec<T>{};
      if (in[u].key < rows) v[u] = load_vec<T>(src + (int64_t)in[u].pos * ld, k - e0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < e && in[u].key != cur) {  // `cur` ended before this entry
        if (cur < rows) {
          if (head)
            put_part<T>(a.part, 2 * chunk, a.kv, vec, sum);
          else
            put<T>(a.out, a.ldo, cur, e0, k, sum, a.scale, a.add);
        }
        head = false;
        cur = in[u].key;
        sum = Vec<T>{};
      }
#pragma unroll
      for (int j = 0; j < NE / 4; ++j) sum.v[j] += v[u].v[j];
    }
  }
  if (cur >= rows) return;
  const bool goes_on = e < a.n && a.in[e].key == cur;
  if (head)
    put_part<T>(a.part, 2 * chunk, a.kv, vec, sum);
  else if (goes_on)
    put_part<T>(a.part, 2 * chunk + 1, a.kv, vec, sum);
  else
    put<T>(a.out, a.ldo, cur, e0, k, sum, a.scale, a.add);
}

// Whether a row begins in `chunk` and goes on in the next (a chunk's last row, so at most one), and whether it is heavy.
enum Crossing { NONE, LIGHT, HEAVY_ROW };
__device__ inline Crossing crossing(const Sums& a, int64_t chunk, uint32_t* key) {
  const int64_t b = chunk * a.chunk, e = b + a.chunk, far = (chunk + HEAVY + 1) * a.chunk;
  if (e >= a.n) return NONE;
  const uint32_t last = a.in[e - 1].key, next = a.in[e].key, first = a.in[b].key, before = a.in[max(b - 1, (int64_t)0)].key,
                 away = a.in[min(far, a.n - 1)].key;  // one wait for all five
  *key = last;
  if (last >= a.rows || next != last || (b > 0 && first == last && before == last)) return NONE;
  return far < a.n && away == last ? HEAVY_ROW : LIGHT;
}

// The rows that cross chunks, in 64 bits. The first blocks, which last longest: HEAVY chunks each, in which one heavy row
// can begin; its partial sums go to the groups of lanes in turn, then the groups' sums are added in order. The
// others: a group of lanes a chunk, the partial sums of the row that begins there in the chunks' order. 13 us in the case
// above: six or seven waits for memory, one after the other.
template <int T>
__global__ __launch_bounds__(256) void k_join_chunks(Sums a, unsigned heavy_blocks) {
  constexpr int NE = Vec<T>::NE, U = 4;
  __shared__ double s_sum[256 * NE];
  __shared__ int s_at;
  __shared__ uint32_t s_key;
  const int groups = 256 / a.lanes, g = threadIdx.x / a.lanes, l = threadIdx.x & (a.lanes - 1);
  const int vec = blockIdx.y * a.lanes + l, e0 = vec * NE;
  double sum[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) sum[j] = 0.0;
  uint32_t key;
  if (blockIdx.x >= heavy_blocks) {
    const int64_t chunk = (int64_t)(blockIdx.x - heavy_blocks) * groups + g;
    if (chunk >= a.chunks || e0 >= a.k || crossing(a, chunk, &key) != LIGHT) return;
    bool more = true;
    for (int64_t c = chunk; more; c += U) {  // U chunks' loads at a time, their keys' beside their sums'
      bool mine[U];
      f32x4 v[U][NE / 4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = min(c + u, a.chunks - 1);
        mine[u] = c + u == chunk || (c + u < a.chunks && a.in[at * a.chunk].key == key);
        const f32x4* part = reinterpret_cast<const f32x4*>(a.part + (2 * at + (at == chunk ? 1 : 0)) * a.kv + (int64_t)e0);
#pragma unroll
        for (int j = 0; j < NE / 4; ++j) v[u][j] = part[j];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        more = more && mine[u];
#pragma unroll
        for (int j = 0; j < NE; ++j) sum[j] += more ? (double)v[u][j >> 2][j & 3] : 0.0;
      }
    }
    Vec<T> r;
#pragma unroll
    for (int j = 0; j < NE; ++j) r.v[j >> 2][j & 3] = (float)sum[j];
    put<T>(a.out, a.ldo, key, e0, a.k, r, a.scale, a.add);
    return;
  }
  if (threadIdx.x == 0) s_at = -1;
  __syncthreads();
  const int64_t first = blockIdx.x * (int64_t)HEAVY;
  if (threadIdx.x < HEAVY && first + threadIdx.x < a.chunks && crossing(a, first + threadIdx.x, &key) == HEAVY_ROW) {
    s_at = threadIdx.x;
    s_key = key;
  }
  __syncthreads();
  if (s_at < 0) return;
  const int64_t chunk = first + s_at;
  key = s_key;
  int64_t lo = chunk + 1, hi = a.chunks;  // the first chunk that does not begin with the row: 256 probes at a time
  while (lo < hi) {
    const int64_t step = (hi - lo + 255) >> 8, at = lo + threadIdx.x * step;
    const int begin = __syncthreads_count(at < hi && a.in[at * a.chunk].key == key);
    if (begin == 0) break;
    hi = min(hi, lo + begin * step);
    lo += (begin - 1) * step + 1;
  }
  if (e0 < a.k) {
#pragma unroll 8
    for (int64_t c = chunk + g; c < lo; c += groups) {
      const f32x4* at = reinterpret_cast<const f32x4*>(a.part + (2 * c + (c == chunk ? 1 : 0)) * a.kv + (int64_t)e0);
#pragma unroll
      for (int j = 0; j < NE; ++j) sum[j] += (double)at[j >> 2][j & 3];
    }
  }
#pragma unroll
  for (int j = 0; j < NE; ++j) s_sum[j * 256 + threadIdx.x] = sum[j];
  __syncthreads();
  if (g == 0 && e0 < a.k) {
    Vec<T> r;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      for (int i = 1; i < groups; ++i) sum[j] += s_sum[j * 256 + i * a.lanes + l];
      r.v[j >> 2][j & 3] = (float)sum[j];
    }
    put<T>(a.out, a.ldo, key, e0, a.k, r, a.scale, a.add);
  }
}

// ---------------------------------------------------------------- host side
struct Plan {
  int passes, bits, rounds, lanes, tiles;
  int64_t blocks, chunk, chunks, kv;
  int64_t o_in[2], o_counts, o_total, o_part, bytes;
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
  p.passes = n <= SMALL ? 0 : (int)div_up(bits, MOST_BITS);
  p.bits = p.passes * 9 >= bits ? 9 : 10;
  p.rounds = n <= 128 * 1024 ? 1 : 4;  // short lists: more blocks, each done sooner
  p.blocks = div_up(n, SORT_THREADS * p.rounds);
  const int64_t vecs = div_up(k, 16 / size_of(type));
  p.lanes = 1;
  while (p.lanes < 64 && p.lanes < vecs) p.lanes <<= 1;
  p.tiles = (int)div_up(vecs, p.lanes);
  // chunks: long enough that partial sums stay few, short enough for 16 waves a compute unit
  p.chunk = 64;
  while (p.chunk > 8 && div_up(n, p.chunk) * p.lanes * p.tiles / 64 < 4096) p.chunk >>= 1;
  p.chunks = div_up(n, p.chunk);
  p.kv = up(k, 16 / size_of(type));
  for (int i = 0; i < 2; ++i) p.o_in[i] = take(8 * n);
  p.o_counts = take(p.passes ? (4ll << p.bits) * p.blocks : 0);
  p.o_total = take(4 << MOST_BITS);
  p.o_part = take(8 * p.chunks * p.kv);
  p.bytes = std::max<int64_t>(at, 256);
  return p;
}

template <int T>
int lookup(hipStream_t st, const void* table, int64_t ld, Ids ids, int64_t n, int k, float scale, void* out, int64_t ldo) {
  const FastDiv per((uint32_t)div_up(k, 16 / size_of(T)));
  const int64_t most = 0x40000000 / per.d;
  for (int64_t i0 = 0; i0 < n; i0 += most) {
    const uint32_t m = (uint32_t)std::min(most, n - i0);
    const unsigned grid = (unsigned)std::min<int64_t>(div_up((int64_t)m * per.d, 1024), 1 << 18);
    k_lookup<T><<<grid, 256, 0, st>>>((const char*)table, ld * size_of(T), ids, i0, m, k, per, scale, (char*)out,
                                      ldo * size_of(T));
    BLP_HIP(hipGetLastError());
  }
  return 0;
}

template <int ROUNDS, int BITS>
int sort(hipStream_t st, const Plan& p, Ids ids, int64_t n, Entry* const* sorted, uint32_t* counts, uint32_t* total, int* last) {
  int cur = 0;
  for (int s = 0; s < p.passes; ++s) {
    const Entry* in = s ? sorted[cur] : nullptr;
    const int to = s ? cur ^ 1 : 0;
    k_digit_counts<ROUNDS, BITS><<<(unsigned)p.blocks, SORT_THREADS, 0, st>>>(ids, in, n, s * BITS, counts);
    BLP_HIP(hipGetLastError());
    k_digit_sums<BITS><<<(1 << BITS) / 16, 1024, 0, st>>>(counts, (int)p.blocks, total);
    BLP_HIP(hipGetLastError());
    k_scatter<ROUNDS, BITS><<<(unsigned)p.blocks, SORT_THREADS, 0, st>>>(ids, in, n, s * BITS, counts, total, sorted[to]);
    BLP_HIP(hipGetLastError());
    cur = to;
  }
  *last = cur;
  return 0;
}

template <int T>
int lookup_grad(hipStream_t st, const Plan& p, const void* dy, int64_t ld, Ids ids, int64_t n, int k, float scale, void* out,
                int64_t ldo, int add, char* ws) {
  const int ES = size_of(T);
  Entry* sorted[2] = {(Entry*)(ws + p.o_in[0]), (Entry*)(ws + p.o_in[1])};
  uint32_t *counts = (uint32_t*)(ws + p.o_counts), *total = (uint32_t*)(ws + p.o_total);
  int cur = 0, rc = 0;
  if (p.passes == 0) {
    if (n > 0) k_place_small<<<(unsigned)div_up(n, PLACED), 512, up(n, 16) * 4, st>>>(ids, (int)n, sorted[0]);
    BLP_HIP(hipGetLastError());
  } else {
    auto run = [&](auto rounds, auto bits) {
      return sort<decltype(rounds)::value, decltype(bits)::value>(st, p, ids, n, sorted, counts, total, &cur);
    };
    using std::integral_constant;
    if (p.rounds == 1)
      rc = p.bits == 9 ? run(integral_constant<int, 1>{}, integral_constant<int, 9>{}) : run(integral_constant<int, 1>{}, integral_constant<int, 10>{});
    else
      rc = p.bits == 9 ? run(integral_constant<int, 4>{}, integral_constant<int, 9>{}) : run(integral_constant<int, 4>{}, integral_constant<int, 10>{});
    if (rc) return rc;
  }
  const Sums a = {sorted[cur], n, p.chunk, p.chunks, (uint32_t)ids.rows, k, p.lanes, scale, (char*)out, ldo * ES, add,
                  (float*)(ws + p.o_part), p.kv};
  const unsigned sum_blocks = (unsigned)div_up(p.chunks * p.lanes, 256), clear_blocks = add ? 0 : (unsigned)div_up(ids.rows, 256);
  if (sum_blocks + clear_blocks == 0) return 0;
  k_chunk_sums<T><<<dim3(sum_blocks + clear_blocks, p.tiles), 256, 0, st>>>(a, (const char*)dy, ld * ES, clear_blocks);
  BLP_HIP(hipGetLastError());
  if (p.chunks > 1) {
    const unsigned light = (unsigned)div_up(p.chunks, 256 / p.lanes), heavies = (unsigned)div_up(p.chunks, HEAVY);
    k_join_chunks<T><<<dim3(light + heavies, p.tiles), 256, 0, st>>>(a, heavies);
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
  BLP_CHECK(fabsf(scale) <= 3.4028235e38f, BLP_E_ARG, "lookup: scale must be finite");
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
  BLP_CHECK(fabsf(scale) <= 3.4028235e38f, BLP_E_ARG, "lookup: scale must be finite");
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
