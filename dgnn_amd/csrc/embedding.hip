// Node (token) embedding: lookup with scaling, and the gradient of the table by sorted ids.
//
//   out_i = scale * table[id_i],   dtable_r = scale * sum over i with id_i = r of grad_i
//
// An id outside [0, rows) names no row: zeros out, no gradient.  Both directions are bound by memory.
// The gradient sorts (id, i) with a stable radix sort, eight bits a pass, so that every row of the
// table is written exactly once, by the sum of its own run in ascending i: no atomics on floats, no
// zeroed table, the same bits every time.  Runs that cross the borders of fixed pieces (all long ones:
// frequent tokens, hub nodes) are summed a piece at a time first.
#include "common.hpp"

using namespace dgnn;

namespace dgnn {

typedef _Float16 half_t;
typedef __bf16 bf16_t;

// N elements of a row in one access of N * sizeof(T) bytes
template <class T, int N>
struct __align__(sizeof(T) * N) Pack {
  T v[N];
};

// PAST: around the caches (accesses of 16 bytes)
template <bool PAST, class T, int N>
__device__ __forceinline__ void store_pack(T *to, const Pack<T, N> &p) {
  if constexpr (PAST) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 v;
    __builtin_memcpy(&v, &p, 16);
    __builtin_nontemporal_store(v, (u32x4 *)to);
  } else {
    *(Pack<T, N> *)to = p;
  }
}

template <class I>
__device__ __forceinline__ int row_of_id(const I *ids, long long i, int rows) {
  const I x = ids[i];
  return x >= 0 && x < (I)rows ? (int)x : rows;           // rows: names none
}

// lanes = threads that share a row (a power of two up to 256).  65536 ids of 1024 bfloat16 45 us, 5.9 TB/s; 196611 of
// 100 floats, from 2.4 million rows, 24 - 36 us, 4.4 TB/s and more (a large copy: 5.1).
template <class T, int N, class I>
__global__ __launch_bounds__(DGNN_BLOCK) void k_embed_fwd(int n, int rows, int dim, int lanes, float scale,
                                                          const I *__restrict__ ids, const T *__restrict__ table,
                                                          T *__restrict__ out) {
  const int per = DGNN_BLOCK / lanes;
  const long long i = (long long)group_in_rows() * per + threadIdx.x / lanes;
  if (i >= n) return;
  const int r = row_of_id(ids, i, rows);
  for (int c = (threadIdx.x & (lanes - 1)) * N; c < dim; c += lanes * N) {
    Pack<T, N> p;
    if (r < rows) {
      p = *(const Pack<T, N> *)(table + (long long)r * dim + c);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        // a float product, then the type: left alone the compiler merges both into v_fma_mixlo_f16, whose
        // single rounding differs from float16's table * scale in the last place now and then
        float y = (float)p.v[j] * scale;
        asm("" : "+v"(y));
        p.v[j] = (T)y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) p.v[j] = (T)0.f;
    }
    *(Pack<T, N> *)(out + i * dim + c) = p;
  }
}

// ------------------------------------------------------------------ stable radix sort of (row, i)
constexpr int SORT_TILE = 1024, SORT_BINS = 256, SORT_SMALL = 8192;
static inline int sort_tiles(int n) { return (n + SORT_TILE - 1) / SORT_TILE; }

template <class I>
struct SortSrc {                       // the first pass reads the ids, later ones the previous pass's pairs
  const I *ids;
  const int *key, *val;
  int rows;
  __device__ __forceinline__ int k(int i) const { return ids ? row_of_id(ids, i, rows) : key[i]; }
  __device__ __forceinline__ int v(int i) const { return ids ? i : val[i]; }
};

// counts[bin * tiles + tile]
template <class I>
__global__ __launch_bounds__(DGNN_BLOCK) void k_sort_count(int n, int shift, SortSrc<I> src, int *__restrict__ counts) {
  __shared__ int bins[SORT_BINS];
  bins[threadIdx.x] = 0;
  __syncthreads();
  const int lo = blockIdx.x * SORT_TILE, hi = min(n, lo + SORT_TILE);
  for (int i = lo + threadIdx.x; i < hi; i += DGNN_BLOCK) atomicAdd(&bins[(src.k(i) >> shift) & (SORT_BINS - 1)], 1);
  __syncthreads();
  counts[(long long)threadIdx.x * gridDim.x + blockIdx.x] = bins[threadIdx.x];
}

// exclusive prefix over the threads of a workgroup of WAVES waves; *total gets the sum
template <int WAVES>
__device__ __forceinline__ int block_prefix(int x, int (&part)[16], int *total) {
  const int lane = lane_id(), wave = wave_in_block();
  int incl = x;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const int up = __shfl_up(incl, w, 64);
    if (lane >= w) incl += up;
  }
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += part[w];
    all += part[w];
  }
  __syncthreads();
  *total = all;
  return before + incl - x;
}

// counts[bin][.] becomes its exclusive prefix over the tiles, totals[bin] the bin's sum; one wave a bin
__global__ __launch_bounds__(DGNN_WAVE) void k_sort_scan(int tiles, int *__restrict__ counts, int *__restrict__ totals) {
  int *x = counts + (long long)blockIdx.x * tiles;
  const int lane = lane_id();
  int carry = 0;
  for (int base = 0; base < tiles; base += 4 * DGNN_WAVE) {
    int v[4], s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = base + lane * 4 + j;
      v[j] = i < tiles ? x[i] : 0;
      s += v[j];
    }
    int incl = s;
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) {
      const int up = __shfl_up(incl, w, 64);
      if (lane >= w) incl += up;
    }
    int run = carry + incl - s;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = base + lane * 4 + j;
      if (i < tiles) x[i] = run;
      run += v[j];
    }
    carry += __shfl(incl, 63, 64);
  }
  if (lane == 0) totals[blockIdx.x] = carry;
}

// Lanes of the wave whose digit equals this lane's (of the lanes that take part).
__device__ __forceinline__ unsigned long long same_digit(int digit, bool on) {
  unsigned long long same = __ballot(on);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const unsigned long long set = __ballot((digit >> b) & 1);
    same &= (digit >> b) & 1 ? set : ~set;
  }
  return same;
}

// The whole sort of up to SORT_SMALL ids in one workgroup, since launches are most of a small sort's time (the whole
// gradient of 2708 rows of 64: 2048 ids 19 us, with three launches a pass 28; 8192 ids 29 and 31): every wave
// owns 512 consecutive positions; a pass counts the wave's digits, turns the counts into first positions
// (digit, then wave) and moves the pairs within LDS in order.
template <class I>
__global__ __launch_bounds__(1024) void k_sort_small(int n, int rows, int passes, const I *__restrict__ ids,
                                                     int *__restrict__ key, int *__restrict__ val) {
  constexpr int WAVES = 16, PART = SORT_SMALL / WAVES;
  __shared__ int at[WAVES][SORT_BINS], ks[2][SORT_SMALL], vs[2][SORT_SMALL], part[16];
  const int lane = lane_id(), wave = wave_in_block();
  for (int i = threadIdx.x; i < n; i += 1024) ks[0][i] = row_of_id(ids, i, rows), vs[0][i] = i;
  for (int p = 0; p < passes; ++p) {
    const int *ki = ks[p & 1], *vi = vs[p & 1];
    int *ko = ks[(p + 1) & 1], *vo = vs[(p + 1) & 1];
    const int shift = 8 * p, lo = wave * PART, hi = min(n, lo + PART);
    for (int i = threadIdx.x; i < WAVES * SORT_BINS; i += 1024) ((int *)at)[i] = 0;
    __syncthreads();
    for (int i = lo + lane; i < hi; i += DGNN_WAVE) atomicAdd(&at[wave][(ki[i] >> shift) & (SORT_BINS - 1)], 1);
    __syncthreads();
    int c[4], s = 0, all;                       // thread t: digit t / 4, waves 4 (t % 4) ..
    const int digit = threadIdx.x >> 2, w0 = 4 * (threadIdx.x & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = at[w0 + j][digit], s += c[j];
    int run = block_prefix<WAVES>(s, part, &all);
#pragma unroll
    for (int j = 0; j < 4; ++j) at[w0 + j][digit] = run, run += c[j];
    __syncthreads();
    for (int base = lo; base < hi; base += DGNN_WAVE) {
      const int i = base + lane;
      const bool on = i < hi;
      const int k = on ? ki[i] : 0, d = (k >> shift) & (SORT_BINS - 1);
      const unsigned long long same = same_digit(d, on);
      const int rank = __popcll(same & ((1ULL << lane) - 1));
      const int to = on ? at[wave][d] + rank : 0;
      wave_lds_sync();
      if (on && rank == 0) at[wave][d] += __popcll(same);
      wave_lds_sync();
      if (on) ko[to] = k, vo[to] = vi[i];
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += 1024) key[i] = ks[passes & 1][i], val[i] = vs[passes & 1][i];
}

// Every wave owns a quarter of the tile; it counts its digits, then walks it again in order: the rank
// of a key among the 64 of a step is the number of lower lanes with its digit.
template <class I>
__global__ __launch_bounds__(DGNN_BLOCK) void k_sort_scatter(int n, int shift, SortSrc<I> src,
                                                             const int *__restrict__ offs, const int *__restrict__ totals,
                                                             int *__restrict__ key, int *__restrict__ val) {
  __shared__ int at[DGNN_WAVES_PER_BLOCK][SORT_BINS], part[16];
  const int lane = lane_id(), wave = wave_in_block();
  for (int w = 0; w < DGNN_WAVES_PER_BLOCK; ++w) at[w][threadIdx.x] = 0;
  __syncthreads();
  constexpr int PART = SORT_TILE / DGNN_WAVES_PER_BLOCK;
  const int lo = blockIdx.x * SORT_TILE + wave * PART, hi = min(n, lo + PART);
  for (int i = lo + lane; i < hi; i += DGNN_WAVE) atomicAdd(&at[wave][(src.k(i) >> shift) & (SORT_BINS - 1)], 1);
  __syncthreads();
  int all, run = offs[(long long)threadIdx.x * gridDim.x + blockIdx.x];
  run += block_prefix<DGNN_WAVES_PER_BLOCK>(totals[threadIdx.x], part, &all);      // the smaller digits
  for (int w = 0; w < DGNN_WAVES_PER_BLOCK; ++w) {
    const int c = at[w][threadIdx.x];
    at[w][threadIdx.x] = run;
    run += c;
  }
  __syncthreads();
  for (int base = lo; base < hi; base += DGNN_WAVE) {
    const int i = base + lane;
    const bool on = i < hi;
    const int k = on ? src.k(i) : 0, digit = (k >> shift) & (SORT_BINS - 1);
    const unsigned long long same = same_digit(digit, on);
    const int rank = __popcll(same & ((1ULL << lane) - 1)), count = __popcll(same);
    const int to = on ? at[wave][digit] + rank : 0;
    wave_lds_sync();
    if (on && rank == 0) at[wave][digit] += count;
    wave_lds_sync();
    if (on) {
      key[to] = k;
      val[to] = src.v(i);
    }
  }
}

// ------------------------------------------------------------------ sums of the runs
__device__ __forceinline__ int first_not_below(const int *__restrict__ key, int lo, int hi, int k) {
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (key[mid] < k) lo = mid + 1; else hi = mid;
  }
  return lo;
}
// the same by a whole wave, 64 probes a step
__device__ __forceinline__ int first_not_below_wave(const int *__restrict__ key, int n, int k) {
  int lo = 0, hi = n;                           // the answer lies in [lo, hi]
  const int lane = lane_id();
  while (lo < hi) {
    const int step = (hi - lo + 63) >> 6, i = lo + lane * step;
    const int below = __popcll(__ballot(i < hi && key[i] < k));
    if (below == 0) return lo;
    lo += (below - 1) * step + 1;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

// Sorted positions are cut into pieces of `run`.  A row whose run crosses a border of pieces gets one partial
// sum per piece it touches: slot 2 p when its run holds the first position of piece p, slot 2 p + 1
// when it begins inside (and leaves through the end).  Whether a run crosses shows in the keys next to the
// borders, so nothing is searched.  64 N columns and one piece a workgroup, its positions dealt to four waves.
// 65536 ids of 1024 bfloat16, most of them frequent ones, 28 us (about 4 TB/s); 196611 of 100 floats 14 us,
// waiting for key, position and row one after the other.
template <class T, int N>
__global__ __launch_bounds__(DGNN_BLOCK) void k_embed_cross(int n, int rows, int dim, int run,
                                                            const int *__restrict__ key, const int *__restrict__ val,
                                                            const T *__restrict__ grad, float *__restrict__ part) {
  __shared__ float sums[DGNN_WAVES_PER_BLOCK][DGNN_WAVE * N];
  __shared__ int counts[2];
  const int lane = lane_id(), wave = wave_in_block();
  const int lo = blockIdx.x * run, hi = min(n, lo + run);
  const int c = (blockIdx.y * DGNN_WAVE + lane) * N;
  const int first = key[lo], last = key[hi - 1];
  const bool before = lo > 0 && key[lo - 1] == first, behind = hi < n && key[hi] == last;
  // the run at the front, if it crosses either border, and the one at the end, if it is another and leaves
  const bool front = first < rows && (before || (behind && first == last)), back = last < rows && behind && first != last;
  if (!front && !back) return;
  if (threadIdx.x < 2) counts[threadIdx.x] = 0;
  __syncthreads();
  for (int i = lo + wave * DGNN_WAVE; i < hi; i += DGNN_BLOCK) {
    const int k = i + lane < hi ? key[i + lane] : rows;
    const int f = __popcll(__ballot(k == first)), b = __popcll(__ballot(k == last));
    if (lane == 0) atomicAdd(&counts[0], f), atomicAdd(&counts[1], b);
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    if (!(which == 0 ? front : back)) continue;
    const int a = which == 0 ? lo : hi - counts[1], b = which == 0 ? lo + counts[0] : hi;
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    if (c < dim) {
#pragma unroll 8
      for (int i = a + wave; i < b; i += DGNN_WAVES_PER_BLOCK) {
        const Pack<T, N> p = *(const Pack<T, N> *)(grad + (long long)val[i] * dim + c);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += (float)p.v[j];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) sums[wave][lane * N + j] = acc[j];
    __syncthreads();
    if (wave == 0 && c < dim)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float t = 0.f;
        for (int w = 0; w < DGNN_WAVES_PER_BLOCK; ++w) t += sums[w][lane * N + j];
        part[(2LL * blockIdx.x + which) * dim + c + j] = t;
      }
    __syncthreads();
  }
}

constexpr int EMBED_ROWS = 256;      // most rows of the table a workgroup writes

// A workgroup writes `per_block` consecutive rows.  It finds the sorted positions that name them, marks
// where each row's run begins and ends, stores zeros to the rows without one as one stream of pieces, and
// gives every other row to `lanes` threads.  A table larger than the 256 MB of cache (PAST) is written around it, so
// that keys and gradients stay in: 2.4 million rows of 100 floats, of which few are named, 209 us, 5.1 TB/s
// (around the cache or not: 203 and 231 before the join in double, the whole step 302 and 339 us, since the kernels next to it
// find more there).  50000 rows of 1024 bfloat16 63 us, 3.7 TB/s: the runs there are a few positions long, each a
// wait of its own.
template <class T, int N, bool PAST>
__global__ __launch_bounds__(DGNN_BLOCK) void k_embed_rows(int n, int rows, int dim, int lanes, int per_block, int run, float scale,
                                                           const int *__restrict__ key, const int *__restrict__ val,
                                                           const T *__restrict__ grad, const float *__restrict__ part,
                                                           T *__restrict__ out) {
  __shared__ int begin[EMBED_ROWS], end[EMBED_ROWS], list[EMBED_ROWS], bounds[2], count;
  const int row0 = blockIdx.x * per_block, mine = min(per_block, rows - row0), wave = wave_in_block();
  if (wave < 2) {
    const int at = first_not_below_wave(key, n, wave == 0 ? row0 : row0 + mine);
    if (lane_id() == 0) bounds[wave] = at;
  }
  if ((int)threadIdx.x < EMBED_ROWS) begin[threadIdx.x] = 0, end[threadIdx.x] = 0;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const int p0 = bounds[0], p1 = bounds[1];
  if (p1 - p0 <= 4 * DGNN_BLOCK) {              // few: read them all, a run begins and ends where the key changes
    for (int i = p0 + threadIdx.x; i < p1; i += DGNN_BLOCK) {
      const int k = key[i];
      if (i == p0 || key[i - 1] != k) begin[k - row0] = i;
      if (i == p1 - 1 || key[i + 1] != k) end[k - row0] = i + 1;
    }
  } else if ((int)threadIdx.x < mine) {         // long runs among them: search
    const int a = first_not_below(key, p0, p1, row0 + threadIdx.x);
    const int b = first_not_below(key, a, p1, row0 + threadIdx.x + 1);
    if (b > a) begin[threadIdx.x] = a, end[threadIdx.x] = b;
  }
  __syncthreads();
  if (wave == 0)                                // the rows that have a run, in order
    for (int b = 0; b < mine; b += DGNN_WAVE) {
      const int r = b + lane_id();
      const bool on = r < mine && end[r] > begin[r];
      const unsigned long long set = __ballot(on);
      if (on) list[count + __popcll(set & ((1ULL << lane_id()) - 1))] = r;
      wave_lds_sync();
      if (lane_id() == 0) count += __popcll(set);
      wave_lds_sync();
    }
  __syncthreads();
  const int groups = DGNN_BLOCK / lanes, group = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
  for (int x = group; x < count; x += groups) {
    const int r = list[x], s = begin[r], e = end[r];
    T *to = out + (long long)(row0 + r) * dim;
    for (int c = lane * N; c < dim; c += lanes * N) {
      float acc[N];
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = 0.f;
      if (s / run == (e - 1) / run) {           // inside one piece
#pragma unroll 8
        for (int i = s; i < e; ++i) {
          const Pack<T, N> p = *(const Pack<T, N> *)(grad + (long long)val[i] * dim + c);
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += (float)p.v[j];
        }
      } else {
        // in double: the pieces of a long run are many (4 sqrt(n) of them if one id is all there is), of like size, and
        // each rounding in float would go the same way (2^20 ids, one row, gradients of 0.1: 4e-5 off).  Four at a time are
        // joined in float first: eight doubled rows in flight take the registers of two waves a SIMD (the step of 309 us takes 343)
        const int q0 = s / run, q1 = (e - 1) / run;
        auto at = [&](int q) { return part + (long long)(2 * q + (q == q0 && s != q * run ? 1 : 0)) * dim + c; };
        double sum[N];
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = 0.;
        int q = q0;
        for (; q + 8 <= q1 + 1; q += 8) {
          float four[2][N];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float *src = at(q + x);
#pragma unroll
            for (int j = 0; j < N; ++j) four[x / 4][j] = x % 4 ? four[x / 4][j] + src[j] : src[j];
          }
#pragma unroll
          for (int j = 0; j < N; ++j) sum[j] += (double)four[0][j] + (double)four[1][j];
        }
        for (; q <= q1; ++q) {
          const float *src = at(q);
#pragma unroll
          for (int j = 0; j < N; ++j) sum[j] += (double)src[j];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = (float)sum[j];
      }
      Pack<T, N> p;
#pragma unroll
      for (int j = 0; j < N; ++j) p.v[j] = (T)(acc[j] * scale);
      store_pack<PAST>(to + c, p);
    }
  }
  // last, so that the stores drain while the next workgroup searches
  const int pieces = dim / N;
  for (int u = threadIdx.x; u < mine * pieces; u += DGNN_BLOCK) {
    const int r = u / pieces;
    if (end[r] > begin[r]) continue;
    Pack<T, N> p;
#pragma unroll
    for (int j = 0; j < N; ++j) p.v[j] = (T)0.f;
    store_pack<PAST>(out + (long long)row0 * dim + (long long)u * N, p);
  }
}

// pieces of sqrt(n) / 4 .. sqrt(n) / 2, at least 64: the longest run possible is summed in float over a quarter of a piece
// by each of four waves (a whole piece where a run stays inside one), then in double over 2 .. 4 sqrt(n) pieces
static inline int embed_run(int n) {
  int r = 64;
  while (16LL * r * r < n) r <<= 1;
  return r;
}
static inline size_t align256(size_t x) { return (x + 255) / 256 * 256; }
struct EmbedPlan {
  int passes, run, pieces;
  size_t pairs, counts, part, total;      // bytes
};
static EmbedPlan embed_plan(int n, int rows, int dim) {
  EmbedPlan p;
  int bits = 1;
  while ((1LL << bits) <= (long long)rows) ++bits;           // keys 0 .. rows
  p.passes = (bits + 7) / 8;
  p.run = embed_run(n);
  p.pieces = (n + p.run - 1) / p.run;
  p.pairs = align256(sizeof(int) * (size_t)n);
  p.counts = align256(sizeof(int) * (size_t)SORT_BINS * (sort_tiles(n) + 1));
  p.part = align256(sizeof(float) * 2 * (size_t)p.pieces * dim);
  p.total = 4 * p.pairs + p.counts + p.part;
  return p;
}

// widest access every row's bytes and all pointers allow: 16, 8, 4 or 2 bytes
static int access_bytes(int dim, int size, const void *a, const void *b) {
  const uintptr_t x = (uintptr_t)a | (uintptr_t)b | (uintptr_t)((size_t)dim * size);
  for (int w = 16; w > size; w >>= 1)
    if (x % w == 0) return w;
  return size;
}
static int access_elements(int bytes, int size) {           // as DGNN_EMBED_DISPATCH has it
  return size == 4 || bytes == 16 ? bytes / size : bytes >= 4 ? 2 : 1;
}
static int row_lanes(int dim, int per) {
  int l = 1;
  while (l < DGNN_BLOCK && l * per < dim) l <<= 1;
  return l;
}

template <class T, int N, class I>
static int launch_embed_fwd(int n, int rows, int dim, float scale, const void *ids, const void *table, void *out,
                            hipStream_t st) {
  const int lanes = row_lanes(dim, N), per = DGNN_BLOCK / lanes;
  hipLaunchKernelGGL((k_embed_fwd<T, N, I>), grid_in_rows((n + (long long)per - 1) / per), dim3(DGNN_BLOCK), 0, st, n, rows,
                     dim, lanes, scale, (const I *)ids, (const T *)table, (T *)out);
  DGNN_LAUNCH_CHECK();
  return DGNN_OK;
}
// as many rows a workgroup as make up for its search, but a thousand workgroups where the rows allow it
static int rows_per_block(int rows, int lanes) {
  const int groups = DGNN_BLOCK / lanes, thousandth = (rows + 1023) / 1024;
  const int most = groups * 16 > EMBED_ROWS / 2 ? EMBED_ROWS : groups * 16;
  return most <= thousandth ? most : thousandth > groups ? thousandth : groups;
}
template <class T, int N>
static int launch_embed_sums(int n, int rows, int dim, float scale, const EmbedPlan &p, const int *key, const int *val,
                             const void *grad, float *part, void *out, hipStream_t st) {
  if (n > p.run) {
    hipLaunchKernelGGL((k_embed_cross<T, N>), dim3((unsigned)p.pieces, (unsigned)((dim + DGNN_WAVE * N - 1) / (DGNN_WAVE * N))),
                       dim3(DGNN_BLOCK), 0, st, n, rows, dim, p.run, key, val, (const T *)grad, part);
    DGNN_LAUNCH_CHECK();
  }
  const int lanes = row_lanes(dim, N), per_block = rows_per_block(rows, lanes);
  auto kernel = k_embed_rows<T, N, false>;
  if constexpr (sizeof(T) * N == 16)
    if ((double)rows * dim * sizeof(T) > 256e6) kernel = k_embed_rows<T, N, true>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + (long long)per_block - 1) / per_block)), dim3(DGNN_BLOCK), 0, st, n, rows, dim,
                     lanes, per_block, p.run, scale, key, val, (const T *)grad, (const float *)part, (T *)out);
  DGNN_LAUNCH_CHECK();
  return DGNN_OK;
}
template <class I>
static int sort_ids(int n, int rows, const void *ids, const EmbedPlan &p, char *ws, const int **key, const int **val,
                    hipStream_t st) {
  int *k[2] = {(int *)ws, (int *)(ws + p.pairs)}, *v[2] = {(int *)(ws + 2 * p.pairs), (int *)(ws + 3 * p.pairs)};
  int *counts = (int *)(ws + 4 * p.pairs), *totals = counts + (size_t)SORT_BINS * sort_tiles(n);
  const int tiles = sort_tiles(n);
  if (n <= SORT_SMALL) {
    hipLaunchKernelGGL(k_sort_small<I>, dim3(1), dim3(1024), 0, st, n, rows, p.passes, (const I *)ids, k[0], v[0]);
    DGNN_LAUNCH_CHECK();
    *key = k[0], *val = v[0];
    return DGNN_OK;
  }
  for (int i = 0; i < p.passes; ++i) {
    const SortSrc<I> src = {i == 0 ? (const I *)ids : nullptr, k[(i + 1) & 1], v[(i + 1) & 1], rows};
    hipLaunchKernelGGL(k_sort_count<I>, dim3(tiles), dim3(DGNN_BLOCK), 0, st, n, 8 * i, src, counts);
    DGNN_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_sort_scan, dim3(SORT_BINS), dim3(DGNN_WAVE), 0, st, tiles, counts, totals);
    DGNN_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_sort_scatter<I>, dim3(tiles), dim3(DGNN_BLOCK), 0, st, n, 8 * i, src, (const int *)counts,
                       (const int *)totals, k[i & 1], v[i & 1]);
    DGNN_LAUNCH_CHECK();
  }
  *key = k[(p.passes - 1) & 1];
  *val = v[(p.passes - 1) & 1];
  return DGNN_OK;
}

static int embed_check(int dtype, int idx_bytes, int n, int rows, int dim) {
  if (dtype < 0 || dtype > 2 || (idx_bytes != 4 && idx_bytes != 8) || n < 0 || rows < 0 || dim < 0) return DGNN_ERR_BAD_ARG;
  if (dim > (1 << 30)) return DGNN_ERR_UNSUPPORTED;          // columns and steps past them are ints
  return DGNN_OK;
}
static bool aligned_to(const void *p, int bytes) { return (uintptr_t)p % bytes == 0; }

}  // namespace dgnn

// one call per element type and access width: EXPR may use T (the element) and N (elements an access)
#define DGNN_EMBED_DISPATCH(dtype, bytes, EXPR)                                   \
  do {                                                                            \
    if ((dtype) == DGNN_F32) {                                                    \
      typedef float T;                                                            \
      if ((bytes) == 16) { constexpr int N = 4; return EXPR; }                    \
      if ((bytes) == 8) { constexpr int N = 2; return EXPR; }                     \
      { constexpr int N = 1; return EXPR; }                                       \
    }                                                                             \
    if ((dtype) == DGNN_BF16) {                                                   \
      typedef bf16_t T;                                                           \
      if ((bytes) == 16) { constexpr int N = 8; return EXPR; }                    \
      if ((bytes) >= 4) { constexpr int N = 2; return EXPR; }                     \
      { constexpr int N = 1; return EXPR; }                                       \
    }                                                                             \
    typedef half_t T;                                                             \
    if ((bytes) == 16) { constexpr int N = 8; return EXPR; }                      \
    if ((bytes) >= 4) { constexpr int N = 2; return EXPR; }                       \
    { constexpr int N = 1; return EXPR; }                                         \
  } while (0)

extern "C" {

int dgnn_embedding_forward(int dtype, int idx_bytes, int n, int rows, int dim, float scale, const void *ids,
                           const void *table, void *out, void *stream) {
  const int rc = embed_check(dtype, idx_bytes, n, rows, dim);
  if (rc != DGNN_OK) return rc;
  if (n == 0 || dim == 0) return DGNN_OK;
  if (!ids || !out || (rows > 0 && !table)) return DGNN_ERR_BAD_ARG;
  const int size = dtype == DGNN_F32 ? 4 : 2;
  if (!aligned_to(ids, idx_bytes) || !aligned_to(table, size) || !aligned_to(out, size)) return DGNN_ERR_ALIGNMENT;
  const int bytes = access_bytes(dim, size, table, out);
  hipStream_t st = (hipStream_t)stream;
  if (idx_bytes == 8)
    DGNN_EMBED_DISPATCH(dtype, bytes, (launch_embed_fwd<T, N, long long>(n, rows, dim, scale, ids, table, out, st)));
  DGNN_EMBED_DISPATCH(dtype, bytes, (launch_embed_fwd<T, N, int>(n, rows, dim, scale, ids, table, out, st)));
}

size_t dgnn_embedding_backward_workspace_bytes(int n, int rows, int dim) {
  if (n <= 0 || rows <= 0 || dim <= 0) return 0;
  return embed_plan(n, rows, dim).total;
}

int dgnn_embedding_backward(int dtype, int idx_bytes, int n, int rows, int dim, float scale, const void *ids,
                            const void *grad, void *grad_table, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = embed_check(dtype, idx_bytes, n, rows, dim);
  if (rc != DGNN_OK) return rc;
  if (n > (1 << 30)) return DGNN_ERR_UNSUPPORTED;            // positions and steps past them are ints
  if (rows == 0 || dim == 0) return DGNN_OK;
  if (!grad_table || (n > 0 && (!ids || !grad))) return DGNN_ERR_BAD_ARG;
  const int size = dtype == DGNN_F32 ? 4 : 2;
  if (!aligned_to(ids, idx_bytes) || !aligned_to(grad, size) || !aligned_to(grad_table, size)) return DGNN_ERR_ALIGNMENT;
  // (columns are the second dimension of a launch, and a workgroup's rows times their pieces are an int)
  const int bytes = access_bytes(dim, size, grad, grad_table), per = access_elements(bytes, size);
  if (dim / (DGNN_WAVE * per) >= 65535 ||
      !launchable(((long long)rows + DGNN_BLOCK) / rows_per_block(rows, row_lanes(dim, per)), DGNN_BLOCK))
    return DGNN_ERR_UNSUPPORTED;
  const EmbedPlan p = embed_plan(n > 0 ? n : 1, rows, dim);
  if (n > 0 && (!workspace || workspace_bytes < p.total)) return DGNN_ERR_WORKSPACE;
  if (n > 0 && !aligned_to(workspace, 16)) return DGNN_ERR_ALIGNMENT;
  hipStream_t st = (hipStream_t)stream;
  const int *key = nullptr, *val = nullptr;
  float *part = nullptr;
  if (n > 0) {
    rc = idx_bytes == 8 ? sort_ids<long long>(n, rows, ids, p, (char *)workspace, &key, &val, st)
                        : sort_ids<int>(n, rows, ids, p, (char *)workspace, &key, &val, st);
    if (rc != DGNN_OK) return rc;
    part = (float *)((char *)workspace + 4 * p.pairs + p.counts);
  }
  DGNN_EMBED_DISPATCH(dtype, bytes, (launch_embed_sums<T, N>(n, rows, dim, scale, p, key, val, grad, part, grad_table, st)));
}

}  // extern "C"
