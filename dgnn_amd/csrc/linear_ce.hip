// Softmax cross entropy of a linear layer, without the logits: z = x W^T is formed a tile at a time.
//
//   lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_i,label(i),  dz_iv = (exp(z_iv - lse_i) - [v = label(i)]) g_i,
//   dx = dz W,  dW = dz^T x
//
// Rows whose label names no class (ignore_index, or outside [0, classes)) take no part: the labelled
// rows are gathered into a dense copy first (padded to whole 16-byte chunks), so the products neither
// spend time on the others nor read what stands in them.  The forward keeps a running maximum and sum
// per (row, class tile) and joins them; the backward rebuilds z a piece of the classes at a time,
// leaves dz in the workspace and multiplies it twice.
#include <string.h>

#include <type_traits>

#include "mma.hpp"

using namespace dgnn;

namespace dgnn {

#define DGNN_LOG2E 1.44269504088896340736f

// ------------------------------------------------------------------ one tile of C^T = A B^T
// WM x WN waves, each BM / WM x BN / WN of the tile; operands are staged BK k elements at a time through
// a ring of STAGES buffers.  An operand lies either with k along its rows (ROW: tile [BM][BK], read
// by row fragments) or with k down its columns (tile [BK][BM], read by transposing column fragments).
template <int BM_, int BN_, int BK_, int WM_, int WN_, int STAGES_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_, STAGES = STAGES_, THREADS = 64 * WM_ * WN_;
  static constexpr int MB = BM / WM / 32, NB = BN / WN / 32;           // 32 x 32 blocks of a wave
};

template <class T, class C, bool AROW, bool BROW>
struct Gemm {
  static constexpr int BM = C::BM, BN = C::BN, BK = C::BK, MB = C::MB, NB = C::NB, S = C::STAGES;
  using TA = Tile<T, AROW ? BK : BM>;
  using TB = Tile<T, BROW ? BK : BN>;
  static constexpr int A_BYTES = BM * BK * (int)sizeof(T), B_BYTES = BN * BK * (int)sizeof(T);
  static constexpr int BYTES = A_BYTES + B_BYTES;      // of a stage

  // an operand: first element of the tile's rows (or columns), how many of them exist, row stride
  struct Operand {
    const T *p;
    int count;                    // rows (ROW) or columns that exist from p on
    unsigned stride;              // bytes between rows
    const int *list = nullptr;    // ROW: the tile's rows are rows list[0 .. count) from p on
    unsigned bytes = 0;           // with a list: what the matrix spans from p on
  };

  // acc[m][n] += over k in [0, kn)
  __device__ static __forceinline__ void run(const Operand &a, const Operand &b, int kn, const lds_ptr (&lds)[4],
                                             acc16 (&acc)[MB][NB]) {
    const int lane = lane_id(), wave = uniform_i32(wave_in_block());
    const int m0 = wave / C::WN * (BM / C::WM), n0 = wave % C::WN * (BN / C::WN);
    // two row operands: consecutive k; against a column operand the order is its transposing read's.  The
    // wave's first row or column is part of the lane's address.
    const int ra = AROW ? (BROW ? TA::row_lane(lane) : TA::row_lane_split(lane)) + m0 * TA::ROW_BYTES
                        : TA::col_lane(lane) ^ (m0 / TA::CHUNK << 4);
    const int rb = BROW ? (AROW ? TB::row_lane(lane) : TB::row_lane_split(lane)) + n0 * TB::ROW_BYTES
                        : TB::col_lane(lane) ^ (n0 / TB::CHUNK << 4);
    Stager<T, AROW ? BK : BM, AROW ? BM : BK, C::THREADS> sa;
    Stager<T, BROW ? BK : BN, BROW ? BN : BK, C::THREADS> sb;
    sa.init(a.stride, AROW ? min(BK, kn) : a.count);
    if (BROW && b.list) sb.init_list(b.list, b.count, b.stride, min(BK, kn));
    else sb.init(b.stride, BROW ? min(BK, kn) : b.count);
    auto stage = [&](int t, auto i) {
      const lds_ptr ta = lds[i.value], tb = ta + A_BYTES;
      const int k0 = t * BK, left = max(0, min(BK, kn - k0));
      // rows end with a whole chunk (rows of dz are padded with zeros): a descriptor that ended inside one would
      // drop the dword the end falls into
      const unsigned row_bytes = (left * (unsigned)sizeof(T) + 15u) & ~15u;
      if (left < BK && left > 0 && k0 > 0) {                       // the last, shorter step
        if (AROW) sa.narrow(left);
        if (BROW) sb.narrow(left);
      }
      if (AROW)
        sa.load(ta, buffer_over(a.p + k0, span_bytes(left > 0 ? min(a.count, BM) : 0, a.stride, row_bytes)));
      else
        sa.load(ta, buffer_over((const char *)a.p + (long long)k0 * a.stride, span_bytes(left, a.stride, min(a.count, BM) * (unsigned)sizeof(T))));
      if (BROW && b.list)
        sb.load(tb, buffer_over(b.p + k0, left > 0 ? b.bytes - k0 * (unsigned)sizeof(T) : 0u));
      else if (BROW)
        sb.load(tb, buffer_over(b.p + k0, span_bytes(left > 0 ? min(b.count, BN) : 0, b.stride, row_bytes)));
      else
        sb.load(tb, buffer_over((const char *)b.p + (long long)k0 * b.stride, span_bytes(left, b.stride, min(b.count, BN) * (unsigned)sizeof(T))));
    };
    auto work = [&](int, auto i) {
      const lds_ptr ta = lds[i.value], tb = ta + A_BYTES;
#pragma unroll
      for (int k = 0; k < BK; k += 16) {
        frag8<T> fa[MB], fb[NB];
#pragma unroll
        for (int x = 0; x < MB; ++x) {
          if constexpr (AROW) fa[x] = BROW ? TA::row_frag(ta, ra, 32 * x, k) : TA::row_frag_split(ta, ra, 32 * x, k);
          else fa[x] = TA::col_frag(ta, ra, k, 32 * x);
        }
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          if constexpr (BROW) fb[x] = AROW ? TB::row_frag(tb, rb, 32 * x, k) : TB::row_frag_split(tb, rb, 32 * x, k);
          else fb[x] = TB::col_frag(tb, rb, k, 32 * x);
        }
        mma_block<MB, NB, T>(fa, fb, acc, T());
      }
    };
    ring<S, decltype(sa)::LOADS + decltype(sb)::LOADS, false>((kn + BK - 1) / BK, stage, work);
  }
  __device__ static __forceinline__ void clear(acc16 (&acc)[MB][NB]) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = acc_zero();
  }
};

// Which tile a workgroup takes.  Consecutive workgroups go to the eight XCDs in turn, so every XCD gets a
// contiguous range of an order that runs over `m` tiles first inside bands of eight `n` tiles: the 32
// workgroups of an XCD then read about 4 + 8 strips of the operands through its L2, not 1 + 32.
struct TileAt {
  int m, n;
};
// ns counts the tiles that have rows, known on the device alone: the workgroups behind them, which find
// nothing to do, are then the last ones and not an XCD's whole share.  n = -1: none left.
__device__ __forceinline__ TileAt tile_at(unsigned id, int ms, int ns) {
  if (id >= (unsigned)ms * (unsigned)ns) return {0, -1};
  const int u = (int)xcd_contiguous_id(id, (unsigned)ms * (unsigned)ns);
  const int band = u / (ms * 8), width = min(8, ns - band * 8), r = u - band * ms * 8;
  return {r / width, band * 8 + r % width};
}

// Tile shapes.  Wide: 16-bit types with enough tiles for every compute unit; two waves a SIMD, 128 KB of
// LDS.  Thin: at most 32 rows, bound by reading the weight (8 x 50000 x 1024 float 55 us, Plain 136; bfloat16 28
// both).  Narrow: at most 64 classes (4096 x 41 x 64 float 5.4 us, Plain 11.0;
// 65536 x 64 x 256 bfloat16, both directions, 235 and 260).
// Plain: the rest, and float, whose matrix instructions are sixteen times slower and bound every shape.
using Wide = Shape<256, 256, 32, 2, 4, 4>;
template <class T> using Plain = Shape<128, 128, sizeof(T) == 2 ? 64 : 16, 2, 2, sizeof(T) == 2 ? 2 : 3>;
template <class T> using Narrow = Shape<64, 64, sizeof(T) == 2 ? 64 : 32, 2, 2, 2>;
template <class T> using Thin = Shape<256, 32, sizeof(T) == 2 ? 64 : 32, 4, 1, 2>;

// ------------------------------------------------------------------ labelled rows
template <class I>
__device__ __forceinline__ int class_of(const I *label, int i, int classes, long long ignore) {
  const long long x = label[i];
  return x != ignore && x >= 0 && x < classes ? (int)x : -1;
}

// list[j] = j-th labelled row, count[0] = how many; one workgroup, in order.  The rows without a label get
// their loss and lse, 0, here.
template <class I>
__global__ __launch_bounds__(1024) void k_ce_rows(int n, int classes, long long ignore, const I *__restrict__ label,
                                                  int *__restrict__ list, int *__restrict__ count,
                                                  float *__restrict__ loss, float *__restrict__ lse) {
  constexpr int PER = 8;                        // labels a thread takes at a time
  __shared__ int part[16];
  const int lane = lane_id(), wave = wave_in_block();
  int carry = 0;
  for (int base = 0; base < n; base += 1024 * PER) {
    const int i = base + threadIdx.x * PER;
    unsigned on = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (i + k < n) {
        if (class_of(label, i + k, classes, ignore) >= 0) on |= 1u << k;
        else if (lse) {
          lse[i + k] = lse[n + i + k] = 0.f;
          if (loss) loss[i + k] = 0.f;
        }
      }
    const int own = __popc(on);
    int incl = own;
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) {
      const int up = __shfl_up(incl, w, 64);
      if (lane >= w) incl += up;
    }
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    int at = carry + incl - own;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) at += part[w];
      carry += part[w];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (on >> k & 1) list[at++] = i + k;
    __syncthreads();
  }
  if (threadIdx.x == 0) count[0] = carry;
}

struct Labels {
  const void *label;
  int bytes, classes;
  long long ignore;
  __device__ __forceinline__ long long at(int row) const {
    return bytes == 8 ? ((const long long *)label)[row] : (long long)((const int *)label)[row];
  }
  __device__ __forceinline__ bool valid(int row) const {
    const long long x = at(row);
    return x != ignore && x >= 0 && x < classes;
  }
};

// to[j, 0 .. ldt) = from[list[j], 0 .. d), zeros behind d; list == NULL: j itself.  j < count (count == NULL: n)
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_gather(int n, int d, int ldt, const int *__restrict__ list,
                                                          const int *__restrict__ count, const T *__restrict__ from,
                                                          long long ldf, int wide, T *__restrict__ to, const Labels labels,
                                                          T *__restrict__ zero) {
  constexpr int VEC = 16 / sizeof(T);
  // the rows of dx that have no label
  if (zero != nullptr)
    for (int r = blockIdx.x; r < n; r += gridDim.x)
      if (!labels.valid(r))
        for (int c = threadIdx.x; c < d; c += DGNN_BLOCK) zero[(long long)r * d + c] = (T)0.f;
  const int per = ldt / VEC, rows = count ? min(n, *count) : n;
  for (long long u = blockIdx.x * (long long)DGNN_BLOCK + threadIdx.x; u < (long long)rows * per; u += (long long)gridDim.x * DGNN_BLOCK) {
    const int j = (int)(u / per), c = (int)(u % per) * VEC;
    const T *src = from + (long long)(list ? list[j] : j) * ldf + c;
    if (wide) {                                   // rows start on 16 bytes and d is whole chunks
      *(u32x4 *)(to + (long long)j * ldt + c) = *(const u32x4 *)src;
    } else {
      T v[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = c + k < d ? src[k] : (T)0.f;
#pragma unroll
      for (int k = 0; k < VEC; ++k) to[(long long)j * ldt + c + k] = v[k];
    }
  }
}

struct CeArgs {
  const void *x, *w;              // rows [n, dk] (gathered: only those with a label), weight [classes, dk]
  int gathered;
  Labels labels;
  const int *list, *count;        // labelled rows in order and how many (NULL: row r is row r, all n take part)
  int n, classes, d, dk;          // dk = d rounded up to whole chunks
  float *part_m, *part_s;         // [class tiles, n]
  float *z_label;                 // [n], by gathered row
  float *lse, *loss;              // by original row, loss [n], lse [2, n]: log-sum and what its rounding to float took
  const float *grad;              // of the loss: n values or one
  int grad_rows, mean;
  const float *grad_top;          // one gradient a row: the largest magnitude
  void *dz;                       // [n, ldz]
  int v0, vn, ldz;                // piece of the classes
  float *acc;                     // split sums [splits][rows][d]
  int splits, first, direct;      // direct: one split of one piece, results go where they belong
  void *dx, *dw;
};

__device__ __forceinline__ int rows_of(const CeArgs &a) { return a.count ? min(a.n, *a.count) : a.n; }
__device__ __forceinline__ int row_at(const CeArgs &a, int r) { return a.list ? a.list[r] : r; }
// A labelled row's results from its largest logit, the log of its sum of exp(z - top) and its label's logit.  top + log
// is never rounded to float before a logit is taken off: with logits of 400 that alone is 1.5e-5, the whole loss and gradient
// of a row that is sure of its label.  The backward gets both parts.
__device__ __forceinline__ void store_row_loss(const CeArgs &a, int row, bool on, float top, double log_sum, float z_label) {
  const double v = (double)top + log_sum;
  const float hi = (float)v;
  a.lse[row] = on ? hi : 0.f;
  a.lse[a.n + row] = on && fabsf(hi) < INFINITY ? (float)(v - (double)hi) : 0.f;
  a.loss[row] = on ? (float)((double)top - (double)z_label + log_sum) : 0.f;
}
// dz is kept in T as (softmax - onehot) g_i / unit and the products carry the factor unit, the largest |g|
// (with the mean's division).  A common factor kept out of dz costs no rounding: rounded into it, one
// g for all rows would put the same error, up to half a step of T, on every gradient.  float16 also has too
// little range for a mean over some thousand rows; there dz runs up to 2^14, so that weights of the softmax
// down to 2^-38 survive, whatever the loss is scaled by.
struct CeScale {
  float unit, by;                 // by: g_i -> g_i / unit before the mean's division
};
template <class T>
__device__ __forceinline__ CeScale ce_scale(const CeArgs &a, int rows) {
  const float range = std::is_same<T, half_t>::value ? 16384.f : 1.f;
  // (not so small that 1 / unit overflows; a NaN or infinite g of the whole loss makes everything NaN)
  float top = a.grad_rows ? *a.grad_top : fabsf(a.grad[0]);
  if (top < 1e-30f) top = 1e-30f;
  const float m = a.mean ? 1.f / (float)max(1, rows) : 1.f;
  return {top * m / range, range / top};
}

// largest finite |g| of the labelled rows, one workgroup
__global__ __launch_bounds__(1024) void k_ce_grad_top(int n, const int *__restrict__ list, const int *__restrict__ count,
                                                      const float *__restrict__ grad, float *__restrict__ top) {
  __shared__ float part[16];
  const int rows = min(n, *count);
  float m = 0.f;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float g = fabsf(grad[list[i]]);
    if (g < INFINITY) m = fmaxf(m, g);
  }
  m = wave_max(m);
  if (lane_id() == 0) part[wave_in_block()] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) m = fmaxf(m, part[w]);
    top[0] = m;
  }
}

// the rows' operand of z
template <class T, class G>
__device__ __forceinline__ typename G::Operand rows_operand(const CeArgs &a, int r0, int rows) {
  const unsigned stride = (unsigned)(a.dk * sizeof(T));
  if (a.gathered || !a.list) return {(const T *)a.x + (long long)r0 * a.dk, rows - r0, stride};
  return {(const T *)a.x, rows - r0, stride, a.list + r0, a.n * stride};
}

// Forward: classes along m, rows along n.  Leaves the tile's maximum and sum of exp for every row and
// the logit of its label.  Bound by the matrix instructions, in 16 bits under the power limit: 8192 x 100003 x 2048
// bfloat16 2.9 - 3.1 ms, 1080 - 1160 TFLOP/s (a large matrix product reaches 1156); 4099 x 19717 x 128 float, nine
// rows in ten labelled, 190 us, 98 TFLOP/s (154).
template <class T, class C>
__global__ __launch_bounds__(C::THREADS, C::THREADS == 512 ? 2 : 1) void k_ce_fwd(const CeArgs a) {
  using G = Gemm<T, C, true, true>;
  DGNN_RING(lds, G::BYTES);
  __shared__ float sm[C::WM][C::BN], ss[C::WM][C::BN], zl[C::BN];
  const int rows = rows_of(a);
  const TileAt tile = tile_at(group_in_rows(), (a.classes + C::BM - 1) / C::BM, (rows + C::BN - 1) / C::BN);
  if (tile.n < 0) return;
  const int v0 = tile.m * C::BM, r0 = tile.n * C::BN;
  acc16 acc[C::MB][C::NB];
  G::clear(acc);
  G::run({(const T *)a.w + (long long)v0 * a.dk, a.classes - v0, (unsigned)(a.dk * sizeof(T))},
         rows_operand<T, G>(a, r0, rows), a.dk, lds, acc);
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int wm = wave / C::WN, m0 = v0 + wm * (C::BM / C::WM), n0 = wave % C::WN * (C::BN / C::WN);
  const bool whole = v0 + C::BM <= a.classes;
#pragma unroll
  for (int j = 0; j < C::NB; ++j) {
    const int col = n0 + 32 * j + (lane & 31), r = r0 + col;
    const long long label = r < rows ? a.labels.at(row_at(a, r)) : -1, want = label == a.labels.ignore ? -1 : label - m0;
    float top = -INFINITY;
    if (want >= 0 && want < C::BM / C::WM) {
#pragma unroll
      for (int i = 0; i < C::MB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * i + acc_row(e, h) == (int)want) {
            if (a.part_m == nullptr) zl[col] = acc[i][j][e];
            else a.z_label[r] = acc[i][j][e];
          }
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < C::MB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (m0 + 32 * i + acc_row(e, h) >= a.classes) acc[i][j][e] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < C::MB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // the difference first: the largest logit then adds exactly one.  Blocks of sixteen are summed by themselves, or
    // a hundred small terms would each be rounded against that one.
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < C::MB; ++i) {
      float block = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) block += __builtin_amdgcn_exp2f((acc[i][j][e] - base) * DGNN_LOG2E);
      sum += block;
    }
    sum += __shfl_xor(sum, 32, 64);
    if (h == 0) sm[wm][col] = top, ss[wm][col] = sum;
  }
  __syncthreads();
  if (threadIdx.x < C::BN && r0 + (int)threadIdx.x < rows) {
    float top = sm[0][threadIdx.x], s = 0.f;
#pragma unroll
    for (int w = 1; w < C::WM; ++w) top = fmaxf(top, sm[w][threadIdx.x]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < C::WM; ++w) s += ss[w][threadIdx.x] * __builtin_amdgcn_exp2f((sm[w][threadIdx.x] - base) * DGNN_LOG2E);
    if (a.part_m == nullptr) {                  // one tile of classes: this is all there is
      const int row = r0 + threadIdx.x;
      store_row_loss(a, row, a.labels.valid(row), base, (double)logf(s), zl[threadIdx.x]);
      return;
    }
    const long long at = (long long)tile.m * a.n + r0 + threadIdx.x;
    a.part_m[at] = top;
    a.part_s[at] = s;
  }
}

// lse and loss of every labelled row from its tiles' pairs: eight rows a workgroup, 32 threads a row
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_join(const CeArgs a, int tiles) {
  const float *__restrict__ pm = a.part_m, *__restrict__ ps = a.part_s;
  const int n = a.n;
  // doubles: a thread may add some thousand tiles' sums of like size, each rounding the same way
  __shared__ float sm[32][8];
  __shared__ double ss[32][8];
  const int c = threadIdx.x & 7, lane = threadIdx.x >> 3, r = blockIdx.x * 8 + c, rows = rows_of(a);
  if ((int)blockIdx.x * 8 >= rows) return;
  float m = -INFINITY;
  double s = 0.;
  if (r < rows) {
#pragma unroll 4
    for (int t = lane; t < tiles; t += 32) {
      const float tm = pm[(long long)t * n + r], ts = ps[(long long)t * n + r], top = fmaxf(m, tm);
      const float base = top == -INFINITY ? 0.f : top;
      s = s * (double)expf(m - base) + (double)ts * (double)expf(tm - base);
      m = top;
    }
  }
  sm[lane][c] = m, ss[lane][c] = s;
  __syncthreads();
  if (lane != 0 || r >= rows) return;
  float top = sm[0][c];
  for (int w = 1; w < 32; ++w) top = fmaxf(top, sm[w][c]);
  const float base = top == -INFINITY ? 0.f : top;
  double sum = 0.;
  for (int w = 0; w < 32; ++w) sum += ss[w][c] * (double)expf(sm[w][c] - base);
  const int row = row_at(a, r);
  store_row_loss(a, row, a.labels.valid(row), base, log(sum), a.z_label[r]);
}
// out[0] = sum of the losses (/ labelled rows), in a fixed order; no labelled row: 0
__global__ __launch_bounds__(1024) void k_ce_reduce(const CeArgs a, int mean, const float *__restrict__ loss, float *__restrict__ out) {
  __shared__ double part[16];
  __shared__ int counts[16];
  double s = 0.;
  int c = 0;
  for (int i = threadIdx.x; i < a.n; i += 1024) {
    s += (double)loss[i];
    if (mean && !a.count) c += a.labels.valid(i);
  }
  for (int w = 32; w > 0; w >>= 1) s += __shfl_xor(s, w, 64), c += __shfl_xor(c, w, 64);
  if (lane_id() == 0) part[wave_in_block()] = s, counts[wave_in_block()] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += part[w], c += counts[w];
    if (a.count) c = *a.count;
    out[0] = (float)(mean ? s / (double)max(1, c) : s);
  }
}

// Turns a workgroup's C^T tile into rows of T through LDS, 32 rows of every wave column at a time in a ring
// buffer of its own, and hands 16-byte pieces to sink(row, column, piece): a lane holds four elements of
// one row, and stored from there every instruction would touch 32 rows.  The ring is drained by then.
template <class T, class C, class Value, class Sink>
__device__ __forceinline__ void rows_of_tile(const lds_ptr (&lds)[4], const Value &value, const Sink &sink) {
  using TL = Tile<T, C::BM>;
  constexpr int PIECES = 32 * TL::CPR;
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int wm = wave / C::WN, wn = wave % C::WN, m0 = wm * (C::BM / C::WM);
#pragma unroll
  for (int j = 0; j < C::NB; ++j) {
    __syncthreads();
    unrolled<0, C::WN>([&](auto b) {
      if (wn != b.value) return;
      const lds_ptr buf = lds[b.value];
#pragma unroll
      for (int i = 0; i < C::MB; ++i)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int m = m0 + 32 * i + 8 * e4 + 4 * h;
          vec4<T> v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = value(i, j, 4 * e4 + e, m + e);
          *(DGNN_LDS vec4<T> *)(buf + TL::chunk_addr(lane & 31, m / TL::CHUNK) + m % TL::CHUNK * (int)sizeof(T)) = v;
        }
    });
    __syncthreads();
    unrolled<0, C::WN>([&](auto b) {
      if (wn != b.value) return;
      const lds_ptr buf = lds[b.value];
      for (int u = wm * 64 + lane; u < PIECES; u += C::WM * 64) {
        const int row = u / TL::CPR, chunk = u % TL::CPR;
        sink(wn * (C::BN / C::WN) + 32 * j + row, chunk * TL::CHUNK, *(const DGNN_LDS u32x4 *)(buf + TL::chunk_addr(row, chunk)));
      }
    });
  }
}
// A piece of a row: as one store, or the elements of it that exist.
template <class T>
__device__ __forceinline__ void store_piece(T *row, int col, int cols, u32x4 piece, bool whole) {
  constexpr int VEC = 16 / sizeof(T);
  if (whole) {
    if (col < cols) *(u32x4 *)(row + col) = piece;
  } else {
    T v[VEC];
    *(u32x4 *)v = piece;
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (col + k < cols) row[col + k] = v[k];
  }
}

// dz of a piece of the classes, [rows, ldz]; columns behind the piece's last class are zeros.  The forward's
// product once more and a store of dz, half a step of T off: at 8192 x 100003 x 2048 bfloat16 3.7 ms in all, 910
// TFLOP/s; what it loses to k_ce_fwd is the turning of tiles for whole-line stores.
template <class T, class C>
__global__ __launch_bounds__(C::THREADS, C::THREADS == 512 ? 2 : 1) void k_ce_dz(const CeArgs a) {
  using G = Gemm<T, C, true, true>;
  static_assert(32 * C::BM * sizeof(T) <= G::BYTES && C::WN <= 4, "the tile as rows fits the ring");
  DGNN_RING(lds, G::BYTES);
  const int rows = rows_of(a);
  const TileAt tile = tile_at(group_in_rows(), a.ldz / C::BM, (rows + C::BN - 1) / C::BN);
  if (tile.n < 0) return;
  const int p0 = tile.m * C::BM, v0 = a.v0 + p0, r0 = tile.n * C::BN;
  acc16 acc[C::MB][C::NB];
  G::clear(acc);
  G::run({(const T *)a.w + (long long)v0 * a.dk, a.classes - v0, (unsigned)(a.dk * sizeof(T))},
         rows_operand<T, G>(a, r0, rows), a.dk, lds, acc);
  const int lane = lane_id(), wave = uniform_i32(wave_in_block()), n0 = wave % C::WN * (C::BN / C::WN);
  const CeScale scale = ce_scale<T>(a, rows);
  // exp(z - lse) = exp2(z log2e - c) f, c the product with the whole lse rounded to float, f what that took
  float c[C::NB], fg[C::NB], g[C::NB];
  int want[C::NB];
#pragma unroll
  for (int j = 0; j < C::NB; ++j) {
    const int r = r0 + n0 + 32 * j + (lane & 31), row = r < rows ? a.list[r] : a.list[0];
    want[j] = (int)(a.labels.at(row) - v0);
    const double t = ((double)a.lse[row] + (double)a.lse[a.n + row]) * (double)DGNN_LOG2E;
    c[j] = (float)t;
    g[j] = a.grad[a.grad_rows ? row : 0] * scale.by;
    fg[j] = g[j] * __builtin_amdgcn_exp2f(fabsf(c[j]) < INFINITY ? (float)((double)c[j] - t) : 0.f);
  }
  const int left = a.vn - p0;                   // classes of this tile
  rows_of_tile<T, C>(
      lds,
      [&](int i, int j, int e, int m) {
        const float y = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], DGNN_LOG2E, -c[j]));
        return (T)(m < left ? fmaf(y, fg[j], m == want[j] ? -g[j] : 0.f) : 0.f);
      },
      [&](int row, int col, u32x4 piece) {
        if (r0 + row < rows) *(u32x4 *)((T *)a.dz + (long long)(r0 + row) * a.ldz + p0 + col) = piece;
      });
}

// A lane's columns of C^T as a row of partial sums, columns m0 .. < d; add: to what an earlier piece left there.
template <class C>
__device__ __forceinline__ void store_sums(float *to, const acc16 (&acc)[C::MB][C::NB], int j, int m0, int d, int h, bool add) {
#pragma unroll
  for (int i = 0; i < C::MB; ++i)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int at = m0 + 32 * i + 8 * e4 + 4 * h;
      const acc16 &c = acc[i][j];
      if (at >= d) continue;
      float4 v = make_float4(c[4 * e4], c[4 * e4 + 1], c[4 * e4 + 2], c[4 * e4 + 3]);
      if (add) {
        const float4 old = *(const float4 *)(to + at);
        v.x += old.x, v.y += old.y, v.z += old.z, v.w += old.w;
      }
      *(float4 *)(to + at) = v;
    }
}

// dx of a piece: C^T[d, rows] += W_piece^T dz^T.  One split of a single piece: straight to dx; else into
// acc[split], added to over the pieces, joined by k_ce_dx_join.  3.1 ms in all at 8192 x 100003 x 2048 bfloat16, 1080
// TFLOP/s.
template <class T, class C>
__global__ __launch_bounds__(C::THREADS, C::THREADS == 512 ? 2 : 1) void k_ce_dx(const CeArgs a, int whole) {
  using G = Gemm<T, C, false, true>;
  DGNN_RING(lds, G::BYTES);
  const int rows = rows_of(a), ms = (a.dk + C::BM - 1) / C::BM, ns = (rows + C::BN - 1) / C::BN;
  const unsigned id = group_in_rows();
  const int split = ns > 0 ? id / (unsigned)(ms * ns) : a.splits;
  if (split >= a.splits) return;
  const TileAt tile = tile_at(id % (unsigned)(ms * ns), ms, ns);
  const int c0 = tile.m * C::BM, r0 = tile.n * C::BN;
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int m0 = c0 + wave / C::WN * (C::BM / C::WM), n0 = wave % C::WN * (C::BN / C::WN);
  acc16 acc[C::MB][C::NB];
  G::clear(acc);
  const int steps = (a.vn + C::BK - 1) / C::BK, per = (steps + a.splits - 1) / a.splits;
  const int ka = min(a.vn, split * per * C::BK), kb = min(a.vn, (split + 1) * per * C::BK);
  G::run({(const T *)a.w + (long long)(a.v0 + ka) * a.dk + c0, a.dk - c0, (unsigned)(a.dk * sizeof(T))},
         {(const T *)a.dz + (long long)r0 * a.ldz + ka, rows - r0, (unsigned)(a.ldz * sizeof(T))}, kb - ka, lds, acc);
  if (a.direct) {
    const float unit = ce_scale<T>(a, rows).unit;
    rows_of_tile<T, C>(
        lds, [&](int i, int j, int e, int) { return (T)(acc[i][j][e] * unit); },
        [&](int row, int col, u32x4 piece) {
          if (r0 + row < rows) store_piece<T>((T *)a.dx + (long long)a.list[r0 + row] * a.d, c0 + col, a.d, piece, whole != 0);
        });
    return;
  }
#pragma unroll
  for (int j = 0; j < C::NB; ++j) {
    const int r = r0 + n0 + 32 * j + (lane & 31);
    if (r < rows) store_sums<C>(a.acc + ((long long)split * a.n + r) * a.dk, acc, j, m0, a.dk, h, !a.first);
  }
}
// dx[list[r]] = sum over the splits, in order
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_dx_join(const CeArgs a) {
  const int rows = rows_of(a), per = a.dk / 4;
  const float unit = ce_scale<T>(a, rows).unit;
  for (long long u = blockIdx.x * (long long)DGNN_BLOCK + threadIdx.x; u < (long long)rows * per; u += (long long)gridDim.x * DGNN_BLOCK) {
    const int r = (int)(u / per), c = (int)(u % per) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < a.splits; ++k) {
      const float4 v = *(const float4 *)(a.acc + ((long long)k * a.n + r) * a.dk + c);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    T *to = (T *)a.dx + (long long)a.list[r] * a.d + c;
    const float f[4] = {s.x * unit, s.y * unit, s.z * unit, s.w * unit};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < a.d) to[j] = (T)f[j];
  }
}
// dW of a piece: C^T[d, classes of the piece] = x^T dz.  splits > 1: partial sums over shares of the rows.  3.0 ms in
// all at 8192 x 100003 x 2048 bfloat16, 1110 TFLOP/s.
template <class T, class C>
__global__ __launch_bounds__(C::THREADS, C::THREADS == 512 ? 2 : 1) void k_ce_dw(const CeArgs a, int whole) {
  using G = Gemm<T, C, false, false>;
  DGNN_RING(lds, G::BYTES);
  const int ms = (a.dk + C::BM - 1) / C::BM, ns = (a.vn + C::BN - 1) / C::BN;
  const unsigned id = group_in_rows();
  const int split = id / (unsigned)(ms * ns);
  if (split >= a.splits) return;
  const TileAt tile = tile_at(id % (unsigned)(ms * ns), ms, ns);
  const int c0 = tile.m * C::BM, p0 = tile.n * C::BN;
  const int rows = rows_of(a);
  acc16 acc[C::MB][C::NB];
  G::clear(acc);
  const int steps = (rows + C::BK - 1) / C::BK, per = (steps + a.splits - 1) / a.splits;
  const int ka = min(rows, split * per * C::BK), kb = min(rows, (split + 1) * per * C::BK);
  G::run({(const T *)a.x + (long long)ka * a.dk + c0, a.dk - c0, (unsigned)(a.dk * sizeof(T))},
         {(const T *)a.dz + (long long)ka * a.ldz + p0, a.ldz - p0, (unsigned)(a.ldz * sizeof(T))}, kb - ka, lds, acc);
  if (a.splits == 1) {
    const float unit = ce_scale<T>(a, rows).unit;
    rows_of_tile<T, C>(
        lds, [&](int i, int j, int e, int) { return (T)(acc[i][j][e] * unit); },
        [&](int row, int col, u32x4 piece) {
          if (p0 + row < a.vn) store_piece<T>((T *)a.dw + (long long)(a.v0 + p0 + row) * a.d, c0 + col, a.d, piece, whole != 0);
        });
    return;
  }
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int m0 = c0 + wave / C::WN * (C::BM / C::WM), n0 = wave % C::WN * (C::BN / C::WN);
#pragma unroll
  for (int j = 0; j < C::NB; ++j) {
    const int p = p0 + n0 + 32 * j + (lane & 31);
    if (p < a.vn) store_sums<C>(a.acc + ((long long)split * a.ldz + p) * a.dk, acc, j, m0, a.dk, h, false);
  }
}
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_dw_join(const CeArgs a) {
  const int per = a.dk / 4;
  const float unit = ce_scale<T>(a, min(a.n, *a.count)).unit;
  for (long long u = blockIdx.x * (long long)DGNN_BLOCK + threadIdx.x; u < (long long)a.vn * per; u += (long long)gridDim.x * DGNN_BLOCK) {
    const int p = (int)(u / per), c = (int)(u % per) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < a.splits; ++k) {
      const float4 v = *(const float4 *)(a.acc + ((long long)k * a.ldz + p) * a.dk + c);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    T *to = (T *)a.dw + (long long)(a.v0 + p) * a.d + c;
    const float f[4] = {s.x * unit, s.y * unit, s.z * unit, s.w * unit};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < a.d) to[j] = (T)f[j];
  }
}

// ------------------------------------------------------------------ plans
static inline size_t align256(size_t x) { return (x + 255) / 256 * 256; }
static inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
static inline unsigned grid_for(long long units) {
  const long long b = (units + DGNN_BLOCK - 1) / DGNN_BLOCK;
  return (unsigned)(b < 1 ? 1 : b > 8192 ? 8192 : b);
}

enum CeShape { CE_PLAIN, CE_WIDE, CE_THIN, CE_NARROW };
struct CePlan {
  int dk, tiles, copy_w, gather, all;                 // class tiles of the forward; all: no list of labelled rows
  CeShape z, dx_shape, dw_shape;
  size_t list, x, w, part, zl, fwd_total;             // bytes
  int piece, pieces, dx_splits, dw_splits;
  size_t dz, dxacc, dwacc, bwd_total;
};
// Wide tiles halve what every product reads from LDS, but there have to be enough of them for 256 compute
// units.  bfloat16, both directions with Wide and with Plain: 8192 x 50000 x 1024 3.64 and 4.16 ms (the forward
// 874 and 956 us), 2048 x 50000 x 512 579 and 625 us.
static CeShape ce_shape(int dtype, long long m, long long n) {
  const long long wide = ((m + 255) / 256) * ((n + 255) / 256);
  return dtype != DGNN_F32 && wide >= 256 ? CE_WIDE : CE_PLAIN;
}
static CePlan ce_plan(int dtype, int n, int classes, int d, const void *x, const void *w) {
  CePlan p;
  memset(&p, 0, sizeof(p));
  const int size = dtype == DGNN_F32 ? 4 : 2, vec = 16 / size;
  p.dk = (d + vec - 1) / vec * vec;
  // rows are read where they are if they are whole, aligned chunks within 32-bit offsets
  p.copy_w = p.dk != d || ((uintptr_t)w & 15) != 0;
  p.gather = p.dk != d || ((uintptr_t)x & 15) != 0 || (long long)n * p.dk * size >= 0x7fffffffLL;
  // up to about 1e9 operations finding the labelled rows costs more than scoring all: 4096 x 41 x 64 float 5.4 us
  // against 16.9, 1024 x 1000 x 256 bfloat16 12.2 against 16.7; 4096 x 1000 x 128 float 27.2 both
  p.all = !p.gather && 2.0 * n * classes * d <= 1e9;
  p.z = classes <= 64 ? CE_NARROW : n <= 32 ? CE_THIN : ce_shape(dtype, classes, n);
  const int class_tile = p.z == CE_NARROW ? 64 : p.z == CE_PLAIN ? 128 : 256;
  p.tiles = ceil_div(classes, class_tile);
  p.list = align256(sizeof(int) * ((size_t)n + 1));
  p.x = align256((size_t)n * p.dk * size);
  p.w = p.copy_w ? align256((size_t)classes * p.dk * size) : 0;
  p.part = align256(sizeof(float) * (size_t)p.tiles * n);
  p.zl = align256(sizeof(float) * (size_t)n);
  p.fwd_total = p.list + (p.gather ? p.x : 0) + p.w + 2 * p.part + 2 * p.zl;
  // pieces: dz of about 2^27 elements, whole tiles (bfloat16 8192 x 100003 x 2048: 14.1 ms with 2^26, 13.7 with 2^27,
  // 14.0 with 1.5 times that, which no longer stays in the 256 MB cache); at most 2^20 columns: 256 rows of a piece stay in 32-bit offsets
  long long cols = (1LL << 27) / n;
  cols = cols < 1024 ? 1024 : cols > (1 << 20) ? 1 << 20 : cols;
  if (cols > classes) cols = classes;
  p.piece = ceil_div(ceil_div(classes, ceil_div(classes, cols)), class_tile) * class_tile;
  p.pieces = ceil_div(classes, p.piece);
  // enough workgroups for every compute unit: split the long axis while tiles are few
  // float: a sum of 10^5 terms in one accumulator has lost three of its seven digits, so none is longer than
  // 4096 terms, or a 64th of the axis
  auto splits = [&](long long tiles, int steps) {
    long long s = tiles > 0 ? 512 / tiles : 1;
    if (dtype == DGNN_F32 && s < (steps + 63) / 64) s = (steps + 63) / 64;
    if (s > steps / 4) s = steps / 4;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
  };
  auto choose = [&](long long cols_of, int steps, CeShape *shape, int *split) {
    const long long wide = (long long)ceil_div(p.dk, 256) * ceil_div(cols_of, 256);
    // a wide tile is worth having if splitting the long axis still gives every compute unit one
    const int s = wide >= 256 ? 1 : (int)((256 + wide - 1) / wide);
    if (dtype != DGNN_F32 && s <= 4 && steps / s >= 16 && p.dk > 128) {
      *shape = CE_WIDE, *split = s;
    } else {
      *shape = CE_PLAIN;
      *split = splits((long long)ceil_div(p.dk, 128) * ceil_div(cols_of, 128), steps);
    }
  };
  choose(n, p.piece / 64, &p.dx_shape, &p.dx_splits);
  choose(p.piece, n / 64, &p.dw_shape, &p.dw_splits);
  p.dz = align256((size_t)n * p.piece * size);
  p.dxacc = p.dx_splits > 1 || p.pieces > 1 ? align256(sizeof(float) * (size_t)p.dx_splits * n * p.dk) : 0;
  p.dwacc = p.dw_splits > 1 ? align256(sizeof(float) * (size_t)p.dw_splits * p.piece * p.dk) : 0;
  p.bwd_total = p.list + p.x + p.w + p.dz + p.dxacc + p.dwacc + 256;
  return p;
}

static int ce_check(int dtype, int label_bytes, int n, int classes, int d) {
  if (dtype < 0 || dtype > 2 || (label_bytes != 4 && label_bytes != 8) || n < 0 || classes <= 0 || d <= 0) return DGNN_ERR_BAD_ARG;
  if (d > 65536 || n > (1 << 22) || classes > (1 << 30)) return DGNN_ERR_UNSUPPORTED;
  return DGNN_OK;
}

// labelled rows -> list, count; gathered x where asked; padded weight where its rows are not whole chunks
template <class T>
static int ce_prepare(const CePlan &p, int n, int classes, int d, bool all, bool gather, const void *x, const void *w, const void *label,
                      int label_bytes, long long ignore, float *loss, float *lse, void *dx, char *ws, CeArgs *a, hipStream_t st) {
  int *list = (int *)ws, *count = list + n;
  T *xc = (T *)(ws + p.list), *wc = (T *)(ws + p.list + (gather ? p.x : 0));
  if (!all) {
    if (label_bytes == 8)
      hipLaunchKernelGGL(k_ce_rows<long long>, dim3(1), dim3(1024), 0, st, n, classes, ignore, (const long long *)label, list, count, loss, lse);
    else
      hipLaunchKernelGGL(k_ce_rows<int>, dim3(1), dim3(1024), 0, st, n, classes, ignore, (const int *)label, list, count, loss, lse);
    DGNN_LAUNCH_CHECK();
  }
  const int per = p.dk / (16 / (int)sizeof(T));
  if (gather) {
    hipLaunchKernelGGL(k_ce_gather<T>, dim3(grid_for((long long)n * per)), dim3(DGNN_BLOCK), 0, st, n, d, p.dk,
                       (const int *)list, (const int *)count, (const T *)x, (long long)d,
                       (int)(p.dk == d && ((uintptr_t)x & 15) == 0), xc, Labels{label, label_bytes, classes, ignore}, (T *)dx);
    DGNN_LAUNCH_CHECK();
  }
  if (p.copy_w) {
    hipLaunchKernelGGL(k_ce_gather<T>, dim3(grid_for((long long)classes * per)), dim3(DGNN_BLOCK), 0, st, classes, d, p.dk,
                       (const int *)nullptr, (const int *)nullptr, (const T *)w, (long long)d, 0, wc, Labels{nullptr, 4, 0, 0}, (T *)nullptr);
    DGNN_LAUNCH_CHECK();
  }
  memset(a, 0, sizeof(*a));
  a->x = gather ? (const void *)xc : x, a->gathered = gather, a->w = p.copy_w ? (const void *)wc : w;
  a->labels = Labels{label, label_bytes, classes, ignore};
  if (!all) a->list = list, a->count = count;
  a->n = n, a->classes = classes, a->d = d, a->dk = p.dk;
  return DGNN_OK;
}

// LAUNCH(kernel, shape's columns along m, along n, splits, args...) for the shape chosen at run time
#define DGNN_CE_LAUNCH(KERNEL, C, ms, ns, splits, ...)                                                          \
  do {                                                                                                         \
    const long long grid_ = (long long)ceil_div(ms, C::BM) * ceil_div(ns, C::BN) * (splits);                    \
    if (grid_ > 0x7fffffffLL) return DGNN_ERR_UNSUPPORTED;                                                     \
    hipLaunchKernelGGL((KERNEL<T, C>), grid_in_rows(grid_), dim3(C::THREADS), 0, st, __VA_ARGS__);           \
    DGNN_LAUNCH_CHECK();                                                                                       \
  } while (0)

template <class T>
static int ce_forward(const CePlan &p, int n, int classes, int d, const void *x, const void *w, const void *label,
                      int label_bytes, long long ignore, int reduction, float *loss, float *lse, char *ws, hipStream_t st) {
  CeArgs a;
  char *at = ws + p.list + (p.gather ? p.x : 0) + p.w;
  float *row = reduction == 0 ? loss : (float *)(at + 2 * p.part + p.zl);
  const int rc = ce_prepare<T>(p, n, classes, d, p.all != 0, p.gather != 0, x, w, label, label_bytes, ignore, row, lse, nullptr, ws, &a, st);
  if (rc != DGNN_OK) return rc;
  a.lse = lse, a.loss = row;
  if (!p.all || p.tiles > 1) a.part_m = (float *)at, a.part_s = (float *)(at + p.part), a.z_label = (float *)(at + 2 * p.part);
  if (p.z == CE_THIN) {
    DGNN_CE_LAUNCH(k_ce_fwd, Thin<T>, classes, n, 1, a);
  } else if (p.z == CE_NARROW) {
    DGNN_CE_LAUNCH(k_ce_fwd, Narrow<T>, classes, n, 1, a);
  } else if (p.z == CE_PLAIN) {
    DGNN_CE_LAUNCH(k_ce_fwd, Plain<T>, classes, n, 1, a);
  } else if constexpr (sizeof(T) == 2) {
    DGNN_CE_LAUNCH(k_ce_fwd, Wide, classes, n, 1, a);
  }
  if (a.part_m) {
    hipLaunchKernelGGL(k_ce_join, dim3(ceil_div(n, 8)), dim3(DGNN_BLOCK), 0, st, a, p.tiles);
    DGNN_LAUNCH_CHECK();
  }
  if (reduction != 0) {
    hipLaunchKernelGGL(k_ce_reduce, dim3(1), dim3(1024), 0, st, a, (int)(reduction == 1), (const float *)row, loss);
    DGNN_LAUNCH_CHECK();
  }
  return DGNN_OK;
}

template <class T>
static int ce_backward(const CePlan &p, int n, int classes, int d, const void *x, const void *w, const void *label,
                       int label_bytes, long long ignore, int reduction, const float *lse, const float *grad, void *dx,
                       void *dw, char *ws, hipStream_t st) {
  CeArgs a;
  const int rc = ce_prepare<T>(p, n, classes, d, false, true, x, w, label, label_bytes, ignore, nullptr, nullptr, dx, ws, &a, st);
  if (rc != DGNN_OK) return rc;
  char *at = ws + p.list + p.x + p.w;
  a.dz = at, a.ldz = p.piece;
  float *dxacc = (float *)(at + p.dz), *dwacc = (float *)(at + p.dz + p.dxacc);
  a.lse = (float *)lse, a.grad = grad, a.grad_rows = reduction == 0, a.mean = reduction == 1;
  a.dx = dx, a.dw = dw;
  if (a.grad_rows) {
    float *top = (float *)(at + p.dz + p.dxacc + p.dwacc);
    hipLaunchKernelGGL(k_ce_grad_top, dim3(1), dim3(1024), 0, st, n, a.list, a.count, grad, top);
    DGNN_LAUNCH_CHECK();
    a.grad_top = top;
  }
  a.direct = p.dx_splits == 1 && p.pieces == 1;
  const int whole_x = p.dk == d && ((uintptr_t)dx & 15) == 0, whole_w = p.dk == d && ((uintptr_t)dw & 15) == 0;
  for (int v0 = 0; v0 < classes; v0 += p.piece) {
    a.v0 = v0, a.vn = classes - v0 < p.piece ? classes - v0 : p.piece, a.first = v0 == 0;
    if (p.z == CE_THIN) {
      DGNN_CE_LAUNCH(k_ce_dz, Thin<T>, p.piece, n, 1, a);
    } else if (p.z == CE_NARROW) {
      DGNN_CE_LAUNCH(k_ce_dz, Narrow<T>, p.piece, n, 1, a);
    } else if (p.z == CE_PLAIN) {
      DGNN_CE_LAUNCH(k_ce_dz, Plain<T>, p.piece, n, 1, a);
    } else if constexpr (sizeof(T) == 2) {
      DGNN_CE_LAUNCH(k_ce_dz, Wide, p.piece, n, 1, a);
    }
    if (dx) {
      a.acc = dxacc, a.splits = p.dx_splits;
      if (p.dx_shape == CE_PLAIN) {
        DGNN_CE_LAUNCH(k_ce_dx, Plain<T>, p.dk, n, p.dx_splits, a, whole_x);
      } else if constexpr (sizeof(T) == 2) {
        DGNN_CE_LAUNCH(k_ce_dx, Wide, p.dk, n, p.dx_splits, a, whole_x);
      }
    }
    if (dw) {
      a.acc = dwacc, a.splits = p.dw_splits;
      if (p.dw_shape == CE_PLAIN) {
        DGNN_CE_LAUNCH(k_ce_dw, Plain<T>, p.dk, a.vn, p.dw_splits, a, whole_w);
      } else if constexpr (sizeof(T) == 2) {
        DGNN_CE_LAUNCH(k_ce_dw, Wide, p.dk, a.vn, p.dw_splits, a, whole_w);
      }
      if (p.dw_splits > 1) {
        hipLaunchKernelGGL(k_ce_dw_join<T>, dim3(grid_for((long long)a.vn * p.dk / 4)), dim3(DGNN_BLOCK), 0, st, a);
        DGNN_LAUNCH_CHECK();
      }
    }
  }
  if (dx && !a.direct) {
    a.acc = dxacc, a.splits = p.dx_splits;
    hipLaunchKernelGGL(k_ce_dx_join<T>, dim3(grid_for((long long)n * p.dk / 4)), dim3(DGNN_BLOCK), 0, st, a);
    DGNN_LAUNCH_CHECK();
  }
  return DGNN_OK;
}

}  // namespace dgnn

extern "C" {

size_t dgnn_linear_ce_workspace_bytes(int dtype, int n, int classes, int d, int backward) {
  if (ce_check(dtype, 4, n, classes, d) != DGNN_OK || n == 0) return 0;
  const CePlan p = ce_plan(dtype, n, classes, d, (const void *)1, (const void *)1);    // the larger case: copies of both
  return backward ? p.bwd_total : p.fwd_total;
}

int dgnn_linear_ce_forward(int dtype, int label_bytes, int n, int classes, int d, long long ignore_index, int reduction,
                           const void *x, const void *w, const void *label, float *loss, float *lse, void *workspace,
                           size_t workspace_bytes, void *stream) {
  const int rc = ce_check(dtype, label_bytes, n, classes, d);
  if (rc != DGNN_OK) return rc;
  if (reduction < 0 || reduction > 2) return DGNN_ERR_BAD_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (n == 0) {
    if (reduction != 0 && loss) {
      CeArgs a;
      memset(&a, 0, sizeof(a));
      hipLaunchKernelGGL(k_ce_reduce, dim3(1), dim3(1024), 0, st, a, 0, (const float *)nullptr, loss);
      DGNN_LAUNCH_CHECK();
    }
    return DGNN_OK;
  }
  if (!x || !w || !label || !loss || !lse) return DGNN_ERR_BAD_ARG;
  const int size = dtype == DGNN_F32 ? 4 : 2;
  if ((uintptr_t)x % size || (uintptr_t)w % size || (uintptr_t)label % label_bytes || ((uintptr_t)loss & 3) || ((uintptr_t)lse & 3))
    return DGNN_ERR_ALIGNMENT;
  const CePlan p = ce_plan(dtype, n, classes, d, x, w);
  if (!workspace || workspace_bytes < p.fwd_total) return DGNN_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return DGNN_ERR_ALIGNMENT;
  if (dtype == DGNN_F32) return ce_forward<float>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, loss, lse, (char *)workspace, st);
  if (dtype == DGNN_BF16) return ce_forward<bf16_t>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, loss, lse, (char *)workspace, st);
  return ce_forward<half_t>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, loss, lse, (char *)workspace, st);
}

int dgnn_linear_ce_backward(int dtype, int label_bytes, int n, int classes, int d, long long ignore_index, int reduction,
                            const void *x, const void *w, const void *label, const float *lse, const float *grad,
                            void *dx, void *dw, void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = ce_check(dtype, label_bytes, n, classes, d);
  if (rc != DGNN_OK) return rc;
  if (reduction < 0 || reduction > 2) return DGNN_ERR_BAD_ARG;
  if (!dx && !dw) return DGNN_OK;
  if (n == 0) return dw ? DGNN_ERR_BAD_ARG : DGNN_OK;
  if (!x || !w || !label || !lse || !grad) return DGNN_ERR_BAD_ARG;
  const int size = dtype == DGNN_F32 ? 4 : 2;
  if ((uintptr_t)x % size || (uintptr_t)w % size || (uintptr_t)dx % size || (uintptr_t)dw % size ||
      (uintptr_t)label % label_bytes || ((uintptr_t)lse & 3) || ((uintptr_t)grad & 3))
    return DGNN_ERR_ALIGNMENT;
  const CePlan p = ce_plan(dtype, n, classes, d, x, w);
  if (!workspace || workspace_bytes < p.bwd_total) return DGNN_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return DGNN_ERR_ALIGNMENT;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DGNN_F32) return ce_backward<float>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, lse, grad, dx, dw, (char *)workspace, st);
  if (dtype == DGNN_BF16) return ce_backward<bf16_t>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, lse, grad, dx, dw, (char *)workspace, st);
  return ce_backward<half_t>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, lse, grad, dx, dw, (char *)workspace, st);
}

}  // extern "C"
