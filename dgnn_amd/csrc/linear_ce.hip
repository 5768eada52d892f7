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
// Block of 4 waves, 2 x 2, each BM / 2 x BN / 2; operands are staged BK k elements at a time,
// double buffered.  An operand lies either with k along its rows (ROW: tile [BM][BK], read by row
// fragments) or with k down its columns (tile [BK][BM], read by transposing column fragments).
template <class T, int BM, int BN, int BK, bool AROW, bool BROW>
struct Gemm {
  static constexpr int THREADS = 256, MB = BM / 64, NB = BN / 64;      // 32 x 32 blocks of a wave
  using TA = Tile<T, AROW ? BK : BM>;
  using TB = Tile<T, BROW ? BK : BN>;
  static constexpr int A_BYTES = BM * BK * (int)sizeof(T), B_BYTES = BN * BK * (int)sizeof(T), S = 2;
  static constexpr int BYTES = A_BYTES + B_BYTES;      // of a stage

  // an operand: first element of the tile's rows (or columns), how many of them exist, row stride
  struct Operand {
    const T *p;
    int count;                    // rows (ROW) or columns that exist from p on
    unsigned stride;              // bytes between rows
  };

  // acc[m][n] += over k in [0, kn)
  __device__ static __forceinline__ void run(const Operand &a, const Operand &b, int kn, char *const (&lds)[S],
                                             acc16 (&acc)[MB][NB]) {
    const int lane = lane_id(), wave = uniform_i32(wave_in_block());
    const int m0 = (wave >> 1) * (BM / 2), n0 = (wave & 1) * (BN / 2);
    // two row operands: consecutive k; against a column operand the order is its transposing read's
    const int ra = AROW ? (BROW ? TA::row_lane(lane) : TA::row_lane_split(lane)) : TA::col_lane(lane);
    const int rb = BROW ? (AROW ? TB::row_lane(lane) : TB::row_lane_split(lane)) : TB::col_lane(lane);
    Stager<T, AROW ? BK : BM, AROW ? BM : BK, THREADS> sa;
    Stager<T, BROW ? BK : BN, BROW ? BN : BK, THREADS> sb;
    sa.init(a.stride, AROW ? min(BK, kn) : a.count);
    sb.init(b.stride, BROW ? min(BK, kn) : b.count);
    auto stage = [&](int t, auto i) {
      char *const ta = lds[i.value], *const tb = ta + A_BYTES;
      const int k0 = t * BK, left = max(0, min(BK, kn - k0));
      // rows end with a whole chunk (rows of dz are padded with zeros): a descriptor that ended inside one would
      // drop the dword the end falls into
      const unsigned row_bytes = (left * (unsigned)sizeof(T) + 15u) & ~15u;
      if (left < BK && left > 0 && k0 > 0) {                       // the last, shorter step
        if (AROW) sa.init(a.stride, left);
        if (BROW) sb.init(b.stride, left);
      }
      if (AROW)
        sa.load(ta, buffer_over(a.p + k0, span_bytes(left > 0 ? min(a.count, BM) : 0, a.stride, row_bytes)));
      else
        sa.load(ta, buffer_over((const char *)a.p + (long long)k0 * a.stride, span_bytes(left, a.stride, min(a.count, BM) * (unsigned)sizeof(T))));
      if (BROW)
        sb.load(tb, buffer_over(b.p + k0, span_bytes(left > 0 ? min(b.count, BN) : 0, b.stride, row_bytes)));
      else
        sb.load(tb, buffer_over((const char *)b.p + (long long)k0 * b.stride, span_bytes(left, b.stride, min(b.count, BN) * (unsigned)sizeof(T))));
    };
    auto work = [&](int, auto i) {
      const char *const ta = lds[i.value], *const tb = ta + A_BYTES;
#pragma unroll
      for (int k = 0; k < BK; k += 16) {
        frag8<T> fa[MB], fb[NB];
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if constexpr (AROW) fa[i] = BROW ? TA::row_frag(ta, ra, m0 + 32 * i, k) : TA::row_frag_split(ta, ra, m0 + 32 * i, k);
          else fa[i] = TA::col_frag(ta, ra, k, m0 + 32 * i);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          if constexpr (BROW) fb[i] = AROW ? TB::row_frag(tb, rb, n0 + 32 * i, k) : TB::row_frag_split(tb, rb, n0 + 32 * i, k);
          else fb[i] = TB::col_frag(tb, rb, k, n0 + 32 * i);
        }
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[i][j] = mma(fa[i], fb[j], acc[i][j]);
      }
    };
    ring<S, decltype(sa)::LOADS + decltype(sb)::LOADS>((kn + BK - 1) / BK, stage, work);
  }
};

// ------------------------------------------------------------------ labelled rows
template <class I>
__device__ __forceinline__ int class_of(const I *label, int i, int classes, long long ignore) {
  const long long x = label[i];
  return x != ignore && x >= 0 && x < classes ? (int)x : -1;
}

// list[j] = j-th labelled row, count[0] = how many; one workgroup, in order
template <class I>
__global__ __launch_bounds__(1024) void k_ce_rows(int n, int classes, long long ignore, const I *__restrict__ label,
                                                  int *__restrict__ list, int *__restrict__ count) {
  __shared__ int part[16];
  __shared__ int carry;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  const int lane = lane_id(), wave = wave_in_block();
  for (int base = 0; base < n; base += 1024) {
    const int i = base + threadIdx.x;
    const bool on = i < n && class_of(label, i, classes, ignore) >= 0;
    const unsigned long long b = __ballot(on);
    if (lane == 0) part[wave] = __popcll(b);
    __syncthreads();
    int at = carry;
    for (int w = 0; w < wave; ++w) at += part[w];
    if (on) list[at + __popcll(b & ((1ULL << lane) - 1))] = i;
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 0; w < 16; ++w) carry += part[w];
    __syncthreads();
  }
  if (threadIdx.x == 0) count[0] = carry;
}

// to[j, 0 .. ldt) = from[list[j], 0 .. d), zeros behind d; list == NULL: j itself.  j < count (count == NULL: n)
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_gather(int n, int d, int ldt, const int *__restrict__ list,
                                                          const int *__restrict__ count, const T *__restrict__ from,
                                                          long long ldf, int wide, T *__restrict__ to) {
  constexpr int VEC = 16 / sizeof(T);
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
  const void *x, *w;              // gathered rows [n, ldx], weight [classes, ldw]
  const void *label;
  const int *list, *count;
  int n, classes, d, dk;          // dk = d rounded up to whole chunks
  long long ldw;                  // elements
  int label_bytes;
  float *part_m, *part_s;         // [class tiles, n]
  float *z_label;                 // [n], by gathered row
  float *lse;                     // [n], by gathered row (backward: by original row)
  const float *grad;              // of the loss: n values or one
  int grad_rows, mean;
  const float *grad_top;          // one gradient a row: the largest magnitude
  void *dz;                       // [n, ldz]
  int v0, vn, ldz;                // piece of the classes
  float *acc;                     // split sums [splits][rows][d]
  int splits, first;
  void *dx, *dw;
};

__device__ __forceinline__ long long label_at(const CeArgs &a, int row) {
  return a.label_bytes == 8 ? ((const long long *)a.label)[row] : (long long)((const int *)a.label)[row];
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

template <class T> constexpr int ce_bk() { return sizeof(T) == 2 ? 64 : 32; }
constexpr int CE_BM = 128, CE_BN = 128;

// Forward: classes along m, rows along n.  Leaves the tile's maximum and sum of exp for every row and
// the logit of its label.
template <class T>
__global__ __launch_bounds__(256) void k_ce_fwd(const CeArgs a) {
  using G = Gemm<T, CE_BM, CE_BN, ce_bk<T>(), true, true>;
  DGNN_RING2(lds, G::BYTES);
  __shared__ float sm[2][CE_BN], ss[2][CE_BN];
  const int vt = blockIdx.x, v0 = vt * CE_BM, r0 = blockIdx.y * CE_BN;
  const int rows = min(a.n, *a.count);
  if (r0 >= rows) return;
  acc16 acc[G::MB][G::NB];
#pragma unroll
  for (int i = 0; i < G::MB; ++i)
#pragma unroll
    for (int j = 0; j < G::NB; ++j) acc[i][j] = acc_zero();
  G::run({(const T *)a.w + (long long)v0 * a.ldw, a.classes - v0, (unsigned)(a.ldw * sizeof(T))},
         {(const T *)a.x + (long long)r0 * a.dk, rows - r0, (unsigned)(a.dk * sizeof(T))}, a.dk, lds, acc);
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int m0 = v0 + (wave >> 1) * (CE_BM / 2), n0 = (wave & 1) * (CE_BN / 2);
#pragma unroll
  for (int j = 0; j < G::NB; ++j) {
    const int col = n0 + 32 * j + (lane & 31), r = r0 + col;
    const long long want = r < rows ? label_at(a, a.list[r]) : -1;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < G::MB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int v = m0 + 32 * i + acc_row(e, h);
        if (v == want) a.z_label[r] = acc[i][j][e];
        if (v >= a.classes) acc[i][j][e] = -INFINITY;
        top = fmaxf(top, acc[i][j][e]);
      }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == -INFINITY ? 0.f : top * DGNN_LOG2E;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < G::MB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], DGNN_LOG2E, -base));
    sum += __shfl_xor(sum, 32, 64);
    if (h == 0) sm[wave >> 1][col] = top, ss[wave >> 1][col] = sum;
  }
  __syncthreads();
  if (threadIdx.x < CE_BN && r0 + (int)threadIdx.x < rows) {
    const float m_a = sm[0][threadIdx.x], m_b = sm[1][threadIdx.x], top = fmaxf(m_a, m_b);
    const float base = top == -INFINITY ? 0.f : top;
    const float s = ss[0][threadIdx.x] * __builtin_amdgcn_exp2f((m_a - base) * DGNN_LOG2E) +
                    ss[1][threadIdx.x] * __builtin_amdgcn_exp2f((m_b - base) * DGNN_LOG2E);
    const long long at = (long long)vt * a.n + r0 + threadIdx.x;
    a.part_m[at] = top;
    a.part_s[at] = s;
  }
}

// lse and loss of every row from its tiles' pairs, one wave a gathered row; rows without a label get 0
// (they are not in the list, so the fill comes first)
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_fill(int n, float *__restrict__ loss, float *__restrict__ lse) {
  const int i = blockIdx.x * DGNN_BLOCK + threadIdx.x;
  if (i < n) {
    if (loss) loss[i] = 0.f;
    lse[i] = 0.f;
  }
}
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_join(int n, int tiles, const int *__restrict__ list,
                                                        const int *__restrict__ count, const float *__restrict__ pm,
                                                        const float *__restrict__ ps, const float *__restrict__ z_label,
                                                        float *__restrict__ loss, float *__restrict__ lse) {
  // 64 rows a workgroup, the tiles dealt to its four waves
  __shared__ float sm[DGNN_WAVES_PER_BLOCK][DGNN_WAVE], ss[DGNN_WAVES_PER_BLOCK][DGNN_WAVE];
  const int lane = lane_id(), wave = wave_in_block(), r = blockIdx.x * DGNN_WAVE + lane, rows = min(n, *count);
  if ((int)blockIdx.x * DGNN_WAVE >= rows) return;
  float m = -INFINITY, s = 0.f;
  if (r < rows)
    for (int t = wave; t < tiles; t += DGNN_WAVES_PER_BLOCK) {
      const float tm = pm[(long long)t * n + r], ts = ps[(long long)t * n + r], top = fmaxf(m, tm);
      const float base = top == -INFINITY ? 0.f : top;
      s = s * expf(m - base) + ts * expf(tm - base);
      m = top;
    }
  sm[wave][lane] = m, ss[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || r >= rows) return;
  float top = sm[0][lane];
  for (int w = 1; w < DGNN_WAVES_PER_BLOCK; ++w) top = fmaxf(top, sm[w][lane]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int w = 0; w < DGNN_WAVES_PER_BLOCK; ++w) sum += ss[w][lane] * expf(sm[w][lane] - base);
  const float v = base + logf(sum);
  lse[list[r]] = v;
  loss[list[r]] = v - z_label[r];
}
// out[0] = sum of the losses (/ labelled rows), in a fixed order; no labelled row: 0
__global__ __launch_bounds__(1024) void k_ce_reduce(int n, int mean, const int *__restrict__ count,
                                                    const float *__restrict__ loss, float *__restrict__ out) {
  __shared__ double part[16];
  double s = 0.;
  for (int i = threadIdx.x; i < n; i += 1024) s += (double)loss[i];
  for (int w = 32; w > 0; w >>= 1) s += __shfl_xor(s, w, 64);
  if (lane_id() == 0) part[wave_in_block()] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += part[w];
    out[0] = (float)(mean ? s / (double)max(1, *count) : s);
  }
}

// dz of a piece of the classes, [rows, ldz]; columns behind the piece's last class are zeros
template <class T>
__global__ __launch_bounds__(256) void k_ce_dz(const CeArgs a) {
  using G = Gemm<T, CE_BM, CE_BN, ce_bk<T>(), true, true>;
  DGNN_RING2(lds, G::BYTES);
  const int p0 = blockIdx.x * CE_BM, v0 = a.v0 + p0, r0 = blockIdx.y * CE_BN;
  const int rows = min(a.n, *a.count);
  if (r0 >= rows) return;
  acc16 acc[G::MB][G::NB];
#pragma unroll
  for (int i = 0; i < G::MB; ++i)
#pragma unroll
    for (int j = 0; j < G::NB; ++j) acc[i][j] = acc_zero();
  G::run({(const T *)a.w + (long long)v0 * a.ldw, a.classes - v0, (unsigned)(a.ldw * sizeof(T))},
         {(const T *)a.x + (long long)r0 * a.dk, rows - r0, (unsigned)(a.dk * sizeof(T))}, a.dk, lds, acc);
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int m0 = p0 + (wave >> 1) * (CE_BM / 2), n0 = (wave & 1) * (CE_BN / 2);
  const CeScale scale = ce_scale<T>(a, rows);
#pragma unroll
  for (int j = 0; j < G::NB; ++j) {
    const int r = r0 + n0 + 32 * j + (lane & 31);
    if (r >= rows) continue;
    const int row = a.list[r];
    const int want = (int)label_at(a, row) - a.v0;
    const float lse = a.lse[row] * DGNN_LOG2E;
    const float g = a.grad[a.grad_rows ? row : 0] * scale.by;
#pragma unroll
    for (int i = 0; i < G::MB; ++i)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int p = m0 + 32 * i + 8 * e4 + 4 * h;
        vec4<T> v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = __builtin_amdgcn_exp2f(fmaf(acc[i][j][4 * e4 + e], DGNN_LOG2E, -lse));
          if (p + e == want) y -= 1.f;
          v[e] = p + e < a.vn ? (T)(y * g) : (T)0.f;
        }
        if (p < a.ldz) *(vec4<T> *)((T *)a.dz + (long long)r * a.ldz + p) = v;
      }
  }
}

// Stores a lane's column of C^T (four consecutive m a group) to row `to`, columns m0 .. < d.
template <class T, int MB>
__device__ __forceinline__ void store_col(T *to, const acc16 (&c)[MB], float by, int m0, int d, int h, bool wide) {
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int at = m0 + 32 * i + 8 * e4 + 4 * h;
      if (wide) {
        vec4<T> v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(c[i][4 * e4 + e] * by);
        if (at < d) *(vec4<T> *)(to + at) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at + e < d) to[at + e] = (T)(c[i][4 * e4 + e] * by);
      }
    }
}

// dx of a piece: C^T[d, rows] += W_piece^T dz^T.  splits == 1 and one piece: straight to dx; else into
// acc[split], continued over the pieces, joined by k_ce_join_acc.
template <class T>
__global__ __launch_bounds__(256) void k_ce_dx(const CeArgs a) {
  constexpr int BK = ce_bk<T>();
  using G = Gemm<T, CE_BM, CE_BN, BK, false, true>;
  DGNN_RING2(lds, G::BYTES);
  const int c0 = blockIdx.x * CE_BM, r0 = blockIdx.y * CE_BN, split = blockIdx.z;
  const int rows = min(a.n, *a.count);
  if (r0 >= rows) return;
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int m0 = c0 + (wave >> 1) * (CE_BM / 2), n0 = (wave & 1) * (CE_BN / 2);
  acc16 acc[G::MB][G::NB];
#pragma unroll
  for (int j = 0; j < G::NB; ++j) {
    const int r = r0 + n0 + 32 * j + (lane & 31);
    const float *old = a.acc + ((long long)split * a.n + r) * a.dk;
#pragma unroll
    for (int i = 0; i < G::MB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int c = m0 + 32 * i + acc_row(e, h);
        acc[i][j][e] = !a.first && r < rows && c < a.dk ? old[c] : 0.f;
      }
  }
  const int steps = (a.vn + BK - 1) / BK, per = (steps + a.splits - 1) / a.splits;
  const int ka = min(a.vn, split * per * BK), kb = min(a.vn, (split + 1) * per * BK);
  G::run({(const T *)a.w + (long long)(a.v0 + ka) * a.ldw + c0, a.dk - c0, (unsigned)(a.ldw * sizeof(T))},
         {(const T *)a.dz + (long long)r0 * a.ldz + ka, rows - r0, (unsigned)(a.ldz * sizeof(T))}, kb - ka, lds, acc);
#pragma unroll
  for (int j = 0; j < G::NB; ++j) {
    const int r = r0 + n0 + 32 * j + (lane & 31);
    acc16 col[G::MB];
#pragma unroll
    for (int i = 0; i < G::MB; ++i) col[i] = acc[i][j];
    if (r < rows) store_col<float, G::MB>(a.acc + ((long long)split * a.n + r) * a.dk, col, 1.f, m0, a.dk, h, true);
  }
}
// dx[list[r]] = sum over the splits, in order
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_dx_join(const CeArgs a) {
  const int rows = min(a.n, *a.count), per = a.dk / 4;
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
// rows without a label: dx = 0
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_ce_dx_zero(const CeArgs a, long long ignore) {
  for (int r = blockIdx.x; r < a.n; r += gridDim.x) {
    const long long x = label_at(a, r);
    if (x != ignore && x >= 0 && x < a.classes) continue;
    for (int c = threadIdx.x; c < a.d; c += DGNN_BLOCK) ((T *)a.dx)[(long long)r * a.d + c] = (T)0.f;
  }
}

// dW of a piece: C^T[d, classes of the piece] = x^T dz.  splits > 1: partial sums over shares of the rows.
template <class T>
__global__ __launch_bounds__(256) void k_ce_dw(const CeArgs a, int wide) {
  constexpr int BK = ce_bk<T>();
  using G = Gemm<T, CE_BM, CE_BN, BK, false, false>;
  DGNN_RING2(lds, G::BYTES);
  const int c0 = blockIdx.x * CE_BM, p0 = blockIdx.y * CE_BN, split = blockIdx.z;
  const int rows = min(a.n, *a.count);
  acc16 acc[G::MB][G::NB];
#pragma unroll
  for (int i = 0; i < G::MB; ++i)
#pragma unroll
    for (int j = 0; j < G::NB; ++j) acc[i][j] = acc_zero();
  const int steps = (rows + BK - 1) / BK, per = (steps + a.splits - 1) / a.splits;
  const int ka = min(rows, split * per * BK), kb = min(rows, (split + 1) * per * BK);
  G::run({(const T *)a.x + (long long)ka * a.dk + c0, a.dk - c0, (unsigned)(a.dk * sizeof(T))},
         {(const T *)a.dz + (long long)ka * a.ldz + p0, a.ldz - p0, (unsigned)(a.ldz * sizeof(T))}, kb - ka, lds, acc);
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int m0 = c0 + (wave >> 1) * (CE_BM / 2), n0 = (wave & 1) * (CE_BN / 2);
  const float unit = ce_scale<T>(a, rows).unit;
#pragma unroll
  for (int j = 0; j < G::NB; ++j) {
    const int p = p0 + n0 + 32 * j + (lane & 31);
    acc16 col[G::MB];
#pragma unroll
    for (int i = 0; i < G::MB; ++i) col[i] = acc[i][j];
    if (p >= a.vn) continue;
    if (a.splits == 1) store_col<T, G::MB>((T *)a.dw + (long long)(a.v0 + p) * a.d, col, unit, m0, a.d, h, wide != 0);
    else store_col<float, G::MB>(a.acc + ((long long)split * a.ldz + p) * a.dk, col, 1.f, m0, a.dk, h, true);
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

struct CePlan {
  int dk, tiles, copy_w;                              // class tiles of the forward
  size_t list, x, w, part, zl, lossrow, fwd_total;    // bytes
  int piece, ldz, dx_splits, dw_splits;
  size_t dz, dxacc, dwacc, bwd_total;
};
static CePlan ce_plan(int dtype, int n, int classes, int d, int aligned_w) {
  CePlan p;
  memset(&p, 0, sizeof(p));
  const int size = dtype == DGNN_F32 ? 4 : 2, vec = 16 / size;
  p.dk = (d + vec - 1) / vec * vec;
  p.copy_w = !aligned_w || p.dk != d;
  p.tiles = ceil_div(classes, CE_BM);
  p.list = align256(sizeof(int) * ((size_t)n + 1));
  p.x = align256((size_t)n * p.dk * size);
  p.w = p.copy_w ? align256((size_t)classes * p.dk * size) : 0;
  p.part = align256(sizeof(float) * (size_t)p.tiles * n);
  p.zl = align256(sizeof(float) * (size_t)n);
  p.lossrow = p.zl;
  p.fwd_total = p.list + p.x + p.w + 2 * p.part + 2 * p.zl;
  // pieces: dz of about 256 MB, whole tiles
  long long cols = (256LL << 20) / ((long long)size * (n > 0 ? n : 1));
  cols = cols < 1024 ? 1024 : cols;
  if (cols > (1 << 20)) cols = 1 << 20;        // 128 rows of a piece stay inside 32-bit offsets
  if (cols > classes) cols = classes;
  const int pieces = ceil_div(classes, cols);
  p.piece = ceil_div(ceil_div(classes, pieces), CE_BM) * CE_BM;
  p.ldz = p.piece;
  // enough workgroups for 256 compute units: split the long axis while tiles are few
  const long long dx_tiles = (long long)ceil_div(p.dk, CE_BM) * ceil_div(n, CE_BN);
  const long long dw_tiles = (long long)ceil_div(p.dk, CE_BM) * ceil_div(p.piece, CE_BN);
  auto splits = [](long long tiles, int steps) {
    long long s = tiles > 0 ? 512 / tiles : 1;
    if (s > steps / 4) s = steps / 4;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
  };
  p.dx_splits = splits(dx_tiles, p.piece / 64);
  p.dw_splits = splits(dw_tiles, n / 64);
  p.dz = align256((size_t)n * p.ldz * size);
  p.dxacc = align256(sizeof(float) * (size_t)p.dx_splits * n * p.dk);
  p.dwacc = p.dw_splits > 1 ? align256(sizeof(float) * (size_t)p.dw_splits * p.ldz * p.dk) : 0;
  p.bwd_total = p.list + p.x + p.w + p.dz + p.dxacc + p.dwacc + 256;
  return p;
}

static int ce_check(int dtype, int label_bytes, int n, int classes, int d) {
  if (dtype < 0 || dtype > 2 || (label_bytes != 4 && label_bytes != 8) || n < 0 || classes <= 0 || d <= 0) return DGNN_ERR_BAD_ARG;
  if (d > 65536 || n > (1 << 22) || classes > (1 << 30)) return DGNN_ERR_UNSUPPORTED;
  return DGNN_OK;
}

// labelled rows -> list, count, gathered x; padded weight where its rows are not whole chunks
template <class T>
static int ce_prepare(const CePlan &p, int n, int classes, int d, const void *x, const void *w, const void *label,
                      int label_bytes, long long ignore, char *ws, CeArgs *a, hipStream_t st) {
  int *list = (int *)ws, *count = list + n;
  T *xc = (T *)(ws + p.list), *wc = (T *)(ws + p.list + p.x);
  if (label_bytes == 8)
    hipLaunchKernelGGL(k_ce_rows<long long>, dim3(1), dim3(1024), 0, st, n, classes, ignore, (const long long *)label, list, count);
  else
    hipLaunchKernelGGL(k_ce_rows<int>, dim3(1), dim3(1024), 0, st, n, classes, ignore, (const int *)label, list, count);
  DGNN_LAUNCH_CHECK();
  const int per = p.dk / (16 / (int)sizeof(T));
  hipLaunchKernelGGL(k_ce_gather<T>, dim3(grid_for((long long)n * per)), dim3(DGNN_BLOCK), 0, st, n, d, p.dk,
                     (const int *)list, (const int *)count, (const T *)x, (long long)d,
                     (int)(p.dk == d && ((uintptr_t)x & 15) == 0), xc);
  DGNN_LAUNCH_CHECK();
  if (p.copy_w) {
    hipLaunchKernelGGL(k_ce_gather<T>, dim3(grid_for((long long)classes * per)), dim3(DGNN_BLOCK), 0, st, classes, d, p.dk,
                       (const int *)nullptr, (const int *)nullptr, (const T *)w, (long long)d, 0, wc);
    DGNN_LAUNCH_CHECK();
  }
  memset(a, 0, sizeof(*a));
  a->x = xc, a->w = p.copy_w ? (const void *)wc : w;
  a->ldw = p.dk;
  a->label = label, a->label_bytes = label_bytes, a->list = list, a->count = count;
  a->n = n, a->classes = classes, a->d = d, a->dk = p.dk;
  return DGNN_OK;
}

template <class T>
static int ce_forward(const CePlan &p, int n, int classes, int d, const void *x, const void *w, const void *label,
                      int label_bytes, long long ignore, int reduction, float *loss, float *lse, char *ws, hipStream_t st) {
  CeArgs a;
  const int rc = ce_prepare<T>(p, n, classes, d, x, w, label, label_bytes, ignore, ws, &a, st);
  if (rc != DGNN_OK) return rc;
  char *at = ws + p.list + p.x + p.w;
  a.part_m = (float *)at, a.part_s = (float *)(at + p.part), a.z_label = (float *)(at + 2 * p.part);
  float *row = reduction == 0 ? loss : (float *)(at + 2 * p.part + p.zl);
  hipLaunchKernelGGL(k_ce_fill, dim3(ceil_div(n, DGNN_BLOCK)), dim3(DGNN_BLOCK), 0, st, n, row, lse);
  DGNN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_ce_fwd<T>, dim3(p.tiles, ceil_div(n, CE_BN)), dim3(256), 0, st, a);
  DGNN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_ce_join, dim3(ceil_div(n, DGNN_WAVE)), dim3(DGNN_BLOCK), 0, st, n, p.tiles, a.list, a.count,
                     (const float *)a.part_m, (const float *)a.part_s, (const float *)a.z_label, row, lse);
  DGNN_LAUNCH_CHECK();
  if (reduction != 0) {
    hipLaunchKernelGGL(k_ce_reduce, dim3(1), dim3(1024), 0, st, n, (int)(reduction == 1), a.count, (const float *)row, loss);
    DGNN_LAUNCH_CHECK();
  }
  return DGNN_OK;
}

template <class T>
static int ce_backward(const CePlan &p, int n, int classes, int d, const void *x, const void *w, const void *label,
                       int label_bytes, long long ignore, int reduction, const float *lse, const float *grad, void *dx,
                       void *dw, char *ws, hipStream_t st) {
  CeArgs a;
  const int rc = ce_prepare<T>(p, n, classes, d, x, w, label, label_bytes, ignore, ws, &a, st);
  if (rc != DGNN_OK) return rc;
  char *at = ws + p.list + p.x + p.w;
  a.dz = at, a.ldz = p.ldz;
  float *dxacc = (float *)(at + p.dz), *dwacc = (float *)(at + p.dz + p.dxacc);
  a.lse = (float *)lse, a.grad = grad, a.grad_rows = reduction == 0, a.mean = reduction == 1;
  a.dx = dx, a.dw = dw;
  if (a.grad_rows) {
    float *top = (float *)(at + p.dz + p.dxacc + p.dwacc);
    hipLaunchKernelGGL(k_ce_grad_top, dim3(1), dim3(1024), 0, st, n, a.list, a.count, grad, top);
    DGNN_LAUNCH_CHECK();
    a.grad_top = top;
  }
  const int wide = d % 4 == 0 && ((uintptr_t)dw & (4 * sizeof(T) - 1)) == 0;
  for (int v0 = 0; v0 < classes; v0 += p.piece) {
    a.v0 = v0, a.vn = classes - v0 < p.piece ? classes - v0 : p.piece, a.first = v0 == 0;
    hipLaunchKernelGGL(k_ce_dz<T>, dim3(p.piece / CE_BM, ceil_div(n, CE_BN)), dim3(256), 0, st, a);
    DGNN_LAUNCH_CHECK();
    if (dx) {
      a.acc = dxacc, a.splits = p.dx_splits;
      hipLaunchKernelGGL(k_ce_dx<T>, dim3(ceil_div(p.dk, CE_BM), ceil_div(n, CE_BN), p.dx_splits), dim3(256), 0, st, a);
      DGNN_LAUNCH_CHECK();
    }
    if (dw) {
      a.acc = dwacc, a.splits = p.dw_splits;
      hipLaunchKernelGGL(k_ce_dw<T>, dim3(ceil_div(p.dk, CE_BM), ceil_div(a.vn, CE_BN), p.dw_splits), dim3(256), 0, st, a, wide);
      DGNN_LAUNCH_CHECK();
      if (p.dw_splits > 1) {
        hipLaunchKernelGGL(k_ce_dw_join<T>, dim3(grid_for((long long)a.vn * p.dk / 4)), dim3(DGNN_BLOCK), 0, st, a);
        DGNN_LAUNCH_CHECK();
      }
    }
  }
  if (dx) {
    a.acc = dxacc, a.splits = p.dx_splits;
    hipLaunchKernelGGL(k_ce_dx_zero<T>, dim3(n < 4096 ? n : 4096), dim3(DGNN_BLOCK), 0, st, a, ignore);
    DGNN_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_ce_dx_join<T>, dim3(grid_for((long long)n * p.dk / 4)), dim3(DGNN_BLOCK), 0, st, a);
    DGNN_LAUNCH_CHECK();
  }
  return DGNN_OK;
}

}  // namespace dgnn

extern "C" {

size_t dgnn_linear_ce_workspace_bytes(int dtype, int n, int classes, int d, int backward) {
  if (ce_check(dtype, 4, n, classes, d) != DGNN_OK || n == 0) return 0;
  const CePlan p = ce_plan(dtype, n, classes, d, 0);
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
      hipLaunchKernelGGL(k_ce_reduce, dim3(1), dim3(1024), 0, st, 0, 0, (const int *)nullptr, (const float *)nullptr, loss);
      DGNN_LAUNCH_CHECK();
    }
    return DGNN_OK;
  }
  if (!x || !w || !label || !loss || !lse) return DGNN_ERR_BAD_ARG;
  const int size = dtype == DGNN_F32 ? 4 : 2;
  if ((uintptr_t)x % size || (uintptr_t)w % size || (uintptr_t)label % label_bytes || ((uintptr_t)loss & 3) || ((uintptr_t)lse & 3))
    return DGNN_ERR_ALIGNMENT;
  const CePlan p = ce_plan(dtype, n, classes, d, ((uintptr_t)w & 15) == 0);
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
  const CePlan p = ce_plan(dtype, n, classes, d, ((uintptr_t)w & 15) == 0);
  if (!workspace || workspace_bytes < p.bwd_total) return DGNN_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return DGNN_ERR_ALIGNMENT;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DGNN_F32) return ce_backward<float>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, lse, grad, dx, dw, (char *)workspace, st);
  if (dtype == DGNN_BF16) return ce_backward<bf16_t>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, lse, grad, dx, dw, (char *)workspace, st);
  return ce_backward<half_t>(p, n, classes, d, x, w, label, label_bytes, ignore_index, reduction, lse, grad, dx, dw, (char *)workspace, st);
}

}  // extern "C"
