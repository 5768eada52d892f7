// Packed attention: what the forward and the backward kernels share.
#pragma once
#include <string.h>

#include "mma.hpp"

namespace dgnn {

struct AttnArgs {
  const void *q, *k, *v, *out, *grad;         // grad: of the output
  void *o, *dq, *dk, *dv;
  void *rest;                                 // [tq, hq, d], what rounding took from the output (may be NULL)
  float *lse;                                 // [hq, tq], natural logarithm (backward: read)
  float *stat;                                // backward: [hq, tq] pairs {lse log2(e) - p_shift (+inf for an empty row), <grad, out>}
  float *part;                                // partial rows (split forward) or gradients (split backward)
  int few, chunk, splits;
  const int *row_ptr, *col_ptr;
  int nseq, tq, tk, hq, hk, g, d, causal;     // g = hq / hk
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head;   // strides in elements; o, grad, dq, dk, dv are contiguous
  float scale;
};

// Boundaries of the segments of `total` packed rows: 0, ptr[0], ..., ptr[nseq], total.  Segment 0 and
// segment nseq + 1 are the rows in front of the first and behind the last sequence, which belong to none.
__device__ __forceinline__ int seg_bound(const int *__restrict__ ptr, int nseq, int total, int s) {
  if (s <= 0) return 0;
  if (s >= nseq + 2) return total;
  return min(max(ptr[s - 1], 0), total);       // whatever ptr holds, no access leaves the tensors
}

struct Segment {
  int seq;                 // sequence, or -1 / nseq for rows that belong to none
  int start, len;          // first row and rows
  int tile;                // which tile of the segment, in units of `rows_per_tile` rows x g
};

// Workgroup -> tile without a list of tiles: segment s owns the tile slots from
// floor(bound(s) g / rows) + s up to the next segment's, at least as many as it has tiles (the spare
// ones find nothing to do).  by_row: the segment that holds row `slot` itself.  The segment of a slot is
// searched with 63 probes a step; the last step's probes are neighbours, so both of its bounds are in two
// lanes already.
__device__ __forceinline__ Segment find_segment(const int *__restrict__ ptr, int nseq, int total, int g, int rows,
                                                int slot, bool last_first, bool by_row = false) {
  int lo = 0, hi = nseq + 2, bound, n, step;
  const int lane = lane_id();
  do {
    step = (hi - lo + 62) / 63;
    const int s = min(lo + lane * step, hi);
    bound = seg_bound(ptr, nseq, total, s);
    n = __popcll(__ballot(s < hi && (unsigned)bound * (unsigned)g / (unsigned)rows + (by_row ? 0 : s) <= (unsigned)slot));
    n = max(n - 1, 0);
    if (step > 1) {
      lo += n * step;
      hi = min(hi, lo + step);
    }
  } while (step > 1);
  lo = uniform_i32(lo + n);
  Segment r;
  r.seq = lo - 1;
  r.start = __builtin_amdgcn_readlane(bound, n);
  r.len = max(__builtin_amdgcn_readlane(bound, n + 1) - r.start, 0);
  r.tile = slot - (int)((unsigned)r.start * (unsigned)g / (unsigned)rows + lo);
  const int tiles = (int)((r.len * (long long)g + rows - 1) / rows);
  if (r.tile < 0 || r.tile >= tiles) r.tile = -1;
  else if (last_first) r.tile = tiles - 1 - r.tile;
  return r;
}
static inline long long tile_slots(int total, int nseq, int g, int rows) {
  return (long long)total * g / rows + nseq + 2;
}
// How the rows of an index are dealt out.  Usually four waves share a tile of 128 packed rows and the tiles
// staged for it (a wave a workgroup is no better where those are fewer than the compute units: 2048 tokens, 8
// heads of 64, bfloat16, forward 33 us against 40).  Short sequences (96 packed rows on average or less): a wave
// alone has 32 rows, and four waves of a workgroup take four heads, since workgroups are then so many and so
// brief that starting them counts; one buffer, because more waves on a compute unit hide more than a
// second buffer (1024 graphs of 1 .. 63 nodes, 8 heads of 32, float: forward 38 us with two buffers, 33 with one).
static inline bool rows_short(int total, int nseq, int g) { return (long long)total * g <= 96LL * nseq; }
// Sequences of equal length leave a spare tile slot at a fixed period, and workgroups are dealt to the XCDs and
// their shader engines in turn: with every second slot spare, half of the card has all the work.  Every 32
// slots are therefore taken in an order of their own, rotated by 3 j mod 8 in the j-th 32: for no period
// up to eight do the rotations and the period cancel, as they would in steps of one for a period of three
// (training step, 512 sequences of 128 tokens, 8 heads of 64, bfloat16: 546 us without, 346 with; 1024 graphs of
// 32 nodes, 8 heads of 32, float: 175 and 126; of 64, two tiles and a spare slot: 301 and 303).
// Only where an eighth of the slots can be spare: long causal sequences are 4 % faster in plain order.
__device__ __forceinline__ int spread(int slot, int slots, int nseq) {
  return slots >> 3 < nseq + 2 && (slot | 31) < slots ? (slot & ~31) | ((slot + (3 * (slot >> 5) & 7)) & 31) : slot;
}
// Workgroup -> key head and tile slot (and split).  Neighbouring workgroups take neighbouring heads: they go to
// the eight XCDs in turn, so the tiles of one head meet in few of them.  HW > 1: wave w has the group's w-th head.
struct HeadSlot {
  int head, slot, split, wave;
};
template <int HW>
__device__ __forceinline__ HeadSlot head_slot(int hk, int nseq, int splits) {
  const int groups = (hk + HW - 1) / HW, wave = HW == 1 ? 0 : uniform_i32(wave_in_block());
  const int rest = blockIdx.x / groups;
  return {(int)(blockIdx.x % groups) * HW + wave, spread(rest / splits, (int)gridDim.x / groups / splits, nseq), rest % splits, wave};
}
// Rows of a segment's sequence in the other index: keys of its queries and the other way round.
__device__ __forceinline__ void other_side(const int *__restrict__ ptr, const int *__restrict__ own, int nseq, int total,
                                           const Segment &seg, int *start, int *len) {
  int s = 0, e = 0;
  if (seg.seq >= 0 && seg.seq < nseq) {
    if (ptr == own) {                          // self attention
      s = min(seg.start, total);
      e = min(seg.start + seg.len, total);
    } else {
      s = seg_bound(ptr, nseq, total, seg.seq + 1);
      e = seg_bound(ptr, nseq, total, seg.seq + 2);
    }
  }
  // into scalar registers whatever the compiler makes of the branches: a buffer descriptor in vector
  // registers costs a loop per load
  *start = uniform_i32(s);
  *len = uniform_i32(max(e - s, 0));
}

// A query row's (or key row's) DP / 16 fragments straight from global memory; columns behind d are zeros.
template <class T, int DP>
__device__ __forceinline__ void load_row_frags(frag8<T> (&f)[DP / 16], const T *row, int d, int h, bool valid) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int c = 16 * s + 8 * h;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[s][j] = (T)0.f;
    if constexpr (sizeof(T) == 2) {
      if (valid && c < d) f[s] = *(const frag8<T> *)(row + c);
    } else {
      if (valid && c < d) {
        const vec4<T> a = *(const vec4<T> *)(row + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[s][j] = a[j];
      }
      if (valid && c + 4 < d) {
        const vec4<T> a = *(const vec4<T> *)(row + c + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[s][4 + j] = a[j];
      }
    }
  }
}
// The transposed result blocks of a lane's row, times `by`, to global memory (d is a multiple of four); what
// the rounding to T took, rounded itself, to `rest`.
template <class T, int DP>
__device__ __forceinline__ void store_row(T *row, const acc16 (&c)[DP / 32], float by, int d, int h, T *rest = nullptr) {
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 32 * b + 8 * i + 4 * h;
      vec4<T> v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (T)(c[b][4 * i + j] * by);
      if (at < d) *(vec4<T> *)(row + at) = v;
      if (rest != nullptr && at < d) {
        vec4<T> lo;
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = (T)(c[b][4 * i + j] * by - (float)v[j]);
        *(vec4<T> *)(rest + at) = lo;
      }
    }
}

int attn_args(int dtype, int nseq, int tq, int tk, int hq, int hk, int d, int causal, float scale, const void *q,
              const void *k, const void *v, const int *row_ptr, const int *col_ptr, const long long *strides,
              AttnArgs *a);

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
#define DGNN_LOG2E 1.44269504088896340736f
#define DGNN_LN2 0.69314718055994530942f

}  // namespace dgnn
