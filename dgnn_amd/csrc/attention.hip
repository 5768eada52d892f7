// Packed attention, forward: every query row of a sequence against the keys of the same sequence.
//
//   z_ij = scale <q_i, k_j>,  p_ij = exp(z_ij - lse_i),  o_i = sum_j p_ij v_j
//
// over the keys the mask leaves (all of the sequence, or j <= i + keys - queries); a row whose mask
// leaves none gives o = 0, lse = -inf.
//
// One workgroup of NW waves owns 32 NW packed rows of one key head: row r is query r / g, head r % g of the
// g query heads that share the key head, so a key tile staged in LDS serves all of them.  The products are
// formed transposed, Z^T = K Q^T and O^T += V^T P^T: a lane then owns one query row, the softmax runs
// inside the lane (one exchange with lane + 32 for the maximum), the rescaling factor is a lane's scalar,
// and the 16 weights a lane holds are, unmoved, its operand of the second product (mma.hpp).
// Key tiles are double buffered, loaded straight to LDS while the previous tile is worked on.
//
// Bound by the matrix instructions and, next to them, the exponentials (one a score against 4 d operations), under
// the power limit that large 16-bit products run into too: 16384 tokens, causal, 16 / 2 heads of 128, float16
// 1.10 ms, 1000 TFLOP/s (a large matrix product reaches 1125); 32 x 2048 tokens, 8 heads of 64, bfloat16
// 0.37 - 0.42 ms, 650 - 740 TFLOP/s.  Weights are rounded to T for the second product, half a step each; their sum is
// of the unrounded ones, in float like every sum here.
#include "attention.hpp"

using namespace dgnn;

namespace dgnn {

// One tile: 32 NW packed rows row0 .. of a sequence (`rows` of them exist) against its keys key0 .. key1 - 1.
// Leaves the lane's unnormalised output row in acc, the reference its weights are relative to (near the maximum
// of z / scale) in m and their sum in l.
template <class T, int DP, int NW, int BN, int S>
struct AttnTile {
  using TL = Tile<T, DP>;
  using SG = Stager<T, DP, BN, 64 * NW>;
  static constexpr int TILE = BN * TL::ROW_BYTES, BYTES = 2 * TILE;
  // log2 of the weight of a score at the reference.  float16: 7, weights then run up to 2^15 and lose nothing before 2^-21
  // of it; at 0, 262144 keys 2^-26 below one other vanished in front of the second product, 0.4 % of the row's sum.
  static constexpr float UP = std::is_same<T, half_t>::value ? 7.f : 0.f;
  static_assert(S == 1 || 2 * SG::LOADS * (S - 2) < 64, "loads in flight are counted in six bits");

  acc16 acc[DP / 32];
  float m, l, c;
  bool valid;
  int head, limit;
  long long tok;

  __device__ __forceinline__ void run(const AttnArgs &a, const lds_ptr (&lds)[4], int qs, int lq, int ks, int lk, int kvh,
                                      long long row0, long long rows, int key0, int key1) {
    const int lane = lane_id(), h = lane >> 5, wave = NW == 1 ? 0 : uniform_i32(wave_in_block());
    const int row_lane = TL::row_lane(lane), col_lane = TL::col_lane(lane);
    // this lane's row
    const long long wrow = row0 + wave * 32, row = wrow + (lane & 31);
    valid = row < rows;
    const int qi = (int)((unsigned)row / (unsigned)a.g);
    head = kvh * a.g + (int)((unsigned)row % (unsigned)a.g);
    tok = qs + (long long)qi;
    // last key it sees; causal: queries and keys end together
    const int shift = lk - lq;
    limit = !valid ? -1 : a.causal ? qi + shift : lk - 1;
    const int last_row = (int)(min(rows, row0 + 32 * NW) - 1);
    const int seen = a.causal ? max(0, min(key1, last_row / a.g + shift + 1)) : key1;
    const int tiles = (max(seen - key0, 0) + BN - 1) / BN;
    // every row of the wave sees the keys up to wave_all, none sees a key behind wave_any
    const int wave_all = a.causal ? min((int)wrow, last_row) / a.g + shift : lk - 1;
    const int wave_any = wrow > last_row ? -1 : a.causal ? min((int)wrow + 31, last_row) / a.g + shift : lk - 1;

    frag8<T> qf[DP / 16];
    load_row_frags<T, DP>(qf, (const T *)a.q + tok * a.q_tok + (long long)head * a.q_head, a.d, h, valid);
    c = a.scale * DGNN_LOG2E;
    // the running maximum is taken before the scale, which must be positive there: the sign goes into
    // q, and a scale of zero becomes q = 0 (a masked score, -inf, stays -inf)
    if (!(c > 0.f)) {
      const bool zero = c == 0.f;
      c = zero ? 1.f : -c;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[s][j] = zero ? (T)0.f : (T)-qf[s][j];
    }

    const unsigned k_stride = (unsigned)(a.k_tok * sizeof(T)), v_stride = (unsigned)(a.v_tok * sizeof(T));
    const unsigned row_bytes = a.d * (unsigned)sizeof(T);
    const T *kbase = (const T *)a.k + (long long)(ks + (long long)key0) * a.k_tok + (long long)kvh * a.k_head;
    const T *vbase = (const T *)a.v + (long long)(ks + (long long)key0) * a.v_tok + (long long)kvh * a.v_head;
    SG st_k, st_v;
    st_k.init(k_stride, a.d);
    st_v.init(v_stride, a.d);
    auto stage = [&](int t, auto i) {
      const int n = t < tiles ? min(BN, key1 - key0 - t * BN) : 0;
      st_k.load(lds[i.value], buffer_over(kbase + (long long)t * BN * a.k_tok, span_bytes(n, k_stride, row_bytes)));
      st_v.load(lds[i.value] + TILE, buffer_over(vbase + (long long)t * BN * a.v_tok, span_bytes(n, v_stride, row_bytes)));
    };

#pragma unroll
    for (int b = 0; b < DP / 32; ++b) acc[b] = acc_zero();
    m = -INFINITY, l = 0.f;

    auto work = [&](int t, auto i) {
      const lds_ptr kt = lds[i.value], vt = kt + TILE;
      const int k0 = key0 + t * BN;
      if (k0 > wave_any) return;
      const int rl = opaque(row_lane), cl = opaque(col_lane);
      acc16 s[BN / 32];
#pragma unroll
      for (int b = 0; b < BN / 32; ++b) {
        s[b] = acc_zero();
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) s[b] = mma(TL::row_frag(kt, rl, 32 * b, 16 * k), qf[k], s[b]);
      }
      if (k0 + BN - 1 > min(wave_all, key1 - 1)) {
        const int last = min(limit, key1 - 1) - k0;
#pragma unroll
        for (int b = 0; b < BN / 32; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * b + acc_row(r, h) > last) s[b][r] = -INFINITY;
      }
      float top = m;
#pragma unroll
      for (int b = 0; b < BN / 32; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      // m is a reference near the maximum, not the maximum itself: it moves only when a score exceeds it by more
      // than 8 (in log2), so weights run up to 256 (times 2^UP), far from any type's end, and most tiles rescale nothing.
      // With 32 rows a wave one of them has a new maximum in nearly every tile of some thousand keys.
      if (__any((top - m) * c > 8.f)) {
        const float by = top == m ? 1.f : exp2_fast((m - top) * c);     // m = -inf: 0
        m = top;
        l *= by;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[b][r] *= by;
      }
      const float mc = m == -INFINITY ? 0.f : base();
#pragma unroll
      for (int b = 0; b < BN / 32; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[b][r] = exp2_fast(fmaf(s[b][r], c, -mc));
          l += s[b][r];
        }
#pragma unroll
      for (int k = 0; k < BN / 16; ++k) {
        const frag8<T> p = frag_of<T>(s[k >> 1], 8 * (k & 1));
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) acc[b] = mma(TL::col_frag(vt, cl, 16 * k, 32 * b), p, acc[b]);
      }
    };
    ring<S, 2 * SG::LOADS, NW == 1>(tiles, stage, work);
    l += __shfl_xor(l, 32, 64);
  }

  // what the scores' exponents are relative to
  __device__ __forceinline__ float base() const { return m * c - UP; }

  __device__ __forceinline__ void finish(const AttnArgs &a, int lk) {
    if (!valid) return;
    const int h = lane_id() >> 5;
    const bool none = limit < 0 || lk == 0;
    if (none) {                                 // not by a factor: weights of zero times a NaN of a row nobody sees is one
#pragma unroll
      for (int b = 0; b < DP / 32; ++b) acc[b] = acc_zero();
    }
    const long long to = (tok * a.hq + head) * a.d;
    store_row<T, DP>((T *)a.o + to, acc, none ? 0.f : 1.f / l, a.d, h, a.rest != nullptr ? (T *)a.rest + to : nullptr);
    if (a.lse != nullptr && h == 0)
      a.lse[(long long)head * a.tq + tok] = none ? -INFINITY : (base() + __builtin_amdgcn_logf(l)) * DGNN_LN2;
  }
};

template <class T, int DP, int NW, int HW, int BN, int S>
__global__ __launch_bounds__(64 * NW * HW, sizeof(T) == 2 ? 2 : 1) void k_attn_fwd(const AttnArgs a) {
  using AT = AttnTile<T, DP, NW, BN, S>;
  DGNN_RING(all, HW * AT::BYTES);
  const int splits = NW > 1 ? a.splits : 1;
  const HeadSlot at = head_slot<HW>(a.hk, a.nseq, splits);
  if (at.head >= a.hk) return;
  const int kvh = at.head;
  const lds_ptr lds[4] = {all[0] + at.wave * AT::BYTES, all[1] + at.wave * AT::BYTES, all[2] + at.wave * AT::BYTES, all[3] + at.wave * AT::BYTES};
  const Segment seg = find_segment(a.row_ptr, a.nseq, a.tq, a.g, 32 * NW, at.slot, a.causal != 0);
  if (seg.tile < 0) return;
  int ks, lk;
  other_side(a.col_ptr, a.row_ptr, a.nseq, a.tk, seg, &ks, &lk);
  const long long row0 = (long long)seg.tile * 32 * NW, rows = (long long)seg.len * a.g;
  int key0 = 0, key1 = lk;
  if (NW > 1 && splits > 1) {                   // an equal share of the keys that the tile's last row sees
    const int seen = a.causal ? min(lk, (int)((min(rows, row0 + 32 * NW) - 1) / a.g) + lk - seg.len + 1) : lk;
    const int per = ((max(seen, 0) + BN - 1) / BN + splits - 1) / splits * BN;
    key0 = uniform_i32(min(at.split * per, lk)), key1 = uniform_i32(min(lk, key0 + per));
  }
  AT t;
  t.run(a, lds, seg.start, seg.len, ks, lk, kvh, row0, rows, key0, key1);
  if (NW == 1 || splits == 1) {
    t.finish(a, lk);
    return;
  }
  if (!t.valid) return;
  float *part = a.part + (((long long)at.split * a.tq + t.tok) * a.hq + t.head) * (a.d + 4);
  store_row<float, DP>(part + 4, t.acc, 1.f, a.d, lane_id() >> 5);
  if (lane_id() < 32) part[0] = t.m == -INFINITY ? -INFINITY : t.base(), part[1] = t.l, part[2] = t.limit >= 0 && lk > 0 ? 1.f : 0.f;
}
// out and lse from the splits' {maximum, sum, whether the row sees a key, -, output}, in order.  One wave a row.
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_attn_merge(const AttnArgs a) {
  const int lane = lane_id();
  const long long r = (long long)blockIdx.x * DGNN_WAVES_PER_BLOCK + uniform_i32(wave_in_block()), stride = (long long)a.tq * a.hq * (a.d + 4);
  if (r >= (long long)a.tq * a.hq) return;
  const float *part = a.part + r * (a.d + 4);
  float top = -INFINITY, sum = 0.f;
  for (int j = 0; j < a.splits; ++j) top = fmaxf(top, part[j * stride]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int j = 0; j < a.splits; ++j) sum = fmaf(part[j * stride + 1], exp2_fast(part[j * stride] - base), sum);
  const bool any = part[2] != 0.f;
  T *out = (T *)a.o + r * a.d;
  for (int c = lane; c < a.d; c += 64) {
    float x = 0.f;
    for (int j = 0; j < a.splits; ++j) x = fmaf(part[j * stride + 4 + c], exp2_fast(part[j * stride] - base), x);
    x = any ? x / sum : 0.f;
    out[c] = (T)x;
    if (a.rest != nullptr) ((T *)a.rest)[r * a.d + c] = (T)(x - (float)(T)x);
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[r % a.hq * a.tq + r / a.hq] = any ? (base + __builtin_amdgcn_logf(sum)) * DGNN_LN2 : -INFINITY;
}

// ------------------------------------------------------------------ few rows, long keys
typedef float f32x4 __attribute__((ext_vector_type(4)));
// a 4 x 1 (lane 4 b + i: row i of block b) times 1 x 4 in sixteen blocks; every group of 2^CB blocks takes the
// first operand of its block BLOCK
template <int CB, int BLOCK>
__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_4x4x1f32(a, b, c, CB, BLOCK, 0);
}
// The same as AttnTile for up to four rows of floats: its float matrix instructions take 32 rows whether they
// are there or not, and bound it at half the memory's rate.  Blocks of 4 x 4 lose nothing (single queries of 32 / 8
// heads of 128: 9 sequences of 32768 keys 418 us against 755, 5.8 TB/s; 16 of 1024 39 against 89).  A tile
// is 32 keys.  Scores: a lane has a key and half of the dims, so blocks 0 - 7 and 8 - 15 take their own dims of q
// and the halves are added.  Output: a lane has DP / 64 columns, and the weights, turned in LDS, are the
// broadcast operand; DP = 32: a column and half of the keys.  Rows lie in the four elements of z and acc.
template <int DP>
struct AttnFour {
  using TL = Tile<float, DP>;
  using SG = Stager<float, DP, 32, 64>;
  static constexpr int TILE = 32 * TL::ROW_BYTES, BYTES = 2 * TILE, VC = DP >= 64 ? DP / 64 : 1;
  static constexpr bool HALVES = DP == 32;      // of the keys, for the output
  f32x4 acc[VC], m, l;                          // l: this lane's share
  float c;

  __device__ __forceinline__ void run(const AttnArgs &a, const lds_ptr (&lds)[4], lds_ptr turn, int qs, int lq, int ks, int lk,
                                      int kvh, int rows, int key0, int key1) {
    const int lane = lane_id(), h = lane >> 5;
    const int k_lane = TL::chunk_addr(lane & 31, h * (DP / 8)), v_lane = HALVES ? TL::chunk_addr(16 * h, (lane & 31) / 4) + lane % 4 * 4 : lane * VC * 4;
    const int shift = lk - lq;
    int last[4], seen = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      last[r] = r >= rows ? -1 : a.causal ? min(key1 - 1, r / a.g + shift) : key1 - 1;
      seen = max(seen, last[r] + 1);
    }
    const int tiles = (max(seen - key0, 0) + 31) / 32;
    c = a.scale * DGNN_LOG2E;
    const float sign = c > 0.f ? 1.f : c < 0.f ? -1.f : 0.f;         // as in AttnTile (NaN: q and c as they are)
    c = sign == 0.f ? (c == 0.f ? 1.f : c) : c * sign;
    float q[DP / 16];
    {
      const int r = lane & 3, b = lane >> 2;
      const float *row = (const float *)a.q + (qs + (long long)(r / a.g)) * a.q_tok + (long long)(kvh * a.g + r % a.g) * a.q_head;
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) {
        const int at = (DP / 2) * (b >> 3) + 8 * j + (b & 7);
        q[j] = r < rows && at < a.d ? row[at] * sign : 0.f;
      }
    }
    const unsigned k_stride = (unsigned)(a.k_tok * 4), v_stride = (unsigned)(a.v_tok * 4), row_bytes = a.d * 4u;
    const float *kbase = (const float *)a.k + (ks + (long long)key0) * a.k_tok + (long long)kvh * a.k_head;
    const float *vbase = (const float *)a.v + (ks + (long long)key0) * a.v_tok + (long long)kvh * a.v_head;
    SG st_k, st_v;
    st_k.init(k_stride, a.d);
    st_v.init(v_stride, a.d);
    auto stage = [&](int t, auto i) {
      const int n = t < tiles ? min(32, key1 - key0 - t * 32) : 0;
      st_k.load(lds[i.value], buffer_over(kbase + (long long)t * 32 * a.k_tok, span_bytes(n, k_stride, row_bytes)));
      st_v.load(lds[i.value] + TILE, buffer_over(vbase + (long long)t * 32 * a.v_tok, span_bytes(n, v_stride, row_bytes)));
    };
#pragma unroll
    for (int v = 0; v < VC; ++v) acc[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY}, l = f32x4{0.f, 0.f, 0.f, 0.f};
    auto work = [&](int t, auto i) {
      const lds_ptr kt = lds[i.value], vt = kt + TILE;
      const int key = key0 + 32 * t + (lane & 31);
      f32x4 z[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      unrolled<0, DP / 8>([&](auto n) {
        constexpr int C = n.value;
        const f32x4 k = *(const DGNN_LDS f32x4 *)TL::at(kt, k_lane, 0, C);
        unrolled<0, 4>([&](auto e) { z[e.value & 1] = mma4<3, 4 * (C & 1) + e.value>(q[C / 2], k[e.value], z[e.value & 1]); });
      });
      f32x4 p;
      bool above = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float s = z[0][r] + z[1][r], both = s + __shfl_xor(s, 32, 64);
        p[r] = key <= last[r] ? both : -INFINITY;
        above |= (p[r] - m[r]) * c > 8.f;
      }
      if (__any(above)) {                       // a reference near the maximum, as in AttnTile
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float top = wave_max(fmaxf(m[r], p[r])), by = top == m[r] ? 1.f : exp2_fast((m[r] - top) * c);
          m[r] = top, l[r] *= by;
#pragma unroll
          for (int v = 0; v < VC; ++v) acc[v][r] *= by;
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float mc = m[r] == -INFINITY ? 0.f : m[r] * c;
        p[r] = exp2_fast(fmaf(p[r], c, -mc));
        l[r] += p[r];
      }
      wave_lds_sync();
      if (h == 0) *(DGNN_LDS f32x4 *)(turn + lane * 16) = p;
      wave_lds_sync();
      constexpr int KEYS = HALVES ? 16 : 32, GROUP = KEYS / 2;         // a lane's keys; of one register of weights
      const lds_ptr own = turn + (HALVES ? 256 * h + lane % 32 * 4 : lane * 4);
      const float w[2] = {*(const DGNN_LDS float *)own, *(const DGNN_LDS float *)(own + 16 * GROUP)};
      unrolled<0, KEYS>([&](auto n) {
        constexpr int K = n.value;
        const lds_ptr at = TL::at(vt, v_lane, K, 0);
        unrolled<0, VC>([&](auto v) {
          acc[v.value] = mma4<HALVES ? 3 : 4, K % GROUP>(w[K / GROUP], *(const DGNN_LDS float *)(at + 4 * v.value), acc[v.value]);
        });
      });
    };
    ring<2, 2 * SG::LOADS, true>(tiles, stage, work);
    if (HALVES) {
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[0][r] += __shfl_xor(acc[0][r], 32, 64);
    }
  }
  // the parts of the rows: {maximum, sum, -, -, output}
  __device__ __forceinline__ void store(const AttnArgs &a, float *part, int rows) const {
    const int lane = lane_id(), col = lane * VC;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float sum = wave_sum(lane < 32 ? l[r] : 0.f);
      if (r >= rows) continue;
      float *to = part + r * (a.d + 4);
      if (lane == 0) to[0] = m[r] == -INFINITY ? -INFINITY : m[r] * c, to[1] = sum;
#pragma unroll
      for (int v = 0; v < VC; ++v)
        if (col + v < a.d) to[4 + col + v] = acc[v][r];             // (DP = 32: d is at most 32)
    }
  }
};

// Single queries and poolings, bound by reading the keys and values: a sequence's first a.few packed rows of a key head are split over chunks of
// a.chunk keys, one wave a chunk, which reads its keys and values once for all query heads of the key
// head; k_attn_join puts the parts together.  Part (slot, key head) holds {output row, maximum, sum} of
// each of the rows.  What rows a sequence has beyond those are dealt to its chunks' workgroups in
// tiles of 32, unsplit.  Two buffers of 32 keys and values: four waves a compute unit keep more loads in flight than
// two with four buffers (9 sequences of 32768 keys, 32 / 8 heads of 128, bfloat16: 230 us against 245, 5.2 TB/s).
template <class T, int DP, bool FOUR>
__global__ __launch_bounds__(64, sizeof(T) == 2 ? 2 : 1) void k_attn_split(const AttnArgs a) {
  using AT = AttnTile<T, DP, 1, 32, 2>;
  DGNN_RING(lds, AT::BYTES);
  const int kvh = blockIdx.x % a.hk, slot = spread(blockIdx.x / a.hk, (int)gridDim.x / a.hk, a.nseq), lane = lane_id(), h = lane >> 5;
  const Segment seg = find_segment(a.col_ptr, a.nseq, a.tk, 1, a.chunk, slot, false);
  if (seg.tile < 0) return;
  int qs, lq;
  other_side(a.row_ptr, a.col_ptr, a.nseq, a.tq, seg, &qs, &lq);
  const long long rows = (long long)lq * a.g;
  const int chunks = (seg.len + a.chunk - 1) / a.chunk;
  float *part = a.part + ((long long)slot * a.hk + kvh) * a.few * (a.d + 4);
  AT t;
  if constexpr (FOUR) {
    __shared__ __align__(16) char turn[512];
    if (rows > 0) {
      AttnFour<DP> f;
      const int n = (int)min(rows, 4LL);
      f.run(a, lds, (lds_ptr)turn, qs, lq, seg.start, seg.len, kvh, n, seg.tile * a.chunk, min(seg.len, (seg.tile + 1) * a.chunk));
      f.store(a, part, n);
    }
  } else if (rows > 0) {
    t.run(a, lds, qs, lq, seg.start, seg.len, kvh, 0, min(rows, (long long)a.few), seg.tile * a.chunk,
          min(seg.len, (seg.tile + 1) * a.chunk));
    if (t.valid) {
      part += (lane & 31) * (a.d + 4);
      store_row<float, DP>(part + 4, t.acc, 1.f, a.d, h);
      if (h == 0) part[0] = t.m == -INFINITY ? -INFINITY : t.base(), part[1] = t.l;
    }
  }
  for (long long row0 = a.few + 32LL * seg.tile; row0 < rows; row0 += 32LL * chunks) {
    __syncthreads();
    t.run(a, lds, qs, lq, seg.start, seg.len, kvh, row0, rows, 0, seg.len);
    t.finish(a, seg.len);
  }
}

// out and lse of the rows k_attn_split left in parts; rows that see no key at all.  One wave a row.
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_attn_join(const AttnArgs a) {
  const int lane = lane_id();
  const long long r = (long long)group_in_rows() * DGNN_WAVES_PER_BLOCK + uniform_i32(wave_in_block());
  if (r >= (long long)a.tq * a.hq) return;
  const int tok = (int)(r / a.hq), head = (int)(r % a.hq);
  const Segment seg = find_segment(a.row_ptr, a.nseq, a.tq, 1, 1, tok, false, true);   // the row's sequence
  const int seq = seg.seq, qs = seg.start, lq = seg.len;
  int ks, lk;
  other_side(a.col_ptr, a.row_ptr, a.nseq, a.tk, seg, &ks, &lk);
  const int qi = tok - qs, packed = qi * a.g + head % a.g;
  const int seen = seq < 0 || seq >= a.nseq ? 0 : a.causal ? max(0, min(lk, qi + lk - lq + 1)) : lk;
  if (seen > 0 && packed >= a.few) return;                          // written unsplit
  T *out = (T *)a.o + r * a.d;
  float *lse = a.lse != nullptr ? a.lse + (long long)head * a.tq + tok : nullptr;
  const int chunks = (seen + a.chunk - 1) / a.chunk;
  const long long slot = (long long)ks / a.chunk + seq + 1, stride = (long long)a.hk * a.few * (a.d + 4);
  const float *part = a.part + ((slot * a.hk + head / a.g) * a.few + packed) * (a.d + 4);
  float top = -INFINITY;
  for (int j = lane; j < chunks; j += 64) top = fmaxf(top, part[j * stride]);
  top = wave_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int j = lane; j < chunks; j += 64) sum += part[j * stride + 1] * exp2_fast(part[j * stride] - base);
  sum = wave_sum(sum);
  for (int c = lane; c < a.d; c += 64) {
    float x = 0.f;
#pragma unroll 4
    for (int j = 0; j < chunks; ++j) x = fmaf(part[j * stride + 4 + c], exp2_fast(part[j * stride] - base), x);
    x = seen > 0 ? x / sum : 0.f;
    out[c] = (T)x;
    if (a.rest != nullptr) ((T *)a.rest)[r * a.d + c] = (T)(x - (float)(T)x);
  }
  if (lse && lane == 0) *lse = seen > 0 ? (base + __builtin_amdgcn_logf(sum)) * DGNN_LN2 : -INFINITY;
}

// ------------------------------------------------------------------ which kernel
// Split: at most 32 packed rows a sequence and 256 keys, on average.  Each way, bfloat16, split and unsplit: 16 single
// queries of 1024 keys 20 and 42 us, 9 of 32768 keys 230 and 1374 us; where the sequences alone fill the card it costs
// something (256 of 1024 keys 226 and 205 us), but a few long ones among short ones cost more the other way.  A
// chunk is a 2048th of all keys times heads (9 x 32768: half of it 242 us, twice 272), within 256 .. 2048.
//
// More rows, but tiles of them for less than half of 512 workgroups: the keys of every tile are split into parts of
// at least 512, by as many as fill those, and joined by k_attn_merge.  Split and unsplit: 4 x 64 rows against 16384
// keys, 32 / 8 heads of 128, causal, bfloat16, 143 and 317 us; 512 rows against as many 194 and 313; 2 x 40 rows
// against 3000 keys, 4 heads of 64, float 55 and 263 us; 1200 x 1200, 4 heads of 128, float 96 and 166; 1100 x 1100, 2 heads of
// 64, bfloat16 15.3 and 19.6; but 3 x 1024 rows, 4 heads of 64, float16 20.6 and 18.3.  Three parts of many rows
// would make a round and a half of workgroups, two are taken (two and three): 1900 x 1900, 8 heads of 32, float 50 and 60
// us; 2048 x 2048, 8 / 2 heads of 64, float 94 and 111, 8 heads of 64, bfloat16 31.6 and 34.9, causal 30.0 and 28.5.
struct AttnPlan {
  int few, chunk;                       // split: rows kept in parts, keys of a chunk (few = 0: not split)
  int splits;                           // tiles of rows: into how many parts the keys are split
  long long slots;
  size_t bytes;
};
static AttnPlan attn_plan(int nseq, int tq, int tk, int hq, int hk, int d) {
  AttnPlan p = {0, 0, 1, 0, 0};
  const long long g = hq / hk, rows = nseq > 0 ? ((long long)tq * g + nseq - 1) / nseq : 0;     // of a sequence, on average
  const long long keys = nseq > 0 ? tk / nseq : 0;
  if (rows == 0) return p;
  if (rows > 32) {
    const long long tiles = ((long long)tq * g / 128 + nseq) * hk;
    long long s = 512 / tiles;
    if (s > keys / 512) s = keys / 512;
    if (s == 3 && rows > 128) s = 2;      // three parts are a round and a half of workgroups
    p.splits = (int)(s < 1 ? 1 : s > 16 ? 16 : s);
    if (p.splits > 1) p.bytes = sizeof(float) * (size_t)p.splits * tq * hq * (d + 4);
    return p;
  }
  if (keys < 256) return p;
  p.few = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
  long long c = ((long long)tk * hk / 2048 + 63) / 64 * 64;
  p.chunk = (int)(c < 256 ? 256 : c > 2048 ? 2048 : c);
  p.slots = tile_slots(tk, nseq, 1, p.chunk);
  p.bytes = sizeof(float) * (size_t)p.slots * hk * p.few * (d + 4);
  return p;
}

template <class T, int DP, int NW, int HW, int BN, int S>
static int launch_rows(const AttnArgs &a, hipStream_t st) {
  const long long groups = tile_slots(a.tq, a.nseq, a.g, 32 * NW) * ((a.hk + HW - 1) / HW) * a.splits;
  const long long rows = (long long)a.tq * a.hq;
  if (!launchable(groups, 64 * NW * HW) || (a.splits > 1 && !launchable(rows, 64))) return DGNN_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((k_attn_fwd<T, DP, NW, HW, BN, S>), dim3((unsigned)groups), dim3(64 * NW * HW), 0, st, a);
  DGNN_LAUNCH_CHECK();
  if (a.splits > 1) {
    hipLaunchKernelGGL(k_attn_merge<T>, dim3((unsigned)((rows + DGNN_WAVES_PER_BLOCK - 1) / DGNN_WAVES_PER_BLOCK)),
                       dim3(DGNN_BLOCK), 0, st, a);
    DGNN_LAUNCH_CHECK();
  }
  return DGNN_OK;
}
template <class T, int DP>
static int launch_fwd(const AttnArgs &a, const AttnPlan &p, hipStream_t st) {
  if (p.few > 0) {
    if (!launchable(p.slots * a.hk, 64)) return DGNN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(p.slots * a.hk));
    const bool four = sizeof(T) == 4 && p.few == 4;
    if constexpr (sizeof(T) == 4) {
      if (four) hipLaunchKernelGGL((k_attn_split<T, DP, true>), grid, dim3(64), 0, st, a);
    }
    if (!four) hipLaunchKernelGGL((k_attn_split<T, DP, false>), grid, dim3(64), 0, st, a);
    DGNN_LAUNCH_CHECK();
    const long long rows = (long long)a.tq * a.hq;
    hipLaunchKernelGGL(k_attn_join<T>, grid_in_rows((rows + DGNN_WAVES_PER_BLOCK - 1) / DGNN_WAVES_PER_BLOCK), dim3(DGNN_BLOCK), 0, st, a);
    DGNN_LAUNCH_CHECK();
    return DGNN_OK;
  }
  if (p.splits > 1 || !rows_short(a.tq, a.nseq, a.g)) return launch_rows<T, DP, 4, 1, 64, 2>(a, st);
  return a.hk >= 4 ? launch_rows<T, DP, 1, 4, 32, 1>(a, st) : launch_rows<T, DP, 1, 1, 32, 1>(a, st);
}
template <class T>
static int launch_fwd_d(const AttnArgs &a, const AttnPlan &p, hipStream_t st) {
  if (a.d <= 32) return launch_fwd<T, 32>(a, p, st);
  if (a.d <= 64) return launch_fwd<T, 64>(a, p, st);
  return launch_fwd<T, 128>(a, p, st);
}

static bool stride_ok(long long s, int size) {
  // a tile of 64 rows stays inside 32-bit offsets, rows start on 16 bytes
  return s >= 0 && s * size % 16 == 0 && s * size < (1LL << 31) / 128;
}
// Checks shared by the two directions; fills `a`.  0, or an error.
int attn_args(int dtype, int nseq, int tq, int tk, int hq, int hk, int d, int causal, float scale, const void *q,
              const void *k, const void *v, const int *row_ptr, const int *col_ptr, const long long *strides,
              AttnArgs *a) {
  if (nseq < 0 || tq < 0 || tk < 0 || hq <= 0 || hk <= 0 || d <= 0 || dtype < 0 || dtype > 2 || hq % hk != 0)
    return DGNN_ERR_BAD_ARG;
  const int size = dtype == DGNN_F32 ? 4 : 2;
  if (d > 128 || d * size % 16 != 0) return DGNN_ERR_UNSUPPORTED;
  if ((long long)tq * hq > 0x7fffffffLL || (long long)tk * hk > 0x7fffffffLL) return DGNN_ERR_UNSUPPORTED;
  if (!row_ptr || !col_ptr || !strides || (tq > 0 && !q) || (tk > 0 && (!k || !v))) return DGNN_ERR_BAD_ARG;
  for (const void *p : {q, k, v})
    if ((uintptr_t)p & 15) return DGNN_ERR_ALIGNMENT;
  if (((uintptr_t)row_ptr | (uintptr_t)col_ptr) & 3) return DGNN_ERR_ALIGNMENT;
  const int toks[3] = {tq, tk, tk}, heads[3] = {hq, hk, hk};
  for (int i = 0; i < 3; ++i) {
    if (toks[i] > 1 && (strides[2 * i] < d || !stride_ok(strides[2 * i], size))) return DGNN_ERR_UNSUPPORTED;
    if (heads[i] > 1 && (strides[2 * i + 1] < 0 || strides[2 * i + 1] * size % 16 != 0)) return DGNN_ERR_UNSUPPORTED;
  }
  memset(a, 0, sizeof(*a));
  a->q = q, a->k = k, a->v = v;
  a->row_ptr = row_ptr, a->col_ptr = col_ptr;
  a->nseq = nseq, a->tq = tq, a->tk = tk, a->hq = hq, a->hk = hk, a->g = hq / hk, a->d = d, a->causal = causal != 0;
  // a dimension of one element may carry any stride: it is never used
  a->q_tok = tq > 1 ? strides[0] : d, a->q_head = hq > 1 ? strides[1] : 0;
  a->k_tok = tk > 1 ? strides[2] : d, a->k_head = hk > 1 ? strides[3] : 0;
  a->v_tok = tk > 1 ? strides[4] : d, a->v_head = hk > 1 ? strides[5] : 0;
  a->scale = scale;
  return DGNN_OK;
}

}  // namespace dgnn

extern "C" {

size_t dgnn_attn_forward_workspace_bytes(int nseq, int tq, int tk, int hq, int hk, int d) {
  if (nseq <= 0 || tq <= 0 || tk <= 0 || hq <= 0 || hk <= 0 || d <= 0 || hq % hk != 0) return 0;
  return attn_plan(nseq, tq, tk, hq, hk, d).bytes;
}

int dgnn_attn_forward(int dtype, int nseq, int tq, int tk, int hq, int hk, int d, int causal, float scale,
                      const void *q, const void *k, const void *v, const long long *strides, const int *row_ptr,
                      const int *col_ptr, void *out, void *out_rest, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  AttnArgs a;
  const int rc = attn_args(dtype, nseq, tq, tk, hq, hk, d, causal, scale, q, k, v, row_ptr, col_ptr, strides, &a);
  if (rc != DGNN_OK) return rc;
  if (tq == 0) return DGNN_OK;
  if (!out) return DGNN_ERR_BAD_ARG;
  if (((uintptr_t)out & 15) || ((uintptr_t)out_rest & 15) || ((uintptr_t)lse & 3)) return DGNN_ERR_ALIGNMENT;
  const AttnPlan p = attn_plan(nseq, tq, tk, hq, hk, d);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return DGNN_ERR_WORKSPACE;
  if (p.bytes > 0 && ((uintptr_t)workspace & 15)) return DGNN_ERR_ALIGNMENT;
  a.o = out;
  a.rest = out_rest;
  a.lse = lse;
  a.part = (float *)workspace, a.few = p.few, a.chunk = p.chunk, a.splits = p.splits;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DGNN_F32) return launch_fwd_d<float>(a, p, st);
  if (dtype == DGNN_BF16) return launch_fwd_d<bf16_t>(a, p, st);
  return launch_fwd_d<half_t>(a, p, st);
}

}  // extern "C"
