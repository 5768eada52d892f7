// Packed attention, backward (formulas of the forward: attention.hip).
//
//   delta_i = <do_i, o_i>,  dv_j = sum_i p_ij do_i,  ds_ij = p_ij (<do_i, v_j> - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// p is rebuilt from the saved lse.  Two kernels, each owning its outputs, so nothing is summed through
// atomics and results do not depend on the order of workgroups: k_attn_bwd_kv keeps 32 keys a wave
// with dk^T and dv^T in accumulators and walks the query tiles of all heads that share the key head;
// k_attn_bwd_q keeps 32 packed query rows a wave and walks the key tiles.  The price is forming z and
// do v^T twice: seven products instead of five.  p and ds are rounded to T for the products that sum over
// them, half a step each; everything else is float.
//
// float16 has neither the range for p of long rows nor for ds = p (<do, v> - delta), whose size is that of the incoming
// gradient divided by the keys: from 2^-14 down every bit of size costs one of precision, below 2^-25 nothing is left
// (4096 keys and gradients of 1e-4: three steps of the type).  p is therefore rounded as 2^12 p, and ds times a
// power of two of the lane's own row (or key), lowered whenever a term outgrows it, like the softmax's running
// maximum (DsScale); both come out of the float sums at the end.  It costs 4 % of a training step of 32 x 2048 tokens, 8
// heads of 64 (1440 us, 1378 without).  bfloat16 has float's range.
#include <utility>

#include "attention.hpp"

using namespace dgnn;

namespace dgnn {

// Rows of a staged tile: 32, or 64 where 32 are too few bytes for one load of every wave.
template <class T, int DP, int NW>
constexpr int bwd_rows() { return 32 * DP * (int)sizeof(T) >= 1024 * NW ? 32 : 64; }

template <class T> constexpr bool scaled() { return std::is_same<T, half_t>::value; }
template <class T> constexpr float p_shift() { return scaled<T>() ? 12.f : 0.f; }        // p is kept times 2^p_shift

// The running power of two of a lane's column of ds (lanes l and l + 32 share one).  It starts above any use, so that
// the first terms set it: the largest term so far lies below 2^15, and was below 2^12 when the factor was set.
template <bool ON>
struct DsScale {
  static constexpr float START = 0x1p60f;       // ds < 2^52 from float16 operands of 128 elements: no overflow
  float by = ON ? START : 1.f;
  // ds holds terms times `by`; sums are what was added up of such terms
  template <int N>
  __device__ __forceinline__ void fit(acc16 &ds, acc16 (&sums)[N]) {
    if constexpr (ON) {
      float top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
      if (__any(top > 32768.f)) {
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // an infinite term stays infinite whatever the factor
        const float change = top > 32768.f && top < INFINITY ? ldexpf(1.f, 12 - __builtin_amdgcn_frexp_expf(top)) : 1.f;
        by *= change;
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] *= change;
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) sums[b][r] *= change;
      }
    }
  }
  __device__ __forceinline__ float out() const { return ON ? 1.f / by : 1.f; }
};

// Long sequences: four waves with 32 keys each share the staged tiles of queries and do, a ring of four, since
// two waves a SIMD (the accumulators' 256 registers) hide little by themselves.  Bound by the matrix instructions
// under the power limit: 32 x 2048 tokens, 8 heads of 64, bfloat16 0.56 - 0.66 ms, 830 - 980 TFLOP/s; 20 k tokens,
// causal, 16 / 4 heads of 128, lengths up to 8000, 1.03 ms, 970 TFLOP/s (a large matrix product reaches 1156).
// 1024 graphs of 1 .. 63 nodes, 8 heads of 32, float: 52 us, waiting for each wave's few loads.
template <class T, int DP, int NW, int HW, int S>
__global__ __launch_bounds__(64 * NW * HW, sizeof(T) == 2 && (NW > 1 || DP < 128) ? 2 : 1) void k_attn_bwd_kv(const AttnArgs a) {
  constexpr int BK = 32 * NW, BQ = bwd_rows<T, DP, NW>(), THREADS = 64 * NW;
  using TL = Tile<T, DP>;
  using SG = Stager<T, DP, BQ, THREADS>;
  // a stage: q tile, do tile, and for every wave its own copy of the statistics (equal load counts)
  constexpr int TILE = BQ * TL::ROW_BYTES, STAT = 2 * BQ * 4;
  constexpr int BYTES = 2 * TILE + NW * STAT;
  DGNN_RING(all, HW * BYTES);
  const HeadSlot at = head_slot<HW>(a.hk, a.nseq, a.splits);
  if (at.head >= a.hk) return;
  const lds_ptr lds[4] = {all[0] + at.wave * BYTES, all[1] + at.wave * BYTES, all[2] + at.wave * BYTES, all[3] + at.wave * BYTES};
  // Two waves a SIMD leave 256 registers; at DP = 128 the accumulators and both operands take 192, and the
  // last fragments of k did not fit (a spill to memory whose wait drains the ring).  They live in LDS: two of them,
  // three with the factor of ds, which is what half of a compute unit's LDS holds next to the ring.  At DP = 64 the factor
  // would cost the third wave of a SIMD, and one of them lives there.
  constexpr int PARK = DP == 128 && sizeof(T) == 2 && NW > 1 ? (scaled<T>() ? 3 : 2) : DP == 64 && scaled<T>() ? 1 : 0, KEPT = DP / 16 - PARK;
  constexpr int PARKERS = THREADS * HW;
  __shared__ __align__(16) char parked[PARK ? PARK * PARKERS * 16 : 16];
  const int lane = lane_id(), h = lane >> 5, wave = NW == 1 ? 0 : uniform_i32(wave_in_block());
  const int row_lane = TL::row_lane(lane), col_lane = TL::col_lane(lane);
  const int kvh = at.head, split = at.split;
  const Segment seg = find_segment(a.col_ptr, a.nseq, a.tk, 1, BK, at.slot, false);
  if (seg.tile < 0) return;
  int qs, lq;
  other_side(a.row_ptr, a.col_ptr, a.nseq, a.tq, seg, &qs, &lq);
  const int lk = seg.len;
  // causal: the first rows of a sequence with more rows than keys see none; what they hold must not be read
  const int blind = a.causal ? max(0, lq - lk) : 0;
  qs += blind, lq -= blind;

  const int key0 = seg.tile * BK + wave * 32, key = key0 + (lane & 31);
  const bool valid = key < lk;
  const long long tok = seg.start + (long long)key;
  // first query that sees a key: query i sees key j when j <= i + lk - lq
  const int first = a.causal ? key - (lk - lq) : 0;
  const int wave_first = a.causal ? key0 - (lk - lq) : 0, wave_all = a.causal ? key0 + 31 - (lk - lq) : 0;
  const int t0 = a.causal ? max(0, seg.tile * BK - (lk - lq)) / BQ : 0;
  const int tiles = (lq + BQ - 1) / BQ, per_head = max(0, tiles - t0);
  // this workgroup's share of the query tiles of all heads
  const int share = (per_head * a.g + a.splits - 1) / a.splits, from = min(split * share, per_head * a.g);
  const int total = min(share, per_head * a.g - from);

  frag8<T> kf[DP / 16], vf[DP / 16];
  load_row_frags<T, DP>(kf, (const T *)a.k + tok * a.k_tok + (long long)kvh * a.k_head, a.d, h, valid);
  load_row_frags<T, DP>(vf, (const T *)a.v + tok * a.v_tok + (long long)kvh * a.v_head, a.d, h, valid);
#pragma unroll
  for (int k = KEPT; k < DP / 16; ++k) *(frag8<T> *)(parked + ((k - KEPT) * PARKERS + threadIdx.x) * 16) = kf[k];
  const float c = a.scale * DGNN_LOG2E;

  const unsigned q_stride = (unsigned)(a.q_tok * sizeof(T)), g_stride = (unsigned)((long long)a.hq * a.d * sizeof(T));
  const unsigned row_bytes = a.d * (unsigned)sizeof(T);
  SG st_q, st_g;
  st_q.init(q_stride, a.d);
  st_g.init(g_stride, a.d);
  // next tile to stage
  int s_head = kvh * a.g + from / max(per_head, 1), s_tile = t0 + from % max(per_head, 1), s_left = total;
  auto stage = [&](int, auto i) {
    // rows behind the end arrive as zeros: p = exp2(0 - 0) = 1 there, on do = 0 and delta = 0
    const int n = s_left > 0 ? min(BQ, lq - s_tile * BQ) : 0;
    const long long tq0 = qs + (long long)s_tile * BQ;
    const auto stat = buffer_over(a.stat + ((long long)s_head * a.tq + tq0) * 2, n * 8u);
#pragma unroll
    for (int w = 0; w < BQ / 32; ++w) load_words(lds[i.value] + 2 * TILE + wave * STAT + 256 * w, stat, (64 * w + lane) * 4u);
    st_q.load(lds[i.value], buffer_over((const T *)a.q + tq0 * a.q_tok + (long long)s_head * a.q_head, span_bytes(n, q_stride, row_bytes)));
    st_g.load(lds[i.value] + TILE, buffer_over((const T *)a.grad + (tq0 * a.hq + s_head) * a.d, span_bytes(n, g_stride, row_bytes)));
    --s_left;
    if (++s_tile == tiles) s_tile = t0, ++s_head;
  };

  acc16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) dk[b] = acc_zero(), dv[b] = acc_zero();
  DsScale<scaled<T>()> ds_scale;

  int w_tile = s_tile;                                       // tile worked on
  auto work = [&](int, auto i) {
    const lds_ptr qt = lds[i.value], gt = qt + TILE;
    const DGNN_LDS float *stt = (const DGNN_LDS float *)(gt + TILE + wave * STAT);
    const int q00 = w_tile * BQ;
    if (++w_tile == tiles) w_tile = t0;
#pragma unroll
    for (int qb = 0; qb < BQ / 32; ++qb) {
      const int q0 = q00 + 32 * qb;
      if (q0 + 31 < wave_first || key0 >= lk) continue;
      const int rl = opaque(row_lane), cl = opaque(col_lane);
      acc16 s = acc_zero(), dp = acc_zero();
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const frag8<T> kk = k < KEPT ? kf[k] : *(const frag8<T> *)(parked + ((k - KEPT) * PARKERS + threadIdx.x) * 16);
        s = mma(TL::row_frag(qt, rl, 32 * qb, 16 * k), kk, s);
        dp = mma(TL::row_frag(gt, rl, 32 * qb, 16 * k), vf[k], dp);
      }
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const DGNN_LDS vec4<float> *st = (const DGNN_LDS vec4<float> *)(stt + 2 * (32 * qb + 8 * r4 + 4 * h));
        const vec4<float> x = st[0], y = st[1];
        const float ls[4] = {x[0], x[2], y[0], y[2]}, de[4] = {x[1], x[3], y[1], y[3]};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * r4 + j;
          s[r] = exp2_fast(fmaf(s[r], c, -ls[j]));
          dp[r] = scaled<T>() ? s[r] * ds_scale.by * (dp[r] - de[j]) : s[r] * (dp[r] - de[j]);
        }
      }
      if (q0 < wave_all) {                      // the diagonal crosses this block
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool seen = q0 + acc_row(r, h) >= first;
          s[r] = seen ? s[r] : 0.f;
          dp[r] = seen ? dp[r] : 0.f;
        }
      }
      ds_scale.fit(dp, dk);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const frag8<T> p = frag_of<T>(s, 8 * k), ds = frag_of<T>(dp, 8 * k);
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
          dv[b] = mma(TL::col_frag(gt, cl, 32 * qb + 16 * k, 32 * b), p, dv[b]);
          dk[b] = mma(TL::col_frag(qt, cl, 32 * qb + 16 * k, 32 * b), ds, dk[b]);
        }
      }
    }
  };
  ring<S, 2 * SG::LOADS + BQ / 32, NW == 1>(total, stage, work);

  // the lane's key once more, rather than in registers throughout the loop
  const int lane2 = opaque(lane), key2 = key0 + (lane2 & 31);
  if (key2 >= lk) return;
  const long long to = ((seg.start + (long long)key2) * a.hk + kvh) * a.d;
  const float of_p = scaled<T>() ? 1.f / (1 << (int)p_shift<T>()) : 1.f, of_ds = a.scale * of_p * ds_scale.out();
  if (a.splits > 1) {
    float *part = a.part + 2 * ((long long)split * a.tk * a.hk * a.d + to);
    store_row<float, DP>(part, dk, of_ds, a.d, lane2 >> 5);
    store_row<float, DP>(part + a.d, dv, of_p, a.d, lane2 >> 5);
    return;
  }
  store_row<T, DP>((T *)a.dk + to, dk, of_ds, a.d, lane2 >> 5);
  store_row<T, DP>((T *)a.dv + to, dv, of_p, a.d, lane2 >> 5);
}

// dk and dv of every (key, key head): the sum of the splits' {dk row, dv row}, in order
template <class T>
__global__ __launch_bounds__(DGNN_BLOCK) void k_attn_bwd_join(const AttnArgs a) {
  const long long rows = (long long)a.tk * a.hk, per = a.d / 4, u = group_in_rows() * (long long)DGNN_BLOCK + threadIdx.x;
  if (u >= rows * per * 2) return;
  const long long row = u / (per * 2);
  const int c = (int)(u % (per * 2)) * 4;
  const float *part = a.part + row * 2 * a.d + c;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < a.splits; ++i) {
    const float4 v = *(const float4 *)(part + i * rows * 2 * a.d);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  vec4<T> o;
  o[0] = (T)s.x, o[1] = (T)s.y, o[2] = (T)s.z, o[3] = (T)s.w;
  *(vec4<T> *)((T *)(c < a.d ? a.dk : a.dv) + row * a.d + (c < a.d ? c : c - a.d)) = o;
}

// The same with the sides changed, as the forward: a lane has one packed query row.  At the sizes above 0.40 - 0.49 ms,
// 0.74 - 0.79 ms (950 - 1010 TFLOP/s) and 45 us.  It runs first and leaves {lse log2(e), <do, o>} of every row for the
// other: a kernel of its own for them read grad a second time, 35 to 48 us of the first two steps, 9 of the last.
template <class T, int DP, int NW, int HW, int S>
__global__ __launch_bounds__(64 * NW * HW, sizeof(T) == 2 ? 2 : 1) void k_attn_bwd_q(const AttnArgs a) {
  constexpr int BM = 32 * NW, BN = bwd_rows<T, DP, NW>(), THREADS = 64 * NW;
  using TL = Tile<T, DP>;
  using SG = Stager<T, DP, BN, THREADS>;
  constexpr int TILE = BN * TL::ROW_BYTES;
  DGNN_RING(all, HW * 2 * TILE);
  const HeadSlot at = head_slot<HW>(a.hk, a.nseq, 1);
  if (at.head >= a.hk) return;
  const lds_ptr lds[4] = {all[0] + at.wave * 2 * TILE, all[1] + at.wave * 2 * TILE, all[2] + at.wave * 2 * TILE, all[3] + at.wave * 2 * TILE};
  const int lane = lane_id(), h = lane >> 5, wave = NW == 1 ? 0 : uniform_i32(wave_in_block());
  const int row_lane = TL::row_lane(lane), col_lane = TL::col_lane(lane);
  const int kvh = at.head;
  const Segment seg = find_segment(a.row_ptr, a.nseq, a.tq, a.g, BM, at.slot, a.causal != 0);
  if (seg.tile < 0) return;
  int ks, lk;
  other_side(a.col_ptr, a.row_ptr, a.nseq, a.tk, seg, &ks, &lk);

  const long long rows = (long long)seg.len * a.g;
  const long long row = (long long)seg.tile * BM + wave * 32 + (lane & 31);
  const bool valid = row < rows;
  const int qi = (int)(row / a.g), head = kvh * a.g + (int)(row % a.g);
  const long long tok = seg.start + (long long)qi;
  const int limit = !valid ? -1 : a.causal ? qi + (lk - seg.len) : lk - 1;
  const long long last_row = min(rows, (long long)(seg.tile + 1) * BM) - 1;
  const int seen = a.causal ? max(0, min(lk, (int)(last_row / a.g) + (lk - seg.len) + 1)) : lk;
  const int tiles = (seen + BN - 1) / BN;
  const long long wrow = (long long)seg.tile * BM + wave * 32;
  const int wave_all = a.causal ? (int)(min(wrow, last_row) / a.g) + (lk - seg.len) : lk - 1;
  const int wave_any = wrow > last_row ? -1
                       : a.causal ? (int)(min(wrow + 31, last_row) / a.g) + (lk - seg.len) : lk - 1;

  frag8<T> qf[DP / 16], gf[DP / 16];
  load_row_frags<T, DP>(qf, (const T *)a.q + tok * a.q_tok + (long long)head * a.q_head, a.d, h, valid);
  load_row_frags<T, DP>(gf, (const T *)a.grad + (tok * a.hq + head) * a.d, a.d, h, valid);
  // <do, o>, o with what its rounding took (`rest`): <do, v_j> - <do, o> cancels in rows that see few keys, and half a
  // step of a 16-bit o is all that was left of it
  float delta = 0.f;
  {
    const long long at = (tok * a.hq + head) * a.d;
    frag8<T> o[DP / 16];
    auto add = [&](const void *from) {
      load_row_frags<T, DP>(o, (const T *)from + at, a.d, h, valid);
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) delta = fmaf((float)o[s][j], (float)gf[s][j], delta);
    };
    add(a.out);
    if (a.rest != nullptr) add(a.rest);
    delta += __shfl_xor(delta, 32, 64);
  }
  // a row that saw no key: p = exp2(z - inf) = 0
  float lse = valid ? a.lse[(long long)head * a.tq + tok] : -INFINITY;
  lse = lse == -INFINITY ? INFINITY : lse * DGNN_LOG2E;
  if (valid && h == 0) ((float2 *)a.stat)[(long long)head * a.tq + tok] = make_float2(lse - p_shift<T>(), delta);
  const float c = a.scale * DGNN_LOG2E;

  const unsigned k_stride = (unsigned)(a.k_tok * sizeof(T)), v_stride = (unsigned)(a.v_tok * sizeof(T));
  const unsigned row_bytes = a.d * (unsigned)sizeof(T);
  const T *kbase = (const T *)a.k + (long long)ks * a.k_tok + (long long)kvh * a.k_head;
  const T *vbase = (const T *)a.v + (long long)ks * a.v_tok + (long long)kvh * a.v_head;
  SG st_k, st_v;
  st_k.init(k_stride, a.d);
  st_v.init(v_stride, a.d);
  auto stage = [&](int t, auto i) {
    const int n = t < tiles ? min(BN, lk - t * BN) : 0;
    st_k.load(lds[i.value], buffer_over(kbase + (long long)t * BN * a.k_tok, span_bytes(n, k_stride, row_bytes)));
    st_v.load(lds[i.value] + TILE, buffer_over(vbase + (long long)t * BN * a.v_tok, span_bytes(n, v_stride, row_bytes)));
  };

  acc16 dq[DP / 32];
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) dq[b] = acc_zero();
  DsScale<scaled<T>()> ds_scale;

  auto work = [&](int t, auto i) {
    const lds_ptr kt = lds[i.value], vt = kt + TILE;
#pragma unroll
    for (int kb = 0; kb < BN / 32; ++kb) {
      const int k0 = t * BN + 32 * kb;
      if (k0 > wave_any) continue;
      const int rl = opaque(row_lane), cl = opaque(col_lane);
      acc16 s = acc_zero(), dp = acc_zero();
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        s = mma(TL::row_frag(kt, rl, 32 * kb, 16 * k), qf[k], s);
        dp = mma(TL::row_frag(vt, rl, 32 * kb, 16 * k), gf[k], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        // (a power of two: the same rounding as the difference's)
        const float diff = scaled<T>() ? fmaf(dp[r], ds_scale.by, -delta * ds_scale.by) : dp[r] - delta;
        dp[r] = exp2_fast(fmaf(s[r], c, -lse)) * diff;
      }
      if (k0 + 31 > wave_all) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = k0 + acc_row(r, h) <= limit ? dp[r] : 0.f;
      }
      ds_scale.fit(dp, dq);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const frag8<T> ds = frag_of<T>(dp, 8 * k);
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) dq[b] = mma(TL::col_frag(kt, cl, 32 * kb + 16 * k, 32 * b), ds, dq[b]);
      }
    }
  };
  ring<S, 2 * SG::LOADS, NW == 1>(tiles, stage, work);

  if (limit < 0) {                              // sees no key: no gradient, whatever the keys hold
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dq[b] = acc_zero();
  }
  if (valid) store_row<T, DP>((T *)a.dq + (tok * a.hq + head) * a.d, dq, a.scale * ds_scale.out(), a.d, h);
}

// Into how many parts the query tiles of a key tile are split.  A key tile's workgroup walks the queries of
// every head that shares the key head, the first ones of a causal sequence all of them: with fewer
// workgroups than four rounds of the card, the longest of them are most of the time.  The parts cost
// writing and reading dk and dv once each in float: 20 k tokens, 16 / 4 heads of 128, causal, lengths up to
// 8000: 1.59 ms unsplit, 1.03 and 0.05 for the join split; 8192 tokens in one sequence, the whole training step 1.92
// and 1.29 ms; 2048 tokens, 8 heads of 64, 135 and 119 us.
static int bwd_splits(int nseq, int tq, int tk, int hq, int hk) {
  if (nseq <= 0 || tk <= 0 || tq <= 0 || rows_short(tk, nseq, 1)) return 1;
  const long long groups = tile_slots(tk, nseq, 1, 128) * hk, steps = (long long)tq / nseq / 32 * (hq / hk);
  long long s = (2047 + groups) / groups;
  if (s > steps / 16) s = steps / 16;
  return (int)(s < 1 ? 1 : s > 8 ? 8 : s);
}
static size_t align256(size_t x) { return (x + 255) / 256 * 256; }

static long long bwd_kv_groups(const AttnArgs &a, int nw, int hw) {
  return tile_slots(a.tk, a.nseq, 1, 32 * nw) * ((a.hk + hw - 1) / hw) * a.splits;
}
static long long bwd_q_groups(const AttnArgs &a, int nw, int hw) {
  return tile_slots(a.tq, a.nseq, a.g, 32 * nw) * ((a.hk + hw - 1) / hw);
}
template <class T, int DP, int NW, int HW, int S>
static int launch_bwd_kv(const AttnArgs &a, hipStream_t st) {
  const long long groups = bwd_kv_groups(a, NW, HW);
  hipLaunchKernelGGL((k_attn_bwd_kv<T, DP, NW, HW, S>), dim3((unsigned)groups), dim3(64 * NW * HW), 0, st, a);
  DGNN_LAUNCH_CHECK();
  if (a.splits > 1) {
    const long long blocks = ((long long)a.tk * a.hk * (a.d / 2) + DGNN_BLOCK - 1) / DGNN_BLOCK;
    hipLaunchKernelGGL(k_attn_bwd_join<T>, grid_in_rows(blocks), dim3(DGNN_BLOCK), 0, st, a);
    DGNN_LAUNCH_CHECK();
  }
  return DGNN_OK;
}
template <class T, int DP, int NW, int HW, int S>
static int launch_bwd_q(const AttnArgs &a, hipStream_t st) {
  const long long groups = bwd_q_groups(a, NW, HW);
  hipLaunchKernelGGL((k_attn_bwd_q<T, DP, NW, HW, S>), dim3((unsigned)groups), dim3(64 * NW * HW), 0, st, a);
  DGNN_LAUNCH_CHECK();
  return DGNN_OK;
}
template <class T, int DP>
static int launch_bwd(const AttnArgs &a, hipStream_t st) {
  int rc = DGNN_OK;
  const bool few_q = rows_short(a.tq, a.nseq, a.g), few_k = a.splits <= 1 && rows_short(a.tk, a.nseq, 1);
  // both of them before either runs
  for (const auto &[few, groups] : {std::pair(few_q, &bwd_q_groups), std::pair(few_k, &bwd_kv_groups)}) {
    const int nw = few ? 1 : 4, hw = few && a.hk >= 4 ? 4 : 1;
    if (!launchable(groups(a, nw, hw), 64 * nw * hw)) return DGNN_ERR_UNSUPPORTED;
  }
  if (a.tq > 0) {
    if (!few_q) rc = launch_bwd_q<T, DP, 4, 1, 4>(a, st);
    else rc = a.hk >= 4 ? launch_bwd_q<T, DP, 1, 4, 1>(a, st) : launch_bwd_q<T, DP, 1, 1, 1>(a, st);
  }
  if (rc == DGNN_OK && a.tk > 0) {
    if (!few_k) rc = launch_bwd_kv<T, DP, 4, 1, 4>(a, st);
    else rc = a.hk >= 4 ? launch_bwd_kv<T, DP, 1, 4, 1>(a, st) : launch_bwd_kv<T, DP, 1, 1, 1>(a, st);
  }
  return rc;
}
template <class T>
static int launch_bwd_d(const AttnArgs &a, hipStream_t st) {
  if (a.d <= 32) return launch_bwd<T, 32>(a, st);
  if (a.d <= 64) return launch_bwd<T, 64>(a, st);
  return launch_bwd<T, 128>(a, st);
}

}  // namespace dgnn

extern "C" {

size_t dgnn_attn_backward_workspace_bytes(int nseq, int tq, int tk, int hq, int hk, int d) {
  if (nseq < 0 || tq < 0 || tk < 0 || hq <= 0 || hk <= 0 || d <= 0 || hq % hk != 0) return 0;
  const int splits = bwd_splits(nseq, tq, tk, hq, hk);
  return align256(2 * sizeof(float) * (size_t)tq * (size_t)hq) +
         (splits > 1 ? 2 * sizeof(float) * (size_t)splits * (size_t)tk * (size_t)hk * (size_t)d : 0);
}

int dgnn_attn_backward(int dtype, int nseq, int tq, int tk, int hq, int hk, int d, int causal, float scale,
                       const void *q, const void *k, const void *v, const long long *strides, const int *row_ptr,
                       const int *col_ptr, const void *out, const void *out_rest, const float *lse, const void *grad, void *dq, void *dk,
                       void *dv, void *workspace, size_t workspace_bytes, void *stream) {
  AttnArgs a;
  const int rc = attn_args(dtype, nseq, tq, tk, hq, hk, d, causal, scale, q, k, v, row_ptr, col_ptr, strides, &a);
  if (rc != DGNN_OK) return rc;
  if (tq > 0 && (!out || !lse || !grad || !dq)) return DGNN_ERR_BAD_ARG;
  if (tk > 0 && (!dk || !dv)) return DGNN_ERR_BAD_ARG;
  for (const void *p : {out, out_rest, grad, (const void *)dq, (const void *)dk, (const void *)dv})
    if ((uintptr_t)p & 15) return DGNN_ERR_ALIGNMENT;
  if (workspace_bytes < dgnn_attn_backward_workspace_bytes(nseq, tq, tk, hq, hk, d) || (tq > 0 && !workspace)) return DGNN_ERR_WORKSPACE;
  if (((uintptr_t)workspace & 15) || ((uintptr_t)lse & 3)) return DGNN_ERR_ALIGNMENT;
  if ((long long)hq * d * (dtype == DGNN_F32 ? 4 : 2) >= (1LL << 31) / 128) return DGNN_ERR_UNSUPPORTED;
  a.out = out, a.lse = (float *)lse, a.rest = (void *)out_rest, a.grad = grad, a.dq = dq, a.dk = dk, a.dv = dv;
  a.stat = (float *)workspace;
  a.splits = bwd_splits(nseq, tq, tk, hq, hk);
  a.part = (float *)((char *)workspace + align256(2 * sizeof(float) * (size_t)tq * (size_t)hq));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DGNN_F32) return launch_bwd_d<float>(a, st);
  if (dtype == DGNN_BF16) return launch_bwd_d<bf16_t>(a, st);
  return launch_bwd_d<half_t>(a, st);
}

}  // extern "C"
