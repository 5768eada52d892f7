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
#include "attention.hpp"

using namespace dgnn;

namespace dgnn {

constexpr int ATTN_BN = 64;                    // keys of a tile

template <class T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 2 : 1) void k_attn_fwd(const AttnArgs a) {
  constexpr int BM = 32 * NW, BN = ATTN_BN, THREADS = 64 * NW;
  using TL = Tile<T, DP>;
  using SG = Stager<T, DP, BN, THREADS>;
  constexpr int TILE = BN * TL::ROW_BYTES, S = 2;
  DGNN_RING(lds, 2 * TILE);
  const int lane = lane_id(), h = lane >> 5, wave = uniform_i32(wave_in_block());
  const int row_lane = TL::row_lane(lane), col_lane = TL::col_lane(lane);
  const int kvh = blockIdx.x % a.hk, slot = blockIdx.x / a.hk;
  const Segment seg = find_segment(a.row_ptr, a.nseq, a.tq, a.g, BM, slot, a.causal != 0);
  if (seg.tile < 0) return;
  int ks, lk;
  other_side(a.col_ptr, a.nseq, a.tk, seg.seq, &ks, &lk);

  // this lane's row
  const long long rows = (long long)seg.len * a.g;
  const long long row = (long long)seg.tile * BM + wave * 32 + (lane & 31);
  const bool valid = row < rows;
  const int qi = (int)(row / a.g), head = kvh * a.g + (int)(row % a.g);
  const long long tok = seg.start + (long long)qi;
  // last key it sees; a.causal: queries and keys end together
  const int limit = !valid ? -1 : a.causal ? qi + (lk - seg.len) : lk - 1;
  const long long last_row = min(rows, (long long)(seg.tile + 1) * BM) - 1;
  const int seen = a.causal ? max(0, min(lk, (int)(last_row / a.g) + (lk - seg.len) + 1)) : lk;
  const int tiles = (seen + BN - 1) / BN;
  // every row of the wave sees keys 0 .. wave_all, none sees a key behind wave_any
  const long long wrow = (long long)seg.tile * BM + wave * 32;
  const int wave_all = a.causal ? (int)(min(wrow, last_row) / a.g) + (lk - seg.len) : lk - 1;
  const int wave_any = wrow > last_row ? -1
                       : a.causal ? (int)(min(wrow + 31, last_row) / a.g) + (lk - seg.len) : lk - 1;

  frag8<T> qf[DP / 16];
  const T *qrow = (const T *)a.q + tok * a.q_tok + (long long)head * a.q_head;
  load_row_frags<T, DP>(qf, qrow, a.d, h, valid);
  float c = a.scale * DGNN_LOG2E;
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

  acc16 acc[DP / 32];
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) acc[b] = acc_zero();
  float m = -INFINITY, l = 0.f;                 // running maximum of z / scale, this half's share of the sum

  auto work = [&](int t, auto i) {
    const char *kt = lds[i.value], *vt = kt + TILE;
    if (t * BN > wave_any) return;
    const int rl = opaque(row_lane), cl = opaque(col_lane);
    acc16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = acc_zero();
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        s[b] = mma(TL::row_frag(kt, rl, 32 * b, 16 * i), qf[i], s[b]);
    }
    if (t * BN + BN - 1 > wave_all) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * BN + 32 * b + acc_row(r, h) > limit) s[b][r] = -INFINITY;
    }
    float top = m;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m)) {
      const float by = top == m ? 1.f : exp2_fast((m - top) * c);     // m = -inf: 0
      m = top;
      l *= by;
#pragma unroll
      for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] *= by;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = exp2_fast(fmaf(s[b][r], c, -mc));
        l += s[b][r];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const frag8<T> p = frag_of<T>(s[i >> 1], 8 * (i & 1));
#pragma unroll
      for (int b = 0; b < DP / 32; ++b) acc[b] = mma(TL::col_frag(vt, cl, 16 * i, 32 * b), p, acc[b]);
    }
  };

  ring<S, 2 * SG::LOADS>(tiles, stage, work);

  if (!valid) return;
  l += __shfl_xor(l, 32, 64);
  const bool none = limit < 0 || lk == 0;
  store_row<T, DP>((T *)a.o + (tok * a.hq + head) * a.d, acc, none ? 0.f : 1.f / l, a.d, h);
  if (a.lse != nullptr && h == 0)
    a.lse[(long long)head * a.tq + tok] = none ? -INFINITY : (m * c + __builtin_amdgcn_logf(l)) * DGNN_LN2;
}

template <class T, int DP>
static int launch_fwd(const AttnArgs &a, hipStream_t st) {
  constexpr int NW = 4;
  const long long slots = tile_slots(a.tq, a.nseq, a.g, 32 * NW);
  if (slots * a.hk > 0x7fffffffLL) return DGNN_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((k_attn_fwd<T, DP, NW>), dim3((unsigned)(slots * a.hk)), dim3(64 * NW), 0, st, a);
  DGNN_LAUNCH_CHECK();
  return DGNN_OK;
}
template <class T>
static int launch_fwd_d(const AttnArgs &a, hipStream_t st) {
  if (a.d <= 32) return launch_fwd<T, 32>(a, st);
  if (a.d <= 64) return launch_fwd<T, 64>(a, st);
  return launch_fwd<T, 128>(a, st);
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

int dgnn_attn_forward(int dtype, int nseq, int tq, int tk, int hq, int hk, int d, int causal, float scale,
                      const void *q, const void *k, const void *v, const long long *strides, const int *row_ptr,
                      const int *col_ptr, void *out, float *lse, void *stream) {
  AttnArgs a;
  const int rc = attn_args(dtype, nseq, tq, tk, hq, hk, d, causal, scale, q, k, v, row_ptr, col_ptr, strides, &a);
  if (rc != DGNN_OK) return rc;
  if (tq == 0) return DGNN_OK;
  if (!out) return DGNN_ERR_BAD_ARG;
  if (((uintptr_t)out & 15) || ((uintptr_t)lse & 3)) return DGNN_ERR_ALIGNMENT;
  a.o = out;
  a.lse = lse;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DGNN_F32) return launch_fwd_d<float>(a, st);
  if (dtype == DGNN_BF16) return launch_fwd_d<bf16_t>(a, st);
  return launch_fwd_d<half_t>(a, st);
}

}  // extern "C"
