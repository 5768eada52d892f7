// Matrix-core building blocks of the dense operators (attention.hip, attention_bwd.hip, linear_ce.hip).
//
// Everything is built from one product, C[32 x 32] += A[32 x 16] B[16 x 32], on 64 lanes.  Lane l
// holds eight elements of A's row l % 32 and eight of B's column l % 32, those of k-half l / 32; the
// result puts column l % 32 of C into lane l, rows 8 (r / 4) + 4 (l / 32) + r % 4 for r = 0 .. 15.
// For 16-bit types that is one v_mfma_f32_32x32x16; for float it is eight v_mfma_f32_32x32x2, where
// element j of both operands feeds product j.  Which k an element stands for does not matter
// as long as A and B agree, so the rows a lane holds of one product are, unmoved, the k elements of
// its column in the next: element j of half h stands for k = 8 (j / 4) + 4 h + j % 4 there.
#pragma once
#include <type_traits>

#include "common.hpp"

namespace dgnn {

// f(integral_constant I) for I = A .. B - 1
template <int A, int B, class F>
__device__ __forceinline__ void unrolled(const F &f) {
  if constexpr (A < B) {
    f(std::integral_constant<int, A>());
    unrolled<A + 1, B>(f);
  }
}

typedef _Float16 half_t;
typedef __bf16 bf16_t;
typedef float acc16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Pointers into LDS carry their address space: a generic pointer is only proven to be one where the
// compiler can see the variable it came from.
#define DGNN_LDS __attribute__((address_space(3)))
typedef DGNN_LDS char *lds_ptr;

template <class T> struct frag8_of;
template <> struct frag8_of<bf16_t> { typedef bf16_t type __attribute__((ext_vector_type(8))); };
template <> struct frag8_of<half_t> { typedef half_t type __attribute__((ext_vector_type(8))); };
template <> struct frag8_of<float> { typedef float type __attribute__((ext_vector_type(8))); };
template <class T> using frag8 = typename frag8_of<T>::type;
template <class T> struct vec4_of;
template <> struct vec4_of<bf16_t> { typedef bf16_t type __attribute__((ext_vector_type(4))); };
template <> struct vec4_of<half_t> { typedef half_t type __attribute__((ext_vector_type(4))); };
template <> struct vec4_of<float> { typedef float type __attribute__((ext_vector_type(4))); };
template <class T> using vec4 = typename vec4_of<T>::type;

__device__ __forceinline__ acc16 mma(frag8<bf16_t> a, frag8<bf16_t> b, acc16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ acc16 mma(frag8<half_t> a, frag8<half_t> b, acc16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ acc16 mma(frag8<float> a, frag8<float> b, acc16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}
// acc[i][j] += a[i] b[j].  float: the eight products of one accumulator depend on each other, so they
// are interleaved over all of them.
template <int MB, int NB, class T>
__device__ __forceinline__ void mma_block(const frag8<T> (&a)[MB], const frag8<T> (&b)[NB], acc16 (&acc)[MB][NB], T) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i][e], b[j][e], acc[i][j], 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = mma(a[i], b[j], acc[i][j]);
  }
}
__device__ __forceinline__ acc16 acc_zero() {
  acc16 c;
#pragma unroll
  for (int r = 0; r < 16; ++r) c[r] = 0.f;
  return c;
}
// row of C that element r of the lane half `h` holds
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// eight consecutive result rows-of-a-lane as the k elements of the next product (round to nearest even)
template <class T>
__device__ __forceinline__ frag8<T> frag_of(const acc16 &c, int first) {
  frag8<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)c[first + j];
  return f;
}

// ------------------------------------------------------------------ global -> LDS tiles
// A tile is ROWS rows of COLS elements, row major, its 16-byte chunks permuted inside each row by
// chunk ^ swizzle(row): sixteen consecutive rows then put the same chunk into different banks (the
// row reads), and four consecutive rows the same pair of chunks (the transposing reads).
template <class T, int COLS>
struct Tile {
  static constexpr int CHUNK = 16 / (int)sizeof(T);          // elements of a 16-byte chunk
  static constexpr int CPR = COLS / CHUNK;                   // chunks of a row
  static constexpr int ROW_BYTES = COLS * (int)sizeof(T);
  static_assert(CPR == 4 || CPR == 8 || CPR >= 16, "rows of at least four chunks");
  __device__ static constexpr __forceinline__ int swizzle(int row) {
    return CPR >= 16 ? ((row & 7) << 1) | ((row >> 3) & 1)
           : CPR == 8 ? (((row >> 1) & 3) << 1) | ((row >> 3) & 1) : (((row >> 2) & 1) << 1) | ((row >> 3) & 1);
  }
  __device__ static __forceinline__ int chunk_addr(int row, int chunk) {
    return row * ROW_BYTES + ((chunk ^ swizzle(row)) << 4);
  }
  // Addresses are a lane's part, computed once, and a constant part.  The permutation is linear in the
  // bits of row and chunk, so where a row is the sum of a lane's and a constant row with no bit in common
  //   addr = (lane's row bytes | lane's chunk ^ swizzle) ^ (constant chunk ^ swizzle) + constant row bytes,
  // one exclusive or a read.
  __device__ static __forceinline__ lds_ptr at(lds_ptr tile, int lane_part, int row, int chunk) {
    return tile + (lane_part ^ ((swizzle(row) ^ chunk) << 4)) + row * ROW_BYTES;
  }
  // A lane's k elements of a product that sums over the columns: eight consecutive ones, of row
  // row0 + lane % 32 (row0 a multiple of 32) from column k0 + 8 (lane / 32).
  __device__ static __forceinline__ int row_lane(int lane) {
    return chunk_addr(lane & 31, (lane >> 5) * (8 / CHUNK));
  }
  __device__ static __forceinline__ frag8<T> row_frag(lds_ptr tile, int part, int row0, int k0) {
    if constexpr (sizeof(T) == 2) {
      return *(const DGNN_LDS frag8<T> *)at(tile, part, row0, k0 / CHUNK);
    } else {
      const vec4<T> a = *(const DGNN_LDS vec4<T> *)at(tile, part, row0, k0 / CHUNK);
      const vec4<T> b = *(const DGNN_LDS vec4<T> *)at(tile, part, row0, k0 / CHUNK + 1);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // The same in the order of the column reads below, columns k0 + 8 (j / 4) + 4 (lane / 32) + j % 4: the other
  // operand of a product with one of those.
  __device__ static __forceinline__ int row_lane_split(int lane) {
    return sizeof(T) == 2 ? chunk_addr(lane & 31, 0) + (lane >> 5) * 8 : chunk_addr(lane & 31, lane >> 5);
  }
  __device__ static __forceinline__ frag8<T> row_frag_split(lds_ptr tile, int part, int row0, int k0) {
    const vec4<T> a = *(const DGNN_LDS vec4<T> *)at(tile, part, row0, k0 / CHUNK);
    const vec4<T> b = *(const DGNN_LDS vec4<T> *)at(tile, part, row0, (k0 + 8) / CHUNK);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // A lane's k elements of a product that sums over the rows, for column col0 + lane % 32 (col0 a multiple of
  // 32): rows row0 + 8 (j / 4) + 4 (lane / 32) + j % 4 (row0 a multiple of 16).  16-bit: ds_read_b64_tr_b16
  // hands each lane of a group of sixteen one column of a 4 x 16 block, lane i supplying the address
  // of row i / 4, columns 4 (i % 4) ...
  __device__ static __forceinline__ int col_lane(int lane) {
    if (sizeof(T) == 2)
      return chunk_addr(4 * (lane >> 5) + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + (lane & 1) * 8;
    return chunk_addr(4 * (lane >> 5), (lane & 31) >> 2) + (lane & 3) * 4;
  }
  __device__ static __forceinline__ frag8<T> col_frag(lds_ptr tile, int part, int row0, int col0) {
    if constexpr (sizeof(T) == 2) {
      typedef DGNN_LDS s16x4 *lds_p;
      union { s16x4 s[2]; frag8<T> f; } u;
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)at(tile, part, row0, col0 / CHUNK));
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)at(tile, part, row0 + 8, col0 / CHUNK));
      return u.f;
    } else {
      frag8<T> f;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = *(const DGNN_LDS T *)at(tile, part, row0 + 8 * (j >> 2) + (j & 3), col0 / CHUNK);
      return f;
    }
  }
};

// Keeps the compiler from computing what depends on x once for all iterations and holding every
// result in a register of its own.
__device__ __forceinline__ int opaque(int x) {
  asm("" : "+v"(x));
  return x;
}

// 128-bit buffer descriptor over `bytes` bytes at p: reads behind them give zeros.  Both are the same in
// all lanes and are made scalars here: where the compiler cannot prove it, every load through the
// descriptor becomes a loop over the lanes' values.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_over(const void *p, unsigned bytes) {
  const unsigned long long at = (unsigned long long)p;
  const unsigned long long lo = (unsigned)uniform_i32((int)at), hi = (unsigned)uniform_i32((int)(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void *)(lo | hi << 32), 0, uniform_i32((int)bytes), 0x00020000);
}
#define DGNN_OOB 0x80000000u                       // an offset behind every descriptor used here

// Stages ROWS x COLS elements into a tile with direct loads to LDS (16 bytes a lane, no registers).  A
// wave's load fills 1024 consecutive bytes of LDS, so the permutation is applied to the address each
// lane reads.  Offsets are relative to the tile's first row and the same for every tile of a
// matrix; `bytes` of the descriptor ends with the last valid row, `cols` (elements) with the last
// valid column: what lies behind either arrives as zeros.
template <class T, int COLS, int ROWS, int THREADS>
struct Stager {
  using TL = Tile<T, COLS>;
  static constexpr int LOADS = (ROWS * TL::CPR + THREADS - 1) / THREADS;
  static_assert(ROWS * TL::CPR % 64 == 0, "whole waves");
  // 64 threads: every wave of the workgroup stages tiles of its own
  __device__ static __forceinline__ int thread() { return THREADS == 64 ? lane_id() : (int)threadIdx.x; }
  unsigned off[LOADS];
  __device__ __forceinline__ void init(unsigned row_stride_bytes, int cols) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = i * THREADS + thread(), row = c / TL::CPR, chunk = (c % TL::CPR) ^ TL::swizzle(row);
      off[i] = chunk * TL::CHUNK < cols ? row * row_stride_bytes + chunk * 16u : DGNN_OOB;
    }
  }
  // the tile's rows are rows list[0], list[1], ... of the matrix; there are `rows` of them
  __device__ __forceinline__ void init_list(const int *__restrict__ list, int rows, unsigned row_stride_bytes, int cols) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = i * THREADS + thread(), row = c / TL::CPR, chunk = (c % TL::CPR) ^ TL::swizzle(row);
      off[i] = chunk * TL::CHUNK < cols && row < rows ? (unsigned)list[row] * row_stride_bytes + chunk * 16u : DGNN_OOB;
    }
  }
  // from now on only `cols` columns exist
  __device__ __forceinline__ void narrow(int cols) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = i * THREADS + thread(), row = c / TL::CPR, chunk = (c % TL::CPR) ^ TL::swizzle(row);
      if (chunk * TL::CHUNK >= cols) off[i] = DGNN_OOB;
    }
  }
  __device__ __forceinline__ void load(lds_ptr tile, __amdgpu_buffer_rsrc_t src) const {
    const int wave = THREADS == 64 ? 0 : uniform_i32(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (ROWS * TL::CPR % THREADS == 0 || i * THREADS + wave * 64 < ROWS * TL::CPR)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(src, tile + (i * THREADS + wave * 64) * 16, 16, (int)off[i], 0, 0, 0);
  }
};

// Waits until at most N of this wave's loads are in flight.  Loads return in order, so the oldest have
// arrived; the memory clobber keeps the compiler from moving LDS reads over it.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "six bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Workgroup barrier that leaves loads to LDS in flight (__syncthreads waits for all of them).  OWN: only
// this wave's LDS reads are waited for, before loads that overwrite what they read.
template <bool OWN>
__device__ __forceinline__ void barrier_in_flight() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (!OWN) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Ring of S tile buffers over `tiles` steps: while a step works on its buffer, the loads of the next
// S - 1 are in flight.  stage(t, i) issues exactly LOADS loads of this wave into buffer i (also behind
// the last tile, where they read nothing), work(t, i) uses buffer i.  Every buffer is a __shared__
// variable of its own and the indices are constants after unrolling: the compiler, which waits for
// all loads to LDS that a read may touch, then knows which those are.
// DGNN_RING declares four; a ring of fewer leaves the others out of the kernel.
#define DGNN_RING(name, bytes)                                                                      \
  __shared__ __align__(16) char name##_0[bytes], name##_1[bytes], name##_2[bytes], name##_3[bytes]; \
  const lds_ptr name[4] = {(lds_ptr)name##_0, (lds_ptr)name##_1, (lds_ptr)name##_2, (lds_ptr)name##_3}
// OWN: the buffers belong to one wave, no barrier is needed.
template <int S, int LOADS, bool OWN, class Stage, class Work>
__device__ __forceinline__ void ring(int tiles, const Stage &stage, const Work &work) {
  if (tiles <= 0) return;
  if constexpr (S == 1) {
    constexpr std::integral_constant<int, 0> i;
    for (int t = 0; t < tiles; ++t) {
      stage(t, i);
      wait_loads<0>();
      barrier_in_flight<OWN>();
      work(t, i);
      barrier_in_flight<OWN>();
    }
    return;
  }
  unrolled<0, S - 1>([&](auto i) { stage(i.value, i); });
  auto step = [&](int t, auto i) {
    wait_loads<S == 1 ? 0 : LOADS * (S - 2)>();
    barrier_in_flight<OWN>();
    stage(t + S - 1, std::integral_constant<int, (i.value + S - 1) % S>());
    work(t, i);
  };
  // whole rounds without a branch, then the rest: joining paths, the compiler would wait for loads of
  // the path that issued fewer
  int t = 0;
  for (; t + S <= tiles; t += S) unrolled<0, S>([&](auto i) { step(t + i.value, i); });
  unrolled<0, S - 1>([&](auto i) {
    if (t + i.value < tiles) step(t + i.value, i);
  });
  wait_loads<0>();                             // the loads behind the last tile still write LDS
}

// One load of 4 bytes a lane to 64 consecutive words of LDS.
__device__ __forceinline__ void load_words(lds_ptr to, __amdgpu_buffer_rsrc_t src, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, to, 4, (int)off, 0, 0, 0);
}

// bytes a descriptor over `rows` rows spans (0 rows: nothing is readable)
__device__ __forceinline__ unsigned span_bytes(int rows, unsigned row_stride_bytes, unsigned row_bytes) {
  return rows > 0 ? (unsigned)(rows - 1) * row_stride_bytes + row_bytes : 0u;
}

}  // namespace dgnn
