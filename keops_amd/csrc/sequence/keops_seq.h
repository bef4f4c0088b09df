// Device helpers shared by the sequence operators (keops_seq_attention.hip, keops_seq_decay.hip, keops_seq_logprobs.hip):
// matrix-core fragments of 32x32 tiles and tiles staged in LDS.
//
// Fragments.  Every product here is a 32x32 tile C += A B, 16 steps of the contraction at a time, of one wavefront; lane l has
// col = l % 32 and half = l / 32.
//   A operand: row = col of the lane, contraction steps 8*half + (0..7);   B operand: column = col, the same steps.
//   C tile: column = col, register r holds row 8*(r/4) + 4*half + r%4.
// The contraction is a sum, so its steps may be numbered in any order as long as A and B agree.  A C tile whose rows become the
// contraction of the next product (probabilities times values) is therefore used as a B operand without moving a value between
// lanes: registers 8s..8s+7 are the steps 16s + 4*half + (0..3) and 16s + 8 + 4*half + (0..3), and the other operand is read
// in that order (frag_cols, frag_rows_split).
//
// Operand types.  bf16 and f16: the 16-bit matrix instructions (products exact, sums in float32).  Split<N>: a number as the sum of
// N bf16 terms, each the rounding of what the ones before leave: two terms hold 16 bits (a float16 exactly, with bf16's range:
// products and probabilities of float16 inputs may leave float16's), three hold a float32.  A product of split operands is the
// sum of the products of terms that are not below its last bit: 3 instructions for two terms, 6 for three (the float32 matrix
// instruction takes the time of 16).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace kseq {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int N> struct Split {};
template <int N> struct SplitX8 { bf16x8 t[N]; };

template <class T> struct Vec;  // eight contraction steps as an operand, four neighbouring values, the element of a tile in LDS
template <> struct Vec<bf16> { typedef bf16x8 x8; typedef bf16x4 x4; typedef bf16 lds; static constexpr int terms = 1; };
template <> struct Vec<f16> { typedef f16x8 x8; typedef f16x4 x4; typedef f16 lds; static constexpr int terms = 1; };
template <int N> struct Vec<Split<N>> { typedef SplitX8<N> x8; typedef bf16 lds; static constexpr int terms = N; };
template <> struct Vec<float> { typedef f32x4 x4; };
template <class T> using lds_t = typename Vec<T>::lds;
template <class T> using frag_t = typename Vec<T>::x8;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

__device__ inline f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; r++) z[r] = 0.f;
  return z;
}

__device__ inline f32x16 mma(const bf16x8& a, const bf16x8& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mma(const f16x8& a, const f16x8& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
template <int N, int M> __device__ inline f32x16 mma(const SplitX8<N>& a, const SplitX8<M>& b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int j = 0; j < M; j++)
      if (i + j < (N > M ? N : M)) c = mma(a.t[i], b.t[j], c);
  return c;
}
template <int M> __device__ inline f32x16 mma(const bf16x8& a, const SplitX8<M>& b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < M; j++) c = mma(a, b.t[j], c);
  return c;
}

// eight float32 values as an operand
template <class T> __device__ inline frag_t<T> to_frag(const float (&x)[8]) {
  frag_t<T> f;
#pragma unroll
  for (int j = 0; j < 8; j++) f[j] = (T)x[j];
  return f;
}
template <int N> __device__ inline SplitX8<N> to_split(const float (&x)[8]) {
  SplitX8<N> f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    float rest = x[j];
#pragma unroll
    for (int n = 0; n < N; n++) {
      const bf16 e = (bf16)rest;
      f.t[n][j] = e;
      rest -= (float)e;
    }
  }
  return f;
}
template <> __device__ inline SplitX8<2> to_frag<Split<2>>(const float (&x)[8]) { return to_split<2>(x); }
template <> __device__ inline SplitX8<3> to_frag<Split<3>>(const float (&x)[8]) { return to_split<3>(x); }

// and back
template <class V> __device__ inline void to_float(const V& f, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = (float)f[j];
}
template <int N> __device__ inline void to_float(const SplitX8<N>& f, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++) {
    x[j] = (float)f.t[N - 1][j];
#pragma unroll
    for (int n = N - 2; n >= 0; n--) x[j] += (float)f.t[n][j];
  }
}

// row of register r of a C tile
__device__ inline constexpr int c_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

// Tiles in LDS: rows of DP elements, a split type's terms one behind the other (N times DP elements of bf16).  No padding: the
// 16-byte piece c of row r lies at place c ^ swizzle(r).  LDS has 64 banks (256 bytes): a row read takes the same piece of 16 rows
// at a time, a transposing read 64 neighbouring bytes of four rows; the exclusive-or spreads both over all banks.
template <class T, int DP> constexpr int tile_stride() { return Vec<T>::terms * DP; }
template <int LENGTH> __device__ inline int swizzle(int row) {  // LENGTH: of a row, in two-byte elements
  if constexpr (LENGTH % 128 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);  // rows begin at the same bank: 16 pieces
  else if constexpr (LENGTH % 128 == 64) return ((row & 2) << 1) | ((row >> 2) & 3);  // 128 bytes apart: 8 pieces
  else return (row >> 2) & 3;                                                   // 64 bytes apart: 4 pieces
}
// offset of element `col` of row `row`
template <class T, int DP> __device__ inline int tile_at(int row, int col) {
  constexpr int LENGTH = tile_stride<T, DP>();
  return row * LENGTH + ((((col >> 3) ^ swizzle<LENGTH>(row)) << 3) | (col & 7));
}

template <class T, class F> __device__ inline frag_t<T> each_term(const F& read) {  // read(n, x): term n of an operand into x
  frag_t<T> f;
  if constexpr (Vec<T>::terms == 1) {
    read(0, f);
  } else {
#pragma unroll
    for (int n = 0; n < Vec<T>::terms; n++) read(n, f.t[n]);
  }
  return f;
}

// contraction steps k0 + 8*half + (0..7) of one row
template <class T, int DP> __device__ inline frag_t<T> frag_rows(const lds_t<T>* tile, int row, int k0, int half) {
  return each_term<T>([&](int n, auto& x) __attribute__((always_inline)) {
    x = *reinterpret_cast<const typename Vec<lds_t<T>>::x8*>(tile + tile_at<T, DP>(row, n * DP + k0 + 8 * half));
  });
}
// contraction steps k0 + 4*half + (0..3), k0 + 8 + 4*half + (0..3) of one row: the order of a C tile's registers
template <class T, int DP> __device__ inline frag_t<T> frag_rows_split(const lds_t<T>* tile, int row, int k0, int half) {
  typedef typename Vec<lds_t<T>>::x4 x4;
  return each_term<T>([&](int n, auto& x) __attribute__((always_inline)) {
    const x4 a = *reinterpret_cast<const x4*>(tile + tile_at<T, DP>(row, n * DP + k0 + 4 * half));
    const x4 b = *reinterpret_cast<const x4*>(tile + tile_at<T, DP>(row, n * DP + k0 + 8 + 4 * half));
    x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  });
}
// The transpose: column c0 + col of rows r0 + 4*half + (0..3) and r0 + 8 + 4*half + (0..3) of a tile in LDS, through the
// transposing LDS read: of each 16 lanes, lane i addresses four neighbouring elements of row i / 4 and receives column i of the
// four rows.
template <class T, int DP> __device__ inline frag_t<T> frag_cols(const lds_t<T>* tile, int r0, int c0, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds4;
  const int i = lane & 15, row = r0 + 4 * (lane >> 5) + (i >> 2), col = c0 + (lane & 16) + 4 * (i & 3);
  return each_term<T>([&](int n, auto& x) __attribute__((always_inline)) {
    union { s16x4 v[2]; typename Vec<lds_t<T>>::x8 x; } u;
    u.v[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + tile_at<T, DP>(row, n * DP + col)));
    u.v[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + tile_at<T, DP>(row + 8, n * DP + col)));
    x = u.x;
  });
}

// registers 8s..8s+7 of a C tile as an operand, rounded to the operand's type
template <class T> __device__ inline frag_t<T> pack(const f32x16& c, int s) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = c[8 * s + j];
  return to_frag<T>(x);
}

// 16 bytes of a row in memory (column `col`) into a tile, times `weight` where the type is split
template <class Tin, class T, int DP> __device__ inline void put_piece(lds_t<T>* tile, int row, int col, const uint4& r, float weight = 1.f) {
  constexpr int VE = 16 / (int)sizeof(Tin);
  if constexpr (Vec<T>::terms == 1) {
    *reinterpret_cast<uint4*>(tile + tile_at<T, DP>(row, col)) = r;
  } else {
    union { uint4 u; Tin e[VE]; } x;
    x.u = r;
    float rest[VE];
#pragma unroll
    for (int j = 0; j < VE; j++) rest[j] = (float)x.e[j] * weight;
#pragma unroll
    for (int n = 0; n < Vec<T>::terms; n++) {
      bf16 t[VE] __attribute__((aligned(16)));
#pragma unroll
      for (int j = 0; j < VE; j++) {
        t[j] = (bf16)rest[j];
        rest[j] -= (float)t[j];
      }
      if constexpr (VE == 8) *reinterpret_cast<uint4*>(tile + tile_at<T, DP>(row, n * DP + col)) = *reinterpret_cast<const uint4*>(t);
      else *reinterpret_cast<uint2*>(tile + tile_at<T, DP>(row, n * DP + col)) = *reinterpret_cast<const uint2*>(t);
    }
  }
}
// four neighbouring values of a row of a tile
template <class T, int DP> __device__ inline void put4(lds_t<T>* tile, int row, int col, float a, float b, float c, float d) {
  float rest[4] = {a, b, c, d};
#pragma unroll
  for (int n = 0; n < Vec<T>::terms; n++) {
    typename Vec<lds_t<T>>::x4 v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[j] = (lds_t<T>)rest[j];
      rest[j] -= (float)v[j];
    }
    *reinterpret_cast<typename Vec<lds_t<T>>::x4*>(tile + tile_at<T, DP>(row, n * DP + col)) = v;
  }
}

// Places in LDS are the same in every turn of a loop.  Formed from a lane that the compiler knows nothing of, they are formed anew
// in each turn (some ten instructions) and do not stay in tens of registers all along.  Where registers are short that is worth
// it (without and with, us): decay_attention of 16 x 16384 tokens, 128 components, 217 and 135, its training at 2x16x4096 392 and 243;
// training of bucket_attention, 2x8x4096^2, 128 components (gradient of the queries) 593 and 568, 2x8x1024^2 float32 337 and 252.
// Where they are not it costs: a forward pass of 8x16384^2 655 and 752, decay_attention of 2x16x2048 float32 112 and 119.
__device__ inline void forget(int& lane, int& half, int& col) {
  asm volatile("" : "+v"(lane));
  half = lane >> 5;
  col = lane & 31;
}

// A tile of ROWS x DP elements on its way from memory to LDS, held in the registers of a workgroup of NT threads: rows from
// `left` on and columns from `dim` on are zeros and are not read, so what lies behind them never enters a product.  `base` is the
// tile's first row, the same for all threads; a thread's offset to it is 32 bits (rows are at most kMaxRowStride apart).
// REVERSE: row r lies r rows before `base`.
constexpr long long kMaxRowStride = 1ll << 23;  // elements: 64 rows of 4 bytes span 2^31 bytes

template <class Tin, class Tc, int ROWS, int DP, int NT = 256, bool REVERSE = false> struct Staged {
  static constexpr int VE = 16 / (int)sizeof(Tin), PER_ROW = DP / VE, TOTAL = ROWS * PER_ROW, N = (TOTAL + NT - 1) / NT;
  uint4 r[N];
  __device__ inline void load(const Tin* base, long long stride, int left, int dim, int tid) {
    const char* lowest = (const char*)(REVERSE ? base - (ROWS - 1) * stride : base);
    const bool whole = left >= ROWS && dim == DP && TOTAL % NT == 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int c = tid + NT * i, row = c / PER_ROW, col = (c % PER_ROW) * VE;
      const unsigned off = ((unsigned)(REVERSE ? ROWS - 1 - row : row) * (unsigned)stride + (unsigned)col) * (unsigned)sizeof(Tin);
      if (whole) {
        r[i] = *reinterpret_cast<const uint4*>(lowest + off);
      } else {
        r[i] = make_uint4(0u, 0u, 0u, 0u);
        if ((TOTAL % NT == 0 || c < TOTAL) && row < left && col < dim) r[i] = *reinterpret_cast<const uint4*>(lowest + off);
      }
    }
  }
  __device__ inline void store(lds_t<Tc>* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int c = tid + NT * i;
      if (TOTAL % NT != 0 && c >= TOTAL) break;
      put_piece<Tin, Tc, DP>(tile, c / PER_ROW, (c % PER_ROW) * VE, r[i]);
    }
  }
  // row j times weights[-j] * scale
  __device__ inline void store(lds_t<Tc>* tile, int tid, const float* weights, float scale) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int c = tid + NT * i, row = c / PER_ROW;
      if (TOTAL % NT != 0 && c >= TOTAL) break;
      put_piece<Tin, Tc, DP>(tile, row, (c % PER_ROW) * VE, r[i], weights[-row] * scale);
    }
  }
};

// contraction steps k0 + 8*half + (0..7) of a row in memory (zeros where the row or the columns do not exist)
template <class Tin, class Tc> __device__ inline frag_t<Tc> frag_global(const Tin* row, bool there, int k0, int half, int dim) {
  constexpr int VE = 16 / (int)sizeof(Tin);
  if constexpr (Vec<Tc>::terms == 1) {
    union { uint4 u; frag_t<Tc> x; } w;
    w.u = make_uint4(0u, 0u, 0u, 0u);
    if (there && k0 + 8 * half < dim) w.u = *reinterpret_cast<const uint4*>(row + k0 + 8 * half);
    return w.x;
  } else {
    float x[8];
#pragma unroll
    for (int p = 0; p < 8 / VE; p++) {
      union { uint4 u; Tin e[VE]; } w;
      w.u = make_uint4(0u, 0u, 0u, 0u);
      const int c = k0 + 8 * half + p * VE;
      if (there && c < dim) w.u = *reinterpret_cast<const uint4*>(row + c);
#pragma unroll
      for (int j = 0; j < VE; j++) x[p * VE + j] = (float)w.e[j];
    }
    return to_frag<Tc>(x);
  }
}

// four neighbouring values of an output row
template <class T> __device__ inline void store4(T* dst, float a, float b, float c, float d) {
  typename Vec<T>::x4 v;
  v[0] = (T)a; v[1] = (T)b; v[2] = (T)c; v[3] = (T)d;
  *reinterpret_cast<typename Vec<T>::x4*>(dst) = v;
}

}  // namespace kseq

// Host side: message behind keops_hip_last_error() (defined in keops_hip.cpp); returns `code`.
int keops_seq_fail(int code, const char* message);

inline bool rows_aligned(const void* p, const int64_t* stride, size_t size) {  // rows that start at multiples of 16 bytes
  return !p || ((uintptr_t)p % 16 == 0 && stride[0] * size % 16 == 0 && stride[1] * size % 16 == 0 && stride[2] * size % 16 == 0);
}

struct SeqDevice {  // makes `device` current, and gives the caller's back
  int before = -1, now;
  explicit SeqDevice(int device) : now(device) {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
    if (before != now) (void)hipSetDevice(now);
  }
  ~SeqDevice() {
    if (before >= 0 && before != now) (void)hipSetDevice(before);
  }
};

inline int seq_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : keops_seq_fail((int)e, what);
}
