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
// Element types.  bf16 and fp16 multiply on the 16-bit matrix instructions (products exact, sums in float32); float32 on
// v_mfma_f32_32x32x2_f32, 8 instructions for the same 16 steps.
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
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T> struct Vec;
template <> struct Vec<bf16> { typedef bf16x8 x8; typedef bf16x4 x4; };
template <> struct Vec<f16> { typedef f16x8 x8; typedef f16x4 x4; };
template <> struct Vec<float> { typedef f32x8 x8; typedef f32x4 x4; };

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
__device__ inline f32x16 mma(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// row of register r of a C tile
__device__ inline constexpr int c_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

// Tiles in LDS: rows of DP elements.  Two-byte elements: no padding, the 16-byte piece c of row r lies at place c ^ swizzle(r).
// LDS has 64 banks (256 bytes): a row read takes the same piece of 16 rows at a time, a transposing read 64 neighbouring bytes of
// four rows; the exclusive-or spreads both over all banks.  float32: rows padded by 16 bytes, no exclusive-or.
template <class T, int DP> constexpr int tile_stride() { return sizeof(T) == 2 ? DP : DP + 4; }
template <class T, int DP> __device__ inline int swizzle(int row) {
  if constexpr (sizeof(T) != 2) return 0;
  else if constexpr (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);           // 256-byte rows: 16 pieces
  else if constexpr (DP == 64) return ((row & 2) << 1) | ((row >> 2) & 3);            // two rows to 256 bytes: 8 pieces
  else return (row >> 2) & 3;                                                         // 64 and 192 bytes: rows begin 64 bytes apart, 4 pieces
}
// offset of element `col` of row `row` (col: a multiple of 16 bytes, or within a piece)
template <class T, int DP> __device__ inline int tile_at(int row, int col) {
  if constexpr (sizeof(T) != 2) return row * tile_stride<T, DP>() + col;
  else return row * DP + ((((col >> 3) ^ swizzle<T, DP>(row)) << 3) | (col & 7));
}

// contraction steps k0 + 8*half + (0..7) of one row
template <class T, int DP> __device__ inline typename Vec<T>::x8 frag_rows(const T* tile, int row, int k0, int half) {
  return *reinterpret_cast<const typename Vec<T>::x8*>(tile + tile_at<T, DP>(row, k0 + 8 * half));
}
// contraction steps k0 + 4*half + (0..3), k0 + 8 + 4*half + (0..3) of one row: the order of a C tile's registers
template <class T, int DP> __device__ inline typename Vec<T>::x8 frag_rows_split(const T* tile, int row, int k0, int half) {
  typedef typename Vec<T>::x4 x4;
  const x4 a = *reinterpret_cast<const x4*>(tile + tile_at<T, DP>(row, k0 + 4 * half));
  const x4 b = *reinterpret_cast<const x4*>(tile + tile_at<T, DP>(row, k0 + 8 + 4 * half));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The transpose: column c0 + col of rows r0 + 4*half + (0..3) and r0 + 8 + 4*half + (0..3) of a tile in LDS.  Two-byte elements
// come through the transposing LDS read: of each 16 lanes, lane i addresses four neighbouring elements of row i / 4 and
// receives column i of the four rows.
template <class T, int DP> __device__ inline typename Vec<T>::x8 frag_cols(const T* tile, int r0, int c0, int lane) {
  const int half = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const int i = lane & 15, row = r0 + 4 * half + (i >> 2), col = c0 + (lane & 16) + 4 * (i & 3);
    union { s16x4 v[2]; typename Vec<T>::x8 x; } u;
    u.v[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + tile_at<T, DP>(row, col)));
    u.v[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + tile_at<T, DP>(row + 8, col)));
    return u.x;
  } else {
    constexpr int ST = tile_stride<T, DP>();
    const T* p = tile + (r0 + 4 * half) * ST + c0 + (lane & 31);
    typename Vec<T>::x8 x;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[j] = p[j * ST];
      x[4 + j] = p[(8 + j) * ST];
    }
    return x;
  }
}

// registers 8s..8s+7 of a C tile as an operand, rounded to the operand's type
template <class T> __device__ inline typename Vec<T>::x8 pack(const f32x16& c, int s) {
  typename Vec<T>::x8 x;
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = (T)c[8 * s + j];
  return x;
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
  __device__ inline void store(Tc* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int c = tid + NT * i, row = c / PER_ROW, col = (c % PER_ROW) * VE;
      if (TOTAL % NT != 0 && c >= TOTAL) break;
      Tc* dst = tile + tile_at<Tc, DP>(row, col);
      if constexpr (sizeof(Tin) == sizeof(Tc)) {
        *reinterpret_cast<uint4*>(dst) = r[i];
      } else {
        union { uint4 u; Tin e[VE]; } x;
        x.u = r[i];
#pragma unroll
        for (int j = 0; j < VE; j++) dst[j] = (Tc)x.e[j];
      }
    }
  }
};

// contraction steps k0 + 8*half + (0..7) of a row in memory (zeros where the row or the columns do not exist)
template <class Tin, class Tc> __device__ inline typename Vec<Tc>::x8 frag_global(const Tin* row, bool there, int k0, int half, int dim) {
  constexpr int VE = 16 / (int)sizeof(Tin);
  typename Vec<Tc>::x8 x;
#pragma unroll
  for (int p = 0; p < 8 / VE; p++) {
    union { uint4 u; Tin e[VE]; } w;
    w.u = make_uint4(0u, 0u, 0u, 0u);
    const int c = k0 + 8 * half + p * VE;
    if (there && c < dim) w.u = *reinterpret_cast<const uint4*>(row + c);
#pragma unroll
    for (int j = 0; j < VE; j++) x[p * VE + j] = (Tc)w.e[j];
  }
  return x;
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
