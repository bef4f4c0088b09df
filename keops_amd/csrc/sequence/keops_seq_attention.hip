// Softmax attention with a learned bias by buckets of the relative position:
//
//   z_ij = scale <q_i, k_j> + bias[h][bucket(j - p_i)],   p_i = query_start + i,   o_i = sum_j softmax_j(z)_ij v_j
//
// and its gradients.  bucket() is a table over the clamped distance -reach..reach, so beyond the reach on either side the bias
// is one number for a head: tiles of pairs that lie there whole take it as a scalar, the others read a table of the head's
// biases by distance in LDS, in which the four neighbouring keys of a lane's registers are neighbours.
#include "../../../include/keops_hip.h"
#include "keops_seq.h"

using namespace kseq;

namespace {

typedef keops_hip_bucket_attention Args;

constexpr int kPad = 96;  // entries of the distance table beyond the reach on each side: a mixed tile of 64 x 32 pairs reads there

__device__ inline int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

struct Span {  // what one sequence of the batch sees
  int klen;    // keys that exist
  int start;   // key position of query 0
};
__device__ inline Span span_of(const Args& A, int b) {
  Span s;
  const int n = (int)A.keys;
  s.klen = A.key_lengths ? clampi(A.key_lengths[b], 0, n) : n;
  s.start = A.query_start ? clampi(A.query_start[b], -(1 << 29), 1 << 29) : (int)A.start;
  return s;
}

// Unit (sequence and key/value head) and block within it of a workgroup: block by block over the units.  With a causal bound the
// blocks are of very different length, and the longest of all units come first.  Workgroups go to the 8 XCDs in turn, so with a
// multiple of 8 units the blocks of one unit share an XCD's L2.
__device__ inline void block_of(unsigned w, int units, int& unit, int& block) {
  unit = w % units;
  block = w / units;
}

// A bias of -6e4 or less (the lowest fp16 is -65504; masks of the type's lowest value) hides its pairs as -inf does: next to such a
// number a float32 logit keeps nothing of the product, and a row of nothing else would be an average of what was masked.
__device__ inline float bias_of(float x) { return x <= -6e4f ? -kInf : x * kLog2e; }

// biases of head h by distance, times log2(e), padded on both sides
__device__ inline void fill_table(float* table, const Args& A, int h, int tid, int nthreads) {
  const int top = 2 * A.reach;
  for (int i = tid; i <= top + 2 * kPad; i += nthreads) table[i] = bias_of(A.bias[(long long)h * A.buckets + A.bucket_of[clampi(i - kPad, 0, top)]]);
}

template <class T> __device__ inline const T* rows_of(const void* p, const int64_t* s, int b, int h) { return (const T*)p + (long long)b * s[0] + (long long)h * s[1]; }
template <class T> __device__ inline T* rows_of(void* p, const int64_t* s, int b, int h) { return (T*)p + (long long)b * s[0] + (long long)h * s[1]; }

// outputs, and what their rounding leaves
template <class Tin> __device__ inline void put_out(const Args& A, int b, int h, int row, int d, float x) {
  const Tin v = (Tin)x;
  rows_of<Tin>(A.out, A.out_stride, b, h)[(long long)row * A.out_stride[2] + d] = v;
  if (A.out_rest) rows_of<Tin>(A.out_rest, A.out_stride, b, h)[(long long)row * A.out_stride[2] + d] = (Tin)(x - (float)v);
}
template <class Tin> __device__ inline float left_of(float x) { return x - (float)(Tin)x; }

// Keys of a staged tile: 32 where 64 would not leave the rows in flight, the logits and the sums in 256 registers.  Forward pass of
// 4x8x4096^2, 64 components, 64 keys 115 us and 32 keys 127; 8x16384^2, 128 components, 64 keys 1557 us (spilled) and 32 keys 672.
template <class Tc, int DP> constexpr int key_tile() { return Vec<Tc>::terms == 1 && DP <= 64 ? 64 : 32; }
// Queries of one, where keys are in registers: 64 against 32, training of 4x8x4096^2, 64 components, 436 and 448 us; 2x8x4096^2, 128
// components, 568 and 582.  (Four tiles of 64 rows of three terms would not fit in LDS.)
template <class Tc> constexpr int query_tile() { return Vec<Tc>::terms == 1 ? 64 : 32; }

// wavefronts a SIMD: wide split rows need more than 256 registers
template <class Tc, int DP> constexpr int waves(int widest = 64) { return Vec<Tc>::terms > 1 && DP > widest ? 1 : 2; }

// logits (base 2, less `less`) of a 32 x 32 tile in place: rows are keys kb + 8g + 4 half + t, the lane's column is the query at
// position pos.  kind: 0 within the reach of the buckets, otherwise the bias is `far`; keys from `lim` on do not count (mask).
__device__ inline void logits_by_key(f32x16& s, float scale2, const float* table, float less, float far, int kind, bool mask, int lim, int kb, int pos,
                                     int half, int reach) {
  if (kind == 0) {
    const float* tp = table + (kb - pos + reach + kPad + 4 * half);
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = fmaf(s[r], scale2, tp[8 * (r / 4) + r % 4]) - less;
  } else {
    const float c = far - less;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = fmaf(s[r], scale2, c);
  }
  if (mask) {
    const int rel = lim - kb - 4 * half;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = 8 * (r / 4) + r % 4 < rel ? s[r] : -kInf;
  }
}

template <class T> constexpr bool is_f16 = false;
template <> constexpr bool is_f16<f16> = true;

// Score gradients as float16 operands: products of probabilities and gradients may lie far below or above float16's range, so each
// lane's column is held times a power of two that puts its largest value so far between 2^13 and 2^15; what has been summed
// follows when that changes.  (Types with float32's range are left alone.)
template <class Tc> struct Scaled {
  template <int ND> __device__ inline void fit(f32x16&, f32x16 (&)[ND]) {}
  __device__ inline float inverse() const { return 1.f; }
};
template <> struct Scaled<f16> {
  float factor = 1.f, most = 0.f;  // most: the largest value that the factor is good for (0: none seen)
  template <int ND> __device__ inline void fit(f32x16& s, f32x16 (&acc)[ND]) {
    float mx = fabsf(s[0]);
#pragma unroll
    for (int r = 1; r < 16; r++) mx = fmaxf(mx, fabsf(s[r]));
    if (__any(mx > most)) {
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      if (mx > most && mx < kInf) {
        const int e = __builtin_amdgcn_frexp_expf(mx);                  // 2^(e-1) <= mx < 2^e
        const float to = __builtin_amdgcn_ldexpf(1.f, min(14 - e, 120)), by = most == 0.f ? 0.f : to / factor;
#pragma unroll
        for (int k = 0; k < ND; k++)
#pragma unroll
          for (int r = 0; r < 16; r++) acc[k][r] *= by;
        factor = to;
        most = 32768.f / to;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] *= factor;
  }
  __device__ inline float inverse() const { return 1.f / factor; }
};

// Where few blocks would leave the chip empty, the tiles that a block walks over are shared by several workgroups, whose float32
// sums are joined: place of one row in the workspace, in records.
__device__ inline long long share_of(const Args& A, int unit, int splits, int split, int h, int row) {
  const int group = A.heads / A.kv_heads;
  return ((long long)(unit * splits + split) * group + h % group) * A.queries + row;
}

// ---- forward --------------------------------------------------------------------------------------------------------------
//
// One pass over the keys with a running reference point and sum.  A workgroup of four wavefronts has 128 queries of one head, a
// wavefront 32 of them, one to a lane pair; tiles of 64 keys are staged in LDS, double buffered, one barrier a tile.  The logits
// are computed transposed (rows keys, columns queries), so a query's sum is an in-lane reduction, and the probabilities enter the
// product with the values as they are (keops_seq.h).
//
// Logits are formed less the reference point, so probabilities are exp2 of one multiply-add.  The point moves only when a logit
// exceeds it by more than 8 (probabilities up to 2^8 lose nothing: the sum is kept in float32 and 16-bit operands have the same
// relative step there).
//
// 8 x 16384^2 causal bf16, 128 components: 672 us, 0.82 Pflop/s (a library product of 8192^3 reaches 1.21); 4x8 x 4096^2, 64
// components: 115 us, 0.60.  Of a SIMD's cycles the matrix instructions take 35 % (64 components: 28 %), vector instructions 39 %
// (51 %): they hardly run side by side, and the exponential, which costs as much as four multiplications, is the largest part.
// Not kept: products a tile ahead of the softmax (162 us for 111), three wavefronts a SIMD (127 with tiles of 32 keys, which two
// take as well), places in LDS formed anew in each turn (752 us for 655), priorities around the products (680 for 673).
template <class Tin, class Tc, int DP>
__global__ void __launch_bounds__(256, (waves<Tc, DP>())) attention_forward(const Args A, int splits, float* part) {
  constexpr int KT = key_tile<Tc, DP>(), SUB = KT / 32, ST = tile_stride<Tc, DP>(), NS = DP / 16, ND = DP / 32;
  typedef typename Vec<Tc>::x8 frag;
  extern __shared__ __align__(16) unsigned char smem[];
  lds_t<Tc>* const ktiles = (lds_t<Tc>*)smem;  // [2][KT][ST]
  lds_t<Tc>* const vtiles = ktiles + 2 * KT * ST;
  float* const table = (float*)(vtiles + 2 * KT * ST);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int group = A.heads / A.kv_heads, M = (int)A.queries, nqb = (M + 127) / 128;
  int unit, block;
  block_of(blockIdx.x, A.batch * A.kv_heads, unit, block);
  const int split = block % splits;
  block /= splits;
  const int b = unit / A.kv_heads, kvh = unit % A.kv_heads, h = kvh * group + block % group, qb = nqb - 1 - block / group;
  const Span sp = span_of(A, b);
  fill_table(table, A, h, tid, 256);

  const int pos_lo = sp.start + qb * 128 + wave * 32, pos_hi = pos_lo + 31, row = qb * 128 + wave * 32 + col, pos = pos_lo + col;
  const Tin* const K = rows_of<Tin>(A.k, A.k_stride, b, kvh);
  const Tin* const V = rows_of<Tin>(A.v, A.v_stride, b, kvh);
  const long long ks = A.k_stride[2], vs = A.v_stride[2];
  frag qf[NS];
  {
    const Tin* q = rows_of<Tin>(A.q, A.q_stride, b, h) + (long long)row * A.q_stride[2];
#pragma unroll
    for (int i = 0; i < NS; i++) qf[i] = frag_global<Tin, Tc>(q, row < M, 16 * i, half, A.dim);
  }
  const int kend = A.causal ? min(sp.klen, sp.start + min(qb * 128 + 128, M)) : sp.klen;  // keys that the workgroup sees
  const int wend = A.causal ? min(kend, pos_hi + 1) : kend;                                // and this wavefront
  const int alltiles = kend > 0 ? (kend + KT - 1) / KT : 0, first = alltiles * split / splits, ntiles = alltiles * (split + 1) / splits;
  const int lim = A.causal ? min(sp.klen, pos + 1) : sp.klen;
  const float scale2 = A.scale * kLog2e;

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; i++) acc[i] = zero16();
  float m = 0.f, l = 0.f, above = -kInf;  // reference point, sum, by what a logit may exceed the reference (-inf: none yet)

  Staged<Tin, Tc, KT, DP> sk, sv;
  const auto fetch = [&](int t) __attribute__((always_inline)) {
    sk.load(K + (long long)t * KT * ks, ks, sp.klen - t * KT, A.dim, tid);
    sv.load(V + (long long)t * KT * vs, vs, sp.klen - t * KT, A.dim, tid);
  };
  const auto put = [&](int t) __attribute__((always_inline)) {
    sk.store(ktiles + (t & 1) * KT * ST, tid);
    sv.store(vtiles + (t & 1) * KT * ST, tid);
  };
  if (first < ntiles) {
    fetch(first);
    put(first);
    if (first + 1 < ntiles) fetch(first + 1);
  }
  __syncthreads();
  const float left = table[0], right = table[2 * A.reach + 2 * kPad];
  for (int t = first; t < ntiles; t++) {
    if constexpr (Vec<Tc>::terms > 1) forget(lane, half, col);
    const lds_t<Tc>* kt = ktiles + (t & 1) * KT * ST;
    const lds_t<Tc>* vt = vtiles + (t & 1) * KT * ST;
    if (t + 1 < ntiles) {
      put(t + 1);
      if (t + 2 < ntiles) fetch(t + 2);
    }
    const int kb = t * KT;
    if (kb < wend) {
      f32x16 s[SUB];
      float mx;
      const int kind = kb - pos_hi >= A.reach ? 1 : (kb + KT - 1 - pos_lo <= -A.reach ? -1 : 0);
      const bool mask = kb + KT > sp.klen || (A.causal && kb + KT - 1 > pos_lo);
      const auto logits = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SUB; u++) {
          s[u] = zero16();
#pragma unroll
          for (int i = 0; i < NS; i++) s[u] = mma(frag_rows<Tc, DP>(kt, 32 * u + col, 16 * i, half), qf[i], s[u]);
        }
#pragma unroll
        for (int u = 0; u < SUB; u++) logits_by_key(s[u], scale2, table, m, kind > 0 ? right : left, kind, mask, lim, kb + 32 * u, pos, half, A.reach);
        mx = s[0][0];
#pragma unroll
        for (int u = 0; u < SUB; u++)
#pragma unroll
          for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[u][r]);
      };
      logits();
      if (__any(mx > above)) {
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > 192.f && above > 0.f)) {
          // so far beyond the reference that nothing before counts, and that the difference may have lost what the logit was made
          // of: such rows begin again, from the products
          if (mx > 192.f && above > 0.f) {
            m = l = 0.f;
            above = -kInf;
#pragma unroll
            for (int k = 0; k < ND; k++) acc[k] = zero16();
          }
          logits();
          mx = fmaxf(mx, __shfl_xor(mx, 32));
        }
        const float d = mx > above ? mx : 0.f, f = above == -kInf ? 0.f : __builtin_amdgcn_exp2f(-d);
        above = mx > above ? 8.f : above;
        m += d;
        l *= f;
#pragma unroll
        for (int u = 0; u < SUB; u++)
#pragma unroll
          for (int r = 0; r < 16; r++) s[u][r] -= d;
#pragma unroll
        for (int k = 0; k < ND; k++)
#pragma unroll
          for (int r = 0; r < 16; r++) acc[k][r] *= f;
      }
#pragma unroll
      for (int u = 0; u < SUB; u++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[u][r] = __builtin_amdgcn_exp2f(s[u][r]);
          l += s[u][r];
        }
      // probabilities rounded to the values' type for the product (2^-9 relative for bf16, as much as the output's own rounding)
#pragma unroll
      for (int u = 0; u < SUB; u++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const frag p = pack<Tc>(s[u], k);
#pragma unroll
          for (int i = 0; i < ND; i++) acc[i] = mma(frag_cols<Tc, DP>(vt, 32 * u + 16 * k, 32 * i, lane), p, acc[i]);
        }
    }
    __syncthreads();
  }
  l += __shfl_xor(l, 32);
  if (splits > 1) {
    if (row < M) {
      float* p = part + share_of(A, unit, splits, split, h, row) * (DP + 4);
      if (half == 0) {
        p[0] = l == 0.f ? -kInf : m;
        p[1] = l;
      }
#pragma unroll
      for (int i = 0; i < ND; i++)
#pragma unroll
        for (int g = 0; g < 4; g++) store4<float>(p + 4 + 32 * i + 8 * g + 4 * half, acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]);
    }
    return;
  }
  if (row < M) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    Tin* o = rows_of<Tin>(A.out, A.out_stride, b, h) + (long long)row * A.out_stride[2];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int d = 32 * i + 8 * g + 4 * half;
        if (d < A.dim) store4<Tin>(o + d, acc[i][4 * g] * inv, acc[i][4 * g + 1] * inv, acc[i][4 * g + 2] * inv, acc[i][4 * g + 3] * inv);
      }
    if (A.out_rest) {
      Tin* rest = rows_of<Tin>(A.out_rest, A.out_stride, b, h) + (long long)row * A.out_stride[2];
#pragma unroll
      for (int i = 0; i < ND; i++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const int d = 32 * i + 8 * g + 4 * half;
          if (d < A.dim)
            store4<Tin>(rest + d, left_of<Tin>(acc[i][4 * g] * inv), left_of<Tin>(acc[i][4 * g + 1] * inv), left_of<Tin>(acc[i][4 * g + 2] * inv),
                        left_of<Tin>(acc[i][4 * g + 3] * inv));
        }
    }
    // base-2 log of the row's sum; a row that sees nothing gets +inf, with which its probabilities are zeros later
    if (A.lse && half == 0) A.lse[((long long)b * A.heads + h) * M + row] = l == 0.f ? kInf : m + __builtin_amdgcn_logf(l);
  }
}

// ---- few queries ----------------------------------------------------------------------------------------------------------
//
// At most 32 rows (queries times heads that share a key/value head): every wavefront holds them all and takes every fourth tile
// of 32 keys of its share of the sequence; keys go from memory to registers as operands, values through the wavefront's own
// piece of LDS for the transposing read.  Shares of a long sequence go to different workgroups, which leave their sums for
// attention_join.  Bound by reading keys and values: 131072 keys of 2 heads, 128 components, 134 MB in 26 us (5.2 TB/s; a copy
// reaches 4.9), 32x8 ragged caches of up to 2048 keys, 64 components, 22 us with the join.
template <class Tin, class Tc, int DP>
__global__ void __launch_bounds__(256, (waves<Tc, DP>(32))) attention_rows(const Args A, int splits, float* part) {
  constexpr int ST = tile_stride<Tc, DP>(), NS = DP / 16, ND = DP / 32, VE = 16 / (int)sizeof(Tin), PER_ROW = DP / VE, NV = 32 * PER_ROW / 64;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
  lds_t<Tc>* const vt = (lds_t<Tc>*)smem + wave * 32 * ST;
  const int group = A.heads / A.kv_heads, M = (int)A.queries, rows = group * M;
  const int unit = blockIdx.x / splits, split = blockIdx.x % splits, b = unit / A.kv_heads, kvh = unit % A.kv_heads;
  const Span sp = span_of(A, b);
  const int h = kvh * group + col / M, qi = col % M;
  const bool there = col < rows;
  const int pos = sp.start + qi;
  int kend = sp.klen;
  if (A.causal) kend = min(kend, sp.start + M);
  if (kend < 0) kend = 0;
  const int share = ((kend + splits - 1) / splits + 127) / 128 * 128, k0 = min(split * share, kend), k1 = min(k0 + share, kend);
  const Tin* const K = rows_of<Tin>(A.k, A.k_stride, b, kvh);
  const Tin* const V = rows_of<Tin>(A.v, A.v_stride, b, kvh);
  typename Vec<Tc>::x8 qf[NS];
  {
    const Tin* q = rows_of<Tin>(A.q, A.q_stride, b, there ? h : 0) + (long long)qi * A.q_stride[2];
#pragma unroll
    for (int i = 0; i < NS; i++) qf[i] = frag_global<Tin, Tc>(q, there, 16 * i, half, A.dim);
  }
  const float* const bias = A.bias + (long long)(there ? h : 0) * A.buckets;
  const float left = bias_of(bias[A.bucket_of[0]]), right = bias_of(bias[A.bucket_of[2 * A.reach]]);
  const int lim = A.causal ? min(sp.klen, pos + 1) : sp.klen, pos_lo = sp.start, pos_hi = sp.start + M - 1;
  const float scale2 = A.scale * kLog2e;
  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; i++) acc[i] = zero16();
  float m = -kInf, l = 0.f;

  typename Vec<Tc>::x8 kf[NS];
  uint4 vr[NV];
  auto fetch = [&](int kb) {
    const int key = kb + col;
    const Tin* kp = K + (long long)key * A.k_stride[2];
#pragma unroll
    for (int i = 0; i < NS; i++) kf[i] = frag_global<Tin, Tc>(kp, key < k1, 16 * i, half, A.dim);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = lane + 64 * i, r = kb + c / PER_ROW, d = (c % PER_ROW) * VE;
      vr[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r < k1 && d < A.dim) vr[i] = *reinterpret_cast<const uint4*>(V + (long long)r * A.v_stride[2] + d);
    }
  };
  const int first = k0 + 32 * wave;
  if (first < k1) fetch(first);
  for (int kb = first; kb < k1; kb += 128) {
    f32x16 s = zero16();
#pragma unroll
    for (int i = 0; i < NS; i++) s = mma(kf[i], qf[i], s);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = lane + 64 * i;
      put_piece<Tin, Tc, DP>(vt, c / PER_ROW, (c % PER_ROW) * VE, vr[i]);
    }
    if (kb + 128 < k1) fetch(kb + 128);
    if (kb - pos_hi >= A.reach || kb + 31 - pos_lo <= -A.reach) {
      const float far = kb - pos_hi >= A.reach ? right : left;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = fmaf(s[r], scale2, far);
    } else {
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int rel = clampi(kb + c_row(r, half) - pos, -A.reach, A.reach);
        s[r] = fmaf(s[r], scale2, bias_of(bias[A.bucket_of[rel + A.reach]]));
      }
    }
    float mx = -kInf;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      s[r] = kb + c_row(r, half) < min(lim, k1) ? s[r] : -kInf;
      mx = fmaxf(mx, s[r]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
      for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][r] *= alpha;
      l *= alpha;
      m = mn;
    }
    const float ms = m == -kInf ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      s[r] = __builtin_amdgcn_exp2f(s[r] - ms);
      l += s[r];
    }
    // the wavefront's own stores to its piece of LDS come before its reads of it
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const typename Vec<Tc>::x8 p = pack<Tc>(s, k);
#pragma unroll
      for (int i = 0; i < ND; i++) acc[i] = mma(frag_cols<Tc, DP>(vt, 16 * k, 32 * i, lane), p, acc[i]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  l += __shfl_xor(l, 32);
  // the four wavefronts' sums, joined in their order
  __syncthreads();
  float* const o4 = (float*)smem;             // [4][rows][DP]
  float* const ml = o4 + 4 * rows * DP;       // [4][rows][2]
  if (there) {
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) o4[(wave * rows + col) * DP + 32 * i + c_row(r, half)] = acc[i][r];
    if (half == 0) {
      ml[(wave * rows + col) * 2] = m;
      ml[(wave * rows + col) * 2 + 1] = l;
    }
  }
  __syncthreads();
  for (int e = tid; e < rows * DP; e += 256) {
    const int r = e / DP, d = e % DP;
    float mm = -kInf, ll = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) mm = fmaxf(mm, ml[(w * rows + r) * 2]);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float mw = ml[(w * rows + r) * 2], a = mw == mm ? 1.f : __builtin_amdgcn_exp2f(mw - mm);
      ll += a * ml[(w * rows + r) * 2 + 1];
      o += a * o4[(w * rows + r) * DP + d];
    }
    const int hr = kvh * group + r / M, qr = r % M;
    if (splits == 1) {
      if (d < A.dim) put_out<Tin>(A, b, hr, qr, d, ll == 0.f ? 0.f : o / ll);
      if (A.lse && d == 0) A.lse[((long long)b * A.heads + hr) * M + qr] = ll == 0.f ? kInf : mm + __builtin_amdgcn_logf(ll);
    } else {
      float* p = part + ((long long)blockIdx.x * rows + r) * (DP + 2);
      p[2 + d] = o;
      if (d == 0) {
        p[0] = mm;
        p[1] = ll;
      }
    }
  }
}

// the shares of one row, joined in an order that is always the same: four groups of threads take every fourth share
template <class Tin> __global__ void __launch_bounds__(512) attention_join(const Args A, int splits, int dp, const float* part) {
  __shared__ float weight[256], sums[4][128], red[8];
  const int tid = threadIdx.x, lane = tid & 63, group = A.heads / A.kv_heads, M = (int)A.queries, rows = group * M;
  const int unit = blockIdx.x / rows, r = blockIdx.x % rows, b = unit / A.kv_heads, h = (unit % A.kv_heads) * group + r / M, qi = r % M;
  const long long step = (long long)rows * (dp + 2);
  const float* p = part + ((long long)unit * splits * rows + r) * (dp + 2);
  float m = -kInf, l = 0.f;
  if (tid < splits) {  // (at most 256)
    m = p[tid * step];
    l = p[tid * step + 1];
  }
  float mm = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
  if (lane == 0) red[tid >> 6] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float a = m == mm ? 1.f : __builtin_amdgcn_exp2f(m - mm);
  if (tid < 256) weight[tid] = a;
  float ll = tid < splits ? a * l : 0.f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ll += __shfl_xor(ll, o);
  __syncthreads();
  if (lane == 0) red[tid >> 6] = ll;
  __syncthreads();
  ll = (red[0] + red[1]) + (red[2] + red[3]);
  const int d = tid & 127, first = tid >> 7;
  float o = 0.f;
  if (d < A.dim) {
#pragma unroll 8
    for (int s = first; s < splits; s += 4) o = fmaf(weight[s], p[s * step + 2 + d], o);
  }
  sums[first][d] = o;
  __syncthreads();
  if (tid < A.dim) {
    o = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
    put_out<Tin>(A, b, h, qi, d, ll == 0.f ? 0.f : o / ll);
  }
  if (A.lse && tid == 0) A.lse[((long long)b * A.heads + h) * M + qi] = ll == 0.f ? kInf : mm + __builtin_amdgcn_logf(ll);
}

// The shares of rows, four components of one to a thread.  GRAD: gradients of queries (sums) and what delta is off by, otherwise
// outputs (sums with reference points).
template <class Tin, bool GRAD> __global__ void __launch_bounds__(256) attention_join_rows(const Args A, int splits, int dp, const float* part) {
  const int quads = A.dim / 4, group = A.heads / A.kv_heads;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x, r = e / quads;  // row: (unit, head of the group, query)
  if (r >= (long long)A.batch * A.heads * A.queries) return;
  const int c = 4 * (int)(e % quads), q = (int)(r % A.queries), g = (int)(r / A.queries % group), unit = (int)(r / A.queries / group);
  const int b = unit / A.kv_heads, h = unit % A.kv_heads * group + g;
  const float* p = part + share_of(A, unit, splits, 0, g, q) * (dp + 4);
  const long long step = (long long)group * A.queries * (dp + 4);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if constexpr (GRAD) {
    float over = 0.f;
    for (int s = 0; s < splits; s++) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + s * step + 4 + c);
      over += p[s * step];
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] += x[j];
    }
    if (c == 0) A.delta[((long long)b * A.heads + h) * A.queries + q] = p[1] + over;
    if (A.grad_q) store4<Tin>(rows_of<Tin>(A.grad_q, A.grad_q_stride, b, h) + (long long)q * A.grad_q_stride[2] + c, o[0], o[1], o[2], o[3]);
  } else {
    float mm = -kInf, l = 0.f;
    for (int s = 0; s < splits; s++) mm = fmaxf(mm, p[s * step]);
    for (int s = 0; s < splits; s++) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + s * step + 4 + c);
      const float m = p[s * step], a = m == mm ? 1.f : __builtin_amdgcn_exp2f(m - mm);
      l = fmaf(a, p[s * step + 1], l);
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = fmaf(a, x[j], o[j]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const long long at = (long long)q * A.out_stride[2] + c;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] *= inv;
    store4<Tin>(rows_of<Tin>(A.out, A.out_stride, b, h) + at, o[0], o[1], o[2], o[3]);
    if (A.out_rest) store4<Tin>(rows_of<Tin>(A.out_rest, A.out_stride, b, h) + at, left_of<Tin>(o[0]), left_of<Tin>(o[1]), left_of<Tin>(o[2]), left_of<Tin>(o[3]));
    if (A.lse && c == 0) A.lse[((long long)b * A.heads + h) * A.queries + q] = l == 0.f ? kInf : mm + __builtin_amdgcn_logf(l);
  }
}

// the same for gradients of keys and values
template <class Tin> __global__ void __launch_bounds__(256) attention_join_keys(const Args A, int splits, int dp, const float* part) {
  const int quads = A.dim / 4;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x, r = e / (2 * quads);  // key: (unit, key)
  if (r >= (long long)A.batch * A.kv_heads * A.keys) return;
  const int x = (int)(e % (2 * quads)), c = 4 * (x % quads), key = (int)(r % A.keys), unit = (int)(r / A.keys), b = unit / A.kv_heads, h = unit % A.kv_heads;
  const bool values = x >= quads;
  const float* p = part + ((long long)unit * splits * A.keys + key) * (2 * dp) + (values ? dp : 0) + c;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; s++) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(p + (long long)s * A.keys * (2 * dp));
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] += y[j];
  }
  Tin* to = values ? rows_of<Tin>(A.grad_v, A.grad_v_stride, b, h) + (long long)key * A.grad_v_stride[2]
                   : rows_of<Tin>(A.grad_k, A.grad_k_stride, b, h) + (long long)key * A.grad_k_stride[2];
  store4<Tin>(to + c, o[0], o[1], o[2], o[3]);
}

// ---- gradient of the queries ------------------------------------------------------------------------------------------------
//
// P = exp2(z - lse), dP = dO V^T, dS = P (dP - delta), dq = scale dS K, laid out as in the forward pass.  delta_i = sum_j P_ij dP_ij
// equals <dO_i, o_i>, but the output is rounded and came from rounded probabilities.  The forward pass of a training call leaves
// what the output's rounding took (out_rest): without it delta adds half as much to the error of dq as the rounding of dS does (rows
// with few keys; 2.6e-3 of dq for 2.3e-3, bf16).  The bias gradient sums rows whose exact sum is zero: a delta off by 2^-9 of itself would
// be most of a far bucket's gradient in a long row.  So dS is formed with <dO_i, o_i>, and the row sums of that dS, which are what
// delta is off by, are added to the delta that the gradient of keys, values and biases uses.
//
// 4x8 x 4096^2 causal bf16, 64 components: 150 us, 0.69 Pflop/s; of a SIMD's cycles matrix instructions take 30 %, vector ones 41 %.
template <class Tin, class Tc, int DP>
__global__ void __launch_bounds__(256, (waves<Tc, DP>(32))) attention_grad_q(const Args A, int splits, float* part) {
  constexpr int KT = key_tile<Tc, DP>(), SUB = KT / 32, ST = tile_stride<Tc, DP>(), NS = DP / 16, ND = DP / 32;
  typedef typename Vec<Tc>::x8 frag;
  extern __shared__ __align__(16) unsigned char smem[];
  lds_t<Tc>* const ktiles = (lds_t<Tc>*)smem;
  lds_t<Tc>* const vtiles = ktiles + 2 * KT * ST;
  float* const table = (float*)(vtiles + 2 * KT * ST);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int group = A.heads / A.kv_heads, M = (int)A.queries, nqb = (M + 127) / 128;
  int unit, block;
  block_of(blockIdx.x, A.batch * A.kv_heads, unit, block);
  const int split = block % splits;
  block /= splits;
  const int b = unit / A.kv_heads, kvh = unit % A.kv_heads, h = kvh * group + block % group, qb = nqb - 1 - block / group;
  const Span sp = span_of(A, b);
  fill_table(table, A, h, tid, 256);

  const int pos_lo = sp.start + qb * 128 + wave * 32, pos_hi = pos_lo + 31, row = qb * 128 + wave * 32 + col, pos = pos_lo + col;
  const Tin* const K = rows_of<Tin>(A.k, A.k_stride, b, kvh);
  const Tin* const V = rows_of<Tin>(A.v, A.v_stride, b, kvh);
  const long long ks = A.k_stride[2], vs = A.v_stride[2];
  frag qf[NS], gf[NS];
  float delta = 0.f;
  {
    const Tin* q = rows_of<Tin>(A.q, A.q_stride, b, h) + (long long)row * A.q_stride[2];
    const Tin* g = rows_of<Tin>(A.grad_out, A.grad_out_stride, b, h) + (long long)row * A.grad_out_stride[2];
    const Tin* o = rows_of<Tin>(A.out, A.out_stride, b, h) + (long long)row * A.out_stride[2];
    const Tin* left = rows_of<Tin>(A.out_rest, A.out_stride, b, h) + (long long)row * A.out_stride[2];
    const bool there = row < M, rest = there && A.out_rest;
#pragma unroll
    for (int i = 0; i < NS; i++) {
      qf[i] = frag_global<Tin, Tc>(q, there, 16 * i, half, A.dim);
      gf[i] = frag_global<Tin, Tc>(g, there, 16 * i, half, A.dim);
      float gx[8], ox[8];
      to_float(gf[i], gx);
      to_float(frag_global<Tin, Tc>(o, there, 16 * i, half, A.dim), ox);
      if constexpr (sizeof(Tin) == 2) {
        float rx[8];
        to_float(frag_global<Tin, Tc>(left, rest, 16 * i, half, A.dim), rx);
#pragma unroll
        for (int j = 0; j < 8; j++) ox[j] += rx[j];
      }
#pragma unroll
      for (int j = 0; j < 8; j++) delta = fmaf(gx[j], ox[j], delta);
    }
    delta += __shfl_xor(delta, 32);
  }
  const long long stat = ((long long)b * A.heads + h) * M + row;
  const float lse = row < M ? A.lse[stat] : kInf;
  const int kend = A.causal ? min(sp.klen, sp.start + min(qb * 128 + 128, M)) : sp.klen;
  const int wend = A.causal ? min(kend, pos_hi + 1) : kend;
  const int alltiles = kend > 0 ? (kend + KT - 1) / KT : 0, first = alltiles * split / splits, ntiles = alltiles * (split + 1) / splits;
  const int nsub = wend > 0 ? (wend + 31) / 32 : 0;
  const int lim = A.causal ? min(sp.klen, pos + 1) : sp.klen;
  const float scale2 = A.scale * kLog2e;

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; i++) acc[i] = zero16();
  float over = 0.f;
  Scaled<Tc> ds_scale;

  Staged<Tin, Tc, KT, DP> sk, sv;
  const auto fetch = [&](int t) __attribute__((always_inline)) {
    sk.load(K + (long long)t * KT * ks, ks, sp.klen - t * KT, A.dim, tid);
    sv.load(V + (long long)t * KT * vs, vs, sp.klen - t * KT, A.dim, tid);
  };
  const auto put = [&](int t) __attribute__((always_inline)) {
    sk.store(ktiles + (t & 1) * KT * ST, tid);
    sv.store(vtiles + (t & 1) * KT * ST, tid);
  };
  if (first < ntiles) {
    fetch(first);
    put(first);
    if (first + 1 < ntiles) fetch(first + 1);
  }
  __syncthreads();
  const float left = table[0], right = table[2 * A.reach + 2 * kPad];
  for (int t = first; t < ntiles; t++) {
    if constexpr (Vec<Tc>::terms > 1 || DP == 128) forget(lane, half, col);
    const lds_t<Tc>* kt = ktiles + (t & 1) * KT * ST;
    const lds_t<Tc>* vt = vtiles + (t & 1) * KT * ST;
    if (t + 1 < ntiles) {
      put(t + 1);
      if (t + 2 < ntiles) fetch(t + 2);
    }
#pragma unroll
    for (int u = 0; u < SUB; u++) {
      const int kb = t * KT + 32 * u;
      if (SUB * t + u >= nsub) continue;
      f32x16 s = zero16(), p;
#pragma unroll
      for (int r = 0; r < 16; r++) p[r] = -delta;
#pragma unroll
      for (int i = 0; i < NS; i++) {
        s = mma(frag_rows<Tc, DP>(kt, 32 * u + col, 16 * i, half), qf[i], s);
        p = mma(frag_rows<Tc, DP>(vt, 32 * u + col, 16 * i, half), gf[i], p);
      }
      const int kind = kb - pos_hi >= A.reach ? 1 : (kb + 31 - pos_lo <= -A.reach ? -1 : 0);
      logits_by_key(s, scale2, table, lse, kind > 0 ? right : left, kind, kb + 32 > sp.klen || (A.causal && kb + 31 > pos_lo), lim, kb, pos, half, A.reach);
#pragma unroll
      for (int r = 0; r < 16; r++) {
        s[r] = __builtin_amdgcn_exp2f(s[r]) * p[r];
        over += s[r];
      }
      ds_scale.fit(s, acc);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const frag ds = pack<Tc>(s, k);
#pragma unroll
        for (int i = 0; i < ND; i++) acc[i] = mma(frag_cols<Tc, DP>(kt, 32 * u + 16 * k, 32 * i, lane), ds, acc[i]);
      }
    }
    __syncthreads();
  }
  over += __shfl_xor(over, 32);
  if (splits > 1) {
    if (row < M) {
      const float back = A.scale * ds_scale.inverse();
      float* p = part + share_of(A, unit, splits, split, h, row) * (DP + 4);
      if (half == 0) {
        p[0] = over;
        p[1] = delta;
      }
#pragma unroll
      for (int i = 0; i < ND; i++)
#pragma unroll
        for (int g = 0; g < 4; g++)
          store4<float>(p + 4 + 32 * i + 8 * g + 4 * half, acc[i][4 * g] * back, acc[i][4 * g + 1] * back, acc[i][4 * g + 2] * back, acc[i][4 * g + 3] * back);
    }
    return;
  }
  if (row < M) {
    if (half == 0) A.delta[stat] = delta + over;
    if (A.grad_q) {
      const float back = A.scale * ds_scale.inverse();
      Tin* o = rows_of<Tin>(A.grad_q, A.grad_q_stride, b, h) + (long long)row * A.grad_q_stride[2];
#pragma unroll
      for (int i = 0; i < ND; i++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const int d = 32 * i + 8 * g + 4 * half;
          if (d < A.dim)
            store4<Tin>(o + d, acc[i][4 * g] * back, acc[i][4 * g + 1] * back, acc[i][4 * g + 2] * back, acc[i][4 * g + 3] * back);
        }
    }
  }
}

// ---- gradients of keys, values and biases -----------------------------------------------------------------------------------
//
// A workgroup has 128 keys of one key/value head, a wavefront 32 of them as columns, and walks over the queries of all heads that
// share them (or over a share of them, joined in order), so no order of additions is left to chance.  Biases: pairs beyond the reach
// add to one sum a side; a 32 x 32 tile within it is summed along its 63 diagonals (each distance is one: lanes are rotated by the
// register's row, so that equal distances meet in a lane) into a table by distance that belongs to the wavefront, and the tables
// become sums by bucket when the head is done.
//
// 4x8 x 4096^2 causal bf16, 64 components: 222 us, 0.62 Pflop/s; of a SIMD's cycles matrix instructions take 27 %, vector ones 39 %;
// the sums and operands of 32 keys take 247 registers, which allows two wavefronts a SIMD.
template <class Tin, class Tc, int DP>
__global__ void __launch_bounds__(256, (Vec<Tc>::terms == 1 && DP <= 64 ? 2 : 1)) attention_grad_kv(const Args A, float* part, int splits, float* share) {
  constexpr int QT = query_tile<Tc>(), ST = tile_stride<Tc, DP>(), NS = DP / 16, ND = DP / 32, SUB = QT / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  lds_t<Tc>* const tiles = (lds_t<Tc>*)smem;            // [2][queries, output gradients][QT][ST]
  float* const stats = (float*)(tiles + 4 * QT * ST);   // [2][lse, delta][QT]
  const int tlen = 2 * A.reach + 1 + 2 * kPad;
  float* const table = stats + 4 * QT;
  float* const sums = table + tlen;                     // [4][tlen]
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int group = A.heads / A.kv_heads, M = (int)A.queries, N = (int)A.keys, nkb = (N + 127) / 128;
  int unit, kblock;
  block_of(blockIdx.x, A.batch * A.kv_heads, unit, kblock);
  const int split = kblock % splits;
  kblock /= splits;
  const int b = unit / A.kv_heads, kvh = unit % A.kv_heads;
  const Span sp = span_of(A, b);
  const int kb = kblock * 128 + wave * 32, key = kb + col;
  const bool want_bias = part != nullptr;
  typename Vec<Tc>::x8 kf[NS], vf[NS];
  {
    const Tin* k = rows_of<Tin>(A.k, A.k_stride, b, kvh) + (long long)key * A.k_stride[2];
    const Tin* v = rows_of<Tin>(A.v, A.v_stride, b, kvh) + (long long)key * A.v_stride[2];
#pragma unroll
    for (int i = 0; i < NS; i++) {
      kf[i] = frag_global<Tin, Tc>(k, key < sp.klen, 16 * i, half, A.dim);
      vf[i] = frag_global<Tin, Tc>(v, key < sp.klen, 16 * i, half, A.dim);
    }
  }
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int i = 0; i < ND; i++) {
    dk[i] = zero16();
    dv[i] = zero16();
  }
  // float16 probabilities are held times 2^15 (1 is 32768; 2^-29 is still a normal number), and the score gradients with them
  constexpr float up = is_f16<Tc> ? 15.f : 0.f, down = is_f16<Tc> ? 1.f / 32768.f : 1.f;
  Scaled<Tc> ds_scale;
  const float scale2 = A.scale * kLog2e;
  // first query tile that can see a key of this workgroup
  int q_first = 0;
  if (A.causal) q_first = max(0, kblock * 128 - sp.start) / QT * QT;
  const int q_end = kblock * 128 < sp.klen ? M : 0;
  const int alltiles = q_end > q_first ? (q_end - q_first + QT - 1) / QT : 0;
  q_first += alltiles * split / splits * QT;  // this workgroup's share of them
  const int ntiles = alltiles * (split + 1) / splits - alltiles * split / splits;

  for (int g = 0; g < group; g++) {
    const int h = kvh * group + g;
    const Tin* const Q = rows_of<Tin>(A.q, A.q_stride, b, h);
    const Tin* const G = rows_of<Tin>(A.grad_out, A.grad_out_stride, b, h);
    const float* const lse = A.lse + ((long long)b * A.heads + h) * M;
    const float* const del = A.delta + ((long long)b * A.heads + h) * M;
    float far_left = 0.f, far_right = 0.f;
    Staged<Tin, Tc, QT, DP> sq, sg;
    float s_lse = -kInf, s_del = 0.f;
    auto fetch = [&](int q0) {
      sq.load(Q + (long long)q0 * A.q_stride[2], A.q_stride[2], M - q0, A.dim, tid);
      sg.load(G + (long long)q0 * A.grad_out_stride[2], A.grad_out_stride[2], M - q0, A.dim, tid);
      if (tid < QT) {  // the negatives, as they are added
        s_lse = q0 + tid < M ? up - lse[q0 + tid] : -kInf;
        s_del = q0 + tid < M ? -del[q0 + tid] : 0.f;
      }
    };
    auto put = [&](int buf) {
      sq.store(tiles + buf * 2 * QT * ST, tid);
      sg.store(tiles + buf * 2 * QT * ST + QT * ST, tid);
      if (tid < QT) {
        stats[buf * 2 * QT + tid] = s_lse;
        stats[buf * 2 * QT + QT + tid] = s_del;
      }
    };
    fill_table(table, A, h, tid, 256);
    if (want_bias)
      for (int i = tid; i < 4 * tlen; i += 256) sums[i] = 0.f;
    if (ntiles > 0) {
      fetch(q_first);
      put(0);
      if (ntiles > 1) fetch(q_first + QT);
    }
    __syncthreads();
    const float left = table[0], right = table[tlen - 1];
    for (int t = 0; t < ntiles; t++) {
      if constexpr (Vec<Tc>::terms > 1) forget(lane, half, col);
      const lds_t<Tc>* qt = tiles + (t & 1) * 2 * QT * ST;
      const lds_t<Tc>* gt = qt + QT * ST;
      const float* st = stats + (t & 1) * 2 * QT;
      if (t + 1 < ntiles) {
        put((t + 1) & 1);
        if (t + 2 < ntiles) fetch(q_first + (t + 2) * QT);
      }
#pragma unroll
      for (int u = 0; u < SUB; u++) {
        const int q0 = q_first + t * QT + 32 * u, pos0 = sp.start + q0;  // position of the tile's first query
        if (kb >= sp.klen || (A.causal && kb > pos0 + 31)) continue;     // nothing in this wavefront's tile
        f32x16 s = zero16(), p, e;
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
          const f32x4 de = *reinterpret_cast<const f32x4*>(st + QT + 32 * u + 8 * g4 + 4 * half);
#pragma unroll
          for (int t4 = 0; t4 < 4; t4++) p[4 * g4 + t4] = de[t4];
        }
#pragma unroll
        for (int i = 0; i < NS; i++) {
          s = mma(frag_rows<Tc, DP>(qt, 32 * u + col, 16 * i, half), kf[i], s);
          p = mma(frag_rows<Tc, DP>(gt, 32 * u + col, 16 * i, half), vf[i], p);
        }
        const int kind = kb - (pos0 + 31) >= A.reach ? 1 : (kb + 31 - pos0 <= -A.reach ? -1 : 0);
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(st + 32 * u + 8 * g4 + 4 * half);
#pragma unroll
          for (int t4 = 0; t4 < 4; t4++) e[4 * g4 + t4] = fmaf(s[4 * g4 + t4], scale2, ls[t4]);
        }
        if (kind == 0) {
          const float* tp = table + (key - pos0 - 4 * half + A.reach + kPad);
#pragma unroll
          for (int r = 0; r < 16; r++) e[r] += tp[-(8 * (r / 4) + r % 4)];
        } else {
          const float far = kind > 0 ? right : left;
#pragma unroll
          for (int r = 0; r < 16; r++) e[r] += far;
        }
        if (kb + 31 >= sp.klen || (A.causal && kb + 31 > pos0)) {
          const int first = key >= sp.klen ? 32 : (A.causal ? key - pos0 - 4 * half : -64);  // first row of the tile that sees the key
#pragma unroll
          for (int r = 0; r < 16; r++) e[r] = 8 * (r / 4) + r % 4 >= first ? e[r] : -kInf;
        }
#pragma unroll
        for (int r = 0; r < 16; r++) {
          e[r] = __builtin_amdgcn_exp2f(e[r]);
          s[r] = e[r] * p[r];
        }
        if (want_bias) {
          if (kind != 0) {
            float x = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r++) x += s[r];
            if (kind > 0) far_right += x; else far_left += x;
          } else {
            // distance of (query row r, key col) is col - row + (kb - pos0): lane c of a half takes the value of key (c + row) % 32
            float up = 0.f, down = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r++) {
              const int from = col + c_row(r, half);
              const float x = __shfl(s[r], (from & 31) | (half << 5));
              if (from < 32) up += x; else down += x;  // distance c, or c - 32
            }
            const float other = __shfl_xor(half ? up : down, 32);
            const float mine = (half ? down : up) + other;
            float* d = sums + wave * tlen + (kb - pos0 + A.reach + kPad + col - 32 * half);
            *d += mine;
          }
        }
        ds_scale.fit(s, dk);
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const typename Vec<Tc>::x8 pf = pack<Tc>(e, k), df = pack<Tc>(s, k);
#pragma unroll
          for (int i = 0; i < ND; i++) {
            dv[i] = mma(frag_cols<Tc, DP>(gt, 32 * u + 16 * k, 32 * i, lane), pf, dv[i]);
            dk[i] = mma(frag_cols<Tc, DP>(qt, 32 * u + 16 * k, 32 * i, lane), df, dk[i]);
          }
        }
      }
      __syncthreads();
    }
    if (want_bias) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        far_left += __shfl_xor(far_left, o);
        far_right += __shfl_xor(far_right, o);
      }
      __syncthreads();
      if (lane == 0) {
        sums[wave * tlen] += far_left;
        sums[wave * tlen + tlen - 1] += far_right;
      }
      __syncthreads();
      for (int i = tid; i < tlen; i += 256) table[i] = ((sums[i] + sums[tlen + i]) + (sums[2 * tlen + i] + sums[3 * tlen + i])) * down;
      __syncthreads();
      if (wave < 2) {  // what lies in the padding belongs to the ends of the reach
        const int at = wave == 0 ? 0 : tlen - kPad;
        float x = table[at + lane] + (lane < kPad - 64 ? table[at + 64 + lane] : 0.f);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
        if (lane == 0) sums[wave] = x;
      }
      __syncthreads();
      if (tid == 0) {
        table[kPad] += sums[0];
        table[tlen - 1 - kPad] += sums[1];
      }
      __syncthreads();
      float* out = part + ((long long)((b * nkb + kblock) * splits + split) * A.heads + h) * A.buckets;
      for (int bu = wave; bu < A.buckets; bu += 4) {
        float x = 0.f;
        for (int e = A.bucket_begin[bu] + lane; e < A.bucket_begin[bu + 1]; e += 64) x += table[A.bucket_order[e] + kPad];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
        if (lane == 0) out[bu] = x;
      }
    }
    __syncthreads();
  }
  if (splits > 1) {
    if (key < N) {
      const float back = A.scale * down * ds_scale.inverse();
      float* p = share + ((long long)(unit * splits + split) * N + key) * (2 * DP);
#pragma unroll
      for (int i = 0; i < ND; i++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const int d = 32 * i + 8 * g + 4 * half;
          store4<float>(p + d, dk[i][4 * g] * back, dk[i][4 * g + 1] * back, dk[i][4 * g + 2] * back, dk[i][4 * g + 3] * back);
          store4<float>(p + DP + d, dv[i][4 * g] * down, dv[i][4 * g + 1] * down, dv[i][4 * g + 2] * down, dv[i][4 * g + 3] * down);
        }
    }
    return;
  }
  if (key < N) {
    const float back = A.scale * down * ds_scale.inverse();
    Tin* ok = rows_of<Tin>(A.grad_k, A.grad_k_stride, b, kvh) + (long long)key * A.grad_k_stride[2];
    Tin* ov = rows_of<Tin>(A.grad_v, A.grad_v_stride, b, kvh) + (long long)key * A.grad_v_stride[2];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int d = 32 * i + 8 * g + 4 * half;
        if (d < A.dim) {
          store4<Tin>(ok + d, dk[i][4 * g] * back, dk[i][4 * g + 1] * back, dk[i][4 * g + 2] * back, dk[i][4 * g + 3] * back);
          store4<Tin>(ov + d, dv[i][4 * g] * down, dv[i][4 * g + 1] * down, dv[i][4 * g + 2] * down, dv[i][4 * g + 3] * down);
        }
      }
  }
}

// gradient of one bias: the workgroups' sums in their order
__global__ void __launch_bounds__(256) attention_grad_bias(const float* part, float* out, int parts, int total) {
  __shared__ double red[256];
  double x = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) x += (double)part[(long long)i * total + blockIdx.x];
  red[threadIdx.x] = x;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[blockIdx.x] = (float)red[0];
}

// ---- host -------------------------------------------------------------------------------------------------------------------

int padded_dim(int dim) { return dim <= 32 ? 32 : (dim <= 64 ? 64 : (dim <= 96 ? 96 : 128)); }

bool aligned(const Args* a) {
  const size_t size = a->dtype == 2 ? 4 : 2;
  return rows_aligned(a->q, a->q_stride, size) && rows_aligned(a->k, a->k_stride, size) && rows_aligned(a->v, a->v_stride, size) &&
         rows_aligned(a->out, a->out_stride, size) && rows_aligned(a->out_rest, a->out_stride, size) && rows_aligned(a->grad_out, a->grad_out_stride, size) &&
         rows_aligned(a->grad_q, a->grad_q_stride, size) && rows_aligned(a->grad_k, a->grad_k_stride, size) && rows_aligned(a->grad_v, a->grad_v_stride, size);
}

const char* check(const Args* a) {
  if (!a) return "bucket attention: null arguments";
  if (a->dtype < 0 || a->dtype > 2) return "bucket attention: dtype must be 0 (bfloat16), 1 (float16) or 2 (float32)";
  const int ve = a->dtype == 2 ? 4 : 8;
  if (a->batch < 1 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads) return "bucket attention: heads must be a multiple of kv_heads";
  if (a->dim < ve || a->dim > 128 || a->dim % ve) return "bucket attention: dim must be a multiple of 16 bytes, at most 128";
  if (a->queries < 1 || a->queries > (1 << 29) || a->keys < 0 || a->keys > (1 << 29)) return "bucket attention: queries or keys out of range";
  if (a->reach < 1 || a->reach > KEOPS_HIP_MAX_REACH || a->buckets < 1 || a->buckets > 2 * a->reach + 1) return "bucket attention: reach or number of buckets out of range";
  if (a->start < -(1 << 29) || a->start > (1 << 29)) return "bucket attention: query_start out of range";
  for (const int64_t* x : {a->q_stride, a->k_stride, a->v_stride, a->grad_out_stride})
    if (x[2] < 0 || x[2] > kMaxRowStride) return "bucket attention: rows too far apart";
  if (!aligned(a)) return "bucket attention: a row does not start at a multiple of 16 bytes";
  if (!a->q || !a->out || !a->bias || !a->bucket_of || (a->keys > 0 && (!a->k || !a->v))) return "bucket attention: null data";
  const int64_t units = (int64_t)a->batch * a->heads;
  if (units * ((a->queries + 127) / 128) > 0x7fffffff || units * ((a->keys + 127) / 128) > 0x7fffffff) return "bucket attention: too many workgroups";
  return nullptr;
}

// The form for few rows against the one for tiles of 128 queries, us: 32x8 caches of up to 2048 keys 25 and 37, 131072 keys for 16
// rows 37 and 344, 4 queries of 32 heads that share 4, 8192 keys, 18 and 53.
bool few_rows(const Args* a) { return a->queries * (a->heads / a->kv_heads) <= 32; }

// Shares of the keys for few rows: two workgroups on every CU, at least 256 keys to a share (two tiles a wavefront).  32x8 caches of
// up to 2048 keys with 256, 512, 1024 and 2048 workgroups: 24.5, 22.4, 24.9 and 31.6 us.  32 rows of 4 sequences, 8192 keys, 64
// components, with at least 128, 256 and 512 keys: 24.0, 18.3, 17.1 us; of one sequence, 128 components: 18.1, 19.0, 22.5.
int splits_of(const Args* a) {
  const int64_t units = (int64_t)a->batch * a->kv_heads;
  int64_t s = 512 / units, most = a->keys / 256;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
}

template <class Tc, int DP> constexpr size_t tile_bytes(int rows) { return 4 * (size_t)rows * tile_stride<Tc, DP>() * 2; }  // two tensors, two buffers
int table_entries(const Args* a) { return 2 * a->reach + 1 + 2 * kPad; }

template <class K> int prepare_lds(K kernel, size_t bytes) {
  if (bytes <= 64 * 1024) return 0;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  return e == hipSuccess ? 0 : keops_seq_fail((int)e, "bucket attention: shared memory");
}

// Workgroups of one block, for `blocks` blocks that walk over `rows` rows: two workgroups on every CU, but shares of at least 256
// rows (128 of float32, whose steps take three times as long), or the join costs more than it gives.  Training of 2x8(2)x2048^2, 64
// components, for 256, 512 and 1024 workgroups: 216, 183, 197 us; 2x8x4096^2, 128 components: 568, 568, 595.  At least 128, 256 and
// 512 rows: a forward pass of 8x300x2000 25, 19, 21 us; at least 64, 128 and 256 of float32, training of 3x6x517x777: 158, 147, 181.
int shares_of(int64_t blocks, int64_t rows, int dtype) {
  int64_t s = blocks < 1 ? 1 : 512 / blocks, most = rows / (dtype == 2 ? 128 : 256);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 16 ? 16 : s));
}
struct Shares {  // of a call's three walks, and where the backward pass's sums lie in its workspace (bytes)
  int forward, q, k;
  size_t forward_bytes, q_at, k_at, backward_bytes;
  explicit Shares(const Args* a) {
    const int64_t qblocks = (int64_t)a->batch * a->heads * ((a->queries + 127) / 128), nkb = (a->keys + 127) / 128, kblocks = (int64_t)a->batch * a->kv_heads * nkb;
    const size_t dp = padded_dim(a->dim), rows = (size_t)a->batch * a->heads * a->queries, keys = (size_t)a->batch * a->kv_heads * a->keys;
    forward = q = shares_of(qblocks, a->keys, a->dtype);
    k = shares_of(kblocks, a->queries, a->dtype);
    forward_bytes = forward > 1 ? (size_t)forward * rows * (dp + 4) * sizeof(float) : 0;
    const size_t bias = a->grad_bias ? (size_t)a->batch * nkb * k * a->heads * a->buckets * sizeof(float) : 0;
    q_at = (bias + 15) / 16 * 16;
    k_at = q_at + (q > 1 ? (size_t)q * rows * (dp + 4) * sizeof(float) : 0);
    backward_bytes = k_at + (k > 1 ? (size_t)k * keys * 2 * dp * sizeof(float) : 0);
  }
};

template <class Tin, class Tc, int DP> struct Passes {
  static int forward(const Args& a, float* work, hipStream_t st) {
    const int group = a.heads / a.kv_heads;
    if (few_rows(&a)) {
      const int rows = group * (int)a.queries, splits = splits_of(&a);
      const size_t v = 4 * 32 * (size_t)tile_stride<Tc, DP>() * 2, o = 4 * (size_t)rows * (DP + 2) * 4, lds = v > o ? v : o;
      if (int e = prepare_lds(attention_rows<Tin, Tc, DP>, lds)) return e;
      attention_rows<Tin, Tc, DP><<<a.batch * a.kv_heads * splits, 256, lds, st>>>(a, splits, work);
      if (splits > 1) attention_join<Tin><<<a.batch * a.kv_heads * rows, 512, 0, st>>>(a, splits, DP, work);
    } else {
      const Shares shares(&a);
      const size_t lds = tile_bytes<Tc, DP>(key_tile<Tc, DP>()) + 4 * (size_t)table_entries(&a);
      if (int e = prepare_lds(attention_forward<Tin, Tc, DP>, lds)) return e;
      const int nqb = (int)((a.queries + 127) / 128);
      attention_forward<Tin, Tc, DP><<<a.batch * a.heads * nqb * shares.forward, 256, lds, st>>>(a, shares.forward, work);
      if (shares.forward > 1) attention_join_rows<Tin, false><<<join_blocks((int64_t)a.batch * a.heads * a.queries * (a.dim / 4)), 256, 0, st>>>(a, shares.forward, DP, work);
    }
    return seq_launched("bucket attention: launch");
  }
  static unsigned join_blocks(int64_t threads) { return (unsigned)((threads + 255) / 256); }
  static int backward(const Args& a, float* work, hipStream_t st) {
    const Shares shares(&a);
    float* const qpart = (float*)((char*)work + shares.q_at), * const kpart = (float*)((char*)work + shares.k_at);
    const int nqb = (int)((a.queries + 127) / 128), nkb = (int)((a.keys + 127) / 128);
    const size_t tb = tile_bytes<Tc, DP>(key_tile<Tc, DP>()), te = 4 * (size_t)table_entries(&a);
    if (int e = prepare_lds(attention_grad_q<Tin, Tc, DP>, tb + te)) return e;
    attention_grad_q<Tin, Tc, DP><<<a.batch * a.heads * nqb * shares.q, 256, tb + te, st>>>(a, shares.q, qpart);
    if (shares.q > 1) attention_join_rows<Tin, true><<<join_blocks((int64_t)a.batch * a.heads * a.queries * (a.dim / 4)), 256, 0, st>>>(a, shares.q, DP, qpart);
    if (nkb > 0) {
      float* part = a.grad_bias ? work : nullptr;
      const size_t lds = tile_bytes<Tc, DP>(query_tile<Tc>()) + 4 * query_tile<Tc>() * sizeof(float) + 5 * te;
      if (int e = prepare_lds(attention_grad_kv<Tin, Tc, DP>, lds)) return e;
      attention_grad_kv<Tin, Tc, DP><<<a.batch * a.kv_heads * nkb * shares.k, 256, lds, st>>>(a, part, shares.k, kpart);
      if (shares.k > 1) attention_join_keys<Tin><<<join_blocks((int64_t)a.batch * a.kv_heads * a.keys * (a.dim / 2)), 256, 0, st>>>(a, shares.k, DP, kpart);
    }
    if (a.grad_bias) attention_grad_bias<<<a.heads * a.buckets, 256, 0, st>>>(work, a.grad_bias, a.batch * nkb * shares.k, a.heads * a.buckets);
    return seq_launched("bucket attention: launch of the backward pass");
  }
};

template <class Tin, class Tc> int dispatch(const Args& a, bool backward, float* work, hipStream_t st) {
  switch (padded_dim(a.dim)) {
    case 32: return backward ? Passes<Tin, Tc, 32>::backward(a, work, st) : Passes<Tin, Tc, 32>::forward(a, work, st);
    case 64: return backward ? Passes<Tin, Tc, 64>::backward(a, work, st) : Passes<Tin, Tc, 64>::forward(a, work, st);
    case 96: return backward ? Passes<Tin, Tc, 96>::backward(a, work, st) : Passes<Tin, Tc, 96>::forward(a, work, st);
    default: return backward ? Passes<Tin, Tc, 128>::backward(a, work, st) : Passes<Tin, Tc, 128>::forward(a, work, st);
  }
}

int enter(const Args* a, bool backward, void* work, size_t work_bytes, int device, void* stream) {
  if (const char* why = check(a)) return keops_seq_fail(-1, why);
  if (backward && (!a->grad_out || !a->lse || !a->delta || (a->keys > 0 && (!a->grad_k || !a->grad_v)) || (a->grad_bias && (!a->bucket_order || !a->bucket_begin))))
    return keops_seq_fail(-1, "bucket attention: null data for the backward pass");
  const size_t need = backward ? keops_hip_bucket_attention_backward_bytes(a) : keops_hip_bucket_attention_forward_bytes(a);
  if (need > work_bytes || (need > 0 && !work)) return keops_seq_fail(-1, "bucket attention: workspace too small");
  SeqDevice on(device);
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == 0) return dispatch<bf16, bf16>(*a, backward, (float*)work, st);
  if (a->dtype == 1) return dispatch<f16, f16>(*a, backward, (float*)work, st);
  return dispatch<float, Split<3>>(*a, backward, (float*)work, st);
}

}  // namespace

extern "C" {

size_t keops_hip_bucket_attention_forward_bytes(const keops_hip_bucket_attention* a) {
  if (check(a)) return 0;
  if (!few_rows(a)) return Shares(a).forward_bytes;
  if (splits_of(a) == 1) return 0;
  const size_t rows = (size_t)(a->heads / a->kv_heads) * a->queries;
  return (size_t)a->batch * a->kv_heads * splits_of(a) * rows * (padded_dim(a->dim) + 2) * sizeof(float);
}

size_t keops_hip_bucket_attention_backward_bytes(const keops_hip_bucket_attention* a) {
  return check(a) ? 0 : Shares(a).backward_bytes;
}

int keops_hip_bucket_attention_forward(const keops_hip_bucket_attention* a, void* work, size_t work_bytes, int device, void* hip_stream) {
  return enter(a, false, work, work_bytes, device, hip_stream);
}

int keops_hip_bucket_attention_backward(const keops_hip_bucket_attention* a, void* work, size_t work_bytes, int device, void* hip_stream) {
  return enter(a, true, work, work_bytes, device, hip_stream);
}

}  // extern "C"
