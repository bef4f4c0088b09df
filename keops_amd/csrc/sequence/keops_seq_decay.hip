// Linear attention with a decay for each head:  S_t = g S_{t-1} + k_t v_t^T,  o_t = scale q_t S_t,  and its gradients, which are
// the same sum with the roles of the inputs exchanged (d = gradient of o):
//   dq = A(d, v, k; S_0^T),   dk = A^rev(v, d, q; dS_T^T),   dv = A^rev(k, q, d; dS_T),   dS_0 = final state of the last one,
// where A^rev walks from the last token to the first.  One kernel serves all of them.
//
// Chunks of 64 tokens: within a chunk the masked product (q k^T) o g^(i-j) times v, across chunks the state, so a token costs
// 4 dim dim_v flop and 64 (dim + dim_v) more.  The state stays in the registers of the wavefronts, each of which has 32 of its
// columns, as a C tile (keops_seq.h) that serves as an operand as it is.
//
// What bounds it is traffic: q, k, v and the outputs once, k and v a second time for the segments' states, and these.  16 x 16384
// tokens, 128 components, bf16: 132 us for 540 MB; training of 4x8x4096, 64 components: 140 us for 500 MB in 8 launches.
#include "../../../include/keops_hip.h"
#include "keops_seq.h"

using namespace kseq;

namespace {

typedef keops_hip_decay_attention Args;

constexpr int kChunk = 64;  // tokens of a chunk
// With 32 tokens also for two terms: float16 training of 4x8x4096, 64 components, 164 us (64 tokens: 216), a prompt of 16 x 16384
// tokens, 128 components, 190 (220): more workgroups fit in LDS.
template <class Tc> constexpr int chunk() { return Vec<Tc>::terms > 1 ? 32 : kChunk; }

// Decayed values as an operand for the state: all of a float32 where the state is a result (or becomes one over the segments
// behind), 16 bits where it only serves outputs that are rounded to 8.  The state itself is float32; as an operand for those
// outputs it is rounded once, as the products within the chunk are.
template <class Tc, bool RESULT> constexpr int update_terms() { return RESULT || Vec<Tc>::terms == 3 ? 3 : 2; }

// powers of the decay in LDS: entry kZero + n holds g^n for n = 0..kChunk, zeros before and behind
constexpr int kZero = 64, kPowers = kZero + kChunk + 8;
__device__ inline float power(float log_decay, long long n) { return n == 0 ? 1.f : (float)exp((double)log_decay * (double)n); }
__device__ inline void fill_powers(float* pw, float log_decay, int tid, int nt) {
  for (int i = tid; i < kPowers; i += nt) pw[i] = i < kZero || i > kZero + kChunk ? 0.f : power(log_decay, i - kZero);
}

template <class T> __device__ inline const T* rows_of(const void* p, const int64_t* s, int b, int h) { return (const T*)p + (long long)b * s[0] + (long long)h * s[1]; }

__device__ inline int length_of(const Args& A, int b) {
  const int t = (int)A.tokens;
  if (!A.lengths) return t;
  const int n = A.lengths[b];
  return n < 0 ? 0 : (n > t ? t : n);
}

// S = g^n S + sum_j weight_j k_j v_j^T of the chunk in LDS (n tokens); wavefront's 32 columns of v
template <class Tc, int DK, int DV, int NT>
__device__ inline void update_state(f32x16 (&S)[DK / 32], const lds_t<Tc>* kt, const lds_t<Tc>* vt, const float* pw, int n, int shift, float scale, int wave,
                                    int lane) {
  const int half = lane >> 5;
  const float all = pw[kZero + n];
#pragma unroll
  for (int i = 0; i < DK / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) S[i][r] *= all;
  const float* w = pw + kZero + n - 1 + shift - 4 * half;  // weight of token j is w[-j], zero behind the chunk's end
#pragma unroll
  for (int s = 0; s < chunk<Tc>() / 16; s++) {
    float x[8];
    to_float(frag_cols<Tc, DV>(vt, 16 * s, 32 * wave, lane), x);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] *= w[-(16 * s + (j & 3) + 2 * (j & 4))] * scale;
    const SplitX8<NT> v = to_split<NT>(x);
#pragma unroll
    for (int i = 0; i < DK / 32; i++) S[i] = mma(frag_cols<Tc, DK>(kt, 16 * s, 32 * i, lane), v, S[i]);
  }
}

// ---- states at the ends of segments -------------------------------------------------------------------------------------------
//
// Few sequences and heads do not fill the chip, so a long sequence is cut into segments: their own states first (this kernel),
// then decay_scan carries them on, then decay_outputs starts every segment from its state.
// A wavefront has 32 columns and half of the rows of a state.  The decayed values, which every row needs, are formed once, on their
// way to LDS, as three bf16 terms each (all 24 bits: these states are results).  16 x 16384 tokens, 128 components: 45 us, 3.7 TB/s
// (58 us with all rows and their own decayed values in each wavefront).
template <class Tin, class Tc, int DK, int DV, bool REV>
__global__ void __launch_bounds__(4 * DV, 2) decay_states(const Args A, int segments, int seg_tokens, float* states) {
  constexpr int C = chunk<Tc>(), NT = 4 * DV, SK = tile_stride<Tc, DK>(), SV = tile_stride<Split<3>, DV>(), I = DK / 64;
  extern __shared__ __align__(16) unsigned char smem[];
  lds_t<Tc>* const kt = (lds_t<Tc>*)smem;
  bf16* const vt = (bf16*)(kt + C * SK);
  float* const pw = (float*)(vt + C * SV);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), column = 32 * (wave % (DV / 32)), row = DK / 2 * (wave / (DV / 32));
  int lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int unit = blockIdx.x / segments, seg = blockIdx.x % segments, b = unit / A.heads, h = unit % A.heads;
  const int len = length_of(A, b), t0 = seg * seg_tokens, t1 = min(len, t0 + seg_tokens);
  fill_powers(pw, A.log_decay[h], tid, NT);
  const Tin* const k = rows_of<Tin>(A.k, A.k_stride, b, h / (A.heads / A.k_heads));
  const Tin* const v = rows_of<Tin>(A.v, A.v_stride, b, h / (A.heads / A.v_heads));
  const long long ks = A.k_stride[2], vs = A.v_stride[2];
  const auto at = [&](int t) -> long long { return REV ? len - 1 - t : t; };  // row of the t-th token of the walk
  f32x16 S[I];
#pragma unroll
  for (int i = 0; i < I; i++) S[i] = zero16();
  Staged<Tin, Tc, C, DK, NT, REV> sk;
  Staged<Tin, Split<3>, C, DV, NT, REV> sv;
  if (t0 < t1) {
    sk.load(k + at(t0) * ks, ks, t1 - t0, A.dim, tid);
    sv.load(v + at(t0) * vs, vs, t1 - t0, A.dim_v, tid);
  }
  for (int t = t0; t < t1; t += C) {
    forget(lane, half, col);
    const int n = min(C, t1 - t);
    __syncthreads();
    sk.store(kt, tid);
    sv.store(vt, tid, pw + kZero + n - 1 + (REV ? 1 : 0), A.update_scale);  // weight of token j: n - 1 - j powers (one more in reverse)
    __syncthreads();
    if (t + C < t1) {
      sk.load(k + at(t + C) * ks, ks, t1 - t - C, A.dim, tid);
      sv.load(v + at(t + C) * vs, vs, t1 - t - C, A.dim_v, tid);
    }
    const float all = pw[kZero + n];
#pragma unroll
    for (int i = 0; i < I; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) S[i][r] *= all;
#pragma unroll
    for (int s = 0; s < C / 16; s++) {
      const SplitX8<3> x = frag_cols<Split<3>, DV>(vt, 16 * s, column, lane);
#pragma unroll
      for (int i = 0; i < I; i++) S[i] = mma(frag_cols<Tc, DK>(kt, 16 * s, row + 32 * i, lane), x, S[i]);
    }
  }
  float* out = states + (long long)blockIdx.x * A.dim * A.dim_v;
  const int c = column + col;
#pragma unroll
  for (int i = 0; i < I; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int d = row + 32 * i + c_row(r, half);
      if (d < A.dim && c < A.dim_v) out[(long long)d * A.dim_v + c] = S[i][r];
    }
}

// States before the segments in place of the segments' own, and the final state.  16 heads of 32 states of 128 x 128: 17 us, 3.9 TB/s.
__global__ void __launch_bounds__(256) decay_scan(const Args A, int segments, int seg_tokens, float* states) {
  const int unit = blockIdx.y, b = unit / A.heads, h = unit % A.heads, size = A.dim * A.dim_v;
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= size) return;
  const int d = e / A.dim_v, c = e % A.dim_v, len = length_of(A, b);
  const float lg = A.log_decay[h], whole = power(lg, seg_tokens);
  float x = A.state_in ? A.state_in[(long long)unit * size + d * A.state_in_stride[0] + c * A.state_in_stride[1]] : 0.f;
  float* s = states + (long long)unit * segments * size + e;
  constexpr int U = 16;  // loads in flight
  for (int g0 = 0; g0 < segments; g0 += U) {
    float own[U];
#pragma unroll
    for (int u = 0; u < U; u++) own[u] = g0 + u < segments ? s[(long long)(g0 + u) * size] : 0.f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int g = g0 + u;
      if (g >= segments) break;
      const int n = min(max(len - g * seg_tokens, 0), seg_tokens);
      s[(long long)g * size] = x;
      x = (n == seg_tokens ? whole : power(lg, n)) * x + own[u];
    }
  }
  if (A.state_out) A.state_out[(long long)unit * size + d * A.state_out_stride[0] + c * A.state_out_stride[1]] = x;
}

// ---- outputs --------------------------------------------------------------------------------------------------------------------

// C tiles (rows: 32 tokens each, columns: the wavefront's 32 components) to memory, 16 bytes a lane, through 4096 bytes of LDS that
// belong to the wavefront (`strip`)
template <class T, bool REV, int U>
__device__ inline void store_rows(T* out, long long stride, const f32x16 (&o)[U], void* strip, int t, int t1, int len, int wave, int lane, int dim_v) {
  constexpr int VE = 16 / (int)sizeof(T), PER_ROW = 32 / VE;
  T* const tile = (T*)strip;
  const int half = lane >> 5, col = lane & 31, row0 = lane / PER_ROW, c = 32 * wave + (lane % PER_ROW) * VE;
  T* const place = tile + 128 * half + col;
#pragma unroll
  for (int u = 0; u < U; u++) {
#pragma unroll
    for (int r = 0; r < 16; r++) place[c_row(r, 0) * 32] = (T)o[u][r];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < PER_ROW / 2; i++) {
      const int row = row0 + i * (64 / PER_ROW), token = t + 32 * u + row;
      const uint4 x = *reinterpret_cast<const uint4*>(tile + row * 32 + (lane % PER_ROW) * VE);
      if (token < t1 && c < dim_v) *reinterpret_cast<uint4*>(out + (long long)(REV ? len - 1 - token : token) * stride + c) = x;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

template <class Tc, int DK, int DV> constexpr size_t query_bytes() {
  constexpr size_t q = (size_t)chunk<Tc>() * tile_stride<Tc, DK>() * 2, o = 4096 * (DV / 32);
  return q > o ? q : o;
}

// Two terms: two wavefronts a SIMD, which leaves no sums in accumulation registers: with one, the compiler stored row 1 of a float32
// tile 32 bytes behind row 0 instead of 128.
// CUT: sequences are cut into segments, whose states are known.  16 x 16384 tokens, 128 components: 78 us, 3.9 TB/s; 4x8x4096, 64
// components: 23 us, 3.6 TB/s.  Two wavefronts for every 32 columns, each with half of the tokens and of the state's rows, which
// makes four a SIMD of two, took 80 and 21 us (training at 128 components 251 for 245).
template <class Tin, class Tc, int DK, int DV, bool REV, bool CUT>
__global__ void __launch_bounds__(2 * DV, (Vec<Tc>::terms == 1 ? (DK <= DV ? 2 : 1) : Vec<Tc>::terms == 2 ? 2 : 1)) decay_outputs(const Args A, int segments, int seg_tokens, const float* states) {
  constexpr int C = chunk<Tc>(), U = C / 32, NT = 2 * DV, NW = DV / 32, SK = tile_stride<Tc, DK>(), SV = tile_stride<Tc, DV>(), SP = tile_stride<Tc, C>();
  extern __shared__ __align__(16) unsigned char smem[];
  lds_t<Tc>* const qt = (lds_t<Tc>*)smem;  // and, once the chunk's queries have been used, the outputs on their way
  lds_t<Tc>* const kt = (lds_t<Tc>*)(smem + query_bytes<Tc, DK, DV>());
  lds_t<Tc>* const vt = kt + C * SK;
  lds_t<Tc>* const pt = vt + C * SV;
  float* const pw = (float*)(pt + C * SP);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int lane = tid & 63, half = lane >> 5, col = lane & 31;
  void* const strip = smem + 4096 * wave;
  const int unit = blockIdx.x / segments, seg = blockIdx.x % segments, b = unit / A.heads, h = unit % A.heads;
  const int len = length_of(A, b), t0 = seg * seg_tokens, t1 = min(len, t0 + seg_tokens);
  const int c = 32 * wave + col, shift = REV ? 0 : 1;
  fill_powers(pw, A.log_decay[h], tid, NT);
  const Tin* const q = rows_of<Tin>(A.q, A.q_stride, b, h / (A.heads / A.q_heads));
  const Tin* const k = rows_of<Tin>(A.k, A.k_stride, b, h / (A.heads / A.k_heads));
  const Tin* const v = rows_of<Tin>(A.v, A.v_stride, b, h / (A.heads / A.v_heads));
  const long long qs = A.q_stride[2], ks = A.k_stride[2], vs = A.v_stride[2];
  const auto at = [&](int t) -> long long { return REV ? len - 1 - t : t; };  // row of the t-th token of the walk
  const long long os = A.out_stride[2], out0 = (long long)b * A.out_stride[0] + (long long)h * A.out_stride[1];

  f32x16 S[DK / 32];
  {
    const float* from = CUT ? states + (long long)blockIdx.x * A.dim * A.dim_v : (A.state_in ? A.state_in + (long long)unit * A.dim * A.dim_v : nullptr);
    const int s0 = (int)(CUT ? A.states_stride[0] : A.state_in_stride[0]), s1 = (int)(CUT ? A.states_stride[1] : A.state_in_stride[1]);
#pragma unroll
    for (int i = 0; i < DK / 32; i++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int d = 32 * i + 8 * g + 4 * half;  // (dim is a multiple of 4)
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (from && d < A.dim && c < A.dim_v) {
          if (s0 == 1) {
            x = *reinterpret_cast<const f32x4*>(from + c * s1 + d);
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = from[(d + j) * s0 + c * s1];
          }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) S[i][4 * g + j] = x[j];
      }
  }
  Staged<Tin, Tc, C, DK, NT, REV> sq, sk;
  Staged<Tin, Tc, C, DV, NT, REV> sv;
  if (t0 < t1) {
    sq.load(q + at(t0) * qs, qs, t1 - t0, A.dim, tid);
    sk.load(k + at(t0) * ks, ks, t1 - t0, A.dim, tid);
    sv.load(v + at(t0) * vs, vs, t1 - t0, A.dim_v, tid);
  }
  for (int t = t0; t < t1; t += C) {
    forget(lane, half, col);
    __syncthreads();
    sq.store(qt, tid);
    sk.store(kt, tid);
    sv.store(vt, tid);
    __syncthreads();
    if (t + C < t1) {
      sq.load(q + at(t + C) * qs, qs, t1 - t - C, A.dim, tid);
      sk.load(k + at(t + C) * ks, ks, t1 - t - C, A.dim, tid);
      sv.load(v + at(t + C) * vs, vs, t1 - t - C, A.dim_v, tid);
    }
    // decayed products within the chunk: 32 x 32 tiles (rows tokens j, columns tokens i >= j), shared through LDS
    for (int tile = wave; tile < U * (U + 1) / 2; tile += NW) {
      const int i0 = tile == 0 ? 0 : 32, j0 = tile == 2 ? 32 : 0;
      f32x16 a = zero16();
#pragma unroll
      for (int s = 0; s < DK / 16; s++) a = mma(frag_rows<Tc, DK>(kt, j0 + col, 16 * s, half), frag_rows<Tc, DK>(qt, i0 + col, 16 * s, half), a);
      const float* w = pw + kZero + i0 + col - j0 - 4 * half;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float x[4];
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = i0 + col >= j0 + 8 * g + 4 * half + u ? a[4 * g + u] * (w[-(8 * g + u)] * A.product_scale) : 0.f;
        put4<Tc, C>(pt, i0 + col, j0 + 8 * g + 4 * half, x[0], x[1], x[2], x[3]);
      }
    }
    // outputs: the state's part first, decayed to each row in float32, then the chunk's own
    f32x16 o[U];
#pragma unroll
    for (int u = 0; u < U; u++) o[u] = zero16();
#pragma unroll
    for (int i = 0; i < DK / 32; i++)
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const typename Vec<Tc>::x8 st = pack<Tc>(S[i], s);
#pragma unroll
        for (int u = 0; u < U; u++) o[u] = mma(frag_rows_split<Tc, DK>(qt, 32 * u + col, 32 * i + 16 * s, half), st, o[u]);
      }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int r = 0; r < 16; r++) o[u][r] *= pw[kZero + 32 * u + c_row(r, half) + shift] * A.query_scale;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < C / 16; s++) {
      const typename Vec<Tc>::x8 vf = frag_cols<Tc, DV>(vt, 16 * s, 32 * wave, lane);
#pragma unroll
      for (int u = s / 2; u < U; u++) o[u] = mma(frag_rows_split<Tc, C>(pt, 32 * u + col, 16 * s, half), vf, o[u]);
    }
    if (A.out_float32) store_rows<float, REV>((float*)A.out + out0, os, o, strip, t, t1, len, wave, lane, A.dim_v);
    else store_rows<Tin, REV>((Tin*)A.out + out0, os, o, strip, t, t1, len, wave, lane, A.dim_v);
    if ((!CUT && A.state_out) || t + C < t1) update_state<Tc, DK, DV, update_terms<Tc, !CUT>()>(S, kt, vt, pw, min(C, t1 - t), REV ? 1 : 0, A.update_scale, wave, lane);
  }
  // tokens behind the sequence
  for (int t = max(t0, len); t < min((int)A.tokens, t0 + seg_tokens); t++)
    for (int d = tid; d < A.dim_v; d += NT) {
      if (A.out_float32) ((float*)A.out)[out0 + t * os + d] = 0.f; else ((Tin*)A.out)[out0 + t * os + d] = (Tin)0.f;
    }
  if (!CUT && A.state_out) {
    float* to = A.state_out + (long long)unit * A.dim * A.dim_v;
#pragma unroll
    for (int i = 0; i < DK / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int d = 32 * i + c_row(r, half);
        if (d < A.dim && c < A.dim_v) to[d * A.state_out_stride[0] + c * A.state_out_stride[1]] = S[i][r];
      }
  }
}

// Sums over the heads that share one, in their order, four components to a thread (2 to 4 us for 3x6x777 tokens).
template <class Tin> __global__ void __launch_bounds__(256) decay_join(const Args A) {
  const int quads = A.dim_v / 4, J = A.joined_heads, group = A.heads / J;
  const long long total = (long long)A.batch * J * A.tokens * quads;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
    const int c = 4 * (int)(e % quads);
    const long long row = e / quads, t = row % A.tokens, unit = row / A.tokens;
    const int b = (int)(unit / J), j = (int)(unit % J);
    const float* p = (const float*)A.out + b * A.out_stride[0] + (long long)j * group * A.out_stride[1] + t * A.out_stride[2] + c;
    f32x4 x = *reinterpret_cast<const f32x4*>(p);
    for (int h = 1; h < group; h++) x += *reinterpret_cast<const f32x4*>(p + h * A.out_stride[1]);
    store4<Tin>((Tin*)A.joined + b * A.joined_stride[0] + j * A.joined_stride[1] + t * A.joined_stride[2] + c, x[0], x[1], x[2], x[3]);
  }
}

// ---- one token ----------------------------------------------------------------------------------------------------------------
//
// One read and one write of the state, float32.  A workgroup has `slice` columns of one head's state, 16 bytes of a row to a
// thread; the sum over the rows is joined in LDS.  64 x 16 states of 128 x 128: 134 MB in 22.4 us (6 TB/s, part of it from the
// cache behind HBM).
struct Strides2 { long long batch, head; };

template <class T>
__global__ void __launch_bounds__(256) decay_step(int heads, int group, int dim, int dim_v, int slice, float scale, const T* q, Strides2 qs, const T* k,
                                                  Strides2 ks, const T* v, Strides2 vs, const float* log_decay, float* state, T* out) {
  __shared__ float qk[2][128];
  __shared__ f32x4 red[256];
  const int unit = blockIdx.x, b = unit / heads, h = unit % heads, tid = threadIdx.x;
  for (int d = tid; d < dim; d += 256) {
    qk[0][d] = (float)q[b * qs.batch + h * qs.head + d] * scale;
    qk[1][d] = (float)k[b * ks.batch + (h / group) * ks.head + d];
  }
  const float g = expf(log_decay[h]);
  const int quads = slice / 4, c = blockIdx.y * slice + 4 * (tid % quads), r0 = tid / quads, step = 256 / quads;
  f32x4 vv = {0.f, 0.f, 0.f, 0.f}, acc = vv;
  const bool there = c < dim_v;
  if (there) {
    const T* vp = v + b * vs.batch + (h / group) * vs.head + c;
#pragma unroll
    for (int j = 0; j < 4; j++) vv[j] = (float)vp[j];
  }
  __syncthreads();
  float* s = state + (long long)unit * dim * dim_v + c;
  if (there) {
    constexpr int U = 8;  // rows of a thread in flight
    for (int d0 = r0; d0 < dim; d0 += U * step) {
      f32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (d0 + u * step < dim) x[u] = *reinterpret_cast<const f32x4*>(s + (long long)(d0 + u * step) * dim_v);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int d = d0 + u * step;
        if (d < dim) {
          const float kk = qk[1][d], qq = qk[0][d];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            x[u][j] = fmaf(g, x[u][j], kk * vv[j]);
            acc[j] = fmaf(qq, x[u][j], acc[j]);
          }
          *reinterpret_cast<f32x4*>(s + (long long)d * dim_v) = x[u];
        }
      }
    }
  }
  red[tid] = acc;
  __syncthreads();
  for (int o = 128; o >= quads; o >>= 1) {
    if (tid < o) {
#pragma unroll
      for (int j = 0; j < 4; j++) red[tid][j] += red[tid + o][j];
    }
    __syncthreads();
  }
  if (tid < quads && there) {
    T* op = out + (long long)unit * dim_v + c;
#pragma unroll
    for (int j = 0; j < 4; j++) op[j] = (T)red[tid][j];
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------

bool aligned(const Args* a) {
  const size_t size = a->dtype == 2 ? 4 : 2;
  return rows_aligned(a->q, a->q_stride, size) && rows_aligned(a->k, a->k_stride, size) && rows_aligned(a->v, a->v_stride, size) &&
         rows_aligned(a->out, a->out_stride, a->out_float32 ? 4 : size) && (!a->joined_heads || rows_aligned(a->joined, a->joined_stride, size)) &&
         (uintptr_t)a->state_in % 16 == 0 && (uintptr_t)a->states % 16 == 0;
}

const char* check(const Args* a) {
  if (!a) return "decay attention: null arguments";
  if (a->dtype < 0 || a->dtype > 2) return "decay attention: dtype must be 0 (bfloat16), 1 (float16) or 2 (float32)";
  const int ve = a->dtype == 2 ? 4 : 8;
  if (a->batch < 1 || a->heads < 1 || a->q_heads < 1 || a->k_heads < 1 || a->v_heads < 1 || a->heads % a->q_heads || a->heads % a->k_heads || a->heads % a->v_heads)
    return "decay attention: heads must be a multiple of the heads of q, k and v";
  if (a->dim < ve || a->dim > 128 || a->dim % ve || a->dim_v < ve || a->dim_v > 128 || a->dim_v % ve)
    return "decay attention: dim and dim_v must be multiples of 16 bytes, at most 128";
  if (a->tokens < 0 || a->tokens > (1 << 29)) return "decay attention: tokens out of range";
  if (a->joined_heads < 0 || (a->joined_heads > 0 && (!a->out_float32 || a->heads % a->joined_heads || (a->tokens > 0 && !a->joined))))
    return "decay attention: joined outputs need float32 outputs, heads that are a multiple of theirs and a place";
  for (const int64_t* x : {a->q_stride, a->k_stride, a->v_stride, a->out_stride})
    if (x[2] < 0 || x[2] > kMaxRowStride) return "decay attention: rows too far apart";
  if (!aligned(a)) return "decay attention: a row does not start at a multiple of 16 bytes";
  if (!a->log_decay || (a->tokens > 0 && (!a->q || !a->k || !a->v || !a->out))) return "decay attention: null data";
  if ((int64_t)a->batch * a->heads > 65535) return "decay attention: more than 65535 sequences times heads";
  return nullptr;
}

// Segments of a sequence: as many workgroups as the chip takes at once, whole chunks each; more of them carry more states, and a few
// more wait for a second turn (220 sequences times heads of 2094 tokens in 3 segments 722 us, in 2 636).  A prompt of
// 16 x 16384 tokens, 128 components, with 256, 512, 768 and 1024 workgroups: 191, 144, 154 and 168 us; training of 4x8x4096, 64
// components, with 256, 512, 768, 1024 and 2048: 237, 167, 148, 148 and 166.
void segments_of(const Args* a, int& segments, int& seg_tokens) {
  const int64_t units = (int64_t)a->batch * a->heads, chunks = (a->tokens + kChunk - 1) / kChunk;
  const int64_t fill = a->dim > 64 || a->dim_v > 64 ? 512 : 1024;  // (the same for exchanged dims: the states are shared)
  int64_t want = fill / units;
  if (want > chunks) want = chunks;
  if (want < 1) want = 1;
  const int64_t per = chunks < 1 ? 1 : (chunks + want - 1) / want;
  segments = (int)(chunks < 1 ? 1 : (chunks + per - 1) / per);
  seg_tokens = (int)(per * kChunk);
}

template <class K> int prepare_lds(K kernel, size_t bytes) {
  if (bytes <= 64 * 1024) return 0;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  return e == hipSuccess ? 0 : keops_seq_fail((int)e, "decay attention: shared memory");
}

template <class Tin, class Tc, int DK, int DV, bool REV> int run(const Args& a, hipStream_t st) {
  float* const work = a.states;
  int segments, seg_tokens;
  segments_of(&a, segments, seg_tokens);
  const int units = a.batch * a.heads;
  constexpr int C = chunk<Tc>();
  const size_t kv = (size_t)C * (tile_stride<Tc, DK>() + tile_stride<Tc, DV>()) * 2, pw = kPowers * sizeof(float);
  const size_t all = query_bytes<Tc, DK, DV>() + kv + (size_t)C * tile_stride<Tc, C>() * 2 + pw;
  if (segments > 1 && !a.states_given) {
    const size_t lds = (size_t)C * (tile_stride<Tc, DK>() + tile_stride<Split<3>, DV>()) * 2 + pw;
    if (int e = prepare_lds(decay_states<Tin, Tc, DK, DV, REV>, lds)) return e;
    decay_states<Tin, Tc, DK, DV, REV><<<units * segments, 4 * DV, lds, st>>>(a, segments, seg_tokens, work);
    decay_scan<<<dim3((a.dim * a.dim_v + 255) / 256, units), 256, 0, st>>>(a, segments, seg_tokens, work);
  }
  const auto outputs = segments > 1 ? decay_outputs<Tin, Tc, DK, DV, REV, true> : decay_outputs<Tin, Tc, DK, DV, REV, false>;
  if (int e = prepare_lds(outputs, all)) return e;
  outputs<<<units * segments, 2 * DV, all, st>>>(a, segments, seg_tokens, work);
  const int64_t joins = a.joined_heads ? ((int64_t)a.batch * a.joined_heads * a.tokens * (a.dim_v / 4) + 255) / 256 : 0;
  if (joins > 0) decay_join<Tin><<<(unsigned)(joins < 65536 ? joins : 65536), 256, 0, st>>>(a);
  return seq_launched("decay attention: launch");
}

template <class Tin, class Tc, bool REV> int by_dims(const Args& a, hipStream_t st) {
  if (a.dim <= 64) return a.dim_v <= 64 ? run<Tin, Tc, 64, 64, REV>(a, st) : run<Tin, Tc, 64, 128, REV>(a, st);
  return a.dim_v <= 64 ? run<Tin, Tc, 128, 64, REV>(a, st) : run<Tin, Tc, 128, 128, REV>(a, st);
}

template <class Tin, class Tc> int dispatch(const Args& a, hipStream_t st) {
  return a.reverse ? by_dims<Tin, Tc, true>(a, st) : by_dims<Tin, Tc, false>(a, st);
}

template <class T>
int step(int batch, int heads, int group, int dim, int dim_v, float scale, const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v,
         const int64_t* vs, const float* log_decay, float* state, void* out, hipStream_t st) {
  // Narrow slices while whole heads would not give two workgroups to a CU: 32 states of 128 x 128 4.1 us (whole heads: 5.1), 320 9.5
  // (9.8), 1024 22.4 whole (slices: 23.1).
  const int units = batch * heads, slice = units >= 512 ? 128 : 32;
  decay_step<T><<<dim3(units, (dim_v + slice - 1) / slice), 256, 0, st>>>(heads, group, dim, dim_v, slice, scale, (const T*)q, Strides2{qs[0], qs[1]},
                                                                          (const T*)k, Strides2{ks[0], ks[1]}, (const T*)v, Strides2{vs[0], vs[1]}, log_decay,
                                                                          state, (T*)out);
  return seq_launched("decay attention step: launch");
}

}  // namespace

extern "C" {

size_t keops_hip_decay_attention_bytes(const keops_hip_decay_attention* a) {
  if (check(a)) return 0;
  int segments, seg_tokens;
  segments_of(a, segments, seg_tokens);
  return segments > 1 ? (size_t)a->batch * a->heads * segments * a->dim * a->dim_v * sizeof(float) : 0;
}

int keops_hip_decay_attention_run(const keops_hip_decay_attention* a, int device, void* hip_stream) {
  if (const char* why = check(a)) return keops_seq_fail(-1, why);
  const size_t need = keops_hip_decay_attention_bytes(a);
  if (need > (size_t)(a->states_bytes > 0 ? a->states_bytes : 0) || (need > 0 && !a->states)) return keops_seq_fail(-1, "decay attention: workspace too small");
  if (a->states_given && need != (size_t)a->states_bytes) return keops_seq_fail(-1, "decay attention: the states given are not of this call's segments");
  if (a->states_given && need > 0 && a->state_out) return keops_seq_fail(-1, "decay attention: no final state where the states are given");
  SeqDevice on(device);
  hipStream_t st = (hipStream_t)hip_stream;
  if (a->dtype == 0) return dispatch<bf16, bf16>(*a, st);
  if (a->dtype == 1) return dispatch<f16, Split<2>>(*a, st);
  return dispatch<float, Split<3>>(*a, st);
}

int keops_hip_decay_attention_step(int dtype, int batch, int heads, int kv_heads, int dim, int dim_v, float scale, const void* q, const int64_t* q_stride,
                                   const void* k, const int64_t* k_stride, const void* v, const int64_t* v_stride, const float* log_decay, float* state,
                                   void* out, int device, void* hip_stream) {
  if (dtype < 0 || dtype > 2) return keops_seq_fail(-1, "decay attention step: dtype must be 0 (bfloat16), 1 (float16) or 2 (float32)");
  if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads) return keops_seq_fail(-1, "decay attention step: heads must be a multiple of kv_heads");
  if (dim < 1 || dim > 128 || dim_v < 4 || dim_v > 128 || dim_v % 4) return keops_seq_fail(-1, "decay attention step: dim at most 128, dim_v a multiple of 4, at most 128");
  if ((int64_t)batch * heads > 0x7fffffff) return keops_seq_fail(-1, "decay attention step: too many workgroups");
  if (!q || !q_stride || !k || !k_stride || !v || !v_stride || !log_decay || !state || !out) return keops_seq_fail(-1, "decay attention step: null data");
  SeqDevice on(device);
  hipStream_t st = (hipStream_t)hip_stream;
  const int group = heads / kv_heads;
  if (dtype == 0) return step<bf16>(batch, heads, group, dim, dim_v, scale, q, q_stride, k, k_stride, v, v_stride, log_decay, state, out, st);
  if (dtype == 1) return step<f16>(batch, heads, group, dim, dim_v, scale, q, q_stride, k, k_stride, v, v_stride, log_decay, state, out, st);
  return step<float>(batch, heads, group, dim, dim_v, scale, q, q_stride, k, k_stride, v, v_stride, log_decay, state, out, st);
}

}  // extern "C"
