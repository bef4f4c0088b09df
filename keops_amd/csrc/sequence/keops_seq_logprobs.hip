// Rows of logits x: log probability of a given token, entropy and the largest alternatives in one sweep, and the gradient.
//
// With m = max x, s = sum e^(x-m), t = sum e^(x-m) (x-m):  lse = m + log s,  entropy = log s - t / s.  Both terms of the entropy
// are non-negative, so nothing cancels; x - m is formed before it is scaled, so large logits lose nothing.  m, s and t are kept
// for each thread (a new maximum m' turns t into e^(m-m') (t + s (m-m'))) and joined at the end.
//
// The K largest: each wavefront keeps a list in LDS, which a value enters when it exceeds the K-th of what the list last held; the
// list is cut to its K largest when it fills.  The first threshold is the K-th largest of the lanes' own maxima, so in the sweep
// almost every vector of a row costs one comparison and no barrier.  Keys are the value's bits in increasing order, then the
// complement of the index, so equal values keep the lowest index and every key is different: the result does not depend on the
// order in which values arrive.
#include "../../../include/keops_hip.h"
#include "keops_seq.h"

using namespace kseq;

namespace {

constexpr int kThreads = 256, kList = 512, kWaveList = 192, kMaxTop = KEOPS_HIP_MAX_TOP, kUnroll = 4;
constexpr float kLn2 = 0.6931471805599453f;
typedef unsigned long long u64;

struct Stat { float m, s, t; };

__device__ inline unsigned ordered(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(u64 key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ inline u64 key_of(float x, long long index) { return ((u64)ordered(x) << 32) | (0xffffffffu - (unsigned)index); }

struct Row {  // columns v0..v1 of a row as 16-byte vectors
  long long first, v0, v1;
  int count;
};
template <class T> __device__ inline Row row_of(const T* x, long long v0, long long v1) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int past = (int)(((uintptr_t)(x + v0) & 15) / sizeof(T));  // elements of the first vector that lie before v0
  Row r;
  r.first = v0 - past;
  r.v0 = v0;
  r.v1 = v1;
  r.count = (int)((v1 - r.first + VE - 1) / VE);
  return r;
}
template <class T> __device__ inline uint4 load_vec(const T* x, const Row& r, int j) {
  constexpr int VE = 16 / (int)sizeof(T);
  const long long i = r.first + (long long)j * VE;
  if (i >= r.v0 && i + VE <= r.v1) return *reinterpret_cast<const uint4*>(x + i);
  union { uint4 u; T e[VE]; } w;
#pragma unroll
  for (int k = 0; k < VE; k++) {
    w.e[k] = (T)-kInf;
    if (i + k >= r.v0 && i + k < r.v1) w.e[k] = x[i + k];
  }
  return w.u;
}
template <class T> __device__ inline void unpack(const uint4& u, float (&x)[16 / sizeof(T)]) {
  union { uint4 u; T e[16 / sizeof(T)]; } w;
  w.u = u;
#pragma unroll
  for (int k = 0; k < (int)(16 / sizeof(T)); k++) x[k] = (float)w.e[k];
}

// element k of a 16-byte vector
template <class T> __device__ inline float element(const uint4& u, int k) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(k == 0 ? u.x : (k == 1 ? u.y : (k == 2 ? u.z : u.w)));
  } else {
    const unsigned w = k < 2 ? u.x : (k < 4 ? u.y : (k < 6 ? u.z : u.w));
    union { unsigned short b; T e; } x;
    x.b = (unsigned short)(k & 1 ? w >> 16 : w);
    return (float)x.e;
  }
}

// LDS accesses of a wavefront before this come before those behind it
__device__ inline void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// list[0..n) -> its `top` largest in decreasing order, in list[0..); returns how many.  All threads of the workgroup.
__device__ inline int cut(u64* list, u64* best, int n, int top, int tid) {
  __syncthreads();
  u64 mine[kList / kThreads];
  int rank[kList / kThreads];
#pragma unroll
  for (int i = 0; i < kList / kThreads; i++) {
    mine[i] = tid + i * kThreads < n ? list[tid + i * kThreads] : 0;
    rank[i] = 0;
  }
#pragma unroll 8
  for (int j = 0; j < n; j++) {
    const u64 o = list[j];
#pragma unroll
    for (int i = 0; i < kList / kThreads; i++) rank[i] += o > mine[i] || (o == mine[i] && j < tid + i * kThreads) ? 1 : 0;  // (0: no key)
  }
#pragma unroll
  for (int i = 0; i < kList / kThreads; i++)
    if (tid + i * kThreads < n && rank[i] < top) best[rank[i]] = mine[i];
  __syncthreads();
  const int left = n < top ? n : top;
  if (tid < left) list[tid] = best[tid];
  __syncthreads();
  return left;
}

// the same for the list of one wavefront (n <= kWaveList different keys)
__device__ inline int cut_wave(u64* list, int n, int top, int lane) {
  constexpr int E = kWaveList / 64;
  u64 mine[E];
  int rank[E];
#pragma unroll
  for (int i = 0; i < E; i++) {
    mine[i] = lane + 64 * i < n ? list[lane + 64 * i] : 0;
    rank[i] = 0;
  }
#pragma unroll 8
  for (int j = 0; j < n; j++) {
    const u64 o = list[j];
#pragma unroll
    for (int i = 0; i < E; i++) rank[i] += o > mine[i] ? 1 : 0;
  }
  wave_fence();
#pragma unroll
  for (int i = 0; i < E; i++)
    if (lane + 64 * i < n && rank[i] < top) list[rank[i]] = mine[i];
  wave_fence();
  return n < top ? n : top;
}

struct Out {
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_index;
};

template <class T>
__device__ inline void finish(const Out& o, long long row, const Stat& st, const T* x, long long vocab, int64_t token, int64_t ignore) {
  const float ls = st.s > 0.f ? __builtin_amdgcn_logf(st.s) * kLn2 : st.s == 0.f ? -kInf : st.s;
  const bool nothing = st.m == -kInf;
  o.lse[row] = nothing ? -kInf : st.m + ls;
  o.entropy[row] = nothing ? 0.f : ls - st.t / st.s;
  float lp;
  if (token == ignore) lp = 0.f;
  else if (token < 0 || token >= vocab) lp = __builtin_nanf("");
  else lp = nothing ? -kInf : ((float)x[token] - st.m) - ls;
  o.logprob[row] = lp;
}
__device__ inline void finish_top(const Out& o, long long at, const Stat& st, u64 key) {
  const float ls = __builtin_amdgcn_logf(st.s) * kLn2;
  o.top_logprob[at] = st.m == -kInf ? -kInf : (value_of(key) - st.m) - ls;
  o.top_index[at] = (int64_t)(0xffffffffu - (unsigned)key);
}

// joins the sums of a wavefront's lanes; every lane gets the result.  The largest m first, so that every lane scales its sums once.
__device__ inline Stat join_lanes(Stat st) {
  float m = st.m, bad = !(st.m < kInf) || st.s != st.s ? 1.f : 0.f;  // +inf or NaN: the row's sums are NaN
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float d = st.m - m, f = st.m == -kInf ? 0.f : __builtin_amdgcn_exp2f(d * kLog2e);
  st.t = f == 0.f ? 0.f : f * (st.t + st.s * d);  // (a factor that has vanished takes its sums with it: s (m - m') may be infinite)
  st.s = f == 0.f ? 0.f : f * st.s;
  if (__any(bad != 0.f)) st.s = st.t = __builtin_nanf("");
  st.m = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    st.s += __shfl_xor(st.s, o);
    st.t += __shfl_xor(st.t, o);
  }
  return st;
}
// joins the threads' sums (NT threads); the first wavefront gets the result
template <int NT> __device__ inline Stat join_all(Stat st, Stat* red, int tid) {
  st = join_lanes(st);
  if ((tid & 63) == 0) red[tid >> 6] = st;
  __syncthreads();
  if (tid < 64) st = join_lanes(tid < NT / 64 ? red[tid] : Stat{-kInf, 0.f, 0.f});
  return st;
}

// One row, or one share of a row's columns (which then leaves its sums and keys in `part`), vectors of 16 bytes, four to a thread on
// their way while four are worked on.  2048 x 50021 float32: 107 us, 3.8 TB/s; 4096 x 131072 bf16: 195 us, 5.5 TB/s (a copy reaches
// 4.9); few rows are bound by the exponentials of one CU.
template <class T, bool TOP, int NT>
__global__ void __launch_bounds__(NT) logprobs_rows(long long vocab, int top, const T* logits, long long stride, const int64_t* tokens, int64_t ignore,
                                                    Out out, int splits, float* part_stat, u64* part_key) {
  constexpr int VE = 16 / (int)sizeof(T), U = kUnroll, NW = NT / 64;
  __shared__ Stat red[NW];
  __shared__ u64 lists[TOP ? NW : 1][TOP ? kWaveList : 1], list[TOP ? NW * kMaxTop : 1], best[TOP ? kMaxTop : 1], floors[NW];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  u64* const own = lists[TOP ? wave : 0];
  int held = 0;  // keys in it
  const long long row = blockIdx.x / splits;
  const int split = blockIdx.x % splits;
  const T* x = logits + row * stride;
  const long long share = (vocab + splits - 1) / splits, v0 = split * share, v1 = v0 + share < vocab ? v0 + share : vocab;
  const Row r = row_of(x, v0, v1 < v0 ? v0 : v1);
  Stat st = {-kInf, 0.f, 0.f};
  u64 least = 0;  // keys up to this one are not among the largest
  float least_value = -kInf, lane_max = -kInf;
  bool lane_any = false;

  // K-th largest of the lanes' maxima, to 16 bits and from below: at least K values reach it
  const auto raise = [&]() __attribute__((always_inline)) {
    const unsigned mine = lane_any ? ordered(lane_max) : 0u;
    unsigned at = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
      const unsigned with = at | 1u << bit;
      if (__popcll(__ballot(mine >= with)) >= top) at = with;
    }
    if ((u64)at << 32 > least) {
      least = (u64)at << 32;
      least_value = value_of(least);
    }
  };

  uint4 next[U];
#pragma unroll
  for (int u = 0; u < U; u++)
    if (tid + u * NT < r.count) next[u] = load_vec(x, r, tid + u * NT);
  for (int j0 = 0; j0 < r.count; j0 += U * NT) {
    uint4 now[U];
#pragma unroll
    for (int u = 0; u < U; u++) now[u] = next[u];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int j = j0 + (U + u) * NT + tid;
      if (j < r.count) next[u] = load_vec(x, r, j);
    }
    float vmax[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      vmax[u] = -kInf;
      if (j0 + u * NT + tid >= r.count) continue;
      float e[VE];
      unpack<T>(now[u], e);
      float mx = e[0];
#pragma unroll
      for (int k = 1; k < VE; k++) mx = fmaxf(mx, e[k]);  // (NaN only if all are: the sums below find the others)
      vmax[u] = mx;
      if (!(mx <= st.m)) {  // a new maximum
        if (st.m != -kInf) {
          const float d = st.m - mx, f = __builtin_amdgcn_exp2f(d * kLog2e);
          st.t = f == 0.f ? 0.f : f * (st.t + st.s * d);
          st.s *= f;
        }
        st.m = mx;
      }
      if (st.m != -kInf) {
#pragma unroll
        for (int k = 0; k < VE; k++) {
          const float d = e[k] - st.m, f = __builtin_amdgcn_exp2f(d * kLog2e);
          st.s += f;
          st.t = fmaf(f, fmaxf(d, -1e4f), st.t);  // (-inf adds nothing: 0 * -1e4)
        }
      } else {
#pragma unroll
        for (int k = 0; k < VE; k++)
          if (e[k] != e[k]) st.m = e[k];  // NaN beside -inf
      }
      if (TOP) {
        lane_max = fmaxf(lane_max, mx);
        lane_any = true;
      }
    }
    if constexpr (TOP) {
      if (j0 == 0) raise();
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (!__any(j0 + u * NT + tid < r.count && !(vmax[u] < least_value))) continue;
        const uint4 cur = now[u];
        const long long i0 = r.first + (long long)(j0 + u * NT + tid) * VE;
        unsigned bits = 0;  // the lane's elements to look at
        if (j0 + u * NT + tid < r.count) {
          float e[VE];
          unpack<T>(cur, e);
#pragma unroll
          for (int k = 0; k < VE; k++)
            if (!(e[k] < least_value)) bits |= 1u << k;
          if (i0 < r.v0) bits &= ~0u << (int)(r.v0 - i0);
          if (i0 + VE > r.v1) bits &= (1u << (int)(r.v1 - i0)) - 1u;
        }
        while (__any(bits != 0)) {
          const int k = bits ? __builtin_ctz(bits) : 0;
          const u64 key = key_of(element<T>(cur, k), i0 + k);
          const bool enters = bits != 0 && key > least;
          bits &= bits - 1;
          const unsigned long long who = __ballot(enters);
          if (enters) own[held + __popcll(who & ((1ull << lane) - 1))] = key;
          held += __popcll(who);
          if (held > kWaveList - 64) {
            // a higher threshold and what it leaves; where that is not enough, the K largest themselves
            raise();
            wave_fence();
            u64 had[kWaveList / 64];
#pragma unroll
            for (int q = 0; q < kWaveList / 64; q++) had[q] = 64 * q + lane < held ? own[64 * q + lane] : 0;
            wave_fence();
            held = 0;
#pragma unroll
            for (int q = 0; q < kWaveList / 64; q++) {
              const unsigned long long stay = __ballot(had[q] > least);
              if (had[q] > least) own[held + __popcll(stay & ((1ull << lane) - 1))] = had[q];
              held += __popcll(stay);
            }
            if (held > kWaveList / 2) {
              wave_fence();
              held = cut_wave(own, held, top, lane);
              if (held == top) {
                least = own[top - 1];
                least_value = value_of(least);
              }
            }
          }
        }
      }
    }
  }
  if constexpr (TOP) {
    wave_fence();
    held = cut_wave(own, held, top, lane);
    if (lane == 0) floors[wave] = held == top ? own[top - 1] : 0;
    if (tid == 0) count = 0;
    __syncthreads();
    // of the wavefronts' lists, what reaches the largest of their last keys, in order
    u64 floor = floors[0];
#pragma unroll
    for (int w = 1; w < NW; w++) floor = floors[w] > floor ? floors[w] : floor;
    if (lane < held && own[lane] >= floor) list[atomicAdd(&count, 1)] = own[lane];
    if (tid < top) best[tid] = 0;
    __syncthreads();
    const int n = count;
    if (tid < n) {
      const u64 mine = list[tid];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; j++) rank += list[j] > mine ? 1 : 0;
      if (rank < top) best[rank] = mine;
    }
  }
  st = join_all<NT>(st, red, tid);
  if (splits == 1) {
    if (tid == 0) finish(out, row, st, x, vocab, tokens[row], ignore);
    if (TOP && tid < top) finish_top(out, row * top + tid, st, best[tid]);
  } else {
    if (tid == 0) {
      float* p = part_stat + (long long)blockIdx.x * 4;
      p[0] = st.m;
      p[1] = st.s;
      p[2] = st.t;
    }
    if (TOP && tid < top) part_key[(long long)blockIdx.x * top + tid] = best[tid];
  }
}

// the shares of one row
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_join(long long vocab, int top, const T* logits, long long stride, const int64_t* tokens, int64_t ignore,
                                                          Out out, int splits, const float* part_stat, const u64* part_key) {
  __shared__ Stat red[4];
  __shared__ u64 list[kList], best[kMaxTop];
  __shared__ int held;
  const int tid = threadIdx.x;
  const long long row = blockIdx.x;
  Stat st = {-kInf, 0.f, 0.f};
  if (tid < splits) {
    const float* p = part_stat + (row * splits + tid) * 4;
    st.m = p[0];
    st.s = p[1];
    st.t = p[2];
  }
  st = join_all<kThreads>(st, red, tid);
  if (tid == 0) finish(out, row, st, logits + row * stride, vocab, tokens[row], ignore);
  if (top == 0) return;
  const u64* keys = part_key + row * splits * top;
  const int all = splits * top;
  // the last of any share's keys is reached by K of them: what lies below the largest such key is out
  u64 floor = tid < splits ? keys[tid * top + top - 1] : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 x = __shfl_xor(floor, o);
    floor = x > floor ? x : floor;
  }
  if ((tid & 63) == 0) best[tid >> 6] = floor;
  if (tid == 0) held = 0;
  __syncthreads();
  floor = best[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; w++) floor = best[w] > floor ? best[w] : floor;
  for (int at = 0; at < all; at += kThreads) {
    const u64 key = at + tid < all ? keys[at + tid] : 0;
    if (key != 0 && key >= floor) list[atomicAdd(&held, 1)] = key;
    __syncthreads();
    const int n = held;
    __syncthreads();
    if (n > kList - kThreads || at + kThreads >= all) {
      const int left = cut(list, best, n, top, tid);
      if (tid == 0) held = left;
      __syncthreads();
    }
  }
  if (tid < top) finish_top(out, row * top + tid, st, list[tid]);
}

// dx = -p (a + c (x - lse + entropy)), a = sum of the incoming gradients of this row's log probabilities, c = that of the
// entropy; the tokens whose log probabilities were returned get theirs added.  One read and one write; the few given tokens are
// written again by threads of the workgroup that has their columns, behind a barrier.  2048 x 50021 float32: 139 us, 5.9 TB/s.
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_grad(long long vocab, int top, const T* logits, long long stride, const int64_t* tokens, int64_t ignore,
                                                          const float* entropy, const float* lse, const int64_t* top_index, const float* g_logprob,
                                                          const float* g_entropy, const float* g_top, T* grad, long long grad_stride, int blocks) {
  constexpr int VE = 16 / (int)sizeof(T), U = kUnroll;
  __shared__ float gs[kMaxTop + 1];
  __shared__ long long is[kMaxTop + 1];
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / blocks, share = (long long)U * kThreads * VE;
  const T* x = logits + row * stride;
  T* dx = grad + row * grad_stride;
  const float l = lse[row], H = entropy[row], c = g_entropy ? g_entropy[row] : 0.f;
  if (tid <= top) {
    float g = 0.f;
    long long i = -1;
    if (tid < top) {
      if (g_top) g = g_top[row * top + tid];
      i = top_index[row * top + tid];
    } else if (g_logprob) {
      const int64_t token = tokens[row];
      if (token != ignore) {
        i = token;
        g = token < 0 || token >= vocab ? __builtin_nanf("") : g_logprob[row];  // no such token: the row's gradient is NaN
      }
    }
    gs[tid] = g;
    is[tid] = i;
  }
  __syncthreads();
  float a = 0.f;
  for (int i = 0; i <= top; i++) a += gs[i];
  const bool nothing = l == -kInf;
  const auto at = [&](float v) {
    const float d = v - l, p = __builtin_amdgcn_exp2f(d * kLog2e);
    return nothing || p == 0.f ? 0.f : -p * fmaf(c, d + H, a);
  };
  // this workgroup's columns begin where the row has 16-byte boundaries
  const int past = (int)(((uintptr_t)x & 15) / sizeof(T));
  const long long b0 = (blockIdx.x % blocks) * share - past, v0 = b0 < 0 ? 0 : b0, v1 = b0 + share < vocab ? b0 + share : vocab;
  const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;
  uint4 in[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const long long i = b0 + (long long)(u * kThreads + tid) * VE;
    if (i >= v0 && i + VE <= v1) in[u] = *reinterpret_cast<const uint4*>(x + i);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const long long i = b0 + (long long)(u * kThreads + tid) * VE;
    if (i >= v0 && i + VE <= v1) {
      float e[VE];
      unpack<T>(in[u], e);
      union { uint4 q; T e[VE]; } w;
#pragma unroll
      for (int k = 0; k < VE; k++) w.e[k] = (T)at(e[k]);
      if (same) {
        *reinterpret_cast<uint4*>(dx + i) = w.q;
      } else {
#pragma unroll
        for (int k = 0; k < VE; k++) dx[i + k] = w.e[k];
      }
    } else {
      for (int k = 0; k < VE; k++)
        if (i + k >= v0 && i + k < v1) dx[i + k] = (T)at((float)x[i + k]);
    }
  }
  __syncthreads();
  if (tid <= top && is[tid] >= v0 && is[tid] < v1) {
    // the token may be among the alternatives too: every writer of a column writes the same sum
    float g = 0.f;
    for (int i = 0; i <= top; i++)
      if (is[i] == is[tid]) g += gs[i];
    dx[is[tid]] = (T)(nothing ? 0.f : at((float)x[is[tid]]) + g);
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------

const char* check(int dtype, int64_t rows, int64_t vocab, int top) {
  if (dtype < 0 || dtype > 2) return "token log probabilities: dtype must be 0 (bfloat16), 1 (float16) or 2 (float32)";
  if (rows < 0 || vocab < 1 || vocab > 0x7fffffff) return "token log probabilities: rows or vocabulary out of range";
  if (top < 0 || top > KEOPS_HIP_MAX_TOP || top > vocab) return "token log probabilities: top must be at most 64 and at most the vocabulary";
  return nullptr;
}

// At most one row to a CU and more than a few vectors of it to a thread: workgroups of 1024 threads, otherwise of 256 (us, 1024
// threads and 256): 4 x 32003 bf16 with 5 alternatives 11.8 and 17.1, 256 x 32000 24.5 and 30.1, 512 x 32000 33.9 and 31.6,
// 1000 x 8192 float32 29.8 and 14.9.  A row of 65536 columns or more is then shared by workgroups while there are less than two on
// a CU: 4 x 131072 17.6 (one workgroup: 47.5; shares of 16384 and 65536 columns 17.2 and 21.0); 4 x 32003 in shares of 4096 11.7 and
// 4.9 for the join and the gap between them.
bool wide(int64_t rows, int64_t vocab) { return rows < 512 && vocab >= 8192; }
int splits_of(int64_t rows, int64_t vocab) {
  if (!wide(rows, vocab)) return 1;
  int64_t s = 512 / rows, most = vocab / 32768;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

template <class T>
int forward(int64_t rows, int64_t vocab, int top, const void* logits, int64_t stride, const int64_t* tokens, int64_t ignore, const Out& out, void* work, hipStream_t st) {
  const int splits = splits_of(rows, vocab);
  u64* keys = (u64*)work;
  float* stats = (float*)(keys + (size_t)rows * splits * top);
  const unsigned grid = (unsigned)(rows * splits);
  const bool w = wide(rows, vocab);
  const auto kernel = top ? (w ? logprobs_rows<T, true, 1024> : logprobs_rows<T, true, 256>) : (w ? logprobs_rows<T, false, 1024> : logprobs_rows<T, false, 256>);
  kernel<<<grid, w ? 1024 : 256, 0, st>>>(vocab, top, (const T*)logits, stride, tokens, ignore, out, splits, stats, keys);
  if (splits > 1) logprobs_join<T><<<(unsigned)rows, kThreads, 0, st>>>(vocab, top, (const T*)logits, stride, tokens, ignore, out, splits, stats, keys);
  return seq_launched("token log probabilities: launch");
}

template <class T>
int backward(int64_t rows, int64_t vocab, int top, const void* logits, int64_t stride, const int64_t* tokens, int64_t ignore, const float* entropy, const float* lse,
             const int64_t* top_index, const float* gl, const float* ge, const float* gt, void* grad, int64_t grad_stride, hipStream_t st) {
  const int64_t share = (int64_t)kUnroll * kThreads * (16 / sizeof(T)), blocks = (vocab + 16 / sizeof(T) - 1 + share - 1) / share;
  if (rows * blocks > 0x7fffffff) return keops_seq_fail(-1, "token log probabilities: too many workgroups");
  logprobs_grad<T><<<(unsigned)(rows * blocks), kThreads, 0, st>>>(vocab, top, (const T*)logits, stride, tokens, ignore, entropy, lse, top_index, gl, ge, gt,
                                                                  (T*)grad, grad_stride, (int)blocks);
  return seq_launched("token log probabilities: launch of the backward pass");
}

}  // namespace

extern "C" {

size_t keops_hip_token_logprobs_bytes(int dtype, int64_t rows, int64_t vocab, int top) {
  if (check(dtype, rows, vocab, top)) return 0;
  const int splits = splits_of(rows, vocab);
  return splits > 1 ? (size_t)rows * splits * (top * sizeof(u64) + 4 * sizeof(float)) : 0;
}

int keops_hip_token_logprobs(int dtype, int64_t rows, int64_t vocab, int top, const void* logits, int64_t row_stride, const int64_t* tokens,
                             int64_t ignore_index, float* logprob, float* entropy, float* lse, float* top_logprob, int64_t* top_index, void* work,
                             size_t work_bytes, int device, void* hip_stream) {
  if (const char* why = check(dtype, rows, vocab, top)) return keops_seq_fail(-1, why);
  if (rows == 0) return 0;
  if (rows * splits_of(rows, vocab) > 0x7fffffff) return keops_seq_fail(-1, "token log probabilities: too many workgroups");
  if (!logits || !tokens || !logprob || !entropy || !lse || (top && (!top_logprob || !top_index))) return keops_seq_fail(-1, "token log probabilities: null data");
  const size_t need = keops_hip_token_logprobs_bytes(dtype, rows, vocab, top);
  if (need > work_bytes || (need > 0 && !work)) return keops_seq_fail(-1, "token log probabilities: workspace too small");
  SeqDevice on(device);
  hipStream_t st = (hipStream_t)hip_stream;
  const Out out = {logprob, entropy, lse, top_logprob, top_index};
  if (dtype == 0) return forward<bf16>(rows, vocab, top, logits, row_stride, tokens, ignore_index, out, work, st);
  if (dtype == 1) return forward<f16>(rows, vocab, top, logits, row_stride, tokens, ignore_index, out, work, st);
  return forward<float>(rows, vocab, top, logits, row_stride, tokens, ignore_index, out, work, st);
}

int keops_hip_token_logprobs_backward(int dtype, int64_t rows, int64_t vocab, int top, const void* logits, int64_t row_stride, const int64_t* tokens,
                                      int64_t ignore_index, const float* entropy, const float* lse, const int64_t* top_index, const float* grad_logprob,
                                      const float* grad_entropy, const float* grad_top, void* grad_logits, int64_t grad_row_stride, int device, void* hip_stream) {
  if (const char* why = check(dtype, rows, vocab, top)) return keops_seq_fail(-1, why);
  if (rows == 0) return 0;
  if (!logits || !tokens || !entropy || !lse || !grad_logits || (top && !top_index)) return keops_seq_fail(-1, "token log probabilities: null data for the backward pass");
  SeqDevice on(device);
  hipStream_t st = (hipStream_t)hip_stream;
  if (dtype == 0)
    return backward<bf16>(rows, vocab, top, logits, row_stride, tokens, ignore_index, entropy, lse, top_index, grad_logprob, grad_entropy, grad_top, grad_logits, grad_row_stride, st);
  if (dtype == 1)
    return backward<f16>(rows, vocab, top, logits, row_stride, tokens, ignore_index, entropy, lse, top_index, grad_logprob, grad_entropy, grad_top, grad_logits, grad_row_stride, st);
  return backward<float>(rows, vocab, top, logits, row_stride, tokens, ignore_index, entropy, lse, top_index, grad_logprob, grad_entropy, grad_top, grad_logits, grad_row_stride, st);
}

}  // extern "C"
