// Rows of logits x: log probability of a given token, entropy and the largest alternatives in one sweep, and the gradient.
//
// With m = max x, s = sum e^(x-m), t = sum e^(x-m) (x-m):  lse = m + log s,  entropy = log s - t / s.  Both terms of the entropy
// are non-negative, so nothing cancels; x - m is formed before it is scaled, so large logits lose nothing.  m, s and t are kept
// for each thread (a new maximum m' turns t into e^(m-m') (t + s (m-m'))) and joined at the end.
//
// The K largest: a value enters a list in LDS when it exceeds the K-th of what the list last held; the list is cut to its K
// largest when half full.  The first threshold is the K-th largest of the threads' own maxima.  Keys are the value's bits in
// increasing order, then the complement of the index, so equal values keep the lowest index and every key is different: the
// result does not depend on the order in which values arrive.
#include "../../../include/keops_hip.h"
#include "keops_seq.h"

using namespace kseq;

namespace {

constexpr int kThreads = 256, kList = 512, kMaxTop = KEOPS_HIP_MAX_TOP, kUnroll = 4;
constexpr float kLn2 = 0.6931471805599453f;
typedef unsigned long long u64;

struct Stat { float m, s, t; };
__device__ inline Stat join(const Stat& a, const Stat& b) {
  if (a.m == -kInf) return b;
  if (b.m == -kInf) return a;
  const float m = fmaxf(a.m, b.m), da = a.m - m, db = b.m - m;
  const float ea = __builtin_amdgcn_exp2f(da * kLog2e), eb = __builtin_amdgcn_exp2f(db * kLog2e);
  Stat r;
  r.m = m;
  r.s = ea * a.s + eb * b.s;
  // (a factor that has vanished takes its sums with it: s (m - m') may be infinite where logits are near the type's lowest value)
  r.t = (ea == 0.f ? 0.f : ea * (a.t + a.s * da)) + (eb == 0.f ? 0.f : eb * (b.t + b.s * db));
  // a value of +inf or NaN makes the row's sums NaN
  if (!(m < kInf)) r.s = r.t = __builtin_nanf("");
  return r;
}

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

// joins the threads' sums; every thread gets the result
__device__ inline Stat join_all(Stat st, Stat* red, int tid) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor(st.m, o);
    b.s = __shfl_xor(st.s, o);
    b.t = __shfl_xor(st.t, o);
    st = join(st, b);
  }
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = st;
  __syncthreads();
  return join(join(red[0], red[1]), join(red[2], red[3]));
}

// one row, or one share of a row's columns (which then leaves its sums and keys in `part`)
template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_rows(long long vocab, int top, const T* logits, long long stride, const int64_t* tokens, int64_t ignore,
                                                          Out out, int splits, float* part_stat, u64* part_key) {
  constexpr int VE = 16 / (int)sizeof(T), U = kUnroll;
  __shared__ Stat red[4];
  __shared__ u64 list[TOP ? kList : 1], best[TOP ? kMaxTop : 1];
  __shared__ unsigned maxima[TOP ? kThreads : 1], cutoff;
  __shared__ int held;
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / splits;
  const int split = blockIdx.x % splits;
  const T* x = logits + row * stride;
  const long long share = (vocab + splits - 1) / splits, v0 = split * share, v1 = v0 + share < vocab ? v0 + share : vocab;
  const Row r = row_of(x, v0, v1 < v0 ? v0 : v1);
  Stat st = {-kInf, 0.f, 0.f};
  u64 least = 0;  // keys up to this one are not among the largest
  float least_value = -kInf;
  if (TOP && tid == 0) held = 0;

  uint4 next[U];
#pragma unroll
  for (int u = 0; u < U; u++)
    if (tid + u * kThreads < r.count) next[u] = load_vec(x, r, tid + u * kThreads);
  for (int j0 = 0; j0 < r.count; j0 += U * kThreads) {
    uint4 now[U];
#pragma unroll
    for (int u = 0; u < U; u++) now[u] = next[u];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int j = j0 + (U + u) * kThreads + tid;
      if (j < r.count) next[u] = load_vec(x, r, j);
    }
    float vmax[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      vmax[u] = -kInf;
      if (j0 + u * kThreads + tid >= r.count) continue;
      float e[VE];
      unpack<T>(now[u], e);
      float mx = e[0];
      bool nan = e[0] != e[0];
#pragma unroll
      for (int k = 1; k < VE; k++) {
        mx = fmaxf(mx, e[k]);
        nan |= e[k] != e[k];
      }
      if (nan) mx = __builtin_nanf("");
      vmax[u] = mx;
      if (!(mx <= st.m)) {  // a new maximum (or NaN, which stays)
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
          st.t += f == 0.f ? 0.f : f * d;  // -inf adds nothing
        }
      }
    }
    if constexpr (TOP) {
      const auto in_row = [&](int u) { return j0 + u * kThreads + tid < r.count; };
      if (j0 == 0) {
        // K-th largest of the threads' maxima: at least K values reach it
        unsigned mine = 0;
#pragma unroll
        for (int u = 0; u < U; u++)
          if (in_row(u)) mine = max(mine, vmax[u] != vmax[u] ? 0xffffffffu : ordered(vmax[u]));
        maxima[tid] = mine;
        if (tid == 0) cutoff = 0;
        __syncthreads();
        int rank = 0;
        for (int i = 0; i < kThreads; i += 4) {
          const uint4 o = *reinterpret_cast<const uint4*>(maxima + i);
          rank += (o.x > mine || (o.x == mine && i < tid)) + (o.y > mine || (o.y == mine && i + 1 < tid)) + (o.z > mine || (o.z == mine && i + 2 < tid)) +
                  (o.w > mine || (o.w == mine && i + 3 < tid));
        }
        if (rank == top - 1) cutoff = mine;
        __syncthreads();
        least = (u64)cutoff << 32;
        if (cutoff == 0xffffffffu) least = 0;
        least_value = least == 0 ? -kInf : value_of(least);
      }
      unsigned wait = 0;  // elements of this thread that may have to go into the list
#pragma unroll
      for (int u = 0; u < U; u++)
        if (in_row(u) && !(vmax[u] < least_value)) wait |= ((1u << VE) - 1u) << (u * VE);
      for (;;) {
        if (wait) {
#pragma unroll
          for (int u = 0; u < U; u++) {
            if (!(wait >> (u * VE) & ((1u << VE) - 1u))) continue;
            float e[VE];
            unpack<T>(now[u], e);
#pragma unroll
            for (int k = 0; k < VE; k++) {
              if (!(wait >> (u * VE + k) & 1u)) continue;
              const long long i = r.first + (long long)(j0 + u * kThreads + tid) * VE + k;
              const u64 key = key_of(e[k], i);
              bool done = i < r.v0 || i >= r.v1 || key <= least;
              if (!done) {
                const int at = atomicAdd(&held, 1);
                if (at < kList) {
                  list[at] = key;
                  done = true;
                }
              }
              if (done) wait &= ~(1u << (u * VE + k));
            }
          }
        }
        __syncthreads();
        const int n = held;
        const bool full = n > kList, last = j0 + U * kThreads >= r.count;
        __syncthreads();
        if (n > kList / 2 || (last && n > 0)) {
          const int left = cut(list, best, full ? kList : n, top, tid);
          if (tid == 0) held = left;
          if (left == top) {
            least = list[top - 1];
            least_value = value_of(least);
          }
          __syncthreads();
        }
        if (!full) break;
      }
    }
  }
  st = join_all(st, red, tid);
  if (splits == 1) {
    if (tid == 0) finish(out, row, st, x, vocab, tokens[row], ignore);
    if (TOP && tid < top) finish_top(out, row * top + tid, st, list[tid]);
  } else {
    if (tid == 0) {
      float* p = part_stat + (long long)blockIdx.x * 4;
      p[0] = st.m;
      p[1] = st.s;
      p[2] = st.t;
    }
    if (TOP && tid < top) part_key[(long long)blockIdx.x * top + tid] = tid < held ? list[tid] : 0;
  }
}

// the shares of one row
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_join(long long vocab, int top, const T* logits, long long stride, const int64_t* tokens, int64_t ignore,
                                                          Out out, int splits, const float* part_stat, const u64* part_key) {
  __shared__ Stat red[4];
  __shared__ u64 list[kList], best[kMaxTop];
  const int tid = threadIdx.x;
  const long long row = blockIdx.x;
  Stat st = {-kInf, 0.f, 0.f};
  if (tid < splits) {
    const float* p = part_stat + (row * splits + tid) * 4;
    st.m = p[0];
    st.s = p[1];
    st.t = p[2];
  }
  st = join_all(st, red, tid);
  if (tid == 0) finish(out, row, st, logits + row * stride, vocab, tokens[row], ignore);
  if (top == 0) return;
  const u64* keys = part_key + row * splits * top;
  const int all = splits * top;
  int n = 0;
  for (int at = 0; at < all;) {  // the list holds the largest so far and as many more as there is room for
    const int take = min(kList - n, all - at);
    __syncthreads();
    for (int i = tid; i < take; i += kThreads) list[n + i] = keys[at + i];
    at += take;
    n = cut(list, best, n + take, top, tid);
  }
  if (tid < top) finish_top(out, row * top + tid, st, list[tid]);
}

// dx = -p (a + c (x - lse + entropy)), a = sum of the incoming gradients of this row's log probabilities, c = that of the
// entropy; the tokens whose log probabilities were returned get theirs added.  One read and one write; the few given tokens are
// written again by threads of the workgroup that has their columns, behind a barrier.
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

// Shares of a row: enough workgroups for four on every CU, at least 4096 columns to a share.
int splits_of(int64_t rows, int64_t vocab) {
  if (rows < 1) return 1;
  int64_t s = 1024 / rows, most = vocab / 4096;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

template <class T>
int forward(int64_t rows, int64_t vocab, int top, const void* logits, int64_t stride, const int64_t* tokens, int64_t ignore, const Out& out, void* work, hipStream_t st) {
  const int splits = splits_of(rows, vocab);
  u64* keys = (u64*)work;
  float* stats = (float*)(keys + (size_t)rows * splits * top);
  const unsigned grid = (unsigned)(rows * splits);
  if (top)
    logprobs_rows<T, true><<<grid, kThreads, 0, st>>>(vocab, top, (const T*)logits, stride, tokens, ignore, out, splits, stats, keys);
  else
    logprobs_rows<T, false><<<grid, kThreads, 0, st>>>(vocab, top, (const T*)logits, stride, tokens, ignore, out, splits, stats, keys);
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
