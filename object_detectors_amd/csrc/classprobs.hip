// Log probabilities of given classes, entropy and the best alternatives of rows of class values, for gfx950.
//
// The reference keeps one score per detection (object_detectors/yolov8_lmi/model.py:223-232, the row NMS emits); the
// rows read here are the ones that score came from: class planes of the head (B, 4+nc+nm, A) at the anchors NMS
// kept, the distance bins behind every box side, or plain rows of a classifier.
//
// Mathematics, one pass over a row: m = max x, s = sum e^(x-m), t = sum e^(x-m)(x-m), kept up to date as m grows
// (s *= e^(m-m'), t = (t + s(m-m')) e^(m-m')); then log Z = m + log s and H = log s - t/s.  s and t are sums of at most
// some hundred terms per lane, added up over the lanes in fp32; values are fp32 whatever the input type.
// The alternatives are ordered by a 64-bit key: the value's bits made monotonic above, the complemented class below, so
// that equal values fall in class order and no two keys are equal (the result does not depend on the order of atomics).
//
// Kernels
//  evidence_rows_kernel    one workgroup of NT threads per row (and per part of a long row): each thread holds J*V values
//                          in registers, so a row is read once.  The best `top`: the top-th best of the 64 per-lane
//                          maxima is a lower bound of the answer; what reaches it (a few dozen of thousands) goes to
//                          LDS and is ranked there by counting.
//  evidence_join_kernel    joins the parts of long rows.
//  evidence_planes_kernel  one thread per row, for rows that lie side by side (class planes): a wave reads 64
//                          neighbouring rows' values of one class at a time; the alternatives sit in registers.
#include <hip/hip_fp16.h>

#include "common.h"

namespace {

struct Evidence {
  const void *x;
  long long classes, cs, n0, n1, s0, s1;
  const int *index;
  long long index_range;
  const int *count;
  const void *labels;
  long long l0, l1;
  int label_dtype, top;
  float *logprob, *entropy, *top_logprob;
  int *top_index;
  unsigned char *ws;
  int parts;           // parts per row (rows kernel)
  long long part_len;  // classes per part
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxTop = LMI_MAX_TOP;

__device__ __forceinline__ float exp_fast(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// monotonic bits: larger value -> larger number; -0 = +0; NaN above everything; never 0
__device__ __forceinline__ unsigned order_bits(float v) {
  unsigned b = __float_as_uint(v + 0.0f);
  b = v != v ? 0x7fffffffu : b;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
typedef unsigned long long u64;
__device__ __forceinline__ u64 make_key(unsigned o, unsigned c) { return ((u64)o << 32) | (0xffffffffu - c); }
__device__ __forceinline__ unsigned key_class(u64 k) { return 0xffffffffu - (unsigned)k; }

// entropy of one yes / no answer
__device__ __forceinline__ float answer_entropy_sigmoid(float x) {
  const float a = fabsf(x), e = exp_fast(-a);
  return log1pf(e) + (e > 0.0f ? a * e / (1.0f + e) : e);   // a infinite: e = 0 and both terms are 0; NaN stays
}
__device__ __forceinline__ float answer_entropy_none(float p) {
  const float a = p == 0.0f ? 0.0f : p * logf(p);
  const float b = p == 1.0f ? 0.0f : (1.0f - p) * log1pf(-p);
  return -a - b;
}
template <int ACT> __device__ __forceinline__ float answer_entropy(float x) {
  return ACT == LMI_PROB_SIGMOID ? answer_entropy_sigmoid(x) : answer_entropy_none(x);
}
// log probability of value x; softmax: m = the reference the row's sums use, log_s = log of the sum
template <int ACT> __device__ __forceinline__ float log_prob(float x, float m, float log_s) {
  if (ACT == LMI_PROB_SOFTMAX) return (x - m) - log_s;
  if (ACT == LMI_PROB_SIGMOID) return fminf(x, 0.0f) - log1pf(expf(-fabsf(x))) + (x != x ? x : 0.0f);   // fminf drops a NaN
  return logf(x);
}

// running sums of a softmax row with respect to m
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// the same sums with respect to m2 >= m
__device__ __forceinline__ void rebase(Sums &a, float m2) {
  if (a.m == m2) return;
  if (a.m == -INFINITY) {   // nothing but -inf so far (or a NaN that already sits in s)
    a.t = a.s;              // 0, or the NaN
  } else {
    const float d = a.m - m2, f = exp_fast(d);
    a.t = (a.t + a.s * fmaxf(d, -200.0f)) * f;
    a.s *= f;
  }
  a.m = m2;
}
__device__ __forceinline__ void add_value(Sums &a, float ref, float x) {
  const float z = x - ref, e = exp_fast(z);
  a.s += e;
  a.t = fmaf(e, fmaxf(z, -200.0f), a.t);   // e is 0 long before z = -200
}
__device__ __forceinline__ void softmax_result(const Sums &a, float &ref, float &log_s, float &h) {
  ref = finite_ref(a.m);
  if (a.s == 0.0f) {   // every value -inf
    log_s = 0.0f;
    h = 0.0f;
  } else {
    log_s = logf(a.s);
    h = log_s - a.t / a.s;
  }
}

__device__ __forceinline__ long long label_of(const Evidence &E, long long o, long long i) {
  const long long at = o * E.l0 + i * E.l1;
  if (E.label_dtype == LMI_I64) return ((const long long *)E.labels)[at];
  if (E.label_dtype == LMI_I32) return ((const int *)E.labels)[at];
  const float f = ((const float *)E.labels)[at];
  return (f >= 0.0f && f < 9.0e15f) ? (long long)f : -1;   // NaN -> -1
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ u64 wave_max_key(u64 v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const u64 w = __shfl_xor(v, d);
    v = w > v ? w : v;
  }
  return v;
}

// the best `top` keys of the workgroup's registers and of the list kept so far -> list (LDS, descending)
constexpr int kCand = 256;
template <int NT> struct TopShared {
  u64 lane_best[NT / 64][64];
  u64 cand[kCand + kMaxTop];
  u64 list[kMaxTop];
  u64 threshold;
  int n;
};
template <int NT, int N, typename Key>
__device__ __forceinline__ void merge_top(TopShared<NT> &L, Key key, int top) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  u64 best = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const u64 k = key(e);
    best = k > best ? k : best;
  }
  L.lane_best[wave][lane] = best;
  if (t == 0) L.n = 0;
  __syncthreads();
  if (wave == 0) {   // the top-th best of 64 lane maxima bounds the top-th best of all values from below
    u64 k = best;
    for (int w = 1; w < NT / 64; ++w) k = L.lane_best[w][lane] > k ? L.lane_best[w][lane] : k;
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < 64; ++j) rank += __shfl(k, j) > k;
    if (rank == top - 1 && k) L.threshold = k;   // keys are distinct unless 0: at most one lane
    if (lane == 0) {
      const u64 any = __ballot(rank == top - 1 && k != 0);
      if (!any) L.threshold = 1;                 // fewer than `top` lanes hold a value: everything is a candidate
    }
  }
  __syncthreads();
  u64 thr = L.threshold;
  const u64 kept = L.list[top - 1];
  thr = kept > thr ? kept : thr;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const u64 k = key(e);
    if (k >= thr) {
      const int at = atomicAdd(&L.n, 1);
      if (at < kCand) L.cand[at] = k;
    }
  }
  __syncthreads();
  int n = L.n;
  if (n <= kCand) {
    if (t < top) L.cand[n + t] = L.list[t];
    __syncthreads();
    n += top;
    if (t < top) L.list[t] = 0;
    __syncthreads();
    for (int i = t; i < n; i += NT) {
      const u64 k = L.cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += L.cand[j] > k;
      if (rank < top && k) L.list[rank] = k;
    }
    __syncthreads();
    return;
  }
  // more candidates than the table holds (values arranged so that few lanes own nearly all of the best): `top` rounds, each
  // taking the best key below the last one
  if (t < top) L.cand[t] = L.list[t];
  __syncthreads();
  u64 last = ~0ull;
  for (int r = 0; r < top; ++r) {
    u64 b = (t < top && L.cand[t] < last) ? L.cand[t] : 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const u64 k = key(e);
      if (k < last && k > b) b = k;
    }
    b = wave_max_key(b);
    if (lane == 0) L.lane_best[wave][0] = b;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) b = L.lane_best[w][0] > b ? L.lane_best[w][0] : b;
    if (t == 0) L.list[r] = b;
    __syncthreads();
    last = b;
  }
}

template <int ACT>
__device__ void store_row(const Evidence &E, long long row, float ref, float log_s, float h, bool has_label, float label_x,
                          const u64 *list, int lane) {
  if (lane == 0) {
    if (E.entropy) E.entropy[row] = h;
    if (E.logprob) E.logprob[row] = has_label ? log_prob<ACT>(label_x, ref, log_s) : NAN;
  }
  if (lane < E.top) {
    const u64 k = list[lane];
    if (E.top_logprob) E.top_logprob[row * E.top + lane] = log_prob<ACT>(order_value((unsigned)(k >> 32)), ref, log_s);
    if (E.top_index) E.top_index[row * E.top + lane] = (int)key_class(k);
  }
}

struct alignas(16) PartHead {
  float m, s, t, pad;
};

template <typename T, int V> struct Pack {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T> struct Pack<T, 1> {
  typedef T type;
};

// V > 1: classes lie side by side and are read in aligned 16-byte groups (the row may start anywhere; the groups at its two ends
// are read value by value).  V == 1: any class stride.
template <typename T, int NT, int J, int V, int ACT>
__device__ __forceinline__ void evidence_row(const Evidence &E, long long row, TopShared<NT> &L, float (&red)[NT / 64][4]) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long long o = row / E.n1, m = row - o * E.n1;
  if (E.count && m >= E.count[o]) return;
  long long i = m;
  if (E.index) {
    i = E.index[row];
    if (i < 0 || i >= E.index_range) {
      if (t == 0 && E.entropy) E.entropy[row] = NAN;
      if (t == 0 && E.logprob) E.logprob[row] = NAN;
      if (t < E.top && E.top_logprob) E.top_logprob[row * E.top + t] = NAN;
      if (t < E.top && E.top_index) E.top_index[row * E.top + t] = -1;
      return;
    }
  }
  const T *x = (const T *)E.x + o * E.s0 + i * E.s1;
  const long long c0 = (long long)blockIdx.y * E.part_len;
  const long long c1 = c0 + E.part_len < E.classes ? c0 + E.part_len : E.classes;
  long long start = c0;
  if (V > 1) start -= (long long)(((uintptr_t)(x + c0) & 15) / sizeof(T));

  if (t < kMaxTop) L.list[t] = 0;
  Sums S = {-INFINITY, 0.0f, 0.0f};   // softmax: sums with respect to the workgroup's m; else t = the entropy
  constexpr int N = J * V;
  for (long long tile = start; tile < c1; tile += (long long)NT * N) {
    float v[N];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const long long e0 = tile + ((long long)j * NT + t) * V;
      if (V > 1 && e0 >= c0 && e0 + V <= c1) {
        typedef typename Pack<T, V>::type P;
        const P p = *(const P *)(x + e0);
#pragma unroll
        for (int u = 0; u < V; ++u) v[j * V + u] = to_float(((const T *)&p)[u]);
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const long long c = e0 + u;
          v[j * V + u] = c >= c0 && c < c1 ? to_float(x[c * (V > 1 ? 1 : E.cs)]) : (ACT == LMI_PROB_NONE ? 0.0f : -INFINITY);
        }
      }
    }
    if (ACT == LMI_PROB_SOFTMAX) {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < N; ++e) mx = fmaxf(mx, v[e]);
      mx = wave_max(mx);
      if (NT > 64) {
        if (lane == 0) red[wave][0] = mx;
        __syncthreads();
        for (int w = 0; w < NT / 64; ++w) mx = fmaxf(mx, red[w][0]);
      }
      rebase(S, fmaxf(S.m, mx));
      const float ref = finite_ref(S.m);
#pragma unroll
      for (int e = 0; e < N; ++e) add_value(S, ref, v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) S.t += answer_entropy<ACT>(v[e]);
    }
    if (E.top) {
      const long long first = tile + (long long)t * V;
      merge_top<NT, N>(L, [&](int e) -> u64 {
        const long long c = first + (e / V) * (NT * V) + e % V;
        return c >= c0 && c < c1 ? make_key(order_bits(v[e]), (unsigned)c) : 0;
      }, E.top);
    } else if (NT > 64 && ACT == LMI_PROB_SOFTMAX) {
      __syncthreads();   // red[][0] is written again by the next tile
    }
  }
  // sums over the workgroup
  S.s = wave_sum(S.s);
  S.t = wave_sum(S.t);
  if (NT > 64) {
    if (lane == 0) {
      red[wave][1] = S.s;
      red[wave][2] = S.t;
    }
    __syncthreads();
    S.s = S.t = 0.0f;
    for (int w = 0; w < NT / 64; ++w) {
      S.s += red[w][1];
      S.t += red[w][2];
    }
  }
  if (wave) return;
  if (E.parts > 1) {
    unsigned char *out = E.ws + (row * E.parts + blockIdx.y) * (sizeof(PartHead) + (long long)kMaxTop * 8);
    if (lane == 0) *(PartHead *)out = PartHead{S.m, S.s, S.t, 0.0f};
    if (lane < E.top) ((u64 *)(out + sizeof(PartHead)))[lane] = L.list[lane];
    return;
  }
  float ref = 0.0f, log_s = 0.0f, h = S.t;
  if (ACT == LMI_PROB_SOFTMAX) softmax_result(S, ref, log_s, h);
  bool has = false;
  float lx = 0.0f;
  if (E.labels && lane == 0) {
    const long long l = label_of(E, o, m);
    has = l >= 0 && l < E.classes;
    if (has) lx = to_float(x[l * E.cs]);
  }
  store_row<ACT>(E, row, ref, log_s, h, has, lx, L.list, lane);
}

template <typename T, int NT, int J, int V, int ACT>
__global__ __launch_bounds__(NT) void evidence_rows_kernel(const Evidence E) {
  __shared__ TopShared<NT> L;
  __shared__ float red[NT / 64][4];
  for (long long row = blockIdx.x; row < E.n0 * E.n1; row += gridDim.x) {   // more rows than a grid holds: several each
    evidence_row<T, NT, J, V, ACT>(E, row, L, red);
    __syncthreads();
  }
}

// one wave per row: lane p holds part p (at most 64), whose list is sorted
template <typename T, int ACT>
__global__ __launch_bounds__(64) void evidence_join_kernel(const Evidence E) {
  __shared__ u64 list[kMaxTop];
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;   // fewer than 128 of them
  const long long o = row / E.n1, m = row - o * E.n1;
  if (E.count && m >= E.count[o]) return;
  const long long i = E.index ? E.index[row] : m;
  if (E.index && (i < 0 || i >= E.index_range)) return;   // written by the parts
  const unsigned char *in = E.ws + (row * E.parts + lane) * (sizeof(PartHead) + (long long)kMaxTop * 8);
  const bool live = lane < E.parts;
  Sums S = {-INFINITY, 0.0f, 0.0f};
  if (live) {
    const PartHead p = *(const PartHead *)in;
    S = Sums{p.m, p.s, p.t};
  }
  float ref = 0.0f, log_s = 0.0f, h;
  if (ACT == LMI_PROB_SOFTMAX) {
    rebase(S, wave_max(S.m));
    S.s = wave_sum(S.s);
    S.t = wave_sum(S.t);
    softmax_result(S, ref, log_s, h);
  } else {
    h = wave_sum(S.t);
  }
  const u64 *keys = (const u64 *)(in + sizeof(PartHead));
  int at = 0;
  u64 head = live && E.top ? keys[0] : 0;
  for (int r = 0; r < E.top; ++r) {
    const u64 b = wave_max_key(head);
    if (lane == 0) list[r] = b;
    if (live && head == b) {
      ++at;
      head = at < E.top ? keys[at] : 0;
    }
  }
  __syncthreads();
  bool has = false;
  float lx = 0.0f;
  if (E.labels && lane == 0) {
    const long long l = label_of(E, o, m);
    has = l >= 0 && l < E.classes;
    if (has) lx = to_float(((const T *)E.x)[o * E.s0 + i * E.s1 + l * E.cs]);
  }
  store_row<ACT>(E, row, ref, log_s, h, has, lx, list, lane);
}

template <typename T, int ACT, int KT>
__global__ __launch_bounds__(256) void evidence_planes_kernel(const Evidence E) {
  const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
  if (row >= E.n0 * E.n1) return;
  const long long o = row / E.n1, i = row - o * E.n1;
  if (E.count && i >= E.count[o]) return;
  const T *x = (const T *)E.x + o * E.s0 + i * E.s1;
  Sums S = {-INFINITY, 0.0f, 0.0f};
  unsigned ord[KT ? KT : 1];
  int cls[KT ? KT : 1];
#pragma unroll
  for (int k = 0; k < KT; ++k) ord[k] = 0, cls[k] = -1;
  constexpr int U = 8;
  const int C = (int)E.classes;
  for (int c = 0; c < C; c += U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = c + u < C ? to_float(x[(long long)(c + u) * E.cs]) : (ACT == LMI_PROB_NONE ? 0.0f : -INFINITY);
    if (ACT == LMI_PROB_SOFTMAX) {
      float mx = S.m;
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, v[u]);
      rebase(S, mx);
      const float ref = finite_ref(mx);
#pragma unroll
      for (int u = 0; u < U; ++u) add_value(S, ref, v[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) S.t += answer_entropy<ACT>(v[u]);
    }
    if (KT) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        unsigned q = c + u < C ? order_bits(v[u]) : 0u;
        int qc = c + u;
        if (q > ord[KT ? KT - 1 : 0]) {   // strictly better than the last kept one: equal values stay in class order
          bool up = false;                // from its place on, everything moves down by one
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            up = up || q > ord[k];
            const unsigned a = ord[k];
            const int b = cls[k];
            ord[k] = up ? q : a;
            cls[k] = up ? qc : b;
            q = up ? a : q;
            qc = up ? b : qc;
          }
        }
      }
    }
  }
  float ref = 0.0f, log_s = 0.0f, h = S.t;
  if (ACT == LMI_PROB_SOFTMAX) softmax_result(S, ref, log_s, h);
  if (E.entropy) E.entropy[row] = h;
  if (E.logprob) {
    float lp = NAN;
    if (E.labels) {
      const long long l = label_of(E, o, i);
      if (l >= 0 && l < C) lp = log_prob<ACT>(to_float(x[l * E.cs]), ref, log_s);
    }
    E.logprob[row] = lp;
  }
#pragma unroll
  for (int k = 0; k < KT; ++k)
    if (k < E.top) {
      if (E.top_logprob) E.top_logprob[row * E.top + k] = log_prob<ACT>(order_value(ord[k]), ref, log_s);
      if (E.top_index) E.top_index[row * E.top + k] = cls[k];
    }
}

// parts per row: long rows of a batch too small to fill the chip are cut into parts of at least 4096 values, at most 64 (one
// per lane of the joining wave)
int split_parts(long long rows, long long classes) {
  if (rows >= 128 || classes <= 8192) return 1;
  const long long p = (classes + 4095) / 4096;
  return (int)(p < 64 ? p : 64);
}

template <typename T, int ACT> int launch(const Evidence &E0, hipStream_t st) {
  Evidence E = E0;
  const long long rows = E.n0 * E.n1;
  // rows side by side and few classes each, or many rows: a thread per row
  const bool planes = !E.index && E.classes <= 65536 && ((E.cs != 1 && E.s1 < E.cs && (rows >= 4096 || E.classes <= 64)) || E.classes <= 8);
  if (planes) {
    const dim3 g((unsigned)((rows + 255) / 256));
    if (E.top == 0) evidence_planes_kernel<T, ACT, 0><<<g, 256, 0, st>>>(E);
    else if (E.top <= 2) evidence_planes_kernel<T, ACT, 2><<<g, 256, 0, st>>>(E);
    else if (E.top <= 8) evidence_planes_kernel<T, ACT, 8><<<g, 256, 0, st>>>(E);
    else evidence_planes_kernel<T, ACT, 32><<<g, 256, 0, st>>>(E);
    return lmi_check_launch("lmi_class_logprobs");
  }
  E.parts = split_parts(rows, E.classes);
  E.part_len = (E.classes + E.parts - 1) / E.parts;
  const dim3 g((unsigned)(rows < (1 << 22) ? rows : (1 << 22)), (unsigned)E.parts);   // grid x workgroup size stays below 2^32
  constexpr int V = 16 / sizeof(T);
  if (E.cs == 1) {
    if (E.part_len <= 1024 - V) evidence_rows_kernel<T, 64, 16 / V, V, ACT><<<g, 64, 0, st>>>(E);
    else if (E.part_len <= 8192 || E.parts > 1) evidence_rows_kernel<T, 256, 16 / V, V, ACT><<<g, 256, 0, st>>>(E);
    else evidence_rows_kernel<T, 512, 32 / V, V, ACT><<<g, 512, 0, st>>>(E);
  } else {
    if (E.part_len <= 128) evidence_rows_kernel<T, 64, 2, 1, ACT><<<g, 64, 0, st>>>(E);
    else evidence_rows_kernel<T, 256, 8, 1, ACT><<<g, 256, 0, st>>>(E);
  }
  if (E.parts > 1) evidence_join_kernel<T, ACT><<<(unsigned)rows, 64, 0, st>>>(E);
  return lmi_check_launch("lmi_class_logprobs");
}

template <typename T> int launch_act(const Evidence &E, int act, hipStream_t st) {
  if (act == LMI_PROB_SOFTMAX) return launch<T, LMI_PROB_SOFTMAX>(E, st);
  if (act == LMI_PROB_SIGMOID) return launch<T, LMI_PROB_SIGMOID>(E, st);
  return launch<T, LMI_PROB_NONE>(E, st);
}

}  // namespace

extern "C" {

int64_t lmi_class_logprobs_workspace_bytes(int64_t rows, int64_t classes, int64_t class_stride, int top) {
  (void)class_stride;
  (void)top;
  if (rows <= 0 || classes <= 0) return 0;
  const int parts = split_parts(rows, classes);
  return parts > 1 ? rows * parts * (int64_t)(sizeof(PartHead) + kMaxTop * 8) : 0;
}

int lmi_class_logprobs(const lmi_logprob_args *a, void *stream) {
  LMI_REQUIRE(a != nullptr, LMI_ERR_BAD_ARG, "lmi_class_logprobs: args is NULL");
  LMI_REQUIRE(a->n0 >= 0 && a->n1 >= 0 && a->classes > 0, LMI_ERR_BAD_ARG, "lmi_class_logprobs: sizes (%lld, %lld) rows of %lld classes",
              (long long)a->n0, (long long)a->n1, (long long)a->classes);
  LMI_REQUIRE(a->activation >= LMI_PROB_SOFTMAX && a->activation <= LMI_PROB_NONE, LMI_ERR_BAD_ARG, "lmi_class_logprobs: unknown activation %d",
              a->activation);
  LMI_REQUIRE(a->top >= 0 && a->top <= LMI_MAX_TOP && a->top <= a->classes, LMI_ERR_BAD_ARG,
              "lmi_class_logprobs: top %d must lie in 0..min(%lld classes, %d)", a->top, (long long)a->classes, LMI_MAX_TOP);
  LMI_REQUIRE(a->classes < (1ll << 31) && a->n0 < (1ll << 31) && a->n1 < (1ll << 31) && a->n0 * a->n1 < (1ll << 31), LMI_ERR_LIMIT,
              "lmi_class_logprobs: rows and classes must each stay below 2^31");
  if (a->n0 == 0 || a->n1 == 0) return LMI_OK;
  LMI_REQUIRE(a->x != nullptr, LMI_ERR_BAD_ARG, "lmi_class_logprobs: x is NULL");
  LMI_REQUIRE(a->class_stride > 0 && a->stride0 >= 0 && a->stride1 >= 0, LMI_ERR_BAD_ARG, "lmi_class_logprobs: negative or zero stride");
  LMI_REQUIRE(!a->labels || (a->label_dtype == LMI_F32 || a->label_dtype == LMI_I32 || a->label_dtype == LMI_I64), LMI_ERR_BAD_ARG,
              "lmi_class_logprobs: labels must be fp32, int32 or int64");
  LMI_REQUIRE(!a->index || a->index_range > 0, LMI_ERR_BAD_ARG, "lmi_class_logprobs: index without a range");
  const int64_t need = lmi_class_logprobs_workspace_bytes(a->n0 * a->n1, a->classes, a->class_stride, a->top);
  LMI_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need), LMI_ERR_WORKSPACE,
              "lmi_class_logprobs: workspace of %lld bytes, %lld needed", (long long)a->workspace_bytes, (long long)need);
  LMI_REQUIRE(need == 0 || lmi_is_aligned(a->workspace, 16), LMI_ERR_ALIGNMENT, "lmi_class_logprobs: workspace must be 16-byte aligned");
  Evidence E;
  E.x = a->x;
  E.classes = a->classes;
  E.cs = a->class_stride;
  E.n0 = a->n0;
  E.n1 = a->n1;
  E.s0 = a->stride0;
  E.s1 = a->stride1;
  E.index = a->index;
  E.index_range = a->index_range;
  E.count = a->count;
  E.labels = a->labels;
  E.l0 = a->label_stride0;
  E.l1 = a->label_stride1;
  E.label_dtype = a->label_dtype;
  E.top = a->top;
  E.logprob = a->logprob;
  E.entropy = a->entropy;
  E.top_logprob = a->top_logprob;
  E.top_index = a->top_index;
  E.ws = (unsigned char *)a->workspace;
  E.parts = 1;
  E.part_len = a->classes;
  hipStream_t st = (hipStream_t)stream;
  if (a->x_dtype == LMI_F32) return launch_act<float>(E, a->activation, st);
  if (a->x_dtype == LMI_F16) return launch_act<_Float16>(E, a->activation, st);
  if (a->x_dtype == LMI_BF16) return launch_act<__bf16>(E, a->activation, st);
  lmi_set_error("lmi_class_logprobs: x must be fp32, fp16 or bf16");
  return LMI_ERR_BAD_ARG;
}

}  // extern "C"
