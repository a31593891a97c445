// Log probabilities of given classes, entropy and the best alternatives of rows of class values, for gfx950.
//
// The reference keeps one score per detection (object_detectors/yolov8_lmi/model.py:223-232, the row NMS emits); the
// rows read here are the ones that score came from: class planes of the head (B, 4+nc+nm, A) at the anchors NMS
// kept, the distance bins behind every box side, or plain rows of a classifier.
//
// Mathematics, one pass over a row: m = max x, s = sum e^(x-m), t = sum e^(x-m)(x-m), kept up to date as m grows
// (s *= e^(m-m'), t = (t + s(m-m')) e^(m-m')); then log Z = m + log s and H = log s - t/s.  Values and sums are fp32 whatever the input type.
// A lane adds up at most 64 terms one after another; where it has more, the sums of such groups are added, and small steps of m applied, with
// what each addition loses carried along, since a long sum of like terms rounds all of them the same way (30011 classes in a thread one by
// one: log s 3e-4 off, an entropy of 16000 by 4; by groups within the bound of a sum of 64 terms, for any length).
// The alternatives are ordered by a 64-bit key: the value's bits made monotonic above, the complemented class below, so
// that equal values fall in class order and no two keys are equal (the result does not depend on the order of atomics).
//
// Kernels
//  evidence_team_kernel    16 lanes per row (a DPP row), up to 128 classes in registers: NMS rows (classes an anchor plane apart, so every
//                          value is a sector of its own: bound by their latency, many rows in flight) and small rows.  The best are
//                          taken one by one: a maximum over the 16 lanes, a ballot for its lowest class.
//  evidence_rows_kernel    a wave (four rows per workgroup) or a workgroup per row, or per part of a long row; 128 bytes of the row per
//                          thread in registers, so that a row is read once and 64 KB of it are in flight.  The top-th best of the 64
//                          lane maxima is a lower bound of the answer; what reaches it (a few dozen of thousands) goes to LDS and
//                          is ranked there by counting.
//  evidence_join_kernel    joins the parts of long rows, the same way.
//  evidence_planes_kernel  one thread per row, for many rows that lie side by side (class planes); the alternatives sit in registers.
#include <hip/hip_fp16.h>

#include <type_traits>

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
  int pairs;           // a row's two alternatives may be written as one word (planes kernel)
  int parts;           // parts per row (rows kernel)
  long long part_len;  // classes per part
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxTop = LMI_MAX_TOP;

__device__ __forceinline__ float exp_fast(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// monotonic bits: larger value -> larger number; -0 = +0; NaN above everything; never 0, never all ones (no key is ~0, from which the rounds start)
__device__ __forceinline__ unsigned order_bits(float v) {
  unsigned b = __float_as_uint(v + 0.0f);
  b = v != v ? 0x7ffffffeu : b;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
typedef unsigned long long u64;
__device__ __forceinline__ u64 make_key(unsigned o, unsigned c) { return ((u64)o << 32) | (0xffffffffu - c); }
__device__ __forceinline__ unsigned key_class(u64 k) { return 0xffffffffu - (unsigned)k; }

// log(1 + d) for -1 <= d <= 1: the logarithm of u = 1 + d rounded, and what the rounding took ((d - (u - 1)) / u, where the division by u in
// [0.5, 2] changes less than half an ulp of the result; below 0.5 nothing was lost)
__device__ __forceinline__ float log_1_plus(float d) {
  const float u = 1.0f + d;
  return fmaf(__builtin_amdgcn_logf(u), 0.6931471805599453f, d - (u - 1.0f));
}
// entropy of one yes / no answer
__device__ __forceinline__ float answer_entropy_sigmoid(float x) {
  const float a = fabsf(x), e = exp_fast(-a);
  return log_1_plus(e) + (e > 0.0f ? a * e * __builtin_amdgcn_rcpf(1.0f + e) : e);   // a infinite: e = 0 and both terms are 0; NaN stays
}
__device__ __forceinline__ float answer_entropy_none(float p) {
  const float a = p == 0.0f ? 0.0f : p * logf(p);
  const float b = p == 1.0f ? 0.0f : (1.0f - p) * log_1_plus(-p);
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
// A row's sums over many groups of values: what each addition loses (Kahan) is carried along.
struct LongSums {
  Sums a = {-INFINITY, 0.0f, 0.0f};
  float lost_s = 0.0f, lost_t = 0.0f;
  __device__ static __forceinline__ void add(float &sum, float &lost, float v) {
    const float y = v - lost, n = sum + y;
    lost = (n - sum) - y;
    sum = n;
  }
  // a group's sums, with respect to g.m >= m
  __device__ __forceinline__ void add(const Sums &g) {
    if (a.m != g.m) {
      const float d = a.m - g.m;
      if (d > -0.25f) {   // a row that climbs slowly takes thousands of such steps: s += s(e^d - 1), e^d - 1 by its series, likewise t
        const float r = d * fmaf(d, fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.0f / 720, 1.0f / 120), 1.0f / 24), 1.0f / 6), 0.5f), 1.0f);
        add(a.t, lost_t, fmaf(a.t, r, a.s * d * (1.0f + r)));
        add(a.s, lost_s, a.s * r);
        a.m = g.m;
      } else {            // what came before fades with every such step
        const float f = a.m == -INFINITY ? 1.0f : exp_fast(d);
        lost_s *= f;
        lost_t *= f;
        rebase(a, g.m);
      }
    }
    add(a.s, lost_s, g.s);
    add(a.t, lost_t, g.t);
  }
  __device__ __forceinline__ void add_entropy(float h) { add(a.t, lost_t, h); }
};
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
    log_s = __builtin_amdgcn_logf(a.s) * 0.6931471805599453f;   // s lies in [1, classes]
    h = fmaf(-a.t, __builtin_amdgcn_rcpf(a.s), log_s);
  }
}

__device__ __forceinline__ long long label_of(const Evidence &E, long long o, long long i) {
  const long long at = o * E.l0 + i * E.l1;
  if (E.label_dtype == LMI_I64) return ((const long long *)E.labels)[at];
  if (E.label_dtype == LMI_I32) return ((const int *)E.labels)[at];
  const float f = ((const float *)E.labels)[at];
  return (f >= 0.0f && f < 9.0e15f) ? (long long)f : -1;   // NaN -> -1
}

// reductions on the data-parallel primitives: within 16 lanes, then across the wave; every lane gets the result
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false); }
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;   // quad_perm [1,0,3,2], [2,3,0,1]; mirror of 8 and of 16 lanes
template <typename F> __device__ __forceinline__ unsigned reduce16(unsigned v, F f) {
  v = f(v, dpp<kXor1>(v));
  v = f(v, dpp<kXor2>(v));
  v = f(v, dpp<kHalfMirror>(v));
  return f(v, dpp<kMirror>(v));
}
struct MaxF {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
};
struct MinF {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b))); }
};
struct SumF {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }
};
struct MaxU {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return a > b ? a : b; }
};
template <typename F> __device__ __forceinline__ float reduce64(float x, F f) {
  unsigned v = reduce16(__float_as_uint(x), f);
  const unsigned a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16), c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return __uint_as_float(f(f(a, b), f(c, d)));
}

// NT threads share a row: one wave (several of them per workgroup, each on its own) or the workgroup
template <int NT> __device__ __forceinline__ void team_sync() {
  if (NT == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

constexpr int kCand = 256;
template <int NT> struct TeamShared {
  float lane_max[NT / 64][64];
  float red[NT / 64][3];
  u64 best[NT / 64];
  u64 cand[kCand + kMaxTop];
  u64 list[kMaxTop];   // the best so far, descending
  float threshold;
  int n;
};

// the top-th largest of the wave's 64 values (rank by counting; equal values share a rank)
__device__ __forceinline__ float kth_of_lanes(float v, int top) {
  int above = 0;
#pragma unroll 16
  for (int j = 0; j < 64; ++j) above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), j)) > v;
  return reduce64(above < top ? v : INFINITY, MinF());
}

// the `top` best of the table's n keys and the list -> list
template <int NT> __device__ __forceinline__ void rank_candidates(TeamShared<NT> &L, int n, int t, int top) {
  if (t < top) L.cand[n + t] = L.list[t];
  team_sync<NT>();
  n += top;
  if (t < top) L.list[t] = 0;
  team_sync<NT>();
  for (int i = t; i < n; i += NT) {
    const u64 k = L.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += L.cand[j] > k;
    if (rank < top && k) L.list[rank] = k;   // keys are distinct unless 0
  }
  team_sync<NT>();
}

__device__ __forceinline__ u64 wave_max_key(u64 v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const u64 w = __shfl_xor(v, d);
    v = w > v ? w : v;
  }
  return v;
}

// More candidates than the table holds (equal values, or values arranged so that few lanes own nearly all of the best): `top` rounds,
// each taking the best key below the last one from key(0) .. key(n - 1), read again.
template <int NT, typename Key> __device__ __forceinline__ void top_by_rounds(TeamShared<NT> &L, Key key, int n, int t, int top) {
  const int lane = t & 63, wave = t >> 6;
  if (t < top) L.cand[t] = L.list[t];
  team_sync<NT>();
  u64 last = ~0ull;
  for (int r = 0; r < top; ++r) {
    u64 b = (t < top && L.cand[t] < last) ? L.cand[t] : 0;
    for (int e = t; e < n; e += NT) {
      const u64 k = key(e);
      if (k < last && k > b) b = k;
    }
    b = wave_max_key(b);
    if (lane == 0) L.best[wave] = b;
    team_sync<NT>();
    for (int w = 0; w < NT / 64; ++w) b = L.best[w] > b ? L.best[w] : b;
    if (t == 0) L.list[r] = b;
    team_sync<NT>();
    last = b;
  }
}

// The values in `p` as if just loaded: what was computed from them is not kept in registers beside them.
template <typename P, int J> __device__ __forceinline__ void forget(P (&p)[J]) {
#pragma unroll
  for (int j = 0; j < J; ++j) asm volatile("" : "+v"(p[j]));
}

template <int ACT>
__device__ __forceinline__ void store_row(const Evidence &E, long long row, float ref, float log_s, float h, bool has_label, float label_x,
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

__device__ __forceinline__ void store_nan(const Evidence &E, long long row, int t) {
  if (t == 0 && E.entropy) E.entropy[row] = NAN;
  if (t == 0 && E.logprob) E.logprob[row] = NAN;
  for (int k = t; k < E.top; k += 16) {
    if (E.top_logprob) E.top_logprob[row * E.top + k] = NAN;
    if (E.top_index) E.top_index[row * E.top + k] = -1;
  }
}

// 16 lanes per row, class j * 16 + l in value j of lane l.  64 x 300 kept rows of 80 classes (fp32, an anchor plane apart): 28 us
// for 1.1 million scattered sectors of 64 bytes (68 MB), 2.4 TB/s; one image's 300 rows: 6.8 us, two
// dependent loads and the arithmetic of one wave.  A wave per row took 52 and 17 us: fewer rows, and so sectors, in flight.
template <typename T, int J, int ACT>
__device__ __forceinline__ void evidence_team(const Evidence &E, long long row, long long rows) {
  const int l = threadIdx.x & 15, group = (threadIdx.x & 63) >> 4;
  bool on = row < rows;
  const long long at = on ? row : 0, o = (unsigned)at / (unsigned)E.n1, m = at - o * E.n1;
  // count, index and label are on their way together: one latency instead of three (64 x 300 rows of 80 classes: 31.5 -> 29.1 us)
  const int count = E.count ? E.count[o] : 0;
  long long i = E.index ? E.index[at] : m;
  long long label = E.labels ? label_of(E, o, m) : -1;
  if (E.count && m >= count) on = false;
  if (on && E.index && (i < 0 || i >= E.index_range)) {
    store_nan(E, row, l);
    on = false;
  }
  if (!on) i = 0;
  const T *x = (const T *)E.x + o * E.s0 + i * E.s1;
  const int C = (int)E.classes;
  float v[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = j * 16 + l;
    v[j] = on && c < C ? to_float(x[c * E.cs]) : (ACT == LMI_PROB_NONE ? 0.0f : -INFINITY);
  }
  if (label >= C) label = -1;
  float lx = 0.0f;   // the label's value, from the lane that has it
#pragma unroll
  for (int j = 0; j < J; ++j) lx = label >> 4 == j ? v[j] : lx;
  lx = __shfl(lx, (int)label & 15, 16);
  float ref = 0.0f, log_s = 0.0f, h = 0.0f;
  if (ACT == LMI_PROB_SOFTMAX) {
    float mx = v[0];
#pragma unroll
    for (int j = 1; j < J; ++j) mx = fmaxf(mx, v[j]);
    Sums S = {__uint_as_float(reduce16(__float_as_uint(mx), MaxF())), 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < J; ++j) add_value(S, finite_ref(S.m), v[j]);
    S.s = __uint_as_float(reduce16(__float_as_uint(S.s), SumF()));
    S.t = __uint_as_float(reduce16(__float_as_uint(S.t), SumF()));
    softmax_result(S, ref, log_s, h);
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j) h += answer_entropy<ACT>(v[j]);
    h = __uint_as_float(reduce16(__float_as_uint(h), SumF()));
  }
  if (on && l == 0) {
    if (E.entropy) E.entropy[row] = h;
    if (E.logprob) E.logprob[row] = label >= 0 ? log_prob<ACT>(lx, ref, log_s) : NAN;
  }
  unsigned ord[J];
#pragma unroll
  for (int j = 0; j < J; ++j) ord[j] = j * 16 + l < C ? order_bits(v[j]) : 0u;
  for (int r = 0; r < E.top; ++r) {
    unsigned b = ord[0];
#pragma unroll
    for (int j = 1; j < J; ++j) b = ord[j] > b ? ord[j] : b;
    b = reduce16(b, MaxU());
    int c = -1;
#pragma unroll
    for (int j = 0; j < J; ++j) {   // the lowest class that has it
      const unsigned hit = (unsigned)(__ballot(ord[j] == b) >> (16 * group)) & 0xffffu;
      if (c < 0 && hit) {
        const int at = __builtin_ctz(hit);
        c = j * 16 + at;
        if (l == at) ord[j] = 0;
      }
    }
    if (on && l == 0) {
      if (E.top_logprob) E.top_logprob[row * E.top + r] = log_prob<ACT>(order_value(b), ref, log_s);
      if (E.top_index) E.top_index[row * E.top + r] = c;
    }
  }
}

template <typename T, int J, int ACT>
__global__ __launch_bounds__(256) void evidence_team_kernel(const Evidence E, long long rows) {
  for (long long first = (long long)blockIdx.x * 16; first < rows; first += (long long)gridDim.x * 16)   // more rows than a grid holds: several each
    evidence_team<T, J, ACT>(E, first + (threadIdx.x >> 4), rows);
}

struct alignas(16) PartHead {
  float m, s, t, pad;
};

// 511 rows of 32001 classes (bf16, top 10): 17.6 us, 1.9 TB/s -- every workgroup's row is in registers at once (two per CU, all of them
// resident), so it is the sum of loading (5.3 us), some 11 vector instructions a value (5) and the tail from the row's threshold to its
// ranked list (5): the two rows of a CU run in step.  2 rows of 200001 (fp32, top 20) in 25 parts: 11 and 5.5
// for the join.  Probabilities of 16 bits (`none`) spill 132 to 144 bytes a lane, held to four waves per SIMD.
// V > 1: classes lie side by side and are read in aligned 16-byte groups (the row may start anywhere; the groups at its two ends
// are read value by value).  V == 1: any class stride.
template <typename T, int V> struct Group {
  typedef T type __attribute__((ext_vector_type(V)));
  __device__ static __forceinline__ float get(const type &p, int u) { return to_float(p[u]); }
  __device__ static __forceinline__ void set(type &p, int u, T x) { p[u] = x; }
};
template <typename T> struct Group<T, 1> {
  typedef T type;
  __device__ static __forceinline__ float get(const type &p, int) { return to_float(p); }
  __device__ static __forceinline__ void set(type &p, int, T x) { p = x; }
};

template <typename T, int NT, int J, int V, int ACT>
__device__ __forceinline__ void evidence_row(const Evidence &E, long long row, int part, int t, TeamShared<NT> &L) {
  typedef Group<T, V> G;
  const int lane = t & 63, wave = t >> 6;
  const long long o = (unsigned)row / (unsigned)E.n1, m = row - o * E.n1;
  if (E.count && m >= E.count[o]) return;
  long long i = m;
  if (E.index) {
    i = E.index[row];
    if (i < 0 || i >= E.index_range) {
      if (t < 16) store_nan(E, row, t);
      return;
    }
  }
  const T *x = (const T *)E.x + o * E.s0 + i * E.s1;
  // this part's classes [c0, c0 + len); a tile starts up to 15 bytes before them, so that groups are aligned
  const long long c0 = (long long)part * E.part_len;
  const int len = (int)(E.classes - c0 < E.part_len ? E.classes - c0 : E.part_len);
  const T *xp = x + c0 * (V > 1 ? 1 : E.cs);
  const int start = V > 1 ? -(int)(((uintptr_t)xp & 15) / sizeof(T)) : 0;

  if (t < kMaxTop) L.list[t] = 0;
  LongSums total;   // softmax: this thread's sums with respect to its own m; else t = the entropy
  constexpr int N = J * V;
  const T absent = (T)(ACT == LMI_PROB_NONE ? 0.0f : -INFINITY);   // adds nothing to the sums
  for (long long tile = start; tile < len; tile += NT * N) {
    typename G::type p[J];
    const long long first = tile + t * V;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const long long e0 = first + j * NT * V;
      if (V > 1 && e0 >= 0 && e0 + V <= len) {
        p[j] = *(const typename G::type *)(xp + e0);
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const long long c = e0 + u;
          G::set(p[j], u, c >= 0 && c < len ? xp[c * (V > 1 ? 1 : E.cs)] : absent);
        }
      }
    }
    // a thread's own sums, group by group as the loads arrive: the exponentials of one run beside the loads of the next
    float mx = -INFINITY;
    Sums S = {total.a.m, 0.0f, 0.0f};   // of this tile
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float g = G::get(p[j], 0);
#pragma unroll
      for (int u = 1; u < V; ++u) g = fmaxf(g, G::get(p[j], u));   // drops NaN
      mx = fmaxf(mx, g);
      if (ACT == LMI_PROB_SOFTMAX) {
        rebase(S, fmaxf(S.m, g));
        const float ref = finite_ref(S.m);
#pragma unroll
        for (int u = 0; u < V; ++u) add_value(S, ref, G::get(p[j], u));
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u) S.t += answer_entropy<ACT>(G::get(p[j], u));
      }
    }
    const bool odd = S.t != S.t || (ACT == LMI_PROB_SOFTMAX && S.s != S.s);   // this thread's part of the tile holds a NaN, or an infinity that made one
    if (ACT == LMI_PROB_SOFTMAX) total.add(S);
    else total.add_entropy(S.t);
    if (E.top) {
      if (NT > 64) {
        L.lane_max[wave][lane] = mx;
        if (t == 0) L.n = 0;
        __syncthreads();
        for (int w = 0; w < NT / 64; ++w) mx = fmaxf(mx, L.lane_max[w][lane]);   // of this lane in every wave
      } else if (t == 0) {
        L.n = 0;
      }
      if (wave == 0) {   // the top-th best of 64 lane maxima bounds the top-th best of all values from below
        const float k = kth_of_lanes(mx, E.top);
        if (lane == 0) L.threshold = k;
      }
    }
    if (E.top) {
      team_sync<NT>();
      float thr = L.threshold;
      if (ACT == LMI_PROB_NONE && thr == 0.0f) thr = -INFINITY;   // perhaps the zeros of lanes without a class: values below zero may be the best there are
      const u64 kept = L.list[E.top - 1];
      if (kept) {
        const float k = order_value((unsigned)(kept >> 32));   // a NaN there: only NaNs can still be better
        thr = k != k ? INFINITY : fmaxf(thr, k);
      }
      forget(p);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float best = G::get(p[j], 0);
#pragma unroll
        for (int u = 1; u < V; ++u) best = fmaxf(best, G::get(p[j], u));
        if (!(best < thr) || odd) {   // few groups
#pragma unroll
          for (int u = 0; u < V; ++u) {
            const float v = G::get(p[j], u);
            const long long c = first + j * (NT * V) + u;
            if (!(v < thr) && c >= 0 && c < len) {   // NaN too
              const int at = atomicAdd(&L.n, 1);
              if (at < kCand) L.cand[at] = make_key(order_bits(v), (unsigned)(c0 + c));
            }
          }
        }
      }
      team_sync<NT>();
      const int n = L.n;
      if (n <= kCand) {
        rank_candidates<NT>(L, n, t, E.top);
      } else {
        const long long lo = tile > 0 ? tile : 0, hi = tile + NT * N < len ? tile + NT * N : len;
        top_by_rounds<NT>(L, [&](int e) -> u64 {
          const long long c = lo + e;
          return make_key(order_bits(to_float(xp[c * (V > 1 ? 1 : E.cs)])), (unsigned)(c0 + c));
        }, (int)(hi - lo), t, E.top);
      }
    }
  }
  // sums over the wave, then over the team
  Sums S = total.a;
  if (ACT == LMI_PROB_SOFTMAX) {
    rebase(S, reduce64(S.m, MaxF()));
    S.s = reduce64(S.s, SumF());
  }
  S.t = reduce64(S.t, SumF());
  if (NT > 64) {
    if (lane == 0) {
      L.red[wave][0] = S.m;
      L.red[wave][1] = S.s;
      L.red[wave][2] = S.t;
    }
    __syncthreads();
    if (wave) return;
    Sums W = {-INFINITY, 0.0f, 0.0f};
    if (lane < NT / 64) W = Sums{L.red[lane][0], L.red[lane][1], L.red[lane][2]};
    if (ACT == LMI_PROB_SOFTMAX) {
      rebase(W, reduce64(W.m, MaxF()));
      W.s = reduce64(W.s, SumF());
    }
    W.t = reduce64(W.t, SumF());
    S = W;
  }
  if (E.parts > 1) {
    unsigned char *out = E.ws + (row * E.parts + part) * (sizeof(PartHead) + (long long)kMaxTop * 8);
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
__global__ __launch_bounds__(NT == 64 ? 256 : NT, 4) void evidence_rows_kernel(const Evidence E) {
  constexpr int kTeams = NT == 64 ? 4 : 1;
  __shared__ TeamShared<NT> L[kTeams];
  const int team = NT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int t = threadIdx.x - team * NT;
  const long long rows = E.n0 * E.n1;
  for (long long row = (long long)blockIdx.x * kTeams + team; row < rows; row += (long long)gridDim.x * kTeams) {   // more rows than a grid holds: several each
    evidence_row<T, NT, J, V, ACT>(E, row, blockIdx.y, t, L[team]);
    team_sync<NT>();
  }
}

// a workgroup per row; lane p of the first wave holds the sums of part p (at most 64); a part's list is sorted
template <typename T, int ACT>
__global__ __launch_bounds__(256) void evidence_join_kernel(const Evidence E) {
  __shared__ TeamShared<256> L;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long long row = blockIdx.x;   // fewer than 256 of them
  const long long o = (unsigned)row / (unsigned)E.n1, m = row - o * E.n1;
  if (E.count && m >= E.count[o]) return;
  const long long i = E.index ? E.index[row] : m;
  if (E.index && (i < 0 || i >= E.index_range)) return;   // written by the parts
  constexpr long long kPart = sizeof(PartHead) + (long long)kMaxTop * 8;
  const unsigned char *base = E.ws + row * E.parts * kPart;
  // thread t: part t / 4, every fourth of its keys from t % 4 on; all loads at once
  u64 keys[kMaxTop / 4];
#pragma unroll
  for (int j = 0; j < kMaxTop / 4; ++j) {
    const int k = j * 4 + (t & 3);
    keys[j] = (t >> 2) < E.parts && k < E.top ? ((const u64 *)(base + (t >> 2) * kPart + sizeof(PartHead)))[k] : 0;
  }
  PartHead head = {-INFINITY, 0.0f, 0.0f, 0.0f};
  u64 best = 0;
  if (lane < E.parts) {
    head = *(const PartHead *)(base + lane * kPart);
    if (E.top) best = *(const u64 *)(base + lane * kPart + sizeof(PartHead));
  }
  Sums S = {head.m, head.s, head.t};
  float ref = 0.0f, log_s = 0.0f, h;
  if (ACT == LMI_PROB_SOFTMAX) {
    rebase(S, reduce64(S.m, MaxF()));
    S.s = reduce64(S.s, SumF());
    S.t = reduce64(S.t, SumF());
    softmax_result(S, ref, log_s, h);
  } else {
    h = reduce64(S.t, SumF());
  }
  if (E.top) {   // the top-th best of the parts' best bounds the answer from below; keys are distinct, so are ranks
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < 64; ++j) above += (u64)__shfl(best, j) > best;
    const u64 sel = __ballot(above == E.top - 1 && best != 0);
    const u64 thr = sel ? (u64)__shfl(best, __builtin_ctzll(sel)) : 1;
    if (t == 0) L.n = 0;
    if (t < kMaxTop) L.list[t] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMaxTop / 4; ++j)
      if (keys[j] >= thr) {
        const int at = atomicAdd(&L.n, 1);
        if (at < kCand) L.cand[at] = keys[j];
      }
    __syncthreads();
    const int n = L.n;
    if (n <= kCand) rank_candidates<256>(L, n, t, E.top);
    else top_by_rounds<256>(L, [&](int e) -> u64 { return e % kMaxTop < E.top ? ((const u64 *)(base + e / kMaxTop * kPart + sizeof(PartHead)))[e % kMaxTop] : 0; },
                            E.parts * kMaxTop, t, E.top);
  }
  if (wave) return;
  bool has = false;
  float lx = 0.0f;
  if (E.labels && lane == 0) {
    const long long l = label_of(E, o, m);
    has = l >= 0 && l < E.classes;
    if (has) lx = to_float(((const T *)E.x)[o * E.s0 + i * E.s1 + l * E.cs]);
  }
  store_row<ACT>(E, row, ref, log_s, h, has, lx, L.list, lane);
}

// insertion into a descending list; equal values stay in class order
template <int KT> __device__ __forceinline__ void insert(float (&val)[KT], int (&cls)[KT], float v, int c) {
  bool up = false;   // from its place on, everything moves down by one
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    up = up || !(v <= val[k]);   // an empty place is NaN
    const float a = val[k];
    const int b = cls[k];
    val[k] = up ? v : a;
    cls[k] = up ? c : b;
    v = up ? a : v;
    c = up ? b : c;
  }
}

// the two best so far, best first; no branch (almost every element of a wave's 64 rows enters some list)
__device__ __forceinline__ void insert2(float (&val)[2], int (&cls)[2], float v, int c) {
  // masks instead of conditions: the compiler makes branches of these
  const int first = -(int)(v > val[0]), second = -(int)(v > val[1]);
  const int next = (c & second) | (cls[1] & ~second);
  val[1] = __builtin_amdgcn_fmed3f(v, val[0], val[1]);
  cls[1] = (cls[0] & first) | (next & ~first);
  val[0] = fmaxf(val[0], v);
  cls[0] = (c & first) | (cls[0] & ~first);
}

// A thread per row, for rows side by side: a wave reads neighbouring rows' values of one class at a time.  The lists are kept by float
// comparisons; a row that holds a NaN (or an infinity that made one) is gone through again in the order that puts NaN first.
// 64 x 4 x 8400 rows of 16 bins (fp16, top 2): 35 us, 3.9 TB/s of 138 MB; the instructions that keep two best beside the softmax
// take as long as the loads.  Two rows of a 16-bit type per thread, read as one word, halve the loads and the threads: a tenth slower
// here and worse for longer lists (64 x 8400 x 80, top 5: 90 us, 74 with one).
template <typename T, int ACT, int KT>
__global__ __launch_bounds__(256) void evidence_planes_kernel(const Evidence E) {
  const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
  if (row >= E.n0 * E.n1) return;
  const long long o = (unsigned)row / (unsigned)E.n1, i = row - o * E.n1;   // fewer than 2^31 rows: a 64-bit division costs as much as four classes
  if (E.count && i >= E.count[o]) return;
  const T *x = (const T *)E.x + o * E.s0 + i * E.s1;
  LongSums total;
  constexpr int KL = KT ? KT : 1;
  float val[KL];
  int cls[KL];
#pragma unroll
  for (int k = 0; k < KT; ++k) val[k] = NAN, cls[k] = -1;
  constexpr int U = KT <= 2 ? 16 : 8;   // loads in flight, and values per update of m
  const int C = (int)E.classes;
  if constexpr (KT == 2) {   // the two best of class 0 and nothing else: what equals -inf after it comes in class order
    val[0] = to_float(x[0]), cls[0] = 0;
    val[1] = -INFINITY, cls[1] = 1;
  }
  auto take = [&](int c, auto all) {   // U classes from c on, or those of them below C
    constexpr bool kAll = decltype(all)::value;
    T w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kAll || c + u < C) w[u] = x[(long long)(c + u) * E.cs];
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = kAll || c + u < C ? to_float(w[u]) : (ACT == LMI_PROB_NONE ? 0.0f : -INFINITY);
    if (ACT == LMI_PROB_SOFTMAX) {
      float mx = total.a.m;
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, v[u]);
      Sums S = {mx, 0.0f, 0.0f};
      const float ref = finite_ref(S.m);
#pragma unroll
      for (int u = 0; u < U; ++u) add_value(S, ref, v[u]);
      total.add(S);
    } else {
      float h = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) h += answer_entropy<ACT>(v[u]);
      total.add_entropy(h);
    }
    if constexpr (KT == 2) {
      if (c > 0) insert2(val, cls, v[0], c);
#pragma unroll
      for (int u = 1; u < U; ++u)
        if (kAll || c + u < C) insert2(val, cls, v[u], c + u);
    } else if constexpr (KT > 0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if ((kAll || c + u < C) && !(v[u] <= val[KL - 1])) insert<KL>(val, cls, v[u], c + u);
    }
  };
  int c = 0;
  for (; c + U <= C; c += U) take(c, std::true_type());
  if (c < C) take(c, std::false_type());
  float ref = 0.0f, log_s = 0.0f, h = total.a.t;
  if (ACT == LMI_PROB_SOFTMAX) softmax_result(total.a, ref, log_s, h);
  if (E.entropy) E.entropy[row] = h;
  if (E.logprob) {
    const long long l = E.labels ? label_of(E, o, i) : -1;
    E.logprob[row] = l >= 0 && l < C ? log_prob<ACT>(to_float(x[l * E.cs]), ref, log_s) : NAN;
  }
  int n = 0;
  if (KT && h != h) {   // first the NaNs by class, then the others
    for (int c = 0; c < C && n < E.top; ++c) {
      const float v = to_float(x[(long long)c * E.cs]);
      if (v != v) {
        if (E.top_logprob) E.top_logprob[row * E.top + n] = NAN;
        if (E.top_index) E.top_index[row * E.top + n] = c;
        ++n;
      }
    }
#pragma unroll
    for (int k = 0; k < KT; ++k) val[k] = NAN, cls[k] = -1;
    for (int c = 0; c < C; ++c) {
      const float v = to_float(x[(long long)c * E.cs]);
      if (v == v && !(v <= val[KL - 1])) insert<KL>(val, cls, v, c);
    }
  }
  if constexpr (KT == 2) {
    if (E.pairs && n == 0) {   // a row's two results as one word
      typedef float f2 __attribute__((ext_vector_type(2)));
      typedef int i2 __attribute__((ext_vector_type(2)));
      *(f2 *)(E.top_logprob + row * 2) = f2{log_prob<ACT>(val[0], ref, log_s), log_prob<ACT>(val[1], ref, log_s)};
      *(i2 *)(E.top_index + row * 2) = i2{cls[0], cls[1]};
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < KT; ++k)
    if (n + k < E.top) {
      if (E.top_logprob) E.top_logprob[row * E.top + n + k] = log_prob<ACT>(val[k], ref, log_s);
      if (E.top_index) E.top_index[row * E.top + n + k] = cls[k];
    }
}

// Parts per row.  A row of up to two tiles of a workgroup of 512 (fp32: 32704 values) is read by one, as fast as parts and their join
// (16 x 32001 bf16: 11 us, 19 in parts of 4096); longer ones of a batch too small to fill the chip are cut into parts of about a tile of 256
// threads, at most 64, one per lane of the joining wave
// (in parts and in one piece, bf16: 2 x 70001 16 and 24 us, 16 x 200001 16 and 50, 100 x 70001 20 and 27, 255 x 70001 30 and 29; 2 x 200001 fp32 16 and 75)
int split_parts(long long rows, long long classes, long long class_stride, int size) {
  const long long unit = class_stride == 1 ? 255 * (128 / size) : 2 * 256 * 8;
  if (rows >= 256 || classes < LMI_LOGPROB_SPLIT_FROM || classes <= 4 * unit) return 1;
  const long long p = (classes + unit - 1) / unit;
  return (int)(p < 64 ? p : 64);
}

template <typename T, int ACT, int KT> void launch_planes(Evidence E, hipStream_t st) {
  const long long rows = E.n0 * E.n1;
  E.pairs = E.top == 2 && E.top_logprob && E.top_index && lmi_is_aligned(E.top_logprob, 8) && lmi_is_aligned(E.top_index, 8);
  evidence_planes_kernel<T, ACT, KT><<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(E);
}

constexpr long long kMaxGrid = 1 << 22;   // workgroups: with their threads below 2^32

template <typename T, int ACT> int launch(const Evidence &E0, hipStream_t st) {
  Evidence E = E0;
  const long long rows = E.n0 * E.n1;
  // Rows side by side: a thread per row where there are enough of them for the chip, the more the longer their lists (fp16, us here and with 16
  // lanes per row: 8400 x 80, top 2 6.9 and 5.9, top 5 28 and 7.5; 4 x 8400 x 80, top 2 7.9 and 12, top 5 24 and 15; 4 x 8400 x 40, top 5
  // 11 and 13; 16 x 8400 x 80, top 5 35 and 40).  Lists of more than eight gain little at best (64 x 8400 x 64, top 20: 225 and 314, x 128
  // 411 and 352).  Up to 8 classes always (64 x 8400 of 4, top 2: 9.7 and 45).
  const long long enough = E.top <= 2 ? 16384 : E.classes <= 40 ? 32768 : 131072;
  const bool planes = !E.index && E.classes <= 65536 && E.top <= 8 && (E.classes <= 8 || (E.cs != 1 && E.s1 < E.cs && rows >= enough));
  if (planes) {
    if (E.top == 0) launch_planes<T, ACT, 0>(E, st);
    else if (E.top <= 2) launch_planes<T, ACT, 2>(E, st);
    else launch_planes<T, ACT, 8>(E, st);
    return lmi_check_launch("lmi_class_logprobs");
  }
  if (E.classes <= 128) {
    const long long teams = (rows + 15) / 16;
    const unsigned g = (unsigned)(teams < kMaxGrid ? teams : kMaxGrid);
    if (E.classes <= 32) evidence_team_kernel<T, 2, ACT><<<g, 256, 0, st>>>(E, rows);
    else evidence_team_kernel<T, 8, ACT><<<g, 256, 0, st>>>(E, rows);
    return lmi_check_launch("lmi_class_logprobs");
  }
  E.parts = split_parts(rows, E.classes, E.cs, sizeof(T));
  E.part_len = (E.classes + E.parts - 1) / E.parts;
  const dim3 g((unsigned)(rows < kMaxGrid ? rows : kMaxGrid), (unsigned)E.parts);
  const dim3 g4((unsigned)((rows + 3) / 4 < kMaxGrid ? (rows + 3) / 4 : kMaxGrid), (unsigned)E.parts);
  constexpr int V = 16 / sizeof(T);   // 128 bytes of a row per thread
  if (E.cs == 1) {
    // The smallest team that holds a row (or part) in one go; with many rows, whose teams fill the chip anyway, a smaller one that
    // goes over the row in tiles (bf16, top 5, a wave / 256 / 512 threads: 512 x 8000 18 / 12 / 14 us, 512 x 32001 49 / 20 / 16,
    // 2048 x 8000 22 / 26 / 46, 2048 x 32001 61 / 47 / 50, 16384 x 8000 94 / 169 / 334, 16384 x 32001 297 / 297 / 330).
    constexpr long long kWave = 63 * 8 * V, kFour = 255 * 8 * V;   // a tile may start up to 15 bytes before its values
    const bool many = rows * E.parts >= 2048;
    if (E.part_len <= (many ? 2 * kWave : kWave)) evidence_rows_kernel<T, 64, 8, V, ACT><<<g4, 256, 0, st>>>(E);
    else if (E.part_len <= kFour || many) evidence_rows_kernel<T, 256, 8, V, ACT><<<g, 256, 0, st>>>(E);
    else evidence_rows_kernel<T, 512, 8, V, ACT><<<g, 512, 0, st>>>(E);
  } else {
    if (E.part_len <= 512) evidence_rows_kernel<T, 64, 8, 1, ACT><<<g4, 256, 0, st>>>(E);
    else evidence_rows_kernel<T, 256, 8, 1, ACT><<<g, 256, 0, st>>>(E);
  }
  if (E.parts > 1) evidence_join_kernel<T, ACT><<<(unsigned)rows, 256, 0, st>>>(E);
  return lmi_check_launch("lmi_class_logprobs");
}

template <typename T> int launch_act(const Evidence &E, int act, hipStream_t st) {
  if (act == LMI_PROB_SOFTMAX) return launch<T, LMI_PROB_SOFTMAX>(E, st);
  if (act == LMI_PROB_SIGMOID) return launch<T, LMI_PROB_SIGMOID>(E, st);
  return launch<T, LMI_PROB_NONE>(E, st);
}

// memory of a call, as addresses [first, last)
struct Range {
  const char *name;
  uintptr_t first, last;
};
// `elements` of `size` bytes each from p on, the last dimension's among them; then two more dimensions
Range range_of(const char *name, const void *p, int64_t size, int64_t elements, int64_t n0 = 1, int64_t s0 = 0, int64_t n1 = 1, int64_t s1 = 0) {
  if (!p) return {name, 0, 0};
  int64_t low = 0, high = elements;
  for (const int64_t d : {(n0 - 1) * s0, (n1 - 1) * s1}) (d < 0 ? low : high) += d;
  return {name, (uintptr_t)p + low * size, (uintptr_t)p + high * size};
}
// the first result that lies in the memory of an input or of a result before it
bool overlapping(const lmi_logprob_args *a, const char *&result, const char *&other) {
  const int64_t rows = a->n0 * a->n1, label = a->label_dtype == LMI_I64 ? 8 : 4;
  const Range all[] = {range_of("x", a->x, a->x_dtype == LMI_F32 ? 4 : 2, (a->classes - 1) * a->class_stride + 1, a->n0, a->stride0,
                                a->index ? a->index_range : a->n1, a->stride1),
                       range_of("labels", a->labels, label, 1, a->n0, a->label_stride0, a->n1, a->label_stride1),
                       range_of("index", a->index, 4, rows), range_of("count", a->count, 4, a->n0), range_of("logprob", a->logprob, 4, rows),
                       range_of("entropy", a->entropy, 4, rows), range_of("top_logprob", a->top_logprob, 4, rows * a->top),
                       range_of("top_index", a->top_index, 4, rows * a->top)};
  for (int i = 4; i < 8; ++i)
    for (int j = 0; j < i; ++j)
      if (all[i].first < all[j].last && all[j].first < all[i].last && all[i].first < all[i].last) {
        result = all[i].name;
        other = all[j].name;
        return true;
      }
  return false;
}

}  // namespace

extern "C" {

int64_t lmi_class_logprobs_workspace_bytes(int64_t rows, int64_t classes, int64_t class_stride, int x_dtype) {
  if (rows <= 0 || classes <= 0) return 0;
  const int parts = split_parts(rows, classes, class_stride, x_dtype == LMI_F32 ? 4 : 2);
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
  const int64_t need = lmi_class_logprobs_workspace_bytes(a->n0 * a->n1, a->classes, a->class_stride, a->x_dtype);
  LMI_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need), LMI_ERR_WORKSPACE,
              "lmi_class_logprobs: workspace of %lld bytes, %lld needed", (long long)a->workspace_bytes, (long long)need);
  LMI_REQUIRE(need == 0 || lmi_is_aligned(a->workspace, 16), LMI_ERR_ALIGNMENT, "lmi_class_logprobs: workspace must be 16-byte aligned");
  const char *result = nullptr, *other = nullptr;
  LMI_REQUIRE(!overlapping(a, result, other), LMI_ERR_BAD_ARG, "lmi_class_logprobs: %s lies in the memory of %s", result, other);
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
  E.pairs = 0;
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
