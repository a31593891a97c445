// MXFP4 (4-bit e2m1 elements, one power-of-two scale per 32) for gfx950: quantising, reading back, and the product of
// quantised weights with activations -- a 1x1 convolution of the network with its folded batch norm and SiLU, or a linear layer.
//
// A block's scale is 2^(floor(log2 max) - 2), so its largest element lands in [4, 8): 6 is the largest magnitude of e2m1, and
// what rounds beyond it stays at 6.  v_cvt_scalef32_pk_fp4_* divides by the scale and rounds to nearest even with that
// saturation; x / 2^e is exact, so nothing is rounded twice.  The products run on v_mfma_scale_f32_32x32x64_f8f6f4 (twice the
// rate of the 16x16x128 form): 64 elements of k per instruction, every lane brings 32 elements of one row and their
// scale byte -- one block --, sums in fp32.  Quantised tensors are kept in that order (see lmi_hip.h), so an operand of a
// wave is one contiguous kilobyte, and the scale bytes of four steps are one word of which the instruction picks a byte; a step of all rows lies together, so
// that what neighbouring workgroups read at a time does, too.
//
// Kernels
//  mx_quantize_kernel     a wave takes 8 rows x 256 elements: four lanes per block, 8 elements each, four steps per lane.
//  mx_dequantize_kernel   8 rows x one step per wave, whole lines written.
//  mx_stream_kernel       the product of many positions that come as floats: 128 of them x up to 320 weight rows per workgroup, streamed along k.
//  mx_rows_kernel         the product of many quantised rows: 128 or 256 of them per workgroup.
//  mx_wave_planes_kernel  shallow 1x1 convolutions (k <= 64): a wave per 64 positions, everything in registers.
//  mx_few_kernel          few positions (a single row, one image's deepest maps): the waves of a workgroup share k.
#include <hip/hip_fp16.h>

#include <type_traits>

#include "common.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

struct Packed {};   // x is quantised already

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// scale byte of a block from the bits of its largest magnitude (an infinity or a NaN has the largest bits: 255)
__device__ __forceinline__ unsigned scale_byte(unsigned magnitude) {
  const unsigned e = magnitude >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
__device__ __forceinline__ float scale_value(unsigned byte) { return __uint_as_float(byte << 23); }   // the conversions use the exponent bits alone: 0 = 2^-127

__device__ __forceinline__ unsigned pack8(const float *v, float scale) {
  unsigned r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
  return r;
}

// 8 elements from p on, `n` of them in the row; VEC: all 8, 16-byte aligned
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T *p, long long n, float (&v)[8]) {
  if (VEC && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      const t8 a = *(const t8 *)p;
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = to_float(a[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = u < n ? to_float(p[u]) : 0.0f;
  }
}

// Bound by HBM: 409600 x 320 fp16 (331 MB in and out) 62 us, 5.3 TB/s; 640 x 2560 fp32 4 us.
// lane = (row of the octet, block of the step, quarter of the block).  The wave reads 8 rows x 128 bytes (16-bit types) per step and writes 8 x 16
// bytes side by side for either block; the scale bytes of its four steps leave as one word.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *x, long long rows, long long k, long long row_stride, unsigned steps, unsigned quads,
                                                          long long units, unsigned *packed, unsigned *scales) {
  const int lane = threadIdx.x & 63, quarter = lane & 3, half = (lane >> 2) & 1, r8 = lane >> 3;
  const long long groups = (rows + 31) >> 5;
  for (long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += (long long)gridDim.x * 4) {   // row octet x four steps
    const long long octet = unit / quads;
    const unsigned quad = (unsigned)(unit - octet * quads);
    const long long row = octet * 8 + r8, group = octet >> 2;
    const int rg = (int)(octet & 3) * 8 + r8;
    const T *p = x + row * row_stride;
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long c0 = ((long long)quad * 4 + i) * 64 + half * 32 + quarter * 8;
      load8<T, VEC>(p + c0, row < rows ? k - c0 : 0, v[i]);
    }
    unsigned word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned m = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) m = max(m, __float_as_uint(v[i][u]) & 0x7fffffffu);
      m = max(m, __shfl_xor(m, 1));
      m = max(m, __shfl_xor(m, 2));
      const unsigned byte = scale_byte(m), step = quad * 4 + i;
      word |= byte << (8 * i);
      if (step < steps) packed[(((step * groups + group) * 2 + half) * 32 + rg) * 4 + quarter] = pack8(v[i], scale_value(byte));
    }
    if (quarter == 0) scales[((quad * groups + group) * 2 + half) * 32 + rg] = word;
  }
}

// Bound by HBM: 409600 x 320 to fp32 (594 MB) 87 us, 6.8 TB/s (195 us with every lane writing its own 32 bytes).
// A wave takes 8 rows x one step.  16-bit results: lane (row, block, quarter) writes 8 of them, a row's eight lanes one line of 128
// bytes.  fp32: a line is one block, so the eight lanes write block 0, then block 1, four elements each, which they get from the lane
// that read them.
template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned *packed, const unsigned *scales, long long rows, long long k, unsigned steps,
                                                            long long units, bool vec, T *out) {
  const int lane = threadIdx.x & 63, quarter = lane & 3, half = (lane >> 2) & 1, r8 = lane >> 3;
  const long long groups = (rows + 31) >> 5;
  for (long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += (long long)gridDim.x * 4) {
    const long long octet = unit / steps;
    const unsigned step = (unsigned)(unit - octet * steps);
    const long long row = octet * 8 + r8, group = octet >> 2;
    const int rg = (int)(octet & 3) * 8 + r8;
    const unsigned word = packed[(((step * groups + group) * 2 + half) * 32 + rg) * 4 + quarter];   // rows beyond the last are zeros there
    const unsigned byte = (scales[(((step >> 2) * groups + group) * 2 + half) * 32 + rg] >> (8 * (step & 3))) & 255u;
    // 2^(byte - 127); the smallest is subnormal, 255 is NaN
    const float s = byte == 255u ? NAN : (byte ? __uint_as_float(byte << 23) : 0x1p-127f);
    T *p = out + row * k + step * 64ll;
    if constexpr (sizeof(T) == 4) {
      const int i = lane & 7;   // of the row's eight lanes
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int from = (lane & ~7) + b * 4 + (i >> 1);
        const unsigned w = (unsigned)__shfl((int)word, from) >> (16 * (i & 1));
        const float sb = __shfl(s, from);
        const f2 lo = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0)), hi = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1));
        const long long left = k - step * 64ll - b * 32 - i * 4;
        T *q = p + b * 32 + i * 4;
        if (row < rows) {
          if (vec && left >= 4) {
            typedef float f4 __attribute__((ext_vector_type(4)));
            __builtin_nontemporal_store(f4{lo.x * sb, lo.y * sb, hi.x * sb, hi.y * sb}, (f4 *)q);
          } else {
            if (left > 0) q[0] = lo.x * sb;
            if (left > 1) q[1] = lo.y * sb;
            if (left > 2) q[2] = hi.x * sb;
            if (left > 3) q[3] = hi.y * sb;
          }
        }
      }
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      t8 v;
      const f2 e0 = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 0)), e1 = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 1)),
               e2 = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 2)), e3 = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 3));
      v[0] = (T)(e0.x * s), v[1] = (T)(e0.y * s), v[2] = (T)(e1.x * s), v[3] = (T)(e1.y * s);
      v[4] = (T)(e2.x * s), v[5] = (T)(e2.y * s), v[6] = (T)(e3.x * s), v[7] = (T)(e3.y * s);
      const long long left = k - step * 64ll - half * 32 - quarter * 8;
      T *q = p + half * 32 + quarter * 8;
      if (row < rows) {
        if (vec && left >= 8) {
          __builtin_nontemporal_store(v, (t8 *)q);
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (u < left) q[u] = v[u];
        }
      }
    }
  }
}

struct Product {
  const void *x;
  const unsigned *xs;
  long long pixels, k, n, xb, xs1;   // xs1: between positions (rows) or channels (planes)
  const uint4 *w;
  const unsigned *ws;
  const float *bias;
  void *y;
  unsigned tiles_pixels;  // tiles of positions per image
  int tiles_n;            // tiles of 32 weight rows
  int split_n;            // tiles of 32 weight rows per wave (mx_wave_planes_kernel)
  int all_steps;          // steps of 64 along k
};

constexpr int kTile = 64;   // positions of a wave

template <int ACT> __device__ __forceinline__ float activate(float v) {
  // v_exp_f32 and v_rcp_f32, an ulp each: an IEEE division here made the results' arithmetic, not their bytes, the bound of shallow products
  if (ACT == LMI_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
  return v;
}

// one block from 32 values
__device__ __forceinline__ uint4 quantize_block(const float (&v)[32], unsigned &byte) {
  unsigned m = 0;
#pragma unroll
  for (int u = 0; u < 32; ++u) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
  byte = scale_byte(m);
  const float s = scale_value(byte);
  return make_uint4(pack8(v, s), pack8(v + 8, s), pack8(v + 16, s), pack8(v + 24, s));
}

// two blocks from 32 words that hold one value of either (two neighbouring pixels of 32 channels), 16-bit types: magnitudes are compared as
// integers, two at a time, and go into the conversion as they are
template <typename T> __device__ __forceinline__ void quantize_pair16(const unsigned (&w)[32], uint4 (&f)[2], unsigned (&byte)[2]) {
  us2 m = {0, 0};
#pragma unroll
  for (int u = 0; u < 32; ++u) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, w[u] & 0x7fff7fffu));
#pragma unroll
  for (int px = 0; px < 2; ++px) {
    const float mag = to_float(__builtin_bit_cast(T, (unsigned short)m[px]));
    byte[px] = scale_byte(__float_as_uint(mag));
    const float s = scale_value(byte[px]);
    unsigned r[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      unsigned a = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned two = __builtin_amdgcn_perm(w[q * 8 + 2 * j + 1], w[q * 8 + 2 * j], px ? 0x07060302u : 0x05040100u);
        if constexpr (__is_same(T, _Float16)) {
          const h2 t = __builtin_bit_cast(h2, two);
          a = j == 0 ? __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(a, t, s, 0) : j == 1 ? __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(a, t, s, 1)
            : j == 2 ? __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(a, t, s, 2) : __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(a, t, s, 3);
        } else {
          const b2 t = __builtin_bit_cast(b2, two);
          a = j == 0 ? __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(a, t, s, 0) : j == 1 ? __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(a, t, s, 1)
            : j == 2 ? __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(a, t, s, 2) : __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(a, t, s, 3);
        }
      }
      r[q] = a;
    }
    f[px] = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

// Columns of the two 32-column subtiles: position 2j + h of the tile is column j of subtile h, so that a lane's two results are
// neighbours.  Rows of a weight tile are permuted the same way on both sides of the product: result i of a lane is weight row
// 16*(lane >> 5) + i of the tile.
__device__ __forceinline__ int weight_lane(int lane) {
  const int r = lane & 31;
  return (lane & 32) + ((r >> 2) & 1) * 16 + (r >> 3) * 4 + (r & 3);
}

__device__ __forceinline__ v8i operand(const uint4 &a) { return v8i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}; }

template <int BYTE> __device__ __forceinline__ void mfma2(f16x (&acc)[2], const uint4 &a, unsigned sa, const uint4 &b0, const uint4 &b1, unsigned sb0, unsigned sb1) {
  acc[0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(a), operand(b0), acc[0], 4, 4, BYTE, (int)sa, BYTE, (int)sb0);
  acc[1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(a), operand(b1), acc[1], 4, 4, BYTE, (int)sa, BYTE, (int)sb1);
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <typename T> struct Raw {   // one step's values of a lane before they are quantised: two pixels of 32 channels
  unsigned v[32];
};
template <> struct Raw<float> {
  f2 v[32];
};

// Addresses are a base that is the same for the wave (scalar registers) plus a 32-bit offset of the lane: the launcher sees to it that
// 32 channels or rows fit.
template <typename W, int ALIGN = sizeof(W)> __device__ __forceinline__ W at(const void *base, unsigned offset) {
  typedef const __attribute__((address_space(1))) char *global;
  typedef W word __attribute__((aligned(ALIGN)));
  global b = (global)base;
  asm("" : "+s"(b));   // kept in scalar registers: without this the sum goes to a pair of vector registers per load
  return *(const __attribute__((address_space(1))) word *)(b + offset);
}
template <typename W, int ALIGN = sizeof(W)> __device__ __forceinline__ W at_any(const void *base, unsigned offset) {   // a base of the lane's own
  typedef W word __attribute__((aligned(ALIGN)));
  return *(const word *)((const char *)base + offset);
}

// `in` channels (32 or more: all) of two neighbouring pixels from base + offset on, one word at whatever address; base is uniform
template <typename T, bool SCALAR = true>
__device__ __forceinline__ void load_planes(const T *base, unsigned offset, long long stride, bool live, int in, Raw<T> &r) {
  typedef typename std::remove_reference<decltype(r.v[0])>::type W;
  if (live && in >= 32) {
#pragma unroll
    for (int u = 0; u < 32; ++u) r.v[u] = SCALAR ? at<W, sizeof(T)>(base + u * stride, offset) : at_any<W, sizeof(T)>(base + u * stride, offset);
  } else if (live && in > 0) {   // the last channels: all loads at once, those beyond read the first again
#pragma unroll
    for (int u = 0; u < 32; ++u) r.v[u] = at_any<W, sizeof(T)>(base + (u < in ? u * stride : 0), offset);
#pragma unroll
    for (int u = 0; u < 32; ++u) r.v[u] = u < in ? r.v[u] : W{};
  } else {
#pragma unroll
    for (int u = 0; u < 32; ++u) r.v[u] = W{};
  }
}
// Planes of odd size (640 -> 320 on 37 x 37 fp16 8.3 us, value by value 24; 64 x 320 -> 320 on 79 x 79 190 and 359): the pair that reaches beyond its plane, `live` == 1, is read one
// pixel earlier, in the same plane, which has at least two; move_pair puts its pixel where it belongs.
template <typename T, bool SCALAR = true>
__device__ __forceinline__ void load_planes_odd(const T *base, unsigned offset, long long stride, int live, int in, Raw<T> &r) {
  load_planes<T, SCALAR>(base - 1, offset + (live == 1 ? 0 : sizeof(T)), stride, live > 0, in, r);
}
template <typename T> __device__ __forceinline__ void move_pair(Raw<T> &r, bool late) {
  if (late) {
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      if constexpr (sizeof(T) == 4) r.v[u] = f2{r.v[u].y, 0.0f};
      else r.v[u] >>= 16;
    }
  }
}
__device__ __forceinline__ void quantize_raw(const Raw<float> &r, uint4 (&f)[2], unsigned (&byte)[2]) {
  float a[32];
#pragma unroll
  for (int u = 0; u < 32; ++u) a[u] = r.v[u].x;
  f[0] = quantize_block(a, byte[0]);
#pragma unroll
  for (int u = 0; u < 32; ++u) a[u] = r.v[u].y;
  f[1] = quantize_block(a, byte[1]);
}
template <typename T> __device__ __forceinline__ void quantize_raw(const Raw<T> &r, uint4 (&f)[2], unsigned (&byte)[2]) { quantize_pair16<T>(r.v, f, byte); }

// the sums of weight tile nt start at the bias
__device__ __forceinline__ void start_sums(const Product &P, int nt, int lane, f16x (&acc)[2]) {
  const long long n0 = (long long)nt * 32 + 16 * (lane >> 5);
  acc[0] = f16x{};
  if (P.bias) {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[0][i] = P.bias[n0 + i < P.n ? n0 + i : P.n - 1];   // rows beyond the last are not stored
  }
  acc[1] = acc[0];
}

// planes: a lane holds 16 weight rows' results of two neighbouring positions.  Results are not read again soon: stored past the caches
// (the 160 x 160 maps of a batch of 64, 48 -> 32 channels: 75 -> 56 us with the sums starting at the bias).
template <typename Y>
__device__ __forceinline__ void store_planes(const Product &P, Y *y, long long p0, int live, int nt, int lane, int act, bool even, const f16x (&acc)[2]) {
  const int px = 2 * (lane & 31), n0 = 16 * (lane >> 5);
  const long long left = P.n - nt * 32ll - n0;
  const unsigned offset = (unsigned)(n0 * P.pixels + px) * sizeof(Y);
  Y *base = y + nt * 32ll * P.pixels + p0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float v0 = acc[0][i], v1 = acc[1][i];
    if (act) {
      v0 = activate<LMI_ACT_SILU>(v0);
      v1 = activate<LMI_ACT_SILU>(v1);
    }
    typedef Y y2 __attribute__((ext_vector_type(2)));
    typedef y2 pair __attribute__((aligned(sizeof(Y))));
    Y *q = (Y *)((char *)(base + i * P.pixels) + offset);
    if ((even ? px : px + 1) < live && i < left) __builtin_nontemporal_store(y2{(Y)v0, (Y)v1}, (pair *)q);
    if (!even && px + 1 == live && i < left) *q = (Y)v0;   // the last of a plane of odd size
  }
}

// rows: a lane holds 16 neighbouring results of either of its two positions (32 apart)
template <typename Y>
__device__ __forceinline__ void store_rows(const Product &P, Y *y, long long p0, int live, int nt, int lane, int act, int vec, const f16x (&acc)[2]) {
  const long long n0 = (long long)nt * 32 + 16 * (lane >> 5);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int px = 32 * h + (lane & 31);
    if (px >= live) continue;
    Y *q = y + (p0 + px) * P.n + n0;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] = acc[h][i];
      if (act) v[i] = activate<LMI_ACT_SILU>(v[i]);
    }
    if (vec && n0 + 16 <= P.n) {
      constexpr int W = 16 / sizeof(Y);
      typedef Y yw __attribute__((ext_vector_type(W)));
#pragma unroll
      for (int j = 0; j < 16 / W; ++j) {
        yw o;
#pragma unroll
        for (int u = 0; u < W; ++u) o[u] = (Y)v[j * W + u];
        ((yw *)q)[j] = o;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (n0 + i < P.n) q[i] = (Y)v[i];
    }
  }
}

// One wave, 64 positions, k of one step (at most 64), everything in registers: what a lane quantises is its operand.  No LDS, no barrier: the
// waves of a CU drift apart, so that some load while others multiply.  Bound by HBM: 64 x 64 -> 32 on 160 x 160 59 us, 5.3 TB/s (69 streamed);
// 16 x 48 -> 32 on 160 x 160 17.5 and 21.  Two steps held that way stream faster: 16 x 128 -> 64 on 80 x 80 13.6 us, 11 streamed.
template <typename T, bool VEC>
__global__ __launch_bounds__(256, 4) void mx_wave_planes_kernel(const Product P, int act, long long tiles) {
  const int lane = threadIdx.x & 63;
  const unsigned tile = blockIdx.x * 4 + wave_id();
  if (tile >= tiles) return;
  const long long image = tile / P.tiles_pixels;
  const long long p0 = (long long)(tile % P.tiles_pixels) * kTile;
  const int live = (int)(P.pixels - p0 < kTile ? P.pixels - p0 : kTile);
  const T *x = (const T *)P.x + image * P.xb + p0;
  const int half = lane >> 5, left = (int)P.k - 32 * half;
  Raw<T> raw;
  const unsigned offset = (unsigned)(half * 32 * P.xs1 + 2 * (lane & 31)) * sizeof(T);
  const int here = live - 2 * (lane & 31);
  if constexpr (VEC) {
    load_planes<T>(x, offset, P.xs1, here > 0, left < 0 ? 0 : left, raw);
  } else {
    load_planes_odd<T>(x, offset, P.xs1, here, left < 0 ? 0 : left, raw);
    move_pair<T>(raw, here == 1);
  }
  uint4 f[2];
  unsigned byte[2];
  quantize_raw(raw, f, byte);
  const int wl = weight_lane(lane);
  const int nt0 = blockIdx.y * P.split_n;
  const int nt1 = nt0 + P.split_n < P.tiles_n ? nt0 + P.split_n : P.tiles_n;
  T *y = (T *)P.y + image * P.pixels * P.n;
  for (int nt = nt0; nt < nt1; ++nt) {
    f16x acc[2];
    start_sums(P, nt, lane, acc);
    mfma2<0>(acc, P.w[nt * 64ll + wl], P.ws[nt * 64ll + wl], f[0], f[1], byte[0], byte[1]);
    store_planes<T>(P, y, p0, live, nt, lane, act, VEC, acc);
  }
}

template <typename T, bool VEC> void launch_wave_planes(Product P, int act, long long batch, hipStream_t st) {
  P.tiles_pixels = (unsigned)((P.pixels + kTile - 1) / kTile);
  const long long tiles = batch * P.tiles_pixels;
  const long long split = tiles < 2048 ? (2048 + tiles - 1) / tiles : 1;
  P.split_n = (int)((P.tiles_n + split - 1) / split);
  const dim3 grid((unsigned)((tiles + 3) / 4), (unsigned)((P.tiles_n + P.split_n - 1) / P.split_n));
  mx_wave_planes_kernel<T, VEC><<<grid, 256, 0, st>>>(P, act, tiles);
}

// Streaming product: 128 positions x up to 64 * NT weight rows per workgroup, k in chunks of two steps.  While the matrix instructions run
// on one chunk, the next chunk's activations and weights are on their way to registers (loads straight to LDS would be waited for
// before the next read of any LDS); an activation block is quantised by the thread that loaded it.  Waves are dealt 2 (positions) x 2 (weight rows), each 64 positions x 32 * NT
// rows of sums in registers: a fragment read from LDS serves 2 or NT matrix instructions.  Bound by HBM: 64 x 1280 -> 320 on 80 x 80 (fp16, 1.31 GB) 273 us, 4.8 TB/s (64 x 320 -> 320: 0.52 GB, 124 us, 4.2); two
// workgroups per CU hold 64 KB of loads in flight and stop for each other at every chunk, which costs the rest to 6.2 TB/s.  The widest tiles (five per wave, planes of
// 16 bits) spill 8 to 12 bytes a lane.
constexpr int kChunkTile = 128;

template <typename T, bool PLANES, bool VEC> struct Chunk;   // what a thread holds of a chunk
// planes: two neighbouring pixels x one block
template <typename T, bool VEC> struct Chunk<T, true, VEC> {
  Raw<T> raw;
  bool late = false;
  __device__ __forceinline__ void load(const Product &P, const T *x, int live, int chunk) {
    const int pair = threadIdx.x & 63;
    const long long c0 = (4ll * chunk + wave_id()) * 32;   // beyond k: in = 0
    const int in = c0 < P.k ? (int)(P.k - c0 < 32 ? P.k - c0 : 32) : 0;
    if constexpr (VEC) {
      load_planes<T>(x + c0 * P.xs1, 2 * pair * sizeof(T), P.xs1, 2 * pair < live, in, raw);
    } else {
      load_planes_odd<T>(x + c0 * P.xs1, 2 * pair * sizeof(T), P.xs1, live - 2 * pair, in, raw);
      late = live - 2 * pair == 1;
    }
  }
  template <int P> __device__ __forceinline__ void put(uint4 (&xb)[2][4][64], unsigned (&xs)[4][64]) {
    const int pair = threadIdx.x & 63, kl = wave_id();
    const int sub = (pair >> 5) * 2, at = (kl & 1) * 32 + (pair & 31);
    uint4 f[2];
    unsigned byte[2];
    if constexpr (!VEC) move_pair<T>(raw, late);
    quantize_raw(raw, f, byte);
#pragma unroll
    for (int px = 0; px < 2; ++px) {
      xb[kl >> 1][sub + px][at] = f[px];
      ((unsigned char *)&xs[sub + px][at])[2 * P + (kl >> 1)] = (unsigned char)byte[px];
    }
  }
};
// rows: eight pieces of 8 elements, four lanes per block
template <typename T, bool VEC> struct Chunk<T, false, VEC> {
  typedef T piece __attribute__((ext_vector_type(8)));
  piece v[8];
  __device__ __forceinline__ void load(const Product &P, const T *x, int live, int chunk) {
    const int t = threadIdx.x;
    const int row = t >> 4;
    const unsigned offset = (unsigned)(row * P.xs1 + (t & 15) * 8) * sizeof(T);
    const T *base = x + chunk * 128ll;
    const long long n = P.k - chunk * 128ll - (t & 15) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T *q = base + i * 16 * P.xs1;
      if (VEC && row + 16 * i < live && n >= 8) {
        v[i] = at<piece>(q, offset);
      } else if (row + 16 * i < live && n > 0) {   // value by value: those beyond the row read its last again
        const T *single = x + (row + 16 * i) * P.xs1 + chunk * 128ll + (t & 15) * 8;
#pragma unroll
        for (int u = 0; u < 8; ++u) v[i][u] = single[u < n ? u : n - 1];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[i][u] = u < n ? v[i][u] : (T)0.0f;
      } else {
        v[i] = piece{};
      }
    }
  }
  template <int P> __device__ __forceinline__ void put(uint4 (&xb)[2][4][64], unsigned (&xs)[4][64]) const {
    const int t = threadIdx.x, quarter = t & 3, block = (t >> 2) & 3;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = (t >> 4) + 16 * i, at = (block & 1) * 32 + (row & 31);
      float e[8];
      unsigned m = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        e[u] = to_float(v[i][u]);
        m = max(m, __float_as_uint(e[u]) & 0x7fffffffu);
      }
      m = max(m, __shfl_xor(m, 1));
      m = max(m, __shfl_xor(m, 2));
      const unsigned byte = scale_byte(m);
      ((unsigned *)&xb[block >> 1][row >> 5][at])[quarter] = pack8(e, scale_value(byte));
      if (quarter == 0) ((unsigned char *)&xs[row >> 5][at])[2 * P + (block >> 1)] = (unsigned char)byte;
    }
  }
};

template <typename T, typename Y, bool PLANES, bool VEC, int NT>
__global__ __launch_bounds__(256, sizeof(Y) == 2 && NT <= (PLANES ? 2 : 1) ? 3 : 2) void mx_stream_kernel(const Product P, int act, int splits, long long tiles, int vec_y) {
  __shared__ uint4 xb[2][2][4][64];
  __shared__ unsigned xs[2][4][64];
  __shared__ uint4 wb[2][2][2 * NT][64];
  __shared__ unsigned wsb[2][(NT + 1) / 2 * 4][64];   // a multiple of the waves
  const int lane = threadIdx.x & 63, wave = wave_id(), wp = wave & 1, wn = wave >> 1;
  // workgroups go round the eight XCDs: the parts of one tile of positions are eight apart, so that they share an L2
  const long long tile = (long long)(blockIdx.x / (8 * splits)) * 8 + (blockIdx.x & 7);
  const int part = (int)(blockIdx.x / 8) % splits;
  if (tile >= tiles) return;
  const long long image = tile / P.tiles_pixels;
  const long long p0 = (tile - image * P.tiles_pixels) * kChunkTile;
  const int live = (int)(P.pixels - p0 < kChunkTile ? P.pixels - p0 : kChunkTile);
  const int S = P.all_steps, chunks = (S + 1) / 2, nt0 = part * 2 * NT;

  // What a wave brings of a chunk: of one of its two steps NT weight fragments, and of four steps their words of scale bytes.
  // Pointers move on from chunk to chunk.
  constexpr int NW = (NT + 1) / 2;
  const int step = wave & 1, wl = weight_lane(lane);   // the weights are put in the order of use: reads of LDS stay linear
  const uint4 *w_src[NT];
  const unsigned *ws_src[NW];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int nt = nt0 + 2 * j + (wave >> 1);
    w_src[j] = P.w + ((long long)step * P.tiles_n + (nt < P.tiles_n ? nt : P.tiles_n - 1)) * 64;
  }
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    const int nt = nt0 + 4 * j + wave;
    ws_src[j] = P.ws + (nt < P.tiles_n ? nt : P.tiles_n - 1) * 64ll;
  }
  u4 w_reg[NT];
  unsigned ws_reg[NW];
  auto load_part = [&](int c, auto parity) {
    if (2 * c + step < S) {   // the second step of the last chunk may be missing: not used then
#pragma unroll
      for (int j = 0; j < NT; ++j) w_reg[j] = at<u4>(w_src[j], wl * 16);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) w_src[j] += 128ll * P.tiles_n;
    if constexpr (decltype(parity)::value == 0) {   // a word of scale bytes serves two chunks
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        ws_reg[j] = at<unsigned>(ws_src[j], wl * 4);
        ws_src[j] += 64ll * P.tiles_n;
      }
    }
  };

  f16x acc[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) start_sums(P, nt0 + wn * NT + t, lane, acc[t]);

  const T *x = (const T *)P.x + image * P.xb + (PLANES ? p0 : p0 * P.xs1);
  Chunk<T, PLANES, VEC> hold;
  load_part(0, std::integral_constant<int, 0>());
  hold.load(P, x, live, 0);

  // Chunk c goes through buffer c & 1, which was read for c - 2 last: every wave is past the barrier of c - 1 by now.
  auto chunk = [&](int c, auto parity) {
    constexpr int B = decltype(parity)::value;
#pragma unroll
    for (int j = 0; j < NT; ++j) *(u4 *)&wb[B][step][2 * j + (wave >> 1)][lane] = w_reg[j];
#pragma unroll
    for (int j = 0; j < NW; ++j) wsb[B][4 * j + wave][lane] = ws_reg[j];
    hold.template put<B>(xb[B], xs[B]);
    if (c + 1 < chunks) {
      load_part(c + 1, std::integral_constant<int, 1 - B>());
      hold.load(P, x, live, c + 1);
    }
    __syncthreads();
    const unsigned sb0 = xs[B][2 * wp][lane], sb1 = xs[B][2 * wp + 1][lane];
    unsigned sa[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) sa[t] = wsb[B][wn * NT + t][lane];
    {
      const uint4 b0 = xb[B][0][2 * wp][lane], b1 = xb[B][0][2 * wp + 1][lane];
#pragma unroll
      for (int t = 0; t < NT; ++t) mfma2<2 * B>(acc[t], wb[B][0][wn * NT + t][lane], sa[t], b0, b1, sb0, sb1);
    }
    if (2 * c + 1 < S) {
      const uint4 b0 = xb[B][1][2 * wp][lane], b1 = xb[B][1][2 * wp + 1][lane];
#pragma unroll
      for (int t = 0; t < NT; ++t) mfma2<2 * B + 1>(acc[t], wb[B][1][wn * NT + t][lane], sa[t], b0, b1, sb0, sb1);
    }
  };
  for (int c = 0; c < chunks; c += 2) {
    chunk(c, std::integral_constant<int, 0>());
    if (c + 1 < chunks) chunk(c + 1, std::integral_constant<int, 1>());
  }

  Y *y = (Y *)P.y + image * P.pixels * P.n;
  const int live_w = live - 64 * wp;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int nt = nt0 + wn * NT + t;
    if (nt < P.tiles_n) {
      if constexpr (PLANES) store_planes<Y>(P, y, p0 + 64 * wp, live_w, nt, lane, act, VEC, acc[t]);
      else store_rows<Y>(P, y, p0 + 64 * wp, live_w, nt, lane, act, vec_y, acc[t]);
    }
  }
}

template <typename T, typename Y, bool PLANES, bool VEC> void launch_stream(Product P, int act, long long batch, hipStream_t st) {
  P.tiles_pixels = (unsigned)((P.pixels + kChunkTile - 1) / kChunkTile);
  const long long tiles = batch * P.tiles_pixels;
  // as many weight rows per workgroup as the registers hold beside a chunk (fp32 and rows read value by value hold more): 1280 -> 320 on 64 maps of 80 x 80
  // with 5 tiles per wave 302 us, with 3 or 4 and the activations read twice through the L2 415;
  // fp32 rows with 4 spill 100 bytes a lane and are faster all the same: 102400 x 1280 -> 256 183 us, 208 with 3
  constexpr int kMaxNT = PLANES && sizeof(Y) == 2 ? 5 : VEC || PLANES ? 4 : 3;
  int splits = (P.tiles_n + 2 * kMaxNT - 1) / (2 * kMaxNT);
  while (tiles * splits < 256 && splits * 2 <= P.tiles_n) splits *= 2;
  int nt = (P.tiles_n + 2 * splits - 1) / (2 * splits);
  splits = (P.tiles_n + 2 * nt - 1) / (2 * nt);
  const int vec_y = (uintptr_t)P.y % 16 == 0 && P.n * sizeof(Y) % 16 == 0;
  const unsigned grid = (unsigned)((tiles + 7) / 8 * 8 * splits);
  if (nt == 1) mx_stream_kernel<T, Y, PLANES, VEC, 1><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 2) mx_stream_kernel<T, Y, PLANES, VEC, 2><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 3) mx_stream_kernel<T, Y, PLANES, VEC, 3><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if constexpr (kMaxNT > 3) {
    if (nt == 4) mx_stream_kernel<T, Y, PLANES, VEC, 4><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
    else mx_stream_kernel<T, Y, PLANES, VEC, kMaxNT><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  }
}

// Quantised rows: 64 * WP of them x 32 * NT * 4 / WP weight rows per workgroup, a wave 64 x 32 * NT.  The weights go through LDS; a wave's rows, which
// at most one other wave needs, come straight into the operands, a chunk of two steps ahead: with both through LDS its traffic (84 KB
// per chunk for 655 k products of 64) kept it as busy as the matrix units, 8192 x 2560 -> 2560 took a tenth longer.  It takes 43 us.  What
// bounds it: the matrix units are busy for half of the time of a deep product (3.8 of the 8.9 PFLOP/s that a loop of
// nothing else reaches: 8192 x 10240 -> 2560 in 114 us, 1.2 us per chunk), the rest are the waits of two workgroups per CU for
// each other's loads; touching lines two chunks ahead, chunks in two sets of registers with smaller tiles, and priorities changed
// nothing or cost; the first loads and 42 MB of results take 19 of the 43 us (the line through k = 2560 and 10240, at k = 0).
template <typename Y, int NT, int WP>
__global__ __launch_bounds__(256, 2) void mx_rows_kernel(const Product P, int act, int splits, long long tiles, int vec_y) {
  constexpr int WN = 4 / WP, NG = NT * WN, NF = (NG + 1) / 2, NW = (NG + 3) / 4;
  __shared__ uint4 wb[2][2][2 * NF][64];
  __shared__ unsigned wsb[2][4 * NW][64];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const long long tile = (long long)(blockIdx.x / (8 * splits)) * 8 + (blockIdx.x & 7);
  const int part = (int)(blockIdx.x / 8) % splits;
  if (tile >= tiles) return;
  const int wp = wave & (WP - 1), wn = wave / WP;
  const long long p0 = (tile * WP + wp) * 64;
  const int S = P.all_steps, nt0 = part * NG;
  const int step = wave & 1, wl = weight_lane(lane);
  const long long groups = (P.pixels + 31) >> 5;
  const uint4 *w_src[NF], *x_src[2];
  const unsigned *ws_src[NW], *xs_src[2];
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int nt = nt0 + 2 * j + (wave >> 1);
    w_src[j] = P.w + ((long long)(step < S ? step : 0) * P.tiles_n + (nt < P.tiles_n ? nt : P.tiles_n - 1)) * 64;
  }
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    const int nt = nt0 + 4 * j + wave;
    ws_src[j] = P.ws + (nt < P.tiles_n ? nt : P.tiles_n - 1) * 64ll;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long g = (p0 >> 5) + h, in = g < groups ? g : groups - 1;
    x_src[h] = (const uint4 *)P.x + in * 64;
    xs_src[h] = P.xs + in * 64;
  }
  u4 w_reg[NF], x_reg[2][2][2];
  unsigned ws_reg[NW], xs_next[2], xs_now[2];
  const int last = S - 1;
  // Loads chunk c; nothing is loaded under a condition, so that the waits in the loop count what is on its way: beyond the last step the
  // pointers stay, and what they read is not used.
  auto load = [&](int c, auto parity) {
    constexpr int B = decltype(parity)::value;
#pragma unroll
    for (int j = 0; j < NF; ++j) w_reg[j] = at<u4>(w_src[j], wl * 16);
    const long long w_move = 2 * c + 2 + step <= last ? 128ll * P.tiles_n : 0;
#pragma unroll
    for (int j = 0; j < NF; ++j) w_src[j] += w_move;
    if constexpr (B == 0) {
      const bool more = 2 * c + 4 <= last;
      const long long ws_move = more ? 64ll * P.tiles_n : 0, xs_move = more ? 64 * groups : 0;
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        ws_reg[j] = at<unsigned>(ws_src[j], wl * 4);
        ws_src[j] += ws_move;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        xs_next[h] = at<unsigned>(xs_src[h], lane * 4);
        xs_src[h] += xs_move;
      }
    }
    const long long second = 2 * c + 1 <= last ? 64 * groups : 0, x_move = 2 * c + 2 <= last ? 128 * groups : 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      x_reg[B][0][h] = at<u4>(x_src[h], lane * 16);
      x_reg[B][1][h] = at<u4>(x_src[h] + second, lane * 16);
      x_src[h] += x_move;
    }
  };
  f16x acc[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) start_sums(P, nt0 + wn * NT + t, lane, acc[t]);
  load(0, std::integral_constant<int, 0>());
  auto put = [&](auto parity) {
    constexpr int B = decltype(parity)::value;
#pragma unroll
    for (int j = 0; j < NF; ++j) *(u4 *)&wb[B][step][2 * j + (wave >> 1)][lane] = w_reg[j];
#pragma unroll
    for (int j = 0; j < NW; ++j) wsb[B][4 * j + wave][lane] = ws_reg[j];
    if constexpr (B == 0) xs_now[0] = xs_next[0], xs_now[1] = xs_next[1];
    __syncthreads();
  };
  unsigned sa[NT];
  auto multiply = [&](auto number) {   // step `number` of four
    constexpr int N = decltype(number)::value, B = N >> 1;
    if constexpr ((N & 1) == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) sa[t] = wsb[B][wn * NT + t][lane];
    }
    const uint4 b0 = __builtin_bit_cast(uint4, x_reg[B][N & 1][0]), b1 = __builtin_bit_cast(uint4, x_reg[B][N & 1][1]);
#pragma unroll
    for (int t = 0; t < NT; ++t) mfma2<N>(acc[t], wb[B][N & 1][wn * NT + t][lane], sa[t], b0, b1, xs_now[0], xs_now[1]);
  };
  constexpr std::integral_constant<int, 0> i0;
  constexpr std::integral_constant<int, 1> i1;
  constexpr std::integral_constant<int, 2> i2;
  constexpr std::integral_constant<int, 3> i3;
  int c = 0;
  for (; 2 * c + 3 < S; c += 2) {   // four steps at a time
    put(i0);
    load(c + 1, i1);
    if constexpr (WP == 2) __builtin_amdgcn_sched_barrier(0);   // loads leave first: 512 x 2560 -> 2560 13.4 us, 14.6 without; at WP = 4 they cost what they gain
    multiply(i0);
    multiply(i1);
    put(i1);
    load(c + 2, i0);
    if constexpr (WP == 2) __builtin_amdgcn_sched_barrier(0);
    multiply(i2);
    multiply(i3);
  }
  if (2 * c < S) {   // up to three more
    put(i0);
    load(c + 1, i1);
    if constexpr (WP == 2) __builtin_amdgcn_sched_barrier(0);   // loads leave first: 512 x 2560 -> 2560 13.4 us, 14.6 without; at WP = 4 they cost what they gain
    multiply(i0);
    if (2 * c + 1 < S) multiply(i1);
    if (2 * c + 2 < S) {
      put(i1);
      multiply(i2);
    }
  }
  const long long live = P.pixels - p0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    if (nt0 + wn * NT + t < P.tiles_n && live > 0) store_rows<Y>(P, (Y *)P.y, p0, (int)(live < 64 ? live : 64), nt0 + wn * NT + t, lane, act, vec_y, acc[t]);
}

template <typename Y, int WP> void launch_rows(const Product &P, int act, hipStream_t st) {
  constexpr int WN = 4 / WP;
  const long long tiles = (P.pixels + 64 * WP - 1) / (64 * WP);
  int splits = (P.tiles_n + 5 * WN - 1) / (5 * WN);   // as many weight tiles as the registers hold
  while (tiles * splits < 256 && splits * 2 * WN <= P.tiles_n * 2) splits *= 2;
  const int nt = (P.tiles_n + WN * splits - 1) / (WN * splits);
  splits = (P.tiles_n + WN * nt - 1) / (WN * nt);
  const int vec_y = (uintptr_t)P.y % 16 == 0 && P.n * sizeof(Y) % 16 == 0;
  const unsigned grid = (unsigned)((tiles + 7) / 8 * 8 * splits);
  if (nt == 1) mx_rows_kernel<Y, 1, WP><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 2) mx_rows_kernel<Y, 2, WP><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 3) mx_rows_kernel<Y, 3, WP><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 4) mx_rows_kernel<Y, 4, WP><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else mx_rows_kernel<Y, 5, WP><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
}

// Few positions: 64 of them x 32 weight rows per workgroup, its eight waves share k.  A wave loads its steps' blocks straight into the
// operands -- no LDS, no barrier before the sums meet; a workgroup's time is the latency of a load or two: a row of 1280 -> 1000 6.5 us, 640 -> 640
// on 20 x 20 7.2.  The row forms spill 16 (bf16) to 48 bytes a lane (fp32), held to four waves per SIMD.
constexpr int kFewWaves = 8;
// Up to this many pairs of tiles, two workgroups per CU (us here and streamed, fp16: 640 -> 320 on 40 x 40, 25 x 10 of them, 7.9 and 9.9;
// 320 -> 160 on 80 x 80, 100 x 5, 7.1 and 7.6; 4 x 640 -> 640 on 20 x 20, 28 x 20, 12.6 and 10.7; 4 x 320 -> 320 on 40 x 40, 100 x 10, 12.1 and
// 9.5; 2000 rows of 1280 -> 160, 32 x 5, 10.4 and 24); quantised rows stream sooner (512 x 5120 -> 640, 8 x 20: 11 and 20; 2048 x 320 ->
// 320, 32 x 10: 6.2 and 4.5)
constexpr long long kFewTiles = 512, kFewTilesPacked = 320;

// blocks kb = 2 * step + (lane >> 5) of the lane's two positions
template <typename T, bool PLANES, bool VEC>
__device__ __forceinline__ void load_few(const Product &P, const T *x, long long p0, int live, int step, int lane, uint4 (&f)[2], unsigned (&byte)[2]) {
  const int j = lane & 31;
  if constexpr (__is_same(T, Packed)) {
    const long long groups = (P.pixels + 31) >> 5;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long group = (p0 >> 5) + h;
      const bool in = 32 * h < live;   // rows of the last group that lie beyond are zeros
      f[h] = in ? ((const uint4 *)P.x)[(step * groups + group) * 64 + lane] : make_uint4(0, 0, 0, 0);
      byte[h] = in ? (P.xs[(step / 4 * groups + group) * 64 + lane] >> (8 * (step & 3))) & 255u : 0u;
    }
  } else {
    const long long c0 = step * 64ll + (lane >> 5) * 32;
    const int in = (int)(P.k - c0 < 0 ? 0 : P.k - c0 < 32 ? P.k - c0 : 32);
    if constexpr (PLANES) {
      Raw<T> raw;
      const T *base = x + step * 64ll * P.xs1;
      const unsigned offset = (unsigned)((lane >> 5) * 32 * P.xs1 + 2 * j) * sizeof(T);
      if constexpr (VEC) {
        load_planes<T, false>(base, offset, P.xs1, 2 * j < live, in, raw);
      } else {
        load_planes_odd<T, false>(base, offset, P.xs1, live - 2 * j, in, raw);
        move_pair<T>(raw, live - 2 * j == 1);
      }
      quantize_raw(raw, f, byte);
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int px = 32 * h + j;
      const T *q = (const T *)((const char *)(x + step * 64ll) + (unsigned)((lane >> 5) * 32 + px * P.xs1) * sizeof(T));
      float v[32];
      if (VEC && px < live && in == 32) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float e[8];
          load8<T, true>(q + 8 * u, 8, e);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[8 * u + i] = e[i];
        }
      } else if (px < live && in == 32) {
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = to_float(q[u]);
      } else if (px < live && in > 0) {   // all loads at once: elements beyond the last read the first again
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = to_float(q[u < in ? u : 0]);
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = u < in ? v[u] : 0.0f;
      } else {
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = 0.0f;
      }
      f[h] = quantize_block(v, byte[h]);
    }
  }
}

template <typename T, typename Y, bool PLANES, bool VEC>
__global__ __launch_bounds__(64 * kFewWaves, 4) void mx_few_kernel(const Product P, int act) {
  __shared__ float part[kFewWaves][32][64];
  const int lane = threadIdx.x & 63, wave = wave_id(), S = P.all_steps;
  const long long image = blockIdx.x / P.tiles_pixels;
  const long long p0 = (long long)(blockIdx.x % P.tiles_pixels) * kTile;
  const int live = (int)(P.pixels - p0 < kTile ? P.pixels - p0 : kTile);
  const int nt = blockIdx.y, wl = weight_lane(lane);
  const uint4 *w = P.w + nt * 64ll + wl;
  const unsigned *ws = P.ws + nt * 64ll + wl;
  f16x acc[2] = {};
  for (int s = wave; s < S; s += kFewWaves) {
    const uint4 a = w[s * 64ll * P.tiles_n];
    const unsigned sa = ws[(s >> 2) * 64ll * P.tiles_n] >> (8 * (s & 3));
    uint4 f[2];
    unsigned byte[2];
    if constexpr (__is_same(T, Packed)) load_few<T, PLANES, VEC>(P, nullptr, p0, live, s, lane, f, byte);
    else load_few<T, PLANES, VEC>(P, (const T *)P.x + image * P.xb + (PLANES ? p0 : p0 * P.xs1), p0, live, s, lane, f, byte);
    mfma2<0>(acc, a, sa, f[0], f[1], byte[0], byte[1]);
  }
  const int waves = S < kFewWaves ? S : kFewWaves;
  constexpr int R = 2048 / (64 * kFewWaves);   // results per thread
  float bias[R] = {};
  if (P.bias) {   // on their way before the sums meet
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long n = nt * 32ll + 16 * (lane >> 5) + ((r * kFewWaves + wave) & 15);
      bias[r] = P.bias[n < P.n ? n : P.n - 1];
    }
  }
  if (wave < waves) {
#pragma unroll
    for (int i = 0; i < 32; ++i) part[wave][i][lane] = acc[i >> 4][i & 15];
  }
  __syncthreads();
  Y *y = (Y *)P.y + image * P.pixels * P.n;
#pragma unroll
  for (int r = 0; r < R; ++r) {   // sums of the waves, in their order
    const int i = r * kFewWaves + wave;
    const int px = PLANES ? 2 * (lane & 31) + (i >> 4) : 32 * (i >> 4) + (lane & 31);
    const long long n = nt * 32ll + 16 * (lane >> 5) + (i & 15);
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < kFewWaves; ++q) v += q < waves ? part[q][i][lane] : 0.0f;
    if (px < live && n < P.n) {
      v += bias[r];
      if (act) v = activate<LMI_ACT_SILU>(v);
      y[PLANES ? n * P.pixels + p0 + px : (p0 + px) * P.n + n] = (Y)v;
    }
  }
}

template <typename T, typename Y, bool PLANES, bool VEC> int launch_by_size(Product P, int act, long long batch, hipStream_t st) {
  P.tiles_pixels = (unsigned)((P.pixels + kTile - 1) / kTile);
  const long long tiles = batch * P.tiles_pixels;
  if (tiles * P.tiles_n <= (__is_same(T, Packed) ? kFewTilesPacked : kFewTiles)) {
    mx_few_kernel<T, Y, PLANES, VEC><<<dim3((unsigned)tiles, (unsigned)P.tiles_n), 64 * kFewWaves, 0, st>>>(P, act);
    return lmi_check_launch("lmi_mx_product");
  }
  if constexpr (PLANES) {
    if (P.all_steps == 1 && tiles >= 512) {
      launch_wave_planes<T, VEC>(P, act, batch, st);
      return lmi_check_launch("lmi_mx_product");
    }
  }
  if constexpr (__is_same(T, Packed)) {
    // 256 rows per workgroup where that leaves work for half of the CUs: 4096 x 1280 -> 1280 12.1 us, 13.2 with 128; 512 x 2560 -> 2560 19 and 13
    if (P.pixels >= 1024 && (P.pixels + 255) / 256 * ((P.tiles_n + 4) / 5) >= 128) launch_rows<Y, 4>(P, act, st);
    else launch_rows<Y, 2>(P, act, st);
  } else {
    launch_stream<T, Y, PLANES, VEC>(P, act, batch, st);
  }
  return lmi_check_launch("lmi_mx_product");
}

// VEC: rows, whole 16-byte words (quantised ones are nothing else); planes, an even size
template <typename T, typename Y, bool PLANES> int launch_product(const Product &P, int act, long long batch, hipStream_t st) {
  if constexpr (__is_same(T, Packed)) {
    return launch_by_size<T, Y, PLANES, true>(P, act, batch, st);
  } else {
    const bool vec = PLANES ? P.pixels % 2 == 0 : (uintptr_t)P.x % 16 == 0 && P.xb * sizeof(T) % 16 == 0 && P.xs1 * sizeof(T) % 16 == 0;
    if (vec) return launch_by_size<T, Y, PLANES, true>(P, act, batch, st);
    return launch_by_size<T, Y, PLANES, false>(P, act, batch, st);
  }
}

bool float_type(int d) { return d == LMI_F32 || d == LMI_F16 || d == LMI_BF16; }

struct Units {
  unsigned steps, quads, grid;
  long long units;
};
// sizes of the quantising kernels' work; false: too large
bool units_of(int64_t rows, int64_t k, Units &u) {
  if (k >= (1ll << 36) || rows >= (1ll << 36)) return false;
  const int64_t steps = (k + 63) / 64, quads = (steps + 3) / 4, octets = (rows + 31) / 32 * 4;
  if (steps >= (1ll << 30) || octets >= (1ll << 40) / quads) return false;
  u.steps = (unsigned)steps;
  u.quads = (unsigned)quads;
  u.units = octets * quads;
  const int64_t wanted = (u.units + 3) / 4;
  u.grid = (unsigned)(wanted < (1 << 23) ? wanted : (1 << 23));
  return true;
}

template <typename T> void quantize(const void *x, int64_t rows, int64_t k, int64_t stride, const Units &u, void *packed, void *scales, hipStream_t st) {
  const bool vec = lmi_is_aligned(x, 16) && stride * sizeof(T) % 16 == 0;
  if (vec) mx_quantize_kernel<T, true><<<u.grid, 256, 0, st>>>((const T *)x, rows, k, stride, u.steps, u.quads, u.units, (unsigned *)packed, (unsigned *)scales);
  else mx_quantize_kernel<T, false><<<u.grid, 256, 0, st>>>((const T *)x, rows, k, stride, u.steps, u.quads, u.units, (unsigned *)packed, (unsigned *)scales);
}
template <typename T> void dequantize(const void *packed, const void *scales, int64_t rows, int64_t k, const Units &u, void *out, hipStream_t st) {
  const bool vec = lmi_is_aligned(out, 16) && k * sizeof(T) % 16 == 0;
  const long long units = u.units / u.quads * u.steps, wanted = (units + 3) / 4;   // octets x steps
  mx_dequantize_kernel<<<(unsigned)(wanted < (1 << 23) ? wanted : (1 << 23)), 256, 0, st>>>((const unsigned *)packed, (const unsigned *)scales, rows, k, u.steps, units, vec, (T *)out);
}

// bytes of a quantised tensor's parts
struct Sizes {
  int64_t packed, scales;
  Sizes(int64_t rows, int64_t k) {
    const int64_t groups = (rows + 31) / 32, steps = (k + 63) / 64;
    packed = groups * steps * 1024;
    scales = groups * ((steps + 3) / 4) * 256;
  }
};

// Rows that come as floats and meet many weight rows are quantised once, into the workspace, where they would be quantised again for
// every 320 weight rows or fewer: 8192 x 1280 -> 2560 (fp16) 34 us, 59 without; 102400 x 1280 -> 640 149 and 183; 128 x 1280 -> 32000 42 and
// 156.  From 320 pairs of tiles on that pays whichever kernel multiplies then (2048 x 1280 -> 320, 320 pairs, both times mx_few_kernel: 10.7 us, as
// floats 15.4; k = 2560 14.3 and 25.5; k = 256 8.6 and 7.4).  Fewer pairs, 256 weight rows or k <= 128 do not pay for the second kernel: 102400 x 1280 -> 160 98 us, 79 without; 8192 x 96 -> 640 11.4 and 9.9.
constexpr int64_t kQuantiseN = 256, kQuantiseK = 128;
bool quantise_first(const lmi_mx_product_args *a) {
  if (a->layout != LMI_MX_ROWS || !float_type(a->x_dtype) || a->batch < 1 || a->n <= kQuantiseN || a->k <= kQuantiseK) return false;
  if (a->batch > 1 && a->x_batch != a->pixels * a->x_stride) return false;   // the rows of the next image do not follow
  if (a->batch >= (1 << 24) || a->pixels < 1 || a->pixels > (1 << 30) / a->batch || a->k >= (1 << 24)) return false;
  return (a->batch * a->pixels + kTile - 1) / kTile * ((a->n + 31) / 32) >= kFewTilesPacked;
}

}  // namespace

extern "C" {

int lmi_mx_quantize(const void *x, int dtype, int64_t rows, int64_t k, int64_t row_stride, uint8_t *packed, uint8_t *scales, void *stream) {
  LMI_REQUIRE(rows >= 0 && k > 0 && row_stride >= 0, LMI_ERR_BAD_ARG, "lmi_mx_quantize: %lld rows of %lld elements", (long long)rows, (long long)k);
  LMI_REQUIRE(float_type(dtype), LMI_ERR_BAD_ARG, "lmi_mx_quantize: x must be fp32, fp16 or bf16");
  if (rows == 0) return LMI_OK;
  LMI_REQUIRE(x && packed && scales, LMI_ERR_BAD_ARG, "lmi_mx_quantize: null pointer");
  LMI_REQUIRE(lmi_is_aligned(packed, 16) && lmi_is_aligned(scales, 4), LMI_ERR_ALIGNMENT, "lmi_mx_quantize: packed must be 16-byte, scales 4-byte aligned");
  Units u;
  LMI_REQUIRE(units_of(rows, k, u), LMI_ERR_LIMIT, "lmi_mx_quantize: too many elements");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LMI_F32) quantize<float>(x, rows, k, row_stride, u, packed, scales, st);
  else if (dtype == LMI_F16) quantize<_Float16>(x, rows, k, row_stride, u, packed, scales, st);
  else quantize<__bf16>(x, rows, k, row_stride, u, packed, scales, st);
  return lmi_check_launch("lmi_mx_quantize");
}

int lmi_mx_dequantize(const uint8_t *packed, const uint8_t *scales, int64_t rows, int64_t k, void *out, int out_dtype, void *stream) {
  LMI_REQUIRE(rows >= 0 && k > 0, LMI_ERR_BAD_ARG, "lmi_mx_dequantize: %lld rows of %lld elements", (long long)rows, (long long)k);
  LMI_REQUIRE(float_type(out_dtype), LMI_ERR_BAD_ARG, "lmi_mx_dequantize: out must be fp32, fp16 or bf16");
  if (rows == 0) return LMI_OK;
  LMI_REQUIRE(packed && scales && out, LMI_ERR_BAD_ARG, "lmi_mx_dequantize: null pointer");
  LMI_REQUIRE(lmi_is_aligned(packed, 16) && lmi_is_aligned(scales, 4), LMI_ERR_ALIGNMENT, "lmi_mx_dequantize: packed must be 16-byte, scales 4-byte aligned");
  Units u;
  LMI_REQUIRE(units_of(rows, k, u), LMI_ERR_LIMIT, "lmi_mx_dequantize: too many elements");
  hipStream_t st = (hipStream_t)stream;
  if (out_dtype == LMI_F32) dequantize<float>(packed, scales, rows, k, u, out, st);
  else if (out_dtype == LMI_F16) dequantize<_Float16>(packed, scales, rows, k, u, out, st);
  else dequantize<__bf16>(packed, scales, rows, k, u, out, st);
  return lmi_check_launch("lmi_mx_dequantize");
}

int64_t lmi_mx_product_workspace_bytes(const lmi_mx_product_args *a) {
  if (!a || !quantise_first(a)) return 0;
  Sizes z(a->batch * a->pixels, a->k);
  return z.packed + z.scales;
}

int lmi_mx_product(const lmi_mx_product_args *a, void *stream) {
  LMI_REQUIRE(a != nullptr, LMI_ERR_BAD_ARG, "lmi_mx_product: args is NULL");
  LMI_REQUIRE(a->batch >= 0 && a->pixels >= 0 && a->k > 0 && a->n > 0, LMI_ERR_BAD_ARG, "lmi_mx_product: batch %lld, pixels %lld, k %lld, n %lld",
              (long long)a->batch, (long long)a->pixels, (long long)a->k, (long long)a->n);
  LMI_REQUIRE(a->act == LMI_ACT_NONE || a->act == LMI_ACT_SILU, LMI_ERR_BAD_ARG, "lmi_mx_product: unknown activation %d", a->act);
  LMI_REQUIRE(a->x_dtype == LMI_MXFP4 || float_type(a->x_dtype), LMI_ERR_BAD_ARG, "lmi_mx_product: x must be fp32, fp16, bf16 or MXFP4");
  LMI_REQUIRE(float_type(a->y_dtype) && (a->x_dtype == LMI_MXFP4 || a->y_dtype == a->x_dtype), LMI_ERR_BAD_ARG,
              "lmi_mx_product: y must be fp32, fp16 or bf16, and of x's type unless x is MXFP4");
  if (a->batch == 0 || a->pixels == 0) return LMI_OK;
  LMI_REQUIRE(a->x && a->w_packed && a->w_scales && a->y, LMI_ERR_BAD_ARG, "lmi_mx_product: null pointer");
  LMI_REQUIRE(a->layout == LMI_MX_ROWS || a->layout == LMI_MX_PLANES, LMI_ERR_BAD_ARG, "lmi_mx_product: unknown layout %d", a->layout);
  const bool rows = a->layout == LMI_MX_ROWS;
  LMI_REQUIRE(a->x_batch >= 0 && a->x_stride >= 0, LMI_ERR_BAD_ARG, "lmi_mx_product: negative stride");
  LMI_REQUIRE(a->x_stride < (1 << 24) && (rows || a->pixels < (1 << 24)), LMI_ERR_LIMIT,
              "lmi_mx_product: rows or channels must lie less than 2^24 elements apart, and a plane hold fewer");
  LMI_REQUIRE(lmi_is_aligned(a->w_packed, 16) && lmi_is_aligned(a->w_scales, 4), LMI_ERR_ALIGNMENT,
              "lmi_mx_product: w_packed must be 16-byte, w_scales 4-byte aligned");
  Product P = {};
  LMI_REQUIRE(rows || a->pixels > 1, LMI_ERR_BAD_ARG, "lmi_mx_product: maps of one position are rows (LMI_MX_ROWS)");
  P.x = a->x;
  P.xs = (const unsigned *)a->x_scales;
  P.pixels = a->pixels;
  P.k = a->k;
  P.n = a->n;
  P.xb = a->x_batch;
  P.xs1 = a->x_stride;
  P.w = (const uint4 *)a->w_packed;
  P.ws = (const unsigned *)a->w_scales;
  P.bias = a->bias;
  P.y = a->y;
  const int64_t blocks = (a->k + LMI_MX_BLOCK - 1) / LMI_MX_BLOCK, tiles_n = (a->n + 31) / 32, tiles_p = (a->pixels + kTile - 1) / kTile;
  LMI_REQUIRE(blocks < (1 << 24) && tiles_n < (1 << 24) && tiles_p < (1 << 24) && a->batch < (1 << 24) && tiles_p * a->batch < (1 << 24), LMI_ERR_LIMIT,
              "lmi_mx_product: k, n or the number of positions is too large");
  P.all_steps = (int)((blocks + 1) / 2);
  P.tiles_n = (int)tiles_n;
  hipStream_t st = (hipStream_t)stream;
  const bool first = quantise_first(a);
  if (first) {
    const int64_t m = a->batch * a->pixels;
    const Sizes z(m, a->k);
    LMI_REQUIRE(a->workspace && a->workspace_bytes >= z.packed + z.scales, LMI_ERR_WORKSPACE, "lmi_mx_product: workspace of %lld bytes, %lld needed",
                (long long)a->workspace_bytes, (long long)(z.packed + z.scales));
    LMI_REQUIRE(lmi_is_aligned(a->workspace, 16), LMI_ERR_ALIGNMENT, "lmi_mx_product: workspace must be 16-byte aligned");
    uint8_t *packed = (uint8_t *)a->workspace, *scales = packed + z.packed;
    const int e = lmi_mx_quantize(a->x, a->x_dtype, m, a->k, a->x_stride, packed, scales, stream);
    if (e != LMI_OK) return e;
    P.x = packed;
    P.xs = (const unsigned *)scales;
    P.pixels = m;
  }
  if (a->x_dtype == LMI_MXFP4) {
    LMI_REQUIRE(rows && a->batch == 1 && a->x_scales && lmi_is_aligned(a->x, 16) && lmi_is_aligned(a->x_scales, 4), LMI_ERR_BAD_ARG,
                "lmi_mx_product: quantised x comes as 16-byte aligned rows with their scales, batch 1");
  }
  if (first || a->x_dtype == LMI_MXFP4) {
    if (a->y_dtype == LMI_F32) return launch_product<Packed, float, false>(P, a->act, 1, st);
    if (a->y_dtype == LMI_F16) return launch_product<Packed, _Float16, false>(P, a->act, 1, st);
    return launch_product<Packed, __bf16, false>(P, a->act, 1, st);
  }
  if (rows) {
    if (a->x_dtype == LMI_F32) return launch_product<float, float, false>(P, a->act, a->batch, st);
    if (a->x_dtype == LMI_F16) return launch_product<_Float16, _Float16, false>(P, a->act, a->batch, st);
    return launch_product<__bf16, __bf16, false>(P, a->act, a->batch, st);
  }
  if (a->x_dtype == LMI_F32) return launch_product<float, float, true>(P, a->act, a->batch, st);
  if (a->x_dtype == LMI_F16) return launch_product<_Float16, _Float16, true>(P, a->act, a->batch, st);
  return launch_product<__bf16, __bf16, true>(P, a->act, a->batch, st);
}

}  // extern "C"
