// MXFP4 (4-bit e2m1 elements, one power-of-two scale per 32) for gfx950: quantising, reading back, and the product of
// quantised weights with activations -- a 1x1 convolution of the network with its folded batch norm and SiLU, or a linear layer.
//
// A block's scale is 2^(floor(log2 max) - 2), so its largest element lands in [4, 8): 6 is the largest magnitude of e2m1, and
// what rounds beyond it stays at 6.  v_cvt_scalef32_pk_fp4_* divides by the scale and rounds to nearest even with that
// saturation; x / 2^e is exact, so nothing is rounded twice.  The products run on v_mfma_scale_f32_32x32x64_f8f6f4 (twice the
// rate of the 16x16x128 form): 64 elements of k per instruction, every lane brings 32 elements of one row and their
// scale byte -- one block --, sums in fp32.  Quantised tensors are kept in that order (see lmi_hip.h), so an operand of a
// wave is one contiguous kilobyte, and the scale bytes of four steps are one word of which the instruction picks a byte.
//
// Kernels
//  mx_quantize_kernel     a wave takes 8 rows x 256 elements: four lanes per block, 8 elements each, four steps per lane.
//  mx_dequantize_kernel   the same shape backwards.
//  mx_product_kernel      64 positions x all of k: activations are read once, quantised in registers (a lane owns whole blocks: 32
//                         channels of one position) and laid into LDS in the matrix instruction's order; then every wave
//                         multiplies them with its share of the weight rows.
#include <hip/hip_fp16.h>

#include <type_traits>

#include "common.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

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

// lane = (row of the octet, block of the step, quarter of the block).  The wave reads 8 rows x 128 bytes (16-bit types) per step and writes 8 x 16
// bytes side by side for either block; the scale bytes of its four steps leave as one word.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *x, long long rows, long long k, long long row_stride, unsigned steps, unsigned quads,
                                                          long long units, unsigned *packed, unsigned *scales) {
  const int lane = threadIdx.x & 63, quarter = lane & 3, half = (lane >> 2) & 1, r8 = lane >> 3;
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
      if (step < steps) packed[(((group * steps + step) * 2 + half) * 32 + rg) * 4 + quarter] = pack8(v[i], scale_value(byte));
    }
    if (quarter == 0) scales[((group * quads + quad) * 2 + half) * 32 + rg] = word;
  }
}

template <typename T> __device__ __forceinline__ void store8(T *p, long long n, bool vec, const float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      ((float4 *)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      ((float4 *)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      t8 a;
#pragma unroll
      for (int u = 0; u < 8; ++u) a[u] = (T)v[u];
      *(t8 *)p = a;
    }
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u < n) p[u] = (T)v[u];
  }
}

// e2m1 code -> value
__device__ __forceinline__ float code_value(unsigned c) {
  const unsigned m = c & 7u;
  const float a = m < 2u ? 0.5f * m : (1.0f + 0.5f * (m & 1u)) * (float)(1u << ((m >> 1) - 1u));
  return (c & 8u) ? -a : a;
}

template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned *packed, const unsigned *scales, long long rows, long long k, unsigned steps,
                                                            unsigned quads, long long units, bool vec, T *out) {
  const int lane = threadIdx.x & 63, quarter = lane & 3, half = (lane >> 2) & 1, r8 = lane >> 3;
  for (long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += (long long)gridDim.x * 4) {
    const long long octet = unit / quads;
    const unsigned quad = (unsigned)(unit - octet * quads);
    const long long row = octet * 8 + r8, group = octet >> 2;
    if (row >= rows) continue;
    const int rg = (int)(octet & 3) * 8 + r8;
    const unsigned word = scales[((group * quads + quad) * 2 + half) * 32 + rg];
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned step = quad * 4 + i;
      w[i] = step < steps ? packed[(((group * steps + step) * 2 + half) * 32 + rg) * 4 + quarter] : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long c0 = ((long long)quad * 4 + i) * 64 + half * 32 + quarter * 8;
      const unsigned byte = (word >> (8 * i)) & 255u;
      // 2^(byte - 127); the smallest is subnormal, 255 is NaN
      const float s = byte == 255u ? NAN : (byte ? __uint_as_float(byte << 23) : 0x1p-127f);
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = code_value((w[i] >> (4 * u)) & 15u) * s;
      store8(out + row * k + c0, k - c0, vec, v);
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
  unsigned blocks;        // blocks of 32 along k
  unsigned tiles_pixels;  // tiles of 64 positions per image
  int tiles_n;            // tiles of 32 weight rows
  int split_n;            // tiles of 32 weight rows per workgroup
  int all_steps;          // steps of 64 along k
  int steps;              // steps that LDS holds (a multiple of 4, or all)
};

constexpr int kTile = 64;   // positions per workgroup

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

// LDS: fragments [step][subtile][64] uint4, then scale words [step / 4][subtile][64]
template <typename T, bool PLANES, bool VEC>
__device__ __forceinline__ void fill(const Product &P, long long image, long long p0, int live, int s0, int ns, uint4 *frags, unsigned char *bytes) {
  const int t = threadIdx.x;
  auto put = [&](int kl, int px, const uint4 &f, unsigned byte) {
    const int at = (px & 1) * 64 + (kl & 1) * 32 + (px >> 1), step = kl >> 1;
    frags[step * 128 + at] = f;
    bytes[((step >> 2) * 128 + at) * 4 + (step & 3)] = (unsigned char)byte;
  };
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if constexpr (__is_same(T, Packed)) {
    const long long g0 = p0 >> 5;
    for (int item = t; item < ns * 128; item += 256) {
      const int step = item >> 7, at = item & 127, px = at & 63, half = at >> 6;   // px: row of the two groups
      const long long g = g0 + (px >> 5);
      uint4 f = zero;
      if (px < live) f = ((const uint4 *)P.x)[((g * P.all_steps + s0 + step) * 2 + half) * 32 + (px & 31)];
      frags[step * 128 + (px & 1) * 64 + half * 32 + (px >> 1)] = f;
    }
    const int quads = (P.all_steps + 3) / 4;
    for (int item = t; item < (ns + 3) / 4 * 128; item += 256) {   // s0 is a multiple of 4
      const int q = item >> 7, at = item & 127, px = at & 63, half = at >> 6;
      const long long g = g0 + (px >> 5);
      unsigned w = 0;
      if (px < live) w = P.xs[((g * quads + s0 / 4 + q) * 2 + half) * 32 + (px & 31)];
      ((unsigned *)bytes)[q * 128 + (px & 1) * 64 + half * 32 + (px >> 1)] = w;
    }
    return;
  } else {
    const T *x = (const T *)P.x + image * P.xb;
    if constexpr (PLANES && VEC) {   // two neighbouring pixels per thread
      for (int item = t; item < ns * 64; item += 256) {
        const int pair = item & 31, kl = item >> 5;
        const unsigned kb = 2 * s0 + kl;
        uint4 f[2] = {zero, zero};
        unsigned byte[2] = {0, 0};
        if (2 * pair < live && kb < P.blocks) {
          const T *q = x + p0 + 2 * pair + (long long)kb * 32 * P.xs1;
          const int in = (int)(P.k - (long long)kb * 32 < 32 ? P.k - (long long)kb * 32 : 32);
          if constexpr (sizeof(T) == 4) {
            float a[32], b[32];
#pragma unroll
            for (int u = 0; u < 32; ++u) {
              const float2 v = u < in ? *(const float2 *)(q + u * P.xs1) : make_float2(0.0f, 0.0f);
              a[u] = v.x;
              b[u] = v.y;
            }
            f[0] = quantize_block(a, byte[0]);
            f[1] = quantize_block(b, byte[1]);
          } else {
            unsigned w[32];
            if (in == 32) {
#pragma unroll
              for (int u = 0; u < 32; ++u) w[u] = *(const unsigned *)(q + u * P.xs1);
            } else {
#pragma unroll
              for (int u = 0; u < 32; ++u) w[u] = u < in ? *(const unsigned *)(q + u * P.xs1) : 0u;
            }
            quantize_pair16<T>(w, f, byte);
          }
        }
        put(kl, 2 * pair, f[0], byte[0]);
        put(kl, 2 * pair + 1, f[1], byte[1]);
      }
    } else {
      for (int item = t; item < ns * 128; item += 256) {
        const int px = item & 63, kl = item >> 6;
        const unsigned kb = 2 * s0 + kl;
        uint4 f = zero;
        unsigned byte = 0;
        if (px < live && kb < P.blocks) {
          const long long c0 = (long long)kb * 32;
          float v[32];
          if constexpr (PLANES) {
            const T *q = x + p0 + px + c0 * P.xs1;
#pragma unroll
            for (int u = 0; u < 32; ++u) v[u] = c0 + u < P.k ? to_float(q[u * P.xs1]) : 0.0f;
          } else {
            const T *q = x + (p0 + px) * P.xs1 + c0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              float e[8];
              load8<T, VEC>(q + 8 * u, P.k - c0 - 8 * u, e);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[8 * u + j] = e[j];
            }
          }
          f = quantize_block(v, byte);
        }
        put(kl, px, f, byte);
      }
    }
  }
}

__device__ __forceinline__ v8i operand(const uint4 &a) { return v8i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}; }

template <int BYTE> __device__ __forceinline__ void mfma2(f16x (&acc)[2], const uint4 &a, unsigned sa, const uint4 &b0, const uint4 &b1, unsigned sb0, unsigned sb1) {
  acc[0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(a), operand(b0), acc[0], 4, 4, BYTE, (int)sa, BYTE, (int)sb0);
  acc[1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(a), operand(b1), acc[1], 4, 4, BYTE, (int)sa, BYTE, (int)sb1);
}

// One quad of steps of G weight tiles: fragments and scale words
template <int G> struct Quad {
  uint4 a[G][4];
  unsigned s[G];
};
template <int G> __device__ __forceinline__ void load_quad(Quad<G> &Q, const uint4 *w, const unsigned *ws, long long tile_w, long long tile_s, int q, int last) {
#pragma unroll
  for (int g = 0; g < G; ++g) {
    Q.s[g] = ws[g * tile_s + q * 64];
#pragma unroll
    for (int i = 0; i < 4; ++i) Q.a[g][i] = w[g * tile_w + (q * 4 + i < last ? q * 4 + i : last) * 64];   // beyond the last step: any of the tile's, not used
  }
}

// Weight tiles nt .. nt + G - 1 times the ns steps in LDS (steps s0 ..), quads q0, q0 + dq, ...  The next quad's weights are on their way
// while the matrix instructions run; every fragment read from LDS serves G of them.
template <int G>
__device__ __forceinline__ void multiply(const Product &P, int nt, int s0, int ns, int q0, int dq, const uint4 *frags, const unsigned *words, int lane, f16x (&acc)[G][2]) {
  const int wl = weight_lane(lane), quads = (P.all_steps + 3) / 4;
  const uint4 *w = P.w + ((long long)nt * P.all_steps + s0) * 64 + wl;
  const unsigned *ws = P.ws + ((long long)nt * quads + s0 / 4) * 64 + wl;
  const long long tile_w = (long long)P.all_steps * 64, tile_s = (long long)quads * 64;
  if (q0 * 4 >= ns) return;
  Quad<G> cur, next;
  load_quad<G>(cur, w, ws, tile_w, tile_s, q0, ns - 1);
  for (int q = q0; q * 4 < ns; q += dq) {
    if ((q + dq) * 4 < ns) load_quad<G>(next, w, ws, tile_w, tile_s, q + dq, ns - 1);
    const unsigned sb0 = words[q * 128 + lane], sb1 = words[q * 128 + 64 + lane];
    const uint4 *f = frags + q * 512 + lane;
    const int left = ns - q * 4;
    {
      const uint4 b0 = f[0], b1 = f[64];
#pragma unroll
      for (int g = 0; g < G; ++g) mfma2<0>(acc[g], cur.a[g][0], cur.s[g], b0, b1, sb0, sb1);
    }
    if (left > 1) {
      const uint4 b0 = f[128], b1 = f[192];
#pragma unroll
      for (int g = 0; g < G; ++g) mfma2<1>(acc[g], cur.a[g][1], cur.s[g], b0, b1, sb0, sb1);
    }
    if (left > 2) {
      const uint4 b0 = f[256], b1 = f[320];
#pragma unroll
      for (int g = 0; g < G; ++g) mfma2<2>(acc[g], cur.a[g][2], cur.s[g], b0, b1, sb0, sb1);
    }
    if (left > 3) {
      const uint4 b0 = f[384], b1 = f[448];
#pragma unroll
      for (int g = 0; g < G; ++g) mfma2<3>(acc[g], cur.a[g][3], cur.s[g], b0, b1, sb0, sb1);
    }
    cur = next;
  }
}

template <typename Y, bool PLANES, bool VEC, int ACT>
__device__ __forceinline__ void store_tile(const Product &P, long long image, long long p0, int live, int nt, int lane, const f16x (&acc)[2]) {
  Y *y = (Y *)P.y + image * P.pixels * P.n;
  const int px = 2 * (lane & 31);
  const long long n0 = (long long)nt * 32 + 16 * (lane >> 5);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const long long n = n0 + i;
    if (n >= P.n) break;
    const float b = P.bias ? P.bias[n] : 0.0f;
    const Y v0 = (Y)activate<ACT>(acc[0][i] + b), v1 = (Y)activate<ACT>(acc[1][i] + b);
    if constexpr (PLANES) {
      Y *q = y + n * P.pixels + p0 + px;
      if (VEC) {
        typedef Y y2 __attribute__((ext_vector_type(2)));
        if (px < live) *(y2 *)q = y2{v0, v1};
      } else {
        if (px < live) q[0] = v0;
        if (px + 1 < live) q[1] = v1;
      }
    } else {
      if (px < live) y[(p0 + px) * P.n + n] = v0;
      if (px + 1 < live) y[(p0 + px + 1) * P.n + n] = v1;
    }
  }
}

// The weight tiles of a workgroup are dealt to its waves in runs of nearly equal length; which wave gets the longer ones turns with the
// workgroup, so that no SIMD gets them all.  A wave takes its run two tiles at a time.  k longer than LDS holds: the positions are
// quantised again for every round of tiles.
// KSPLIT: one weight tile per workgroup, its waves share k (few positions).
template <typename T, typename Y, bool PLANES, bool VEC, int ACT, bool KSPLIT>
__global__ __launch_bounds__(256, KSPLIT ? 1 : 3) void mx_product_kernel(const Product P) {
  extern __shared__ uint4 lds[];
  uint4 *frags = lds;
  unsigned char *bytes = (unsigned char *)(lds + (long long)P.steps * 128);
  const unsigned *words = (const unsigned *)bytes;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long image = blockIdx.x / P.tiles_pixels;
  const long long p0 = (long long)(blockIdx.x % P.tiles_pixels) * kTile;
  const int live = (int)(P.pixels - p0 < kTile ? P.pixels - p0 : kTile);
  const int nt0 = blockIdx.y * P.split_n;
  const int nt1 = nt0 + P.split_n < P.tiles_n ? nt0 + P.split_n : P.tiles_n;
  const bool once = P.all_steps <= P.steps;
  if constexpr (KSPLIT) {
    f16x acc[1][2] = {};
    for (int s0 = 0; s0 < P.all_steps; s0 += P.steps) {
      const int ns = P.all_steps - s0 < P.steps ? P.all_steps - s0 : P.steps;
      __syncthreads();   // LDS is free again
      fill<T, PLANES, VEC>(P, image, p0, live, s0, ns, frags, bytes);
      __syncthreads();
      multiply<1>(P, nt0, s0, ns, wave, 4, frags, words, lane, acc);
    }
    __syncthreads();   // sums of the four waves, in their order
    float *part = (float *)lds;   // [3][32][64]
    if (wave) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) part[((wave - 1) * 32 + h * 16 + i) * 64 + lane] = acc[0][h][i];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
#pragma unroll
          for (int w = 0; w < 3; ++w) acc[0][h][i] += part[(w * 32 + h * 16 + i) * 64 + lane];
        }
      store_tile<Y, PLANES, VEC, ACT>(P, image, p0, live, nt0, lane, acc[0]);
    }
  } else {
    const int count = nt1 - nt0, turn = (wave + blockIdx.x) & 3;
    const int mine = count / 4 + (turn < count % 4), first = nt0 + turn * (count / 4) + (turn < count % 4 ? turn : count % 4);
    const int rounds = ((count + 3) / 4 + 1) / 2;   // of the longest run
    for (int r = 0; r < rounds; ++r) {
      const int nt = first + 2 * r, have = mine - 2 * r;
      f16x acc[2][2] = {};
      for (int s0 = 0; s0 < P.all_steps; s0 += P.steps) {
        const int ns = P.all_steps - s0 < P.steps ? P.all_steps - s0 : P.steps;
        if (!once || r == 0) {
          __syncthreads();   // LDS is free again
          fill<T, PLANES, VEC>(P, image, p0, live, s0, ns, frags, bytes);
          __syncthreads();
        }
        if (have >= 2) {
          multiply<2>(P, nt, s0, ns, 0, 1, frags, words, lane, acc);
        } else if (have == 1) {
          f16x one[1][2] = {{acc[0][0], acc[0][1]}};
          multiply<1>(P, nt, s0, ns, 0, 1, frags, words, lane, one);
          acc[0][0] = one[0][0];
          acc[0][1] = one[0][1];
        }
      }
      if (have >= 1) store_tile<Y, PLANES, VEC, ACT>(P, image, p0, live, nt, lane, acc[0]);
      if (have >= 2) store_tile<Y, PLANES, VEC, ACT>(P, image, p0, live, nt + 1, lane, acc[1]);
    }
  }
}

// One wave, 64 positions, all of k (at most 128) in registers: what a lane quantises is its operand.  No LDS, no barrier: the waves of
// a CU drift apart, so that some load while others multiply.
constexpr int kWaveSteps = 2;   // deeper ones stream faster: 64 x 192 -> 192 on 80 x 80: 80 us here, 68 streamed; 128 -> 640: 141 and 172; 48 -> 32 on 160 x 160: 56 and 84
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <typename T, bool PLANES> struct Raw;   // one step's values of a lane before they are quantised
template <> struct Raw<float, true> {
  float2 v[32];
};
template <typename T> struct Raw<T, true> {
  unsigned v[32];
};
template <typename T> struct Raw<T, false> {
  float v[8][8];
};

// Addresses are a base that is the same for the wave (scalar registers) plus a 32-bit offset of the lane: the launcher sees to it that
// 32 channels or rows fit.
template <typename W> __device__ __forceinline__ const W *at(const void *base, unsigned offset) { return (const W *)((const char *)base + offset); }

// `in` channels (32 or more: all) of two neighbouring pixels from base + offset on; base is uniform
template <typename T> __device__ __forceinline__ void load_planes(const T *base, unsigned offset, long long stride, bool live, int in, Raw<T, true> &r) {
  typedef typename std::remove_reference<decltype(r.v[0])>::type W;
  if (live && in >= 32) {
#pragma unroll
    for (int u = 0; u < 32; ++u) r.v[u] = *at<W>(base + u * stride, offset);
  } else {   // positions beyond the image, the last channels
#pragma unroll
    for (int u = 0; u < 32; ++u) r.v[u] = live && u < in ? *at<W>(base + u * stride, offset) : W{};
  }
}
__device__ __forceinline__ void quantize_raw(const Raw<float, true> &r, uint4 (&f)[2], unsigned (&byte)[2]) {
  float a[32];
#pragma unroll
  for (int u = 0; u < 32; ++u) a[u] = r.v[u].x;
  f[0] = quantize_block(a, byte[0]);
#pragma unroll
  for (int u = 0; u < 32; ++u) a[u] = r.v[u].y;
  f[1] = quantize_block(a, byte[1]);
}
template <typename T> __device__ __forceinline__ void quantize_raw(const Raw<T, true> &r, uint4 (&f)[2], unsigned (&byte)[2]) { quantize_pair16<T>(r.v, f, byte); }

// the sums of weight tile nt start at the bias
__device__ __forceinline__ void start_sums(const Product &P, int nt, int lane, f16x (&acc)[2]) {
  const long long n0 = (long long)nt * 32 + 16 * (lane >> 5);
  acc[0] = f16x{};
  if (P.bias) {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[0][i] = n0 + i < P.n ? P.bias[n0 + i] : 0.0f;
  }
  acc[1] = acc[0];
}

// planes: a lane holds 16 weight rows' results of two neighbouring positions.  Results are not read again soon: stored past the caches
// (the 160 x 160 maps of a batch of 64, 48 -> 32 channels: 75 -> 56 us with the sums starting at the bias).
template <typename Y>
__device__ __forceinline__ void store_planes(const Product &P, Y *y, long long p0, int live, int nt, int lane, int act, const f16x (&acc)[2]) {
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
    if (px < live && i < left) __builtin_nontemporal_store(y2{(Y)v0, (Y)v1}, (y2 *)((char *)(base + i * P.pixels) + offset));
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

template <typename T>
__global__ __launch_bounds__(256, 4) void mx_wave_planes_kernel(const Product P, int act, long long tiles) {
  const int lane = threadIdx.x & 63;
  const unsigned tile = blockIdx.x * 4 + wave_id();
  if (tile >= tiles) return;
  const long long image = tile / P.tiles_pixels;
  const long long p0 = (long long)(tile % P.tiles_pixels) * kTile;
  const int live = (int)(P.pixels - p0 < kTile ? P.pixels - p0 : kTile);
  const T *x = (const T *)P.x + image * P.xb + p0;
  const unsigned offset = (unsigned)((lane >> 5) * 32 * P.xs1 + 2 * (lane & 31)) * sizeof(T);
  const bool mine = 2 * (lane & 31) < live;
  const int S = P.all_steps, half = lane >> 5;
  uint4 f[kWaveSteps][2];
  unsigned sw[2] = {};
  Raw<T, true> raw;
#pragma unroll
  for (int s = 0; s < kWaveSteps; ++s) {
    if (s < S) {
      const int left = (int)(P.k - 64ll * s) - 32 * half;
      load_planes<T>(x + 64ll * s * P.xs1, offset, P.xs1, mine, left < 0 ? 0 : left, raw);
      unsigned byte[2];
      quantize_raw(raw, f[s], byte);
      sw[0] |= byte[0] << (8 * s);
      sw[1] |= byte[1] << (8 * s);
    }
  }
  const int wl = weight_lane(lane);
  const int nt0 = blockIdx.y * P.split_n;
  const int nt1 = nt0 + P.split_n < P.tiles_n ? nt0 + P.split_n : P.tiles_n;
  T *y = (T *)P.y + image * P.pixels * P.n;
  for (int nt = nt0; nt < nt1; ++nt) {
    f16x acc[2];
    start_sums(P, nt, lane, acc);
    const uint4 *w = P.w + (long long)nt * S * 64 + wl;
    const unsigned sa = P.ws[nt * 64 + wl];
    uint4 a[kWaveSteps];
#pragma unroll
    for (int s = 0; s < kWaveSteps; ++s) a[s] = w[(s < S ? s : S - 1) * 64];
    mfma2<0>(acc, a[0], sa, f[0][0], f[0][1], sw[0], sw[1]);
    if (S > 1) mfma2<1>(acc, a[1], sa, f[1][0], f[1][1], sw[0], sw[1]);
    store_planes<T>(P, y, p0, live, nt, lane, act, acc);
  }
}

template <typename T> bool launch_wave_planes(Product P, int act, long long batch, hipStream_t st) {
  const long long tiles = batch * P.tiles_pixels;
  if (P.all_steps > kWaveSteps || tiles < 512) return false;
  const long long split = tiles < 2048 ? (2048 + tiles - 1) / tiles : 1;
  P.split_n = (int)((P.tiles_n + split - 1) / split);
  const dim3 grid((unsigned)((tiles + 3) / 4), (unsigned)((P.tiles_n + P.split_n - 1) / P.split_n));
  mx_wave_planes_kernel<T><<<grid, 256, 0, st>>>(P, act, tiles);
  return true;
}

// Streaming product: 128 positions x up to 64 * NT weight rows per workgroup, k in chunks of two steps.  While the matrix instructions run
// on one chunk, the next chunk's activations are on their way to registers and its weights on their way to LDS; an
// activation block is quantised by the thread that loaded it.  Waves are dealt 2 (positions) x 2 (weight rows), each 64 positions x 32 * NT
// rows of sums in registers: a fragment read from LDS serves 2 or NT matrix instructions.
constexpr int kChunkTile = 128;

template <typename T, bool PLANES> struct Chunk;   // what a thread holds of a chunk
// planes: two neighbouring pixels x one block
template <typename T> struct Chunk<T, true> {
  Raw<T, true> raw;
  __device__ __forceinline__ void load(const Product &P, const T *x, int live, int chunk) {
    const int pair = threadIdx.x & 63;
    const long long c0 = (4ll * chunk + wave_id()) * 32;
    load_planes<T>(x + c0 * P.xs1, 2 * pair * sizeof(T), P.xs1, 2 * pair < live, c0 < P.k ? (int)(P.k - c0 < 32 ? P.k - c0 : 32) : 0, raw);
  }
  __device__ __forceinline__ void put(uint4 (&xb)[2][4][64], unsigned (&xs)[4][64]) const {
    const int pair = threadIdx.x & 63, kl = wave_id();
    const int sub = (pair >> 5) * 2, at = (kl & 1) * 32 + (pair & 31);
    uint4 f[2];
    unsigned byte[2];
    quantize_raw(raw, f, byte);
#pragma unroll
    for (int px = 0; px < 2; ++px) {
      xb[kl >> 1][sub + px][at] = f[px];
      ((unsigned char *)&xs[sub + px][at])[kl >> 1] = (unsigned char)byte[px];
    }
  }
};
// rows: eight pieces of 8 elements, four lanes per block
template <typename T> struct Chunk<T, false> {
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
      if (row + 16 * i < live && n >= 8) {
        v[i] = *at<piece>(q, offset);
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) v[i][u] = row + 16 * i < live && u < n ? *at<T>(q, offset + u * sizeof(T)) : (T)0.0f;
      }
    }
  }
  __device__ __forceinline__ void put(uint4 (&xb)[2][4][64], unsigned (&xs)[4][64]) const {
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
      if (quarter == 0) ((unsigned char *)&xs[row >> 5][at])[block >> 1] = (unsigned char)byte;
    }
  }
};

// 64 lanes x SIZE bytes from src (per lane) to dst (the wave's base; lane l lands at l * SIZE).  Complete for the workgroup after a
// wait for vmcnt(0) and a barrier.
template <int SIZE> __device__ __forceinline__ void to_lds(const void *src, void *dst) {
  const auto from = (const __attribute__((address_space(1))) void *)src;
  const auto to = (__attribute__((address_space(3))) void *)dst;
  if constexpr (SIZE == 16) __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds(from, to, 4, 0, 0);
}

template <typename T, typename Y, bool PLANES, int NT>
__global__ __launch_bounds__(256, NT <= 2 ? 3 : 2) void mx_stream_kernel(const Product P, int act, int splits, long long tiles, int vec_y) {
  __shared__ uint4 xb[2][2][4][64];
  __shared__ unsigned xs[2][4][64];
  __shared__ uint4 wb[2][2][2 * NT][64];
  __shared__ unsigned wsb[2][2 * NT][64];
  const int lane = threadIdx.x & 63, wave = wave_id(), wp = wave & 1, wn = wave >> 1;
  // workgroups go round the eight XCDs: the parts of one tile of positions are eight apart, so that they share an L2
  const long long tile = (long long)(blockIdx.x / (8 * splits)) * 8 + (blockIdx.x & 7);
  const int part = (int)(blockIdx.x / 8) % splits;
  if (tile >= tiles) return;
  const long long image = tile / P.tiles_pixels;
  const long long p0 = (tile - image * P.tiles_pixels) * kChunkTile;
  const int live = (int)(P.pixels - p0 < kChunkTile ? P.pixels - p0 : kChunkTile);
  const int S = P.all_steps, quads = (S + 3) / 4, chunks = (S + 1) / 2, nt0 = part * 2 * NT;

  auto load_weights = [&](int c, int buf) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {   // 4 * NT fragments over four waves
      const int id = j * 4 + wave, step = id & 1, t = id >> 1;
      const int nt = nt0 + t < P.tiles_n ? nt0 + t : P.tiles_n - 1, s = 2 * c + step < S ? 2 * c + step : S - 1;
      to_lds<16>(P.w + ((long long)nt * S + s) * 64 + lane, &wb[buf][step][t][0]);
    }
#pragma unroll
    for (int j = 0; j < (NT + 1) / 2; ++j) {
      const int t = j * 4 + wave;
      if (t < 2 * NT) {
        const int nt = nt0 + t < P.tiles_n ? nt0 + t : P.tiles_n - 1;
        to_lds<4>(P.ws + ((long long)nt * quads + c / 2) * 64 + lane, &wsb[buf][t][0]);
      }
    }
  };
  const long long g0 = p0 >> 5;   // Packed: first group of rows
  auto load_packed = [&](int c, int buf) {
    const unsigned char *base = (const unsigned char *)P.x;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int id = j * 4 + wave, step = id & 1, sub = id >> 1;
      const long long groups = (P.pixels + 31) >> 5, g = g0 + sub < groups ? g0 + sub : groups - 1;
      const int s = 2 * c + step < S ? 2 * c + step : S - 1;
      to_lds<16>(base + ((g * S + s) * 64 + lane) * 16, &xb[buf][step][sub][0]);
    }
    const long long groups = (P.pixels + 31) >> 5, g = g0 + wave < groups ? g0 + wave : groups - 1;
    to_lds<4>(P.xs + (g * quads + c / 2) * 64 + lane, &xs[buf][wave][0]);
  };

  f16x acc[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) start_sums(P, nt0 + wn * NT + t, lane, acc[t]);
  const int wl = weight_lane(lane);
  auto multiply_chunk = [&](int c, int buf) {
    const int shift = 16 * (c & 1);
    unsigned sb0 = xs[buf][2 * wp][lane], sb1 = xs[buf][2 * wp + 1][lane];
    if constexpr (__is_same(T, Packed)) sb0 >>= shift, sb1 >>= shift;
    unsigned sa[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) sa[t] = wsb[buf][wn * NT + t][wl] >> shift;
    {
      const uint4 b0 = xb[buf][0][2 * wp][lane], b1 = xb[buf][0][2 * wp + 1][lane];
#pragma unroll
      for (int t = 0; t < NT; ++t) mfma2<0>(acc[t], wb[buf][0][wn * NT + t][wl], sa[t], b0, b1, sb0, sb1);
    }
    if (2 * c + 1 < S) {
      const uint4 b0 = xb[buf][1][2 * wp][lane], b1 = xb[buf][1][2 * wp + 1][lane];
#pragma unroll
      for (int t = 0; t < NT; ++t) mfma2<1>(acc[t], wb[buf][1][wn * NT + t][wl], sa[t], b0, b1, sb0, sb1);
    }
  };

  if constexpr (__is_same(T, Packed)) {
    load_weights(0, 0);
    load_packed(0, 0);
    for (int c = 0; c < chunks; ++c) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this chunk's weights and rows are in LDS
      __syncthreads();
      if (c + 1 < chunks) {
        load_weights(c + 1, (c + 1) & 1);
        load_packed(c + 1, (c + 1) & 1);
      }
      multiply_chunk(c, c & 1);
    }
  } else {
    const T *x = (const T *)P.x + image * P.xb + (PLANES ? p0 : p0 * P.xs1);
    Chunk<T, PLANES> hold;
    load_weights(0, 0);
    hold.load(P, x, live, 0);
    for (int c = 0; c < chunks; ++c) {
      hold.put(xb[c & 1], xs[c & 1]);                    // chunk c - 2 used this buffer: every wave is past the barrier of c - 1
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this chunk's weights are in LDS
      __syncthreads();
      if (c + 1 < chunks) {
        load_weights(c + 1, (c + 1) & 1);                // chunk c - 1 used this buffer: every wave is past it
        hold.load(P, x, live, c + 1);
      }
      multiply_chunk(c, c & 1);
    }
  }

  Y *y = (Y *)P.y + image * P.pixels * P.n;
  const int live_w = live - 64 * wp;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int nt = nt0 + wn * NT + t;
    if (nt < P.tiles_n) {
      if constexpr (PLANES) store_planes<Y>(P, y, p0 + 64 * wp, live_w, nt, lane, act, acc[t]);
      else store_rows<Y>(P, y, p0 + 64 * wp, live_w, nt, lane, act, vec_y, acc[t]);
    }
  }
}

template <typename T, typename Y, bool PLANES> bool launch_stream(Product P, int act, long long batch, hipStream_t st) {
  P.tiles_pixels = (unsigned)((P.pixels + kChunkTile - 1) / kChunkTile);
  const long long tiles = batch * P.tiles_pixels;
  constexpr int kMaxNT = sizeof(Y) == 4 && !__is_same(T, Packed) ? 4 : 5;
  int splits = (P.tiles_n + 2 * kMaxNT - 1) / (2 * kMaxNT);
  while (tiles * splits < 256 && splits * 2 <= P.tiles_n) splits *= 2;
  int nt = (P.tiles_n + 2 * splits - 1) / (2 * splits);
  splits = (P.tiles_n + 2 * nt - 1) / (2 * nt);
  const int vec_y = (uintptr_t)P.y % 16 == 0 && P.n * sizeof(Y) % 16 == 0;
  const unsigned grid = (unsigned)((tiles + 7) / 8 * 8 * splits);
  if (nt == 1) mx_stream_kernel<T, Y, PLANES, 1><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 2) mx_stream_kernel<T, Y, PLANES, 2><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 3) mx_stream_kernel<T, Y, PLANES, 3><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else if (nt == 4) mx_stream_kernel<T, Y, PLANES, 4><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  else mx_stream_kernel<T, Y, PLANES, kMaxNT><<<grid, 256, 0, st>>>(P, act, splits, tiles, vec_y);
  return true;
}

constexpr int kMaxSteps = 28;   // 59.5 KB of LDS
size_t lds_bytes(int steps) { return (size_t)steps * 2048 + (size_t)((steps + 3) / 4) * 512; }

template <typename T, typename Y, bool PLANES, bool VEC, int ACT> int launch_product(Product P, long long batch, hipStream_t st) {
  P.steps = P.all_steps < kMaxSteps ? P.all_steps : kMaxSteps;
  const long long tiles = batch * P.tiles_pixels;
  // few positions: the weight rows are split over workgroups too, until there are about two per CU
  long long split = 1;
  if (tiles < 512) split = (512 + tiles - 1) / tiles;
  P.split_n = (int)((P.tiles_n + split - 1) / split);
  const dim3 grid((unsigned)tiles, (unsigned)((P.tiles_n + P.split_n - 1) / P.split_n));
  const size_t lds = lds_bytes(P.steps);
  if (P.split_n == 1) {
    const size_t parts = 3 * 32 * 64 * 4;
    mx_product_kernel<T, Y, PLANES, VEC, ACT, true><<<grid, 256, lds > parts ? lds : parts, st>>>(P);
  } else {
    mx_product_kernel<T, Y, PLANES, VEC, ACT, false><<<grid, 256, lds, st>>>(P);
  }
  return lmi_check_launch("lmi_mx_product");
}

template <typename T, typename Y, bool PLANES> int launch_act(const Product &P, int act, long long batch, hipStream_t st) {
  constexpr long long kStreamFrom = 4096;
  if constexpr (__is_same(T, Packed)) {
    if (batch * P.pixels >= kStreamFrom && launch_stream<T, Y, false>(P, act, batch, st)) return lmi_check_launch("lmi_mx_product");
  }
  // planes: two pixels of a channel in one load, and of a result in one store; rows: 16-byte loads
  const uintptr_t align = PLANES ? 2 * sizeof(Y) : 16;
  bool vec = false;
  if constexpr (!__is_same(T, Packed)) {
    vec = P.xs1 < (1 << 24) && P.pixels < (1 << 24) && (uintptr_t)P.x % align == 0 && P.xb * sizeof(Y) % align == 0 && P.xs1 * sizeof(Y) % align == 0;
    if (PLANES) vec = vec && P.pixels % 2 == 0 && (uintptr_t)P.y % align == 0;
    if constexpr (PLANES) {
      if (vec && launch_wave_planes<T>(P, act, batch, st)) return lmi_check_launch("lmi_mx_product");
    }
    if (vec && batch * P.pixels >= kStreamFrom && launch_stream<T, Y, PLANES>(P, act, batch, st)) return lmi_check_launch("lmi_mx_product");
    if (vec)
      return act == LMI_ACT_SILU ? launch_product<T, Y, PLANES, true, LMI_ACT_SILU>(P, batch, st) : launch_product<T, Y, PLANES, true, LMI_ACT_NONE>(P, batch, st);
  }
  return act == LMI_ACT_SILU ? launch_product<T, Y, PLANES, false, LMI_ACT_SILU>(P, batch, st) : launch_product<T, Y, PLANES, false, LMI_ACT_NONE>(P, batch, st);
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
  mx_dequantize_kernel<<<u.grid, 256, 0, st>>>((const unsigned *)packed, (const unsigned *)scales, rows, k, u.steps, u.quads, u.units, vec, (T *)out);
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

int64_t lmi_mx_product_workspace_bytes(const lmi_mx_product_args *) { return 0; }

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
  LMI_REQUIRE(lmi_is_aligned(a->w_packed, 16) && lmi_is_aligned(a->w_scales, 4), LMI_ERR_ALIGNMENT,
              "lmi_mx_product: w_packed must be 16-byte, w_scales 4-byte aligned");
  Product P = {};
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
  P.blocks = (unsigned)blocks;
  P.all_steps = (int)((blocks + 1) / 2);
  P.tiles_n = (int)tiles_n;
  P.tiles_pixels = (unsigned)tiles_p;
  hipStream_t st = (hipStream_t)stream;
  if (a->x_dtype == LMI_MXFP4) {
    LMI_REQUIRE(rows && a->batch == 1 && a->x_scales && lmi_is_aligned(a->x, 16) && lmi_is_aligned(a->x_scales, 4), LMI_ERR_BAD_ARG,
                "lmi_mx_product: quantised x comes as 16-byte aligned rows with their scales, batch 1");
    if (a->y_dtype == LMI_F32) return launch_act<Packed, float, false>(P, a->act, 1, st);
    if (a->y_dtype == LMI_F16) return launch_act<Packed, _Float16, false>(P, a->act, 1, st);
    return launch_act<Packed, __bf16, false>(P, a->act, 1, st);
  }
  if (rows) {
    if (a->x_dtype == LMI_F32) return launch_act<float, float, false>(P, a->act, a->batch, st);
    if (a->x_dtype == LMI_F16) return launch_act<_Float16, _Float16, false>(P, a->act, a->batch, st);
    return launch_act<__bf16, __bf16, false>(P, a->act, a->batch, st);
  }
  if (a->x_dtype == LMI_F32) return launch_act<float, float, true>(P, a->act, a->batch, st);
  if (a->x_dtype == LMI_F16) return launch_act<_Float16, _Float16, true>(P, a->act, a->batch, st);
  return launch_act<__bf16, __bf16, true>(P, a->act, a->batch, st);
}

}  // extern "C"
