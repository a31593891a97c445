// MXFP4 (4-bit e2m1 elements, one power-of-two scale per 32) for gfx950: quantising, reading back, and the product of
// quantised weights with activations -- a 1x1 convolution of the network with its folded batch norm and SiLU, or a linear layer.
//
// A block's scale is 2^(floor(log2 max) - 2), so its largest element lands in [4, 8): 6 is the largest magnitude of e2m1, and
// what rounds beyond it stays at 6.  v_cvt_scalef32_pk_fp4_* divides by the scale and rounds to nearest even with that
// saturation; x / 2^e is exact, so nothing is rounded twice.  The products run on v_mfma_scale_f32_32x32x64_f8f6f4: 64 elements of k
// per instruction, every lane brings 32 elements of one row and their scale byte -- one block --, sums in fp32.
//
// Kernels
//  mx_quantize_kernel     four lanes per block of a row, 8 elements each.
//  mx_dequantize_kernel   eight elements per thread.
//  mx_product_kernel      64 positions x all of k: activations are read once, quantised in registers (a lane owns whole blocks: 32
//                         channels of one position) and laid into LDS in the matrix instruction's order; then every wave
//                         multiplies them with its share of the weight rows.
#include <hip/hip_fp16.h>

#include "common.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));

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

template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *x, long long rows, long long k, long long row_stride, unsigned blocks,
                                                          unsigned char *packed, unsigned char *scales) {
  const long long quads = rows * blocks * 4;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < quads; q += (long long)gridDim.x * 256) {   // quads % 4 == 0: the four lanes stay together
    const long long block = q >> 2;
    const long long row = block / blocks;
    const long long c0 = (block - row * blocks) * LMI_MX_BLOCK + (q & 3) * 8;
    const T *p = x + row * row_stride + c0;
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = c0 + u < k ? to_float(p[u]) : 0.0f;
    unsigned m = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
    m = max(m, __shfl_xor(m, 1));
    m = max(m, __shfl_xor(m, 2));
    const unsigned byte = scale_byte(m);
    ((unsigned *)packed)[q] = pack8(v, scale_value(byte));
    if ((q & 3) == 0) scales[block] = (unsigned char)byte;
  }
}

// e2m1 code -> value
__device__ __forceinline__ float code_value(unsigned c) {
  const unsigned m = c & 7u;
  const float a = m < 2u ? 0.5f * m : (1.0f + 0.5f * (m & 1u)) * (float)(1u << ((m >> 1) - 1u));
  return (c & 8u) ? -a : a;
}

template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned char *packed, const unsigned char *scales, long long rows,
                                                            long long k, unsigned blocks, T *out) {
  const long long quads = rows * blocks * 4;
  for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < quads; q += (long long)gridDim.x * 256) {
    const long long block = q >> 2;
    const long long row = block / blocks;
    const long long c0 = (block - row * blocks) * LMI_MX_BLOCK + (q & 3) * 8;
    const unsigned w = ((const unsigned *)packed)[q], byte = scales[block];
    // 2^(byte - 127); the smallest is subnormal, 255 is NaN
    const float s = byte == 255u ? NAN : (byte ? __uint_as_float(byte << 23) : 0x1p-127f);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (c0 + u < k) out[row * k + c0 + u] = (T)(code_value((w >> (4 * u)) & 15u) * s);
  }
}

struct Product {
  const void *x;
  const unsigned char *xs;
  long long pixels, k, n, xb, xs1;   // xs1: between positions (rows) or channels (planes)
  const unsigned char *w, *ws;
  const float *bias;
  void *y;
  unsigned blocks;        // blocks of 32 along k
  unsigned tiles_pixels;  // tiles of 64 positions per image
  int tiles_n;            // tiles of 32 weight rows
  int split_n;            // tiles of 32 weight rows per workgroup
  int steps;              // steps of 64 along k that LDS holds
};

constexpr int kTile = 64;   // positions per workgroup

template <int ACT> __device__ __forceinline__ float activate(float v) {
  if (ACT == LMI_ACT_SILU) return v / (1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
  return v;
}

// block kb of position p -> 16 bytes and the scale byte
template <typename T, bool PLANES>
__device__ __forceinline__ void load_block(const Product &P, const T *x, long long p, unsigned kb, uint4 &frag, unsigned &byte) {
  float v[LMI_MX_BLOCK];
  unsigned m = 0;
  const long long c0 = (long long)kb * LMI_MX_BLOCK;
  const T *q = x + p * (PLANES ? 1 : P.xs1) + c0 * (PLANES ? P.xs1 : 1);
#pragma unroll
  for (int u = 0; u < LMI_MX_BLOCK; ++u) {
    v[u] = c0 + u < P.k ? to_float(q[u * (PLANES ? P.xs1 : 1)]) : 0.0f;
    m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
  }
  byte = scale_byte(m);
  const float s = scale_value(byte);
  frag = make_uint4(pack8(v, s), pack8(v + 8, s), pack8(v + 16, s), pack8(v + 24, s));
}
template <bool PLANES>
__device__ __forceinline__ void load_packed(const Product &P, long long p, unsigned kb, uint4 &frag, unsigned &byte) {
  const long long block = p * P.blocks + kb;
  frag = ((const uint4 *)P.x)[block];
  byte = P.xs[block];
}

template <typename T, typename Y, bool PLANES, int ACT>
__global__ __launch_bounds__(256) void mx_product_kernel(const Product P) {
  extern __shared__ uint4 lds[];   // [step][2][64] fragments, then [step][2][64] scale bytes
  uint4 *frags = lds;
  unsigned char *bytes = (unsigned char *)(lds + (long long)P.steps * 128);
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long long image = blockIdx.x / P.tiles_pixels;
  const long long p0 = (long long)(blockIdx.x % P.tiles_pixels) * kTile;
  const int live = (int)(P.pixels - p0 < kTile ? P.pixels - p0 : kTile);
  const int nt0 = blockIdx.y * P.split_n;
  const int nt1 = nt0 + P.split_n < P.tiles_n ? nt0 + P.split_n : P.tiles_n;
  const int all_steps = (int)(P.blocks + 1) / 2;
  const bool once = all_steps <= P.steps;
  Y *y = (Y *)P.y + image * P.pixels * P.n;

  for (int g0 = nt0; g0 < nt1; g0 += 4) {   // every wave takes one tile of a group of four
    const int nt = g0 + wave;
    f16x acc[2] = {};
    for (int s0 = 0; s0 < all_steps; s0 += P.steps) {
      const int ns = all_steps - s0 < P.steps ? all_steps - s0 : P.steps;
      if (!once || g0 == nt0) {
        __syncthreads();   // LDS is free again
        for (int item = t; item < ns * 2 * kTile; item += 256) {
          const int px = item % kTile, kl = item / kTile;
          const unsigned kb = 2 * s0 + kl;
          uint4 frag = make_uint4(0, 0, 0, 0);
          unsigned byte = 0;
          if (px < live && kb < P.blocks) {
            if constexpr (__is_same(T, Packed)) load_packed<PLANES>(P, p0 + px, kb, frag, byte);
            else load_block<T, PLANES>(P, (const T *)P.x + image * P.xb, p0 + px, kb, frag, byte);
          }
          const int at = ((kl >> 1) * 2 + (px >> 5)) * 64 + (kl & 1) * 32 + (px & 31);
          frags[at] = frag;
          bytes[at] = (unsigned char)byte;
        }
        __syncthreads();
      }
      if (nt < nt1) {
        const long long n = (long long)nt * 32 + (lane & 31);
        const long long wrow = (n < P.n ? n : P.n - 1) * P.blocks;
        for (int s = 0; s < ns; ++s) {
          const unsigned kb = 2 * (s0 + s) + (lane >> 5);
          uint4 a = make_uint4(0, 0, 0, 0);
          unsigned sa = 0;
          if (kb < P.blocks) {
            a = ((const uint4 *)P.w)[wrow + kb];
            sa = P.ws[wrow + kb];
          }
          const v8i av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 b = frags[(s * 2 + h) * 64 + lane];
            const v8i bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
            acc[h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc[h], 4, 4, 0, (int)sa, 0, (int)bytes[(s * 2 + h) * 64 + lane]);
          }
        }
      }
    }
    if (nt < nt1) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int px = h * 32 + (lane & 31);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const long long n = (long long)nt * 32 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
          if (px < live && n < P.n) {
            const float v = activate<ACT>(acc[h][i] + (P.bias ? P.bias[n] : 0.0f));
            y[PLANES ? n * P.pixels + p0 + px : (p0 + px) * P.n + n] = (Y)v;
          }
        }
      }
    }
  }
}

constexpr int kStepBytes = 128 * 17;   // LDS of one step of 64 along k
constexpr int kMaxSteps = 28;          // 59.5 KB

template <typename T, typename Y, bool PLANES, int ACT> int launch_product(Product P, long long batch, hipStream_t st) {
  const int all_steps = (int)(P.blocks + 1) / 2;
  P.steps = all_steps < kMaxSteps ? all_steps : kMaxSteps;
  const long long tiles = batch * P.tiles_pixels;
  // few positions: the weight rows are split over workgroups too, until there are about two per CU
  long long split = 1;
  if (tiles < 512) split = (512 + tiles - 1) / tiles;
  P.split_n = (int)((P.tiles_n + split - 1) / split);
  const unsigned gy = (unsigned)((P.tiles_n + P.split_n - 1) / P.split_n);
  mx_product_kernel<T, Y, PLANES, ACT><<<dim3((unsigned)tiles, gy), 256, (size_t)P.steps * kStepBytes, st>>>(P);
  return lmi_check_launch("lmi_mx_product");
}

template <typename T, typename Y, bool PLANES> int launch_act(const Product &P, int act, long long batch, hipStream_t st) {
  return act == LMI_ACT_SILU ? launch_product<T, Y, PLANES, LMI_ACT_SILU>(P, batch, st) : launch_product<T, Y, PLANES, LMI_ACT_NONE>(P, batch, st);
}

bool float_type(int d) { return d == LMI_F32 || d == LMI_F16 || d == LMI_BF16; }

}  // namespace

extern "C" {

int lmi_mx_quantize(const void *x, int dtype, int64_t rows, int64_t k, int64_t row_stride, uint8_t *packed, uint8_t *scales, void *stream) {
  LMI_REQUIRE(rows >= 0 && k > 0 && row_stride >= 0, LMI_ERR_BAD_ARG, "lmi_mx_quantize: %lld rows of %lld elements", (long long)rows, (long long)k);
  LMI_REQUIRE(float_type(dtype), LMI_ERR_BAD_ARG, "lmi_mx_quantize: x must be fp32, fp16 or bf16");
  if (rows == 0) return LMI_OK;
  LMI_REQUIRE(x && packed && scales, LMI_ERR_BAD_ARG, "lmi_mx_quantize: null pointer");
  LMI_REQUIRE(lmi_is_aligned(packed, 16), LMI_ERR_ALIGNMENT, "lmi_mx_quantize: packed must be 16-byte aligned");
  const int64_t blocks = (k + LMI_MX_BLOCK - 1) / LMI_MX_BLOCK;
  LMI_REQUIRE(blocks < (1ll << 31) && rows < (1ll << 40) / blocks, LMI_ERR_LIMIT, "lmi_mx_quantize: too many elements");
  const int64_t wanted = (rows * blocks * 4 + 255) / 256;
  const unsigned grid = (unsigned)(wanted < (1 << 23) ? wanted : (1 << 23));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LMI_F32) mx_quantize_kernel<<<grid, 256, 0, st>>>((const float *)x, rows, k, row_stride, (unsigned)blocks, packed, scales);
  else if (dtype == LMI_F16) mx_quantize_kernel<<<grid, 256, 0, st>>>((const _Float16 *)x, rows, k, row_stride, (unsigned)blocks, packed, scales);
  else mx_quantize_kernel<<<grid, 256, 0, st>>>((const __bf16 *)x, rows, k, row_stride, (unsigned)blocks, packed, scales);
  return lmi_check_launch("lmi_mx_quantize");
}

int lmi_mx_dequantize(const uint8_t *packed, const uint8_t *scales, int64_t rows, int64_t k, void *out, int out_dtype, void *stream) {
  LMI_REQUIRE(rows >= 0 && k > 0, LMI_ERR_BAD_ARG, "lmi_mx_dequantize: %lld rows of %lld elements", (long long)rows, (long long)k);
  LMI_REQUIRE(float_type(out_dtype), LMI_ERR_BAD_ARG, "lmi_mx_dequantize: out must be fp32, fp16 or bf16");
  if (rows == 0) return LMI_OK;
  LMI_REQUIRE(packed && scales && out, LMI_ERR_BAD_ARG, "lmi_mx_dequantize: null pointer");
  LMI_REQUIRE(lmi_is_aligned(packed, 16), LMI_ERR_ALIGNMENT, "lmi_mx_dequantize: packed must be 16-byte aligned");
  const int64_t blocks = (k + LMI_MX_BLOCK - 1) / LMI_MX_BLOCK;
  LMI_REQUIRE(blocks < (1ll << 31) && rows < (1ll << 40) / blocks, LMI_ERR_LIMIT, "lmi_mx_dequantize: too many elements");
  const int64_t wanted = (rows * blocks * 4 + 255) / 256;
  const unsigned grid = (unsigned)(wanted < (1 << 23) ? wanted : (1 << 23));
  hipStream_t st = (hipStream_t)stream;
  if (out_dtype == LMI_F32) mx_dequantize_kernel<<<grid, 256, 0, st>>>(packed, scales, rows, k, (unsigned)blocks, (float *)out);
  else if (out_dtype == LMI_F16) mx_dequantize_kernel<<<grid, 256, 0, st>>>(packed, scales, rows, k, (unsigned)blocks, (_Float16 *)out);
  else mx_dequantize_kernel<<<grid, 256, 0, st>>>(packed, scales, rows, k, (unsigned)blocks, (__bf16 *)out);
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
  LMI_REQUIRE(lmi_is_aligned(a->w_packed, 16), LMI_ERR_ALIGNMENT, "lmi_mx_product: w_packed must be 16-byte aligned");
  Product P = {};
  P.x = a->x;
  P.xs = a->x_scales;
  P.pixels = a->pixels;
  P.k = a->k;
  P.n = a->n;
  P.xb = a->x_batch;
  P.xs1 = a->x_stride;
  P.w = a->w_packed;
  P.ws = a->w_scales;
  P.bias = a->bias;
  P.y = a->y;
  const int64_t blocks = (a->k + LMI_MX_BLOCK - 1) / LMI_MX_BLOCK, tiles_n = (a->n + 31) / 32, tiles_p = (a->pixels + kTile - 1) / kTile;
  LMI_REQUIRE(blocks < (1 << 24) && tiles_n < (1 << 24) && tiles_p < (1 << 24) && a->batch < (1 << 24) && tiles_p * a->batch < (1 << 24), LMI_ERR_LIMIT,
              "lmi_mx_product: k, n or the number of positions is too large");
  P.blocks = (unsigned)blocks;
  P.tiles_n = (int)tiles_n;
  P.tiles_pixels = (unsigned)tiles_p;
  hipStream_t st = (hipStream_t)stream;
  if (a->x_dtype == LMI_MXFP4) {
    LMI_REQUIRE(rows && a->batch == 1 && a->x_scales && lmi_is_aligned(a->x, 16), LMI_ERR_BAD_ARG,
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
