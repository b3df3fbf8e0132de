// q8.hip -- 8-bit rows and their integer product: RMSNorm with the residual's addition and 8-bit rows out, quantisation of activations
// and of SwiGLU products, the read-back, and C = sa[m] sw[n] (A8 . W8^T) + bias on the integer matrix cores (gfx950).
#include "q8.hpp"

using namespace wj;

namespace {

struct RowArgs {
  const void* x; int64_t ldx; int xt;          // input rows and their type
  const void* delta; int64_t ldd; int dt;      // NULL: none
  const float* w; float eps;                   // NULL: no norm
  void* resid; int64_t ldr;                    // NULL: not stored
  int block;                                   // > 0: SwiGLU over alternating blocks of gate and up columns
  int8_t* codes; int64_t ldc;
  float* scale;
  int cols;
};

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + expf(-g)) * u; }

// sum and maximum over a workgroup of 4 waves
__device__ __forceinline__ float group_sum(float v, float* part) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}
__device__ __forceinline__ float group_max(float v, float* part) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

// One workgroup per row, any type, stride and alignment: the row lives in LDS as float32 between its three passes (read and sum of
// squares; maximum; codes).
__global__ __launch_bounds__(256) void q8_rows_kernel(const RowArgs a) {
  extern __shared__ float row[];
  __shared__ float part[4];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  float ss = 0.f;
  for (int c = tid; c < a.cols; c += 256) {
    float v;
    if (a.block) {
      const int64_t g = r * a.ldx + (int64_t)(c / a.block) * 2 * a.block + c % a.block;
      v = silu_mul(ld_any(a.x, a.xt, g), ld_any(a.x, a.xt, g + a.block));
    } else {
      v = ld_any(a.x, a.xt, r * a.ldx + c);
    }
    if (a.delta) v += ld_any(a.delta, a.dt, r * a.ldd + c);
    if (a.resid) st_any(a.resid, a.xt, r * a.ldr + c, v);
    ss += v * v;
    row[c] = v;
  }
  float top = 0.f;
  if (a.w) {
    const float s = rsqrtf(group_sum(ss, part) / (float)a.cols + a.eps);
    for (int c = tid; c < a.cols; c += 256) {
      const float y = row[c] * s * a.w[c];
      row[c] = y;
      top = fmaxf(top, mag(y));
    }
  } else {
    for (int c = tid; c < a.cols; c += 256) top = fmaxf(top, mag(row[c]));
  }
  const RowQuant q(group_max(top, part));
  for (int c = tid; c < a.cols; c += 256) a.codes[r * a.ldc + c] = (int8_t)q.code(row[c]);
  if (tid == 0) a.scale[r] = q.scale;
}

__global__ __launch_bounds__(256) void q8_dequantize_kernel(const int8_t* __restrict__ codes, int64_t ldc, const float* __restrict__ scale,
                                                            int dtype, void* __restrict__ out, int64_t ldo, int cols) {
  const int64_t r = blockIdx.x;
  const float s = scale[r];
  for (int c = threadIdx.x; c < cols; c += 256) st_any(out, dtype, r * ldo + c, (float)codes[r * ldc + c] * s);
}

// --------------------------------------------------------------------------------------------
// int8 product
// --------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

struct GemmQ8Args {
  const int8_t* a; int64_t lda; const float* sa;
  const int8_t* w; int64_t ldw; const float* sw;
  const float* bias;
  void* out; int64_t ldo; int dtype;
  int64_t m; int n, k;
};

__device__ __forceinline__ i32x4_t mfma_i8(i32x4_t a, i32x4_t b, i32x4_t c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// Any base, stride and size: 64 x 64 tile, k step 64, operands gathered byte by byte into LDS, 4 waves of 16 rows x 64 columns.
__global__ __launch_bounds__(256) void q8_gemm_any_kernel(const GemmQ8Args g) {
  __shared__ __attribute__((aligned(16))) int8_t la[64 * 80], lw[64 * 80];      // rows 80 bytes apart: 16-byte reads, few bank conflicts
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * 64;
  const int n0 = blockIdx.x * 64;
  i32x4_t acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = i32x4_t{0, 0, 0, 0};
  const int r = tid >> 2, c0 = (tid & 3) * 16;
  for (int k0 = 0; k0 < g.k; k0 += 64) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int k = k0 + c0 + e;
      la[r * 80 + c0 + e] = k < g.k && m0 + r < g.m ? g.a[(m0 + r) * g.lda + k] : (int8_t)0;
      lw[r * 80 + c0 + e] = k < g.k && n0 + r < g.n ? g.w[(int64_t)(n0 + r) * g.ldw + k] : (int8_t)0;
    }
    __syncthreads();
    const i32x4_t af = *reinterpret_cast<const i32x4_t*>(&la[(wave * 16 + (lane & 15)) * 80 + (lane >> 4) * 16]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc[j] = mfma_i8(*reinterpret_cast<const i32x4_t*>(&lw[(j * 16 + (lane & 15)) * 80 + (lane >> 4) * 16]), af, acc[j]);
  }
  // weights first: lane (r = lane & 15, q = lane >> 4) holds columns 4 q .. 4 q + 3 of row r
  const int64_t m = m0 + wave * 16 + (lane & 15);
  if (m >= g.m) return;
  const float sa = g.sa[m];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + j * 16 + (lane >> 4) * 4 + e;
      if (n < g.n) st_any(g.out, g.dtype, m * g.ldo + n, (float)acc[j][e] * (sa * g.sw[n]) + (g.bias ? g.bias[n] : 0.f));
    }
}

int launch_rows(const char* who, wj_ctx* ctx, const RowArgs& a, int64_t rows, void* stream) {
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  static AttrOnce attr;
  const size_t lds = (size_t)a.cols * 4;
  if (attr.need()) {
    WJ_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(q8_rows_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 32768 * 4));
    attr.done();
  }
  hipLaunchKernelGGL(q8_rows_kernel, dim3((unsigned)rows), dim3(256), lds, ctx->pick(stream), a);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}

}  // namespace

extern "C" {

int wj_q8_rmsnorm(wj_ctx* ctx, int dtype, const void* x_dev, int64_t ldx, int delta_dtype, const void* delta_dev, int64_t ldd,
                  const float* w_dev, float eps, void* residual_dev, int64_t ldr, int8_t* codes_dev, int64_t ldc, float* scale_dev,
                  int64_t rows, int cols, void* stream) {
  WJ_REQUIRE(ctx, "wj_q8_rmsnorm: NULL context");
  WJ_REQUIRE(known_dtype(dtype) && (!delta_dev || known_dtype(delta_dtype)), "wj_q8_rmsnorm: unknown dtype");
  WJ_REQUIRE(rows >= 0 && rows <= 0x7fffffff && cols >= 1 && cols <= 32768, "wj_q8_rmsnorm: %lld rows of %d columns (at most 2^31 - 1 rows of 1 .. 32768)", (long long)rows, cols);
  if (rows == 0) return WJ_OK;
  WJ_REQUIRE(x_dev && w_dev && codes_dev && scale_dev, "wj_q8_rmsnorm: NULL argument");
  WJ_REQUIRE(eps >= 0.f, "wj_q8_rmsnorm: eps must not be negative");
  WJ_REQUIRE(ldx >= 0 && ldd >= 0 && (rows == 1 || (ldc >= cols && (!residual_dev || ldr >= cols))), "wj_q8_rmsnorm: output rows overlap (stride below %d columns)", cols);
  RowArgs a{x_dev, ldx, dtype, delta_dev, ldd, delta_dtype, w_dev, eps, residual_dev, ldr, 0, codes_dev, ldc, scale_dev, cols};
  return launch_rows("wj_q8_rmsnorm", ctx, a, rows, stream);
}

int wj_q8_quantize(wj_ctx* ctx, int dtype, const void* x_dev, int64_t ldx, int swiglu_block, int8_t* codes_dev, int64_t ldc,
                   float* scale_dev, int64_t rows, int cols, void* stream) {
  WJ_REQUIRE(ctx, "wj_q8_quantize: NULL context");
  WJ_REQUIRE(known_dtype(dtype), "wj_q8_quantize: unknown dtype %d", dtype);
  WJ_REQUIRE(rows >= 0 && rows <= 0x7fffffff && cols >= 1 && cols <= 32768, "wj_q8_quantize: %lld rows of %d columns (at most 2^31 - 1 rows of 1 .. 32768)", (long long)rows, cols);
  WJ_REQUIRE(swiglu_block >= 0 && (swiglu_block == 0 || cols % swiglu_block == 0), "wj_q8_quantize: %d columns are no whole number of SwiGLU blocks of %d", cols, swiglu_block);
  if (rows == 0) return WJ_OK;
  WJ_REQUIRE(x_dev && codes_dev && scale_dev, "wj_q8_quantize: NULL argument");
  WJ_REQUIRE(ldx >= 0 && (rows == 1 || ldc >= cols), "wj_q8_quantize: output rows overlap (stride below %d columns)", cols);
  RowArgs a{x_dev, ldx, dtype, nullptr, 0, 0, nullptr, 0.f, nullptr, 0, swiglu_block, codes_dev, ldc, scale_dev, cols};
  return launch_rows("wj_q8_quantize", ctx, a, rows, stream);
}

int wj_q8_dequantize(wj_ctx* ctx, const int8_t* codes_dev, int64_t ldc, const float* scale_dev, int dtype, void* out_dev, int64_t ldo,
                     int64_t rows, int cols, void* stream) {
  WJ_REQUIRE(ctx, "wj_q8_dequantize: NULL context");
  WJ_REQUIRE(known_dtype(dtype), "wj_q8_dequantize: unknown dtype %d", dtype);
  WJ_REQUIRE(rows >= 0 && rows <= 0x7fffffff && cols >= 0, "wj_q8_dequantize: %lld rows of %d columns", (long long)rows, cols);
  if (rows == 0 || cols == 0) return WJ_OK;
  WJ_REQUIRE(codes_dev && scale_dev && out_dev, "wj_q8_dequantize: NULL argument");
  WJ_REQUIRE(ldc >= 0 && (rows == 1 || ldo >= cols), "wj_q8_dequantize: output rows overlap (stride below %d columns)", cols);
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  hipLaunchKernelGGL(q8_dequantize_kernel, dim3((unsigned)rows), dim3(256), 0, ctx->pick(stream), codes_dev, ldc, scale_dev, dtype, out_dev, ldo, cols);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}

int64_t wj_q8_gemm_workspace(wj_ctx* ctx, int64_t m, int n, int k) {
  (void)ctx; (void)m; (void)n; (void)k;
  return 0;
}

int wj_q8_gemm(wj_ctx* ctx, const int8_t* a_dev, int64_t lda, const float* a_scale_dev, const int8_t* w_dev, int64_t ldw,
               const float* w_scale_dev, const float* bias_dev, int dtype, void* out_dev, int64_t ldo, int64_t m, int n, int k,
               void* workspace_dev, int64_t workspace_bytes, void* stream) {
  WJ_REQUIRE(ctx, "wj_q8_gemm: NULL context");
  WJ_REQUIRE(known_dtype(dtype), "wj_q8_gemm: unknown dtype %d", dtype);
  WJ_REQUIRE(m >= 0 && m <= (int64_t)65535 * 64 && n >= 0 && k >= 0 && k <= 131071, "wj_q8_gemm: %lld x %d x %d (at most 4194240 rows; k at most 131071: the sum is 32 bits wide)",
             (long long)m, n, k);
  if (m == 0 || n == 0) return WJ_OK;
  WJ_REQUIRE(a_scale_dev && w_scale_dev && out_dev && (k == 0 || (a_dev && w_dev)), "wj_q8_gemm: NULL argument");
  WJ_REQUIRE(lda >= 0 && ldw >= 0 && (m == 1 || ldo >= n), "wj_q8_gemm: output rows overlap (stride below %d columns)", n);
  WJ_REQUIRE(workspace_bytes >= wj_q8_gemm_workspace(ctx, m, n, k), "wj_q8_gemm: %lld bytes of workspace, %lld needed", (long long)workspace_bytes,
             (long long)wj_q8_gemm_workspace(ctx, m, n, k));
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  const GemmQ8Args g{a_dev, lda, a_scale_dev, w_dev, ldw, w_scale_dev, bias_dev, out_dev, ldo, dtype, m, n, k};
  hipLaunchKernelGGL(q8_gemm_any_kernel, dim3((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64)), dim3(256), 0, ctx->pick(stream), g);
  WJ_LAUNCH_CHECK();
  (void)workspace_dev;
  return WJ_OK;
}

}  // extern "C"
