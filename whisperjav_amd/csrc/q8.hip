// q8.hip -- 8-bit rows and their integer product: RMSNorm with the residual's addition and 8-bit rows out, quantisation of activations
// and of SwiGLU products, the read-back, and C = sa[m] sw[n] (A8 . W8^T) + bias on the integer matrix cores (gfx950).
#include <type_traits>

#include "q8.hpp"

using namespace wj;

namespace {

// --------------------------------------------------------------------------------------------
// Rows.  WPR waves hold one row in registers, 8 consecutive columns per lane and step (at most 4 steps): one read of the inputs, one
// write of the outputs, the sum of squares and the maximum over lanes by shuffles (and over waves through LDS).  Bound by memory: the
// norm of 2048 float32 + float16 columns moves 11 bytes per element.  Rows of any stride and base are read with wide loads (gfx950
// serves unaligned ones).  One wave per row when there are rows to fill the chip with (no barrier between the passes); else 4 or 16, which
// shortens the chain of loads of a call that is bound by latency.
// --------------------------------------------------------------------------------------------
struct RowArgs {
  const void* x; int64_t ldx;
  const void* delta; int64_t ldd;
  const float* w; float eps;                   // norm only
  void* resid; int64_t ldr;                    // NULL: not stored
  int block;                                   // SwiGLU only: width of the alternating blocks of gate and up columns
  int8_t* codes; int64_t ldc;
  float* scale;
  int64_t rows;
  int cols;
};
enum RowMode { ROW_NORM, ROW_PLAIN, ROW_SWIGLU };
struct NoType {};                              // "no delta"
constexpr int kSteps = 4;

template <typename T> struct Raw8 { uint32_t w[8 * sizeof(T) / 4]; };      // 8 elements as they lie in memory
template <typename T> __device__ __forceinline__ Raw8<T> ld_raw8(const T* p) {
  Raw8<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
__device__ __forceinline__ void widen8(const Raw8<float>& r, float v[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r.w[e]);
}
__device__ __forceinline__ void widen8(const Raw8<f16_t>& r, float v[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) unpack2<f16_t>(r.w[e], v[2 * e], v[2 * e + 1]);
}
__device__ __forceinline__ void widen8(const Raw8<bf16_t>& r, float v[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) unpack2<bf16_t>(r.w[e], v[2 * e], v[2 * e + 1]);
}
template <typename T> __device__ __forceinline__ void st8(T* p, const float v[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = to_T<T>(v[e]);
  __builtin_memcpy(p, t, sizeof(t));
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + expf(-g)) * u; }

template <int WPR> __device__ __forceinline__ float row_sum(float v, float* part) {
  v = wave_sum(v);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) v += part[w];
  }
  return v;
}
template <int WPR> __device__ __forceinline__ float row_max(float v, float* part) {
  v = wave_max(v);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) v = fmaxf(v, part[w]);
  }
  return v;
}

template <RowMode MODE, int WPR, typename X, typename D>
__global__ __launch_bounds__(WPR == 1 ? 256 : WPR * 64) void q8_rows_kernel(const RowArgs a) {
  __shared__ float part[2][WPR];
  const int64_t r = WPR == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
  if (r >= a.rows) return;                     // WPR == 1 only, where no barrier follows
  const int tid = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const X* x = reinterpret_cast<const X*>(a.x) + r * a.ldx;
  const int whole = a.cols & ~7;               // columns in whole groups of 8
  float v[kSteps][8];
  if constexpr (MODE == ROW_SWIGLU) {
    // the group's 8 gate columns lie together when groups do not straddle blocks
    const bool wide = a.block % 8 == 0 || a.block == a.cols;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = (s * WPR * 64 + tid) * 8;
      if (c < whole && wide) {
        const X* g = x + (int64_t)(c / a.block) * 2 * a.block + c % a.block;
        float gate[8], up[8];
        const Raw8<X> rg = ld_raw8(g), ru = ld_raw8(g + a.block);
        widen8(rg, gate); widen8(ru, up);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[s][e] = silu_mul(gate[e], up[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[s][e] = 0.f;
          if (c + e < a.cols) {
            const X* g = x + (int64_t)((c + e) / a.block) * 2 * a.block + (c + e) % a.block;
            v[s][e] = silu_mul(Elem<X>::ld(g), Elem<X>::ld(g + a.block));
          }
        }
      }
    }
  } else {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = (s * WPR * 64 + tid) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s][e] = 0.f;
      if (c < whole) widen8(ld_raw8(x + c), v[s]);
      else
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (c + e < a.cols) v[s][e] = Elem<X>::ld(x + c + e);
    }
  }
  float ss = 0.f, top = 0.f;
  if constexpr (MODE == ROW_NORM) {
    if constexpr (!std::is_same<D, NoType>::value) {
      const D* d = reinterpret_cast<const D*>(a.delta) + r * a.ldd;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int c = (s * WPR * 64 + tid) * 8;
        if (c < whole) {
          float t[8];
          widen8(ld_raw8(d + c), t);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[s][e] += t[e];
        } else {
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (c + e < a.cols) v[s][e] += Elem<D>::ld(d + c + e);
        }
      }
    }
    if (a.resid) {
      X* o = reinterpret_cast<X*>(a.resid) + r * a.ldr;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int c = (s * WPR * 64 + tid) * 8;
        if (c < whole) st8<X>(o + c, v[s]);
        else
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (c + e < a.cols) o[c + e] = to_T<X>(v[s][e]);
      }
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += v[s][e] * v[s][e];
    const float scale = rsqrtf(row_sum<WPR>(ss, part[0]) / (float)a.cols + a.eps);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = (s * WPR * 64 + tid) * 8;
      if (c < whole) {
        float w[8];
        widen8(ld_raw8(a.w + c), w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[s][e] = v[s][e] * scale * w[e];
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (c + e < a.cols) v[s][e] = v[s][e] * scale * a.w[c + e];
      }
    }
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, mag(v[s][e]));
  const RowQuant q(row_max<WPR>(top, part[1]));
  int8_t* o = a.codes + r * a.ldc;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int c = (s * WPR * 64 + tid) * 8;
    if (c < whole) {
      const uint32_t w[2] = {pack4(q.code(v[s][0]), q.code(v[s][1]), q.code(v[s][2]), q.code(v[s][3])),
                             pack4(q.code(v[s][4]), q.code(v[s][5]), q.code(v[s][6]), q.code(v[s][7]))};
      __builtin_memcpy(o + c, w, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (c + e < a.cols) o[c + e] = (int8_t)q.code(v[s][e]);
    }
  }
  if (tid == 0) a.scale[r] = q.scale;
}

// Read-back: a workgroup takes whole rows' groups of 8 columns in turn, one wide load and store each.
template <typename T>
__global__ __launch_bounds__(256) void q8_dequantize_kernel(const int8_t* __restrict__ codes, int64_t ldc, const float* __restrict__ scale,
                                                            T* __restrict__ out, int64_t ldo, int64_t rows, int cols) {
  const int groups = (cols + 7) >> 3;
  const int64_t total = rows * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / groups;
    const int c = (int)(i - r * groups) * 8;
    const float s = scale[r];
    const int8_t* p = codes + r * ldc + c;
    T* o = out + r * ldo + c;
    if (c + 8 <= cols) {
      uint32_t w[2];
      __builtin_memcpy(w, p, 8);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3))) * s;
      st8<T>(o, v);
    } else {
      for (int e = 0; c + e < cols; ++e) o[e] = to_T<T>((float)p[e] * s);
    }
  }
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

// ---- host side ---------------------------------------------------------------------------------

template <RowMode MODE, int WPR, typename X, typename D>
int start_rows(const RowArgs& a, hipStream_t s) {
  const int64_t groups = WPR == 1 ? (a.rows + 3) / 4 : a.rows;
  hipLaunchKernelGGL((q8_rows_kernel<MODE, WPR, X, D>), dim3((unsigned)groups), dim3(WPR == 1 ? 256 : WPR * 64), 0, s, a);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}
template <RowMode MODE, typename X, typename D>
int pick_rows(const RowArgs& a, hipStream_t s) {
  if (a.cols <= 2048 && a.rows >= 2048) return start_rows<MODE, 1, X, D>(a, s);
  if (a.cols <= 8192) return start_rows<MODE, 4, X, D>(a, s);
  return start_rows<MODE, 16, X, D>(a, s);
}
template <RowMode MODE, typename X>
int pick_delta(const RowArgs& a, int delta_dtype, hipStream_t s) {
  if constexpr (MODE == ROW_NORM) {
    if (a.delta) {
      if (delta_dtype == WJ_F32) return pick_rows<MODE, X, float>(a, s);
      if (delta_dtype == WJ_F16) return pick_rows<MODE, X, f16_t>(a, s);
      return pick_rows<MODE, X, bf16_t>(a, s);
    }
  }
  return pick_rows<MODE, X, NoType>(a, s);
}
template <RowMode MODE>
int launch_rows(wj_ctx* ctx, int dtype, int delta_dtype, const RowArgs& a, void* stream) {
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  hipStream_t s = ctx->pick(stream);
  if (dtype == WJ_F32) return pick_delta<MODE, float>(a, delta_dtype, s);
  if (dtype == WJ_F16) return pick_delta<MODE, f16_t>(a, delta_dtype, s);
  return pick_delta<MODE, bf16_t>(a, delta_dtype, s);
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
  const RowArgs a{x_dev, ldx, delta_dev, ldd, w_dev, eps, residual_dev, ldr, 0, codes_dev, ldc, scale_dev, rows, cols};
  return launch_rows<ROW_NORM>(ctx, dtype, delta_dtype, a, stream);
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
  const RowArgs a{x_dev, ldx, nullptr, 0, nullptr, 0.f, nullptr, 0, swiglu_block, codes_dev, ldc, scale_dev, rows, cols};
  return swiglu_block ? launch_rows<ROW_SWIGLU>(ctx, dtype, 0, a, stream) : launch_rows<ROW_PLAIN>(ctx, dtype, 0, a, stream);
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
  const int64_t groups = (rows * (((int64_t)cols + 7) / 8) + 255) / 256;
  const dim3 grid((unsigned)(groups < 8192 ? groups : 8192));
  hipStream_t s = ctx->pick(stream);
  if (dtype == WJ_F32) hipLaunchKernelGGL(q8_dequantize_kernel<float>, grid, dim3(256), 0, s, codes_dev, ldc, scale_dev, (float*)out_dev, ldo, rows, cols);
  else if (dtype == WJ_F16) hipLaunchKernelGGL(q8_dequantize_kernel<f16_t>, grid, dim3(256), 0, s, codes_dev, ldc, scale_dev, (f16_t*)out_dev, ldo, rows, cols);
  else hipLaunchKernelGGL(q8_dequantize_kernel<bf16_t>, grid, dim3(256), 0, s, codes_dev, ldc, scale_dev, (bf16_t*)out_dev, ldo, rows, cols);
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
