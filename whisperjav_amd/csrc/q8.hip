// q8.hip -- 8-bit rows and their integer product: RMSNorm with the residual's addition and 8-bit rows out, quantisation of activations
// and of SwiGLU products, the read-back, and C = sa[m] sw[n] (A8 . W8^T) + bias on the integer matrix cores (gfx950).
#include <type_traits>

#include "q8.hpp"
#include "q8_plan.hpp"

using namespace wj;

namespace {

// --------------------------------------------------------------------------------------------
// Rows.  WPR waves hold one row in registers, 8 consecutive columns per lane and step (at most 4 steps): one read of the inputs, one
// write of the outputs, the sum of squares and the maximum over lanes by shuffles (and over waves through LDS).  Bound by memory: the
// norm of 16384 x 2048 float32 + float16 moves 11 bytes per element (369 MB with the weight) in 73 us, 5.0 TB/s, back to back in cold caches;
// one row takes 4.2 us, which is the launch and two round trips.  Everything a row needs is requested before its first value is used.  Rows of any stride and base are read with wide loads (gfx950
// serves unaligned ones).  One wave per row when there are rows to fill the chip with (no barrier between the passes); else 4, which
// shortens the chain of loads of a call that is bound by latency (see pick_rows).
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

__device__ __forceinline__ float silu_mul(float g, float u) { return g * __builtin_amdgcn_rcpf(1.f + expf(-g)) * u; }      // v_rcp_f32: 1 ulp

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
  const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t r = WPR == 1 ? group * 4 + (threadIdx.x >> 6) : group;
  if (r >= a.rows) return;                     // whole workgroups, or whole waves of one without barriers
  const int tid = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const X* x = reinterpret_cast<const X*>(a.x) + r * a.ldx;
  const int whole = a.cols & ~7;               // columns in whole groups of 8; the one group after them goes element by element
  const bool tail = a.cols & 7;
  auto col = [&](int s) { return (s * WPR * 64 + tid) * 8; };
  float v[kSteps][8], ss = 0.f, top = 0.f;
  if constexpr (MODE == ROW_SWIGLU) {
    // a group's 8 gate columns lie together when groups do not straddle blocks
    if (a.block % 8 == 0 || a.block == a.cols) {
      Raw8<X> gate[kSteps] = {}, up[kSteps] = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int c = col(s);
        if (c < whole) {
          const X* g = x + (int64_t)(c / a.block) * 2 * a.block + c % a.block;
          gate[s] = ld_raw8(g);
          up[s] = ld_raw8(g + a.block);
        }
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[s][e] = 0.f;
        if (s * WPR * 512 < a.cols) {                  // a step that lies past the row is left out: its exponentials would cost like others
          float g[8], u[8];
          widen8(gate[s], g); widen8(up[s], u);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[s][e] = silu_mul(g[e], u[e]);
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = col(s) + e;
          v[s][e] = 0.f;
          if (c < whole) {
            const X* g = x + (int64_t)(c / a.block) * 2 * a.block + c % a.block;
            v[s][e] = silu_mul(Elem<X>::ld(g), Elem<X>::ld(g + a.block));
          }
        }
    }
    if (tail)
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (col(s) == whole)
#pragma unroll
          for (int e = 0; e < 7; ++e) {
            const int c = whole + e;
            const X* g = x + (int64_t)(c / a.block) * 2 * a.block + c % a.block;
            if (c < a.cols) v[s][e] = silu_mul(Elem<X>::ld(g), Elem<X>::ld(g + a.block));
          }
  } else {
    // everything the row needs is requested before the first value is used
    constexpr bool HAS_DELTA = !std::is_same<D, NoType>::value;
    typedef typename std::conditional<HAS_DELTA, D, f16_t>::type DT;
    const DT* d = reinterpret_cast<const DT*>(a.delta) + r * a.ldd;
    Raw8<X> rx[kSteps] = {};
    Raw8<DT> rd[kSteps] = {};
    Raw8<float> rw[kSteps] = {};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = col(s);
      if (c < whole) {
        rx[s] = ld_raw8(x + c);
        if constexpr (HAS_DELTA) rd[s] = ld_raw8(d + c);
        if constexpr (MODE == ROW_NORM) rw[s] = ld_raw8(a.w + c);
      }
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      widen8(rx[s], v[s]);
      if constexpr (HAS_DELTA) {
        float t[8];
        widen8(rd[s], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[s][e] += t[e];
      }
    }
    if (tail)
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (col(s) == whole)
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (whole + e < a.cols) {
              v[s][e] = Elem<X>::ld(x + whole + e);
              if constexpr (HAS_DELTA) v[s][e] += Elem<D>::ld(d + whole + e);
              if constexpr (MODE == ROW_NORM) rw[s].w[e] = __float_as_uint(a.w[whole + e]);
            }
    if constexpr (MODE == ROW_NORM) {
      if (a.resid) {
        X* o = reinterpret_cast<X*>(a.resid) + r * a.ldr;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int c = col(s);
          if (c < whole) st8<X>(o + c, v[s]);
          else if (c == whole)
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
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e)            // past the row: zeros, unless the row itself is not finite
          v[s][e] = v[s][e] * scale * __uint_as_float(rw[s].w[e]);
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
    const int c = col(s);
    if (c < whole) {
      const uint32_t w[2] = {pack4(q.code(v[s][0]), q.code(v[s][1]), q.code(v[s][2]), q.code(v[s][3])),
                             pack4(q.code(v[s][4]), q.code(v[s][5]), q.code(v[s][6]), q.code(v[s][7]))};
      __builtin_memcpy(o + c, w, 8);
    } else if (c == whole) {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (c + e < a.cols) o[c + e] = (int8_t)q.code(v[s][e]);
    }
  }
  if (tid == 0) a.scale[r] = q.scale;
}

// Read-back: a workgroup takes whole rows' groups of 8 columns in turn, one wide load and store each.  16383 x 2040 to bfloat16 (100 MB): 15 to 20 us, 5 TB/s
// and more where the codes are still in the caches that they were written to.
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
// int8 product.  v_mfma_i32_16x16x64_i8: a lane's operand is 16 consecutive codes of one row, so an int8 tile lies in LDS exactly as a
// 16-bit tile of half the columns would, and twice the products come out of the same bytes.  The weights go first, which leaves a lane with
// 4 consecutive output columns of one row.  Codes past k inside a row's last 16 bytes may be anything: they are cleared on the activations'
// side, which is enough.  int32 sums are exact, so the kernels agree bit for bit whatever their order.
// --------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

struct GemmQ8Args {
  const int8_t* a; int64_t lda; const float* sa;
  const int8_t* w; int64_t ldw; const float* sw;
  const float* bias;
  void* out; int64_t ldo;
  int64_t m; int n, k;
  int32_t* slab; int ksplit;           // ksplit > 1: raw sums [ksplit][m][n] instead of out
};

__device__ __forceinline__ i32x4_t mfma_i8(i32x4_t a, i32x4_t b, i32x4_t c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// the bytes of a 16-byte piece that lie before `valid` (<= 0: none, >= 16: all)
__device__ __forceinline__ i32x4_t piece_mask(int valid) {
  i32x4_t m;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int b = min(4, max(0, valid - 4 * d));
    m[d] = b == 4 ? -1 : (int)((1u << (8 * b)) - 1u);
  }
  return m;
}

// Barrier without the fence of __syncthreads(), which would wait for every LDS-DMA request in flight: the kernels order their LDS
// traffic themselves (a counted s_waitcnt vmcnt by the waves that issued the DMA, the barrier, then the reads; s_waitcnt lgkmcnt(0) by
// the readers before the barrier that hands a buffer back).
__device__ __forceinline__ void q8_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void dma16(const int8_t* src, int8_t* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

__device__ __forceinline__ void ld4_to(const float* p, int n, int limit, float v[4]) {       // p[n .. n + 3], clamped below `limit`
  if (n + 4 <= limit) __builtin_memcpy(v, p + n, 16);
  else
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p[min(n + e, limit - 1)];
}

template <typename T> __device__ __forceinline__ uint32_t pack_any(float lo, float hi) {
  return (uint32_t)__builtin_bit_cast(uint16_t, to_T<T>(lo)) | ((uint32_t)__builtin_bit_cast(uint16_t, to_T<T>(hi)) << 16);
}

// 16 bytes of output, at any element alignment; PAST: past the caches
template <bool PAST> __device__ __forceinline__ void st16(void* p, u32x4_t w) {
  typedef uint32_t at2_t __attribute__((ext_vector_type(4), aligned(2)));
  if constexpr (PAST) __builtin_nontemporal_store((at2_t)w, reinterpret_cast<at2_t*>(p));
  else *reinterpret_cast<at2_t*>(p) = w;
}

// out = acc * (sa * sw) + bias of RI x 4 fragments of 16 x 16, wave origin (mw, nw).  16-bit types: lanes 16 apart trade halves of
// neighbouring fragments (v_permlane16_swap), so that a lane stores 8 consecutive columns at once.
template <typename T, bool PAST, int RI>
__device__ __forceinline__ void q8_epilogue(const GemmQ8Args& g, int64_t mw, int nw, int lane, i32x4_t (&acc)[RI][4]) {
  const int li = lane & 15, q = lane >> 4;
  float sw[4][4], bias[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = nw + j * 16 + q * 4;
    ld4_to(g.sw, n, g.n, sw[j]);
    if (g.bias) ld4_to(g.bias, n, g.n, bias[j]);
    else
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[j][e] = 0.f;
  }
  float sa[RI];
#pragma unroll
  for (int i = 0; i < RI; ++i) sa[i] = g.sa[min(mw + i * 16 + li, g.m - 1)];
#pragma unroll
  for (int i = 0; i < RI; ++i) {
    const int64_t m = mw + i * 16 + li;
    T* row = reinterpret_cast<T*>(g.out) + min(m, g.m - 1) * g.ldo;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = nw + j * 16 + q * 4;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j][e] * (sa[i] * sw[j][e]) + bias[j][e];
        if (m < g.m) {
          if (n + 4 <= g.n) st16<PAST>(row + n, u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
          else
#pragma unroll
            for (int e = 0; e < 3; ++e)
              if (n + e < g.n) row[n + e] = v[e];
        }
      }
    } else {
#pragma unroll
      for (int jp = 0; jp < 4; jp += 2) {
        float va[4], vb[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          va[e] = (float)acc[i][jp][e] * (sa[i] * sw[jp][e]) + bias[jp][e];
          vb[e] = (float)acc[i][jp + 1][e] * (sa[i] * sw[jp + 1][e]) + bias[jp + 1][e];
        }
        const uint32_t a0 = pack_any<T>(va[0], va[1]), a1 = pack_any<T>(va[2], va[3]);
        const uint32_t b0 = pack_any<T>(vb[0], vb[1]), b1 = pack_any<T>(vb[2], vb[3]);
        const auto s0 = __builtin_amdgcn_permlane16_swap(a0, b0, false, false);
        const auto s1 = __builtin_amdgcn_permlane16_swap(a1, b1, false, false);
        const u32x4_t w = {(uint32_t)s0[0], (uint32_t)s1[0], (uint32_t)s0[1], (uint32_t)s1[1]};
        const int n8 = nw + (jp + (q & 1)) * 16 + (q >> 1) * 8;
        if (m < g.m) {
          if (n8 + 8 <= g.n) st16<PAST>(row + n8, w);
          else
#pragma unroll
            for (int e = 0; e < 7; ++e)
              if (n8 + e < g.n) reinterpret_cast<uint16_t*>(row)[n8 + e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

// Tile order: workgroups go to the 8 XCDs in turn, so each XCD takes a contiguous run of tiles, in groups of 8 row panels walked column by
// column: an XCD's L2 sees few panels of either operand at a time.
__device__ __forceinline__ void tile_of(int lin, int nx, int ny, int* tx, int* ty) {
  const int total = nx * ny, q8 = total >> 3, r8 = total & 7, xcd = lin & 7;
  const int tile = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (lin >> 3);
  const int per_group = 8 * nx, group = tile / per_group, first = group * 8, rows = min(8, ny - first), in = tile - group * per_group;
  *ty = first + in % rows;
  *tx = in / rows;
}

// 256 x 256 tile, 8 waves (2 x 4, 128 x 64 each), k in pairs of 64 + 64 codes (128-byte row segments), two 64 KiB buffers.  The two waves of
// every SIMD run one barrier apart: one group reads its fragments (and requests the next pair) while the other runs 32 products on
// fragments in registers.  Barrier sequence after the prologue barrier P, every wave in every barrier:
//   group 0:        MEM(0) B0 MFMA(0) B1 MEM(1) B2 MFMA(1) B3 ...      group 1:  B0 MEM(0) B1 MFMA(0) B2 MEM(1) B3 ...
//   MEM(2p) reads half 0 of pair p and requests pair p + 1 into the other buffer; MEM(2p + 1) reads half 1 and waits for the requests.
// WAR: the other buffer held pair p - 1, read last in group 1's MEM(2p - 1), retired before B(4p - 1); MEM(2p) starts after it.
// RAW: both groups have waited for pair p + 1 by B(4p + 3); it is first read after that.
// 128-byte LDS rows, 16-byte piece c of row r in place c ^ (r & 7).
// 16384 x 12288 x 2048 in 387 .. 402 us, 2.05 .. 2.13 POP/s: the matrix pipe is busy half of the cycles, at a clock that falls to 2 GHz under it.
template <typename T, bool PAST>
__global__ __launch_bounds__(512) void q8_gemm_big_kernel(const GemmQ8Args g, int nx, int ny) {
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];      // [buffer][A | W][256][128]
  constexpr int STAGE = 2 * 256 * 128;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  int tx, ty;
  tile_of(blockIdx.x, nx, ny, &tx, &ty);
  const int64_t m0 = (int64_t)ty * 256;
  const int n0 = tx * 256;
  const int8_t* ga[4];
  const int8_t* gw[4];
  const int c = (lane & 7) ^ ((lane >> 3) & 7);                    // rows of a request start at multiples of 8: row & 7 = lane >> 3
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = (wave * 4 + q) * 8 + (lane >> 3);
    ga[q] = g.a + min(m0 + row, g.m - 1) * g.lda + c * 16;
    gw[q] = g.w + (int64_t)min(n0 + row, g.n - 1) * g.ldw + c * 16;
  }
  const int np = (g.k + 127) / 128;
  // pieces that lie wholly past k are fetched from the row's start instead (in bounds; cleared below like every code past k)
  auto issue = [&](int p, int buf) __attribute__((always_inline)) {
    const int back = p == np - 1 && p * 128 + c * 16 >= g.k ? p * 128 + c * 16 : 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      dma16(ga[q] - back, &lds[buf * STAGE + (wave * 4 + q) * 1024]);
      dma16(gw[q] - back, &lds[buf * STAGE + 256 * 128 + (wave * 4 + q) * 1024]);
      ga[q] += 128;
      gw[q] += 128;
    }
  };
  i32x4_t acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
  const int off0 = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const int off1 = (lane & 15) * 128 + (((4 + (lane >> 4)) ^ (lane & 7)) << 4);
  const int a_base = wm * 128 * 128, w_base = 256 * 128 + wn * 64 * 128;

  issue(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  q8_barrier();                 // P
  if (wm == 1) q8_barrier();    // B0
  i32x4_t af[8], wf[4];
#define WJ_Q8_READ(buf, off)                                                                                                    \
  {                                                                                                                             \
    const int8_t* ls = &lds[(buf) * STAGE];                                                                                     \
    _Pragma("unroll") for (int j = 0; j < 4; ++j) wf[j] = *reinterpret_cast<const i32x4_t*>(&ls[w_base + j * 2048 + (off)]);    \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) af[i] = *reinterpret_cast<const i32x4_t*>(&ls[a_base + i * 2048 + (off)]);    \
  }
#define WJ_Q8_CLEAR(h)                                                                       \
  if (p == np - 1 && (g.k & 127)) {                                                          \
    const i32x4_t mask = piece_mask(g.k - (p * 128 + (h) * 64 + (lane >> 4) * 16));          \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) af[i] &= mask;                             \
  }
#define WJ_Q8_MFMA()                                                                         \
  __builtin_amdgcn_s_setprio(1);                                                             \
  _Pragma("unroll") for (int i = 0; i < 8; ++i)                                              \
    _Pragma("unroll") for (int j = 0; j < 4; ++j) acc[i][j] = mfma_i8(wf[j], af[i], acc[i][j]); \
  __builtin_amdgcn_s_setprio(0);
  for (int p = 0; p < np; ++p) {
    const int b = p & 1;
    WJ_Q8_READ(b, off0)
    if (p + 1 < np) issue(p + 1, b ^ 1);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    WJ_Q8_CLEAR(0)
    q8_barrier();
    WJ_Q8_MFMA()
    q8_barrier();
    WJ_Q8_READ(b, off1)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    WJ_Q8_CLEAR(1)
    q8_barrier();
    WJ_Q8_MFMA()
    q8_barrier();
  }
  if (wm == 0) q8_barrier();    // every wave has taken part in the same number of barriers
#undef WJ_Q8_READ
#undef WJ_Q8_CLEAR
#undef WJ_Q8_MFMA
  q8_epilogue<T, PAST, 8>(g, m0 + wm * 128, n0 + wn * 64, lane, acc);
}

// BM x 128 tile, k steps of 128 codes, a ring of 3 buffers with 2 steps requested ahead (BM = 64: two workgroups per CU).  Eight waves: (2 x 2, BM / 2 x 64 each) twice,
// each four taking one half of every step's codes, so that the two waves of a SIMD overlap one's LDS reads with the other's products; the
// two halves' sums meet in LDS at the end, each four finishing half of the rows.  For calls with too few 256-tiles to fill the chip;
// ksplit > 1: slices of k on the grid's second axis write raw sums, joined by q8_gemm_join_kernel.  Bound by LDS traffic (DMA in, fragments out):
// 0.38 us per step of a 64-row tile (300 x 2048 x 8192; 0.23 with the DMA taken away); 240 x 12288 x 2048 takes 128-row tiles, 14 us.
template <typename T, int BM>
__global__ __launch_bounds__(512) void q8_gemm_tile_kernel(const GemmQ8Args g, int nx, int ny) {
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];      // [stage][A: BM | W: 128][128]
  constexpr int NS = 3, STAGE = (BM + 128) * 128, RI = BM / 32, QA = BM / 64;      // 16-row blocks and requests of a wave
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = wave >> 2, wm = (wave >> 1) & 1, wn = wave & 1;
  int tx, ty;
  tile_of(blockIdx.x, nx, ny, &tx, &ty);
  const int64_t m0 = (int64_t)ty * BM;
  const int n0 = tx * 128;
  const int steps = (g.k + 127) / 128;
  const int s_begin = (int)((int64_t)steps * blockIdx.y / g.ksplit), s_end = (int)((int64_t)steps * (blockIdx.y + 1) / g.ksplit);
  const int nk = s_end - s_begin;
  const int c = (lane & 7) ^ ((lane >> 3) & 7);
  const int8_t* ga[QA];
#pragma unroll
  for (int q = 0; q < QA; ++q) ga[q] = g.a + min(m0 + (wave * QA + q) * 8 + (lane >> 3), g.m - 1) * g.lda + c * 16 + (int64_t)s_begin * 128;
  const int8_t* gw0 = g.w + (int64_t)min(n0 + wave * 16 + (lane >> 3), g.n - 1) * g.ldw + c * 16 + (int64_t)s_begin * 128;
  const int8_t* gw1 = g.w + (int64_t)min(n0 + wave * 16 + 8 + (lane >> 3), g.n - 1) * g.ldw + c * 16 + (int64_t)s_begin * 128;
  auto issue = [&](int s, int buf) __attribute__((always_inline)) {
    const int back = s == steps - 1 && s * 128 + c * 16 >= g.k ? s * 128 + c * 16 : 0;
#pragma unroll
    for (int q = 0; q < QA; ++q) { dma16(ga[q] - back, &lds[buf * STAGE + (wave * QA + q) * 1024]); ga[q] += 128; }
    dma16(gw0 - back, &lds[buf * STAGE + BM * 128 + wave * 2048]);
    dma16(gw1 - back, &lds[buf * STAGE + BM * 128 + wave * 2048 + 1024]);
    gw0 += 128; gw1 += 128;
  };
  i32x4_t acc[RI][4];
#pragma unroll
  for (int i = 0; i < RI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int st = 0; st < NS - 1; ++st)
    if (st < nk) issue(s_begin + st, st);
  const int off = (lane & 15) * 128 + (((half * 4 + (lane >> 4)) ^ (lane & 7)) << 4);
  int buf = 0;
  for (int kt = 0; kt < nk; ++kt) {
    // the step after kt may stay in flight
    if (kt + 1 < nk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(QA + 2) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // step kt is visible to all; the buffer of step kt - 1 is free (its reads were retired before this barrier)
    q8_barrier();
    if (kt + NS - 1 < nk) issue(s_begin + kt + NS - 1, buf == 0 ? NS - 1 : buf - 1);
    const int8_t* la = &lds[buf * STAGE + wm * (BM / 2) * 128 + off];
    const int8_t* lw = &lds[buf * STAGE + BM * 128 + wn * 64 * 128 + off];
    i32x4_t af[RI], wf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) wf[j] = *reinterpret_cast<const i32x4_t*>(lw + j * 2048);
#pragma unroll
    for (int i = 0; i < RI; ++i) af[i] = *reinterpret_cast<const i32x4_t*>(la + i * 2048);
    if (s_begin + kt == steps - 1 && (g.k & 127)) {
      const i32x4_t mask = piece_mask(g.k - ((s_begin + kt) * 128 + half * 64 + (lane >> 4) * 16));
#pragma unroll
      for (int i = 0; i < RI; ++i) af[i] &= mask;
    }
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma_i8(wf[j], af[i], acc[i][j]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    buf = buf == NS - 1 ? 0 : buf + 1;
  }
  // this half finishes one half of the wave's rows and hands the others over
  __syncthreads();
  i32x4_t* swap = reinterpret_cast<i32x4_t*>(lds);
#pragma unroll
  for (int i = 0; i < RI / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) swap[((wave * (RI / 2) + i) * 4 + j) * 64 + lane] = half ? acc[i][j] : acc[RI / 2 + i][j];
  __syncthreads();
  i32x4_t sum[RI / 2][4];
#pragma unroll
  for (int i = 0; i < RI / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = (half ? acc[RI / 2 + i][j] : acc[i][j]) + swap[(((wave ^ 4) * (RI / 2) + i) * 4 + j) * 64 + lane];
  const int64_t mw = m0 + wm * (BM / 2) + half * (BM / 4);
  const int nw = n0 + wn * 64;
  if (g.ksplit == 1) {
    q8_epilogue<T, false, RI / 2>(g, mw, nw, lane, sum);
    return;
  }
#pragma unroll
  for (int i = 0; i < RI / 2; ++i) {
    const int64_t m = mw + i * 16 + (lane & 15);
    if (m >= g.m) continue;
    int32_t* row = g.slab + ((int64_t)blockIdx.y * g.m + m) * g.n;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = nw + j * 16 + (lane >> 4) * 4;
      if (n + 4 <= g.n) __builtin_memcpy(row + n, &sum[i][j], 16);
      else
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (n + e < g.n) row[n + e] = sum[i][j][e];
    }
  }
}

// out = epilogue of the slices' sums, 4 columns per lane
template <typename T>
__global__ __launch_bounds__(256) void q8_gemm_join_kernel(const GemmQ8Args g) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
  const int64_t m = blockIdx.y;
  if (n >= g.n) return;
  float sw[4], bias[4] = {0.f, 0.f, 0.f, 0.f};
  ld4_to(g.sw, n, g.n, sw);
  if (g.bias) ld4_to(g.bias, n, g.n, bias);
  const float sa = g.sa[m];
  const bool whole = n + 4 <= g.n;
  i32x4_t v[8], sum = i32x4_t{0, 0, 0, 0};             // all slices (at most 8) are requested before the first is added
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    v[s] = i32x4_t{0, 0, 0, 0};
    if (s < g.ksplit) {
      const int32_t* p = g.slab + ((int64_t)s * g.m + m) * g.n + n;
      if (whole) __builtin_memcpy(&v[s], p, 16);
      else
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (n + e < g.n) v[s][e] = p[e];
    }
  }
#pragma unroll
  for (int s = 0; s < 8; ++s) sum += v[s];
  T t[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] = to_T<T>((float)sum[e] * (sa * sw[e]) + bias[e]);
  T* o = reinterpret_cast<T*>(g.out) + m * g.ldo + n;
  if (whole) __builtin_memcpy(o, t, sizeof(t));
  else
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (n + e < g.n) o[e] = t[e];
}

// Few rows (at most 16 MT): bound by the weights' bytes.  A workgroup owns 16 output columns, its 8 waves split k, the weights go straight
// from memory into the operands (every byte once), the 8 partial tiles meet in LDS.  1 x 4096 x 2048 in 3.9 us: the launch and one round trip;
// 8 steps ahead instead of 4 take 4.6 (requests past a wave's share of k).
template <typename T, int MT>
__global__ __launch_bounds__(512) void q8_gemm_rows_kernel(const GemmQ8Args g) {
  __shared__ __attribute__((aligned(16))) int red[8 * MT * 256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  constexpr int UNR = MT == 1 ? 4 : 2;
  const int steps = (g.k + 63) / 64, per = (steps + 7) / 8;
  const int s_begin = wave * per, s_end = min(steps, s_begin + per);
  const int8_t* wr = g.w + (int64_t)min(n0 + li, g.n - 1) * g.ldw;
  i32x4_t acc[MT];
  const int8_t* ar[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    acc[t] = i32x4_t{0, 0, 0, 0};
    ar[t] = g.a + min((int64_t)t * 16 + li, g.m - 1) * g.lda;
  }
  for (int s0 = s_begin; s0 < s_end; s0 += UNR) {
    i32x4_t wv[UNR], av[UNR][MT];
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int k = (s0 + u) * 64 + q * 16;
      const bool in = s0 + u < s_end && k < g.k;
      const int kc = in ? k : 0;
      wv[u] = *reinterpret_cast<const i32x4_t*>(wr + kc);
      const i32x4_t mask = piece_mask(in ? g.k - k : 0);
#pragma unroll
      for (int t = 0; t < MT; ++t) av[u][t] = *reinterpret_cast<const i32x4_t*>(ar[t] + kc) & mask;
    }
#pragma unroll
    for (int u = 0; u < UNR; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = mfma_i8(wv[u], av[u][t], acc[t]);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) *reinterpret_cast<i32x4_t*>(&red[(wave * MT * 16 + t * 16 + li) * 16 + q * 4]) = acc[t];
  __syncthreads();
  for (int o = tid; o < MT * 64; o += 512) {
    const int64_t m = o >> 2;
    const int n = n0 + (o & 3) * 4;
    if (m >= g.m || n >= g.n) continue;
    i32x4_t sum = i32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += *reinterpret_cast<const i32x4_t*>(&red[(w * MT * 16 + (int)m) * 16 + (o & 3) * 4]);
    float sw[4], bias[4] = {0.f, 0.f, 0.f, 0.f};
    ld4_to(g.sw, n, g.n, sw);
    if (g.bias) ld4_to(g.bias, n, g.n, bias);
    const float sa = g.sa[m];
    T* row = reinterpret_cast<T*>(g.out) + m * g.ldo + n;
    T t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = to_T<T>((float)sum[e] * (sa * sw[e]) + bias[e]);
    if (n + 4 <= g.n) __builtin_memcpy(row, t, sizeof(t));
    else
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (n + e < g.n) row[e] = t[e];
  }
}

// Any base, stride and size (the caller's own layout, not a path to be fast on: 16384 x 12288 x 2048 takes 21 ms): 64 x 64 tile, k step 64, operands gathered byte by byte into LDS, 4 waves of 16 rows x 64 columns.
__global__ __launch_bounds__(256) void q8_gemm_any_kernel(const GemmQ8Args g, int dtype) {
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
      if (n < g.n) st_any(g.out, dtype, m * g.ldo + n, (float)acc[j][e] * (sa * g.sw[n]) + (g.bias ? g.bias[n] : 0.f));
    }
}

// ---- host side ---------------------------------------------------------------------------------

template <RowMode MODE, int WPR, typename X, typename D>
int start_rows(const RowArgs& a, hipStream_t s) {
  const int64_t groups = WPR == 1 ? (a.rows + 3) / 4 : a.rows;
  const int64_t nx = groups < (1 << 21) ? groups : 1 << 21;          // a grid's axis holds 2^32 threads
  hipLaunchKernelGGL((q8_rows_kernel<MODE, WPR, X, D>), dim3((unsigned)nx, (unsigned)((groups + nx - 1) / nx)), dim3(WPR == 1 ? 256 : WPR * 64), 0, s, a);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}
// Waves per row, us per call in a graph, norm (float32 + float16) / bfloat16 quantisation / float16 SwiGLU:
//   1 wave against 4: 24 x 2048 4.2, 3.3, 5.2 / 4.0, 3.1, 3.7; 512 x 2048 5.1, 3.5, 5.5 / 5.0, 3.5, 4.4; 1024 x 2048 6.4, 3.7, 5.7 / 7.1, 4.5, 6.1;
//     1024 x 512 4.1, 3.1, 3.8 / 5.3, 4.1, 5.3; 16384 x 2048 56, 18, 41 / 60, 29, 47;
//   4 waves against 16: 1 x 8192 4.3, 3.2, 5.1 / 5.2, 3.7, 5.0; 256 x 6144 5.7, 3.6, 5.2 / 6.5, 4.3, 5.7; 2048 x 4096 17, 7, 14 / 35, 16, 30.
// So 16 are for rows that 4 cannot hold, beyond 8192 columns.
template <RowMode MODE, typename X, typename D>
int pick_rows(const RowArgs& a, hipStream_t s) {
  if (a.cols <= 2048 && a.rows >= 1024) return start_rows<MODE, 1, X, D>(a, s);
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

template <typename K>
int allow_lds(K kernel, AttrOnce& once, int bytes) {
  if (once.need()) {
    WJ_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    once.done();
  }
  return WJ_OK;
}

template <typename T, int BM>
int start_tile(const GemmQ8Args& g, hipStream_t s) {
  static AttrOnce once;
  constexpr int lds = 3 * (BM + 128) * 128;
  if (int rc = allow_lds(q8_gemm_tile_kernel<T, BM>, once, lds)) return rc;
  const int nx = (g.n + 127) / 128, ny = (int)((g.m + BM - 1) / BM);
  hipLaunchKernelGGL((q8_gemm_tile_kernel<T, BM>), dim3((unsigned)nx * ny, g.ksplit), dim3(512), lds, s, g, nx, ny);
  WJ_LAUNCH_CHECK();
  if (g.ksplit > 1) {
    hipLaunchKernelGGL(q8_gemm_join_kernel<T>, dim3((unsigned)((g.n + 1023) / 1024), (unsigned)g.m), dim3(256), 0, s, g);
    WJ_LAUNCH_CHECK();
  }
  return WJ_OK;
}

template <typename T, bool PAST>
int start_big(const GemmQ8Args& g, hipStream_t s) {
  static AttrOnce once;
  constexpr int lds = 2 * 2 * 256 * 128;
  if (int rc = allow_lds(q8_gemm_big_kernel<T, PAST>, once, lds)) return rc;
  const int nx = (g.n + 255) / 256, ny = (int)((g.m + 255) / 256);
  hipLaunchKernelGGL((q8_gemm_big_kernel<T, PAST>), dim3((unsigned)nx * ny), dim3(512), lds, s, g, nx, ny);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}

template <typename T>
int launch_gemm_q8(GemmQ8Args g, hipStream_t s) {
  const GemmPlan p = plan_gemm(g.m, g.n, g.k);
  g.ksplit = p.ksplit;
  switch (p.kind) {
    case GEMM_ROWS: {
      const dim3 grid((unsigned)((g.n + 15) / 16));
      if (g.m <= 16) hipLaunchKernelGGL((q8_gemm_rows_kernel<T, 1>), grid, dim3(512), 0, s, g);
      else if (g.m <= 32) hipLaunchKernelGGL((q8_gemm_rows_kernel<T, 2>), grid, dim3(512), 0, s, g);
      else hipLaunchKernelGGL((q8_gemm_rows_kernel<T, 4>), grid, dim3(512), 0, s, g);
      WJ_LAUNCH_CHECK();
      return WJ_OK;
    }
    case GEMM_BIG: return g.m * g.n * (int64_t)sizeof(T) > (int64_t)256 << 20 ? start_big<T, true>(g, s) : start_big<T, false>(g, s);
    case GEMM_TILE128: return start_tile<T, 128>(g, s);
    default: return start_tile<T, 64>(g, s);
  }
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
  (void)ctx;
  if (m <= 0 || n <= 0 || k < 0) return 0;
  const GemmPlan p = plan_gemm(m, n, k);
  return p.ksplit > 1 ? (int64_t)p.ksplit * m * n * 4 : 0;
}

int wj_q8_gemm(wj_ctx* ctx, const int8_t* a_dev, int64_t lda, const float* a_scale_dev, const int8_t* w_dev, int64_t ldw,
               const float* w_scale_dev, const float* bias_dev, int dtype, void* out_dev, int64_t ldo, int64_t m, int n, int k,
               void* workspace_dev, int64_t workspace_bytes, void* stream) {
  WJ_REQUIRE(ctx, "wj_q8_gemm: NULL context");
  WJ_REQUIRE(known_dtype(dtype), "wj_q8_gemm: unknown dtype %d", dtype);
  WJ_REQUIRE(m >= 0 && m <= (int64_t)65535 * 64 && n >= 0 && k >= 0 && k <= 131071, "wj_q8_gemm: %lld x %d x %d (at most 4194240 rows; k at most 131071: the sum is 32 bits wide)",
             (long long)m, n, k);
  WJ_REQUIRE(n <= (1 << 27) - 16, "wj_q8_gemm: %d columns (at most 2^27 - 16: a grid's axis holds 2^32 threads, 32 for each)", n);
  if (m == 0 || n == 0) return WJ_OK;
  WJ_REQUIRE(a_scale_dev && w_scale_dev && out_dev && (k == 0 || (a_dev && w_dev)), "wj_q8_gemm: NULL argument");
  WJ_REQUIRE(lda >= 0 && ldw >= 0 && (m == 1 || ldo >= n), "wj_q8_gemm: output rows overlap (stride below %d columns)", n);
  WJ_REQUIRE(workspace_bytes >= wj_q8_gemm_workspace(ctx, m, n, k), "wj_q8_gemm: %lld bytes of workspace, %lld needed", (long long)workspace_bytes,
             (long long)wj_q8_gemm_workspace(ctx, m, n, k));
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  hipStream_t s = ctx->pick(stream);
  const GemmQ8Args g{a_dev, lda, a_scale_dev, w_dev, ldw, w_scale_dev, bias_dev, out_dev, ldo, m, n, k, reinterpret_cast<int32_t*>(workspace_dev), 1};
  // the fast kernels fetch rows in 16-byte pieces
  const bool pieces = aligned_to(a_dev, 16) && aligned_to(w_dev, 16) && (m == 1 || lda % 16 == 0) && (n == 1 || ldw % 16 == 0);
  if (pieces && k > 0) {
    WJ_REQUIRE(workspace_dev || wj_q8_gemm_workspace(ctx, m, n, k) == 0, "wj_q8_gemm: NULL workspace");
    WJ_REQUIRE(aligned_to(workspace_dev, 16), "wj_q8_gemm: the workspace is not 16-byte aligned");
    if (dtype == WJ_F32) return launch_gemm_q8<float>(g, s);
    if (dtype == WJ_F16) return launch_gemm_q8<f16_t>(g, s);
    return launch_gemm_q8<bf16_t>(g, s);
  }
  hipLaunchKernelGGL(q8_gemm_any_kernel, dim3((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64)), dim3(256), 0, s, g, dtype);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}

}  // extern "C"
