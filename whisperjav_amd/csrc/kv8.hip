// kv8.hip -- the 8-bit key / value cache: rows quantised as they are written, read back, and the attention over it (gfx950).
#include <type_traits>

#include "q8.hpp"
#include "q8_plan.hpp"

using namespace wj;

namespace {

struct Kv8Args {
  wj_kv8 c;
  wj_kv8_batch b;
};

__device__ __forceinline__ Span span_of(const Kv8Args& a, int b) {
  // the same for every lane: kept in scalar registers
  auto uni = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  return span_from(uni(a.b.slots_dev[b]), uni(a.b.starts_dev[b]), uni(a.b.starts_dev[b + 1]), uni(a.b.lens_dev[b]), a.c.slots, a.b.rows);
}

// Writing: HD / 8 lanes hold one head's row of K and of V, 8 elements each, read and written with one wide access per lane and tensor; the
// maximum goes over the lanes by exchanges.  Bound by memory: a 16-bit row of 128 moves 256 + 128 + 4 bytes; 20 k rows of 8 heads of K and V are
// written in 26 us (4.9 TB/s) and read back in 21 (5.9).  A workgroup takes (row, head) pairs of one sequence in turn.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv8_write_kernel(const Kv8Args a, const T* __restrict__ k, int64_t ldk, const T* __restrict__ v,
                                                        int64_t ldv) {
  constexpr int L = HD / 8, PER = 256 / L;
  const Span s = span_of(a, blockIdx.y);
  if (s.slot < 0) return;
  const int l8 = (threadIdx.x % L) * 8, heads = a.c.heads;
  const int64_t tasks = (int64_t)s.n * heads;
  for (int64_t task = (int64_t)blockIdx.x * PER + threadIdx.x / L; task < tasks; task += (int64_t)gridDim.x * PER) {
    const int t = (int)(task / heads), head = (int)(task - (int64_t)t * heads), pos = s.pos0 + t;
    if (pos < 0 || pos >= a.c.ctx) continue;                    // all lanes of a row alike
    const Raw8<T> rk = ld_raw8(k + (int64_t)(s.first + t) * ldk + head * HD + l8), rv = ld_raw8(v + (int64_t)(s.first + t) * ldv + head * HD + l8);
    float xk[8], xv[8], tk = 0.f, tv = 0.f;
    widen8(rk, xk); widen8(rv, xv);
#pragma unroll
    for (int e = 0; e < 8; ++e) { tk = fmaxf(tk, mag(xk[e])); tv = fmaxf(tv, mag(xv[e])); }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) { tk = fmaxf(tk, __shfl_xor(tk, o, 64)); tv = fmaxf(tv, __shfl_xor(tv, o, 64)); }
    const RowQuant qk(tk), qv(tv);
    const int64_t row = ((int64_t)s.slot * heads + head) * a.c.ctx + pos;
    *reinterpret_cast<uint2*>(a.c.k_dev + row * HD + l8) = make_uint2(pack4(qk.code(xk[0]), qk.code(xk[1]), qk.code(xk[2]), qk.code(xk[3])),
                                                                      pack4(qk.code(xk[4]), qk.code(xk[5]), qk.code(xk[6]), qk.code(xk[7])));
    *reinterpret_cast<uint2*>(a.c.v_dev + row * HD + l8) = make_uint2(pack4(qv.code(xv[0]), qv.code(xv[1]), qv.code(xv[2]), qv.code(xv[3])),
                                                                      pack4(qv.code(xv[4]), qv.code(xv[5]), qv.code(xv[6]), qv.code(xv[7])));
    if (l8 == 0) { a.c.k_scale_dev[row] = qk.scale; a.c.v_scale_dev[row] = qv.scale; }
  }
}

__device__ __forceinline__ void codes8(uint2 w, float s, float v[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = (float)(int8_t)(w.x >> (8 * e)) * s;
    v[4 + e] = (float)(int8_t)(w.y >> (8 * e)) * s;
  }
}

template <typename T, int HD>
__global__ __launch_bounds__(256) void kv8_read_kernel(const Kv8Args a, T* __restrict__ k, int64_t ldk, T* __restrict__ v, int64_t ldv) {
  constexpr int L = HD / 8, PER = 256 / L;
  const Span s = span_of(a, blockIdx.y);
  const int l8 = (threadIdx.x % L) * 8, heads = a.c.heads;
  const int64_t tasks = (int64_t)s.n * heads;
  for (int64_t task = (int64_t)blockIdx.x * PER + threadIdx.x / L; task < tasks; task += (int64_t)gridDim.x * PER) {
    const int t = (int)(task / heads), head = (int)(task - (int64_t)t * heads), pos = s.pos0 + t;
    float xk[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, xv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (s.slot >= 0 && pos >= 0 && pos < a.c.ctx) {
      const int64_t row = ((int64_t)s.slot * heads + head) * a.c.ctx + pos;
      const uint2 wk = *reinterpret_cast<const uint2*>(a.c.k_dev + row * HD + l8), wv = *reinterpret_cast<const uint2*>(a.c.v_dev + row * HD + l8);
      codes8(wk, a.c.k_scale_dev[row], xk);
      codes8(wv, a.c.v_scale_dev[row], xv);
    }
    st8<T>(k + (int64_t)(s.first + t) * ldk + head * HD + l8, xk);
    st8<T>(v + (int64_t)(s.first + t) * ldv + head * HD + l8, xv);
  }
}

// --------------------------------------------------------------------------------------------
// Attention over the cache.
//
// Per key / value head the rows of a sequence are its (new row, query head of the group) pairs, r = t * per + g; a workgroup takes
// 16 RT of them and a range of positions, its waves (four, or eight for 16 rows) take 32 positions at a time in turn.  Codes go from memory straight into the
// operands of the matrix cores: S^T = K Q^T per 16 positions, the positions of two such products permuted so that the weights leave the
// first product in the order the second one, O^T += V^T P^T, wants them.  An int8 code is exact in float16 (byte | 0x6400 is 1024 + byte,
// minus 1152), so the products lose nothing of the cache; the query is carried in units of a power of two that bounds its row, exact for
// 16-bit types, as a high and a low half (22 bits) for float32.
//
// Weights: with x = scale * log2(e) * ks * (q . k), the numerator of a position is 2^x vs, and 16 bits must hold it whatever the
// scales are.  So the running reference of a row is M = max(x + exponent of vs) - 11, numerators are 2^(x - M) vs (at most 2^15), the
// denominator sums 2^(x - M) in float32.  A scale has an exponent of up to 128, which puts the denominator's terms down at 2^-117, where the exponential
// gives nothing below 2^-126: M and with it the exponentials are carried 20 binades higher, the scales and the denominator's terms taken 20 lower.
// Exponents below -90 count as -90, so that a term is at most 2^105: scales below 2^-105 lose bits of their numerators.
// M moves only when the largest numerator would pass 2^15.  The smallest step of a half, 2^-24, is then 2^-34 of the row's largest numerator or
// less: what a weight can lose for being small.  A numerator goes into the product as a high and a low half (21 bits or more): the results are
// those of the float32 form.  With one half a float16 row ends up 3.0e-4 off instead of 2.1e-4 and a bfloat16 row 1.671e-3 instead of 1.658e-3
// (8 % of its values are not the nearest ones, against 0.06 %); the second product costs nothing where memory bounds the call (512 sequences
// 124 us) and 11 to 16 % of a bfloat16 prompt pass (32 prompts 142 -> 157 us).
// --------------------------------------------------------------------------------------------
struct AttnArgs {
  Kv8Args s;
  const void* q; int64_t ldq;
  void* out; int64_t ldo;
  int n_heads, per, causal;
  uint32_t per_inv;          // ceil(2^32 / per): r / per is the high word of r * per_inv for r < 2^28 (per = 1: 0, see over_per)
  float scale2;              // scale * log2(e)
  int chunk, nsplit;         // positions per workgroup; workgroups per row block (the last takes what is left)
  float* part;               // nsplit > 1: numerator sums [row * n_heads + head][nsplit][dim]
  float2* ml;                // ... and (M, denominator)
};

constexpr float kRoom = 31.f, kSlack = 35.f, kDown = 0x1p-20f;
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

// Eight numerators as high and low halves.  The high ones are cut off instead of rounded, two at an instruction: the low ones hold what is left.
__device__ __forceinline__ void split_halves(const float (&w)[8], f16x8_t (&out)[2]) {
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(w[2 * j], w[2 * j + 1]);
    hi[j] = __builtin_bit_cast(uint32_t, h);
    lo[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(w[2 * j] - (float)h[0], w[2 * j + 1] - (float)h[1]));
  }
  out[0] = __builtin_bit_cast(f16x8_t, make_uint4(hi[0], hi[1], hi[2], hi[3]));
  out[1] = __builtin_bit_cast(f16x8_t, make_uint4(lo[0], lo[1], lo[2], lo[3]));
}

__device__ __forceinline__ uint32_t h2_less(uint32_t w) {      // two halves, 1152 taken off each
  const h2_t c = {(_Float16)1152.f, (_Float16)1152.f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, w) - c);
}
// 8 codes of one position -> 8 halves
__device__ __forceinline__ f16x8_t codes_to_h8(uint32_t a, uint32_t b) {
  a ^= 0x80808080u; b ^= 0x80808080u;
  uint4 r;
  r.x = h2_less(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u));
  r.y = h2_less(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u));
  r.z = h2_less(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u));
  r.w = h2_less(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u));
  return __builtin_bit_cast(f16x8_t, r);
}
// byte E of two positions' words (already ^ 0x80808080) -> two halves
template <int E> __device__ __forceinline__ uint32_t codes_pair(uint32_t first, uint32_t second) {
  return h2_less(__builtin_amdgcn_perm(second, first, 0x0c000c00u | ((uint32_t)(4 + E) << 16) | (uint32_t)E) | 0x64006400u);
}

__device__ __forceinline__ float quad_max(float x) {      // over the four lanes that share lane & 15
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t v = __float_as_uint(x);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

__device__ __forceinline__ float scale_exponent(float vs) {      // of a value scale, bounded so that 2^(x - M) and its sums stay in range
  return vs == 0.f ? -90.f : fmaxf((float)__builtin_amdgcn_frexp_expf(vs), -90.f);
}

__device__ __forceinline__ int over_per(const AttnArgs& a, int r) { return a.per == 1 ? r : (int)__umulhi((uint32_t)r, a.per_inv); }

// the positions that rows r0 .. of a block may see at most, and the row's own
__device__ __forceinline__ int row_limit(const AttnArgs& a, const Span& s, int r) {
  if (s.slot < 0) return 0;
  return max(0, min(a.s.c.ctx, a.causal ? s.pos0 + over_per(a, r) + 1 : s.len));
}

// The query operands of row r: piece c holds dims lg * (HD / 4) + 8 c (or, INTERLEAVED, 32 c + 8 lg), NP halves each; returns what a product
// counts in units of log2.  float16 rows go in as they are.  The others are counted in units of a power of two that bounds the row: a
// bfloat16 value is then exact in float16 down to 2^-14 of the row's largest, a float32 one is its high and its low half (22 bits).
// A row that is not finite makes NaN of its own scores.
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
template <typename T, int HD, int NP, bool INTERLEAVED>
__device__ __forceinline__ float load_query(const AttnArgs& a, const Span& s, int kvh, int r, int rows, int lg, f16x8_t (&qf)[NP][HD / 32]) {
  constexpr int KS = HD / 32;
  Raw8<T> raw[KS];
#pragma unroll
  for (int c = 0; c < KS; ++c)
#pragma unroll
    for (int w = 0; w < (int)(2 * sizeof(T)); ++w) raw[c].w[w] = 0u;
  if (r < rows) {
    const int t = over_per(a, r);
    const T* p = reinterpret_cast<const T*>(a.q) + (int64_t)(s.first + t) * a.ldq + (kvh * a.per + r - t * a.per) * HD;
#pragma unroll
    for (int c = 0; c < KS; ++c) raw[c] = ld_raw8(p + (INTERLEAVED ? 32 * c + 8 * lg : lg * (HD / 4) + 8 * c));
  }
  if constexpr (std::is_same<T, f16_t>::value) {
#pragma unroll
    for (int c = 0; c < KS; ++c) qf[0][c] = __builtin_bit_cast(f16x8_t, raw[c]);
    return a.scale2;
  } else {
    float v[KS][8], top = 0.f;
    if constexpr (sizeof(T) == 2) {
      u16x2_t t = {0, 0};
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int w = 0; w < 4; ++w) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2_t, raw[c].w[w] & 0x7fff7fffu));
      top = mag(__uint_as_float((uint32_t)max(t[0], t[1]) << 16));
    }
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      widen8(raw[c], v[c]);
      if constexpr (sizeof(T) == 4)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, mag(v[c][e]));
    }
    top = quad_max(top);
    const bool fine = top < INFINITY;
    const int ex = top > 0.f && fine ? max(__builtin_amdgcn_frexp_expf(top), -120) : 0;
    const float down = fine ? ldexpf(1.f, -ex) : 0.f;
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = v[c][e] * down;
        const f16_t hi = f2h(x);
        qf[0][c][e] = hi;
        if constexpr (NP == 2) qf[1][c][e] = f2h(x - h2f(hi));
      }
    return fine ? ldexpf(a.scale2, ex) : __uint_as_float(0x7fc00000u);
  }
}

template <typename T, int N> __device__ __forceinline__ void st_out(T* p, const float* v) {      // any alignment: gfx950 serves wide unaligned stores
  T t[N];
#pragma unroll
  for (int e = 0; e < N; ++e) t[e] = to_T<T>(v[e]);
  __builtin_memcpy(p, t, sizeof(t));
}

// A denominator brought to a reference that is -by higher, in two steps: beyond 2^-126 the factor would be zero.  The numerators add nothing to
// the result then, but the denominator may hold the weights of positions whose values are that much smaller.
__device__ __forceinline__ float lower_sum(float sum, float by) {
  const float f = __builtin_amdgcn_exp2f(0.5f * by);
  return sum * f * f;
}

// Parts of one row over different positions, each with its reference and denominator: brought to the largest reference and added.  A part
// that saw nothing (reference -inf, zeros) adds nothing; one that holds a NaN makes one of the sum.
template <int N> struct Part {
  float top = -INFINITY, sum = 0.f, o[N] = {};
  __device__ __forceinline__ void see(float2 ml) { top = fmaxf(top, ml.x); }
  __device__ __forceinline__ void add(float2 ml, const float* part) {
    const float by = ml.x - (top == -INFINITY ? 0.f : top), f = __builtin_amdgcn_exp2f(by);
    sum += lower_sum(ml.y, by);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = fmaf(part[e], f, o[e]);
  }
  __device__ __forceinline__ void finish(bool seen) {
    const float inv = 1.f / sum;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = seen ? o[e] * inv : 0.f;
  }
};

// Bound by memory where there are many sequences: 512 of 250 .. 1000 positions, 16 heads on 8 of 128, 124 us, 5.5 TB/s.  One sequence of 448
// positions takes 7.6 us: the launch, two turns of each wave, and the meeting in LDS.
template <typename T, int HD, int RT, int NV>      // NV waves
__global__ __launch_bounds__(NV * 64, sizeof(T) == 4 && RT == 2 ? 1 : 2) void kv8_attn_rows_kernel(const AttnArgs a) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;                              // halves of a query
  constexpr int NE = HD / 16;                  // 16-dim tiles of the output; a lane's output dims are NE consecutive ones, four times
  constexpr int KW = HD / 64;                  // 16-byte pieces of a key per lane
  constexpr int LDO = HD + 4;
  __shared__ __attribute__((aligned(16))) float lo[NV * 16 * LDO];
  __shared__ float2 lml[NV * 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
  const int kvh = blockIdx.y;
  const Span s = span_of(a.s, blockIdx.z);
  const int split = blockIdx.x % a.nsplit, blocks = gridDim.x / a.nsplit;
  const int64_t rows = (int64_t)s.n * a.per;
  for (int64_t r0 = (int64_t)(blockIdx.x / a.nsplit) * 16 * RT; r0 < rows; r0 += (int64_t)blocks * 16 * RT) {
    const int first = (int)r0, last = (int)min(rows, r0 + 16 * RT) - 1;
    const int every = row_limit(a, s, first), all = row_limit(a, s, last);      // positions that every row / some row of the block sees
    const int kbeg = split * a.chunk;
    const int kend = split == a.nsplit - 1 ? all : min(all, kbeg + a.chunk);
    if (split > 0 && kbeg >= kend) continue;                                    // the join does not read this part
    const int64_t row0 = ((int64_t)max(s.slot, 0) * a.s.c.heads + kvh) * a.s.c.ctx;
    const int8_t* kp = a.s.c.k_dev + row0 * HD;
    const int8_t* vp = a.s.c.v_dev + row0 * HD;
    const float* ksp = a.s.c.k_scale_dev + row0;
    const float* vsp = a.s.c.v_scale_dev + row0;

    f16x8_t qf[RT][NP][HD / 32];
    float unit[RT], M[RT], l[RT];
    int limit[RT];
    f32x4_t o[RT][NE];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = first + t * 16 + li;
      unit[t] = load_query<T, HD, NP, false>(a, s, kvh, r, (int)rows, lg, qf[t]);
      limit[t] = r <= last ? min(kend, row_limit(a, s, r)) : kend;
      M[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) o[t][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    auto tile = [&](const int kt, auto masked_tag) __attribute__((always_inline)) {
      constexpr bool MASKED = decltype(masked_tag)::value;
      // codes of this lane's keys (two rows of K, eight of V) and scales of its eight positions kt + 8 lg ..
      uint4 kw[2][KW];
      uint32_t vw[8][HD / 64];
      float ks[8], vs[8];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        int key = kt + 8 * (li >> 2) + 4 * t2 + (li & 3);
        if (MASKED) key = min(key, kend - 1);
#pragma unroll
        for (int c = 0; c < KW; ++c) kw[t2][c] = *reinterpret_cast<const uint4*>(kp + (int64_t)key * HD + lg * (HD / 4) + c * 16);
      }
      if (MASKED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = min(kt + 8 * lg + j, kend - 1);
          ks[j] = ksp[key]; vs[j] = vsp[key];
        }
      } else {
        __builtin_memcpy(ks, ksp + kt + 8 * lg, 32);
        __builtin_memcpy(vs, vsp + kt + 8 * lg, 32);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        int key = kt + 8 * lg + j;
        if (MASKED) key = min(key, kend - 1);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(vp + (int64_t)key * HD + li * (HD / 16));
        if constexpr (HD == 128) {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
          vw[j][0] = u.x; vw[j][1] = u.y;
        } else {
          vw[j][0] = *src;
        }
      }
      float ex[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) { ex[j] = scale_exponent(vs[j]); vs[j] *= kDown; }
      f32x4_t st[RT][2];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
#pragma unroll
        for (int t = 0; t < RT; ++t) st[t][t2] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KW; ++c) {
          const f16x8_t k0 = codes_to_h8(kw[t2][c].x, kw[t2][c].y), k1 = codes_to_h8(kw[t2][c].z, kw[t2][c].w);
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              st[t][t2] = mfma16(k0, qf[t][p][2 * c], st[t][t2]);
              st[t][t2] = mfma16(k1, qf[t][p][2 * c + 1], st[t][t2]);
            }
        }
      }
      f16x8_t pf[RT][2];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float x[8], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = st[t][j >> 2][j & 3] * ks[j];
          const bool in = !MASKED || kt + 8 * lg + j < limit[t];
          top = fmaxf(top, in ? fmaf(x[j], unit[t], ex[j]) : -INFINITY);
        }
        top = quad_max(top);
        if (top > M[t] + kSlack) {
          const float by = M[t] - (top - kRoom), f = __builtin_amdgcn_exp2f(by);      // the first time: 0 on zeros
          M[t] = top - kRoom;
          l[t] = lower_sum(l[t], by);
#pragma unroll
          for (int e = 0; e < NE; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][e][r] *= f;
        }
        const float m = M[t] == -INFINITY ? 0.f : M[t];
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = !MASKED || kt + 8 * lg + j < limit[t];
          const float p = in ? __builtin_amdgcn_exp2f(fmaf(x[j], unit[t], -m)) : 0.f;
          l[t] = fmaf(p, kDown, l[t]);
          w[j] = in ? p * vs[j] : 0.f;
        }
        split_halves(w, pf[t]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) vw[j][c] ^= 0x80808080u;
      auto value_tile = [&](auto e_tag) __attribute__((always_inline)) {
        constexpr int E = decltype(e_tag)::value, C = E >> 2, B = E & 3;
        uint4 u;
        u.x = codes_pair<B>(vw[0][C], vw[1][C]); u.y = codes_pair<B>(vw[2][C], vw[3][C]);
        u.z = codes_pair<B>(vw[4][C], vw[5][C]); u.w = codes_pair<B>(vw[6][C], vw[7][C]);
        const f16x8_t vf = __builtin_bit_cast(f16x8_t, u);
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int p = 0; p < 2; ++p) o[t][E] = mfma16(vf, pf[t][p], o[t][E]);
      };
      value_tile(std::integral_constant<int, 0>{}); value_tile(std::integral_constant<int, 1>{});
      value_tile(std::integral_constant<int, 2>{}); value_tile(std::integral_constant<int, 3>{});
      if constexpr (HD == 128) {
        value_tile(std::integral_constant<int, 4>{}); value_tile(std::integral_constant<int, 5>{});
        value_tile(std::integral_constant<int, 6>{}); value_tile(std::integral_constant<int, 7>{});
      }
    };
    for (int kt = kbeg + 32 * wave; kt < kend; kt += 32 * NV) {
      if (kt + 32 <= min(every, kend)) tile(kt, std::false_type{});
      else tile(kt, std::true_type{});
    }

    // the waves' parts meet in LDS, 16 rows at a time
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (first + t * 16 > last) break;
      __syncthreads();
      const float lsum = quad_sum(l[t]);
      if (lg == 0) lml[wave * 16 + li] = make_float2(M[t], lsum);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float* d = &lo[(wave * 16 + li) * LDO + NE * (4 * lg + r)];
#pragma unroll
        for (int e = 0; e < NE; e += 4) *reinterpret_cast<float4*>(d + e) = make_float4(o[t][e][r], o[t][e + 1][r], o[t][e + 2][r], o[t][e + 3][r]);
      }
      __syncthreads();
      const int row = tid >> 4, r = first + t * 16 + row, d0 = (tid & 15) * NE;
      if (tid < 256 && r <= last) {
        Part<NE> p;
#pragma unroll
        for (int w = 0; w < NV; ++w) p.see(lml[w * 16 + row]);
#pragma unroll
        for (int w = 0; w < NV; ++w) p.add(lml[w * 16 + row], &lo[(w * 16 + row) * LDO + d0]);
        const int t1 = over_per(a, r);
        const int64_t at = s.first + t1, head = kvh * a.per + r - t1 * a.per;
        if (a.nsplit == 1) {
          p.finish(row_limit(a, s, r) > 0);
          st_out<T, NE>(reinterpret_cast<T*>(a.out) + at * a.ldo + head * HD + d0, p.o);
        } else {
          const int64_t slot = (at * a.n_heads + head) * a.nsplit + split;
          if ((tid & 15) == 0) a.ml[slot] = make_float2(p.top, p.sum);
#pragma unroll
          for (int e = 0; e < NE; e += 4) *reinterpret_cast<float4*>(a.part + slot * HD + d0 + e) = make_float4(p.o[e], p.o[e + 1], p.o[e + 2], p.o[e + 3]);
        }
      }
    }
  }
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// `bytes` bytes from p as a buffer: loads past them give zeros
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(void* p, int bytes) { return __builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, 0x00027000); }

// Many rows: 128 rows of one key / value head per workgroup, 32 per wave, positions 64 at a time through LDS.  The codes are widened to
// halves ONCE per workgroup on their way into LDS (both operands in the order the products read them: K rows permuted, V transposed in
// registers, 8 positions of one dimension per 16-byte piece), which the rows kernel above does once per wave.  The next 64 positions are
// in flight (registers) while this wave's products run.  Two buffers, one barrier per step, two workgroups per CU.  Bound by the vector unit
// (widening, softmax; busy 50 % of the cycles) beside the matrix pipe (24 %): 32 bfloat16 prompts of 250 .. 1000 positions, 16 heads on 8 of 128, 157 us
// (299 with 32 rows per workgroup, when a numerator was one half); 4 of 4000 positions, 32 heads on 8, 823 us, 637 TFLOP/s of what the causal mask
// leaves; float16 148 and 791 us.
template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void kv8_attn_tile_kernel(const AttnArgs a, int blocks) {
  constexpr int NP = 1;
  constexpr int NE = HD / 16, KS = HD / 32;
  constexpr int KB = 64 * HD * 2, VB = 64 * HD * 2, BUF = KB + VB + 3 * 256;       // K [64][HD], V^T [HD][64], then ks, 2^-20 vs, exponents of vs [64]
  constexpr int KL = HD / 64;                                                      // 16-byte pieces of K per thread
  extern __shared__ __attribute__((aligned(16))) char lds_t[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
  // Workgroups go to the 8 XCDs in turn: all row blocks of one (sequence, head) on one XCD.  Under a causal mask later blocks see more: the
  // last blocks of every (sequence, head) come first, so that short ones fill the end.
  const int groups = a.s.b.seqs * a.s.c.heads, per_xcd = (groups + 7) >> 3;
  const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3, rank = idx / per_xcd, group = (idx - rank * per_xcd) * 8 + xcd;
  if (group >= groups) return;
  const int seq = group / a.s.c.heads, kvh = group - seq * a.s.c.heads;
  const Span s = span_of(a.s, seq);
  const int rows = s.n * a.per, n_blocks = (rows + 127) >> 7;
  const int64_t row0 = ((int64_t)max(s.slot, 0) * a.s.c.heads + kvh) * a.s.c.ctx;
  const auto k_buf = buffer_of(a.s.c.k_dev + row0 * HD, a.s.c.ctx * HD), v_buf = buffer_of(a.s.c.v_dev + row0 * HD, a.s.c.ctx * HD);
  const auto ks_buf = buffer_of(a.s.c.k_scale_dev + row0, a.s.c.ctx * 4), vs_buf = buffer_of(a.s.c.v_scale_dev + row0, a.s.c.ctx * 4);
  // (a sequence of fewer blocks sits out the first ranks; one of more than `blocks` takes several)
  for (int block = n_blocks > blocks ? n_blocks - 1 - rank : blocks - 1 - rank; block >= 0; block -= blocks) {
    if (block >= n_blocks) break;
    const int first = block * 128, last = min(rows, first + 128) - 1;
    const int wfirst = first + wave * 32, wlast = min(last, wfirst + 31);
    const int kend = row_limit(a, s, last);                                        // positions the workgroup walks
    const int wend = wfirst <= last ? row_limit(a, s, wlast) : 0, every = wfirst <= last ? row_limit(a, s, wfirst) : 0;

    // this thread's share of 64 positions: KL pieces of K; 8 positions x 4 dimensions of V (HD = 64: half of the threads); one scale.
    // Positions behind kend are fetched like the others (their weights are cleared); those behind the slot's last one read as zeros, which is
    // what a buffer load gives past its range.
    u32x4_t rk[KL];
    uint32_t rv[8], rs = 0;
    const int vd = tid % (HD / 4), vg = tid / (HD / 4);                            // V: dimensions 4 vd .., positions 8 vg ..
    const bool has_v = HD == 128 || vg < 8;
    auto fetch = [&](int kt) __attribute__((always_inline)) {
      const int k = kt * HD + tid * 16, v = kt * HD + vg * 8 * HD + vd * 4;        // bytes from the slot's first position
#pragma unroll
      for (int i = 0; i < KL; ++i) rk[i] = __builtin_amdgcn_raw_buffer_load_b128(k_buf, k + i * 4096, 0, 0);
      if (has_v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) rv[j] = __builtin_amdgcn_raw_buffer_load_b32(v_buf, v + j * HD, 0, 0);
      }
      if (tid < 64) rs = __builtin_amdgcn_raw_buffer_load_b32(ks_buf, (kt + tid) * 4, 0, 0);
      else if (tid < 128) rs = __builtin_amdgcn_raw_buffer_load_b32(vs_buf, (kt + tid - 64) * 4, 0, 0);
    };
    int k_put[KL];                                                                 // the first of a piece's two halves; the second: ^ 16
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int u = i * 256 + tid, key = u / (HD / 16), c = (u % (HD / 16)) * 2;
      // the row this position has in the first product's operand
      const int row = (key >> 5) * 32 + ((key >> 2) & 1) * 16 + ((key >> 3) & 3) * 4 + (key & 3);
      k_put[i] = row * (HD * 2) + ((c ^ (row & (HD / 8 - 1))) << 4);
    }
    const int v_put[2] = {KB + vd * 512 + ((vg ^ ((2 * vd) & 7)) << 4), KB + vd * 512 + ((vg ^ ((2 * vd + 1) & 7)) << 4)};
    auto put = [&](int buf) __attribute__((always_inline)) {
      char* b = lds_t + buf * BUF;
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        *reinterpret_cast<f16x8_t*>(b + k_put[i]) = codes_to_h8(rk[i].x, rk[i].y);
        *reinterpret_cast<f16x8_t*>(b + (k_put[i] ^ 16)) = codes_to_h8(rk[i].z, rk[i].w);
      }
      if (has_v) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = rv[j] ^ 0x80808080u;
        char* v = b + v_put[0];
        char* v2 = b + v_put[1];
        *reinterpret_cast<uint4*>(v) = make_uint4(codes_pair<0>(w[0], w[1]), codes_pair<0>(w[2], w[3]), codes_pair<0>(w[4], w[5]), codes_pair<0>(w[6], w[7]));
        *reinterpret_cast<uint4*>(v + 128) = make_uint4(codes_pair<1>(w[0], w[1]), codes_pair<1>(w[2], w[3]), codes_pair<1>(w[4], w[5]), codes_pair<1>(w[6], w[7]));
        *reinterpret_cast<uint4*>(v2 + 256) = make_uint4(codes_pair<2>(w[0], w[1]), codes_pair<2>(w[2], w[3]), codes_pair<2>(w[4], w[5]), codes_pair<2>(w[6], w[7]));
        *reinterpret_cast<uint4*>(v2 + 384) = make_uint4(codes_pair<3>(w[0], w[1]), codes_pair<3>(w[2], w[3]), codes_pair<3>(w[4], w[5]), codes_pair<3>(w[6], w[7]));
      }
      float* sc = reinterpret_cast<float*>(b + KB + VB);
      if (tid < 64) sc[tid] = __uint_as_float(rs);
      else if (tid < 128) { sc[tid] = __uint_as_float(rs) * kDown; sc[64 + tid] = scale_exponent(__uint_as_float(rs)); }
    };

    if (kend > 0) fetch(0);                // in flight while the queries are read
    f16x8_t qf[2][NP][KS];
    float unit[2], M[2], l[2];
    int limit[2];
    f32x4_t o[2][NE];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = wfirst + t * 16 + li;
      unit[t] = load_query<T, HD, NP, true>(a, s, kvh, r, rows, lg, qf[t]);
      limit[t] = r <= last ? row_limit(a, s, r) : kend;
      M[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) o[t][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // this lane's place in the buffers.  Pieces are swapped within their rows (K: 16 pieces of a 256-byte row or 8 of a 128-byte one; V: 8)
    // so that the 16 lanes that LDS serves together (0-3, 12-15, 20-27 and so on) reach different banks
    int k_at[KS], v_at[2];
#pragma unroll
    for (int c = 0; c < KS; ++c) k_at[c] = li * (HD * 2) + (((c * 4 + lg) ^ (li & (HD / 8 - 1))) << 4);
    v_at[0] = KB + li * 128 + ((lg ^ (li >> 1)) << 4);
    v_at[1] = v_at[0] ^ 64;
    // 32 positions: half H of the buffer's 64
    auto tile = [&](const int kt, const int buf, auto half_tag, auto masked_tag) __attribute__((always_inline)) {
      constexpr int H = decltype(half_tag)::value;
      constexpr bool MASKED = decltype(masked_tag)::value;
      const char* b = lds_t + buf * BUF;
      float ks[8], vs[8], ex[8];
      {
        const float* sc = reinterpret_cast<const float*>(b + KB + VB) + H * 32 + lg * 8;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          *reinterpret_cast<float4*>(ks + j) = *reinterpret_cast<const float4*>(sc + j);
          *reinterpret_cast<float4*>(vs + j) = *reinterpret_cast<const float4*>(sc + 64 + j);
          *reinterpret_cast<float4*>(ex + j) = *reinterpret_cast<const float4*>(sc + 128 + j);
        }
      }
      const int key0 = kt + H * 32 + lg * 8;
      f32x4_t st[2][2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        st[0][kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        st[1][kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          const f16x8_t kf = *reinterpret_cast<const f16x8_t*>(b + k_at[c] + (H * 32 + kb * 16) * (HD * 2));
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int p = 0; p < NP; ++p) st[t][kb] = mfma16(kf, qf[t][p][c], st[t][kb]);
        }
      }
      f16x8_t pf[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float x[8], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = st[t][j >> 2][j & 3] * ks[j];
          const bool in = !MASKED || key0 + j < limit[t];
          top = fmaxf(top, in ? fmaf(x[j], unit[t], ex[j]) : -INFINITY);
        }
        top = quad_max(top);
        if (top > M[t] + kSlack) {
          const float by = M[t] - (top - kRoom), f = __builtin_amdgcn_exp2f(by);
          M[t] = top - kRoom;
          l[t] = lower_sum(l[t], by);
#pragma unroll
          for (int e = 0; e < NE; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][e][r] *= f;
        }
        const float m = M[t] == -INFINITY ? 0.f : M[t];
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = !MASKED || key0 + j < limit[t];
          const float p = in ? __builtin_amdgcn_exp2f(fmaf(x[j], unit[t], -m)) : 0.f;
          l[t] = fmaf(p, kDown, l[t]);
          w[j] = in ? p * vs[j] : 0.f;
        }
        split_halves(w, pf[t]);
      }
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const f16x8_t vf = *reinterpret_cast<const f16x8_t*>(b + v_at[H] + e * 2048);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int p = 0; p < 2; ++p) o[t][e] = mfma16(vf, pf[t][p], o[t][e]);
      }
    };

    __syncthreads();                       // the block before has read its last buffer
    if (kend > 0) put(0);
    __syncthreads();
    int buf = 0;
    for (int kt = 0; kt < kend; kt += 64, buf ^= 1) {
      const bool more = kt + 64 < kend;
      if (more) fetch(kt + 64);
      if (kt + 32 <= every) tile(kt, buf, std::integral_constant<int, 0>{}, std::false_type{});
      else if (kt < wend) tile(kt, buf, std::integral_constant<int, 0>{}, std::true_type{});
      if (kt + 64 <= every) tile(kt, buf, std::integral_constant<int, 1>{}, std::false_type{});
      else if (kt + 32 < wend) tile(kt, buf, std::integral_constant<int, 1>{}, std::true_type{});
      if (more) put(buf ^ 1);
      __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float sum = quad_sum(l[t]);
      const int r = wfirst + t * 16 + li;
      if (r > last) continue;
      const float inv = limit[t] > 0 ? 1.f / sum : 0.f;      // a row that sees nothing has added nothing: zeros
      const int t1 = over_per(a, r);
      T* out = reinterpret_cast<T*>(a.out) + (int64_t)(s.first + t1) * a.ldo + (kvh * a.per + r - t1 * a.per) * HD + lg * 4;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = o[t][e][i] * inv;
        st_out<T, 4>(out + e * 16, v);
      }
    }
  }
}

// The parts of every row's positions joined, in order: 16 lanes per (row, head)
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv8_attn_join_kernel(const AttnArgs a, int block_rows) {
  constexpr int NE = HD / 16;
  const Span s = span_of(a.s, blockIdx.y);
  const int d0 = (threadIdx.x & 15) * NE;
  const int total = s.n * a.n_heads;
  for (int i = blockIdx.x * 16 + (threadIdx.x >> 4); i < total; i += gridDim.x * 16) {
    const int t = i / a.n_heads, head = i - t * a.n_heads, r = t * a.per + head % a.per;
    const int last = min(s.n * a.per, (r / block_rows + 1) * block_rows) - 1;         // of the row's block: its workgroups went by that limit
    const int parts = min(a.nsplit, max(1, (row_limit(a, s, last) + a.chunk - 1) / a.chunk));
    const int64_t slot = ((int64_t)(s.first + t) * a.n_heads + head) * a.nsplit;
    Part<NE> p;
    for (int j = 0; j < parts; ++j) p.see(a.ml[slot + j]);
    for (int j = 0; j < parts; ++j) p.add(a.ml[slot + j], a.part + (slot + j) * HD + d0);
    p.finish(row_limit(a, s, r) > 0);
    st_out<T, NE>(reinterpret_cast<T*>(a.out) + (int64_t)(s.first + t) * a.ldo + head * HD + d0, p.o);
  }
}

// the launch's sizes go by the hints as far as they can be true
int most_new(const wj_kv8_batch& b) { return wj::most_new(b.max_new, b.rows); }
AttnPlan plan_attention(const wj_kv8& c, const wj_kv8_batch& b, int n_heads) {
  return wj::plan_attention(c.heads, c.ctx, c.dim, b.seqs, most_new(b), b.max_len, n_heads);
}

int check_kv8(const char* who, wj_ctx* ctx, const wj_kv8* c, const wj_kv8_batch* b, int dtype) {
  WJ_REQUIRE(ctx && c && b, "%s: NULL argument", who);
  WJ_REQUIRE(known_dtype(dtype), "%s: unknown dtype %d", who, dtype);
  WJ_REQUIRE(c->dim == 64 || c->dim == 128, "%s: head dimension %d (64 and 128 are built)", who, c->dim);
  WJ_REQUIRE(c->slots >= 0 && c->ctx >= 0 && c->heads >= 1 && c->heads <= 65535, "%s: a cache of %d slots, %d heads, %d positions", who, c->slots, c->heads, c->ctx);
  WJ_REQUIRE(b->seqs >= 0 && b->seqs <= 65535 && b->rows >= 0 && b->max_new >= 0 && b->max_len >= 0, "%s: a batch of %d sequences (at most 65535), %d rows", who,
             b->seqs, b->rows);
  WJ_REQUIRE(b->seqs == 0 || (b->slots_dev && b->starts_dev && b->lens_dev), "%s: NULL batch array", who);
  const bool empty = (int64_t)c->slots * c->ctx == 0;
  WJ_REQUIRE(empty || (c->k_dev && c->k_scale_dev && c->v_dev && c->v_scale_dev), "%s: NULL cache array", who);
  WJ_REQUIRE(aligned_to(c->k_dev, 16) && aligned_to(c->v_dev, 16) && aligned_to(c->k_scale_dev, 4) && aligned_to(c->v_scale_dev, 4),
             "%s: the cache's codes are not 16-byte aligned (scales: 4)", who);
  return WJ_OK;
}

// (row, head) pairs of a sequence over workgroups, one turn each (four turns: 1500 x 20 heads of 64 6.7 us instead of 5.3, 32 x 640 x 8 heads of 128
// 24.9 instead of 24.8; reading 4.9 / 3.9 and 22.8 / 21.6)
dim3 pair_grid(int64_t pairs, int per, int seqs) {
  const int64_t groups = (pairs + per - 1) / per;
  return dim3((unsigned)(groups < 65536 ? groups : 65536), seqs);
}
template <typename T, int HD>
int start_write(const wj_kv8* c, const wj_kv8_batch* b, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t pairs, hipStream_t s) {
  hipLaunchKernelGGL((kv8_write_kernel<T, HD>), pair_grid(pairs, 256 / (HD / 8), b->seqs), dim3(256), 0, s, Kv8Args{*c, *b}, (const T*)k, ldk, (const T*)v, ldv);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}
template <typename T, int HD>
int start_read(const wj_kv8* c, const wj_kv8_batch* b, void* k, int64_t ldk, void* v, int64_t ldv, int64_t pairs, hipStream_t s) {
  hipLaunchKernelGGL((kv8_read_kernel<T, HD>), pair_grid(pairs, 256 / (HD / 8), b->seqs), dim3(256), 0, s, Kv8Args{*c, *b}, (T*)k, ldk, (T*)v, ldv);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}
int launch_write(const wj_kv8* c, const wj_kv8_batch* b, int dtype, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t pairs, hipStream_t s) {
  if (c->dim == 128) {
    if (dtype == WJ_F32) return start_write<float, 128>(c, b, k, ldk, v, ldv, pairs, s);
    if (dtype == WJ_F16) return start_write<f16_t, 128>(c, b, k, ldk, v, ldv, pairs, s);
    return start_write<bf16_t, 128>(c, b, k, ldk, v, ldv, pairs, s);
  }
  if (dtype == WJ_F32) return start_write<float, 64>(c, b, k, ldk, v, ldv, pairs, s);
  if (dtype == WJ_F16) return start_write<f16_t, 64>(c, b, k, ldk, v, ldv, pairs, s);
  return start_write<bf16_t, 64>(c, b, k, ldk, v, ldv, pairs, s);
}
int launch_read(const wj_kv8* c, const wj_kv8_batch* b, int dtype, void* k, int64_t ldk, void* v, int64_t ldv, int64_t pairs, hipStream_t s) {
  if (c->dim == 128) {
    if (dtype == WJ_F32) return start_read<float, 128>(c, b, k, ldk, v, ldv, pairs, s);
    if (dtype == WJ_F16) return start_read<f16_t, 128>(c, b, k, ldk, v, ldv, pairs, s);
    return start_read<bf16_t, 128>(c, b, k, ldk, v, ldv, pairs, s);
  }
  if (dtype == WJ_F32) return start_read<float, 64>(c, b, k, ldk, v, ldv, pairs, s);
  if (dtype == WJ_F16) return start_read<f16_t, 64>(c, b, k, ldk, v, ldv, pairs, s);
  return start_read<bf16_t, 64>(c, b, k, ldk, v, ldv, pairs, s);
}

template <typename T, int HD, int RT>
int start_attention(const AttnArgs& a, int waves, hipStream_t s) {
  const int64_t rows = (int64_t)most_new(a.s.b) * a.per;
  const dim3 grid((unsigned)((rows + 16 * RT - 1) / (16 * RT) * a.nsplit), a.s.c.heads, a.s.b.seqs);
  if constexpr (RT == 1) {
    if (waves == 8) {
      hipLaunchKernelGGL((kv8_attn_rows_kernel<T, HD, RT, 8>), grid, dim3(512), 0, s, a);
      WJ_LAUNCH_CHECK();
      return WJ_OK;
    }
  }
  hipLaunchKernelGGL((kv8_attn_rows_kernel<T, HD, RT, 4>), grid, dim3(256), 0, s, a);
  WJ_LAUNCH_CHECK();
  if (a.nsplit > 1) {
    const int64_t groups = ((int64_t)most_new(a.s.b) * a.n_heads + 15) / 16;
    hipLaunchKernelGGL((kv8_attn_join_kernel<T, HD>), dim3((unsigned)groups, a.s.b.seqs), dim3(256), 0, s, a, 16 * RT);
    WJ_LAUNCH_CHECK();
  }
  return WJ_OK;
}
template <typename T, int HD>
int start_tile(const AttnArgs& a, hipStream_t s) {
  static AttrOnce once;
  constexpr int lds = 2 * (64 * HD * 4 + 768);
  if (once.need()) {
    WJ_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kv8_attn_tile_kernel<T, HD>), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    once.done();
  }
  const int64_t rows = (int64_t)most_new(a.s.b) * a.per, blocks = (rows + 127) / 128, groups = (int64_t)a.s.b.seqs * a.s.c.heads;
  hipLaunchKernelGGL((kv8_attn_tile_kernel<T, HD>), dim3((unsigned)((groups + 7) / 8 * 8 * blocks)), dim3(256), lds, s, a, (int)blocks);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}
template <int HD, typename T>
int pick_rows(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  if (p.rt == 0) {
    if constexpr (sizeof(T) == 2) return start_tile<T, HD>(a, s);
  }
  return p.rt == 1 ? start_attention<T, HD, 1>(a, p.waves, s) : start_attention<T, HD, 2>(a, p.waves, s);
}
template <int HD>
int pick_type(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t s) {
  if (dtype == WJ_F32) return pick_rows<HD, float>(a, p, s);
  if (dtype == WJ_F16) return pick_rows<HD, f16_t>(a, p, s);
  return pick_rows<HD, bf16_t>(a, p, s);
}

}  // namespace

extern "C" {

int wj_kv8_write(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int dtype, const void* k_dev, int64_t ldk, const void* v_dev,
                 int64_t ldv, void* stream) {
  if (int rc = check_kv8("wj_kv8_write", ctx, cache, batch, dtype)) return rc;
  if (batch->seqs == 0 || batch->rows == 0 || (int64_t)cache->slots * cache->ctx == 0) return WJ_OK;
  WJ_REQUIRE(k_dev && v_dev, "wj_kv8_write: NULL argument");
  WJ_REQUIRE(ldk >= 0 && ldv >= 0, "wj_kv8_write: negative stride");
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  const int64_t pairs = (int64_t)most_new(*batch) * cache->heads;
  return launch_write(cache, batch, dtype, k_dev, ldk, v_dev, ldv, pairs, ctx->pick(stream));
}

int wj_kv8_read(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int dtype, void* k_dev, int64_t ldk, void* v_dev, int64_t ldv,
                void* stream) {
  if (int rc = check_kv8("wj_kv8_read", ctx, cache, batch, dtype)) return rc;
  if (batch->seqs == 0 || batch->rows == 0) return WJ_OK;
  WJ_REQUIRE((int64_t)cache->slots * cache->ctx > 0, "wj_kv8_read: an empty cache");
  WJ_REQUIRE(k_dev && v_dev, "wj_kv8_read: NULL argument");
  WJ_REQUIRE(batch->rows == 1 || (ldk >= cache->heads * cache->dim && ldv >= cache->heads * cache->dim), "wj_kv8_read: output rows overlap");
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  const int64_t pairs = (int64_t)most_new(*batch) * cache->heads;
  return launch_read(cache, batch, dtype, k_dev, ldk, v_dev, ldv, pairs, ctx->pick(stream));
}

int64_t wj_kv8_attention_workspace(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int n_heads) {
  (void)ctx;
  if (!cache || !batch || batch->seqs <= 0 || batch->rows <= 0 || n_heads <= 0 || cache->heads <= 0 || n_heads % cache->heads) return 0;
  const AttnPlan p = plan_attention(*cache, *batch, n_heads);
  return p.nsplit > 1 ? (int64_t)batch->rows * n_heads * p.nsplit * (cache->dim * 4 + 8) : 0;
}

int wj_kv8_attention(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int dtype, const void* q_dev, int64_t ldq, void* out_dev,
                     int64_t ldo, int n_heads, float scale, int causal, void* workspace_dev, int64_t workspace_bytes, void* stream) {
  if (int rc = check_kv8("wj_kv8_attention", ctx, cache, batch, dtype)) return rc;
  WJ_REQUIRE(n_heads >= 1 && n_heads % cache->heads == 0 && n_heads / cache->heads <= 16, "wj_kv8_attention: %d query heads on %d key / value heads (a multiple, at most 16 each)",
             n_heads, cache->heads);
  if (batch->seqs == 0 || batch->rows == 0) return WJ_OK;
  WJ_REQUIRE((int64_t)cache->slots * cache->ctx > 0, "wj_kv8_attention: an empty cache");
  WJ_REQUIRE(q_dev && out_dev, "wj_kv8_attention: NULL argument");
  WJ_REQUIRE((int64_t)batch->rows * n_heads < (int64_t)1 << 28, "wj_kv8_attention: %d rows of %d heads (below 2^28 in all)", batch->rows, n_heads);
  WJ_REQUIRE(ldq >= 0 && (batch->rows == 1 || ldo >= (int64_t)n_heads * cache->dim), "wj_kv8_attention: output rows overlap");
  const int64_t need = wj_kv8_attention_workspace(ctx, cache, batch, n_heads);
  WJ_REQUIRE(workspace_bytes >= need && (workspace_dev || need == 0), "wj_kv8_attention: %lld bytes of workspace, %lld needed", (long long)workspace_bytes, (long long)need);
  WJ_REQUIRE(aligned_to(workspace_dev, 16), "wj_kv8_attention: the workspace is not 16-byte aligned");
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  const AttnPlan p = plan_attention(*cache, *batch, n_heads);
  AttnArgs a{Kv8Args{*cache, *batch}, q_dev, ldq, out_dev, ldo, n_heads, n_heads / cache->heads, causal, 0, scale * 1.44269504088896340736f,
             p.chunk, p.nsplit, reinterpret_cast<float*>(workspace_dev), nullptr};
  if (a.per > 1) a.per_inv = (uint32_t)((((uint64_t)1 << 32) + a.per - 1) / a.per);
  a.ml = reinterpret_cast<float2*>(a.part + (int64_t)batch->rows * n_heads * p.nsplit * cache->dim);
  hipStream_t s = ctx->pick(stream);
  if (cache->dim == 128) return pick_type<128>(a, p, dtype, s);
  return pick_type<64>(a, p, dtype, s);
}

}  // extern "C"
