// q8_plan.hpp -- plain arithmetic of the 8-bit operators, the same on the host and in the kernels: which rows a sequence owns, which kernel a
// call takes.
#pragma once

#include <stdint.h>

namespace wj {

// What a sequence of a call owns.  first .. first + n - 1: its rows of the row arrays; pos0: position of the first of them
struct Span { int slot, first, n, len, pos0; };

// Whatever the arrays hold, the rows lie inside 0 .. rows - 1 and no position passes 32 bits: a sequence that starts before row 0 or ends before
// it starts owns no rows, a negative length is none (its rows lie before position 0).
constexpr Span span_from(int slot, int first, int last, int len, int slots, int rows) {
  const bool there = first >= 0 && first < rows && last > first;
  const int n = there ? (last < rows ? last : rows) - first : 0, positions = len > 0 ? len : 0;
  return Span{slot >= 0 && slot < slots ? slot : -1, there ? first : rows, n, positions, positions - n};
}

// Which kernel a product takes, from its size alone (the workspace follows from it).  Measured on the MI355X, us per call in a graph (both sides of a pair
// in one run; runs differ by up to 10 %):
//   rows / tile: 16 x 5176 x 5824 10.3 / 11.5, 48 x 4096 x 2048 6.3 / 8.6, 64 x 4096 x 2048 7.1 / 9.4, 64 x 12288 x 2048 17.0 / 10.3,
//     32 x 5176 x 5824 14.2 / 11.8: the rows kernel reads the activations once per 16 columns, so beyond 16 rows it is for products where
//     that is at most 36 MiB;
//   tile / big: 2048 x 4096 x 2048 27.6 / 29.6, 3000 x 2048 x 6144 53 / 67, 512 x 12288 x 2048 22 / 30, 1024 x 12288 x 2048 40 / 32,
//     3000 x 4096 x 2048 39 / 31, 1500 x 12288 x 2048 58 / 58: a round of 256 big tiles, filled or not, takes as long as 1000 small ones;
//   tile of 64 / 128 rows: 512 x 5176 x 5824 39 / 31, 3000 x 1190 x 3808 31 / 25, 240 x 12288 x 2048 15.6 / 15.2, 384 x 5176 x 5824 24 / 31, 512 x
//     12288 x 2048 22.6 / 26.9: the larger pays where small ones would share CUs unevenly and large ones have a CU each;
//   big, stores past the caches: 16384 x 12288 x 2048 (402 MB out) 440 -> 398, 8192 x 12288 x 2048 (201 MB) 188 -> 208: for outputs beyond the
//     256 MiB of the memory-side cache;
//   tile, slices 1 / 2 / 4: 100 x 4096 x 2048 10.0 / 11.1 / 11.6, 100 x 2048 x 6144 23 / 15 / 12.5, 512 x 2048 x 6144 22.5 / 19.1 / 19.8: a
//     slice saves its share of the 0.4 us that a step takes and the join costs 3 us, so it pays from 16 steps a slice while CUs are idle.
enum GemmKind { GEMM_ROWS, GEMM_BIG, GEMM_TILE, GEMM_TILE128 };
struct GemmPlan { GemmKind kind; int ksplit; };
constexpr GemmPlan plan_gemm(int64_t m, int n, int k) {
  if (m <= 16 || (m <= 64 && m * k * ((n + 15) / 16) <= (int64_t)36 << 20)) return {GEMM_ROWS, 1};
  const int64_t t256 = ((m + 255) / 256) * ((n + 255) / 256), t64 = ((m + 63) / 64) * ((n + 127) / 128);
  if (t64 > 1000 * ((t256 + 255) / 256)) return {GEMM_BIG, 1};
  if (t64 > 256 && ((m + 127) / 128) * ((n + 127) / 128) <= 256) return {GEMM_TILE128, 1};
  const int steps = (k + 127) / 128;
  int ks = 1;
  while (ks < 8 && t64 * ks * 2 <= 256 && steps > 16 * ks) ks *= 2;
  return {GEMM_TILE, ks};
}

// the launch's sizes go by the hints as far as they can be true
constexpr int most_new(int max_new, int rows) { return max_new < 1 ? 1 : max_new < rows ? max_new : rows; }

// Rows and waves per workgroup and parts per row, from the call's sizes alone (the workspace follows from them).  Measured on the MI355X (us a
// call in a graph; float16, 8 heads of 128 and 1 .. 4 queries each unless said otherwise):
//   16 rows, up to 1024 positions, four / eight waves: 16 sequences x 500 9.1 / 8.2, 16 x 1000 13.5 / 11.9, 64 x 500 13.2 / 15.8, 200 x 500
//     36 / 49: eight where there are fewer than 256 workgroups (four parts and a join: 9.8 and 12.5, and 3.5 us more for the host);
//   16 rows, more positions, one / two / four / eight parts: 1 x 4000 33 / 22 / 16 / 13, 16 x 4000 40 / 28 / 27 / 30, 64 x 1500 33 / 36 / 37 / 39,
//     16 x 20 heads of 64 x 4000 45 / 37 / 34 / 37 (more parts were not measured);
//   32 rows: 1 x 1000 16 / 14 / 12 / 12, 16 x 1000 18 / 17 / 19 / 25, 16 x 4000 53 / 35 / 34 / 40, 64 x 1000 29 / 39 / 49 / 72, 1 x 500 10.6 / 11 / 10.3.
// So parts make up to 512 workgroups, of 256 positions or more, at most 8.
// The 128-row kernel against 32 rows per workgroup, new rows x queries per head, positions: 16 x 100 x 1, 500 25.7 / 19.0; 8 x 128 x 2, 1500 63.5 / 40;
//   32 x 33 x 2, 500 26.1 / 26.0; 32 x 100 x 1, 500 and 1500 28.0 / 32.3 and 66 / 69; 4 x 500 x 2, 500 24.5 / 29.5; 16 x 500 x 2, 500 45 / 101;
//   of 64 dims 32 x 100 x 1, 500 and 1500 20.9 / 21.8 and 53 / 47 (one border for both dims: this last one is on its wrong side): a CU holds two of its workgroups, so it is for calls of more than three blocks
//   of 32 rows per CU; up to 64 rows a sequence its waves would stand half idle (16 x 64 rows 24.0 / 12.6, 32 x 64 25.2 / 19.1).
struct AttnPlan { int rt, waves, nsplit, chunk; };        // rt: 16-row blocks per workgroup, 0: the 128-row kernel (16-bit types; float32 rows take two blocks)
constexpr int kWhole = 0x40000000;
constexpr AttnPlan plan_attention(int heads, int ctx, int dim, int seqs, int new_rows, int max_len, int n_heads) {
  const int per = n_heads / heads;
  const int64_t rows = (int64_t)new_rows * per;
  const int64_t tiles = (int64_t)seqs * heads * ((rows + 127) / 128);
  const int64_t blocks32 = (int64_t)seqs * heads * ((rows + 31) / 32);
  if (rows > 64 && blocks32 > 768 && tiles < 1 << 22 && (int64_t)ctx * dim < 0x7fff0000) return {0, 4, 1, kWhole};
  const int rt = rows <= 16 ? 1 : 2;
  const int64_t groups = (int64_t)seqs * heads * ((rows + 16 * rt - 1) / (16 * rt));
  const int len = max_len < ctx ? (max_len > 0 ? max_len : 1) : ctx;
  if (rt == 1 && len <= 1024) return {1, len > 128 && groups < 256 ? 8 : 4, 1, kWhole};
  int64_t parts = (512 + groups - 1) / groups;
  parts = parts > 8 ? 8 : parts;
  parts = parts > (len + 255) / 256 ? (len + 255) / 256 : parts;
  if (parts <= 1 || (rt == 2 && len <= 512)) return {rt, 4, 1, kWhole};
  const int chunk = (int)(((len + parts - 1) / parts + 127) / 128 * 128);
  return {rt, 4, (len + chunk - 1) / chunk, chunk};
}

}  // namespace wj
