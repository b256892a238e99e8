// Products of matrices that are held as pairs of halves (pairs.cu), for the operators that work on matrices (fcloss.cu, muon.cu).
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace vlb {

// A matrix of single-precision values x as  x * 2^e = hi + lo * 2^-11  with hi = half(x * 2^e), lo = half((x * 2^e - hi) * 2^11): 22 significant bits where the
// largest magnitude lies in [2^14, 2^15) for everything down to 2^-28 of it, an error of 2^-50 of it below that.  e belongs to 64 rows -- the rows of a k-block where
// they are the reduction -- or is one number.  Rows of ld halves, ld a multiple of 64; what lies between cols and ld is not read.
struct Pair {
  __half *hi, *lo;
  int rows, cols;
  long long ld;
};

inline long long pair_ld(int cols) { return (cols + 63ll) / 64 * 64; }
inline size_t pair_bytes(int rows, int cols) { return 2 * sizeof(__half) * (size_t)rows * pair_ld(cols); }
inline Pair pair_at(void* p, int rows, int cols)
{
  long long const ld = pair_ld(cols);
  return {(__half*)p, (__half*)p + (size_t)rows * ld, rows, cols, ld};
}

// A side of a product: its rows are the matrix's rows and the reduction runs along the columns, or (byCols) the other way round.  lower: of a symmetric
// matrix only the tiles on and under the diagonal are there, as a symmetric product with the same tiles left them.
struct PairSide { Pair m; bool byCols, lower; };

// The exponents of a pair: one per 64 rows, on the device, or a number.
struct PairExp { int const* blocks; int value; };

enum PairKind {
  kPairOut = 0,      // out = [out +] alpha * product
  kPairSeen = 1,     // of the predictions product + bias: largest, sum of exponentials and the label's, per row and half a tile's columns
  kPairGrad = 2,     // (exp(product + bias - lse) - [column is the label]) per row, as a pair scaled by 2^14, and its sums over 32 rows
  kPairPoly = 3      // to = alpha * product + beta * add, as a pair; or w -= rate * that
};

struct PairEpilogue {
  PairExp ea, eb;                   // exponents of the two sides
  float alpha, beta;
  float* out; long long ldc;        // kPairOut (beta 0 or 1); kPairPoly with out: out -= rate * value
  float rate;
  float const *bias, *labels;       // kPairSeen, kPairGrad: columns are the classes firstClass + 0, 1, ...; classes of all pieces for the labels' check
  int firstClass, classes;
  float2* parts; float* label;      // kPairSeen: parts[(2 * column tile + half) * M + row]; the label's prediction per row
  float const* lse; float* db;      // kPairGrad: db[(row / 32) * to.ld + column]; status is told of labels above the classes
  int* status;
  Pair to, add; int toExp, addExp;  // kPairGrad (to), kPairPoly
};

struct PairProduct {
  PairSide a, b;
  int M, N, K;
  bool symmetric;                   // the product is symmetric: only the tiles on and under the diagonal are made
  PairEpilogue e;
};

constexpr int kMaxPairProducts = 16;

// Scratch for the partial results of reductions that are cut, at most.
constexpr size_t kPairSplitBytes = 64u << 20;

// Parts per row that kPairSeen writes of N columns.
inline int pair_parts(int N, int tile) { return 2 * ceil_div(N, tile); }

// A matrix of floats, rows one after the other, to be made a pair, with the exponent of the largest finite magnitude of each 64 rows, left in exps.
// labels (or NULL): rows whose label is not in 1 ... classes count as zeros, whatever they hold.
struct PairSource { Pair to; float const* x; int* exps; float const* labels; int classes; };

// One or two of them.  partial: pair_partials(rows) words of scratch for each, one after the other.
inline size_t pair_partials(int rows) { return (size_t)ceil_div(rows, 64) + 1024; }
void make_pairs(vlb_ctx* ctx, PairSource const* s, int count, unsigned* partial);

// The tiles, 256 x 256 or 128 x 128, that take less time for these products, all of them together.
int pair_tile(vlb_ctx* ctx, PairProduct const* p, int count);

// All products of one kind in one launch, with tiles of `tile` rows and columns.  split: kPairSplitBytes of scratch, 16-byte aligned.
int products_of_pairs(vlb_ctx* ctx, PairKind kind, PairProduct const* p, int count, void* split, int tile);

#ifdef __CUDACC__
// 32 bytes at once, 32-byte aligned
__device__ __forceinline__ void store32(void* p, uint32_t const (&v)[8])
{
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// The exponent that brings the magnitude m into [2^14, 2^15); at most 116, so that 2^e and its inverse are normal numbers.
__device__ __forceinline__ int pair_exp(float m) { return m > 0.f ? min(141 - (int)(__float_as_uint(m) >> 23), 116) : 0; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }        // -126 <= e <= 127

// hi and lo of a value that has been multiplied by 2^e.  An infinity or a not-a-number is all hi.
__device__ __forceinline__ void pair_of(float v, __half& hi, __half& lo)
{
  hi = __float2half_rn(v);
  float const h = __half2float(hi);
  lo = __float2half_rn(fabsf(h) <= 65504.f ? (v - h) * 2048.f : 0.f);
}
// 16 neighbouring values of a row, multiplied by 2^e, into a pair: a whole sector per lane and part
__device__ __forceinline__ void store_pair16(Pair const& to, long long row, int col, float const* v)
{
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    __half h0, l0, h1, l1;
    pair_of(v[2 * i], h0, l0);
    pair_of(v[2 * i + 1], h1, l1);
    hi[i] = (uint32_t)__half_as_ushort(h0) | ((uint32_t)__half_as_ushort(h1) << 16);
    lo[i] = (uint32_t)__half_as_ushort(l0) | ((uint32_t)__half_as_ushort(l1) << 16);
  }
  store32(to.hi + row * to.ld + col, hi);
  store32(to.lo + row * to.ld + col, lo);
}
#endif

}  // namespace vlb
