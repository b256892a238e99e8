// Products of matrices held as pairs of halves, on tcgen05 / TMEM with operands delivered by tensor-map copies.
//
// D[i][j] = sum over k of A(i, k) * B(j, k), where A and B are row-major matrices of halves, hi and lo (pairs.cuh), either of which may be read along its rows or
// along its columns: the tensor core takes K-major and MN-major tiles alike, so no operand is ever transposed, and of a symmetric matrix only the tiles on and
// under the diagonal are made and kept: what lies above is read along the other index.  A product of two values is three products of
// halves, lo*hi + hi*lo + hi*hi (lo*lo, 2^-22, is dropped); every k-block of 64 is an accumulation chain of its own in tensor memory, small terms first, then
// hi*hi on the accumulator scaled by 2^-11, and is added to the tile's single-precision running sum, which eight drain warps hold in registers: the tensor
// core truncates when it adds, and twelve additions have no time to pile up.
//
// A tile is 256 x 256 on a pair of CTAs (cta_group::2: each loads 128 rows of A and 128 of B and holds 128 rows of the accumulator) or 128 x 128 on one.
// Roles of a CTA's warps: 0-7 drain (warp w: TMEM lanes 32 (w % 4), half w / 4 of the columns), 8 loads A, 10 loads B, 9 issues the MMAs (of the pair's first
// CTA), 11 completes the warpgroup that gives registers to the drain warps (setmaxnreg moves them by whole warpgroups; a pair's drain threads hold 128 sums each).
// Persistent: CTAs walk the work (product, tile, range of the reduction) in a fixed order (item_at); pipeline indices run through, so a tile's epilogue overlaps the next
// tile's first chains.  A reduction that is cut leaves its partial sums in scratch; the drain warps that take a tile's last ticket add them up in the order of
// the ranges, so results do not depend on timing.
#include "pairs.cuh"
#include "tc_common.cuh"
#include <math.h>

namespace {

using vlb::PairEpilogue; using vlb::PairKind; using vlb::PairProduct; using vlb::Pair;
using vlb::kPairOut; using vlb::kPairSeen; using vlb::kPairGrad; using vlb::kPairPoly;
using vlb::pow2; using vlb::store_pair16;

constexpr int kThreads = 384, kDrainWarps = 8;
constexpr int kLaunchRegs = 168, kDrainRegs = 224, kOtherRegs = 56;     // registers per thread: 8 * 224 + 4 * 56 = 12 * 168
constexpr int kDepth = 64;                       // halves of a k-block: 128 bytes, a row of the swizzle
constexpr int kHalfTile = 128 * kDepth * 2;      // bytes of one operand's hi or lo part of a stage.  Along the rows: hi, lo; along the columns: hi and lo of 64 rows, twice
constexpr int kStageBytes = 4 * kHalfTile, kStages = 3;
constexpr int kRing = 8;                         // barriers of finished k-blocks; more than a waiter can fall behind (3 stages, 4 accumulators)
constexpr int kPatch = 32 * 33;                  // floats of a warp's patch
constexpr size_t kSmem = (size_t)kStages * kStageBytes + kDrainWarps * kPatch * sizeof(float) + 1024;       // (the stages begin at a multiple of 1024)

struct Product {
  int M, N, kBlocks, tilesM, tilesN, splits, work;      // work: items in front of and including this product's
  int byColsA, byColsB, lowerA, lowerB, symmetric;
  int same;                                             // both sides are one matrix: a tile on the diagonal is loaded once
  int slot0; long long part0;                           // tickets and partial results in front of this product's, per CTA of a pair
  PairEpilogue e;
};

template <int kMax> struct Batch {
  CUtensorMap map[4 * kMax];                            // of each product A along its rows, along its columns, B likewise
  Product p[kMax];
  int count, work, three;
  int lead, behind, even;                               // item_at
  int idle;                                             // test switch: nothing is loaded, so that every wait runs out
  float* split;
  int* tickets;
  int* status;
};

// The t-th item of place c of C, or -1: first the longest ones, the first product's `lead` items, with a stride; then the others, of which the `behind` places
// that had one more of the long ones take `even` less than they otherwise would.  Derivatives of 2047 images, 50001 classes (32 tiles of 782 k-blocks beside 784 of
// 32): 1277 us with a stride throughout, 927 so.
template <int kMax>
__device__ __forceinline__ int item_at(Batch<kMax> const& b, int c, int C, int t)
{
  int const first = c < b.lead ? (b.lead - c + C - 1) / C : 0;
  if (t < first) return c + t * C;
  t -= first;
  int w = b.lead + t * C + c;
  if (t >= b.even) {
    if (c < b.behind) return -1;
    w = b.lead + b.even * C + (t - b.even) * (C - b.behind) + c - b.behind;
  }
  return w < b.work ? w : -1;
}

struct Item { int prod, tile, tm, tn, split, kb0, kb1; };

template <int kMax>
__device__ __forceinline__ Item item_of(Batch<kMax> const& b, int w)
{
  Item t;
  t.prod = 0;
  while (kMax > 1 && w >= b.p[t.prod].work) ++t.prod;
  Product const& p = b.p[t.prod];
  if (t.prod) w -= b.p[t.prod - 1].work;
  t.tile = w; t.split = 0;
  t.kb0 = 0; t.kb1 = p.kBlocks;
  if (p.splits > 1) {                                   // (at most 64, of at most 2^25 k-blocks)
    t.tile = w / p.splits;
    t.split = w - t.tile * p.splits;
    t.kb0 = (int)((unsigned)p.kBlocks * (unsigned)t.split / (unsigned)p.splits);
    t.kb1 = (int)((unsigned)p.kBlocks * (unsigned)(t.split + 1) / (unsigned)p.splits);
  }
  if (p.symmetric) {
    int i = (int)((sqrtf(8.f * t.tile + 1.f) - 1.f) * 0.5f);
    while (i * (i + 1) / 2 > t.tile) --i;
    while ((i + 1) * (i + 2) / 2 <= t.tile) ++i;
    t.tm = i; t.tn = t.tile - i * (i + 1) / 2;
  } else {
    // groups of eight row tiles, column by column: what runs at one time reads few different tiles
    int const per = 8 * p.tilesN, g = t.tile / per, r = t.tile - g * per, rows = min(8, p.tilesM - 8 * g);
    t.tn = r / rows; t.tm = 8 * g + r - t.tn * rows;
  }
  return t;
}

// Whether k-block kb of a side's tile t is read along the columns.
__device__ __forceinline__ bool along_cols(int byCols, int lower, int t, int tile, int kb) { return byCols || (lower && kb * kDepth >= (t + 1) * tile); }

// ------------------------------------------------------------------ PTX
__device__ __forceinline__ uint32_t rank_in_cluster() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync()
{ asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the same shared-memory place in the cluster's first CTA
__device__ __forceinline__ uint32_t in_first(uint32_t addr)
{ uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr)); return r; }
// Relaxed: what it tells of are loads from tensor memory that have been waited for.  (With release semantics in the cluster the arrival waits for the whole
// of the tensor core's work under way: 2200 cycles per k-block of a pair instead of 1800.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar)
{ asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

template <int kCtas>
__device__ __forceinline__ void load_box(uint32_t dst, CUtensorMap const* map, int x, int y, uint32_t bar)
{
  if (kCtas == 2)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar) : "memory");
  else
    tma_load_3d(dst, map, x, y, 0, bar);
}

template <int kCtas>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
  if (kCtas == 2)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// d = a*b + d * 2^-11
template <int kCtas>
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc)
{
  if (kCtas == 2)
    asm volatile("{\n .reg .pred p;\n setp.eq.b32 p, %3, %3;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, 11;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.eq.b32 p, %3, %3;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, 11;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
}
// arrives on the barrier of each CTA of the pair when the MMAs issued so far are through
template <int kCtas>
__device__ __forceinline__ void commit(uint32_t bar)
{
  if (kCtas == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    umma_commit(bar);
}
// the end of all MMAs issued so far; bounded like every wait
template <int kCtas>
__device__ __forceinline__ void finish_mma(uint32_t bar) { commit<kCtas>(bar); mbar_wait(bar, 0u, kWaitCycles); }
template <int kCtas>
__device__ __forceinline__ void alloc_tmem(uint32_t dst)
{
  if (kCtas == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, 512);
  }
}
template <int kCtas>
__device__ __forceinline__ void free_tmem(uint32_t t)
{
  if (kCtas == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(t) : "memory");
  else            tmem_dealloc(t, 512);
}
// ------------------------------------------------------------------ epilogues
// acc: kCols columns from col0 on of row `row` (a lane's); the warp has the same columns of the rows row0 + 0 .. 31.  Global memory is read and written by rows
// of 128 bytes, eight lanes each, and turned into a row per lane in the warp's patch: 32 rows of eight 16-byte places, place c of row r at c ^ (r % 8), so
// that both ways are free of conflicts.
__device__ __forceinline__ uint4& patch_at(float* patch, int row, int place) { return ((uint4*)patch)[row * 8 + (place ^ (row & 7))]; }

// Rows of 64 halves or 32 floats, `pitch` bytes apart, into or out of a lane's eight uint4; rows: those that exist.
__device__ __forceinline__ void fetch_rows(uint4 (&v)[8], char const* from, long long pitch, int rows)
{
  int const lane = threadIdx.x & 31, r0 = lane >> 3, c = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = r0 + 4 * i < rows ? *(uint4 const*)(from + (r0 + 4 * i) * pitch + 16 * c) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void turn_rows(uint4 (&v)[8], float* patch)
{
  int const lane = threadIdx.x & 31, r0 = lane >> 3, c = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) patch_at(patch, r0 + 4 * i, c) = v[i];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = patch_at(patch, lane, i);
  __syncwarp();
}
__device__ __forceinline__ void store_rows(uint4 const (&v)[8], char* to, long long pitch, int rows, float* patch)
{
  int const lane = threadIdx.x & 31, r0 = lane >> 3, c = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) patch_at(patch, lane, i) = v[i];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint4 const q = patch_at(patch, r0 + 4 * i, c);
    if (r0 + 4 * i < rows) *(uint4*)(to + (r0 + 4 * i) * pitch + 16 * c) = q;
  }
  __syncwarp();
}

// Two values, scaled, as hi and lo: four instructions each.  An infinity leaves a not-a-number in lo (pair_of has the test that a matrix of any values needs; what
// products and exponentials give here is finite, or has been spoilt already).
__device__ __forceinline__ void two_pairs(float a, float b, uint32_t& hi, uint32_t& lo)
{
  __half2 const h = __floats2half2_rn(a, b);
  float2 const f = __half22float2(h);
  __half2 const l = __floats2half2_rn((a - f.x) * 2048.f, (b - f.y) * 2048.f);
  hi = *(uint32_t const*)&h; lo = *(uint32_t const*)&l;
}

// 64 neighbouring values of a row per lane, times f, into a pair.
__device__ __forceinline__ void store_pair64(Pair const& to, int row0, int col, int rows, float const* v, float f, float* patch)
{
  uint4 hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    two_pairs(v[8 * i] * f, v[8 * i + 1] * f, hi[i].x, lo[i].x); two_pairs(v[8 * i + 2] * f, v[8 * i + 3] * f, hi[i].y, lo[i].y);
    two_pairs(v[8 * i + 4] * f, v[8 * i + 5] * f, hi[i].z, lo[i].z); two_pairs(v[8 * i + 6] * f, v[8 * i + 7] * f, hi[i].w, lo[i].w);
  }
  store_rows(hi, (char*)(to.hi + row0 * to.ld + col), to.ld * 2, rows, patch);
  store_rows(lo, (char*)(to.lo + row0 * to.ld + col), to.ld * 2, rows, patch);
}

// out = combine(out or 0, value) for the columns of a tile, whatever the alignment of out.
template <int kCols, class F>
__device__ __forceinline__ void update_rows(float* out, long long ldc, int M, int N, bool readOld, float const (&acc)[kCols], int row0, int col0, float* patch, F combine)
{
  int const lane = threadIdx.x & 31, rows = min(32, M - row0);
  bool const vec = ((uintptr_t)out & 15) == 0 && (ldc & 3) == 0;
#pragma unroll
  for (int g = 0; g < kCols / 32; ++g) {
    int const c0 = col0 + g * 32;
    float* const o = out + row0 * ldc + c0;
    if (vec && c0 + 32 <= N) {
      uint4 q[8];
      if (readOld) { fetch_rows(q, (char const*)o, ldc * 4, rows); turn_rows(q, patch); }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        auto one = [&](uint32_t old, int k) { return __float_as_uint(combine(readOld ? __uint_as_float(old) : 0.f, acc[g * 32 + 4 * i + k])); };
        q[i] = make_uint4(one(q[i].x, 0), one(q[i].y, 1), one(q[i].z, 2), one(q[i].w, 3));
      }
      store_rows(q, (char*)o, ldc * 4, rows, patch);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) patch[lane * 33 + i] = acc[g * 32 + i];
      __syncwarp();
      if (c0 + lane < N)
        for (int r = 0; r < rows; r += 8) {
          float old[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) old[i] = readOld && r + i < rows ? o[(r + i) * ldc + lane] : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) if (r + i < rows) o[(r + i) * ldc + lane] = combine(old[i], patch[(r + i) * 33 + lane]);
        }
      __syncwarp();
    }
  }
}

// What the epilogue of a tile takes from global memory, fetched before its products: the sides' scales, and for predictions the row's label and lse and, in the
// warp's patch, the columns' biases (-inf beyond the last column).  Fetched when they are needed they cost 2 us per tile.
struct Ahead { float fa, fb[2], label, lse; };             // fb: of the thread's first and second 64 columns

// The factor that takes the exponent of row `row` of a side back; a side whose rows are the reduction has its factors in the chains.
__device__ __forceinline__ float unscale(vlb::PairExp const& e, int byCols, int row)
{ return e.blocks ? (byCols ? 1.f : pow2(-__ldg(e.blocks + row / 64))) : pow2(-e.value); }

template <int kKind, int kCols>
__device__ __forceinline__ Ahead fetch_ahead(Product const& p, int row, int col0, float* patch)
{
  PairEpilogue const& e = p.e;
  Ahead a = {unscale(e.ea, p.byColsA, min(row, p.M - 1)), {}, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kCols / 64; ++i) a.fb[i] = unscale(e.eb, p.byColsB, min(col0 + 64 * i, p.N - 1));
  if (kKind == kPairSeen || kKind == kPairGrad) {
    if (row < p.M) {
      a.label = __ldg(e.labels + row);
      if (kKind == kPairGrad) a.lse = __ldg(e.lse + row);
    }
#pragma unroll
    for (int i = 0; i < kCols; i += 32) {
      int const c = col0 + i + (int)(threadIdx.x & 31);
      patch[i + (threadIdx.x & 31)] = c < p.N ? (e.bias ? __ldg(e.bias + c) : 0.f) : -INFINITY;
    }
    __syncwarp();
  }
  return a;
}

template <int kCols>
__device__ __forceinline__ void finish_out(Product const& p, Ahead const& ahead, float (&acc)[kCols], int row0, int col0, float* patch)
{
  PairEpilogue const& e = p.e;
  float const fa = ahead.fa, alpha = e.alpha;
#pragma unroll
  for (int i = 0; i < kCols; ++i) acc[i] *= ahead.fb[i / 64];
  update_rows(e.out, e.ldc, p.M, p.N, e.beta != 0.f, acc, row0, col0, patch, [&](float old, float v) { return v * fa * alpha + old; });
}

// predictions = product + bias in place, -inf beyond the last column
template <int kCols>
__device__ __forceinline__ void predictions(Ahead const& a, float (&acc)[kCols], float* patch)
{
#pragma unroll
  for (int i = 0; i < kCols; i += 4) {
    float4 const b = *(float4 const*)(patch + i);
    float const f = a.fb[i / 64];
    acc[i] = fmaf(acc[i] * a.fa, f, b.x); acc[i + 1] = fmaf(acc[i + 1] * a.fa, f, b.y);
    acc[i + 2] = fmaf(acc[i + 2] * a.fa, f, b.z); acc[i + 3] = fmaf(acc[i + 3] * a.fa, f, b.w);
  }
  __syncwarp();
}

// (Fast exponentials here and in finish_grad, one for every element of a tile: off by at most 2 + 1.2 |z - base| units of the last place, where rounding the difference itself costs
// |z - base| / 2.)
template <int kCols>
__device__ __forceinline__ void finish_seen(Product const& p, Ahead const& ahead, float (&acc)[kCols], int row, int col0, float* patch)
{
  PairEpilogue const& e = p.e;
  predictions(ahead, acc, patch);
  bool const in = row < p.M;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kCols; ++i) top = fmaxf(top, acc[i]);
  // an infinite largest value is none to subtract: the exponentials below it are then 0 or infinite, as the definition has them
  float const base = isinf(top) ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kCols; ++i) sum += __expf(acc[i] - base);
  if (in) e.parts[(long long)(col0 / kCols) * p.M + row] = make_float2(top, sum);
  int const at = in ? min(max((int)ahead.label - 1, 0), e.classes - 1) - e.firstClass - col0 : -1;
  bool const here = at >= 0 && at < kCols && col0 + at < p.N;
  if (__any_sync(0xffffffffu, here)) {
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < kCols; ++i) z = i == at ? acc[i] : z;
    if (here) e.label[row] = z;
  }
}

// Sums over the 32 lanes of 32 values each: afterwards lane l holds the sum of v[l] in v[0].
__device__ __forceinline__ float lane_sums(float (&v)[32])
{
  int const lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    bool const up = lane & s;
#pragma unroll
    for (int i = 0; i < s; ++i) {
      float const send = up ? v[i] : v[i + s], keep = up ? v[i + s] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, s);
    }
  }
  return v[0];
}

template <int kCols>
__device__ __forceinline__ void finish_grad(Product const& p, Ahead const& ahead, float (&acc)[kCols], int row0, int row, int col0, float* patch)
{
  PairEpilogue const& e = p.e;
  predictions(ahead, acc, patch);
  float const l = ahead.label, lse = ahead.lse;               // (rows behind the last: label 0)
  bool const real = l > 0.f && l <= (float)e.classes;
  if (l > (float)e.classes && e.status) atomicExch(e.status, kStatusBadLabel);
  int const at = min(max((int)l - 1, 0), e.classes - 1) - e.firstClass - col0;
  // 64 columns at a time, so that the stores of one group are on their way while the next is computed
#pragma unroll
  for (int c0 = 0; c0 < kCols; c0 += 64) {
    float v[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = real ? __expf(acc[c0 + i] - lse) : 0.f;
    if (__any_sync(0xffffffffu, real && at >= c0 && at < c0 + 64)) {
#pragma unroll
      for (int i = 0; i < 64; ++i) v[i] -= real && c0 + i == at ? 1.f : 0.f;
    }
    if (e.db) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float t[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) t[i] = v[g * 32 + i];
        float const s = lane_sums(t);
        int const c = col0 + c0 + g * 32 + (threadIdx.x & 31);
        if (row0 < p.M && c < p.N) e.db[(long long)(row0 / 32) * e.to.ld + c] = s;
      }
    }
    if (col0 + c0 < e.to.ld) store_pair64(e.to, row0, col0 + c0, min(32, p.M - row0), v, pow2(e.toExp), patch);
  }
}

template <int kCols>
__device__ __forceinline__ void finish_poly(Product const& p, Ahead const& ahead, float (&acc)[kCols], int row0, int col0, float* patch)
{
  PairEpilogue const& e = p.e;
  int const rows = min(32, p.M - row0);
  float const f = e.alpha * ahead.fa * ahead.fb[0];            // (one number on either side)
#pragma unroll
  for (int i = 0; i < kCols; ++i) acc[i] *= f;
  if (e.beta != 0.f) {
    float const fh = e.beta * pow2(-e.addExp), fl = fh * (1.f / 2048.f);
    auto two = [&](uint32_t w, float k, float& a, float& b) {
      float2 const v = __half22float2(*(__half2 const*)&w);
      a = fmaf(v.x, k, a); b = fmaf(v.y, k, b);
    };
#pragma unroll
    for (int i = 0; i < kCols; i += 64) {
      if (col0 + i >= e.add.ld) continue;
      uint4 q[2][8];
      fetch_rows(q[0], (char const*)(e.add.hi + row0 * e.add.ld + col0 + i), e.add.ld * 2, rows);
      fetch_rows(q[1], (char const*)(e.add.lo + row0 * e.add.ld + col0 + i), e.add.ld * 2, rows);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        turn_rows(q[part], patch);
        float const k = part ? fl : fh;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          two(q[part][c].x, k, acc[i + 8 * c], acc[i + 8 * c + 1]); two(q[part][c].y, k, acc[i + 8 * c + 2], acc[i + 8 * c + 3]);
          two(q[part][c].z, k, acc[i + 8 * c + 4], acc[i + 8 * c + 5]); two(q[part][c].w, k, acc[i + 8 * c + 6], acc[i + 8 * c + 7]);
        }
      }
    }
  }
  if (e.out) {
    update_rows(e.out, e.ldc, p.M, p.N, true, acc, row0, col0, patch, [&](float old, float v) { return old - e.rate * v; });
    return;
  }
#pragma unroll
  for (int i = 0; i < kCols; i += 64)
    if (col0 + i < e.to.ld) store_pair64(e.to, row0, col0 + i, rows, &acc[i], pow2(e.toExp), patch);
}

// ------------------------------------------------------------------ the kernel
template <int kKind, int kMax, int kCtas>
__global__ void __launch_bounds__(kThreads, 1)
pairs_kernel(const __grid_constant__ Batch<kMax> batch)
{
  constexpr int kTileRows = 128 * kCtas, kTileCols = 128 * kCtas, kCols = kTileCols / 2, kAcc = 512 / kTileCols;
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t full[kStages], done[kRing], empty[kAcc], last;
  __shared__ uint32_t tmemAt;
  __shared__ int ticket;
  uint32_t const base = (smem_u32(raw) + 1023u) & ~1023u;
  int const warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t const rank = kCtas == 2 ? rank_in_cluster() : 0u;
  int const place = (int)blockIdx.x / kCtas, places = (int)gridDim.x / kCtas;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(&full[i]), 2);
    for (int i = 0; i < kRing; ++i) mbar_init(smem_u32(&done[i]), 1);
    for (int i = 0; i < kAcc; ++i) mbar_init(smem_u32(&empty[i]), kDrainWarps * kCtas);
    mbar_init(smem_u32(&last), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) alloc_tmem<kCtas>(smem_u32(&tmemAt));
  tc_fence_before();
  __syncthreads();
  if (kCtas == 2) cluster_sync();
  tc_fence_after();
  uint32_t const tmem = tmemAt;
  if (threadIdx.x == 8 * 32 && place < batch.work) {       // the maps of the first item, on their way before there is anything to load
    CUtensorMap const* const map = batch.map + 4 * item_of(batch, place).prod;
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("prefetch.tensormap [%0];" ::"l"(map + i) : "memory");
  }
  vlb::pdl_wait();

  bool dead = false;                 // a wait ran out: nothing is waited for any more, the work is walked through to the end
  if (warp < kDrainWarps) {
    // (a single CTA's drain threads hold 64 sums and do with what they have)
    if (kCtas == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
    int const quarter = warp & 3, half = warp >> 2;
    float* const patch = (float*)(raw + (base - smem_u32(raw)) + kStages * kStageBytes) + warp * kPatch;
    uint32_t const lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * kCols);
    int j = 0;
    for (int i = 0, w; (w = item_at(batch, place, places, i)) >= 0; ++i) {
      Item const t = item_of(batch, w);
      Product const& p = batch.p[t.prod];
      int const row0 = t.tm * kTileRows + (int)rank * 128 + quarter * 32, col0 = t.tn * kTileCols + half * kCols;
      bool const any = row0 < p.M && col0 < p.N;            // rows and columns behind the matrix need no sums
      Ahead const ahead = fetch_ahead<kKind, kCols>(p, row0 + lane, col0, patch);
      float acc[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
      // exponents that change with the k-block: of a side whose rows are the reduction
      int const* const chainExp = kKind != kPairOut ? nullptr : p.byColsA && p.e.ea.blocks ? p.e.ea.blocks : p.byColsB ? p.e.eb.blocks : nullptr;
      int nextExp = kKind == kPairOut && chainExp ? __ldg(chainExp + t.kb0) : 0;
      for (int kb = t.kb0; kb < t.kb1; ++kb, ++j) {
        float const f = pow2(-nextExp);
        if (kKind == kPairOut && chainExp && kb + 1 < t.kb1) nextExp = __ldg(chainExp + kb + 1);
        if (!dead && !mbar_wait(smem_u32(&done[j % kRing]), (uint32_t)(j / kRing) & 1u)) dead = true;
        if (dead) continue;
        tc_fence_after();
        int const buf = j % kAcc;
        uint32_t const at = lanes + (uint32_t)(buf * kTileCols);
        if (any) {
          uint32_t r[2][16];
          tmem_ld16_issue(at, r[0]);
#pragma unroll
          for (int g = 0; g < kCols / 16; ++g) {
            tmem_ld_wait();
            if (g + 1 < kCols / 16) tmem_ld16_issue(at + 16u * (g + 1), r[(g + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float const v = __uint_as_float(r[g & 1][i]);
              acc[g * 16 + i] = kKind == kPairOut ? fmaf(v, f, acc[g * 16 + i]) : acc[g * 16 + i] + v;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (kCtas == 2) mbar_arrive_cluster(in_first(smem_u32(&empty[buf])));
          else            mbar_arrive(smem_u32(&empty[buf]));
        }
      }
      if (p.splits > 1) {
        // a tile's partial sums: [tile and CTA][range][column / 4][drain thread]
        int const slot = (p.slot0 + t.tile) * kCtas + (int)rank;
        float4* const all = (float4*)batch.split + (p.part0 * kCtas + (long long)(t.tile * kCtas + (int)rank) * p.splits) * (kCols / 4) * 256 + threadIdx.x;
        float4* const mine = all + (long long)t.split * (kCols / 4) * 256;
        if (any) {
#pragma unroll
          for (int i = 0; i < kCols / 4; ++i) mine[i * 256] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        }
        __threadfence();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (threadIdx.x == 0) ticket = atomicAdd(batch.tickets + slot, 1);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ticket != p.splits - 1) continue;
        __threadfence();
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
        for (int s = 0; any && s < p.splits; ++s) {
#pragma unroll
          for (int i = 0; i < kCols / 4; ++i) {
            float4 const v = __ldcg(all + (long long)(s * (kCols / 4) + i) * 256);
            acc[4 * i] += v.x; acc[4 * i + 1] += v.y; acc[4 * i + 2] += v.z; acc[4 * i + 3] += v.w;
          }
        }
        if (threadIdx.x == 0) batch.tickets[slot] = 0;
      }
      if (row0 >= p.M || (!any && kKind != kPairSeen)) continue;       // (half a tile's columns have a part, if an empty one)
      if (kKind == kPairOut)  finish_out(p, ahead, acc, row0, col0, patch);
      if (kKind == kPairSeen) finish_seen(p, ahead, acc, row0 + lane, col0, patch);
      if (kKind == kPairGrad) finish_grad(p, ahead, acc, row0, row0 + lane, col0, patch);
      if (kKind == kPairPoly) finish_poly(p, ahead, acc, row0, col0, patch);
    }
    if (dead && lane == 0) atomicCAS(batch.status, 0, 42);
  } else {
    if (kCtas == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8 || warp == 10) {
      if (lane == 0) {
        bool const isA = warp == 8;
        int it = 0;
        uint32_t const bytes = (batch.three ? 2u : 1u) * kHalfTile;
        for (int i = 0, w; !dead && !batch.idle && (w = item_at(batch, place, places, i)) >= 0; ++i) {
          Item const t = item_of(batch, w);
          Product const& p = batch.p[t.prod];
          int const tile = isA ? t.tm : t.tn, byCols = isA ? p.byColsA : p.byColsB, lower = isA ? p.lowerA : p.lowerB, r0 = tile * kTileRows + (int)rank * 128;
          CUtensorMap const* const map = batch.map + 4 * t.prod + (isA ? 0 : 2);
          for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
            int const s = it % kStages, before = it - kStages;
            if (before >= 0 && !mbar_wait(smem_u32(&done[before % kRing]), (uint32_t)(before / kRing) & 1u)) { dead = true; break; }
            uint32_t const mine = smem_u32(&full[s]), bar = kCtas == 2 ? in_first(mine) : mine;
            if (!isA && p.same && t.tm == t.tn) {
              if (rank == 0) mbar_arrive(mine);
              continue;
            }
            if (rank == 0) mbar_arrive_expect_tx(mine, bytes * kCtas);
            uint32_t const to = base + (uint32_t)s * kStageBytes + (isA ? 0u : 2u * kHalfTile);
            if (along_cols(byCols, lower, tile, kTileRows, kb)) {
              load_box<kCtas>(to, map + 1, r0, kb * kDepth, bar);
              load_box<kCtas>(to + kHalfTile, map + 1, r0 + 64, kb * kDepth, bar);
            } else {
              load_box<kCtas>(to, map, kb * kDepth, r0, bar);
            }
          }
        }
        if (dead) atomicCAS(batch.status, 0, 40);
        // copies still on their way when a wait ran out -- this warp's, or that of the warp which issues the products and had these copies left to wait for -- land
        // before the block ends
        if (rank == 0)
          for (int j = max(0, it - kStages); j < it; ++j) mbar_wait(smem_u32(&full[j % kStages]), (uint32_t)(j / kStages) & 1u, kWaitCycles);
      }
    } else if (warp == 9) {
      if (lane == 0 && rank == 0) {
        // k-block j has its operands and an accumulator
        auto ready = [&](int j) {
          return mbar_wait(smem_u32(&full[j % kStages]), (uint32_t)(j / kStages) & 1u) &&
                 (j < kAcc || mbar_wait(smem_u32(&empty[j % kAcc]), (uint32_t)(j / kAcc - 1) & 1u));
        };
        int j = 0, w = item_at(batch, place, places, 0);
        if (w >= 0) dead = !ready(0);                       // (where both products have few items there are places without any)
        for (int i = 0, after; !dead && w >= 0; ++i, w = after) {
          after = item_at(batch, place, places, i + 1);
          Item const t = item_of(batch, w);
          Product const& p = batch.p[t.prod];
          for (int kb = t.kb0; kb < t.kb1 && !dead; ++kb, ++j) {
            int const s = j % kStages, acc = j % kAcc;
            // the next k-block is waited for when the tensor core still has the end of this one to work on: 250 cycles per k-block
            bool const more = kb + 1 < t.kb1 || after >= 0;
            tc_fence_after();
            uint32_t const st = base + (uint32_t)s * kStageBytes, d = tmem + (uint32_t)(acc * kTileCols);
            bool const ca = along_cols(p.byColsA, p.lowerA, t.tm, kTileRows, kb), cb = along_cols(p.byColsB, p.lowerB, t.tn, kTileCols, kb);
            uint32_t const idesc = (1u << 4) | (ca ? 1u << 15 : 0u) | (cb ? 1u << 16 : 0u) | ((uint32_t)(kTileCols >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
            uint64_t const stepA = (ca ? 2048u : 32u) >> 4, stepB = (cb ? 2048u : 32u) >> 4;
            uint64_t const aH = make_desc(st, kHalfTile, 1024), aL = aH + ((ca ? kHalfTile / 2 : kHalfTile) >> 4);
            uint64_t const bH = p.same && t.tm == t.tn ? aH : make_desc(st + 2 * kHalfTile, kHalfTile, 1024), bL = bH + ((cb ? kHalfTile / 2 : kHalfTile) >> 4);
            if (batch.three) {
#pragma unroll
              for (int k = 0; k < kDepth / 16; ++k) {
                mma<kCtas>(d, aL + stepA * k, bH + stepB * k, idesc, k > 0 ? 1u : 0u);
                mma<kCtas>(d, aH + stepA * k, bL + stepB * k, idesc, 1u);
              }
              mma_scaled<kCtas>(d, aH, bH, idesc);
              if (more) dead = !ready(j + 1);
#pragma unroll
              for (int k = 1; k < kDepth / 16; ++k) mma<kCtas>(d, aH + stepA * k, bH + stepB * k, idesc, 1u);
            } else {
#pragma unroll
              for (int k = 0; k < kDepth / 16; ++k) {
                mma<kCtas>(d, aH + stepA * k, bH + stepB * k, idesc, k > 0 ? 1u : 0u);
                if (k == 0 && more) dead = !ready(j + 1);
              }
            }
            commit<kCtas>(smem_u32(&done[j % kRing]));
          }
        }
        if (dead) atomicCAS(batch.status, 0, 41);
        // tensor memory is given back only when nothing writes to it any more
        finish_mma<kCtas>(smem_u32(&last));
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (kCtas == 2) cluster_sync();
  tc_fence_after();
  if (warp == 9) free_tmem<kCtas>(tmem);
}

// ------------------------------------------------------------------ pairs of single-precision matrices
__device__ __forceinline__ bool is_real(float const* labels, long long row, int classes)
{
  if (!labels) return true;
  float const l = __ldg(labels + row);
  return l > 0.f && l <= (float)classes;
}
__device__ __forceinline__ unsigned finite_bits(float v)
{
  unsigned const b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// 64 rows, which share an exponent, are cut into segments of columns where there are few of them: a block takes one.  First the blocks' largest magnitudes, in a launch
// of their own, then the pairs.  (Both in one launch by blocks that have all of their 64 rows, the second reading from L2: 124 us instead of 44 + 65 for 50001 x 1000,
// 472 instead of 130 + 268 for 100000 x 2048: what L2 holds of them is too few blocks to keep the memory busy.)
constexpr int kSplitThreads = 512;

struct SplitJob {
  vlb::PairSource s;
  unsigned* partial;                          // largest magnitude of each block
  int block0, segments, groups, vec;          // first block; segments of 64 rows; columns / 16 of a segment
  vlb::FastDiv31 perRow;                      // by groups
};
struct SplitJobs { SplitJob j[2]; int count; };

// Sixteen neighbouring floats from p on, by 16-byte loads whatever the alignment of p; those in front of `begin` and from `end` on are not touched.
__device__ __forceinline__ void load16(float (&v)[16], float const* p, float const* begin, float const* end)
{
  int const s = (int)((uintptr_t)p >> 2) & 3;
  float const* const q = p - s;
  float t[20];
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    float const* const a = q + 4 * i;
    if (a >= begin && a + 4 <= end) {
      float4 const f = __ldg((float4 const*)a);
      t[4 * i] = f.x; t[4 * i + 1] = f.y; t[4 * i + 2] = f.z; t[4 * i + 3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) t[4 * i + k] = a + k >= begin && a + k < end ? __ldg(a + k) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 19; ++i) t[i] = s & 1 ? t[i + 1] : t[i];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = s & 2 ? t[i + 2] : t[i];
}

// f(row, column, sixteen values) for the columns of a block; rows that count as zeros give zeros.
template <class F>
__device__ __forceinline__ void each16(SplitJob const& j, int rb, int seg, F f)
{
  vlb::Pair const& to = j.s.to;
  int const first = seg * j.groups, most = min(j.groups, (int)(to.ld / 16) - first);
  float const* const end = j.s.x + (long long)to.rows * to.cols;
#pragma unroll 2
  for (int t = threadIdx.x; t < 64 * j.groups; t += kSplitThreads) {
    int const r = j.perRow(t), g = t - r * j.groups, c = (first + g) * 16;
    long long const row = rb * 64ll + r;
    if (row >= to.rows || g >= most) continue;
    float v[16];
    float const* const p = j.s.x + row * to.cols + c;
    if (j.vec && c + 16 <= to.cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float4 const q = __ldg((float4 const*)p + i);
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
      }
    } else {
      load16(v, p, j.s.x, end);
    }
    bool const real = is_real(j.s.labels, row, j.s.classes);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = real && c + i < to.cols ? v[i] : 0.f;
    f(row, c, v);
  }
}

__device__ __forceinline__ unsigned block_max(unsigned m)
{
  __shared__ unsigned all[kSplitThreads / 32];
  m = __reduce_max_sync(0xffffffffu, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = m;
  __syncthreads();
  m = all[0];
#pragma unroll
  for (int i = 1; i < kSplitThreads / 32; ++i) m = max(m, all[i]);
  return m;
}

__global__ void __launch_bounds__(kSplitThreads)
largest_kernel(const __grid_constant__ SplitJobs jobs)
{
  vlb::pdl_wait();
  SplitJob const& j = jobs.j[jobs.count > 1 && (int)blockIdx.x >= jobs.j[1].block0];
  int const block = (int)blockIdx.x - j.block0, rb = block / j.segments;
  unsigned m = 0;
  each16(j, rb, block - rb * j.segments, [&](long long, int, float const (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, finite_bits(v[i]));
  });
  m = block_max(m);
  if (threadIdx.x == 0) j.partial[block] = m;
}

__global__ void __launch_bounds__(kSplitThreads)
make_pair_kernel(const __grid_constant__ SplitJobs jobs)
{
  vlb::pdl_wait();
  SplitJob const& j = jobs.j[jobs.count > 1 && (int)blockIdx.x >= jobs.j[1].block0];
  int const block = (int)blockIdx.x - j.block0, rb = block / j.segments, seg = block - rb * j.segments;
  unsigned m = 0;
  for (int i = threadIdx.x; i < j.segments; i += kSplitThreads) m = max(m, __ldg(j.partial + rb * j.segments + i));
  m = block_max(m);
  int const e = vlb::pair_exp(__uint_as_float(m));
  if (seg == 0 && threadIdx.x == 0) j.s.exps[rb] = e;
  float const f = pow2(e);
  each16(j, rb, seg, [&](long long row, int c, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= f;
    store_pair16(j.s.to, row, c, v);
  });
}

// ------------------------------------------------------------------ host
// The maps of a side, along its rows and along its columns: hi and lo (or hi alone) in one copy.  A way that no tile is read in has the other one's map: the kernel
// asks for both ahead of time.
bool encode_side(CUtensorMap* map, vlb::PairSide const& s, bool three)
{
  EncodeTiledFn const encode = encode_tiled();
  if (!encode) return false;
  cuuint64_t const dims[3] = {(cuuint64_t)s.m.cols, (cuuint64_t)s.m.rows, 2};
  cuuint64_t const strides[2] = {(cuuint64_t)s.m.ld * 2, (cuuint64_t)((char*)s.m.lo - (char*)s.m.hi)};
  cuuint32_t const one[3] = {1, 1, 1};
  bool const read[2] = {!s.byCols, s.byCols || s.lower};
  for (int along = 0; along < 2; ++along) {
    if (!read[along]) continue;
    cuuint32_t const box[3] = {64, along ? 64u : 128u, three ? 2u : 1u};
    if (encode(map + along, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, s.m.hi, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  for (int along = 0; along < 2; ++along)
    if (!read[along]) map[along] = map[1 - along];
  return true;
}

int tiles_of(PairProduct const& p, int tile)
{
  int const m = vlb::ceil_div(p.M, tile), n = vlb::ceil_div(p.N, tile);
  return p.symmetric ? m * (m + 1) / 2 : m * n;
}

// Microseconds that a tile takes, measured: per k-block; for the hand-over of partial sums and for each of them; for its beginning and end.  A launch with a tile for every SM, or
// for every two (kPairSeen, 128 and 256 images, 18944 classes): 6.9 and 9.9 us with one k-block, 13.7 and 18.3 with 8, 23.3 and 29.5 with 16, 43.0 and 51.2 with 32, 74.9 and
// 88.4 with 64.  Eight tiles of 64 and 128 k-blocks, cut: 21.4 and 28.1.
struct TileCost { double block, cut, part, ends; };
constexpr TileCost kCost[2] = {{1., 3., 0.55, 5.}, {1., 3., 1.1, 7.}};           // 128 x 128 on one CTA, 256 x 256 on two

// Ranges of a reduction of kBlocks k-blocks where there are fewer tiles than places: the number that takes least time as long as all of them run at once.
int splits_of(int kBlocks, long long tiles, int clusters, int ctas)
{
  TileCost const& c = kCost[ctas - 1];
  int best = 1;
  double least = kBlocks * c.block;
  for (int s = 2; s <= 64 && s * tiles <= clusters && 2 * s <= kBlocks; ++s) {
    double const t = vlb::ceil_div(kBlocks, s) * c.block + c.cut + s * c.part;
    if (t < least) { least = t; best = s; }
  }
  return best;
}

template <int kKind, int kMax, int kCtas>
int run(vlb_ctx* ctx, PairProduct const* given, int count, void* split)
{
  constexpr int kTile = 128 * kCtas;
  TileCost const& cost = kCost[kCtas - 1];
  Batch<kMax> b;
  b.three = ctx->precision != VLB_PRECISION_TF32;
  b.idle = ctx->testSwitch & 1;
  int const clusters = ctx->smCount / kCtas;
  long long tiles = 0;
  double total = 0;
  int order[vlb::kMaxPairProducts], splits[vlb::kMaxPairProducts], blocks[vlb::kMaxPairProducts];
  for (int i = 0; i < count; ++i) {
    order[i] = i;
    blocks[i] = vlb::ceil_div(given[i].K, kDepth);
    tiles += tiles_of(given[i], kTile);
    total += tiles_of(given[i], kTile) * (blocks[i] * cost.block + cost.ends);
  }
  double const share = total / clusters;                // what a place has to do
  for (int i = 0; i < count; ++i) {
    splits[i] = splits_of(blocks[i], tiles, clusters, kCtas);
    // a tile that would take more than half of it is cut too, beside others
    if (splits[i] == 1 && count > 1 && blocks[i] >= 64) splits[i] = std::max(1, std::min(16, (int)ceil(2 * blocks[i] * cost.block / share)));
  }
  std::stable_sort(order, order + count, [&](int x, int y) { return vlb::ceil_div(blocks[x], splits[x]) > vlb::ceil_div(blocks[y], splits[y]); });
  size_t const partBytes = sizeof(float) * 128 * kTile;
  int slot = 0;
  long long part = 0, work = 0;
  double rest = 0;                                      // time of all but the first product's items
  for (int i = 0; i < count; ++i) {
    PairProduct const& q = given[order[i]];
    Product& d = b.p[i];
    d.M = q.M; d.N = q.N; d.kBlocks = blocks[order[i]];
    d.tilesM = vlb::ceil_div(q.M, kTile); d.tilesN = vlb::ceil_div(q.N, kTile);
    int const t = tiles_of(q, kTile), s = splits[order[i]];
    bool const fits = (slot + t) * kCtas < 4095 && (size_t)((part + (long long)t * s) * kCtas) * partBytes <= vlb::kPairSplitBytes;
    d.splits = fits ? s : 1;
    d.slot0 = slot; d.part0 = part;
    if (d.splits > 1) { slot += t; part += (long long)t * d.splits; }
    work += (long long)t * d.splits;
    if (work > INT32_MAX / 4) return vlb::set_error(ctx, VLB_IllegalArgument, "the matrices are too large");
    d.work = (int)work;
    if (i) rest += (double)t * d.splits * (vlb::ceil_div(d.kBlocks, d.splits) * cost.block + cost.ends);
    d.byColsA = q.a.byCols; d.byColsB = q.b.byCols; d.lowerA = q.a.lower; d.lowerB = q.b.lower; d.symmetric = q.symmetric;
    d.same = q.symmetric && q.a.m.hi == q.b.m.hi && q.a.byCols == q.b.byCols && q.a.lower == q.b.lower;
    d.e = q.e;
    if (!encode_side(&b.map[4 * i], q.a, b.three) || !encode_side(&b.map[4 * i + 2], q.b, b.three))
      return vlb::set_error(ctx, VLB_Cuda, "a tensor map could not be made");
  }
  int const places = (int)std::min<long long>(clusters, work);
  b.lead = count > 1 ? b.p[0].work : (int)work;
  b.behind = b.lead % places;
  b.even = (int)work;
  if (count > 1 && work > b.lead && b.behind) {
    double const one = vlb::ceil_div(b.p[0].kBlocks, b.p[0].splits) * cost.block + cost.ends, each = rest / (double)(work - b.lead);
    long long const others = work - b.lead;
    int const near = (int)std::max(0., ((b.lead * one + rest) / places - (b.lead / places + 1) * one) / each);
    double least = 1e30;
    for (int e : {near, near + 1, vlb::ceil_div(others, places)}) {
      double const behind = (b.lead / places + 1) * one + std::min<long long>(e, vlb::ceil_div(others, places)) * each;
      double const ahead = (b.lead / places) * one + (e + vlb::ceil_div(std::max(0ll, others - (long long)e * places), places - b.behind)) * each;
      if (std::max(behind, ahead) < least) { least = std::max(behind, ahead); b.even = e; }
    }
  }
  b.count = count; b.work = (int)work;
  b.split = (float*)split;
  b.tickets = ctx->deviceStatus + 64;
  b.status = ctx->deviceStatus;
  auto const kernel = pairs_kernel<kKind, kMax, kCtas>;
  static bool ready[64];
  if (!ready[ctx->device & 63]) {
    cudaError_t const e = vlb::allow_max_dynamic_smem(kernel);
    if (e != cudaSuccess) return vlb::set_error(ctx, VLB_Cuda, cudaGetErrorString(e));
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess || (kCtas == 2 && a.numRegs != kLaunchRegs))        // the drain warps would wait for registers for ever
      return vlb::set_error(ctx, VLB_Cuda, "products_of_pairs: the kernel was built with another number of registers");
    ready[ctx->device & 63] = true;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCtas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(places * kCtas)); cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem; cfg.stream = ctx->stream; cfg.attrs = attr; cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, b);
  VLB_LAUNCHED(ctx, 1);
  return vlb::check_launch(ctx, "products_of_pairs");
}

template <int kKind, int kMax>
int run_kind(vlb_ctx* ctx, PairProduct const* p, int count, void* split, int tile)
{
  return tile == 256 ? run<kKind, kMax, 2>(ctx, p, count, split) : run<kKind, kMax, 1>(ctx, p, count, split);
}

}  // namespace

namespace vlb {

void make_pairs(vlb_ctx* ctx, PairSource const* s, int count, unsigned* partial)
{
  SplitJobs jobs;
  jobs.count = count;
  int blocks = 0;
  for (int i = 0; i < count; ++i) {
    SplitJob& j = jobs.j[i];
    j.s = s[i];
    j.partial = partial;
    partial += pair_partials(s[i].to.rows);
    j.vec = ((uintptr_t)s[i].x & 15) == 0 && s[i].to.cols % 4 == 0;
    int const rowBlocks = ceil_div(s[i].to.rows, 64), all = (int)(s[i].to.ld / 16);
    // two blocks per SM where 64 rows at a time do not give as many; sixteen columns of all 64 rows, two per thread, at least
    int const want = std::min(ceil_div(all, 16), std::max(1, 2 * ctx->smCount / rowBlocks));
    j.groups = ceil_div(all, want);
    j.segments = ceil_div(all, j.groups);
    j.perRow = FastDiv31(j.groups);
    j.block0 = blocks;
    blocks += rowBlocks * j.segments;
  }
  launch(ctx->stream, largest_kernel, (unsigned)blocks, kSplitThreads, 0, jobs);
  launch(ctx->stream, make_pair_kernel, (unsigned)blocks, kSplitThreads, 0, jobs);
  VLB_LAUNCHED(ctx, 2);
}

int pair_tile(vlb_ctx* ctx, PairProduct const* p, int count)
{
  double time[2];
  for (int ctas = 1; ctas <= 2; ++ctas) {
    int const clusters = ctx->smCount / ctas;
    TileCost const& c = kCost[ctas - 1];
    long long tiles = 0;
    for (int i = 0; i < count; ++i) tiles += tiles_of(p[i], 128 * ctas);
    double sum = 0, longest = 0;
    for (int i = 0; i < count; ++i) {
      int const kb = ceil_div(p[i].K, kDepth), s = splits_of(kb, tiles, clusters, ctas);
      double const t = ceil_div(kb, s) * c.block + c.ends + (s > 1 ? c.cut + s * c.part : 0);
      sum += tiles_of(p[i], 128 * ctas) * (kb * c.block + c.ends);
      longest = std::max(longest, t);
    }
    time[ctas - 1] = std::max(sum / clusters, longest);
  }
  return time[1] < time[0] ? 256 : 128;
}

int products_of_pairs(vlb_ctx* ctx, PairKind kind, PairProduct const* p, int count, void* split, int tile)
{
  switch (kind) {
    case kPairOut:  return run_kind<kPairOut, 2>(ctx, p, count, split, tile);
    case kPairSeen: return run_kind<kPairSeen, 1>(ctx, p, count, split, tile);
    case kPairGrad: return run_kind<kPairGrad, 1>(ctx, p, count, split, tile);
    default:        return count > 1 ? run_kind<kPairPoly, kMaxPairProducts>(ctx, p, count, split, tile) : run_kind<kPairPoly, 1>(ctx, p, count, split, tile);
  }
}

cudaError_t pairs_set_wait_limit(long long cycles, cudaStream_t stream)
{
  long long const v = cycles == 0 ? kWaitCycles : cycles;
  return cudaMemcpyToSymbolAsync(gWaitCycles, &v, sizeof(v), 0, cudaMemcpyHostToDevice, stream);
}

}  // namespace vlb
