// The Newton-Schulz steps of matrices of at most 128 rows or columns, all steps in one launch: a matrix belongs to a cluster of CTAs and stays in their shared memory
// from the first step to the last.  As launches of products (pairs.cu) a step takes three, of 8 us each whatever the size: the way from one launch's stores to the
// next one's loads is most of them.
//
// X, the matrix or its transpose, has m <= 128 rows; CTA r of the cluster has up to 256 of its columns, as pairs of halves (pairs.cuh) in the layout that the tensor
// core reads both along the rows (A = X X': the columns are the reduction) and along the columns (Q X: the rows are).  A step:
//   A = X X'        every CTA for its columns, in chains of 64; each CTA then adds up a share of the elements over the cluster's shared memories and leaves the
//                   totals in the same places of all of them
//   Q = b A + c A A every CTA for itself
//   X = a X + Q X   every CTA its columns, in place
// The arithmetic is that of pairs.cu: three products of halves each, chains of 64 products, sums in single precision.
// Sixteen warps move data between registers, tensor memory and shared memory: warp w has TMEM lanes (rows) 32 (w % 4) ... and quarter w / 4 of the columns.  One of
// their threads issues the MMAs: nothing else could be done meanwhile, and without a warp for it a thread has 128 registers.
#include "muon_small.cuh"
#include "pairs.cuh"
#include "tc_common.cuh"

namespace {

using vlb::SmallMatrix; using vlb::SmallSteps; using vlb::pow2;
using vlb::kSmallMost; using vlb::kSmallSide; using vlb::kSmallLong;

constexpr int kThreads = 512;
constexpr int kPart = 128 * 128, kBlock = 2 * kPart;          // bytes of 128 rows x 64 halves, and of hi and lo of them
constexpr int kMostBlocks = 4;                                // 64-column blocks of X in a CTA
constexpr size_t kSmem = (size_t)(kMostBlocks + 2) * kBlock + 1024;

struct Matrices { SmallMatrix m[kSmallMost]; SmallSteps steps; int* status; int cluster, idle; };      // idle: test switch, no wait is answered

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// d = a*b + d * 2^-11
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc)
{
  asm volatile("{\n .reg .pred p;\n setp.eq.b32 p, %3, %3;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, 11;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
}
// A chain of 64 products per element: small terms first.  step: what 16 of the reduction are in a descriptor.
__device__ __forceinline__ void chain(uint32_t d, uint64_t aH, uint64_t aL, uint64_t stepA, uint64_t bH, uint64_t bL, uint64_t stepB, uint32_t idesc, bool three)
{
  if (three) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mma(d, aL + stepA * k, bH + stepB * k, idesc, k > 0 ? 1u : 0u);
      mma(d, aH + stepA * k, bL + stepB * k, idesc, 1u);
    }
    mma_scaled(d, aH, bH, idesc);
#pragma unroll
    for (int k = 1; k < 4; ++k) mma(d, aH + stepA * k, bH + stepB * k, idesc, 1u);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) mma(d, aH + stepA * k, bH + stepB * k, idesc, k > 0 ? 1u : 0u);
  }
}

__device__ __forceinline__ void cluster_sync()
{ asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// the same shared-memory place in the cluster's CTA `rank`
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank)
{ uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank)); return r; }
__device__ __forceinline__ float4 load_cluster(uint32_t addr)
{
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_cluster(uint32_t addr, float4 v)
{ asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory"); }

// Eight neighbouring halves of a row of a block: place c of row r lies at c ^ (r % 8), the 128-byte swizzle.
__device__ __forceinline__ uint4& place(char* block, int row, int c) { return *(uint4*)(block + row * 128 + ((c ^ (row & 7)) << 4)); }

// Eight values of a row, scaled, into hi (block) and lo (block + kPart).
__device__ __forceinline__ void put8(char* block, int row, int c, float const* v)
{
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 const p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    float2 const f = __half22float2(p);
    __half2 const q = __floats2half2_rn((v[2 * i] - f.x) * 2048.f, (v[2 * i + 1] - f.y) * 2048.f);
    h[i] = *(uint32_t const*)&p; l[i] = *(uint32_t const*)&q;
  }
  place(block, row, c) = make_uint4(h[0], h[1], h[2], h[3]);
  place(block + kPart, row, c) = make_uint4(l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void get8(char* block, int row, int c, float (&v)[8])
{
  uint4 const h = place(block, row, c), l = place(block + kPart, row, c);
  uint32_t const hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 const a = __half22float2(*(__half2 const*)&hs[i]), b = __half22float2(*(__half2 const*)&ls[i]);
    v[2 * i] = fmaf(b.x, 1.f / 2048.f, a.x); v[2 * i + 1] = fmaf(b.y, 1.f / 2048.f, a.y);
  }
}

__global__ void __launch_bounds__(kThreads, 1)
small_kernel(const __grid_constant__ Matrices all, bool three)
{
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t through, last;
  __shared__ uint32_t tmemAt;
  __shared__ double sums[kThreads / 32];
  char* const base = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  char* const gramAt = base + kMostBlocks * kBlock;           // A, then Q: two blocks
  int const warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = all.cluster, rank = (int)blockIdx.x % G, which = (int)blockIdx.x / G;
  if (threadIdx.x == 0) { mbar_init(smem_u32(&through), 1); mbar_init(smem_u32(&last), 1); asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
  if (warp == 0) tmem_alloc(smem_u32(&tmemAt), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t const tmem = tmemAt;
  vlb::pdl_wait();

  SmallMatrix const& mat = all.m[which];
  SmallSteps const& st = all.steps;
  bool const tall = mat.rows > mat.cols;
  int const m = tall ? mat.cols : mat.rows, n = tall ? mat.rows : mat.cols;
  int const per = ((n + G - 1) / G + 63) / 64 * 64, j0 = rank * per, mine = max(0, min(per, n - j0)), blocks = per / 64;      // columns j0 ... j0 + mine - 1
  int const rowBlocks = m > 64 ? 2 : 1;
  uint32_t phase = 0;
  bool dead = false;
  int const quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;
  bool const rowsIn = quarter * 32 < m, in = rowsIn && part * 32 < m;            // whether the warp has rows of X, and elements of A
  uint32_t const lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  // the factor that normalises
  double sum = 0;
  for (int i = threadIdx.x; i < mat.partCount; i += kThreads) sum += mat.parts[i];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < kThreads / 32; ++i) sum += sums[i];
  float const norm = (float)(1. / (sqrt(sum) + st.epsilon));
  // X: a thread takes eight neighbouring columns of a row; neighbouring threads what is neighbouring in memory
  float const f0 = pow2(st.x[0]);
#pragma unroll 4
  for (int t = threadIdx.x; t < 128 * per / 8; t += kThreads) {
    int const r = tall ? t % 128 : t / (per / 8), c = tall ? t / 128 : t % (per / 8);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int const j = c * 8 + i;
      bool const in = r < m && j < mine;
      size_t const at = tall ? (size_t)(j0 + j) * mat.cols + r : (size_t)r * mat.cols + j0 + j;
      v[i] = in ? __ldg(mat.u + at) * norm * f0 : 0.f;
    }
    put8(base + c / 8 * kBlock, r, c % 8, v);
  }
  uint32_t const xAt = smem_u32(base), gramAddr = smem_u32(gramAt);
  uint64_t const rowStep = 32 >> 4, colStep = 2048 >> 4;
  uint32_t const square = (1u << 4) | (128u >> 3 << 17) | (128u >> 4 << 24), next = (1u << 4) | (1u << 16) | ((uint32_t)(per >> 3) << 17) | (128u >> 4 << 24);
  // What the threads wrote is handed to the tensor core, `issue` starts its work, and all wait for the end of it.
  auto multiply = [&](auto issue) {
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) {
      tc_fence_after();
      if (!all.idle) issue();
      if (!all.idle) umma_commit(smem_u32(&through));
    }
    __syncwarp();
    if (!dead && !mbar_wait(smem_u32(&through), phase)) dead = true;
    phase ^= 1u;
    __syncwarp();
    tc_fence_after();
  };
  float4* const gramSums = (float4*)gramAt;                 // [column / 4][row]: side by side for a warp
  for (int k = 0; k < st.count; ++k) {
    float const unX = pow2(-st.x[k]), toA = pow2(st.gram[k]), unA = pow2(-st.gram[k]), toQ = pow2(st.poly[k]), unQ = pow2(-st.poly[k]), toX = pow2(st.x[k + 1]);
    multiply([&] {
      for (int b = 0; b < blocks; ++b) {
        uint64_t const h = make_desc(xAt + b * kBlock, 16, 1024), l = make_desc(xAt + b * kBlock + kPart, 16, 1024);
        chain(tmem + 128 * b, h, l, rowStep, h, l, rowStep, square, three);
      }
    });
    // A: 32 columns of a row
    float g[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) g[i] = 0.f;
    if (in)
      for (int b = 0; b < blocks; ++b) {
        uint32_t r[32];
        tmem_ld16_issue(lanes + (uint32_t)(128 * b + 32 * part), r);
        tmem_ld16_issue(lanes + (uint32_t)(128 * b + 32 * part + 16), r + 16);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) g[i] += __uint_as_float(r[i]);
      }
    if (G > 1 && in) {
      // (nothing reads Q any more)
#pragma unroll
      for (int i = 0; i < 8; ++i) gramSums[(8 * part + i) * 128 + row] = make_float4(g[4 * i], g[4 * i + 1], g[4 * i + 2], g[4 * i + 3]);
    }
    __syncwarp();
    cluster_sync();
    if (G > 1) {
      // a place is read and written by one thread of the cluster alone
      int const rows = (m + 31) / 32 * 32, places = (m + 3) / 4 * rows, share = (places + G - 1) / G, end = min((rank + 1) * share, places);
      for (int i = rank * share + (int)threadIdx.x; i < end; i += kThreads) {
        uint32_t const at = gramAddr + 16u * (uint32_t)(i / rows * 128 + i % rows);
        float4 v[8], t = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 8; ++c) if (c < G) v[c] = load_cluster(in_cta(at, c));
#pragma unroll
        for (int c = 0; c < 8; ++c) if (c < G) { t.x += v[c].x; t.y += v[c].y; t.z += v[c].z; t.w += v[c].w; }
#pragma unroll
        for (int c = 0; c < 8; ++c) if (c < G) store_cluster(in_cta(at, c), t);
      }
    }
    __syncwarp();
    cluster_sync();
    if (G > 1) {
      if (in) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float4 const v = 8 * part + i < (m + 3) / 4 ? gramSums[(8 * part + i) * 128 + row] : make_float4(0, 0, 0, 0);
          g[4 * i] = v.x; g[4 * i + 1] = v.y; g[4 * i + 2] = v.z; g[4 * i + 3] = v.w;
        }
      }
      __syncthreads();                                             // before A takes the places of the totals
    }
    char* const gramBlock = gramAt + part / 2 * kBlock;
    int const gramPlace = part % 2 * 4;
#pragma unroll
    for (int i = 0; i < 32; ++i) g[i] = g[i] * unX * unX;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = g[8 * c + i] * toA;
      put8(gramBlock, row, gramPlace + c, v);               // (zeros behind the last row and column)
    }
    multiply([&] {
      for (int b = 0; b < rowBlocks; ++b) {
        uint64_t const h = make_desc(gramAddr + b * kBlock, 16, 1024), l = make_desc(gramAddr + b * kBlock + kPart, 16, 1024);
        chain(tmem + 128 * b, h, l, rowStep, h, l, rowStep, square, three);
      }
    });
    // Q = b A + c A A
    if (in) {
      float const fa = st.c * unA * unA;
#pragma unroll
      for (int i = 0; i < 32; ++i) g[i] *= st.b;
      for (int b = 0; b < rowBlocks; ++b) {
        uint32_t r[32];
        tmem_ld16_issue(lanes + (uint32_t)(128 * b + 32 * part), r);
        tmem_ld16_issue(lanes + (uint32_t)(128 * b + 32 * part + 16), r + 16);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) g[i] = fmaf(fa, __uint_as_float(r[i]), g[i]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = g[8 * c + i] * toQ;
        put8(gramBlock, row, gramPlace + c, v);
      }
    }
    multiply([&] {
      for (int b = 0; b < rowBlocks; ++b) {                     // rows 64 b ... of X are the reduction
        uint64_t const h = make_desc(gramAddr + b * kBlock, 16, 1024), l = make_desc(gramAddr + b * kBlock + kPart, 16, 1024);
        uint64_t const xh = make_desc(xAt + b * 64 * 128, kBlock, 1024), xl = make_desc(xAt + kPart + b * 64 * 128, kBlock, 1024);
        chain(tmem + 256 * b, h, l, rowStep, xh, xl, colStep, next, three);
      }
    });
    // X = a X + Q X, the warp's quarter of the columns, sixteen at a time
    bool const last = k + 1 == st.count;
    if (rowsIn)
      for (int c16 = part * (per / 64); c16 < (part + 1) * (per / 64); ++c16) {
        uint32_t r[2][16];
        tmem_ld16_issue(lanes + (uint32_t)(16 * c16), r[0]);
        if (rowBlocks > 1) tmem_ld16_issue(lanes + (uint32_t)(256 + 16 * c16), r[1]);
        char* const block = base + c16 / 4 * kBlock;
        float v[2][8];
#pragma unroll
        for (int q = 0; q < 2; ++q) get8(block, row, c16 % 4 * 2 + q, v[q]);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float const t = __uint_as_float(r[0][8 * q + i]) + (rowBlocks > 1 ? __uint_as_float(r[1][8 * q + i]) : 0.f);
            v[q][i] = st.a * (v[q][i] * unX) + t * unQ * unX;
          }
          if (!last) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q][i] *= toX;
            put8(block, row, c16 % 4 * 2 + q, v[q]);
          } else {
            int const j = 16 * c16 + 8 * q;
            float* const w = mat.w + (tall ? (size_t)(j0 + j) * mat.cols + row : (size_t)row * mat.cols + j0 + j);
            size_t const step = tall ? mat.cols : 1;
            float old[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) old[i] = row < m && j + i < mine ? w[i * step] : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) if (row < m && j + i < mine) w[i * step] = old[i] - mat.rate * v[q][i];
          }
        }
      }
  }
  if (dead && lane == 0) atomicCAS(all.status, 0, 44);
  // products that still run when the wait of the thread that issued them ran out end before the shared memory and the tensor memory that they use is given back
  if (dead && threadIdx.x == 0) { umma_commit(smem_u32(&last)); mbar_wait(smem_u32(&last), 0u, kWaitCycles); }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

}  // namespace

namespace vlb {

bool small_fits(int rows, int cols, int steps)
{
  return std::min(rows, cols) <= kSmallSide && std::max(rows, cols) <= kSmallLong && steps > 0 && steps <= kSmallSteps;
}

int small_matrices(vlb_ctx* ctx, SmallMatrix const* m, int count, SmallSteps const& steps)
{
  Matrices all;
  int longest = 0;
  for (int i = 0; i < count; ++i) { all.m[i] = m[i]; longest = std::max(longest, std::max(m[i].rows, m[i].cols)); }
  all.steps = steps;
  all.status = ctx->deviceStatus;
  all.idle = ctx->testSwitch & 1;
  // as many CTAs to a matrix as its longer side has 128 columns for, at most eight (64 x 576: 58 us; with 256 each 70)
  all.cluster = 1;
  while (all.cluster < 8 && all.cluster * 128 < longest) all.cluster *= 2;
  static bool ready[64];
  if (!ready[ctx->device & 63]) {
    cudaError_t const e = allow_max_dynamic_smem(small_kernel);
    if (e != cudaSuccess) return set_error(ctx, VLB_Cuda, cudaGetErrorString(e));
    ready[ctx->device & 63] = true;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = all.cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(count * all.cluster)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = kSmem; cfg.stream = ctx->stream;
  cfg.attrs = attr; cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, small_kernel, all, ctx->precision != VLB_PRECISION_TF32);
  VLB_LAUNCHED(ctx, 1);
  return check_launch(ctx, "small_matrices");
}

cudaError_t small_set_wait_limit(long long cycles, cudaStream_t stream)
{
  long long const v = cycles == 0 ? kWaitCycles : cycles;
  return cudaMemcpyToSymbolAsync(gWaitCycles, &v, sizeof(v), 0, cudaMemcpyHostToDevice, stream);
}

}  // namespace vlb
