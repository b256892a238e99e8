// Layer normalisation over the channels of a position (include/vlb.h has the formulas) -- HBM bound: 8 bytes per value forward, 12 backward.
//
// A position's values are read once and held in registers through all passes over them: the mean, then the sum of squared differences from it (backward
// together with the two sums of the derivative), then the result.  One position per image (tokens; P = 1): a position is a run of C floats and belongs to a warp or
// a block.  Maps (P > 1): values of a position lie P floats apart, so that neighbouring positions belong to neighbouring lanes, and a block's warps share the
// channels.  Both count positions through the batch.  What does not fit the registers is read again for each pass, from L2.
//
// The sums over positions (dG, dB) are kept per channel by the threads that see it; each block leaves its part, and a second kernel adds the parts in order.
#include "tc_common.cuh"
#include <algorithm>

namespace {

// Blocks of a backward pass, at most: eight per SM, and parts of 64 MB.
int most_parts(vlb_ctx* ctx, int C) { return (int)std::max<long long>(1, std::min<long long>(8 * ctx->smCount, (64ll << 20) / (8ll * C))); }

__device__ __forceinline__ float warp_sum(float v)
{
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums over the kThreads threads of a row, in each of them; red: [kCount][32] floats, not in use by an earlier call's readers any more.
template <int kThreads, int kCount>
__device__ __forceinline__ void row_sums(float (&v)[kCount], float (*red)[32])
{
#pragma unroll
  for (int k = 0; k < kCount; ++k) v[k] = warp_sum(v[k]);
  if (kThreads == 32) return;
  int const lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < kCount; ++k) red[k][warp] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kCount; ++k) v[k] = warp_sum(lane < kThreads / 32 ? red[k][lane] : 0.f);
}

// ------------------------------------------------------------------ positions that are rows
// A row belongs to kThreads threads, each with kVec times four neighbouring channels (kWide) or 4 kVec channels kThreads apart.
template <int kThreads, int kVec, bool kWide>
struct Row {
  static constexpr int kValues = 4 * kVec;
  static __device__ __forceinline__ int channel(int i)
  {
    int const t = threadIdx.x % kThreads;
    return kWide ? 4 * (t + kThreads * (i / 4)) + i % 4 : t + kThreads * i;
  }
  static __device__ __forceinline__ void load(float (&v)[kValues], float const* __restrict__ p, int C)
  {
    if (kWide) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        float4 const q = channel(4 * i) < C ? __ldg((float4 const*)(p + channel(4 * i))) : make_float4(0, 0, 0, 0);
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kValues; ++i) v[i] = channel(i) < C ? __ldg(p + channel(i)) : 0.f;
    }
  }
  static __device__ __forceinline__ void store(float* __restrict__ p, float const (&v)[kValues], int C)
  {
    if (kWide) {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (channel(4 * i) < C) *(float4*)(p + channel(4 * i)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kValues; ++i) if (channel(i) < C) p[channel(i)] = v[i];
    }
  }
};

constexpr int block_of(int rowThreads) { return rowThreads < 128 ? 128 : rowThreads; }

template <int kThreads, int kVec, bool kWide>
__global__ void __launch_bounds__(block_of(kThreads))
rows_fwd_kernel(float* __restrict__ y, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ b, int rows, int C, float eps)
{
  using R = Row<kThreads, kVec, kWide>;
  vlb::pdl_wait();
  __shared__ float red[2][1][32];
  int const row = (int)blockIdx.x * (block_of(kThreads) / kThreads) + (int)threadIdx.x / kThreads;
  if (kThreads == 32 && row >= rows) return;
  float v[R::kValues];
  R::load(v, x + (size_t)row * C, C);
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < R::kValues; ++i) s[0] += v[i];
  row_sums<kThreads>(s, red[0]);
  float const mean = s[0] / (float)C;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < R::kValues; ++i) { v[i] -= mean; s[0] += R::channel(i) < C ? v[i] * v[i] : 0.f; }
  row_sums<kThreads>(s, red[1]);
  float const r = 1.f / sqrtf(s[0] / (float)C + eps);
  float gv[R::kValues], bv[R::kValues];
  R::load(gv, g, C);
  R::load(bv, b, C);
#pragma unroll
  for (int i = 0; i < R::kValues; ++i) v[i] = fmaf(gv[i], v[i] * r, bv[i]);
  R::store(y + (size_t)row * C, v, C);
}

// Groups of neighbouring rows in turn to the blocks, `per` rows to a row's threads.  kWide: they come by bulk copies, kStages groups on their way or in use, so that
// the reductions of one row (half of the time otherwise) do not keep the memory waiting: 16384 x 4096 175 -> 126 us, the copy rate.  Without 16-byte alignment every thread loads
// its own values.  parts: [block][2][C], dG then dB.
constexpr int kStages = 3;

template <int kThreads, int kVec, bool kWide>
__global__ void __launch_bounds__(block_of(kThreads))
rows_bwd_kernel(float* __restrict__ dx, float* __restrict__ parts, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ dy,
                int rows, int C, int per, float eps, int* status, int idle)
{
  using R = Row<kThreads, kVec, kWide>;
  constexpr int kRows = block_of(kThreads) / kThreads, kWarps = block_of(kThreads) / 32;
  extern __shared__ __align__(128) float staged[];         // [stage][x or dy][per * kRows rows]
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages];
  __shared__ float red[2][4][32];
  __shared__ float other[kRows > 1 ? (kRows - 1) * 2 * 32 * R::kValues : 1];
  int const group = per * kRows, groups = (rows + group - 1) / group, mine = ((int)blockIdx.x < groups) ? (groups - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
  if (kWide) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < kStages; ++i) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), kWarps); }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  vlb::pdl_wait();
  bool dead = false;                                       // a wait ran out: nothing is waited for any more
  int asked = 0;                                           // groups that were asked for
  auto fetch = [&](int it) {                               // by one thread
    if (idle) return;                                      // (test switch: nothing comes, so that every wait runs out)
    int const st = it % kStages, row0 = ((int)blockIdx.x + it * (int)gridDim.x) * group, count = min(group, rows - row0);
    if (it >= kStages && !dead && !mbar_wait(smem_u32(&empty[st]), (uint32_t)(it / kStages - 1) & 1u)) dead = true;
    if (dead) return;
    uint32_t const bytes = (uint32_t)count * C * 4, to = smem_u32(staged + (size_t)st * 2 * group * C);
    mbar_arrive_expect_tx(smem_u32(&full[st]), 2 * bytes);
    bulk_copy_g2s(to, x + (size_t)row0 * C, bytes, smem_u32(&full[st]));
    bulk_copy_g2s(to + (uint32_t)group * C * 4, dy + (size_t)row0 * C, bytes, smem_u32(&full[st]));
    asked = it + 1;
  };
  if (kWide && threadIdx.x == 0)
    for (int it = 0; it < min(mine, kStages - 1); ++it) fetch(it);
  float gv[R::kValues], dg[R::kValues] = {}, db[R::kValues] = {};
  R::load(gv, g, C);
  float const n = (float)C;
  int even = 0;
  for (int it = 0; it < mine; ++it) {
    int const st = it % kStages, row0 = ((int)blockIdx.x + it * (int)gridDim.x) * group;
    if (kWide) {
      if (threadIdx.x == 0 && it + kStages - 1 < mine) fetch(it + kStages - 1);
      if (!dead && !mbar_wait(smem_u32(&full[st]), (uint32_t)(it / kStages) & 1u)) dead = true;
    }
    for (int k = 0; k < per; ++k, even ^= 1) {
      int const local = k * kRows + (int)threadIdx.x / kThreads, row = row0 + local;
      if (row >= rows) break;                              // (a block has one row at a time where its threads meet at barriers)
      float v[R::kValues], d[R::kValues];
      if (kWide) {
        float const* const from = staged + ((size_t)st * 2 * group + local) * C;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          int const c = R::channel(4 * i);
          float4 const p = c < C ? *(float4 const*)(from + c) : make_float4(0, 0, 0, 0), q = c < C ? *(float4 const*)(from + (size_t)group * C + c) : make_float4(0, 0, 0, 0);
          v[4 * i] = p.x; v[4 * i + 1] = p.y; v[4 * i + 2] = p.z; v[4 * i + 3] = p.w;
          d[4 * i] = q.x; d[4 * i + 1] = q.y; d[4 * i + 2] = q.z; d[4 * i + 3] = q.w;
        }
      } else {
        R::load(v, x + (size_t)row * C, C);
        R::load(d, dy + (size_t)row * C, C);
      }
      float m[1] = {0.f};
#pragma unroll
      for (int i = 0; i < R::kValues; ++i) m[0] += v[i];
      row_sums<kThreads>(m, red[even] + 3);
      float const mean = m[0] / n;
      float s[3] = {};
#pragma unroll
      for (int i = 0; i < R::kValues; ++i) {
        v[i] = R::channel(i) < C ? v[i] - mean : 0.f;
        float const gd = gv[i] * d[i];
        s[0] += v[i] * v[i]; s[1] += gd; s[2] += gd * v[i];
      }
      row_sums<kThreads>(s, red[even]);
      float const r = 1.f / sqrtf(s[0] / n + eps), m1 = s[1] / n, m2 = s[2] * r / n;
#pragma unroll
      for (int i = 0; i < R::kValues; ++i) {
        float const xh = v[i] * r;
        dg[i] += d[i] * xh; db[i] += d[i];
        v[i] = r * (gv[i] * d[i] - m1 - xh * m2);
      }
      if (dx) R::store(dx + (size_t)row * C, v, C);
    }
    if (kWide) {
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&empty[st]));
    }
  }
  if (dead) atomicCAS(status, 0, 43);
  // copies still on their way when the wait of the thread that asked for them ran out land before the block ends
  if (kWide && threadIdx.x == 0 && dead)
    for (int it = max(0, asked - kStages); it < asked; ++it) mbar_wait(smem_u32(&full[it % kStages]), (uint32_t)(it / kStages) & 1u, kWaitCycles);
  if (!parts) return;
  if (kRows > 1) {
    // the block's warps, added in order
    int const w = (int)threadIdx.x / 32, lane = threadIdx.x & 31;
    if (w) {
#pragma unroll
      for (int i = 0; i < R::kValues; ++i) {
        other[((w - 1) * 2 * R::kValues + i) * 32 + lane] = dg[i];
        other[((w - 1) * 2 * R::kValues + R::kValues + i) * 32 + lane] = db[i];
      }
    }
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int i = 0; i < R::kValues; ++i)
      for (int k = 0; k < kRows - 1; ++k) {
        dg[i] += other[(k * 2 * R::kValues + i) * 32 + lane];
        db[i] += other[(k * 2 * R::kValues + R::kValues + i) * 32 + lane];
      }
  }
  float* const p = parts + (size_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int i = 0; i < R::kValues; ++i)
    if (R::channel(i) < C) { p[R::channel(i)] = dg[i]; p[C + R::channel(i)] = db[i]; }
}

// Rows of any length, a block per row: the values are read again for each pass, the block's sums over rows are kept in parts themselves.
__global__ void __launch_bounds__(1024)
rows_fwd_long_kernel(float* __restrict__ y, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ b, int C, float eps)
{
  vlb::pdl_wait();
  __shared__ float red[2][1][32];
  float const* const xp = x + (size_t)blockIdx.x * C;
  float s[1] = {0.f};
#pragma unroll 8
  for (int c = threadIdx.x; c < C; c += 1024) s[0] += __ldg(xp + c);
  row_sums<1024>(s, red[0]);
  float const mean = s[0] / (float)C;
  s[0] = 0.f;
#pragma unroll 8
  for (int c = threadIdx.x; c < C; c += 1024) { float const d = __ldg(xp + c) - mean; s[0] += d * d; }
  row_sums<1024>(s, red[1]);
  float const r = 1.f / sqrtf(s[0] / (float)C + eps);
#pragma unroll 4
  for (int c = threadIdx.x; c < C; c += 1024) y[(size_t)blockIdx.x * C + c] = fmaf(__ldg(g + c), (__ldg(xp + c) - mean) * r, __ldg(b + c));
}

__global__ void __launch_bounds__(1024)
rows_bwd_long_kernel(float* __restrict__ dx, float* __restrict__ parts, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ dy,
                     int rows, int C, float eps)
{
  vlb::pdl_wait();
  __shared__ float red[2][4][32];
  float const n = (float)C;
  float* const own = parts ? parts + (size_t)blockIdx.x * 2 * C : nullptr;
  int even = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x, even ^= 1) {
    bool const first = row == (int)blockIdx.x;
    float const *const xp = x + (size_t)row * C, *const dp = dy + (size_t)row * C;
    float m[1] = {0.f};
#pragma unroll 8
    for (int c = threadIdx.x; c < C; c += 1024) m[0] += __ldg(xp + c);
    row_sums<1024>(m, red[even] + 3);
    float const mean = m[0] / n;
    float s[3] = {};
#pragma unroll 4
    for (int c = threadIdx.x; c < C; c += 1024) {
      float const v = __ldg(xp + c) - mean, gd = __ldg(g + c) * __ldg(dp + c);
      s[0] += v * v; s[1] += gd; s[2] += gd * v;
    }
    row_sums<1024>(s, red[even]);
    float const r = 1.f / sqrtf(s[0] / n + eps), m1 = s[1] / n, m2 = s[2] * r / n;
#pragma unroll 4
    for (int c = threadIdx.x; c < C; c += 1024) {
      float const xh = (__ldg(xp + c) - mean) * r, d = __ldg(dp + c);
      if (dx) dx[(size_t)row * C + c] = r * (__ldg(g + c) * d - m1 - xh * m2);
      if (own) {
        own[c] = first ? d * xh : own[c] + d * xh;
        own[C + c] = first ? d : own[C + c] + d;
      }
    }
  }
}

// ------------------------------------------------------------------ positions of maps
// A block takes tiles of kQ neighbouring positions: a thread has kPos neighbouring ones -- 4, by 16-byte accesses, where planes and tensors allow it, or 1 -- of
// kValues channels in its registers, a warp's lanes kQ / kPos groups of positions of as many channels as fit.  Small blocks, several to an SM, and many
// values to a thread: what waits at one block's sums is covered by the loads of another's, and the sums over channels go over few warps.  28 x 28 x 512 x 64 forward:
// 36 us, by one block of 16 warps and 32 positions 49; backward 67 and 176 (a block of 32 warps); 64 x 64 x 64 x 64 backward 40, by blocks of 8 warps with 4 channels to
// a thread 169.  Tiles that come ahead through a ring in shared memory gained nothing over that: 36 / 38 us forward, 67 / 68 backward.
// A launch takes the smallest shape that holds the channels.  With the next larger one, 28 x 28 and 27 x 29 (accesses of 16 and of 4 bytes), 40 million values, us:
//   channels          32         64         128        256        512        1024
//   28 x 28 forward   62 (81)    68 (78)    69 (86)    60 (88)    60 (91)    68 (111)
//           backward  112 (135)  89 (141)   90 (146)   92 (157)   106 (179)  131 (242)
//   27 x 29 forward   64 (109)   64 (97)    71 (102)   71 (108)   82 (126)   92 (138)
//           backward  109 (186)  104 (174)  107 (180)  118 (186)  126 (200)  137 (247)
struct Place { size_t at; bool in; };

__device__ __forceinline__ Place place_of(long long q, long long positions, int P, int C)
{
  bool const in = q < positions;
  unsigned const t = (unsigned)(in ? q : positions - 1), n = t / (unsigned)P;
  return {(size_t)n * P * C + (t - n * P), in};
}

// A kernel for maps: warps, positions of a tile and of a thread, channels of a thread, blocks that an SM holds.
template <int W, int Q, int P, int V, int B>
struct Shape { static constexpr int kWarps = W, kQ = Q, kPos = P, kValues = V, kPerSm = B; };

template <class T>
struct Strip {
  static constexpr int kWarps = T::kWarps, kQ = T::kQ, kPos = T::kPos, kValues = T::kValues;
  static constexpr int kLanes = kQ / kPos, kChannels = 32 / kLanes, kPass = kWarps * kChannels;       // lanes of a channel; channels of a warp's row, of a row of all warps
  static __device__ __forceinline__ int channel(int i) { return i * kPass + (int)(threadIdx.x >> 5) * kChannels + (int)(threadIdx.x & 31) / kLanes; }
  // the thread's first position; those behind the batch's last (all kPos of them) repeat earlier ones
  static __device__ __forceinline__ Place place(int tile, long long positions, int P, int C)
  {
    long long const q = (long long)tile * kQ + (threadIdx.x & 31) % kLanes * kPos;
    Place const p = place_of(min(q, positions - kPos), positions, P, C);
    return {p.at, q < positions};
  }
  static __device__ __forceinline__ void load(float (&v)[kValues][kPos], float const* __restrict__ from, int P, int C)
  {
#pragma unroll
    for (int i = 0; i < kValues; ++i) {
      bool const in = channel(i) < C;
      float const* const p = from + (size_t)P * channel(i);
      if (kPos == 4) {
        float4 const q = in ? __ldg((float4 const*)p) : make_float4(0, 0, 0, 0);
        v[i][0] = q.x; v[i][1 % kPos] = q.y; v[i][2 % kPos] = q.z; v[i][3 % kPos] = q.w;
      } else {
        v[i][0] = in ? __ldg(p) : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void store(float* __restrict__ p, float const (&v)[kPos])
  {
    if (kPos == 4) *(float4*)p = make_float4(v[0], v[1 % kPos], v[2 % kPos], v[3 % kPos]);
    else *p = v[0];
  }
  // sums over the block's channels, position by position
  template <int kCount>
  static __device__ __forceinline__ void totals(float (&v)[kCount][kPos], float (*red)[kWarps][kQ])
  {
    int const lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = lane % kLanes * kPos;
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
#pragma unroll
      for (int p = 0; p < kPos; ++p)
        for (int o = kLanes; o < 32; o <<= 1) v[k][p] += __shfl_xor_sync(0xffffffffu, v[k][p], o);
      if (lane < kLanes) store(&red[k][warp][at], v[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      float t[kPos] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (kPos == 4) {
          float4 const q = *(float4 const*)&red[k][w][at];
          t[0] += q.x; t[1 % kPos] += q.y; t[2 % kPos] += q.z; t[3 % kPos] += q.w;
        } else {
          t[0] += red[k][w][at];
        }
      }
#pragma unroll
      for (int p = 0; p < kPos; ++p) v[k][p] = t[p];
    }
  }
};

template <class T>
__global__ void __launch_bounds__(T::kWarps * 32, T::kPerSm)
maps_fwd_kernel(float* __restrict__ y, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ b, long long positions, int tiles,
                int P, int C, float eps)
{
  using S = Strip<T>;
  constexpr int kPos = S::kPos, kValues = S::kValues;
  __shared__ __align__(16) float red[2][2][S::kWarps][S::kQ];
  vlb::pdl_wait();
  float const n = (float)C;
  int even = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, even ^= 1) {
    Place const at = S::place(tile, positions, P, C);
    float v[kValues][kPos], s[1][kPos] = {}, mean[kPos], r[kPos];
    S::load(v, x + at.at, P, C);
#pragma unroll
    for (int i = 0; i < kValues; ++i)
#pragma unroll
      for (int p = 0; p < kPos; ++p) s[0][p] += v[i][p];
    S::totals(s, red[even]);
#pragma unroll
    for (int p = 0; p < kPos; ++p) { mean[p] = s[0][p] / n; s[0][p] = 0.f; }
#pragma unroll
    for (int i = 0; i < kValues; ++i)
#pragma unroll
      for (int p = 0; p < kPos; ++p) { v[i][p] -= mean[p]; s[0][p] += S::channel(i) < C ? v[i][p] * v[i][p] : 0.f; }
    S::totals(s, red[even] + 1);
#pragma unroll
    for (int p = 0; p < kPos; ++p) r[p] = 1.f / sqrtf(s[0][p] / n + eps);
    float* to = y + at.at + (size_t)P * S::channel(0);
    if (at.in)
#pragma unroll
      for (int i = 0; i < kValues; ++i, to += (size_t)P * S::kPass)
        if (S::channel(i) < C) {
          float const gc = __ldg(g + S::channel(i)), bc = __ldg(b + S::channel(i));
#pragma unroll
          for (int p = 0; p < kPos; ++p) v[i][p] = fmaf(gc, v[i][p] * r[p], bc);
          S::store(to, v[i]);
        }
  }
}

// More channels than that: the values are read again for each pass.
template <int kWarps>
__global__ void __launch_bounds__(kWarps * 32)
maps_fwd_long_kernel(float* __restrict__ y, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ b, long long positions, int P, int C,
                     float eps)
{
  using S = Strip<Shape<kWarps, 32, 1, 1, 1>>;
  __shared__ float red[2][1][kWarps][32];
  vlb::pdl_wait();
  int const warp = threadIdx.x >> 5;
  Place const at = S::place(blockIdx.x, positions, P, C);
  float const* const xp = x + at.at;
  float m[1][1] = {}, s[1][1] = {};
#pragma unroll 8
  for (int c = warp; c < C; c += kWarps) m[0][0] += __ldg(xp + (size_t)P * c);
  S::totals(m, red[0]);
  float const mean = m[0][0] / (float)C;
#pragma unroll 8
  for (int c = warp; c < C; c += kWarps) { float const v = __ldg(xp + (size_t)P * c) - mean; s[0][0] += v * v; }
  S::totals(s, red[1]);
  float const r = 1.f / sqrtf(s[0][0] / (float)C + eps);
  if (!at.in) return;
#pragma unroll 8
  for (int c = warp; c < C; c += kWarps) y[at.at + (size_t)P * c] = fmaf(__ldg(g + c), (__ldg(xp + (size_t)P * c) - mean) * r, __ldg(b + c));
}

// Sums over groups of kLanes neighbouring lanes of kCount values, both powers of two: lane l ends with v[0 ...] the totals of the values
// l % kLanes % kCount * (kCount / kLanes) ... (kCount / kLanes of them, or one).
template <int kLanes, int kCount>
__device__ __forceinline__ void lane_sums(float (&v)[kCount])
{
  int const lane = threadIdx.x & 31;
  constexpr int kFew = kCount < kLanes ? kCount : kLanes;
#pragma unroll
  for (int s = kFew / 2, half = kCount / 2; s > 0; s >>= 1, half >>= 1) {
    bool const up = lane & s;
#pragma unroll
    for (int i = 0; i < kCount / 2; ++i) {
      if (i >= half) break;
      float const send = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, s);
    }
  }
#pragma unroll
  for (int s = kFew; s < kLanes; s <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], s);
}

// Tiles in turn to the blocks.  parts: [block][2][C].
template <class T>
__global__ void __launch_bounds__(T::kWarps * 32, T::kPerSm)
maps_bwd_kernel(float* __restrict__ dx, float* __restrict__ parts, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ dy,
                long long positions, int tiles, int P, int C, float eps)
{
  using S = Strip<T>;
  constexpr int kPos = S::kPos, kValues = S::kValues, kLanes = S::kLanes;
  constexpr int kOwn = kValues > kLanes ? kValues / kLanes : 1;              // channels whose sums over positions end with a lane
  __shared__ __align__(16) float red[2][4][S::kWarps][S::kQ];
  vlb::pdl_wait();
  float const n = (float)C;
  float sumG[kOwn] = {}, sumB[kOwn] = {};
  int even = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, even ^= 1) {
    Place const at = S::place(tile, positions, P, C);
    float v[kValues][kPos], d[kValues][kPos], m[1][kPos] = {}, s[3][kPos] = {};
    S::load(v, x + at.at, P, C);
    S::load(d, dy + at.at, P, C);
#pragma unroll
    for (int i = 0; i < kValues; ++i)
#pragma unroll
      for (int p = 0; p < kPos; ++p) m[0][p] += v[i][p];
    S::totals(m, red[even] + 3);
#pragma unroll
    for (int p = 0; p < kPos; ++p) m[0][p] /= n;
#pragma unroll
    for (int i = 0; i < kValues; ++i) {
      bool const real = S::channel(i) < C;
      float const gc = real ? __ldg(g + S::channel(i)) : 0.f;
#pragma unroll
      for (int p = 0; p < kPos; ++p) {
        v[i][p] = real ? v[i][p] - m[0][p] : 0.f;
        float const gd = gc * d[i][p];
        s[0][p] += v[i][p] * v[i][p]; s[1][p] += gd; s[2][p] += gd * v[i][p];
      }
    }
    S::totals(s, red[even]);
    float r[kPos], m1[kPos], m2[kPos];
#pragma unroll
    for (int p = 0; p < kPos; ++p) { r[p] = 1.f / sqrtf(s[0][p] / n + eps); m1[p] = s[1][p] / n; m2[p] = s[2][p] * r[p] / n; }
    float* to = dx + at.at + (size_t)P * S::channel(0);
    float tG[kValues], tB[kValues];
#pragma unroll
    for (int i = 0; i < kValues; ++i, to += (size_t)P * S::kPass) {
      tG[i] = tB[i] = 0.f;
#pragma unroll
      for (int p = 0; p < kPos; ++p) { v[i][p] *= r[p]; tG[i] += d[i][p] * v[i][p]; tB[i] += d[i][p]; }
      if (S::channel(i) < C && dx && at.in) {
        float const gc = __ldg(g + S::channel(i));
        float o[kPos];
#pragma unroll
        for (int p = 0; p < kPos; ++p) o[p] = r[p] * (gc * d[i][p] - m1[p] - v[i][p] * m2[p]);
        S::store(to, o);
      }
      if (!at.in) tG[i] = tB[i] = 0.f;
    }
    if (parts) {
      lane_sums<kLanes>(tG);
      lane_sums<kLanes>(tB);
#pragma unroll
      for (int k = 0; k < kOwn; ++k) { sumG[k] += tG[k]; sumB[k] += tB[k]; }
    }
  }
  int const lane = threadIdx.x & 31;
  if (!parts || lane % kLanes >= kValues) return;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    int const c = S::channel(lane % kLanes * kOwn + k);
    if (c < C) { parts[(size_t)blockIdx.x * 2 * C + c] = sumG[k]; parts[((size_t)blockIdx.x * 2 + 1) * C + c] = sumB[k]; }
  }
}

// Any number of channels: the values are read again for each pass, the block's sums over positions are kept in parts themselves.
template <int kWarps>
__global__ void __launch_bounds__(kWarps * 32)
maps_bwd_long_kernel(float* __restrict__ dx, float* __restrict__ parts, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ dy,
                     long long positions, int tiles, int P, int C, float eps)
{
  vlb::pdl_wait();
  using M = Strip<Shape<kWarps, 32, 1, 1, 1>>;
  __shared__ float red[2][4][kWarps][32];
  int const warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float const n = (float)C;
  float* const own = parts ? parts + (size_t)blockIdx.x * 2 * C : nullptr;
  int even = 0;
  bool first = true;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, even ^= 1, first = false) {
    Place const at = M::place(tile, positions, P, C);
    float const *const xp = x + at.at, *const dp = dy + at.at;
    float m[1][1] = {};
#pragma unroll 8
    for (int c = warp; c < C; c += kWarps) m[0][0] += __ldg(xp + (size_t)P * c);
    M::totals(m, red[even] + 3);
    float const mean = m[0][0] / n;
    float s[3][1] = {};
#pragma unroll 4
    for (int c = warp; c < C; c += kWarps) {
      float const v = __ldg(xp + (size_t)P * c) - mean, gd = __ldg(g + c) * __ldg(dp + (size_t)P * c);
      s[0][0] += v * v; s[1][0] += gd; s[2][0] += gd * v;
    }
    M::totals(s, red[even]);
    float const r = 1.f / sqrtf(s[0][0] / n + eps), m1 = s[1][0] / n, m2 = s[2][0] * r / n;
    for (int c0 = warp; c0 < C; c0 += kWarps * 16) {
      float t[32];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        int const c = c0 + kWarps * i;
        float const xh = c < C ? (__ldg(xp + (size_t)P * c) - mean) * r : 0.f, d = c < C ? __ldg(dp + (size_t)P * c) : 0.f;
        if (dx && at.in && c < C) dx[at.at + (size_t)P * c] = r * (__ldg(g + c) * d - m1 - xh * m2);
        t[i] = at.in ? d * xh : 0.f; t[16 + i] = at.in ? d : 0.f;
      }
      if (own) {
        lane_sums<32>(t);
        float const sum = t[0];
        int const c = c0 + kWarps * (lane % 16);
        float* const p = own + (lane < 16 ? 0 : C) + c;
        if (c < C) *p = first ? sum : *p + sum;
      }
    }
  }
}

// dG and dB from the parts of `count` blocks, kCols columns per block, in a fixed order.
template <int kCols>
__global__ void __launch_bounds__(1024)
sum_blocks_kernel(float* __restrict__ dg, float* __restrict__ db, float const* __restrict__ parts, int count, int C)
{
  vlb::pdl_wait();
  __shared__ float all[32][kCols];
  int const tx = threadIdx.x % kCols, ty = threadIdx.x / kCols, c = (int)blockIdx.x * kCols + tx;
  float s = 0.f;
  if (c < 2 * C) {
#pragma unroll 4
    for (int i = ty; i < count; i += 1024 / kCols) s += __ldg(parts + (size_t)i * 2 * C + c);
  }
#pragma unroll
  for (int o = kCols; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) < kCols) all[threadIdx.x >> 5][tx] = s;
  __syncthreads();
  if (ty) return;
  s = all[0][tx];
#pragma unroll
  for (int i = 1; i < 32; ++i) s += all[i][tx];
  if (c < C) { if (dg) dg[c] = s; }
  else if (c < 2 * C) { if (db) db[c - C] = s; }
}

// Positions, and channels twice over, are walked through with 32-bit counters.
bool bad_shape(int H, int W, int C, int N)
{ return H <= 0 || W <= 0 || C <= 0 || N <= 0 || (long long)H * W > INT32_MAX || (long long)H * W * N > INT32_MAX - (1 << 20) || C > (1 << 30) - (1 << 20); }

bool wide(int C, std::initializer_list<void const*> ps)
{
  uintptr_t all = 0;
  for (void const* p : ps) all |= (uintptr_t)p;
  return C % 4 == 0 && (all & 15) == 0;
}

// Threads per row: as few as hold it with sixteen values each.  f(threads, vec) for the smallest that do; false for rows that are too long.
template <class F>
bool with_row(int C, F f)
{
  if (C <= 128)   { f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{}); return true; }
  if (C <= 256)   { f(std::integral_constant<int, 32>{}, std::integral_constant<int, 2>{}); return true; }
  if (C <= 512)   { f(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{}); return true; }
  if (C <= 1024)  { f(std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{}); return true; }
  if (C <= 2048)  { f(std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{}); return true; }
  if (C <= 4096)  { f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{}); return true; }
  if (C <= 8192)  { f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{}); return true; }
  return false;
}

}  // namespace

namespace vlb {

cudaError_t lnorm_set_wait_limit(long long cycles, cudaStream_t stream)
{
  long long const v = cycles == 0 ? kWaitCycles : cycles;
  return cudaMemcpyToSymbolAsync(gWaitCycles, &v, sizeof(v), 0, cudaMemcpyHostToDevice, stream);
}

}  // namespace vlb

extern "C" {

int vlb_lnorm_forward(vlb_ctx* ctx, float* Y, float const* X, float const* g, float const* b, int H, int W, int C, int N, double eps)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, !bad_shape(H, W, C, N), "lnorm_forward: bad shape");
  VLB_REQUIRE(ctx, Y && X && g && b, "lnorm_forward: null tensor");
  VLB_REQUIRE(ctx, vlb::on_its_device(ctx), "lnorm_forward: the context belongs to another device than the current one");
  VLB_REQUIRE(ctx, eps >= 0, "lnorm_forward: epsilon is negative");
  int const P = H * W, positions = P * N;
  bool done = false;
  if (P == 1) {
    bool const vec = wide(C, {Y, X, g, b});
    done = with_row(C, [&](auto threads, auto count) {
      constexpr int kThreads = decltype(threads)::value, kVec = decltype(count)::value, kRows = block_of(kThreads) / kThreads;
      auto const kernel = vec ? rows_fwd_kernel<kThreads, kVec, true> : rows_fwd_kernel<kThreads, kVec, false>;
      vlb::launch(ctx->stream, kernel, (unsigned)vlb::ceil_div(N, kRows), block_of(kThreads), 0, Y, X, g, b, N, C, (float)eps);
    });
    if (!done) vlb::launch(ctx->stream, rows_fwd_long_kernel, (unsigned)N, 1024, 0, Y, X, g, b, C, (float)eps);
    done = true;
  }
  if (!done) {
    auto run = [&](auto shape) {
      using T = decltype(shape);
      int const tiles = vlb::ceil_div(positions, T::kQ);
      vlb::launch(ctx->stream, maps_fwd_kernel<T>, (unsigned)std::min(tiles, ctx->smCount * T::kPerSm), T::kWarps * 32, 0, Y, X, g, b, (long long)positions, tiles, P, C, (float)eps);
    };
    if (wide(P, {Y, X})) {
      if (C <= 32)        run(Shape<2, 32, 4, 4, 16>{});
      else if (C <= 64)   run(Shape<2, 32, 4, 8, 12>{});
      else if (C <= 128)  run(Shape<4, 32, 4, 8, 8>{});
      else if (C <= 256)  run(Shape<8, 32, 4, 8, 4>{});
      else if (C <= 512)  run(Shape<8, 16, 4, 8, 4>{});
      else if (C <= 1024) run(Shape<8, 16, 4, 16, 2>{});
      else if (C <= 2048) run(Shape<16, 8, 4, 8, 2>{});
      else done = true;
    } else {
      if (C <= 32)        run(Shape<2, 32, 1, 16, 16>{});
      else if (C <= 64)   run(Shape<4, 32, 1, 16, 8>{});
      else if (C <= 128)  run(Shape<4, 32, 1, 32, 6>{});
      else if (C <= 256)  run(Shape<8, 32, 1, 32, 4>{});
      else if (C <= 512)  run(Shape<8, 16, 1, 32, 4>{});
      else if (C <= 1024) run(Shape<16, 16, 1, 32, 2>{});
      else if (C <= 2048) run(Shape<16, 8, 1, 32, 2>{});
      else done = true;
    }
    if (done) vlb::launch(ctx->stream, maps_fwd_long_kernel<32>, (unsigned)vlb::ceil_div(positions, 32), 1024, 0, Y, X, g, b, (long long)positions, P, C, (float)eps);
  }
  VLB_LAUNCHED(ctx, 1);
  return vlb::check_launch(ctx, "vlb_lnorm_forward");
}

int vlb_lnorm_backward(vlb_ctx* ctx, float* dX, float* dG, float* dB, float const* X, float const* g, float const* dY,
                       int H, int W, int C, int N, double eps)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, !bad_shape(H, W, C, N), "lnorm_backward: bad shape");
  VLB_REQUIRE(ctx, X && g && dY, "lnorm_backward: null tensor");
  VLB_REQUIRE(ctx, vlb::on_its_device(ctx), "lnorm_backward: the context belongs to another device than the current one");
  VLB_REQUIRE(ctx, eps >= 0, "lnorm_backward: epsilon is negative");
  if (!dX && !dG && !dB) return VLB_Success;
  int const P = H * W, positions = P * N, most = most_parts(ctx, C);
  float* parts = nullptr;
  if (dG || dB) {
    parts = (float*)vlb::workspace(ctx, sizeof(float) * 2 * (size_t)C * most);
    if (!parts) return vlb::pass_error(ctx, ctx->lastError, "vlb_lnorm_backward");
  }
  int blocks = 0;
  cudaError_t failed = cudaSuccess;
  if (P == 1) {
    bool const vec = wide(C, {dX, X, g, dY});
    with_row(C, [&](auto threads, auto count) {
      constexpr int kThreads = decltype(threads)::value, kVec = decltype(count)::value, kRows = block_of(kThreads) / kThreads;
      // Groups of rows of 16 KB, for four blocks of 128 threads per SM or as many threads in larger ones; and as many blocks as fit the device at once, which a block's
      // three groups of X and dY decide where it has a row to a warp: with two blocks per SM 16384 x 512 takes 28.5 us, with four, of which two wait, 32.6.
      int const perSm = std::max(1, std::min(4, 512 / block_of(kThreads))), per = kThreads == 32 ? std::max(1, std::min(4096 / (C * kRows), N / (kRows * ctx->smCount * perSm))) : 1;
      size_t const smem = vec ? sizeof(float) * kStages * 2 * per * kRows * C : 0, other = 2048 + sizeof(float) * (kRows - 1) * 2 * 32 * 4 * kVec;
      int const fit = std::max(1, std::min(perSm, (int)(228 * 1024 / (smem + other))));
      blocks = std::min(vlb::ceil_div(N, kRows * per), std::min(most, ctx->smCount * fit));
      auto const kernel = vec ? rows_bwd_kernel<kThreads, kVec, true> : rows_bwd_kernel<kThreads, kVec, false>;
      static bool ready[64];                               // (of this kernel and device)
      if (smem > 32 * 1024 && !ready[ctx->device & 63]) {
        failed = vlb::allow_max_dynamic_smem(kernel);
        ready[ctx->device & 63] = failed == cudaSuccess;
      }
      if (failed == cudaSuccess)
        vlb::launch(ctx->stream, kernel, (unsigned)blocks, block_of(kThreads), smem, dX, parts, X, g, dY, N, C, per, (float)eps, ctx->deviceStatus, ctx->testSwitch & 1);
    });
    if (failed != cudaSuccess) return vlb::set_error(ctx, VLB_Cuda, cudaGetErrorString(failed));
    if (!blocks) {
      blocks = std::min(N, std::min(most, ctx->smCount * 2));
      vlb::launch(ctx->stream, rows_bwd_long_kernel, (unsigned)blocks, 1024, 0, dX, parts, X, g, dY, N, C, (float)eps);
    }
  }
  if (!blocks) {
    auto run = [&](auto shape) {
      using T = decltype(shape);
      int const tiles = vlb::ceil_div(positions, T::kQ);
      blocks = std::min(tiles, std::min(most, ctx->smCount * T::kPerSm));
      vlb::launch(ctx->stream, maps_bwd_kernel<T>, (unsigned)blocks, T::kWarps * 32, 0, dX, parts, X, g, dY, (long long)positions, tiles, P, C, (float)eps);
    };
    if (wide(P, {dX, X, dY})) {
      if (C <= 32)        run(Shape<2, 32, 4, 4, 8>{});
      else if (C <= 64)   run(Shape<2, 32, 4, 8, 8>{});
      else if (C <= 128)  run(Shape<4, 32, 4, 8, 4>{});
      else if (C <= 256)  run(Shape<4, 16, 4, 8, 4>{});
      else if (C <= 512)  run(Shape<4, 8, 4, 8, 4>{});
      else if (C <= 1024) run(Shape<4, 8, 4, 16, 2>{});
      else if (C <= 2048) run(Shape<16, 8, 4, 8, 1>{});
    } else {
      if (C <= 32)        run(Shape<2, 32, 1, 16, 8>{});
      else if (C <= 64)   run(Shape<4, 32, 1, 16, 6>{});
      else if (C <= 128)  run(Shape<4, 32, 1, 32, 4>{});
      else if (C <= 256)  run(Shape<8, 32, 1, 32, 2>{});
      else if (C <= 512)  run(Shape<8, 16, 1, 32, 2>{});
      else if (C <= 1024) run(Shape<8, 8, 1, 32, 2>{});
      else if (C <= 2048) run(Shape<16, 8, 1, 32, 1>{});
    }
    if (C > 2048) {
      int const tiles = vlb::ceil_div(positions, 32);
      blocks = std::min(tiles, std::min(most, ctx->smCount * 2));
      vlb::launch(ctx->stream, maps_bwd_long_kernel<16>, (unsigned)blocks, 512, 0, dX, parts, X, g, dY, (long long)positions, tiles, P, C, (float)eps);
    }
  }
  VLB_LAUNCHED(ctx, 1);
  if (parts) {
    // columns of a block: few, where 32 would leave most of the device idle
    if (2ll * C >= 32ll * ctx->smCount) vlb::launch(ctx->stream, sum_blocks_kernel<32>, (unsigned)vlb::ceil_div(2ll * C, 32), 1024, 0, dG, dB, parts, blocks, C);
    else                                vlb::launch(ctx->stream, sum_blocks_kernel<8>, (unsigned)vlb::ceil_div(2ll * C, 8), 1024, 0, dG, dB, parts, blocks, C);
    VLB_LAUNCHED(ctx, 1);
  }
  return vlb::check_launch(ctx, "vlb_lnorm_backward");
}

}  // extern "C"
