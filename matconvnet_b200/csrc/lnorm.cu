// Layer normalisation over the channels of a position (include/vlb.h has the formulas).
#include "common.cuh"

namespace {

constexpr int kThreads = 256;

// Sum of a and of b over the block, in every thread; red: 2 * 32 floats of shared memory.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2* red)
{
  for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int i = 0; i < (int)blockDim.x / 32; ++i) { s.x += red[i].x; s.y += red[i].y; }
  return s;
}

struct Moments { float mean, r; };

__device__ __forceinline__ Moments moments_of(float const* x, size_t P, int C, float eps, float2* red)
{
  float s = 0.f;
  for (int c = threadIdx.x; c < C; c += blockDim.x) s += x[P * c];
  float const mean = block_sum2(s, 0.f, red).x / (float)C;
  float v = 0.f;
  for (int c = threadIdx.x; c < C; c += blockDim.x) { float const d = x[P * c] - mean; v += d * d; }
  return {mean, 1.f / sqrtf(block_sum2(v, 0.f, red).x / (float)C + eps)};
}

// A block per position: P positions of an image, values of a position P floats apart.
__global__ void lnorm_fwd_kernel(float* __restrict__ y, float const* __restrict__ x, float const* __restrict__ g, float const* __restrict__ b,
                                 int P, int C, float eps)
{
  vlb::pdl_wait();
  __shared__ float2 red[32];
  size_t const at = blockIdx.x / P * ((size_t)P * C) + blockIdx.x % P;
  Moments const m = moments_of(x + at, P, C, eps, red);
  for (int c = threadIdx.x; c < C; c += blockDim.x) y[at + (size_t)P * c] = g[c] * ((x[at + (size_t)P * c] - m.mean) * m.r) + b[c];
}

__global__ void lnorm_dx_kernel(float* __restrict__ dx, Moments* __restrict__ moments, float const* __restrict__ x, float const* __restrict__ g,
                                float const* __restrict__ dy, int P, int C, float eps)
{
  vlb::pdl_wait();
  __shared__ float2 red[32];
  size_t const at = blockIdx.x / P * ((size_t)P * C) + blockIdx.x % P;
  Moments const m = moments_of(x + at, P, C, eps, red);
  if (threadIdx.x == 0) moments[blockIdx.x] = m;
  if (!dx) return;
  float s = 0.f, sx = 0.f;
  for (int c = threadIdx.x; c < C; c += blockDim.x) {
    float const gd = g[c] * dy[at + (size_t)P * c];
    s += gd; sx += gd * ((x[at + (size_t)P * c] - m.mean) * m.r);
  }
  float2 const t = block_sum2(s, sx, red);
  for (int c = threadIdx.x; c < C; c += blockDim.x) {
    size_t const i = at + (size_t)P * c;
    dx[i] = m.r * (g[c] * dy[i] - t.x / (float)C - (x[i] - m.mean) * m.r * (t.y / (float)C));
  }
}

// A block per channel.
__global__ void lnorm_dparam_kernel(float* __restrict__ dg, float* __restrict__ db, Moments const* __restrict__ moments, float const* __restrict__ x,
                                    float const* __restrict__ dy, int P, int C, int positions)
{
  vlb::pdl_wait();
  __shared__ float2 red[32];
  float s = 0.f, sx = 0.f;
  for (int p = threadIdx.x; p < positions; p += blockDim.x) {
    size_t const i = p / P * ((size_t)P * C) + p % P + (size_t)P * blockIdx.x;
    s += dy[i]; sx += dy[i] * ((x[i] - moments[p].mean) * moments[p].r);
  }
  float2 const t = block_sum2(s, sx, red);
  if (threadIdx.x == 0) {
    if (dg) dg[blockIdx.x] = t.y;
    if (db) db[blockIdx.x] = t.x;
  }
}

bool bad_shape(int H, int W, int C, int N) { return H <= 0 || W <= 0 || C <= 0 || N <= 0 || (long long)H * W * N > INT32_MAX; }

}  // namespace

extern "C" {

int vlb_lnorm_forward(vlb_ctx* ctx, float* Y, float const* X, float const* g, float const* b, int H, int W, int C, int N, double eps)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, !bad_shape(H, W, C, N), "lnorm_forward: bad shape");
  VLB_REQUIRE(ctx, Y && X && g && b, "lnorm_forward: null tensor");
  VLB_REQUIRE(ctx, eps >= 0, "lnorm_forward: epsilon is negative");
  vlb::launch(ctx->stream, lnorm_fwd_kernel, (unsigned)(H * W * N), kThreads, 0, Y, X, g, b, H * W, C, (float)eps);
  VLB_LAUNCHED(ctx, 1);
  return vlb::check_launch(ctx, "vlb_lnorm_forward");
}

int vlb_lnorm_backward(vlb_ctx* ctx, float* dX, float* dG, float* dB, float const* X, float const* g, float const* dY,
                       int H, int W, int C, int N, double eps)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, !bad_shape(H, W, C, N), "lnorm_backward: bad shape");
  VLB_REQUIRE(ctx, X && g && dY, "lnorm_backward: null tensor");
  VLB_REQUIRE(ctx, eps >= 0, "lnorm_backward: epsilon is negative");
  int const positions = H * W * N;
  Moments* const m = (Moments*)vlb::workspace(ctx, sizeof(Moments) * (size_t)positions);
  if (!m) return vlb::pass_error(ctx, ctx->lastError, "vlb_lnorm_backward");
  vlb::launch(ctx->stream, lnorm_dx_kernel, (unsigned)positions, kThreads, 0, dX, m, X, g, dY, H * W, C, (float)eps);
  if (dG || dB) vlb::launch(ctx->stream, lnorm_dparam_kernel, (unsigned)C, kThreads, 0, dG, dB, m, X, dY, H * W, C, positions);
  VLB_LAUNCHED(ctx, dG || dB ? 2 : 1);
  return vlb::check_launch(ctx, "vlb_lnorm_backward");
}

}  // extern "C"
