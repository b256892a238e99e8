// The Muon solver (include/vlb.h has the formulas).
#include "products.cuh"
#include <math.h>
#include <algorithm>

namespace {

constexpr int kThreads = 256, kMaxParts = 592;

// Momentum; u = what is to be orthogonalised; a part of the sum of its squares per block, in double precision.
__global__ void __launch_bounds__(kThreads)
momentum_kernel(float* __restrict__ u, float* __restrict__ s1, float const* __restrict__ w, float const* __restrict__ g, size_t n, float gradMult,
                float decay, float momentum, int nesterov, double* __restrict__ parts)
{
  vlb::pdl_wait();
  double sum = 0;
  for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < n; i += (size_t)gridDim.x * kThreads) {
    float const d = gradMult * g[i] + decay * w[i], m = momentum * s1[i] + d, v = nesterov ? d + momentum * m : m;
    s1[i] = m;
    u[i] = v;
    sum += (double)v * v;
  }
  __shared__ double all[kThreads / 32];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads / 32; ++i) sum += all[i];
    parts[blockIdx.x] = sum;
  }
}

__global__ void normalise_kernel(float* __restrict__ u, size_t n, double const* __restrict__ parts, int count, double epsilon)
{
  vlb::pdl_wait();
  double sum = 0;
  for (int i = 0; i < count; ++i) sum += parts[i];
  float const f = (float)(1. / (sqrt(sum) + epsilon));
  for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < n; i += (size_t)gridDim.x * kThreads) u[i] *= f;
}

__global__ void step_kernel(float* __restrict__ w, float const* __restrict__ x, size_t n, float rate)
{
  vlb::pdl_wait();
  for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < n; i += (size_t)gridDim.x * kThreads) w[i] -= rate * x[i];
}

}  // namespace

extern "C" {

int vlb_muon_update_many(vlb_ctx* ctx, int count, vlb_muon_param const* u, double gradMult, vlb_muon_opts const* o)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, count >= 0 && (u || count == 0) && o, "muon_update_many: null argument");
  VLB_REQUIRE(ctx, o->steps >= 0 && o->epsilon >= 0, "muon_update_many: steps and epsilon must not be negative");
  size_t most = 0;
  for (int i = 0; i < count; ++i) {
    VLB_REQUIRE(ctx, u[i].rows > 0 && u[i].cols > 0, "muon_update_many: bad shape");
    VLB_REQUIRE(ctx, u[i].W && u[i].S1 && u[i].G, "muon_update_many: null tensor");
    size_t const m = std::min(u[i].rows, u[i].cols);
    most = std::max(most, 2 * (size_t)u[i].rows * u[i].cols + 2 * m * m);
  }
  if (count == 0) return VLB_Success;
  double* const parts = (double*)vlb::workspace(ctx, sizeof(double) * kMaxParts + sizeof(float) * most);
  if (!parts) return vlb::pass_error(ctx, ctx->lastError, "vlb_muon_update_many");
  for (int i = 0; i < count; ++i) {
    int const rows = u[i].rows, cols = u[i].cols, m = std::min(rows, cols);
    size_t const n = (size_t)rows * cols;
    float *x = (float*)(parts + kMaxParts), *next = x + n, *const a = next + n, *const q = a + (size_t)m * m;
    unsigned const grid = vlb::grid_for(n, kThreads, kMaxParts);
    vlb::launch(ctx->stream, momentum_kernel, grid, kThreads, 0, x, u[i].S1, u[i].W, u[i].G, n, (float)gradMult, (float)u[i].decay,
                (float)o->momentum, o->nesterov, parts);
    vlb::launch(ctx->stream, normalise_kernel, grid, kThreads, 0, x, n, parts, (int)grid, o->epsilon);
    for (int k = 0; k < o->steps; ++k) {
      vlb::Operand const byRow = {x, cols, 1}, byCol = {x, 1, cols};
      if (rows <= cols) vlb::products_exact(ctx, a, m, m, m, cols, byRow, byRow, 1.f, 0.f, nullptr, nullptr);
      else              vlb::products_exact(ctx, a, m, m, m, rows, byCol, byCol, 1.f, 0.f, nullptr, nullptr);
      vlb::products_exact(ctx, q, m, m, m, m, {a, m, 1}, {a, m, 1}, (float)o->c, (float)o->b, a, nullptr);
      if (rows <= cols) vlb::products_exact(ctx, next, cols, rows, cols, rows, {q, m, 1}, byCol, 1.f, (float)o->a, x, nullptr);
      else              vlb::products_exact(ctx, next, cols, rows, cols, cols, byRow, {q, m, 1}, 1.f, (float)o->a, x, nullptr);
      std::swap(x, next);
    }
    vlb::launch(ctx->stream, step_kernel, grid, kThreads, 0, u[i].W, x, n, (float)(u[i].lr * sqrt(std::max(1., (double)rows / cols))));
    VLB_LAUNCHED(ctx, 3);
  }
  return vlb::check_launch(ctx, "vlb_muon_update_many");
}

}  // extern "C"
