// A fully connected prediction layer and the softmax loss behind it, in pieces of classes (include/vlb.h has the formulas).
#include "products.cuh"
#include <algorithm>

namespace {

using vlb::Operand;

constexpr int kThreads = 256;

// What the pieces so far have shown of an image's predictions: the largest, the sum of exp(z - largest), the label's.
struct Seen { float top, sum, label; };

struct Label { bool real; int at; };

// As vlb_softmaxloss_*: class 0 skips the image, a class above K too and is reported.
__device__ __forceinline__ Label label_of(float const* labels, int n, int K, int* status)
{
  float const l = labels[n];
  bool const tooBig = l > (float)K;
  if (tooBig && status) atomicExch(status, kStatusBadLabel);
  return {l > 0.f && !tooBig, min(max((int)l - 1, 0), K - 1)};
}

__device__ __forceinline__ float block_reduce(float v, bool isMax, float* red)
{
  for (int o = 16; o > 0; o >>= 1) { float const u = __shfl_xor_sync(0xffffffffu, v, o); v = isMax ? fmaxf(v, u) : v + u; }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kThreads / 32; ++i) v = isMax ? fmaxf(v, red[i]) : v + red[i];
  return v;
}

// An image's place in one sum: exp(-inf - -inf) does not arise, a largest value that is not finite gives what the definition gives.
__device__ __forceinline__ float exp_below(float z, float top) { return z == top ? 1.f : expf(z - top); }

// z: N x ld, columns k0 .. k0 + cols - 1 of the predictions.  A block per image.
__global__ void seen_kernel(Seen* __restrict__ seen, float const* __restrict__ z, long long ld, int cols, int k0, int K, float const* __restrict__ labels)
{
  vlb::pdl_wait();
  __shared__ float red[32];
  int const n = blockIdx.x;
  Label const l = label_of(labels, n, K, nullptr);
  if (!l.real) return;
  float const* const row = z + n * ld;
  float m = -INFINITY;
  for (int c = threadIdx.x; c < cols; c += kThreads) m = fmaxf(m, row[c]);
  m = block_reduce(m, true, red);
  Seen s = k0 ? seen[n] : Seen{-INFINITY, 0.f, 0.f};
  float const top = fmaxf(m, s.top);
  float sum = 0.f;
  for (int c = threadIdx.x; c < cols; c += kThreads) sum += exp_below(row[c], top);
  sum = block_reduce(sum, false, red);
  if (threadIdx.x == 0) {
    if (l.at >= k0 && l.at < k0 + cols) s.label = row[l.at - k0];
    s.sum = (s.sum == 0.f ? 0.f : s.sum * exp_below(s.top, top)) + sum;
    s.top = top;
    seen[n] = s;
  }
}

__global__ void loss_kernel(float* __restrict__ loss, float* __restrict__ lse, Seen const* __restrict__ seen, float const* __restrict__ labels, int N, int K,
                            int* status)
{
  vlb::pdl_wait();
  __shared__ float red[32];
  double sum = 0;
  for (int n = threadIdx.x; n < N; n += kThreads) {
    Label const l = label_of(labels, n, K, status);
    float v = 0.f;
    if (l.real) { v = seen[n].top + logf(seen[n].sum); sum += (double)v - seen[n].label; }
    if (lse) lse[n] = v;
  }
  __shared__ double all[kThreads];
  all[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads; ++i) sum += all[i];
    if (loss) *loss = (float)(sum / N);
  }
}

// z -> dz in place.  A block per image.
__global__ void dz_kernel(float* __restrict__ z, long long ld, int cols, int k0, int K, float const* __restrict__ labels, float const* __restrict__ lse,
                          float scale, int* status)
{
  vlb::pdl_wait();
  int const n = blockIdx.x;
  Label const l = label_of(labels, n, K, status);
  float* const row = z + n * ld;
  for (int c = threadIdx.x; c < cols; c += kThreads)
    row[c] = l.real ? (expf(row[c] - lse[n]) - (k0 + c == l.at ? 1.f : 0.f)) * scale : 0.f;
}

// X without the images that are skipped, whose values may be anything.
__global__ void real_rows_kernel(float* __restrict__ out, float const* __restrict__ x, int D, int K, float const* __restrict__ labels)
{
  vlb::pdl_wait();
  size_t const at = (size_t)blockIdx.x * D;
  bool const real = label_of(labels, blockIdx.x, K, nullptr).real;
  for (int d = threadIdx.x; d < D; d += kThreads) out[at + d] = real ? x[at + d] : 0.f;
}

// db[c] = sum over the images of dz.  A thread per class.
__global__ void db_kernel(float* __restrict__ db, float const* __restrict__ dz, long long ld, int cols, int N)
{
  vlb::pdl_wait();
  int const c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int n = 0; n < N; ++n) s += dz[n * ld + c];
  db[c] = s;
}

// Classes per piece: predictions of a piece up to 64 MB.
int piece_of(int N, int K) { return (int)std::min<long long>(K, std::max<long long>(64, (16ll << 20) / N / 64 * 64)); }

}  // namespace

extern "C" {

int vlb_fc_softmaxloss_forward(vlb_ctx* ctx, float* loss, float* lse, float const* X, float const* F, float const* b, float const* labels,
                               int H, int W, int C, int N, int K)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, H > 0 && W > 0 && C > 0 && N > 0 && K > 0 && (long long)H * W * C <= INT32_MAX, "fc_softmaxloss_forward: bad shape");
  VLB_REQUIRE(ctx, loss && X && F && labels, "fc_softmaxloss_forward: null tensor");
  int const D = H * W * C, piece = piece_of(N, K);
  char* const ws = (char*)vlb::workspace(ctx, sizeof(float) * (size_t)N * piece + sizeof(Seen) * (size_t)N);
  if (!ws) return vlb::pass_error(ctx, ctx->lastError, "vlb_fc_softmaxloss_forward");
  float* const z = (float*)ws;
  Seen* const seen = (Seen*)(z + (size_t)N * piece);
  for (int k0 = 0; k0 < K; k0 += piece) {
    int const cols = std::min(piece, K - k0);
    vlb::products_exact(ctx, z, piece, N, cols, D, {X, D, 1}, {F + (size_t)k0 * D, D, 1}, 1.f, 0.f, nullptr, b ? b + k0 : nullptr);
    vlb::launch(ctx->stream, seen_kernel, (unsigned)N, kThreads, 0, seen, z, (long long)piece, cols, k0, K, labels);
    VLB_LAUNCHED(ctx, 1);
  }
  vlb::launch(ctx->stream, loss_kernel, 1, kThreads, 0, loss, lse, seen, labels, N, K, ctx->deviceStatus);
  VLB_LAUNCHED(ctx, 1);
  return vlb::check_launch(ctx, "vlb_fc_softmaxloss_forward");
}

int vlb_fc_softmaxloss_backward(vlb_ctx* ctx, float* dX, float* dF, float* db, float const* X, float const* F, float const* b,
                                float const* labels, float const* lse, double dzdy, int H, int W, int C, int N, int K)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, H > 0 && W > 0 && C > 0 && N > 0 && K > 0 && (long long)H * W * C <= INT32_MAX, "fc_softmaxloss_backward: bad shape");
  VLB_REQUIRE(ctx, X && F && labels, "fc_softmaxloss_backward: null tensor");
  int const D = H * W * C, piece = piece_of(N, K);
  size_t const ND = (size_t)N * D;
  float* const z = (float*)vlb::workspace(ctx, sizeof(float) * ((size_t)N * piece + N + ND) + sizeof(Seen) * (size_t)N);
  if (!z) return vlb::pass_error(ctx, ctx->lastError, "vlb_fc_softmaxloss_backward");
  float *const real = z + (size_t)N * piece, *const own = real + ND;
  Seen* const seen = (Seen*)(own + N);
  vlb::launch(ctx->stream, real_rows_kernel, (unsigned)N, kThreads, 0, real, X, D, K, labels);
  VLB_LAUNCHED(ctx, 1);
  for (int pass = lse ? 1 : 0; pass < 2; ++pass) {
    for (int k0 = 0; k0 < K; k0 += piece) {
      int const cols = std::min(piece, K - k0);
      float const* const f = F + (size_t)k0 * D;
      vlb::products_exact(ctx, z, piece, N, cols, D, {real, D, 1}, {f, D, 1}, 1.f, 0.f, nullptr, b ? b + k0 : nullptr);
      if (pass == 0) {
        vlb::launch(ctx->stream, seen_kernel, (unsigned)N, kThreads, 0, seen, z, (long long)piece, cols, k0, K, labels);
        VLB_LAUNCHED(ctx, 1);
        continue;
      }
      vlb::launch(ctx->stream, dz_kernel, (unsigned)N, kThreads, 0, z, (long long)piece, cols, k0, K, labels, lse ? lse : own,
                  (float)(dzdy / N), ctx->deviceStatus);
      VLB_LAUNCHED(ctx, 1);
      if (dX) vlb::products_exact(ctx, dX, D, N, D, cols, {z, piece, 1}, {f, 1, D}, 1.f, k0 ? 1.f : 0.f, dX, nullptr);
      if (dF) vlb::products_exact(ctx, dF + (size_t)k0 * D, D, cols, D, N, {z, 1, piece}, {real, 1, D}, 1.f, 0.f, nullptr, nullptr);
      if (db) {
        vlb::launch(ctx->stream, db_kernel, (unsigned)vlb::ceil_div(cols, kThreads), kThreads, 0, db + k0, z, (long long)piece, cols, N);
        VLB_LAUNCHED(ctx, 1);
      }
    }
    if (pass == 0) {
      vlb::launch(ctx->stream, loss_kernel, 1, kThreads, 0, nullptr, own, seen, labels, N, K, nullptr);
      VLB_LAUNCHED(ctx, 1);
    }
  }
  return vlb::check_launch(ctx, "vlb_fc_softmaxloss_backward");
}

}  // extern "C"
