// Matrix products on CUDA cores: the arithmetic of VLB_PRECISION_FP32.
#include "products.cuh"

namespace {

using vlb::Strided;

constexpr int kTile = 64, kDepth = 16;

__global__ void __launch_bounds__(256)
products_exact_kernel(float* __restrict__ C, long long ldc, int M, int N, int K, int tilesM, Strided a, Strided b, float alpha, float beta,
                      float const* D, float const* __restrict__ bias)
{
  vlb::pdl_wait();
  __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4];
  int const i0 = (int)(blockIdx.x % tilesM) * kTile, j0 = (int)(blockIdx.x / tilesM) * kTile;
  int const tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  // neighbouring threads read neighbouring elements: along the reduction where that is the fast index, along the rows otherwise
  bool const aK = a.ks == 1, bK = b.ks == 1;
  for (int k0 = 0; k0 < K; k0 += kDepth) {
    for (int t = threadIdx.x; t < kTile * kDepth; t += 256) {
      int const ai = aK ? t / kDepth : t % kTile, ak = aK ? t % kDepth : t / kTile;
      int const bi = bK ? t / kDepth : t % kTile, bk = bK ? t % kDepth : t / kTile;
      as[ak][ai] = i0 + ai < M && k0 + ak < K ? a.p[(i0 + ai) * a.rs + (k0 + ak) * a.ks] : 0.f;
      bs[bk][bi] = j0 + bi < N && k0 + bk < K ? b.p[(j0 + bi) * b.rs + (k0 + bk) * b.ks] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      float4 const u = *(float4 const*)&as[k][ty * 4], v = *(float4 const*)&bs[k][tx * 4];
      float const us[4] = {u.x, u.y, u.z, u.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(us[i], vs[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int const r = i0 + ty * 4 + i, c = j0 + tx * 4 + j;
      if (r >= M || c >= N) continue;
      float o = alpha * acc[i][j];
      if (beta != 0.f) o += beta * D[r * ldc + c];
      if (bias) o += bias[c];
      C[r * ldc + c] = o;
    }
}

}  // namespace

namespace vlb {

void products_exact(vlb_ctx* ctx, float* C, long long ldc, int M, int N, int K, Strided a, Strided b, float alpha, float beta, float const* D,
                    float const* bias)
{
  int const tm = ceil_div(M, kTile), tn = ceil_div(N, kTile);
  launch(ctx->stream, products_exact_kernel, dim3((unsigned)((long long)tm * tn)), 256, 0, C, ldc, M, N, K, tm, a, b, alpha, beta, D, bias);
  VLB_LAUNCHED(ctx, 1);
}

}  // namespace vlb
