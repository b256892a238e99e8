// Matrix products of the operators that work on matrices (fcloss.cu, muon.cu).
#pragma once
#include "common.cuh"

namespace vlb {

// Element (row i, reduction index k) of an operand: p[i * rs + k * ks].
struct Strided { float const* p; long long rs, ks; };

// C[i * ldc + j] = alpha * sum_k A(i, k) * B(j, k) + beta * D[i * ldc + j] + bias[j] on CUDA cores, every product exact and every sum in single
// precision.  D may be C; D (with beta 0) and bias may be NULL.
void products_exact(vlb_ctx* ctx, float* C, long long ldc, int M, int N, int K, Strided a, Strided b, float alpha, float beta, float const* D,
                    float const* bias);

}  // namespace vlb
