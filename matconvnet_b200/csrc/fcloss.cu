// A fully connected prediction layer and the softmax loss behind it, in pieces of classes (include/vlb.h has the formulas).
#include "pairs.cuh"
#include "products.cuh"
#include <algorithm>

namespace {

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

// ------------------------------------------------------------------ on pairs of halves (pairs.cu)
struct Part { float top, sum; };

__device__ __forceinline__ Part together(Part a, Part b)
{
  float const top = fmaxf(a.top, b.top), base = isinf(top) ? 0.f : top;      // (as where the parts come from)
  return {top, a.sum * expf(a.top - base) + b.sum * expf(b.top - base)};
}

// kCount parts into one, so that their exponentials do not wait for one another; part(i) is the i-th.
template <int kCount, class F>
__device__ __forceinline__ Part joined(Part p, F part)
{
  Part q[kCount];
  float top = p.top;
#pragma unroll
  for (int i = 0; i < kCount; ++i) { q[i] = part(i); top = fmaxf(top, q[i].top); }
  float const base = isinf(top) ? 0.f : top;
  float sum = p.sum * expf(p.top - base);
#pragma unroll
  for (int i = 0; i < kCount; ++i) sum += q[i].sum * expf(q[i].top - base);
  return {top, sum};
}

// lse of 32 images per block from the parts of their predictions, and the loss by the block that is through last, which adds the blocks' sums in their order.
// lse and labels: of the images first ... first + rows - 1; sums: one per block of 32 images of all `blocks`.  more: pieces of classes are still to come, and the parts
// so far are left as one, the first.
__global__ void __launch_bounds__(1024)
lse_kernel(float* __restrict__ loss, float* __restrict__ lse, float2* parts, int count, bool more, float const* __restrict__ label,
           float const* __restrict__ labels, int rows, int first, int N, int K, double* sums, int blocks, int* ticket, int* status)
{
  vlb::pdl_wait();
  __shared__ Part all[32][33];
  int const tx = threadIdx.x & 31, ty = threadIdx.x >> 5, row = (int)blockIdx.x * 32 + tx;
  Part p = {-INFINITY, 0.f};
  if (row < rows)
    for (int i0 = ty; i0 < count; i0 += 32 * 8)
      p = joined<8>(p, [&](int k) {
        int const i = i0 + 32 * k;
        float2 const v = i < count ? parts[(long long)i * rows + row] : make_float2(-INFINITY, 0.f);
        return Part{v.x, v.y};
      });
  all[ty][tx] = p;
  __syncthreads();
  if (ty) return;
  p = joined<31>(p, [&](int i) { return all[i + 1][tx]; });
  if (more) {
    if (row < rows) parts[row] = make_float2(p.top, p.sum);          // (an image's parts are read by this block alone)
    return;
  }
  double term = 0;
  if (row < rows) {
    Label const l = label_of(labels, row, K, status);
    float v = 0.f;
    if (l.real) { v = p.top + logf(p.sum); term = (double)v - label[row]; }
    if (lse) lse[row] = v;
  }
  for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
  if (!loss) return;
  bool mine = false;
  if (tx == 0) {
    sums[first / 32 + blockIdx.x] = term;
    __threadfence();
    mine = atomicAdd(ticket, 1) == blocks - 1;
    __threadfence();
  }
  if (!__shfl_sync(0xffffffffu, (int)mine, 0)) return;
  double sum = 0;
  for (int i = tx; i < blocks; i += 32) sum += __ldcg(sums + i);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (tx == 0) { *loss = (float)(sum / N); *ticket = 0; }
}

// db[c] (+)= scale * sum of the rows of parts: 32 columns to a block, its warps the rows in turn.
__global__ void __launch_bounds__(kThreads)
db_parts_kernel(float* __restrict__ db, float const* __restrict__ parts, long long ld, int cols, int rows, float scale, bool add)
{
  vlb::pdl_wait();
  __shared__ float all[kThreads / 32][33];
  int const tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int r = ty; r < rows; r += kThreads / 32) s += __ldg(parts + r * ld + c);
  }
  all[ty][tx] = s;
  __syncthreads();
  if (ty || c >= cols) return;
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) s += all[i][tx];
  db[c] = add ? db[c] + s * scale : s * scale;
}

constexpr int kMostImages = 16384;          // images at a time
constexpr int kDzExp = 14;                  // derivatives of the predictions, at most 1 in magnitude, times 2^14
constexpr size_t kMostScratch = 1u << 30;   // what the pieces of classes may take

// The call's scratch, cut up.  withSeen: the log-sum-exp are computed, from parts of what the pieces of classes show (the first: what the pieces before them showed).
struct Plan {
  int images, piece;                        // images at a time, classes at a time
  size_t bytes;
  int *expX, *expF;                         // exponents of X and of the piece of F
  unsigned* partial;
  char *x, *f, *dz, *split;
  float2* parts; float *label, *lse, *db;
  double* sums;

  Plan(int N, int D, int K, bool back, bool withSeen, size_t scratch, char* at = nullptr)
  {
    images = std::min(N, kMostImages);
    // (the parts of many images of few features, 8 bytes for 64 classes, can be more than the pairs: as much again at most)
    size_t const perClass = 4 * (size_t)vlb::pair_ld(D) + (back ? 4 * (size_t)images + (size_t)images / 8 + 64 : 0);
    long long const most = std::max<long long>(256, (long long)(scratch / std::max(perClass, withSeen ? (size_t)images / 8 : 0)) / 256 * 256);
    int const pieces = vlb::ceil_div(K, most);
    piece = (int)std::min<long long>(K, vlb::ceil_div(vlb::ceil_div(K, pieces), 256) * 256ll);
    bytes = 0;
    auto take = [&](size_t n) { char* const p = at + bytes; bytes += (n + 255) / 256 * 256; return p; };
    expX = (int*)take(sizeof(int) * (size_t)vlb::ceil_div(images, 64));
    expF = (int*)take(sizeof(int) * (size_t)vlb::ceil_div(piece, 64));
    partial = (unsigned*)take(sizeof(unsigned) * (vlb::pair_partials(images) + vlb::pair_partials(piece)));
    x = take(vlb::pair_bytes(images, D));
    f = take(vlb::pair_bytes(piece, D));
    split = take(vlb::kPairSplitBytes);
    parts = withSeen ? (float2*)take(sizeof(float2) * (size_t)images * (vlb::pair_parts(piece, 128) + (pieces > 1 ? 1 : 0))) : nullptr;
    label = withSeen ? (float*)take(sizeof(float) * (size_t)images) : nullptr;
    lse = back && withSeen ? (float*)take(sizeof(float) * (size_t)images) : nullptr;
    sums = back ? nullptr : (double*)take(sizeof(double) * (size_t)vlb::ceil_div(N, 32));
    dz = back ? take(vlb::pair_bytes(images, piece)) : nullptr;
    db = back ? (float*)take(sizeof(float) * (size_t)vlb::ceil_div(images, 32) * vlb::pair_ld(piece)) : nullptr;
  }
};

// A plan whose scratch there is: smaller pieces where there is less.
bool plan_for(vlb_ctx* ctx, Plan& plan, int N, int D, int K, bool back, bool withSeen)
{
  for (size_t scratch = kMostScratch; scratch >= (16u << 20); scratch /= 4) {
    plan = Plan(N, D, K, back, withSeen, scratch);
    void* const p = scratch / 4 >= (16u << 20) ? vlb::try_workspace(ctx, plan.bytes) : vlb::workspace(ctx, plan.bytes);
    if (p) { plan = Plan(N, D, K, back, withSeen, scratch, (char*)p); return true; }
  }
  return false;
}

struct Problem {
  vlb_ctx* ctx;
  float const *X, *F, *b, *labels;
  int N, D, K;
};

// The pair of a piece of F, and before the first piece that of the images n0 ....
struct Sides { vlb::Pair x, f; };

Sides sides(Problem const& q, Plan const& plan, int n0, int k0, bool withImages)
{
  int const rows = std::min(plan.images, q.N - n0), cols = std::min(plan.piece, q.K - k0);
  Sides const s = {vlb::pair_at(plan.x, rows, q.D), vlb::pair_at(plan.f, cols, q.D)};
  vlb::PairSource const from[2] = {{s.f, q.F + (size_t)k0 * q.D, plan.expF, nullptr, 0}, {s.x, q.X + (size_t)n0 * q.D, plan.expX, q.labels + n0, q.K}};
  vlb::make_pairs(q.ctx, from, withImages ? 2 : 1, plan.partial);
  return s;
}

vlb::PairProduct predictions(Problem const& q, Plan const& plan, vlb::Pair x, vlb::Pair f, int n0, int k0)
{
  vlb::PairProduct p = {};
  p.a = {x, false, false}; p.b = {f, false, false};
  p.M = x.rows; p.N = f.rows; p.K = q.D;
  p.e.ea.blocks = plan.expX; p.e.eb.blocks = plan.expF;
  p.e.bias = q.b ? q.b + k0 : nullptr;
  p.e.labels = q.labels + n0;
  p.e.firstClass = k0; p.e.classes = q.K;
  return p;
}

// lse of images n0 ... and, after the last of them, the loss (either may be null).  The pairs of the images and of the last piece are left.
int seen(Problem const& q, Plan const& plan, int n0, float* lse, float* loss, int* status)
{
  int const rows = std::min(plan.images, q.N - n0);
  for (int k0 = 0; k0 < q.K; k0 += plan.piece) {
    Sides const s = sides(q, plan, n0, k0, k0 == 0);
    vlb::PairProduct p = predictions(q, plan, s.x, s.f, n0, k0);
    int const before = k0 ? 1 : 0;          // what the pieces before this one have shown
    p.e.parts = plan.parts + (size_t)before * rows; p.e.label = plan.label;
    int const tile = vlb::pair_tile(q.ctx, &p, 1);
    if (int const rc = vlb::products_of_pairs(q.ctx, vlb::kPairSeen, &p, 1, plan.split, tile)) return rc;
    vlb::launch(q.ctx->stream, lse_kernel, (unsigned)vlb::ceil_div(rows, 32), 1024, 0, loss, lse, plan.parts, before + vlb::pair_parts(s.f.rows, tile),
                q.K - k0 > plan.piece, plan.label, q.labels + n0, rows, n0, q.N, q.K, plan.sums, vlb::ceil_div(q.N, 32), q.ctx->deviceStatus + 64 + 4095, status);
    VLB_LAUNCHED(q.ctx, 1);
  }
  return VLB_Success;
}

int forward_on_pairs(Problem const& q, float* loss, float* lse)
{
  Plan plan(1, 1, 1, false, false, 0);
  if (!plan_for(q.ctx, plan, q.N, q.D, q.K, false, true)) return q.ctx->lastError;
  vlb::ProfScope prof(q.ctx, vlb::kProfFc);
  prof.rec.flops = 2.0 * q.N * q.D * q.K;
  for (int n0 = 0; n0 < q.N; n0 += plan.images)
    if (int const rc = seen(q, plan, n0, lse ? lse + n0 : nullptr, loss, q.ctx->deviceStatus)) return rc;
  return vlb::check_launch(q.ctx, "vlb_fc_softmaxloss_forward");
}

int backward_on_pairs(Problem const& q, float* dX, float* dF, float* db, float const* lse, float scale)
{
  Plan plan(1, 1, 1, false, false, 0);
  if (!plan_for(q.ctx, plan, q.N, q.D, q.K, true, !lse)) return q.ctx->lastError;
  vlb::ProfScope prof(q.ctx, vlb::kProfFc);
  prof.rec.flops = 2.0 * q.N * q.D * q.K * ((dX ? 1 : 0) + (dF ? 1 : 0) + (lse ? 1 : 2));
  for (int n0 = 0; n0 < q.N; n0 += plan.images) {
    if (!lse)
      if (int const rc = seen(q, plan, n0, plan.lse, nullptr, nullptr)) return rc;
    for (int k0 = 0; k0 < q.K; k0 += plan.piece) {
      int const cols = std::min(plan.piece, q.K - k0);
      Sides const s = sides(q, plan, n0, k0, lse && k0 == 0);
      vlb::Pair const x = s.x, f = s.f, dz = vlb::pair_at(plan.dz, x.rows, cols);
      vlb::PairProduct p = predictions(q, plan, x, f, n0, k0);
      p.e.lse = lse ? lse + n0 : plan.lse;
      p.e.to = dz; p.e.toExp = kDzExp; p.e.db = db ? plan.db : nullptr;
      p.e.status = q.ctx->deviceStatus;
      if (int const rc = vlb::products_of_pairs(q.ctx, vlb::kPairGrad, &p, 1, plan.split, vlb::pair_tile(q.ctx, &p, 1))) return rc;
      if (db) {
        vlb::launch(q.ctx->stream, db_parts_kernel, (unsigned)vlb::ceil_div(cols, 32), kThreads, 0, db + k0, plan.db, dz.ld, cols,
                    vlb::ceil_div(x.rows, 32), scale, n0 > 0);
        VLB_LAUNCHED(q.ctx, 1);
      }
      // both derivatives in one launch, the longer reduction first
      vlb::PairProduct two[2] = {};
      int count = 0;
      if (dX) {
        vlb::PairProduct& d = two[count++];
        d.a = {dz, false, false}; d.b = {f, true, false};
        d.M = x.rows; d.N = q.D; d.K = cols;
        d.e.eb.blocks = plan.expF;
        d.e.out = dX + (size_t)n0 * q.D; d.e.beta = k0 ? 1.f : 0.f;
      }
      if (dF) {
        vlb::PairProduct& d = two[count++];
        d.a = {dz, true, false}; d.b = {x, true, false};
        d.M = cols; d.N = q.D; d.K = x.rows;
        d.e.eb.blocks = plan.expX;
        d.e.out = dF + (size_t)k0 * q.D; d.e.beta = n0 ? 1.f : 0.f;
      }
      for (int i = 0; i < count; ++i) { two[i].e.ea.value = kDzExp; two[i].e.alpha = scale; two[i].e.ldc = q.D; }
      if (count == 2 && two[1].K > two[0].K) std::swap(two[0], two[1]);
      if (count)
        if (int const rc = vlb::products_of_pairs(q.ctx, vlb::kPairOut, two, count, plan.split, vlb::pair_tile(q.ctx, two, count))) return rc;
    }
  }
  return vlb::check_launch(q.ctx, "vlb_fc_softmaxloss_backward");
}

// ------------------------------------------------------------------ few images: on CUDA cores, bound by reading F
// Up to sixteen images: F is read as it is, once forward and twice backward (and its derivative written); with the images in shared memory a class costs as
// many multiplications as there are images, exact ones, which the cores do in the time that its row takes to arrive.  Microseconds forward / backward, F not in L2, here and on
// pairs:
//   images                          1                    8                    12                   16
//   32000 classes, 1024 features    39/75   132/219      59/139   122/208     84/257   120/208     92/256   122/209
//   81631 classes,  242 features    37/66   108/192      45/129    97/187     66/248    97/187     72/262   108/193
//    1000 classes, 4096 features    21/23    38/63       47/63     38/63      53/82     38/63      (twelve images fill the shared memory)
// Forward sixteen images are the limit of what the sums of a class take in registers; backward the second launch is the slower one from nine images on, and so is all of it where
// few classes of long rows leave most warps idle.  There the products stay exact for the more that they take.
constexpr int kFew = 16;
constexpr int kFewFloats = 49152;             // images that fit shared memory: 192 KB
constexpr int kFewWarps = 16;

bool few_images(int N, long long D) { return N <= kFew && N * D <= kFewFloats; }

struct FewArgs {
  float const *x, *f, *b, *labels, *lse;
  int N, D, K;
  int* status;
  float2* parts; float* label;                // forward: parts[block * N + n]
  float *loss, *lseOut; int* ticket;          // and the results, from the block that is through last
  float *dz, *db; float scale;                // backward: dz[class * kImages + n]
};

// The exponentials are fast ones: off by at most 2 + 1.2 |z - lse| units of the last place, where rounding the difference itself costs |z - lse| / 2.
// Predictions, kRows classes at a time to the warps of all blocks in turn (neighbouring ones to different blocks); forward their largest and sum of exponentials, backward the derivatives.
template <int kImages, int kRows, bool kBack, bool kWide>
__global__ void __launch_bounds__(kFewWarps * 32, 1)
few_predict_kernel(FewArgs a)
{
  vlb::pdl_wait();
  extern __shared__ __align__(16) float xs[];               // [n][D rounded up to a multiple of 128]
  __shared__ float info[2][kFew];                           // label + 1, or 0 for an image that is skipped; lse
  int const lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ld = (a.D + 127) / 128 * 128;
  if (threadIdx.x < a.N) {
    Label const l = label_of(a.labels, threadIdx.x, a.K, blockIdx.x == 0 ? a.status : nullptr);
    info[0][threadIdx.x] = l.real ? (float)(l.at + 1) : 0.f;
    info[1][threadIdx.x] = kBack ? a.lse[threadIdx.x] : 0.f;
  }
  __syncthreads();
  for (int n = 0; n < a.N; ++n) {
    bool const real = info[0][n] > 0.f;                     // (what a skipped image holds is not looked at)
    for (int d = threadIdx.x; d < ld; d += kFewWarps * 32) xs[n * ld + d] = real && d < a.D ? a.x[(size_t)n * a.D + d] : 0.f;
  }
  __syncthreads();
  int const n = lane % kImages, k1 = a.K;
  int const at = n < a.N ? (int)info[0][n] - 1 : -1;        // the label's class, -1: skipped
  float const lse = n < a.N ? info[1][n] : 0.f;
  float top = -INFINITY, sum = 0.f;
  for (int k = (warp * (int)gridDim.x + (int)blockIdx.x) * kRows; k < k1; k += kFewWarps * (int)gridDim.x * kRows) {
    float acc[kRows * kImages] = {};
    float const* f[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) f[r] = a.f + (size_t)min(k + r, k1 - 1) * a.D;
#pragma unroll 4
    for (int d = kWide ? 4 * lane : lane; d < ld; d += 128) {      // four neighbouring columns, or four 32 apart
      float4 w[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (kWide) {
          w[r] = d < a.D ? __ldg((float4 const*)(f[r] + d)) : make_float4(0, 0, 0, 0);
        } else {
          w[r].x = d < a.D ? __ldg(f[r] + d) : 0.f; w[r].y = d + 32 < a.D ? __ldg(f[r] + d + 32) : 0.f;
          w[r].z = d + 64 < a.D ? __ldg(f[r] + d + 64) : 0.f; w[r].w = d + 96 < a.D ? __ldg(f[r] + d + 96) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < kImages; ++i) {
        if (kImages > 1 && i >= a.N) break;
        float const* const xi = xs + i * ld + d;
        float4 const q = kWide ? *(float4 const*)xi : make_float4(xi[0], xi[32], xi[64], xi[96]);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          acc[r * kImages + i] = fmaf(w[r].x, q.x, fmaf(w[r].y, q.y, fmaf(w[r].z, q.z, fmaf(w[r].w, q.w, acc[r * kImages + i]))));
      }
    }
    // lane l: class k + l / kImages % kRows of image l % kImages
    constexpr int kCount = kRows * kImages;
#pragma unroll
    for (int s = kCount / 2; s > 0; s >>= 1) {
      bool const up = lane & s;
#pragma unroll
      for (int i = 0; i < s; ++i) {
        float const send = up ? acc[i] : acc[i + s], keep = up ? acc[i + s] : acc[i];
        acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, s);
      }
    }
#pragma unroll
    for (int s = kCount; s < 32; s <<= 1) acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], s);
    int const c = k + lane / kImages % kRows;
    bool const mine = c < k1 && n < a.N && lane < kCount;
    float const z = acc[0] + (a.b && c < k1 ? __ldg(a.b + c) : 0.f);
    if (!kBack) {
      if (mine) {
        float const t = fmaxf(top, z), base = isinf(t) ? 0.f : t;
        sum = sum * __expf(top - base) + __expf(z - base);
        top = t;
        if (c == at) a.label[n] = z;
      }
    } else {
      float v = mine && at >= 0 ? (__expf(z - lse) - (c == at ? 1.f : 0.f)) * a.scale : 0.f;
      if (c < k1 && lane < kCount) a.dz[(size_t)c * kImages + n] = v;
      if (a.db) {
#pragma unroll
        for (int s = 1; s < kImages; s <<= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
        if (n == 0 && c < k1 && lane < kCount) a.db[c] = v;
      }
    }
  }
  if (kBack) return;
  // lanes of one image, then the block's warps
  Part p = {top, sum};
#pragma unroll
  for (int s = kImages; s < 32; s <<= 1) {
    Part const q = {__shfl_xor_sync(0xffffffffu, p.top, s), __shfl_xor_sync(0xffffffffu, p.sum, s)};
    p = lane & s ? together(q, p) : together(p, q);          // (in the lanes' order, so that all of them hold the same)
  }
  __shared__ Part all[kFewWarps][kFew];
  if (lane < kImages) all[warp][lane] = p;
  __syncthreads();
  __shared__ bool last;
  __shared__ double term[kFew];
  if (threadIdx.x < 32) {
    if (lane < a.N) {
      p = all[0][lane];
      for (int w = 1; w < kFewWarps; ++w) p = together(p, all[w][lane]);
      __stcg(a.parts + blockIdx.x * a.N + lane, make_float2(p.top, p.sum));
    }
    __threadfence();
    __syncwarp();
    if (lane == 0) last = atomicAdd(a.ticket, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (warp < a.N) {
    p = {-INFINITY, 0.f};
    for (int i = lane; i < (int)gridDim.x; i += 32) { float2 const q = __ldcg(a.parts + i * a.N + warp); p = together(p, {q.x, q.y}); }
    for (int s = 1; s < 32; s <<= 1) {
      Part const q = {__shfl_xor_sync(0xffffffffu, p.top, s), __shfl_xor_sync(0xffffffffu, p.sum, s)};
      p = lane & s ? together(q, p) : together(p, q);
    }
    if (lane == 0) {
      bool const real = info[0][warp] > 0.f;
      float const v = real ? p.top + logf(p.sum) : 0.f;
      term[warp] = real ? (double)v - __ldcg(a.label + warp) : 0.;
      if (a.lseOut) a.lseOut[warp] = v;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0;
    for (int i = 0; i < a.N; ++i) sum += term[i];
    if (a.loss) *a.loss = (float)(sum / a.N);
    *a.ticket = 0;
  }
}

// dF of the block's classes, and the block's part of dX: parts[block][n][D].  A thread has four neighbouring columns (kWide) or four kFewThreads apart.
constexpr int kFewThreads = 128;

template <int kImages, bool kWide>
__global__ void __launch_bounds__(kFewThreads, kImages <= 4 ? 8 : 2)
few_derivatives_kernel(float* __restrict__ dF, float* __restrict__ parts, float const* __restrict__ x, float const* __restrict__ f, float const* __restrict__ dz,
                       float const* __restrict__ labels, int N, int D, int K, int perBlock)
{
  vlb::pdl_wait();
  int const c0 = (int)blockIdx.y * 4 * kFewThreads + (kWide ? 4 : 1) * (int)threadIdx.x, k0 = (int)blockIdx.x * perBlock, k1 = min(k0 + perBlock, K);
  auto col = [&](int i) { return kWide ? c0 + i : c0 + kFewThreads * i; };
  float xv[kImages][4] = {}, acc[kImages][4] = {};
#pragma unroll
  for (int n = 0; n < kImages; ++n)
    if (n < N && label_of(labels, n, K, nullptr).real)
#pragma unroll
      for (int i = 0; i < 4; ++i) if (col(i) < D) xv[n][i] = __ldg(x + (size_t)n * D + col(i));
  // rows of F are asked for kAhead classes before they are used
  constexpr int kAhead = 4;
  float w[kAhead][4] = {};
  auto fetch = [&](float (&v)[4], int k) {
    if (!parts || k >= k1) return;
    float const* const p = f + (size_t)k * D;
    if (kWide) {
      float4 const q = col(0) < D ? __ldg((float4 const*)(p + col(0))) : make_float4(0, 0, 0, 0);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = col(i) < D ? __ldg(p + col(i)) : 0.f;
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) fetch(w[u], k0 + u);
  for (int kb = k0; kb < k1; kb += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      int const k = kb + u;
      if (k >= k1) break;
      float o[4] = {}, g[kImages];
      if (kImages >= 4) {
#pragma unroll
        for (int n = 0; n < kImages / 4; ++n) {
          float4 const q = __ldg((float4 const*)(dz + (size_t)k * kImages) + n);
          g[4 * n % kImages] = q.x; g[(4 * n + 1) % kImages] = q.y; g[(4 * n + 2) % kImages] = q.z; g[(4 * n + 3) % kImages] = q.w;
        }
      } else {
#pragma unroll
        for (int n = 0; n < kImages; ++n) g[n] = __ldg(dz + (size_t)k * kImages + n);
      }
#pragma unroll
      for (int n = 0; n < kImages; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) { acc[n][i] = fmaf(g[n], w[u][i], acc[n][i]); o[i] = fmaf(g[n], xv[n][i], o[i]); }
      fetch(w[u], k + kAhead);
      if (dF) {
        if (kWide) {
          if (col(0) < D) *(float4*)(dF + (size_t)k * D + col(0)) = make_float4(o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) if (col(i) < D) dF[(size_t)k * D + col(i)] = o[i];
        }
      }
    }
  }
  if (!parts) return;
#pragma unroll
  for (int n = 0; n < kImages; ++n)
    if (n < N)
#pragma unroll
      for (int i = 0; i < 4; ++i) if (col(i) < D) parts[((size_t)blockIdx.x * N + n) * D + col(i)] = acc[n][i];
}

// dX = the sum of the blocks' parts, in order: 32 elements to a block.
__global__ void __launch_bounds__(1024)
few_sum_kernel(float* __restrict__ dX, float const* __restrict__ parts, int count, int n)
{
  vlb::pdl_wait();
  __shared__ float all[32][33];
  int const tx = threadIdx.x & 31, ty = threadIdx.x >> 5, at = (int)blockIdx.x * 32 + tx;
  float s = 0.f;
  if (at < n) {
#pragma unroll 4
    for (int i = ty; i < count; i += 32) s += __ldg(parts + (size_t)i * n + at);
  }
  all[ty][tx] = s;
  __syncthreads();
  if (ty) return;
  for (int i = 1; i < 32; ++i) s += all[i][tx];
  if (at < n) dX[at] = s;
}

// f(images, rows): the smallest number of images, a power of two, that holds N, and the classes that a warp takes at a time.
template <class F>
void with_images(int N, F f)
{
  using std::integral_constant;
  if (N == 1)      f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (N == 2) f(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  else if (N <= 4) f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (N <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
  else             f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
}

bool aligned(int D, void const* f) { return D % 4 == 0 && ((uintptr_t)f & 15) == 0; }

template <bool kBack>
int few_predict(Problem const& q, FewArgs a, int& blocks)
{
  int rc = VLB_Success;
  with_images(q.N, [&](auto images, auto rows) {
    constexpr int kImages = decltype(images)::value, kRows = decltype(rows)::value;
    blocks = std::min(q.ctx->smCount, vlb::ceil_div(q.K, kRows));
    auto const kernel = aligned(q.D, q.F) ? few_predict_kernel<kImages, kRows, kBack, true> : few_predict_kernel<kImages, kRows, kBack, false>;
    size_t const smem = sizeof(float) * (size_t)q.N * vlb::ceil_div(q.D, 128) * 128;
    static bool ready[64][2];
    bool& r = ready[q.ctx->device & 63][aligned(q.D, q.F)];
    if (smem > 32 * 1024 && !r) {
      cudaError_t const e = vlb::allow_max_dynamic_smem(kernel);
      if (e != cudaSuccess) { rc = vlb::set_error(q.ctx, VLB_Cuda, cudaGetErrorString(e)); return; }
      r = true;
    }
    vlb::launch(q.ctx->stream, kernel, (unsigned)blocks, kFewWarps * 32, smem, a);
    VLB_LAUNCHED(q.ctx, 1);
  });
  return rc;
}

FewArgs few_args(Problem const& q)
{
  FewArgs a = {};
  a.x = q.X; a.f = q.F; a.b = q.b; a.labels = q.labels;
  a.N = q.N; a.D = q.D; a.K = q.K;
  return a;
}

// lse and loss (either may be null); scratch: few_scratch(q) bytes.
size_t few_scratch(Problem const& q) { return (sizeof(float2) * q.ctx->smCount + sizeof(float)) * kFew; }

int few_seen(Problem const& q, float* loss, float* lse, char* scratch, int* status)
{
  FewArgs a = few_args(q);
  a.parts = (float2*)scratch;
  a.label = (float*)(a.parts + (size_t)q.ctx->smCount * kFew);
  a.loss = loss; a.lseOut = lse; a.ticket = q.ctx->deviceStatus + 64 + 4095; a.status = status;
  int blocks = 0;
  return few_predict<false>(q, a, blocks);
}

int forward_few(Problem const& q, float* loss, float* lse)
{
  char* const scratch = (char*)vlb::workspace(q.ctx, few_scratch(q));
  if (!scratch) return q.ctx->lastError;
  if (int const rc = few_seen(q, loss, lse, scratch, q.ctx->deviceStatus)) return rc;
  return vlb::check_launch(q.ctx, "vlb_fc_softmaxloss_forward");
}

int backward_few(Problem const& q, float* dX, float* dF, float* db, float const* lse, float scale)
{
  // eight blocks per SM, as far as the parts of dX stay within 16 MB (81631 x 242, three images: 116 us with four per SM, 81 with eight and rows asked for ahead)
  int const columns = vlb::ceil_div(q.D, 4 * kFewThreads);
  int const most = dX ? (int)std::max<long long>(q.ctx->smCount, (4 << 20) / ((long long)q.N * q.D)) : INT32_MAX;
  int const chunks = std::min(std::min(q.K, most), std::max(1, 8 * q.ctx->smCount / columns)), per = vlb::ceil_div(q.K, chunks);
  int const count = vlb::ceil_div(q.K, per);
  size_t const seen = (few_scratch(q) + 255) / 256 * 256, dzBytes = (sizeof(float) * (size_t)q.K * kFew + 255) / 256 * 256;
  char* const scratch = (char*)vlb::workspace(q.ctx, seen + 256 + dzBytes + (dX ? sizeof(float) * (size_t)count * q.N * q.D : 0));
  if (!scratch) return q.ctx->lastError;
  float *const own = (float*)(scratch + seen), *const dz = (float*)(scratch + seen + 256), *const parts = dX ? (float*)(scratch + seen + 256 + dzBytes) : nullptr;
  if (!lse)
    if (int const rc = few_seen(q, nullptr, own, scratch, nullptr)) return rc;
  FewArgs a = few_args(q);
  a.lse = lse ? lse : own; a.dz = dz; a.db = db; a.scale = scale; a.status = q.ctx->deviceStatus;
  int blocks = 0;
  if (int const rc = few_predict<true>(q, a, blocks)) return rc;
  if (dX || dF)
    with_images(q.N, [&](auto images, auto) {
      constexpr int kImages = decltype(images)::value;
      bool const wide = aligned(q.D, q.F) && (!dF || aligned(q.D, dF));
      vlb::launch(q.ctx->stream, wide ? few_derivatives_kernel<kImages, true> : few_derivatives_kernel<kImages, false>, dim3((unsigned)count, (unsigned)columns),
                  kFewThreads, 0, dF, parts, q.X, q.F, dz, q.labels, q.N, q.D, q.K, per);
      VLB_LAUNCHED(q.ctx, 1);
    });
  if (dX) {
    vlb::launch(q.ctx->stream, few_sum_kernel, (unsigned)vlb::ceil_div((long long)q.N * q.D, 32), 1024, 0, dX, parts, count, q.N * q.D);
    VLB_LAUNCHED(q.ctx, 1);
  }
  return vlb::check_launch(q.ctx, "vlb_fc_softmaxloss_backward");
}

// Classes per piece: predictions of a piece up to 64 MB.
int piece_of(int N, int K) { return (int)std::min<long long>(K, std::max<long long>(64, (16ll << 20) / N / 64 * 64)); }

// Images, classes and features are walked through with 32-bit counters, in strides of up to kStride.
bool good_shape(int H, int W, int C, int N, int K)
{
  constexpr int kStride = 1 << 20;
  return H > 0 && W > 0 && C > 0 && N > 0 && K > 0 && (long long)H * W <= INT32_MAX && (long long)H * W * C <= INT32_MAX - kStride && N <= INT32_MAX - kStride && K <= INT32_MAX - kStride;
}

}  // namespace

extern "C" {

int vlb_fc_softmaxloss_forward(vlb_ctx* ctx, float* loss, float* lse, float const* X, float const* F, float const* b, float const* labels,
                               int H, int W, int C, int N, int K)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, good_shape(H, W, C, N, K), "fc_softmaxloss_forward: bad shape");
  VLB_REQUIRE(ctx, loss && X && F && labels, "fc_softmaxloss_forward: null tensor");
  VLB_REQUIRE(ctx, vlb::on_its_device(ctx), "fc_softmaxloss_forward: the context belongs to another device than the current one");
  int const D = H * W * C;
  if (few_images(N, D)) return vlb::pass_error(ctx, forward_few({ctx, X, F, b, labels, N, D, K}, loss, lse), "vlb_fc_softmaxloss_forward");
  if (ctx->precision != VLB_PRECISION_FP32)
    return vlb::pass_error(ctx, forward_on_pairs({ctx, X, F, b, labels, N, D, K}, loss, lse), "vlb_fc_softmaxloss_forward");
  int const piece = piece_of(N, K);
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
  VLB_REQUIRE(ctx, good_shape(H, W, C, N, K), "fc_softmaxloss_backward: bad shape");
  VLB_REQUIRE(ctx, X && F && labels, "fc_softmaxloss_backward: null tensor");
  VLB_REQUIRE(ctx, vlb::on_its_device(ctx), "fc_softmaxloss_backward: the context belongs to another device than the current one");
  int const D = H * W * C;
  if (few_images(N, D))
    return vlb::pass_error(ctx, backward_few({ctx, X, F, b, labels, N, D, K}, dX, dF, db, lse, (float)(dzdy / N)), "vlb_fc_softmaxloss_backward");
  if (ctx->precision != VLB_PRECISION_FP32)
    return vlb::pass_error(ctx, backward_on_pairs({ctx, X, F, b, labels, N, D, K}, dX, dF, db, lse, (float)(dzdy / N)), "vlb_fc_softmaxloss_backward");
  int const piece = piece_of(N, K);
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
