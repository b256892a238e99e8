// The Muon solver (include/vlb.h has the formulas).
#include "muon_small.cuh"
#include "pairs.cuh"
#include "products.cuh"
#include <math.h>
#include <algorithm>
#include <vector>

namespace {

constexpr int kThreads = 256, kMaxParts = 592;

constexpr int kMost = vlb::kMaxPairProducts;          // parameters in one pass

// One parameter's share of a launch over several: blocks block0 ... block0 + blocks - 1.
struct Job {
  float *w, *s1; float const* g; float* u;
  size_t n;
  float decay, rate;
  double* parts;                     // sums of squares, one per block of momentum_kernel
  int partCount, block0, blocks, vec;
  vlb::Pair x;
  int rowsPer; vlb::FastDiv31 perRow;  // make_x_kernel: rows of a block, sixteen columns at a time (by groups of columns, of which there are up to 2^27)
};
struct Jobs { Job j[kMost]; int count; };

__device__ __forceinline__ Job const& job_of(Jobs const& jobs, int& block)
{
  int i = 0;
  while (i + 1 < jobs.count && block >= jobs.j[i + 1].block0) ++i;
  block -= jobs.j[i].block0;
  return jobs.j[i];
}

__device__ __forceinline__ double block_sum(double sum)
{
  __shared__ double all[kThreads / 32];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = all[0];
  for (int i = 1; i < kThreads / 32; ++i) sum += all[i];
  return sum;
}

// Momentum; u = what is to be orthogonalised; a part of the sum of its squares per block, in double precision.
__global__ void __launch_bounds__(kThreads)
momentum_kernel(const __grid_constant__ Jobs jobs, float gradMult, float momentum, int nesterov)
{
  vlb::pdl_wait();
  int block = blockIdx.x;
  Job const& j = job_of(jobs, block);
  double sum = 0;
  auto one = [&](float w, float& m, float g) {
    float const d = gradMult * g + j.decay * w;
    m = momentum * m + d;
    float const v = nesterov ? d + momentum * m : m;
    sum += (double)v * v;
    return v;
  };
  size_t const step = (size_t)j.blocks * kThreads;
  if (j.vec) {
    for (size_t i = (size_t)block * kThreads + threadIdx.x; i < j.n / 4; i += step) {
      float4 const w = ((float4 const*)j.w)[i], g = ((float4 const*)j.g)[i];
      float4 m = ((float4 const*)j.s1)[i], v;
      v.x = one(w.x, m.x, g.x); v.y = one(w.y, m.y, g.y); v.z = one(w.z, m.z, g.z); v.w = one(w.w, m.w, g.w);
      ((float4*)j.s1)[i] = m;
      ((float4*)j.u)[i] = v;
    }
  } else {
    for (size_t i = (size_t)block * kThreads + threadIdx.x; i < j.n; i += step) {
      float m = j.s1[i];
      j.u[i] = one(j.w[i], m, j.g[i]);
      j.s1[i] = m;
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) j.parts[block] = sum;
}

__device__ __forceinline__ float norm_factor(Job const& j, double epsilon)
{
  double sum = 0;
  for (int i = threadIdx.x; i < j.partCount; i += kThreads) sum += j.parts[i];
  return (float)(1. / (sqrt(block_sum(sum)) + epsilon));
}

// u / (|u| + epsilon), as a pair scaled by 2^e
__global__ void __launch_bounds__(kThreads)
make_x_kernel(const __grid_constant__ Jobs jobs, double epsilon, int e)
{
  vlb::pdl_wait();
  int block = blockIdx.x;
  Job const& j = job_of(jobs, block);
  float const norm = norm_factor(j, epsilon), f = vlb::pow2(e);
  int const groups = (int)(j.x.ld / 16);
  for (int t = threadIdx.x; t < j.rowsPer * groups; t += kThreads) {
    int const r = j.perRow(t), c = (t - r * groups) * 16;
    long long const row = (long long)block * j.rowsPer + r;
    if (row >= j.x.rows) break;
    float const* const p = j.u + row * j.x.cols + c;
    float v[16];
    if (j.x.cols % 4 == 0 && c + 16 <= j.x.cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float4 const q = __ldg((float4 const*)p + i);
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = c + i < j.x.cols ? __ldg(p + i) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = v[i] * norm * f;
    vlb::store_pair16(j.x, row, c, v);
  }
}

// u / (|u| + epsilon) in place
__global__ void __launch_bounds__(kThreads)
normalise_kernel(const __grid_constant__ Jobs jobs, double epsilon)
{
  vlb::pdl_wait();
  int block = blockIdx.x;
  Job const& j = job_of(jobs, block);
  float const f = norm_factor(j, epsilon);
  for (size_t i = (size_t)block * kThreads + threadIdx.x; i < j.n; i += (size_t)j.blocks * kThreads) j.u[i] *= f;
}

// w -= rate * x
__global__ void __launch_bounds__(kThreads)
subtract_kernel(float* __restrict__ w, float const* __restrict__ x, size_t n, float rate)
{
  vlb::pdl_wait();
  for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < n; i += (size_t)gridDim.x * kThreads) w[i] -= rate * x[i];
}

// Without a Newton-Schulz step.
__global__ void __launch_bounds__(kThreads)
step_kernel(const __grid_constant__ Jobs jobs, double epsilon)
{
  vlb::pdl_wait();
  int block = blockIdx.x;
  Job const& j = job_of(jobs, block);
  float const f = norm_factor(j, epsilon);
  for (size_t i = (size_t)block * kThreads + threadIdx.x; i < j.n; i += (size_t)j.blocks * kThreads) j.w[i] -= j.rate * (j.u[i] * f);
}

// The largest magnitude of a polynomial over [0, s], with 2% for what lies between the samples.
template <class F>
double most(F f, double s)
{
  double m = 0;
  for (int i = 0; i <= 1024; ++i) m = std::max(m, fabs(f(s * i / 1024)));
  return 1.02 * m;
}

// The exponent that keeps magnitudes up to m below 2^15.
int exp_below_half(double m)
{
  if (!(m < 1e30)) return -100;
  return m < 1e-25 ? 97 : 14 - (int)ceil(log2(m));
}

// The exponents of the halves through the steps: every element of a matrix is at most its largest singular value, which the polynomials bound.
struct Exponents {
  std::vector<int> x, gram, poly;
  explicit Exponents(vlb_muon_opts const& o)
  {
    double s = 1;
    x.push_back(exp_below_half(s));
    for (int k = 0; k < o.steps; ++k) {
      double const s2 = s * s;
      gram.push_back(exp_below_half(s2));
      poly.push_back(exp_below_half(most([&](double t) { return t * (o.b + t * o.c); }, s2)));
      s = most([&](double t) { return t * (o.a + t * t * (o.b + t * t * o.c)); }, s);
      x.push_back(exp_below_half(s));
    }
  }
};

// What momentum_kernel and those that share its blocks need; u and parts are set.  Returns the number of blocks.
int set_up(Jobs& jobs, int count, vlb_muon_param const* u)
{
  jobs.count = count;
  int blocks = 0;
  for (int i = 0; i < count; ++i) {
    Job& j = jobs.j[i];
    j.w = u[i].W; j.s1 = u[i].S1; j.g = u[i].G;
    j.n = (size_t)u[i].rows * u[i].cols;
    j.decay = (float)u[i].decay;
    j.rate = (float)(u[i].lr * sqrt(std::max(1., (double)u[i].rows / u[i].cols)));
    j.vec = j.n % 4 == 0 && (((uintptr_t)j.w | (uintptr_t)j.s1 | (uintptr_t)j.g) & 15) == 0;
    j.block0 = blocks;
    j.blocks = j.partCount = (int)vlb::grid_for((j.n + 3) / 4, kThreads, kMaxParts);
    blocks += j.blocks;
  }
  return blocks;
}

// The scratch of a pass, cut up from `at` on.
struct Layout {
  size_t bytes = 0;
  bool small = true;                 // all are: all steps in one launch.  (Beside larger ones they cost next to nothing in the launches that those need.)
  char* split;
  Jobs jobs = {};
  vlb::Pair x[2][kMost], a[kMost], q[kMost];

  Layout(int count, vlb_muon_param const* u, int steps, char* at)
  {
    auto take = [&](size_t n) { char* const p = at + bytes; bytes += (n + 255) / 256 * 256; return p; };
    for (int i = 0; i < count; ++i) small = small && vlb::small_fits(u[i].rows, u[i].cols, steps);
    split = take(small ? 0 : vlb::kPairSplitBytes);
    for (int i = 0; i < count; ++i) {
      int const rows = u[i].rows, cols = u[i].cols, m = std::min(rows, cols);
      jobs.j[i].u = (float*)take(sizeof(float) * (size_t)rows * cols);
      jobs.j[i].parts = (double*)take(sizeof(double) * kMaxParts);
      if (small) continue;
      x[0][i] = vlb::pair_at(take(vlb::pair_bytes(rows, cols)), rows, cols);
      x[1][i] = vlb::pair_at(take(vlb::pair_bytes(rows, cols)), rows, cols);
      a[i] = vlb::pair_at(take(vlb::pair_bytes(m, m)), m, m);
      q[i] = vlb::pair_at(take(vlb::pair_bytes(m, m)), m, m);
    }
  }
};

int update_on_pairs(vlb_ctx* ctx, int count, vlb_muon_param const* u, double gradMult, vlb_muon_opts const* o)
{
  char* const at = (char*)vlb::workspace(ctx, Layout(count, u, o->steps, nullptr).bytes);
  if (!at) return ctx->lastError;
  Layout l(count, u, o->steps, at);
  bool const small = l.small;
  char* const split = l.split;
  Jobs& jobs = l.jobs;
  auto const &x = l.x;
  auto const &a = l.a, &q = l.q;
  int blocks = set_up(jobs, count, u);
  vlb::launch(ctx->stream, momentum_kernel, (unsigned)blocks, kThreads, 0, jobs, (float)gradMult, (float)o->momentum, o->nesterov);
  VLB_LAUNCHED(ctx, 1);
  if (o->steps == 0) {
    vlb::launch(ctx->stream, step_kernel, (unsigned)blocks, kThreads, 0, jobs, o->epsilon);
    VLB_LAUNCHED(ctx, 1);
    return VLB_Success;
  }
  Exponents const e(*o);
  if (small) {
    vlb::SmallMatrix m[kMost];
    vlb::SmallSteps steps = {};
    steps.count = o->steps; steps.epsilon = o->epsilon;
    steps.a = (float)o->a; steps.b = (float)o->b; steps.c = (float)o->c;
    std::copy(e.x.begin(), e.x.end(), steps.x); std::copy(e.gram.begin(), e.gram.end(), steps.gram); std::copy(e.poly.begin(), e.poly.end(), steps.poly);
    for (int i = 0; i < count; ++i) m[i] = {u[i].W, jobs.j[i].u, jobs.j[i].parts, jobs.j[i].partCount, u[i].rows, u[i].cols, jobs.j[i].rate};
    return vlb::small_matrices(ctx, m, count, steps);
  }
  blocks = 0;
  for (int i = 0; i < count; ++i) {
    Job& j = jobs.j[i];
    j.x = x[0][i];
    int const groups = (int)(j.x.ld / 16);
    j.rowsPer = std::max(1, 512 / groups);
    j.perRow = vlb::FastDiv31(groups);
    j.block0 = blocks;
    j.blocks = vlb::ceil_div(j.x.rows, j.rowsPer);
    blocks += j.blocks;
  }
  vlb::launch(ctx->stream, make_x_kernel, (unsigned)blocks, kThreads, 0, jobs, o->epsilon, e.x[0]);
  VLB_LAUNCHED(ctx, 1);
  vlb::PairProduct step[3 * kMost];
  vlb::PairProduct *const gram = step, *const poly = step + count, *const next = step + 2 * count;
  for (int k = 0; k < o->steps; ++k) {
    int const ex = e.x[k], ea = e.gram[k], eq = e.poly[k];
    for (int i = 0; i < count; ++i) {
      int const rows = u[i].rows, cols = u[i].cols, m = std::min(rows, cols);
      bool const tall = rows > cols;
      vlb::Pair const& xi = x[k & 1][i];
      vlb::PairProduct &g = gram[i] = {}, &p = poly[i] = {}, &n = next[i] = {};
      g.a = g.b = {xi, tall, false};
      g.M = g.N = m; g.K = std::max(rows, cols);
      g.symmetric = true;
      g.e.ea.value = g.e.eb.value = ex; g.e.alpha = 1.f; g.e.to = a[i]; g.e.toExp = ea;
      p.a = p.b = {a[i], false, true};
      p.M = p.N = p.K = m;
      p.symmetric = true;
      p.e.ea.value = p.e.eb.value = ea; p.e.alpha = (float)o->c; p.e.beta = (float)o->b; p.e.add = a[i]; p.e.addExp = ea; p.e.to = q[i]; p.e.toExp = eq;
      n.a = tall ? vlb::PairSide{xi, false, false} : vlb::PairSide{q[i], false, true};
      n.b = tall ? vlb::PairSide{q[i], false, true} : vlb::PairSide{xi, true, false};
      n.M = rows; n.N = cols; n.K = m;
      n.e.ea.value = tall ? ex : eq; n.e.eb.value = tall ? eq : ex;
      n.e.alpha = 1.f; n.e.beta = (float)o->a; n.e.add = xi; n.e.addExp = ex;
      if (k + 1 < o->steps) { n.e.to = x[(k + 1) & 1][i]; n.e.toExp = e.x[k + 1]; }
      else                  { n.e.out = u[i].W; n.e.ldc = cols; n.e.rate = jobs.j[i].rate; }
    }
    int const tile = vlb::pair_tile(ctx, step, 3 * count);          // (one for all: what one product leaves of a symmetric matrix the next one reads)
    for (int set = 0; set < 3; ++set)
      if (int const rc = vlb::products_of_pairs(ctx, vlb::kPairPoly, step + set * count, count, split, tile)) return rc;
  }
  return VLB_Success;
}

size_t exact_bytes(vlb_muon_param const& u)
{
  size_t const n = (size_t)u.rows * u.cols, m = std::min(u.rows, u.cols);
  return sizeof(double) * kMaxParts + sizeof(float) * (2 * n + 2 * m * m);
}

// VLB_PRECISION_FP32: products on CUDA cores, one parameter after the other.
int update_exact(vlb_ctx* ctx, vlb_muon_param const& u, double gradMult, vlb_muon_opts const* o)
{
  int const rows = u.rows, cols = u.cols, m = std::min(rows, cols);
  size_t const n = (size_t)rows * cols;
  Jobs jobs = {};
  jobs.j[0].parts = (double*)vlb::workspace(ctx, exact_bytes(u));
  if (!jobs.j[0].parts) return ctx->lastError;
  float *x = jobs.j[0].u = (float*)(jobs.j[0].parts + kMaxParts), *next = x + n, *const a = next + n, *const q = a + (size_t)m * m;
  unsigned const blocks = (unsigned)set_up(jobs, 1, &u);
  vlb::launch(ctx->stream, momentum_kernel, blocks, kThreads, 0, jobs, (float)gradMult, (float)o->momentum, o->nesterov);
  vlb::launch(ctx->stream, normalise_kernel, blocks, kThreads, 0, jobs, o->epsilon);
  for (int k = 0; k < o->steps; ++k) {
    vlb::Strided const byRow = {x, cols, 1}, byCol = {x, 1, cols};
    if (rows <= cols) vlb::products_exact(ctx, a, m, m, m, cols, byRow, byRow, 1.f, 0.f, nullptr, nullptr);
    else              vlb::products_exact(ctx, a, m, m, m, rows, byCol, byCol, 1.f, 0.f, nullptr, nullptr);
    vlb::products_exact(ctx, q, m, m, m, m, {a, m, 1}, {a, m, 1}, (float)o->c, (float)o->b, a, nullptr);
    if (rows <= cols) vlb::products_exact(ctx, next, cols, rows, cols, rows, {q, m, 1}, byCol, 1.f, (float)o->a, x, nullptr);
    else              vlb::products_exact(ctx, next, cols, rows, cols, cols, byRow, {q, m, 1}, 1.f, (float)o->a, x, nullptr);
    std::swap(x, next);
  }
  vlb::launch(ctx->stream, subtract_kernel, blocks, kThreads, 0, u.W, x, n, jobs.j[0].rate);
  VLB_LAUNCHED(ctx, 3);
  return VLB_Success;
}

bool overlap(void const* p, size_t n, void const* q, size_t m) { return (char const*)p < (char const*)q + m && (char const*)q < (char const*)p + n; }

// Whether what one of them writes is anything of the other's.
bool overlap(vlb_muon_param const& a, vlb_muon_param const& b)
{
  size_t const n = sizeof(float) * (size_t)a.rows * a.cols, m = sizeof(float) * (size_t)b.rows * b.cols;
  for (void const* p : {(void const*)a.W, (void const*)a.S1})
    for (void const* q : {(void const*)b.W, (void const*)b.S1, (void const*)b.G})
      if (overlap(p, n, q, m)) return true;
  return overlap(b.W, m, a.G, n) || overlap(b.S1, m, a.G, n);
}

// Items first ... end - 1 go through all steps together: as many as fit a pass, each of them apart from those in front of it.
int end_of_pass(int first, int count, vlb_muon_param const* u, bool exact)
{
  int end = first + 1;
  for (; end < count && end - first < (exact ? 1 : kMost); ++end)
    for (int i = first; i < end; ++i)
      if (overlap(u[i], u[end])) return end;
  return end;
}

}  // namespace

extern "C" {

int vlb_muon_update_many(vlb_ctx* ctx, int count, vlb_muon_param const* u, double gradMult, vlb_muon_opts const* o)
{
  if (!ctx) return VLB_IllegalArgument;
  VLB_REQUIRE(ctx, count >= 0 && (u || count == 0) && o, "muon_update_many: null argument");
  VLB_REQUIRE(ctx, o->steps >= 0 && o->epsilon >= 0, "muon_update_many: steps and epsilon must not be negative");
  VLB_REQUIRE(ctx, o->steps < 65536, "muon_update_many: fewer than 65536 steps expected");       // (their exponents are computed before the first one)
  for (int i = 0; i < count; ++i) {
    // (32-bit counters, in strides below a million)
    VLB_REQUIRE(ctx, u[i].rows > 0 && u[i].cols > 0 && std::max(u[i].rows, u[i].cols) <= INT32_MAX - (1 << 20), "muon_update_many: bad shape");
    VLB_REQUIRE(ctx, u[i].W && u[i].S1 && u[i].G, "muon_update_many: null tensor");
  }
  VLB_REQUIRE(ctx, vlb::on_its_device(ctx), "muon_update_many: the context belongs to another device than the current one");
  bool const exact = ctx->precision == VLB_PRECISION_FP32;
  // the scratch of the pass that needs most is there before the first one: a call that cannot have it has changed nothing
  size_t most = 0;
  for (int first = 0, end; first < count; first = end) {
    end = end_of_pass(first, count, u, exact);
    most = std::max(most, exact ? exact_bytes(u[first]) : Layout(end - first, u + first, o->steps, nullptr).bytes);
  }
  if (most && !vlb::workspace(ctx, most)) return vlb::pass_error(ctx, ctx->lastError, "vlb_muon_update_many");
  for (int first = 0, end; first < count; first = end) {
    end = end_of_pass(first, count, u, exact);
    int const rc = exact ? update_exact(ctx, u[first], gradMult, o) : update_on_pairs(ctx, end - first, u + first, gradMult, o);
    if (rc) return vlb::pass_error(ctx, rc, "vlb_muon_update_many");
  }
  return vlb::check_launch(ctx, "vlb_muon_update_many");
}

}  // extern "C"
