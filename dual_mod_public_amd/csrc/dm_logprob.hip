// Log probabilities of given tokens, entropies, the most likely tokens and the logits' gradient (dm_logprob_rows,
// dm_logprob_rows_bwd).
#include "dm_common.h"
#include "dm_error.h"

#include <algorithm>

using namespace dm;

namespace {

constexpr float INF = __builtin_inff();
constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct LpArgs {
  const T* x;
  T* dx;   // nullptr: no gradient
  const int64_t* target;
  float *logp, *lse, *entropy, *stats, *top_logp;
  int64_t* top_ids;
  const float *g_logp, *g_entropy;
  long ld, ld_d;
  int rows, cols, top;
};

// The statistics of a row: lse = M + log_z where the maximum M is finite.
struct RowStats {
  float M, log_z, lse, entropy;
  DM_DEV float logp(float x) const {
    if (lse == -INF) return -INF;
    if (fabsf(lse) < INF) return (x - M) - log_z;
    return x - lse;   // NaN, or +inf in the row
  }
};

DM_DEV float exp_of(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }

// The order of the most likely tokens as one number per column: by value (NaN first, -0 as 0), then the lower id.
DM_DEV uint64_t order_of(float x, int id) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t o = x != x ? 0xffffffffu : (b >> 31 ? ~b : b | 0x80000000u);
  return (uint64_t)o << 32 | (uint32_t)~id;
}

template <int NT> struct Shared {
  float f[3][NT / 64];
  uint64_t key[NT / 64];
};

DM_DEV uint64_t wave_max_u64(uint64_t k) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t lo = __shfl_xor((uint32_t)k, o, 64), hi = __shfl_xor((uint32_t)(k >> 32), o, 64);
    const uint64_t other = (uint64_t)hi << 32 | lo;
    k = other > k ? other : k;
  }
  return k;
}

// What a row's gradient is made of: dx[v] = -p (g + gh (logp(v) + H)), + g at the target.
struct RowGrad {
  float g, gh;
  bool zero, nan;   // a row of zeros, of NaN
};
template <typename T> DM_DEV RowGrad row_grad(const LpArgs<T>& a, long r, float lse) {
  RowGrad w;
  const long t = a.target ? a.target[r] : -1;
  w.g = a.g_logp && t >= 0 ? a.g_logp[r] : 0.f;
  w.gh = a.g_entropy ? a.g_entropy[r] : 0.f;
  w.zero = (w.g == 0.f && w.gh == 0.f) || lse == -INF;
  w.nan = !w.zero && (!(fabsf(lse) < INF) || (w.g != 0.f && t >= a.cols));
  return w;
}
template <typename T> DM_DEV float grad_of(const RowStats& s, const RowGrad& w, float x) {
  const float lp = s.logp(x), p = exp_of(lp);
  return -p * (w.g + w.gh * (fmaxf(lp, -1e30f) + s.entropy));   // p = 0 at -inf
}

// One row by one block, element by element: every case.
template <typename T, int NT>
DM_DEV void any_row(const LpArgs<T>& a, long r, Shared<NT>& sh) {
  const T* x = a.x + r * a.ld;
  const int n = a.cols, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long t = a.target ? a.target[r] : -1;
  const float xt = t >= 0 && t < n ? to_f(x[t]) : 0.f;
  float m = -INF;
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += NT) {
    const float v = to_f(x[i]);
    bad |= v != v;
    m = fmaxf(m, v);
  }
  bad = __syncthreads_or(bad);
  m = wave_max(m);
  if (lane == 0) sh.f[0][wave] = m;
  __syncthreads();
  RowStats s;
  s.M = sh.f[0][0];
  for (int w = 1; w < NT / 64; ++w) s.M = fmaxf(s.M, sh.f[0][w]);
  if (bad) {
    s.M = s.lse = s.entropy = s.log_z = __builtin_nanf("");
  } else if (fabsf(s.M) == INF) {
    s.lse = s.log_z = s.M;
    s.entropy = s.M > 0 ? __builtin_nanf("") : 0.f;
  } else {
    float z = 0.f, q = 0.f;
    for (int i = threadIdx.x; i < n; i += NT) {
      const float d = to_f(x[i]) - s.M, e = exp_of(d);
      z += e;
      q += e * fmaxf(d, -1e30f);
    }
    z = wave_sum(z);
    q = wave_sum(q);
    if (lane == 0) sh.f[1][wave] = z, sh.f[2][wave] = q;
    __syncthreads();
    z = q = 0.f;
    for (int w = 0; w < NT / 64; ++w) z += sh.f[1][w], q += sh.f[2][w];
    s.log_z = logf(z);
    s.lse = s.M + s.log_z;
    s.entropy = s.log_z - q / z;
  }
  if (threadIdx.x == 0) {
    if (a.logp) a.logp[r] = t < 0 ? 0.f : t < n ? s.logp(xt) : __builtin_nanf("");
    if (a.lse) a.lse[r] = s.lse;
    if (a.entropy) a.entropy[r] = s.entropy;
    if (a.stats) a.stats[2 * r] = s.M, a.stats[2 * r + 1] = s.log_z;
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < a.top; ++j) {   // the next one in order after `last`
    uint64_t best = 0;
    for (int i = threadIdx.x; i < n; i += NT) {
      const uint64_t k = order_of(to_f(x[i]), i);
      if (k < last && k > best) best = k;
    }
    best = wave_max_u64(best);
    __syncthreads();
    if (lane == 0) sh.key[wave] = best;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) best = max(best, sh.key[w]);
    last = best;
    if (threadIdx.x == 0) {
      const int id = ~(uint32_t)best;
      a.top_ids[r * a.top + j] = id;
      a.top_logp[r * a.top + j] = s.logp(to_f(x[id]));
    }
  }
  __syncthreads();   // the row is read; its buffers are free again
  if (!a.dx) return;
  const RowGrad w = row_grad(a, r, s.lse);
  T* dx = a.dx + r * a.ld_d;
  for (int i = threadIdx.x; i < n; i += NT)
    dx[i] = from_f<T>(w.zero ? 0.f : w.nan ? __builtin_nanf("") : grad_of<T>(s, w, to_f(x[i])) + (i == t ? w.g : 0.f));
}

template <typename T> __global__ __launch_bounds__(256) void k_logprob_rows(LpArgs<T> a) {
  __shared__ Shared<256> sh;
  for (long r = blockIdx.x; r < a.rows; r += gridDim.x) any_row<T, 256>(a, r, sh);
}

template <typename T> __global__ __launch_bounds__(256) void k_logprob_bwd(LpArgs<T> a) {
  for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    RowStats s;
    s.M = a.stats[2 * r];
    s.log_z = a.stats[2 * r + 1];
    s.lse = s.M + s.log_z;
    s.entropy = a.g_entropy ? a.entropy[r] : 0.f;
    const RowGrad w = row_grad(a, r, s.lse);
    const long t = a.target ? a.target[r] : -1;
    const T* x = a.x + r * a.ld;
    T* dx = a.dx + r * a.ld_d;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < a.cols; i += gridDim.x * 256)
      dx[i] = from_f<T>(w.zero ? 0.f : w.nan ? __builtin_nanf("") : grad_of<T>(s, w, to_f(x[i])) + (i == t ? w.g : 0.f));
  }
}

constexpr int MAX_BLOCKS = 1 << 20;   // a grid's blocks per dimension; further rows by the same blocks

template <typename T> LpArgs<T> typed(const dm_logprob_args* a) {
  return {(const T*)a->logits, (T*)a->dlogits, a->target, a->logp, a->lse, a->entropy, a->stats, a->top_logp,
          a->top_ids, a->g_logp, a->g_entropy, a->ld, a->ld_d, a->rows, a->cols, a->top};
}

template <typename T> void run_rows(const LpArgs<T>& a, hipStream_t s) {
  hipLaunchKernelGGL(k_logprob_rows<T>, dim3(std::min(a.rows, MAX_BLOCKS)), dim3(256), 0, s, a);
}
template <typename T> void run_bwd(const LpArgs<T>& a, hipStream_t s) {
  hipLaunchKernelGGL(k_logprob_bwd<T>, dim3(cdiv(a.cols, 4096), std::min(a.rows, 65535)), dim3(256), 0, s, a);
}

bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// what both entry points ask of their arguments
int check_logprob(const dm_logprob_args* a, bool bwd) {
  DM_REQUIRE(a != nullptr, DM_ERR_INVALID, "null arguments");
  DM_REQUIRE(a->dtype == DM_BF16 || a->dtype == DM_F32, DM_ERR_INVALID, "dtype %d", a->dtype);
  DM_REQUIRE(a->rows >= 0 && a->cols > 0 && a->ld >= a->cols, DM_ERR_INVALID, "rows=%d cols=%d ld=%lld", a->rows, a->cols,
             (long long)a->ld);
  if (a->rows == 0) return DM_OK;
  const size_t e = esz(a->dtype);
  DM_REQUIRE(a->logits && aligned_to(a->logits, e), DM_ERR_INVALID, "null or unaligned logits");
  DM_REQUIRE(!a->logp || a->target, DM_ERR_INVALID, "logp without targets");
  if (!bwd) {
    DM_REQUIRE(a->top >= 0 && a->top <= DM_TOP_MAX && a->top <= a->cols, DM_ERR_INVALID, "top=%d of cols=%d (at most %d)",
               a->top, a->cols, DM_TOP_MAX);
    DM_REQUIRE(a->top == 0 || (a->top_logp && a->top_ids), DM_ERR_INVALID, "null output of the most likely tokens");
    if (!a->dlogits) return DM_OK;
  }
  DM_REQUIRE(a->dlogits && aligned_to(a->dlogits, e) && a->ld_d >= a->cols, DM_ERR_INVALID, "null or unaligned dlogits, ld_d=%lld",
             (long long)a->ld_d);
  DM_REQUIRE(a->g_logp || a->g_entropy, DM_ERR_INVALID, "a gradient without coefficients");
  DM_REQUIRE(!a->g_logp || a->target, DM_ERR_INVALID, "g_logp without targets");
  DM_REQUIRE(!bwd || (a->stats && (a->entropy || !a->g_entropy)), DM_ERR_INVALID, "the forward's stats (and entropy) are needed");
  const uintptr_t x = reinterpret_cast<uintptr_t>(a->logits), d = reinterpret_cast<uintptr_t>(a->dlogits);
  const size_t xe = ((size_t)(a->rows - 1) * a->ld + a->cols) * e, de = ((size_t)(a->rows - 1) * a->ld_d + a->cols) * e;
  DM_REQUIRE((x == d && a->ld == a->ld_d) || x + xe <= d || d + de <= x, DM_ERR_INVALID, "dlogits overlaps the logits in part");
  return DM_OK;
}

}  // namespace

extern "C" {

int dm_logprob_rows(const dm_logprob_args* a, void* stream) {
  const int rc = check_logprob(a, false);
  if (rc || a->rows == 0) return rc;
  if (a->dtype == DM_BF16) run_rows(typed<bf16>(a), S(stream));
  else run_rows(typed<float>(a), S(stream));
  DM_HIP(hipGetLastError());
  return DM_OK;
}

int dm_logprob_rows_bwd(const dm_logprob_args* a, void* stream) {
  const int rc = check_logprob(a, true);
  if (rc || a->rows == 0) return rc;
  if (a->dtype == DM_BF16) run_bwd(typed<bf16>(a), S(stream));
  else run_bwd(typed<float>(a), S(stream));
  DM_HIP(hipGetLastError());
  return DM_OK;
}

}  // extern "C"
