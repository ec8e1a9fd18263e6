// One AdamW step over many tensors, with 32-bit or 8-bit states, and the global gradient norm it clips by
// (dm_adamw_step, dm_grad_norm).
#include "dm_common.h"
#include "dm_error.h"

#include <algorithm>
#include <cmath>

using namespace dm;

namespace {

constexpr int BLOCK = DM_ADAMW_BLOCK;
constexpr int CHUNK = 16 * BLOCK;      // elements per launched block: four 256-element blocks per wave
constexpr int NORM_PARTS = 1024;       // partial sums of the norm

// the plan: the tensors, then the tensor of each chunk
struct PlanTensor {
  float* p;
  const void* g;
  long n, block0, chunk0;   // chunk0: the tensor's first chunk
  float weight_decay, lr_scale;
  int g_bf16, pad;
};
// what the step's kernels share: written by k_adamw_begin
struct Control {
  double norm;
  float coef, rate, v_scale, lr;   // c, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
  uint32_t key;                    // the step's hash
  int skip;
};
static_assert(sizeof(Control) + 64 + NORM_PARTS * sizeof(double) <= DM_ADAMW_WORKSPACE, "workspace");
struct Workspace {
  Control* c;
  double* part;
};
Workspace carve(void* base) { return {(Control*)base, (double*)((char*)base + 64)}; }

struct AdamArgs {
  const PlanTensor* tensors;
  const int* chunk_tensor;
  void *m, *v;
  uint8_t *me, *ve;
  float b1, c1, b2, c2, eps;   // c = 1 - b
  const Control* c;
};

DM_DEV float grad_at(const PlanTensor& t, long i) {
  return t.g_bf16 ? to_f(((const bf16*)t.g)[i]) : ((const float*)t.g)[i];
}

DM_DEV double block_sum(double x, double* red) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) x += red[w];
  return x;
}

// part[b] = sum of g^2 over chunks b, b + NORM_PARTS, ...
__global__ __launch_bounds__(256) void k_grad_sumsq(const PlanTensor* tensors, const int* chunk_tensor, long n_chunks,
                                                    double* part) {
  __shared__ double red[4];
  double s = 0.;
  for (long c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const PlanTensor t = tensors[chunk_tensor[c]];
    const long i0 = (c - t.chunk0) * CHUNK;
    for (long i = i0 + threadIdx.x; i < min(i0 + CHUNK, t.n); i += 256) {
      const double g = grad_at(t, i);
      s += g * g;
    }
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// A 32-bit hash: two odd multipliers and three shifts.
DM_DEV uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 13;
  x *= 0xBB67AE85u;
  return x ^ x >> 16;
}

struct BeginArgs {
  Control* c;
  const double* part;
  int parts;   // 0: no norm
  double beta1, beta2, max_norm;
  int skip_nonfinite;
  uint32_t seed;
  const float* lr;
  int64_t* steps;
  float* norm;
  int* skipped;
};
// one block: the norm from its parts and the step's scalars
__global__ __launch_bounds__(256) void k_adamw_begin(BeginArgs a) {
  __shared__ double red[4];
  double s = 0.;
  for (int i = threadIdx.x; i < a.parts; i += 256) s += a.part[i];
  s = block_sum(s, red);
  if (threadIdx.x > 0) return;
  const double norm = sqrt(s);
  if (a.parts > 0 && a.norm) *a.norm = (float)norm;
  if (!a.steps) return;   // the norm alone
  Control c;
  c.norm = norm;
  c.skip = a.skip_nonfinite && !(norm < __builtin_inf());
  if (c.skip) {
    *a.skipped += 1;
    *a.c = c;
    return;
  }
  const int64_t t = *a.steps + 1;
  *a.steps = t;
  c.coef = 1.f;
  if (a.max_norm > 0.) {
    const double k = a.max_norm / (norm + 1e-6);
    c.coef = k < 1. || k != k ? (float)k : 1.f;
  }
  c.lr = *a.lr;
  c.rate = (float)(c.lr / (1. - pow(a.beta1, (double)t)));
  c.v_scale = (float)(1. / sqrt(1. - pow(a.beta2, (double)t)));
  c.key = mix(a.seed + (uint32_t)t * 0x9E3779B1u);
  *a.c = c;
}

// m and v of one element from its gradient; each product and sum rounded by itself, so that the codes made from them
// do not depend on how a compiler contracts them
DM_DEV void moments(const AdamArgs& a, float g, float& m, float& v) {
#pragma clang fp contract(off)
  const float m0 = a.b1 * m, m1 = a.c1 * g, v0 = a.b2 * v, v1 = a.c2 * (g * g);
  m = m0 + m1;
  v = v0 + v1;
}
DM_DEV float updated(const AdamArgs& a, const Control& c, const PlanTensor& t, float p, float m, float v) {
  const float keep = (float)(1. - (double)c.lr * t.lr_scale * t.weight_decay);
  return p * keep - c.rate * t.lr_scale * (m / (sqrtf(v) * c.v_scale + a.eps));
}

__global__ __launch_bounds__(256) void k_adamw32(AdamArgs a) {
  const Control c = *a.c;
  if (c.skip) return;
  const PlanTensor t = a.tensors[a.chunk_tensor[blockIdx.x]];
  const long i0 = (blockIdx.x - t.chunk0) * CHUNK;
  float* ms = (float*)a.m + t.block0 * BLOCK;
  float* vs = (float*)a.v + t.block0 * BLOCK;
  for (long i = i0 + threadIdx.x; i < min(i0 + CHUNK, t.n); i += 256) {
    float m = ms[i], v = vs[i];
    moments(a, grad_at(t, i) * c.coef, m, v);
    ms[i] = m;
    vs[i] = v;
    t.p[i] = updated(a, c, t, t.p[i], m, v);
  }
}

// The two code formats: a normal code is the exponent and the three upper mantissa bits of a, less (EXP - 1) << 3,
// EXP the exponent field of the smallest normal a; below it the grid is 2^-GRID.
struct First {
  static constexpr int EXP = 112, GRID = 18;
};
struct Second {
  static constexpr int EXP = 96, GRID = 34;
};
template <typename F> DM_DEV float decoded(uint32_t code, int e) {   // code without sign
  const float a = code >= 8 ? __uint_as_float((code + ((F::EXP - 1) << 3)) << 20) : ldexpf((float)code, -F::GRID);
  return e == 255 ? __builtin_nanf("") : ldexpf(a, e - 125);
}
// x >= 0 rounded by the 20 random bits r20; e: its block's exponent
template <typename F> DM_DEV uint32_t encoded(float x, int e, uint32_t r20) {
  const float a = ldexpf(x, 125 - e);
  if (a >= ldexpf(1.f, 3 - F::GRID)) return ((__float_as_uint(a) + r20) >> 20) - ((F::EXP - 1) << 3);
  return (uint32_t)(ldexpf(a, F::GRID) + ldexpf((float)r20, -20));
}
// the exponent field of a block's largest magnitude, 255 where one is not below 2^127; every lane of the wave
DM_DEV int block_exponent(float largest, bool bad) {
  const int e = __float_as_uint(wave_max(largest)) >> 23;
  return __any(bad) ? 255 : max(e, 1);
}
DM_DEV bool too_large(float x) { return !(fabsf(x) < 0x1p127f); }

// a wave per 256-element block, four elements per lane
__global__ __launch_bounds__(256) void k_adamw8(AdamArgs a) {
  const Control c = *a.c;
  if (c.skip) return;
  const PlanTensor t = a.tensors[a.chunk_tensor[blockIdx.x]];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b = wave; b < CHUNK / BLOCK; b += 4) {
    const long i0 = (blockIdx.x - t.chunk0) * CHUNK + b * BLOCK;
    if (i0 >= t.n) return;
    const long blk = t.block0 + i0 / BLOCK, at = blk * BLOCK + 4 * lane;
    const int me = a.me[blk], ve = a.ve[blk];
    const uint32_t mc = *(const uint32_t*)((const uint8_t*)a.m + at), vc = *(const uint32_t*)((const uint8_t*)a.v + at);
    const uint32_t key = mix(c.key + (uint32_t)blk * 0x9E3779B1u);
    float m[4], v[4], mmax = 0.f, vmax = 0.f;
    bool mbad = false, vbad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long i = i0 + 4 * lane + j;
      const uint32_t cm = mc >> 8 * j & 255, cv = vc >> 8 * j & 255;
      m[j] = decoded<First>(cm & 127, me);
      m[j] = cm & 128 ? -m[j] : m[j];
      v[j] = decoded<Second>(cv, ve);
      if (i < t.n) {
        moments(a, grad_at(t, i) * c.coef, m[j], v[j]);
        t.p[i] = updated(a, c, t, t.p[i], m[j], v[j]);
      } else {
        m[j] = v[j] = 0.f;
      }
      mmax = fmaxf(mmax, fabsf(m[j]));
      vmax = fmaxf(vmax, v[j]);
      mbad |= too_large(m[j]);
      vbad |= too_large(v[j]);
    }
    const int me1 = block_exponent(mmax, mbad), ve1 = block_exponent(vmax, vbad);
    uint32_t mo = 0, vo = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t r = mix(key + (4 * lane + j) * 0x9E3779B1u);
      uint32_t cm = me1 == 255 ? 0 : encoded<First>(fabsf(m[j]), me1, (r & 0xffff) << 4 | 8);
      cm |= m[j] < 0.f && cm ? 128 : 0;
      uint32_t cv = ve1 == 255 ? 0 : encoded<Second>(v[j], ve1, r >> 16 << 4 | 8);
      if (v[j] > 0.f && cv == 0) cv = 1;
      mo |= cm << 8 * j;
      vo |= cv << 8 * j;
    }
    *(uint32_t*)((uint8_t*)a.m + at) = mo;
    *(uint32_t*)((uint8_t*)a.v + at) = vo;
    if (lane == 0) {
      a.me[blk] = me1;
      a.ve[blk] = ve1;
    }
  }
}

template <typename F> __global__ __launch_bounds__(256) void k_adamw_values(const uint8_t* codes, const uint8_t* exps, long n_blocks, bf16* out) {
  const int lane = threadIdx.x & 63;
  for (long b = blockIdx.x * 4L + (threadIdx.x >> 6); b < n_blocks; b += gridDim.x * 4L) {
    const uint32_t c = *(const uint32_t*)(codes + b * BLOCK + 4 * lane);
    const int e = exps[b];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t q = c >> 8 * j & 255;
      const bool neg = F::GRID == First::GRID && q & 128;
      const float x = decoded<F>(F::GRID == First::GRID ? q & 127 : q, e);
      out[b * BLOCK + 4 * lane + j] = from_f<bf16>(neg ? -x : x);
    }
  }
}

long chunks_of(long n) { return (n + CHUNK - 1) / CHUNK; }

int check_tensors(const dm_adamw_tensor* t, int n, long* chunks) {
  DM_REQUIRE(t != nullptr && n > 0, DM_ERR_INVALID, "%d tensors", n);
  *chunks = 0;
  for (int i = 0; i < n; ++i) {
    DM_REQUIRE(t[i].n >= 0 && t[i].block0 >= 0, DM_ERR_INVALID, "tensor %d: n=%lld block0=%lld", i, (long long)t[i].n,
               (long long)t[i].block0);
    DM_REQUIRE(t[i].g_dtype == DM_F32 || t[i].g_dtype == DM_BF16, DM_ERR_INVALID, "tensor %d: gradient dtype %d", i, t[i].g_dtype);
    if (t[i].n == 0) continue;
    DM_REQUIRE(t[i].p && reinterpret_cast<uintptr_t>(t[i].p) % 4 == 0, DM_ERR_INVALID, "tensor %d: null or unaligned parameter", i);
    DM_REQUIRE(t[i].g && reinterpret_cast<uintptr_t>(t[i].g) % esz(t[i].g_dtype) == 0, DM_ERR_INVALID,
               "tensor %d: null or unaligned gradient", i);
    *chunks += chunks_of(t[i].n);
  }
  DM_REQUIRE(*chunks > 0 && *chunks < (1L << 24), DM_ERR_INVALID, "%ld chunks of %d elements", *chunks, CHUNK);
  return DM_OK;
}
size_t tensor_bytes(int n) { return (size_t)n * sizeof(PlanTensor); }

int check_plan(const dm_adamw_args* a) {
  DM_REQUIRE(a != nullptr, DM_ERR_INVALID, "null arguments");
  DM_REQUIRE(a->plan && aligned16(a->plan) && a->n_tensors > 0 && a->n_chunks > 0 && a->n_chunks < (1L << 24), DM_ERR_INVALID,
             "null or unaligned plan, %d tensors, %lld chunks", a->n_tensors, (long long)a->n_chunks);
  DM_REQUIRE(a->workspace && aligned16(a->workspace) && a->workspace_bytes >= DM_ADAMW_WORKSPACE, DM_ERR_WORKSPACE,
             "workspace %zu < %d bytes", a->workspace_bytes, DM_ADAMW_WORKSPACE);
  return DM_OK;
}
const int* chunk_map(const dm_adamw_args* a) { return (const int*)((const char*)a->plan + tensor_bytes(a->n_tensors)); }
int run_sumsq(const dm_adamw_args* a, double* part, hipStream_t s) {
  const int parts = (int)std::min<long>(a->n_chunks, NORM_PARTS);
  hipLaunchKernelGGL(k_grad_sumsq, dim3(parts), dim3(256), 0, s, (const PlanTensor*)a->plan, chunk_map(a), a->n_chunks, part);
  return parts;
}

}  // namespace

extern "C" {

size_t dm_adamw_plan_bytes(const dm_adamw_tensor* t, int32_t n_tensors) {
  long chunks = 0;
  return check_tensors(t, n_tensors, &chunks) ? 0 : tensor_bytes(n_tensors) + chunks * sizeof(int);
}

int dm_adamw_plan(const dm_adamw_tensor* t, int32_t n_tensors, void* plan, size_t plan_bytes, int64_t* n_chunks) {
  long chunks = 0;
  const int rc = check_tensors(t, n_tensors, &chunks);
  if (rc) return rc;
  const size_t need = tensor_bytes(n_tensors) + chunks * sizeof(int);
  DM_REQUIRE(plan && n_chunks && plan_bytes >= need, DM_ERR_WORKSPACE, "plan %zu < %zu bytes", plan_bytes, need);
  PlanTensor* out = (PlanTensor*)plan;
  int* map = (int*)((char*)plan + tensor_bytes(n_tensors));
  long c = 0;
  for (int i = 0; i < n_tensors; ++i) {
    out[i] = {t[i].p, t[i].g, t[i].n, t[i].block0, c, t[i].weight_decay, t[i].lr_scale, t[i].g_dtype == DM_BF16, 0};
    for (long k = chunks_of(t[i].n); k > 0; --k) map[c++] = i;
  }
  *n_chunks = chunks;
  return DM_OK;
}

int dm_adamw_step(const dm_adamw_args* a, void* stream) {
  const int rc = check_plan(a);
  if (rc) return rc;
  DM_REQUIRE(a->state_bits == 32 || a->state_bits == 8, DM_ERR_INVALID, "state_bits %d (32 or 8)", a->state_bits);
  DM_REQUIRE(a->exp_avg && a->exp_avg_sq && aligned16(a->exp_avg) && aligned16(a->exp_avg_sq), DM_ERR_INVALID,
             "null or unaligned state");
  DM_REQUIRE(a->state_bits == 32 || (a->exp_avg_exponent && a->exp_avg_sq_exponent), DM_ERR_INVALID, "null block exponents");
  DM_REQUIRE(a->beta1 >= 0. && a->beta1 < 1. && a->beta2 >= 0. && a->beta2 < 1. && (float)a->eps > 0.f && a->eps < HUGE_VAL,
             DM_ERR_INVALID, "beta1=%g beta2=%g eps=%g", a->beta1, a->beta2, a->eps);
  DM_REQUIRE(a->max_norm < HUGE_VAL, DM_ERR_INVALID, "max_norm=%g", a->max_norm);
  const bool norm = a->max_norm > 0. || a->skip_nonfinite;
  DM_REQUIRE(a->lr && a->steps && (a->norm || !norm) && (a->skipped || !a->skip_nonfinite), DM_ERR_INVALID, "null scalar");
  hipStream_t s = S(stream);
  const Workspace w = carve(a->workspace);
  const int parts = norm ? run_sumsq(a, w.part, s) : 0;
  hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(256), 0, s,
                     BeginArgs{w.c, w.part, parts, a->beta1, a->beta2, a->max_norm, a->skip_nonfinite, a->seed, a->lr, a->steps,
                               a->norm, a->skipped});
  const AdamArgs k{(const PlanTensor*)a->plan, chunk_map(a), a->exp_avg, a->exp_avg_sq, a->exp_avg_exponent,
                   a->exp_avg_sq_exponent, (float)a->beta1, (float)(1. - a->beta1), (float)a->beta2, (float)(1. - a->beta2),
                   (float)a->eps, w.c};
  if (a->state_bits == 32) hipLaunchKernelGGL(k_adamw32, dim3(a->n_chunks), dim3(256), 0, s, k);
  else hipLaunchKernelGGL(k_adamw8, dim3(a->n_chunks), dim3(256), 0, s, k);
  DM_HIP(hipGetLastError());
  return DM_OK;
}

int dm_grad_norm(const dm_adamw_args* a, void* stream) {
  const int rc = check_plan(a);
  if (rc) return rc;
  DM_REQUIRE(a->norm, DM_ERR_INVALID, "null norm");
  const Workspace w = carve(a->workspace);
  BeginArgs b{};
  b.part = w.part;
  b.parts = run_sumsq(a, w.part, S(stream));
  b.norm = a->norm;
  hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(256), 0, S(stream), b);
  DM_HIP(hipGetLastError());
  return DM_OK;
}

int dm_adamw_values(const uint8_t* codes, const uint8_t* exponents, int64_t n_blocks, int32_t second, void* out, void* stream) {
  DM_REQUIRE(n_blocks >= 0 && n_blocks < (1L << 40), DM_ERR_INVALID, "n_blocks=%lld", (long long)n_blocks);
  if (n_blocks == 0) return DM_OK;
  DM_REQUIRE(codes && exponents && out && aligned16(codes) && aligned16(out), DM_ERR_INVALID, "null or unaligned operand");
  const dim3 grid((unsigned)std::min<long>((n_blocks + 3) / 4, 1 << 16));
  if (second) hipLaunchKernelGGL(k_adamw_values<Second>, grid, dim3(256), 0, S(stream), codes, exponents, (long)n_blocks, (bf16*)out);
  else hipLaunchKernelGGL(k_adamw_values<First>, grid, dim3(256), 0, S(stream), codes, exponents, (long)n_blocks, (bf16*)out);
  DM_HIP(hipGetLastError());
  return DM_OK;
}

}  // extern "C"
