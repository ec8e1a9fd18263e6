// One AdamW step over many tensors, with 32-bit or 8-bit states, and the global gradient norm it clips by
// (dm_adamw_step, dm_adamw_step_counted, dm_grad_norm).
//
// Three launches whatever the number of tensors: the sum of g^2 in NORM_PARTS parts (only where the norm is asked for),
// one block that makes the step's scalars from them and from the step count, and the update, a block per chunk of a tensor;
// a plan in device memory says which. All of it streams: 543M parameters (fp32 gradients) move 15.2 GB, and 2.2 GB for
// the norm, in 3.01 ms (5.8 TB/s, where a large copy reaches 5.0); with 8-bit states 8.7 and 2.2 GB in 1.81 ms (6.0 TB/s).
// A small model's step (2.9M) takes 21 us, of which 4 are the scalars' launch (3.3 with one step count for all tensors).
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
struct Rates {
  float rate, v_scale;   // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
};
// what the step's kernels share: written by k_adamw_begin
struct Control {
  float coef, lr;   // c
  Rates all;        // of every tensor, where they have no step counts of their own
  uint32_t key;     // the step's hash
  int skip;
};
static_assert(sizeof(Control) + 64 + NORM_PARTS * sizeof(double) <= DM_ADAMW_WORKSPACE, "workspace");
struct Workspace {
  Control* c;
  double* part;
  Rates* rates;   // per tensor, with step counts of their own
};
Workspace carve(void* base) {
  return {(Control*)base, (double*)((char*)base + 64), (Rates*)((char*)base + DM_ADAMW_WORKSPACE)};
}

struct AdamArgs {
  const PlanTensor* tensors;
  const int* chunk_tensor;
  void *m, *v;
  uint8_t *me, *ve;
  float b1, c1, b2, c2, eps;   // c = 1 - b
  const Control* c;
  const Rates* rates;          // nullptr: Control's for all
};

DM_DEV float grad_at(const PlanTensor& t, long i) {
  return t.g_bf16 ? __uint_as_float((uint32_t)ld_global<uint16_t>((const bf16*)t.g + i) << 16) : ld_global<float>((const float*)t.g + i);
}
// Vectors in global memory, aligned to A bytes. PAST: with the non-temporal hint, for what is larger than the caches
// keep from one kernel to the next (see Stream).
template <typename V, int A, bool PAST, typename P> DM_DEV V load(const P* p) {
  typedef V VA __attribute__((aligned(A)));
  const auto* q = (const __attribute__((address_space(1))) VA*)p;
  if constexpr (PAST) return __builtin_nontemporal_load(q);
  else return *q;
}
template <int A, bool PAST, typename V, typename P> DM_DEV void store(P* p, const V& v) {
  typedef V VA __attribute__((aligned(A)));
  auto* q = (__attribute__((address_space(1))) VA*)p;
  if constexpr (PAST) __builtin_nontemporal_store(v, q);
  else *q = v;
}
DM_DEV u32x4 pack8(const float* v) {
  const uint4 r = pack16<bf16>(v);
  return u32x4{r.x, r.y, r.z, r.w};
}
// Four gradients from i on. Parameters and gradients may be views at any element of a buffer: their vectors are aligned
// to their elements only.
template <bool BF16, bool PAST> DM_DEV floatx4 grads4(const PlanTensor& t, long i) {
  if constexpr (BF16) {
    const u32x2 r = load<u32x2, 2, PAST>((const bf16*)t.g + i);
    return floatx4{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16),
                   __uint_as_float(r[1] & 0xffff0000u)};
  } else {
    return load<floatx4, 4, PAST>((const float*)t.g + i);
  }
}
// What goes past the caches. A small model's step finds its data in the last one, of 256 MB (2.9M parameters, 80 MB). A
// larger step's parameters and states, read and written, only push one another and what else the program uses out. Steps of
// three models in turn, kept / states and parameters past / gradients past as well: 6M parameters 47 / 42 / 44 us, 15M 103 /
// 84 / 91, 47M 299 / 254 / 263; with 8-bit states 38 / 37 / 37, 75 / 64 / 64, 189 / 164 / 166. (One model's steps with nothing
// between them find more of it: 6M 40 / 42 / 41, 15M 80 / 84 / 89, 47M 297 / 230 / 256.) The gradients stay as long as they
// fit by themselves, since the norm has read them just before; beyond, they go past too (543M: 3.24 / 3.09 / 3.01 ms, with
// 8-bit states 2.02 / 1.79 / 1.81).
enum class Stream { KEPT, STATES, ALL };
constexpr double CACHE_BYTES = 256 << 20;

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

template <bool BF16, bool PAST> DM_DEV void add_squares(const PlanTensor& t, long i, long end, double (&s)[4]) {
  constexpr int STEP = 256 * 4, IN_FLIGHT = 4;
  i += 4 * threadIdx.x;
  for (; i + (IN_FLIGHT - 1) * STEP + 3 < end; i += IN_FLIGHT * STEP) {
    floatx4 g[IN_FLIGHT];
#pragma unroll
    for (int k = 0; k < IN_FLIGHT; ++k) g[k] = grads4<BF16, PAST>(t, i + k * STEP);
#pragma unroll
    for (int k = 0; k < IN_FLIGHT; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += (double)g[k][j] * g[k][j];
  }
  for (; i < end; i += STEP)
    for (int j = 0; j < 4 && i + j < end; ++j) {
      const double g = grad_at(t, i + j);
      s[j] += g * g;
    }
}
// part[b] = sum of g^2 over the b-th run of chunks. The squares of fp32 are exact in 64 bits, so the norm is the same for
// any order of the sum but for its last bits. A run's chunks are neighbours, so a tensor's entry is read once per run and
// tensor (chunk by chunk in a stride each waited for two dependent loads: 1.05 ms for 543M fp32 gradients). Bound by reading
// them: 0.37 ms, 5.8 TB/s.
template <bool PAST>
__global__ __launch_bounds__(256) void k_grad_sumsq(const PlanTensor* tensors, const int* chunk_tensor, long n_chunks, double* part) {
  __shared__ double red[4];
  double s[4] = {0., 0., 0., 0.};
  const long end = (blockIdx.x + 1) * n_chunks / gridDim.x;
  for (long c = blockIdx.x * n_chunks / gridDim.x; c < end;) {
    const PlanTensor t = tensors[chunk_tensor[c]];
    const long first = (c - t.chunk0) * CHUNK, last = min((end - t.chunk0) * CHUNK, t.n);   // this run's part of the tensor
    if (t.g_bf16) add_squares<true, PAST>(t, first, last, s);
    else add_squares<false, PAST>(t, first, last, s);
    c = t.chunk0 + (last + CHUNK - 1) / CHUNK;
  }
  const double x = block_sum((s[0] + s[1]) + (s[2] + s[3]), red);
  if (threadIdx.x == 0) part[blockIdx.x] = x;
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
  double log2_beta1, log2_beta2, max_norm;
  int skip_nonfinite;
  uint32_t seed;
  const float* lr;
  int64_t* steps;
  float* norm;
  int* skipped;
  const PlanTensor* tensors;
  int n_tensors;
  int64_t* tensor_steps;   // nullptr: all tensors' are *steps
  Rates* rates;
};
DM_DEV Rates rates_at(const BeginArgs& a, int64_t t) {
  const double power1 = exp2(t * a.log2_beta1), power2 = exp2(t * a.log2_beta2);
  return {(float)(*a.lr / (1. - power1)), (float)(1. / sqrt(1. - power2))};
}
// one block: the norm from its parts and the step's scalars; a thread per tensor counts its steps and makes its rates
__global__ __launch_bounds__(256) void k_adamw_begin(BeginArgs a) {
  __shared__ double red[4];
  const bool step = a.steps != nullptr;   // else the norm alone
  const int i = threadIdx.x;
  int64_t t = step ? *a.steps + 1 : 0, ti = t;
  long n = 0;
  if (step && a.tensor_steps && i < a.n_tensors) n = a.tensors[i].n, ti = a.tensor_steps[i] + 1;
  double s = 0.;
  for (int k = i; k < a.parts; k += 256) s += a.part[k];
  const Rates r = step ? rates_at(a, ti) : Rates{};
  s = block_sum(s, red);
  const double norm = sqrt(s);
  const bool skip = a.skip_nonfinite && !(norm < __builtin_inf());
  if (step && !skip && a.tensor_steps) {
    if (n > 0) a.tensor_steps[i] = ti, a.rates[i] = r;
    for (int k = i + 256; k < a.n_tensors; k += 256)
      if (a.tensors[k].n > 0) a.rates[k] = rates_at(a, a.tensor_steps[k] += 1);
  }
  if (i > 0) return;
  if (a.parts > 0 && a.norm) *a.norm = (float)norm;
  if (!step) return;
  Control c{};
  c.skip = skip;
  if (skip) {
    *a.skipped += 1;
    *a.c = c;
    return;
  }
  *a.steps = t;
  c.coef = 1.f;
  if (a.max_norm > 0.) {
    const double k = a.max_norm / (norm + 1e-6);
    c.coef = k < 1. || k != k ? (float)k : 1.f;
  }
  c.lr = *a.lr;
  c.all = r;
  c.key = mix(a.seed + (uint32_t)t * 0x9E3779B1u);
  *a.c = c;
}

// m and v of one element from its gradient; each product and sum rounded by itself, so that the codes made from them
// do not depend on how a compiler contracts them
DM_DEV void moments(const AdamArgs& a, float b1, float b2, float g, float& m, float& v) {
#pragma clang fp contract(off)
  const float m0 = b1 * m, m1 = a.c1 * g, v0 = b2 * v, v1 = a.c2 * (g * g);
  m = m0 + m1;
  v = v0 + v1;
}
// The parameters' part of a step, per tensor.
struct Update {
  float keep, rate, v_scale, eps;
  DM_DEV Update(const AdamArgs& a, const Control& c, const Rates& r, const PlanTensor& t)
      : keep((float)(1. - (double)c.lr * t.lr_scale * t.weight_decay)), rate(r.rate * t.lr_scale), v_scale(r.v_scale), eps(a.eps) {}
  // A square root and a reciprocal of one ulp each. The root's instruction takes numbers below 2^-126 for 0, so small ones
  // are scaled up before it; the reciprocal's would too, but eps is not below 2^-126.
  DM_DEV float of(float p, float m, float v) const {
    const bool small = v < 0x1p-96f;
    const float root = __builtin_amdgcn_sqrtf(small ? v * 0x1p32f : v);
    const float denom = fmaf(root, small ? v_scale * 0x1p-16f : v_scale, eps);
    return p * keep - rate * (m * __builtin_amdgcn_rcpf(denom));
  }
};

// A block per chunk; bound by its 28 bytes per element (543M: 15.2 GB in 2.64 ms).
template <bool BF16, Stream S> DM_DEV void step32(const AdamArgs& a, const Control& c, const Update& u, const PlanTensor& t, long i0, float* ms, float* vs) {
  constexpr int STEP = 256 * 4, N = CHUNK / STEP;
  constexpr bool PAST = S != Stream::KEPT;
  if (i0 + CHUNK <= t.n) {
    i0 += 4 * threadIdx.x;
    floatx4 p[N], g[N], m[N], v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long i = i0 + k * STEP;
      g[k] = grads4<BF16, S == Stream::ALL>(t, i);
      m[k] = load<floatx4, 16, PAST>(ms + i);
      v[k] = load<floatx4, 16, PAST>(vs + i);
      p[k] = load<floatx4, 4, PAST>(t.p + i);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long i = i0 + k * STEP;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float m1 = m[k][j], v1 = v[k][j];
        moments(a, a.b1, a.b2, g[k][j] * c.coef, m1, v1);
        m[k][j] = m1;
        v[k][j] = v1;
        p[k][j] = u.of(p[k][j], m1, v1);
      }
      store<16, PAST>(ms + i, m[k]);
      store<16, PAST>(vs + i, v[k]);
      store<4, PAST>(t.p + i, p[k]);
    }
    return;
  }
  for (long i = i0 + threadIdx.x; i < t.n; i += 256) {
    float m = ms[i], v = vs[i];
    moments(a, a.b1, a.b2, grad_at(t, i) * c.coef, m, v);
    ms[i] = m;
    vs[i] = v;
    t.p[i] = u.of(t.p[i], m, v);
  }
}
template <Stream S> __global__ __launch_bounds__(256) void k_adamw32(AdamArgs a) {
  const Control c = *a.c;
  if (c.skip) return;
  const int ti = a.chunk_tensor[blockIdx.x];
  const PlanTensor t = a.tensors[ti];
  const Update u(a, c, a.rates ? a.rates[ti] : c.all, t);
  const long i0 = (blockIdx.x - t.chunk0) * CHUNK;
  float* ms = (float*)a.m + t.block0 * BLOCK;
  float* vs = (float*)a.v + t.block0 * BLOCK;
  if (t.g_bf16) step32<true, S>(a, c, u, t, i0, ms, vs);
  else step32<false, S>(a, c, u, t, i0, ms, vs);
}

// The two code formats. Shifted to the place of an fp32 number's exponent and upper mantissa bits, a code is one, its
// smallest binade fp32's subnormal numbers; the value is that number times 2^(e - BIAS), e the block's exponent.
struct First {
  static constexpr int BIAS = 14;
};
struct Second {
  static constexpr int BIAS = 30;
};
template <typename F> DM_DEV float decoded(uint32_t code, int e) { return ldexpf(__uint_as_float(code << 20), e - F::BIAS); }
// x >= 0 rounded by the 20 random bits r20 (in the smallest binade after fp32's own rounding, to 2^-20 of a code)
template <typename F> DM_DEV uint32_t encoded(float x, int e, uint32_t r20) {
  return (__float_as_uint(ldexpf(x, F::BIAS - e)) + r20) >> 20;
}
// the exponent field of a block's largest magnitude, 255 where one is not below 2^127; every lane of the wave
DM_DEV int block_exponent(float largest, bool bad) {
  const int e = __float_as_uint(wave_max(largest)) >> 23;
  return __any(bad) ? 255 : max(e, 1);
}
DM_DEV bool too_large(float x) { return !(fabsf(x) < 0x1p127f); }

// A wave per run of four 256-element blocks, four elements per lane and block: a block's largest magnitude is a wave's
// reduction, its codes 4 bytes per lane. Bound by its 16 bytes per element (543M: 8.7 GB in 1.55 ms); the 89 vector
// instructions per element, a hash of two quarter-rate products among them, run beside the streams.
template <bool BF16, Stream S> DM_DEV void step8(const AdamArgs& a, const Control& c, const Update& u, const PlanTensor& t, long i0) {
  constexpr int N = CHUNK / BLOCK / 4;
  constexpr bool PAST = S != Stream::KEPT;
  const int lane = threadIdx.x & 63;
  const long blk0 = t.block0 + i0 / BLOCK;
  floatx4 p[N], g[N];
  uint32_t mc[N], vc[N];
  int me[N], ve[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const long i = i0 + k * BLOCK + 4 * lane;
    g[k] = p[k] = floatx4{0.f, 0.f, 0.f, 0.f};
    mc[k] = vc[k] = me[k] = ve[k] = 0;
    if (i0 + k * BLOCK >= t.n) continue;
    if (i + 3 < t.n) {
      g[k] = grads4<BF16, S == Stream::ALL>(t, i);
      p[k] = load<floatx4, 4, PAST>(t.p + i);
    } else {
      for (int j = 0; j < 3; ++j)
        if (i + j < t.n) g[k][j] = grad_at(t, i + j), p[k][j] = t.p[i + j];
    }
    mc[k] = load<uint32_t, 4, PAST>((const uint8_t*)a.m + (blk0 + k) * BLOCK + 4 * lane);
    vc[k] = load<uint32_t, 4, PAST>((const uint8_t*)a.v + (blk0 + k) * BLOCK + 4 * lane);
    me[k] = a.me[blk0 + k];
    ve[k] = a.ve[blk0 + k];
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const long i = i0 + k * BLOCK + 4 * lane;
    if (i0 + k * BLOCK >= t.n) return;
    // a block of NaN stays one
    const float b1 = me[k] == 255 ? __builtin_nanf("") : a.b1, b2 = ve[k] == 255 ? __builtin_nanf("") : a.b2;
    const uint32_t key = mix(c.key + (uint32_t)(blk0 + k) * 0x9E3779B1u) + lane * (4 * 0x9E3779B1u);
    float m[4], v[4], mmax = 0.f, vmax = 0.f;
    bool mbad = false, vbad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t cm = mc[k] >> 8 * j & 255;
      m[j] = decoded<First>(cm & 127, me[k]);
      m[j] = cm & 128 ? -m[j] : m[j];
      v[j] = decoded<Second>(vc[k] >> 8 * j & 255, ve[k]);
      moments(a, b1, b2, g[k][j] * c.coef, m[j], v[j]);
      p[k][j] = u.of(p[k][j], m[j], v[j]);
      if (i + j >= t.n) m[j] = v[j] = 0.f;   // behind the tensor's end
      mmax = fmaxf(mmax, fabsf(m[j]));
      vmax = fmaxf(vmax, v[j]);
      mbad |= too_large(m[j]);
      vbad |= too_large(v[j]);
    }
    const int me1 = block_exponent(mmax, mbad), ve1 = block_exponent(vmax, vbad);
    uint32_t mo = 0, vo = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t r = mix(key + j * 0x9E3779B1u);
      uint32_t cm = encoded<First>(fabsf(m[j]), me1, (r & 0xffff) << 4 | 8);
      cm |= cm ? __float_as_uint(m[j]) >> 24 & 128 : 0;
      const uint32_t cv = max(encoded<Second>(v[j], ve1, r >> 16 << 4 | 8), v[j] > 0.f ? 1u : 0u);
      mo |= cm << 8 * j;
      vo |= cv << 8 * j;
    }
    store<4, PAST>((uint8_t*)a.m + (blk0 + k) * BLOCK + 4 * lane, me1 == 255 ? 0 : mo);
    store<4, PAST>((uint8_t*)a.v + (blk0 + k) * BLOCK + 4 * lane, ve1 == 255 ? 0 : vo);
    if (lane == 0) {
      a.me[blk0 + k] = me1;
      a.ve[blk0 + k] = ve1;
    }
    if (i + 3 < t.n) {
      store<4, PAST>(t.p + i, p[k]);
    } else {
      for (int j = 0; j < 3; ++j)
        if (i + j < t.n) t.p[i + j] = p[k][j];
    }
  }
}
template <Stream S> __global__ __launch_bounds__(256) void k_adamw8(AdamArgs a) {
  const Control c = *a.c;
  if (c.skip) return;
  const int ti = a.chunk_tensor[blockIdx.x];
  const PlanTensor t = a.tensors[ti];
  const Update u(a, c, a.rates ? a.rates[ti] : c.all, t);
  const long i0 = (blockIdx.x - t.chunk0) * CHUNK + (threadIdx.x >> 6) * (CHUNK / 4);
  if (i0 >= t.n) return;
  if (t.g_bf16) step8<true, S>(a, c, u, t, i0);
  else step8<false, S>(a, c, u, t, i0);
}

// Eight codes per lane: the numbers of a wave's store follow one another. Bound by 3 bytes per element (543M: 0.28 ms).
template <typename F, bool PAST> __global__ __launch_bounds__(256) void k_adamw_values(const uint8_t* codes, const uint8_t* exps, long n_blocks, bf16* out) {
  constexpr bool SIGNED = F::BIAS == First::BIAS;
  constexpr int N = 4;   // vectors in flight
  const long n = n_blocks * (BLOCK / 8), step = gridDim.x * 256L;
  for (long i0 = blockIdx.x * 256L + threadIdx.x; i0 < n; i0 += N * step) {
    u32x2 c[N];
    int e[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long i = min(i0 + k * step, n - 1);
      c[k] = load<u32x2, 8, PAST>(codes + 8 * i);
      e[k] = exps[i / (BLOCK / 8)];
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (i0 + k * step >= n) return;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t q = c[k][j / 4] >> 8 * (j % 4) & 255;
        v[j] = decoded<F>(SIGNED ? q & 127 : q, e[k]);
        if (SIGNED && q & 128) v[j] = -v[j];
        if (e[k] == 255) v[j] = __builtin_nanf("");
      }
      store<16, PAST>(out + 8 * (i0 + k * step), pack8(v));
    }
  }
}

constexpr long MAX_CHUNKS = 1L << 24;   // of a launch
constexpr long MAX_BLOCKS = 1L << 40;   // of the states
long chunks_of(long n) { return (n + CHUNK - 1) / CHUNK; }

int check_tensors(const dm_adamw_tensor* t, int n, long* chunks) {
  DM_REQUIRE(t != nullptr && n > 0, DM_ERR_INVALID, "%d tensors", n);
  *chunks = 0;
  for (int i = 0; i < n; ++i) {
    DM_REQUIRE(t[i].n >= 0 && t[i].n < MAX_CHUNKS * CHUNK && t[i].block0 >= 0 && t[i].block0 < MAX_BLOCKS, DM_ERR_INVALID, "tensor %d: n=%lld block0=%lld", i, (long long)t[i].n,
               (long long)t[i].block0);
    DM_REQUIRE(t[i].g_dtype == DM_F32 || t[i].g_dtype == DM_BF16, DM_ERR_INVALID, "tensor %d: gradient dtype %d", i, t[i].g_dtype);
    if (t[i].n == 0) continue;
    DM_REQUIRE(t[i].p && reinterpret_cast<uintptr_t>(t[i].p) % 4 == 0, DM_ERR_INVALID, "tensor %d: null or unaligned parameter", i);
    DM_REQUIRE(t[i].g && reinterpret_cast<uintptr_t>(t[i].g) % esz(t[i].g_dtype) == 0, DM_ERR_INVALID,
               "tensor %d: null or unaligned gradient", i);
    *chunks += chunks_of(t[i].n);
  }
  DM_REQUIRE(*chunks > 0 && *chunks < MAX_CHUNKS, DM_ERR_INVALID, "%ld chunks of %d elements", *chunks, CHUNK);
  return DM_OK;
}
size_t tensor_bytes(int n) { return (size_t)n * sizeof(PlanTensor); }

int check_plan(const dm_adamw_args* a) {
  DM_REQUIRE(a != nullptr, DM_ERR_INVALID, "null arguments");
  DM_REQUIRE(a->plan && aligned16(a->plan) && a->n_tensors > 0 && a->n_chunks > 0 && a->n_chunks < MAX_CHUNKS, DM_ERR_INVALID,
             "null or unaligned plan, %d tensors, %lld chunks", a->n_tensors, (long long)a->n_chunks);
  DM_REQUIRE(a->workspace && aligned16(a->workspace) && a->workspace_bytes >= DM_ADAMW_WORKSPACE, DM_ERR_WORKSPACE,
             "workspace %zu < %d bytes", a->workspace_bytes, DM_ADAMW_WORKSPACE);
  return DM_OK;
}
const int* chunk_map(const dm_adamw_args* a) { return (const int*)((const char*)a->plan + tensor_bytes(a->n_tensors)); }
double elements(const dm_adamw_args* a) { return (double)a->n_chunks * CHUNK; }   // at most
Stream stream_of(const dm_adamw_args* a) {   // by fp32 gradients
  if (elements(a) * 4 > CACHE_BYTES) return Stream::ALL;
  return elements(a) * (a->state_bits == 32 ? 28 : 16) > CACHE_BYTES / 2 ? Stream::STATES : Stream::KEPT;
}
int run_sumsq(const dm_adamw_args* a, double* part, hipStream_t s) {
  const int parts = (int)std::min<long>(a->n_chunks, NORM_PARTS);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(parts), dim3(256), 0, s, (const PlanTensor*)a->plan, chunk_map(a), (long)a->n_chunks, part);
  };
  if (elements(a) * 4 > CACHE_BYTES) go(k_grad_sumsq<true>);
  else go(k_grad_sumsq<false>);
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

int dm_adamw_step(const dm_adamw_args* a, void* stream) { return dm_adamw_step_counted(a, nullptr, stream); }

int dm_adamw_step_counted(const dm_adamw_args* a, int64_t* tensor_steps, void* stream) {
  const int rc = check_plan(a);
  if (rc) return rc;
  DM_REQUIRE(a->state_bits == 32 || a->state_bits == 8, DM_ERR_INVALID, "state_bits %d (32 or 8)", a->state_bits);
  DM_REQUIRE(a->exp_avg && a->exp_avg_sq && aligned16(a->exp_avg) && aligned16(a->exp_avg_sq), DM_ERR_INVALID,
             "null or unaligned state");
  DM_REQUIRE(a->state_bits == 32 || (a->exp_avg_exponent && a->exp_avg_sq_exponent), DM_ERR_INVALID, "null block exponents");
  DM_REQUIRE(a->beta1 >= 0. && a->beta1 < 1. && a->beta2 >= 0. && a->beta2 < 1. && (float)a->eps >= 0x1p-126f && (float)a->eps < INFINITY,
             DM_ERR_INVALID, "beta1=%g beta2=%g eps=%g", a->beta1, a->beta2, a->eps);
  DM_REQUIRE(a->max_norm < HUGE_VAL, DM_ERR_INVALID, "max_norm=%g", a->max_norm);
  const bool norm = a->max_norm > 0. || a->skip_nonfinite;
  DM_REQUIRE(a->lr && a->steps && (a->norm || !norm) && (a->skipped || !a->skip_nonfinite), DM_ERR_INVALID, "null scalar");
  DM_REQUIRE(reinterpret_cast<uintptr_t>(tensor_steps) % 8 == 0, DM_ERR_INVALID, "unaligned tensor_steps");
  const size_t need = DM_ADAMW_WORKSPACE + (tensor_steps ? a->n_tensors * sizeof(Rates) : 0);
  DM_REQUIRE(a->workspace_bytes >= need, DM_ERR_WORKSPACE, "workspace %zu < %zu bytes", a->workspace_bytes, need);
  hipStream_t s = S(stream);
  const Workspace w = carve(a->workspace);
  Rates* rates = tensor_steps ? w.rates : nullptr;
  const int parts = norm ? run_sumsq(a, w.part, s) : 0;
  hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(256), 0, s,
                     BeginArgs{w.c, w.part, parts, std::log2(a->beta1), std::log2(a->beta2), a->max_norm, a->skip_nonfinite, a->seed, a->lr, a->steps,
                               a->norm, a->skipped, (const PlanTensor*)a->plan, a->n_tensors, tensor_steps, rates});
  const AdamArgs k{(const PlanTensor*)a->plan, chunk_map(a), a->exp_avg, a->exp_avg_sq, a->exp_avg_exponent,
                   a->exp_avg_sq_exponent, (float)a->beta1, (float)(1. - a->beta1), (float)a->beta2, (float)(1. - a->beta2),
                   (float)a->eps, w.c, rates};
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a->n_chunks), dim3(256), 0, s, k); };
  switch (stream_of(a)) {
    case Stream::KEPT: a->state_bits == 32 ? go(k_adamw32<Stream::KEPT>) : go(k_adamw8<Stream::KEPT>); break;
    case Stream::STATES: a->state_bits == 32 ? go(k_adamw32<Stream::STATES>) : go(k_adamw8<Stream::STATES>); break;
    case Stream::ALL: a->state_bits == 32 ? go(k_adamw32<Stream::ALL>) : go(k_adamw8<Stream::ALL>); break;
  }
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
  DM_REQUIRE(n_blocks >= 0 && n_blocks < MAX_BLOCKS, DM_ERR_INVALID, "n_blocks=%lld", (long long)n_blocks);
  if (n_blocks == 0) return DM_OK;
  DM_REQUIRE(codes && exponents && out && aligned16(codes) && aligned16(out), DM_ERR_INVALID, "null or unaligned operand");
  const dim3 grid((unsigned)std::min<long>((n_blocks + 31) / 32, 1 << 16));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, S(stream), codes, exponents, (long)n_blocks, (bf16*)out);
  };
  if (n_blocks * BLOCK * 3. > CACHE_BYTES) second ? go(k_adamw_values<Second, true>) : go(k_adamw_values<First, true>);
  else second ? go(k_adamw_values<Second, false>) : go(k_adamw_values<First, false>);
  DM_HIP(hipGetLastError());
  return DM_OK;
}

}  // extern "C"
