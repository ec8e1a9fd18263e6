// Log probabilities of given tokens, entropies, the most likely tokens and the logits' gradient (dm_logprob_rows,
// dm_logprob_rows_bwd).
//
// A row x of V logits: M = max x, Z = sum e^(x - M), lse = M + log Z, logp(v) = x_v - lse, and the entropy
// log Z - sum e^(x - M) (x - M) / Z, all from one pass over the row: each thread keeps its own maximum and two sums
// relative to it, joined over the block once (rescaled by 2 to the difference of their references). The gradient
// -p (g + gh (logp + H)) + g [target] needs lse and H, so a row's logits wait in registers for them: 16 vectors of
// 16 bytes in each of 256 threads hold 32768 bf16 logits, and the row is read and written once.
// The `top` most likely tokens: the 64 lanes' largest logits are logits of 64 different places, so the top-th of them is
// reached by at least `top` of the row; the few tens of logits that reach it are listed in LDS and ranked there. A row with
// more than 1024 such logits (equal ones or of few values, or masked by a finite number with fewer lanes of allowed ones than
// `top`) and one of -inf are scanned once per alternative instead: 64 rows of 50257 bf16 with 8 alternatives 83 to 100 us
// (ordinary ones 12), 4096 of 32000 1.34 to 1.42 ms (53).
// Bound by HBM (44 us for 262 MB of logits, 6.0 TB/s; with the gradient 524 MB in 98 us, 5.4 TB/s; a large copy reaches
// 5.0 to 5.4); close behind come the 11 vector instructions per logit, 4 of whose slots are the exponential.
#include "dm_common.h"
#include "dm_error.h"

#include <algorithm>

using namespace dm;

namespace {

constexpr float INF = __builtin_inff(), NAN_ = __builtin_nanf("");
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float FLOOR = -0x1p100f;   // fills the places of a tile without a logit; no reference of a sum is lower
constexpr int CANDIDATES = 1024;   // of a row's most likely tokens, in LDS

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

// The statistics of a row: lse = M + log_z, M its maximum.
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
DM_DEV uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : (b >> 31 ? ~b : b | 0x80000000u);
}
DM_DEV uint64_t order_of(float x, int id) { return (uint64_t)order_of(x) << 32 | (uint32_t)~id; }
DM_DEV float value_of(uint32_t order) { return __uint_as_float(order >> 31 ? order & 0x7fffffffu : ~order); }
constexpr uint32_t ORDER_OF_MINUS_INF = 0x007fffffu;

template <int NT> struct Shared {
  float m[NT / 64], z[NT / 64], q[NT / 64];
  uint64_t key[NT / 64];
  float largest[NT];            // each thread's largest logit
  int count;                    // candidates found
  uint64_t cand[CANDIDATES];
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

// What a row's gradient is made of: dx[v] = -p (g + gh (logp(v) + H)), + g at the target, as p (a + b y) with
// y = logp(v) log2 e, p = 2^y.
struct GradCoef {
  float g, gh;
  template <typename T> DM_DEV GradCoef(const LpArgs<T>& a, long r, long target)
      : g(a.g_logp && target >= 0 ? a.g_logp[r] : 0.f), gh(a.g_entropy ? a.g_entropy[r] : 0.f) {}
};
struct RowGrad {
  float M, l2z, a, b, g;
  bool fill;      // every element the same:
  float value;    // 0 or NaN
  DM_DEV float of(float x) const {
    const float y = fmaf(x - M, LOG2E, -l2z), p = __builtin_amdgcn_exp2f(y);
    // p = 0 at -inf. Each product with p for itself: b y would pass fp32's range for a large b, and 0 times it is NaN
    return fmaf(p * b, fmaxf(y, -1e30f), p * a);
  }
  DM_DEV RowGrad(const GradCoef& k, const RowStats& s, bool no_token)
      : M(s.M), l2z(s.log_z * LOG2E), a(-k.g - (k.gh == 0.f ? 0.f : k.gh * s.entropy)), b(-k.gh * LN2), g(k.g) {
    const bool zero = (g == 0.f && k.gh == 0.f) || s.lse == -INF;
    fill = zero || !(fabsf(s.lse) < INF) || (g != 0.f && no_token);
    value = zero ? 0.f : NAN_;
  }
};

// A row in 16-byte vectors: the columns before the first and behind the last whole aligned vector (at most
// 2 (V - 1), one per thread) and the vectors between them.
template <typename T> struct RowSpan {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* x;
  int n, c0, nvec;
  DM_DEV RowSpan(const T* row, int cols) : x(row), n(cols) {
    c0 = min(n, (int)(-(long)(reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (V - 1)));
    nvec = (n - c0) / V;
  }
  DM_DEV int edge_col(int e) const {   // the e-th single column, -1: there is none
    const int c = e < c0 ? e : c0 + nvec * V + (e - c0);
    return c < n ? c : -1;
  }
  DM_DEV int col(int q) const { return c0 + q * V; }
  // vector q0 + lane, q0 the same in every lane: a scalar base and one 32-bit lane offset for all of a thread's loads.
  // ONCE: no kernel of the call reads it again, and it goes past the caches (4096 rows of 32000 bf16: 44 us, kept 49;
  // with the gradient 98 and 107; but 2000 rows of 100003 read twice 236, kept 197)
  template <bool ONCE> DM_DEV u32x4 vec(int q0, int lane) const {
    const auto* p = (const __attribute__((address_space(1))) u32x4*)(reinterpret_cast<const char*>(x + c0 + (long)q0 * V) + 16u * lane);
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return *p;
  }
};
template <typename T> DM_DEV void unpack(const u32x4& r, float* v) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  }
}

// x is computed here, not where it is used (all of a tile's summands would wait in registers until then)
DM_DEV void here(float& x) { asm volatile("" : "+v"(x)); }

// bf16 numbers as 16-bit integers: those >= 0 order as signed ones, above all others; the negative ones as unsigned ones
// the other way round.
typedef short shortx2 __attribute__((ext_vector_type(2)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
DM_DEV shortx2 signed_pair(uint32_t x) { return __builtin_bit_cast(shortx2, x); }
DM_DEV ushortx2 unsigned_pair(uint32_t x) { return __builtin_bit_cast(ushortx2, x); }
DM_DEV float bf16_value(int bits) { return __uint_as_float((uint32_t)bits << 16); }

// A thread's part of one tile of a row: NV vectors and (first tile) one single column, FLOOR where there is none.
template <typename T, int NT, int NV> struct Tile {
  static constexpr int V = RowSpan<T>::V;
  static constexpr uint32_t FILL = sizeof(T) == 2 ? 0xf180f180u : 0xf1800000u;
  u32x4 raw[NV];
  float edge;
  int nv;   // vectors that any of the block's threads has
  template <bool ONCE> DM_DEV void load(const RowSpan<T>& row, int tile) {
    nv = (row.nvec + NT - 1) / NT - tile * NV;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q0 = (tile * NV + i) * NT;
      raw[i] = u32x4{FILL, FILL, FILL, FILL};
      if (q0 + (int)threadIdx.x < row.nvec) raw[i] = row.template vec<ONCE>(q0, threadIdx.x);
    }
    const int c = tile == 0 ? row.edge_col(threadIdx.x) : -1;
    edge = c >= 0 ? to_f(row.x[c]) : FLOOR;
  }
  // vector i's logits, converted where they are used: kept from pass to pass the converted ones would take twice the
  // registers of the row (the statement hides from the compiler that it has converted them before)
  DM_DEV void get(int i, float (&v)[V]) {
    asm volatile("" : "+v"(raw[i]));
    unpack<T>(raw[i], v);
  }
  // the thread's largest logit, FLOOR at least; NaN is passed over or taken
  DM_DEV float largest() {
    float m = fmaxf(edge, FLOOR);
    if constexpr (sizeof(T) == 2) {
      shortx2 p = signed_pair(FILL);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i >= nv) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) p = __builtin_elementwise_max(p, signed_pair(raw[i][j]));
      }
      int best = max((int)p[0], (int)p[1]);
      if (__any(best < 0)) {   // somebody has negative ones only
        ushortx2 u = unsigned_pair(FILL);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (i >= nv) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) u = __builtin_elementwise_min(u, unsigned_pair(raw[i][j]));
        }
        if (best < 0) best = min((int)u[0], (int)u[1]);
      }
      m = fmaxf(m, bf16_value(best));
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i >= nv) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, __uint_as_float(raw[i][j]));
      }
    }
    return m;
  }
  // whether one of a vector's logits may reach `bound`
  DM_DEV bool reaches(int i, float bound) {
    if constexpr (sizeof(T) == 2) {
      if (bound > 0.f) {
        const shortx2 p = __builtin_elementwise_max(__builtin_elementwise_max(signed_pair(raw[i][0]), signed_pair(raw[i][1])),
                                                    __builtin_elementwise_max(signed_pair(raw[i][2]), signed_pair(raw[i][3])));
        return max((int)p[0], (int)p[1]) >= (int)(__float_as_uint(bound) >> 16);   // bound: rounded down to bf16's bits
      }
    }
    float v[V];
    unpack<T>(raw[i], v);
    float m = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = fmaxf(m, v[j]);
    return m >= bound;
  }
};

// A thread's sums over its logits relative to a reference m: with y = x log2 e + c and c = -m log2 e (rounded: it is c
// that counts, so far rows lose nothing), z = sum of 2^y and q = sum of 2^y y.
struct Sums {
  float m, c, z, q;
  DM_DEV Sums() : m(FLOOR), c(-FLOOR * LOG2E), z(0.f), q(0.f) {}
  DM_DEV void refer(float to) {
    const float c1 = -to * LOG2E, d = c1 - c, f = __builtin_amdgcn_exp2f(d);
    q = f > 0.f ? f * (q + z * d) : 0.f;
    z *= f;
    m = to;
    c = c1;
  }
  template <typename T, int NT, int NV> DM_DEV void add(Tile<T, NT, NV>& t) {
    float zt = 0.f, qt = 0.f;
    pass<false>(t, zt, qt);
    if (__any(qt != qt)) {   // -inf among them: 0 times -inf
      zt = qt = 0.f;
      pass<true>(t, zt, qt);
    }
    z += zt;
    q += qt;
  }
  template <bool CLAMP, typename T, int NT, int NV> DM_DEV void pass(Tile<T, NT, NV>& t, float& zt, float& qt) {
    auto one = [&](float x) {
      const float y = fmaf(x, LOG2E, c), e = __builtin_amdgcn_exp2f(y);
      zt += e;
      qt = fmaf(e, CLAMP ? fmaxf(y, -1e30f) : y, qt);
    };
    one(t.edge);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i >= t.nv) continue;
      float v[Tile<T, NT, NV>::V];
      t.get(i, v);
#pragma unroll
      for (int j = 0; j < Tile<T, NT, NV>::V; ++j) one(v[j]);
      here(zt);
      here(qt);
    }
  }
  // the block's sums in every thread
  template <int NT> DM_DEV void join(Shared<NT>& sh) {
    refer(wave_max(m));
    z = wave_sum(z);
    q = wave_sum(q);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) sh.m[wave] = m, sh.z[wave] = z, sh.q[wave] = q;
    __syncthreads();
    const int w = threadIdx.x % (NT / 64);   // each wave's lanes join all waves' sums
    m = sh.m[w], z = sh.z[w], q = sh.q[w];
    c = -m * LOG2E;
    refer(lanes_max<1, NT / 128>(m));
    z = lanes_sum<1, NT / 128>(z);
    q = lanes_sum<1, NT / 128>(q);
  }
};

// A row's statistics element by element: rows with a NaN, +inf, or nothing above FLOOR.
template <typename T, int NT> DM_DEV RowStats slow_stats(const T* x, int n, Shared<NT>& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = -INF;
  int nan = 0;
  for (int i = threadIdx.x; i < n; i += NT) {
    const float v = to_f(x[i]);
    nan |= v != v;
    m = fmaxf(m, v);
  }
  m = wave_max(m);
  __syncthreads();   // the sums in sh have been read
  if (lane == 0) sh.m[wave] = m;
  nan = __syncthreads_or(nan);
  RowStats s;
  s.M = sh.m[0];
  for (int w = 1; w < NT / 64; ++w) s.M = fmaxf(s.M, sh.m[w]);
  if (nan) s.M = NAN_;
  s.lse = s.log_z = s.M;
  s.entropy = s.M == -INF ? 0.f : NAN_;
  if (nan || fabsf(s.M) == INF) return s;
  float z = 0.f, q = 0.f;
  for (int i = threadIdx.x; i < n; i += NT) {
    const float d = to_f(x[i]) - s.M, e = exp_of(d);
    z += e;
    q += e * fmaxf(d, -1e30f);
  }
  z = wave_sum(z);
  q = wave_sum(q);
  if (lane == 0) sh.z[wave] = z, sh.q[wave] = q;
  __syncthreads();
  z = q = 0.f;
  for (int w = 0; w < NT / 64; ++w) z += sh.z[w], q += sh.q[w];
  s.log_z = logf(z);
  s.lse = s.M + s.log_z;
  s.entropy = s.log_z - q / z;
  return s;
}

// The row's `top` largest in order, found one after the other: any row, any values.
template <typename T, int NT> DM_DEV void slow_top(const LpArgs<T>& a, long r, const RowStats& s, Shared<NT>& sh) {
  const T* x = a.x + r * a.ld;
  uint64_t last = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.cols; i += NT) {
      const uint64_t k = order_of(to_f(x[i]), i);
      if (k < last && k > best) best = k;
    }
    best = wave_max_u64(best);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.key[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) best = max(best, sh.key[w]);
    last = best;
    if (threadIdx.x == 0) {
      const int id = ~(uint32_t)best;
      a.top_ids[r * a.top + j] = id;
      a.top_logp[r * a.top + j] = s.logp(to_f(x[id]));
    }
  }
  __syncthreads();   // the row has been read
}

// A bound that at least `top` of the row's logits reach, or the least number: of the 64 lanes' largest logits the top-th.
template <typename T, int NT> DM_DEV float top_bound(int top, const Shared<NT>& sh) {
  float g = -INF;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) g = fmaxf(g, sh.largest[w * 64 + (threadIdx.x & 63)]);
  const uint32_t o = order_of(g);
  uint32_t bound = 0;   // its upper bits: rounded down it lets a few more pass
#pragma unroll
  for (int bit = 31; bit >= (sizeof(T) == 2 ? 16 : 13); --bit) {
    const uint32_t b = bound | 1u << bit;
    if (__popcll(__ballot(o >= b)) >= top) bound = b;
  }
  return bound <= ORDER_OF_MINUS_INF ? -3.402823466e38f : value_of(bound);
}
template <int NT> DM_DEV void take(float x, int col, Shared<NT>& sh) {
  const int at = atomicAdd(&sh.count, 1);
  if (at < CANDIDATES) sh.cand[at] = order_of(x, col);
}
// this tile's logits of at least `bound` (a number) into the list
template <typename T, int NT, int NV> DM_DEV void take_tile(const RowSpan<T>& row, Tile<T, NT, NV>& t, int tile, float bound, Shared<NT>& sh) {
  constexpr int V = RowSpan<T>::V;
  const int c = tile == 0 ? row.edge_col(threadIdx.x) : -1;
  if (c >= 0 && t.edge >= bound) take(t.edge, c, sh);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i >= t.nv) continue;
    const int q = (tile * NV + i) * NT + threadIdx.x;
    if (!t.reaches(i, bound) || q >= row.nvec) continue;
    float v[V];
    t.get(i, v);
    uint32_t hit = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) hit |= v[j] >= bound ? 1u << j : 0u;
    while (hit) {   // one, as a rule
      const int j = __builtin_ctz(hit), k = j * (int)sizeof(T) / 4;
      hit &= hit - 1;
      uint32_t w = t.raw[i][0];
      w = k == 1 ? t.raw[i][1] : w;
      w = k == 2 ? t.raw[i][2] : w;
      w = k == 3 ? t.raw[i][3] : w;
      if constexpr (sizeof(T) == 2) w = j & 1 ? w & 0xffff0000u : w << 16;
      take(__uint_as_float(w), row.col(q) + j, sh);
    }
  }
}
// the c candidates in order; behind them, where they are fewer, the lowest ids of probability 0
template <typename T, int NT> DM_DEV void write_top(const LpArgs<T>& a, long r, const RowStats& s, int c, const Shared<NT>& sh) {
  float* lp = a.top_logp + r * a.top;
  int64_t* ids = a.top_ids + r * a.top;
  for (int i = threadIdx.x; i < c; i += NT) {
    const uint64_t k = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < c; ++j) rank += sh.cand[j] > k;
    if (rank >= a.top) continue;
    ids[rank] = (uint32_t)~(uint32_t)k;
    lp[rank] = s.logp(value_of(k >> 32));
  }
  if (c < a.top && (int)threadIdx.x < a.top) {   // the first `top` columns hold enough of them
    int before = 0;
    bool taken = false;
    for (int j = 0; j < c; ++j) {
      const uint32_t id = ~(uint32_t)sh.cand[j];
      before += id < threadIdx.x;
      taken |= id == threadIdx.x;
    }
    const int at = c + threadIdx.x - before;
    if (!taken && at < a.top) {
      ids[at] = threadIdx.x;
      lp[at] = -INF;
    }
  }
}

// Vector q0 + lane of a row's gradient dx (RowSpan::vec's addressing), element by element where dx lies otherwise in its
// 16 bytes than x.
template <typename T> DM_DEV void store_grad(T* dx, const RowSpan<T>& row, int q0, int lane, const float* v, bool aligned) {
  constexpr int V = RowSpan<T>::V;
  T* p = reinterpret_cast<T*>(reinterpret_cast<char*>(dx + row.c0 + (long)q0 * V) + 16u * lane);
  if (aligned) {
    store_vec_nt<T, V>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = from_f<T>(v[j]);
  }
}
template <typename T> DM_DEV bool same_alignment(const T* dx, const RowSpan<T>& row) {
  return ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(row.x)) & 15) == 0;
}
// the gradient of vector q0 + lane from its logits v
template <typename T>
DM_DEV void grad_vec(T* dx, const RowSpan<T>& row, int q0, int lane, float* v, const RowGrad& w, int target, bool aligned) {
  constexpr int V = RowSpan<T>::V;
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = w.of(v[j]);
  const int at = target - row.col(q0 + lane);
  if ((unsigned)at < (unsigned)V) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += at == j ? w.g : 0.f;
  }
  store_grad(dx, row, q0, lane, v, aligned);
}
template <typename T> DM_DEV void grad_edge(T* dx, int c, float x, const RowGrad& w, int target) {
  if (c >= 0) dx[c] = from_f<T>(w.of(x) + (c == target ? w.g : 0.f));
}
template <typename T, int NT> DM_DEV void fill_row(const RowSpan<T>& row, float value, T* dx) {
  constexpr int V = RowSpan<T>::V;
  float v[V];
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = value;
  for (int q = threadIdx.x; q < row.nvec; q += NT) store_grad(dx, row, 0, q, v, same_alignment(dx, row));
  const int c = row.edge_col(threadIdx.x);
  if (c >= 0) dx[c] = from_f<T>(value);
}
template <typename T, int NT, int NV>
DM_DEV void store_tile(const RowSpan<T>& row, Tile<T, NT, NV>& t, int tile, const RowGrad& w, int target, T* dx) {
  const bool aligned = same_alignment(dx, row);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int q0 = (tile * NV + i) * NT;
    if (i >= t.nv || q0 + (int)threadIdx.x >= row.nvec) continue;
    float v[RowSpan<T>::V];
    t.get(i, v);
    grad_vec(dx, row, q0, threadIdx.x, v, w, target, aligned);
  }
  if (tile == 0) grad_edge(dx, row.edge_col(threadIdx.x), t.edge, w, target);
}

// A block per row, the row in tiles of NT NV vectors held in registers. ONCE: the gradient's rows are one tile.
template <typename T, int NT, int NV, bool GRAD, bool ONCE> __global__ __launch_bounds__(NT, 4) void k_logprob_rows(LpArgs<T> a) {
  __shared__ Shared<NT> sh;
  for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const RowSpan<T> row(a.x + r * a.ld, a.cols);
    // (also where it is 1: known to be, the row's values would be kept converted between the passes, and spilled)
    const int tiles = max(1, (row.nvec + NT * NV - 1) / (NT * NV));
    const long t = a.target ? a.target[r] : -1;
    const float xt = t >= 0 && t < a.cols ? to_f(row.x[t]) : 0.f;
    const GradCoef coef(a, r, t);   // (null without a gradient)
    Sums u;
    Tile<T, NT, NV> tile;
    if (a.top && threadIdx.x == 0) sh.count = 0;
    for (int i = 0; i < tiles; ++i) {
      tile.template load<ONCE>(row, i);
      u.refer(fmaxf(u.m, tile.largest()));
      u.add(tile);
      if (a.top) {   // the bound only rises from tile to tile
        sh.largest[threadIdx.x] = u.m > FLOOR ? u.m : -INF;
        __syncthreads();
        take_tile(row, tile, i, top_bound<T>(a.top, sh), sh);
        if (i + 1 < tiles) __syncthreads();
      }
    }
    u.join(sh);
    RowStats s;
    const bool slow = !(u.z > 0.f && u.z < INF) || u.m <= FLOOR;
    if (slow) {
      s = slow_stats<T, NT>(row.x, a.cols, sh);
    } else {
      s.M = u.m;
      const float l2 = __builtin_amdgcn_logf(u.z), shift = fmaf(u.m, LOG2E, u.c);   // what c's rounding left
      // neither is below 0 but for the roundings of the two instructions, where one token has all of the probability
      s.log_z = fmaxf((l2 - shift) * LN2, 0.f);
      s.lse = s.M + s.log_z;
      s.entropy = fmaxf((l2 - u.q / u.z) * LN2, 0.f);
    }
    if (threadIdx.x == 0) {
      if (a.logp) a.logp[r] = t < 0 ? 0.f : t < a.cols ? s.logp(xt) : NAN_;
      if (a.lse) a.lse[r] = s.lse;
      if (a.entropy) a.entropy[r] = s.entropy;
      if (a.stats) a.stats[3 * r] = s.M, a.stats[3 * r + 1] = s.log_z, a.stats[3 * r + 2] = s.entropy;
    }
    if (a.top) {
      const int c = sh.count;
      if (slow || c > CANDIDATES) slow_top<T, NT>(a, r, s, sh);
      else write_top<T, NT>(a, r, s, c, sh);
    }
    if constexpr (GRAD) {
      const RowGrad w(coef, s, t >= a.cols);
      const int target = t < a.cols ? (int)t : -1;
      T* dx = a.dx + r * a.ld_d;
      if (w.fill) {
        fill_row<T, NT>(row, w.value, dx);
      } else {
        for (int i = 0; i < tiles; ++i) {
          if (!ONCE) tile.template load<true>(row, i);
          store_tile(row, tile, i, w, target, dx);
        }
      }
    }
    __syncthreads();   // sh is free again
  }
}

// The gradient after the forward, element by element. NT threads per part of a row, NV vectors each; 256 / NT parts per
// block. Bound by reading the logits and writing the gradient: 999 rows of 50257 bf16, 201 MB, 39 us (5.2 TB/s).
template <typename T, int NT, int NV> __global__ __launch_bounds__(256) void k_logprob_bwd(LpArgs<T> a, int parts) {
  const long items = (long)a.rows * parts;
  for (long it = blockIdx.x * (256L / NT) + threadIdx.x / NT; it < items; it += gridDim.x * (256L / NT)) {
    const long r = it / parts;
    const int q0 = (int)(it % parts) * NT * NV + threadIdx.x % NT;
    RowStats s;
    s.M = a.stats[3 * r];
    s.log_z = a.stats[3 * r + 1];
    s.entropy = a.stats[3 * r + 2];
    s.lse = s.M + s.log_z;
    const long t = a.target ? a.target[r] : -1;
    const RowGrad w(GradCoef(a, r, t), s, t >= a.cols);
    const int target = t < a.cols ? (int)t : -1;
    const RowSpan<T> row(a.x + r * a.ld, a.cols);
    T* dx = a.dx + r * a.ld_d;
    const bool aligned = same_alignment(dx, row);
    u32x4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[i] = u32x4{0, 0, 0, 0};
      if (!w.fill && q0 + i * NT < row.nvec) raw[i] = row.template vec<true>(0, q0 + i * NT);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = q0 + i * NT;
      if (q >= row.nvec) continue;
      float v[RowSpan<T>::V];
      unpack<T>(raw[i], v);
      if (w.fill) {
#pragma unroll
        for (int j = 0; j < RowSpan<T>::V; ++j) v[j] = w.value;
        store_grad(dx, row, 0, q, v, aligned);
      } else {
        grad_vec(dx, row, 0, q, v, w, target, aligned);
      }
    }
    const int c = it % parts == 0 ? row.edge_col(q0) : -1;
    if (c >= 0 && w.fill) dx[c] = from_f<T>(w.value);
    else if (c >= 0) grad_edge(dx, c, to_f(row.x[c]), w, target);
  }
}

constexpr int MAX_COLS = DM_LOGPROB_COLS;   // a row's bytes in 32 bits
constexpr int MAX_BLOCKS = 1 << 20;   // of a grid; further rows by the same blocks

template <typename T> LpArgs<T> typed(const dm_logprob_args* a) {
  return {(const T*)a->logits, (T*)a->dlogits, a->target, a->logp, a->lse, a->entropy, a->stats, a->top_logp,
          a->top_ids, a->g_logp, a->g_entropy, a->ld, a->ld_d, a->rows, a->cols, a->top};
}

template <bool GRAD, typename T, int NT, int NV, bool ONCE = true> void launch_rows(const LpArgs<T>& a, hipStream_t s) {
  hipLaunchKernelGGL((k_logprob_rows<T, NT, NV, GRAD, ONCE>), dim3(std::min(a.rows, MAX_BLOCKS)), dim3(NT), 0, s, a);
}
// The threads of a row and their vectors per tile, by the row's 16-byte vectors (bf16: 8 logits, fp32: 4).
// Fewer rows than CUs: as many threads as a block has, since nothing else hides a row's latencies (one row of 32000 bf16
// with 5 alternatives 7.0 us, at 256 threads 9.6; without them 4.9, where a block of so many threads takes 3.8 for a row
// of 8). Up to a row per CU that is faster, from two on the CU's other blocks hide them better: 1024 and 256 threads take
// for 64, 255, 320, 1000 rows of 50257 bf16 7.5 / 9.8, 8.6 / 11.1, 14.2 / 12.3, 29 / 21 us, with 8 alternatives 10.4 / 17.5,
// 11.6 / 18.4, 19.8 / 20.3, 40 / 28; of 12000 bf16 4.7 / 4.5, 5.1 / 4.8, 8.0 / 5.7, 15 / 8. Several blocks per row have not
// been tried: joined by a second launch they would cost that launch.
// Otherwise the smallest blocks that fill a CU's memory pipes while others of the CU wait at their barriers (4096 rows of
// 32000 bf16: 64 threads of 4 vectors 47 us, 256 of 8 44, 1024 of 4 72). With the gradient a row is best read once and
// held until it is written (the same rows: 256 threads of 16 vectors, all of a row, 98 us; of 8 vectors, read twice,
// 114); rows past 65536 fp32 or 131072 bf16 are read twice (2000 rows of 100003 bf16: 186 us held, 197 read twice).
template <typename T> void run_rows(const LpArgs<T>& a, hipStream_t s) {
  const int nvec = cdiv(a.cols, RowSpan<T>::V);
  const bool few = a.rows < 256 && nvec > 256 * 4;
  if (!a.dx) {
    if (nvec <= 64 * 4) launch_rows<false, T, 64, 4>(a, s);
    else if (nvec <= 256 * 4) launch_rows<false, T, 256, 4>(a, s);
    else if (!few) launch_rows<false, T, 256, 8>(a, s);
    else if (nvec <= 1024 * 4) launch_rows<false, T, 1024, 4>(a, s);
    else launch_rows<false, T, 1024, 16>(a, s);
  } else {
    if (nvec <= 64 * 4) launch_rows<true, T, 64, 4>(a, s);
    else if (nvec <= 64 * 8) launch_rows<true, T, 64, 8>(a, s);
    else if (nvec <= 256 * 4) launch_rows<true, T, 256, 4>(a, s);
    else if (few && nvec <= 1024 * 4) launch_rows<true, T, 1024, 4>(a, s);
    else if (nvec <= 256 * 16) launch_rows<true, T, 256, 16>(a, s);
    else if (!few && nvec <= 512 * 16) launch_rows<true, T, 512, 16>(a, s);
    else if (nvec <= 1024 * 16) launch_rows<true, T, 1024, 16>(a, s);
    else launch_rows<true, T, 1024, 16, false>(a, s);
  }
}
template <typename T> void run_bwd(const LpArgs<T>& a, hipStream_t s) {
  const int nvec = cdiv(a.cols, RowSpan<T>::V);
  auto go = [&](auto kernel, int nt, int nv) {
    const int parts = cdiv(nvec, nt * nv);
    const long items = (long)a.rows * parts;
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<long>((items + 256 / nt - 1) / (256 / nt), MAX_BLOCKS)), dim3(256), 0, s, a, parts);
  };
  if (nvec <= 64 * 4) go(k_logprob_bwd<T, 64, 4>, 64, 4);
  else go(k_logprob_bwd<T, 256, 4>, 256, 4);
}

bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// whether what a call writes lies in anything else that it reads or writes (dlogits in the logits' place aside)
bool outputs_overlap(const dm_logprob_args* a, bool bwd) {
  typedef unsigned __int128 wide;
  struct Range {
    const void* p;
    wide bytes;
  };
  const wide n = a->rows, e = esz(a->dtype);
  const bool in_place = a->dlogits == a->logits && a->ld_d == a->ld;
  const Range out[] = {{in_place ? nullptr : a->dlogits, ((n - 1) * a->ld_d + a->cols) * e}, {bwd ? nullptr : a->logp, n * 4},
                       {bwd ? nullptr : a->lse, n * 4}, {bwd ? nullptr : a->entropy, n * 4}, {bwd ? nullptr : a->stats, n * 12},
                       {bwd || !a->top ? nullptr : a->top_logp, n * a->top * 4}, {bwd || !a->top ? nullptr : a->top_ids, n * a->top * 8}};
  const Range in[] = {{a->logits, ((n - 1) * a->ld + a->cols) * e}, {a->target, n * 8}, {a->dlogits ? a->g_logp : nullptr, n * 4},
                      {a->dlogits ? a->g_entropy : nullptr, n * 4}, {bwd ? a->stats : nullptr, n * 12}};
  auto meet = [](const Range& r, const Range& s) {
    const wide p = reinterpret_cast<uintptr_t>(r.p), q = reinterpret_cast<uintptr_t>(s.p);
    return p && q && p < q + s.bytes && q < p + r.bytes;
  };
  // rows of one stride side by side: the gradient's columns in the gaps of the logits'
  const wide row = a->ld * e, used = a->cols * e;
  const wide gap = a->dlogits && a->ld_d == a->ld
                       ? ((wide)reinterpret_cast<uintptr_t>(a->dlogits) + ((wide)1 << 100) * row - reinterpret_cast<uintptr_t>(a->logits)) % row
                       : 0;
  const bool beside = gap >= used && gap + used <= row;
  for (const Range& r : out) {
    for (const Range& s : in)
      if (meet(r, s) && !(beside && &r == out && &s == in)) return true;
    for (const Range& s : out)
      if (&s != &r && meet(r, s)) return true;
  }
  // written over the logits, the gradient meets the other inputs and outputs where the logits do
  if (in_place)
    for (const Range& s : in)
      if (&s != in && meet(in[0], s)) return true;
  return false;
}

// what both entry points ask of their arguments
int check_logprob(const dm_logprob_args* a, bool bwd) {
  DM_REQUIRE(a != nullptr, DM_ERR_INVALID, "null arguments");
  DM_REQUIRE(a->dtype == DM_BF16 || a->dtype == DM_F32, DM_ERR_INVALID, "dtype %d", a->dtype);
  DM_REQUIRE(a->rows >= 0 && a->cols > 0 && a->cols <= MAX_COLS && a->ld >= a->cols, DM_ERR_INVALID,
             "rows=%d cols=%d ld=%lld (at most %d columns)", a->rows, a->cols, (long long)a->ld, MAX_COLS);
  if (a->rows == 0) return DM_OK;
  const size_t e = esz(a->dtype);
  DM_REQUIRE(a->logits && aligned_to(a->logits, e), DM_ERR_INVALID, "null or unaligned logits");
  DM_REQUIRE(!a->logp || a->target, DM_ERR_INVALID, "logp without targets");
  if (!bwd) {
    DM_REQUIRE(a->top >= 0 && a->top <= DM_TOP_MAX && a->top <= a->cols, DM_ERR_INVALID, "top=%d of cols=%d (at most %d)",
               a->top, a->cols, DM_TOP_MAX);
    DM_REQUIRE(a->top == 0 || (a->top_logp && a->top_ids), DM_ERR_INVALID, "null output of the most likely tokens");
  }
  if (bwd || a->dlogits) {
    DM_REQUIRE(a->dlogits && aligned_to(a->dlogits, e) && a->ld_d >= a->cols, DM_ERR_INVALID, "null or unaligned dlogits, ld_d=%lld",
               (long long)a->ld_d);
    DM_REQUIRE(a->g_logp || a->g_entropy, DM_ERR_INVALID, "a gradient without coefficients");
    DM_REQUIRE(!a->g_logp || a->target, DM_ERR_INVALID, "g_logp without targets");
    DM_REQUIRE(!bwd || a->stats, DM_ERR_INVALID, "the forward's stats are needed");
  }
  DM_REQUIRE(!outputs_overlap(a, bwd), DM_ERR_INVALID, "an output overlaps an input or another output");
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
