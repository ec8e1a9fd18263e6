// Drafted tokens against the target's probabilities, from given random numbers (dm_verify_drafts).
//
// A sequence's rows of logits x (target) and y (draft) are distributions p and q at its temperature T; the draft d of a row
// is accepted where u0 q(d) < p(d), and the first row without an accepted draft gets a token by its place u1 in the sums of
// r = max(p - q, 0) (of p where nothing was drafted, or r is 0). Whether a number falls on this or that side of a sum of
// 10^5 probabilities is decided in 64 bits throughout: exponentials, their sums and the places.
#include "dm_common.h"
#include "dm_error.h"

#include <algorithm>

using namespace dm;

namespace {

constexpr float INF = __builtin_inff(), NAN_ = __builtin_nanf("");
constexpr int PART = 4096;      // columns of a block's part of a row

// 2^(w / 32) for w <= 0 (w = 32 x / (T ln 2) for e^(x / T), x a difference of logits) to within a few units of 2^-53: 2^(n / 32)
// 2^(f / 32) with n the nearest whole number to w, the 32 roots from a table in LDS (one in each pair of its banks), and for 2^(f / 32)
// its Taylor sum up to f^6 with that term spread over f^2 and f^4 (less the Chebyshev polynomial of its degree: |f| <= 1/2 leaves
// 1.4e-16). With f^4 for the last term 1.3e-12 was left, and drafts and places as near as that to their border were decided
// wrongly (one more instruction: 64 sequences of up to 8 fp32 rows of 50257 51.3 -> 52.1 us a call). Little more than half of the
// instructions of the library's
// function, whose range is not needed here. Below 2^-1000 it stays there, which a sum of at least 1 does not see;
// a probability is 0 there (prob_of). No NaN.
__constant__ const double ROOTS[32] = {      // 2^(i / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
constexpr int LEAST = 1000;
struct Roots {
  double v[32];            // 2^(i / 32 - LEAST)
  DM_DEV void fill() {     // a barrier has to follow
    if (threadIdx.x < 32) v[threadIdx.x] = ROOTS[threadIdx.x] * 0x1p-1000;
  }
};
DM_DEV double scale_of(double T) { return 32.0 / (T * 0.6931471805599453); }
DM_DEV double exp_of(double w, const Roots& roots) {
  constexpr double SHIFT = 0x1.8p52 + 32 * LEAST;      // the sum with it holds n + 32 LEAST in its low bits
  w = fmax(w, -32.0 * LEAST);
  const double big = w + SHIFT, f = w - (big - SHIFT);
  double e = fma(f, 3.973709984549416e-11, 9.172616498033084e-09);
  e = fma(e, f, 1.693850972437182e-06);
  e = fma(e, f, 0.0002345961981972034);
  e = fma(e, f, 0.02166084939249829);
  e = fma(e, f, 1.0);
  const uint32_t k = (uint32_t)__double_as_longlong(big);
  const uint64_t root = (uint64_t)__double_as_longlong(roots.v[k & 31]);
  return e * __longlong_as_double((long long)(root + ((uint64_t)(k >> 5) << 52)));
}

// ... as a probability: 0 below 2^-1000, and of a logit of -inf
DM_DEV double prob_of(double w, const Roots& roots) { return w > -32.0 * LEAST ? exp_of(w, roots) : 0.0; }

// A part's sum of exp((x - m) / T) relative to its own maximum, with the first place of that; m is NaN where the part holds
// one.
struct Part {
  double z;
  float m;
  int arg;
};
// What a sequence's rows say: the row that gets a new token, and how.
struct Choice {
  double zp, zq;      // sums of exponentials of its target and draft rows (zq 0: p alone)
  float mp, mq;       // their maxima
  int row;            // token row
  int drop;           // a column that counts 0 (the draft without a distribution), -1: none
  int token;          // -2: to be drawn; else there is nothing more to do
  double scale, T;    // scale_of its temperature, and that
  double log_zp;
  float u;            // its place
};

struct VerifyArgs {
  const void *x, *y;
  const int64_t* ids;
  const float *u, *temperature;
  const int32_t* starts;
  int64_t* tokens;
  int32_t* accepted;
  float* logp;
  Part* parts;        // [2][N][n_parts]
  double* sums;       // [B][2][n_parts]: of r and of p, over the chosen row's parts
  Choice* choice;     // [B]
  long ld_x, ld_y;
  int N, B, V, n_parts;
};

struct Rows {
  int first, n;
  DM_DEV Rows(const VerifyArgs& a, int b) {
    first = min(max(a.starts[b], 0), a.N);
    n = min(max(a.starts[b + 1], first), a.N) - first;
  }
};

// The sequence of token row t, the same in all lanes of a wave; -1: none.
DM_DEV int sequence_of(const VerifyArgs& a, int t) {
  int n = 0;     // sequences that start at t or before
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + (threadIdx.x & 63);
    n += __popcll(__ballot(b < a.B && a.starts[b] <= t));
  }
  if (n == 0) return -1;
  const Rows r(a, n - 1);
  return t >= r.first && t < r.first + r.n ? n - 1 : -1;
}
// a temperature of 0 is greedy; the log probabilities are those at 1 then
DM_DEV double divisor(float T) { return T == 0.f ? 1.0 : (double)T; }

// sums and minima over a wave without the LDS crossbar (lane_pair)
template <int O> DM_DEV double pair_sum(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const LanePair lo = lane_pair<O>(__uint_as_float((uint32_t)u)), hi = lane_pair<O>(__uint_as_float((uint32_t)(u >> 32)));
  const auto join = [](float l, float h) { return __longlong_as_double((long long)((uint64_t)__float_as_uint(h) << 32 | __float_as_uint(l))); };
  return join(lo.a, hi.a) + join(lo.b, hi.b);
}
DM_DEV double wave_sum_double(double v) {
  return pair_sum<32>(pair_sum<16>(pair_sum<8>(pair_sum<4>(pair_sum<2>(pair_sum<1>(v))))));
}
template <int O> DM_DEV int pair_min(int v) {
  const LanePair p = lane_pair<O>(__uint_as_float((uint32_t)v));
  return min((int)__float_as_uint(p.a), (int)__float_as_uint(p.b));
}
DM_DEV int wave_min(int v) { return pair_min<32>(pair_min<16>(pair_min<8>(pair_min<4>(pair_min<2>(pair_min<1>(v)))))); }

// N elements from column c on; -inf behind the row. Rows have their elements' alignment only.
template <typename T, int N> DM_DEV void load_columns(const T* x, int c, int cols, float (&v)[N]) {
  constexpr int V = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += V) {
    if (c + i + V <= cols) {
      const auto r = ld_global_a<typename RawV<T, V>::type, (int)sizeof(T)>(x + c + i);
      float u[V];
      unpackv<T, V>(r, u);
#pragma unroll
      for (int e = 0; e < V; ++e) v[i + e] = u[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[i + e] = c + i + e < cols ? to_f(x[c + i + e]) : -INF;
    }
  }
}

// One block per row and part of it, of the target and of the draft (blockIdx.z): 64 sequences of 1 to 8 rows of 50257 in fp32, target
// and draft (108 MB), 30.6 us, 3.5 TB/s; 48 of 1 to 6 rows of 100003 in bf16, target alone (35 MB), 21. Bound by the rows first, which
// take 20 and 12 us of that without any exponentials, then by those in 64 bits (21 instructions each).
template <typename T> __global__ __launch_bounds__(256) void k_verify_parts(VerifyArgs a) {
  constexpr int V = 16 / (int)sizeof(T), EACH = PART / 256;
  __shared__ Roots roots;
  __shared__ float sm[4];
  __shared__ double sz[4];
  __shared__ int sarg[4], snan[4];
  const int t = blockIdx.y, c0 = blockIdx.x * PART, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool draft = blockIdx.z;
  const T* x = draft ? (const T*)a.y + t * a.ld_y : (const T*)a.x + t * a.ld_x;
  float v[EACH / V][V];
#pragma unroll
  for (int i = 0; i < EACH / V; ++i) load_columns(x, c0 + (threadIdx.x + 256 * i) * V, a.V, v[i]);
  const int b = sequence_of(a, t);
  if (b < 0) return;
  const Rows rows(a, b);
  const float temperature = a.temperature[b];
  if (draft && (t == rows.first + rows.n - 1 || temperature == 0.f)) return;
  const double scale = scale_of(divisor(temperature));
  roots.fill();
  float m = -INF;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    m = fmaxf(m, v[i / V][i % V]);
    nan |= v[i / V][i % V] != v[i / V][i % V];
  }
  m = wave_max(m);
  nan = __ballot(nan) != 0;
  if (lane == 0) sm[wave] = m, snan[wave] = nan;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  // the difference first: at a temperature of 10^-6 a product's rounding would be as large as the logits' steps
  const double top = m == -INF ? 0.0 : (double)m;
  double z = 0.0;
  int arg = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < EACH; ++i) z += exp_of(((double)v[i / V][i % V] - top) * scale, roots);
  z = m == -INF ? 0.0 : wave_sum_double(z);
  if (temperature == 0.f) {
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (v[i / V][i % V] == m) arg = min(arg, c0 + ((int)threadIdx.x + 256 * (i / V)) * V + i % V);
    arg = wave_min(arg);
  }
  if (lane == 0) sz[wave] = z, sarg[wave] = arg;
  __syncthreads();
  if (threadIdx.x) return;
  Part p;
  p.z = (sz[0] + sz[1]) + (sz[2] + sz[3]);
  p.m = snan[0] | snan[1] | snan[2] | snan[3] ? NAN_ : m;
  p.arg = min(min(sarg[0], sarg[1]), min(sarg[2], sarg[3]));
  a.parts[((long)draft * a.N + t) * a.n_parts + blockIdx.x] = p;
}

// A row's parts joined by a wave: the maximum (NaN if there is one), the sum relative to it and the first place of it.
DM_DEV Part join_parts(const VerifyArgs& a, bool draft, int t, double scale, const Roots& roots) {
  const Part* p = a.parts + ((long)draft * a.N + t) * a.n_parts;
  const int lane = threadIdx.x & 63;
  float m = -INF;
  bool nan = false;
  for (int i = lane; i < a.n_parts; i += 64) {
    m = fmaxf(m, p[i].m);
    nan |= p[i].m != p[i].m;
  }
  m = wave_max(m);
  double z = 0.0;
  int arg = 0x7fffffff;
  for (int i = lane; i < a.n_parts; i += 64) {
    if (p[i].m == m) arg = min(arg, p[i].arg);
    z += p[i].z * (p[i].m == -INF ? 0.0 : exp_of(((double)p[i].m - m) * scale, roots));
  }
  Part r;
  r.z = wave_sum_double(z);
  r.arg = wave_min(arg);
  r.m = __ballot(nan) ? NAN_ : m;
  return r;
}
// whether a number is a temperature
DM_DEV bool is_temperature(float T) { return T >= 0.f && T < INF; }
// whether the parts are those of a distribution: something finite, no NaN, no +inf
DM_DEV bool is_distribution(const Part& p) { return fabsf(p.m) < INF; }

// 4 columns of the chosen row's p, and r
template <typename T> struct Residual {
  float x[4];
  double p[4], r[4];
  DM_DEV Residual(const VerifyArgs& a, const Choice& ch, int c, const Roots& roots) {
    float y[4];
    load_columns((const T*)a.x + ch.row * a.ld_x, c, a.V, x);
    if (ch.zq > 0.0) load_columns((const T*)a.y + ch.row * a.ld_y, c, a.V, y);
    const double ip = 1.0 / ch.zp, iq = ch.zq > 0.0 ? 1.0 / ch.zq : 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = prob_of(((double)x[i] - ch.mp) * ch.scale, roots) * ip;
      const double q = ch.zq > 0.0 ? prob_of(((double)y[i] - ch.mq) * ch.scale, roots) * iq : 0.0;
      r[i] = c + i == ch.drop ? 0.0 : fmax(p[i] - q, 0.0);
    }
  }
};

struct Deciding {
  Part p[16], q[16];
  bool refused[16];
  Choice choice;
};

// A block decides over a sequence's rows (a wave each, 16 at a time); writes: and writes what is decided.
template <typename T> DM_DEV void decide(const VerifyArgs& a, int b, bool writes, const Roots& roots, Deciding& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float temperature = a.temperature[b];
  const Rows rows(a, b);
  if (rows.n == 0) {
    if (threadIdx.x == 0) {
      sh.choice.token = -1;
      if (writes) a.accepted[b] = 0, a.choice[b].token = -1;
    }
    return;
  }
  const double by = divisor(temperature), scale = scale_of(by);
  const bool greedy = temperature == 0.f;
  int end = 0, i0 = 0;
  for (;; i0 += 16) {      // the last row takes no draft, so one of them ends it
    const int i = i0 + wave;
    if (i < rows.n) {
      const int t = rows.first + i;
      const bool last = i == rows.n - 1, with_q = !last && a.y && !greedy;
      const long d = last ? -1 : a.ids[t + 1];
      const float u = a.u[2 * t];
      const bool in_range = d >= 0 && d < a.V;
      const float xd = in_range ? to_f(((const T*)a.x)[t * a.ld_x + d]) : 0.f;
      const float yd = in_range && with_q ? to_f(((const T*)a.y)[t * a.ld_y + d]) : 0.f;
      const Part p = join_parts(a, false, t, scale, roots);
      Part q;
      q.z = 0.0, q.m = 0.f, q.arg = 0;
      if (with_q) q = join_parts(a, true, t, scale, roots);
      const bool valid = is_temperature(temperature) && is_distribution(p) && is_distribution(q);
      bool ok = false;
      if (greedy) {
        ok = !last && d == p.arg && p.m == p.m && p.m > -INF;
      } else if (valid && in_range) {
        const double qd = !with_q ? 1.0 : prob_of(((double)yd - q.m) * scale, roots) / q.z;
        ok = (double)u * qd < prob_of(((double)xd - p.m) * scale, roots) / p.z;
      }
      if (lane == 0) {
        sh.p[wave] = p, sh.q[wave] = q;
        sh.refused[wave] = !ok;
        if (ok && writes) a.tokens[t] = d, a.logp[t] = valid ? (float)(((double)xd - p.m) / by - log(p.z)) : NAN_;
      }
    }
    __syncthreads();
    const uint64_t first = __ballot(lane < 16 && i0 + lane < rows.n && sh.refused[lane & 15]);
    if (first) {
      end = i0 + __ffsll((unsigned long long)first) - 1;
      break;
    }
    __syncthreads();
  }
  const int t = rows.first + end;
  if (threadIdx.x == 0) {
    const bool last = end == rows.n - 1;
    const Part p = sh.p[end - i0], q = sh.q[end - i0];
    Choice ch;
    ch.zp = p.z, ch.zq = q.z, ch.mp = p.m, ch.mq = q.m, ch.row = t, ch.scale = scale, ch.u = a.u[2 * t + 1];
    ch.drop = last || a.y ? -1 : (int)max(-1l, min((long)a.ids[t + 1], 0x7fffffffl));
    ch.token = greedy ? (p.m == p.m && p.m > -INF ? p.arg : -1) : is_temperature(temperature) && is_distribution(p) && is_distribution(q) ? -2 : -1;
    ch.T = by, ch.log_zp = log(p.z);
    sh.choice = ch;
    if (writes) {
      a.choice[b] = ch;
      a.accepted[b] = end;
      if (ch.token != -2) a.tokens[t] = ch.token, a.logp[t] = ch.token >= 0 && is_distribution(p) ? (float)-ch.log_zp : NAN_;
    }
  }
  if (writes)
    for (int i = end + 1 + threadIdx.x; i < rows.n; i += 1024) a.tokens[rows.first + i] = -1, a.logp[rows.first + i] = 0.f;
}

// The sums of r and p over part `part` of the chosen row, by a block, into a.sums.
template <typename T> DM_DEV void sum_part(const VerifyArgs& a, const Choice& ch, int b, int part, const Roots& roots, double (&sums)[2][16]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Residual<T> v(a, ch, part * PART + threadIdx.x * 4, roots);
  const double r = wave_sum_double((v.r[0] + v.r[1]) + (v.r[2] + v.r[3])), s = wave_sum_double((v.p[0] + v.p[1]) + (v.p[2] + v.p[3]));
  if (lane == 0) sums[0][wave] = r, sums[1][wave] = s;
  __syncthreads();
  if (threadIdx.x < 2) {
    double sum = 0.0;
    for (int w = 0; w < 16; ++w) sum += sums[threadIdx.x][w];
    a.sums[((long)b * 2 + threadIdx.x) * a.n_parts + part] = sum;
  }
}

// The sums of r and p over each part of a sequence's chosen row, as in k_verify_parts bound by the exponentials. DECIDE: each block
// decides over the sequence by itself, a launch less (one sequence of 4 drafts 8.5 us, 5.5 and 5.1 apart; 64 of 13 parts 26, 6.4
// and 8.4 apart).
template <typename T, bool DECIDE> __global__ __launch_bounds__(1024) void k_verify_sums(VerifyArgs a) {
  const int b = blockIdx.y;
  __shared__ Roots roots;
  __shared__ double sums[2][16];
  __shared__ Deciding sh;
  roots.fill();
  __syncthreads();
  if constexpr (DECIDE) {
    decide<T>(a, b, blockIdx.x == 0, roots, sh);
    __syncthreads();
  }
  const Choice ch = DECIDE ? sh.choice : a.choice[b];
  if (ch.token != -2 || (!DECIDE && ch.zq == 0.0)) return;
  sum_part<T>(a, ch, b, blockIdx.x, roots, sums);
}

// the sum over the lanes up to this one, by moves inside the rows of 16 lanes and broadcasts of the rows' last lanes
template <int CTRL, int ROWS> DM_DEV double moved(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
DM_DEV double wave_upto(double v) {
  v += moved<0x111, 0xf>(v);     // row_shr 1, 2, 4, 8
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);     // row_bcast 15, 31
  v += moved<0x143, 0xc>(v);
  return v;
}

// A block: the part of the chosen row in which the place lies, then the thread, then the column. ahead: the first wave's sums of r
// of parts 0 .. 63. Bound by latency: the sums, then the part's logits.
struct Picking {
  double base, place, sums[16];
  int part, plain, hit[16], most[16];
};
template <typename T> DM_DEV void pick(const VerifyArgs& a, const Choice& ch, const double* sums_of, double ahead, const Roots& roots, Picking& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave == 0) {
    const double* s = sums_of;
    double total = 0.0;
    for (int kind = 0; kind < 2; ++kind) {      // r, and p where r is 0
      if (kind) s += a.n_parts;
      total = kind ? (lane < a.n_parts ? s[lane] : 0.0) : ahead;
      for (int i = lane + 64; i < a.n_parts; i += 64) total += s[i];
      total = wave_sum_double(total);
      if (lane == 0) sh.plain = kind;
      if (total > 0.0) break;
    }
    const double to = (double)ch.u * total;
    // the part in which the sum passes the place; by rounding none: the last part with any
    double before = 0.0, found_base = 0.0;
    int found = -1, any = 0;
    double any_base = 0.0;
    for (int i0 = 0; i0 < a.n_parts && found < 0; i0 += 64) {
      const int i = i0 + lane;
      const double mine = s == sums_of && i0 == 0 ? ahead : i < a.n_parts ? s[i] : 0.0, upto = before + wave_upto(mine);
      const uint64_t over = __ballot(mine > 0.0 && upto > to), some = __ballot(mine > 0.0);
      if (some) {
        const int l = 63 - __clzll((long long)some);
        any = i0 + l, any_base = __shfl(upto - mine, l, 64);
      }
      if (over) {
        const int l = __ffsll((unsigned long long)over) - 1;
        found = i0 + l, found_base = __shfl(upto - mine, l, 64);
      }
      before = __shfl(upto, 63, 64);
    }
    if (lane == 0) {
      sh.part = found < 0 ? any : found;
      sh.base = found < 0 ? any_base : found_base;
      sh.place = to;
    }
  }
  __syncthreads();
  const int c0 = sh.part * PART + threadIdx.x * 4;
  const Residual<T> v(a, ch, c0, roots);
  double r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = sh.plain ? v.p[i] : v.r[i];
  const double mine = (r[0] + r[1]) + (r[2] + r[3]), upto = wave_upto(mine);
  if (lane == 63) sh.sums[wave] = upto;
  __syncthreads();
  double before = sh.base;
  for (int w = 0; w < wave; ++w) before += sh.sums[w];
  before += upto - mine;
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    before += r[i];
    if (r[i] > 0.0) last = c0 + i;
    if (before > sh.place && r[i] > 0.0) first = min(first, c0 + i);
  }
  // columns ascend with the lanes and the waves
  const uint64_t hits = __ballot(first != 0x7fffffff), some = __ballot(last >= 0);
  if (hits && lane == __ffsll((unsigned long long)hits) - 1) sh.hit[wave] = first;
  else if (!hits && lane == 0) sh.hit[wave] = -1;
  if (some && lane == 63 - __clzll((long long)some)) sh.most[wave] = last;
  else if (!some && lane == 0) sh.most[wave] = -1;
  __syncthreads();
  int token = -1;
#pragma unroll
  for (int w = 0; w < 16; ++w)
    if (sh.most[w] >= 0) token = sh.most[w];
#pragma unroll
  for (int w = 15; w >= 0; --w)
    if (sh.hit[w] >= 0) token = sh.hit[w];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c0 + i == token) a.tokens[ch.row] = token, a.logp[ch.row] = (float)(((double)v.x[i] - ch.mp) / ch.T - ch.log_zp);
  if (token < 0 && threadIdx.x == 0) a.tokens[ch.row] = -1, a.logp[ch.row] = NAN_;
}
// blocks from the sequences' number on: 16 rows each, of which those of no sequence get token -1
DM_DEV bool rows_of_none(const VerifyArgs& a) {
  if ((int)blockIdx.x < a.B) return false;
  const int t = ((int)blockIdx.x - a.B) * 16 + (threadIdx.x >> 6);
  if (t < a.N && sequence_of(a, t) < 0 && (threadIdx.x & 63) == 0) a.tokens[t] = -1, a.logp[t] = 0.f;
  return true;
}

// A sequence per block, 5 to 7 us at any size.
template <typename T> __global__ __launch_bounds__(1024) void k_verify_pick(VerifyArgs a) {
  if (rows_of_none(a)) return;
  __shared__ Roots roots;
  __shared__ Picking sh;
  const double* sums_of = a.sums + (long)blockIdx.x * 2 * a.n_parts;
  const double ahead = threadIdx.x < 64 && (int)threadIdx.x < a.n_parts ? sums_of[threadIdx.x] : 0.0;      // beside the choice
  const Choice ch = a.choice[blockIdx.x];
  if (ch.token != -2) return;
  roots.fill();
  __syncthreads();
  pick<T>(a, ch, sums_of, ahead, roots, sh);
}

// A sequence per block. Where no draft distribution is subtracted, the chosen row's sums are those of its parts, but for the
// part of a draft that counts 0: written here, so that only a call with draft distributions takes a launch for them (48
// sequences, rows of 100003 in bf16: 6.4 us for 4.8 and 10.3 apart). PICK (a call without them): the token too (10.0 us; 6.6 and 5.4
// apart, and a launch).
template <typename T, bool PICK> __global__ __launch_bounds__(1024) void k_verify_decide(VerifyArgs a) {
  if (PICK && rows_of_none(a)) return;
  __shared__ Roots roots;
  __shared__ Deciding sh;
  __shared__ Picking picking;
  __shared__ double sums[2][16];
  roots.fill();
  __syncthreads();
  const int b = blockIdx.x;
  decide<T>(a, b, true, roots, sh);
  __syncthreads();
  const Choice ch = sh.choice;
  if (ch.token != -2 || ch.zq > 0.0) return;
  const int own = ch.drop >= 0 && ch.drop < a.V ? ch.drop / PART : -1;
  const Part* p = a.parts + (long)ch.row * a.n_parts;
  double* to = a.sums + (long)b * 2 * a.n_parts;
  for (int i = threadIdx.x; i < a.n_parts; i += 1024)
    if (i != own) to[i] = to[a.n_parts + i] = p[i].z / ch.zp * prob_of(((double)p[i].m - ch.mp) * ch.scale, roots);
  if (own >= 0) sum_part<T>(a, ch, b, own, roots, sums);
  if constexpr (PICK) {
    __syncthreads();
    const double ahead = threadIdx.x < 64 && (int)threadIdx.x < a.n_parts ? to[threadIdx.x] : 0.0;
    pick<T>(a, ch, to, ahead, roots, picking);
  }
}

int n_parts(int V) { return cdiv(V, PART); }
size_t parts_bytes(const dm_verify_args* a) { return align256((size_t)2 * a->rows * n_parts(a->cols) * sizeof(Part)); }
size_t sums_bytes(const dm_verify_args* a) { return align256((size_t)2 * a->B * n_parts(a->cols) * sizeof(double)); }

template <typename T> void run_verify(const VerifyArgs& p, hipStream_t s) {
  hipLaunchKernelGGL(k_verify_parts<T>, dim3(p.n_parts, p.N, p.y ? 2 : 1), dim3(256), 0, s, p);
  const dim3 picks(p.B + cdiv(p.N, 16));
  if (!p.y) {
    hipLaunchKernelGGL((k_verify_decide<T, true>), picks, dim3(1024), 0, s, p);
    return;
  }
  if ((long)p.n_parts * p.B <= 256) {      // a block per CU
    hipLaunchKernelGGL((k_verify_sums<T, true>), dim3(p.n_parts, p.B), dim3(1024), 0, s, p);
  } else {
    hipLaunchKernelGGL((k_verify_decide<T, false>), dim3(p.B), dim3(1024), 0, s, p);
    hipLaunchKernelGGL((k_verify_sums<T, false>), dim3(p.n_parts, p.B), dim3(1024), 0, s, p);
  }
  hipLaunchKernelGGL(k_verify_pick<T>, picks, dim3(1024), 0, s, p);
}

}  // namespace

extern "C" {

size_t dm_verify_workspace_bytes(const dm_verify_args* a) {
  if (!a || a->rows <= 0 || a->B <= 0 || a->cols <= 0 || a->cols > DM_LOGPROB_COLS) return 0;
  return parts_bytes(a) + sums_bytes(a) + align256((size_t)a->B * sizeof(Choice));
}

int dm_verify_drafts(const dm_verify_args* a, void* stream) {
  DM_REQUIRE(a != nullptr, DM_ERR_INVALID, "null arguments");
  DM_REQUIRE(a->dtype == DM_BF16 || a->dtype == DM_F32, DM_ERR_INVALID, "dtype %d", a->dtype);
  DM_REQUIRE(a->rows >= 0 && a->rows <= 65535 && a->B >= 0 && a->B <= 65535, DM_ERR_INVALID, "rows=%d B=%d (at most 65535)", a->rows, a->B);
  DM_REQUIRE(a->cols > 0 && a->cols <= DM_LOGPROB_COLS && a->ld >= a->cols && (!a->draft_logits || a->ld_draft >= a->cols), DM_ERR_INVALID,
             "cols=%d ld=%lld ld_draft=%lld (at most %d columns)", a->cols, (long long)a->ld, (long long)a->ld_draft, DM_LOGPROB_COLS);
  if (a->B == 0 || a->rows == 0) {
    DM_REQUIRE(a->rows == 0 && a->B == 0, DM_ERR_INVALID, "rows=%d B=%d", a->rows, a->B);
    return DM_OK;
  }
  DM_REQUIRE(a->logits && a->ids && a->uniforms && a->temperature && a->starts && a->tokens && a->accepted && a->logp, DM_ERR_INVALID,
             "null argument");
  const size_t e = esz(a->dtype);
  DM_REQUIRE(reinterpret_cast<uintptr_t>(a->logits) % e == 0 && reinterpret_cast<uintptr_t>(a->draft_logits) % e == 0, DM_ERR_INVALID,
             "unaligned logits");
  const size_t need = dm_verify_workspace_bytes(a);
  DM_REQUIRE(a->workspace && aligned16(a->workspace) && a->workspace_bytes >= need, DM_ERR_WORKSPACE, "workspace %zu < %zu bytes",
             a->workspace_bytes, need);
  char* ws = (char*)a->workspace;
  VerifyArgs p = {a->logits, a->draft_logits, a->ids, a->uniforms, a->temperature, a->starts, a->tokens, a->accepted, a->logp,
                  (Part*)ws, (double*)(ws + parts_bytes(a)), (Choice*)(ws + parts_bytes(a) + sums_bytes(a)), a->ld, a->ld_draft,
                  a->rows, a->B, a->cols, n_parts(a->cols)};
  if (a->dtype == DM_BF16) run_verify<bf16>(p, S(stream));
  else run_verify<float>(p, S(stream));
  DM_HIP(hipGetLastError());
  return DM_OK;
}

}  // extern "C"
