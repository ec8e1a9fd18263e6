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
constexpr int EACH = PART / 256;

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
  int row;            // token row, -1: none
  int drop;           // a column that counts 0 (the draft without a distribution), -1: none
  int token;          // -2: to be drawn; else the token, -1 where there is no distribution
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

// the sequence of token row t, -1: none
DM_DEV int sequence_of(const VerifyArgs& a, int t) {
  int lo = 0, hi = a.B;
  while (lo + 1 < hi) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const Rows r(a, lo);
  return t >= r.first && t < r.first + r.n ? lo : -1;
}
// a temperature of 0 is greedy; the log probabilities are those at 1 then
DM_DEV double divisor(float T) { return T == 0.f ? 1.0 : (double)T; }

DM_DEV double wave_sum_double(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One block per row and part of it, of the target and of the draft (blockIdx.z).
template <typename T> __global__ __launch_bounds__(256) void k_verify_parts(VerifyArgs a) {
  const int t = blockIdx.y, c0 = blockIdx.x * PART;
  const bool draft = blockIdx.z;
  const int b = sequence_of(a, t);
  if (b < 0) return;
  const Rows rows(a, b);
  if (draft && t == rows.first + rows.n - 1) return;
  const T* x = (draft ? (const T*)a.y + t * a.ld_y : (const T*)a.x + t * a.ld_x) + c0;
  const int n = min(PART, a.V - c0);
  const double inv = 1.0 / divisor(a.temperature[b]);
  float v[EACH];
  float m = -INF;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int c = threadIdx.x + 256 * i;
    v[i] = c < n ? to_f(x[c]) : -INF;
    m = fmaxf(m, v[i]);
    nan |= v[i] != v[i];
  }
  __shared__ float sm[4];
  __shared__ double sz[4];
  __shared__ int sarg[4], snan;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) snan = 0;
  m = wave_max(m);
  if (lane == 0) sm[wave] = m;
  __syncthreads();
  if (nan) snan = 1;
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const double ref = m == -INF ? 0.0 : (double)m;
  double z = 0.0;
  int arg = 0x7fffffff;
#pragma unroll
  for (int i = EACH - 1; i >= 0; --i) {
    if (v[i] == m) arg = threadIdx.x + 256 * i;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) z += exp(((double)v[i] - ref) * inv);
  z = wave_sum_double(z);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) arg = min(arg, __shfl_xor(arg, o, 64));
  if (lane == 0) sz[wave] = z, sarg[wave] = arg;
  __syncthreads();
  if (threadIdx.x) return;
  Part p;
  p.z = (sz[0] + sz[1]) + (sz[2] + sz[3]);
  p.m = snan ? NAN_ : m;
  p.arg = c0 + min(min(sarg[0], sarg[1]), min(sarg[2], sarg[3]));
  a.parts[((long)draft * a.N + t) * a.n_parts + blockIdx.x] = p;
}

// A row's parts joined by a wave: the maximum (NaN if there is one), the sum relative to it and the first place of it.
DM_DEV Part join_parts(const VerifyArgs& a, bool draft, int t, double inv) {
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
    z += p[i].z * (p[i].m == -INF ? 0.0 : exp(((double)p[i].m - m) * inv));
  }
  Part r;
  r.z = wave_sum_double(z);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) arg = min(arg, __shfl_xor(arg, o, 64));
  r.arg = arg;
  r.m = __ballot(nan) ? NAN_ : m;
  return r;
}
// whether the parts are those of a distribution: something finite, no NaN, no +inf
DM_DEV bool is_distribution(const Part& p) { return fabsf(p.m) < INF; }

// Every block of a sequence's parts decides over its rows (a wave each, in turn), the first one writes what is decided; then
// each sums its part of the chosen row.
template <typename T> __global__ __launch_bounds__(256) void k_verify_choose(VerifyArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rows rows(a, b);
  __shared__ Choice ch;
  __shared__ int end;
  __shared__ double sums[2][4];
  if (threadIdx.x == 0) end = rows.n;
  __syncthreads();
  const float temperature = a.temperature[b];
  const double inv = 1.0 / divisor(temperature);
  const bool greedy = temperature == 0.f;
  for (int i = wave; i < rows.n; i += 4) {
    const int t = rows.first + i;
    const bool last = i == rows.n - 1;
    const Part p = join_parts(a, false, t, inv);
    Part q;
    q.z = 0.0, q.m = 0.f;
    if (!last && a.y && !greedy) q = join_parts(a, true, t, inv);
    const long d = last ? -1 : a.ids[t + 1];
    const bool in_range = d >= 0 && d < a.V;
    bool ok = false;
    double pd = 0.0, lp = NAN_;
    const bool valid = is_distribution(p) && is_distribution(q);
    if (valid && in_range) {
      lp = ((double)to_f(((const T*)a.x)[t * a.ld_x + d]) - p.m) * inv;
      pd = exp(lp) / p.z;
      lp -= log(p.z);
    }
    if (greedy) {
      ok = !last && d == p.arg && p.m == p.m && p.m > -INF;
    } else if (valid && in_range) {
      const double qd = a.y ? exp(((double)to_f(((const T*)a.y)[t * a.ld_y + d]) - q.m) * inv) / q.z : 1.0;
      ok = (double)a.u[2 * t] * qd < pd;
    }
    if (!ok && lane == 0) atomicMin(&end, i);
    if (ok && blockIdx.x == 0 && lane == 0) {
      a.tokens[t] = d;
      a.logp[t] = (float)lp;
    }
  }
  __syncthreads();
  const int e = end;
  if (rows.n == 0) {
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.accepted[b] = 0;
      a.choice[b].row = -1;
    }
    return;
  }
  const int t = rows.first + e;
  const bool last = e == rows.n - 1;
  if (wave == 0) {
    const Part p = join_parts(a, false, t, inv);
    Part q;
    q.z = 0.0, q.m = 0.f, q.arg = 0;
    const bool with_q = !last && a.y && !greedy;
    if (with_q) q = join_parts(a, true, t, inv);
    if (lane == 0) {
      ch.zp = p.z, ch.zq = with_q ? q.z : 0.0, ch.mp = p.m, ch.mq = q.m, ch.row = t;
      ch.drop = last || a.y ? -1 : (int)max(-1l, min((long)a.ids[t + 1], 0x7fffffffl));
      ch.token = greedy ? (p.m == p.m && p.m > -INF ? p.arg : -1) : is_distribution(p) && is_distribution(q) ? -2 : -1;
      if (blockIdx.x == 0) {
        a.choice[b] = ch;
        a.accepted[b] = e;
      }
    }
  }
  // the rows behind
  if (blockIdx.x == 0)
    for (int i = e + 1 + threadIdx.x; i < rows.n; i += 256) a.tokens[rows.first + i] = -1, a.logp[rows.first + i] = 0.f;
  __syncthreads();
  if (ch.token != -2) return;
  double r = 0.0, s = 0.0;
  const T* x = (const T*)a.x + t * a.ld_x;
  const T* y = (const T*)a.y + t * a.ld_y;
  const int c0 = blockIdx.x * PART + threadIdx.x * EACH;
  for (int i = 0; i < EACH; ++i) {
    const int c = c0 + i;
    if (c >= a.V) break;
    const double pc = exp(((double)to_f(x[c]) - ch.mp) * inv) / ch.zp;
    const double qc = ch.zq > 0.0 ? exp(((double)to_f(y[c]) - ch.mq) * inv) / ch.zq : 0.0;
    s += pc;
    r += c == ch.drop ? 0.0 : fmax(pc - qc, 0.0);
  }
  r = wave_sum_double(r);
  s = wave_sum_double(s);
  if (lane == 0) sums[0][wave] = r, sums[1][wave] = s;
  __syncthreads();
  if (threadIdx.x < 2)
    a.sums[((long)b * 2 + threadIdx.x) * a.n_parts + blockIdx.x] =
        (sums[threadIdx.x][0] + sums[threadIdx.x][1]) + (sums[threadIdx.x][2] + sums[threadIdx.x][3]);
}

// One block per sequence: the part of the chosen row in which the place lies, then the thread, then the column. Rows of no
// sequence get token -1.
template <typename T> __global__ __launch_bounds__(256) void k_verify_pick(VerifyArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (b == a.B) {
    for (int t = threadIdx.x; t < a.N; t += 256)
      if (sequence_of(a, t) < 0) a.tokens[t] = -1, a.logp[t] = 0.f;
    return;
  }
  const Choice ch = a.choice[b];
  if (ch.row < 0) return;
  const double inv = 1.0 / divisor(a.temperature[b]);
  const T* x = (const T*)a.x + ch.row * a.ld_x;
  const T* y = (const T*)a.y + ch.row * a.ld_y;
  __shared__ double base, place, sums[4];
  __shared__ int part, plain, hit[4], positive[4];
  int token = ch.token;
  if (token == -2) {
    if (threadIdx.x == 0) {
      const double* s = a.sums + (long)b * 2 * a.n_parts;
      double total = 0.0;
      for (int i = 0; i < a.n_parts; ++i) total += s[i];
      plain = !(total > 0.0);
      if (plain) {
        s += a.n_parts;
        total = 0.0;
        for (int i = 0; i < a.n_parts; ++i) total += s[i];
      }
      place = (double)a.u[2 * ch.row + 1] * total;
      // the part after whose sum the place lies; past the last one's (by rounding) the last with any
      double before = 0.0;
      part = -1;
      int any = 0;
      double any_base = 0.0;
      for (int i = 0; i < a.n_parts; ++i) {
        if (s[i] > 0.0) any = i, any_base = before;
        if (before + s[i] > place) {
          part = i, base = before;
          break;
        }
        before += s[i];
      }
      if (part < 0) part = any, base = any_base;
    }
    __syncthreads();
    const int c0 = part * PART + threadIdx.x * EACH;
    double r[EACH], mine = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int c = c0 + i;
      r[i] = 0.0;
      if (c < a.V) {
        const double pc = exp(((double)to_f(x[c]) - ch.mp) * inv) / ch.zp;
        const double qc = !plain && ch.zq > 0.0 ? exp(((double)to_f(y[c]) - ch.mq) * inv) / ch.zq : 0.0;
        r[i] = !plain && c == ch.drop ? 0.0 : fmax(pc - qc, 0.0);
      }
      mine += r[i];
    }
    double sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    double before = base + (sum - mine);
    for (int w = 0; w < wave; ++w) before += sums[w];
    int first = 0x7fffffff, most = -1;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      before += r[i];
      if (r[i] > 0.0) most = c0 + i;
      if (before > place && r[i] > 0.0 && first == 0x7fffffff) first = c0 + i;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64)), most = max(most, __shfl_xor(most, o, 64));
    if (lane == 0) hit[wave] = first, positive[wave] = most;
    __syncthreads();
    token = min(min(hit[0], hit[1]), min(hit[2], hit[3]));
    if (token == 0x7fffffff) token = max(max(positive[0], positive[1]), max(positive[2], positive[3]));
  }
  if (threadIdx.x == 0) {
    a.tokens[ch.row] = token;
    a.logp[ch.row] = token < 0 ? NAN_ : (float)(((double)to_f(x[token]) - ch.mp) * inv - log(ch.zp));
  }
}

int n_parts(int V) { return cdiv(V, PART); }
size_t parts_bytes(const dm_verify_args* a) { return align256((size_t)2 * a->rows * n_parts(a->cols) * sizeof(Part)); }
size_t sums_bytes(const dm_verify_args* a) { return align256((size_t)2 * a->B * n_parts(a->cols) * sizeof(double)); }

template <typename T> void run_verify(const VerifyArgs& p, hipStream_t s) {
  hipLaunchKernelGGL(k_verify_parts<T>, dim3(p.n_parts, p.N, p.y ? 2 : 1), dim3(256), 0, s, p);
  hipLaunchKernelGGL(k_verify_choose<T>, dim3(p.n_parts, p.B), dim3(256), 0, s, p);
  hipLaunchKernelGGL(k_verify_pick<T>, dim3(p.B + 1), dim3(256), 0, s, p);
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
