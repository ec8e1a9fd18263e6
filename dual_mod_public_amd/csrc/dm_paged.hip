// Attention of new tokens over a paged cache (dm_paged_write, dm_paged_attention) and eviction from it
// (dm_paged_evict).
//
// Sequence b has lengths[b] cached rows with its new tokens, whose rows are the last ones; row r lies in page
// table[b, r / page] of [n_pages, h_kv, page, dh]. The query rows of a sequence and key head are its n tokens times
// the g = h / h_kv heads that share the key head, token by token, in tiles of TILE_Q.
//
// How the work is split is decided on the device, from the lengths (a captured call is replayed with other ones): every
// kernel derives the same plan from them (find_item), in which a sequence's rows are cut into as many pieces as bring the
// whole call to about `want` pieces (one each where they are few). Partial results of a query tile (unnormalised sums with their maximum) wait in the
// workspace and k_paged_join adds them in the order of the pieces, so a call's results repeat bit for bit.
#include "dm_common.h"
#include "dm_error.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace dm;

namespace {

constexpr float INF = __builtin_inff(), NAN_ = __builtin_nanf("");
constexpr float LOG2E = 1.4426950408889634f;
constexpr int CUS = 256;
constexpr float LAST_CACHE = 1 << 28;      // bytes
constexpr int TILE_Q = 16;      // query rows of a tile
constexpr int TILE_K = 64;      // cached rows that the plan counts in

struct PagedArgs {
  const void *q, *K, *V, *k_rows, *v_rows;
  void* o;
  float *lse, *weights, *part;         // part: the pieces' sums, then their maxima and sums of exponentials
  const int32_t *table, *lengths, *starts;
  long q_token, q_head, k_page, v_page, kr_token, kr_head, vr_token, vr_head;
  int B, h, h_kv, g, n_pages, cols, page_shift, N, window;
  float scale2;                        // scale log2 e
  int want, least;                     // the plan: pieces wanted, least tiles of cached rows in one
  float* scores;                       // N h cols * page of them, before the scale, for the weights; nullptr: not kept
};

// A sequence as the call gives it. A table that does not hold its rows, or fewer rows than new tokens: bad, NaN results.
struct Seq {
  int first, n, len;
  bool bad;
  DM_DEV Seq() : first(0), n(0), len(0), bad(false) {}
  DM_DEV Seq(const PagedArgs& a, int b) {
    len = a.lengths[b];
    if (a.starts) {
      first = min(max(a.starts[b], 0), a.N);
      n = min(max(a.starts[b + 1], first), a.N) - first;
    } else {
      first = b;
      n = len != 0;   // an empty place of the batch
    }
    bad = len < n || len > (a.cols << a.page_shift);
    if (bad) len = n;
  }
  // rows [low, high) that token j reads (with a self pair its own row is not among them)
  DM_DEV int high(const PagedArgs& a, int j) const { return len - n + j + (a.k_rows ? 0 : 1); }
  DM_DEV int low(const PagedArgs& a, int j) const { return a.window ? max(0, len - n + j - a.window + 1) : 0; }
  DM_DEV int tiles_k(const PagedArgs& a) const {   // of all its tokens' rows
    if (n == 0 || bad) return 0;
    return (max(0, high(a, n - 1) - (low(a, 0) & -TILE_K)) + TILE_K - 1) / TILE_K;
  }
};

struct Item {
  int b = -1;      // -1: there is none
  Seq s;
  int tile, piece, pieces, slot;   // slot of the query tile's piece 0 in the workspace, where pieces > 1
  float tiles_k;                   // tiles of cached rows of all sequences
};

// The sum over the lanes up to this one, by moves inside the rows of 16 lanes and broadcasts of the rows' last lanes.
DM_DEV int wave_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);     // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);     // row_bcast 15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);     // row_bcast 31 into rows 2 and 3
  return v;
}

// The plan: sequence b's query tiles (of ROWS query rows; 1 with ROWS = 0) times its pieces, in order. PIECES: find item
// number `at` of those; otherwise of the query tiles alone. Called by whole waves. Items and slots are fewer than the blocks
// of a launch; the cost (query tiles times tiles of cached rows) may pass 32 bits and is summed in fp32, rounded up, so that a
// piece's tiles are never too few for the slots that the workspace has.
template <int ROWS, bool PIECES> DM_DEV Item find_item(const PagedArgs& a, int at) {
  const int lane = threadIdx.x & 63;
  auto tiles_q = [&](const Seq& s) { return ROWS ? (s.n * a.g + ROWS - 1) / (ROWS ? ROWS : 1) : (s.n > 0); };
  Seq s;
  Item it;
  float cost = 0.f, tiles_k = 0.f;
  for (int b = lane; b < a.B; b += 64) {
    s = Seq(a, b);
    tiles_k += (float)s.tiles_k(a);
    cost += (float)tiles_q(s) * (float)s.tiles_k(a);
  }
  it.tiles_k = wave_sum(tiles_k);
  cost = wave_sum(cost) * (1.f + 1e-4f);                   // 1024 + 6 additions of half a step, 2^-24, each
  const int each = max(a.least, (int)fminf(ceilf(cost / (float)a.want), 1e9f));   // tiles of cached rows per piece
  int done = 0, slots = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    if (a.B > 64) s = b < a.B ? Seq(a, b) : Seq();
    const int tq = b < a.B ? tiles_q(s) : 0;
    const int pieces = tq ? max(1, (s.tiles_k(a) + each - 1) / each) : 1;
    const int mine = PIECES ? tq * pieces : tq, kept = pieces > 1 ? tq * pieces : 0;
    const int upto = wave_upto(mine), kept_upto = wave_upto(kept);
    const uint64_t hit = __ballot(mine > 0 && done + upto > at);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int rest = at - (done + __shfl(upto - mine, l, 64));
      if (rest < 0 || rest >= __shfl(mine, l, 64)) return it;     // (starts that do not ascend: more than 32 bits of tiles)
      it.b = b0 + l;
      it.s.first = __shfl(s.first, l, 64);
      it.s.n = __shfl(s.n, l, 64);
      it.s.len = __shfl(s.len, l, 64);
      it.s.bad = __shfl((int)s.bad, l, 64);
      it.pieces = __shfl(pieces, l, 64);
      it.tile = PIECES ? rest / it.pieces : rest;
      if (ROWS) it.tile = __shfl(tq, l, 64) - 1 - it.tile;      // the tiles with the most rows to read first
      it.piece = PIECES ? rest % it.pieces : 0;
      it.slot = slots + __shfl(kept_upto - kept, l, 64) + it.tile * it.pieces;
      return it;
    }
    done += __shfl(upto, 63, 64);
    slots += __shfl(kept_upto, 63, 64);
  }
  return it;
}

// A number that every lane holds, as a scalar: quotients come from vector instructions, and what is computed from them (rows,
// pages, addresses) would stay with those.
DM_DEV int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// the item in scalar registers: every lane holds the same
DM_DEV void make_uniform(Item& it) {
  auto u = [](int& x) { x = __builtin_amdgcn_readfirstlane(x); };
  u(it.b), u(it.s.first), u(it.s.n), u(it.s.len), u(it.tile), u(it.piece), u(it.pieces), u(it.slot);
  it.s.bad = __builtin_amdgcn_readfirstlane((int)it.s.bad);
}

// ---- rows into the pages ---------------------------------------------------------------------
// A wave per token and 256 of its 16-byte pieces of key and value rows (tokens in turn where there are more of them than a launch
// has threads). The token's sequence is searched for by all lanes, a 64th at a time. Bound by latency for few tokens (4 us for 200),
// by the bytes for many: 10000 tokens of 16 key heads of 64 in fp32 (168 MB moved) 30 us, 5.6 TB/s (62 with a thread per 16 bytes,
// its quotients and a binary search), 4096 tokens of 8 key heads of 128 in bf16 9.7.
template <typename T> __global__ __launch_bounds__(256) void k_paged_write(PagedArgs a, int dh_shift) {
  constexpr int V = 16 / (int)sizeof(T), SHIFT = sizeof(T) == 2 ? 3 : 2, EACH = 4;
  const int lane = threadIdx.x & 63, per_shift = dh_shift - SHIFT, half = a.h_kv << per_shift;
  const int in_page = (1 << a.page_shift) - 1;
  for (long at = blockIdx.x * 4L + (threadIdx.x >> 6); at < a.N; at += gridDim.x * 4L) {
    const int t = uniform((int)at);
    int b = t;
    if (a.starts) {   // the last sequence that starts at t or before
      b = 0;
      for (int n = a.B; n > 1;) {
        const int step = (n + 63) >> 6, i = lane * step;
        const uint64_t before = __ballot(i < n && a.starts[b + min(i, n - 1)] <= t);
        const int k = max(0, (int)__popcll(before) - 1) * step;
        b += k;
        n = min(step, n - k);
      }
      b = uniform(b);
    }
    const Seq s(a, b);
    if (s.bad || t < s.first || t >= s.first + s.n) continue;
    const int row = s.len - s.n + (t - s.first);
    const int page = a.table[(long)b * a.cols + (row >> a.page_shift)];
    if (page < 0 || page >= a.n_pages) continue;
    const T* k = (const T*)a.k_rows + t * a.kr_token;
    const T* v = (const T*)a.v_rows + t * a.vr_token;
    T* const K = (T*)a.K + page * a.k_page + ((long)(row & in_page) << dh_shift);
    T* const Vp = (T*)a.V + page * a.v_page + ((long)(row & in_page) << dh_shift);
    u32x4 x[EACH];
    T* to[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = ((int)blockIdx.y * EACH + e) * 64 + lane;
      const bool value = i >= half;
      const int j = value ? i - half : i, c = j >> per_shift, at_v = (j & ((1 << per_shift) - 1)) * V;
      to[e] = nullptr;
      if (j >= half) continue;
      x[e] = ld_global<u32x4>((value ? v + c * a.vr_head : k + c * a.kr_head) + at_v);
      to[e] = (value ? Vp : K) + ((long)c << (a.page_shift + dh_shift)) + at_v;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (to[e]) *reinterpret_cast<u32x4*>(to[e]) = x[e];
  }
}

// ---- the read ----------------------------------------------------------------------------------
template <typename T, int DH> struct Tile {
  // tiles of 16 cached rows in a wave's step (fp32 rows of 128 two at a time leave room for one wave per SIMD: 16 tokens over 4096
  // rows on 8 key heads 131 us instead of 99, 512 tokens over 8192 rows, 16 heads on 8, 427 instead of 313)
  static constexpr int NT = sizeof(T) == 4 && DH == 128 ? 1 : 2;
  static constexpr int KT = 16 * NT;
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr int LDV = DH + (sizeof(T) == 2 ? 16 : 4);      // 8 rows (fp32: 4 groups) fill the banks once
  static constexpr int NF = DH * (int)sizeof(T) / 64;             // 16-byte loads of a lane for 16 rows in fragments
  static constexpr int NV = KT * DH * (int)sizeof(T) / 1024;      // 16-byte loads of a lane for the step's V rows
  static constexpr int VPR = DH / V;
  static constexpr int NDT = DH / 16;
  // per SIMD at least: what the registers of rows on their way leave (bf16 rows of 64: 115 registers, 4 waves fit; asked for 4 the
  // compiler keeps fewer loads on their way: 64 sequences of 100 to 8192 rows 97 us instead of 92 through the last cache)
  static constexpr int WAVES = sizeof(T) == 2 || DH == 128 ? 3 : 2;
};

// S^T = K Q^T of NT tiles of 16 cached rows and 16 query rows, from a lane's 16-byte chunks of each: bf16 lane l holds columns
// 8 (l / 16) .. + 7 of a 32-column step, fp32 4 (l / 16) .. + 3 of 16 columns (the same in K and Q, so the order of the
// columns in an instruction does not matter). In fp32 two chains of sums take turns, of LENGTH chunks (of 16 products) each, whose
// sums are added to the score: short chains round less. Outputs' errors in the 2-norm and us a call of 16 tokens over 4096 rows of 128,
// 32 heads on 8, with one chain of 128 products 1.12e-6 and 98, two of 64 6.8e-7 and 100 to 104, four of 32 4.6e-7 and 115, two of 16 four
// times 4.0e-7 and 101 to 103; 512 tokens over 8192 rows 661, 647, 650 and 604.
template <typename T, int LENGTH, int NT, int NF> DM_DEV void mma_scores(const u32x4 (&k)[NT][NF], const u32x4 (&q)[NF], floatx4 (&acc)[NT]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = zero4();
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[t] = Mfma<bf16>::mma(__builtin_bit_cast(bf16x8, k[t][i]), __builtin_bit_cast(bf16x8, q[i]), acc[t]);
  } else {
#pragma unroll
    for (int i0 = 0; i0 < NF; i0 += 2 * LENGTH) {
      floatx4 part[2][NT];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < NT; ++t) part[c][t] = zero4();
#pragma unroll
      for (int i = i0; i < i0 + 2 * LENGTH; i += 2)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              part[c][t] = Mfma<float>::mma(__uint_as_float(k[t][i + c][j]), __uint_as_float(q[i + c][j]), part[c][t]);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = i0 ? acc[t] + (part[0][t] + part[1][t]) : part[0][t] + part[1][t];
    }
  }
}

// Scores are held as they come from the products and scaled where their exponential is taken, in one rounding with the reference that
// is subtracted. Maxima are taken before the scale, so that is positive there: queries carry its sign, or 0 (and then it is 1).
DM_DEV float positive_scale(float scale2) { return scale2 == 0.f ? 1.f : fabsf(scale2); }
template <typename T> DM_DEV void carry_sign(u32x4& q, float scale2) {
  constexpr uint32_t SIGN = sizeof(T) == 2 ? 0x80008000u : 0x80000000u, LOW = sizeof(T) == 2 ? 0x7f80u : 0u, TOP = 0x7f800000u;
  const uint32_t flip = scale2 < 0.f ? SIGN : 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t zero = (LOW && (q[e] & LOW) == LOW ? 0x7fc0u : 0u) | ((q[e] & TOP) == TOP ? 0x7fc00000u : 0u);   // NaN where not finite
    q[e] = scale2 == 0.f ? zero : q[e] ^ flip;
  }
}
// The logarithm of a sum z relative to a reference in units of ln 2, rounded once.
DM_DEV float log_of(float ref, float z) { return z == 0.f ? -INF : (float)(((double)ref + __builtin_amdgcn_logf(z)) * 0.6931471805599453); }

template <typename T> DM_DEV bool any_nonfinite(const u32x4& v) {
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 2) bad |= (v[j] & 0x7f80u) == 0x7f80u || (v[j] & 0x7f800000u) == 0x7f800000u;
    else bad |= (v[j] & 0x7f800000u) == 0x7f800000u;
  }
  return bad;
}

// Steps in which a query row does not read every row, and some value among them is not finite: a product with a probability
// of 0 would make it NaN. Such values count 0 in the product; at the end a second one, of 1 for each row that is read with 1
// for +inf, 2^7 for -inf and 2^14 for NaN (of at most 32 rows, exact in bf16 and fp32), says what to add.
DM_DEV float split_nonfinite(float v) {      // the code of a value
  const uint32_t u = __float_as_uint(v), top = u & 0x7fffffffu;
  return top < 0x7f800000u ? 0.f : top > 0x7f800000u ? 16384.f : u >> 31 ? 128.f : 1.f;
}
template <typename T> DM_DEV void clear_nonfinite(u32x4& v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 2) {
      if ((v[j] & 0x7f80u) == 0x7f80u) v[j] &= 0xffff0000u;
      if ((v[j] & 0x7f800000u) == 0x7f800000u) v[j] &= 0xffffu;
    } else {
      if ((v[j] & 0x7f800000u) == 0x7f800000u) v[j] = 0;
    }
  }
}
DM_DEV float said_by(float code) {
  const int c = (int)code;
  float x = 0.f;
  if (c & 0x7f) x += INF;
  if ((c >> 7) & 0x7f) x -= INF;
  if (c >> 14) x = NAN_;
  return x;
}

// O^T[16 columns][16 query rows] += V^T P^T over 32 rows. Lane l's probabilities are those of rows 16 t + 4 (l / 16) + i
// of query row l % 16, which is how the scores' tiles leave them; V's fragments take their rows in the same order.
// Beside values in bf16 a probability is the sum of two bf16 numbers, each with a product of its own: itself cut to 8 bits, and
// what is left rounded, 2^-15 of it at most. Outputs are then off by 1.65e-3 in the 2-norm, which is their own rounding; with
// probabilities rounded to bf16 once 1.95e-3 to 2.2e-3, in the same time (64 sequences of 100 to 8192 rows 90 us a call, 24 chunks of
// up to 8 tokens 39, 16 chunks of 24 tokens over 4096 rows 69).
DM_DEV i16x8 values_fragment(const bf16* v, int ldv) {
  const int lane = threadIdx.x & 63, grp = lane >> 4, s = lane & 15;
  v += (4 * grp + (s >> 2)) * ldv + 4 * (s & 3);
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(v));
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(v + 16 * ldv));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int N> DM_DEV bf16x8 to_bf16x8(const float (&p)[N], int at) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (bf16)p[at + i];
  return r;
}
// The second part is never 0 where the first is not (2^-24 of the probability at least): its product with an infinite value would be
// NaN.
template <typename T, int N> struct Probabilities;
template <> struct Probabilities<bf16, 8> {
  bf16x8 cut, left;
  DM_DEV Probabilities(const float (&p)[8]) {
    u32x4 c;
    float l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t top = __float_as_uint(p[i]) & 0xffff0000u;
      c[i >> 1] = i & 1 ? c[i >> 1] | top : top >> 16;
      l[i] = fmaxf(p[i] - __uint_as_float(top), p[i] * 0x1p-24f);
    }
    cut = __builtin_bit_cast(bf16x8, c);
    left = to_bf16x8(l, 0);
  }
};
template <int N> struct Probabilities<float, N> {
  const float (&p)[N];
  DM_DEV Probabilities(const float (&p)[N]) : p(p) {}
};
template <int LDV> DM_DEV floatx4 mma_values(const bf16* Vs, const Probabilities<bf16, 8>& p, floatx4 acc) {
  const bf16x8 v = __builtin_bit_cast(bf16x8, values_fragment(Vs, LDV));
  return Mfma<bf16>::mma(v, p.left, Mfma<bf16>::mma(v, p.cut, acc));
}
template <int LDV, int N> DM_DEV floatx4 mma_values(const float* Vs, const Probabilities<float, N>& p, floatx4 acc) {
  const int lane = threadIdx.x & 63, grp = lane >> 4, s = lane & 15;
#pragma unroll
  for (int i = 0; i < N; ++i) acc = Mfma<float>::mma(Vs[(16 * (i >> 2) + 4 * grp + (i & 3)) * LDV + s], p.p[i], acc);
  return acc;
}

// The page of rows r .. that lie in one (pages hold 16 rows or more and begin at a multiple of 16). needed: some query of
// the tile reads some of them. A page outside the pool is read as page 0 and marks the tile's results. The table is read through
// the scalar cache: a vector load of it would be waited for together with all rows that are on their way (two prompts' chunks
// of 2048 tokens over 16384 rows 2.50 ms so, 1.66 with scalar loads), and pages are looked up a step ahead of their rows.
DM_DEV int page_of(const PagedArgs& a, const int32_t* table, int r, bool needed, bool& bad) {
  typedef const __attribute__((address_space(4))) int32_t* Scalar;
  const int p = needed ? ((Scalar)table)[r >> a.page_shift] : 0;
  const bool in = p >= 0 && p < a.n_pages;
  bad |= !in;
  return in ? p : 0;
}

// Row r of V, nullptr: not among [t_low, t_high), or of no page of the pool.
template <typename T> DM_DEV const T* value_row(const PagedArgs& a, const int32_t* table, int c, int r, int t_low, int t_high, int dh) {
  const int page = r >= t_low && r < t_high ? table[r >> a.page_shift] : -1;
  if (page < 0 || page >= a.n_pages) return nullptr;
  return (const T*)a.V + page * a.v_page + (((long)c << a.page_shift) + (r & ((1 << a.page_shift) - 1))) * dh;
}
// (rows in steps of 32)
DM_DEV long scores_at(const PagedArgs& a, const Seq& s, int c) {
  return ((long)s.first * a.h_kv + (long)c * s.n) * a.g * ((((long)a.cols << a.page_shift) + 31) & -32L);
}

// One block: a query tile of 16 rows, a key head and a piece of its cached rows. The four waves take steps of 32 rows in
// turn, each with a running maximum m and sum z per query row (scores in units of ln 2) and O^T in registers, and are
// joined through LDS. S^T = K Q^T rather than S = Q K^T: a lane then holds scores of one query row only, the maximum needs two
// exchanges, and the probabilities are already the operand of the product with V, whose columns come from LDS transposed. K goes
// to the matrix cores straight from memory. The next step's rows of K and V are on their way in registers meanwhile.
// Bound by the rows' bytes: 64 sequences of 100 to 8192 rows of 64 on 16 key heads (484 MB) 83.5 us, 5.8 TB/s, of random pages of
// 64 rows; more blocks per CU or more rows on their way bring nothing. One token over 1024 rows 11 us in one piece per head, most of
// it latency: the plan, the table, the rows.
// KEEP: the scores are kept for the weights (of the lanes behind the last query row too, which work on that one again: a store
// that some lanes skip would have the next rows' loads wait for it, 276 instead of 273 us). 32 sequences of 3000 to 16384 rows of
// 128 on 8 key heads, 1.28 GB: 229 us without, 273 with; past the last cache 204 and 268 (of which 5 where they stay in L2,
// 55 for the 40 MB in memory). Computing the scores again costs 172.
template <typename T, int DH, bool KEEP> __global__ __launch_bounds__(256, (Tile<T, DH>::WAVES)) void k_paged_read(PagedArgs a) {
  using C = Tile<T, DH>;
  constexpr int NP = 4 * C::NT;      // scores of a lane in a step
  constexpr int VBYTES = C::KT * C::LDV * (int)sizeof(T), OBYTES = TILE_Q * DH * 4;
  __shared__ __attribute__((aligned(16))) char smem[4 * (VBYTES > OBYTES ? VBYTES : OBYTES)];
  __shared__ float sm[4][TILE_Q], sz[4][TILE_Q];
  const int c = uniform(blockIdx.x % a.h_kv), lane = threadIdx.x & 63, grp = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Item it = find_item<TILE_Q, true>(a, blockIdx.x / a.h_kv);
  if (it.b < 0) return;
  make_uniform(it);
  const Seq& s = it.s;
  const int rows = s.n * a.g, rho0 = it.tile * TILE_Q;            // query rows of the sequence, the tile's first
  const int j_first = uniform(rho0 / a.g), j_last = uniform((min(rho0 + TILE_Q, rows) - 1) / a.g);
  // the lane's query row; behind the last one that one again
  const int rho = min(rho0 + col, rows - 1), j = rho / a.g, head = c * a.g + rho % a.g;
  const int high = s.high(a, j), low = s.low(a, j);
  // the tile's rows, and this piece's
  const int t_low = s.low(a, j_first), t_high = s.bad ? 0 : s.high(a, j_last);
  const int base = t_low & -TILE_K, tiles = max(0, (t_high - base + TILE_K - 1) / TILE_K);
  const int each = uniform((tiles + it.pieces - 1) / it.pieces);
  const int k0 = base + it.piece * each * TILE_K, k1 = min(k0 + each * TILE_K, t_high);
  // rows from this on and below that are read by all query rows of the tile
  const int all_low = s.low(a, j_last), all_high = s.high(a, j_first);

  u32x4 qf[C::NF];
  {
    const T* q = (const T*)a.q + (long)(s.first + j) * a.q_token + (long)head * a.q_head;
#pragma unroll
    for (int i = 0; i < C::NF; ++i) qf[i] = ld_global<u32x4>(q + i * 4 * C::V + grp * C::V), carry_sign<T>(qf[i], a.scale2);
  }
  const float scale2 = positive_scale(a.scale2);
  floatx4 O[C::NDT];
#pragma unroll
  for (int d = 0; d < C::NDT; ++d) O[d] = zero4();
  float m = -INF, z = 0.f;    // z: this lane's share
  if (a.k_rows && it.piece == 0 && wave == 0) {   // the self pair: one more row
    const long kr = (long)(s.first + j) * a.kr_token + (long)c * a.kr_head, vr = (long)(s.first + j) * a.vr_token + (long)c * a.vr_head;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < C::NF; ++i) {
      const u32x4 k = ld_global<u32x4>((const T*)a.k_rows + kr + i * 4 * C::V + grp * C::V);
      float x[C::V], y[C::V];
      unpack16<T>(uint4{k[0], k[1], k[2], k[3]}, x);
      unpack16<T>(uint4{qf[i][0], qf[i][1], qf[i][2], qf[i][3]}, y);
#pragma unroll
      for (int e = 0; e < C::V; ++e) dot = fmaf(x[e], y[e], dot);
    }
    dot = xor_sum<32>(xor_sum<16>(dot));
    m = dot * scale2;
    const float p = __builtin_amdgcn_exp2f(fmaf(dot, scale2, m == -INF ? 0.f : -m));
    z = grp == 0 ? p : 0.f;
#pragma unroll
    for (int d = 0; d < C::NDT; ++d) {
      float v[4];
      unpack4<T>(ld_global<typename Raw4<T>::type>((const T*)a.v_rows + vr + 16 * d + 4 * grp), v);
#pragma unroll
      for (int i = 0; i < 4; ++i) O[d][i] = p * v[i];
    }
  }

  // kept scores of the lane's query row: [cached rows / 32][query rows][32] for each sequence and key head
  float* scores = a.scores + scores_at(a, s, c) + 32L * rho + 4 * grp;
  const int32_t* table = a.table + (long)it.b * a.cols;
  const int in_page = (1 << a.page_shift) - 1;
  T* Vs = reinterpret_cast<T*>(smem) + wave * C::KT * C::LDV;
  bool bad = s.bad, odd = false;
  u32x4 kf[C::NT][C::NF], vf[C::NV];
  int pages[C::NT];
  auto look_up = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < C::NT; ++t) pages[t] = page_of(a, table, r0 + 16 * t, r0 + 16 * t < t_high && r0 + 16 * t + 16 > t_low, bad);
  };
  // Rows that one tile reads pass the last cache by where the call's are more than it holds: 64 sequences of 2048 rows of 64 on 16
  // key heads (512 MiB) 81 us, 6.6 TB/s, instead of 92.6; 32 of 8192 rows of 128 on 8 (1 GiB) 168 instead of 197. Fewer rows find
  // themselves there where they were read before (24 sequences of 50 to 4001 rows 21 us, past it 25.8), those of two tiles are
  // read by the second one there or in L2 (32 sequences of 4096 rows, two tiles, 121 us, past it 154).
  const bool stream = rows <= TILE_Q && uniform(it.tiles_k * (2.f * TILE_K * DH * sizeof(T)) * a.h_kv > LAST_CACHE);
  auto load_rows = [&](int r0, auto passing) __attribute__((always_inline)) {
    auto ld = [&](const T* p) {
      if constexpr (passing) return __builtin_nontemporal_load((const __attribute__((address_space(1))) u32x4*)p);
      else return ld_global<u32x4>(p);
    };
#pragma unroll
    for (int t = 0; t < C::NT; ++t) {
      const int r = r0 + 16 * t;
      const long page = pages[t];
      const long off = (((long)c << a.page_shift) + (r & in_page)) * DH;
      const T* K = (const T*)a.K + page * a.k_page + off;
      const T* Vp = (const T*)a.V + page * a.v_page + off;
#pragma unroll
      for (int i = 0; i < C::NF; ++i) kf[t][i] = ld(K + col * DH + i * 4 * C::V + grp * C::V);
#pragma unroll
      for (int i = 0; i < C::NV / C::NT; ++i) {
        const int v = i * 64 + lane;
        vf[t * (C::NV / C::NT) + i] = ld(Vp + v * C::V);
      }
    }
  };
  auto load = [&](int r0) __attribute__((always_inline)) {
    if (stream) {      // (the compiler would make one of both sides but for what differs before and behind the loads)
      asm volatile("; rows pass the last cache by");
      load_rows(r0, std::true_type());
      asm volatile("; passed");
    } else {
      asm volatile("; rows may stay in the last cache");
      load_rows(r0, std::false_type());
      asm volatile("; stayed");
    }
  };
  int r0 = k0 + C::KT * wave;
  if (r0 < k1) look_up(r0), load(r0), look_up(min(r0 + 4 * C::KT, k1));
  for (; r0 < k1; r0 += 4 * C::KT) {
    const bool masked = r0 < all_low || r0 + C::KT > all_high;
    if (masked) {
#pragma unroll
      for (int i = 0; i < C::NV; ++i) {
        const int row = r0 + (i * 64 + lane) / C::VPR;
        if (row < t_low || row >= t_high) vf[i] = u32x4{0, 0, 0, 0};   // whatever lies there
        if (any_nonfinite<T>(vf[i])) odd = true, clear_nonfinite<T>(vf[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < C::NV; ++i) {
      const int v = i * 64 + lane;
      *reinterpret_cast<u32x4*>(Vs + v / C::VPR * C::LDV + (v % C::VPR) * C::V) = vf[i];
    }
    float p[NP];      // of rows r0 + 16 (i / 4) + 4 grp + i % 4
    floatx4 acc[C::NT];
    mma_scores<T, 1>(kf, qf, acc);
#pragma unroll
    for (int i = 0; i < NP; ++i) p[i] = acc[i >> 2][i & 3];
    if (masked) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = r0 + 16 * (i >> 2) + 4 * grp + (i & 3);
        if (r < low || r >= high) p[i] = -INF;
      }
    }
    float top = p[0];
#pragma unroll
    for (int i = 1; i < NP; ++i) top = fmaxf(top, p[i]);
    if constexpr (KEEP) {
      float* x = scores + (long)(r0 >> 5) * (32L * rows) + (r0 & 31);
      *reinterpret_cast<floatx4*>(x) = floatx4{p[0], p[1], p[2], p[3]};
      if constexpr (C::NT == 2) *reinterpret_cast<floatx4*>(x + 16) = floatx4{p[4], p[5], p[6], p[7]};
    }
    if (r0 + 4 * C::KT < k1) load(r0 + 4 * C::KT), look_up(min(r0 + 8 * C::KT, k1));
    top = xor_max<32>(xor_max<16>(top)) * scale2;
    // the reference follows the maximum only where that has risen by 2^8: sums and probabilities are relative to it
    if (__ballot(top > m + 8.f)) {
      const float was = m;
      m = fmaxf(m, top);
      const float alpha = __builtin_amdgcn_exp2f(was - (m == -INF ? 0.f : m));
      z *= alpha;
#pragma unroll
      for (int d = 0; d < C::NDT; ++d) O[d] *= alpha;
    }
    const float ref = m == -INF ? 0.f : m;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], scale2, -ref));
      z += p[i];
    }
    __builtin_amdgcn_wave_barrier();   // LDS operations of one wave complete in order
    const Probabilities<T, NP> both(p);
#pragma unroll
    for (int d = 0; d < C::NDT; ++d) O[d] = mma_values<C::LDV>(Vs + 16 * d, both, O[d]);
    __builtin_amdgcn_wave_barrier();
  }
  if (__ballot(odd)) {      // see split_nonfinite
    for (r0 = k0 + C::KT * wave; r0 < k1; r0 += 4 * C::KT) {
      if (r0 >= all_low && r0 + C::KT <= all_high) continue;
      float read[NP];
      const T* v[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = r0 + 16 * (i >> 2) + 4 * grp + (i & 3);
        read[i] = r < low || r >= high ? 0.f : 1.f;
        v[i] = value_row<T>(a, table, c, r, t_low, t_high, DH);
      }
      for (int d = 0; d < C::NDT; ++d) {
        float x[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) x[i] = v[i] ? to_f(v[i][16 * d + col]) : 0.f;
        floatx4 said = zero4();
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int i = 0; i < NP; ++i) x[i] = split_nonfinite(x[i]);
          said = Mfma<bf16>::mma(to_bf16x8(x, 0), to_bf16x8(read, 0), said);
        } else {
#pragma unroll
          for (int i = 0; i < NP; ++i) said = Mfma<float>::mma(split_nonfinite(x[i]), read[i], said);
        }
#pragma unroll
        for (int dd = 0; dd < C::NDT; ++dd)
#pragma unroll
          for (int i = 0; i < 4; ++i) O[dd][i] += dd == d ? said_by(said[i]) : 0.f;
      }
    }
  }
  z = xor_sum<32>(xor_sum<16>(z));
  if (bad) z = NAN_;
  if (grp == 0) sm[wave][col] = m, sz[wave][col] = z;
  __syncthreads();
  float M = fmaxf(fmaxf(sm[0][col], sm[1][col]), fmaxf(sm[2][col], sm[3][col]));
  const float mine = __builtin_amdgcn_exp2f(m - (M == -INF ? 0.f : M));
  float* Os = reinterpret_cast<float*>(smem) + wave * TILE_Q * DH;
#pragma unroll
  for (int d = 0; d < C::NDT; ++d)
    *reinterpret_cast<floatx4*>(Os + col * DH + 16 * d + 4 * grp) = O[d] * mine;
  __syncthreads();
  // 16 threads per query row, DH / 16 columns each
  constexpr int E = DH / 16;
  const int row = threadIdx.x >> 4, e0 = (threadIdx.x & 15) * E;
  M = fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row]));
  const float ref = M == -INF ? 0.f : M;
  float Z = 0.f, x[E];
#pragma unroll
  for (int w = 0; w < 4; ++w) Z += sz[w][row] * __builtin_amdgcn_exp2f(sm[w][row] - ref);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) x[e] += reinterpret_cast<float*>(smem)[(w * TILE_Q + row) * DH + e0 + e];
  }
  if (rho0 + row >= rows) return;
  if (it.pieces > 1) {
    const long at = ((long)(it.slot + it.piece) * a.h_kv + c) * TILE_Q + row;
    float* part = a.part + at * (DH + 2);
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<floatx2*>(part + e0 + e) = floatx2{x[e], x[e + 1]};
    if (e0 == 0) *reinterpret_cast<floatx2*>(part + DH) = floatx2{M, Z};
    return;
  }
  const long at = (long)(s.first + (rho0 + row) / a.g) * a.h + c * a.g + (rho0 + row) % a.g;
  const float inv = Z == 0.f ? 0.f : 1.f / Z;
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = Z == 0.f ? 0.f : x[e] * inv;
#pragma unroll
  for (int e = 0; e < E; e += 4) st4<T>((T*)a.o + at * DH + e0 + e, x + e);
  if (e0 == 0) a.lse[at] = log_of(ref, Z);
}

// ---- the read of many query rows -------------------------------------------------------------------
typedef float floatx16 __attribute__((ext_vector_type(16)));
DM_DEV floatx16 mma32(const u32x4& a, const u32x4& b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// V^T's fragment for 32 columns and 16 rows: lane l column l % 32, rows 4 (l / 32) + 0..3 and 8 + those, the order in which
// a 32 x 32 tile of scores leaves its rows to its lanes.
DM_DEV i16x8 values_fragment32(const bf16* v, int ldv) {
  const int lane = threadIdx.x & 63, s = lane & 15;
  v += (4 * (lane >> 5) + (s >> 2)) * ldv + 16 * ((lane >> 4) & 1) + 4 * (s & 3);
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(v));
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(v + 8 * ldv));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int DH> struct WideTile {
  static constexpr int KT = 64;            // cached rows of a step
  static constexpr int LDK = DH + 8;       // 16 rows' 16-byte pieces fill the banks once
  static constexpr int LDV = DH + 32;      // 4 rows' 64-byte pieces do
  static constexpr int KS = KT * LDK, VS = KT * LDV;      // a buffer of K, of V
  static constexpr int VPR = DH / 8, NK = DH / 16, ND = DH / 32;
};

// One block: a tile of 32 NW query rows (32 per wave), a key head and a piece of its cached rows, which pass through LDS in
// steps of 64 that all waves share. Scores as 32 x 32 tiles S^T = K Q^T: a lane holds one query row's scores, so maximum and
// sum need one exchange per step. The next step's scores run on the matrix cores while this one's exponentials run on the
// vector units, and this one's product with V beside the next one's maximum: K is a step ahead of V (two buffers each, their
// rows on their way in registers; rows sent to LDS directly were slower, since the compiler then waits for all of them before
// it reads V transposed). Rows of K are padded by 16 bytes, of V by 64: no bank conflicts.
// Probabilities are rounded to bf16 once before the product with V (their sum is not): outputs are off by 2.3e-3 in the 2-norm
// instead of 1.65e-3. In two parts, as the read of few rows takes them, the call below takes 1.47 ms instead of 1.06, 16 chunks of
// 64 tokens over 4096 rows 167 us instead of 131: half as many matrix instructions again, and as many vector ones.
// Bound by the matrix cores beside the exponentials: two prompts' chunks of 2048 tokens over 16384 rows, 32 heads of 128 on 8
// key heads (1.01 Tflop) 1.13 ms after a pause and 1.03 in a run of calls, 0.9 to 0.98 Pflop/s (a library product of 8192^3
// 1.10); the matrix cores are busy 48 % of the cycles at the clock that the power leaves. With 16-row tiles 4.1 ms.
template <int DH, int NW> __global__ __launch_bounds__(64 * NW, 8 / NW) void k_paged_read_wide(PagedArgs a) {
  using C = WideTile<DH>;
  constexpr int NT = 64 * NW, ROWS = 32 * NW, NL = C::KT * C::VPR / NT;    // 16-byte loads per thread of K and of V
  extern __shared__ __attribute__((aligned(16))) char smem[];
  bf16* const Ks = reinterpret_cast<bf16*>(smem);
  bf16* const Vs = Ks + 2 * C::KS;
  __shared__ int any_odd, any_bad;
  const int c = uniform(blockIdx.x % a.h_kv), lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Item it = find_item<ROWS, true>(a, blockIdx.x / a.h_kv);
  if (it.b < 0) return;
  make_uniform(it);
  const Seq& s = it.s;
  const int rows = s.n * a.g, rho0 = it.tile * ROWS;
  const int j_first = uniform(rho0 / a.g), j_last = uniform((min(rho0 + ROWS, rows) - 1) / a.g);
  const int rho = rho0 + 32 * wave + col, j = rho / a.g, head = c * a.g + rho % a.g;
  const bool live = rho < rows;
  const int high = live ? s.high(a, j) : 0, low = live ? s.low(a, j) : 0;
  const int t_low = s.low(a, j_first), t_high = s.bad ? 0 : s.high(a, j_last);
  const int base = t_low & -TILE_K, tiles = max(0, (t_high - base + TILE_K - 1) / TILE_K);
  const int each = uniform((tiles + it.pieces - 1) / it.pieces);
  const int k0 = base + it.piece * each * TILE_K, k1 = min(k0 + each * TILE_K, t_high);
  // rows from this on and below that are read by all of the wave's live query rows
  const int all_low = s.low(a, uniform(min(rho0 + 32 * wave + 31, rows - 1) / a.g));
  const int all_high = s.high(a, uniform(min(rho0 + 32 * wave, rows - 1) / a.g));

  u32x4 qf[C::NK];
  {
    const bf16* q = (const bf16*)a.q + (long)(s.first + j) * a.q_token + (long)head * a.q_head;
#pragma unroll
    for (int i = 0; i < C::NK; ++i) {
      qf[i] = live ? ld_global<u32x4>(q + 16 * i + 8 * half) : u32x4{0, 0, 0, 0};
      carry_sign<bf16>(qf[i], a.scale2);
    }
  }
  const float scale2 = positive_scale(a.scale2);
  floatx16 O[C::ND];
#pragma unroll
  for (int d = 0; d < C::ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[d][i] = 0.f;
  float m = -INF, z = 0.f;     // z: this lane's share
  if (a.k_rows && it.piece == 0) {
    const long kr = (long)(s.first + j) * a.kr_token + (long)c * a.kr_head, vr = (long)(s.first + j) * a.vr_token + (long)c * a.vr_head;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < C::NK; ++i) {
      const u32x4 k = live ? ld_global<u32x4>((const bf16*)a.k_rows + kr + 16 * i + 8 * half) : u32x4{0, 0, 0, 0};
      float x[8], y[8];
      unpack16<bf16>(uint4{k[0], k[1], k[2], k[3]}, x);
      unpack16<bf16>(uint4{qf[i][0], qf[i][1], qf[i][2], qf[i][3]}, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(x[e], y[e], dot);
    }
    dot = xor_sum<32>(dot);
    m = dot * scale2;
    const float p = __builtin_amdgcn_exp2f(fmaf(dot, scale2, m == -INF ? 0.f : -m));
    z = half == 0 ? p : 0.f;
#pragma unroll
    for (int d = 0; d < C::ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (live) unpack4<bf16>(ld_global<u32x2>((const bf16*)a.v_rows + vr + 32 * d + 8 * i + 4 * half), v);
#pragma unroll
        for (int e = 0; e < 4; ++e) O[d][4 * i + e] = p * v[e];
      }
  }

  const int32_t* table = a.table + (long)it.b * a.cols;
  const int in_page = (1 << a.page_shift) - 1;
  bool bad = s.bad;
  // load i of a wave: 64 / VPR (4 or 8) rows, of one page; the lane's place from the first of them on
  constexpr int AT_ONCE = 64 / C::VPR;
  const int my_row = lane / C::VPR, my_col = lane % C::VPR * 8;
  const uint32_t my_off = (uint32_t)(my_row * DH + my_col) * 2;
  auto first_row = [&](int i) { return (i * NW + wave) * AT_ONCE; };
  struct Rows {
    int page[NL];
    u32x4 x[NL];
  } kr, vr;
  auto look_up = [&](Rows& w, int r0) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = r0 + first_row(i);
      w.page[i] = page_of(a, table, r, r < t_high && r + AT_ONCE > t_low, bad);
    }
  };
  auto load = [&](Rows& w, int r0, const void* pages, long stride) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const long off = w.page[i] * stride + (((long)c << a.page_shift) + ((r0 + first_row(i)) & in_page)) * DH;
      w.x[i] = ld_global<u32x4>((const char*)((const bf16*)pages + off) + my_off);
    }
  };
  auto store_k = [&](int buf) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      *reinterpret_cast<u32x4*>(Ks + buf * C::KS + (first_row(i) + my_row) * C::LDK + my_col) = kr.x[i];
  };
  const int edge_low = s.low(a, j_last), edge_high = s.high(a, j_first);   // rows that all query rows of the tile read
  // In steps that some query row does not read all of, values that are not finite count 0 here (a product with a probability
  // of 0 would make it NaN) and are added at the end, for the query rows that read them.
  auto is_edge = [&](int r0) { return r0 < edge_low || r0 + C::KT > edge_high; };
  auto store_v = [&](int r0, int buf) {
    if (is_edge(r0)) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int r = r0 + first_row(i) + my_row;
        if (r < t_low || r >= t_high) vr.x[i] = u32x4{0, 0, 0, 0};    // whatever lies there
        if (any_nonfinite<bf16>(vr.x[i])) {
          any_odd = 1;
          clear_nonfinite<bf16>(vr.x[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i)
      *reinterpret_cast<u32x4*>(Vs + buf * C::VS + (first_row(i) + my_row) * C::LDV + my_col) = vr.x[i];
  };
  auto scores = [&](int buf, floatx16 (&S)[2]) {
    const bf16* K = Ks + buf * C::KS + col * C::LDK + 8 * half;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[t][i] = 0.f;
#pragma unroll
    for (int i = 0; i < C::NK; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) S[t] = mma32(*reinterpret_cast<const u32x4*>(K + 32 * t * C::LDK + 16 * i), qf[i], S[t]);
  };
  // scores of rows r0 + 32 t + 8 (i / 4) + 4 half + i % 4 in S[t][i]
  auto is_masked = [&](int r0) { return r0 < all_low || r0 + C::KT > all_high; };
  auto mask = [&](int r0, floatx16 (&S)[2]) {
    const int from = low - r0 - 4 * half, to = high - r0 - 4 * half;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 32 * t + 8 * (i >> 2) + (i & 3);
        if (r < from || r >= to) S[t][i] = -INF;
      }
  };
  auto largest = [&](const floatx16 (&S)[2]) {
    float top = S[0][0];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i) top = __builtin_elementwise_maximum(top, S[0][i]);
      top = __builtin_elementwise_maximum(top, S[1][i]);
    }
    const LanePair both = lane_pair<32>(top);
    return __builtin_elementwise_maximum(both.a, both.b) * scale2;
  };
  auto follow = [&](float top) {     // as in k_paged_read
    if (__ballot(top > m + 8.f)) {
      const float was = m;
      m = fmaxf(m, top);
      const float alpha = __builtin_amdgcn_exp2f(was - (m == -INF ? 0.f : m));
      z *= alpha;
#pragma unroll
      for (int d = 0; d < C::ND; ++d) O[d] *= alpha;
    }
  };
  // the exponentials number at .. at + n - 1 of a step's 32, packed eight by eight
  u32x4 p[4];
  float e[32], sum[2];
  auto exponentials = [&](const floatx16 (&S)[2], float ref, int at, int n) {
#pragma unroll
    for (int i = at; i < at + n; ++i) {
      e[i] = __builtin_amdgcn_exp2f(fmaf(S[i >> 4][i & 15], scale2, -ref));
      sum[i & 1] = i < 2 ? e[i] : sum[i & 1] + e[i];
      if ((i & 7) == 7) p[i >> 3] = __builtin_bit_cast(u32x4, to_bf16x8(e, i - 7));
    }
  };
  // V^T's fragments of columns 64 u and rows 16 k of the step, and the products with them: number i = (k, u)
  constexpr int PAIRS = C::ND / 2;
  u32x4 vf[2];
  auto read_v = [&](const bf16* V, int i) {
#pragma unroll
    for (int d = 0; d < 2; ++d)
      vf[d] = __builtin_bit_cast(u32x4, values_fragment32(V + 16 * (i / PAIRS) * C::LDV + 64 * (i % PAIRS) + 32 * d, C::LDV));
  };
  if (threadIdx.x == 0) any_odd = any_bad = 0;
  __syncthreads();
  const int steps = k0 < k1 ? (k1 - k0 + C::KT - 1) / C::KT : 0;
  // step n's first row. Past the last step the next 64 rows again and again: a load's rows lie in one page from any multiple
  // of 16 on, but not from k1 on
  auto step_row = [&](int n) { return k0 + min(n, steps) * C::KT; };
  if (steps) {
    look_up(kr, k0), load(kr, k0, a.K, a.k_page);
    vr = kr, load(vr, k0, a.V, a.v_page);
    store_k(0), store_v(k0, 0);
    look_up(kr, step_row(1)), load(kr, step_row(1), a.K, a.k_page), store_k(1);
#pragma unroll
    for (int i = 0; i < NL; ++i) vr.page[i] = kr.page[i];       // V follows K by a step
    look_up(kr, step_row(2));
    __syncthreads();
    floatx16 S[2];
    scores(0, S);
    if (is_masked(k0)) mask(k0, S);
    follow(largest(S));
    __syncthreads();
    auto step = [&](int n, auto masked) {
      const int buf = n & 1;
      int next[NL];
      load(kr, step_row(n + 2), a.K, a.k_page);      // (past the last step: of page 0, not used)
      load(vr, step_row(n + 1), a.V, a.v_page);
#pragma unroll
      for (int i = 0; i < NL; ++i) next[i] = kr.page[i];
      look_up(kr, step_row(n + 3));
      // Each matrix product stands beside a share of the vector work, in this order (the compiler's own puts all
      // exponentials first, and each LDS read right before its product): the next step's scores beside the first 24 exponentials,
      // the products with V beside the others and the next maximum.
      floatx16 T[2];
      const float ref = m == -INF ? 0.f : m;
      const bf16* K = Ks + (buf ^ 1) * C::KS + col * C::LDK + 8 * half;
      const bf16* V = Vs + buf * C::VS;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) T[t][i] = 0.f;
      u32x4 kf[2] = {*reinterpret_cast<const u32x4*>(K), *reinterpret_cast<const u32x4*>(K + 32 * C::LDK)};
#pragma unroll
      for (int i = 0; i < C::NK; ++i) {
        const u32x4 k0 = kf[0], k1 = kf[1];
        if (i + 1 < C::NK) {
#pragma unroll
          for (int t = 0; t < 2; ++t) kf[t] = *reinterpret_cast<const u32x4*>(K + 32 * t * C::LDK + 16 * (i + 1));
        } else {
          read_v(V, 0);
        }
        T[0] = mma32(k0, qf[i], T[0]);
        T[1] = mma32(k1, qf[i], T[1]);
        exponentials(S, ref, i * (24 / C::NK), 24 / C::NK);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (masked) mask(step_row(n + 1), T);
      float top = T[0][0];
#pragma unroll
      for (int i = 0; i < 4 * PAIRS; ++i) {
        const u32x4 v0 = vf[0], v1 = vf[1];
        if (i + 1 < 4 * PAIRS) read_v(V, i + 1);
        const int d = 2 * (i % PAIRS);
        O[d] = mma32(v0, p[i / PAIRS], O[d]);
        O[d + 1] = mma32(v1, p[i / PAIRS], O[d + 1]);
        if (i < 2 * PAIRS) {
          exponentials(S, ref, 24 + i * (4 / PAIRS), 4 / PAIRS);
        } else {     // NaN where a score is NaN: the reference stays then, and the sum becomes NaN
#pragma unroll
          for (int x = (i - 2 * PAIRS) * (8 / PAIRS); x < (i - 2 * PAIRS + 1) * (8 / PAIRS); ++x) {
            top = __builtin_elementwise_maximum(top, T[0][x]);
            top = __builtin_elementwise_maximum(top, T[1][x]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      z += sum[0] + sum[1];
      const LanePair both = lane_pair<32>(top);
      follow(__builtin_elementwise_maximum(both.a, both.b) * scale2);
      S[0] = T[0], S[1] = T[1];
      // into the buffers of K of step n and V of step n - 1, which every wave has done with since the last barrier
      store_k(buf);
      store_v(step_row(n + 1), buf ^ 1);
#pragma unroll
      for (int i = 0; i < NL; ++i) vr.page[i] = next[i];
      __syncthreads();
    };
    for (int n = 0; n + 1 < steps; ++n) {
      if (is_masked(step_row(n + 1))) step(n, std::true_type());
      else step(n, std::false_type());
    }
    exponentials(S, m == -INF ? 0.f : m, 0, 32);
    z += sum[0] + sum[1];
    const bf16* V = Vs + ((steps - 1) & 1) * C::VS;
#pragma unroll
    for (int i = 0; i < 4 * PAIRS; ++i) {
      read_v(V, i);
#pragma unroll
      for (int d = 0; d < 2; ++d) O[2 * (i % PAIRS) + d] = mma32(vf[d], p[i / PAIRS], O[2 * (i % PAIRS) + d]);
    }
  }
  __syncthreads();
  if (any_odd) {
    for (int r0 = k0; r0 < k1; r0 += 16) {
      if (!is_edge(k0 + (r0 - k0) / C::KT * C::KT)) continue;
      float read[8];
      const bf16* v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {      // the lane's rows
        const int r = r0 + 8 * (i >> 2) + 4 * half + (i & 3);
        read[i] = r < low || r >= high ? 0.f : 1.f;
        v[i] = value_row<bf16>(a, table, c, r, t_low, t_high, DH);
      }
#pragma unroll
      for (int d = 0; d < C::ND; ++d) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = split_nonfinite(v[i] ? to_f(v[i][32 * d + col]) : 0.f);
        floatx16 said;
#pragma unroll
        for (int i = 0; i < 16; ++i) said[i] = 0.f;
        said = mma32(__builtin_bit_cast(u32x4, to_bf16x8(x, 0)), __builtin_bit_cast(u32x4, to_bf16x8(read, 0)), said);
#pragma unroll
        for (int i = 0; i < 16; ++i) O[d][i] += said_by(said[i]);
      }
    }
  }
  z = xor_sum<32>(z);
  if (bad) any_bad = 1;      // seen by the waves whose rows lie there
  __syncthreads();
  if (any_bad) z = NAN_;
  if (!live) return;
  const float ref = m == -INF ? 0.f : m;
  if (it.pieces > 1) {
    float* part = a.part + (((long)(it.slot + it.piece) * a.h_kv + c) * ROWS + 32 * wave + col) * (DH + 2);
#pragma unroll
    for (int d = 0; d < C::ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 2) *reinterpret_cast<floatx2*>(part + 32 * d + 8 * (i >> 2) + 4 * half + (i & 3)) = floatx2{O[d][i], O[d][i + 1]};
    if (half == 0) *reinterpret_cast<floatx2*>(part + DH) = floatx2{m, z};
    return;
  }
  const long at = (long)(s.first + j) * a.h + head;
  const float inv = 1.f / z;
#pragma unroll
  for (int d = 0; d < C::ND; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = z == 0.f ? 0.f : O[d][4 * i + e] * inv;
      st4<bf16>((bf16*)a.o + at * DH + 32 * d + 8 * i + 4 * half, x);
    }
  if (half == 0) a.lse[at] = log_of(ref, z);
}

// The pieces of a query tile, in their order: 16 threads a query row. Bound by latency: the plan, the maxima, then eight pieces'
// columns at a time (one token in eight pieces 4 us, 64 sequences 6, 8192 query rows of 8 key heads 11).
template <typename T, int DH, int ROWS> __global__ __launch_bounds__(256) void k_paged_join(PagedArgs a) {
  const int c = blockIdx.x % a.h_kv;
  Item it = find_item<ROWS, false>(a, blockIdx.x / a.h_kv);
  if (it.b < 0 || it.pieces == 1) return;
  make_uniform(it);
  constexpr int E = DH / 16;
  const int row = blockIdx.y * 16 + (threadIdx.x >> 4), e0 = (threadIdx.x & 15) * E, rho = it.tile * ROWS + row;
  if (rho >= it.s.n * a.g) return;
  const long step = (long)a.h_kv * ROWS * (DH + 2);
  const float* part = a.part + (((long)it.slot * a.h_kv + c) * ROWS + row) * (DH + 2);
  float M = -INF, Z = 0.f, x[E];
  // the row's 16 threads share its pieces' maxima and sums, then each adds its columns
  const int lane16 = threadIdx.x & 15;
  for (int i = lane16; i < it.pieces; i += 16) M = fmaxf(M, part[i * step + DH]);
  M = group16_max(M);
  const float ref = M == -INF ? 0.f : M;
  for (int i = lane16; i < it.pieces; i += 16) {
    const floatx2 mz = *reinterpret_cast<const floatx2*>(part + i * step + DH);
    Z += __builtin_amdgcn_exp2f(mz[0] - ref) * mz[1];
  }
  Z = group16_sum(Z);
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll 8
  for (int i = 0; i < it.pieces; ++i) {
    const float* p = part + i * step;
    const float f = __builtin_amdgcn_exp2f(p[DH] - ref);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const floatx2 v = *reinterpret_cast<const floatx2*>(p + e0 + e);
      x[e] = fmaf(f, v[0], x[e]);
      x[e + 1] = fmaf(f, v[1], x[e + 1]);
    }
  }
  const long at = (long)(it.s.first + rho / a.g) * a.h + c * a.g + rho % a.g;
  const float inv = 1.f / Z;
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = Z == 0.f ? 0.f : x[e] * inv;
#pragma unroll
  for (int e = 0; e < E; e += 4) st4<T>((T*)a.o + at * DH + e0 + e, x + e);
  if (e0 == 0) a.lse[at] = log_of(ref, Z);
}

// ---- the weights -------------------------------------------------------------------------------
// The logarithm of a sum in units of ln 2, with what a sum of 0 (no row read, or scores of -inf) stands for: weights of 0.
DM_DEV float lse_of(float lse) { return lse == -INF ? INF : lse * LOG2E; }

// weights[b, c, r] += the sum over the sequence's query rows of exp(score - lse), from scores that the read kept: a thread
// takes 4 cached rows and goes over the query rows; 32 cached rows of one query row lie together, a cache line for both sides (12
// chunks of 13 fp32 tokens over 1824 to 6130 rows, 32 heads on 16: 18.8 us, with 4 rows of all query rows together 45.5). 32
// sequences of 3000 to 16384 rows, 32 heads on 8 key heads: 14.5 us; 24 chunks of up to 8 tokens over 50 to 4001 rows on 16
// heads 5.8 (four query rows on their way; with one 1.8 more, with eight the other call 4 more).
__global__ __launch_bounds__(256) void k_paged_weights_of(PagedArgs a) {
  constexpr int AT_ONCE = 4;      // query rows on their way
  const int c = uniform(blockIdx.x % a.h_kv);
  Item it = find_item<0, true>(a, blockIdx.x / a.h_kv);
  if (it.b < 0) return;
  make_uniform(it);
  const Seq& s = it.s;
  if (s.bad) return;
  const int t_low = s.low(a, 0), t_high = s.high(a, s.n - 1);
  const int base = t_low & -TILE_K, tiles = max(0, (t_high - base + TILE_K - 1) / TILE_K);
  const int each = uniform((tiles + it.pieces - 1) / it.pieces);
  const int k0 = base + it.piece * each * TILE_K, k1 = min(k0 + each * TILE_K, t_high);
  const long cap = (long)a.cols << a.page_shift;
  const float scale2 = positive_scale(a.scale2);
  float* w = a.weights + ((long)it.b * a.h_kv + c) * cap;
  for (int r = k0 + 4 * threadIdx.x; r < k1; r += 1024) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int rows = s.n * a.g;
    const float* x = a.scores + scores_at(a, s, c) + (long)(r >> 5) * (32L * rows) + (r & 31);
    const float* lse = a.lse + (long)s.first * a.h + c * a.g;
    int j = 0, i = 0;      // the query row's token and head
    for (int rho = 0; rho < rows; rho += AT_ONCE) {
      floatx4 v[AT_ONCE];
      float lse2[AT_ONCE];
      int token[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        v[u] = *reinterpret_cast<const floatx4*>(x + 32L * min(rho + u, rows - 1));
        lse2[u] = lse[(long)min(j, s.n - 1) * a.h + i];
        token[u] = j;
        if (++i == a.g) i = 0, ++j;
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int low = s.low(a, token[u]), high = token[u] < s.n ? s.high(a, token[u]) : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += r + e >= low && r + e < high ? __builtin_amdgcn_exp2f(fmaf(v[u][e], scale2, -lse_of(lse2[u]))) : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r + e >= t_low && r + e < t_high) w[r + e] += sum[e];
  }
}

// The same with the scores computed again: a wave holds 32 cached rows as fragments and goes over all query tiles, so each
// weight has one writer and one order of its sum. fp32, seven sequences of up to 130 tokens over up to 1501 rows, a window of
// 256: 15 us, most of it latency.
template <typename T, int DH> __global__ __launch_bounds__(256) void k_paged_weights(PagedArgs a) {
  using C = Tile<T, DH>;
  constexpr int KT = 32;      // cached rows of a step
  const int c = uniform(blockIdx.x % a.h_kv), lane = threadIdx.x & 63, grp = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Item it = find_item<0, true>(a, blockIdx.x / a.h_kv);
  if (it.b < 0) return;
  make_uniform(it);
  const Seq& s = it.s;
  if (s.bad) return;
  const int rows = s.n * a.g, t_low = s.low(a, 0), t_high = s.high(a, s.n - 1);
  const int base = t_low & -TILE_K, tiles = max(0, (t_high - base + TILE_K - 1) / TILE_K);
  const int each = uniform((tiles + it.pieces - 1) / it.pieces);
  const int k0 = base + it.piece * each * TILE_K, k1 = min(k0 + each * TILE_K, t_high);
  const int32_t* table = a.table + (long)it.b * a.cols;
  const int in_page = (1 << a.page_shift) - 1;
  float* w = a.weights + ((long)it.b * a.h_kv + c) * ((long)a.cols << a.page_shift);
  // Few query rows: each wave takes cached rows of its own; many: the waves share them and take the query tiles in turn
  // (the call above 15 us so, 23 without)
  __shared__ float part[2][4][KT];
  const bool shared = rows > 4 * TILE_Q;
  const int step = shared ? KT : 4 * KT, q_first = shared ? TILE_Q * wave : 0, q_step = shared ? 4 * TILE_Q : TILE_Q;
  int buf = 0;
  for (int r0 = k0 + (shared ? 0 : KT * wave); r0 < k1; r0 += step, buf ^= 1) {
    u32x4 kf[2][C::NF];
    bool bad = false;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = r0 + 16 * t;
      const long page = page_of(a, table, r, r < t_high && r + 16 > t_low, bad);
      const T* K = (const T*)a.K + page * a.k_page + (((long)c << a.page_shift) + (r & in_page)) * DH;
#pragma unroll
      for (int i = 0; i < C::NF; ++i) kf[t][i] = ld_global<u32x4>(K + col * DH + i * 4 * C::V + grp * C::V);
    }
    float sum[2][4] = {};
    // the tokens that read one of these rows; a tile of their query rows is on its way while the one before is used
    const int past = s.len - s.n;
    const int j0 = max(0, r0 - past + (a.k_rows ? 1 : 0)), j1 = a.window ? min((long)s.n, (long)r0 - past + KT - 1 + a.window) : s.n;
    u32x4 qf[C::NF];
    float lse2 = 0.f;
    auto fetch = [&](int rho0) {
      const int rho = min(rho0 + col, rows - 1), j = rho / a.g, head = c * a.g + rho % a.g;
      const T* q = (const T*)a.q + (long)(s.first + j) * a.q_token + (long)head * a.q_head;
#pragma unroll
      for (int i = 0; i < C::NF; ++i) qf[i] = ld_global<u32x4>(q + i * 4 * C::V + grp * C::V);
      lse2 = lse_of(a.lse[(long)(s.first + j) * a.h + head]);
    };
    int rho0 = j0 * a.g + q_first;
    if (rho0 < j1 * a.g) fetch(rho0);
    for (; rho0 < j1 * a.g; rho0 += q_step) {
      const int rho = rho0 + col, j = rho / a.g;
      const bool live = rho < rows;
      const int high = live ? s.high(a, j) : 0, low = live ? s.low(a, j) : 0;
      floatx4 acc[2];
      const float minus = -lse2;
      mma_scores<T, C::NF / 2>(kf, qf, acc);    // (two chains: more of them take more registers than leave room for three waves)
      if (rho0 + q_step < j1 * a.g) fetch(rho0 + q_step);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = r0 + 16 * t + 4 * grp + i;
          if (r >= low && r < high) sum[t][i] += __builtin_amdgcn_exp2f(fmaf(acc[t][i], a.scale2, minus));
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + 16 * t + 4 * grp + i;
        const float x = group16_sum(sum[t][i]);
        if (shared) {
          if (col == 0) part[buf][wave][r - r0] = bad ? NAN_ : x;
        } else if (col == 0 && r >= t_low && r < t_high) {
          w[r] += bad ? NAN_ : x;
        }
      }
    if (shared) {     // (the other buffer's sums are read before the next barrier)
      __syncthreads();
      const int r = r0 + threadIdx.x;
      if (threadIdx.x < KT && r >= t_low && r < t_high)
        w[r] += (part[buf][0][threadIdx.x] + part[buf][1][threadIdx.x]) + (part[buf][2][threadIdx.x] + part[buf][3][threadIdx.x]);
    }
  }
}

// The same for many query rows: a block takes 64 cached rows, each wave all of them against 32 query rows at a time (every
// fragment of Q is used twice), the waves' sums are added through LDS. Bound by the exponentials beside the products: two
// prompts' chunks of 2048 tokens over 16384 rows, 32 heads of 128 on 8 key heads: 0.86 ms, with 16-row tiles 1.84.
template <int DH> __global__ __launch_bounds__(256, 2) void k_paged_weights_wide(PagedArgs a) {
  constexpr int NK = DH / 16;
  __shared__ float part[2][4][TILE_K];
  const int c = uniform(blockIdx.x % a.h_kv), lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Item it = find_item<0, true>(a, blockIdx.x / a.h_kv);
  if (it.b < 0) return;
  make_uniform(it);
  const Seq& s = it.s;
  if (s.bad) return;
  const int rows = s.n * a.g, t_low = s.low(a, 0), t_high = s.high(a, s.n - 1), past = s.len - s.n;
  const int base = t_low & -TILE_K, tiles = max(0, (t_high - base + TILE_K - 1) / TILE_K);
  const int each = uniform((tiles + it.pieces - 1) / it.pieces);
  const int k0 = base + it.piece * each * TILE_K, k1 = min(k0 + each * TILE_K, t_high);
  const int32_t* table = a.table + (long)it.b * a.cols;
  const int in_page = (1 << a.page_shift) - 1;
  float* w = a.weights + ((long)it.b * a.h_kv + c) * ((long)a.cols << a.page_shift);
  int buf = 0;
  for (int r0 = k0; r0 < k1; r0 += TILE_K, buf ^= 1) {
    u32x4 kf[2][NK];
    bool bad = false;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int page[2];     // of 16 rows each
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + 32 * t + 16 * e;
        page[e] = page_of(a, table, r, r < t_high && r + 16 > t_low, bad);
      }
      const long at = ((long)c << a.page_shift) + ((r0 + 32 * t + col) & in_page);
      const bf16* K = (const bf16*)a.K + (col < 16 ? page[0] : page[1]) * a.k_page + at * DH + 8 * half;
#pragma unroll
      for (int i = 0; i < NK; ++i) kf[t][i] = ld_global<u32x4>(K + 16 * i);
    }
    const int j0 = max(0, r0 - past + (a.k_rows ? 1 : 0)), j1 = a.window ? min((long)s.n, (long)r0 - past + TILE_K - 1 + a.window) : s.n;
    float sum[2][16];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[t][i] = 0.f;
    u32x4 qf[NK];
    float lse2 = INF;
    auto fetch = [&](int rho0) {
      const int rho = min(rho0 + col, rows - 1), j = rho / a.g, head = c * a.g + rho % a.g;
      const bf16* q = (const bf16*)a.q + (long)(s.first + j) * a.q_token + (long)head * a.q_head + 8 * half;
#pragma unroll
      for (int i = 0; i < NK; ++i) qf[i] = ld_global<u32x4>(q + 16 * i);
      lse2 = rho0 + col < rows ? lse_of(a.lse[(long)(s.first + j) * a.h + head]) : INF;
    };
    int rho0 = j0 * a.g + 32 * wave;
    if (rho0 < j1 * a.g) fetch(rho0);
    for (; rho0 < j1 * a.g; rho0 += 128) {
      const int j = min(rho0 + col, rows - 1) / a.g;
      const float minus = -lse2;
      floatx16 S[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) S[t][i] = 0.f;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        S[0] = mma32(kf[0][i], qf[i], S[0]);
        S[1] = mma32(kf[1][i], qf[i], S[1]);
      }
      if (rho0 + 128 < j1 * a.g) fetch(rho0 + 128);
      const int first = uniform(rho0 / a.g), last = uniform((min(rho0 + 32, rows) - 1) / a.g);
      if (r0 < s.low(a, last) || r0 + TILE_K > s.high(a, first)) {
        const int from = s.low(a, j) - r0 - 4 * half, to = s.high(a, j) - r0 - 4 * half;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = 32 * t + 8 * (i >> 2) + (i & 3);
            sum[t][i] += r < from || r >= to ? 0.f : __builtin_amdgcn_exp2f(fmaf(S[t][i], a.scale2, minus));
          }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[t][i] += __builtin_amdgcn_exp2f(fmaf(S[t][i], a.scale2, minus));
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = lanes_sum<1, 16>(sum[t][i]);
        if (col == 0) part[buf][wave][32 * t + 8 * (i >> 2) + 4 * half + (i & 3)] = bad ? NAN_ : x;
      }
    __syncthreads();     // (the other buffer's sums are read before the next barrier)
    const int r = r0 + threadIdx.x;
    if (threadIdx.x < TILE_K && r >= t_low && r < t_high)
      w[r] += (part[buf][0][threadIdx.x] + part[buf][1][threadIdx.x]) + (part[buf][2][threadIdx.x] + part[buf][3][threadIdx.x]);
  }
}

// ---- eviction ------------------------------------------------------------------------------------
struct EvictArgs {
  const void *K, *V;
  void *K_out, *V_out;
  const float* weights;
  float* weights_out;
  const int32_t *table, *lengths, *new_table;
  int32_t *rows, *lengths_out;
  long k_page, v_page;
  int B, h, n_pages, cols, new_cols, page_shift, keep, sinks, recent;
};

// The order of weights as whole numbers (NaN above all, -0 as 0).
DM_DEV uint32_t weight_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : (b >> 31 ? ~b : b | 0x80000000u);
}

// One block per sequence and key head: the weight of the last row to be kept by its bits, eight at a time from the top
// (a histogram over the rows that agree so far), then the rows in order: those above it, and of those equal to it the first.
// A thread takes 4 rows in turn; the first KEYS * 4096 rows' weights stay in registers. Eight histograms, by lane, since weights
// share their first bits; one set for each pass, cleared before the first. Bound by its passes'
// latencies (one sequence of 2304 rows and 16 heads 8.4 us, 32 of 3000 to 16384 rows and 8 heads 15.3; with scans by shuffles,
// one set of histograms and a sum over the waves' totals in each thread 15.7 and 22.4).
constexpr int KEYS = 4, COPIES = 8, COPY = 256 + 8;      // a copy's first banks lie 8 behind the one's before
struct Selection {
  int hist[4][COPIES * COPY];
  int total[KEYS][16];      // rows kept of wave w's turn k, ties << 16
  int digit, above;
};

// of the need-th largest: its digit, and how many rows have a larger one. By the first wave: lane l takes digits 4 (63 - l) ..
// + 3, from the largest.
DM_DEV void find_digit(Selection& sh, const int* hist, int need) {
  const int lane = threadIdx.x & 63, d0 = 4 * (63 - lane);
  typedef int intx4 __attribute__((ext_vector_type(4)));
  intx4 n = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < COPIES; ++k) n += *reinterpret_cast<const intx4*>(hist + k * COPY + d0);
  const int sum = (n[0] + n[1]) + (n[2] + n[3]), upto = wave_upto(sum);
  int above = upto - sum;
  if (above < need && upto >= need) {
    int d = 3;
    while (d > 0 && above + n[d] < need) above += n[d--];
    sh.digit = d0 + d;
    sh.above = above;
  }
}

__global__ __launch_bounds__(1024) void k_evict_select(EvictArgs a) {
  __shared__ Selection sh;
  const int c = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long cap = (long)a.cols << a.page_shift;
  const int len = a.lengths[b] < 0 || a.lengths[b] > cap ? 0 : a.lengths[b];
  const int left = min(len, a.keep);
  int32_t* rows = a.rows + ((long)b * a.h + c) * a.keep;
  if (c == 0 && threadIdx.x == 0) a.lengths_out[b] = left;
  for (long i = left + (long)threadIdx.x; i < a.keep; i += 1024) rows[i] = -1;     // (keep may be any more than there are)
  if (len <= a.keep) {
    for (int i = threadIdx.x; i < left; i += 1024) rows[i] = i;
    return;
  }
  const float* w = a.weights + ((long)b * a.h + c) * cap;
  const int lo = a.sinks, hi = len - a.recent;      // rows that may go
  // rows 4 q .. 4 q + 3 (the capacity is a multiple of 16)
  auto keys_of = [&](int q, uint32_t (&u)[4]) {
    if (4 * q < len) {
      const floatx4 v = *reinterpret_cast<const floatx4*>(w + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = weight_order(v[e]);
    }
  };
  uint32_t held[KEYS][4];
#pragma unroll
  for (int k = 0; k < KEYS; ++k) keys_of(threadIdx.x + 1024 * k, held[k]);
  uint32_t key = 0;
  int need = a.keep - a.sinks - a.recent;           // of them stay (less than there are)
  if (need > 0) {
    for (int i = threadIdx.x; i < 4 * COPIES * COPY; i += 1024) (&sh.hist[0][0])[i] = 0;
    __syncthreads();
    for (int shift = 24; shift >= 0; shift -= 8) {
      int* hist = sh.hist[shift >> 3];
      const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      auto count = [&](int q, const uint32_t (&u)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * q + e >= lo && 4 * q + e < hi && (u[e] & mask) == key)
            atomicAdd(hist + (lane & (COPIES - 1)) * COPY + ((u[e] >> shift) & 255), 1);
      };
#pragma unroll
      for (int k = 0; k < KEYS; ++k) count(threadIdx.x + 1024 * k, held[k]);
      for (int q = threadIdx.x + 1024 * KEYS; 4 * q < hi; q += 1024) {
        uint32_t u[4];
        keys_of(q, u);
        count(q, u);
      }
      __syncthreads();
      if (wave == 0) find_digit(sh, hist, need);
      __syncthreads();
      key |= (uint32_t)sh.digit << shift;
      need -= sh.above;
    }
  } else {
    key = 0xffffffffu;
  }
  // need: how many of the rows equal to key stay
  int at = 0, equal = 0;
  for (int q0 = 0; 4 * q0 < len; q0 += 1024 * KEYS) {
    int sure[KEYS], tie[KEYS], before[KEYS];     // bits of a thread's rows; rows of the wave before the thread's, ties << 16
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
      const int q = q0 + threadIdx.x + 1024 * k;
      uint32_t u[4];
      if (q0) keys_of(q, u);
      else u[0] = held[k][0], u[1] = held[k][1], u[2] = held[k][2], u[3] = held[k][3];
      sure[k] = tie[k] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * q + e;
        if (i < len && (i < lo || i >= hi || u[e] > key)) sure[k] |= 1 << e;
        else if (i < len && u[e] == key) tie[k] |= 1 << e;
      }
      const int mine = __popc(sure[k]) + (__popc(tie[k]) << 16);
      const int upto = wave_upto(mine);
      before[k] = upto - mine;
      if (lane == 63) sh.total[k][wave] = upto;
    }
    __syncthreads();
    // rows before each wave's turn (16384 rows at most: ties stay below 32 bits)
    const int turn = sh.total[lane >> 4][lane & 15], turns = wave_upto(turn);
#pragma unroll
    for (int k = 0; k < KEYS; ++k) {
      const int ahead = before[k] + __builtin_amdgcn_readlane(turns - turn, 16 * k + wave);
      int s = at + (ahead & 0xffff), t = equal + (ahead >> 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool is_sure = sure[k] >> e & 1, is_tie = tie[k] >> e & 1;
        if (is_sure || (is_tie && t < need)) rows[s + min(t, need)] = 4 * (q0 + (int)threadIdx.x + 1024 * k) + e;
        s += is_sure;
        t += is_tie;
      }
    }
    const int all = __builtin_amdgcn_readlane(turns, 63);
    at += all & 0xffff;
    equal += all >> 16;
    __syncthreads();
  }
}

// One thread per 16 bytes of a kept row of K and of V. Bound by the rows' bytes: 32 sequences, 4096 kept rows of 128 on 8 heads
// each (1.08 GB) 222 us, 4.85 TB/s, what a large copy reaches.
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a, int row_bytes, int esize) {
  const int c = blockIdx.y, b = blockIdx.z, per = row_bytes / 16;
  const long at = blockIdx.x * 256L + threadIdx.x;
  const long i = at / per;
  const int v = (int)(at % per);
  const long cap = (long)a.cols << a.page_shift, new_cap = (long)a.new_cols << a.page_shift;
  if (i >= new_cap) return;
  const int len = a.lengths[b] < 0 || a.lengths[b] > cap ? 0 : a.lengths[b];
  const int left = min(len, a.keep), in_page = (1 << a.page_shift) - 1;
  if (i >= left) {
    if (v == 0) a.weights_out[((long)b * a.h + c) * new_cap + i] = 0.f;
    return;
  }
  const int r = a.rows[((long)b * a.h + c) * a.keep + i];
  if (v == 0) a.weights_out[((long)b * a.h + c) * new_cap + i] = a.weights[((long)b * a.h + c) * cap + r];
  const int src = a.table[(long)b * a.cols + (r >> a.page_shift)], dst = a.new_table[(long)b * a.new_cols + (i >> a.page_shift)];
  if (dst < 0 || dst >= a.n_pages) return;
  const bool bad = src < 0 || src >= a.n_pages;
  const long from = (((long)c << a.page_shift) + (r & in_page)) * row_bytes + v * 16;
  const long to = (((long)c << a.page_shift) + (i & in_page)) * row_bytes + v * 16;
  u32x4 k = {~0u, ~0u, ~0u, ~0u}, x = k;   // NaN in either type
  if (!bad) {
    k = *reinterpret_cast<const u32x4*>((const char*)a.K + src * a.k_page * esize + from);
    x = *reinterpret_cast<const u32x4*>((const char*)a.V + src * a.v_page * esize + from);
  }
  *reinterpret_cast<u32x4*>((char*)a.K_out + dst * a.k_page * esize + to) = k;
  *reinterpret_cast<u32x4*>((char*)a.V_out + dst * a.v_page * esize + to) = x;
}

// ---- host ------------------------------------------------------------------------------------------
int log2_of(int x) {
  for (int i = 0; i < 31; ++i)
    if (x == 1 << i) return i;
  return -1;
}

long query_tiles(const dm_paged_args* a, int rows) { return (long)a->n_tokens * (a->h / a->h_kv) / rows + a->B; }
// the most tiles of cached rows that a query tile can have, by the table's and the window's rows
long most_tiles(const dm_paged_args* a) {
  const long rows = (long)a->table_cols * a->page;
  return (a->window ? std::min(rows, (long)a->window + a->n_tokens + TILE_K) : rows) / TILE_K + 1;
}
// The plan's numbers: about `blocks` blocks over the key heads, but no more than there can be: blocks without a piece cost their
// look at the plan (one token over 1024 rows in pieces: 8.2 us with 8 blocks per CU wanted, 7.0 with 5, 6.0 with those that there can be).
int wanted(const dm_paged_args* a, int blocks, long tiles, int least) {
  return (int)std::max(1L, std::min((long)cdiv(blocks, a->h_kv), tiles * ((most_tiles(a) + least - 1) / least)));
}
constexpr int WEIGHT_BLOCKS = 8 * CUS;

// Which read a call takes, by the mean number of query rows of a sequence and key head: tiles of 16 rows while two of them
// hold those, of 128, or of 256 (us, bf16, 16 sequences of 4096 rows, 16 heads of 64 and 32 of 128 on 8 key heads:
// 24 rows 59 / 69 / 115 and 60 / 62 / 82, 48 rows 71 / 66 / 115 and 76 / 62 / 86, 256 rows 297 / 120 / 134 and 302 / 112 / 119,
// 512 rows 559 / 221 / 215 and 583 / 188 / 188; two sequences of 16384 rows, 8192 query rows: 4206 / 1340 / 1061). Pieces:
// what fills the CUs with the blocks that one holds (at 8192 query rows 1, 2 and 4 times as many: 1150, 1184, 1206 us).
// In one piece, with no join, while a tile's keys take no more than 128 KiB, or 256 with blocks for half of the CUs (a call / its
// kernels in a graph, pieces -> whole: one token, 16 heads of 64, 256 rows 18.1 / 8.9 -> 14.0 / 6.5 us, 512 rows 18.0 / 9.3 ->
// 13.4 / 7.8, 1024 rows 18.1 / 9.2 -> 13.4 / 10.4, 2048 rows 17.0 / 9.5 -> 14.5 / 14.3; 8 tokens over 2048 rows 23.4 / 24.0 ->
// 20.4 / 21.0; 7 chunks of 65 fp32 tokens, 8 heads of 64 on 4, over 1024 rows 43 -> 34). The larger tiles: up to 512 rows with
// blocks for half of the CUs (16 chunks of 64 tokens, 8 heads of 64, over 128, 512 and 1024 rows 21.9 -> 17.6, 21.6 -> 16.8 and
// 22.3 -> 24.9; 33 of 100 tokens, 16 heads of 128, 43 -> 33, 63 -> 54.5 and 106 -> 92; one of 1024 rows among 16 of 70 21 -> 33.6).
bool in_one_piece(const dm_paged_args* a) {
  const long bytes = (most_tiles(a) - 1) * TILE_K * a->dh * (long)esz(a->dtype);
  return bytes <= (query_tiles(a, TILE_Q) * a->h_kv >= CUS / 2 ? 256 << 10 : 128 << 10);
}
struct Form {
  int rows, blocks, least;     // query rows of a tile; blocks wanted; least tiles of cached rows in a piece
};
Form form_of(const dm_paged_args* a) {
  const int64_t mean = (int64_t)a->n_tokens * (a->h / a->h_kv) / a->B;
  if (a->dtype != DM_BF16 || mean <= 2 * TILE_Q) return {TILE_Q, 5 * CUS, in_one_piece(a) ? (int)most_tiles(a) : 2};
  Form f = mean <= 512 ? Form{128, 2 * CUS, 2} : Form{256, CUS, 2};
  if (most_tiles(a) <= 9 && query_tiles(a, f.rows) * a->h_kv >= CUS / 2) f.least = (int)most_tiles(a);
  return f;
}
// The scores of a call with weights are kept where they take no more room than the pages' keys, and 1 GiB: they lie under the table's
// whole width, which may be far more than the sequences' rows, and a pool may leave little memory beside it. Else they are computed
// again from the keys (us a call, kept / again: 64 tokens over 32768 rows, 32 heads of 128 on 8 key heads, 256 MiB of scores 1832 /
// 2354; 16 chunks of 8, 512 MiB, 791 / 848; fp32, 8 chunks of 32 over 16384 rows, 512 MiB, 981 / 1408).
constexpr double SCORE_BYTES = 1 << 30;
size_t score_floats(const dm_paged_args* a) {
  if (!a->weights || form_of(a).rows != TILE_Q) return 0;
  const double n = (double)a->n_tokens * a->h * (((int64_t)a->table_cols * a->page + 31) & -32);
  return n * 4 <= std::min(SCORE_BYTES, (double)a->n_pages * a->h_kv * a->page * a->dh * esz(a->dtype)) ? (size_t)n : 0;
}
int wanted(const dm_paged_args* a, const Form& f) { return wanted(a, f.blocks, query_tiles(a, f.rows), f.least); }
bool in_pieces(const dm_paged_args* a, const Form& f) { return most_tiles(a) > f.least; }
size_t part_floats(const dm_paged_args* a) {
  const Form f = form_of(a);
  return !in_pieces(a, f) ? 0 : (size_t)2 * wanted(a, f) * a->h_kv * f.rows * (a->dh + 2);
}
size_t part_bytes(const dm_paged_args* a) { return align256(part_floats(a) * 4); }

int check_pages(int dtype, int dh, int page, int n_pages, int cols, int B, int h_kv, const void* K, const void* V, int64_t k_page,
                int64_t v_page) {
  DM_REQUIRE(dtype == DM_BF16 || dtype == DM_F32, DM_ERR_INVALID, "dtype %d", dtype);
  DM_REQUIRE(dh == 64 || dh == 128, DM_ERR_UNSUPPORTED, "dh=%d (64 or 128)", dh);
  DM_REQUIRE(log2_of(page) >= 4 && page <= DM_PAGE_MAX, DM_ERR_UNSUPPORTED, "page=%d rows (a power of two, 16..%d)", page, DM_PAGE_MAX);
  DM_REQUIRE(B > 0 && h_kv > 0 && n_pages > 0 && cols > 0 && (int64_t)cols * page <= DM_PAGED_ROWS, DM_ERR_INVALID,
             "B=%d h_kv=%d n_pages=%d table_cols=%d of %d rows (at most %d rows)", B, h_kv, n_pages, cols, page, DM_PAGED_ROWS);
  DM_REQUIRE(B <= 65535 && h_kv <= 65535 && (int64_t)B * h_kv <= DM_PAGED_HEADS, DM_ERR_INVALID, "B=%d h_kv=%d (at most 65535, %d in all)",
             B, h_kv, DM_PAGED_HEADS);
  const int64_t least = (int64_t)h_kv * page * dh, unit = dtype == DM_BF16 ? 8 : 4;
  DM_REQUIRE(K && V && aligned16(K) && aligned16(V) && k_page >= least && v_page >= least && k_page % unit == 0 && v_page % unit == 0,
             DM_ERR_INVALID, "null or unaligned pages, strides %lld %lld (at least %lld, 16-byte steps)", (long long)k_page,
             (long long)v_page, (long long)least);
  return DM_OK;
}

int check_rows(const char* what, const void* p, int64_t token, int64_t head, int dtype) {
  const int64_t unit = dtype == DM_BF16 ? 8 : 4;
  DM_REQUIRE(p && aligned16(p) && token >= 0 && head >= 0 && token % unit == 0 && head % unit == 0, DM_ERR_INVALID,
             "%s: null or unaligned, strides %lld %lld (16-byte steps)", what, (long long)token, (long long)head);
  return DM_OK;
}

int check_paged(const dm_paged_args* a, bool write) {
  DM_REQUIRE(a != nullptr, DM_ERR_INVALID, "null arguments");
  if (const int rc = check_pages(a->dtype, a->dh, a->page, a->n_pages, a->table_cols, a->B, a->h_kv, a->K, a->V, a->k_page, a->v_page)) return rc;
  DM_REQUIRE(a->n_tokens >= 0 && (a->starts || a->n_tokens == a->B), DM_ERR_INVALID,
             "n_tokens=%d (without starts one per sequence, B=%d)", a->n_tokens, a->B);
  DM_REQUIRE(a->table && a->lengths, DM_ERR_INVALID, "null table or lengths");
  if (a->n_tokens == 0) return DM_OK;
  DM_REQUIRE((int64_t)a->n_tokens * std::max(a->h_kv, write ? 0 : a->h) <= DM_PAGED_TOKENS, DM_ERR_INVALID,
             "%d tokens of %d heads (at most %d rows)", a->n_tokens, std::max(a->h_kv, write ? 0 : a->h), DM_PAGED_TOKENS);
  if (write || a->k_rows || a->v_rows) {
    if (const int rc = check_rows("k_rows", a->k_rows, a->k_token, a->k_head, a->dtype)) return rc;
    if (const int rc = check_rows("v_rows", a->v_rows, a->v_token, a->v_head, a->dtype)) return rc;
  }
  if (write) return DM_OK;
  DM_REQUIRE(a->h > 0 && a->h % a->h_kv == 0 && a->h / a->h_kv <= 1024, DM_ERR_INVALID, "h=%d h_kv=%d", a->h, a->h_kv);
  DM_REQUIRE(a->window >= 0 && std::fabs(a->scale * LOG2E) < INF, DM_ERR_INVALID, "window=%d scale=%g (below 2.3e38)", a->window, a->scale);
  if (const int rc = check_rows("q", a->q, a->q_token, a->q_head, a->dtype)) return rc;
  DM_REQUIRE(a->o && aligned16(a->o) && a->lse, DM_ERR_INVALID, "null or unaligned o, null lse");
  const size_t need = dm_paged_workspace_bytes(a);
  DM_REQUIRE(a->workspace_bytes >= need && (need == 0 || (a->workspace && aligned16(a->workspace))), DM_ERR_WORKSPACE,
             "workspace %zu < %zu bytes", a->workspace_bytes, need);
  return DM_OK;
}

PagedArgs paged(const dm_paged_args* a) {
  PagedArgs r = {};
  r.q = a->q, r.K = a->K, r.V = a->V, r.k_rows = a->k_rows, r.v_rows = a->v_rows, r.o = a->o, r.lse = a->lse, r.weights = a->weights;
  r.part = (float*)a->workspace, r.table = a->table, r.lengths = a->lengths, r.starts = a->starts;
  r.q_token = a->q_token, r.q_head = a->q_head, r.k_page = a->k_page, r.v_page = a->v_page;
  r.kr_token = a->k_token, r.kr_head = a->k_head, r.vr_token = a->v_token, r.vr_head = a->v_head;
  r.B = a->B, r.h = a->h, r.h_kv = a->h_kv, r.g = a->h_kv ? a->h / a->h_kv : 1, r.n_pages = a->n_pages, r.cols = a->table_cols;
  r.page_shift = log2_of(a->page), r.N = a->n_tokens, r.window = a->window, r.scale2 = a->scale * LOG2E;
  return r;
}

template <int DH, int NW> int launch_wide(const PagedArgs& p, unsigned blocks, hipStream_t s) {
  constexpr int BYTES = 2 * (WideTile<DH>::KS + WideTile<DH>::VS) * 2;
  DM_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&k_paged_read_wide<DH, NW>), hipFuncAttributeMaxDynamicSharedMemorySize,
                             BYTES));     // of the current device, so in every call
  hipLaunchKernelGGL((k_paged_read_wide<DH, NW>), dim3(blocks), dim3(64 * NW), BYTES, s, p);
  return DM_OK;
}

template <typename T, int DH> int run_attention(const dm_paged_args* a, hipStream_t s) {
  const Form f = form_of(a);
  PagedArgs p = paged(a);
  p.want = wanted(a, f), p.least = f.least;
  if (score_floats(a)) p.scores = (float*)((char*)a->workspace + part_bytes(a));
  const long tiles = query_tiles(a, f.rows);
  const unsigned blocks = (unsigned)((p.want + tiles) * a->h_kv);
  const bool join = in_pieces(a, f);
  const dim3 joined((unsigned)(tiles * a->h_kv), f.rows / 16);
  if (f.rows == TILE_Q) {
    if (p.scores) hipLaunchKernelGGL((k_paged_read<T, DH, true>), dim3(blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_paged_read<T, DH, false>), dim3(blocks), dim3(256), 0, s, p);
    if (join) hipLaunchKernelGGL((k_paged_join<T, DH, TILE_Q>), joined, dim3(256), 0, s, p);
  }
  if constexpr (sizeof(T) == 2) {
    if (f.rows == 128) {
      if (const int rc = launch_wide<DH, 4>(p, blocks, s)) return rc;
      if (join) hipLaunchKernelGGL((k_paged_join<T, DH, 128>), joined, dim3(256), 0, s, p);
    } else if (f.rows == 256) {
      if (const int rc = launch_wide<DH, 8>(p, blocks, s)) return rc;
      if (join) hipLaunchKernelGGL((k_paged_join<T, DH, 256>), joined, dim3(256), 0, s, p);
    }
  }
  if (a->weights) {
    p.least = p.scores ? 1024 / TILE_K : 1;     // a round of a block's threads; a step
    p.want = wanted(a, WEIGHT_BLOCKS, a->B, p.least);
    const dim3 grid((unsigned)((p.want + (long)a->B) * a->h_kv));
    if (p.scores) {
      hipLaunchKernelGGL(k_paged_weights_of, grid, dim3(256), 0, s, p);
    } else {
      if constexpr (sizeof(T) == 2) {
        if (f.rows != TILE_Q) hipLaunchKernelGGL(k_paged_weights_wide<DH>, grid, dim3(256), 0, s, p);
      }
      if (f.rows == TILE_Q) hipLaunchKernelGGL((k_paged_weights<T, DH>), grid, dim3(256), 0, s, p);
    }
  }
  DM_HIP(hipGetLastError());
  return DM_OK;
}

}  // namespace

extern "C" {

size_t dm_paged_workspace_bytes(const dm_paged_args* a) {
  if (!a || a->h_kv <= 0 || a->B <= 0 || a->h < a->h_kv || a->n_tokens < 0 || (a->dh != 64 && a->dh != 128)) return 0;
  return part_bytes(a) + score_floats(a) * 4;
}

int dm_paged_write(const dm_paged_args* a, void* stream) {
  const int rc = check_paged(a, true);
  if (rc || a->n_tokens == 0) return rc;
  const PagedArgs p = paged(a);
  const int pieces = a->h_kv * 2 * (a->dh * (int)esz(a->dtype) / 16);      // 16 bytes each, of a token
  const dim3 grid((unsigned)std::min(cdiv(a->n_tokens, 4), 1 << 20), cdiv(pieces, 256));
  if (a->dtype == DM_BF16) hipLaunchKernelGGL(k_paged_write<bf16>, grid, dim3(256), 0, S(stream), p, log2_of(a->dh));
  else hipLaunchKernelGGL(k_paged_write<float>, grid, dim3(256), 0, S(stream), p, log2_of(a->dh));
  DM_HIP(hipGetLastError());
  return DM_OK;
}

int dm_paged_attention(const dm_paged_args* a, void* stream) {
  const int rc = check_paged(a, false);
  if (rc || a->n_tokens == 0) return rc;
  if (a->dtype == DM_BF16) return a->dh == 64 ? run_attention<bf16, 64>(a, S(stream)) : run_attention<bf16, 128>(a, S(stream));
  return a->dh == 64 ? run_attention<float, 64>(a, S(stream)) : run_attention<float, 128>(a, S(stream));
}

int dm_paged_evict(const dm_evict_args* a, void* stream) {
  DM_REQUIRE(a != nullptr, DM_ERR_INVALID, "null arguments");
  if (const int rc = check_pages(a->dtype, a->dh, a->page, a->n_pages, a->table_cols, a->B, a->h_kv, a->K, a->V, a->k_page, a->v_page)) return rc;
  const int64_t cap = (int64_t)a->table_cols * a->page, new_cap = (int64_t)a->new_cols * a->page;
  DM_REQUIRE(a->keep > 0 && a->sinks >= 0 && a->recent >= 0 && (int64_t)a->sinks + a->recent <= a->keep, DM_ERR_INVALID,
             "keep=%d sinks=%d recent=%d", a->keep, a->sinks, a->recent);
  DM_REQUIRE(a->new_cols > 0 && new_cap <= DM_PAGED_ROWS && new_cap >= std::min<int64_t>(a->keep, cap), DM_ERR_INVALID,
             "new_cols=%d pages do not hold %d rows", a->new_cols, a->keep);
  DM_REQUIRE(a->table && a->lengths && a->new_table && a->weights && a->weights_out && a->rows && a->lengths_out, DM_ERR_INVALID,
             "null argument");
  DM_REQUIRE(a->weights != a->weights_out && a->lengths != a->lengths_out, DM_ERR_INVALID, "an output in an input's place");
  EvictArgs p = {};
  p.K = a->K, p.V = a->V, p.K_out = a->K, p.V_out = a->V, p.weights = a->weights, p.weights_out = a->weights_out;
  p.table = a->table, p.lengths = a->lengths, p.new_table = a->new_table, p.rows = a->rows, p.lengths_out = a->lengths_out;
  p.k_page = a->k_page, p.v_page = a->v_page, p.B = a->B, p.h = a->h_kv, p.n_pages = a->n_pages, p.cols = a->table_cols;
  p.new_cols = a->new_cols, p.page_shift = log2_of(a->page), p.keep = a->keep, p.sinks = a->sinks, p.recent = a->recent;
  const int bytes = a->dh * (int)esz(a->dtype);
  hipLaunchKernelGGL(k_evict_select, dim3(a->h_kv, a->B), dim3(1024), 0, S(stream), p);
  hipLaunchKernelGGL(k_evict_move, dim3((unsigned)((new_cap * (bytes / 16) + 255) / 256), a->h_kv, a->B), dim3(256), 0, S(stream), p, bytes,
                     (int)esz(a->dtype));
  DM_HIP(hipGetLastError());
  return DM_OK;
}

}  // extern "C"
