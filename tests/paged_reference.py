"""The paged cache's operators from their definitions, in 64 bits on the CPU, one sequence and head at a time."""

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # half a step of a rounding, relative to the value


def gather(pages, table, b, n):
    """The first n rows of sequence b: [h_kv, n, dh] in 64 bits."""
    page = pages.shape[2]
    r = torch.arange(n)
    at = table[b, r // page].long()
    return pages[at, :, r % page].transpose(0, 1).double()


def attention(q, K, V, table, lengths, counts, k_self=None, v_self=None, window=0, scale=None):
    """(o, lse, added weights, bound of o, bound of lse, bound of the weights), all CPU tensors in 64 bits.

    The bounds count roundings. A score is a sum of dh products: at most (dh + 8) u sum |q k| scale off (u = 2^-24), and its
    exponential's argument, a difference of numbers of up to |s| and |lse| in units of ln 2, another 8 u (|s| + |lse|); sums
    over L rows L u. A probability, and with it each output's share, is off by d = that; with bf16 it is rounded once more
    before the product with V, and the output once."""
    N, h, dh = q.shape
    cap = table.shape[1] * K.shape[2]
    h_kv = K.shape[1]
    g = h // h_kv
    scale = 1 / math.sqrt(dh) if scale is None else scale
    u, half = 2.0 ** -24, HALF[q.dtype]
    q = q.double()
    o, bo = torch.zeros(N, h, dh, dtype=torch.float64), torch.zeros(N, h, dh, dtype=torch.float64)
    lse, bl = torch.full((N, h), -math.inf, dtype=torch.float64), torch.zeros(N, h, dtype=torch.float64)
    w, bw = (torch.zeros(len(lengths), h_kv, cap, dtype=torch.float64) for _ in range(2))
    t0 = 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        for c in range(h_kv):
            Kc, Vc = gather(K, table, b, length)[c], gather(V, table, b, length)[c]
            for a in range(c * g, c * g + g):
                for j in range(n):
                    t, p = t0 + j, length - n + j
                    high = p if k_self is not None else p + 1
                    low = max(0, p - window + 1) if window else 0
                    k, v = Kc[low:high], Vc[low:high]
                    if k_self is not None:
                        k = torch.cat([k, k_self[t, c].double()[None]])
                        v = torch.cat([v, v_self[t, c].double()[None]])
                    if not len(k):
                        continue
                    s = scale * (k @ q[t, a])
                    total = torch.logsumexp(s, 0)
                    e = torch.exp(s - total)
                    o[t, a], lse[t, a] = e @ v, total
                    d = u * ((dh + 8) * (abs(scale) * (k.abs() @ q[t, a].abs())).max() + 8 * (s.abs().max() + total.abs()) + len(k) + 16)
                    share = e @ v.abs()
                    bo[t, a] = share * (2 * d + (half if half > u else 0)) + half * o[t, a].abs()
                    bl[t, a] = d + 2 * u * total.abs()
                    m = max(0, high - low)
                    w[b, c, low:low + m] += e[:m]
                    bw[b, c, low:low + m] += 2 * d * e[:m]
        t0 += n
    return o, lse, w, bo, bl, bw + 16 * u * w


def evict(weights, lengths, keep, sinks, recent):
    """rows [B, h_kv, keep] by sorting (weight, -row)."""
    B, h, _ = weights.shape
    rows = torch.full((B, h, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for c in range(h):
            w = weights[b, c].tolist()
            order = sorted(range(n), key=lambda r: (not (r < sinks or r >= n - recent), -math.inf if math.isnan(w[r]) else -w[r], r))
            kept = sorted(order[:min(n, keep)]) if n > keep else range(n)
            for i, r in enumerate(kept):
                rows[b, c, i] = r
    return rows


def verify(x, ids, u, counts, y, temperature):
    """(tokens, accepted, logp) of rows x (64 bits), row by row."""
    N, V = x.shape
    tokens, logp = torch.full((N,), -1, dtype=torch.int64), torch.zeros(N, dtype=torch.float64)
    accepted, t = [], 0

    def dist(row, T):
        return torch.log_softmax(row.double() / (T or 1.0), 0)

    def proper(row, T):
        m = row.max()
        return not row.isnan().any() and m > -math.inf and (T == 0 or m < math.inf)

    for b, n in enumerate(counts):
        T, taken = float(temperature[b]), 0
        for j in range(n):
            i, last = t + j, j == n - 1
            d = None if last else int(ids[i + 1])
            has_y = y is not None and not last and T > 0
            if not proper(x[i], T) or (has_y and not proper(y[i], T)):
                logp[i] = math.nan
                break
            lp = dist(x[i], T)
            best = int((x[i] == x[i].max()).nonzero()[0])
            q = dist(y[i], T).exp() if has_y else None
            if not last and 0 <= d < V:
                ok = d == best if T == 0 else float(u[i, 0]) * (float(q[d]) if has_y else 1.0) < float(lp[d].exp())
                if ok:
                    tokens[i], logp[i], taken = d, lp[d], taken + 1
                    continue
            if T == 0:
                v = best
            else:
                r = lp.exp()
                if has_y:
                    r = (r - q).clamp(min=0)
                elif not last and 0 <= d < V:
                    r = r.clone()
                    r[d] = 0
                if float(r.sum()) == 0:
                    r = lp.exp()
                s = r.cumsum(0)
                v = min(int((s <= float(u[i, 1]) * s[-1]).sum()), int(r.nonzero()[-1]))
            tokens[i], logp[i] = v, lp[v]
            break
        accepted.append(taken)
        t += n
    return tokens, torch.tensor(accepted, dtype=torch.int32), logp
