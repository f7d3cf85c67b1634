"""Token log probabilities and top-logit distillation from their definitions, in
64 bits, one row at a time; with each value the most that fp32 arithmetic may be
off.  U = 2^-24 is one rounding: an exponential of d costs 4 |d| + 4 of them
(difference, scale, the factor log2 e, the exponential itself), a sum over V
values a chain of at most V / 256 + 24.  FLUSH: the hardware's exponential gives
0 where the result would be subnormal, so a probability may be off by the
smallest normal number (which counts where a teacher's mass of 1e-39 meets a
log probability of -1e38)."""
import math

import torch

U = 2.0 ** -24
FLUSH = 2.0 ** -126
INF = math.inf


def half(t):
    """(relative, absolute) error of one rounding to type t."""
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def _row(x, T):
    """lp, its error, entropy, its error; None for a row of only -inf."""
    u = x.double()
    if torch.isnan(u).any() or (u == INF).any():
        nan = torch.full_like(u, math.nan)
        return nan, nan, math.nan, math.nan
    M = u.max()
    if M == -INF:
        return None
    n = len(u) / 256 + 24
    d = (u - M) / T
    L = float(torch.logsumexp(d, 0))
    p = (d - L).exp()
    f = torch.where(p > 0, d, 0.0)                       # finite where it counts
    e_L = U * (float((p * (4 * f.abs() + 4)).sum()) + n + 2 * abs(L))
    lp = d - L
    e_lp = U * (3 * d.abs() + 2 * lp.abs()) + e_L
    H = L - float((p * f).sum())
    e_H = 2 * e_L + U * (float((p * f.abs() * (4 * f.abs() + 2 * n + 8)).sum()) + 2 * abs(H))
    return lp, e_lp, H, e_H


def order(x):
    """Indices by falling value, ties to the lower index, any NaN first (a device
    sort may put a NaN with its sign bit set last)."""
    x = torch.where(torch.isnan(x), math.nan, x.double())
    return torch.sort(x, dim=-1, descending=True, stable=True)[1]


def token_logprobs(x, targets, k=0, T=1.0, ignore=-100, g=None, gh=None):
    """Dict of (value, error) lists over the rows of x (N, V)."""
    N, V = x.shape
    out = {'logprobs': [], 'entropy': [], 'top_logprobs': [], 'top_ids': [], 'dlogits': []}
    zero = torch.zeros(V, dtype=torch.float64, device=x.device)

    def put(name, v, e=0.0):
        out[name].append((v, e))
    for i in range(N):
        t = None if targets is None else int(targets[i])
        if t is not None and t == ignore:
            put('logprobs', 0.0)
            put('entropy', 0.0)
            put('top_ids', torch.full((k,), -1))
            put('top_logprobs', torch.full((k,), -INF))
            put('dlogits', zero, zero)
            continue
        ids = order(x[i])[:k]
        put('top_ids', ids.cpu())
        r = _row(x[i], T)
        if r is None:
            put('logprobs', math.nan if t is not None and not 0 <= t < V else -INF)
            put('entropy', 0.0)
            put('top_logprobs', torch.full((k,), -INF))
            put('dlogits', zero, zero)
            continue
        lp, e_lp, H, e_H = r
        put('top_logprobs', lp[ids], e_lp[ids])
        put('entropy', H, e_H)
        bad = t is not None and not 0 <= t < V
        if t is not None:
            put('logprobs', math.nan if bad else float(lp[t]), 0.0 if bad else float(e_lp[t]))
        if g is None and gh is None:
            continue
        p = lp.exp()
        live = p > 0
        f, e_f = torch.where(live, lp, 0.0), torch.where(live, e_lp, 0.0)
        e_p = p * (e_f + 4 * U * (1 + f.abs())) + FLUSH
        d, e = torch.zeros_like(p), torch.zeros_like(p)
        if g is not None:
            gi = math.nan if bad else float(g[i])
            d, e = d - gi * p, e + abs(gi) * e_p
            if not bad:
                d[t] += gi
        if gh is not None:
            b = float(gh[i])
            d = d - b * p * torch.where(live, f + H, 0.0)
            e = e + abs(b) * (e_p * (f + H).abs() + p * (e_f + e_H + 2 * U * (f.abs() + abs(H))))
        mass = (abs(float(g[i])) * p if g is not None else 0) + \
            (abs(float(gh[i])) * p * (f.abs() + abs(H)) if gh is not None else 0)
        put('dlogits', d / T, (e + 6 * U * (mass + d.abs())) / T)
    return out


def distill(x, ids, teacher, T=1.0, g=None):
    N, V = x.shape
    out = {'loss': [], 'dlogits': []}
    zero = torch.zeros(V, dtype=torch.float64, device=x.device)
    for i in range(N):
        row, t = ids[i].tolist(), teacher[i].double().tolist()
        slots = [(a, b) for a, b in zip(row, t) if a != -1]
        if all(b == -INF and 0 <= a < V for a, b in slots):
            out['loss'].append((0.0, 0.0))
            out['dlogits'].append((zero, zero))
            continue
        bad = any(not 0 <= a < V or math.isnan(b) or b == INF for a, b in slots)
        r = _row(x[i], T)
        top = max(b for _, b in slots)
        mass = [math.exp((b - top) / T) if not bad else math.nan for _, b in slots]
        Z = math.fsum(mass)
        K = len(slots)
        # log q: difference, scale, and the sum's log
        e_lq = [U * (4 * abs(b - top) / T + 4 + K + 2 * abs(math.log(Z))) if not bad and m
                else 0.0 for (_, b), m in zip(slots, mass)]
        loss = err = 0.0
        q_at, e_at = {}, {}
        for (a, b), m, el in zip(slots, mass, e_lq):
            q = m / Z
            if q == 0:
                continue
            if bad or r is not None and math.isnan(r[2]):
                loss = math.nan
                continue
            lq = (b - top) / T - math.log(Z)
            lp, e_lp = (-INF, 0.0) if r is None else (float(r[0][a]), float(r[1][a]))
            e_q = q * (el + 4 * U * (1 + abs(lq))) + FLUSH
            loss += q * (lq - lp)
            if math.isfinite(lp):
                err += e_q * abs(lq - lp) + q * (el + e_lp + (K + 4) * U * (abs(lq) + abs(lp)))
            q_at[a], e_at[a] = q_at.get(a, 0.0) + q, e_at.get(a, 0.0) + e_q + K * U * q
        out['loss'].append((loss, err))
        if g is None:
            continue
        if r is None:
            out['dlogits'].append((zero, zero))
            continue
        lp, e_lp, _, _ = r
        p = lp.exp()
        f, e_f = torch.where(p > 0, lp, 0.0), torch.where(p > 0, e_lp, 0.0)
        d, e = p.clone() if not bad else p * math.nan, p * (e_f + 4 * U * (1 + f.abs())) + FLUSH
        for a in q_at:
            d[a] -= q_at[a]
            e[a] += e_at[a]
        s = abs(float(g[i])) / T
        out['dlogits'].append((d * (float(g[i]) / T), s * (e + 6 * U * p) + 4 * U * s * d.abs()))
    return out


def check(name, got, want):
    """`got` (N, ...) against a list of (value, error) a row."""
    rel, tiny = half(got.dtype)
    for i, (ref, err) in enumerate(want):
        v = got[i].detach().double()
        ref = torch.as_tensor(ref, dtype=torch.float64, device=v.device)
        err = torch.as_tensor(err, dtype=torch.float64, device=v.device)
        same = (v == ref) | (torch.isnan(v) & torch.isnan(ref))
        off, allow = (v - ref).abs(), err + (ref.abs() + err) * rel + tiny
        # a value that may be off past the type's largest number may round to infinity:
        # q_1 m + q_2 m with m the largest and q_1 + q_2 = 1 + U is one such sum
        over = torch.isinf(v) & (v * ref > 0) & (ref.abs() + allow > torch.finfo(got.dtype).max)
        ok = same | (off <= allow) | over
        assert ok.all(), (name, i, int((~ok).sum()), v[~ok][:4].tolist(), ref[~ok][:4].tolist(),
                          float((off / allow)[~ok].max()))


def check_ids(got, want):
    for i, (ref, _) in enumerate(want):
        assert torch.equal(got[i].cpu(), ref), (i, got[i].tolist()[:8], ref.tolist()[:8])


def edge_rows(V, dtype, device='cpu'):
    """Rows that masks and degenerate heads make, and a name for each."""
    g = torch.Generator().manual_seed(V)
    low = torch.finfo(dtype).min
    base = torch.randn(V, generator=g) * 3
    spike = torch.full((V,), low)
    spike[V // 2] = 1.0
    half_masked = base.clone()
    half_masked[::2] = -INF
    one = torch.full((V,), -INF)
    one[V - 1] = 2.0
    few = torch.full((V,), low)
    few[:min(V, 3)] = torch.tensor([0.5, -0.5, 0.25])[:min(V, 3)]
    zeros = torch.zeros(V)
    zeros[1::3] = -0.0
    nan = base.clone()
    nan[V // 3] = math.nan
    pinf = base.clone()
    pinf[V // 3] = INF
    up = torch.arange(V, dtype=torch.float32) / V
    rows = {'ordinary': base, 'all_masked': torch.full((V,), -INF),
            'all_lowest': torch.full((V,), low), 'spike_over_lowest': spike,
            'few_over_lowest': few, 'half_masked': half_masked, 'one_left': one,
            'zeros_of_both_signs': zeros, 'equal': torch.full((V,), 1.5),
            'rising': up, 'falling': -up, 'steps': (base * 2).round(), 'nan': nan,
            'plus_inf': pinf, 'large': base * 300, 'offset': base + 1000}
    return list(rows), torch.stack(list(rows.values())).to(dtype).to(device)
