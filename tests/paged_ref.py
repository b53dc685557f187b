"""64-bit restatement of the paged operators' definitions for tests: the 4-bit quantisation, block tables and attention."""
import math

import torch

PAGE, GROUP, LARGEST = 64, 32, 57120.0


def quantise(x):
    """The values that 4 bits hold of x [..., 32 m]: (c - 8) s with s a seventh of the largest magnitude to 8 significant bits."""
    y = x.double()
    y = torch.where(y.isnan(), torch.zeros_like(y), y).clamp(-LARGEST, LARGEST).unflatten(-1, (-1, GROUP))
    a = y.abs().amax(-1, keepdim=True)
    t = a / torch.full_like(a, 7.0)
    e = (torch.frexp(t).exponent - 8).clamp(min=-24)
    u = ((e.long() + 1023) << 52).view(torch.float64)
    s = torch.round(t / u) * u
    c = torch.where(s > 0, torch.round(y / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(y)).clamp(-7, 7)
    return (c * s).flatten(-2)


def tables(cached, new, table, free, tokens, page):
    """Lists in, (table, slots, positions, starts, lengths, pages) out, one token at a time."""
    table = [list(r) for r in table]
    slots, positions, starts, lengths, taken = [], [], [0], [], 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        have = -(-c // page)
        for pos in range(c, c + n):
            pi = pos // page
            if pi >= have and pos % page == 0 and pi < len(table[r]):
                at = taken + pi - have
                table[r][pi] = free[at] if at < len(free) else -1
            held = table[r][pi] if pi < len(table[r]) else -1
            slots.append(held * page + pos % page if held >= 0 else -1)
            positions.append(pos)
        taken += -(-(c + n) // page) - have
        starts.append(starts[-1] + n)
        lengths.append(c + n)
    pad = tokens - len(slots)
    return table, slots + [-1] * pad, positions + [-1] * pad, starts, lengths, taken


def attend(q, k, v, lengths, starts, scale, window=None, indices=None, seen_keys=None):
    """q [N,H,dk]; k, v lists of [T, G, d] per request.  -> o, L, M and the sums that bound their errors: A = sum p |v|, B = largest sum of
    |q k| scale over the visible keys, V = sum |v| over them (all 64-bit; rows behind the last request: nan).  seen_keys(r): extra mask [T]
    of a request."""
    q = q.double()
    N, H, dk = q.shape
    G, dv = k[0].shape[1], v[0].shape[2]
    hp = H // G
    o = torch.full((N, H, dv), math.nan, dtype=torch.float64, device=q.device)
    A, V, L = o.clone(), o.clone(), o[..., 0].clone()
    M, B = L.clone(), L.clone()
    for r in range(len(lengths)):
        T = k[r].shape[0]
        j = torch.arange(T, device=q.device)
        for i in range(starts[r], starts[r + 1]):
            pos = lengths[r] - starts[r + 1] + i
            for g in range(G):
                see = j <= pos
                if window is not None:
                    see &= j > pos - window
                if indices is not None:
                    see &= (j[:, None] // PAGE == indices[i, g][None, :]).any(1)
                if seen_keys is not None:
                    see &= seen_keys(r)
                hs = slice(g * hp, (g + 1) * hp)
                kk, vv = k[r][see, g].double(), v[r][see, g].double()
                if kk.shape[0] == 0:
                    o[i, hs], A[i, hs], V[i, hs], L[i, hs], M[i, hs], B[i, hs] = 0, 0, 0, -math.inf, -math.inf, 0
                    continue
                x = q[i, hs] @ kk.T * scale
                m = x.max(1).values
                p = torch.exp(x - m[:, None])
                s = p.sum(1)
                o[i, hs], A[i, hs] = p @ vv / s[:, None], p @ vv.abs() / s[:, None]
                L[i, hs], M[i, hs], V[i, hs] = torch.log(s), m, vv.abs().sum(0)
                B[i, hs] = (q[i, hs].abs() @ kk.T.abs()).max(1).values * scale
    return o, L, M, A, B, V


def check(got, want, dtype, keys, dk):
    """Outputs within what the arithmetic allows.  A logit is a sum of dk products in 32 bits: off by at most dk 2^-24 B.  Relative to the
    row, probabilities are off by twice that and the sum over the keys by keys 2^-24; for bf16 queries probabilities are rounded to
    fp16 (by 2^-11 of themselves, below 2^-14 by 2^-25: half a step of the subnormal numbers; the row's largest is at least 1, so the sum
    that divides them is too) and the output to bf16 (2^-8)."""
    (o, L, M), (ro, rL, rM, A, B, V) = got, want
    rows = ~rL.isnan()
    logit = dk * 2.0 ** -24 * B + 2.0 ** -23 * rM.abs().nan_to_num(0, 0, 0)
    sums = keys * 2.0 ** -24
    rel = 2 * logit + sums + (2.0 ** -11 + 2.0 ** -20 if dtype == torch.bfloat16 else 0) + 2.0 ** -22
    tol = rel[..., None] * A + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23) * ro.abs() + (2.0 ** -25 * V if dtype == torch.bfloat16 else 0) + 1e-30
    err = (o.double() - ro).abs()
    assert bool((err <= tol)[rows].all()), f"output off by up to {((err / tol)[rows]).max().item():.3g} of its bound"
    fin = rows & (rM > -math.inf)
    assert torch.equal((M == -math.inf)[rows], (rM == -math.inf)[rows]) and torch.equal((L == -math.inf)[rows], (rL == -math.inf)[rows])
    for name, x, y, t in (("M", M, rM, logit), ("L", L, rL, logit * 2 + sums + 2.0 ** -22 * (1 + rL.abs().nan_to_num(0, 0, 0)))):
        e = (x.double() - y).abs()
        assert bool((e <= t)[fin].all()), f"{name} off by up to {(e / t)[fin].max().item():.3g} of its bound"
