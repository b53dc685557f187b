"""The operators of paged serving as measurable cases: block tables, the 4-bit cache, attention over it.

A case is a dict of plain values; ``prepare`` builds what a program holds before the call, ``run`` makes one pass.  The kinds:

* ``tables``  block table, slot map and positions of a step from the requests' lengths;
* ``append``  a step's keys and values quantised into their slots, and those tokens read back as the values they stand for;
* ``attend``  attention of a step's queries over the pages: all earlier keys, a sliding window, or selected blocks of 64.

The cache is one byte tensor ``[pages, groups, page bytes]``.  A page holds 64 tokens as four records of 16; a record holds, for
each 32 of the dk + dv dimensions, 256 bytes of codes, then for each of them 16 scales in fp16 (``_unpack``).  The plain form and
the framework read the same bytes.
"""
import math
import os
import sys

import torch

own = False

# head configurations: the paper's (and the benchmark's), one of 128-wide heads, the small test configuration
HEADS = {"paper": dict(H=64, G=4, dk=192, dv=128), "square": dict(H=32, G=2, dk=128, dv=128), "small": dict(H=8, G=2, dk=64, dv=64)}
PAGE, GROUP, REC = 64, 32, 16
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one step of a server in steady state: every request brings one token, some of them open a page
        dict(name="tables_decode_256", kind="tables", S=256, cached=8192, prompts=0, new=1, width=512),
        # a step that admits prompts among requests that generate
        dict(name="tables_mixed_1000", kind="tables", S=1000, cached=4096, prompts=60, new=900, width=1024),
        # the tokens of a decoded batch
        dict(name="append_decode_64", kind="append", heads="paper", dtype="bf16", N=64),
        # a chunk of prompts
        dict(name="append_chunk_8k", kind="append", heads="paper", dtype="bf16", N=8192),
        # fp32 tokens of a small model, an odd number of them
        dict(name="append_fp32_1001", kind="append", heads="small", dtype="fp32", N=1001),
        # a chat turn being generated: one sequence, one token
        dict(name="attend_decode_b1_2k", kind="attend", heads="paper", dtype="bf16", S=1, cached=2100, new=1),
        # batched generation over contexts of very different lengths
        dict(name="attend_decode_b64_32k", kind="attend", heads="paper", dtype="bf16", S=64, cached=32000, new=1),
        # fp32 decoding with the small heads
        dict(name="attend_fp32_b8_4k", kind="attend", heads="small", dtype="fp32", S=8, cached=4100, new=1),
        # drafted tokens checked together, sliding window
        dict(name="attend_draft_window", kind="attend", heads="square", dtype="bf16", S=32, cached=9000, new=4, window=512),
        # the selected blocks of generated tokens in long contexts
        dict(name="attend_selected_b32_64k", kind="attend", heads="paper", dtype="bf16", S=32, cached=65000, new=1, n=16),
        # prompts from an empty cache, each of its own length
        dict(name="attend_prompts_ragged", kind="attend", heads="square", dtype="bf16", S=7, cached=0, new=1500),
        # a chunk of a long prompt
        dict(name="attend_chunk_2k_30k", kind="attend", heads="paper", dtype="bf16", S=1, cached=30000, new=2000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "append", "attend", "attend", "attend", "attend", "attend"])
    if kind == "tables":
        S = _log(rng, 1, 4000)
        return dict(kind=kind, S=S, cached=_log(rng, 1, 30000), prompts=rng.randint(0, min(S, 30)), new=_log(rng, 1, 1500), width=rng.randint(512, 1500))
    if kind == "append":
        return dict(kind=kind, heads=rng.choice(["paper", "paper", "square", "small"]), dtype=rng.choice(["bf16", "bf16", "fp32"]), N=_log(rng, 1, 12000))
    heads = rng.choice(["paper", "paper", "square", "small"])
    form = rng.choice(["decode", "decode", "draft", "window", "selected", "chunk", "chunk"])
    c = dict(kind=kind, heads=heads, dtype="bf16")
    if form == "chunk":
        S = rng.choice([1, 1, 2, 5])
        new = _log(rng, 20, 2000)
        c.update(S=S, cached=rng.choice([0, _log(rng, 1, 30000)]) // S, new=max(2, new // S))
        if rng.random() < 0.3:
            c.update(window=rng.choice([128, 500, 512, 2000]))
        return c
    S = _log(rng, 1, 128)
    c.update(S=S, cached=_log(rng, 1, 1000000 // S if S > 16 else 60000), new=1 if form == "decode" else rng.randint(1, 8))
    if form == "decode" and rng.random() < 0.2:
        c.update(dtype="fp32", cached=min(c["cached"], 100000 // S))
    if form == "window":
        c.update(window=rng.choice([128, 500, 512, 2000]))
    if form == "selected":
        c.update(n=rng.choice([8, 16, 17]))
    return c


# ------------------------------------------------------------------------------------------------ inputs

def _lengths(case, gen):
    """Cached and new tokens of each request (int32, host): one request as the case says, several spread below that, in any order."""
    S, cached, new = case["S"], case["cached"], case["new"]

    def spread(top, least, count=S):
        x = _spread(top, least, count)
        return torch.tensor(x, dtype=torch.int32)[torch.randperm(count, generator=gen)]

    if case["kind"] == "tables":
        n = torch.ones(S, dtype=torch.int32)
        c = spread(cached, 0)
        at = torch.randperm(S, generator=gen)[:case["prompts"]]
        n[at], c[at] = spread(new, 1, len(at)), 0
        return c, n
    if new <= 8:
        return spread(cached, min(cached, 1)), torch.full((S,), new, dtype=torch.int32)
    return spread(cached, 0), spread(new, 1)


def _spread(top, least, count):
    """``count`` lengths from ``top`` down towards ``least``, more long ones than short ones."""
    return [max(least, round(top - (top - least) * (i / count) ** 1.4)) for i in range(count)]


def _pages(n):
    return -(-n // PAGE)


def _storage(pages, G, dk, dv, gen):
    """Pages full of quantised normal values: codes as rounding N(0, 2.7) gives them, scales around 1/2.7."""
    rec = (dk + dv) // GROUP
    st = torch.empty(pages, G, PAGE // REC, rec * 288, device="cuda", dtype=torch.uint8)
    nib = torch.randn(2, 4096, generator=gen, device="cuda").mul_(2.7).round_().clamp_(-7, 7).add_(8).to(torch.uint8)
    table = nib[0] | (nib[1] << 4)
    step = max(1, (1 << 26) // st[0].numel())
    for p in range(0, pages, step):
        part = st[p:p + step]
        at = torch.randint(0, 4096, (*part.shape[:3], rec * 256), generator=gen, device="cuda", dtype=torch.int32)
        part[..., :rec * 256] = table[at]
        s = torch.randn(*part.shape[:3], rec * 16, generator=gen, device="cuda").mul_(0.25).exp_().div_(2.7).bfloat16().half()
        part[..., rec * 256:] = s.view(torch.uint8)
    return st.view(pages, G, -1)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    cg = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "tables":
        c, n = _lengths(case, gen)
        have, need = _pages(c), _pages(c + n) - _pages(c)
        total, P = int((have + need).sum()), case["width"]
        ids = torch.randperm(total + 100, generator=gen, dtype=torch.int32)
        table = torch.full((case["S"], P), -1, dtype=torch.int32)
        used = torch.arange(P)[None] < have[:, None]
        table[used] = ids[:int(have.sum())]
        return dict(kind="tables", cached=c.cuda(), new=n.cuda(), table=table.cuda(), free=ids[int(have.sum()):].cuda(), tokens=int(n.sum()))
    h = HEADS[case["heads"]]
    H, G, dk, dv = h["H"], h["G"], h["dk"], h["dv"]
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "append":
        N = case["N"]
        pages = _pages(N) + 8
        k = torch.randn(N, G, dk, generator=cg, device="cuda")
        k *= torch.randn(dk, generator=cg, device="cuda").mul_(0.5).exp_()          # channels of different size, as keys have them
        v = torch.randn(N, G, dv, generator=cg, device="cuda")
        if N > 512:                                                                 # prompts: runs of slots, pages in any order
            slots = torch.randperm(pages, generator=gen)[:, None] * PAGE + torch.arange(PAGE)
            slots = slots.reshape(-1)[:N]
        else:                                                                       # one token of each request
            slots = torch.randperm(pages * PAGE, generator=gen)[:N]
        return dict(kind="append", k=k.to(dt), v=v.to(dt), slots=slots.cuda(), G=G, dk=dk, dv=dv,
                    storage=torch.zeros(pages, G, 4 * (dk + dv) // GROUP * 288, device="cuda", dtype=torch.uint8))
    c, n = _lengths(case, gen)
    ln, S = c + n, case["S"]
    per = _pages(ln)
    total, P = int(per.sum()), int(per.max()) + 3
    ids = torch.randperm(total + 5, generator=gen, dtype=torch.int32)
    table = torch.full((S, P), -1, dtype=torch.int32)
    table[torch.arange(P)[None] < per[:, None]] = ids[:total]
    starts = torch.zeros(S + 1, dtype=torch.int32)
    starts[1:] = n.cumsum(0)
    N = int(n.sum())
    st = dict(kind="attend", q=torch.randn(N, H, dk, generator=cg, device="cuda").to(dt), storage=_storage(total + 5, G, dk, dv, cg),
              table=table.cuda(), lengths=ln.cuda(), starts=starts.cuda(), max_new=int(n.max()), G=G, dk=dk, dv=dv, window=case.get("window"),
              indices=None)
    if "n" in case:
        row = torch.repeat_interleave(torch.arange(S), n.long())
        last = (ln[row] - n[row] + (torch.arange(N) - starts[row])).long() // PAGE  # block of each token's own position
        pick = torch.rand(N, G, case["n"], generator=gen).mul_(last[:, None, None] + 1).long()
        pick[..., 0], pick[..., 1], pick[..., 2] = 0, last[:, None], (last[:, None] - 1).clamp(min=0)
        pick = pick.sort(-1).values
        pick[..., 1:][pick[..., 1:] == pick[..., :-1]] = -1                         # a short context has fewer blocks than places
        st["indices"] = pick.to(torch.int32).cuda()
    return st


# ------------------------------------------------------------------------------------------------ the plain forms

def _unpack(st, dk, dv):
    """[..., page bytes] -> the values held, keys [..., 64, dk] and values [..., 64, dv] in fp32."""
    lead, gk, gv = st.shape[:-1], dk // GROUP, dv // GROUP
    rec = st.reshape(*lead, 4, (gk + gv) * 288)
    codes = rec[..., :(gk + gv) * 256].reshape(*lead, 4, gk + gv, 8, 4, 8)          # 8 x 4 lanes of 8 bytes
    scales = rec[..., (gk + gv) * 256:].contiguous().view(torch.float16).float()
    scales = scales.view(*lead, 4, gk + gv, 4, 2, 2).movedim(-4, -1)                # [pair, tile, odd], group
    scales = scales.transpose(-4, -3).reshape(*lead, PAGE, gk + gv)                 # token 16 r + 8 tile + 2 pair + odd
    x = torch.stack((codes & 15, codes >> 4), dim=-1).float() - 8                   # [r, group, 8, 4, 8 bytes, 2]
    n = len(lead)
    d = list(range(n))
    # keys: lane = 4 (token % 8) + j, word = tile, nibble = dimension 8 j + e
    k = x.narrow(n + 1, 0, gk).reshape(*lead, 4, gk, 8, 4, 2, 8).permute(*d, n, n + 4, n + 2, n + 1, n + 3, n + 5).reshape(*lead, PAGE, dk)
    # values: lane = 4 (dimension % 8) + pair, half word = 2 tile + odd, nibble = dimension / 8
    v = x.narrow(n + 1, gk, gv).reshape(*lead, 4, gv, 8, 4, 2, 2, 4).permute(*d, n, n + 4, n + 3, n + 5, n + 1, n + 6, n + 2).reshape(*lead, PAGE, dv)
    return k * scales[..., :gk].repeat_interleave(GROUP, -1), v * scales[..., gk:].repeat_interleave(GROUP, -1)


def _power2(e):
    """2^e of whole numbers, exact."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantise(x):
    """The values that 4 bits hold of x [..., 32 m], in 64 bits (a quotient next to a border has to fall on its side)."""
    x = x.double().nan_to_num(0.0, 57120.0, -57120.0).clamp(-57120, 57120).unflatten(-1, (-1, GROUP))
    t = x.abs().amax(-1, keepdim=True)
    t = t / torch.full_like(t, 7)                                                   # (by a plain 7 it would be times its reciprocal)
    u = _power2((torch.frexp(t).exponent - 8).clamp(min=-24))
    s = torch.round(t / u) * u
    code = torch.where(s > 0, torch.round(x / s.clamp(min=2.0 ** -24)), torch.zeros_like(x)).clamp(-7, 7)
    return (code + 8).to(torch.uint8).flatten(-2), s.squeeze(-1).half()


def _write(st, slots, k, v, dk, dv):
    """Quantised tokens into their bytes."""
    gk, gv = dk // GROUP, dv // GROUP
    kc, ks = _quantise(k)
    vc, vs = _quantise(v)
    N, G = kc.shape[:2]
    rec = st.view(st.shape[0], G, 4, (gk + gv) * 288)
    page, r = slots // PAGE, slots % PAGE // REC
    tile, n, pair, odd = slots % 16 // 8, slots % 8, slots % 8 // 2, slots % 2
    dev = st.device
    g = torch.arange(G, device=dev).view(1, G, 1)
    two = lambda t: t.view(N, 1, 1)
    kb = kc[..., 0::2] | (kc[..., 1::2] << 4)                                       # [N,G,dk/2]: 16 bytes a group, 4 a word
    b = torch.arange(dk // 2, device=dev).view(1, 1, -1)
    rec[two(page), g, two(r), b // 16 * 256 + (two(n) * 4 + b % 16 // 4) * 8 + two(tile) * 4 + b % 4] = kb
    vb = vc.view(N, G, gv, 4, 8)                                                    # dimension 32 g + 8 e + n
    vb = torch.stack((vb[..., 0, :] | (vb[..., 1, :] << 4), vb[..., 2, :] | (vb[..., 3, :] << 4)), -1).reshape(N, G, gv * 16)
    b = torch.arange(gv * 16, device=dev).view(1, 1, -1)
    rec[two(page), g, two(r), (gk + b // 16) * 256 + (b % 16 // 2 * 4 + two(pair)) * 8 + two(2 * tile + odd) * 2 + b % 2] = vb
    sc = torch.cat((ks, vs), -1).contiguous().view(torch.uint8)
    b = torch.arange(2 * (gk + gv), device=dev).view(1, 1, -1)
    rec[two(page), g, two(r), (gk + gv) * 256 + b // 2 * 32 + two(4 * pair + 2 * tile + odd) * 2 + b % 2] = sc


def _tables(s):
    c, n, table, free = s["cached"].long(), s["new"].long(), s["table"], s["free"]
    dev, N = table.device, s["tokens"]
    have, all_ = (c + PAGE - 1) // PAGE, (c + n + PAGE - 1) // PAGE
    need = all_ - have
    first = need.cumsum(0) - need
    col = torch.arange(table.shape[1], device=dev)[None]
    fresh = (col >= have[:, None]) & (col < all_[:, None])
    table = torch.where(fresh, free[(first[:, None] + col - have[:, None]).clamp(0, len(free) - 1)], table)
    starts = torch.cat((n.new_zeros(1), n.cumsum(0)))
    i = torch.arange(N, device=dev)
    row = torch.searchsorted(starts[1:], i, right=True)
    pos = c[row] + i - starts[row]
    slots = table[row, pos // PAGE].long() * PAGE + pos % PAGE
    return table, slots, pos.int(), starts.int(), (c + n).int(), need.sum().int().view(1)


def _softmax_rows(x, v):
    """Logits x [..., keys] (-inf where masked) and values -> output, log of the sum, maximum."""
    M = x.amax(-1)
    p = x.sub_(M.clamp(min=-3e38)[..., None]).exp_()
    l = p.sum(-1)
    return torch.matmul(p, v) / torch.where(l > 0, l, torch.ones_like(l))[..., None], l.log(), M


def _attend(s):
    q, table, G, dk, dv = s["q"].float(), s["table"].long(), s["G"], s["dk"], s["dv"]
    N, H = q.shape[:2]
    S, dev, hp, scale = table.shape[0], q.device, H // G, dk ** -0.5
    starts, lengths = s["starts"].long(), s["lengths"].long()
    i = torch.arange(N, device=dev)
    row = torch.searchsorted(starts[1:], i, right=True)
    at = i - starts[row]
    pos = lengths[row] - (starts[row + 1] - starts[row]) + at
    if s["indices"] is not None:
        idx = s["indices"].long()
        page = table[row[:, None, None], idx.clamp(min=0)].clamp(min=0)
        k, v = _unpack(s["storage"][page, torch.arange(G, device=dev)[None, :, None]], dk, dv)
        k, v = k.view(N, G, -1, dk), v.view(N, G, -1, dv)
        j = (idx[..., None] * PAGE + torch.arange(PAGE, device=dev)).view(N, G, -1)
        seen = (idx >= 0).repeat_interleave(PAGE, -1) & (j <= pos[:, None, None])
        x = torch.matmul(q.view(N, G, hp, dk) * scale, k.transpose(-1, -2)).masked_fill_(~seen[:, :, None], float("-inf"))
        o, l, M = _softmax_rows(x, v)
        return o.reshape(N, H, dv).to(s["q"].dtype), l.reshape(N, H), M.reshape(N, H)
    k, v = _unpack(s["storage"][table.clamp(min=0)], dk, dv)                         # [S,P,G,64,d]
    k, v = (t.transpose(1, 2).reshape(S, G, -1, t.shape[-1]) for t in (k, v))
    T, most = k.shape[2], s["max_new"]
    qs = q.new_zeros(S, most, H, dk)
    qs[row, at] = q * scale
    qs = qs.view(S, most, G, hp, dk).permute(0, 2, 1, 3, 4).reshape(S, G, most * hp, dk)
    ps = torch.full((S, most), -1, device=dev)
    ps[row, at] = pos
    j = torch.arange(T, device=dev)
    seen = j <= ps[..., None]
    if s["window"] is not None:
        seen &= j > ps[..., None] - s["window"]
    x = torch.matmul(qs, k.transpose(-1, -2)).view(S, G, most, hp, T).masked_fill_(~seen[:, None, :, None], float("-inf"))
    o, l, M = _softmax_rows(x.view(S, G, most * hp, T), v)
    back = lambda t: t.view(S, G, most, hp, -1).permute(0, 2, 1, 3, 4).reshape(S, most, H, -1)[row, at]
    return back(o).to(s["q"].dtype), back(l)[..., 0], back(M)[..., 0]


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "tables":
        return _tables(s)
    if s["kind"] == "append":
        _write(s["storage"], s["slots"], s["k"], s["v"], s["dk"], s["dv"])
        k, v = _unpack(s["storage"], s["dk"], s["dv"])                              # [pages,G,64,d]
        page, t = s["slots"] // PAGE, s["slots"] % PAGE
        return k[page, :, t], v[page, :, t]
    return _attend(s)


def _run_own(s):
    pkg = os.path.join(os.getcwd(), "nsa-test_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from nsa.paged import PagedCache4, block_tables
    if s["kind"] == "tables":
        step = block_tables(s["cached"], s["new"], s["table"], s["free"], s["tokens"])
        return s["table"], step.slots, step.positions, step.starts, step.lengths, step.pages
    cache = PagedCache4(s["storage"], s["dk"], s["dv"])
    if s["kind"] == "append":
        cache.append(s["k"], s["v"], s["slots"])
        return cache.read(s["slots"])
    return cache.attend(s["q"], s["table"], s["lengths"], s["starts"], window=s["window"], indices=s["indices"], max_new=s["max_new"])


# ------------------------------------------------------------------------------------------------ work and exact values

def _seen_keys(case):
    """(keys read for the requests, keys seen by the tokens, tokens) of a case."""
    S, w = case["S"], case.get("window")
    cached = _spread(case["cached"], min(case["cached"], 1) if case["new"] <= 8 else 0, S)
    new = [case["new"]] * S if case["new"] <= 8 else _spread(case["new"], 1, S)
    read = seen = 0
    # the orders of the two are drawn apart: each takes the other's mean
    for c, n in zip(cached, [sum(new) / S] * S):
        most = min(case["n"] * PAGE * n if "n" in case else c + n, n + w - 1 if w is not None else c + n)
        per = min(c + n / 2, case["n"] * PAGE if "n" in case else w if w is not None else c + n)
        read, seen = read + most, seen + n * per
    return read, seen, sum(new)


def work(case):
    if case["kind"] == "tables":
        S, n = case["S"], case["prompts"]
        tokens = S - n + sum(_spread(case["new"], 1, n))
        return {"bytes": 16 * S + 12 * tokens + 8 * (tokens / PAGE + S / PAGE), "flops": 4 * tokens}
    h = HEADS[case["heads"]]
    d, e = h["dk"] + h["dv"], 2 if case["dtype"] == "bf16" else 4
    held = h["G"] * d // GROUP * 18
    if case["kind"] == "append":
        return {"bytes": case["N"] * (h["G"] * d * (e + 4) + 2 * held + 16), "flops": case["N"] * h["G"] * d * 6}
    read, seen, tokens = _seen_keys(case)
    return {"bytes": read * held + tokens * h["H"] * (d * e + 8), "flops": 2 * h["H"] * d * seen}


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    if case["kind"] == "append":
        return tuple(_held64(s[name]) for name in ("k", "v"))
    dk, dv, G, q = s["dk"], s["dv"], s["G"], s["q"].double()
    N, H = q.shape[:2]
    hp = H // G
    starts, lengths, table = s["starts"].tolist(), s["lengths"].tolist(), s["table"].long()
    o = q.new_zeros(N, H, dv)
    L, M = q.new_full((N, H), -math.inf), q.new_full((N, H), -math.inf)

    def rows(at, g, k, v, seen):
        """Tokens `at` of group g over keys k, v [T, d] where seen [tokens, T]."""
        x = torch.einsum("nhd,td->nht", q[at, g * hp:(g + 1) * hp], k) / math.sqrt(dk)
        x = torch.where(seen[:, None], x, torch.full_like(x, -math.inf))
        m = x.max(-1).values
        p = torch.exp(x - torch.where(m > -math.inf, m, torch.zeros_like(m))[..., None])
        l = p.sum(-1)
        o[at, g * hp:(g + 1) * hp] = torch.einsum("nht,td->nhd", p, v) / l.clamp(min=1e-300)[..., None]
        L[at, g * hp:(g + 1) * hp], M[at, g * hp:(g + 1) * hp] = torch.log(l), m

    for r in range(table.shape[0]):
        a, b = starts[r], starts[r + 1]
        for g in range(G):
            held = _unpack64(s["storage"][table[r, :-(-lengths[r] // PAGE)], g], dk, dv)
            k, v = (t.reshape(-1, t.shape[-1]) for t in held)
            j = torch.arange(k.shape[0], device=q.device)
            for lo in range(a, b, 128):
                at = torch.arange(lo, min(b, lo + 128), device=q.device)
                pos = lengths[r] - b + at
                seen = j[None] <= pos[:, None]
                if s["window"] is not None:
                    seen = seen & (j[None] > pos[:, None] - s["window"])
                if s["indices"] is not None:
                    seen = seen & (j[None, :, None] // PAGE == s["indices"][at, g][:, None, :]).any(-1)
                rows(at, g, k, v, seen)
    return o, L, M


def _held64(x):
    """Each value as 4 bits hold it, from the definition: the group's largest seventh to 8 significant bits, the nearest multiple."""
    y = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    a = torch.max(torch.abs(y), dim=-1, keepdim=True).values
    t = a / torch.full_like(a, 7.0)
    bits = torch.where(t >= 2.0 ** -16, t, torch.full_like(t, 2.0 ** -17)).view(torch.int64)
    step = (((bits >> 52) - 7) << 52).view(torch.float64)                           # the power of two of t, by its bits, 7 places down
    s = torch.round(t / step) * step
    return torch.where(s > 0, torch.round(y / s).clamp(-7, 7) * s, torch.zeros_like(y)).reshape(x.shape)


def _unpack64(pages, dk, dv):
    """The values of pages [P, page bytes] one token place and dimension at a time: byte addresses from the layout's definition."""
    dev, P = pages.device, pages.shape[0]
    groups = (dk + dv) // GROUP
    t = torch.arange(PAGE, device=dev)[:, None]
    rec, tile, pair, odd = t // 16 * (groups * 288), t % 16 // 8, t % 8 // 2, t % 2

    def part(first, width, address):
        d = torch.arange(width, device=dev)[None]
        byte, high = address(d % GROUP)
        code = pages[:, rec + (first + d // GROUP) * 256 + byte].double()
        code = torch.where(high.expand(PAGE, width) > 0, torch.floor(code / 16), torch.remainder(code, 16))
        at = rec + groups * 256 + (first + d // GROUP) * 32 + 2 * (4 * pair + 2 * tile + odd)
        bits = pages[:, at].int() + 256 * pages[:, at + 1].int()
        e, m = bits // 1024, bits % 1024                                            # fp16, no sign
        return (code - 8) * torch.where(e > 0, (1024 + m) * torch.exp2(e.double() - 25), m * 2.0 ** -24)

    k = part(0, dk, lambda d: ((t % 8 * 4 + d // 8) * 8 + tile * 4 + d % 8 // 2, d % 2))
    v = part(dk // GROUP, dv, lambda d: ((d % 8 * 4 + pair) * 8 + (2 * tile + odd) * 2 + d // 16, d // 8 % 2))
    return k, v
