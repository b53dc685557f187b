"""Paged serving where it can go wrong: many short requests, queries and lengths beyond the ordinary, steps taken apart."""
import math
import random

import pytest
import torch

from tests import paged_ref as ref
from tests.test_paged import BF, F32, HEADS, ODD_HEADS, Served


def by_request(s, q, lengths=None, scale=None, window=None, held=None):
    """``ref.attend`` for all tokens of a request and group at once (64 bits): o, L, M, A, B, V.  held[r]: the positions of keys s.k[r], where not all are there."""
    q, N, H = q.double(), q.shape[0], q.shape[1]
    G, dk, dv = s.k[0].shape[1], s.dk, s.v[0].shape[2]
    hp, scale = H // G, s.dk ** -0.5 if scale is None else scale
    o = torch.full((N, H, dv), math.nan, dtype=torch.float64, device=q.device)
    A, V, L = o.clone(), o.clone(), o[..., 0].clone()
    M, B = L.clone(), L.clone()
    for r, length in enumerate(s.lengths if lengths is None else lengths):
        a, b = s.starts[r], s.starts[r + 1]
        if a == b:
            continue
        j = torch.arange(length, device=q.device) if held is None else held[r]
        pos = length - b + torch.arange(a, b, device=q.device)
        see = j <= pos[:, None]
        if window is not None:
            see &= j > pos[:, None] - window
        for g in range(G):
            at = (slice(a, b), slice(g * hp, (g + 1) * hp))
            k, v = s.k[r][:len(j), g].double(), s.v[r][:len(j), g].double()
            mask = lambda x, y: torch.where(see[:, None], x, torch.full_like(x, y))
            x = mask(q[at] @ k.T * scale, -math.inf)
            M[at] = x.amax(-1)
            p = torch.exp(x - M[at][..., None])
            l = p.sum(-1, keepdim=True)
            o[at], A[at], L[at] = p @ v / l, p @ v.abs() / l, torch.log(l[..., 0])
            B[at] = mask(q[at].abs() @ k.abs().T * abs(scale), 0.0).amax(-1)
            V[at] = (see.double() @ v.abs())[:, None].expand(-1, hp, -1)
    return o, L, M, A, B, V


# ------------------------------------------------------------------------------------------------ many short requests

def _rows(hp, *rows):
    """New tokens that make so many rows (token, head) of a group, rounded up."""
    return [-(-r // hp) for r in rows]


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("pattern", [(160, 96), (256, 80, 128, 96, 80), (96, 80, 128, 256), (300, 90, 90, 90, 90, 90), None])
@pytest.mark.parametrize("window", [None, 30])
def test_many_pieces_a_block(heads, pattern, window):
    """Hundreds of short requests: a block has more of them than it holds at once, with one row tile or two in any order."""
    hp = heads[0] // heads[1]
    rng = random.Random(30)
    S = 1200 // heads[1]
    rows = [rng.choice([80, 96, 128, 129, 200, 256, 257, 400]) for _ in range(S)] if pattern is None else [pattern[i % len(pattern)] for i in range(S)]
    new = _rows(hp, *rows)
    s = Served([n + rng.choice([0, 1, rng.randint(0, 150)]) for n in new], new, *heads, BF, seed=30)
    got = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, window=window)
    ref.check(got, by_request(s, s.q, window=window), BF, max(s.lengths), s.dk)
    for _ in range(5):
        again = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, window=window)
        assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("every", [3, 5, 9, 1000])
def test_a_padded_step_of_mostly_single_tokens(heads, every):
    """Room for 256 rows a request, of which most bring one token: all are one kernel's, and most pieces have one row tile."""
    hp, S = heads[0] // heads[1], 1000 // heads[1]
    most = 256 // hp
    rng = random.Random(every)
    new = [most if i % every == 0 else rng.choice([1, 1, 1, 2]) for i in range(S)]
    s = Served([n + rng.randint(0, 200) for n in new], new, *heads, BF, seed=31)
    N = s.starts[-1]
    q = torch.cat((s.q, s.q.new_full((S * most - N, *s.q.shape[1:]), math.nan)))
    o, L, M = s.cache.attend(q, s.table, s.len_dev, s.starts_dev, max_new=most)
    ref.check((o[:N], L[:N], M[:N]), by_request(s, s.q), BF, max(s.lengths), s.dk)


# ------------------------------------------------------------------------------------------------ queries beyond the ordinary

# (lengths, new tokens): segments that one block has whole, segments that many blocks share, several row tiles, prompts
LAYOUTS = [([40, 7, 64], [1, 1, 1]), ([20000, 5], [1, 1]), ([90, 3000, 33], [3, 2, 4]), ([150, 40, 60], [150, 40, 60]), ([6000], [40])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heads", [(BF, HEADS[0]), (BF, HEADS[1]), (BF, HEADS[2]), (F32, HEADS[2]), (BF, ODD_HEADS[0])])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("form", ["all", "window", "selected"])
def test_rows_that_are_not_finite(dtype, heads, layout, form):
    """A NaN or an infinity in a query makes that row NaN however the work is cut, and no other row anything else."""
    s = Served(*layout, *heads, dtype, seed=32)
    N, H, dk = s.q.shape
    kw = dict(window=dict(window=33), all={}, selected=dict(indices=torch.randint(0, -(-min(s.lengths) // 64), (N, heads[1], 3), dtype=torch.int32).cuda()))[form]
    clean = s.q.clone()
    rng = random.Random(33)
    bad = torch.zeros(N, H, dtype=torch.bool, device="cuda")
    for _ in range(min(5, N * H // 2)):
        i, h = rng.randrange(N), rng.randrange(H)
        bad[i, h] = True
        clean[i, h] = 0
        what = rng.choice([math.nan, math.inf, -math.inf])
        if rng.random() < 0.3:
            s.q[i, h] = what
        else:
            s.q[i, h, rng.randrange(dk)] = what
    got = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, **kw)
    want = s.cache.attend(clean, s.table, s.len_dev, s.starts_dev, **kw)
    assert want[0].isfinite().all()
    blind = want[2] == -math.inf                    # (a row may see nothing of the named blocks: then its query does not count)
    for x, y in zip(got, want):
        assert x[bad & ~blind].isnan().all() and torch.equal(x[~bad | blind], y[~bad | blind])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_rows_that_are_not_finite_and_see_nothing(dtype, new):
    s = Served([200, 90], [new, 1], *HEADS[2], dtype, seed=34)
    s.q[0] = math.nan
    s.table[:] = -1
    o, L, M = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
    assert not o.any() and (L == -math.inf).all() and (M == -math.inf).all()


# ------------------------------------------------------------------------------------------------ more units than 32 bits count

@pytest.mark.gpu
def test_more_units_of_work_than_32_bits_count():
    """The longest table there may be, with six pages in it: 320 row tiles of 8 388 608 pages are 2.7e9 units of work, behind and in front of
    requests of a page."""
    from types import SimpleNamespace

    from nsa.paged import PagedCache4
    H, dk, P, new = 16, 32, 1 << 23, [1, 160, 2]
    lengths = [60, P * 64, 40]
    pages = {0: [0], 1: [0, 1, P // 2, P - 3, P - 2, P - 1], 2: [0]}
    table = torch.full((3, P), -1, dtype=torch.int32, device="cuda")
    c = PagedCache4.empty(8, 1, dk, dk)
    s = SimpleNamespace(lengths=lengths, starts=[0, 1, 161, 163], dk=dk, k=[], v=[])
    gen = torch.Generator(device="cuda").manual_seed(40)
    rn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    held, at = [], 0
    for r in range(3):
        ids = torch.arange(at, at + len(pages[r]), device="cuda")
        at += len(pages[r])
        table[r, torch.tensor(pages[r], device="cuda")] = ids.int()
        slots = (ids[:, None] * 64 + torch.arange(64, device="cuda")).view(-1)
        c.append(rn(len(slots), 1, dk), rn(len(slots), 1, dk), slots)
        k, v = c.read(slots)
        s.k.append(k)
        s.v.append(v)
        held.append((torch.tensor(pages[r], device="cuda")[:, None] * 64 + torch.arange(64, device="cuda")).view(-1))
    q = rn(163, H, dk)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    got = c.attend(q, table, i32(lengths), i32(s.starts))
    # 384 keys and at most 296 partial results a row
    ref.check(got, by_request(s, q, held=held), F32, 1000, dk)


# ------------------------------------------------------------------------------------------------ block tables of lengths beyond reason

LIMIT = 2 ** 30 - 1


def _bounded_tables(cached, new, table, free, tokens, page):
    """slots and positions as nsa_block_tables finds them, sums of lengths held below 2^30: every page it reads or writes is one of its own."""
    hold = lambda x: min(max(x, 0), 2 ** 29)
    c, n = [hold(x) for x in cached], [hold(x) for x in new]
    have = [-(-x // page) for x in c]
    need = [-(-(x + y) // page) - h for x, y, h in zip(c, n, have)]
    first, opened, taken, t = [], [], 0, 0
    for x, y in zip(n, need):
        t, taken = min(t + x, LIMIT), min(taken + y, LIMIT)
        first.append(t - x)
        opened.append(taken - y)
    table = [list(r) for r in table]
    rows = []
    for i in range(min(tokens, t)):
        r, up = 0, len(c)
        while up - r > 1:
            mid = (r + up) // 2
            r, up = (mid, up) if first[mid] <= i else (r, mid)
        pos = c[r] + i - first[r]
        at = pos // page
        assert pos >= 0 and first[r] >= 0 and opened[r] >= 0
        rows.append((r, pos, at, opened[r] + at - have[r] if at >= have[r] else None))
    before = [list(x) for x in table]
    for r, pos, at, f in rows:
        if at < len(table[r]) and f is not None and pos % page == 0:
            table[r][at] = free[f] if f < len(free) else -1
    slots, positions = [], []
    for r, pos, at, f in rows:
        id = -1
        if at < len(table[r]):
            id = before[r][at] if f is None else free[f] if f < len(free) else -1
        slots.append(id * page + pos % page if id >= 0 else -1)
        positions.append(pos)
    pad = [-1] * (tokens - len(rows))
    return table, slots + pad, positions + pad, first + [t], [x + y for x, y in zip(c, n)], taken


def _wild_lengths(S, seed):
    rng = random.Random(seed)
    some = [0, 0, 1, 5, 2 ** 29, 2 ** 30, 2 ** 31 - 1, -1, -2 ** 31, rng.randint(0, 2 ** 31 - 1)]
    if seed == 0:
        return [0] * S, [2 ** 29] * S
    if seed == 1:                                   # sums at their limit, then requests without tokens
        return [0] * S, [2 ** 31 - 1 if i < S * 3 // 4 else 0 for i in range(S)]
    if seed == 2:
        return [2 ** 31 - 1] * S, [70 if i == 0 else rng.choice(some) for i in range(S)]
    return [rng.choice(some) for _ in range(S)], [rng.choice(some) for _ in range(S)]


def _wrapping_lengths(seed):
    """(Sums of these that wrap around 32 bits would give a token of theirs a page number below zero.)"""
    rng = random.Random(seed)
    S = rng.choice([5, 6, 8, 9, 12, 40])
    return [rng.choice([0, 0, 100, 2 ** 29]) for _ in range(S)], [rng.choice([0, 1, 2 ** 29, 2 ** 29, 2 ** 31 - 1, 5]) for _ in range(S)]


def _check_bounded(c, n, page, tokens):
    """No entry outside the table and the free list is read or written."""
    from nsa.paged import block_tables
    S, P = len(c), 5
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    around = torch.full((S + 2000, P), 12345678, dtype=torch.int32, device="cuda")       # an entry of it would give itself away
    table = around[1000:1000 + S]
    host = [[r * P + i for i in range(P)] for r in range(S)]
    table.copy_(i32(host))
    free = list(range(100000, 100050))
    want = _bounded_tables(c, n, host, free, tokens, page)
    step = block_tables(i32(c), i32(n), table, i32(free), tokens, page)
    assert table.tolist() == want[0]
    assert [x.tolist() for x in step[:4]] == [want[1], want[2], want[3], want[4]] and step.pages.tolist() == [want[5]]
    assert (around[:1000] == 12345678).all() and (around[1000 + S:] == 12345678).all()


@pytest.mark.gpu
@pytest.mark.parametrize("S", [4, 40, 300, 1100])
@pytest.mark.parametrize("page", [1, 64, 65536])
@pytest.mark.parametrize("seed", [0, 1, 2, 3, 4])
def test_block_tables_of_lengths_beyond_reason(S, page, seed):
    _check_bounded(*_wild_lengths(S, 5 * seed + S if seed > 2 else seed), page, 2000)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [27, 1171, 1241, 1892, 1958])
def test_block_tables_of_sums_that_would_wrap(seed):
    _check_bounded(*_wrapping_lengths(seed), 64, 64)


# ------------------------------------------------------------------------------------------------ one key far above many

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,new", [(BF, 1), (BF, 16), (F32, 1)])
@pytest.mark.parametrize("heads", HEADS)
def test_one_key_far_above_a_long_tail(dtype, new, heads):
    """A first key whose logit is 12 to 21 above those of 50 000 others, in segments that a block has whole: what the others add up to is
    still there, each off by no more than 2^-32 of the first.  (Its own value is 0, so nothing else shows.)"""
    from types import SimpleNamespace

    from nsa.paged import PagedCache4
    H, G, dk, dv = heads
    hp, T = H // G, 50000
    S = (592 if new == 1 else 148) // G                     # as many segments of one length as there are thread blocks
    pages = -(-T // 64)
    c = PagedCache4.empty(pages, G, dk, dv)
    k, v = torch.zeros(T, G, dk, device="cuda"), torch.ones(T, G, dv, device="cuda")
    k[0], v[0] = 1, 0
    slots = torch.arange(T, device="cuda")
    c.append(k, v, slots)
    k, v = c.read(slots)
    up = torch.linspace(12, 21, hp, device="cuda").repeat(G) / dk ** 0.5          # logit = up * dk * dk^-1/2
    q = up[None, :, None].expand(new, H, dk).to(dtype).contiguous()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = torch.arange(pages, device="cuda", dtype=torch.int32).repeat(S, 1)
    o, L, M = c.attend(q.repeat(S, 1, 1), table, i32([T] * S), i32([new * r for r in range(S + 1)]))
    for x in (o, L, M):
        assert torch.equal(x.view(S, new, *x.shape[1:]), x[:new].expand(S, *x[:new].shape))
    s = SimpleNamespace(lengths=[T], starts=[0, new], dk=dk, k=[k], v=[v])
    want = by_request(s, q)
    ref.check((o[:new], L[:new], M[:new]), want, dtype, T, dk)
    ro, rL, rM, A, B, V = want
    # the probabilities' own roundings are 2^-11; logits and 32-bit sums as in ref.check
    rel = 2 * (dk * 2.0 ** -24 * B + 2.0 ** -23 * rM) + T * 2.0 ** -24 + 2.0 ** -22 + (2.0 ** -11 if dtype == BF else 0)
    tol = rel[..., None] * A + (2.0 ** -8 if dtype == BF else 2.0 ** -23) * ro + (2.0 ** -32 * V if dtype == BF else 0)
    err = (o[:new].double() - ro).abs()
    assert bool((err <= tol).all()), f"off by up to {(err / tol).max().item():.3g} of the bound"


# ------------------------------------------------------------------------------------------------ queries and scales at the ends of their range

@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("size", [1e6, 1e8, 1e10, 1e20, 1e33, 1e36])
def test_large_queries(new, heads, size):
    """Logits of 1e6 to 1e37: hardly more than the largest key counts."""
    s = Served([300], [new], *heads, BF, seed=41)
    H, G, dk, _ = heads
    s.q.mul_(size)
    o, L, M = s.check()
    x = torch.einsum("nghd,tgd->nght", s.q.double().unflatten(1, (G, H // G)), s.k[0].double()).reshape(new, H, 300) * dk ** -0.5
    near = torch.einsum("nghd,tgd->nght", s.q.double().abs().unflatten(1, (G, H // G)), s.k[0].double().abs()).reshape(new, H, 300).amax(-1) * dk ** -0.5
    x = x.masked_fill(torch.arange(300, device="cuda") > 300 - new + torch.arange(new, device="cuda")[:, None, None], -math.inf)
    top, at = x.topk(2, -1)
    sure = top[..., 0] - top[..., 1] > 2 * dk * 2.0 ** -24 * near + 1000          # further apart than a logit is off
    assert sure.float().mean() > 0.9
    first = s.v[0][at[..., 0], torch.arange(H, device="cuda") // (H // G)]           # [new, H, dv]
    assert torch.equal(o[sure], first[sure].bfloat16()) and not L[sure].any() and M.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_scales_near_zero(dtype, new):
    """Scales down to the smallest numbers there are: the mean of what a row sees."""
    s = Served([300, 70], [new, 1], *HEADS[2], dtype, seed=42)
    for size in (1.0, 1e-30):
        s.q.mul_(size)
        for scale in (1e-12, 1e-25, 1e-38, 1e-44, -1e-30):
            scale = torch.tensor(scale).item()              # (as 32 bits have it)
            o, L, M = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, scale=scale)
            ro, rL, rM, A, B, V = by_request(s, s.q, scale=scale)
            # 32 bits keep no relative precision below 2^-126: largest logits are off by as much besides what ref.check allows
            assert bool(((M - rM).abs() <= 64 * 2.0 ** -24 * B + 2.0 ** -23 * rM.abs() + 2.0 ** -126).all())
            ref.check((o, L, rM), (ro, rL, rM, A, B, V), dtype, 300, 64)


# ------------------------------------------------------------------------------------------------ some of a step's requests

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heads", [(BF, HEADS[0]), (BF, HEADS[2]), (F32, HEADS[2]), (BF, ODD_HEADS[0])])
@pytest.mark.parametrize("form", ["all", "window", "selected"])
@pytest.mark.parametrize("first,last", [(1, 5), (2, 4), (0, 3), (3, 3), (4, 5)])
def test_some_requests_of_a_step(dtype, heads, form, first, last):
    """Slices of the tables, lengths and starts of a step: only the rows of those requests are written."""
    s = Served([200, 90, 64, 333, 70], [3, 1, 40, 2, 60], *heads, dtype, seed=50)
    N, G = s.starts[-1], heads[1]
    gen = torch.Generator().manual_seed(51)
    kw = dict(window=33) if form == "window" else {}
    if form == "selected":
        kw = dict(indices=torch.randint(-1, 6, (N, G, 4), generator=gen, dtype=torch.int32).cuda())
    want = ref.attend(s.q, s.k, s.v, s.lengths, s.starts, s.dk ** -0.5, **kw)
    out = torch.full((N, heads[0], heads[3]), 5.0, device="cuda", dtype=dtype)
    o, L, M = s.cache.attend(s.q, s.table[first:last], s.len_dev[first:last], s.starts_dev[first:last + 1], out=out, **kw)
    a, b = s.starts[first], s.starts[last]
    ref.check([x[a:b] for x in (o, L, M)], [x[a:b] for x in want], dtype, 333, s.dk) if a < b else None
    assert (out[:a] == 5).all() and (out[b:] == 5).all()


# ------------------------------------------------------------------------------------------------ refusals (no GPU)

def test_counts_beyond_32_bits():
    """Counts that 32 bits would cut short are refused, not cut."""
    from nsa import _lib as L
    from nsa.paged import PagedCache4, block_tables
    one, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    for tokens, page in ((2 ** 32 + 2, 64), (2 ** 30 + 1, 64), (2, 2 ** 32 + 64), (2, 65537)):
        with pytest.raises(ValueError, match="tokens"):
            block_tables(one, one, table, one, tokens, page)
    assert L.lib.nsa_block_tables(16, 16, 16, 4, 16, 16, 16, 16, 16, 16, 1, 4, 1, 2 ** 30 + 1, 64, None) == -1
    c = PagedCache4.empty(2, 2, 64, 64, device="cpu")
    with pytest.raises(RuntimeError):               # (a bound of any size is one: what is missing is the GPU)
        c.attend(torch.zeros(3, 4, 64), table, one, torch.zeros(3, dtype=torch.int32), max_new=2 ** 40)


@pytest.mark.gpu
def test_a_bound_beyond_32_bits():
    s = Served([90, 40], [30, 1], *HEADS[0], BF, seed=52)
    s.check(max_new=2 ** 40)


def test_table_rows_that_overlap():
    from nsa import _lib as L
    from nsa.paged import PagedCache4
    i32 = dict(dtype=torch.int32)
    c = PagedCache4.empty(2, 2, 64, 64, device="cpu")
    q, lengths, starts = torch.zeros(2, 4, 64), torch.ones(2, **i32), torch.arange(3, **i32)
    for table in (torch.zeros(1, 3, **i32).expand(2, 3), torch.zeros(5, **i32).as_strided((2, 3), (2, 1))):
        with pytest.raises(ValueError, match="overlap"):
            c.attend(q, table, lengths, starts)
    with pytest.raises(RuntimeError):               # a row of its own needs no distance
        c.attend(q[:1], torch.zeros(1, 3, **i32).expand(1, 3), lengths[:1], starts[:2])
    d = dict(N=1, S=2, P=3, H=4, G=2, dk=64, dv=64, n_pages=1, n_sel=0, window=0, max_new=0, dtype=1, scale=1.0, s0=256, s1=64, ld=2, q=16, cache=16,
             table=16, lengths=16, starts=16, indices=0, out=16, L=16, M=16)
    assert L.lib.nsa_cache4_attn_fwd(L.CACHE4_DESC.pack(*d.values()), 16, 1 << 40, None) == -1 and b"overlap" in L.lib.nsa_last_error()


def test_scales_that_are_not_finite():
    from nsa import _lib as L
    from nsa.paged import PagedCache4
    i32 = dict(dtype=torch.int32)
    c = PagedCache4.empty(2, 2, 64, 64, device="cpu")
    d = dict(N=1, S=1, P=3, H=4, G=2, dk=64, dv=64, n_pages=1, n_sel=0, window=0, max_new=0, dtype=1, scale=1.0, s0=256, s1=64, ld=3, q=16, cache=16,
             table=16, lengths=16, starts=16, indices=0, out=16, L=16, M=16)
    for scale in (math.nan, math.inf, -math.inf):
        with pytest.raises(ValueError, match="scale"):
            c.attend(torch.zeros(1, 4, 64), torch.zeros(1, 3, **i32), torch.ones(1, **i32), torch.arange(2, **i32), scale=scale)
        assert L.lib.nsa_cache4_attn_fwd(L.CACHE4_DESC.pack(*{**d, "scale": scale}.values()), 16, 1 << 40, None) == -1 and b"scale" in L.lib.nsa_last_error()


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits

@pytest.mark.gpu
def test_pages_behind_4_gigabytes():
    """The last pages of a cache of 6 GB: the same bits as in a small one, written, read and attended to."""
    from nsa.paged import PagedCache4
    H, G, dk, dv = HEADS[0]
    pages = 130000
    big = PagedCache4(torch.empty(pages, G, 64 * 180, device="cuda", dtype=torch.uint8), dk, dv)
    assert big.storage.numel() > 5 << 30
    for dtype, new in ((BF, 1), (BF, 20), (F32, 2)):
        s = Served([700, 90], [new, 1], H, G, dk, dv, dtype, seed=53)
        n = s.cache.storage.shape[0]
        table = torch.where((s.table >= 0) & (s.table < n), s.table + (pages - n), s.table)
        for r, length in enumerate(s.lengths):
            pos = torch.arange(length, device="cuda")
            slots = table[r, pos // 64].long() * 64 + pos % 64
            big.append(s.k[r], s.v[r], slots)              # (what the small cache holds is held exactly again)
            assert all(torch.equal(x, y) for x, y in zip(big.read(slots), (s.k[r], s.v[r])))
        idx = torch.randint(-1, 12, (s.starts[-1], G, 5), dtype=torch.int32).cuda()
        for kw in ({}, dict(window=70), dict(indices=idx)):
            want = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, **kw)
            assert all(torch.equal(x, y) for x, y in zip(want, big.attend(s.q, table, s.len_dev, s.starts_dev, **kw)))
