"""Paged serving: block tables, the 4-bit cache and attention over it, against 64-bit restatements of their definitions."""
import math
import random

import pytest
import torch

from tests import paged_ref as ref

BF, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------ refusals (no GPU)

def test_page_bytes():
    from nsa._lib import lib
    assert lib.nsa_cache4_page_bytes(192, 128) == 64 * 180
    for bad in ((0, 128), (192, 0), (100, 128), (192, 48), (288, 128), (-32, 64)):
        assert lib.nsa_cache4_page_bytes(*bad) == 0


def test_refusals_of_the_library():
    from nsa import _lib as L
    lib, one = L.lib, 16          # a pointer that is never followed
    assert lib.nsa_block_tables(one, one, one, 3, one, one, one, one, one, one, 1, 4, 1, 1, 64, None) == -1      # rows closer than they are long
    assert lib.nsa_block_tables(one, one, one, 4, one, one, one, one, one, one, 16385, 4, 1, 1, 64, None) == -1
    assert b"16384" in lib.nsa_last_error()
    assert lib.nsa_block_tables(one, one, one, 4, one, None, one, one, one, one, 1, 4, 1, 1, 64, None) == -1
    assert lib.nsa_block_tables(one, one, one, 4, one, one, one, one, one, one, 1, 4, 1, 1, 0, None) == -1
    assert lib.nsa_cache4_append(one, one, None, one, one, 1, 1, 1, 64, 64, 1, None) == -1
    assert lib.nsa_cache4_append(one, one, L.i64([1] * 6), one, one, 1, 1, 1, 64, 40, 1, None) == -1
    assert lib.nsa_cache4_append(one, one, L.i64([1] * 6), one, 8, 1, 1, 1, 64, 64, 1, None) == -1               # misaligned cache
    assert lib.nsa_cache4_read(one, one, one, 24, 1, 1, 1, 64, 64, 0, None) == -1

    def attn(ws=one, nbytes=1 << 40, **kw):
        d = dict(N=1, S=1, P=1, H=4, G=2, dk=64, dv=64, n_pages=1, n_sel=0, window=0, max_new=0, dtype=1, scale=1.0, s0=256, s1=64, ld=1,
                 q=one, cache=one, table=one, lengths=one, starts=one, indices=0, out=one, L=one, M=one)
        d.update(kw)
        return lib.nsa_cache4_attn_fwd(L.CACHE4_DESC.pack(*d.values()), ws, nbytes, None)

    for kw in (dict(H=3), dict(G=0), dict(dk=80), dict(dv=512), dict(dtype=2), dict(n_sel=33, indices=one), dict(n_sel=4), dict(n_sel=4, indices=one, window=3),
               dict(window=-1), dict(N=-1), dict(P=2), dict(q=0), dict(out=0), dict(M=0), dict(starts=0), dict(cache=8), dict(P=1 << 24, ld=1 << 24)):
        assert attn(**kw) == -1, kw
    assert attn(ws=0) == -3 and attn(nbytes=16) == -3 and attn(ws=8) == -3
    assert attn(N=0) == 0 and attn(S=0) == 0


def test_refusals_of_the_package():
    from nsa.paged import PagedCache4, block_tables
    i32 = dict(dtype=torch.int32)
    t, one = torch.zeros(2, 3, **i32), torch.zeros(2, **i32)
    for bad in (dict(cached=one.long()), dict(new=torch.zeros(3, **i32)), dict(table=t.t()), dict(free_pages=t), dict(tokens=-1), dict(page_tokens=0),
                dict(table=t[:1].expand(2, 3)), dict(table=one)):
        with pytest.raises(ValueError):
            block_tables(**{**dict(cached=one, new=one, table=t, free_pages=one, tokens=2), **bad})
    with pytest.raises(RuntimeError):               # no CPU path
        block_tables(one, one, t, one, 2)
    for st, dk in ((torch.zeros(2, 2, 100, dtype=torch.uint8), 64), (torch.zeros(2, 2, 64 * 72), 64), (torch.zeros(2, 2, 64 * 72, dtype=torch.uint8), 65)):
        with pytest.raises(ValueError):
            PagedCache4(st, dk, 64)
    c = PagedCache4.empty(2, 2, 64, 64, device="cpu")
    k, slots = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int64)
    for args in ((k[:, :1], k, slots), (k, k[:2], slots), (k, k, slots[:2]), (k, k, slots.int()), (k, k, torch.zeros(6, dtype=torch.int64)[::2])):
        with pytest.raises(ValueError):
            c.append(*args)
    with pytest.raises(TypeError):
        c.append(k.half(), k.half(), slots)
    with pytest.raises(TypeError):
        c.append(k, k.bfloat16(), slots)
    with pytest.raises(TypeError):
        c.read(slots, torch.float16)
    q, lens, starts, idx = torch.zeros(3, 4, 64), torch.zeros(2, **i32), torch.zeros(3, **i32), torch.zeros(3, 2, 5, **i32)
    good = dict(q=q, table=t, lengths=lens, starts=starts)
    for bad in (dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(lengths=starts), dict(starts=lens), dict(table=t.long()), dict(window=0),
                dict(window=5, indices=idx), dict(indices=idx[:2]), dict(indices=idx[..., :0]), dict(indices=torch.zeros(3, 2, 33, **i32)),
                dict(indices=idx.transpose(0, 1).contiguous().transpose(0, 1)), dict(out=q.bfloat16()), dict(out=torch.zeros(3, 4, 32)), dict(max_new=-1)):
        with pytest.raises(ValueError):
            c.attend(**{**good, **bad})
    with pytest.raises(TypeError):
        c.attend(**{**good, "q": q.double()})
    with pytest.raises(RuntimeError):
        c.attend(**good)


# ------------------------------------------------------------------------------------------------ block tables

def _tables_case(rng, S, P, page, most_cached, most_new, spare):
    cached = [rng.choice([0, rng.randint(0, most_cached), page, page - 1 if page > 1 else 1]) for _ in range(S)]
    new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(S)]
    table, ids = [], list(range(sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 10))
    rng.shuffle(ids)
    for c in cached:
        have = -(-c // page)
        table.append([ids.pop() for _ in range(have)] + [-7] * (P - have))
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
    return cached, new, table, ids[:max(0, need + spare)]


def _check_tables(step, table, want):
    assert table.tolist() == want[0]
    assert [x.tolist() for x in step[:4]] == [want[1], want[2], want[3], want[4]] and step.pages.tolist() == [want[5]]
    assert [x.dtype for x in step] == [torch.int64] + [torch.int32] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("S,page,cached,new,spare,pad", [(1, 64, 5000, 3000, 3, 0), (1, 64, 0, 1, 0, 0), (3, 64, 200, 200, 1, 5), (7, 16, 100, 90, -3, 0),
                                                         (257, 64, 500, 30, 2, 1), (300, 1, 9, 9, -40, 9), (1000, 64, 3000, 70, 0, 4000), (2500, 48, 300, 3, 8, 0)])
def test_block_tables(S, page, cached, new, spare, pad):
    from nsa.paged import block_tables
    rng = random.Random(S + page)
    P = -(-(cached + new) // page) + 1
    c, n, table, free = _tables_case(rng, S, P, page, cached, new, spare)
    tokens = sum(n) + pad
    want = ref.tables(c, n, table, free, tokens, page)
    wide = torch.full((S, P + 3), -9, dtype=torch.int32, device="cuda")
    t = wide[:, :P]                                             # rows further apart than they are long
    t.copy_(torch.tensor(table, dtype=torch.int32))
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (c, n, free)]
    step = block_tables(dev[0], dev[1], t, dev[2], tokens, page)
    _check_tables(step, t, want)
    assert (wide[:, P:] == -9).all()
    again = block_tables(dev[0], dev[1], t, dev[2], tokens, page)      # the same step again: the same pages
    _check_tables(again, t, want)


@pytest.mark.gpu
def test_block_tables_that_do_not_fit():
    """Rows too short, no requests, no tokens, lengths below zero and beyond reason: no fault, slot -1 for what has no page."""
    from nsa.paged import block_tables
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = 5
    step = block_tables(dev(60, 0), dev(100, 3), table, dev(8, 9, 3, 4), 110)
    want = ref.tables([60, 0], [100, 3], [[5, -1], [-1, -1]], [8, 9, 3, 4], 110, 64)
    _check_tables(step, table, want)
    assert step.slots[4:68].tolist() == list(range(8 * 64, 9 * 64)) and (step.slots[68:100] == -1).all()
    empty = block_tables(dev(), dev(), table[:0], dev(), 3)
    assert empty.slots.tolist() == [-1] * 3 and empty.starts.tolist() == [0] and empty.pages.tolist() == [0]
    none = block_tables(dev(7), dev(0), table[:1].clone(), dev(), 0)
    assert none.slots.numel() == 0 and none.lengths.tolist() == [7]
    before = table.clone()
    big = block_tables(dev(-5, 2 ** 31 - 1), dev(2 ** 31 - 1, -2 ** 31), table, dev(2), 70)
    assert big.positions.tolist() == list(range(70)) and big.slots[:64].tolist() == list(range(128, 192)) and (big.slots[64:] == -1).all()
    assert torch.equal(table[1], before[1])


# ------------------------------------------------------------------------------------------------ tokens in and out

def _held(x):
    return ref.quantise(x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,G,dk,dv", [(1, 1, 32, 32), (3, 4, 192, 128), (64, 2, 128, 128), (200, 2, 64, 64), (130, 3, 96, 160), (33, 1, 256, 256), (2111, 4, 192, 128)])
def test_append_and_read(dtype, N, G, dk, dv):
    """Quantised values equal the definition's bit for bit; other tokens of the same pages keep theirs."""
    from nsa.paged import PagedCache4
    gen = torch.Generator(device="cuda").manual_seed(N * dk)
    pages = N // 64 + 3
    c = PagedCache4.empty(pages, G, dk, dv)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    every = torch.randperm(pages * 64, generator=gen, device="cuda")
    old_k, old_v = rn(pages * 64, G, dk).to(dtype), rn(pages * 64, G, dv).to(dtype)
    c.append(old_k, old_v, every)
    k, v = (rn(N, G, dk) * rn(N, G, 1).exp()).to(dtype), (rn(N, G, dv) * 100).to(dtype)
    slots = every[:N].contiguous()
    c.append(k, v, slots)
    rk, rv = c.read(slots)
    assert rk.dtype == F32 and torch.equal(rk.double(), _held(k)) and torch.equal(rv.double(), _held(v))
    rk, rv = c.read(every[N:].contiguous())
    assert torch.equal(rk.double(), _held(old_k[N:])) and torch.equal(rv.double(), _held(old_v[N:]))
    bk, bv = c.read(slots, BF)
    assert torch.equal(bk, _held(k).float().bfloat16()) and torch.equal(bv, _held(v).float().bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_values_at_the_edges(dtype):
    """Zeros, infinities, NaN, values below and above what 4 bits with an fp16 scale hold, exact ties, one large value among small ones."""
    from nsa.paged import PagedCache4
    x = torch.zeros(24, 1, 32)
    x[1, 0, 3], x[2, 0, 4], x[3, 0, 5] = math.inf, -math.inf, math.nan
    x[4] = torch.randn(32) * 1e-7
    x[5] = torch.randn(32) * 1e-6
    x[6] = torch.randn(32) * 3e38
    x[7] = torch.randn(32) * 2e4
    x[8], x[8, 0, 0] = 1e-3, 1e4
    x[9] = torch.arange(32).float() / 2 - 7                       # scale 1: every second quotient is a tie
    x[10] = 7.0 * 2 ** -24
    x[11] = 3.4 * 2 ** -24
    x[12] = 57120.0
    x[13] = 57300.0
    x[14] = 1e-45
    for i in range(15, 24):                                       # a seventh right at a border of 8 bits, and its neighbours in 32 bits
        edge = torch.tensor(7 * (128 + 0.5 + i % 3) * 2.0 ** (i - 18))
        x[i, 0, 0] = [edge, torch.nextafter(edge, edge * 2), torch.nextafter(edge, edge / 2)][i // 3 % 3]
        x[i, 0, 1:] = torch.linspace(-1, 1, 31) * edge
    x = x.to(dtype).cuda()
    c = PagedCache4.empty(1, 1, 32, 32)
    slots = torch.arange(24, device="cuda")
    c.append(x, x.flip(0).contiguous(), slots)
    k, v = c.read(slots)
    assert torch.equal(k.double(), _held(x)) and torch.equal(v.double(), _held(x.flip(0)))
    assert k.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_strides_and_slots_outside(dtype):
    """Time-contiguous keys as the projections write them, views off 16-byte boundaries, broadcast heads; slots that are no slots."""
    from nsa.paged import PagedCache4
    G, dk, dv, N = 2, 64, 96, 21
    base = torch.randn(G, dk, N + 3, device="cuda").to(dtype)
    k = base[..., 1:N + 1].permute(2, 0, 1)                       # strides (1, dk * T, T)
    wide = torch.randn(N, G * dv + 5, device="cuda").to(dtype)
    v = wide[:, 3:3 + G * dv].unflatten(1, (G, dv))               # rows off alignment
    slots = torch.arange(N, device="cuda") * 3
    slots[4], slots[5], slots[6], slots[7] = -1, 64 * 2, 2 ** 40, -2 ** 60
    c = PagedCache4.empty(2, G, dk, dv)
    c.append(k, v, slots)
    rk, rv = c.read(slots)
    ok = (slots >= 0) & (slots < 128)
    assert torch.equal(rk[ok].double(), _held(k)[ok]) and torch.equal(rv[ok].double(), _held(v)[ok])
    assert not rk[~ok].any() and not rv[~ok].any()
    rest = torch.tensor([s for s in range(128) if s not in slots.tolist()], device="cuda")
    assert not c.read(rest)[0].any() and not c.read(rest)[1].any()
    one = torch.randn(1, 1, dk, device="cuda").to(dtype).expand(N, G, dk)
    c.append(one, v, torch.arange(N, device="cuda"))
    assert torch.equal(c.read(torch.arange(N, device="cuda"))[0].double(), _held(one))
    c.append(k[:0], v[:0], slots[:0])
    assert c.read(slots[:0])[0].shape == (0, G, dk)


# ------------------------------------------------------------------------------------------------ attention

class Served:
    """Requests with random contents in a cache: pages in random order, table rows longer than needed."""

    def __init__(self, lengths, new, H, G, dk, dv, dtype, seed=0, extra=2, strided_q=False):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        host = random.Random(seed)
        from nsa.paged import PagedCache4
        self.lengths, self.new, S = lengths, new, len(lengths)
        per = [-(-n // 64) for n in lengths]
        ids = list(range(sum(per) + 2))
        host.shuffle(ids)
        P = max(per) + extra
        self.table_host = [[ids.pop() for _ in range(p)] + [host.choice([-1, 10 ** 6, -5])] * (P - p) for p in per]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.table, self.len_dev = i32(self.table_host).view(S, P), i32(lengths)
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.starts_dev = i32(self.starts)
        N = self.starts[-1]
        self.cache = PagedCache4.empty(sum(per) + 2, G, dk, dv)
        self.k, self.v = [], []
        for r, n in enumerate(lengths):
            k, v = torch.randn(n, G, dk, generator=gen, device="cuda"), torch.randn(n, G, dv, generator=gen, device="cuda")
            pos = torch.arange(n, device="cuda")
            slots = self.table[r, pos // 64].long() * 64 + pos % 64
            self.cache.append(k, v, slots)
            k, v = self.cache.read(slots)
            self.k.append(k)
            self.v.append(v)
        q = torch.randn(N, H, dk, generator=gen, device="cuda").to(dtype)
        if strided_q:
            q = torch.empty(H, N, dk + 8, device="cuda", dtype=dtype)[..., :dk].permute(1, 0, 2).copy_(q)
        self.q, self.dtype, self.dk = q, dtype, dk

    def check(self, scale=None, window=None, indices=None, max_new=None, seen_keys=None):
        got = self.cache.attend(self.q, self.table, self.len_dev, self.starts_dev, scale=scale, window=window, indices=indices, max_new=max_new)
        want = ref.attend(self.q, self.k, self.v, self.lengths, self.starts, scale or self.dk ** -0.5, window, indices, seen_keys)
        ref.check(got, want, self.dtype, max(self.lengths + [1]), self.dk)
        return got


HEADS = [(64, 4, 192, 128), (32, 2, 128, 128), (8, 2, 64, 64)]
ODD_HEADS = [(3, 3, 96, 160), (10, 2, 32, 256), (20, 1, 256, 32), (48, 2, 64, 64), (7, 1, 192, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", HEADS + ODD_HEADS)
def test_decode(heads, dtype):
    """One token a request; lengths of one token, around page and record borders, empty requests among them."""
    lengths = [1, 64, 65, 63, 16, 17, 130, 1000, 2]
    Served(lengths, [1] * 9, *heads, dtype, seed=1).check()
    Served([300, 5, 77], [1, 0, 1], *heads, dtype, seed=2).check(max_new=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", HEADS + ODD_HEADS[:2])
@pytest.mark.parametrize("window", [None, 1, 40, 64, 500])
def test_several_tokens_and_windows(heads, dtype, window):
    Served([5, 600, 64, 90], [5, 3, 0, 4], *heads, dtype, seed=3, strided_q=True).check(window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heads", [(BF, HEADS[0]), (BF, HEADS[1]), (BF, HEADS[2]), (F32, HEADS[2]), (BF, ODD_HEADS[0])])
@pytest.mark.parametrize("window", [None, 70])
def test_chunks(dtype, heads, window):
    """Prompts from an empty cache, chunks behind cached tokens and single tokens in one step."""
    Served([150, 333, 40, 259, 1], [150, 70, 1, 64, 1], *heads, dtype, seed=4).check(window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", HEADS + ODD_HEADS[1:4])
@pytest.mark.parametrize("n", [1, 5, 16, 32])
def test_selected_blocks(heads, dtype, n):
    """Block lists with repetitions, negative entries, blocks in the future and behind the table, and none at all."""
    s = Served([700, 64, 1, 333], [3, 1, 1, 40], *heads, dtype, seed=5)
    G = heads[1]
    gen = torch.Generator().manual_seed(n)
    idx = torch.randint(-2, 13, (s.starts[-1], G, n), generator=gen, dtype=torch.int32)
    idx[1] = -1                                         # a token that sees nothing
    idx[2] = idx[2, :, :1]                              # one block, again and again
    idx[3, :, 0] = 2 ** 31 - 1
    s.check(indices=idx.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", HEADS)
def test_long_and_uneven(heads, dtype):
    """Segments that many blocks share, next to short ones; a long cache split over the whole GPU."""
    Served([20000, 3, 4000, 64], [1, 1, 2, 1], *heads, dtype, seed=6).check()
    Served([9000], [1], *heads, dtype, seed=7).check(window=5000)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_missing_pages_and_lengths_that_do_not_fit(dtype):
    """Keys on pages that the table does not give are not seen; a request shorter than its new tokens has rows that see nothing."""
    s = Served([300, 200, 100], [2, 1, 1], *HEADS[2], dtype, seed=8)
    s.table[0, 1], s.table[1, 0] = -1, 10 ** 8
    gone = {0: (64, 128), 1: (0, 64)}

    def seen(r):
        j = torch.arange(s.lengths[r], device="cuda")
        return ~((j >= gone[r][0]) & (j < gone[r][1])) if r in gone else torch.ones_like(j, dtype=torch.bool)

    s.check(seen_keys=seen)
    s.table[:] = -1
    o, L, M = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
    assert not o.any() and (L == -math.inf).all() and (M == -math.inf).all()
    short = Served([2, 70], [2, 1], *HEADS[2], dtype, seed=9)
    o, L, M = short.cache.attend(short.q, short.table, short.len_dev - torch.tensor([1, 0], dtype=torch.int32, device="cuda"), short.starts_dev)
    assert not o[0].any() and (M[0] == -math.inf).all() and o[1:].isfinite().all() and (M[1:] > -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", [HEADS[0], HEADS[2], ODD_HEADS[0]])
@pytest.mark.parametrize("new", [1, 60])
def test_bytes_never_written_do_not_matter(heads, dtype, new):
    """What lies behind the last token of a page and on pages of nobody is NaN here: no output changes."""
    s = Served([77, 1 + new, 130], [new, 1, new], *heads, dtype, seed=10)
    before = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, window=50)
    all_before = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
    held = [s.cache.read(s.table[r, torch.arange(n, device="cuda") // 64].long() * 64 + torch.arange(n, device="cuda") % 64) for r, n in enumerate(s.lengths)]
    s.cache.storage.fill_(255)                          # fp16 NaN in every scale
    slots = [s.table[r, torch.arange(n, device="cuda") // 64].long() * 64 + torch.arange(n, device="cuda") % 64 for r, n in enumerate(s.lengths)]
    for (k, v), at in zip(held, slots):
        s.cache.append(k, v, at)                        # what was held is held exactly again
    for a, b in zip(before, s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, window=50)):
        assert torch.equal(a, b)
    for a, b in zip(all_before, s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_behind_the_last_request_stay(dtype):
    s = Served([70, 200], [1, 3], *HEADS[0], dtype, seed=11)
    q = torch.cat((s.q, torch.full((5, *s.q.shape[1:]), math.nan, device="cuda", dtype=dtype)))
    out = torch.full((9, 64, 128), 3.0, device="cuda", dtype=dtype)
    o, L, M = s.cache.attend(q, s.table, s.len_dev, s.starts_dev, out=out)
    assert o is out and (out[4:] == 3.0).all() and out[:4].isfinite().all()
    idx = torch.zeros(9, 4, 3, dtype=torch.int32, device="cuda")
    s.cache.attend(q, s.table, s.len_dev, s.starts_dev, indices=idx, out=out)
    assert (out[4:] == 3.0).all()
    ref.check(s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev),
              ref.attend(s.q, s.k, s.v, s.lengths, s.starts, 192 ** -0.5), dtype, 200, 192)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_logits_far_apart(dtype, new):
    """Queries of very different sizes: rows of zeros, tiny rows, rows whose softmax is one key."""
    s = Served([400, 90], [new, 1], *HEADS[2], dtype, seed=12)
    s.q[:, 0] = 0
    s.q[:, 1] *= 1e-6
    s.q[:, 2] *= 30
    s.q[:, 3] *= 1e-30
    s.q[:, 4, 5:] *= 1e-8
    s.check()
    s.check(scale=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_queries_of_any_layout(dtype):
    """Rows off 16-byte boundaries, strided dimensions, heads before tokens: through the package and straight into the library."""
    from nsa import ops
    H, G, dk, dv = HEADS[0]
    s = Served([300, 70], [3, 1], H, G, dk, dv, dtype, seed=15)
    want = ref.attend(s.q, s.k, s.v, s.lengths, s.starts, dk ** -0.5)
    odd = torch.empty(4 * H * (dk + 1) + 1, device="cuda", dtype=dtype)[1:].view(4, H, dk + 1)[..., :dk].copy_(s.q)
    for q in (odd, torch.empty(dk, H, 4, device="cuda", dtype=dtype).permute(2, 1, 0).copy_(s.q),
              torch.empty(4 * H * dk + 3, device="cuda", dtype=dtype)[3:].view(4, H, dk).copy_(s.q)):
        ref.check(s.cache.attend(q, s.table, s.len_dev, s.starts_dev), want, dtype, 300, dk)
    ref.check(ops.cache4_attn(odd, s.cache.storage, s.table, s.len_dev, s.starts_dev, None, dk, dv, 0, dk ** -0.5, 0), want, dtype, 300, dk)


@pytest.mark.gpu
def test_same_bits_twice_and_on_another_stream():
    for dtype, new in ((BF, 1), (F32, 1), (BF, 50)):
        s = Served([3000, 500, 64], [new, 1, new], *HEADS[0], dtype, seed=13)
        a = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
        b = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [HEADS[0], HEADS[2], ODD_HEADS[0]])
def test_bounds_that_are_not_reached(heads):
    """As many rows as requests times max_new (a padded step, captured or not), but some requests bring fewer tokens, one none."""
    s = Served([300, 40, 5, 129], [16, 3, 0, 1], *heads, BF, seed=16)
    N = s.starts[-1]
    want = ref.attend(s.q, s.k, s.v, s.lengths, s.starts, s.dk ** -0.5)
    for rows, most in ((64, 16), (20, 5), (N, 16), (N, 1), (N, 10 ** 6), (N, None)):
        q = torch.cat((s.q, s.q.new_full((rows - N, *s.q.shape[1:]), math.nan)))
        o, L, M = s.cache.attend(q, s.table, s.len_dev, s.starts_dev, max_new=most)
        ref.check((o[:N], L[:N], M[:N]), want, BF, 300, s.dk)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_more_requests_than_are_counted_at_once(dtype):
    """5000 requests of 1 to 3 cached tokens and 0 to 2 new ones, and one long one behind them all."""
    rng = random.Random(17)
    new = [rng.choice([0, 1, 2]) for _ in range(5000)] + [1]
    s = Served([n + rng.randint(0, 2) for n in new[:-1]] + [700], new, 4, 2, 64, 64, dtype, seed=17, extra=0)
    s.check()
    idx = torch.randint(-1, 3, (s.starts[-1], 2, 4), dtype=torch.int32)
    s.check(indices=idx.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_scales_that_turn_or_level_the_logits(dtype, new, scale):
    s = Served([200, 90], [new, 1], *HEADS[2], dtype, seed=18)
    got = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, scale=scale)
    o, L, M, A, B, V = ref.attend(s.q, s.k, s.v, s.lengths, s.starts, scale)
    ref.check(got, (o, L, M, A, B.abs(), V), dtype, 200, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_an_output_tensor_off_its_boundary(new):
    s = Served([200, 90], [new, 1], *HEADS[0], BF, seed=19)
    want = ref.attend(s.q, s.k, s.v, s.lengths, s.starts, s.dk ** -0.5)
    buf = torch.full(((new + 1) * 64 * 128 + 9,), 7.0, device="cuda", dtype=BF)
    out = buf[3:3 + (new + 1) * 64 * 128].view(new + 1, 64, 128)
    ref.check(s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, out=out), want, BF, 200, 192)
    assert (buf[:3] == 7).all() and (buf[-6:] == 7).all()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    a, b = Served([9000, 30], [1, 1], *HEADS[0], BF, seed=20), Served([700, 400], [100, 60], *HEADS[0], BF, seed=21)
    go = lambda s: s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
    want = go(a), go(b)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                got[k].append(go(s))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for k in range(2) for g in got[k] for x, y in zip(g, want[k]))


@pytest.mark.gpu
def test_refuses_after_a_device_time_out():
    from nsa import _lib as L
    s = Served([100, 90], [1, 60], *HEADS[2], BF, seed=22)
    want = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
    assert L.lib.nsa_selftest_wait_timeout(1 << 16, None) == 0
    try:
        with pytest.raises(L.NSAKernelError, match="time-out"):
            s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)
    finally:
        assert L.lib.nsa_device_timeouts(1) == 1
    assert all(torch.equal(x, y) for x, y in zip(want, s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev)))


# ------------------------------------------------------------------------------------------------ a server's steps

def _serve(steps, H, G, dk, dv, dtype, step_fn):
    """Steps of requests that join, generate and leave; every step's attention against the values the cache holds."""
    from nsa.paged import PagedCache4
    gen = torch.Generator(device="cuda").manual_seed(20)
    S, P, pages = len(steps[0]), 12, 40
    cache = PagedCache4.empty(pages, G, dk, dv)
    table = torch.full((S, P), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, generator=gen, device="cuda").int()
    cached = torch.zeros(S, dtype=torch.int32, device="cuda")
    hk, hv = [torch.zeros(0, G, dk, device="cuda")] * S, [torch.zeros(0, G, dv, device="cuda")] * S
    bound = max(sum(n) for n in steps)
    for new in steps:
        n = torch.tensor(new, dtype=torch.int32, device="cuda")
        rn = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)
        q, k, v = rn(bound, H, dk), rn(bound, G, dk), rn(bound, G, dv)
        step, o, L, M, win = step_fn(cache, cached, n, table, free, bound, q, k, v)
        at = 0
        for r, m in enumerate(new):
            hk[r], hv[r] = torch.cat((hk[r], ref.quantise(k[at:at + m]).float())), torch.cat((hv[r], ref.quantise(v[at:at + m]).float()))
            at += m
        lengths, starts = [x.shape[0] for x in hk], [sum(new[:i]) for i in range(S + 1)]
        assert step.lengths.tolist() == lengths and step.starts.tolist() == starts
        for got, w in (((o, L, M), None), (win, 100)):
            want = ref.attend(q, hk, hv, lengths, starts, dk ** -0.5, window=w)
            ref.check(got, want, dtype, max(lengths), dk)
        cached = step.lengths.clone()
        free = free[int(step.pages):].contiguous()
    return cache, table


STEPS = [[100, 0, 64, 1], [1, 30, 1, 1], [1, 1, 1, 1], [1, 1, 0, 150], [28, 1, 200, 1], [1, 1, 1, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads", HEADS)
def test_a_run_of_steps(heads, dtype):
    from nsa.paged import block_tables

    def step_fn(cache, cached, n, table, free, bound, q, k, v):
        step = block_tables(cached, n, table, free, bound)
        cache.append(k, v, step.slots)
        return (step, *cache.attend(q, table, step.lengths, step.starts), cache.attend(q, table, step.lengths, step.starts, window=100))

    _serve(STEPS, *heads, dtype, step_fn)


@pytest.mark.gpu
def test_a_first_call_under_capture():
    """A process whose first attention call on the device is captured."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from nsa.paged import PagedCache4, block_tables
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
c = PagedCache4.empty(4, 2, 64, 64)
k, q, table = torch.randn(100, 2, 64, device="cuda").bfloat16(), torch.randn(100, 8, 64, device="cuda").bfloat16(), torch.full((1, 3), -1, dtype=torch.int32, device="cuda")
zero, n, free = i32(0), i32(100), i32(3, 0, 1)
torch.cuda.synchronize()
def go():
    step = block_tables(zero, n, table, free, 100)
    c.append(k, k, step.slots)
    return c.attend(q, table, step.lengths, step.starts)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = go()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, go())) and out[0].isfinite().all() and out[0].any()
"""
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=os.path.join(root, "nsa-test_b200")), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
def test_a_captured_step_replayed_with_other_lengths():
    from nsa.paged import block_tables
    H, G, dk, dv = HEADS[0]
    held = {}

    def step_fn(cache, cached, n, table, free, bound, q, k, v):
        def go(b):
            step = block_tables(b["cached"], b["n"], table, b["free"], bound)
            cache.append(b["k"], b["v"], step.slots)
            return (step, *cache.attend(b["q"], table, step.lengths, step.starts), cache.attend(b["q"], table, step.lengths, step.starts, window=100))

        new = dict(cached=cached, n=n, free=torch.cat((free, free.new_full((40 - len(free),), -1))), q=q, k=k, v=v)
        if not held:
            held["b"] = {a: b.clone() for a, b in new.items()}
            b = held["b"]
            b["n"].zero_()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                go(b)                                   # no tokens: nothing is written
            torch.cuda.current_stream().wait_stream(side)
            held["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(held["graph"]):
                held["out"] = go(b)
        for a, b in new.items():
            held["b"][a].copy_(b)
        held["graph"].replay()
        return held["out"]

    _serve(STEPS, H, G, dk, dv, BF, step_fn)


@pytest.mark.gpu
def test_against_the_branches_of_the_layer():
    """Window and selected blocks over the pages against the layer's own branches on the values that the cache holds (fp32, one sequence)."""
    from nsa import ops
    H, G, dk, dv, T, n = 8, 2, 64, 64, 300, 4
    s = Served([T], [T], H, G, dk, dv, F32, seed=14)
    q, k, v = s.q.permute(1, 0, 2)[None].contiguous(), s.k[0].permute(1, 2, 0)[None].contiguous(), s.v[0].permute(1, 0, 2)[None].contiguous()
    close = lambda a, b: (a.permute(1, 0, *range(2, a.dim())) - b[0]).abs().max().item() < 2e-5 * max(1.0, b.abs().max().item())
    o, L, M = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, window=100)
    assert all(close(a, b) for a, b in zip((o, L, M), ops.sliding_fwd(q, k, v, 100, dk ** -0.5)))
    idx = torch.randint(0, 5, (T, G, n), dtype=torch.int32, device="cuda")
    idx[..., 0] = (torch.arange(T, device="cuda") // 64)[:, None]
    o, L, M = s.cache.attend(s.q, s.table, s.len_dev, s.starts_dev, indices=idx)
    assert all(close(a, b) for a, b in zip((o, L, M), ops.slc_fwd(q, k, v, idx.permute(1, 0, 2)[None].contiguous(), 64, dk ** -0.5)))
