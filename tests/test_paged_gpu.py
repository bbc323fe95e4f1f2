"""Paged K/V cache: writer, reader and attention against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tinycoder_inference_b200 import capi, ops

pytestmark = pytest.mark.gpu
F64 = torch.float64


class Paged:
    """A pool with sequences of `lens` rows whose last `new` ones are the call's tokens.  What no sequence holds is
    NaN (fp16, scales) or -128; table entries past a sequence's pages name no page."""

    def __init__(self, store, nH, nKV, hd, lens, new, page, seed=0, fill=True, ragged=True, extra=3):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.store, self.nH, self.nKV, self.hd, self.page = store, nH, nKV, hd, page
        self.lens_h, self.new_h, self.g = lens, new, g
        held = [-(-n // page) for n in lens]
        self.num, per = sum(held) + extra, max(1, max(held))
        order = torch.randperm(self.num, device="cuda", generator=g).to(torch.int32)
        self.pages = torch.full((len(lens), per), -1, dtype=torch.int32, device="cuda")
        self.pages[::2] = self.num
        at = 0
        for b, n in enumerate(held):
            self.pages[b, :n] = order[at:at + n]
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        starts = np.concatenate([[0], np.cumsum(new)])
        self.tokens = int(starts[-1])
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda") if ragged else None
        shape = (self.num, page, nKV, hd)
        self.ks = self.vs = None
        if store == "i8":
            self.kc = torch.full(shape, -128, dtype=torch.int8, device="cuda")
            self.vc = torch.full_like(self.kc, -128)
            self.ks = torch.full(shape[:3], float("nan"), device="cuda")
            self.vs = torch.full_like(self.ks, float("nan"))
        else:
            self.kc = torch.full(shape, float("nan"), dtype=torch.float16, device="cuda")
            self.vc = torch.full_like(self.kc, float("nan"))
        if fill:
            for b, n in enumerate(lens):
                r = self.rows(b, 0, n)
                for c, s in ((self.kc, self.ks), (self.vc, self.vs)):
                    x = self.normal(n, nKV, hd)
                    if store == "i8":
                        c.view(-1, nKV, hd)[r] = (x * 42).round().clamp(-127, 127).to(torch.int8)
                        s.view(-1, nKV)[r] = 0.024 * torch.exp(0.3 * self.normal(n, nKV))
                    else:
                        c.view(-1, nKV, hd)[r] = x.half()

    def normal(self, *shape):
        return torch.randn(shape, device="cuda", generator=self.g)

    def rows(self, b, first, end):
        p = torch.arange(first, end, device="cuda")
        return self.pages[b].long()[p // self.page] * self.page + p % self.page

    def values(self, b, n):
        out = []
        for c, s in ((self.kc, self.ks), (self.vc, self.vs)):
            x = c.view(-1, self.nKV, self.hd)[self.rows(b, 0, n)].to(F64)
            if self.store == "i8":
                x = x * s.view(-1, self.nKV)[self.rows(b, 0, n)].to(F64)[..., None]
            out.append(x)
        return out

    def attend(self, q, ws, max_tokens=0, scale=None):
        out = torch.full_like(q, 77.0)
        ops.attn_paged(q, self.kc, self.vc, self.pages, self.lens, out, ws, starts=self.starts, max_tokens=max_tokens,
                       ks=self.ks, vs=self.vs, invSqrt=scale)
        return out

    def check(self, q, out, scale=None):
        """out against softmax attention in 64 bits, each value within what the kernel's arithmetic may cost:
        scores are off by their products' 2^-21 (q as an fp16 pair) and at most hd / 16 + 3 additions and scalings of 2^-23 each,
        relative to sum |q k|; p by 2^-22 (exp2), its pair by 2^-21, fp16 p by 2^-11; sums by 2^-23 for every tile and 8 joins;
        an fp16 result is rounded by 2^-11.  Everything twice: numerator and denominator.  What a weight is off by however small it
        is: 2^13 p (times the scale of V's row, relative to at most twice the largest scale) is held in fp16, whose smallest step 2^-24
        rounds by 2^-25: 2^-38 of a weight of 1, 2^-37 with the scale, for each of n rows.  (A peaked row whose largest
        weight meets an int8 value of 0 has nothing else: p = 8e-21 then is the whole result.)"""
        scale = 1.0 / math.sqrt(self.hd) if scale is None else scale
        half = q.dtype == torch.float16
        group, at = self.nH // self.nKV, 0
        for b, (n, m) in enumerate(zip(self.lens_h, self.new_h)):
            if m == 0:
                continue
            k, v = self.values(b, n)
            qq, got = q[at:at + m].to(F64), out[at:at + m].to(F64)
            at += m
            see = torch.arange(n, device="cuda")[None, :] <= torch.arange(n - m, n, device="cuda")[:, None]
            if self.store == "i8":
                most = 127.0 * self.vs.view(-1, self.nKV)[self.rows(b, 0, n)].max().item() if n else 0.0
            else:
                most = v.abs().max().item() if n else 0.0
            for h in range(self.nH):
                kh, vh = k[:, h // group], v[:, h // group]
                x = (qq[:, h] @ kh.T * scale).masked_fill(~see, -math.inf)
                top = x.amax(-1, keepdim=True) if n else torch.zeros((m, 1), device="cuda", dtype=F64)
                p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total > 0, total, 1.0)
                want, mass = p @ vh, p @ vh.abs()
                size = (qq[:, h].abs() @ kh.abs().T * scale).masked_fill(~see, 0.0)
                size = size.amax(-1, keepdim=True) if n else top
                c = 2 * (size * (2.0 ** -21 + (self.hd / 16 + 3) * 2.0 ** -23) + 2.0 ** -22 + 2.0 ** -21 + (n / 64 + 8) * 2.0 ** -23)
                tol = (c + (2.0 ** -11 if half else 0.0)) * mass + (2.0 ** -11 * want.abs() * 1.01 + 2.0 ** -25 if half else 0.0) + 2.0 ** -37 * n * most + 1e-30
                err = (got[:, h] - want).abs()
                assert (err <= tol).all(), (f"sequence {b} head {h}: {err.max().item():.3e}, {(err / tol).max().item():.2f} x the bound at "
                                            f"{np.unravel_index(int((err / tol).argmax()), tuple(err.shape))}")


@pytest.fixture(scope="module")
def ws():
    return ops.paged_workspace()


MODELS = [("f16", 14, 2, 64), ("f16", 8, 4, 64), ("f16", 28, 4, 128), ("f16", 40, 8, 128), ("f16", 16, 2, 256), ("f16", 4, 4, 256),
          ("i8", 28, 4, 128), ("i8", 8, 2, 128), ("i8", 16, 2, 256), ("i8", 16, 4, 256)]


@pytest.mark.parametrize("store,nH,nKV,hd", MODELS)
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("lens,page", [([1], 16), ([64, 65, 63], 16), ([130, 1, 7, 1000], 8), ([517, 2100], 24), ([1025] * 5, 128)])
def test_steps(ws, store, nH, nKV, hd, io, lens, page):
    """One new token each: a decode step."""
    c = Paged(store, nH, nKV, hd, lens, [1] * len(lens), page, ragged=False)
    q = c.normal(c.tokens, nH, hd).to(io)
    c.check(q, c.attend(q, ws))
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,nH,nKV,hd", MODELS)
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("lens,new,page", [([200, 77], [2, 2], 16), ([300, 5, 90], [5, 5, 1], 64), ([70, 400, 9], [0, 33, 9], 16), ([0, 130, 0], [0, 130, 0], 32),
                                           ([500, 129, 1], [120, 1, 1], 40)])
def test_chunks(ws, store, nH, nKV, hd, io, lens, new, page):
    """Drafted tokens, chunks behind earlier rows, whole prompts, and sequences without new tokens."""
    c = Paged(store, nH, nKV, hd, lens, new, page)
    q = c.normal(c.tokens, nH, hd).to(io)
    for most in (0, max(new)):
        c.check(q, c.attend(q, ws, most))
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,nH,nKV,hd", MODELS)
@pytest.mark.parametrize("lens,new,page", [([300], [300], 16), ([1500, 1, 700, 64, 2000], [900, 1, 3, 64, 300], 32), ([3000], [128], 8),
                                           ([40, 500], [90, 400], 16), ([1027, 900], [37, 19], 64), ([5000], [20], 48)])
def test_chunks_of_many_rows(ws, store, nH, nKV, hd, lens, new, page):
    """Whole prompts, chunks behind long prefixes, both beside single tokens, items of one and of two query tiles, runs that end
    inside an item; more new tokens than rows."""
    c = Paged(store, nH, nKV, hd, lens, new, page)
    q = c.normal(c.tokens, nH, hd).half()
    c.check(q, c.attend(q, ws, max(new)))
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,hd", [("f16", 64), ("f16", 128), ("f16", 256), ("i8", 128), ("i8", 256)])
@pytest.mark.parametrize("seed", range(4))
def test_random_batches(ws, store, hd, seed):
    r = np.random.default_rng(seed)
    nKV = int(r.integers(1, 5))
    nH = nKV * int(r.integers(1, 17))
    batch = int(r.integers(1, 50))
    new = [int(r.choice([0, 1, 1, 1, r.integers(2, 9), r.integers(1, 60)])) for _ in range(batch)]
    new[0] = max(1, new[0])
    lens = [n + int(r.choice([0, 1, r.integers(0, 300), r.integers(0, 2000)])) for n in new]
    c = Paged(store, nH, nKV, hd, lens, new, int(r.choice([8, 16, 32, 48, 256])), seed=seed)
    for io in (torch.float32, torch.float16):
        q = c.normal(c.tokens, nH, hd).to(io)
        c.check(q, c.attend(q, ws, int(r.choice([0, 1, max(new)]))))
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,hd,heads", [("f16", 64, 128), ("i8", 128, 128), ("f16", 256, 71)])
def test_one_kv_head_for_many_q_heads(ws, store, hd, heads):
    c = Paged(store, heads, 1, hd, [333, 20], [3, 1], 16)
    for io in (torch.float32, torch.float16):
        q = c.normal(c.tokens, heads, hd).to(io)
        c.check(q, c.attend(q, ws))


@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("store,hd", [("f16", 128), ("i8", 128), ("f16", 64)])
def test_tokens_ahead_of_the_first_row_see_nothing(ws, store, hd, io):
    """More new tokens than rows: the first of them have no row, and their outputs are zero."""
    c = Paged(store, 8, 2, hd, [3, 100], [40, 30], 16)
    q = c.normal(c.tokens, 8, hd).to(io)
    out = c.attend(q, ws)
    assert (out[:37] == 0).all()
    c.check(q, out)


def test_rows_behind_the_last_sequence_are_left(ws):
    c = Paged("f16", 8, 2, 128, [50, 60], [4, 3], 16)
    q = c.normal(12, 8, 128)
    out = torch.full_like(q, 5.0)
    ops.attn_paged(q, c.kc, c.vc, c.pages, c.lens, out, ws, starts=c.starts)
    assert (out[7:] == 5.0).all()
    c.check(q[:7], out[:7])
    k_out = torch.full((12, 2, 128), 5.0, device="cuda")
    v_out = k_out.clone()
    ops.paged_read(c.kc, c.vc, c.pages, c.lens, k_out, v_out, starts=c.starts)
    assert (k_out[7:] == 5.0).all() and (v_out[7:] == 5.0).all() and not (k_out[:7] == 5.0).any()


@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0])
@pytest.mark.parametrize("store", ["f16", "i8"])
def test_scores_of_other_sizes(ws, store, scale):
    """Flat and peaked softmax rows, and q values whose fp16 pair would run out of range without a power of two of its own."""
    c = Paged(store, 8, 2, 128, [700, 90], [2, 9], 16, seed=3)
    q = c.normal(c.tokens, 8, 128)
    c.check(q, c.attend(q, ws, scale=scale / math.sqrt(128)), scale / math.sqrt(128))
    for size in (1e-30, 1e30):
        c.check(q * size, c.attend(q * size, ws, scale=scale / math.sqrt(128) / size), scale / math.sqrt(128) / size)


def test_v_scales_that_lie_far_apart(ws):
    c = Paged("i8", 8, 2, 128, [900], [1], 16, seed=5)
    r = c.rows(0, 0, 900)
    for powers in (torch.linspace(-20, 0, 900, device="cuda"), torch.linspace(0, -20, 900, device="cuda"), torch.linspace(90, 70, 900, device="cuda")):
        c.vs.view(-1, 2)[r] = torch.exp2(powers)[:, None].expand(-1, 2).contiguous()
        q = c.normal(c.tokens, 8, 128)
        c.check(q, c.attend(q, ws))
    c.vs.view(-1, 2)[r] = 0.0
    assert (c.attend(c.normal(c.tokens, 8, 128), ws) == 0).all()


def rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([(a.double() * c - (b * s).double()).float(), (a.double() * s + (b * c).double()).float()], -1)


@pytest.mark.parametrize("store,nH,nKV,hd", MODELS)
@pytest.mark.parametrize("lens,new,page", [([1], [1], 8), ([65, 40, 7, 129], [1, 40, 0, 128], 16), ([5000, 300], [2500, 300], 32)])
@pytest.mark.parametrize("turn", [True, False])
def test_write_and_read(store, nH, nKV, hd, lens, new, page, turn):
    """Stored bytes, scales, q and what is read back, to the bit."""
    c = Paged(store, nH, nKV, hd, lens, new, page, fill=False)
    before = [t.clone() if t is not None else None for t in (c.kc, c.vc, c.ks, c.vs)]
    k, v, q = c.normal(c.tokens, nKV, hd), c.normal(c.tokens, nKV, hd), c.normal(c.tokens, nH, hd)
    k[0, 0] = 0.0                                   # a row of zeros has the scale 1
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rope_tables(max(lens), hd, 1e4))
    row = torch.cat([c.rows(b, n - m, n) for b, (n, m) in enumerate(zip(lens, new))])
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)])
    want_k, want_q = (rotated(k, cos[pos], sin[pos]), rotated(q, cos[pos], sin[pos])) if turn else (k, q)
    tables = dict(cosT=cos, sinT=sin) if turn else {}
    q16, q32, qi = torch.empty_like(q, dtype=torch.float16), torch.empty_like(q), q.clone()
    for qq, q_out in ((q, q16), (q, q32), (qi, None), (None, None)):
        ops.paged_write(k, v, c.kc, c.vc, c.pages, c.lens, starts=c.starts, ks=c.ks, vs=c.vs, q=qq, q_out=q_out, **tables)
    assert torch.equal(q16, want_q.half()) and torch.equal(q32, want_q) and torch.equal(qi, want_q)
    back = {}
    for x, pool, old, s, olds in ((want_k, c.kc, before[0], c.ks, before[2]), (v, c.vc, before[1], c.vs, before[3])):
        want = old.clone().view(-1, nKV, hd)
        if store == "i8":
            amax = x.abs().amax(-1)
            sc = torch.where(amax > 0, amax / torch.full_like(amax, 127.0), 1.0)
            q8 = torch.round(x / sc[..., None]).clamp(-128, 127)
            want[row] = q8.to(torch.int8)
            wants = olds.clone().view(-1, nKV)
            wants[row] = sc
            assert torch.equal(s.view(torch.int32), wants.view_as(s).view(torch.int32))
            back[len(back)] = q8 * sc[..., None]
        else:
            want[row] = x.half()
            back[len(back)] = x.half().float()
        assert torch.equal(pool.view(torch.int8), want.view_as(pool).view(torch.int8))
    for dt in (torch.float32, torch.float16):
        ko, vo = torch.empty((c.tokens, nKV, hd), dtype=dt, device="cuda"), torch.empty((c.tokens, nKV, hd), dtype=dt, device="cuda")
        ops.paged_read(c.kc, c.vc, c.pages, c.lens, ko, vo, starts=c.starts, ks=c.ks, vs=c.vs)
        assert torch.equal(ko, back[0].to(dt)) and torch.equal(vo, back[1].to(dt))
    assert ops.device_status() == 0


def test_rows_without_a_page_are_reported(ws):
    """Pages outside the pool, lengths past the table and positions past the rotation tables: nothing outside is touched."""
    c = Paged("f16", 8, 2, 64, [40, 64], [3, 64], 16)
    c.pages[0, 2] = 1 << 30
    bit = 32
    k = c.normal(c.tokens, 2, 64)
    kc = c.kc.clone()
    ops.paged_write(k, k, c.kc, c.vc, c.pages, c.lens, starts=c.starts)
    assert ops.device_status(raise_on_flags=False) == bit
    row = c.rows(1, 0, 64)
    kc.view(-1, 2, 64)[row] = k[3:].half()
    assert torch.equal(c.kc.view(torch.int16), kc.view(torch.int16))
    ko, vo = torch.full_like(k, 9.0), torch.full_like(k, 9.0)
    ops.paged_read(c.kc, c.vc, c.pages, c.lens, ko, vo, starts=c.starts)
    assert ops.device_status(raise_on_flags=False) == bit
    assert (ko[:3] == 0).all() and torch.equal(ko[3:], k[3:].half().float())
    q = c.normal(c.tokens, 8, 64)
    out = c.attend(q, ws)
    assert ops.device_status(raise_on_flags=False) == bit
    c.lens_h, c.new_h = c.lens_h[1:], c.new_h[1:]
    c.pages = c.pages[1:]
    c.check(q[3:], out[3:])
    # a length past the table
    lens = torch.tensor([65], dtype=torch.int32, device="cuda")
    pages = c.pages[:, :4].contiguous()
    ops.attn_paged(q[:1].contiguous(), c.kc, c.vc, pages, lens, torch.empty_like(q[:1]), ws)
    assert ops.device_status(raise_on_flags=False) == bit
    ops.paged_write(k[:1].contiguous(), k[:1].contiguous(), c.kc, c.vc, pages, lens)
    assert ops.device_status(raise_on_flags=False) == bit
    # a position past the tables
    t = torch.ones((10, 32), device="cuda")
    lens.fill_(11)
    qq = q[:1].clone()
    ops.paged_write(k[:1].contiguous(), k[:1].contiguous(), c.kc, c.vc, pages, lens, q=qq, cosT=t, sinT=t)
    assert ops.device_status(raise_on_flags=False) == bit and torch.equal(qq, q[:1])
    assert ops.device_status() == 0


def test_refusals_of_tensors(ws):
    c = Paged("i8", 8, 2, 128, [40], [2], 16, ragged=False)
    q = c.normal(2, 8, 128)
    out = torch.empty_like(q)
    go = lambda **kw: ops.attn_paged(**{**dict(q=q, kc=c.kc, vc=c.vc, pages=c.pages, lens=c.lens, out=out, ws=ws, ks=c.ks, vs=c.vs), **kw})
    go()
    for bad in (dict(out=out.half()), dict(q=q.double()), dict(vc=c.vc[:1]), dict(pages=c.pages.long()), dict(lens=c.lens.float()), dict(ks=None),
                dict(ks=c.ks[..., :1].contiguous()), dict(ws=ws.half()), dict(q=q[..., :64].contiguous()), dict(starts=c.lens), dict(kc=c.kc.float()),
                dict(out=out[:1])):
        with pytest.raises((ValueError, TypeError)):
            go(**bad)
    for bad in (dict(q=q.transpose(0, 1)), dict(pages=c.pages.cpu())):
        with pytest.raises(AssertionError):
            go(**bad)
    with pytest.raises(capi.TcError) as e:
        go(ws=ws[:-1])
    assert e.value.code == capi.TC_EWORKSPACE
    with pytest.raises(capi.TcError):
        go(q=c.normal(2, 7, 128), out=torch.empty((2, 7, 128), device="cuda"))
