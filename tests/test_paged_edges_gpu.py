"""Attention over a paged cache where its arithmetic is at its edges, against plain implementations in 64 bits."""
import math

import pytest
import torch

from tests.test_paged_gpu import Paged
from tinycoder_inference_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ws():
    return ops.paged_workspace()


def set_scales(c, pattern):
    """V's scales of every sequence from `pattern`, a function of the row numbers of a sequence (f32)."""
    for b, n in enumerate(c.lens_h):
        row = torch.arange(n, device="cuda", dtype=torch.float64)
        c.vs.view(-1, c.nKV)[c.rows(b, 0, n)] = pattern(row, n).float()[:, None].expand(-1, c.nKV).contiguous()


def where(cond, low):
    return lambda row, n: torch.where(cond(row), torch.full_like(row, low), 0.02 + 0.01 * torch.sin(row))


SCALES = {
    # tiles of 64 rows whose V scales are 0 (rows that a caller zeroed), below what a power of two of f32 holds, and subnormal: the first one,
    # every second one, a thousand rows where runs begin, the last ones
    "zero_first": where(lambda r: r < 64, 0.0), "zero_second": where(lambda r: (r // 64) % 2 == 1, 0.0), "zero_even": where(lambda r: (r // 64) % 2 == 0, 0.0),
    "zero_middle": where(lambda r: (r >= 1000) & (r < 2000), 0.0), "zero_last": where(lambda r: r >= 700, 0.0),
    "tiny_first": where(lambda r: r < 64, 2.0 ** -125), "tiny_middle": where(lambda r: (r >= 500) & (r < 1900), 2.0 ** -118),
    "subnormal_first": where(lambda r: r < 128, 1e-42), "small_first": where(lambda r: r < 192, 2.0 ** -70),
    "up": lambda r, n: torch.exp2(torch.linspace(-20, 0, n, device="cuda", dtype=torch.float64)),
    "down": lambda r, n: torch.exp2(torch.linspace(0, -20, n, device="cuda", dtype=torch.float64)),
    "far_up": lambda r, n: torch.exp2(torch.linspace(-125, 0, n, device="cuda", dtype=torch.float64)),
    "far_down": lambda r, n: torch.exp2(torch.linspace(0, -125, n, device="cuda", dtype=torch.float64)),
}


@pytest.mark.parametrize("pattern", SCALES)
@pytest.mark.parametrize("nH,nKV,hd", [(8, 2, 128), (14, 1, 128), (16, 2, 256)])
@pytest.mark.parametrize("io", [torch.float16, torch.float32])
def test_v_scales_of_any_size(ws, nH, nKV, hd, io, pattern):
    """Single tokens, drafts, and chunks of one and of two query tiles; items in one run and in many."""
    for lens, new in (([900, 70], [1, 1]), ([1300, 128], [3, 2]), ([2600, 300], [20, 13]), ([2100, 130], [90, 130]), ([5000], [17])):
        c = Paged("i8", nH, nKV, hd, lens, new, 16, seed=len(lens) + new[0])
        set_scales(c, SCALES[pattern])
        q = c.normal(c.tokens, nH, hd).to(io)
        c.check(q, c.attend(q, ws, max(new)))
    assert ops.device_status() == 0


@pytest.mark.parametrize("scale", [0.0, 1e-42, 2.0 ** -126, 2.0 ** -100])
@pytest.mark.parametrize("nH,nKV,hd", [(8, 2, 128), (16, 2, 256)])
def test_all_v_scales_tiny_or_zero(ws, nH, nKV, hd, scale):
    """What an fp16 result cannot show is 0, and so is 0."""
    for new in (1, 5, 20, 100):
        c = Paged("i8", nH, nKV, hd, [1000, 130], [new, 1], 32, seed=new)
        set_scales(c, lambda row, n: torch.full_like(row, scale))
        q = c.normal(c.tokens, nH, hd).half()
        assert (c.attend(q, ws, new) == 0).all()
    assert ops.device_status() == 0


def sink(store, nH, nKV, hd, lens, new, drop, seed):
    """Rows whose weight is 2^-drop of the first row's, which holds V = 0: the small weights are the whole result.  Every q head
    has a factor of its own near 1, so the weights' roundings differ from head to head and agree within one."""
    c = Paged(store, nH, nKV, hd, lens, new, 16, seed=seed)
    q = torch.zeros((c.tokens, nH, hd), device="cuda")
    q[:, :, 0] = math.sqrt(hd) * math.log(2.0) * (1.0 + torch.arange(nH, device="cuda") / (64.0 * nH))
    for b, n in enumerate(lens):
        r = c.rows(b, 0, n)
        k, v = torch.zeros((n, nKV, hd), device="cuda"), c.normal(n, nKV, hd).abs() + 0.5
        k[1:, :, 0] = -drop
        v[0] = 0.0
        if store == "i8":
            c.kc.view(-1, nKV, hd)[r] = (k * 4).to(torch.int8)
            c.ks.view(-1, nKV)[r] = 0.25
            c.vc.view(-1, nKV, hd)[r] = (v * 20).round().clamp(0, 127).to(torch.int8)
            c.vs.view(-1, nKV)[r] = 0.04
        else:
            c.kc.view(-1, nKV, hd)[r] = k.half()
            c.vc.view(-1, nKV, hd)[r] = v.half()
    return c, q


@pytest.mark.parametrize("drop", [12, 20, 24])
@pytest.mark.parametrize("store,nH,nKV,hd", [("f16", 14, 2, 64), ("f16", 28, 4, 128), ("f16", 16, 2, 256), ("i8", 28, 4, 128), ("i8", 16, 2, 256)])
def test_f32_results_of_small_weights(ws, store, nH, nKV, hd, drop):
    """A row of large weight that holds nothing, and many of small ones: an f32 result stays one."""
    for lens, new in (([300], [1]), ([100, 1000], [1, 1]), ([260, 90], [3, 2]), ([700], [40])):
        c, q = sink(store, nH, nKV, hd, lens, new, drop, seed=drop)
        c.check(q, c.attend(q, ws, max(new)))
    assert ops.device_status() == 0


@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0])
@pytest.mark.parametrize("store,nH,nKV,hd", [("f16", 14, 2, 64), ("f16", 8, 2, 128), ("f16", 16, 2, 256), ("i8", 8, 2, 128), ("i8", 16, 2, 256)])
def test_flat_and_peaked_rows_of_fp16_queries(ws, store, nH, nKV, hd, scale):
    """Scores of other sizes, through the forms for few and for many query rows."""
    for lens, new in (([700, 90], [1, 1]), ([700, 90], [2, 9]), ([2500, 128], [20, 40]), ([1900, 300], [150, 300])):
        c = Paged(store, nH, nKV, hd, lens, new, 16, seed=3)
        q = c.normal(c.tokens, nH, hd).half()
        for most in (max(new), 0):
            c.check(q, c.attend(q, ws, most, scale=scale / math.sqrt(hd)), scale / math.sqrt(hd))
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,hd", [("f16", 64), ("f16", 128), ("f16", 256), ("i8", 128), ("i8", 256)])
@pytest.mark.parametrize("io", [torch.float16, torch.float32])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_rise_or_fall_along_a_sequence(ws, store, hd, io, rising):
    """Every tile moves the running maximum, or none behind the first one does."""
    for lens, new in (([2000], [1]), ([1500, 400], [4, 4]), ([1300, 500], [130, 30])):
        c = Paged(store, 8, 2, hd, lens, new, 16, seed=7)
        q = c.normal(c.tokens, 8, hd).to(io)
        q[:, :, 0] = 0.5 * math.sqrt(hd)
        for b, n in enumerate(lens):
            r = c.rows(b, 0, n)
            ramp = torch.linspace(-30.0, 30.0, n, device="cuda") * (1.0 if rising else -1.0)
            if store == "i8":
                c.ks.view(-1, 2)[r] = 0.25
                c.kc.view(-1, 2, hd)[r] = (c.normal(n, 2, hd) * 4).round().clamp(-8, 8).to(torch.int8)
                c.kc.view(-1, 2, hd)[r, :, 0] = (ramp * 4).round().to(torch.int8)[:, None]
            else:
                c.kc.view(-1, 2, hd)[r, :, 0] = ramp.half()[:, None]
        c.check(q, c.attend(q, ws, max(new)))
    assert ops.device_status() == 0


class Without(Paged):
    """A cache whose first sequence has a table entry outside the pool and whose second one has a length past its table."""

    def spoil(self, page):
        self.pages[0, self.lens_h[0] // self.page // 2] = page
        self.lens[1] = self.pages.shape[1] * self.page + 5


@pytest.mark.parametrize("store,hd", [("f16", 64), ("f16", 128), ("f16", 256), ("i8", 128), ("i8", 256)])
@pytest.mark.parametrize("io", [torch.float16, torch.float32])
@pytest.mark.parametrize("new", [1, 3, 40, 200])
def test_bad_tables_touch_nothing_else(ws, store, hd, io, new):
    """Entries that name no page and lengths past the table are reported; other sequences' results and tokens of no sequence are as they
    were, whichever form takes the call, K and V and the scales of an int8 row."""
    for page in (1 << 30, -1, -2 ** 31):
        c = Without(store, 8, 2, hd, [900, 700, 800, 450], [new] * 4, 16, seed=new)
        q = torch.zeros((c.tokens + 5, 8, hd), device="cuda", dtype=io)
        q[:c.tokens] = c.normal(c.tokens, 8, hd).to(io)
        out = torch.full_like(q, 5.0)
        c.spoil(page)
        ops.attn_paged(q, c.kc, c.vc, c.pages, c.lens, out, ws, starts=c.starts, max_tokens=new, ks=c.ks, vs=c.vs)
        assert ops.device_status(raise_on_flags=False) == 32
        assert (out[c.tokens:] == 5.0).all()
        c.lens_h, c.new_h, c.pages = c.lens_h[2:], c.new_h[2:], c.pages[2:]
        c.check(q[2 * new:4 * new], out[2 * new:4 * new])
        assert ops.device_status() == 0


@pytest.mark.parametrize("store", ["f16", "i8"])
def test_bad_tables_of_the_writer_and_the_reader(store):
    """Rows without a page are not stored and read back as zeros; all others are what they are without them."""
    nKV, hd, new = 2, 128, 100
    c = Without(store, 8, nKV, hd, [300, 300, 300], [new] * 3, 16, seed=1, fill=False)
    k, v = c.normal(c.tokens, nKV, hd), c.normal(c.tokens, nKV, hd)
    c.pages[0, 300 // 16 - 1] = -1           # rows 272 .. 287 of the first sequence
    c.lens[1] = c.pages.shape[1] * 16 + 5    # the second one's last five rows lie past the table
    pools = [t.clone() if t is not None else None for t in (c.kc, c.vc, c.ks, c.vs)]
    ops.paged_write(k, v, c.kc, c.vc, c.pages, c.lens, starts=c.starts, ks=c.ks, vs=c.vs)
    assert ops.device_status(raise_on_flags=False) == 32
    ko, vo = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    ops.paged_read(c.kc, c.vc, c.pages, c.lens, ko, vo, starts=c.starts, ks=c.ks, vs=c.vs)
    assert ops.device_status(raise_on_flags=False) == 32
    lost = torch.zeros(c.tokens, dtype=torch.bool, device="cuda")
    lost[72:88] = True                       # tokens at rows 272 .. 287 (tokens 0 .. 99 are rows 200 .. 299)
    lost[195:200] = True
    for got, x, pool, old in ((ko, k, c.kc, pools[0]), (vo, v, c.vc, pools[1])):
        assert (got[lost] == 0).all()
        if store == "f16":
            assert torch.equal(got[~lost], x[~lost].half().float())
        else:  # half a step of a row's largest / 127
            assert ((got - x)[~lost].abs() <= x[~lost].abs().amax(-1, keepdim=True) / 127 * 0.5001).all()
        # stored rows: those that were not lost, no others
        changed = (pool.view(-1, nKV * hd) != old.view(-1, nKV * hd)).any(-1) & ~(torch.isnan(pool.view(-1, nKV * hd).float()).all(-1))
        assert changed.sum().item() == (~lost).sum().item()


@pytest.mark.parametrize("store,io", [("f16", torch.float32), ("f16", torch.float16), ("i8", torch.float32), ("i8", torch.float16)])
def test_values_of_tokens_between_tokens_of_no_sequence(ws, store, io):
    """`starts` that begin behind the first token and end ahead of the last one, with the items of a long prompt."""
    tokens, hd = 4000, 128
    c = Paged(store, 8, 4, hd, [tokens, 40], [tokens - 9, 3], 16, seed=6)
    c.starts += 4
    q = c.normal(tokens, 8, hd).to(io)
    out = torch.full_like(q, 5.0)
    ops.attn_paged(q, c.kc, c.vc, c.pages, c.lens, out, ws, starts=c.starts, ks=c.ks, vs=c.vs)
    assert (out[:4] == 5).all() and (out[tokens - 2:] == 5).all()
    c.check(q[4:tokens - 2], out[4:tokens - 2])
    assert ops.device_status() == 0


def off(x):
    """The same values at an address that is a multiple of 16 bytes and not of 32."""
    n = 16 // x.element_size()
    flat = torch.empty(x.numel() + 3 * n, dtype=x.dtype, device="cuda")
    at = n if flat.data_ptr() % 32 == 0 else 2 * n
    y = flat[at:at + x.numel()].view(x.shape)
    y.copy_(x)
    assert y.data_ptr() % 32 == 16
    return y


@pytest.mark.parametrize("store,hd", [("f16", 64), ("f16", 128), ("f16", 256), ("i8", 128), ("i8", 256)])
@pytest.mark.parametrize("io", [torch.float16, torch.float32])
def test_arrays_at_16_bytes(ws, store, hd, io):
    """Every array at an odd multiple of 16 bytes, through every form: the same bits as at wider alignments."""
    other = off(ws)
    for lens, new in (([300, 65], [1, 1]), ([900, 65], [3, 2]), ([1200, 65], [40, 60]), ([1500, 400], [200, 400])):
        c = Paged(store, 8, 2, hd, lens, new, 16, seed=new[0])
        q = c.normal(c.tokens, 8, hd).to(io)
        k, v, cos = c.normal(c.tokens, 2, hd), c.normal(c.tokens, 2, hd), c.normal(max(lens), hd // 2)
        results = []
        for place in (lambda t: t, off):
            kc, vc, qq, out, q32, q_out = (place(t) for t in (c.kc.clone(), c.vc.clone(), q, torch.zeros_like(q), q.float(), torch.zeros_like(q)))
            ks, vs = (t.clone() if t is not None else None for t in (c.ks, c.vs))
            w = ws if place is not off else other
            ops.attn_paged(qq, kc, vc, c.pages, c.lens, out, w, starts=c.starts, max_tokens=max(new), ks=ks, vs=vs)
            ops.paged_write(place(k), place(v), kc, vc, c.pages, c.lens, starts=c.starts, ks=ks, vs=vs, q=q32, q_out=q_out, cosT=place(cos), sinT=place(cos))
            ko, vo = place(torch.zeros_like(k).to(io)), place(torch.zeros_like(k).to(io))
            ops.paged_read(kc, vc, c.pages, c.lens, ko, vo, starts=c.starts, ks=ks, vs=vs)
            results.append([out, q_out, ko, vo])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        c.check(q, results[1][0])
    assert ops.device_status() == 0


@pytest.mark.parametrize("io", [torch.float16, torch.float32])
@pytest.mark.parametrize("store", ["f16", "i8"])
def test_a_page_of_two_sequences(ws, store, io):
    """Sequences that share the pages of a common beginning (and one that has a page twice): each as if they were its own."""
    for new in (1, 3, 40, 150):
        c = Paged(store, 8, 2, 128, [700, 700, 700], [new] * 3, 32, seed=new)
        c.pages[1, :15] = c.pages[0, :15]
        c.pages[2, 3] = c.pages[2, 9]
        q = c.normal(c.tokens, 8, 128).to(io)
        c.check(q, c.attend(q, ws, new))
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,io", [("f16", torch.float16), ("i8", torch.float16), ("i8", torch.float32)])
def test_calls_of_one_workspace_behind_each_other(store, io):
    """Calls of different forms and sizes in a row, nothing between them: each takes the workspace as the one before left it."""
    w = ops.paged_workspace()
    calls = []
    for seed, (lens, new) in enumerate((([3000, 90], [1, 1]), ([2500], [300]), ([40, 3000, 7], [3, 2, 7]), ([1], [1]), ([2000] * 40, [1] * 40), ([1500, 900], [700, 1]))):
        c = Paged(store, 28, 4, 128, lens, new, 16, seed=seed)
        q = c.normal(c.tokens, 28, 128).to(io)
        calls.append((c, q, torch.full_like(q, 9.0)))
    torch.cuda.synchronize()
    for _ in range(3):
        for c, q, out in calls:
            ops.attn_paged(q, c.kc, c.vc, c.pages, c.lens, out, w, starts=c.starts, max_tokens=max(c.new_h), ks=c.ks, vs=c.vs)
    for c, q, out in calls:
        c.check(q, out)
    assert ops.device_status() == 0
