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
