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
