"""The paged calls as a serving program makes them: one after another, captured and replayed, on several streams, with the sizes
at the ends of their ranges."""
import math

import numpy as np
import pytest
import torch

from tests.test_paged_gpu import Paged, rotated
from tinycoder_inference_b200 import capi, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ws():
    return ops.paged_workspace()


@pytest.mark.parametrize("store,io", [("f16", torch.float32), ("f16", torch.float16), ("i8", torch.float32), ("i8", torch.float16)])
def test_a_session_from_prompt_to_tokens_and_back(ws, store, io):
    """Two prompts are written and attended to, then four steps of one token each; every output against 64 bits over what the
    store holds; in the end the rows come back."""
    nH, nKV, hd, page = 14, 2, 128, 16
    prompts, steps = [100, 37], 4
    c = Paged(store, nH, nKV, hd, [n + steps for n in prompts], [0, 0], page, fill=False)
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rope_tables(256, hd, 1e6))
    told = {0: [], 1: []}
    for i in range(steps + 1):
        new = prompts if i == 0 else [1, 1]
        lens = [n + i for n in prompts]
        starts = np.concatenate([[0], np.cumsum(new)])
        c.starts = torch.tensor(starts, dtype=torch.int32, device="cuda") if i == 0 else None
        c.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        c.lens_h, c.new_h = lens, new
        t = int(starts[-1])
        q, k, v = c.normal(t, nH, hd), c.normal(t, nKV, hd), c.normal(t, nKV, hd)
        pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)])
        want = rotated(q, cos[pos], sin[pos])
        q_out = torch.empty_like(q, dtype=io)
        ops.paged_write(k, v, c.kc, c.vc, c.pages, c.lens, starts=c.starts, ks=c.ks, vs=c.vs, q=q, q_out=q_out, cosT=cos, sinT=sin)
        assert torch.equal(q_out, want.to(io))
        c.check(q_out, c.attend(q_out, ws, max(new)))
        for b in range(2):
            told[b].append(v[starts[b]:starts[b + 1]])
    starts = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device="cuda")
    ko = torch.empty((sum(lens), nKV, hd), device="cuda")
    vo = torch.empty_like(ko)
    ops.paged_read(c.kc, c.vc, c.pages, c.lens, ko, vo, starts=starts, ks=c.ks, vs=c.vs)
    told = torch.cat([torch.cat(told[0]), torch.cat(told[1])])
    if store == "f16":
        assert torch.equal(vo, told.half().float())
    else:  # half a step of a row's largest / 127
        assert ((vo - told).abs() <= told.abs().amax(-1, keepdim=True) / 127 * 0.5001).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,io,lens", [("i8", torch.float32, [70, 300]), ("f16", torch.float16, [1, 900]), ("i8", torch.float16, [500, 40])])
def test_a_captured_step_follows_its_tables(store, io, lens):
    """Lengths, pages and new rows may change between replays; two graphs may share a workspace as long as they follow each other."""
    nH, nKV, hd, page, room = 28, 4, 128, 16, 1152   # (more than any length below)
    ws = ops.paged_workspace()
    ws.fill_(float("nan"))                   # what it holds does not matter
    c = Paged(store, nH, nKV, hd, [room, room], [1, 1], page, ragged=False)
    q, k, v = (c.normal(2, n, hd) for n in (nH, nKV, nKV))
    qo, out = torch.empty_like(q, dtype=io), torch.empty_like(q, dtype=io)
    c.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def step():
        ops.paged_write(k, v, c.kc, c.vc, c.pages, c.lens, ks=c.ks, vs=c.vs, q=q, q_out=qo)
        ops.attn_paged(qo, c.kc, c.vc, c.pages, c.lens, out, ws, ks=c.ks, vs=c.vs)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i in range(6):
        now = [n + 37 * i for n in lens]
        c.lens.copy_(torch.tensor(now, dtype=torch.int32))
        c.pages.copy_(c.pages.flip(0))
        for t in (q, k, v):
            t.copy_(c.normal(*t.shape))
        graphs[i % 2].replay()
        c.lens_h, c.new_h = now, [1, 1]
        c.check(qo, out)
        first = out.clone()
        graphs[(i + 1) % 2].replay()          # the same again, to the bit
        assert torch.equal(out, first)
    assert ops.device_status() == 0


def test_streams_with_workspaces_of_their_own():
    cases = []
    for i in range(3):
        c = Paged(("f16", "i8", "f16")[i], 8, 2, 128, [3000 + 100 * i, 77], [1, 60], 16, seed=i)
        io = (torch.float16, torch.float16, torch.float32)[i]
        cases.append((c, c.normal(c.tokens, 8, 128).to(io), ops.paged_workspace(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [None] * 3
    for _ in range(5):
        for i, (c, q, w, s) in enumerate(cases):
            with torch.cuda.stream(s):
                outs[i] = c.attend(q, w)
    torch.cuda.synchronize()
    for (c, q, _, _), out in zip(cases, outs):
        c.check(q, out)
    assert ops.device_status() == 0


@pytest.mark.parametrize("store,io", [("i8", torch.float32), ("f16", torch.float16)])
def test_the_same_call_gives_the_same_bits(ws, store, io):
    c = Paged(store, 28, 4, 128, [4000, 900, 65, 1], [1, 200, 3, 1], 16, seed=9)
    q = c.normal(c.tokens, 28, 128).to(io)
    first = c.attend(q, ws)
    for _ in range(5):
        assert torch.equal(c.attend(q, ws), first)


@pytest.mark.parametrize("store,hd,io,new", [("f16", 64, torch.float32, None), ("f16", 128, torch.float32, None), ("f16", 128, torch.float16, 4),
                                             ("f16", 128, torch.float32, 2), ("f16", 64, torch.float16, 1), ("i8", 128, torch.float16, 2),
                                             ("i8", 256, torch.float32, 3), ("f16", 128, torch.float16, None), ("i8", 128, torch.float16, None)])
def test_a_stage_is_not_handed_back_under_its_readers(ws, store, hd, io, new):
    """Uneven sequences whose blocks end their items at different times, a hundred times over: a tile that is written under the
    slowest warp's last loads shows as a few weights that differ from run to run."""
    if new is None:
        c = Paged(store, 21, 3, hd, [220, 345, 2910, 110, 322, 449], [204, 345, 279, 110, 322, 362], 128)
    else:
        c = Paged(store, 21, 3, hd, [220, 345, 2910, 1110, 322, 4449] * 3, [new] * 18, 128, ragged=False)
    q = c.normal(c.tokens, 21, hd).to(io)
    first = c.attend(q, ws)
    c.check(q, first)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(100):
        differ += (c.attend(q, ws) != first).any()
    assert differ.item() == 0


@pytest.mark.parametrize("batch", [33, 129, 300])
@pytest.mark.parametrize("store,io", [("i8", torch.float16), ("f16", torch.float32)])
def test_many_sequences(ws, batch, store, io):
    r = np.random.default_rng(batch)
    new = [int(r.choice([0, 1, 1, 2, 40])) for _ in range(batch)]
    new[-1] = 1
    lens = [n + int(r.integers(0, 200)) for n in new]
    c = Paged(store, 4, 2, 128, lens, new, 16, seed=batch)
    q = c.normal(c.tokens, 4, 128).to(io)
    c.check(q, c.attend(q, ws, 40))


@pytest.mark.parametrize("store,hd,io", [("i8", 128, torch.float32), ("f16", 64, torch.float32), ("f16", 128, torch.float16), ("i8", 256, torch.float16)])
def test_a_long_sequence(ws, store, hd, io):
    """100000 rows: long sums keep f32 accuracy, splits and merges of many blocks."""
    for new in (1, 5, 40):
        c = Paged(store, 4, 1, hd, [100000], [new], 128, seed=new)
        q = c.normal(new, 4, hd).to(io)
        c.check(q, c.attend(q, ws))


@pytest.mark.parametrize("io", [torch.float32, torch.float16])
def test_pages_far_into_a_pool(ws, io):
    """Offsets past 32 bits: rows in the last pages of pools of 5 GB."""
    nKV, hd, page, n = 4, 128, 64, 300
    num = (5 << 30) // (page * nKV * hd)
    for store in ("i8", "f16"):
        pages_n = num if store == "i8" else num // 2
        kc = torch.empty((pages_n, page, nKV, hd), dtype=torch.int8 if store == "i8" else torch.float16, device="cuda")
        vc = torch.empty_like(kc)
        ks, vs = (torch.empty((pages_n, page, nKV), device="cuda") for _ in range(2)) if store == "i8" else (None, None)
        c = Paged(store, 8, nKV, hd, [n], [n], page, seed=1, fill=False)
        c.kc, c.vc, c.ks, c.vs, c.num = kc, vc, ks, vs, pages_n
        per = -(-n // page)
        c.pages = torch.arange(pages_n - 1, pages_n - 1 - per, -1, dtype=torch.int32, device="cuda")[None].contiguous()
        k, v, q = c.normal(n, nKV, hd), c.normal(n, nKV, hd), c.normal(n, 8, hd)
        ops.paged_write(k, v, kc, vc, c.pages, c.lens, ks=ks, vs=vs)
        ko, vo = torch.empty_like(k), torch.empty_like(v)
        ops.paged_read(kc, vc, c.pages, c.lens, ko, vo, ks=ks, vs=vs)
        if store == "f16":
            assert torch.equal(ko, k.half().float()) and torch.equal(vo, v.half().float())
        else:  # half a step of a row's largest / 127
            assert ((vo - v).abs() <= v.abs().amax(-1, keepdim=True) / 127 * 0.5001).all()
        q = q.to(io)
        c.check(q, c.attend(q, ws))
        del kc, vc, ks, vs, c
        torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens", [12, 4000])
def test_tokens_of_no_sequence_are_left(ws, tokens):
    """`starts` may begin behind the first token and end ahead of the last one."""
    nKV, hd = 4, 128
    c = Paged("f16", 8, nKV, hd, [tokens, 40], [tokens - 9, 3], 16, seed=6)
    c.starts += 4
    new = tokens - 6
    q, k = c.normal(tokens, 8, hd), c.normal(tokens, nKV, hd)
    out, kc = torch.full_like(q, 5.0), c.kc.clone()
    ops.paged_write(k, k, c.kc, c.vc, c.pages, c.lens, starts=c.starts, q=q, q_out=out)
    row = torch.cat([c.rows(b, n - m, n) for b, (n, m) in enumerate(zip(c.lens_h, c.new_h))])
    kc.view(-1, nKV, hd)[row] = k[4:4 + new].half()
    assert torch.equal(c.kc.view(torch.int16), kc.view(torch.int16))
    for t, want in ((out, q),):
        assert torch.equal(t[4:4 + new], want[4:4 + new]) and (t[:4] == 5).all() and (t[4 + new:] == 5).all()
    ko = torch.full_like(k, 5.0)
    vo = ko.clone()
    ops.paged_read(c.kc, c.vc, c.pages, c.lens, ko, vo, starts=c.starts)
    assert torch.equal(vo[4:4 + new], k[4:4 + new].half().float()) and (vo[:4] == 5).all() and (vo[4 + new:] == 5).all()
    for io in (torch.float32, torch.float16):
        out = torch.full((tokens, 8, hd), 5.0, dtype=io, device="cuda")
        ops.attn_paged(q.to(io), c.kc, c.vc, c.pages, c.lens, out, ws, starts=c.starts)
        assert (out[:4] == 5).all() and (out[4 + new:] == 5).all()
        if tokens < 100:
            c.check(q[4:4 + new].to(io), out[4:4 + new])
    assert ops.device_status() == 0


@pytest.mark.parametrize("max_tokens", [0, 1, 7, 1000])
def test_the_hint_does_not_change_what_is_computed(ws, max_tokens):
    for store, io in (("f16", torch.float16), ("i8", torch.float16), ("f16", torch.float32), ("i8", torch.float32)):
        c = Paged(store, 14, 2, 128, [400, 33, 90], [90, 1, 5], 16, seed=2)
        q = c.normal(c.tokens, 14, 128).to(io)
        c.check(q, c.attend(q, ws, max_tokens))


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("new", [1, 20, 300])
def test_what_lies_behind_a_sequence_does_not_matter(ws, store, io, new):
    """Infinities and NaN in the rest of a page and in other pages, lengths that end inside a tile and a page."""
    c = Paged(store, 8, 2, 128, [300 + new, 3 + new], [new, new], 64, ragged=False, seed=4)
    q = c.normal(c.tokens, 8, 128).to(io)
    first = c.attend(q, ws)
    c.check(q, first)
    flat = torch.ones(c.num * 64, dtype=torch.bool, device="cuda")
    for b, n in enumerate(c.lens_h):
        flat[c.rows(b, 0, n)] = False
    for pool, scale in ((c.kc, c.ks), (c.vc, c.vs)):
        if store == "i8":
            pool.view(-1, 2, 128)[flat] = 127
            scale.view(-1, 2)[flat] = float("inf")
        else:
            pool.view(-1, 2, 128)[flat] = float("inf")
    assert torch.equal(c.attend(q, ws), first)


def test_wrong_devices_and_null_tensors(ws):
    c = Paged("f16", 8, 2, 64, [40], [1], 16, ragged=False)
    q = c.normal(1, 8, 64)
    with pytest.raises((TypeError, ValueError, AssertionError)):
        ops.attn_paged(q, c.kc, None, c.pages, c.lens, torch.empty_like(q), ws)
    with pytest.raises((TypeError, ValueError, AssertionError)):
        ops.attn_paged(q.cpu(), c.kc, c.vc, c.pages, c.lens, torch.empty_like(q), ws)
    with pytest.raises(capi.TcError):
        ops.attn_paged(q, c.kc, c.vc, c.pages, c.lens, torch.empty_like(q), ws, invSqrt=-1.0)
    ops.attn_paged(q[:0].contiguous(), c.kc, c.vc, c.pages, c.lens, q[:0].contiguous(), ws)     # no tokens: nothing to do
    assert math.isfinite(q.sum().item()) and ops.device_status() == 0
