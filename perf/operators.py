"""The paged K/V cache and the attention over it, as a serving program drives them.

Sessions share one pool of pages ([page][row][kv head][head_dim], fp16 or int8 with a scale per row and
kv head); a table gives every session its pages, `lens` its rows, `starts` the new tokens of a ragged
batch.  Three operators, all through `tinycoder_inference_b200.ops`:

  write   the new tokens' K and V (f32) into the pages, rotated on the way, with q rotated to the type
          that attention takes.  Over an int8 store the rows are read back, as a prompt that attends to
          what the store holds does
  read    the rows of every session back into contiguous f32 / fp16 rows (a session that leaves the pool)
  attend  the new tokens' attention over their sessions' rows: one token each (a decode step), a few
          (drafted tokens), chunks of prompts behind earlier rows, whole prompts, and mixtures
"""
from __future__ import annotations

import math
import random

import torch

own = False

# (q heads, kv heads) per head_dim: the shapes of the benchmark, the planner's models and the tests
SHAPES = {64: [(14, 2), (8, 4)], 128: [(28, 4), (12, 2), (40, 8), (8, 2)], 256: [(16, 2), (16, 4), (8, 4)]}
PAGES = [16, 32, 64, 128]
ROPE_THETA = 1e6
TYPES = {"f16": torch.float16, "f32": torch.float32}


def _case(name, op, store, heads, kv_heads, head_dim, batch, past, new, page, io, mix, **more):
    """past, new: ranges of the rows that a session has and of the tokens that it brings."""
    c = {"name": name, "op": op, "store": store, "q_heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "batch": batch, "past_lo": past[0], "past_hi": past[1], "new_lo": new[0], "new_hi": new[1], "page": page,
         "io": io, "mix": mix}
    c.update(more)
    return c


def listed():
    return [
        # a decode step of 64 sessions puts its tokens away: launches and latency
        _case("write_step_i8", "write", "i8", 28, 4, 128, 64, (0, 4095), (1, 1), 16, "f16", 1),
        # five prompts of a 32B-shaped model enter the fp16 cache in one call
        _case("write_prompts_f16", "write", "f16", 40, 8, 128, 5, (0, 0), (300, 2500), 32, "f16", 2),
        # sixteen sessions leave an int8 pool as fp16 rows
        _case("read_i8", "read", "i8", 28, 4, 128, 16, (0, 0), (500, 8000), 64, "f16", 3),
        # one short session of a small model, to the f32 rows of the contiguous store
        _case("read_f16_small", "read", "f16", 14, 2, 64, 1, (0, 0), (2047, 2047), 16, "f32", 4),
        # a token of a single user's session, f32 results: the smallest attention call
        _case("step_i8_single", "attend", "i8", 28, 4, 128, 1, (8190, 8190), (1, 1), 16, "f32", 5),
        # a decode step of 64 sessions of a 32B-shaped model on the fp16 store
        _case("step_f16_batch", "attend", "f16", 40, 8, 128, 64, (511, 8191), (1, 1), 16, "f16", 6),
        # a serving mix on the int8 store, contexts up to 32768
        _case("step_i8_ragged", "attend", "i8", 28, 4, 128, 32, (511, 32767), (1, 1), 64, "f16", 7),
        # drafted tokens of a gated model go through the target at once
        _case("draft_i8_gated", "attend", "i8", 16, 2, 256, 16, (1000, 6000), (2, 6), 32, "f32", 8),
        # short chunks of a small model whose caller wants f32 results
        _case("chunk_f16_exact", "attend", "f16", 14, 2, 64, 3, (100, 900), (37, 200), 16, "f32", 9),
        # chunks of prompts and single tokens of other sessions in one call
        _case("mixed_f16", "attend", "f16", 28, 4, 128, 8, (0, 8000), (1, 512), 16, "f16", 10),
        # 512-token chunks of two long prompts over the int8 store
        _case("chunk_i8_long", "attend", "i8", 28, 4, 128, 2, (3500, 16000), (512, 512), 64, "f16", 11),
        # four whole prompts of a 7B-shaped model: the largest call
        _case("prompts_f16", "attend", "f16", 28, 4, 128, 4, (0, 0), (1500, 4096), 128, "f16", 12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _padded(case):
    """(cache values, scores x head_dim) that a padded batch of the case has."""
    rows = case["past_hi"] + case["new_hi"]
    cache = case["batch"] * rows * case["kv_heads"] * case["head_dim"]
    return cache, case["batch"] * case["new_hi"] * rows * case["q_heads"] * case["head_dim"]


def draw(rng):
    most = [max(x) for x in zip(*(_padded(c) for c in listed() if c["op"] == "attend"))]
    while True:
        op = rng.choice(["write", "read", "attend", "attend", "attend"])
        store = rng.choice(["f16", "i8"])
        head_dim = rng.choice([128, 128, 256] if store == "i8" else [64, 128, 256])
        heads, kv_heads = rng.choice(SHAPES[head_dim])
        io = rng.choice(["f16", "f16", "f32"])
        batch, past, page = _log(rng, 1, 64), _log(rng, 1, 32768) - 1, rng.choice(PAGES)
        if op == "read":
            past, new = 0, _log(rng, 1, 16384)
        elif op == "write":
            new = _log(rng, 1, 4096)
        else:  # f32 results: steps, drafts and short chunks
            new = rng.choice([1, _log(rng, 2, 16), _log(rng, 16, 512 if io == "f32" else 4096)])
        lo = rng.choice([1, new, max(1, new // 2)])
        case = _case("", op, store, heads, kv_heads, head_dim, batch, (rng.choice([0, past // 8, past]), past), (lo, new),
                     page, io, rng.randrange(1 << 20))
        del case["name"]
        cache, scores = _padded(case)
        if op == "attend" and cache <= most[0] and scores <= most[1] // (8 if io == "f32" else 1):
            return case
        if op != "attend" and case["batch"] * new * heads * head_dim <= 48_000_000 and cache <= most[0]:
            return case


def _lengths(case):
    """(rows of every session, its new tokens among them; new tokens)."""
    r = random.Random(case["mix"])
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    return [r.randint(case["past_lo"], case["past_hi"]) + n for n in new], new


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    lens, new = _lengths(case)
    R, nH, nKV, hd, op = case["page"], case["q_heads"], case["kv_heads"], case["head_dim"], case["op"]
    tokens, per_seq = sum(new), -(-max(lens) // R)
    used = [-(-n // R) for n in lens]
    num = sum(used) + 3                      # a pool has pages that nobody holds
    order = torch.randperm(num, device=dev, generator=g).to(torch.int32)
    pages = torch.full((case["batch"], per_seq), num, dtype=torch.int32, device=dev)  # past a session's pages: no page
    at = 0
    for b, n in enumerate(used):
        pages[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = {"case": dict(case), "pages": pages, "lens": torch.tensor(lens, dtype=torch.int32, device=dev),
         "starts": torch.tensor(starts, dtype=torch.int32, device=dev) if case["new_lo"] < case["new_hi"] else None,
         "tokens": tokens, "max_new": max(new), "max_len": max(lens), "ks": None, "vs": None}

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, device=dev, generator=g, dtype=dtype)

    shape = (num, R, nKV, hd)
    for name, scale in (("k", "ks"), ("v", "vs")):
        if op == "write":
            s[name + "c"] = torch.zeros(shape, dtype=torch.int8 if case["store"] == "i8" else torch.float16, device=dev)
        elif case["store"] == "i8":
            s[name + "c"] = (normal(*shape, dtype=torch.float16) * 42).round().clamp(-127, 127).to(torch.int8)
        else:
            s[name + "c"] = normal(*shape, dtype=torch.float16)
        if case["store"] == "i8":
            # a row's largest of 127 values of deviation 1 is near 3
            s[scale] = torch.zeros(shape[:3], device=dev) if op == "write" else 0.024 * (1 + 0.2 * normal(*shape[:3])).clamp(0.2, 3)
    if op == "write":
        s["q"], s["k"], s["v"] = normal(tokens, nH, hd), normal(tokens, nKV, hd), normal(tokens, nKV, hd)
        s["q_out"] = torch.zeros((tokens, nH, hd), dtype=TYPES[case["io"]], device=dev)
        angle = torch.arange(max(lens), dtype=torch.float64, device=dev)[:, None] * (
            ROPE_THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=dev) / hd))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if op == "attend":
        s["q"] = normal(tokens, nH, hd).to(TYPES[case["io"]])
        s["out"] = torch.zeros_like(s["q"])
    if op == "read" or (op == "write" and case["store"] == "i8"):
        rows = (tokens, nKV, hd)
        back = torch.float16 if op == "write" else TYPES[case["io"]]
        s["k_out"], s["v_out"] = torch.zeros(rows, dtype=back, device=dev), torch.zeros(rows, dtype=back, device=dev)
    if own and op == "attend":
        from tinycoder_inference_b200 import ops
        s["ws"] = ops.paged_workspace()
    return s


def run(s):
    case = s["case"]
    if own:
        from tinycoder_inference_b200 import ops
        if case["op"] == "attend":
            ops.attn_paged(s["q"], s["kc"], s["vc"], s["pages"], s["lens"], s["out"], s["ws"], starts=s["starts"],
                           max_tokens=s["max_new"], ks=s["ks"], vs=s["vs"])
            return s["out"]
        if case["op"] == "write":
            ops.paged_write(s["k"], s["v"], s["kc"], s["vc"], s["pages"], s["lens"], starts=s["starts"], ks=s["ks"],
                            vs=s["vs"], q=s["q"], q_out=s["q_out"], cosT=s["cos"], sinT=s["sin"])
            if case["store"] != "i8":
                return {"q": s["q_out"], "k": s["kc"], "v": s["vc"]}
        ops.paged_read(s["kc"], s["vc"], s["pages"], s["lens"], s["k_out"], s["v_out"], starts=s["starts"], ks=s["ks"],
                       vs=s["vs"])
        if case["op"] == "write":
            return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"], "ks": s["ks"], "vs": s["vs"]}
        return {"k": s["k_out"], "v": s["v_out"]}
    return {"attend": _plain_attend, "write": _plain_write, "read": _plain_read}[case["op"]](s)


# ---- the operators in elementary torch operations -----------------------------------------------------

def _tokens(s):
    """Sequence and position of every new token."""
    case, dev = s["case"], s["lens"].device
    t = torch.arange(s["tokens"], device=dev)
    starts = s["starts"] if s["starts"] is not None else torch.arange(case["batch"] + 1, device=dev) * case["new_hi"]
    starts = starts.long()
    seq = (t[:, None] >= starts[None, 1:]).sum(1)
    return seq, t - starts[seq], s["lens"].long()[seq] - (starts[seq + 1] - t)


def _rows(s, seq, pos):
    """Rows of the pool, pages one behind another."""
    R = s["case"]["page"]
    return s["pages"][seq, pos // R].long() * R + pos % R


def _rotated(x, c, sn):
    """x0 c - x1 s, x0 s + x1 c of the pairs (j, j + head_dim / 2): the second product rounded, then one fused step."""
    a, b = x.chunk(2, dim=-1)
    c, sn = c[:, None, :], sn[:, None, :]
    return torch.cat([(a.double() * c - (b * sn).double()).float(), (a.double() * sn + (b * c).double()).float()], -1)


def _plain_write(s):
    case = s["case"]
    seq, _, pos = _tokens(s)
    row = _rows(s, seq, pos)
    c, sn = s["cos"][pos], s["sin"][pos]
    s["q_out"].copy_(_rotated(s["q"], c, sn))
    out = {"q": s["q_out"]}
    for name, x in (("k", _rotated(s["k"], c, sn)), ("v", s["v"])):
        pool = s[name + "c"].view(-1, case["kv_heads"], case["head_dim"])
        if case["store"] == "f16":
            pool[row] = x.half()
            out[name] = s[name + "c"]
            continue
        amax = x.abs().amax(-1)
        scale = torch.where(amax > 0, amax / torch.full_like(amax, 127.0), 1.0)
        q8 = torch.round(x / scale[..., None]).clamp(-128, 127)
        pool[row] = q8.to(torch.int8)
        s[name + "s"].view(-1, case["kv_heads"])[row] = scale
        out[name + "s"] = s[name + "s"]
        s[name + "_out"].copy_(pool[row].float() * s[name + "s"].view(-1, case["kv_heads"])[row][..., None])
        out[name] = s[name + "_out"]
    return out


def _values(s, name, row):
    """Rows of a pool as f32."""
    case = s["case"]
    x = s[name + "c"].view(-1, case["kv_heads"], case["head_dim"])[row].float()
    if case["store"] == "i8":
        x = x * s[name + "s"].view(-1, case["kv_heads"])[row][..., None]
    return x


def _plain_read(s):
    seq, _, pos = _tokens(s)
    row = _rows(s, seq, pos)
    for name in ("k", "v"):
        s[name + "_out"].copy_(_values(s, name, row))
    return {"k": s["k_out"], "v": s["v_out"]}


def _plain_attend(s):
    case, dev = s["case"], s["lens"].device
    nH, nKV, hd, B, n, L = case["q_heads"], case["kv_heads"], case["head_dim"], case["batch"], s["max_new"], s["max_len"]
    seq, i, pos = _tokens(s)
    j = torch.arange(L, device=dev)
    held = j[None, :] < s["lens"][:, None]
    b = torch.arange(B, device=dev)[:, None]
    row = torch.where(held, _rows(s, b, torch.where(held, j[None, :], 0)), 0)
    q = torch.zeros((B, n, nH, hd), device=dev)
    q[seq, i] = s["q"].float()
    last = torch.full((B, n), -1, device=dev)          # the last row that a token sees
    last[seq, i] = pos
    q = q.view(B, n, nKV, nH // nKV, hd).permute(0, 2, 3, 1, 4).reshape(B, nKV, -1, hd)
    k = _values(s, "k", row).permute(0, 2, 3, 1)        # [B][kv head][head_dim][L]
    scores = (torch.matmul(q, k) / math.sqrt(hd)).view(B, nKV, nH // nKV, n, L)
    del k
    scores.masked_fill_(j[None, None, None, None, :] > last[:, None, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(top > -math.inf, top, 0.0)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    v = _values(s, "v", row).permute(0, 2, 1, 3) * held[:, None, :, None]
    o = torch.matmul(scores.view(B, nKV, -1, L), v).view(B, nKV, nH // nKV, n, hd)
    o = o / torch.where(total > 0, total, 1.0)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(B, n, nH, hd)[seq, i])
    return s["out"]


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    lens, new = _lengths(case)
    R, nH, nKV, hd = case["page"], case["q_heads"], case["kv_heads"], case["head_dim"]
    i8 = case["store"] == "i8"
    f64 = torch.float64

    def rows_of(b, first, end):
        p = torch.arange(first, end, device=s["lens"].device)
        return s["pages"][b].long()[p // R] * R + p % R

    def held(name, r):
        x = s[name + "c"].reshape(-1, nKV, hd)[r].to(f64)
        return x * s[name + "s"].reshape(-1, nKV)[r].to(f64).unsqueeze(-1) if i8 else x

    if case["op"] == "read":
        where = [rows_of(b, n - m, n) for b, (n, m) in enumerate(zip(lens, new))]
        return {name: torch.cat([held(name, r) for r in where]) for name in ("k", "v")}
    if case["op"] == "write":
        p = torch.cat([torch.arange(n - m, n, device=s["lens"].device) for n, m in zip(lens, new)])
        r = torch.cat([rows_of(b, n - m, n) for b, (n, m) in enumerate(zip(lens, new))])
        turn = torch.complex(s["cos"].to(f64), s["sin"].to(f64))[p].unsqueeze(1)

        def rotate(x):
            z = torch.complex(x[..., :hd // 2].to(f64), x[..., hd // 2:].to(f64)) * turn
            return torch.cat([z.real, z.imag], -1)

        out = {"q": rotate(s["q"])}
        for name, x in (("k", rotate(s["k"])), ("v", s["v"].to(f64))):
            if not i8:
                pool = s[name + "c"].to(f64)
                pool.view(-1, nKV, hd)[r] = x
                out[name] = pool
                continue
            a = x.abs().amax(-1) / 127
            a = torch.where(a == 0, torch.ones_like(a), a)
            scales = s[name + "s"].to(f64)
            scales.view(-1, nKV)[r] = a
            out[name + "s"] = scales
            out[name] = torch.round(x / a.unsqueeze(-1)) * a.unsqueeze(-1)
        return out
    outs, at, group = [], 0, nH // nKV
    for b, (n, m) in enumerate(zip(lens, new)):
        r = rows_of(b, 0, n)
        k, v = held("k", r), held("v", r)
        q = s["q"][at:at + m].to(f64)
        at += m
        o = torch.empty((m, nH, hd), dtype=f64, device=q.device)
        step = max(1, (1 << 28) // (n * group))  # tokens at a time
        for t in range(0, m, step):
            e = min(m, t + step)
            see = torch.arange(n, device=q.device)[None, :] <= torch.arange(n - m + t, n - m + e, device=q.device)[:, None]
            for h in range(nKV):
                x = torch.einsum("tgd,jd->gtj", q[t:e, h * group:(h + 1) * group], k[:, h]) * hd ** -0.5
                w = torch.softmax(x.masked_fill(~see, float("-inf")), -1)
                o[t:e, h * group:(h + 1) * group] = torch.einsum("gtj,jd->tgd", w, v[:, h])
        outs.append(o)
    return torch.cat(outs)


def work(case):
    lens, new = _lengths(case)
    nH, nKV, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    io = 2 if case["io"] == "f16" else 4
    row = 2 * nKV * (hd + 4 if case["store"] == "i8" else 2 * hd)  # K and V of a row in the store
    tokens = sum(new)
    table = 4 * sum(-(-n // case["page"]) for n in lens) + 4 * case["batch"]
    if case["op"] == "read":
        return {"bytes": tokens * (row + 2 * nKV * hd * io) + table, "flops": 0}
    if case["op"] == "write":
        moved = tokens * (nH * hd * (4 + io) + 2 * nKV * hd * 4 + row) + 4 * hd * max(lens if case["batch"] == 1 else new)
        if case["store"] == "i8":
            moved += tokens * (row + 2 * nKV * hd * 2)
        return {"bytes": moved, "flops": 6 * tokens * (nH + nKV) * hd}
    seen = sum((n - m) * m + m * (m + 1) // 2 for n, m in zip(lens, new))
    return {"bytes": sum(lens) * row + 2 * tokens * nH * hd * io + table, "flops": 4 * seen * nH * hd}
