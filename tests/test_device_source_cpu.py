"""Rules for the device code that reading decides, not a run (breaking one may hang a GPU)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinycoder_inference_b200", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_asm_that_synchronises_is_volatile():
    """An asm statement that is not volatile is a function of its operands: the compiler may move it to where its result
    is used, say under a test of the lane, and a warp-wide operation is then run by part of the warp."""
    seen, bad = 0, []
    for name in SOURCES:
        for m in re.finditer(r"\basm\b(\s+volatile\b)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)", _code(name)):
            if re.search(r"\.sync\b|\bbar\.|\bbarrier\.|mbarrier\.|tcgen05\.|cp\.async|griddepcontrol", m.group(2)):
                seen += 1
                if not m.group(1):
                    bad.append((name, m.group(2).strip()))
    assert seen > 30 and bad == []


def test_tensor_memory_is_given_back_behind_the_warps_that_issue():
    """A wait that ran out in some warps must not free tensor memory that others still issue products into: in front of each
    deallocation stands a barrier of the block, or the one that the issuing warps arrive at when they are through."""
    found = 0
    for name in SOURCES:
        lines = _code(name).splitlines()
        for i, line in enumerate(lines):
            if "tmemDealloc(" not in line or "__device__" in line:
                continue
            found += 1
            before = "\n".join(x for x in lines[:i] if x.strip()).splitlines()[-5:]
            barrier = re.search(r"__syncthreads\(\)|namedBarSync\((kIssuedBar), ", "\n".join(before))
            assert barrier, (name, i + 1)
            if barrier.group(1):
                assert "namedBarArrive(kIssuedBar, " in "\n".join(lines[:i]), (name, i + 1)
    assert found >= 2


def _roles(name, *marks):
    """The code of a kernel's roles: what stands between one mark and the next."""
    code = _code(name)
    at = [code.index(m) for m in marks]
    assert at == sorted(at), name
    return [code[a:b] for a, b in zip(at, at[1:] + [len(code)])]


def test_paged_tiles_wait_for_the_last_release_of_every_slot():
    """A release of a K or V slot arrives when the products behind it are complete, at a barrier in the block's own memory: somebody
    has to wait for the last ones before the block leaves, over either kind of pages.  The waiting warp has to have seen the
    slot's last tile come in, or a parity wait may take an older phase for the last one: over fp16 pages the producers, which
    wait for every release themselves, over int8 ones the issuing warps, which wait for every tile."""
    producer, values, converters, issuers, softmax = _roles(
        "paged_tiles.cu", "if (warp == 8) {", "else if (!I8 && warp == 13)", "else if (I8 && warp >= 13)", "else if (warp >= 9 && warp < 13)", "else if (!(kOne && warp >= 4))")
    assert "drain(kEmpty, gk, NK" in producer and "drain(vEmpty, gv, NV" in values
    behind = issuers[issuers.index("g += it.nTiles;"):]
    assert re.search(r"if \(I8 && ok && x == 0u\)", behind)
    assert "drain(kEmpty, g, NK" in behind and "drain(vEmpty, g, NV" in behind


def test_prefill_commits_to_no_barrier_that_nobody_waits_for():
    """At head_dim 256 (kAhead) the softmax threads go by pvBuf: a commit to pvDone would be an arrival that no wait sees before the
    block leaves."""
    code = _code("prefill_f16.cu")
    assert re.search(r"kAhead\s*\?\s*pfWait<kCall>\(&pvBuf", code)
    commits = re.findall(r"[^\n]*umaCommit\(&pvDone\[x\]\)[^\n]*", code)
    assert len(commits) == 1 and "if (!kAhead)" in commits[0]


def test_the_query_tiles_last_release_is_waited_for():
    """The score warps commit to qFree with an item's last product; the producer waits for it ahead of the next item, so the last
    item's needs a wait of its own, in the producer, behind its loop over the items."""
    for name, loop in (("prefill_f16.cu", "item = next;"), ("paged_tiles.cu", "while (ok && w.next(p));")):
        code = _code(name)
        producer = code[code.index("if (warp == 8) {"):]
        behind = producer[producer.index(loop):]
        behind = behind[:re.search(r"else if \((!I8 && warp == 13|warp >= 9)\)", behind).start()]
        for x in "01":
            assert re.search(r"pfWait<kCall>\(&qFree\[%s\], \(n - 1u\) & 1u" % x, behind), (name, x)


def test_int8_decode_releases_only_stages_that_are_filled_again():
    """A stage's release is waited for by the request of the tile that takes it next.  Where there is none, nobody waits, and the
    arrival may come after the block has left: there is no commit then."""
    code = _code("decode_i8_tc.cu")
    assert len(re.findall(r"mbarWait<true>\(&emptyBar\[", code)) == 1 and "if (it >= NS && !mbarWait<true>(&emptyBar[s]" in code
    commits = re.findall(r"[^\n]*umaCommit\(&emptyBar\[s\]\)[^\n]*", code)
    assert len(commits) == 1 and "if (j + NS < nTiles)" in commits[0]


def test_shared_memory_is_handed_back_behind_the_loads_from_it():
    """A warp that releases a buffer it has loaded from makes the arrival wait for those loads (releaseStage: its address depends on
    what was loaded); an arrival by itself can overtake them, and the buffer's next contents then come in under the slowest warp."""
    common = _code("tc_common.cuh")
    assert "mbarArrive(bar + (used & zero))" in common[common.index("void releaseStage("):]
    seen = 0
    for name in SOURCES:
        code = _code(name)
        if "mbarInit(&emptyBar[s], VW + 1)" in code or "mbarInit(&empty[i], L::NW)" in code:  # rings that warps with loads release
            seen += code.count("releaseStage(&empty")
            assert not re.search(r"mbarArrive\(&empty", code), name
    assert seen == 4
