"""Wait states of the kernels' LDS-DMA requests (buffer_load ... lds), read off the gfx950 listing: between the write of M0 and the load the
hardware asks software for one, between a vector instruction's write of a scalar operand of it and the load for five.  The compiler keeps to
that for its own instructions; it does not look into inline asm."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lidiff_amd", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith((".hip", ".h")))


def scalar_registers(token):
    m = re.match(r"s\[(\d+):(\d+)\]$", token)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"s(\d+)$", token)
    return {int(m[1])} if m else set()


def short_requests(listing):
    """(requests, those behind too few wait states), a scan in the listing's order."""
    requests, short, at, m0, by_vector = 0, [], 0, -100, {}
    for number, line in enumerate(listing.split("\n"), 1):
        text = line.split(";")[0].strip()
        if not text or text.startswith(".") or text.endswith(":"):
            continue
        op, _, rest = text.partition(" ")
        operands = [o.strip() for o in rest.split(",")]
        if op == "s_nop":
            at += int(operands[0], 0) + 1
            continue
        if op.startswith("buffer_load") and re.search(r"\blds\b", rest):
            requests += 1
            used = set().union(*(scalar_registers(o.split()[0]) for o in operands if o))
            if at - m0 - 1 < 1 or any(at - by_vector.get(r, -100) - 1 < 5 for r in used):
                short.append((number, text))
        if operands[0] == "m0":
            m0 = at
        if op.startswith("v_"):
            by_vector.update((r, at) for r in scalar_registers(operands[0]))
        elif op.startswith("s_"):
            for r in scalar_registers(operands[0]):
                by_vector.pop(r, None)
        at += 1
    return requests, short


def test_the_scan_sees_what_it_looks_for():
    request = "\tbuffer_load_dwordx4 v1, s[4:7], s8 offen lds\n"
    assert short_requests("\ts_mov_b32 m0, s3\n" + request) == (1, [(2, request.strip())])
    assert short_requests("\ts_mov_b32 m0, s3\n\ts_nop 0\n" + request) == (1, [])
    assert short_requests("\tv_readfirstlane_b32 s5, v2\n\ts_mov_b32 m0, s3\n\ts_nop 2\n" + request)[1]
    assert short_requests("\tv_readfirstlane_b32 s5, v2\n\ts_mov_b32 m0, s3\n\ts_nop 3\n" + request) == (1, [])
    assert short_requests("\tv_readfirstlane_b32 s9, v2\n\ts_mov_b32 m0, s3\n\ts_nop 0\n" + request) == (1, [])


@pytest.mark.parametrize("source", SOURCES)
def test_inline_requests_bring_their_wait_states(source):
    """Every asm string that writes M0 waits five instructions before its load and names M0 among what it writes."""
    text = open(os.path.join(CSRC, source)).read()
    for m in re.finditer(r'asm volatile\("[^"]*s_mov_b32 m0.*?\);', text, re.S):
        assert re.search(r"m0, %0\\n\\ts_nop 3\\n\\tbuffer_load", m[0]) and '"m0"' in m[0], m[0]


# (attention_fwd.hip: descriptors from v_readfirstlane close to their requests; spconv_split3.hip: the shortest of the others)
@pytest.mark.parametrize("source", ["spconv_split3.hip", "attention_fwd.hip"])
def test_requests_of_the_listing_keep_their_distance(tmp_path, source):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    from lidiff_amd.csrc.build import NO_PACKED_F32
    out = os.path.join(tmp_path, "kernel.s")
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-x", "hip", "--cuda-device-only", "-S", os.path.join(CSRC, source), "-o", out]
                       + NO_PACKED_F32, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    requests, short = short_requests(open(out).read())
    assert requests > 50 and not short, (requests, len(short), short[:5])
