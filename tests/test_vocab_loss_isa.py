"""Build-time checks (no GPU) of what the streaming kernels of ns_linear_loss.hip count by hand, on the gfx950 assembly of the source as it is built:
the s_waitcnt vmcnt(n) in front of a tile's first K steps allow for exactly the stores that the tile before issues, so the compiler must neither
merge, split nor spill around them."""
import os
import re
import subprocess

import pytest

from neuspeech1_amd import build

pytestmark = pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc (cross-compiles gfx950 without a GPU)")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("isa") / "ll.s")
    flags = [f for f in build.flags_of("ns_linear_loss.hip") if f != "-fPIC"]
    subprocess.run([build.HIPCC, *flags, "-S", "--cuda-device-only", os.path.join(build.CSRC, "ns_linear_loss.hip"), "-o", out], check=True, capture_output=True)
    text = open(out).read()
    return {m.group(1): m.group(2) for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)\.Lfunc_end", text, re.S | re.M)}


def pick(kernels, part):
    got = {n: b for n, b in kernels.items() if part in n}
    assert got
    return got


def count(body, pattern):
    return len(re.findall(pattern, body))


def test_no_packed_fp32_and_no_scratch(kernels):
    for name, body in kernels.items():
        assert not re.search(r"v_pk_(add|mul|fma)_f32", body), name
        if "ll_" in name:
            assert not re.search(r"\bscratch_", body), name


@pytest.mark.parametrize("mode,dual,x4,x1", [(0, 0, 0, 4), (0, 1, 0, 6), (1, 0, 16, 12), (1, 1, 16, 14), (2, 0, 16, 0), (2, 1, 16, 0)])
def test_stores_per_tile_of_the_logits_kernel(kernels, mode, dual, x4, x1):
    """mode 1 (kept): 16 stores of the tile + 8 of the strips' maxima = the 24 that vmcnt(32) allows for beside 8 DMA pieces; the join of the statistics is
    there twice (loop, end).  mode 2 (dz): the 16 of vmcnt(24)."""
    for name, body in pick(kernels, f"ll_logits_kernel").items():
        if f"Li{mode}ELb{dual}" not in name:
            continue
        assert count(body, r"global_store_dwordx4") == x4 and count(body, r"global_store_dword\b") == x1, name
        assert count(body, r"v_mfma") == 128
        want = {0: (0, 0), 1: (4, 0), 2: (0, 4)}[mode]
        assert (count(body, r"vmcnt\(32\)"), count(body, r"vmcnt\(24\)")) == want, name


def test_the_transposed_products_never_drain_their_ring(kernels):
    """between the DMA pieces and the transposed fragment reads hipcc inserts no wait of its own (it would be vmcnt(0) in every phase)"""
    for part in ("ll_dh_kernel", "ll_dw_kernel"):
        for name, body in pick(kernels, part).items():
            loop = body[body.index("ds_read_b64_tr"):]
            loop = loop[:[m.end() for m in re.finditer(r"v_mfma", loop)][-1]]
            assert "vmcnt(0)" not in loop, name
