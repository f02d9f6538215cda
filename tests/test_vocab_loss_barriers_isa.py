"""Build-time check (no GPU) on the gfx950 assembly of ns_linear_loss.hip: shared memory that every wave reads is not written over before all of them have read it."""
import os
import re
import subprocess

import pytest

from neuspeech1_amd import build

pytestmark = pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc (cross-compiles gfx950 without a GPU)")
COUNT_AT = 4096 * 8 + 128 * 4        # ll_add_entries: the batch's number of entries, behind LL_LIST pairs, 64 counts and 64 prefixes


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("isa") / "ll.s")
    flags = [f for f in build.flags_of("ns_linear_loss.hip") if f != "-fPIC"]
    subprocess.run([build.HIPCC, *flags, "-S", "--cuda-device-only", os.path.join(build.CSRC, "ns_linear_loss.hip"), "-o", out], check=True, capture_output=True)
    return {m.group(1): m.group(2) for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)\.Lfunc_end", open(out).read(), re.S | re.M)}


def reached_without_a_barrier(body, start, target):
    """lines that match `target` on some path from a line that matches `start`, no s_barrier between"""
    lines = [ln.split(";")[0].strip() for ln in body.splitlines()]
    label = {ln[:-1]: i for i, ln in enumerate(lines) if re.fullmatch(r"\.LBB\w+:", ln)}
    starts = [i for i, ln in enumerate(lines) if re.search(start, ln)]
    todo, seen, hits = [i + 1 for i in starts], set(), []
    while todo:
        i = todo.pop()
        while i < len(lines) and i not in seen:
            seen.add(i)
            op, _, arg = lines[i].partition(" ")
            if op in ("s_barrier", "s_endpgm"):
                break
            if re.search(target, lines[i]):
                hits.append(lines[i])
            if op == "s_branch":
                i = label[arg.strip()]
                continue
            if op.startswith("s_cbranch"):
                todo.append(label[arg.strip()])
            i += 1
    return starts, hits


def test_the_walk_sees_a_missing_barrier_and_a_loop():
    body = "ds_read_b32 v1, v2 offset:8\n.LBB0_1:\ns_cbranch_scc1 .LBB0_3\n.LBB0_2:\ns_barrier\ns_branch .LBB0_1\n.LBB0_3:\nds_write2_b64 v1, v[2:3], v[4:5]\ns_endpgm\n"
    assert len(reached_without_a_barrier(body, "offset:8", "ds_write2_b64")[1]) == 1
    assert not reached_without_a_barrier(body.replace(".LBB0_3:\n", ".LBB0_3:\ns_barrier\n"), "offset:8", "ds_write2_b64")[1]


def test_no_wave_stages_dw_over_a_count_that_another_has_yet_to_read(kernels):
    """ll_dw_kernel: where no entry names the tile nothing but this barrier stands between the last read of the number of entries and the 16-bit epilogue, which
    stages dW over it"""
    got = {n: b for n, b in kernels.items() if "ll_dw_kernel" in n}
    assert len(got) == 2
    for name, body in got.items():
        starts, hits = reached_without_a_barrier(body, rf"ds_read_b32 .*offset:{COUNT_AT}\b", r"ds_write(2|2st64)?_b64 ")
        assert starts, name
        assert not hits, (name, hits[:2])
