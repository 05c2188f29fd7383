"""Bounded waits in front of barriers that only some warps reach: a wait that runs out in one warp never leaves another behind."""
import os
import re

import pytest

from onnx_genai_b200.specs import epilogue_votes

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "kernels")


@pytest.mark.parametrize("warps,tiles,barriers", [(2, 1, 1), (2, 3, 2), (4, 2, 2), (3, 2, 4)])
def test_warps_that_decide_together_all_reach_the_end(warps, tiles, barriers):
    r = epilogue_votes.check(warps, tiles, barriers)
    assert r.ok and r.states > 10, str(r)


def test_a_warp_that_decides_alone_leaves_the_others_in_the_groups_barrier():
    r = epilogue_votes.check(2, 1, 1, vote=False)
    assert not r.ok and r.kind == "deadlock" and any("gives up" in s for s in r.trace) and any("sees" in s for s in r.trace), str(r)


def _body(path, name):
    """The function's text, from its name to the line that closes it."""
    with open(os.path.join(KERNELS, path), encoding="utf-8") as f:
        text = f.read()
    start = re.search(r"^OGB_DEVICE void %s\(" % name, text, flags=re.M).start()
    return text[start:text.index("\n}\n", start)]


@pytest.mark.parametrize("path,name,vote", [("gemm_int8.cu", "i8_epilogue", "i8_group_all("), ("gemm_rows.cuh", "rows_epilogue", "rows_epi_all(")])
def test_the_epilogues_vote_before_any_warp_leaves_a_tile(path, name, vote):
    body = _body(path, name)
    wait = body.index("&bars->tmem_full[buf]" if "&bars->tmem_full[buf]" in body else "&tmem_full[buf]")
    line = body[body.rindex("\n", 0, wait):body.index("\n", wait)]
    assert vote in line, "each warp goes by its own wait:" + line
    assert "continue;" not in body[:wait]


def _loop(path, first):
    """The text of the loop whose body begins with `first` (a regular expression), from there to its closing brace."""
    with open(os.path.join(KERNELS, path), encoding="utf-8") as f:
        text = f.read()
    start = re.search(first, text).start()
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth < 0:
            return text[start:i]
    raise AssertionError(path)


def test_prefill_over_expanded_pages_leaves_its_loop_as_one():
    body = _loop("attention_fp8.cu", r"[^\n]*mbar_wait\(&full_bar\[stage\], phase\)[^\n]*\n(?=[^}]*// warp w expands page w)")
    assert body.count("break;") == 1 and re.search(r"if \(!compute_bar_all\(there\)\) \{ ok = false; break; \}", body)
    assert body.index("compute_bar_all(there)") < body.index("compute_bar_sync()")


def test_a_warp_that_meets_the_barriers_it_owes_leaves_nobody_behind():
    r = epilogue_votes.check(3, 3, 1, vote=False, owes=True)
    assert r.ok and r.states > 10, str(r)


def test_decode_over_one_byte_pages_counts_the_barriers_that_a_warp_owes():
    body = _loop("attention_fp8_tc.cu", r"      const int s = i % kTcStages, b = i & 1;\n      stamp.begin\(\);\n      ok = ")
    with open(os.path.join(KERNELS, "attention_fp8_tc.cu"), encoding="utf-8") as f:
        behind = f.read().split(body)[1]
    # one barrier a block, and one behind the loop for warps that got that far
    assert body.count("compute_bar_sync();") == 1 and behind[:behind.index("__syncthreads()")].count("compute_bar_sync();") == 2
    ahead, rest = body.split("compute_bar_sync();")
    assert ahead.count("break;") == ahead.count("owed = n_blocks - i + 1; break;") == 1
    assert rest.count("break;") == rest.count("owed = n_blocks - i; break;") == 2
    assert "for (; owed > 0; --owed) compute_bar_sync();" in behind[:behind.index("} else {")]
