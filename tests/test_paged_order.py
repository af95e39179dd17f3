"""What the paged kernels read before they wait for the launch in front of them, and why that is finished work (a check of the sources; no GPU).

A kernel that is launched early starts when every block of the one in front has triggered.  All kernels of the cache wait before they trigger, so that at that moment
everything ahead of the kernel in front has ended; what its successor reads without a wait of its own may therefore be anything but that kernel's own output.  The
attention kernel behind the prefix kernel relies on it for positions, pages, queries, keys and values, the merge and the choice for a row's place."""
import os
import re

import pytest

from yasakani_b200 import build


def code(name):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(build.CSRC, name)).read(), flags=re.S)


def body(text, kernel):
    at = text.index("{", re.search(rf"\b{kernel}\(const [^)]*\)", text).end() - 1)
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i]


KERNELS = [("paged_append.cu", "paged_append_kernel"), ("paged_select.cu", "paged_score_kernel"), ("paged_select.cu", "paged_choose_kernel"),
           ("paged_attn.cu", "paged_attn_kernel"), ("paged_attn.cu", "paged_merge_kernel"), ("paged_prefix.cu", "paged_prefix_kernel")]


@pytest.mark.parametrize("file,kernel", KERNELS)
def test_every_kernel_waits_before_it_triggers(file, kernel):
    b = body(code(file), kernel)
    wait, trigger = b.index("pdl_wait()"), b.index("pdl_launch()")
    assert wait < trigger and b.count("pdl_launch()") == 1
    assert not b[wait + len("pdl_wait()"):trigger].strip(" ;\n"), "something between the wait and the trigger"
    first = b[:wait]
    if kernel == "paged_attn_kernel":                            # its wait is left out behind the prefix kernel alone, and made up for by blocks without work, by the producer and by the compute warps
        assert re.search(r"if \(!P\.beside\) $", first) and not re.search(r"\b(P\.(R|q|ids|qml|qacc)\b|place_of|page_of)", first)
        assert b.count("if (P.beside) pdl_wait();") == 3
    elif kernel == "paged_merge_kernel":
        assert re.findall(r"\b(place_of\S*|page_of\S*|P\.(?:span|ml|pacc|qml|qacc)\b)", first) == ["place_of<true>(P.R,"]
    elif kernel == "paged_choose_kernel":
        assert re.findall(r"\b(place_of\S*|page_of\S*|P\.(?:approx|exact|q|kmean)\b)", first) == ["place_of<true>(P.R,"] and "if (P.scored) w = place_of<true>" in first
    else:
        assert not re.search(r"place_of|page_of|__ldc|\bP\.(q|k|v|k_in|v_in|q_in|kmean|rope)\b", first)


def test_early_reads_come_past_l1():
    """An SM's first-level cache may hold lines from before; only reads behind a kernel's own wait may meet them."""
    attn = body(code("paged_attn.cu"), "paged_attn_kernel")
    assert re.findall(r"\b(?:place_of|page_of)(?:<\w+>)?\(", attn) == ["place_of<true>(", "page_of<true>("]
    common = code("paged_common.cuh")
    assert "PAST_L1 ? __ldcg(p) : *p" in common
    assert not re.search(r"[^_](R|P\.R)\.(seq|pos|table)\s*(\+|\[)", re.sub(r"read_index<PAST_L1>\([^)]*\)", "", common))
    # the attention kernel's only other way to memory ahead of a wait is by asynchronous copies; chosen blocks exclude a shared part
    assert "P.ids[" in attn and re.search(r"if \(P\.ids\)", attn) and "a->ids && a->shared > 0" in code("paged_abi.cu")


def test_no_kernel_writes_positions_or_tables():
    for file in sorted({f for f, _ in KERNELS}):
        assert not re.search(r"\b(?:R|P\.R)\.(?:seq|pos|table)\[[^\]]*\]\s*=[^=]", code(file)), file
    assert "const int* table" in code("paged_common.cuh") and "const int* seq; const int* pos;" in code("paged_common.cuh")


def test_the_prefix_kernel_is_the_one_in_front():
    launch = code("paged_attn.cu")
    assert "splits > 0 && first == 0 ? 1 : 0" in launch         # beside: the first launch behind the prefix kernel, nothing in between
    a, b = launch.index("launch_paged_prefix(c, r, a, splits, w, st)"), launch.index("for (int first = 0; first < r.rows")
    assert not re.search(r"launch_|<<<", launch[a + len("launch_paged_prefix"):b])
