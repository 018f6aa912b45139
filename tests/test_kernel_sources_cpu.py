"""Rules that the kernels' sources keep and that no run can show reliably."""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "laya_js_b200" / "csrc"


def _body(text: str, start: int) -> str:
    """The braces that open at or after `start`, with what they hold."""
    i = text.index("{", start)
    depth = 0
    for j in range(i, len(text)):
        depth += {"{": 1, "}": -1}.get(text[j], 0)
        if depth == 0:
            return text[i:j + 1]
    raise AssertionError("unbalanced braces")


def test_adapter_epilogues_meet_before_warp_wide_loads():
    """tcgen05.ld is .sync.aligned: undefined in a warp whose lanes have parted.
    Rows of one warp belong to different requests there, so the load itself
    brings the lanes together, and the lanes agree on a wait that ran out."""
    text = (CSRC / "lc_adapters_tc.cu").read_text()
    load = _body(text, text.index("void tmem_ld16("))
    assert load.index("__syncwarp()") < load.index("asm volatile")
    waits = re.findall(r"^.*mbar_wait\(&tfull\[acc\].*$", text, re.M)
    assert len(waits) == 2 and all("__all_sync(0xffffffffu, mbar_wait(" in w for w in waits)


def test_gemm_epilogues_meet_before_warp_wide_loads():
    text = (CSRC / "lc_gemm.cu").read_text()
    for load in ("tmem_ld64(tbase + u * 64, racc);", "tmem_ld32(tbase + u * 64, ra);"):
        at = text.index(load, text.index("epilogue_tma(" if "64(" in load else "k_gemm_tc(const"))
        lines = text[:at].rstrip().splitlines()
        assert lines[-1].strip().startswith("__syncwarp()"), lines[-1]


def test_the_per_thread_stream_is_not_taken_for_one_stream():
    """cudaStreamPerThread is one handle value for a different stream in every
    thread: nothing kept for a stream may be kept for it, and two uses of it
    are not in order."""
    core = (CSRC / "lc_core.cu").read_text()
    body = re.sub(r"//.*", "", _body(core, core.index("bool permanent_stream()")))
    assert "cudaStreamLegacy" in body and "cudaStreamPerThread" not in body
    enter = (CSRC / "lc_adapters.cu").read_text()
    assert "st != cudaStreamPerThread) return;" in _body(enter, enter.index("void plan_enter("))


def test_a_flush_reads_the_adapters_error_word_only_after_their_kernels():
    """Every flush and every host-to-host forward takes the device errors; a
    word of kernels that did not run would cost each a blocking copy."""
    text = (CSRC / "lc_adapters_tc.cu").read_text()
    body = _body(text, text.index("std::string take_adapter_errors()"))
    assert body.index('if (!launched) return "";') < body.index("cudaMemcpyFromSymbol")
    for entry in ("void adapter_shrink_tc(", "void adapter_outer_tc("):
        assert "launched = true;" in _body(text, text.index(entry))
