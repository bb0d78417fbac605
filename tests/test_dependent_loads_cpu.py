"""Kernels of the 8-bit cache and of sampling start while the kernel before them in the stream still runs.  What that kernel
may have written has to come by coherent loads behind the wait, so none of their sources may ask for read-only ones."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "demonic_b200" / "csrc"


@pytest.mark.parametrize("name", ["kv8.cuh", "kv8.cu", "kv8_pages.cu", "sample.cu"])
def test_no_read_only_loads(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    found = re.findall(r"\.nc\b|__ldg\b|ldg_stream16|__restrict__", text)
    assert not found, f"{name}: {found}"


def test_the_coherent_streaming_load_stays_behind_the_wait():
    text = (CSRC / "gemv.cuh").read_text()
    body = text[text.index("uint4 ld_stream16("):]
    body = body[:body.index("return")]
    assert "asm volatile" in body and "ld.global.L1" in body
    assert "asm volatile" in text[text.index("void griddep_wait()"):].split("\n")[0]
