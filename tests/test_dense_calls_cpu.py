"""Calls around 16-bit pages, as far as they can be looked at without a GPU: what a kernel reads before its wait,
frequencies of long contexts, sizes and refusals."""

import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "flashquant_b200", "csrc")


def _kernel(source, name):
    """The body of a kernel, comments left out."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, source)).read())
    at = text.index("{", text.index(name + "(const DenseArgs p)"))
    depth, end = 1, at + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
    return text[at:end]


@pytest.mark.parametrize("name", ["dense_decode_kernel", "dense_join_kernel"])
def test_nothing_is_read_before_the_wait(name):
    """Launched while the kernels before it may still run, a kernel sees what those wrote only behind a wait of its own:
    before it no memory that the arguments point to is touched."""
    body = _kernel("dense_decode.cu", name)
    assert body.count("griddepcontrol.wait") == 1
    before = body[:body.index("griddepcontrol.wait")]
    args = re.search(r"struct DenseArgs \{(.*?)\n\};", open(os.path.join(CSRC, "dense_decode.cu")).read(), re.S).group(1)
    pointers = [n for line in re.findall(r"[^;]*\*[^;]*;", args) for n in re.findall(r"\*?\b(\w+)\b(?=\s*[,;])", line)]
    assert {"q", "k", "v", "out", "lse", "table", "lens", "status", "tickets", "bounds", "pieces"} <= set(pointers)
    for n in pointers:
        assert not re.search(r"\bp\.%s\b" % n, before), n
