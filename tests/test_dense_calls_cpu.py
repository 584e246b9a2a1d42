"""Calls around 16-bit pages, as far as they can be looked at without a GPU: what a kernel reads before its wait,
frequencies of long contexts, sizes and refusals."""

import os
import re

import pytest
import torch

import flashquant_b200 as fq
from flashquant_b200 import _native as N
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


def _decode_args(**kw):
    pages = torch.zeros(4, 16, 8, 128, dtype=torch.float16)
    return {**dict(q=torch.zeros(2, 8, 128, dtype=torch.float16), key_cache=pages, value_cache=pages,
                   block_table=torch.zeros(2, 2, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32)), **kw}


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(1 << 28), torch.zeros(1 << 12, dtype=torch.uint8)[::2],
                                       torch.zeros(1 << 12), torch.zeros(64, 64, dtype=torch.uint8).t()])
def test_workspaces_that_are_not_plain_bytes(monkeypatch, workspace):
    """A workspace whose number of values is not the number of bytes behind its address is refused before anything else."""
    monkeypatch.setattr(N, "require_cuda", lambda *t: None)
    with pytest.raises(ValueError, match="workspace"):
        fq.split_k_paged_decode_dense(**_decode_args(workspace=workspace))


@pytest.mark.parametrize("block_size", [2 ** 32 + 16, 2 ** 31, 2 ** 64 + 1, 0, -16])
def test_block_sizes_beyond_32_bits(monkeypatch, block_size):
    monkeypatch.setattr(N, "require_cuda", lambda *t: None)
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="block_size"):
        fq.plan_paged_step(i32, i32, i32.view(2, 1), i32, i32[:1], block_size, 8)
    with pytest.raises(ValueError, match="block_size"):
        fq.release_pages(i32.bool(), i32, i32.view(2, 1), i32, i32[:1], block_size)
