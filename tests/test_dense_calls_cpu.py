"""Calls around 16-bit pages, as far as they can be looked at without a GPU: what a kernel reads before its wait,
frequencies of long contexts, sizes and refusals."""

import math
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


# fp64, a few operations of 2^-53 each on exponents and logarithms of at most 20: 1e-13 covers them and the ramp's slope
@pytest.mark.parametrize("rd, base, factor, length, high", [(128, 10000.0, 4.0, 65536, 32.0), (128, 10000.0, 16.0, 131072, 32.0),
                                                            (64, 10000.0, 40.0, 4096, 32.0), (128, 1e6, 4.0, 32768, 32.0),
                                                            (64, 10000.0, 8.0, 1 << 20, 32.0), (128, 10000.0, 8.0, 64, 32.0),
                                                            (2, 10000.0, 8.0, 4096, 32.0), (128, 10000.0, 4.0, 65536, None)])
def test_yarn_is_the_published_blend(rd, base, factor, length, high):
    """With the ramp's end in the table and behind it (the slowest frequency makes more than one turn)."""
    index = lambda n: rd * math.log(length / (n * 2 * math.pi)) / (2 * math.log(base))
    first, last = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), rd - 1)
    if first == last:
        last += 0.001
    want = []
    for j in range(rd // 2):
        w = base ** (-2.0 * j / rd)
        ramp = min(max((j - first) / (last - first), 0.0), 1.0)
        want.append(w / factor * ramp + w * (1 - ramp))
    kw = {} if high is None else dict(high=high)
    got, scale = fq.rotary_frequencies(rd, base, "yarn", factor, length, **kw)
    assert got.tolist() == pytest.approx(want, rel=1e-13) and scale == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)


def test_the_slowest_frequency_is_divided_no_further_than_its_turns_ask_for():
    plain, _ = fq.rotary_frequencies(128, 10000.0)
    f, _ = fq.rotary_frequencies(128, 10000.0, "yarn", 16.0, 131072, 1.0, 32.0)
    assert 131072 * plain[-1] / (2 * math.pi) > 1.0 and f[-1] / plain[-1] > 2.0 / 16.0


def test_where_the_turns_end_by_default():
    for scaling, high in (("wavelength", 4.0), ("yarn", 32.0)):
        a, b = (fq.rotary_frequencies(64, 10000.0, scaling, 8.0, 4096, **kw)[0] for kw in ({}, dict(high=high)))
        assert torch.equal(a, b)
