"""Step plans, rotary positions, append to and attention over 16-bit pages, against the definitions in 64 bits.

Tolerances are sums of what each rounding may do, at most; u = 2^-24 is half a step of fp32.
  attention   the output's own rounding, eps / 2 of the value.  A score of D products and its scaling is off by
              (D + 16) u of sum |q k|, which moves a weight by that share, numerator and denominator: 4 S (D + 16) u with
              S the largest scale * sum |q k| (natural units; the factor 4 also holds the exponential's 2 u).  A weight as two
              16-bit terms: 2^-17.  The running sums take n / 16 products and as many rescalings, 2 u each and once
              more for the sum of the weights: n u / 4; a join of a few hundred pieces the same once more.  All of these
              relative to sum p |v| / sum p.
  logarithm   S (D + 16) u, n u / 4 as above, and 4 u of its value and of log2 n.
  rotary      the angle after the whole turns are dropped: 2 pi * 2^-53 * 4 of the turns, pi u; sine and cosine 4 u; two
              products, the factor and a sum 4 u: 12 u of |a| + |b| and the share of the turns; the output's own rounding.
"""

import math
import random
import threading

import pytest
import torch

import flashquant_b200 as fq
from flashquant_b200 import _native as N
from flashquant_b200 import dense
from flashquant_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF, HF = torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# --------------------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------------------
class Batch:
    """Permuted pages of ``lens`` tokens; everything that no token of the batch stands in is NaN."""

    def __init__(self, lens, hq, hkv, d, dtype, block=16, layout="two", window=0, spare=3, width=None, seed=0, blocks=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        counts = [-(-n // block) for n in lens]
        total = blocks or sum(counts) + spare
        self.lens, self.hq, self.hkv, self.d, self.block, self.window = lens, hq, hkv, d, block, window
        shape = {"two": (2, total, block, hkv, d), "token": (total, block, 2, hkv, d), "heads": (2, total, hkv, block, d),
                 "padded": (2, total, block, hkv, d + 8)}[layout]
        pages = torch.full(shape, float("nan"), dtype=dtype, device=DEV)
        if layout == "token":
            self.k, self.v = pages[:, :, 0], pages[:, :, 1]
        elif layout == "heads":
            self.k, self.v = (p.transpose(1, 2) for p in pages)
        else:
            self.k, self.v = pages[0][..., :d], pages[1][..., :d]
        ids = torch.randperm(total, generator=g, device=DEV).int()
        self.table = torch.full((len(lens), width or max(max(counts), 1)), 1 << 30, dtype=torch.int32, device=DEV)
        at, self.rows = 0, []
        for i, (n, c) in enumerate(zip(lens, counts)):
            self.table[i, :c] = ids[at:at + c]
            at += c
            tok = torch.arange(max(0, n - window) if window else 0, n, device=DEV)
            page, row = self.table[i][tok // block].long(), tok % block
            k = torch.randn(len(tok), hkv, d, generator=g, device=DEV)
            k[..., ::max(1, d // 4)] *= 6.0
            self.k[page, row], self.v[page, row] = k.to(dtype), torch.randn(len(tok), hkv, d, generator=g, device=DEV).to(dtype)
            self.rows.append((page, row))
        self.q = torch.randn(len(lens), hq, d, generator=g, device=DEV).to(dtype)
        self.sl = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def call(self, **kw):
        return fq.split_k_paged_decode_dense(self.q, self.k, self.v, self.table, self.sl, window=self.window, **kw)

    def check(self, out, lse=None, scale=None, only=None):
        scale = 1.0 / math.sqrt(self.d) if scale is None else scale
        for i in range(len(self.lens)) if only is None else only:
            page, row = self.rows[i]
            n = len(page)
            if n == 0:
                assert not out[i].any() and (lse is None or bool((lse[i] == -math.inf).all()))
                continue
            g = self.hq // self.hkv
            q = self.q[i].double().view(self.hkv, g, self.d)
            k, v = (x[page, row].double().transpose(0, 1) for x in (self.k, self.v))
            s = scale * q @ k.transpose(1, 2)
            p = torch.softmax(s, -1)
            want = (p @ v).view(self.hq, self.d)
            S = abs(scale) * float((q.abs() @ k.abs().transpose(1, 2)).max())
            share = 4 * S * (self.d + 16) * U + 2.0 ** -17 + n * U / 2
            tol = half_step(out.dtype) * want.abs() + share * (p @ v.abs()).view(self.hq, self.d) * (1 + half_step(out.dtype))
            tol += torch.finfo(out.dtype).smallest_normal * half_step(out.dtype)  # (a rounding below the normal numbers)
            bad = ((out[i].double() - want).abs() > tol) | out[i].isnan()
            assert not bad.any(), (i, n, (out[i].double() - want).abs().max().item(), tol.min().item())
            if lse is not None:
                w = torch.logsumexp(s, -1).flatten()
                t = S * (self.d + 16) * U + n * U / 4 + 4 * U * (w.abs() + math.log2(n + 1) + 1)
                assert bool(((lse[i].double() - w).abs() <= t).all()), (i, (lse[i].double() - w).abs().max().item())


HEADS = [(32, 8, 128), (64, 8, 128), (8, 1, 128), (16, 16, 64), (40, 10, 96), (20, 2, 256), (48, 2, 128), (71, 1, 64),
         (8, 8, 256), (12, 4, 96), (1, 1, 128), (16, 1, 256)]


@pytest.mark.parametrize("hq, hkv, d", HEADS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_head_layouts(hq, hkv, d, dtype):
    b = Batch([1, 0, 17, 300, 16, 2049, 15, 33], hq, hkv, d, dtype, seed=hq + d)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("lens", [[1], [0], [15], [16], [17], [900], [9000], [5, 5, 5], [0, 0, 7], [1] * 300, [64] * 40,
                                  [131, 1, 4000, 0, 77, 2500], [3] * 1000 + [5000] + [0] * 100])
@pytest.mark.parametrize("hq, hkv, d", [(32, 8, 128), (8, 1, 64)])
def test_decode_lengths(lens, hq, hkv, d):
    b = Batch(lens, hq, hkv, d, BF, seed=len(lens))
    out, lse = b.call(return_lse=True)
    b.check(out, lse, only=range(0, len(lens), max(1, len(lens) // 50)))
    assert not out.isnan().any()


@pytest.mark.parametrize("block", [16, 32, 48, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 15, 16, 17, 250, 4000])
def test_decode_windows_and_pages(block, window):
    b = Batch([1, 0, 16, 250, 777, 3001], 16, 4, 128, HF, block=block, window=window, seed=window)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("layout", ["two", "token", "heads", "padded"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_cache_layouts(layout, dtype):
    b = Batch([33, 500, 1, 1200], 32, 8, 128, dtype, layout=layout)
    b.check(b.call())


def test_decode_scales_and_large_scores():
    b = Batch([100, 2000], 32, 8, 128, BF)
    for scale in (0.01, 1.0, -0.3, 0.0):
        out, lse = b.call(sm_scale=scale, return_lse=True)
        b.check(out, lse, scale=scale)
    b.q.mul_(20)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


def test_decode_arguments_of_other_layouts():
    """Strided queries, a wider block table, a given output: the same bits; the converting path the same."""
    b = Batch([40, 700, 9], 32, 8, 128, BF, width=60)
    want = b.call()
    b.check(want)
    joint = torch.randn(3, 48, 128, device=DEV).to(BF)
    joint[:, :32] = b.q
    out = torch.empty_like(want)
    table = b.table.t().contiguous().t()
    for q in (joint[:, :32], b.q.transpose(0, 1).contiguous().transpose(0, 1), b.q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(fq.split_k_paged_decode_dense(q, b.k, b.v, b.table, b.sl), want)
        got = fq.split_k_paged_decode_dense(q, b.k, b.v, table, b.sl, out=out)
        assert got is out and torch.equal(out, want)
    lens = torch.stack([b.sl, b.sl], 1)[:, 0]
    assert torch.equal(fq.split_k_paged_decode_dense(b.q, b.k, b.v, b.table, lens), want)
    ws = torch.zeros(N.load().fq_dense_paged_decode_workspace_bytes(3, 32, 8, 128), dtype=torch.uint8, device=DEV)
    for _ in range(3):
        assert torch.equal(b.call(workspace=ws), want)
    assert K.workspace_status(ws) == 0 and not ws[:32768].any()


def test_decode_refusals():
    b = Batch([40, 700], 32, 8, 128, BF)
    args = dict(q=b.q, key_cache=b.k, value_cache=b.v, block_table=b.table, seq_lens=b.sl)

    def refused(error=ValueError, **kw):
        with pytest.raises(error):
            fq.split_k_paged_decode_dense(**{**args, **kw})
    refused(q=b.q[0])
    refused(q=b.q.half())
    refused(TypeError, q=b.q.float())
    refused(key_cache=b.k[..., :64])
    refused(key_cache=b.k.transpose(2, 3))
    refused(value_cache=b.v[:-1])
    refused(block_table=b.table.long())
    refused(block_table=b.table[:1])
    refused(seq_lens=b.sl[:1])
    refused(seq_lens=b.sl.long())
    refused(window=-1)
    refused(out=torch.empty(2, 32, 64, dtype=BF, device=DEV))
    refused(N.FlashQuantNativeError, workspace=torch.zeros(1024, dtype=torch.uint8, device=DEV))
    refused(N.FlashQuantNativeError, out=torch.zeros(2 * 32 * 128 + 2, dtype=BF, device=DEV)[2:].view(2, 32, 128))
    refused(N.FlashQuantNativeError, q=torch.zeros(2, 12, 128, dtype=BF, device=DEV))
    refused(N.FlashQuantNativeError, seq_lens=b.sl.cpu())
    odd = torch.zeros(8 * 16 * 8 * 128 + 1, dtype=BF, device=DEV)[1:].view(8, 16, 8, 128)
    refused(N.FlashQuantNativeError, key_cache=odd, value_cache=odd)
    small = torch.zeros(8, 8, 8, 128, dtype=BF, device=DEV)
    refused(N.FlashQuantNativeError, key_cache=small, value_cache=small)


def test_decode_pages_out_of_range():
    """The tokens of a page that does not exist are skipped, a length beyond the block table is cut, the rest
    of the batch is as it was; both leave their mark."""
    b = Batch([40, 700, 90, 33], 32, 8, 128, BF)
    want = b.call()
    ws = torch.zeros(N.load().fq_dense_paged_decode_workspace_bytes(4, 32, 8, 128), dtype=torch.uint8, device=DEV)
    b.table[1, 3], b.table[1, 9] = -1, b.k.shape[0]
    out = b.call(workspace=ws)
    assert torch.equal(out[[0, 2, 3]], want[[0, 2, 3]])
    page, row = b.rows[1]
    seen = [i for i in range(700) if i // 16 not in (3, 9)]
    b.rows[1] = page[seen], row[seen]
    b.check(out, only=[1])
    assert K.workspace_status(ws, reset=True) == N.FQ_DEV_BAD_BLOCK_INDEX and K.workspace_status(ws) == 0
    b.table[1] = -5  # no page at all: nothing is seen
    out, lse = b.call(workspace=ws, return_lse=True)
    assert not out[1].any() and bool((lse[1] == -math.inf).all()) and torch.equal(out[[0, 2, 3]], want[[0, 2, 3]])
    assert K.workspace_status(ws, reset=True) == N.FQ_DEV_BAD_BLOCK_INDEX
    full = Batch([64, 48], 32, 8, 128, BF)
    want = full.call()
    full.sl[0], full.sl[1] = 2 ** 31 - 1, 64
    full.table[1, 3] = full.table[1, 0]
    out = full.call(workspace=ws)
    assert torch.equal(out[0], want[0]) and K.workspace_status(ws, reset=True) == N.FQ_DEV_BAD_BLOCK_INDEX
    full.sl[0] = -7
    assert not full.call(workspace=ws)[0].any() and K.workspace_status(ws) == 0


def test_decode_offsets_beyond_32_bits():
    blocks = (1 << 31) // (16 * 8 * 128) + 4000
    b = Batch([3000], 32, 8, 128, BF, blocks=blocks)
    assert int(b.table[0, :188].max()) * 16 * 8 * 128 > 1 << 31
    b.check(b.call())


def test_decode_repeats_bit_for_bit():
    b = Batch([4000, 1, 777, 2100, 60], 32, 8, 128, BF)
    want = b.call()
    assert all(torch.equal(b.call(), want) for _ in range(50))
    c = Batch([30000], 8, 1, 128, HF)
    want = c.call()
    assert all(torch.equal(c.call(), want) for _ in range(50))


@pytest.mark.parametrize("hq, hkv, d, lens, window", [
    (32, 8, 128, [230001, 3, 131072, 0, 77000, 60123], 0), (8, 1, 128, [1500000, 17, 2300000], 0),
    (16, 16, 64, [300000, 1, 180007, 90000], 0), (20, 2, 256, [70000, 500000, 16, 430000], 0),
    (32, 8, 128, [400000, 5, 390007], 300000), (32, 8, 128, [900 - i % 300 for i in range(620)], 0)])
def test_decode_long_lists(hq, hkv, d, lens, window):
    """Lists of which warps take a part when they are free (1.9 GB of keys and values; the last is one of too many
    sequences for that): right, and the same bits whoever takes what; the workspace's head is left as it was."""
    b = Batch(lens, hq, hkv, d, BF, block=64, window=window)
    ws = torch.zeros(N.load().fq_dense_paged_decode_workspace_bytes(len(lens), hq, hkv, d), dtype=torch.uint8, device=DEV)
    out, lse = b.call(return_lse=True, workspace=ws)
    b.check(out, lse, only=range(0, len(lens), max(1, len(lens) // 40)))
    for _ in range(15):
        assert torch.equal(b.call(workspace=ws), out)
    assert not ws[:32768].any()


def test_decode_on_two_streams():
    a, b = Batch([4000, 9, 1300], 32, 8, 128, BF), Batch([2, 5000], 8, 1, 64, HF, seed=5)
    want = a.call(), b.call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(30):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(x.call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for out, w in zip(got, want) for o in out)


def test_two_recorded_decodes_side_by_side():
    """Two graphs recorded on one stream and replayed on two at the same time share no workspace, and eager
    calls run between them."""
    a, b = Batch([9000, 9, 1300], 32, 8, 128, BF), Batch([7000, 20, 3100], 32, 8, 128, BF, seed=5)
    want = a.call(), b.call()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for x in (a, b):
            x.call()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(x.call())
            graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = a.call()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
    a.sl.fill_(0)  # the lengths are read by the replay
    graphs[0].replay()
    torch.cuda.synchronize()
    assert not outs[0].any()
    for graph in graphs:
        graph.reset()


def test_recorded_behind_a_fork():
    """Behind work of two streams, a copy and a fill, with a workspace of the call's own and a given one."""
    b = Batch([4000, 3, 700], 32, 8, 128, BF)
    want = b.call()
    ws = torch.zeros(N.load().fq_dense_paged_decode_workspace_bytes(3, 32, 8, 128), dtype=torch.uint8, device=DEV)
    q, side, main = b.q.clone(), torch.cuda.Stream(), torch.cuda.Stream()
    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            b.q.zero_()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                b.q.copy_(q)
                lens = b.sl + 0
                one = fq.split_k_paged_decode_dense(b.q, b.k, b.v, b.table, lens, workspace=ws)
            two = fq.split_k_paged_decode_dense(q, b.k, b.v, b.table, b.sl)
            main.wait_stream(side)
            three = fq.split_k_paged_decode_dense(b.q, b.k, b.v, b.table, lens, workspace=ws)
            four = three * 1
        for _ in range(10):
            for x in (one, two, three, four):
                x.zero_()
            graph.replay()
            main.synchronize()
            assert all(torch.equal(x, want) for x in (one, two, three, four))
        graph.reset()


def test_recorded_clusters_and_long_prompts():
    """Pieces joined by clusters, and rotary positions of a prompt, in a recorded graph."""
    b = Batch([60000, 2, 9000], 8, 1, 128, HF)
    want = b.call()
    b.check(want)
    q, k = heads(3000, (8, 1), 128, HF, joint=True)
    freq, _ = fq.rotary_frequencies(128, device=DEV)
    pos = torch.randint(0, 9000, (3000,), device=DEV)
    turned_q, turned_k = fq.rotary_embed(q, k, pos, freq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x, y = fq.rotary_embed(q, k, pos, freq)
        out = b.call()
    for _ in range(5):
        out.zero_(), x.zero_(), y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(x, turned_q) and torch.equal(y, turned_k)
    graph.reset()


def test_what_follows_waits_for_all_of_a_decode():
    """A batch of which no unit has to be joined, long enough to be under way when what follows it is launched:
    eager and recorded, the reader of its output sees all of it."""
    b = Batch([16000] * 4 + [1] * 400, 64, 8, 128, BF)
    b.table[:4] = b.table[:1]  # (the long ones share pages)
    b.rows[:4] = [b.rows[0]] * 4
    want = b.call()
    b.check(want, only=[0, 3, 4, 403])
    short = Batch([300] * 200, 16, 16, 64, HF)
    want_short = short.call()
    out, copy = torch.empty_like(want_short), torch.empty_like(want_short)
    for _ in range(30):
        out.fill_(float("nan"))
        short.call(out=out)
        copy.copy_(out)
        assert torch.equal(copy, want_short)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for x, y in ((short, out),):
            y.fill_(float("nan"))
            x.call(out=y)
            copy.copy_(y)
            first = b.call()
            second = first + 0
    for _ in range(20):
        copy.zero_(), second.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(copy, want_short) and torch.equal(second, want)
    graph.reset()


def test_decodes_from_two_threads_on_one_stream():
    a, b = Batch([4000, 9, 1300], 32, 8, 128, BF), Batch([2, 5000, 77], 32, 8, 128, BF, seed=5)
    want = a.call(), b.call()
    torch.cuda.synchronize()
    wrong = []

    def work(x, w):
        outs = [x.call() for _ in range(60)]
        torch.cuda.synchronize()
        wrong.extend(o for o in outs if not torch.equal(o, w))
    threads = [threading.Thread(target=work, args=z) for z in zip((a, b), want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_calls_without_anything_to_do():
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    pages = torch.zeros(2, 16, 8, 128, dtype=BF, device=DEV)
    q = torch.zeros(0, 32, 128, dtype=BF, device=DEV)
    out, lse = fq.split_k_paged_decode_dense(q, pages, pages, none.view(0, 4), none, return_lse=True)
    assert out.shape == (0, 32, 128) and lse.shape == (0, 32)
    freq, _ = fq.rotary_frequencies(128, device=DEV)
    kv = torch.zeros(0, 8, 128, dtype=BF, device=DEV)
    assert [x.shape[0] for x in fq.rotary_embed(q, kv, none, freq)] == [0, 0]
    assert fq.rotary_append_dense(q, kv, kv, pages, pages, none, none, freq).shape == (0, 32, 128)
    q = torch.randn(3, 32, 128, device=DEV).to(BF)  # a block table without columns: no tokens
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert not fq.split_k_paged_decode_dense(q, pages, pages, none.view(3, 0), zero).any()
    heads = torch.zeros(4, 0, 128, dtype=BF, device=DEV)
    x, y = fq.rotary_embed(heads, heads, torch.arange(4, device=DEV), freq)
    assert x.shape == y.shape == (4, 0, 128)
    room = fq.plan_paged_step(none, none, none.view(0, 4), none, zero[:1], 16, 0)
    assert room.cu_seqlens_q.tolist() == [0] and room.slot_mapping.numel() == 0 and int(room.free_count) == 0
    assert int(fq.release_pages(none.bool(), none, none.view(0, 4), none, zero[:1], 16)) == 0


def test_decode_through_ctypes_alone(monkeypatch):
    b = Batch([40, 700], 32, 8, 128, BF)
    want, lse = b.call(return_lse=True)
    monkeypatch.setattr(K, "_host_module", K._ConvertingCalls())
    got = b.call(return_lse=True)
    assert torch.equal(got[0], want) and torch.equal(got[1], lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    graph.reset()


# --------------------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------------------
def turned(x, positions, freq, layout, scale, inverse=False):
    """(values, tolerance) in 64 bits."""
    angle = positions.double()[:, None] * freq.to(x.device)
    cos, sin = angle.cos()[:, None] * scale, angle.sin()[:, None] * scale * (-1 if inverse else 1)
    share = (12 * U + 2 * math.pi * 2.0 ** -51 * (angle.abs() / (2 * math.pi)))[:, None] * scale
    rd, y = 2 * freq.numel(), x.double().clone()
    a, b = (y[..., :rd // 2], y[..., rd // 2:rd]) if layout == "half" else (y[..., 0:rd:2], y[..., 1:rd:2])
    a, b = a.clone(), b.clone()
    tol = torch.zeros_like(y)
    if layout == "half":
        y[..., :rd // 2], y[..., rd // 2:rd] = a * cos - b * sin, b * cos + a * sin
        tol[..., :rd // 2] = tol[..., rd // 2:rd] = (a.abs() + b.abs()) * share
    else:
        y[..., 0:rd:2], y[..., 1:rd:2] = a * cos - b * sin, b * cos + a * sin
        tol[..., 0:rd:2] = tol[..., 1:rd:2] = (a.abs() + b.abs()) * share
    h = half_step(x.dtype)
    tol[..., :rd] = tol[..., :rd] * (1 + h) + h * y[..., :rd].abs() + torch.finfo(x.dtype).smallest_normal * h
    return y, tol


def close(got, want):
    y, tol = want
    off = (got.double() - y).abs()
    assert bool((off <= tol).all()), (off.max().item(), (off / tol.clamp(min=1e-300)).max().item())


def heads(n, h, d, dtype, seed=0, joint=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, sum(h), d, generator=g, device=DEV).to(dtype)
    parts = torch.split(x, h, 1)
    return parts if joint else tuple(p.contiguous() for p in parts)


@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d, rd", [(128, 128), (128, 64), (64, 64), (96, 96), (80, 32), (96, 24), (256, 128), (128, 2), (6, 4),
                                   (128, 0), (5, 4), (7, 0), (9, 6), (1024, 512)])
def test_rotary(dtype, layout, d, rd):
    n = 37
    q, k = heads(n, (6, 2), d, dtype, seed=d + rd, joint=d == 96)
    freq = fq.rotary_frequencies(rd, 500000.0, device=DEV)[0] if rd else torch.zeros(0, dtype=torch.float64, device=DEV)
    pos = torch.randint(0, 1 << 20, (n,), device=DEV)
    for scale, inverse in ((1.0, False), (1.25, True)):
        got = fq.rotary_embed(q, k, pos, freq, layout=layout, scale=scale, inverse=inverse)
        for g, x in zip(got, (q, k)):
            close(g, turned(x, pos, freq, layout, scale, inverse))
            assert torch.equal(g[..., rd:], x[..., rd:])


@pytest.mark.parametrize("n", [1, 2, 591, 593, 3000])
def test_rotary_token_counts_and_position_types(n):
    q, k = heads(n, (32, 8), 128, BF, joint=True)
    freq, scale = fq.rotary_frequencies(128, 10000.0, "yarn", 4.0, 4096, 1.0, 32.0)
    pos = torch.randint(0, 40000, (n,), device=DEV)
    got = fq.rotary_embed(q, k, pos, freq.to(DEV), scale=scale)
    for g, x in zip(got, (q, k)):
        close(g, turned(x, pos, freq, "half", scale))
    other = fq.rotary_embed(q, k, pos.int(), freq, scale=scale)  # (frequencies on the CPU: converted)
    assert torch.equal(other[0], got[0]) and torch.equal(other[1], got[1])
    alone, none = fq.rotary_embed(q, None, pos, freq.to(DEV), scale=scale)
    assert none is None and torch.equal(alone, got[0])


def test_rotary_far_positions():
    q, k = heads(64, (4, 4), 128, torch.float32)
    freq, _ = fq.rotary_frequencies(128, 10000.0, device=DEV)
    pos = torch.randint(1 << 29, 1 << 31, (64,), device=DEV)
    for layout in ("half", "interleaved"):
        for g, x in zip(fq.rotary_embed(q, k, pos, freq, layout=layout), (q, k)):
            close(g, turned(x, pos, freq, layout, 1.0))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_rotary_in_place_padded_and_misaligned(layout, dtype):
    """In place and out of it, rows at odd addresses and of odd strides: the same bits; rows with a negative
    position stay as they are."""
    n, d = 33, 64
    q, k = heads(n, (5, 3), d, dtype)
    freq, _ = fq.rotary_frequencies(48, device=DEV)
    pos = torch.randint(0, 5000, (n,), device=DEV)
    pos[[3, 32]] = -1
    live = pos >= 0
    want = fq.rotary_embed(q, k, pos.clamp(min=0), freq, layout=layout)
    qi, ki = q.clone(), k.clone()
    got = fq.rotary_embed(qi, ki, pos, freq, layout=layout, out=(qi, ki))
    assert got[0] is qi or got[0].data_ptr() == qi.data_ptr()
    for i, w, x in ((qi, want[0], q), (ki, want[1], k)):
        assert torch.equal(i[live], w[live]) and torch.equal(i[~live], x[~live])
    room = torch.zeros(n * 9 * (d + 1) + 1, dtype=dtype, device=DEV)[1:].view(n, 9, d + 1)
    odd_q, odd_k = room[:, :5, :d], room[:, 5:8, 1:]
    odd_q.copy_(q), odd_k.copy_(k)
    got = fq.rotary_embed(odd_q, odd_k, pos.clamp(min=0), freq, layout=layout)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    fq.rotary_embed(odd_q, odd_k, pos, freq, layout=layout, out=(odd_q, odd_k))
    assert torch.equal(odd_q[live], want[0][live]) and torch.equal(odd_k[~live], k[~live])
    assert not room[:, 8].any() and not room[:, :5, d:].any()
    turned_heads = fq.rotary_embed(q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(1, 2).contiguous().transpose(1, 2),
                                   pos.clamp(min=0), freq, layout=layout)
    assert torch.equal(turned_heads[0], want[0]) and torch.equal(turned_heads[1], want[1])


def test_rotary_inverse_is_the_gradient():
    """R^T g is the derivative of <g, R x>: against the formula's, and against differences in 64 bits."""
    x, _ = heads(9, (4, 1), 64, torch.float32)
    g = torch.randn_like(x)
    freq, _ = fq.rotary_frequencies(64, device=DEV)
    pos = torch.randint(0, 3000, (9,), device=DEV)
    for layout in ("half", "interleaved"):
        back, _ = fq.rotary_embed(g, None, pos, freq, layout=layout, scale=1.5, inverse=True)
        y = x.double().requires_grad_()
        turned_y = turned(y, pos, freq, layout, 1.5)[0]
        (grad,) = torch.autograd.grad((turned_y * g.double()).sum(), y)
        tol = turned(g, pos, freq, layout, 1.5, True)[1]
        assert bool(((back.double() - grad).abs() <= tol).all())
        step = torch.randn_like(y)  # linear: one difference is exact but for its rounding in 64 bits
        f = lambda z: (turned(z, pos, freq, layout, 1.5)[0] * g.double()).sum()
        diff = f(y + step) - f(y - step)
        assert abs(float(diff.detach()) / 2 - float((back.double() * step).sum())) <= float((tol * step.abs()).sum()) + 1e-9


def test_rotary_refusals():
    q, k = heads(5, (4, 2), 64, BF)
    freq, _ = fq.rotary_frequencies(64, device=DEV)
    pos = torch.arange(5, device=DEV)
    ok = dict(q=q, k=k, positions=pos, frequencies=freq)

    def refused(error=ValueError, **kw):
        with pytest.raises(error):
            fq.rotary_embed(**{**ok, **kw})
    refused(layout="neither")
    refused(positions=pos[:4])
    refused(positions=pos.float())
    refused(frequencies=torch.ones(33, device=DEV))
    refused(k=k[:4])
    refused(k=k.half())
    refused(k=k[..., :32])
    refused(TypeError, q=q.double())
    refused(out=(q, k[:, :1]))
    refused(out=(torch.zeros(1, 1, 64, dtype=BF, device=DEV).expand(5, 4, 64), k))
    refused(k=None, out=(q, k))
    refused(N.FlashQuantNativeError, positions=pos.cpu())


# --------------------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("pages", ["two", "token", "heads", "odd"])
@pytest.mark.parametrize("n, hq, hkv, d, rd", [(1, 32, 8, 128, 128), (700, 8, 1, 64, 32), (45, 6, 3, 96, 96), (33, 2, 2, 256, 64)])
def test_append(dtype, layout, pages, n, hq, hkv, d, rd):
    q, k, v = heads(n, (hq, hkv, hkv), d, dtype, joint=n != 45)
    block = 32
    total = -(-2 * n // block) + 1
    shape = {"two": (2, total, block, hkv, d), "token": (total, block, 2, hkv, d), "heads": (2, total, hkv, block, d),
             "odd": (2, total, block, hkv, d + 1)}[pages]
    buf = torch.zeros(shape, dtype=dtype, device=DEV)
    if pages == "token":
        kc, vc = buf[:, :, 0], buf[:, :, 1]
    elif pages == "heads":
        kc, vc = (x.transpose(1, 2) for x in buf)
    else:
        kc, vc = buf[0][..., :d], buf[1][..., :d]
    freq, scale = fq.rotary_frequencies(rd, 10000.0, "linear", 2.0, device=DEV)
    pos = torch.randint(0, 1 << 17, (n,), device=DEV)
    slots = torch.randperm(total * block, device=DEV)[:n]
    slots[n // 2:n // 2 + 3:2] = -1
    if n > 1:
        slots[n - 1], pos[0] = total * block, -1
    stored = (slots >= 0) & (slots < total * block)
    q_old = q.clone()
    got = fq.rotary_append_dense(q, k, v, kc, vc, slots, pos, freq, layout=layout, scale=scale)
    live = pos >= 0
    wq, wk = fq.rotary_embed(q, k, pos.clamp(min=0), freq, layout=layout, scale=scale)
    close(wk, turned(k, pos.clamp(min=0), freq, layout, scale))
    assert torch.equal(got[live], wq[live]) and torch.equal(q, q_old)
    want_k, want_v = torch.zeros(total * block, hkv, d, dtype=dtype, device=DEV), torch.zeros(total * block, hkv, d, dtype=dtype, device=DEV)
    want_k[slots[stored & live]], want_v[slots[stored]] = wk[stored & live], v[stored]
    assert torch.equal(kc.reshape(-1, hkv, d), want_k) and torch.equal(vc.reshape(-1, hkv, d), want_v)
    if pages == "odd":
        assert not buf[..., d:].any()
    # 32-bit slots and positions, q in place, the converting path
    buf.zero_()
    joint = q.clone()
    back = fq.rotary_append_dense(joint, k, v, kc, vc, slots.int(), pos.int(), freq.cpu(), layout=layout, scale=scale, q_out=joint)
    assert back is joint and torch.equal(joint[live], wq[live]) and torch.equal(joint[~live], q[~live])
    assert torch.equal(kc.reshape(-1, hkv, d), want_k) and torch.equal(vc.reshape(-1, hkv, d), want_v)


def test_append_without_rotation():
    k, v = heads(20, (4, 4), 128, BF)
    kc, vc = (torch.zeros(3, 16, 4, 128, dtype=BF, device=DEV) for _ in range(2))
    slots = torch.randperm(48, device=DEV)[:20]
    assert fq.rotary_append_dense(None, k, v, kc, vc, slots) is None
    assert torch.equal(kc.view(48, 4, 128)[slots], k) and torch.equal(vc.view(48, 4, 128)[slots], v)
    assert int((kc.view(48, -1).abs().sum(1) > 0).sum()) == 20
    freq, _ = fq.rotary_frequencies(128, device=DEV)
    pos = torch.arange(20, device=DEV)
    assert fq.rotary_append_dense(None, k, v, kc, vc, slots, pos, freq) is None
    close(kc.view(48, 4, 128)[slots], turned(k, pos, freq, "half", 1.0))


def test_append_offsets_beyond_32_bits():
    blocks = (1 << 31) // (16 * 8 * 128) + 10
    kc, vc = (torch.empty(blocks, 16, 8, 128, dtype=BF, device=DEV) for _ in range(2))
    q, k, v = heads(4, (8, 8, 8), 128, BF)
    slots = torch.tensor([blocks * 16 - 1, 5, blocks * 16 - 40, 0], device=DEV)
    freq, _ = fq.rotary_frequencies(128, device=DEV)
    pos = torch.arange(4, device=DEV)
    fq.rotary_append_dense(q, k, v, kc, vc, slots, pos, freq)
    assert torch.equal(vc.view(-1, 8, 128)[slots], v)
    assert torch.equal(kc.view(-1, 8, 128)[slots], fq.rotary_embed(k, None, pos, freq)[0])


def test_append_refusals():
    q, k, v = heads(5, (8, 4, 4), 64, BF)
    kc, vc = (torch.zeros(3, 16, 4, 64, dtype=BF, device=DEV) for _ in range(2))
    freq, _ = fq.rotary_frequencies(64, device=DEV)
    i = torch.arange(5, device=DEV)
    ok = dict(q=q, key=k, value=v, key_cache=kc, value_cache=vc, slot_mapping=i, positions=i, frequencies=freq)

    def refused(error=ValueError, **kw):
        with pytest.raises(error):
            fq.rotary_append_dense(**{**ok, **kw})
    refused(value=v[:, :2])
    refused(key_cache=kc[:, :, :2])
    refused(value_cache=vc[:2])
    refused(key_cache=kc.half())
    refused(key_cache=kc[:, :1].expand(3, 16, 4, 64))
    refused(value_cache=vc.as_strided((3, 16, 4, 64), (4096, 64, 64, 1)))
    refused(slot_mapping=i[:3])
    refused(slot_mapping=i.float())
    refused(positions=None)
    refused(frequencies=None)
    refused(positions=None, frequencies=None)
    refused(q=None, q_out=q)
    refused(q=q[:, :, :32])
    refused(TypeError, q=q.float(), key=k.float(), value=v.float(), key_cache=kc.float(), value_cache=vc.float())
    refused(N.FlashQuantNativeError, slot_mapping=i.cpu())


# --------------------------------------------------------------------------------------
# step plans
# --------------------------------------------------------------------------------------
def plan_oracle(context, query, table, free, count, block, room):
    """Request by request."""
    table, width = [list(r) for r in table], len(table[0]) if table else 0
    lens, cu, slots, pos, served = [], [0], [], [], []
    height, closed = count, False
    for i, (c, n) in enumerate(zip(context, query)):
        valid = c >= 0 and n >= 0 and -(-(c + n) // block) <= width
        fresh = range(-(-c // block), -(-(c + n) // block)) if valid and n else range(0)
        if valid and n and (len(fresh) > height or len(slots) + n > room):
            closed = True
        ok = valid and (n == 0 or not closed)
        if ok and n:
            for page in fresh:
                height -= 1
                table[i][page] = free[height]
            for at in range(c, c + n):
                slots.append(table[i][at // block] * block + at % block)
                pos.append(at)
        served.append(ok)
        lens.append(min(max(c, 0), width * block) + (n if ok else 0))
        cu.append(len(slots))
    pad = [-1] * (room - len(slots))
    return table, lens, cu, slots + pad, pos + pad, served, height


def plan_case(rng, requests, width, block, new, blocks, tight=1.0):
    context = [rng.randint(0, max(0, width * block - 2)) for _ in range(requests)]
    query = [rng.choice([0, 1, 1, min(new, width * block - c)]) if new > 1 else 1 for c in context]
    ids = list(range(blocks))
    rng.shuffle(ids)
    table = [[-1] * width for _ in range(requests)]
    for row, c in zip(table, context):
        for j in range(-(-c // block)):
            row[j] = rng.randrange(blocks)
    grow = sum(max(0, -(-(c + n) // block) - -(-c // block)) for c, n in zip(context, query))
    count = min(blocks, int(grow * tight))
    return context, query, table, ids, count


def run_plan(context, query, table, free, count, block, room, in_place=False):
    i32 = dict(dtype=torch.int32, device=DEV)
    t = torch.tensor(table, **i32).view(len(context), -1) if table else torch.zeros(0, 4, **i32)
    height = torch.tensor([count], **i32)
    p = fq.plan_paged_step(torch.tensor(context, **i32), torch.tensor(query, **i32), t, torch.tensor(free, **i32), height,
                           block, room, free_count_out=height if in_place else None)
    assert in_place or int(height) == count
    assert [x.dtype for x in p] == [torch.int32, torch.int32, torch.int64, torch.int64, torch.bool, torch.int32]
    return (t.tolist(), *(x.tolist() for x in p[:5]), int(p.free_count))


@pytest.mark.parametrize("requests", [1, 2, 33, 511, 512, 513, 1500, 4096])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("tight", [1.0, 0.6])
def test_plan(requests, new, tight):
    rng = random.Random(requests * new)
    for block in (16, 1, 24):
        context, query, table, free, count = plan_case(rng, requests, 8, block, new, 3000, tight)
        total = sum(query)
        for room in {total + 5, total, int(total * tight)}:
            want = plan_oracle(context, query, table, free, count, block, room)
            got = run_plan(context, query, table, free, count, block, room, in_place=room == total)
            for g, w in zip(got, want):
                assert g == w


def test_plan_at_its_edges():
    free = list(range(100, 164))
    cases = [([], [], [], 64, 16, 8), ([0], [0], [[7, 7]], 64, 16, 4), ([0], [32], [[7, 7]], 64, 16, 32),
             ([0], [33], [[7, 7]], 64, 16, 40), ([-1, 5], [3, 2], [[1, 2], [3, 4]], 64, 16, 9),
             ([5, 5], [-2, 2], [[1, 2], [3, 4]], 64, 16, 9), ([2 ** 31 - 1, 1], [2 ** 31 - 1, 1], [[1, 2], [3, 4]], 64, 16, 9),
             ([16, 0, 16], [1, 0, 1], [[1, 2], [3, 4], [5, 6]], 1, 16, 9), ([16, 3, 0], [1, 1, 0], [[1, 2], [3, 4], [5, 6]], 0, 16, 9),
             ([0, 1], [5, 1], [[1, 2], [3, 4]], 64, 16, 0), ([0, 1], [5, 1], [[1, 2], [3, 4]], 64, 16, 4),
             ([1000], [2], [[1, 2]], 64, 16, 4), ([31, 40], [1, 0], [[1, 2], [3, 4]], 64, 16, 4)]
    for context, query, table, count, block, room in cases:
        got = run_plan(context, query, table, free, count, block, room)
        want = plan_oracle(context, query, table, free, count, block, room)
        assert got == tuple(want) or (not table and got[1:] == tuple(want)[1:]), (context, query, got, want)
    # a height outside the stack is cut to it
    assert run_plan([0], [20], [[1, 2]], [9, 8, 7], 1000, 16, 20)[0] == [[7, 8]]
    assert run_plan([0], [20], [[1, 2]], [9, 8, 7], -4, 16, 20)[5] == [False]


@pytest.mark.parametrize("requests, width, block", [(1, 3, 16), (40, 8, 16), (700, 9, 1), (4096, 5, 32)])
def test_release_and_plan_again(requests, width, block):
    rng = random.Random(requests)
    context, _, table, _, _ = plan_case(rng, requests, width, block, 1, 3000)
    table = [[rng.randrange(1 << 20) for _ in r] for r in table]
    if requests > 3:
        context[1], context[2] = -3, width * block + 1000
    done = [rng.random() < 0.4 for _ in context]
    pages = [row[:max(0, min(-(-c // block), width))] if f else [] for c, row, f in zip(context, table, done)]
    flat = [p for r in pages for p in r]
    i32 = dict(dtype=torch.int32, device=DEV)
    for start, capacity in ((5, 5 + len(flat)), (0, len(flat) + 9), (5, 5 + len(flat) // 2), (3, 1 << 16)):
        free = torch.full((capacity,), -7, **i32)
        height = torch.tensor([start], **i32)
        args = torch.tensor(done, device=DEV), torch.tensor(context, **i32), torch.tensor(table, **i32)
        out = fq.release_pages(*args, free, height, block)
        kept = flat[:capacity - start]
        assert int(out) == start + len(kept) and int(height) == start
        assert free.tolist() == [-7] * start + kept + [-7] * (capacity - start - len(kept))
        assert fq.release_pages(args[0], args[1].long(), args[2], free, height, block, free_count_out=height) is height
        assert int(height) == start + len(kept)
    # what was released is what the next step takes, last in first out
    height = torch.tensor([start + len(flat)], **i32)
    if flat:
        t = torch.zeros(1, width, **i32)
        zero = torch.zeros(1, **i32)
        fq.plan_paged_step(zero, zero + 1, t, free, height, block, 4, free_count_out=height)
        assert t[0, 0].item() == flat[-1] and int(height) == start + len(flat) - 1


def test_plan_views_and_refusals():
    i32 = dict(dtype=torch.int32, device=DEV)
    wide = torch.full((3, 10), 5, **i32)
    free, one = torch.arange(40, **i32), torch.tensor([40], **i32)
    context, query = torch.tensor([0, 17, 3], **i32), torch.tensor([17, 0, 20], **i32)
    plain = wide[:, :4].contiguous()
    a = fq.plan_paged_step(context, query, plain, free, one, 16, 50)
    b = fq.plan_paged_step(context.long(), torch.stack([query, query], 1)[:, 0], wide[:, :4], free, one, 16, 50)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(wide[:, :4], plain) and bool((wide[:, 4:] == 5).all())
    ok = dict(context_lens=context, query_lens=query, block_table=plain, free_blocks=free, free_count=one, block_size=16, max_tokens=50)

    def refused(error=ValueError, **kw):
        with pytest.raises(error):
            fq.plan_paged_step(**{**ok, **kw})
    refused(context_lens=context[:2])
    refused(query_lens=query.float())
    refused(block_table=plain.long())
    refused(block_table=plain.t())
    refused(block_table=plain[:1].expand(3, 4))
    refused(free_blocks=free.view(2, 20))
    refused(free_count=free)
    refused(free_count_out=one.long())
    refused(max_tokens=-1)
    refused(block_size=0)
    refused(N.FlashQuantNativeError, block_table=plain.cpu())
    with pytest.raises(ValueError):
        fq.release_pages(context, context, plain, free, one, 16)


# --------------------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("recorded", [False, True])
def test_steps_of_a_batch(consts, recorded):
    """Prompts, then decode steps: plan, rotary positions and append, attention, for a layer of 16-bit pages and a
    compressed one over the same block tables.  The first against attention over all keys in 64 bits, the second
    against the same calls with tables made on the host.  Eager, and the decode steps as one recorded graph."""
    n, hq, hkv, d, block, width, dtype = 5, 32, 8, 128, 16, 20, BF
    i32 = dict(dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    rot, bk, bv, ck, cv = (consts[x].contiguous().to(DEV) for x in (
        "rotation_128_0", "boundaries_128_3", "boundaries_128_4", "centroids_128_3", "centroids_128_4"))
    blocks = 64
    kc, vc = (torch.full((blocks, block, hkv, d), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    packed, packed_host = (torch.zeros(blocks, block, hkv * (d + 8), dtype=torch.uint8, device=DEV) for _ in range(2))
    freq, scale = fq.rotary_frequencies(d, 500000.0, "wavelength", 4.0, device=DEV)
    table, free = torch.zeros(n, width, **i32), torch.randperm(blocks, generator=g, device=DEV).int()
    height, context = torch.tensor([blocks], **i32), torch.zeros(n, **i32)
    seen = [[[], []] for _ in range(n)]          # rotated keys, values of each request
    prompt = [17, 1, 90, 16, 130]
    qkv = torch.zeros(300, hq + 2 * hkv, d, dtype=dtype, device=DEV)
    step_q = torch.zeros(n, hq, d, dtype=dtype, device=DEV)
    query = torch.tensor(prompt, **i32)

    def append(room):
        plan = fq.plan_paged_step(context, query, table, free, height, block, room, free_count_out=height)
        q, k, v = (x[:room] for x in torch.split(qkv, (hq, hkv, hkv), 1))
        q = fq.rotary_append_dense(q, k, v, kc, vc, plan.slot_mapping, plan.positions, freq, scale=scale)
        _, turned_k = fq.rotary_embed(q, k, plan.positions, freq, scale=scale)
        fq.tq4_compress_append(turned_k, v, packed, plan.slot_mapping, rot, bk, bv)
        context.copy_(plan.seq_lens)
        return plan, q, turned_k

    def decode():
        plan, q, turned_k = append(n)
        step_q.copy_(q)
        return (plan, q, turned_k, fq.split_k_paged_decode_dense(step_q, kc, vc, table, plan.seq_lens),
                fq.split_k_paged_decode(step_q, packed, table, plan.seq_lens, ck, cv, rot, hkv, d, block))

    qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV))
    plan, q, turned_k = append(300)
    assert plan.served.all() and plan.cu_seqlens_q.tolist() == [0, 17, 18, 108, 124, 254] and int(plan.slot_mapping[254]) == -1
    total = sum(prompt)
    for i in range(n):
        lo, hi = plan.cu_seqlens_q[i].item(), plan.cu_seqlens_q[i + 1].item()
        seen[i][0].append(turned_k[lo:hi].clone())
        seen[i][1].append(qkv[lo:hi, hq + hkv:].clone())
    query.fill_(1)
    graph, made = None, None
    if recorded:
        keep = [x.clone() for x in (context, table, height, kc, vc, packed)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                made = decode()
        torch.cuda.synchronize()
        for x, y in zip((context, table, height, kc, vc, packed), keep):
            x.copy_(y)
    for step in range(20):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV))
        if recorded:
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
        else:
            made = decode()
        plan, q, turned_k, out, out4 = made
        assert plan.served.all() and context.tolist() == [p + step + 1 for p in prompt]
        for i in range(n):
            seen[i][0].append(turned_k[i:i + 1].clone())
            seen[i][1].append(qkv[i:i + 1, hq + hkv:].clone())
            at = torch.arange(context[i].item(), device=DEV)
            slots = table[i][at // block].long() * block + at % block
            keys, values = (torch.cat(x) for x in seen[i])
            assert torch.equal(kc.view(-1, hkv, d)[slots], keys) and torch.equal(vc.view(-1, hkv, d)[slots], values)
            assert plan.slot_mapping[i].item() == slots[-1].item() and plan.positions[i].item() == at[-1].item()
        if step % 5 == 0:
            b = Batch.__new__(Batch)
            b.lens, b.hq, b.hkv, b.d, b.k, b.v, b.q = context.tolist(), hq, hkv, d, kc, vc, q
            b.rows = [(table[i][torch.arange(m, device=DEV) // block].long(), torch.arange(m, device=DEV) % block)
                      for i, m in enumerate(b.lens)]
            b.check(out)
            host_table = torch.zeros(n, width, **i32)
            packed_host.zero_()
            at = 0
            for i in range(n):
                pages = -(-b.lens[i] // block)
                host_table[i, :pages] = torch.arange(at, at + pages, **i32)
                at += pages
                tok = torch.arange(b.lens[i], device=DEV)
                slots = host_table[i][tok // block].long() * block + tok % block
                packed_host.view(-1, packed.shape[2])[slots] = packed.view(-1, packed.shape[2])[table[i][tok // block].long() * block + tok % block]
            again = fq.split_k_paged_decode(q.contiguous(), packed_host, host_table, context, ck, cv, rot, hkv, d, block)
            assert torch.equal(out4, again)
    pages = sum(-(-(p + 20) // block) for p in prompt)
    assert height.item() == blocks - pages
    done = torch.tensor([True] * n, device=DEV)
    fq.release_pages(done, context, table, free, height, block, free_count_out=height)
    assert height.item() == blocks and sorted(free.tolist()) == list(range(blocks))
    if graph is not None:
        graph.reset()
