"""Calls around 16-bit pages that a program may make and the other tests do not: tolerances are those of
test_gpu_dense.py, most comparisons are of bits."""

import threading

import pytest
import torch

import flashquant_b200 as fq
from flashquant_b200 import _native as N
from flashquant_b200 import kernels as K
from test_gpu_dense import BF, DEV, HF, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("seqs", [3, 700])
def test_lengths_written_right_before_the_call(seqs, recorded):
    """Both kernels of a decode go by the lengths that the kernel before the call has written, not by older ones."""
    g = torch.Generator().manual_seed(seqs)
    longest = 6000 if seqs == 3 else 90
    b = Batch([longest] * seqs, 32, 8, 128, BF, spare=0)
    lens = torch.randint(0, longest + 1, (12, seqs), generator=g).int().to(DEV)
    want = []
    for n in lens:
        b.sl.copy_(n)
        torch.cuda.synchronize()
        want.append(b.call(return_lse=True))
        torch.cuda.synchronize()
    source = torch.empty_like(b.sl)
    copied = lambda: (b.sl.copy_(source), b.call(return_lse=True))[1]
    graph = None
    if recorded:
        source.copy_(lens[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = copied()
    for step in range(60):
        source.copy_(lens[step % 12])
        if recorded:
            graph.replay()
        else:
            made = copied()
        for x, w in zip(made, want[step % 12]):
            assert torch.equal(x, w)
    if graph is not None:
        graph.reset()


@pytest.mark.parametrize("paths", ["both converted", "one converted"])
def test_decodes_of_converted_arguments_from_two_threads(monkeypatch, paths):
    """Calls whose arguments are converted (a whole number for the scale, lengths a column of a table) share the stream's
    workspace with those of other threads like all others."""
    a, b = Batch([4000, 9, 1300], 32, 8, 128, BF), Batch([2, 5000, 77], 32, 8, 128, BF, seed=5)
    b.sl = torch.stack([b.sl, b.sl], 1)[:, 0]
    want = a.call(sm_scale=1.0), b.call()
    torch.cuda.synchronize()
    if paths == "both converted":
        monkeypatch.setattr(K, "_host_module", K._ConvertingCalls())
    wrong = []

    def work(x, w, kw):
        outs = [x.call(**kw) for _ in range(300)]
        torch.cuda.synchronize()
        wrong.extend(o for o in outs if not torch.equal(o, w))
    threads = [threading.Thread(target=work, args=z)
               for z in zip((a, b), want, (dict(sm_scale=1 if paths == "both converted" else 1.0), {}))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63])
def test_windows_beyond_32_bits_see_all(window):
    b = Batch([40, 700, 9], 32, 8, 128, BF)
    want = b.call()
    b.window = window
    assert torch.equal(b.call(), want)


I32 = dict(dtype=torch.int32, device=DEV)


def test_lengths_beyond_32_bits_are_too_long():
    """64-bit lengths that do not fit into 32 bits: more pages than a row holds (or negative), not what their low bits say."""
    table = torch.tensor([[3, 4], [5, 6], [7, 8], [9, 10], [11, 12]], **I32)
    context = torch.tensor([2 ** 32 + 3, 0, -2 ** 32 + 3, 2, 2 ** 31 + 1], device=DEV)
    query = torch.tensor([1, 2 ** 32 + 1, 1, 1, 0], device=DEV)
    free, height = torch.arange(50, 60, **I32), torch.tensor([10], **I32)
    plan = fq.plan_paged_step(context, query, table.clone(), free, height, 16, 8)
    assert plan.served.tolist() == [False, False, False, True, False]
    assert plan.cu_seqlens_q.tolist() == [0, 0, 0, 0, 1, 1] and plan.slot_mapping.tolist() == [9 * 16 + 2] + [-1] * 7
    assert plan.seq_lens.tolist() == [32, 0, 0, 3, 32] and int(plan.free_count) == 10
    done = torch.ones(5, dtype=torch.bool, device=DEV)
    stack = torch.full((20,), -1, **I32)
    out = fq.release_pages(done, context, table, stack, torch.zeros(1, **I32), 16)
    assert int(out) == 5 and stack[:5].tolist() == [3, 4, 9, 11, 12]


@pytest.mark.parametrize("recorded", [False, True])
def test_a_step_that_not_every_request_takes_part_in(consts, recorded):
    """Requests that are finished, wait or are not served stand between others: rows of tokens are compact, those of the
    decodes are not.  Each token's row is that of its request in a call whose rows a list has put in their places."""
    r, hq, hkv, d, block, width, room = 7, 32, 8, 128, 16, 8, 5
    g = torch.Generator(device=DEV).manual_seed(4)
    rot, bk, bv, ck, cv = (consts[x].contiguous().to(DEV) for x in (
        "rotation_128_0", "boundaries_128_3", "boundaries_128_4", "centroids_128_3", "centroids_128_4"))
    blocks = 64
    kc, vc = (torch.randn(blocks, block, hkv, d, generator=g, device=DEV).to(BF) for _ in range(2))
    packed = torch.zeros(blocks, block, hkv * (d + 8), dtype=torch.uint8, device=DEV)
    every = torch.arange(blocks * block, device=DEV)
    fq.tq4_compress_append(kc.view(-1, hkv, d), vc.view(-1, hkv, d), packed, every, rot, bk, bv)
    table0 = torch.randperm(blocks, generator=g, device=DEV).int()[:r * width].view(r, width).contiguous()
    free = torch.arange(56, 64, **I32)
    freq, scale = fq.rotary_frequencies(d, device=DEV)
    context, query, height, table = torch.zeros(r, **I32), torch.zeros(r, **I32), torch.zeros(1, **I32), table0.clone()
    qkv = torch.randn(room, hq + 2 * hkv, d, generator=g, device=DEV).to(BF)
    tokens = torch.arange(room, **I32)

    def step():
        plan = fq.plan_paged_step(context, query, table, free, height, block, room, free_count_out=height)
        first = plan.cu_seqlens_q[:-1].clamp(max=room - 1)
        owner = torch.searchsorted(plan.cu_seqlens_q[1:], tokens, right=True).clamp(max=r - 1)
        q, k, v = torch.split(qkv, (hq, hkv, hkv), 1)
        rq, rk = fq.rotary_embed(q, k, plan.positions, freq, scale=scale)
        fq.tq4_compress_append(rk, v, packed, plan.slot_mapping, rot, bk, bv)
        out4 = fq.split_k_paged_decode(rq[first], packed, table, plan.seq_lens, ck, cv, rot, hkv, d, block)[owner]
        q = fq.rotary_append_dense(q, k, v, kc, vc, plan.slot_mapping, plan.positions, freq, scale=scale)
        out = fq.split_k_paged_decode_dense(q[first], kc, vc, table, plan.seq_lens)[owner]
        return plan, q, out4, out

    # contexts, new tokens, pages left; who is served with a token
    cases = [([5, 17, 40, 3, 90, 60, 33], [0, 1, 0, 1, 1, 0, 1], 8, [1, 3, 4, 6]),
             ([5, 16, 40, 3, 96, 60, 33], [1, 1, 0, 1, 1, 0, 1], 1, [0, 1, 3]),   # no page for the fifth
             ([5, 17, 40, 3, 90, 60, 33], [1, 1, 1, 1, 1, 1, 1], 8, [0, 1, 2, 3, 4]),  # no row for the sixth
             ([5, -1, 128, 3, 90, 60, 33], [1, 1, 1, 0, 0, 1, 0], 8, [0, 5]),     # one is no request, one is full
             ([5, 17, 40, 3, 90, 60, 33], [0] * 7, 8, [])]
    graph = None
    if recorded:
        context.fill_(1)
        query[:room].fill_(1)
        height.fill_(8)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                made = step()
        torch.cuda.synchronize()
    for lens, new, pages, served in cases * 2:
        context.copy_(torch.tensor(lens)), query.copy_(torch.tensor(new)), height.fill_(pages), table.copy_(table0)
        torch.cuda.synchronize()
        if recorded:
            graph.replay()
            torch.cuda.synchronize()
        else:
            made = step()
        plan, q, out4, out = made
        assert [i for i in range(r) if plan.served[i] and new[i]] == served
        each = torch.zeros(r, hq, d, dtype=BF, device=DEV)  # a row a request, by the list
        for row, i in enumerate(served):
            assert int(plan.seq_lens[i]) == lens[i] + 1 and int(plan.positions[row]) == lens[i]
            each[i] = q[row]
        want = fq.split_k_paged_decode_dense(each, kc, vc, table, plan.seq_lens)
        want4 = fq.split_k_paged_decode(each, packed, table, plan.seq_lens, ck, cv, rot, hkv, d, block)
        assert torch.equal(out[:len(served)], want[served]) and torch.equal(out4[:len(served)], want4[served])
    if graph is not None:
        graph.reset()


def test_status_of_replays():
    """A recorded call leaves its status in the workspace it was given; the stream's own says nothing of it."""
    b = Batch([40, 700], 32, 8, 128, BF)
    want = b.call()
    stream = fq.dense_workspace(DEV, 2, 32, 8, 128)
    ws = torch.zeros_like(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        given, own = b.call(workspace=ws), b.call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(given, want) and torch.equal(own, want) and K.workspace_status(ws) == 0
    page = int(b.table[0, 1])
    b.table[0, 1] = b.k.shape[0]
    graph.replay()
    assert K.workspace_status(ws, reset=True) == N.FQ_DEV_BAD_BLOCK_INDEX and K.workspace_status(stream) == 0
    assert torch.equal(given, own) and torch.equal(given[1], want[1])
    b.table[0, 1] = page
    graph.replay()
    assert K.workspace_status(ws) == 0 and torch.equal(given, want) and not ws[:32768].any()
    graph.reset()


@pytest.mark.parametrize("converted", [False, True])
def test_workspaces_are_as_large_as_they_have_to_be(monkeypatch, converted):
    """Heads of another kind take a workspace of their own size, not twice the one before."""
    if converted:
        monkeypatch.setattr(K, "_host_module", K._ConvertingCalls())
    need = lambda *heads: N.load().fq_dense_paged_decode_workspace_bytes(1, *heads)
    small, large = sorted([(16, 1, 256), (16, 1, 64)], key=lambda h: need(*h))
    with torch.cuda.stream(torch.cuda.Stream()):
        for heads, size in ((small, need(*small)), (large, need(*large)), (small, need(*large))):  # (the larger one stays)
            b = Batch([50, 3000], *heads, HF)
            b.check(b.call())
            assert fq.dense_workspace(DEV, 2, *heads).numel() == size
        ws = fq.dense_workspace(DEV, 2, *large)
        assert ws.numel() == need(*large) and not ws[:32768].any()
        torch.cuda.current_stream().synchronize()


@pytest.mark.parametrize("hq, hkv, d", [(32, 8, 128), (64, 8, 128), (8, 1, 64), (128, 8, 128)])
@pytest.mark.parametrize("n", [65, 296, 444, 445, 593, 888, 889, 1185])
def test_rotary_around_the_bounds_of_its_rule(hq, hkv, d, n):
    """However many tokens are taken at a time: the bits of a few tokens alone."""
    x = torch.randn(n, hq + hkv, d, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV).to(BF)
    q, k = torch.split(x, (hq, hkv), 1)
    freq, _ = fq.rotary_frequencies(d, device=DEV)
    pos = torch.randint(0, 1 << 17, (n,), device=DEV)
    got = fq.rotary_embed(q, k, pos, freq)
    for i in range(0, n, 64):
        part = fq.rotary_embed(q[i:i + 64], k[i:i + 64], pos[i:i + 64], freq)
        assert all(torch.equal(g[i:i + 64], w) for g, w in zip(got, part))


@pytest.mark.parametrize("converted", [1, 2])
def test_compressed_attention_of_converted_arguments_from_two_threads(consts, converted):
    """Attention over a compressed cache: calls of one thread, or of both, go through the conversion."""
    bnd, c, rot = (consts[n].contiguous().to(DEV) for n in ("boundaries_128_4", "centroids_128_4", "rotation_128_0"))
    cases = []
    for i in range(2):
        x = torch.randn(2 * 8 * 600, 1, 128, device=DEV, generator=torch.Generator(DEV).manual_seed(i)).half()
        p, n = fq.tq4_compress(x, rot, bnd)
        q = torch.randn(2, 32, 1, 128, device=DEV).half()
        args = (q, p.view(2, 8, 600, 64), n.view(2, 8, 600, 1), p.view(2, 8, 600, 64), n.view(2, 8, 600, 1), c, c, rot)
        want = fq.fused_tq_attention(*args, sm_scale=1.0)
        cases.append((args, 1 if i < converted else 1.0, want))
    torch.cuda.synchronize()
    wrong = []

    def run(args, scale, want):
        outs = [fq.fused_tq_attention(*args, sm_scale=scale) for _ in range(300)]
        wrong.extend(i for i, o in enumerate(outs) if not torch.equal(o, want))
    threads = [threading.Thread(target=run, args=case) for case in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("hq, hkv, d", [(2, 2, 256), (16, 1, 256), (8, 8, 128), (4, 1, 64), (6, 2, 96)])
def test_as_many_sequences_as_a_call_takes(hq, hkv, d):
    lens = [(7 * i) % 40 for i in range(2047)] + [3000]
    b = Batch(lens, hq, hkv, d, HF)
    out, lse = b.call(return_lse=True)
    b.check(out, lse, only=[0, 1, 2, 40, 777, 2040, 2046, 2047])
    assert not out.isnan().any() and not out[::40].any()
    b.sl.zero_()
    assert not b.call().any()


@pytest.mark.parametrize("hq, hkv", [(1024, 1), (1024, 1024), (1000, 8), (17, 17)])
def test_as_many_heads_as_a_call_takes(hq, hkv):
    b = Batch([40, 0, 1, 500], hq, hkv, 64, BF)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


def test_rotary_offsets_beyond_32_bits():
    n, hq, d = (1 << 31) // (32 * 128) + 300, 32, 128
    q = torch.empty(n, hq, d, dtype=BF, device=DEV)
    q[-400:] = torch.randn(400, hq, d, device=DEV).to(BF)
    q[:-400] = 0
    freq, _ = fq.rotary_frequencies(d, device=DEV)
    pos = torch.arange(n, device=DEV)
    want, _ = fq.rotary_embed(q[-400:].clone(), None, pos[-400:], freq)
    got, _ = fq.rotary_embed(q, None, pos, freq)
    assert torch.equal(got[-400:], want) and not got[:-400].any()
    fq.rotary_embed(q, None, pos, freq, out=(q, None))
    assert torch.equal(q[-400:], want) and not q[:-400].any()


@pytest.mark.parametrize("requests", [3, 900])
def test_recorded_plans_in_place(requests):
    """A plan and a release that update the stack's height in place, replayed with other lengths: large enough for several
    CTAs, the pages are those that the calls take when they are made one by one."""
    width, block, blocks, room = 40, 16, 40000, 9000
    g = torch.Generator().manual_seed(requests)
    context, query = torch.zeros(requests, **I32), torch.zeros(requests, **I32)
    done, table = torch.zeros(requests, dtype=torch.bool, device=DEV), torch.zeros(requests, width, **I32)
    free, height = torch.randperm(blocks, generator=g).int().to(DEV), torch.tensor([blocks], **I32)
    state = [table, free, height]

    def step():
        plan = fq.plan_paged_step(context, query, table, free, height, block, room, free_count_out=height)
        fq.release_pages(done, plan.seq_lens, table, free, height, block, free_count_out=height)
        return plan
    graph = torch.cuda.CUDAGraph()
    step()  # (nothing is asked for)
    with torch.cuda.graph(graph):
        made = step()
    for i in range(8):
        new = torch.randint(0, 600, (requests,), generator=g).int().to(DEV)
        query.copy_(torch.where((context + new) <= width * block, new, torch.zeros_like(new)))
        done.copy_(torch.rand(requests, generator=g) < 0.4)
        before = [x.clone() for x in state]
        plan = step()
        want = [x.clone() for x in (*plan, *state)]
        for x, y in zip(state, before):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((*made, *state), want):
            assert torch.equal(x, y)
        context.copy_(torch.where(done, torch.zeros_like(context), plan.seq_lens))
        held = int(((context + block - 1) // block).sum())
        assert int(height) == blocks - held and plan.served.any()
        mine = [table[r, :(int(context[r]) + block - 1) // block] for r in range(requests)]
        assert torch.equal(torch.cat([*mine, free[:int(height)]]).sort().values, torch.arange(blocks, **I32))
    graph.reset()


def test_results_take_part_in_what_follows():
    """Results that share one allocation: under inference mode, as inputs of a gradient, one of them kept alone."""
    q, k = (torch.randn(9, h, 128, device=DEV).to(BF) for h in (8, 2))
    freq, _ = fq.rotary_frequencies(128, device=DEV)
    pos = torch.arange(9, device=DEV)
    a, b = fq.rotary_embed(q, k, pos, freq)
    with torch.inference_mode():
        c, d = fq.rotary_embed(q, k, pos, freq)
        assert torch.equal(a, c) and torch.equal(b, d) and c.is_inference()
        c.add_(1)
    w = torch.ones(128, device=DEV, dtype=BF, requires_grad=True)
    (a * w).float().sum().backward()
    assert torch.isfinite(w.grad).all()
    kept = b.clone()
    del a, c, d
    for _ in range(20):
        torch.randn(9, 8, 128, device=DEV)
    assert torch.equal(b, kept) and b.is_contiguous()
