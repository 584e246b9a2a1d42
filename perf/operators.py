"""The operators around a paged cache whose pages hold 16-bit keys and values, as timed cases.

``listed()`` names twelve cases, ``draw()`` gives further sizes and options of the same kinds,
``prepare()`` makes what a serving program holds before the call, ``run()`` is one pass: the package's
entry points where ``own`` is true, elementary torch operations where it is not.  ``exact()`` says in 64
bits what comes out.

Kinds:
  plan     block tables, slots and positions of a step from the lengths of its requests
  release  the pages of finished requests go back to the pool
  rotary   rotary positions of the queries and keys of a step
  append   the same, with the keys and values written to their pages
  decode   attention of one new token per sequence over the pages
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a decode step of 256 running requests: one token each, a few of them cross into a new page
        _plan("plan_step_256", requests=256, context=4096, new=1, spare=0),
        # a prefill step: 64 requests with chunks of up to 1024 tokens behind a part-filled cache
        _plan("plan_prompts_64x1024", requests=64, context=2048, new=1024, spare=100),
        # a few requests of a small batch end
        _release("release_64", requests=64, context=4096, share=0.1),
        # a large batch is drained: half of its requests end at once
        _release("release_1024", requests=1024, context=8192, share=0.5),
        # one decode step of 32 sequences at far positions, all of the head rotated
        _rotary("rotary_step_32", tokens=32, far=131072),
        # a prompt batch of odd length, fp16, pairs side by side, half of the head rotated, q and k
        # slices of one projection
        _rotary("rotary_prompt_7001", tokens=7001, far=8192, dtype="fp16", layout="interleaved", rd=64,
                joint=True),
        # the new tokens of 32 sequences
        _append("append_step_32", tokens=32, far=131072),
        # a prompt batch, frequencies scaled by their wavelength for a longer context
        _append("append_prompt_8192", tokens=8192, far=32768, scaling="wavelength", joint=True),
        # one user at a short context: latency counts
        _decode("decode_1x900", seqs=1, context=900),
        # the batch of an 8B-shaped layer
        _decode("decode_32x4096", seqs=32, context=4096),
        # 70B-shaped long contexts, ragged 32k .. 128k, eight query heads per KV head
        _decode("decode_long_8x131072", seqs=8, context=131072, ragged=True, hq=64),
        # small heads, one KV head per query head, fp16, each sequence sees its last 1000 tokens, with the
        # logarithms of the sums
        _decode("decode_window_48x6000", seqs=48, context=6000, ragged=True, hq=16, hkv=16, d=64,
                dtype="fp16", window=1000, lse=True),
    ]


def _named(name, c):
    return {**c, "name": name} if name else c


def _plan(name, **kw):
    return _named(name, {"kind": "plan", "block": 16, **kw})


def _release(name, **kw):
    return _named(name, {"kind": "release", "block": 16, **kw})


_HEADS = {"hq": 32, "hkv": 8, "d": 128, "dtype": "bf16"}
_ROPE = {"rd": 128, "layout": "half", "scaling": "none", "joint": False, **_HEADS}


def _rotary(name, **kw):
    return _named(name, {"kind": "rotary", "inverse": False, **_ROPE, **kw})


def _append(name, **kw):
    return _named(name, {"kind": "append", "block": 16, **_ROPE, **kw})


def _decode(name, **kw):
    return _named(name, {"kind": "decode", "block": 16, "ragged": False, "window": 0, "lse": False,
                         "rows": False, "empty": 0, **_HEADS, **kw})


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["plan", "release", "rotary", "append", "decode"], [2, 1, 3, 3, 5])[0]
    if kind in ("plan", "release"):
        block = rng.choice([16, 16, 16, 32, 64])
        requests = _log(rng, 1, 1024)
        context = _log(rng, 20, min(131072, (1 << 20) * block // requests // 4))
        if kind == "release":
            return _release(None, requests=requests, context=context, share=rng.choice([0.05, 0.3, 1.0]),
                            block=block)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(4096, 65536 // requests)))
        return _plan(None, requests=requests, context=context, new=new, spare=rng.choice([0, 7, 1000]),
                     block=block)
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (8, 1), (16, 16), (20, 2), (40, 10)])
    if kind == "decode":
        c = _decode(None, hq=hq, hkv=hkv, d=rng.choice([128, 128, 64, 96, 256]),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), block=rng.choice([16, 16, 32, 64, 256]))
        c["seqs"] = _log(rng, 1, 256)
        room = 512 * 1024 * 8 * 128 // (hkv * c["d"])  # tokens in 2.1 GB of pages
        c["context"] = _log(rng, 1, max(1, min(131072, room // c["seqs"])))
        c["ragged"] = rng.random() < 0.7
        c["window"] = rng.choice([0, 0, 0, 127, 4096])
        c["lse"] = rng.random() < 0.3
        c["rows"] = rng.random() < 0.3
        c["empty"] = 0 if c["lse"] else rng.choice([0, 0, 3])
        return c
    d = rng.choice([128, 128, 64, 96, 256])
    c = dict(hq=hq, hkv=hkv, d=d, rd=rng.choice([d, d, d // 2, d // 4]), tokens=_log(rng, 1, 16384),
             layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "wavelength"]),
             joint=rng.random() < 0.5, far=_log(rng, 64, 1 << 20))
    c["tokens"] = max(1, min(c["tokens"], 7000 * 40 * 128 // ((hq + 2 * hkv) * d)))
    if kind == "rotary":
        return _rotary(None, dtype=rng.choice(["bf16", "fp16", "fp32"]), inverse=rng.random() < 0.25, **c)
    return _append(None, dtype=rng.choice(["bf16", "bf16", "fp16"]), block=rng.choice([16, 16, 32, 64]), **c)


# --------------------------------------------------------------------------------------
# sizes
# --------------------------------------------------------------------------------------
def _pages(tokens, block):
    return -(-tokens // block)


def _requests(c):
    """(context, new tokens) of every request of a plan or release: they belong to the case."""
    n, hi = c["requests"], c["context"]
    r = random.Random(7919 * n + hi)
    new = c.get("new", 0)
    out = []
    for _ in range(n):
        m = new if new <= 1 else r.randint(max(1, new // 4), new)
        out.append((r.randint(0 if new > 1 else 1, hi), m))
    return out


def _lengths(c):
    """Tokens of every sequence, ragged ones from a quarter of ``context``, ``empty`` rows of none behind."""
    n, hi = c["seqs"], c["context"]
    r = random.Random(1000003 * n + hi)
    lo = max(1, hi // 4)
    return [r.randint(lo, hi) if c["ragged"] else hi for _ in range(n)] + [0] * c["empty"]


def _finished(c):
    r = random.Random(31 * c["requests"] + c["context"])
    done = [r.random() < c["share"] for _ in range(c["requests"])]
    done[0] = True
    return done


def work(case):
    c, kind = case, case["kind"]
    if kind == "plan":
        reqs, b = _requests(c), c["block"]
        tokens = sum(n for _, n in reqs)
        grown = sum(_pages(k + n, b) - _pages(k, b) for k, n in reqs)
        # lengths in and out, pages taken (read, written), the open page of each request, slots and positions
        return {"bytes": len(reqs) * (8 + 8 + 1) + 8 * grown + 4 * len(reqs) + 16 * (tokens + c["spare"]),
                "flops": 0}
    if kind == "release":
        pages = sum(_pages(k, c["block"]) for (k, _), f in zip(_requests(c), _finished(c)) if f)
        return {"bytes": 8 * pages + 5 * c["requests"], "flops": 0}
    size = 4 if c["dtype"] == "fp32" else 2
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    if kind == "rotary":
        n = c["tokens"]
        return {"bytes": 2 * n * (hq + hkv) * d * size + 8 * n + 4 * c["rd"],
                "flops": 3 * n * (hq + hkv) * c["rd"]}
    if kind == "append":
        n = c["tokens"]
        return {"bytes": 2 * n * (hq + 2 * hkv) * d * size + 16 * n + 4 * c["rd"],
                "flops": 3 * n * (hq + hkv) * c["rd"]}
    lens = _lengths(c)
    seen = [min(n, c["window"]) if c["window"] else n for n in lens]
    total = sum(seen)
    b = 2 * total * hkv * d * size + 2 * len(lens) * hq * d * size + 4 * len(lens)
    b += 4 * sum(_pages(n, c["block"]) for n in seen) + (4 * len(lens) * hq if c["lse"] else 0)
    return {"bytes": b, "flops": 4 * d * hq * total}


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _frequencies(c):
    """Angles per position, in 64 bits: a geometric series; for longer contexts four times slower
    ("linear"), or that for wavelengths beyond 8192 positions, unchanged below 2048, blended between."""
    j = torch.arange(0, c["rd"], 2, dtype=torch.float64)
    w = torch.pow(torch.tensor(500000.0, dtype=torch.float64), -j / c["rd"])
    if c["scaling"] == "linear":
        return w / 4
    if c["scaling"] == "wavelength":
        turn = 2 * math.pi / w
        keep = ((8192 / turn - 1) / 3).clamp(0, 1)
        return w * keep + w / 4 * (1 - keep)
    return w


def _heads(g, dev, c):
    """q, k, v of the new tokens, a few key channels times ten; slices of one projection where joint."""
    n, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
    x = torch.randn(n, hq + 2 * hkv, d, generator=g, device=dev)
    x[:, hq:hq + hkv, ::max(1, d // 4)] *= 10.0
    x = x.to(_DTYPES[c["dtype"]])
    parts = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    return parts if c["joint"] else tuple(p.contiguous() for p in parts)


def prepare(case, seed):
    c, kind = case, case["kind"]
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": c}
    if kind in ("plan", "release"):
        reqs, b = _requests(c), c["block"]
        order = torch.randperm(len(reqs), generator=g, device=dev)
        pairs = torch.tensor(reqs, dtype=torch.int32, device=dev)[order]
        s["context"], s["new"] = pairs[:, 0].contiguous(), pairs[:, 1].contiguous()
        width = _pages(c["context"] + c.get("new", 0), b)
        held = sum(_pages(k, b) for k, _ in reqs)
        blocks = 2 * sum(_pages(k + n, b) for k, n in reqs) + 64
        ids = torch.randperm(blocks, generator=g, device=dev).int()
        cols = torch.arange(width, device=dev)
        mine = cols[None] < ((s["context"] + b - 1) // b)[:, None]
        s["table"] = torch.full((len(reqs), width), -1, dtype=torch.int32, device=dev)
        s["table"][mine] = ids[:held]
        s["free"] = torch.full((blocks,), -1, dtype=torch.int32, device=dev)
        s["free"][:blocks - held] = ids[held:]
        s["count"] = torch.tensor([blocks - held], dtype=torch.int32, device=dev)
        s["room"] = sum(n for _, n in reqs) + c.get("spare", 0)
        if kind == "release":
            s["done"] = torch.tensor(_finished(c), device=dev)[order]
        return s
    if kind in ("rotary", "append"):
        s["q"], s["k"], s["v"] = _heads(g, dev, c)
        s["positions"] = torch.randint(c["far"], (c["tokens"],), generator=g, device=dev)
        s["freq"] = _frequencies(c).to(dev)
        if kind == "append":
            blocks = _pages(2 * c["tokens"], c["block"]) + 1
            shape = (blocks, c["block"], c["hkv"], c["d"])
            s["k_pages"] = torch.zeros(shape, dtype=s["k"].dtype, device=dev)
            s["v_pages"] = torch.zeros(shape, dtype=s["k"].dtype, device=dev)
            s["slots"] = torch.randperm(blocks * c["block"], generator=g, device=dev)[:c["tokens"]]
        return s
    lens, b, h, d = _lengths(c), c["block"], c["hkv"], c["d"]
    dtype = _DTYPES[c["dtype"]]
    counts = [_pages(n, b) for n in lens]
    blocks = sum(counts)
    # keys and values of a token side by side ("rows"), or in two buffers
    pages = torch.empty((blocks, b, 2, h, d) if c["rows"] else (2, blocks, b, h, d), dtype=dtype, device=dev)
    flat = pages.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=g, device=dev))
    s["k_pages"], s["v_pages"] = (pages[:, :, 0], pages[:, :, 1]) if c["rows"] else (pages[0], pages[1])
    s["k_pages"][..., ::max(1, d // 4)] *= 10.0
    s["q"] = torch.randn(len(lens), c["hq"], d, generator=g, device=dev).to(dtype)
    ids = torch.randperm(blocks, generator=g, device=dev).int()
    s["table"] = torch.zeros(len(lens), max(counts), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(counts):
        s["table"][i, :n] = ids[at:at + n]
        at += n
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    return s


# --------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------
def run(state):
    return _calls(state) if own else _PLAIN[state["case"]["kind"]](state)


def _calls(s):
    import flashquant_b200 as fq
    c = s["case"]
    kind = c["kind"]
    if kind == "plan":
        p = fq.plan_paged_step(s["context"], s["new"], s["table"], s["free"], s["count"], c["block"], s["room"])
        return {"table": s["table"], "lens": p.seq_lens, "starts": p.cu_seqlens_q, "slots": p.slot_mapping,
                "positions": p.positions, "served": p.served, "count": p.free_count}
    if kind == "release":
        count = fq.release_pages(s["done"], s["context"], s["table"], s["free"], s["count"], c["block"])
        return {"free": s["free"], "count": count}
    if kind == "rotary":
        q, k = fq.rotary_embed(s["q"], s["k"], s["positions"], s["freq"], layout=c["layout"], scale=_scale(c),
                               inverse=c["inverse"])
        return {"q": q, "k": k}
    if kind == "append":
        q = fq.rotary_append_dense(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], s["positions"],
                                   s["freq"], layout=c["layout"], scale=_scale(c))
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    out = fq.split_k_paged_decode_dense(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                                        window=c["window"], return_lse=c["lse"])
    return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}


def _scale(c):
    """What the rotated values are multiplied with besides: a little more than one where the context is stretched."""
    return 1.0 if c["scaling"] != "linear" else 0.1 * math.log(4.0) + 1.0


def _plain_plan(s):
    b, table, free, room = s["case"]["block"], s["table"], s["free"], s["room"]
    ctx, new, count = s["context"].long(), s["new"].long(), s["count"].long()
    width = table.shape[1]
    have, need = (ctx + b - 1) // b, (ctx + new + b - 1) // b
    valid = (ctx >= 0) & (new >= 0) & (need <= width)
    new = torch.where(valid, new, 0)
    grow = torch.where(new > 0, need - have, 0)
    fits = (grow.cumsum(0) <= count) & (new.cumsum(0) <= room)
    served = valid & ((new == 0) | fits)
    new, grow = torch.where(served, new, 0), torch.where(served, grow, 0)
    before = grow.cumsum(0) - grow
    cols = torch.arange(width, device=table.device)[None]
    taken = (cols >= have[:, None]) & (cols < (have + grow)[:, None])
    source = count - 1 - (before - have)[:, None] - cols
    table.copy_(torch.where(taken, free[torch.where(taken, source, 0)], table))
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(room, device=table.device)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    used = r < len(ctx)
    r = torch.where(used, r, 0)
    at = ctx[r] + t - starts[r]
    page = torch.where(used, at // b, 0)
    slots = torch.where(used, table[r, page].long() * b + at % b, -1)
    return {"table": table, "lens": (ctx.clamp(0, width * b) + new).int(), "starts": starts.int(), "slots": slots,
            "positions": torch.where(used, at, -1), "served": served, "count": (count - grow.sum()).int()}


def _plain_release(s):
    b, table, free, count = s["case"]["block"], s["table"], s["free"], s["count"].long()
    pages = torch.where(s["done"], (s["context"].long() + b - 1) // b, 0)
    cols = torch.arange(table.shape[1], device=table.device)[None]
    mine = cols < pages[:, None]
    to = count + (pages.cumsum(0) - pages)[:, None] + cols
    at = torch.arange(free.numel(), device=free.device)
    # the entries that go, in order of their place; the others are sent behind the stack
    grown = torch.cat([free, free.new_zeros(1)])
    grown[torch.where(mine, to, free.numel())] = table
    total = count + pages.sum()
    free.copy_(torch.where((at >= count) & (at < total), grown[:-1], free))
    return {"free": free, "count": total.int()}


def _turned(x, positions, freq, c, inverse=False):
    """Rotary positions in 32 bits, the angles in 64; not rounded."""
    angle = positions.double()[:, None] * freq[None]
    cos, sin = angle.cos().float()[:, None] * _scale(c), angle.sin().float()[:, None] * _scale(c)
    sin = -sin if inverse else sin
    rd = c["rd"]
    x = x.float()
    head, rest = x[..., :rd], x[..., rd:]
    if c["layout"] == "half":
        a, b = head[..., :rd // 2], head[..., rd // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _plain_rotary(s):
    c = s["case"]
    return {n: _turned(s[n], s["positions"], s["freq"], c, c["inverse"]).to(s[n].dtype) for n in ("q", "k")}


def _plain_append(s):
    c = s["case"]
    q, k = (_turned(s[n], s["positions"], s["freq"], c).to(s[n].dtype) for n in ("q", "k"))
    s["k_pages"].view(-1, c["hkv"], c["d"])[s["slots"]] = k
    s["v_pages"].view(-1, c["hkv"], c["d"])[s["slots"]] = s["v"]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_decode(s):
    c = s["case"]
    b, hq, h, d = c["block"], c["hq"], c["hkv"], c["d"]
    outs, lses = [], []
    for i, n in enumerate(_lengths(c)):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            outs.append(torch.zeros(h, hq // h, d, device=s["q"].device))
            continue
        ids = s["table"][i, first // b:_pages(n, b)]
        lo, hi = first % b, n - first // b * b
        k, v = (s[x][ids].flatten(0, 1)[lo:hi].permute(1, 0, 2).float() for x in ("k_pages", "v_pages"))
        q = s["q"][i].float().view(h, hq // h, d)
        score = (q @ k.transpose(1, 2)) * (1.0 / math.sqrt(d))
        top = score.amax(-1, keepdim=True)
        e = (score - top).exp()
        total = e.sum(-1, keepdim=True)
        outs.append(e @ v / total)
        lses.append((top + total.log()).flatten())
    out = torch.stack(outs).view(len(outs), hq, d).to(s["q"].dtype)
    return {"out": out, "lse": torch.stack(lses)} if c["lse"] else {"out": out}


_PLAIN = {"plan": _plain_plan, "release": _plain_release, "rotary": _plain_rotary, "append": _plain_append,
          "decode": _plain_decode}


# --------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s, case)


def _exact_plan(s, c):
    """Request by request, as a scheduler on the host does it."""
    b, room = c["block"], s["room"]
    table, stack = s["table"].cpu().numpy().copy(), s["free"].cpu().tolist()
    height = free = s["count"].item()
    lens, starts, slots, positions, served = [], [0], [], [], []
    for i, (have, new) in enumerate(zip(s["context"].tolist(), s["new"].tolist())):
        fresh = range(-(-have // b), -(-(have + new) // b))
        ok = len(fresh) <= height and len(slots) + new <= room  # the cases hold no request that does not fit
        assert ok
        for page in fresh:
            height -= 1
            table[i, page] = stack[height]
        for at in range(have, have + new):
            slots.append(int(table[i, at // b]) * b + at % b)
            positions.append(at)
        lens.append(have + new)
        starts.append(len(slots))
        served.append(ok)
    assert free - height >= 0
    pad = [-1] * (room - len(slots))
    i32 = dict(dtype=torch.int32)
    return {"table": torch.from_numpy(table), "lens": torch.tensor(lens, **i32), "starts": torch.tensor(starts, **i32),
            "slots": torch.tensor(slots + pad), "positions": torch.tensor(positions + pad),
            "served": torch.tensor(served), "count": torch.tensor([height], **i32)}


def _exact_release(s, c):
    stack, height = s["free"].cpu().tolist(), s["count"].item()
    rows = s["table"].cpu().tolist()
    for done, have, row in zip(s["done"].tolist(), s["context"].tolist(), rows):
        for page in row[:-(-have // c["block"])] if done else []:
            stack[height] = page
            height += 1
    return {"free": torch.tensor(stack, dtype=torch.int32), "count": torch.tensor([height], dtype=torch.int32)}


def _exact_turn(x, s, c, sign):
    """As products of complex numbers, scale * exp(i * sign * position * frequency)."""
    angle = sign * s["positions"].double()[:, None] * s["freq"]
    unit = torch.polar(torch.full_like(angle, _scale(c)), angle)[:, None]
    rd, x = c["rd"], x.double()
    head = x[..., :rd]
    pairs = head.unflatten(-1, (2, -1)).transpose(-1, -2) if c["layout"] == "half" else head.unflatten(-1, (-1, 2))
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    if c["layout"] == "half":
        turned = turned.transpose(-1, -2)
    out = x.clone()
    out[..., :rd] = turned.flatten(-2)
    return out


def _exact_rotary(s, c):
    return {n: _exact_turn(s[n], s, c, -1.0 if c["inverse"] else 1.0) for n in ("q", "k")}


def _exact_append(s, c):
    out = {"q": _exact_turn(s["q"], s, c, 1.0)}
    b = c["block"]
    for name, new in (("k_pages", _exact_turn(s["k"], s, c, 1.0)), ("v_pages", s["v"].double())):
        pages = s[name].double()
        pages[s["slots"] // b, s["slots"] % b] = new
        out[name] = pages
    return out


def _exact_decode(s, c):
    b, hq, h, d = c["block"], c["hq"], c["hkv"], c["d"]
    out = torch.zeros(len(s["lens"]), hq, d, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device=out.device)
    for i, n in enumerate(_lengths(c)):
        at = torch.arange(max(0, n - c["window"]) if c["window"] else 0, n, device=out.device)
        page, row = s["table"][i][at // b].long(), at % b
        for kv in range(h if n else 0):
            k, v = s["k_pages"][page, row, kv].double(), s["v_pages"][page, row, kv].double()
            heads = slice(kv * (hq // h), (kv + 1) * (hq // h))
            score = s["q"][i, heads].double() @ k.T / math.sqrt(d)
            lse[i, heads] = torch.logsumexp(score, 1)
            out[i, heads] = torch.softmax(score, 1) @ v
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


_EXACT = {"plan": _exact_plan, "release": _exact_release, "rotary": _exact_rotary, "append": _exact_append,
          "decode": _exact_decode}
