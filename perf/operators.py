"""The decoder-step operators measured: what they are fed, their plain forms, and what they have to move.

Three operators stand between the embedding row of a drawn token (ssb_sample_embed_rows) and the LM head
(ssb_lm_head_argmax) of a device-resident decode loop:

  append   RMS norms of the query and key heads, the rotation of both, and the keys and values written into
           a paged key-value cache (Sampler.norm_rope_append)
  step     attention of one new token, or of a few draft rows, per sequence over that cache (Sampler.attend)
  prompt   the same call for the rows of prompts

A case is one call. `own` selects the framework's entry points; otherwise `run` computes the plain form.
"""
import math
import random

import torch

own = False

_ENGINE = []


def _engine():
    """The engine context a program creates once per device."""
    if not _ENGINE:
        import os
        import sys
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "speech.cpp_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import speech_sampler
        _ENGINE.extend([speech_sampler.Sampler(0), speech_sampler])
    return _ENGINE


def _append(name, **kw):
    c = dict(name=name, op="append", seqs=1, rows=1, ragged=1, len_min=1, len_max=1, heads=16, kv_heads=8, dim=128,
             rope_dim=128, interleaved=False, dtype="bf16", page=64, layout="heads")
    c.update(kw)
    return c


def _attend(name, op, **kw):
    c = dict(name=name, op=op, seqs=1, rows=1, ragged=1, len_min=1, len_max=1, heads=16, kv_heads=8, dim=128,
             dtype="bf16", page=64, layout="heads", window=0, sinks=0)
    c.update(kw)
    return c


def listed():
    return [
        # the single stream of a talker: one row, where only latency counts
        _append("append-one-row", len_min=411, len_max=411),
        # one decode step of a text decoder's batch: 256 streams
        _append("append-256-streams", seqs=256, len_min=1, len_max=300, layout="positions"),
        # prompts of a batch, ragged, fp32 rows with half of each head rotated in adjacent pairs
        _append("append-prompts-f32", seqs=9, rows=1500, len_min=1500, len_max=2001, rope_dim=64, interleaved=True,
                dtype="f32", page=16),
        # a talker's first frames: a short cache, latency again
        _attend("step-one-short", "step", len_min=37, len_max=37, page=16),
        # one stream far into a recording: all of the GPU on one sequence
        _attend("step-one-long", "step", len_min=120001, len_max=120001),
        # the streams of a server, each somewhere between its first token and its eight thousandth
        _attend("step-64-streams", "step", seqs=64, len_min=1, len_max=8000),
        # draft rows to verify, one to five per stream, on four query heads per key head
        _attend("step-verify-drafts", "step", seqs=24, rows=5, len_min=300, len_max=4001, heads=32, page=32,
                layout="positions"),
        # endless dialogues: a window of 2000 positions and four first tokens, the pages between them freed
        _attend("step-dialogues-window", "step", seqs=128, len_min=100, len_max=30000, window=2000, sinks=4, page=16),
        # an fp32 cache
        _attend("step-16-streams-f32", "step", seqs=16, len_min=200, len_max=3001, dtype="f32"),
        # one 512-row block of a chunked prompt behind 4000 cached positions
        _attend("prompt-block-512", "prompt", rows=512, len_min=4512, len_max=4512),
        # whole prompts of a batch, ragged
        _attend("prompt-8-ragged", "prompt", seqs=8, rows=6000, len_min=1000, len_max=6001, heads=32),
        # one long recording under a window with first tokens kept
        _attend("prompt-long-window", "prompt", rows=16001, len_min=16001, len_max=16001, window=1024, sinks=4, page=128,
                layout="positions"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "step", "step", "prompt"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (16, 2), (8, 8), (12, 4), (16, 1)])
    dim = rng.choice([64, 128, 128])
    common = dict(op=op, ragged=rng.randrange(1, 1 << 20), heads=heads, kv_heads=kv_heads, dim=dim,
                  page=rng.choice([16, 32, 64, 128]), layout=rng.choice(["heads", "positions"]))
    if op == "append":
        seqs = _log_int(rng, 1, 256)
        rows = _log_int(rng, 1, max(1, 13000 // seqs))
        lo = _log_int(rng, rows, rows + 300)
        return dict(common, seqs=seqs, rows=rows, len_min=lo, len_max=lo + rng.randrange(0, 200),
                    rope_dim=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.3,
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    sinks = rng.randrange(0, 9) if window else 0
    if op == "step":
        seqs = _log_int(rng, 1, 128)
        rows = rng.choice([1, 1, rng.randrange(2, 7)])
        hi = _log_int(rng, 8, min(120000, 400000 // seqs))
        lo = _log_int(rng, 1, hi)
        return dict(common, seqs=seqs, rows=rows, len_min=lo, len_max=hi, window=window, sinks=sinks,
                    dtype="f32" if rng.random() < 0.2 else "bf16")
    seqs = _log_int(rng, 1, 8)
    rows = _log_int(rng, 130, 14000 // seqs)
    lo = _log_int(rng, max(1, rows // 4), rows)
    return dict(common, seqs=seqs, rows=rows, len_min=lo, len_max=rows + rng.choice([0, _log_int(rng, 1, 4000)]),
                window=window, sinks=sinks, dtype="bf16")


def _lengths(case):
    """(cached length, new rows) of every sequence, a function of the case alone. The length counts the new rows."""
    rng = random.Random(case["ragged"])
    lens = [rng.randint(case["len_min"], case["len_max"]) for _ in range(case["seqs"])]
    if case["op"] == "prompt":
        rows = [min(n, case["rows"]) for n in lens]
    elif case["op"] == "append" or case["rows"] == 1:
        rows = [min(n, case["rows"]) for n in lens]
    else:
        rows = [min(n, rng.randint(1, case["rows"])) for n in lens]
    return lens, rows


def _seen(length, rows, window, sinks):
    """The positions that some of the last `rows` positions of a sequence see, as (start, stop) ranges."""
    lo = max(0, length - rows - window + 1) if window else 0
    return [(0, length)] if lo <= sinks else [(0, sinks), (lo, length)]


def work(case):
    lens, rows = _lengths(case)
    e = 2 if case["dtype"] == "bf16" else 4
    d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
    n = sum(rows)
    if case["op"] == "append":
        row = (2 * hq + 4 * hk) * d * e
        return {"bytes": n * (row + 4) + case["seqs"] * 12 + 8 * d, "flops": n * (hq + hk) * d * 7}
    pairs = seen = 0
    w, sinks = case["window"], case["sinks"]
    for length, r in zip(lens, rows):
        seen += sum(b - a for a, b in _seen(length, r, w, sinks))
        for p in ([length - 1] if r == 1 else range(length - r, length)):
            pairs += sum(b - a for a, b in _seen(p + 1, 1, w, sinks))
    return {"bytes": seen * hk * d * 2 * e + n * hq * (2 * d * e + 4) + 4 * (seen // case["page"] + 2 * case["seqs"]),
            "flops": 4 * d * hq * pairs}


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    lens, rows = _lengths(case)
    s, d, hq, hk, ps = case["seqs"], case["dim"], case["heads"], case["kv_heads"], case["page"]
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    held = []  # the (sequence, page of the sequence) pairs whose pages exist
    for i, (length, r) in enumerate(zip(lens, rows)):
        keep = set()
        for a, b in _seen(length, r, window, sinks):
            if b > a:
                keep.update(range(a // ps, (b - 1) // ps + 1))
        held.extend((i, p) for p in sorted(keep))
    pages = len(held) + 1
    order = torch.randperm(pages, device=dev, generator=g)[: len(held)].to(torch.int32)
    table = torch.full((s, max((n + ps - 1) // ps for n in lens)), -1, dtype=torch.int32, device=dev)
    at = torch.tensor(held, dtype=torch.int64, device=dev)
    table[at[:, 0], at[:, 1]] = order
    if case["layout"] == "heads":  # one head's positions of a page lie together
        pool = torch.randn(2, pages, hk, ps, d, device=dev, generator=g).to(dt).transpose(2, 3)
    else:  # one position's heads lie together
        pool = torch.randn(2, pages, ps, hk, d, device=dev, generator=g).to(dt)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    state = {"case": case, "k": pool[0], "v": pool[1], "table": table, "rows": rows, "lens": lens,
             "lens_dev": torch.tensor(lens, dtype=torch.int32, device=dev),
             "starts": torch.tensor(starts, dtype=torch.int32, device=dev),
             "uniform": min(rows) == max(rows)}
    n = starts[-1]
    if case["op"] == "append":
        qkv = torch.randn(n, (hq + 2 * hk) * d, device=dev, generator=g).to(dt)  # one projection's output rows
        state["q"] = qkv[:, : hq * d].view(n, hq, d)
        state["new_k"] = qkv[:, hq * d: (hq + hk) * d].view(n, hk, d)
        state["new_v"] = qkv[:, (hq + hk) * d:].view(n, hk, d)
        state["q_weight"] = 1 + 0.3 * torch.randn(d, device=dev, generator=g)
        state["k_weight"] = 1 + 0.3 * torch.randn(d, device=dev, generator=g)
        half = case["rope_dim"] // 2
        state["inv_freq"] = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        state["out"] = torch.empty(n, hq, d, dtype=dt, device=dev)
    else:
        state["q"] = torch.randn(n, hq, d, device=dev, generator=g).to(dt)
        state["out"] = torch.empty(n, hq, d, dtype=dt, device=dev)
        state["lse"] = torch.empty(n, hq, dtype=torch.float32, device=dev)
    if own:
        engine, ss = _engine()
        state["engine"] = engine
        state["cache"] = ss.KvCache(state["k"], state["v"], table)
    return state


def run(state):
    case = state["case"]
    if own:
        ragged = {} if state["uniform"] else {"row_start": state["starts"]}
        if case["op"] == "append":
            state["engine"].norm_rope_append(
                state["q"], state["new_k"], state["new_v"], state["cache"], state["lens_dev"], state["inv_freq"],
                q_weight=state["q_weight"], k_weight=state["k_weight"], eps=1e-6, interleaved=case["interleaved"],
                max_rows=max(state["rows"]), q_out=state["out"], stream=torch.cuda.current_stream(), **ragged)
            return {"q": state["out"], "k": state["k"], "v": state["v"]}
        state["engine"].attend(
            state["q"], state["cache"], state["lens_dev"], scale=case["dim"] ** -0.5, window=case["window"],
            sinks=case["sinks"], max_rows=max(state["rows"]), max_length=max(state["lens"]), out=state["out"],
            lse=state["lse"], stream=torch.cuda.current_stream(), **ragged)
        return {"out": state["out"], "lse": state["lse"]}
    return _plain_append(state) if case["op"] == "append" else _plain_attend(state)


def _positions(state):
    """(sequence, position) of every row."""
    rows, lens = state["starts"].diff().long(), state["lens_dev"].long()
    seq = torch.repeat_interleave(torch.arange(len(state["rows"]), device=rows.device), rows, output_size=sum(state["rows"]))
    at = torch.arange(sum(state["rows"]), device=rows.device) - state["starts"][:-1].long()[seq]
    return seq, lens[seq] - rows[seq] + at


def _plain_append(state):
    case = state["case"]
    seq, pos = _positions(state)
    angle = pos.double()[:, None] * state["inv_freq"][None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    rot = case["rope_dim"]

    def shaped(x, weight):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
        head, rest = x[..., :rot], x[..., rot:]
        if case["interleaved"]:
            a, b = head[..., 0::2], head[..., 1::2]
            head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = head.chunk(2, -1)
            head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([head, rest], -1)

    dt = state["q"].dtype
    page = state["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    state["k"][page, slot] = shaped(state["new_k"], state["k_weight"]).to(dt)
    state["v"][page, slot] = state["new_v"]
    return {"q": shaped(state["q"], state["q_weight"]).to(dt), "k": state["k"], "v": state["v"]}


def _plain_attend(state):
    case = state["case"]
    hk, d, ps, window, sinks = case["kv_heads"], case["dim"], case["page"], case["window"], case["sinks"]
    group = case["heads"] // hk
    out, lse = torch.empty_like(state["out"]), torch.empty_like(state["lse"])
    row = 0
    for s, (length, rows) in enumerate(zip(state["lens"], state["rows"])):
        done = 0
        while done < rows:
            first = length - rows + done
            most = max(64, window) if window else rows  # a block's ranges stay within twice its window
            n = min(rows - done, most, max(1, (1 << 27) // (case["heads"] * min(length, 2 * most if window else length))))
            idx = torch.cat([torch.arange(a, b, device="cuda") for a, b in _seen(first + n, n, window, sinks)])
            page, slot = state["table"][s, idx // ps].long(), idx % ps
            k = state["k"][page, slot].float().permute(1, 2, 0)  # [kv_heads, dim, positions]
            v = state["v"][page, slot].float().transpose(0, 1)   # [kv_heads, positions, dim]
            q = state["q"][row: row + n].float().view(n, hk, group, d).permute(1, 0, 2, 3).reshape(hk, n * group, d)
            x = (torch.matmul(q, k) * d ** -0.5).view(hk, n, group, -1)
            p = torch.arange(first, first + n, device="cuda")[:, None]
            ok = idx[None] <= p
            if window:
                ok &= (idx[None] > p - window) | (idx[None] < sinks)
            x = x.masked_fill(~ok[None, :, None], -math.inf)
            top = x.amax(-1, keepdim=True)
            w = torch.exp(x - top)
            total = w.sum(-1, keepdim=True)
            o = torch.matmul(w.view(hk, n * group, -1), v).view(hk, n, group, d) / total
            out[row: row + n] = o.permute(1, 0, 2, 3).reshape(n, hk * group, d).to(out.dtype)
            lse[row: row + n] = (top + torch.log(total))[..., 0].permute(1, 0, 2).reshape(n, hk * group)
            row += n
            done += n
    return {"out": out, "lse": lse}


def exact(case, seed):
    """The operators' definitions in 64 bits."""
    st = prepare(case, seed)
    table, ps, d = st["table"].cpu().tolist(), case["page"], case["dim"]
    if case["op"] == "append":
        where, turn = [], []
        for s, (length, rows) in enumerate(zip(st["lens"], st["rows"])):
            for p in range(length - rows, length):
                where.append(table[s][p // ps] * ps + p % ps)
                turn.append(p)
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                        torch.tensor(turn, dtype=torch.float64, device="cuda")[:, None] * st["inv_freq"])
        where = torch.tensor(where, device="cuda")

        def turned(x, weight):
            x = x.double()
            x = weight.double() * x / ((x * x).sum(-1, keepdim=True) / d + 1e-6).sqrt()
            r = case["rope_dim"]
            if case["interleaved"]:
                y = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * z[:, None]
                x[..., :r] = torch.view_as_real(y).reshape(*x.shape[:-1], r)
            else:
                y = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2: r].contiguous()) * z[:, None]
                x[..., : r // 2], x[..., r // 2: r] = y.real, y.imag
            return x

        k, v = st["k"].double(), st["v"].double()
        k[where // ps, where % ps] = turned(st["new_k"], st["k_weight"])
        v[where // ps, where % ps] = st["new_v"].double()
        return {"q": turned(st["q"], st["q_weight"]), "k": k, "v": v}

    n, hq = st["q"].shape[:2]
    group = hq // case["kv_heads"]
    out = torch.empty(n, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.empty(n, hq, dtype=torch.float64, device="cuda")
    base = 0
    for s, (length, rows) in enumerate(zip(st["lens"], st["rows"])):
        held = torch.tensor([table[s][j // ps] * ps + j % ps if table[s][j // ps] >= 0 else -1 for j in range(length)],
                            device="cuda")
        for h in range(case["kv_heads"]):
            for a in range(0, rows, 1024):
                b = min(rows, a + 1024)
                p0, p1 = length - rows + a, length - rows + b  # the block's positions
                low = max(0, p0 - case["window"] + 1) if case["window"] else 0
                j = torch.arange(length, device="cuda")[:p1]
                j = j[(j >= low) | (j < case["sinks"])]
                k = st["k"][:, :, h][held[j] // ps, held[j] % ps].double()
                v = st["v"][:, :, h][held[j] // ps, held[j] % ps].double()
                at = torch.arange(p0, p1, device="cuda")
                hidden = j[None] > at[:, None]
                if case["window"]:
                    hidden |= (at[:, None] - j[None] >= case["window"]) & (j[None] >= case["sinks"])
                for g in range(h * group, (h + 1) * group):
                    x = st["q"][base + a: base + b, g].double() @ k.T / math.sqrt(d)
                    x[hidden] = -math.inf
                    lse[base + a: base + b, g] = torch.logsumexp(x, 1)
                    out[base + a: base + b, g] = torch.softmax(x, 1) @ v
        base += rows
    return {"out": out, "lse": lse}
