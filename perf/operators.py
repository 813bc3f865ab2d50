"""Performance cases of serving from a paged key-value cache, and of prompts with a window and sinks.

A case is a dict of plain values whose ``op`` names the operator; ``listed()`` gives fixed ones, ``draw(rng)``
one more of the same ranges.  ``prepare`` makes the inputs of a case, ``run`` is one pass, ``work`` the bytes
and operations one pass cannot do without, ``exact`` the outputs in 64 bits.

Where ``own`` is false, ``run`` computes the operators in their plain form out of elementary torch operations;
where it is true, it makes the calls that a user makes of the framework.

Operators
  tables    ops.paged_tables: block tables and slot maps of a step from the lengths of its requests
  prepare   ops.qkv_prepare_paged: norms, rotation (either layout, part of the head, scaled) and append to the pages
  decode    ops.sdpa_decode_paged: one new token of each sequence over its pages, with or without window and sinks
  prefill   ops.sdpa_prefill with a window and the first tokens that stay visible
"""
import math

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # The smallest step there is: one new token of each of a few chats.
        dict(name="tables_few", op="tables", batch=8, lo=100, hi=4000, prompts=0, chunk=1, page=16, lengths=1),
        # A serving step that mixes new tokens of most requests with prompt chunks of some.
        dict(name="tables_mixed", op="tables", batch=509, lo=0, hi=9000, prompts=37, chunk=512, page=32, lengths=2),
        # A burst of new prompts: every token's slot and position, every page from the free list.
        dict(name="tables_prompts", op="tables", batch=64, lo=0, hi=0, prompts=64, chunk=8192, page=64, lengths=3),
        # One new token of each sequence of a serving batch: norms, rotation of a quarter of the head.
        dict(name="prepare_tokens", op="prepare", tokens=64, past=32768, nq=24, nkv=4, hd=256, rotary=64, interleaved=False,
             norm=True, theta=1e6, scale=1.0, page=16),
        # A ragged prompt chunk far into a context that was stretched: no norms, neighbours as pairs.
        dict(name="prepare_chunk", op="prepare", tokens=1531, past=500000, nq=28, nkv=4, hd=128, rotary=128, interleaved=True,
             norm=False, theta=1e4, scale=16.0, page=32),
        # Prompt processing: norms and rotation of whole heads.
        dict(name="prepare_prompt", op="prepare", tokens=16384, past=0, nq=32, nkv=16, hd=128, rotary=128, interleaved=False,
             norm=True, theta=1e4, scale=1.0, page=64),
        # One user's chat at a small depth: the latency of a token's attention, gate fused.
        dict(name="decode_one", op="decode", batch=1, lo=513, hi=513, nq=24, nkv=4, hd=256, page=16, window=0, sinks=0, gate=True,
             lengths=4),
        # Many streams of any length through layers with a window and sinks: most of the cache is never read.
        dict(name="decode_window", op="decode", batch=48, lo=300, hi=65536, nq=28, nkv=4, hd=128, page=32, window=1024, sinks=4,
             gate=False, lengths=5),
        # A serving batch: 64 sequences of 1 K to 32 K keys, gated.
        dict(name="decode_batch", op="decode", batch=64, lo=1024, hi=32768, nq=24, nkv=4, hd=256, page=64, window=0, sinks=0,
             gate=True, lengths=6),
        # A short prompt of odd length through one layer.
        dict(name="prefill_short", op="prefill", batch=1, seq=701, kv=701, nq=8, nkv=4, hd=128, window=256, sinks=4, gate=False),
        # A chunk of a long prompt at head dim 256 behind a ragged past, gated.
        dict(name="prefill_chunk", op="prefill", batch=1, seq=2048, kv=5049, nq=24, nkv=4, hd=256, window=1024, sinks=64, gate=True),
        # Prompts of a full batch.
        dict(name="prefill_batch", op="prefill", batch=4, seq=8192, kv=8192, nq=32, nkv=16, hd=128, window=1024, sinks=4,
             gate=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


#: (query heads, KV heads, head dim) of the configurations, the tests and the bench program
HEADS = [(8, 4, 128), (16, 8, 256), (32, 16, 128), (24, 4, 256), (16, 2, 128), (28, 4, 128), (16, 8, 128), (8, 2, 256), (7, 7, 128),
         (16, 1, 128)]
PAGES = [16, 16, 32, 48, 64, 128, 256]
#: most operations of a drawn prefill, most bytes of a drawn decode: under what the largest listed cases take
MOST_FLOPS = 1.2e11
MOST_BYTES = 3.0e9


def draw(rng):
    op = rng.choice(["tables", "prepare", "prepare", "decode", "decode", "decode", "prefill", "prefill"])
    if op == "tables":
        batch = _log(rng, 1, 1024)
        prompts = rng.choice([0, rng.randint(0, batch), batch])
        return dict(op=op, batch=batch, lo=0, hi=_log(rng, 1, 20000), prompts=prompts, chunk=_log(rng, 1, max(2, min(8192, 400000 // batch))),
                    page=rng.choice(PAGES), lengths=rng.randrange(1 << 20))
    nq, nkv, hd = rng.choice(HEADS)
    if op == "prepare":
        return dict(op=op, tokens=_log(rng, 1, 8192), past=_log(rng, 1, 1000000), nq=nq, nkv=nkv, hd=hd,
                    rotary=rng.choice([hd, hd, hd // 2, hd // 4, 48]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.6,
                    theta=rng.choice([1e4, 1e6]), scale=rng.choice([1.0, 1.0, 4.0, 32.0]), page=rng.choice(PAGES))
    if op == "decode":
        windowed = rng.random() < 0.5
        c = dict(op=op, batch=_log(rng, 1, 128), lo=0, hi=_log(rng, 16, 131072), nq=nq, nkv=nkv, hd=hd, page=rng.choice(PAGES),
                 window=_log(rng, 16, 8192) if windowed else 0, sinks=rng.choice([0, 1, 4, 16, 100]) if windowed else 0,
                 gate=rng.random() < 0.4, lengths=rng.randrange(1 << 20))
        c["hi"] = max(16, min(c["hi"], int(MOST_BYTES / (4 * nkv * hd * c["batch"]))))
        c["lo"] = int(c["hi"] * rng.choice([0.0, 0.1, 1.0]))
        return c
    c = dict(op=op, batch=rng.choice([1, 1, 2, 4]), seq=_log(rng, 1, 8192), kv=0, nq=nq, nkv=nkv, hd=hd, window=_log(rng, 32, 4096),
             sinks=rng.choice([1, 4, 4, 64, 128, 500]), gate=rng.random() < 0.4)
    past = _log(rng, 1, 8192) if rng.random() < 0.5 else 0
    c["kv"] = c["seq"] + past
    while work(c)["flops"] > MOST_FLOPS:  # fewer queries, the rest of the call as it is
        c["seq"] = max(32, int(c["seq"] * 0.8))
        c["kv"] = c["seq"] + past
    return c


# ---------------------------------------------------------------------------
# What follows from a case
# ---------------------------------------------------------------------------
def _spread(seed, n, lo, hi):
    """n whole numbers of [lo, hi], over their logarithm where the range is wide, the first of them hi."""
    out = []
    for i in range(n):
        seed = (seed * 6364136223846793005 + 1442695040888963407) % (1 << 64)
        u = (seed >> 11) / float(1 << 53)
        v = math.exp(math.log(lo + 1) + u * (math.log(hi + 1) - math.log(lo + 1))) - 1 if hi > 10 * (lo + 1) else lo + u * (hi - lo)
        out.append(min(hi, max(lo, int(round(v)))))
    if out:
        out[0] = hi
    return out


def _step(c):
    """(tokens in the cache, new tokens) of every request of a step."""
    past = _spread(c["lengths"] * 2 + 1, c["batch"], c["lo"], c["hi"])
    chunks = _spread(c["lengths"] * 2 + 2, c["prompts"], min(c["chunk"], 1), c["chunk"])
    new = [1] * c["batch"]
    for i, n in enumerate(chunks):  # spread over the batch
        new[i * c["batch"] // c["prompts"]] = n
    return past, new


def _seen(length, window, sinks):
    """Keys that one token at the end of `length` keys sees."""
    return length if not window else min(length, window + min(sinks, max(0, length - window)))


def _pairs(seq, kv, window, sinks):
    """(query, key) pairs of one head; query i sits at position kv - seq + i."""
    return sum(_seen(p + 1, window, sinks) for p in range(kv - seq, kv))


def _pages_of(lens, page):
    return [-(-n // page) for n in lens]


def work(case):
    c, op = case, case["op"]
    if op == "tables":
        past, new = _step(c)
        total = [p + n for p, n in zip(past, new)]
        fresh = sum(_pages_of(total, c["page"])) - sum(_pages_of(past, c["page"]))
        behind = sum(1 for p, n in zip(past, new) if p % c["page"] and n)  # pages that are continued: read from the table
        return {"bytes": 4.0 * (2 * sum(new) + 2 * fresh + behind + 5 * c["batch"]), "flops": 4.0 * sum(new)}
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    if op == "prepare":
        return {"bytes": c["tokens"] * (4.0 * (nq + 2 * nkv) * hd + 8), "flops": c["tokens"] * (nq + nkv) * (3.0 * c["rotary"] + (4.0 * hd if c["norm"] else 0))}
    if op == "decode":
        keys = sum(_seen(n, c["window"], c["sinks"]) for n in _spread(c["lengths"], c["batch"], c["lo"], c["hi"]))
        return {"bytes": 4.0 * keys * nkv * hd + c["batch"] * nq * hd * 2.0 * (3 if c["gate"] else 2) + c["batch"] * nq * 4.0,
                "flops": 4.0 * hd * nq * keys}
    seen = min(c["kv"], c["seq"] + c["window"] - 1 + c["sinks"])
    return {"bytes": c["batch"] * (2.0 * hd * (c["seq"] * nq * (3 if c["gate"] else 2) + 2 * seen * nkv) + 4.0 * c["seq"] * nq),
            "flops": 4.0 * hd * nq * c["batch"] * _pairs(c["seq"], c["kv"], c["window"], c["sinks"])}


# ---------------------------------------------------------------------------
# Inputs: N(0, 1) bf16 drawn on the device, norm weights near one, pages in no order
# ---------------------------------------------------------------------------
def _frequencies(c):
    """Radians a position of every pair, and the factor on cosine and sine: contexts stretched `scale` times turn the slow
    pairs more slowly and leave the fast ones, with a ramp between (YaRN, arXiv:2309.00071)."""
    half, factor = c["rotary"] // 2, c["scale"]
    inv = c["theta"] ** (-2.0 * torch.arange(half, dtype=torch.float64) / c["rotary"])
    if factor == 1.0:
        return inv, 1.0
    turns = 4096.0 * inv / (2 * math.pi)  # over the length that the model was trained on
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return inv * keep + inv / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def rnd(*shape, by=1.0):
        t = torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.bfloat16)
        return t if by == 1.0 else t.mul_(by)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)

    def shuffled(n):
        return torch.randperm(n, generator=g, device=DEVICE).to(torch.int32)

    s, op, page = dict(case), case["op"], case.get("page", 0)
    if op == "tables":
        past, new = _step(case)
        held, need = _pages_of(past, page), _pages_of([p + n for p, n in zip(past, new)], page)
        order = shuffled(sum(need) + 7)
        width = max(max(need), 1)
        table = torch.full((case["batch"], width), -1, dtype=torch.int32)
        order_host, at = order.cpu(), 0
        for b, n in enumerate(held):
            table[b, :n] = order_host[at:at + n]
            at += n
        s.update(past=ints(past), new=ints(new), table=table.to(DEVICE), free=order[at:].contiguous(), tokens=sum(new))
        return s
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    if op == "prepare":
        tokens = case["tokens"]
        pages = -(-tokens // page) + 3
        inv, mscale = _frequencies(case)
        s.update(q=rnd(tokens, nq, hd), k=rnd(tokens, nkv, hd), v=rnd(tokens, nkv, hd), q_out=torch.empty(tokens, nq, hd, device=DEVICE, dtype=torch.bfloat16),
                 kp=rnd(pages, page, nkv, hd), vp=rnd(pages, page, nkv, hd), inv=inv.to(DEVICE), mscale=mscale,
                 qw=rnd(hd, by=0.1).add_(1.0) if case["norm"] else None, kw=rnd(hd, by=0.1).add_(1.0) if case["norm"] else None)
        at = torch.arange(tokens, device=DEVICE)
        s["positions"] = (case["past"] + at).to(torch.int32)
        s["slots"] = (shuffled(pages)[at // page] * page + at % page).to(torch.int32)
        return s
    if op == "decode":
        lens = _spread(case["lengths"], case["batch"], case["lo"], case["hi"])
        need = _pages_of(lens, page)
        pages = sum(need) + 5
        order, at = shuffled(pages).cpu(), 0
        table = torch.full((case["batch"], max(max(need), 1)), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        s.update(q=rnd(case["batch"], nq, hd), kp=rnd(pages, page, nkv, hd), vp=rnd(pages, page, nkv, hd), table=table.to(DEVICE),
                 lens=ints(lens), g=rnd(case["batch"], nq, hd) if case["gate"] else None, lens_host=lens)
        return s
    s.update(q=rnd(case["batch"], case["seq"], nq, hd), k=rnd(case["batch"], case["kv"], nkv, hd), v=rnd(case["batch"], case["kv"], nkv, hd),
             g=rnd(case["batch"], case["seq"], nq, hd) if case["gate"] else None)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_tables(s):
    page, past, new = s["page"], s["past"].long(), s["new"].long()
    total = past + new
    held, need = (past + page - 1) // page, (total + page - 1) // page
    begin = torch.zeros(s["batch"] + 1, dtype=torch.long, device=past.device)
    begin[1:] = new.cumsum(0)
    taken = (need - held).cumsum(0) - (need - held)  # pages that the requests in front take
    column = torch.arange(s["table"].shape[1], device=past.device)[None]
    fresh = (column >= held[:, None]) & (column < need[:, None])
    pick = (taken[:, None] + column - held[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][pick], s["table"])
    token = torch.arange(s["tokens"], device=past.device)
    request = torch.searchsorted(begin[1:], token, right=True)
    position = past[request] + token - begin[request]
    slots = table[request, position // page].long() * page + position % page
    return slots.int(), position.int(), begin.int(), total.int(), (need - held).sum().int().view(1), table


def _plain_rows(x, weight, s):
    """Norm and rotation of rows (tokens, heads, hd), in 32 bits; the angles in 64."""
    y = x.float()
    if s["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    angle = s["positions"].double()[:, None] * s["inv"][None]
    cos, sin = (angle.cos() * s["mscale"]).float()[:, None], (angle.sin() * s["mscale"]).float()[:, None]
    half = s["rotary"] // 2
    if s["interleaved"]:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype)


def _plain_prepare(s):
    at = s["slots"].long()
    s["q_out"].copy_(_plain_rows(s["q"], s["qw"], s))
    s["kp"].view(-1, s["nkv"], s["hd"])[at] = _plain_rows(s["k"], s["kw"], s)
    s["vp"].view(-1, s["nkv"], s["hd"])[at] = s["v"]
    return s["q_out"], s["kp"], s["vp"]


def _gated(out, gate):
    return out if gate is None else out * torch.sigmoid(gate.to(out.dtype))


def _plain_decode(s):
    nq, nkv, hd, page = s["nq"], s["nkv"], s["hd"], s["page"]
    out = torch.zeros(s["batch"], nq, hd, device=s["q"].device)
    lse = torch.full((s["batch"], nq), -math.inf, device=s["q"].device)
    for b, n in enumerate(s["lens_host"]):
        if n == 0:
            continue
        at = torch.arange(n, device=s["q"].device)
        if s["window"] and n > s["window"]:
            at = at[(at >= n - s["window"]) | (at < s["sinks"])]
        at = s["table"][b].long()[at // page] * page + at % page
        k, v = s["kp"].view(-1, nkv, hd)[at].float(), s["vp"].view(-1, nkv, hd)[at].float()
        q = s["q"][b].float().view(nkv, nq // nkv, hd)
        score = torch.matmul(q, k.permute(1, 2, 0)) * hd ** -0.5
        top = score.amax(-1, keepdim=True)
        e = torch.exp(score - top)
        z = e.sum(-1, keepdim=True)
        out[b] = (torch.matmul(e, v.transpose(0, 1)) / z).view(nq, hd)
        lse[b] = (top + torch.log(z)).view(nq)
    return _gated(out, s["g"]).to(s["q"].dtype), lse


def _plain_prefill(s):
    batch, seq, kv, nq, nkv, hd = s["batch"], s["seq"], s["kv"], s["nq"], s["nkv"], s["hd"]
    group, off, rows = nq // nkv, s["kv"] - s["seq"], 512
    out, lse = torch.empty_like(s["q"]), torch.empty(batch, seq, nq, device=s["q"].device)
    for t0 in range(0, seq, rows):  # rows of queries, the keys that some of them see
        t1 = min(seq, t0 + rows)
        lo = max(0, t0 + off - s["window"] + 1)
        first = min(lo, s["sinks"])
        at = torch.cat((torch.arange(first, device=out.device), torch.arange(lo, t1 + off, device=out.device)))
        own_at = torch.arange(t0 + off, t1 + off, device=out.device)[:, None]
        seen = (at[None] <= own_at) & ((at[None] > own_at - s["window"]) | (at[None] < s["sinks"]))
        k, v = s["k"][:, at].float().permute(0, 2, 3, 1), s["v"][:, at].float().transpose(1, 2)
        q = s["q"][:, t0:t1].float().view(batch, t1 - t0, nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, nkv, group * (t1 - t0), hd)
        score = (torch.matmul(q, k) * hd ** -0.5).view(batch, nkv, group, t1 - t0, -1)
        score = torch.where(seen, score, -math.inf)
        top = score.amax(-1, keepdim=True)
        e = torch.exp(score - top)
        z = e.sum(-1, keepdim=True)
        o = torch.matmul(e.view(batch, nkv, group * (t1 - t0), -1), v).view(batch, nkv, group, t1 - t0, hd) / z
        o = o.permute(0, 3, 1, 2, 4).reshape(batch, t1 - t0, nq, hd)
        out[:, t0:t1] = _gated(o, None if s["g"] is None else s["g"][:, t0:t1]).to(out.dtype)
        lse[:, t0:t1] = (top + torch.log(z)).squeeze(-1).permute(0, 3, 1, 2).reshape(batch, t1 - t0, nq)
    return out, lse


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"tables": _plain_tables, "prepare": _plain_prepare, "decode": _plain_decode, "prefill": _plain_prefill}[op](s)
    from arcaine_b200 import ops
    if op == "tables":
        slots, positions, begin, kv_len, used = ops.paged_tables(s["new"], s["past"], s["table"], s["free"], page_size=s["page"],
                                                                 num_tokens=s["tokens"])
        return slots, positions, begin, kv_len, used, s["table"]
    if op == "prepare":
        ops.qkv_prepare_paged(s["q"], s["k"], s["v"], s["positions"], s["inv"], k_pages=s["kp"], v_pages=s["vp"], slots=s["slots"],
                              norm=s["norm"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6, interleaved=s["interleaved"],
                              mscale=s["mscale"], q_out=s["q_out"])
        return s["q_out"], s["kp"], s["vp"]
    if op == "decode":
        out, _, lse = ops.sdpa_decode_paged(s["q"], s["kp"], s["vp"], s["table"], s["lens"], scale=s["hd"] ** -0.5,
                                            window=s["window"] or ops.NO_WINDOW, sinks=s["sinks"], gate=s["g"], return_partial=True)
        return out, lse
    return ops.sdpa_prefill(s["q"], s["k"], s["v"], scale=s["hd"] ** -0.5, mask_type=ops.MASK_CAUSAL, window=s["window"], sinks=s["sinks"],
                            gate=s["g"], return_lse=True)


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_tables(s):
    page, past, new, free = s["page"], s["past"].tolist(), s["new"].tolist(), s["free"].tolist()
    table = s["table"].tolist()
    slots, positions, begin, used = [], [], [0], 0
    for b, (p, n) in enumerate(zip(past, new)):
        for column in range(-(-p // page), -(-(p + n) // page)):
            table[b][column] = free[used]
            used += 1
        for at in range(p, p + n):
            positions.append(at)
            slots.append(table[b][at // page] * page + at % page)
        begin.append(begin[-1] + n)
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (slots, positions, begin, [p + n for p, n in zip(past, new)], [used], table))


def _exact_prepare(s):
    def rows(x, weight):
        y = x.double()
        if s["norm"]:
            y = y / torch.sqrt(torch.mean(y ** 2, dim=2, keepdim=True) + 1e-6) * weight.double()
        n = s["rotary"] // 2
        first = torch.arange(n, device=x.device) * (2 if s["interleaved"] else 1)
        second = first + (1 if s["interleaved"] else n)
        turn = torch.polar(torch.full((1, 1), s["mscale"], dtype=torch.float64, device=x.device).expand(x.shape[0], n),
                           torch.outer(s["positions"].double(), s["inv"]))
        z = torch.complex(y[:, :, first], y[:, :, second]) * turn[:, None, :]
        y[:, :, first], y[:, :, second] = z.real, z.imag
        return y

    kp, vp = s["kp"].double(), s["vp"].double()
    page, offset = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    kp[page, offset] = rows(s["k"], s["kw"])
    vp[page, offset] = s["v"].double()
    return rows(s["q"], s["qw"]), kp, vp


def _exact_attention(q, k, v, hidden, scale):
    """(rows, hd) over (keys, hd), hidden (rows, keys) or None: results and log-sum-exps."""
    score = (q @ k.T) * scale
    if hidden is not None:
        score.masked_fill_(hidden, -math.inf)
    lse = torch.logsumexp(score, dim=1)
    return torch.exp(score - lse[:, None]) @ v, lse


def _exact_decode(s):
    nq, nkv, hd, page = s["nq"], s["nkv"], s["hd"], s["page"]
    out = torch.zeros(s["batch"], nq, hd, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((s["batch"], nq), -math.inf, dtype=torch.float64, device=s["q"].device)
    group = nq // nkv
    for b, n in enumerate(s["lens_host"]):
        if n == 0:
            continue
        used = s["table"][b, :-(-n // page)].long()
        first = max(0, n - s["window"]) if s["window"] else 0
        keep = torch.ones(n, dtype=torch.bool, device=out.device)
        keep[min(s["sinks"], first):first] = False
        for h in range(nkv):
            k = s["kp"][used, :, h].reshape(-1, hd)[:n][keep].double()
            v = s["vp"][used, :, h].reshape(-1, hd)[:n][keep].double()
            o, l = _exact_attention(s["q"][b, h * group:(h + 1) * group].double(), k, v, None, hd ** -0.5)
            out[b, h * group:(h + 1) * group], lse[b, h * group:(h + 1) * group] = o, l
    if s["g"] is not None:
        out = out / (1.0 + torch.exp(-s["g"].double()))
    return out, lse


def _exact_prefill(s):
    batch, seq, kv, nq, nkv, hd = s["batch"], s["seq"], s["kv"], s["nq"], s["nkv"], s["hd"]
    group, off, rows = nq // nkv, kv - seq, 1024
    out = torch.empty(batch, seq, nq, hd, dtype=torch.float64, device=s["q"].device)
    lse = torch.empty(batch, seq, nq, dtype=torch.float64, device=s["q"].device)
    for b in range(batch):
        for h in range(nkv):
            k, v = s["k"][b, :, h].double(), s["v"][b, :, h].double()
            for t0 in range(0, seq, rows):
                t1 = min(seq, t0 + rows)
                lo, hi = max(0, t0 + off - s["window"] + 1), t1 + off
                near = torch.cat((k[:min(lo, s["sinks"])], k[lo:hi])), torch.cat((v[:min(lo, s["sinks"])], v[lo:hi]))
                key = torch.cat((torch.arange(min(lo, s["sinks"])), torch.arange(lo, hi))).to(out.device)
                at = torch.arange(t0 + off, t1 + off, device=out.device).unsqueeze(1)
                hidden = (key > at) | ((at - key >= s["window"]) & (key >= s["sinks"]))
                for i in range(group):
                    o, l = _exact_attention(s["q"][b, t0:t1, h * group + i].double(), *near, hidden, hd ** -0.5)
                    out[b, t0:t1, h * group + i], lse[b, t0:t1, h * group + i] = o, l
    if s["g"] is not None:
        out = out / (1.0 + torch.exp(-s["g"].double()))
    return out, lse


def exact(case, seed):
    return {"tables": _exact_tables, "prepare": _exact_prepare, "decode": _exact_decode, "prefill": _exact_prefill}[case["op"]](prepare(case, seed))
