"""Paged KV cache: tables, pre-processing with append, decode; each against its definition in 64 bits, and a run of them together.

Tolerances, derived: a bf16 rounding is off by at most half a step, 2^-8 of the value.  Attention rounds its probabilities for the second
product (2^-8 of sum p |v| at most, p normalised) and its result; fp32 sums and scores add less than 2^-9 of sum p |v| at these sizes.  Pre-processing
rounds once; its fp32 arithmetic adds less than 2^-18 of the pair (a row's reciprocal root, a weight, two products, a sum, an angle within 2^-21)."""
import math
import random

import pytest
import torch

from helpers import seeded_bf16

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def clean_status():
    from arcaine_b200 import ops
    ops.clear_device_status()
    yield
    ops.clear_device_status()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------
def plain_tables(new, past, table, free, page, num_tokens, begin=0):
    table = [list(r) for r in table]
    slots, positions, token_begin, used = [], [], [0], 0
    for b, (n, p) in enumerate(zip(new, past)):
        for column in range(-(-p // page), -(-(p + n) // page)):
            table[b][column] = free[begin + used] if begin + used < len(free) else -1
            used += 1
        for at in range(p, p + n):
            positions.append(at)
            slots.append(table[b][at // page] * page + at % page if table[b][at // page] >= 0 else -1)
        token_begin.append(len(slots))
    pad = [-1] * (num_tokens - len(slots))
    return slots + pad, positions + pad, token_begin, [n + p for n, p in zip(new, past)], [used], table


def make_step(seed, batch, page, most_past, most_new, short=0, begin=0):
    r = random.Random(seed)
    past = [r.choice([0, r.randint(0, most_past), page * r.randint(0, most_past // page), max(0, page * r.randint(0, most_past // page) - 1)]) for _ in range(batch)]
    new = [r.choice([0, 1, 1, r.randint(0, most_new)]) for _ in range(batch)]
    held = [-(-p // page) for p in past]
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    ids = list(range(sum(need) + begin + 3))
    r.shuffle(ids)
    width = max(need) + 2
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    free = ids[at:]
    return new, past, table, free[:len(free) - 3 - short], width


@pytest.mark.parametrize("batch,page,most_past,most_new,short,begin", [
    (1, 16, 40, 40, 0, 0), (3, 16, 0, 100, 0, 0), (8, 48, 500, 3, 0, 5), (33, 32, 900, 700, 0, 0), (257, 64, 300, 130, 0, 11),
    (2048, 16, 64, 5, 0, 0), (100, 256, 5000, 3000, 0, 0), (17, 16, 100, 90, 9, 2), (5, 16, 30, 30, 1000, 0)])
@pytest.mark.parametrize("pad", [0, 37])
def test_tables(batch, page, most_past, most_new, short, begin, pad):
    from arcaine_b200 import ops
    new, past, table, free, width = make_step(batch * 7 + page, batch, page, most_past, most_new, short, begin)
    tokens = sum(new) + pad
    wide = torch.full((batch, width + 5), -9, dtype=torch.int32, device=DEV)  # rows further apart than they are wide
    wide[:, :width] = ints(table)
    got = ops.paged_tables(ints(new), ints(past) if most_past else None, wide[:, :width], ints(free), page_size=page, num_tokens=tokens,
                           free_begin=ints([begin]) if begin else None)
    want = plain_tables(new, past, table, free, page, tokens, begin)
    for g, w in zip(got, want):
        assert g.dtype == torch.int32 and g.tolist() == w
    assert wide[:, :width].tolist() == want[5] and bool((wide[:, width:] == -9).all())
    assert ops.device_status() == (0, 0)
    # into tensors of the caller's; the same table again gives the same step
    out = tuple(torch.full_like(g, 5) for g in got)
    again = ops.paged_tables(ints(new), ints(past), wide[:, :width], ints(free), page_size=page, num_tokens=tokens,
                             free_begin=ints([begin]) if begin else None, out=out)
    assert again is out and all(torch.equal(a, g) for a, g in zip(again, got))


@pytest.mark.parametrize("new,past,tokens,detail", [([3, -1, 2], [4, 4, 4], 9, 1), ([3, 1, 2], [4, 4, -4], 9, 2), ([3, 1, 2], [4, 48, 4], 9, 1),
                                                    ([3, 49, 2], [0, 0, 0], 99, 1), ([3, 2**31 - 1, 2], [4, 2**31 - 1, 4], 9, 1), ([3, 4, 3], [4, 4, 4], 9, 3)])
def test_tables_bad_lengths_write_nothing(new, past, tokens, detail):
    from arcaine_b200 import ops
    table = torch.full((3, 3), 7, dtype=torch.int32, device=DEV)
    out = tuple(torch.full((n,), 5, dtype=torch.int32, device=DEV) for n in (tokens, tokens, 4, 3, 1))
    ops.paged_tables(ints(new), ints(past), table, ints(list(range(9))), page_size=16, num_tokens=tokens, out=out)
    assert ops.device_status() == (10, detail)
    assert bool((table == 7).all()) and all(bool((t == 5).all()) for t in out)
    ops.clear_device_status()


def test_tables_of_lengths_about_31_bits():
    """A row of large pages may name more keys than 32 bits count: what passes them is refused, what does not is served."""
    from arcaine_b200 import ops
    page, last = 2**30, 2**31 - 1
    for past, new, fits in ((last, 2, False), (last - 1, 2, False), (2, last, False), (last - 2, 2, True), (last, 0, True)):
        table = ints([[0, 1, -7, -7], [0, 1, -7, -7]])
        out = tuple(torch.full((n,), 5, dtype=torch.int32, device=DEV) for n in (2, 2, 3, 2, 1))
        ops.paged_tables(ints([0, new]), ints([7, past]), table, ints([3, 4]), page_size=page, num_tokens=2, out=out)
        assert ops.device_status() == ((0, 0) if fits else (10, 1))
        ops.clear_device_status()
        if fits:
            want = plain_tables([0, new], [7, past], [[0, 1, -7, -7]] * 2, [3, 4], page, 2)
            assert [t.tolist() for t in out] == list(want[:5]) and table.tolist() == want[5]
        else:
            assert bool((table[:, 2:] == -7).all()) and all(bool((t == 5).all()) for t in out)


def test_tables_refusals():
    from arcaine_b200 import ops
    one, table, free = ints([1, 1]), torch.zeros(2, 4, dtype=torch.int32, device=DEV), ints([1, 2, 3])
    good = dict(page_size=16, num_tokens=2)
    with pytest.raises(ValueError, match="past_len"):
        ops.paged_tables(one, ints([1]), table, free, **good)
    with pytest.raises(ValueError, match="block_table"):
        ops.paged_tables(one, None, table.t(), free, **good)
    with pytest.raises(ValueError, match="block_table"):
        ops.paged_tables(one, None, table.long(), free, **good)
    with pytest.raises(ValueError, match="num_tokens"):
        ops.paged_tables(one, None, table, free, page_size=16, num_tokens=-1)
    with pytest.raises(ops.ArcError):
        ops.paged_tables(one, None, table, free, page_size=15, num_tokens=2)
    past = ints([3, 4])
    with pytest.raises(ValueError, match="kv_len overlaps"):
        ops.paged_tables(one, past, table, free, **good, out=(ints([0, 0]), ints([0, 0]), ints([0, 0, 0]), past, ints([0])))
    shared = ints([0, 0, 0, 0])
    with pytest.raises(ValueError, match="positions overlaps"):
        ops.paged_tables(one, past, table, free, **good, out=(shared[:2], shared[1:3], ints([0, 0, 0]), ints([0, 0]), ints([0])))
    with pytest.raises(ValueError, match="out must be"):
        ops.paged_tables(one, past, table, free, **good, out=(shared[:2],))


# ---------------------------------------------------------------------------
# pre-processing
# ---------------------------------------------------------------------------
def plain_rows(x, positions, inv, interleaved, norm, weight, mscale, eps=1e-6):
    """In 64 bits: rows (tokens, heads, hd) and the size that each value's rounding errors go by."""
    y = x.double()
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    size = y.abs()
    half = 0 if inv is None else inv.numel()
    if half:
        a = torch.arange(half, device=x.device) * (2 if interleaved else 1)
        b = a + (1 if interleaved else half)
        angle = positions.double()[:, None] * inv[None]
        c, s = angle.cos()[:, None] * mscale, angle.sin()[:, None] * mscale
        ya, yb = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = ya * c - yb * s, ya * s + yb * c
        size = size.clone()
        size[..., a] = size[..., b] = (ya.abs() + yb.abs()) * max(1.0, abs(mscale))
    return y, size


def assert_rows(got, want, size):
    off = (got.double() - want).abs()
    room = want.abs() * 2.0 ** -8 + size * 2.0 ** -18 + 1e-30
    assert bool((off <= room).all()), f"off by {(off / room).max().item():.2f} of the tolerance"


PREPARE = [  # tokens, nq, nkv, hd, rotary, interleaved, norm, v_norm, weights, page, far
    (1, 8, 4, 128, 128, False, True, False, True, 16, 0), (3, 24, 4, 256, 64, False, True, False, True, 16, 777),
    (64, 24, 4, 256, 256, True, False, False, False, 48, 10**6), (37, 7, 7, 128, 48, True, True, True, True, 32, 2**31 - 200),
    (130, 28, 4, 128, 128, False, False, False, False, 64, 500000), (5, 4, 2, 512, 512, False, True, True, True, 16, 9),
    (19, 4, 1, 512, 96, True, True, False, False, 16, 123456789), (2500, 8, 2, 128, 32, False, True, False, True, 128, 0),
    (11, 16, 1, 128, 0, False, True, False, True, 256, 50), (700, 5, 5, 256, 16, True, True, False, True, 16, 31)]


@pytest.mark.parametrize("tokens,nq,nkv,hd,rotary,interleaved,norm,v_norm,weights,page,far", PREPARE)
def test_prepare(tokens, nq, nkv, hd, rotary, interleaved, norm, v_norm, weights, page, far):
    """Rows of a fused projection, some tokens padding, some not appended; everything else stays as it was."""
    from arcaine_b200 import ops
    width = (nq + 2 * nkv) * hd + 8
    fused = seeded_bf16(tokens, width, seed=tokens + hd).cuda()
    q = fused[:, :nq * hd].view(tokens, nq, hd)
    k = fused[:, nq * hd:(nq + nkv) * hd].view(tokens, nkv, hd)
    v = fused[:, (nq + nkv) * hd:(nq + 2 * nkv) * hd].view(tokens, nkv, hd)
    qw, kw = [(1 + 0.2 * seeded_bf16(hd, seed=s).float()).bfloat16().cuda() if weights and norm else None for s in (2, 3)]
    inv, mscale = ops.rope_frequencies(rotary, 1e4, scaling="yarn", factor=8.0, original_len=4096, device=DEV) if rotary else (None, 1.0)
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens].int()
    positions = (far + torch.arange(tokens)).int()
    if tokens > 4:
        positions[::5] = -1   # padding
        slots[1::5] = -1      # not appended
    slots, positions = slots.to(DEV), positions.to(DEV)
    both = torch.full((pages, 2, page, nkv, hd), 7.0, dtype=torch.bfloat16, device=DEV)  # K and V pages side by side
    kp, vp = both[:, 0], both[:, 1]
    q_out = torch.full((tokens, nq, hd), 9.0, dtype=torch.bfloat16, device=DEV)
    k_out = torch.full((tokens, nkv, hd), 9.0, dtype=torch.bfloat16, device=DEV)
    before = fused.clone()
    ops.qkv_prepare_paged(q, k, v, positions, inv, k_pages=kp, v_pages=vp, slots=slots, norm=norm, v_norm=v_norm, q_weight=qw, k_weight=kw,
                          interleaved=interleaved, mscale=mscale, q_out=q_out, k_out=k_out)
    assert ops.device_status() == (0, 0)
    assert torch.equal(fused, before)
    live = positions >= 0
    wq, sq = plain_rows(q, positions, inv, interleaved, norm, qw, mscale)
    wk, sk = plain_rows(k, positions, inv, interleaved, norm, kw, mscale)
    wv, sv = plain_rows(v, positions, None, False, v_norm, None, 1.0)
    assert_rows(q_out[live], wq[live], sq[live])
    assert_rows(k_out[live], wk[live], sk[live])
    assert bool((q_out[~live] == 9.0).all()) and bool((k_out[~live] == 9.0).all())
    stored = live & (slots >= 0)
    at = slots[stored].long()
    assert torch.equal(kp[at // page, at % page], k_out[stored])
    if v_norm:
        assert_rows(vp[at // page, at % page], wv[stored], sv[stored])
    else:
        assert torch.equal(vp[at // page, at % page], v[stored])
    rest = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    rest[at] = False
    rest = rest.view(pages, page)
    assert bool((kp[rest] == 7.0).all()) and bool((vp[rest] == 7.0).all())
    # in place, without a cache: the same rows
    ops.qkv_prepare_paged(q, k, v, positions, inv, norm=norm, v_norm=v_norm, q_weight=qw, k_weight=kw, interleaved=interleaved, mscale=mscale)
    assert torch.equal(q[live], q_out[live]) and torch.equal(k[live], k_out[live])
    assert torch.equal(q[~live], before[:, :nq * hd].view(tokens, nq, hd)[~live])
    assert torch.equal(fused[:, -8:], before[:, -8:])


def test_prepare_angles_of_far_positions():
    """Positions close to multiples of pi, the numerators of its convergents among them: the sine is small, and bf16 shows the angle to 2^-8 of
    it.  A position may be off by 1e-6 rad: three roundings to 64 bits, 3 * 2^-53 * 2^31 = 7.2e-7, and one to fp32, 2 pi 2^-26 = 9.4e-8."""
    from decimal import Decimal, getcontext

    from arcaine_b200 import ops
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    far = [355, 103993, 80143857, 165707065, 245850922, 411557987, 1068966896, 2 * 1068966896, 2**31 - 1, 2**31 - 2, 1068966896 + 355, 1068966896 + 103993]
    far += [int(round(pi * n)) for n in range(650000000, 683000000, 1999999)]
    x = torch.zeros(len(far), 1, 128, dtype=torch.bfloat16, device=DEV)
    x[..., 0] = 1.0
    inv = torch.zeros(8, dtype=torch.float64, device=DEV)
    inv[0] = 1.0
    ops.qkv_prepare_paged(x, None, None, ints(far), inv, norm=False)
    for at, c, s in zip(far, x[:, 0, 0].tolist(), x[:, 0, 8].tolist()):
        half_turns = int((Decimal(at) / pi).to_integral_value())
        rest = float(Decimal(at) - pi * half_turns)
        want = math.sin(rest) * (-1) ** half_turns, math.cos(rest) * (-1) ** half_turns
        assert abs(s - want[0]) <= 1e-6 + 2.0 ** -8 * abs(want[0]), at
        assert abs(c - want[1]) <= 1e-6 + 2.0 ** -8 * abs(want[1]), at


def test_prepare_only_queries_or_only_keys():
    from arcaine_b200 import ops
    q, k = seeded_bf16(9, 4, 128, seed=1).cuda(), seeded_bf16(9, 2, 128, seed=2).cuda()
    positions, inv = ints(list(range(9))), ops.rope_frequencies(128, device=DEV)[0]
    both_q, both_k, alone_q, alone_k = q.clone(), k.clone(), q.clone(), k.clone()
    ops.qkv_prepare_paged(both_q, both_k, None, positions, inv)
    ops.qkv_prepare_paged(alone_q, None, None, positions, inv)
    ops.qkv_prepare_paged(None, alone_k, None, positions, inv)
    assert torch.equal(both_q, alone_q) and torch.equal(both_k, alone_k)
    pages = torch.zeros(1, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    ops.qkv_prepare_paged(None, k, None, positions, inv, k_pages=pages, slots=positions)
    assert torch.equal(pages[0, :9], alone_k) and bool((pages[0, 9:] == 0).all())


def test_prepare_bad_slots_are_not_written():
    from arcaine_b200 import ops
    k, v = seeded_bf16(6, 2, 128, seed=1).cuda(), seeded_bf16(6, 2, 128, seed=2).cuda()
    for bad, token in ((48, 3), (-2, 3), (2**31 - 1, 3)):
        kp, vp = (torch.full((4, 16, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        ops.qkv_prepare_paged(None, k, v, ints(list(range(6))), None, k_pages=kp[:3], v_pages=vp[:3], slots=ints([5, 6, 7, bad, 8, 9]), norm=False)
        assert ops.device_status() == (10, token)
        assert bool((kp[3] == 7.0).all()) and torch.equal(kp[0, [5, 6, 7, 8, 9]], k[[0, 1, 2, 4, 5]])
        ops.clear_device_status()


@pytest.mark.parametrize("bad", [[0], [0, 12345, 29999]])
def test_prepare_bad_slots_cost_no_other_token(bad):
    """CTAs that start behind another stream's kernel find the status that a bad slot of their own call has set."""
    from arcaine_b200 import ops
    tokens, page = 30000, 16
    q, k, v = (seeded_bf16(tokens, n, 128, seed=n).cuda() for n in (4, 2, 2))
    positions, inv = torch.arange(tokens, dtype=torch.int32, device=DEV), ops.rope_frequencies(128, device=DEV)[0]
    slots = torch.arange(tokens, dtype=torch.int32, device=DEV)
    good = torch.ones(tokens, dtype=torch.bool, device=DEV)
    for t in bad:
        slots[t], good[t] = 2**30 + t, False
    want_q, want_k = q.clone(), k.clone()
    ops.qkv_prepare_paged(want_q, want_k, None, positions, inv)
    side, busy = torch.cuda.Stream(), seeded_bf16(8192, 8192, seed=9).cuda()

    def call(got_q, kp, vp):
        ops.qkv_prepare_paged(got_q, k, v, positions, inv, k_pages=kp, v_pages=vp, slots=slots)

    for captured in (False, True):
        got_q, kp, vp = q.clone(), *(torch.full((tokens // page + 1, page, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call(got_q, kp, vp)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.mm(busy, busy)
        if captured:
            graph.replay()
        else:
            call(got_q, kp, vp)
        code, detail = ops.device_status()
        assert code == 10 and detail in bad
        assert torch.equal(got_q, want_q)
        for pages, rows in ((kp, want_k), (vp, v)):
            pages = pages.view(-1, 2, 128)
            assert torch.equal(pages[:tokens][good], rows[good])
            assert bool((pages[:tokens][~good] == 7.0).all()) and bool((pages[tokens:] == 7.0).all())
        # a later call finds a status that is not its own: nothing is done
        later = q.clone()
        call(later, kp.fill_(5.0), vp.fill_(5.0))
        assert torch.equal(later, q) and bool((kp == 5.0).all()) and bool((vp == 5.0).all())
        assert ops.device_status() == (code, detail)
        ops.clear_device_status()


def test_a_step_of_no_tokens():
    from arcaine_b200 import ops
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    slots, positions, begin, kv_len, used = ops.paged_tables(ints([0, 0]), ints([3, 0]), table, ints([]), page_size=16, num_tokens=0)
    assert slots.shape == positions.shape == (0,) and begin.tolist() == [0, 0, 0] and kv_len.tolist() == [3, 0] and used.tolist() == [0]
    q, k = (torch.empty(0, n, 128, dtype=torch.bfloat16, device=DEV) for n in (4, 2))
    pages = torch.full((2, 16, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    launches = ops.launch_count()
    ops.qkv_prepare_paged(q, k, k, positions, ops.rope_frequencies(128, device=DEV)[0], k_pages=pages, v_pages=pages, slots=slots)
    ops.qkv_prepare_paged(q, None, None, positions, None, q_out=q.clone())
    assert ops.launch_count() == launches and bool((pages == 7.0).all()) and ops.device_status() == (0, 0)


def test_prepare_refusals():
    from arcaine_b200 import ops
    q, k = seeded_bf16(4, 4, 128, seed=1).cuda(), seeded_bf16(4, 2, 128, seed=2).cuda()
    positions, pages = ints([0, 1, 2, 3]), torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    inv = ops.rope_frequencies(128, device=DEV)[0]
    for args, kw, text in (((None, None, None), {}, "needs q or k"), ((q, None, k), {}, "v needs k"), ((q, k, k), dict(k_pages=pages), "go together"),
                           ((q, k, k), dict(k_pages=pages, v_pages=pages), "slots"), ((q, k, None), dict(k_pages=pages, v_pages=pages), "v_pages needs v"),
                           ((q, k[:3], None), {}, "k must be"), ((q, k, None), dict(norm=False, q_weight=q[0, 0]), "norm=True"),
                           ((q, k, k), dict(k_pages=pages, v_pages=pages[:1], slots=positions), "same number"),
                           ((q, k, k), dict(k_pages=pages[..., :64], v_pages=pages, slots=positions), "k_pages must be"),
                           ((q.transpose(0, 1), None, None), {}, "must be contiguous"), ((q, None, None), dict(k_pages=pages), "need k and v")):
        with pytest.raises(ValueError, match=text):
            ops.qkv_prepare_paged(*args, positions, inv, **kw)
    with pytest.raises(ValueError, match="float64"):
        ops.qkv_prepare_paged(q, None, None, positions, inv.float())
    with pytest.raises(ValueError, match="inv_freq"):
        ops.qkv_prepare_paged(q, None, None, positions, torch.cat((inv, inv)))
    with pytest.raises(ops.ArcError):
        ops.qkv_prepare_paged(q, None, None, positions, inv[:7])
    with pytest.raises(ValueError, match="positions"):
        ops.qkv_prepare_paged(q, None, None, positions[:3], inv)


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def visible(n, window, sinks):
    at = torch.arange(n, device=DEV)
    return at if window is None or window >= n else at[(at >= n - window) | (at < sinks)]


def plain_decode(q, kp, vp, table, lens, window, sinks, scale, gate=None):
    """In 64 bits: results, log-sum-exps, and sum p |v|."""
    batch, nq, hd = q.shape
    page, nkv = kp.shape[1:3]
    out = torch.zeros(batch, nq, hd, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    lse = torch.full((batch, nq), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        at = visible(n, window, sinks)
        where = table[b].long()[at // page], at % page
        k, v = kp[where].double().transpose(0, 1), vp[where].double().transpose(0, 1)  # (nkv, keys, hd)
        s = torch.matmul(q[b].double().view(nkv, nq // nkv, hd), k.transpose(1, 2)) * scale
        lse[b] = torch.logsumexp(s, -1).view(nq)
        p = torch.softmax(s, -1)
        out[b], size[b] = torch.matmul(p, v).view(nq, hd), torch.matmul(p, v.abs()).view(nq, hd)
    if gate is not None:
        out, size = out * torch.sigmoid(gate.double()), size * torch.sigmoid(gate.double())
    return out, lse, size


def assert_attention(out, lse, want, want_lse, size, rounded=True):
    off = (out.double() - want).abs()
    room = size * (2.0 ** -8 + 2.0 ** -9) + (want.abs() * 2.0 ** -8 if rounded else 0.0) + 1e-30
    assert bool(torch.isfinite(out).all())
    assert bool((off <= room).all()), f"off by {(off / room).max().item():.2f} of the tolerance"
    if lse is not None:
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all())
        # scores of hd products in fp32: 2^-24 of their absolute sum each; logarithm and exponentials a few 2^-22
        assert bool(((lse.double() - want_lse).abs()[~empty] <= 2e-4 + 2.0 ** -20 * want_lse.abs()[~empty]).all())


def paged_case(lens, page, nq, nkv, hd, window, sinks, seed, interleave=False, poison=True):
    """A batch whose pool holds NaN wherever no token of it looks, and a table whose other entries are not pages."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(0, n) // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g).int()
    width = max(max(need), 1) + 1
    table = torch.full((len(lens), width), -5, dtype=torch.int32)
    table[:, ::2] = 10**9
    at = 0
    shape = (pages, 2, page, nkv, hd) if interleave else (2, pages, page, nkv, hd)
    both = torch.full(shape, math.nan if poison else 3.0, dtype=torch.bfloat16, device=DEV)
    kp, vp = (both[:, 0], both[:, 1]) if interleave else (both[0], both[1])
    if poison:
        vp.fill_(math.inf)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        own = order[at:at + need[b]]
        at += need[b]
        seen = visible(n, window, sinks)
        columns = torch.unique(seen // page).cpu()
        table[b, columns] = own[columns]
        where = own.to(DEV).long()[seen // page], seen % page
        kp[where] = torch.randn(len(seen), nkv, hd, generator=g).bfloat16().to(DEV)
        vp[where] = torch.randn(len(seen), nkv, hd, generator=g).bfloat16().to(DEV)
    q = torch.randn(len(lens), nq, hd, generator=g).bfloat16().to(DEV)
    gate = torch.randn(len(lens), nq, hd, generator=g).bfloat16().to(DEV)
    return q, kp, vp, table.to(DEV), gate


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300, 1000, -3]


@pytest.mark.parametrize("nq,nkv,hd", [(8, 4, 128), (24, 4, 256), (7, 7, 128), (16, 1, 128), (16, 2, 256), (28, 4, 128), (32, 16, 128), (4, 4, 256), (9, 3, 256)])
@pytest.mark.parametrize("ctas", [0, 148])  # (0: the library's choice, here nearly always one launch; else two)
@pytest.mark.parametrize("page,window,sinks", [(16, None, 0), (48, None, 3), (32, 20, 0), (64, 17, 4), (16, 1, 1), (256, 100, 40), (16, 33, 17), (128, 64, 1000)])
def test_decode_edges(nq, nkv, hd, page, window, sinks, ctas):
    """Lengths about the ends of slices and pages, behind windows and sinks of all sizes; what nobody sees is NaN and infinite."""
    from arcaine_b200 import ops
    scale = hd ** -0.5
    launches = ops.launch_count()
    q, kp, vp, table, gate = paged_case(EDGES, page, nq, nkv, hd, window, sinks, seed=nq + page, interleave=page == 32)
    w = ops.NO_WINDOW if window is None else window
    want, want_lse, size = plain_decode(q, kp, vp, table, EDGES, window, sinks, scale)
    out, o32, lse = ops.sdpa_decode_paged(q, kp, vp, table, ints(EDGES), scale=scale, window=w, sinks=sinks, return_partial=True, num_ctas=ctas)
    assert ops.device_status() == (0, 0) and ops.launch_count() - launches == (2 if ctas or (nkv == 16 and window is None) else 1)
    assert_attention(out, lse, want, want_lse, size)
    assert_attention(o32, None, want, want_lse, size, rounded=False)
    want, _, size = plain_decode(q, kp, vp, table, EDGES, window, sinks, scale, gate)
    got = ops.sdpa_decode_paged(q, kp, vp, table, ints(EDGES), scale=scale, window=w, sinks=sinks, gate=gate, num_ctas=ctas)
    assert_attention(got, None, want, want_lse, size)
    again = ops.sdpa_decode_paged(q, kp, vp, table, ints(EDGES), scale=scale, window=w, sinks=sinks, gate=gate, num_ctas=ctas)
    assert torch.equal(got, again)


@pytest.mark.parametrize("nq,nkv,hd", [(9, 1, 256), (16, 1, 256), (24, 2, 256), (39, 3, 256), (9, 1, 128), (60, 4, 128)])
@pytest.mark.parametrize("ctas", [0, 148])
@pytest.mark.parametrize("page,window,sinks", [(16, None, 0), (32, 20, 0), (64, 17, 4), (16, 33, 17)])
def test_decode_wide_groups(nq, nkv, hd, page, window, sinks, ctas):
    """More than eight query heads to a KV head: two warps divide them, the second with fewer heads than the first."""
    from arcaine_b200 import ops
    q, kp, vp, table, gate = paged_case(EDGES, page, nq, nkv, hd, window, sinks, seed=nq + page, interleave=page == 32)
    more = dict(scale=hd ** -0.5, window=ops.NO_WINDOW if window is None else window, sinks=sinks, num_ctas=ctas)
    want, want_lse, size = plain_decode(q, kp, vp, table, EDGES, window, sinks, hd ** -0.5)
    out, o32, lse = ops.sdpa_decode_paged(q, kp, vp, table, ints(EDGES), return_partial=True, **more)
    assert ops.device_status() == (0, 0)
    assert_attention(out, lse, want, want_lse, size)
    assert_attention(o32, None, want, want_lse, size, rounded=False)
    want, _, size = plain_decode(q, kp, vp, table, EDGES, window, sinks, hd ** -0.5, gate)
    assert_attention(ops.sdpa_decode_paged(q, kp, vp, table, ints(EDGES), gate=gate, **more), None, want, want_lse, size)


@pytest.mark.parametrize("lens,page,nq,nkv,hd,window,sinks,ctas", [
    ([5000], 16, 24, 4, 256, None, 0, 0), ([70001, 3], 64, 16, 2, 128, None, 0, 0), ([9000] * 40, 32, 28, 4, 128, 1024, 4, 0), ([513], 16, 8, 8, 128, None, 0, 0),
    ([800, 7, 2000, 0, 31], 16, 8, 2, 256, None, 0, 1), ([800, 7, 2000, 0, 31], 16, 8, 4, 128, 500, 20, 3), ([3000, 100], 48, 32, 16, 128, None, 0, 1000),
    ([1] * 2000, 16, 4, 4, 128, None, 0, 0), ([300] * 129, 128, 16, 1, 256, 64, 1, 0), ([0, 0, 0], 16, 8, 4, 128, None, 0, 0),
    ([0, 0, 0], 16, 8, 4, 128, None, 0, 7), ([5000, 4000, 17], 16, 8, 4, 256, 4090, 2**31 - 1, 0), ([5000, 4000, 17], 32, 16, 2, 128, 2**31 - 2, 9, 0),
    ([4096] * 9, 16, 4, 2, 128, None, 0, 1), ([257] * 700, 16, 8, 1, 256, None, 0, 0)])
def test_decode_sizes(lens, page, nq, nkv, hd, window, sinks, ctas):
    from arcaine_b200 import ops
    q, kp, vp, table, _ = paged_case(lens, page, nq, nkv, hd, window, sinks, seed=len(lens))
    want, want_lse, size = plain_decode(q, kp, vp, table, lens, window, sinks, hd ** -0.5)
    out, _, lse = ops.sdpa_decode_paged(q, kp, vp, table, ints(lens), scale=hd ** -0.5, window=ops.NO_WINDOW if window is None else window, sinks=sinks,
                                        return_partial=True, num_ctas=ctas)
    assert ops.device_status() == (0, 0)
    assert_attention(out, lse, want, want_lse, size)


def test_decode_length_on_the_host_and_own_buffers():
    from arcaine_b200 import ops
    lens = [300, 300, 300]
    q, kp, vp, table, gate = paged_case(lens, 32, 8, 2, 128, None, 0, seed=3)
    wide = torch.full((3, 9, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    gates = torch.zeros_like(wide)
    gates[:, :8] = gate
    ws = ops.Workspace(torch.device(DEV))
    got = ops.sdpa_decode_paged(q, kp, vp, table, 300, scale=0.1, gate=gates[:, :8], out=wide[:, :8], workspace=ws)
    assert got.data_ptr() == wide.data_ptr() and bool((wide[:, 8] == 5.0).all())
    assert torch.equal(got, ops.sdpa_decode_paged(q, kp, vp, table, ints(lens), scale=0.1, gate=gate))
    none, o32, lse = ops.sdpa_decode_paged(q, kp, vp, table, 300, scale=0.1, want_out=False, return_partial=True)
    assert none is None and o32.dtype == torch.float32
    assert torch.equal(ops.sdpa_decode_paged(q, kp, vp, table, 300, scale=0.1, out=q), o32.bfloat16())  # over the queries
    assert ops.device_status() == (0, 0)


def test_views_of_one_head_or_one_token():
    """Where a dimension has one element its stride means nothing: transposed views are taken as they come."""
    from arcaine_b200 import ops
    positions, inv = ints([3, 4, 5]), ops.rope_frequencies(128, device=DEV)[0]
    k = seeded_bf16(1, 3, 128, seed=1).cuda().transpose(0, 1)  # (3, 1, 128)
    want_k = k.contiguous()
    pool = torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16, device=DEV)  # one head, in front of the rows
    want_pool = torch.zeros(2, 16, 1, 128, dtype=torch.bfloat16, device=DEV)
    slots = ints([17, 0, 18])
    ops.qkv_prepare_paged(None, want_k.clone(), want_k.clone(), positions, inv, k_pages=want_pool, v_pages=want_pool.clone(), slots=slots)
    ops.qkv_prepare_paged(None, k, k.clone(), positions, inv, k_pages=pool.transpose(1, 2), v_pages=pool.clone().transpose(1, 2), slots=slots)
    assert torch.equal(pool.transpose(1, 2), want_pool) and bool(want_pool.any())
    q = seeded_bf16(4, 1, 128, seed=2).cuda().transpose(0, 1)  # (1, 4, 128)
    got, want = torch.empty_like(q), torch.empty_like(q)
    ops.qkv_prepare_paged(q, None, None, positions[:1], inv, q_out=got)
    ops.qkv_prepare_paged(q.clone(memory_format=torch.contiguous_format).reshape(4, 128)[None], None, None, positions[:1], inv, q_out=want)
    assert torch.equal(got, want)
    pages, table = seeded_bf16(2, 1, 16, 128, seed=3).cuda(), ints([[1, 0]])
    dense = pages.transpose(1, 2).reshape(2, 16, 1, 128).clone()
    out = torch.empty(4, 1, 128, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    ops.sdpa_decode_paged(q, pages.transpose(1, 2), pages.transpose(1, 2), table, 20, scale=0.1, out=out)
    want = ops.sdpa_decode_paged(q.reshape(4, 128)[None], dense, dense, table, 20, scale=0.1)
    assert ops.device_status() == (0, 0) and torch.equal(out, want)


def test_tables_of_one_column_out_of_a_transposed_list():
    """(B, 1) with a stride of B behind the last dimension, which has one element."""
    from arcaine_b200 import ops
    pages, q = seeded_bf16(5, 16, 2, 128, seed=3).cuda(), seeded_bf16(3, 4, 128, seed=4).cuda()
    table = ints([[4, 0, 2]]).t()
    assert table.stride() == (1, 3)
    lens = ints([16, 1, 9])
    got = ops.sdpa_decode_paged(q, pages, pages, table, lens, scale=0.1)
    assert torch.equal(got, ops.sdpa_decode_paged(q, pages, pages, table.clone(memory_format=torch.contiguous_format), lens, scale=0.1))
    new, past, table = ints([1, 2, 0]), ints([3, 0, 0]), ints([[4, -7, -7]]).t()
    step = ops.paged_tables(new, past, table, ints([1, 3]), page_size=16, num_tokens=3)
    want = plain_tables([1, 2, 0], [3, 0, 0], [[4], [-7], [-7]], [1, 3], 16, 3)
    assert [t.tolist() for t in step] == list(want[:5]) and table.tolist() == want[5]
    with pytest.raises(ValueError, match="block_table"):  # rows in one place
        ops.sdpa_decode_paged(q, pages, pages, ints([[0]]).expand(3, 1), lens, scale=0.1)
    assert ops.device_status() == (0, 0)


def test_decode_infinite_and_missing_numbers_stay_in_their_row():
    from arcaine_b200 import ops
    lens = [700, 700, 700]
    q, kp, vp, table, _ = paged_case(lens, 16, 4, 2, 128, None, 0, seed=5)
    want = ops.sdpa_decode_paged(q, kp, vp, table, 700, scale=0.09)
    want2 = ops.sdpa_decode_paged(q, kp, vp, table, 700, scale=0.09, num_ctas=148)
    for value in (math.nan, math.inf):
        bad = q.clone()
        bad[1, 0, 5] = value
        for ctas, w in ((0, want), (148, want2)):
            out, _, lse = ops.sdpa_decode_paged(bad, kp, vp, table, 700, scale=0.09, return_partial=True, num_ctas=ctas)
            assert bool(torch.isnan(out[1, 0]).all()) and bool(torch.isnan(lse[1, 0]))
            keep = torch.ones(3, 4, dtype=torch.bool, device=DEV)
            keep[1, 0] = False
            assert torch.equal(out[keep], w[keep]) and bool(torch.isfinite(lse[keep]).all())


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("batch,nq,nkv,ctas,n", [(2, 4, 2, 0, 300), (130, 8, 2, 0, 100), (1, 2, 1, 148, 300), (20, 8, 2, 148, 300), (200, 8, 2, 148, 100)])
@pytest.mark.parametrize("value,factor", [(-math.inf, 1.0), (-1e38, 100.0)])
def test_decode_scores_of_minus_infinity(hd, batch, nq, nkv, ctas, n, value, factor):
    """Keys whose scores are all -inf, or pass fp32: zeros and a log-sum-exp of -inf, as without keys, in one launch and behind each merge.  The
    first sequence has one key with a score of its own, which takes all the weight."""
    from arcaine_b200 import ops
    page = 16
    width = -(-n // page)
    table = torch.arange(batch * width, dtype=torch.int32, device=DEV).view(batch, width)
    kp = torch.full((batch * width, page, nkv, hd), value, dtype=torch.bfloat16, device=DEV)
    vp = seeded_bf16(batch * width, page, nkv, hd, seed=hd).cuda()
    q = ((1 + seeded_bf16(batch, nq, hd, seed=2).float().abs()) * factor).bfloat16().cuda()
    for one in (False, True):
        if one:
            kp[width - 1, 0] = 0.5
        out, o32, lse = ops.sdpa_decode_paged(q, kp, vp, table, ints([n] * batch), scale=0.1, return_partial=True, num_ctas=ctas)
        assert bool((out[int(one):] == 0).all()) and bool((o32[int(one):] == 0).all()) and bool((lse[int(one):] == -math.inf).all())
        if one:
            seen = vp[width - 1, 0].repeat_interleave(nq // nkv, 0)
            assert torch.equal(out[0], seen) and bool(torch.isfinite(lse[0]).all())
    assert ops.device_status() == (0, 0)


def test_decode_large_scores():
    """One key takes all the weight, and scores of some thousand neither overflow nor lose the others' rows."""
    from arcaine_b200 import ops
    lens = [500, 33]
    q, kp, vp, table, _ = paged_case(lens, 16, 4, 1, 128, None, 0, seed=6, poison=False)
    q = (q.float() * 60).bfloat16()
    want, want_lse, size = plain_decode(q, kp, vp, table, lens, None, 0, 1.0)
    for ctas in (0, 148):
        out, _, lse = ops.sdpa_decode_paged(q, kp, vp, table, ints(lens), scale=1.0, return_partial=True, num_ctas=ctas)
        large_scores_hold(out, lse, want, want_lse, size)


def large_scores_hold(out, lse, want, want_lse, size):
    # a score is off by up to 128 products in fp32, of values up to 800: 2^-24 * 128 * 800 * 4 = 0.025, and so is the exponent
    assert bool(((lse.double() - want_lse).abs() <= 0.03).all())
    assert bool(((out.double() - want).abs() <= size * (2 * 0.026 + 2.0 ** -8) + want.abs() * 2.0 ** -8).all())


def test_decode_far_pages():
    """A pool whose last pages lie behind 2^32 elements."""
    from arcaine_b200 import ops
    nkv, hd, page = 8, 128, 64
    pages = (2**32 // (page * nkv * hd)) + 40
    pool = torch.empty(pages, page, nkv, hd, dtype=torch.bfloat16, device=DEV)
    lens = [250, 64]
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[pages - 1, 0, pages - 7, pages - 2], [pages - 30, 0, 0, 0]], dtype=torch.int32)
    for b, n in enumerate(lens):
        for c in range(-(-n // page)):
            pool[table[b, c]] = torch.randn(page, nkv, hd, generator=g).bfloat16().to(DEV)
    q = torch.randn(2, 16, hd, generator=g).bfloat16().to(DEV)
    out, _, lse = ops.sdpa_decode_paged(q, pool, pool, table.to(DEV), ints(lens), scale=0.08, return_partial=True)
    want, want_lse, size = plain_decode(q, pool, pool, table.to(DEV), lens, None, 0, 0.08)
    assert_attention(out, lse, want, want_lse, size)
    # and the append there
    k = seeded_bf16(3, nkv, hd, seed=4).cuda()
    at = ints([(pages - 1) * page + 63, 5, (pages - 3) * page + 1])
    ops.qkv_prepare_paged(None, k, k, ints([1, 2, 3]), None, k_pages=pool, v_pages=pool, slots=at, norm=False)
    assert torch.equal(pool[at.long() // page, at.long() % page], k)
    assert ops.device_status() == (0, 0)


@pytest.mark.parametrize("what", ["page", "negative page", "length"])
def test_decode_bad_pages_and_lengths(what):
    from arcaine_b200 import ops
    lens = [100, 90, 80]
    q, kp, vp, table, _ = paged_case(lens, 16, 8, 2, 128, None, 0, seed=7)
    if what == "length":
        lens[1] = table.shape[1] * 16 + 1
    else:
        table[1, 2] = kp.shape[0] if what == "page" else -1
    out = torch.full_like(q, 5.0)
    ops.sdpa_decode_paged(q, kp, vp, table, ints(lens), scale=1.0, out=out)
    assert ops.device_status() == (10, 1)
    for sequences in (1, 3):  # (nothing while the status is set, in either form)
        out.fill_(5.0)
        ops.sdpa_decode_paged(q[:sequences], kp, vp, table[:sequences], ints([1] * sequences), scale=1.0, out=out[:sequences], num_ctas=3 - sequences)
        assert bool((out == 5.0).all())
    ops.clear_device_status()


def test_decode_refusals():
    from arcaine_b200 import ops
    q, kp, vp, table, gate = paged_case([30, 20], 16, 8, 2, 128, None, 0, seed=8)
    lens = ints([30, 20])
    for kw, text in ((dict(gate=gate[:1]), "gate"), (dict(out=q[:, :4]), "out"), (dict(window=2**40), "window")):
        with pytest.raises(ValueError, match=text):
            ops.sdpa_decode_paged(q, kp, vp, table, lens, scale=1.0, **kw)
    with pytest.raises(ValueError, match="kv_len"):
        ops.sdpa_decode_paged(q, kp, vp, table, lens[:1], scale=1.0)
    with pytest.raises(ValueError, match="block_table"):
        ops.sdpa_decode_paged(q, kp, vp, table[:1], lens, scale=1.0)
    with pytest.raises(ValueError, match="v_pages"):
        ops.sdpa_decode_paged(q, kp, vp[..., :64], table, lens, scale=1.0)
    with pytest.raises(ValueError, match="same number"):
        ops.sdpa_decode_paged(q, kp, vp[:, :8], table, lens, scale=1.0)
    for kw in (dict(window=0), dict(sinks=-1), dict(scale=-1.0)):
        with pytest.raises(ops.ArcError):
            ops.sdpa_decode_paged(q, kp, vp, table, lens, **{"scale": 1.0, **kw})
    with pytest.raises(ops.ArcError):
        ops.sdpa_decode_paged(q, kp, vp, table, 10**6, scale=1.0)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
class Layer:
    """One layer's attention of a server with a paged cache, and the same kept whole in 64 bits."""

    def __init__(self, requests, page, nq, nkv, hd, window, sinks, interleaved, most, seed):
        from arcaine_b200 import ops
        self.page, self.nq, self.nkv, self.hd, self.window, self.sinks, self.interleaved = page, nq, nkv, hd, window, sinks, interleaved
        self.g = torch.Generator().manual_seed(seed)
        width = -(-most // page)
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(requests * width, generator=self.g).int().to(DEV)
        self.cursor = ints([0])
        self.kv_len = ints([0] * requests)
        self.kp, self.vp = (torch.full((requests * width, page, nkv, hd), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.inv, self.mscale = ops.rope_frequencies(hd // 2, 1e4, scaling="linear", factor=2.0, device=DEV)
        self.qw, self.kw = (torch.ones(hd).add_(0.1 * torch.randn(hd, generator=self.g)).bfloat16().to(DEV) for _ in range(2))
        self.keys, self.values = [[] for _ in range(requests)], [[] for _ in range(requests)]

    def rows(self, tokens):
        return [torch.randn(tokens, n, self.hd, generator=self.g).bfloat16().to(DEV) for n in (self.nq, self.nkv, self.nkv)]

    def tables(self, new, num_tokens):
        from arcaine_b200 import ops
        slots, positions, begin, self.kv_len, used = ops.paged_tables(new, self.kv_len, self.table, self.free, page_size=self.page, num_tokens=num_tokens,
                                                                      free_begin=self.cursor)
        self.cursor = self.cursor + used
        return slots, positions

    def prepare(self, q, k, v, slots, positions, **kw):
        from arcaine_b200 import ops
        ops.qkv_prepare_paged(q, k, v, positions, self.inv, k_pages=self.kp, v_pages=self.vp, slots=slots, q_weight=self.qw, k_weight=self.kw,
                              interleaved=self.interleaved, mscale=self.mscale, **kw)

    def keep(self, b, q, k, v, positions):
        """Rotated queries in 64 bits as they were rounded; keys and values join the request's."""
        q, _ = plain_rows(q, positions, self.inv, self.interleaved, True, self.qw, self.mscale)
        k, _ = plain_rows(k, positions, self.inv, self.interleaved, True, self.kw, self.mscale)
        self.keys[b].append(k)
        self.values[b].append(v.double())
        return q

    def attend(self, b, q, at):
        """One token at position `at` in 64 bits: result and sum p |v|."""
        k, v = torch.cat(self.keys[b])[:at + 1], torch.cat(self.values[b])[:at + 1]
        seen = visible(at + 1, self.window, self.sinks)
        k, v = k[seen].transpose(0, 1), v[seen].transpose(0, 1)
        p = torch.softmax(torch.matmul(q.view(self.nkv, -1, self.hd), k.transpose(1, 2)) * self.hd ** -0.5, -1)
        return torch.matmul(p, v).view(self.nq, self.hd), torch.matmul(p, v.abs()).view(self.nq, self.hd)


@pytest.mark.parametrize("page,nq,nkv,hd,window,sinks,interleaved", [(16, 8, 4, 128, 90, 5, False), (32, 24, 4, 256, None, 0, True), (48, 16, 8, 256, 130, 1, False)])
def test_prompts_then_tokens(page, nq, nkv, hd, window, sinks, interleaved):
    """Prompts of several requests, then tokens of some of them at a time: every layer call of a server.  Queries and keys are rounded to
    bf16 before the scores: 2^-8 of each factor, so a score is off by a few 2^-8 of sum |q k| / sqrt(hd), about 1, and the
    probabilities by as much; 0.05 of sum p |v| bounds it (|score error| < 0.025 on both sides of the softmax)."""
    from arcaine_b200 import ops
    layer = Layer(4, page, nq, nkv, hd, window, sinks, interleaved, 400, seed=hd + page)
    w = ops.NO_WINDOW if window is None else window
    prompts = [200, 0, 37, 129]
    slots, positions = layer.tables(ints(prompts), sum(prompts))
    q, k, v = layer.rows(sum(prompts))
    raw = q.clone(), k.clone(), v.clone()
    layer.prepare(q, k, v, slots, positions, k_out=k)
    begin = 0
    for b, n in enumerate(prompts):
        if n == 0:
            continue
        part = slice(begin, begin + n)
        begin += n
        out = ops.sdpa_prefill(q[part], k[part], v[part], scale=hd ** -0.5, mask_type=ops.MASK_CAUSAL, window=w, sinks=sinks)
        exact = layer.keep(b, *(t[part] for t in raw), positions[part])
        for at in (0, n // 2, n - 1):
            want, size = layer.attend(b, exact[at], at)
            assert bool(((out[at].double() - want).abs() <= 0.05 * size + want.abs() * 2.0 ** -8).all())
    lens = list(prompts)
    for step in range(40):
        new = [int(i != step % 4) for i in range(4)]
        slots, positions = layer.tables(ints(new), 4)  # room for four tokens; three come
        q, k, v = layer.rows(4)
        raw = q.clone(), k.clone(), v.clone()
        layer.prepare(q, k, v, slots, positions)
        assert torch.equal(q[3], raw[0][3])  # (the padding)
        owners = [b for b in range(4) if new[b]]
        queries = torch.zeros(4, nq, hd, dtype=torch.bfloat16, device=DEV)
        queries[owners] = q[:3]
        out = ops.sdpa_decode_paged(queries, layer.kp, layer.vp, layer.table, layer.kv_len, scale=hd ** -0.5, window=w, sinks=sinks)
        for i, b in enumerate(owners):
            exact = layer.keep(b, *(t[i:i + 1] for t in raw), positions[i:i + 1])
            lens[b] += 1
            want, size = layer.attend(b, exact[0], lens[b] - 1)
            assert bool(((out[b].double() - want).abs() <= 0.05 * size + want.abs() * 2.0 ** -8).all())
    assert layer.kv_len.tolist() == lens and ops.device_status() == (0, 0)


def test_a_step_from_a_captured_graph():
    """Tables, append and decode in one graph, replayed while lengths, pages and rows change; two such graphs side by side."""
    from arcaine_b200 import ops
    page, nq, nkv, hd, batch = 16, 8, 4, 128, 3

    def build(seed):
        layer = Layer(batch, page, nq, nkv, hd, 40, 4, False, 200, seed)
        state = dict(new=ints([1] * batch), past=ints([0] * batch), rows=layer.rows(batch))
        state["work"] = [t.clone() for t in state["rows"]]

        def step():
            slots, positions, _, kv_len, used = ops.paged_tables(state["new"], state["past"], layer.table, layer.free, page_size=page, num_tokens=batch,
                                                                 free_begin=layer.cursor)
            for w, r in zip(state["work"], state["rows"]):
                w.copy_(r)
            layer.prepare(*state["work"], slots, positions)
            out = ops.sdpa_decode_paged(state["work"][0], layer.kp, layer.vp, layer.table, kv_len, scale=hd ** -0.5, window=40, sinks=4)
            state["past"].copy_(kv_len)
            layer.cursor.add_(used)
            return out

        return layer, state, step

    results = []
    for graphed in (False, True):
        sides = [build(1), build(2)]
        graphs, outs = [], []
        if graphed:
            for layer, state, step in sides:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                saved = [t.clone() for t in (layer.table, layer.cursor, state["past"], layer.kp, layer.vp)]
                with torch.cuda.stream(side):
                    step()
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    outs.append(step())
                for t, s in zip((layer.table, layer.cursor, state["past"], layer.kp, layer.vp), saved):
                    t.copy_(s)
                graphs.append(graph)
            streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = []
        g = torch.Generator().manual_seed(9)
        for i in range(50):
            for n, (layer, state, step) in enumerate(sides):
                for r in state["rows"]:
                    r.copy_(torch.randn(r.shape, generator=g).bfloat16())
                state["new"].copy_(ints([1, int(i % 2 == 0), int(i % 3 != n)]))
            torch.cuda.synchronize()
            if graphed:
                for graph, stream in zip(graphs, streams):
                    with torch.cuda.stream(stream):
                        graph.replay()
                torch.cuda.synchronize()
                got.append([o.clone() for o in outs])
            else:
                got.append([step().clone() for _, _, step in sides])
        results.append(got)
    assert ops.device_status() == (0, 0)
    for plain, replayed in zip(*results):
        for a, b in zip(plain, replayed):
            assert torch.equal(a, b)


def test_calls_on_two_streams_and_off_the_current_one():
    from arcaine_b200 import ops
    cases = [paged_case([900, 40, 3000], 32, 24, 4, 256, None, 0, seed=s) for s in (1, 2)]
    lens = ints([900, 40, 3000])
    want = [ops.sdpa_decode_paged(q, kp, vp, table, lens, scale=0.06, gate=gate) for q, kp, vp, table, gate in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (q, kp, vp, table, gate) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.sdpa_decode_paged(q, kp, vp, table, lens, scale=0.06, gate=gate))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)
    assert ops.device_status() == (0, 0)
