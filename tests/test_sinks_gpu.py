"""Prefill behind a window with the first tokens visible, against the definition in 64 bits.

Tolerance: bf16 roundings of the probabilities (2^-8 of sum p |v|) and of the result (2^-8 of it), and 2^-9 of sum p |v| for the fp32 sums, scores and
rescales in between."""
import math
import os
import subprocess
import sys

import pytest
import torch

from helpers import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def inputs(batch, seq, kv, nq, nkv, hd, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(batch, n, h, hd, generator=g, device=DEV).bfloat16() for n, h in ((seq, nq), (kv, nkv), (kv, nkv), (seq, nq))]


def plain(q, k, v, window, sinks, scale, gate=None):
    batch, seq, nq, hd = q.shape
    kv, nkv = k.shape[1:3]
    at = torch.arange(kv - seq, kv, device=DEV)[:, None]
    key = torch.arange(kv, device=DEV)[None]
    hidden = (key > at) | ((key <= at - window) & (key >= sinks))
    out, size = (torch.empty(batch, seq, nq, hd, dtype=torch.float64, device=DEV) for _ in range(2))
    lse = torch.empty(batch, seq, nq, dtype=torch.float64, device=DEV)
    for b in range(batch):
        for h in range(nq):
            kk, vv = k[b, :, h // (nq // nkv)].double(), v[b, :, h // (nq // nkv)].double()
            s = (q[b, :, h].double() @ kk.T * scale).masked_fill(hidden, -math.inf)
            lse[b, :, h] = torch.logsumexp(s, -1)
            p = torch.where(torch.isinf(lse[b, :, h])[:, None], 0.0, torch.softmax(s, -1))
            out[b, :, h], size[b, :, h] = p @ vv, p @ vv.abs()
    if gate is not None:
        out, size = out * torch.sigmoid(gate.double()), size * torch.sigmoid(gate.double())
    return out, lse, size


def check(got, lse, want, want_lse, size):
    off = (got.double() - want).abs()
    room = size * (2.0 ** -8 + 2.0 ** -9) + want.abs() * 2.0 ** -8 + 1e-30
    assert bool(torch.isfinite(got).all())
    assert bool((off <= room).all()), f"off by {(off / room).max().item():.2f} of the tolerance"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty)
    assert bool(((lse.double() - want_lse).abs()[~empty] <= 2e-4 + 2.0 ** -20 * want_lse.abs()[~empty]).all())


CASES = [  # batch, seq, kv, nq, nkv, hd, window, sinks, splits
    (1, 1, 1, 4, 2, 128, 1, 1, 0), (1, 1, 700, 4, 2, 128, 100, 4, 0), (1, 129, 129, 4, 4, 128, 1, 1, 0), (2, 300, 300, 8, 4, 128, 64, 4, 0),
    (1, 500, 1300, 7, 7, 128, 200, 130, 0), (1, 513, 513, 4, 1, 128, 128, 128, 0), (1, 400, 2000, 2, 2, 128, 300, 700, 0), (1, 700, 700, 3, 1, 128, 90, 5, 0),
    (2, 1024, 1024, 32, 16, 128, 300, 4, 0), (1, 2100, 2100, 28, 4, 128, 513, 260, 0), (1, 3000, 3300, 9, 9, 128, 400, 3, 0),  # (two tiles a CTA)
    (1, 300, 5000, 4, 2, 128, 1500, 200, 0), (1, 64, 4000, 4, 2, 128, 700, 100, 3), (1, 200, 150, 4, 2, 128, 30, 5, 0),
    (1, 1, 1, 4, 2, 256, 1, 1, 0), (1, 33, 900, 8, 4, 256, 50, 4, 0), (2, 300, 300, 16, 8, 256, 64, 4, 0), (1, 260, 700, 5, 5, 256, 150, 20, 0),
    (1, 128, 3000, 8, 8, 256, 1000, 140, 0), (1, 128, 3000, 8, 8, 256, 1000, 140, 2), (1, 100, 3000, 4, 2, 256, 900, 300, 3), (1, 100, 3000, 4, 2, 256, 900, 300, 4),
    (1, 100, 3000, 4, 2, 256, 900, 300, 6), (1, 2000, 2500, 24, 4, 256, 512, 64, 0), (4, 900, 900, 16, 8, 256, 256, 8, 0), (1, 2600, 2600, 9, 3, 256, 100, 600, 0),
    (1, 200, 150, 4, 2, 256, 30, 5, 0), (1, 384, 384, 8, 4, 256, 1, 2, 0),
    (1, 500, 900, 8, 4, 128, 100, 2**31 - 1, 0), (1, 2100, 2100, 28, 4, 128, 300, 2**31 - 1, 0), (1, 500, 900, 8, 4, 256, 100, 2**31 - 1, 0),
    (2, 1499, 1499, 28, 4, 128, 490, 64, 0), (1, 300, 900, 8, 4, 256, 200, 65, 0), (1, 300, 900, 8, 4, 256, 200, 63, 0), (1, 700, 1500, 9, 3, 256, 128, 1, 0)]


@pytest.mark.parametrize("batch,seq,kv,nq,nkv,hd,window,sinks,splits", CASES)
def test_sinks(batch, seq, kv, nq, nkv, hd, window, sinks, splits):
    one_call(batch, seq, kv, nq, nkv, hd, window, sinks, splits)


def one_call(batch, seq, kv, nq, nkv, hd, window, sinks, splits):
    from arcaine_b200 import ops
    ops.clear_device_status()
    q, k, v, gate = inputs(batch, seq, kv, nq, nkv, hd, seed=seq + kv)
    kw = dict(scale=hd ** -0.5, mask_type=ops.MASK_CAUSAL, window=window, sinks=sinks, num_splits=splits, return_lse=True)
    out, lse = ops.sdpa_prefill(q, k, v, **kw)
    assert ops.device_status() == (0, 0)
    want, want_lse, size = plain(q, k, v, window, sinks, hd ** -0.5)
    check(out, lse, want, want_lse, size)
    again, _ = ops.sdpa_prefill(q, k, v, **kw)
    assert torch.equal(out, again)
    gated, lse = ops.sdpa_prefill(q, k, v, gate=gate, **kw)
    assert ops.device_status() == (0, 0)
    check(gated, lse, want * torch.sigmoid(gate.double()), want_lse, size * torch.sigmoid(gate.double()))


@pytest.mark.parametrize("hd", [128, 256])
def test_sinks_that_change_nothing(hd):
    """Behind no window, or one that hides nothing, sinks change no key.  Head dim 128: bit for bit.  At 256 the parts of a call are weighted by
    log-sum-exps that leave out the rounding of the largest probability, up to 2^-8 of a part's sum, which those of calls
    without sinks keep in: both are held to the definition."""
    from arcaine_b200 import ops
    q, k, v, gate = inputs(1, 300, 500, 8, 4, hd, seed=3)
    causal = dict(scale=0.08, mask_type=ops.MASK_CAUSAL)
    want = ops.sdpa_prefill(q, k, v, **causal)
    exact, want_lse, size = plain(q, k, v, 500, 0, 0.08, gate)
    for window in (ops.NO_WINDOW, 500, 10**6):
        got, lse = ops.sdpa_prefill(q, k, v, window=window, sinks=7, return_lse=True, **causal)
        if hd == 128:
            assert torch.equal(got, want)
        check(got, lse, *plain(q, k, v, 500, 0, 0.08))
        got, lse = ops.sdpa_prefill(q, k, v, window=window, sinks=7, gate=gate, return_lse=True, **causal)
        check(got, lse, exact, want_lse, size)
    assert torch.equal(ops.sdpa_prefill(q, k, v, window=90, sinks=0, gate=gate, **causal), ops.sdpa_prefill(q, k, v, window=90, gate=gate, **causal))


@pytest.mark.parametrize("hd,seq", [(128, 400), (128, 2500), (256, 400), (256, 1800)])
def test_sinks_strides_copies_and_aliases(hd, seq):
    """Rows of a fused projection, output over the queries, and copies of the output."""
    from arcaine_b200 import ops
    nq, nkv, window, sinks = 16, 8, 200, 6
    g = torch.Generator(device=DEV).manual_seed(1)
    fused = torch.randn(1, seq, (nq + 2 * nkv) * hd, generator=g, device=DEV).bfloat16()
    q = fused[..., :nq * hd].unflatten(-1, (nq, hd))
    k = fused[..., nq * hd:(nq + nkv) * hd].unflatten(-1, (nkv, hd))
    v = fused[..., (nq + nkv) * hd:].unflatten(-1, (nkv, hd))
    kw = dict(scale=hd ** -0.5, mask_type=ops.MASK_CAUSAL, window=window, sinks=sinks)
    copy = torch.zeros(1, seq, nq, hd, dtype=torch.bfloat16, device=DEV)
    addresses = torch.tensor([copy.data_ptr()], dtype=torch.int64, device=DEV)
    out, lse = ops.sdpa_prefill(q, k, v, out_copies=addresses, return_lse=True, **kw)
    want, want_lse, size = plain(q, k, v, window, sinks, hd ** -0.5)
    check(out, lse, want, want_lse, size)
    assert torch.equal(copy, out)
    ops.sdpa_prefill(q, k, v, out=q, **kw)
    assert torch.equal(q, out) and ops.device_status() == (0, 0)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("seq,kv,nq,nkv", [(1, 130, 8, 4), (33, 33, 16, 1), (130, 400, 7, 7), (1100, 1100, 16, 8), (2300, 2300, 28, 4)])
def test_sinks_gated_rows_of_a_wider_tensor(seq, kv, nq, nkv, hd):
    """The gate and the output are parts of wider rows, and copies of the output go elsewhere; what lies beside them is left alone."""
    from arcaine_b200 import ops
    ops.clear_device_status()
    q, k, v, _ = inputs(2, seq, kv, nq, nkv, hd, seed=seq)
    g = torch.Generator(device=DEV).manual_seed(9)
    rows = 4 * torch.randn(2, seq, nq * hd + 16, generator=g, device=DEV).bfloat16()
    wide, copy = torch.full_like(rows, 7.0), torch.full_like(rows, 5.0)
    gate, out = (t[..., 8:8 + nq * hd].unflatten(-1, (nq, hd)) for t in (rows, wide))
    addresses = torch.tensor([copy.data_ptr() + 16], dtype=torch.int64, device=DEV)  # (laid out like the output)
    got, lse = ops.sdpa_prefill(q, k, v, scale=hd ** -0.5, mask_type=ops.MASK_CAUSAL, window=200, sinks=6, gate=gate, out=out, out_copies=addresses, return_lse=True)
    assert ops.device_status() == (0, 0)
    want, want_lse, size = plain(q, k, v, 200, 6, hd ** -0.5)
    weight = torch.sigmoid(gate.double())
    check(got, lse, want * weight, want_lse, size * weight)
    assert bool((wide[..., :8] == 7.0).all()) and bool((wide[..., 8 + nq * hd:] == 7.0).all())
    assert torch.equal(copy[..., 8:8 + nq * hd], wide[..., 8:8 + nq * hd])
    assert bool((copy[..., :8] == 5.0).all()) and bool((copy[..., 8 + nq * hd:] == 5.0).all())


FORCED = r"""
import sys
sys.path.insert(0, sys.argv[1] + '/tests')
import test_sinks_gpu as t
from helpers import ROOT
for group in ((4, 2), (3, 1), (5, 5), (8, 1)):  # two heads of a group on one tile of tokens, or two tiles of one head
    for seq, kv in ((1, 300), (129, 129), (500, 500), (300, 800), (700, 650), (1300, 1300)):
        for window, sinks in ((1, 1), (30, 4), (128, 128), (129, 200), (250, 64), (300, 600), (490, 7), (513, 260)):
            t.one_call(1, seq, kv, *group, 128, window, sinks, 1)
"""


@pytest.mark.parametrize("kernel", ["pair", "single"])
def test_both_kernels_of_head_dim_128(kernel):
    """The library chooses between them by size; here each takes all calls, in a process of its own (the choice is read once)."""
    env = dict(os.environ, ARC_SDPA_PREFILL_KERNEL=kernel, PYTHONPATH=ROOT)
    done = subprocess.run([sys.executable, "-c", FORCED, ROOT], env=env, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]


def test_sinks_refusals():
    from arcaine_b200 import ops
    q, k, v, _ = inputs(1, 64, 64, 4, 2, 128, seed=2)
    ids = torch.full((64,), -1, dtype=torch.int32, device=DEV)
    with pytest.raises(ops.ArcError):
        ops.sdpa_prefill(q, k, v, scale=1.0, sinks=4)
    with pytest.raises(ops.ArcError):
        ops.sdpa_prefill(q, k, v, scale=1.0, mask_type=ops.MASK_CAUSAL, window=8, sinks=-1)
    with pytest.raises(ops.ArcError):
        ops.sdpa_prefill(q, k, v, scale=1.0, mask_type=ops.MASK_CAUSAL, window=8, sinks=4, block_ids=ids)
    with pytest.raises(ValueError, match="sinks"):
        ops.sdpa_prefill(q, k, v, scale=1.0, mask_type=ops.MASK_CAUSAL, window=8, sinks=2**35)
