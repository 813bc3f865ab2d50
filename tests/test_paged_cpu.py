"""The paged cache and prefill sinks without a GPU: layouts of the parameter structs, statuses decided before any CUDA call,
arguments the binding refuses, rotation frequencies."""
import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def mirrors():
    from arcaine_b200 import _lib
    return [("arc_paged_tables_params", _lib.PagedTablesParams), ("arc_qkv_prepare_paged_params", _lib.QkvPreparePagedParams),
            ("arc_sdpa_decode_paged_params", _lib.DecodePagedParams), ("arc_sdpa_prefill_params", _lib.PrefillParams)]


def test_struct_mirrors_have_the_layout_the_header_declares(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "arc_sdpa.h")).read(), flags=re.S)
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "arc_sdpa.h"', 'int main(void) {']
    for cname, mirror in mirrors():
        body = re.search(r"typedef struct " + cname + r" \{(.*?)\} " + cname + ";", text, flags=re.S).group(1)
        names = [n.split()[-1] for decl in body.split(";") if decl.strip() for n in decl.replace("*", " ").split(",")]
        assert names == [f[0] for f in mirror._fields_], cname
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in mirror._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ['  return 0;', '}']))
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    seen = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for cname, mirror in mirrors():
        assert int(seen[cname]) == ctypes.sizeof(mirror)
        for f, _ in mirror._fields_:
            assert int(seen[f"{cname}.{f}"]) == getattr(mirror, f).offset, f"{cname}.{f}"


class Memory:
    """Host addresses that pass alignment checks; nothing reads them."""

    def __init__(self):
        self.buf = (ctypes.c_uint8 * 65536)()
        self.base = ctypes.addressof(self.buf) + (-ctypes.addressof(self.buf)) % 64


def test_tables_refusals():
    from arcaine_b200 import _lib
    lib, m = _lib.load(), Memory()

    def call(**kw):
        p = _lib.PagedTablesParams(batch=4, num_tokens=9, page_size=16, table_width=8, free_count=3, table_stride=8)
        for i, f in enumerate(("new_len", "past_len", "block_table", "free_pages", "free_begin", "slots", "positions", "token_begin", "kv_len", "pages_used")):
            setattr(p, f, m.base + 256 * i)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.arc_paged_tables(ctypes.byref(p), None)

    assert lib.arc_paged_tables(None, None) == _lib.ARC_ERR_NULL_POINTER
    for kw in (dict(batch=0), dict(num_tokens=-1), dict(table_width=0), dict(table_stride=7), dict(page_size=0), dict(page_size=8), dict(page_size=24),
               dict(free_count=-1)):
        assert call(**kw) == _lib.ARC_ERR_BAD_SHAPE, kw
    assert call(batch=2049) == _lib.ARC_ERR_TOO_LARGE
    assert call(num_tokens=2**30 + 1) == call(num_tokens=2**31 - 1) == _lib.ARC_ERR_TOO_LARGE
    for f in ("new_len", "block_table", "free_pages", "slots", "positions", "token_begin", "kv_len", "pages_used"):
        assert call(**{f: None}) == _lib.ARC_ERR_NULL_POINTER, f
    assert call(kv_len=m.base + 2) == _lib.ARC_ERR_ALIGNMENT


def test_prepare_refusals():
    from arcaine_b200 import _lib
    lib, m = _lib.load(), Memory()

    def call(**kw):
        p = _lib.QkvPreparePagedParams(tokens=2, nq=2, nkv=1, hd=128, page_size=16, num_pages=4, rotary_dim=128, norm_qk=1, q_stride=256, k_stride=128,
                                       v_stride=128, q_out_stride=256, k_out_stride=128, v_out_stride=128, k_stride_page=2048, k_stride_t=128,
                                       v_stride_page=2048, v_stride_t=128, eps=1e-6, mscale=1.0)
        for f in ("q", "k", "v", "q_out", "k_pages", "v_pages", "slots", "positions", "inv_freq"):
            setattr(p, f, m.base)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.arc_qkv_prepare_paged(ctypes.byref(p), None)

    assert lib.arc_qkv_prepare_paged(None, None) == _lib.ARC_ERR_NULL_POINTER
    assert call(hd=64) == _lib.ARC_ERR_UNSUPPORTED_HEAD_DIM
    for kw in (dict(tokens=-1), dict(rotary_dim=24), dict(rotary_dim=144), dict(rotary_dim=-16), dict(eps=float("nan")), dict(eps=-1.0),
               dict(mscale=float("inf")), dict(page_size=8), dict(page_size=20), dict(num_pages=0), dict(q_stride=128), dict(q_out_stride=128),
               dict(k_stride_t=64), dict(k_stride_page=1024), dict(v_stride_page=1024), dict(nq=0), dict(nkv=0)):
        assert call(**kw) == _lib.ARC_ERR_BAD_SHAPE, kw
    for kw in (dict(positions=None), dict(slots=None), dict(inv_freq=None), dict(q_out=None), dict(k=None), dict(k_pages=None, v_pages=None),
               dict(q=None, k=None, v=None)):
        assert call(**kw) == _lib.ARC_ERR_NULL_POINTER, kw
    for kw in (dict(q=m.base + 8), dict(k_pages=m.base + 2), dict(inv_freq=m.base + 4), dict(slots=m.base + 1), dict(q_stride=260), dict(k_stride=-128),
               dict(v_stride_page=2052)):
        assert call(**kw) == _lib.ARC_ERR_ALIGNMENT, kw
    assert call(num_pages=1 << 27, page_size=16) == _lib.ARC_ERR_TOO_LARGE
    assert call(tokens=0) == _lib.ARC_OK


def test_prepare_of_no_tokens_needs_no_addresses():
    """A step without tokens: empty tensors have no address."""
    from arcaine_b200 import _lib
    p = _lib.QkvPreparePagedParams(tokens=0, nq=2, nkv=1, hd=128, page_size=16, num_pages=4, rotary_dim=128, norm_qk=1, eps=1e-6, mscale=1.0)
    assert _lib.load().arc_qkv_prepare_paged(ctypes.byref(p), None) == _lib.ARC_OK
    p.rotary_dim = 24
    assert _lib.load().arc_qkv_prepare_paged(ctypes.byref(p), None) == _lib.ARC_ERR_BAD_SHAPE


def test_decode_refusals():
    from arcaine_b200 import _lib
    lib, m = _lib.load(), Memory()

    def call(**kw):
        p = _lib.DecodePagedParams(batch=2, nq=4, nkv=2, hd=128, page_size=16, num_pages=4, table_width=3, window=_lib.NO_WINDOW, q_stride_b=512,
                                   o_stride_b=512, table_stride=3, k_stride_page=4096, k_stride_t=256, v_stride_page=4096, v_stride_t=256, scale=1.0)
        for f in ("q", "k_pages", "v_pages", "out", "block_table", "kv_len"):
            setattr(p, f, m.base)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.arc_sdpa_decode_paged(ctypes.byref(p), None)

    assert lib.arc_sdpa_decode_paged(None, None) == _lib.ARC_ERR_NULL_POINTER
    for kw in (dict(q=None), dict(k_pages=None), dict(v_pages=None), dict(block_table=None), dict(out=None), dict(out=None, out_f32=m.base, gate=m.base)):
        assert call(**kw) == _lib.ARC_ERR_NULL_POINTER, kw
    for kw in (dict(batch=0), dict(nq=3), dict(nkv=0), dict(table_width=0), dict(table_stride=2), dict(scale=0.0), dict(scale=float("nan")), dict(window=0),
               dict(window=-5), dict(sinks=-1), dict(page_size=12), dict(page_size=0), dict(num_pages=0), dict(kv_len=None, kv_len_uniform=-1),
               dict(kv_len=None, kv_len_uniform=49), dict(q_stride_b=256), dict(o_stride_b=256), dict(k_stride_t=128), dict(v_stride_page=2048),
               dict(num_ctas=-1)):
        assert call(**kw) == _lib.ARC_ERR_BAD_SHAPE, kw
    assert call(hd=64) == _lib.ARC_ERR_UNSUPPORTED_HEAD_DIM
    assert call(nq=34) == _lib.ARC_ERR_UNSUPPORTED_GQA
    assert call(batch=2049) == _lib.ARC_ERR_TOO_LARGE
    assert call(num_pages=1 << 28) == _lib.ARC_ERR_TOO_LARGE
    for kw in (dict(q=m.base + 8), dict(gate=m.base + 2), dict(block_table=m.base + 2), dict(k_stride_t=260), dict(v_stride_page=-4096), dict(q_stride_b=516)):
        assert call(**kw) == _lib.ARC_ERR_ALIGNMENT, kw


def test_cpu_tensors_are_refused():
    from arcaine_b200 import ops
    i, x = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.paged_tables(i, None, i.view(4, 1), i, page_size=16, num_tokens=4)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.qkv_prepare_paged(x, None, None, i, None)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.sdpa_decode_paged(x, x, x, i.view(4, 1), 3, scale=1.0)


def test_rope_frequencies():
    from arcaine_b200 import ops
    inv, m = ops.rope_frequencies(64, 1e4, device="cpu")
    assert m == 1.0 and inv.dtype == torch.float64 and inv.shape == (32,)
    assert torch.allclose(inv, torch.tensor([1e4 ** (-f / 32) for f in range(32)], dtype=torch.float64), rtol=1e-15)
    lin, m = ops.rope_frequencies(64, 1e4, scaling="linear", factor=4.0, device="cpu")
    assert m == 1.0 and torch.allclose(lin, inv / 4, rtol=1e-15)
    ntk, m = ops.rope_frequencies(64, 1e4, scaling="ntk", factor=4.0, device="cpu")
    assert m == 1.0 and ntk[0] == 1.0 and math.isclose(ntk[-1], inv[-1] / 4, rel_tol=1e-12)
    yarn, m = ops.rope_frequencies(64, 1e4, scaling="yarn", factor=4.0, original_len=4096, device="cpu")
    assert math.isclose(m, 0.1 * math.log(4.0) + 1.0)
    turns = 4096 * inv / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], inv[turns >= 32]) and torch.allclose(yarn[turns <= 1], inv[turns <= 1] / 4, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and bool(((yarn < inv) & (yarn > inv / 4))[between].all())
    one, m = ops.rope_frequencies(64, 1e4, scaling="yarn", factor=1.0, original_len=4096, device="cpu")
    assert m == 1.0 and torch.allclose(one, inv, rtol=1e-15)
    for kw in (dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=64, theta=0.0), dict(rotary_dim=64, scaling="other"),
               dict(rotary_dim=64, scaling="linear", factor=0.5), dict(rotary_dim=64, scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**kw, device="cpu")


@pytest.mark.parametrize("theta,length,factor,low,high", [(1e6, 32768, 4.0, 23, 40), (1e4, 4096, 8.0, 20, 46), (1e6, 8192, 8.0, 17, 34)])
def test_yarn_ramp_goes_by_the_index_of_the_pair(theta, length, factor, low, high):
    """Of 64 pairs: up to `low` as they are, from `high` on divided, linear in the index between them.  low and high are worked out by hand:
    pair f turns length theta^(-f / 64) / (2 pi) times, so that the ends are the last whole f with 32 turns or more and the first with
    one or less."""
    from arcaine_b200 import ops
    turns = [length * theta ** (-f / 64) / (2 * math.pi) for f in range(64)]
    assert turns[low] >= 32 > turns[low + 1] and turns[high] <= 1 < turns[high - 1]
    inv = ops.rope_frequencies(128, theta, device="cpu")[0]
    got, m = ops.rope_frequencies(128, theta, scaling="yarn", factor=factor, original_len=length, device="cpu")
    assert math.isclose(m, 0.1 * math.log(factor) + 1.0)
    for f in range(64):
        share = min(1.0, max(0.0, (f - low) / (high - low)))  # of the divided frequency
        assert math.isclose(got[f].item(), inv[f].item() * (1.0 - share + share / factor), rel_tol=1e-12), f


def test_yarn_ends_outside_the_pairs():
    from arcaine_b200 import ops
    inv = ops.rope_frequencies(32, 1e4, device="cpu")[0]
    # the fastest pair turns 16 times: the ramp begins with it; the slowest 10^5 times: all are left
    got = ops.rope_frequencies(32, 1e4, scaling="yarn", factor=4.0, original_len=101, device="cpu")[0]
    assert got[0] == inv[0] and bool((got[1:] < inv[1:]).all())
    assert torch.equal(ops.rope_frequencies(32, 1e4, scaling="yarn", factor=4.0, original_len=2**31 - 1, beta_fast=64.0, beta_slow=32.0, device="cpu")[0], inv)
    for kw in (dict(theta=1.0), dict(theta=0.5), dict(beta_slow=0.0), dict(beta_slow=-1.0), dict(beta_fast=1.0), dict(beta_slow=math.nan)):
        with pytest.raises(ValueError, match="yarn needs"):
            ops.rope_frequencies(64, **{"theta": 1e4, **kw}, scaling="yarn", factor=2.0, original_len=4096, device="cpu")
