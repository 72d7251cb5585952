"""Codebook attributes: codebook_lookup, code_log_probs and code_balance_loss
against 64-bit restatements (oracle/torch_ref.py), forward and backward, at the
sizes, types, strides and masks where they can go wrong; their refusals (CPU); and
a run of them together in front of the rasterizer.

Tolerances. u = 2^-24 is half a step of fp32, eps(t)/2 of a result's type t. A sum
of n products in fp32 is off by at most (n + 1) u times the sum of their
magnitudes. exp(x) as ex2(x log2 e) is off by u|x| for x, as much for the product,
and 2^-22 for the function, relatively: REL_EXP below, for |x| <= 64 (smaller
values do not count next to the 1 of the largest logit, and a row of one logit has
no others).
"""
from __future__ import annotations

import ctypes
import itertools
import math
import multiprocessing
import re
import time
from multiprocessing.shared_memory import SharedMemory
from pathlib import Path

import pytest
import torch

import torch_gsplat_bridge_fast as tgb
from oracle import torch_ref as TR
from torch_gsplat_bridge_fast import _native as N
from torch_gsplat_bridge_fast.rasterize import _host, _ops

U = 2.0**-24
REL_EXP = 128 * U + 4 * U
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = math.inf
DEV = "cuda:0"


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half a step of the smallest numbers of a type (fp16 results may be subnormal)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _close(got, ref, tol, dtype):
    """|got - ref| <= tol + the rounding to dtype; the same non-finite values."""
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine)
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)])
    tol = torch.as_tensor(tol, dtype=torch.float64, device=ref.device).expand(ref.shape)
    bound = tol + _half_step(dtype) * (ref.abs() + tol) + _tiny(dtype)
    over = ((got - ref).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"over by {over.max().item()} (|ref| <= {ref[fine].abs().max().item()})"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ---- refusals ------------------------------------------------------------------
def _z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call, match", [
    (lambda: tgb.codebook_lookup(_z(0, 3), _z(2, dtype=torch.int32)), "at least one row"),
    (lambda: tgb.codebook_lookup(_z(4, 0), _z(2, dtype=torch.int32)), "at least one row"),
    (lambda: tgb.codebook_lookup(_z(4, 3), _z(2)), "int32 or int64"),
    (lambda: tgb.codebook_lookup(_z(4, 3, dtype=torch.float64), _z(2, dtype=torch.int32)), "float32, bfloat16"),
    (lambda: tgb.codebook_lookup(_z(4, 3), _z(2, dtype=torch.int32), _z(2, 1)), "weights must have"),
    (lambda: tgb.codebook_lookup(_z(4, 3), _z(2, 0, dtype=torch.int32), _z(2, 0)), "weights must have"),
    (lambda: tgb.codebook_lookup(_z(4, 3), _z(2, 1, dtype=torch.int32), _z(2, 1, dtype=torch.float16)), "float32"),
    (lambda: tgb.codebook_lookup(_z(4, 3), _z(2, dtype=torch.int32), out_dtype=torch.float64), "out_dtype"),
    (lambda: tgb.codebook_lookup(_z(4, 3), _z(2, dtype=torch.int32)), "CUDA device"),
    (lambda: tgb.code_log_probs(_z(4, 0)), "at least one code"),
    (lambda: tgb.code_log_probs(_z(4, 3), _z(3, dtype=torch.int32)), "codes must have the shape"),
    (lambda: tgb.code_log_probs(_z(4, 3), top_k=4), "top_k"),
    (lambda: tgb.code_log_probs(_z(4, 64), top_k=33), "top_k"),
    (lambda: tgb.code_log_probs(_z(4, 64), top_k=-1), "top_k"),
    (lambda: tgb.code_log_probs(_z(4, 3, dtype=torch.float64)), "float32, bfloat16"),
    (lambda: tgb.code_log_probs(_z(4, 3)), "CUDA device"),
    (lambda: tgb.code_balance_loss(_z(4, 3), _z(3, dtype=torch.int32)), "codes must have the shape"),
    (lambda: tgb.code_balance_loss(_z(4, 3), _z(4, 0, dtype=torch.int32)), "codes must have the shape"),
    (lambda: tgb.code_balance_loss(_z(4, 3), _z(4, 1)), "int32 or int64"),
    (lambda: tgb.code_balance_loss(_z(4, 3), _z(4, 1, dtype=torch.int64)), "CUDA device"),
    (lambda: tgb.spherical_harmonics_colors(_z(4, 9, 3), _z(5, 3), codes=_z(4, dtype=torch.int32)), "codes must have"),
    (lambda: tgb.spherical_harmonics_colors(_z(4, 9, 3), _z(4, 3), code_weights=_z(4, 1)), "need codes"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_c_entries_refuse_before_any_launch():
    L = N.load()
    one = 256  # a pointer that is never followed: each call is refused first
    fwd = lambda td=0, od=0, rows=4, bag=1, c=8, dim=3, table=one, stride=3, codes=one, cb=4, out=one, st=one: \
        L.gsb_codebook_forward(td, od, rows, bag, c, dim, table, stride, codes, cb, None, 1.0, out, st, None)
    assert fwd(td=3) == 2 and fwd(od=-1) == 2 and fwd(od=1) == 2 and fwd(td=1, od=2) == 2
    for bad in (dict(rows=-1), dict(bag=0), dict(c=0), dict(dim=0), dict(cb=2), dict(table=None), dict(codes=None),
                dict(out=None), dict(st=None), dict(stride=-1)):
        assert fwd(**bad) == 1, bad
    assert fwd(rows=1 << 30) == 4 and fwd(rows=1 << 20, bag=1 << 11) == 4 and fwd(c=(1 << 31) - 1) == 4
    assert fwd(rows=0, table=None, codes=None, out=None) == 0
    assert L.gsb_codebook_backward_workspace_size(1 << 30, 1, 8, 3) == 0
    assert L.gsb_codebook_backward_workspace_size(1000, 2, 8, 3) > 2000 * 16
    bwd = lambda table=one, g=one, gt=one, gw=None, ws=one, n=0: \
        L.gsb_codebook_backward(0, 0, 4, 1, 8, 3, table, 3, one, 4, None, 1.0, g, gt, gw, one, ws, n, None)
    assert bwd() == 3 and bwd(ws=None, n=1 << 20) == 3 and bwd(g=None, n=1 << 20) == 1
    assert bwd(table=None, gw=one, n=1 << 20) == 1
    lp = lambda dt=0, rows=4, c=8, z=one, stride=8, codes=one, cb=4, k=2, lp=one, ent=one, tl=one, tc=one, st=one: \
        L.gsb_code_log_probs_forward(dt, rows, c, z, stride, codes, cb, k, lp, ent, tl, tc, None, st, None, 0, None)
    assert L.gsb_code_log_probs_workspace_size(1000, 512, 4) == 0
    assert L.gsb_code_log_probs_workspace_size(3, 100000, 4) > 0 and lp(c=100000) == 3
    assert lp(dt=7) == 2 and lp(rows=1 << 31) == 4 and lp(rows=0, z=None) == 0
    for bad in (dict(c=0), dict(cb=1), dict(k=9), dict(k=-1), dict(k=33, c=64), dict(z=None), dict(codes=None),
                dict(lp=None), dict(ent=None), dict(tl=None), dict(tc=None), dict(st=None), dict(rows=-1)):
        assert lp(**bad) == 1, bad
    lb = lambda z=one, codes=one, tc=one, st=one, dz=one, gl=one, gt=one: \
        L.gsb_code_log_probs_backward(0, 4, 8, z, 8, codes, 4, 2, tc, st, gl, None, gt, dz, None)
    for bad in (dict(z=None), dict(codes=None), dict(tc=None), dict(st=None), dict(dz=None)):
        assert lb(**bad) == 1, bad
    n = L.gsb_code_balance_workspace_size(4, 8)
    assert n > 0 and L.gsb_code_balance_workspace_size(-1, 8) == 0
    assert L.gsb_code_balance_state_floats(8) >= 8 and L.gsb_code_balance_state_floats(0) == 0
    bl = lambda rows=4, bag=1, z=one, codes=one, loss=one, cnt=one, state=one, st=one, ws=one, n=n: \
        L.gsb_code_balance_forward(0, rows, 8, bag, z, 8, codes, 4, loss, cnt, None, state, st, ws, n, None)
    for bad in (dict(bag=0), dict(z=None), dict(codes=None), dict(loss=None), dict(cnt=None), dict(state=None),
                dict(st=None)):
        assert bl(**bad) == 1, bad
    assert bl(ws=None) == 3 and bl(n=n - 1) == 3 and bl(rows=1 << 30, bag=2) == 4
    bb = lambda z=one, st=one, state=one, g=one, dz=one: \
        L.gsb_code_balance_backward(0, 4, 8, z, 8, st, state, g, dz, None)
    for bad in (dict(z=None), dict(st=None), dict(state=None), dict(g=None), dict(dz=None)):
        assert bb(**bad) == 1, bad


def _record_errors(name):
    """Two errors in a row for each number that the reader puts into word 8, then that number in word 9."""
    shm = SharedMemory(name)
    w = memoryview(shm.buf).cast("I")
    try:
        done = w[9] = 0xFFFFFFFF
        while (t := w[8]) != 0xFFFFFFFF:
            if t == done:
                continue
            for _ in range(t % 50):  # at any time
                pass
            w[3], w[1] = 9, 2 * t & 0xFFFFFFFF
            w[3], w[1] = 9, 2 * t + 1 & 0xFFFFFFFF
            w[9] = done = t
    finally:
        w.release()
        shm.close()


def test_errors_recorded_while_others_are_read_are_not_lost():
    """What a kernel writes into the status words while the host takes an earlier error is in that result or in
    the next. The kernel is another process here, the mapped words shared memory."""
    take = _host().take_status_error
    shm = SharedMemory(create=True, size=64)
    w = memoryview(shm.buf).cast("I")
    probe = ctypes.c_char.from_buffer(shm.buf)
    address = ctypes.addressof(probe)
    writer = multiprocessing.get_context("spawn").Process(target=_record_errors, args=(shm.name,), daemon=True)
    lost = t = 0
    try:
        for i in range(16):
            w[i] = 0
        w[8] = 0xFFFFFFFE  # a number to begin with: the writer is there once it has answered
        assert take(address) == (0, 0)
        writer.start()
        while w[9] != 0xFFFFFFFE:
            assert writer.is_alive()
        assert take(address) == (0xFFFFFFFD, 9)
        stop = time.monotonic() + 4.0
        while time.monotonic() < stop:
            t += 1
            w[8], last, done = t, 0, False
            for turn in itertools.count(1):
                assert turn % 65536 or writer.is_alive()
                flags, site = take(address)
                if flags:
                    assert site == 9
                    last = flags
                elif done:
                    break
                done = w[9] == t
            lost += last != 2 * t + 1
    finally:
        w[8] = 0xFFFFFFFF
        writer.join(60)
        w.release()
        del probe
        shm.close()
        shm.unlink()
    assert t > 0 and lost == 0


# ---- the 64-bit restatements themselves, against differences --------------------
def _directional(f, x, v, h=1e-5):
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


def test_restatements_match_differences():
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    codes = torch.tensor([[0, 4, -1], [2, 2, 1], [-1, -1, -1], [4, 0, 3]])
    T, w, up = r(5, 2, 3), r(4, 3), r(4, 2, 3)
    z, gl, gh, gt = r(4, 5), r(4), r(4), r(4, 2)
    z[1, 2], z[2] = -INF, -INF
    one = torch.tensor([1, 0, 3, -1])

    def log_probs(x):
        lp, ent, tl, _ = TR.code_log_probs_reference(x, one, 2)
        keep = torch.tensor([True, True, False, True])
        return (lp * gl)[keep].sum() + (ent * gh).sum() + (tl * gt)[keep].sum()

    for f, x in ((lambda x: (TR.codebook_lookup_reference(x, codes, w, 1.5) * up).sum(), T),
                 (lambda x: (TR.codebook_lookup_reference(T, codes, x, 1.5) * up).sum(), w),
                 (log_probs, z), (lambda x: TR.code_balance_reference(x, codes)[0], z)):
        x = x.clone().requires_grad_(True)
        grad, = torch.autograd.grad(f(x), x)
        v = r(*x.shape)
        with torch.no_grad():
            assert abs(_directional(f, x, v) - (grad * v).sum()) <= 1e-8 * (1 + grad.abs().max() * v.abs().sum())


# ---- lookup --------------------------------------------------------------------
def _lookup_case(rows, C, row, bag, dtype, seed, *, empty=0.1, skew=3.0, wide=False):
    g = _gen(seed)
    table = (torch.randn(C, *row, device=DEV, generator=g) * 0.5).to(dtype)
    shape = (rows, bag) if bag else (rows,)
    codes = (torch.rand(shape, device=DEV, generator=g) ** skew * C).long().clamp_(max=C - 1)
    codes[torch.rand(shape, device=DEV, generator=g) < empty] = -1
    w = torch.randn(shape, device=DEV, generator=g) if bag else None
    return table, codes if wide else codes.int(), w


def _check_lookup(table, codes, w, scale, out_dtype, seed=5):
    table = table.detach().requires_grad_(True)
    w = None if w is None else w.detach().requires_grad_(True)
    out = tgb.codebook_lookup(table, codes, w, scale=scale, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    up = torch.randn(out.shape, device=DEV, generator=_gen(seed)).to(out_dtype)
    leaves = [table] + ([w] if w is not None else [])
    grads = torch.autograd.grad(out, leaves, up)
    with torch.no_grad():
        plain = tgb.codebook_lookup(table, codes, w, scale=scale, out_dtype=out_dtype)
    assert torch.equal(plain, out)
    T = table.detach().double().requires_grad_(True)
    W = None if w is None else w.detach().double().requires_grad_(True)
    ref = TR.codebook_lookup_reference(T, codes, W, scale)
    ref_g = torch.autograd.grad(ref, [T] + ([W] if W is not None else []), up.double())
    # Sums of magnitudes: the same formulas on absolute values.
    Ta = T.detach().abs().requires_grad_(True)
    Wa = None if W is None else W.detach().abs().requires_grad_(True)
    mag = TR.codebook_lookup_reference(Ta, codes, Wa, abs(scale))
    mag_g = torch.autograd.grad(mag, [Ta] + ([Wa] if Wa is not None else []), up.double().abs())
    J = codes.shape[-1] if w is not None else 1
    _close(out.detach(), ref.detach(), (J + 2) * U * mag.detach(), out_dtype)
    used = torch.bincount(codes[codes >= 0].long().reshape(-1), minlength=table.shape[0])
    n = used.reshape(-1, *([1] * (table.ndim - 1))).double()
    _close(grads[0], ref_g[0], (n + 3) * U * mag_g[0], table.dtype)
    assert grads[0].dtype == table.dtype and grads[0].shape == table.shape
    if w is not None:
        dim = max(1, table[0].numel())
        _close(grads[1], ref_g[1], (dim + 3) * U * mag_g[1], torch.float32)
    return out, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, C, row, bag, wide", [
    (1, 1, (1,), 0, False), (1, 9, (16, 3), 4, True), (2, 3, (3,), 1, False), (63, 5, (4, 3), 0, True),
    (257, 70, (9, 3), 3, False), (1000, 1000, (59,), 0, False), (4099, 33, (16, 3), 2, False),
    (20000, 7, (8,), 8, True), (5001, 40000, (11,), 0, False), (300, 17, (300,), 2, False), (77, 6, (1030,), 5, True),
])
def test_lookup_matches_reference(dtype, rows, C, row, bag, wide):
    table, codes, w = _lookup_case(rows, C, row, bag, dtype, seed=rows + C, wide=wide)
    _check_lookup(table, codes, w, 1.25, dtype)
    _check_lookup(table, codes, w, -0.5, torch.float32)


@pytest.mark.gpu
def test_lookup_out_types_mix():
    table, codes, w = _lookup_case(515, 40, (9, 3), 2, torch.float32, seed=8)
    _check_lookup(table, codes, w, 1.0, torch.float32)
    for dtype, other in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16)):
        with pytest.raises(ValueError, match="out_dtype"):
            tgb.codebook_lookup(table.to(dtype), codes, w, out_dtype=other)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["one code", "all empty", "two codes", "sorted", "unused"])
def test_lookup_uneven_use(kind):
    """Every splat on one code (a run through all blocks), no code at all, rows never used."""
    rows, C = 70001, 300
    table, codes, w = _lookup_case(rows, C, (16, 3), 0, torch.float32, seed=11, empty=0.0)
    if kind == "one code":
        codes.fill_(C - 1)
    elif kind == "all empty":
        codes.fill_(-7)
    elif kind == "two codes":
        codes.fill_(3)[rows // 3] = 4
    elif kind == "sorted":
        codes = codes.sort().values
    else:
        codes.clamp_(max=5)
    out, (g,) = _check_lookup(table, codes, w, 1.0, torch.float32)
    if kind == "all empty":
        assert not out.any() and not g.any()


@pytest.mark.gpu
@pytest.mark.parametrize("slots", [1, 31, 32, 33, 1000, 4096, 4097, 8191, 8192, 8193])
@pytest.mark.parametrize("C", [1, 7, 100_003])
def test_lookup_gradient_of_few_slots(slots, C):
    """Small whole numbers, whose sums are exact in any order; codes that tie, empty slots."""
    g = _gen(slots + C)
    codes = torch.randint(-1, C, (slots,), device=DEV, generator=g)
    if C > 1000:
        codes[::3] = codes[0].item()
    table = torch.zeros(C, 5, device=DEV, requires_grad=True)
    up = torch.randint(-8, 9, (slots, 5), device=DEV, generator=g).float()
    got, = torch.autograd.grad(tgb.codebook_lookup(table, codes), table, up)
    ref = torch.zeros(C + 1, 5, device=DEV).index_add_(0, torch.where(codes < 0, C, codes), up)[:C]
    assert torch.equal(got, ref)
    codes[-1] = C
    with pytest.raises(RuntimeError, match="out of bounds"):
        _ops().codebook_bwd(up, table.detach(), codes, None, 1.0, True, False)
        tgb.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_lookup_shapes_strides_and_offsets(dtype):
    g = _gen(21)
    big = (torch.randn(50, 16, 3, device=DEV, generator=g)).to(dtype)
    codes = torch.randint(-1, 50, (6, 7, 2), device=DEV, generator=g)
    w = torch.randn(6, 7, 2, device=DEV, generator=g)
    for table in (big[:, :9], big[:, 1:5], big[1::2][:20], big.transpose(1, 2), big[:, 0, 0], big[:1].expand(50, 16, 3)):
        c = codes.clamp(max=table.shape[0] - 1)
        _check_lookup(table, c, w, 1.0, torch.float32)
        _check_lookup(table, c.transpose(0, 1), w.transpose(0, 1), 1.0, dtype)
        _check_lookup(table, c[..., 0], None, 2.0, dtype)
        _check_lookup(table, c[2, 3, 1], None, 1.0, dtype)
    # A gradient that is broadcast (sum().backward() hands on an expanded one).
    t = big.clone().requires_grad_(True)
    tgb.codebook_lookup(t, codes.clamp(max=49), w).float().sum().backward()
    r = big.double().requires_grad_(True)
    TR.codebook_lookup_reference(r, codes.clamp(max=49), w.double()).sum().backward()
    _close(t.grad, r.grad, 90 * U * w.abs().sum().double(), dtype)


@pytest.mark.gpu
def test_lookup_of_nothing():
    table = torch.randn(5, 3, device=DEV).requires_grad_(True)
    for shape in ((0,), (0, 4), (3, 0)):
        out = tgb.codebook_lookup(table, torch.zeros(shape, dtype=torch.int32, device=DEV))
        assert out.shape == (*shape, 3)
        g, = torch.autograd.grad(out.sum(), table)
        assert g.shape == table.shape and not g.any()
    w = torch.zeros(0, 2, device=DEV, requires_grad=True)
    out = tgb.codebook_lookup(table, torch.zeros(0, 2, dtype=torch.int32, device=DEV), w)
    gt, gw = torch.autograd.grad(out.sum(), (table, w))
    assert out.shape == (0, 3) and not gt.any() and gw.shape == (0, 2)


@pytest.mark.gpu
def test_lookup_gradient_of_many_slots():
    """More than 2^22 slots: the sort takes its prefixes another way."""
    rows, C = (1 << 20) + 77, 3001
    table, codes, w = _lookup_case(rows, C, (3,), 4, torch.float32, seed=12)
    w = w.round()  # whole numbers: sums of them are exact below 2^24
    t = table.detach().requires_grad_(True)
    g, = torch.autograd.grad(tgb.codebook_lookup(t, codes, w).sum(), t)
    keep = codes >= 0
    ref = torch.zeros(C, device=DEV, dtype=torch.float64).index_add_(0, codes[keep].long(), w[keep].double())
    assert ref.abs().max() < 2**24
    assert torch.equal(g.double(), ref[:, None].expand(C, 3))


@pytest.mark.gpu
def test_lookup_only_what_is_asked():
    table, codes, w = _lookup_case(100, 9, (5,), 2, torch.float32, seed=30)
    w.requires_grad_(True)
    out = tgb.codebook_lookup(table, codes, w)
    g, = torch.autograd.grad(out.sum(), w)
    t2 = table.clone().requires_grad_(True)
    g2 = torch.autograd.grad(tgb.codebook_lookup(t2, codes, w).sum(), (t2, w))
    assert torch.equal(g, g2[1])
    with pytest.raises(RuntimeError):  # once differentiable
        g3, = torch.autograd.grad(tgb.codebook_lookup(t2, codes, w).square().sum(), t2, create_graph=True)
        torch.autograd.grad(g3.sum(), t2)


@pytest.mark.gpu
def test_bad_codes_are_reported_and_taken_as_empty():
    table = torch.randn(10, 4, device=DEV, requires_grad=True)
    codes = torch.tensor([1, 10, 3, 2**31 - 1], dtype=torch.int32, device=DEV)
    logits = torch.randn(4, 10, device=DEV, requires_grad=True)
    calls = [lambda: tgb.codebook_lookup(table, codes), lambda: tgb.codebook_lookup(table, codes.long() + 2**40),
             lambda: tgb.code_log_probs(logits, codes), lambda: tgb.code_balance_loss(logits, codes)]
    for call in calls:  # GSPLAT_B200_CHECK: reported by the call itself, once
        with pytest.raises(RuntimeError, match="out of bounds"):
            call()
    tgb.check_device_errors()


@pytest.mark.gpu
def test_bad_codes_later(monkeypatch):
    """Without the debug check the error is raised by the next call or by
    check_device_errors(), once, and the results are those of empty slots."""
    monkeypatch.setenv("GSPLAT_B200_CHECK", "0")
    g = _gen(4)
    table = torch.randn(10, 4, device=DEV, generator=g).requires_grad_(True)
    logits = torch.randn(40, 10, device=DEV, generator=g).requires_grad_(True)
    good = torch.randint(0, 10, (40,), device=DEV, generator=g, dtype=torch.int32)
    bad, empty = good.clone(), good.clone()
    bad[3::7], empty[3::7] = 10, -1

    def passes(codes):
        out = tgb.codebook_lookup(table, codes)
        torch.cuda.synchronize()
        first = None
        try:
            lp = tgb.code_log_probs(logits, codes, top_k=2)
        except RuntimeError as e:
            first = str(e)
            lp = tgb.code_log_probs(logits, codes, top_k=2)
        res = [out, lp.log_probs, lp.entropy]
        torch.cuda.synchronize()
        try:
            tgb.check_device_errors()
        except RuntimeError:
            pass
        return first, res

    first, res = passes(bad)
    assert first is not None and "out of bounds" in first
    none, ref = passes(empty)
    assert none is None
    for a, b in zip(res, ref):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="out of bounds"):
        tgb.code_balance_loss(logits, bad)
        tgb.check_device_errors()
    tgb.check_device_errors()


# ---- log probabilities ---------------------------------------------------------
def _logits(rows, C, dtype, seed, *, spread=2.5, pad=0, masked=0.0, low=-INF):
    g = _gen(seed)
    full = (torch.randn(rows, C + pad, device=DEV, generator=g) * spread).to(dtype)
    z = full[:, :C]
    if masked:
        z.masked_fill_(torch.rand(rows, C, device=DEV, generator=g) < masked, low)
    return z


def _row_terms(z):
    """x = z - max, p and 1 + log-ish scale of each row, for the tolerances."""
    zd = z.detach().double()
    m = zd.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    x = (zd - m).clamp(min=-64.0)
    e = torch.where(torch.isinf(zd), torch.zeros_like(x), x.exp())
    s = e.sum(-1, keepdim=True).clamp(min=1.0)
    return x, e / s, REL_EXP + (z.shape[-1] / 32 + 32) * U


def _check_log_probs(z, codes, k, *, use=(True, True, True), seed=6):
    z = z.detach().requires_grad_(True)
    r = tgb.code_log_probs(z, codes, top_k=k)
    ref_in = z.detach().double().requires_grad_(True)
    lp, ent, tl, tc = TR.code_log_probs_reference(ref_in, codes, k)
    x, p, d = _row_terms(z)
    C = z.shape[-1]
    assert torch.equal(r.top_codes.long(), tc) and r.top_codes.dtype == torch.int32
    for got, ref in ((r.log_probs, lp), (r.top_log_probs, tl)):
        if ref is not None:
            mag = torch.where(torch.isinf(ref), torch.zeros_like(ref), ref.detach().abs())
            _close(got.detach(), ref.detach(), 4 * U * mag + d, torch.float32)
    # H = log1p(s) - mu: d of each; |mu| <= H + log C.
    _close(r.entropy.detach(), ent.detach(), 2 * d * (1 + ent.detach().abs() + math.log(C)), torch.float32)
    with torch.no_grad():
        plain = tgb.code_log_probs(z, codes, top_k=k)
    for a, b in zip(plain, r):
        assert (a is None and b is None) or torch.equal(a, b)
    g = _gen(seed)
    outs, refs, ups = [], [], []
    for want, got, ref in ((use[0] and codes is not None, r.log_probs, lp), (use[1], r.entropy, ent), (use[2] and k > 0, r.top_log_probs, tl)):
        if want:
            up = torch.randn(got.shape, device=DEV, generator=g)
            outs.append(got), refs.append(torch.where(torch.isinf(ref), torch.zeros_like(ref), ref)), ups.append(up)
    if not outs:
        return r
    dz, = torch.autograd.grad(outs, z, ups)
    assert dz.dtype == z.dtype and dz.shape == z.shape
    # -inf values of the result have no derivative in the restatement; the operator's own rule
    # (sum over all of them times p) is the formula's.
    rows = z.detach().reshape(-1, C)
    pr = p.reshape(-1, C)
    some = (rows > -INF).any(-1, keepdim=True)
    lead = torch.zeros(rows.shape[0], 1, device=DEV, dtype=torch.float64)
    dref = torch.zeros(rows.shape, device=DEV, dtype=torch.float64)
    mag = torch.zeros_like(dref)
    i = 0
    if use[0] and codes is not None:
        up = torch.where(codes >= 0, ups[i].double(), 0.0).reshape(-1, 1)
        dref.scatter_add_(1, codes.clamp(min=0).long().reshape(-1, 1), up)
        mag.scatter_add_(1, codes.clamp(min=0).long().reshape(-1, 1), up.abs())
        lead += up
        i += 1
    gh = torch.zeros_like(lead)
    if use[1]:
        gh = ups[i].double().reshape(-1, 1)
        i += 1
    if use[2] and k > 0:
        up = ups[i].double().reshape(-1, k)
        dref.scatter_add_(1, tc.reshape(-1, k), up)
        mag.scatter_add_(1, tc.reshape(-1, k), up.abs())
        lead += up.sum(-1, keepdim=True)
        mag_lead = up.abs().sum(-1, keepdim=True)
    else:
        mag_lead = torch.zeros_like(lead)
    mag_lead = mag_lead + lead.abs()
    lpz = torch.log_softmax(torch.where(some, rows.double(), 0.0), -1)
    H = ent.detach().reshape(-1, 1)
    pd = lpz.exp()
    t = torch.where(pd > 0, torch.where(torch.isinf(lpz), torch.zeros_like(lpz), lpz) + H, torch.zeros_like(lpz))
    dref = torch.where(some, dref - pd * lead - gh * pd * t, torch.zeros_like(dref))
    mag = mag + pd * (mag_lead + gh.abs() * (t.abs() + 1 + math.log(C)))
    _close(dz.reshape(-1, C), dref, torch.where(some, 4 * d * mag, 0.0), z.dtype)
    return r


def _codes_for(z, seed, empty=0.1):
    g = _gen(seed)
    lead, C = z.shape[:-1], z.shape[-1]
    c = torch.randint(0, C, lead, device=DEV, generator=g, dtype=torch.int32)
    return torch.where(torch.rand(lead, device=DEV, generator=g) < empty, -1, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, C, k", [
    (1, 1, 1), (3, 2, 2), (5, 8, 0), (1, 31, 31), (129, 16, 2), (33, 32, 32), (700, 64, 4), (65, 100, 3), (40, 256, 16),
    (9, 1000, 32), (17, 1025, 1), (6, 4096, 8), (3, 8191, 5), (2, 20011, 7), (1, 70001, 32), (1, 262147, 3),
])
def test_log_probs_match_reference(dtype, rows, C, k):
    z = _logits(rows, C, dtype, seed=rows * 7 + C)
    _check_log_probs(z, _codes_for(z, 3), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, C, k", [(37, 24, 6), (50, 333, 8), (7, 5003, 4), (2, 40001, 9)])
@pytest.mark.parametrize("masked", [0.5, 0.97])
def test_log_probs_masked(dtype, rows, C, k, masked):
    z = _logits(rows, C, dtype, seed=C, pad=5, masked=masked)
    z[0] = -INF  # nothing left
    z[-1] = -INF
    z[-1, C // 2] = 1.5  # one code left
    _check_log_probs(z, _codes_for(z, 3), k)
    z = _logits(rows, C, dtype, seed=C, pad=3, masked=masked, low=torch.finfo(dtype).min)
    z[0] = torch.finfo(dtype).min  # an even row of lowest values
    _check_log_probs(z, _codes_for(z, 4), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [16, 200, 3000, 9000, 33000])
def test_log_probs_ties_and_certainty(dtype, C):
    z = torch.zeros(7, C, device=DEV, dtype=dtype)
    z[1] = 2.0  # all equal: the lowest codes come first
    z[2, ::2] = 1.0
    z[3, -1], z[3, 0] = 30.0, -30.0  # one code almost certain: H and 1 - p are small differences
    z[4, C // 3] = 12.0
    z[5, 0] = -0.0  # equal to +0
    z[6] = torch.arange(C, device=DEV).flip(0).remainder(7).to(dtype)
    codes = torch.tensor([0, C - 1, 1, C - 1, C // 3, 0, 3], device=DEV)
    r = _check_log_probs(z, codes, min(32, C))
    # Relative, not absolute: log p = -log1p(s), s = (C - 1) exp(-30 or so).
    s = (C - 2) * math.exp(-30.0) + math.exp(-60.0)
    assert abs(r.log_probs[3].item() + math.log1p(s)) <= (2 * REL_EXP + (C / 32 + 32) * U) * s
    h = math.log1p(s) + ((C - 2) * 30 * math.exp(-30.0) + 60 * math.exp(-60.0)) / (1 + s)
    assert abs(r.entropy[3].item() - h) <= (2 * REL_EXP + (C / 32 + 32) * U) * h


@pytest.mark.gpu
@pytest.mark.parametrize("C", [24, 700, 20000])
def test_log_probs_certain_gradient_is_relative(C):
    """d log p / d z at an almost certain code is 1 - p, not a difference of two ones."""
    z = torch.zeros(2, C, device=DEV).requires_grad_(True)
    with torch.no_grad():
        z[:, 5] = 25.0
    r = tgb.code_log_probs(z, torch.full((2,), 5, device=DEV), top_k=1)
    s = (C - 1) * math.exp(-25.0)
    for out in (r.log_probs, r.top_log_probs):
        g, = torch.autograd.grad(out.sum(), z, retain_graph=True)
        q = s / (1 + s)
        assert abs(g[0, 5].item() - q) <= (3 * REL_EXP + (C / 32 + 32) * U) * q


@pytest.mark.gpu
@pytest.mark.parametrize("use", [(True, False, False), (False, True, False), (False, False, True), (True, True, False)])
@pytest.mark.parametrize("C", [40, 2500])
def test_log_probs_part_of_the_gradients(use, C):
    z = _logits(19, C, torch.float32, seed=2)
    _check_log_probs(z, _codes_for(z, 5), 4, use=use)
    if not use[0]:
        _check_log_probs(z, None, 4, use=use)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_shapes_and_strides(dtype):
    z = _logits(24, 1001, dtype, seed=9, pad=23)
    _check_log_probs(z[1:], _codes_for(z[1:], 1), 3)  # odd offset
    _check_log_probs(z[:, 1:], _codes_for(z, 1), 3)
    _check_log_probs(z[::3], _codes_for(z[::3], 1), 3)
    t = _logits(64, 30, dtype, seed=9).t()  # strided values
    _check_log_probs(t, _codes_for(t, 1), 3)
    e = _logits(1, 300, dtype, seed=10).expand(5, 300)
    _check_log_probs(e, _codes_for(e, 1), 3)
    b = _logits(24, 50, dtype, seed=11).reshape(4, 6, 50)
    _check_log_probs(b, _codes_for(b, 1).long(), 3)
    _check_log_probs(b.transpose(0, 1), _codes_for(b.transpose(0, 1), 1), 3)
    one = _logits(1, 50, dtype, seed=12)[0]
    _check_log_probs(one, torch.tensor(7, device=DEV), 3)
    for shape in ((0, 5), (3, 0, 5)):
        r = tgb.code_log_probs(torch.zeros(shape, device=DEV, dtype=dtype), top_k=2)
        assert r.log_probs is None and r.entropy.shape == shape[:-1] and r.top_codes.shape == (*shape[:-1], 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, C, k", [(101, 7, 3), (70, 61, 2), (40, 129, 9), (37, 255, 4), (9, 1027, 3),
                                        (5, 5001, 2), (3, 20001, 5)])
@pytest.mark.parametrize("offset", [1, 3, 6])
def test_rows_between_16_byte_boundaries(dtype, rows, C, k, offset):
    """Contiguous rows of odd length from an odd address on: the first row begins inside a
    16-byte piece whose other values are no part of the tensor."""
    g = _gen(C + offset)
    flat = (torch.randn(rows * C + offset + 8, device=DEV, generator=g) * 2.5).to(dtype)
    flat[:offset], flat[offset + rows * C :] = math.nan, math.nan
    z = flat[offset : offset + rows * C].view(rows, C)
    _check_log_probs(z, _codes_for(z, 1), k)
    codes = torch.randint(-1, C, (rows, 2), device=DEV, generator=g)
    _check_balance(z, codes, 10.0)
    assert flat[:offset].isnan().all() and flat[offset + rows * C :].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C, k", [(20, 20), (100, 32), (400, 12), (3001, 32)])
def test_alternatives_around_nan_and_ties(dtype, C, k):
    """NaN comes after every number, from the lowest code on; equal values by code."""
    g = _gen(C)
    z = torch.randint(-2, 3, (33, C), device=DEV, generator=g).to(dtype)  # five values: many ties
    r = tgb.code_log_probs(z, top_k=k)
    assert torch.equal(r.top_codes.long(), torch.argsort(z.float(), dim=-1, descending=True, stable=True)[:, :k])
    z[:, :] = math.nan  # and fewer numbers than alternatives
    for row in range(33):
        keep = torch.randperm(C, device=DEV, generator=g)[: min(k // 2, C)]
        z[row, keep] = torch.randn(keep.numel(), device=DEV, generator=g).to(dtype)
    r = tgb.code_log_probs(z, top_k=k)
    low = torch.where(z.isnan(), -INF, z.float())
    ref = torch.argsort(low, dim=-1, descending=True, stable=True)[:, :k]
    assert torch.equal(r.top_codes.long(), ref)
    assert r.log_probs is None and r.entropy.isnan().all() and r.top_log_probs.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("C", [12, 500, 9001])
def test_log_probs_not_finite(C):
    z = torch.zeros(4, C, device=DEV)
    z[0, 3], z[1, 2] = math.nan, INF
    z[2] = 3e38
    z[3, 1::2] = -3e38
    r = tgb.code_log_probs(z, torch.zeros(4, dtype=torch.int32, device=DEV), top_k=3)
    assert r.log_probs[:2].isnan().all() and r.entropy[:2].isnan().all() and r.top_log_probs[:2].isnan().all()
    assert r.top_codes[0].tolist() == [0, 1, 2] and r.top_codes[1].tolist() == [2, 0, 1]
    assert abs(r.entropy[2].item() - math.log(C)) <= 1e-5 and abs(r.entropy[3].item() - math.log((C + 1) // 2)) <= 1e-5


# ---- balance -------------------------------------------------------------------
def _check_balance(z, codes, up=1.0):
    z = z.detach().requires_grad_(True)
    r = tgb.code_balance_loss(z, codes)
    C = z.shape[-1]
    x = z.detach().double().reshape(-1, C).requires_grad_(True)
    J = codes.numel() // max(1, x.shape[0])
    loss, counts = TR.code_balance_reference(x, codes.reshape(-1, J))
    assert r.counts.dtype == torch.int32 and torch.equal(r.counts.long(), counts)
    d = REL_EXP + (C / 32 + 32) * U
    _close(r.loss.detach(), loss.detach(), 3 * d * loss.detach().abs(), torch.float32)
    with torch.no_grad():
        plain = tgb.code_balance_loss(z, codes)
    assert torch.equal(plain.loss, r.loss) and torch.equal(plain.counts, r.counts)
    dz, = torch.autograd.grad(r.loss, z, torch.tensor(up, device=DEV))
    ref, = torch.autograd.grad(loss, x, torch.tensor(up, device=DEV, dtype=torch.float64))
    assert dz.dtype == z.dtype and dz.shape == z.shape
    # dz_c = k p_c ((n_c - n_a) - dr): magnitudes |n_c - n_a| + sum p |n - n_a|, a the row's first largest.
    zz = x.detach()
    some = (zz > -INF).any(-1, keepdim=True)
    p = torch.softmax(torch.where(some, zz, 0.0), -1)
    n = counts.double()
    off = (n - n[zz.argmax(-1)][:, None]).abs()
    k = up * C / max(1, int(counts.sum())) / max(1, int((codes.reshape(-1, J) >= 0).any(-1).sum()))
    # The restatement's own error, in 64 bits: it forms n_c - sum p n from values as large as n (C products and
    # C sums of them, 2^-53 each), where the operator forms n_c - n_a without any. At a row whose largest p is
    # 1 - 1e-26 the true value, 1e-26 n, is below that, and the restatement gives 0.
    own = 2.0**-53 * (2 * C + 4) * (n + (p * n).sum(-1, keepdim=True))
    tol = abs(k) * p * (4 * d * (off + (p * off).sum(-1, keepdim=True)) + own)
    _close(dz.reshape(-1, C), ref, tol, z.dtype)
    return r


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, C, bag", [
    (1, 1, 1), (2, 3, 2), (31, 8, 1), (512, 64, 1), (130, 33, 4), (1000, 256, 2), (77, 1000, 8), (40, 1031, 1),
    (21, 5000, 3), (5, 17000, 2), (3, 70001, 1),
])
def test_balance_matches_reference(dtype, rows, C, bag):
    z = _logits(rows, C, dtype, seed=rows + C, pad=C % 3)
    codes = z.topk(bag, -1).indices.int()
    codes[2::5] = -1
    if bag > 1:
        codes[1::3, 0] = -1
    up = max(1.0, rows * min(C, rows * bag) / 16)
    _check_balance(z, codes, up)
    if bag == 1:
        _check_balance(z, codes[:, 0].long(), up)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [20, 600, 9001])
def test_balance_masks(C):
    z = _logits(64, C, torch.float32, seed=C, masked=0.6)
    z[5] = -INF
    z[6] = torch.finfo(torch.float32).min
    z[7, 3] = 60.0  # one code almost certain
    codes = torch.randint(-1, C, (64, 2), device=DEV, generator=_gen(1))
    _check_balance(z, codes, 100.0)
    _check_balance(z.reshape(4, 16, C), codes.reshape(4, 16, 2), 100.0)
    none = _check_balance(z, torch.full((64,), -1, device=DEV), 100.0)
    assert none.loss.item() == 0.0 and not none.counts.any()
    empty = tgb.code_balance_loss(torch.zeros(0, C, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV))
    assert empty.loss.item() == 0.0 and empty.counts.shape == (C,) and not empty.counts.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [20, 301, 600, 9001])
def test_balance_rows_without_a_code_may_hold_anything(dtype, C):
    """They take no part: the loss, and the others' gradient, as if they held zeros, and
    no gradient of their own."""
    z = _logits(40, C, dtype, seed=C)
    codes = torch.randint(0, C, (40, 2), device=DEV, generator=_gen(3))
    codes[1::4] = -1
    clean = z.clone()
    clean[1::4] = 0.0
    z[1], z[5], z[9], z[13, 2], z[17, 1], z[21] = math.nan, INF, -INF, math.nan, INF, torch.finfo(dtype).max
    _check_balance(clean, codes, 50.0)
    got, ref = [], []
    for x, out in ((z, got), (clean, ref)):
        x = x.detach().requires_grad_(True)
        r = tgb.code_balance_loss(x, codes)
        out += [r.loss.detach(), r.counts, *torch.autograd.grad(r.loss, x, torch.tensor(50.0, device=DEV))]
    # Rows of a warp may take another way than with zeros beside them: both results are within the bounds of
    # _check_balance, so within twice those (off is at most the largest count), and each is rounded.
    d = REL_EXP + (C / 32 + 32) * U
    n, loss = int(got[1].max()), ref[0].double()
    _close(got[0], loss, 6 * d * loss + U * loss, torch.float32)
    assert torch.equal(got[1], ref[1])
    k = 50.0 * C / int(got[1].sum()) / 30
    tol = 8 * k * d * torch.softmax(clean.double(), -1) * 2 * n
    _close(got[2], ref[2].double(), tol + _half_step(dtype) * (ref[2].double().abs() + tol), dtype)
    assert not got[2][1::4].any() and got[2][0].any()


@pytest.mark.gpu
def test_balance_certain_rows_are_relative():
    """One row, one code: dz at it is k p (1 - p), with 1 - p far below a step of fp32."""
    for C in (24, 3000, 40000):
        z = torch.zeros(1, C, device=DEV)
        z[0, 5] = 25.0
        _check_balance(z, torch.tensor([5], device=DEV), 1.0e6)
        z = z.requires_grad_(True)
        g, = torch.autograd.grad(tgb.code_balance_loss(z, torch.tensor([5], device=DEV)).loss, z)
        s = (C - 1) * math.exp(-25.0)
        ref = C * s / (1 + s) ** 2
        assert abs(g[0, 5].item() - ref) <= 4 * (REL_EXP + (C / 32 + 32) * U) * ref


@pytest.mark.gpu
@pytest.mark.parametrize("C", [16, 60, 300, 5000])
def test_balance_of_many_codes_a_row(C):
    """More codes a row than lanes that take it."""
    z = _logits(19, C, torch.bfloat16, seed=C)
    codes = torch.randint(-1, C, (19, 45), device=DEV, generator=_gen(2))
    codes[3] = -1
    codes[4, :44] = -1
    _check_balance(z, codes, 50.0)


@pytest.mark.gpu
def test_balance_of_even_use_is_one():
    C = 128
    z = torch.zeros(C * 3, C, device=DEV)
    r = tgb.code_balance_loss(z, torch.arange(C * 3, device=DEV) % C)
    assert abs(r.loss.item() - 1.0) <= 1e-6 and r.counts.tolist() == [3] * C


# ---- all of them ---------------------------------------------------------------
@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call():
    table, codes, w = _lookup_case(30000, 50, (9, 3), 3, torch.float32, seed=1)
    z = _logits(3000, 900, torch.bfloat16, seed=2)
    table.requires_grad_(True), w.requires_grad_(True), z.requires_grad_(True)
    c = _codes_for(z, 2)

    def run():
        out = tgb.codebook_lookup(table, codes, w)
        lp = tgb.code_log_probs(z, c, top_k=4)
        bal = tgb.code_balance_loss(z, lp.top_codes)
        loss = out.square().sum() + lp.log_probs.sum() + lp.entropy.sum() + lp.top_log_probs.sum() + bal.loss
        return [out, *lp, *bal, *torch.autograd.grad(loss, (table, w, z))]

    first = run()
    for _ in range(3):
        for a, b in zip(run(), first):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_rows_behind_2_31_values():
    """Offsets beyond 32 bits, in logits and in a looked-up result."""
    C = (1 << 15) + 1
    rows = (1 << 16) + 3
    z = torch.zeros(rows, C, device=DEV, dtype=torch.bfloat16)
    z[-2:] = _logits(2, C, torch.bfloat16, seed=3)
    z.requires_grad_(True)
    codes = torch.full((rows,), -1, device=DEV, dtype=torch.int32)
    codes[-2:] = 7
    r = tgb.code_log_probs(z, codes, top_k=2)
    b = tgb.code_balance_loss(z, codes)
    g, = torch.autograd.grad(r.log_probs.sum() + b.loss, z)
    tail = z.detach()[-2:].requires_grad_(True)
    rt, bt = tgb.code_log_probs(tail, codes[-2:], top_k=2), tgb.code_balance_loss(tail, codes[-2:])
    gt, = torch.autograd.grad(rt.log_probs.sum() + bt.loss, tail)
    assert torch.equal(r.top_codes[-2:], rt.top_codes) and torch.equal(b.counts, bt.counts)
    _close(r.log_probs[-2:].detach(), rt.log_probs.detach().double(), 1e-5, torch.float32)
    _close(g[-2:], gt.double(), 2.0**-6 * gt.abs().max().item(), torch.bfloat16)
    assert not g[:1000].any()
    del z, g, r, b
    table = torch.randn(9, 2051, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    n = (1 << 20) + 7
    out = tgb.codebook_lookup(table, (torch.arange(n, device=DEV) % 9).int())
    assert torch.equal(out[-9:], table.detach()[torch.arange(n - 9, n, device=DEV) % 9])
    up = torch.zeros_like(out)
    up[-1] = 1.0
    g, = torch.autograd.grad(out, table, up)
    assert g[(n - 1) % 9].eq(1).all() and g.float().sum().item() == 2051


@pytest.mark.gpu
def test_side_stream_and_device_guard():
    table, codes, w = _lookup_case(5000, 60, (27,), 2, torch.float32, seed=1)
    z = _logits(500, 300, torch.float32, seed=2)
    c = _codes_for(z, 2)

    def run():
        t, ww, zz = (x.detach().requires_grad_(True) for x in (table, w, z))
        out = tgb.codebook_lookup(t, codes, ww)
        lp = tgb.code_log_probs(zz, c, top_k=4)
        bal = tgb.code_balance_loss(zz, lp.top_codes)
        loss = out.square().sum() + lp.entropy.sum() + lp.top_log_probs.sum() + bal.loss
        return [out.detach(), *torch.autograd.grad(loss, (t, ww, zz))]

    ref = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_training_passes_replay(monkeypatch):
    """Two graphs of forward and backward, replayed in turn on new inputs, with the
    eager results of the same inputs; bad codes in a replay are reported after it."""
    monkeypatch.setenv("GSPLAT_B200_CHECK", "0")

    def make(seed, rows):
        table, codes, w = _lookup_case(rows, 60, (9, 3), 2, torch.float32, seed=seed)
        z = _logits(rows, 130, torch.float32, seed=seed + 1)
        return [table, w, z], codes, _codes_for(z, seed + 2)

    def run(leaves, codes, c):
        t, w, z = (x.detach().requires_grad_(True) for x in leaves)
        out = tgb.codebook_lookup(t, codes, w)
        lp = tgb.code_log_probs(z, c, top_k=3)
        bal = tgb.code_balance_loss(z, lp.top_codes)
        loss = out.square().sum() + lp.log_probs.sum() + lp.entropy.sum() + lp.top_log_probs.sum() + bal.loss
        return [out.detach(), bal.counts, *torch.autograd.grad(loss, (t, w, z))]

    graphs = []
    for seed, rows in ((1, 3000), (5, 1700)):
        state = make(seed, rows)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*state)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run(*state)
        graphs.append((g, state, outs, rows))
    for turn in range(3):
        for g, (leaves, codes, c), outs, rows in graphs:
            new, ncodes, nc = make(100 + turn, rows)
            for a, b in zip([*leaves, codes, c], [*new, ncodes, nc]):
                a.copy_(b)
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, state, outs, rows in graphs:
            for a, b in zip(outs, run(*state)):
                assert torch.equal(a, b)
    graphs[0][1][1][7, 0] = 60  # a code behind the codebook
    graphs[0][0].replay()
    with pytest.raises(RuntimeError, match="out of bounds"):
        tgb.check_device_errors()
    tgb.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_codebook_colors(dtype):
    """spherical_harmonics_colors with codes is the lookup in front of it."""
    g = _gen(3)
    book = (torch.randn(40, 16, 3, device=DEV, generator=g) * 0.3).to(dtype)
    means = torch.randn(500, 3, device=DEV, generator=g) * 4
    c2w = torch.eye(4, device=DEV).repeat(2, 1, 1)
    c2w[:, :3, 3] = torch.randn(2, 3, device=DEV, generator=g) * 9
    codes = torch.randint(0, 40, (500, 2), device=DEV, generator=g, dtype=torch.int32)
    w = torch.softmax(torch.randn(500, 2, device=DEV, generator=g), -1)
    up = torch.randn(2, 500, 3, device=DEV, generator=g)
    for degree, cc, ww in ((3, codes, w), (2, codes[:, 0], None), (0, codes[:, 1].long(), None)):
        K = (degree + 1) ** 2
        a = book.clone().requires_grad_(True)
        out = tgb.spherical_harmonics_colors(a, means, c2w, degree=degree, codes=cc, code_weights=ww)
        b = book.clone().requires_grad_(True)
        sh = tgb.codebook_lookup(b[:, :K], cc, ww, out_dtype=torch.float32)
        ref = tgb.spherical_harmonics_colors(sh, means, c2w, degree=degree)
        assert torch.equal(out, ref)
        out.backward(up), ref.backward(up)
        assert torch.equal(a.grad, b.grad) and a.grad[:, :K].any() and not a.grad[:, K:].any()


@pytest.mark.gpu
def test_learning_codes_through_the_rasterizer():
    """Logits -> alternatives -> weighted lookup -> SH colours -> image, with the
    entropy and the balance loss: the gradients of logits and codebook against
    differences of the loss along their own direction."""
    G, C, K, H, W = 400, 24, 4, 48, 64
    g = _gen(17)
    means = torch.randn(G, 3, device=DEV, generator=g) * 0.8 + torch.tensor([0.0, 0.0, 4.0], device=DEV)
    scales = torch.rand(G, 3, device=DEV, generator=g) * 0.1 + 0.05
    quats = torch.nn.functional.normalize(torch.randn(G, 4, device=DEV, generator=g), dim=-1)
    opac = torch.rand(G, device=DEV, generator=g) * 0.5 + 0.3
    c2w = torch.eye(4, device=DEV)[None]
    cfg = tgb.RasterConfig(H, W)
    target = torch.rand(1, H, W, 3, device=DEV, generator=g)
    book = (torch.randn(C, 9, 3, device=DEV, generator=g) * 0.2).requires_grad_(True)
    logits = torch.randn(G, C, device=DEV, generator=g)
    # The chosen codes stand 3 above the others, so that they stay the same ones along the step.
    logits.scatter_add_(1, logits.topk(K, -1).indices, torch.full((G, K), 3.0, device=DEV))
    logits.requires_grad_(True)

    def loss_of(book, logits):
        p = tgb.code_log_probs(logits, top_k=K)
        w = torch.softmax(p.top_log_probs, -1)
        colors = tgb.spherical_harmonics_colors(book, means, c2w, degree=2, codes=p.top_codes, code_weights=w)
        b = means[None], scales[None], quats[None], opac[None]
        image = tgb.rasterize_pinhole_gaussians(*b, colors, 50.0, 50.0, W / 2, H / 2, c2w, config=cfg)
        fit = (image.double() - target.double()).square().mean()
        return fit + 1e-3 * p.entropy.double().mean() + 1e-2 * tgb.code_balance_loss(logits, p.top_codes).loss.double()

    loss = loss_of(book, logits)
    grads = torch.autograd.grad(loss, (book, logits))
    for i, (x, gx) in enumerate(zip((book, logits), grads)):
        v = gx / gx.norm()
        h = 0.05 if i == 0 else 0.02
        with torch.no_grad():
            args = [book, logits]
            args[i] = x + h * v
            up = loss_of(*args)
            args[i] = x - h * v
            down = loss_of(*args)
        # What is left is the third derivative's h^2 / 6, and 2^-24 of the pixels over h.
        assert abs((up - down).item() / (2 * h) - gx.norm().item()) <= 0.05 * gx.norm().item()

@pytest.mark.gpu
def test_backward_ops_refuse_tensors_of_other_devices():
    """The registered backward ops check what a caller hands back to them."""
    ops = _ops()
    z = _logits(6, 40, torch.float32, seed=1)
    codes = _codes_for(z, 1).clamp(min=0)
    _, ent, top, tc, stats = ops.code_log_probs_fwd(z, codes, 3, True)
    args = [torch.ones(6, device=DEV), torch.ones_like(ent), torch.ones_like(top), z, codes, tc, stats]
    assert ops.code_log_probs_bwd(*args).shape == z.shape
    for i in (0, 1, 2, 4, 5, 6):
        with pytest.raises(ValueError):
            ops.code_log_probs_bwd(*args[:i], args[i].cpu(), *args[i + 1 :])
    loss, _, stats, state = ops.code_balance_fwd(z, codes, True)
    args = [torch.ones_like(loss), z, stats, state]
    assert ops.code_balance_bwd(*args).shape == z.shape
    for i in (0, 2, 3):
        with pytest.raises(ValueError):
            ops.code_balance_bwd(*args[:i], args[i].cpu(), *args[i + 1 :])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [40, 41, 600, 9001])
@pytest.mark.parametrize("low", [-1e4, -1e18, -1e30, -1e34, -1e37, -9e37])
def test_entropy_gradient_at_very_low_logits(dtype, C, low):
    """Finite values far below the others (masks of a large number): their gradient is 0, the others' what it is
    without them, whatever the size of the incoming gradient. fp16 has no such values."""
    z = _logits(7, C, dtype, seed=C)
    z[0, 1::2] = low
    z[1, :-1] = low  # one code stands: p = 1, H = 0
    z[2] = low  # an even row
    z[3, 2:] = low
    z[3, :2] = 0.5  # two even codes
    z[4, :] += 2000.0
    z[4, C // 2 :] = low
    z[5, : C // 2] = low
    z[5, C // 3] = low * 1.5
    x = z.double()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    H = -(p * lp.clamp(min=-1e6)).sum(-1, keepdim=True)
    t = torch.where(p > 0, lp + H, 0.0)
    d = REL_EXP + (C / 32 + 32) * U
    for rows in (slice(0, 7), *(slice(i, i + 1) for i in range(7))):  # rows of a warp may go one way together
        for gh in (1.0, 10.0, 64.0, 65536.0, 1e9, 1e30):
            leaf = z[rows].detach().requires_grad_(True)
            ent = tgb.code_log_probs(leaf).entropy
            dz, = torch.autograd.grad(ent, leaf, torch.full_like(ent, gh))
            q, u = p[rows], t[rows]
            _close(dz, -gh * q * u, 4 * d * gh * q * (u.abs() + 1 + math.log(C)), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, C", [(1, 70001), (2, 30011), (1, 262147), (3, 9001), (2, 40)])
def test_best_code_behind_nan(dtype, rows, C):
    """NaN comes after -inf too, where a row is split into parts and some of them hold NaN alone."""
    first = C // 2 + 3
    z = torch.full((rows, C), -INF, device=DEV, dtype=dtype)
    z[:, :first] = math.nan
    for k in (1, 2):
        r = tgb.code_log_probs(z, top_k=k)
        assert r.top_codes.tolist() == [list(range(first, first + k))] * rows and r.top_log_probs.isnan().all()
    z[-1] = math.nan
    assert tgb.code_log_probs(z, top_k=1).top_codes[-1].item() == 0
    z[:, -1] = -3.0
    assert tgb.code_log_probs(z, top_k=1).top_codes[:, 0].tolist() == [C - 1] * rows


@pytest.mark.gpu
def test_lookup_gradient_beside_errors_of_other_calls():
    """Status words that hold an earlier call's error: the sort's waits must not take it for their own. Two
    streams at once, so that blocks wait for others; whole numbers, whose sums are exact."""
    L = N.load()
    n, C = (1 << 21) + 5, 70_003
    g = _gen(9)
    codes = torch.randint(-1, C, (n,), device=DEV, generator=g, dtype=torch.int32)
    up = torch.randint(-8, 9, (n,), device=DEV, generator=g).float()
    ref = torch.zeros(C + 1, device=DEV).index_add_(0, torch.where(codes < 0, C, codes), up)[:C]
    status = torch.zeros(16, dtype=torch.int32, device=DEV)
    status[1], status[3] = N.DEVERR_BOUNDS, 9
    before = status.clone()
    size = L.gsb_codebook_backward_workspace_size(n, 1, C, 1)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ws = [torch.full((size,), 255, dtype=torch.uint8, device=DEV) for _ in streams]
    got = [[torch.full((C,), math.nan, device=DEV) for _ in range(6)] for _ in streams]
    torch.cuda.synchronize()
    for turn in range(6):
        for s, w, out in zip(streams, ws, got):
            rc = L.gsb_codebook_backward(0, 0, n, 1, C, 1, None, 1, codes.data_ptr(), 4, None, 1.0, up.data_ptr(),
                                         out[turn].data_ptr(), None, status.data_ptr(), w.data_ptr(), size,
                                         s.cuda_stream)
            assert rc == 0
    torch.cuda.synchronize()
    for out in got:
        for t in out:
            assert torch.equal(t, ref)
    assert torch.equal(status, before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [48, 27, 300, 400])
@pytest.mark.parametrize("bag", [0, 2])
@pytest.mark.parametrize("kind", ["one code", "two codes", "sorted", "even"])
def test_lookup_gradients_of_much_used_codes_are_exact(dtype, dim, bag, kind):
    """Runs that cross stretches and blocks, in rows of whole pieces, odd rows and rows of two tiles: small
    whole numbers, whose sums (below 2^24) are exact in any order and are rounded once to the result's type. A
    block that is left out or counted twice shows in every column."""
    rows, C = (70001, 300) if dim < 300 else (20011, 40)
    g = _gen(dim + bag)
    shape = (rows, bag) if bag else (rows,)
    codes = torch.randint(0, C, shape, device=DEV, generator=g)
    if kind == "one code":
        codes.fill_(C - 1)
    elif kind == "two codes":
        codes.fill_(3)[rows // 3 :] = 4
    elif kind == "sorted":
        codes = codes.reshape(-1).sort().values.reshape(shape)
    codes[torch.rand(shape, device=DEV, generator=g) < 0.1] = -1
    whole = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, device=DEV, generator=g).float()
    table = whole(-3, 3, C, dim).to(dtype).requires_grad_(True)
    w = whole(-2, 2, *shape).requires_grad_(True) if bag else None
    up = whole(1, 4, rows, dim)  # of one sign: sums that nothing cancels
    out = tgb.codebook_lookup(table, codes, w, out_dtype=torch.float32)
    T = table.detach().double()
    cc = codes.reshape(rows, -1)
    ww = (w.detach() if bag else torch.ones(rows, 1, device=DEV)).double() * (cc >= 0)
    picked = T[cc.clamp(min=0)]
    assert torch.equal(out.detach().double(), (picked * ww[..., None]).sum(1))
    grads = torch.autograd.grad(out, (table, w) if bag else (table,), up)
    ref = torch.zeros(C, dim, device=DEV, dtype=torch.float64)
    for j in range(cc.shape[1]):
        ref.index_add_(0, cc[:, j].clamp(min=0), up.double() * ww[:, j, None])
    assert ref.abs().max() < 2**24
    assert torch.equal(grads[0], ref.to(dtype))
    if bag:
        assert torch.equal(grads[1].double(), (picked * up.double()[:, None]).sum(-1) * (cc >= 0))


# ---- the sources ---------------------------------------------------------------
def test_local_arrays_read_wide_are_aligned():
    """A local array of narrow values that is read as one 16-byte (or 8-byte) value lies on such a boundary
    only if it says so: nothing else promises it once the array is in memory."""
    csrc = Path(N.__file__).resolve().parents[1] / "csrc"
    for path in sorted((*csrc.glob("*.cu"), *csrc.glob("*.cuh"))):
        text = path.read_text()
        for name in set(re.findall(r"\*reinterpret_cast<(?:const )?(?:uint|int|float)[24]\*>\((\w+)\)", text)):
            plain = re.findall(rf"^\s*(?!extern|__shared__|.*__align__|.*alignas)[\w:<>]+ {name}\[[^]]*\];", text, re.M)
            assert not plain, f"{path.name}: {plain}"
