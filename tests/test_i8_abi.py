"""Layers in 8-bit integers without a GPU: sizes, refusals (all before any device call), the binding's checks, and the oracle's
own properties."""
import numpy as np
import pytest
import torch

import densecore_amd as dc
from oracle import i8 as I

OK, INVALID, UNSUPPORTED, BAD_SHAPE, MISALIGNED, WORKSPACE, NO_DEVICE = 0, -1, -2, -3, -4, -5, -7
F32, F16, Q8_0 = 0, 1, 8
BIG = 0x10000000
NO_GPU = not torch.cuda.is_available()


def quantize(t=F32, x=0x100000, m=4, k=64, xs=None, q=0x200000, qs=None, s=0x300000):
    return dc.lib().dcq_quantize_i8(t, x, m, k, (k * (2 if t == F16 else 4)) if xs is None else xs, q, k if qs is None else qs, s, None)


@pytest.mark.parametrize("kw,want", [
    (dict(t=Q8_0), UNSUPPORTED), (dict(m=0), BAD_SHAPE), (dict(m=1 << 22), BAD_SHAPE), (dict(k=0), BAD_SHAPE), (dict(k=40), BAD_SHAPE),
    (dict(k=131072), BAD_SHAPE), (dict(x=None), INVALID), (dict(q=None), INVALID), (dict(s=None), INVALID), (dict(xs=128), INVALID),
    (dict(qs=48), INVALID), (dict(xs=(1 << 24) + 16), INVALID), (dict(xs=264), MISALIGNED), (dict(qs=72), MISALIGNED),
    (dict(x=0x100008), MISALIGNED), (dict(q=0x200004), MISALIGNED), (dict(s=0x300002), MISALIGNED), (dict(q=0x100100), INVALID),
    (dict(s=0x200010), INVALID), (dict(s=0x100000), INVALID),
])
def test_quantize_refusals(kw, want):
    assert quantize(**kw) == want


def norm(t=F32, x=0x100000, xs=None, r=0x200000, rs=None, h=0x300000, hs=None, w=0x400000, eps=1e-6, m=4, k=64, q=0x500000, qs=None,
         s=0x600000, y=None, ys=0):
    f = k * 4
    return dc.lib().dcq_rms_norm_i8(t, x, (f if t == F32 else f // 2) if xs is None else xs, r, f if rs is None else rs, h,
                                    f if hs is None else hs, w, eps, m, k, q, k if qs is None else qs, s, y, ys, None)


@pytest.mark.parametrize("kw,want", [
    (dict(t=2), UNSUPPORTED), (dict(m=0), BAD_SHAPE), (dict(m=1 << 22), BAD_SHAPE), (dict(k=8), BAD_SHAPE), (dict(w=None), INVALID),
    (dict(q=None, s=None), INVALID), (dict(q=None), INVALID), (dict(s=None), INVALID), (dict(r=None), INVALID), (dict(h=None), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(eps=float("inf")), INVALID), (dict(x=None), INVALID),
    (dict(rs=128), INVALID), (dict(hs=128), INVALID), (dict(r=0x200004), MISALIGNED), (dict(h=0x300008), MISALIGNED),
    (dict(w=0x400004), MISALIGNED), (dict(y=0x700004, ys=256), MISALIGNED), (dict(y=0x700000, ys=128), INVALID),
    (dict(h=0x100000), INVALID), (dict(h=0x200010, hs=272), INVALID), (dict(h=0x200000, hs=272), INVALID), (dict(q=0x200000), INVALID),
    (dict(q=0x300000), INVALID), (dict(s=0x500010), INVALID), (dict(y=0x300000, ys=256), INVALID), (dict(s=0x400000), INVALID),
])
def test_norm_refusals(kw, want):
    assert norm(**kw) == want


def product(w=0x1000000, ws=0x2000000, n=24, k=64, wst=None, x=0x3000000, xs=0x4000000, m=5, xst=None, r=None, rst=0, t=F32, y=0x5000000,
            yst=None, wk=None, wkb=0):
    return dc.lib().dcq_mul_mat_i8(w, ws, n, k, k if wst is None else wst, x, xs, m, k if xst is None else xst, r, rst, t, y,
                                   n * (2 if t == F16 else 4) if yst is None else yst, wk, wkb, None)


SPLIT = dict(n=2560, k=9728, m=100)  # few tiles, long K: the workspace holds planes


@pytest.mark.parametrize("kw,want", [
    (dict(t=Q8_0), UNSUPPORTED), (dict(m=0), BAD_SHAPE), (dict(n=0), BAD_SHAPE), (dict(k=24), BAD_SHAPE), (dict(k=131072), BAD_SHAPE),
    (dict(m=(1 << 22) + 1), BAD_SHAPE), (dict(m=1 << 18, n=1 << 16), BAD_SHAPE), (dict(w=None), INVALID), (dict(ws=None), INVALID),
    (dict(x=None), INVALID), (dict(xs=None), INVALID), (dict(y=None), INVALID), (dict(wst=48), INVALID), (dict(xst=48), INVALID),
    (dict(yst=92), INVALID), (dict(wst=72), MISALIGNED), (dict(w=0x1000008), MISALIGNED), (dict(x=0x3000004), MISALIGNED),
    (dict(ws=0x2000002), MISALIGNED), (dict(y=0x5000002), MISALIGNED), (dict(yst=98), MISALIGNED), (dict(t=F16, y=0x5000001), MISALIGNED),
    (dict(r=0x6000000, rst=92), INVALID), (dict(r=0x6000002), MISALIGNED), (dict(r=0x6000000, rst=98), MISALIGNED),
    (dict(y=0x1000000), INVALID), (dict(y=0x4000000), INVALID), (dict(r=0x5000010, rst=96), INVALID), (dict(r=0x5000000), INVALID),
    (dict(r=0x5000000, rst=96, t=F16, yst=96), INVALID),
    (dict(wk=BIG, wkb=256, **SPLIT), WORKSPACE), (dict(wk=BIG + 16, wkb=1 << 30, **SPLIT), MISALIGNED),
    (dict(wk=0x5000100, wkb=1 << 30, **SPLIT), INVALID),
])
def test_product_refusals(kw, want):
    assert product(**kw) == want


def test_product_workspace():
    size = dc.mul_mat_i8_workspace_size
    assert size(1, 9728, 2560) == 0 and size(2048, 8192, 2048) == 0 and size(0, 1, 16) == 0 and size(1, 1, 24) == 0
    need = size(100, 2560, 9728)
    assert need > 0 and need % (100 * 2560 * 4) < 256  # whole planes
    if NO_GPU:
        assert product() == NO_DEVICE and product(r=0x5000000, rst=96) == NO_DEVICE
        assert product(**SPLIT) == NO_DEVICE and product(wk=BIG, wkb=need, **SPLIT) == NO_DEVICE


def route(t=F32, x=0x100000, xs=None, m=4, e=64, sc=0, bias=None, g=1, kept=1, best=1, k=8, scale=1.0, ids=0x200000, wt=0x300000):
    return dc.lib().dcq_moe_route(t, x, e * (2 if t == F16 else 4) if xs is None else xs, m, e, sc, bias, g, kept, best, k, 1, scale, ids,
                                  wt, None)


@pytest.mark.parametrize("kw,want", [
    (dict(t=8), UNSUPPORTED), (dict(sc=2), UNSUPPORTED), (dict(m=0), BAD_SHAPE), (dict(e=0), BAD_SHAPE), (dict(e=513), BAD_SHAPE),
    (dict(k=0), BAD_SHAPE), (dict(k=65), BAD_SHAPE), (dict(e=4, k=5), BAD_SHAPE), (dict(g=0), BAD_SHAPE), (dict(g=3), BAD_SHAPE),
    (dict(e=130, g=65), BAD_SHAPE), (dict(g=4, kept=5), BAD_SHAPE), (dict(kept=0), BAD_SHAPE), (dict(best=0), BAD_SHAPE),
    (dict(best=3), BAD_SHAPE), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(x=None), INVALID),
    (dict(ids=None), INVALID), (dict(wt=None), INVALID), (dict(xs=128), INVALID), (dict(xs=258), MISALIGNED), (dict(x=0x100002), MISALIGNED),
    (dict(bias=0x400002), MISALIGNED), (dict(ids=0x200001), MISALIGNED), (dict(ids=0x100000), INVALID), (dict(wt=0x200010), INVALID),
    (dict(bias=0x300000), INVALID),
])
def test_route_refusals(kw, want):
    assert route(**kw) == want


def plan(ids=0x100000, m=4, k=2, e=8, p=BIG, size=1 << 20):
    return dc.lib().dcq_moe_plan(ids, m, k, e, p, size, None)


@pytest.mark.parametrize("kw,want", [
    (dict(m=0), BAD_SHAPE), (dict(k=0), BAD_SHAPE), (dict(e=0), BAD_SHAPE), (dict(e=513), BAD_SHAPE), (dict(m=1 << 22), BAD_SHAPE),
    (dict(k=513), BAD_SHAPE), (dict(ids=None), INVALID), (dict(p=None), INVALID), (dict(size=256), WORKSPACE), (dict(ids=0x100002), MISALIGNED),
    (dict(p=BIG + 16), MISALIGNED), (dict(ids=BIG + 64), INVALID),
])
def test_plan_refusals(kw, want):
    assert plan(**kw) == want


def up(p=BIG, size=1 << 20, m=4, k=2, e=8, wg=0x1000000, wgs=0x1800000, wu=0x2000000, wus=0x2800000, n=32, width=64, row=None, per=None,
       x=0x3000000, xs=0x3800000, xst=None, t=F32, h=0x4000000, hst=None):
    row = width if row is None else row
    return dc.lib().dcq_moe_gate_up_i8(p, size, m, k, e, wg, wgs, wu, wus, n, width, row, row * n if per is None else per, x, xs,
                                       width if xst is None else xst, t, h, n * (2 if t == F16 else 4) if hst is None else hst, None)


@pytest.mark.parametrize("kw,want", [
    (dict(t=8), UNSUPPORTED), (dict(m=0), BAD_SHAPE), (dict(e=600), BAD_SHAPE), (dict(n=0), BAD_SHAPE), (dict(n=131073), BAD_SHAPE),
    (dict(width=40), BAD_SHAPE), (dict(m=1 << 20, k=2, n=1024, size=1 << 40), BAD_SHAPE), (dict(m=1 << 20, xst=8192, n=16, size=1 << 40), BAD_SHAPE),
    (dict(p=None), INVALID), (dict(size=512), WORKSPACE), (dict(p=BIG + 16), MISALIGNED), (dict(wg=None), INVALID), (dict(wu=None), INVALID),
    (dict(wgs=None), INVALID), (dict(wus=None), INVALID), (dict(x=None), INVALID), (dict(xs=None), INVALID), (dict(h=None), INVALID),
    (dict(row=48), INVALID), (dict(per=1024), INVALID), (dict(row=72), MISALIGNED), (dict(per=2056), MISALIGNED), (dict(xst=72), MISALIGNED),
    (dict(hst=126), INVALID), (dict(hst=130), MISALIGNED), (dict(wgs=0x1800002), MISALIGNED), (dict(h=0x1000000), INVALID),
    (dict(h=BIG), INVALID), (dict(h=0x3800000), INVALID),
])
def test_gate_up_refusals(kw, want):
    assert up(**kw) == want


def down(p=BIG, size=1 << 20, m=4, k=2, e=8, w=0x1000000, ws=0x1800000, n=32, width=64, row=None, per=None, h=0x3000000, hs=0x3800000,
         hst=None, wt=0x3900000, r=None, rst=0, t=F32, y=0x4000000, yst=None, wk=2 * BIG, wkb=1 << 30):
    row = width if row is None else row
    return dc.lib().dcq_moe_down_i8(p, size, m, k, e, w, ws, n, width, row, row * n if per is None else per, h, hs,
                                    width if hst is None else hst, wt, r, rst, t, y, n * (2 if t == F16 else 4) if yst is None else yst, wk,
                                    wkb, None)


@pytest.mark.parametrize("kw,want", [
    (dict(t=2), UNSUPPORTED), (dict(k=0), BAD_SHAPE), (dict(width=8), BAD_SHAPE), (dict(n=131073), BAD_SHAPE), (dict(p=None), INVALID),
    (dict(w=None), INVALID), (dict(ws=None), INVALID), (dict(h=None), INVALID), (dict(hs=None), INVALID), (dict(wt=None), INVALID),
    (dict(y=None), INVALID), (dict(wk=None), WORKSPACE), (dict(wkb=512), WORKSPACE), (dict(wk=2 * BIG + 8), MISALIGNED),
    (dict(r=0x5000000, rst=64), INVALID), (dict(r=0x5000002, rst=128), MISALIGNED), (dict(r=0x4000010, rst=128), INVALID),
    (dict(y=0x3900000), INVALID), (dict(y=2 * BIG), INVALID), (dict(wk=BIG), INVALID), (dict(wt=0x3900002), MISALIGNED),
    (dict(r=0x4000000, rst=128, t=F16, yst=128), INVALID),
])
def test_down_refusals(kw, want):
    assert down(**kw) == want


@pytest.mark.skipif(not NO_GPU, reason="asks for the refusal of a missing device")
def test_valid_calls_reach_the_device_check():
    assert quantize() == quantize(t=F16) == norm() == norm(r=None, h=None) == norm(h=0x200000) == norm(q=None, s=None, y=0x700000, ys=256) == \
        norm(t=F16) == route() == route(t=F16, sc=1, bias=0x400000, g=8, kept=4, best=2) == plan() == up() == up(t=F16) == down() == \
        down(r=0x4000000, rst=128) == NO_DEVICE


def test_sizes():
    assert dc.moe_plan_size(0, 8, 128) == 0 and dc.moe_plan_size(5, 8, 513) == 0
    # offsets, order and experts in rows of 64 numbers, then 16 bytes for each tile: 40 slots in tiles of 16 of 129 groups
    assert dc.moe_plan_size(5, 8, 128) == 4 * (192 + 64 + 64) + 16 * ((40 + 129 * 15) // 16)
    assert dc.moe_down_i8_workspace_size(5, 8, 100) == 16128 and dc.moe_down_i8_workspace_size(5, 8, 1 << 18) == 0


# ---------------------------------------------------------------- the binding's own checks (CPU tensors: refused)
def test_binding_refuses_what_is_not_on_the_gpu():
    x, q, s = torch.zeros((2, 32)), torch.zeros((2, 32), dtype=torch.int8), torch.zeros(2)
    for call in (lambda: dc.quantize_i8(x), lambda: dc.quantize_i8(x.double()), lambda: dc.quantize_i8([1.0]),
                 lambda: dc.rms_norm_i8(x, s, 1e-6, q=q, s=s), lambda: dc.rms_norm(x, s, 1e-6, y=x), lambda: dc.mul_mat_i8(q, s, q, s),
                 lambda: dc.mul_mat_i8(x, s, q, s), lambda: dc.moe_route(x, 2), lambda: dc.moe_plan(s, 4),
                 lambda: dc.moe_gate_up_i8(q, q, s, q, s, q, s, 2), lambda: dc.moe_down_i8(q, q, s, q, s, x)):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- the oracle's own properties
def test_oracle_quantize():
    x = np.array([[1.0, -2.0, 0.5, 127.0], [0, 0, 0, 0], [1, 2, np.inf, 0], [-254.0, 1.0, 3.0, 5.0]])
    q, s = I.quantize(x)
    assert q.tolist() == [[1, -2, 0, 127], [0, 0, 0, 0], [0, 0, 0, 0], [-127, 0, 2, 2]]  # 0.5, 1.5, 2.5: halves to even
    assert s[0] == 1 and s[1] == 0 and np.isnan(s[2]) and s[3] == 2
    big = np.random.default_rng(0).standard_normal((50, 200))
    q, s = I.quantize(big)
    assert (np.abs(big - q * s[:, None].astype(np.float64)) <= s[:, None] * 0.5001).all() and (np.abs(q).max(1) == 127).all()


def test_oracle_norm_is_the_norm():
    r = np.random.default_rng(1)
    x, w, res = r.standard_normal((3, 64)).astype(np.float32), r.standard_normal(64).astype(np.float32), r.standard_normal((3, 64))
    h, q, s, y = I.rms_norm(x, w, 1e-5, res.astype(np.float32))
    want = torch.nn.functional.rms_norm(torch.from_numpy(h).double(), (64,), torch.from_numpy(w).double(), 1e-5).numpy()
    assert np.allclose(y, want, rtol=1e-7) and np.allclose(s, np.abs(want).max(1) / 127, rtol=1e-7)
    assert (np.abs(want - q * s[:, None]) <= 0.5001 * s[:, None]).all()


def test_oracle_route():
    x = np.log(np.array([[1.0, 2, 3, 4], [4, 4, 1, 1]]))
    ids, w = I.route(x, 2)
    assert ids.tolist() == [[3, 2], [0, 1]] and np.allclose(w, [[4 / 7, 3 / 7], [0.5, 0.5]])
    ids, w = I.route(x, 2, renorm=False, scale=10)
    assert np.allclose(w, [[4, 3], [4, 4]])
    ids, _ = I.route(x, 2, bias=np.array([5.0, 0, 0, 0]))  # the bias chooses, and has no part in the weights
    assert ids[0].tolist() == [0, 3]
    ids, _ = I.route(np.array([[0.0, 3, 2, 2]]), 2, scoring="sigmoid", n_group=2, topk_group=1, group_best=2)
    assert ids.tolist() == [[2, 3]]
    ids, _ = I.route(np.array([[0.0, 3, 2, 2]]), 2, scoring="sigmoid", n_group=2, topk_group=1, group_best=1)
    assert ids.tolist() == [[1, 0]]
    ids, w = I.route(np.array([[-np.inf, 1.0, -np.inf, -np.inf]]), 2)
    assert ids.tolist() == [[1, -1]] and w.tolist() == [[1, 0]]


def test_oracle_experts():
    r = np.random.default_rng(2)
    w, ws = r.integers(-127, 128, (2, 3, 16), dtype=np.int8), r.uniform(0.1, 1, (2, 3))
    x, xs = r.integers(-127, 128, (2, 16), dtype=np.int8), r.uniform(0.001, 0.01, 2)
    ids = np.array([[1, -1], [0, 0]])
    h, gate, _ = I.gate_up(ids, 2, w, ws, w, ws, x, xs)
    full = np.einsum("enk,en,mk,m->men", w.astype(float), ws, x.astype(float), xs)
    assert np.allclose(gate, [full[0, 1], 0 * full[0, 0], full[1, 0], full[1, 0]])
    assert np.allclose(h, gate ** 2 / (1 + np.exp(-gate)))
    y, _ = I.down(ids, 2, w, ws, x[[0, 0, 1, 1]], xs[[0, 0, 1, 1]], np.array([[0.5, np.nan], [1, 2]]))
    assert np.allclose(y, [0.5 * full[0, 1], 3 * full[1, 0]])
