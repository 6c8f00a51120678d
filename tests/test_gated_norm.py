"""gated_norm: RMSNorm and SiLU gate after a block, scaled residual add and the
next block's RMSNorm, against the formulas in 64 bits; refusals on the CPU."""
import ctypes
import itertools

import pytest
import torch

from cpu_mamba_b200 import _lib, ops

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def reference(x, gate, weight, residual, scale, nxt, eps, group, before):
    """(u or r, n) in 64 bits, and the size of r's two terms."""
    u = x.double()
    act = None if gate is None else torch.nn.functional.silu(gate.double())

    def rms(t, width):
        t = t.unflatten(-1, (-1, width))
        return (t / (t.pow(2).mean(-1, keepdim=True) + eps).sqrt()).flatten(-2)

    if act is not None and not before:
        u = u * act
    if weight is not None:
        u = rms(u, group or x.shape[-1]) * weight.double()
    if act is not None and before:
        u = u * act
    if residual is None:
        return u, None, u.abs()
    s = scale.double() if torch.is_tensor(scale) else (1.0 if scale is None else scale)
    r = residual.double() + s * u
    n = None if nxt is None else rms(r, x.shape[-1]) * nxt.double()
    return r, n, residual.double().abs() + (s * u).abs()


def run_case(rows, W, dtype, rdtype, gate, weight, residual, scale, nxt, group, before, seed=0):
    g = torch.Generator().manual_seed(seed + rows + W)

    def rand(*shape, dt=dtype):
        return torch.randn(*shape, generator=g).to(dt)

    x = rand(rows, W) * 3
    z = rand(rows, W) if gate else None
    w = rand(W) if weight else None
    res = rand(rows, W, dt=rdtype) if residual else None
    sc = (rand(W) if scale == "vector" else scale) if residual else None
    nw = rand(W, dt=F32) if nxt and residual else None
    cuda = [t.cuda() if torch.is_tensor(t) else t for t in (x, z, w, res, sc, nw)]
    got = ops.gated_norm(cuda[0], gate=cuda[1], weight=cuda[2], residual=cuda[3],
                         residual_scale=cuda[4], next_weight=cuda[5], eps=1e-4, group_size=group,
                         norm_before_gate=before)
    want = reference(x, z, w, res, sc, nw, 1e-4, group, before)
    first, second = got if nw is not None else (got, None)
    half = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
    # fp32 arithmetic: a sum of W squares added in at most 16 + log2(W) + 16 levels
    # of rounding (halved by the root), SiLU within 4 + |z| units, ten products:
    # 64 units of 2^-24 of the terms' sizes; then one rounding to the output's type
    unit = 64 * 2.0 ** -24
    d = (first.double().cpu() - want[0]).abs()
    assert first.dtype == (rdtype if residual else dtype)
    assert bool((d <= unit * want[2] + half[first.dtype] * want[0].abs() + 1e-30).all()), d.max()
    if second is not None:
        # n inherits r's error, relative to the row: unit * the terms' sizes / rms(r)
        rms = (want[0].pow(2).mean(-1, keepdim=True) + 1e-4).sqrt()
        d = (second.double().cpu() - want[1]).abs()
        tol = 2 * unit * (want[2] / rms * nw.double().abs() + want[1].abs())
        assert second.dtype == dtype
        assert bool((d <= tol + half[dtype] * want[1].abs() + 1e-30).all()), d.max()


@gpu
@pytest.mark.parametrize("rows,W,group", [(1, 1, None), (3, 17, None), (5, 96, 32), (2, 100, 10),
                                          (64, 1024, None), (7, 1536, 64), (3, 4096, 512),
                                          (2, 16384, None), (2, 6000, 2000), (9, 768, 96),
                                          (3, 5000, None), (2, 16383, None), (4, 1029, 3)])
@pytest.mark.parametrize("dtype,rdtype", [(F32, F32), (BF16, BF16), (BF16, F32)])
def test_all_parts(rows, W, group, dtype, rdtype):
    for before in (True, False):
        run_case(rows, W, dtype, rdtype, True, True, True, "vector", True, group, before)


@gpu
@pytest.mark.parametrize("rows,W", [(2500, 64), (2401, 768), (2369, 17), (2400, 1000), (2400, 96)])
@pytest.mark.parametrize("dtype,rdtype", [(F32, F32), (BF16, F32)])
def test_many_rows(rows, W, dtype, rdtype):
    run_case(rows, W, dtype, rdtype, True, True, True, 0.5, True, None, True)
    run_case(rows, W, dtype, rdtype, True, True, False, None, False, 8 if W % 8 == 0 else None,
             False)
    if W % 24 == 0:
        run_case(rows, W, dtype, rdtype, False, True, True, None, True, 24, True)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_combination_of_parts(dtype):
    for gate, weight, residual, nxt in itertools.product((False, True), repeat=4):
        run_case(4, 256, dtype, dtype, gate, weight, residual, 0.25 if residual else None,
                 nxt, None, False)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_in_place_and_graph(dtype):
    """Halves of one projection's rows, the residual updated in place, a replay."""
    g = torch.Generator().manual_seed(3)
    xz = torch.randn(2, 50, 2 * 256, generator=g).to(dtype).cuda()
    x, z = xz[..., :256], xz[..., 256:]
    w = torch.rand(256, generator=g).cuda()
    want = ops.gated_norm(x.contiguous(), gate=z.contiguous(), weight=w)
    assert torch.equal(ops.gated_norm(x, gate=z, weight=w), want)
    assert torch.equal(ops.gated_norm(x.transpose(0, 1), gate=z.transpose(0, 1), weight=w),
                       want.transpose(0, 1))
    off = torch.randn(50 * 257 + 1, generator=g).to(dtype).cuda()[1:].reshape(50, 257)[:, :256]
    a = ops.gated_norm(off, weight=w)
    b = ops.gated_norm(off.contiguous(), weight=w)      # other tiles, other order of the sum
    assert (a.float() - b.float()).abs().max() <= (1e-5 if dtype == F32 else 2 ** -7) * b.abs().max()
    res = torch.randn(2, 50, 256, generator=g).cuda()
    r, n = ops.gated_norm(x, gate=z, weight=w, residual=res, next_weight=w)
    mine = res.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r2, n2 = ops.gated_norm(x, gate=z, weight=w, residual=mine, next_weight=w, out=mine)
    assert r2.data_ptr() == mine.data_ptr()
    graph.replay()
    assert torch.equal(mine, r) and torch.equal(n2, n)


@gpu
def test_zero_rows_and_zero_row():
    x = torch.zeros(3, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    assert bool((ops.gated_norm(x, weight=w) == 0).all())
    assert ops.gated_norm(x[:0], weight=w).shape == (0, 64)


@gpu
def test_torch_ops():
    x, z = torch.randn(2, 4, 96, device="cuda").unbind(0)
    w = torch.rand(96, device="cuda")
    assert torch.equal(torch.ops.mamba_b200.gated_norm(x, z, w, 32), ops.gated_norm(
        x, gate=z, weight=w, group_size=32))
    r, n = torch.ops.mamba_b200.gated_norm_residual(x, z, w, x, None, w)
    r2, n2 = ops.gated_norm(x, gate=z, weight=w, residual=x, next_weight=w)
    assert torch.equal(r, r2) and torch.equal(n, n2)


@gpu
def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    w = torch.rand(64, device="cuda")
    f = ops.gated_norm
    bad = [lambda: f(x, weight=w[:63]), lambda: f(x, gate=x[:3]), lambda: f(x, gate=x.bfloat16()),
           lambda: f(x, weight=w.bfloat16()), lambda: f(x, weight=w.double()),
           lambda: f(x, weight=w, group_size=7), lambda: f(x, weight=w, group_size=0),
           lambda: f(x, next_weight=w), lambda: f(x, residual_scale=2.0),
           lambda: f(x, residual=x.bfloat16()), lambda: f(x, residual=x[:2]),
           lambda: f(x, weight=w, out=x.bfloat16()), lambda: f(x, weight=w, out=x.t()),
           lambda: f(x, weight=w.cpu()), lambda: f(x[0, 0], weight=w)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        f(x.double(), weight=w)
    with pytest.raises(RuntimeError, match="16384"):
        f(torch.zeros(1, 16385, device="cuda"))


@pytest.mark.parametrize("kw,code", [({"dtype": 4}, 1), ({"dtype": 0, "residual_dtype": 1}, 1),
                                     ({"rows": -1}, 2), ({"width": 0}, 2), ({"width": 16385}, 2),
                                     ({"group": 5}, 2), ({}, 1), ({"x": 16, "out": 16,
                                                                  "next_weight": 16}, 1)])
def test_c_entry_refuses(kw, code):
    d = _lib.GatedNorm()
    d.rows, d.width = 2, 64
    for n, v in kw.items():
        setattr(d, n, v)
    assert _lib.lib().mb2_gated_norm(ctypes.byref(d), None) == code
    assert b"gated_norm" in _lib.lib().mb2_last_error()


def test_c_entry_nothing_to_do_and_cpu_tensors():
    d = _lib.GatedNorm()
    d.width = 8
    assert _lib.lib().mb2_gated_norm(ctypes.byref(d), None) == 0
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_norm(torch.zeros(2, 8))
