"""The gated recurrence where it can go wrong beside test_gated_recurrence.py's cases."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from cpu_mamba_b200 import _lib, ops
from test_gated_recurrence import BF16, F32, HALF, U, call, close, make, reference

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [12, 150])
def test_low_input_gates(dtype, T):
    """Input gates whose sigmoids are small but normal numbers, from a zero state: the
    prompt, its gradients and single tokens to the relative bounds of other gates."""
    case = {"B": 3, "T": T, "D": 64, "dtype": dtype}
    st = make(case)
    g = torch.Generator().manual_seed(T)
    st["i"] = (-40 - 46 * torch.rand(3, T, 64, generator=g)).to(dtype).cuda()
    want, tol = reference(case, st)
    for k, v in call(st, grad=True).items():
        close(k, v, want[k], tol[k], case)
    state = torch.zeros(3, 64, device="cuda")
    for t in range(T):
        h = ops.gated_recurrence_step(st["x"][:, t], st["i"][:, t], st["r"][:, t], st["decay"],
                                      state)
        close("step", h, want["h"][:, t], tol["h"][:, t], case)
    close("state", state, want["last"], tol["last"], case)
    assert float(state.abs().max()) > 1e-25              # none of it is what 1e-37 lets pass


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_low_input_gates_among_others(dtype):
    """Some low gates, in other warps' tokens and beside other channels: the same bounds, and
    channels and tokens that do not see them keep their bits."""
    case = {"B": 2, "T": 400, "D": 72, "dtype": dtype, "state": True}
    st = make(case)
    clean = call(st)
    st["i"][0, 100:300:7, 5], st["i"][1, 250, 70] = -60.0, -80.0
    want, tol = reference(case, st)
    got = call(st, grad=True)
    for k, v in got.items():
        close(k, v, want[k], tol[k], case)
    same = torch.ones(2, 400, 72, dtype=torch.bool)
    same[0, 100:, 5], same[1, 250:, 70] = False, False
    assert torch.equal(got["h"][same], clean["h"][same])


@pytest.mark.parametrize("which", ["x", "input_gate", "decay_gate", "decay", "initial_state"])
def test_forward_mode_is_refused(which):
    """A dual tensor's tangent is not dropped: the call is refused, without gradients too."""
    v = {"x": torch.zeros(1, 2, 4), "input_gate": torch.zeros(1, 2, 4),
         "decay_gate": torch.zeros(1, 2, 4), "decay": torch.zeros(4),
         "initial_state": torch.zeros(1, 4)}
    with fwd.dual_level():
        v[which] = fwd.make_dual(v[which], torch.ones_like(v[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_recurrence(**v)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_recurrence(**v)


@gpu
def test_other_tensors_of_a_dual_level():
    """A call that has no dual tensor among its own runs as always."""
    x = torch.randn(1, 5, 8, device="cuda")
    want = ops.gated_recurrence(x, x, x, x[0, 0])
    with fwd.dual_level():
        fwd.make_dual(torch.ones(2), torch.ones(2))
        assert torch.equal(ops.gated_recurrence(x, x, x, x[0, 0]), want)


@gpu
def test_dual_gradients_are_refused():
    x = torch.randn(1, 5, 8, device="cuda", requires_grad=True)
    v = x.detach()
    h, last = ops.gated_recurrence(x, v, v, v[0, 0], return_final_state=True)
    with fwd.dual_level():
        for y in (h, last):
            dy = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, [x], [dy], retain_graph=True)


def relative(got, want, rel):
    """got within rel of want, and its rounding, all of one sign."""
    d = (got.double().cpu() - want).abs()
    ok = d <= (rel + HALF[got.dtype] * (1 + rel)) * want.abs() + 1e-37
    assert bool(ok.all()), float((d / want.abs()).max())


def sharper(v):
    """sigmoid(-v) over 1 - sigmoid(v) in 64 bits, which is off by up to 1e-3 at v = 30."""
    v = v.double().cpu()
    return torch.sigmoid(-v) / (1 - torch.sigmoid(v))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 9, 200])
def test_gradients_of_open_gates(dtype, T):
    """Gates at 12 .. 30, whose 1 - sigmoid is 6e-6 .. 9e-14: the gates' gradients have that
    as a factor, to its own few units.  Inputs of one sign, so that nothing cancels: u = 2^-24,
    a sigmoid and 1 - sigmoid are off by 7 + 2 |v| units (the exponential's argument twice,
    the exponential 4, sum, reciprocal and product), 1 - a^2 by the same and 19 more, G and h
    by what a token's decay (8 units and |log a| times its own) and sum (2) add up to."""
    B, D = 3, 64
    g = torch.Generator().manual_seed(T)

    def rand(*s):
        return torch.rand(*s, generator=g).to(dtype).cuda()

    case = {"B": B, "T": T, "D": D, "dtype": dtype, "state": True}
    st = make(case)
    high = (12 + 18 * torch.rand(B, T, D, generator=g)).to(dtype).cuda()
    gate = 67 * U                                        # 7 + 2 * 30
    # |log a| <= 0.11, so ea <= 0.11 (gate + 11 U) + 8 U; eb: half of y's, input gate's, 8
    token = 0.11 * (gate + 11 * U) + 10 * U
    eb = 0.5 * (gate + 19 * U) + gate + 8 * U
    # dinput_gate = G m i x (1 - i): x and dh positive
    for r in (st["r"], high):
        s = {**st, "x": rand(B, T, D) + 0.5, "dh": rand(B, T, D) + 0.5, "i": high, "r": r,
             "dlast": st["dlast"].abs()}
        want, _ = reference(case, s)
        # (an r at -5 multiplies |log a| by less, so that the same bounds hold)
        relative(call(s, grad=True)["di"], want["di"] * sharper(high),
                 T * token + eb + gate + 12 * U)
    # ddecay_gate = G r (a h - a^2 i x / m) log a (1 - r): h positive, x negative and small
    s = {**st, "x": -(rand(B, T, D) + 0.5) * 2.0 ** -40, "dh": rand(B, T, D) + 0.5, "r": high,
         "h0": (st["h0"].abs() + 1) * 1e3, "dlast": st["dlast"].abs()}
    want, _ = reference(case, s)
    relative(call(s, grad=True)["dr"], want["dr"] * sharper(high),
             2 * T * token + 2 * token + eb + 3 * gate + 40 * U)
    # open altogether
    s["i"], s["r"] = torch.full_like(high, math.inf), torch.full_like(high, math.inf)
    got = call(s, grad=True)
    assert bool((got["di"] == 0).all()) and bool((got["dr"] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_low_and_far_gates(dtype):
    """Both gates over the whole range at once, -100 .. 100, and closed and open ones: finite,
    within the reference's bounds wherever its own 64 bits tell 1 - sigmoid (gates below 12).
    Decay gates whose 1 - a^2 is below 2^-120 count as closed: m, below 2^-60, counts as 0 in
    h = .. + m i x, dx = G m i, dinput_gate = dx x (1 - i), and in ddecay_gate's G i x m / 2
    (r log a / m is -m / 2 there).  |x| and |dh| are below 6, so |G| below 6 (T + 1); with the
    sum over T tokens every output is off by less than 2^-60 36 (T + 1) T."""
    B, T, D = 2, 230, 64
    case = {"B": B, "T": T, "D": D, "dtype": dtype, "state": True}
    st = make(case)
    assert all(float(st[k].abs().max()) < 6 for k in ("x", "dh", "dlast"))
    closed = 2.0 ** -60 * 36 * (T + 1) * T
    g = torch.Generator().manual_seed(3)
    far = 200 * torch.rand(2, B, T, D, generator=g) - 100
    far[:, :, ::50], far[:, :, 1::50] = math.inf, -math.inf
    # (from -80 to -100 sigmoids leave the normal numbers, where they count as 0)
    far = torch.where((far < -80) & (far > -100), -80.0, far).to(dtype).cuda()
    st["i"], st["r"] = far[0], far[1]
    got = call(st, grad=True)
    want, tol = reference(case, st)
    for k, v in got.items():
        assert bool(v.isfinite().all()), k
    for k in ("h", "last", "dh0", "dx"):
        close(k, got[k], want[k], tol[k] + closed, case)
    low = ((far[0] < 12) & (far[1] < 12)).cpu()
    for k in ("di", "dr"):
        close(k, got[k][low.cuda()], want[k][low], tol[k][low] + closed, case)


@gpu
def test_states_advanced_in_place_are_seen_by_autograd():
    """A state that a backward pass still needs and a step has advanced: an error, as for
    torch's own operations in place, and no gradient of the wrong state."""
    x = torch.randn(1, 5, 8, device="cuda")
    decay = torch.full((8,), -5.0, device="cuda", requires_grad=True)
    state = torch.randn(1, 8, device="cuda")
    h = ops.gated_recurrence(x, x, x, decay, initial_state=state)
    version = state._version
    ops.gated_recurrence_step(x[:, 0], x[:, 0], x[:, 0], decay.detach(), state)
    assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h.sum(), [decay])
    with torch.inference_mode():                          # (these have no versions)
        state = torch.zeros(1, 8, device="cuda")
    ops.gated_recurrence_step(x[:, 0], x[:, 0], x[:, 0], decay.detach(), state)


@gpu
def test_other_tensors_written_in_place_are_seen_by_autograd():
    w = torch.randn(3, 40, device="cuda", requires_grad=True)
    p = torch.sigmoid(w)                                  # keeps its output for the gradient
    z = p.detach()
    assert ops.adjust_logits(z, temperature=2.0, out=z) is z
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        p.sum().backward()
    p = torch.sigmoid(w)
    ops.adjust_logits(p.detach(), temperature=2.0)        # a new tensor: p is as it was
    p.sum().backward()
    p = torch.sigmoid(w)
    ops.reorder_states([p.detach()], torch.tensor([[2, 1, 0]], device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        p.sum().backward()


# Calls of many tiles: each CTA takes several, across sequences, strips and batch rows
def check_channels(case, st, channels, got):
    """The outputs of some channels (they do not touch) against the reference's."""
    part = {k: v if v is None or k == "cu" else v[..., channels].contiguous()
            for k, v in st.items()}
    want, tol = reference({**case, "D": len(channels)}, part)
    for k, v in got.items():
        close(k, v[..., channels], want[k], tol[k], case)


@gpu
@pytest.mark.parametrize("D", [1536, 1537])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_tiles_than_ctas(dtype, D):
    """2 x 1500 tokens are 30 tiles of 104 and more of fewer in 24 or 25 strips: from 720 to
    1900 for 296 CTAs.  Dense, and as a pack of ragged sequences with rows of none."""
    channels = [0, 1, 31, 32, 63, 64, 700, 767, 768, 1471, 1472, 1535, D - 1]
    case = {"B": 2, "T": 1500, "D": D, "dtype": dtype, "state": True}
    st = make(case)
    check_channels(case, st, channels, call(st, grad=True))
    case = {"B": 1, "T": 3000, "D": D, "dtype": dtype, "state": True,
            "cu": [3, 700, 700, 1801, 1802, 2900, 2990]}
    st = make(case)
    check_channels(case, st, channels, call(st, grad=True))
    assert _lib.device_status() == 0


@gpu
@pytest.mark.parametrize("off", [-1, 0, 1])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 128), (BF16, 64), (BF16, 136)])
def test_packs_of_whole_tiles(dtype, D, off):
    """Rows of 16-byte chunks and sequences of several tiles, so that most tiles need no marks;
    they end at, one before and one behind the ends of tiles (104, 64, 56 and 40 tokens), tiles
    begin with a sequence, end with one and hold several."""
    cu = [0, 312 + off, 448 + off, 704 + off, 705 + off, 1064 + off, 1200 + off, 1664 + off, 1900]
    for first, behind in ((0, 0), (5, 70)):
        case = {"B": 1, "T": 1900 + behind, "D": D, "dtype": dtype, "state": True,
                "cu": [first] + cu[1:]}
        st = make(case)
        want, tol = reference(case, st)
        for k, v in call(st, grad=True).items():
            close(k, v, want[k], tol[k], case)


@gpu
@pytest.mark.parametrize("dtype,limit", [(F32, 1 << 21), (BF16, 1 << 22)])
def test_strides_around_the_limit_of_short_offsets(dtype, limit):
    """Token strides at which a tile's offsets (up to 104 rows) still fit 32 bits, and at which
    they no longer do; the last rows are more than 2^31 elements away."""
    T, D = 1100 if dtype == F32 else 600, 64
    case = {"B": 1, "T": T, "D": D, "dtype": dtype, "state": True}
    st = make(case)
    want = call(st, grad=True)
    store = torch.empty(T * limit, dtype=dtype, device="cuda")
    assert (T - 1) * (limit - 8) > 1 << 31
    for stride in (limit - 8, limit):
        far = store.as_strided((1, T, D), (0, stride, 1))
        for name in ("x", "i", "dh"):
            far.copy_(st[name])
            got = call({**st, name: far}, grad=True)
            assert all(torch.equal(got[k], want[k]) for k in want), (stride, name)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_past_32_bits(dtype):
    """Few tokens, and batch rows, more than 2^31 elements apart from first to last."""
    far = (1 << 30) + 64
    store = torch.empty(2 * far + 4096, dtype=dtype, device="cuda")
    for B, T, strides in ((1, 3, (0, far, 1)), (3, 1, (far, 64, 1)), (3, 60, (far, 64, 1))):
        case = {"B": B, "T": T, "D": 64, "dtype": dtype, "state": True}
        st = make(case)
        want = call(st, grad=True)
        view = store.as_strided((B, T, 64), strides)
        for name in ("x", "i", "r", "dh"):
            view.copy_(st[name])
            got = call({**st, name: view}, grad=True)
            assert all(torch.equal(got[k], want[k]) for k in want), (B, T, name)


# batches of which a CTA takes several sequences, the last ones unevenly
@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,D", [(2400, 64), (2500, 75), (5001, 4), (700, 2048), (301, 4098)])
def test_step_of_many_sequences(dtype, B, D):
    """Two steps against the formula: bounds as reference's, for all sequences at once."""
    g = torch.Generator().manual_seed(B + D)

    def rand(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).to(dtype).cuda()

    x, i, r = rand(2, B, D), rand(2, B, D, scale=1.5), rand(2, B, D, scale=1.5)
    decay = (torch.rand(D, generator=g) * 3 - 6).cuda()
    state = torch.randn(B, D, generator=g).cuda()
    want = state.double()
    e = torch.zeros_like(want)
    for t in range(2):
        h = ops.gated_recurrence_step(x[t], i[t], r[t], decay, state)
        vr, vi = r[t].double(), i[t].double()
        la = -8 * torch.nn.functional.softplus(decay.double()) * torch.sigmoid(vr)
        a = torch.exp(la)
        b = (-torch.expm1(2 * la)).sqrt() * torch.sigmoid(vi) * x[t].double()
        er, ei = (7 + 2 * vr.abs()) * U, (7 + 2 * vi.abs()) * U
        eg = er + 11 * U
        size = (a * want).abs() + b.abs()
        e = (a * e + (la.abs() * eg + 8 * U) * (a * want).abs()
             + (0.5 * (eg + 8 * U) + ei + 8 * U) * b.abs() + 2 * U * size)
        want = a * want + b
        assert bool(((state.double() - want).abs() <= e + 1e-37).all())
        assert bool(((h.double() - want).abs() <= e + HALF[dtype] * (want.abs() + e)).all())
