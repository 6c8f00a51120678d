"""The gated recurrence where it can go wrong beside test_gated_recurrence.py's cases."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from cpu_mamba_b200 import ops
from test_gated_recurrence import BF16, F32, call, close, make, reference

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
