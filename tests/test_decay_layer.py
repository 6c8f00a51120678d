"""The operators as a model would use them together: a layer that projects, runs
decay attention, norms and gates its heads, projects back and adds the residual
with the next norm -- over a prompt and then token by token -- and beam search
over its states, against the same layer in 64 bits token by token."""
import pytest
import torch

from cpu_mamba_b200 import ops

pytestmark = pytest.mark.gpu


class Layer:
    """One residual layer of H heads (dk x dv) on width D; states (B, H, dk, dv)."""

    def __init__(self, D, H, dk, dv, dtype, seed):
        r = torch.Generator().manual_seed(seed)

        def w(*s):
            return (torch.randn(*s, generator=r) * s[-1] ** -0.5).to(dtype)

        self.H, self.dk, self.dv = H, dk, dv
        self.qkvz = w(2 * dk + 2 * H * dv, D)
        self.out = w(D, H * dv)
        self.norm = (torch.rand(H * dv, generator=r) + 0.5).to(dtype)
        self.next = (torch.rand(D, generator=r) + 0.5).to(dtype)
        self.scale = (torch.rand(D, generator=r) + 0.5).to(dtype)
        self.g = torch.log1p(-torch.exp2(-3.0 - torch.arange(H).float()))

    def cuda(self):
        for n, t in list(vars(self).items()):
            if torch.is_tensor(t):
                setattr(self, n, t.cuda())
        return self

    def split(self, p):
        dk, n = self.dk, self.H * self.dv
        return (p[..., :dk].unsqueeze(-2), p[..., dk:2 * dk].unsqueeze(-2),
                p[..., 2 * dk:2 * dk + n].unflatten(-1, (self.H, self.dv)), p[..., 2 * dk + n:])

    def after(self, o, z, x):
        u = ops.gated_norm(o.flatten(-2), gate=z, weight=self.norm, group_size=self.dv)
        return ops.gated_norm(ops.linear(u, self.out), residual=x, residual_scale=self.scale,
                              next_weight=self.next)

    def prompt(self, x):
        q, k, v, z = self.split(ops.linear(x, self.qkvz))
        o, state = ops.decay_attention(q, k, v, self.g, scale=self.dk ** -0.5,
                                       return_final_state=True)
        return *self.after(o, z, x), state

    def step(self, x, state):
        q, k, v, z = self.split(ops.linear(x, self.qkvz))
        o = ops.decay_attention_step(q, k, v, self.g, state, scale=self.dk ** -0.5)
        return self.after(o, z, x)

    def reference(self, x, state=None):
        """In 64 bits over (B, T, D): (residual, next norm, final state)."""
        d = torch.float64
        q, k, v, z = self.split(x.to(d) @ self.qkvz.to(d).t())
        B, T = x.shape[:2]
        s = torch.zeros(B, self.H, self.dk, self.dv, dtype=d) if state is None else state.to(d)
        a = self.g.to(d).exp().reshape(1, -1, 1, 1)
        outs = []
        for t in range(T):
            s = a * s + k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2)
            outs.append((q[:, t].unsqueeze(-1) * s).sum(-2) * self.dk ** -0.5)
        o = torch.stack(outs, 1)
        u = o / (o.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
        u = u.flatten(-2) * self.norm.to(d) * torch.nn.functional.silu(z)
        r = x.to(d) + self.scale.to(d) * (u @ self.out.to(d).t())
        n = r / (r.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * self.next.to(d)
        return r, n, s


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 0.04)])
def test_prompt_then_tokens_through_a_layer(dtype, tol):
    """fp32: sums of up to 192 products behind one another, 1e-6 each.  bf16: five
    roundings of 2^-8 of activations of size 1 to 4 on the way (projection, heads,
    norm, output, residual), added as a random walk: 2^-8 sqrt(5) 4 = 0.035."""
    D, H, dk, dv, B, T, n = 192, 3, 64, 64, 2, 150, 3
    cpu = Layer(D, H, dk, dv, dtype, seed=1)
    x = torch.randn(B, T + n, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    r_ref, n_ref, s_ref = cpu.reference(x)
    gpu = Layer(D, H, dk, dv, dtype, seed=1).cuda()
    xc = x.cuda()
    r, nx, state = gpu.prompt(xc[:, :T])
    rs, ns = [r], [nx]
    for t in range(T, T + n):
        r, nx = gpu.step(xc[:, t], state)
        rs.append(r.unsqueeze(1))
        ns.append(nx.unsqueeze(1))
    r, nx = torch.cat(rs, 1).double().cpu(), torch.cat(ns, 1).double().cpu()
    assert (r - r_ref).abs().max() <= tol and (nx - n_ref).abs().max() <= tol
    assert (state.double().cpu() - s_ref).abs().max() <= tol * s_ref.abs().max()


def test_beams_over_the_layer():
    """A beam search step by step: selection, states following their parents, the
    next token through the layer; the winning beam's own sequence run alone gives
    the same logits."""
    D, H, dk, dv, K, V = 64, 2, 32, 32, 3, 50
    layer = Layer(D, H, dk, dv, torch.float32, seed=3)
    E = torch.randn(V, D, generator=torch.Generator().manual_seed(4))
    prompt = torch.randn(1, 20, D, generator=torch.Generator().manual_seed(5))
    gpu = Layer(D, H, dk, dv, torch.float32, seed=3).cuda()
    Ec = E.cuda()
    _, nx, state = gpu.prompt(prompt.cuda())
    logits = nx[:, -1] @ Ec.t()
    scores, _, tok = ops.beam_select(logits.unsqueeze(1), torch.zeros(1, 1, device="cuda"), num=K)
    state = state.repeat_interleave(K, 0)
    history = [[t] for t in tok[0].tolist()]
    for _ in range(4):
        _, nx = gpu.step(Ec[tok.flatten()], state)
        logits = (nx @ Ec.t()).reshape(1, K, V)
        scores, par, tok = ops.beam_select(logits, scores)
        ops.reorder_states({"s": [state]}, par)
        history = [history[p] + [t] for p, t in zip(par[0].tolist(), tok[0].tolist())]
    total = 0.0
    seq = prompt
    for t in history[0]:
        _, n_ref, _ = layer.reference(seq)
        total += torch.log_softmax(n_ref[:, -1] @ E.double().t(), -1)[0, t].item()
        seq = torch.cat([seq, E[t][None, None]], 1)
    # five log probabilities of logits of size 8 sqrt(64) with 2e-5 each
    assert abs(total - scores[0, 0].item()) <= 5 * 2e-4 * 8
    _, _, s_ref = layer.reference(seq[:, :-1])
    assert (state[0].double().cpu() - s_ref[0]).abs().max() <= 2e-5 * s_ref.abs().max()
