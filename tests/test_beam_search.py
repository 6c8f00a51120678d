"""Beam search: the selection over beams and vocabulary against a 64-bit sort,
the in-place reordering of states against indexing, and the search itself (its
graph-captured loop over a MambaStack) against a plain search over whole
sequences; refusals on the CPU."""
import ctypes

import pytest
import torch

import oracle
from cpu_mamba_b200 import CPUMamba, MambaStack, _lib, ops
from cpu_mamba_b200.generate import BeamLoop, TiedEmbeddingSampler, beam_search

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def reference(logits, scores, num, finished=None, pad=0):
    """(all candidates' values (B, K V), the best num's flat indices): a stable
    sort in 64 bits.  A beam without a finite normaliser or score has none."""
    x = logits.double()
    x = torch.where(x.isnan().any(-1, keepdim=True), torch.nan, x)
    c = torch.log_softmax(x, -1) + scores.double()[..., None]
    if finished is not None:
        for b, k in finished.nonzero().tolist():
            c[b, k] = -torch.inf
            c[b, k, pad] = scores[b, k].double()
    c = torch.where(scores.isfinite()[..., None], c, -torch.inf)
    c = torch.where(c.isnan(), -torch.inf, c).flatten(1)
    return c, c.sort(dim=-1, descending=True, stable=True).indices[:, :num]


# fp32 exponentials (2 + 1.2 |x| units of 2^-23, weighted by e^-|x|: below 2^-21) in
# sums of at most 45 roundings on any path: 2^-21 + 45 2^-24 of the normaliser
LSE = 2.0 ** -21 + 45 * 2.0 ** -24


def check(logits, scores, num, finished=None, pad=0, exact=False):
    B, K, V = logits.shape
    c, want = reference(logits, scores, num, finished, pad)
    got = ops.beam_select(logits.cuda(), scores.cuda(), num=num, pad_token=pad,
                          finished=None if finished is None else finished.cuda())
    s, p, t = (x.cpu() for x in got)
    assert s.shape == p.shape == t.shape == (B, num)
    assert s.dtype == F32 and p.dtype == t.dtype == torch.int64
    flat = p * V + t
    assert bool(((p >= 0) & (p < K) & (t >= 0) & (t < V)).all())
    assert all(len(set(r)) == num for r in flat.tolist())
    best = c.gather(1, want)
    if exact:
        assert torch.equal(flat, want)
    # candidates nearer to one another than two normalisers' errors may change places
    mine = c.gather(1, flat)
    tie = (mine == best) | ((mine - best).abs() <= 2 * LSE)
    assert bool(tie.all())
    gap = torch.ones_like(best, dtype=torch.bool)
    gap[:, 1:] &= (best[:, :-1] - best[:, 1:]) > 2 * LSE
    gap[:, :-1] &= (best[:, :-1] - best[:, 1:]) > 2 * LSE
    nxt = c.sort(dim=-1, descending=True).values
    if nxt.shape[1] > num:
        gap[:, -1] &= (best[:, -1] - nxt[:, num]) > 2 * LSE
    assert bool((flat == want)[gap].all())
    ok = ((s.double() - mine).abs() <= LSE + 2.0 ** -24 * mine.abs()) | (s.double() == mine)
    assert bool(ok.all()), (s, mine)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,K,V,num", [(1, 1, 1, 1), (2, 3, 5, 15), (1, 2, 7, 4), (3, 4, 100, 8),
                                       (2, 5, 8191, 5), (2, 4, 8192, 8), (1, 3, 8200, 6),
                                       (2, 8, 50257, 16), (1, 32, 16400, 64), (1, 2, 131073, 33),
                                       (149, 4, 9001, 3), (150, 4, 17000, 12)])
def test_select(B, K, V, num, dtype):
    g = torch.Generator().manual_seed(V + K)
    logits = (torch.randn(B, K, V, generator=g) * 3).to(dtype)
    scores = -torch.rand(B, K, generator=g) * 4
    check(logits, scores, num)
    fin = torch.rand(B, K, generator=g) < 0.4
    check(logits, scores, num, fin, pad=V // 2)


@gpu
@pytest.mark.parametrize("K,V", [(29, 9000), (31, 9000), (32, 9000)])
def test_select_lists_around_the_shared_memory_limit(K, V):
    """58, 62 and 64 lists of 64 entries: 44776, 47864 and 49408 bytes staged."""
    g = torch.Generator().manual_seed(K)
    check(torch.randn(1, K, V, generator=g) * 3, torch.zeros(1, K), 64)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_ties_go_to_the_lowest_index(dtype):
    """All logits equal; logits on a coarse grid; equal beams."""
    flat = torch.zeros(2, 3, 20000, dtype=dtype)
    s = torch.tensor([[-1.0, -1.0, -0.5], [0.0, 0.0, 0.0]])
    check(flat, s, 20, exact=True)
    g = torch.Generator().manual_seed(1)
    grid = torch.randint(-3, 4, (2, 1, 9000), generator=g).to(dtype).expand(2, 4, 9000)
    check(grid, torch.full((2, 4), -2.0), 40, exact=True)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_masks(dtype):
    """Masked logits, a beam with nothing left, NaN and +inf rows, dead beams,
    all beams dead, fewer finite candidates than asked for."""
    inf = float("inf")
    g = torch.Generator().manual_seed(2)
    B, K, V = 6, 3, 10000
    x = torch.randn(B, K, V, generator=g).to(dtype)
    s = -torch.rand(B, K, generator=g)
    x[0, :, 7:] = -inf                        # 7 tokens left in each beam
    x[1, 0] = -inf                            # nothing left
    x[2, 1, 5000] = float("nan")
    x[3, 2, 9999] = inf
    s[4, 1:] = -inf                           # the first step of a search
    s[5] = -inf
    check(x, s, 30)
    x[:, :, 3:] = -inf
    check(x, s, 12)                           # at most 9 finite ones
    fin = torch.zeros(B, K, dtype=torch.bool)
    fin[:, 1] = True
    check(x, s, 12, fin, pad=2)
    check(x, s, 12, torch.ones_like(fin), pad=9999)
    check(torch.full((1, 2, 60000), -1e30, dtype=dtype), torch.zeros(1, 2), 5, exact=True)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_strides(dtype):
    """Rows that start off every 16-byte boundary, an expanded beam index."""
    g = torch.Generator().manual_seed(3)
    big = torch.randn(2, 3, 1003, generator=g).to(dtype).cuda()
    part = big[:, :, 1:1000]
    s = -torch.rand(2, 3, generator=g).cuda()
    a = ops.beam_select(part, s, num=6)
    b = ops.beam_select(part.contiguous(), s, num=6)
    for x, y in zip(a[1:], b[1:]):
        assert torch.equal(x, y)
    assert (a[0] - b[0]).abs().max() <= 2 * LSE
    row = big[:, 0].unsqueeze(1)
    s1 = torch.tensor([[0.0, -1.0, -1.0]] * 2)
    check(row.expand(2, 3, 1003).cpu(), s1, 5)
    e = ops.beam_select(row.expand(2, 3, 1003), s1.cuda(), num=5)
    f = ops.beam_select(row.expand(2, 3, 1003).contiguous(), s1.cuda(), num=5)
    assert all(torch.equal(x, y) for x, y in zip(e, f)) or (e[0] - f[0]).abs().max() <= 2 * LSE


@gpu
def test_select_graph_and_side_stream():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 4, 9000, generator=g).cuda()
    s = -torch.rand(2, 4, generator=g).cuda()
    want = ops.beam_select(x, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.beam_select(x, s)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for y in (x, x.flip(0).contiguous()):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, ops.beam_select(y, s), y))
    for gr, out, y in graphs * 2:
        for t in out:
            t.zero_()
        gr.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, ops.beam_select(y, s)))
    t = torch.ops.mamba_b200.beam_select(x, s, 4)
    assert all(torch.equal(a, b) for a, b in zip(want, t))


# -------------------------------------------------------------------- reorder
@gpu
@pytest.mark.parametrize("B,K", [(1, 1), (3, 2), (2, 4), (1, 7), (2, 13), (1, 32)])
def test_reorder(B, K):
    g = torch.Generator().manual_seed(K)
    shapes = [((17, 3), F32), ((64, 16), F32), ((33,), BF16), ((5,), torch.uint8),
              ((4096,), BF16), ((), torch.int64), ((3, 0), F32), ((7,), torch.float64)]
    parents = torch.randint(0, K, (B, K), generator=g)
    for par in (parents, torch.arange(K).expand(B, K), parents * 0, parents.int()):
        ts = [(torch.randn(B * K, *s, generator=g) * 50).to(d) for s, d in shapes]
        cuda = [t.cuda() for t in ts]
        nested = {"a": cuda[0], "rest": [cuda[1], tuple(cuda[2:])]}
        assert ops.reorder_states(nested, par.cuda()) is nested
        at = (torch.arange(B)[:, None] * K + par).flatten().long()
        for t, c in zip(ts, cuda):
            assert torch.equal(c.cpu(), t[at])


@gpu
def test_reorder_many_tensors_misaligned_and_out_of_range():
    B, K = 2, 3
    ts = [torch.randn(B * K, 5 + i, device="cuda") for i in range(150)]
    off = torch.randn(1 + B * K * 8, device="cuda")
    ts.append(off[1:].reshape(B * K, 8))
    before = [t.clone() for t in ts]
    par = torch.tensor([[1, 7, -1], [2, 0, 1]], device="cuda")
    ops.reorder_states(ts, par)
    at = torch.tensor([1, 1, 2, 5, 3, 4], device="cuda")
    assert all(torch.equal(t, b[at]) for t, b in zip(ts, before))
    torch.ops.mamba_b200.reorder_states(ts[:2], par)
    assert torch.equal(ts[0], before[0][at][at])
    assert ops.reorder_states([], par) == []


# --------------------------------------------------------------- whole search
def _stack(dtype, n=2, dm=64, S=16):
    s = MambaStack(n, dm, d_state=S)
    for i, layer in enumerate(s.layers):
        layer.mixer.load_state_dict(oracle.make_block_params(dm, S, seed=7 + i))
    return s.to("cuda", dtype)


def _plain_search(model, sampler, prompt, n, K, eos=None):
    """The search over whole sequences: every step runs each beam's sequence from
    the start and ranks all candidates in 64 bits."""
    B = prompt.shape[0]
    E, out, all_scores = sampler.E, [], []
    for b in range(B):
        beams = [([], 0.0)]
        for _ in range(n):
            cand = []
            for i, (toks, sc) in enumerate(beams):
                if eos is not None and toks and toks[-1] == eos:
                    cand.append((-sc, i, eos))
                    continue
                x = prompt[b:b + 1]
                if toks:
                    x = torch.cat([x, E[torch.tensor(toks, device=E.device)].to(x.dtype)[None]], 1)
                lp = torch.log_softmax(sampler.logits(model(x)[:, -1]).double()[0], -1).cpu()
                top = lp.topk(min(2 * K, lp.numel()))
                cand += [(-(sc + v), i, t) for v, t in zip(top.values.tolist(),
                                                           top.indices.tolist())]
            cand.sort()
            beams = [(beams[i][0] + [t], -v) for v, i, t in cand[:K]]
        out.append([t for t, _ in beams])
        all_scores.append([s for _, s in beams])
    return out, all_scores


@gpu
def test_search_matches_a_plain_one():
    model = _stack(F32)
    g = torch.Generator().manual_seed(5)
    E = torch.randn(90, 64, generator=g).cuda()
    sampler = TiedEmbeddingSampler(E * 0.4, norm_weight=torch.ones(64, device="cuda"))
    prompt = torch.randn(2, 9, 64, generator=g).cuda()
    with torch.no_grad():
        want, ws = _plain_search(model, sampler, prompt, 7, 3)
    eos = want[0][0][3]
    for e in (None, eos):
        if e is not None:
            with torch.no_grad():
                want, ws = _plain_search(model, sampler, prompt, 7, 3, eos=e)
        for per in (1, 2, 16):
            tok, sc = beam_search(model, sampler, prompt, 7, 3, eos_token=e, steps_per_graph=per)
            assert tok.tolist() == want
            # seven log probabilities of logits that carry the fp32 block's 1e-5 each
            assert (sc.double().cpu() - torch.tensor(ws).double()).abs().max() <= 7 * 2e-4


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_search_single_block_one_beam_is_greedy(dtype):
    block = CPUMamba(64, 16)
    block.load_state_dict(oracle.make_block_params(64, 16, seed=3))
    block = block.to("cuda", dtype)
    g = torch.Generator().manual_seed(6)
    E = torch.randn(50, 64, generator=g).to(dtype).cuda()
    prompt = torch.randn(3, 5, 64, generator=g).to(dtype).cuda()
    from cpu_mamba_b200.generate import generate
    tok, _ = generate(block, TiedEmbeddingSampler(E), prompt, 9)
    beam, sc = beam_search(block, TiedEmbeddingSampler(E), prompt, 9, 1)
    assert torch.equal(beam[:, 0], tok) and bool(torch.isfinite(sc).all())
    one, _ = beam_search(block, TiedEmbeddingSampler(E), prompt, 1, 4)
    assert one.shape == (3, 4, 1) and torch.equal(one[:, 0, 0], tok[:, 0])


@gpu
def test_search_length_penalty_and_refusals():
    model = _stack(F32)
    g = torch.Generator().manual_seed(8)
    E = torch.randn(40, 64, generator=g).cuda()
    s = TiedEmbeddingSampler(E * 0.2)
    prompt = torch.randn(1, 4, 64, generator=g).cuda()
    t0, s0 = beam_search(model, s, prompt, 6, 4, eos_token=1)
    t1, s1 = beam_search(model, s, prompt, 6, 4, eos_token=1, length_penalty=1.0)
    length = torch.where((t1 == 1).any(-1), (t1 == 1).int().argmax(-1) + 1, 6)
    ranked = s1 / length
    assert bool((ranked[:, :-1] >= ranked[:, 1:]).all())
    assert sorted(s0[0].tolist()) == sorted(s1[0].tolist())
    for call in (lambda: beam_search(model, s, prompt, 0, 2), lambda: beam_search(model, s, prompt, 2, 0),
                 lambda: beam_search(model, s, prompt, 2, 41),
                 lambda: beam_search(model, s, prompt, 2, 2, eos_token=40),
                 lambda: BeamLoop(model, s, None, None, None, steps_per_graph=0)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------- refusals
@pytest.mark.parametrize("args,code", [((7, 1, 1, 8, 1, 0), 1), ((0, -1, 1, 8, 1, 0), 2),
                                       ((0, 1, 33, 8, 1, 0), 2), ((0, 1, 1, 8, 65, 0), 2),
                                       ((0, 1, 1, 8, 9, 0), 2), ((0, 1, 1, 8, 0, 0), 2),
                                       ((0, 1, 1, (1 << 20) + 1, 1, 0), 2),
                                       ((0, 1, 1, 8, 1, 8), 2), ((0, 1, 1, 8, 1, -1), 2),
                                       ((0, 5000, 32, 8, 1, 0), 2), ((0, 1, 1, 8, 1, 0), 1),
                                       ((0, 0, 1, 8, 1, 0), 0)])
def test_select_c_entry_refuses(args, code):
    dt, B, K, V, num, pad = args
    f = _lib.lib().mb2_beam_select
    assert f(dt, None, V, V, None, None, pad, B, K, V, num, None, None, None, None, 0, None) == code
    if code == 1 and dt == 0:
        p = ctypes.c_void_p(256)
        assert f(dt, p, V, V, p, None, pad, B, K, V, num, p, p, p, p, 4, None) == 6


def test_reorder_c_entry_refuses():
    f = _lib.lib().mb2_reorder_rows
    ptrs, sizes = (ctypes.c_void_p * 1)(None), (ctypes.c_int64 * 1)(16)
    assert f(ptrs, sizes, 1, 256, 1, 33, None) == 2
    assert f(ptrs, sizes, 1, 256, 70000, 2, None) == 2
    assert f(ptrs, sizes, 1, 256, 1, 2, None) == 1            # null tensor
    assert f(ptrs, sizes, 1, None, 1, 2, None) == 1
    assert f(None, None, 0, None, 1, 2, None) == 0
    sizes[0] = 0
    assert f(ptrs, sizes, 1, 256, 1, 2, None) == 0            # nothing to move


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.beam_select(torch.zeros(1, 1, 4), torch.zeros(1, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.reorder_states([torch.zeros(2, 4)], torch.zeros(1, 2, dtype=torch.long))


@gpu
def test_refusals():
    x, s = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, device="cuda")
    f, par = ops.beam_select, torch.zeros(2, 3, dtype=torch.long, device="cuda")
    st = torch.zeros(6, 4, device="cuda")
    for call in (lambda: f(x[0], s), lambda: f(x, s[:1]), lambda: f(x, s.double()),
                 lambda: f(x, s, num=0), lambda: f(x, s, num=25), lambda: f(x, s, num=-1),
                 lambda: f(x, s, pad_token=8), lambda: f(x, s, finished=s),
                 lambda: f(x, s.cpu()), lambda: ops.reorder_states(st[:5], par),
                 lambda: ops.reorder_states(st.t().contiguous().t(), par),
                 lambda: ops.reorder_states(st.cpu(), par),
                 lambda: ops.reorder_states(st, par.float()),
                 lambda: ops.reorder_states(st, par[0])):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        f(x.double(), s)


@pytest.mark.parametrize("bases", [(4096, 4096), (4096, 4096 + 47), (4096 + 47, 4096)])
def test_reorder_c_entry_refuses_overlap(bases):
    """Two tensors of 2 x 3 rows of 8 bytes."""
    ptrs, sizes = (ctypes.c_void_p * 2)(*bases), (ctypes.c_int64 * 2)(8, 8)
    assert _lib.lib().mb2_reorder_rows(ptrs, sizes, 2, 4096, 2, 3, None) == 1
    assert b"overlap" in _lib.lib().mb2_last_error()


@gpu
def test_reorder_refuses_the_same_tensor_twice():
    x = torch.randn(6, 5, device="cuda")
    keep = x.clone()
    parents = torch.tensor([[1, 1, 0], [2, 0, 1]], device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        ops.reorder_states([x, {"h": x}], parents)
    assert torch.equal(x, keep)
    a, b = x[:, :0], torch.randn(12, 4, device="cuda")
    ops.reorder_states([a.contiguous(), b[:6], b[6:]], parents)      # neighbours in one buffer


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [7, 2047, 2049, 16383, 16384, 16385, 16391, 40000])
def test_select_around_the_slices(V, dtype):
    """Rows off 16 bytes; two tokens left of a row; rising logits, whose best all
    stand in the last slice."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(1, 2, V + 3, generator=g) * 3).to(dtype)[..., 3:]
    check(x, torch.zeros(1, 2), min(64, 2 * V))
    check(x.sort(-1).values, torch.zeros(1, 2), min(64, 2 * V))
    few = torch.full((1, 2, V), -torch.inf, dtype=dtype)
    few[..., V // 2], few[..., V - 1] = 1.0, 0.5
    check(few, torch.tensor([[-1.0, -2.0]]), 3)


class Bf16Sampler(TiedEmbeddingSampler):
    """A sampler whose logits are bf16 (a head that is not widened)."""

    def logits(self, y):
        return super().logits(y).to(BF16)


@gpu
def test_search_over_bf16_logits():
    model = _stack(F32)
    g = torch.Generator().manual_seed(12)
    E = torch.randn(40, 64, generator=g).cuda()
    prompt = torch.randn(2, 4, 64, generator=g).cuda()
    tok, sc = beam_search(model, Bf16Sampler(E), prompt, 5, 3)
    assert tok.shape == (2, 3, 5) and sc.dtype == F32 and bool(torch.isfinite(sc).all())
    with torch.no_grad():
        y, _ = model.forward_with_final_state(prompt)
        first = torch.log_softmax(Bf16Sampler(E).logits(y[:, -1]).double(), -1)
    one, s1 = beam_search(model, Bf16Sampler(E), prompt, 1, 3)
    want = first.sort(dim=-1, descending=True, stable=True)
    assert torch.equal(one[..., 0], want.indices[:, :3])
    assert ((s1.double() - want.values[:, :3]).abs() <= LSE + 2.0 ** -24 * want.values[:, :3].abs()).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1008, 9000, 20000])
def test_select_reads_an_expanded_beam_index(V, dtype):
    """Logits shared by a batch's beams (stride 0), each row at a 16-byte boundary as in
    the copy it is compared with: the same bits; and with logits on a coarse grid and
    equal scores, ties by beam and token as in 64 bits."""
    B, K, num = 2, 3, 12
    g = torch.Generator().manual_seed(V)
    row = torch.randn(B, 1, V, generator=g).to(dtype).cuda()
    s = torch.tensor([[0.0, -1.0, -0.3], [-2.0, -2.5, 0.0]]).cuda()
    wide = row.expand(B, K, V)
    assert wide.stride(1) == 0
    got, want = ops.beam_select(wide, s, num=num), ops.beam_select(wide.contiguous(), s, num=num)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    c, at = reference(wide.cpu(), s.cpu(), num)
    assert torch.equal((got[1] * V + got[2]).cpu(), at)
    assert bool(((got[0].double().cpu() - c.gather(1, at)).abs()
                 <= LSE + 2.0 ** -24 * c.gather(1, at).abs()).all())
    grid = torch.randint(-3, 4, (B, 1, V), generator=g).to(dtype).cuda().expand(B, K, V)
    same = torch.full((B, K), -2.0, device="cuda")
    got = ops.beam_select(grid, same, num=40)
    _, at = reference(grid.cpu(), same.cpu(), 40)
    assert torch.equal((got[1] * V + got[2]).cpu(), at)


def test_reorder_c_entry_without_memory_returns_an_error():
    """Four million empty tensors in a process without room for the list of them."""
    import pathlib
    import subprocess
    import sys
    code = """
import ctypes, resource
from cpu_mamba_b200 import _lib
f, n = _lib.lib().mb2_reorder_rows, 1 << 22
ptrs, sizes = (ctypes.c_void_p * n)(), (ctypes.c_int64 * n)()
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (8 << 20), resource.RLIM_INFINITY))
rc = f(ptrs, sizes, n, 256, 1, 2, None)
resource.setrlimit(resource.RLIMIT_AS, (resource.RLIM_INFINITY, resource.RLIM_INFINITY))
print(rc, _lib.lib().mb2_last_error())
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=str(pathlib.Path(__file__).resolve().parent.parent))
    assert r.returncode == 0, r.stderr
    assert r.stdout.startswith("4 b'reorder_rows"), r.stdout
