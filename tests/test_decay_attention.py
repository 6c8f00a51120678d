"""Decay attention, S_t = e^{g_t} S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t:
the prompt form (dense and packed) and the one-token form, against the
recurrence in 64 bits; refusals on the CPU."""
import pytest
import torch

from cpu_mamba_b200 import _lib, ops

gpu = pytest.mark.gpu


def reference(q, k, v, g, scale, h0=None):
    """(o, final state, bound): the recurrence in 64 bits for (B, T, H, width)
    inputs with all heads spelled out, and the same recurrence on absolute
    values, which bounds the sum of the magnitudes of an output's terms."""
    q, k, v = q.double(), k.double(), v.double()
    B, T, H, dv = v.shape
    s = torch.zeros(B, H, q.shape[-1], dv, dtype=torch.float64) if h0 is None else h0.double()
    m = s.abs()
    o, ob = torch.empty(B, T, H, dv, dtype=torch.float64), torch.empty(B, T, H, dv).double()
    for t in range(T):
        a = torch.exp(g[:, t].double())[..., None, None]
        kv = k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2)
        s, m = a * s + kv, a * m + kv.abs()
        o[:, t] = scale * (q[:, t].unsqueeze(-1) * s).sum(-2)
        ob[:, t] = abs(scale) * (q[:, t].abs().unsqueeze(-1) * m).sum(-2)
    return o, s, ob, m


def spread(x, H):
    return x.repeat_interleave(H // x.shape[2], dim=2)


def make(B, T, H, Hq, Hk, Hv, dk, dv, dtype, seed, per_head=False, strong=False):
    r = torch.Generator().manual_seed(seed)
    q = torch.randn(B, T, Hq, dk, generator=r).to(dtype)
    k = torch.randn(B, T, Hk, dk, generator=r).to(dtype)
    v = torch.randn(B, T, Hv, dv, generator=r).to(dtype)
    top = 30.0 if strong else 0.3
    g = -torch.rand(H, generator=r) * top if per_head else -torch.rand(B, T, H, generator=r) * top
    h0 = torch.randn(B, H, dk, dv, generator=r) * 2
    return q, k, v, g, h0


def tolerance(dtype, T, dk, o, ob):
    """fp32: an output is a sum of terms that pass through at most 3 roundings a
    token (decay, product, sum), dk additions and a few factors, each off by
    2^-24 relative: (3 T + dk + 32) 2^-24 times the sum of the terms' sizes.
    bf16 adds the output's rounding (2^-8 of it) and, on the tensor cores, the
    rounding to bf16 of the decayed scores and of the carried state (2^-8 of
    each term)."""
    f = (3 * T + dk + 32) * 2.0 ** -24
    if dtype == torch.float32:
        return f * ob
    return 2.0 ** -8 * (1 + 2.0 ** -8) * (o.abs() + ob) + f * ob


def state_tolerance(T, m):
    # fp32 throughout: 3 roundings a token and a few factors; bf16 inputs whose
    # decayed values are split into three bf16 parts lose 2^-26 more of a term
    return (3 * T + 32) * 2.0 ** -24 * m + 1e-30


def check(o, s, ref, dtype, T, dk):
    ro, rs, ob, m = ref
    d = (o.double().cpu() - ro).abs()
    assert bool((d <= tolerance(dtype, T, dk, ro, ob) + 1e-30).all()), (
        d / (tolerance(dtype, T, dk, ro, ob) + 1e-30)).max().item()
    if s is not None:
        d = (s.double().cpu() - rs).abs()
        assert bool((d <= state_tolerance(T, m)).all()), (d / state_tolerance(T, m)).max().item()


SHAPES = [  # B, T, H, Hq, Hk, Hv, dk, dv
    (1, 1, 1, 1, 1, 1, 1, 1),
    (2, 2, 2, 1, 2, 2, 3, 5),
    (2, 15, 4, 2, 1, 4, 16, 16),
    (1, 16, 2, 2, 2, 1, 32, 64),
    (3, 17, 6, 3, 6, 2, 20, 36),
    (2, 64, 2, 1, 1, 2, 64, 64),
    (1, 127, 2, 2, 2, 2, 128, 128),
    (1, 128, 3, 1, 1, 3, 128, 64),
    (2, 129, 2, 1, 1, 2, 64, 72),
    (1, 300, 2, 2, 1, 2, 24, 64),
    (1, 257, 1, 1, 1, 1, 104, 200),
    (1, 70, 1, 1, 1, 1, 200, 33),
    (1, 40, 2, 1, 2, 2, 256, 130),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_prompt_matches_the_recurrence(shape, dtype):
    B, T, H, Hq, Hk, Hv, dk, dv = shape
    q, k, v, g, h0 = make(*shape, dtype, seed=T + dk, per_head=T % 2 == 0)
    ref = reference(spread(q, H), spread(k, H), spread(v, H), g.expand(B, T, H), 0.7, h0)
    o, s = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), scale=0.7,
                               initial_state=h0.cuda(), return_final_state=True)
    assert o.dtype == dtype and o.shape == (B, T, H, dv) and s.dtype == torch.float32
    check(o, s, ref, dtype, T, dk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strong_decays_and_resets(dtype):
    """Decays down to e^-30 a token, a reset (g = -inf) in the middle, no
    initial state."""
    B, T, H, dk, dv = 2, 150, 2, 64, 64
    q, k, v, g, _ = make(B, T, H, 1, 2, 2, dk, dv, dtype, seed=3, strong=True)
    g[:, :50] *= 0.01
    g[0, 70, 0] = float("-inf")
    g[1, 0, 1] = float("-inf")
    g[:, 100:] = 0.0
    ref = reference(spread(q, H), spread(k, H), v, g, 1.0)
    o, s = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), return_final_state=True)
    check(o, s, ref, dtype, T, dk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weak_decay_over_a_long_sequence(dtype):
    """A head that forgets over 4096 tokens: the products of thousands of equal
    decays hold (all terms positive, so nothing hides in cancellation)."""
    B, T, H, dk, dv = 1, 6000, 1, 8, 8
    r = torch.Generator().manual_seed(1)
    q = torch.rand(B, T, H, dk, generator=r).to(dtype)
    k = torch.rand(B, T, H, dk, generator=r).to(dtype)
    v = torch.rand(B, T, H, dv, generator=r).to(dtype)
    g = torch.log1p(torch.tensor([-2.0 ** -12]))
    ref = reference(q, k, v, g.expand(B, T, H), 1.0)
    o, s = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), return_final_state=True)
    rel = ((s.double().cpu() - ref[1]) / ref[1]).abs().max().item()
    # 6000 sums of positive terms in fp32, each rounding within 2^-24 and of either
    # sign: 5 sqrt(6000) 2^-24 = 2.3e-5 bounds their random walk
    assert rel <= 2.3e-5, rel
    check(o, s, ref, dtype, T, dk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_sequences(dtype):
    """Lengths 0, 1, odd, over several tiles; rows behind the last sequence."""
    lens = [5, 0, 1, 130, 63, 200, 17]
    H, dk, dv = 4, 64, 48
    T = sum(lens) + 9
    q, k, v, g, _ = make(1, T, H, 2, 1, 4, dk, dv, dtype, seed=11)
    h0 = torch.randn(len(lens), H, dk, dv, generator=torch.Generator().manual_seed(2))
    cu = torch.tensor([0] + lens).cumsum(0)
    # what stands behind the last sequence must not matter
    for t in (q, k, v):
        t[:, -9:] = float("nan")
    out = torch.full((1, T, H, dv), 7.0, dtype=dtype, device="cuda")
    args = [t.cuda() for t in (q, k, v, g)]
    o, s = ops.decay_attention(*args, initial_state=h0.cuda(), cu_seqlens=cu.cuda(),
                               return_final_state=True, out=out)
    assert o.data_ptr() == out.data_ptr() and bool((out[:, -9:] == 7).all())
    new = ops.decay_attention(*args, initial_state=h0.cuda(), cu_seqlens=cu.cuda().int())
    assert bool((new[:, -9:] == 0).all()) and torch.equal(new[:, :-9], out[:, :-9])
    for i, n in enumerate(lens):
        a, b = int(cu[i]), int(cu[i + 1])
        if n == 0:
            assert torch.equal(s[i].cpu(), h0[i])
            continue
        ref = reference(spread(q[:, a:b], H), spread(k[:, a:b], H), v[:, a:b], g[:, a:b], 1.0,
                        h0[i:i + 1])
        check(o[:, a:b], s[i:i + 1], ref, dtype, n, dk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 3000, 1, 1, 1, 1, 64, 64), (2, 1537, 2, 1, 1, 2, 32, 40),
                                   (1, 2049, 1, 1, 1, 1, 128, 128)])
def test_few_heads_run_in_segments(shape, dtype):
    """Long prompts of few heads are cut along their tokens."""
    B, T, H, _, _, _, dk, dv = shape
    q, k, v, g, h0 = make(*shape, dtype, seed=T)
    g *= 0.05
    ref = reference(spread(q, H), spread(k, H), v, g, 1.0, h0)
    args = [t.cuda() for t in (q, k, v, g)]
    start = h0.cuda()
    o, s = ops.decay_attention(*args, initial_state=start, return_final_state=True)
    check(o, s, ref, dtype, T, dk)
    # its workspace is its own call's: two captured calls replayed in turn
    graphs = []
    for scale in (1.0, 2.0):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, ops.decay_attention(*args, scale=scale, initial_state=start)))
    for gr, _ in graphs * 2:
        gr.replay()
    assert torch.equal(graphs[0][1], o)
    ref2 = tuple(2 * t if i in (0, 2) else t for i, t in enumerate(ref))
    check(graphs[1][1], None, ref2, dtype, T, dk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_segments(dtype):
    """Ragged packed sequences long enough to be cut; an empty one keeps its
    state; overlapping offsets stay inside the tensors and the workspace."""
    lens = [1300, 0, 2, 2300, 129]
    H, dk, dv, T = 1, 64, 64, 3731 + 5
    q, k, v, g, _ = make(1, T, H, 1, 1, 1, dk, dv, dtype, seed=21)
    g *= 0.1
    h0 = torch.randn(len(lens), H, dk, dv, generator=torch.Generator().manual_seed(2))
    cu = torch.tensor([0] + lens).cumsum(0)
    args = [t.cuda() for t in (q, k, v, g)]
    o, s = ops.decay_attention(*args, initial_state=h0.cuda(), cu_seqlens=cu.cuda(),
                               return_final_state=True)
    assert bool((o[:, T - 5:] == 0).all())
    for i, n in enumerate(lens):
        a, b = int(cu[i]), int(cu[i + 1])
        if n == 0:
            assert torch.equal(s[i].cpu(), h0[i])
            continue
        ref = reference(q[:, a:b], k[:, a:b], v[:, a:b], g[:, a:b], 1.0, h0[i:i + 1])
        check(o[:, a:b], s[i:i + 1], ref, dtype, n, dk)
    bad = torch.tensor([0, T, 0, T, 0, T], device="cuda")
    ops.decay_attention(*args, initial_state=h0.cuda(), cu_seqlens=bad, return_final_state=True)
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_column_slices(dtype):
    """q, k, v as slices of one projection's rows, and transposed (heads before
    tokens) inputs, give the bits of contiguous ones."""
    B, T, H, dk, dv = 2, 140, 2, 64, 64
    r = torch.Generator().manual_seed(9)
    x = torch.randn(B, T, 2 * dk + H * dv + 8, generator=r).to(dtype).cuda()
    q, k = x[..., :dk].unsqueeze(2), x[..., dk:2 * dk].unsqueeze(2)
    v = x[..., 2 * dk:2 * dk + H * dv].unflatten(-1, (H, dv))
    g = (-torch.rand(B, T, H, generator=r)).cuda()
    a = ops.decay_attention(q, k, v, g)
    b = ops.decay_attention(q.contiguous(), k.contiguous(), v.contiguous(), g)
    assert torch.equal(a, b)
    vt = v.transpose(1, 2).contiguous().transpose(1, 2)
    gt = g.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.decay_attention(q, k, vt, gt), a)
    odd = torch.randn(B, T, 1 + H * dv, generator=r).to(dtype).cuda()
    vo = odd[..., 1:].unflatten(-1, (H, dv))                 # rows off every 16-byte boundary
    check(ops.decay_attention(q, k, vo, g), None,
          reference(spread(q.cpu(), H), spread(k.cpu(), H), vo.cpu(), g.cpu(), 1.0), dtype, T, dk)
    rev = v.transpose(2, 3).contiguous().transpose(2, 3)     # last index not contiguous
    assert torch.equal(ops.decay_attention(q, k, rev, g), a)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_later_tokens_do_not_reach_back(dtype):
    """Infinities and NaN in a token leave every earlier output as it was."""
    B, T, H, dk, dv = 1, 200, 2, 64, 64
    q, k, v, g, h0 = make(B, T, H, 1, 1, 2, dk, dv, dtype, seed=4)
    args = [t.cuda() for t in (q, k, v, g)]
    clean = ops.decay_attention(*args, initial_state=h0.cuda())
    v[:, 150, 0] = float("inf")
    k[:, 170] = float("nan")
    got = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), initial_state=h0.cuda())
    ref = reference(spread(q, H), spread(k, H), v, g, 1.0, h0)
    check(got[:, :150], None, tuple(t[:, :150] if t.dim() == 4 and t.shape[1] == T else t
                                    for t in ref), dtype, T, dk)
    assert bool(torch.isfinite(got[:, :150]).all())
    assert bool(torch.isfinite(got[:, 150:170, 1]).all())
    assert not bool(torch.isfinite(got[:, 150:, 0]).any())
    assert bool(torch.isnan(got[:, 170:]).all())
    assert torch.equal(clean[:, :128], got[:, :128])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1, 1), (3, 6, 3, 1, 2, 20, 36),
                                   (5, 4, 4, 4, 4, 128, 128), (2, 2, 1, 1, 2, 64, 300),
                                   (70, 8, 1, 1, 8, 128, 64), (1, 2, 1, 2, 1, 256, 33)])
def test_one_token(shape, dtype):
    B, H, Hq, Hk, Hv, dk, dv = shape
    q, k, v, g, h0 = make(B, 1, H, Hq, Hk, Hv, dk, dv, dtype, seed=dk)
    ref = reference(spread(q, H), spread(k, H), spread(v, H), g, 0.5, h0)
    s = h0.cuda()
    o = ops.decay_attention_step(q[:, 0].cuda(), k[:, 0].cuda(), v[:, 0].cuda(), g[:, 0].cuda(), s,
                                 scale=0.5)
    assert o.shape == (B, H, dv) and o.dtype == dtype
    check(o.unsqueeze(1), s, ref, dtype, 1, dk)
    s2 = h0.cuda()
    gh = g[0, 0].clone()
    o2 = ops.decay_attention_step(q[:1, 0].cuda(), k[:1, 0].cuda(), v[:1, 0].cuda(), gh.cuda(),
                                  s2[:1], scale=0.5)
    assert torch.equal(o2[0], o[0]) and torch.equal(s2[0], s[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """A prompt's final state continued token by token, on a side stream and as a
    replayed graph, gives the outputs of the whole sequence."""
    B, T, n, H, dk, dv = 2, 90, 4, 2, 64, 64
    q, k, v, g, _ = make(B, T, H, 1, 1, 2, dk, dv, dtype, seed=6)
    ref = reference(spread(q, H), spread(k, H), v, g, 1.0)
    q, k, v, g = (t.cuda() for t in (q, k, v, g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, s = ops.decay_attention(*(t[:, :T - n] for t in (q, k, v, g)), return_final_state=True)
        outs = [o]
        outs += [ops.decay_attention_step(q[:, T - n], k[:, T - n], v[:, T - n], g[:, T - n],
                                          s).unsqueeze(1)]
    torch.cuda.current_stream().wait_stream(side)
    cur = [t[:, 0].clone() for t in (q, k, v, g)]
    graph = torch.cuda.CUDAGraph()
    keep = s.clone()
    with torch.cuda.graph(graph):
        y = ops.decay_attention_step(*cur, s)
    assert torch.equal(s, keep)
    for t in range(T - n + 1, T):
        for c, x in zip(cur, (q, k, v, g)):
            c.copy_(x[:, t])
        graph.replay()
        outs.append(y.clone().unsqueeze(1))
    check(torch.cat(outs, 1), s, ref, dtype, T, dk)


@gpu
def test_prompt_in_a_graph_matches_eager():
    q, k, v, g, h0 = (t.cuda() for t in make(2, 300, 4, 1, 1, 4, 64, 64, torch.bfloat16, seed=8))
    cu = torch.tensor([0, 100, 300], device="cuda", dtype=torch.int32)
    a = ops.decay_attention(q, k, v, g, initial_state=h0)
    p = ops.decay_attention(q[:1], k[:1], v[:1], g[:1], cu_seqlens=cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ya = ops.decay_attention(q, k, v, g, initial_state=h0)
        yp = ops.decay_attention(q[:1], k[:1], v[:1], g[:1], cu_seqlens=cu)
    for _ in range(2):
        ya.fill_(3)
        yp.fill_(3)
        graph.replay()
        assert torch.equal(ya, a) and torch.equal(yp, p)


@gpu
def test_broken_offsets_stay_inside():
    """Offsets out of order or out of range address no row outside the tensors
    (they are clamped); no sequence at all leaves zeros."""
    q, k, v, g, _ = (t.cuda() for t in make(1, 50, 2, 1, 1, 2, 32, 32, torch.float32, seed=5))
    for cu in ([0, 40, 20, 99], [-5, 10, 10, 50], [50, 50]):
        o = ops.decay_attention(q, k, v, g, cu_seqlens=torch.tensor(cu, device="cuda"))
        assert o.shape == v.shape
    z, s = ops.decay_attention(q, k, v, g, cu_seqlens=torch.zeros(1, device="cuda").int(),
                               return_final_state=True)
    assert s.shape[0] == 0


@gpu
def test_empty_prompt_returns_the_state():
    q, k, v, g, h0 = (t.cuda() for t in make(2, 0, 2, 1, 1, 2, 32, 32, torch.float32, seed=5))
    o, s = ops.decay_attention(q, k, v, g, initial_state=h0, return_final_state=True)
    assert o.shape == (2, 0, 2, 32) and torch.equal(s, h0)
    _, s = ops.decay_attention(q, k, v, g, return_final_state=True)
    assert bool((s == 0).all())


@gpu
def test_torch_ops():
    q, k, v, g, h0 = (t.cuda() for t in make(1, 20, 2, 1, 1, 2, 16, 16, torch.float32, seed=5))
    o, s = ops.decay_attention(q, k, v, g, initial_state=h0, return_final_state=True)
    o2, s2 = torch.ops.mamba_b200.decay_attention(q, k, v, g, 1.0, h0, None)
    assert torch.equal(o, o2) and torch.equal(s, s2)
    st = s.clone()
    y = torch.ops.mamba_b200.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], st, 1.0)
    assert torch.equal(y, ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s))
    assert torch.equal(s, st)


# ------------------------------------------------------------- refusals (CPU)
def desc(**kw):
    d = _lib.DecayAttn()
    d.batch, d.seqlen, d.heads, d.q_heads, d.k_heads, d.v_heads, d.dk, d.dv = 1, 4, 2, 1, 1, 2, 8, 8
    for n, x in kw.items():
        setattr(d, n, x)
    return d


@pytest.mark.parametrize("kw,code", [({"dtype": 5}, 1), ({"batch": -1}, 2), ({"dk": 257}, 2),
                                     ({"dk": 0}, 2), ({"dv": 0}, 2), ({"q_heads": 3}, 2),
                                     ({"v_heads": 0}, 2), ({"heads": 0}, 2), ({}, 1),
                                     ({"batch": 2, "cu_seqlens": 16, "n_seqs": 1}, 2)])
def test_c_entry_refuses(kw, code):
    import ctypes
    lib = _lib.lib()
    assert lib.mb2_decay_attention(ctypes.byref(desc(**kw)), None, 0, None) == code
    assert b"decay_attention" in lib.mb2_last_error()
    assert lib.mb2_decay_attention_step(ctypes.byref(desc(**kw)), None, None) == code
    assert lib.mb2_decay_attention(None, None, 0, None) == 1


def test_c_entry_nothing_to_do():
    import ctypes
    lib = _lib.lib()
    assert lib.mb2_decay_attention(ctypes.byref(desc(batch=0)), None, 0, None) == 0
    assert lib.mb2_decay_attention_step(ctypes.byref(desc(batch=0)), None, None) == 0


def test_cpu_tensors_are_refused():
    q, k, v, g, h0 = make(1, 4, 2, 1, 1, 2, 8, 8, torch.float32, seed=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.decay_attention(q, k, v, g)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], h0)


@gpu
def test_refusals():
    q, k, v, g, h0 = (t.cuda() for t in make(2, 6, 4, 1, 2, 4, 8, 8, torch.float32, seed=1))
    f = ops.decay_attention
    bad = [
        lambda: f(q[0], k, v, g), lambda: f(q, k.bfloat16(), v, g), lambda: f(q, k, v, g.double()),
        lambda: f(q[:, :5], k, v, g), lambda: f(q[..., :7], k, v, g), lambda: f(q, k, v, g[..., :3]),
        lambda: f(q, k, v, g[:, :, 0]), lambda: f(q, k, v, g, initial_state=h0[:1]),
        lambda: f(q, k, v, g, initial_state=h0.bfloat16()),
        lambda: f(q, k, v, g, cu_seqlens=torch.tensor([0, 6], device="cuda")),
        lambda: f(q[:1], k[:1], v[:1], g[:1], cu_seqlens=torch.tensor([0., 6.], device="cuda")),
        lambda: f(q, k, v, g, out=v.bfloat16()), lambda: f(q, k, v, g, out=v[:, :5]),
        lambda: f(q, k, v.cpu(), g),
        lambda: ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], h0[:, :3]),
        lambda: ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], h0.transpose(2, 3)),
        lambda: ops.decay_attention_step(q, k, v, g, h0),
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        f(q.double(), k.double(), v.double(), g)
    wide = torch.zeros(1, 3, 1, 257, device="cuda")
    with pytest.raises(RuntimeError, match="257"):
        f(wide, wide, wide, torch.zeros(1, device="cuda"))


# ---------------------------------------- widths and rows off 16-byte groups
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 200, 4, 2, 1, 4, 87, 64), (1, 260, 3, 1, 3, 1, 64, 14),
                                   (3, 129, 2, 2, 2, 2, 10, 51), (40, 70, 8, 1, 2, 8, 33, 67),
                                   (1, 1100, 1, 1, 1, 1, 127, 121)])
def test_odd_widths(shape, dtype):
    """States in and out, at an address off 16 bytes."""
    B, T, H, Hq, Hk, Hv, dk, dv = shape
    q, k, v, g, h0 = make(*shape, dtype, seed=T + dv)
    ref = reference(spread(q, H), spread(k, H), spread(v, H), g.expand(B, T, H), 0.7, h0)
    o, s = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), scale=0.7,
                               initial_state=h0.cuda(), return_final_state=True)
    check(o, s, ref, dtype, T, dk)
    shifted = torch.empty(h0.numel() + 1, device="cuda")[1:].view(h0.shape).copy_(h0)
    o2, s2 = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), scale=0.7,
                                 initial_state=shifted, return_final_state=True)
    check(o2, s2, ref, dtype, T, dk)


@gpu
@pytest.mark.parametrize("dv", [64, 61])
def test_odd_packed_rows_outside_the_sequences_stay(dv):
    """An `out` with other strides: rows behind the last sequence and columns
    between its rows keep what they held; broadcast q, one sequence empty."""
    T, H, dk, dtype = 700, 3, 45, torch.bfloat16
    q, k, v, g, h0 = make(1, T, H, 1, 1, H, dk, dv, dtype, seed=dv)
    cu = torch.tensor([0, 250, 250, 640], dtype=torch.int32)
    h0 = torch.randn(3, H, dk, dv, generator=torch.Generator().manual_seed(2))
    hold = torch.full((1, T, H, dv + 5), 7.0, dtype=dtype, device="cuda")
    out = hold[..., 3:3 + dv]
    o, s = ops.decay_attention(q.cuda().expand(1, T, H, dk), k.cuda(), v.cuda(), g.cuda(),
                               cu_seqlens=cu.cuda(), initial_state=h0.cuda(),
                               return_final_state=True, out=out)
    assert o.data_ptr() == out.data_ptr()
    assert bool((hold[:, 640:] == 7).all())
    assert bool((hold[..., :3] == 7).all() and (hold[..., 3 + dv:] == 7).all())
    for i in range(3):
        a, b = cu[i].item(), cu[i + 1].item()
        if a == b:
            assert torch.equal(s[i].cpu(), h0[i])
            continue
        w = slice(a, b)
        ref = reference(spread(q[:, w], H), spread(k[:, w], H), v[:, w], g[:, w], 1.0, h0[i:i + 1])
        check(o[:, w], s[i:i + 1], ref, dtype, b - a, dk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_odd_widths_in_a_graph_and_on_two_streams(dtype):
    q, k, v, g, h0 = (t.cuda() for t in make(2, 333, 4, 1, 1, 4, 50, 39, dtype, seed=3))
    want = ops.decay_attention(q, k, v, g, initial_state=h0)
    other = ops.decay_attention(k, q, v, g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.decay_attention(q, k, v, g, initial_state=h0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        y.fill_(3)
        torch.cuda.synchronize()
        got = []
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                got.append(ops.decay_attention(*((q, k) if i % 2 == 0 else (k, q)), v, g,
                                               initial_state=h0 if i % 2 == 0 else None))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert all(torch.equal(x, other if i % 2 else want) for i, x in enumerate(got))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,T", [(1, 9), (8, 31), (148, 33), (300, 40), (2100, 20)])
def test_few_and_many_walks(heads, T, dtype):
    """Both spreads of a state over lanes, with decays that end a run inside a
    group of tokens, at every place in it."""
    for dk, dv in ((16, 24), (30, 64), (64, 32), (120, 8), (180, 4)):
        q, k, v, g, h0 = make(1, T, heads, 1, 1, heads, dk, dv, dtype, seed=heads + dk)
        g = g.clone()
        g[0, ::7, ::2] = -6.0
        g[0, 3::5, 1::3] = -3.5
        ref = reference(spread(q, heads), spread(k, heads), v, g, 1.0, h0)
        o, s = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(),
                                   initial_state=h0.cuda(), return_final_state=True)
        check(o, s, ref, dtype, T, dk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,dv", [(200, 64), (200, 37), (40, 16)])
def test_rows_outside_the_packed_sequences(T, dv, dtype):
    """Rows before the first sequence, too: zero in a new output, kept in `out`."""
    q, k, v, g, _ = make(1, T, 2, 1, 1, 2, 32, dv, dtype, seed=T)
    cu = torch.tensor([7, 20, T - 9], device="cuda")
    args = [t.cuda() for t in (q, k, v, g)]
    torch.full((1, T, 2, dv), float("nan"), dtype=dtype, device="cuda")    # freed: its bytes stay
    new = ops.decay_attention(*args, cu_seqlens=cu)
    assert bool((new[:, :7] == 0).all() and (new[:, T - 9:] == 0).all())
    out = torch.full((1, T, 2, dv), 7.0, dtype=dtype, device="cuda")
    ops.decay_attention(*args, cu_seqlens=cu, out=out)
    assert bool((out[:, :7] == 7).all() and (out[:, T - 9:] == 7).all())
    assert torch.equal(out[:, 7:T - 9], new[:, 7:T - 9])
    for a, b in ((7, 20), (20, T - 9)):
        ref = reference(spread(q[:, a:b], 2), spread(k[:, a:b], 2), v[:, a:b], g[:, a:b], 1.0)
        check(new[:, a:b], None, ref, dtype, b - a, 32)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", [(18, 63), (65, 62), (66, 63), (129, 64), (250, 129), (24, 64),
                                   (48, 64), (49, 64), (97, 64), (3, 4), (256, 256)])
def test_one_token_by_every_size_of_block(dk, dv, dtype):
    """Few and many threads, by rows of 16 and of 4 bytes; an address off 16 bytes."""
    q, k, v, g, h0 = make(3, 1, 4, 2, 1, 4, dk, dv, dtype, seed=dk + dv)
    ref = reference(spread(q, 4), spread(k, 4), v, g, 1.0, h0)
    one = [t[:, 0].cuda() for t in (q, k, v, g)]
    for s in (h0.cuda(), torch.empty(h0.numel() + 1, device="cuda")[1:].view(h0.shape).copy_(h0)):
        o = ops.decay_attention_step(*one, s)
        check(o.unsqueeze(1), s, ref, dtype, 1, dk)


# ------------------------------------------------- hand-overs between the roles
def beside_copies(call, times):
    """The results of ``call`` on one stream while another one copies: loads then
    come late and out of order."""
    a = torch.zeros(1 << 26, device="cuda")
    b = torch.empty_like(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(times):
        with torch.cuda.stream(side):
            b.copy_(a)
        got.append(call())
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    return got


@gpu
def test_v_has_arrived_before_it_is_multiplied():
    """The same bits whenever the loads of v come; each sequence ends inside a chunk,
    before one whose first token holds infinities."""
    lens = [300, 129, 1, 500, 77, 640, 255]
    H, dk, dv, dtype = 40, 128, 64, torch.bfloat16
    q, k, v, g, _ = make(1, sum(lens), H, 1, 1, H, dk, dv, dtype, seed=31)
    cu = torch.tensor([0] + lens).cumsum(0)
    clean = v.clone()
    v[:, cu[1:-1], :, ::3] = float("-inf")
    args = [t.cuda() for t in (q, k, v, g)]
    got = beside_copies(lambda: ops.decay_attention(*args, cu_seqlens=cu.cuda()), 30)
    assert all(torch.equal(o.view(torch.int16), got[0].view(torch.int16)) for o in got)
    w = slice(0, lens[0])                                # the sequence without them
    ref = reference(spread(q[:, w], H), spread(k[:, w], H), clean[:, w], g[:, w], 1.0)
    check(got[0][:, w], None, ref, dtype, lens[0], dk)


@gpu
def test_many_short_spans_and_long_ones_keep_their_hand_overs():
    """Sequences of one chunk and of many, side by side, several items a CTA."""
    r = torch.Generator().manual_seed(5)
    lens = [int(n) for n in torch.randint(1, 3, (40,), generator=r) * 127] + [2000, 1, 128, 129, 0]
    H, dk, dv, dtype = 32, 64, 64, torch.bfloat16
    q, k, v, g, _ = make(1, sum(lens), H, 1, 1, H, dk, dv, dtype, seed=32)
    h0 = torch.randn(len(lens), H, dk, dv, generator=r)
    cu = torch.tensor([0] + lens).cumsum(0)
    args = [t.cuda() for t in (q, k, v, g)]
    got = beside_copies(lambda: ops.decay_attention(*args, cu_seqlens=cu.cuda(), return_final_state=True,
                                                    initial_state=h0.cuda()), 20)
    assert all(torch.equal(x, y) for pair in got for x, y in zip(pair, got[0]))
    for i in (0, 7, 40, 42, 43):
        w = slice(int(cu[i]), int(cu[i + 1]))
        ref = reference(spread(q[:, w], H), spread(k[:, w], H), v[:, w], g[:, w], 1.0, h0[i:i + 1])
        check(got[0][0][:, w], got[0][1][i:i + 1], ref, dtype, lens[i], dk)


@gpu
def test_keys_behind_a_sequence_do_not_reach_it():
    """The bits of a call without them, whatever keys follow a sequence's last token."""
    lens = [300, 129, 1, 500, 77, 640, 255]
    H, dk, dv, dtype = 40, 128, 64, torch.bfloat16
    q, k, v, g, _ = make(1, sum(lens), H, 1, 1, H, dk, dv, dtype, seed=33)
    cu = torch.tensor([0] + lens).cumsum(0)
    args = [t.cuda() for t in (q, k, v, g)]
    want = ops.decay_attention(*args, cu_seqlens=cu.cuda())
    bad = args[1].clone()                     # every second sequence without a finite key
    keep = torch.zeros(sum(lens), dtype=torch.bool, device="cuda")
    for i in range(len(lens)):
        w = slice(int(cu[i]), int(cu[i + 1]))
        keep[w] = i % 2 == 0
        if i % 2:
            bad[:, w] = float("nan") if i % 4 == 1 else float("inf")
    got = beside_copies(lambda: ops.decay_attention(args[0], bad, *args[2:], cu_seqlens=cu.cuda()), 30)
    for o in got:
        assert torch.equal(o[:, keep], want[:, keep])
        assert not bool(torch.isfinite(o[:, ~keep]).any())


@gpu
@pytest.mark.parametrize("shape", [(1, 128, 3, 1, 1, 3, 128, 64), (2, 129, 2, 1, 1, 2, 64, 72),
                                   (1, 300, 2, 2, 1, 2, 24, 64), (2, 515, 4, 1, 2, 4, 128, 128),
                                   (1, 2049, 1, 1, 1, 1, 128, 64), (3, 200, 4, 2, 1, 4, 87, 50),
                                   (148, 20, 1, 1, 1, 1, 16, 8)])
def test_bf16_outputs_are_rounded_once(shape):
    """A bf16 prompt's output is the formula's, rounded to bf16 (2^-8 of it): scores and
    carried states enter their products in two bf16 parts, which lose 2^-8 2^-8 of a term."""
    B, T, H, _, _, _, dk, dv = shape
    q, k, v, g, h0 = make(*shape, torch.bfloat16, seed=T + dv)
    ro, rs, ob, m = reference(spread(q, H), spread(k, H), spread(v, H), g, 0.7, h0)
    o, s = ops.decay_attention(q.cuda(), k.cuda(), v.cuda(), g.cuda(), scale=0.7,
                               initial_state=h0.cuda(), return_final_state=True)
    terms = (2.0 ** -16 + (3 * T + dk + 32) * 2.0 ** -24) * ob
    tol = 2.0 ** -8 * (ro.abs() + terms) + terms + 1e-30
    d = (o.double().cpu() - ro).abs()
    assert bool((d <= tol).all()), (d / tol).max().item()
    d = (s.double().cpu() - rs).abs()
    assert bool((d <= state_tolerance(T, m)).all()), (d / state_tolerance(T, m)).max().item()


def fastest(call, times=5):
    best = float("inf")
    for _ in range(times):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        call()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@gpu
def test_a_state_that_is_not_finite_costs_its_own_columns_only():
    """One NaN in h0: its column is NaN, every other output keeps its bits, and the call
    takes no longer (a row that is computed again costs hundreds of times a chunk; a
    call next to it on the stream and the clocks stay within a factor of 4)."""
    B, T, H, dk, dv = 2, 1024, 8, 128, 64
    q, k, v, g, h0 = (t.cuda() for t in make(B, T, H, 1, 1, H, dk, dv, torch.bfloat16, seed=41))
    bad = h0.clone()
    bad[:, :, 17, 5] = float("nan")
    clean = ops.decay_attention(q, k, v, g, initial_state=h0)
    got = ops.decay_attention(q, k, v, g, initial_state=bad)
    keep = torch.arange(dv, device="cuda") != 5
    assert torch.equal(got[..., keep], clean[..., keep])
    assert bool(torch.isnan(got[..., 5]).all())
    for x in (float("inf"), float("-inf")):
        bad[:, :, 17, 5] = x
        got = ops.decay_attention(q, k, v, g, initial_state=bad)
        assert torch.equal(got[..., keep], clean[..., keep])
        want = torch.sign(q[..., 17].float()).expand(B, T, H) * x
        assert torch.equal(got[..., 5].float(), want)
    # (no segments: their states carry it from one to the next)
    wide = [t.repeat_interleave(24, 0) for t in (q, k, v, g, h0, bad)]
    plain = fastest(lambda: ops.decay_attention(*wide[:4], initial_state=wide[4]))
    assert fastest(lambda: ops.decay_attention(*wide[:4], initial_state=wide[5])) <= 4 * plain


@gpu
@pytest.mark.parametrize("dv", [64, 40])
def test_rows_before_an_infinity_are_rounded_once(dv):
    """Rows that share a chunk with a later infinity are computed again, to the same
    accuracy as all others."""
    B, T, H, dk = 2, 300, 3, 128
    q, k, v, g, h0 = make(B, T, H, 1, 1, H, dk, dv, torch.bfloat16, seed=42)
    ro, _, ob, _ = reference(spread(q, H), spread(k, H), v, g, 1.0, h0)
    v[:, 200] = float("inf")
    v[1, 37, 1, 3] = float("nan")
    o = ops.decay_attention(*(t.cuda() for t in (q, k, v, g)), initial_state=h0.cuda())
    terms = (2.0 ** -16 + (3 * T + dk + 32) * 2.0 ** -24) * ob
    d = (o.double().cpu() - ro).abs()
    ok = d <= 2.0 ** -8 * (ro.abs() + terms) + terms + 1e-30
    ok[1, 37:, 1, 3] = True
    assert bool(ok[:, :200].all()) and not bool(torch.isfinite(o[:, 200:]).any())
    assert bool(torch.isnan(o[1, 37:, 1, 3]).all())


def kinds(x):
    """0 finite, 1 +inf, -1 -inf, 2 NaN"""
    k = torch.where(x.isnan(), 2.0, 0.0)
    return torch.where(x.isinf(), x.sign().double(), k.double())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,B", [(400, 3), (100, 3), (20, 40), (2049, 1)])
def test_infinities_stay_infinities_in_the_state(T, B, dtype):
    """An infinite v or k leaves the infinities of the recurrence in the final state (and
    in the outputs behind an infinite k), on both paths and in segments; every other
    element is finite and right."""
    H, dk, dv = 3, 64, 40
    q, k, v, g, h0 = make(B, T, H, H, H, H, dk, dv, dtype, seed=T)
    g *= min(1.0, 200 / T)
    inf = float("inf")
    v[:, T // 3, 0, 7] = inf
    v[:, T // 2, 0, 11] = -inf
    k[:, T // 4, 1, 30] = inf
    k[:, T - 1, 1, 33] = -inf
    ref = reference(q, k, v, g, 1.0, h0)
    o, s = ops.decay_attention(*(t.cuda() for t in (q, k, v, g)), initial_state=h0.cuda(),
                               return_final_state=True)
    s, o = s.double().cpu(), o.double().cpu()
    assert torch.equal(kinds(s), kinds(ref[1]))
    fine = kinds(ref[1]) == 0
    assert bool(((s - ref[1]).abs() <= state_tolerance(T, ref[3]))[fine].all())
    assert torch.equal(kinds(o[:, :, 1:]), kinds(ref[0][:, :, 1:]))
    cols = [c for c in range(dv) if c not in (7, 11)]
    assert bool(o[:, :, 0, cols].isfinite().all())
    assert not bool(o[:, T // 3:, 0, 7].isfinite().any())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dv", [64, 61])
def test_offsets_that_fall(dv, dtype):
    """A sequence whose end is not behind its start is empty, and the others are computed
    wherever they stand: with rows as they are and with rows that are laid out again."""
    T, H, dk = 400, 2, 64
    q, k, v, g, _ = make(1, T, H, 1, 1, H, dk, dv, dtype, seed=dv)
    h0 = torch.randn(4, H, dk, dv, generator=torch.Generator().manual_seed(2))
    args = [t.cuda() for t in (q, k, v, g)]
    for cu in ([150, 390, 20, 140, 10], [300, 399, 0, 0, 250], [0, 100, 90, 90, 90]):
        out = torch.full((1, T, H, dv), 7.0, dtype=dtype, device="cuda")
        held = torch.zeros(T, dtype=torch.bool)
        n = len(cu) - 1
        kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"), initial_state=h0.cuda(),
                  return_final_state=True)
        new, s = ops.decay_attention(*args, **kw)
        ops.decay_attention(*args, out=out, **kw)
        for i in range(n):
            w = slice(cu[i], cu[i + 1])
            if cu[i + 1] <= cu[i]:
                assert torch.equal(s[i].cpu(), h0[i])
                continue
            held[w] = True
            ref = reference(spread(q[:, w], H), spread(k[:, w], H), v[:, w], g[:, w], 1.0, h0[i:i + 1])
            check(new[:, w], s[i:i + 1], ref, dtype, cu[i + 1] - cu[i], dk)
        assert torch.equal(out[:, held.cuda()], new[:, held.cuda()])
        assert bool((out[:, ~held.cuda()] == 7).all())
        assert bool((new[:, ~held.cuda()] == 0).all())


@gpu
def test_an_expanded_out_is_refused():
    """Rows, heads or sequences that would be written to one place."""
    q, k, v, g, _ = (t.cuda() for t in make(2, 6, 4, 1, 2, 4, 8, 8, torch.float32, seed=1))
    for i in range(3):
        shape = [1 if j == i else n for j, n in enumerate(v.shape)]
        with pytest.raises(RuntimeError, match="one place"):
            ops.decay_attention(q, k, v, g, out=torch.empty(shape, device="cuda").expand(v.shape))
    one = torch.empty_like(v[:1]).expand(1, 6, 4, 8)
    assert ops.decay_attention(q[:1], k[:1], v[:1], g[:1], out=one).data_ptr() == one.data_ptr()


@pytest.mark.parametrize("heads,tokens,dk,dv", [(1900, 32768, 32, 64), (20, 600, 250, 64)])
def test_segments_are_planned_for_the_walks_that_fit(heads, tokens, dk, dv):
    """12 one-warp walks of 32 rows share an SM, and one narrow walk of more than 128 rows
    has it for itself: these calls (two uneven rounds) are cut along their tokens, which
    shows in their workspace."""
    import ctypes
    d = desc(heads=heads, v_heads=1, seqlen=tokens, dk=dk, dv=dv)
    assert _lib.lib().mb2_decay_attention_workspace_bytes(ctypes.byref(d)) >= 2 * heads * dk * dv * 4
