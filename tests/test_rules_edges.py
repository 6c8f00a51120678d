"""LogitRules where they can go wrong beside test_gated_layer.py's cases."""
import pytest
import torch

from cpu_mamba_b200.generate import BeamLoop, LogitRules, TiedEmbeddingSampler
from test_gated_layer import Model

gpu = pytest.mark.gpu


def masks(rows, words, kind):
    """A mask with rows of its own, in the ways a program may hold it; and its buffer."""
    g = torch.Generator().manual_seed(rows + words)
    bits = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=g).int().cuda()
    if kind == "contiguous":
        return bits, bits
    if kind == "wider":
        buf = torch.full((rows, words + 3), 7, dtype=torch.int32, device="cuda")
        buf[:, 1:1 + words] = bits
        return buf[:, 1:1 + words], buf
    buf = bits.t().contiguous()                           # words first
    return buf.t(), buf


@gpu
@pytest.mark.parametrize("kind", ["contiguous", "wider", "transposed"])
def test_masks_follow_their_beams(kind):
    mask, buf = masks(6, 3, kind)
    before = mask.clone()
    rules = LogitRules(6, 4, prompt_tokens=torch.arange(6, device="cuda")[:, None], mask=mask)
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]], device="cuda")
    flat = torch.tensor([2, 0, 0, 4, 4, 5], device="cuda")
    rules.reorder(parents)
    assert rules.mask is mask and torch.equal(mask, before[flat])
    assert torch.equal(rules.tokens[:, 0], flat)
    if kind == "wider":
        assert bool((buf[:, 0] == 7).all()) and bool((buf[:, 4:] == 7).all())


@gpu
def test_one_mask_for_all_stays():
    row = torch.randint(-2 ** 31, 2 ** 31, (1, 3)).int().cuda()
    kept = row.clone()
    rules = LogitRules(6, 4, mask=row.expand(6, 3))
    rules.reorder(torch.tensor([[2, 0, 0], [1, 1, 2]], device="cuda"))
    assert torch.equal(row, kept)


@gpu
@pytest.mark.parametrize("kind", ["contiguous", "wider", "transposed"])
def test_beams_under_masks_of_their_own(kind):
    """A grammar that forbids each token once it was used, told beam by beam between the
    steps: setting the loop up leaves the masks as they were, no beam repeats a token, and
    each beam's mask is that of its own sequence."""
    model = Model(seed=12)
    B, K, V, n = 2, 4, 90, 12
    prompt = torch.randint(0, V, (B, 5), generator=torch.Generator().manual_seed(13)).cuda()
    _, state = model.forward_with_final_state(model.E[prompt].repeat_interleave(K, 0))
    mask, _ = masks(B * K, 3, kind)
    mask.fill_(-1)
    first = torch.tensor([[3, 14, 15, 9], [2, 6, 53, 58]], device="cuda")
    rows = torch.arange(B * K, device="cuda")

    def forbid(tokens):
        t = tokens.flatten()
        mask[rows, t // 32] &= ~(1 << (t % 32)).int()

    forbid(first)
    before = mask.clone()
    rules = LogitRules(B * K, n + 1, mask=mask)
    rules.append(first.flatten())
    loop = BeamLoop(model, TiedEmbeddingSampler(model.E, rules=rules), state, first,
                    torch.zeros(B, K, device="cuda"), steps_per_graph=1)
    torch.cuda.synchronize()
    assert torch.equal(mask, before)
    moved = False
    for _ in range(n):
        loop.run(1)
        moved = moved or bool((loop.parents[0] != torch.arange(K, device="cuda")).any())
        forbid(loop.last)
    assert moved
    tokens = loop.result()[0].reshape(B * K, -1)
    assert torch.equal(rules.tokens, tokens)
    for row, words in zip(tokens.tolist(), mask.tolist()):
        assert len(set(row)) == n + 1
        assert {t for t in range(V) if not words[t // 32] >> (t % 32) & 1} == set(row)


@gpu
@pytest.mark.parametrize("temperature", [0.3, 0.7, 1.0, 1.9])
def test_rules_that_ask_for_nothing(temperature):
    """The same logits, bit for bit, and so the same tokens as without rules."""
    model = Model(seed=14)
    y = torch.randn(5, 48, generator=torch.Generator().manual_seed(15)).cuda()
    plain = TiedEmbeddingSampler(model.E, temperature)
    z = plain.logits(y)
    rules = LogitRules(5, 8)
    assert torch.equal(rules.adjust(z.clone(), temperature), z / temperature)
    torch.manual_seed(1)
    want = plain(y)[1]
    torch.manual_seed(1)
    assert torch.equal(TiedEmbeddingSampler(model.E, temperature, rules=rules)(y)[1], want)
    assert torch.equal(rules.tokens[:, 0], want)
