"""The paged 4-bit model (tendo_b200/paged.py): its logits against the same
model in 64 bits with the cache rounded to 4 bits, drafts against none, and
pages that come back.

A K or V value that lies within an fp32 rounding of the middle between two
codes may be held one code off, which moves the logits by far less than the
2e-2 of max |logit| allowed; any mistake of place or mask moves them by more.
"""
import math

import numpy as np
import pytest

from test_gpu_kv4 import quantize_rows, rope, values_of

pytestmark = pytest.mark.gpu

CFG = dict(vocab=500, dim=256, layers=2, heads=8, kv_heads=2, hidden=384, max_seq=256, rope_base=10000.0, eps=1e-5)


@pytest.fixture(scope="module")
def model(cuda):
    from tendo_b200.paged import PagedLlama

    return PagedLlama(CFG, num_blocks=64, block_size=16, max_requests=5, seed=3)


def _norm(x):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + CFG["eps"])


def reference(model, seq):
    """Logits [len, V] of one sequence in 64 bits, K and V rounded to 4 bits."""
    f = lambda t: t.detach().cpu().numpy().astype(np.float64)  # noqa: E731
    w64 = lambda q: f(q[0]) * f(q[1])[:, None]  # noqa: E731
    H, Hkv, D = CFG["heads"], CFG["kv_heads"], model.D
    n = len(seq)
    x = f(model.embed)[seq]
    c, s = (f(t)[:n, None] for t in (model.cos, model.sin))
    for w in model.layers:
        rows = (_norm(x) @ w64(w["qkv"]).T).reshape(n, H + 2 * Hkv, D)
        q = rope(rows[:, :H], c, s)
        held = [values_of(*quantize_rows(t.astype(np.float32))).astype(np.float64)
                for t in (rope(rows[:, H:H + Hkv], c, s), rows[:, H + Hkv:])]
        k, v = (np.repeat(t, H // Hkv, 1) for t in held)
        z = np.einsum("ihd,jhd->hij", q, k) / math.sqrt(D) + np.triu(np.full((n, n), -np.inf), 1)
        p = np.exp(z - z.max(-1, keepdims=True))
        a = np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), v).reshape(n, H * D)
        x = x + a @ w64(w["o"]).T
        h = _norm(x)
        gate = h @ w64(w["gate"]).T
        x = x + (gate / (1 + np.exp(-gate)) * (h @ w64(w["up"]).T)) @ w64(w["down"]).T
    return _norm(x) @ f(model.lm_head).T


def test_logits_of_ragged_requests(model, cuda):
    import torch

    rng = np.random.default_rng(1)
    seqs = [rng.integers(0, CFG["vocab"], n).tolist() for n in (37, 1, 100, 16)]
    want = [reference(model, s) for s in seqs]

    def check(got, rows):
        assert np.abs(got - rows).max() <= 2e-2 * np.abs(rows).max()

    # prompts in two parts, then single tokens with one request rolled back and one finished
    first = [20, 1, 61, 0, 0]
    flat = [t for s, n in zip(seqs, first) for t in s[:n]]
    got = model.forward(torch.tensor(flat, device=cuda), [0] * 5, first).cpu().numpy()
    at = 0
    for b, n in enumerate(first[:4]):
        if n:
            check(got[at:at + n], want[b][:n])
            at += n
    ctx, new = [12, 0, 61, 0, 0], [25, 0, 39, 16, 0]  # request 0 takes 8 positions again
    flat = [t for s, c, n in zip(seqs, ctx, new) for t in s[c:c + n]]
    got = model.forward(torch.tensor(flat, device=cuda), ctx, new).cpu().numpy()
    at = 0
    for b in (0, 2, 3):
        check(got[at:at + new[b]], want[b][ctx[b]:ctx[b] + new[b]])
        at += new[b]
    model._plan([0] * 5, [0] * 5)
    assert int(model.count) == 64 and sorted(model.free.tolist()) == list(range(64))


def test_drafts_change_passes_and_not_tokens(model):
    """At a temperature that leaves one word a time, drafts give the same tokens in fewer passes."""
    prompts = [[5, 6, 7, 8, 5, 6, 7, 8, 5], [40], [3, 9] * 20]
    plain, n0 = model.generate(prompts, 40, drafts=0, temperature=1e-4)
    drafted, n4 = model.generate(prompts, 40, drafts=4, temperature=1e-4)
    assert [len(t) for t in plain] == [40, 40, 40]
    assert drafted == plain
    assert n0 == 40 and n4 <= n0
    assert int(model.count) == 64


def test_no_room_raises_and_changes_nothing(model, tb):
    import torch

    before = model.table.clone(), model.free.clone(), int(model.count)
    with pytest.raises(tb.ShapeError):
        model.forward(torch.zeros(256 * 5, dtype=torch.int64, device="cuda"), [0] * 5, [256] * 5)
    assert torch.equal(model.table, before[0]) and torch.equal(model.free, before[1]) and int(model.count) == before[2]
    with pytest.raises(tb.ShapeError):
        model.generate([[1]] * 6, 3)


def test_command_runs(cuda, capsys):
    from tendo_b200 import paged

    paged.main()
    out = capsys.readouterr().out
    assert "256 of 256 pages free" in out


def test_nothing_runs_past_the_longest_sequence(cuda, tb):
    """max_seq that is no multiple of the block: a request may fill it and not one position more, although the
    block table's last page reaches further than the RoPE tables."""
    import torch

    from tendo_b200.paged import PagedLlama

    model = PagedLlama(dict(CFG, layers=1, max_seq=37), num_blocks=8, block_size=16, max_requests=2, seed=3)
    rng = np.random.default_rng(2)
    seq = rng.integers(0, CFG["vocab"], 38).tolist()
    ids = lambda a, b: torch.tensor(seq[a:b], device=cuda)  # noqa: E731
    got = model.forward(ids(0, 37), [0, 0], [37, 0]).cpu().numpy()
    want = reference(model, seq[:37])
    assert np.abs(got - want).max() <= 2e-2 * np.abs(want).max()
    before = model.table.clone(), int(model.count), list(model.held)
    with pytest.raises(tb.ShapeError):
        model.forward(ids(37, 38), [37, 0], [1, 0])
    assert torch.equal(model.table, before[0]) and int(model.count) == before[1] and model.held == before[2]
    with pytest.raises(tb.ShapeError):
        model.generate([seq[:5], seq[:30]], 9)  # 38 positions; the last token's own is never taken
    out, _ = model.generate([seq[:5], seq[:30]], 8, drafts=4)
    assert [len(t) for t in out] == [8, 8] and int(model.count) == 8


def test_generate_refuses_what_it_cannot_sample(model, tb):
    """A prompt without tokens has no distribution to draw from, and a temperature must be above 0."""
    with pytest.raises(tb.ShapeError):
        model.generate([[], [1, 2]], 3)
    for t in (0.0, -1.0, float("nan")):
        with pytest.raises(tb.ShapeError):
            model.generate([[1, 2]], 3, temperature=t)
    assert int(model.count) == 64


def test_drafts_are_accepted_and_refused(model, monkeypatch):
    """Greedy continuations of three prompts, whose best word leads by 0.0069 of logits up to 1.5 all the way (a
    few 1e-4 is what another grouping of rows moves them by): drafts taken from them are accepted, so there are
    fewer passes; drafts of other tokens are refused, and their positions taken again."""
    prompts = [[431, 41, 490, 413],
               [317, 471, 392, 63, 18, 432, 203, 29, 238, 190, 215, 214, 157, 244, 245, 488, 346, 387, 4, 154, 491],
               [318, 255, 134, 153, 20, 37, 8, 87, 406, 324, 456, 251, 303, 485, 364, 316, 271, 279, 467, 138, 407, 335,
                1, 197, 428]]
    plain, n0 = model.generate(prompts, 40, drafts=0, temperature=1e-5)
    text = [p + t for p, t in zip(prompts, plain)]
    assert n0 == 40

    def lookup(seq, most, wrong):
        """What follows, with every `wrong`-th position's token another one."""
        s = next(t for t in text if t[:len(seq)] == seq)
        ahead = enumerate(s[len(seq):len(seq) + most], len(seq))
        return [(x + 1) % CFG["vocab"] if wrong and i % wrong == 0 else x for i, x in ahead]

    passes = {}
    for wrong in (0, 3, 1):  # none, every third, all
        monkeypatch.setattr(model, "lookup", lambda seq, most, w=wrong: lookup(seq, most, w))
        tokens, passes[wrong] = model.generate(prompts, 40, drafts=4, temperature=1e-5)
        assert tokens == plain
        assert int(model.count) == 64
    # all accepted: the prompt's pass, then five tokens a pass; all refused: a token a pass
    assert passes[0] == 1 + 8 and passes[0] < passes[3] < passes[1] == 40
