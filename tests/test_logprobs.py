"""Log probabilities of given tokens, entropies and the likeliest tokens, against 64 bits.

Tolerances.  With t = x - m, exact to 2^-24 of itself, log p = t - log S.  A term e^t of S is off by |t| 2^-24 (its argument) and a few 2^-24,
where terms count |t| is below 128; a lane adds V / 512 of them or fewer, each sum off by 2^-24: S is off by (V / 512 + 160) 2^-24 of itself, and log S by that.
(Where S is near 1, log S is the sum of the other terms.)  The entropy is log S - A / S, A a sum of t e^t of one sign: A / S, below 16 here, is off by as much of
itself.  Then four roundings of the result."""
import math

import pytest
import torch

DEV = "cuda:0"
F32 = torch.float32


@pytest.fixture(scope="module")
def ops():
    from palm_infra_amd.kernels import ops
    return ops


def plain(x, tokens, top):
    x = x.double()
    t = x - x.amax(1, keepdim=True)                     # (x less the sum's logarithm itself loses it beside logits of 1e38, in 64 bits too)
    logp = t - t.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0 * p).sum(1)
    bad = x.isnan().any(1) | (x == math.inf).any(1) | (x == -math.inf).all(1)
    entropy[bad] = math.nan
    logp[bad] = math.nan
    t = tokens.long()
    given = torch.where((t >= 0) & (t < x.shape[1]), logp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0], math.nan)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return given, entropy, ids, logp.gather(1, ids), bad


def near(got, want, V, parts=1.0):
    off = 2.0 ** -24 * ((V / 512 + 160) * parts + 4 * want.abs().nan_to_num(0, 0, 0))
    return bool(((got.double() == want) | (got.isnan() & want.isnan()) | ((got.double() - want).abs() <= off)).all())


def check(ops, x, tokens, top):
    given, entropy, ids, best = ops.token_logprobs(x.to(DEV), tokens.to(DEV), top)
    w_given, w_entropy, w_ids, w_best, bad = plain(x, tokens, top)
    V = x.shape[1]
    assert near(given.cpu(), w_given, V) and near(entropy.cpu(), w_entropy, V, 17.0) and near(best.cpu(), w_best, V)
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu().long()[~bad], w_ids[~bad])
    assert ids.numel() == 0 or (int(ids.min()) >= 0 and int(ids.max()) < x.shape[1])


def logits(n, V, seed, kind):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=g) * 3
    if kind == "sure":
        x[torch.arange(n), torch.randint(0, V, (n,), generator=g)] += torch.linspace(5, 60, n)
    elif kind == "rounded":
        x = x.bfloat16().float()
    elif kind == "equal":
        x = torch.full((n, V), -0.75)
        x[:, ::3] = 0.0
        x[:, ::6] = -0.0
    elif kind == "rising":
        x = torch.arange(V).float().expand(n, V).contiguous() * 1e-3
    elif kind == "falling":
        x = torch.arange(V).flip(0).float().expand(n, V).contiguous() * 1e-3
    elif kind == "masked":
        x[torch.rand(n, V, generator=g) < 0.98] = -math.inf
        x[:, V // 2] = 1.0
        x[0] = -math.inf
        x[0, V - 1] = 3.0
    elif kind == "lowest":
        x[:, 1:] = torch.finfo(F32).min
        x[n // 2] = torch.finfo(F32).min
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["random", "sure", "rounded", "equal", "rising", "falling", "masked", "lowest"])
@pytest.mark.parametrize("n,V", [(1, 1), (2, 7), (3, 64), (5, 1000), (1, 4097), (4, 50257), (2, 151936), (300, 1025), (257, 9001), (260, 3)])
def test_against_64_bits(ops, n, V, kind):
    x = logits(n, V, n + V, kind)
    tokens = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    tokens[0] = x[0].argmax()
    for top in (0, 1, 5, 20, 64):
        if top <= V:
            check(ops, x, tokens, top)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["random", "rounded", "equal", "masked", "lowest"])
@pytest.mark.parametrize("n,V", [(1, 32768), (7, 20001), (1, 32769), (5, 33001), (100, 40000), (175, 32769), (176, 32769), (239, 32770), (240, 32769)])
def test_by_slices_and_a_block_for_each_row(ops, n, V, kind):
    """At both sides of where the one begins and the other ends."""
    x = logits(n, V, n + V, kind)
    tokens = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    for top in (0, 5, 64):
        check(ops, x, tokens, top)


@pytest.mark.gpu
def test_rows_that_are_none_by_slices(ops):
    x = logits(6, 60000, 3, "random")
    x[0] = -math.inf
    x[1, 59999] = math.nan
    x[2, 5] = math.inf
    x[3, :1024] = -math.inf
    x[4, 700:] = -math.inf
    tokens = torch.tensor([0, 1, 5, 0, 1999, -1], dtype=torch.int32)
    check(ops, x, tokens, 20)
    given, entropy, ids, best = ops.token_logprobs(x.to(DEV), tokens.to(DEV), 3)
    assert given[3] == -math.inf and given[4] == -math.inf and bool(given[5].isnan()) and bool(entropy[:3].isnan().all()) and bool(best[:3].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["random", "rounded", "masked"])
@pytest.mark.parametrize("n,V", [(1, 262143), (2, 262145), (3, 400001), (1, 1500007), (180, 151936), (180, 262144), (241, 262145), (177, 300001)])
def test_large_vocabularies(ops, n, V, kind):
    """Groups of more than 16 logits, and as many of them as a block holds; some of the rows are looked at."""
    some = sorted({0, n // 2, n - 1})
    x = torch.randn(n, V, generator=torch.Generator().manual_seed(V))
    x[some] = logits(len(some), V, n, kind)
    tokens = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    x_dev, t_dev = x.to(DEV), tokens.to(DEV)
    for top in (0, 20, 64):
        given, entropy, ids, best = [t[some].cpu() for t in ops.token_logprobs(x_dev, t_dev, top)]
        w_given, w_entropy, w_ids, w_best, _ = plain(x[some], tokens[some], top)
        assert near(given, w_given, V) and near(entropy, w_entropy, V, 17.0) and near(best, w_best, V)
        assert torch.equal(ids.long(), w_ids)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 300])
def test_rows_that_are_none(ops, n):
    x = logits(n, 2000, 3, "random")
    x[0] = -math.inf
    x[1, 1999] = math.nan
    x[2, 5] = math.inf
    x[3, :1024] = -math.inf
    x[4, 700:] = -math.inf
    tokens = torch.tensor([0, 1, 5, 0, 1999] + [1] * (n - 5), dtype=torch.int32)
    check(ops, x, tokens, 20)
    given, entropy, ids, best = ops.token_logprobs(x.to(DEV), tokens.to(DEV), 3)
    assert given[3] == -math.inf and given[4] == -math.inf and bool(entropy[:3].isnan().all()) and bool(best[:3].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 256])
def test_tokens_outside_the_vocabulary_and_none(ops, n):
    x = logits(n, 300, 3, "random")
    tokens = torch.tensor([-1, 300, 299, 2 ** 31 - 1] + [0] * (n - 4), dtype=torch.int32)
    given, entropy, ids, best = ops.token_logprobs(x.to(DEV), tokens.to(DEV), 2)
    assert given.isnan().tolist() == [True, True, False, True] + [False] * (n - 4)
    none, entropy2, ids2, best2 = ops.token_logprobs(x.to(DEV), None, 2)
    assert none is None and torch.equal(entropy, entropy2) and torch.equal(ids, ids2) and torch.equal(best, best2)


@pytest.mark.gpu
def test_a_sure_model_is_not_rounded_away(ops):
    """log p of a token of probability 1 - 1e-6 to five places."""
    x = torch.zeros(3, 151936)
    x[:, 77] = torch.tensor([math.log(151935.0 * 10 ** e) for e in (4, 6, 8)])
    given, entropy, _, _ = ops.token_logprobs(x.to(DEV), torch.full((3,), 77, dtype=torch.int32, device=DEV))
    want, went = plain(x, torch.full((3,), 77), 0)[:2]
    assert bool(((given.cpu().double() - want).abs() <= 2e-5 * want.abs()).all()) and bool(((entropy.cpu().double() - went).abs() <= 2e-5 * went.abs()).all())


@pytest.mark.gpu
def test_the_same_row_alone_and_among_others_and_captured(ops):
    x = logits(300, 5000, 4, "rounded").to(DEV)
    tokens = torch.arange(300, dtype=torch.int32, device=DEV)
    many = ops.token_logprobs(x, tokens, 8)
    few = ops.token_logprobs(x[:9], tokens[:9], 8)
    assert torch.equal(many[2][:9], few[2])
    for a, b in ((many[0][:9], few[0]), (many[1][:9], few[1]), (many[3][:9], few[3])):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    y = x[:9].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.token_logprobs(y, tokens[:9], 8)
    for turn in range(3):
        y.copy_(x[9 * turn:9 * turn + 9])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, ops.token_logprobs(x[9 * turn:9 * turn + 9].contiguous(), tokens[:9], 8)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_no_rows(ops):
    given, entropy, ids, best = ops.token_logprobs(torch.empty((0, 10), device=DEV), torch.empty((0,), dtype=torch.int32, device=DEV), 4)
    assert given.shape == entropy.shape == (0,) and ids.shape == best.shape == (0, 4)


def test_refusals(ops, monkeypatch):
    x, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="GPU only"):
        ops.token_logprobs(x, t)
    monkeypatch.setattr(ops, "_dev", lambda what, *tensors: None)
    for args, match in (((x[0], t, 0), "not float32 \\[rows, vocab\\]"), ((x.double(), t, 0), "not float32"), ((x, t.long(), 0), "int32"), ((x, t[:1], 0), "for 2 rows"),
                        ((x, t, 11), "11 likeliest of 10"), ((x, t, -1), "-1 likeliest"), ((torch.zeros(2, 100), t, 65), "64 at most")):
        with pytest.raises(ops.KernelError, match=match):
            ops.token_logprobs(*args)
