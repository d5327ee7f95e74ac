"""Windowed streams that keep their first positions, branches of a sequence and log probabilities, as a user has them: through the engine,
the generation loop and the command line, one, two and all three together, against the plain implementation."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import plain_qwen3 as P
import tiny

ROOT = Path(__file__).resolve().parent.parent
CASES = [(name, dtype) for name in ("A", "B", "C", "D") for dtype in ("float32", "bfloat16")]
_engines = {}


def engine_for(model_dirs, name, dtype, window=None, kept=0, **more):
    from palm_infra_amd.engine import Engine
    key = (name, dtype, window, kept, tuple(sorted(more.items())))
    if key not in _engines:
        _engines[key] = Engine.from_dir(model_dirs[name][dtype], dtype=dtype, window=window, kept=kept, **{"max_tokens": 64 * 24, **more})
    return _engines[key]


def plain_logits(model_dirs, name, dtype, ids, window=None, kept=0):
    """The plain implementation's logits with the mask of a window and first positions."""
    def attention(q, k, v, scale, _=None):
        n, nh, hd = q.shape
        group = nh // k.shape[1]
        i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
        seen = (j <= i) & ((j > i - window) | (j < kept)) if window else j <= i
        out = torch.zeros(n, nh, hd, dtype=torch.float64)
        for h in range(nh):
            s = (q[:, h].double() @ k[:, h // group].double().T * scale).masked_fill(~seen, -math.inf)
            out[:, h] = torch.softmax(s, -1) @ v[:, h // group].double()
        return out
    cfg, w = P.read_model(model_dirs[name][dtype])
    real, P.causal_attention = P.causal_attention, attention
    try:
        return P.logits(cfg, w, ids)
    finally:
        P.causal_attention = real


# ---- streams --------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("name,dtype", CASES)
@pytest.mark.parametrize("window,kept", [(20, 3), (64, 64), (33, 70), (10, 0)])
def test_prompts_whole_in_pieces_and_token_by_token(model_dirs, name, dtype, window, kept):
    from palm_infra_amd.engine import StepEntry
    eng = engine_for(model_dirs, name, dtype, window, kept)
    pool = tiny.LogitsPool(dtype, f"{name} window {window} kept {kept}")
    a, b, c = tiny.prompts(name, [200, 90, 150], seed=7)
    refs = [plain_logits(model_dirs, name, dtype, ids, window, kept) for ids in (a, b, c)]
    slots = [eng.open() for _ in range(3)]
    cuts = [120, 90, 1]                                      # two prompts, one whole, and a first token, in one step
    got = eng.step([StepEntry(s, ids[:n], list(range(n))) for s, ids, n in zip(slots, (a, b, c), cuts)])
    row = 0
    for ref, n in zip(refs, cuts):
        pool.add(got[row:row + n], ref[:n])
        row += n
    got = eng.step([StepEntry(slots[0], a[120:157], list(range(37))), StepEntry(slots[2], c[1:4], [0, 1, 2])])
    pool.add(got, torch.cat([refs[0][120:157], refs[2][1:4]]))
    for t in range(40):                                      # single tokens, recorded from the second on
        got = eng.step([StepEntry(slots[0], [a[157 + t]], [0]), StepEntry(slots[2], [c[4 + t]], [0])])
        pool.add(got, torch.stack([refs[0][157 + t], refs[2][4 + t]]))
    pool.check()
    for g in eng.cache.paged_groups:
        assert sum(p >= 0 for p in g.table.slot_pages[slots[0]]) <= (window + 62) // 64 + 1 + (kept + 63) // 64
    for s in slots:
        eng.close(s)
    eng.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_stream_longer_than_the_cache(model_dirs, dtype):
    """1,900 tokens through a cache of 1,408: the window moves on, the first positions stay."""
    from palm_infra_amd.engine import StepEntry
    eng = engine_for(model_dirs, "D", dtype, 50, 4, max_tokens=64 * 22, stream_tokens=1950)
    ids = tiny.prompts("D", [1900], seed=3)[0]
    ref = plain_logits(model_dirs, "D", dtype, ids, 50, 4)
    slot = eng.open()
    pool = tiny.LogitsPool(dtype, "a stream")
    pool.add(eng.step([StepEntry(slot, ids[:1860], [0, 700, 1500, 1859])]), ref[[0, 700, 1500, 1859]])
    for t in range(1860, 1900):
        pool.add(eng.step([StepEntry(slot, [ids[t]], [0])]), ref[t:t + 1])
    pool.check()
    assert eng.length(slot) == 1900 and eng.cache.paged_groups[0].table.pages.held_count <= 3
    eng.close(slot)
    results, _ = eng.generate([ids[:1500], ids[:40]], temperature=0.0, max_new_tokens=30, ignore_eos=True)
    assert [len(r.token_ids) for r in results] == [30, 30]
    eng.cache.check()
    assert eng.cache.slots.held_count == 0


def test_a_window_is_for_designs_without_windows_of_their_own():
    from palm_infra_amd.config import ConfigError, config_from_dict, preset_dict
    from palm_infra_amd.engine import Engine
    cfg = config_from_dict(tiny.CONFIGS["A"])
    windowed = cfg.with_window(64, 4)
    assert windowed.spec().layers[0].parts["mixer"].params["window"] == 64 and windowed.spec().layers[0].parts["mixer"].params["kept"] == 4
    assert cfg.spec().layers[0].parts["mixer"].params["window"] is None and windowed.to_dict() == cfg.to_dict()
    assert Engine._windowed(cfg, None, 0) is cfg
    for window, kept in ((0, 0), (-5, 0), (10, -1)):
        with pytest.raises(ConfigError):
            cfg.with_window(window, kept)
    with pytest.raises(ValueError, match="stand behind a window"):
        Engine._windowed(cfg, None, 4)
    with pytest.raises(ValueError, match="part of the model"):
        Engine._windowed(config_from_dict(preset_dict("tiny-biguzen")), 64, 4)


# ---- branches -------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("name,dtype", CASES)
@pytest.mark.parametrize("length", [5, 64, 100])
def test_branches_go_on_as_the_sequence_would(model_dirs, name, dtype, length):
    from palm_infra_amd.engine import StepEntry
    eng = engine_for(model_dirs, name, dtype)
    ids, other, third = (tiny.prompts(name, [n], seed=s)[0] for n, s in ((length + 24, 1), (24, 2), (24, 3)))
    ways = [ids, ids[:length] + other, ids[:length] + third]
    refs = [plain_logits(model_dirs, name, dtype, w) for w in ways]
    slot = eng.open()
    eng.step([StepEntry(slot, ids[:length], [length - 1])])
    slots = [slot] + eng.fork(slot, 2)
    pool = tiny.LogitsPool(dtype, f"{name} branches at {length}")
    for t in range(length, length + 20):
        got = eng.step([StepEntry(s, [w[t]], [0]) for s, w in zip(slots, ways)])
        pool.add(got, torch.stack([r[t] for r in refs]))
        if t == length + 7:
            eng.close(eng.open())
            eng.compact()
    got = eng.step([StepEntry(s, w[length + 20:], [3]) for s, w in zip(slots, ways)])
    pool.add(got, torch.stack([r[length + 23] for r in refs]))
    pool.check()
    eng.cache.check()
    for s in slots:
        eng.close(s)
    eng.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("preset", ["tiny-sebesun", "tiny-pazilorn", "tiny-matalix", "tiny-biguzen", "tiny-vovalix", "tiny-nirotar"])
def test_branches_of_every_design(preset, dtype):
    """States, compressed rows and windowed keys too: a branch's tokens are those of the whole sequence run by itself."""
    from palm_infra_amd.config import config_from_dict, preset_dict
    from palm_infra_amd.engine import Engine, StepEntry
    eng = Engine.from_config(config_from_dict(preset_dict(preset)), seed=2, dtype=dtype, max_tokens=64 * 16)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, eng.vocab_size, (90,), generator=g).tolist()
    more = torch.randint(0, eng.vocab_size, (2, 12), generator=g).tolist()

    def run(tokens, fork_at=None):
        slot = eng.open()
        eng.step([StepEntry(slot, tokens[:77], [])])
        if fork_at is not None:
            branch, = eng.fork(slot)
            # the first sequence goes on by itself, then makes way
            eng.step([StepEntry(slot, [7], [0])])
            eng.step([StepEntry(slot, [9], [0])])
            eng.close(slot)
            eng.compact()
            slot = branch
        out = [eng.step([StepEntry(slot, [t], [0])])[0].clone() for t in tokens[77:]]
        eng.close(slot)
        eng.cache.check()
        return torch.stack(out)
    for tail in more:
        assert torch.equal(run(ids[:77] + tail), run(ids[:77] + tail, fork_at=77))


@pytest.mark.gpu
def test_several_answers_are_those_of_the_prompt_given_several_times(model_dirs):
    """The draws of answer j of prompt i are stream i * answers + j's: as if each answer were a request of its own."""
    eng = engine_for(model_dirs, "D", "float32")
    prompts = tiny.prompts("D", [70, 5, 64], seed=4)
    for options in (dict(temperature=0.8, seed=3), dict(temperature=0.8, seed=3, repeat_penalty=1.3), dict(temperature=0.0)):
        apart, _ = eng.generate([p for p in prompts for _ in range(3)], max_new_tokens=20, ignore_eos=True, max_batch=9, **options)
        got, metrics = eng.generate(prompts, max_new_tokens=20, ignore_eos=True, max_batch=9, answers=3, **options)
        assert [r.token_ids for r in got] == [r.token_ids for r in apart] and len(got) == 9
        assert metrics.generated_tokens == 180
        few, _ = eng.generate(prompts, max_new_tokens=20, ignore_eos=True, max_batch=4, answers=3, **options)      # a prompt at a time
        assert [r.token_ids for r in few] == [r.token_ids for r in apart]
    eng.cache.check()
    assert eng.cache.slots.held_count == 0


# ---- log probabilities ----------------------------------------------------------------------------------------------

def plain_scores(ref, following):
    logp = torch.log_softmax(ref.double(), -1)
    return logp[torch.arange(len(following)), torch.tensor(following)], -(logp.exp() * logp).sum(-1), logp


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_scores_of_given_tokens(model_dirs, name):
    """float32 logits are within 1e-4 of the plain ones, so a log probability is within twice that (its own logit and the sum's), and an entropy by 2e-4 times
    the spread of log p."""
    eng = engine_for(model_dirs, name, "float32")
    prompts = tiny.prompts(name, [100, 1, 37, 2], seed=9)
    for pieces in (2048, 30):
        eng.SCORED_ROWS = pieces
        for ids, s in zip(prompts, eng.score(prompts, 4)):
            assert len(s.logprobs) == len(s.entropies) == len(s.alternatives) == len(ids) - 1
            if len(ids) == 1:
                assert s.total == 0.0
                continue
            given, entropy, logp = plain_scores(plain_logits(model_dirs, name, "float32", ids)[:-1], ids[1:])
            assert float((torch.tensor(s.logprobs) - given).abs().max()) <= 2.1e-4
            assert bool(((torch.tensor(s.entropies) - entropy).abs() <= 2.1e-4 * (1 + logp.abs().amax(-1))).all())
            assert abs(s.total - float(given.sum())) <= 2.1e-4 * len(ids)
            for row, others in zip(logp, s.alternatives):
                assert [p for _, p in others] == sorted((p for _, p in others), reverse=True)
                assert all(abs(float(row[t]) - p) <= 2.1e-4 for t, p in others)
                assert float(row.topk(4).values[-1]) - others[-1][1] <= 4.2e-4
    eng.SCORED_ROWS = type(eng).SCORED_ROWS
    assert eng.cache.slots.held_count == 0
    with pytest.raises(ValueError, match="at least one token"):
        eng.score([[]])
    with pytest.raises(ValueError, match="outside the vocabulary"):
        eng.score([[1, eng.vocab_size]])
    with pytest.raises(ValueError, match="outside the vocabulary"):
        eng.score([[1, -1, 2]])
    with pytest.raises(ValueError, match="alternatives"):
        eng.score([[1, 2]], 65)
    assert eng.cache.slots.held_count == 0


@pytest.mark.gpu
@pytest.mark.parametrize("options", [dict(temperature=0.0), dict(temperature=0.9, seed=1), dict(temperature=0.9, presence_penalty=0.5)])
def test_generation_tells_what_scoring_its_result_tells(model_dirs, options):
    eng = engine_for(model_dirs, "D", "float32")
    prompts = tiny.prompts("D", [9, 70], seed=5)
    plain, _ = eng.generate(prompts, max_new_tokens=15, ignore_eos=True, **options)
    got, _ = eng.generate(prompts, max_new_tokens=15, ignore_eos=True, logprobs=3, **options)
    assert [r.token_ids for r in got] == [r.token_ids for r in plain] and plain[0].scores is None
    for p, r, s in zip(prompts, got, eng.score([p + r.token_ids for p, r in zip(prompts, got)], 3)):
        assert len(r.scores.logprobs) == len(r.scores.alternatives) == 15
        tail = len(p) - 1
        assert torch.allclose(torch.tensor(r.scores.logprobs), torch.tensor(s.logprobs[tail:]), atol=4.2e-4, rtol=0)
        if options["temperature"] == 0.0:
            assert [a[0][0] for a in r.scores.alternatives] == r.token_ids
    with pytest.raises(ValueError, match="0 to 64"):
        eng.generate(prompts, logprobs=65)


# ---- together -------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_likeliest_of_several_endless_answers(model_dirs, dtype):
    """A prompt runs once, its sequence is forked, the branches run on as windowed streams longer than the cache, and their log probabilities choose among
    them: as the same with every answer a request of its own, and as the plain implementation scores them."""
    eng = engine_for(model_dirs, "D", dtype, 40, 4, max_tokens=64 * 120, stream_tokens=64 * 150)
    prompt = tiny.prompts("D", [150], seed=6)[0]
    options = dict(max_new_tokens=60, ignore_eos=True, temperature=0.9, seed=5, logprobs=2)
    apart, _ = eng.generate([prompt] * 4, **options)
    got, _ = eng.generate([prompt], answers=4, **options)
    if dtype == "float32":
        assert [r.token_ids for r in got] == [r.token_ids for r in apart]
    assert len({tuple(r.token_ids) for r in got}) > 1
    for r in got:
        ids = prompt + r.token_ids
        ref = plain_logits(model_dirs, "D", dtype, ids, 40, 4)[len(prompt) - 1:-1]
        given = plain_scores(ref, r.token_ids)[0]
        near = 2.1e-4 if dtype == "float32" else 2 * tiny.BFLOAT16_MAX_REL * float(ref.double().pow(2).mean().sqrt())     # (two logits' errors)
        assert float((torch.tensor(r.scores.logprobs) - given).abs().max()) <= near
    best = max(range(4), key=lambda i: got[i].scores.total)
    rescored = eng.score([prompt + r.token_ids for r in got])
    totals = [sum(s.logprobs[len(prompt) - 1:]) for s in rescored]
    assert totals[best] >= max(totals) - (0.05 if dtype == "float32" else 60.0)
    eng.cache.check()
    assert eng.cache.slots.held_count == 0


@pytest.mark.gpu
def test_the_command_line(model_dirs):
    def chat(*args):
        r = subprocess.run([sys.executable, str(ROOT / "bin" / "palm_chat"), "--package", str(model_dirs["D"]["float32"]), "--dtype", "float32", *args],
                           capture_output=True, text=True, timeout=110)
        return r.returncode, r.stdout, r.stderr
    rc, out, err = chat("--prompt-ids", "1,2,3,4", "--max-new-tokens", "5", "--temperature", "0", "--ignore-eos", "--answers", "2", "--logprobs", "1",
                        "--window", "64", "--kept", "4", "--n-ctx", "4096", "--stream-tokens", "9000")
    assert rc == 0, err
    lines = out.strip().splitlines()
    assert lines[0].startswith("[0] ") and lines[1].startswith("[1] ") and lines[0][4:] == lines[1][4:]
    assert lines[2].startswith("[0] total -") and "of 5 tokens" in lines[2] and "entropy" in lines[3]
    rc, out, err = chat("--prompt-ids", "1,2,3,4", "--score", "--logprobs", "2")
    assert rc == 0 and out.startswith("[0] total -") and len(out.strip().splitlines()) == 4, err
    rc, out, err = chat("--prompt-ids", "1,2", "--kept", "4")
    assert rc == 1 and "stand behind a window" in err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("preset", ["tiny-sebesun", "tiny-pazilorn", "tiny-vovalix"])
def test_branches_of_designs_whose_convolutions_have_one_tap(preset, dtype):
    """Such a convolution keeps no earlier inputs: its state has no elements."""
    from palm_infra_amd.config import config_from_dict, preset_dict
    from palm_infra_amd.engine import Engine, StepEntry

    def one_tap(x):
        if isinstance(x, dict):
            return {k: 1 if k == "conv" and v is not None else one_tap(v) for k, v in x.items()}
        return [one_tap(v) for v in x] if isinstance(x, list) else x
    eng = Engine.from_config(config_from_dict(one_tap(preset_dict(preset))), seed=2, dtype=dtype, max_tokens=64 * 16)
    assert any(g.table is None and g.data.numel() == 0 for g in eng.cache.groups)
    ids = torch.randint(0, eng.vocab_size, (90,), generator=torch.Generator().manual_seed(5)).tolist()

    def run(fork):
        slot = eng.open()
        eng.step([StepEntry(slot, ids[:77], [])])
        if fork:
            branch, = eng.fork(slot)
            eng.step([StepEntry(slot, [7], [0])])
            eng.close(slot)
            slot = branch
        out = torch.stack([eng.step([StepEntry(slot, [t], [0])])[0].clone() for t in ids[77:]])
        eng.close(slot)
        eng.cache.check()
        return out
    assert torch.equal(run(False), run(True))
    results, _ = eng.generate([ids[:9]], answers=2, temperature=0.0, max_new_tokens=3, ignore_eos=True)
    assert results[0].token_ids == results[1].token_ids and len(results[0].token_ids) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_totals_that_choose_among_answers_are_the_answers_own(model_dirs, dtype):
    """Each answer's log probabilities against 64 bits of the logits of the very steps that drew it, made again: the prompt once, the same forks, the four tokens together.

    Bounds.  The same steps give the same logits, so a log probability is off by the operator's own rounding, (V / 512 + 160 + 4 |log p|) 2^-24 (tests of
    ``token_logprobs``), a total by the sum of those.  Scoring the whole answer in pieces is another pass: logits of two passes are each within the gate's 5 % of
    their mean square of the exact ones (bfloat16; 1e-4 in float32), a log probability is a logit less a mean of logits, so a total of 60 is off by 60 x 2 x 2 of that
    if every error had one sign."""
    from palm_infra_amd.engine import StepEntry
    eng = engine_for(model_dirs, "D", dtype, 40, 4, max_tokens=64 * 120, stream_tokens=64 * 150)
    prompt = tiny.prompts("D", [150], seed=8)[0]
    got, _ = eng.generate([prompt], answers=4, max_new_tokens=60, ignore_eos=True, temperature=0.9, seed=7, logprobs=0)
    slot = eng.open()
    logits = eng.step([StepEntry(slot, prompt, [len(prompt) - 1])])
    slots = [slot] + eng.fork(slot, 3)
    rows = [logits.repeat_interleave(4, dim=0)]
    for t in range(59):
        rows.append(eng.step([StepEntry(s, [r.token_ids[t]], [0]) for s, r in zip(slots, got)]).clone())
    for s in slots:
        eng.close(s)
    rows = torch.stack(rows).double().cpu()                                     # [tokens, answers, vocabulary]
    tokens = torch.tensor([r.token_ids for r in got]).T
    exact = torch.log_softmax(rows, -1).gather(2, tokens[..., None])[..., 0]
    told = torch.tensor([r.scores.logprobs for r in got], dtype=torch.float64).T
    off = (rows.shape[2] / 512 + 160 + 4 * exact.abs()) * 2.0 ** -24
    assert bool(((told - exact).abs() <= off).all())
    totals, room = exact.sum(0), float(off.sum(0).max())
    best = max(range(4), key=lambda i: got[i].scores.total)
    assert float(totals[best]) >= float(totals.max()) - 2 * room
    # (another answer's total is not within it: the comparison tells them apart)
    assert float((totals.sort().values[1:] - totals.sort().values[:-1]).min()) > 4 * room
    logit_off = 1e-4 if dtype == "float32" else tiny.BFLOAT16_RMS_REL * float(rows.pow(2).mean().sqrt())
    rescored = [sum(s.logprobs[len(prompt) - 1:]) for s in eng.score([prompt + r.token_ids for r in got])]
    bound = 60 * 2 * 2 * logit_off
    assert all(abs(r.scores.total - s) <= bound for r, s in zip(got, rescored))
    assert rescored[best] >= max(rescored) - 2 * bound
