"""Attention with a window and first positions that stay visible, against its definition in 64 bits.

The pages that no query sees are one page full of NaN, and so is what lies behind each sequence's end: what is read of them shows.

Tolerances, for an output o = sum w v of weights that sum to one.  A score is a sum of hd products, off by at most hd 2^-24 sum |q k| scale (each
of hd roundings relative to a partial sum), which scales its weight by e^(2 of those) at most, with the maximum's own; exponentials are off by
a few 2^-24 and a sum of N of them by N 2^-24.  bfloat16 on the matrix cores: a weight is rounded by 2^-8 relative to it, in the sum of weights too, and the
result once more by 2^-8 of itself."""
import math

import pytest
import torch

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from palm_infra_amd.kernels import ops
    return ops


class Case:
    """A step over a cache: ``seqs`` are (tokens before, new tokens)."""

    def __init__(self, seqs, nh, nkv, hd, window, kept, dtype, seed=0, q_scale=2.0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.nh, self.nkv, self.hd, self.window, self.kept, self.dtype = seqs, nh, nkv, hd, window, kept, dtype
        lists = []
        for start, new in seqs:
            pages, first = (start + new + 63) // 64, max(0, start - window + 1) // 64
            lists.append([p for p in range(pages) if new and (p < (kept + 63) // 64 or p >= first)])
        n_pages = sum(map(len, lists))
        width = max(max((s + n + 63) // 64 for s, n in seqs), 1)
        order = torch.randperm(n_pages, generator=g).tolist()
        slots = torch.randperm(len(seqs) + 2, generator=g).tolist()[:len(seqs)]
        self.table = torch.full((len(seqs) + 2, width), n_pages, dtype=torch.int32)
        self.k = torch.randn(n_pages + 1, nkv, 64, hd, generator=g).to(dtype)
        self.v = torch.randn(n_pages + 1, nkv, hd, 64, generator=g).to(dtype)
        self.k[n_pages], self.v[n_pages] = math.nan, math.nan
        for slot, pages, (start, new) in zip(slots, lists, seqs):
            for p in pages:
                self.table[slot, p] = order.pop()
            if pages and (start + new) % 64:
                last = self.table[slot, pages[-1]]
                self.k[last, :, (start + new) % 64:] = math.nan
                self.v[last, :, :, (start + new) % 64:] = math.nan
        self.cu = [0]
        for _, new in seqs:
            self.cu.append(self.cu[-1] + new)
        self.q = (torch.randn(self.cu[-1], nh * hd, generator=g) * q_scale).to(dtype)
        self.slots = slots

    def place(self, b, j):
        return int(self.table[self.slots[b], j // 64]), j % 64

    def run(self, ops, fn=None, **more):
        i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        fn = fn or ops.attention_kept
        return fn(self.q.to(DEV), self.k.to(DEV), self.v.to(DEV), self.table.to(DEV), i(self.slots), i([s for s, _ in self.seqs]),
                  i([n for _, n in self.seqs]), i(self.cu), max(n for _, n in self.seqs), max(s + n for s, n in self.seqs), self.nh, self.nkv,
                  self.hd, self.hd ** -0.5, self.window, self.kept, **more).cpu()

    def plain(self):
        """The results and how far a kernel's may be from them."""
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        off = torch.zeros_like(out)
        G, hd, scale = self.nh // self.nkv, self.hd, self.hd ** -0.5
        rounding = 2.0 ** -8 if self.dtype == BF16 else 2.0 ** -24
        for b, (start, new) in enumerate(self.seqs):
            for i in range(new):
                p = start + i
                keys = torch.arange(p + 1)
                keys = keys[(keys > p - self.window) | (keys < self.kept)]
                page, at = self.table[self.slots[b]].long()[keys // 64], keys % 64
                row = self.cu[b] + i
                q = self.q[row].double().view(self.nh, hd)
                k, v = self.k[page, :, at].double(), self.v[page, :, :, at].double()     # [keys, nkv, hd]
                k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
                s = (q * k).sum(-1) * scale                                           # [keys, nh]
                w = torch.softmax(s, 0)[..., None]
                o = (w * v).sum(0)
                ds = hd * 2.0 ** -24 * ((q * k).abs().sum(-1) * scale).amax(0)[:, None]
                weigh = (w * v.abs()).sum(0)
                e = weigh * (4 * ds + (len(keys) + 16) * 2.0 ** -24 + (2 * rounding if self.dtype == BF16 else 0)) + rounding * (o.abs() + weigh * 2 * rounding)
                out[row], off[row] = o.reshape(-1), e.reshape(-1)
        return out, off

    def check(self, got):
        want, off = self.plain()
        assert got.dtype == self.dtype and got.shape == self.q.shape
        same = torch.where(torch.isfinite(want), (got.double() - want).abs() <= off, (got.double() == want) | (got.isnan() & want.isnan()))
        assert bool(same.all()), (int((~same).sum()), float((got.double() - want).abs().nan_to_num(9e9).max()))


SHAPES = [(4, 2, 16), (5, 1, 64), (8, 8, 128), (6, 2, 20), (3, 1, 6), (40, 2, 32), (2, 1, 80), (4, 4, 192), (10, 2, 128), (4, 1, 512)]
LONG = [(4, 2, 64), (8, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("window,kept", [(1, 0), (1, 1), (5, 4), (64, 64), (100, 3), (70, 130), (4096, 4)])
def test_prompts_pieces_and_single_tokens(ops, nh, nkv, hd, window, kept, dtype):
    case = Case([(0, 1), (0, 70), (250, 17), (130, 0), (400, 1), (64, 64), (63, 2)], nh, nkv, hd, window, kept, dtype, seed=hd + window)
    case.check(case.run(ops))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("window,kept", [(1, 0), (1, 1), (5, 4), (64, 64), (100, 3), (70, 130), (4096, 4)])
def test_a_step_of_single_tokens(ops, nh, nkv, hd, window, kept, dtype):
    case = Case([(n, 1) for n in (0, 1, 63, 64, 65, 127, 500, 301, 200)], nh, nkv, hd, window, kept, dtype, seed=hd + window)
    case.check(case.run(ops))


@pytest.mark.gpu
@pytest.mark.parametrize("sequences", [2, 63, 64, 65, 130])
@pytest.mark.parametrize("nh,nkv,hd", LONG)
@pytest.mark.parametrize("plan", [None, (False, 1, 1), (False, 2, 3)])
def test_prompts_of_many_sequences_beside_single_tokens(ops, nh, nkv, hd, sequences, plan):
    """One long prompt (at either end or within), the others a token, some, or none."""
    for longest in (0, sequences // 2, sequences - 1):
        seqs = [(40 * b % 300, (0, 1, 33, 1)[b % 4]) for b in range(sequences)]
        seqs[longest] = (17, 300)
        case = Case(seqs, nh, nkv, hd, 100, 3, BF16, seed=longest)
        case.check(case.run(ops, plan=plan))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", LONG)
@pytest.mark.parametrize("seqs", [[(5000, 1)], [(3000, 1), (70, 1), (2047, 1)], [(3000, 5)], [(0, 700)], [(900, 300), (0, 65)]])
@pytest.mark.parametrize("window,kept", [(1000, 4), (2048, 129), (333, 64)])
def test_long_rows_of_pages(ops, nh, nkv, hd, seqs, window, kept, dtype):
    case = Case(seqs, nh, nkv, hd, window, kept, dtype, seed=len(seqs))
    case.check(case.run(ops))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 16), (8, 2, 64), (8, 2, 128), (6, 2, 20)])
@pytest.mark.parametrize("seqs", [[(0, 200)], [(300, 30), (290, 1)], [(310, 1), (200, 1)]])
def test_what_masked_places_hold_does_not_show(ops, nh, nkv, hd, seqs, dtype):
    """Infinities and NaN in keys and values: a query that sees such a value has it in its result, the others do not."""
    case = Case(seqs, nh, nkv, hd, 90, 3, dtype, seed=5)
    for b, (start, new) in enumerate(seqs):
        for j, what in ((20, math.inf), (100, math.nan), (150, -math.inf), (215, math.inf), (start + new - 2, math.nan)):
            page, at = case.place(b, j) if j < start + new else (len(case.k) - 1, 0)
            if page == len(case.k) - 1:
                continue
            case.v[page, 0, :3, at] = what
        for j in (40, 120):                                     # keys too, where no query's window reaches them
            if j < start - 90 and case.place(b, j)[0] != len(case.k) - 1:
                case.k[case.place(b, j)[0], :, j % 64] = math.nan
                case.v[case.place(b, j)[0], :, :, j % 64] = math.inf
    case.check(case.run(ops))


PAGED = [(4, 2, 64), (8, 8, 64), (8, 1, 64), (8, 2, 128), (5, 1, 128), (16, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", PAGED)
@pytest.mark.parametrize("lengths", [[0], [63], [64, 0], [5000], [0, 1, 63, 64, 65, 127, 500, 301, 200], [3000, 70, 2047], [n * 37 % 700 for n in range(128)]])
@pytest.mark.parametrize("window,kept", [(1, 0), (1, 1), (5, 4), (64, 64), (100, 3), (70, 130), (4096, 4)])
def test_single_tokens_cut_by_pages(ops, nh, nkv, hd, lengths, window, kept):
    """By pages, whatever the sizes; then with infinities and NaN where a query sees them, and where it does not."""
    case = Case([(n, 1) for n in lengths], nh, nkv, hd, window, kept, BF16, seed=hd + window + len(lengths))
    case.check(case.run(ops, by_pages=True))
    if len(lengths) > 16:
        return
    for b, n in enumerate(lengths):
        for j, what in ((2, math.inf), (n // 2, math.nan), (n - 70, -math.inf), (n - 101, math.inf)):
            if 0 <= j < n and case.place(b, j)[0] != len(case.k) - 1:
                case.v[case.place(b, j)[0], 0, :3, j % 64] = what
                if kept <= j <= n - window:                      # (a key that is not seen too)
                    case.k[case.place(b, j)[0], :, j % 64] = math.nan
    case.check(case.run(ops, by_pages=True))


@pytest.mark.gpu
@pytest.mark.parametrize("by_pages", [True, False, None])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (4, 2, 80)])
@pytest.mark.parametrize("counts", [[1, 0, 1, 0, 1, 1], [0, 0, 1], [1, 0, 0], [0, 0], [0, 1, 1, 1, 0], [n % 3 // 2 for n in range(128)], [int(n == 77) for n in range(128)],
                                    [int(n % 30 < 12) for n in range(100)]])
@pytest.mark.parametrize("rows", [0, 1, 200])
def test_single_tokens_of_some_sequences(ops, nh, nkv, hd, counts, dtype, by_pages, rows):
    """Sequences without a query (nothing is read of theirs) between the others, and rows behind the last, as many as make one for each sequence or more."""
    case = Case([(130 * n % 1700 + n, c) for n, c in enumerate(counts)], nh, nkv, hd, 200, 4, dtype, seed=len(counts))
    q = case.q
    behind = len(counts) - sum(counts) if rows == 1 else rows
    case.q = torch.cat([q, torch.full((behind, nh * hd), math.nan, dtype=dtype)])
    if case.q.shape[0] == 0:
        return
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    got = ops.attention_kept(case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), case.table.to(DEV), i(case.slots), i([s for s, _ in case.seqs]), i(counts), i(case.cu), 1,
                             max(s + n for s, n in case.seqs), nh, nkv, hd, hd ** -0.5, 200, 4, by_pages=by_pages).cpu()
    case.q = q
    case.check(got[:q.shape[0]])


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 80), (24, 2, 128), (140, 1, 64)])
def test_single_tokens_that_are_not_served_by_pages(ops, nh, nkv, hd):
    case = Case([(200, 1), (70, 1)], nh, nkv, hd, 90, 4, BF16, seed=1)
    assert torch.equal(case.run(ops, by_pages=True), case.run(ops, by_pages=False))


@pytest.mark.gpu
@pytest.mark.parametrize("by_pages", [True, False])
@pytest.mark.parametrize("planes", [0, 1, 2, 3])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (8, 1, 128)])
@pytest.mark.parametrize("window,kept", [(1, 1), (64, 64), (100, 3), (70, 130), (4096, 4)])
def test_from_the_projection(ops, nh, nkv, hd, window, kept, planes, by_pages):
    """The step that makes queries, keys and values of the joined projection's rows: the new ones arrive in the cache, nothing else is touched."""
    lengths = [0, 1, 63, 64, 300, 65, 500, 129, 1000]
    case = Case([(n, 1) for n in lengths], nh, nkv, hd, window, kept, BF16, seed=window + planes)
    k, v, B = case.k.clone(), case.v.clone(), len(lengths)
    new_k, new_v = torch.zeros(B, nkv, hd, dtype=BF16), torch.zeros(B, nkv, hd, dtype=BF16)
    for b, n in enumerate(lengths):
        page, at = case.place(b, n)
        new_k[b], new_v[b] = k[page, :, at], v[page, :, :, at]
        k[page, :, at], v[page, :, :, at] = math.nan, math.nan
    rows = torch.cat([case.q, new_k.flatten(1), new_v.flatten(1)], 1)
    if planes:                                                   # of which all but one are nothing: the sum is exact
        rows = torch.stack([rows.float() if p == planes // 2 else torch.zeros(rows.shape) for p in range(planes)])
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    k_dev, v_dev = k.to(DEV), v.to(DEV)
    got = ops.attention_decode_fused(rows.to(DEV), k_dev, v_dev, case.table.to(DEV), i(case.slots), i(lengths), nh, nkv, hd, hd ** -0.5, window, 3, kept=kept,
                                     pages=by_pages)
    case.check(got.cpu())
    bits = lambda t: t.cpu().view(torch.int16)
    assert torch.equal(bits(k_dev), bits(case.k)) and torch.equal(bits(v_dev), bits(case.v))


@pytest.mark.gpu
def test_a_captured_step_cut_by_pages_replays_with_new_contents(ops):
    starts = [500, 70, 1500, 0, 64, 900]
    cases = [Case([(n, 1) for n in starts], 8, 2, 128, 300, 4, BF16, seed=s) for s in (8, 9)]
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    held = [t.to(DEV) for t in (cases[0].q, cases[0].k, cases[0].v, cases[0].table)] + [i(cases[0].slots), i(starts), i([1] * 6), i(cases[0].cu)]
    args = (1, 1501, 8, 2, 128, 128 ** -0.5, 300, 4)
    ops.attention_kept(*held, *args, by_pages=True)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.attention_kept(*held, *args, by_pages=True)))
    for turn in range(4):
        now = cases[turn % 2]
        for t, new in zip(held, (now.q, now.k, now.v, now.table, torch.tensor(now.slots, dtype=torch.int32))):
            t.copy_(new.to(DEV))
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            now.check(out.cpu())
        now.check(ops.attention_kept(*held, *args, by_pages=True).cpu())


PLANS = [(False, 1, 1), (False, 2, 1), (False, 1, 3), (False, 2, 5), (False, 1, 16), (False, 2, 2), (True, 0, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (5, 1, 128), (24, 1, 64), (40, 1, 128), (2, 2, 64), (3, 1, 128), (140, 1, 64)])
@pytest.mark.parametrize("window,kept", [(40, 4), (200, 65)])
def test_every_way_a_prompt_goes(ops, nh, nkv, hd, window, kept, plan):
    """Two halves, slices (more of them than pages too), 64 columns a wave: whatever the plan, and with values that only some queries see."""
    if plan[0] and hd != 128:
        pytest.skip("heads of 128 only")
    case = Case([(0, 60), (500, 37), (130, 0), (320, 1)], nh, nkv, hd, window, kept, BF16, seed=nh)
    case.check(case.run(ops, plan=plan))
    for b, j in ((0, 10), (1, 480), (1, 520), (3, 300), (1, 2)):
        case.v[case.place(b, j)[0], 0, :5, j % 64] = math.inf if j % 20 else math.nan
    case.check(case.run(ops, plan=plan))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (5, 1, 128), (6, 2, 20), (4, 2, 80)])
@pytest.mark.parametrize("seqs", [[(1500, 1), (90, 1)], [(700, 130), (0, 65), (200, 1)], [(0, 400)]])
@pytest.mark.parametrize("max_new,max_total", [(0, 0), (0, 5000), (300, 0)])
def test_the_longest_sequence_sizes_the_work_only(ops, nh, nkv, hd, seqs, dtype, max_new, max_total):
    """Too small or too large a longest sequence, and more new tokens than any sequence has."""
    case = Case(seqs, nh, nkv, hd, 333, 70, dtype, seed=hd)
    width = 80
    table = torch.full((case.table.shape[0], width), len(case.k) - 1, dtype=torch.int32)
    table[:, :case.table.shape[1]] = case.table
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    most = max(n for _, n in seqs)
    got = ops.attention_kept(case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), table.to(DEV), i(case.slots), i([s for s, _ in seqs]), i([n for _, n in seqs]), i(case.cu),
                             most + max_new, max_total, nh, nkv, hd, hd ** -0.5, 333, 70).cpu()
    case.check(got)


@pytest.mark.gpu
def test_prescaled_queries(ops):
    """Queries that carry scale and log2 e already, rounded with them: as the step hands them over."""
    case = Case([(0, 60), (500, 37)], 8, 2, 128, 90, 4, BF16, seed=2)
    plain = Case([(0, 60), (500, 37)], 8, 2, 128, 90, 4, BF16, seed=2)
    factor = ops.prefill_q_scale(128, BF16, 128 ** -0.5)
    assert factor != 1.0
    case.q = (case.q.float() * factor).to(BF16)
    plain.q = case.q.double() / (128 ** -0.5 * ops.LOG2E)
    want, off = plain.plain()
    for plan in [p for p in PLANS] + [None]:
        got = case.run(ops, plan=plan, q_prescaled=True)
        assert bool(((got.double() - want).abs() <= off).all())


@pytest.mark.gpu
def test_without_first_positions_it_is_the_window_alone(ops):
    """The framework's other window, on the same step."""
    case = Case([(0, 90), (200, 33), (77, 1)], 8, 2, 64, 50, 0, F32, seed=3)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    case.k[-1], case.v[-1] = 0, 0
    other = ops.attention_exact(case.q.to(DEV), case.k.to(DEV), case.v.to(DEV), case.table.to(DEV), i(case.slots), i([0, 200, 77]), i([90, 33, 1]),
                                i(case.cu), 90, 8, 2, 64, 64 ** -0.5, 50).cpu()
    assert torch.allclose(case.run(ops), other, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
def test_a_captured_step_replays_with_new_contents(ops):
    case = Case([(500, 1), (70, 1), (1500, 1)], 8, 2, 128, 300, 4, BF16, seed=8)
    other = Case([(500, 1), (70, 1), (1500, 1)], 8, 2, 128, 300, 4, BF16, seed=9)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    held = [t.to(DEV) for t in (case.q, case.k, case.v, case.table)] + [i(case.slots), i([500, 70, 1500]), i([1, 1, 1]), i(case.cu)]
    args = (1, 1501, 8, 2, 128, 128 ** -0.5, 300, 4)
    ops.attention_kept(*held, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_kept(*held, *args)
    for turn in range(4):
        now = (case, other)[turn % 2]
        for t, new in zip(held, (now.q, now.k, now.v, now.table, torch.tensor(now.slots, dtype=torch.int32))):
            t.copy_(new.to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        now.check(out.cpu())
        now.check(ops.attention_kept(*held, *args).cpu())


def _refused(ops, match, **change):
    z = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype)
    a = dict(q=z(3, 8 * 16, dtype=F32), k_cache=z(5, 2, 64, 16, dtype=F32), v_cache=z(5, 2, 16, 64, dtype=F32), block_table=z(3, 4), seq_slot=z(2), seq_start=z(2),
             seq_new=z(2), cu_new=z(3), max_new=2, max_total=200, nh=8, nkv=2, hd=16, scale=0.25, window=64, kept=4)
    a.update(change)
    with pytest.raises(ops.KernelError, match=match):
        ops.attention_kept(**a)


def test_refusals(ops, monkeypatch):
    _refused(ops, "GPU only")
    monkeypatch.setattr(ops, "_dev", lambda what, *tensors: None)       # the checks behind that one need no GPU
    z = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype)
    _refused(ops, "not a multiple", nh=7)
    _refused(ops, "is not \\[n, 8\\*16\\]", q=z(3, 100, dtype=F32))
    _refused(ops, "key cache", k_cache=z(5, 2, 32, 16, dtype=F32))
    _refused(ops, "value cache", v_cache=z(5, 2, 64, 16, dtype=F32))
    _refused(ops, "page table", block_table=z(12))
    _refused(ops, "queries are torch.bfloat16", q=z(3, 8 * 16, dtype=BF16))
    _refused(ops, "neither float32 nor bfloat16", q=z(3, 128, dtype=torch.float16), k_cache=z(5, 2, 64, 16, dtype=torch.float16),
             v_cache=z(5, 2, 16, 64, dtype=torch.float16))
    _refused(ops, "differ in length", seq_new=z(3))
    _refused(ops, "differ in length", cu_new=z(2))
    _refused(ops, "window of 0", window=0)
    _refused(ops, "-1 first ones", kept=-1)
    _refused(ops, "room for 256", max_total=257)
    _refused(ops, "-1 new tokens", max_new=-1)
    _refused(ops, "int32", seq_slot=z(2, dtype=torch.int64))


def test_plans_of_prompts(ops, monkeypatch):
    """A way that there is, for any sizes; slices only where they find pages, and not where blocks are many."""
    class Lib:
        palm_attention_prefill_wide_serves = staticmethod(lambda: 1)
    monkeypatch.setattr(ops, "attention_lib", lambda hd: Lib)
    ops.kept_plan.cache_clear()
    assert ops.kept_plan(100, 1, 100, 4, 2, 80, 64, 4) == (False, 0, 1)
    for rows, n, total, nh, nkv, hd, window, kept in [(2, 1, 2, 4, 2, 64, 1, 0), (64, 1, 6064, 32, 8, 128, 4096, 4), (8192, 1, 8192, 32, 8, 128, 2048, 64), (5, 64, 900, 64, 1, 64, 1 << 29, 1 << 29),
                                                      (60000, 1, 60000, 32, 8, 128, 8192, 4), (300, 300, 40000, 160, 1, 128, 5000, 0)]:
        wide, halves, slices = ops.kept_plan(rows, n, total, nh, nkv, hd, window, kept)
        assert (wide and (halves, slices) == (0, 1) and hd == 128) or (halves in (1, 2) and 1 <= slices <= 16)
        assert slices <= -(-total // 64)
    assert ops.kept_plan(64, 1, 6064, 32, 8, 128, 4096, 4)[2] >= 8 and ops.kept_plan(8192, 1, 8192, 32, 8, 128, 2048, 64) == (False, 1, 1)
    ops.kept_plan.cache_clear()


def test_slices_fill_the_chip_and_leave_no_wave_without_a_page(ops):
    n = ops.attention_kept_lib().palm_attention_kept_slices
    assert n(1, 1, 64, 32, 8, 2048, 4) == 1                     # one page
    assert n(1, 1, 5001, 32, 8, 2048, 4) == 9                   # 33 pages for four waves
    assert n(1, 1, 1 << 24, 32, 8, 1 << 24, 0) == 64            # 8 blocks, 512 wanted
    assert n(64, 1, 5001, 32, 8, 2048, 4) == 1
    assert n(1, 2000, 2000, 32, 8, 2048, 4) == 1


def test_large_steps_of_single_tokens_are_cut_by_pages(ops):
    assert not ops.kept_by_pages(1, 8, 128, 5000) and not ops.kept_by_pages(64, 8, 128, 400) and not ops.kept_by_pages(3, 2, 64, 1 << 15)
    assert ops.kept_by_pages(48, 8, 128, 4224) and ops.kept_by_pages(64, 8, 64, 1000) and ops.kept_by_pages(1, 8, 128, 1 << 20)


def test_a_steps_way_is_chosen_from_the_keys_that_its_sequences_see(ops, monkeypatch):
    """Of a windowed layer with first positions: the window's and those, not the sequences' lengths."""
    from palm_infra_amd.parts.attention import Attention
    asked = []
    monkeypatch.setattr(ops, "decode_pages_pays", lambda *a: asked.append(a) or True)
    part = object.__new__(Attention)
    part.dtype, part.hd, part.nh, part.nkv, part.window, part.kept = BF16, 128, 8, 2, 100, 30
    assert part.decode_form([5, 400], 512)
    assert asked == [([6, 130], 8, 2, 128, 130)]
    part.window, part.kept = None, 0
    part.decode_form([5, 400], 512)
    assert asked[1] == ([6, 401], 8, 2, 128, 512)


def test_short_rows_of_single_tokens_are_not_cut(ops):
    assert ops.kept_slices(1, 32, 8, 3 * 64, 3) == 1 and ops.kept_slices(1, 32, 8, 3 * 64 + 1, 3) == 4 and ops.kept_slices(1, 32, 8, 5 * 64, 5) == 1
    assert ops.kept_slices(30, 32, 8, 640, 3) == 1 and ops.kept_slices(30, 32, 8, 641, 3) == ops.decode_slices(30, 32, 8, 641)
    assert ops.kept_slices(1, 160, 1, 320, 3) == 5 and ops.kept_slices(24, 160, 1, 320, 3) == 1


def _ways(ops, dtype, hd, single):
    """Every kernel that serves the step: named, as arguments of ``Case.run``."""
    ways = [dict(), dict(fn=ops.attention_kept_exact)]
    if dtype == BF16 and hd in ops.MFMA_HEAD_DIMS:
        ways += [dict(by_pages=True), dict(by_pages=False)] if single else [dict(plan=p) for p in PLANS if hd == 128 or (hd == 64 and not p[0])]
    return ways


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (4, 2, 80), (6, 2, 20), (4, 1, 512)])
@pytest.mark.parametrize("page", range(5))
def test_keys_that_are_no_numbers_show_wherever_their_page_falls(ops, nh, nkv, hd, dtype, page):
    """A query that sees a NaN among the keys has NaN, also if all that it sees of a page are such (its own key alone on the page, or the whole page), and whichever
    wave, slice or block walks over the page; the other kv heads' queries have their numbers."""
    for seqs in ([(64 * page, 1), (64 * page + 63, 1), (330, 1), (3000, 1)], [(0, 330), (64 * page, 30), (3000, 3)]):
        case = Case(seqs, nh, nkv, hd, 4096, 4, dtype, seed=page)
        for b, (start, new) in enumerate(seqs):
            at = page + 20 if start == 3000 else page
            case.k[case.place(b, 64 * at)[0], 0] = math.nan
        assert bool(case.plain()[0].isnan().any(1).all()) or seqs[0][1] > 1
        for way in _ways(ops, dtype, hd, seqs[0][1] == 1):
            case.check(case.run(ops, **way))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (4, 2, 80), (6, 2, 20)])
@pytest.mark.parametrize("kept", [0, 3, 67, 130])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_the_windows_first_key_alone_on_its_page_is_no_number(ops, nh, nkv, hd, dtype, kept, what):
    """The key 63 of a page is all that the window reaches of it, behind none to three pages of first positions."""
    start = 64 * 9 + 20
    case = Case([(start, 1), (start - 20, 1), (40, 1)], nh, nkv, hd, start - (64 * 5 + 63) + 1, kept, dtype, seed=kept)
    case.k[case.place(0, 64 * 5 + 63)[0], 0, 63] = what
    for way in _ways(ops, dtype, hd, True):
        case.check(case.run(ops, **way))


@pytest.mark.parametrize("hd", [64, 128, 80])
def test_the_kernels_without_first_positions_are_a_library_of_their_own(ops, hd):
    """The code of those with them would lie between, and decode steps that never run it took longer."""
    plain, kept = ops.attention_lib(hd), ops.attention_kept_hd_lib(hd)
    for name in ("decode", "decode_fused", "decode_pages", "prefill_wide"):
        assert hasattr(plain, f"palm_attention_{name}") and not hasattr(plain, f"palm_attention_{name}_kept")
        assert hasattr(kept, f"palm_attention_{name}_kept") and not hasattr(kept, f"palm_attention_{name}")
    assert plain.palm_attention_decode_pages_work(32, 8) == kept.palm_attention_decode_pages_work(32, 8)
    with pytest.raises(ops.KernelError, match="steps of 16"):
        ops.attention_kept_hd_lib(72)
