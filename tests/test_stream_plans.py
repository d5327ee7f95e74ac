"""Which streams and answers run together, against the pages that they really hold, and what a stream's page lists cost (the cache's books on the
host, no GPU)."""
import random

import pytest
import torch

from palm_infra_amd.cache import CacheFull, KVNeed, ModelCache
from palm_infra_amd.engine import Engine
from palm_infra_amd.engine.generate import RequestTooLong, plan_batches


class Books:
    """What ``Engine.held_tokens`` looks at, and the steps that the generation loop makes, on a cache without kernels."""

    def __init__(self, window, kept, max_tokens, stream_tokens, max_seqs=64):
        self.cache = ModelCache([[KVNeed(1, 2, window, kept=kept)]], [None], max_tokens, max_seqs, None, torch.float32, "cpu", stream_tokens=stream_tokens)
        self.step_tokens_least = max(1024, 2 * window)          # as the engine has it

    def held_tokens(self, *a):
        return Engine.held_tokens(self, *a)

    def feed(self, growth):
        self.cache.reserve(growth)
        self.cache.commit(growth)

    def run(self, prompts, answers, new):
        """The batch's prompts in pieces of ``step_tokens_least``, the forks, then ``new`` single tokens of all.  The most pages held."""
        table, most = self.cache.paged_groups[0].table, 0
        firsts, left = [self.cache.open() for _ in prompts], list(prompts)
        while any(left):
            now = [(s, min(n, self.step_tokens_least)) for s, n in zip(firsts, left) if n]
            self.cache.reserve(now)
            most = max(most, table.pages.held_count)
            self.cache.commit(now)
            left = [n - min(n, self.step_tokens_least) for n in left]
        slots = firsts + [b for s in firsts if answers > 1 for b in self.cache.fork(s, answers - 1)]
        for _ in range(new):
            self.cache.reserve([(s, 1) for s in slots])
            most = max(most, table.pages.held_count)
            self.cache.commit([(s, 1) for s in slots])
        for s in slots:
            self.cache.close(s)
        self.cache.check()
        return most


def test_answers_need_no_room_for_a_prompt_of_their_own():
    """Two endless answers to a short question: 66 pages each of 256."""
    b = Books(4096, 4, 16384, 1 << 20)
    assert b.held_tokens(20100, 0) == 66 * 64 and b.held_tokens(100, 100) == 2 * 64
    assert plan_batches([100], 20000, 64, 16384, 1 << 20, 2, b.held_tokens) == [[0]]
    assert plan_batches([100], 20000, 64, 16384, 1 << 20, 3, b.held_tokens) == [[0]]
    with pytest.raises(RequestTooLong, match="in 4 sequences do not fit"):
        plan_batches([100], 20000, 64, 16384, 1 << 20, 4, b.held_tokens)
    # three streams of their own run together too; a long prompt takes its piece and runs alone
    assert plan_batches([100, 100, 100, 100], 20000, 64, 16384, 1 << 20, 1, b.held_tokens) == [[0, 1, 2], [3]]
    assert plan_batches([100, 30000], 20000, 64, 16384, 1 << 20, 1, b.held_tokens) == [[0], [1]]
    # with the length alone it is room for any way to get there
    assert b.held_tokens(20000) == (64 + 128 + 1 + 1) * 64 == b.held_tokens(20000, 20000) and b.held_tokens(100) == 2 * 64


@pytest.mark.parametrize("seed", range(12))
def test_what_is_planned_together_fits(seed):
    """Batches as planned, run to their full lengths: never more pages than the cache has, whatever the prompts."""
    rng = random.Random(seed)
    window, kept, answers = rng.choice([1, 40, 64, 65, 300]), rng.choice([0, 3, 64, 130]), rng.choice([1, 1, 2, 3, 5])
    b = Books(window, kept, 64 * rng.choice([40, 70, 130]), 64 * 400)
    prompts = [rng.choice([1, 63, 64, 65, 200, 1023, 1025, 3000, rng.randint(1, 2500)]) for _ in range(8)]
    new, planned = rng.choice([1, 64, 150, 700]), []
    for batch in plan_batches(prompts, new, 64, b.cache.max_tokens, b.cache.max_seq_tokens, answers, b.held_tokens):
        need = sum(max(b.held_tokens(prompts[i], prompts[i]), answers * b.held_tokens(prompts[i] + new, 0)) for i in batch)
        assert b.run([prompts[i] for i in batch], answers, new) * 64 <= need <= b.cache.max_tokens
        planned += batch
    assert planned == list(range(8))


def test_a_page_border_costs_the_same_however_long_the_stream_is():
    """What reaches the device's page table there are the new page and the one given back, not the whole list: the places before the window are never
    written again."""
    c = ModelCache([[KVNeed(1, 2, 130, kept=4)]], [None], 64 * 12, 3, None, torch.float32, "cpu", stream_tokens=1 << 22)
    group, s = c.paged_groups[0], c.open()
    sent = []
    real = torch.Tensor.index_copy_

    def counted(self, dim, index, source):
        sent.append(index.numel())
        return real(self, dim, index, source)
    for _ in range(5000):                                       # 320,000 tokens, a page at a time
        c.reserve([(s, 64)])
        c.commit([(s, 64)])
    marked = group.table_dev[s, 1000:4000].clone()
    group.table_dev[s, 1000:4000] = 7                           # places that were given back long ago
    torch.Tensor.index_copy_ = counted
    try:
        for _ in range(64 * 20):
            c.reserve([(s, 1)])
            c.commit([(s, 1)])
    finally:
        torch.Tensor.index_copy_ = real
    assert bool((group.table_dev[s, 1000:4000] == 7).all()) and bool((marked == c.paged_groups[0].pad_page).all())
    # 20 new pages, and 20 given back
    assert len(sent) <= 40 and sum(sent) <= 40
    c.close(s)
    assert c.lengths[s] == 0
    group.sync()
    assert bool((group.table_dev == group.pad_page).all())


def test_the_device_has_every_list_as_the_books_have_it():
    """After any traffic, all of the table: the pages listed, the spare page elsewhere."""
    rng = random.Random(11)
    needs = [[KVNeed(1, 4)], [KVNeed(1, 4, 100)], [KVNeed(1, 4, 90, kept=70)]]
    c = ModelCache(needs, [None] * 3, 64 * 60, 10, 2000, torch.float32, "cpu")
    live = []
    for turn in range(500):
        what = rng.random()
        try:
            if what < 0.25:
                live.append(c.open())
            elif what < 0.35 and live:
                live += c.fork(rng.choice(live), rng.randint(1, 2))
            elif what < 0.5 and live:
                c.close(live.pop(rng.randrange(len(live))))
            elif what < 0.55:
                c.compact()
            elif live:
                for _ in range(rng.choice([1, 1, 70])):
                    s = rng.choice(live)
                    c.reserve([(s, rng.choice([1, 1, 5, 64, 130]))]) if rng.random() < 0.1 else None     # (room taken and not used)
                    n = rng.choice([1, 1, 5, 64])
                    c.reserve([(s, n)])
                    c.commit([(s, n)])
        except CacheFull:
            pass
        for g in c.paged_groups:
            g.sync()
            want = torch.full_like(g.table_dev, g.pad_page)
            for slot, pages in enumerate(g.table.slot_pages):
                for j, p in enumerate(pages):
                    want[slot, j] = p if p >= 0 else g.pad_page
            assert torch.equal(g.table_dev, want) and torch.equal(g.table_host, want)
