"""Pages copied to other pages: every byte that is to be moved, and none beside."""
import pytest
import torch

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from palm_infra_amd.kernels import ops
    return ops


def _pages(layers, pages, heads, hd, dtype, vheads=None, vd=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(layers, pages, heads, 64, hd, generator=g).to(dtype), torch.randn(layers, pages, vheads or heads, vd or hd, 64, generator=g).to(dtype))


def _plain(k, v, src, dst, tokens):
    k, v = k.clone(), v.clone()
    a, b = k.clone(), v.clone()
    for s, d, n in zip(src, dst, tokens or [64] * len(src)):
        a[:, d, :, :n] = k[:, s, :, :n]
        b[:, d, :, :, :n] = v[:, s, :, :, :n]
    return a, b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layers,heads,hd,vheads,vd", [(1, 1, 2, None, None), (3, 2, 16, None, None), (2, 8, 128, None, None), (5, 3, 20, 1, 7), (2, 1, 6, 2, 33)])
@pytest.mark.parametrize("src,dst,tokens", [([0], [1], [37]), ([0], [1], [0]), ([4, 4, 4, 2, 2], [0, 1, 3, 6, 7], [1, 1, 64, 63, 17]), ([5, 6, 7], [0, 1, 2], None), ([], [], [])])
def test_against_indexing(ops, layers, heads, hd, vheads, vd, src, dst, tokens, dtype):
    k, v = _pages(layers, 9, heads, hd, dtype, vheads, vd)
    want = _plain(k, v, src, dst, tokens)
    k, v = k.to(DEV), v.to(DEV)
    ops.copy_pages(k, v, src, dst, tokens)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("n,fan", [(700, 1), (170, 3), (1, 600), (161, 1), (5, 64)])
def test_more_copies_than_a_launch_takes(ops, n, fan):
    k, v = _pages(2, n * (1 + fan) + 1, 1, 4, BF16, seed=n)
    order = torch.randperm(n * (1 + fan), generator=torch.Generator().manual_seed(n)).tolist()
    src = [s for s in order[:n] for _ in range(fan)]
    tokens = [1 + (i * 29) % 64 for i in range(n * fan)]
    want = _plain(k, v, src, order[n:], tokens)
    k, v = k.to(DEV), v.to(DEV)
    ops.copy_pages(k, v, src, order[n:], tokens)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("row", [(), (1,), (3, 5), (576,)])
def test_rows_and_states(ops, row, dtype):
    g = torch.Generator().manual_seed(1)
    rows = torch.randn((3, 6, 64) + row, generator=g).to(dtype)
    want = rows.clone()
    want[:, 4, :33], want[:, 5, :64] = rows[:, 1, :33], rows[:, 0]
    got = rows.to(DEV)
    ops.copy_rows(got, [1, 0], [4, 5], [33, 64])
    assert torch.equal(got.cpu(), want)
    states = torch.randn((3, 6) + row, generator=g).to(dtype)
    want = states.clone()
    want[:, 4], want[:, 2] = states[:, 1], states[:, 1]
    got = states.to(DEV)
    if dtype == BF16 and not row:                       # two bytes a state
        assert got[0, 0].numel() == 1
    ops.copy_states(got, [1, 1], [4, 2])
    assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
def test_a_view_that_starts_anywhere(ops):
    """Storage that does not start on 16 bytes: moved by smaller pieces."""
    flat = torch.randn(1 + 2 * 5 * 64 * 8, generator=torch.Generator().manual_seed(2)).to(BF16)
    got = flat.to(DEV)
    ops.copy_rows(got[1:].view(2, 5, 64, 8), [0], [3], [9])
    want = flat.clone()
    want[1:].view(2, 5, 64, 8)[:, 3, :9] = flat[1:].view(2, 5, 64, 8)[:, 0, :9]
    assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
def test_on_a_stream_of_its_own_and_captured(ops):
    k, v = (t.to(DEV) for t in _pages(2, 6, 2, 16, BF16))
    before = k.clone(), v.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages(k, v, [0, 0], [3, 4], [5, 64])
    torch.cuda.synchronize()
    assert torch.equal(k, before[0])                    # recorded, not run
    for turn in range(3):
        k.normal_(), v.normal_()
        want = _plain(k.cpu(), v.cpu(), [0, 0], [3, 4], [5, 64])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.copy_pages(k, v, [1], [5])
    stream.synchronize()
    assert torch.equal(k[:, 5], k[:, 1]) and torch.equal(v[:, 5], v[:, 1])


def test_refusals(ops, monkeypatch):
    k, v = _pages(2, 6, 2, 16, BF16)
    with pytest.raises(ops.KernelError, match="GPU only"):
        ops.copy_pages(k, v, [0], [1])
    monkeypatch.setattr(ops, "_dev", lambda what, *tensors: None)

    def on_host(device, lib, name, *args):              # the library's own checks stand before its launches
        ops.library.call(lib, name, None, *args)
    monkeypatch.setattr(ops, "_call_on", on_host)
    for src, dst, tokens, match in (([0], [6], None, "from page 0 to 6 of 6"), ([-1], [1], None, "from page -1"), ([0, 1], [2, 2], None, "written twice"),
                                    ([0, 1], [1, 2], None, "both read and written"), ([3], [3], None, "both read and written"), ([0], [1], [65], "has 65 of 64"),
                                    ([0], [1], [-1], "has -1 of 64"), ([0], [1, 2], None, "1 sources, 2 destinations"), ([0], [1], [1, 2], "2 counts"),
                                    ([0.5], [1], None, "whole numbers"), ([1 << 40], [1], None, "whole numbers")):
        with pytest.raises(ops.KernelError, match=match):
            ops.copy_pages(k, v, src, dst, tokens)
    with pytest.raises(ops.KernelError, match="keys"):
        ops.copy_pages(k[0], v, [0], [1])
    with pytest.raises(ops.KernelError, match="values"):
        ops.copy_pages(k, v.float(), [0], [1])
    with pytest.raises(ops.KernelError, match="neither float32 nor bfloat16"):
        ops.copy_pages(k.half(), v.half(), [0], [1])
    with pytest.raises(ops.KernelError, match="rows"):
        ops.copy_rows(k, [0], [1])
    with pytest.raises(ops.KernelError, match="elements of 8 bytes"):
        ops.copy_states(torch.zeros(2, 3, dtype=torch.float64), [0], [1])
    ops.copy_pages(k, v, [], [])


def test_pages_and_states_too_large_are_refused(ops, monkeypatch):
    """Sizes go to the library as 32-bit numbers."""
    monkeypatch.setattr(ops, "_dev", lambda what, *tensors: None)
    with pytest.raises(ops.KernelError, match="more than 2\\^30 bytes"):
        ops.copy_states(torch.empty(1, 2, 1 << 28, device="meta"), [0], [1])
    with pytest.raises(ops.KernelError, match="more than 2\\^30 bytes"):
        ops.copy_rows(torch.empty(1, 2, 64, 1 << 23, dtype=BF16, device="meta"), [0], [1])
    with pytest.raises(ops.KernelError, match="2\\^31 pages"):
        ops.copy_states(torch.empty(1 << 16, 1 << 16, 1, device="meta"), [0], [1])


def test_states_of_no_elements_are_nothing_to_copy(ops, monkeypatch):
    monkeypatch.setattr(ops, "_dev", lambda what, *tensors: None)
    monkeypatch.setattr(ops, "_call_on", lambda device, lib, name, *args: ops.library.call(lib, name, None, *args))
    for shape in ((2, 5, 0, 7), (2, 5, 0), (1, 5, 3, 0)):
        ops.copy_states(torch.zeros(shape), [0, 0, 4], [1, 2, 3])
        with pytest.raises(ops.KernelError, match="from page 0 to 5 of 5"):
            ops.copy_states(torch.zeros(shape), [0], [5])
        with pytest.raises(ops.KernelError, match="written twice"):
            ops.copy_states(torch.zeros(shape), [0, 1], [2, 2])
    with pytest.raises(ops.KernelError, match="are not \\[layers, slots"):
        ops.copy_states(torch.zeros(0), [0], [1])


@pytest.mark.gpu
def test_states_of_no_elements_on_the_device(ops):
    ops.copy_states(torch.zeros((3, 4, 0, 6), device=DEV), [0, 0], [1, 3])
    torch.cuda.synchronize()
