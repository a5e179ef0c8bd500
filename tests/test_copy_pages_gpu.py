"""Pages copied within stores: to the bit, every element size, and the calls that are refused."""

import numpy as np
import pytest
import torch

from tesseract_b200 import kernels

pytestmark = pytest.mark.gpu

SHAPES = [
    # entries, pages, page shape, moves
    (1, 2, (8,), 1),
    (16, 40, (2, 8, 16, 64), 3),
    (3, 200, (2, 2, 8, 16), 100),
    (2, 31, (257,), 15),             # states: 32-bit rows of odd width are copied word by word
    (5, 17, (1,), 8),
    (1, 9000, (4,), 4400),           # more moves than one launch takes
    (2, 64, (16391,), 7),            # pieces that end inside a page
]


def moves_of(rng, pages, count):
    places = rng.permutation(pages)
    return places[:count], places[count:2 * count]


def expected(store, sources, targets):
    out = store.clone()
    for s, t in zip(sources, targets):
        out[:, int(t)] = store[:, int(s)]
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
@pytest.mark.parametrize("shape", SHAPES)
def test_moves_pages_bit_by_bit(shape, dtype):
    entries, pages, page, count = shape
    rng = np.random.RandomState(pages + count)
    store = torch.randint(0, 256, (entries, pages, *page, dtype.itemsize), dtype=torch.uint8, device="cuda")
    store = store.view(dtype)[..., 0]
    store = store.contiguous()
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[dtype.itemsize]
    sources, targets = moves_of(rng, pages, count)
    want = expected(store.view(bits), sources, targets)
    kernels.copy_pages([(store, sources, targets)])
    assert torch.equal(store.view(bits), want)


def test_a_source_may_go_to_several_targets():
    store = torch.randn(4, 12, 2, 3, 8, device="cuda")
    want = expected(store, [5, 5, 5, 0], [1, 2, 9, 11])
    kernels.copy_pages([(store, [5, 5, 5, 0], [1, 2, 9, 11])])
    assert torch.equal(store, want)


def test_many_stores_in_one_call_and_empty_ones():
    rng = np.random.RandomState(5)
    stores, moves, wants = [], [], []
    for i in range(19):
        store = torch.randn(1 + i % 3, 20 + i, 1 + 3 * i, device="cuda")
        sources, targets = moves_of(rng, store.shape[1], i % 7)
        stores.append(store)
        moves.append((store, sources.tolist(), targets.tolist()))
        wants.append(expected(store, sources, targets))
    moves.append((torch.empty(0, 4, 8, device="cuda"), [0], [1]))
    moves.append((torch.empty(2, 4, 0, device="cuda"), [0], [1]))
    before = kernels.launch_count
    kernels.copy_pages(moves)
    assert kernels.launch_count - before == 2             # eight stores a launch: 16 of the 19 have moves, the empty two nothing to move
    for store, want in zip(stores, wants):
        assert torch.equal(store, want)


def test_nothing_to_do_launches_nothing():
    before = kernels.launch_count
    kernels.copy_pages([])
    kernels.copy_pages([(torch.zeros(2, 3, 4, device="cuda"), [], [])])
    assert kernels.launch_count == before


def test_pages_that_start_off_a_16_byte_boundary():
    whole = torch.arange(2 * 10 * 12 + 3, dtype=torch.float32, device="cuda")
    for offset in (1, 2, 3):
        store = whole.clone()[offset:offset + 2 * 10 * 12].view(2, 10, 12)
        want = expected(store, [1, 7], [2, 0])
        kernels.copy_pages([(store, [1, 7], [2, 0])])
        assert torch.equal(store, want)
    odd = torch.arange(7 * 5 * 3 + 1, dtype=torch.uint8, device="cuda")[1:].view(5, 7, 3)
    want = expected(odd, [1, 6], [2, 0])
    kernels.copy_pages([(odd, [1, 6], [2, 0])])
    assert torch.equal(odd, want)


def test_on_another_stream():
    store = torch.zeros(8, 100, 2, 8, 16, 64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        store[:, 3] = 7.0
        kernels.copy_pages([(store, [3], [90])])
        got = store[:, 90].clone()
    torch.cuda.current_stream().wait_stream(side)
    assert bool((got == 7.0).all())


@pytest.mark.parametrize("sources, targets, message", [
    ([0], [3], "outside"), ([3], [0], "outside"), ([-1], [0], "outside"), ([0], [-1], "outside"),
    ([0, 1], [2, 2], "twice"), ([0, 1], [1, 2], "twice"), ([1], [1], "twice"),
    ([0], [1, 2], "as many"), ([0.5], [1], "integers"), ([2 ** 40], [1], "outside"),
])
def test_refusals_copy_nothing(sources, targets, message):
    store = torch.randn(2, 3, 8, device="cuda")
    kept = store.clone()
    with pytest.raises(kernels.KernelError, match=message):
        kernels.copy_pages([(store, sources, targets)])
    assert torch.equal(store, kept)


def test_refuses_what_is_not_a_store():
    store = torch.randn(4, 6, 8, device="cuda")
    for bad in (store.transpose(0, 1), store[:, :, ::2], torch.randn(4, 6, 8), torch.zeros(5, device="cuda")):
        with pytest.raises(kernels.KernelError):
            kernels.copy_pages([(bad, [0], [1])])
    with pytest.raises(kernels.KernelError, match="once"):
        kernels.copy_pages([(store, [0], [1]), (store, [2], [3])])
    with pytest.raises(kernels.KernelError, match="once"):
        kernels.copy_pages([(store[1:], [0], [1]), (store[:3], [2], [3])])
    kernels.copy_pages([(store[2:], [0], [1]), (store[:2], [2], [3])])        # side by side
    assert torch.equal(store[2:, 1], store[2:, 0]) and torch.equal(store[:2, 3], store[:2, 2])
    with pytest.raises(kernels.KernelError, match="host"):
        kernels.copy_pages([(store, torch.tensor([0], device="cuda"), [1])])
