"""Attention of decoded rows with keys in common, against the definition in 64 bits.

Tolerances, with the scores' and values' sizes of the inputs below (|q . k| * scale up to about 6, |v| about 1).  32 bits: a
score is off by head_dim roundings of partial sums, at most head_dim * 2^-24 * sum |q_i k_i| * scale <= 256 * 2^-24 * 16 * ... in
the worst case and sqrt(head_dim) of that in the usual one; weights and sums follow it: 2e-5 relative to the largest value covers
every size below with a factor of ten.  bfloat16: inputs are exact in 64 bits as they stand; the weights' rounding (relative 2^-9,
zero mean) and the result's (2^-9 of it): 2^-8 of the largest value of a row's keys and 2^-8 of the result itself.
"""

import math

import numpy as np
import pytest
import torch

from tesseract_b200 import kernels, plan
from tesseract_b200.parts.base import SharedRows

pytestmark = pytest.mark.gpu


class Case:
    """``groups``: for each, the keys in common and how many keys each of its rows reads in all (0: none)."""

    def __init__(self, groups, heads=8, kv_heads=2, dim=64, page=16, dtype=torch.bfloat16, seed=0, poison=True, gap=0):
        rng = np.random.RandomState(seed)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        lengths = [n for _, rows in groups for n in rows]
        rows = len(lengths)
        place = rng.permutation(rows)
        columns = max(1, max(-(-n // page) for n in lengths))
        table = np.zeros((rows, columns), dtype=np.int32)
        at, row, members, copies = 1, 0, [], []
        for prefix, counts in groups:
            common = prefix // page
            shared = np.arange(at, at + common)
            at += common
            mine, first = [], None
            for n in counts:
                need = -(-n // page)
                b = int(place[row])
                table[b, :common] = shared
                table[b, common:need] = np.arange(at, at + need - common)
                at += max(0, need - common)
                if prefix % page and need > common:
                    if first is None:
                        first = int(table[b, common])
                    else:
                        copies.append((first, int(table[b, common]), prefix % page))
                mine.append(b)
                row += 1
            members.append(mine)
        order = np.concatenate([[0], 1 + rng.permutation(at - 1)]).astype(np.int32)
        table = order[table]
        cache = torch.randn(at, 2, kv_heads, page, dim, generator=gen, device="cuda")
        for a, b, n in copies:
            cache[int(order[b]), :, :, :n] = cache[int(order[a]), :, :, :n].clone()
        self.last = np.zeros(rows, dtype=np.int64)
        self.last[place] = np.asarray(lengths) - 1
        cache = cache.to(dtype)
        if poison:                                   # what lies behind a row's last key, and the scratch page
            cache[0] = math.nan
            for b in range(rows):
                n = int(self.last[b]) + 1
                if n % page:
                    cache[int(table[b, n // page]), :, :, n % page:] = math.nan
        self.cache = cache
        # (strides of their own: the queries are columns of a wider product, the table rows of a wider table)
        wide = torch.randn(rows, (heads + 2 * kv_heads) * dim + gap, generator=gen, device="cuda").to(dtype)
        self.q = wide[:, :heads * dim]
        wide_table = torch.full((rows, columns + 5), 1 << 30, dtype=torch.int32)
        wide_table[:, :columns] = torch.from_numpy(table)
        self.table = wide_table.cuda()[:, :columns]
        self.positions = torch.from_numpy(self.last.astype(np.int32)).cuda()
        self.scale = 1.0 / math.sqrt(dim)
        self.shared = SharedRows.of(members, [p for p, _ in groups], self.last.tolist(), "cuda")

    def choice(self):
        return plan.shared_attention(self.dtype, num_heads=self.heads, num_kv_heads=self.kv_heads, head_dim=self.dim,
                                     page_size=self.page, shared=self.shared)

    def run(self, choice=None):
        out = torch.full((self.q.shape[0], self.heads * self.dim + 16), 7.0, dtype=self.dtype, device="cuda")
        view = out[:, :self.heads * self.dim]
        got = kernels.attention_shared(self.q, view, self.cache, self.positions, self.table, self.shared, self.heads,
                                       self.kv_heads, self.dim, self.page, self.scale, choice or self.choice())
        assert got is view and bool((out[:, self.heads * self.dim:] == 7.0).all())
        return view

    def definition(self):
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        limit = torch.zeros(self.q.shape[0], 1, dtype=torch.float64, device="cuda")
        for b, last in enumerate(self.last):
            if last < 0:
                continue
            pages = self.table[b, :last // self.page + 1].long()
            kv = self.cache[pages].double().permute(1, 2, 0, 3, 4).reshape(2, self.kv_heads, -1, self.dim)[:, :, :last + 1]
            q = self.q[b].double().view(self.kv_heads, -1, self.dim)
            weights = torch.softmax(q @ kv[0].transpose(1, 2) * self.scale, dim=-1)
            out[b] = (weights @ kv[1]).reshape(-1)
            limit[b] = kv[1].abs().max()
        return out, limit

    def check(self, choice=None):
        got = self.run(choice).double()
        want, limit = self.definition()
        if self.dtype == torch.float32:
            bound = 2e-5 * limit
        else:
            bound = 2.0 ** -8 * (limit + want.abs())
        assert bool(torch.isfinite(got).all())
        worst = float(((got - want).abs() - bound).max())
        assert worst <= 0, worst
        return got


DTYPES = [torch.bfloat16, torch.float32]

GROUPS = {
    "one row, one key": [(0, [1])],
    "two rows of one key": [(1, [1, 1])],
    "less than a block in common": [(63, [64, 70, 63])],
    "a block to the key": [(64, [64, 65, 100])],
    "blocks, an odd length": [(201, [201, 202, 230, 400])],
    "rows without a key": [(0, [0]), (130, [131, 140]), (0, [0, 5])],
    "nothing in common": [(0, [50, 300, 1, 129])],
    "groups of all sizes": [(500, [501] * 9), (64, [90]), (1000, [1300, 1001]), (0, [7, 8]), (129, [130 + i for i in range(20)])],
    "long": [(5000, [5001, 5100, 5555]), (0, [3001])],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", GROUPS)
def test_groups(name, dtype):
    Case(GROUPS[name], dtype=dtype, seed=len(name)).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 64), (32, 8, 128), (24, 8, 128), (4, 2, 16), (4, 4, 32), (20, 4, 80),
                                                  (3, 1, 48), (16, 1, 128), (40, 2, 64), (8, 2, 256), (6, 2, 240), (5, 5, 96),
                                                  (64, 1, 64), (18, 2, 112)])
def test_head_layouts(heads, kv_heads, dim, dtype):
    Case([(300, [301, 340, 420, 303, 305]), (77, [100, 99]), (0, [33])], heads, kv_heads, dim, dtype=dtype, seed=dim).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 128, 256, 1000])
def test_page_sizes(page, dtype):
    for dim in (64, 128):
        Case([(260, [261, 390, 300]), (190, [191, 192] + [200] * 20), (5, [6, 70])], 8, 2, dim, page, dtype, seed=page).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 3, 4, 5, 8, 16, 17, 31, 32, 33, 64, 65, 100])
def test_tiles_of_rows(rows, dtype):
    for dim in (64, 128):
        Case([(450, [451 + 3 * i % 97 for i in range(rows)])], 8, 2, dim, dtype=dtype, seed=rows).check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_cut_gives_the_same_numbers(dtype):
    """Runs of any length, more runs than there are blocks, and no sharing at all."""
    case = Case([(700, [701, 900, 1500, 702]), (320, [321, 333] + [350] * 12), (0, [640, 0])], 8, 2, 64, dtype=dtype, seed=3)
    base = case.choice()
    for prefix_parts, prefix_run, tail_parts, tail_run in [(1, 1, 1, 1), (64, 1, 64, 1), (3, 2, 2, 3), (2, 100, 5, 1), (0, 1, 7, 2),
                                                           (40, 1, 1, 9)]:
        choice = type(base)(**{**base.__dict__, "prefix_parts": prefix_parts, "prefix_run": prefix_run, "tail_parts": tail_parts,
                               "tail_run": tail_run})
        case.check(choice)
    more = type(base)(**{**base.__dict__, "tiles": base.tiles + 5})
    assert torch.equal(case.run(more), case.run(base))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 112, 128, 144, 192, 208, 256])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 16, 24, 33, 70])
def test_both_forms(rows, dim, dtype):
    """The form with the larger tiles (in bfloat16 the tensor cores') and the other, at every count of rows, whichever the plan takes."""
    case = Case([(1030, [1031 + 7 * i % 90 for i in range(rows)]), (192, [200, 250])], 8, 2, dim, dtype=dtype, seed=rows)
    alone = rows == 1                                # (a row alone has nothing in common with another)
    for wide in (False, True):
        tile = kernels.attention_shared_tile(dtype, wide)
        tiles = sum(-(-n * 4 // tile) for n in ((2,) if alone else (rows, 2)))
        for parts, run, warps in ((1, 1, 0), (5, 2, 2)):
            case.check(plan.SharedAttentionPlan(tiles, parts, run, 2, 1, wide, warps))
    assert kernels.tcgen05_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_share_nothing_in_one_launch(dtype):
    """No common part and one run a row: the results are written at once, the zeros of rows without keys too."""
    for dim in (48, 64, 128):
        case = Case([(0, [0]), (128, [200, 140]), (0, [1]), (0, [0, 70, 0])], 8, 2, dim, dtype=dtype, seed=4)
        before = kernels.launch_count
        got = case.check(plan.SharedAttentionPlan(0, 0, 1, 1, 1))
        assert kernels.launch_count == before + 1
        rows = case.shared.members.tolist()
        assert not bool(got[[rows[0], rows[4], rows[6]]].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_bits_every_time(dtype):
    case = Case([(900, [901 + 5 * i for i in range(40)])], 32, 8, 128, dtype=dtype, seed=9)
    first = case.run().clone()
    for _ in range(3):
        assert torch.equal(case.run(), first)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_leap(dtype):
    """Maxima that rise late (a key far above all before it), and keys whose scores are far below the first."""
    for direction in (1.0, -1.0):
        case = Case([(640, [641, 700, 720, 655] + [660] * 16)], 8, 2, 128, dtype=dtype, seed=11)
        steps = torch.linspace(0.05, 6.0, 16, device="cuda") if direction > 0 else torch.linspace(6.0, 0.05, 16, device="cuda")
        case.cache[:, 0] = (case.cache[:, 0].float() * steps[None, None, :, None]).to(dtype)
        case.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_stays_in_its_rows(dtype):
    """A NaN among the keys of one row's own pages, and one among the common keys of one group."""
    case = Case([(128, [140, 150, 160]), (192, [200, 210]), (0, [40])], 8, 2, 64, dtype=dtype, seed=5)
    want, _ = case.definition()
    rows = [int(r) for r in case.shared.members.tolist()]
    case.cache[int(case.table[rows[1], 139 // 16]), :, :, 139 % 16] = math.nan
    case.cache[int(case.table[rows[3], 2]), :, :, 5] = math.nan
    got = case.run().double()
    assert bool(torch.isnan(got[rows[1]]).all()) and bool(torch.isnan(got[rows[3]]).all()) and bool(torch.isnan(got[rows[4]]).all())
    for b in (rows[0], rows[2], rows[5]):
        assert float((got[b] - want[b]).abs().max()) < 2.0 ** -6


@pytest.mark.parametrize("dtype", DTYPES)
def test_on_another_stream_and_behind_its_inputs(dtype):
    case = Case([(256, [257, 300, 280])], 8, 2, 64, dtype=dtype, seed=2)
    want = case.run().clone()
    side = torch.cuda.Stream()
    kept = case.q
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(kept)
        torch.cuda._sleep(2_000_000)
        late.copy_(kept)
        case.q = late
        got = case.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_pages_past_the_reach_of_32_bits():
    """A cache of more than 2^31 numbers whose pages in use lie at its end."""
    pages, page, kv_heads, dim = 70_000, 16, 8, 128
    cache = torch.zeros(pages, 2, kv_heads, page, dim, dtype=torch.bfloat16, device="cuda")
    assert cache.numel() > 2 ** 31
    case = Case([(300, [301, 330, 350, 360, 310, 305])], 32, kv_heads, dim, seed=1)
    used = case.cache.shape[0]
    cache[pages - used:] = case.cache
    case.table = case.table + (pages - used)
    case.cache = cache
    case.check()


def test_shared_rows_refuse_what_is_no_grouping():
    for groups, prefixes, positions in [([[0, 1]], [0], [5]), ([[0], [0]], [0, 0], [5]), ([[0]], [0], [5, 5]), ([[0, 1]], [7], [5, 9]),
                                        ([[0, 1]], [-1], [5, 9]), ([[0, 1], []], [1, 0], [5, 9]), ([[0, 1]], [1, 1], [5, 9])]:
        with pytest.raises(ValueError):
            SharedRows.of(groups, prefixes, positions, "cuda")


def test_refusals():
    case = Case([(100, [101, 120])], 8, 2, 64, poison=False)
    out = torch.empty(case.q.shape, dtype=case.dtype, device="cuda")
    good = dict(q=case.q, out=out, cache=case.cache, positions=case.positions, block_table=case.table, shared=case.shared,
                num_heads=8, num_kv_heads=2, head_dim=64, page_size=16, scale=0.125, choice=case.choice())
    kernels.attention_shared(**good)
    wide = torch.randn(2, 8 * 64 + 3, device="cuda").bfloat16()
    small = Case([(100, [101, 120, 130])], 8, 2, 64)
    for name, value in [("q", case.q.float()), ("q", case.q[:, :100]), ("q", case.q[:1]), ("q", wide[:, :512]), ("q", wide[:, 1:513]),
                        ("out", out.float()), ("out", out.cpu()), ("cache", case.cache.transpose(2, 3)), ("cache", case.cache.float()),
                        ("positions", case.positions.long()), ("positions", case.positions[:1]), ("block_table", case.table.long()),
                        ("block_table", case.table[:1]), ("page_size", 8), ("num_heads", 4), ("head_dim", 32),
                        ("shared", small.shared), ("scale", 0.0), ("scale", -1.0), ("scale", math.nan)]:
        with pytest.raises(kernels.KernelError):
            kernels.attention_shared(**{**good, name: value})
    many = Case([(1030, [1040] * 40)], 8, 2, 64)
    short = type(many.choice())(**{**many.choice().__dict__, "tiles": many.choice().tiles - 1})
    with pytest.raises(kernels.KernelError, match="tiles"):
        many.run(short)
    for dim in (8, 24, 272):
        with pytest.raises(kernels.KernelError):
            kernels.attention_shared(torch.zeros(2, 8 * dim, device="cuda"), torch.zeros(2, 8 * dim, device="cuda"),
                                     torch.zeros(20, 2, 2, 16, dim, device="cuda"), case.positions, case.table, case.shared, 8, 2, dim,
                                     16, 1.0, case.choice())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix_parts, tail_parts, wide, kernels_run", [(0, 1, False, 1), (0, 1, True, 1), (0, 3, False, 2), (0, 3, True, 2),
                                                                       (2, 1, False, 2), (2, 3, True, 3)])
def test_every_kernel_of_a_call_is_counted(prefix_parts, tail_parts, wide, kernels_run, dtype):
    """One kernel where results are written at once, one more where runs are put together, one more for common parts in large tiles;
    and those are the kernels that the device saw."""
    case = Case([(640, [700 + 9 * i for i in range(24)])], 8, 2, 64, dtype=dtype, seed=6)
    tiles = case.shared.tiles(4, kernels.attention_shared_tile(dtype, wide))
    choice = plan.SharedAttentionPlan(tiles, prefix_parts, 2, tail_parts, 2, wide)
    out = torch.empty(case.q.shape, dtype=dtype, device="cuda")

    def call():
        kernels.attention_shared(case.q, out, case.cache, case.positions, case.table, case.shared, 8, 2, 64, 16, case.scale, choice)

    call()
    torch.cuda.synchronize()
    before = kernels.launch_count
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as seen:
        call()
        torch.cuda.synchronize()
    assert kernels.launch_count - before == kernels_run
    names = [event.name for event in seen.events() if "shared_" in event.name]
    assert len(names) == kernels_run or not names        # (nothing where the device gives no record)
