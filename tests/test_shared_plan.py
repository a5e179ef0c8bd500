"""How attention over rows with keys in common is cut, and what of its kernel a run cannot show (no GPU needed)."""

import os
import re
from types import SimpleNamespace

import pytest
import torch

from tesseract_b200 import kernels, plan
from tesseract_b200.parts.base import SharedRows, shared_arrays

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tesseract_b200", "csrc")
SMS = 148


def choose(groups, heads=32, kv_heads=8, dim=128, dtype=torch.bfloat16, page=16, room=None):
    rows, members, prefixes, positions = 0, [], [], []
    for prefix, counts in groups:
        members.append(list(range(rows, rows + len(counts))))
        prefixes.append(prefix)
        positions += [n - 1 for n in counts]
        rows += len(counts)
    shared = SharedRows.of(members, prefixes, positions, "cpu")
    shared.room = room
    return shared, plan.shared_attention(dtype, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, page_size=page, shared=shared,
                                         sms=SMS)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("groups", [
    [(0, [1])], [(0, [0])], [(200, [205] * 4)], [(2048, [2100] * 16)], [(32768, [32900] * 64)], [(0, [70000])],
    [(300 * k, [300 * k + 10 * j for j in range(1, 2 + k)]) for k in range(1, 9)], [(131072, [131073, 131080])], [(64, [65] * 500)],
])
def test_runs_cover_every_key_and_fit_the_chip(groups, dim, dtype):
    shared, choice = choose(groups, dim=dim, dtype=dtype)
    fold, kv_heads = 4, 8
    assert 1 <= choice.tail_parts <= plan.SHARED_MAX_PARTS and 0 <= choice.prefix_parts <= plan.SHARED_MAX_PARTS
    if choice.prefix_parts == 0:
        assert choice.tiles == 0 and not choice.wide
        assert plan.saved_blocks(shared.sizes, shared.blocks) < plan.SHARED_MIN_SAVED
    else:
        tile = kernels.attention_shared_tile(dtype, choice.wide)
        assert choice.tiles == sum(-(-n * fold // tile) for n, b in zip(shared.sizes, shared.blocks) if b)
        runs = [(-(-n * fold // tile), -(-b // choice.prefix_run)) for n, b in zip(shared.sizes, shared.blocks) if b]
        assert choice.prefix_parts == min(plan.SHARED_MAX_PARTS, max(r for _, r in runs))
        # at most what is resident at once, unless every tile is one run already
        assert sum(t * r for t, r in runs) * kv_heads <= 4 * SMS or max(r for _, r in runs) == 1


@pytest.mark.parametrize("dtype, heads, kv_heads, dim, groups, wide", [
    (torch.bfloat16, 32, 8, 64, [(8192, [8200] * 8)], False), (torch.bfloat16, 32, 8, 64, [(8192, [8200] * 16)], True),
    (torch.bfloat16, 32, 8, 64, [(8192, [8200] * 4)] * 16, False), (torch.bfloat16, 32, 8, 128, [(8192, [8200] * 4)] * 16, False),
    (torch.bfloat16, 32, 8, 128, [(2048, [2100] * 16)], True), (torch.bfloat16, 32, 8, 64, [(2048, [2100] * 16)], False), (torch.bfloat16, 20, 4, 80, [(32768, [32800] * 64)], True),
    (torch.bfloat16, 8, 2, 256, [(8192, [8200] * 2)], True), (torch.bfloat16, 4, 2, 16, [(8192, [8200] * 64)], False),
    (torch.float32, 32, 8, 64, [(2048, [2100] * 4)], False), (torch.float32, 32, 8, 64, [(2048, [2100] * 8)], True),
])
def test_which_form_takes_the_keys_in_common(dtype, heads, kv_heads, dim, groups, wide):
    _, choice = choose(groups, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    assert choice.wide == wide and choice.prefix_parts > 0
    assert choice.wide or choice.warps == 0                           # (common parts want the large blocks)


def test_what_is_shared_and_what_not():
    assert choose([(200, [205] * 4)])[1].prefix_parts == 0            # three rows times three blocks: every row reads its own
    assert choose([(2048, [2100] * 16)])[1].prefix_parts > 0
    assert choose([(4096, [5000])])[1].prefix_parts == 0              # alone
    block = 64 * 8 * 64 * 2 * 2
    assert not plan.sharing_pays((8,), (32,), block) and plan.sharing_pays((32,), (32,), block)
    assert plan.sharing_pays((4,), (64,), block) and not plan.sharing_pays((4,), (63,), block)         # long ones from a third on
    assert not plan.sharing_pays((2,), (64,), block) and not plan.sharing_pays((), (), block)
    assert not plan.sharing_pays((1, 1), (0, 0), block) and not plan.sharing_pays((4,), (100,), 0)


def test_the_plan_of_a_prompts_continuations():
    mixer = SimpleNamespace(num_heads=32, num_kv_heads=8, head_dim=128)
    assert plan.continuations(torch.bfloat16, mixer, 1, 4096, 16, SMS) is None
    assert plan.continuations(torch.bfloat16, mixer, 8, 1024, 16, SMS) is None
    choice = plan.continuations(torch.bfloat16, mixer, 64, 4096, 16, SMS)
    assert choice == choose([(4096, [4100] * 64)])[1] and choice.wide
    assert not plan.continuations(torch.float32, SimpleNamespace(num_heads=8, num_kv_heads=8, head_dim=256), 2, 16384, 16, SMS).wide


def test_a_captured_plan_has_tiles_for_every_grouping_of_as_many_groups():
    for room in (8, 16, 32):
        _, choice = choose([(4096, [4200] * (room // 2)), (2048, [2100] * (room - room // 2))], room=room)
        tile = kernels.attention_shared_tile(torch.bfloat16, choice.wide)
        for first in range(0, room + 1):
            assert choice.tiles >= -(-first * 4 // tile) + -(-(room - first) * 4 // tile)
    for heads in (8, 20, 24, 40, 48, 56):
        for groups in ([16], [3, 13], [5, 5, 6], [2] * 8, [1, 15], [7, 9]):
            _, choice = choose([(8192, [8200] * n) for n in groups], heads=heads, room=16)
            tile, fold = kernels.attention_shared_tile(torch.bfloat16, choice.wide), heads // 8
            assert choice.tiles >= sum(-(-n * fold // tile) for n in groups if n > 1)


def test_arrays_of_a_step():
    arrays, sizes, blocks, tails, row_blocks = shared_arrays([[2, 0], [1], [3]], [130, 500, 0], [140, 600, 129, -1])
    members, start, leader, prefix, common = [a.tolist() for a in arrays]
    assert members == [2, 0, 1, 3] and start == [0, 2, 3, 4] and leader == [2, 1, 3]
    assert prefix == [128, 0, 0] and common == [128, 0, 128, 0]       # whole blocks, and nothing for a row alone
    assert sizes == (2, 1, 1) and blocks == (2, 0, 0) and tails == (1, 10, 1, 0) and row_blocks == (2, 0, 2, 0)


def test_tensor_memory_that_a_product_used_is_touched_behind_a_fence():
    """attend_tc: a softmax thread that waited for a product's commit reads or writes what the product used only behind
    ``tcgen05.fence::after_thread_sync``."""
    with open(os.path.join(CSRC, "attention_shared.cu")) as handle:
        code = re.sub(r"//[^\n]*", "", handle.read())
    softmax = code[code.index("const uint32_t lane_base"):code.index("__global__ void __launch_bounds__(kTcThreads")]
    waiting, waits, touches = False, 0, 0
    for event in re.finditer(r"(?P<wait>mbar_wait\((?:o_full|s_full))|(?P<fence>tc_fence_after\(\))|"
                             r"(?P<touch>tmem_(?:load|store)\w*\(tmem_[ops]\b|\"r\"\(tmem_o)", softmax):
        if event["wait"]:
            waiting, waits = True, waits + 1
        elif event["fence"]:
            waiting = False
        else:
            touches += 1
            assert not waiting
    assert waits == 2 and touches >= 5                                # (o_full is waited for in product_done alone)


def test_what_is_under_way_is_waited_for_before_a_block_that_gave_up_leaves():
    """attend_tc: whichever warp's wait runs out, and whenever, the copies and products that others have issued are waited for once
    nobody issues any more (behind a barrier of the whole block), and in front of the barrier behind which tensor memory goes back."""
    with open(os.path.join(CSRC, "attention_shared.cu")) as handle:
        code = re.sub(r"//[^\n]*", "", handle.read())
    body = code[code.index("__device__ void attend_tc"):code.index("shared_tc_kernel")]
    barriers = [m.start() for m in re.finditer(r"__syncthreads\(\)", body)]
    issued = [m.start() for m in re.finditer(r"tma_load_kv\(|umma_ss\(|umma_ts\(|umma_commit\(", body)]
    settled = [m.start() for m in re.finditer(r"settle\(", body)]
    last, before = barriers[-1], barriers[-2]
    assert max(issued) < before < min(settled) < max(settled) < last < body.index("tcgen05.dealloc")
    given_up = body[before:last]
    assert re.match(r"__syncthreads\(\);\s*if \(abort_flag\) \{", given_up)
    for barrier in ("k_full", "v_full", "k_empty", "v_empty"):
        assert barrier in given_up


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 64), (32, 8, 128), (32, 32, 128), (32, 32, 256), (64, 16, 128), (8, 8, 256),
                                                  (16, 1, 128), (48, 48, 80)])
def test_a_step_that_leaves_the_ordinary_path_shares(heads, kv_heads, dim, dtype):
    """Wherever ``sharing_pays`` sends a decode step here, its plan reads keys in common once; large blocks pay from few on."""
    block_bytes = 64 * 2 * kv_heads * dim * (2 if dtype == torch.bfloat16 else 4)
    assert plan.shared_block_bytes(dtype, kv_heads, dim) == block_bytes
    paid = few = 0
    for rows in (2, 3, 4, 8, 31, 64):
        for blocks in (1, 2, 5, 12, 15, 33, 63, 64, 65, 200):
            shared, choice = choose([(64 * blocks, [64 * blocks + 10] * rows)], heads, kv_heads, dim, dtype)
            if plan.sharing_pays(shared.sizes, shared.blocks, block_bytes):
                assert choice.prefix_parts > 0 and choice.tiles > 0
                paid += 1
                few += plan.saved_blocks(shared.sizes, shared.blocks) < plan.SHARED_MIN_SAVED
    assert paid and (few > 0) == (block_bytes * (plan.SHARED_MIN_SAVED - 1) >= plan.SHARED_MIN_BYTES)


def cut(blocks, parts, run):
    """How the kernel cuts a row's or a common part's blocks: how many runs, and the blocks of one."""
    if blocks == 0:
        return 0, 0
    n = min(parts, -(-blocks // run))
    each = -(-blocks // n)
    return -(-blocks // each), each


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 64), (32, 8, 128), (8, 2, 256), (20, 4, 80)])
@pytest.mark.parametrize("rows", [2, 4, 8, 16, 32])
@pytest.mark.parametrize("groups", [1, 3])
def test_a_captured_plan_is_as_good_for_later_steps(groups, rows, heads, kv_heads, dim, dtype):
    """A step is captured right behind a fork; its rows then grow, and its groups share more, within its tables' width: a row's
    own keys are cut into runs of 1,024 or about those of a plan made for that step, its common part into runs that leave room for rows'
    own beside them."""
    def made(common, own, reach=None):
        prefixes = [64 * common * (k + 2) // (groups + 1) // 64 * 64 for k in range(groups)]
        shared, fresh = choose([(p, [p + 64 * own - 9] * rows) for p in prefixes], heads, kv_heads, dim, dtype)
        if reach is None:
            return shared, fresh
        shared.reach, shared.plans = reach, {}
        return shared, plan.shared_attention(dtype, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, page_size=16, shared=shared,
                                             sms=SMS)

    for reach in (64, 128, 512):
        shared, captured = made(reach // 2 + 1, 1, reach)
        assert captured == made(reach // 2 + 1, reach // 2 - 1, reach)[1]
        if plan.saved_blocks(shared.sizes, shared.blocks) < plan.SHARED_MIN_SAVED:
            continue
        assert captured.prefix_parts > 0
        for common in (reach // 2 + 1, 3 * reach // 4, reach - 2):
            for own in sorted({1, 2, 5, reach // 8, reach // 3, reach - common}):
                if common + own > reach:
                    continue
                shared, fresh = made(common, own)
                if fresh.wide != captured.wide or fresh.prefix_parts == 0:
                    continue                                            # (near the threshold; both sides' times are there)
                mine, best = cut(own, captured.tail_parts, captured.tail_run), cut(own, fresh.tail_parts, fresh.tail_run)
                assert mine[1] <= max(16, best[1] + 1, 1.25 * best[1]) and mine[0] <= best[0] + max(1, best[0] // 4)
                mine = [cut(b, captured.prefix_parts, captured.prefix_run) for b in shared.blocks]
                best = [cut(b, fresh.prefix_parts, fresh.prefix_run) for b in shared.blocks]
                assert max(r for _, r in mine) <= 2 * max(r for _, r in best) + 1
                assert sum(n for n, _ in mine) <= 2 * sum(n for n, _ in best) + groups
