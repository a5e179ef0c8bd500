"""The kernel plan: which kernel, in which form, every operation of a step takes.

One place decides, for a data type, a row count and the sizes of an operation, which of this package's kernels
runs it (the reference resolves one plan per model and prints it: src/cuda/kernel_plan.rs:140-161, 168-239).
The parts ask these functions and do what the answer says; ``describe`` prints the answers for a whole model
(``tesseract --print-plan``); ``tests/test_kernel_choices.py`` pins them.  There is no other backend to dispatch
to: a size no kernel takes is an error where the part is built or called.

Thresholds, with the measurement behind each:

* ``DECODE_LINEAR_MAX_ROWS`` (16): up to this many rows a product streams its weights once through the skinny
  ``decode_linear`` kernel (mma.sync, 16 warps splitting K), with the residual addition and the RMSNorm in front
  and SwiGLU or a 32-bit store behind folded in.  Against the library product with norm and activation kernels
  of their own a decode step of 16 rows of the 1B sizes takes 0.94 instead of 1.33 ms.
* ``SKINNY_MAX_ROWS`` (128): from 17 rows up to here a product streams its weights through ``skinny_tcgen05``
  (tcgen05 with the weights as the 128-row operand, K splits as a thread-block cluster), with SwiGLU or a 32-bit
  store behind it, and with the same division of a norm's work between the product in front of it and the product
  behind it as ``decode_linear`` has.
* ``FUSED_GATE_UP_MIN_ROWS`` (17): above ``SKINNY_MAX_ROWS`` gate/up + SwiGLU is one tcgen05 GEMM (100 against
  114 us per product at 2,048 rows).
* Plain bfloat16 products over more than 128 rows (QKV, O, down, the head) call the library GEMM, where the
  reference calls one (src/cuda/cublas.rs:49-92).
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from functools import lru_cache
from types import SimpleNamespace
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import kernels

DECODE_LINEAR_MAX_ROWS = 16
SKINNY_MAX_ROWS = kernels.SKINNY_MAX_ROWS
FUSED_GATE_UP_MIN_ROWS = 17
MAX_ATTENTION_SPLITS = kernels.MAX_ATTENTION_SPLITS
CLUSTER_SPLITS = 8            # up to this many splits merge inside a thread-block cluster; more go through scratch

BF16, F32, SWIGLU = "bf16", "f32", "swiglu"
GATED_SILU, GATED_GELU = "gated_silu", "gated_gelu"       # the rounded product's gate and up, activated: what a kernel behind it gives
OVER_GATE_AND_UP = (SWIGLU, GATED_SILU, GATED_GELU)
_EPILOGUE_CODE = {BF16: kernels.EPI_BF16, F32: kernels.EPI_F32, SWIGLU: kernels.EPI_SWIGLU, GATED_SILU: kernels.EPI_GATED_SILU,
                  GATED_GELU: kernels.EPI_GATED_GELU}


@lru_cache(maxsize=None)
def _decode_linear_takes(rows: int, out_features: int, in_features: int, prologue: int) -> bool:
    return kernels.decode_linear_supported(rows, out_features, in_features, prologue)


@lru_cache(maxsize=None)
def _skinny_takes(rows: int, out_features: int, in_features: int, epilogue: int) -> bool:
    return kernels.skinny_tcgen05_supported(rows, out_features, in_features, epilogue)


@lru_cache(maxsize=None)
def _gemm_tcgen05_takes(rows: int, out_features: int, in_features: int, epilogue: int) -> bool:
    return kernels.gemm_tcgen05_supported(rows, out_features, in_features, epilogue)


@lru_cache(maxsize=None)
def _attention_tcgen05_takes(num_heads: int, num_kv_heads: int, head_dim: int, page_size: int) -> bool:
    return kernels.attention_tcgen05_supported(num_heads, num_kv_heads, head_dim, page_size)


@dataclass(frozen=True)
class ProductPlan:
    """``kernel``: ``gemm_f32`` (true 32-bit FFMA), ``decode_linear`` (weight streaming, at most 16 rows),
    ``skinny_tcgen05`` (weight streaming on the tensor-memory cores, at most 128 rows), ``gemm_tcgen05`` (this
    package's tensor-memory GEMM: CTA pairs on 256-row tiles above 128 rows) or ``library``.
    ``norm_folded``: the RMSNorm (and the residual addition) in front runs inside the product's kernel.  ``epilogue``: what the kernel stores;
    ``activation_apart``: an activation was asked for but runs as a kernel of its own behind the product.
    ``prepares_norm``: the product also does the work of the norm BEHIND it (new residual, rows times the norm's
    weights, sums of squares); the product behind that then runs with ``norm="prepared"`` (``takes_prepared``): it
    takes those rows as they are and applies the scale to its 32-bit sums."""

    kernel: str
    norm_folded: bool = False
    epilogue: str = BF16
    activation_apart: bool = False
    prepares_norm: bool = False
    takes_prepared: bool = False

    @property
    def epilogue_code(self) -> int:
        return _EPILOGUE_CODE[self.epilogue]

    def __str__(self) -> str:
        extras = [f"{self.epilogue} store"]
        if self.takes_prepared:
            extras.insert(0, "rows prepared by the product in front, the norm's scale on the sums")
        elif self.norm_folded:
            extras.insert(0, "add+norm folded in front")
        if self.activation_apart:
            extras.append("activation as a kernel of its own")
        if self.prepares_norm:
            extras.append("does the following add+norm's work")
        return f"{self.kernel} ({', '.join(extras)})"


def product(dtype: torch.dtype, rows: int, out_features: int, in_features: int, *, epilogue: str = BF16,
            norm: Optional[str] = None, contiguous_rows: bool = True, follow: bool = False) -> ProductPlan:
    """The kernel for ``[rows, in] @ [out, in]^T``.  ``norm``: ``"norm"`` or ``"add_norm"`` if an RMSNorm (with the
    residual addition) stands in front and may be folded in, ``"prepared"`` if the product in front has done that
    norm's work; ``epilogue``: ``bf16``, ``f32`` (logits), or ``swiglu``, ``gated_silu`` or ``gated_gelu`` (the weight's rows interleave
    eight gates and eight up projections; in front of the last two a norm always runs on its own); ``follow``: an addition and an
    RMSNorm of the product's own width follow it."""
    if dtype == torch.float32:
        return ProductPlan("gemm_f32", False, F32, activation_apart=epilogue in OVER_GATE_AND_UP)
    if epilogue in (GATED_SILU, GATED_GELU):
        norm = None                   # (the kernels have these epilogues without a norm in front)
    if rows <= DECODE_LINEAR_MAX_ROWS and contiguous_rows:
        if norm == "prepared":
            if _decode_linear_takes(rows, out_features, in_features, kernels.PRO_NONE):
                return ProductPlan("decode_linear", True, epilogue, takes_prepared=True)
            apart = epilogue in OVER_GATE_AND_UP
            return ProductPlan("library", False, BF16 if apart else epilogue, activation_apart=apart)
        if follow and norm is None and epilogue == BF16 and _decode_linear_takes(rows, out_features, in_features,
                                                                                kernels.PRO_NONE):
            return ProductPlan("decode_linear", False, BF16, prepares_norm=True)
        if norm is not None:
            prologue = kernels.PRO_NORM if norm == "norm" else kernels.PRO_ADD_NORM
            if _decode_linear_takes(rows, out_features, in_features, prologue):
                return ProductPlan("decode_linear", True, epilogue)
        if _decode_linear_takes(rows, out_features, in_features, kernels.PRO_NONE):
            return ProductPlan("decode_linear", False, epilogue)
    if DECODE_LINEAR_MAX_ROWS < rows <= SKINNY_MAX_ROWS and in_features % 8 == 0:
        # (rows whose stride is no multiple of 8 elements are refused by the kernel's caller, which then copies)
        if norm == "prepared" and _skinny_takes(rows, out_features, in_features, _EPILOGUE_CODE[epilogue]):
            return ProductPlan("skinny_tcgen05", True, epilogue, takes_prepared=True)
        if (follow and norm is None and epilogue == BF16
                and _skinny_takes(rows, out_features, in_features, kernels.EPI_ADD_NORM)):
            return ProductPlan("skinny_tcgen05", False, BF16, prepares_norm=True)
        if norm != "prepared" and _skinny_takes(rows, out_features, in_features, _EPILOGUE_CODE[epilogue]):
            return ProductPlan("skinny_tcgen05", False, epilogue)
    if (epilogue == SWIGLU and rows >= FUSED_GATE_UP_MIN_ROWS
            and _gemm_tcgen05_takes(rows, out_features, in_features, kernels.EPI_SWIGLU)):
        return ProductPlan("gemm_tcgen05", False, SWIGLU)
    if epilogue in OVER_GATE_AND_UP:
        return ProductPlan("library", False, BF16, activation_apart=True)
    return ProductPlan("library", False, epilogue)


MASKED_PROMPT_MIN_ROWS = 257      # from here on a step's masked attention may go to the tensor cores


@lru_cache(maxsize=None)
def _prompt_mma_takes(dtype: torch.dtype, key_dim: int, value_dim: int) -> bool:
    return kernels.attention_prompt_mma_supported(dtype, key_dim, value_dim)


def masked_attention(dtype: torch.dtype, rows: int, key_dim: int, value_dim: int, sink: bool = False,
                     gated: bool = False, heads_per_kv: int = 1) -> str:
    """The kernel for attention with 32-bit scores and weights over keys and values of separate widths.  On the
    tensor cores (bfloat16, no sink, no gate, head sizes the kernels are built for): ``"attention_prompt_mma"`` for
    steps of more than 256 rows (2,048 rows of 32 heads of 64 under a window of 512: 87 us against 555 for
    ``attention_masked``), ``"attention_rows_mma"`` for steps of fewer (a block a row and kv head; at most 16 query
    heads a kv head).  ``"attention_masked"`` otherwise."""
    if not sink and not gated and dtype == torch.bfloat16 and _prompt_mma_takes(dtype, key_dim, value_dim):
        if rows >= MASKED_PROMPT_MIN_ROWS:
            return "attention_prompt_mma"
        if heads_per_kv <= 16:
            return "attention_rows_mma"
    return "attention_masked"


def latent_attention(dtype: torch.dtype, entry: int, rank: int) -> str:
    """The kernel for attention over cached latent vectors of ``entry`` numbers whose first ``rank`` are the value:
    ``"attention_latent_mma"`` in bfloat16 for the sizes it is built for (2,048 prompt rows of 16 heads over vectors of
    576 under a window of 512: 6.3 ms on ``attention_masked``), ``"attention_masked"`` otherwise."""
    return "attention_latent_mma" if kernels.attention_latent_mma_supported(dtype, entry, rank) else "attention_masked"


def attention_splits(num_seqs: int, num_kv_heads: int, max_context: int, head_dim: int = 64,
                     sms: Optional[int] = None) -> int:
    """How many key splits the decode kernel uses.

    A CTA's warps (eight up to a head size of 64, six up to 128, four above) each stream their share of the tiles
    of 16 keys at about 0.65 microseconds a tile of 64-wide heads (wider heads in proportion); merging splits
    costs about 2.5 microseconds inside a thread-block cluster (up to 8 splits) and 5 through scratch memory; two
    CTAs fit an SM up to a head size of 128, one above.  The choice minimises that estimate over the split counts
    that keep all CTAs resident at once (at most 32: one sequence of 131,072 tokens reads its keys at 5.2 TB/s
    with 32 splits, 4.5 with 16)."""
    tiles = -(-max_context // 16)
    warps = 8 if head_dim <= 64 else 6 if head_dim <= 128 else 4
    ctas = max(1, num_seqs * num_kv_heads)
    per_sm = 2 if head_dim <= 128 else 1
    tile_cost = 0.65 * max(1.0, head_dim / 64.0)
    limit = max(1, min(MAX_ATTENTION_SPLITS, per_sm * (sms or kernels.sm_count()) // ctas))
    best, best_cost = 1, float("inf")
    for splits in range(1, limit + 1):
        per_warp = -(-(-(-tiles // splits)) // warps)
        merge = 0.0 if splits == 1 else 2.5 if splits <= CLUSTER_SPLITS else 5.0
        cost = tile_cost * per_warp + merge + 0.15 * splits
        if cost < best_cost:
            best, best_cost = splits, cost
    return best


def prompt_key_splits(tile_ctas: int, max_context: int, head_dim: int = 64, sms: Optional[int] = None) -> int:
    """CTAs per tile of the tcgen05 prompt kernel.  A tile of 128 folded rows walks over its key blocks (128 keys
    up to head size 64, else 64) one after the other, and two CTAs fit an SM: a step with fewer tiles than that (a
    512-token portion of one prompt is 128 tiles of the 1B sizes) leaves SMs idle while every tile walks its whole
    context.  Such a step gives each tile to several CTAs, each over a run of at least 2,048 keys, as many as are
    resident at once (at most 8); the last one to finish adds the runs.  Leaving and adding the partial rows costs
    about 10 microseconds (a round of stores, a fence, a counter, three rounds of loads from L2), and two CTAs on an
    SM share its exponential unit, so short contexts lose, at either head size: a 512-token portion at context
    2,048 takes 27.3 us alone and 32.6 shared by two (head size 128: 42.9 and 53.5), at 3,072 38.6 and 39.0 (61.0
    and 62.8), at 4,096 50.3 and 45.0 (78.6 and 72.3), at 8,192 94.4 and 68.5 (150 and 110); ``head_dim`` is taken for
    the callers' sake and does not enter."""
    resident = 2 * (sms or kernels.sm_count())
    return max(1, min(8, resident // max(1, tile_ctas), max_context // 2048))


@dataclass(frozen=True)
class AttentionPlan:
    """``fused_decode``: one kernel rotates q and the new key, writes the cache page and attends (a pure decode
    step).  Otherwise a rotation + cache-write kernel runs first and ``prompt`` (``tcgen05``, ``mma_tiles`` or
    None) takes the sequences with more than 16 folded rows (new tokens x query heads per kv head), ``split``
    (True/False) the others through the split decode kernel.  ``rows``: the 32-bit path's one kernel.
    ``splits``/``merge``: key splits of the split kernel and how they meet (``none``, ``cluster``, ``scratch``).
    ``key_splits``: CTAs per tile of the tcgen05 prompt kernel (``prompt_key_splits``)."""

    fused_decode: bool = False
    prompt: Optional[str] = None
    split: bool = False
    rows: bool = False
    splits: int = 1
    key_splits: int = 1

    @property
    def merge(self) -> str:
        return "none" if self.splits == 1 else "cluster" if self.splits <= CLUSTER_SPLITS else "scratch"

    def __str__(self) -> str:
        if self.rows:
            return "attention_rows (a warp, in steps of few rows a block, per row and head; fixed order)"
        if self.fused_decode:
            return f"attention_decode (rotation and cache write folded in; {self.splits} split(s), merge: {self.merge})"
        parts = ["rope_kv_write"]
        if self.prompt:
            shared = f", {self.key_splits} CTAs a tile" if self.key_splits > 1 else ""
            parts.append(f"attention_{self.prompt} for prompt portions{shared}")
        if self.split:
            parts.append(f"attention_decode for short sequences ({self.splits} split(s), merge: {self.merge})")
        return " + ".join(parts)


def attention(dtype: torch.dtype, *, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
              new_tokens: Sequence[int], max_context: int, rotary_in_kernel: bool = True,
              prompt_kernel: str = "tcgen05", sms: Optional[int] = None) -> AttentionPlan:
    """The attention kernels of a step whose sequences bring ``new_tokens`` tokens each."""
    if dtype == torch.float32:
        return AttentionPlan(rows=True)
    fold = num_heads // num_kv_heads
    seqs = len(new_tokens)
    if rotary_in_kernel and fold <= 16 and all(n == 1 for n in new_tokens):
        return AttentionPlan(fused_decode=True, splits=attention_splits(seqs, num_kv_heads, max_context, head_dim, sms))
    long_seqs = any(n * fold > 16 for n in new_tokens)
    short_seqs = any(n * fold <= 16 for n in new_tokens)
    prompt = None
    if long_seqs:
        prompt = "mma_tiles"
        if prompt_kernel == "tcgen05" and _attention_tcgen05_takes(num_heads, num_kv_heads, head_dim, page_size):
            prompt = "tcgen05"
    splits = attention_splits(seqs, num_kv_heads, max_context, head_dim, sms) if short_seqs else 1
    key_splits = 1
    if prompt == "tcgen05":
        tile_ctas = -(-(max(new_tokens) * fold) // 128) * num_kv_heads * seqs      # the kernel's grid, per key split
        key_splits = prompt_key_splits(tile_ctas, max_context, head_dim, sms)
    return AttentionPlan(prompt=prompt, split=short_seqs, splits=splits, key_splits=key_splits)


@dataclass(frozen=True)
class SharedAttentionPlan:
    """How ``attention_shared`` cuts a step: ``tiles`` tiles of all groups' folded rows (``wide``: larger tiles, in bfloat16 on
    the tcgen05 tensor cores), common parts in at most ``prefix_parts`` runs of at least ``prefix_run`` blocks of 64 keys each (0
    parts: nothing is shared, every row reads its own keys), what lies behind in at most ``tail_parts`` of at least ``tail_run``."""

    tiles: int
    prefix_parts: int
    prefix_run: int
    tail_parts: int
    tail_run: int
    wide: bool = False
    warps: int = 0           # of a block: 2, or (0) as many as let two blocks share a multiprocessor


# Blocks of 64 keys in a run: a tile of 16 keys for each of eight warps, twice; in 32 bits one of 32 for each of four.
SHARED_MIN_RUN = {torch.bfloat16: 4, torch.float32: 2}
SHARED_MAX_PARTS = 64


# Blocks of 64 keys that rows need not read themselves from where on common parts are taken by themselves: below, one launch over
# every row's own keys is faster (4 rows of 32 heads of 64 at 200 keys: 4.2 us on the device, 7.0 with a launch to put parts together).
# Blocks of many or large heads are worth it from fewer on: wherever a decode step would share (`sharing_pays`), its plan does.
SHARED_MIN_SAVED = 64
# The same in bytes of keys and values from where on a decode step takes ``attention_shared`` at all: below, the kernel that rotates,
# writes and attends in one launch is faster, as it finds the common pages in L2.  Behind many keys in common a third of that: that
# kernel's runs are longer then.  A step with and without, ms: of the 1B sizes, 8 rows at 2,048 keys (29 MB) 0.756 and 0.702, 16 at 2,048
# (63) 0.852 and 0.839, 8 at 6,144 (88) 0.797 and 0.847, 32 at 2,048 (130) 1.001 and 1.067, 32 at 8,192 1.091 and 1.927; 4 at 4,096 (25)
# 0.761 and 0.807, 8 at 4,096 (59) 0.773 and 0.776, 2 at 16,000 (33) 0.792 and 0.794; of 8 layers of the 8B sizes, 16 at 1,024 (63)
# 1.064 and 1.056, 8 at 3,072 (88) 0.986 and 0.990, 4 at 4,096 (50) 0.959 and 1.015, 32 at 8,192 1.140 and 2.098.
SHARED_MIN_BYTES = 72 << 20
SHARED_LONG = 64                # blocks of 64 keys


# Where the form with the larger tiles is faster by more than the 3 us of host time that its launch costs.  bfloat16 (a tile of it
# works for 128 rows whatever it holds): tiles of 16 folded rows of a group beyond the first two, or the first (at head sizes above
# 128, where small tiles hold few keys, all of them and two more), times its blocks of common keys, kv heads and head size.  Device
# time with small tiles and with large: 32 heads on 8 of 64, 8 rows at 8,192 keys 12.4 and 14.5 us, 16 at 2,048 11.5 and 11.2, 16 at
# 8,192 19.9 and 16.9, 64 at 8,192 100.8 and 22.9, 16 groups of 4 at 8,192 51.6 and 65.9; of 128, 4 rows at 8,192 15.8 and 18.0, 8 at
# 2,048 13.9 and 12.4, 64 at 8,192 114 and 32, 16 groups of 4 at 8,192 96.6 and 98.7; 20 on 4 of 80, 8 rows at 2,048 10.9 and 12.0, 8
# at 8,192 16.3 and 15.5, 64 at 32,768 338 and 45; 8 on 2 of 256, 2 rows at 8,192 17.8 and 15.2, 64 at 32,768 365 and 45; 4 on 2 of
# 16, 64 rows at 8,192 10.2 and 11.7, at 32,768 22.9 and 16.1.
SHARED_WIDE_FREE = {64: 2, 128: 1, 256: -2}
SHARED_WIDE_MIN = 49152
# 32 bits: tiles of 8 folded rows beyond a group's first times its blocks of common keys, by head size.  32 heads on 8 of 64, 4 rows at
# 2,048 keys 12.1 and 13.8, 8 16.6 and 15.0, 64 93.5 and 51.2, 16 groups of 2 at 4,096 77.2 and 74.7, of 4 129.7 and 100.9; of 128 16.7
# and 18.3, 23.9 and 21.2, 172.8 and 96.3, 133.6 and 138.7, 225.1 and 207.2; 8 on 2 of 256, 16 rows at 4,096 keys 32.1 and 35.5, 32 at
# 2,048 40.9 and 38.3, 32 at 8,192 154.9 and 83.3.
SHARED_WIDE_MIN_F32 = {64: 64, 128: 64, 256: 460}
# Blocks of threads that share a multiprocessor, by the head size that they are made for: of the form with the larger tiles, and of
# the 32-bit one with the small.
SHARED_WIDE_RESIDENT = {torch.bfloat16: {64: 2, 128: 2, 256: 1}, torch.float32: {64: 4, 128: 3, 256: 2}}
SHARED_F32_RESIDENT = {64: 4, 128: 4, 256: 2}


# A captured step keeps its plan while keys in common and rows' own grow within its tables' width.  So it is laid out for as many runs
# as a fresh plan gives the longest that the table can name (the common parts in the proportions that they have), and shorter ones
# are cut into as many as they have blocks for.  What it cannot know is how much of the chip the other kind takes: common parts that
# share a launch with rows' own leave them two fifths, and rows' own in front of a launch of large tiles begin a second run only at
# so many blocks, up to a head size.  Device time of a plan kept from right behind the fork, of a fresh one and of a captured one, us:
# 32 heads on 8 of 64, 4 rows at 4,160 keys in common and 16 of their own 9.4, 9.4 and 9.9, 4,000 27.3, 17.5 and 17.5, at 8,256 and
# 8,092 49.9, 25.2 and 23.4; of 128, 8 rows at 4,160 and 500 16.3, 20.3 and 16.5, 4,000 49.2, 36.9 and 37.0; in 32 bits, 8 rows of 64
# at 4,160 and 16 23.1, 23.1 and 29.4 (blocks of threads that find no run), 4,000 231, 63 and 63.
CAPTURED_ROOM = 0.6
CAPTURED_TAIL_RUN = {torch.bfloat16: 16, torch.float32: 4}
CAPTURED_TAIL_RUN_UP_TO = {torch.bfloat16: 128, torch.float32: 256}


def shared_block_bytes(dtype: torch.dtype, num_kv_heads: int, head_dim: int) -> int:
    """Bytes of the keys and values of a block of 64 tokens in one layer."""
    return 64 * 2 * num_kv_heads * head_dim * torch.empty((), dtype=dtype).element_size()


def saved_blocks(sizes: Sequence[int], blocks: Sequence[int]) -> int:
    """Blocks of 64 keys that the rows of groups (``sizes`` rows, ``blocks`` blocks in common each) need not read a second time."""
    return sum((n - 1) * b for n, b in zip(sizes, blocks))


def sharing_pays(sizes: Sequence[int], blocks: Sequence[int], block_bytes: int) -> bool:
    """Whether a decode step reads common keys once a group rather than once a row, with ``block_bytes`` of keys and values in a
    block of 64 of one layer."""
    least = SHARED_MIN_BYTES // 3 if max(blocks, default=0) >= SHARED_LONG else SHARED_MIN_BYTES
    return saved_blocks(sizes, blocks) * block_bytes >= max(1, least)


def shared_attention(dtype: torch.dtype, *, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, shared,
                     sms: Optional[int] = None) -> SharedAttentionPlan:
    """The plan of attention over groups of rows with keys in common (``shared``: a :class:`SharedRows`, which keeps its plans: the
    layers of a step ask for the same one)."""
    key = (dtype, num_heads, num_kv_heads, head_dim, page_size, sms)
    choice = shared.plans.get(key)
    if choice is None:
        choice = _shared_attention(dtype, num_heads // num_kv_heads, num_kv_heads, head_dim, page_size, shared,
                                   sms or kernels.sm_count())
        shared.plans[key] = choice
    return choice


def _shared_runs(tiles: np.ndarray, blocks: np.ndarray, target: int, shortest: int) -> int:
    """The shortest runs (in blocks, ``shortest`` at least) with which all tiles' runs are at most ``target``: one more, and the
    chip goes round a second time for it."""
    longest = int(blocks.max())
    run = max(shortest, -(-int((tiles * blocks).sum()) // target))
    while run < longest and int((tiles * -(-blocks // run)).sum()) > target:
        run += 1 + run // 16
    return run


def _shared_attention(dtype, fold, num_kv_heads, head_dim, page_size, shared, sms) -> SharedAttentionPlan:
    sizes, blocks = np.asarray(shared.sizes), np.asarray(shared.blocks)
    tails = np.asarray(shared.tails)
    if (saved_blocks(shared.sizes, shared.blocks) < SHARED_MIN_SAVED        # every row reads its own
            and not sharing_pays(shared.sizes, shared.blocks, shared_block_bytes(dtype, num_kv_heads, head_dim))):
        tails = tails + np.asarray(shared.row_blocks)
        blocks = np.zeros_like(blocks)
    captured = shared.reach is not None
    if captured:
        tails = np.full_like(tails, shared.reach)
        blocks = -(-blocks * shared.reach // max(1, int(blocks.max())))
    rows = np.where(blocks > 0, sizes * fold, 0)
    sixteens = -(-rows // 16)
    padded = 64 if head_dim <= 64 else 128 if head_dim <= 128 else 256            # (a kernel's head size)
    if dtype == torch.float32:
        wide = int((np.maximum(-(-rows // 8) - 1, 0) * blocks).sum()) > SHARED_WIDE_MIN_F32[padded]
    else:
        beyond = np.where(sixteens > 0, np.maximum(sixteens - SHARED_WIDE_FREE[padded], 0), 0)
        wide = int((beyond * blocks).sum()) * num_kv_heads * head_dim > SHARED_WIDE_MIN
    wide = wide and kernels.attention_shared_wide(dtype, head_dim, page_size)
    tile = kernels.attention_shared_tile(dtype, wide)
    tiles = -(-rows // tile)
    # (large) blocks of threads that are resident at once, a kv head
    target = max(1, (SHARED_F32_RESIDENT[padded] if dtype == torch.float32 else 2) * sms // num_kv_heads)
    # rows' own keys, a block of threads each: large blocks where they are few or share a launch with common parts, small ones (and
    # all of them at once) where they are many
    tails = np.maximum(tails, 1)
    tail_tiles = np.full(tails.shape, -(-fold // kernels.attention_shared_tile(dtype)))
    warps = 2 if dtype != torch.float32 and int(tail_tiles.sum()) > target and (wide or not tiles.any()) else 0
    small = 4 if head_dim <= 64 else 2 if head_dim <= 128 else 1        # as many small ones are resident beside a large one's room
    shortest = 1 if wide and dtype == torch.float32 else SHARED_MIN_RUN[dtype]
    tail_run = _shared_runs(tail_tiles, tails, target if warps == 0 else small * target, SHARED_MIN_RUN[dtype])
    tail_parts = min(SHARED_MAX_PARTS, -(-int(tails.max()) // tail_run))
    if captured:
        tail_run = SHARED_MIN_RUN[dtype]
        if wide and padded <= CAPTURED_TAIL_RUN_UP_TO[dtype]:
            tail_run = CAPTURED_TAIL_RUN[dtype]
    prefix_parts, prefix_run = 0, 1
    if tiles.any():
        room = target
        if wide:
            room = max(1, SHARED_WIDE_RESIDENT[dtype][padded] * sms // num_kv_heads)
        else:                                   # in one launch with the rows' own: at once with them where those are much of the work
            left = target - int((tail_tiles * -(-tails // tail_run)).sum())
            few = int((tiles * blocks).sum()) > 4 * int((tail_tiles * tails).sum())
            room = int(target * CAPTURED_ROOM) if captured else target if few or 2 * left < target else left
        prefix_run = _shared_runs(tiles, blocks, room, shortest)
        prefix_parts = min(SHARED_MAX_PARTS, -(-int(blocks.max()) // prefix_run))
        if captured:                            # (a table is chosen for rows of more than half its width)
            prefix_run = _shared_runs(tiles, -(-blocks // 2), room, shortest)
    # (tensors that are refilled with other groupings of so many rows in as many groups: none has more tiles, as a group's last tile
    # holds at least what both a tile and a row's heads are multiples of)
    count = int(tiles.sum())
    if shared.room is not None:
        count = (shared.room * fold + int((blocks > 0).sum()) * (tile - math.gcd(fold, tile))) // tile
    return SharedAttentionPlan(count, prefix_parts, prefix_run, tail_parts, tail_run, wide, warps)


def continuations(dtype, mixer, rows: int, context: int, page_size: int, sms: Optional[int] = None
                  ) -> Optional[SharedAttentionPlan]:
    """The plan of a decode step of ``rows`` continuations of one prompt of ``context`` tokens, if it reads their common keys once."""
    common = context // 64
    shared = SimpleNamespace(sizes=(rows,), blocks=(common,), tails=(1,) * rows, row_blocks=(common,) * rows, room=None, reach=None,
                             plans={})
    if not sharing_pays(shared.sizes, shared.blocks, shared_block_bytes(dtype, mixer.num_kv_heads, mixer.head_dim)):
        return None
    return shared_attention(dtype, num_heads=mixer.num_heads, num_kv_heads=mixer.num_kv_heads, head_dim=mixer.head_dim,
                            page_size=page_size, shared=shared, sms=sms)


def describe(model, row_counts: Sequence[int] = (1, 8, 16, 17, 64, 512, 2048), context: int = 4096,
             page_size: int = 16, sms: Optional[int] = None) -> str:
    """The plan of a built model as text: for every distinct layer and the head, the kernel of each operation at
    each of ``row_counts`` (a decode step of that many sequences; from 17 rows on also one prompt portion of
    that many rows)."""
    from .parts.attention import Attention
    from .parts.mlp import SwiGLU

    dtype = model.runtime.dtype
    lines: List[str] = [f"kernel plan for {model.spec.architecture} in {str(dtype).replace('torch.', '')} "
                        f"(context {context}, pages of {page_size})"]
    seen = {}
    for index, block in enumerate(model.layers):
        ff_spec = model.spec.layers[index].feed_forward
        key = (repr(model.spec.layers[index].mixer.params), repr(ff_spec.params if ff_spec is not None else None))
        if key in seen:
            seen[key].append(index)
            continue
        seen[key] = [index]
    for key, layers in seen.items():
        block = model.layers[layers[0]]
        lines.append(f"layers {layers[0]}..{layers[-1]} ({len(layers)}): mixer '{block.mixer.kind}', "
                     f"feed-forward '{block.feed_forward.kind if block.feed_forward is not None else None}'")
        for rows in row_counts:
            lines.append(f"  {rows} rows")
            mixer, ffn = block.mixer, block.feed_forward
            down_prepares = False
            if isinstance(ffn, SwiGLU):
                down_prepares = product(dtype, rows, ffn.down_proj.out_features, ffn.down_proj.in_features,
                                        follow=True).prepares_norm
            if isinstance(mixer, Attention):
                qkv = mixer.qkv_proj
                lines.append(f"    qkv      {product(dtype, rows, qkv.out_features, qkv.in_features, norm='add_norm')}")
                if down_prepares:
                    behind = product(dtype, rows, qkv.out_features, qkv.in_features, norm='prepared')
                    lines.append(f"             behind a layer whose down product prepared the norm: {behind}")
                decode = attention(dtype, num_heads=mixer.num_heads, num_kv_heads=mixer.num_kv_heads,
                                   head_dim=mixer.head_dim, page_size=page_size, new_tokens=[1] * rows,
                                   max_context=context, prompt_kernel=mixer.prompt_kernel, sms=sms)
                lines.append(f"    attend   decode step: {decode}")
                together = None if mixer.window else continuations(dtype, mixer, rows, context, page_size, sms)
                if together is not None:
                    lines.append(f"             of one prompt's continuations: {together}")
                if rows >= 17:
                    portion = attention(dtype, num_heads=mixer.num_heads, num_kv_heads=mixer.num_kv_heads,
                                        head_dim=mixer.head_dim, page_size=page_size, new_tokens=[rows],
                                        max_context=context, prompt_kernel=mixer.prompt_kernel, sms=sms)
                    lines.append(f"             one portion: {portion}")
                o = mixer.o_proj
                o_plan = product(dtype, rows, o.out_features, o.in_features, follow=True)
                lines.append(f"    o        {o_plan}")
            elif hasattr(mixer, "products"):
                lines.append(f"    mixer    '{mixer.kind}' (its own kernels between the products)")
                for name, linear, epilogue in mixer.products():
                    lines.append(f"      {name:10s} {product(dtype, rows, linear.out_features, linear.in_features, epilogue=epilogue)}")
                if hasattr(mixer, "attention_choice"):
                    lines.append(f"      attend     {mixer.attention_choice(rows)}")
                elif hasattr(mixer, "sides"):              # mixers side by side: each one's attention kernel
                    for side in mixer.sides:
                        if hasattr(side, "attention_choice"):
                            lines.append(f"      attend     '{side.kind}': {side.attention_choice(rows)}")
                elif hasattr(mixer, "num_kv_heads") and hasattr(mixer, "value_dim") and not hasattr(mixer, "taps"):
                    per = mixer.num_heads // mixer.num_kv_heads
                    lines.append(f"      attend     {masked_attention(dtype, rows, mixer.key_dim, mixer.value_dim, heads_per_kv=per)}")
            else:
                lines.append(f"    mixer    '{mixer.kind}' (its own code)")
            if isinstance(ffn, SwiGLU):
                gu, down = ffn.gate_up_proj, ffn.down_proj
                epilogue = SWIGLU if ffn.interleaved else BF16
                prepared = isinstance(mixer, Attention) and o_plan.prepares_norm
                lines.append(f"    gate/up  {product(dtype, rows, gu.out_features, gu.in_features, epilogue=epilogue, norm='prepared' if prepared else 'add_norm')}")
                lines.append(f"    down     {product(dtype, rows, down.out_features, down.in_features, follow=True)}")
            elif ffn is not None and hasattr(ffn, "products"):
                choices = [(name, product(dtype, rows, linear.out_features, linear.in_features, epilogue=epilogue))
                           for name, linear, epilogue in ffn.products()]
                inside = any(choice.epilogue in OVER_GATE_AND_UP for _, choice in choices)
                lines.append(f"    feed-forward '{ffn.kind}' "
                             f"({'activated by the product in front' if inside else 'its own kernel between the products'})")
                lines.extend(f"      {name:10s} {choice}" for name, choice in choices)
            elif ffn is not None:
                lines.append(f"    feed-forward '{ffn.kind}' (its own code)")
            gates = getattr(block, "gates", None)
            if gates is not None and hasattr(gates, "products"):
                lines.append(f"    residual gates '{gates.kind}' (the weighting, the addition and the next norm are one kernel)")
                for name, linear, epilogue in gates.products():
                    lines.append(f"      {name:10s} {product(dtype, rows, linear.out_features, linear.in_features, epilogue=epilogue)}")
    for index, injection in enumerate(getattr(model, "injections", ())):
        entries = [i for i, entry in enumerate(model.spec.run_order) if entry.inject == index]
        lines.append(f"injection '{injection.kind}' in front of run entries {entries}")
        for rows in row_counts:
            for name, linear, epilogue in (injection.products() if hasattr(injection, "products") else []):
                lines.append(f"  {rows} rows  {name:10s} {product(dtype, rows, linear.out_features, linear.in_features, epilogue=epilogue)}")
    proj = getattr(model.head, "proj", None)
    if proj is not None:
        lines.append("head (wanted rows only)")
        for rows in row_counts:
            text = f"  {rows} rows  {product(dtype, rows, proj.out_features, proj.in_features, epilogue=F32, norm='add_norm')}"
            behind = product(dtype, rows, proj.out_features, proj.in_features, epilogue=F32, norm='prepared')
            if behind.takes_prepared:
                text += f"; on every row of a step: {behind}"
            lines.append(text)
    return "\n".join(lines)
