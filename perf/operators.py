"""What the operators behind many continuations of one prompt cost.

A server that continues a prompt in several ways (parallel samples, beams, questions about one document) stores the prompt's
keys once, reads them once a step for all continuations, and asks how probable what it produced is:

``copy_pages``        a fork copies the page that is still being filled (and a request's states), a compaction moves pages down
``attention_shared``  one decoded row a continuation: the keys in common read once for all rows of a group, each row's own behind
``token_logprobs``    log probabilities of given tokens, the entropy, and the most probable alternatives, from 32-bit logits

Layer sizes are those of ``bench.py`` (the 1B and 8B Llama sizes, the 3B's 24 heads) and of the tests; page sizes and contexts
those of the engine's options.  A row of attention reads keys 0 to its position; a row at position -1 (one that pads a captured
step up to its size) reads nothing and gives zeros.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}

# ----------------------------------------------------------------------------- cases


def _copy(name, dtype, entries, pages, moved, page, slots=0, state=0):
    """``page``: numbers of a page of one entry; ``slots``, ``state``: as many states of that many 32-bit numbers are copied in the
    same call."""
    return {"name": name, "op": "copy_pages", "dtype": dtype, "entries": entries, "pages": pages, "moved": moved, "page": page,
            "slots": slots, "state": state}


def _attention(name, dtype, heads, kv_heads, dim, page_size, groups, least, most, prefix_least, prefix_most, tail_most, padding=0):
    """``groups`` groups of ``least`` to ``most`` rows over ``prefix_least`` to ``prefix_most`` keys in common, and 1 to
    ``tail_most`` keys of each row's own."""
    return {"name": name, "op": "attention_shared", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page_size": page_size, "groups": groups, "least": least, "most": most, "prefix_least": prefix_least,
            "prefix_most": prefix_most, "tail_most": tail_most, "padding": padding, "lengths": groups * 7919 + most}


def _logprobs(name, rows, vocab, top, apart=0, allowed=1.0):
    """``apart``: numbers between the end of a row and the next; ``allowed``: the share of the vocabulary that is not masked."""
    return {"name": name, "op": "token_logprobs", "rows": rows, "vocab": vocab, "top": top, "apart": apart, "allowed": allowed}


def listed():
    return [
        # four beams of the 1B model part: the page being filled of three of them, in all 16 layers (the smallest call)
        _copy("fork_beams_4", "bfloat16", 16, 2048, 3, 2 * 8 * 16 * 64),
        # 31 samples of one prompt split off at the 8B sizes of a model that keeps a state per request as well
        _copy("fork_samples_31_states", "bfloat16", 32, 1024, 31, 2 * 8 * 16 * 128, 31, 16 * 128 * 128),
        # a pool is compacted: 1,500 pages of 32-bit keys and values move
        _copy("compact_1500_f32", "float32", 8, 4096, 1500, 2 * 8 * 16 * 64),
        # four beams behind a short question
        _attention("beams_4_at_200", "bfloat16", 32, 8, 64, 16, 1, 4, 4, 200, 200, 12),
        # sixteen samples of one prompt of the headline length
        _attention("samples_16_at_2k", "bfloat16", 32, 8, 64, 16, 1, 16, 16, 2048, 2048, 200),
        # a busy server: requests of six system prompts of all lengths, padded up to a captured size
        _attention("six_prompts_8b", "bfloat16", 32, 8, 128, 16, 6, 3, 17, 300, 6000, 500, 3),
        # 64 questions about one long document
        _attention("document_64_at_32k", "bfloat16", 32, 8, 128, 16, 1, 64, 64, 32768, 32768, 300),
        # the 32-bit path: beams at an odd length
        _attention("beams_8_f32", "float32", 32, 8, 64, 16, 1, 8, 8, 1111, 1111, 40),
        # four beams choose their next tokens
        _logprobs("beams_4_top_8", 4, 128256, 8),
        # a decode step of 64 rows with the twenty best
        _logprobs("step_64_top_20", 64, 128256, 20),
        # a constrained step: nine tenths of an odd vocabulary masked, rows apart
        _logprobs("masked_33_top_5", 33, 50257, 5, 7, 0.1),
        # every place of a prompt is scored
        _logprobs("prompt_1536_top_1", 1536, 128256, 1),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["copy_pages", "attention_shared", "attention_shared", "token_logprobs"])
    limit = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op == "copy_pages":
            dtype = rng.choice(["bfloat16", "float32"])
            heads, size, dim = rng.choice([1, 2, 4, 8]), rng.choice([8, 16, 32, 64]), rng.choice([16, 64, 80, 128, 256])
            states = rng.random() < 0.4
            pages = _log_int(rng, 16, 4096)
            case = _copy("", dtype, rng.randint(1, 32), pages, _log_int(rng, 1, pages // 2), 2 * heads * size * dim,
                         _log_int(rng, 1, 48) if states else 0, rng.choice([257, 4096, 65536, 100003]) if states else 0)
            if 4 * (case["entries"] * pages * case["page"] + 97 * case["entries"] * case["state"]) > 3e9:
                continue
        elif op == "attention_shared":
            dtype = "float32" if rng.random() < 0.2 else "bfloat16"
            heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (24, 8, 128), (16, 4, 64), (4, 2, 16), (20, 4, 80), (16, 1, 128),
                                               (8, 8, 64), (8, 2, 256), (48, 2, 64)])
            groups = _log_int(rng, 1, 16)
            most = _log_int(rng, 1, 64)
            longest = _log_int(rng, 16, 32768)
            case = _attention("", dtype, heads, kv_heads, dim, rng.choice([8, 16, 16, 16, 32, 64]), groups, rng.randint(1, most), most,
                              _log_int(rng, 1, longest), longest, _log_int(rng, 1, 700), rng.randint(0, 3))
            case["lengths"] = rng.randrange(1 << 30)
            if groups * most > 128:
                continue
        else:
            case = _logprobs("", _log_int(rng, 1, 1536), _log_int(rng, 256, 150000), rng.choice([1, 2, 5, 8, 20, 40, 64]),
                             rng.choice([0, 0, 1, 7, 64]), rng.choice([1.0, 1.0, 0.5, 0.01]))
        if _cost(case) <= limit:
            del case["name"]
            return case


def _lengths(case):
    """The sizes of the groups, their keys in common, and the position of every row, group by group."""
    rng = np.random.RandomState(case["lengths"] % (1 << 31))
    sizes = rng.randint(case["least"], case["most"] + 1, case["groups"])
    prefixes = rng.randint(case["prefix_least"], case["prefix_most"] + 1, case["groups"])
    tails = [rng.randint(1, case["tail_most"] + 1, n) for n in sizes]
    return sizes, prefixes, [p + t - 1 for p, t in zip(prefixes, tails)]


def work(case):
    if case["op"] == "copy_pages":
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": 2 * case["entries"] * (case["moved"] * case["page"] * size + case["slots"] * case["state"] * 4), "flops": 0}
    if case["op"] == "attention_shared":
        sizes, prefixes, positions = _lengths(case)
        size = 2 if case["dtype"] == "bfloat16" else 4
        keys = int(sum(prefixes)) + sum(int((p + 1 - shared).sum()) for shared, p in zip(prefixes, positions))
        rows = int(sum(sizes)) + case["padding"]
        scores = sum(int((p + 1).sum()) for p in positions)
        return {"bytes": size * case["dim"] * (2 * case["kv_heads"] * keys + 2 * case["heads"] * rows),
                "flops": 4 * case["dim"] * case["heads"] * scores}
    return {"bytes": case["rows"] * (4 * case["vocab"] + 4 + 8 + 8 * case["top"]), "flops": 0}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / (1e15 if case.get("dtype") == "bfloat16" else 5e13))


# ----------------------------------------------------------------------------- what a program has in hand


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _inputs(case, seed):
    """Everything on the device from the seed alone; index lists as numpy arrays on the host."""
    gen, host = _generator(seed), np.random.RandomState(int(seed) % (1 << 31))
    if case["op"] == "copy_pages":
        def moves(count, pages):
            places = host.permutation(pages)
            return places[:count].astype(np.int32), places[count:2 * count].astype(np.int32)

        store = torch.randn(case["entries"], case["pages"], case["page"], generator=gen, device="cuda", dtype=torch.float32
                            ).to(DTYPES[case["dtype"]])
        out = [(store, *moves(case["moved"], case["pages"]))]
        if case["slots"]:
            states = torch.randn(case["entries"], 2 * case["slots"] + 1, case["state"], generator=gen, device="cuda")
            out.append((states, *moves(case["slots"], 2 * case["slots"] + 1)))
        return out
    if case["op"] == "attention_shared":
        sizes, prefixes, positions = _lengths(case)
        dtype, size, dim = DTYPES[case["dtype"]], case["page_size"], case["dim"]
        rows = int(sum(sizes)) + case["padding"]
        columns = max(-(-int(p.max() + 1) // size) for p in positions)
        table = np.zeros((rows, columns), dtype=np.int32)
        at, row, groups = 1, 0, []
        for n, shared, last in zip(sizes, prefixes, positions):
            common = int(shared) // size                       # whole pages are shared, the page being filled is a copy
            for k in range(int(n)):
                pages = -(-(int(last[k]) + 1) // size)
                table[row, :common] = np.arange(at, at + common)
                own_at = at + common + (sum(-(-(int(p) + 1) // size) - common for p in last[:k]))
                table[row, common:pages] = np.arange(own_at, own_at + pages - common)
                row += 1
            at += common + sum(-(-(int(p) + 1) // size) - common for p in last)
            groups.append(list(range(row - int(n), row)))
        order = np.concatenate([[0], 1 + host.permutation(at - 1)]).astype(np.int32)    # pages lie anywhere in the pool
        table = order[table]
        last = np.concatenate([p for p in positions] + [np.full(case["padding"], -1)]).astype(np.int32)
        groups += [[r] for r in range(row, rows)]
        prefixes = np.concatenate([prefixes, np.zeros(case["padding"])]).astype(np.int32)
        # rows stand in the batch in any order
        place = host.permutation(rows)
        table[place], last[place] = table.copy(), last.copy()
        groups = [[int(place[r]) for r in g] for g in groups]
        cache = torch.randn(at, 2, case["kv_heads"], size, dim, generator=gen, device="cuda")
        # the page being filled holds the same numbers in every row of its group
        for g, shared in zip(groups, prefixes):
            common, rest = int(shared) // size, int(shared) % size
            if rest:
                others = torch.from_numpy(table[g[1:], common].astype(np.int64)).cuda()
                cache[others, :, :, :rest] = cache[int(table[g[0], common]), :, :, :rest].clone()
        # a row's projections as they leave the fused product: queries, then the new key and value; scores of a few units
        qkv = torch.randn(rows, (case["heads"] + 2 * case["kv_heads"]) * dim, generator=gen, device="cuda") * 1.5
        return {"qkv": qkv.to(dtype), "cache": cache.to(dtype), "table": torch.from_numpy(table).cuda(),
                "positions": torch.from_numpy(last).cuda(), "groups": groups, "prefixes": [int(p) for p in prefixes],
                "last": [int(p) for p in last]}
    width = case["vocab"] + case["apart"]
    logits = torch.randn(case["rows"], width, generator=gen, device="cuda") * 2.5
    logits = logits[:, :case["vocab"]]
    if case["allowed"] < 1.0:
        masked = torch.rand(case["rows"], case["vocab"], generator=gen, device="cuda") >= case["allowed"]
        masked[:, case["vocab"] // 2] = False                  # something is always allowed
        logits.masked_fill_(masked, -math.inf)
    tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda", dtype=torch.int32)
    return {"logits": logits, "tokens": tokens}


def prepare(case, seed):
    state = {"case": dict(case)}
    if case["op"] == "copy_pages":
        state["moves"] = _inputs(case, seed)
        if not own:
            state["moves"] = [(store, torch.from_numpy(a.astype(np.int64)).cuda(), torch.from_numpy(b.astype(np.int64)).cuda())
                              for store, a, b in state["moves"]]
        return state
    state.update(_inputs(case, seed))
    if case["op"] == "attention_shared":
        state["q"] = state["qkv"][:, :case["heads"] * case["dim"]]
        state["out"] = torch.empty(state["q"].shape, dtype=state["q"].dtype, device="cuda")
        if own:
            from tesseract_b200.parts.base import SharedRows

            state["shared"] = SharedRows.of(state["groups"], state["prefixes"], state["last"], "cuda")
        else:
            state["members"] = [torch.tensor(g, device="cuda") for g in state["groups"]]
    return state


# ----------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "copy_pages":
        for store, sources, targets in state["moves"]:
            store[:, targets] = store[:, sources]
        return [store for store, _, _ in state["moves"]]
    if case["op"] == "attention_shared":
        return _attend(case, state)
    return _logprobs_plain(state["logits"], state["tokens"], case["top"])


def _run_own(case, state):
    from tesseract_b200 import kernels, plan

    if case["op"] == "copy_pages":
        kernels.copy_pages(state["moves"])
        return [store for store, _, _ in state["moves"]]
    if case["op"] == "attention_shared":
        shared = state["shared"]
        choice = plan.shared_attention(state["q"].dtype, num_heads=case["heads"], num_kv_heads=case["kv_heads"],
                                       head_dim=case["dim"], page_size=case["page_size"], shared=shared)
        return kernels.attention_shared(state["q"], state["out"], state["cache"], state["positions"], state["table"], shared,
                                        case["heads"], case["kv_heads"], case["dim"], case["page_size"],
                                        1.0 / math.sqrt(case["dim"]), choice)
    return list(kernels.token_logprobs(state["logits"], state["tokens"], case["top"]))


def _attend(case, state):
    """Group by group: the keys in common gathered once and scored for all of its rows, each row's own behind them."""
    heads, kv_heads, dim, size = case["heads"], case["kv_heads"], case["dim"], case["page_size"]
    fold, out, scale = heads // kv_heads, state["out"], 1.0 / math.sqrt(dim)
    out.zero_()
    for members, rows, shared in zip(state["members"], state["groups"], state["prefixes"]):
        last = [state["last"][r] for r in rows]
        if max(last) < 0:
            continue
        common = min(shared, min(last) + 1)
        span = max(last) + 1 - common
        q = state["q"].index_select(0, members).float().view(len(rows), kv_heads, fold, dim)
        table = state["table"].index_select(0, members).long()
        first = torch.arange(common, device="cuda")
        own_keys = common + torch.arange(span, device="cuda")
        pages = state["cache"][table[0, first // size], :, :, first % size].float()              # [common, 2, kv, dim]
        reach = own_keys.clamp(max=table.shape[1] * size - 1)
        tails = state["cache"][table[:, reach // size], :, :, (reach % size).expand(len(rows), -1)].float()   # [n, span, 2, kv, dim]
        scores = torch.cat([torch.einsum("nkgd,lkd->nkgl", q, pages[:, 0]),
                            torch.einsum("nkgd,nlkd->nkgl", q, tails[:, :, 0])], dim=-1) * scale
        ends = state["positions"].index_select(0, members)
        visible = torch.cat([torch.ones(len(rows), common, dtype=torch.bool, device="cuda"), own_keys <= ends[:, None]], dim=1)
        scores = scores.masked_fill(~visible[:, None, None, :], -math.inf)
        weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
        weights = weights / weights.sum(dim=-1, keepdim=True)
        tails = torch.where(visible[:, common:, None, None], tails[:, :, 1], torch.zeros((), device="cuda"))
        made = torch.einsum("nkgl,lkd->nkgd", weights[..., :common], pages[:, 1])
        made = made + torch.einsum("nkgl,nlkd->nkgd", weights[..., common:], tails)
        out.index_copy_(0, members, made.reshape(len(rows), heads * dim).to(out.dtype))
    return out


def _logprobs_plain(logits, tokens, top):
    got, entropy, values, ids = [], [], [], []
    for at in range(0, logits.shape[0], 256):
        x = logits[at:at + 256]
        shifted = x - x.amax(dim=1, keepdim=True)
        e = torch.exp(shifted)
        total = e.sum(dim=1, keepdim=True)
        logs = torch.log(total)
        given = tokens[at:at + 256].long()[:, None]
        got.append((shifted.gather(1, given) - logs)[:, 0])
        weighted = torch.where(e > 0, shifted * e, torch.zeros((), device=x.device))
        entropy.append((logs - weighted.sum(dim=1, keepdim=True) / total)[:, 0])
        best, where = torch.sort(shifted, dim=1, descending=True, stable=True)      # ties: the lowest id first
        values.append(best[:, :top] - logs)
        ids.append(where[:, :top].to(torch.int32))
    return [torch.cat(got), torch.cat(entropy), torch.cat(values), torch.cat(ids)]


# ----------------------------------------------------------------------------- from the definition, in 64 bits


def exact(case, seed):
    made = _inputs(case, seed)
    if case["op"] == "copy_pages":
        out = []
        for store, sources, targets in made:
            comes_from = torch.arange(store.shape[1])
            comes_from[torch.from_numpy(targets).long()] = torch.from_numpy(sources).long()
            out.append(store.index_select(1, comes_from.cuda()))
        return out
    if case["op"] == "attention_shared":
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        out = torch.zeros(len(made["last"]), heads * dim, dtype=torch.float64, device="cuda")
        for row, last in enumerate(made["last"]):
            if last < 0:
                continue
            pages = made["table"][row, :last // case["page_size"] + 1].long()
            kv = made["cache"][pages].double().permute(1, 2, 0, 3, 4).reshape(2, kv_heads, -1, dim)[:, :, :last + 1]
            q = made["qkv"][row, :heads * dim].double().view(kv_heads, heads // kv_heads, dim)
            weights = torch.softmax(q @ kv[0].transpose(1, 2) / math.sqrt(dim), dim=-1)
            out[row] = (weights @ kv[1]).reshape(-1)
        return out
    got, entropy, values, ids = [], [], [], []
    for row in range(case["rows"]):
        x = made["logits"][row].double()
        logs = x - torch.logsumexp(x, dim=0)
        got.append(logs[made["tokens"][row].long()])
        entropy.append(torch.special.entr(torch.exp(logs)).sum())
        order = torch.argsort(logs, descending=True, stable=True)[:case["top"]]
        values.append(logs[order])
        ids.append(order.to(torch.int32))
    return [torch.stack(got), torch.stack(entropy), torch.stack(values), torch.stack(ids)]
