"""What the operators behind a request's say in its next token cost.

A server that lets a request shape what comes next (penalties for tokens it has had, biases on tokens, a grammar's mask, and cuts of
the distribution) keeps a history of tokens a request, and on every step takes the step's logits to one token a row:

``note_tokens``    a request's known tokens go into its history: a bit for every token it has had, and how often it generated each
``shape_logits``   penalties, biases and the mask applied to 32-bit logits, written out (beam search ranks what comes out)
``choose_tokens``  the same on the way to a token: greedy, or drawn after top-k, min-p and top-p, for a given uniform draw

The rules, for a logit ``l`` of a token that the request has had ``c`` times in its answer::

    x = l;   x = x / repetition if x > 0 else x * repetition   (tokens of the prompt and the answer)
    x = x - frequency * c;   x = x - presence if c > 0;   x = x + bias;   -inf where the mask does not allow the token

in 64 bits, rounded once.  The choice: with a temperature of 0 the lowest id of the largest; else z = x * (1 / temperature) and
d = z - max z in 32 bits each, weights exp(d) in 64, tokens ranked by descending d, equal ones by id; of the rank the first
``top_k``, of those weights of ``min_p`` and more, of those the shortest beginning that holds ``top_p`` of their mass; and of what is
left the first token whose cumulative weight passes the draw's share of the whole.  A row without a cut is drawn from in the order of ids
(with z - max z rounded once).

The vocabulary is that of ``bench.py``'s layer sizes and others of common sizes, row counts those of the engine's decode steps.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

# ----------------------------------------------------------------------------- cases


def _note(name, rows, vocab, least, most, answered):
    """``rows`` requests of ``least`` to ``most`` known tokens, of which the last ``answered`` (a share) were generated."""
    return {"name": name, "op": "note_tokens", "rows": rows, "vocab": vocab, "least": least, "most": most, "answered": answered,
            "lengths": rows * 7919 + most}


def _rules(op, name, rows, vocab, history, biases, allowed, apart, spread):
    """``history``: the most tokens that a row's request has had (0: no penalties); ``biases``: tokens with a bias; ``allowed``: the
    share of the vocabulary that the mask leaves (1: no mask); ``apart``: numbers between the end of a row and the next; ``spread``:
    standard deviation of the logits."""
    return {"name": name, "op": op, "rows": rows, "vocab": vocab, "history": history, "biases": biases, "allowed": allowed,
            "apart": apart, "spread": spread, "lengths": rows * 7919 + history}


def _shape(name, rows, vocab, history, biases, allowed, apart=0):
    return _rules("shape_logits", name, rows, vocab, history, biases, allowed, apart, 2.5)


def _choose(name, rows, vocab, history, biases, allowed, temperature, top_k, top_p, min_p, apart=0, spread=2.5, mixed=False):
    """``mixed``: rows take turns with the case's settings, none of the cuts, greedy, top-k alone and min-p alone."""
    case = _rules("choose_tokens", name, rows, vocab, history, biases, allowed, apart, spread)
    case.update(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, mixed=mixed)
    return case


def listed():
    return [
        # a request is admitted: its prompt goes into its history
        _note("admit_1", 1, 128256, 200, 200, 0.0),
        # requests come back with all that they had: prompts and answers of up to 8,192 tokens
        _note("resume_32", 32, 128256, 1, 8192, 0.4),
        # four beams under a repetition penalty and a few biases
        _shape("beams_4", 4, 128256, 2000, 16, 1.0),
        # a decode step whose rows all have a grammar, penalties and biases
        _shape("grammar_64", 64, 128256, 4000, 16, 0.1),
        # biases alone, an odd vocabulary, rows apart
        _shape("biases_33_odd", 33, 50257, 0, 300, 1.0, 7),
        # one chat, nucleus sampling (the smallest choice)
        _choose("top_p_1", 1, 128256, 0, 0, 1.0, 0.8, 0, 0.9, 0.0),
        # greedy rows under penalties
        _choose("greedy_8", 8, 128256, 1000, 0, 1.0, 0.0, 0, 1.0, 0.0),
        # sixteen chats with a list of candidates and a floor
        _choose("top_k_16", 16, 128256, 2000, 0, 1.0, 0.7, 50, 0.95, 0.05),
        # a busy server: every kind of request in one step, penalties, biases and grammars in all
        _choose("mixed_64", 64, 128256, 4000, 16, 0.5, 1.0, 200, 0.9, 0.02, mixed=True),
        # creative writing: a hot, flat distribution whose nucleus is a large part of the vocabulary
        _choose("flat_32", 32, 128256, 2000, 0, 1.0, 1.5, 0, 0.95, 0.0, spread=1.2),
        # an odd vocabulary under a tight grammar, rows apart
        _choose("grammar_33_odd", 33, 50257, 300, 5, 0.01, 0.9, 0, 0.9, 0.0, 7),
        # the largest step that the engine's options allow for, nucleus sampling
        _choose("top_p_256", 256, 128256, 0, 0, 1.0, 0.8, 0, 0.9, 0.0),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["note_tokens", "shape_logits", "choose_tokens", "choose_tokens"])
    limit = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        vocab = _log_int(rng, 256, 150000) if rng.random() < 0.6 else rng.choice([32000, 50257, 128256, 151936])
        rows = _log_int(rng, 1, 256)
        if op == "note_tokens":
            most = _log_int(rng, 1, 16384)
            case = _note("", min(rows, 64), vocab, rng.randint(1, most), most, rng.choice([0.0, 0.4, 1.0]))
            case["lengths"] = rng.randrange(1 << 30)
        else:
            shared = (rows, vocab, rng.choice([0, 0, 1, _log_int(rng, 2, 8192)]), rng.choice([0, 0, 1, 16, 300]),
                      rng.choice([1.0, 1.0, 0.9, 0.1, 0.003]))
            apart = rng.choice([0, 0, 1, 7, 64])
            if op == "shape_logits":
                case = _shape("", *shared, apart)
            else:
                case = _choose("", *shared, rng.choice([0.0, 0.3, 0.7, 1.0, 1.7]), rng.choice([0, 0, 1, 5, 50, 1000]),
                               rng.choice([1.0, 0.99, 0.9, 0.5]), rng.choice([0.0, 0.0, 0.01, 0.1]), apart,
                               rng.choice([0.7, 1.5, 2.5, 4.0]), rng.random() < 0.3)
            case["lengths"] = rng.randrange(1 << 30)
        if _cost(case) <= limit:
            del case["name"]
            return case


def _lengths(case):
    """How many tokens every row's request has had, and how many of them were its prompt's."""
    rng = np.random.RandomState(case["lengths"] % (1 << 31))
    if case["op"] == "note_tokens":
        counts = rng.randint(case["least"], case["most"] + 1, case["rows"])
        return counts, counts - (counts * case["answered"]).astype(np.int64)
    counts = rng.randint(case["history"] // 10, case["history"] + 1, case["rows"])
    return counts, counts // 2


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    bits = 4 * -(-vocab // 32)
    had = int(_lengths(case)[0].sum())
    if case["op"] == "note_tokens":
        return {"bytes": 4 * had + 8 * rows + rows * (4 * vocab + bits), "flops": 0}
    # a bit a token for what was had and one for the mask, the counts of tokens that were had, the biases
    rules = (rows * bits + 4 * had if case["history"] else 0) + (rows * bits if case["allowed"] < 1.0 else 0) + 8 * rows * case["biases"]
    return {"bytes": rows * 4 * vocab + rules + (4 * vocab * rows if case["op"] == "shape_logits" else 36 * rows), "flops": 0}


def _cost(case):
    return work(case)["bytes"]


# ----------------------------------------------------------------------------- what a program has in hand


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _pack(bits):
    """Truth values ``[n, V]`` as int32 words, bit ``i % 32`` of word ``i // 32``."""
    rows, vocab = bits.shape
    words = -(-vocab // 32)
    whole = torch.zeros(rows, words * 32, dtype=torch.int64, device=bits.device)
    whole[:, :vocab] = bits
    packed = (whole.view(rows, words, 32) << torch.arange(32, device=bits.device)).sum(dim=2)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _known_tokens(case, gen):
    """Every row's known tokens one behind the other (few of them often, as in text), their row and their place in it."""
    counts, prompts = _lengths(case)
    total = int(counts.sum())
    tokens = (torch.rand(total, generator=gen, device="cuda", dtype=torch.float64) ** 3 * case["vocab"]).to(torch.int32)
    row = torch.from_numpy(np.repeat(np.arange(case["rows"]), counts)).cuda()
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    place = torch.arange(total, device="cuda") - torch.from_numpy(starts[:-1].astype(np.int64)).cuda()[row]
    return tokens, row, place, torch.from_numpy(starts).cuda(), torch.from_numpy(prompts.astype(np.int32)).cuda()


def _inputs(case, seed):
    """Everything on the device, from the seed alone.  A row's rules are those of its slot."""
    gen, host = _generator(seed), np.random.RandomState(int(seed) % (1 << 31))
    rows, vocab = case["rows"], case["vocab"]
    slots = rows + 3
    made = {"slots": torch.from_numpy(host.permutation(slots)[:rows].astype(np.int32)).cuda()}
    tokens, row, place, starts, prompts = _known_tokens(case, gen)
    if case["op"] == "note_tokens":
        made.update(tokens=tokens, row=row, place=place, starts=starts, prompts=prompts)
        return made
    at = made["slots"].long()
    counts = torch.zeros(slots, vocab, dtype=torch.int32, device="cuda")
    had = torch.zeros(slots, vocab, dtype=torch.bool, device="cuda")
    had[at[row], tokens.long()] = True
    counts.view(-1).index_add_(0, at[row] * vocab + tokens.long(), (place >= prompts[row]).to(torch.int32))
    penalties = torch.rand(slots, 3, generator=gen, device="cuda") * torch.tensor([0.4, 0.8, 0.5], device="cuda")
    penalties[:, 0] += 1.0
    made.update(had=had, counts=counts, penalties=penalties)
    ids = torch.rand(slots, vocab, generator=gen, device="cuda").argsort(dim=1)[:, :min(case["biases"], vocab)] if case["biases"] else None
    made["bias_ids"] = ids
    made["biases"] = torch.randn(ids.shape, generator=gen, device="cuda") * 3.0 if ids is not None else None
    made["allowed"] = None
    if case["allowed"] < 1.0:
        allowed = torch.rand(slots, vocab, generator=gen, device="cuda") < case["allowed"]
        allowed[:, vocab // 2] = True                          # something may always come next
        made["allowed"] = allowed
    logits = torch.randn(rows, vocab + case["apart"], generator=gen, device="cuda") * case["spread"]
    made["logits"] = logits[:, :vocab]
    if case["op"] == "choose_tokens":
        n = rows
        turn = torch.arange(n, device="cuda") % 5 if case["mixed"] else torch.zeros(n, dtype=torch.long, device="cuda")
        made["temperature"] = torch.full((n,), case["temperature"], device="cuda").masked_fill(turn == 2, 0.0)
        made["top_k"] = torch.full((n,), case["top_k"], dtype=torch.int32, device="cuda").masked_fill((turn == 1) | (turn == 4), 0)
        made["top_p"] = torch.full((n,), case["top_p"], dtype=torch.float64, device="cuda").masked_fill((turn == 1) | (turn >= 3), 1.0)
        made["min_p"] = torch.full((n,), case["min_p"], dtype=torch.float64, device="cuda").masked_fill((turn == 1) | (turn == 3), 0.0)
        made["uniform"] = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return made


def prepare(case, seed):
    state = {"case": dict(case)}
    state.update(_inputs(case, seed))
    rows, vocab = case["rows"], case["vocab"]
    if own:
        from tesseract_b200.sampling import TokenRules

        rules = TokenRules(rows + 3, vocab, "cuda", biases=case.get("biases", 0))
        state["rules"] = rules
        if case["op"] != "note_tokens":
            penalties = state["penalties"].double().tolist()
            for slot in range(rows + 3):
                repetition, presence, frequency = penalties[slot] if case["history"] else (1.0, 0.0, 0.0)
                rules.set(slot, repetition=repetition, presence=presence, frequency=frequency)
            rules.seen.copy_(_pack(state["had"]))
            rules.counts.copy_(state["counts"])
            if case["biases"]:
                rules.set_biases(state["bias_ids"], state["biases"])
            if state["allowed"] is not None:
                rules.set_masks(_pack(state["allowed"]))
    elif case["op"] == "note_tokens":
        state["counts"] = torch.zeros(rows + 3, vocab, dtype=torch.int32, device="cuda")
        state["seen"] = torch.zeros(rows + 3, -(-vocab // 32), dtype=torch.int32, device="cuda")
    elif state["allowed"] is not None or case["history"]:
        # (the plain form reads its bits from the same words)
        state["seen"] = _pack(state["had"])
        state["masks"] = _pack(state["allowed"]) if state["allowed"] is not None else None
    for name in ("had", "allowed"):
        state.pop(name, None)
    if case["op"] == "shape_logits":
        state["out"] = torch.empty(rows, vocab, device="cuda")
    elif case["op"] == "choose_tokens":
        state["out"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    return state


# ----------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "note_tokens":
        return _note_plain(case, state)
    if case["op"] == "shape_logits":
        return _shape_plain(case, state)
    return _choose_plain(_shape_plain(case, state), state)


def _run_own(case, state):
    from tesseract_b200 import kernels

    rules, slots = state["rules"], state["slots"]
    if case["op"] == "note_tokens":
        kernels.note_tokens(rules, slots, state["tokens"], starts=state["starts"], prompts=state["prompts"], restart=True)
        return [rules.counts, rules.seen]
    if case["op"] == "shape_logits":
        return kernels.shape_logits(state["logits"], state["out"], rules, slots)
    return kernels.choose_tokens(state["logits"], state["temperature"], state["uniform"], state["out"], top_k=state["top_k"],
                                 top_p=state["top_p"], min_p=state["min_p"], rules=rules, slots=slots)


def _note_plain(case, state):
    at, vocab, counts, seen = state["slots"].long(), case["vocab"], state["counts"], state["seen"]
    row, tokens = state["row"], state["tokens"].long()
    mine = torch.zeros(case["rows"], vocab, dtype=torch.int32, device=counts.device)
    mine.view(-1).index_add_(0, row * vocab + tokens, (state["place"] >= state["prompts"][row]).to(torch.int32))
    had = torch.zeros(case["rows"], vocab, dtype=torch.bool, device=counts.device)
    had[row, tokens] = True
    counts[at] = mine
    seen[at] = _pack(had)
    return [counts, seen]


def _bits(words, vocab):
    return ((words[:, :, None] >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1).view(words.shape[0], -1)[:, :vocab] != 0


def _shape_plain(case, state):
    at, vocab = state["slots"].long(), case["vocab"]
    x = state["logits"].double()
    if case["history"]:
        repetition, presence, frequency = (p[:, None] for p in state["penalties"][at].double().unbind(1))
        seen, counts = _bits(state["seen"][at], vocab), state["counts"][at].double()
        x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
        x = x - frequency * counts
        x = torch.where(counts > 0, x - presence, x)
    if case["biases"]:
        x = x.scatter_add(1, state["bias_ids"][at], state["biases"][at].double())
    if case["allowed"] < 1.0:
        x = torch.where(_bits(state["masks"][at], vocab), x, torch.full((), -math.inf, dtype=x.dtype, device=x.device))
    return x.float()


def _choose_plain(x, state):
    temperature, vocab = state["temperature"][:, None], x.shape[1]
    best, lowest = x.amax(dim=1, keepdim=True), x.argmax(dim=1)
    first = torch.arange(vocab, device=x.device).expand_as(x)
    lowest = torch.where(x == best, first, vocab).amin(dim=1)
    inverse = 1.0 / torch.where(temperature > 0, temperature, torch.ones_like(temperature))
    k, top_p, min_p = state["top_k"][:, None], state["top_p"][:, None], state["min_p"][:, None]
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    cut = (k < vocab) | (top_p < 1) | (min_p > 0)
    scaled = x * inverse
    once = (x.double() * inverse.double() - (best * inverse).double()).float()
    d = torch.where(cut, scaled - best * inverse, once)
    order = torch.where(cut, torch.sort(d, dim=1, descending=True, stable=True)[1], first)
    weights = torch.exp(d.double()).gather(1, order)
    weights = torch.where((first < k) & (weights >= min_p), weights, torch.zeros_like(weights))
    sums = torch.cumsum(weights, dim=1)
    kept = ((sums < sums[:, -1:] * top_p).sum(dim=1, keepdim=True) + 1).clamp(max=vocab)
    kept = torch.where(top_p < 1, kept, vocab)
    mass = sums.gather(1, kept - 1)
    picked = (sums <= state["uniform"][:, None] * mass).sum(dim=1, keepdim=True)
    token = order.gather(1, torch.minimum(picked, kept - 1))[:, 0]
    return torch.where(state["temperature"] > 0, token, lowest).to(torch.int32)


# ----------------------------------------------------------------------------- from the definition, in 64 bits


def _shaped(case, made, row):
    slot = int(made["slots"][row])
    x = made["logits"][row].cpu().numpy().astype(np.float64)
    if case["history"]:
        repetition, presence, frequency = made["penalties"][slot].cpu().numpy().astype(np.float64)
        had, times = made["had"][slot].cpu().numpy(), made["counts"][slot].cpu().numpy()
        for token in np.flatnonzero(had):
            x[token] = x[token] / repetition if x[token] > 0 else x[token] * repetition
            x[token] -= frequency * times[token]
            x[token] -= presence if times[token] else 0.0
    if case["biases"]:
        x[made["bias_ids"][slot].cpu().numpy()] += made["biases"][slot].cpu().numpy()
    if case["allowed"] < 1.0:
        x[~made["allowed"][slot].cpu().numpy()] = -np.inf
    return x


def exact(case, seed):
    made = _inputs(case, seed)
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "note_tokens":
        counts = np.zeros((rows + 3, vocab), dtype=np.int32)
        seen = np.zeros((rows + 3, -(-vocab // 32) * 32), dtype=np.uint8)
        tokens, slots = made["tokens"].cpu().numpy(), made["slots"].cpu().numpy()
        starts, prompts = made["starts"].cpu().numpy(), made["prompts"].cpu().numpy()
        for row in range(rows):
            known = tokens[starts[row]:starts[row + 1]]
            seen[slots[row], known] = 1
            counts[slots[row]] = np.bincount(known[prompts[row]:], minlength=vocab)
        return [counts, np.packbits(seen, axis=1, bitorder="little").view(np.int32)]
    if case["op"] == "shape_logits":
        return np.stack([_shaped(case, made, row) for row in range(rows)])
    out = np.empty(rows, dtype=np.int32)
    for row in range(rows):
        x = _shaped(case, made, row).astype(np.float32)
        temperature = np.float32(made["temperature"][row].item())
        if temperature <= 0:
            out[row] = int(np.argmax(x))
            continue
        inverse = np.float32(1.0) / temperature
        k, top_p, min_p = int(made["top_k"][row]), float(made["top_p"][row]), float(made["min_p"][row])
        k = k if 0 < k < vocab else vocab
        if k < vocab or top_p < 1.0 or min_p > 0.0:
            scaled = x * inverse
            d = (scaled - scaled.max()).astype(np.float64)
            rank = np.argsort(-d, kind="stable")[:k]
        else:
            top = np.float64(x.max() * inverse)
            d = (x.astype(np.float64) * np.float64(inverse) - top).astype(np.float32).astype(np.float64)
            rank = np.arange(vocab)
        weights = np.exp(d[rank])
        rank, weights = rank[weights >= min_p], weights[weights >= min_p]
        sums = np.cumsum(weights)
        if top_p < 1.0:
            sums = sums[:int(np.searchsorted(sums, sums[-1] * top_p, side="left")) + 1]
        target = float(made["uniform"][row]) * sums[-1]
        out[row] = rank[min(int(np.searchsorted(sums, target, side="right")), len(sums) - 1)]
    return out
