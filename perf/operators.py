"""What lies between a model's logits over a byte-pair vocabulary and its tokens, as measured work.

Kinds of case (`case["op"]`):

- ``masks``: a grammar, given as an automaton over bytes, becomes one bit per (state, token).
- ``step``: one decoding step of a batch under a grammar: the states move by the drawn tokens, and the
  rows of bits of the new states are made.
- ``adjust``: penalties for repeated tokens, biases and masks on logits, as a serving step calls it.
- ``adjust_grad``: the same with its gradients, as training under the same constraints calls it.
- ``draw``: temperature, top-k, top-p and min-p, and one token a row by a given uniform number.
- ``logprobs`` / ``logprobs_grad``: log-probabilities of given tokens, without and with their gradient.

Where ``own`` is false ``run`` computes them by elementary torch operations; where it is true it calls the
framework.
"""
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_MOST_BYTES = 16  # the longest token of the vocabularies made here


# ---- the cases ---------------------------------------------------------------------------------


def listed():
    return [
        # a small grammar compiled for the vocabulary that the command line trains (300 tokens)
        {"name": "masks_64x300", "op": "masks", "states": 64, "vocab": 300},
        # a grammar of a record format, for the vocabulary of the 1 GiB corpus
        {"name": "masks_600x32000", "op": "masks", "states": 600, "vocab": 32000},
        # a large schema, for the largest vocabulary there is
        {"name": "masks_2048x65535", "op": "masks", "states": 2048, "vocab": 65535},
        # one sequence, and a batch, decoding under a grammar
        {"name": "step_1x32000", "op": "step", "rows": 1, "states": 600, "vocab": 32000},
        {"name": "step_256x32000", "op": "step", "rows": 256, "states": 600, "vocab": 32000},
        # one sequence's logits, short history
        {"name": "adjust_1x4096", "op": "adjust", "rows": 1, "vocab": 4096, "type": "f32", "history": 65, "biases": 4},
        # a serving batch with everything on, histories up to 2000 tokens
        {"name": "adjust_256x32000", "op": "adjust", "rows": 256, "vocab": 32000, "type": "bf16", "history": 2000, "biases": 32},
        # training under the constraints that the answers were drawn with
        {"name": "adjust_grad_4096x32000", "op": "adjust_grad", "rows": 4096, "vocab": 32000, "type": "bf16", "history": 500,
         "biases": 8},
        # one answer at a time
        {"name": "draw_1x32000", "op": "draw", "rows": 1, "vocab": 32000, "type": "f32", "filter": "all"},
        # a large batch over the largest vocabulary: half the rows drawn freely, half with the filters of a chat service
        {"name": "draw_1000x65535", "op": "draw", "rows": 1000, "vocab": 65535, "type": "f32", "filter": "mixed"},
        # scoring a few sentences
        {"name": "logprobs_33x4096", "op": "logprobs", "rows": 33, "vocab": 4096, "type": "f16"},
        # the loss of a training step and its gradient
        {"name": "logprobs_grad_8192x32000", "op": "logprobs_grad", "rows": 8192, "vocab": 32000, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["masks", "step", "adjust", "adjust_grad", "draw", "logprobs", "logprobs_grad"])
    vocab = min(65535, _log(rng, 257, 65535) | rng.randrange(2))
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "masks":
        return {"op": op, "states": _log(rng, 1, 2048), "vocab": vocab}
    if op == "step":
        return {"op": op, "rows": _log(rng, 1, 512), "states": _log(rng, 2, 2048), "vocab": vocab}
    most = {"adjust": 512 * 32000, "adjust_grad": 4096 * 32000, "draw": 1000 * 65535, "logprobs": 8192 * 32000,
            "logprobs_grad": 8192 * 32000}[op] // vocab
    if kind == "f32":
        most //= 2
    rows = _log(rng, 1, max(2, min(most, 16384)))
    case = {"op": op, "rows": rows, "vocab": vocab, "type": kind}
    if op == "draw":
        case["filter"] = rng.choice(["none", "all", "mixed"])
    if op in ("adjust", "adjust_grad"):
        case["history"] = _log(rng, 1, 4000)
        case["biases"] = rng.randrange(0, 65)
    return case


# ---- inputs ------------------------------------------------------------------------------------


def _vocabulary(vocab, rng):
    """A merge table like a trained one, level by level, frequent tokens more often, at most 16 bytes a token; and each token's
    bytes (zero behind its end) and length. The last id has no bytes: it ends an answer."""
    text = np.frombuffer(b" etaoinshrdlucmfwypvbgk.,0123456789\"{}[]:ETAOINSHRDLU-_/\n", dtype=np.uint8)
    n = vocab - 257
    first, second = np.zeros(n, np.int64), np.zeros(n, np.int64)
    length = np.ones(vocab, np.int64)
    length[-1] = 0
    data = np.zeros((vocab, _MOST_BYTES), np.uint8)
    data[:256, 0] = np.arange(256)
    place = np.arange(_MOST_BYTES)
    at = 0
    for part in (0.05, 0.15, 0.3, 0.5, 0.75, 1.0):
        end = max(at, int(round(n * part)))
        m = end - at
        for side in (first, second):
            byte = np.where(rng.random(m) < 0.97, text[(len(text) * rng.random(m) ** 2).astype(np.int64)], rng.integers(0, 256, m))
            token = 256 + (at * rng.random(m) ** 1.5).astype(np.int64)
            side[at:end] = np.where((at > 0) & (rng.random(m) < 0.7), token, byte)
        long = length[first[at:end]] + length[second[at:end]] > _MOST_BYTES
        for side in (first, second):
            side[at:end] = np.where(long, text[rng.integers(0, len(text), m)], side[at:end])
        a, b = first[at:end], second[at:end]
        length[256 + at:256 + end] = length[a] + length[b]
        behind = place - length[a][:, None]
        data[256 + at:256 + end] = np.where(behind < 0, data[a], data[b[:, None], np.clip(behind, 0, _MOST_BYTES - 1)])
        at = end
    data[place >= length[:, None]] = 0
    return np.stack([first, second, np.arange(256, vocab - 1)], 1).astype(np.uint16), length, data


def _automaton(states, rng):
    """States of three sorts, as grammars of records have: inside a string (nearly every byte, mostly back to itself), inside a
    number, and structure (a few bytes)."""
    table = np.full((states, 256), -1, np.int64)
    sort = rng.random(states)
    to = lambda *shape: rng.integers(0, states, shape)  # noqa: E731
    printable = np.arange(32, 127)
    for s in np.nonzero(sort < 0.25)[0]:
        table[s, printable] = s
        table[s, 128:] = s
        table[s, [34, 92]] = to(2)
    for s in np.nonzero((sort >= 0.25) & (sort < 0.45))[0]:
        table[s, 48:58] = s
        table[s, [44, 46, 93, 125]] = to(4)
    for s in np.nonzero(sort >= 0.45)[0]:
        table[s, rng.choice(printable, 3)] = to(3)
        table[s, 32] = s
    accepting = rng.random(states) < 0.1
    return table.astype(np.int32), accepting


def _decoding(rows, table, length, data, rng):
    """The batch's states and the tokens that were drawn in them: allowed ones, the end of the answer in some rows; and some rows
    that are no longer in use (state -1)."""
    states = rng.integers(0, len(table), rows)
    tried = (len(length) * rng.random((rows, 64)) ** 3).astype(np.int64)
    at = np.broadcast_to(states[:, None], tried.shape)
    for j in range(_MOST_BYTES):
        moved = np.where(at < 0, -1, table[at, data[tried, j]])
        at = np.where(j < length[tried], moved, at)
    fits = (at >= 0) & (length[tried] > 0)
    one_byte = np.argmax((table[states] >= 0) * rng.random((rows, 256)), 1)
    tokens = np.where(fits.any(1), tried[np.arange(rows), np.argmax(fits, 1)], one_byte)
    idle = rng.random(rows)
    tokens = np.where((idle > 0.95) & (rows > 1), len(length) - 1, tokens)
    states = np.where((idle < 0.05) & (rows > 1), -1, states)
    return states.astype(np.int32), tokens.astype(np.int32)


def _logits(g, rows, vocab, kind):
    """A model's logits: a bulk of unlikely tokens, and a tail of likely ones."""
    z = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.0)
    z.add_(torch.rand(rows, vocab, generator=g, device="cuda").pow_(300).mul_(14.0)).sub_(3.0)
    return z.to(_TYPES[kind])


def _words(vocab):
    return (vocab + 31) // 32


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    vocab, op = case["vocab"], case["op"]
    s = {"case": case}
    if op in ("masks", "step"):
        merges, length, data = _vocabulary(vocab, rng)
        table, accepting = _automaton(case["states"], rng)
        s["merges"] = merges  # the trained table, on the host as the tokenizer has it
        s["bytes"] = torch.from_numpy(data).cuda()
        s["length"] = torch.from_numpy(length).cuda()
        s["next"] = torch.from_numpy(table).cuda()
        s["accepting"] = torch.from_numpy(accepting).cuda()
        s["end"] = vocab - 1
        if op == "step":
            states, tokens = _decoding(case["rows"], table, length, data, rng)
            s["states"] = torch.from_numpy(states).cuda()
            s["tokens"] = torch.from_numpy(tokens).cuda()
        if own:  # a program lays its vocabulary out once, for all its grammars
            s["vocabulary"] = _framework().Vocabulary(merges, vocab_size=vocab, end_token=vocab - 1)
        return s
    rows, kind = case["rows"], case["type"]
    s["logits"] = _logits(g, rows, vocab, kind)
    if op == "draw":
        many = case["filter"] != "none"
        some = torch.rand(rows, generator=g, device="cuda") < (1.0 if case["filter"] == "all" else 0.5)
        on = some & many
        s["uniforms"] = torch.rand(rows, generator=g, device="cuda")
        s["temperature"] = 0.6 + 0.6 * torch.rand(rows, generator=g, device="cuda")
        k = torch.randint(1, 200, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["top_k"] = torch.where(on, k, torch.zeros_like(k))
        p = 0.8 + 0.19 * torch.rand(rows, generator=g, device="cuda")
        s["top_p"] = torch.where(on, p, torch.ones_like(p))
        s["min_p"] = torch.where(on, torch.full_like(p, 0.01), torch.zeros_like(p))
        return s
    if op in ("logprobs", "logprobs_grad"):
        s["tokens"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        s["tokens"][torch.rand(rows, generator=g, device="cuda") < 0.05] = -1  # padding: not scored
        s["grad"] = torch.randn(rows, generator=g, device="cuda") / rows
        s["logits"].requires_grad_(op == "logprobs_grad")
        return s
    hist, nb = case["history"], case["biases"]
    s["history"] = (vocab * torch.rand(rows, hist, generator=g, device="cuda", dtype=torch.float64).pow_(2)).to(torch.int32)
    s["lengths"] = torch.randint(0, hist + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    s["prompt_lengths"] = (s["lengths"] * torch.rand(rows, generator=g, device="cuda")).to(torch.int32)
    s["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=g, device="cuda")
    s["presence"] = torch.rand(rows, generator=g, device="cuda")
    s["frequency"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
    s["bias"] = torch.randn(vocab, generator=g, device="cuda") * 0.1
    s["bias_tokens"] = torch.randint(0, vocab, (rows, nb), generator=g, device="cuda", dtype=torch.int32)
    s["bias_values"] = torch.randn(rows, nb, generator=g, device="cuda")
    states = 64
    open_ = torch.randint(-(2 ** 31), 2 ** 31, (states, _words(vocab)), generator=g, device="cuda")
    s["masks"] = (open_ | torch.randint(-(2 ** 31), 2 ** 31, open_.shape, generator=g, device="cuda")).to(torch.int32)
    s["states"] = torch.randint(0, states, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if op == "adjust_grad":
        s["grad"] = torch.randn(rows, vocab, generator=g, device="cuda").to(_TYPES[kind])
        for name in ("logits", "bias", "bias_values"):
            s[name].requires_grad_(True)
    return s


# ---- one pass ----------------------------------------------------------------------------------


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zig-bpe_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import zbpe

    return zbpe


def _history(s):
    return {k: s[k] for k in ("history", "lengths", "prompt_lengths", "repetition", "presence", "frequency", "bias", "bias_tokens",
                              "bias_values", "masks", "states")}


def _run_own(s):
    zbpe, op = _framework(), s["case"]["op"]
    if op == "masks":
        return zbpe.Grammar(s["vocabulary"], s["next"], s["accepting"]).masks()
    if op == "step":
        grammar = zbpe.Grammar(s["vocabulary"], s["next"], s["accepting"])
        states = grammar.advance(s["states"], s["tokens"])
        return states, grammar.masks(states)
    if op == "adjust":
        return zbpe.adjust_logits(s["logits"], **_history(s))
    if op == "adjust_grad":
        out = zbpe.adjust_logits(s["logits"], **_history(s))
        return (out.detach(), *torch.autograd.grad(out, [s["logits"], s["bias"], s["bias_values"]], s["grad"]))
    if op == "draw":
        return zbpe.draw_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                min_p=s["min_p"])
    if op == "logprobs":
        return zbpe.token_logprobs(s["logits"], s["tokens"])
    out = zbpe.token_logprobs(s["logits"], s["tokens"])
    return out.detach(), torch.autograd.grad(out, s["logits"], s["grad"])[0]


def _walk(s, states):
    """[rows, vocab]: the state after each token from each of `states`; the state past the last one is the dead one."""
    n = s["next"].shape[0]
    table = torch.full((n + 1, 256), n, dtype=torch.int32, device="cuda")
    table[:n] = torch.where((s["next"] < 0) | (s["next"] >= n), n, s["next"])
    table = table.reshape(-1)
    at = torch.where((states < 0) | (states >= n), n, states).to(torch.int32)[:, None].expand(-1, s["length"].shape[0])
    for j in range(_MOST_BYTES):
        moved = table[at.to(torch.int64) * 256 + s["bytes"][:, j]]
        at = torch.where(j < s["length"], moved, at)
    return at


def _bits(s, states):
    n = s["next"].shape[0]
    alive = _walk(s, states) != n
    inside = (states >= 0) & (states < n)
    alive[:, s["end"]] = inside & s["accepting"][torch.where(inside, states, 0).to(torch.int64)]
    rows, vocab = alive.shape
    words = _words(vocab)
    padded = torch.zeros(rows, words * 32, dtype=torch.bool, device="cuda")
    padded[:, :vocab] = alive
    weights = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
    packed = (padded.view(rows, words, 32) * weights).sum(2)
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)


def _advanced(s):
    n = s["next"].shape[0]
    states, tokens = s["states"], s["tokens"].to(torch.int64)
    inside = (states >= 0) & (states < n)
    at = torch.where(inside, states, 0).to(torch.int64)
    ended = torch.where(s["accepting"][at], at, -1)
    for j in range(_MOST_BYTES):
        moved = s["next"][torch.where(at < 0, 0, at), s["bytes"][tokens, j].to(torch.int64)].to(torch.int64)
        at = torch.where((j < s["length"][tokens]) & (at >= 0), moved, at)
    at = torch.where(tokens == s["end"], ended, at)
    return torch.where(inside, at, -1).to(torch.int32)


def _adjusted(s):
    """What the penalties, biases and masks make of the logits, in 32 bits; also the factor of each logit and what the masks allow."""
    rows, vocab = s["logits"].shape
    z = s["logits"].detach().float()
    place = torch.arange(s["history"].shape[1], device="cuda")
    ids = s["history"].to(torch.int64)
    used = place < s["lengths"][:, None]
    seen = torch.zeros(rows, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, ids, used.to(torch.int32))
    count = torch.zeros(rows, vocab, dtype=torch.int32, device="cuda").scatter_add_(
        1, ids, (used & (place >= s["prompt_lengths"][:, None])).to(torch.int32))
    theta = s["repetition"][:, None]
    factor = torch.where(seen > 0, torch.where(z > 0, 1 / theta, theta), 1.0)
    z = torch.where(seen > 0, torch.where(z > 0, z / theta, z * theta), z)
    z = z - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    z = z + s["bias"].detach()
    z = z + torch.zeros(rows, vocab, device="cuda").scatter_add_(1, s["bias_tokens"].to(torch.int64), s["bias_values"].detach())
    v = torch.arange(vocab, device="cuda")
    allowed = (s["masks"][s["states"].to(torch.int64)][:, v >> 5] >> (v & 31)) & 1 != 0
    return torch.where(allowed, z, -torch.inf).to(s["logits"].dtype), factor, allowed


def _adjusted_grad(s):
    out, factor, allowed = _adjusted(s)
    g = torch.where(allowed, s["grad"].float(), 0.0)
    return (out, (g * factor).to(s["logits"].dtype), g.sum(0), g.gather(1, s["bias_tokens"].to(torch.int64)))


def _drawn(s):
    """In 64 bits: a token is drawn by where sums end."""
    z = s["logits"].double()
    z = torch.where(torch.isnan(z), -torch.inf, z)
    rows, vocab = z.shape
    top = z.amax(1, keepdim=True)
    w = torch.exp((z - top) / s["temperature"].double()[:, None])
    _, order = torch.sort(z, dim=1, descending=True, stable=True)
    sorted_w = w.gather(1, order)
    rank = torch.arange(vocab, device="cuda")
    k = s["top_k"][:, None]
    kept = (rank < k) | (k <= 0)
    sorted_w = torch.where(kept, sorted_w, 0.0)
    before = torch.cumsum(sorted_w, 1) - sorted_w
    p = s["top_p"].double()[:, None]
    kept &= (before < p * sorted_w.sum(1, keepdim=True)) | (p >= 1)
    kept &= sorted_w >= s["min_p"].double()[:, None]
    weights = torch.zeros_like(w).scatter_(1, order, torch.where(kept, sorted_w, 0.0))
    ends = torch.cumsum(weights, 1)
    total = ends[:, -1:]
    token = (ends <= s["uniforms"].double()[:, None] * total).sum(1, keepdim=True).clamp_(max=vocab - 1)
    logprob = torch.log(weights.gather(1, token) / total)
    return token[:, 0].to(torch.int32), logprob[:, 0].float()


def _scored(s, grad):
    z = s["logits"].detach().float()
    scored = s["tokens"] >= 0
    token = torch.where(scored, s["tokens"], 0)[:, None]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    logprob = torch.where(scored, (z.gather(1, token) - top - torch.log(total))[:, 0], 0.0)
    if not grad:
        return logprob
    g = torch.where(scored, s["grad"], 0.0)[:, None]
    d = (e / total).mul_(-g)
    d.scatter_add_(1, token, g)
    return logprob, d.to(s["logits"].dtype)


@torch.no_grad()
def _run_plain(s):
    op = s["case"]["op"]
    if op == "masks":
        return _bits(s, torch.arange(s["next"].shape[0], device="cuda"))
    if op == "step":
        states = _advanced(s)
        return states, _bits(s, states)
    if op == "adjust":
        return _adjusted(s)[0]
    if op == "adjust_grad":
        return _adjusted_grad(s)
    if op == "draw":
        return _drawn(s)
    return _scored(s, op == "logprobs_grad")


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    vocab, op = case["vocab"], case["op"]
    words = _words(vocab)
    if op in ("masks", "step"):
        rows = case.get("rows", case["states"])
        # each state's row of the automaton, the tokens' bytes (about 6 a token), the bits; a lookup for each state and token
        return {"bytes": 1024 * min(rows, case["states"]) + 6 * vocab + 4 * rows * words, "flops": rows * vocab}
    rows, e = case["rows"], _SIZE[case["type"]]
    n = rows * vocab
    if op == "draw":
        return {"bytes": n * e + 28 * rows, "flops": 4 * n}
    if op == "logprobs":
        return {"bytes": n * e + 12 * rows, "flops": 4 * n}
    if op == "logprobs_grad":
        return {"bytes": 2 * n * e + 16 * rows, "flops": 8 * n}
    inputs = 4 * vocab + 4 * 64 * words + rows * (4 * case["history"] + 8 * case["biases"] + 24)
    if op == "adjust":
        return {"bytes": 2 * n * e + inputs, "flops": 2 * n}
    return {"bytes": 4 * n * e + inputs + 4 * vocab + 4 * rows * case["biases"], "flops": 4 * n}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------


def _exact_tokens(s):
    """[vocab, states + 1]: the state after each token, composed along the merges: a token moves as its halves do, one after
    the other. The last state is the dead one."""
    table = s["next"].cpu().numpy().astype(np.int64)
    n = len(table)
    table = np.where((table < 0) | (table >= n), n, table)
    after = np.empty((s["case"]["vocab"], n + 1), np.int32)
    after[:256, :n] = table.T
    after[:256, n] = n
    after[-1] = n
    for a, b, c in s["merges"].tolist():
        after[c] = after[b][after[a]]
    return after


def _exact_masks(s, states, after):
    n = after.shape[1] - 1
    accepting = np.append(s["accepting"].cpu().numpy(), False)
    rows = np.where((states < 0) | (states >= n), n, states)
    out = np.zeros((len(rows), _words(len(after))), np.int32)
    for i, r in enumerate(rows):
        alive = after[:, r] != n
        alive[s["end"]] = accepting[r]
        bits = np.zeros(out.shape[1] * 32, bool)
        bits[:len(alive)] = alive
        out[i] = np.packbits(bits, bitorder="little").view(np.int32)
    return out


def _exact_adjust(s, grad):
    host = {k: v.detach().cpu() for k, v in s.items() if isinstance(v, torch.Tensor)}
    z = host["logits"].double().numpy()
    rows, vocab = z.shape
    h = {k: host[k].numpy() for k in ("history", "lengths", "prompt_lengths", "bias_tokens", "masks", "states")}
    f = {k: host[k].double().numpy() for k in ("repetition", "presence", "frequency", "bias", "bias_values")}
    out = np.empty_like(z)
    dz, db, dv = np.empty_like(z) if grad else None, np.zeros(vocab), np.zeros(h["bias_tokens"].shape)
    up = host["grad"].double().numpy() if grad else None
    for r in range(rows):
        ids = h["history"][r, :h["lengths"][r]]
        theta = f["repetition"][r]
        y, slope = z[r].copy(), np.ones(vocab)
        old = np.unique(ids)
        slope[old] = np.where(z[r, old] > 0, 1 / theta, theta)
        y[old] *= slope[old]
        new, count = np.unique(ids[h["prompt_lengths"][r]:], return_counts=True)
        y[new] -= f["frequency"][r] * count + f["presence"][r]
        y += f["bias"]
        np.add.at(y, h["bias_tokens"][r], f["bias_values"][r])
        allowed = np.unpackbits(h["masks"][h["states"][r]].view(np.uint8), bitorder="little")[:vocab] != 0
        out[r] = np.where(allowed, y, -np.inf)
        if grad:
            u = up[r] * allowed
            dz[r] = u * slope
            db += u
            dv[r] = u[h["bias_tokens"][r]]
    return (out, dz, db, dv) if grad else out


def _exact_draw(s):
    z = s["logits"].double().cpu().numpy()
    get = {k: s[k].double().cpu().numpy() for k in ("uniforms", "temperature", "top_k", "top_p", "min_p")}
    rows, vocab = z.shape
    token, logprob = np.zeros(rows, np.int32), np.zeros(rows)
    for r in range(rows):
        w = np.exp((z[r] - z[r].max()) / get["temperature"][r])
        k = int(get["top_k"][r])
        if k > 0 or get["top_p"][r] < 1 or get["min_p"][r] > 0:
            order = np.argsort(-z[r], kind="stable")[:k if k > 0 else vocab]
            sums = np.concatenate([[0.0], np.cumsum(w[order])])
            kept = sums[:-1] < get["top_p"][r] * sums[-1] if get["top_p"][r] < 1 else np.ones(len(order), bool)
            kept = order[kept & (w[order] >= get["min_p"][r])]
            ids = np.sort(kept)
        else:
            ids = np.arange(vocab)
        ends = np.cumsum(w[ids])
        at = min(int(np.searchsorted(ends, get["uniforms"][r] * ends[-1], side="right")), len(ids) - 1)
        token[r], logprob[r] = ids[at], np.log(w[ids[at]] / ends[-1])
    return token, logprob


def _exact_logprobs(s, grad):
    """Rows in pieces, by 64-bit logarithms of sums."""
    z, tokens = s["logits"].detach(), s["tokens"]
    logprob, parts = [], []
    for at in range(0, z.shape[0], 512):
        x, t = z[at:at + 512].double(), tokens[at:at + 512]
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        one = torch.zeros_like(lp)
        rows = torch.nonzero(t >= 0)[:, 0]
        one[rows, t[rows]] = 1.0
        logprob.append(torch.where(t >= 0, torch.where(one > 0, lp, 0.0).sum(1), 0.0))
        if grad:
            parts.append((one - lp.exp()) * torch.where(t >= 0, s["grad"][at:at + 512].double(), 0.0)[:, None])
    return (torch.cat(logprob), torch.cat(parts)) if grad else torch.cat(logprob)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op in ("masks", "step"):
        after = _exact_tokens(s)
        if op == "masks":
            return _exact_masks(s, np.arange(case["states"]), after)
        states, tokens = s["states"].cpu().numpy(), s["tokens"].cpu().numpy()
        n = case["states"]
        accepting = s["accepting"].cpu().numpy()
        moved = np.array([n if a < 0 else (a if accepting[a] else n) if t == s["end"] else after[t, a] for a, t in zip(states, tokens)])
        moved = np.where(moved == n, -1, moved).astype(np.int32)
        return moved, _exact_masks(s, moved, after)
    if op in ("adjust", "adjust_grad"):
        return _exact_adjust(s, op == "adjust_grad") if case["rows"] * (case["vocab"] + 8 * case["history"]) < 2 ** 28 else None
    if op == "draw":
        return _exact_draw(s) if case["rows"] * case["vocab"] <= 2 ** 26 else None
    return _exact_logprobs(s, op == "logprobs_grad")
