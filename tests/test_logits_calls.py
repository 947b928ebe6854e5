"""Calls of the operators between a model's logits and its tokens that their definitions allow, or refuse, at the edges:
tensors written in place, forward-mode derivatives, memory that overlaps, numbers, temperatures, devices, messages.

Tolerances count roundings as test_logits.py does: u = 2^-24 for each 32-bit operation.
"""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import zbpe
from test_logits import INF, U, adjust_case, check_draw, close, cuda, gpu, half_step, some_automaton, some_merges, to_gpu


# ---- tensors that are written in place -----------------------------------------------------------------------------------------


def test_out_with_a_gradient_is_refused():
    z = torch.zeros(2, 300)
    out = torch.zeros(2, 300, requires_grad=True)
    with pytest.raises(zbpe.InvalidArgument, match="out goes without gradients"):
        zbpe.adjust_logits(z, out=out)


@gpu
def test_writing_out_is_seen_by_earlier_operations():
    """what an operation saved for its backward pass is overwritten through `out`: the backward pass raises, as for torch's own
    operations in place"""
    z, x = adjust_case(4, 300, 1)
    z, g = z.cuda(), to_gpu(x)
    rng = np.random.default_rng(0)
    merges = np.array(some_merges(300, rng, np.arange(97, 103)))
    grammar = zbpe.Grammar(zbpe.Vocabulary(merges, 300), cuda(some_automaton(5, rng, np.arange(97, 103))[0]))
    states = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    buffer = grammar.masks(states)
    zg = z.clone().requires_grad_()
    # one buffer of masks, made anew at the next step
    y = zbpe.adjust_logits(zg, masks=buffer)
    grammar.masks(states, out=buffer)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, zg, torch.ones_like(y))
    # logits that were scored, adjusted in place
    work = zg * 1.0
    lp = zbpe.token_logprobs(work, torch.tensor([1, 2, 3, 4], device="cuda"))
    with torch.no_grad():
        zbpe.adjust_logits(work, **g, out=work)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(lp, zg, torch.ones_like(lp))
    # the same through a view, and by torch's own operation that saved it
    work = (zg * 1.0).view(2, 2, 300)
    y = work.exp().sum() + (work * work).sum()
    with torch.no_grad():
        zbpe.adjust_logits(work[:1], bias=g["bias"], out=work[:1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, zg)


@gpu
def test_out_without_anything_saved():
    """an `out` that learns may be written under no_grad, any may in inference mode, where tensors have no versions"""
    z, x = adjust_case(4, 300, 1)
    z, g = z.cuda(), to_gpu(x)
    want = zbpe.adjust_logits(z, **g)
    leaf = torch.zeros(4, 300, device="cuda", requires_grad=True)
    with torch.no_grad():
        assert zbpe.adjust_logits(z, **g, out=leaf) is leaf
    assert torch.equal(leaf.detach(), want)
    with pytest.raises(zbpe.InvalidArgument, match="out goes without gradients"):
        zbpe.adjust_logits(z, **g, out=leaf)
    with torch.inference_mode():
        fresh = torch.zeros(4, 300, device="cuda")
        assert torch.equal(zbpe.adjust_logits(z, **g, out=fresh), want)
        ours = torch.zeros_like(want)
        zbpe.adjust_logits(ours, bias=g["bias"], out=ours)
    before = z._version
    zbpe.adjust_logits(z, **g)  # (what is only read keeps its version)
    assert z._version == before


# ---- forward-mode derivatives --------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_is_refused(device):
    """a tangent that no operator here carries is not dropped: the call raises, whatever requires_grad and no_grad say"""
    z, x = adjust_case(4, 300, 1)
    z, x = z.to(device), {k: v.to(device) for k, v in x.items()}
    t = torch.ones(4, device=device)
    tokens = torch.zeros(4, dtype=torch.int64, device=device)
    with forward_ad.dual_level():
        dual = lambda a: forward_ad.make_dual(a, torch.ones_like(a))  # noqa: E731
        calls = [lambda: zbpe.adjust_logits(dual(z), **x), lambda: zbpe.adjust_logits(dual(z)[:, 1:], bias=x["bias"][1:]),
                 lambda: zbpe.token_logprobs(dual(z), tokens), lambda: zbpe.token_logprobs(z, tokens, temperature=dual(t)),
                 lambda: zbpe.adjust_logits(dual(z), out=torch.empty_like(z)), lambda: zbpe.adjust_logits(z, out=dual(torch.empty_like(z)))]
        for name in ("bias", "bias_values", "repetition", "presence", "frequency"):
            calls.append(lambda name=name: zbpe.adjust_logits(z, **{**x, name: dual(x[name])}))
        for call in calls:
            with pytest.raises(zbpe.InvalidArgument, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(zbpe.InvalidArgument, match="tangent"):
                call()
        if device == "cpu":
            return
        # nothing is dropped where nothing is differentiated: inference mode, logits that are cut off, the draw
        want = zbpe.token_logprobs(z, tokens)
        assert torch.equal(zbpe.token_logprobs(dual(z).detach(), tokens), want)
        d = dual(z)
        with torch.inference_mode():
            assert torch.equal(zbpe.token_logprobs(d, tokens), want)
        zbpe.draw_tokens(dual(z), torch.zeros(4, device=device))


# ---- memory that overlaps ------------------------------------------------------------------------------------------------------


def bytes_of(data, outer, inner, rows, per, cols, element):
    """the addresses of a matrix's elements, by zbpe_rows' rule"""
    r = np.arange(rows)
    starts = data + ((r // per) * outer + (r % per) * inner) * element
    return set((starts[:, None] + np.arange(cols * element)).reshape(-1).tolist()) if rows else set()


def test_memory_that_is_written_against_all_that_is_read():
    """Matrices and arrays at random places of a small memory: a gradient that shares a byte with anything that the call reads is
    refused for that, any other one reaches the check behind it (of the workspace, which is missing here: nothing is launched)."""
    from zbpe import logits as ops

    L, rng = ops._library(), np.random.default_rng(0)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        rows, per, cols = int(rng.integers(1, 9)), int(rng.integers(1, 5)), int(rng.integers(1, 12))
        kind = int(rng.integers(0, 3))
        element = 4 if kind == 0 else 2
        inside = lambda: int(rng.integers(0, 500) // 8 * 8) + 4096  # noqa: E731

        def matrix(n, size, apart):
            inner = int(rng.choice([n, n + rng.integers(0, 20), 2 * n, 0 if not apart else n]))
            outer = int(rng.choice([inner * per, max(inner * (per - 1) + n, 0) + rng.integers(0, 20)]))
            if rng.random() < 0.3:  # rows of different outer steps between each other
                outer, inner = int(n + rng.integers(0, 6)), int((n + 6) * ((rows + per - 1) // per) + rng.integers(0, 6))
            if rng.random() < 0.1:
                return inside() + 600, -outer, -inner
            return inside(), outer, inner

        if rng.random() < 0.5:  # the same strides for all, at different places
            strides = matrix(cols, element, True)[1:]
            places = [(inside(), *strides) for _ in range(3)]
        else:
            places = [matrix(cols, element, i == 0) for i in range(3)]
        wide_up = rng.random() < 0.3
        hist = matrix(5, 4, False) if rng.random() < 0.5 else None
        arrays = {}
        for name, n in (("lengths", 4 * rows), ("prompt", 4 * rows), ("theta", 4 * rows), ("presence", 4 * rows), ("frequency", 4 * rows),
                        ("bias", 4 * cols), ("tokens", 8 * rows), ("values", 8 * rows), ("masks", 4 * 6), ("states", 4 * rows)):
            if rng.random() < 0.15:
                arrays[name] = (inside(), n)
        if ("tokens" in arrays) != ("values" in arrays):
            arrays.pop("tokens", None), arrays.pop("values", None)
        if "masks" not in arrays:
            arrays.pop("states", None)
        elif "states" not in arrays:
            arrays.pop("masks")
        place = lambda name: arrays.get(name, (0, 0))[0]  # noqa: E731
        (gp, go, gi), (zp, zo, zi), (up, uo, ui) = places
        args = ops._ADJUST.pack(
            ops._ADJUST.size, cols, rows, per, zp, zo, zi, kind, up, uo, ui, 0 if wide_up else kind,
            *((hist[0], hist[1], hist[2], 3) if hist else (0, 0, 0, 0)), 5 if hist else 0, place("lengths"), place("prompt"), place("theta"),
            place("presence"), place("frequency"), place("bias"), place("tokens"), place("values"), 2 if "tokens" in arrays else 0, 1,
            place("masks"), 6 if "masks" in arrays else 0, place("states"))
        status = L.zbpe_adjust_logits_grad(0, None, args, ops._MATRIX.pack(gp, go, gi, kind), 64, 0, 64, 0)
        message = L.zbpe_last_error(None).decode()
        assert status == 5
        if "the rows of grad_logits overlap" in message:
            continue
        read = bytes_of(zp, zo, zi, rows, per, cols, element) | bytes_of(up, uo, ui, rows, per, cols, 4 if wide_up else element)
        if hist:
            read |= bytes_of(*hist, rows, per, 5, 4)
        for at, n in arrays.values():
            read |= set(range(at, at + n))
        overlap = bool(bytes_of(gp, go, gi, rows, per, cols, element) & read)
        assert ("grad_logits overlaps" in message) == overlap and ("workspace of 0 bytes" in message) != overlap, (message, args)
        seen[overlap] += 1
    assert min(seen.values()) > 500


def test_masks_and_states_that_overlap_what_is_read():
    from zbpe import logits as ops

    L = ops._library()
    grammar = ops._GRAMMAR.pack(1 << 20, 1 << 21, 300, -1, 1 << 22, 1 << 23, 5, 1 << 24)  # (words: 10)
    for states, out, words in ((4096, 4096, "states"), (4096 + 196, 4096, "states"), (4096, 4096 + 8, "states"),
                               (4096, (1 << 22) + 5000, "automaton"), (4096, (1 << 22) - 196, "automaton"), (4096, (1 << 23) - 8, "automaton"),
                               (4096, (1 << 24) + 300 * 32, "index")):
        assert L.zbpe_grammar_masks(0, None, grammar, states, 5, out) == 5
        assert "masks overlaps" in L.zbpe_last_error(None).decode() and words in L.zbpe_last_error(None).decode()
    for states, tokens, out, words in ((4096, 8192, 4100, "states"), (4096, 8192, 8188, "tokens"), (4096, 8192, 1 << 22, "automaton")):
        assert L.zbpe_grammar_advance(0, None, grammar, states, tokens, 5, out) == 5
        assert "out overlaps" in L.zbpe_last_error(None).decode() and words in L.zbpe_last_error(None).decode()


def test_out_that_overlaps_in_part():
    """the forward call, and the scores' gradient, by the same rule"""
    from zbpe import logits as ops

    L = ops._library()
    none = (0, 0, 0, 0)

    def adjust(z, out, rows=4, inner=4, history=none, n=0, bias=0):
        return L.zbpe_adjust_logits(0, None, ops._ADJUST.pack(ops._ADJUST.size, 300, rows, inner, *z, *out, *history, n, 0, 0, 0, 0, 0, bias, 0, 0, 0, 0, 0, 0, 0))

    base = 1 << 20
    for z, out, kw, words in (((base, 0, 300, 0), (base + 4, 0, 300, 0), {}, "the logits"),         # one column on
                              ((base, 0, 300, 0), (base + 1200, 0, 300, 0), {}, "the logits"),      # one row on
                              ((base, 0, 300, 1), (base, 0, 300, 0), {}, "the logits"),             # 32 bits over 16
                              ((base, 0, 600, 0), (base + 1196, 0, 600, 0), {}, "the logits"),      # beside each other but for one
                              ((base, 0, 300, 0), (base, 0, 301, 0), {}, "the logits"),             # other strides
                              ((base, 0, 0, 0), (base - 1200, 0, 300, 0), {}, "the logits"),        # a broadcast row among them
                              ((base, 0, 300, 0), (2 * base, 0, 300, 0), {"history": (2 * base + 4796, 0, 50, 3), "n": 50}, "history"),
                              ((base, 0, 300, 0), (2 * base, 0, 300, 0), {"bias": 2 * base - 1196}, "bias"),
                              ((base, 0, 300, 0), (base, 0, 300, 0), {"bias": base + 2400}, "bias")):
        assert adjust(z, out, **kw) == 5
        assert f"out overlaps {words}" in L.zbpe_last_error(None).decode()
    for grad, words in ((base + 4, "the logits"), (2 * base - 8, "the tokens"), (3 * base, "grad"), (4 * base + 24, "stats")):
        args = ops._LOGPROBS.pack(ops._LOGPROBS.size, 300, 4, 4, base, 0, 300, 0, 2 * base, 3, 0, 0, 4 * base)
        assert L.zbpe_token_logprobs_grad(0, None, args, 3 * base, ops._MATRIX.pack(grad, 0, 300, 0)) == 5
        assert f"grad_logits overlaps {words}" in L.zbpe_last_error(None).decode()


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_out_beside_the_logits(kind):
    """what shares a buffer and no element is written as before: halves of rows, alternate rows, another dtype's rows in between;
    what shares some is refused and not touched"""
    z, x = adjust_case(12, 700, 4, kind=kind)
    g = to_gpu(x)
    want = zbpe.adjust_logits(z.cuda(), **g)
    wide = torch.full((12, 1500), 7.0, dtype=kind, device="cuda")
    halves = wide[:, 3:703], wide[:, 703:1403]
    rows = wide.view(24, 750)[:, 1:701]
    for source, out in (halves, halves[::-1], (rows[::2], rows[1::2])):
        wide.fill_(7.0)
        source.copy_(z)
        assert zbpe.adjust_logits(source, **g, out=out) is out
        assert torch.equal(out, want) and torch.equal(source, z.cuda())
        assert int((wide == 7).sum()) >= 12 * 100
    three = wide[:, 3:703].view(3, 4, 700)
    three.copy_(z.view(3, 4, 700))
    shaped = {k: v.view(3, 4, *v.shape[1:]) if k not in ("bias", "masks") else v for k, v in g.items()}
    assert torch.equal(zbpe.adjust_logits(three, **shaped, out=three).reshape(12, 700), want)  # in place, by another view
    row = wide[5:6, :700]
    row.copy_(z[:1])
    spread = torch.cat([wide[:5], wide[6:], wide[:1]])[:, :700]
    assert zbpe.adjust_logits(row.expand(12, -1), **g, out=spread) is spread
    buffer = torch.arange(13 * 700, device="cuda").view(13, 700).to(kind)
    was = buffer.clone()
    for source, out in ((buffer[:12], buffer[1:]), (buffer[1:], buffer[:12]), (buffer[:12, :-1], buffer[:12, 1:]),
                        (buffer[1:2].expand(12, -1), buffer[:12])):
        terms = {"presence": 1.0, "history": g["history"]}
        with pytest.raises(zbpe.InvalidArgument, match="out overlaps the logits"):
            zbpe.adjust_logits(source, **terms, out=out)
    bias = torch.zeros(12 * 700, device="cuda")
    with pytest.raises(zbpe.InvalidArgument, match="out overlaps bias"):
        zbpe.adjust_logits(z.float().cuda(), bias=bias[700:1400], out=bias.view(12, 700))
    masks = torch.zeros(13, 22, dtype=torch.int32, device="cuda")
    with pytest.raises(zbpe.InvalidArgument, match="out overlaps masks"):
        zbpe.adjust_logits(torch.zeros(1, 20, device="cuda"), masks=masks[:1], out=masks[:1, 1:21].view(torch.float32))
    grammar = zbpe.Grammar(zbpe.Vocabulary([], 300), torch.zeros(13 * 10, 256, dtype=torch.int32))
    states = torch.zeros(130, dtype=torch.int32, device="cuda")
    with pytest.raises(zbpe.InvalidArgument, match="masks overlaps states"):
        grammar.masks(states[:13], out=states.view(13, 10))
    torch.cuda.synchronize()
    assert torch.equal(buffer, was) and not bias.any() and not masks.any() and not states.any()


# ---- numbers that stand for all rows -------------------------------------------------------------------------------------------


@gpu
def test_numbers_for_whole_values():
    """a number for an int32 argument is whole and fits, or is refused; it is never cut off"""
    z, x = adjust_case(4, 300, 1)
    z, g, u = z.cuda(), to_gpu(x), torch.full((4,), 0.6, device="cuda")
    for bad in (0.5, 1.5, -0.5, float("nan"), INF, -INF, 2 ** 31, 2 ** 40, -2 ** 31 - 1, 1e30):
        with pytest.raises(zbpe.InvalidArgument, match="top_k"):
            zbpe.draw_tokens(z, u, top_k=bad)
        for name in ("lengths", "prompt_lengths"):
            with pytest.raises(zbpe.InvalidArgument, match=name):
                zbpe.adjust_logits(z, history=g["history"], **{name: bad})
        with pytest.raises(zbpe.InvalidArgument, match="states"):
            zbpe.adjust_logits(z, masks=g["masks"], states=bad)
    whole = zbpe.draw_tokens(z, u, top_k=torch.full((4,), 3, dtype=torch.int32, device="cuda"))
    for good in (3, 3.0):
        assert torch.equal(zbpe.draw_tokens(z, u, top_k=good)[0], whole[0])
    every = zbpe.draw_tokens(z, u)
    for good in (0, -1, 2 ** 31 - 1, -2 ** 31, False):
        assert torch.equal(zbpe.draw_tokens(z, u, top_k=good)[0], every[0])
    zbpe.draw_tokens(z, u, temperature=1, top_p=1e300, min_p=0.5)  # (a float argument takes any number)


# ---- temperatures of log-probabilities -----------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [300, 4099])
def test_logprobs_at_any_temperature(cols, kind):
    """From the smallest to infinite; 0, negative ones, NaN and subnormal ones count as 2^-126. Logits are eighths, so that no value
    comes near the border of what 32 bits hold; one row spans more than 32 bits can (3e38 - -3e38).

    An exponent e = d / T is off by 5 U |e|, and by what 1 / T loses where it is subnormal (half of 2^-149, twice in the scale,
    relative to 1 / T); for T infinite it is |d| 2^-148 at most in place of 0."""
    rng = np.random.default_rng(cols)
    ts = np.float32([INF, 3e38, 1e38, 1e20, 1e3, 1e-3, 1e-20, 2e-38, 2.0 ** -126, 1e-38, 1e-40, 1e-45, 0.0, -1.0, float("nan")])
    rows = 2 * len(ts)
    z = torch.from_numpy(np.round(rng.standard_normal((rows, cols)) * 16) / 8).to(kind)
    z[:, 5] = -INF
    big = torch.finfo(kind).max * 0.9
    z[:len(ts), 7], z[:len(ts), 9] = big, -big
    z[:len(ts):2, 11] = big  # ties of the largest
    tokens = torch.from_numpy(rng.choice([0, 5, 7, 9, 11, 20], rows))
    tokens[len(ts):] = torch.from_numpy(rng.integers(0, cols, len(ts)))
    tokens[len(ts) + 3] = -1
    t32 = torch.from_numpy(np.tile(ts, 2))
    up = torch.from_numpy(rng.uniform(-2, 2, rows)).float()
    zg = z.cuda().requires_grad_()
    y = zbpe.token_logprobs(zg, tokens.cuda(), temperature=t32.cuda())
    got, = torch.autograd.grad(y, zg, up.cuda())

    t = t32.double().numpy()[:, None]
    t = np.where(t >= 2.0 ** -126, t, 2.0 ** -126)
    d = z.double().numpy()
    d = d - d.max(1, keepdims=True)
    none = np.isneginf(d)
    e = np.where(none, -np.inf, np.where(none, 0, d) / t)
    w = np.exp(e)
    p = w / w.sum(1, keepdims=True)
    loss = np.where(np.isinf(t), 0.0, np.where(np.isinf(t), 0.0, t) * 2.0 ** -148)
    off = np.where(p > 0, np.where(np.isinf(t), np.abs(np.where(none, 0, d)) * 2.0 ** -148, np.abs(np.where(p > 0, e, 0)) * (5 * U + loss)), 0.0)
    mean = (p * off).sum(1)
    at = np.arange(rows), np.maximum(tokens.numpy(), 0)
    scored = tokens.numpy() >= 0
    want = np.where(scored, np.where(none[at], -np.inf, e[at] - np.log(w.sum(1))), 0.0)
    bound = np.where(scored & np.isfinite(want), U * (370 + 8 * np.abs(want)) + mean + np.abs(np.where(none[at], 0, d[at])) * 2.0 ** -148 + np.abs(
        np.where(none[at], 0, e[at])) * loss[:, 0], 0)
    with np.errstate(over="ignore"):
        narrow = want.astype(np.float32).astype(np.float64)  # (past what 32 bits hold: -inf)
    close(y, np.where(np.isinf(narrow), narrow, want), bound)
    hot = np.zeros((rows, cols))
    hot[at] = 1
    g = np.where(scored, up.double().numpy() / t[:, 0], 0.0)[:, None]
    want = g * (hot - p)
    relative, least = half_step(kind)
    rough = np.abs(g) * (p * (off + mean[:, None] + 370 * U) + (4 * U + loss) * (hot + p)) + np.abs(up.double().numpy())[:, None] * 2.0 ** -147
    close(got, want, rough + (np.abs(want) + rough) * relative + least + np.abs(g) * 2.0 ** -126)
    # one number for all rows
    for number in (INF, 0.0, 0):
        a = zbpe.token_logprobs(z.cuda(), tokens.cuda(), temperature=number)
        b = zbpe.token_logprobs(z.cuda(), tokens.cuda(), temperature=torch.full((rows,), float(number), device="cuda"))
        assert torch.equal(a.view(torch.int32), b.view(torch.int32)) and not a.isnan().any()


@gpu
def test_logprobs_of_a_draw_at_an_infinite_temperature():
    """the log-probability that draw_tokens gives is the score of its token, masked tokens among the row"""
    z = torch.randn(6, 700, device="cuda")
    z[:, ::3] = -INF
    tokens, logprobs = zbpe.draw_tokens(z, torch.rand(6, device="cuda"), temperature=INF)
    # log of 466: 7 roundings of its sum of ones (exact), exponents within |d| 2^-148, one of logf (2 U relative), one more
    np.testing.assert_allclose(zbpe.token_logprobs(z, tokens, temperature=INF).cpu().numpy(), logprobs.cpu().numpy(), rtol=8 * U, atol=0)


@gpu
@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.3])
def test_logprobs_gradient_far_from_the_largest(temperature):
    """32-bit logits that are eighths, so that their distances are exact, down to 80 temperatures below the largest: an element of
    the gradient is off by its own few roundings there too. The exponential: 3 U (the instruction's 2, the correction's one);
    the sum: 2 U, 3 U of the mean distance from the largest (below 3 here), and 4 + 6 additions and a rescaling; g / T, g / s,
    their product and 1 / T: 5 U; together under 32 U."""
    rng = np.random.default_rng(8)
    cols = 256
    z = torch.from_numpy(np.round(-rng.random((40, cols)) * 80 * temperature * 8) / 8).float()
    z[:, 0] = 0
    t = np.float64(np.float32(temperature))
    e = z.double().numpy() / t
    p = np.exp(e) / np.exp(e).sum(1, keepdims=True)
    assert (-p * e).sum(1).max() < 3
    tokens = torch.zeros(40, dtype=torch.int64)
    zg = z.cuda().requires_grad_()
    y = zbpe.token_logprobs(zg, tokens.cuda(), temperature=temperature)
    got, = torch.autograd.grad(y, zg, torch.ones_like(y))
    want = -p / t
    got = got.double().cpu().numpy()
    worst = (np.abs(got - want) / np.abs(want))[:, 1:].max() / U
    assert worst < 32, worst


# ---- without torch -------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("blocked", [True, False])
def test_the_tokenizer_does_not_need_torch(blocked):
    """`from zbpe import *` takes the tokenizer alone, whether torch can be imported or not; the operators' names are there when
    they are asked for"""
    code = ("import sys\n" + ("sys.modules['torch'] = None\n" if blocked else "") + "from zbpe import *\nimport zbpe\n"
            "assert BasicTokenizer is zbpe.BasicTokenizer and Merges().as_array() is not None\n"
            "assert sys.modules.get('torch') is None\n"
            + ("try:\n    zbpe.draw_tokens\nexcept ImportError:\n    print('fine')\n" if blocked else
               "assert 'draw_tokens' in dir(zbpe) and zbpe.draw_tokens and sys.modules['torch']\nprint('fine')\n"))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": os.path.dirname(os.path.dirname(zbpe.__file__))})
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr


# ---- devices -------------------------------------------------------------------------------------------------------------------


def test_a_grammar_needs_a_vocabulary_on_a_gpu():
    v = zbpe.Vocabulary([(97, 98, 256)], 300, device="cpu")
    assert v.lengths()[[0, 256, 299]].tolist() == [1, 2, 0]
    with pytest.raises(zbpe.InvalidArgument, match="not on a GPU"):
        zbpe.Grammar(v, torch.zeros(3, 256, dtype=torch.int32))


@gpu
def test_bits_per_byte_on_another_device():
    v = zbpe.Vocabulary([(97, 98, 256)], 300, device="cpu")
    z, tokens = torch.zeros(4, 300, device="cuda"), torch.tensor([1, 2, 256, -1], device="cuda")
    with pytest.raises(zbpe.InvalidArgument, match="the vocabulary is on cpu"):
        v.bits_per_byte(z, tokens)
    there = zbpe.Vocabulary([(97, 98, 256)], 300, device="cuda")
    np.testing.assert_allclose(float(there.bits_per_byte(z, tokens)), 3 * np.log2(300) / 4, rtol=400 * U)


# ---- messages ------------------------------------------------------------------------------------------------------------------


def test_an_older_message_is_not_taken_for_a_later_failure():
    """zbpe_last_error(NULL) after a call without a context that has no message: not that of an operator's call before it"""
    L = zbpe.load_library()
    for fail in (lambda: L.zbpe_create(0, None), lambda: L.zbpe_comm_unique_id(None), lambda: L.zbpe_create_dist(0, 1, 1, None, None),
                 lambda: L.zbpe_create_dist_host(0, 0, 0, zbpe.COLLECTIVE_FN(), None, None), lambda: L.zbpe_upload(None, None, 0),
                 lambda: L.zbpe_tokens(None, None, 0, None), lambda: L.zbpe_zig_order_winner(None, None, None, 0, 0, 0, None)):
        assert L.zbpe_adjust_logits(0, None, None) == 5 and b"no arguments" in L.zbpe_last_error(None)
        assert fail() == 5
        assert L.zbpe_last_error(None) == b"null context"
    assert L.zbpe_draw_tokens(0, None, None) == 5 and b"zbpe_draw_tokens" in L.zbpe_last_error(None)


# ---- small uniform numbers -----------------------------------------------------------------------------------------------------


@gpu
def test_draw_by_a_very_small_uniform():
    """The token is the first at which the sum exceeds u times the whole, exactly, also where u is no multiple of 2^-64: column 0
    weighs x steps of 2^-47 beside 60000 columns of 2^47 steps, and u times the whole lies just above x, or just below it."""
    cols = 60001
    cases = []
    for x in range(3, 4000):
        z0 = np.float32(np.log(x * 2.0 ** -47))
        near = np.exp(np.float64(z0)) * 2.0 ** 47
        if abs(near - np.round(near)) > 0.25:  # (far from where the weight's own rounding turns)
            continue
        x = int(np.round(near))
        whole = 60000 * 2 ** 47 + x
        u = np.float32(x / whole)
        if int(float(u).hex().split("p")[1]) > -41:
            continue
        for v in (u, np.nextafter(u, np.float32(1)), np.nextafter(u, np.float32(0))):
            exact = int(float(v) * 2.0 ** 100) * whole  # (u is a multiple of 2^-100 here; times 2^100)
            assert int(float(v) * 2.0 ** 100) == float(v) * 2.0 ** 100
            first = 0 if x * 2 ** 100 > exact else 1
            cut_off = 0 if x > (int(float(v) * 2.0 ** 64) * whole) >> 64 else 1
            cases.append((z0, v, first, first != cut_off))
    assert sum(c[3] for c in cases) > 20, "cases in which cutting u off at 2^-64 would draw another token"
    cases = [c for c in cases if c[3]][:24] + cases[:24]
    z = torch.zeros(len(cases), cols)
    z[:, 0] = torch.tensor([float(c[0]) for c in cases])
    tokens, _ = zbpe.draw_tokens(z.cuda(), torch.tensor([float(c[1]) for c in cases]).cuda())
    assert tokens.tolist() == [c[2] for c in cases]
    tiny = torch.tensor([2.0 ** -149, 2.0 ** -126, 2.0 ** -64, 0.0], device="cuda")
    assert zbpe.draw_tokens(torch.zeros(4, 300, device="cuda"), tiny)[0].tolist() == [0] * 4


# ---- merge tables --------------------------------------------------------------------------------------------------------------


def test_a_table_of_other_rows_is_no_table_of_triples():
    """3 pairs are 6 numbers, as 2 triples are"""
    for bad in ([[97, 98], [99, 100], [101, 102]], np.zeros((3, 2, 2), np.int64), np.zeros((3, 4), np.uint16), [[97] * 6]):
        with pytest.raises(zbpe.InvalidArgument, match="triples"):
            zbpe.token_bytes(bad)
    want = zbpe.token_bytes([[97, 98, 256], [256, 99, 257]])
    for good in ([97, 98, 256, 256, 99, 257], [[[97, 98, 256]], [[256, 99, 257]]]):
        got = zbpe.token_bytes(good)
        assert (got[0] == want[0]).all() and (got[1] == want[1]).all()
    assert len(zbpe.token_bytes(np.zeros((0, 2)))[0]) == 257


# ---- draws from many tokens ----------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [700, 1024, 1025, 5000, 32000, 65536])
@pytest.mark.parametrize("shape", ["normal", "levels", "flat", "steep"])
def test_draw_with_large_cuts(shape, cols, kind):
    """Cuts that leave more tokens than a workgroup has threads: by rank (top_k), by share (top_p), one after the other, and within
    thousands of equal logits, where the cut lies between two ids. `steep`: all but a few logits lie in one narrow range."""
    rng = np.random.default_rng(cols)
    rows = 8
    z = rng.standard_normal((rows, cols))
    if shape == "levels":
        z = np.round(z)
    elif shape == "flat":
        z = np.full((rows, cols), 0.25)
    elif shape == "steep":
        z = -2 + z * 1e-3
        z[:, rng.integers(0, cols, 5)] = rng.integers(0, 3, (rows, 5))
    z = torch.from_numpy(z).to(kind)
    t = np.float32(1 + rng.random(rows))
    k = np.int32([cols // 2, cols - 1, cols * 3 // 4, 641, 0, 0, cols * 7 // 8, 0])
    p = np.float32([1.0, 1.0, 0.6, 1.0, 0.5, 0.9, 0.95, 0.97])
    m = np.float32([0, 0, 0, 0, 0, 0, 0.01, 0.02])
    check_draw(z, rng, t, k, p, m)
