"""Calls of the operators between a model's logits and its tokens that their definitions allow, or refuse, at the edges:
tensors written in place, forward-mode derivatives, memory that overlaps, numbers, temperatures, devices, messages.

Tolerances count roundings as test_logits.py does: u = 2^-24 for each 32-bit operation.
"""
import ctypes
import subprocess
import sys

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import zbpe
from test_logits import INF, U, adjust_case, close, cuda, gpu, half_step, kept_weights, pack, some_automaton, some_merges, to_gpu


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
