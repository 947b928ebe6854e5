"""The operators between a model's logits and its tokens (zbpe/logits.py) against plain 64-bit implementations.

Tolerances count roundings: u = 2^-24 for each 32-bit operation relative to the largest term it handles, and half a step of
the result's type (finfo.eps / 2 relative, half the smallest subnormal absolute) for the last rounding.
"""
import ctypes

import numpy as np
import pytest
import torch

import zbpe
from helpers import c1_text

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")
gpu = pytest.mark.gpu


def half_step(t):
    f = torch.finfo(t)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def close(got, want, bound):
    """got (tensor) within `bound` (absolute, elementwise) of want (float64 array); equal where want is not finite."""
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    worst = np.abs(got - np.where(finite, want, 0)) - bound
    worst = np.where(finite, worst, -1.0)
    assert not (worst > 0).any() and not np.isnan(got[finite]).any(), f"off by {np.nanmax(np.abs(got - want)[finite])}, {worst.max()} over the bound"


# ---- vocabularies and automata for the tests ----------------------------------------------------------------------------------


def tokens_of(merges, size):
    """bytes of every token, None where it has none"""
    out = [bytes([v]) for v in range(256)] + [None] * (size - 256)
    made = {}
    for a, b, c in merges:
        if c >= 256:
            made.setdefault(c, (a, b))
    def get(v):
        if out[v] is None and v in made:
            out[v] = get(made[v][0]) + get(made[v][1])
        return out[v]
    for v in range(size):
        get(v)
    return out


def some_merges(size, rng, alphabet, most=12, skip=0.0):
    """triples for the ids from 256 on; a share `skip` of the ids is made by no merge"""
    data = {v: bytes([v]) for v in alphabet}
    ids, out = list(alphabet), []
    for c in range(256, size):
        if rng.random() < skip:
            continue
        while True:
            a, b = (int(ids[rng.integers(len(ids))]) for _ in range(2))
            if len(data[a]) + len(data[b]) <= most:
                break
        data[c] = data[a] + data[b]
        ids.append(c)
        out.append((a, b, c))
    return out


def some_automaton(states, rng, alphabet, odd=True):
    table = np.full((states, 256), -1, np.int32)
    for s in range(states):
        kind = rng.integers(4)
        if kind == 0:
            table[s, alphabet] = s
        elif kind == 1:
            table[s, alphabet] = rng.integers(0, states, len(alphabet))
        elif kind == 2:
            few = rng.choice(alphabet, min(3, len(alphabet)), replace=False)
            table[s, few] = rng.integers(0, states, len(few))
        table[s, rng.integers(0, 256, 4)] = rng.integers(0, states, 4)
    if odd and states:  # any value that is no state refuses the byte
        table[rng.integers(0, states, 8), rng.integers(0, 256, 8)] = rng.choice([states, -7, 2 ** 31 - 1, -2 ** 31], 8)
    return table, rng.random(states) < 0.4


def walk(table, s, data):
    for b in data:
        if not 0 <= s < len(table):
            return -1
        s = int(table[s, b])
    return s if 0 <= s < len(table) else -1


def allowed_after(table, accepting, tokens, end, s):
    on = np.zeros(len(tokens), bool)
    if 0 <= s < len(table):
        for v, data in enumerate(tokens):
            on[v] = bool(data) and walk(table, s, data) >= 0
        if end is not None:
            on[end] = accepting[s]
    return on


def unpack(masks, size):
    words = masks.cpu().numpy()
    assert words.shape[-1] == (size + 31) // 32
    bits = np.unpackbits(np.ascontiguousarray(words).view(np.uint8), axis=-1, bitorder="little").astype(bool)
    assert not bits[..., size:].any(), "bits past the vocabulary"
    return bits[..., :size]


def pack(on):
    words = (on.shape[-1] + 31) // 32
    wide = np.zeros((*on.shape[:-1], words * 32), bool)
    wide[..., :on.shape[-1]] = on
    return torch.from_numpy(np.packbits(wide, axis=-1, bitorder="little").view(np.int32))


# ---- on the host ---------------------------------------------------------------------------------------------------------------


def test_token_bytes():
    rng = np.random.default_rng(1)
    merges = some_merges(700, rng, np.arange(97, 103), skip=0.1)
    shuffled = [merges[i] for i in rng.permutation(len(merges))]  # a merge may stand before its halves' merges
    extra = [(1, 2, merges[0][2]), (9, 9, 65)]                    # a second merge of a token, and one of a byte: passed over
    want = tokens_of(merges, 720)
    for table in (merges, shuffled + extra):
        offsets, data = zbpe.token_bytes(np.array(table), 720)
        assert [bytes(data[offsets[v]:offsets[v + 1]]) for v in range(720)] == [w or b"" for w in want]
    offsets, data = zbpe.token_bytes([])
    assert len(offsets) == 257 and bytes(data) == bytes(range(256))
    m = zbpe.Merges()
    m.put(zbpe.CharPair(97, 98), 300)
    offsets, data = zbpe.token_bytes(m)
    assert len(offsets) == 302 and bytes(data[256:]) == b"ab" and offsets[300] == 256


def test_token_bytes_agree_with_decode():
    t = zbpe.BasicTokenizer()
    for a, b, c in some_merges(400, np.random.default_rng(2), np.arange(256)):
        t.merges.put(zbpe.CharPair(a, b), c)
    offsets, data = zbpe.token_bytes(t.merges)
    for v in range(400):
        assert bytes(data[offsets[v]:offsets[v + 1]]) == t.decode([v])


def test_token_bytes_deep_and_long():
    """a chain as deep as the vocabulary (no recursion), and doublings past 2^31 bytes"""
    chain = [(97 if c == 256 else c - 1, 98, c) for c in range(256, 20000)]
    offsets, data = zbpe.token_bytes(np.array(chain[::-1]))
    assert offsets[-1] - offsets[-2] == 19745 and bytes(data[offsets[300]:offsets[301]]) == b"a" + b"b" * 45
    doubled = [(97, 97, 256)] + [(c - 1, c - 1, c) for c in range(257, 256 + 40)]
    with pytest.raises(zbpe.InvalidArgument, match="2\\^31"):
        zbpe.token_bytes(np.array(doubled))
    with pytest.raises(zbpe.InvalidArgument, match="2\\^31"):
        zbpe.token_bytes(np.array(doubled[:30] + [(285, 285, c) for c in range(286, 300)]))


@pytest.mark.parametrize("merges, size, error, words", [
    ([(300, 1, 256)], 400, "InvalidToken", "no merge makes"),
    ([(65535, 1, 256)], 400, "InvalidToken", "no merge makes"),
    ([(256, 1, 256)], None, "InvalidToken", "made from it"),
    ([(257, 1, 256), (1, 256, 257)], None, "InvalidToken", "made from it"),
    ([(1, 2, 400)], 400, "InvalidArgument", "outside a vocabulary"),
    ([(1, 2, 256)], 255, "InvalidArgument", "vocab_size"),
    ([(1, 2, 256)], 65537, "InvalidArgument", "vocab_size"),
    ([(1, 2, 65536)], None, "InvalidArgument", "outside 0"),
    ([(-1, 2, 256)], None, "InvalidArgument", "outside 0"),
    ([1, 2], None, "InvalidArgument", "triples"),
    ([1.5, 2, 256], None, "InvalidArgument", "triples"),
])
def test_token_bytes_refusals(merges, size, error, words):
    with pytest.raises(getattr(zbpe, error), match=words):
        zbpe.token_bytes(merges, size)


@pytest.mark.parametrize("size, skip", [(256, 0.0), (257, 1.0), (700, 0.2), (8192, 0.0), (8255, 0.1), (20000, 0.5)])
def test_vocab_index(size, skip):
    """every token once in its slice, in the order of its bytes; nothing written past the end"""
    rng = np.random.default_rng(size)
    merges = some_merges(size, rng, np.arange(256), most=30, skip=skip)
    offsets, data = zbpe.token_bytes(np.array(merges).reshape(-1, 3), size)
    L = zbpe.load_library()
    n = (size + 63) // 64 * 64
    assert L.zbpe_vocab_index_size(size) == n * 32 + n // 32
    index = np.full(n * 32 + n // 32 + 64, 0xAA, np.uint8)
    assert L.zbpe_vocab_index(offsets.ctypes.data, data.ctypes.data, size, index.ctypes.data) == 0
    assert (index[-64:] == 0xAA).all()
    heads, tails = index[:n * 16].reshape(n, 16), index[n * 16:n * 32].reshape(n, 16)
    bounds = index[n * 32:n * 32 + n // 32].reshape(-1, 2)
    classes = heads[:, :8].copy().view(np.uint64)[:, 0]
    of_byte = {}
    for base in range(0, size, 8192):
        ids = [v for v in range(base, min(base + 8192, size)) if offsets[v] < offsets[v + 1]]
        got = []
        for e in range(base, base + len(ids)):
            v, length = int(heads[e, 8]) + 256 * int(heads[e, 9]) + base, int(heads[e, 10])
            b = data[offsets[v]:offsets[v + 1]].tobytes()
            got.append((v, b[:8]))
            assert length == min(len(b), 22)
            assert heads[e, 11:].tobytes() + tails[e].tobytes() == b[:21].ljust(21, b"\0")
            if len(b) == 1:
                of_byte[b[0]] = int(classes[e])
            want = 0
            for c in b:
                want |= of_byte[c] if c in of_byte else 0
            if base or len(of_byte) == 256:
                assert int(classes[e]) == want
        assert sorted(v for v, _ in got) == ids
        keys = [b.ljust(8, b"\0") for _, b in got]
        assert keys == sorted(keys)
        end = min(base + 8192, n)
        assert not heads[base + len(ids):end].any() and not tails[base + len(ids):end].any()
        for at in range(base, end, 64):
            first = [data[offsets[v]] for v, _ in got[at - base:at - base + 64]]
            assert tuple(bounds[at // 64]) == ((min(first), max(first)) if first else (255, 0))
    assert all(bin(c).count("1") == 1 for c in of_byte.values())


def test_vocab_index_refusals():
    L = zbpe.load_library()
    offsets, data, index = np.array([0, 2, 1], np.uint32), np.zeros(4, np.uint8), np.zeros(4096, np.uint8)
    for size, words in ((2, "offsets of token 1 fall"), (0, "vocabulary of 0"), (65537, "vocabulary of 65537")):
        assert L.zbpe_vocab_index(offsets.ctypes.data, data.ctypes.data, size, index.ctypes.data) == 5
        assert words in L.zbpe_last_error(None).decode()
    assert L.zbpe_vocab_index(offsets.ctypes.data, data.ctypes.data, 2, None) == 5
    assert L.zbpe_vocab_index_size(0) == 0 and L.zbpe_vocab_index_size(65537) == 0


def test_operators_refuse_tensors_off_the_gpu():
    z = torch.zeros(2, 300)
    for call in (lambda: zbpe.adjust_logits(z), lambda: zbpe.draw_tokens(z, torch.zeros(2)),
                 lambda: zbpe.token_logprobs(z, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(zbpe.InvalidArgument, match="not on a GPU"):
            call()
    for bad, words in ((torch.zeros(2, 300, dtype=torch.float64), "float64"), (torch.zeros(2, 0), "0 columns"),
                       (torch.zeros(()), "axis"), (torch.zeros(1, 65537), "65537 columns"), ([1.0], "not a tensor")):
        with pytest.raises(zbpe.InvalidArgument, match=words):
            zbpe.token_logprobs(bad, torch.zeros(2, dtype=torch.int64))


def test_c_entries_refuse_before_any_device_work():
    """arguments are judged on the host: each of these is refused without a GPU, with a message and nothing launched"""
    from zbpe import logits as ops

    L = ops._library()
    assert [L.zbpe_struct_size(i) for i in (-1, 4)] == [0, 0]
    f32, bad = (4096, 300, 300, 0), (4096, 300, 300, 9)

    def refused(status, words):
        assert status == 5 and words in L.zbpe_last_error(None).decode(), (status, L.zbpe_last_error(None))

    def adjust(size=ops._ADJUST.size, cols=300, rows=2, inner=1, z=f32, out=f32, history=(0, 0, 0, 0), hlen=0, n_biases=0, words=0,
               masks=0, mask_rows=0):
        return L.zbpe_adjust_logits(0, None, ops._ADJUST.pack(size, cols, rows, inner, *z, *out, *history, hlen, 0, 0, 0, 0, 0, 0, 0, 0,
                                                              n_biases, words, masks, mask_rows, 0))

    refused(L.zbpe_adjust_logits(0, None, None), "no arguments")
    refused(adjust(size=8), "another version")
    refused(adjust(cols=0), "columns")
    refused(adjust(cols=65537), "columns")
    refused(adjust(rows=-1), "rows")
    refused(adjust(inner=0), "inner")
    refused(adjust(z=bad), "data type 9")
    refused(adjust(z=(0, 300, 300, 0)), "no logits")
    refused(adjust(out=(4096, 300, 300, 1)), "type of the logits")
    refused(adjust(out=(4096, 10, 300, 0)), "overlap")
    refused(adjust(rows=6, inner=3, out=(4096, 301, 300, 0)), "overlap")
    refused(adjust(history=(4096, 8, 8, 0), hlen=8), "history")
    refused(adjust(history=(4096, 8, 8, 3), hlen=-1), "history")
    refused(adjust(history=(4096, 8, 8, 3), hlen=2 ** 31), "2^31")
    refused(adjust(n_biases=1025), "1025 biases")
    refused(adjust(n_biases=4), "without values")
    refused(adjust(masks=4096, words=9, mask_rows=2), "9 words")
    refused(adjust(masks=4096, words=10, mask_rows=3 - 3), "rows of masks")

    def draw(size=ops._DRAW.size, z=f32, uniforms=4096, tokens=4096):
        return L.zbpe_draw_tokens(0, None, ops._DRAW.pack(size, 300, 2, 1, *z, uniforms, 0, 0, 0, 0, tokens, 0))

    refused(draw(size=0), "another version")
    refused(draw(z=bad), "data type 9")
    refused(draw(uniforms=0), "no uniforms")
    refused(draw(tokens=0), "no tokens")

    def logprobs(kind=3, tokens=4096, out=4096):
        return ops._LOGPROBS.pack(ops._LOGPROBS.size, 300, 2, 1, *f32, tokens, kind, 0, out, 0)

    refused(L.zbpe_token_logprobs(0, None, logprobs(kind=0)), "tokens of data type 0")
    refused(L.zbpe_token_logprobs(0, None, logprobs(tokens=0)), "no tokens")
    refused(L.zbpe_token_logprobs(0, None, logprobs(out=0)), "no logprobs")
    refused(L.zbpe_token_logprobs_grad(0, None, logprobs(), 4096, None), "type of the logits")

    def masks(vocab=300, end=-1, states=5, rows=5, next=4096, out=4096, index=4096):
        return L.zbpe_grammar_masks(0, None, ops._GRAMMAR.pack(4096, 4096, vocab, end, next, 0, states, index), None, rows, out)

    refused(masks(vocab=0), "vocabulary of 0")
    refused(masks(end=300), "end token")
    refused(masks(states=1 << 23), "states")
    refused(masks(rows=-1), "rows")
    refused(masks(next=0), "missing")
    refused(masks(out=0), "no masks")
    refused(masks(index=0), "no index")
    assert L.zbpe_adjust_workspace(0, 300) == 0 and L.zbpe_adjust_workspace(-1, 300) == 0


# ---- grammars --------------------------------------------------------------------------------------------------------------------


def cuda(x):
    return torch.as_tensor(x).cuda()


ALPHABET = np.frombuffer(b"abc {}:,01\"\xc3\xa9", np.uint8).astype(np.int64)


@gpu
@pytest.mark.parametrize("size, states, end", [(256, 1, None), (257, 3, 256), (300, 64, 299), (1000, 33, 0), (4097, 130, 4096), (700, 5, 400)])
def test_masks_and_advance(size, states, end):
    rng = np.random.default_rng(size)
    merges = some_merges(size, rng, ALPHABET, skip=0.1)
    table, accepting = some_automaton(states, rng, ALPHABET)
    tokens = tokens_of(merges, size)
    want = np.stack([allowed_after(table, accepting, tokens, end, s) for s in range(states)])
    v = zbpe.Vocabulary(np.array(merges).reshape(-1, 3), size, end)
    g = zbpe.Grammar(v, cuda(table), cuda(accepting))
    assert v.words == (size + 31) // 32 and v.lengths().tolist() == [len(t or b"") for t in tokens]
    np.testing.assert_array_equal(unpack(g.masks(), size), want)

    # rows of states, the same state twice, states outside the automaton
    rows = np.concatenate([rng.integers(0, states, 70), [-1, states, 2 ** 31 - 1, -2 ** 31]]).astype(np.int32)
    inside = (rows >= 0) & (rows < states)
    wanted = np.where(inside[:, None], want[np.where(inside, rows, 0)], False)
    np.testing.assert_array_equal(unpack(g.masks(cuda(rows)), size), wanted)
    np.testing.assert_array_equal(unpack(g.masks(cuda(rows[:70].reshape(7, 10))), size), wanted[:70].reshape(7, 10, -1))
    for r in (0, 69, 71):  # one row alone
        np.testing.assert_array_equal(unpack(g.masks(cuda(rows[r:r + 1])), size), wanted[r:r + 1])

    drawn = rng.integers(0, size, len(rows))
    some = [np.nonzero(w)[0] for w in wanted]
    drawn = np.array([rng.choice(s) if len(s) and rng.random() < 0.7 else d for s, d in zip(some, drawn)]).astype(np.int32)
    drawn[:3] = [-1, size, 2 ** 31 - 1]
    after = np.array([-1 if not 0 <= s < states else s if t < 0 else -1 if t >= size else (s if accepting[s] else -1) if t == end
                      else walk(table, s, tokens[t]) if tokens[t] else -1 for s, t in zip(rows.tolist(), drawn.tolist())])
    np.testing.assert_array_equal(g.advance(cuda(rows), cuda(drawn)).cpu().numpy(), after)


@gpu
def test_masks_of_long_tokens_and_wide_automata():
    """tokens of 1 to 6000 bytes over a counter of 70000 states (past 16 bits), and no accepting states"""
    n = 70000
    table = np.full((n, 256), -1, np.int32)
    table[:-1, 97] = np.arange(1, n)
    merges = [(97, 97, 256)] + [(c - 1, c - 1, c) for c in range(257, 268)] + [(256 + i % 12, 97 + i % 2, 268 + i) for i in range(60)]
    size = 400
    tokens = tokens_of(merges, size)
    v = zbpe.Vocabulary(np.array(merges), size, 399)
    g = zbpe.Grammar(v, torch.from_numpy(table))  # (from the host)
    rows = np.array([0, 1, 65535, 65536, n - 4097, n - 4096, n - 2, n - 1], np.int32)
    want = np.stack([[bool(t) and set(t) == {97} and s + len(t) < n for t in tokens] for s in rows])
    np.testing.assert_array_equal(unpack(g.masks(cuda(rows)), size), want)
    for v_ in (97, 256, 267, 268, 269):
        got = g.advance(cuda(rows), torch.full((len(rows),), v_, dtype=torch.int32, device="cuda"))
        assert got.tolist() == [walk(table, s, tokens[v_]) for s in rows.tolist()]


@gpu
def test_masks_of_every_state_of_a_large_automaton():
    """rows against the same rows asked for by state, over the sizes where the kernel's split changes"""
    rng = np.random.default_rng(5)
    merges = some_merges(5000, rng, np.arange(256), skip=0.01)
    v = zbpe.Vocabulary(np.array(merges), 5001, 5000)
    for states in (1, 2, 63, 257, 1500):
        table, accepting = some_automaton(states, rng, np.arange(32, 127))
        g = zbpe.Grammar(v, cuda(table), cuda(accepting))
        whole = g.masks()
        order = torch.randperm(states).int().cuda()
        assert torch.equal(whole[order.long()], g.masks(order))
        one = int(rng.integers(states))
        tokens = tokens_of(merges, 5001)
        np.testing.assert_array_equal(unpack(whole[one], 5001), allowed_after(table, accepting, tokens, 5000, one))


@gpu
def test_masks_of_many_rows_over_several_slices():
    """rows enough that a workgroup takes several slices of ids; tokens longer than the index holds; states with many successors"""
    rng = np.random.default_rng(11)
    size, end = 20000, 12345
    merges = some_merges(size, rng, ALPHABET, most=40, skip=0.02)
    table, accepting = some_automaton(60, rng, ALPHABET)
    table[0, ALPHABET] = 0
    table[1, ALPHABET] = np.arange(len(ALPHABET)) + 1
    accepting[0] = True
    tokens = tokens_of(merges, size)
    assert max(len(t) for t in tokens if t) > 30
    g = zbpe.Grammar(zbpe.Vocabulary(np.array(merges), size, end), cuda(table), cuda(accepting))
    few = np.array([0, 1, 2, 59, -1, 60], np.int32)
    want = np.stack([allowed_after(table, accepting, tokens, end, int(s)) for s in few])
    for rows in (len(few), 400, 1500, 3000, 6000):
        pick = np.concatenate([np.arange(len(few)), rng.integers(0, len(few), rows - len(few))])
        got = g.masks(cuda(few[pick]))
        np.testing.assert_array_equal(unpack(got[:len(few)], size), want)
        assert torch.equal(got, got[:len(few)][torch.from_numpy(pick).cuda()])


@gpu
def test_grammar_edges_and_refusals():
    v = zbpe.Vocabulary([], 256)
    g = zbpe.Grammar(v, torch.zeros(0, 256, dtype=torch.int32))  # no states: nothing is allowed, nothing moves
    assert g.masks().shape == (0, 8)
    s = torch.tensor([0, -1], dtype=torch.int32, device="cuda")
    assert not g.masks(s).any() and g.advance(s, s).tolist() == [-1, -1]
    assert g.masks(s[:0]).shape == (0, 8) and g.advance(s[:0], s[:0]).shape == (0,)
    g = zbpe.Grammar(v, torch.tensor([[2 ** 32] * 256, [0] * 256]))  # (a wide type: no state either)
    assert unpack(g.masks(), 256).tolist() == [[False] * 256, [True] * 256]
    out = torch.full((2, 8), 7, dtype=torch.int32, device="cuda")
    assert g.masks(out=out) is out and out[0].tolist() == [0] * 8
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    for call, words in ((lambda: zbpe.Grammar(v, torch.zeros(3, 255, dtype=torch.int32)), "shape"),
                        (lambda: zbpe.Grammar(v, torch.zeros(3, 256)), "whole numbers"),
                        (lambda: zbpe.Grammar(v, torch.zeros(3, 256, dtype=torch.int32), torch.zeros(2, dtype=torch.bool)), "3 states"),
                        (lambda: zbpe.Grammar(v, torch.zeros(3, 256, dtype=torch.int32), torch.zeros(3)), "bool"),
                        (lambda: zbpe.Grammar([], torch.zeros(3, 256, dtype=torch.int32)), "not a Vocabulary"),
                        (lambda: zbpe.Vocabulary([], 300, 300), "end_token"),
                        (lambda: zbpe.Vocabulary([], 300, -1), "end_token"),
                        (lambda: g.masks(t.long()), "int32"), (lambda: g.masks(t.cpu()), "on cpu"),
                        (lambda: g.masks(t, out=t), "packed"), (lambda: g.advance(t, t[:2]), "shape"),
                        (lambda: g.advance(t, t.long()), "int32")):
        with pytest.raises(zbpe.InvalidArgument, match=words):
            call()


# ---- penalties, biases and masks -----------------------------------------------------------------------------------------------------


def adjust_case(rows, cols, seed, history=40, biases=6, mask_rows=5, kind=torch.float32, wide=False, scale=4.0):
    rng = np.random.default_rng(seed)
    z = torch.from_numpy(rng.standard_normal((rows, cols)) * scale).to(kind)
    if rows * cols > 4:
        z.view(-1)[rng.integers(0, rows * cols, 3)] = 0.0
    ids = rng.integers(-3, cols + 3, (rows, history))  # (some outside the vocabulary)
    ids[:, ::3] = rng.integers(0, min(cols, 7), ids[:, ::3].shape)  # often the same
    lengths = rng.integers(-2, history + 3, rows)
    x = dict(history=torch.from_numpy(ids).to(torch.int64 if wide else torch.int32), lengths=torch.from_numpy(lengths).int(),
             prompt_lengths=torch.from_numpy(rng.integers(-2, history + 3, rows)).int(),
             repetition=torch.from_numpy(1 + rng.random(rows)).float(), presence=torch.from_numpy(rng.random(rows) - 0.3).float(),
             frequency=torch.from_numpy(rng.random(rows) - 0.3).float(), bias=torch.from_numpy(rng.standard_normal(cols)).float(),
             bias_tokens=torch.from_numpy(rng.integers(-2, cols + 2, (rows, biases))).int(),
             bias_values=torch.from_numpy(rng.standard_normal((rows, biases))).float())
    if biases > 2:
        x["bias_tokens"][:, 1] = x["bias_tokens"][:, 0]  # the same token twice
    on = rng.random((mask_rows, cols)) < 0.6
    on[0] = False  # a mask that leaves nothing
    x["masks"] = pack(on)
    x["states"] = torch.from_numpy(rng.integers(-1, mask_rows + 1, rows)).int()
    return z, x


def adjust_oracle(z, x, up=None):
    """(y, bound without the last rounding[, dz, dbias, dbias_values, their bounds])"""
    z = z.detach().double().numpy()
    rows, cols = z.shape
    get = lambda k, default: np.broadcast_to(np.float64(default), rows) if x.get(k) is None else np.broadcast_to(  # noqa: E731
        np.asarray(x[k].detach() if isinstance(x[k], torch.Tensor) else x[k], np.float64), rows)
    y, most = z.copy(), np.abs(z)
    slope = np.ones_like(z)
    if x.get("history") is not None:
        h = x["history"].numpy()
        n = np.clip(get("lengths", h.shape[1]), 0, h.shape[1]).astype(int)
        prompt, theta = get("prompt_lengths", 0), get("repetition", 1)
        for r in range(rows):
            for v in set(h[r, :n[r]].tolist()):
                if not 0 <= v < cols:
                    continue
                slope[r, v] = 1 / theta[r] if y[r, v] > 0 else theta[r]
                y[r, v] *= slope[r, v]
                c = int((h[r, max(int(prompt[r]), 0):n[r]] == v).sum())
                most[r, v] = max(most[r, v], abs(y[r, v]))
                if c:
                    y[r, v] -= get("frequency", 0)[r] * c
                    y[r, v] -= get("presence", 0)[r]
                    most[r, v] += abs(get("frequency", 0)[r]) * c + abs(get("presence", 0)[r])
    if x.get("bias") is not None:
        y += x["bias"].detach().double().numpy()
        most += np.abs(x["bias"].detach().double().numpy())
    if x.get("bias_tokens") is not None:
        t, val = x["bias_tokens"].numpy(), x["bias_values"].detach().double().numpy()
        for r in range(rows):
            for v, b in zip(t[r], val[r]):
                if 0 <= v < cols:
                    y[r, v] += b
                    most[r, v] += abs(b)
    allowed = np.ones_like(z, bool)
    if x.get("masks") is not None:
        on = unpack(x["masks"], cols).reshape(-1, cols)
        states = x["states"].numpy().reshape(-1) if x.get("states") is not None else np.arange(rows) if len(on) != 1 else np.zeros(rows, int)
        good = (states >= 0) & (states < len(on))
        allowed = on[np.where(good, states, 0)] & good[:, None]
    y = np.where(allowed, y, -np.inf)
    # a rounding for each of: *theta, f*c, -, -, + bias, + row's sum; one for each further entry of that sum
    nb = 0 if x.get("bias_tokens") is None else x["bias_tokens"].shape[1]
    bound = (6 + nb) * U * np.where(np.isfinite(most), most, 0)
    if up is None:
        return y, bound
    g = np.where(allowed, up.double().numpy(), 0)
    dz = g * slope
    dv = np.zeros((rows, nb))
    for r in range(rows):
        for j in range(nb):
            v = int(x["bias_tokens"][r, j])
            dv[r, j] = g[r, v] if 0 <= v < cols else 0
    return y, bound, dz, g.sum(0), dv, rows * U * np.abs(g).sum(0)


def to_gpu(x):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in x.items()}


def check_adjust(z, x, kind, **kw):
    y, bound = adjust_oracle(z, x)
    relative, least = half_step(kind)
    got = zbpe.adjust_logits(z.cuda(), **to_gpu(x), **kw)
    assert got.dtype == kind
    close(got, y, bound + (np.where(np.isfinite(y), np.abs(y), 0) + bound) * relative + least)
    return got


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 31), (3, 257), (2, 4096), (5, 4099), (7, 12345), (1, 65536)])
def test_adjust(rows, cols, kind):
    z, x = adjust_case(rows, cols, rows + cols, kind=kind, wide=rows == 7)
    check_adjust(z, x, kind)


@gpu
@pytest.mark.parametrize("names", [(), ("history",), ("history", "repetition"), ("history", "lengths", "frequency"),
                                   ("history", "prompt_lengths", "presence"), ("bias",), ("bias_tokens", "bias_values"), ("masks", "states")])
def test_adjust_by_parts(names):
    z, x = adjust_case(6, 1001, 3)
    check_adjust(z, {k: x[k] for k in names}, torch.float32)


@gpu
@pytest.mark.parametrize("history, biases", [(0, 0), (1, 1), (63, 2), (5000, 64), (300, 1024)])
def test_adjust_sizes_of_history_and_biases(history, biases):
    z, x = adjust_case(3, 6000, history + biases, history=history, biases=biases)
    check_adjust(z, x, torch.float32)


@gpu
def test_adjust_numbers_masks_of_rows_and_one_for_all():
    z, x = adjust_case(4, 777, 9, mask_rows=4)
    one = dict(history=x["history"], repetition=1.5, presence=1, frequency=-0.25)
    y, bound = adjust_oracle(z, one)
    close(zbpe.adjust_logits(z.cuda(), **to_gpu(one)), y, bound + np.abs(y) * U)
    check_adjust(z, {"masks": x["masks"]}, torch.float32)
    check_adjust(z, {"masks": x["masks"][1]}, torch.float32)
    check_adjust(z, {"masks": x["masks"][1:2]}, torch.float32)
    wide = torch.cat([x["masks"], torch.full((4, 9), -1, dtype=torch.int32)], 1)  # (rows of masks longer than the vocabulary)
    got = zbpe.adjust_logits(z.cuda(), masks=wide.cuda())
    assert torch.equal(got, zbpe.adjust_logits(z.cuda(), masks=x["masks"].cuda()))


@gpu
@pytest.mark.parametrize("kind", TYPES)
def test_adjust_strides_axes_and_out(kind):
    """views of wider buffers at odd starts, three and four axes, broadcast rows, transposed histories; `out` in place and wider"""
    z, x = adjust_case(12, 1003, 4, kind=kind)
    want = check_adjust(z, x, kind)
    g = to_gpu(x)
    wide = torch.full((12, 1100), 9.0, dtype=kind, device="cuda")
    view = wide[:, 5:1008]
    view.copy_(z)
    assert torch.equal(zbpe.adjust_logits(view, **g), want)
    h = g["history"].t().contiguous().t()
    assert torch.equal(zbpe.adjust_logits(view, **{**g, "history": h}), want)
    shaped = {k: v.view(3, 4, *v.shape[1:]) if k not in ("bias", "masks") else v for k, v in g.items()}
    cut = wide.view(3, 4, 1100)[..., 5:1008]
    assert torch.equal(zbpe.adjust_logits(cut, **shaped), want.view(3, 4, -1))
    four = {k: v.view(3, 1, 4, *v.shape[1:]) if k not in ("bias", "masks") else v for k, v in g.items()}
    assert torch.equal(zbpe.adjust_logits(cut[:, None], **four), want.view(3, 1, 4, -1))
    long = torch.zeros(4, 3, 1100, dtype=kind, device="cuda").transpose(0, 1)  # time before batch in memory
    long[..., 5:1008] = cut
    assert torch.equal(zbpe.adjust_logits(long[..., 5:1008], **shaped), want.view(3, 4, -1))
    assert torch.equal(zbpe.adjust_logits(z.cuda().t().contiguous().t(), **g), want)  # columns apart
    same = z[:1].cuda().expand(12, -1)
    assert torch.equal(zbpe.adjust_logits(same, **g), zbpe.adjust_logits(same.contiguous(), **g))
    out = torch.full((12, 1100), 9.0, device="cuda")  # 32 bits, in rows that are apart
    close(zbpe.adjust_logits(view, **g, out=out[:, 5:1008]), *adjust_f32(z, x))
    assert (out[:, :5] == 9).all() and (out[:, 1008:] == 9).all()
    assert zbpe.adjust_logits(view, **g, out=view) is view and torch.equal(view, want)
    assert (wide[:, :5] == 9).all() and (wide[:, 1008:] == 9).all(), "written past the rows"
    one = {k: v[0] if k not in ("bias", "masks") else v for k, v in g.items()}
    assert torch.equal(zbpe.adjust_logits(z[0].cuda(), **one), want[0])
    none = {k: v[:0] if k not in ("bias", "masks") else v for k, v in g.items()}
    assert zbpe.adjust_logits(z[:0].cuda(), **none).shape == (0, 1003)


def adjust_f32(z, x):
    y, bound = adjust_oracle(z, x)
    return y, bound + (np.where(np.isfinite(y), np.abs(y), 0) + bound) * U + 2.0 ** -150


@gpu
@pytest.mark.parametrize("kind", TYPES)
def test_adjust_infinities_nan_and_lowest(kind):
    low = torch.finfo(kind).min
    z = torch.tensor([[INF, -INF, float("nan"), low, 0.0, -0.0, 1.0, torch.finfo(kind).max]], dtype=kind)
    on = torch.tensor([[True] * 8, [False] * 8, [False, False, False, True, True, True, True, True]])
    got = zbpe.adjust_logits(z.expand(3, -1).cuda(), masks=pack(on.numpy()).cuda())
    assert torch.equal(got[0].cpu().view(torch.uint8), z[0].view(torch.uint8))  # every bit kept, -0 and NaN too
    assert (got[1] == -INF).all() and (got[2, :3] == -INF).all() and torch.equal(got[2, 3:].cpu(), z[0, 3:])
    h = torch.arange(8, dtype=torch.int32).view(1, 8)
    got = zbpe.adjust_logits(z.cuda(), history=h.cuda(), repetition=2.0).cpu()[0].float()
    assert got[0] == INF and got[1] == -INF and got[2].isnan() and got[3] == -INF and got[4] == 0 and got[6] == 0.5
    assert got[7] == torch.finfo(kind).max / 2


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 257), (70, 4099), (2100, 301), (1, 65536)])
def test_adjust_gradients(rows, cols, kind):
    z, x = adjust_case(rows, cols, rows * 3 + cols, kind=kind, history=25)
    up = torch.from_numpy(np.random.default_rng(1).standard_normal((rows, cols))).to(kind)
    _, _, dz, db, dv, db_bound = adjust_oracle(z, x, up)
    g = to_gpu(x)
    zg = z.cuda().requires_grad_()
    g["bias"].requires_grad_()
    g["bias_values"].requires_grad_()
    got = torch.autograd.grad(zbpe.adjust_logits(zg, **g), [zg, g["bias"], g["bias_values"]], up.cuda())
    relative, least = half_step(kind)
    assert got[0].dtype == kind
    close(got[0], dz, np.abs(dz) * (relative + 2 * U) + least)
    close(got[1], db, db_bound)
    close(got[2], dv, np.abs(dv) * 0)
    # one at a time, and only what is asked for
    for i, name in enumerate(("logits", "bias", "bias_values")):
        z1 = z.cuda().requires_grad_(i == 0)
        g1 = {k: v.detach().requires_grad_(k == name) if v.is_floating_point() else v for k, v in g.items()}
        leaf = z1 if i == 0 else g1[name]
        assert torch.equal(torch.autograd.grad(zbpe.adjust_logits(z1, **g1), leaf, up.cuda())[0], got[i])


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("history, biases, wide", [(1300, 3, True), (2600, 700, False)])
def test_adjust_runs_of_rows(kind, history, biases, wide):
    """several rows and slices for a workgroup, histories and biases longer than one load of it, rows cut out of a wider tensor"""
    lead, cols = (20, 15), 9001
    z, x = adjust_case(300, cols, history, history=history, biases=biases, kind=kind, wide=wide)
    up = torch.from_numpy(np.random.default_rng(2).standard_normal((300, cols))).to(kind)
    y, bound, dz, db, dv, db_bound = adjust_oracle(z, x, up)
    g = {k: v.view(*lead, *v.shape[1:]) if k not in ("bias", "masks") else v for k, v in to_gpu(x).items()}
    whole = torch.zeros(20, 17, cols, dtype=kind, device="cuda")
    whole[:, 1:16] = z.view(*lead, cols).cuda()
    zg = whole[:, 1:16].requires_grad_()
    g["bias"].requires_grad_()
    g["bias_values"].requires_grad_()
    out = zbpe.adjust_logits(zg, **g)
    relative, least = half_step(kind)
    close(out.view(300, cols), y, bound + (np.where(np.isfinite(y), np.abs(y), 0) + bound) * relative + least)
    got = torch.autograd.grad(out, [zg, g["bias"], g["bias_values"]], up.view(*lead, cols).cuda())
    close(got[0].reshape(300, cols), dz, np.abs(dz) * (relative + 2 * U) + least)
    close(got[1], db, db_bound)
    close(got[2].reshape(300, -1), dv, np.abs(dv) * 0)
    # in place, and nothing beside the rows
    target = whole.clone()
    with torch.no_grad():
        zbpe.adjust_logits(target[:, 1:16], **g, out=target[:, 1:16])
    assert torch.equal(target[:, 1:16], out) and not target[:, 0].any() and not target[:, 16].any()


@gpu
def test_adjust_gradients_by_differences():
    """central differences of the 64-bit function along random directions, where no logit changes sign"""
    z, x = adjust_case(4, 300, 8, history=30)
    z = torch.where(z.abs() < 0.1, 0.5, z)
    w = torch.from_numpy(np.random.default_rng(3).standard_normal((4, 300))).float()
    f = lambda z, x: float(np.where(np.isfinite(o := adjust_oracle(z, x)[0]), o * w.numpy(), 0).sum())  # noqa: E731
    g = to_gpu(x)
    zg = z.cuda().requires_grad_()
    g["bias"].requires_grad_()
    g["bias_values"].requires_grad_()
    out = zbpe.adjust_logits(zg, **g)
    grads = torch.autograd.grad(torch.where(out > -INF, out, 0.0).mul(w.cuda()).sum(), [zg, g["bias"], g["bias_values"]])
    h = 1e-3
    for grad, base, name in zip(grads, (z, x["bias"], x["bias_values"]), ("z", "bias", "bias_values")):
        d = torch.from_numpy(np.random.default_rng(5).standard_normal(tuple(base.shape)))
        ends = [f(base.double() + s * d, x) if name == "z" else f(z, {**x, name: base.double() + s * d}) for s in (h, -h)]
        # the function is linear on this interval: the difference is exact up to 64-bit roundings (2^-52 of the sum / h), the
        # gradient's entries are off by U of themselves and the bias's sum by 4 U
        size = float((grad.double().cpu() * d).abs().sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - float((grad.double().cpu() * d).sum())) < 8 * U * size + 1e-9


@gpu
def test_adjust_gradient_views_and_broadcast_gradients():
    """a gradient that is broadcast (from a sum) or a cut of a wider tensor; logits that are"""
    z, x = adjust_case(6, 515, 2)
    g = to_gpu(x)
    wide = torch.zeros(2, 3, 600, device="cuda")
    wide[..., 3:518] = z.view(2, 3, -1)
    wide.requires_grad_()
    shaped = {k: v.view(2, 3, *v.shape[1:]) if k not in ("bias", "masks") else v for k, v in g.items()}
    _, _, dz, _, _, _ = adjust_oracle(z, x, torch.ones(6, 515))
    torch.where((out := zbpe.adjust_logits(wide[..., 3:518], **shaped)) > -INF, out, 0.0).sum().backward()
    want = np.zeros((2, 3, 600))
    want[..., 3:518] = dz.reshape(2, 3, -1)
    close(wide.grad, want, np.abs(want) * 3 * U)
    z1 = z.cuda().requires_grad_()
    out = zbpe.adjust_logits(z1, **g)
    got = torch.autograd.grad(out, z1, torch.ones(1, 1, device="cuda").expand(6, 515))[0]
    close(got, dz, np.abs(dz) * 3 * U)


@gpu
def test_adjust_refusals():
    z, x = adjust_case(4, 300, 1)
    g, z = to_gpu(x), z.cuda()
    def no(words, **kw):
        with pytest.raises(zbpe.InvalidArgument, match=words):
            zbpe.adjust_logits(z, **kw)
    no("history", repetition=1.5)
    no("history", lengths=g["lengths"])
    no("float32", history=g["history"].float())
    no("shape", history=g["history"][:3])
    no("shape", history=g["history"], lengths=g["lengths"][:3])
    no("int64", history=g["history"], lengths=g["lengths"].long())
    no("detach", history=g["history"], repetition=g["repetition"].clone().requires_grad_())
    no("neither", history=g["history"], repetition="1")
    no("bias is not", bias=g["bias"][:299])
    no("bias is not", bias=g["bias"].half())
    no("bias_values", bias_tokens=g["bias_tokens"])
    no("different shapes", bias_tokens=g["bias_tokens"], bias_values=g["bias_values"][:, :3])
    no("1025 biases", bias_tokens=torch.zeros(4, 1025, dtype=torch.int32, device="cuda"), bias_values=torch.zeros(4, 1025, device="cuda"))
    no("too narrow", masks=g["masks"][:, :9])
    no("rows are", masks=g["masks"][:3])
    no("no rows", masks=g["masks"][:0], states=g["states"])
    no("without masks", states=g["states"])
    no("on cpu", masks=x["masks"])
    no("int64", masks=g["masks"].long())
    no("out is not", out=torch.zeros(4, 300, dtype=torch.float16, device="cuda"))
    no("out is not", out=torch.zeros(4, 301, device="cuda"))
    no("strides", out=torch.zeros(300, 4, device="cuda").t())
    no("overlap", out=torch.zeros(1, 300, device="cuda").expand(4, 300))
    with pytest.raises(zbpe.InvalidArgument, match="without gradients"):
        zbpe.adjust_logits(z.clone().requires_grad_(), out=z)


# ---- the draw ---------------------------------------------------------------------------------------------------------------------------


def kept_weights(z, t, k, p, m):
    """float64 weights of one row's tokens, 0 where the filters drop them"""
    z = np.where(np.isnan(z), -np.inf, z)
    top = z.max()
    w = np.where(z == top, 1.0, np.exp((np.where(z == top, 0.0, z - (top if np.isfinite(top) else 0.0)) / t)) if np.isfinite(top) else 0.0)
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -np.inf]
    if k > 0:
        order = order[:k]
    if p < 1:
        s = np.cumsum(w[order])
        order = order[np.concatenate([[0.0], s[:-1]]) < p * s[-1]] if p > 0 else order[:1]
    order = order[w[order] >= min(m, 1.0)] if m > 0 else order
    out = np.zeros_like(w)
    out[order] = w[order]
    return out


def draw_case(rows, cols, seed, kind, ties=False):
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((rows, cols)) * 3
    if ties:
        z = np.round(z * 2) / 2
    return torch.from_numpy(z).to(kind), rng


def check_draw(z, rng, t, k, p, m):
    """Draws the row's tokens at the middle of intervals of the kept weights (a border is off by less than 2^-30 of the whole);
    p lies in the middle between two sums, m between two weights."""
    rows = z.shape[0]
    z64 = z.double().numpy()
    u, want, logprob = np.zeros(rows, np.float32), np.zeros(rows, np.int32), np.zeros(rows)
    for r in range(rows):
        if 0 < p[r] < 1:
            w = kept_weights(z64[r], t[r], k[r], 1.0, 0.0)
            w = np.sort(w)[::-1] / w.sum()
            s = np.cumsum(w)
            i = min(int(np.searchsorted(s, p[r])), int((w > 2.0 ** -20).sum()) - 1)  # (a middle that float32 can name)
            p[r] = np.float32(s[i] - w[i] / 2)
        if 0 < m[r] < 1:
            w = np.unique(kept_weights(z64[r], t[r], k[r], 1.0, 0.0))
            i = int(np.searchsorted(w, m[r]))
            m[r] = np.float32((w[i - 1] + w[min(i, len(w) - 1)]) / 2 if i else m[r])
        w = kept_weights(z64[r], t[r], k[r], float(p[r]), float(m[r]))
        ends = np.cumsum(w) / w.sum()
        wide = np.nonzero(w / w.sum() > 2.0 ** -20)[0]  # (a middle that float32 can name)
        v = int(rng.choice(wide))
        u[r] = np.float32(ends[v] - w[v] / w.sum() / 2)
        want[r], logprob[r] = v, np.log(w[v] / w.sum())
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()  # noqa: E731
    got = zbpe.draw_tokens(z.cuda(), torch.from_numpy(u).cuda(), temperature=f(t), top_k=torch.from_numpy(np.asarray(k, np.int32)).cuda(),
                           top_p=f(p), min_p=f(m))
    np.testing.assert_array_equal(got[0].cpu().numpy(), want)
    # one rounding to 32 bits; 2^-40: 64-bit sums of weights in steps of 2^-47
    close(got[1], logprob, np.abs(logprob) * U + 2.0 ** -40)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 257, 2048, 2049, 8192, 8193, 32000, 32769, 65535, 65536])
def test_draw(cols, kind):
    rows = 24
    for ties in (False, True):
        z, rng = draw_case(rows, cols, cols, kind, ties)
        t = np.float32(0.4 + rng.random(rows))
        k = np.where(rng.random(rows) < 0.5, rng.integers(1, min(cols, 300) + 1, rows), rng.integers(-1, 1, rows)).astype(np.int32)
        p = np.where(rng.random(rows) < 0.5, 0.3 + 0.69 * rng.random(rows), rng.choice([1.0, 2.0], rows)).astype(np.float32)
        m = np.where(rng.random(rows) < 0.5, 0.3 * rng.random(rows), rng.choice([0.0, -1.0], rows)).astype(np.float32)
        check_draw(z, rng, t, k, p, m)


@gpu
def test_draw_top_p_among_ties():
    """eight equal logits and 300 far below: top_p keeps the first of the equal ones, by id"""
    z = torch.full((8, 308), -40.0, device="cuda")
    at = torch.arange(8, device="cuda") * 37 + 5
    z[:, at] = 2.0
    p = (torch.arange(8, device="cuda") + 0.5) / 8
    tokens, logprobs = zbpe.draw_tokens(z, torch.full((8,), 0.99999, device="cuda"), top_p=p)
    assert tokens.tolist() == at.tolist()
    # the sum over eight equal weights is exact
    np.testing.assert_allclose(logprobs.cpu().numpy(), -np.log(np.arange(1, 9)), rtol=2 * U, atol=0)
    tokens, _ = zbpe.draw_tokens(z, torch.full((8,), 0.99999, device="cuda"), top_k=torch.arange(1, 9, device="cuda").int())
    assert tokens.tolist() == at.tolist()


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [300, 5000, 65536])
def test_draw_extremes(cols, kind):
    z, rng = draw_case(9, cols, 1, kind, ties=True)
    u = torch.rand(9, generator=torch.Generator().manual_seed(1)).cuda()
    first = torch.from_numpy(np.argmax(z.double().numpy(), 1))
    for kw in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=1), dict(top_p=0.0),
               dict(top_p=-1.0), dict(top_k=1, top_p=0.5, min_p=0.5)):
        kw = {k: torch.full((9,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda") for k, v in kw.items()}
        tokens, logprobs = zbpe.draw_tokens(z.cuda(), u, **kw)
        assert torch.equal(tokens.cpu().long(), first) and (logprobs == 0).all()
    # min_p of 1 or more keeps the ties of the largest
    tokens, logprobs = zbpe.draw_tokens(z.cuda(), torch.full((9,), 0.9999999, device="cuda"), min_p=3.0)
    top = z.double().numpy().max(1)
    last = [np.nonzero(row == m)[0] for row, m in zip(z.double().numpy(), top)]
    assert tokens.tolist() == [int(i[-1]) for i in last]
    np.testing.assert_allclose(logprobs.cpu().numpy(), [-np.log(len(i)) for i in last], rtol=2 * U, atol=0)
    # uniforms outside [0, 1) are the nearest inside; the last token with a weight, not the last column
    z[:, -1] = -INF
    a, _ = zbpe.draw_tokens(z.cuda(), torch.tensor([0.0, -3.0, float("nan")] * 3, device="cuda"), min_p=0.5)
    b, _ = zbpe.draw_tokens(z.cuda(), torch.tensor([1.0, 7.0, INF] * 3, device="cuda"), min_p=0.5)
    w = [np.nonzero(kept_weights(row, 1.0, 0, 1.0, 0.5))[0] for row in z.double().numpy()]
    assert a.tolist() == [int(i[0]) for i in w] and b.tolist() == [int(i[-1]) for i in w]
    # one value a row: every token alike
    flat = torch.full((9, cols), -1.5, dtype=kind, device="cuda")
    at = torch.arange(9, device="cuda") * (cols // 9)
    tokens, logprobs = zbpe.draw_tokens(flat, ((at + 0.5) / cols).float())
    assert tokens.tolist() == at.tolist()
    np.testing.assert_allclose(logprobs.cpu().numpy(), -np.log(cols), rtol=2 * U, atol=0)


@gpu
@pytest.mark.parametrize("kind", TYPES)
def test_draw_masked_rows_infinities_and_nan(kind):
    z = torch.zeros(6, 1000, dtype=kind)
    z[0] = -INF                         # nothing
    z[1] = float("nan")                 # nothing either
    z[2] = -INF
    z[2, 77] = -5.0                     # one token
    z[3, [5, 9]] = INF                  # +inf holds all the weight
    z[4] = torch.finfo(kind).min        # the lowest value is a value like any other
    z[5, ::2] = float("nan")
    z[5, 1::2] = -INF
    z[5, 3] = torch.finfo(kind).min
    for kw in ({}, dict(temperature=0.5, top_k=3, top_p=0.9, min_p=0.1), dict(temperature=INF), dict(temperature=1e-38), dict(temperature=0.0)):
        kw = {k: torch.full((6,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda") for k, v in kw.items()}
        tokens, logprobs = zbpe.draw_tokens(z.cuda(), torch.full((6,), 0.75, device="cuda"), **kw)
        tokens, logprobs = tokens.tolist(), logprobs.tolist()
        assert tokens[:3] == [-1, -1, 77] and logprobs[:3] == [-INF, -INF, 0.0] and tokens[5] == 3
        greedy = "temperature" in kw and float(kw["temperature"][0]) == 0
        assert tokens[3] == (5 if greedy else 9) and tokens[4] == (0 if greedy else 2 if "top_k" in kw else 750)


@gpu
def test_draw_strides_axes_and_refusals():
    z, rng = draw_case(12, 700, 7, torch.bfloat16)
    u = torch.rand(12, generator=torch.Generator().manual_seed(2)).cuda()
    want = zbpe.draw_tokens(z.cuda(), u, temperature=0.7, top_k=50)
    wide = torch.zeros(3, 4, 800, dtype=torch.bfloat16, device="cuda")
    wide[..., 3:703] = z.view(3, 4, -1).cuda()
    got = zbpe.draw_tokens(wide[..., 3:703], u.view(3, 4), temperature=0.7, top_k=50)
    assert torch.equal(got[0].view(-1), want[0]) and torch.equal(got[1].view(-1), want[1])
    one = zbpe.draw_tokens(z[4].cuda(), u[4], temperature=0.7, top_k=50)
    assert one[0].shape == () and one[0] == want[0][4]
    none = zbpe.draw_tokens(z[:0].cuda(), u[:0])
    assert none[0].shape == (0,) and none[1].shape == (0,)
    for words, args, kw in (("shape", (z.cuda(), u[:11]), {}), ("not a tensor", (z.cuda(), 0.5), {}), ("float64", (z.cuda(), u.double()), {}),
                            ("on cpu", (z.cuda(), u.cpu()), {}), ("int64", (z.cuda(), u), {"top_k": torch.ones(12, dtype=torch.int64, device="cuda")}),
                            ("neither", (z.cuda(), u), {"top_p": "0.5"})):
        with pytest.raises(zbpe.InvalidArgument, match=words):
            zbpe.draw_tokens(*args, **kw)


# ---- log-probabilities ------------------------------------------------------------------------------------------------------------------


def logprobs_oracle(z, tokens, t=1.0):
    z = z.detach().double().numpy() / np.broadcast_to(np.asarray(t, np.float64).reshape(-1, 1), (z.shape[0], 1))
    top = z.max(1, keepdims=True)
    lse = np.log(np.exp(z - top).sum(1, keepdims=True)) + top
    tokens = tokens.numpy()
    y = np.take_along_axis(z, np.maximum(tokens, 0)[:, None], 1)[:, 0] - lse[:, 0]
    return np.where(tokens < 0, 0.0, y), np.exp(z - lse)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (5, 2), (9, 255), (65, 2048), (66, 2049), (3, 32001), (2, 65536), (2000, 300)])
def test_logprobs(rows, cols, kind):
    """The sum of exponentials: each is off by the roundings of its argument d (5 U |d|, and the mean of |d| under the softmax is
    at most log V < 12), by 2 U of its own, and by those of at most 300 additions; the result's own roundings are 8 U |y|."""
    rng = np.random.default_rng(rows + cols)
    z = torch.from_numpy(rng.standard_normal((rows, cols)) * 4).to(kind)
    tokens = torch.from_numpy(rng.integers(0, cols, rows))
    if rows > 3:
        tokens[1] = -1
        tokens[2] = -100
    t = torch.from_numpy(np.float32(0.5 + rng.random(rows)))
    up = torch.from_numpy(rng.standard_normal(rows)).float()
    relative, least = half_step(kind)
    for temperature in (None, t):
        inverse = 1.0 if temperature is None else (1 / t.double()).numpy()
        y, p = logprobs_oracle(z, tokens, 1.0 if temperature is None else t)
        for ids in (tokens, tokens.int()):
            zg = z.cuda().requires_grad_()
            kw = {} if temperature is None else {"temperature": t.cuda()}
            plain = zbpe.token_logprobs(zg.detach(), ids.cuda(), **kw)
            close(plain, y, U * (370 + 8 * np.abs(y)))
            out = zbpe.token_logprobs(zg, ids.cuda(), **kw)
            assert torch.equal(out.detach(), plain)
            got, = torch.autograd.grad(out, zg, up.cuda())
            hot = np.zeros((rows, cols))
            hot[np.arange(rows), np.maximum(tokens.numpy(), 0)] = 1
            g = np.where(tokens.numpy() < 0, 0.0, up.double().numpy() * inverse)[:, None]
            want = g * (hot - p)
            # p's relative error as above, with |d| of this element; g's own 2 U; then one rounding to the type
            off = np.abs(g) * U * (p * (370 + 8 * np.abs(np.log(np.maximum(p, 1e-300)))) + 4 * hot)
            assert got.dtype == kind
            close(got, want, off + (np.abs(want) + off) * relative + least + np.abs(g) * 2.0 ** -126)


@gpu
def test_logprobs_extremes():
    nan = float("nan")
    z = torch.zeros(8, 600)
    z[0] = -INF
    z[1] = -INF
    z[1, 7] = 3.0
    z[2] = torch.finfo(torch.float32).min
    z[3, 5] = INF
    z[4, 5] = nan
    z[5] = 3e38
    z[6, 1] = -INF
    tokens = torch.tensor([3, 7, 9, 5, 8, 1, 1, 600])
    zg = z.cuda().requires_grad_()
    y = zbpe.token_logprobs(zg, tokens.cuda())
    got = y.tolist()
    assert got[0] == -INF and got[1] == 0 and got[6] == -INF
    assert abs(got[2] + np.log(600)) < 400 * U and abs(got[5] + np.log(600)) < 400 * U
    assert np.isnan(got[3]) and np.isnan(got[4]) and np.isnan(got[7])
    d, = torch.autograd.grad(y, zg, torch.ones(8, device="cuda"))
    assert (d[0] == 0).all() and (d[1] == 0).all() and d[7].isnan().all() and d[4].isnan().any()
    assert d[6, 1] == 1 and (d[6, 2:] < 0).all()
    empty = zbpe.token_logprobs(z[:0].cuda(), tokens[:0].cuda())
    assert empty.shape == (0,)
    zero = torch.zeros(0, 600, device="cuda", requires_grad=True)
    assert torch.autograd.grad(zbpe.token_logprobs(zero, tokens[:0].cuda()).sum(), zero)[0].shape == (0, 600)


@gpu
def test_logprobs_of_a_language_models_batch():
    """[batch, time, V] logits cut to predict the next token, against torch's own in 64 bits, weighted by a broadcast gradient;
    and what a text costs in bits a byte"""
    rng = np.random.default_rng(4)
    merges = some_merges(400, rng, np.arange(97, 110))
    v = zbpe.Vocabulary(np.array(merges), 400)
    z = torch.from_numpy(rng.standard_normal((3, 9, 400))).float().cuda().requires_grad_()
    ids = torch.from_numpy(rng.integers(0, 400, (3, 9))).cuda()
    ids[1, 5:] = -1
    y = zbpe.token_logprobs(z[:, :-1], ids[:, 1:])
    z64 = z.detach().double().requires_grad_()
    scored = ids[:, 1:] >= 0
    want = z64[:, :-1].log_softmax(-1).gather(-1, ids[:, 1:].clamp(min=0)[..., None])[..., 0] * scored
    # values and gradients below 16, sums of 400: 370 + 8 * 16 roundings
    np.testing.assert_allclose(y.detach().cpu().numpy(), want.detach().cpu().numpy(), rtol=0, atol=500 * U)
    got, = torch.autograd.grad(y.sum(), z)
    ref, = torch.autograd.grad(want.sum(), z64)
    np.testing.assert_allclose(got.cpu().numpy(), ref.cpu().numpy(), rtol=0, atol=500 * U)
    tokens = tokens_of(merges, 400)
    n = sum(len(tokens[i]) for i in ids[:, 1:].flatten().tolist() if i >= 0)
    bits = v.bits_per_byte(z[:, :-1], ids[:, 1:])
    np.testing.assert_allclose(float(bits.detach()), float(-want.detach().sum() / np.log(2) / n), rtol=500 * U)
    torch.autograd.grad(bits, z)
    for words, args, kw in (("shape", (z, ids[:, 1:]), {}), ("float32", (z, z[..., 0]), {}), ("on cpu", (z, ids.cpu()), {}),
                            ("detach", (z, ids), {"temperature": torch.ones(3, 9, device="cuda", requires_grad=True)})):
        with pytest.raises(zbpe.InvalidArgument, match=words):
            zbpe.token_logprobs(*args, **kw)


# ---- together ---------------------------------------------------------------------------------------------------------------------------


def number_list():
    """[1,23,456]: a list of numbers without leading zeros"""
    table = np.full((6, 256), -1, np.int32)
    digits, first = np.arange(48, 58), np.arange(49, 58)
    table[0, ord("[")] = 1
    for s in (1, 4):           # 1: after "[", 4: after ","
        table[s, first] = 2
        table[s, 48] = 3
    table[1, ord("]")] = 5
    table[2, digits] = 2       # 2: inside a number, 3: behind a 0
    for s in (2, 3):
        table[s, ord(",")] = 4
        table[s, ord("]")] = 5
    return table, np.arange(6) == 5


@gpu
def test_tokenizer_answers_under_a_grammar(engine):
    """train, then decode a batch step by step under a grammar with everything on: every answer is of the grammar's language, the
    log-probabilities are those of token_logprobs of the adjusted logits, and the prompt's cost in bits a byte is finite"""
    import re

    tok = zbpe.BasicTokenizer(engine=engine)
    tok.train(b"[1,20,300,4] [10,200,31] [100,2000] " * 40 + c1_text()[:4000], 400)
    size = 401  # one more id ends an answer
    table, accepting = number_list()
    grammar = tok.grammar(table, accepting, vocabSize=size, endToken=400)
    rows, steps = 33, 24
    gen = torch.Generator(device="cuda").manual_seed(0)
    states = torch.zeros(rows, dtype=torch.int32, device="cuda")
    history = torch.full((rows, steps), -1, dtype=torch.int32, device="cuda")
    allowed = grammar.masks()
    for step in range(steps):
        z = torch.randn(rows, size, generator=gen, device="cuda", dtype=torch.float32).bfloat16()
        z[:, 400] += 2
        u = torch.rand(rows, generator=gen, device="cuda")
        lengths = torch.full((rows,), step, dtype=torch.int32, device="cuda")
        terms = dict(history=history, lengths=lengths, repetition=1.2, frequency=0.1, presence=0.1)
        tokens, logprobs, after = tok.nextTokens(z, u, grammar=grammar, states=states, temperature=0.9, **terms)
        adjusted = zbpe.adjust_logits(z, masks=allowed, states=states, **terms)
        again = zbpe.token_logprobs(adjusted, tokens, temperature=0.9)
        # the scores' own error (370 + 8 |y| roundings, |y| < 32)
        np.testing.assert_allclose(logprobs.cpu().numpy(), again.cpu().numpy(), rtol=0, atol=626 * U)
        done = history[:, :step].eq(400).any(1)
        tokens = torch.where(done, 400, tokens)
        states = torch.where(done, states, after)
        assert (states >= 0).all()
        history[:, step] = tokens
    whole = 0
    for row in history.tolist():
        end = row.index(400) if 400 in row else len(row)
        text = tok.decode(row[:end]).decode()
        if end < len(row):
            whole += 1
            assert re.fullmatch(r"\[((0|[1-9][0-9]*)(,(0|[1-9][0-9]*))*)?\]", text), text
        else:
            assert re.match(r"\[[0-9,]*$", text), text
    assert whole
    ids = torch.tensor(tok.encode(b"[1,20,300]")).cuda()
    cost = tok.bitsPerByte(torch.zeros(len(ids), size, device="cuda"), ids)
    np.testing.assert_allclose(float(cost), len(ids) * np.log2(size) / 10, rtol=400 * U)
    free, logprob, none = tok.nextTokens(torch.zeros(2, size, device="cuda"), torch.zeros(2, device="cuda"))
    assert none is None and free.tolist() == [0, 0]
    for kw in (dict(grammar=grammar), dict(states=states), dict(grammar=grammar, states=states, masks=allowed)):
        with pytest.raises(zbpe.InvalidArgument):
            tok.nextTokens(torch.zeros(rows, size, device="cuda"), torch.zeros(rows, device="cuda"), **kw)


def step_inputs(seed, rows=5, size=900):
    rng = np.random.default_rng(seed)
    return (torch.from_numpy(rng.standard_normal((rows, size))).to(torch.bfloat16).cuda(), torch.from_numpy(rng.random(rows)).float().cuda(),
            torch.from_numpy(rng.integers(-1, 7, rows)).int().cuda(), torch.from_numpy(rng.integers(0, size, (rows, 50))).int().cuda())


@gpu
def test_a_captured_step_replays():
    """grammar, penalties, draw and scores captured into one graph; replayed on new inputs, with eager work between the replays"""
    rng = np.random.default_rng(6)
    merges = some_merges(900, rng, ALPHABET)
    table, accepting = some_automaton(7, rng, ALPHABET)
    grammar = zbpe.Grammar(zbpe.Vocabulary(np.array(merges), 900, 0), cuda(table), cuda(accepting))

    def step(z, u, s, h):
        masks = grammar.masks(s)
        y = zbpe.adjust_logits(z, history=h, repetition=1.3, frequency=0.2, masks=masks)
        tokens, logprobs = zbpe.draw_tokens(y, u, temperature=0.8, top_k=40, top_p=0.9)
        return masks, y, tokens, logprobs, grammar.advance(s, tokens), zbpe.token_logprobs(z, tokens)

    held = step_inputs(0)
    step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*held)
    for seed in range(1, 5):
        new = step_inputs(seed)
        want = step(*new)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)


@gpu
def test_captured_gradients_replay():
    z, x = adjust_case(40, 500, 3)
    g = to_gpu(x)
    tokens = torch.randint(0, 500, (40,), device="cuda")
    z = z.cuda().requires_grad_()
    g["bias"].requires_grad_()
    g["bias_values"].requires_grad_()
    del g["masks"], g["states"]

    def step():
        y = zbpe.token_logprobs(zbpe.adjust_logits(z, **g), tokens)
        return torch.autograd.grad(y, [z, g["bias"], g["bias_values"]], torch.ones_like(y))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        with torch.no_grad():
            z.add_(torch.randn_like(z))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@gpu
def test_streams_and_repeats():
    """two streams at once, each on its own inputs, give what one gives; the same call twice gives the same bits"""
    z, x = adjust_case(64, 9000, 12, kind=torch.bfloat16)
    g = to_gpu(x)
    z = z.cuda().requires_grad_()
    g["bias"].requires_grad_()
    u = torch.rand(64, device="cuda")

    def all_of():
        y = zbpe.adjust_logits(z, **g)
        lp = zbpe.token_logprobs(z, torch.zeros(64, dtype=torch.int64, device="cuda"))
        return [y.detach(), *zbpe.draw_tokens(y, u, top_p=0.9, top_k=100), lp.detach(),
                *torch.autograd.grad([y, lp], [z, g["bias"]], [torch.ones_like(y), torch.ones_like(lp)])]

    want = all_of()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(all_of())
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(r, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@gpu
def test_offsets_past_32_bits():
    """rows that start behind 2^31 elements"""
    rows, cols = 33000, 65536
    z = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    at = torch.arange(rows, device="cuda") * 7919 % cols
    z[torch.arange(rows, device="cuda"), at] = 20.0
    tokens, _ = zbpe.draw_tokens(z, torch.full((rows,), 0.5, device="cuda"), top_k=1)
    assert torch.equal(tokens.long(), at)
    want = -np.log1p((cols - 1) * np.exp(-20.0))
    y = zbpe.token_logprobs(z, at)
    assert float((y.double() - want).abs().max()) < 370 * U
    zbpe.adjust_logits(z, history=at.int()[:, None], presence=19.0, out=z)
    assert bool((z.gather(1, at[:, None]) == 1).all()) and bool((z[-1].sum() == 1))
    z.requires_grad_()
    d, = torch.autograd.grad(zbpe.token_logprobs(z, at), z, torch.ones(rows, device="cuda"))
    got = d.gather(1, at[:, None])[:, 0].double()
    want = 1 - np.e / (np.e + cols - 1)
    assert float((got - want).abs().max()) < 2.0 ** -11 + 370 * U
