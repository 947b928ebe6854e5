"""The operators between a model's logits over a byte-pair vocabulary and its tokens, on torch tensors.

  Vocabulary, Grammar   which tokens an automaton over bytes allows, as one bit a token; the automaton's step by a token
  adjust_logits         penalties for repeated tokens, biases and masks on logits, with gradients
  draw_tokens           temperature, top-k, top-p, min-p, and one token a row by a given uniform number
  token_logprobs        log-probabilities of given tokens, with the gradient

They run on libzbpe.so's kernels (include/zbpe.h states each one's definition), on the tensors' device and its current
stream, wait for nothing and can be captured into a HIP graph. Logits are float32, float16 or bfloat16 with any number of
leading axes, ``[..., V]`` with V up to 65536; a per-row tensor has the leading axes' shape, and a plain number stands for
all rows (a whole one for an int32 tensor). Tensors of the wrong type, shape or device raise InvalidArgument before anything is launched. Results of a captured
call are those of the eager one, bit for bit; no result depends on the order in which workgroups run. A backward pass is captured
as any of torch's: warmed up on a side stream, and while no eager graph of the same leaves is alive (torch ties a leaf's gradient
to the stream that first used it).
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _STATUS, InternalError, InvalidArgument, Merges, ZbpeError, _ptr, load_library, vocabStart

MAX_VOCAB = 65536
_FLOATS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INTS = {torch.int32: 3, torch.int64: 4}
_KINDS = {**_FLOATS, **_INTS}

# include/zbpe.h's structures, field by field ("@": native alignment, as a C compiler lays them out)
_ROWS = "Pqqi0q"
_GRAMMAR = struct.Struct("@PPiiPPiP")
_ADJUST = struct.Struct("@Iiqq" + 3 * _ROWS + "qPPPPPPPPiiPqP")
_DRAW = struct.Struct("@Iiqq" + _ROWS + "PPPPPPP")
_LOGPROBS = struct.Struct("@Iiqq" + _ROWS + "PiPPP")
_MATRIX = struct.Struct("@" + _ROWS)
_NO_ROWS = (0, 0, 0, 0)

_checked = None


def _library() -> ctypes.CDLL:
    global _checked
    if _checked is None:
        L = load_library()
        for which, layout in enumerate((_ADJUST, _DRAW, _LOGPROBS, _GRAMMAR)):
            if L.zbpe_struct_size(which) != layout.size:
                raise ImportError(f"structure {which} of the library is {L.zbpe_struct_size(which)} B, this binding's is {layout.size} B")
        _checked = L
    return _checked


def _check(status: int) -> None:
    if status:
        raise _STATUS.get(status, ZbpeError)(_library().zbpe_last_error(None).decode())


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)  # (what torch.cuda.current_stream wraps in two objects)


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise InvalidArgument(message)


# (Checks on the way of every call make their messages only when they fail.)


def _is_tensor(x, name: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise InvalidArgument(f"{name} is not a tensor")


def _no_gradient(**named) -> None:
    for name, x in named.items():
        if isinstance(x, torch.Tensor) and x.requires_grad:
            raise InvalidArgument(f"{name} has no gradient here: detach it")


def _no_tangent(**named) -> None:
    """No operator here has a forward-mode derivative. (A tensor with a tangent does not require a gradient, so that torch's own
    refusal is not reached; and no_grad does not switch tangents off.)"""
    if not torch._C._is_fwd_grad_enabled():
        return
    for name, x in named.items():
        if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise InvalidArgument(f"{name} has a tangent, and there is no forward-mode derivative here: detach it")


def _written(out: torch.Tensor) -> None:
    """A caller's tensor was written by its pointer: torch is told, so that a backward pass that needs what stood there raises."""
    torch.autograd.graph.increment_version(out)


class _Rows:
    """How the rows of one call are numbered: by the logits' leading axes, in two levels."""

    __slots__ = ("lead", "cols", "inner", "rows", "device", "index")

    def __init__(self, logits: torch.Tensor, name: str = "logits"):
        _is_tensor(logits, name)
        if logits.dtype not in _FLOATS:
            raise InvalidArgument(f"{name} is {logits.dtype} (float32, float16 or bfloat16)")
        if not (logits.dim() >= 1):
            raise InvalidArgument(f"{name} has no axis of columns")
        self.lead, self.cols = logits.shape[:-1], logits.shape[-1]
        if not (1 <= self.cols <= MAX_VOCAB):
            raise InvalidArgument(f"{name} has {self.cols} columns (1 to {MAX_VOCAB})")
        if not (logits.is_cuda):
            raise InvalidArgument(f"{name} is on {logits.device}, not on a GPU")
        self.device = logits.device
        self.index = self.device.index
        self.rows = self.lead.numel()
        self.inner = max(self.lead[-1], 1) if self.lead else 1

    def matrix(self, t: torch.Tensor, keep: list):
        """(pointer, outer stride, inner stride, dtype) of a [*lead, n] tensor, copied only when two strides do not say it."""
        n = t.shape[-1]
        if t.is_contiguous():
            return (t.data_ptr(), self.inner * n, n, _KINDS.get(t.dtype, 0))
        if t.dim() == 2 and t.stride(1) == 1 and t.numel():
            step = t.stride(0)
            return (t.data_ptr(), self.inner * step, step, _KINDS.get(t.dtype, 0))
        if t.dim() != 3:
            try:
                t = t.view(-1, self.inner, n) if t.numel() else t
            except RuntimeError:
                t = t.contiguous().view(-1, self.inner, n)
        if t.numel() and n > 1 and t.stride(-1) != 1:
            t = t.contiguous()
        keep.append(t)
        kind = _KINDS.get(t.dtype, 0)
        if not t.numel():
            return (t.data_ptr(), n, n, kind)
        return (t.data_ptr(), t.stride(0), t.stride(1), kind)

    def on(self, t: torch.Tensor, name: str) -> None:
        _is_tensor(t, name)
        if t.get_device() != self.index:
            raise InvalidArgument(f"{name} is on {t.device}, the logits are on {self.device}")

    def per_row(self, x, name: str, dtype: torch.dtype, keep: list) -> int:
        """Pointer of one value a row; a number stands for all rows, None for the default."""
        if x is None:
            return 0
        if not isinstance(x, torch.Tensor):
            if not isinstance(x, (int, float)):
                raise InvalidArgument(f"{name} is neither a tensor nor a number")
            if dtype == torch.int32:
                if not (-(2 ** 31) <= x < 2 ** 31 and x == int(x)):
                    raise InvalidArgument(f"{name} is {x}, not a whole number of 32 bits")
            elif abs(x) > 3.4e38:  # (rounded to 32 bits as a tensor's values are: infinite from half a step past the largest)
                x = ctypes.c_float(min(max(x, -1e39), 1e39)).value
            x = torch.full(self.lead, x, dtype=dtype, device=self.device)
        elif x.dtype == dtype and x.shape == self.lead and x.get_device() == self.index and x.is_contiguous():
            return x.data_ptr()  # (the usual case; the caller holds it)
        self.on(x, name)
        if x.dtype != dtype:
            raise InvalidArgument(f"{name} is {x.dtype} ({dtype})")
        if x.shape != self.lead:
            raise InvalidArgument(f"{name} has shape {tuple(x.shape)}, the rows are {tuple(self.lead)}")
        x = x.contiguous()
        keep.append(x)
        return x.data_ptr()

    def tokens(self, x: torch.Tensor, name: str, keep: list):
        self.on(x, name)
        if x.dtype not in _INTS:
            raise InvalidArgument(f"{name} is {x.dtype} (int32 or int64)")
        if x.shape != self.lead:
            raise InvalidArgument(f"{name} has shape {tuple(x.shape)}, the rows are {tuple(self.lead)}")
        x = x.contiguous()
        keep.append(x)
        return x.data_ptr(), _INTS[x.dtype]


# ---- grammars ------------------------------------------------------------------------------------------------------------


def _triples(merges) -> np.ndarray:
    if isinstance(merges, Merges):
        merges = merges.as_array()
    a = np.asarray(merges)
    _need(a.size == 0 or (a.dtype.kind in "iu" and a.size % 3 == 0), "merges are triples of whole numbers: first, second, new token")
    _need(a.ndim < 2 or a.shape[-1] == 3 or a.size == 0, "merges are triples of whole numbers: first, second, new token")
    _need(a.size == 0 or (a.min() >= 0 and a.max() <= 0xFFFF), "a merge's token is outside 0 .. 65535")
    return np.ascontiguousarray(a.reshape(-1, 3), dtype=np.uint16)


def token_bytes(merges, vocab_size: Optional[int] = None):
    """The bytes of every token, as decode gives them: (offsets uint32 [vocab_size + 1], bytes uint8). A token that no merge
    makes has none. vocab_size: up to the largest token when not given. Host only."""
    a = _triples(merges)
    if vocab_size is None:
        vocab_size = max(vocabStart, int(a[:, 2].max()) + 1 if len(a) else 0)
    if not (isinstance(vocab_size, (int, np.integer)) and vocabStart <= vocab_size <= MAX_VOCAB):
        raise InvalidArgument(f"vocab_size is {vocab_size} ({vocabStart} to {MAX_VOCAB})")
    L = _library()
    triples = a if len(a) else np.zeros(3, np.uint16)
    offsets, n = np.zeros(vocab_size + 1, np.uint32), ctypes.c_size_t(0)
    _check(L.zbpe_vocab_bytes(_ptr(triples), len(a), vocab_size, _ptr(offsets), None, 0, ctypes.byref(n)))
    data = np.zeros(n.value, np.uint8)
    _check(L.zbpe_vocab_bytes(_ptr(triples), len(a), vocab_size, _ptr(offsets), _ptr(data), n.value, ctypes.byref(n)))
    return offsets, data


class Vocabulary:
    """The tokens of a merge table, laid out on a device once for all grammars over them.

    merges: Merges, or triples (first, second, new token) as Engine.train returns them. vocab_size: how many ids the model has;
    those that no merge makes are never allowed. end_token: the id that ends an answer, allowed in accepting states alone."""

    def __init__(self, merges, vocab_size: Optional[int] = None, end_token: Optional[int] = None, device=None):
        offsets, data = token_bytes(merges, vocab_size)
        self.size = len(offsets) - 1
        self.end_token = -1 if end_token is None else int(end_token)
        if not (end_token is None or 0 <= self.end_token < self.size):
            raise InvalidArgument(f"end_token is {end_token}, the vocabulary has {self.size} tokens")
        self.words = (self.size + 31) // 32
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.offsets = torch.from_numpy(offsets.view(np.int32)).to(self.device)
        self.bytes = torch.from_numpy(data).to(self.device)
        L = _library()
        index = np.empty(L.zbpe_vocab_index_size(self.size), np.uint8)
        _check(L.zbpe_vocab_index(_ptr(offsets), _ptr(data), self.size, _ptr(index)))
        self.index = torch.from_numpy(index).to(self.device)

    def lengths(self) -> torch.Tensor:
        """Bytes of each token, int32 [size]; 0 where it has none."""
        return self.offsets[1:] - self.offsets[:-1]

    def bits_per_byte(self, logits: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        """What a text costs under a model, in bits for each of its bytes: comparable between vocabularies, as a loss per token
        is not. logits [..., V] predict tokens [...]; negative tokens (padding) count for nothing. A 0-d float32 tensor, with a
        gradient with respect to the logits. A token past the vocabulary makes it NaN. (Its sums are torch's, which a captured
        graph does not replay safely: call it outside of one.)"""
        _is_tensor(logits, "logits")
        if logits.device != self.device:
            raise InvalidArgument(f"logits are on {logits.device}, the vocabulary is on {self.device}")
        nats = token_logprobs(logits, tokens)
        known = (tokens >= 0) & (tokens < self.size)
        n = torch.where(known, self.lengths()[torch.where(known, tokens, 0).long()], 0).sum()
        wrong = torch.where(tokens < self.size, 0.0, torch.nan).sum()
        return (nats.double().sum() / (n.double() * -np.log(2.0)) + wrong).float()


class Grammar:
    """An automaton over bytes, read by whole tokens.

    next: int32 [states, 256], the state after each byte; any value that is no state (-1) refuses it. accepting: bool [states],
    where an answer may end (none when not given)."""

    def __init__(self, vocabulary: Vocabulary, next, accepting=None):
        _need(isinstance(vocabulary, Vocabulary), "vocabulary is not a Vocabulary")
        device = vocabulary.device
        if device.type != "cuda":
            raise InvalidArgument(f"vocabulary is on {device}, not on a GPU")
        next = torch.as_tensor(next)
        if not (next.dim() == 2 and next.shape[1] == 256):
            raise InvalidArgument(f"next has shape {tuple(next.shape)} (states, 256)")
        n = next.shape[0]
        if not (n < 1 << 23):
            raise InvalidArgument(f"{n} states (fewer than 2^23)")
        if next.is_floating_point() or next.is_complex() or next.dtype == torch.bool:
            raise InvalidArgument(f"next is {next.dtype} (whole numbers)")
        if next.dtype != torch.int32:
            next = torch.where((next < 0) | (next >= n), -1, next).to(torch.int32)
        self.next = next.to(device).contiguous()
        self.accepting = None
        if accepting is not None:
            accepting = torch.as_tensor(accepting)
            if not (accepting.dtype in (torch.bool, torch.uint8)):
                raise InvalidArgument(f"accepting is {accepting.dtype} (bool)")
            if accepting.shape != (n,):
                raise InvalidArgument(f"accepting has shape {tuple(accepting.shape)}, there are {n} states")
            self.accepting = accepting.to(device).contiguous()
        self.vocabulary, self.states = vocabulary, n

    def _packed(self) -> bytes:
        v = self.vocabulary
        return _GRAMMAR.pack(v.offsets.data_ptr(), v.bytes.data_ptr(), v.size, v.end_token, self.next.data_ptr(),
                             0 if self.accepting is None else self.accepting.data_ptr(), self.states, v.index.data_ptr())

    def _vector(self, x: torch.Tensor, name: str) -> torch.Tensor:
        _is_tensor(x, name)
        if x.device != self.next.device:
            raise InvalidArgument(f"{name} is on {x.device}, the grammar is on {self.next.device}")
        if x.dtype != torch.int32:
            raise InvalidArgument(f"{name} is {x.dtype} (int32)")
        return x.contiguous()

    def masks(self, states: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """int32 [..., words]: bit v % 32 of word v / 32 says whether token v may follow, for each of `states` (int32), or for
        every state of the automaton in order. In a state outside the automaton nothing may."""
        device = self.next.device
        if states is not None:
            states = self._vector(states, "states")
        lead = (self.states,) if states is None else states.shape
        shape = (*lead, self.vocabulary.words)
        written = out is not None
        if out is None:
            out = torch.empty(shape, dtype=torch.int32, device=device)
        else:
            _is_tensor(out, "out")
            if not (out.dtype == torch.int32 and out.shape == shape and out.device == device and out.is_contiguous()):
                raise InvalidArgument(f"out is not a packed int32 tensor of shape {tuple(shape)} on {device}")
        rows = self.states if states is None else states.numel()
        _check(_library().zbpe_grammar_masks(device.index, _stream(device), self._packed(),
                                             None if states is None else states.data_ptr(), rows, out.data_ptr()))
        if written:
            _written(out)
        return out

    def advance(self, states: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        """The states after `tokens` (int32 both, of one shape): -1 where the grammar refuses the token. A negative token
        leaves its state as it is."""
        states, tokens = self._vector(states, "states"), self._vector(tokens, "tokens")
        if states.shape != tokens.shape:
            raise InvalidArgument(f"states have shape {tuple(states.shape)}, tokens {tuple(tokens.shape)}")
        out = torch.empty_like(states)
        device = self.next.device
        _check(_library().zbpe_grammar_advance(device.index, _stream(device), self._packed(), states.data_ptr(), tokens.data_ptr(),
                                               states.numel(), out.data_ptr()))
        return out


# ---- penalties, biases and masks --------------------------------------------------------------------------------------------


class _Terms(NamedTuple):
    """The arguments of adjust_logits besides the logits, as given."""

    history: Optional[torch.Tensor]
    lengths: Optional[torch.Tensor]
    prompt_lengths: Optional[torch.Tensor]
    repetition: object
    presence: object
    frequency: object
    bias: Optional[torch.Tensor]
    bias_tokens: Optional[torch.Tensor]
    bias_values: Optional[torch.Tensor]
    masks: Optional[torch.Tensor]
    states: Optional[torch.Tensor]


def _pack_adjust(at: _Rows, logits: torch.Tensor, out: torch.Tensor, x: _Terms, keep: list) -> bytes:
    history, length = _NO_ROWS, 0
    if x.history is not None:
        at.on(x.history, "history")
        if x.history.dtype not in _INTS:
            raise InvalidArgument(f"history is {x.history.dtype} (int32 or int64)")
        if not (x.history.shape[:-1] == at.lead and x.history.dim() == len(at.lead) + 1):
            raise InvalidArgument(f"history has shape {tuple(x.history.shape)}, the rows are {tuple(at.lead)}")
        length = x.history.shape[-1]
        history = at.matrix(x.history, keep)
    else:
        for name in ("lengths", "prompt_lengths", "repetition", "presence", "frequency"):
            if getattr(x, name) is not None:
                raise InvalidArgument(f"{name} without a history")
    bias = 0
    if x.bias is not None:
        at.on(x.bias, "bias")
        if not (x.bias.dtype == torch.float32 and x.bias.shape == (at.cols,)):
            raise InvalidArgument(f"bias is not float32 of {at.cols} values")
        t = x.bias.contiguous()
        keep.append(t)
        bias = t.data_ptr()
    n_biases, bias_tokens, bias_values = 0, 0, 0
    _need((x.bias_tokens is None) == (x.bias_values is None), "bias_tokens go with bias_values")
    if x.bias_tokens is not None:
        for name, kind in (("bias_tokens", torch.int32), ("bias_values", torch.float32)):
            t = getattr(x, name)
            at.on(t, name)
            if t.dtype != kind:
                raise InvalidArgument(f"{name} is {t.dtype} ({kind})")
            if not (t.dim() == len(at.lead) + 1 and t.shape[:-1] == at.lead):
                raise InvalidArgument(f"{name} has shape {tuple(t.shape)}, the rows are {tuple(at.lead)}")
        n_biases = x.bias_tokens.shape[-1]
        _need(x.bias_values.shape == x.bias_tokens.shape, "bias_tokens and bias_values have different shapes")
        t, v = x.bias_tokens.contiguous(), x.bias_values.contiguous()
        keep += [t, v]
        bias_tokens, bias_values = t.data_ptr(), v.data_ptr()
    masks, mask_words, mask_rows, states = 0, 0, 0, 0
    if x.masks is not None:
        at.on(x.masks, "masks")
        if x.masks.dtype != torch.int32:
            raise InvalidArgument(f"masks are {x.masks.dtype} (int32)")
        if not (x.masks.dim() >= 1 and x.masks.shape[-1] >= (at.cols + 31) // 32):
            raise InvalidArgument(f"masks of shape {tuple(x.masks.shape)} are too narrow for {at.cols} columns")
        if not (x.masks.numel() > 0 or at.rows == 0):
            raise InvalidArgument(f"masks of shape {tuple(x.masks.shape)} have no rows")
        t = x.masks.contiguous()
        keep.append(t)
        masks, mask_words, mask_rows = t.data_ptr(), t.shape[-1], t.shape[:-1].numel()
        if x.states is None:
            if not (t.shape[:-1] == at.lead or mask_rows == 1):
                raise InvalidArgument(f"masks of shape {tuple(t.shape)}, the rows are {tuple(at.lead)}")
        else:
            states = at.per_row(x.states, "states", torch.int32, keep)
    else:
        _need(x.states is None, "states without masks")
    f32, i32 = torch.float32, torch.int32
    return _ADJUST.pack(
        _ADJUST.size, at.cols, at.rows, at.inner, *at.matrix(logits, keep), *at.matrix(out, keep), *history, length,
        at.per_row(x.lengths, "lengths", i32, keep), at.per_row(x.prompt_lengths, "prompt_lengths", i32, keep),
        at.per_row(x.repetition, "repetition", f32, keep), at.per_row(x.presence, "presence", f32, keep),
        at.per_row(x.frequency, "frequency", f32, keep), bias, bias_tokens, bias_values, n_biases, mask_words, masks, mask_rows, states)


def _adjust(logits: torch.Tensor, out: torch.Tensor, x: _Terms) -> torch.Tensor:
    at, keep = _Rows(logits), []
    args = _pack_adjust(at, logits, out, x, keep)
    _check(_library().zbpe_adjust_logits(at.device.index, _stream(at.device), args))
    return out


class _Adjust(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, bias_values, x: _Terms, dtype):
        out = torch.empty(logits.shape, dtype=dtype, device=logits.device)
        x = x._replace(bias=bias, bias_values=bias_values)
        _adjust(logits, out, x)
        tensors = [t if isinstance(t, torch.Tensor) else None for t in x]
        ctx.numbers = [None if isinstance(t, torch.Tensor) else t for t in x]
        ctx.save_for_backward(logits, *tensors)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        logits, *tensors = ctx.saved_tensors
        x = _Terms(*[n if t is None else t for t, n in zip(tensors, ctx.numbers)])
        at, keep = _Rows(logits), []
        args = _pack_adjust(at, logits, grad, x, keep)
        wants = ctx.needs_input_grad
        d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if wants[0] else None
        d_bias = torch.empty_like(x.bias, memory_format=torch.contiguous_format) if wants[1] else None
        d_values = torch.empty_like(x.bias_values, memory_format=torch.contiguous_format) if wants[2] else None
        L = _library()
        space = L.zbpe_adjust_workspace(at.rows, at.cols) if wants[1] else 0
        workspace = torch.empty(space, dtype=torch.uint8, device=at.device) if space else None
        rows = None if d_logits is None else _MATRIX.pack(*at.matrix(d_logits, keep))
        _check(L.zbpe_adjust_logits_grad(at.device.index, _stream(at.device), args, rows, 0 if d_bias is None else d_bias.data_ptr(),
                                         0 if d_values is None else d_values.data_ptr(), 0 if workspace is None else workspace.data_ptr(), space))
        return d_logits, d_bias, d_values, None, None


def adjust_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                  prompt_lengths: Optional[torch.Tensor] = None, repetition=None, presence=None, frequency=None,
                  bias: Optional[torch.Tensor] = None, bias_tokens: Optional[torch.Tensor] = None,
                  bias_values: Optional[torch.Tensor] = None, masks: Optional[torch.Tensor] = None,
                  states: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits with penalties for the row's earlier tokens, biases and a mask, in the logits' type. In this order:

      repetition      a logit whose token is in the row's history: z / repetition where z > 0, else z * repetition
      frequency       minus frequency * how often the token is in the history behind the prompt
      presence        minus presence when it is there at all
      bias            float32 [V], for all rows
      bias_values     float32 [..., n] (n up to 1024), each added to the row's token bias_tokens (int32 [..., n])
      masks           int32 [m, words] (Grammar.masks): -inf where the row's bit is 0. states (int32 [...]) names each row's
                      row of masks, outside 0 .. m - 1: nothing is allowed; without it, one row for all or one for each

    history: int32 or int64 [..., n]; lengths and prompt_lengths (int32 [...]): how many of a row's tokens count, and how
    many of these are the prompt's. History and bias tokens outside 0 .. V - 1 are passed over.

    Gradients go to logits, bias and bias_values; tangents (forward mode) are refused. out: where to write (the logits' type or
    float32; it may be the logits themselves, and otherwise shares no memory with them or another argument), without gradients."""
    x = _Terms(history, lengths, prompt_lengths, repetition, presence, frequency, bias, bias_tokens, bias_values, masks, states)
    _is_tensor(logits, "logits")
    learns = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (logits, bias, bias_values))
    if torch.is_grad_enabled():
        _no_gradient(repetition=repetition, presence=presence, frequency=frequency)
    if forward_ad._current_level >= 0:  # (otherwise no tensor has one)
        _no_tangent(logits=logits, bias=bias, bias_values=bias_values, repetition=repetition, presence=presence, frequency=frequency,
                    out=out)
    if out is not None:
        _is_tensor(out, "out")
        _need(not learns and not (out.requires_grad and torch.is_grad_enabled()), "out goes without gradients")
        if not (out.shape == logits.shape and out.device == logits.device and out.dtype in (logits.dtype, torch.float32)):
            raise InvalidArgument(f"out is not {logits.dtype} or float32 of shape {tuple(logits.shape)} on {logits.device}")
        _need(_Rows(logits).matrix(out, [])[0] == out.data_ptr(), "out has strides that its rows cannot be written by")
        _adjust(logits, out, x)
        _written(out)
        return out
    if learns:
        return _Adjust.apply(logits, bias, bias_values, x, logits.dtype)
    return _adjust(logits, torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), x)


# ---- the draw ---------------------------------------------------------------------------------------------------------------


def draw_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token a row: (tokens int32 [...], logprobs float32 [...], the drawn token's among the kept ones).

    Tokens are weighed by exp(z / temperature) and ranked by z, larger first, then by id. top_k keeps the first ranks (0 or
    less: all), top_p of these the first whose predecessors hold less than this share of their sum, min_p of these the
    ones with at least this share of the largest weight. The token is the first, by id, at which the sum of the kept
    weights exceeds uniforms (float32 [...], in [0, 1)) times the whole. A temperature of 0 or less takes the largest
    logit. A row without a logit above -inf gives token -1; NaN counts as -inf. Neither result has a gradient: token_logprobs
    scores drawn tokens with one."""
    at, keep = _Rows(logits), []
    logits = logits.detach()
    _is_tensor(uniforms, "uniforms")
    f32 = torch.float32
    tokens = torch.empty(at.lead, dtype=torch.int32, device=at.device)
    logprobs = torch.empty(at.lead, dtype=f32, device=at.device)
    args = _DRAW.pack(_DRAW.size, at.cols, at.rows, at.inner, *at.matrix(logits, keep), at.per_row(uniforms, "uniforms", f32, keep),
                      at.per_row(temperature, "temperature", f32, keep), at.per_row(top_k, "top_k", torch.int32, keep),
                      at.per_row(top_p, "top_p", f32, keep), at.per_row(min_p, "min_p", f32, keep), tokens.data_ptr(),
                      logprobs.data_ptr())
    _check(_library().zbpe_draw_tokens(at.device.index, _stream(at.device), args))
    return tokens, logprobs


# ---- log-probabilities --------------------------------------------------------------------------------------------------------


def _pack_logprobs(at: _Rows, logits, tokens, temperature, logprobs, stats, keep: list) -> bytes:
    return _LOGPROBS.pack(_LOGPROBS.size, at.cols, at.rows, at.inner, *at.matrix(logits, keep), *at.tokens(tokens, "tokens", keep),
                          at.per_row(temperature, "temperature", torch.float32, keep),
                          0 if logprobs is None else logprobs.data_ptr(), 0 if stats is None else stats.data_ptr())


def _logprobs(logits, tokens, temperature, stats):
    at, keep = _Rows(logits), []
    out = torch.empty(at.lead, dtype=torch.float32, device=at.device)
    args = _pack_logprobs(at, logits, tokens, temperature, out, stats, keep)
    _check(_library().zbpe_token_logprobs(at.device.index, _stream(at.device), args))
    return out


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        stats = torch.empty((*logits.shape[:-1], 2), dtype=torch.float32, device=logits.device)
        out = _logprobs(logits, tokens, temperature, stats)
        number = None if isinstance(temperature, torch.Tensor) else temperature
        ctx.number = number
        ctx.save_for_backward(logits, tokens, stats, temperature if number is None else None)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        logits, tokens, stats, temperature = ctx.saved_tensors
        at, keep = _Rows(logits), []
        args = _pack_logprobs(at, logits, tokens, ctx.number if temperature is None else temperature, None, stats, keep)
        grad = grad.contiguous()
        d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _check(_library().zbpe_token_logprobs_grad(at.device.index, _stream(at.device), args, grad.data_ptr(),
                                                   _MATRIX.pack(*at.matrix(d_logits, keep))))
        return d_logits, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature=None) -> torch.Tensor:
    """float32 [...]: the log-probability of each row's token (int32 or int64 [...]) under softmax(logits / temperature), with
    the gradient with respect to the logits (tangents are refused). Negative tokens (padding) are not scored: 0, and no gradient. A token past the
    last column gives NaN; so does +inf or NaN among the logits. A row of -inf alone gives -inf, and no gradient. A
    temperature below 2^-126 (0, negative ones and NaN too) counts as 2^-126: all weight is the largest logits'."""
    _is_tensor(logits, "logits")
    if torch.is_grad_enabled():
        _no_gradient(temperature=temperature)
    if forward_ad._current_level >= 0:
        _no_tangent(logits=logits, temperature=temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Logprobs.apply(logits, tokens, temperature)
    return _logprobs(logits.detach(), tokens, temperature, None)
