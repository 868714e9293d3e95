"""Token-by-token Fastmax attention with a carried moment state.

The reference generates text by running the whole model, and with it the attention operator, on the full token
window for every new token (transformer/eval.py:8-32: `logits = model(token_chunk)` inside the loop over
`max_new_tokens`).  Fastmax attention does not need that: everything a later query needs from the keys and
values seen so far is the fixed-size moment state S = sum_j Phi(k_j)^T [v_j | 1].  `FastmaxDecoder` keeps that
state on the device; `prefill` runs the causal operator over a prompt and leaves the state behind, `step`
feeds one token per (batch, head) through `fastmax_decode_step`, whose cost does not depend on how many tokens
came before.

Several drafted tokens at once: `verify` gives the attention of a tree of drafted tokens without changing the state, `accept` takes
the path that the caller keeps into it.  `cache.FastmaxCache` does the same for sequences that come, go and branch.

The q/k normalisation of the operator (`normalize=True`) divides by the largest token norm of the whole
sequence and therefore cannot be evaluated incrementally; the decoder takes un-normalised q and k, as the
reference's CPU implementations do by default (fastattention_einops.py:78-82).
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _ext


class FastmaxDecoder:
    """Causal Fastmax attention over a growing sequence.

    batch, heads, d, p: problem geometry (d in {16, 32, 64}; p = polynomial order 1 or 2).
    temperature, a0, a1, a2: as in `fastmax_custom` (scores are q.k / temperature).
    The state is float32 (batch, heads, rows, d + 4) in the layout of `fastmax_forward`'s state_out and is
    updated in place by every call, so a step that was captured into a CUDA graph goes on from whatever was read last.
    """

    def __init__(self, batch, heads, d, p=2, temperature=1.0, a0=1.0, a1=1.0, a2=0.5, device="cuda"):
        if d not in (16, 32, 64):
            raise ValueError("head dim must be 16, 32 or 64")
        if p not in (1, 2):
            raise ValueError("p must be 1 or 2")
        self.batch, self.heads, self.d, self.p = int(batch), int(heads), int(d), int(p)
        self.inv_temperature = 1.0 / float(temperature)
        self.a0, self.a1, self.a2 = float(a0), float(a1), float(a2)
        self.state = _lib.new_state(self.batch, self.heads, self.d, self.p, device)
        self.tokens_seen = 0

    def reset(self):
        self.state.zero_()
        self.tokens_seen = 0

    def _check(self, t, name):
        shape = t.shape
        if shape[0] != self.batch or shape[1] != self.heads or shape[-1] != self.d:
            raise ValueError(f"{name}: expected ({self.batch}, {self.heads}, ..., {self.d}), got {tuple(t.shape)}")

    def prefill(self, q, k, v):
        """Causal attention of a (b, h, n, d) block that continues the sequence seen so far.  Returns o (b, h, n, d)
        and adds the block's keys and values to the state."""
        check_prompts(q, k, v, self.batch, self.state)
        with torch.cuda.device(self.state.device.index):
            before = self.state if self.tokens_seen else None
            # the state keeps its memory, which a captured step reads; the call does not take one array as both of its states
            o, _, state = _lib.forward(q, k, v, True, self.inv_temperature, self.a0, self.a1, self.a2, self.p, state_in=before,
                                       want_state=True, flags=_lib.FLAG_PAIRWISE, state_out=None if self.tokens_seen else self.state)
            if before is not None:
                self.state.copy_(state)
        self.tokens_seen += q.shape[2]
        return o

    def step(self, q, k, v, out=None):
        """One new token per (batch, head): q, k, v are (b, h, d) or (b, h, 1, d).  Returns o shaped like q."""
        for t, name in ((q, "q"), (k, "k"), (v, "v")):
            self._check(t, name)
        # through the extension: the ctypes binding costs 20 us of interpreter time per token, the kernel 7 us for eight heads
        o = _ext().decode_step(q, k, v, self.state, self.inv_temperature, self.a0, self.a1, self.a2, self.p, out)
        self.tokens_seen += 1
        return o

    def verify(self, q, k, v, parents=None, lengths=None, out=None):
        """Attention of drafted tokens, (b, h, n, d) with n <= 64, that leaves the state as it is: node i sees the sequence so far, its
        ancestors and itself.  parents: int32 (b, n), the parent of each node (a node before it, or -1: the sequence itself); None: a chain.
        lengths: int32 (b,), nodes of each sequence.  Returns o (b, h, n, d); rows behind a sequence's nodes stay as they are in
        `out`, zero without one.  Can be captured into a CUDA graph with parents and lengths on the device."""
        return _ext().tree_attention(q, k, v, self.state, None, tree_parents(parents, q), per_sequence(lengths, q, "lengths", 0, q.shape[2]),
                                     self.inv_temperature, self.a0, self.a1, self.a2, self.p, out)

    def accept(self, k, v, last, parents=None):
        """Takes drafted tokens into the state: the path from the root to node last[i] for every sequence i, nothing where last[i] is
        -1.  k, v, parents as `verify` had them; last: int32 (b,).  Can be captured with last and parents on the device.  tokens_seen, one number
        for all sequences, grows by the longest path that the drafts can have: from then on it is a bound, not a length."""
        _ext().tree_accept(k, v, self.state, per_sequence(last, k, "last", -1, k.shape[2] - 1), None, tree_parents(parents, k), self.p)
        self.tokens_seen += k.shape[2]


def check_prompts(q, k, v, batch, state):
    """Prompts' q, k, v for the `batch` sequences of `state` (float32 (..., heads, rows, d + 4)): all of it is refused here, before anything is
    launched, since the binding that prompts go through takes the sizes, the type and the device of all three from q."""
    shape, sizes = q.shape, state.shape
    if len(shape) != 4 or k.shape != shape or v.shape != shape or shape[0] != batch or shape[1] != sizes[-3] or shape[3] != sizes[-1] - 4:
        raise ValueError(f"q, k, v: expected ({batch}, {sizes[-3]}, n, {sizes[-1] - 4}), got {tuple(shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if shape[2] == 0:
        raise ValueError("a prompt needs a token")
    dtype, device = q.dtype, state.device
    _lib.dtype_code(q)
    if k.dtype != dtype or v.dtype != dtype:
        raise RuntimeError(f"dtypes differ: q {dtype}, k {k.dtype}, v {v.dtype}")
    if q.stride(3) != 1 or k.stride(3) != 1 or v.stride(3) != 1:
        raise RuntimeError("the head dim must be contiguous")
    if device.type != "cuda" or q.device != device or k.device != device or v.device != device:
        raise RuntimeError(f"q, k, v must be CUDA tensors on the state's device {device}, got {q.device}, {k.device}, {v.device}")


def _is_there(x):
    return x is None or (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.int32)


def per_sequence(x, like, name, low, high):
    """One number per sequence as an int32 tensor beside `like`.  What lies on the host is checked to be in low .. high and copied, for which
    the call waits and which cannot be captured; what lies on the device is not read here (the kernels treat other numbers as their
    documentation says), and int32 there goes on as it is."""
    if _is_there(x):
        return x
    x = _whole(x, name)
    if tuple(x.shape) != (like.shape[0],):
        raise ValueError(f"{name}: expected ({like.shape[0]},), got {tuple(x.shape)}")
    if not x.is_cuda and bool(((x < low) | (x > high)).any()):
        raise ValueError(f"{name}: numbers from {low} to {high} expected")
    return _int32(x, like, low, high)


def tree_parents(parents, like):
    """The parents of (b, n) nodes as an int32 tensor beside `like` (b, h, n, d); checked as in per_sequence."""
    if _is_there(parents):
        return parents
    parents = _whole(parents, "parents")
    if like.dim() != 4 or tuple(parents.shape) != (like.shape[0], like.shape[2]):
        raise ValueError(f"parents: expected (b, n) for (b, h, n, d) tensors, got {tuple(parents.shape)}")
    if not parents.is_cuda and bool(((parents < -1) | (parents >= torch.arange(parents.shape[1]))).any()):
        raise ValueError("parents: every node needs a parent before it, or -1")
    return _int32(parents, like, -1, like.shape[2])


def _whole(x, name):
    x = torch.as_tensor(x)
    if x.dtype.is_floating_point or x.dtype.is_complex or x.dtype in (torch.bool, torch.uint64):   # uint64: not all of it fits below
        raise TypeError(f"{name}: whole numbers of up to 64 bits with a sign expected, got {x.dtype}")
    return x.to(torch.int64)   # bounds are compared in 64 bits: a narrow type does not hold them all


def _int32(x, like, low, high):
    if x.is_cuda:   # what is out of range stays so when it loses its upper bits
        x = x.clamp(low - 1, high + 1)
    else:
        refuse_capture(like.device)
    return x.to(device=like.device, dtype=torch.int32)


def refuse_capture(device):
    """For what copies from the host and waits for it: said before the copy, so that the capture goes on without the call."""
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("numbers on the host cannot go into a CUDA graph: pass int32 tensors on the device")
