"""Serving with a cache of moment states: many sequences that come, go, branch and check drafted tokens.

A sequence's state does not grow with its length, so its place in the cache is ONE page, float32 (layers, heads, rows, d + 4), and sequences
do not share pages.  `table` says which page each place of the batch holds (-1: none); all calls of a model's layers take the
whole batch and leave the places without a page alone.  `arrange` forks, ends and begins sequences, on the device and in one call, so beam
search needs no synchronisation; a page is copied only where a second sequence goes on from it.  Nothing here has a counterpart in
the reference, whose generation loop keeps no state (transformer/eval.py:8-32).
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _ext
from .decoding import check_prompts, per_sequence, refuse_capture, tree_parents


class FastmaxCache:
    """Moment states of up to `places` sequences in `pages` pages (as many as places unless given).

    heads, d, p, temperature, a0, a1, a2: as in `FastmaxDecoder`.  layers: attention layers whose states share a page.
    state: float32 (pages, layers, heads, rows, d + 4).  table: int32 (places,), the page of each place or -1.  Both are updated in
    place by every call, on the current stream.  With sources, parents, lengths and last on the device no call waits for it, and all of them
    can be captured into a CUDA graph; numbers on the host (lists, tensors there; `begin`, `end` and `prefill` have them always) are copied
    first, for which the call waits, and are refused during a capture.
    Nothing here records gradients; outputs must not share memory with the state, those of `verify` not with its inputs either.
    """

    NOTHING, EMPTY = -1, -2   # sources of `arrange` that are no places

    def __init__(self, places, heads, d, p=2, temperature=1.0, a0=1.0, a1=1.0, a2=0.5, layers=1, pages=None, device="cuda"):
        if d not in (16, 32, 64):
            raise ValueError("head dim must be 16, 32 or 64")
        if p not in (1, 2):
            raise ValueError("p must be 1 or 2")
        self.places, self.pages = int(places), int(places if pages is None else pages)
        self.layers, self.heads, self.d, self.p = int(layers), int(heads), int(d), int(p)
        if min(self.places, self.pages, self.layers, self.heads) < 1 or max(self.places, self.pages) > _lib.CACHE_PAGES:
            raise ValueError(f"1 to {_lib.CACHE_PAGES} places and pages, and at least one layer and head")
        self.inv_temperature = 1.0 / float(temperature)
        self.a0, self.a1, self.a2 = float(a0), float(a1), float(a2)
        self.state = _lib.new_state(self.pages * self.layers, self.heads, self.d, self.p, device).unflatten(0, (self.pages, self.layers))
        self.table = torch.full((self.places,), -1, dtype=torch.int32, device=device)
        self._states = self.state.unbind(1)   # a layer's (pages, heads, rows, d + 4)

    # ---- pages -----------------------------------------------------------------------------------------------------------
    def arrange(self, sources):
        """sources (places,): what place i goes on from afterwards: the sequence that place sources[i] held before, NOTHING, or EMPTY, a
        new sequence.  A page stays with the lowest place that goes on from it, the others get copies in free pages, the lowest first.
        Returns int32 (1,) on the device: how many places found no free page; those hold nothing."""
        return _ext().cache_arrange(self.state, self.table, per_sequence(sources, self.table, "sources", -2, self.places - 1))

    def begin(self, places):
        """Starts an empty sequence in each of these places (numbers on the host: not for capture), whatever they held.  Returns what arrange
        returns."""
        return self.arrange(self._with(places, self.EMPTY))

    def end(self, places):
        """Frees the pages of these places (numbers on the host: not for capture)."""
        self.arrange(self._with(places, self.NOTHING))

    def _distinct(self, places):
        places = [int(i) for i in places]
        if any(i < 0 or i >= self.places for i in places) or len(set(places)) != len(places):
            raise ValueError(f"places: different numbers from 0 to {self.places - 1} expected, got {places}")
        return places

    def _with(self, places, source):
        sources = torch.arange(self.places, dtype=torch.int32)
        sources[self._distinct(places)] = source
        return sources

    def compact(self):
        """Moves the live pages to the front of `state`, so that state[:n] holds all of them.  Returns n as int32 (1,) on the device."""
        return _ext().cache_compact(self.state, self.table)

    # ---- one layer's attention ---------------------------------------------------------------------------------------------
    def _layer(self, layer):
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer: 0 to {self.layers - 1} expected, got {layer}")
        return self._states[layer]

    def prefill(self, q, k, v, places, layer=0, continues=False):
        """Causal attention of prompts, (len(places), h, n, d), whose sequences are in `places` (different numbers on the host; they have
        their pages).  The layer's states are replaced by the prompts', or with `continues` extended.  Returns o.  Not for capture."""
        places = self._distinct(places)
        states = self._layer(layer)
        check_prompts(q, k, v, len(places), states)
        if not places:
            return q.new_empty(q.shape)
        refuse_capture(q.device)
        index = self.table[torch.tensor(places, device=self.table.device)]
        before = None
        if continues:
            before = torch.zeros((len(places), *states.shape[1:]), dtype=torch.float32, device=states.device)
            _ext().pages_copy(states, before, index, None, len(places))
        with torch.cuda.device(states.device.index):
            o, _, after = _lib.forward(q, k, v, True, self.inv_temperature, self.a0, self.a1, self.a2, self.p, state_in=before, want_state=True,
                                       flags=_lib.FLAG_PAIRWISE)
        _ext().pages_copy(after, states, None, index, len(places))
        return o

    def step(self, q, k, v, layer=0, out=None):
        """One new token per place: q, k, v are (places, h, d) or (places, h, 1, d).  Returns o shaped like q; rows of places without a
        page stay as they are in `out`, zero without one."""
        return _ext().decode_step_paged(q, k, v, self._layer(layer), self.table, self.inv_temperature, self.a0, self.a1, self.a2, self.p, out)

    def verify(self, q, k, v, parents=None, lengths=None, layer=0, out=None):
        """Attention of drafted tokens, (places, h, n, d) with n <= 64, as in FastmaxDecoder.verify.  Rows of places without a page and rows
        behind a place's nodes stay as they are in `out`, zero without one."""
        return _ext().tree_attention(q, k, v, self._layer(layer), self.table, tree_parents(parents, q), per_sequence(lengths, q, "lengths", 0, q.shape[2]),
                                     self.inv_temperature, self.a0, self.a1, self.a2, self.p, out)

    def accept(self, k, v, last, parents=None, layer=0):
        """Takes the path to node last[i] into the state of place i, as in FastmaxDecoder.accept.  Every layer takes its own k and v."""
        _ext().tree_accept(k, v, self._layer(layer), per_sequence(last, k, "last", -1, k.shape[2] - 1), self.table, tree_parents(parents, k), self.p)
