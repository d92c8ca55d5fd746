"""Beam search over a target on the 8-bit cache: every request's hypotheses are rows of
one step, their caches forked pages of one pool.

One step, all on the device (one HIP graph a side of the caches):
  pages_fork + copy   the tables of the hypotheses that go on (their sources)
  embed, layers       row b at its own position; a hybrid's GatedDeltaNet layers read
                      the window and state of the source (gdn_layer_batch)
  LM head             logits [rows, V]
  beam_select         the next hypotheses: sums, tokens, parents, sources

The reference decodes one sequence (api.py:29-170); it has no beam search.
"""
from __future__ import annotations

import ctypes as C
import time
from dataclasses import dataclass
from typing import Any

import torch

from . import _native as N
from .cache import PAGE, Qwen35Cache
from .pool import HypothesisCache


@dataclass
class BeamHypothesis:
    """Generated tokens (the stop token included), their summed log-probability and
    whether they end with a stop token."""
    tokens: list[int]
    score: float
    finished: bool


class BeamDecoder:
    """``groups`` requests of ``beams`` hypotheses each on a target's engine (of
    ``groups * beams`` rows at most ``max_nodes``). ``start`` runs the prompts,
    ``step`` one token of every hypothesis; ``hypotheses`` reads the result."""

    def __init__(self, target, prompts, beams: int, max_new_tokens: int, stop_token: int = -1, pad_token: int = 0,
                 length_penalty: float = 1.0, use_graph: bool = True):
        eng = self.eng = target.model.engine
        self.target = target
        self.prompts = [[int(t) for t in p] for p in prompts]
        if not self.prompts or min(len(p) for p in self.prompts) < 1:
            raise ValueError("every prompt holds a token")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be positive")
        if not 1 <= beams <= 64:
            raise ValueError("beams in [1, 64]")
        c = eng.cfg
        if not -1 <= stop_token < c.vocab_size or not 0 <= pad_token < c.vocab_size:
            raise ValueError("stop and pad tokens of the vocabulary")
        if any(t < 0 or t >= c.vocab_size for p in self.prompts for t in p):
            raise ValueError("token id outside the vocabulary")
        self.groups, self.beams, self.max_new = len(self.prompts), beams, max_new_tokens
        self.longest = max(len(p) for p in self.prompts) + max_new_tokens
        if self.longest > eng.max_past:
            raise ValueError(f"{self.longest} positions exceed the engine's max_past {eng.max_past}")
        rows = self.rows = self.groups * beams
        # the prompts, and every hypothesis' own: its tokens, a page begun, a copy
        pages = sum((len(p) + PAGE - 1) // PAGE for p in self.prompts) + rows * ((max_new_tokens + PAGE - 1) // PAGE + 2)
        self.cache = HypothesisCache(eng, rows, pages)
        self.use_graph = use_graph
        self._graphs: dict = {}
        dev = eng.dev
        i32 = dict(dtype=torch.int32, device=dev)
        self.scores = torch.zeros(rows, dtype=torch.float32, device=dev)
        self.parents, self.lengths, self.finished = (torch.zeros(rows, **i32) for _ in range(3))
        self.history = torch.zeros(max_new_tokens, 2, rows, **i32)  # tokens, parents
        self.made = 0
        a = self._select = N.BeamArgs()
        a.type = N.T_F32; a.ld_logits = c.vocab_size; a.vocab = c.vocab_size
        a.groups = self.groups; a.num_select = beams
        a.eos_token = stop_token; a.pad_token = pad_token; a.length_penalty = float(length_penalty)
        self.tokens = self.cache.tokens
        for name, t in (("scores", self.scores), ("tokens", self.tokens), ("parents", self.parents),
                        ("lengths", self.lengths), ("finished", self.finished), ("sources", self.cache.sources)):
            setattr(a, name + "_out", t.data_ptr())
        a.beams = beams
        size = eng.lib.dtree_beam_select_workspace_bytes(C.byref(a))
        if not size:
            N.check(N.E_ARG, "beam select")
        self.workspace = torch.empty(size, dtype=torch.uint8, device=dev)
        a.workspace = self.workspace.data_ptr(); a.workspace_bytes = size
        if eng.logits is None:
            eng.logits = torch.zeros(eng.MP, c.vocab_size, dtype=torch.float32, device=dev)
        eng.reserve_hypotheses(self.cache, self.longest)

    # ---- launches ----------------------------------------------------------------
    def _launch_select(self, logits: torch.Tensor, beams: int, st: int) -> None:
        a = self._select
        a.logits = logits.data_ptr()
        a.beams = beams
        first = beams != self.beams or not self.made  # the prompts' rows: no sums yet
        a.scores = None if first else self.scores.data_ptr()
        a.lengths = None if first else self.lengths.data_ptr()
        a.finished = None if first else self.finished.data_ptr()
        N.check(self.eng.lib.dtree_beam_select(C.byref(a), st), "beam select")

    def _record(self) -> None:
        self.history[self.made, 0].copy_(self.tokens)
        self.history[self.made, 1].copy_(self.parents)
        self.made += 1

    def _sequence(self, i: int):
        """Sequence i as the engine's prefill takes a cache, and the windows and states
        that it leaves (a hybrid's)."""
        kv, eng = self.cache.pool.sequence(i), self.eng
        if self.cache.windows is None:
            return kv
        c = Qwen35Cache(eng.cfg, PAGE, device=eng.dev, kv_bits=8)
        c.kv = kv
        return c

    def start(self) -> None:
        """The prompts, one after another, and the first tokens."""
        if self.made:
            raise RuntimeError("the prompts have run: a decoder is used once")
        with torch.cuda.device(self.scores.device):
            self._start()

    def _start(self) -> None:
        eng, cache = self.eng, self.cache
        cache.pool.start([len(p) for p in self.prompts])
        first = torch.empty(self.groups, eng.cfg.vocab_size, dtype=torch.float32, device=eng.dev)
        for g, prompt in enumerate(self.prompts):
            seq = self._sequence(g)
            logits, _ = self.target.forward_with_hidden_states(torch.tensor([prompt]), seq, list(eng.layer_ids))
            first[g].copy_(logits[0, -1])
            if cache.windows is not None:
                cache.windows[cache.turn, :, g].copy_(seq.windows)
                cache.states[cache.turn, :, g].copy_(seq.states)
        cache.pool._sequences.clear()  # (the tables are the device's from here on)
        cache.pool._set_rooms([(0, 0)] * self.rows)
        cache.positions.zero_()
        cache.positions[:self.groups].copy_(torch.tensor([len(p) for p in self.prompts], dtype=torch.int32))
        self._launch_select(first, 1, eng.stream_handle())
        self._record()

    def _launch_step(self, advance: int, st: int) -> None:
        self.eng.launch_hypotheses(self.cache, advance, st)
        self._launch_select(self.eng.logits, self.beams, st)

    def step(self) -> None:
        """One token of every hypothesis that goes on."""
        if not 1 <= self.made < self.max_new:
            raise RuntimeError("start() comes first, and max_new_tokens bounds the steps")
        with torch.cuda.device(self.scores.device):
            self._step()

    def _step(self) -> None:
        eng, cache = self.eng, self.cache
        # a hypothesis is as long as its prompt and the tokens that it has fed
        cache.max_past = eng.attn_grid_past(min(self.longest - self.max_new + self.made - 1, eng.max_past))
        advance = 0 if self.made == 1 else 1
        st = eng.stream_handle()
        if self.use_graph and advance:  # (the step behind the prompts is one of its kind)
            N.check(eng.lib.dtree_graph_launch(C.c_void_p(self._graph()), st), "graph launch")
        else:
            self._launch_step(advance, st)
        cache.flip()
        self._record()

    def _graph(self) -> int:
        # (a graph holds the engine's buffers: those of its hidden layers may change)
        eng = self.eng
        eng._destroy_pending()
        key = (self.cache.turn, self.cache.max_past, tuple(eng.layer_ids), eng.hidden.data_ptr())
        if key not in self._graphs:
            lib = eng.lib
            side = torch.cuda.Stream(device=eng.dev)
            side.wait_stream(torch.cuda.current_stream())
            N.check(lib.dtree_graph_begin(side.cuda_stream), "graph begin")
            ex = C.c_void_p()
            try:
                self._launch_step(1, side.cuda_stream)
            except Exception:
                lib.dtree_graph_end(side.cuda_stream, C.byref(ex))
                raise
            N.check(lib.dtree_graph_end(side.cuda_stream, C.byref(ex)), "graph end")
            torch.cuda.current_stream().wait_stream(side)
            self._graphs[key] = ex.value
        return self._graphs[key]

    def done(self) -> bool:
        """Whether every hypothesis has ended (waits for the device)."""
        self.cache.pool.check()
        return bool(((self.finished != 0) | (self.parents < 0)).all())

    def hypotheses(self) -> list[list[BeamHypothesis]]:
        """Every request's hypotheses, best first."""
        self.cache.pool.check()
        hist = self.history[:self.made].cpu()
        scores, lengths, finished = self.scores.tolist(), self.lengths.tolist(), self.finished.tolist()
        last = hist[-1, 1].tolist()
        out = []
        for g in range(self.groups):
            best = []
            for i in range(g * self.beams, (g + 1) * self.beams):
                if last[i] < 0:  # fewer continuations than beams
                    continue
                toks, at = [], i
                for t in range(self.made - 1, -1, -1):
                    toks.append(int(hist[t, 0, at]))
                    at = int(hist[t, 1, at])
                best.append(BeamHypothesis(toks[::-1][:lengths[i]], scores[i], bool(finished[i])))
            out.append(best)
        return out

    def release(self) -> None:
        """Destroys the captured steps (after the device is done with them)."""
        if self._graphs:
            torch.cuda.synchronize(self.eng.dev)
            for g in self._graphs.values():
                self.eng.lib.dtree_graph_destroy(C.c_void_p(g))
            self._graphs.clear()

    def __del__(self):
        # (may run at any point, during a capture too: the engine destroys them at a launch)
        graphs = self.__dict__.get("_graphs")
        if graphs:
            self.eng._dead_graphs.extend(graphs.values())


def beam_generate(target, prompts, num_beams: int = 4, max_new_tokens: int = 256, stop_token_ids=None, pad_token: int = 0,
                  length_penalty: float = 1.0, use_graph: bool = True) -> tuple[list[list[BeamHypothesis]], dict[str, Any]]:
    """Beam search of every prompt (lists of token ids): their ``num_beams`` best
    continuations by summed log-probability / length ** length_penalty, best first, and
    metrics. A hypothesis that reaches the stop token stays among the beams with its sum
    and competes. Requests are decoded together, as many as the engine's rows hold."""
    eng = target.model.engine
    stops = sorted(target.stop_token_ids() if stop_token_ids is None else {int(t) for t in stop_token_ids})
    if len(stops) > 1:
        raise ValueError("beam search takes one stop token")
    together = eng.max_nodes // num_beams if num_beams > 0 else 0
    if together < 1:
        raise ValueError(f"num_beams {num_beams}: the engine steps up to {eng.max_nodes} rows (max_nodes)")
    prompts = [list(p) for p in prompts]
    out, steps, prefill_time = [], 0, 0.0
    began = time.perf_counter()
    for at in range(0, len(prompts), together):
        d = BeamDecoder(target, prompts[at:at + together], num_beams, max_new_tokens, stops[0] if stops else -1, pad_token,
                        length_penalty, use_graph)
        t0 = time.perf_counter()
        d.start()
        over = d.done()
        prefill_time += time.perf_counter() - t0
        while not over and d.made < max_new_tokens:
            d.step()
            steps += 1
            over = d.done()
        out += d.hypotheses()
        d.release()
    total = time.perf_counter() - began
    tokens = sum(len(h[0].tokens) for h in out if h)
    metrics = {"decode_mode": "beam", "num_beams": num_beams, "length_penalty": length_penalty,
               "num_input_tokens": sum(len(p) for p in prompts), "num_output_tokens": tokens, "steps": steps,
               "prefill_time_s": prefill_time, "decode_time_s": total - prefill_time, "total_time_s": total,
               "peak_memory_gb": (torch.cuda.max_memory_allocated() / 1e9) if torch.cuda.is_available() else 0.0}
    return out, metrics
