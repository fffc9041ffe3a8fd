"""Serving loop over any registered model: requests with their own state, a step that feeds one request's next tokens, a
first-come scheduler that cuts prompts into portions and interleaves decoding, and token sampling.

`Engine.step` is the only place that runs a model; generation (`submit` / `run` / `generate`) and trace replay both go through it.
"""
from __future__ import annotations

import math
from collections import deque
from ctypes import c_float
from dataclasses import dataclass, field

import torch

import seq_ops as S
from seq_state import StatePool


@dataclass
class SamplingParams:
    max_new: int = 16
    temperature: float = 0.0     # 0: greedy
    top_k: int = 0               # 0: all tokens
    seed: int = 0
    stop: tuple = ()             # token ids that end the request (kept in the output)
    repetition: float = 1.0      # what the logits of all tokens so far are divided by (negative ones: multiplied)
    presence: float = 0.0        # taken off the logits of generated tokens,
    frequency: float = 0.0       # and as often as they were generated
    bias: tuple = ()             # (token id, added to its logit) pairs
    allowed: object = None       # callable: generated tokens so far -> ids that may come next, None: all

    def adjusts(self) -> bool:
        return self.repetition != 1.0 or self.presence != 0.0 or self.frequency != 0.0 or bool(self.bias) or self.allowed is not None


@dataclass
class Request:
    rid: object
    prompt: list
    params: SamplingParams
    fed: int = 0                                   # prompt tokens already run
    out: list = field(default_factory=list)
    done: bool = False
    said: torch.Tensor | None = None               # prompt and generated tokens on the device, for the penalties
    bias: tuple | None = None                      # (ids, values) on the device


class Engine:
    def __init__(self, model, max_tokens: int, portion: int = 2048, max_live: int = 8):
        """max_tokens: capacity of one request's state; portion: most prompt tokens a step runs; max_live: requests with a state at once."""
        if portion < 1 or max_live < 1:
            raise ValueError("portion and max_live must be positive")
        self.model, self.portion, self.max_live = model, portion, max_live
        self.pool = StatePool(model, max_tokens)
        self.waiting, self.live, self.finished = deque(), deque(), {}
        self.failed = {}             # request id: (exception, tokens generated so far) of requests that ended so
        self._next = 0

    # ---- the step ----------------------------------------------------------------------------------------------------
    def step(self, rid, tokens, want=(), end: bool = False):
        """Feed `tokens` to request rid (a new id starts a sequence) and return the fp32 logits at the places `want` among them, or None.
        end: the request is finished after this step and its state goes back to the pool."""
        V = self.model.vocab
        for t in tokens:
            if not 0 <= t < V:
                raise ValueError(f"token {t} outside the vocabulary of {V}")
        for w in want:
            if not 0 <= w < len(tokens):
                raise ValueError(f"place {w} among {len(tokens)} tokens")
        st = self.pool.get(rid) if rid in self.pool else self.pool.acquire(rid)
        out = self.model.forward(torch.tensor([list(tokens)], dtype=torch.int64), st, list(want)) if len(tokens) else None
        if end:
            self.pool.release(rid)
        return out

    def end(self, rid):
        if rid in self.pool:
            self.pool.release(rid)

    # ---- generation ----------------------------------------------------------------------------------------------------
    def submit(self, prompt, params: SamplingParams | None = None):
        params = params or SamplingParams()
        if not prompt:
            raise ValueError("empty prompt")
        r, p, f = (c_float(v).value for v in (params.repetition, params.presence, params.frequency))      # as the kernel takes them
        if not 0.0 < r < math.inf:
            raise ValueError("the repetition penalty is a positive factor")
        total = {}
        for t, v in params.bias:
            total[t] = total.get(t, 0.0) + c_float(v).value
        if any(math.isnan(v - p - f) for v in (0.0, *total.values())):
            raise ValueError("presence, frequency and biases that add up to no number")
        if any(not 0 <= t < self.model.vocab for t, _ in params.bias):
            raise ValueError(f"a bias for a token outside the vocabulary of {self.model.vocab}")
        if len(params.bias) > 4096:
            raise ValueError(f"{len(params.bias)} biases, at most 4096")
        if len(prompt) + params.max_new > self.pool.capacity:
            raise ValueError(f"{len(prompt)} + {params.max_new} tokens exceed the capacity {self.pool.capacity}")
        rid = ("gen", self._next)
        self._next += 1
        self.waiting.append(Request(rid, list(prompt), params))
        return rid

    def schedule(self):
        """The request that the next step serves: requests are admitted in order while there is room, a prompt that has started is
        finished first, then the live requests decode in turn."""
        while self.waiting and len(self.live) < self.max_live:
            self.live.append(self.waiting.popleft())
        for r in self.live:
            if r.fed < len(r.prompt):
                return r
        return self.live[0] if self.live else None

    def run_one(self) -> bool:
        """One scheduled step; False when there is nothing left to do."""
        r = self.schedule()
        if r is None:
            return False
        if r.fed < len(r.prompt):
            part = r.prompt[r.fed:r.fed + self.portion]
            r.fed += len(part)
            logits = self.step(r.rid, part, [len(part) - 1] if r.fed == len(r.prompt) else ())
        else:
            logits = self.step(r.rid, [r.out[-1]], [0])
        if logits is not None and r.params.max_new > 0:
            try:
                self._take(r, logits)
            except Exception as e:       # its settings failed: it ends, the others go on with the next call
                self.live.remove(r)
                self.end(r.rid)
                self.failed[r.rid] = (e, r.out)
                e.add_note(f"request {r.rid!r} after {len(r.out)} tokens")
                raise
        if r.done or (r.fed == len(r.prompt) and len(r.out) >= r.params.max_new):
            self.live.remove(r)
            self.end(r.rid)
            self.finished[r.rid] = r.out
        elif r.fed == len(r.prompt):
            self.live.remove(r)          # to the back: the others decode next
            self.live.append(r)
        return True

    def _take(self, r: Request, logits: torch.Tensor):
        p = r.params
        at = torch.tensor([r.fed + len(r.out)], dtype=torch.int32, device=logits.device)
        if p.adjusts():
            logits = self._adjust(r, logits)
        tok = int(S.sample(logits, at, p.temperature, p.top_k, p.seed).item())
        r.out.append(tok)
        r.done = tok in p.stop

    def _adjust(self, r: Request, logits: torch.Tensor) -> torch.Tensor:
        """The request's settings on its logits fp32 [1, V]."""
        p, dev, V = r.params, logits.device, logits.shape[1]
        kw = {}
        if p.repetition != 1.0 or p.presence != 0.0 or p.frequency != 0.0:
            n, n_prompt = len(r.prompt) + len(r.out), len(r.prompt)
            if r.said is None:
                r.said = torch.tensor([r.prompt + [0] * p.max_new], dtype=torch.int64, device=dev)
            if r.out:
                S.put(r.said[0, n - 1:n], torch.tensor(r.out[-1:]))
            counts = torch.tensor([[n], [n_prompt]], dtype=torch.int32, device=dev)
            kw = dict(tokens=r.said, lengths=counts[0], prompt_lengths=counts[1], repetition=p.repetition, presence=p.presence, frequency=p.frequency)
        if p.bias:
            if r.bias is None:
                r.bias = (torch.tensor([[t for t, _ in p.bias]], dtype=torch.int64, device=dev), torch.tensor([[b for _, b in p.bias]], dtype=torch.float32, device=dev))
            kw.update(bias_ids=r.bias[0], bias=r.bias[1])
        ids = p.allowed(list(r.out)) if p.allowed is not None else None
        if ids is not None:
            ids = torch.tensor(sorted({int(t) for t in (ids.tolist() if hasattr(ids, "tolist") else ids)}), dtype=torch.int64)      # numbers: equal elements of a tensor are different objects
            if ids.numel() == 0 or ids[0] < 0 or ids[-1] >= V:
                raise ValueError(f"request {r.rid!r}: no token is allowed, or one outside the vocabulary of {V}")
            words = torch.zeros((V + 31) // 32, dtype=torch.int64)
            words.index_add_(0, ids >> 5, 1 << (ids & 31))
            kw["mask"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).view(1, -1).to(dev)
        return S.adjust_logits(logits, **kw)

    def cancel(self, rid):
        """Whatever has become of a submitted request, nothing of it stays."""
        self.waiting = deque(r for r in self.waiting if r.rid != rid)
        self.live = deque(r for r in self.live if r.rid != rid)
        self.end(rid)
        self.finished.pop(rid, None)
        self.failed.pop(rid, None)

    def run(self) -> dict:
        """Until every submitted request is finished: {request id: generated tokens} of all finished so far. A request that fails raises and is in `failed`; the next call goes on with the others."""
        while self.run_one():
            pass
        return self.finished

    def generate(self, prompts, params: SamplingParams | None = None):
        """Generated tokens of every prompt, in order. Where one of them fails, none of them stays."""
        ids = []
        try:
            for p in prompts:
                ids.append(self.submit(p, params))
            while True:
                try:
                    if not self.run_one():
                        return [self.finished.pop(i) for i in ids]
                except Exception as e:
                    rid = next((i for i, (error, _) in self.failed.items() if error is e), None)
                    if rid is None or rid in ids:
                        raise            # else the request of another caller, who finds it in `failed`
        except BaseException:
            for i in ids:
                self.cancel(i)
            raise
