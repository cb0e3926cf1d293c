"""Continuous batching for LLMEngine over the paged key-value cache.

With ``LLMArgs(kv_cache="paged")`` (or ``"paged_e4m3"``: 8-bit pages) the
engine keeps one PagedKVCache for all requests instead of a dense, padded
cache for each group: a request joins at any step as soon as a row and its
pages are free, its prompt is read in one packed pass without padding, every
decode step runs all active requests, and its pages go back when it ends.

The model's layers are transformers' own; only their attention is replaced,
through its AttentionInterface: the new keys and values go into the pages
(ops/paged.py write_kv), and decode_attention or prompt_attention reads them.
"""

from __future__ import annotations

import math
import threading
from collections import deque
from typing import Any, Deque, List, Optional

NAME = "beta9_paged"
KINDS = ("dense", "paged", "paged_e4m3")


class Step:
    """What one forward pass tells its layers' attention."""

    def __init__(self, cache, plan, active=None):
        self.cache, self.plan, self.active = cache, plan, active  # active: of a decode step's rows


def attention(module, query, key, value, attention_mask, scaling=None, paged_step=None, **kwargs):
    """transformers' attention signature; query [1, heads, tokens, dim]."""
    if paged_step is None:
        raise RuntimeError("this model's attention runs on a paged cache: call it through the engine")
    if kwargs.get("sliding_window") is not None or kwargs.get("softcap") is not None or kwargs.get("s_aux") is not None:
        raise ValueError("the paged cache serves full attention only, without windows, caps or sinks")
    step, layer = paged_step, module.layer_idx
    cache, plan = step.cache, step.plan
    q, k, v = (x[0].transpose(0, 1) for x in (query, key, value))  # [tokens, heads, dim]
    cache.write(layer, k, v, plan)
    if step.active is None:
        out = cache.prompt(layer, q, plan, scaling)
    else:
        out = cache.decode(layer, q, plan, scaling, step.active)
    return out.unsqueeze(0), None


def register() -> str:
    """Makes the attention known to transformers; returns its name there."""
    from transformers import AttentionInterface, AttentionMaskInterface

    AttentionInterface.register(NAME, attention)
    AttentionMaskInterface.register(NAME, lambda *args, **kwargs: None)  # lengths and positions say it all
    return NAME


def sample(logits, temperature: float) -> Optional[int]:
    """A token at a temperature above zero; None if the largest logit is not
    a finite number."""
    import torch

    top = logits.max()
    if not math.isfinite(top.item()):
        return None
    # The largest is taken off first, and the temperature kept in range: the quotients then pass 32 bits only towards -inf,
    # whose weight is 0, and a temperature next to zero takes the largest.
    t = min(max(temperature, 2.0**-100), 2.0**100)
    return int(torch.multinomial(torch.softmax((logits - top) / t, dim=-1), 1).item())


class PagedDecoder:
    """Rows, pages and steps of one engine's model."""

    def __init__(self, model, args, eos_id: Optional[int], dtype, device: str):
        import torch

        from ..ops.paged import MAX_HEAD_DIM, PagedKVCache

        cfg = model.config
        heads = cfg.num_attention_heads
        dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // heads
        kv_heads = getattr(cfg, "num_key_value_heads", None) or heads
        kinds = set(getattr(cfg, "layer_types", None) or ["full_attention"])
        if dim % 8 or dim > MAX_HEAD_DIM or kinds != {"full_attention"}:
            raise ValueError(
                f"kv_cache={args.kv_cache!r} needs full attention in every layer and a head dim that is a "
                f"multiple of 8 up to {MAX_HEAD_DIM}; this model has {sorted(kinds)} and {dim}"
            )
        # without layer types, a window is that of every layer
        for name, set_to in (
            ("sliding_window", None if getattr(cfg, "layer_types", None) else getattr(cfg, "sliding_window", None)),
            ("attn_logit_softcapping", getattr(cfg, "attn_logit_softcapping", None)),
        ):
            if set_to is not None:
                raise ValueError(
                    f"kv_cache={args.kv_cache!r} serves attention without windows or caps; this model has {name} = {set_to}"
                )
        if device != "cpu" and dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"kv_cache={args.kv_cache!r} needs dtype='bfloat16' on a GPU, not {args.dtype!r}")
        model.set_attn_implementation(register())
        self.model, self.args, self.eos_id, self.device = model, args, eos_id, device
        size = args.kv_page_size
        pages = args.kv_pages or args.max_num_seqs * -(-args.max_model_len // size)
        e4m3 = args.kv_cache == "paged_e4m3"
        self.cache = PagedKVCache(
            cfg.num_hidden_layers, kv_heads, dim, pages, size, args.max_num_seqs, args.max_model_len,
            torch.float8_e4m3fn if e4m3 else dtype, device,
            *((args.kv_scale, args.kv_scale) if e4m3 else ()),
        )
        self.rows: List[Any] = [None] * args.max_num_seqs  # request of each row
        self.lens = [0] * args.max_num_seqs  # tokens held, as the GPU has them
        self.reserved = [0] * args.max_num_seqs  # pages a row may come to hold
        self.waiting: List[Any] = []
        # A step whose loop was stopped runs on in its thread; the next one waits for it. What it ends stays here until a loop
        # takes it. Requests go from `waiting` to `rows` to `_ended`, and are entered in the next before they leave the last,
        # so that a loop that looks at the three in this order beside a running step misses none.
        self._ended: Deque[Any] = deque()
        self._freed: List[int] = []
        self._lock = threading.Lock()
        self.broken: Optional[Exception] = None  # why no step can be run any more

    @property
    def active(self) -> bool:
        return bool(self.waiting) or any(r is not None for r in self.rows)

    def submit(self, req) -> None:
        """A request for the next step."""
        self.waiting.append(req)

    def take_ended(self) -> List[Any]:
        """The requests that ended since the last call."""
        ended = []
        while self._ended:
            ended.append(self._ended.popleft())
        return ended

    def _most(self, req) -> int:
        """Tokens the request can come to hold: its last one is never written."""
        return min(len(req.prompt_ids) + req.max_tokens - 1, self.args.max_model_len)

    def _admit(self) -> List[int]:
        """Rows of the waiting requests that start now, in their order."""
        started = []
        while self.waiting:
            req = self.waiting[0]
            if req.max_tokens <= 0 or not req.prompt_ids:
                if not req.prompt_ids:
                    req.error = ValueError("the prompt has no tokens")
                self._ended.append(req)
                self.waiting.pop(0)
                continue
            pages = self.cache.pages_for(self._most(req))
            if len(req.prompt_ids) > self.args.max_model_len or pages > self.cache.pages:
                req.error = ValueError(
                    f"a request of {len(req.prompt_ids)} + {req.max_tokens} tokens does not fit the cache: "
                    f"{self.args.max_model_len} tokens a row, {self.cache.pages} pages of {self.cache.page_size}"
                )
                self._ended.append(req)
                self.waiting.pop(0)
                continue
            free = [r for r, q in enumerate(self.rows) if q is None]
            if not free or sum(self.reserved) + pages > self.cache.pages:
                break  # first come, first served
            row = free[0]
            self.rows[row], self.reserved[row], self.lens[row] = req, pages, 0
            self.waiting.pop(0)
            started.append(row)
        return started

    def _forward(self, rows: List[int], ids: List[int], new: List[int], decode: bool) -> List[Optional[int]]:
        """One pass over the packed tokens of `rows`; each row's next token,
        None where its logits give none."""
        import torch

        put = lambda x, t: torch.tensor(x, dtype=t, device=self.device)  # noqa: E731
        new_lens = [0] * len(self.rows)
        for row, n in zip(rows, new):
            new_lens[row] = n
            self.lens[row] += n
        plan = self.cache.plan(put(new_lens, torch.int32), len(ids))
        step = Step(self.cache, plan, self.cache.active(plan, put(rows, torch.long)) if decode else None)
        ends = put([sum(new[: i + 1]) - 1 for i in range(len(new))], torch.long)
        logits = self.model(
            input_ids=put([ids], torch.long),
            position_ids=plan.positions.long().unsqueeze(0),
            use_cache=False,
            logits_to_keep=ends,
            paged_step=step,
        ).logits[0].float()
        tokens = logits.argmax(-1).tolist()
        for i, row in enumerate(rows):
            t = self.rows[row].temperature
            if t > 0:
                tokens[i] = sample(logits[i], t)
        return tokens

    def _take(self, rows: List[int], tokens: List[Optional[int]]) -> None:
        for row, token in zip(rows, tokens):
            req = self.rows[row]
            if token is None:
                req.error = ValueError("no token can be drawn: the model's logits are not finite")
            else:
                req.out_ids.append(token)
            full = self.lens[row] >= self.args.max_model_len
            if token is None or (self.eos_id is not None and token == self.eos_id) or len(req.out_ids) >= req.max_tokens or full:
                self._ended.append(req)
                self.rows[row] = None
                self._freed.append(row)

    def _end(self, req, error: Exception) -> None:
        req.error = error
        self._ended.append(req)

    def _fail(self, error: Exception) -> None:
        """After a step that raised: ends every request with its error, and
        starts again with an empty cache. If that raises too, the requests
        of all later steps end with an error."""
        import torch

        for row, req in enumerate(self.rows):
            if req is not None:
                self._end(req, error)
                self.rows[row] = None
        while self.waiting:
            self._end(self.waiting[0], error)
            self.waiting.pop(0)
        n = len(self.rows)
        self.lens, self.reserved = [0] * n, [0] * n
        if self.broken is None:
            try:
                self.cache.release(torch.ones(n, dtype=torch.bool, device=self.device))
            except Exception as e:
                self.broken = RuntimeError(f"the paged cache could not be reset after an error: {e}")

    def step(self) -> None:
        """Reads the waiting prompts that fit, decodes one token of every
        active request. An error ends the requests and is not raised."""
        with self._lock:
            try:
                if self.broken is not None:
                    raise self.broken
                self._step()
            except Exception as e:
                self._fail(e)

    def _step(self) -> None:
        import torch

        self._freed = []
        with torch.inference_mode():
            started = self._admit()
            if started:
                prompts = sorted(started)  # the plan packs by row
                ids = [self.rows[r].prompt_ids for r in prompts]
                self._take(prompts, self._forward(prompts, sum(ids, []), [len(i) for i in ids], False))
            rows = [r for r, q in enumerate(self.rows) if q is not None]
            if rows:
                last = [self.rows[r].out_ids[-1] for r in rows]
                self._take(rows, self._forward(rows, last, [1] * len(rows), True))
            if self._freed:
                done = torch.zeros(len(self.rows), dtype=torch.bool)
                done[self._freed] = True
                self.cache.release(done.to(self.device))
                for row in self._freed:
                    self.reserved[row] = self.lens[row] = 0
