"""A key-value cache in pages that requests of any length share, on gfx950.

Four operators and the cache object that holds their state:

- ``plan_step``: block tables, slots and positions of a step's new tokens,
  computed on the GPU from the requests' lengths; ``release_pages`` gives
  the pages of finished requests back;
- ``write_kv``: new keys and values into their pages;
- ``decode_attention``: attention of one new token of each request;
- ``prompt_attention``: causal attention of packed new tokens, any number
  of each request, behind what the cache already holds of it.

The cache holds keys and values as [pages, kv heads, page size, head dim],
in the type of the queries (bfloat16, float16) or in float8_e4m3fn with one
scale each for keys and values. Head dims are multiples of 8 up to 256; the
attention kernels compute with 64, 128 or 256, so these cost least. Page
sizes are 16 to 256 in powers of two. ``tables[r, i]`` is the page of request
r's tokens i * page_size and on. Lengths, tables and slots stay on the GPU: no
call copies to the host or waits, and every one can be captured into a HIP
graph. Workspaces belong to the call, so calls on several streams, or from
several captured graphs, share nothing but the tensors they are given.

All are for inference: an input that requires a gradient is refused while
gradients are recorded. Wrong shapes and values raise ValueError, wrong
types TypeError. As in ops/gemm.py, a missing extension on a GPU host is a
hard error, and CPU tensors take a plain torch path (any floating type).
"""

from __future__ import annotations

import math
import threading
from typing import NamedTuple, Optional, Tuple

import torch

from .gemm import E4M3_MAX

MAX_REQUESTS = 4096
MAX_HEAD_DIM = 256
PAGE_SIZES = (16, 32, 64, 128, 256)

_ext = None
_tried = False
_loading = threading.Lock()


def _load():
    global _ext, _tried
    if not _tried:
        with _loading:  # a second thread's first call waits for the import
            if not _tried:
                try:
                    from . import _paged_ext

                    _ext = _paged_ext
                except ImportError as e:
                    if torch.cuda.is_available():
                        raise RuntimeError(
                            f"gfx950 paged-cache extension missing on a GPU host: {e}; "
                            "run __graft_entry__.build()"
                        )
                _tried = True
    return _ext


def has_native() -> bool:
    return _load() is not None


def _native(t: torch.Tensor):
    """The extension for a GPU tensor, None for a CPU one."""
    if not t.is_cuda:
        return None
    ext = _load()
    if ext is None:
        raise RuntimeError("the paged cache's operators need the native extension on a GPU")
    return ext


class StepPlan(NamedTuple):
    """Where one step's new tokens go. T tokens, packed by request; B requests."""

    slots: torch.Tensor  # int32 [T]: page * page_size + place in the page; -1 where a token got none
    positions: torch.Tensor  # int32 [T]: place in the token's request; 0 where it got no slot
    cu_new: torch.Tensor  # int32 [B + 1]: request r's tokens are rows cu_new[r] .. cu_new[r + 1] - 1
    kv_lens: torch.Tensor  # int32 [B]: tokens to attend to after the write; 0 where the request got no slots
    lens: torch.Tensor  # int32 [B]: tokens held after the step
    free_count: torch.Tensor  # int32 [1]: pages left on the free stack


def plan_step(
    tables: torch.Tensor,
    lens: torch.Tensor,
    new_lens: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    page_size: int,
    num_tokens: int,
) -> StepPlan:
    """Slots for the new tokens of a step, pages taken from the free stack.

    tables [B, M], lens [B] (tokens held), new_lens [B] (tokens that come;
    0 for an idle row), free_pages [N] (a stack, its top at
    free_count[0] - 1), free_count [1], all int32; B at most 4096. The new
    tokens are packed by request into ``num_tokens`` rows; rows behind the
    last get slot -1.

    A request is served whole or not at all: it gets nothing if its row has
    no room for its tokens, its rows pass ``num_tokens``, or the stack has
    too few pages for it and those before it; so once one finds too few,
    none behind it that needs a page gets one. Its slots are then -1, its
    kv_lens 0, and it holds what it held. New entries of ``tables`` are
    written in place; lens and free_count come back anew, so a step counts
    once the caller stores them (``PagedKVCache.plan`` does)."""
    ext = _native(tables)
    if ext is not None:
        return StepPlan(*ext.plan_step(tables, lens, new_lens, free_pages, free_count, page_size, num_tokens))
    return _plan_plain(tables, lens, new_lens, free_pages, free_count, page_size, num_tokens)


def release_pages(
    tables: torch.Tensor,
    lens: torch.Tensor,
    done: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    page_size: int,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The pages of the requests marked in ``done`` (bool [B]) back onto the
    free stack, in the order of the requests: returns (lens, free_count),
    lens 0 where done. free_pages is written in place above its top. Store
    both before the next call: a request given back twice would have its
    pages on the stack twice."""
    ext = _native(tables)
    if ext is not None:
        return tuple(ext.release_pages(tables, lens, done, free_pages, free_count, page_size))
    return _release_plain(tables, lens, done, free_pages, free_count, page_size)


def write_kv(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> None:
    """cache[slot of t] = k[t], v[t] for k, v [T, kv heads, head dim] (rows
    and heads may be strided: slices of one fused projection do). Tokens
    whose slot is negative or past the cache are skipped. An 8-bit cache
    holds the value divided by its scale, clamped to +-448, rounded to the
    nearest. Slots must differ: which of two tokens with one slot stays is
    not defined (``plan_step`` gives none twice). k and v must not lie in the
    places that are written."""
    ext = _native(k)
    if ext is not None:
        ext.write_kv(k, v, k_cache, v_cache, slots, k_scale, v_scale)
        return
    _write_plain(k, v, k_cache, v_cache, slots, k_scale, v_scale)


def decode_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    tables: torch.Tensor,
    kv_lens: torch.Tensor,
    scale: Optional[float] = None,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """softmax(scale * q k^T) v for one token of each request: q
    [B, heads, head dim], row r over the first kv_lens[r] tokens of request
    r. heads is a multiple of the cache's; head h reads kv head
    h // (heads // kv heads). scale is 1 / sqrt(head dim) if not given. A
    row with no tokens gives zeros; scores that are NaN, or all -inf, give
    NaN, however the keys are split. ``out`` (contiguous) is written if
    given."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ext = _native(q)
    if ext is not None:
        return ext.decode_attention(q, k_cache, v_cache, tables, kv_lens, scale, k_scale, v_scale, out)
    return _attend_plain(q, k_cache, v_cache, tables, kv_lens, None, scale, k_scale, v_scale, out)


def prompt_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    tables: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_new: torch.Tensor,
    scale: Optional[float] = None,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention of packed new tokens: q [T, heads, head dim], request
    r's rows cu_new[r] .. cu_new[r + 1] - 1 are its last tokens among its
    kv_lens[r], which the cache holds already (``write_kv`` comes first).
    The j-th of n new rows sees the first kv_lens[r] - n + j + 1 tokens; a
    row that sees none gives zeros, one whose scores are NaN or all -inf NaN.
    Rows behind the last request are zero in
    a new result, and left as they are in ``out`` (contiguous)."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ext = _native(q)
    if ext is not None:
        return ext.prompt_attention(q, k_cache, v_cache, tables, kv_lens, cu_new, scale, k_scale, v_scale, out)
    return _attend_plain(q, k_cache, v_cache, tables, kv_lens, cu_new, scale, k_scale, v_scale, out)


class PagedKVCache:
    """Pages, block tables and lengths of up to ``requests`` requests, for
    all layers of one model. A step:

        plan = cache.plan(new_lens, num_tokens)   # once, commits the step
        for layer in range(layers):
            cache.write(layer, k, v, plan)
            o = cache.decode(layer, q, plan)      # or cache.prompt(...)

    and ``cache.release(done)`` when requests end. ``decode`` takes one row
    of q for each request of the cache; if only some have a new token, their
    rows alone, with ``active=cache.active(plan, rows)``. plan, write, decode and
    prompt may be captured into a graph; its replays read and advance the
    same state. Steps of one cache run in order, on one stream at a time."""

    def __init__(
        self,
        layers: int,
        kv_heads: int,
        head_dim: int,
        pages: int,
        page_size: int = 64,
        requests: int = 32,
        max_len: int = 2048,
        dtype: torch.dtype = torch.bfloat16,
        device: str = "cuda:0",
        k_scale: float = 1.0,
        v_scale: float = 1.0,
    ):
        if min(layers, kv_heads, pages, requests, max_len) < 1:
            raise ValueError("layers, kv_heads, pages, requests and max_len must be positive")
        self.page_size, self.k_scale, self.v_scale = _page_size(page_size), k_scale, v_scale
        shape = (layers, pages, kv_heads, page_size, head_dim)
        like = torch.empty(shape, dtype=dtype, device="meta")
        _check_caches(like[0], like[0], like[0])
        _check_scales(like, k_scale, v_scale)
        _check_table(torch.empty((requests, self.pages_for(max_len)), dtype=torch.int32, device="meta"), like, page_size)
        # zeros, not what the memory held: no page is read before it is written, but dumps and snapshots see all
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        ints = dict(dtype=torch.int32, device=device)
        self.tables = torch.full((requests, self.pages_for(max_len)), -1, **ints)
        self._state = torch.zeros(requests + 1, **ints)
        self._state[requests] = pages
        self.lens, self.free_count = self._state[:requests], self._state[requests:]
        self.free_pages = torch.arange(pages, **ints)

    @property
    def pages(self) -> int:
        return self.free_pages.shape[0]

    def pages_for(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def plan(self, new_lens: torch.Tensor, num_tokens: int) -> StepPlan:
        """plan_step for this cache, its lengths and free stack advanced."""
        plan = plan_step(
            self.tables, self.lens, new_lens, self.free_pages, self.free_count, self.page_size, num_tokens
        )
        self.lens.copy_(plan.lens)
        self.free_count.copy_(plan.free_count)
        return plan

    def release(self, done: torch.Tensor) -> None:
        """Ends the requests marked in done (bool [requests])."""
        lens, count = release_pages(
            self.tables, self.lens, done, self.free_pages, self.free_count, self.page_size
        )
        self.lens.copy_(lens)
        self.free_count.copy_(count)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: StepPlan) -> None:
        write_kv(k, v, self.k[layer], self.v[layer], plan.slots, self.k_scale, self.v_scale)

    def active(self, plan: StepPlan, rows: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Tables and lengths of the requests ``rows`` (int64, ascending as
        the plan packs them), for all layers of a decode step."""
        return self.tables[rows], plan.kv_lens[rows]

    def decode(
        self,
        layer: int,
        q: torch.Tensor,
        plan: StepPlan,
        scale: Optional[float] = None,
        active: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
    ) -> torch.Tensor:
        tables, kv_lens = (self.tables, plan.kv_lens) if active is None else active
        return decode_attention(
            q, self.k[layer], self.v[layer], tables, kv_lens, scale, self.k_scale, self.v_scale
        )

    def prompt(self, layer: int, q: torch.Tensor, plan: StepPlan, scale: Optional[float] = None) -> torch.Tensor:
        return prompt_attention(
            q, self.k[layer], self.v[layer], self.tables, plan.kv_lens, plan.cu_new, scale, self.k_scale, self.v_scale
        )


# -- the plain path of CPU tensors ------------------------------------------


def _require(ok: bool, message: str, error=ValueError) -> None:
    if not ok:
        raise error(message)


def _page_size(page_size: int) -> int:
    _require(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}, is {page_size}")
    return page_size


def _check(t: torch.Tensor, like: torch.Tensor, name: str) -> None:
    _require(t.device == like.device, f"{name} must be on {like.device}, is on {t.device}")
    _require(
        not (torch.is_grad_enabled() and t.requires_grad),
        f"{name} requires a gradient: the paged cache's operators have none",
        RuntimeError,
    )


def _check_ints(t: torch.Tensor, like: torch.Tensor, dims: int, name: str) -> None:
    _check(t, like, name)
    _require(t.dtype == torch.int32, f"{name} must be int32, is {t.dtype}", TypeError)
    _require(
        t.dim() == dims and (t.numel() == 0 or t.stride(-1) == 1),
        f"{name} must have {dims} dimension(s), the last without gaps",
    )


def _check_table(tables: torch.Tensor, like: torch.Tensor, page_size: int) -> None:
    _page_size(page_size)
    _check_ints(tables, like, 2, "tables")
    _require(tables.shape[0] <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests, got {tables.shape[0]}")
    _require(
        tables.shape[1] >= 1 and tables.shape[1] * page_size <= 2**30,
        "a table row must name at least 1 and at most 2^30 slots",
    )


def _check_stack(tables, lens, other, name, free_pages, free_count, page_size) -> None:
    _check_table(tables, tables, page_size)
    n = tables.shape[0]
    _require(n >= 1, "tables must have a row")
    _require(n == 1 or tables.stride(0) >= tables.shape[1], "the rows of tables must not overlap")
    _check_ints(lens, tables, 1, "lens")
    _check_ints(free_pages, tables, 1, "free_pages")
    _check_ints(free_count, tables, 1, "free_count")
    _check(other, tables, name)
    _require(
        lens.shape[0] == n and other.shape == (n,),
        f"lens and {name} must have one value for each of the {n} rows of tables",
    )
    _require(free_count.shape[0] == 1, "free_count must have one value")
    _require(free_pages.shape[0] * page_size < 2**31, "the cache must have fewer than 2^31 slots")


def _check_caches(k_cache, v_cache, like) -> None:
    _check(k_cache, like, "k_cache")
    _check(v_cache, like, "v_cache")
    _require(
        k_cache.dim() == 4 and k_cache.shape == v_cache.shape,
        "k_cache and v_cache must be [pages, kv heads, page size, head dim] of one shape",
    )
    _require(k_cache.is_contiguous() and v_cache.is_contiguous(), "k_cache and v_cache must be contiguous")
    _require(
        k_cache.dtype == v_cache.dtype and k_cache.dtype in (like.dtype, torch.float8_e4m3fn),
        f"k_cache and v_cache must both be {like.dtype} or float8_e4m3fn",
        TypeError,
    )
    pages, heads, page_size, dim = k_cache.shape
    _page_size(page_size)
    _require(pages >= 1 and heads >= 1, "the cache must have a page and a head")
    _require(pages * page_size < 2**31, "the cache must have fewer than 2^31 slots")
    _require(pages * page_size * heads < 2**32, "the cache must have fewer than 2^32 rows of a head")
    _require(
        dim % 8 == 0 and 8 <= dim <= MAX_HEAD_DIM,
        f"head dim must be a multiple of 8, at most {MAX_HEAD_DIM}, is {dim}",
    )


def _check_scales(cache, k_scale, v_scale) -> None:
    for name, x in (("k_scale", k_scale), ("v_scale", v_scale)):
        _require(
            2.0**-126 <= x <= 2.0**126, f"{name} must be a positive number that fits 32 bits, and its inverse too, is {x}"
        )
    _require(
        cache.dtype == torch.float8_e4m3fn or (k_scale == 1.0 and v_scale == 1.0),
        "only a float8_e4m3fn cache has scales",
    )


def _plan_plain(tables, lens, new_lens, free_pages, free_count, page_size, num_tokens) -> StepPlan:
    _check_stack(tables, lens, new_lens, "new_lens", free_pages, free_count, page_size)
    _check_ints(new_lens, tables, 1, "new_lens")
    _require(0 <= num_tokens < 2**31, f"num_tokens must be 0 or more and fit 31 bits, is {num_tokens}")
    n, width = tables.shape
    pool = free_pages.shape[0]
    available = min(max(int(free_count[0]), 0), pool)
    slots = torch.full((num_tokens,), -1, dtype=torch.int32)
    positions = torch.zeros(num_tokens, dtype=torch.int32)
    cu, kv_lens, after = [0], [], []
    wanted = taken = 0
    for r, (held, new) in enumerate(zip(lens.tolist(), new_lens.tolist())):
        held, new = min(max(held, 0), width * page_size), max(new, 0)
        start = cu[-1]
        cu.append(start + new)
        fits = new > 0 and held + new <= width * page_size and cu[-1] <= num_tokens
        have, want = -(-held // page_size), -(-(held + new) // page_size)
        wanted += want - have if fits else 0
        if fits and (want == have or wanted <= available):
            for c in range(have, want):
                tables[r, c] = free_pages[available - 1 - taken]
                taken += 1
            at = torch.arange(held, held + new)
            page = tables[r, at // page_size].long()
            known = (page >= 0) & (page < pool)
            slots[start : cu[-1]] = torch.where(known, page * page_size + at % page_size, -1).to(torch.int32)
            positions[start : cu[-1]] = at.to(torch.int32)
            kv_lens.append(held + new)
            after.append(held + new)
        else:
            kv_lens.append(0)
            after.append(held)
    ints = lambda x: torch.tensor(x, dtype=torch.int64).clamp(max=2**31 - 1).to(torch.int32)  # noqa: E731
    return StepPlan(slots, positions, ints(cu), ints(kv_lens), ints(after), ints([available - taken]))


def _release_plain(tables, lens, done, free_pages, free_count, page_size):
    _check_stack(tables, lens, done, "done", free_pages, free_count, page_size)
    _require(done.dtype == torch.bool, f"done must be bool, is {done.dtype}", TypeError)
    pool, width = free_pages.shape[0], tables.shape[1]
    count = min(max(int(free_count[0]), 0), pool)
    after = lens.clamp(0, width * page_size)
    for r in done.nonzero()[:, 0].tolist():
        given = -(-int(after[r]) // page_size)
        kept = min(given, pool - count)
        free_pages[count : count + kept] = tables[r, :kept]
        count += kept
        after[r] = 0
    return after, torch.tensor([count], dtype=torch.int32)


def _write_plain(k, v, k_cache, v_cache, slots, k_scale, v_scale) -> None:
    _check(k, k, "k")
    _check(v, k, "v")
    _require(k.is_floating_point(), f"k must be a floating type, is {k.dtype}", TypeError)
    _require(v.dtype == k.dtype, f"v must be {k.dtype} like k, is {v.dtype}", TypeError)
    _check_caches(k_cache, v_cache, k)
    pages, heads, page_size, dim = k_cache.shape
    _require(
        k.dim() == 3 and k.shape == v.shape and k.shape[1:] == (heads, dim),
        f"k and v must be [tokens, {heads}, {dim}] for this cache",
    )
    _require(k.shape[0] < min(2**31, 2**32 // (heads * (dim // 8))), "too many tokens")
    _require(
        k.numel() == 0 or (k.stride(2) == 1 and v.stride(2) == 1), "k and v must have no gaps along the head dim"
    )
    _check_ints(slots, k, 1, "slots")
    _require(
        slots.shape[0] == k.shape[0],
        f"slots must have one value for each of the {k.shape[0]} tokens, has {slots.shape[0]}",
    )
    _check_scales(k_cache, k_scale, v_scale)
    kept = ((slots >= 0) & (slots < pages * page_size)).nonzero()[:, 0]
    at = slots[kept].long()
    for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        value = x[kept]
        if cache.dtype == torch.float8_e4m3fn:
            inverse = (1.0 / torch.tensor(scale, dtype=torch.float32)).item()
            value = (value.float() * inverse).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
            cache, value = cache.view(torch.uint8), value.view(torch.uint8)
        cache[at // page_size, :, at % page_size] = value


def _attend_plain(q, k_cache, v_cache, tables, kv_lens, cu_new, scale, k_scale, v_scale, out):
    _check(q, q, "q")
    _require(q.is_floating_point(), f"q must be a floating type, is {q.dtype}", TypeError)
    _check_caches(k_cache, v_cache, q)
    pages, kv_heads, page_size, dim = k_cache.shape
    _require(q.dim() == 3 and q.shape[2] == dim, f"q must be [rows, heads, {dim}] for this cache")
    rows, heads = q.shape[:2]
    _require(heads <= 65535 and (not heads or rows < 2**31 // heads), "too many rows or heads")
    _require(
        heads >= 1 and heads % kv_heads == 0, f"q's {heads} heads must be a multiple of the cache's {kv_heads}"
    )
    _require(q.numel() == 0 or q.stride(2) == 1, "q must have no gaps along the head dim")
    _check_table(tables, q, page_size)
    _check_ints(kv_lens, q, 1, "kv_lens")
    requests, width = tables.shape
    _require(
        kv_lens.shape[0] == requests, f"kv_lens must have one value for each of the {requests} rows of tables"
    )
    if cu_new is not None:
        _check_ints(cu_new, q, 1, "cu_new")
        _require(cu_new.shape[0] == requests + 1, f"cu_new must have {requests + 1} values, has {cu_new.shape[0]}")
        tiles = rows * (heads // kv_heads) // 128 + requests
        _require((tiles + 256) * kv_heads < 2**24, "too many rows, requests or heads")
    else:
        _require(rows == requests, f"q must have one row for each of the {requests} rows of tables")
    _check_scales(k_cache, k_scale, v_scale)
    _require(abs(scale * k_scale * math.log2(math.e)) < 2.0**128, "scale must be finite, also by k_scale in 32 bits")
    if out is not None:
        _check(out, q, "out")
        _require(out.dtype == q.dtype, f"out must be {q.dtype} like q, is {out.dtype}", TypeError)
        _require(out.shape == q.shape and out.is_contiguous(), "out must be contiguous and of q's shape")
        if q.numel():
            span = sum((n - 1) * s for n, s in zip(q.shape, q.stride())) + 1
            a, b, size = out.data_ptr(), q.data_ptr(), q.element_size()
            _require(a + out.numel() * size <= b or b + span * size <= a, "out must not overlap q")
    else:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    work = torch.float64 if q.dtype == torch.float64 else torch.float32
    ends = cu_new.tolist() if cu_new is not None else list(range(requests + 1))
    for r, length in enumerate(kv_lens.tolist()):
        first, last = max(ends[r], 0), min(ends[r + 1], rows)
        if last <= first:
            continue
        length = min(max(length, 0), width * page_size)
        at = torch.arange(length)
        page = tables[r, at // page_size].long()
        known = (page >= 0) & (page < pages)
        # absent tokens take a present token's place in the product and are masked
        page = torch.where(known, page, 0)
        group = heads // kv_heads
        k = k_cache.view(torch.uint8) if k_cache.dtype == torch.float8_e4m3fn else k_cache
        v = v_cache.view(torch.uint8) if v_cache.dtype == torch.float8_e4m3fn else v_cache
        k = k[page, :, at % page_size].view(k_cache.dtype).to(work).repeat_interleave(group, dim=1) * k_scale
        v = v[page, :, at % page_size].view(v_cache.dtype).to(work).repeat_interleave(group, dim=1) * v_scale
        seen = known[None] & (at[None] <= torch.arange(length - (ends[r + 1] - first), length + last - ends[r + 1])[:, None])
        scores = torch.matmul(q[first:last].to(work).transpose(0, 1), k.permute(1, 2, 0)) * scale
        scores = scores.masked_fill(~seen, -math.inf)
        any_seen = seen.any(-1)[None, :, None]
        p = torch.softmax(torch.where(any_seen, scores, 0.0), dim=-1).masked_fill(~seen, 0.0)
        # a token that a row does not see adds nothing to it, infinities and NaN included: 0 * inf would
        finite = torch.isfinite(v).all(-1).all(-1)
        o = torch.matmul(p, torch.where(finite[:, None, None], v, 0.0).transpose(0, 1))
        for j in (~finite).nonzero()[:, 0].tolist():
            o = torch.where(seen[None, :, j, None], o + p[:, :, j, None] * v[j][:, None], o)
        out[first:last] = o.transpose(0, 1).to(q.dtype)
    return out
