"""The paged key-value cache's operators, measured: the step's plan, the write, one token's attention, the prompt's attention.

A cache holds keys and values as [pages, kv heads, page size, head dim]; `tables[request, i]` is the page of the request's tokens
i * page_size and on. `run` computes each operator from elementary torch operations, or, where `own` is true, with beta9_amd.ops.paged.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "fp16": 2, "e4m3": 1}
E4M3_MAX = 448.0


# ---- cases ----------------------------------------------------------------


def listed():
    return [
        # one decode step of the LLM server at its full batch (32 sequences, at most 2048 tokens each)
        dict(name="plan_decode", op="plan", kind="decode", requests=32, longest=2048, new=1, page=64, room=1.0),
        # a full queue of prompts admitted at once, the pool too small for the last of them
        dict(name="plan_prompts", op="plan", kind="prompts", requests=509, longest=1024, new=1000, page=16, room=0.9),
        # pages of a quarter of the sequences given back
        dict(name="release", op="release", requests=256, longest=8192, page=64),
        # the new token of each sequence, per layer of the transformer model (8 kv heads of 128)
        dict(name="write_decode", op="write", tokens=32, heads=32, kv=8, dim=128, page=64, type="bf16", cache="bf16"),
        # a chunk of prompts, of an odd length, into an 8-bit cache
        dict(name="write_prompts_e4m3", op="write", tokens=16381, heads=32, kv=8, dim=128, page=64, type="bf16", cache="e4m3"),
        # a single chat a few hundred tokens in, on the LLM server's default model (16 heads of 64): latency counts
        dict(name="decode_one", op="decode", requests=1, longest=333, even=True, heads=16, kv=16, dim=64, page=16, type="fp16", cache="fp16"),
        # the server's batch of 32 at ragged lengths, on the transformer model's heads
        dict(name="decode_batch", op="decode", requests=32, longest=2048, even=False, heads=32, kv=8, dim=128, page=64, type="bf16", cache="bf16"),
        # one very long document under question
        dict(name="decode_long", op="decode", requests=1, longest=131071, even=True, heads=32, kv=8, dim=128, page=64, type="bf16", cache="bf16"),
        # a full card: many ragged requests on an 8-bit cache
        dict(name="decode_full_e4m3", op="decode", requests=128, longest=8192, even=False, heads=32, kv=8, dim=128, page=128, type="bf16", cache="e4m3"),
        # the benchmark's request: 256 tokens of one prompt
        dict(name="prompt_256", op="prompt", requests=1, new=256, held=0, even=True, heads=32, kv=8, dim=128, page=64, type="bf16", cache="bf16"),
        # ragged prompts behind a cached beginning, on the LLM server's default heads
        dict(name="prompt_ragged", op="prompt", requests=13, new=1500, held=700, even=False, heads=16, kv=16, dim=64, page=32, type="fp16", cache="fp16"),
        # one long document read at once
        dict(name="prompt_long", op="prompt", requests=1, new=8192, held=0, even=True, heads=32, kv=8, dim=128, page=64, type="bf16", cache="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["plan", "release", "write", "decode", "decode", "prompt", "prompt"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        kind = rng.choice(["decode", "prompts"])
        case = dict(op=op, kind=kind, requests=_spread(rng, 1, 509), longest=_spread(rng, 16, 4096),
                    new=1 if kind == "decode" else _spread(rng, 8, 1000), page=page, room=rng.choice([1.0, 1.0, 0.8]))
        return case
    if op == "release":
        return dict(op=op, requests=_spread(rng, 1, 256), longest=_spread(rng, 16, 8192), page=page)
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 16, 64), (16, 16, 128), (16, 2, 64), (40, 8, 128), (24, 1, 64)])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    cache = rng.choice([kind, kind, "e4m3"])
    case = dict(op=op, heads=heads, kv=kv, dim=dim, page=page, type=kind, cache=cache)
    if op == "write":
        return dict(case, tokens=_spread(rng, 1, 16381))
    if op == "decode":
        requests = _spread(rng, 1, 128)
        tokens = 2_000_000 // (requests * max(kv, heads // 4))
        return dict(case, requests=requests, longest=_spread(rng, 1, min(131071, tokens)), even=rng.random() < 0.3)
    requests = _spread(rng, 1, 16)
    new = _spread(rng, 1, int(8192 / math.sqrt(requests) / 2))
    return dict(case, requests=requests, new=new, held=rng.choice([0, _spread(rng, 1, new)]), even=rng.random() < 0.3)


def _lengths(case):
    """[(tokens held, new tokens)] of the case's requests: the sizes belong to the case, their order to the seed."""
    rng = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    op, n = case["op"], case["requests"]
    if op == "plan":
        got = [(rng.randint(0, case["longest"]), 1 if case["kind"] == "decode" else rng.randint(1, case["new"])) for _ in range(n)]
        # some rows idle, as in a batch that is not full
        return [(h, 0) if i and rng.random() < 0.1 else (h, w) for i, (h, w) in enumerate(got)]
    if op == "release":
        return [(rng.randint(1, case["longest"]), 0) for _ in range(n)]
    if op == "decode":
        got = [case["longest"] if case["even"] or not i else rng.randint(1, case["longest"]) for i in range(n)]
        return [(0 if i and not case["even"] and rng.random() < 0.05 else h, 1) for i, h in enumerate(got)]  # 0: an idle row
    full = lambda most, i, low: most if case["even"] or not i else rng.randint(low, most)  # noqa: E731
    return [(full(case["held"], i, 0), full(case["new"], i, 0)) for i in range(n)]


def work(case):
    op = case["op"]
    if op == "write":
        return dict(bytes=case["tokens"] * (4 + 2 * case["kv"] * case["dim"] * (SIZE[case["type"]] + SIZE[case["cache"]])), flops=0)
    lens, page = _lengths(case), case["page"]
    if op == "plan":
        fresh = sum(-(-(h + n) // page) - -(-h // page) for h, n in lens)
        return dict(bytes=8 * len(lens) + 8 * fresh + 8 * sum(n for _, n in lens) + 12 * len(lens), flops=0)
    if op == "release":
        return dict(bytes=9 * len(lens) + 8 * sum(-(-h // page) for h, _ in lens) // 4, flops=0)
    width = case["dim"] * SIZE[case["cache"]]
    if op == "decode":
        tokens, pairs, rows = sum(h for h, _ in lens), sum(h for h, _ in lens), len(lens)
    else:
        tokens, rows = sum(h + n for h, n in lens), sum(n for _, n in lens)
        pairs = sum(h * n + n * (n + 1) // 2 for h, n in lens)
    return dict(bytes=2 * tokens * case["kv"] * width + 2 * rows * case["heads"] * case["dim"] * SIZE[case["type"]],
                flops=4 * case["dim"] * case["heads"] * pairs)


# ---- inputs ---------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(lens, page, width, pages, gen):
    """Block tables over shuffled pages, and the pages left, as a stack."""
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    counts = _ints([-(-n // page) for n in lens])
    column = torch.arange(width, device="cuda", dtype=torch.int32)
    held = column[None] < counts[:, None]
    place = (counts.cumsum(0) - counts)[:, None] + column[None]
    tables = torch.where(held, order[torch.where(held, place, 0).long()], -1).to(torch.int32)
    return tables, order[int(counts.sum()):].contiguous()


def _normal(shape, gen, kind, columns=None):
    x = torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32)
    if columns is not None:
        x = x * columns  # a few channels of the keys are larger than the others, as in trained models
    return x.to(TYPES[kind])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, page = case["op"], case["page"]
    state = dict(op=op, page=page)
    if op == "write":
        heads, kv, dim, tokens = case["heads"], case["kv"], case["dim"], case["tokens"]
        qkv = _normal((tokens, heads + 2 * kv, dim), gen, case["type"])
        pages = -(-tokens // page) + 3
        slots = torch.randperm(pages, device="cuda", generator=gen)[:, None] * page + torch.arange(page, device="cuda")[None]
        slots = slots.reshape(-1)[:tokens] if tokens > pages else torch.randperm(pages * page, device="cuda", generator=gen)[:tokens]
        state["slots"] = slots.to(torch.int32)
        if tokens > 8:
            state["slots"][tokens // 2] = -1  # a token without a page
        state["k"], state["v"] = qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        state["k_cache"] = torch.zeros((pages, kv, page, dim), device="cuda", dtype=TYPES[case["cache"]])
        state["v_cache"] = torch.zeros_like(state["k_cache"])
        state["scales"] = (0.0123, 0.0117) if case["cache"] == "e4m3" else (1.0, 1.0)
        return state
    lens = _lengths(case)
    random.Random(seed).shuffle(lens)
    if op in ("plan", "release"):
        held = [h for h, _ in lens]
        fresh = sum(-(-(h + n) // page) - -(-h // page) for h, n in lens)
        spare = int(case.get("room", 1.0) * fresh)
        pages = sum(-(-h // page) for h in held) + spare + 1
        width = -(-(case["longest"] + case.get("new", 0)) // page)
        state["tables"], free = _tables(held, page, width, pages, gen)
        state["lens"], state["free"] = _ints(held), torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        state["free"][: len(free)] = free
        state["free_count"] = _ints([len(free)])
        if op == "plan":
            state["new"], state["tokens"] = _ints([n for _, n in lens]), sum(n for _, n in lens)
        else:
            state["done"] = torch.rand(len(lens), device="cuda", generator=gen) < 0.25
        return state
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    total = [h if op == "decode" else h + n for h, n in lens]
    pages = sum(-(-n // page) for n in total) + 1
    state["tables"], _ = _tables(total, page, -(-max(total) // page), pages, gen)
    columns = torch.ones(dim, device="cuda")
    columns[3::29] = 2.5
    state["scales"] = (0.031, 0.019) if case["cache"] == "e4m3" else (1.0, 1.0)
    state["k_cache"] = torch.empty((pages, kv, page, dim), device="cuda", dtype=TYPES[case["cache"]])
    state["v_cache"] = torch.empty_like(state["k_cache"])
    for first in range(0, pages, 1 << 12):
        for cache, scale, wide in ((state["k_cache"], state["scales"][0], columns), (state["v_cache"], state["scales"][1], None)):
            part = cache[first:first + (1 << 12)]
            x = torch.randn(part.shape, device="cuda", generator=gen)
            x = (x if wide is None else x * wide) / scale
            part.copy_(x.clamp(-E4M3_MAX, E4M3_MAX) if case["cache"] == "e4m3" else x)
    state["kv_lens"] = _ints(total)
    rows = len(lens) if op == "decode" else sum(n for _, n in lens)
    qkv = _normal((rows, heads + 2 * kv, dim), gen, case["type"])
    state["q"] = qkv[:, :heads]
    if op == "prompt":
        ends = [0]
        for _, n in lens:
            ends.append(ends[-1] + n)
        state["cu_new"], state["most"] = _ints(ends), max(n for _, n in lens)
    return state


# ---- one pass -------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plan, "release": _release, "write": _write, "decode": _decode, "prompt": _prompt}[state["op"]](state)


def _run_own(s):
    from beta9_amd.ops import paged

    if s["op"] == "plan":
        p = paged.plan_step(s["tables"], s["lens"], s["new"], s["free"], s["free_count"], s["page"], s["tokens"])
        return [s["tables"], p.slots, p.positions, p.cu_new, p.kv_lens, p.lens, p.free_count]
    if s["op"] == "release":
        lens, count = paged.release_pages(s["tables"], s["lens"], s["done"], s["free"], s["free_count"], s["page"])
        return [s["free"], lens, count]
    if s["op"] == "write":
        paged.write_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["scales"][0], v_scale=s["scales"][1])
        return [s["k_cache"], s["v_cache"]]
    more = dict(k_scale=s["scales"][0], v_scale=s["scales"][1])
    if s["op"] == "decode":
        return paged.decode_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], **more)
    return paged.prompt_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu_new"], **more)


def _plan(s):
    tables, lens, new, page, tokens = s["tables"], s["lens"], s["new"], s["page"], s["tokens"]
    device, width = tables.device, tables.shape[1]
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32, device=device)
    cu[1:] = new.cumsum(0)
    have, want = (lens + page - 1) // page, (lens + new + page - 1) // page
    fits = (new > 0) & (lens + new <= width * page) & (cu[1:] <= tokens)
    need = torch.where(fits, want - have, 0)
    taken = need.cumsum(0)
    granted = fits & ((need == 0) | (taken <= s["free_count"]))
    need = torch.where(granted, need, 0)
    # the k-th page taken lies k below the stack's top
    column = torch.arange(width, device=device)
    place = s["free_count"] - 1 - ((taken - need)[:, None] + column[None] - have[:, None])
    fresh = (column[None] >= have[:, None]) & (column[None] < (have + need)[:, None])
    tables.copy_(torch.where(fresh, s["free"][torch.where(fresh, place, 0)], tables))
    t = torch.arange(tokens, device=device)
    request = torch.searchsorted(cu[1:].contiguous(), t.to(torch.int32), right=True).clamp(max=len(lens) - 1)
    at = lens[request] + t - cu[request]
    page_of = tables[request, torch.where(granted[request], at // page, 0)]
    ok = granted[request] & (t < cu[-1])
    slots = torch.where(ok, page_of * page + at % page, -1).to(torch.int32)
    positions = torch.where(ok, at, 0).to(torch.int32)
    after = torch.where(granted, lens + new, lens)
    count = s["free_count"] - need.sum()
    return [tables, slots, positions, cu, torch.where(granted, after, 0), after, count.to(torch.int32)]


def _release(s):
    tables, lens, done, page = s["tables"], s["lens"], s["done"], s["page"]
    give = torch.where(done, (lens + page - 1) // page, 0)
    column = torch.arange(tables.shape[1], device=tables.device)
    given = column[None] < give[:, None]
    place = s["free_count"] + (give.cumsum(0) - give)[:, None] + column[None]
    s["free"].index_put_((place[given].long(),), tables[given])
    return [s["free"], torch.where(done, 0, lens), (s["free_count"] + give.sum()).to(torch.int32)]


def _write(s):
    kept = (s["slots"] >= 0).nonzero()[:, 0]
    slots = s["slots"][kept].long()
    for_cache = lambda x, scale: x[kept].float() if scale == 1.0 else (x[kept].float() / scale).clamp(-E4M3_MAX, E4M3_MAX)  # noqa: E731
    page = s["page"]
    kind = s["k_cache"].dtype
    # 8-bit floats are moved as whole numbers: torch's indexed write does not take them
    raw = torch.uint8 if kind == torch.float8_e4m3fn else torch.int16
    s["k_cache"].view(raw)[slots // page, :, slots % page] = for_cache(s["k"], s["scales"][0]).to(kind).view(raw)
    s["v_cache"].view(raw)[slots // page, :, slots % page] = for_cache(s["v"], s["scales"][1]).to(kind).view(raw)
    return [s["k_cache"], s["v_cache"]]


def _gathered(cache, tables, scale):
    """[requests, kv heads, tokens, dim] in 32 bits."""
    # a part of a row that holds no page reads page 0 and is masked
    got = cache.view(torch.uint8)[tables.clamp(min=0).long()].view(cache.dtype)
    b, m, kv, page, dim = got.shape
    return got.permute(0, 2, 1, 3, 4).reshape(b, kv, m * page, dim).float() * scale


def _softmax_product(scores, seen, values):
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, values) / torch.where(total == 0, 1.0, total)


def _decode(s):
    q, tables = s["q"], s["tables"]
    b, heads, dim = q.shape
    k, v = _gathered(s["k_cache"], tables, s["scales"][0]), _gathered(s["v_cache"], tables, s["scales"][1])
    kv, tokens = k.shape[1], k.shape[2]
    grouped = q.float().reshape(b, kv, heads // kv, dim)
    scores = torch.matmul(grouped, k.transpose(-1, -2)) * dim**-0.5
    seen = torch.arange(tokens, device=q.device)[None] < s["kv_lens"][:, None]
    return _softmax_product(scores, seen[:, None, None], v).reshape(b, heads, dim).to(q.dtype)


def _prompt(s):
    q, tables, cu, most = s["q"], s["tables"], s["cu_new"].long(), s["most"]
    rows, heads, dim = q.shape
    k, v = _gathered(s["k_cache"], tables, s["scales"][0]), _gathered(s["v_cache"], tables, s["scales"][1])
    b, kv, tokens = k.shape[:3]
    new = cu[1:] - cu[:-1]
    column = torch.arange(most, device=q.device)
    real = column[None] < new[:, None]
    row = (cu[:-1, None] + column[None]).clamp(max=rows - 1)
    padded = q.float()[row].reshape(b, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dim)
    scores = (torch.matmul(padded, k.transpose(-1, -2)) * dim**-0.5).reshape(b, kv, heads // kv, most, tokens)
    position = (s["kv_lens"] - new)[:, None] + column[None]
    key = torch.arange(tokens, device=q.device)
    seen = (key[None, None] <= position[:, :, None]) & (key[None, None] < s["kv_lens"][:, None, None])
    o = _softmax_product(scores, seen[:, None, None], v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(b, most, heads, dim)
    return o[real].to(q.dtype)  # requests in order, each with its own tokens in order: the packed rows


# ---- the definition in 64 bits --------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("plan", "release"):
        return None
    page = s["page"]
    if case["op"] == "write":
        out = []
        for x, cache, scale in ((s["k"], s["k_cache"], s["scales"][0]), (s["v"], s["v_cache"], s["scales"][1])):
            flat = cache.double().permute(0, 2, 1, 3).reshape(-1, cache.shape[1], cache.shape[3])
            for first in range(0, case["tokens"], 4096):
                at = s["slots"][first:first + 4096].long()
                value = x[first:first + 4096].double()
                if cache.dtype == torch.float8_e4m3fn:
                    value = (value / scale).clamp(-E4M3_MAX, E4M3_MAX)
                flat[at[at >= 0]] = value[at >= 0]
            out.append(flat.reshape(cache.shape[0], page, cache.shape[1], cache.shape[3]).permute(0, 2, 1, 3))
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    lens = s["kv_lens"].tolist()
    ends = s["cu_new"].tolist() if case["op"] == "prompt" else list(range(len(lens) + 1))
    for i, n in enumerate(lens):
        held = s["tables"][i, : -(-n // page)].long()
        first, last = ends[i], ends[i + 1]
        for h in range(kv):
            k = s["k_cache"][:, h].view(torch.uint8)[held].view(s["k_cache"].dtype).reshape(-1, dim)[:n].double() * s["scales"][0]
            v = s["v_cache"][:, h].view(torch.uint8)[held].view(s["v_cache"].dtype).reshape(-1, dim)[:n].double() * s["scales"][1]
            for g in range(h * heads // kv, (h + 1) * heads // kv):
                x = s["q"][first:last, g].double() @ k.T / math.sqrt(dim)
                if last - first > 1:
                    late = torch.arange(n, device="cuda")[None] > torch.arange(n - (last - first), n, device="cuda")[:, None]
                    x[late] = -math.inf
                out[first:last, g] = torch.softmax(x, dim=-1) @ v
    return out
