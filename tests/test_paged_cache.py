"""The paged key-value cache's operators against plain implementations in 64
bits, on CPU tensors and, marked gpu, through the gfx950 kernels."""

import math
import random

import pytest

torch = pytest.importorskip("torch")

from beta9_amd.ops import paged  # noqa: E402

DEVICES = [
    "cpu",
    pytest.param(
        "cuda",
        marks=[pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs MI355X")],
    ),
]
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
both = pytest.mark.parametrize("device", DEVICES)


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def cache_like(x, dtype, scale):
    """x as an 8-bit cache or a plain one holds it."""
    if dtype == torch.float8_e4m3fn:
        return (x.float() / scale).clamp(-448, 448).to(dtype)
    return x.to(dtype)


def values_of(cache, scale=1.0):
    return cache.cpu().to(torch.float64) * scale


# -- plan and release -------------------------------------------------------


def plan_oracle(tables, lens, new, stack, page, tokens):
    """plan_step on lists. `stack`: the free pages, the top last."""
    tables, stack = [list(t) for t in tables], list(stack)
    slots, positions, cu, kv, after = [-1] * tokens, [0] * tokens, [0], [], []
    wanted, available = 0, len(stack)
    for r in range(len(lens)):
        start, end = cu[-1], cu[-1] + new[r]
        cu.append(end)
        have, want = math.ceil(lens[r] / page), math.ceil((lens[r] + new[r]) / page)
        ok = new[r] > 0 and want <= len(tables[r]) and end <= tokens
        if ok:
            wanted += want - have
            ok = want == have or wanted <= available
        if ok:
            for c in range(have, want):
                tables[r][c] = stack.pop()
            for j in range(new[r]):
                at = lens[r] + j
                slots[start + j] = tables[r][at // page] * page + at % page
                positions[start + j] = at
        kv.append(lens[r] + new[r] if ok else 0)
        after.append(lens[r] + new[r] if ok else lens[r])
    return tables, slots, positions, cu, kv, after, len(stack)


def plan_inputs(rng, requests, page, longest, most_new, width, spare):
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, longest)]) for _ in range(requests)]
    lens = [min(n, longest, width * page) for n in lens]
    new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(requests)]
    held = sum(math.ceil(n / page) for n in lens)
    pages = list(range(held + spare))
    rng.shuffle(pages)
    tables = []
    for n in lens:
        count = math.ceil(n / page)
        tables.append([pages.pop() for _ in range(count)] + [-1] * (width - count))
    return tables, lens, new, pages, held + spare


@both
@pytest.mark.parametrize(
    "requests,page,longest,most_new,width,spare,short",
    [
        (1, 16, 40, 1, 4, 9, 0),
        (5, 16, 100, 50, 10, 40, 0),
        (33, 64, 500, 70, 9, 20, 0),  # too few pages for some
        (257, 32, 200, 90, 8, 300, 0),  # rows that overflow
        (700, 128, 900, 300, 12, 900, 0),
        (4096, 16, 64, 20, 6, 9000, 0),
        (9, 16, 50, 30, 8, 60, 25),  # fewer token rows than tokens
        (3, 256, 1000, 5000, 30, 0, 0),  # no free page at all
    ],
)
def test_plan_step(device, requests, page, longest, most_new, width, spare, short):
    rng = random.Random(requests * 1000 + page)
    tables, lens, new, stack, pool = plan_inputs(rng, requests, page, longest, most_new, width, spare)
    tokens = max(0, sum(new) - short) + (3 if not short else 0)
    want = plan_oracle(tables, lens, new, stack, page, tokens)
    # rows of a wider tensor, so that their stride is not their width
    wide = torch.full((requests, width + 3), -7, dtype=torch.int32, device=device)
    t = wide[:, :width]
    t.copy_(ints(tables, device))
    free = ints(stack + [-1] * (pool - len(stack)), device)
    count = ints([len(stack)], device)
    for _ in range(2):  # a plan that is not stored can be made again
        p = paged.plan_step(t, ints(lens, device), ints(new, device), free, count, page, tokens)
        assert t.tolist() == want[0]
        for got, expected in zip(p, want[1:6]):
            assert got.dtype == torch.int32 and got.tolist() == expected
        assert p.free_count.tolist() == [want[6]]
    assert count.tolist() == [len(stack)] and (wide[:, width:] == -7).all()


@both
def test_plan_step_bounds_what_it_reads(device):
    """Values that a caller's mistake leaves on the GPU stay inside the tensors."""
    tables = ints([[0, 99], [-5, 1], [2, 3]], device)
    p = paged.plan_step(
        tables, ints([3, 2, 1000], device), ints([2, 1, 1], device), ints([4, 5, 6, 0, 0, 0, 0], device), ints([50], device), 16, 4
    )
    # row 1 holds a page that the pool does not have; row 2 is full
    assert p.slots.tolist() == [3, 4, -1, -1]
    assert p.cu_new.tolist() == [0, 2, 3, 4] and p.kv_lens.tolist() == [5, 3, 0] and p.lens.tolist() == [5, 3, 32]
    assert p.free_count.tolist() == [7]
    p = paged.plan_step(tables, ints([3, 2, -4], device), ints([-2, 0, 1], device), ints([4, 5], device), ints([-1], device), 16, 1)
    assert p.slots.tolist() == [-1] and p.free_count.tolist() == [0] and p.lens.tolist() == [3, 2, 0]
    p = paged.plan_step(tables, ints([3, 2, 1], device), ints([0, 0, 0], device), ints([4, 5], device), ints([1], device), 16, 0)
    assert p.slots.shape == (0,) and p.kv_lens.tolist() == [0, 0, 0]


@both
@pytest.mark.parametrize("requests,page,longest", [(1, 16, 50), (40, 32, 300), (300, 64, 1000), (4096, 16, 40)])
def test_release_pages(device, requests, page, longest):
    rng = random.Random(requests)
    tables, lens, _, stack, pool = plan_inputs(rng, requests, page, longest, 1, math.ceil(longest / page), 11)
    done = [rng.random() < 0.5 for _ in range(requests)]
    expected = list(stack)
    for r in range(requests):
        if done[r]:
            expected += tables[r][: math.ceil(lens[r] / page)]
    free = ints(stack + [-1] * (pool - len(stack)), device)
    after, count = paged.release_pages(
        ints(tables, device), ints(lens, device), torch.tensor(done, device=device), free, ints([len(stack)], device), page
    )
    assert count.tolist() == [len(expected)]
    assert free.tolist() == expected + [-1] * (pool - len(expected))
    assert after.tolist() == [0 if d else n for d, n in zip(done, lens)]


@both
def test_release_stays_inside_the_stack(device):
    free = ints([7, 7, 7], device)
    after, count = paged.release_pages(
        ints([[1, 2], [5, 6]], device), ints([17, 900], device), torch.tensor([True, True], device=device), free, ints([2], device), 16
    )
    assert free.tolist() == [7, 7, 1] and count.tolist() == [3] and after.tolist() == [0, 0]


# -- write ------------------------------------------------------------------


@both
@pytest.mark.parametrize("kind,cached", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")])
@pytest.mark.parametrize("tokens,heads,dim,page,offset", [(1, 1, 8, 16, 0), (37, 3, 80, 16, 0), (300, 8, 128, 64, 0), (65, 2, 64, 32, 1)])
def test_write_kv(device, kind, cached, tokens, heads, dim, page, offset):
    """Exactly the value, or the nearest e4m3, at each slot, and nothing else changed. offset 1: rows off the 16-byte grid."""
    gen = torch.Generator().manual_seed(tokens)
    fused = (torch.randn((tokens, 2 * heads + 1, dim + offset), generator=gen) * 3).to(TYPES[kind]).to(device)
    k, v = fused[:, :heads, offset:], fused[:, heads : 2 * heads, offset:]
    k[0, 0, :6] = torch.tensor([math.nan, math.inf, -math.inf, 60000.0, -60000.0, 0.0])
    pages = tokens // page + 2
    k_cache = torch.full((pages, heads, page, dim), 1.0).to(TYPES[cached]).to(device)
    v_cache = k_cache.clone()
    slots = torch.randperm(pages * page, generator=gen)[:tokens].to(torch.int32)
    if tokens > 5:
        slots[3], slots[4] = -1, pages * page  # skipped
    scales = (0.03125, 0.5) if cached == "e4m3" else (1.0, 1.0)  # powers of two: the quotient is exact
    before = values_of(k_cache)
    paged.write_kv(k, v, k_cache, v_cache, slots.to(device), *scales)
    for x, cache, scale in ((k, k_cache, scales[0]), (v, v_cache, scales[1])):
        want = before.clone()
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                want[slot // page, :, slot % page] = values_of(cache_like(x[t].cpu(), TYPES[cached], scale))
        assert torch.equal(values_of(cache).nan_to_num(7.5), want.nan_to_num(7.5))
        assert torch.equal(values_of(cache).isnan(), want.isnan())


@both
def test_write_kv_rounds_every_quotient_to_the_nearest(device):
    """All finite bf16 values against the list of e4m3 values, by a scale that is no power of two."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x[x.isfinite()]
    x = torch.cat([x, x.new_zeros(-len(x) % 128)]).reshape(-1, 1, 128)
    scale = 0.37
    k_cache = torch.zeros((len(x) // 16 + 1, 1, 16, 128), device=device).to(torch.float8_e4m3fn)
    v_cache = k_cache.clone()
    paged.write_kv(x.to(device), x.to(device), k_cache, v_cache, torch.arange(len(x), dtype=torch.int32, device=device), scale, 1.0)
    grid = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double()
    grid = grid[grid.isfinite()].unique()
    quotient = (x.double().flatten() / scale).clamp(-448, 448)
    got = values_of(k_cache).reshape(-1)[: quotient.numel()]
    up = torch.searchsorted(grid, quotient).clamp(1, len(grid) - 1)
    nearest = torch.minimum((grid[up] - quotient).abs(), (quotient - grid[up - 1]).abs())
    # 1 / scale and its product with x are rounded to 32 bits, half a step each: a quotient that lies that near to the
    # middle of two values may go to either
    assert ((got - quotient).abs() <= nearest + quotient.abs() * 2 * 2**-24 * 1.01).all()


# -- attention --------------------------------------------------------------


def attention_oracle(q, k_cache, v_cache, tables, kv_lens, cu, scale, k_scale, v_scale):
    """The formula in 64 bits, row by row, and for each result how far off it may be."""
    kind = q.dtype
    half = torch.finfo(kind).eps / 2
    q, k_cache, v_cache = q.cpu().double(), values_of(k_cache, k_scale), values_of(v_cache, v_scale)
    rows, heads, dim = q.shape
    pages, kv_heads, page, _ = k_cache.shape
    out, off = torch.zeros_like(q), torch.zeros_like(q)
    for r, length in enumerate(kv_lens):
        length = max(0, min(length, len(tables[r]) * page))
        first, last = cu[r], min(cu[r + 1], rows)
        at = torch.arange(length)
        entry = torch.tensor(tables[r] + [0], dtype=torch.int64)[at // page]
        known = (entry >= 0) & (entry < pages)
        at, entry = at[known], entry[known]
        for h in range(heads if last > first else 0):
            k, v = k_cache[entry, h * kv_heads // heads, at % page], v_cache[entry, h * kv_heads // heads, at % page]
            x = q[first:last, h]
            sees = at[None] <= torch.arange(length - (cu[r + 1] - first), length + last - cu[r + 1])[:, None]
            any_key = sees.any(1, keepdim=True)
            s = ((x @ k.T) * scale).masked_fill(~sees, -math.inf)
            w = torch.softmax(torch.where(any_key, s, 0.0), 1).masked_fill(~sees, 0.0)
            out[first:last, h] = w @ v
            # Each score is a sum of dim products in 32 bits: off by (dim + 4) half steps of its terms' sizes, and as
            # much, relatively, is its exponential; numerator and denominator both. The exponent's argument in base 2
            # is rounded once more, to half a step of its size. A probability may be rounded to the result's type
            # before its product with v, the sums to 32 bits, the result to its type.
            size = ((x.abs() @ k.abs().T) * abs(scale)).masked_fill(~sees, 0.0).amax(1, keepdim=True) if len(at) else 0.0
            score = (dim + 4 + 2) * 2**-24 * size + 2**-22
            sums = (len(at) + 8) * 2**-24
            off[first:last, h] = half * out[first:last, h].abs() + (half + 2 * score + 2 * sums) * (w @ v.abs()) * (1 + half)
            if kind == torch.float16:
                off[first:last, h] += 2**-25  # half a step of its subnormals
    return out, off


def make_cache(gen, lens, heads, dim, page, kind, cached, device, holes=False):
    """Tables over shuffled pages; every slot that no token holds is NaN, inf or the type's largest."""
    counts = [math.ceil(n / page) for n in lens]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=gen).tolist()
    width = max(max(counts), 1) + 1
    tables = [[order.pop() for _ in range(c)] + [123456789] * (width - c) for c in counts]
    scales = (0.02, 0.015) if cached == "e4m3" else (1.0, 1.0)
    made = []
    for scale in scales:
        x = torch.full((pages, heads, page, dim), math.nan)
        x[..., 1::3] = 448 * scale if cached == "e4m3" else math.inf
        for r, n in enumerate(lens):
            for c in range(counts[r]):
                m = min(page, n - c * page)
                x[tables[r][c], :, :m] = torch.randn((heads, m, dim), generator=gen)
        made.append(cache_like(x, TYPES[cached], scale) if cached == "e4m3" else x.to(TYPES[kind]))
    if holes:
        for row, entry in zip(tables, (-1, pages, 2**31 - 1, -(2**31))):
            row[0] = entry
    return made[0].to(device), made[1].to(device), tables, scales


HEADS = [(1, 1), (4, 4), (8, 2), (5, 1), (20, 1), (6, 2)]
KINDS = [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")]


def check_attention(got, q, cache, lens, cu, scale=None):
    k_cache, v_cache, tables, scales = cache
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, off = attention_oracle(q, k_cache, v_cache, tables, lens, cu, scale, *scales)
    assert got.dtype == q.dtype and got.shape == q.shape
    far = (got.cpu().double() - want).abs()
    assert (far <= off).all(), f"off by {far.max():.3g}, at most {float((far / off.clamp(min=1e-30)).max()):.3g} of what is allowed"


def run_decode(q, cache, lens, **more):
    k_cache, v_cache, tables, scales = cache
    d = q.device
    return paged.decode_attention(q, k_cache, v_cache, ints(tables, d), ints(lens, d), k_scale=scales[0], v_scale=scales[1], **more)


def run_prompt(q, cache, lens, cu, **more):
    k_cache, v_cache, tables, scales = cache
    d = q.device
    return paged.prompt_attention(
        q, k_cache, v_cache, ints(tables, d), ints(lens, d), ints(cu, d), k_scale=scales[0], v_scale=scales[1], **more
    )


@both
@pytest.mark.parametrize("kind,cached", KINDS)
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_decode_attention(device, kind, cached, dim, heads, kv_heads):
    page = {8: 16, 64: 16, 80: 64, 128: 32, 256: 128}[dim]
    gen = torch.Generator().manual_seed(heads * dim)
    lens = [0, 1, 2, 31, 32, 33, 64, 127, 0, 129, 257, 300]
    cache = make_cache(gen, lens, kv_heads, dim, page, kind, cached, device)
    q = torch.randn((len(lens), heads, dim), generator=gen).to(TYPES[kind]).to(device)
    got = run_decode(q, cache, lens)
    check_attention(got, q, cache, lens, list(range(len(lens) + 1)))
    assert (got[0] == 0).all() and (got[8] == 0).all()


@both
@pytest.mark.parametrize("kind,cached", KINDS)
@pytest.mark.parametrize("lens", [[5000], [1, 2049, 7, 4100], [640] * 40])
def test_decode_attention_over_long_rows(device, kind, cached, lens):
    gen = torch.Generator().manual_seed(len(lens))
    cache = make_cache(gen, lens, 2, 64, 64, kind, cached, device)
    q = (torch.randn((len(lens), 4, 64), generator=gen) * 2).to(TYPES[kind]).to(device)
    check_attention(run_decode(q, cache, lens), q, cache, lens, list(range(len(lens) + 1)))


@both
@pytest.mark.parametrize("kind,cached", KINDS)
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_prompt_attention(device, kind, cached, dim, heads, kv_heads):
    page = {8: 16, 64: 16, 80: 64, 128: 32, 256: 128}[dim]
    gen = torch.Generator().manual_seed(heads * dim + 1)
    new = [1, 0, 3, 40, 0, 1, 17]
    held = [0, 5, 60, 0, 0, 130, 33]
    lens = [h + n for h, n in zip(held, new)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    cache = make_cache(gen, lens, kv_heads, dim, page, kind, cached, device)
    q = torch.randn((cu[-1], heads, dim), generator=gen).to(TYPES[kind]).to(device)
    check_attention(run_prompt(q, cache, lens, cu), q, cache, lens, cu)


@both
@pytest.mark.parametrize("kind,cached", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 128)])
def test_prompt_attention_over_many_tiles(device, kind, cached, dim, page):
    gen = torch.Generator().manual_seed(dim)
    new, held = [150, 2, 333], [1, 500, 0]
    lens = [h + n for h, n in zip(held, new)]
    cu = [0, 150, 152, 485]
    cache = make_cache(gen, lens, 2, dim, page, kind, cached, device)
    q = (torch.randn((cu[-1], 4, dim), generator=gen) * 2).to(TYPES[kind]).to(device)
    check_attention(run_prompt(q, cache, lens, cu), q, cache, lens, cu)


@both
@pytest.mark.parametrize("cached", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim", range(8, 257, 8))
def test_every_head_dim(device, dim, cached):
    """Decode split and joined, prompts in tiles and with split keys; the cache's neighbours hold no numbers."""
    gen = torch.Generator().manual_seed(dim)
    lens, new = [700, 0, 65], [70, 0, 3]
    cu = [0, 70, 70, 73]
    cache = make_cache(gen, lens, 2, dim, 64, "bf16", cached, device)
    wide = (cache[0], cache[1], [t + [0] * 20 for t in cache[2]], cache[3])  # room for more keys: split and joined
    q = torch.randn((73, 4, dim), generator=gen).to(torch.bfloat16).to(device)
    for c in (cache, wide):
        check_attention(run_decode(q[:3], c, lens), q[:3], cache, lens, [0, 1, 2, 3])
        check_attention(run_prompt(q, c, lens, cu), q, cache, lens, cu)


FEW = [([7], [3000]), ([1, 0, 40, 3], [2500, 900, 0, 1023]), ([130], [1100])]
MANY = ([2] * 70, [600 + 13 * i for i in range(70)])


@both
@pytest.mark.parametrize(
    "kind,cached,dim,heads,kv_heads,new,held",
    [(*k, *d, *x) for k in KINDS for d in [(64, 4, 4), (128, 8, 2), (128, 5, 1), (64, 40, 1)] for x in FEW]
    + [("bf16", "bf16", 128, 8, 2, *MANY)],
)
def test_prompt_attention_of_few_rows_over_many_keys(device, kind, cached, dim, heads, kv_heads, new, held):
    """The last tokens of a request behind a long beginning, one, several and more than 64 requests."""
    gen = torch.Generator().manual_seed(len(new) + dim)
    lens = [h + n for h, n in zip(held, new)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    cache = make_cache(gen, lens, kv_heads, dim, 32, kind, cached, device)
    q = (torch.randn((cu[-1] + 3, heads, dim), generator=gen) * 2).to(TYPES[kind]).to(device)
    got = run_prompt(q, cache, lens, cu)
    assert (got[cu[-1] :] == 0).all()
    check_attention(got[: cu[-1]], q[: cu[-1]], cache, lens, cu)


@both
@pytest.mark.parametrize("requests", [64, 65, 130])
@pytest.mark.parametrize("kind,cached,dim", [("bf16", "bf16", 128), ("fp16", "fp16", 64), ("bf16", "e4m3", 80)])
def test_prompts_of_many_requests(device, kind, cached, dim, requests):
    """As many as a server may admit at once, their keys not split: up to 64 are ordered by their lengths, more are not."""
    rng = random.Random(requests)
    gen = torch.Generator().manual_seed(requests + dim)
    new = [rng.choice([0, 1, rng.randint(2, 90)]) for _ in range(requests)]
    held = [rng.choice([0, 0, rng.randint(1, 120)]) for _ in range(requests)]
    lens = [h + n for h, n in zip(held, new)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    cache = make_cache(gen, lens, 2, dim, 16, kind, cached, device)
    q = torch.randn((cu[-1], 4, dim), generator=gen).to(TYPES[kind]).to(device)
    check_attention(run_prompt(q, cache, lens, cu), q, cache, lens, cu)


@both
@pytest.mark.parametrize("kind,cached,dim", [("bf16", "bf16", 128), ("fp16", "fp16", 64), ("bf16", "e4m3", 80), ("bf16", "bf16", 256)])
@pytest.mark.parametrize("lens", [[333], [1], [256, 0, 1, 17, 63], [300] * 32])
def test_short_rows_of_a_table_as_wide_as_a_server_makes_it(device, kind, cached, dim, lens):
    """Room for 2048 tokens a row: the operators choose their form by it. One token of each row, and the rows' whole prompts."""
    gen = torch.Generator().manual_seed(len(lens) + dim)
    k_cache, v_cache, tables, scales = make_cache(gen, lens, 2, dim, 64, kind, cached, device)
    cache = (k_cache, v_cache, [t + [-1] * (32 - len(t)) for t in tables], scales)
    q = torch.randn((sum(lens), 4, dim), generator=gen).to(TYPES[kind]).to(device)
    one = torch.randn((len(lens), 4, dim), generator=gen).to(TYPES[kind]).to(device)
    check_attention(run_decode(one, cache, lens), one, cache, lens, list(range(len(lens) + 1)))
    if len(lens) < 32:
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        check_attention(run_prompt(q, cache, lens, cu), q, cache, lens, cu)


@both
@pytest.mark.parametrize("dim", [64, 128])
def test_split_keys_with_bad_entries_and_values(device, dim):
    """The same with an entry that names no page, and a later token that is not finite, in different parts of the keys."""
    gen = torch.Generator().manual_seed(dim)
    k_cache, v_cache, tables, scales = make_cache(gen, [2100], 2, dim, 16, "bf16", "bf16", device)
    cache = (k_cache, v_cache, tables, scales)
    q = torch.randn((60, 4, dim), generator=gen).to(torch.bfloat16).to(device)
    tables[0][20], tables[0][100] = -1, 1 << 30
    clean = run_prompt(q, cache, [2100], [0, 60])
    check_attention(clean, q, cache, [2100], [0, 60])
    v_cache[tables[0][2090 // 16], 0, 2090 % 16, 3] = math.nan
    got = run_prompt(q, cache, [2100], [0, 60])
    check_attention(got[:50], q[:50], cache, [2090], [0, 50])
    check_attention(got[:, 2:], q[:, 2:], (k_cache[:, 1:], v_cache[:, 1:], tables, scales), [2100], [0, 60])
    assert got[50:, :2, 3].isnan().all() and got[50:, :2, 4:].isfinite().all()


@both
@pytest.mark.parametrize("dim", [80, 64, 128])
def test_attention_with_entries_that_name_no_page(device, dim):
    """Their tokens count as absent, whatever the other pages hold."""
    gen = torch.Generator().manual_seed(3)
    lens = [20, 70, 33, 16, 40]
    cache = make_cache(gen, lens, 1, dim, 16, "bf16", "bf16", device, holes=True)
    q = torch.randn((5, 2, dim), generator=gen).to(torch.bfloat16).to(device)
    got = run_decode(q, cache, lens)
    check_attention(got, q, cache, lens, list(range(6)))
    assert (got[3] == 0).all()
    cu = [0, 20, 50, 60, 70, 72]
    q = torch.randn((72, 2, dim), generator=gen).to(torch.bfloat16).to(device)
    check_attention(run_prompt(q, cache, lens, cu), q, cache, lens, cu)


@both
@pytest.mark.parametrize("dim", [80, 64, 128])
def test_lengths_past_the_table_end_with_it(device, dim):
    gen = torch.Generator().manual_seed(4)
    k_cache, v_cache, tables, scales = make_cache(gen, [32, 32], 1, dim, 16, "bf16", "bf16", device)
    cache = (k_cache, v_cache, [t[:2] for t in tables], scales)
    q = torch.randn((2, 1, dim), generator=gen).to(torch.bfloat16).to(device)
    got = run_decode(q, cache, [2**31 - 1, -3])
    check_attention(got, q, cache, [32, 0], [0, 1, 2])
    # more new rows than tokens: the first rows see nothing
    q = torch.randn((40, 1, dim), generator=gen).to(torch.bfloat16).to(device)
    got = run_prompt(q, cache, [32, 0], [0, 40, 40])
    check_attention(got, q, cache, [32, 0], [0, 40, 40])
    assert (got[:8] == 0).all()


@both
@pytest.mark.parametrize("dim", [80, 64, 128])
@pytest.mark.parametrize("rows", [1, 30, 41, 160])
def test_fewer_rows_than_new_tokens(device, dim, rows):
    """The first rows of a step: what each of them sees does not change."""
    gen = torch.Generator().manual_seed(rows)
    lens, cu = [90, 100, 700], [0, 40, 140, 170]
    cache = make_cache(gen, lens, 2, dim, 16, "bf16", "bf16", device)
    q = torch.randn((170, 4, dim), generator=gen).to(torch.bfloat16).to(device)
    want, off = attention_oracle(q, *cache[:3], lens, cu, dim**-0.5, *cache[3])
    got = run_prompt(q[:rows], cache, lens, cu)
    assert got.shape[0] == rows
    assert ((got.cpu().double() - want[:rows]).abs() <= off[:rows]).all()


@both
@pytest.mark.parametrize("dim", [80, 64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_later_tokens_do_not_reach_earlier_rows(device, dim, bad):
    """A value or key that is not finite changes the rows that see it and no others."""
    gen = torch.Generator().manual_seed(5)
    k_cache, v_cache, tables, scales = make_cache(gen, [200], 2, dim, 16, "bf16", "bf16", device)
    q = torch.randn((200, 4, dim), generator=gen).to(torch.bfloat16).to(device)
    for which in (0, 1):
        caches = [k_cache.clone(), v_cache.clone()]
        caches[which][tables[0][150 // 16], 1, 150 % 16, 7] = bad
        got = run_prompt(q, (*caches, tables, scales), [200], [0, 200])
        cache = (k_cache, v_cache, tables, scales)
        check_attention(got[:150], q[:150], cache, [150], [0, 150])
        check_attention(got[:, :2], q[:, :2], (k_cache[:, :1], v_cache[:, :1], tables, scales), [200], [0, 200])
        touched = got[150:, 2:].isfinite() if which == 0 else got[150:, 2:, 7].isfinite()
        if which == 0 and bad == math.inf:
            # q * inf is +inf (no value for the row: inf - inf) or -inf (the token's weight is 0)
            negative = q[150:, 2:, 7] < 0
            assert (touched == negative[..., None]).all()
        else:
            assert not touched.any()
        if which == 1:
            rest = [d for d in range(dim) if d != 7]
            want, off = attention_oracle(q, k_cache, v_cache, tables, [200], [0, 200], dim**-0.5, *scales)
            assert ((got.cpu().double() - want).abs() <= off)[:, :, rest].all()


@both
@pytest.mark.parametrize("dim", [80, 64, 128])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(device, dim, bad):
    gen = torch.Generator().manual_seed(8)
    lens = [1, 40, 700, 33]
    k_cache, v_cache, tables, scales = make_cache(gen, lens, 1, dim, 16, "bf16", "bf16", device)
    cache = (k_cache, v_cache, tables, scales)
    q = torch.randn((4, 2, dim), generator=gen).to(torch.bfloat16).to(device)
    for cu in (None, [0, 1, 2, 3, 4]):
        run = lambda: run_decode(q, cache, lens) if cu is None else run_prompt(q, cache, lens, cu)  # noqa: E731
        clean = run()
        keep = v_cache.clone()
        for r, n in enumerate(lens[:3]):
            v_cache[tables[r][(n - 1) // 16], 0, (n - 1) % 16, 5] = bad
        got = run()
        v_cache.copy_(keep)
        assert torch.equal(got[3], clean[3])
        assert torch.equal(got[:3, :, 5].float().nan_to_num(3.0, 1.0, -1.0), torch.full((3, 2), bad, device=device).nan_to_num(3.0, 1.0, -1.0))
        want, off = attention_oracle(q, k_cache, v_cache, tables, lens, [0, 1, 2, 3, 4], dim**-0.5, *scales)
        rest = [d for d in range(dim) if d != 5]
        assert ((got.cpu().double() - want).abs() <= off)[..., rest].all()


# A row whose scores are not all numbers, in the operator's split and unsplit forms: `room` is the pages of 16 that a table
# row has, which decides between them.
NUMBERLESS = pytest.mark.parametrize("kind,cached,dim", [("bf16", "bf16", 64), ("fp16", "fp16", 128), ("bf16", "e4m3", 80), ("bf16", "bf16", 256)])


def check_all_but(got, q, cache, lens, cu, places):
    """NaN at the places (row, head); the other rows are what they are beside a finite q, to what rounding allows. Their bits
    may differ: the rows of a wave move their running maxima together, and so round probabilities at one scale or another."""
    want, off = attention_oracle(q, *cache[:3], lens, cu, q.shape[-1] ** -0.5, *cache[3])
    got = got.cpu().double()
    for r, head in places:
        assert got[r, head].isnan().all()
        got[r, head] = want[r, head]
    assert ((got - want).abs() <= off).all()


@both
@NUMBERLESS
@pytest.mark.parametrize("lens,room", [([300, 0, 17, 300], 20), ([5000, 0, 17, 4100], 320), ([700] * 300, 44)])
def test_a_query_that_is_no_number_in_decode(device, kind, cached, dim, lens, room):
    """Its row is NaN, however its keys are split, and no other; without keys it is zero all the same."""
    gen = torch.Generator().manual_seed(dim)
    k_cache, v_cache, tables, scales = make_cache(gen, lens, 2, dim, 16, kind, cached, device)
    cache = (k_cache, v_cache, [t + [0] * (room - len(t)) for t in tables], scales)
    q = torch.randn((len(lens), 4, dim), generator=gen).to(TYPES[kind]).to(device)
    bad, places = q.clone(), [(0, 1), (1, 0), (2, 3)]
    for r, head in places:
        bad[r, head, dim // 2] = math.nan
    got = run_decode(bad, cache, lens)
    check_all_but(got, q, cache, lens, list(range(len(lens) + 1)), [p for p in places if lens[p[0]]])


@both
@NUMBERLESS
def test_a_stretch_of_keys_that_are_no_numbers_in_decode(device, kind, cached, dim):
    """Whole chunks of it, the first, inner ones and the last: they make the heads that read them NaN."""
    gen = torch.Generator().manual_seed(dim)
    for first, last in ((0, 512), (1024, 2048), (4864, 5000)):
        k_cache, v_cache, tables, scales = make_cache(gen, [5000], 2, dim, 16, kind, cached, device)
        q = torch.randn((1, 4, dim), generator=gen).to(TYPES[kind]).to(device)
        raw = torch.uint8 if cached == "e4m3" else torch.int16  # 0x7f..: NaN in each of the types
        for t in range(first, last):
            k_cache.view(raw)[tables[0][t // 16], 1, t % 16, dim - 1] = 0x7F if cached == "e4m3" else 0x7FFF
        got = run_decode(q, (k_cache, v_cache, tables, scales), [5000])
        assert got[:, 2:].isnan().all()
        check_attention(got[:, :2], q[:, :2], (k_cache[:, :1], v_cache[:, :1], tables, scales), [5000], [0, 1])

@both
@NUMBERLESS
@pytest.mark.parametrize("new,held,room", [([40, 3], [100, 0], 12), ([7, 0, 3], [3000, 0, 900], 200), ([300, 300], [0, 700], 66)])
def test_a_query_that_is_no_number_in_a_prompt(device, kind, cached, dim, new, held, room):
    gen = torch.Generator().manual_seed(dim)
    lens = [h + n for h, n in zip(held, new)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    k_cache, v_cache, tables, scales = make_cache(gen, lens, 2, dim, 16, kind, cached, device)
    cache = (k_cache, v_cache, [t + [0] * (room - len(t)) for t in tables], scales)
    q = torch.randn((cu[-1], 4, dim), generator=gen).to(TYPES[kind]).to(device)
    bad = q.clone()
    places = [(0, 1), (2, 3), (cu[-1] - 1, 0)]
    for r, head in places:
        bad[r, head, dim // 2] = math.nan
    check_all_but(run_prompt(bad, cache, lens, cu), q, cache, lens, cu, places)


@both
@NUMBERLESS
def test_a_newest_key_that_is_no_number_alone_in_its_part(device, kind, cached, dim):
    """1025 keys are four parts of 256 and one of a single key, the row's own; 1030 with the last six tokens new."""
    gen = torch.Generator().manual_seed(dim)
    for n in (1, 6):
        length = 1024 + n
        k_cache, v_cache, tables, scales = make_cache(gen, [length], 2, dim, 16, kind, cached, device)
        q = torch.randn((n, 4, dim), generator=gen).to(TYPES[kind]).to(device)
        raw = torch.uint8 if cached == "e4m3" else torch.int16
        k_cache.view(raw)[tables[0][1024 // 16], 1, 0, 0] = 0x7F if cached == "e4m3" else 0x7FFF
        got = run_prompt(q, (k_cache, v_cache, tables, scales), [length], [0, n])
        assert got[:, 2:].isnan().all()
        check_attention(got[:, :2], q[:, :2], (k_cache[:, :1], v_cache[:, :1], tables, scales), [length], [0, n])

def infinite_keys(gen, lens, dim, kind, device, room, where=lambda t: True):
    """A cache of two kv heads; the keys t of the first that `where` names hold inf in dim 7, so that a query negative there
    has the score -inf."""
    k_cache, v_cache, tables, scales = make_cache(gen, lens, 2, dim, 16, kind, kind, device)
    for r, n in enumerate(lens):
        t = torch.tensor([t for t in range(n) if where(t)], dtype=torch.int64)
        if len(t):
            k_cache[torch.tensor(tables[r], dtype=torch.int64)[t // 16].to(device), 0, (t % 16).to(device), 7] = math.inf
    return k_cache, v_cache, [t + [0] * (room - len(t)) for t in tables], scales


@both
@pytest.mark.parametrize("kind,dim", [("bf16", 64), ("fp16", 128), ("bf16", 80), ("fp16", 256)])
@pytest.mark.parametrize("lens,room", [([1, 0, 40, 300], 20), ([1, 0, 700, 5000], 320)])
def test_scores_of_minus_infinity_in_decode(device, kind, dim, lens, room):
    """Where all that a row sees have it, the softmax is 0 / 0: NaN. Where some have, they weigh nothing."""
    gen = torch.Generator().manual_seed(dim)
    q = torch.randn((4, 4, dim), generator=gen).to(TYPES[kind]).to(device)
    q[:, :2, 7] = -1.0
    cache = infinite_keys(gen, lens, dim, kind, device, room)
    got = run_decode(q, cache, lens)
    assert got[[0, 2, 3], :2].isnan().all() and (got[1] == 0).all()
    check_attention(got[:, 2:], q[:, 2:], (cache[0][:, 1:], cache[1][:, 1:], *cache[2:]), lens, [0, 1, 2, 3, 4])
    # the same as if those keys were absent: pages 0 and 4 to 19 of each row
    gone = lambda t: t // 16 == 0 or 4 <= t // 16 < 20  # noqa: E731
    cache = infinite_keys(gen, lens, dim, kind, device, room, gone)
    got = run_decode(q, cache, lens)
    left = [[-1 if gone(16 * i) else p for i, p in enumerate(t)] for t in cache[2]]
    some = [r for r, n in enumerate(lens) if any(not gone(t) for t in range(n))]
    want = [lens[r] for r in some]
    cache = (cache[0][:, :1], cache[1][:, :1], [left[r] for r in some], cache[3])
    check_attention(got[some, :2], q[some, :2], cache, want, list(range(len(some) + 1)))

@both
@pytest.mark.parametrize("kind,dim", [("bf16", 64), ("fp16", 128), ("bf16", 80), ("fp16", 256)])
@pytest.mark.parametrize("length,rows,room", [(90, 90, 8), (90, 100, 8), (3000, 5, 200)])
def test_scores_of_minus_infinity_in_a_prompt(device, kind, dim, length, rows, room):
    """The same, and rows that see no key stay zero."""
    gen = torch.Generator().manual_seed(dim)
    q = torch.randn((rows, 4, dim), generator=gen).to(TYPES[kind]).to(device)
    q[:, :2, 7] = -1.0
    none = max(0, rows - length)
    cache = infinite_keys(gen, [length], dim, kind, device, room)
    got = run_prompt(q, cache, [length], [0, rows])
    assert (got[:none] == 0).all() and got[none:, :2].isnan().all()
    check_attention(got[:, 2:], q[:, 2:], (cache[0][:, 1:], cache[1][:, 1:], *cache[2:]), [length], [0, rows])
    # the first three pages and a later stretch: as if those keys were absent
    gone = lambda t: t < 48 or 512 <= t < 1104  # noqa: E731
    cache = infinite_keys(gen, [length], dim, kind, device, room, gone)
    got = run_prompt(q, cache, [length], [0, rows])
    first = none + 48 if rows >= length else 0  # the first row that sees another
    assert (got[:none] == 0).all() and got[none:first, :2].isnan().all()
    left = [[-1 if gone(16 * i) else p for i, p in enumerate(cache[2][0])]]
    check_attention(got[first:, :2], q[first:, :2], (cache[0][:, :1], cache[1][:, :1], left, cache[3]), [length], [0, rows - first])


@both
@pytest.mark.parametrize("dim", [80, 64, 128])
def test_scores_far_apart(device, dim):
    """Scores of thousands, all equal scores, and a maximum that comes first or last."""
    gen = torch.Generator().manual_seed(6)
    cache = make_cache(gen, [300, 300, 300], 1, dim, 64, "fp16", "fp16", device)
    q = torch.randn((3, 2, dim), generator=gen).half().to(device)
    q[0] *= 200
    q[1] = 0
    tables = cache[2]
    cache[0][tables[2][0], 0, 0] = q[2, 0] * 4
    cache[0][tables[2][4], 0, 300 - 257] = q[2, 1] * 4
    check_attention(run_decode(q, cache, [300] * 3), q, cache, [300] * 3, [0, 1, 2, 3])
    check_attention(run_decode(q, cache, [300] * 3, scale=-0.5), q, cache, [300] * 3, [0, 1, 2, 3], scale=-0.5)
    check_attention(run_prompt(q, cache, [300] * 3, [0, 1, 2, 3], scale=0.01), q, cache, [300] * 3, [0, 1, 2, 3], scale=0.01)


@both
@pytest.mark.parametrize("dim", [80, 64, 128])
def test_strided_queries_and_given_results(device, dim):
    gen = torch.Generator().manual_seed(7)
    lens, cu = [90, 0, 33], [0, 50, 50, 60]
    cache = make_cache(gen, lens, 2, dim, 16, "bf16", "bf16", device)
    for offset in (0, 1, 8):  # 1: rows off the 16-byte grid
        fused = torch.randn((64, 9, dim + offset), generator=gen).to(torch.bfloat16).to(device)
        q = fused[:, 2:6, offset:]
        out = torch.full((64, 4, dim), 5.0, dtype=torch.bfloat16, device=device)
        got = run_prompt(q, cache, lens, cu, out=out)
        assert got.data_ptr() == out.data_ptr() and (out[60:] == 5).all()
        check_attention(out[:60], q[:60], cache, lens, cu)
        fresh = run_prompt(q, cache, lens, cu)
        assert (fresh[60:] == 0).all() and torch.equal(fresh[:60], out[:60])
        q = q.transpose(0, 1)[:, :3].transpose(0, 1)
        out = torch.full((3, 4, dim), 5.0, dtype=torch.bfloat16, device=device)
        run_decode(q, cache, lens, out=out)
        check_attention(out, q, cache, lens, [0, 1, 2, 3])


@both
def test_empty_calls(device):
    cache = torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16, device=device)
    none = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device=device)
    tables, zero = ints([[0, 1]], device), ints([0], device)
    assert paged.decode_attention(none, cache, cache, tables[:0], zero[:0]).shape == (0, 4, 64)
    assert paged.prompt_attention(none, cache, cache, tables, zero, ints([0, 0], device)).shape == (0, 4, 64)
    paged.write_kv(none[:, :2], none[:, :2], cache, cache.clone(), zero[:0])
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device=device)
    assert (paged.prompt_attention(q, cache, cache, tables[:0], zero[:0], zero) == 0).all()


# -- refusals ---------------------------------------------------------------


def good(device):
    bf16 = dict(dtype=torch.bfloat16, device=device)
    return dict(
        q=torch.zeros((3, 4, 64), **bf16),
        k_cache=torch.zeros((5, 2, 16, 64), **bf16),
        v_cache=torch.zeros((5, 2, 16, 64), **bf16),
        tables=torch.zeros((3, 2), dtype=torch.int32, device=device),
        kv_lens=torch.zeros(3, dtype=torch.int32, device=device),
    )


@both
@pytest.mark.parametrize(
    "change,error",
    [
        (dict(q=lambda x: x.int()), TypeError),
        (dict(q=lambda x: x[0]), ValueError),
        (dict(q=lambda x: x[:2]), ValueError),
        (dict(q=lambda x: x[:, :3]), ValueError),
        (dict(q=lambda x: x[..., :32]), ValueError),
        (dict(q=lambda x: x.repeat(1, 1, 2)[..., ::2]), ValueError),
        (dict(q=lambda x: x.requires_grad_()), RuntimeError),
        (dict(k_cache=lambda x: x.half()), TypeError),
        (dict(v_cache=lambda x: x.to(torch.float8_e4m3fn)), TypeError),
        (dict(k_cache=lambda x: x[:4]), ValueError),
        (dict(k_cache=lambda x: x.transpose(1, 2), v_cache=lambda x: x.transpose(1, 2)), ValueError),
        (dict(k_cache=lambda x: x[:, :, :10].contiguous(), v_cache=lambda x: x[:, :, :10].contiguous()), ValueError),
        (dict(k_cache=lambda x: x[0], v_cache=lambda x: x[0]), ValueError),
        (dict(k_cache=lambda x: x[:0], v_cache=lambda x: x[:0]), ValueError),
        (dict(tables=lambda x: x.long()), TypeError),
        (dict(tables=lambda x: x[0]), ValueError),
        (dict(tables=lambda x: x[:, :0]), ValueError),
        (dict(tables=lambda x: x.t().contiguous().t()), ValueError),
        (dict(tables=lambda x: x[:2]), ValueError),
        (dict(kv_lens=lambda x: x.float()), TypeError),
        (dict(kv_lens=lambda x: x[:2]), ValueError),
        (dict(kv_lens=lambda x: x.repeat(2)[::2]), ValueError),
        (dict(scale=math.nan), ValueError),
        (dict(k_scale=2.0), ValueError),
        (dict(v_scale=0.0), ValueError),
        (dict(k_scale=math.inf), ValueError),
        (dict(out=lambda q: q.clone().half()), TypeError),
        (dict(out=lambda q: q), ValueError),
        (dict(out=lambda q: q.clone()[:, :2]), ValueError),
        (dict(out=lambda q: torch.cat([q, q], 1)[:, :4]), ValueError),
    ],
)
def test_attention_refusals(device, change, error):
    args, more = good(device), {}
    for name, f in change.items():
        if name in args:
            args[name] = f(args[name])
        else:
            more[name] = f(args["q"]) if callable(f) else f
    with pytest.raises(error):
        paged.decode_attention(*args.values(), **more)
    cu = torch.zeros(4, dtype=torch.int32, device=device)
    if set(change) != {"q"} or error is not ValueError or args["q"].shape[1:] != (4, 64) or args["q"].stride(2) != 1:
        with pytest.raises(error):
            paged.prompt_attention(*args.values(), cu, **more)
    args = good(device)
    for bad, e in ((cu[:3], ValueError), (cu.long(), TypeError), (cu.repeat(2)[::2], ValueError)):
        with pytest.raises(e):
            paged.prompt_attention(*args.values(), bad)


@both
@pytest.mark.parametrize(
    "more",
    [dict(scale=1e39), dict(scale=-1e300), dict(k_scale=1e30, scale=1e10), dict(k_scale=1e-40), dict(v_scale=1e39), dict(v_scale=1e-50)],
)
def test_scales_that_32_bits_do_not_hold_are_refused(device, more):
    args = good(device)
    args["k_cache"], args["v_cache"] = (args[n].to(torch.float8_e4m3fn) for n in ("k_cache", "v_cache"))
    cu = torch.zeros(4, dtype=torch.int32, device=device)
    with pytest.raises(ValueError):
        paged.decode_attention(*args.values(), **more)
    with pytest.raises(ValueError):
        paged.prompt_attention(*args.values(), cu, **more)
    if "scale" not in more:
        k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=device)
        with pytest.raises(ValueError):
            paged.write_kv(k, k, args["k_cache"], args["v_cache"], ints([0, 1], device), **more)


@both
def test_more_work_than_a_launch_takes_is_refused(device):
    """Sizes that take no memory: a row of each stands for all, or most requests bring nothing."""
    bf16 = dict(dtype=torch.bfloat16, device=device)
    cache = torch.zeros((1, 2048, 16, 8), **bf16)
    tokens = 2**21
    slots = ints([-1], device).repeat(tokens)
    k = torch.zeros((1, 2048, 8), **bf16).expand(tokens, -1, -1)
    with pytest.raises(ValueError, match="too many tokens"):
        paged.write_kv(k, k, cache, cache, slots)
    cache = torch.zeros((1, 8192, 16, 8), **bf16)
    q = torch.zeros((1, 8192, 8), **bf16)
    tables, lens, cu = ints([[0]], device).repeat(4096, 1), ints([0], device).repeat(4096), ints([0], device).repeat(4097)
    with pytest.raises(ValueError, match="too many"):
        paged.prompt_attention(q, cache, cache, tables, lens, cu)


@both
def test_head_dims_are_refused_that_no_kernel_takes(device):
    for dim in (4, 12, 264):
        q = torch.zeros((1, 1, dim), dtype=torch.bfloat16, device=device)
        cache = torch.zeros((1, 1, 16, dim), dtype=torch.bfloat16, device=device)
        with pytest.raises(ValueError):
            paged.decode_attention(q, cache, cache, ints([[0]], device), ints([0], device))
        with pytest.raises(ValueError):
            paged.write_kv(q, q, cache, cache, ints([0], device))


@both
@pytest.mark.parametrize(
    "change,error",
    [
        (dict(k=lambda x: x.int()), TypeError),
        (dict(v=lambda x: x.half()), TypeError),
        (dict(k=lambda x: x[:, :1]), ValueError),
        (dict(k=lambda x: x[:, :1], v=lambda x: x[:, :1]), ValueError),
        (dict(k=lambda x: x.repeat(1, 1, 2)[..., ::2]), ValueError),
        (dict(slots=lambda x: x.long()), TypeError),
        (dict(slots=lambda x: x[:1]), ValueError),
        (dict(slots=lambda x: x[None]), ValueError),
        (dict(k_cache=lambda x: x[:, :, :, :32]), ValueError),
        (dict(k_scale=0.5), ValueError),
        (dict(v_scale=-1.0), ValueError),
        (dict(k=lambda x: x.requires_grad_()), RuntimeError),
    ],
)
def test_write_refusals(device, change, error):
    bf16 = dict(dtype=torch.bfloat16, device=device)
    args = dict(k=torch.zeros((2, 2, 64), **bf16), v=torch.zeros((2, 2, 64), **bf16))
    args |= dict(k_cache=torch.zeros((5, 2, 16, 64), **bf16), v_cache=torch.zeros((5, 2, 16, 64), **bf16), slots=ints([0, 1], device))
    for name, f in change.items():
        args[name] = f(args[name]) if callable(f) else f
    with pytest.raises(error):
        paged.write_kv(**args)


@both
@pytest.mark.parametrize(
    "change,error",
    [
        (dict(page_size=24), ValueError),
        (dict(page_size=8), ValueError),
        (dict(page_size=512), ValueError),
        (dict(num_tokens=-1), ValueError),
        (dict(tables=lambda x: x.float()), TypeError),
        (dict(tables=lambda x: x[:0]), ValueError),
        (dict(tables=lambda x: x.repeat(3000, 1)), ValueError),
        (dict(tables=lambda x: x[:1].expand(2, 2)), ValueError),
        (dict(lens=lambda x: x[:1]), ValueError),
        (dict(lens=lambda x: x.long()), TypeError),
        (dict(new_lens=lambda x: x[:1]), ValueError),
        (dict(new_lens=lambda x: x.long()), TypeError),
        (dict(free_pages=lambda x: x[None]), ValueError),
        (dict(free_pages=lambda x: x.repeat(2)[::2]), ValueError),
        (dict(free_count=lambda x: x.repeat(2)), ValueError),
        (dict(free_count=lambda x: x.float()), TypeError),
    ],
)
def test_plan_refusals(device, change, error):
    args = dict(tables=ints([[0, 1], [2, 3]], device), lens=ints([1, 1], device), new_lens=ints([1, 1], device))
    args |= dict(free_pages=ints([4, 5], device), free_count=ints([2], device), page_size=16, num_tokens=2)
    for name, f in change.items():
        args[name] = f(args[name]) if callable(f) else f
    with pytest.raises(error):
        paged.plan_step(**args)
    if "new_lens" in change or "num_tokens" in change:
        return
    args["done"] = torch.zeros(2, dtype=torch.bool, device=device)
    del args["new_lens"], args["num_tokens"]
    with pytest.raises(error):
        paged.release_pages(**args)


@both
def test_release_refusals(device):
    tables, lens = ints([[0, 1], [2, 3]], device), ints([1, 1], device)
    free, count = ints([4, 5], device), ints([1], device)
    for done, error in ((ints([0, 0], device), TypeError), (torch.zeros(3, dtype=torch.bool, device=device), ValueError)):
        with pytest.raises(error):
            paged.release_pages(tables, lens, done, free, count, 16)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs MI355X")
def test_tensors_of_two_devices_are_refused():
    args = good("cuda")
    for name in ("k_cache", "v_cache", "tables", "kv_lens"):
        with pytest.raises(ValueError):
            paged.decode_attention(**{**args, name: args[name].cpu()})
    with pytest.raises((ValueError, TypeError)):
        paged.decode_attention(**{**args, "q": args["q"].cpu()})
    with pytest.raises(TypeError):
        paged.decode_attention(**{n: x.float() if x.is_floating_point() else x for n, x in args.items()})


# -- the operators together -------------------------------------------------


class Dense:
    """A request's keys, values and last output in 64 bits, beside the paged cache."""

    def __init__(self, layers, kv_heads, dim):
        self.k = [torch.zeros((0, kv_heads, dim), dtype=torch.float64) for _ in range(layers)]
        self.v = [torch.zeros((0, kv_heads, dim), dtype=torch.float64) for _ in range(layers)]


@both
@pytest.mark.parametrize("kind,cached,dim", [("bf16", "bf16", 64), ("fp16", "fp16", 128), ("bf16", "e4m3", 128), ("bf16", "bf16", 80)])
def test_requests_come_and_go(device, kind, cached, dim):
    """A server's steps on one cache: prompts in parts, decoding, ends, rows and pages used again, a pool that runs short.
    Every output is compared with attention over the request's own keys and values, as the cache holds them."""
    rng = random.Random(dim)
    gen = torch.Generator().manual_seed(dim)
    layers, heads, kv_heads, rows, page = 2, 4, 2, 6, 16
    scales = (0.03125, 0.0625) if cached == "e4m3" else (1.0, 1.0)
    cache = paged.PagedKVCache(layers, kv_heads, dim, 17, page, rows, 200, TYPES[cached], device, *scales)
    dense = [Dense(layers, kv_heads, dim) for _ in range(rows)]
    refused = 0
    for step in range(24):
        decode = step % 3 != 0
        held = cache.lens.tolist()
        if decode:
            new = [1] * rows
        else:
            new = [rng.choice([0, rng.randint(1, 70)]) for _ in range(rows)]
        total = sum(new)
        plan = cache.plan(ints(new, device), total + (0 if decode else 5))
        served = [n > 0 and k > 0 for n, k in zip(new, plan.kv_lens.tolist())]
        refused += sum(n > 0 and not s for n, s in zip(new, served))
        assert cache.lens.tolist() == [h + (n if s else 0) for h, n, s in zip(held, new, served)]
        cu = plan.cu_new.tolist()
        for layer in range(layers):
            fused = torch.randn((plan.slots.shape[0], heads + 2 * kv_heads, dim), generator=gen).to(TYPES[kind]).to(device)
            q, k, v = fused[:, :heads], fused[:, heads : heads + kv_heads], fused[:, heads + kv_heads :]
            cache.write(layer, k, v, plan)
            out = (cache.decode if decode else cache.prompt)(layer, q, plan)
            for r in range(rows):
                part = slice(cu[r], cu[r + 1])
                if not served[r]:
                    assert (out[part] == 0).all()
                    continue
                d = dense[r]
                for x, have, scale in ((k, d.k, scales[0]), (v, d.v, scales[1])):
                    have[layer] = torch.cat([have[layer], values_of(cache_like(x[part].cpu(), TYPES[cached], scale), scale)])
                n = len(d.k[layer])
                # one page that holds all of the request's tokens
                whole = (d.k[layer][None].transpose(1, 2).contiguous(), d.v[layer][None].transpose(1, 2).contiguous())
                want, off = attention_oracle(q[part], *whole, [[0]], [n], [0, new[r]], dim**-0.5, 1.0, 1.0)
                assert ((out[part].cpu().double() - want).abs() <= off).all()
            assert (out[cu[-1] :] == 0).all()
        # no page has two owners
        used = [cache.tables[r, : cache.pages_for(n)].tolist() for r, n in enumerate(cache.lens.tolist())]
        stack = cache.free_pages[: int(cache.free_count)].tolist()
        assert sorted(sum(used, []) + stack) == list(range(cache.pages))
        if step % 4 == 3:
            done = [rng.random() < 0.5 for _ in range(rows)]
            cache.release(torch.tensor(done, device=device))
            for r in range(rows):
                if done[r]:
                    dense[r] = Dense(layers, kv_heads, dim)
    assert refused  # the pool did run short


@both
def test_cache_arguments(device):
    with pytest.raises(ValueError):
        paged.PagedKVCache(1, 1, 64, 4, page_size=20, device=device)
    with pytest.raises(ValueError):
        paged.PagedKVCache(0, 1, 64, 4, device=device)
    for more in (dict(head_dim=12), dict(head_dim=264), dict(requests=4097), dict(pages=2**27, page_size=16), dict(max_len=2**31)):
        with pytest.raises(ValueError):
            paged.PagedKVCache(**(dict(layers=1, kv_heads=1, head_dim=64, pages=4, device=device) | more))
    for more in (dict(k_scale=0.5), dict(dtype=torch.float8_e4m3fn, v_scale=0.0)):
        with pytest.raises(ValueError):
            paged.PagedKVCache(1, 1, 64, 4, device=device, **more)
    cache = paged.PagedKVCache(1, 2, 64, 4, 16, 2, 40, device=device)
    assert cache.tables.shape == (2, 3) and cache.pages == 4 and cache.pages_for(17) == 2 and cache.k.dtype == torch.bfloat16


@both
def test_transformer_model_over_the_cache(device):
    """Prompts in two parts and a decode step give what the whole sequences give at once."""
    from beta9_amd.models.transformer import TransformerServingModel

    torch.manual_seed(0)
    # 4 heads of 64; a scale that keeps the random layers' outputs near their inputs' size
    model = TransformerServingModel(hidden=256, inter=512, layers=2, n_heads=4, n_kv_heads=2, device=device)
    for b in model.blocks:
        for w in (b.attn_norm, b.mlp_norm):
            w.fill_(1.0)
    lens = [70, 1, 33]
    x = [torch.randn((n + 1, 256), device=device).to(torch.bfloat16) for n in lens]
    cache = model.new_cache(requests=3, max_len=100, page_size=16)
    first = [40, 0, 33]
    got = [[], [], []]
    for part in ([(0, f) for f in first], [(f, n) for f, n in zip(first, lens)]):
        new = ints([b - a for a, b in part], device)
        y = model.prompt(torch.cat([v[a:b] for v, (a, b) in zip(x, part)]), new, cache)
        for r, piece in enumerate(y.split([b - a for a, b in part])):
            got[r].append(piece)
    y = model.decode(torch.stack([v[n] for v, n in zip(x, lens)]), cache)
    for r in range(3):
        got[r].append(y[r : r + 1])
    for r in range(3):
        whole = x[r]
        for b in model.blocks:
            whole = b.forward(whole)
        a, b = torch.cat(got[r]).double(), whole.double()
        # both round attention, projections, norms and sums to bf16, in 2 layers of 9 operations each: 36 roundings of
        # half a step, 2^-8, that add up as independent ones; the maximum over 256 x 71 values is within 5 deviations
        assert float((a - b).abs().max() / b.std()) <= 5 * (2 * 2 * 9) ** 0.5 * 2**-8


# -- streams, graphs, threads -----------------------------------------------

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs MI355X")]


@both
def test_infer_decode(device, monkeypatch):
    from beta9_amd.models import bench_handler
    from beta9_amd.models.transformer import TransformerServingModel

    torch.manual_seed(0)
    model = TransformerServingModel(hidden=256, inter=512, layers=2, n_heads=4, n_kv_heads=2, device=device)
    for b in model.blocks:
        for w in (b.attn_norm, b.mlp_norm):
            w.fill_(1.0)
    monkeypatch.setattr(bench_handler, "_model", model)
    r = bench_handler.infer(tokens=5, decode_steps=3, requests=2)
    assert r["requests"] == 2 and r["tokens_per_sec"] > 0 and math.isfinite(r["checksum"])
    for bad in ((0, 5, 3), (2, 0, 3), (2, 5, 0), (5000, 1, 1)):
        with pytest.raises(ValueError):
            model.infer_decode(*bad)
    monkeypatch.setattr(bench_handler, "_model", object())
    with pytest.raises(ValueError):
        bench_handler.infer(tokens=5, decode_steps=3)


class Loop:
    """A decode step of two layers over a cache of its own, its inputs changed from outside."""

    def __init__(self, seed, rows=5, heads=8, kv_heads=2, dim=128):
        self.gen = torch.Generator().manual_seed(seed)
        self.rows, self.heads, self.kv_heads, self.dim = rows, heads, kv_heads, dim
        self.cache = paged.PagedKVCache(2, kv_heads, dim, 40, 16, rows, 700, device="cuda")
        self.one = torch.ones(rows, dtype=torch.int32, device="cuda")
        self.fused = torch.zeros((2, rows, heads + 2 * kv_heads, dim), dtype=torch.bfloat16, device="cuda")
        n = [3, 17, 0, 40, 1]
        plan = self.cache.plan(ints(n, "cuda"), sum(n))
        x = torch.randn((2, sum(n), 2 * kv_heads, dim), generator=self.gen).to(torch.bfloat16).cuda()
        for layer in range(2):
            self.cache.write(layer, x[layer, :, :kv_heads], x[layer, :, kv_heads:], plan)

    def fresh(self):
        self.fused.copy_(torch.randn(self.fused.shape, generator=self.gen))

    def step(self):
        h, kv = self.heads, self.kv_heads
        plan = self.cache.plan(self.one, self.rows)
        out = []
        for layer in range(2):
            x = self.fused[layer]
            self.cache.write(layer, x[:, h : h + kv], x[:, h + kv :], plan)
            out.append(self.cache.decode(layer, x[:, :h], plan))
            out.append(self.cache.prompt(layer, x[:, :h], plan))
        return out + list(plan)

    def state(self):
        return [self.cache.lens, self.cache.free_count, self.cache.tables, self.cache.k, self.cache.v]


def captured(loop):
    """The step in a graph, and its outputs; the state is as before the capture."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = loop.step()
    return graph, out


class TestOnTheGpu:
    pytestmark = gpu

    def test_two_captured_steps_replayed_in_turn(self):
        """Two caches' steps in graphs of their own, an eager twin of each beside them, many replays with other work and
        synchronizations between: every replay gives what the eager step gives, bit by bit."""
        loops, twins = [Loop(1), Loop(2)], [Loop(1), Loop(2)]
        for x in twins:
            x.fresh(), x.step()  # code is loaded before the capture
        for x in loops:
            x.fresh(), x.step()
        graphs = [captured(x) for x in loops]
        for turn in range(8):
            for which in (0, 1) if turn % 2 else (1, 0):
                loop, twin, (graph, out) = loops[which], twins[which], graphs[which]
                loop.fresh(), twin.fresh()
                graph.replay()
                want = twin.step()
                torch.randn((512, 512), device="cuda").sum()
                if turn % 3 == 0:
                    torch.cuda.synchronize()
                for a, b in zip(out + loop.state(), want + twin.state()):
                    assert torch.equal(a, b)
        assert loops[0].cache.lens.tolist() == [3 + 9, 17 + 9, 9, 40 + 9, 1 + 9]

    def test_calls_on_several_streams_at_once(self):
        """The same calls on three streams, enqueued without waiting, give the bits of the calls one by one."""
        gen = torch.Generator().manual_seed(9)
        jobs = []
        for lens, heads, kv_heads, dim in (([900, 30, 2000], 8, 2, 128), ([64] * 30, 4, 4, 64), ([5000], 16, 1, 128)):
            cache = make_cache(gen, lens, kv_heads, dim, 16, "bf16", "bf16", "cuda")
            q = torch.randn((sum(min(n, 100) for n in lens), heads, dim), generator=gen).to(torch.bfloat16).cuda()
            cu = [0]
            for n in lens:
                cu.append(cu[-1] + min(n, 100))
            jobs.append((q, cache, lens, cu))
        calls = lambda q, cache, lens, cu: (run_decode(q[: len(lens)], cache, lens), run_prompt(q, cache, lens, cu))  # noqa: E731
        want = [calls(*j) for j in jobs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in jobs]
        got = []
        for _ in range(10):
            for stream, job in zip(streams, jobs):
                stream.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(stream):
                    got.append(calls(*job))
        torch.cuda.synchronize()
        for i, pair in enumerate(got):
            for a, b in zip(pair, want[i % len(jobs)]):
                assert torch.equal(a, b)

    def test_runs_are_the_same_bit_by_bit(self):
        gen = torch.Generator().manual_seed(10)
        lens = [3000, 1, 700, 0, 2500]
        cache = make_cache(gen, lens, 2, 128, 64, "bf16", "e4m3", "cuda")
        q = torch.randn((5, 8, 128), generator=gen).to(torch.bfloat16).cuda()
        first = run_decode(q, cache, lens)
        for _ in range(5):
            assert torch.equal(run_decode(q, cache, lens), first)

    def test_slots_past_two_to_the_31_bytes(self):
        """A cache of more than 4 GB a side: offsets pass 32 bits."""
        pages, page, dim = 140_000, 64, 128
        k = torch.empty((pages, 2, page, dim), dtype=torch.bfloat16, device="cuda")
        v = torch.empty_like(k)
        gen = torch.Generator().manual_seed(11)
        rows = [pages - 1, 0, pages - 2, 70_001]
        n = 250
        x = torch.randn((n, 6, dim), generator=gen).to(torch.bfloat16).cuda()
        slots = torch.cat([torch.arange(p * page, (p + 1) * page, dtype=torch.int32) for p in rows])[:n].cuda()
        paged.write_kv(x[:, 2:4], x[:, 4:], k, v, slots)
        small_k = torch.stack([k[p] for p in rows])
        small_v = torch.stack([v[p] for p in rows])
        near, far = [[0, 1, 2, 3]], [rows]
        q = x[:, :2].repeat(1, 2, 1)
        for run, more in ((run_decode, ()), (run_prompt, ([0, n],))):
            rows_of_q = q[:1] if run is run_decode else q
            small = run(rows_of_q, (small_k, small_v, near, (1.0, 1.0)), [n], *more)
            check_attention(small, rows_of_q, (small_k, small_v, near, (1.0, 1.0)), [n], more[0] if more else [0, 1])
            assert torch.equal(run(rows_of_q, (k, v, far, (1.0, 1.0)), [n], *more), small)

    def test_another_current_device(self):
        if torch.cuda.device_count() < 2:
            pytest.skip("one GPU")
        loop = Loop(3)
        loop.fresh()
        with torch.cuda.device(1):
            out = loop.step()
        assert all(t.device == loop.fused.device for t in out)
