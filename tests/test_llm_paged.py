"""The LLM engine over the paged key-value cache."""

import asyncio
import threading
from concurrent.futures import ThreadPoolExecutor

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")

from beta9_amd.integrations import LLMArgs  # noqa: E402
from beta9_amd.integrations.llm import LLMEngine, _Request  # noqa: E402


def args(**more):
    base = dict(
        hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, max_model_len=128,
        max_num_seqs=3, kv_page_size=16,
    )
    return LLMArgs(**{**base, **more})


def ids_of(engine, prompts, steps):
    """Greedy tokens of all prompts at once, by the engine's own decode."""

    async def main():
        reqs = [_Request(engine.tokenizer.encode(p), n, 0.0) for p, n in zip(prompts, steps)]
        engine._queue = asyncio.Queue()  # a queue belongs to one event loop
        await engine.start()
        for r in reqs:
            await engine._queue.put(r)
        for r in reqs:
            await asyncio.wait_for(r.done.wait(), 120)
        await engine.stop()
        return [r.out_ids for r in reqs], [r.error for r in reqs]

    return asyncio.run(main())


PROMPTS = ["hello", "a longer prompt than the others, over three pages of sixteen", "x", "abc" * 9, "last one", "q" * 40]
STEPS = [5, 20, 1, 12, 33, 7]


def alone(engine, prompt, steps):
    """The same model without any cache, in 64 bits: the whole sequence again for each token."""
    engine.model.set_attn_implementation("eager")
    model = engine.model.double()
    ids = engine.tokenizer.encode(prompt)
    out = []
    with torch.inference_mode():
        for _ in range(steps):
            logits = model(input_ids=torch.tensor([ids], device=engine.device), use_cache=False).logits[0, -1]
            out.append(int(logits.argmax()))
            ids = ids + out[-1:]
            if out[-1] == engine.eos_id:
                break
    return out


def test_paged_tokens_are_the_models():
    """More requests than rows, joining as rows become free; each gets the tokens it would get alone."""
    if torch.cuda.is_available():
        pytest.skip("32-bit caches are the CPU's")
    got, errors = ids_of(LLMEngine(args(kv_cache="paged")), PROMPTS, STEPS)
    assert errors == [None] * len(PROMPTS)
    reference = LLMEngine(args())
    for prompt, steps, tokens in zip(PROMPTS, STEPS, got):
        assert tokens == alone(reference, prompt, steps)


def test_paged_with_few_pages_and_small_rows():
    """Requests wait for pages; one that can never fit is refused, and the others go on. The second prompt's 61 tokens and
    19 of the 20 that it asks for (the last is not held) fill five pages of 16 exactly."""
    engine = LLMEngine(args(kv_cache="paged", kv_pages=5))
    got, errors = ids_of(engine, PROMPTS, STEPS)
    assert errors == [None] * len(PROMPTS)
    assert [len(t) <= n for t, n in zip(got, STEPS)] == [True] * len(PROMPTS)
    engine = LLMEngine(args(kv_cache="paged", kv_pages=4))
    got, errors = ids_of(engine, PROMPTS, STEPS)
    assert isinstance(errors[1], ValueError) and errors[:1] + errors[2:] == [None] * 5
    assert engine.paged.cache.free_count.tolist() == [4] and engine.paged.cache.lens.tolist() == [0, 0, 0]
    assert sorted(engine.paged.cache.free_pages.tolist()) == list(range(4))
    # a request ends where its row does
    engine = LLMEngine(args(kv_cache="paged", max_model_len=32))
    got, errors = ids_of(engine, ["hello"], [100])
    assert errors == [None] and len(got[0]) <= 32 - 6 + 1
    if engine.eos_id not in got[0]:
        assert len(got[0]) == 32 - 6 + 1


def test_paged_e4m3_and_sampling_run():
    engine = LLMEngine(args(kv_cache="paged_e4m3"))
    assert engine.paged.cache.k.dtype == torch.float8_e4m3fn

    async def main():
        try:
            return await asyncio.gather(*[engine.generate(p, 6, temperature=0.8) for p in PROMPTS])
        finally:
            await engine.stop()

    assert all(isinstance(t, str) for t in asyncio.run(main()))


def test_paged_refusals():
    with pytest.raises(ValueError, match="kv_cache"):
        LLMEngine(args(kv_cache="none"))
    with pytest.raises(ValueError, match="head dim"):
        LLMEngine(args(kv_cache="paged", hidden_size=48, num_attention_heads=4))
    with pytest.raises(ValueError, match="page_size"):
        LLMEngine(args(kv_cache="paged", kv_page_size=17))
    if torch.cuda.is_available():
        with pytest.raises(ValueError, match="dtype"):
            LLMEngine(args(kv_cache="paged", dtype="float32"))
    engine = LLMEngine(args(kv_cache="paged"))
    got, errors = ids_of(engine, ["hello", "ok"], [0, 2])
    assert got[0] == [] and errors == [None, None] and len(got[1]) in (1, 2)
    with pytest.raises(RuntimeError, match="engine"):
        engine.model(input_ids=torch.tensor([[1, 2]], device=engine.device), use_cache=False)


def test_a_step_that_raises_ends_its_requests_and_no_more():
    engine = LLMEngine(args(kv_cache="paged"))
    whole, failed = engine.paged._forward, []

    def forward(*a):
        if not failed:
            failed.append(True)
            whole(*a)
            raise RuntimeError("planned")
        return whole(*a)

    engine.paged._forward = forward
    _, errors = ids_of(engine, ["hello", "there"], [3, 3])
    assert any(isinstance(e, RuntimeError) for e in errors)
    got, errors = ids_of(engine, ["hello"], [3])
    assert errors == [None] and 1 <= len(got[0]) <= 3
    assert engine.paged.cache.free_count.tolist() == [engine.paged.cache.pages]


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs MI355X")
@pytest.mark.parametrize("kind", ["paged", "paged_e4m3"])
@pytest.mark.parametrize("heads", [4, 2])  # head dims of 64 and 128
def test_paged_on_the_gpu(kind, heads):
    """bf16: the first token of each prompt is within rounding of the best one in 64 bits."""
    more = dict(hidden_size=256, intermediate_size=512, num_attention_heads=heads, kv_page_size=32)
    engine = LLMEngine(args(kv_cache=kind, **more))
    got, errors = ids_of(engine, PROMPTS, STEPS)
    assert errors == [None] * len(PROMPTS)
    assert engine.paged.cache.free_count.tolist() == [engine.paged.cache.pages]
    model = LLMEngine(args(**more)).model.double()
    model.set_attn_implementation("eager")
    for prompt, tokens in zip(PROMPTS, got):
        ids = torch.tensor([engine.tokenizer.encode(prompt)], device="cuda")
        with torch.inference_mode():
            logits = model(input_ids=ids, use_cache=False).logits[0, -1]
        # bf16 rounds what each of the 2 x 7 products and 4 sums of two layers gives: logits may be off by their spread
        # times a few 2^-8, e4m3 keys and values by 2^-4 of theirs; a wrong row or page moves them by the whole spread
        off = {"paged": 0.25, "paged_e4m3": 0.75}[kind]
        assert float(logits.max() - logits[tokens[0]]) <= off * float(logits.std())


def together(engine, requests):
    """generate() of (prompt, max_tokens, temperature) at once; each one's text or exception."""

    async def main():
        calls = [engine.generate(*r) for r in requests]
        try:
            return await asyncio.wait_for(asyncio.gather(*calls, return_exceptions=True), 120)
        finally:
            await engine.stop()

    return asyncio.run(main())


@pytest.mark.parametrize("temperature", [1e-40, 1e-300, 5e-324])
def test_a_temperature_next_to_zero_is_greedy_and_leaves_the_others_alone(temperature):
    want = together(LLMEngine(args(kv_cache="paged")), [("hello", 8, 0.0), ("bad", 8, 0.0)])
    got = together(LLMEngine(args(kv_cache="paged")), [("hello", 8, 0.0), ("bad", 8, temperature)])
    assert got == want


def test_a_temperature_without_bound_runs():
    got = together(LLMEngine(args(kv_cache="paged")), [("hello", 8, 1e300), ("there", 8, float("inf")), ("x", 3, float("nan"))])
    assert all(isinstance(t, str) for t in got)


def test_logits_that_are_no_numbers_end_their_own_request_only():
    want = together(LLMEngine(args(kv_cache="paged")), [("hello", 8, 0.0)])
    engine = LLMEngine(args(kv_cache="paged"))
    forward, calls = engine.model.forward, []

    def planted(*a, **more):
        out = forward(*a, **more)
        calls.append(out.logits.shape[1])
        if len(calls) == 3:  # a decode step of both requests: the second one's
            out.logits[0, 1, 7] = float("nan")
        return out

    engine.model.forward = planted
    got = together(engine, [("hello", 8, 0.0), ("there", 8, 0.5)])
    assert calls[2] == 2 and got[:1] == want
    assert isinstance(got[1], ValueError) and "finite" in str(got[1])
    assert engine.paged.cache.free_count.tolist() == [engine.paged.cache.pages]


class Held:
    """The engine's forward passes wait, from the first one on, until they are let go."""

    def __init__(self, engine):
        self.entered, self.go, forward = threading.Event(), threading.Event(), engine.paged._forward

        def wait(*a):
            self.entered.set()
            assert self.go.wait(60)
            return forward(*a)

        engine.paged._forward = wait


@pytest.mark.parametrize("another", [True, False])
def test_a_request_that_ends_in_a_step_whose_loop_was_stopped(another):
    """It is answered when the engine runs again, with another request or without one, in that step or after it."""
    for early in (False, True):
        engine = LLMEngine(args(kv_cache="paged"))
        held = Held(engine)

        async def main():
            in_thread = asyncio.get_event_loop().run_in_executor
            first = asyncio.create_task(engine.generate("hello", 1))
            assert await in_thread(None, held.entered.wait, 60)
            await engine.stop()
            if not early:
                held.go.set()
                while engine.paged.active:
                    await asyncio.sleep(0.01)
            if another:
                second = asyncio.create_task(engine.generate("there", 2))
                await asyncio.sleep(0)
            else:
                await engine.start()
            await asyncio.sleep(0.05)
            held.go.set()
            try:
                got = [await asyncio.wait_for(first, 30)]
                return got + ([await asyncio.wait_for(second, 30)] if another else [])
            finally:
                await engine.stop()

        got = asyncio.run(main())
        want = together(LLMEngine(args(kv_cache="paged")), [("hello", 1, 0.0), ("there", 2, 0.0)])
        assert got == want[: len(got)]


def test_a_request_whose_step_was_stopped_before_it_began():
    """The step waits for a thread when the loop is stopped, and never runs; its request is not lost with it."""
    engine = LLMEngine(args(kv_cache="paged"))
    busy, go = threading.Event(), threading.Event()

    def hold():
        busy.set()
        assert go.wait(60)

    async def main():
        loop = asyncio.get_event_loop()
        loop.set_default_executor(ThreadPoolExecutor(1))
        other = loop.run_in_executor(None, hold)
        while not busy.is_set():
            await asyncio.sleep(0.01)
        first = asyncio.create_task(engine.generate("hello", 3))
        await asyncio.sleep(0.05)
        await engine.stop()
        go.set()
        await other
        second = asyncio.create_task(engine.generate("there", 2))
        try:
            return [await asyncio.wait_for(t, 30) for t in (second, first)]
        finally:
            await engine.stop()

    want = together(LLMEngine(args(kv_cache="paged")), [("there", 2, 0.0), ("hello", 3, 0.0)])
    assert asyncio.run(main()) == want


def test_a_cache_that_cannot_be_reset_ends_every_request():
    """As after a device error, which the release meets again: those in flight, those that wait, and all later ones."""
    engine = LLMEngine(args(kv_cache="paged", max_num_seqs=2))

    def planted(*a):
        raise RuntimeError("planned")

    engine.paged._forward = engine.paged.cache.release = planted
    got = together(engine, [("hello", 3, 0.0), ("there", 3, 0.0), ("waits", 3, 0.0)])
    assert [type(e) for e in got] == [RuntimeError] * 3 and not engine.paged.active
    engine._queue = asyncio.Queue()
    got = together(engine, [("later", 3, 0.0)])
    assert isinstance(got[0], RuntimeError) and "reset" in str(got[0])


@pytest.mark.parametrize("kind", ["dense", "paged"])
def test_a_loop_that_has_finished_is_begun_again(kind):
    engine = LLMEngine(args(kv_cache=kind))

    async def main():
        first = await engine.generate("hello", 2)
        engine._task.cancel()
        await asyncio.wait([engine._task])
        try:
            return first, await asyncio.wait_for(engine.generate("hello", 2), 30)
        finally:
            await engine.stop()

    first, second = asyncio.run(main())
    assert first == second


def test_models_that_need_more_than_full_attention_are_refused_when_built():
    """A window for all layers is no layer type, and a cap on the scores neither: both came out at the first request."""
    from transformers import Gemma2Config, Gemma2ForCausalLM, MistralConfig, MistralForCausalLM

    from beta9_amd.integrations.llm_paged import PagedDecoder

    sizes = dict(
        vocab_size=300, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
        head_dim=16, max_position_embeddings=128,
    )
    build = lambda model: PagedDecoder(model.eval(), args(kv_cache="paged"), None, torch.float32, "cpu")  # noqa: E731
    with pytest.raises(ValueError, match="sliding_window"):
        build(MistralForCausalLM(MistralConfig(sliding_window=32, **sizes)))
    full = dict(layer_types=["full_attention"] * 2, **sizes)
    with pytest.raises(ValueError, match="softcapping"):
        build(Gemma2ForCausalLM(Gemma2Config(attn_logit_softcapping=30.0, **full)))
    # without a window and a cap they are served
    for model in (
        MistralForCausalLM(MistralConfig(sliding_window=None, **sizes)),
        Gemma2ForCausalLM(Gemma2Config(attn_logit_softcapping=None, query_pre_attn_scalar=16, **full)),
    ):
        decoder, req = build(model), _Request([5, 6, 7], 4, 0.0)
        decoder.submit(req)
        while decoder.active:
            decoder.step()
        assert decoder.take_ended() == [req] and req.error is None
        ids = [5, 6, 7]
        model.set_attn_implementation("eager")
        with torch.inference_mode():
            for token in req.out_ids:
                logits = model(input_ids=torch.tensor([ids]), use_cache=False).logits[0, -1]
                # the same sums in another order: about 20 one after the other, of at most 128 terms, each off by 2^-24 a term
                assert float(logits.max() - logits[token]) <= 1e-3 * float(logits.std())
                ids.append(token)
        assert len(req.out_ids) == 4


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs MI355X")
@pytest.mark.parametrize("kind", ["paged", "paged_e4m3"])
@pytest.mark.parametrize("heads", [4, 2])
def test_every_token_of_the_paged_engine_on_the_gpu(kind, heads):
    """Each token, those of the decode steps too, is within rounding of the best one in 64 bits behind the tokens before it."""
    more = dict(hidden_size=256, intermediate_size=512, num_attention_heads=heads, kv_page_size=32)
    engine = LLMEngine(args(kv_cache=kind, **more))
    engine.eos_id = engine.paged.eos_id = None
    got, errors = ids_of(engine, PROMPTS, STEPS)
    assert errors == [None] * len(PROMPTS) and [len(t) for t in got] == STEPS
    model = LLMEngine(args(**more)).model.double()
    model.set_attn_implementation("eager")
    # as for the first token: two layers' 2 x 7 products and 4 sums round to bf16, and with them each key and value that the
    # cache holds, in e4m3 to 2^-4; a wrong row, page or position moves logits by their whole spread
    off = {"paged": 0.25, "paged_e4m3": 0.75}[kind]
    for prompt, tokens in zip(PROMPTS, got):
        ids = engine.tokenizer.encode(prompt)
        with torch.inference_mode():
            whole = torch.tensor([ids + tokens[:-1]], device="cuda")
            logits = model(input_ids=whole, use_cache=False).logits[0, len(ids) - 1 :]
        far = logits.max(-1).values - logits.gather(1, torch.tensor(tokens, device="cuda")[:, None])[:, 0]
        assert (far <= off * logits.std(-1)).all()


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs MI355X")
def test_sampling_on_the_gpu():
    """Temperatures of any size beside each other, and logits that are no numbers."""
    engine = LLMEngine(args(kv_cache="paged"))
    got = together(engine, [(p, 6, t) for p, t in zip(PROMPTS, (1e-40, 0.8, 1e300, float("inf"), 0.0, 1e-300))])
    assert all(isinstance(t, str) for t in got)
    engine._queue, forward = asyncio.Queue(), engine.model.forward

    def planted(*a, **more):
        out = forward(*a, **more)
        out.logits[0, -1, 7] = float("nan")
        return out

    engine.model.forward = planted
    got = together(engine, [("hello", 3, 0.0), ("there", 3, 0.5)])
    assert isinstance(got[0], str) and isinstance(got[1], ValueError)
    assert engine.paged.cache.free_count.tolist() == [engine.paged.cache.pages]
