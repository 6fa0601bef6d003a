"""Several prompts in one pass, and answers drawn by given numbers, on the operators' plain forms (CPU); see test_generate.py for the bound."""
import pytest
import torch

from mccl_b200 import ops
from mccl_b200.models import Generator, build_decoder
from tests.generate_checks import dequantized, reference_logits, rms, sharpen

FAMILIES = {"gelu": {}, "swiglu": dict(act="swiglu", norm="rmsnorm", pos="rope", tied=False)}


def model_of(family, device="cpu", **changes):
    torch.manual_seed(0)
    return sharpen(build_decoder("tiny", **{**FAMILIES[family], **changes}).to(device))


@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("weights", ["bf16", "w4"])
def test_prompts_together(family, weights):
    model = model_of(family)
    gen = Generator(model, max_sequences=5, page_size=8, weights=weights, group=64)
    texts = [torch.randint(0, 512, (n,)) for n in (1, 30, 17, 8)]
    rows, logits = gen.prefill_together([t[:-1] if len(t) > 1 else t for t in texts])
    assert [gen.cache.length(r) for r in rows] == [1, 29, 16, 7]
    matrices = dequantized(model, 64) if weights == "w4" else None
    next_logits = gen.step(rows[1:], torch.stack([t[-1] for t in texts[1:]]))
    with torch.no_grad():
        want = torch.stack([reference_logits(model, t[:-1] if len(t) > 1 else t, matrices)[-1] for t in texts])
        then = torch.stack([reference_logits(model, t, matrices)[-1] for t in texts[1:]])
        whole = rms(torch.stack([model(t[None])[0, -1] for t in texts[1:]]).float() - torch.stack([reference_logits(model, t)[-1] for t in texts[1:]]))
    assert rms(logits.float() - want) <= 3 * whole and rms(next_logits.float() - then) <= 3 * whole   # few rows scatter more than many


def test_a_window_in_one_pass():
    model = model_of("swiglu")
    gen = Generator(model, max_sequences=2, page_size=4, window=10, sinks=2)
    one = Generator(model, max_sequences=2, page_size=4, window=10, sinks=2)
    tokens = torch.randint(0, 512, (40,))
    rows, logits = gen.prefill_together([tokens, tokens[:7]])
    row, want = one.prefill(tokens)
    scale = rms(want.float())
    assert rms(logits[0].float() - want.float()) < 0.1 * scale
    assert gen.cache.free_pages == gen.cache.pages.shape[2] - len([p for r in rows for p in gen.cache.row_pages(r) if p >= 0])
    assert min(gen.cache.row_pages(rows[0])) == -1
    a, b = gen.step([rows[0]], [3]), one.step([row], [3])
    assert rms(a.float() - b.float()) < 0.1 * scale


def test_refusals_leave_nothing_behind():
    gen = Generator(model_of("gelu"), max_sequences=2, pages=3, page_size=8)
    free = gen.cache.free_pages
    for bad in ([[1], []], [[1], [2], [3]], [[1] * 20, [2] * 9], [[1], [600]], [[1] * 65]):
        with pytest.raises(RuntimeError):
            gen.prefill_together(bad)
        assert gen.cache.free_pages == free and gen.cache.rows == []
    rows, logits = gen.prefill_together([])
    assert rows == [] and logits.shape == (0, 512)


def test_generate_draws_by_given_numbers():
    model = model_of("gelu")
    gen = Generator(model, max_sequences=3, page_size=8)
    prompts = [[1, 2, 3], [4], [5, 6]]
    draw = lambda **o: gen.generate(prompts, 6, generator=torch.Generator().manual_seed(7), **o)
    a = draw(temperature=1.0, top_k=20, top_p=0.9, min_p=0.01, together=True)
    assert a == draw(temperature=1.0, top_k=20, top_p=0.9, min_p=0.01, together=True) and all(len(t) == 6 for t in a)
    assert draw(temperature=1.0, top_k=1) == gen.generate(prompts, 6)
    # the first tokens are what the operator draws from the prompts' logits
    rows, logits = gen.prefill_together(prompts)
    u = torch.rand(3, generator=torch.Generator().manual_seed(7))
    assert [t[0] for t in a] == ops.sample(logits.float(), u, temperature=1.0, top_k=20, top_p=0.9, min_p=0.01).tolist()
    for r in rows:
        gen.free(r)
    assert gen.generate(prompts, 3, together=True) == gen.generate(prompts, 3) and gen.cache.rows == []
    for bad in ({"top_p": 1.5}, {"top_k": -1}, {"min_p": -0.1}):
        with pytest.raises(RuntimeError):
            draw(temperature=1.0, **bad)
        assert gen.cache.rows == []


def test_logits_that_are_not_finite_are_refused():
    model = model_of("gelu")
    with torch.no_grad():
        model.ln_f.weight.fill_(float("nan"))
    gen = Generator(model, max_sequences=1, page_size=8)
    with pytest.raises(RuntimeError, match="not finite"):
        gen.generate([[1]], 2, temperature=1.0, top_p=0.9)
    assert gen.cache.rows == []
