"""The paged cache's bookkeeping, and answering token by token on the operators' plain forms.

Logits of the generator and of the model's own forward over the whole text are both computed with bf16 activations; neither is nearer to the model in 32
bits by construction, so the generator may be off by at most twice as much (root mean square) as that forward."""
import dataclasses

import pytest
import torch

from mccl_b200 import ops
from mccl_b200.models import Generator, PagedKVCache, build_decoder
from tests.generate_checks import dequantized, reference_logits, rms, sharpen

FAMILIES = {"gelu": {}, "swiglu": dict(act="swiglu", norm="rmsnorm", pos="rope", tied=False)}


def cache_of(pages=10, rows=4, page_size=4, layers=2):
    return PagedKVCache(layers, 2, 8, pages=pages, max_sequences=rows, max_positions=32, page_size=page_size, device="cpu", dtype=torch.float16)


def fill(cache, row, length, seed):
    """`length` positions of a sequence with values of their own; returns them."""
    g = torch.Generator().manual_seed(seed)
    cache.reserve([row], [length])
    kv = torch.randn(cache.pages.shape[0], 2, length, 2, 8, generator=g).half()
    positions = torch.arange(length, dtype=torch.int32)
    for i in range(cache.pages.shape[0]):
        ops.paged_append(kv[i, 0], kv[i, 1], cache.keys(i), cache.values(i), cache.table, positions, rows=torch.full((length,), row, dtype=torch.int32))
    cache.set_length(row, length)
    return kv


def read(cache, row):
    length = cache.length(row)
    at = torch.arange(length)
    page = cache.table[row, at // cache.page_size].long()
    assert (page >= 0).all()
    return torch.stack([cache.pages[:, :, p, :, o] for p, o in zip(page.tolist(), (at % cache.page_size).tolist())], dim=2)


def test_sequences_keep_what_they_hold():
    cache = cache_of(pages=12)
    a, b = cache.add(), cache.add()
    assert (a, b) == (0, 1)
    kv_a, kv_b = fill(cache, a, 10, 1), fill(cache, b, 4, 2)
    assert cache.free_pages == 12 - 3 - 1
    assert torch.equal(read(cache, a), kv_a) and torch.equal(read(cache, b), kv_b)
    c, d = cache.fork(a, 2)
    assert cache.free_pages == 8 - 2   # two full pages are shared, the last one is copied twice
    assert cache.row_pages(c)[:2] == cache.row_pages(a)[:2] and len({cache.row_pages(r)[2] for r in (a, c, d)}) == 3
    assert all(torch.equal(read(cache, r), kv_a) for r in (c, d)) and cache.lengths.tolist() == [10, 4, 10, 10]
    # what one sequence appends, the others do not see
    cache.reserve([c], [11])
    one = torch.ones(1, 2, 8).half()
    ops.paged_append(one, one, cache.keys(0), cache.values(0), cache.table, torch.tensor([10], dtype=torch.int32), rows=torch.tensor([c], dtype=torch.int32))
    cache.set_length(c, 11)
    assert torch.equal(read(cache, a), kv_a) and torch.equal(read(cache, c)[:, :, :10], kv_a)
    with pytest.raises(RuntimeError, match="rows are taken"):
        cache.add()
    cache.free(a)
    assert cache.free_pages == 7 and torch.equal(read(cache, d), kv_a)   # its full pages have other owners
    cache.free(c)
    cache.free(b)
    cache.free(d)
    assert cache.free_pages == 12 and (cache.table == -1).all() and cache.rows == []


def test_fork_of_whole_pages_copies_nothing():
    cache = cache_of()
    a = cache.add()
    kv = fill(cache, a, 8, 3)
    (b,) = cache.fork(a)
    assert cache.free_pages == 8 and cache.row_pages(a) == cache.row_pages(b) and torch.equal(read(cache, b), kv)
    (c,) = cache.fork(cache.add())   # an empty one
    assert cache.length(c) == 0 and cache.row_pages(c) == []


@pytest.mark.parametrize("seed", range(5))
def test_compact(seed):
    g = torch.Generator().manual_seed(seed)
    cache = cache_of(pages=40, rows=12)
    held = {}
    for step in range(30):
        kind = int(torch.randint(0, 4, (1,), generator=g))
        if kind <= 1 and len(cache.rows) < 12 and cache.free_pages >= 8:
            row = cache.add()
            held[row] = fill(cache, row, int(torch.randint(1, 30, (1,), generator=g)), step)
        elif kind == 2 and held and len(cache.rows) < 12 and cache.free_pages >= 1:
            row = sorted(held)[int(torch.randint(0, len(held), (1,), generator=g))]
            (new,) = cache.fork(row)
            held[new] = held[row]
        elif kind == 3 and held:
            row = sorted(held)[int(torch.randint(0, len(held), (1,), generator=g))]
            cache.free(row)
            del held[row]
        if step % 7 == 6:
            used = cache.compact()
            taken = {p for r in cache.rows for p in cache.row_pages(r)}
            assert taken == set(range(used)) and cache.free_pages == 40 - used
        assert all(torch.equal(read(cache, r), kv) for r, kv in held.items())
    assert cache.compact() == cache.compact()


def test_pages_that_nobody_will_see():
    cache = cache_of(pages=8, rows=2)
    a = cache.add()
    fill(cache, a, 27, 1)   # 7 pages of 4
    (b,) = cache.fork(a)
    assert cache.free_pages == 0
    # the first page stays for one sink, the window of 10 reaches back to position 18 of the next token
    assert cache.drop_unseen([a], 10, 1) == 0                # the other sequence still has them
    assert cache.row_pages(a)[1:4] == [-1] * 3 and cache.row_pages(a)[0] >= 0 and -1 not in cache.row_pages(a)[4:]
    assert cache.table[a, 1:4].tolist() == [-1] * 3 and -1 not in cache.row_pages(b)
    assert cache.drop_unseen([b], 10, 1) == 3 and cache.free_pages == 3
    assert cache.drop_unseen([a, b], 10, 1) == 0
    (c,) = cache.fork(a) if len(cache.rows) < 2 else (None,)
    cache.free(a)
    cache.free(b)
    assert cache.free_pages == 8


def test_a_full_cache_changes_nothing():
    cache = cache_of(pages=4)
    a, b = cache.add(), cache.add()
    kv = fill(cache, a, 9, 1)
    before = cache.table.clone()
    for call in (lambda: cache.reserve([a, b], [16, 8]), lambda: cache.reserve([b], [33]), lambda: cache.fork(a, 2), lambda: cache.set_length(b, 1), lambda: cache.advance([a, b], 1),
                 lambda: cache.length(3), lambda: cache.free(3), lambda: cache.reserve([3], [1])):
        with pytest.raises(RuntimeError, match="PagedKVCache"):
            call()
        assert torch.equal(cache.table, before) and cache.free_pages == 1 and cache.rows == [a, b] and torch.equal(read(cache, a), kv)
    for bad in (dict(pages=0), dict(max_sequences=0), dict(page_size=0), dict(max_positions=0)):
        with pytest.raises(RuntimeError, match="PagedKVCache"):
            PagedKVCache(1, 1, 8, device="cpu", **{**dict(pages=1, max_sequences=1, max_positions=1), **bad})
    with pytest.raises(RuntimeError, match="head_dim"):
        PagedKVCache(1, 1, 12, device="cpu", pages=1, max_sequences=1, max_positions=1)


@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("weights", ["bf16", "w4"])
def test_steps_are_the_whole_text(family, weights):
    torch.manual_seed(0)
    model = sharpen(build_decoder("tiny", **FAMILIES[family]))
    tokens = torch.randint(0, 512, (30,))
    gen = Generator(model, max_sequences=2, page_size=8, weights=weights, group=64)
    row, logits = gen.prefill(tokens[:11])
    got = torch.stack([logits] + [gen.step([row], tokens[i:i + 1])[0] for i in range(11, 30)]).float()
    with torch.no_grad():
        want = reference_logits(model, tokens, dequantized(model, 64) if weights == "w4" else None)[10:]
        whole = rms(model(tokens[None])[0, 10:].float() - reference_logits(model, tokens)[10:])
    assert rms(got - want) <= 2 * whole and rms(want) > 10 * whole
    assert gen.cache.length(row) == 30


def test_sequences_side_by_side_and_forks():
    torch.manual_seed(1)
    model = sharpen(build_decoder("tiny"))
    gen = Generator(model, max_sequences=4, page_size=8)
    a, _ = gen.prefill([1, 2, 3])
    b, _ = gen.prefill(list(range(9)))
    (c,) = gen.fork(b)
    together = gen.step([c, a, b], [7, 8, 9])
    alone = Generator(model, max_sequences=4, page_size=8)
    for k, (prompt, token) in enumerate(((list(range(9)), 7), ([1, 2, 3], 8), (list(range(9)), 9))):
        row, _ = alone.prefill(prompt)
        assert torch.allclose(alone.step([row], [token])[0].float(), together[k].float(), atol=0.03)
    assert [gen.cache.length(r) for r in (a, b, c)] == [4, 10, 10]


def test_a_window():
    torch.manual_seed(2)
    model = sharpen(build_decoder("tiny", act="swiglu", norm="rmsnorm", pos="rope", tied=False))
    tokens = torch.randint(0, 512, (40,))
    gen = Generator(model, max_sequences=1, page_size=4, pages=6, window=9, sinks=2)   # 24 positions' room for 40
    row, logits = gen.prefill(tokens[:20])
    got = torch.stack([logits] + [gen.step([row], tokens[i:i + 1])[0] for i in range(20, 40)]).float()
    with torch.no_grad():
        want = reference_logits(model, tokens, window=9, sinks=2)[19:]
        whole = rms(model(tokens[None])[0, 19:].float() - reference_logits(model, tokens)[19:])
    assert rms(got - want) <= 2 * whole and rms(want - reference_logits(model, tokens)[19:]) > 10 * whole
    assert gen.cache.free_pages >= 1


def test_generate():
    torch.manual_seed(3)
    model = sharpen(build_decoder("tiny"))
    gen = Generator(model, max_sequences=3, page_size=8)
    prompts = [[5], list(range(20)), [9, 8, 7]]
    texts = gen.generate(prompts, 6)
    assert [len(t) for t in texts] == [6, 6, 6] and gen.cache.free_pages == gen.cache.pages.shape[2] and gen.cache.rows == []
    # greedy: each token is the likeliest behind what was there
    for prompt, text in zip(prompts, texts):
        row, logits = gen.prefill(prompt)
        for token in text:
            assert logits.float().max() - logits.float()[token] <= 0.03
            logits = gen.step([row], [token])[0]
        gen.free(row)
    assert gen.generate(prompts, 6, stop=texts[1][0])[1] == texts[1][:1]
    assert len(gen.generate([[1] * 62], 10)[0]) == 3    # positions 62 and 63, and the token behind them
    g = torch.Generator().manual_seed(0)
    drawn = gen.generate([[1, 2]], 5, temperature=1.0, generator=g)
    assert drawn == gen.generate([[1, 2]], 5, temperature=1.0, generator=g.manual_seed(0))
    assert gen.generate([], 5) == [] and gen.generate([[1]], 0) == [[]]
    assert gen.cache.rows == []


def test_refusals():
    model = build_decoder("tiny")
    for kw in (dict(weights="int8"), dict(window=0), dict(sinks=1), dict(window=3, sinks=-1), dict(max_positions=65)):
        with pytest.raises(RuntimeError):
            Generator(model, **kw)
    with pytest.raises(RuntimeError):
        Generator(torch.nn.Linear(2, 2))
    wrapped = build_decoder("tiny")
    wrapped.blocks[0].up = torch.nn.Linear(128, 512)
    with pytest.raises(RuntimeError, match="replaced"):
        Generator(wrapped)
    gen = Generator(model, max_sequences=2, pages=3, page_size=16)
    row, _ = gen.prefill([1, 2])
    for call in (lambda: gen.prefill([]), lambda: gen.prefill([1] * 65), lambda: gen.step([row, row], [1, 2]), lambda: gen.step([row], [1, 2]), lambda: gen.step([1], [1]),
                 lambda: gen.prefill([1] * 40)):
        with pytest.raises(RuntimeError):
            call()
    assert gen.cache.rows == [row] and gen.cache.length(row) == 2 and gen.cache.free_pages == 2
    assert gen.step([], []).shape == (0, 512)


def test_a_fork_that_goes_back():
    torch.manual_seed(4)
    model = sharpen(build_decoder("tiny"))
    prompt = list(range(16))
    gen, alone = Generator(model, max_sequences=3, page_size=8), Generator(model, max_sequences=3, page_size=8)
    a, _ = gen.prefill(prompt)
    (b,) = gen.fork(a)
    gen.cache.set_length(b, 13)
    for tokens in ((40, 50), (41, 51), (42, 52), (43, 53)):
        got = gen.step([a, b], tokens)
    one, _ = alone.prefill(prompt)
    two, _ = alone.prefill(prompt[:13])
    for tokens in ((40, 50), (41, 51), (42, 52), (43, 53)):
        want = torch.cat([alone.step([r], [t]) for r, t in zip((one, two), tokens)])
    assert torch.allclose(got.float(), want.float(), atol=0.03)


class Adapted(type(build_decoder("tiny").blocks[0].up)):
    def forward(self, x, native, act="none", residual=None):
        return super().forward(x, native, act, residual) * 1.5


class Scaled(torch.nn.Embedding):
    def forward(self, ids):
        return super().forward(ids) * 2.0


def _adapter(model):
    model.blocks[1].up.__class__ = Adapted


def _embedding(model):
    model.tok.__class__ = Scaled


def _own_forward(model):
    first = model.blocks[0].proj
    stock = first.forward
    first.forward = lambda *a, **k: stock(*a, **k) * 1.5


def _own_head(model):
    model.head_weight = lambda: model.tok.weight * 2.0


def _other_heads(model):
    model.blocks[0].cfg = dataclasses.replace(model.cfg, n_heads=2)


CHANGES = {"adapter": _adapter, "embedding": _embedding, "forward": _own_forward, "head": _own_head, "heads": _other_heads,
           "hook-block": lambda m: m.blocks[0].register_forward_hook(lambda mod, args, out: out * 1.5),
           "hook-projection": lambda m: m.blocks[1].qkv.register_forward_pre_hook(lambda mod, args: (args[0] * 1.5, *args[1:])),
           "hook-norm": lambda m: m.ln_f.register_forward_hook(lambda mod, args, out: out * 1.5),
           "hook-embedding": lambda m: m.tok.register_forward_hook(lambda mod, args, out: out * 1.5),
           "hook-model": lambda m: m.register_forward_hook(lambda mod, args, out: out * 1.5)}


@pytest.mark.parametrize("change", list(CHANGES))
def test_a_changed_model_is_refused(change):
    model = build_decoder("tiny")
    CHANGES[change](model)
    with pytest.raises(RuntimeError, match="Generator"):
        Generator(model)


def test_hooks_of_all_modules_are_refused():
    model = build_decoder("tiny")
    handle = torch.nn.modules.module.register_module_forward_hook(lambda mod, args, out: None)
    try:
        with pytest.raises(RuntimeError, match="Generator"):
            Generator(model)
    finally:
        handle.remove()
    Generator(model)


def _norms(model):
    for i, m in enumerate(m for m in model.modules() if hasattr(m, "eps") and hasattr(m, "kind")):
        m.eps = (0.02, 0.1, 0.5)[i % 3]


def _parametrized(model):
    class Half(torch.nn.Module):
        def forward(self, w):
            return w * 0.5
    torch.nn.utils.parametrize.register_parametrization(model.blocks[0].up, "weight", Half())


@pytest.mark.parametrize("change", [_norms, _parametrized])
@pytest.mark.parametrize("family", list(FAMILIES))
def test_a_changed_model_that_can_be_answered_for(family, change):
    """What a norm adds under its root, and a weight that is computed, are the module's own."""
    if family == "swiglu" and change is _parametrized:
        pytest.skip("one family shows it")
    torch.manual_seed(5)
    model = sharpen(build_decoder("tiny", **FAMILIES[family]))
    before = Generator(model).prefill(range(10))[1].float()
    change(model)
    gen = Generator(model)
    row, first = gen.prefill(range(10))
    got = torch.stack([first, gen.step([row], [10])[0]]).float()
    with torch.no_grad():
        want = model(torch.arange(11)[None])[0, 9:].float()
    assert rms(got[0] - before) > 10 * rms(got - want) and torch.allclose(got, want, atol=0.05)


def test_tokens_outside_the_vocabulary():
    gen = Generator(build_decoder("tiny"), max_sequences=2)
    row, _ = gen.prefill([1, 2])
    free = gen.cache.free_pages
    for bad in (512, -1, 2 ** 40):
        for call in (lambda: gen.prefill([1, bad]), lambda: gen.step([row], [bad]), lambda: gen.step([row], torch.tensor([bad])), lambda: gen.generate([[1], [bad]], 2)):
            with pytest.raises(RuntimeError, match="vocabulary"):
                call()
            assert gen.cache.rows == [row] and gen.cache.length(row) == 2 and gen.cache.free_pages == free
    gen.step([row], [511])


def test_temperatures_near_zero():
    """What is drawn is among the likeliest: bf16 logits may be equal."""
    torch.manual_seed(7)
    gen = Generator(sharpen(build_decoder("tiny")), max_sequences=1)
    for temperature in (1e-20, 1e-39, 1e-46):
        for prompt in ([1, 2], [3]):
            (text,) = gen.generate([prompt], 4, temperature=temperature)
            row, logits = gen.prefill(prompt)
            for token in text:
                assert logits[token] == logits.max()
                logits = gen.step([row], [token])[0]
            gen.free(row)
    assert gen.cache.rows == []


def test_no_token_is_drawn_from_logits_that_are_no_numbers():
    model = build_decoder("tiny")
    with torch.no_grad():
        model.ln_f.weight[3] = float("nan")
    gen = Generator(model, max_sequences=2)
    with pytest.raises(RuntimeError, match="Generator"):
        gen.generate([[1, 2]], 3, temperature=1.0)
    assert gen.cache.rows == []


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_weights_that_are_no_numbers_are_not_quantized(value):
    w = torch.randn(20, 128)
    w[17, 100] = value
    with pytest.raises(RuntimeError, match="quantize_w4"):
        ops.quantize_w4(w, 64)
    w[17, 100] = 0.0
    ops.quantize_w4(w, 64)
    with pytest.raises(RuntimeError, match="quantize_w4"):
        ops.quantize_w4(torch.tensor([3e38, -3e38]).repeat(1, 16), 32)     # a range that no scale spans
    assert ops.quantize_w4(w[:0], 64).shape == (0, 128)
