"""Answering token by token on the native operators, see test_generate.py for the bound."""
import gc

import pytest
import torch

from mccl_b200 import ops
from mccl_b200.models import Generator, PagedKVCache, build_decoder
from tests.generate_checks import dequantized, reference_logits, rms, sharpen

pytestmark = pytest.mark.gpu
MODELS = {"tiny": ("tiny", {}), "70m": ("70m", dict(n_layers=3)), "110m": ("110m", dict(n_layers=2, vocab=1000)),
          "swiglu": ("1.3b", dict(n_layers=2, vocab=1024, max_seq=512)), "swiglu-narrow": ("1.3b", dict(n_layers=2, vocab=512, d_model=192, n_heads=3, d_ff=320, max_seq=300))}


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("weights", ["bf16", "w4"])
@pytest.mark.parametrize("graph", [True, False])
def test_steps_are_the_whole_text(name, weights, graph):
    torch.manual_seed(0)
    preset, changes = MODELS[name]
    model = sharpen(build_decoder(preset, **changes).cuda())
    count = min(model.cfg.max_seq, 150)
    tokens = torch.randint(0, model.cfg.vocab, (count,), device="cuda")
    gen = Generator(model, max_sequences=2, page_size=16, weights=weights, group=64, use_graph=graph)
    first = count * 2 // 3
    row, logits = gen.prefill(tokens[:first])
    got = torch.stack([logits] + [gen.step([row], tokens[i:i + 1])[0] for i in range(first, count)]).float()
    with torch.no_grad():
        want = reference_logits(model, tokens, dequantized(model, 64) if weights == "w4" else None)[first - 1:]
        whole = rms(model(tokens[None])[0, first - 1:].float() - reference_logits(model, tokens)[first - 1:])
    assert rms(got - want) <= 2 * whole and rms(want) > 10 * whole


@pytest.mark.parametrize("weights", ["bf16", "w4"])
def test_many_sequences(weights):
    torch.manual_seed(1)
    model = sharpen(build_decoder("70m", n_layers=2).cuda())
    gen = Generator(model, max_sequences=40, page_size=16, weights=weights)
    lengths = [1 + 5 * i % 97 for i in range(40)]
    texts = [torch.randint(0, 32000, (n + 3,), device="cuda") for n in lengths]
    rows = [gen.prefill(t[:n])[0] for t, n in zip(texts, lengths)]
    matrices = dequantized(model, 128) if weights == "w4" else None
    for step in range(3):
        got = gen.step(rows, torch.stack([t[n + step] for t, n in zip(texts, lengths)]))
    with torch.no_grad():
        want = torch.stack([reference_logits(model, t, matrices)[-1] for t in texts])
        whole = rms(torch.stack([model(t[None])[0, -1] for t in texts]).float() - torch.stack([reference_logits(model, t)[-1] for t in texts]))
    assert rms(got.float() - want) <= 2 * whole
    # fewer of them, in another order, forked and moved
    for r in rows[5:30]:
        gen.free(r)
    new = gen.fork(rows[2], 2)
    gen.cache.compact()
    again = [rows[35], new[0], rows[2], new[1], rows[0]]
    out = gen.step(again, torch.tensor([7, 8, 8, 9, 10]))
    with torch.no_grad():
        for k, (i, token) in enumerate(((35, 7), (2, 8), (2, 8), (2, 9), (0, 10))):
            text = torch.cat((texts[i], torch.tensor([token], device="cuda")))
            assert rms(out[k].float() - reference_logits(model, text, matrices)[-1]) <= 3 * whole   # one row alone scatters more than the mean of many
    assert torch.equal(out[1], out[2])


def test_a_window():
    torch.manual_seed(2)
    model = sharpen(build_decoder("1.3b", n_layers=2, vocab=512, d_model=256, n_heads=4, d_ff=512, max_seq=400).cuda())
    tokens = torch.randint(0, 512, (400,), device="cuda")
    gen = Generator(model, max_sequences=1, page_size=16, pages=10, window=100, sinks=5)   # 160 positions' room for 400
    row, logits = gen.prefill(tokens[:200])
    got = torch.stack([logits] + [gen.step([row], tokens[i:i + 1])[0] for i in range(200, 400)]).float()
    with torch.no_grad():
        want = reference_logits(model, tokens, window=100, sinks=5)[199:]
        whole = rms(model(tokens[None])[0, 199:].float() - reference_logits(model, tokens)[199:])
    assert rms(got - want) <= 2 * whole


def test_native_kernels_run():
    model = build_decoder("tiny").cuda()
    gen = Generator(model, max_sequences=2, weights="w4", group=64, use_graph=False)
    row, _ = gen.prefill([1, 2, 3])
    before = ops.launch_count()
    gen.step([row], [4])
    # per layer: two norms, four 4-bit products, append, attention; the last norm and the vocabulary projection
    assert ops.launch_count() - before >= 2 * 8 + 2


def test_cache_on_the_gpu():
    cache = PagedKVCache(3, 2, 32, pages=20, max_sequences=4, max_positions=64, page_size=16)
    a = cache.add()
    cache.reserve([a], [40])
    cache.pages[:, :, cache.row_pages(a)] = torch.randn(3, 2, 3, 2, 16, 32, device="cuda").bfloat16()
    cache.set_length(a, 40)
    held = cache.pages[:, :, cache.row_pages(a)].clone()
    b, c = cache.fork(a, 2)
    cache.free(a)
    assert cache.compact() == 4
    for row in (b, c):
        assert torch.equal(cache.pages[:, :, cache.row_pages(row)], held)
        assert cache.table[row, :3].tolist() == cache.row_pages(row)


def test_generate():
    torch.manual_seed(3)
    model = sharpen(build_decoder("70m", n_layers=2).cuda())
    gen = Generator(model, max_sequences=3, weights="w4")
    texts = gen.generate([[5], list(range(20)), [9, 8, 7]], 6)
    assert [len(t) for t in texts] == [6, 6, 6] and gen.cache.rows == []
    assert texts == gen.generate([[5], list(range(20)), [9, 8, 7]], 6)


def test_a_step_is_captured_on_a_stream_of_the_models_device(monkeypatch):
    """Without a stream of its own a capture takes one of the device that was current at the process's first capture."""
    model = build_decoder("tiny").cuda()
    gen = Generator(model, max_sequences=2)
    row, _ = gen.prefill([1, 2, 3])
    seen, stock = [], torch.cuda.graph

    class Graph(stock):
        def __init__(self, graph, pool=None, stream=None, **kw):
            seen.append((stream, torch.cuda.current_device()))
            super().__init__(graph, pool=pool, stream=stream, **kw)

    monkeypatch.setattr(torch.cuda, "graph", Graph)
    gen.step([row], [4])
    (stream, current), = seen
    assert stream is not None and stream.device == gen.device and current == gen.device.index


def test_prompts_and_steps_run_with_the_models_device_current(monkeypatch):
    model = build_decoder("tiny").cuda()
    gen = Generator(model, max_sequences=2)
    entered, stock = [], torch.cuda.device

    class Device(stock):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    monkeypatch.setattr(torch.cuda, "device", Device)
    row, _ = gen.prefill([1, 2, 3])
    assert entered[:1] == [gen.device.index]
    for _ in range(2):      # captured, replayed
        entered.clear()
        gen.step([row], [4])
        assert entered[:1] == [gen.device.index]


def test_garbage_with_graphs_does_not_break_a_capture():
    """A generator in a reference cycle, with its graph, that nobody has collected when another one captures."""
    model = build_decoder("tiny").cuda()
    gen = Generator(model, max_sequences=2)
    row, _ = gen.prefill([1, 2, 3])
    stock, calls, kept = gen._one, [], []

    def one(rows, ids):
        calls.append(gc.isenabled())
        if torch.cuda.is_current_stream_capturing():
            kept.pop()
            for _ in range(3):
                [[] for _ in range(3 * gc.get_threshold()[0])]      # allocations enough for the collector to run by itself
        return stock(rows, ids)

    gen._one = one
    other = Generator(model, max_sequences=2)
    other.step([other.prefill([1, 2])[0]], [3])
    other.me = other
    kept.append(other)
    threshold = gc.get_threshold()
    gc.collect()
    del other
    try:
        gc.set_threshold(50, 1, 1)
        logits = gen.step([row], [4])
    finally:
        gc.set_threshold(*threshold)
        gen._one = stock
    assert calls == [True, False] and gc.isenabled()
    again = Generator(model, max_sequences=2)
    assert torch.equal(logits, again.step([again.prefill([1, 2, 3])[0]], [4]))


@pytest.mark.parametrize("preset,changes", [("tiny", {}), ("1.3b", dict(n_layers=1, vocab=500, d_model=128, n_heads=2, d_ff=256, max_seq=64))])
def test_tokens_outside_the_vocabulary(preset, changes):
    """On the host they are refused; on the device, where looking would mean waiting, they count as token 0, as they do where whole texts are scored."""
    torch.manual_seed(6)
    model = build_decoder(preset, **changes).cuda()
    gen = Generator(model, max_sequences=4, page_size=16)
    with pytest.raises(RuntimeError, match="vocabulary"):
        gen.prefill([1, model.cfg.vocab])
    rows = [gen.prefill([1, 2])[0] for _ in range(3)]
    with pytest.raises(RuntimeError, match="vocabulary"):
        gen.step(rows, [0, -1, 3])
    got = gen.step(rows, torch.tensor([0, -1, 2 ** 40], device="cuda"))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    first = gen.prefill(torch.tensor([1, model.cfg.vocab], device="cuda"))
    again = Generator(model, max_sequences=1, page_size=16)
    assert torch.equal(first[1], again.prefill([1, 0])[1])
