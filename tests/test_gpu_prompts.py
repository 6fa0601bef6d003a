"""Several prompts in one pass on the native operators, and a training step over packed texts; see test_generate.py for the bound on logits."""
import math

import pytest
import torch

from mccl_b200 import ops
from mccl_b200.models import Generator, build_decoder
from tests.generate_checks import dequantized, reference_logits, rms, sharpen

pytestmark = pytest.mark.gpu
MODELS = {"tiny": ("tiny", {}), "70m": ("70m", dict(n_layers=3)), "110m": ("110m", dict(n_layers=2, vocab=1000)),
          "swiglu": ("1.3b", dict(n_layers=2, vocab=1024, max_seq=512)), "swiglu-narrow": ("1.3b", dict(n_layers=2, vocab=512, d_model=192, n_heads=3, d_ff=320, max_seq=300))}


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("weights", ["bf16", "w4"])
def test_prompts_together(name, weights):
    torch.manual_seed(0)
    preset, changes = MODELS[name]
    model = sharpen(build_decoder(preset, **changes).cuda())
    lengths = [min(n, model.cfg.max_seq - 1) for n in (1, 200, 37, 129, 5, 64)]
    texts = [torch.randint(0, model.cfg.vocab, (n + 1,), device="cuda") for n in lengths]
    gen = Generator(model, max_sequences=6, page_size=16, weights=weights, group=64)
    rows, first = gen.prefill_together([t[:-1] for t in texts])
    then = gen.step(rows, torch.stack([t[-1] for t in texts]))
    matrices = dequantized(model, 64) if weights == "w4" else None
    with torch.no_grad():
        want = [torch.stack([reference_logits(model, t, matrices)[-1] for t in x]) for x in ([t[:-1] for t in texts], texts)]
        whole = rms(torch.stack([model(t[None])[0, -1] for t in texts]).float() - torch.stack([reference_logits(model, t)[-1] for t in texts]))
    assert rms(first.float() - want[0]) <= 3 * whole and rms(then.float() - want[1]) <= 3 * whole
    assert rms(want[0]) > 10 * whole


def test_a_window_in_one_pass():
    torch.manual_seed(2)
    model = sharpen(build_decoder("1.3b", n_layers=2, vocab=512, d_model=256, n_heads=4, d_ff=512, max_seq=400).cuda())
    tokens = torch.randint(0, 512, (400,), device="cuda")
    gen = Generator(model, max_sequences=1, page_size=16, window=100, sinks=5)
    rows, logits = gen.prefill_together([tokens[:390]])
    got = torch.stack([logits[0]] + [gen.step(rows, tokens[i:i + 1])[0] for i in range(390, 400)]).float()
    with torch.no_grad():
        want = reference_logits(model, tokens, window=100, sinks=5)[389:]
        whole = rms(model(tokens[None])[0, 389:].float() - reference_logits(model, tokens)[389:])
    assert rms(got - want) <= 3 * whole


def test_generate_together_and_by_given_numbers():
    torch.manual_seed(3)
    model = sharpen(build_decoder("70m", n_layers=2).cuda())
    gen = Generator(model, max_sequences=4, page_size=16)
    prompts = [torch.randint(0, 32000, (n,)).tolist() for n in (3, 120, 17)]
    draw = lambda **o: gen.generate(prompts, 8, temperature=1.0, generator=torch.Generator().manual_seed(7), **o)
    a = draw(top_k=50, top_p=0.95, min_p=1e-3, together=True)
    assert a == draw(top_k=50, top_p=0.95, min_p=1e-3, together=True) and all(len(t) == 8 for t in a)
    assert all(len(t) == 8 for t in gen.generate(prompts, 8, temperature=0.7, top_p=0.9, generator=torch.Generator("cuda").manual_seed(1)))
    rows, logits = gen.prefill_together(prompts)
    u = torch.rand(3, generator=torch.Generator().manual_seed(7)).cuda()
    assert [t[0] for t in a] == ops.sample(logits.float(), u, temperature=1.0, top_k=50, top_p=0.95, min_p=1e-3).tolist()
    for r in rows:
        gen.free(r)
    with torch.no_grad():
        model.ln_f.weight.fill_(math.nan)
    broken = Generator(model, max_sequences=1)
    with pytest.raises(RuntimeError, match="not finite"):
        broken.generate([[1]], 2, temperature=1.0, top_p=0.9)


def test_on_a_stream_of_its_own():
    model = sharpen(build_decoder("tiny").cuda())
    gen = Generator(model, max_sequences=3, page_size=16)
    prompts = [[1, 2, 3], [4] * 40, [5, 6]]
    want = gen.prefill_together(prompts)[1].clone()
    for r in gen.cache.rows:
        gen.free(r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gen.prefill_together(prompts)[1]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def block(x, w, w_out, rope, positions, offsets, heads, kv_heads, dim, **options):
    """An attention block over packed texts: projection, rotation, attention, projection back."""
    qkv = (x @ w.T).view(-1, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    q, k = ops.rotary(q, k, rope=rope, positions=positions, layout="half")
    return x + ops.packed_attention(q, k, v, offsets, **options).flatten(1) @ w_out.T


@pytest.mark.parametrize("options", [{}, {"window": 50, "sinks": 3}])
def test_a_training_step_over_packed_texts(options):
    """Gradients of a block's input and weights: packed, and text by text with the plain forms in 32 bits.  In bf16 every product and sum of the block is rounded: their errors
    are compared with those of the plain forms carried out on the same bf16 tensors, of which no more than twice is allowed."""
    torch.manual_seed(4)
    heads, kv_heads, dim, width = 4, 2, 64, 256
    lengths = [130, 1, 77, 300]
    n = sum(lengths)
    positions = torch.cat([torch.arange(m, dtype=torch.int32) for m in lengths])
    offsets = torch.cumsum(torch.tensor([0] + lengths), 0).to(torch.int32)
    rope = ops.rotary_tables(400, 32, device="cpu")
    x = torch.randn(n, width).to(torch.bfloat16)
    w = (torch.randn((heads + 2 * kv_heads) * dim, width) * width ** -0.5).to(torch.bfloat16)
    w_out = (torch.randn(width, heads * dim) * width ** -0.5).to(torch.bfloat16)
    g = torch.randn(n, width).to(torch.bfloat16)

    def grads(device, dtype):
        leaves = [t.to(device, dtype).requires_grad_() for t in (x, w, w_out)]
        y = block(*leaves, tuple(t.to(device) for t in rope), positions.to(device), offsets.to(device), heads, kv_heads, dim, **options)
        return [t.float().cpu() for t in (y.detach(), *torch.autograd.grad(y, leaves, g.to(device, dtype)))]

    exact, plain, got = grads("cpu", torch.float32), grads("cpu", torch.bfloat16), grads("cuda", torch.bfloat16)
    for a, b, c in zip(exact, plain, got):
        assert rms(c - a) <= 2 * rms(b - a) and rms(a) > 20 * rms(b - a)
