"""Writing tokens into a paged cache and copying its pages.  Unrotated values have to arrive bit by bit; a rotated one is a c - b s in fp32 with
three roundings of at most 2^-24 (|a| + |b|) each, rounded once to 16 bits (u of itself)."""
import pytest
import torch

from mccl_b200 import ops

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rope_tables(rows, dim):
    inv = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / dim))
    f = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float32), inv)
    return f.cos(), f.sin()


def make(tokens, sequences, heads, kv_heads, dim, page, dtype=torch.bfloat16, longest=300, seed=0):
    g = torch.Generator().manual_seed(seed)
    width = -(-longest // page)
    pages = sequences * width + 5
    table = torch.randperm(pages, generator=g)[:sequences * width].view(sequences, width).to(torch.int32).cuda()
    places = torch.randperm(sequences * longest, generator=g)[:tokens]
    rows, positions = (places // longest).to(torch.int32).cuda(), (places % longest).to(torch.int32).cuda()
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g).to(dtype).cuda()
    k_pages, v_pages = (torch.randn(pages, kv_heads, page, dim, generator=g).to(dtype).cuda() for _ in range(2))
    return *qkv.split([heads, kv_heads, kv_heads], dim=1), k_pages, v_pages, table, rows, positions


def rotated(x, positions, cos, sin):
    """(value, bound) in 64 bits."""
    c, s = cos[positions.long()].double()[:, None], sin[positions.long()].double()[:, None]
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    both = (a.abs() + b.abs()).repeat_interleave(2, dim=-1)
    return y, UNIT[x.dtype] * y.abs() + 3 * 2.0 ** -24 * both + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)   # fp16: steps of 2^-24 at the low end


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("tokens,sequences,heads,kv_heads,dim,page", [
    (1, 1, 8, 8, 64, 64), (7, 7, 4, 2, 128, 16), (64, 64, 16, 16, 128, 64), (301, 3, 8, 1, 32, 24), (1000, 5, 3, 3, 72, 16), (513, 2, 40, 8, 256, 1), (33, 4, 2, 2, 8, 7)])
def test_append(tokens, sequences, heads, kv_heads, dim, page, rope, dtype):
    q, k, v, k_pages, v_pages, table, rows, positions = make(tokens, sequences, heads, kv_heads, dim, page, dtype, longest=max(300, tokens))
    cos, sin = rope_tables(max(300, tokens), dim)
    before = k_pages.clone(), v_pages.clone()
    out = ops.paged_append(k, v, k_pages, v_pages, table, positions, rows=rows, q=q if rope else None, rope=(cos, sin) if rope else None)
    index, at = table[rows.long(), positions.long() // page].long(), positions.long() % page
    assert torch.equal(v_pages[index, :, at], v)
    if rope:
        for got, x in ((k_pages[index, :, at], k), (out, q)):
            want, bound = rotated(x, positions, cos, sin)
            assert got.dtype == dtype and ((got.double() - want).abs() <= bound).all()
        assert out.is_contiguous() and out.shape == q.shape
    else:
        assert out is None and torch.equal(k_pages[index, :, at], k)
    # nothing else moved
    for pages, old in zip((k_pages, v_pages), before):
        old[index, :, at] = pages[index, :, at]
        assert torch.equal(pages, old)


def test_rotation_has_the_bits_of_the_whole_text():
    """A key that goes into the cache is the key that attention over the whole text rotates."""
    from mccl_b200 import _C
    qkv = torch.randn(2, 50, 3, 4, 64, dtype=torch.bfloat16, device="cuda")
    cos, sin = rope_tables(64, 64)
    qk = _C.rope_qk_fwd(qkv, cos, sin)
    k_pages, v_pages = (torch.zeros(8, 4, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    rows = torch.arange(2, dtype=torch.int32, device="cuda").repeat_interleave(50)
    positions = torch.arange(50, dtype=torch.int32, device="cuda").repeat(2)
    flat = qkv.view(100, 3, 4, 64)
    q = ops.paged_append(flat[:, 1], flat[:, 2], k_pages, v_pages, table, positions, rows=rows, q=flat[:, 0], rope=(cos, sin))
    assert torch.equal(q.view(2, 50, 4, 64), qk[:, :, 0])
    index, at = table[rows.long(), positions.long() // 16].long(), positions.long() % 16
    assert torch.equal(k_pages[index, :, at].view(2, 50, 4, 64), qk[:, :, 1])


def test_tokens_that_have_no_place():
    q, k, v, k_pages, v_pages, table, rows, positions = make(40, 4, 4, 2, 64, 16)
    cos, sin = rope_tables(300, 64)
    before = k_pages.clone(), v_pages.clone()
    positions[0], positions[1], positions[2], positions[3] = -1, table.shape[1] * 16, 2 ** 31 - 1, -2 ** 31
    rows[4], rows[5], rows[6] = -1, 4, 2 ** 31 - 1
    table[rows[7], positions[7] // 16] = -1
    table[rows[8], positions[8] // 16] = k_pages.shape[0]
    index = torch.full((40,), -1, device="cuda")
    ok = (positions >= 0) & (positions < table.shape[1] * 16) & (rows >= 0) & (rows < 4)
    index[ok] = table[rows[ok].long(), positions[ok].long() // 16].long()
    ok &= (index >= 0) & (index < k_pages.shape[0]) & (positions < 300)
    assert 20 < ok.sum() < 40 and not ok[:9].any()
    out = ops.paged_append(k, v, k_pages, v_pages, table, positions, rows=rows, q=q, rope=(cos, sin))
    assert not out[~ok].any() and out[ok].abs().amax(-1).min() > 0
    at = positions.long() % 16
    assert torch.equal(v_pages[index[ok], :, at[ok]], v[ok])
    for pages, old in zip((k_pages, v_pages), before):
        old[index[ok], :, at[ok]] = pages[index[ok], :, at[ok]]
        assert torch.equal(pages, old)


def test_positions_beyond_the_rotation_tables():
    q, k, v, k_pages, v_pages, table, rows, positions = make(5, 1, 2, 2, 64, 16)
    positions.copy_(torch.tensor([0, 99, 100, 101, 250]))
    before = v_pages.clone()
    out = ops.paged_append(k, v, k_pages, v_pages, table, positions, rows=rows, q=q, rope=rope_tables(100, 64))
    assert out[:2].any() and not out[2:].any()
    assert (v_pages != before).flatten(1).any(1).sum() == 2


@pytest.mark.parametrize("layout", ["heads", "tokens", "layers"])
def test_strides_of_the_cache(layout):
    q, k, v, k_pages, v_pages, table, rows, positions = make(100, 3, 4, 2, 64, 16)
    want = k_pages.clone(), v_pages.clone()
    ops.paged_append(k, v, *want, table, positions, rows=rows)
    if layout == "tokens":
        got = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k_pages, v_pages)]
    elif layout == "heads":
        got = [k_pages.clone(), v_pages.clone()]
    else:
        cache = torch.stack((k_pages, v_pages), dim=1).unsqueeze(0).repeat(3, 1, 1, 1, 1, 1)
        got = [cache[1, :, 0], cache[1, :, 1]]
    ops.paged_append(k.contiguous(), v, *got, table, positions, rows=rows)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_decode_and_no_tokens():
    # without rows, token t is of row t
    q, k, v, k_pages, v_pages, table, rows, positions = make(4, 4, 4, 2, 64, 16)
    other = k_pages.clone(), v_pages.clone()
    ops.paged_append(k, v, k_pages, v_pages, table, positions)
    ops.paged_append(k, v, *other, table, positions, rows=torch.arange(4, dtype=torch.int32, device="cuda"))
    assert torch.equal(k_pages, other[0]) and torch.equal(v_pages, other[1])
    out = ops.paged_append(k[:0], v[:0], k_pages, v_pages, table, positions[:0], rows=rows[:0], q=q[:0], rope=rope_tables(300, 64))
    assert out.shape == (0, 4, 64) and torch.equal(k_pages, other[0])


def test_append_beyond_32_bits():
    pages = 5 * 2 ** 30 // (16 * 2 * 64)
    cache = torch.zeros(pages, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    k, v = torch.randn(2, 3, 2, 64, device="cuda").to(torch.bfloat16)
    table = torch.tensor([[pages - 1], [pages - 7], [2]], dtype=torch.int32, device="cuda")
    positions = torch.tensor([15, 3, 0], dtype=torch.int32, device="cuda")
    ops.paged_append(k, v, cache, cache.clone(), table, positions)
    assert torch.equal(cache[table[:, 0].long(), :, positions.long()], k)
    assert cache[pages - 8:].any(-1).sum() == 4 and cache[:3].any(-1).sum() == 2
    ops.copy_pages(cache, table[:1, 0].contiguous(), torch.tensor([pages - 3], dtype=torch.int32, device="cuda"))
    assert torch.equal(cache[pages - 3], cache[pages - 1]) and cache[pages - 8:].any(-1).sum() == 6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8, torch.int64])
@pytest.mark.parametrize("shape,dim", [((9, 2, 16, 64), 0), ((3, 2, 21, 4, 16, 32), 2), ((2, 50, 3), 1), ((2, 50, 1), 1), ((30,), 0), ((4, 7, 300, 8, 40), 1), ((5, 11, 3), -2)])
def test_copy_pages(shape, dim, dtype):
    pages = torch.randint(0, 100, shape, device="cuda").to(dtype)
    n = shape[dim]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(0))
    for count in {1, n // 2}:
        src, dst = order[:count].to(torch.int32).cuda(), order[count:2 * count].to(torch.int32).cuda()
        got, want = pages.clone(), pages.clone()
        want.index_copy_(dim, dst.long(), pages.index_select(dim, src.long()))
        assert ops.copy_pages(got, src, dst, dim=dim) is got or True
        assert torch.equal(got, want)


def test_copy_pages_shared_sources_and_bad_pairs():
    pages = torch.randn(2, 20, 4, 16, 64, device="cuda")
    src = torch.tensor([3, 3, -1, 20, 5, 3], dtype=torch.int32, device="cuda")
    dst = torch.tensor([0, 1, 2, 4, 20, 19], dtype=torch.int32, device="cuda")
    want = pages.clone()
    want[:, [0, 1, 19]] = pages[:, [3]]
    ops.copy_pages(pages, src, dst, dim=1)
    assert torch.equal(pages, want)
    assert torch.equal(ops.copy_pages(pages, src[:0], dst[:0], dim=1), want)
    # one layer's keys out of a cache of layers; the dimensions before the pages with one stride
    cache = torch.randn(3, 2, 20, 4, 64, device="cuda")
    want = cache.clone()
    want[1, :, 7], want[1, :, 2] = cache[1, :, 3], cache[1, :, 4]
    ops.copy_pages(cache[1], torch.tensor([3, 4], dtype=torch.int32, device="cuda"), torch.tensor([7, 2], dtype=torch.int32, device="cuda"), dim=1)
    assert torch.equal(cache, want)
    # more pairs than a grid has rows
    many = torch.arange(140000, dtype=torch.float32, device="cuda").view(70000, 2).repeat(2, 1)
    ops.copy_pages(many, torch.arange(70000, dtype=torch.int32, device="cuda"), torch.arange(70000, 140000, dtype=torch.int32, device="cuda").flip(0).contiguous())
    assert torch.equal(many[70000:], many[:70000].flip(0))


def test_refusals():
    q, k, v, k_pages, v_pages, table, rows, positions = make(4, 4, 4, 2, 64, 16)
    rope = rope_tables(300, 64)

    def refused(*args, **kw):
        with pytest.raises(RuntimeError, match="paged_append"):
            ops.paged_append(*args, **kw)

    refused(k.float(), v.float(), k_pages, v_pages, table, positions)
    refused(k, v.half(), k_pages, v_pages, table, positions)
    refused(k, v[:3], k_pages, v_pages, table, positions)
    refused(k[:, :1], v[:, :1], k_pages, v_pages, table, positions)
    refused(k, v, k_pages.half(), v_pages, table, positions)
    refused(k, v, k_pages, v_pages[1:], table, positions)
    refused(k, v, k_pages, v_pages, table, positions.long())
    refused(k, v, k_pages, v_pages, table, positions[:3])
    refused(k, v, k_pages, v_pages, table, positions, rows=rows[:3])
    refused(k, v, k_pages, v_pages, table, positions, rows=rows.cpu())
    refused(k, v, k_pages, v_pages, table, positions, q=q)
    refused(k, v, k_pages, v_pages, table, positions, q=q[:3], rope=rope)
    refused(k, v, k_pages, v_pages, table, positions, q=q[..., :32], rope=rope)
    refused(k, v, k_pages, v_pages, table, positions, rope=(rope[0][:, :16], rope[1][:, :16]))
    refused(k, v, k_pages, v_pages, table, positions, rope=(rope[0].double(), rope[1].double()))
    refused(k, v, k_pages, v_pages, table, positions, rope=(rope[0], rope[1][:10]))
    refused(k[..., ::2], v[..., ::2], k_pages, v_pages, table, positions)
    refused(k.clone().requires_grad_(), v, k_pages, v_pages, table, positions)
    one, two = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (1, 2))
    for args, kw in (((k_pages, one.long(), two), {}), ((k_pages, one, torch.cat((two, two))), {}), ((k_pages, one, two), {"dim": 4}),
                     ((k_pages.transpose(1, 2), one, two), {}), ((k_pages[:1].expand(4, -1, -1, -1), one, two), {}), ((k_pages, one.cpu(), two.cpu()), {}),
                     ((k_pages.view(2, 3, -1, 2, 16, 64)[:, :2] if k_pages.shape[0] % 6 == 0 else k_pages.unsqueeze(0).expand(3, -1, -1, -1, -1), one, two), {"dim": 1})):
        with pytest.raises(RuntimeError, match="copy_pages"):
            ops.copy_pages(*args, **kw)
