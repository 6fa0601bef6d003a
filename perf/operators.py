"""The operators that let a decoder answer token by token, as cases that can be timed and compared.

  attention  ``ops.paged_attention``: one new token per sequence over a paged key-value cache
  append     ``ops.paged_append``: keys and values of new tokens into the cache's pages, with rotary positions where the model has them
  copy       ``ops.copy_pages``: pages of all layers copied to other pages (forked sequences, a cache that is compacted)
  w4         ``ops.linear_w4``: a linear layer with 4-bit weights and group scales

With ``own`` false every operator is computed from elementary torch operations in 32 bits, rounded once at the end; with ``own`` true by
the package's own kernels.  Head counts and widths are those of the package's presets (70m: 8 x 64, 110m: 12 x 64, 1.3b: 16 x 128), and
heads that share keys and values, which the operators take as well.
"""
import math

import torch

#: whether `run` calls the package's operators; otherwise their plain forms
own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------------ cases ----
def _attention(name, batch, heads, kv_heads, dim, page, longest, spread, window=0, sinks=0, dtype="bf16"):
    return {"name": name, "op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "longest": longest, "spread": spread, "window": window, "sinks": sinks, "dtype": dtype}


def _append(name, tokens, sequences, heads, kv_heads, dim, page, rope, dtype="bf16"):
    return {"name": name, "op": "append", "tokens": tokens, "sequences": sequences, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "rope": rope, "dtype": dtype}


def _copy(name, layers, pages, copies, heads, dim, page, dtype="bf16"):
    return {"name": name, "op": "copy", "layers": layers, "pages": pages, "copies": copies, "heads": heads, "dim": dim, "page": page, "dtype": dtype}


def _w4(name, rows, n, k, group, act="none", bias=False, residual=False):
    return {"name": name, "op": "w4", "rows": rows, "n": n, "k": k, "group": group, "act": act, "bias": bias, "residual": residual}


def listed():
    return [
        # one short answer of the 70m model: nothing but latency
        _attention("attention-one-short", 1, 8, 8, 64, 64, 37, 0.0),
        # a serving batch of the 1.3b model, every sequence at another point of its 2048 positions
        _attention("attention-ragged", 64, 16, 16, 128, 64, 2048, 1.0),
        # two very long documents, four query heads to each head of keys and values: few rows, the length has to be split
        _attention("attention-long", 2, 32, 8, 128, 64, 131009, 0.01),
        # a stream that keeps its first tokens and the last thousand, small pages, fp16
        _attention("attention-window", 48, 16, 4, 128, 16, 16384, 0.9, window=1024, sinks=4, dtype="fp16"),
        # a decode step of the 1.3b model: one token for each of 64 sequences
        _append("append-step", 64, 64, 16, 16, 128, 64, True),
        # a prompt of the 1.3b model goes into the cache
        _append("append-prompt", 1537, 1, 16, 16, 128, 64, True),
        # eight sequences of the 70m model fork: each takes a copy of its last page in 16 layers
        _copy("copy-fork", 16, 64, 8, 8, 64, 64),
        # a cache of 12 layers of the 1.3b widths is compacted: half its pages move
        _copy("copy-compact", 12, 132, 61, 16, 128, 64),
        # one token through an attention output projection of the 1.3b model
        _w4("w4-one", 1, 2048, 2048, 128, residual=True),
        # four sequences through a vocabulary projection
        _w4("w4-head", 4, 32000, 2048, 64),
        # a batch of sequences through the 110m model's up projection
        _w4("w4-batch", 48, 3072, 768, 128, act="gelu", bias=True),
        # a prompt through the 1.3b model's gate and up projections
        _w4("w4-prompt", 1537, 16384, 2048, 128),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "copy", "w4", "w4", "w4"])
    if op == "attention":
        dim = rng.choice([32, 64, 64, 72, 96, 128, 128, 128, 256])
        kv_heads, group = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 8])
        batch = _log_uniform(rng, 1, 96)
        most = min(131072, int(2.5e8 / (batch * kv_heads * dim)))
        longest = _log_uniform(rng, 1, max(1, most))
        window = rng.choice([0, 0, 0, _log_uniform(rng, 1, 4096)])
        return _attention(None, batch, kv_heads * group, kv_heads, dim, rng.choice([16, 32, 64, 128, 24]), longest, rng.choice([0.0, 0.5, 1.0]),
                          window, rng.choice([0, 1, 4, 37]) if window else 0, rng.choice(["bf16", "bf16", "fp16"]))
    if op == "append":
        sequences = _log_uniform(rng, 1, 128)
        tokens = sequences if rng.random() < 0.5 else max(sequences, _log_uniform(rng, 1, 4096))
        kv_heads, group = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4])
        return _append(None, tokens, sequences, kv_heads * group, kv_heads, rng.choice([32, 64, 96, 128]), rng.choice([16, 32, 64, 24]),
                       rng.random() < 0.6, rng.choice(["bf16", "bf16", "fp16"]))
    if op == "copy":
        heads, dim, page = rng.choice([1, 4, 8, 12, 16]), rng.choice([32, 64, 128]), rng.choice([16, 32, 64, 24])
        layers = rng.choice([1, 2, 12, 16, 24])
        pages = max(2, min(256, int(4e8 / (layers * heads * dim * page))))
        pages = _log_uniform(rng, 2, pages)
        return _copy(None, layers, pages, _log_uniform(rng, 1, pages // 2), heads, dim, page, rng.choice(["bf16", "fp16"]))
    group = rng.choice([32, 64, 128, 128])
    k = group * _log_uniform(rng, 1, 8192 // group)
    n = 8 * _log_uniform(rng, 1, 4096)
    rows = rng.choice([1, 1, 2, _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 2048)])
    rows = max(1, min(rows, int(5e10 / (n * k))))
    act = rng.choice(["none", "none", "gelu"])
    return _w4(None, rows, n, k, group, act, rng.random() < 0.4, act == "none" and rng.random() < 0.4)


# ----------------------------------------------------------------------------------------------------------- inputs ----
def _lengths(case, gen):
    """Lengths of the sequences: the longest one is as long as the case says, the others up to `spread` of it shorter."""
    cut = torch.rand(case["batch"], generator=gen) * case["spread"]
    cut[0] = 0.0
    return [max(1, int(case["longest"] * (1.0 - c))) for c in cut.tolist()]


def _table(needed, width, total, gen):
    """Page tables over one shared pool of `total` pages in a random order (-1 behind a sequence's last page)."""
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(needed), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(needed):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def _rotations(positions, dim, device):
    inv = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, device=device, dtype=torch.float32) / dim))
    angle = torch.outer(torch.arange(positions, device=device, dtype=torch.float32), inv)
    return angle.cos(), angle.sin()


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=dev, device="cuda", dtype=dtype)

    if case["op"] == "attention":
        dtype, dim, page = _DTYPES[case["dtype"]], case["dim"], case["page"]
        lengths = _lengths(case, gen)
        needed = [-(-n // page) for n in lengths]
        total = sum(needed)
        table = _table(needed, max(needed), total, gen)
        # queries as a model has them: part of the fused projection's output
        qkv = normal(case["batch"], case["heads"] + 2 * case["kv_heads"], dim, dtype=dtype)
        return {"op": "attention", "q": qkv[:, :case["heads"]], "k_pages": normal(total, case["kv_heads"], page, dim, dtype=dtype),
                "v_pages": normal(total, case["kv_heads"], page, dim, dtype=dtype), "table": table.cuda(),
                "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "scale": dim ** -0.5,
                "window": case["window"] or None, "sinks": case["sinks"]}
    if case["op"] == "append":
        dtype, dim, page, count, tokens = _DTYPES[case["dtype"]], case["dim"], case["page"], case["sequences"], case["tokens"]
        new = [tokens // count + (i < tokens % count) for i in range(count)]
        before = torch.randint(0, 512, (count,), generator=gen).tolist()   # what each sequence has in the cache already
        width, total = -(-(512 + max(new)) // page), sum(-(-(512 + n) // page) for n in new)
        table = _table([-(-(b + n) // page) for b, n in zip(before, new)], width, total, gen)
        rows = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(new)])
        positions = torch.cat([torch.arange(b, b + n, dtype=torch.int32) for b, n in zip(before, new)])
        qkv = normal(tokens, case["heads"] + 2 * case["kv_heads"], dim, dtype=dtype)
        q, k, v = qkv.split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        return {"op": "append", "q": q, "k": k, "v": v, "k_pages": normal(total, case["kv_heads"], page, dim, dtype=dtype),
                "v_pages": normal(total, case["kv_heads"], page, dim, dtype=dtype), "table": table.cuda(), "rows": rows.cuda(),
                "positions": positions.cuda(), "rope": _rotations(512 + max(new), dim, "cuda") if case["rope"] else None}
    if case["op"] == "copy":
        pages = normal(case["layers"], 2, case["pages"], case["heads"], case["page"], case["dim"], dtype=_DTYPES[case["dtype"]])
        order = torch.randperm(case["pages"], generator=gen).to(torch.int32)
        n = case["copies"]
        return {"op": "copy", "pages": pages, "src": order[:n].cuda(), "dst": order[n:2 * n].cuda()}
    n, k, group, rows = case["n"], case["k"], case["group"], case["rows"]
    codes = torch.randint(0, 16, (n, k), generator=dev, device="cuda", dtype=torch.uint8)
    zeros = torch.randint(6, 10, (n, k // group), generator=dev, device="cuda", dtype=torch.uint8)
    scales = (0.02 / 4.6 * (0.5 + torch.rand(n, k // group, generator=dev, device="cuda"))).to(torch.bfloat16)
    state = {"op": "w4", "x": normal(rows, k, dtype=torch.bfloat16), "act": case["act"], "group": group,
             "bias": normal(n, dtype=torch.float32) * 0.1 if case["bias"] else None,
             "residual": normal(rows, n, dtype=torch.bfloat16) if case["residual"] else None}
    if own:
        from mccl_b200 import ops
        state["weight"] = ops.W4Weight.from_codes(codes, scales, zeros)
    else:
        state.update(codes=codes, zeros=zeros, scales=scales)
    return state


# ------------------------------------------------------------------------------------------------------------- runs ----
def _plain_attention(s):
    q, k_pages, v_pages, table = s["q"], s["k_pages"], s["v_pages"], s["table"]
    batch, heads, dim = q.shape
    kv_heads, page = k_pages.shape[1], k_pages.shape[2]
    span = table.shape[1] * page
    block = max(1, int(2 ** 29 // (span * kv_heads * dim)))   # sequences whose keys and values are gathered at a time
    at = torch.arange(span, device=q.device)
    out = []
    for b in range(0, batch, block):
        n = min(block, batch - b)
        index = table[b:b + n].long().clamp(min=0)
        length = s["lengths"][b:b + n, None].long()
        seen = at < length
        if s["window"] is not None:
            seen = seen & ((at >= length - s["window"]) | (at < s["sinks"]))
        seen = seen[:, None, None, :]
        k = k_pages[index].permute(0, 2, 1, 3, 4).reshape(n, kv_heads, span, dim).float()
        score = torch.matmul(q[b:b + n].float().reshape(n, kv_heads, heads // kv_heads, dim), k.transpose(2, 3)) * s["scale"]
        del k
        score = torch.where(seen, score, float("-inf"))
        p = torch.where(seen, torch.exp(score - score.amax(-1, keepdim=True)), 0.0)
        v = v_pages[index].permute(0, 2, 1, 3, 4).reshape(n, kv_heads, span, dim).float()
        v = torch.where(seen.transpose(2, 3), v, 0.0)
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out.append(torch.where(seen.any(-1, keepdim=True), o, 0.0).reshape(n, heads, dim).to(q.dtype))
    return torch.cat(out)


def _plain_append(s):
    def rotate(x):
        if s["rope"] is None:
            return x
        cos, sin = (t[s["positions"].long()][:, None] for t in s["rope"])
        a, b = x[..., 0::2].float(), x[..., 1::2].float()
        return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2).to(x.dtype)

    page = s["k_pages"].shape[2]
    positions = s["positions"].long()
    index = s["table"][s["rows"].long(), positions // page].long()
    s["k_pages"][index, :, positions % page] = rotate(s["k"])
    s["v_pages"][index, :, positions % page] = s["v"]
    pages = [s["k_pages"], s["v_pages"]]
    return pages if s["rope"] is None else [rotate(s["q"])] + pages


def _plain_w4(s):
    n, k = s["codes"].shape
    w = s["codes"].view(n, -1, s["group"]).float() - s["zeros"].float()[..., None]
    w = (w * s["scales"].float()[..., None]).view(n, k)
    y = torch.matmul(s["x"].float(), w.t())
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * 2 ** -0.5))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def run(state):
    s, op = state, state["op"]
    if own:
        from mccl_b200 import ops
        if op == "attention":
            return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], scale=s["scale"], window=s["window"],
                                       sinks=s["sinks"])
        if op == "append":
            q = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["positions"], rows=s["rows"],
                                 q=s["q"] if s["rope"] is not None else None, rope=s["rope"])
            pages = [s["k_pages"], s["v_pages"]]
            return pages if s["rope"] is None else [q] + pages
        if op == "copy":
            return ops.copy_pages(s["pages"], s["src"], s["dst"], dim=2)
        return ops.linear_w4(s["x"], s["weight"], s["bias"], act=s["act"], residual=s["residual"])
    if op == "attention":
        return _plain_attention(s)
    if op == "append":
        return _plain_append(s)
    if op == "copy":
        s["pages"][:, :, s["dst"].long()] = s["pages"][:, :, s["src"].long()]
        return s["pages"]
    return _plain_w4(s)


# ------------------------------------------------------------------------------------------------------------- work ----
def work(case):
    if case["op"] == "attention":
        # the lengths of a case depend on the seed: half of the spread is what they lose on average
        mean = case["longest"] if case["batch"] == 1 else case["longest"] * (1.0 - case["spread"] / 2 * (case["batch"] - 1) / case["batch"])
        if case["window"]:
            mean = min(mean, case["window"] + case["sinks"])
        seen = case["batch"] * max(1.0, mean)
        return {"bytes": seen * case["kv_heads"] * case["dim"] * 4 + 2 * case["batch"] * case["heads"] * case["dim"] * 2,
                "flops": 4.0 * seen * case["heads"] * case["dim"]}
    if case["op"] == "append":
        rotated = case["heads"] + case["kv_heads"] if case["rope"] else 0
        moved = (case["heads"] if case["rope"] else 0) + 2 * case["kv_heads"]
        return {"bytes": 2.0 * case["tokens"] * moved * case["dim"] * 2, "flops": 3.0 * case["tokens"] * rotated * case["dim"]}
    if case["op"] == "copy":
        return {"bytes": 2.0 * case["layers"] * 2 * case["copies"] * case["heads"] * case["page"] * case["dim"] * 2, "flops": 0.0}
    m, n, k = case["rows"], case["n"], case["k"]
    return {"bytes": n * k / 2 + 2.5 * n * (k // case["group"]) + 2.0 * m * k + 2.0 * m * n * (2 if case["residual"] else 1) + 4.0 * n * case["bias"],
            "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------------------------------------------------ exact ----
def exact(case, seed):
    global own
    was, own = own, False   # the inputs as numbers, not laid out
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "attention":
        page, group = case["page"], case["heads"] // case["kv_heads"]
        out = torch.zeros(case["batch"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        for b, length in enumerate(s["lengths"].tolist()):
            seen = list(range(length))
            if case["window"]:
                seen = [j for j in seen if j < case["sinks"] or length - j <= case["window"]]
            j = torch.tensor(seen, device="cuda")
            at = s["table"][b].long()[torch.div(j, page, rounding_mode="floor")]
            for h in range(case["kv_heads"]):
                k, v = (s[name][at, h, j % page].double() for name in ("k_pages", "v_pages"))
                weight = torch.softmax(s["q"][b, h * group:(h + 1) * group].double() @ k.T * case["dim"] ** -0.5, dim=-1)
                out[b, h * group:(h + 1) * group] = weight @ v
        return out
    if case["op"] == "append":
        page, half = case["page"], case["dim"] // 2
        turned = {}
        for name in ("q", "k"):
            x = s[name].double()
            if case["rope"]:
                p = s["positions"].long()
                z = torch.view_as_complex(x.reshape(x.shape[0], x.shape[1], half, 2)) * torch.complex(s["rope"][0].double(), s["rope"][1].double())[p].unsqueeze(1)
                x = torch.view_as_real(z).reshape(x.shape)
            turned[name] = x
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        slot = s["table"].long()[s["rows"].long(), s["positions"].long() // page] * page + s["positions"].long() % page
        k_pages.transpose(1, 2)[slot // page, slot % page] = turned["k"]
        v_pages.transpose(1, 2)[slot // page, slot % page] = s["v"].double()
        return [turned["q"], k_pages, v_pages] if case["rope"] else [k_pages, v_pages]
    if case["op"] == "copy":
        return None
    w = s["codes"].double() - s["zeros"].double().repeat_interleave(case["group"], dim=1)
    w = w * s["scales"].double().repeat_interleave(case["group"], dim=1)
    y = s["x"].double() @ w.T
    if case["bias"]:
        y = y + s["bias"].double()
    if case["act"] == "gelu":
        y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2.0))
    if case["residual"]:
        y = y + s["residual"].double()
    return y
