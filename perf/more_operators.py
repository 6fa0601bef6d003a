"""The operators around whole prompts and packed texts, as cases that can be timed and compared.

  prompt   ``ops.packed_attention``: causal attention of texts of different lengths, one behind the other without padding; query heads may
           share keys and values, a text may have keys before its first query, positions may see a window and the first few only
  train    the same with its gradients of queries, keys and values
  rotary   ``ops.rotary``: queries and keys turned by their positions, neighbouring or half-a-head pairs, the whole head or a part of it;
           with gradients where a model trains
  sample   ``ops.sample``: a token per row of logits from a given random number, under temperature, top-k, top-p and min-p

With ``own`` false every operator is computed from elementary torch operations in 32 bits (64 where tokens are chosen), rounded once at the end;
with ``own`` true by the package's own kernels.  Head counts and widths are those of the package's presets (70m: 8 x 64, 110m: 12 x 64,
1.3b: 16 x 128), and heads that share keys and values.
"""
import math

import torch

#: whether `run` calls the package's operators; otherwise their plain forms
own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------ cases ----
def _attention(name, op, texts, longest, spread, heads, kv_heads, dim, window=0, sinks=0, before=0, spare=0, dtype="bf16"):
    """`texts` of `longest` new tokens down to `spread` of it shorter, each behind up to `before` earlier keys; `spare` rows belong to no text."""
    return {"name": name, "op": op, "texts": texts, "longest": longest, "spread": spread, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": sinks, "before": before, "spare": spare, "dtype": dtype}


def _rotary(name, tokens, heads, kv_heads, dim, rotated, layout, factor=1.0, grad=False, dtype="bf16"):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": rotated, "layout": layout,
            "factor": factor, "grad": grad, "dtype": dtype}


def _sample(name, rows, vocab, temperature, top_k=0, top_p=1.0, min_p=0.0, each=False, dtype="bf16"):
    """`each`: every row has a temperature, top-k, top-p and min-p of its own, around the ones given."""
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "each": each, "dtype": dtype}


def listed():
    return [
        # one short prompt of the 70m model: nothing but latency
        _attention("prompt-short", "prompt", 1, 37, 0.0, 8, 8, 64),
        # sixteen prompts of the 1.3b model, up to its 2048 positions, in one pass
        _attention("prompt-ragged", "prompt", 16, 2048, 1.0, 16, 16, 128),
        # one long document, four query heads to each head of keys and values
        _attention("prompt-long", "prompt", 1, 16381, 0.0, 32, 8, 128),
        # four long streams that keep their first tokens and the last thousand, fp16
        _attention("prompt-window", "prompt", 4, 8192, 0.5, 16, 4, 128, window=1024, sinks=4, dtype="fp16"),
        # a part of eight prompts behind what is in the cache already, widths of the 110m model
        _attention("prompt-behind", "prompt", 8, 130, 0.5, 12, 4, 64, before=4096),
        # a step of the 70m model on texts of up to 256 tokens
        _attention("train-short", "train", 32, 256, 0.8, 8, 8, 64),
        # a step of the 1.3b model on packed texts of up to 2048 tokens
        _attention("train-ragged", "train", 8, 2048, 0.9, 16, 16, 128, spare=77),
        # long texts, shared keys and values
        _attention("train-long", "train", 1, 8192, 0.0, 16, 4, 128),
        # a decode step of the 1.3b model: one token for each of 64 sequences
        _rotary("rotary-step", 64, 16, 16, 128, 128, "interleaved"),
        # packed training texts, half of each head turned in halves, positions scaled to reach further
        _rotary("rotary-train", 16384, 32, 8, 128, 64, "half", factor=4.0, grad=True),
        # one answer of the package's vocabulary
        _sample("sample-one", 1, 32000, 0.8, top_k=50, top_p=0.9),
        # a serving batch over a large vocabulary, every request with settings of its own
        _sample("sample-batch", 64, 128000, 1.0, top_p=0.95, min_p=0.01, each=True, dtype="fp32"),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "train", "train", "rotary", "sample", "sample"])
    if op in ("prompt", "train"):
        dim = rng.choice([32, 64, 64, 72, 96, 128, 128, 128])
        kv_heads, group = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 1, 2, 3, 4, 8])
        texts = _log_uniform(rng, 1, 64)
        # no more scores than the largest listed case of the kind has
        most = 6e9 if op == "prompt" else 1e9
        longest = _log_uniform(rng, 1, max(1, min(16384, int(math.sqrt(most / (texts * kv_heads * group))), int(1.2e5 / texts))))
        before = 0
        if op == "prompt" and rng.random() < 0.3:
            longest = min(longest, 512)
            before = _log_uniform(rng, 1, 8192)
        window = rng.choice([0, 0, 0, _log_uniform(rng, 1, 4096)])
        return _attention(None, op, texts, longest, rng.choice([0.0, 0.5, 1.0]), kv_heads * group, kv_heads, dim, window,
                          rng.choice([0, 1, 4, 37]) if window else 0, before, rng.choice([0, 0, 5]), "bf16" if op == "train" else rng.choice(["bf16", "bf16", "fp16"]))
    if op == "rotary":
        dim = rng.choice([32, 64, 72, 96, 128, 128, 256])
        rotated = rng.choice([dim, dim, dim // 2 // 8 * 8 or 8, 16])
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        return _rotary(None, _log_uniform(rng, 1, 16384), kv_heads * rng.choice([1, 1, 2, 4]), kv_heads, dim, rotated, rng.choice(["interleaved", "half"]),
                       rng.choice([1.0, 2.0, 8.0]), rng.random() < 0.4, rng.choice(["bf16", "bf16", "fp16"]))
    rows = _log_uniform(rng, 1, 256)
    return _sample(None, rows, _log_uniform(rng, 100, min(200000, int(1.6e7 / rows))), rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 2.0]), rng.choice([0, 0, 1, 20, 64, 1000]),
                   rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]), rng.choice([0.0, 0.0, 0.05]), rng.random() < 0.5, rng.choice(["bf16", "fp16", "fp32"]))


# ----------------------------------------------------------------------------------------------------------- inputs ----
def _spread(case, longest):
    """Lengths from the longest down to `spread` of it shorter, in even steps: a text that is left without tokens is one too."""
    return [int(longest * (1.0 - case["spread"] * i / max(1, case["texts"] - 1))) for i in range(case["texts"])]


def _lengths(case, longest, gen):
    """The same lengths in an order of the seed's."""
    lengths = _spread(case, longest)
    return [lengths[i] for i in torch.randperm(len(lengths), generator=gen).tolist()]


def _offsets(lengths):
    return torch.cumsum(torch.tensor([0] + lengths), 0).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=dev, device="cuda", dtype=dtype)

    if case["op"] in ("prompt", "train"):
        lengths = _lengths(case, case["longest"], gen)
        rows, heads, kv_heads, dim = sum(lengths) + case["spare"], case["heads"], case["kv_heads"], case["dim"]
        state = {"op": case["op"], "lengths": lengths, "key_lengths": lengths, "offsets": _offsets(lengths).cuda(), "k_offsets": None,
                 "scale": dim ** -0.5, "window": case["window"] or None, "sinks": case["sinks"]}
        if case["before"]:
            # the earlier keys lie in front of the new ones, as they come out of a cache
            state["key_lengths"] = [n + m for n, m in zip(lengths, _lengths(case, case["before"], gen))]
            state["k_offsets"] = _offsets(state["key_lengths"]).cuda()
            kv = normal(sum(state["key_lengths"]) + case["spare"], 2, kv_heads, dim)
            q, k, v = normal(rows, heads, dim), kv[:, 0], kv[:, 1]
        else:
            # queries, keys and values as a model has them: parts of the fused projection's output
            q, k, v = normal(rows, heads + 2 * kv_heads, dim).split([heads, kv_heads, kv_heads], dim=1)
        if case["op"] == "train":
            q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
            state["grad"] = normal(rows, heads, dim)
        state.update(q=q, k=k, v=v)
        return state
    if case["op"] == "rotary":
        tokens, heads, kv_heads, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        q, k, _ = normal(tokens, heads + 2 * kv_heads, dim).split([heads, kv_heads, kv_heads], dim=1)
        longest = min(tokens, 4096) if case["grad"] else 4096
        angle = torch.arange(longest, dtype=torch.float64) / case["factor"]
        angle = torch.outer(angle, 10000.0 ** (-torch.arange(0, case["rotated"], 2, dtype=torch.float64) / case["rotated"]))
        # packed texts count up from zero each; steps are anywhere
        positions = torch.arange(tokens) % longest if case["grad"] else torch.randint(0, longest, (tokens,), generator=gen)
        state = {"op": "rotary", "rope": (angle.cos().float().cuda(), angle.sin().float().cuda()), "positions": positions.to(torch.int32).cuda(), "layout": case["layout"],
                 "grads": None}
        if case["grad"]:
            q, k = (t.detach().requires_grad_() for t in (q, k))
            state["grads"] = normal(tokens, heads, dim), normal(tokens, kv_heads, dim)
        state.update(q=q, k=k)
        return state
    # logits as a model has them: most tokens far below a few likely ones
    rows, vocab = case["rows"], case["vocab"]
    logits = 2.0 * torch.randn(rows, vocab, generator=dev, device="cuda")
    logits += 8.0 * torch.rand(rows, vocab, generator=dev, device="cuda") ** 64
    settings = {"temperature": case["temperature"], "top_k": case["top_k"], "top_p": case["top_p"], "min_p": case["min_p"]}
    if case["each"]:
        some = torch.rand(3, rows, generator=gen)
        settings["temperature"] = (case["temperature"] * (0.5 + some[0])).cuda()
        settings["top_k"] = torch.where(some[1] < 0.5, case["top_k"], case["top_k"] // 2 + 3).to(torch.int32).cuda()
        settings["top_p"] = torch.where(some[2] < 0.3, 1.0, case["top_p"] * (1.0 - 0.2 * some[1])).cuda()
        settings["min_p"] = (case["min_p"] * 2.0 * some[2]).cuda()
    return {"op": "sample", "logits": logits.to(dtype), "uniform": torch.rand(rows, generator=dev, device="cuda"), **settings}


# ------------------------------------------------------------------------------------------------------------- runs ----
def _texts(s):
    """(first query, first key, queries, keys) of every text."""
    at, key = 0, 0
    for n, m in zip(s["lengths"], s["key_lengths"]):
        yield at, key, n, m
        at, key = at + n, key + m


def _seen(n, m, window, sinks, device):
    """Which of m keys the last n positions see."""
    i, j = torch.arange(m - n, m, device=device)[:, None], torch.arange(m, device=device)[None]
    seen = j <= i
    return seen if window is None else seen & ((j > i - window) | (j < sinks))


def _plain_attention(s):
    q, k, v, grad = s["q"].detach(), s["k"].detach(), s["v"].detach(), s.get("grad")
    group = q.shape[1] // k.shape[1]
    o = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    dq, dk, dv = (torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)) if grad is not None else (None,) * 3
    for at, key, n, m in _texts(s):
        if n == 0:
            continue
        seen = _seen(n, m, s["window"], s["sinks"], q.device)
        block = max(1, int(2 ** 29 // (n * m * group)))   # heads of keys and values whose scores are held at a time
        for h in range(0, k.shape[1], block):
            kv = slice(h, min(h + block, k.shape[1]))
            qh = slice(kv.start * group, kv.stop * group)

            def rows(t, first, count, part):   # [kv heads, group, count, dim]
                return t[first:first + count, part].float().transpose(0, 1).unflatten(0, (kv.stop - kv.start, -1))

            qq, kk, vv = rows(q, at, n, qh), rows(k, key, m, kv), rows(v, key, m, kv)
            p = torch.matmul(qq, kk.transpose(2, 3)) * s["scale"]
            p = torch.where(seen, p, float("-inf"))
            p = torch.exp(p - p.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o[at:at + n, qh] = torch.matmul(p, vv).flatten(0, 1).transpose(0, 1).to(q.dtype)
            if grad is not None:
                gg = rows(grad, at, n, qh)
                dv[key:key + m, kv] = torch.matmul(p.transpose(2, 3), gg).sum(1).transpose(0, 1).to(v.dtype)
                ds = torch.matmul(gg, vv.transpose(2, 3))
                ds = p * (ds - (p * ds).sum(-1, keepdim=True)) * s["scale"]
                dq[at:at + n, qh] = torch.matmul(ds, kk).flatten(0, 1).transpose(0, 1).to(q.dtype)
                dk[key:key + m, kv] = torch.matmul(ds.transpose(2, 3), qq).sum(1).transpose(0, 1).to(k.dtype)
    return o if grad is None else [o, dq, dk, dv]


def _turn(x, cos, sin, layout):
    """x [tokens, heads, dim] in 32 bits, its first 2 * cos.shape[1] elements turned; the result in x's type."""
    half = cos.shape[1]
    y = x.float()
    part = y[..., :2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if layout == "interleaved" else (part[..., :half], part[..., half:])
    c, s = cos[:, None], sin[:, None]
    a, b = a * c - b * s, a * s + b * c
    part = torch.stack((a, b), dim=-1).flatten(-2) if layout == "interleaved" else torch.cat((a, b), dim=-1)
    return torch.cat((part, y[..., 2 * half:]), dim=-1).to(x.dtype)


def _plain_rotary(s):
    cos, sin = (t[s["positions"].long()] for t in s["rope"])
    out = [_turn(t.detach(), cos, sin, s["layout"]) for t in (s["q"], s["k"])]
    if s["grads"] is not None:
        out += [_turn(g, cos, -sin, s["layout"]) for g in s["grads"]]   # the transpose of a rotation turns the other way
    return out


def _plain_sample(s):
    logits = s["logits"].double()
    rows, vocab = logits.shape

    def each(name):   # settings count as 32-bit numbers
        t = s[name] if torch.is_tensor(s[name]) else torch.tensor(s[name], dtype=torch.float32, device=logits.device)
        return t.double().expand(rows)[:, None]

    temperature, top_k, top_p, min_p = (each(name) for name in ("temperature", "top_k", "top_p", "min_p"))
    high = logits.amax(-1, keepdim=True)
    weight = torch.exp((logits - high) / torch.where(temperature > 0, temperature, 1.0))
    sorted_weight, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    sorted_weight = weight.gather(1, order)
    rank = torch.arange(vocab, device=logits.device)
    kept = (top_k <= 0) | (rank < top_k)
    total = torch.cumsum(torch.where(kept, sorted_weight, 0.0), -1)
    kept = kept & ((top_p >= 1) | (rank == 0) | (total - sorted_weight < top_p * total[:, -1:]))
    kept = kept & (sorted_weight >= min_p)
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    total = torch.cumsum(torch.where(kept, weight, 0.0), -1)
    passed = total > s["uniform"].double()[:, None] * total[:, -1:]
    index = torch.arange(vocab, device=logits.device)
    drawn = torch.where(passed & kept, index, vocab).amin(-1)
    likeliest = torch.where(logits == high, index, vocab).amin(-1)
    return torch.where(temperature[:, 0] > 0, drawn, likeliest)


def run(state):
    s, op = state, state["op"]
    if not own:
        return _plain_sample(s) if op == "sample" else _plain_rotary(s) if op == "rotary" else _plain_attention(s)
    from mccl_b200 import ops
    if op in ("prompt", "train"):
        o = ops.packed_attention(s["q"], s["k"], s["v"], s["offsets"], s["k_offsets"], scale=s["scale"], window=s["window"], sinks=s["sinks"])
        return o if op == "prompt" else [o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["grad"])]
    if op == "rotary":
        q, k = ops.rotary(s["q"], s["k"], rope=s["rope"], positions=s["positions"], layout=s["layout"])
        return [q, k] if s["grads"] is None else [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), s["grads"])]
    return ops.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


# ------------------------------------------------------------------------------------------------------------- work ----
def work(case):
    if case["op"] in ("prompt", "train"):
        lengths, before = _spread(case, case["longest"]), _spread(case, case["before"])
        most = case["window"] + case["sinks"] if case["window"] else sum(lengths) + sum(before)
        # positions see what is before them, themselves and no more than the window and the first few (every length is as likely to meet any other)
        mean = sum(before) // case["texts"]
        pairs = float(sum(min(p + 1, most) for n in lengths for p in range(mean, mean + n)))
        rows = sum(lengths) + case["spare"]
        keys = rows + sum(before)
        q, kv = 2.0 * rows * case["heads"] * case["dim"], 2.0 * keys * case["kv_heads"] * case["dim"]
        if case["op"] == "prompt":
            return {"bytes": 2 * q + 2 * kv, "flops": 4.0 * pairs * case["heads"] * case["dim"]}
        # two products forward, five backward
        return {"bytes": 4 * q + 4 * kv, "flops": 14.0 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "rotary":
        elements = float(case["tokens"]) * (case["heads"] + case["kv_heads"])
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * elements * case["dim"] * 4 + 4.0 * case["tokens"], "flops": passes * 3.0 * elements * case["rotated"]}
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": float(case["rows"]) * (case["vocab"] * size + 12), "flops": 4.0 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------------------------------------------------ exact ----
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("prompt", "train"):
        group, train = case["heads"] // case["kv_heads"], case["op"] == "train"
        leaves = [s[name].detach().double() for name in ("q", "k", "v")]
        o = torch.zeros_like(leaves[0])
        grads = [torch.zeros_like(t) for t in leaves]
        starts, key_starts = s["offsets"].tolist(), (s["offsets"] if s["k_offsets"] is None else s["k_offsets"]).tolist()
        for b in range(case["texts"]):
            rows, keys = slice(starts[b], starts[b + 1]), slice(key_starts[b], key_starts[b + 1])
            n, m = rows.stop - rows.start, keys.stop - keys.start
            if n == 0:
                continue
            at = torch.arange(n, device="cuda") + (m - n)
            back = at.unsqueeze(1) - torch.arange(m, device="cuda")   # how far behind the query a key is
            hidden = back < 0
            if case["window"]:
                hidden |= (back >= case["window"]) & (torch.arange(m, device="cuda") >= case["sinks"])
            for h in range(case["heads"]):
                qq, kk, vv = leaves[0][rows, h], leaves[1][keys, h // group], leaves[2][keys, h // group]
                score = (qq @ kk.T).mul_(case["dim"] ** -0.5).masked_fill_(hidden, -math.inf)
                weight = score.sub_(torch.logsumexp(score, 1, keepdim=True)).exp_()
                o[rows, h] = weight @ vv
                if train:
                    g = s["grad"][rows, h].double()
                    inner = (g * o[rows, h]).sum(1, keepdim=True)
                    ds = (g @ vv.T).sub_(inner).mul_(weight).mul_(case["dim"] ** -0.5)
                    grads[0][rows, h] = ds @ kk
                    grads[1][keys, h // group] += ds.T @ qq
                    grads[2][keys, h // group] += weight.T @ g
        return [o, *grads] if train else o
    if case["op"] == "rotary":
        half, out = case["rotated"] // 2, []
        turn = torch.complex(s["rope"][0].double(), s["rope"][1].double())[s["positions"].long()].unsqueeze(1)
        for x, z in ((s["q"], turn), (s["k"], turn)) + (() if s["grads"] is None else tuple((g, turn.conj()) for g in s["grads"])):
            y = x.detach().double().clone()
            pairs = y[..., :2 * half].unflatten(-1, (half, 2) if case["layout"] == "interleaved" else (2, half))
            along = -1 if case["layout"] == "interleaved" else -2
            turned = torch.view_as_real(torch.complex(pairs.select(along, 0).contiguous(), pairs.select(along, 1).contiguous()) * z)
            y[..., :2 * half] = (turned if along == -1 else turned.transpose(-1, -2)).flatten(-2)
            out.append(y)
        return out
    import numpy as np
    logits, uniform = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
    chosen = []
    for r in range(case["rows"]):
        t, k, p, low = (float(s[name][r]) if torch.is_tensor(s[name]) else float(np.float32(s[name])) for name in ("temperature", "top_k", "top_p", "min_p"))
        x = logits[r]
        if t <= 0:
            chosen.append(int(x.argmax()))
            continue
        weight = np.exp((x - x.max()) / t)
        order = np.lexsort((np.arange(len(x)), -x))   # likeliest first, equal ones by their number
        if k > 0:
            order = order[:int(k)]
        if p < 1:
            sums = np.cumsum(weight[order])
            order = order[:1 + int(np.searchsorted(sums, p * sums[-1]))]
        order = np.sort(order[weight[order] >= low])
        sums = np.cumsum(weight[order])
        chosen.append(int(order[min(len(order) - 1, np.searchsorted(sums, uniform[r] * sums[-1], side="right"))]))
    return torch.tensor(chosen, device="cuda")
