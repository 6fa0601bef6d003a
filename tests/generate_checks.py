"""Shared by the CPU and GPU tests of the generator: the decoder in 32 bits, and errors against it."""
import torch
import torch.nn.functional as F


def reference_logits(model, tokens, matrices=None, window=None, sinks=0):
    """Logits [S, V] of a decoder for tokens [S] in fp32.  matrices: what a Linear's weight is replaced by; window / sinks as the generator's."""
    cfg, w = model.cfg, (lambda m: m.weight.float() if matrices is None else matrices[m])
    S, H, hd = len(tokens), cfg.n_heads, cfg.head_dim

    def norm(m, x):
        if cfg.norm == "layernorm":
            return F.layer_norm(x, x.shape[-1:], m.weight, m.bias, cfg.eps)
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.eps) * m.weight

    def linear(m, x):
        return F.linear(x, w(m), m.bias)

    i, j = torch.arange(S, device=tokens.device)[:, None], torch.arange(S, device=tokens.device)[None]
    seen = j <= i
    if window is not None:
        seen &= (j > i - window) | (j < sinks)
    x = model.tok.weight[tokens]
    if model.pos is not None:
        x = x + model.pos.weight[:S]
    for b in model.blocks:
        q, k, v = linear(b.qkv, norm(b.ln1, x)).view(S, 3, H, hd).unbind(1)
        if cfg.pos == "rope":
            inv = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device=x.device, dtype=torch.float32) / hd))
            angle = torch.outer(torch.arange(S, device=x.device, dtype=torch.float32), inv)[:, None]

            def turn(t):
                a, c = t[..., 0::2], t[..., 1::2]
                return torch.stack((a * angle.cos() - c * angle.sin(), a * angle.sin() + c * angle.cos()), -1).flatten(-2)
            q, k = turn(q), turn(k)
        s = torch.einsum("ihd,jhd->hij", q, k) * hd ** -0.5
        p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
        x = x + linear(b.proj, torch.einsum("hij,jhd->ihd", p, v).reshape(S, -1))
        h = norm(b.ln2, x)
        if cfg.act == "swiglu":
            gate, up = linear(b.gate_up, h).chunk(2, -1)
            h = F.silu(gate) * up
        else:
            h = F.gelu(linear(b.up, h))
        x = x + linear(b.down, h)
    return F.linear(norm(model.ln_f, x), model.head_weight())


def dequantized(model, group):
    """What 4 bits make of each layer's matrices."""
    from mccl_b200 import ops
    out = {}
    for b in model.blocks:
        for m in (b.qkv, b.proj, b.gate_up if model.cfg.act == "swiglu" else b.up, b.down):
            out[m] = ops.quantize_w4(m.weight, group)._plain().float()
    return out


def sharpen(model):
    """Larger weights: at their initial size every layer adds so little that an error in one would hardly be seen."""
    with torch.no_grad():
        for b in model.blocks:
            for m in b.children():
                if hasattr(m, "weight") and m.weight.dim() == 2:
                    m.weight.mul_(4.0)
                    if m.bias is not None:
                        m.bias.normal_(0.0, 0.1)
    return model


def rms(x):
    return x.float().pow(2).mean().sqrt().item()
