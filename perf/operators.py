"""Operators that can be timed next to their plain forms: products with 8-bit floating-point weights (dense projections and the experts of
an MoE layer) and the router's balance loss.

Weights are E4M3 with one f32 scale for each block of 128 x 128, the layout of FP8 checkpoints.  Rows of activations are f32; they become E4M3 with
one scale for each 128 columns, the smallest power of two that keeps the block's largest magnitude at or below 448, so that dividing by it is exact.
A product is  y[n][m] = sum over column blocks b of  x_scale[n][b] * w_scale[m/128][b] * (sum over the block's columns of xq * wq).

The experts take the pairs (token << 4) | slot sorted by expert, with offsets[experts + 1]; gate/up writes h[token][slot][n_ff] = silu(gate x) * (up x),
down writes contrib[token][slot][n_embd] = routing weight * down h.

The balance loss of T router rows is  coef * E / (N * k) * sum_e counts[e] * P[e],  N tokens that the mask leaves, counts[e] of their N * k selections, P[e] the
mean of their softmax probabilities; its gradient goes to the logits (the counts have none).  Logits that are not finite count as -3.4e38, as the
selection takes them, and get no gradient.
"""
import importlib
import math

import numpy as np
import torch

own = False

FLOOR = -3.4e38
_contexts = {}


def _linear(name, n, M, K):
    return {"name": name, "op": "linear", "n": n, "M": M, "K": K}


def _experts(name, op, tokens, experts=256, used=8):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "used": used, "n_embd": 2048, "n_ff": 512}


def _balance(name, tokens, experts, used, mask, ties=False):
    return {"name": name, "op": "balance", "tokens": tokens, "experts": experts, "used": used, "mask": mask, "blocked": ties}


def listed():
    return [
        # one stream's decode step: a projection outside the experts, where latency is all
        _linear("linear_1", 1, 4096, 2048),
        # the same for 16 slots, the wide way in
        _linear("linear_16", 16, 2048, 4096),
        # the head of the model for one token: a matrix that is read once from HBM
        _linear("linear_head", 1, 151936, 2048),
        # the rest of a prompt, into a matrix whose sizes fit no tile
        _linear("linear_77_odd", 77, 1000, 1040),
        # a prompt chunk's projection
        _linear("linear_1000", 1000, 4096, 2048),
        # a long prompt in one chunk, the largest projection
        _linear("linear_4096", 4096, 8192, 4096),
        # decode, 16 slots: about 101 of 256 experts have a pair or two each
        _experts("gateup_16", "gateup", 16),
        # a long prompt: 128 pairs an expert on average
        _experts("gateup_4096", "gateup", 4096),
        # decode on the wider layer (512 experts, top 10)
        _experts("down_5_512x10", "down", 5, 512, 10),
        # a long prompt
        _experts("down_4096", "down", 4096),
        # a short batch on its way through a fine-tuning step, padded, with experts that are switched off by an infinite logit
        _balance("balance_77", 77, 512, 10, True, True),
        # a training batch of 16 sequences of 2048 tokens
        _balance("balance_32768", 32768, 256, 8, False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "gateup", "down", "balance"))
    if op == "linear":
        n, M, K = _log_int(rng, 1, 4096), _log_int(rng, 100, 65536), 16 * rng.randint(8, 256)
        while n * M * K > 4096 * 8192 * 4096 or n * M > 1 << 28:
            M = max(1, M // 2)
        return {"op": op, "n": n, "M": M, "K": K}
    wide = rng.random() < 0.3
    if op == "balance":
        return {"op": op, "tokens": _log_int(rng, 1, 32768), "experts": rng.choice((60, 128, 256)) if not wide else 512, "used": rng.choice((4, 8)) if not wide else 10,
                "mask": rng.random() < 0.5, "blocked": rng.random() < 0.3}
    return {"op": op, "tokens": _log_int(rng, 1, 2048 if wide else 4096), "experts": 512 if wide else rng.choice((64, 128, 256)), "used": 10 if wide else 8,
            "n_embd": 256 * rng.randint(4, 8), "n_ff": 256 * rng.randint(1, 2)}


# ------------------------------------------------------------------ what a user's program has in hand

class State:
    pass


def _blocks(K):
    return (K + 127) // 128


def _fp8_weights(gen, mats, M, K):
    """Weights of a trained layer's size as a checkpoint holds them: E4M3 bytes [mats][M][K], f32 scales [mats][M/128][K/128]."""
    mb, kb = _blocks(M), _blocks(K)
    w = torch.empty((mats, M, K), dtype=torch.uint8, device="cuda")
    scale = torch.empty((mats, mb, kb), device="cuda")
    for at in range(0, mats, 32):
        m = min(32, mats - at)
        v = torch.randn((m, M, K), device="cuda", generator=gen) * 0.02
        v = torch.nn.functional.pad(v, (0, kb * 128 - K, 0, mb * 128 - M)).view(m, mb, 128, kb, 128)
        v *= torch.rand((m, mb, 1, kb, 1), device="cuda", generator=gen) + 0.5
        s = v.abs().amax(dim=(2, 4), keepdim=True) / 448
        q = (v / s).to(torch.float8_e4m3fn).view(torch.uint8).view(m, mb * 128, kb * 128)
        w[at:at + m] = q[:, :M, :K]
        scale[at:at + m] = s.view(m, mb, kb)
    return w, scale


def _rows(gen, *shape):
    """Rows behind a norm: N(0, 1), some columns of every row larger, as activations have them."""
    x = torch.randn(shape, device="cuda", generator=gen)
    return x * (1 + 9 * (torch.rand(shape[-1:], device="cuda", generator=gen) < 0.01))


def _selection(gen, tokens, experts, used):
    """Selection records [tokens][40 words], as the library's selection writes them."""
    logits = torch.randn((tokens, experts), device="cuda", generator=gen) + 0.5 * torch.randn((1, experts), device="cuda", generator=gen)
    top, ids = logits.topk(used, dim=1)
    sel = torch.zeros((tokens, 40), dtype=torch.int32, device="cuda")
    sel[:, :used] = ids.int()
    sel[:, 16:16 + used] = torch.softmax(top, 1).view(torch.int32)
    return logits, sel


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = State()
    s.case, op = case, case["op"]
    if op == "linear":
        n, M, K = case["n"], case["M"], case["K"]
        w, scale = _fp8_weights(gen, 1, M, K)
        s.w, s.w_scale = w[0], scale[0]
        s.x = _rows(gen, n, K)
        s.q, s.scale = torch.empty((n, K), dtype=torch.uint8, device="cuda"), torch.empty((n, _blocks(K)), device="cuda")
        s.y = torch.empty((n, M), device="cuda")
    elif op == "balance":
        T, E, k = case["tokens"], case["experts"], case["used"]
        s.logits, s.sel = _selection(gen, T, E, k)
        if case["blocked"]:
            s.logits[:, torch.randperm(E, device="cuda", generator=gen)[:E // 16]] = -math.inf
            s.sel[:, :k] = s.logits.topk(k, dim=1).indices.int()
        s.mask = (torch.rand(T, device="cuda", generator=gen) < 0.8).to(torch.uint8) if case["mask"] else None
        s.coef = 1e-2
        s.d_loss = torch.rand(1, device="cuda", generator=gen) + 0.5
        s.counts = torch.empty(E + 1, dtype=torch.int32, device="cuda")
        s.probs, s.loss, s.d_logits = torch.empty(E, device="cuda"), torch.empty(1, device="cuda"), torch.empty((T, E), device="cuda")
    else:
        T, E, k, D, F = case["tokens"], case["experts"], case["used"], case["n_embd"], case["n_ff"]
        _, s.sel = _selection(gen, T, E, k)
        expert = s.sel[:, :k].reshape(-1).long()
        order = torch.argsort(expert, stable=True)
        s.pairs = ((order // k << 4) | order % k).int()
        count = torch.bincount(expert, minlength=E)
        s.offsets = torch.cat([count.new_zeros(1), count.cumsum(0)]).int()
        s.most = int(count.max())                       # pairs of the busiest expert
        s.used = count.nonzero().view(-1)               # experts that have pairs
        s.place = (count.cumsum(0) - count)[s.used]
        if op == "gateup":
            s.gate, s.gate_scale = _fp8_weights(gen, E, F, D)
            s.up, s.up_scale = _fp8_weights(gen, E, F, D)
            s.x = _rows(gen, T, D)
            s.out = torch.zeros((T, k + 1, F), device="cuda")
        else:
            s.down, s.down_scale = _fp8_weights(gen, E, D, F)
            s.x = _rows(gen, T * (k + 1), F) * torch.rand((T * (k + 1), 1), device="cuda", generator=gen)
            s.out = torch.zeros((T, k, D), device="cuda")
        s.q = torch.empty(s.x.shape, dtype=torch.uint8, device="cuda")
        s.scale = torch.empty((s.x.shape[0], _blocks(s.x.shape[1])), device="cuda")
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ one pass

def _context(n_embd=2048, n_ff=512, experts=256, used=8):
    """The library context that a program opens once for its layer's sizes."""
    key = (n_embd, n_ff, experts, used)
    if key not in _contexts:
        qk = importlib.import_module("qwen-kernel_b200")
        _contexts[key] = qk.Context(qk.synth.Dims(n_embd=n_embd, n_ff=n_ff, n_expert=experts, n_used=used), n_layer=1, max_tokens=1, device=torch.cuda.current_device())
    return _contexts[key]


def _own(s):
    c, op = s.case, s.case["op"]
    if op == "linear":
        ctx = _context()
        ctx.fp8_quantize(s.x, c["n"], c["K"], s.q, s.scale)
        ctx.fp8_gemm(s.w, s.w_scale, s.q, s.scale, s.y, c["M"], c["K"], c["n"])
        return s.y, s.q.view(torch.float8_e4m3fn), s.scale
    if op == "balance":
        ctx = _context(experts=c["experts"], used=c["used"])
        ctx.moe_balance(s.logits, s.sel, s.mask, c["tokens"], s.coef, s.counts, s.probs, s.loss)
        ctx.moe_balance_grad(s.logits, s.mask, s.counts, c["tokens"], s.coef, s.d_loss, s.d_logits)
        return s.loss, s.counts, s.probs, s.d_logits
    ctx = _context(c["n_embd"], c["n_ff"], c["experts"], c["used"])
    ctx.fp8_quantize(s.x, s.x.shape[0], s.x.shape[1], s.q, s.scale)
    if op == "gateup":
        ctx.moe_gateup_grouped_fp8(s.gate, s.gate_scale, s.up, s.up_scale, s.q, s.scale, s.offsets, s.pairs, s.out, c["tokens"])
    else:
        ctx.moe_down_grouped_fp8(s.down, s.down_scale, s.q, s.scale, s.sel, s.offsets, s.pairs, s.out, c["tokens"])
    return s.out


def _quantize(x):
    """E4M3 rows and their scales, the smallest power of two for each 128 columns that keeps the largest magnitude at or below 448 (1 for zeros)."""
    n, K = x.shape
    pad = _blocks(K) * 128 - K
    v = torch.nn.functional.pad(x, (0, pad)).view(n, -1, 128)
    most = v.abs().amax(2)
    m, e = torch.frexp(most)                                     # most = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    scale = torch.where(most > 0, torch.ldexp(torch.ones_like(most), (e - 9 + (m > 0.875)).clamp(min=-126)), torch.ones_like(most))
    return (v / scale[:, :, None]).to(torch.float8_e4m3fn).view(n, -1)[:, :K], scale


def _expand(q, scale, rows):
    """f32 values of E4M3 with a scale for each `rows` x 128."""
    s = scale.repeat_interleave(rows, -2)[..., :q.shape[-2], :].repeat_interleave(128, -1)[..., :q.shape[-1]]
    return q.view(torch.float8_e4m3fn).float() * s


def run(s):
    if own:
        return _own(s)
    c, op = s.case, s.case["op"]
    if op == "linear":
        q, scale = _quantize(s.x)
        return torch.matmul(_expand(q, scale, 1), _expand(s.w, s.w_scale, 128).t()), q, scale
    if op == "balance":
        E, k = c["experts"], c["used"]
        keep = torch.ones_like(s.logits[:, 0]) if s.mask is None else (s.mask != 0).float()
        fine = torch.isfinite(s.logits)
        v = torch.where(fine, s.logits, FLOOR)
        p = torch.exp(v - v.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        N = keep.double().sum()
        counts = torch.zeros(E + 1, dtype=torch.float64, device="cuda")
        counts.index_add_(0, s.sel[:, :k].reshape(-1).long(), keep.double().repeat_interleave(k))
        counts[E] = N
        per = torch.where(N > 0, 1 / N.clamp(min=1), 0)
        probs = (p.double() * keep[:, None]).sum(0) * per
        f = counts[:E] * (s.coef * E / k) * per                  # d loss / d probs
        loss = (f * probs).sum()
        g = (f * per * s.d_loss).float()
        d = p * (g - (p * g).sum(1, keepdim=True)) * keep[:, None]
        return loss.float().view(1), counts.int(), probs.float(), torch.where(fine, d, 0)
    k, T = c["used"], c["tokens"]
    q, scale = _quantize(s.x)
    rows = _expand(q, scale, 1)
    span = torch.arange(s.most, device="cuda")
    at = s.place[:, None] + span                                 # [used experts][most] places in the list of pairs
    real = span < (s.offsets[s.used + 1] - s.offsets[s.used])[:, None]
    pair = s.pairs[at.clamp(max=s.pairs.numel() - 1)].long()
    token, slot = pair >> 4, pair & 15
    if op == "gateup":
        x = rows[token]                                          # [used experts][most][n_embd]
        g = torch.matmul(x, _expand(s.gate[s.used], s.gate_scale[s.used], 128).transpose(1, 2))
        u = torch.matmul(x, _expand(s.up[s.used], s.up_scale[s.used], 128).transpose(1, 2))
        h = g / (1 + torch.exp(-g)) * u
        out = torch.zeros((T, k + 1, c["n_ff"]), device="cuda")
        out[token[real], slot[real]] = h[real]
        return out
    y = torch.matmul(rows[token * (k + 1) + slot], _expand(s.down[s.used], s.down_scale[s.used], 128).transpose(1, 2))
    w = s.sel[:, 16:16 + k].view(torch.float32)
    out = torch.zeros((T, k, c["n_embd"]), device="cuda")
    out[token[real], slot[real]] = y[real] * w[token[real], slot[real]][:, None]
    return out


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_rows(x):
    """(values, scales, E4M3 values) in 64 bits: the rounding to E4M3 spelt out, 4 significant bits, steps of 2^-9 below 2^-6, ties to even."""
    n, K = x.shape
    v = torch.zeros((n, _blocks(K) * 128), dtype=torch.float64, device=x.device)
    v[:, :K] = x
    v = v.view(n, -1, 128)
    most = v.abs().max(dim=2).values
    scale = torch.exp2(torch.ceil(torch.log2(most / 448)))
    scale = torch.where(most > 448 * scale, 2 * scale, scale)    # (a logarithm that was rounded across a whole number)
    scale = torch.where(most <= 224 * scale, scale / 2, scale)
    scale = torch.where(most > 0, scale.clamp(min=2.0**-126), torch.ones_like(scale))
    t = v / scale[:, :, None]
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0**-6))) - 3)
    q = torch.round(t / step) * step
    return (q * scale[:, :, None]).view(n, -1)[:, :K], scale, q.view(n, -1)[:, :K]


def _exact_weights(w, scale):
    """One matrix [M][K] in 64 bits, the bits of E4M3 taken apart."""
    b = w.to(torch.int64)
    e, m = b >> 3 & 15, (b & 7).double()
    v = torch.where(e > 0, (8 + m) * torch.exp2((e - 10).double()), m * 2.0**-9)
    v = torch.where(b >= 128, -v, v)
    M, K = w.shape
    at_m, at_k = torch.arange(M, device=w.device) // 128, torch.arange(K, device=w.device) // 128
    return v * scale.double()[at_m][:, at_k]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        v, scale, q = _exact_rows(s.x)
        y = torch.empty((case["n"], case["M"]), dtype=torch.float64, device="cuda")
        for m in range(0, case["M"], 8192):                      # (a multiple of 128)
            y[:, m:m + 8192] = v @ _exact_weights(s.w[m:m + 8192], s.w_scale[m // 128:m // 128 + 64]).T
        return y, q, scale
    if op == "balance":
        T, E, k = case["tokens"], case["experts"], case["used"]
        logits, ids = s.logits.double().cpu().numpy(), s.sel.cpu().numpy()[:, :k]
        keep = np.ones(T, bool) if s.mask is None else s.mask.cpu().numpy() != 0
        fine = np.isfinite(logits)
        z = np.where(fine, logits, FLOOR)
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        N = int(keep.sum())
        counts = np.bincount(ids[keep].reshape(-1), minlength=E)[:E]
        probs = p[keep].sum(0) / max(N, 1)
        unit = s.coef * E / (max(N, 1) * k)
        loss = unit * (counts * probs).sum()
        weight = unit * counts / max(N, 1) * float(s.d_loss)
        grad = np.zeros((T, E))
        grad[keep] = p[keep] * (weight - (p[keep] @ weight)[:, None])
        grad[~fine] = 0
        return np.array([loss]), np.append(counts, N).astype(np.int32), probs, grad
    k, F, D = case["used"], case["n_ff"], case["n_embd"]
    v, _, _ = _exact_rows(s.x)
    offsets, pairs = s.offsets.tolist(), s.pairs.long()
    out = torch.zeros(s.out.shape, dtype=torch.float64, device="cuda")
    w = s.sel[:, 16:16 + k].view(torch.float32).double()
    for e in range(case["experts"]):
        mine = pairs[offsets[e]:offsets[e + 1]]
        if mine.numel() == 0:
            continue
        token, slot = mine // 16, mine % 16
        if op == "gateup":
            g = v[token] @ _exact_weights(s.gate[e], s.gate_scale[e]).T
            u = v[token] @ _exact_weights(s.up[e], s.up_scale[e]).T
            out[token, slot] = g * torch.sigmoid(g) * u
        else:
            out[token, slot] = (v[token * (k + 1) + slot] @ _exact_weights(s.down[e], s.down_scale[e]).T) * w[token, slot][:, None]
    return out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "linear":
        n, M, K = case["n"], case["M"], case["K"]
        return {"bytes": M * K + 4 * _blocks(M) * _blocks(K) + 4 * n * K + n * K + 4 * n * _blocks(K) + 4 * n * M, "flops": 2 * n * M * K}
    T, E, k = case["tokens"], case["experts"], case["used"]
    if op == "balance":
        return {"bytes": 8 * T * E + 4 * T * k + 8 * E, "flops": 12 * T * E}
    D, F = case["n_embd"], case["n_ff"]
    live = E * (1 - (1 - k / E) ** T)                            # experts that T independent rows choose, on average
    if op == "gateup":
        return {"bytes": live * 2 * F * D + 4 * T * D + 4 * T * k * F, "flops": 4 * T * k * F * D}
    return {"bytes": live * F * D + 4 * T * k * F + 4 * T * k * D, "flops": 2 * T * k * F * D}
