"""The transformer operators over packs of sequences, as cases with inputs, plain forms and 64-bit results.

Three operators, five calls:

  attention        ``ops.attention_pack_mode``: softmax attention inside every sequence of a pack, forward
  attention_train  the same with the gradients of q, k and v
  cache            ``ops.cached_attention``: the newest tokens of every sequence against its cached keys and values
  norm             ``ops.layer_norm`` (optionally of a sum, as a post-norm layer calls it), forward
  norm_train       the same with the gradients of the input, the weight and the bias

``own`` selects what ``run`` executes: the plain form (elementary torch operations in 32 bits, rounded once at the end)
or the calls that a user makes of ``vision3d_amd.ops``.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------- the cases
def _attention(name, op, dtype, heads, kv_heads, dim, batch, tokens, keys=0, causal=False, edge=False, fused=False):
    """``keys`` = 0: self-attention (the keys are the queries' own sequences), else the keys' total.  ``edge``: an empty
    sequence, one of a single token and, where the keys are apart, one with no keys are in the pack.  ``fused``: q, k and
    v are views of one (tokens, heads + 2 kv_heads, dim) projection."""
    return {"name": name, "op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "batch": batch,
            "tokens": tokens, "keys": keys, "causal": causal, "edge": edge, "fused": fused}


def _cache(name, dtype, heads, kv_heads, dim, batch, tokens, capacity):
    return {"name": name, "op": "cache", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "batch": batch, "tokens": tokens, "capacity": capacity}


def _norm(name, op, dtype, rows, channels, residual):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "channels": channels, "residual": residual}


def listed():
    return [
        # the norm behind the attention of a handful of query tokens: one launch, latency is all there is to it
        _norm("norm fp32 16x256", "norm", "float32", 16, 256, False),
        # post-norm layer over the points of four 30k-point scenes at 256 channels
        _norm("norm fp32 120000x256 sum", "norm", "float32", 120000, 256, True),
        # training of a wide layer in bf16 over a large pack
        _norm("norm train bf16 65536x1024", "norm_train", "bfloat16", 65536, 1024, True),
        # an odd channel count: rows start at every alignment
        _norm("norm train fp16 20011x771", "norm_train", "float16", 20011, 771, False),
        # cross-attention between the superpoints of 32 pairs of scenes, 4 heads of 64, full precision
        _attention("cross fp32 4x64", "attention", "float32", 4, 4, 64, 32, 16384, keys=15003),
        # a prompt: six sequences, grouped heads, causal, q / k / v straight out of one projection
        _attention("prompt bf16 32/8x128", "attention", "bfloat16", 32, 8, 128, 6, 12288, causal=True, fused=True),
        # a pack with an empty sequence, one of one token and one without keys; odd head count and head size
        _attention("ragged fp16 6/3x80", "attention", "float16", 6, 3, 80, 19, 7001, keys=9003, causal=True, edge=True),
        # training step of a causal layer with grouped heads
        _attention("train bf16 16/4x128", "attention_train", "bfloat16", 16, 4, 128, 5, 8192, causal=True),
        # training step of the superpoint transformer: full precision, every pair of a sequence
        _attention("train fp32 4x64", "attention_train", "float32", 4, 4, 64, 16, 8000, edge=True),
        # one stream, a short cache: the smallest step there is
        _cache("step fp32 1x500", "float32", 4, 4, 64, 1, 1, 512),
        # one new token for each of 32 streams, grouped heads
        _cache("step bf16 32x8192", "bfloat16", 32, 8, 128, 32, 1, 8192),
        # four tokens at a time against few long caches
        _cache("steps fp16 6x32768", "float16", 16, 2, 128, 6, 4, 32768),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cost(case):
    """What a case costs the plain form: pairs times channels for the attentions, values for the norms."""
    if case["op"].startswith("norm"):
        return case["rows"] * case["channels"] * 40.0
    if case["op"] == "cache":
        return 1.0 * case["batch"] * case["capacity"] * (case["kv_heads"] * case["dim"] * 8 + 16 * case["heads"] * case["tokens"])
    q, s = _pack_lengths(case)
    steps = 3.0 if case["op"] == "attention_train" else 1.0
    return steps * case["batch"] * case["heads"] * max(q) * max(s) * (case["dim"] + 40)


_most = {}


def draw(rng):
    if not _most:
        for c in listed():
            _most[c["op"]] = max(_most.get(c["op"], 0.0), _cost(c))
    op = rng.choice(["norm", "norm_train", "attention", "attention", "attention_train", "cache"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    while True:
        if op.startswith("norm"):
            case = _norm("", op, dtype, _log_int(rng, 1, 120000), _log_int(rng, 16, 4096), rng.random() < 0.5)
        else:
            kv = rng.choice([1, 2, 3, 4, 8])
            heads = kv * rng.choice([1, 1, 2, 4, 8])
            dim = rng.choice([32, 40, 64, 72, 80, 96, 100, 128, 128, 192, 256])
            if op == "cache":
                case = _cache("", dtype, heads, kv, dim, _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 5]),
                              _log_int(rng, 64, 32768))
            else:
                batch = _log_int(rng, 1, 48)
                tokens = batch * _log_int(rng, 24, 2400) + rng.randrange(batch)
                keys = 0 if rng.random() < 0.6 else batch * _log_int(rng, 24, 2400) + rng.randrange(batch)
                case = _attention("", op, dtype, heads, kv, dim, batch, tokens, keys, causal=rng.random() < 0.5,
                                  edge=batch > 6 and rng.random() < 0.5, fused=keys == 0 and rng.random() < 0.5)
        if _cost(case) <= _most[op]:
            del case["name"]
            return case


# --------------------------------------------------------------------------------------------------------- the inputs
def _ragged(rng, count, total):
    share = [rng.uniform(0.2, 1.0) for _ in range(count)]
    whole = sum(share)
    lengths = [int(total * s / whole) for s in share]
    lengths[0] += total - sum(lengths)
    return lengths


def _pack_lengths(case):
    """The lengths of a pack's sequences (queries, keys): a function of the case alone."""
    rng = random.Random(case["tokens"] * 1000003 + case["keys"] * 101 + case["batch"])
    q = _ragged(rng, case["batch"], case["tokens"])
    s = list(q) if case["keys"] == 0 else _ragged(rng, case["batch"], case["keys"])
    if case["edge"]:
        for lengths in (q, s) if case["keys"] else (q,):
            lengths[0] += lengths[3] + lengths[4] - 1
            lengths[3], lengths[4] = 0, 1
        if case["keys"]:
            s[0] += s[5]
            s[5] = 0
        else:
            s = list(q)
    return q, s


def _cache_lengths(case):
    """How many rows of each cache are filled, the new tokens among them."""
    rng = random.Random(case["capacity"] * 1000003 + case["batch"])
    low = max(case["tokens"], case["capacity"] // 4)
    lengths = [rng.randint(low, case["capacity"]) for _ in range(case["batch"])]
    lengths[0] = max(low, case["capacity"] - 12)
    return lengths


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case, "dtype": dtype}
    if case["op"].startswith("norm"):
        rows, channels = case["rows"], case["channels"]
        # activations of one channel share an offset and a scale, as behind a linear layer
        spread = torch.rand((channels,), generator=gen, device=DEVICE) * 2 + 0.2
        offset = torch.randn((channels,), generator=gen, device=DEVICE) * 0.5
        x = torch.randn((rows, channels), generator=gen, device=DEVICE)
        state["feats"] = (x * spread + offset).to(dtype)
        state["residual"] = _randn(gen, (rows, channels), dtype) if case["residual"] else None
        state["weight"] = (torch.rand((channels,), generator=gen, device=DEVICE) + 0.5).to(dtype)
        state["bias"] = _randn(gen, (channels,), dtype, 0.2)
        if case["op"] == "norm_train":
            state["grad"] = _randn(gen, (rows, channels), dtype)
            for k in ("feats", "weight", "bias"):
                state[k].requires_grad_(True)
        return state
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "cache":
        b, t, cap = case["batch"], case["tokens"], case["capacity"]
        state["q"] = _randn(gen, (b, t, heads, dim), dtype, 1.5)
        state["k"] = _randn(gen, (b, cap, kv, dim), dtype)
        state["v"] = _randn(gen, (b, cap, kv, dim), dtype)
        state["lengths"] = torch.tensor(_cache_lengths(case), device=DEVICE)
        return state
    q_lengths, s_lengths = _pack_lengths(case)
    nq, ns = sum(q_lengths), sum(s_lengths)
    if case["fused"]:
        qkv = _randn(gen, (nq, heads + 2 * kv, dim), dtype, 1.2)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        q = _randn(gen, (nq, heads, dim), dtype, 1.5)
        k = _randn(gen, (ns, kv, dim), dtype)
        v = _randn(gen, (ns, kv, dim), dtype)
    if case["op"] == "attention_train":
        state["grad"] = _randn(gen, (nq, heads, dim), dtype)
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    state.update(q=q, k=k, v=v, q_lengths=torch.tensor(q_lengths, device=DEVICE),
                 s_lengths=torch.tensor(s_lengths, device=DEVICE), longest=(max(q_lengths), max(s_lengths)))
    return state


# ------------------------------------------------------------------------------------------------------ the plain forms
def _rows_of(lengths, longest):
    """(B, longest) row of every place of the padded batch, and which places are a sequence's own."""
    place = torch.arange(longest, device=lengths.device)
    first = lengths.cumsum(0) - lengths
    valid = place < lengths[:, None]
    return torch.where(valid, first[:, None] + place, 0), valid


def _softmax_parts(scores, seen):
    """exp(score - largest) of what is seen and its sum, in 32 bits; a row that sees nothing has zeros and a sum of 1."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p, torch.where(total == 0, 1.0, total)


def _fold(x, kv):
    """(B, L, H, D) -> (B, kv, H / kv * L, D): the query heads of a key head under one another."""
    b, n, h, d = x.shape
    return x.view(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, h // kv * n, d)


def _unfold(x, n):
    b, kv, rows, d = x.shape
    return x.view(b, kv, rows // n, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, kv * (rows // n), d)


def _plain_attention(s):
    case, dtype = s["case"], s["dtype"]
    kv, scale = case["kv_heads"], case["dim"] ** -0.5
    nq, ns = s["longest"]
    q_rows, q_valid = _rows_of(s["q_lengths"], nq)
    s_rows, s_valid = _rows_of(s["s_lengths"], ns)
    q = _fold(s["q"].detach().float()[q_rows], kv)
    k = s["k"].detach().float()[s_rows].transpose(1, 2).contiguous()
    v = s["v"].detach().float()[s_rows].transpose(1, 2).contiguous()
    seen = s_valid[:, None, :]
    if case["causal"]:  # the last query of a sequence sees all of its keys
        last = torch.arange(nq, device=q.device) + (s["s_lengths"] - s["q_lengths"])[:, None]
        seen = seen & (torch.arange(ns, device=q.device) <= last[:, :, None])
    seen = seen.expand(-1, nq, -1).repeat(1, case["heads"] // kv, 1)[:, None]
    p, total = _softmax_parts(torch.matmul(q, k.transpose(2, 3)) * scale, seen)
    p = p / total
    out = torch.matmul(p, v)
    if case["op"] == "attention":
        return _unfold(out, nq)[q_valid].to(dtype)
    g = _fold(s["grad"].float()[q_rows] * q_valid[:, :, None, None], kv)
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * out).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    grads = [_unfold(dq, nq)[q_valid]] + [x.transpose(1, 2)[s_valid] for x in (dk, dv)]
    return [_unfold(out, nq)[q_valid].to(dtype)] + [x.to(dtype) for x in grads]


def _plain_cache(s):
    case = s["case"]
    kv, t = case["kv_heads"], case["tokens"]
    q = _fold(s["q"].float(), kv)
    k = s["k"].float().transpose(1, 2).contiguous()
    v = s["v"].float().transpose(1, 2).contiguous()
    last = s["lengths"][:, None] - t + torch.arange(t, device=q.device)
    seen = torch.arange(case["capacity"], device=q.device) <= last[:, :, None]
    p, total = _softmax_parts(torch.matmul(q, k.transpose(2, 3)) * case["dim"] ** -0.5,
                              seen.repeat(1, case["heads"] // kv, 1)[:, None])
    return _unfold(torch.matmul(p, v) / total, t).to(s["dtype"])


EPS = 1e-5


def _plain_norm(s):
    x = s["feats"].detach().float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    w, b = s["weight"].detach().float(), s["bias"].detach().float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    unit = centred * rstd
    y = (unit * w + b).to(s["dtype"])
    if s["case"]["op"] == "norm":
        return y
    g = s["grad"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - unit * (gw * unit).mean(1, keepdim=True))
    return [y] + [t.to(s["dtype"]) for t in (dx, (g * unit).sum(0), g.sum(0))]


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from vision3d_amd import ops

    case = s["case"]
    if case["op"] == "cache":
        return ops.cached_attention(s["q"], s["k"], s["v"], s["lengths"])
    if case["op"].startswith("attention"):
        out = ops.attention_pack_mode(s["q"], s["k"], s["v"], s["q_lengths"], s["s_lengths"], causal=case["causal"])
        if case["op"] == "attention":
            return out
        return [out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])]
    y = ops.layer_norm(s["feats"], s["weight"], s["bias"], eps=EPS, residual=s["residual"])
    if case["op"] == "norm":
        return y
    return [y, *torch.autograd.grad(y, (s["feats"], s["weight"], s["bias"]), s["grad"])]


def run(state):
    if own:
        return _own(state)
    if state["case"]["op"] == "cache":
        return _plain_cache(state)
    return _plain_norm(state) if state["case"]["op"].startswith("norm") else _plain_attention(state)


# ------------------------------------------------------------------------------------------------------ what it has to do
def _pairs(case):
    """Pairs of a query token and a key that it sees, of all sequences."""
    if case["op"] == "cache":
        t = case["tokens"]
        return sum(max(0, n - t + 1 + i) for n in _cache_lengths(case) for i in range(t))
    q, s = _pack_lengths(case)
    if not case["causal"]:
        return sum(a * b for a, b in zip(q, s))
    total = 0
    for a, b in zip(q, s):  # queries see b - a + 1 ... b keys; the first ones may see none
        least = b - a + 1
        total += sum(range(max(least, 0), b + 1)) if b > 0 else 0
    return total


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"].startswith("norm"):
        n = case["rows"] * case["channels"]
        moved = 3 if case["residual"] else 2
        if case["op"] == "norm":
            return {"bytes": n * size * moved, "flops": 8.0 * n}
        return {"bytes": n * size * (moved + 2), "flops": 20.0 * n}
    per_pair = case["heads"] * case["dim"]
    if case["op"] == "cache":
        rows = sum(_cache_lengths(case))
        return {"bytes": size * (2 * rows * case["kv_heads"] * case["dim"] + 2 * case["batch"] * case["tokens"] * per_pair),
                "flops": 4.0 * per_pair * _pairs(case)}
    q, s = _pack_lengths(case)
    once = size * (2 * sum(q) * per_pair + 2 * sum(s) * case["kv_heads"] * case["dim"])
    if case["op"] == "attention":
        return {"bytes": once, "flops": 4.0 * per_pair * _pairs(case)}
    return {"bytes": 2 * once, "flops": 14.0 * per_pair * _pairs(case)}


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def _attend(q, k, v, causal, scale):
    """One sequence in 64 bits: q (T, H, D), k and v (S, KV, D) -> (T, H, D), by torch.softmax over each row's keys."""
    t, h, _ = q.shape
    n, kv, _ = k.shape
    if n == 0:
        return q * 0
    group = h // kv
    parts = []
    for i in range(h):
        logits = (q[:, i] @ k[:, i // group].T.contiguous()) * scale
        if causal:
            hidden = torch.ones((t, n), dtype=torch.bool, device=q.device).triu(n - t + 1)
            none = hidden.all(1, keepdim=True)
            weights = torch.softmax(logits.masked_fill(hidden & ~none, float("-inf")), 1).masked_fill(none, 0.0)
        else:
            weights = torch.softmax(logits, 1)
        parts.append(weights @ v[:, i // group])
    return torch.stack(parts, 1)


def _exact_pack(case, s):
    leaves = [s[n].detach().double().contiguous().requires_grad_("grad" in s) for n in ("q", "k", "v")]
    q, k, v = leaves
    q_lengths, s_lengths = _pack_lengths(case)
    outs, grads, at_q, at_s = [], [torch.zeros_like(x) for x in leaves], 0, 0
    for a, b in zip(q_lengths, s_lengths):
        rows, keys = slice(at_q, at_q + a), slice(at_s, at_s + b)
        at_q, at_s = at_q + a, at_s + b
        mine = [x.detach()[at].requires_grad_("grad" in s) for x, at in ((q, rows), (k, keys), (v, keys))]
        out = _attend(*mine, case["causal"], case["dim"] ** -0.5)
        outs.append(out.detach())
        if "grad" in s and a and b:
            got = torch.autograd.grad(out, mine, s["grad"][rows].double())
            for whole, at, g in zip(grads, (rows, keys, keys), got):
                whole[at] = g
    out = torch.cat(outs)
    return [out, *grads] if "grad" in s else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cache":
        outs = []
        for b, n in enumerate(_cache_lengths(case)):
            outs.append(_attend(s["q"][b].double(), s["k"][b, :n].double(), s["v"][b, :n].double(), True,
                                case["dim"] ** -0.5))
        return torch.stack(outs)
    if case["op"].startswith("attention"):
        return _exact_pack(case, s)
    x, w, b = (s[n].detach().double().requires_grad_(True) for n in ("feats", "weight", "bias"))
    total = x if s["residual"] is None else x + s["residual"].double()
    var, mean = torch.var_mean(total, dim=1, keepdim=True, correction=0)
    y = (total - mean) * torch.rsqrt(var + EPS) * w + b
    if case["op"] == "norm":
        return y.detach()
    return [y.detach(), *torch.autograd.grad(y, (x, w, b), s["grad"].double())]
