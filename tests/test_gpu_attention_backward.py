"""The gradients of ops.attention_pack_mode against the formulas in 64 bits and against differences, and a transformer
layer of all three operators over a pack."""
import pytest
import torch

from vision3d_amd import ops

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ULP = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _sequence(q, k, v, g, causal, scale, dtype):
    """One sequence of one query head in 64 bits: (T,D), (S,D) -> dq, dk, dv and the bounds of their errors.

    A score is a sum of D products in 32 bits: off by es = 2 (D + 4) half steps of sum |q| |k| in p's relative terms (its own
    and the log-sum's).  p and ds are rounded to the type before they meet v, k and q.  dp is a sum of D products, delta a
    sum over an output that was rounded to the type and carries the forward's error.  Sums over rows or keys: 64 steps for
    the instructions' order plus one per 32 terms."""
    t, d = q.shape
    s = k.shape[0]
    half, own = _half(dtype), (_half(dtype) if dtype != torch.float32 else ULP)
    seen = torch.ones((t, s), dtype=torch.bool)
    if causal:
        seen = torch.arange(s)[None] <= torch.arange(t)[:, None] + (s - t)
    logits = (q @ k.T) * scale
    logits = logits.masked_fill(~seen, float("-inf"))
    none = ~seen.any(1, keepdim=True)
    p = torch.softmax(logits.masked_fill(none, 0.0), 1).masked_fill(~seen, 0.0)
    o = p @ v
    dp, delta = g @ v.T, (g * o).sum(1, keepdim=True)
    inner = dp - delta
    ds = p * inner
    es = (2 * (d + 4) * ULP * ((q.abs() @ k.abs().T) * scale).amax(1, keepdim=True)) if s else torch.zeros(t, 1, dtype=q.dtype)
    steps = (64 + max(s, t) / 32) * ULP
    o_err = half * o.abs() + (p @ v.abs()) * (own + es + steps)
    delta_err = (g.abs() * o_err).sum(1, keepdim=True) + (d + 4) * ULP * (g.abs() * o.abs()).sum(1, keepdim=True)
    dp_err = (d + 4) * ULP * (g.abs() @ v.abs().T)
    ds_err = p * (inner.abs() * (own + es + steps) + dp_err + delta_err)
    p_err = p * (own + es + steps)
    dq, dk, dv = (ds @ k) * scale, (ds.T @ q) * scale, p.T @ g
    add = steps * scale
    errs = (ds_err @ k.abs() * scale + add * (ds.abs() @ k.abs()), ds_err.T @ q.abs() * scale + add * (ds.abs().T @ q.abs()),
            p_err.T @ g.abs() + steps * (p.T @ g.abs()))
    return (dq, dk, dv), errs


def _expect(q, k, v, g, q_lengths, s_lengths, causal, scale, dtype):
    q, k, v, g = (t.double() for t in (q, k, v, g))
    h, kv = q.shape[1], k.shape[1]
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    errs = [torch.zeros_like(t) for t in (q, k, v)]
    at, key = 0, 0
    for a, b in zip(q_lengths, s_lengths):
        rows, keys = slice(at, at + a), slice(key, key + b)
        at, key = at + a, key + b
        for i in range(h):
            j = i // (h // kv)
            got, err = _sequence(q[rows, i], k[keys, j], v[keys, j], g[rows, i], causal, scale, dtype)
            grads[0][rows, i], errs[0][rows, i] = got[0], err[0]
            for n in (1, 2):
                grads[n][keys, j] += got[n]
                errs[n][keys, j] += err[n]
    return grads, errs


def _inputs(q_lengths, s_lengths, heads, kv, dim, dtype, seed, spare=0):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda n, h: torch.randn((n, h, dim), generator=gen).to(dtype)
    nq, ns = sum(q_lengths) + spare, sum(s_lengths) + spare
    return mk(nq, heads), mk(ns, kv), mk(ns, kv), mk(nq, heads)


def _check(dtype, q_lengths, s_lengths, heads, kv, dim, causal, seed=0, spare=0):
    q, k, v, g = _inputs(q_lengths, s_lengths, heads, kv, dim, dtype, seed, spare)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = ops.attention_pack_mode(*leaves, torch.tensor(q_lengths).to(DEV), torch.tensor(s_lengths).to(DEV), causal=causal)
    with torch.no_grad():
        plain = ops.attention_pack_mode(*leaves, torch.tensor(q_lengths).to(DEV), torch.tensor(s_lengths).to(DEV), causal=causal)
    assert torch.equal(plain, out)
    got = torch.autograd.grad(out, leaves, g.to(DEV), retain_graph=True)
    again = torch.autograd.grad(out, leaves, g.to(DEV))
    want, errs = _expect(q, k, v, g, q_lengths, s_lengths, causal, dim ** -0.5, dtype)
    for name, a, b, ref, err in zip("qkv", got, again, want, errs):
        assert a.dtype == dtype and torch.equal(a, b), name
        off = (a.cpu().double() - ref).abs()
        tol = err + _half(dtype) * ref.abs() + ULP
        assert (off <= tol).all(), f"d{name}: {(off / tol).max().item():.2f} of the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [8, 32, 33, 64, 80, 100, 128, 192, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_head_sizes(dtype, dim, causal):
    _check(dtype, [70, 1, 0, 33, 5], [70, 1, 0, 33, 5], 2, 1, dim, causal, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (6, 3), (8, 1), (14, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_heads_and_cross_lengths(dtype, heads, kv, causal):
    _check(dtype, [37, 90, 11, 0, 1, 129], [64, 31, 0, 40, 1, 65], heads, kv, 64, causal, seed=heads, spare=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_tile_borders(dtype):
    for n in (1, 31, 32, 33, 64, 65, 127, 128, 129, 257):
        _check(dtype, [n], [n], 1, 1, 64, True, seed=n)
    _check(dtype, [3], [700], 2, 1, 128, False)
    _check(dtype, [700], [3], 2, 1, 128, False)
    _check(dtype, [300], [200], 4, 1, 64, True)  # the first hundred queries see nothing


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("count", [2, 63, 64, 65, 200])
def test_numbers_of_sequences(count, causal):
    # up to 64 sequences are looked up one to a lane and, causal, numbered by work; more are divided among the lanes
    gen = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 70, (count,), generator=gen).tolist()
    lengths[count // 2] = 300
    keys = torch.randint(0, 70, (count,), generator=gen).tolist()
    keys[-1] = 200
    _check(torch.bfloat16, lengths, keys, 2, 1, 32, causal, seed=count, spare=5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_do(dtype):
    q, k, v, g = (t.to(DEV).requires_grad_(True) for t in _inputs([7], [9], 2, 1, 32, dtype, 0))
    none, zero = torch.zeros(0, dtype=torch.long, device=DEV), torch.zeros(2, dtype=torch.long, device=DEV)
    for lengths in (none, zero):  # no sequence, or only empty ones: zeros everywhere
        out = ops.attention_pack_mode(q, k, v, lengths, causal=True)
        grads = torch.autograd.grad(out, (q, k, v), g.detach())
        for t in (out, *grads):
            assert torch.equal(t, torch.zeros_like(t))
    for qs, ks in ((q[:0], k), (q, k[:0]), (q[:0], k[:0])):  # no queries, no keys, neither
        vs = v[:ks.shape[0]]
        out = ops.attention_pack_mode(qs, ks, vs, torch.tensor([qs.shape[0]]), torch.tensor([ks.shape[0]]))
        grads = torch.autograd.grad(out, (q, k, v), g[:qs.shape[0]].detach())
        for t in (out, *grads):
            assert torch.equal(t, torch.zeros_like(t))


@pytest.mark.gpu
def test_lengths_that_overrun_are_cut():
    q, k, v, g = (t.to(DEV).requires_grad_(True) for t in _inputs([60], [60], 2, 1, 32, torch.float32, 3))
    grads = []
    for lengths in ([20, 40], [20, 4000, 7], [-3, 20, 1 << 62, 1 << 62]):
        out = ops.attention_pack_mode(q, k, v, torch.tensor(lengths, device=DEV), causal=True)
        grads.append([out, *torch.autograd.grad(out, (q, k, v), g.detach())])
    for other in grads[1:]:
        for a, b in zip(grads[0], other):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_strided_leaves_and_part_of_them():
    lengths = torch.tensor([50, 77], device=DEV)
    qkv = torch.randn((127, 8, 64), device=DEV, requires_grad=True)
    g = torch.randn((127, 4, 64), device=DEV)
    out = ops.attention_pack_mode(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], lengths, causal=True)
    (whole,) = torch.autograd.grad(out, qkv, g)
    parts = [qkv.detach()[:, s].contiguous().requires_grad_(True) for s in (slice(0, 4), slice(4, 6), slice(6, 8))]
    out = ops.attention_pack_mode(*parts, lengths, causal=True)
    got = torch.autograd.grad(out, parts, g.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(torch.cat(got, 1), whole)
    out = ops.attention_pack_mode(parts[0].detach(), parts[1], parts[2].detach(), lengths, causal=True)
    (dk,) = torch.autograd.grad(out, parts[1], g)
    assert torch.equal(dk, got[1])
    # queries, keys and values of one tensor: autograd adds the three gradients
    x = torch.randn((127, 2, 32), device=DEV, requires_grad=True)
    out = ops.attention_pack_mode(x, x, x, lengths)
    (dx,) = torch.autograd.grad(out, x, g[:, :2, :32])
    want, _ = _expect(*(x.detach().cpu(),) * 3, g[:, :2, :32].cpu(), [50, 77], [50, 77], False, 32 ** -0.5, torch.float32)
    assert (dx.cpu().double() - sum(want)).abs().max() < 1e-4


@pytest.mark.gpu
def test_neighbouring_sequences_do_not_reach():
    lengths = torch.tensor([90, 40], device=DEV)
    q, k, v, g = (t.to(DEV) for t in _inputs([90, 40], [90, 40], 2, 1, 64, torch.bfloat16, 1))

    def grads(q, k, v, g):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(ops.attention_pack_mode(*leaves, lengths), leaves, g)

    clean = grads(q, k, v, g)
    for bad in (float("inf"), float("nan")):
        q2, k2, v2, g2 = (t.clone() for t in (q, k, v, g))
        for t in (q2, k2, v2, g2):
            t[85:90] = bad
        got = grads(q2, k2, v2, g2)
        for a, b in zip(got, clean):
            assert torch.equal(a[90:], b[90:]) and torch.isnan(a[:90]).any()


@pytest.mark.gpu
def test_against_differences():
    q_lengths, s_lengths = [6, 3], [5, 7]
    q, k, v, g = (t.double() for t in _inputs(q_lengths, s_lengths, 2, 1, 16, torch.float32, 4))
    lengths = [torch.tensor(n, device=DEV) for n in (q_lengths, s_lengths)]
    leaves = [t.float().to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(ops.attention_pack_mode(*leaves, *lengths, causal=True), leaves, g.float().to(DEV))

    def f(q, k, v):
        total, at, key = 0.0, 0, 0
        for a, b in zip(q_lengths, s_lengths):
            for i in range(2):
                logits = (q[at:at + a, i] @ k[key:key + b, 0].T) * 0.25
                seen = torch.arange(b)[None] <= torch.arange(a)[:, None] + (b - a)
                none = ~seen.any(1, keepdim=True)
                p = torch.softmax(logits.masked_fill(~seen & ~none, float("-inf")), 1).masked_fill(none, 0.0)
                total = total + ((p @ v[key:key + b, 0]) * g[at:at + a, i]).sum()
            at, key = at + a, key + b
        return total

    base, h = [q, k, v], 1e-5
    for n, leaf in enumerate(base):
        for i in range(0, leaf.numel(), 5):
            step = torch.zeros(leaf.numel(), dtype=torch.float64)
            step[i] = h
            up, down = list(base), list(base)
            up[n], down[n] = leaf + step.view_as(leaf), leaf - step.view_as(leaf)
            slope = ((f(*up) - f(*down)) / (2 * h)).item()
            # 1e-10 from the differences, 32-bit steps of sums of size ~ 10 from the kernel
            assert abs(got[n].reshape(-1)[i].item() - slope) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_graph_replays(dtype):
    from vision3d_amd import ext

    lengths = torch.tensor([130, 0, 45], device=DEV)
    q, k, v, g = (t.to(DEV) for t in _inputs([175], [175], 4, 2, 64, dtype, 2))
    out, lse = torch.empty_like(q), torch.empty((175, 4), device=DEV)
    grads = [torch.empty_like(t) for t in (q, k, v)]

    def step():
        ext.attention_pack_forward(q, k, v, lengths, lengths, out, lse, 0.125, True)
        ext.attention_pack_backward(g, q, k, v, out, lse, lengths, lengths, *grads, 0.125, True)

    step()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]  # two graphs, each with a workspace of its own
    for graph in graphs:
        with torch.cuda.graph(graph):
            step()
    for n in range(4):
        q.mul_(1.1)
        step()
        torch.cuda.synchronize()
        eager = [t.clone() for t in [out] + grads]
        for graph in graphs:
            for t in [out] + grads:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(eager, [out] + grads):
                assert torch.equal(a, b), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_a_transformer_layer_over_a_pack(dtype):
    """Post-norm layer over ragged clouds: project, self-attend, add and norm, then the newest token of every cloud against
    a cache of the same keys and values -- outputs and gradients against the layer in 64 bits."""
    gen = torch.Generator().manual_seed(7)
    lengths, heads, kv, dim = [150, 1, 64, 0, 85], 4, 2, 32
    channels, n = heads * dim, sum(lengths)
    mk = lambda *s, scale=1.0: (torch.randn(s, generator=gen) * scale).to(dtype)
    x, wq = mk(n, channels), mk((heads + 2 * kv) * dim, channels, scale=channels ** -0.5)
    wo, w, b, g = mk(channels, channels, scale=channels ** -0.5), mk(channels, scale=0.3) + 1, mk(channels), mk(n, channels)
    w = w.to(dtype)

    def layer(x, wq, wo, w, b, native):
        qkv = (x @ wq.T).view(n, heads + 2 * kv, dim)
        parts = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        if native:
            att = ops.attention_pack_mode(*parts, torch.tensor(lengths, device=DEV), causal=True)
            return ops.layer_norm(att.reshape(n, channels) @ wo.T, w, b, residual=x), qkv, att
        outs, at = [], 0
        for m in lengths:
            for i in range(heads):
                q, k, v = parts[0][at:at + m, i], parts[1][at:at + m, i // 2], parts[2][at:at + m, i // 2]
                hidden = torch.ones(m, m, dtype=torch.bool).triu(1)
                outs.append(torch.softmax((q @ k.T * dim ** -0.5).masked_fill(hidden, float("-inf")), 1) @ v)
            at += m
        att = torch.cat([torch.stack(outs[i:i + heads], 1) for i in range(0, len(outs), heads)])
        t = att.reshape(n, channels) @ wo.T + x
        u = (t - t.mean(1, keepdim=True)) / (t.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
        return u * w + b, qkv, att

    base = [x, wq, wo, w, b]
    exact = [t.double().requires_grad_(True) for t in base]
    want, _, _ = layer(*exact, native=False)
    want_grads = torch.autograd.grad(want, exact, g.double())
    leaves = [t.to(DEV).requires_grad_(True) for t in base]
    got, qkv, att = layer(*leaves, native=True)
    grads = torch.autograd.grad(got, leaves, g.to(DEV))
    # a dozen roundings to the type lie between the input and any of these (projections, attention, norm and back), each
    # relative to values of the result's size: in the 2-norm at most 12 half steps; fp32 products sum up to 300 terms
    bound = 12 * _half(dtype) if dtype != torch.float32 else 300 * ULP
    for a, ref in zip([got, *grads], [want, *want_grads]):
        assert (a.detach().cpu().double() - ref.detach()).norm() <= bound * ref.norm()
    with torch.no_grad():
        cache = torch.full((len(lengths), 160, 2 * kv, dim), float("nan"), dtype=dtype, device=DEV)
        last, at = [], 0
        for i, m in enumerate(lengths):
            cache[i, :m] = qkv[at:at + m, heads:]
            at += m
            last.append(at - 1 if m else 0)
        new = ops.cached_attention(qkv[last, :heads].unsqueeze(1), cache[:, :, :kv], cache[:, :, kv:],
                                   torch.tensor(lengths, device=DEV))
        for i, m in enumerate(lengths):
            ref = att[last[i]] if m else torch.zeros_like(att[0])
            # the same products summed in another order: each side within its rounding of outputs below 4
            assert (new[i, 0].double() - ref.double()).abs().max() <= 4 * (2 * _half(dtype) + 64 * ULP) * 2


@pytest.mark.gpu
def test_refusals():
    from vision3d_amd import ext

    q, k, v, g = (t.to(DEV) for t in _inputs([10], [10], 4, 2, 16, torch.float32, 0))
    n, lse = torch.tensor([10], device=DEV), torch.zeros((10, 4), device=DEV)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    with pytest.raises(RuntimeError, match="target_grads must be contiguous"):
        ext.attention_pack_backward(g.transpose(0, 1), q, k, v, q, lse, n, n, dq, dk, dv, 0.25, False)
    with pytest.raises(RuntimeError, match="lse must have shape"):
        ext.attention_pack_backward(g, q, k, v, q, lse[:9], n, n, dq, dk, dv, 0.25, False)
    with pytest.raises(RuntimeError, match="k_grads must have shape"):
        ext.attention_pack_backward(g, q, k, v, q, lse, n, n, dq, dq, dv, 0.25, False)
    with pytest.raises(RuntimeError, match="scale must be positive"):
        ext.attention_pack_backward(g, q, k, v, q, lse, n, n, dq, dk, dv, -0.25, False)
    leaf = q.clone().requires_grad_(True)
    out = ops.attention_pack_mode(leaf, k, v, n)
    upstream = g.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(out, leaf, upstream, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):  # no second derivative
        grad.sum().backward()


def _dense(q, k, v, g, scale):
    """One sequence of one head without a mask, in 64 bits: dq, dk, dv."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    p = torch.softmax((q @ k.T) * scale, 1)
    o = p @ v
    ds = p * (g @ v.T - (g * o).sum(1, keepdim=True))
    return (ds @ k) * scale, (ds.T @ q) * scale, p.T @ g


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 192])
@pytest.mark.parametrize("size", [2.0 ** -16, 2.0 ** -10, 1.0, 2.0 ** 10])
@pytest.mark.parametrize("dtype", TYPES)
def test_small_and_large_gradients(dtype, size, dim):
    # ds is about grad . v / keys: with 2500 keys and gradients of 2^-10 it lies at 2^-18, where fp16 has a few bits left
    n = 2500
    q, k, v, g = (t[:, 0] for t in _inputs([n], [n], 1, 1, dim, dtype, seed=dim))
    g = (g.double() * size).to(dtype)
    leaves = [t.view(n, 1, dim).to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = ops.attention_pack_mode(*leaves, torch.tensor([n], device=DEV))
    got = torch.autograd.grad(out, leaves, g.view(n, 1, dim).to(DEV))
    # In the 2-norm: p or ds, delta and the gradient itself are rounded (half a step each, of separate entries) and each of
    # the 32-bit sums adds at most its 100 steps; a fourth half step for their products.  The result's own rounding is
    # at least half a subnormal step.
    bound = 4 * _half(dtype) if dtype != torch.float32 else 100 * ULP
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for name, a, ref in zip("qkv", got, _dense(q, k, v, g, dim ** -0.5)):
        off = (a[:, 0].cpu().double() - ref).norm()
        tol = bound * ref.norm() + least * ref.numel() ** 0.5
        assert off <= tol, f"d{name}: {(off / tol).item():.2f} of the tolerance"


@pytest.mark.gpu
def test_rows_of_very_different_gradients():
    # one row's ds does not take the others' bits: each row's dq, and every dk, as if it were alone
    n, dim = 300, 64
    q, k, v, g = (t[:, 0] for t in _inputs([n], [n], 1, 1, dim, torch.float16, seed=1))
    g = (g.double() * 2.0 ** torch.linspace(-20, 10, n)[torch.randperm(n, generator=torch.Generator().manual_seed(0))][:, None]).half()
    g[7], g[200] = 0, 0  # and rows without any
    leaves = [t.view(n, 1, dim).to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(ops.attention_pack_mode(*leaves, torch.tensor([n], device=DEV)), leaves, g.view(n, 1, dim).to(DEV))
    want = _dense(q, k, v, g, dim ** -0.5)
    for a, ref in zip(got, want):
        off = (a[:, 0].cpu().double() - ref).norm(dim=1)
        assert (off <= 4 * 2.0 ** -11 * ref.norm(dim=1) + 2.0 ** -25 * dim ** 0.5).all()
    assert not got[0][7].any() and not got[0][200].any()


@pytest.mark.gpu
def test_products_beyond_the_type():
    # ds reaches 2^17, past fp16's largest number; the gradients do not
    n, dim = 4, 64
    q, k, v, g = (t[:, 0].double() for t in _inputs([n], [n], 1, 1, dim, torch.float16, seed=2))
    q, k, v, g = (q * 2.0 ** -6).half(), (k * 2.0 ** -6).half(), (v * 2.0 ** 5).half(), (g * 2.0 ** 10).half()
    p = torch.softmax(q.double() @ k.double().T / 8, 1)
    assert (p * (g.double() @ v.double().T)).abs().max() > 70000
    leaves = [t.view(n, 1, dim).to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(ops.attention_pack_mode(*leaves, torch.tensor([n], device=DEV)), leaves, g.view(n, 1, dim).to(DEV))
    for a, ref in zip(got, _dense(q, k, v, g, 0.125)):
        assert (a[:, 0].cpu().double() - ref).norm() <= 4 * 2.0 ** -11 * ref.norm()


@pytest.mark.gpu
def test_values_gradients_of_many_keys():
    # a hundred thousand equal keys: p = 10^-5 is a subnormal fp16 number with half its bits
    n, dim = 100001, 32
    q, g = torch.ones(1, 1, dim), torch.full((1, 1, dim), 384.0)
    k, v = torch.full((n, 1, dim), 0.25), torch.ones(n, 1, dim)
    leaves = [t.half().to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = ops.attention_pack_mode(*leaves, torch.tensor([1], device=DEV), torch.tensor([n], device=DEV))
    dv = torch.autograd.grad(out, leaves, g.half().to(DEV))[2].double()
    # p and the gradient are rounded; the log-sum of n equal terms is off by its own half step (17 of them, in the exponent)
    want = 384.0 / n
    assert (dv - want).abs().max() <= want * (2 * 2.0 ** -11 + 32 * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_thousands_of_short_sequences(dtype):
    # more than a wave's lanes squared: the table of the sequences is searched in three steps
    gen = torch.Generator().manual_seed(11)
    lengths = torch.randint(0, 4, (4500,), generator=gen).tolist()
    lengths[4000] = 150
    _check(dtype, lengths, lengths[::-1], 2, 1, 32, True, seed=5, spare=300)


@pytest.mark.gpu
def test_overrunning_lengths_of_many_sequences():
    gen = torch.Generator().manual_seed(12)
    lengths = torch.randint(0, 4, (2000,), generator=gen).tolist()
    n = sum(lengths)
    q, k, v, g = (t.to(DEV).requires_grad_(True) for t in _inputs([n], [n], 2, 1, 32, torch.float32, 3))
    lengths[-1] += 2
    bad = [-7] + lengths
    bad[-1] = 1 << 62  # cut at the end, what follows has no rows
    bad += [5] * 100 + [1 << 62]
    grads = []
    for some in (lengths[:-1] + [lengths[-1] - 2], bad):
        out = ops.attention_pack_mode(q, k, v, torch.tensor(some, device=DEV), causal=True)
        grads.append([out, *torch.autograd.grad(out, (q, k, v), g.detach())])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_only_the_gradients_that_are_wanted(dtype):
    from vision3d_amd import ext

    n = torch.tensor([130, 0, 45], device=DEV)
    q, k, v, g = (t.to(DEV) for t in _inputs([175], [175], 4, 2, 64, dtype, 2, spare=4))

    def grads(*wanted):
        leaves = [t.clone().requires_grad_(w) for t, w in zip((q, k, v), wanted)]
        out = ops.attention_pack_mode(*leaves, n, causal=True)
        return torch.autograd.grad(out, [t for t in leaves if t.requires_grad], g)

    dq, dk, dv = grads(True, True, True)
    for wanted, want in (((1, 0, 0), [dq]), ((0, 1, 0), [dk]), ((0, 0, 1), [dv]), ((0, 1, 1), [dk, dv]), ((1, 0, 1), [dq, dv])):
        for a, b in zip(grads(*map(bool, wanted)), want):
            assert torch.equal(a, b)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    ext.attention_pack_forward(q, k, v, n, n, out, lse, 0.125, True)
    a, b = torch.empty_like(q), [torch.empty_like(k), torch.empty_like(v)]
    ext.attention_pack_backward(g, q, k, v, out, lse, n, n, None, None, None, 0.125, True)
    ext.attention_pack_backward(g, q, k, v, out, lse, n, n, a, None, None, 0.125, True)
    ext.attention_pack_backward(g, q, k, v, out, lse, n, n, None, *b, 0.125, True)
    both = [torch.empty_like(t) for t in (q, k, v)]
    ext.attention_pack_backward(g, q, k, v, out, lse, n, n, *both, 0.125, True)
    for x, y in zip([a, *b], both):
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="come together"):
        ext.attention_pack_backward(g, q, k, v, out, lse, n, n, a, b[0], None, 0.125, True)


@pytest.mark.gpu
def test_frozen_keys_and_values_save_their_kernel():
    n = torch.tensor([8192], device=DEV)
    q, k, v = (torch.randn((8192, 8, 64), device=DEV).to(torch.bfloat16) for _ in range(3))

    def least(*wanted):
        leaves = [t.clone().requires_grad_(w) for t, w in zip((q, k, v), wanted)]
        out, wanted = ops.attention_pack_mode(*leaves, n), [t for t in leaves if t.requires_grad]
        times = []
        for _ in range(6):
            marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            marks[0].record()
            torch.autograd.grad(out, wanted, q, retain_graph=True)
            marks[1].record()
            torch.cuda.synchronize()
            times.append(marks[0].elapsed_time(marks[1]))
        return min(times)

    whole = least(True, True, True)  # dq takes two fifths of it
    assert least(True, False, False) < 0.75 * whole and least(False, True, True) < 0.9 * whole
