"""ops.attention_pack_mode and ops.cached_attention against the definition in 64 bits: types, head sizes, grouped heads,
ragged packs (empty sequences, sequences without keys, rows behind the last one), strides, masked infinities, refusals."""
import pytest
import torch

from vision3d_amd import ops

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _one(q, k, v, causal, scale):
    """One sequence in 64 bits: (T,H,D), (S,KV,D) -> out, its bound sum_j p |v|, the largest error of a score."""
    t, h, d = q.shape
    s, kv, _ = k.shape
    group = h // kv
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    worst = torch.zeros(t, h, 1, dtype=torch.float64)
    lse = torch.full((t, h), float("-inf"), dtype=torch.float64)
    for i in range(h):
        kk, vv = k[:, i // group], v[:, i // group]
        for row in range(t):
            n = min(s, max(0, row + s - t + 1)) if causal else s
            if n == 0:
                continue
            logits = (kk[:n] @ q[row, i]) * scale
            p = torch.softmax(logits, 0)
            out[row, i] = p @ vv[:n]
            size[row, i] = p @ vv[:n].abs()
            lse[row, i] = torch.logsumexp(logits, 0)
            worst[row, i] = (kk[:n].abs() @ q[row, i].abs()).max() * scale
    return out, size, worst, lse


def _tolerance(dtype, out, size, worst, d):
    """The output's own rounding; the probabilities' rounding before they meet the values (16-bit types); a score is a sum
    of d products in 32 bits, off by at most d + 4 half steps of sum |q| |k| (exp2's argument included), which moves its
    probability and the sum of them by that much; 64 steps for the exponentials and the sums over keys."""
    scores = (d + 4) * 2.0 ** -24 * worst
    p = _half(dtype) if dtype != torch.float32 else 0.0
    return _half(dtype) * out.abs() + size * (p + 2 * scores + 64 * 2.0 ** -24) + 2.0 ** -24


def _pack(q_lengths, s_lengths, heads, kv, dim, dtype, seed=0, spare=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda n, h: (torch.randn((n, h, dim), generator=gen) * spread).to(dtype)
    return (mk(sum(q_lengths) + spare, heads), mk(sum(s_lengths) + spare, kv), mk(sum(s_lengths) + spare, kv))


def _expect(q, k, v, q_lengths, s_lengths, causal, scale):
    outs, sizes, worsts, at, key = [], [], [], 0, 0
    for a, b in zip(q_lengths, s_lengths):
        o, s, w, _ = _one(q[at:at + a].double(), k[key:key + b].double(), v[key:key + b].double(), causal, scale)
        outs.append(o), sizes.append(s), worsts.append(w)
        at, key = at + a, key + b
    return torch.cat(outs), torch.cat(sizes), torch.cat(worsts)


def _check(dtype, q_lengths, s_lengths, heads, kv, dim, causal, seed=0, spare=0, scale=None, spread=1.0):
    q, k, v = _pack(q_lengths, s_lengths, heads, kv, dim, dtype, seed, spare, spread)
    out = ops.attention_pack_mode(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(q_lengths).to(DEV),
                                  torch.tensor(s_lengths).to(DEV), scale=scale, causal=causal).cpu()
    n = sum(q_lengths)
    want, size, worst = _expect(q, k, v, q_lengths, s_lengths, causal, dim ** -0.5 if scale is None else scale)
    assert out.dtype == dtype and out.shape == q.shape
    assert torch.equal(out[n:], torch.zeros_like(out[n:]))
    off = (out[:n].double() - want).abs()
    tol = _tolerance(dtype, want, size, worst, dim)
    assert (off <= tol).all(), f"{(off / tol).max().item():.2f} of the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [8, 32, 33, 40, 64, 80, 96, 100, 128, 192, 200, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_head_sizes(dtype, dim, causal):
    _check(dtype, [70, 1, 0, 33, 5], [70, 1, 0, 33, 5], 2, 1, dim, causal, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (6, 3), (8, 1), (14, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_heads_and_cross_lengths(dtype, heads, kv, causal):
    # more keys than queries, fewer (the first queries see nothing), none, no queries, one of each
    _check(dtype, [37, 90, 11, 0, 1, 129], [64, 31, 0, 40, 1, 65], heads, kv, 64, causal, seed=heads, spare=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_tile_borders(dtype):
    for n in (1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 257):
        _check(dtype, [n], [n], 1, 1, 64, True, seed=n)
        _check(dtype, [3], [n], 2, 1, 64, False, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows_many_keys(dtype):
    # the keys are divided over workgroups and joined
    _check(dtype, [1], [1500], 1, 1, 128, True)
    _check(dtype, [1, 1, 2], [900, 3, 1300], 4, 2, 64, True)
    _check(dtype, [40], [1100], 2, 2, 80, False)


@pytest.mark.gpu
def test_many_short_sequences():
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 9, (5000,), generator=gen).tolist()  # more sequences than a wave looks up at once
    _check(torch.float32, lengths, lengths, 1, 1, 16, True)
    lengths = torch.randint(0, 40, (130,), generator=gen).tolist()
    _check(torch.bfloat16, lengths, lengths[::-1], 2, 1, 32, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores_and_scale(dtype):
    # scores of some hundreds: the sums live on the running maximum
    _check(dtype, [70, 20], [140, 20], 2, 1, 64, True, scale=1.0, spread=3.0)
    _check(dtype, [70, 20], [140, 20], 2, 1, 64, False, scale=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    lengths = torch.tensor([50, 77], device=DEV)
    for dim in (40, 64):
        gen = torch.Generator().manual_seed(dim)
        qkv = torch.randn((127, 8, dim + 3), generator=gen).to(dtype).to(DEV)
        q, k, v = qkv[:, :4, 1:dim + 1], qkv[:, 4:6, 2:dim + 2], qkv[:, 6:, 3:]  # views at odd elements
        got = ops.attention_pack_mode(q, k, v, lengths, causal=True)
        assert torch.equal(got, ops.attention_pack_mode(q.contiguous(), k.contiguous(), v.contiguous(), lengths, causal=True))
        flip = lambda t: t.transpose(0, 2).contiguous().transpose(0, 2)  # the last dimension is not contiguous
        assert torch.equal(got, ops.attention_pack_mode(flip(q), flip(k), flip(v), lengths.cpu().int(), causal=True))
        heads_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(got, ops.attention_pack_mode(heads_first(q), heads_first(k), heads_first(v), lengths, causal=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_what_is_not_seen_does_not_reach(dtype, bad):
    q, k, v = (t.to(DEV) for t in _pack([90, 40], [90, 40], 2, 1, 64, dtype))
    lengths = torch.tensor([90, 40], device=DEV)
    clean = ops.attention_pack_mode(q, k, v, lengths, causal=True)
    k2, v2 = k.clone(), v.clone()
    k2[70], v2[70] = bad, bad  # seen by queries 70 ... 89 of the first sequence only
    got = ops.attention_pack_mode(q, k2, v2, lengths, causal=True)
    assert torch.equal(got[:70], clean[:70]) and torch.equal(got[90:], clean[90:])
    assert not torch.isfinite(got[70:90]).all(dim=2).any()
    v2 = v.clone()
    v2[70, 0, 5] = bad  # a value alone spoils its own column only
    got = ops.attention_pack_mode(q, k, v2, lengths, causal=True)
    assert torch.equal(got[:70], clean[:70]) and torch.equal(got[90:], clean[90:])
    assert not torch.isfinite(got[70:90, :, 5]).any()
    others = [c for c in range(64) if c != 5]
    off = (got[70:90][:, :, others].double() - clean[70:90][:, :, others].double()).abs()
    assert (off <= 4 * _half(dtype) * (1 + clean[70:90][:, :, others].double().abs())).all()
    # a query's infinity or NaN stays with the query; without a mask the next sequence is still not reached
    q2 = q.clone()
    q2[11] = bad
    got = ops.attention_pack_mode(q2, k, v, lengths, causal=True)
    keep = [i for i in range(130) if i != 11]
    assert torch.equal(got[keep], clean[keep])
    v2 = v.clone()
    v2[89] = bad
    clean = ops.attention_pack_mode(q, k, v, lengths)
    assert torch.equal(ops.attention_pack_mode(q, k, v2, lengths)[90:], clean[90:])


@pytest.mark.gpu
def test_lengths_that_do_not_fit():
    q, k, v = (t.to(DEV) for t in _pack([60], [60], 1, 1, 32, torch.float32))
    want = ops.attention_pack_mode(q, k, v, torch.tensor([20, 40], device=DEV))
    got = ops.attention_pack_mode(q, k, v, torch.tensor([20, 4000, 7], device=DEV))  # cut at the total
    assert torch.equal(got, want)
    got = ops.attention_pack_mode(q, k, v, torch.tensor([-5, 20, 40, -(1 << 62)], device=DEV))
    assert torch.equal(got, want)
    got = ops.attention_pack_mode(q, k, v, torch.tensor([20, 1 << 62, 1 << 62], device=DEV))
    assert torch.equal(got, want)
    none = torch.zeros(0, dtype=torch.long, device=DEV)
    assert torch.equal(ops.attention_pack_mode(q, k, v, none), torch.zeros_like(q))
    assert ops.attention_pack_mode(q[:0], k, v, torch.tensor([0], device=DEV), torch.tensor([60], device=DEV)).shape == (0, 1, 32)
    got = ops.attention_pack_mode(q, k[:0], v[:0], torch.tensor([60], device=DEV), torch.tensor([0], device=DEV))
    assert torch.equal(got, torch.zeros_like(q))


def _check_cache(dtype, lengths, tokens, capacity, heads, kv, dim, seed=0):
    gen = torch.Generator().manual_seed(seed)
    b = len(lengths)
    q = torch.randn((b, tokens, heads, dim), generator=gen).to(dtype)
    k = torch.randn((b, capacity, kv, dim), generator=gen).to(dtype)
    v = torch.randn((b, capacity, kv, dim), generator=gen).to(dtype)
    for i, n in enumerate(lengths):  # rows past a length may hold anything
        k[i, max(n, 0):], v[i, max(n, 0):] = float("nan"), float("inf")
    got = ops.cached_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(lengths).to(DEV)).cpu()
    for i, n in enumerate(lengths):
        n = min(max(n, 0), capacity)
        want, size, worst, _ = _one(q[i].double(), k[i, :n].double(), v[i, :n].double(), True, dim ** -0.5)
        off = (got[i].double() - want).abs()
        tol = _tolerance(dtype, want, size, worst, dim)
        assert (off <= tol).all(), f"{(off / tol).max().item():.2f} of the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (8, 2, 128), (6, 3, 80), (40, 1, 33), (4, 4, 256), (2, 1, 32), (4, 2, 192)])
def test_cache(dtype, heads, kv, dim):
    _check_cache(dtype, [300, 1, 0, 129, 77, 512], 1, 512, heads, kv, dim, seed=dim)
    _check_cache(dtype, [70, 3, 600], 5, 600, heads, kv, dim, seed=dim + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_cache_lengths(dtype):
    _check_cache(dtype, [2500, 2499, 2049, 64], 1, 2500, 4, 1, 128)
    _check_cache(dtype, [9], 3, 9, 2, 2, 64)
    _check_cache(dtype, [2], 7, 40, 2, 1, 64)     # more new tokens than rows: the first see nothing
    _check_cache(dtype, [-3, 50], 1, 40, 2, 1, 64)  # cut to [0, capacity]
    _check_cache(dtype, [31 * (i % 5) + i for i in range(70)], 1, 200, 2, 1, 64)


@pytest.mark.gpu
def test_cache_equals_the_packs_last_rows():
    lengths = [140, 33, 260]
    q, k, v = (t.to(DEV) for t in _pack(lengths, lengths, 8, 2, 128, torch.bfloat16))
    whole = ops.attention_pack_mode(q, k, v, torch.tensor(lengths, device=DEV), causal=True)
    cap = 300
    kc, vc = (torch.full((3, cap, 2, 128), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    at = 0
    for i, n in enumerate(lengths):
        kc[i, :n], vc[i, :n] = k[at:at + n], v[at:at + n]
        at += n
    ends = torch.tensor(lengths).cumsum(0) - 1
    last = ops.cached_attention(q[ends.to(DEV)].unsqueeze(1), kc, vc, torch.tensor(lengths, device=DEV))
    off = (last[:, 0].double() - whole[ends.to(DEV)].double()).abs()
    # two sums of the same products in another order: each is within its rounding of the exact value
    assert off.max() <= 4 * _half(torch.bfloat16) * 2


@pytest.mark.gpu
def test_cache_beyond_32_bit_offsets():
    # 2^31 elements of keys and as many of values in one cache: only the last rows carry weight
    capacity, kv, dim = (1 << 21) + 70, 8, 128
    k = torch.zeros((1, capacity, kv, dim), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    gen = torch.Generator().manual_seed(0)
    n = capacity - 5
    tail = torch.randn((3, kv, dim), generator=gen).to(torch.bfloat16)
    k[0, n - 3:n], v[0, n - 3:n] = 2.0, tail.to(DEV)
    k[0, n:], v[0, n:] = float("nan"), float("nan")
    q = torch.full((1, 1, 16, dim), 2.0, dtype=torch.bfloat16, device=DEV)
    got = ops.cached_attention(q, k, v, torch.tensor([n], device=DEV))[0, 0].double().cpu()
    # the three rows' scores are 4 * 128 / sqrt(128) = 45.25, all others 0: their weight is 2^21 e^-45 of the whole
    want = tail.double().mean(0).repeat_interleave(2, 0)
    assert (got - want).abs().max() <= 2.0 ** -8 * 4 + 1e-6
    pack = ops.attention_pack_mode(q[0], k[0, :n], v[0, :n], torch.tensor([1], device=DEV), torch.tensor([n], device=DEV))
    assert (pack[0].double().cpu() - want).abs().max() <= 2.0 ** -8 * 4 + 1e-6


@pytest.mark.gpu
def test_shared_and_far_rows():
    # a key row for all (stride 0), rows far apart (a stride beyond what a tile's offsets hold is copied), overlapping rows
    q, k, v = (t.to(DEV) for t in _pack([50], [50], 2, 2, 64, torch.float16))
    n = torch.tensor([50], device=DEV)
    shared = k[:1].expand(50, 2, 64)
    assert torch.equal(ops.attention_pack_mode(q, shared, v, n), ops.attention_pack_mode(q, shared.contiguous(), v, n))
    want = ops.attention_pack_mode(q, k, v, n, causal=True)
    for stride in (1 << 21, 1 << 22, 1 << 23):  # elements between rows
        far = torch.empty(50 * stride, dtype=torch.float16, device=DEV).view(50, stride)[:, :128].view(50, 2, 64)
        far.copy_(k)
        assert torch.equal(ops.attention_pack_mode(q, far, v, n, causal=True), want)
        far.copy_(q)
        assert torch.equal(ops.attention_pack_mode(far, k, v, n, causal=True), want)
        del far
    # one row, one head: their strides mean nothing
    one = torch.randn(1, 64, device=DEV).half()
    odd = [one.as_strided((1, 1, 64), st) for st in ((1, 1, 1), (3, 1 << 40, 1), (1 << 40, 5, 1), (0, 0, 1))]
    for t in odd:
        got = ops.attention_pack_mode(t, t, t, torch.tensor([1], device=DEV))
        assert torch.equal(got.view(1, 64), one)
        got = ops.cached_attention(t[None], t[None], t[None], torch.tensor([1], device=DEV))
        assert torch.equal(got.view(1, 64), one)
        leaf = t.detach().requires_grad_(True)
        out = ops.attention_pack_mode(leaf, t, t, torch.tensor([1], device=DEV))
        # one key: its weight is 1 whatever q is, so ds = dp - delta is 0 but for the two sums of 64 products each, taken in
        # different orders: off by at most 64 + 4 half steps of sum |v| apiece; dq = scale ds k, then rounded (half a step,
        # subnormal 2^-25)
        grad = torch.autograd.grad(out, leaf, torch.ones_like(out))[0].double()
        ds = 2 * 68 * 2.0 ** -24 * one.double().abs().sum()
        assert (grad.abs() <= 0.125 * ds * one.double().abs().max() * (1 + 2.0 ** -11) + 2.0 ** -25).all()
    over = torch.randn(50 * 32 + 128, device=DEV).to(torch.float16).as_strided((50, 2, 64), (32, 64, 1))
    assert torch.equal(ops.attention_pack_mode(q, over, over, n), ops.attention_pack_mode(q, over.contiguous(), over.contiguous(), n))


@pytest.mark.gpu
def test_other_stream_and_graph_replays():
    from vision3d_amd import ext

    lengths = torch.tensor([1, 1, 1], device=DEV)
    keys = torch.tensor([700, 0, 1800], device=DEV)
    q, k, v = (t.to(DEV) for t in _pack([3], [2500], 4, 2, 64, torch.float16))
    want = ops.attention_pack_mode(q, k, v, lengths, keys)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.attention_pack_mode(q, k, v, lengths, keys)
    side.synchronize()
    assert torch.equal(got, want)
    out, cached = torch.empty_like(q), torch.empty_like(q).view(3, 1, 4, 64)
    cache_k, cache_v = k.view(-1)[:3 * 800 * 128].view(3, 800, 2, 64), v.view(-1)[:3 * 800 * 128].view(3, 800, 2, 64)

    def step():
        ext.attention_pack_forward(q, k, v, lengths, keys, out, None, 0.125, False)
        ext.cached_attention(q.view(3, 1, 4, 64), cache_k, cache_v, keys, cached, 0.125)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(4):
        q.mul_(1.25)
        keys[0] -= 100  # the lengths are device data: a replay follows them
        step()
        torch.cuda.synchronize()
        eager = [out.clone(), cached.clone()]
        out.fill_(float("nan")), cached.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(cached, eager[1]), n


@pytest.mark.gpu
def test_refusals():
    q, k, v = (t.to(DEV) for t in _pack([10], [10], 4, 2, 16, torch.float32))
    n = torch.tensor([10], device=DEV)
    with pytest.raises(RuntimeError, match="multiple of the key heads"):
        ops.attention_pack_mode(q[:, :3], k, v, n)
    with pytest.raises(RuntimeError, match="expected scalar type"):
        ops.attention_pack_mode(q, k.half(), v.half(), n)
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        ops.attention_pack_mode(q.double(), k.double(), v.double(), n)
    with pytest.raises(RuntimeError, match="expected q_feats"):
        ops.attention_pack_mode(q, k, v[:5], n)
    with pytest.raises(RuntimeError, match="expected q_feats"):
        ops.attention_pack_mode(q[:, :, :8], k, v, n)
    with pytest.raises(RuntimeError, match="s_lengths must have shape"):
        ops.attention_pack_mode(q, k, v, n, torch.tensor([5, 5], device=DEV))
    with pytest.raises(RuntimeError, match="must have 3 dimensions"):
        ops.attention_pack_mode(q[0], k, v, n)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="scale must be positive"):
            ops.attention_pack_mode(q, k, v, n, scale=scale)
    with pytest.raises(RuntimeError, match="head size 257"):
        big = torch.zeros((4, 1, 257), device=DEV)
        ops.attention_pack_mode(big, big, big, torch.tensor([4], device=DEV))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.cached_attention(q.view(1, 10, 4, 16).requires_grad_(True), k.view(1, 10, 2, 16), v.view(1, 10, 2, 16), n)
    q = q.detach()
    with pytest.raises(RuntimeError, match="expected q_feats"):
        ops.cached_attention(q.view(2, 5, 4, 16), k.view(1, 10, 2, 16), v.view(1, 10, 2, 16), torch.tensor([5, 5], device=DEV))
    with pytest.raises(RuntimeError, match="lengths must have shape"):
        ops.cached_attention(q.view(1, 10, 4, 16), k.view(1, 10, 2, 16), v.view(1, 10, 2, 16), torch.tensor([5, 5], device=DEV))


def test_refusals_without_a_gpu():
    from vision3d_amd import _lib

    t = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="attention_pack_mode: CUDA tensors required"):
        ops.attention_pack_mode(t, t, t, torch.tensor([4]))
    with pytest.raises(RuntimeError, match="cached_attention: CUDA tensors required"):
        ops.cached_attention(t[None], t[None], t[None], torch.tensor([4]))
    lib = _lib.lib()
    none = [None] * 8

    def pack(dtype=1, b=1, nq=4, ns=4, h=2, kv=1, d=8, scale=1.0):
        return lib.v3d_attention_pack_fwd(*none, dtype, b, nq, ns, h, kv, d, None, scale, 0, None, 0, 0, None)

    assert pack(dtype=5) == -1 and pack(h=3, kv=2) == -1 and pack(d=0) == -1 and pack(b=-1) == -1
    assert pack(scale=0.0) == -1 and pack(scale=float("nan")) == -1 and pack() == -1  # null pointers
    assert pack(d=7) == -1 and pack(dtype=0, d=3) == -1  # less than 16 bytes
    assert pack(d=257) == -4 and pack(nq=1 << 30) == -4 and pack(ns=(1 << 30) + 1) == -4
    assert pack(nq=0) == 0
    # the workspace is asked for only where the keys are divided
    assert lib.v3d_attention_pack_workspace_bytes(4, 100000, 100000, 8, 8, 64) == 0
    assert lib.v3d_attention_pack_workspace_bytes(1, 1, 100000, 8, 8, 64) > 0
    assert lib.v3d_cached_attention_workspace_bytes(1, 1, 64, 8, 8, 64) == 0
    assert lib.v3d_cached_attention_workspace_bytes(1, 1, 100000, 8, 8, 64) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("count", [32768, 1 << 20])
@pytest.mark.parametrize("dtype", TYPES)
def test_many_weak_keys_behind_a_strong_one(dtype, count):
    # each weak key's probability is 2^-25.2 of the strong one's, in fp16 at the edge of nothing; together they are the output
    k = torch.zeros(1, count, 1, 64, dtype=dtype, device=DEV)
    v = torch.ones_like(k)
    k[0, 0], v[0, 0] = 2.1875, 0.0
    q = torch.ones(1, 1, 1, 64, dtype=dtype, device=DEV)
    strong = torch.tensor(8 * 2.1875, dtype=torch.float64).exp().item()
    want = (count - 1) / (count - 1 + strong)
    cached = ops.cached_attention(q, k, v, torch.tensor([count], device=DEV))
    one, n = torch.tensor([1], device=DEV), torch.tensor([count], device=DEV)
    pack = ops.attention_pack_mode(q[0], k[0], v[0], one, n)
    several = ops.attention_pack_mode(q[0].expand(300, 1, 64).contiguous(), k[0], v[0], one * 300, n)
    # the probability and the output are rounded to the type (equal values: all in the same direction); scores are exact,
    # exp2's argument off by a half step of 25, the 32-bit sums by a step per 64 keys of a lane and per joined part
    tol = want * (2 * _half(dtype) + (26 + count / 64 + 128) * 2.0 ** -24)
    for out in (cached, pack, several):
        assert (out.double() - want).abs().max() <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 192])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e9, 1e15])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_beyond_the_exponents(dtype, size, dim):
    # scores of up to 1e30: the row's maximum takes all, whatever 32-bit numbers can no longer tell apart
    if dtype == torch.float16:
        size = min(size, 2e4)
    n = 1500
    gen = torch.Generator().manual_seed(dim)
    sign = torch.randint(0, 2, (n, 1, dim), generator=gen) * 2.0 - 1
    k = (sign * size).to(dtype)
    assert torch.unique(sign, dim=0).shape[0] == n
    k = k.to(DEV)  # distinct signs: a key's own product is dim size^2, any other's at least 2 size^2 less
    v = torch.randn((n, 1, dim), generator=gen).to(dtype).to(DEV)
    pick = torch.randint(0, n, (400,), generator=gen).to(DEV)
    one, few, many = (torch.tensor([m], device=DEV) for m in (1, 40, 400))
    keys = torch.tensor([n], device=DEV)
    for q, lengths in ((k[pick], many), (k[pick[:40]], few), (k[pick[:1]], one)):
        assert torch.equal(ops.attention_pack_mode(q, k, v, lengths, keys), v[pick[:q.shape[0]]])
    got = ops.cached_attention(k[pick[:3]].unsqueeze(1), k.expand(3, n, 1, dim).reshape(3, n, 1, dim),
                               v.expand(3, n, 1, dim).reshape(3, n, 1, dim), keys.expand(3).contiguous())
    assert torch.equal(got[:, 0], v[pick[:3]])
    # all of them equally far below zero: the plain mean
    least = ops.attention_pack_mode(-k[:1].expand(40, 1, dim).contiguous(), k[:1].expand(n, 1, dim), v, few, keys)
    want = v.double().mean(0)
    size = v.double().abs().mean(0)
    assert ((least.double() - want).abs() <= 2 * _half(dtype) * size + 200 * 2.0 ** -24 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_newest_token_of_a_long_projection(dtype):
    # one token a sequence, the sequences 5.7 million elements apart: more than a tile's offsets, but no tile spans two of them
    x = torch.randn((3, 1400, 32, 128), device=DEV).to(dtype)
    k, v = (torch.randn((3, 100, 8, 128), device=DEV).to(dtype) for _ in range(2))
    n = torch.tensor([100, 30, 77], device=DEV)
    want = ops.cached_attention(x[:, -1:].contiguous(), k, v, n)
    assert torch.equal(ops.cached_attention(x[:, -1:], k, v, n), want)
    assert torch.equal(ops.cached_attention(x[:, -1:].transpose(1, 2).contiguous().transpose(1, 2), k, v, n), want)
    five = ops.cached_attention(x[:, -5:].contiguous(), k, v, n)  # several tokens: copied by the op
    assert torch.equal(ops.cached_attention(x[:, -5:], k, v, n), five)


@pytest.mark.gpu
def test_heads_first_layouts_up_to_the_tiles_offsets():
    # queries of 8 heads on one key head, 38 million elements from head to head: within a tile's offsets (7 of them), taken as
    # they are; 80 million: beyond, copied
    n = torch.tensor([300000], device=DEV)
    k = torch.randn((64, 1, 128), device=DEV).to(torch.bfloat16)
    s = torch.tensor([64], device=DEV)
    for rows in (300000, 620000):
        x = torch.randn((8, rows, 128), device=DEV, dtype=torch.bfloat16)[:, :300000].transpose(0, 1)
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = ops.attention_pack_mode(x, k, k, n, s)
        copied = torch.cuda.max_memory_allocated() - before > 1.5 * got.numel() * 2
        assert copied == (rows == 620000)
        assert torch.equal(got, ops.attention_pack_mode(x.contiguous(), k, k, n, s))
        del got, x


@pytest.mark.gpu
def test_heads_first_cache_is_not_copied():
    # the distance between a cache's key heads is 64-bit: no tile spans two of them
    k = torch.randn((1, 8, 530000, 128), device=DEV, dtype=torch.bfloat16).transpose(1, 2)
    q = torch.randn((1, 1, 32, 128), device=DEV, dtype=torch.bfloat16)
    n = torch.tensor([200], device=DEV)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = ops.cached_attention(q, k, k, n)
    assert torch.cuda.max_memory_allocated() - before < 1 << 26
    near = k[:, :200].contiguous()
    want = ops.attention_pack_mode(q[0], near[0], near[0], torch.tensor([1], device=DEV), n)
    # the same products summed in another order: each side within its rounding of outputs below 4
    assert (got[0].double() - want.double()).abs().max() <= 4 * 4 * _half(torch.bfloat16)


@pytest.mark.gpu
def test_cost_of_many_sequences():
    # sixteen times as many short sequences cost about sixteen times as much, forward and backward (not the square of it)
    def least(count):
        lengths = torch.full((count,), 4, device=DEV)
        leaves = [torch.randn((4 * count, 8, 32), device=DEV).to(torch.bfloat16).requires_grad_(True) for _ in range(3)]
        times = [[], []]
        for _ in range(6):
            marks = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
            marks[0].record()
            out = ops.attention_pack_mode(*leaves, lengths)
            marks[1].record()
            torch.autograd.grad(out, leaves, leaves[0].detach())
            marks[2].record()
            torch.cuda.synchronize()
            for i in range(2):
                times[i].append(marks[i].elapsed_time(marks[i + 1]))
        return [min(t) for t in times]

    few, many = least(2048), least(32768)
    assert many[0] < 48 * few[0] and many[1] < 48 * few[1]


def test_launches_beyond_the_limit_are_refused():
    # three million sequences of four tokens, eight key heads: more workgroups than a launch holds; nothing is read before
    import ctypes

    from vision3d_amd import _lib

    lib, at = _lib.lib(), ctypes.c_void_p(1 << 20)
    strides, cache = (ctypes.c_int64 * 6)(64, 8, 64, 8, 64, 8), (ctypes.c_int64 * 8)(64, 8, 64, 64, 8, 64, 64, 8)
    count = 3_000_000

    def pack(count, heads):
        return lib.v3d_attention_pack_fwd(at, at, at, at, at, at, None, None, 1, count, 4 * count, 4 * count, heads, heads, 8,
                                          strides, 1.0, 0, at, 1 << 40, 0, None)

    assert pack(count, 8) == -4 and pack(1 << 24, 1) == -4
    assert lib.v3d_attention_pack_bwd(at, at, at, at, at, None, at, at, at, at, at, at, 1, count, 4 * count, 4 * count, 8, 8, 8,
                                      strides, 1.0, 0, at, 1 << 40, 0, None) == -4
    assert lib.v3d_attention_pack_bwd(at, at, at, at, at, None, at, at, at, at, at, at, 1, 10, 40, 1 << 30, 8, 8, 8,
                                      strides, 1.0, 0, at, 1 << 40, 0, None) == -4
    assert lib.v3d_cached_attention(at, at, at, at, at, 1, count, 1, 1, 8, 8, 8, cache, 1.0, at, 1 << 40, 0, None) == -4


@pytest.mark.gpu
def test_forward_mode_is_refused():
    # no forward-mode derivatives: a tangent is refused, not dropped; what carries none goes through
    import torch.autograd.forward_ad as fw

    x, w = torch.randn((10, 2, 16), device=DEV), torch.ones(16, device=DEV)
    n = torch.tensor([10], device=DEV)
    calls = [lambda t: ops.attention_pack_mode(t, x, x, n), lambda t: ops.attention_pack_mode(x, x, t, n),
             lambda t: ops.layer_norm(t), lambda t: ops.layer_norm(x, w, residual=t), lambda t: ops.layer_norm(x, t[0, 0])]
    cached = lambda t: ops.cached_attention(x[None], t[None], x[None], n)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in calls:
                    with pytest.raises(NotImplementedError):
                        call(dual)
                with pytest.raises(RuntimeError, match="no gradient"):
                    cached(dual)
                for call in calls + [cached]:
                    call(x)
