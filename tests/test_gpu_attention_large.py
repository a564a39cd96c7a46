"""ops.attention_pack_mode on packs large enough for the 128-row kernel and for undivided key tiles of the backward, against
the definition in 64 bits over a padded batch; every test says which kernels it reaches."""
import ctypes

import pytest
import torch

from vision3d_amd import _lib, ops

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ULP = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _plan(lengths, keys, heads, kv, dim, spare=0, dtype=torch.float32):
    """(rows of a forward tile, parts of its keys, parts of a backward key tile's rows, parts of a backward row tile's keys)."""
    out = [ctypes.c_int() for _ in range(4)]
    rc = _lib.lib().v3d_attention_pack_plan(TYPES.index(dtype), len(lengths), sum(lengths) + spare, sum(keys) + spare, heads, kv,
                                            dim, *(ctypes.byref(x) for x in out))
    assert rc == 0
    return out[0].value, out[1].value, out[3].value, out[2].value


def _rows(lengths):
    """(B, longest) row in the pack of every place of a padded batch, and which places are a sequence's own."""
    n = torch.tensor(lengths, device=DEV)
    place = torch.arange(max(max(lengths), 1), device=DEV)
    valid = place < n[:, None]
    return torch.where(valid, (n.cumsum(0) - n)[:, None] + place, 0), valid


def _padded(x, rows, valid):
    return torch.where(valid[..., None], x.double()[rows], 0.0)


def _expect(q, k, v, lengths, keys, causal, g=None):
    """Per query head over the padded batch, in 64 bits.  Forward: out, sum_j p |v|, largest sum |q| |k| of a row.  With g: the
    three gradients and the bounds of their errors."""
    (nq, heads, dim), (ns, kv, _) = q.shape, k.shape
    scale = dim ** -0.5
    q_rows, q_valid = _rows(lengths)
    s_rows, s_valid = _rows(keys)
    seen = s_valid[:, None, :] & q_valid[:, :, None]
    if causal:
        last = torch.arange(q_rows.shape[1], device=DEV) + torch.tensor(keys, device=DEV)[:, None] - torch.tensor(
            lengths, device=DEV)[:, None]
        seen = seen & (torch.arange(s_rows.shape[1], device=DEV) <= last[:, :, None])
    none = ~seen.any(2, keepdim=True)
    n_q, n_s = sum(lengths), sum(keys)
    out, size = torch.zeros(nq, heads, dim, dtype=torch.float64, device=DEV), torch.zeros(nq, heads, dim, dtype=torch.float64, device=DEV)
    worst = torch.zeros(nq, heads, 1, dtype=torch.float64, device=DEV)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (q, k, v)] if g is not None else None
    errs = [torch.zeros_like(t) for t in grads] if g is not None else None
    half, own = _half(q.dtype), (_half(q.dtype) if q.dtype != torch.float32 else ULP)
    steps = (64 + max(max(lengths), max(keys)) / 32) * ULP
    for h in range(heads):
        j = h // (heads // kv)
        qq, kk, vv = _padded(q[:, h], q_rows, q_valid), _padded(k[:, j], s_rows, s_valid), _padded(v[:, j], s_rows, s_valid)
        kt, vt = kk.transpose(1, 2).contiguous(), vv.transpose(1, 2).contiguous()
        logits = (torch.bmm(qq, kt) * scale).masked_fill(~seen, float("-inf")).masked_fill(none, 0.0)
        p = torch.softmax(logits, 2).masked_fill(~seen, 0.0)
        o, pv = torch.bmm(p, vv), torch.bmm(p, vv.abs())
        reach = (torch.bmm(qq.abs(), kt.abs()) * scale).masked_fill(~seen, 0.0).amax(2, keepdim=True)
        out[:n_q, h], size[:n_q, h], worst[:n_q, h] = o[q_valid], pv[q_valid], reach[q_valid]
        if g is None:
            continue
        gg = _padded(g[:, h], q_rows, q_valid)
        ga = gg.abs()
        delta = (gg * o).sum(2, keepdim=True)
        inner = torch.bmm(gg, vt) - delta
        ds = p * inner
        es = 2 * (dim + 4) * ULP * reach
        o_err = half * o.abs() + pv * (own + es + steps)
        delta_err = (ga * o_err).sum(2, keepdim=True) + (dim + 4) * ULP * (ga * o.abs()).sum(2, keepdim=True)
        ds_err = p * (inner.abs() * (own + es + steps) + (dim + 4) * ULP * torch.bmm(ga, vt.abs()) + delta_err)
        p_err = p * (own + es + steps)
        turn = lambda t: t.transpose(1, 2).contiguous()
        grads[0][:n_q, h] = (torch.bmm(ds, kk) * scale)[q_valid]
        errs[0][:n_q, h] = (scale * torch.bmm(ds_err, kk.abs()) + steps * scale * torch.bmm(ds.abs(), kk.abs()))[q_valid]
        grads[1][:n_s, j] += (torch.bmm(turn(ds), qq) * scale)[s_valid]
        errs[1][:n_s, j] += (scale * torch.bmm(turn(ds_err), qq.abs()) + steps * scale * torch.bmm(turn(ds.abs()), qq.abs()))[s_valid]
        grads[2][:n_s, j] += torch.bmm(turn(p), gg)[s_valid]
        errs[2][:n_s, j] += (torch.bmm(turn(p_err), ga) + steps * torch.bmm(turn(p), ga))[s_valid]
    return (out, size, worst) if g is None else (grads, errs)


def _inputs(lengths, keys, heads, kv, dim, dtype, seed, spare=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda n, h: torch.randn((n, h, dim), generator=gen, device=DEV).to(dtype)
    nq, ns = sum(lengths) + spare, sum(keys) + spare
    return mk(nq, heads), mk(ns, kv), mk(ns, kv), mk(nq, heads)


def _tensors(*lists):
    return tuple(torch.tensor(t, device=DEV) for t in lists)


def _forward(dtype, lengths, keys, heads, kv, dim, causal, seed=0, spare=0):
    """The output's own rounding; the probabilities' rounding (16-bit types); a score is off by d + 4 half steps of
    sum |q| |k|, which moves its probability and the sum of them; 64 steps for the exponentials and the sums over keys."""
    q, k, v, _ = _inputs(lengths, keys, heads, kv, dim, dtype, seed, spare)
    got = ops.attention_pack_mode(q, k, v, *_tensors(lengths, keys), causal=causal)
    want, size, worst = _expect(q, k, v, lengths, keys, causal)
    p = _half(dtype) if dtype != torch.float32 else 0.0
    tol = _half(dtype) * want.abs() + size * (p + 2 * (dim + 4) * ULP * worst + 64 * ULP) + ULP
    off = (got.double() - want).abs()
    assert got.dtype == dtype and (off <= tol).all(), f"{(off / tol).max().item():.2f} of the tolerance"
    assert not got[sum(lengths):].any()


def _gradients(dtype, lengths, keys, heads, kv, dim, causal, seed=0, spare=0):
    q, k, v, g = _inputs(lengths, keys, heads, kv, dim, dtype, seed, spare)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = ops.attention_pack_mode(*leaves, *_tensors(lengths, keys), causal=causal)
    got = torch.autograd.grad(out, leaves, g)
    want, errs = _expect(*(t.detach() for t in (q, k, v)), lengths, keys, causal, g)
    for name, a, ref, err in zip("qkv", got, want, errs):
        off = (a.double() - ref).abs()
        tol = err + _half(dtype) * ref.abs() + ULP
        assert a.dtype == dtype and (off <= tol).all(), f"d{name}: {(off / tol).max().item():.2f} of the tolerance"
    for a, n in zip(got, (sum(lengths), sum(keys), sum(keys))):
        assert not a[n:].any()


# an empty sequence, one of one token, one without keys, more and fewer keys than queries, tile borders
LENGTHS, KEYS = [300, 1, 0, 131, 257, 400, 33, 128, 250], [64, 500, 40, 131, 0, 450, 1, 128, 300]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 80, 96, 100, 128, 160, 192, 200, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_head_sizes(dtype, dim, causal):
    assert _plan(LENGTHS, KEYS, 6, 3, dim, 77)[:2] == (128, 1)
    _forward(dtype, LENGTHS, KEYS, 6, 3, dim, causal, seed=dim, spare=77)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv", [(7, 7), (20, 2), (24, 1), (9, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_heads(dtype, heads, kv, causal):
    if heads == 24:
        lengths = [4 * n for n in LENGTHS]
        assert _plan(lengths, KEYS, heads, kv, 64)[0] == 128
        _forward(dtype, lengths, KEYS, heads, kv, 64, causal, seed=heads)
    else:
        assert _plan(LENGTHS, KEYS, heads, kv, 64)[0] == 128
        _forward(dtype, LENGTHS, KEYS, heads, kv, 64, causal, seed=heads)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_divided_keys(dtype, dim, causal):
    # two parts of 128-row tiles joined; the second part of the short sequences has no keys at all
    lengths, keys = [700, 500, 300], [2600, 1900, 40]
    assert _plan(lengths, keys, 6, 3, dim, 50)[:2] == (128, 2)
    _forward(dtype, lengths, keys, 6, 3, dim, causal, seed=dim, spare=50)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("count", [64, 65, 200, 256, 257, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_numbers_of_sequences(dtype, count, causal):
    # one to a lane (causal: numbered by work), a few to a lane, in the table
    gen = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 6400 // count, (count,), generator=gen).tolist()
    keys = torch.randint(0, 6400 // count, (count,), generator=gen).tolist()
    lengths[count // 2], keys[-1] = 300, 270
    assert _plan(lengths, keys, 16, 2, 32, 9)[0] == 128
    _forward(dtype, lengths, keys, 16, 2, 32, causal, seed=count, spare=9)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dim,keys", [(64, 0), (128, 0), (256, 0), (64, 1500), (256, 1500)])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_seen_does_not_reach(dtype, dim, keys, bad):
    lengths = [600, 400, 500]
    s = [n + keys for n in lengths]  # the last rows of the keys are the queries' own places
    assert _plan(lengths, s, 6, 3, dim)[:2] == (128, 1 if keys == 0 else 3)
    q, k, v, _ = _inputs(lengths, s, 6, 3, dim, dtype, 3)
    args = _tensors(lengths, s)
    clean = ops.attention_pack_mode(q, k, v, *args, causal=True)
    at = keys + 350  # seen by the queries 350 ... 599 of the first sequence
    rest = [i for i in range(1500) if not 350 <= i < 600]
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at] = bad, bad
    got = ops.attention_pack_mode(q, k2, v2, *args, causal=True)
    assert torch.equal(got[rest], clean[rest]) and not torch.isfinite(got[350:600]).all(dim=2).any()
    v2 = v.clone()
    v2[at, 1, 5] = bad  # spoils the column of the two heads that read it, where it is seen
    got = ops.attention_pack_mode(q, k, v2, *args, causal=True)
    assert torch.equal(got[rest], clean[rest])
    spoiled = ~torch.isfinite(got)
    assert spoiled[350:600, 2:4, 5].all() and spoiled.sum() == 250 * 2
    # the other columns: the same products, the tile's values added one by one
    off = (torch.where(spoiled, 0.0, got.double()) - torch.where(spoiled, 0.0, clean.double())).abs()
    assert (off <= 4 * _half(dtype) * (1 + clean.double().abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_that_do_not_fit_and_views(dtype, causal):
    lengths = [600, 400, 500]
    gen = torch.Generator(device=DEV).manual_seed(1)
    qkv = torch.randn((1500, 12, 83), generator=gen, device=DEV).to(dtype)
    q, k, v = qkv[:, :6, 1:81], qkv[:, 6:9, 2:82], qkv[:, 9:, 3:]  # views at odd elements
    assert _plan(lengths, lengths, 6, 3, 80)[0] == 128
    want = ops.attention_pack_mode(q.contiguous(), k.contiguous(), v.contiguous(), *_tensors(lengths), causal=causal)
    for some in (lengths, [600, 400, 1 << 62, 7], [-9, 600, 400, 500, -(1 << 62)], [600, 400, 500] + [0] * 90):
        assert _plan(lengths + [0] * (len(some) - 3), lengths, 6, 3, 80)[:2] == (128, 1)
        assert torch.equal(ops.attention_pack_mode(q, k, v, *_tensors(some), causal=causal), want)
    flip = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.attention_pack_mode(flip(q), flip(k), flip(v), *_tensors(lengths), causal=causal), want)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_undivided_key_tiles(dtype, dim, causal):
    # so many sequences that no key tile's rows are divided: dk and dv leave the kernel in the type
    gen = torch.Generator().manual_seed(dim)
    lengths, keys = torch.randint(0, 9, (600,), generator=gen).tolist(), torch.randint(0, 9, (600,), generator=gen).tolist()
    lengths[7], keys[7], keys[500] = 150, 200, 90
    assert _plan(lengths, keys, 4, 2, dim, 200)[2] == 1
    _gradients(dtype, lengths, keys, 4, 2, dim, causal, seed=dim, spare=200)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_long_packs(dtype, dim, causal):
    # 128-row tiles forward, whole key tiles of eight heads backward, up to 64 sequences (causal: numbered by work)
    lengths = [700, 1, 0, 900, 257, 400, 33, 128, 810, 1300, 640, 1000, 1024, 901, 100]
    keys = lengths[::-1]
    assert _plan(lengths, keys, 8, 8, dim) == (128, 1, 1, 1)
    _gradients(dtype, lengths, keys, 8, 8, dim, causal, seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_divided_row_tiles(dtype, dim, causal):
    # few queries, many keys: the keys of a row tile are divided; the short sequence's later parts have none, the last has no keys
    lengths, keys = [140, 70, 1, 0, 200], [2900, 1500, 700, 40, 0]
    assert _plan(lengths, keys, 4, 2, dim, 30, dtype)[3] == (8 if dtype == torch.float32 else 2)
    _gradients(dtype, lengths, keys, 4, 2, dim, causal, seed=dim, spare=30)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_replays_of_divided_tiles(dtype):
    # every kernel of a training step under capture: the table, the norms, both divided gradients and their joins
    from vision3d_amd import ext

    lengths, keys = [2] * 260, [5] * 259 + [160000 // 260 * 260 - 5 * 259]
    q, k, v, g = _inputs(lengths, keys, 2, 1, 64, dtype, 4)
    assert _plan(lengths, keys, 2, 1, 64, 0, dtype)[2] == 1
    few = [60, 50], [1500, 1400]
    q2, k2, v2, g2 = _inputs(*few, 2, 1, 64, dtype, 5)
    plan = _plan(*few, 2, 1, 64, 0, dtype)
    assert plan[2] > 1 and plan[3] > 1
    args, args2 = _tensors(lengths, keys), _tensors(*few)
    outs = [[torch.empty_like(t) for t in (a, a, b, c)] + [torch.empty(a.shape[:2], device=DEV)] for a, b, c in ((q, k, v), (q2, k2, v2))]

    def step():
        for (a, b, c, d, n), (out, dq, dk, dv, lse) in zip(((q, k, v, g, args), (q2, k2, v2, g2, args2)), outs):
            ext.attention_pack_forward(a, b, c, *n, out, lse, 0.125, True)
            ext.attention_pack_backward(d, a, b, c, out, lse, *n, dq, dk, dv, 0.125, True)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(4):
        q.mul_(1.1), g2.mul_(0.5)
        args[1][7] += 3  # the lengths are device data: a replay follows them
        args[1][-1] -= 3
        step()
        torch.cuda.synchronize()
        eager = [t.clone() for o in outs for t in o]
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, (t for o in outs for t in o)):
            assert torch.equal(a, b), n


def test_the_plan_refuses_what_is_no_pack():
    plan, none = _lib.lib().v3d_attention_pack_plan, [None] * 4
    assert plan(0, 1, 10, 10, 4, 2, 64, *none) == 0
    assert plan(0, 1, 10, 10, 4, 3, 64, *none) == -1 and plan(0, -1, 10, 10, 4, 2, 64, *none) == -1
    assert plan(3, 1, 10, 10, 4, 2, 64, *none) == -1 and plan(0, 1, 10, 10, 4, 2, 257, *none) == -4
