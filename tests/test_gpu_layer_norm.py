"""ops.layer_norm against the definition in 64 bits: forward, gradients, types, odd sizes, refusals."""
import numpy as np
import pytest
import torch

from vision3d_amd import ops

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# every launch geometry of the three types: 16 / 32 / 64 threads a row, one and two vectors of 64, 256 and 1024 threads
CHANNELS = [1, 3, 64, 100, 127, 256, 257, 512, 771, 1024, 1500, 2048, 4096, 4099, 8192]


def _formula(x, r, w, b, eps, g=None):
    t = x if r is None else x + r
    mean = t.mean(1, keepdim=True)
    var = ((t - mean) ** 2).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    u = (t - mean) * rstd
    y = u * w + b
    if g is None:
        return y, u, t, rstd
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - u * (gw * u).mean(1, keepdim=True))
    return y, u, t, rstd, dx, (g * u).sum(0), g.sum(0)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _unit_error(t, rstd):
    """How far the normalised value may be off, relative to max(1, |u|): 32-bit sums of up to 16 values a thread and 10
    joining steps are off by at most 26 half steps of mean |t|, the difference to the mean by one of |t|, the variance by
    26 relative steps (half of that in rstd); every step counted at its largest, times 2 for the products around them."""
    size = t.abs().amax(1, keepdim=True) * rstd
    return 2 * 2.0 ** -24 * (27 * size + 20 + size)


def _inputs(rows, channels, dtype, residual, seed=0, wdtype=None):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=gen)
    x = (mk(rows, channels) * 2 + mk(channels)).to(dtype)
    r = mk(rows, channels).to(dtype) if residual else None
    w = (mk(channels) * 0.3 + 1).to(wdtype or dtype)
    b = mk(channels).to(wdtype or dtype)
    g = mk(rows, channels).to(dtype)
    return x, r, w, b, g


def _d(t):
    return None if t is None else t.double()


def _c(t):
    return None if t is None else t.to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", CHANNELS)
def test_forward_and_gradients(dtype, channels):
    for rows, residual in ((1, False), (5, True), (67, False), (1030, True)):
        if rows * channels > 1030 * 1030:
            rows = 130
        x, r, w, b, g = _inputs(rows, channels, dtype, residual, seed=rows)
        y, u, t, rstd, dx, dw, db = _formula(_d(x), _d(r), _d(w), _d(b), 1e-5, _d(g))
        leaves = [v.to(DEV).requires_grad_(True) for v in ([x, w, b] + ([r] if residual else []))]
        out = ops.layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3] if residual else None)
        grads = torch.autograd.grad(out, leaves, g.to(DEV))
        e = _unit_error(t, rstd)
        big = u.abs().clamp(min=1)
        half = _half(dtype)
        tol = half * y.abs() + e * big * w.double().abs() + 2.0 ** -23 * (y.abs() + b.double().abs()) + 2.0 ** -24
        assert out.dtype == dtype and out.shape == x.shape
        assert ((out.cpu().double() - y).abs() <= tol).all()
        # dx: every term is bounded by the row's largest |gw| (1 + |u| + |u| mean|u|...): each factor is off by e or 30 steps
        gw = (g.double() * w.double()).abs()
        most = gw.amax(1, keepdim=True) + gw + big * (gw * u.abs()).mean(1, keepdim=True)
        tol = half * dx.abs() + rstd * most * (4 * e * big + 60 * 2.0 ** -24) + 2.0 ** -24
        assert ((grads[0].cpu().double() - dx).abs() <= tol).all()
        if residual:
            assert torch.equal(grads[3], grads[0])
        # column sums: at most rows + 80 additions of 32-bit values
        steps = (rows + 80) * 2.0 ** -24
        tol = half * dw.abs() + steps * (g.double() * u).abs().sum(0) + (g.double().abs() * e * big).sum(0) + 2.0 ** -24
        assert ((grads[1].cpu().double() - dw).abs() <= tol).all()
        assert ((grads[2].cpu().double() - db).abs() <= half * db.abs() + steps * g.double().abs().sum(0)).all()
        # the same bits a second time, without gradients and from the same leaves
        with torch.no_grad():
            again = ops.layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3] if residual else None)
        assert torch.equal(again, out)


@pytest.mark.gpu
def test_gradient_against_differences():
    x, r, w, b, g = (v.double() for v in _inputs(3, 20, torch.float32, True, seed=5))
    leaves = [v.float().to(DEV).requires_grad_(True) for v in (x, r, w, b)]
    out = ops.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    grads = torch.autograd.grad(out, leaves, g.float().to(DEV))
    f = lambda a, c, d, e: (_formula(a, c, d, e, 1e-5)[0] * g).sum()
    h = 1e-5
    base = [x, r, w, b]
    for k, leaf in enumerate(base):
        flat = leaf.reshape(-1)
        for i in range(0, flat.numel(), 7):
            step = torch.zeros_like(flat)
            step[i] = h
            up, down = list(base), list(base)
            up[k], down[k] = (flat + step).view_as(leaf), (flat - step).view_as(leaf)
            slope = ((f(*up) - f(*down)) / (2 * h)).item()
            # central differences: third derivatives of order 1 times h^2, rounding 1e-16 / h; kernel: 1e-5 of sizes ~ 10
            assert abs(grads[k].reshape(-1)[i].item() - slope) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_weights_in_fp32_and_absent(dtype):
    x, r, w, b, g = _inputs(33, 200, dtype, True, wdtype=torch.float32)
    for weight, bias in ((w, b), (None, None), (w, None), (None, b)):
        wd = torch.ones(200).double() if weight is None else weight.double()
        bd = torch.zeros(200).double() if bias is None else bias.double()
        y, u, t, rstd, dx, dw, db = _formula(_d(x), _d(r), wd, bd, 1e-3, _d(g))
        leaf = x.to(DEV).requires_grad_(True)
        extra = [v.to(DEV).requires_grad_(True) for v in (weight, bias) if v is not None]
        it = iter(extra)
        wt = next(it) if weight is not None else None
        bt = next(it) if bias is not None else None
        out = ops.layer_norm(leaf, wt, bt, eps=1e-3, residual=r.to(DEV))
        tol = _half(dtype) * y.abs() + 1e-5 * (wd.abs() * u.abs().clamp(min=1) + bd.abs())
        assert ((out.cpu().double() - y).abs() <= tol).all()
        grads = torch.autograd.grad(out, [leaf] + extra, g.to(DEV))
        want = [dx] + ([dw] if weight is not None else []) + ([db] if bias is not None else [])
        for got, ref in zip(grads[1:], want[1:]):
            assert got.dtype == torch.float32
            assert ((got.cpu().double() - ref).abs() <= 2e-5 * (1 + ref.abs())).all()
        assert ((grads[0].cpu().double() - dx).abs() <= _half(dtype) * dx.abs() + 1e-5 * (1 + dx.abs())).all()


@pytest.mark.gpu
def test_batched_strided_empty_and_nonfinite():
    x = torch.randn(4, 6, 5, 32, device=DEV)
    y = ops.layer_norm(x.transpose(1, 2))
    want = _formula(x.transpose(1, 2).reshape(-1, 32).cpu().double(), None, 1.0, 0.0, 1e-5)[0]
    assert y.shape == (4, 5, 6, 32) and (y.reshape(-1, 32).cpu().double() - want).abs().max() < 1e-5
    e = torch.randn(0, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    out = ops.layer_norm(e, w)
    ge, gw = torch.autograd.grad(out, (e, w), torch.zeros_like(out))
    assert out.shape == (0, 16) and ge.shape == (0, 16) and torch.equal(gw, torch.zeros_like(gw))
    # a row of one value everywhere: variance 0; a row with an infinity spoils itself alone
    x = torch.randn(9, 300, device=DEV)
    x[2] = 7.25
    clean = ops.layer_norm(x)
    assert torch.equal(clean[2], torch.zeros_like(clean[2]))
    x[4, 17] = float("inf")
    got = ops.layer_norm(x)
    assert torch.isnan(got[4]).all()
    keep = [i for i in range(9) if i != 4]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.gpu
def test_accumulated_gradients_are_apart():
    x, r, w, b, g = (v.to(DEV).requires_grad_(True) for v in _inputs(40, 64, torch.float32, True))
    for k in range(2):  # the second pass adds to what the first left
        ops.layer_norm(x, w, b, residual=r).backward(g.detach())
    want = torch.autograd.grad(ops.layer_norm(x, w, b, residual=r), (x, w, b), g.detach())
    for leaf, one in zip((x, w, b), want):
        assert torch.equal(leaf.grad, one + one)
    assert torch.equal(r.grad, x.grad)
    x.grad.zero_()  # one gradient for two inputs, but not one tensor
    assert torch.equal(r.grad, want[0] + want[0])
    # a frozen input, frozen weights: only what is asked for
    (gr,) = torch.autograd.grad(ops.layer_norm(x.detach(), w.detach(), b.detach(), residual=r), r, g.detach())
    assert torch.equal(gr, want[0])
    (gb,) = torch.autograd.grad(ops.layer_norm(x.detach(), None, b), b, g.detach())
    assert torch.equal(gb, torch.autograd.grad(ops.layer_norm(x.detach(), torch.ones_like(w), b), b, g.detach())[0])


@pytest.mark.gpu
def test_other_stream_and_graph_replays():
    x, r, w, b, g = (v.to(DEV) for v in _inputs(300, 333, torch.bfloat16, True))
    want = ops.layer_norm(x, w, b, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.layer_norm(x, w, b, residual=r)
    side.synchronize()
    assert torch.equal(got, want)

    from vision3d_amd import ext
    rows = x.shape[0]
    y, stats = torch.empty_like(x), x.new_empty((2, rows), dtype=torch.float32)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)

    def step():
        ext.layer_norm_forward(x, r, w, b, y, stats, 1e-5)
        ext.layer_norm_backward(g, x, r, w, stats, dx, dw, db)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        x.add_(0.25)
        step()
        torch.cuda.synchronize()
        eager = [t.clone() for t in (y, dx, dw, db)]
        for t in (y, dx, dw, db):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(eager, (y, dx, dw, db)):
            assert torch.equal(a, c), k


@pytest.mark.gpu
def test_refusals():
    x = torch.randn(4, 8, device=DEV)
    with pytest.raises(RuntimeError, match="residual must have the shape"):
        ops.layer_norm(x, residual=x[:2])
    with pytest.raises(RuntimeError, match="weight must have shape"):
        ops.layer_norm(x, torch.ones(7, device=DEV))
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        ops.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="V3D_ERR_INVALID_ARGUMENT"):
        ops.layer_norm(x, torch.ones(8, device=DEV, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="V3D_ERR_INVALID_ARGUMENT"):
        ops.layer_norm(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="V3D_ERR_SIZE_LIMIT"):
        ops.layer_norm(torch.zeros(2, 8193, device=DEV))
    with pytest.raises(RuntimeError, match="expected scalar type"):
        ops.layer_norm(x, residual=x.half())


def test_refusals_without_a_gpu():
    from vision3d_amd import _lib

    with pytest.raises(RuntimeError, match="layer_norm: CUDA tensors required"):
        ops.layer_norm(torch.zeros(3, 4))
    lib = _lib.lib()
    assert lib.v3d_layer_norm_fwd(None, None, None, None, None, None, None, 7, 7, 1, 1, 1e-5, 0, None) == -1
    assert lib.v3d_layer_norm_fwd(None, None, None, None, None, None, None, 1, 2, 1, 1, 1e-5, 0, None) == -1
    assert lib.v3d_layer_norm_fwd(None, None, None, None, None, None, None, 0, 0, 1, 1, 1e-5, 0, None) == -1
    assert lib.v3d_layer_norm_fwd(None, None, None, None, None, None, None, 1, 1, 1, 16385, 1e-5, 0, None) == -4
    assert lib.v3d_layer_norm_fwd(None, None, None, None, None, None, None, 0, 0, 0, 1, 1e-5, 0, None) == 0
    assert lib.v3d_layer_norm_bwd_workspace_bytes(0, 8) == 0
    assert lib.v3d_layer_norm_bwd_workspace_bytes(10 ** 7, 1000) == 1024 * 1000 * 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("channels", [8193, 8200, 12289, 16384])
def test_widest_rows(dtype, channels):
    test_forward_and_gradients(dtype, channels)  # 1024 threads, two vectors each


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(131072 + 777, 8), (65536 + 9, 200), (8192 + 5, 4099)])
def test_more_rows_than_workgroups_take_at_once(dtype, rows, channels):
    # the forward's 8192 workgroups take 16, 8 (4) and 1 rows at a time: the last ones come in a second round
    x, r, w, b, g = (None if v is None else v.to(DEV) for v in _inputs(rows, channels, dtype, True, seed=rows))
    y, u, t, rstd, dx, dw, db = _formula(_d(x), _d(r), _d(w), _d(b), 1e-5, _d(g))
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    out = ops.layer_norm(*leaves, residual=r)
    grads = torch.autograd.grad(out, leaves, g)
    e, big, half = _unit_error(t, rstd), u.abs().clamp(min=1), _half(dtype)
    tol = half * y.abs() + e * big * w.detach().double().abs() + 2.0 ** -23 * (y.abs() + b.detach().double().abs()) + 2.0 ** -24
    assert ((out.detach().double() - y).abs() <= tol).all()
    gw = (g.double() * w.detach().double()).abs()
    most = gw.amax(1, keepdim=True) + gw + big * (gw * u.abs()).mean(1, keepdim=True)
    assert ((grads[0].double() - dx).abs() <= half * dx.abs() + rstd * most * (4 * e * big + 60 * 2.0 ** -24) + 2.0 ** -24).all()
    steps = (rows + 80) * 2.0 ** -24
    tol = half * dw.abs() + steps * (g.double() * u).abs().sum(0) + (g.double().abs() * e * big).sum(0) + 2.0 ** -24
    assert ((grads[1].double() - dw).abs() <= tol).all()
    assert ((grads[2].double() - db).abs() <= half * db.abs() + steps * g.double().abs().sum(0)).all()
