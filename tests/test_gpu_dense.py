"""GPU: linear and gated_ffn against 64-bit forms of the same formulas, forward and backward."""
import math

import pytest
import torch

from tests import dense_ref as ref

pytestmark = pytest.mark.gpu

GAMMA = 0.1
ACTS = ["none", "relu", "silu", "gelu_tanh", "era"]
BF16, F32 = torch.bfloat16, torch.float32


def rand(gen, *shape, std=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=gen, dtype=torch.float32) * std).to(dtype)


def d64(t):
    return None if t is None else t.detach().double().cpu()


def leaf(t):
    return None if t is None else t.cuda().requires_grad_()


def run_linear(T, K, N, act="none", dtype=BF16, bias=True, residual=True, seed=0, wdtype=None,
               train=True):
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(seed)
    wd = wdtype or dtype
    x, w = rand(gen, T, K, dtype=dtype), rand(gen, N, K, std=K ** -0.5, dtype=wd)
    b = rand(gen, N, std=0.1, dtype=wd) if bias else None
    r = rand(gen, T, N, dtype=dtype) if residual else None
    dy = rand(gen, T, N, dtype=dtype)
    leaves = [leaf(t) for t in (x, w, b, r)]
    with torch.set_grad_enabled(train):
        y = vb.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act, gamma=GAMMA)
    # fp32 parameters of a bf16 call are cast to bf16
    want = ref.linear(d64(x), d64(w.to(dtype)), d64(None if b is None else b.to(dtype)), d64(r),
                      d64(dy) if train else None, act, GAMMA, dtype, wd)
    assert y.dtype == dtype
    ref.check("y", y, *want["y"], 1, dtype)
    if not train:
        assert not y.requires_grad
        return
    have = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, have, dy.cuda())
    names = [n for n, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None]
    for n, g, t in zip(names, grads, have):
        assert g.dtype == t.dtype
        if n == "dr":
            assert torch.equal(g.cpu(), dy)
        else:
            ref.check(n, g, *want[n], 3, BF16 if BF16 in (dtype, g.dtype) else F32)


# one token, the small-batch form's edges (8, 9, 16 | 17), tiles and their edges (256, 257)
@pytest.mark.parametrize("T", [1, 2, 8, 9, 16, 17, 63, 128, 129, 256, 257])
@pytest.mark.parametrize("K,N", [(64, 64), (40, 24), (136, 264)])
def test_linear_sizes(T, K, N):
    run_linear(T, K, N, act="silu", seed=T + K)


# widths that no 16-byte load divides, single columns
@pytest.mark.parametrize("T,K,N", [(1, 1, 1), (5, 33, 7), (16, 65, 1), (17, 1, 3), (33, 257, 129),
                                   (300, 31, 513), (129, 7, 255)])
@pytest.mark.parametrize("act", ["none", "era"])
def test_linear_odd(T, K, N, act):
    run_linear(T, K, N, act=act, seed=T)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [3, 70])
@pytest.mark.parametrize("bias,residual", [(True, True), (True, False), (False, True), (False, False)])
def test_linear_forms(act, T, bias, residual):
    run_linear(T, 72, 48, act=act, bias=bias, residual=residual, seed=T)


@pytest.mark.parametrize("T,K,N", [(1, 40, 24), (7, 33, 5), (130, 96, 200), (64, 1000, 16),
                                   (1000, 24, 40)])
@pytest.mark.parametrize("act", ["none", "gelu_tanh"])
def test_linear_f32(T, K, N, act):
    run_linear(T, K, N, act=act, dtype=F32, seed=T)


@pytest.mark.parametrize("T,K,N", [(300, 8192, 256), (2000, 264, 40), (150, 40, 6000)])
def test_linear_f32_long_sums(T, K, N):
    """Sums of thousands of terms stay at fp32's own error, in every product: below 1e-6 by norm
    (two thousand roundings to nearest of independent sign, sqrt(2000) 2^-24 = 2.7e-6, would
    already be over; a truncating accumulator reaches 9e-6 at 8192 terms)."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(T)
    x, w, dy = (rand(gen, *s, dtype=F32) for s in ((T, K), (N, K), (T, N)))
    lx, lw = leaf(x), leaf(w)
    y = vb.linear(lx, lw)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy.cuda())
    x, w, dy = x.double(), w.double(), dy.double()
    for got, want in ((y, x @ w.t()), (dx, dy @ w), (dw, dy.t() @ x)):
        assert float((d64(got) - want).norm() / want.norm()) < 1e-6


@pytest.mark.parametrize("T", [5, 90])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, F32), (F32, BF16)])
def test_linear_parameters_of_another_type(T, dtype, wdtype):
    run_linear(T, 48, 40, act="era", dtype=dtype, wdtype=wdtype, seed=3)


# k divided over SMs (few tiles, long sums) and many tiles
@pytest.mark.parametrize("T,K,N", [(64, 4096, 256), (40, 2048, 520), (33, 1000, 1100), (17, 130, 2500),
                                   (128, 6000, 136), (65, 64, 20000), (200, 4096, 256), (2100, 72, 136),
                                   (3000, 256, 2304), (513, 512, 4096)])
def test_linear_splits(T, K, N):
    run_linear(T, K, N, act="gelu_tanh", seed=1)


@pytest.mark.parametrize("T", [1, 12, 40, 300])
@pytest.mark.parametrize("act", ["none", "era"])
def test_linear_inference(T, act):
    run_linear(T, 264, 104, act=act, seed=2, train=False)


def test_linear_empty_batch():
    import velvetoptimizer_b200 as vb
    for dtype in (BF16, F32):
        x = torch.zeros(0, 40, device="cuda", dtype=dtype, requires_grad=True)
        w = torch.randn(24, 40, device="cuda").to(dtype).requires_grad_()
        b = torch.zeros(24, device="cuda", dtype=dtype, requires_grad=True)
        y = vb.linear(x, w, b, activation="era")
        assert y.shape == (0, 24)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == x.shape and not dw.any() and not db.any()


def views(gen, T, K, dtype=BF16):
    """The same kinds of x that a program holds: slices, transposes, expansions, odd starts."""
    base = rand(gen, T + 2, 2 * K + 16, dtype=dtype).cuda()
    yield base[1:T + 1, 8:8 + K]                       # aligned column slice, long pitch
    yield base[1:T + 1, 3:3 + K]                       # starts between 16-byte boundaries
    yield rand(gen, K, T, dtype=dtype).cuda().t()      # columns contiguous
    yield rand(gen, 1, K, dtype=dtype).cuda().expand(T, K)
    yield rand(gen, T, 2 * K, dtype=dtype).cuda()[:, ::2]
    yield rand(gen, 2 * T, K, dtype=dtype).cuda()[::2]
    flat = rand(gen, T * (K + 1) + 1, dtype=dtype).cuda()
    yield flat[1:1 + T * (K + 1)].view(T, K + 1)[:, :K]  # an odd pitch


@pytest.mark.parametrize("T", [6, 130])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_strides(T, dtype):
    import velvetoptimizer_b200 as vb
    K, N = 64, 56
    gen = torch.Generator().manual_seed(0)
    w0 = rand(gen, N, K, std=0.1, dtype=dtype).cuda()
    dys = list(views(gen, T, N, dtype))
    for i, x in enumerate(views(gen, T, K, dtype)):
        wide = rand(gen, N, K + 24, std=0.1, dtype=dtype).cuda()
        for w in (w0, wide[:, 8:8 + K], wide[:, 5:5 + K], w0.t().contiguous().t()):
            dy, r = dys[i], dys[(i + 1) % len(dys)]
            lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
            y = vb.linear(lx, lw, residual=r, activation="silu")
            dx, dw = torch.autograd.grad(y, (lx, lw), dy)
            want = ref.linear(d64(x), d64(w), None, d64(r), d64(dy), "silu", GAMMA, dtype)
            for n, g in (("y", y), ("dx", dx), ("dw", dw)):
                ref.check(f"{n} of view {i}", g, *want[n], 3, dtype)


def test_linear_batched_and_1d():
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    x, w = rand(gen, 2, 3, 5, 40).cuda(), rand(gen, 24, 40).cuda()
    y = vb.linear(x, w)
    assert y.shape == (2, 3, 5, 24)
    assert torch.equal(y.reshape(30, 24), vb.linear(x.reshape(30, 40), w))
    assert torch.equal(vb.linear(x[0, 0, 0], w), vb.linear(x[0, 0, :1], w)[0])


@pytest.mark.parametrize("T", [4, 200])
def test_linear_partial_gradients(T):
    """Only what is asked for is computed, with the same bits."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    base = [rand(gen, T, 72).cuda(), rand(gen, 88, 72, std=0.1).cuda(), rand(gen, 88).cuda(),
            rand(gen, T, 88).cuda()]
    dy = rand(gen, T, 88).cuda()

    def grads(mask):
        p = [t.clone().requires_grad_(bool(m)) for t, m in zip(base, mask)]
        y = vb.linear(p[0], p[1], p[2], residual=p[3], activation="era")
        return torch.autograd.grad(y, [t for t in p if t.requires_grad], dy)

    full = grads((1, 1, 1, 1))
    for mask in [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 1, 0), (0, 1, 1, 1)]:
        want = [g for g, m in zip(full, mask) if m]
        assert all(torch.equal(a, b) for a, b in zip(grads(mask), want)), mask


def run_ffn(T, H, I, act="era", dtype=BF16, bias=True, residual=True, seed=0, wdtype=None, train=True):
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(seed)
    wd = wdtype or dtype
    x = rand(gen, T, H, dtype=dtype)
    ws = [rand(gen, I, H, std=H ** -0.5, dtype=wd), rand(gen, I, H, std=H ** -0.5, dtype=wd),
          rand(gen, H, I, std=I ** -0.5, dtype=wd)]
    bs = [rand(gen, n, std=0.1, dtype=wd) if bias else None for n in (I, I, H)]
    r = rand(gen, T, H, dtype=dtype) if residual else None
    dy = rand(gen, T, H, dtype=dtype)
    leaves = [leaf(t) for t in (x, *ws, *bs, r)]
    with torch.set_grad_enabled(train):
        y = vb.gated_ffn(*leaves[:7], residual=leaves[7], activation=act, gamma=GAMMA)
    to = lambda t: None if t is None else d64(t.to(dtype))  # noqa: E731
    want = ref.gated_ffn(d64(x), *map(to, ws), *map(to, bs), d64(r), d64(dy) if train else None,
                         act, GAMMA, dtype, wd)
    # h and y rounded
    ref.check("y", y, *want["y"], 2, dtype)
    if not train:
        return
    have = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, have, dy.cuda())
    names = [n for n, t in zip(("dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd", "dr"), leaves)
             if t is not None]
    for n, g, t in zip(names, grads, have):
        assert g.dtype == t.dtype
        if n == "dr":
            assert torch.equal(g.cpu(), dy)
        else:  # dg or du (or h), then the gradient rounded
            ref.check(n, g, *want[n], 2, dtype)


@pytest.mark.parametrize("T", [1, 8, 9, 16, 17, 100, 128, 129, 256, 300])
@pytest.mark.parametrize("H,I", [(64, 128), (40, 72), (136, 264)])
def test_gated_ffn_sizes(T, H, I):
    run_ffn(T, H, I, seed=T)


@pytest.mark.parametrize("T,H,I", [(1, 1, 1), (3, 33, 17), (16, 7, 129), (17, 31, 1), (70, 129, 65),
                                   (260, 65, 257)])
def test_gated_ffn_odd(T, H, I):
    run_ffn(T, H, I, seed=T)


@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("T", [3, 70])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True)])
def test_gated_ffn_forms(act, T, bias, residual):
    run_ffn(T, 72, 104, act=act, bias=bias, residual=residual, seed=T)


@pytest.mark.parametrize("T,H,I", [(1, 40, 24), (9, 33, 21), (140, 72, 200), (70, 520, 48)])
def test_gated_ffn_f32(T, H, I):
    run_ffn(T, H, I, dtype=F32, seed=T)


@pytest.mark.parametrize("T", [5, 90])
def test_gated_ffn_f32_parameters(T):
    run_ffn(T, 48, 72, wdtype=F32, seed=3)


@pytest.mark.parametrize("T,H,I", [(40, 1024, 2048), (1500, 256, 640), (700, 520, 1304)])
def test_gated_ffn_splits(T, H, I):
    run_ffn(T, H, I, seed=1)


@pytest.mark.parametrize("T", [1, 12, 40, 300])
def test_gated_ffn_inference(T):
    run_ffn(T, 264, 520, seed=2, train=False)


def test_gated_ffn_empty_batch():
    import velvetoptimizer_b200 as vb
    for dtype in (BF16, F32):
        x = torch.zeros(0, 40, device="cuda", dtype=dtype, requires_grad=True)
        ws = [torch.randn(s, device="cuda").to(dtype).requires_grad_() for s in ((24, 40), (24, 40), (40, 24))]
        y = vb.gated_ffn(x, *ws)
        got = torch.autograd.grad(y, (x, *ws), torch.zeros_like(y))
        assert y.shape == (0, 40) and not any(g.any() for g in got)


def test_gated_ffn_partial_gradients():
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    T, H, I = 150, 72, 104
    base = [rand(gen, T, H), rand(gen, I, H, std=0.1), rand(gen, I, H, std=0.1), rand(gen, H, I, std=0.1),
            rand(gen, I), rand(gen, I), rand(gen, H), rand(gen, T, H)]
    base = [t.cuda() for t in base]
    dy = rand(gen, T, H).cuda()

    def grads(mask):
        p = [t.clone().requires_grad_(bool(m)) for t, m in zip(base, mask)]
        y = vb.gated_ffn(*p[:7], residual=p[7])
        return torch.autograd.grad(y, [t for t in p if t.requires_grad], dy)

    full = grads([1] * 8)
    for i in range(8):
        one = grads([j == i for j in range(8)])
        # one weight's gradient alone may be divided over k differently: within two roundings
        assert torch.allclose(one[0].float(), full[i].float(), rtol=2 ** -7, atol=1e-3), i


@pytest.mark.parametrize("T", [6, 60, 200])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gated_ffn_strides(T, dtype):
    import velvetoptimizer_b200 as vb
    H, I = 40, 56
    gen = torch.Generator().manual_seed(0)
    # a transposed weight, a slice with a long pitch, one that starts between 16-byte boundaries
    wg = rand(gen, H, I, std=0.2, dtype=dtype).cuda().t()
    wu = rand(gen, I, H + 24, std=0.2, dtype=dtype).cuda()[:, 8:8 + H]
    wd = rand(gen, H * I + 3, std=0.2, dtype=dtype).cuda()[3:].view(H, I)
    bs = [rand(gen, 2 * n, dtype=dtype).cuda()[::2] for n in (I, I, H)]
    dys = list(views(gen, T, H, dtype))
    for i, x in enumerate(views(gen, T, H, dtype)):
        dy, r = dys[i], dys[(i + 2) % len(dys)]
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd, *bs)]
        y = vb.gated_ffn(*leaves, residual=r)
        got = torch.autograd.grad(y, leaves, dy)
        want = ref.gated_ffn(*(d64(t) for t in (x, wg, wu, wd, *bs)), d64(r), d64(dy), "era", GAMMA, dtype)
        ref.check(f"y of view {i}", y, *want["y"], 2, dtype)
        for n, g in zip(("dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd"), got):
            ref.check(f"{n} of view {i}", g, *want[n], 2, dtype)


# More than 2^31 elements in an operand.  Only the last rows (or features) have a gradient, so the
# sums over all rows are those of the last ones: a form of their size is the whole reference.
def last_rows(T, N, R, gen):
    dy = torch.zeros(T, N, device="cuda", dtype=BF16)
    dy[-R:] = rand(gen, R, N).cuda()
    return dy


def test_linear_rows_past_32_bits():
    import velvetoptimizer_b200 as vb
    T, K, N, R = 270_000, 64, 8192, 40
    gen = torch.Generator().manual_seed(0)
    x = rand(gen, T, K).cuda().requires_grad_()
    w = rand(gen, N, K, std=K ** -0.5).cuda().requires_grad_()
    b = rand(gen, N, std=0.1).cuda().requires_grad_()
    y = vb.linear(x, w, b, activation="silu")
    assert y.numel() > 2 ** 31
    dy = last_rows(T, N, R, gen)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = ref.linear(d64(x[-R:]), d64(w), d64(b), None, d64(dy[-R:]), "silu", GAMMA, BF16)
    ref.check("y", y[-R:], *want["y"], 1, BF16)
    ref.check("dx", dx[-R:], *want["dx"], 3, BF16)
    ref.check("dw", dw, *want["dw"], 3, BF16)
    ref.check("db", db, *want["db"], 3, BF16)
    assert not dx[:-R].any()
    del y, dy, dx
    torch.cuda.empty_cache()


def test_gated_ffn_rows_past_32_bits():
    import velvetoptimizer_b200 as vb
    T, H, I, R = 270_000, 64, 8192, 40
    gen = torch.Generator().manual_seed(0)
    leaves = [t.cuda().requires_grad_() for t in (
        rand(gen, T, H), rand(gen, I, H, std=H ** -0.5), rand(gen, I, H, std=H ** -0.5),
        rand(gen, H, I, std=I ** -0.5), rand(gen, I, std=0.1), rand(gen, I, std=0.1),
        rand(gen, H, std=0.1))]
    y = vb.gated_ffn(*leaves, activation="silu")
    dy = last_rows(T, H, R, gen)
    got = torch.autograd.grad(y, leaves, dy)
    want = ref.gated_ffn(d64(leaves[0][-R:]), *(d64(t) for t in leaves[1:]), None, d64(dy[-R:]), "silu",
                         GAMMA, BF16)
    ref.check("y", y[-R:], *want["y"], 2, BF16)
    assert not got[0][:-R].any()
    ref.check("dx", got[0][-R:], *want["dx"], 2, BF16)
    for n, g in zip(("dwg", "dwu", "dwd", "dbg", "dbu", "dbd"), got[1:]):
        ref.check(n, g, *want[n], 2, BF16)
    del y, dy, got
    torch.cuda.empty_cache()


# the streaming form, the decode form and the pair form on a weight whose last rows lie that far
@pytest.mark.parametrize("T", [1, 40, 200])
def test_linear_weight_past_32_bits(T):
    import velvetoptimizer_b200 as vb
    K, N, R = 65_544, 32_840, 72
    gen = torch.Generator().manual_seed(0)
    x = rand(gen, T, K).cuda().requires_grad_()
    w = torch.zeros(N, K, device="cuda", dtype=BF16)
    w[-R:] = rand(gen, R, K, std=K ** -0.5).cuda()
    w.requires_grad_()
    assert w.numel() > 2 ** 31
    y = vb.linear(x, w)
    assert not y[:, :-R].any()
    dy = torch.zeros(T, N, device="cuda", dtype=BF16)
    dy[:, -R:] = rand(gen, T, R).cuda()
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = ref.linear(d64(x), d64(w[-R:]), None, None, d64(dy[:, -R:]), "none", GAMMA, BF16)
    ref.check("y", y[:, -R:], *want["y"], 1, BF16)
    ref.check("dx", dx, *want["dx"], 3, BF16)
    ref.check("dw", dw[-R:], *want["dw"], 3, BF16)
    assert not dw[:-R].any()
    del w, dw
    torch.cuda.empty_cache()


def test_far_values_stay_finite():
    """Pre-activations far out in the tails: the derivative's polynomial must not overflow."""
    import velvetoptimizer_b200 as vb
    for dtype in (BF16, F32):
        for T in (4, 40):
            x = torch.ones(T, 8, device="cuda", dtype=dtype)
            x[1::2] = -1
            w = torch.full((16, 8), 1e18, device="cuda", dtype=dtype)
            for act in ACTS:
                lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
                y = vb.linear(lx, lw, activation=act)
                assert torch.isfinite(y).all(), act
                dx, dw = torch.autograd.grad(y, (lx, lw), torch.ones_like(y))
                assert torch.isfinite(dx).all() and torch.isfinite(dw).all(), act


def test_nan_and_inf_pass_through():
    import velvetoptimizer_b200 as vb
    for dtype in (BF16, F32):
        for T in (4, 40):
            x = torch.zeros(T, 16, device="cuda", dtype=dtype)
            x[1, 3], x[2, 5] = float("nan"), float("inf")
            w = torch.ones(24, 16, device="cuda", dtype=dtype)
            for act in ACTS:
                y = vb.linear(x, w, activation=act)
                assert torch.isnan(y[1]).all() and torch.isinf(y[2]).all(), (act, dtype, T)
                assert torch.isfinite(y[0]).all() and torch.isfinite(y[3:]).all()


@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan"), 3.4e38])
def test_f32_special_values(T, bad):
    """fp32 products with an operand that has no sum of bf16 parts: the same infinities and NaNs
    as fp32 arithmetic gives, and the other values as exact as ever."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(T)
    K, N = 72, 40
    for where in ("x", "w", "dy", None):
        x, w, dy = (rand(gen, *s, dtype=F32) for s in ((T, K), (N, K), (T, N)))
        w[5, 7] = 0.0  # infinity times zero
        if where:
            {"x": x, "w": w, "dy": dy}[where][2, 7] = bad
        lx, lw = leaf(x), leaf(w)
        y = vb.linear(lx, lw)
        dx, dw = torch.autograd.grad(y, (lx, lw), dy.cuda())
        for got, a, b in ((y, x, w.t()), (dx, dy, w), (dw, dy.t(), x)):
            want, got = a @ b, got.detach().cpu()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
            assert torch.equal(got[want.isinf()], want[want.isinf()])
            ok = want.isfinite()
            a64, b64 = a.double(), b.double()
            exact = (a64 @ b64)[ok]
            bound = ((a64.abs() @ b64.abs()) * (a.shape[1] + 2) * 2.0 ** -23)[ok]
            assert ((got[ok].double() - exact).abs() <= bound + 2.0 ** -24 * exact.abs()).all()
    p = [rand(gen, T, 24, dtype=F32), rand(gen, 48, 24, dtype=F32), rand(gen, 48, 24, dtype=F32),
         rand(gen, 24, 48, dtype=F32)]
    p[0][1, 3] = bad
    leaves = [leaf(t) for t in p]
    y = vb.gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert not torch.isfinite(y[1]).all() and torch.isfinite(y[0]).all()
    if math.isfinite(bad):
        return
    assert not torch.isfinite(grads[0][1]).all() and torch.isfinite(grads[0][0]).all()


@pytest.mark.parametrize("T", [5, 100])
def test_gradients_against_differences(T):
    """fp32: <gradient, v> against the difference of the operators' own values along v.

    With f = <dy, op(p)> the central difference has a truncation error of eps^2 / 6 |f'''| and a
    rounding error of about |f| 2^-23 sqrt(n) / eps; at eps = 2^-6 both are below 1e-3 of the
    norms used here, the allowance is 5e-3 of |gradient| |v|.
    """
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(5)
    H, I = 24, 40
    p = [rand(gen, T, H, dtype=F32), rand(gen, I, H, std=0.2, dtype=F32),
         rand(gen, I, H, std=0.2, dtype=F32), rand(gen, H, I, std=0.2, dtype=F32),
         rand(gen, I, dtype=F32), rand(gen, I, dtype=F32), rand(gen, H, dtype=F32)]
    p = [t.cuda() for t in p]
    dy, dz = rand(gen, T, H, dtype=F32).cuda(), rand(gen, T, I, dtype=F32).cuda()

    def ffn(q):
        return vb.gated_ffn(*q)

    def lin(q):
        return vb.linear(q[0], q[1], q[4], activation="era")

    for fn, cot, used in ((ffn, dy, range(7)), (lin, dz, (0, 1, 4))):
        leaves = [t.clone().requires_grad_() for t in p]
        grads = torch.autograd.grad(fn(leaves), [leaves[i] for i in used], cot)
        for i, g in zip(used, grads):
            v = torch.randn(p[i].shape, generator=gen).cuda()
            eps = 2.0 ** -6 / float(v.abs().max())
            with torch.no_grad():
                at = [[(t + s * eps * v) if j == i else t for j, t in enumerate(p)] for s in (1, -1)]
                diff = (cot.double() * (fn(at[0]).double() - fn(at[1]).double())).sum() / (2 * eps)
            dot = (g.double() * v.double()).sum()
            assert abs(float(dot - diff)) <= 5e-3 * float(g.norm() * v.norm()), i


def test_same_bits_every_run():
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    for T, H, I in ((12, 264, 520), (64, 1024, 2048), (700, 256, 640)):
        p = [rand(gen, T, H), rand(gen, I, H, std=0.05), rand(gen, I, H, std=0.05),
             rand(gen, H, I, std=0.05), rand(gen, I), rand(gen, I), rand(gen, H)]
        p = [t.cuda().requires_grad_() for t in p]
        dy = rand(gen, T, H).cuda()
        first = None
        for _ in range(4):
            y = vb.gated_ffn(*p)
            got = [y, *torch.autograd.grad(y, p, dy)]
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_captured_and_replayed():
    """Forward and backward in a CUDA graph, replayed on new inputs."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    for T in (8, 150):
        H, I = 72, 136
        shapes = ((T, H), (I, H), (I, H), (H, I), (I,), (I,), (H,))
        p = [rand(gen, *s, std=0.1).cuda().requires_grad_() for s in shapes]
        dy = rand(gen, T, H).cuda()

        def step():
            y = vb.linear(vb.gated_ffn(*p, residual=p[0]), p[1], p[4], activation="silu")
            return [y, *torch.autograd.grad(y.float().square().sum(), p)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for k in range(2):
            with torch.no_grad():
                p[0].copy_(rand(gen, T, H, std=0.1 * (k + 1)))
            graph.replay()
            torch.cuda.synchronize()
            captured = [t.detach().clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(captured, step()))
        del graph, out, dy


def test_two_streams_and_two_threads():
    """Calls at the same time, each with its own workspace and context, give the same bits."""
    import threading

    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    T, H, I = 64, 1024, 2048
    sets = []
    for _ in range(2):
        p = [rand(gen, T, H), rand(gen, I, H, std=0.05), rand(gen, I, H, std=0.05),
             rand(gen, H, I, std=0.05)]
        sets.append([t.cuda() for t in p])
    alone = [vb.gated_ffn(*p) for p in sets]
    torch.cuda.synchronize()
    got = [[], []]

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[k].append(vb.gated_ffn(*sets[k]))
        s.synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(got[k]) == 20 and all(torch.equal(g, alone[k]) for g in got[k])


def test_refusals():
    import velvetoptimizer_b200 as vb
    x = torch.zeros(4, 16, device="cuda", dtype=BF16)
    w = torch.zeros(24, 16, device="cuda", dtype=BF16)
    with pytest.raises(TypeError):
        vb.linear(x.half(), w)
    with pytest.raises(TypeError):
        vb.linear(x, w.half())
    with pytest.raises(ValueError):
        vb.linear(x, w[:, :8])
    with pytest.raises(ValueError):
        vb.linear(x, w, torch.zeros(23, device="cuda", dtype=BF16))
    with pytest.raises(ValueError):
        vb.linear(x, w.cpu())
    with pytest.raises(ValueError):
        vb.linear(x, w, activation="tanh")
    with pytest.raises(ValueError):
        vb.linear(x, w, residual=torch.zeros(4, 16, device="cuda", dtype=BF16))
    with pytest.raises(TypeError):
        vb.linear(x, w, residual=torch.zeros(4, 24, device="cuda"))
    with pytest.raises(ValueError):
        vb.linear(x, torch.zeros(0, 16, device="cuda", dtype=BF16))
    with pytest.raises(ValueError):
        vb.gated_ffn(x, w, w, w.t(), activation="none")
    with pytest.raises(ValueError):
        vb.gated_ffn(x, w, w, w)
    with pytest.raises(ValueError):
        vb.gated_ffn(x, w, w[:8], w.t())


def test_gradients_have_no_gradient():
    import velvetoptimizer_b200 as vb
    for act in ("none", "silu"):
        x = torch.randn(20, 16, device="cuda", requires_grad=True)
        w = torch.randn(24, 16, device="cuda", requires_grad=True)
        y = vb.linear(x, w, activation=act)
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated"):
            g.square().sum().backward()


def test_changed_input_is_noticed():
    import velvetoptimizer_b200 as vb
    x = torch.randn(20, 16, device="cuda", dtype=BF16).requires_grad_()
    w = torch.randn(24, 16, device="cuda", dtype=BF16).requires_grad_()
    y = vb.linear(x, w, activation="silu")
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_backward_twice():
    import velvetoptimizer_b200 as vb
    x = torch.randn(20, 16, device="cuda", dtype=BF16).requires_grad_()
    ws = [torch.randn(s, device="cuda", dtype=BF16).requires_grad_() for s in ((24, 16), (24, 16), (16, 24))]
    for y, ps in ((vb.linear(x, ws[0], activation="silu"), (x, ws[0])), (vb.gated_ffn(x, *ws), (x, *ws))):
        dy = torch.randn_like(y)
        a = torch.autograd.grad(y, ps, dy, retain_graph=True)
        b = torch.autograd.grad(y, ps, dy)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, ps, dy)


def test_first_call_of_a_thread_inside_a_capture():
    """A new thread's first call makes its context: nothing in that may disturb a capture."""
    import threading

    import velvetoptimizer_b200 as vb
    x = torch.randn(40, 64, device="cuda").to(BF16)
    w = torch.randn(48, 64, device="cuda").to(BF16)
    want = vb.linear(x, w)
    torch.cuda.synchronize()
    got, failed = [], []

    def work():
        try:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = vb.linear(x, w)
            graph.replay()
            torch.cuda.synchronize()
            got.append(y.clone())
        except Exception as e:
            failed.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not failed and torch.equal(got[0], want)


def test_traced():
    """Under a tracer the registered ops run, with the eager path's results and gradients."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    p = [rand(gen, 40, 64), rand(gen, 72, 64, std=0.1), rand(gen, 72, 64, std=0.1),
         rand(gen, 64, 72, std=0.1), rand(gen, 72)]
    p = [t.cuda().requires_grad_() for t in p]
    dy = rand(gen, 40, 72).cuda()

    def fn(x, wg, wu, wd, b):
        return vb.linear(vb.gated_ffn(x, wg, wu, wd, b, residual=x), wg, b, activation="silu")

    traced = torch.compile(fn, backend="aot_eager", fullgraph=True)
    y, t = fn(*p), traced(*p)
    assert torch.equal(y, t)
    for a, b in zip(torch.autograd.grad(y, p, dy), torch.autograd.grad(t, p, dy)):
        assert torch.equal(a, b)


def test_errors_of_the_library_surface():
    """A status of the C ABI arrives as VmoeError with its text."""
    from velvetoptimizer_b200 import _lib
    from velvetoptimizer_b200.dense import ops_for
    o = ops_for(torch.device("cuda"))
    d = _lib.VmoeLinear(4, 8, 8, 8, 8, 8, _lib.VMOE_BF16, 9, 0.1, _lib.VMOE_BF16)
    import ctypes
    with pytest.raises(_lib.VmoeError, match="unknown activation"):
        o.check(o.lib.vmoe_linear_workspace_size(o.ptr, d, 0, ctypes.c_size_t()), "size")


@pytest.mark.parametrize("change,code", [
    (dict(tokens=-1), 1), (dict(in_features=0), 1), (dict(out_features=0), 1), (dict(ldx=7), 1),
    (dict(ldw=7), 1), (dict(dtype=2), 1), (dict(activation=5), 1), (dict(grad_dtype=3), 1),
    (dict(gamma=float("nan"), activation=4), 1), (dict(tokens=1 << 31), 1)])
def test_abi_refusals(change, code):
    import ctypes

    from velvetoptimizer_b200 import _lib
    from velvetoptimizer_b200.dense import ops_for
    o = ops_for(torch.device("cuda"))
    base = dict(tokens=4, in_features=8, out_features=8, ldx=8, ldw=8, ldr=8, dtype=_lib.VMOE_BF16,
                activation=0, gamma=0.1, grad_dtype=_lib.VMOE_BF16)
    d = _lib.VmoeLinear(**{**base, **change})
    n = ctypes.c_size_t()
    assert o.lib.vmoe_linear_workspace_size(o.ptr, d, 0, n) == code
    x = torch.zeros(64, device="cuda", dtype=BF16)
    p = x.data_ptr()
    assert o.lib.vmoe_linear_forward(o.ptr, d, p, p, None, None, p, None, None, 0, None) == code


def test_abi_pointer_refusals():
    import ctypes

    from velvetoptimizer_b200 import _lib
    from velvetoptimizer_b200.dense import ops_for
    o = ops_for(torch.device("cuda"))
    bf = _lib.VMOE_BF16
    d = _lib.VmoeLinear(40, 64, 64, 64, 64, 64, bf, 0, 0.1, bf)
    buf = torch.zeros(1 << 20, device="cuda", dtype=torch.uint8)
    p = buf.data_ptr()
    ws = p + (1 << 19)
    n = ctypes.c_size_t()
    f, b = o.lib.vmoe_linear_forward, o.lib.vmoe_linear_backward
    assert f(o.ptr, d, None, p, None, None, p, None, ws, 1 << 19, None) == 1   # no x
    assert f(o.ptr, d, p, None, None, None, p, None, ws, 1 << 19, None) == 1   # no weight
    assert f(o.ptr, d, p, p, None, None, None, None, ws, 1 << 19, None) == 1   # no y
    assert f(o.ptr, d, p + 2, p, None, None, p, None, ws, 1 << 19, None) == 1  # unaligned x
    assert f(o.ptr, d, p + 1, p, None, None, p, None, ws, 1 << 19, None) == 1
    # 400 rows: the bias gradient's partial sums need a workspace (40 rows need none)
    d = _lib.VmoeLinear(400, 64, 64, 64, 64, 64, bf, 0, 0.1, bf)
    assert o.lib.vmoe_linear_workspace_size(o.ptr, d, 1, n) == 0 and n.value > 0
    args = (p, p, None, p, 64, p, p, p)
    assert b(o.ptr, d, *args, None, 0, None) == _lib.VMOE_ERR_WORKSPACE
    assert b(o.ptr, d, *args, ws, n.value - 1, None) == _lib.VMOE_ERR_WORKSPACE
    assert b(o.ptr, d, *args, ws + 16, n.value, None) == _lib.VMOE_ERR_WORKSPACE
    assert b(o.ptr, d, p, p, None, p, 65, p, p, p, ws, n.value, None) == 1     # a pitch it cannot read
    act = _lib.VmoeLinear(400, 64, 64, 64, 64, 64, bf, 2, 0.1, bf)
    assert o.lib.vmoe_linear_workspace_size(o.ptr, act, 1, n) == 0
    assert b(o.ptr, act, *args, ws, n.value, None) == 1                        # no z
    ffn = _lib.VmoeGatedFfn(40, 64, 64, 64, 64, bf, 4, 0.1, bf)
    w = _lib.VmoeFfnWeights(p, p, p)
    s = ctypes.c_size_t()
    assert o.lib.vmoe_gated_ffn_workspace_size(o.ptr, ffn, 0, n, s) == 0 and s.value > 0
    g = o.lib.vmoe_gated_ffn_forward
    assert g(o.ptr, ffn, p, w, None, p, None, 0, ws, n.value - 1, None) == _lib.VMOE_ERR_WORKSPACE
    assert g(o.ptr, ffn, p, w, None, p, p, s.value - 1, ws, n.value, None) == _lib.VMOE_ERR_WORKSPACE
    assert g(o.ptr, ffn, p, _lib.VmoeFfnWeights(p, None, p), None, p, None, 0, ws, n.value, None) == 1
    torch.cuda.synchronize()
    assert not buf.any()  # nothing ran


def module_inputs(dtype, wdtype, T=50, H=72, I=104):
    from velvetoptimizer_b200 import FeedForward, MoEConfig
    torch.manual_seed(0)
    m = FeedForward(MoEConfig(hidden_size=H, intermediate_size=I, flylora_rank=4, flylora_alpha=8.0))
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn_like(p) * (0.2 if p.dim() == 1 else p.shape[1] ** -0.5))
    m = m.cuda().to(wdtype)
    x = torch.randn(2, T // 2, H).to(dtype).cuda()
    return m, x, torch.randn(2, T // 2, H).to(dtype).cuda()


@pytest.mark.parametrize("dtype,wdtype", [(BF16, F32), (BF16, BF16), (F32, F32)])
def test_feed_forward_trains(dtype, wdtype):
    """FeedForward's gradients, the FlyLoRA factors' among them, against 64-bit autograd of the
    unfolded branch.  Norm-wise: the rounding of the folded weight, of g and u, of dg and du (or
    h), and of the gradient: five."""
    m, x, dy = module_inputs(dtype, wdtype)
    r = torch.randn_like(x)
    lx = x.clone().requires_grad_()
    y = m(lx, residual=r)
    grads = torch.autograd.grad(y, [lx, *m.parameters()], dy)

    def fly(p, v):
        q = dict(p)
        base = v @ q["base.weight"].t() + q["base.bias"]
        low = v @ q["lora_down.weight"].t() + q["lora_down.bias"]
        return base + 2.0 * (low @ q["lora_up.weight"].t() + q["lora_up.bias"])

    import copy
    ref64 = copy.deepcopy(m).double().cpu()
    v = x.double().cpu().requires_grad_()
    g = fly(ref64.gate_proj.named_parameters(), v)
    u = fly(ref64.up_proj.named_parameters(), v)
    out = r.double().cpu() + ref64.down_proj(ref.act(g, "era", GAMMA) * u)
    want = torch.autograd.grad(out, [v, *ref64.parameters()], dy.double().cpu())
    limit = 5 * 2.0 ** -8 if BF16 in (dtype, wdtype) else 1e-5
    names = ["x"] + [n for n, _ in m.named_parameters()]
    for n, a, b in zip(["y"] + names, [y.detach(), *grads], [out.detach(), *want]):
        assert a.dtype == (dtype if n in ("x", "y") else wdtype)
        rel = float((a.double().cpu() - b).norm() / b.norm())
        assert rel <= limit, (n, rel)


def test_feed_forward_f32_is_forward_only():
    m, x, _ = module_inputs(F32, F32)
    with pytest.warns(UserWarning, match="no gradient"):
        y = m(x)
    assert not y.requires_grad
    with torch.no_grad():
        assert torch.equal(y, m(x))


def test_feed_forward_without_gradients_is_unchanged():
    """Under no_grad the packed path runs, and agrees with the training path."""
    m, x, _ = module_inputs(BF16, F32)
    with torch.no_grad():
        a = m(x)
    assert len(m._packed) == 1
    b = m(x)
    assert b.requires_grad and not a.requires_grad
    # two roundings each (h and out), and the packed path's tanh.approx (2^-11)
    assert float((a.float() - b.float()).norm() / a.float().norm()) <= 4 * 2.0 ** -8


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_flylora_linear_alone(dtype):
    from velvetoptimizer_b200 import FlyLoRALinear
    torch.manual_seed(0)
    m = FlyLoRALinear(40, 56, rank=4, alpha=8.0).cuda()
    with torch.no_grad():
        m.lora_up.weight.normal_(std=0.1)
    x = torch.randn(3, 7, 40, device="cuda").to(dtype)
    r = torch.randn(3, 7, 56, device="cuda").to(dtype)
    y = m(x, residual=r, activation="silu")
    d = lambda t: t.detach().double()  # noqa: E731
    z = d(x) @ d(m.base.weight).t() + d(m.base.bias) + 2.0 * (
        (d(x) @ d(m.lora_down.weight).t() + d(m.lora_down.bias)) @ d(m.lora_up.weight).t()
        + d(m.lora_up.bias))
    want = d(r) + z * torch.sigmoid(z)
    # the folded weight and the result rounded
    limit = 2 * 2.0 ** -8 if dtype == BF16 else 1e-6
    assert float((d(y) - want).norm() / want.norm()) <= limit
    y.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


def test_training_steps_together():
    """The operators as a step uses them: block, projection, backward, clipping, update; the
    clipped gradients against the same step in 64 bits."""
    import copy

    import velvetoptimizer_b200 as vb
    m, x, dy = module_inputs(BF16, F32)
    head = vb.FlyLoRALinear(72, 40, rank=4, alpha=8.0).cuda()
    with torch.no_grad():
        head.lora_up.weight.normal_(std=0.1)
    ps = [*m.parameters(), *head.parameters()]
    opt = torch.optim.SGD(ps, lr=0.1)
    for step in range(2):
        ref_m, ref_h = copy.deepcopy(m).double().cpu(), copy.deepcopy(head).double().cpu()
        opt.zero_grad()
        y = head(m(x, residual=x), activation="gelu_tanh")
        y.float().square().mean().backward()
        norm = vb.clip_grad_norm_(ps, 0.05)

        def eff(q):
            return (q.base.weight + 2.0 * q.lora_up.weight @ q.lora_down.weight,
                    q.base.bias + 2.0 * (q.lora_up.weight @ q.lora_down.bias + q.lora_up.bias))

        v = x.double().cpu()
        (gw, gb), (uw, ub), (hw, hb) = eff(ref_m.gate_proj), eff(ref_m.up_proj), eff(ref_h)
        h = ref.act(v @ gw.t() + gb, "era", GAMMA) * (v @ uw.t() + ub)
        out = ref.act((v + ref_m.down_proj(h)) @ hw.t() + hb, "gelu_tanh", GAMMA)
        rp = [*ref_m.parameters(), *ref_h.parameters()]
        want = torch.autograd.grad(out.square().mean(), rp)
        n64 = math.sqrt(sum(float(g.square().sum()) for g in want))
        # ten roundings lie between the inputs and a gradient: weights, g, u, h, y (twice: the
        # loss's gradient squares it), z, dz, dg, and the block's output
        assert abs(float(norm) - n64) <= 10 * 2.0 ** -8 * n64
        for p, g in zip(ps, want):
            g = g * min(1.0, 0.05 / (n64 + 1e-6))
            assert float((p.grad.double().cpu() - g).norm()) <= 11 * 2.0 ** -8 * float(g.norm()) + 1e-9
        opt.step()


def test_device_status_clean():
    from velvetoptimizer_b200.dense import _native
    torch.cuda.synchronize()
    assert _native().device_status(torch.zeros(1, device="cuda")) == 0
