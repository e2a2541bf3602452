"""GPU: grad_norm and clip_grad_norm_ against 64-bit sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def params(gen, shapes, dtypes, std=1.0):
    ps = []
    for s, d in zip(shapes, dtypes):
        p = torch.nn.Parameter(torch.zeros(s, device="cuda", dtype=d))
        p.grad = (torch.randn(s, generator=gen) * std).to(d).cuda()
        ps.append(p)
    return ps


def norm64(ts, p):
    flat = torch.cat([t.detach().double().cpu().reshape(-1) for t in ts]) if ts else torch.zeros(0)
    if flat.numel() == 0:
        return 0.0
    return float(flat.abs().max()) if p == math.inf else float((flat.abs() ** p).sum() ** (1 / p))


def check_clip(ps, max_norm, p=2.0):
    """The norm is one rounding to fp32 off its 64-bit value (the fp64 sums' error is far below);
    a scaled gradient is off by the factor's rounding and its own, 2^-24 + u."""
    import velvetoptimizer_b200 as vb
    before = [q.grad.detach().clone() for q in ps]
    want = norm64(before, p)
    norm = vb.clip_grad_norm_(ps, max_norm, p)
    assert norm.dtype == F32 and norm.shape == () and norm.is_cuda
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    coef = min(1.0, max_norm / (want + 1e-6))
    for q, b in zip(ps, before):
        if coef == 1.0:
            assert torch.equal(q.grad, b)
            continue
        ref = b.double().cpu() * coef
        err = (q.grad.double().cpu() - ref).abs()
        # below the smallest normal number the rounding is absolute
        assert (err <= (U[b.dtype] + 2.0 ** -23) * ref.abs() + torch.finfo(b.dtype).tiny * U[b.dtype] * 2).all()


SIZES = [1, 2, 3, 7, 8, 9, 31, 63, 255, 257, 4095, 4096, 4097, 8191, 8192, 8193, 12345, 100003]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("clipped", [True, False])
def test_sizes(dtype, p, clipped):
    gen = torch.Generator().manual_seed(0)
    for n in SIZES:
        ps = params(gen, [(n,)], [dtype])
        check_clip(ps, norm64([ps[0].grad], p) * (0.3 if clipped else 3.0), p)
    ps = params(gen, [(n,) for n in SIZES], [dtype] * len(SIZES))
    check_clip(ps, 1.0 if clipped else 1e9, p)


@pytest.mark.parametrize("first", range(1, 9))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_odd_starts(first, dtype):
    """Views into one buffer from any element on; what lies around them stays as it was."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(first)
    sizes = [5, 4099, 1, 17, 20000, 3]
    flat = torch.randn(first + sum(sizes) + 2 * len(sizes) + 9, generator=gen).to(dtype).cuda()
    was = flat.clone()
    at, views = first, []
    for s in sizes:
        views.append(flat[at:at + s])
        at += s + 2
    want = norm64(views, 2.0)
    assert abs(float(vb.grad_norm(views)) - want) <= 2.0 ** -23 * want
    assert torch.equal(flat, was)
    ps = [torch.nn.Parameter(torch.zeros_like(v)) for v in views]
    for q, v in zip(ps, views):
        q.grad = v
    vb.clip_grad_norm_(ps, want / 2)
    inside = torch.zeros_like(flat, dtype=torch.bool)
    at = first
    for s in sizes:
        inside[at:at + s] = True
        at += s + 2
    assert torch.equal(flat[~inside], was[~inside])
    ref = was.double() * (want / 2 / (want + 1e-6))
    assert ((flat.double() - ref).abs()[inside] <= (U[dtype] + 2.0 ** -23) * ref.abs()[inside]).all()


@pytest.mark.parametrize("n", [63, 64, 65, 1023, 1024, 1025, 2500])
def test_many_tensors(n):
    """The kernel parameters hold 64 or 1024 tensors; longer lists take several launches."""
    gen = torch.Generator().manual_seed(n)
    shapes = [(1 + (7 * i) % 50,) for i in range(n)]
    dtypes = [BF16 if i % 3 == 0 else F32 for i in range(n)]
    check_clip(params(gen, shapes, dtypes), 2.0)
    check_clip(params(gen, shapes, dtypes), 1e9)


def test_large():
    gen = torch.Generator().manual_seed(0)
    check_clip(params(gen, [(5000, 1999), (3, 1000003), (129,)], [F32, BF16, F32]), 10.0)


def test_tensor_past_32_bits():
    """Ones at the ends of a tensor of more than 2^31 elements: the norm and the factor are exact."""
    import velvetoptimizer_b200 as vb
    n = 2 ** 31 + 4099
    p = torch.nn.Parameter(torch.empty(n, device="cuda", dtype=BF16))
    p.grad = torch.zeros(n, device="cuda", dtype=BF16)
    p.grad[:2] = 1
    p.grad[-2:] = 1
    assert float(vb.clip_grad_norm_([p], 1.0)) == 2.0
    # 1 / (2 + 1e-6) rounds to 0.5 as bf16
    assert p.grad[:2].tolist() == [0.5, 0.5] and p.grad[-2:].tolist() == [0.5, 0.5]
    assert not p.grad[2:-2].any()
    del p
    torch.cuda.empty_cache()


def test_no_fp32_overflow_or_loss():
    import velvetoptimizer_b200 as vb
    for dtype, v in ((F32, 1e30), (BF16, 1e30), (F32, 1e-30)):
        t = torch.full((1000,), v, device="cuda", dtype=dtype)
        want = norm64([t], 2.0)
        assert abs(float(vb.grad_norm([t])) - want) <= 2.0 ** -23 * want
    # 2^25 equal terms: a single fp32 sum would stop at 2^24
    t = torch.ones(1 << 25, device="cuda")
    assert float(vb.grad_norm([t], 1)) == float(1 << 25)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_non_finite(bad, p):
    import velvetoptimizer_b200 as vb
    for dtype in (F32, BF16):
        for where in (0, 777, 4999):
            t = torch.ones(5000, device="cuda", dtype=dtype)
            t[where] = bad
            q = torch.nn.Parameter(torch.zeros_like(t))
            q.grad = t.clone()
            other = torch.nn.Parameter(torch.zeros(4, device="cuda"))
            other.grad = torch.ones(4, device="cuda")
            with pytest.raises(RuntimeError):
                vb.clip_grad_norm_([q, other], 1.0, p, error_if_nonfinite=True)
            assert torch.equal(q.grad.nan_to_num(7.0), t.nan_to_num(7.0))
            norm = float(vb.clip_grad_norm_([q, other], 1.0, p))
            if math.isnan(bad):
                assert math.isnan(norm) and q.grad.isnan().all() and other.grad.isnan().all()
            else:
                assert norm == math.inf
                assert q.grad[where].isnan() and int(q.grad.isnan().sum()) == 1
                assert not other.grad.any()


def test_zero_and_empty():
    import velvetoptimizer_b200 as vb
    z = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    z.grad = torch.zeros_like(z)
    assert float(vb.clip_grad_norm_([z], 1.0)) == 0.0 and not z.grad.any()
    e = torch.nn.Parameter(torch.zeros(0, 5, device="cuda"))
    e.grad = torch.zeros_like(e)
    assert float(vb.clip_grad_norm_([e], 1.0)) == 0.0
    assert float(vb.clip_grad_norm_([e, z], 1.0, math.inf)) == 0.0
    none = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert float(vb.clip_grad_norm_([none], 1.0)) == 0.0
    one = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    one.grad = torch.full((3,), 2.0, device="cuda")
    assert float(vb.clip_grad_norm_(iter([none, one, e]), 0.0)) == pytest.approx(math.sqrt(12))
    assert not one.grad.any()


def test_shared_gradients_count_once():
    import velvetoptimizer_b200 as vb
    p = torch.nn.Parameter(torch.zeros(1000, device="cuda"))
    p.grad = torch.ones_like(p)
    q = torch.nn.Parameter(torch.zeros(1000, device="cuda"))
    q.grad = p.grad
    assert float(vb.clip_grad_norm_([p, q, p], 1.0)) == pytest.approx(math.sqrt(1000))
    assert torch.allclose(p.grad, torch.full_like(p.grad, 1 / math.sqrt(1000)))
    flat = torch.ones(100, device="cuda")
    with pytest.raises(ValueError):
        vb.grad_norm([flat[:60], flat[50:]])
    with pytest.raises(ValueError):
        vb.grad_norm([flat, flat[:60]])


def test_strides():
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    base = torch.randn(40, 60, generator=gen).cuda()
    p = torch.nn.Parameter(torch.zeros(60, 40, device="cuda"))
    p.grad = base.t()                      # dense in another order
    q = torch.nn.Parameter(torch.zeros(40, 20, device="cuda"))
    wide = torch.randn(40, 60, generator=gen).cuda()
    was = wide.clone()
    q.grad = wide[:, 10:30]                # rows with gaps
    check_clip([p, q], 1.0)
    assert torch.equal(wide[:, :10], was[:, :10]) and torch.equal(wide[:, 30:], was[:, 30:])
    e = torch.randn(1, 60, generator=gen).cuda().expand(40, 60)
    want = norm64([e], 2.0)
    assert abs(float(vb.grad_norm(e)) - want) <= 2.0 ** -23 * want
    r = torch.nn.Parameter(torch.zeros(40, 60, device="cuda"))
    r.grad = e
    with pytest.raises(ValueError):
        vb.clip_grad_norm_(r, 1.0)


def test_captured_and_same_bits():
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    shapes = [(257, 129)] * 70 + [(3,)] * 30
    ps = params(gen, shapes, [F32, BF16] * 50)
    fresh = [q.grad.clone() for q in ps]

    def step():
        for q, f in zip(ps, fresh):
            q.grad.copy_(f)
        return vb.clip_grad_norm_(ps, 1.0)

    first = float(step())
    want = [q.grad.clone() for q in ps]
    for _ in range(3):
        assert float(step()) == first
        assert all(torch.equal(q.grad, w) for q, w in zip(ps, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step()
    for _ in range(2):
        for f in fresh:
            f.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        got = [q.grad.clone() for q in ps]
        n = float(norm)
        assert float(step()) == n and all(torch.equal(g, q.grad) for g, q in zip(got, ps))


def test_scaling_counts_as_a_change():
    import velvetoptimizer_b200 as vb
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    p.grad = torch.ones(8, device="cuda")
    v = p.grad._version
    vb.grad_norm([p.grad])
    assert p.grad._version == v
    vb.clip_grad_norm_([p], 0.5)
    assert p.grad._version > v


def test_refusals():
    import velvetoptimizer_b200 as vb
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    p.grad = torch.ones_like(p)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            vb.clip_grad_norm_([p], bad)
    with pytest.raises(ValueError):
        vb.clip_grad_norm_([p], 1.0, 3.0)
    with pytest.raises(TypeError):
        vb.grad_norm([torch.zeros(3, device="cuda", dtype=torch.float16)])
    with pytest.raises(RuntimeError):
        vb.grad_norm([torch.zeros(3)])
    assert torch.equal(p.grad, torch.ones_like(p))


def test_layer_step():
    """A mixture layer's gradients, as its training loop clips them."""
    import velvetoptimizer_b200 as vb
    torch.manual_seed(0)
    layer = vb.MoELayer(vb.MoEConfig(hidden_size=64, intermediate_size=128, moe_num_experts=4)).cuda()
    x = torch.randn(2, 40, 64, device="cuda", dtype=BF16)
    out, aux = layer(x)
    (out.float().square().mean() + 0.01 * aux).backward()
    ps = list(layer.parameters())
    check_clip([q for q in ps if q.grad is not None], 1e-3)


def test_shared_gradients_that_are_not_dense_count_once():
    """Row-gapped, transposed and strided gradients that several parameters share."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    for dtype in (F32, BF16):
        for cut in (lambda w: w[:, 10:30], lambda w: w[:, ::2], lambda w: w[::3, 1:]):
            wide = torch.randn(40, 60, generator=gen).to(dtype).cuda()
            was, g = wide.clone(), cut(wide)
            want = norm64([g], 2.0)
            assert float(vb.grad_norm([g, g])) == pytest.approx(want, rel=2.0 ** -22)
            ps = [torch.nn.Parameter(torch.zeros_like(g)) for _ in range(3)]
            for q in ps[:2]:
                q.grad = g
            ps[2] = torch.nn.Parameter(torch.zeros_like(g.t()))
            ps[2].grad = g.t()
            norm = vb.clip_grad_norm_([*ps, ps[0]], want / 2)
            assert float(norm) == pytest.approx(want, rel=2.0 ** -22)
            ref = cut(was).double() * (0.5 * want / (want + 1e-6))
            assert ((g.double() - ref).abs() <= (U[dtype] + 2.0 ** -22) * ref.abs()).all()
            outside = torch.ones_like(wide, dtype=torch.bool)
            cut(outside)[:] = False
            assert torch.equal(wide[outside], was[outside])


def test_overlapping_gradients_that_are_not_dense_are_refused():
    import velvetoptimizer_b200 as vb
    wide = torch.ones(40, 60, device="cuda")
    for a, b in ((wide, wide[:, 10:30]), (wide[:, :20], wide[:, 19:40]), (wide[::2], wide[30:]),
                 (wide[:, ::2], wide[:, ::3]), (wide[:, 10:30], wide[5])):
        for pair in ((a, b), (b, a)):
            with pytest.raises(ValueError, match="overlap"):
                vb.grad_norm(list(pair))
            ps = [torch.nn.Parameter(torch.zeros_like(t)) for t in pair]
            for q, t in zip(ps, pair):
                q.grad = t
            with pytest.raises(ValueError, match="overlap"):
                vb.clip_grad_norm_(ps, 1.0)
    assert (wide == 1).all()
    # apart, however they interleave
    parts = [wide[:, :10], wide[:, 10:30], wide[:, 30::2], wide[:, 31::2]]
    assert float(vb.grad_norm(parts)) == pytest.approx(math.sqrt(2400))
    ps = [torch.nn.Parameter(torch.zeros_like(t)) for t in parts]
    for q, t in zip(ps, parts):
        q.grad = t
    vb.clip_grad_norm_(ps, 1.0)
    assert torch.allclose(wide, torch.full_like(wide, 1 / math.sqrt(2400)))


def test_expanded_tensors_count_once():
    """The same expansion twice is one tensor; another one of the same memory overlaps it."""
    import velvetoptimizer_b200 as vb
    row = torch.randn(1, 60, device="cuda")
    e = row.expand(40, 60)
    want = norm64([e], 2.0)
    assert float(vb.grad_norm([e, e, row.expand(40, 60)])) == pytest.approx(want, rel=2.0 ** -22)
    for other in (row.expand(10, 60), row):
        with pytest.raises(ValueError, match="overlap"):
            vb.grad_norm([e, other])
