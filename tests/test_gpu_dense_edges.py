"""GPU: linear, gated_ffn and the gradient norm at the edges: row ends, non-finite values, tangents,
tracers, status words, refusals of the C ABI."""
import ctypes

import pytest
import torch

from tests import dense_ref as ref
from tests.test_gpu_dense import BF16, F32, GAMMA, d64, leaf, rand, run_ffn, run_linear

pytestmark = pytest.mark.gpu


# fp32 gradients of a bf16 call, at row lengths that end inside 8 columns: multiples of 4, and not
@pytest.mark.parametrize("T", [5, 90, 300])
@pytest.mark.parametrize("K,N", [(4, 24), (12, 40), (100, 36), (1004, 260), (260, 1004), (10, 6),
                                 (101, 7)])
def test_linear_f32_gradients_at_row_ends(T, K, N):
    run_linear(T, K, N, act="silu", dtype=BF16, wdtype=F32, seed=T + K)


@pytest.mark.parametrize("T", [5, 90, 300])
@pytest.mark.parametrize("H,I", [(12, 40), (40, 12), (100, 36), (1004, 260), (260, 1004), (10, 6)])
def test_gated_ffn_f32_gradients_at_row_ends(T, H, I):
    run_ffn(T, H, I, dtype=BF16, wdtype=F32, seed=T + H)


def ops():
    from velvetoptimizer_b200 import _lib
    return _lib, _lib.Ops(torch.cuda.current_device())


GUARD = 64


class Guarded:
    """A buffer of n elements with words after it that must stay as they are."""

    def __init__(self, shape, dtype):
        self.n = 1
        for s in shape:
            self.n *= s
        self.buf = torch.full((self.n + GUARD,), 7.0, device="cuda", dtype=dtype)
        self.t = self.buf[:self.n].view(shape)

    def ptr(self):
        return self.buf.data_ptr()

    def check(self):
        assert (self.buf[self.n:] == 7.0).all()


@pytest.mark.parametrize("T", [5, 90, 300])
@pytest.mark.parametrize("K,N", [(100, 36), (4, 260), (1004, 12), (9, 5)])
def test_nothing_is_written_past_the_gradients(T, K, N):
    """What lies behind dW, db and dx keeps its value (linear through the C ABI)."""
    _lib, o = ops()
    gen = torch.Generator().manual_seed(T)
    bf = _lib.VMOE_BF16
    x, w, dy = rand(gen, T, K).cuda(), rand(gen, N, K).cuda(), rand(gen, T, N).cuda()
    d = _lib.VmoeLinear(T, K, N, K, K, N, bf, 0, 0.1, _lib.VMOE_F32)
    n = ctypes.c_size_t()
    o.check(o.lib.vmoe_linear_workspace_size(o.ptr, d, 1, n), "size")
    ws = torch.empty(n.value + 256, device="cuda", dtype=torch.uint8)
    dx, dw, db = Guarded((T, K), BF16), Guarded((N, K), F32), Guarded((N,), F32)
    stream = torch.cuda.current_stream().cuda_stream
    o.check(o.lib.vmoe_linear_backward(o.ptr, d, x.data_ptr(), w.data_ptr(), None, dy.data_ptr(), N,
                                       dx.ptr(), dw.ptr(), db.ptr(), ws.data_ptr(), n.value,
                                       stream), "backward")
    torch.cuda.synchronize()
    want = ref.linear(d64(x), d64(w), None, None, d64(dy), "none", GAMMA, BF16, F32)
    for name, g in (("dx", dx), ("dw", dw), ("db", db)):
        g.check()
        ref.check(name, g.t, *want[name], 3, BF16)


@pytest.mark.parametrize("T", [5, 90, 300])
@pytest.mark.parametrize("H,I", [(100, 36), (36, 100), (12, 260)])
def test_nothing_is_written_past_the_blocks_gradients(T, H, I):
    _lib, o = ops()
    gen = torch.Generator().manual_seed(T)
    bf = _lib.VMOE_BF16
    x, dy = rand(gen, T, H).cuda(), rand(gen, T, H).cuda()
    w = [rand(gen, *s, std=s[1] ** -0.5).cuda() for s in ((I, H), (I, H), (H, I))]
    d = _lib.VmoeGatedFfn(T, H, I, H, H, bf, 2, 0.1, _lib.VMOE_F32)
    n, s = ctypes.c_size_t(), ctypes.c_size_t()
    o.check(o.lib.vmoe_gated_ffn_workspace_size(o.ptr, d, 1, n, s), "size")
    m = ctypes.c_size_t()
    o.check(o.lib.vmoe_gated_ffn_workspace_size(o.ptr, d, 0, m, None), "size")
    ws = torch.empty(max(n.value, m.value) + 256, device="cuda", dtype=torch.uint8)
    saved = torch.empty(s.value, device="cuda", dtype=torch.uint8)
    y = Guarded((T, H), BF16)
    shapes = dict(dx=(T, H), dwg=(I, H), dwu=(I, H), dwd=(H, I), dbg=(I,), dbu=(I,), dbd=(H,))
    g = {k: Guarded(v, BF16 if k == "dx" else F32) for k, v in shapes.items()}
    stream = torch.cuda.current_stream().cuda_stream
    vw = _lib.VmoeFfnWeights(*[t.data_ptr() for t in w])
    vg = _lib.VmoeFfnGrads(*[g[k].ptr() for k in ("dwg", "dwu", "dwd", "dbg", "dbu", "dbd")])
    o.check(o.lib.vmoe_gated_ffn_forward(o.ptr, d, x.data_ptr(), vw, None, y.ptr(), saved.data_ptr(),
                                         s.value, ws.data_ptr(), m.value, stream), "forward")
    o.check(o.lib.vmoe_gated_ffn_backward(o.ptr, d, x.data_ptr(), vw, dy.data_ptr(), H, g["dx"].ptr(),
                                          vg, saved.data_ptr(), s.value, ws.data_ptr(), n.value,
                                          stream), "backward")
    torch.cuda.synchronize()
    want = ref.gated_ffn(d64(x), *map(d64, w), None, None, None, None, d64(dy), "silu", GAMMA, BF16, F32)
    for name, t in (("y", y), *g.items()):
        t.check()
        ref.check(name, t.t, *want[name], 2, BF16)


def test_abi_refuses_addresses_between_elements():
    """Every operand that is read or written by elements is refused when it starts between two."""
    _lib, o = ops()
    buf = torch.zeros(1 << 20, device="cuda", dtype=torch.uint8)
    p, ws, n = buf.data_ptr(), buf.data_ptr() + (1 << 19), 1 << 19
    bad = _lib.VMOE_ERR_INVALID_ARG
    for dtype, elt, gdtype in ((_lib.VMOE_BF16, 2, _lib.VMOE_F32), (_lib.VMOE_F32, 4, _lib.VMOE_F32)):
        for T in (0, 4, 40):
            d = _lib.VmoeLinear(T, 64, 64, 64, 64, 64, dtype, 2, 0.1, gdtype)
            f = [p, p, p, p, p, p]                       # x, w, bias, residual, y, z
            for i in range(2, 6):
                a = list(f)
                a[i] += elt // 2
                if T:
                    assert o.lib.vmoe_linear_forward(o.ptr, d, *a, ws, n, None) == bad, (dtype, i)
            for i in range(6):                           # x, w, z, dy | lddy | dx, dw, db
                a = [p, p, p, p, 64, p, p, p]
                at = (2, 3, 5, 6, 7, 0)[i]
                a[at] += 2 if at in (6, 7) else elt // 2
                if T or at > 4:
                    assert o.lib.vmoe_linear_backward(o.ptr, d, *a, ws, n, None) == bad, (dtype, at)
            e = _lib.VmoeGatedFfn(T, 64, 64, 64, 64, dtype, 2, 0.1, gdtype)
            w = [p] * 6
            for i in (3, 4, 5, 6, 7):                    # biases, residual, y
                a, q = list(w), [p, p]
                if i < 6:
                    a[i] += elt // 2
                else:
                    q[i - 6] += elt // 2
                if T:
                    assert o.lib.vmoe_gated_ffn_forward(o.ptr, e, p, _lib.VmoeFfnWeights(*a), q[0], q[1],
                                                        None, 0, ws, n, None) == bad, (dtype, i)
            for i in range(7):                           # gradients, dx
                a, dx = list(w), p
                if i < 6:
                    a[i] += 2
                else:
                    dx += elt // 2
                assert o.lib.vmoe_gated_ffn_backward(
                    o.ptr, e, p, _lib.VmoeFfnWeights(*w), p, 64, dx, _lib.VmoeFfnGrads(*a), p, n, ws, n,
                    None) == bad, (dtype, i)
    ptrs, counts = (ctypes.c_void_p * 1)(p), (ctypes.c_int64 * 1)(8)
    types = (ctypes.c_int32 * 1)(_lib.VMOE_F32)
    assert o.lib.vmoe_grad_norm(o.ptr, ptrs, counts, types, 1, 2, 1.0, p + 2, ws, n, None) == bad
    torch.cuda.synchronize()
    assert not buf.any()  # nothing ran


@pytest.mark.parametrize("dtype", [0, 1])
def test_sizes_past_64_bits_are_refused(dtype):
    """Sizes whose workspace would not fit 64 bits: refused, never a small number."""
    _lib, o = ops()
    n, s, big = ctypes.c_size_t(), ctypes.c_size_t(), (1 << 31) - 1
    for T, K, N in ((big, big, 8), (big, 8, big), (8, big, big), (big, big, big), (1 << 20, (1 << 20) + 1, 8)):
        d = _lib.VmoeLinear(T, K, N, K, K, N, dtype, 2, 0.1, dtype)
        e = _lib.VmoeGatedFfn(T, K, N, K, K, dtype, 2, 0.1, dtype)
        for backward in (0, 1):
            assert o.lib.vmoe_linear_workspace_size(o.ptr, d, backward, n) == _lib.VMOE_ERR_UNSUPPORTED_SHAPE
            assert o.lib.vmoe_gated_ffn_workspace_size(o.ptr, e, backward, n, s) == _lib.VMOE_ERR_UNSUPPORTED_SHAPE
    T, I = 1 << 20, 1 << 20  # the largest: its sizes are what the formulas give
    e = _lib.VmoeGatedFfn(T, 8, I, 8, 8, dtype, 2, 0.1, dtype)
    assert o.lib.vmoe_gated_ffn_workspace_size(o.ptr, e, 1, n, s) == 0
    elt = 2 if dtype == _lib.VMOE_BF16 else 4
    assert s.value == T * I * (8 + elt) and n.value > 2 * T * I * elt


@pytest.mark.parametrize("T", [5, 33, 300, 4001])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_bias_sums_take_in_real_rows_alone(T, bad):
    """An infinite down weight makes dh infinite, not NaN, where dy has one sign: so are the gate's
    and the up's bias gradients, whatever the number of rows is in the last block of 32."""
    import velvetoptimizer_b200 as vb
    H, I = 40, 72
    x = torch.full((T, H), 0.5, device="cuda", dtype=BF16)
    wg, wu = (torch.full((I, H), 0.125, device="cuda", dtype=BF16) for _ in range(2))
    wd = torch.full((H, I), 0.25, device="cuda", dtype=BF16)
    wd[3, 7] = bad
    bg, bu = (torch.zeros(I, device="cuda", dtype=BF16).requires_grad_() for _ in range(2))
    y = vb.gated_ffn(x, wg, wu, wd, bg, bu, activation="silu")
    dbg, dbu = torch.autograd.grad(y, (bg, bu), torch.ones_like(y))
    for g in (dbg, dbu):
        assert g[7] == bad
        rest = torch.cat([g[:7], g[8:]])
        assert torch.isfinite(rest).all() and (rest > 0).all()


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_tangents_are_refused(grad, dtype, wdtype):
    """A tangent in any argument raises; without one, calls inside a dual level run as ever."""
    import torch.autograd.forward_ad as fwd

    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    lin = [rand(gen, 2, 3, 16, dtype=dtype), rand(gen, 24, 16, dtype=wdtype), rand(gen, 24, dtype=wdtype),
           rand(gen, 2, 3, 24, dtype=dtype)]
    ffn = [rand(gen, 6, 16, dtype=dtype), rand(gen, 24, 16, dtype=wdtype), rand(gen, 24, 16, dtype=wdtype),
           rand(gen, 16, 24, dtype=wdtype), rand(gen, 24, dtype=wdtype), rand(gen, 24, dtype=wdtype),
           rand(gen, 16, dtype=wdtype), rand(gen, 6, 16, dtype=dtype)]
    for fn, args in ((lambda a: vb.linear(*a[:3], residual=a[3], activation="silu"), lin),
                     (lambda a: vb.gated_ffn(*a[:7], residual=a[7]), ffn)):
        args = [t.cuda().requires_grad_(grad) for t in args]
        want = fn(args)
        with fwd.dual_level():
            assert torch.equal(fn(args), want)
            for i in range(len(args)):
                a = list(args)
                a[i] = fwd.make_dual(a[i], torch.ones_like(a[i]))
                with pytest.raises(NotImplementedError, match="tangent"):
                    fn(a)
            if grad:
                dy = fwd.make_dual(torch.ones_like(want), torch.ones_like(want))
                with pytest.raises(NotImplementedError, match="tangent"):
                    torch.autograd.grad(fn(args), args, dy)
    g = torch.ones(8, device="cuda")
    with fwd.dual_level():
        assert float(vb.grad_norm([g])) == pytest.approx(8 ** 0.5)
        with pytest.raises(NotImplementedError, match="tangent"):
            vb.grad_norm([fwd.make_dual(g, g)])


def test_tracers_record_the_registered_ops():
    """make_fx and torch.jit.trace on real tensors record the ops, not their results; a dispatch
    mode sees them; results and gradients are the eager path's."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)

    def inputs():
        return [rand(gen, 40, 64).cuda(), *(rand(gen, *s, std=0.1).cuda()
                                            for s in ((72, 64), (72, 64), (64, 72), (72,)))]

    def fn(x, wg, wu, wd, b):
        return vb.linear(vb.gated_ffn(x, wg, wu, wd, b, residual=x), wg, b, activation="silu")

    def step(*p):
        p = [t.detach().requires_grad_() for t in p]
        y = fn(*p)
        return [y, *torch.autograd.grad(y.float().sum(), p)]

    p, q = inputs(), inputs()
    for kw in (dict(), dict(tracing_mode="fake")):
        graph = make_fx(fn, **kw)(*p)
        names = [str(n.target) for n in graph.graph.nodes if "vesper_moe" in str(n.target)]
        assert [n.split(".")[1] for n in names] == ["gated_ffn_forward", "linear_forward"]
        assert torch.equal(graph(*q), fn(*q))
    graph = make_fx(step)(*p)
    names = {str(n.target).split(".")[1] for n in graph.graph.nodes if "vesper_moe" in str(n.target)}
    assert names == {f"{a}_{b}" for a in ("linear", "gated_ffn") for b in ("forward", "backward")}
    assert all(torch.equal(a, b) for a, b in zip(graph(*q), step(*q)))
    with torch.no_grad():
        traced = torch.jit.trace(fn, tuple(p))
        assert torch.equal(traced(*q), fn(*q))
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.__name__.split(".")[0])
            return func(*args, **(kwargs or {}))

    want = fn(*p)
    with Mode():
        assert torch.equal(fn(*p), want)
    assert "linear_forward" in seen and "gated_ffn_forward" in seen


class OpsHead(ctypes.Structure):
    """The beginning of struct vmoe_ops (csrc/ops_host.h)."""
    _fields_ = [("device", ctypes.c_int), ("num_sms", ctypes.c_int), ("sm100", ctypes.c_bool),
                ("status", ctypes.c_void_p)]


def test_a_wait_that_gave_up_on_another_thread_is_reported():
    """The status that a kernel of any thread's context leaves reaches every thread's question, is
    cleared by it, and is not handed on to later contexts.  The status is written from the host."""
    import threading

    import velvetoptimizer_b200 as vb
    from velvetoptimizer_b200.dense import _native
    _lib = ops()[0]
    cudart = ctypes.CDLL("libcudart.so.12")
    index = torch.cuda.current_device()

    def leave(code):
        o = _lib.Ops(index)
        head = ctypes.cast(o.ptr, ctypes.POINTER(OpsHead)).contents
        assert head.device == index and head.num_sms > 0 and head.sm100
        word = ctypes.c_int(code)
        rc = cudart.cudaMemcpy(ctypes.c_void_p(head.status), ctypes.byref(word), ctypes.c_size_t(4), 1)
        o.close()
        assert rc == 0

    x = torch.zeros(1, device="cuda")
    for ask in (vb.device_status, lambda: vb.device_status(index), lambda: vb.device_status("cuda"),
                lambda: _native().device_status(x), lambda: vb.device_status(x.device)):
        assert ask() == 0
        t = threading.Thread(target=leave, args=(0x103,))
        t.start()
        t.join()
        with pytest.raises(_lib.VmoeError, match="0x103") as e:
            ask()
        assert e.value.code == _lib.VMOE_ERR_TIMEOUT
        assert ask() == 0
    assert _lib.Ops(index).device_status(torch.cuda.current_stream().cuda_stream) == 0


def same_as_fp32(got, a, b):
    """a @ b in fp32's infinities and NaNs, every other value within its sum's bound."""
    got, want = got.detach().cpu(), a @ b
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    ok = want.isfinite()
    a64, b64 = a.double(), b.double()
    exact = (a64 @ b64)[ok]
    bound = ((a64.abs() @ b64.abs()) * (a.shape[1] + 2) * 2.0 ** -23)[ok]
    assert ((got[ok].double() - exact).abs() <= bound + 2.0 ** -24 * exact.abs()).all()


@pytest.mark.parametrize("T,K,N", [(3, 72, 40), (40, 72, 40), (300, 72, 40), (150, 200, 130),
                                   (40, 2048, 264), (17, 33, 300)])
def test_f32_products_that_overflow(T, K, N):
    """Finite operands whose products leave fp32's range: infinity, as fp32 arithmetic gives, in
    every product and beside values as exact as ever.  All terms of such a sum have one sign, so
    that it does not depend on their order."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(T)
    x, w, dy = (rand(gen, *s, dtype=F32) for s in ((T, K), (N, K), (T, N)))
    x[2], w[5] = (x[2].abs() + 0.1) * 1.5e30, (w[5].abs() + 0.1) * 1.5e30
    dy[1, 5], dy[2, 7] = 1.7e30, -1.7e30
    lx, lw = leaf(x), leaf(w)
    y = vb.linear(lx, lw)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy.cuda())
    assert float(y[2, 5]) == float("inf") and (dx[1] == float("inf")).all() and (dw[7] == -float("inf")).all()
    for got, a, b in ((y, x, w.t()), (dx, dy, w), (dw, dy.t(), x)):
        same_as_fp32(got, a, b)


@pytest.mark.parametrize("T", [3, 40, 300])
def test_f32_products_that_just_fit(T):
    """x y below fp32's largest number though the operands round, as bf16, to a product above it."""
    import velvetoptimizer_b200 as vb
    v = 2.0 ** 64 * (1 - 2.0 ** -10)
    x, w = torch.zeros(T, 40), torch.zeros(24, 40)
    x[1, 3], w[7, 3] = v, -v
    y = vb.linear(x.cuda(), w.cuda(), residual=torch.ones(T, 24, device="cuda"))
    want = torch.ones(T, 24, dtype=torch.float64)
    want[1, 7] -= v * v
    assert torch.isfinite(y).all()
    assert ((y.double().cpu() - want).abs() <= 2.0 ** -23 * want.abs()).all()


@pytest.mark.parametrize("T", [3, 40, 300])
def test_f32_gated_products_that_overflow(T):
    """An overflowing gate (one row), an overflowing dh (another) and overflowing weight gradients:
    infinite where fp32 is, the other rows as ever."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(T)
    H, I = 40, 72
    p = [rand(gen, *s, dtype=F32).abs() for s in ((T, H), (I, H), (I, H), (H, I))]
    x, wg, wu, wd = p
    dy = rand(gen, T, H, dtype=F32).abs()
    x[2] = (x[2] + 0.1) * 1.3e30
    wg[9] = (wg[9] + 0.1) * 1.5e30
    wd[3] = (wd[3] + 0.1) * 1.7e20
    dy[1, 3] = 1.9e30
    leaves = [leaf(t) for t in p]
    y = vb.gated_ffn(*leaves, activation="relu")
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    ref64 = [t.double().requires_grad_() for t in p]
    g, u = ref64[0] @ ref64[1].t(), ref64[0] @ ref64[2].t()
    want = (torch.relu(g) * u) @ ref64[3].t()
    exact = torch.autograd.grad(want, ref64, dy.double())
    inf = float("inf")
    assert (y[2] == inf).all() and (grads[0][1] == inf).all()
    big = torch.finfo(F32).max
    for name, a, b in zip(("y", "dx", "dwg", "dwu", "dwd"), (y, *grads), (want, *exact)):
        a, b = a.detach().double().cpu(), b.detach()
        over = b > big
        assert not a.isnan().any(), name
        assert (a[over] == inf).all(), name
        # far from overflow in every intermediate: rows of x and dy without large values
        rows = [i for i in range(T) if i not in (1, 2)]
        if name in ("y", "dx"):
            ok = b[rows] < 1e30
            assert ((a[rows] - b[rows])[ok].abs() <= 1e-5 * b[rows][ok]).all(), name


CAPTURE = """
import gc, torch, velvetoptimizer_b200 as vb
torch.manual_seed(0)
def leaf(*s): return torch.randn(*s, device="cuda").to(torch.bfloat16).requires_grad_()
x, w, b = leaf(40, 64), leaf(72, 64), leaf(72)
ws = [leaf(72, 64), leaf(72, 64), leaf(64, 72)]
deep = leaf(4, 10, 64)  # reaches linear through a view
cases = ((lambda: vb.linear(x, w, b, activation="silu"), [x, w, b]),
         (lambda: vb.gated_ffn(x, *ws), [x, *ws]),
         (lambda: vb.linear(deep, w), [deep, w]))
def backward(fn, ps, how):
    y = fn()
    if how == "grad":
        return torch.autograd.grad(y.float().square().sum(), ps)
    y.float().square().sum().backward()
for fn, ps in cases:
    want = backward(fn, ps, "grad")
    for how in ("grad", "backward"):
        for p in ps: p.grad = torch.zeros_like(p)
        alive = fn()
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(graph):
                backward(fn, ps, how)
            raise SystemExit("the capture was not refused")
        except RuntimeError as e:
            assert "alive" in str(e), e
        del alive, graph
        gc.collect()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = backward(fn, ps, how)
        graph.replay()
        torch.cuda.synchronize()
        got = got or [p.grad for p in ps]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del graph, got
    for p in ps: p.grad = None
    # an eager backward with an eager graph alive is as ever, and so is a captured forward
    alive = fn()
    assert all(torch.equal(a, b) for a, b in zip(backward(fn, ps, "grad"), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fn()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alive)
    del alive, y, graph
    gc.collect()
print("captured")
"""


def test_captured_backward_beside_a_living_eager_graph_is_refused():
    """It would end the process (the leaves' gradients are accumulated on the default stream); it
    raises before that, the process goes on, and without the eager graph the capture works."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE], cwd=root, capture_output=True, text=True,
                       timeout=180)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("change", [lambda m: m.cpu(), lambda m: m.double(), lambda m: m.half(),
                                    lambda m: m.cpu().double()])
def test_feed_forward_takes_parameters_of_any_kind(change):
    """In grad mode and under no_grad alike: parameters of another device or floating type than
    the kernels read; their gradients come back in their own place and type."""
    from tests.test_gpu_dense import module_inputs
    m, x, dy = module_inputs(BF16, F32)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(p.half())  # exact in every type
    want = torch.autograd.grad(m(x, residual=x), list(m.parameters()), dy)
    plain = m(x)
    m = change(m)
    with torch.no_grad():
        packed = m(x)
    # two roundings each (h and out), and the packed path's tanh.approx (2^-11)
    assert float((packed.float() - plain.detach().float()).norm() / plain.detach().float().norm()) <= 4 * 2.0 ** -8
    # the fold's last bit may differ with its device and type, and with it a folded weight's
    # rounding to bf16: one step of 2^-8 at most in y and in the gradients
    near = lambda a, b: float((a.double().cpu() - b.double().cpu()).norm() / b.double().norm())  # noqa: E731
    assert near(m(x).detach(), plain.detach()) <= 2.0 ** -8
    got = torch.autograd.grad(m(x, residual=x), list(m.parameters()), dy)
    for p, g, w in zip(m.parameters(), got, want):
        assert g.dtype == p.dtype and g.device == p.device
        assert near(g, w) <= 2.0 ** -8 + 2.0 ** -11


def test_another_architecture_is_refused_in_both_types():
    _lib, o = ops()
    ctypes.cast(o.ptr, ctypes.POINTER(OpsHead)).contents.sm100 = False
    n = ctypes.c_size_t()
    for dtype in (_lib.VMOE_F32, _lib.VMOE_BF16):
        for backward in (0, 1):
            d = _lib.VmoeLinear(40, 64, 64, 64, 64, 64, dtype, 2, 0.1, dtype)
            e = _lib.VmoeGatedFfn(40, 64, 64, 64, 64, dtype, 2, 0.1, dtype)
            with pytest.raises(_lib.VmoeError, match="sm_100") as err:
                o.check(o.lib.vmoe_linear_workspace_size(o.ptr, d, backward, n), "size")
            assert err.value.code == _lib.VMOE_ERR_UNSUPPORTED_SHAPE
            with pytest.raises(_lib.VmoeError, match="sm_100"):
                o.check(o.lib.vmoe_gated_ffn_workspace_size(o.ptr, e, backward, n, None), "size")


@pytest.mark.parametrize("T", [4, 40, 200])
def test_negated_views(T):
    """Views that torch negates when they are read, in every place."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    for dtype in (F32, BF16):
        x, w, b, r, dy = (rand(gen, *s, dtype=dtype).cuda()
                          for s in ((T, 64), (72, 64), (72,), (T, 72), (T, 72)))
        ws = [rand(gen, *s, dtype=dtype).cuda() for s in ((72, 64), (72, 64), (64, 72), (72,), (72,), (64,))]
        for neg in (lambda t: torch._neg_view(-t), lambda t: t):
            def run():
                p = [neg(t).detach().requires_grad_() for t in (x, w, b, *ws)]
                y = vb.linear(*p[:3], residual=neg(r), activation="silu")
                z = vb.gated_ffn(p[0], *p[3:], residual=neg(x))
                g = torch.autograd.grad((y, z), p, (neg(dy), neg(x)))
                return [t.resolve_neg() for t in (y, z, *g)]
            if neg(x).is_neg():
                got = run()
            else:
                assert all(torch.equal(a, c) for a, c in zip(got, run()))
        g = torch._neg_view(x.clone())
        assert torch.equal(vb.grad_norm([g]), vb.grad_norm([x]))


@pytest.mark.parametrize("T", [8, 100, 400])
def test_era_far_down(T):
    """bf16 ERA below zero, where softplus is log2(1 + e^z): its logarithm is off by at most 2^-22
    near 1, so y by gamma 2^-22 beside its rounding; it ends in 0, never below."""
    import velvetoptimizer_b200 as vb
    z = torch.linspace(-40, -5, T).to(BF16)
    y = vb.linear(z[:, None].cuda(), torch.ones(8, 1, device="cuda", dtype=BF16), activation="era",
                  gamma=GAMMA)
    v = z.double()[:, None].expand(T, 8)
    gelu = v * torch.sigmoid(1.5957691216057308 * (v + 0.044715 * v ** 3))
    want = gelu + GAMMA * torch.log1p(torch.exp(v))
    bound = 2.0 ** -8 * want.abs() + GAMMA * 2.0 ** -22 + 2.0 ** -18 * gelu.abs()
    got = y.double().cpu()
    assert ((got - want).abs() <= bound).all()
    assert (got[z < -20] >= 0).all() and (got[z < -20] <= GAMMA * 2.0 ** -22).all()


@pytest.mark.parametrize("T,K,N", [(40, 72, 40), (300, 2048, 40), (300, 300, 130), (64, 4096, 264)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_f32_all_not_a_number(T, K, N, act):
    """Every sum of a product formed again, with k divided and not: what fp32 gives."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(T)
    x, w, dy = (rand(gen, *s, dtype=F32) for s in ((T, K), (N, K), (T, N)))
    for bad, at in ((float("nan"), slice(None)), (float("inf"), slice(0, T, 2))):
        v = x.clone()
        v[at] = bad
        w1 = w.abs() + 0.5
        lx, lw = leaf(v), leaf(w1)
        y = vb.linear(lx, lw, activation=act)
        if act == "none":
            dx, dw = torch.autograd.grad(y, (lx, lw), dy.abs().cuda())
            same_as_fp32(dx, dy.abs(), w1)
            same_as_fp32(dw, dy.abs().t(), v)
            same_as_fp32(y, v, w1.t())
        else:
            want = torch.nn.functional.silu(v @ w1.t())
            got = y.detach().cpu()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        # the same bits again
        assert torch.equal(vb.linear(lx, lw, activation=act).nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [5, 90, 300])
def test_relu_cuts_off_whatever_the_gradient_is(T, dtype):
    """Where relu is 0 no gradient passes, an infinite or NaN one neither; where its input is NaN the
    gradient passes, as the value does."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(T)
    K, N = 24, 40
    x, w, dy = (rand(gen, *s, dtype=dtype) for s in ((T, K), (N, K), (T, N)))
    x[3] = float("nan")
    z = x.double() @ w.double().t()
    for i, bad in enumerate((float("inf"), float("nan"), -float("inf"))):
        off = (z[i] < -1).nonzero()[0]
        dy[i, off] = bad
    lx, lw = leaf(x), leaf(w)
    y = vb.linear(lx, lw, activation="relu")
    dx, dw = torch.autograd.grad(y, (lx, lw), dy.cuda())
    keep = ~(z <= 0)
    dz = torch.where(keep, dy.double(), 0.0)
    want = dz @ w.double()
    assert y[3].isnan().all() and torch.isfinite(dx).all() and dw.isnan().all()
    lim = 4 * ref.U[dtype] if dtype == BF16 else 1e-5
    assert float((d64(dx) - want).norm() / want.norm()) <= lim
    # the block: dg alone is cut off (du is dh times relu's own 0)
    wu, wd = rand(gen, N, K, dtype=dtype), torch.zeros(K, N, dtype=dtype)
    wd[0] = 1
    g, dout = torch.zeros(T, K, dtype=dtype), torch.zeros(T, K, dtype=dtype)
    dout[1, 0] = float("inf")
    g[:, 1] = 1
    wg = torch.zeros(N, K, dtype=dtype)
    wg[:, 1] = -1.0
    bg = torch.zeros(N, dtype=dtype)
    p = [leaf(t) for t in (g, wg, wu, wd, bg)]
    y = vb.gated_ffn(*p, activation="relu")
    dbg, = torch.autograd.grad(y, p[4], dout.cuda())
    assert not dbg.any()


def test_saved_tensor_hooks_and_checkpoints():
    """What the forward keeps goes through the hooks: on the CPU and back, or formed again."""
    from torch.utils.checkpoint import checkpoint

    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    for dtype in (BF16, F32):
        p = [rand(gen, 60, 72, dtype=dtype), *(rand(gen, *s, std=0.1, dtype=dtype)
                                               for s in ((104, 72), (104, 72), (72, 104), (40, 72)))]
        p = [t.cuda().requires_grad_() for t in p]
        dy = rand(gen, 60, 40, dtype=dtype).cuda()

        def fn(x, wg, wu, wd, wp):
            return vb.linear(vb.gated_ffn(x, wg, wu, wd, residual=x), wp, activation="silu")

        want = torch.autograd.grad(fn(*p), p, dy)
        with torch.autograd.graph.save_on_cpu():
            y = fn(*p)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, p, dy), want))
        y = checkpoint(fn, *p, use_reentrant=False)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, p, dy), want))


def test_f32_captured_with_and_without_infinities():
    """A captured fp32 call replayed on finite and other inputs in turn: nothing of one replay
    is left for the next."""
    import velvetoptimizer_b200 as vb
    gen = torch.Generator().manual_seed(0)
    x = rand(gen, 150, 300, dtype=F32).cuda()
    w = rand(gen, 130, 300, dtype=F32).cuda().requires_grad_()
    dy = rand(gen, 150, 130, dtype=F32).cuda()
    good = x.clone()
    bad = x.clone()
    bad[7, 11], bad[100] = float("inf"), float("nan")

    def step():
        lx = x.detach().requires_grad_()
        y = vb.linear(lx, w, activation="silu")
        return [y, *torch.autograd.grad(y, (lx, w), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for values in (bad, good, bad, bad, good):
        x.copy_(values)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    assert torch.isfinite(got[0]).all()
