"""Products with bias, activation and residual in the epilogue and their backward pass, against the formulas in 64 bits.

Tolerances: a result is rounded once, half a step of its type relative to the value.  Before that: a sum of K products in fp32, K * 2^-24
of the sum of magnitudes; an activation has a slope of 1.13 at most and is evaluated to 2^-20 of its argument's size (the exponential's
two units in the last place, and 1 + erf, which cancels), its slope to 2^-19; bias and residual one rounding each.  Backward rounds dpre
to the operands' type: half a step of each factor."""
import ctypes

import pytest
import torch

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def act_of(x, act):
    if act == "relu":
        return torch.relu(x)      # slope 0 at 0
    if act == "gelu":
        return x * torch.special.ndtr(x)
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)))
    if act == "silu":
        return x * torch.sigmoid(x)
    return x


def slope_of(x, act):
    x = x.detach().requires_grad_()
    return torch.autograd.grad(act_of(x, act).sum(), x)[0]


def close(got, want, delta):
    f = torch.finfo(got.dtype)
    bound = f.eps / 2 * (want.abs() + delta) + delta + f.smallest_normal * f.eps
    return bool(((got.double() - want).abs() <= bound).all())


def product(a, b):
    """a @ b and the bound of its roundings"""
    a, b = a.double(), b.double()
    return a @ b, a.shape[1] * 2.0 ** -24 * (a.abs() @ b.abs())


def check_forward(x, w, bias, act, res, y, pre):
    x = x.reshape(-1, x.shape[-1])
    want, delta = product(x, w.t())
    if bias is not None:
        want, delta = want + bias.double(), delta + 2.0 ** -24 * (want.abs() + bias.double().abs())
    assert pre is None or close(pre.reshape(want.shape), want, delta)
    out = act_of(want, act)
    delta = 1.13 * delta + (0 if act in ("none", "relu") else 2.0 ** -20 * want.abs())
    if res is not None:
        r = res.double().reshape(want.shape)
        out, delta = out + r, delta + 2.0 ** -23 * (out.abs() + r.abs())
    assert close(y.reshape(want.shape), out, delta)


def check_backward(dy, x, w, act, pre, dx, dw, db):
    n, k = w.shape
    dy, x = dy.double().reshape(-1, n), x.double().reshape(-1, k)
    if act == "none":
        dpre, err, half = dy, torch.zeros_like(dy), 0.0
    else:
        f = torch.finfo(w.dtype)
        dpre = dy * slope_of(pre.double().reshape(-1, n), act)
        err = 2.0 ** -19 * dy.abs()
        half = f.eps / 2 * 1.01
    step = err + half * dpre.abs() + (0 if act == "none" else torch.finfo(w.dtype).smallest_normal * torch.finfo(w.dtype).eps)
    if dx is not None:
        want, delta = product(dpre, w)
        assert dx.dtype == w.dtype and close(dx.reshape(want.shape), want, delta * 1.01 + step @ w.double().abs())
    if dw is not None:
        want, delta = product(dpre.t(), x)
        assert dw.dtype == w.dtype and close(dw, want, delta * 1.01 + step.t() @ x.abs())
    if db is not None:
        assert db.dtype == w.dtype and close(db, dpre.sum(0), (dy.shape[0] + 32) * 2.0 ** -24 * dpre.abs().sum(0) + err.sum(0))


def inputs(t, k, n, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
    return rn(t, k), (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype).to(DEV), rn(n), rn(t, n), rn(t, n), rn(t, n)


def run_both(x, w, b, res, dy, pre, act):
    from hyc_lora_release_b200.operators import linear_kernels as lk
    for bias, r, save in ((b, res, True), (None, None, False), (b, None, True)):
        y, p = lk.linear_act_forward(x, w, bias, act, residual=r, save_pre=save)
        assert y.shape == dy.shape and y.is_contiguous() and (p is None) == (not save)
        check_forward(x, w, bias, act, r, y, p)
    out = lk.linear_act_backward(dy, x, w, act, pre=None if act == "none" else pre)
    check_backward(dy, x, w, act, pre, *out)
    return out


SIZES = [(1, 64, 64), (1, 4096, 1032), (2, 8, 8), (3, 40, 16), (7, 1000, 72), (15, 264, 520), (16, 128, 256), (17, 136, 264), (33, 512, 4096), (63, 2000, 136),
         (64, 256, 1000), (100, 72, 2048), (128, 1024, 128), (129, 640, 384), (200, 1504, 2000), (255, 320, 256), (256, 4096, 64), (257, 128, 512),
         (300, 2048, 2056), (333, 11008, 264), (511, 256, 1024), (512, 64, 4096), (513, 520, 1288), (777, 1000, 1000), (1025, 264, 776), (2100, 512, 2048),
         (4097, 128, 3000), (9000, 64, 136)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_sizes(size, dtype):
    act = ACTS[SIZES.index(size) % 5]
    x, w, b, res, dy, pre = inputs(*size, DTYPES[dtype], sum(size))
    run_both(x, w, b, res, dy, pre, act)
    from hyc_lora_release_b200.operators import linear_kernels as lk
    lk.raise_on_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [5, 1200])
def test_activations(act, t):
    """Arguments from -inf to inf: a product with the identity hands them to the epilogue as they are."""
    from hyc_lora_release_b200.operators import linear_kernels as lk
    n = 64
    for dtype in DTYPES.values():
        v = torch.cat((torch.linspace(-12, 12, t * n - 20), torch.tensor([0.0, -0.0, 1e-6, -1e-6, 30.0, -30.0, 100.0, -100.0, 1e4, -1e4,
                                                                         6e4, -6e4, 20.0, -20.0, 8.5, -8.5, 5.9, -5.9, 4.4, -4.4])))
        x = v.view(t, n).to(dtype).to(DEV)
        eye = torch.eye(n, dtype=dtype, device=DEV)
        y, pre = lk.linear_act_forward(x, eye, None, act, save_pre=True)
        assert torch.equal(pre, x)
        check_forward(x, eye, None, act, None, y, None)
        ones = torch.ones_like(x)
        dx, _, db = lk.linear_act_backward(ones, x, eye, act, pre=None if act == "none" else x, needs_grad=(True, False, True))
        check_backward(ones, x, eye, act, x, dx, None, db)
        x[1, 3] = float("nan")
        y, _ = lk.linear_act_forward(x, eye, None, act)
        assert bool(y[1].isnan().all()) and not bool(y[0].isnan().any()) and not bool(y[2:].isnan().any())


@pytest.mark.gpu
def test_layouts():
    """Rows with strides of their own, leading dimensions, operands off 16 bytes, expanded gradients, transposed weights."""
    from hyc_lora_release_b200.operators import linear_kernels as lk
    for t in (24, 700):
        k, n = 264, 136
        x, w, b, res, dy, pre = inputs(t, k, n, torch.bfloat16, t)
        want = run_both(x, w, b, res, dy, pre, "silu")
        wide = lambda a, c: torch.cat((a, a), 1)[:, :a.shape[1]] if c == 0 else torch.cat((a, a[:, :c]), 1)[:, :a.shape[1]]
        for c in (0, 3, 8):
            got = run_both(wide(x, c), wide(w, c), b, wide(res, c), wide(dy, c), wide(pre, c), "silu")
            assert all(torch.equal(p, q) for p, q in zip(want, got))
        off = lambda a: torch.empty(a.numel() + 1, dtype=a.dtype, device=DEV)[1:].view(a.shape).copy_(a)
        got = run_both(off(x), off(w), off(b), off(res), off(dy), off(pre), "silu")
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        got = run_both(x.t().contiguous().t(), w.t().contiguous().t(), b, res.t().contiguous().t(), dy.t().contiguous().t(), pre, "silu")
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        split = lambda a: a.view(2, t // 4, 2, -1)
        got = run_both(split(x), w, b, split(res), split(dy), split(pre), "silu")
        assert got[0].shape == (2, t // 4, 2, k) and all(torch.equal(p.reshape(q.shape), q) for p, q in zip(got, want))
        for shape in ((1, n), (t, 1), (1, 1)):
            g = torch.randn(shape, device=DEV).to(torch.bfloat16).expand(t, n)
            run_both(x, w, b, res, g, pre, "relu")
            run_both(x, w, b, res, g, pre, "none")
        y, _ = lk.linear_act_forward(x[0], w, b, "gelu")
        assert y.shape == (n,)
        y, _ = lk.linear_act_forward(x, w, b, residual=res[:1].expand(t, n))
        check_forward(x, w, b, "none", res[:1].expand(t, n), y, None)


@pytest.mark.gpu
def test_what_is_asked_for():
    from hyc_lora_release_b200.operators import linear_kernels as lk
    x, w, b, res, dy, pre = inputs(50, 72, 136, torch.float16, 1)
    whole = lk.linear_act_backward(dy, x, w, "gelu", pre=pre)
    for bits in range(8):
        needs = tuple(bool(bits >> i & 1) for i in range(3))
        got = lk.linear_act_backward(dy, x, w, "gelu", pre=pre, needs_grad=needs)
        for g, v, need in zip(got, whole, needs):
            assert (g is None) == (not need) and (g is None or torch.equal(g, v))
    empty = x[:0]
    y, p = lk.linear_act_forward(empty, w, b, "gelu", residual=res[:0], save_pre=True)
    assert y.shape == p.shape == (0, 136)
    dx, dw, db = lk.linear_act_backward(dy[:0], empty, w, "gelu", pre=pre[:0])
    assert dx.shape == (0, 72) and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.gpu
def test_rows_do_not_depend_on_their_neighbours_and_nothing_else_is_written():
    """NaN behind the last row of every operand's storage, results in the middle of a larger buffer's life: only what belongs is read."""
    from hyc_lora_release_b200.operators import linear_kernels as lk
    for t, k, n in ((5, 136, 264), (300, 72, 520), (1100, 264, 136)):
        x, w, b, res, dy, pre = inputs(t, k, n, torch.bfloat16, t)
        want = lk.linear_act_forward(x, w, b, "gelu", residual=res, save_pre=True) + lk.linear_act_backward(dy, x, w, "gelu", pre=pre)

        def nan_around(a):
            big = torch.full((a.shape[0] + 300, a.shape[1] + 8), float("nan"), dtype=a.dtype, device=DEV)
            big[:a.shape[0], :a.shape[1]] = a
            return big[:a.shape[0], :a.shape[1]]
        x, w, res, dy = (nan_around(a) for a in (x, w, res, dy))
        got = lk.linear_act_forward(x, w, b, "gelu", residual=res, save_pre=True) + lk.linear_act_backward(dy, x, w, "gelu", pre=pre)
        assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.gpu
def test_same_bits_again_and_in_graphs_on_another_stream():
    from hyc_lora_release_b200.operators import linear_kernels as lk
    cases = [inputs(t, k, n, torch.bfloat16, t) for t, k, n in ((3, 4096, 512), (400, 1024, 1024), (1500, 512, 1288))]

    def both():
        out = []
        for x, w, b, res, dy, pre in cases:
            out += [*lk.linear_act_forward(x, w, b, "gelu_tanh", residual=res, save_pre=True), *lk.linear_act_backward(dy, x, w, "gelu_tanh", pre=pre)]
        return out
    first = both()
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = both()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, side))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, both()))
    for case in cases:
        case[0].mul_(-2)
        case[4].mul_(0.5)
    again = both()
    for graph, out in graphs[::-1]:
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, again))
    lk.raise_on_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS[2:])
def test_gradients_against_differences(act):
    """Central differences of the 64-bit formula along one direction (truncation of order step^2); the kernels' gradients carry 16-bit
    roundings, half a step of dpre and half a step of the result for each term of the sum."""
    from hyc_lora_release_b200.operators import linear_kernels as lk
    x, w, b, _, dy, _ = inputs(40, 64, 72, torch.float16, 3)
    _, pre = lk.linear_act_forward(x, w, b, act, save_pre=True)
    dx, dw, db = lk.linear_act_backward(dy, x, w, act, pre=pre)
    g = torch.Generator().manual_seed(4)
    vx, vw, vb = (torch.randn(t.shape, generator=g, dtype=torch.float64).to(DEV) for t in (x, w, b))

    def loss(step):
        return (act_of((x.double() + step * vx) @ (w.double() + step * vw).t() + b.double() + step * vb, act) * dy.double()).sum()
    difference = (loss(1e-4) - loss(-1e-4)) / 2e-4
    parts = torch.cat([(p.double() * v).reshape(-1) for p, v in ((dx, vx), (dw, vw), (db, vb))])
    # pre is off by half a step of up to 8 (its own type), and the second derivatives are at most 1.2
    terms = (dy.double().abs() @ w.double().abs() * vx.abs()).sum() + (dy.double().abs().t() @ x.double().abs() * vw.abs()).sum() + (dy.double().abs().sum(0) * vb.abs()).sum()
    assert abs(float(parts.sum() - difference)) <= 2.0 ** -11 * float(terms) * (1.13 * 2 + 1.2 * 8) + 1e-6 * float(terms)


@pytest.mark.gpu
def test_refusals():
    from hyc_lora_release_b200.operators import linear_kernels as lk
    x, w, b, res, dy, pre = inputs(6, 64, 72, torch.bfloat16, 5)

    def fwd(x=x, w=w, b=b, act="none", **kw):
        return lk.linear_act_forward(x, w, b, act, **kw)

    def bwd(dy=dy, x=x, w=w, act="gelu", pre=pre):
        return lk.linear_act_backward(dy, x, w, act, pre=pre)
    for call in (lambda: fwd(act="tanh"), lambda: fwd(x.float(), w.float(), b.float()), lambda: fwd(w=w.half()), lambda: fwd(w=w[:, :60], x=x[:, :60]),
                 lambda: fwd(w=w[:70], b=b[:70]), lambda: fwd(x=x[:, :56]), lambda: fwd(w=w[None]), lambda: fwd(b=b[:64]), lambda: fwd(b=b.float()),
                 lambda: fwd(residual=res[:5]), lambda: fwd(residual=res.float()), lambda: fwd(residual=res[0]), lambda: bwd(pre=None), lambda: bwd(pre=pre[:5]),
                 lambda: bwd(dy=dy[:5]), lambda: bwd(dy=dy.half()), lambda: bwd(pre=pre.float())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="different devices|only on CUDA"):
        fwd(w=w.cpu())


class Args(ctypes.Structure):
    _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("pre", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("ld_a", ctypes.c_int64), ("ld_b", ctypes.c_int64), ("ld_res", ctypes.c_int64), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int), ("depth", ctypes.c_int), ("a_mn", ctypes.c_int), ("b_mn", ctypes.c_int), ("type", ctypes.c_int), ("act", ctypes.c_int)]


def test_the_library_refuses_before_it_launches():
    from hyc_lora_release_b200._lib import lib
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) & ~15

    def call(**change):
        a = Args(p, p, None, None, None, p, 64, 64, 0, 8, 64, 64, 0, 0, 0, 0)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.hyc_linear_act_tcgen05(ctypes.byref(a), None)
    assert lib.hyc_linear_act_tcgen05(None, None) == -1 and call(rows=0) == 0
    assert call(type=2) == call(act=5) == call(act=-1) == call(a_mn=1) == -8
    for change in (dict(rows=-1), dict(rows=1 << 30), dict(cols=60), dict(cols=0), dict(depth=60), dict(depth=0), dict(ld_a=56), dict(ld_b=56), dict(a_mn=1, b_mn=1, rows=9),
                   dict(b_mn=1, cols=72), dict(residual=p, ld_res=8)):
        assert call(**change) == -3, change
    assert call(a=None) == call(b=None) == call(out=None) == -1
    for change in (dict(a=p + 2), dict(b=p + 8), dict(out=p + 2), dict(pre=p + 2), dict(bias=p + 1), dict(residual=p + 2, ld_res=64), dict(ld_a=68), dict(ld_b=68),
                   dict(residual=p, ld_res=68)):
        assert call(**change) == -4, change
    dpre = lib.hyc_linear_act_dpre
    assert dpre(p, 64, p, p, None, 8, 64, 2, 0, None, 0, None) == dpre(p, 64, p, p, None, 8, 64, 0, 5, None, 0, None) == -8
    assert dpre(p, 64, p, p, None, -1, 64, 0, 0, None, 0, None) == dpre(p, 64, p, p, None, 8, 60, 0, 0, None, 0, None) == -3
    assert dpre(None, 64, p, p, None, 8, 64, 0, 0, None, 0, None) == dpre(p, 64, None, p, None, 8, 64, 0, 1, None, 0, None) == -1
    assert dpre(p, 60, p, p, None, 8, 64, 0, 0, None, 0, None) == dpre(p + 2, 64, p, p, None, 8, 64, 0, 0, None, 0, None) == -4
    need = lib.hyc_linear_act_dpre_workspace_bytes(64)
    assert need > 0 and dpre(p, 64, p, p, p, 8, 64, 0, 0, p, need - 1, None) == dpre(p, 64, p, p, p, 8, 64, 0, 0, None, need, None) == -5
    assert lib.hyc_linear_status(None) == -1


@pytest.mark.gpu
def test_the_status_waits_for_every_stream():
    """Work on a stream that the default one does not wait for has ended when the status has been read."""
    from hyc_lora_release_b200.operators import linear_kernels as lk
    x, w, b, _, _, _ = inputs(64, 64, 64, torch.bfloat16, 1)
    big = torch.randn(8192, 8192, device=DEV).to(torch.bfloat16)
    stream, done = torch.cuda.Stream(), torch.cuda.Event()

    def work(times):
        with torch.cuda.stream(stream):
            for _ in range(times):
                big @ big
            lk.linear_act_forward(x, w, b)
            done.record()
    work(1)                      # (memory and code are there: nothing else waits for the device)
    torch.cuda.synchronize()
    work(60)                     # tens of milliseconds
    lk.raise_on_device_errors()
    assert done.query()


def test_the_status_is_of_the_device_that_is_meant(monkeypatch):
    from hyc_lora_release_b200.operators import linear_kernels as lk
    asked = []

    class Host:
        @staticmethod
        def linear_status(device):
            asked.append(device)
            return 0
    monkeypatch.setattr(lk, "host", Host)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for device in (None, "cuda", torch.device("cuda"), "cuda:0", torch.device("cuda", 2), 1):
        lk.raise_on_device_errors(device)
    assert asked == [3, 3, 3, 0, 2, 1]
    with pytest.raises(ValueError):
        lk.raise_on_device_errors("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("t", [4, 600])
def test_gelu_far_out_on_the_left(t, dtype):
    """x Phi(x) for x from -14 to -1, where it is small: relative to itself.  Before the one rounding: the tail's rational function 2^-17;
    the exponential's argument, up to 90 and rounded three times, 3 * 90 * 2^-24 < 2^-15; its two units, the quotient's and the products' 2^-20."""
    from hyc_lora_release_b200.operators import linear_kernels as lk
    k = 512
    x = torch.linspace(-14, -1, t * k).view(t, k).to(DTYPES[dtype]).to(DEV)
    y, _ = lk.linear_act_forward(x, torch.eye(k, dtype=x.dtype, device=DEV), None, "gelu")
    want = x.double() * torch.special.erfc(-x.double() / 2 ** 0.5) / 2
    f = torch.finfo(x.dtype)
    # (a result below fp32's smallest normal number may be 0)
    assert bool(((y.double() - want).abs() <= want.abs() * (f.eps / 2 + 2.0 ** -14) + f.smallest_normal * f.eps + 2.0 ** -126).all())
