"""Norms of query and key heads with the rotary embedding, forward and backward, against the formulas in 64 bits.

Tolerance: a result is rounded once, half a step of its type relative to the value, and smallest subnormals where they end.  Before
that the fp32 chain: a sum over a head is 16 fused products in a row and five additions across lanes (21 roundings), its root and
quotient two, products and rotation six: under 2^5 roundings of 2^-24 each, relative to the magnitudes that are added up."""
import ctypes

import pytest
import torch

EPS = 1e-6
FP32_CHAIN = 2.0 ** -19
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _tables(length, rot, dtype):
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(length, dtype=torch.float64)[:, None] * freq[None]
    a = torch.cat((a, a), 1)
    return a.cos().to(dtype).to(DEV), a.sin().to(dtype).to(DEV)


def _angles(cos, sin, pos, b, m, rot):
    at = torch.arange(m, device=DEV).expand(b, m) if pos is None else pos.long().expand(b, m)
    cos, sin = cos.reshape(cos.shape[-2:]), sin.reshape(sin.shape[-2:])
    return cos.double()[at][:, :, None, :rot // 2], sin.double()[at][:, :, None, :rot // 2]


def _turn(n, c, s, rot):
    h = rot // 2
    return torch.cat((n[..., :h] * c - n[..., h:rot] * s, n[..., h:rot] * c + n[..., :h] * s, n[..., rot:]), -1)


def plain_forward(x, w, c, s, rot, eps=EPS):
    """-> (value, magnitude that the roundings refer to)"""
    x = x.double()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return _turn(n, c, s, rot), _turn(n.abs(), c.abs(), -s.abs(), rot).abs() + _turn(n.abs(), c.abs(), s.abs(), rot).abs()


def plain_backward(dy, x, w, c, s, rot, eps=EPS):
    """-> (dx, dw) and the magnitudes that their roundings refer to"""
    x, dy, w = x.double(), dy.double(), w.double()
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    g = _turn(dy, c, -s, rot)
    mag = _turn(dy.abs(), c.abs(), -s.abs(), rot).abs() + _turn(dy.abs(), c.abs(), s.abs(), rot).abs()
    xn = x * r
    dx = r * (g * w - xn * (g * w * xn).mean(-1, keepdim=True))
    dx_mag = r * (mag * w.abs() + xn.abs() * (mag * w.abs() * xn.abs()).mean(-1, keepdim=True))
    return dx, (g * xn).sum((0, 1, 2)), dx_mag, (mag * xn.abs()).sum((0, 1, 2))


def close(got, want, mag, chain=FP32_CHAIN):
    f = torch.finfo(got.dtype)
    delta = chain * mag
    bound = f.eps / 2 * (want.abs() + delta) + delta + f.smallest_normal * f.eps
    return bool(((got.double() - want).abs() <= bound).all())


def _inputs(b, m, hq, hk, d, dtype, packed, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, m, hq + 2 * hk, d, generator=g).to(dtype).to(DEV)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    if not packed:
        q, k = q.contiguous(), k.contiguous()
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype).to(DEV) for _ in range(2)]
    dy = [torch.randn(b, m, h, d, generator=g).to(dtype).to(DEV) for h in (hq, hk)]
    return q, k, w, dy


def _check(q, k, w, dy, cos, sin, pos, rot, eps=EPS):
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    b, m = q.shape[:2]
    c, s = _angles(cos, sin, pos, b, m, rot)
    out = qn.qk_norm_rope_forward(q, k, *w, cos, sin, eps, position_ids=pos, rotary_dim=rot)
    grads = qn.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, eps, position_ids=pos, rotary_dim=rot)
    for i, x in enumerate((q, k)):
        assert out[i].shape == x.shape and out[i].dtype == x.dtype and out[i].is_contiguous()
        assert close(out[i], *plain_forward(x, w[i], c, s, rot, eps))
        dx, dw, dx_mag, dw_mag = plain_backward(dy[i], x, w[i], c, s, rot, eps)
        assert grads[i].dtype == x.dtype and grads[2 + i].dtype == w[i].dtype and grads[2 + i].shape == w[i].shape
        assert close(grads[i], dx, dx_mag)
        # the weights' gradients: a chain over tokens and heads on top
        assert close(grads[2 + i], dw, dw_mag, (x.shape[0] * x.shape[1] * x.shape[2] + 32) * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,rot", [(16, 16), (32, 16), (64, 64), (80, 80), (96, 48), (128, 128), (256, 64), (272, 272), (512, 512)])
def test_head_sizes(dtype, d, rot):
    t = DTYPES[dtype]
    q, k, w, dy = _inputs(2, 5, 3, 1, d, t, packed=True, seed=d + rot)
    _check(q, k, w, dy, *_tables(5, rot, torch.float32), None, rot)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,rot", [(48, 48), (48, 16), (80, 32), (96, 96), (112, 112), (144, 144), (160, 96), (192, 192), (240, 240), (288, 288)])
@pytest.mark.parametrize("hq,hk", [(1, 1), (7, 3), (24, 11)])
def test_heads_that_share_a_warp(dtype, d, rot, hq, hk):
    """Head sizes with any number of lanes, head counts that fill their last warp or do not."""
    q, k, w, dy = _inputs(2, 9, hq, hk, d, DTYPES[dtype], packed=True, seed=d + hq)
    _check(q, k, w, dy, *_tables(9, rot, torch.float32), None, rot)


@pytest.mark.gpu
@pytest.mark.parametrize("b,m,hq,hk", [(1, 1, 1, 1), (8, 1, 32, 8), (1, 257, 7, 7), (3, 333, 12, 4), (2, 1500, 32, 32), (300, 3, 5, 1)])
@pytest.mark.parametrize("table", ["bf16", "fp32"])
def test_sizes_and_positions(b, m, hq, hk, table):
    q, k, w, dy = _inputs(b, m, hq, hk, 128, torch.bfloat16, packed=(b + m) % 2 == 0, seed=b + m)
    cos, sin = _tables(4096, 128, DTYPES[table])
    first = torch.randint(0, 4096 - m, (b, 1), generator=torch.Generator().manual_seed(m)).to(DEV)
    for pos in (None, first + torch.arange(m, device=DEV), (first[:1] + torch.arange(m, device=DEV)).int(),
                torch.arange(m, device=DEV).flip(0)[None].expand(b, m)):
        _check(q, k, w, dy, cos, sin, pos, 128)


@pytest.mark.gpu
def test_layouts():
    """Heads in front of the sequence, channels that are not adjacent, begins off 16 bytes, expanded gradients, wide tables."""
    b, m, h, d = 2, 37, 4, 64
    t = torch.bfloat16
    q, k, w, dy = _inputs(b, m, h, h, d, t, packed=False, seed=1)
    cos, sin = _tables(50, d, torch.float32)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert not turned.is_contiguous()
    spread = torch.empty(b, m, h, 2 * d, dtype=t, device=DEV)[..., ::2].copy_(k)
    _check(turned, spread, w, dy, cos, sin, None, d)
    off = torch.empty(b * m * h * d + 1, dtype=t, device=DEV)[1:].view(b, m, h, d).copy_(q)
    off_w = torch.empty(d + 1, dtype=t, device=DEV)[1:].copy_(w[0])
    _check(off, k, (off_w, w[1]), dy, cos, sin, None, d)
    wide = [torch.cat((x, x), 1)[:, :d + 3] for x in (cos, sin)]                 # row strides that are no multiple of 16 bytes
    _check(q, k, w, dy, *[x[:, :d + 3].contiguous() for x in wide], None, d)
    _check(q, k, w, dy, cos[None, None], sin[None, None], None, d)
    for shape in ((b, m, h, 1), (1, 1, 1, d), (b, 1, h, d)):
        g = [torch.randn(shape, device=DEV).to(t).expand(b, m, h, d) for _ in range(2)]
        _check(q, k, w, g, cos, sin, None, d)
    _check(q, k, [x.float() for x in w], dy, cos, sin, None, d)


@pytest.mark.gpu
def test_values():
    """Heads of zeros, of one value, large and tiny ones, a large eps; NaN and infinities stay in their head."""
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    b, m, h, d = 1, 8, 4, 64
    q, k, w, dy = _inputs(b, m, h, h, d, torch.float32, packed=False, seed=2)
    q[0, 0] = 0
    q[0, 1] = 3
    q[0, 2] *= 1e15
    q[0, 3] *= 1e-12
    cos, sin = _tables(m, d, torch.float32)
    _check(q, k, w, dy, cos, sin, None, d)
    _check(q, k, w, dy, cos, sin, None, d, eps=1.0)
    good = qn.qk_norm_rope_forward(q, k, *w, cos, sin, EPS)[0]
    q[0, 4, 1, 7] = float("nan")
    q[0, 5, 2, 8] = float("inf")
    bad = qn.qk_norm_rope_forward(q, k, *w, cos, sin, EPS)[0]
    grads = qn.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, EPS)[0]
    assert bool(bad[0, 4, 1].isnan().all()) and bool(bad[0, 5, 2, 8].isnan())
    keep = torch.ones(b, m, h, dtype=torch.bool, device=DEV)
    keep[0, 4, 1] = keep[0, 5, 2] = False
    assert torch.equal(bad[keep], good[keep]) and bool(grads[keep].isfinite().all())


@pytest.mark.gpu
def test_positions_outside_of_the_tables():
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    q, k, w, dy = _inputs(2, 3, 2, 1, 64, torch.bfloat16, packed=False, seed=3)
    cos, sin = _tables(10, 32, torch.float32)
    pos = torch.tensor([[0, -1, 9], [10, 1 << 40, 3]], device=DEV)
    out = qn.qk_norm_rope_forward(q, k, *w, cos, sin, EPS, position_ids=pos, rotary_dim=32)[0]
    bad = (pos < 0) | (pos > 9)
    assert bool(out[bad][..., :32].isnan().all()) and bool(out[bad][..., 32:].isfinite().all()) and bool(out[~bad].isfinite().all())


@pytest.mark.gpu
def test_nothing_to_do_and_frozen_weights():
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    cos, sin = _tables(4, 64, torch.float32)
    w = [torch.ones(64, dtype=torch.bfloat16, device=DEV)] * 2
    for shape in ((0, 4), (4, 0)):
        q, k = torch.empty(*shape, 2, 64, dtype=torch.bfloat16, device=DEV), torch.empty(*shape, 1, 64, dtype=torch.bfloat16, device=DEV)
        out = qn.qk_norm_rope_forward(q, k, *w, cos, sin, EPS)
        assert out[0].shape == q.shape and out[1].shape == k.shape
        grads = qn.qk_norm_rope_backward(q, k, q, k, *w, cos, sin, EPS)
        assert bool((grads[2] == 0).all()) and bool((grads[3] == 0).all())
    q, k, w, dy = _inputs(1, 4, 2, 2, 64, torch.bfloat16, packed=True, seed=4)
    with_w, frozen = (qn.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, EPS, needs_weight_grad=x) for x in (True, False))
    assert frozen[2] is None and frozen[3] is None and torch.equal(frozen[0], with_w[0]) and torch.equal(frozen[1], with_w[1])


@pytest.mark.gpu
def test_same_bits_again_and_in_graphs_on_another_stream():
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    q, k, w, dy = _inputs(2, 700, 8, 2, 128, torch.bfloat16, packed=True, seed=5)
    cos, sin = _tables(700, 128, torch.bfloat16)

    def both():
        return qn.qk_norm_rope_forward(q, k, *w, cos, sin, EPS) + qn.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, EPS)
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
    q.neg_()
    again = both()
    for graph, out in graphs[::-1]:
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the 64-bit formula along one direction: truncation of order step^2 = 1e-8 of the sum's magnitude, the
    kernel's fp32 chains above it."""
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    q, k, w, dy = _inputs(1, 9, 3, 2, 64, torch.float32, packed=False, seed=6)
    cos, sin = _tables(9, 64, torch.float32)
    c, s = _angles(cos, sin, None, 1, 9, 64)
    grads = qn.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, EPS)
    g = torch.Generator().manual_seed(7)
    for i, x in enumerate((q, k)):
        vx, vw = torch.randn(x.shape, generator=g, dtype=torch.float64).to(DEV), torch.randn(64, generator=g, dtype=torch.float64).to(DEV)

        def loss(step):
            return (plain_forward(x.double() + step * vx, w[i].double() + step * vw, c, s, 64)[0] * dy[i].double()).sum()
        difference = (loss(1e-4) - loss(-1e-4)) / 2e-4
        parts = torch.cat(((grads[i].double() * vx).reshape(-1), grads[2 + i].double() * vw))
        assert abs(float(parts.sum() - difference)) <= 1e-5 * float(parts.abs().sum())


@pytest.mark.gpu
def test_refusals():
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    q, k, w, dy = _inputs(2, 4, 2, 1, 64, torch.bfloat16, packed=False, seed=8)
    cos, sin = _tables(4, 64, torch.float32)

    def fwd(q=q, k=k, w=w, cos=cos, sin=sin, **kw):
        return qn.qk_norm_rope_forward(q, k, w[0], w[1], cos, sin, EPS, **kw)
    for call in (lambda: fwd(k=k[:1]), lambda: fwd(k=k.half()), lambda: fwd(q=q.double(), k=k.double()), lambda: fwd(q=q[..., :40], k=k[..., :40]),
                 lambda: fwd(q=q[0]), lambda: fwd(w=(w[0][:32], w[1])), lambda: fwd(w=(w[0].float(), w[1])), lambda: fwd(rotary_dim=24),
                 lambda: fwd(rotary_dim=80), lambda: fwd(rotary_dim=0), lambda: fwd(cos=cos[:3], sin=sin[:3]), lambda: fwd(cos=cos[:, :16], sin=sin[:, :16]),
                 lambda: fwd(cos=cos[:3]), lambda: fwd(position_ids=torch.zeros(2, 3, dtype=torch.int64, device=DEV)),
                 lambda: fwd(position_ids=torch.zeros(2, 4, device=DEV)), lambda: fwd(position_ids=torch.zeros(3, 4, dtype=torch.int64, device=DEV)),
                 lambda: qn.qk_norm_rope_backward(dy[0][:1], dy[1], q, k, *w, cos, sin, EPS),
                 lambda: qn.qk_norm_rope_backward(dy[0].float(), dy[1], q, k, *w, cos, sin, EPS)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="different devices|only on CUDA"):
        fwd(cos=cos.cpu(), sin=sin.cpu())


class Args(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p * 2), ("dy", ctypes.c_void_p * 2), ("weight", ctypes.c_void_p * 2), ("out", ctypes.c_void_p * 2),
                ("x_stride", ctypes.c_int64 * 6), ("dy_stride", ctypes.c_int64 * 6), ("cos_t", ctypes.c_void_p), ("sin_t", ctypes.c_void_p),
                ("ld_cos", ctypes.c_int64), ("ld_sin", ctypes.c_int64), ("table_rows", ctypes.c_int64), ("position_ids", ctypes.c_void_p),
                ("pos_stride", ctypes.c_int64 * 2), ("pos_is_int64", ctypes.c_int), ("batch", ctypes.c_int64), ("seq", ctypes.c_int64),
                ("heads", ctypes.c_int * 2), ("head_dim", ctypes.c_int), ("rotary_dim", ctypes.c_int), ("type", ctypes.c_int),
                ("w_type", ctypes.c_int), ("table_type", ctypes.c_int), ("eps", ctypes.c_float)]


def test_the_library_refuses_before_it_launches():
    """Sizes, alignment and missing pointers are errors of the call, found without a device."""
    from hyc_lora_release_b200._lib import lib
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) & ~15

    def call(backward=False, **change):
        a = Args()
        for name in ("x", "dy", "weight", "out"):
            getattr(a, name)[0] = getattr(a, name)[1] = p
        a.x_stride[:] = a.dy_stride[:] = [512, 128, 64] * 2
        a.cos_t = a.sin_t = p
        a.ld_cos = a.ld_sin = 64
        a.table_rows, a.batch, a.seq, a.head_dim, a.rotary_dim = 4, 0, 4, 64, 64
        a.heads[0] = a.heads[1] = 2
        for name, value in change.items():
            if isinstance(value, tuple):
                getattr(a, name)[value[0]] = value[1]
            else:
                setattr(a, name, value)
        if backward:
            return lib.hyc_qk_norm_rope_bwd(ctypes.byref(a), p, p, None, 0, None)
        return lib.hyc_qk_norm_rope_fwd(ctypes.byref(a), None)
    assert call() == 0                                                     # no tokens
    assert lib.hyc_qk_norm_rope_fwd(None, None) == -1
    for change in (dict(head_dim=24), dict(head_dim=528), dict(rotary_dim=8), dict(rotary_dim=80), dict(heads=(0, 0)), dict(heads=(1, 65537)),
                   dict(batch=-1), dict(batch=1 << 31), dict(batch=1 << 20, seq=1 << 20), dict(batch=1, table_rows=3), dict(batch=1, ld_cos=24)):
        assert call(**change) == -3, change
    assert call(type=3) == call(w_type=-1) == call(table_type=7) == -8
    for change in (dict(x=(1, None)), dict(weight=(0, None)), dict(out=(0, None)), dict(cos_t=None)):
        assert call(batch=1, **change) == -1, change
    for change in (dict(x=(0, p + 2)), dict(weight=(1, p + 8)), dict(out=(1, p + 4)), dict(x_stride=(2, 68)), dict(ld_sin=68, table_type=0), dict(sin_t=p + 4)):
        assert call(batch=1, **change) == -4, change
    assert call(backward=True) == -5                                       # no workspace


@pytest.mark.gpu
def test_tables_that_are_one_row_for_all_positions():
    """Expanded tables (row stride 0) and tables whose rows overlap."""
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    q, k, w, dy = _inputs(2, 6, 3, 2, 64, torch.bfloat16, packed=False, seed=9)
    for t in DTYPES.values():
        cos, sin = _tables(6, 64, t)
        for c, s in ((cos[3:4].expand(6, 64), sin[3:4].expand(6, 64)), (cos[3:4].expand(6, 64), sin),
                     (cos.reshape(-1).as_strided((6, 32), (16, 1)), sin.reshape(-1).as_strided((6, 32), (16, 1)))):
            _check(q, k, w, dy, c, s, None, 64)
            got = qn.qk_norm_rope_forward(q, k, *w, c, s, EPS)
            want = qn.qk_norm_rope_forward(q, k, *w, c.contiguous(), s.contiguous(), EPS)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def _weight_gradients_close(got, want, mag, chain):
    """-> whether they are within the bound, the bound"""
    f = torch.finfo(got.dtype)
    bound = f.eps / 2 * (want.abs() + chain * mag) + chain * mag + f.smallest_normal * f.eps
    return bool(((got.double() - want).abs() <= bound).all()), bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,b,m,hq,hk,d,rot", [("bf16", 2, 1500, 32, 32, 128, 128), ("bf16", 4, 2048, 32, 8, 128, 128), ("fp16", 3, 1333, 12, 12, 64, 32),
                                                   ("fp32", 2, 1500, 24, 8, 96, 96), ("fp32", 1, 2000, 8, 2, 512, 512), ("bf16", 2, 3000, 7, 1, 80, 80)])
def test_weight_gradients_of_many_tokens(dtype, b, m, hq, hk, d, rot):
    """Sums over all tokens and heads, as the kernel takes them: the grid has at least two blocks per 32 SMs and tensor, of eight warps that
    share a tensor's heads evenly but for one token's each, and a lane adds up the heads of its place in the warp; then the warp's
    heads (32 at most), eight warps, and the blocks, every 32nd by a thread (10 at most) and five steps of a tree.  In roundings of 2^-24 relative to the
    magnitudes, on top of a head's own chain.  The gradients are far above that: half of one, or one without an eightieth of the tokens, would not pass."""
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    t = DTYPES[dtype]
    q, k, w, dy = _inputs(b, m, hq, hk, d, t, packed=True, seed=m)
    for x, g in ((q, dy[0]), (k, dy[1])):      # gradients that follow the heads: the sums grow with the number of tokens
        g.copy_(g.float() + x.float())
    cos, sin = _tables(m, rot, torch.float32)
    one, zero = torch.ones_like(cos), torch.zeros_like(sin)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for c_table, s_table in ((cos, sin), (one, zero)):
        c, s = _angles(c_table, s_table, None, b, m, rot)
        grads = qn.qk_norm_rope_backward(*dy, q, k, *w, c_table, s_table, EPS, rotary_dim=rot)
        for i, x in enumerate((q, k)):
            _, want, _, mag = plain_backward(dy[i], x, w[i], c, s, rot)
            heads = x.shape[0] * x.shape[1] * x.shape[2]
            lane = heads / (sms // 32 * 2 * 8) + x.shape[2]      # (a warp's heads, all in one place: more than a lane has)
            chain = FP32_CHAIN + (lane + 32 + 8 + 10 + 5) * 2.0 ** -24
            fits, bound = _weight_gradients_close(grads[2 + i], want, mag, chain)
            assert fits
            if s_table is zero:
                assert bool((bound < want.abs() / 80).all())
                assert not _weight_gradients_close(grads[2 + i] / 2, want, mag, chain)[0]
                share = plain_backward(dy[i][:, :m // 80 + 1], x[:, :m // 80 + 1], w[i], c[:, :m // 80 + 1], s[:, :m // 80 + 1], rot)[1]
                assert not _weight_gradients_close(grads[2 + i], want + share, mag, chain)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,rot", [(64, 32), (80, 32), (96, 48), (128, 64), (320, 160)])
def test_infinities_in_channels_that_are_not_turned(dtype, d, rot):
    """Behind rotary_dim every channel is on its own: an infinity there is in no other channel's result, nor in another's weight gradient."""
    from hyc_lora_release_b200.operators import qk_norm_kernels as qn
    t = DTYPES[dtype]
    cos, sin = _tables(7, rot, torch.float32)
    for at in range(rot, d):
        q, k, w, dy = _inputs(1, 7, 3, 2, d, t, packed=False, seed=d)
        q[0, 2, 1, at] = float("inf")
        dy[1][0, 3, 0, at] = float("inf")
        out = qn.qk_norm_rope_forward(q, k, *w, cos, sin, EPS, rotary_dim=rot)[0][0, 2, 1]
        want = torch.zeros(d, device=DEV)
        want[at] = float("nan")                          # (a root of infinity: everything else is 0)
        assert torch.equal(out.isnan(), want.isnan()) and bool((out[~want.isnan()] == 0).all())
        dw = qn.qk_norm_rope_backward(*dy, q, k, *w, cos, sin, EPS, rotary_dim=rot)[3]
        others = torch.arange(d, device=DEV) != at
        assert bool(dw[others].isfinite().all()) and not bool(dw[at].isfinite())
