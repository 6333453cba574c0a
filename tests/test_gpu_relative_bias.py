"""Softmax with a learned bias per bucket of relative positions, forward and backward, against the formulas in 64 bits.

Tolerances: a result is rounded once, half a step of its type relative to the value.  Before that, fp32:
  forward   an exponent is three roundings of numbers up to X (the largest |scale s| + |bias| + |mask| of a place that counts in
            its row), off by 2^-22 X at most, and so relatively is an exponential and the row's sum; the exponential itself
            and a sum of chains of at most 32 + 5 + 16 + 8 additions: 2^-17
  backward  a row's product sum is chains of the same lengths: 2^-18 of the sum of magnitudes; a difference and two products:
            2^-22; the table's sums: chains of 32 rows and of 1024 / 32 + 6 distances, then 64 bits: 2^-17 of the magnitudes"""
import ctypes
import math

import pytest
import torch

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def bucket_by_definition(r, side, distance):
    """exact + floor((side - exact) * log(r / exact) / log(distance / exact)), counted in whole numbers"""
    exact = side // 2
    if r < exact:
        return r
    t = 0
    while t + 1 < side - exact and r ** (side - exact) * exact ** (t + 1) >= distance ** (t + 1) * exact ** (side - exact):
        t += 1
    return exact + t


def bucket_index(buckets, n, cols, offset):
    """[n, cols] entry of the table, from the definition"""
    side = buckets.num_buckets // 2 if buckets.bidirectional else buckets.num_buckets
    one = torch.tensor([bucket_by_definition(r, side, buckets.max_distance) for r in range(buckets.max_distance + 1)])
    d = torch.arange(cols)[None] - torch.arange(n)[:, None] - offset
    if buckets.bidirectional:
        return (one[d.abs().clamp_max(buckets.max_distance)] + side * (d > 0)).to(DEV)
    return one[(-d).clamp(0, buckets.max_distance)].to(DEV)


def visible(n, cols, causal, offset):
    if not causal:
        return torch.ones(n, cols, dtype=torch.bool, device=DEV)
    return torch.arange(cols, device=DEV)[None] <= torch.arange(n, device=DEV)[:, None] + offset


def plain_forward(scores, scale, table, buckets, mask, causal, offset):
    """-> (probabilities, largest magnitude of an exponent's parts per row)"""
    n, cols = scores.shape[2:]
    see = visible(n, cols, causal, offset)
    bias = table.double()[bucket_index(buckets, n, cols, offset)].permute(2, 0, 1)
    x = scores.double() * scale + bias
    mag = (scores.double() * scale).abs() + bias.abs()
    if mask is not None:
        x, mag = x + mask.double(), mag + mask.double().abs()
    x = x.masked_fill(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    return p, torch.where(p > 0, mag, torch.zeros_like(mag)).amax(-1, keepdim=True)


def forward_close(got, want, X):
    f = torch.finfo(got.dtype)
    rel = 2.0 ** -22 * X * 2 + 2.0 ** -17
    return bool(((got.double() - want).abs() <= want * (rel + f.eps / 2) + f.smallest_normal * f.eps + 2.0 ** -126).all())


def plain_backward(a, grad, scale, buckets, causal, offset):
    """-> scores' and table's gradients, each with the bound of its roundings before the last"""
    n, cols = a.shape[2:]
    see = visible(n, cols, causal, offset)
    a, g = a.double().masked_fill(~see, 0), grad.double().masked_fill(~see, 0)
    dot, mag = (a * g).sum(-1, keepdim=True), (a * g).abs().sum(-1, keepdim=True)
    ds = a * (g - dot)
    err = a.abs() * (2.0 ** -22 * (g.abs() + dot.abs()) + 2.0 ** -18 * mag)
    hit = torch.nn.functional.one_hot(bucket_index(buckets, n, cols, offset), buckets.num_buckets).double()
    table, table_err = (torch.einsum("bhnc,nck->kh", v, hit) for v in (ds, err + 2.0 ** -17 * ds.abs()))
    return ds * scale, err * abs(scale), table, table_err


def grad_close(got, want, err):
    f = torch.finfo(got.dtype)
    return bool(((got.double() - want).abs() <= (want.abs() + err) * f.eps / 2 + err + f.smallest_normal * f.eps).all())


def _inputs(b, h, n, cols, dtype, buckets, causal, offset, seed):
    g = torch.Generator().manual_seed(seed)
    scores = (10 * torch.randn(b, h, n, cols, generator=g)).to(dtype).to(DEV)
    table = torch.randn(buckets.num_buckets, h, generator=g).to(dtype).to(DEV)
    grad = torch.randn(b, h, n, cols, generator=g).to(dtype).to(DEV)
    x = (scores.float() * 0.125).masked_fill(~visible(n, cols, causal, offset), -math.inf)
    return scores, table, torch.softmax(x, -1).nan_to_num(0.0).to(dtype), grad


def _check(scores, table, a, grad, buckets, mask=None, causal=False, offset=0, scale=0.125):
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    got = rb.softmax_forward_relative_bias(scores, scale, table, buckets, attention_mask=mask, causal=causal, q_offset=offset)
    assert got.shape == scores.shape and got.dtype == scores.dtype
    assert forward_close(got, *plain_forward(scores, scale, table, buckets, mask, causal, offset))
    ds, dt = rb.softmax_backward_relative_bias(a, grad, scale, buckets, causal=causal, q_offset=offset)
    want, err, want_t, err_t = plain_backward(a, grad, scale, buckets, causal, offset)
    assert ds.dtype == a.dtype and dt.dtype == torch.float32 and dt.shape == table.shape
    assert grad_close(ds, want, err) and grad_close(dt, want_t, err_t)
    return got, ds, dt


@pytest.mark.parametrize("side", [2, 3, 4, 7, 8, 16, 31, 32, 64, 128])
@pytest.mark.parametrize("distance", [65, 128, 200, 1000, 8192])
def test_edges_are_the_definition(side, distance):
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    for buckets in (RelativeBuckets(side, distance, False), RelativeBuckets(2 * side, distance, True)):
        edges = buckets.edges.tolist()
        assert len(edges) == side and edges == sorted(edges) and edges[0] == 0
        for r in sorted({0, 1, distance - 1, distance, *edges, *[e - 1 for e in edges[1:]]}):
            if r >= 0:
                assert sum(e <= r for e in edges) - 1 == bucket_by_definition(r, side, distance), r


def test_bucket_refusals():
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    assert RelativeBuckets(32, 128, True).edges.tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91]
    for args in ((31, 128, True), (2, 128, True), (1, 128, False), (0, 128, False), (258, 1000, True), (129, 1000, False), (32, 8, True), (32, 8193, True)):
        with pytest.raises(ValueError):
            RelativeBuckets(*args)


class Args(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("out", ctypes.c_void_p), ("table", ctypes.c_void_p), ("mask", ctypes.c_void_p),
                ("mask_b", ctypes.c_int64), ("mask_h", ctypes.c_int64), ("mask_row", ctypes.c_int64), ("host_edges", ctypes.c_void_p),
                ("batch", ctypes.c_int64), ("n", ctypes.c_int64), ("cols", ctypes.c_int64), ("q_offset", ctypes.c_int64), ("heads", ctypes.c_int),
                ("side", ctypes.c_int), ("both", ctypes.c_int), ("causal", ctypes.c_int), ("type", ctypes.c_int), ("table_type", ctypes.c_int),
                ("mask_type", ctypes.c_int), ("scale", ctypes.c_float)]


def test_the_library_refuses_before_it_launches():
    from hyc_lora_release_b200._lib import lib
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) & ~15
    edges = (ctypes.c_int32 * 4)(0, 1, 5, 9)

    def call(backward=False, **change):
        a = Args(p, p, p, p, None, 0, 0, 0, ctypes.addressof(edges), 0, 4, 64, 0, 2, 4, 1, 0, 0, 0, 0, 1.0)
        for name, value in change.items():
            setattr(a, name, value)
        if backward:
            return lib.hyc_softmax_relative_bias_bwd(ctypes.byref(a), p, None, 0, None)
        return lib.hyc_softmax_relative_bias_fwd(ctypes.byref(a), None)
    assert call() == call(n=0, batch=3) == 0
    assert lib.hyc_softmax_relative_bias_fwd(None, None) == -1 and call(host_edges=None) == -1
    for change in (dict(cols=0), dict(cols=131073), dict(heads=0), dict(batch=-1), dict(n=1 << 31), dict(batch=1 << 20, n=1 << 20), dict(side=0), dict(side=129),
                   dict(q_offset=1 << 30)):
        assert call(**change) == -3, change
    for values in ((1, 2, 3, 4), (0, 5, 4, 9), (0, 1, 2, 8193)):
        wrong = (ctypes.c_int32 * 4)(*values)
        assert call(host_edges=ctypes.addressof(wrong)) == -3
    assert call(type=3) == call(table_type=-1) == call(mask=p, mask_type=9) == -8
    assert call(batch=1, x=None) == call(batch=1, table=None) == call(backward=True, batch=1, grad=None) == -1
    assert call(batch=1, x=p + 1) == call(batch=1, mask=p + 1) == -4
    assert call(backward=True, batch=1) == -5
    assert lib.hyc_softmax_relative_bias_bwd(ctypes.byref(Args(host_edges=ctypes.addressof(edges), cols=4, heads=1, side=4)), None, None, 0, None) == -1


COLS = [1, 2, 7, 8, 31, 64, 255, 256, 257, 260, 512, 777, 1000, 1023, 1024, 1025, 1030, 1032]


@pytest.mark.gpu
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_row_lengths(cols, dtype):
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    for n, both, causal, offset in ((1, True, False, 0), (37, True, False, 3), (40, False, True, cols - 40), (70, True, True, 0)):
        buckets = RelativeBuckets(32, 128, both)
        _check(*_inputs(2, 3, n, cols, DTYPES[dtype], buckets, causal, offset, cols + n), buckets, causal=causal, offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1537, 2048, 4097, 4098, 5000, 16384, 16392, 20001, 40002, 131072])
def test_long_rows(cols):
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    for dtype, n, heads, both, causal in (("bf16", 3, 2, True, False), ("fp16", 1, 5, False, True), ("fp32", 5, 1, False, True)):
        buckets = RelativeBuckets(64, 1000, both)
        offset = cols - n
        _check(*_inputs(1, heads, n, cols, DTYPES[dtype], buckets, causal, offset, cols), buckets, causal=causal, offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("n,cols,heads", [(600, 600, 12), (1500, 1500, 4), (2048, 2048, 3), (1100, 3000, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_whole_maps(n, cols, heads, causal):
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    buckets = RelativeBuckets(32, 128, not causal)
    _check(*_inputs(2, heads, n, cols, torch.bfloat16, buckets, causal, 0, n + cols), buckets, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("num,distance,both", [(4, 3, True), (2, 5, False), (8, 64, True), (32, 128, False), (64, 256, True), (256, 8192, True), (128, 8192, False),
                                               (200, 120, True)])
def test_bucket_forms(num, distance, both):
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    buckets = RelativeBuckets(num, distance, both)
    for n, cols, offset in ((50, 300, -20), (50, 300, 500), (64, 1200, 40)):
        _check(*_inputs(1, 3, n, cols, torch.float32, buckets, False, offset, num + n), buckets, offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [200, 257, 1500])
def test_masks(cols):
    """Every layout and type of a mask; ends of sequences; rows that nothing or only the type's lowest value is left to."""
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    b, h, n = 2, 3, 20
    buckets = rb.RelativeBuckets(32, 128, True)
    scores, table, a, grad = _inputs(b, h, n, cols, torch.bfloat16, buckets, False, 0, cols)
    g = torch.Generator().manual_seed(1)
    for shape in ((b, h, n, cols), (1, 1, n, cols), (b, 1, 1, cols), (1, h, 1, cols), (1, 1, 1, cols)):
        for t in DTYPES.values():
            for low in (-math.inf, torch.finfo(t).min):
                mask = torch.where(torch.rand(shape, generator=g) < 0.7, torch.randn(shape, generator=g), low).to(t).to(DEV)
                _check(scores, table, a, grad, buckets, mask=mask)
                _check(scores, table, a, grad, buckets, mask=mask, causal=True, offset=5)
    wide = torch.randn(b, 1, n, cols + 3, generator=g).to(DEV)[..., 1:cols + 1]
    _check(scores, table, a, grad, buckets, mask=wide)
    _check(scores, table, a, grad, buckets, mask=wide.expand(b, h, n, cols))
    _check(scores, table, a, grad, buckets, mask=torch.randn(b, 1, cols, n, generator=g).to(DEV).transpose(2, 3))
    mask = torch.zeros(b, 1, n, cols, dtype=torch.bfloat16, device=DEV)
    mask[0, 0, 3] = -math.inf
    mask[1, 0, 4] = torch.finfo(torch.bfloat16).min
    got, _, _ = _check(scores, table, a, grad, buckets, mask=mask)
    assert bool((got[0, :, 3] == 0).all())
    assert torch.equal(got[1, :, 4], torch.full_like(got[1, :, 4], 1 / cols))
    # rows in front of the first column see nothing
    got, ds, _ = _check(scores, table, a, grad, buckets, causal=True, offset=-4)
    assert bool((got[:, :, :4] == 0).all()) and bool((ds[:, :, :4] == 0).all())


@pytest.mark.gpu
def test_what_a_causal_row_does_not_see_does_not_count():
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    for n in (300, 1300):
        buckets = rb.RelativeBuckets(32, 128, False)
        scores, table, a, grad = _inputs(1, 2, n, n, torch.float16, buckets, True, 0, n)
        want = rb.softmax_forward_relative_bias(scores, 0.125, table, buckets, causal=True), *rb.softmax_backward_relative_bias(a, grad, 0.125, buckets, causal=True)
        hidden = ~visible(n, n, True, 0)
        for value in (math.nan, math.inf, -math.inf):
            s2, a2, g2 = (t.masked_fill(hidden, value) for t in (scores, a, grad))
            got = rb.softmax_forward_relative_bias(s2, 0.125, table, buckets, causal=True), *rb.softmax_backward_relative_bias(a2, g2, 0.125, buckets, causal=True)
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        # a NaN that is seen stays in its row
        scores[0, 1, 200, 7] = math.nan
        got = rb.softmax_forward_relative_bias(scores, 0.125, table, buckets, causal=True)
        assert bool(got[0, 1, 200, :201].isnan().all()) and int(got.isnan().sum()) == 201


@pytest.mark.gpu
def test_layouts():
    """Begins off 16 bytes, heads behind the rows, expanded gradients, tables of other types and layouts, results in place."""
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    buckets = rb.RelativeBuckets(32, 128, True)
    for n, cols in ((30, 512), (10, 2048)):
        scores, table, a, grad = _inputs(2, 4, n, cols, torch.bfloat16, buckets, False, 0, n)
        whole = _check(scores, table, a, grad, buckets)
        for skip in (1, 2):
            moved = [torch.empty(t.numel() + skip, dtype=t.dtype, device=DEV)[skip:].view(t.shape).copy_(t) for t in (scores, a, grad)]
            _check(moved[0], table, moved[1], moved[2], buckets)
        turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (scores, a, grad)]
        again = _check(turned[0], table, turned[1], turned[2], buckets)
        assert all(torch.equal(x, y) for x, y in zip(whole, again))
        for shape in ((2, 4, n, 1), (1, 1, 1, cols), (1, 4, 1, 1)):
            _check(scores, table, a, torch.randn(shape, device=DEV).to(torch.bfloat16).expand(grad.shape), buckets)
        _check(scores, table.float(), a, grad, buckets)
        _check(scores, table.t().contiguous().t(), a, grad, buckets)
        mine = scores.clone()
        assert rb.softmax_forward_relative_bias(mine, 0.125, table, buckets, inplace=True) is not None and torch.equal(mine, whole[0])


@pytest.mark.gpu
def test_same_bits_again_and_in_graphs_on_another_stream():
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    buckets = rb.RelativeBuckets(32, 128, False)
    scores, table, a, grad = _inputs(2, 4, 333, 333, torch.bfloat16, buckets, True, 0, 3)
    long = _inputs(1, 2, 9, 20000, torch.bfloat16, buckets, True, 19991, 4)

    def both():
        return (rb.softmax_forward_relative_bias(scores, 0.125, table, buckets, causal=True),
                *rb.softmax_backward_relative_bias(a, grad, 0.125, buckets, causal=True),
                rb.softmax_forward_relative_bias(long[0], 0.125, long[1], buckets, causal=True, q_offset=19991),
                *rb.softmax_backward_relative_bias(long[2], long[3], 0.125, buckets, causal=True, q_offset=19991))
    first = both()
    assert all(torch.equal(x, y) for x, y in zip(first, both()))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = both()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, y) for x, y in zip(first, side))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, both()))
    scores.neg_()
    grad.mul_(0.5)
    again = both()
    for graph, out in graphs[::-1]:
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(out, again))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """The last rows of a map of more than 2^32 bytes and 2^31 elements, against the same rows on their own."""
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    n, cols = 66000, 32768
    buckets = rb.RelativeBuckets(32, 128, True)
    scores = torch.zeros(1, 1, n, cols, dtype=torch.bfloat16, device=DEV)
    scores[0, 0, -7:] = torch.randn(7, cols, device=DEV)
    table = torch.randn(32, 1, device=DEV)
    got = rb.softmax_forward_relative_bias(scores, 0.5, table, buckets, inplace=True)[:, :, -7:]
    tail = torch.zeros(1, 1, 7, cols, dtype=torch.bfloat16, device=DEV)
    torch.manual_seed(0)
    fresh = torch.randn(7, cols, device=DEV).to(torch.bfloat16)
    scores[0, 0, -7:] = fresh
    tail[0, 0] = fresh
    got = rb.softmax_forward_relative_bias(scores, 0.5, table, buckets, inplace=True)[:, :, -7:]
    want, X = plain_forward(tail, 0.5, table, buckets, None, False, n - 7)
    assert forward_close(got, want, X)
    # backward: the tail alone has a gradient
    grad = torch.zeros_like(scores)
    grad[0, 0, -7:] = torch.randn(7, cols, device=DEV)
    ds, dt = rb.softmax_backward_relative_bias(scores, grad, 0.5, buckets)
    want, err, want_t, err_t = plain_backward(got, grad[:, :, -7:], 0.5, buckets, False, n - 7)
    assert grad_close(ds[:, :, -7:], want, err) and grad_close(dt, want_t, err_t) and bool((ds[:, :, :-7:1000] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("b,h,n,cols", [(4, 16, 1, 1670), (3, 1, 3, 1277), (8, 12, 1, 4000), (2, 3, 1, 13384)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_table_gradient_of_few_rows(b, h, n, cols, dtype):
    """A bucket that holds nearly all of a row, whose sum nearly cancels.  In units of 2^-24: one rounding per element (a g is exact in
    fp32), the row's product sum off by its own rounding and by at most 3 + 2 additions of a lane before 64 bits, and the result's."""
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets, softmax_backward_relative_bias
    buckets, offset = RelativeBuckets(8, 64, False), cols - n
    g = torch.Generator(device=DEV).manual_seed(cols)
    dt = DTYPES[dtype]
    a = torch.softmax(torch.randn(b, h, n, cols, generator=g, device=DEV) * 1.5, -1)
    a = a.masked_fill(~visible(n, cols, True, offset), 0.0).to(dt)
    grad = (torch.randn(b, h, n, cols, generator=g, device=DEV) * 0.05).to(dt)
    _, got = softmax_backward_relative_bias(a, grad, 0.125, buckets, causal=True, q_offset=offset)
    x = a.double()
    prod = x * grad.double()
    dot, mag = prod.sum(-1, keepdim=True), prod.abs().sum(-1, keepdim=True)
    ds = x * (grad.double() - dot)
    err = ds.abs() + x * (dot.abs() + 5 * mag)
    hit = torch.nn.functional.one_hot(bucket_index(buckets, n, cols, offset), 8).double()
    want, bound = (torch.einsum("bhij,ijk->kh", v, hit) for v in (ds, err))
    assert bool(((got.double() - want).abs() <= 2.0 ** -24 * (bound + want.abs())).all())


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of the 64-bit formula along one direction of scores and table (truncation of order step^2)."""
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    for n, cols, causal in ((40, 40, True), (33, 70, False)):
        buckets = rb.RelativeBuckets(16, 40, not causal)
        scores, table, _, grad = _inputs(2, 2, n, cols, torch.float32, buckets, causal, 0, n)
        a = rb.softmax_forward_relative_bias(scores, 0.125, table, buckets, causal=causal)
        ds, dt = rb.softmax_backward_relative_bias(a, grad, 0.125, buckets, causal=causal)
        g = torch.Generator().manual_seed(2)
        vs, vt = (torch.randn(t.shape, generator=g, dtype=torch.float64).to(DEV) for t in (scores, table))

        def loss(step):
            return (plain_forward(scores.double() + step * vs, 0.125, table.double() + step * vt, buckets, None, causal, 0)[0] * grad.double()).sum()
        difference = (loss(1e-4) - loss(-1e-4)) / 2e-4
        parts = torch.cat(((ds.double() * vs).reshape(-1), (dt.double() * vt).reshape(-1)))
        assert abs(float(parts.sum() - difference)) <= 1e-5 * float(parts.abs().sum())


@pytest.mark.gpu
def test_empty_and_refusals():
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    buckets = rb.RelativeBuckets(32, 128, True)
    scores, table, a, grad = _inputs(2, 3, 5, 16, torch.bfloat16, buckets, False, 0, 1)
    for empty in (scores[:0], scores[:, :, :0]):
        assert rb.softmax_forward_relative_bias(empty, 1.0, table, buckets).shape == empty.shape
        ds, dt = rb.softmax_backward_relative_bias(empty, empty, 1.0, buckets)
        assert ds.shape == empty.shape and bool((dt == 0).all())

    def fwd(scores=scores, table=table, buckets=buckets, **kw):
        return rb.softmax_forward_relative_bias(scores, 1.0, table, buckets, **kw)
    zeros = lambda *s: torch.zeros(s, device=DEV)
    for call in (lambda: fwd(scores[0]), lambda: fwd(scores[..., :0]), lambda: fwd(scores[:, :0], table[:, :0]), lambda: fwd(scores.double()),
                 lambda: fwd(table=table[:31]), lambda: fwd(table=table[:, :2]), lambda: fwd(table=table.double()), lambda: fwd(q_offset=1 << 40),
                 lambda: fwd(buckets=rb.RelativeBuckets(32, 128, False), table=table[:16]), lambda: fwd(attention_mask=zeros(2, 1, 5, 15)),
                 lambda: fwd(attention_mask=zeros(5, 16)), lambda: fwd(attention_mask=zeros(2, 2, 5, 16)), lambda: fwd(attention_mask=zeros(3, 1, 5, 16)),
                 lambda: fwd(attention_mask=zeros(1, 1, 4, 16)), lambda: fwd(attention_mask=zeros(2, 1, 5, 16).bool()),
                 lambda: fwd(scores.transpose(2, 3), inplace=True), lambda: rb.softmax_backward_relative_bias(a, grad[:1], 1.0, buckets),
                 lambda: rb.softmax_backward_relative_bias(a, grad.float(), 1.0, buckets)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="different devices|only on CUDA"):
        fwd(table=table.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,b,h,n,cols,offset", [
    ("bf16", 2, 20, 900, 760, 0), ("bf16", 2, 20, 900, 768, 0), ("fp16", 2, 16, 1500, 1280, 0), ("bf16", 1, 20, 1700, 1536, 0), ("bf16", 1, 16, 2000, 1792, 0),
    ("bf16", 2, 20, 700, 768, 400), ("bf16", 2, 20, 300, 1536, 2000), ("fp32", 2, 16, 900, 768, 0), ("bf16", 2, 20, 900, 766, 0), ("fp16", 2, 20, 900, 767, 3),
    ("bf16", 1, 20, 300, 4864, 4864), ("fp16", 1, 20, 400, 4870, 4600)])
def test_causal_rows_behind_the_last_column(dtype, b, h, n, cols, offset):
    """Rows whose own position lies behind the map's last column see all of it, and the diagonals' sums leave the columns on the right:
    columns that end at or close to a block of 256 inside a warp's span, more rows than columns, and keys that all lie behind."""
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets, softmax_backward_relative_bias
    buckets = RelativeBuckets(32, 128, False)
    g = torch.Generator(device=DEV).manual_seed(cols)
    see = visible(n, cols, True, offset)
    x = torch.randn(b, h, n, cols, generator=g, device=DEV).masked_fill(~see, -math.inf)
    a, grad = torch.softmax(x, -1).to(DTYPES[dtype]), torch.randn(b, h, n, cols, generator=g, device=DEV).to(DTYPES[dtype])
    ds, dt = softmax_backward_relative_bias(a, grad, 0.125, buckets, causal=True, q_offset=offset)
    want, err, want_t, err_t = plain_backward(a, grad, 0.125, buckets, True, offset)
    assert grad_close(ds, want, err) and grad_close(dt, want_t, err_t)


def test_buckets_made_where_another_device_is_the_default():
    """A model that is built under a device's context: the edges are host data all the same."""
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    with torch.device("meta"):
        buckets = RelativeBuckets(32, 128, True)
    assert buckets.edges.device.type == "cpu" and torch.equal(buckets.edges, RelativeBuckets(32, 128, True).edges)


@pytest.mark.gpu
@pytest.mark.parametrize("n,cols", [(6, 200), (40, 1001), (6, 1500), (6, 20000)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_values_close_to_the_types_lowest(n, cols, dtype):
    """Scores, table entries and masks at and near the ends of a type's range are numbers like others: a row of nothing but the lowest
    value shares its 1, the largest of several far ones takes it all, and beside ordinary ones they are 0.  Where the exponents of a row are far
    out, two of them are equal or so far apart that one exponential is 0: what is left are the sum's and the result's roundings."""
    from hyc_lora_release_b200.operators import relative_bias_kernels as rb
    t = DTYPES[dtype]
    low = torch.finfo(t).min
    buckets = rb.RelativeBuckets(32, 128, True)
    scores, table, _, _ = _inputs(2, 3, n, cols, t, buckets, False, 0, n + cols)
    scores[0, :, 0] = low                                # nothing else
    scores[0, :, 1, ::2] = low                           # beside ordinary ones
    scores[0, :, 2] = low / 2
    scores[0, :, 2, 5] = low / 4                         # the largest of far ones
    scores[1, :, 0] = -low / 2
    scores[1, :, 0, 3] = -low * 0.75                     # far on the other side
    mask = torch.zeros(2, 1, n, cols, dtype=t, device=DEV)
    mask[1, :, 1] = low * 0.875
    mask[1, :, 1, 7] = low * 0.6875                      # masks keep their order
    mask[1, :, 2] = low
    far = {(0, 0), (0, 2), (1, 0), (1, 1), (1, 2)}
    one_value = table.clone()
    one_value[:] = low                                   # .. and so does a table of them
    for given_table, m, everywhere in ((table, mask, False), (table.float(), mask.float(), False), (one_value, None, True)):
        s = torch.zeros_like(scores) if everywhere else scores
        want, X = plain_forward(s, 1.0, given_table, buckets, m, False, 0)
        got = rb.softmax_forward_relative_bias(s, 1.0, given_table, buckets, attention_mask=m)
        for i in range(2):
            for row in range(n):
                x = torch.zeros_like(X[i, :, row]) if everywhere or (i, row) in far else X[i, :, row]
                assert forward_close(got[i, :, row], want[i, :, row], x), (i, row)
        assert bool((got.double().sum(-1) - 1).abs().max() < 0.02)
    # -infinity is still nothing
    scores[0, :, 0] = -math.inf
    got = rb.softmax_forward_relative_bias(scores, 1.0, table, buckets)
    assert bool((got[0, :, 0] == 0).all())


FIRST_CALL = """
import ctypes, torch
from hyc_lora_release_b200.operators import relative_bias_kernels as rb
driver = ctypes.CDLL("libcuda.so.1")

class Params(ctypes.Structure):      # CUDA_KERNEL_NODE_PARAMS_v2
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3), ("smem", ctypes.c_uint),
                ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kernel", ctypes.c_void_p), ("context", ctypes.c_void_p)]

scores = torch.zeros(2, 32, 40, 8192, dtype=torch.bfloat16, device="cuda")
mask, table, buckets = torch.zeros(1, 1, 1, 8192, device="cuda"), torch.zeros(32, 32, device="cuda"), rb.RelativeBuckets(32, 128, True)
torch.cuda.synchronize()

def launch():
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        rb.softmax_forward_relative_bias(scores, 1.0, table, buckets, attention_mask=mask)
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert driver.cuGraphGetNodes(raw, None, ctypes.byref(count)) == 0 and count.value == 1
    node, p = (ctypes.c_void_p * 1)(), Params()
    assert driver.cuGraphGetNodes(raw, node, ctypes.byref(count)) == 0
    assert driver.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node[0]), ctypes.byref(p)) == 0
    return list(p.grid) + list(p.block) + [p.smem]

first, second = launch(), launch()
assert first == second, (first, second)
print("same", first)
"""


@pytest.mark.gpu
def test_the_first_call_is_cut_as_later_ones_are():
    """In a process of its own: what one launch of long rows is, recorded on the first call and on the second."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr
