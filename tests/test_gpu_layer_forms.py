"""A layer built from the operators of other layer forms, as a training step runs them: projection with bias, norms and rotation of q and k,
softmax with a learned position bias, output projection with residual, MLP product with an activation and one with residual, and back.

Every operator is checked on what the step hands it (the tolerances of its own tests).  The gradients of the whole are compared with
autograd on the formulas in 64 bits, in norm: a path through the step passes at most 24 roundings to bf16, each off by half a step
(2^-8) relative to the norm, and products of random factors carry a relative error on as it is: 24 * 2^-8."""
import math
import threading

import pytest
import torch

import test_gpu_linear as tl
import test_gpu_qk_norm as tq
import test_gpu_relative_bias as tr

pytestmark = pytest.mark.gpu
DEV, BF16 = "cuda", torch.bfloat16
B, M, H, KV, D, INNER = 2, 197, 4, 2, 64, 520
HIDDEN, EPS, SCALE = H * D, 1e-6, D ** -0.5


def _parameters(seed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s, std=1.0: (std * torch.randn(*s, generator=g)).to(BF16).to(DEV)
    wide = (H + 2 * KV) * D
    return dict(x=rn(B, M, HIDDEN), wqkv=rn(wide, HIDDEN, std=HIDDEN ** -0.5), bqkv=rn(wide, std=0.3), qw=1 + rn(D, std=0.2), kw=1 + rn(D, std=0.2),
                table=rn(32, H), wo=rn(HIDDEN, HIDDEN, std=HIDDEN ** -0.5), bo=rn(HIDDEN, std=0.3), wu=rn(INNER, HIDDEN, std=HIDDEN ** -0.5),
                bu=rn(INNER, std=0.3), wd=rn(HIDDEN, INNER, std=INNER ** -0.5), bd=rn(HIDDEN, std=0.3)), rn(B, M, HIDDEN)


def _tables():
    return tq._tables(M, D, torch.float32)


def _by_group(t):      # heads of k or v for every head of q
    return t.repeat_interleave(H // KV, 2)


def _step(p, dy, cos, sin, buckets):
    """-> result, gradients by name, and what every operator was given and gave"""
    from hyc_lora_release_b200.operators import linear_kernels as lk, qk_norm_kernels as qn, relative_bias_kernels as rb
    seen = {}
    qkv, _ = lk.linear_act_forward(p["x"], p["wqkv"], p["bqkv"])
    heads = qkv.view(B, M, H + 2 * KV, D)
    q0, k0, v = heads[:, :, :H], heads[:, :, H:H + KV], _by_group(heads[:, :, H + KV:]).transpose(1, 2)
    q, k = qn.qk_norm_rope_forward(q0, k0, p["qw"], p["kw"], cos, sin, EPS)
    qt, kt = q.transpose(1, 2), _by_group(k).transpose(1, 2)
    scores = qt @ kt.transpose(2, 3)
    a = rb.softmax_forward_relative_bias(scores, SCALE, p["table"], buckets, causal=True)
    o = (a @ v).transpose(1, 2).reshape(B, M, HIDDEN)
    x1, _ = lk.linear_act_forward(o, p["wo"], p["bo"], residual=p["x"])
    u, pre = lk.linear_act_forward(x1, p["wu"], p["bu"], "gelu", save_pre=True)
    y, _ = lk.linear_act_forward(u, p["wd"], p["bd"], residual=x1)

    du, dwd, dbd = lk.linear_act_backward(dy, u, p["wd"])
    dx1, dwu, dbu = lk.linear_act_backward(du, x1, p["wu"], "gelu", pre=pre)
    g1 = dx1 + dy
    do, dwo, dbo = lk.linear_act_backward(g1, o, p["wo"])
    dot = do.view(B, M, H, D).transpose(1, 2)
    da, dv = dot @ v.transpose(2, 3), a.transpose(2, 3) @ dot
    ds, dtable = rb.softmax_backward_relative_bias(a, da, SCALE, buckets, causal=True)
    dq, dk = (ds @ kt).transpose(1, 2), (ds.transpose(2, 3) @ qt).transpose(1, 2)
    sum_group = lambda t: t.reshape(B, M, KV, H // KV, D).sum(3)
    dk = sum_group(dk)
    dq0, dk0, dqw, dkw = qn.qk_norm_rope_backward(dq, dk, q0, k0, p["qw"], p["kw"], cos, sin, EPS)
    dqkv = torch.cat((dq0, dk0, sum_group(dv.transpose(1, 2))), 2).view(B, M, -1)
    dx, dwqkv, dbqkv = lk.linear_act_backward(dqkv, p["x"], p["wqkv"])
    grads = dict(x=dx + g1, wqkv=dwqkv, bqkv=dbqkv, qw=dqw, kw=dkw, table=dtable, wo=dwo, bo=dbo, wu=dwu, bu=dbu, wd=dwd, bd=dbd)
    seen.update(locals())
    return y, grads, seen


def _exact(p, dy, cos, sin, buckets):
    w = {n: t.double().requires_grad_() for n, t in p.items()}
    heads = (w["x"] @ w["wqkv"].t() + w["bqkv"]).view(B, M, H + 2 * KV, D)
    c, s = tq._angles(cos, sin, None, B, M, D)

    def norm(t, weight):
        return tq._turn(t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * weight, c, s, D)
    q, k = norm(heads[:, :, :H], w["qw"]), _by_group(norm(heads[:, :, H:H + KV], w["kw"]))
    sc = torch.einsum("bihd,bjhd->bhij", q, k) * SCALE + w["table"][tr.bucket_index(buckets, M, M, 0)].permute(2, 0, 1)
    a = torch.softmax(sc.masked_fill(~tr.visible(M, M, True, 0), -math.inf), -1)
    o = torch.einsum("bhij,bjhd->bihd", a, _by_group(heads[:, :, H + KV:])).reshape(B, M, HIDDEN)
    x1 = o @ w["wo"].t() + w["bo"] + w["x"]
    y = tl.act_of(x1 @ w["wu"].t() + w["bu"], "gelu") @ w["wd"].t() + w["bd"] + x1
    return y.detach(), dict(zip(w, torch.autograd.grad((y * dy.double()).sum(), list(w.values()))))


def _setup(seed):
    from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
    return (*_parameters(seed), *_tables(), RelativeBuckets(32, 128, False))


def test_every_operator_on_what_the_step_hands_it():
    p, dy, cos, sin, buckets = _setup(1)
    y, grads, t = _step(p, dy, cos, sin, buckets)
    tl.check_forward(p["x"], p["wqkv"], p["bqkv"], "none", None, t["qkv"], None)
    tl.check_forward(t["o"], p["wo"], p["bo"], "none", p["x"], t["x1"], None)
    tl.check_forward(t["x1"], p["wu"], p["bu"], "gelu", None, t["u"], t["pre"])
    tl.check_forward(t["u"], p["wd"], p["bd"], "none", t["x1"], y, None)
    tl.check_backward(dy, t["u"], p["wd"], "none", None, t["du"], t["dwd"], t["dbd"])
    tl.check_backward(t["du"], t["x1"], p["wu"], "gelu", t["pre"], t["dx1"], t["dwu"], t["dbu"])
    tl.check_backward(t["g1"], t["o"], p["wo"], "none", None, t["do"], t["dwo"], t["dbo"])
    tl.check_backward(t["dqkv"], p["x"], p["wqkv"], "none", None, t["dx"], t["dwqkv"], t["dbqkv"])
    assert tr.forward_close(t["a"], *tr.plain_forward(t["scores"], SCALE, p["table"], buckets, None, True, 0))
    ds, err, dtable, err_t = tr.plain_backward(t["a"], t["da"], SCALE, buckets, True, 0)
    assert tr.grad_close(t["ds"], ds, err) and tr.grad_close(t["dtable"], dtable, err_t)
    c, s = tq._angles(cos, sin, None, B, M, D)
    for x, w, out, g, dx, dw in ((t["q0"], p["qw"], t["q"], t["dq"], t["dq0"], t["dqw"]), (t["k0"], p["kw"], t["k"], t["dk"], t["dk0"], t["dkw"])):
        assert tq.close(out, *tq.plain_forward(x, w, c, s, D))
        want, want_w, mag, mag_w = tq.plain_backward(g, x, w, c, s, D)
        assert tq.close(dx, want, mag) and tq.close(dw, want_w, mag_w, (x.shape[0] * x.shape[1] * x.shape[2] + 32) * 2.0 ** -24)


def test_gradients_of_the_whole_step():
    p, dy, cos, sin, buckets = _setup(2)
    y, grads, _ = _step(p, dy, cos, sin, buckets)
    want_y, want = _exact(p, dy, cos, sin, buckets)
    assert float((y.double() - want_y).norm() / want_y.norm()) <= 24 * 2.0 ** -8
    for name, g in grads.items():
        assert g.shape == want[name].shape
        assert float((g.double() - want[name]).norm() / want[name].norm()) <= 24 * 2.0 ** -8, name


def test_a_step_as_a_graph_beside_an_eager_one():
    """The step has no state: recorded, replayed with other inputs and interleaved with eager steps on another stream, the same bits."""
    p, dy, cos, sin, buckets = _setup(3)
    other, dy2, *_ = _setup(4)
    _step(p, dy, cos, sin, buckets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grads, _ = _step(p, dy, cos, sin, buckets)
    for n in p:
        p[n].copy_(other[n])
    dy.copy_(dy2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph.replay()
    with torch.cuda.stream(stream):
        y2, grads2, _ = _step(other, dy2, cos, sin, buckets)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads)


def test_steps_of_several_threads_at_once():
    """Each with a stream of its own: tensor memory, shared memory and workspaces are each call's own."""
    p, dy, cos, sin, buckets = _setup(5)
    y, grads, _ = _step(p, dy, cos, sin, buckets)
    torch.cuda.synchronize()
    wrong = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                y2, grads2, _ = _step(p, dy, cos, sin, buckets)
                if not (torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads)):
                    wrong.append(1)
            stream.synchronize()
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
