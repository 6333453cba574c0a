"""Operators of a transformer layer that is built otherwise than the fused one, each with its backward pass: what is
measured, in plain torch operations and through the framework's entry points (``own``).

  qknorm   RMS norms of the query and key heads with the rotary embedding in the same pass
           (``operators.qk_norm_kernels.qk_norm_rope_forward / _backward``)
  relbias  softmax of attention scores with a learned bias per bucket of relative positions, and its gradient
           (``operators.relative_bias_kernels.softmax_forward_relative_bias / softmax_backward_relative_bias``)
  linear   a product with bias, activation and residual in its epilogue
           (``operators.linear_kernels.linear_act_forward / linear_act_backward``)

A layer runs them in this order: projections (linear), norms and rotation of q and k, scores, softmax, output projection
with the residual, MLP products with an activation.
"""
import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # eight sequences that generate, one token each at a position of its own: latency
        dict(name="qknorm-fwd-8x1-decode", op="qknorm", way="fwd", batch=8, seq=1, hq=32, hk=8, d=128, rot=128, dtype="bf16", table="fp32",
             packed=True, positions=True),
        # a full micro-batch of grouped heads, q and k as slices of one projection's result
        dict(name="qknorm-fwd-4x2048", op="qknorm", way="fwd", batch=4, seq=2048, hq=32, hk=8, d=128, rot=128, dtype="bf16", table="bf16",
             packed=True, positions=False),
        # training step of one long sequence, as many key as query heads, with the gradients of both norm weights
        dict(name="qknorm-bwd-1x2048", op="qknorm", way="bwd", batch=1, seq=2048, hq=32, hk=32, d=128, rot=128, dtype="bf16", table="bf16",
             packed=False, positions=False),
        # a small model on a ragged batch, half of each head rotated
        dict(name="qknorm-bwd-3x333", op="qknorm", way="bwd", batch=3, seq=333, hq=12, hk=12, d=64, rot=32, dtype="fp16", table="fp32",
             packed=True, positions=True),
        # one token of each of eight sequences over a cache of odd length: latency, few long rows
        dict(name="relbias-fwd-8x32x1x1537", op="relbias", way="fwd", batch=8, heads=32, n=1, cols=1537, buckets=32, distance=128,
             both=False, causal=True, mask="padding", dtype="fp16"),
        # an encoder's map at the size of the map benchmark, padded batch
        dict(name="relbias-fwd-4x32x512", op="relbias", way="fwd", batch=4, heads=32, n=512, cols=512, buckets=32, distance=128,
             both=True, causal=False, mask="padding", dtype="bf16"),
        # training step of one long causal sequence: map and its gradient in, gradients of scores and table out
        dict(name="relbias-bwd-1x32x2048", op="relbias", way="bwd", batch=1, heads=32, n=2048, cols=2048, buckets=32, distance=128,
             both=False, causal=True, mask="none", dtype="bf16"),
        # a padded instruction batch of an odd length
        dict(name="relbias-bwd-2x12x333", op="relbias", way="bwd", batch=2, heads=12, n=333, cols=333, buckets=64, distance=256,
             both=True, causal=False, mask="none", dtype="bf16"),
        # one token through an MLP's first product: the weight is what is read
        dict(name="linear-fwd-1tok", op="linear", way="fwd", tokens=1, k=4096, n=11008, act="gelu_tanh", bias=True, residual=False,
             pre=False, dtype="bf16"),
        # output product of a ragged batch, residual added
        dict(name="linear-fwd-333tok", op="linear", way="fwd", tokens=333, k=11008, n=4096, act="none", bias=True, residual=True,
             pre=False, dtype="fp16"),
        # the largest forward product of a micro-batch, what backward needs saved
        dict(name="linear-fwd-8192tok", op="linear", way="fwd", tokens=8192, k=4096, n=14336, act="gelu", bias=True, residual=False,
             pre=True, dtype="bf16"),
        # training step of the MLP's first product: gradients of input, weight and bias
        dict(name="linear-bwd-2048tok", op="linear", way="bwd", tokens=2048, k=4096, n=11008, act="silu", bias=True, residual=False,
             pre=True, dtype="bf16"),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of ``step`` between the two, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    """One case of the same ranges: any operator, direction, type and size, no dearer than the largest listed one."""
    op, way = rng.choice(["qknorm", "relbias", "linear"]), rng.choice(["fwd", "bwd"])
    while True:
        if op == "qknorm":
            hk = rng.choice([1, 2, 4, 8, 12, 32])
            d = rng.choice([64, 80, 96, 128, 256])
            c = dict(op=op, way=way, batch=_spread(rng, 1, 16), seq=1 if way == "fwd" and rng.random() < 0.3 else _spread(rng, 1, 8192),
                     hq=hk * rng.choice([1, 2, 4, 7]), hk=hk, d=d, rot=rng.choice([d, d, d // 32 * 16]),
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), table=rng.choice(["bf16", "fp32"]),
                     packed=rng.random() < 0.5, positions=rng.random() < 0.5)
            if c["batch"] * c["seq"] * (c["hq"] + c["hk"]) * d <= 4 * 2048 * 40 * 128:
                return c
        elif op == "relbias":
            form = rng.choice(["self", "self", "token", "other"])
            cols = _spread(rng, 1, 2048) if form != "token" else _spread(rng, 16, 32768)
            n = cols if form == "self" else (1 if form == "token" else _spread(rng, 1, 2048))
            causal = form == "token" or rng.random() < 0.5
            if causal and n > cols:
                n = cols
            c = dict(op=op, way=way, batch=_spread(rng, 1, 16), heads=rng.choice([1, 3, 8, 12, 16, 32]), n=n, cols=cols,
                     buckets=rng.choice([8, 32, 64]), distance=rng.choice([64, 128, 256, 1000]), both=rng.random() < 0.5, causal=causal,
                     mask=rng.choice(["none", "padding", "full"]) if way == "fwd" else "none", dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            if c["batch"] * c["heads"] * n * cols <= 32 * 2048 * 2048 // (2 if c["dtype"] == "fp32" else 1):
                return c
        else:
            c = dict(op=op, way=way, tokens=_spread(rng, 1, 8192), k=_spread(rng, 64, 14336, 8), n=_spread(rng, 64, 14336, 8),
                     act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7,
                     residual=way == "fwd" and rng.random() < 0.5, pre=way == "bwd" or rng.random() < 0.5,
                     dtype=rng.choice(["bf16", "bf16", "fp16"]))
            if c["tokens"] * c["k"] * c["n"] * (2 if way == "bwd" else 1) <= 8192 * 4096 * 14336:
                return c


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std)

    if case["op"] == "qknorm":
        b, m, hq, hk, d, rot = (case[x] for x in ("batch", "seq", "hq", "hk", "d", "rot"))

        def heads():
            # channels of unlike size, as projections give them; packed: slices of one [.., (hq + 2 hk) d] result
            size = torch.exp(rn(d, std=0.5))
            if case["packed"]:
                qkv = (rn(b, m, hq + 2 * hk, d) * size).to(dt)
                return qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
            return (rn(b, m, hq, d) * size).to(dt), (rn(b, m, hk, d) * size).to(dt)
        q, k = heads()
        length = m if not case["positions"] else max(4096, m)
        s = dict(case=case, q=q, k=k, qw=(1 + rn(d, std=0.2)).to(dt), kw=(1 + rn(d, std=0.2)).to(dt), rot=rot)
        freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * freq[None]
        angle = torch.cat((angle, angle), 1)
        s["cos"], s["sin"] = angle.cos().to(DTYPES[case["table"]]), angle.sin().to(DTYPES[case["table"]])
        s["pos"] = None
        if case["positions"]:      # every sequence begins somewhere of its own
            first = torch.randint(0, length - m + 1, (b, 1), generator=g, device="cuda")
            s["pos"] = first + torch.arange(m, device="cuda")[None]
        if case["way"] == "bwd":
            s["dq"], s["dk"] = rn(b, m, hq, d).to(dt), rn(b, m, hk, d).to(dt)
        return s
    if case["op"] == "relbias":
        b, h, n, cols = (case[x] for x in ("batch", "heads", "n", "cols"))
        s = dict(case=case, scale=0.125, offset=cols - n if case["causal"] else 0, table=rn(case["buckets"], h).to(dt), mask=None)
        if own:
            from hyc_lora_release_b200.operators.relative_bias_kernels import RelativeBuckets
            s["buckets"] = RelativeBuckets(case["buckets"], case["distance"], case["both"])
        scores = rn(b, h, n, cols, std=12.0)
        low = torch.finfo(dt).min
        if case["mask"] == "padding":      # ends of the sequences, additive
            end = torch.randint((cols + 1) // 2, cols + 1, (b, 1), generator=g, device="cuda")
            s["mask"] = torch.where(torch.arange(cols, device="cuda")[None] < end, 0.0, low).to(dt).view(b, 1, 1, cols)
        elif case["mask"] == "full":       # a tenth of the places of every row
            s["mask"] = torch.where(torch.rand(1, 1, n, cols, generator=g, device="cuda") < 0.9, 0.0, low).to(dt)
        if case["way"] == "fwd":
            s["scores"] = scores.to(dt)
            return s
        x = scores * s["scale"]
        if case["causal"]:
            x = x.masked_fill(_later(n, cols, s["offset"]), -math.inf)
        s["a"] = torch.softmax(x, -1).to(dt)
        s["grad"] = rn(b, h, n, cols, std=0.05).to(dt)
        return s
    t, k, n = case["tokens"], case["k"], case["n"]
    s = dict(case=case, x=rn(t, k).to(dt), w=rn(n, k, std=k ** -0.5).to(dt), b=None, res=None, pre=None)
    if case["bias"]:
        s["b"] = rn(n, std=0.5).to(dt)
    if case["residual"]:
        s["res"] = rn(t, n).to(dt)
    if case["way"] == "bwd":
        s["dy"] = rn(t, n, std=0.1).to(dt)
        s["pre"] = rn(t, n).to(dt) if case["act"] != "none" else None
    return s


def _later(n, cols, offset):
    """Columns behind a row's own position."""
    return torch.arange(cols, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + offset


# ------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    return (_own if own else _plain)[case["op"], case["way"]](s)


def _rope(x, s, inverse=False):
    rot, half = s["rot"], s["rot"] // 2
    m = x.shape[1]
    pos = s["pos"] if s["pos"] is not None else torch.arange(m, device=x.device)[None]
    c, sn = s["cos"][:, :half].float()[pos][:, :, None], s["sin"][:, :half].float()[pos][:, :, None]
    if inverse:
        sn = -sn
    x1, x2 = x[..., :half], x[..., half:rot]
    return torch.cat((x1 * c - x2 * sn, x2 * c + x1 * sn, x[..., rot:]), -1)


def _plain_qknorm_fwd(s):
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        f = x.float()
        y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * w.float()
        out.append(_rope(y, s).to(x.dtype))
    return tuple(out)


def _plain_qknorm_bwd(s):
    grads, weights = [], []
    for x, w, dy in ((s["q"], s["qw"], s["dq"]), (s["k"], s["kw"], s["dk"])):
        f = x.float()
        r = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
        xn = f * r
        dn = _rope(dy.float(), s, inverse=True)
        weights.append((dn * xn).double().sum((0, 1, 2)).to(w.dtype))
        dxn = dn * w.float()
        grads.append((r * (dxn - xn * (dxn * xn).mean(-1, keepdim=True))).to(x.dtype))
    return (*grads, *weights)


def _edges(side, distance):
    """Smallest distance of each bucket of one side: one bucket per distance up to half of them, the rest evenly over the
    logarithm up to ``distance``, in whole numbers."""
    exact = side // 2
    rest = side - exact
    edges = list(range(exact))
    for t in range(rest):
        want = exact ** (rest - t) * distance ** t      # distance_t ** rest
        r = int(round(exact * (distance / exact) ** (t / rest)))
        while r ** rest >= want:
            r -= 1
        edges.append(r + 1)
    return edges


def _bucket_map(case, n, cols, offset):
    side = case["buckets"] // 2 if case["both"] else case["buckets"]
    edges = torch.tensor(_edges(side, case["distance"]), device="cuda")
    ahead = torch.arange(cols, device="cuda")[None] - (torch.arange(n, device="cuda")[:, None] + offset)
    if case["both"]:
        return torch.bucketize(ahead.abs(), edges, right=True) - 1 + side * (ahead > 0)
    return torch.bucketize((-ahead).clamp_min(0), edges, right=True) - 1


def _plain_relbias_fwd(s):
    case = s["case"]
    n, cols = case["n"], case["cols"]
    bias = s["table"].float()[_bucket_map(case, n, cols, s["offset"])].permute(2, 0, 1)
    x = s["scores"].float() * s["scale"] + bias
    if s["mask"] is not None:
        x = x + s["mask"].float()
    if case["causal"]:
        x = x.masked_fill(_later(n, cols, s["offset"]), -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m)
    return (p / p.sum(-1, keepdim=True)).to(s["scores"].dtype)


def _plain_relbias_bwd(s):
    case = s["case"]
    a, grad = s["a"].float(), s["grad"].float()
    ds = a * (grad - (a * grad).sum(-1, keepdim=True))
    # sums over whole maps that nearly cancel: in 64 bits
    hit = (_bucket_map(case, case["n"], case["cols"], s["offset"]).reshape(1, -1) == torch.arange(case["buckets"], device="cuda")[:, None])
    table = hit.double() @ ds.double().sum(0).reshape(case["heads"], -1).t()
    return (ds * s["scale"]).to(s["a"].dtype), table.float()


def _activation(x, act):
    if act == "relu":
        return x.clamp_min(0)
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / math.pi) ** 0.5 * (x + 0.044715 * x ** 3)))
    if act == "silu":
        return x * torch.sigmoid(x)
    return x


def _slope(x, act):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        th = torch.tanh(c * (x + 0.044715 * x ** 3))
        return 0.5 * (1 + th) + 0.5 * x * (1 - th * th) * c * (1 + 3 * 0.044715 * x * x)
    sg = torch.sigmoid(x)
    return sg * (1 + x * (1 - sg))


def _plain_linear_fwd(s):
    case, dt = s["case"], s["x"].dtype
    pre = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        pre = pre + s["b"].float()
    y = _activation(pre, case["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    return (y.to(dt), pre.to(dt)) if case["pre"] else (y.to(dt),)


def _plain_linear_bwd(s):
    case, dt = s["case"], s["x"].dtype
    dpre = s["dy"].float()
    if case["act"] != "none":
        dpre = dpre * _slope(s["pre"].float(), case["act"])
    out = [(dpre @ s["w"].float()).to(dt), (dpre.t() @ s["x"].float()).to(dt)]
    if case["bias"]:
        out.append(dpre.sum(0).to(dt))
    return tuple(out)


def _own_qknorm_fwd(s):
    from hyc_lora_release_b200.operators.qk_norm_kernels import qk_norm_rope_forward
    return qk_norm_rope_forward(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], EPS, position_ids=s["pos"], rotary_dim=s["rot"])


def _own_qknorm_bwd(s):
    from hyc_lora_release_b200.operators.qk_norm_kernels import qk_norm_rope_backward
    return qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], EPS, position_ids=s["pos"],
                                 rotary_dim=s["rot"])


def _own_relbias_fwd(s):
    from hyc_lora_release_b200.operators.relative_bias_kernels import softmax_forward_relative_bias
    return softmax_forward_relative_bias(s["scores"], s["scale"], s["table"], s["buckets"], attention_mask=s["mask"],
                                         causal=s["case"]["causal"], q_offset=s["offset"])


def _own_relbias_bwd(s):
    from hyc_lora_release_b200.operators.relative_bias_kernels import softmax_backward_relative_bias
    return softmax_backward_relative_bias(s["a"], s["grad"], s["scale"], s["buckets"], causal=s["case"]["causal"], q_offset=s["offset"])


def _own_linear_fwd(s):
    from hyc_lora_release_b200.operators.linear_kernels import linear_act_forward
    y, pre = linear_act_forward(s["x"], s["w"], s["b"], s["case"]["act"], residual=s["res"], save_pre=s["case"]["pre"])
    return (y, pre) if s["case"]["pre"] else (y,)


def _own_linear_bwd(s):
    from hyc_lora_release_b200.operators.linear_kernels import linear_act_backward
    bias = s["case"]["bias"]
    out = linear_act_backward(s["dy"], s["x"], s["w"], s["case"]["act"], pre=s["pre"], needs_grad=(True, True, bias))
    return out if bias else out[:2]


_plain = {("qknorm", "fwd"): _plain_qknorm_fwd, ("qknorm", "bwd"): _plain_qknorm_bwd, ("relbias", "fwd"): _plain_relbias_fwd,
          ("relbias", "bwd"): _plain_relbias_bwd, ("linear", "fwd"): _plain_linear_fwd, ("linear", "bwd"): _plain_linear_bwd}
_own = {("qknorm", "fwd"): _own_qknorm_fwd, ("qknorm", "bwd"): _own_qknorm_bwd, ("relbias", "fwd"): _own_relbias_fwd,
        ("relbias", "bwd"): _own_relbias_bwd, ("linear", "fwd"): _own_linear_fwd, ("linear", "bwd"): _own_linear_bwd}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "qknorm":
        tokens = case["batch"] * case["seq"]
        x = tokens * (case["hq"] + case["hk"]) * case["d"]
        length = min(tokens, max(4096, case["seq"])) if case["positions"] else case["seq"]
        tables = 2 * length * (case["rot"] // 2) * BYTES[case["table"]] + (8 * tokens if case["positions"] else 0)
        small = (2 if case["way"] == "fwd" else 4) * case["d"] * e
        return {"bytes": (2 if case["way"] == "fwd" else 3) * x * e + tables + small, "flops": (8 if case["way"] == "fwd" else 20) * x}
    if case["op"] == "relbias":
        b, h, n, cols = (case[x] for x in ("batch", "heads", "n", "cols"))
        places = n * cols
        if case["causal"]:      # what is behind a row's position need not be read, and is written as zeros
            places = sum(min(cols, i + cols - n + 1) for i in range(n))
        mask = {"none": 0, "padding": b * cols * e, "full": places * e}[case["mask"]]
        table = case["buckets"] * h * (e if case["way"] == "fwd" else 4)
        maps = b * h * e * ((1 if case["way"] == "fwd" else 2) * places + n * cols)
        return {"bytes": maps + mask + table, "flops": 8 * b * h * places}
    t, k, n = case["tokens"], case["k"], case["n"]
    if case["way"] == "fwd":
        elements = t * k + n * k + t * n * (1 + (case["pre"] is True) + case["residual"]) + n * case["bias"]
        return {"bytes": e * elements, "flops": 2 * t * k * n}
    elements = 2 * t * k + 2 * n * k + t * n * (2 if case["act"] != "none" else 1) + n * case["bias"]
    return {"bytes": e * elements, "flops": 4 * t * k * n}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _exact[case["op"], case["way"]](case, s)


def _turn(s, b, m):
    """Rotations [b, m, 1, rot / 2] as complex numbers."""
    z = torch.complex(s["cos"].double(), s["sin"].double())[:, :s["rot"] // 2]
    where = s["pos"] if s["pos"] is not None else torch.arange(m, device="cuda").expand(b, m)
    return z[where.reshape(-1)].view(b, m, 1, -1)


def _exact_qknorm_fwd(case, s):
    out = []
    h = s["rot"] // 2
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        v = x.double()
        v = v / ((v * v).sum(-1, keepdim=True) / case["d"] + EPS).sqrt() * w.double()
        z = torch.complex(v[..., :h], v[..., h:2 * h]) * _turn(s, case["batch"], case["seq"])
        v[..., :h], v[..., h:2 * h] = z.real, z.imag
        out.append(v)
    return tuple(out)


def _exact_qknorm_bwd(case, s):
    dx, dw = [], []
    h, d = s["rot"] // 2, case["d"]
    for x, w, dy in ((s["q"], s["qw"], s["dq"]), (s["k"], s["kw"], s["dk"])):
        g = dy.double().clone()
        z = torch.complex(g[..., :h], g[..., h:2 * h]) * _turn(s, case["batch"], case["seq"]).conj()
        g[..., :h], g[..., h:2 * h] = z.real, z.imag
        v = x.double()
        rms = ((v * v).sum(-1, keepdim=True) / d + EPS).sqrt()
        dw.append(torch.einsum("bmhd,bmhd->d", g, v / rms))
        gw = g * w.double()
        dx.append(gw / rms - v * (gw * v).sum(-1, keepdim=True) / (d * rms ** 3))
    return (*dx, *dw)


@functools.lru_cache(None)
def _bucket_of(distance, side, limit):
    """Bucket of one distance: counted from the definition bucket = exact + floor(rest * log(r / exact) / log(limit / exact)), as powers."""
    first = side // 2
    if distance < first:
        return distance
    rest, t = side - first, 0
    while t + 1 < rest and distance ** rest >= first ** (rest - t - 1) * limit ** (t + 1):
        t += 1
    return first + t


def _exact_bias_index(case, s):
    n, cols = case["n"], case["cols"]
    side = case["buckets"] // 2 if case["both"] else case["buckets"]
    lowest = -(n - 1 + s["offset"])
    row = []
    for ahead in range(lowest, cols - s["offset"]):
        if case["both"]:
            row.append(_bucket_of(min(abs(ahead), case["distance"]), side, case["distance"]) + (side if ahead > 0 else 0))
        else:
            row.append(_bucket_of(min(max(-ahead, 0), case["distance"]), side, case["distance"]))
    row = torch.tensor(row, device="cuda")
    at = torch.arange(cols, device="cuda")[None] - torch.arange(n, device="cuda")[:, None] + (n - 1)
    return row, at


def _exact_relbias_fwd(case, s):
    row, at = _exact_bias_index(case, s)
    x = s["scores"].double().mul_(s["scale"])
    x += s["table"].double()[row].t()[:, at][None]
    if s["mask"] is not None:
        x += s["mask"].double()
    if case["causal"]:
        x = torch.where(at <= case["n"] - 1 + s["offset"], x, -math.inf)
    return torch.softmax(x, -1)


def _exact_relbias_bwd(case, s):
    row, at = _exact_bias_index(case, s)
    a, g = s["a"].double(), s["grad"].double()
    ds = a * g - a * torch.einsum("bhnc,bhnc->bhn", a, g)[..., None]
    # sums along the diagonals first, then of the distances of a bucket
    n, cols, h = case["n"], case["cols"], case["heads"]
    diagonal = torch.zeros(h, n + cols - 1, dtype=torch.float64, device="cuda")
    total = ds.sum(0)
    for i in range(n):
        diagonal[:, n - 1 - i:n - 1 - i + cols] += total[:, i]
    table = torch.stack([diagonal[:, row == k].sum(1) for k in range(case["buckets"])])
    return ds * s["scale"], table


def _exact_pre(s):
    pre = s["x"].double() @ s["w"].double().t()
    return pre if s["b"] is None else pre + s["b"].double()


def _exact_act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, 0.0)
    if act == "gelu":      # x times the normal distribution's mass below x
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _exact_slope(v, act):
    if act == "none":
        return torch.ones_like(v)
    if act == "relu":
        return torch.where(v > 0, 1.0, 0.0).double()
    if act == "gelu":
        return torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":      # x sigma(u): sigma + x sigma (1 - sigma) u'
        u, du = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3), 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * v * v)
    else:
        u, du = v, 1.0
    sg = 1 / (1 + torch.exp(-u))
    return sg + v * sg * (1 - sg) * du


def _exact_linear_fwd(case, s):
    pre = _exact_pre(s)
    y = _exact_act(pre, case["act"])
    if s["res"] is not None:
        y = y + s["res"].double()
    return (y, pre) if case["pre"] else (y,)


def _exact_linear_bwd(case, s):
    g = s["dy"].double()
    if case["act"] != "none":
        g = g * _exact_slope(s["pre"].double(), case["act"])
    out = (g @ s["w"].double(), g.t() @ s["x"].double())
    return (*out, g.sum(0)) if case["bias"] else out


_exact = {("qknorm", "fwd"): _exact_qknorm_fwd, ("qknorm", "bwd"): _exact_qknorm_bwd, ("relbias", "fwd"): _exact_relbias_fwd,
          ("relbias", "bwd"): _exact_relbias_bwd, ("linear", "fwd"): _exact_linear_fwd, ("linear", "bwd"): _exact_linear_bwd}
