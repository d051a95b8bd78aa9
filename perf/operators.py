"""Operators of 8-bit integer layers: rows quantised where they are made, their products with quantised weights, and layers trained with them.

A row ``y`` is held as whole numbers ``q`` of 8 bits and one scale: ``scale = max |y| / 127``, ``q = round(127 y / max |y|)`` with ties to the even
number; a weight matrix ``[out, in]`` has one scale per row, that is per output channel.  Half of a row's largest value lies on a tie, and bf16 rows often
hold it: all forms here multiply before they divide, which is exact there.

* ``norm``: ``h = x + residual`` (rounded to the rows' type) and the root-mean-square norm of ``h`` with a weight, quantised.
* ``glu``: ``act(gate) up`` of the two halves of a joint product's rows, quantised.
* ``product``: ``scale_x scale_w (q_x q_w^T) + bias + residual`` of quantised rows and weights.
* ``train``: a layer's forward and backward pass.  ``x`` and the weights are quantised, the product is made of them, and the gradients are those of
  the product at the values that the whole numbers stand for, ``dx = dy w'`` and ``dw = dy^T x'`` (the rounding counts as having slope one), so that
  of the activations the 8-bit rows are all that is kept.  Several projections of the same rows share them.
* ``mlp``: the second half of a decoder layer as a server runs it: the norm with its residual, the joint product of gate and up, their gated
  activation, the down product with the residual added.

Quantised rows come back as the values that they stand for, in bf16.  Widths are those of this repository's configs (``config/*.yaml``) and of its
serving benchmark (``levanter_b200/inference/bench_decode.py``)."""
import math

import torch

own = False

TINY = 2.0 ** -100  # rows whose largest magnitude is below this are stored as zeros
EPS = 1e-5


def listed():
    return [
        # one user's token at the width of the serving benchmark's 8B model: the latency of a call
        dict(name="norm_1", kind="norm", rows=1, cols=4096, dtype="bfloat16", residual=True),
        # a full prefill step of the engine
        dict(name="norm_16384", kind="norm", rows=16384, cols=4096, dtype="bfloat16", residual=True),
        # a decode round of 64 users, the 8B model's feed-forward width
        dict(name="glu_64", kind="glu", rows=64, cols=14336, act="silu"),
        # a training micro-batch of the 7B model, evaluated
        dict(name="glu_8192", kind="glu", rows=8192, cols=11008, act="silu"),
        # one user: gate and up of the 8B model side by side
        dict(name="product_1", kind="product", rows=1, cols=4096, outs=28672, dtype="bfloat16", bias=False, residual=False),
        # 64 users: q, k and v of the 8B model side by side
        dict(name="product_64", kind="product", rows=64, cols=4096, outs=6144, dtype="bfloat16", bias=False, residual=False),
        # a short ragged batch of GPT-2 small, its joint projection with a bias; a result in 32 bits, as a caller that goes on in it asks for
        dict(name="product_333", kind="product", rows=333, cols=768, outs=2304, dtype="float32", bias=True, residual=False),
        # prompts through the 8B model's down projection, the residual added on the way
        dict(name="product_8192", kind="product", rows=8192, cols=14336, outs=4096, dtype="bfloat16", bias=False, residual=True),
        # fine-tuning on a small ragged batch, GPT-2 small
        dict(name="train_999", kind="train", rows=999, cols=768, outs=2304, parts=1, bias=True),
        # the training benchmark's micro-batch: gate and up of the 7B model
        dict(name="train_8192", kind="train", rows=8192, cols=4096, outs=11008, parts=2, bias=False),
        # a decode round of 8 users through the 8B model's feed-forward half
        dict(name="mlp_8", kind="mlp", rows=8, cols=4096, outs=14336, act="silu"),
        # one prompt through that of the 1B model
        dict(name="mlp_2000", kind="mlp", rows=2000, cols=2048, outs=8192, act="silu"),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, odd=0.5):
    n = _log_uniform(rng, lo, hi)
    return n if rng.random() < odd else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["norm", "glu", "product", "product", "train", "mlp"])
    act = rng.choice(["silu", "silu", "gelu_new"])
    if kind == "norm":
        cols = _size(rng, 512, 8192)
        return dict(kind=kind, rows=_log_uniform(rng, 1, (16384 * 4096) // cols // 2), cols=cols, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]),
                    residual=rng.random() < 0.6)
    if kind == "glu":
        cols = _size(rng, 512, 14336)
        return dict(kind=kind, rows=_log_uniform(rng, 1, (8192 * 11008) // cols), cols=cols, act=act)
    if kind == "product":
        cols = _size(rng, 128, 14336)
        outs = _size(rng, 128, min(28672, (4096 * 28672) // cols))
        return dict(kind=kind, rows=_log_uniform(rng, 1, min(16384, (8192 * 14336 * 4096) // (cols * outs))), cols=cols, outs=outs,
                    dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), bias=rng.random() < 0.3, residual=rng.random() < 0.3)
    if kind == "train":
        cols, outs = (_log_uniform(rng, 128, 4096) // 8 * 8 for _ in range(2))
        return dict(kind=kind, rows=_log_uniform(rng, 16, 8192), cols=cols, outs=outs, parts=rng.randint(1, 3), bias=rng.random() < 0.3)
    cols = _size(rng, 512, 4096, odd=0.3)
    return dict(kind=kind, rows=_log_uniform(rng, 1, 4096), cols=cols, outs=_size(rng, 512, 14336, odd=0.3), act=act)


# ---------------------------------------------------------------------------------------------------------------- inputs from a seed
class _Maker:
    """Tensors from one seed: activations with a few channels that stand out, as a transformer's have, and weights as an initialised model's."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed % (1 << 62))

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32) * std).to(dtype)

    def rows(self, rows, cols, dtype=torch.bfloat16):
        loud = 1.0 + 7.0 * (torch.rand(cols, generator=self.g, device="cuda") < 0.01).float()
        return (torch.randn(rows, cols, generator=self.g, device="cuda") * loud).to(dtype)

    def norm_weight(self, cols):
        return self.normal(cols, std=0.1, dtype=torch.float32).add_(1.0).bfloat16()

    def int8(self, x):
        """Whole numbers and scales as a program keeps them: rows start at multiples of 16 bytes."""
        q, s = _quantize(x.float())
        held = torch.zeros(x.shape[0], -(-x.shape[1] // 16) * 16, dtype=torch.int8, device="cuda")[:, :x.shape[1]]
        return held.copy_(q), s.squeeze(-1)


def prepare(case, seed):
    m, kind, T, C = _Maker(seed * 31 + 7), case["kind"], case["rows"], case["cols"]
    st = dict(case)
    if kind == "norm":
        dt = getattr(torch, case["dtype"])
        st.update(x=m.rows(T, C, dt), r=m.normal(T, C, std=0.5, dtype=dt) if case["residual"] else None, w=m.norm_weight(C))
    elif kind == "glu":
        st.update(y=m.rows(T, 2 * C))
    elif kind == "product":
        (q, s), (wq, ws) = m.int8(m.rows(T, C)), m.int8(m.normal(case["outs"], C, std=0.02))
        st.update(q=q, s=s, wq=wq, ws=ws, b=m.normal(case["outs"], std=0.1) if case["bias"] else None,
                  r=m.normal(T, case["outs"]) if case["residual"] else None)
    elif kind == "train":
        n, F = case["parts"], case["outs"]
        st.update(x=m.rows(T, C), w=m.normal(n, F, C, std=0.02), b=m.normal(n, F, std=0.1) if case["bias"] else None, dy=m.normal(n, T, F, std=0.01))
    else:
        F = case["outs"]
        (gu, gus), (d, ds) = m.int8(m.normal(2 * F, C, std=0.02)), m.int8(m.normal(C, F, std=0.02))
        st.update(x=m.rows(T, C), r=m.normal(T, C, std=0.5), w=m.norm_weight(C), gu=gu, gus=gus, d=d, ds=ds)
    return st


# ---------------------------------------------------------------------------------------------------------------- the plain form, in 32 bits
def _quantize(y, factor=1.0):
    """Whole numbers (in 32-bit floats) and the scale of every row of ``factor y``, with a positive factor per row."""
    top = y.abs().amax(-1, keepdim=True)
    live = top * factor >= TINY
    return torch.where(live, torch.round(y * 127.0 / top), 0.0), torch.where(live, top * factor / 127.0, 0.0)


def _norm(x, r, w):
    """``h``, and the whole numbers and scales of its norm, whose factor of the row leaves the whole numbers as they are."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = h.float()
    return h, *_quantize(f * w.float(), torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS))


def _act(g, name):
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _product(q, s, wq, ws):
    return (q @ wq.float().t()) * s * ws


def _plain(st):
    kind = st["kind"]
    if kind == "norm":
        h, q, s = _norm(st["x"], st["r"], st["w"])
        return {"rows": (q * s).bfloat16(), "scale": s.squeeze(-1), "h": h if st["residual"] else None}
    if kind == "glu":
        g, u = st["y"].float().chunk(2, dim=-1)
        q, s = _quantize(_act(g, st["act"]) * u)
        return {"rows": (q * s).bfloat16(), "scale": s.squeeze(-1)}
    if kind == "product":
        y = _product(st["q"].float(), st["s"][:, None], st["wq"], st["ws"])
        if st["b"] is not None:
            y = y + st["b"].float()
        if st["r"] is not None:
            y = y + st["r"].float()
        return {"y": y.to(getattr(torch, st["dtype"]))}
    if kind == "train":
        w = st["w"].float().flatten(0, 1)
        q, s = _quantize(st["x"].float())
        wq, ws = _quantize(w)
        y = (q @ wq.t()) * s * ws.squeeze(-1)
        if st["b"] is not None:
            y = y + st["b"].float().flatten()
        dy = st["dy"].float().transpose(0, 1).flatten(1)  # [rows, parts * outs]
        dx, dw = dy @ (wq * ws), dy.t() @ (q * s)
        return {"y": y.bfloat16().unflatten(1, (st["parts"], -1)).unbind(1), "dx": dx.bfloat16(), "dw": dw.bfloat16().unflatten(0, (st["parts"], -1)).unbind(0),
                "db": None if st["b"] is None else dy.sum(0).bfloat16().unflatten(0, (st["parts"], -1)).unbind(0)}
    h, *rows = _norm(st["x"], st["r"], st["w"])
    g, u = _product(*rows, st["gu"], st["gus"]).bfloat16().float().chunk(2, dim=-1)
    out = _product(*_quantize(_act(g, st["act"]) * u), st["d"], st["ds"]) + h.float()
    return {"h": h, "y": out.bfloat16()}


# ---------------------------------------------------------------------------------------------------------------- the framework's operators
def _own(st):
    from levanter_b200.ops import int8 as I
    from levanter_b200.utils.activation import ActivationFunctionEnum as Act

    kind = st["kind"]
    if kind == "norm":
        rows, h = I.rms_norm_int8(st["x"], st["w"], EPS, residual=st["r"])
        return {"rows": rows.dequantize(), "scale": rows.scale, "h": h}
    if kind == "glu":
        C = st["cols"]
        rows = I.gated_activation_int8(st["y"][:, :C], st["y"][:, C:], Act(st["act"]))
        return {"rows": rows.dequantize(), "scale": rows.scale}
    if kind == "product":
        y = I.int8_product(I.Int8Rows(st["q"], st["s"]), I.Int8Rows(st["wq"], st["ws"]), bias=st["b"], residual=st["r"], out_dtype=getattr(torch, st["dtype"]))
        return {"y": y}
    if kind == "train":
        x = st["x"].detach().requires_grad_()
        ws = [w.detach().requires_grad_() for w in st["w"].unbind(0)]
        bs = None if st["b"] is None else [b.detach().requires_grad_() for b in st["b"].unbind(0)]
        ys = I.int8_linear_many(x, ws, bs)
        g = torch.autograd.grad(ys, [x, *ws, *(bs or [])], list(st["dy"].unbind(0)))
        n = st["parts"]
        return {"y": [y.detach() for y in ys], "dx": g[0], "dw": g[1:1 + n], "db": g[1 + n:] if bs else None}
    F = st["outs"]
    rows, h = I.rms_norm_int8(st["x"], st["w"], EPS, residual=st["r"])
    y = I.int8_product(rows, I.Int8Rows(st["gu"], st["gus"]))
    mid = I.gated_activation_int8(y[:, :F], y[:, F:], Act(st["act"]))
    return {"h": h, "y": I.int8_product(mid, I.Int8Rows(st["d"], st["ds"]), residual=h)}


def run(st):
    if own:
        return _own(st)
    return _plain(st)


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, T, C = case["kind"], case["rows"], case["cols"]
    if kind == "norm":
        e = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": T * C * (e * (3 if case["residual"] else 1) + 2) + 4 * T + 2 * C, "flops": 6 * T * C}
    if kind == "glu":
        return {"bytes": T * C * 6 + 4 * T, "flops": 10 * T * C}
    N = case["outs"]
    if kind == "product":
        e = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": T * C + N * C + 4 * (T + N) + T * N * (e + (2 if case["residual"] else 0)) + (2 * N if case["bias"] else 0), "flops": 2 * T * N * C}
    if kind == "train":
        n = case["parts"]
        return {"bytes": 4 * T * C + 4 * n * N * C + 4 * n * T * N + (4 * n * N if case["bias"] else 0), "flops": 6 * n * T * N * C}
    return {"bytes": 8 * T * C + 2 * C + 3 * N * C + 4 * (2 * N + C), "flops": 6 * T * N * C}


# ---------------------------------------------------------------------------------------------------------------- the definition, in 64 bits
def _held(y, factor=None):
    """The values that 8-bit rows of ``y`` (times a factor per row) stand for, and their scales."""
    most = y.abs().max(dim=-1).values
    steps = (127 * y / most[:, None]).round()
    most = most if factor is None else most * factor
    gone = most < TINY
    scale = (most / 127).masked_fill(gone, 0)
    return steps.masked_fill(gone[:, None], 0) * scale[:, None], scale


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]

    def gate(y):
        g, u = y[:, :y.shape[1] // 2], y[:, y.shape[1] // 2:]
        if case["act"] == "silu":
            return g * torch.sigmoid(g) * u
        return g * 0.5 * (1 + torch.tanh((g + 0.044715 * g ** 3) * (2 / math.pi) ** 0.5)) * u

    def normed(x, r, w):
        h = x if r is None else (x.double() + r.double()).to(x.dtype)
        d = h.double()
        return h, *_held(d * w.double(), (d.pow(2).mean(dim=-1) + EPS) ** -0.5)

    if kind == "norm":
        h, held, scale = normed(st["x"], st["r"], st["w"])
        return {"rows": held, "scale": scale, "h": h.double() if case["residual"] else None}
    if kind == "glu":
        held, scale = _held(gate(st["y"].double()))
        return {"rows": held, "scale": scale}
    if kind == "product":
        y = torch.mm(st["q"].double() * st["s"].double()[:, None], (st["wq"].double() * st["ws"].double()[:, None]).t())
        for term in (st["b"], st["r"]):
            if term is not None:
                y += term.double()
        return {"y": y}
    if kind == "train":
        x = _held(st["x"].double())[0]
        ws = [_held(w.double())[0] for w in st["w"]]
        dys = [g.double() for g in st["dy"]]
        ys = [torch.mm(x, w.t()) for w in ws]
        if st["b"] is not None:
            ys = [y + b.double() for y, b in zip(ys, st["b"])]
        dx = sum(torch.mm(g, w) for g, w in zip(dys, ws))
        return {"y": ys, "dx": dx, "dw": [torch.mm(g.t(), x) for g in dys], "db": None if st["b"] is None else [g.sum(dim=0) for g in dys]}
    h, held, _ = normed(st["x"], st["r"], st["w"])
    joint = torch.mm(held, (st["gu"].double() * st["gus"].double()[:, None]).t()).bfloat16().double()
    out = torch.mm(_held(gate(joint))[0], (st["d"].double() * st["ds"].double()[:, None]).t()) + h.double()
    return {"h": h.double(), "y": out}
