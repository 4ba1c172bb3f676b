"""A decoder's layer in 8-bit integers, as cases to be measured: products of rows and weights of 8 bits with a scale for each token and each
channel, the gated feed-forward block of such products, and the norms behind and before a block with its gate and its factor on the residual.
`own` says whether a case runs through this framework or in its plain form."""
import math

import torch

own = False

HIDDEN, FFN, EPS = 4096, 14336, 1e-5


# ---- cases ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one generating request at the fused q/k/v projection: the smallest product, all latency
        dict(name="mm_one", op="mm", rows=1, k=HIDDEN, n=6144, bias=False, f32=False),
        # a decode batch at the output projection: weights decide
        dict(name="mm_decode", op="mm", rows=64, k=HIDDEN, n=HIDDEN, bias=False, f32=False),
        # a classifier's logits of a mixed step, in f32 with a bias, nothing a multiple of anything
        dict(name="mm_odd", op="mm", rows=301, k=1111, n=5003, bias=True, f32=True),
        # prompts at the fused q/k/v projection
        dict(name="mm_prompt", op="mm", rows=8192, k=HIDDEN, n=6144, bias=True, f32=False),
        # one generated token through the feed-forward block
        dict(name="ffn_one", op="ffn", rows=1, k=HIDDEN, f=FFN, act="silu"),
        # a decode batch through it
        dict(name="ffn_decode", op="ffn", rows=96, k=HIDDEN, f=FFN, act="silu"),
        # a step's pieces of prompts through a block of odd widths
        dict(name="ffn_ragged", op="ffn", rows=777, k=2222, f=5777, act="gelu"),
        # prompts through it: the largest call
        dict(name="ffn_prompt", op="ffn", rows=8192, k=HIDDEN, f=FFN, act="gelu_tanh"),
        # norms around a block's end for one token
        dict(name="norm_one", op="norm", rows=1, n=HIDDEN, post=True, gate="none", h_f32=False, y_f32=False),
        # a mixed step: the residual in f32, a gate for each channel, an odd width
        dict(name="norm_mixed", op="norm", rows=333, n=5003, post=True, gate="channel", h_f32=True, y_f32=False),
        # prompts, with a gate that the model computes for each token
        dict(name="norm_prompt", op="norm", rows=8192, n=HIDDEN, post=True, gate="row", h_f32=False, y_f32=False),
        # the second half of a layer for a decode batch: norms into 8 bits, the block, norms in front of the next one
        dict(name="layer_decode", op="layer", rows=128, k=HIDDEN, f=FFN, act="silu"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["mm", "mm", "ffn", "ffn", "norm", "norm", "layer"])
    most = {o: max(work(c)["flops"] for c in listed() if c["op"] == o) for o in ("mm", "ffn", "norm", "layer")}
    most["layer"] = most["ffn"]
    while True:
        rows = _log(rng, 1, 8192)
        if op == "mm":
            k, n = rng.choice([(HIDDEN, HIDDEN), (HIDDEN, 6144), (FFN, HIDDEN), (_log(rng, 64, 16384), _log(rng, 64, 32768)), (16 * _log(rng, 4, 1024), 8 * _log(rng, 8, 4096))])
            case = dict(op=op, rows=rows, k=k, n=n, bias=rng.random() < 0.4, f32=rng.random() < 0.2)
        elif op == "norm":
            case = dict(op=op, rows=rows, n=rng.choice([HIDDEN, 8 * _log(rng, 8, 2048), _log(rng, 64, 16384)]), post=rng.random() < 0.7,
                        gate=rng.choice(["none", "channel", "row", "sigmoid"]), h_f32=rng.random() < 0.4, y_f32=rng.random() < 0.2)
        else:
            k, f = rng.choice([(HIDDEN, FFN), (2048, 8192), (_log(rng, 64, 8192), _log(rng, 128, 16384)), (64 * rng.randint(4, 96), 64 * rng.randint(8, 224))])
            case = dict(op=op, rows=rows, k=k, f=f, act=rng.choice(["silu", "silu", "gelu", "gelu_tanh"]))
        w = work(case)
        if w["flops"] <= most[op] and w["bytes"] <= 2e9:
            return case


def work(case):
    rows = case["rows"]
    if case["op"] == "mm":
        k, n = case["k"], case["n"]
        return {"bytes": 2 * rows * k + n * k + 4 * n * (2 if case["bias"] else 1) + rows * n * (4 if case["f32"] else 2), "flops": 2 * rows * n * k}
    if case["op"] == "norm":
        n = case["n"]
        gate = {"none": 0, "channel": n, "row": rows * n, "sigmoid": rows * n}[case["gate"]]
        return {"bytes": rows * n * ((8 if case["h_f32"] else 4) + (4 if case["y_f32"] else 2) + 2) + 2 * gate + 2 * n * (2 if case["post"] else 1), "flops": 14 * rows * n}
    k, f = case["k"], case["f"]
    block = {"bytes": 3 * f * k + 4 * (2 * f + k) + 4 * rows * k, "flops": 6 * rows * f * k}
    if case["op"] == "layer":  # y and h come, h and the next block's input go
        block = {"bytes": block["bytes"] + 4 * rows * k, "flops": block["flops"] + 28 * rows * k}
    return block


# ---- what a case holds ----------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    bf16 = lambda t: t.to(torch.bfloat16)  # noqa: E731

    def weight(n, k):
        """[n, k] in 8 bits, a scale for each of n."""
        w = normal(n, k) * k ** -0.5
        scale = w.abs().amax(1) / 127
        return torch.round(w / scale[:, None]).to(torch.int8), scale

    def activations(rows, k):
        """Some channels are much larger than the others."""
        return bf16(normal(rows, k) * torch.where(torch.rand(k, generator=g, device="cuda") < 0.004, 12.0, 1.0))

    rows = case["rows"]
    if case["op"] == "mm":
        w, scale = weight(case["n"], case["k"])
        return dict(x=activations(rows, case["k"]), w=w, w_scale=scale, bias=normal(case["n"]) if case["bias"] else None)
    norm_of = lambda n: bf16(1 + 0.2 * normal(n))  # noqa: E731
    if case["op"] == "norm":
        n, f32 = case["n"], lambda t, wide: t if wide else bf16(t)
        gate = {"none": lambda: None, "channel": lambda: bf16(0.5 + 0.3 * normal(n)), "row": lambda: bf16(0.5 + normal(rows, n)), "sigmoid": lambda: bf16(2 * normal(rows, n))}
        return dict(h=f32(3 * normal(rows, n), case["h_f32"]), y=f32(normal(rows, n), case["y_f32"]), gate=gate[case["gate"]](),
                    post_weight=norm_of(n) if case["post"] else None, norm_weight=norm_of(n), scale=0.22)
    k, f = case["k"], case["f"]
    state = dict(zip(("gate", "gate_scale", "up", "up_scale", "down", "down_scale"), (*weight(f, k), *weight(f, k), *weight(k, f))))
    if case["op"] == "ffn":
        return dict(state, x=activations(rows, k))
    return dict(state, h=bf16(3 * normal(rows, k)), y=bf16(normal(rows, k)), post_weight=norm_of(k), norm_weight=norm_of(k), end_weight=norm_of(k), next_weight=norm_of(k), scale=0.22)


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        from dmlx_b200 import device
        if case["op"] == "mm":
            state["weight"] = device.I8Weight(state["w"], state["w_scale"])
            state["rows"] = device.I8Rows(case["rows"], case["k"])
        elif case["op"] in ("ffn", "layer"):
            state["gate_up"] = device.I8Weight.gated(state["gate"], state["gate_scale"], state["up"], state["up_scale"])
            state["down_weight"] = device.I8Weight(state["down"], state["down_scale"])
            state["rows"] = device.I8Rows(case["rows"], case["k"], case["f"])
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        from dmlx_b200 import device
        if case["op"] == "mm":
            return device.i8_mm(s["weight"], s["rows"], s["x"], bias=s["bias"], f32=case["f32"])
        if case["op"] == "ffn":
            return device.i8_ffn(s["gate_up"], s["down_weight"], s["rows"], s["x"], activation=case["act"])
        if case["op"] == "norm":
            return device.residual_norm(s["h"], s["y"], s["norm_weight"], post_weight=s["post_weight"], gate=s["gate"], gate_sigmoid=case["gate"] == "sigmoid",
                                        scale=s["scale"], eps=EPS)
        h, _ = device.residual_norm(s["h"], s["y"], s["norm_weight"], post_weight=s["post_weight"], scale=s["scale"], eps=EPS, rows=s["rows"], h_dtype=torch.float32)
        y = device.i8_ffn(s["gate_up"], s["down_weight"], s["rows"], activation=case["act"], f32=True)
        return device.residual_norm(h, y, s["next_weight"], post_weight=s["end_weight"], scale=s["scale"], eps=EPS, h_dtype=torch.bfloat16)
    if case["op"] == "mm":
        y = _product(s["x"].float(), s["w"], s["w_scale"])
        if s["bias"] is not None:
            y = y + s["bias"]
        return y if case["f32"] else y.to(torch.bfloat16)
    if case["op"] == "ffn":
        return _feed_forward(s, s["x"].float()).to(torch.bfloat16)
    if case["op"] == "norm":
        h, x = _norms(s["h"], s["y"].float(), s["gate"], case["gate"] == "sigmoid", s["post_weight"], s["norm_weight"], s["scale"])
        return h.to(s["h"].dtype), x.to(torch.bfloat16)
    h, x = _norms(s["h"], s["y"].float(), None, False, s["post_weight"], s["norm_weight"], s["scale"])
    h, x = _norms(h, _feed_forward(s, x), None, False, s["end_weight"], s["next_weight"], s["scale"])
    return h.to(torch.bfloat16), x.to(torch.bfloat16)


def _product(x, w, w_scale):
    """The rows in 8 bits, a row's largest at 127, times w."""
    most = x.abs().amax(1, keepdim=True)
    q = torch.round(x * 127 / most)
    return q @ w.float().T * w_scale * (most / 127)


def _feed_forward(s, x):
    gate, up = _product(x, s["gate"], s["gate_scale"]), _product(x, s["up"], s["up_scale"])
    act = s["case"]["act"]
    if act == "silu":
        gate = gate / (1 + torch.exp(-gate))
    elif act == "gelu":
        gate = 0.5 * gate * (1 + torch.erf(gate * 0.5 ** 0.5))
    else:
        gate = 0.5 * gate * (1 + torch.tanh((2 / math.pi) ** 0.5 * (gate + 0.044715 * gate ** 3)))
    return _product(gate * up, s["down"], s["down_scale"])


def _norm(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _norms(h, y, gate, sigmoid, post_weight, norm_weight, scale):
    if post_weight is not None:
        y = _norm(y, post_weight)
    if gate is not None:
        y = y * (1 / (1 + torch.exp(-gate.float())) if sigmoid else gate.float())
    h = h.float() + scale * y
    return h, _norm(h, norm_weight)


# ---- the definitions, in 64 bits ------------------------------------------------------------------------------------------------
def _exact_product(x, w, scale):
    largest = torch.linalg.vector_norm(x, float("inf"), dim=-1)[:, None]
    steps = (127.0 * x).div(largest).round()
    return torch.einsum("tk,nk->tn", steps, w.double()) * largest.div(127.0) * scale.double()[None]


def _exact_block(s, x):
    a, b = _exact_product(x, s["gate"], s["gate_scale"]), _exact_product(x, s["up"], s["up_scale"])
    act = s["case"]["act"]
    if act == "silu":
        a = a * torch.sigmoid(a)
    else:
        a = torch.nn.functional.gelu(a, approximate="tanh" if act == "gelu_tanh" else "none")
    return _exact_product(a * b, s["down"], s["down_scale"])


def _exact_norm(x, weight):
    return weight.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)


def exact(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["op"] == "mm":
        y = _exact_product(s["x"].double(), s["w"], s["w_scale"])
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "ffn":
        return _exact_block(s, s["x"].double())
    y = s["y"].double()
    if s["post_weight"] is not None:
        y = _exact_norm(y, s["post_weight"])
    if case["op"] == "norm" and s["gate"] is not None:
        y = y * (torch.sigmoid(s["gate"].double()) if case["gate"] == "sigmoid" else s["gate"].double())
    h = s["h"].double() + s["scale"] * y
    x = _exact_norm(h, s["norm_weight"])
    if case["op"] == "norm":
        return h, x
    h = h + s["scale"] * _exact_norm(_exact_block(s, x), s["end_weight"])
    return h, _exact_norm(h, s["next_weight"])
