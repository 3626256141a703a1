"""What is measured of the operators that the models here train with: the gated
feed-forward projection of a transformer layer, group normalisation with its activation
on channels-last images, and the distillation loss against a teacher's top logits.

    listed()            the cases
    draw(rng)           another case of the same ranges
    prepare(case, seed) inputs as a training or an evaluating program has them in hand
    run(state)          one pass; outputs and, where a case trains, every gradient
    work(case)          bytes and operations that a pass cannot do without
    exact(case, seed)   the same outputs from the definitions in 64 bits

`own`: false, `run` is the plain form (elementary torch operations in 32 bits, rounded
once); true, it calls `stdml_collective_experimental_b200.ops`.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# gated    h = act(x Wg^T + bg) * (x Wu^T + bu); tokens x hidden -> tokens x ffn
# norm     y = act(group_norm(x) * w + b [+ residual]); images x channels x high x wide,
#          channels last; w and b are 32-bit parameters
# distill  per row a * CE(z, label) + (1 - a) * t^2 * KL(teacher || softmax(z / t)), the
#          teacher's distribution being that of its `top` largest logits; without labels
#          t^2 * KL alone.  `absent`: some rows have fewer teacher entries, some none.
#          `padded`: the rows of the logits lie further apart than they are long
# train    forward and backward; otherwise forward alone


def listed():
    return [
        # one token of an encoder that answers: the weights' way through the chip is all there is
        {"name": "gated_token_768x2048_bf16", "op": "gated", "tokens": 1, "hidden": 768, "ffn": 2048,
         "dtype": "bf16", "act": "gelu", "bias": True, "train": False},
        # BERT-base's hidden size, 32 sequences of 128 tokens; two thirds of the plain block's
        # width, which keeps the number of parameters near that of the ungated block
        {"name": "gated_bert_base_4096_bf16", "op": "gated", "tokens": 4096, "hidden": 768,
         "ffn": 2048, "dtype": "bf16", "act": "gelu", "bias": True, "train": True},
        # what is left of a batch without its padding, and sizes that no tile divides
        {"name": "gated_ragged_1037_f16", "op": "gated", "tokens": 1037, "hidden": 1000, "ffn": 2730,
         "dtype": "f16", "act": "silu", "bias": False, "train": True},
        # BERT-large's hidden size in the type that parameters have by default
        {"name": "gated_bert_large_512_f32", "op": "gated", "tokens": 512, "hidden": 1024,
         "ffn": 2736, "dtype": "f32", "act": "gelu", "bias": True, "train": True},
        # the largest: long batches of a wide model
        {"name": "gated_wide_16384_bf16", "op": "gated", "tokens": 16384, "hidden": 4096,
         "ffn": 11008, "dtype": "bf16", "act": "silu", "bias": False, "train": True},
        # the last block of ResNet-50 on one image that is to be classified
        {"name": "norm_last_block_x1_bf16", "op": "norm", "images": 1, "channels": 2048, "high": 7,
         "wide": 7, "groups": 32, "dtype": "bf16", "act": "relu", "residual": True, "train": False},
        # the stem of ResNet-50, a rank's batch
        {"name": "norm_stem_x64_bf16", "op": "norm", "images": 64, "channels": 64, "high": 112,
         "wide": 112, "groups": 32, "dtype": "bf16", "act": "relu", "residual": False, "train": True},
        # the end of one of its blocks, where the shortcut is added
        {"name": "norm_block_x32_f16", "op": "norm", "images": 32, "channels": 256, "high": 56,
         "wide": 56, "groups": 32, "dtype": "f16", "act": "relu", "residual": True, "train": True},
        # three channels to a group, an image of odd sides, 32 bits
        {"name": "norm_odd_x3_f32", "op": "norm", "images": 3, "channels": 90, "high": 53, "wide": 37,
         "groups": 30, "dtype": "f32", "act": "silu", "residual": False, "train": True},
        # the image classifiers' 1000 classes, a rank's batch
        {"name": "distill_classes_x256_f32", "op": "distill", "rows": 256, "classes": 1000, "top": 5,
         "dtype": "f32", "t": 4.0, "alpha": 0.5, "labels": True, "absent": False, "padded": False,
         "train": True},
        # BERT's vocabulary, the masked positions of a batch
        {"name": "distill_bert_vocab_2048_bf16", "op": "distill", "rows": 2048, "classes": 30522,
         "top": 64, "dtype": "bf16", "t": 2.0, "alpha": 0.3, "labels": True, "absent": True,
         "padded": False, "train": True},
        # the largest: every position of a batch counts, a vocabulary of many languages
        {"name": "distill_wide_4096_bf16", "op": "distill", "rows": 4096, "classes": 128256,
         "top": 100, "dtype": "bf16", "t": 1.0, "alpha": 0.0, "labels": False, "absent": False,
         "padded": False, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gated", "norm", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.7
    if op == "gated":
        most = (1 << 36) if dtype == "f32" else (1 << 39)
        while True:
            tokens, hidden, ffn = _log(rng, 1, 16384), _log(rng, 64, 4096), _log(rng, 64, 11008)
            if rng.random() < 0.6:
                hidden, ffn = -(-hidden // 64) * 64, -(-ffn // 64) * 64
            if tokens * hidden * ffn <= most:
                break
        return {"op": op, "tokens": tokens, "hidden": hidden, "ffn": ffn, "dtype": dtype,
                "act": rng.choice(["gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.5,
                "train": train}
    if op == "norm":
        while True:
            images, groups = _log(rng, 1, 64), rng.choice([1, 8, 16, 30, 32, 32])
            channels = groups * _log(rng, 1, 64)
            high, wide = _log(rng, 1, 512), _log(rng, 1, 512)
            # a group has at least 16 values
            if channels <= 2048 and 16 <= high * wide * channels // groups and \
                    images * channels * high * wide <= 64 * 64 * 112 * 112:
                break
        return {"op": op, "images": images, "channels": channels, "high": high, "wide": wide,
                "groups": groups, "dtype": dtype, "act": rng.choice(["none", "relu", "silu", "gelu"]),
                "residual": rng.random() < 0.4, "train": train}
    while True:
        rows, classes = _log(rng, 1, 4096), _log(rng, 10, 128256)
        if rows * classes <= (1 << 28):
            break
    return {"op": op, "rows": rows, "classes": classes, "top": _log(rng, 1, min(classes, 128)),
            "dtype": dtype, "t": rng.choice([0.7, 1.0, 2.0, 4.0]), "alpha": rng.choice([0.0, 0.25, 0.5, 0.9]),
            "labels": rng.random() < 0.6, "absent": rng.random() < 0.4, "padded": rng.random() < 0.3,
            "train": train}


# ------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=g) * scale

    s = {"case": dict(case)}
    if case["op"] == "gated":
        t, k, f = case["tokens"], case["hidden"], case["ffn"]
        # what a layer norm gives, weights of the usual initialisation
        s["x"] = normal(t, k).to(dt)
        s["w_gate"], s["w_up"] = (normal(f, k, scale=k ** -0.5).to(dt) for _ in range(2))
        s["b_gate"], s["b_up"] = (normal(f, scale=0.1).to(dt) for _ in range(2)) if case["bias"] else (None, None)
        leaves = ("x", "w_gate", "w_up", "b_gate", "b_up")
        s["grad"] = normal(t, f).to(dt)
    elif case["op"] == "norm":
        n, c, h, w = case["images"], case["channels"], case["high"], case["wide"]

        def image(scale, shift):
            v = normal(n, h, w, c) * scale + shift
            return v.to(dt).permute(0, 3, 1, 2)

        # a convolution's output: channels of their own scale and offset
        s["x"] = image(0.5 + torch.rand(c, device=dev, generator=g), normal(c, scale=0.5))
        s["residual"] = image(1.0, 0.0).relu() if case["residual"] else None
        s["weight"], s["bias"] = 1 + normal(c, scale=0.2), normal(c, scale=0.2)
        leaves = ("x", "residual", "weight", "bias")
        s["grad"] = image(1.0, 0.0)
    else:
        r, v, k = case["rows"], case["classes"], case["top"]
        far = v + 24 if case["padded"] else v
        s["logits"] = normal(r, far, scale=2.0).to(dt)[:, :v]
        # a teacher that agrees with the student in part
        top = torch.topk(s["logits"].float() + normal(r, v, scale=2.0), k, dim=1)
        s["top"], s["index"] = top.values.to(dt), top.indices
        if case["absent"]:
            last = torch.randint(0, k + 1, (r, 1), device=dev, generator=g)
            s["index"] = s["index"].masked_fill(torch.arange(k, device=dev) >= last, -1)
        s["labels"] = None
        if case["labels"]:
            s["labels"] = torch.randint(0, v, (r,), device=dev, generator=g)
            s["labels"] = s["labels"].masked_fill(torch.rand(r, device=dev, generator=g) < 0.1, -100)
        leaves = ("logits",)
    if case["train"]:
        for name in leaves:
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_()
    return s


# ------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"gated": _plain_gated, "norm": _plain_norm, "distill": _plain_distill}[s["case"]["op"]](s)


def _own(s):
    from stdml_collective_experimental_b200 import ops
    case = s["case"]
    if case["op"] == "gated":
        leaves = {k: s[k] for k in ("x", "w_gate", "w_up", "b_gate", "b_up") if s[k] is not None}
        out = ops.gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], activation=case["act"])
    elif case["op"] == "norm":
        leaves = {k: s[k] for k in ("x", "residual", "weight", "bias") if s[k] is not None}
        out = ops.group_norm(s["x"], case["groups"], s["weight"], s["bias"], eps=1e-5,
                             activation=None if case["act"] == "none" else case["act"],
                             residual=s["residual"])
    else:
        leaves = {"logits": s["logits"]}
        out = ops.distill_loss(s["logits"], s["top"], s["index"], s["labels"], temperature=case["t"],
                               alpha=case["alpha"])
    if not case["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, list(leaves.values()), s.get("grad"))
    return {"out": out, **dict(zip(leaves, grads))}


# ------------------------------------------------------------------------- plain forms
_SQRT_HALF, _GAUSS, _CUBE = math.sqrt(0.5), 1 / math.sqrt(2 * math.pi), 0.044715


def _act(name, z):
    """The activation and its derivative."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(z * _SQRT_HALF))
        return z * c, c + z * _GAUSS * torch.exp(-0.5 * z * z)
    if name == "gelu_tanh":
        a = 2 * _GAUSS  # sqrt(2 / pi)
        th = torch.tanh(a * (z + _CUBE * z * z * z))
        return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * a * (1 + 3 * _CUBE * z * z)
    return z, torch.ones_like(z)


def _plain_gated(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    a, da = _act(case["act"], g)
    out = {"out": (a * u).to(dt)}
    if case["train"]:
        dh = s["grad"].float()
        dg, du = dh * u * da, dh * a
        out |= {"x": (dg @ wg + du @ wu).to(dt), "w_gate": (dg.t() @ x).to(dt), "w_up": (du.t() @ x).to(dt)}
        if case["bias"]:
            out |= {"b_gate": dg.sum(0).to(dt), "b_up": du.sum(0).to(dt)}
    return out


def _plain_norm(s):
    case, dt = s["case"], s["x"].dtype
    n, c, h, w = s["x"].shape
    many = (n, h * w, case["groups"], c // case["groups"])
    # the derivative of relu jumps at zero: values next to it are placed in 64 bits
    wide = torch.float64 if case["act"] == "relu" else torch.float32

    def rows(t):  # channels last, as they lie in memory
        return t.permute(0, 2, 3, 1).to(wide).reshape(many)

    x, wt, b = rows(s["x"]), s["weight"].to(wide).reshape(many[2:]), s["bias"].to(wide).reshape(many[2:])
    x = x - x.mean((1, 3), keepdim=True)
    rstd = (x.square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()
    xh = x * rstd
    z = xh * wt + b
    if case["residual"]:
        z = z + rows(s["residual"])
    y, dact = _act(case["act"], z)

    def image(t):
        return t.to(dt).reshape(n, h, w, c).permute(0, 3, 1, 2)

    out = {"out": image(y)}
    if case["train"]:
        dz = rows(s["grad"]) * dact
        dxh = dz * wt
        dx = rstd * (dxh - dxh.mean((1, 3), keepdim=True) - xh * (dxh * xh).mean((1, 3), keepdim=True))
        out |= {"x": image(dx), "weight": (dz * xh).sum((0, 1)).reshape(c).float(),
                "bias": dz.sum((0, 1)).reshape(c).float()}
        if case["residual"]:
            out["residual"] = image(dz)
    return out


def _plain_distill(s):
    case, dt = s["case"], s["logits"].dtype
    t = case["t"]
    z = s["logits"].float()
    there = s["index"] >= 0
    at = s["index"].clamp(min=0)
    has = there.any(1)
    p = torch.where(there, s["top"].float() / t, -math.inf)
    p = p - torch.where(has, p.amax(1), 0.0)[:, None]
    p = p - torch.where(has, p.exp().sum(1), 1.0).log()[:, None]
    pe = p.exp()

    def log_softmax(v):
        v = v - v.amax(1, keepdim=True)
        return v - v.exp().sum(1, keepdim=True).log()

    q = log_softmax(z / t)
    kl = (pe * torch.where(there, p - q.gather(1, at), 0.0)).sum(1)
    if case["labels"]:
        counts = s["labels"] >= 0
        label = s["labels"].clamp(min=0)[:, None]
        q1 = log_softmax(z)
        a, b = case["alpha"], 1 - case["alpha"]
        loss = b * t * t * kl - a * q1.gather(1, label)[:, 0]
    else:
        counts, a, b = has, 0.0, 1.0
        loss = t * t * kl
    each = torch.where(counts, 1.0, 0.0) / counts.sum().clamp(min=1)
    out = {"out": (loss * each).sum()}
    if case["train"]:
        d = q.exp_().mul_(has[:, None].float()).scatter_add_(1, at, -pe).mul_(b * t)
        if case["labels"]:
            d += a * q1.exp_().scatter_add_(1, label, -torch.ones_like(label, dtype=q1.dtype))
        out["logits"] = d.mul_(each[:, None]).to(dt)
    return out


# ------------------------------------------------------------------------- costs
def work(case):
    b = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "gated":
        t, k, f = case["tokens"], case["hidden"], case["ffn"]
        bias = 2 * f if case["bias"] else 0
        read, flops = t * k + 2 * f * k + bias, 4 * t * k * f
        if not case["train"]:
            return {"bytes": b * (read + t * f), "flops": flops}
        return {"bytes": b * (2 * read + 2 * t * f), "flops": 3 * flops}
    if case["op"] == "norm":
        n = case["images"] * case["channels"] * case["high"] * case["wide"]
        images = 3 if case["residual"] else 2  # x, y
        if case["train"]:
            images += 3 if case["residual"] else 2  # dy, dx
        return {"bytes": b * images * n + 16 * case["channels"], "flops": n * (30 if case["train"] else 10)}
    n, k = case["rows"] * case["classes"], case["rows"] * case["top"]
    return {"bytes": b * n * (2 if case["train"] else 1) + (b + 8) * k + (8 * case["rows"] if case["labels"] else 0),
            "flops": n * (10 if case["train"] else 5)}


# ------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions in 64 bits; the gradients by differentiating them."""
    s = prepare(case, seed)
    names = [k for k in ("x", "w_gate", "w_up", "b_gate", "b_up", "residual", "weight", "bias", "logits")
             if s.get(k) is not None]
    leaf = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names}
    nn = torch.nn.functional
    act = {"gelu": nn.gelu, "gelu_tanh": lambda v: nn.gelu(v, approximate="tanh"), "silu": nn.silu,
           "relu": nn.relu, "none": lambda v: v}
    up = s["grad"].double() if case["op"] != "distill" else None
    if case["op"] == "gated":
        gate, lin = (nn.linear(leaf["x"], leaf["w_" + k], leaf.get("b_" + k)) for k in ("gate", "up"))
        out = act[case["act"]](gate) * lin
    elif case["op"] == "norm":
        v = leaf["x"].reshape(case["images"], case["groups"], -1)
        var, mean = torch.var_mean(v, dim=2, unbiased=False, keepdim=True)
        z = ((v - mean) / torch.sqrt(var + 1e-5)).reshape(leaf["x"].shape)
        z = z * leaf["weight"].view(1, -1, 1, 1) + leaf["bias"].view(1, -1, 1, 1)
        out = act[case["act"]](z + leaf["residual"] if case["residual"] else z)
    else:
        z, t = leaf["logits"], case["t"]
        top = s["top"].double().div(t).masked_fill(s["index"] < 0, -math.inf)
        some = ~torch.isneginf(top).all(1)
        pt = torch.zeros(len(z), case["classes"], dtype=torch.float64, device=z.device)
        pt[some] = pt[some].scatter_add(1, s["index"][some].clamp(min=0), torch.softmax(top[some], 1))
        rows = nn.kl_div(torch.log_softmax(z / t, 1), pt, reduction="none").sum(1) * t * t
        if case["labels"]:
            hard = nn.cross_entropy(z, s["labels"], ignore_index=-100, reduction="none")
            rows = case["alpha"] * hard + (1 - case["alpha"]) * rows
            live = s["labels"] != -100
        else:
            live = some
        out = rows[live].sum() / max(1, int(live.sum()))
    got = {"out": out.detach()}
    if case["train"]:
        got |= dict(zip(names, torch.autograd.grad(out, [leaf[k] for k in names], up)))
    return got
