"""What the training operators cost: cases, plain forms, and the calls a user makes of ``videoitg_amd.ops``.

Four operators of one fine-tuning step of the frame selector (sizes: the Qwen2-7B widths of ``ITGConfig``, the 512-frame prompt of 512 x 25 visual
tokens + 60 text tokens, one rank of an eight-way split of it):

* ``embed`` / ``embed_grad``   token embedding lookup with a scale, and its gradient;
* ``ffn`` / ``ffn_grad``       the gated feed-forward's [gate | up] projection + SiLU * up (weight rows interleaved [32 gate | 32 up]), and its backward;
* ``clip``                     the global gradient norm over a list of tensors, and the clipped gradients;
* ``head``                     per-frame mean + linear score, the grounding loss, and their gradients.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCAB, HIDDEN, FFN = 152064, 3584, 18944


def listed():
    return [
        # the text of one prompt around <image>: a handful of rows, all latency
        {"name": "embed_prompt", "op": "embed", "n": 60, "d": HIDDEN, "vocab": VOCAB, "table": "fp16", "out": "fp32", "scale": 1.0, "pad": 0.0},
        # a full text batch at the tokenizer's maximum length
        {"name": "embed_batch", "op": "embed", "n": 20480, "d": HIDDEN, "vocab": VOCAB, "table": "bf16", "out": "bf16", "scale": 59.866518188383064, "pad": 0.1},
        # its gradient as a dense tensor of the table's type: every row of the vocabulary is written
        {"name": "embed_grad_dense", "op": "embed_grad", "n": 20480, "d": HIDDEN, "vocab": VOCAB, "dout": "bf16", "table": "bf16", "scale": 1.0, "pad": 0.1, "accumulate": False},
        # added to a running fp32 gradient: only the rows of the batch are touched, a third of the tokens are one and the same
        {"name": "embed_grad_add", "op": "embed_grad", "n": 5003, "d": HIDDEN, "vocab": VOCAB, "dout": "fp32", "table": "fp32", "scale": 0.5, "pad": 0.33, "accumulate": True},
        # one token through one feed-forward: the weight's bytes
        {"name": "ffn_token", "op": "ffn", "m": 1, "d": HIDDEN, "f": FFN, "dtype": "bf16", "save": False},
        # the whole 512-frame prompt, pre-activations kept for the backward pass
        {"name": "ffn_video", "op": "ffn", "m": 12860, "d": HIDDEN, "f": FFN, "dtype": "bf16", "save": True},
        {"name": "ffn_grad_video", "op": "ffn_grad", "m": 12860, "d": HIDDEN, "f": FFN, "dtype": "bf16"},
        # one rank of eight, a ragged share, in the reference's own dtype
        {"name": "ffn_grad_rank", "op": "ffn_grad", "m": 1607, "d": HIDDEN, "f": FFN, "dtype": "fp16"},
        # head + projector only: a few tensors, latency
        {"name": "clip_head", "op": "clip", "kind": "projector", "d": HIDDEN, "f": 1152, "layers": 1, "dtype": "fp32", "max_norm": 1.0, "sigma": 0.01},
        # four decoder layers: matrices in 16 bit, norms and biases in fp32
        {"name": "clip_layers", "op": "clip", "kind": "decoder", "d": HIDDEN, "f": FFN, "layers": 4, "dtype": "bf16", "max_norm": 1.0, "sigma": 0.001},
        # the reference workload's head: 512 frames x 25 tokens
        {"name": "head_512", "op": "head", "frames": 512, "tokens": 25, "d": HIDDEN, "h": "fp32", "dh": "fp32", "positive": 0.06},
        # a short clip keeps a 16 x 16 grid per frame
        {"name": "head_clip", "op": "head", "frames": 61, "tokens": 256, "d": HIDDEN, "h": "bf16", "dh": "bf16", "positive": 0.3},
    ]


def _span(rng, lo, hi):
    """a whole number of [lo, hi], spread evenly over its logarithm"""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "ffn", "ffn", "ffn_grad", "ffn_grad", "clip", "head"])
    if op == "embed":
        return {"op": op, "n": _span(rng, 1, 20480), "d": 4 * _span(rng, 32, 1024), "vocab": _span(rng, 300, VOCAB), "table": rng.choice(["bf16", "fp16", "fp32"]),
                "out": rng.choice(["bf16", "fp16", "fp32"]), "scale": round(rng.uniform(0.5, 2.0), 3), "pad": round(rng.uniform(0.0, 0.5), 3)}
    if op == "embed_grad":
        table = rng.choice(["bf16", "fp16", "fp32"])
        add = table == "fp32" and rng.random() < 0.5
        return {"op": op, "n": _span(rng, 1, 20480), "d": 4 * _span(rng, 32, 640), "vocab": _span(rng, 300, 100000), "dout": rng.choice(["bf16", "fp16", "fp32"]),
                "table": table, "scale": round(rng.uniform(0.5, 2.0), 3), "pad": round(rng.uniform(0.0, 0.9), 3), "accumulate": add}
    if op == "ffn":
        return {"op": op, "m": _span(rng, 1, 12860), "d": 64 * _span(rng, 4, 56), "f": 32 * _span(rng, 8, 592), "dtype": rng.choice(["bf16", "fp16"]), "save": rng.random() < 0.5}
    if op == "ffn_grad":
        return {"op": op, "m": _span(rng, 1, 12860), "d": 64 * _span(rng, 4, 56), "f": 32 * _span(rng, 8, 592), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "clip":
        return {"op": op, "kind": rng.choice(["projector", "decoder"]), "d": _span(rng, 100, HIDDEN), "f": _span(rng, 300, 9000), "layers": rng.randint(1, 4),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "max_norm": round(rng.uniform(0.1, 5.0), 3), "sigma": rng.choice([0.0001, 0.001, 0.01])}
    return {"op": op, "frames": _span(rng, 1, 600), "tokens": _span(rng, 1, 30), "d": 8 * _span(rng, 32, 512), "h": rng.choice(["bf16", "fp16", "fp32"]),
            "dh": rng.choice(["bf16", "fp16", "fp32"]), "positive": round(rng.uniform(0.0, 0.6), 3)}


def _shapes(case):
    """(shape, dtype name) of the gradients that one clipping call sees"""
    d, f, kind = case["d"], case["f"], case["dtype"]
    if case["kind"] == "projector":
        one = [((d, f), kind), ((d,), "fp32"), ((d, d), kind), ((d,), "fp32"), ((1, d), "fp32"), ((1,), "fp32")]
    else:
        kv = max(1, d // 7)
        one = [((d + 2 * kv, d), kind), ((d + 2 * kv,), "fp32"), ((d, d), kind), ((2 * f, d), kind), ((d, f), kind), ((d,), "fp32"), ((d,), "fp32")]
    return one * case["layers"]


def _ids(case, g):
    """token ids as a prompt batch has them: a long-tailed vocabulary, a share of one repeated id, and slots that hold no token (negative ids)"""
    n, vocab = case["n"], case["vocab"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (u ** 3 * vocab).long().clamp_(max=vocab - 1)
    kind = torch.rand(n, generator=g, device="cuda")
    ids[kind < case["pad"]] = vocab // 3
    ids[kind > 0.97] = -200
    return ids


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype="fp32", scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(DT[dtype])

    def randn_tall(rows, cols, dtype, scale):
        """the same, in pieces: no second copy of a large matrix in 32 bits"""
        out = torch.empty(rows, cols, device="cuda", dtype=DT[dtype])
        for i in range(0, rows, 8192):
            out[i:i + 8192] = randn(min(8192, rows - i), cols, scale=scale)
        return out

    s = {"case": case}
    op = case["op"]
    if op == "embed":
        s["ids"] = _ids(case, g)
        s["table"] = randn_tall(case["vocab"], case["d"], case["table"], 0.02)
        s["out"] = torch.empty(case["n"], case["d"], device="cuda", dtype=DT[case["out"]])
    elif op == "embed_grad":
        s["ids"] = _ids(case, g)
        s["dout"] = randn(case["n"], case["d"], dtype=case["dout"], scale=0.1)
        s["dtable"] = (randn_tall(case["vocab"], case["d"], case["table"], 0.1) if case["accumulate"] else
                       torch.empty(case["vocab"], case["d"], device="cuda", dtype=DT[case["table"]]))
    elif op in ("ffn", "ffn_grad"):
        m, d, f, dt = case["m"], case["d"], case["f"], case["dtype"]
        s["x"] = randn(m, d, dtype=dt)
        s["w"] = randn_tall(2 * f, d, dt, d ** -0.5)
        if op == "ffn":
            s["out"] = torch.empty(m, f, device="cuda", dtype=DT[dt])
            s["gu"] = torch.empty(m, 2 * f, device="cuda", dtype=DT[dt]) if case["save"] else None
        else:
            s["gu"] = randn_tall(m, 2 * f, dt, 1.0)
            s["dout"] = randn_tall(m, f, dt, 0.05)
            s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
    elif op == "clip":
        s["grads"] = [randn(*shape, dtype=kind, scale=case["sigma"]) for shape, kind in _shapes(case)]
        s["outs"] = [torch.empty_like(t) for t in s["grads"]]
    else:
        frames, tokens, d = case["frames"], case["tokens"], case["d"]
        s["h"] = randn(frames * tokens, d, dtype=case["h"])
        s["w"], s["b"] = randn(d, scale=d ** -0.5 * 5), randn(1)
        s["labels"] = (torch.rand(frames, generator=g, device="cuda") < case["positive"]).float()
        s["logits"], s["pooled"] = torch.empty(frames, device="cuda"), torch.empty(frames, d, device="cuda")
        s["dh"] = torch.empty(frames * tokens, d, device="cuda", dtype=DT[case["dh"]])
        s["dw"], s["db"] = torch.empty(d, device="cuda"), torch.empty(1, device="cuda")
    return s


def _halves(t):
    """[..., 2 f] laid as [32 gate | 32 up] blocks -> gate [..., f], up [..., f]"""
    b = t.unflatten(-1, (-1, 2, 32))
    return b[..., 0, :].flatten(-2), b[..., 1, :].flatten(-2)


def _interleave(gate, up):
    return torch.stack([gate.unflatten(-1, (-1, 32)), up.unflatten(-1, (-1, 32))], -2).flatten(-3)


def _run_own(s):
    from videoitg_amd import ops
    c = s["case"]
    op = c["op"]
    if op == "embed":
        return {"out": ops.embed_lookup(s["ids"], s["table"], s["out"], scale=c["scale"])}
    if op == "embed_grad":
        return {"dtable": ops.embed_backward(s["ids"], s["dout"], s["dtable"], scale=c["scale"], accumulate=c["accumulate"])}
    if op == "ffn":
        ops.swiglu(s["x"], s["w"], s["out"], gu=s["gu"])
        return {"out": s["out"], "gu": s["gu"]}
    if op == "ffn_grad":
        ops.swiglu_backward(s["dout"], s["gu"], s["x"], s["w"], dx=s["dx"], dw=s["dw"])
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "clip":
        return {"norm": ops.clip_grad_norm(s["grads"], c["max_norm"], outs=s["outs"]), "grads": s["outs"]}
    ops.pool_score_save(s["h"], c["frames"], c["tokens"], c["d"], s["w"], s["b"], s["logits"], s["pooled"])
    loss, _, dlogits = ops.bce_loss_backward(s["logits"], s["labels"])
    ops.pool_score_backward(s["pooled"], c["frames"], c["tokens"], c["d"], s["w"], dlogits, s["dh"], dw=s["dw"], db=s["db"])
    return {"logits": s["logits"], "loss": loss, "dlogits": dlogits, "dh": s["dh"], "dw": s["dw"], "db": s["db"]}


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    op = c["op"]
    if op in ("embed", "embed_grad"):
        ids = s["ids"]
        known = (ids >= 0) & (ids < c["vocab"])
        at = torch.where(known, ids, 0)
        if op == "embed":
            rows = s["table"][at].float() * c["scale"]
            return {"out": torch.where(known[:, None], rows, 0.0).to(DT[c["out"]])}
        rows = torch.where(known[:, None], s["dout"].float() * c["scale"], 0.0)
        if c["accumulate"]:
            s["dtable"].index_add_(0, at, rows)
            return {"dtable": s["dtable"]}
        return {"dtable": torch.zeros(c["vocab"], c["d"], device=rows.device).index_add_(0, at, rows).to(DT[c["table"]])}
    if op == "ffn":
        gate, up = _halves(s["x"].float() @ s["w"].float().t())
        out = (gate * torch.sigmoid(gate) * up).to(DT[c["dtype"]])
        return {"out": out, "gu": _interleave(gate, up).to(DT[c["dtype"]]) if c["save"] else None}
    if op == "ffn_grad":
        gate, up = _halves(s["gu"].float())
        dout, sig = s["dout"].float(), torch.sigmoid(gate)
        dgu = _interleave(dout * up * sig * (1.0 + gate * (1.0 - sig)), dout * gate * sig)
        return {"dx": (dgu @ s["w"].float()).to(DT[c["dtype"]]), "dw": (dgu.t() @ s["x"].float()).to(DT[c["dtype"]])}
    if op == "clip":
        norm = torch.stack([t.double().square().sum() for t in s["grads"]]).sum().sqrt()
        factor = torch.clamp(c["max_norm"] / (norm + 1e-6), max=1.0).float()
        return {"norm": norm.float().reshape(1), "grads": [(t.float() * factor).to(t.dtype) for t in s["grads"]]}
    w, y, n = s["w"], s["labels"], c["frames"]
    pooled = s["h"].float().view(n, c["tokens"], c["d"]).mean(1)
    z = (pooled * w).sum(1) + s["b"]
    positives = y.sum()
    weight = torch.sqrt((n - positives) / torch.clamp(positives, min=1.0)).clamp(max=5.0)
    softplus = torch.log1p(torch.exp(-z.abs())) + torch.clamp(-z, min=0.0)
    loss = ((1.0 - y) * z + (1.0 + (weight - 1.0) * y) * softplus).mean()
    dz = ((1.0 - y) - (1.0 + (weight - 1.0) * y) * torch.sigmoid(-z)) / n
    dh = (dz / c["tokens"])[:, None] * w
    dh = dh[:, None, :].expand(n, c["tokens"], c["d"]).reshape(n * c["tokens"], c["d"]).to(DT[c["dh"]])
    return {"logits": z, "loss": loss, "dlogits": dz, "dh": dh, "dw": (dz[:, None] * pooled).sum(0), "db": dz.sum().reshape(1)}


def work(case):
    op = case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if op == "embed":
        return {"bytes": case["n"] * (8 + case["d"] * (size[case["table"]] + size[case["out"]])), "flops": case["n"] * case["d"]}
    if op == "embed_grad":
        # an added gradient reads and writes the touched rows only: at most one for each token that is no repeat
        rows = min(case["vocab"], max(1, int(case["n"] * (1.0 - case["pad"]) * 0.9))) if case["accumulate"] else case["vocab"]
        return {"bytes": case["n"] * (8 + case["d"] * size[case["dout"]]) + rows * case["d"] * size[case["table"]] * (2 if case["accumulate"] else 1),
                "flops": 2 * case["n"] * case["d"]}
    if op == "ffn":
        m, d, f = case["m"], case["d"], case["f"]
        return {"bytes": 2 * (m * d + 2 * f * d + m * f * (3 if case["save"] else 1)), "flops": 4 * m * d * f}
    if op == "ffn_grad":
        m, d, f = case["m"], case["d"], case["f"]
        return {"bytes": 2 * (3 * m * f + 2 * m * d + 4 * f * d), "flops": 8 * m * d * f}
    if op == "clip":
        n = [(math.prod(shape), size[kind]) for shape, kind in _shapes(case)]
        return {"bytes": sum(k * b * 3 for k, b in n), "flops": sum(3 * k for k, _ in n)}
    n = case["frames"] * case["tokens"] * case["d"]
    return {"bytes": n * (size[case["h"]] + size[case["dh"]]) + 16 * case["frames"] + 12 * case["d"], "flops": 4 * n}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("embed", "embed_grad"):
        ids = s["ids"]
        good = torch.nonzero((ids >= 0) & (ids < case["vocab"])).flatten()
        if op == "embed":
            out = torch.zeros(case["n"], case["d"], device="cuda", dtype=torch.float64)
            out[good] = s["table"].index_select(0, ids[good]).double() * case["scale"]
            return {"out": out}
        # the sum of each distinct token's rows, set into the table
        token, which = torch.unique(ids[good], return_inverse=True)
        sums = torch.zeros(token.numel(), case["d"], device="cuda", dtype=torch.float64)
        sums.scatter_add_(0, which[:, None].expand(-1, case["d"]), s["dout"][good].double())
        table = s["dtable"].double() if case["accumulate"] else torch.zeros(case["vocab"], case["d"], device="cuda", dtype=torch.float64)
        table[token] += sums * case["scale"]
        return {"dtable": table}
    if op == "ffn":
        m, f = case["m"], case["f"]
        w = s["w"].view(f // 32, 2, 32, case["d"])
        gate = s["x"].double() @ w[:, 0].reshape(f, -1).double().t()
        up = s["x"].double() @ w[:, 1].reshape(f, -1).double().t()
        gu = None
        if case["save"]:
            gu = torch.empty(m, f // 32, 2, 32, device="cuda", dtype=torch.float64)
            gu[:, :, 0], gu[:, :, 1] = gate.view(m, -1, 32), up.view(m, -1, 32)
            gu = gu.view(m, 2 * f)
        return {"out": up.mul_(gate.div_(1.0 + torch.exp(-gate))), "gu": gu}
    if op == "ffn_grad":
        m, f, d = case["m"], case["f"], case["d"]
        gu, w = s["gu"].view(m, f // 32, 2, 32), s["w"].view(f // 32, 2, 32, d)
        gate, dout = gu[:, :, 0].reshape(m, f).double(), s["dout"].double()
        grow = torch.exp(-gate)                                     # silu(g) = g / (1 + e^-g), silu'(g) = (1 + e^-g + g e^-g) / (1 + e^-g)^2
        dup = dout * gate / (1.0 + grow)
        dgate = dout * gu[:, :, 1].reshape(m, f).double() * (1.0 + grow + gate * grow) / (1.0 + grow).square()
        dw = torch.empty(f // 32, 2, 32, d, device="cuda", dtype=torch.float64)
        x = s["x"].double()
        dw[:, 0], dw[:, 1] = (dgate.t() @ x).view(-1, 32, d), (dup.t() @ x).view(-1, 32, d)
        dx = dgate @ w[:, 0].reshape(f, d).double() + dup @ w[:, 1].reshape(f, d).double()
        return {"dx": dx, "dw": dw.view(2 * f, d)}
    if op == "clip":
        total = sum(float(torch.linalg.vector_norm(t.double())) ** 2 for t in s["grads"])
        norm = math.sqrt(total)
        factor = min(1.0, case["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor([norm], dtype=torch.float64), "grads": [t.double() * factor for t in s["grads"]]}
    n, k, d = case["frames"], case["tokens"], case["d"]
    h, w, y = s["h"].double().view(n, k, d), s["w"].double(), s["labels"].double()
    pooled = h.sum(1) / k
    z = pooled @ w + s["b"].double()
    positives = float(y.sum())
    weight = min(5.0, math.sqrt((n - positives) / max(1.0, positives)))
    log_p, log_q = torch.nn.functional.logsigmoid(z), torch.nn.functional.logsigmoid(-z)
    loss = -(weight * y * log_p + (1.0 - y) * log_q).sum() / n
    dz = (torch.sigmoid(z) * (1.0 - y) - weight * y * torch.sigmoid(-z)) / n
    dh = torch.einsum("t,d->td", dz / k, w).repeat_interleave(k, 0)
    return {"logits": z, "loss": loss, "dlogits": dz, "dh": dh, "dw": pooled.t() @ dz, "db": dz.sum().reshape(1)}
