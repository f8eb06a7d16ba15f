"""The training operators' workloads: LayerNorm forward and backward, the classifier's Linear + softmax cross entropy with
its gradients, and the global gradient norm with clipping.

`listed()` names fixed cases and `draw(rng)` one more of the same ranges; `prepare` makes a case's inputs on the GPU from a
seed, `run` takes one pass through the operator -- the package's entry points where `own` is true, elementary torch
operations in 32 bits where it is false -- and `exact` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}
IGNORE = -100


def listed():
    return [
        # the temporal encoder's norm while serving: 8 clips of 128 frames, width 512, fp32 residual stream in, bf16 GEMM
        # operand out
        {"name": "norm_encoder_forward", "op": "norm", "rows": 1024, "d": 512, "x": "fp32", "w": "fp32", "y": "bf16",
         "train": False},
        # a width that no vector divides, as a concatenation of features gives it; forward and backward
        {"name": "norm_odd_train", "op": "norm", "rows": 1237, "d": 777, "x": "bf16", "w": "fp32", "y": "bf16", "train": True},
        # frames of a long training batch at ResNet-50's feature width, forward and backward
        {"name": "norm_long_train", "op": "norm", "rows": 65536, "d": 2048, "x": "bf16", "w": "bf16", "y": "bf16",
         "train": True},
        # tuning the 2000-class head on pooled features of 8 clips: fp32 masters, one small step, latency counts
        {"name": "loss_head_8_clips", "op": "loss", "n": 8, "classes": 2000, "d": 512, "x": "fp32", "bias": True,
         "smoothing": 0.0, "ignored": 0.0, "train": True},
        # a label per frame, 8 clips of 128 frames, smoothed labels
        {"name": "loss_frames", "op": "loss", "n": 1024, "classes": 2000, "d": 512, "x": "bf16", "bias": True,
         "smoothing": 0.1, "ignored": 0.1, "train": True},
        # nothing divides anything: odd width, odd vocabulary, a third of the frames unlabelled
        {"name": "loss_odd", "op": "loss", "n": 777, "classes": 5003, "d": 509, "x": "bf16", "bias": True,
         "smoothing": 0.0, "ignored": 0.33, "train": True},
        # fp32 training of a mid-sized open vocabulary on I3D-wide features
        {"name": "loss_fp32", "op": "loss", "n": 2048, "classes": 8192, "d": 1024, "x": "fp32", "bias": True,
         "smoothing": 0.0, "ignored": 0.05, "train": True},
        # the loss alone, as validation computes it
        {"name": "loss_validation", "op": "loss", "n": 4096, "classes": 32768, "d": 1024, "x": "bf16", "bias": True,
         "smoothing": 0.0, "ignored": 0.05, "train": False},
        # a large token vocabulary at ResNet-50's feature width: the largest matrix work
        {"name": "loss_large", "op": "loss", "n": 8192, "classes": 32768, "d": 2048, "x": "bf16", "bias": False,
         "smoothing": 0.0, "ignored": 0.05, "train": True},
        # gradients of the classifier end alone (last norm + 100-class head)
        {"name": "clip_head", "op": "clip", "layers": 0, "d": 512, "ffn": 0, "classes": 100, "g": "fp32", "out": "fp32",
         "factor": 0.5},
        # gradients of the two-stream model's encoder: 4 layers of width 512 and its 2000-class head
        {"name": "clip_encoder", "op": "clip", "layers": 4, "d": 512, "ffn": 2048, "classes": 2000, "g": "fp32", "out": "fp32",
         "factor": 0.5},
        # a large encoder's bf16 gradients clipped into the fp32 buffers its optimizer reads
        {"name": "clip_large", "op": "clip", "layers": 16, "d": 1280, "ffn": 5120, "classes": 32768, "g": "bf16", "out": "fp32",
         "factor": 0.5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "loss", "clip"])
    if op == "norm":
        rows = _log_int(rng, 1, 65536)
        d = _log_int(rng, 16, min(16384, 65536 * 2048 // rows))
        return {"op": "norm", "rows": rows, "d": d, "x": rng.choice(["fp32", "bf16", "bf16"]), "w": rng.choice(["fp32", "bf16"]),
                "y": rng.choice(["fp32", "bf16", "bf16"]), "train": rng.random() < 0.7}
    if op == "loss":
        x = rng.choice(["fp32", "bf16", "bf16"])
        # an fp32 case is bounded by the listed fp32 one, a bf16 case by the largest
        most = 2048 * 8192 * 1024 if x == "fp32" else 8192 * 32768 * 2048
        n = _log_int(rng, 1, 8192)
        d = _log_int(rng, 8, 4096)
        classes = _log_int(rng, 2, max(2, min(65536, most // (n * d))))
        return {"op": "loss", "n": n, "classes": classes, "d": d, "x": x, "bias": rng.random() < 0.6,
                "smoothing": rng.choice([0.0, 0.0, 0.1]), "ignored": rng.choice([0.0, 0.05, 0.5]),
                "train": rng.random() < 0.75}
    d = _log_int(rng, 16, 1280)
    layers = rng.randint(0, 16)
    return {"op": "clip", "layers": layers, "d": d, "ffn": d * rng.randint(1, 4) + rng.randint(0, 3),
            "classes": _log_int(rng, 2, 32768), "g": rng.choice(["fp32", "bf16"]), "out": rng.choice(["fp32", "bf16"]),
            "factor": rng.choice([0.01, 0.5, 2.0])}


def _shapes(case):
    """parameter shapes of a post-norm encoder with a classifier head"""
    d, f, c = case["d"], case["ffn"], case["classes"]
    layer = [(3 * d, d), (3 * d,), (d, d), (d,), (f, d), (f,), (d, f), (d,), (d,), (d,), (d,), (d,)]
    return layer * case["layers"] + [(d,), (d,), (c, d), (c,)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        # a residual stream: an offset, and a few channels that stand out
        x = randn(rows, d).mul_(1.5).add_(0.3)
        x[:, ::97] *= 8.0
        st = {"x": x.to(DTYPES[case["x"]]), "w": (1.0 + 0.1 * randn(d)).to(DTYPES[case["w"]]),
              "b": (0.1 * randn(d)).to(DTYPES[case["w"]])}
        if case["train"]:
            st["dy"] = (1e-2 * randn(rows, d)).to(DTYPES[case["y"]])
    elif case["op"] == "loss":
        n, v, d = case["n"], case["classes"], case["d"]
        t = torch.randint(0, v, (n,), generator=g, device="cuda")
        w = randn(v, d).mul_(2.0 / math.sqrt(d))
        # features that point, some strongly, to their class: losses from near nought to large ones
        x = randn(n, d) + (2.5 * torch.rand(n, 1, generator=g, device="cuda")) * w[t]
        drop = torch.rand(n, generator=g, device="cuda") < case["ignored"]
        drop[0] = False
        t[drop] = IGNORE
        st = {"x": x.to(DTYPES[case["x"]]), "w": w.to(DTYPES[case["x"]]), "t": t,
              "b": (0.1 * randn(v)).to(DTYPES[case["x"]]) if case["bias"] else None}
    else:
        dt = DTYPES[case["g"]]
        # tensors of one model differ in the size of their gradients
        grads = [(randn(*s) * (1e-3 * 4.0 ** (i % 5 - 2))).to(dt) for i, s in enumerate(_shapes(case))]
        norm = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
        # the optimizer's gradients lie in one buffer, tensor behind tensor
        flat = torch.empty(sum(t.numel() for t in grads), dtype=DTYPES[case["out"]], device="cuda")
        out = [o.view(t.shape) for o, t in zip(flat.split([t.numel() for t in grads]), grads)]
        st = {"g": grads, "flat": flat, "out": out, "max_norm": case["factor"] * norm}
    st["case"] = case
    return st


def run(state):
    case = state["case"]
    return {"norm": _norm, "loss": _loss, "clip": _clip}[case["op"]](case, state)


def _norm(case, st):
    x, w, b, eps = st["x"], st["w"], st["b"], 1e-5
    yt = DTYPES[case["y"]]
    if own:
        from video_asl_recognition_amd import training
        y, mean, rstd = training.layer_norm_fwd(x, w, b, eps, out_dtype=yt)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = training.layer_norm_bwd(st["dy"], x, w, mean, rstd)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    xf, wf = x.float(), w.float()
    xc = xf - xf.mean(1, keepdim=True)
    rstd = torch.rsqrt(xc.square().mean(1, keepdim=True) + eps)
    h = xc * rstd
    y = (h * wf + b.float()).to(yt)
    if not case["train"]:
        return {"y": y}
    dy = st["dy"].float()
    gg = dy * wf
    dx = rstd * (gg - gg.mean(1, keepdim=True) - h * (gg * h).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dw": (dy * h).sum(0).to(w.dtype), "db": dy.sum(0).to(w.dtype)}


def _loss(case, st):
    x, w, b, t, s = st["x"], st["w"], st["b"], st["t"], case["smoothing"]
    if own:
        from video_asl_recognition_amd import training
        if not case["train"]:
            loss, lse = training.linear_cross_entropy_fwd(x, w, t, b, ignore_index=IGNORE, label_smoothing=s, reduction="none")
            return {"loss": loss, "lse": lse}
        loss, dx, dw, db = training.linear_cross_entropy_grad(x, w, t, b, ignore_index=IGNORE, label_smoothing=s)
        return {"loss": loss, "dx": dx, "dw": dw, "db": db} if b is not None else {"loss": loss, "dx": dx, "dw": dw}
    xf, wf = x.float(), w.float()
    z = xf @ wf.t()
    if b is not None:
        z += b.float()
    v = z.shape[1]
    keep = t != IGNORE
    at = torch.where(keep, t, torch.zeros_like(t))[:, None]
    top = z.max(1, keepdim=True).values
    lse = top + (z - top).exp().sum(1, keepdim=True).log()
    rows = (lse - (1.0 - s) * z.gather(1, at)).squeeze(1)
    if s:
        rows = rows - s * z.mean(1)
    rows = torch.where(keep, rows, torch.zeros_like(rows))
    if not case["train"]:
        return {"loss": rows, "lse": lse.squeeze(1)}
    count = keep.sum().float()
    p = (z - lse).exp() - s / v
    p.scatter_add_(1, at, torch.full_like(lse, -(1.0 - s)))
    p *= (keep.float() / count)[:, None]
    p = torch.where(keep[:, None], p, torch.zeros_like(p))
    out = {"loss": rows.sum() / count, "dx": (p @ wf).to(x.dtype), "dw": (p.t() @ xf).to(w.dtype)}
    if b is not None:
        out["db"] = p.sum(0).to(b.dtype)
    return out


def _clip(case, st):
    if own:
        from video_asl_recognition_amd import training
        norm = training.clip_grads(st["g"], st["max_norm"], out=st["out"])
        return {"norm": norm, "out": st["flat"]}
    norm = torch.stack([t.float().square().sum() for t in st["g"]]).sum().sqrt()
    c = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for t, o in zip(st["g"], st["out"]):
        o.copy_(t.float() * c)
    return {"norm": norm, "out": st["flat"]}


def work(case):
    if case["op"] == "norm":
        e, d = case["rows"] * case["d"], case["d"]
        sx, sw, sy = SIZE[case["x"]], SIZE[case["w"]], SIZE[case["y"]]
        nbytes, flops = e * (sx + sy) + 2 * d * sw, 8 * e
        if case["train"]:
            nbytes += e * (sy + sx) + 2 * d * sw
            flops += 15 * e
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "loss":
        n, v, d, s = case["n"], case["classes"], case["d"], SIZE[case["x"]]
        once = (n * d + v * d + (v if case["bias"] else 0)) * s
        if not case["train"]:
            return {"bytes": once + 12 * n, "flops": 2 * n * v * d}
        return {"bytes": 2 * once + 8 * n, "flops": 6 * n * v * d}
    e = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": e * (SIZE[case["g"]] + SIZE[case["out"]]), "flops": 3 * e}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "clip":
        squares = 0.0
        for t in st["g"]:
            squares += float((t.double() ** 2).sum())
        norm = math.sqrt(squares)
        scale = min(1.0, st["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda"),
                "out": torch.cat([t.double().flatten() for t in st["g"]]).mul_(scale)}
    x, w = st["x"].double(), st["w"].double()
    b = None if st["b"] is None else st["b"].double()
    if case["op"] == "norm":
        var, mu = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        y = (x - mu) / sd * w + b
        if not case["train"]:
            return {"y": y}
        dy = st["dy"].double()
        h = (x - mu) / sd
        u = dy * w
        dx = (u - u.mean(1, keepdim=True) - h * (u * h).mean(1, keepdim=True)) / sd
        return {"y": y, "dx": dx, "dw": (dy * h).sum(0), "db": dy.sum(0)}
    t, s, v = st["t"], case["smoothing"], case["classes"]
    logp = x @ w.t()
    if b is not None:
        logp += b
    lse = torch.logsumexp(logp, 1)
    logp -= lse[:, None]
    kept = torch.nonzero(t != IGNORE).squeeze(1)
    rows = torch.zeros(case["n"], dtype=torch.float64, device="cuda")
    rows[kept] = -(1.0 - s) * logp[kept, t[kept]] - (s / v) * logp[kept].sum(1) if s else -logp[kept, t[kept]]
    if not case["train"]:
        return {"loss": rows, "lse": lse}
    grad = torch.zeros_like(logp)
    grad[kept] = logp[kept].exp() - s / v
    grad[kept, t[kept]] -= 1.0 - s
    grad /= kept.numel()
    out = {"loss": rows.sum() / kept.numel(), "dx": grad @ w, "dw": grad.t() @ x}
    if b is not None:
        out["db"] = grad.sum(0)
    return out
