"""The workloads of the learning operators: group norm with an activation, distillation from a
teacher's top logits, and the product of 8-bit operands with a scale for each block of 128.

`own` false runs each operator in its plain form (elementary torch operations in 32 bits, 64 where
32 lose what matters); `own` true makes the calls a user makes of the framework.  `exact` gives the
same outputs from the definitions in 64 bits."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f64": 8, "f16": 2, "bf16": 2}
_FP8 = torch.float8_e4m3fn


def _pcu():
    import importlib

    return importlib.import_module("fusion-pcu_b200")


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the loss of a few evaluated positions, over a large vocabulary: latency counts
        {"name": "distill_eval_4x131072", "op": "distill", "mode": "loss", "dtype": "bf16", "rows": 4, "vocab": 131072,
         "k": 32, "temperature": 1.0, "pad": 0, "ragged": False},
        # a training step's loss and gradient, a whole batch of positions, some of them padding
        {"name": "distill_step_4096x131072", "op": "distill", "mode": "step", "dtype": "bf16", "rows": 4096,
         "vocab": 131072, "k": 64, "temperature": 2.0, "pad": 0, "ragged": True},
        # the same in binary32 with an odd vocabulary in padded rows, an odd number of teacher entries
        {"name": "distill_step_777x50003", "op": "distill", "mode": "step", "dtype": "f32", "rows": 777, "vocab": 50003,
         "k": 17, "temperature": 1.5, "pad": 5, "ragged": True},
        # the gradient alone, its upstream known only after the forward pass
        {"name": "distill_backward_2048x32768", "op": "distill", "mode": "backward", "dtype": "bf16", "rows": 2048,
         "vocab": 32768, "k": 128, "temperature": 1.0, "pad": 0, "ragged": False},
        # a hidden layer of the 4-layer MLP (batch 8192, width 4096): one position per sample
        {"name": "norm_8192x4096_relu", "op": "norm", "mode": "forward", "dtype": "f32", "batch": 8192, "positions": 1,
         "channels": 4096, "groups": 32, "act": "relu", "affine": True, "pad": 0},
        # feature maps of odd extent (63 x 65 positions), channels last
        {"name": "norm_5x4095x320_silu", "op": "norm", "mode": "forward", "dtype": "bf16", "batch": 5, "positions": 4095,
         "channels": 320, "groups": 32, "act": "silu", "affine": True, "pad": 0},
        # the MLP layer's backward pass
        {"name": "norm_backward_8192x4096_relu", "op": "norm", "mode": "backward", "dtype": "f32", "batch": 8192,
         "positions": 1, "channels": 4096, "groups": 32, "act": "relu", "affine": True, "pad": 0},
        # feature maps' backward pass
        {"name": "norm_backward_16x1024x640_silu", "op": "norm", "mode": "backward", "dtype": "bf16", "batch": 16,
         "positions": 1024, "channels": 640, "groups": 32, "act": "silu", "affine": True, "pad": 0},
        # one row through a quantised layer: the weights' bytes count
        {"name": "block_1x4096x16384", "op": "block", "mode": "product", "dtype": "bf16", "out": "bf16", "rows": 1,
         "inner": 4096, "columns": 16384},
        # a hidden layer of the 4-layer MLP, whole batch
        {"name": "block_8192x4096x4096", "op": "block", "mode": "product", "dtype": "bf16", "out": "bf16", "rows": 8192,
         "inner": 4096, "columns": 4096},
        # odd extents in every direction, binary32 in and out
        {"name": "block_300x1111x1000", "op": "block", "mode": "product", "dtype": "f32", "out": "f32", "rows": 300,
         "inner": 1111, "columns": 1000},
        # laying out a weight matrix once: scales for tiles of 128 x 128
        {"name": "block_weights_16384x4096", "op": "block", "mode": "weights", "dtype": "f32", "out": "f32", "rows": 16384,
         "inner": 4096, "columns": 1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["distill", "norm", "block"])
    if op == "distill":
        rows, vocab = _log(rng, 1, 4096), _log(rng, 130, 200000)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32", "f32", "f64"])
        while rows * vocab * _BYTES[dtype] > 1 << 29:
            rows = max(1, rows // 2)
        return {"op": op, "mode": rng.choice(["loss", "step", "backward"]), "dtype": dtype, "rows": rows, "vocab": vocab,
                "k": min(_log(rng, 1, 256), vocab // 2), "temperature": rng.choice([0.7, 1.0, 2.0, 4.0]),
                "pad": rng.choice([0, 0, 1, 8]), "ragged": rng.random() < 0.5}
    if op == "norm":
        groups, width = _log(rng, 1, 64), _log(rng, 1, 200)
        batch, positions = _log(rng, 1, 4096), _log(rng, 1, 16384)
        if groups == 1 and width == 1 and positions == 1:
            width = 8
        dtype = rng.choice(["bf16", "bf16", "f16", "f32", "f32", "f64"])
        if width * positions < 4:  # a handful of values has a variance near zero now and then
            width += 3
        while batch > 1 and batch * positions * groups * width * _BYTES[dtype] > 1 << 27:
            batch = max(1, batch // 2)
        while batch * positions * groups * width * _BYTES[dtype] > 1 << 27:
            positions = positions // 2
        return {"op": op, "mode": rng.choice(["forward", "backward"]), "dtype": dtype, "batch": batch,
                "positions": positions, "channels": groups * width, "groups": groups,
                "act": rng.choice(["none", "relu", "silu", "gelu"]), "affine": rng.random() < 0.75,
                "pad": rng.choice([0, 0, 1, 8])}
    rows, inner, columns = _log(rng, 1, 8192), _log(rng, 64, 16384), _log(rng, 64, 16384)
    while rows * inner * columns > 1 << 36:
        rows = max(1, rows // 2)
    weights = rng.random() < 0.2
    return {"op": op, "mode": "weights" if weights else "product", "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "rows": rows, "inner": inner,
            "columns": 1 if weights else columns}


def work(case):
    b = _BYTES[case["dtype"]]
    if case["op"] == "distill":
        n = case["rows"] * case["vocab"]
        passes = 1 if case["mode"] == "loss" else 2
        return {"bytes": passes * n * b + case["rows"] * case["k"] * (12 if b <= 4 else 16), "flops": 4 * passes * n}
    if case["op"] == "norm":
        n = case["batch"] * case["positions"] * case["channels"]
        return {"bytes": (2 if case["mode"] == "forward" else 3) * n * b,
                "flops": (10 if case["mode"] == "forward" else 20) * n}
    m, k, n = case["rows"], case["inner"], case["columns"]
    if case["mode"] == "weights":
        return {"bytes": m * k * (b + 1), "flops": 2 * m * k}
    return {"bytes": m * k * (b + 1) + n * k + m * n * _BYTES[case["out"]], "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _padded(values, dtype, pad):
    """`values` as a view whose rows are `pad` elements longer than they are read."""
    if not pad:
        return values.to(dtype).contiguous()
    base = torch.zeros(values.shape[:-1] + (values.shape[-1] + pad,), dtype=dtype, device="cuda")
    base[..., :values.shape[-1]] = values
    return base[..., :values.shape[-1]]


def _distill_inputs(case, seed):
    g = _generator(seed)
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    dtype = _TYPES[case["dtype"]]
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    teacher = _normal(g, (rows, vocab))
    teacher *= 3.0
    top_logits, top_indices = teacher.topk(k, dim=1)
    teacher *= 0.7
    teacher += _normal(g, (rows, vocab))
    logits = _padded(teacher, dtype, case["pad"])
    del teacher
    weights = None
    if case["ragged"]:
        # a tenth of the positions is padding; some have fewer teacher entries than k
        weights = (torch.rand(rows, generator=g, device="cuda") > 0.1).to(wide)
        kept = torch.randint(1, k + 1, (rows, 1), generator=g, device="cuda")
        top_indices = torch.where(torch.arange(k, device="cuda")[None, :] < kept, top_indices, -1)
    upstream = torch.full((1,), 1.0 / rows, dtype=wide, device="cuda")
    if case["mode"] == "backward":
        upstream = torch.rand(rows, generator=g, device="cuda").to(wide) + 0.5
    return {"logits": logits, "indices": top_indices.contiguous(), "top": top_logits.to(wide).contiguous(),
            "weights": weights, "upstream": upstream}


def _norm_inputs(case, seed):
    g = _generator(seed)
    n, s, c = case["batch"], case["positions"], case["channels"]
    dtype = _TYPES[case["dtype"]]
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    scale, shift = torch.rand(c, generator=g, device="cuda") + 0.5, _normal(g, (c,))
    x = _padded(_normal(g, (n, s, c)) * scale + 0.5 * shift, dtype, case["pad"])
    given = {"x": x, "weight": None, "bias": None, "dy": None}
    if case["affine"]:
        given["weight"] = (1.0 + 0.2 * _normal(g, (c,))).to(wide)
        given["bias"] = (0.2 * _normal(g, (c,))).to(wide)
    if case["mode"] == "backward":
        given["dy"] = _padded(_normal(g, (n, s, c)), dtype, case["pad"])
    return given


def _room(columns):
    """The row stride of 8-bit codes: whole 16-byte pieces."""
    return (columns + 15) // 16 * 16


def _block_inputs(case, seed):
    g = _generator(seed)
    x = _normal(g, (case["rows"], case["inner"])) * torch.exp(_normal(g, (case["rows"], 1)))
    given = {"x": x.to(_TYPES[case["dtype"]])}
    if case["mode"] == "product":
        w = _normal(g, (case["columns"], case["inner"])) / math.sqrt(case["inner"])
        codes, given["w_scales"] = _quantize(w, 128)
        given["w"] = torch.zeros((case["columns"], _room(case["inner"])), dtype=torch.uint8, device="cuda").view(_FP8)
        given["w"].view(torch.uint8)[:, :case["inner"]] = codes.view(torch.uint8)
        given["w"] = given["w"][:, :case["inner"]]
    return given


def prepare(case, seed):
    """Inputs, and the buffers for results that a program keeps from step to step."""
    if case["op"] == "distill":
        given = _distill_inputs(case, seed)
        wide = given["top"].dtype
        given["loss"] = torch.empty(case["rows"], dtype=wide, device="cuda")
        given["stats"] = torch.empty((case["rows"], 2), dtype=wide, device="cuda")
        if case["mode"] == "backward":
            given["stats"] = _distill_plain(case, given, "loss")[1]
        if case["mode"] != "loss":
            given["gradient"] = torch.empty((case["rows"], case["vocab"]), dtype=given["logits"].dtype, device="cuda")
    elif case["op"] == "norm":
        given = _norm_inputs(case, seed)
        wide = torch.float64 if given["x"].dtype == torch.float64 else torch.float32
        if case["mode"] == "backward":
            given["stats"] = _norm_forward_plain(case, given)[1]
        else:
            given["stats"] = torch.empty((case["batch"], case["groups"], 2), dtype=wide, device="cuda")
        given["out"] = torch.empty(given["x"].shape, dtype=given["x"].dtype, device="cuda")
    else:
        given = _block_inputs(case, seed)
        m, k = case["rows"], case["inner"]
        high = 1 if case["mode"] == "product" else 128
        given["codes"] = torch.empty((m, _room(k)), dtype=torch.uint8, device="cuda").view(_FP8)[:, :k]
        given["scales"] = torch.empty((-(-m // high), -(-k // 128)), dtype=torch.float32, device="cuda")
        if case["mode"] == "product":
            given["out"] = torch.empty((m, case["columns"]), dtype=_TYPES[case["out"]], device="cuda")
    given["status"] = torch.full((2,), -1, dtype=torch.int64, device="cuda")
    given["case"] = case
    return given


# ------------------------------------------------------------------------------------ plain forms

def _distill_plain(case, s, mode):
    wide = s["top"].dtype
    t = case["temperature"]
    z = s["logits"].to(wide)
    keep = torch.ones(z.shape[0], dtype=torch.bool, device=z.device) if s["weights"] is None else s["weights"] != 0
    weight = torch.ones_like(s["top"][:, 0]) if s["weights"] is None else s["weights"]
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp((z - top) / t)
    total = e.sum(dim=1, keepdim=True)
    # the teacher's softmax and the rows' losses are differences of logarithms: in 64 bits
    present = s["indices"] >= 0
    some = present.any(dim=1)
    at = torch.where(present, s["indices"], 0)
    a = torch.where(present, s["top"].double() / t, -math.inf)
    a = a - torch.where(some, a.amax(dim=1), 0.0)[:, None]
    pe = torch.exp(a)
    psum = torch.where(some, pe.sum(dim=1), 1.0)[:, None]
    p = pe / psum
    stats = torch.where(keep[:, None], torch.cat([top, total], dim=1), torch.tensor([0.0, 1.0], dtype=wide, device=z.device))
    loss = gradient = None
    if mode != "backward":
        ln_q = (z.gather(1, at).double() - top.double()) / t - torch.log(total.double())
        ln_p = torch.where(p > 0, a - torch.log(psum), 0.0)
        terms = torch.where(p > 0, p * (ln_p - ln_q), 0.0)
        loss = torch.where(keep, weight.double() * t * t * terms.sum(dim=1), 0.0).to(wide)
    if mode != "loss":
        factor = torch.where(keep & some, s["upstream"] * weight * t, 0.0)[:, None]
        e /= total
        e.scatter_add_(1, at, torch.where(present, -p, 0.0).to(wide))
        e *= factor
        gradient = e.to(s["logits"].dtype)
    return loss, stats, gradient


def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


_EPS = 1e-5


def _norm_forward_plain(case, s):
    n, p, c = s["x"].shape
    g = case["groups"]
    wide = torch.float64 if s["x"].dtype == torch.float64 else torch.float32
    x = s["x"].to(wide).reshape(n, p, g, c // g)
    mean = x.mean(dim=(1, 3), keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + _EPS)
    z = (d * rstd).reshape(n, p, c)
    if s["weight"] is not None:
        z = z * s["weight"] + s["bias"]
    y = _act(z, case["act"]).to(s["x"].dtype)
    return y, torch.stack([mean.reshape(n, g), rstd.reshape(n, g)], dim=2)


def _norm_backward_plain(case, s):
    n, p, c = s["x"].shape
    g = case["groups"]
    wide = s["stats"].dtype
    mean, rstd = s["stats"][:, None, :, None, 0], s["stats"][:, None, :, None, 1]
    h = ((s["x"].to(wide).reshape(n, p, g, c // g) - mean) * rstd).reshape(n, p, c)
    if case["act"] == "relu":  # a step at 0: the side that z is on, in 64 bits
        z = s["x"].double().reshape(n, p, g, c // g) - mean.double()
        z = (z * rstd.double()).reshape(n, p, c)
    else:
        z = h
    z = z if s["weight"] is None else z * s["weight"] + s["bias"]
    dz = s["dy"].to(wide) * _act_slope(z, case["act"]).to(wide)
    dw, db = None, None
    if s["weight"] is not None:
        dw, db = (dz * h).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
        dz = dz * s["weight"]
    dz, h = dz.reshape(n, p, g, c // g), h.reshape(n, p, g, c // g)
    c1 = dz.mean(dim=(1, 3), keepdim=True)
    c2 = (dz * h).mean(dim=(1, 3), keepdim=True)
    dx = (rstd * (dz - c1 - h * c2)).reshape(n, p, c).to(s["x"].dtype)
    return dx, dw, db


def _quantize(x, high):
    """Codes and scales of blocks of `high` rows and 128 columns: the scale is the smallest power of
    two that brings the block's largest magnitude to 448 or below (1 for a block of zeros), so a
    quotient by it is exact."""
    x = x.float()
    m, k = x.shape
    mb, kb = -(-m // high), -(-k // 128)
    full = torch.zeros((mb * high, kb * 128), dtype=torch.float32, device=x.device)
    full[:m, :k] = x
    full = full.reshape(mb, high, kb, 128)
    amax = full.abs().amax(dim=(1, 3))
    part, power = torch.frexp(amax)  # amax = part 2^power, part in [0.5, 1); 448 = 0.875 2^9
    power = torch.where(part > 0.875, power - 8, power - 9).clamp(min=-126)
    scales = torch.where(amax > 0, (power + 127 << 23).to(torch.int32).view(torch.float32), 1.0)
    codes = (full / scales[:, None, :, None]).reshape(mb * high, kb * 128)[:m, :k].to(_FP8)
    return codes, scales


def _widen(codes, scales, high):
    """The values that codes and scales stand for."""
    m, k = codes.shape
    return codes.float() * scales.repeat_interleave(high, 0)[:m].repeat_interleave(128, 1)[:, :k]


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "distill":
            loss, stats, gradient = _distill_plain(case, state, case["mode"])
            return {"loss": loss, "stats": None if case["mode"] == "backward" else stats, "gradient": gradient}
        if case["op"] == "norm":
            if case["mode"] == "forward":
                return list(_norm_forward_plain(case, state))
            return list(_norm_backward_plain(case, state))
        codes, scales = _quantize(state["x"], 1 if case["mode"] == "product" else 128)
        if case["mode"] == "weights":
            return [codes, scales]
        out = _widen(codes, scales, 1) @ _widen(state["w"], state["w_scales"], 128).t()
        return [out.to(_TYPES[case["out"]]), codes, scales]

    pcu = _pcu()
    status = state["status"]
    if case["op"] == "distill":
        if case["mode"] == "loss":
            pcu.distill_loss(state["logits"], state["indices"], state["top"], temperature=case["temperature"],
                             row_weights=state["weights"], loss=state["loss"], stats=state["stats"], status=status[:1])
            return {"loss": state["loss"], "stats": state["stats"], "gradient": None}
        if case["mode"] == "step":
            pcu.distill_loss_step(state["logits"], state["indices"], state["top"], upstream=state["upstream"],
                                  temperature=case["temperature"], row_weights=state["weights"], loss=state["loss"],
                                  stats=state["stats"], gradient=state["gradient"], status=status[:1])
            return {"loss": state["loss"], "stats": state["stats"], "gradient": state["gradient"]}
        pcu.distill_loss_backward(state["logits"], state["indices"], state["top"], state["stats"],
                                  upstream=state["upstream"], temperature=case["temperature"],
                                  row_weights=state["weights"], gradient=state["gradient"], status=status[:1])
        return {"loss": None, "stats": None, "gradient": state["gradient"]}
    if case["op"] == "norm":
        if case["mode"] == "forward":
            return list(pcu.group_norm(state["x"], case["groups"], state["weight"], state["bias"],
                                       activation=case["act"], eps=_EPS, out=state["out"], stats=state["stats"],
                                       status=status[:1]))
        return list(pcu.group_norm_backward(state["x"], state["dy"], case["groups"], state["stats"], state["weight"],
                                            state["bias"], activation=case["act"], dx=state["out"], status=status[:1]))
    if case["mode"] == "weights":
        return list(pcu.block_quantize(state["x"], 128, codes=state["codes"], scales=state["scales"], status=status[:1]))
    codes, scales = pcu.block_quantize(state["x"], 1, codes=state["codes"], scales=state["scales"], status=status[:1])
    out = pcu.block_matmul(codes, scales, state["w"], state["w_scales"], out=state["out"], status=status[1:])
    return [out, codes, scales]


# ------------------------------------------------------------------------------------ 64 bits

def _distill_exact(case, seed):
    s = _distill_inputs(case, seed)
    rows, vocab = s["logits"].shape
    t = float(case["temperature"])
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    stats = torch.zeros((rows, 2), dtype=torch.float64, device="cuda")
    gradient = None if case["mode"] == "loss" else torch.zeros((rows, vocab), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // vocab)
    for i in range(0, rows, step):
        z = s["logits"][i:i + step].double()
        j = s["indices"][i:i + step]
        there = j >= 0
        m = z.max(dim=1).values
        total = ((z - m[:, None]) / t).exp().sum(dim=1)
        ln_q = (z - m[:, None]) / t - total.log()[:, None]
        u = (s["top"][i:i + step].double() / t).masked_fill(~there, -math.inf)
        any_ = there.any(dim=1)
        u = u.masked_fill(~any_[:, None], 0.0)
        ln_p = u - torch.logsumexp(u, dim=1, keepdim=True)
        p = ln_p.exp() * there
        w = torch.ones_like(m) if s["weights"] is None else s["weights"][i:i + step].double()
        use = (w != 0).double()
        chosen = ln_q.gather(1, j.clamp(min=0))
        loss[i:i + step] = w * t * t * (p * torch.where(there, ln_p - chosen, 0.0)).sum(dim=1)
        stats[i:i + step, 0] = m * use
        stats[i:i + step, 1] = total * use + (1 - use)
        if gradient is not None:
            up = s["upstream"].double().expand(rows)[i:i + step]
            d = ln_q.exp()
            d.scatter_add_(1, j.clamp(min=0), -p)
            gradient[i:i + step] = d * (up * w * any_ * t)[:, None]
    if case["mode"] == "backward":
        return {"loss": None, "stats": None, "gradient": gradient}
    return {"loss": loss, "stats": stats, "gradient": gradient}


def _norm_exact(case, seed):
    s = _norm_inputs(case, seed)
    n, p, c = s["x"].shape
    g = case["groups"]
    d = c // g
    x = s["x"].double().reshape(n, p, g, d).transpose(1, 2).reshape(n, g, p * d)
    var, mean = torch.var_mean(x, dim=2, correction=0)
    r = (var + _EPS).rsqrt()

    def spread(v):  # [n, g, p * d] -> [n, p, c]
        return v.reshape(n, g, p, d).transpose(1, 2).reshape(n, p, c)

    w = torch.ones(c, dtype=torch.float64, device="cuda") if s["weight"] is None else s["weight"].double()
    b = torch.zeros(c, dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"].double()
    if case["mode"] == "backward":  # the statistics that the call is given, as they were rounded
        wide = torch.float64 if s["x"].dtype == torch.float64 else torch.float32
        given = _norm_forward_plain(case, s)[1]
        mean, r = given[..., 0].to(wide).double(), given[..., 1].to(wide).double()
    h = (x - mean[..., None]) * r[..., None]
    z = spread(h) * w + b
    act = case["act"]
    if act == "none":
        y, slope = z, torch.ones_like(z)
    elif act == "relu":
        y, slope = z.clamp(min=0), (z > 0).double()
    elif act == "silu":
        q = torch.sigmoid(z)
        y, slope = z * q, q + z * q * (1 - q)
    else:
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        y, slope = z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if case["mode"] == "forward":
        return [y, torch.stack([mean, r], dim=2)]
    dz = s["dy"].double() * slope
    dw, db = (dz * spread(h)).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    k = (dz * w).reshape(n, p, g, d).transpose(1, 2).reshape(n, g, p * d)
    dx = r[..., None] * (k - k.mean(dim=2, keepdim=True) - h * (k * h).mean(dim=2, keepdim=True))
    if s["weight"] is None:
        dw = db = None
    return [spread(dx), dw, db]


def _power(e):
    """2^e for whole e, exactly (a power function on the device is not)."""
    return (e.to(torch.int64) + 1023 << 52).view(torch.float64)


def _e4m3(v):
    """The nearest value of 4 exponent and 3 fraction bits (ties to even), as a 64-bit value."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30)))
    e = torch.where(_power(e) > v.abs(), e - 1, e)
    e = torch.where(_power(e + 1) <= v.abs(), e + 1, e)
    step = _power(e.clamp(min=-6.0) - 3)
    return torch.round(v / step) * step


def _block_exact(case, seed):
    s = _block_inputs(case, seed)
    m, k = s["x"].shape
    high = 1 if case["mode"] == "product" else 128
    x = s["x"].double()
    full = torch.nn.functional.pad(x, (0, -k % 128, 0, -m % high)).unflatten(1, (-1, 128)).unflatten(0, (-1, high))
    amax = full.abs().amax(dim=3).amax(dim=1)
    power = torch.ceil(torch.log2(torch.where(amax > 0, amax / 448, 1.0)))
    for _ in range(2):  # log2's own rounding next to a power of two
        at = _power(power)
        power = torch.where(at * 448 < amax, power + 1, torch.where(at * 224 >= amax, power - 1, power))
    scales = torch.where(amax > 0, _power(power.clamp(min=-126)), 1.0)
    wide = scales.repeat_interleave(high, 0)[:m].repeat_interleave(128, 1)[:, :k]
    codes = _e4m3(x / wide)
    if case["mode"] == "weights":
        return [codes, scales]
    w = s["w"].double() * s["w_scales"].double().repeat_interleave(128, 0)[:case["columns"]].repeat_interleave(128, 1)[:, :k]
    return [(codes * wide) @ w.t(), codes, scales]


def exact(case, seed):
    return {"distill": _distill_exact, "norm": _norm_exact, "block": _block_exact}[case["op"]](case, seed)
