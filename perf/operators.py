"""Cases of the 4-bit linear layer (forward, input gradient) and of the top-logit distillation loss (with its gradient).

`run` computes a case either in elementary torch operations (`own` false) or through graphite_amd (`own` true);
`exact` computes it in 64 bits, from the definitions, independently of both.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _w4(name, op, n, k, m, group, dtype, zeros, bias=False, relu=False):
    return dict(name=name, op=op, n=n, k=k, m=m, group=group, dtype=dtype, zeros=zeros, bias=bias, relu=relu)


def _kd(name, n, v, top, dtype, rest, tau, shared=False):
    return dict(name=name, op="distill", n=n, v=v, top=top, dtype=dtype, rest=rest, tau=tau, shared=shared)


def listed():
    return [
        # one query of the victim: its first linear layer (2048 -> 1024), where the time is latency
        _w4("forward_f32_one_query", "forward", 1, 2048, 1024, 64, "f32", True, bias=True, relu=True),
        # one evaluation of a candidate mask: a hundred transformed images through the same layer
        _w4("forward_f32_hundred", "forward", 100, 2048, 1024, 64, "f32", True, bias=True, relu=True),
        # one chunk of a scoring call (8192 images per chunk is the framework's default)
        _w4("forward_f32_chunk", "forward", 8192, 2048, 1024, 64, "f32", True, bias=True, relu=True),
        # a wide layer for a single row in a 16-bit type: bound by the weights' bytes
        _w4("forward_bf16_one_row_wide", "forward", 1, 8192, 8192, 128, "bf16", True),
        # a handful of rows, no dimension a multiple of anything
        _w4("forward_f16_few_rows_odd", "forward", 7, 5001, 4999, 32, "f16", False, bias=True),
        # a large batch in bf16: bound by the matrix units
        _w4("forward_bf16_batch", "forward", 4096, 4096, 4096, 128, "bf16", True),
        # the whitebox step: gradients of a hundred transformed images through the 2048 -> 1024 layer
        _w4("gradient_f32_hundred", "gradient", 100, 2048, 1024, 64, "f32", True),
        # the same direction for a large batch in bf16
        _w4("gradient_bf16_batch", "gradient", 2048, 4096, 4096, 128, "bf16", True),
        # the whitebox step's loss: a hundred images, 43 classes, one teacher answer of five scores for all of them
        _kd("distill_f32_hundred", 100, 43, 5, "f32", True, 2.0, shared=True),
        # a thousand classes in half precision, the teacher's ten best
        _kd("distill_f16_thousand_classes", 1000, 1000, 10, "f16", False, 1.0),
        # wide rows in bf16, sixty-four teacher logits and the mass of the others
        _kd("distill_bf16_wide", 4096, 32768, 64, "bf16", True, 1.5),
        # few very wide odd rows in 32 bits
        _kd("distill_f32_widest_odd", 515, 100003, 32, "f32", True, 1.0),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["forward", "forward", "gradient", "distill", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "distill":
        v = _log(rng, 2, 131072)
        n = _log(rng, 1, max(1, min(8192, 50_000_000 // v)))
        return dict(op="distill", n=n, v=v, top=rng.randint(1, min(128, v)), dtype=dtype, rest=rng.random() < 0.5,
                    tau=rng.choice([0.5, 1.0, 1.5, 2.0, 4.0]), shared=rng.random() < 0.25)
    k, m = _log(rng, 33, 8192), _log(rng, 10, 8192)
    n = _log(rng, 1, max(1, min(8192, 30_000_000_000 // (k * m))))
    return dict(op=kind, n=n, k=k, m=m, group=rng.choice([32, 64, 128, 256]), dtype=dtype, zeros=rng.random() < 0.6,
                bias=kind == "forward" and rng.random() < 0.5, relu=kind == "forward" and rng.random() < 0.5)


def work(case):
    e = SIZE[case["dtype"]]
    n = case["n"]
    if case["op"] == "distill":
        t = 1 if case["shared"] else n
        return {"bytes": 2 * n * case["v"] * e + 4 * n + t * case["top"] * 12 + (4 * t if case["rest"] else 0),
                "flops": 6 * n * case["v"]}
    k, m = case["k"], case["m"]
    groups = -(-k // case["group"])
    weights = m * (-(-k // 2)) + m * groups * (e + (1 if case["zeros"] else 0)) + (4 * m if case["bias"] else 0)
    return {"bytes": weights + n * (k + m) * e, "flops": 2 * n * m * k}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _quantise(w, group, zeros, dtype):
    """Round-to-nearest 4-bit weights of w [m,k]: (packed [m, ceil(k/2)] uint8, scales [m,groups], zeros [m,groups])."""
    m, k = w.shape
    groups = -(-k // group)
    pad = torch.zeros((m, groups * group), device=w.device)
    pad[:, :k] = w
    g = pad.view(m, groups, group)
    if zeros:
        lo, hi = g.amin(2).clamp(max=0.0), g.amax(2).clamp(min=0.0)
        s = ((hi - lo) / 15.0).clamp(min=1e-8).to(dtype)
        z = torch.round(-lo / s.float()).clamp(0, 15)
    else:
        s = (g.abs().amax(2) / 7.0).clamp(min=1e-8).to(dtype)
        z = torch.full_like(s, 8.0, dtype=torch.float32)
    q = (torch.round(g / s.float()[:, :, None]) + z[:, :, None]).clamp(0, 15).to(torch.uint8).view(m, -1)
    if q.shape[1] % 2:
        q = torch.nn.functional.pad(q, (0, 1))
    packed = (q[:, 0::2] | (q[:, 1::2] << 4))[:, :(k + 1) // 2].contiguous()
    if k % 2:
        packed[:, -1] &= 15
    return packed, s, (z.to(torch.uint8) if zeros else None)


def _make(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dt = DT[case["dtype"]]
    n = case["n"]
    if case["op"] == "distill":
        v, top = case["v"], case["top"]
        rows = 1 if case["shared"] else n
        z = randn(n, v) * 2.5
        t = (z[:rows] * 0.7 + randn(rows, v) * 1.8).contiguous()
        val, idx = torch.topk(t, top, dim=1)
        lse = torch.logsumexp(t / case["tau"], dim=1) if case["rest"] else None
        gl = torch.rand(n, generator=g, device="cuda") * (2.0 / n)
        return dict(z=z.to(dt), idx=idx, top=val, lse=lse, gl=gl)
    k, m = case["k"], case["m"]
    w = randn(m, k) * (1.0 / math.sqrt(k))
    q, s, z = _quantise(w, case["group"], case["zeros"], dt)
    if case["op"] == "forward":
        x = randn(n, k)
        if case["relu"]:
            x = torch.relu(x)                       # what a rectified layer hands on
        x = x.to(dt)
    else:
        x = (randn(n, m) / n).to(dt)
    return dict(q=q, s=s, z=z, x=x, b=randn(m) * 0.1 if case["bias"] else None)


def prepare(case, seed):
    st = _make(case, seed)
    st["case"] = case
    if own and case["op"] != "distill":
        from graphite_amd.linear_w4 import LinearW4
        st["layer"] = LinearW4(st["q"], st["s"], st["z"], bias=st["b"], group=case["group"], in_features=case["k"],
                               input_grad=case["op"] == "gradient")
    return st


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _weights32(st, case):
    """[m,k] f32 weights of the packed ones."""
    q, k = st["q"], case["k"]
    nib = torch.stack((q & 15, q >> 4), dim=2).view(q.shape[0], -1)[:, :k].float()
    z = st["z"].float() if st["z"] is not None else torch.full_like(st["s"], 8.0, dtype=torch.float32)
    grp = torch.arange(k, device=q.device) // case["group"]
    return (nib - z[:, grp]) * st["s"].float()[:, grp]


def _distill32(st, case):
    tau = case["tau"]
    u = st["z"].float() / tau
    e = torch.exp(u - u.amax(1, keepdim=True))
    lse = u.amax(1) + torch.log(e.sum(1))
    q = e / e.sum(1, keepdim=True)
    n = u.shape[0]
    # the teacher's side in 64 bits: what its named classes leave over is a difference next to zero
    idx, t = st["idx"].expand(n, -1), st["top"].expand(n, -1).double() / tau
    lq = u.gather(1, idx) - lse[:, None]
    if case["rest"]:
        p = torch.exp(t - st["lse"][:, None].double())
        pr = (1.0 - p.sum(1)).clamp(min=0.0).float()
        p = p.float()
        other = torch.ones_like(q).scatter_(1, idx, 0.0)
        qr = (q * other).sum(1)
        live = (pr > 0) & (qr > 0)
        ratio = torch.where(live, pr / torch.where(live, qr, torch.ones_like(qr)), torch.zeros_like(pr))
        # no mass and no class left over: nothing to add
        tail = torch.where(live, pr * torch.log(torch.where(live, ratio, torch.ones_like(ratio))), torch.zeros_like(pr))
        grad = q - q * other * ratio[:, None]
    else:
        p = torch.exp(t - t.amax(1, keepdim=True))
        p = (p / p.sum(1, keepdim=True)).float()
        tail = torch.zeros_like(lse)
        grad = q
    lp = torch.where(p > 0, torch.log(torch.where(p > 0, p, torch.ones_like(p))), torch.zeros_like(p))
    loss = tau * tau * ((p * (lp - lq)).sum(1) + tail)
    grad = grad.scatter_add(1, idx, -p) * (tau * st["gl"])[:, None]
    return loss, grad.to(st["z"].dtype)


def run(state):
    case = state["case"]
    if case["op"] == "distill":
        if own:
            from graphite_amd.distill import topk_distill
            return topk_distill(state["z"], state["idx"], state["top"], tau=case["tau"], teacher_lse=state["lse"],
                                grad_loss=state["gl"])
        return _distill32(state, case)
    if own:
        if case["op"] == "forward":
            return state["layer"].forward(state["x"], relu=case["relu"])
        return state["layer"].input_grad(state["x"])
    w = _weights32(state, case)
    x = state["x"].float()
    if case["op"] == "gradient":
        return torch.matmul(x, w).to(state["x"].dtype)
    y = torch.matmul(x, w.t())
    if state["b"] is not None:
        y = y + state["b"]
    if case["relu"]:
        y = torch.clamp(y, min=0.0)
    return y.to(state["x"].dtype)


# ------------------------------------------------------------------------------------------------
# 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_distill(st, case):
    tau, n = case["tau"], case["n"]
    losses, grads = [], []
    rows = max(1, 16_000_000 // case["v"])
    for r0 in range(0, n, rows):
        u = st["z"][r0:r0 + rows].double() / tau
        c = u.shape[0]
        shared = st["idx"].shape[0] == 1
        idx = st["idx"].expand(c, -1) if shared else st["idx"][r0:r0 + rows]
        t = (st["top"].expand(c, -1) if shared else st["top"][r0:r0 + rows]).double() / tau
        log_q = u - torch.logsumexp(u, dim=1, keepdim=True)
        target = torch.zeros_like(u)
        named = torch.zeros_like(u, dtype=torch.bool).scatter_(1, idx, True)
        if case["rest"]:
            lse = (st["lse"].expand(c) if shared else st["lse"][r0:r0 + rows]).double()
            target.scatter_(1, idx, torch.exp(t - lse[:, None]))
        else:
            target.scatter_(1, idx, torch.softmax(t, dim=1))
        loss = torch.special.xlogy(target, target).sum(1) - (target * log_q).sum(1)
        if case["rest"]:
            rest = (1.0 - target.sum(1)).clamp(min=0.0)
            log_qr = torch.logsumexp(log_q.masked_fill(named, -math.inf), dim=1)
            none = torch.isinf(log_qr) | (rest == 0)
            loss = loss + torch.where(none, torch.zeros_like(rest), torch.special.xlogy(rest, rest) - rest * log_qr)
            inner = torch.exp(log_q - torch.where(none, torch.zeros_like(rest), log_qr)[:, None])
            share = torch.where(named, torch.zeros_like(u), inner * torch.where(none, torch.zeros_like(rest), rest)[:, None])
            target = target + share
        losses.append(tau * tau * loss)
        grads.append((torch.exp(log_q) - target) * (tau * st["gl"][r0:r0 + rows].double())[:, None])
    return torch.cat(losses), torch.cat(grads)


def exact(case, seed):
    st = _make(case, seed)
    if case["op"] == "distill":
        return _exact_distill(st, case)
    k, group = case["k"], case["group"]
    m = case["m"]
    codes = torch.zeros((m, 2 * st["q"].shape[1]), dtype=torch.float64, device=st["q"].device)
    codes[:, 0::2] = (st["q"] % 16).double()
    codes[:, 1::2] = torch.div(st["q"], 16, rounding_mode="floor").double()
    w = torch.empty((m, k), dtype=torch.float64, device=codes.device)
    for g in range(-(-k // group)):
        a, b = g * group, min(k, (g + 1) * group)
        zero = st["z"][:, g:g + 1].double() if st["z"] is not None else 8.0
        w[:, a:b] = (codes[:, a:b] - zero) * st["s"][:, g:g + 1].double()
    x = st["x"].double()
    if case["op"] == "gradient":
        return torch.matmul(x, w)
    y = torch.matmul(x, w.t())
    if st["b"] is not None:
        y = y + st["b"].double()
    return torch.relu(y) if case["relu"] else y
