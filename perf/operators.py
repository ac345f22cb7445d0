"""Operators of gated recurrent blocks: the gated scan, the block norm and the linear layer with 4-bit weights.

A case is a dict of plain values; ``kind`` names the operator and its direction:

  scan       h_t = a_t h_{t-1} + u_t over a sequence, from a carried state; a = sigmoid(gate) or the gate itself,
             u = (1 - a) x ("leaky") or x
  scan_train the same forward pass and then its gradients from the gradient of h
  norm       r' = r + alpha * s * act(gate) * rms_norm(y), z = rms_norm(r'): the norm behind one block, its gate and
             residual scale, and the norm in front of the next block
  norm_bwd   its gradients
  w4         y = x W^T + b with 4-bit weights, a scale (and a zero point) for each group along K

``run`` computes the plain form in elementary torch operations in 32 bits, or, with ``own`` set, calls the framework.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6


def listed():
    return [
        # decode: one token for each of 16 users, the gate and the input are halves of one projection
        dict(name="scan_step_b16_bf16", kind="scan", dtype="bf16", T=1, B=16, D=2048, gate="sigmoid", leaky=True,
             batch_first=True, ragged=False, carry=True),
        # prefill or training forward of one layer, a batch of eight sequences
        dict(name="scan_t2048_b8_bf16", kind="scan", dtype="bf16", T=2048, B=8, D=2048, gate="sigmoid", leaky=True,
             batch_first=True, ragged=False, carry=False),
        # one long document, a chunk of it with the state of the chunk before
        dict(name="scan_t32768_b1_fp16", kind="scan", dtype="fp16", T=32768, B=1, D=1024, gate="sigmoid", leaky=True,
             batch_first=True, ragged=False, carry=True),
        # a padded batch of odd sizes in the framework's own order (time outermost), ready-made decays
        dict(name="scan_ragged_t1031_fp32", kind="scan", dtype="fp32", T=1031, B=6, D=1001, gate="value", leaky=False,
             batch_first=False, ragged=True, carry=True),
        # training: forward and backward pass of the second case
        dict(name="scan_train_t2048_b8_bf16", kind="scan_train", dtype="bf16", T=2048, B=8, D=2048, gate="sigmoid",
             leaky=True, batch_first=True, ragged=False, carry=False),
        # decode: norm, gate and residual between two blocks for four users
        dict(name="norm_m4_bf16", kind="norm", dtype="bf16", M=4, D=4096, gate="silu", post=True, pre=True),
        # the same in training, 16384 tokens
        dict(name="norm_m16384_bf16", kind="norm", dtype="bf16", M=16384, D=2048, gate="silu", post=True, pre=True),
        # and its backward pass
        dict(name="norm_bwd_m16384_bf16", kind="norm_bwd", dtype="bf16", M=16384, D=2048, gate="silu", post=True,
             pre=True),
        # a small model trained in fp32, odd width
        dict(name="norm_bwd_m1023_fp32", kind="norm_bwd", dtype="fp32", M=1023, D=1001, gate="sigmoid", post=True,
             pre=True),
        # the 512 -> 1000 classifier of the ResNet-18 with 4-bit weights, one image
        dict(name="w4_m1_512_1000_fp16", kind="w4", dtype="fp16", M=1, K=512, N=1000, G=64, zeros=False, bias=True),
        # decode: a square projection for one user
        dict(name="w4_m1_4096_bf16", kind="w4", dtype="bf16", M=1, K=4096, N=4096, G=128, zeros=False, bias=False),
        # decode: the widest projection of a block for 16 users, zero points
        dict(name="w4_m16_8192_bf16", kind="w4", dtype="bf16", M=16, K=8192, N=16384, G=128, zeros=True, bias=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    kind = rng.choice(["scan", "scan", "scan_train", "norm", "norm_bwd", "w4", "w4"])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind in ("scan", "scan_train"):
        c["T"] = _log_int(rng, 1, 32768 if kind == "scan" else 8192)
        c["B"] = _log_int(rng, 1, 64)
        c["D"] = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            c["D"] = (c["D"] + 7) // 8 * 8
        c["gate"] = rng.choice(["sigmoid", "sigmoid", "value"])
        c["leaky"] = rng.random() < 0.6
        c["batch_first"] = rng.random() < 0.7
        c["ragged"] = c["B"] > 1 and rng.random() < 0.3
        c["carry"] = rng.random() < 0.5
    elif kind in ("norm", "norm_bwd"):
        c["M"] = _log_int(rng, 1, 32768)
        c["D"] = _log_int(rng, 128, 16384)
        if rng.random() < 0.6:
            c["D"] = (c["D"] + 7) // 8 * 8
        c["gate"] = rng.choice(["none", "sigmoid", "silu", "silu"])
        c["post"] = rng.random() < 0.8
        c["pre"] = rng.random() < 0.8
    else:
        c["G"] = rng.choice([32, 64, 128])
        c["M"] = _log_int(rng, 1, 64)
        c["K"] = 32 * _log_int(rng, 4, 512)     # the last group may be a short one
        c["N"] = _log_int(rng, 64, 32768)
        c["zeros"] = rng.random() < 0.5
        c["bias"] = rng.random() < 0.5
    return c


def draw(rng):
    """One more case of the same ranges that costs no more than the largest listed one of its kind."""
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["kind"], (0, 0))
        most[c["kind"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= most[c["kind"]][0] and w["flops"] <= most[c["kind"]][1]:
            return c


# ------------------------------------------------------------------------------------------------ inputs ----
def _steps(case):
    """Valid steps of each sequence of a padded batch: from none to all."""
    T, B = case["T"], case["B"]
    if not case["ragged"]:
        return [T] * B
    return [T * i // (B - 1) for i in range(B)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device=dev) * std + mean).to(dtype)

    s = dict(case=case)
    if case["kind"] in ("scan", "scan_train"):
        T, B, D = case["T"], case["B"], case["D"]
        lead = (B, T) if case["batch_first"] else (T, B)
        if case["gate"] == "sigmoid":       # input and gate logits are the two halves of one projection's rows
            proj = normal(*lead, 2 * D)
            proj[..., D:].mul_(1.5).add_(2.0)   # most gates between 0.5 and 0.99
            s["x"], s["g"] = proj[..., :D], proj[..., D:]
        else:
            s["x"] = normal(*lead, D)
            s["g"] = torch.sigmoid(normal(*lead, D, std=1.5, mean=2.0, dtype=torch.float32)).to(dt)
        s["h0"] = normal(B, D, std=0.5, dtype=torch.float32) if case["carry"] else None
        s["lengths"] = None
        if case["ragged"]:
            steps = torch.tensor(_steps(case), device=dev, dtype=torch.int32)
            s["lengths"] = steps[torch.randperm(B, generator=gen, device=dev)].contiguous()
        if case["kind"] == "scan_train":
            s["dh"] = normal(*lead, D)
            s["dh_last"] = normal(B, D, dtype=torch.float32) if case["carry"] else None
    elif case["kind"] in ("norm", "norm_bwd"):
        M, D = case["M"], case["D"]
        s["y"] = normal(M, D, std=2.0)
        s["gate"] = normal(M, D) if case["gate"] != "none" else None
        s["r"] = normal(M, D, std=3.0)
        s["w_post"] = normal(D, std=0.2, mean=1.0) if case["post"] else None
        s["scale"] = normal(D, std=0.05, mean=0.3)
        s["w_pre"] = normal(D, std=0.2, mean=1.0) if case["pre"] else None
        if case["kind"] == "norm_bwd":
            s["dr"] = normal(M, D)
            s["dz"] = normal(M, D) if case["pre"] else None
    else:
        M, K, N, G = case["M"], case["K"], case["N"], case["G"]
        groups = -(-K // G)
        s["x"] = normal(M, K)
        s["q"] = torch.randint(0, 256, (N, K // 2), generator=gen, device=dev, dtype=torch.uint8)
        s["scales"] = (torch.rand(N, groups, generator=gen, device=dev) * 0.01 + 0.005).to(dt)
        s["zeros"] = (torch.randint(0, 16, (N, groups), generator=gen, device=dev, dtype=torch.uint8)
                      if case["zeros"] else None)
        s["bias"] = normal(N) if case["bias"] else None
    return s


# ------------------------------------------------------------------------------------------- plain forms ----
def _gates(s):
    """a, 1 - a, the input u of each step and which steps count, time outermost."""
    case = s["case"]
    x, g = s["x"].float(), s["g"].float()
    if case["batch_first"]:
        x, g = x.transpose(0, 1), g.transpose(0, 1)
    if case["gate"] == "sigmoid":
        e = torch.exp(-g.abs())
        big, small = 1 / (1 + e), e / (1 + e)
        a, b = torch.where(g >= 0, big, small), torch.where(g >= 0, small, big)
    else:
        a, b = g, 1 - g
    u = b * x if case["leaky"] else x
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(case["T"], device=x.device)[:, None] < s["lengths"][None, :])[..., None]
        a, u = torch.where(live, a, 1.0), torch.where(live, u, 0.0)
    return x, a, b, u, live


def _states(a, u, h0):
    """All h_t = a_t h_{t-1} + u_t, time outermost: the span that each step's (product, sum) covers doubles."""
    if h0 is not None:
        u = torch.cat([(u[0] + a[0] * h0)[None], u[1:]])
    span = 1
    while span < a.shape[0]:
        u = torch.cat([u[:span], u[span:] + a[span:] * u[:-span]])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return u


def _order(case, t, dt):
    return (t.transpose(0, 1) if case["batch_first"] else t).to(dt).contiguous()


def _scan(s):
    case = s["case"]
    x, a, b, u, live = _gates(s)
    hs = _states(a, u, s["h0"])
    last = hs[-1].clone()
    if live is not None:
        hs = torch.where(live, hs, 0.0)
    return _order(case, hs, DTYPES[case["dtype"]]), last


def _scan_train(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    x, a, b, u, live = _gates(s)
    hs = _states(a, u, s["h0"])
    first = torch.zeros_like(u[0]) if s["h0"] is None else s["h0"]
    before = torch.cat([first[None], hs[:-1]])
    dh = s["dh"].float()
    dh = dh.transpose(0, 1) if case["batch_first"] else dh
    if live is not None:
        dh = torch.where(live, dh, 0.0)
    # lam_t = dh_t + a_{t+1} lam_{t+1}: the same recurrence from the end
    lams = _states(torch.cat([torch.ones_like(first)[None], a.flip(0)[:-1]]), dh.flip(0), s["dh_last"]).flip(0)
    dx = b * lams if case["leaky"] else lams
    dg = lams * (before - x if case["leaky"] else before)
    if case["gate"] == "sigmoid":
        dg = dg * a * b
    if live is not None:
        dx, dg = torch.where(live, dx, 0.0), torch.where(live, dg, 0.0)
        hs = torch.where(live, hs, 0.0)
    return _order(case, hs, dt), _order(case, dx, dt), _order(case, dg, dt), a[0] * lams[0]


def _act(kind, gate):
    """The gate's activation and its derivative."""
    if kind == "none":
        return None, None
    g = gate.float()
    p = 1 / (1 + torch.exp(-g))
    if kind == "sigmoid":
        return p, p * (1 - p)
    return g * p, p * (1 + g * (1 - p))


def _rstd(v):
    return torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)


def _norm_parts(s):
    case = s["case"]
    y, r = s["y"].float(), s["r"].float()
    act, dact = _act(case["gate"], s["gate"])
    n = y * _rstd(y) if case["post"] else y
    coef = s["scale"].float() * (s["w_post"].float() if case["post"] else 1.0)
    inner = n if act is None else n * act
    return y, r, act, dact, n, coef, r + coef * inner, inner


def _norm(s):
    dt = DTYPES[s["case"]["dtype"]]
    out = _norm_parts(s)[6]
    z = out * _rstd(out) * s["w_pre"].float() if s["case"]["pre"] else None
    return out.to(dt), None if z is None else z.to(dt)


def _norm_grad(v, dn):
    """Gradient of v * rstd(v) for the gradient dn of its result."""
    r = _rstd(v)
    return r * dn - v * r ** 3 * (v * dn).mean(-1, keepdim=True)


def _norm_bwd(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    y, r, act, dact, n, coef, out, inner = _norm_parts(s)
    total, dw_pre = s["dr"].float(), None
    if case["pre"]:
        dz = s["dz"].float()
        total = total + _norm_grad(out, dz * s["w_pre"].float())
        dw_pre = (dz * out * _rstd(out)).sum(0)
    q = (total * inner).sum(0)
    dscale = q * s["w_post"].float() if case["post"] else q
    dw_post = q * s["scale"].float() if case["post"] else None
    dn = total * coef if act is None else total * coef * act
    dy = _norm_grad(y, dn) if case["post"] else dn
    dgate = None if act is None else (total * coef * n * dact).to(dt)
    return dy.to(dt), dgate, total.to(dt), dw_post, dscale, dw_pre


def _weights(s, dtype):
    case = s["case"]
    q = torch.stack([s["q"] & 15, s["q"] >> 4], -1).reshape(case["N"], case["K"]).to(dtype)
    group = torch.arange(case["K"], device=q.device) // case["G"]
    zero = 8.0 if s["zeros"] is None else s["zeros"].to(dtype)[:, group]
    return (q - zero) * s["scales"].to(dtype)[:, group]


def _w4(s):
    y = s["x"].float() @ _weights(s, torch.float32).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


_PLAIN = {"scan": _scan, "scan_train": _scan_train, "norm": _norm, "norm_bwd": _norm_bwd, "w4": _w4}


def _own(s):
    case = s["case"]
    if case["kind"] in ("scan", "scan_train"):
        from triton_snn_fusion_b200.runtime import temporal_gated_scan_backend as scan
        kw = dict(gate=case["gate"], leaky=case["leaky"], lengths=s["lengths"], batch_first=case["batch_first"])
        f = scan.run_temporal_gated_scan(s["x"], s["g"], s["h0"], save_for_backward=case["kind"] == "scan_train", **kw)
        if case["kind"] == "scan":
            return f.h_seq, f.h_last
        r = scan.run_temporal_gated_scan_backward(s["dh"], s["x"], s["g"], s["h0"], f.ckpt, dh_last=s["dh_last"], **kw)
        return f.h_seq, r.dx, r.dgate, r.dh_init
    if case["kind"] in ("norm", "norm_bwd"):
        from triton_snn_fusion_b200.runtime import block_norm_backend as norm
        kw = dict(gate=s["gate"], residual=s["r"], w_post=s["w_post"], res_scale=s["scale"], w_pre=s["w_pre"],
                  gate_act=case["gate"], post_norm=case["post"], pre_norm=case["pre"], eps=EPS)
        if case["kind"] == "norm":
            r = norm.run_block_norm(s["y"], **kw)
            return r.res_out, r.z
        r = norm.run_block_norm_backward(s["dr"], s["dz"], s["y"], **kw)
        return r.dy, r.dgate, r.dresidual, r.dw_post, r.dres_scale, r.dw_pre
    from triton_snn_fusion_b200.runtime import linear_w4_backend as w4
    return w4.run_linear_w4(s["x"], s["q"], s["scales"], s["zeros"], s["bias"], group_size=case["G"])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


# -------------------------------------------------------------------------------------------------- work ----
def work(case):
    sz = SIZE[case["dtype"]]
    if case["kind"] in ("scan", "scan_train"):
        T, B, D = case["T"], case["B"], case["D"]
        live, n = sum(_steps(case)) * D, T * B * D
        state = 4 * B * D
        if case["kind"] == "scan":
            return {"bytes": sz * (2 * live + n) + state * (2 if case["carry"] else 1), "flops": 8 * live}
        return {"bytes": sz * (3 * live + 3 * n) + state * (3 if case["carry"] else 1), "flops": 24 * live}
    if case["kind"] in ("norm", "norm_bwd"):
        M, D = case["M"], case["D"]
        gate, pre = case["gate"] != "none", case["pre"]
        params = 1 + case["post"] + pre
        if case["kind"] == "norm":
            return {"bytes": sz * (M * D * (3 + gate + pre) + params * D), "flops": 16 * M * D}
        return {"bytes": sz * (M * D * (5 + 2 * gate + pre) + params * D) + 4 * params * D, "flops": 40 * M * D}
    M, K, N, G = case["M"], case["K"], case["N"], case["G"]
    groups = -(-K // G)
    return {"bytes": N * K // 2 + N * groups * (sz + case["zeros"]) + sz * (M * K + M * N + N * case["bias"]),
            "flops": 2 * M * N * K}


# ----------------------------------------------------------------------------------- 64-bit definitions ----
def _walk(a, u, h):
    """h_t = a_t h_{t-1} + u_t step by step."""
    out = torch.empty_like(u)
    for t in range(a.shape[0]):
        h = torch.addcmul(u[t], a[t], h)
        out[t] = h
    return out


def _exact_scan(case, s, backward):
    T, B = case["T"], case["B"]
    flip = (lambda t: t.transpose(0, 1)) if case["batch_first"] else (lambda t: t)
    x, g = flip(s["x"].double()), flip(s["g"].double())
    a = torch.sigmoid(g) if case["gate"] == "sigmoid" else g.clone()
    one_less = torch.sigmoid(-g) if case["gate"] == "sigmoid" else 1 - g
    u = x * one_less if case["leaky"] else x.clone()
    steps = torch.full((B,), T, device=x.device) if s["lengths"] is None else s["lengths"].long()
    pad = torch.arange(T, device=x.device).view(T, 1, 1) >= steps.view(1, B, 1)
    a = a.masked_fill(pad, 1.0)
    u = u.masked_fill(pad, 0.0)
    h0 = torch.zeros_like(u[0]) if s["h0"] is None else s["h0"].double()
    h = _walk(a, u, h0)
    seq = flip(h.masked_fill(pad, 0.0))
    if not backward:
        return seq, h[-1]
    prev = torch.cat((h0[None], h[:-1]))
    dh = flip(s["dh"].double()).masked_fill(pad, 0.0)
    end = torch.zeros_like(h0) if s["dh_last"] is None else s["dh_last"].double()
    after = torch.cat((a[1:], torch.ones_like(a[:1])))      # lam_t = a_{t+1} lam_{t+1} + dh_t
    lam = _walk(after.flip(0), dh.flip(0), end).flip(0)
    dx = (lam * one_less if case["leaky"] else lam).masked_fill(pad, 0.0)
    da = lam * (prev - x if case["leaky"] else prev)
    dg = (da * torch.sigmoid(g) * one_less if case["gate"] == "sigmoid" else da).masked_fill(pad, 0.0)
    return seq, flip(dx), flip(dg), a[0] * lam[0]


def _exact_norm(case, s, backward):
    names = ["y", "gate", "r", "w_post", "scale", "w_pre"]
    v = {k: None if s[k] is None else s[k].double().requires_grad_(backward) for k in names}
    D = case["D"]

    def rms(t):
        return t / torch.sqrt(t.pow(2).sum(-1, keepdim=True) / D + EPS)

    n = rms(v["y"]) * v["w_post"] if case["post"] else v["y"]
    if case["gate"] == "sigmoid":
        n = n * torch.sigmoid(v["gate"])
    elif case["gate"] == "silu":
        n = n * v["gate"] * torch.sigmoid(v["gate"])
    out = v["r"] + v["scale"] * n
    z = rms(out) * v["w_pre"] if case["pre"] else None
    if not backward:
        return out, z
    total = (out * s["dr"].double()).sum()
    if z is not None:
        total = total + (z * s["dz"].double()).sum()
    have = [k for k in names if v[k] is not None]
    got = dict(zip(have, torch.autograd.grad(total, [v[k] for k in have])))
    return tuple(got.get(k) for k in names)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("scan", "scan_train"):
        return _exact_scan(case, s, case["kind"] == "scan_train")
    if case["kind"] in ("norm", "norm_bwd"):
        return _exact_norm(case, s, case["kind"] == "norm_bwd")
    low, high = s["q"].bitwise_and(15).double(), s["q"].bitwise_right_shift(4).double()
    full = torch.empty(case["N"], case["K"], dtype=torch.float64, device=low.device)
    full[:, 0::2], full[:, 1::2] = low, high
    out = torch.zeros(case["M"], case["N"], dtype=torch.float64, device=low.device)
    for k in range(s["scales"].shape[1]):
        cut = slice(k * case["G"], min((k + 1) * case["G"], case["K"]))
        zero = 8.0 if s["zeros"] is None else s["zeros"][:, k:k + 1].double()
        out += s["x"][:, cut].double() @ ((full[:, cut] - zero) * s["scales"][:, k:k + 1].double()).t()
    return out if s["bias"] is None else out + s["bias"].double()
