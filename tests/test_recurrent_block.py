"""The gated-block operators together, as a model runs them: a training step and a decoding loop of one block, each
against the same block in 64 bits."""
import pytest
import torch

from oracle import recurrent_oracle as orc

DEV = "cuda"
pytestmark = pytest.mark.gpu


def _params(D, H, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, std=1.0, mean=0.0: torch.randn(*s, generator=g) * std + mean  # noqa: E731
    return dict(w_pre=rnd(D, std=0.1, mean=1.0), w_in=rnd(3 * H, D, std=D ** -0.5), w_out=rnd(D, H, std=H ** -0.5),
                w_post=rnd(D, std=0.1, mean=1.0), scale=rnd(D, std=0.05, mean=0.5), w_next=rnd(D, std=0.1, mean=1.0))


def _reference(p, x, h0):
    """x [B,T,D] fp64 with gradients -> residual stream and normed input of the next block, and the state."""
    rms = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    u = (rms(x) * p["w_pre"]) @ p["w_in"].t()
    v, f, o = u.chunk(3, -1)
    a = torch.sigmoid(f)
    h, hs = h0, []
    for t in range(x.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * v[:, t]
        hs.append(h)
    y = torch.stack(hs, 1) @ p["w_out"].t()
    gate = o[..., :x.shape[-1]]
    res = x + p["scale"] * (gate * torch.sigmoid(gate)) * (rms(y) * p["w_post"])
    return res, rms(res) * p["w_next"], h


def test_training_step_of_a_block():
    """Forward and backward of norm -> projection -> scan -> projection -> norm, gate, residual, norm in fp32, every
    product of the projections a plain matmul. Tolerance: the scan's bound is under 1e-5 of a state's scale over 150 steps,
    a matmul of K = 96 products adds 96 * 2^-24, the norms 2^-16: 2e-4 of each tensor's largest value covers their chain."""
    from triton_snn_fusion_b200.runtime.block_norm_backend import run_block_norm, run_block_norm_backward
    from triton_snn_fusion_b200.runtime.temporal_gated_scan_backend import run_temporal_gated_scan, run_temporal_gated_scan_backward

    B, T, D, H = 3, 150, 96, 96
    p64 = {k: v.double().requires_grad_() for k, v in _params(D, H).items()}
    g = torch.Generator().manual_seed(1)
    x64 = torch.randn(B, T, D, generator=g).double().requires_grad_()
    h64 = torch.randn(B, H, generator=g).double().requires_grad_()
    res, z, last = _reference(p64, x64, h64)
    dres, dz, dlast = (torch.randn(t.shape, generator=g).double() for t in (res, z, last))
    names = list(p64)
    want = torch.autograd.grad((res * dres).sum() + (z * dz).sum() + (last * dlast).sum(), [x64, h64] + [p64[k] for k in names])

    p = {k: v.detach().float().to(DEV) for k, v in p64.items()}
    x, h0, dres, dz, dlast = (t.detach().float().to(DEV) for t in (x64, h64, dres, dz, dlast))
    norm = run_block_norm(None, residual=x, w_pre=p["w_pre"], post_norm=False)
    u = norm.z @ p["w_in"].t()
    v, f, o = u[..., :H], u[..., H:2 * H], u[..., 2 * H:]       # views: rows of the projection
    s = run_temporal_gated_scan(v, f, h0, batch_first=True, save_for_backward=True)
    y = s.h_seq @ p["w_out"].t()
    kw = dict(gate=o, residual=x, w_post=p["w_post"], res_scale=p["scale"], w_pre=p["w_next"], gate_act="silu")
    out = run_block_norm(y, **kw)

    gb = run_block_norm_backward(dres, dz, y, **kw)
    dy2 = gb.dy.reshape(-1, D)
    gs = run_temporal_gated_scan_backward((gb.dy @ p["w_out"]), v, f, h0, s.ckpt, dh_last=dlast, batch_first=True)
    du = torch.cat([gs.dx, gs.dgate, gb.dgate], -1)
    gn = run_block_norm_backward(gb.dresidual, du @ p["w_in"], None, residual=x, w_pre=p["w_pre"], post_norm=False)
    got = [gn.dresidual, gs.dh_init, gn.dw_pre, du.reshape(-1, 3 * H).t() @ norm.z.reshape(-1, D),
           dy2.t() @ s.h_seq.reshape(-1, H), gb.dw_post, gb.dres_scale, gb.dw_pre]
    for name, a, b in zip(["res", "z", "state", "dx", "dh0"] + ["d" + k for k in names],
                          [out.res_out, out.z, s.h_last] + got, [res, z, last] + list(want)):
        b = b.detach()
        worst = float((a.double().cpu() - b).abs().max() / b.abs().max())
        assert worst <= 2e-4, (name, worst)


def test_decoding_with_4_bit_projections_captured_once():
    """Tokens one by one with 4-bit projections, the state updated in place, the step captured into a graph and replayed:
    the same numbers as the calls one by one, and as the whole sequence in one call of each operator (bf16; the orders of
    the scan's sums differ, so that one is held to the rounding of its bf16 tensors, 2^-8, through a block)."""
    from triton_snn_fusion_b200.runtime.block_norm_backend import run_block_norm
    from triton_snn_fusion_b200.runtime.linear_w4_backend import quantize_linear_w4, run_linear_w4
    from triton_snn_fusion_b200.runtime.temporal_gated_scan_backend import run_temporal_gated_scan

    B, T, D, H = 2, 12, 128, 128
    p = {k: v.to(DEV).bfloat16() for k, v in _params(D, H).items()}
    q_in, q_out = quantize_linear_w4(p["w_in"], 64), quantize_linear_w4(p["w_out"], 64, symmetric=False)
    x = torch.randn(B, T, D, generator=torch.Generator().manual_seed(2)).to(DEV).bfloat16()

    def block(xt, state, **scan):
        z = run_block_norm(None, residual=xt, w_pre=p["w_pre"], post_norm=False).z
        u = run_linear_w4(z, *q_in, group_size=64)
        s = run_temporal_gated_scan(u[..., :H], u[..., H:2 * H], state, batch_first=True, **scan)
        y = run_linear_w4(s.h_seq, *q_out, group_size=64)
        return run_block_norm(y, gate=u[..., 2 * H:], residual=xt, w_post=p["w_post"], res_scale=p["scale"], w_pre=p["w_next"],
                              gate_act="silu").z

    state = torch.zeros(B, H, device=DEV)
    eager = torch.cat([block(x[:, t:t + 1], state, h_last_out=state) for t in range(T)], 1)
    token, state2 = x[:, :1].clone(), torch.zeros(B, H, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(token, state2, h_last_out=state2)
    state2.zero_()
    steps = []
    for t in range(T):
        token.copy_(x[:, t:t + 1])
        graph.replay()
        steps.append(out.clone())
    assert torch.equal(torch.cat(steps, 1), eager) and torch.equal(state2, state)
    whole = block(x, torch.zeros(B, H, device=DEV))
    assert float((whole.float() - eager.float()).abs().max()) <= 4 * 2.0 ** -8 * float(eager.float().abs().max())
    assert orc.half_step(torch.bfloat16) == 2.0 ** -8
