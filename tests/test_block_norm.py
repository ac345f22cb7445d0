"""The norms around a block and their gradients against the 64-bit oracle; each value within its counted error."""
import pytest
import torch

from oracle import recurrent_oracle as orc
from triton_snn_fusion_b200 import _lib
from triton_snn_fusion_b200.runtime import block_norm_backend as ops

DEV = "cuda"
gpu = pytest.mark.gpu


def _inputs(M, D, dtype, act="silu", post=True, pre=True, y=True, res=True, scale=True, w_dtype=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, std=1.0, mean=0.0, dt=dtype: (torch.randn(*s, generator=g) * std + mean).to(dt)  # noqa: E731
    w_dtype = w_dtype or dtype
    return dict(
        y=rnd(M, D, std=2.0) if y else None,
        gate=rnd(M, D).clamp(-8, 8) if y and act != "none" else None,
        residual=rnd(M, D, std=3.0) if res else None,
        w_post=rnd(D, std=0.2, mean=1.0, dt=w_dtype) if y and post else None,
        res_scale=rnd(D, std=0.05, mean=0.3, dt=w_dtype) if y and scale else None,
        w_pre=rnd(D, std=0.2, mean=1.0, dt=w_dtype) if pre else None), rnd(M, D), rnd(M, D)


def _dev(t):
    return None if t is None else t.to(DEV)


def _check(M, D, dtype, act="silu", post=True, pre=True, y=True, alpha=1.0, eps=1e-6, has_dro=True, has_dz=True, **kw):
    v, dro, dz = _inputs(M, D, dtype, act, post, pre, y, **kw)
    post, act = post and y, act if y else "none"
    opt = dict(gate_act=act, alpha=alpha, post_norm=post, pre_norm=pre, eps=eps)
    par = (v["y"], v["gate"], v["residual"], v["w_post"], v["res_scale"], v["w_pre"], act, post)
    dv = {k: _dev(t) for k, t in v.items()}
    dy = dv.pop("y")
    f = ops.run_block_norm(dy, **dv, **opt)
    ref, err, _ = orc.block_norm(*par, pre, alpha, eps)
    assert (f.z is None) == (not pre) and (f.res_out is None) == (not y)
    if y:
        orc.assert_within(f.res_out, ref["res_out"], err["res_out"], "res_out")
    if pre:
        orc.assert_within(f.z, ref["z"], err["z"], "z")
    dro, dz = dro if has_dro else None, dz if pre and has_dz else None
    r = ops.run_block_norm_backward(_dev(dro), _dev(dz), dy, **dv, **opt)
    ref, err = orc.block_norm_backward(dro, dz, *par, pre, alpha, eps)
    have = dict(dy=v["y"], dgate=v["gate"], dresidual=1, dw_post=v["w_post"], dres_scale=v["res_scale"], dw_pre=v["w_pre"])
    for name, of in have.items():
        got = getattr(r, name)
        assert (got is None) == (of is None), name
        if got is not None and name in ref:
            orc.assert_within(got, ref[name], err[name], name)
        elif got is not None:
            assert not bool(got.any()), name
    return f, r


@gpu
@pytest.mark.parametrize("D", [1, 2, 7, 8, 31, 64, 100, 256, 257, 1000, 1001, 2048, 2056, 4096, 5000, 8192, 16384, 16383])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_widths_and_types(D, dtype):
    _check(5, D, dtype, seed=D)


@gpu
@pytest.mark.parametrize("M,D", [(1, 64), (2, 512), (3, 4096), (149, 96), (593, 128), (700, 2048), (2500, 72), (5001, 33)])
def test_row_counts(M, D):
    _check(M, D, torch.bfloat16, seed=M)


@gpu
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("res", [True, False])
def test_forms(act, post, pre, res):
    for dtype in (torch.float32, torch.bfloat16):
        for D in (136, 333):
            _check(40, D, dtype, act, post, pre, res=res, alpha=0.7)


@gpu
def test_optional_parameters_and_gradients():
    for dtype in (torch.float32, torch.float16):
        _check(33, 200, dtype, scale=False)
        _check(33, 200, dtype, w_dtype=torch.float32)
        _check(33, 200, dtype, has_dz=False)
        _check(33, 200, dtype, has_dro=False)
        _check(33, 200, dtype, y=False)                 # the norm in front of the first block
        _check(33, 200, dtype, y=False, has_dro=False)


@gpu
def test_rows_of_zeros_and_large_values():
    M, D = 6, 512
    for dtype in (torch.float32, torch.bfloat16):
        v, dro, dz = _inputs(M, D, dtype)
        v["y"][0] = 0
        v["residual"][0] = 0
        v["y"][1] = 0
        v["y"][2] *= 2.0 ** 40
        v["residual"][3] *= 2.0 ** 40
        v["y"][4] *= 2.0 ** -40
        dv = {k: _dev(t) for k, t in v.items()}
        y = dv.pop("y")
        par = (v["y"], v["gate"], v["residual"], v["w_post"], v["res_scale"], v["w_pre"], "silu", True)
        f = ops.run_block_norm(y, **dv, gate_act="silu")
        ref, err, _ = orc.block_norm(*par, True, 1.0, 1e-6)
        orc.assert_within(f.res_out, ref["res_out"], err["res_out"], "res_out")
        orc.assert_within(f.z, ref["z"], err["z"], "z")
        r = ops.run_block_norm_backward(_dev(dro), _dev(dz), y, **dv, gate_act="silu")
        ref, err = orc.block_norm_backward(dro, dz, *par, True, 1.0, 1e-6)
        for n in ("dy", "dgate", "dresidual"):
            got = getattr(r, n)
            keep = [0, 1, 2, 3, 5]      # row 4: y is lost beside eps in its norm; its gradient is checked alone
            orc.assert_within(got[keep], ref[n][keep], err[n][keep], n)
            orc.assert_within(got[4:5], ref[n][4:5], err[n][4:5], n)


@gpu
def test_gate_logits_at_the_ends_of_their_type():
    M, D = 4, 256
    for dtype in (torch.float32, torch.bfloat16):
        v, dro, dz = _inputs(M, D, dtype)
        low = torch.finfo(dtype).min
        v["gate"][0] = low
        v["gate"][1] = -200.0
        v["gate"][2] = 200.0
        dv = {k: _dev(t) for k, t in v.items()}
        y = dv.pop("y")
        for act in ("sigmoid", "silu"):
            f = ops.run_block_norm(y, **dv, gate_act=act)
            r = ops.run_block_norm_backward(_dev(dro), _dev(dz), y, **dv, gate_act=act)
            # closed gates: the block adds nothing and takes no gradient
            assert torch.equal(f.res_out[:2].cpu(), v["residual"][:2])
            assert not bool(r.dgate[:2].any()) and not bool(r.dy[:2].any())
            for t in (*f, *r):
                assert bool(torch.isfinite(t).all())


@gpu
def test_a_bad_row_stays_alone():
    M, D = 300, 96
    v, dro, dz = _inputs(M, D, torch.bfloat16)
    dv = {k: _dev(t) for k, t in v.items()}
    y = dv.pop("y")
    a, ga = ops.run_block_norm(y, **dv, gate_act="silu"), ops.run_block_norm_backward(_dev(dro), _dev(dz), y, **dv, gate_act="silu")
    y2 = y.clone()
    y2[77, 3] = float("nan")
    b, gb = ops.run_block_norm(y2, **dv, gate_act="silu"), ops.run_block_norm_backward(_dev(dro), _dev(dz), y2, **dv, gate_act="silu")
    keep = torch.arange(M, device=DEV) != 77
    for p, q in zip((*a, *ga[:3]), (*b, *gb[:3])):
        assert torch.equal(p[keep], q[keep])
    assert bool(b.z[77].isnan().all())


@gpu
@pytest.mark.parametrize("off", [0, 1, 8])
def test_strided_rows_leading_dimensions_and_in_place(off):
    B, T, D = 3, 5, 72
    v, dro, dz = _inputs(B * T, D, torch.bfloat16)
    wide = torch.zeros(B, T, 2 * D + off, dtype=torch.bfloat16, device=DEV)
    yv, gv = wide[..., off:off + D], wide[..., off + D:]
    yv.copy_(v["y"].view(B, T, D))
    gv.copy_(v["gate"].view(B, T, D))
    par = (v["y"], v["gate"], v["residual"], v["w_post"], v["res_scale"], v["w_pre"], "silu", True)
    ref, err, _ = orc.block_norm(*par, True, 1.0, 1e-6)
    w = dict(w_post=_dev(v["w_post"]), res_scale=_dev(v["res_scale"]), w_pre=_dev(v["w_pre"]), gate_act="silu")
    r = _dev(v["residual"]).view(B, T, D)
    rt = r.transpose(0, 1).contiguous().transpose(0, 1)      # batch inside time: rows without a common stride
    f = ops.run_block_norm(yv, gate=gv, residual=rt, **w)
    assert f.z.shape == (B, T, D) and f.z.is_contiguous()
    orc.assert_within(f.z.reshape(-1, D), ref["z"], err["z"])
    g = ops.run_block_norm_backward(_dev(dro).view(B, T, D), _dev(dz).view(B, T, D), yv, gate=gv, residual=rt, **w)
    gref, gerr = orc.block_norm_backward(dro, dz, *par, True, 1.0, 1e-6)
    for n in ("dy", "dgate", "dresidual"):
        orc.assert_within(getattr(g, n).reshape(-1, D), gref[n], gerr[n], n)
    keep = r.clone()
    f2 = ops.run_block_norm(yv, gate=gv, residual=keep, res_inplace=True, **w)
    assert f2.res_out is keep and torch.equal(keep, f.res_out) and torch.equal(f2.z, f.z)


@gpu
def test_no_rows():
    D = 16
    e = torch.empty(0, D, device=DEV)
    one = torch.ones(D, device=DEV)
    f = ops.run_block_norm(e, gate=e, residual=e, w_post=one, res_scale=one, w_pre=one, gate_act="silu")
    assert f.z.shape == (0, D)
    r = ops.run_block_norm_backward(e, e, e, gate=e, residual=e, w_post=one, res_scale=one, w_pre=one, gate_act="silu")
    assert all(not bool(t.any()) for t in (r.dw_post, r.dres_scale, r.dw_pre))


@gpu
def test_results_repeat_and_graphs_do_not_share_a_workspace():
    M, D = 1200, 1024
    sets = []
    for seed in (1, 2):
        v, dro, dz = _inputs(M, D, torch.bfloat16, seed=seed)
        dv = {k: _dev(t) for k, t in v.items()}
        sets.append((_dev(dro), _dev(dz), dv.pop("y"), dv))
    run = lambda s: ops.run_block_norm_backward(*s[:3], **s[3], gate_act="silu")  # noqa: E731
    first = [run(s) for s in sets]
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(s)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):      # both graphs in flight at the same time
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for want, (_, got) in zip(first, graphs):
        assert all(torch.equal(p, q) for p, q in zip(want, got))


@gpu
def test_more_than_2_to_32_bytes():
    """One row repeated 132000 times (4.3 GB a result): each row comes out as the first; the parameters' gradients are that
    row's times the number of rows, to within a rounding a row added in fp32 (at most 132040 units of 2^-24)."""
    M, D = 132000, 16384
    v, dro, dz = _inputs(1, D, torch.bfloat16)
    dv = {k: _dev(t) for k, t in v.items()}
    rows = lambda t: _dev(t).expand(M, D)  # noqa: E731
    w = dict(w_post=dv["w_post"], res_scale=dv["res_scale"], w_pre=dv["w_pre"], gate_act="silu")
    one = ops.run_block_norm(dv["y"], gate=dv["gate"], residual=dv["residual"], **w)
    f = ops.run_block_norm(rows(v["y"]), gate=rows(v["gate"]), residual=rows(v["residual"]), **w)
    for m in (0, M // 2, M - 1):
        assert torch.equal(f.z[m], one.z[0]) and torch.equal(f.res_out[m], one.res_out[0])
    del f
    one = ops.run_block_norm_backward(_dev(dro), _dev(dz), dv["y"], gate=dv["gate"], residual=dv["residual"], **w)
    r = ops.run_block_norm_backward(rows(dro), rows(dz), rows(v["y"]), gate=rows(v["gate"]), residual=rows(v["residual"]), **w)
    for m in (0, M // 2, M - 1):
        assert torch.equal(r.dy[m], one.dy[0]) and torch.equal(r.dgate[m], one.dgate[0]) and torch.equal(r.dresidual[m], one.dresidual[0])
    for a, b in zip(r[3:], one[3:]):
        assert bool(((a.double() - M * b.double()).abs() <= (M + 40) * 2.0 ** -24 * M * b.double().abs()).all())


@gpu
def test_gradients_against_differences():
    """Central differences of the forward pass for J = sum(dres_out * res_out) + sum(dz * z): step 2^-6, fp32."""
    v, dro, dz = _inputs(7, 64, torch.float32)
    dv = {k: _dev(t) for k, t in v.items()}
    dro, dz = _dev(dro), _dev(dz)
    y = dv["y"]
    grads = ops.run_block_norm_backward(dro, dz, y, gate_act="silu", **{k: t for k, t in dv.items() if k != "y"})

    def J(d):
        f = ops.run_block_norm(d["y"], gate_act="silu", **{k: t for k, t in d.items() if k != "y"})
        return float((f.res_out.double() * dro.double()).sum() + (f.z.double() * dz.double()).sum())

    g = torch.Generator(device=DEV).manual_seed(1)
    for k, grad in zip(("y", "gate", "residual", "w_post", "res_scale", "w_pre"), grads):
        d = torch.randn(dv[k].shape, generator=g, device=DEV)
        e = 2.0 ** -6
        slope = (J({**dv, k: dv[k] + e * d}) - J({**dv, k: dv[k] - e * d})) / (2 * e)
        prod = grad.double() * d.double()
        assert abs(slope - float(prod.sum())) <= 1e-2 * float(prod.norm()), k


# ---------------------------------------------------------------------------------------------- refusals ----
def _c(fn, base, **kw):
    a = dict(base, **kw)
    return getattr(_lib.lib, fn)(*a.values()), _lib.lib.snnb_last_error().decode()


def test_c_refusals():
    base = dict(y=4096, ys=64, g=8192, gs=64, r=12288, rs=64, wp=16384, sc=20480, wr=24576, ro=28672, z=32768, M=4, D=64,
                alpha=1.0, eps=1e-6, act=2, post=1, dt=1, wdt=1, stream=None)
    for kw, code, text in ((dict(D=16385), 2, "16384"), (dict(D=0), 1, "positive"), (dict(M=-1), 1, "rows"),
                           (dict(act=0), 1, "gate"), (dict(g=None), 1, "gate"), (dict(act=3), 1, "activation"),
                           (dict(dt=3), 1, "dtype"), (dict(wdt=2), 1, "parameter dtype"), (dict(eps=-1.0), 1, "eps"),
                           (dict(y=None), 1, "belong to y"), (dict(post=0), 1, "w_post"), (dict(ro=None, z=None), 1, "neither"),
                           (dict(z=None), 1, "w_pre"), (dict(ro=12288, rs=128), 1, "in place"), (dict(gs=-1), 1, "stride"), (dict(z=28672), 1, "z shares"), (dict(z=12288), 1, "z shares"),
                           (dict(ro=4096), 1, "res_out shares")):
        st, msg = _c("snnb_block_norm", base, **kw)
        assert st == code and text in msg, (kw, st, msg)


def test_c_backward_refusals():
    base = dict(dro=4096, dos=64, dz=8192, dzs=64, y=12288, ys=64, g=16384, gs=64, r=20480, rs=64, wp=24576, sc=28672,
                wr=32768, dy=36864, dg=40960, dr=45056, dwp=49152, dsc=53248, dwr=57344, ws=65536, wb=1 << 30, M=4, D=64,
                alpha=1.0, eps=1e-6, act=2, post=1, dt=1, wdt=1, stream=None)
    for kw, text in ((dict(dro=None, dz=None), "neither"), (dict(dz=None), "w_pre without dz"), (dict(dy=None), "dy belongs"),
                     (dict(dg=None), "dgate belongs"), (dict(wb=16), "workspace too small"), (dict(ws=None), "workspace"),
                     (dict(ws=65540), "aligned"), (dict(dy=12288), "one of the inputs"), (dict(dg=45056), "one buffer")):
        st, msg = _c("snnb_block_norm_backward", base, **kw)
        assert st == 1 and text in msg, (kw, st, msg)


def test_refusals_name_their_reason():
    x = torch.zeros(4, 8)
    w = torch.ones(8)
    for a, kw, text in ((x, {}, "unsupported_device"), (x, dict(gate=x), "unsupported_gate"),
                        (x, dict(gate_act="silu"), "unsupported_gate"), (x, dict(gate_act="gelu"), "unsupported_gate"),
                        (x, dict(residual=x[:3]), "unsupported_shape"), (x, dict(residual=x.half()), "unsupported_dtype"),
                        (x, dict(w_post=w[:7]), "unsupported_shape"), (x, dict(w_post=w.half()), "unsupported_dtype"),
                        (x, dict(w_post=w, post_norm=False), "unsupported_form"),
                        (x, dict(w_pre=w, pre_norm=False), "unsupported_form"), (None, dict(residual=x), "unsupported_form"),
                        (torch.zeros(2, 16385), {}, "unsupported_shape"), (x, dict(eps=-1.0), "unsupported_eps"),
                        (x, dict(eps=float("nan")), "unsupported_eps"), (None, {}, "expected a Tensor")):
        with pytest.raises(RuntimeError, match=text):
            ops.run_block_norm(a, **kw)
    with pytest.raises(RuntimeError, match="neither dres_out nor dz"):
        ops.run_block_norm_backward(None, None, x)
    with pytest.raises(RuntimeError, match="dz is"):
        ops.run_block_norm_backward(x, x[:2], x)


@gpu
@pytest.mark.parametrize("M,D,row", [(3 * 444 * 16 + 8, 64, 8), (444 * 8 + 4, 63, 4)])
def test_rows_behind_the_last_add_nothing_to_the_parameters(M, D, row):
    """Several rows share a block, and in the last round some have none left: an infinite gradient of the row before makes an
    infinite sum in its column, not NaN."""
    v, dro, _ = _inputs(M, D, torch.bfloat16)
    dro[row, 3] = float("inf")
    r = ops.run_block_norm_backward(_dev(dro), None, _dev(v["y"]), gate=_dev(v["gate"]), residual=_dev(v["residual"]),
                                    w_post=_dev(v["w_post"]), res_scale=_dev(v["res_scale"]), gate_act="silu", pre_norm=False)
    q = float("inf") * float((v["y"][row, 3].float() * v["gate"][row, 3].float()).sign())
    for got, w in ((r.dw_post, v["res_scale"]), (r.dres_scale, v["w_post"])):
        assert float(got[3]) == q * float(w[3].float().sign())
        got[3] = 0
        assert bool(torch.isfinite(got).all())


@gpu
@pytest.mark.parametrize("M", [1, 5, 37])
@pytest.mark.parametrize("D", [8, 63, 64, 128, 200, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eps_zero_with_groups_that_have_no_row(M, D, dtype):
    """Narrow rows share a block, and with these row counts some of its groups have none: with eps = 0 the norm of such a row
    is infinite, which must not reach the parameters' gradients. No row is zero, so every value is defined."""
    for post, pre, has_dz in ((True, True, True), (True, True, False), (False, True, True), (True, False, False)):
        _, r = _check(M, D, dtype, post=post, pre=pre, has_dz=has_dz, eps=0.0, seed=M + D)
        assert all(bool(torch.isfinite(t).all()) for t in r if t is not None)


def test_activations_and_eps_of_other_kinds_are_refused():
    x = torch.zeros(4, 8)
    for bad in (None, ["silu"], {}):
        with pytest.raises(RuntimeError, match="unsupported_gate"):
            ops.run_block_norm(x, gate=x, gate_act=bad)
    for bad in (None, "small", "0.5", torch.ones(2)):
        with pytest.raises(RuntimeError, match="unsupported_eps"):
            ops.run_block_norm(x, eps=bad)
        with pytest.raises(RuntimeError, match="unsupported_alpha"):
            ops.run_block_norm(x, alpha=bad)
