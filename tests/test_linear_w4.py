"""The linear layer with 4-bit weights against the 64-bit oracle; each value within its counted error."""
import pytest
import torch

from oracle import recurrent_oracle as orc
from triton_snn_fusion_b200 import _lib
from triton_snn_fusion_b200.runtime import linear_w4_backend as ops

DEV = "cuda"
gpu = pytest.mark.gpu


def _inputs(M, K, N, G, dtype, zeros=True, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // G)
    x = torch.randn(M, K, generator=g).to(dtype)
    q = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(N, groups, generator=g) * 0.01 + 0.005).to(dtype)
    z = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(N, generator=g).to(dtype) if bias else None
    return x, q, s, z, b


def _dev(t):
    return None if t is None else t.to(DEV)


def _check(M, K, N, G, dtype, **kw):
    x, q, s, z, b = _inputs(M, K, N, G, dtype, **kw)
    y = ops.run_linear_w4(_dev(x), _dev(q), _dev(s), _dev(z), _dev(b), group_size=G)
    ref, err = orc.linear_w4(x, q, s, z, b, G)
    orc.assert_within(y, ref, err, f"M={M} K={K} N={N} G={G}")
    return y


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("K", [32, 64, 96, 160, 512, 544, 1056, 4096])
def test_depths_groups_and_types(dtype, G, K):
    _check(1, K, 48, G, dtype, seed=K)
    _check(5, K, 33, G, dtype, zeros=False, bias=False, seed=K + 1)


@gpu
@pytest.mark.parametrize("M", [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 64, 65, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_counts(M, dtype):
    _check(M, 416, 70, 64, dtype, seed=M)


@gpu
@pytest.mark.parametrize("N", [1, 2, 7, 8, 15, 16, 17, 31, 100, 1000, 5001])
def test_widths(N):
    _check(1, 512, N, 128, torch.float16, seed=N)
    _check(9, 96, N, 64, torch.bfloat16, seed=N)


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 16384, 64), (16, 8192, 512), (3, 2048, 4096), (1, 4096, 20000), (32, 12288, 80)])
def test_larger_layers(M, K, N):
    for dtype in (torch.bfloat16, torch.float32):
        _check(M, K, N, 128, dtype)


@gpu
def test_every_weight_value_and_zero_point():
    """One weight at a time: x is a unit vector, so each output is one weight times its scale, exactly."""
    K, N, G = 64, 16 * 16, 32
    q = torch.arange(16, dtype=torch.uint8).repeat(N // 16)[:, None].expand(N, K)
    q = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
    z = torch.arange(16, dtype=torch.uint8).repeat_interleave(16)[:, None].expand(N, 2).contiguous()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        s = torch.full((N, 2), 0.25, dtype=dtype)
        x = torch.zeros(K, K, dtype=dtype)
        x.fill_diagonal_(1)
        y = ops.run_linear_w4(_dev(x), _dev(q), _dev(s), _dev(z), group_size=G).cpu()
        assert torch.equal(y.double(), orc.unpack_w4(q, s, z, G).t())
    # zero points up to 127 are numbers like any other
    z = torch.full((N, 2), 100, dtype=torch.uint8)
    y = ops.run_linear_w4(_dev(x), _dev(q), _dev(s), _dev(z), group_size=G).cpu()
    assert torch.equal(y.double(), orc.unpack_w4(q, s, z, G).t())


@gpu
def test_position_of_each_weight():
    """Random weights against unit vectors: every (n, k) must land on its own x."""
    K, N, G = 288, 40, 128
    _, q, s, z, _ = _inputs(1, K, N, G, torch.float16)
    for dtype in (torch.float16, torch.float32):
        x = torch.eye(K).to(dtype)
        s2 = torch.full_like(s, 0.5).to(dtype)
        y = ops.run_linear_w4(_dev(x), _dev(q), _dev(s2), _dev(z), group_size=G).cpu()
        assert torch.equal(y.double(), orc.unpack_w4(q, s2, z, G).t())


@gpu
def test_strided_tokens_leading_dimensions_and_out():
    B, T, K, N, G = 2, 3, 128, 24, 64
    x, q, s, z, b = _inputs(B * T, K, N, G, torch.bfloat16)
    ref, err = orc.linear_w4(x, q, s, z, b, G)
    for off in (0, 1, 8):
        wide = torch.full((B, T, K + off + 2), float("nan"), dtype=torch.bfloat16, device=DEV)
        v = wide[..., off:off + K]
        v.copy_(x.view(B, T, K))
        y = ops.run_linear_w4(v, _dev(q), _dev(s), _dev(z), _dev(b), group_size=G)
        assert y.shape == (B, T, N)
        orc.assert_within(y.reshape(-1, N), ref, err)
    out = torch.empty(B * T, N, dtype=torch.bfloat16, device=DEV)
    assert ops.run_linear_w4(_dev(x), _dev(q), _dev(s), _dev(z), _dev(b), group_size=G, out=out) is out
    orc.assert_within(out, ref, err)
    q8 = torch.zeros(N * K // 2 + 8, dtype=torch.uint8, device=DEV)[8:].view(N, K // 2)      # not 16-byte aligned: copied
    q8.copy_(q)
    orc.assert_within(ops.run_linear_w4(_dev(x), q8, _dev(s), _dev(z), _dev(b), group_size=G), ref, err)
    assert ops.run_linear_w4(torch.empty(0, K, device=DEV).bfloat16(), _dev(q), _dev(s), group_size=G).shape == (0, N)


@gpu
def test_a_bad_token_stays_alone():
    x, q, s, z, b = (_dev(t) for t in _inputs(12, 512, 64, 128, torch.bfloat16))
    a = ops.run_linear_w4(x, q, s, z, b)
    for bad in (float("nan"), float("inf")):
        x2 = x.clone()
        x2[4, 100] = bad
        c = ops.run_linear_w4(x2, q, s, z, b)
        keep = torch.arange(12, device=DEV) != 4
        assert torch.equal(a[keep], c[keep]) and not bool(torch.isfinite(c[4]).any())


@gpu
def test_fp32_tokens_keep_their_bits():
    """fp32 tokens of very different sizes: each is widened as a whole, not rounded to 16 bits on the way."""
    K, N, G = 256, 32, 64
    x, q, s, z, b = _inputs(3, K, N, G, torch.float32)
    x *= torch.logspace(-20, 20, K)
    y = ops.run_linear_w4(_dev(x), _dev(q), _dev(s), _dev(z), _dev(b), group_size=G)
    ref, err = orc.linear_w4(x, q, s, z, b, G)
    orc.assert_within(y, ref, err)


@gpu
def test_results_repeat_also_in_a_graph():
    x, q, s, z, b = (_dev(t) for t in _inputs(4, 2048, 640, 128, torch.bfloat16))
    a = ops.run_linear_w4(x, q, s, z, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = ops.run_linear_w4(x, q, s, z, b)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, c)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantized_weights_are_the_nearest(symmetric, dtype):
    """Each weight within half a step of what it is read back as (the zero point of an asymmetric group is rounded, which
    moves its ends by at most another half; 2^-8 for the scale's own rounding to 16 bits)."""
    g = torch.Generator().manual_seed(0)
    w = torch.randn(20, 160, generator=g).to(dtype)
    w[3] = 0
    w[4, :128] = 0.5
    for G in (32, 64, 128):
        r = ops.quantize_linear_w4(w, G, symmetric)
        assert r.q_weight.shape == (20, 80) and r.scales.shape == (20, -(-160 // G)) and r.scales.dtype == dtype
        back = orc.unpack_w4(r.q_weight, r.scales, r.zeros, G)
        step = r.scales.double()[:, torch.arange(160) // G]
        assert bool(((back - w.double()).abs() <= step * (0.5 if symmetric else 1.0) + 15 * 2.0 ** -8 * step).all())
        assert not bool(back[3].any())
    with pytest.raises(RuntimeError, match="unsupported_shape"):
        ops.quantize_linear_w4(torch.zeros(4, 33))


def test_c_refusals():
    base = dict(x=4096, xs=64, q=8192, s=12288, z=None, b=None, y=16384, ys=32, M=2, K=64, N=32, G=32, dt=1, stream=None)
    for kw, code, text in ((dict(K=48), 2, "multiple of 32"), (dict(G=16), 1, "groups"), (dict(q=8200), 1, "aligned"),
                           (dict(x=None), 1, "null pointer"), (dict(ys=31), 1, "stride"), (dict(xs=-1), 1, "stride"),
                           (dict(N=0), 1, "positive"), (dict(dt=3), 1, "dtype"), (dict(M=-1), 1, "positive")):
        a = dict(base, **kw)
        st = _lib.lib.snnb_linear_w4(*a.values())
        assert st == code and text in _lib.lib.snnb_last_error().decode(), (kw, st, _lib.lib.snnb_last_error())


def test_refusals_name_their_reason():
    x, q, s = torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 2)
    for args, kw, text in (((x, q, s), dict(group_size=32), "unsupported_device"), ((x, q, s), dict(group_size=16), "unsupported_group"),
                           ((x[:, :48], q, s), dict(group_size=32), "unsupported_shape"),
                           ((x, q[:, :31], s), dict(group_size=32), "unsupported_shape"),
                           ((x, q.int(), s), dict(group_size=32), "unsupported_dtype"),
                           ((x, q, s.half()), dict(group_size=32), "unsupported_dtype"),
                           ((x, q, s, torch.zeros(8, 2)), dict(group_size=32), "unsupported_dtype"),
                           ((x, q, s, None, torch.zeros(9)), dict(group_size=32), "unsupported_shape"),
                           ((x, q[:0], s[:0]), dict(group_size=32), "no rows"), (([x], q, s), {}, "expected a Tensor")):
        with pytest.raises(RuntimeError, match=text):
            ops.run_linear_w4(*args, **kw)


def test_sizes_whose_offsets_would_wrap_are_refused():
    """A row of 2^31 - 32 weights: the step behind its last one has no 32-bit number. The addresses are never read."""
    for K in (2 ** 31 - 32, 2 ** 30 + 32):
        assert _lib.lib.snnb_linear_w4(4096, K, 4096, 4096, None, None, 8192, 1, 1, K, 1, 128, _lib.F32, None) == 1
        assert b"too large" in _lib.lib.snnb_last_error()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 12, 40])
def test_infinite_tokens(dtype, M):
    """An infinite value gives infinities of the weight's sign, and no number only where that weight is zero."""
    K, N, G = 256, 40, 64
    x, q, s, z, b = _inputs(M, K, N, G, dtype)
    for k, v in ((100, float("inf")), (255, -float("inf")), (0, float("inf"))):
        x2 = x.clone()
        x2[M // 2, k] = v
        y = ops.run_linear_w4(_dev(x2), _dev(q), _dev(s), _dev(z), _dev(b), group_size=G)[M // 2].double().cpu()
        weight = (q[:, k // 2] >> (4 * (k % 2)) & 15).double() - z[:, k // G].double()
        want = weight * v
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(nan=0.0, posinf=2, neginf=-2), want.nan_to_num(nan=0.0, posinf=2, neginf=-2))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 12, 40])
def test_large_zero_points(dtype, M):
    """Zero points up to 127 are numbers like any other, in each type. A larger one is outside what is documented: fp16 still
    has its value, the other types have no number for it and answer NaN in its rows alone."""
    K, N, G = 256, 70, 64
    x, q, s, _, b = _inputs(M, K, N, G, dtype)
    zs = torch.tensor([0, 15, 16, 63, 64, 100, 126, 127], dtype=torch.uint8)
    z = zs[(torch.arange(N)[:, None] + 3 * torch.arange(K // G)) % 8].contiguous()
    ref, err = orc.linear_w4(x, q, s, z, b, G)
    y = ops.run_linear_w4(_dev(x), _dev(q), _dev(s), _dev(z), _dev(b), group_size=G)
    orc.assert_within(y, ref, err)
    z[5, 1], z[40, 3] = 128, 255
    ref, err = orc.linear_w4(x, q, s, z, b, G)
    y2 = ops.run_linear_w4(_dev(x), _dev(q), _dev(s), _dev(z), _dev(b), group_size=G)
    if dtype == torch.float16:
        orc.assert_within(y2, ref, err)
    else:
        assert bool(y2[:, [5, 40]].isnan().all())
        keep = [n for n in range(N) if n not in (5, 40)]
        assert torch.equal(y2[:, keep], y[:, keep])


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 6e-7), (torch.float16, 2e-7), (torch.float16, 4e-6), (torch.float16, 6e4),
                                        (torch.bfloat16, 3e38), (torch.float32, 3e38), (torch.float32, 1e-44)])
def test_quantized_weights_at_the_ends_of_the_types(symmetric, dtype, size):
    """Groups so small that their scale is a subnormal number, which rounds by up to half of itself, and groups as wide as the
    type: each weight within half a step of what it is read back as (a whole one with a rounded zero point; 2^-8 of the widest
    weight, 15 steps, for the scale's rounding), and the step no wider than a seventh (fifteenth) of the group or the type's
    smallest number, whichever is more, up to that rounding."""
    G = 32
    w = ((torch.rand(6, 64, generator=torch.Generator().manual_seed(1)) * 2 - 1) * size).to(dtype)
    r = ops.quantize_linear_w4(w, G, symmetric)
    assert bool(torch.isfinite(r.scales).all())
    step = r.scales.double()[:, torch.arange(64) // G]
    back = orc.unpack_w4(r.q_weight, r.scales, r.zeros, G)
    assert bool(((back - w.double()).abs() <= step * ((0.5 if symmetric else 1.0) + 15 * 2.0 ** -8)).all())
    g = w.double().view(6, 2, G)
    exact = g.abs().amax(-1) / 7 if symmetric else (g.amax(-1).clamp(min=0) - g.amin(-1).clamp(max=0)) / 15
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert bool((r.scales.double() <= exact * (1 + 2.0 ** -8) + tiny).all())


def test_quantizing_a_parameter_keeps_no_graph():
    """The 4-bit weights of a model's parameter are plain tensors: they must not hold the full weight through autograd."""
    w = torch.nn.Parameter(torch.randn(8, 64, generator=torch.Generator().manual_seed(0)))
    for symmetric in (True, False):
        r = ops.quantize_linear_w4(w, 32, symmetric)
        plain = ops.quantize_linear_w4(w.detach(), 32, symmetric)
        for a, b in zip(r, plain):
            assert (a is None) == (b is None)
            if a is not None:
                assert not a.requires_grad and a.grad_fn is None and torch.equal(a, b)


def test_quantizer_refusals_name_their_reason():
    w = torch.randn(4, 64, generator=torch.Generator().manual_seed(0))
    bad = w.clone()
    bad[1, 3] = float("nan")
    wide = w.clone()
    wide[2, 60] = -float("inf")
    for args, text in ((([1.0],), "expected a Tensor"), ((w[0],), "dimensions"), ((w.double(),), "unsupported_dtype"),
                       ((w, 48), "unsupported_shape"), ((w, 64.0), "unsupported_shape"), ((w, "64"), "unsupported_shape"),
                       ((w[:, :40],), "unsupported_shape"), ((w[:, :0],), "unsupported_shape"),
                       ((bad, 32), "unsupported_value"), ((wide, 32, False), "unsupported_value")):
        with pytest.raises(RuntimeError, match=text):
            ops.quantize_linear_w4(*args)


def test_group_sizes_and_outputs_of_other_kinds_are_refused():
    x, q, s = torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1)
    for group in (64.0, "64", None, [64]):
        with pytest.raises(RuntimeError, match="unsupported_group_size"):
            ops.run_linear_w4(x, q, s, group_size=group)


@gpu
def test_outputs_that_are_no_tensors_are_refused():
    x, q, s, _, _ = (_dev(t) for t in _inputs(2, 64, 8, 64, torch.float32, zeros=False, bias=False))
    for out in ([[0.0] * 8] * 2, 1.0):
        with pytest.raises(RuntimeError, match="unsupported_output"):
            ops.run_linear_w4(x, q, s, group_size=64, out=out)


@gpu
def test_the_microbenchmark_rotates_weights_that_fit_the_cache(capsys):
    from triton_snn_fusion_b200 import microbench
    microbench.main(["w4", "--M", "2", "--K", "4096", "--N", "8192"])       # 16.8 MB of weights: 25 of them are 400 MB
    assert "(25 rotating weights)" in capsys.readouterr().out


def test_a_group_size_may_be_any_whole_number_type():
    import numpy as np
    w = torch.randn(4, 64, generator=torch.Generator().manual_seed(0))
    assert all(torch.equal(a, b) for a, b in zip(ops.quantize_linear_w4(w, np.int64(32), False), ops.quantize_linear_w4(w, 32, False)))
    with pytest.raises(RuntimeError, match="unsupported_device"):       # and nothing else
        ops.run_linear_w4(w, *ops.quantize_linear_w4(w, 32), group_size=np.int32(32))
