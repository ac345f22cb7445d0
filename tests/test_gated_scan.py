"""The gated scan and its gradients against the 64-bit oracle; each value within its counted rounding error."""
import ctypes

import pytest
import torch

from oracle import recurrent_oracle as orc
from triton_snn_fusion_b200 import _lib
from triton_snn_fusion_b200.runtime import temporal_gated_scan_backend as ops

DEV = "cuda"
gpu = pytest.mark.gpu


def _inputs(T, B, D, dtype, kind, seed=0, state=torch.float32, carry=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, B, D, generator=g).to(dtype)
    gate = (torch.randn(T, B, D, generator=g) * 1.5 + 2).clamp(-8, 8)
    gate = (gate if kind == "sigmoid" else torch.sigmoid(gate)).to(dtype)
    h0 = (torch.randn(B, D, generator=g) * 0.5).to(state) if carry else None
    dh = torch.randn(T, B, D, generator=g).to(dtype)
    dl = torch.randn(B, D, generator=g).to(state) if carry else None
    return x, gate, h0, dh, dl


def _dev(t, batch_first=False):
    if t is None:
        return None
    t = t.to(DEV)
    return t.transpose(0, 1).contiguous() if batch_first and t.dim() == 3 else t


def _check(T, B, D, dtype, kind, leaky, *, lengths=None, batch_first=False, state=torch.float32, carry=True, seed=0):
    x, gate, h0, dh, dl = _inputs(T, B, D, dtype, kind, seed, state, carry)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    kw = dict(gate=kind, leaky=leaky, batch_first=batch_first, lengths=None if n is None else n.to(DEV))
    back = (lambda t: t.transpose(0, 1)) if batch_first else (lambda t: t)
    f = ops.run_temporal_gated_scan(_dev(x, batch_first), _dev(gate, batch_first), _dev(h0), save_for_backward=True, **kw)
    h, eh, last, el = orc.gated_scan(x, gate, h0, kind, leaky, n)
    orc.assert_within(back(f.h_seq), h, eh, "h_seq")
    orc.assert_within(f.h_last, last, el, "h_last")
    assert f.h_last.dtype == (state if carry else torch.float32)
    r = ops.run_temporal_gated_scan_backward(_dev(dh, batch_first), _dev(x, batch_first), _dev(gate, batch_first), _dev(h0),
                                             f.ckpt, dh_last=_dev(dl), **kw)
    ref, err = orc.gated_scan_backward(dh, dl, x, gate, h0, kind, leaky, n)
    for name, got, want, e in zip(("dx", "dgate", "dh_init"), (back(r.dx), back(r.dgate), r.dh_init), ref, err):
        orc.assert_within(got, want, e, name)
    return f, r


@gpu
@pytest.mark.parametrize("T", [0, 1, 2, 7, 8, 9, 31, 32, 33, 127, 128, 129, 300, 1031])
@pytest.mark.parametrize("D", [64, 77])
def test_lengths_from_none_to_long(T, D):
    _check(T, 3, D, torch.float32, "sigmoid", True, seed=T)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["sigmoid", "value"])
@pytest.mark.parametrize("leaky", [True, False])
@pytest.mark.parametrize("batch_first", [True, False])
def test_types_gates_and_orders(dtype, kind, leaky, batch_first):
    for T, B, D in ((1, 5, 200), (6, 2, 333), (29, 3, 130), (261, 2, 136)):
        _check(T, B, D, dtype, kind, leaky, batch_first=batch_first, seed=T)


@gpu
@pytest.mark.parametrize("T,B,D", [(4099, 1, 64), (2500, 1, 33), (5000, 2, 264), (700, 1, 2048), (9, 1, 1), (130, 70, 1),
                                   (1, 1, 1), (1, 300, 512), (8, 40, 1000), (32, 33, 1024), (200, 2, 5000)])
def test_shapes_of_every_split(T, B, D):
    _check(T, B, D, torch.bfloat16, "sigmoid", True, batch_first=True, seed=D)


@gpu
@pytest.mark.parametrize("batch_first", [True, False])
@pytest.mark.parametrize("D", [96, 101])
def test_padded_batches(batch_first, D):
    # empty, one step, a tile's end and one behind it, all, and values that are clamped
    for T in (5, 30, 270, 1100):
        n = [0, 1, min(T, 128), min(T, 129), T, T - 1, -3, T + 7]
        f, r = _check(T, len(n), D, torch.bfloat16, "sigmoid", True, lengths=n, batch_first=batch_first, seed=T)
        for t in (f.h_seq, r.dx, r.dgate):
            t = t if batch_first else t.transpose(0, 1)
            for b, k in enumerate(n):
                assert not bool(t[b, max(0, min(k, T)):].any())


@gpu
@pytest.mark.parametrize("T", [10, 15, 16, 17, 24, 40, 63, 64, 65])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_short_tiles(T, dtype):
    """Sequences of one short tile, whole and padded, with the last channels of a tile missing and with rows that start
    anywhere."""
    n = [0, 1, 8, 9, T - 1, T, T + 3]
    for D in (200, 75):
        for kind, leaky in (("sigmoid", True), ("value", False)):
            _check(T, len(n), D, dtype, kind, leaky, lengths=n, batch_first=D == 200, seed=T)
            _check(T, 3, D, dtype, kind, leaky, batch_first=D == 75, state=dtype, seed=T + 1)


@gpu
def test_padding_is_not_read():
    T, B, D = 300, 3, 72
    n = torch.tensor([0, 17, 200], dtype=torch.int32)
    x, gate, h0, dh, dl = (t.to(DEV) for t in _inputs(T, B, D, torch.bfloat16, "sigmoid"))
    kw = dict(lengths=n.to(DEV), save_for_backward=True)
    a = ops.run_temporal_gated_scan(x, gate, h0, **kw)
    ga = ops.run_temporal_gated_scan_backward(dh, x, gate, h0, a.ckpt, dh_last=dl, lengths=n.to(DEV))
    for bad in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).min):
        x2, g2, d2 = x.clone(), gate.clone(), dh.clone()
        for b, k in enumerate(n.tolist()):
            x2[k:, b] = bad
            g2[k:, b] = bad
            d2[k:, b] = bad
        r = ops.run_temporal_gated_scan(x2, g2, h0, **kw)
        assert torch.equal(r.h_seq, a.h_seq) and torch.equal(r.h_last, a.h_last)
        gr = ops.run_temporal_gated_scan_backward(d2, x2, g2, h0, r.ckpt, dh_last=dl, lengths=n.to(DEV))
        assert all(torch.equal(p, q) for p, q in zip(gr, ga))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_state_in_the_activation_type(dtype):
    f, r = _check(200, 2, 96, dtype, "sigmoid", True, state=dtype)
    assert f.h_last.dtype == dtype and r.dh_init.dtype == dtype
    x, gate, *_ = _inputs(3, 2, 96, dtype, "sigmoid")
    assert ops.run_temporal_gated_scan(x.to(DEV), gate.to(DEV), state_dtype=dtype).h_last.dtype == dtype


@gpu
def test_zero_state_is_none_or_a_scalar():
    _check(140, 2, 40, torch.float32, "sigmoid", True, carry=False)
    x, gate, *_ = (t.to(DEV) for t in _inputs(140, 2, 40, torch.float32, "sigmoid"))
    a = ops.run_temporal_gated_scan(x, gate, None)
    b = ops.run_temporal_gated_scan(x, gate, torch.tensor(0.0, device=DEV))
    c = ops.run_temporal_gated_scan(x, gate, torch.zeros(2, 40, device=DEV))
    assert torch.equal(a.h_seq, b.h_seq) and torch.equal(a.h_seq, c.h_seq)


@gpu
def test_decoding_step_by_step_in_place_equals_one_call():
    T, B, D = 21, 4, 160
    x, gate, h0, *_ = (t.to(DEV) for t in _inputs(T, B, D, torch.bfloat16, "sigmoid"))
    state = h0.clone()
    steps = []
    for t in range(T):
        r = ops.run_temporal_gated_scan(x[t:t + 1], gate[t:t + 1], state, h_last_out=state)
        assert r.h_last is state
        steps.append(r.h_seq)
    xs, gs = x.cpu(), gate.cpu()
    h, eh, last, el = orc.gated_scan(xs, gs, h0.cpu(), "sigmoid", True)
    orc.assert_within(torch.cat(steps), h, eh)
    orc.assert_within(state, last, el)
    # a long sequence, in place as well
    x, gate, h0, *_ = _inputs(3000, 1, 512, torch.bfloat16, "sigmoid")
    state = h0.to(DEV)
    ops.run_temporal_gated_scan(x.to(DEV), gate.to(DEV), state, h_last_out=state)
    _, _, last, el = orc.gated_scan(x, gate, h0, "sigmoid", True)
    orc.assert_within(state, last, el)


@gpu
@pytest.mark.parametrize("D,off", [(64, 0), (64, 1), (72, 4), (61, 3)])
def test_rows_of_wider_tensors(D, off):
    """x and gate inside one projection, an output inside a wider buffer whose other columns stay as they were."""
    T, B = 150, 2
    for batch_first in (True, False):
        x, gate, h0, dh, dl = _inputs(T, B, D, torch.bfloat16, "sigmoid", seed=off)
        lead = (B, T) if batch_first else (T, B)
        put = (lambda t: t.transpose(0, 1)) if batch_first else (lambda t: t)
        wide = torch.zeros(*lead, 2 * D + off + 3, dtype=torch.bfloat16, device=DEV)
        xv, gv = wide[..., off:off + D], wide[..., off + D:off + 2 * D]
        xv.copy_(put(x))
        gv.copy_(put(gate))
        buf = torch.full((*lead, D + 5), 7.0, dtype=torch.bfloat16, device=DEV)
        f = ops.run_temporal_gated_scan(xv, gv, h0.to(DEV), batch_first=batch_first, h_seq_out=buf[..., 2:2 + D],
                                        save_for_backward=True)
        h, eh, *_ = orc.gated_scan(x, gate, h0, "sigmoid", True)
        orc.assert_within(put(f.h_seq), h, eh)
        assert bool((buf[..., :2] == 7).all()) and bool((buf[..., 2 + D:] == 7).all())
        wd = torch.zeros(*lead, D + off, dtype=torch.bfloat16, device=DEV)
        wd[..., off:].copy_(put(dh))
        r = ops.run_temporal_gated_scan_backward(wd[..., off:], xv, gv, h0.to(DEV), f.ckpt, batch_first=batch_first)
        ref, err = orc.gated_scan_backward(dh, None, x, gate, h0, "sigmoid", True)
        for got, want, e in zip((put(r.dx), put(r.dgate), r.dh_init), ref, err):
            orc.assert_within(got, want, e)


@gpu
def test_expanded_and_transposed_inputs():
    T, B, D = 40, 3, 48
    x, gate, h0, *_ = _inputs(T, B, D, torch.float32, "sigmoid")
    h, eh, *_ = orc.gated_scan(x[:, :1].expand(T, B, D), gate[:1].expand(T, B, D), h0, "sigmoid", True)
    f = ops.run_temporal_gated_scan(x[:, :1].to(DEV).expand(T, B, D), gate[:1].to(DEV).expand(T, B, D), h0.to(DEV))
    orc.assert_within(f.h_seq, h, eh)
    xt = x.permute(2, 0, 1).contiguous().to(DEV).permute(1, 2, 0)      # channels outermost: copied
    h, eh, *_ = orc.gated_scan(x, gate, h0, "sigmoid", True)
    orc.assert_within(ops.run_temporal_gated_scan(xt, gate.to(DEV), h0.to(DEV)).h_seq, h, eh)


@gpu
def test_closed_and_open_gates():
    """Logits at the type's ends: a closed gate drops the past, an open one keeps it."""
    T, B, D = 200, 1, 64
    x = torch.randn(T, B, D).to(torch.bfloat16).to(DEV)
    big = torch.finfo(torch.bfloat16).max
    for v in (big, float("inf")):
        f = ops.run_temporal_gated_scan(x, torch.full_like(x, -v))
        assert torch.equal(f.h_seq, x)
        h0 = torch.randn(B, D, device=DEV)
        f = ops.run_temporal_gated_scan(x, torch.full_like(x, v), h0)
        assert torch.equal(f.h_last, h0) and torch.equal(f.h_seq, h0.to(x.dtype).expand(T, B, D))


@gpu
def test_a_bad_value_stays_in_its_channel_and_its_future():
    T, B, D = 400, 2, 64
    x, gate, *_ = (t.to(DEV) if t is not None else None for t in _inputs(T, B, D, torch.float32, "sigmoid", carry=False))
    clean = ops.run_temporal_gated_scan(x, gate).h_seq
    x[137, 1, 5] = float("nan")
    h = ops.run_temporal_gated_scan(x, gate).h_seq
    assert bool(h[137:, 1, 5].isnan().all())
    h[137:, 1, 5] = clean[137:, 1, 5]
    assert torch.equal(h, clean)


@gpu
def test_results_repeat_bit_for_bit_and_in_a_graph_on_another_stream():
    x, gate, h0, dh, dl = (t.to(DEV) for t in _inputs(1500, 2, 512, torch.bfloat16, "sigmoid"))

    def both():
        f = ops.run_temporal_gated_scan(x, gate, h0, save_for_backward=True)
        return (*f, *ops.run_temporal_gated_scan_backward(dh, x, gate, h0, f.ckpt, dh_last=dl))

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        graphs.append((graph, out))
    for _ in range(2):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for got in (second, graphs[0][1], graphs[1][1]):
        assert all(torch.equal(p, q) for p, q in zip(first, got))


@gpu
def test_more_than_2_to_32_bytes():
    """A constant input and gate, never stored more than once: every state is x (1 - a^(t+1)), which is x in bf16 from step
    100 on (a <= 0.9, 0.9^100 < 2^-15). h takes 4.3 GB."""
    T, D = 33000, 65536
    x = torch.randn(1, 1, D, generator=torch.Generator().manual_seed(0)).to(DEV).bfloat16()
    gate = (torch.rand(1, 1, D, generator=torch.Generator().manual_seed(1)) * 4 - 2).to(DEV).bfloat16()
    h = ops.run_temporal_gated_scan(x.expand(T, 1, D), gate.expand(T, 1, D)).h_seq
    for t in (200, T // 2, T - 129, T - 1):
        orc.assert_within(h[t], x[0].double(), x[0].double().abs() * 2.0 ** -12)
    del h
    # the same where a row is more than 2^22 values apart from the next
    wide = torch.empty(40, 1 << 23, dtype=torch.bfloat16, device=DEV)
    xs, gs, h0, *_ = _inputs(40, 1, 64, torch.bfloat16, "sigmoid")
    wide[:, :64].copy_(xs[:, 0])
    wide[:, 1 << 22:(1 << 22) + 64].copy_(gs[:, 0])
    f = ops.run_temporal_gated_scan(wide[:, None, :64], wide[:, None, 1 << 22:(1 << 22) + 64], h0.to(DEV))
    want, err, *_ = orc.gated_scan(xs, gs, h0, "sigmoid", True)
    orc.assert_within(f.h_seq, want, err)


@gpu
def test_gradients_against_differences():
    """Central differences of the kernel's own forward pass in a random direction, for the value
    J = sum(dh * h) + sum(dh_last * h_last). With a step e the difference has the truncation error
    e^2 J'''/6 and the rounding of J / e: e = 2^-6 and fp32 states leave about 1e-3 of its scale."""
    T, B, D = 150, 2, 64
    x, gate, h0, dh, dl = (t.to(DEV) for t in _inputs(T, B, D, torch.float32, "sigmoid"))
    for leaky in (True, False):
        f = ops.run_temporal_gated_scan(x, gate, h0, leaky=leaky, save_for_backward=True)
        grads = ops.run_temporal_gated_scan_backward(dh, x, gate, h0, f.ckpt, dh_last=dl, leaky=leaky)

        def J(*a):
            r = ops.run_temporal_gated_scan(*a, leaky=leaky)
            return float((r.h_seq.double() * dh.double()).sum() + (r.h_last.double() * dl.double()).sum())

        g = torch.Generator(device=DEV).manual_seed(1)
        args = [x, gate, h0]
        for i, grad in enumerate(grads):
            v = torch.randn(args[i].shape, generator=g, device=DEV)
            e = 2.0 ** -6
            plus, minus = list(args), list(args)
            plus[i], minus[i] = args[i] + e * v, args[i] - e * v
            slope = (J(*plus) - J(*minus)) / (2 * e)
            want = float((grad.double() * v.double()).sum())
            scale = float((grad.double() * v.double()).norm())
            assert abs(slope - want) <= 1e-2 * scale, (i, slope, want, scale)


# ---------------------------------------------------------------------------------------------- refusals ----
def test_checkpoint_rows():
    rows = _lib.lib.snnb_gated_scan_ckpt_rows
    assert [rows(t) for t in (0, 1, 128, 129, 256, 257)] == [0, 0, 0, 1, 1, 2]


def _c_call(**kw):
    """snnb_gated_scan with stand-in addresses that no launch follows: every argument error is found on the host."""
    a = dict(x=4096, xt=64, xb=64, g=8192, gt=64, gb=64, h0=None, n=None, h=12288, ht=64, hb=64, hl=None, ck=None,
             T=2, B=1, D=64, kind=1, leaky=1, dt=1, sdt=0, stream=None)
    a.update(kw)
    return _lib.lib.snnb_gated_scan(*a.values()), _lib.lib.snnb_last_error().decode()


def test_c_refusals():
    for kw, text in ((dict(x=None), "null pointer"), (dict(g=None), "null pointer"), (dict(h=None), "null pointer"),
                     (dict(T=-1), "negative"), (dict(kind=2), "gate kind"), (dict(dt=3), "dtype"), (dict(sdt=2), "state dtype"),
                     (dict(xt=-64), "negative stride"), (dict(ht=32), "overlap"), (dict(B=2, hb=64, ht=64), "overlap"),
                     (dict(h0=65536, hl=65536 + 16), "overlap"), (dict(T=1 << 40), "too large"),
                     (dict(h=4096), "one of the inputs"), (dict(h=8192), "one of the inputs"),
                     (dict(T=1 << 30, B=1 << 18, D=1 << 18, hb=1 << 18, ht=1 << 36, x=None), "null pointer")):
        status, msg = _c_call(**kw)
        assert status == 1 and text in msg, (kw, status, msg)


def test_c_backward_refusals():
    base = dict(dh=4096, dht=64, dhb=64, dl=None, x=8192, xt=64, xb=64, g=12288, gt=64, gb=64, h0=None, ck=None, n=None,
                dx=16384, dxt=64, dxb=64, dg=20480, dgt=64, dgb=64, di=None, T=129, B=1, D=64, kind=1, leaky=1, dt=1,
                sdt=0, stream=None)
    for kw, text in ((dict(), "checkpoints"), (dict(T=2, dx=None), "null pointer"), (dict(T=2, dxt=8), "overlap"),
                     (dict(T=2, dl=65536, di=65540), "overlap"), (dict(T=2, dx=4096), "one of the inputs"),
                     (dict(T=2, dg=16384), "one buffer")):
        a = dict(base, **kw)
        assert _lib.lib.snnb_gated_scan_backward(*a.values()) == 1
        assert text in _lib.lib.snnb_last_error().decode(), kw


def test_refusals_name_their_reason():
    x = torch.zeros(4, 2, 8)
    run = ops.run_temporal_gated_scan
    for args, kw, text in (((x, x), {}, "unsupported_device"), ((x[0], x[0]), {}, "unsupported_rank"),
                           ((x, x[:3]), {}, "unsupported_shape"), ((x, x.half()), {}, "unsupported_dtype"),
                           ((x.double(), x.double()), {}, "unsupported_dtype"), ((x, x), dict(gate="exp"), "unsupported_gate"),
                           ((x, x, torch.zeros(2, 9)), {}, "unsupported_shape"),
                           ((x, x, torch.zeros(2, 8).half()), {}, "unsupported_dtype"),
                           ((x, x), dict(lengths=torch.zeros(2)), "unsupported_dtype"),
                           ((x, x), dict(lengths=torch.zeros(3, dtype=torch.int32)), "unsupported_shape"),
                           ((x, x), dict(state_dtype=torch.float16), "unsupported_dtype"), (([x], x), {}, "expected a Tensor")):
        with pytest.raises(RuntimeError, match=text):
            run(*args, **kw)
    with pytest.raises(RuntimeError, match="dh_seq"):
        ops.run_temporal_gated_scan_backward(x[:2], x, x)
    long = torch.zeros(130, 1, 4)
    with pytest.raises(RuntimeError, match="ckpt"):
        ops.run_temporal_gated_scan_backward(long, long, long)


@gpu
def test_output_refusals_on_the_device():
    x = torch.zeros(4, 2, 8, device=DEV)
    with pytest.raises(RuntimeError, match="h_seq_out"):
        ops.run_temporal_gated_scan(x, x, h_seq_out=torch.zeros(4, 2, 9, device=DEV))
    with pytest.raises(RuntimeError, match="h_last_out"):
        ops.run_temporal_gated_scan(x, x, h_last_out=torch.zeros(2, 8, device=DEV).half())
    with pytest.raises(RuntimeError, match="overlap"):
        ops.run_temporal_gated_scan(x, x, h_seq_out=torch.zeros(1, 2, 8, device=DEV).expand(4, 2, 8))


def test_states_that_are_no_tensors_are_refused():
    """A carried state is a tensor, a 0-dim tensor or None; anything else was once taken for zeros without a word."""
    x = torch.zeros(4, 2, 8)
    for bad in (1.0, [[0.0] * 8] * 2, "zeros"):
        with pytest.raises(RuntimeError, match="h_init is"):
            ops.run_temporal_gated_scan(x, x, bad)
        with pytest.raises(RuntimeError, match="h_init is"):
            ops.run_temporal_gated_scan_backward(x, x, x, bad)
        with pytest.raises(RuntimeError, match="dh_last is"):
            ops.run_temporal_gated_scan_backward(x, x, x, dh_last=bad)


@gpu
def test_outputs_that_are_no_tensors_are_refused():
    x = torch.zeros(4, 2, 8, device=DEV)
    for bad in ([0.0], 1.0):
        with pytest.raises(RuntimeError, match="unsupported_output: h_seq_out"):
            ops.run_temporal_gated_scan(x, x, h_seq_out=bad)
        with pytest.raises(RuntimeError, match="unsupported_output: h_last_out"):
            ops.run_temporal_gated_scan(x, x, h_last_out=bad)


def test_gates_of_other_kinds_are_refused():
    x = torch.zeros(4, 2, 8)
    for bad in (None, 1, ["sigmoid"], {}):
        with pytest.raises(RuntimeError, match="unsupported_gate"):
            ops.run_temporal_gated_scan(x, x, gate=bad)


@gpu
@pytest.mark.parametrize("T", [6, 60, 500, 3000])
@pytest.mark.parametrize("D", [64, 65])
def test_an_infinite_state_stays_in_its_channel_and_its_future(T, D):
    """Small gates, whose products over a tile are 0 in fp32: the state stays infinite or becomes NaN, never a number again;
    the steps before it and the other channels are those of a clean input, and so for an infinite gradient the other way."""
    x, gate, _, dh, _ = _inputs(T, 2, D, torch.float32, "sigmoid", carry=False)
    x, gate, dh = x.to(DEV), (gate - 5).to(DEV), dh.to(DEV)
    clean = ops.run_temporal_gated_scan(x, gate, save_for_backward=True)
    t = T // 2
    x2 = x.clone()
    x2[t, 1, 5] = float("inf")
    h = ops.run_temporal_gated_scan(x2, gate).h_seq
    assert not bool(torch.isfinite(h[t:, 1, 5]).any()) and float(h[t, 1, 5]) == float("inf")
    h[t:, 1, 5] = clean.h_seq[t:, 1, 5]
    assert torch.equal(h, clean.h_seq)
    want = ops.run_temporal_gated_scan_backward(dh, x, gate, None, clean.ckpt)
    dh2 = dh.clone()
    dh2[t, 1, 5] = -float("inf")
    got = ops.run_temporal_gated_scan_backward(dh2, x, gate, None, clean.ckpt)
    assert not bool(torch.isfinite(got.dx[:t + 1, 1, 5]).any()) and not bool(torch.isfinite(got.dh_init[1, 5]))
    got.dx[:t + 1, 1, 5] = want.dx[:t + 1, 1, 5]
    got.dgate[:t + 1, 1, 5] = want.dgate[:t + 1, 1, 5]
    got.dh_init[1, 5] = want.dh_init[1, 5]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("T,B,D", [(0, 2, 8), (5, 0, 8), (5, 2, 0), (200, 0, 8), (0, 0, 0)])
@pytest.mark.parametrize("batch_first", [True, False])
def test_empty_sizes(T, B, D, batch_first):
    """Nothing to compute: outputs of the right shapes, and without a step the state is handed on."""
    x = torch.randn((B, T, D) if batch_first else (T, B, D), device=DEV)
    h0, dl = torch.randn(B, D, device=DEV), torch.randn(B, D, device=DEV)
    f = ops.run_temporal_gated_scan(x, x, h0, batch_first=batch_first, save_for_backward=True)
    assert f.h_seq.shape == x.shape and f.h_last.shape == (B, D)
    r = ops.run_temporal_gated_scan_backward(x, x, x, h0, f.ckpt, dh_last=dl, batch_first=batch_first)
    assert r.dx.shape == x.shape and r.dgate.shape == x.shape and r.dh_init.shape == (B, D)
    if T == 0:
        assert torch.equal(f.h_last, h0) and torch.equal(r.dh_init, dl)
    n = torch.zeros(B, dtype=torch.int32, device=DEV)
    f = ops.run_temporal_gated_scan(x, x, h0, batch_first=batch_first, lengths=n)
    assert torch.equal(f.h_last, h0) and not bool(f.h_seq.any())


@gpu
@pytest.mark.parametrize("D", [64, 61])
def test_one_step_of_a_padded_batch(D):
    """A decoding step in which some sequences have ended: their state stays and their row is zero."""
    _check(1, 5, D, torch.bfloat16, "sigmoid", True, lengths=[1, 0, 1, 0, 3], batch_first=True)
    _check(1, 5, D, torch.float32, "value", False, lengths=[0, 0, 1, -1, 1])
