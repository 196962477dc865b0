"""laya_rope on the B200 against the rotation in 64 bits.

Tolerance, per element: with |a|, |b| the pair's values and m the factor on cos
and sin, the kernel's f32 cosine and sine are off by at most 2^-33 turn of
angle (7e-10), half a step of the reduced argument (pi/4 * 2^-24) and two steps
of sincospi (2^-23), together under 1.8e-7; the factor and the two products and
sum add four roundings of 2^-24.  So |error| <= 4.3e-7 m (|a| + |b|) before the
last rounding, which is off by at most eps/2 of the value (or 2^-25 for f16
values under its normal range).
"""
import math

import numpy as np
import pytest
import torch

from laya_rust_b200 import engine as E
from laya_rust_b200 import modelgen, ops, workloads

pytestmark = pytest.mark.gpu
DT = {ops.F16: torch.float16, ops.BF16: torch.bfloat16, ops.F32: torch.float32}


def oracle(x, pos, freqs, rot, layout, inverse, m):
    """(rotated in 64 bits, error bound before the last rounding)."""
    x = x.double().cpu()
    ang = pos.double().cpu()[:, None] * torch.from_numpy(np.asarray(freqs))[None, :]
    c, s = m * torch.cos(ang)[:, None, :], m * torch.sin(ang)[:, None, :] * (-1 if inverse else 1)
    out, tol = x.clone(), torch.zeros_like(x)
    i = np.arange(rot // 2)
    i0, i1 = (i, i + rot // 2) if layout == ops.ROPE_HALF else (2 * i, 2 * i + 1)
    a, b = x[..., i0], x[..., i1]
    out[..., i0], out[..., i1] = a * c - b * s, b * c + a * s
    tol[..., i0] = tol[..., i1] = 4.3e-7 * m * (a.abs() + b.abs())
    return out, tol


def check(got, want, tol):
    half_step = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    err = (got.double().cpu() - want).abs()
    lim = tol + half_step * (want.abs() + tol) + tiny
    assert bool((err <= lim).all()), float((err - lim).max())


def view(t):
    return t.data_ptr(), t.stride(0), t.stride(1)


def rt(x, out):
    return ops.RopeTensor(x.data_ptr(), out.data_ptr(), x.shape[1], x.stride(0), x.stride(1), out.stride(0), out.stride(1))


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("type", [ops.F16, ops.BF16, ops.F32])
@pytest.mark.parametrize("layout", [ops.ROPE_HALF, ops.ROPE_INTERLEAVED])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 64, 64), (1, 32, 64, 64), (5, 3, 64, 32), (33, 16, 64, 64),
                                                  (7, 2, 80, 20), (9, 5, 18, 6), (3, 1, 2, 2), (300, 12, 128, 128),
                                                  (2, 3, 512, 512), (17, 4, 96, 48), (3, 2, 511, 2), (40, 2, 510, 300), (1000, 40, 256, 256), (700, 70, 64, 64), (130, 40, 128, 64), (11, 7, 37, 36)])
def test_against_64_bits(type, layout, tokens, heads, dim, rot):
    g = torch.Generator(device="cuda").manual_seed(tokens * 1000 + dim + rot)
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(DT[type])
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    freqs, _ = ops.rope_freqs(10000.0, rot)
    for inverse, m in ((False, 1.0), (True, 1.25)):
        out = torch.full_like(x, float("nan"))
        ops.rope(ops.RopeSpec(type, dim, rot, freqs, layout, inverse, m), [rt(x, out)], tokens, pos=pos.data_ptr(),
                 stream=stream())
        check(out, *oracle(x, pos, freqs, rot, layout, inverse, m))


@pytest.mark.parametrize("type", [ops.F16, ops.BF16, ops.F32])
@pytest.mark.parametrize("layout", [ops.ROPE_HALF, ops.ROPE_INTERLEAVED])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(50, 6, 40, 24), (50, 6, 64, 24), (9, 3, 120, 40), (900, 7, 24, 24), (5, 1, 56, 8),
                                                  (3000, 40, 128, 64), (700, 20, 96, 80), (33, 5, 511, 510), (20000, 9, 64, 64),
                                                  (4, 6, 512, 8), (2, 3, 500, 2)])
def test_odd_numbers_of_pieces(type, layout, inplace, tokens, heads, dim, rot):
    """Turned and copied parts that are an odd number of pieces, and walks of many tiles."""
    x = torch.randn(tokens, heads, dim, device="cuda").to(DT[type])
    out = x.clone() if inplace else torch.full_like(x, float("nan"))
    freqs, _ = ops.rope_freqs(10000.0, rot)
    ops.rope(ops.RopeSpec(type, dim, rot, freqs, layout), [rt(out if inplace else x, out)], tokens, pos0=3, stream=stream())
    check(out, *oracle(x, torch.arange(3, 3 + tokens), freqs, rot, layout, False, 1.0))
    assert torch.equal(out[..., rot:], x[..., rot:])


def test_far_and_negative_positions():
    freqs, _ = ops.rope_freqs(10000.0, 64)
    pos = torch.tensor([0, 1, -1, 2**31 - 1, -2**31, 2**30 + 7, 123456789, -987654321], dtype=torch.int32, device="cuda")
    x = torch.randn(8, 2, 64, device="cuda")
    out = torch.empty_like(x)
    ops.rope(ops.RopeSpec(ops.F32, 64, 64, freqs), [rt(x, out)], 8, pos=pos.data_ptr(), stream=stream())
    # the oracle's own product rounds at 2^31 radians by 2^-22 (f64: 2^-53 relative); the kernel's frequency by 2^31 2^-65 turn
    want, tol = oracle(x, pos, freqs, 64, ops.ROPE_HALF, False, 1.0)
    far = (pos.double().abs() * 2.0 ** -52).cpu()[:, None, None] * (x.double().abs().cpu().amax() * 2)
    check(out, want, tol + far)


def test_counted_positions_and_four_tensors_in_one_launch():
    freqs, _ = ops.rope_freqs(160000.0, 64)
    xs = [torch.randn(77, h, 64, device="cuda").half() for h in (16, 1, 5, 8)]
    outs = [torch.empty_like(x) for x in xs]
    ops.rope(ops.RopeSpec(ops.F16, 64, 64, freqs), [rt(x, o) for x, o in zip(xs, outs)], 77, pos0=1000, stream=stream())
    pos = torch.arange(1000, 1077, dtype=torch.int32)
    for x, o in zip(xs, outs):
        check(o, *oracle(x, pos, freqs, 64, ops.ROPE_HALF, False, 1.0))


@pytest.mark.parametrize("layout", [ops.ROPE_HALF, ops.ROPE_INTERLEAVED])
def test_in_place_in_a_packed_buffer_touches_nothing_else(layout):
    """q and k columns of a q|k|v buffer whose rows are wider still; v, the row
    tails, the unrotated dims and the rows behind the last token stay."""
    T, H, D, R = 40, 4, 64, 32
    freqs, _ = ops.rope_freqs(10000.0, R)
    buf = torch.randn(T + 9, 3 * H * D + 24, device="cuda").to(torch.bfloat16)
    keep = buf.clone()
    q, k = (buf[:, i * H * D:(i + 1) * H * D].unflatten(1, (H, D)) for i in (0, 1))
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    ops.rope(ops.RopeSpec(ops.BF16, D, R, freqs, layout), [rt(q, q), rt(k, k)], T, pos=pos.data_ptr(), stream=stream())
    for i, v in ((0, q), (1, k)):
        was = keep[:T, i * H * D:(i + 1) * H * D].unflatten(1, (H, D))
        check(v[:T], *oracle(was, pos, freqs, R, layout, False, 1.0))
        assert torch.equal(v[:T, :, R:], was[:, :, R:])
    assert torch.equal(buf[:, 2 * H * D:], keep[:, 2 * H * D:]) and torch.equal(buf[T:], keep[T:])


@pytest.mark.parametrize("type", [ops.F16, ops.F32])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 4])
def test_odd_strides_offsets_and_orders(type, shift):
    """Head-major inputs, odd strides, views that start off every alignment."""
    T, H, D, R = 13, 3, 24, 16
    es = 2 if type == ops.F16 else 4
    freqs, _ = ops.rope_freqs(10000.0, R)
    raw = torch.randn(H * (T * 27 + 5) + 8, device="cuda").to(DT[type])
    x = raw[shift:].as_strided((T, H, D), (27, T * 27 + 5, 1))
    oraw = torch.full((T * (H * 31 + 3) + 8,), 7.0, device="cuda", dtype=DT[type])
    o = oraw[shift:].as_strided((T, H, D), (H * 31 + 3, 31, 1))
    assert x.data_ptr() % es == 0
    for layout in (ops.ROPE_HALF, ops.ROPE_INTERLEAVED):
        oraw.fill_(7.0)
        ops.rope(ops.RopeSpec(type, D, R, freqs, layout), [rt(x, o)], T, pos0=5, stream=stream())
        check(o, *oracle(x, torch.arange(5, 5 + T), freqs, R, layout, False, 1.0))
        left = torch.ones_like(oraw, dtype=torch.bool)
        left[shift:].as_strided((T, H, D), (H * 31 + 3, 31, 1)).fill_(False)
        assert bool((oraw[left] == 7.0).all())


@pytest.mark.parametrize("type", [ops.F16, ops.F32])
def test_offsets_past_32_bits(type):
    """Heads, then tokens, more than 2^32 elements apart."""
    far = (1 << 32) + 8
    freqs, _ = ops.rope_freqs(10000.0, 32)
    raw = torch.empty(far + 3 * 48, device="cuda", dtype=DT[type])
    wide, near = raw.as_strided((3, 2, 48), (48, far, 1)), torch.randn(3, 2, 48, device="cuda").to(DT[type])
    ops.rope(ops.RopeSpec(type, 48, 32, freqs), [rt(near, wide)], 3, pos0=9, stream=stream())
    check(wide, *oracle(near, torch.arange(9, 12), freqs, 32, ops.ROPE_HALF, False, 1.0))
    wide = raw.as_strided((2, 3, 48), (far, 48, 1))
    wide.copy_(torch.randn(2, 3, 48, device="cuda"))
    near = torch.empty(2, 3, 48, device="cuda", dtype=DT[type])
    ops.rope(ops.RopeSpec(type, 48, 32, freqs), [rt(wide, near)], 2, pos0=9, stream=stream())
    check(near, *oracle(wide, torch.arange(9, 11), freqs, 32, ops.ROPE_HALF, False, 1.0))
    del raw, wide
    torch.cuda.empty_cache()


def test_many_tokens_of_one_pair():
    n = 3000001
    x, o = torch.randn(n, 1, 2, device="cuda"), torch.empty(n, 1, 2, device="cuda")
    ops.rope(ops.RopeSpec(ops.F32, 2, 2, [0.37]), [rt(x, o)], n, stream=stream())
    check(o, *oracle(x, torch.arange(n), [0.37], 2, ops.ROPE_HALF, False, 1.0))


def test_repeated_input_rows():
    """Stride 0 over heads: one key read for every head."""
    freqs, _ = ops.rope_freqs(10000.0, 64)
    x = torch.randn(6, 1, 64, device="cuda").half()
    o = torch.empty(6, 8, 64, device="cuda", dtype=torch.float16)
    xe = x.expand(6, 8, 64)
    ops.rope(ops.RopeSpec(ops.F16, 64, 64, freqs), [rt(xe, o)], 6, stream=stream())
    check(o, *oracle(xe, torch.arange(6), freqs, 64, ops.ROPE_HALF, False, 1.0))


def test_inverse_is_the_gradient():
    """The gradient of sum(w . rope(x)) is the inverse rotation of w: against
    autograd of the rotation in 64 bits, and against differences."""
    T, H, D, R = 5, 2, 32, 20
    freqs, _ = ops.rope_freqs(10000.0, R)
    w = torch.randn(T, H, D, device="cuda")
    dx = torch.empty_like(w)
    ops.rope(ops.RopeSpec(ops.F32, D, R, freqs, ops.ROPE_INTERLEAVED, True, 1.5), [rt(w, dx)], T, pos0=3, stream=stream())
    x = torch.randn(T, H, D, dtype=torch.float64, requires_grad=True)
    pos = torch.arange(3, 3 + T)

    def f(v):
        ang = pos.double()[:, None] * torch.from_numpy(freqs)[None]
        z = torch.view_as_complex(v[..., :R].unflatten(-1, (R // 2, 2)).contiguous()) * torch.polar(
            torch.full_like(ang, 1.5), ang)[:, None]
        return (torch.cat([torch.view_as_real(z).flatten(-2), v[..., R:]], -1) * w.double().cpu()).sum()

    f(x).backward()
    check(dx, x.grad, 4.3e-7 * 1.5 * 2 * w.double().cpu().abs().amax() * torch.ones_like(x.grad))
    with torch.no_grad():
        for idx in ((0, 0, 0), (2, 1, 7), (4, 0, 19), (3, 1, 31)):
            e = torch.zeros_like(x)
            e[idx] = 0.5          # f is linear: a difference of any width is exact to 64-bit rounding
            assert abs(float(f(x + e) - f(x - e)) - float(dx[idx])) < 1e-5


def test_infinities_and_nan_stay_in_their_pair():
    freqs, _ = ops.rope_freqs(10000.0, 64)
    x = torch.randn(3, 2, 64, device="cuda")
    clean = torch.empty_like(x)
    ops.rope(ops.RopeSpec(ops.F32, 64, 64, freqs), [rt(x, clean)], 3, pos0=1, stream=stream())
    x[1, 0, 5], x[2, 1, 40] = float("nan"), float("inf")
    out = torch.empty_like(x)
    ops.rope(ops.RopeSpec(ops.F32, 64, 64, freqs), [rt(x, out)], 3, pos0=1, stream=stream())
    hit = torch.zeros_like(x, dtype=torch.bool)
    for t, h, d in ((1, 0, 5), (1, 0, 37), (2, 1, 40), (2, 1, 8)):
        hit[t, h, d] = True
    assert bool((~torch.isfinite(out[hit])).all()) and torch.equal(out[~hit], clean[~hit])


def test_another_stream_and_a_replayed_graph():
    freqs, _ = ops.rope_freqs(10000.0, 64)
    sp = ops.RopeSpec(ops.F16, 64, 64, freqs)
    x = torch.randn(50, 16, 64, device="cuda").half()
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.rope(sp, [rt(x, out)], 50, pos=pos.data_ptr(), stream=s.cuda_stream)
    s.synchronize()
    check(out, *oracle(x, pos, freqs, 64, ops.ROPE_HALF, False, 1.0))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.rope(sp, [rt(x, out)], 50, pos=pos.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    x.copy_(torch.randn(50, 16, 64, device="cuda"))
    pos.add_(777)
    g.replay()
    torch.cuda.synchronize()
    check(out, *oracle(x, pos, freqs, 64, ops.ROPE_HALF, False, 1.0))


def test_memory_that_is_not_the_device_s_is_refused():
    freqs, _ = ops.rope_freqs(10000.0, 64)
    sp = ops.RopeSpec(ops.F32, 64, 64, freqs)
    dev, host = torch.randn(2, 1, 64, device="cuda"), torch.randn(2, 1, 64)
    pos = torch.zeros(2, dtype=torch.int32)
    for x, o, p in ((host, dev, 0), (dev, host, 0), (dev, dev, pos.data_ptr())):
        with pytest.raises(E.LayaError, match="not a device address"):
            ops.rope(sp, [rt(x, o)], 2, pos=p, stream=stream())
    with pytest.raises(E.LayaError, match="device out of range"):
        ops.rope(sp, [rt(dev, dev)], 2, device=torch.cuda.device_count(), stream=stream())


# ---- the engine with stretched frequencies --------------------------------------
@pytest.fixture(scope="module")
def engine():
    e = E.Engine(modelgen.cached_model(seed=0), device=0)
    yield e
    e.close()


def test_engine_scaling_on_and_off(engine):
    """Scaling changes the answers, a factor of 1 leaves them within the f32
    tables' own error, and taking it back restores every bit."""
    req = workloads.long_state(seed=3)
    base = engine.forward(req)
    try:
        ops.set_rope_scaling(engine, ops.RopeScaling(ops.ROPE_LINEAR, 1.0), ops.RopeScaling(ops.ROPE_LINEAR, 1.0))
        same = engine.forward(req)
        ops.set_rope_scaling(engine, ops.RopeScaling(ops.ROPE_PARTS, 8.0, 512.0, 1.0, 32.0))
        far = [engine.forward(req) for _ in range(3)]          # eager, captured, replayed
    finally:
        ops.set_rope_scaling(engine)
    again = engine.forward(req)
    on = base.logits > -9999
    # angles differ by the model's own f32 product, at most 512 * 2^-24: far inside the f16 rounding of q and k
    assert np.abs(same.logits[on] - base.logits[on]).max() < 2e-2
    assert np.abs(far[0].logits[on] - base.logits[on]).max() > 1e-4
    for o in far[1:]:
        assert np.array_equal(o.logits, far[0].logits) and np.array_equal(o.act, far[0].act)
    assert np.array_equal(again.logits, base.logits) and np.array_equal(again.act, base.act)


def test_engine_layers_read_their_own_scaling(engine):
    """A stretch of the windowed layers' frequencies reaches a windowed layer
    and leaves a global one bit for bit."""
    req = workloads.long_state(seed=4)
    plan = engine.plan(req)
    x = np.random.default_rng(1).standard_normal((plan.stats()[0], 1024)).astype(np.float32)
    outs = []
    try:
        for f in (1.0, 2.0, 4.0):
            ops.set_rope_scaling(engine, None, ops.RopeScaling(ops.ROPE_LINEAR, f))
            plan.set_hidden(x)
            plan.run_layer(1)
            outs.append(plan.hidden())
            plan.set_hidden(x)
            plan.run_layer(3)          # a global layer: not scaled
            outs.append(plan.hidden())
    finally:
        ops.set_rope_scaling(engine)
        plan.close()
    assert np.array_equal(outs[1], outs[3]) and np.array_equal(outs[1], outs[5])
    assert np.abs(outs[0] - outs[2]).max() > 1e-3 and np.abs(outs[2] - outs[4]).max() > 1e-3


def test_engine_refuses_bad_scaling_and_keeps_its_tables(engine):
    req = workloads.long_state(seed=5)
    base = engine.forward(req)
    for bad in (ops.RopeScaling(ops.ROPE_LINEAR, 0.0), ops.RopeScaling(9, 2.0), ops.RopeScaling(ops.ROPE_PARTS, 2.0)):
        with pytest.raises(E.LayaError) as ei:
            ops.set_rope_scaling(engine, bad)
        assert ei.value.code == E.LAYA_E_INVALID
    assert np.array_equal(engine.forward(req).logits, base.logits)
