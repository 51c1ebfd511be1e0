"""What the gated linear recurrence and AdamW refuse, through the Python layer and the C entry points, and the recurrence's
gradient formulas against differences.  Nothing here needs a GPU: every refusal comes before a launch."""
import ctypes

import numpy as np
import pytest
import torch

from tests import glr_reference as ref


@pytest.fixture(scope="module")
def hip():
    from baselines_amd import hip
    return hip


@pytest.fixture(scope="module")
def _lib():
    from baselines_amd import _lib
    return _lib


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


# -- recurrence ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("resets", [False, True])
def test_gradient_formulas_agree_with_differences(resets):
    """Central differences of the 64-bit forward pass: their own error is the step squared (1e-5 squared times derivatives of
    order one) and the rounding of a sum of 100 terms over the step, 100 * 1e-16 / 1e-5 = 1e-9."""
    g = torch.Generator().manual_seed(3)
    T, E, H = 9, 2, 3
    f, x, w = (torch.randn(T, E, H, generator=g, dtype=torch.float64) for _ in range(3))
    h0, wl = (torch.randn(E, H, generator=g, dtype=torch.float64) for _ in range(2))
    b = torch.randn(H, generator=g, dtype=torch.float64)
    r = torch.rand(T, E, generator=g) < 0.3 if resets else None
    if resets:
        r[0, 0] = True
    loss = lambda: float((ref.forward(f, x, h0, r, b)[0] * w).sum() + (ref.forward(f, x, h0, r, b)[1] * wl).sum())      # noqa: E731
    df, dx, dh0, dbias = ref.backward(f, x, h0, r, b, w, wl)
    for t, grad in ((f, df), (x, dx), (h0, dh0), (b, dbias)):
        flat, gflat = t.view(-1), grad.reshape(-1)
        for i in range(flat.numel()):
            keep = float(flat[i])
            flat[i] = keep + 1e-5
            up = loss()
            flat[i] = keep - 1e-5
            down = loss()
            flat[i] = keep
            assert abs((up - down) / 2e-5 - float(gflat[i])) < 1e-7


def test_forward_refusals(hip):
    f, x = z(4, 3, 8), z(4, 3, 8)
    for bad, err in (
            (dict(x=z(4, 8)), TypeError), (dict(x=z(4, 3, 8, dtype=torch.float64)), TypeError), (dict(x=None), TypeError),
            (dict(f=z(4, 3, 8, dtype=torch.bfloat16)), TypeError), (dict(f=z(4, 3, 7)), ValueError), (dict(f=None), TypeError),
            (dict(f=z(4, 8, 3).transpose(1, 2)), ValueError),
            (dict(resets=z(4, 3)), TypeError), (dict(resets=z(3, 4, dtype=torch.bool)), ValueError),
            (dict(bias=z(8, dtype=torch.bfloat16)), TypeError), (dict(bias=z(7)), ValueError), (dict(bias=z(16)[::2]), ValueError),
            (dict(h0=z(3, 8, dtype=torch.float64)), TypeError), (dict(h0=z(8, 3)), ValueError), (dict(h0=z(8, 3).t()), ValueError),
            (dict(y=z(4, 3, 8, dtype=torch.float16)), TypeError), (dict(y=x), ValueError), (dict(y=f), ValueError),
            (dict(y=z(1, 3, 8).expand(4, 3, 8)), ValueError), (dict(y=z(4, 3, 9)[..., :8].as_strided((4, 3, 8), (24, 7, 1))), ValueError),
            (dict(h_last=z(3, 7)), ValueError)):
        args = dict(f=f, x=x)
        args.update(bad)
        with pytest.raises(err):
            hip.glr_forward(**args)
    h0 = z(3, 8)
    with pytest.raises(ValueError, match="h_last overlaps h0"):
        hip.glr_forward(f, x, h0=h0, h_last=h0)
    joint = z(4, 3, 24)
    with pytest.raises(ValueError, match="y overlaps f"):
        hip.glr_forward(joint[..., :8], joint[..., 8:16], y=joint[..., 4:12])
    # rows that take turns in one buffer are told apart: this gets as far as the missing GPU
    with pytest.raises(TypeError, match="device tensor"):
        hip.glr_forward(joint[..., :8], joint[..., 8:16], y=joint[..., 16:])
    with pytest.raises(TypeError, match="device tensor"):
        hip.glr_forward(f, x)


def test_step_refusals(hip):
    f, x, s = z(3, 8), z(3, 8), z(3, 8)
    for bad, err in ((dict(x=z(1, 3, 8)), TypeError), (dict(f=z(3, 7)), ValueError), (dict(f=z(3, 8, dtype=torch.float16)), TypeError),
                     (dict(state=None), TypeError), (dict(state=z(3, 8, dtype=torch.bfloat16)), TypeError), (dict(state=z(3, 9)[:, :8]), ValueError),
                     (dict(resets=z(3)), TypeError), (dict(resets=z(4, dtype=torch.bool)), ValueError), (dict(bias=z(3)), ValueError),
                     (dict(y=s), ValueError), (dict(y=x), ValueError), (dict(f=z(8, 3).t()), ValueError)):
        args = dict(f=f, x=x, state=s)
        args.update(bad)
        with pytest.raises(err):
            hip.glr_step(**args)
    with pytest.raises(TypeError, match="device tensor"):
        hip.glr_step(f, x, s)


def test_backward_refusals(hip):
    f, x, dy = z(20, 3, 8), z(20, 3, 8), z(20, 3, 8)
    saved = hip.GlrSaved(z(2, 3, 8), x.shape, x.dtype)
    for bad, err in ((dict(saved=None), TypeError), (dict(saved=hip.GlrSaved(z(2, 3, 8), (19, 3, 8), x.dtype)), ValueError),
                     (dict(saved=hip.GlrSaved(z(2, 3, 8), x.shape, torch.float16)), ValueError), (dict(dy=z(20, 3, 7)), ValueError),
                     (dict(dh_last=z(3, 7)), ValueError), (dict(df=dy), ValueError), (dict(dx=f), ValueError), (dict(df=x), ValueError)):
        args = dict(f=f, x=x, dy=dy, saved=saved)
        args.update(bad)
        with pytest.raises(err):
            hip.glr_backward(**args)
    d = z(20, 3, 8)
    with pytest.raises(ValueError, match="dx overlaps df"):
        hip.glr_backward(f, x, dy, saved, df=d, dx=d)
    with pytest.raises(TypeError, match="device tensor"):
        hip.glr_backward(f, x, dy, saved)


def test_c_entry_refuses_bad_recurrences(_lib):
    L, one = _lib.lib, ctypes.c_void_p(256)
    seq, null, neg = _lib.Seq(256, 24, 8), _lib.Seq(None, 24, 8), _lib.Seq(256, -1, 8)
    fwd = lambda dt=0, T=4, E=3, H=8, f=seq, x=seq, r=None, h0=None, y=seq, hl=None: L.ppo2hip_glr_forward(      # noqa: E731
        dt, T, E, H, f, x, None, r, h0, y, hl, None, None, 0, None)
    for kw in (dict(dt=3), dict(dt=-1), dict(T=-1), dict(E=-1), dict(H=-1), dict(E=1 << 16, H=1 << 15), dict(f=null), dict(x=None), dict(y=neg),
               dict(r=null), dict(h0=one, hl=one)):
        assert fwd(**kw) == _lib.EINVAL and L.ppo2hip_last_error(), kw
    assert fwd(E=0) == 0 and fwd(H=0) == 0 and fwd(T=0) == 0
    bwd = lambda saved=one, dy=seq, dhl=None, dh0=None, dbias=None: L.ppo2hip_glr_backward(      # noqa: E731
        0, 4, 3, 8, seq, seq, None, None, saved, dy, dhl, seq, seq, dbias, dh0, None, 0, None)
    assert bwd(saved=None) == _lib.EINVAL
    assert bwd(dy=null) == _lib.EINVAL
    assert bwd(dhl=one, dh0=one) == _lib.EINVAL
    assert bwd(dbias=one) == _lib.ENOSPACE
    assert L.ppo2hip_glr_saved_floats(33, 2, 5) == 3 * 10 and L.ppo2hip_glr_saved_floats(0, 2, 5) == 0


# -- AdamW --------------------------------------------------------------------------------------------------------------

def test_plan_refusals(hip):
    p = z(5, 4)
    for args, err in (((([],), {}), ValueError), ((([p, p],), {}), ValueError), ((([p, p.view(-1)[3:7]],), {}), ValueError),
                      ((([z(4, dtype=torch.float16)],), {}), TypeError), ((([p, 3.0],), {}), TypeError), ((([z(4, 5).t()],), {}), ValueError),
                      ((([p],), dict(state_bits=4)), ValueError), ((([p],), dict(decay=[1, 0])), ValueError),
                      ((([p],), dict(grad_dtype=torch.float16)), TypeError)):
        with pytest.raises(err):
            hip.AdamWPlan(*args[0], **args[1])
    with pytest.raises(TypeError, match="GPU"):
        hip.AdamWPlan([p])


def test_c_entry_refuses_bad_lists(_lib):
    L = _lib.lib
    T = _lib.AdamwTensor
    good = (T * 2)(T(256, 300, 0, 0, 1.0, 0), T(4096, 1, 1, 1, 0.0, 0))
    assert L.ppo2hip_adamw_state_elements(good, 2, 32) == 301
    assert L.ppo2hip_adamw_state_elements(good, 2, 8) == 512 + 256
    for bad in (T(None, 3, 0, 0, 1, 0), T(256, -1, 0, 0, 1, 0), T(256, 3, 2, 0, 1, 0), T(256, 3, 0, 2, 1, 0)):
        assert L.ppo2hip_adamw_state_elements((T * 1)(bad), 1, 32) == _lib.EINVAL
    assert L.ppo2hip_adamw_state_elements(good, 2, 16) == _lib.EINVAL
    need = L.ppo2hip_adamw_plan_bytes(good, 2)
    buf = np.zeros(need, np.uint8)
    assert L.ppo2hip_adamw_plan_fill(good, 2, 32, buf.ctypes.data, need - 1) == _lib.ENOSPACE
    assert L.ppo2hip_adamw_plan_fill(good, 2, 32, None, need) == _lib.EINVAL
    assert L.ppo2hip_adamw_plan_fill(good, 2, 32, buf.ctypes.data, need) == 0
    one, grads = ctypes.c_void_p(256), (ctypes.c_void_p * 2)(256, 256)
    step = lambda bits=32, plan=one, g=grads, m=one, ms=None, v=one, vs=None, t=1, b1=.9, b2=.999, eps=1e-8, clip=0.0: L.ppo2hip_adamw_step(      # noqa: E731,E501
        good, 2, bits, plan, g, m, ms, v, vs, 1e-3, t, b1, b2, eps, 0.0, 1.0, clip, None, None, 0, None)
    for kw in (dict(bits=16), dict(plan=None), dict(g=None), dict(m=None), dict(v=None), dict(t=0), dict(b1=1.0), dict(b1=-.1), dict(b2=1.0),
               dict(eps=-1.0), dict(bits=8), dict(bits=8, ms=one)):
        assert step(**kw) == _lib.EINVAL and L.ppo2hip_last_error(), kw
    assert step(clip=1.0) == _lib.ENOSPACE
    assert L.ppo2hip_adamw_state(good, 2, one, one, one, one, one, 2, one, one, None) == _lib.EINVAL
    assert L.ppo2hip_adamw_state(good, 2, one, one, None, one, one, 0, one, one, None) == _lib.EINVAL


def test_c_entry_refuses_what_a_launch_or_a_lane_cannot_address(_lib):
    """Lanes carry 32-bit byte offsets and a launch 2^32 threads: sizes beyond either are refused before anything runs."""
    L, one = _lib.lib, ctypes.c_void_p(256)
    seq = _lib.Seq(256, 0, 0)
    fwd = lambda T, E, H, dt=0: L.ppo2hip_glr_forward(dt, T, E, H, seq, seq, None, None, None, seq, None, None, one, 1 << 62, None)      # noqa: E731
    bwd = lambda T, E, H, dt=0: L.ppo2hip_glr_backward(      # noqa: E731
        dt, T, E, H, seq, seq, None, None, one, seq, None, seq, seq, None, None, one, 1 << 62, None)
    for call in (fwd, bwd):
        for T, E, H in ((2, 1, 1 << 26), (1000, 31, (1 << 26) - 1), (1000, 1 << 30, 1), (1 << 30, 1 << 20, 1)):
            assert call(T, E, H) == _lib.EINVAL and L.ppo2hip_last_error(), (T, E, H)
    # tiles of 64 columns, a workgroup of 1024 threads each: 2^22 of them
    assert fwd(256, 1 << 5, 1 << 23) == _lib.EINVAL and b"one launch" in L.ppo2hip_last_error()


def test_c_entry_refuses_lists_and_norms_that_do_not_fit(_lib):
    L, one = _lib.lib, ctypes.c_void_p(256)
    T = _lib.AdamwTensor
    long = (T * 2)(T(256, 1 << 34, 0, 0, 1.0, 0), T(4096, 1 << 34, 0, 0, 1.0, 0))
    assert L.ppo2hip_adamw_state_elements(long, 1, 32) == 1 << 34
    assert L.ppo2hip_adamw_state_elements(long, 2, 32) == _lib.EINVAL and b"elements in one list" in L.ppo2hip_last_error()
    good, grads = (T * 1)(T(256, 300, 0, 0, 1.0, 0)), (ctypes.c_void_p * 1)(256)
    step = lambda clip, plan=one, ws=one: L.ppo2hip_adamw_step(      # noqa: E731
        good, 1, 32, plan, grads, one, None, one, None, 1e-3, 1, .9, .999, 1e-8, 0.0, 1.0, clip, None, ws, 1 << 20, None)
    for clip in (1e-60, float("nan")):
        assert step(clip) == _lib.EINVAL and b"max_grad_norm" in L.ppo2hip_last_error()
    assert step(1.0, ws=ctypes.c_void_p(264)) == _lib.EINVAL and step(1.0, plan=ctypes.c_void_p(264)) == _lib.EINVAL


def test_c_entry_refuses_bad_steps(_lib):
    L, one = _lib.lib, ctypes.c_void_p(256)
    step = lambda dt=0, E=3, H=8, f=one, fe=8, x=one, r=None, re=1, s=one, y=one: L.ppo2hip_glr_step(      # noqa: E731
        dt, E, H, f, fe, x, 8, None, r, re, s, y, 8, None)
    for kw in (dict(dt=3), dict(E=-1), dict(H=-1), dict(H=1 << 26), dict(f=None), dict(x=None), dict(y=None), dict(s=None), dict(fe=-8),
               dict(r=one, re=-1)):
        assert step(**kw) == _lib.EINVAL and L.ppo2hip_last_error(), kw
    assert step(E=0, s=None) == 0 and step(H=0) == 0


def test_a_state_in_place_meets_no_input(hip):
    """glr_step writes the state while other workgroups still read: an input in the state's memory is refused, one beside it is not."""
    E, H = 3, 8
    buf = z(200)
    state = buf[40:64].view(E, H)
    f, x = z(E, H), z(E, H)
    rows = lambda at, step: buf.as_strided((E, H), (step, 1), at)      # noqa: E731
    flags = lambda at, step: buf.view(torch.uint8).as_strided((E,), (step,), at)      # noqa: E731
    for bad in (dict(x=state), dict(f=state), dict(x=rows(48, 8)), dict(f=rows(33, 0)), dict(x=rows(63, 8)), dict(f=rows(0, 20)), dict(f=rows(25, 9)),
                dict(bias=buf[33:41]), dict(bias=buf[63:71]), dict(resets=flags(159, 1)[:E]), dict(resets=flags(100, 70)), dict(resets=flags(255, 1))):
        args = dict(f=f, x=x, state=state)
        args.update(bad)
        with pytest.raises(ValueError, match="state overlaps %s" % list(bad)[0]):
            hip.glr_step(**args)
    # as far as the missing GPU
    for good in (dict(x=rows(64, 8)), dict(f=rows(16, 8)), dict(x=rows(32, 32)), dict(bias=buf[32:40]), dict(bias=buf[64:72]),
                 dict(resets=flags(157, 1)), dict(resets=flags(256, 1)), dict(resets=flags(159, 97))):
        args = dict(f=f, x=x, state=state)
        args.update(good)
        with pytest.raises(TypeError, match="device tensor"):
            hip.glr_step(**args)
    for shape in ((0, 8), (3, 0)):
        with pytest.raises(TypeError, match="device tensor"):
            hip.glr_step(z(*shape), z(*shape), z(*shape))
